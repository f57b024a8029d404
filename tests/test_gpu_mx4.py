"""Microscaled 4-bit rows and products on the GPU (include/eif_hip_mx.h) against the definition in 64 bits."""
import numpy as np
import pytest

import mx4_ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}


def dev(a, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(getattr(torch, TYPES[dtype]))


def host(t):
    return t.cpu().numpy()


def rows_on_gpu(gpu, x, ldc=0, lds=0, values=True):
    """codes, scales, values of mx4_quant_rows, in buffers filled with 0xA5 / NaN."""
    import torch
    r, k = x.shape
    kp = mx4_ref.kpad(k)
    c = torch.full((r, max(ldc, kp // 2)), 0xA5, dtype=torch.uint8, device="cuda")
    s = torch.full((r, max(lds, kp // 32)), 0xA5, dtype=torch.uint8, device="cuda")
    v = torch.full((r, k), float("nan"), device="cuda") if values else None
    gpu.mx4_quant_rows(x, c, s, v)
    torch.cuda.synchronize()
    return c, s, v


def special_rows(rng, rows, cols):
    """Rows over the whole range of FP32, with ties, zeros, infinities and NaN in some blocks."""
    x = mx4_ref.activations(rng, rows, cols) * np.exp2(rng.integers(-140, 100, (rows, 1))).astype(np.float32)
    x = x.astype(np.float32)
    for r in range(rows):
        kind = r % 8
        b = 32 * int(rng.integers(0, -(-cols // 32)))
        at = b + int(rng.integers(0, min(32, cols - b)))
        if kind == 1:
            x[r] = 0.0
        elif kind == 2:
            x[r, at] = np.inf
        elif kind == 3:
            x[r, at] = np.nan
        elif kind == 4:
            x[r, at] = -np.inf
        elif kind == 5:   # multiples of an eighth of the scale: every tie
            x[r] = rng.integers(-64, 65, cols) / 8.0
        elif kind == 6:
            x[r] = -0.0
            x[r, at] = 3.4e38
        elif kind == 7:
            x[r] = rng.integers(-3, 4, cols) * 2.0 ** -149
    return x


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (16, 32), (17, 33), (9, 256), (8, 257), (5, 1000), (40, 2560), (1, 8192),
                                       (300, 511), (2, 20011)])
def test_quant_rows(gpu, type, rows, cols):
    rng = np.random.default_rng(rows * 1000 + cols)
    with np.errstate(over="ignore"):
        x = dev(special_rows(rng, rows, cols), type)
    c, s, v = rows_on_gpu(gpu, x)
    xh = host(x.float())
    wc, ws = mx4_ref.quantise(xh)
    assert np.array_equal(host(s), ws)
    assert np.array_equal(host(c), wc)
    want = mx4_ref.values(wc, ws, cols).astype(np.float32)
    got = host(v)
    assert np.array_equal(got, want, equal_nan=True)
    assert np.array_equal(np.signbit(got) | np.isnan(got), np.signbit(want) | np.isnan(want))


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,ldx,off", [(7, 300, 301, 0), (7, 300, 304, 1), (5, 64, 70, 3), (6, 512, 516, 4), (3, 1030, 1031, 1)])
def test_quant_strides(gpu, type, rows, cols, ldx, off):
    """Rows of any stride and alignment; operand rows of wider buffers, whose bytes beyond are left as they were."""
    import torch
    rng = np.random.default_rng(cols + off)
    buf = dev(mx4_ref.activations(rng, 1, rows * ldx + off)[0], type)
    x = torch.as_strided(buf, (rows, cols), (ldx, 1), off)
    kp = mx4_ref.kpad(cols)
    c, s, v = rows_on_gpu(gpu, x, kp // 2 + 48, kp // 32 + 24)
    wc, ws = mx4_ref.quantise(host(x.float()))
    assert np.array_equal(host(c)[:, :kp // 2], wc) and (host(c)[:, kp // 2:] == 0xA5).all()
    assert np.array_equal(host(s)[:, :kp // 32], ws) and (host(s)[:, kp // 32:] == 0xA5).all()
    # values alone, and codes alone
    alone = torch.full((rows, cols + 5), float("nan"), device="cuda")
    gpu.mx4_quant_rows(x, values=alone[:, 2:2 + cols])
    c2, s2, _ = rows_on_gpu(gpu, x, values=False)
    torch.cuda.synchronize()
    assert torch.equal(alone[:, 2:2 + cols], v) and alone[:, :2].isnan().all() and alone[:, 2 + cols:].isnan().all()
    assert torch.equal(c2, c[:, :kp // 2]) and torch.equal(s2, s[:, :kp // 32])


class Case:
    """A weight (a stack of `experts`), its values, and operand rows with theirs."""

    def __init__(self, gpu, seed, n, k, m, experts=1, on_device=True, edges=False):
        rng = np.random.default_rng(seed)
        w = mx4_ref.matrix(rng, experts * n, k)
        a = mx4_ref.activations(rng, m, k)
        if edges and m > 2:
            a[1] = 0.0
        wc, ws = mx4_ref.quantise(w)
        # the matrix comes in tight rows
        wc, ws = wc[:, :(k + 1) // 2].copy(), ws[:, :-(-k // 32)].copy()
        self.wv = mx4_ref.values(wc, ws, k).reshape(experts, n, k)
        wc, ws = wc.reshape(experts, n, -1), ws.reshape(experts, n, -1)
        self.w = gpu.Mx4Weight(n, k, dev(wc) if on_device else wc, dev(ws) if on_device else ws, experts=experts)
        self.a = a
        ac, as_ = mx4_ref.quantise(a)
        self.av = mx4_ref.values(ac, as_, k)
        self.ac, self.as_ = dev(ac), dev(as_)
        self.bias = rng.standard_normal((experts, n)).astype(np.float32)


def out(m, n, pad=0):
    import torch
    return torch.full((m, n + pad), float("nan"), device="cuda")[:, :n]


def check(y, want, tol):
    got = host(y).astype(np.float64)
    bad = ~(np.abs(got - want) <= tol) & ~(np.isnan(got) & np.isnan(want))
    assert not bad.any(), (np.argwhere(bad)[:5].tolist(), got[bad][:5], want[bad][:5], tol[bad][:5] if tol.shape == got.shape else tol)


LINEAR = [  # rows, cols, tokens
    (16, 32, 1), (1, 1, 1), (5, 7, 3), (17, 33, 2), (64, 256, 16), (100, 300, 17), (129, 1000, 31), (896, 4864, 1), (2560, 2560, 1),
    (4864, 896, 5), (300, 6912, 24), (2560, 1024, 33), (640, 2560, 63), (1152, 896, 64), (512, 512, 65), (257, 777, 127),
    (1000, 1536, 128), (2048, 2048, 129), (384, 4096, 200), (130, 257, 255), (1152, 896, 257), (2304, 2560, 512), (31, 8192, 300),
    (4096, 640, 700),
]


@pytest.mark.parametrize("n,k,m", LINEAR)
def test_linear(gpu, n, k, m):
    import torch
    c = Case(gpu, n + k + m, n, k, m, on_device=m % 2 == 0, edges=True)
    for bias in (None, c.bias[0]):
        y = out(m, n)
        c.w.linear(c.ac, c.as_, y, None if bias is None else dev(bias))
        torch.cuda.synchronize()
        check(y, *mx4_ref.product(c.av, c.wv[0], bias))


@pytest.mark.parametrize("n,k,m", [(32, 64, 1), (64, 300, 3), (13824, 256, 1), (160, 2560, 16), (96, 1000, 17), (352, 2560, 40),
                                   (2816, 512, 64), (1024, 1536, 130), (2048, 896, 300), (544, 1111, 513)])
def test_linear_gated(gpu, n, k, m):
    import torch
    c = Case(gpu, n + k + m, n, k, m, edges=True)
    for bias in (None, c.bias[0]):
        y = out(m, n // 2)
        c.w.linear(c.ac, c.as_, y, None if bias is None else dev(bias), glu=True)
        torch.cuda.synchronize()
        check(y, *mx4_ref.product(c.av, c.wv[0], bias, glu=True))


@pytest.mark.parametrize("m", [1, 20, 150])
def test_linear_strides(gpu, m):
    """Operand rows in wider buffers, output rows of any stride and alignment; what lies between is left as it was."""
    import torch
    n, k = 130, 700
    c = Case(gpu, m, n, k, m)
    kp = c.w.kpad
    ac = torch.full((m, kp // 2 + 32), 0x77, dtype=torch.uint8, device="cuda")
    as_ = torch.full((m, kp // 32 + 16), 0xFF, dtype=torch.uint8, device="cuda")
    ac[:, 16:16 + kp // 2], as_[:, 8:8 + kp // 32] = c.ac, c.as_
    for off, ldy in ((1, 133), (3, 140), (0, 132)):
        buf = torch.full((m * ldy + 8,), float("nan"), device="cuda")
        y = torch.as_strided(buf, (m, n), (ldy, 1), off)
        c.w.linear(ac[:, 16:], as_[:, 8:], y)
        torch.cuda.synchronize()
        check(y, *mx4_ref.product(c.av, c.wv[0]))
        assert int(buf.isnan().sum()) == buf.numel() - m * n


@pytest.mark.parametrize("m", [1, 16, 40, 200])
def test_linear_not_finite(gpu, m):
    """A NaN scale in an operand row or a matrix row reaches that row's or column's outputs, and no others."""
    import torch
    n, k = 96, 600
    rng = np.random.default_rng(m)
    a, w = mx4_ref.activations(rng, m, k), mx4_ref.matrix(rng, n, k)
    a[m // 2, 599], w[37, 5] = np.inf, np.nan
    (ac, as_), (wc, ws) = mx4_ref.quantise(a), mx4_ref.quantise(w)
    wt = gpu.Mx4Weight(n, k, dev(wc), dev(ws))
    y = out(m, n)
    wt.linear(dev(ac), dev(as_), y)
    torch.cuda.synchronize()
    want, tol = mx4_ref.product(mx4_ref.values(ac, as_, k), mx4_ref.values(wc, ws, k))
    assert np.isnan(want).sum() == m + n - 1
    check(y, want, tol)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,k,m,glu", [(16, 32, 1, False), (3, 5, 2, False), (2560, 2560, 1, False), (100, 257, 3, False),
                                       (64, 1000, 5, True), (13824, 300, 1, True), (896, 4864, 8, False), (160, 6912, 7, True),
                                       (48, 16384, 8, False), (40000, 1024, 1, False), (33000, 544, 6, False), (4096, 4096, 4, False)])
def test_linear_rows(gpu, type, n, k, m, glu):
    """The product of rows quantised within the call is that of the quantised rows."""
    import torch
    c = Case(gpu, n + k + m, n, k, m)
    x = dev(np.pad(c.a, ((0, 0), (0, 3))), type)
    x = x[:, 1:1 + k] if m % 2 else x[:, :k]
    av = mx4_ref.values(*mx4_ref.quantise(host(x.float())), k)
    for bias in (None, c.bias[0]):
        y = out(m, n // 2 if glu else n, 3)
        c.w.linear_rows(x, y, None if bias is None else dev(bias), glu=glu)
        torch.cuda.synchronize()
        check(y, *mx4_ref.product(av, c.wv[0], bias, glu))


def test_linear_rows_not_finite(gpu):
    import torch
    n, k, m = 64, 300, 3
    c = Case(gpu, 1, n, k, m)
    a = c.a.copy()
    a[1, 299] = np.nan
    a[2] = 0.0
    y = out(m, n)
    c.w.linear_rows(dev(a), y)
    torch.cuda.synchronize()
    check(y, *mx4_ref.product(mx4_ref.values(*mx4_ref.quantise(a), k), c.wv[0]))


def spread(rng, m, experts, how):
    """Counts of rows by expert that add up to m."""
    if how == "one":
        n = np.zeros(experts, int)
        n[experts // 2] = m
        return n
    if how == "last":
        n = np.zeros(experts, int)
        n[-1] = m
        return n
    p = rng.random(experts) ** 3 + 1e-9
    return rng.multinomial(m, p / p.sum())


def grouped_want(c, offsets, idx, m, n, glu, bias):
    want, tol = np.full((m, n // 2 if glu else n), np.nan), np.zeros((m, n // 2 if glu else n))
    for e in range(len(offsets) - 1):
        rows = np.arange(max(offsets[e], 0), min(offsets[e + 1], m))
        src = rows if idx is None else idx[rows]
        keep = (src >= 0) & (src < len(c.av))
        if keep.any():
            want[rows[keep]], tol[rows[keep]] = mx4_ref.product(c.av[src[keep]], c.wv[e], bias[e] if bias is not None else None, glu)
    return want, tol


GROUPED = [  # experts, rows, cols, tokens, rows of y, spread
    (1, 64, 300, 5, 9, "ragged"), (4, 33, 100, 7, 1, "ragged"), (8, 96, 512, 8, 32, "ragged"), (32, 160, 1000, 3, 24, "ragged"),
    (3, 256, 257, 50, 200, "ragged"), (5, 128, 640, 300, 700, "ragged"), (70, 64, 256, 20, 150, "ragged"), (200, 32, 64, 40, 500, "ragged"),
    (6, 96, 768, 200, 333, "one"), (129, 64, 300, 64, 64, "last"), (1500, 16, 64, 30, 900, "ragged"), (2, 640, 2560, 600, 1200, "ragged"),
]


@pytest.mark.parametrize("experts,n,k,t,m,how", GROUPED)
@pytest.mark.parametrize("glu", [False, True])
def test_grouped(gpu, experts, n, k, t, m, how, glu):
    import torch
    n = -(-n // 32) * 32 if glu else n
    c = Case(gpu, experts + n + m, n, k, t, experts=experts)
    rng = np.random.default_rng(m)
    offsets = np.concatenate([[0], np.cumsum(spread(rng, m, experts, how))]).astype(np.int32)
    idx = rng.integers(0, t, m).astype(np.int32)
    for bias in (None, c.bias):
        y = out(m, n // 2 if glu else n)
        c.w.linear_grouped(c.ac, c.as_, dev(offsets), y, dev(idx), None if bias is None else dev(bias), glu)
        torch.cuda.synchronize()
        check(y, *grouped_want(c, offsets, idx, m, n, glu, bias))


@pytest.mark.parametrize("m", [12, 90, 400])
def test_grouped_rows_left(gpu, m):
    """Rows before the first and behind the last group, and rows whose index names no row, are left as they were."""
    import torch
    experts, n, k, t = 5, 80, 300, 37
    c = Case(gpu, m, n, k, t, experts=experts)
    rng = np.random.default_rng(m)
    offsets = (np.concatenate([[0], np.cumsum(spread(rng, m - 4, experts, "ragged"))]) + 2).astype(np.int32)
    idx = rng.integers(0, t, m).astype(np.int32)
    idx[::5], idx[3::7] = -1, t
    idx[2] = 2 ** 31 - 1
    y = out(m, n)
    c.w.linear_grouped(c.ac, c.as_, dev(offsets), y, dev(idx))
    torch.cuda.synchronize()
    want, tol = grouped_want(c, offsets, idx, m, n, False, None)
    assert np.isnan(want[[0, 1, 2, 3, 5, -2, -1]]).all() and not np.isnan(want[4]).any()
    check(y, want, tol)
    # no index: row i takes operand row i, of which there are fewer
    y = out(m, n)
    c.w.linear_grouped(c.ac, c.as_, dev(offsets), y)
    torch.cuda.synchronize()
    check(y, *grouped_want(c, offsets, np.arange(m), m, n, False, None))


def test_grouped_offsets_cut(gpu):
    """Offsets beyond the rows are taken as if cut to them; no rows at all leaves everything."""
    import torch
    experts, n, k, m = 4, 64, 256, 50
    c = Case(gpu, 3, n, k, m, experts=experts)
    for offsets in ([-7, 10, 10, 45, 2 ** 31 - 1], [-2 ** 31, 0, 0, 0, 0], [50, 60, 70, 80, 90], [0, 50, 50, 50, 50]):
        offsets = np.array(offsets, np.int32)
        y = out(m, n)
        c.w.linear_grouped(c.ac, c.as_, dev(offsets), y)
        torch.cuda.synchronize()
        check(y, *grouped_want(c, np.clip(offsets.astype(np.int64), 0, m), None, m, n, False, None))


LARGE = [  # rows, token rows: the tiles of 256x128, 128x128, 128x64 and 128x32 (rows x token rows)
    (4130, 3070), (9920, 600), (2880, 1101), (1100, 300)]


def large(gpu, n, k, m, experts=1):
    """A weight, operand rows and biases made on the GPU, and their values in 64 bits there."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(n + k + m)

    def packed(rows, scale):
        x = torch.randn((rows, k), device="cuda", generator=g) * scale
        c, s, v = rows_on_gpu(gpu, x * torch.exp2(torch.randn((rows, 1), device="cuda", generator=g)))
        return c, s, v.double()

    wc, ws, wv = packed(experts * n, k ** -0.5)
    w = gpu.Mx4Weight(n, k, wc, ws, experts=experts)
    ac, as_, av = packed(m, 1.0)
    return w, wv.reshape(experts, n, k), ac, as_, av, torch.randn((experts, n), device="cuda", generator=g)


def product_on_gpu(a, w, bias, glu):
    """mx4_ref.product on GPU tensors."""
    import torch
    k = a.shape[1]
    y = a @ w.T + bias.double()
    tol = (-(-k // 32) + 16) * 2.0 ** -23 * (a.abs() @ w.abs().T) + 2.0 ** -126 + 2.0 ** -23 * (y.abs() + bias.double().abs())
    if not glu:
        return y, tol
    (g, u), (tg, tu) = y.chunk(2, 1), tol.chunk(2, 1)
    silu = g * torch.sigmoid(g)
    return silu * u, 1.1 * tg * (u.abs() + tu) + (silu.abs() + 1.1 * tg) * tu + 2.0 ** -21 * (silu * u).abs() + 2.0 ** -126


def check_on_gpu(y, want, tol):
    bad = ~((y.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())


@pytest.mark.parametrize("n,m", LARGE)
@pytest.mark.parametrize("k", [256, 300, 700, 1024, 1300, 2304])
@pytest.mark.parametrize("glu", [False, True])
def test_linear_large(gpu, n, m, k, glu):
    import torch
    n = -(-2 * n // 32) * 32 if glu else n
    w, wv, ac, as_, av, bias = large(gpu, n, k, m)
    want, tol = product_on_gpu(av, wv[0], bias[0], glu)
    cols = n // 2 if glu else n
    for pad in (0, 3):   # rows of y whose 16-byte stores are whole, and others
        y = torch.full((m, cols + pad), float("nan"), device="cuda")[:, :cols]
        w.linear(ac, as_, y, bias[0], glu=glu)
        check_on_gpu(y, want, tol)


@pytest.mark.parametrize("n,m,experts", [(2304, 6000, 7), (1280, 3000, 20), (640, 3600, 40), (1100, 700, 9)])
@pytest.mark.parametrize("k", [300, 1536, 2304])
@pytest.mark.parametrize("glu", [False, True])
def test_grouped_large(gpu, n, m, experts, k, glu):
    import torch
    n = -(-2 * n // 32) * 32 if glu else n
    t = m // 3
    w, wv, ac, as_, av, bias = large(gpu, n, k, t, experts)
    rng = np.random.default_rng(m)
    offsets = np.concatenate([[0], np.cumsum(spread(rng, m - 5, experts, "ragged"))]).astype(np.int32) + 2
    idx = rng.integers(0, t, m).astype(np.int32)
    idx[::11] = -1
    y = torch.full((m, n // 2 if glu else n), float("nan"), device="cuda")
    w.linear_grouped(ac, as_, dev(offsets), y, dev(idx), bias, glu)
    left = np.ones(m, bool)
    for e in range(experts):
        rows = np.arange(offsets[e], offsets[e + 1])
        rows = rows[idx[rows] >= 0]
        left[rows] = False
        if len(rows):
            at = torch.from_numpy(rows).cuda()
            check_on_gpu(y[at], *product_on_gpu(av[torch.from_numpy(idx[rows]).cuda().long()], wv[e], bias[e], glu))
    assert y[torch.from_numpy(left).cuda()].isnan().all()


def test_grouped_offsets_in_any_order(gpu):
    """Offsets that decrease or ranges that overlap: every output written is that of some expert whose range holds it."""
    import torch
    experts, n, k, m = 70, 32, 256, 200
    c = Case(gpu, 4, n, k, m, experts=experts)
    rng = np.random.default_rng(8)
    for offsets in (rng.integers(-50, 300, experts + 1), np.tile([0, m], 36)[:experts + 1], np.arange(experts, -1, -1)):
        offsets = offsets.astype(np.int32)
        y = out(m, n)
        c.w.linear_grouped(c.ac, c.as_, dev(offsets), y)
        torch.cuda.synchronize()
        got = host(y).astype(np.float64)
        fits = np.isnan(got)
        for e in range(experts):
            rows = np.arange(max(offsets[e], 0), min(max(offsets[e + 1], 0), m))
            want, tol = mx4_ref.product(c.av[rows], c.wv[e])
            fits[rows] |= np.abs(got[rows] - want) <= tol
        assert fits.all()


FAR = [(1, 40), (3, 40), (40, 40), (300, 40)]   # token rows, rows


@pytest.mark.parametrize("m,n", FAR)
def test_offsets_beyond_32_bits(gpu, m, n):
    """Rows so far apart that the last ones lie behind 2^32 bytes: operands, outputs, the quantiser's inputs and outputs."""
    import torch
    k = 300
    c = Case(gpu, m, n, k, m)
    far = (5 << 30) // max(m - 1, 1) // 16 * 16 + 1024
    codes = torch.empty(far * (m - 1) + 4096, dtype=torch.uint8, device="cuda").as_strided((m, 256), (far, 1))
    scales = torch.empty(far * (m - 1) + 4096, dtype=torch.uint8, device="cuda").as_strided((m, 16), (far, 1))
    x = torch.empty(far // 4 * (m - 1) + 4096, device="cuda").as_strided((m, k), (far // 4, 1))
    y = torch.empty(far // 4 * (m - 1) + 4096, device="cuda").as_strided((m, n), (far // 4, 1))
    x.copy_(dev(c.a))
    y.fill_(float("nan"))
    gpu.mx4_quant_rows(x, codes, scales)
    assert torch.equal(codes, c.ac) and torch.equal(scales, c.as_)
    want = mx4_ref.product(c.av, c.wv[0])
    c.w.linear(codes, scales, y)
    check(y, *want)
    y.fill_(float("nan"))
    c.w.linear_grouped(codes, scales, dev(np.array([0, m], np.int32)), y)
    check(y, *want)
    if m <= 8:
        y.fill_(float("nan"))
        c.w.linear_rows(x, y)
        check(y, *want)


@pytest.mark.parametrize("m,n", [(300, 4096), (600, 10240)])
def test_operand_rows_behind_31_bits(gpu, m, n):
    """Operand rows that span between 2^31 and 2^32 bytes, through the forms whose loads take 32-bit offsets."""
    import torch
    k = 1000
    w, wv, ac, as_, av, bias = large(gpu, n, k, m)
    far = (7 << 29) // m // 16 * 16
    codes = torch.empty(far * m, dtype=torch.uint8, device="cuda").as_strided((m, 512), (far, 1))
    codes.copy_(ac)
    y = out(m, n)
    w.linear(codes, as_, y, bias[0])
    check_on_gpu(y, *product_on_gpu(av, wv[0], bias[0], False))
    idx = torch.arange(m - 1, -1, -1, device="cuda", dtype=torch.int32)
    y = out(m, n)
    w.linear_grouped(codes, as_, dev(np.array([0, m], np.int32)), y, idx, bias)
    check_on_gpu(y, *product_on_gpu(av.flip(0), wv[0], bias[0], False))


@pytest.mark.parametrize("m", [3, 60, 200])
def test_stack_beyond_32_bits(gpu, m):
    """A stack of matrices of more than 2^32 bytes: the last one's products, at some of its rows."""
    import torch
    experts, n, k = 5, 65536, 32768
    g = torch.Generator(device="cuda").manual_seed(m)
    wc = torch.randint(0, 256, (experts, n, k // 2), dtype=torch.uint8, device="cuda", generator=g)
    ws = torch.randint(120, 126, (experts, n, k // 32), dtype=torch.uint8, device="cuda", generator=g)
    w = gpu.Mx4Weight(n, k, wc, ws, experts=experts)
    assert w.bytes > 1 << 32
    ac, as_ = mx4_ref.quantise(mx4_ref.activations(np.random.default_rng(m), m, k))
    y = out(m, n)
    w.linear_grouped(dev(ac), dev(as_), dev(np.array([0, 0, 0, 0, 0, m], np.int32)), y)
    torch.cuda.synchronize()
    assert not y.isnan().any()
    at = [0, 1, 17, 32767, 40000, 65520, 65535]
    want, tol = mx4_ref.product(mx4_ref.values(ac, as_, k), mx4_ref.values(host(wc[4, at]), host(ws[4, at]), k))
    check(y[:, at], want, tol)


def test_run_together(gpu):
    """A routed feed-forward: token rows quantised, the experts' gated product on gathered rows, its outputs quantised, the
    down product, each step against the definition on the step's own inputs."""
    import torch
    experts, dim, hidden, t, top = 6, 320, 224, 45, 2
    rng = np.random.default_rng(5)
    up = Case(gpu, 11, 2 * hidden, dim, t, experts=experts)
    down = Case(gpu, 12, dim, hidden, 1, experts=experts)
    ids = np.argsort(rng.random((t, experts)) * np.arange(1, experts + 1), 1)[:, :top].ravel()
    order = np.argsort(ids, kind="stable")
    idx = (order // top).astype(np.int32)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(ids, minlength=experts))]).astype(np.int32)
    m = t * top
    x = dev(up.a)
    c, s, _ = rows_on_gpu(gpu, x)
    h = out(m, hidden)
    up.w.linear_grouped(c, s, dev(offsets), h, dev(idx), glu=True)
    hc, hs, _ = rows_on_gpu(gpu, h)
    y = out(m, dim)
    down.w.linear_grouped(hc, hs, dev(offsets), y, bias=dev(down.bias))
    torch.cuda.synchronize()
    check(h, *grouped_want(up, offsets, idx, m, 2 * hidden, True, None))
    wc, ws = mx4_ref.quantise(host(h))
    assert np.array_equal(host(hc), wc) and np.array_equal(host(hs), ws)
    down.av = mx4_ref.values(wc, ws, hidden)
    check(y, *grouped_want(down, offsets, None, m, dim, False, down.bias))


@pytest.mark.parametrize("m", [4, 100])
def test_graph_replays(gpu, m):
    """The whole run captured: every replay, with eager work between, gives the eager bits."""
    import torch
    experts, n, k = 3, 128, 512
    c = Case(gpu, m, n, k, m, experts=experts)
    one = Case(gpu, m + 1, n, k, 1)
    x = dev(c.a)
    codes, scales = torch.zeros_like(c.ac), torch.zeros_like(c.as_)
    offsets, idx = dev(np.array([0, m // 2, m // 2, m], np.int32)), dev(np.arange(m, dtype=np.int32)[::-1].copy())
    ys = [out(m, n), out(m, n // 2), out(min(m, 8), n)]

    def step():
        gpu.mx4_quant_rows(x, codes, scales)
        one.w.linear(codes, scales, ys[0])
        c.w.linear_grouped(codes, scales, offsets, ys[1], idx, glu=True)
        one.w.linear_rows(x[:8], ys[2])

    step()
    torch.cuda.synchronize()
    want = [y.clone() for y in ys]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(4):
        for y in ys:
            y.fill_(float("nan"))
        codes.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ys, want))
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ys, want))


def test_two_graphs_on_one_weight(gpu):
    """Two graphs that share a weight and its operands, replayed in turn and on two streams at once."""
    import torch
    n, k, m = 512, 1536, 150
    c = Case(gpu, 21, n, k, m)
    ys, graphs = [out(m, n), out(m, n)], []
    c.w.linear(c.ac, c.as_, ys[0])
    torch.cuda.synchronize()
    want = ys[0].clone()
    for y in ys:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.w.linear(c.ac, c.as_, y)
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for y in ys:
            y.fill_(float("nan"))
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, want) for y in ys)


def test_threads(gpu):
    """Calls of several threads at once, each on a stream of its own."""
    import threading

    import torch
    n, k = 320, 1024
    c = Case(gpu, 33, n, k, 40)
    offsets = dev(np.array([0, 40], np.int32))
    bad = []

    def work():
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for i in range(20):
                y = out(40, n)
                if i % 2:
                    c.w.linear(c.ac, c.as_, y)
                else:
                    c.w.linear_grouped(c.ac, c.as_, offsets, y)
                st.synchronize()
                if not (np.abs(host(y) - want) <= tol).all():
                    bad.append(i)

    want, tol = mx4_ref.product(c.av, c.wv[0])
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_streams(gpu):
    """Calls on two streams at once, on one weight."""
    import torch
    n, k = 256, 2560
    c = Case(gpu, 9, n, k, 64)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    ys = [out(64, n) for _ in range(8)]
    torch.cuda.synchronize()
    for i, y in enumerate(ys):
        c.w.linear(c.ac, c.as_, y, stream=streams[i % 2])
    torch.cuda.synchronize()
    want, tol = mx4_ref.product(c.av, c.wv[0])
    for y in ys:
        check(y, want, tol)
