"""Low-rank adapters of many requests on the GPU (include/eif_hip_adapters.h) against the definition in 64 bits."""
import numpy as np
import pytest

import moe_ref
import mx4_ref
from test_gpu_moe import dev, host

pytestmark = pytest.mark.gpu


class Case:
    """Adapters of ragged ranks in every slot but the last, which is empty."""

    def __init__(self, gpu, seed, slots, rows, cols, rank, weights="bf16", on_device=True, ranks=None):
        import torch
        rng = np.random.default_rng(seed)
        dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[weights]
        self.h = gpu.Adapters(slots, rows, cols, rank, dt)
        self.pairs, self.rows = {}, rows
        for s in range(slots - 1 if slots > 1 else 1):
            r = ranks[s] if ranks else max(1, rank >> (s % 3))
            a, b = rng.standard_normal((r, cols)) / np.sqrt(cols), rng.standard_normal((rows, r)) / np.sqrt(r)
            a, b = torch.from_numpy(a).to(dt), torch.from_numpy(b).to(dt)
            scale = 0.5 + 0.25 * s
            self.h.set(s, a.cuda() if on_device else a, b.cuda() if on_device else b, scale)
            self.pairs[s] = (a.double().numpy(), b.double().numpy(), scale)

    def check(self, x, slot, y, base=None, pairs=None):
        want, tol = moe_ref.adapters(host(x), slot, self.pairs if pairs is None else pairs, base, self.rows)
        got = host(y).astype(np.float64)
        bad = ~(np.abs(got - want) <= tol)
        assert not bad.any(), (np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4], tol[bad][:4])


def slots_of(rng, m, slots, kind):
    if kind == "one":
        return np.zeros(m, np.int32)
    if kind == "runs":   # a prompt after another
        cuts = np.sort(rng.integers(0, m + 1, 5))
        return rng.integers(-1, slots, 6)[np.searchsorted(cuts, np.arange(m), side="right")].astype(np.int32)
    s = rng.integers(-2, slots + 2, m).astype(np.int32)
    s[rng.random(m) < 0.05] = 2 ** 31 - 1
    s[rng.random(m) < 0.05] = -2 ** 31
    return s


SHAPES = [  # rows, cols, rank, slots, tokens
    (1, 1, 1, 1, 1), (16, 32, 16, 2, 1), (17, 33, 3, 3, 5), (100, 300, 8, 4, 17), (2560, 2560, 16, 4, 1), (1025, 4100, 40, 3, 9),
    (640, 896, 64, 5, 48), (300, 2048, 256, 3, 33), (64, 64, 16, 20, 64), (70, 130, 16, 4, 65), (2560, 512, 16, 6, 100), (129, 1000, 33, 4, 200),
    (512, 4096, 64, 5, 300), (1000, 640, 80, 3, 130), (96, 264, 256, 4, 90), (4096, 256, 16, 9, 1100), (31, 8200, 20, 3, 150),
    # tiles of 16 and of 32 rows
    (1, 1, 1, 1, 513), (17, 33, 3, 3, 600), (260, 300, 16, 20, 777), (70, 1000, 33, 4, 259), (520, 264, 64, 30, 1025), (96, 130, 200, 4, 300),
    (33, 70, 16, 5, 4099), (130, 300, 40, 33, 4096), (200, 512, 64, 6, 5001), (40, 264, 130, 3, 4200), (640, 96, 16, 2, 8193),
]


@pytest.mark.parametrize("rows,cols,rank,slots,m", SHAPES)
def test_linear(gpu, rows, cols, rank, slots, m):
    import torch
    for i, (xt, wt) in enumerate((("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("bf16", "f16"), ("f16", "f32"))):
        rng = np.random.default_rng(rows + cols + i)
        c = Case(gpu, i, slots, rows, cols, rank, wt, on_device=i % 2 == 0)
        x = dev(mx4_ref.activations(rng, m, cols), xt)
        for kind in ("one", "runs", "any"):
            slot = slots_of(rng, m, slots, kind)
            base = rng.standard_normal((m, rows)).astype(np.float32) if kind != "one" else None
            y = torch.full((m, rows), float("nan"), device="cuda")
            c.h.linear(x, dev(slot), y, None if base is None else dev(base))
            torch.cuda.synchronize()
            c.check(x, slot, y, base)
        c.h.close()


@pytest.mark.parametrize("m", [5, 77, 300, 4100])
@pytest.mark.parametrize("rows,cols", [(260, 512), (257, 515), (33, 40)])
def test_strides_and_in_place(gpu, m, rows, cols):
    """Rows of any stride and alignment; the base is y itself; what lies between is left as it was."""
    import torch
    c = Case(gpu, m, 4, rows, cols, 24)
    rng = np.random.default_rng(rows)
    slot = slots_of(rng, m, 4, "any")
    for xoff, ldx, yoff, ldy, xt in ((0, cols, 0, rows, "f32"), (1, cols + 3, 1, rows + 5, "f32"), (4, cols + 8, 4, rows + 8, "bf16"),
                                     (3, cols + 1, 2, rows + 2, "f16"), (8, cols + 8, 0, rows + 3, "bf16")):
        xb = dev(mx4_ref.activations(rng, 1, m * ldx + xoff)[0], xt)
        x = torch.as_strided(xb, (m, cols), (ldx, 1), xoff)
        yb = dev(rng.standard_normal(m * ldy + yoff + 8).astype(np.float32))
        before = host(yb).copy()
        y = torch.as_strided(yb, (m, rows), (ldy, 1), yoff)
        base = host(y).copy()
        c.h.linear(x, dev(slot), y, y)
        torch.cuda.synchronize()
        c.check(x, slot, y, base)
        inside = torch.zeros_like(yb, dtype=torch.bool)
        torch.as_strided(inside, (m, rows), (ldy, 1), yoff).fill_(True)
        out = ~host(inside)
        assert np.array_equal(host(yb)[out], before[out])


@pytest.mark.parametrize("m", [6, 70, 600, 4200])
@pytest.mark.parametrize("types", [("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f16"), ("f32", "f32")])
def test_not_finite(gpu, m, types):
    """An infinity or NaN in a row reaches that row alone, and not through the zeros beyond its adapter's rank."""
    import torch
    rows, cols = 80, 200
    c = Case(gpu, 3, 3, rows, cols, 12, types[1], ranks=[1, 5])
    rng = np.random.default_rng(m)
    x = mx4_ref.activations(rng, m, cols)
    slot = (np.arange(m) % 4 - 1).astype(np.int32)   # none, two adapters, an empty slot
    x[:, 7] = 0.0
    x[1, 7], x[2, 7], x[0, 7], x[3, 7] = np.inf, np.nan, np.nan, np.inf
    y = torch.full((m, rows), 5.0, device="cuda")
    base = rng.standard_normal((m, rows)).astype(np.float32)
    c.h.linear(dev(x, types[0]), dev(slot), y, dev(base))
    torch.cuda.synchronize()
    got = host(y)
    with np.errstate(invalid="ignore"):
        a, b, scale = c.pairs[0]
        want = scale * ((x[1].astype(np.float64) @ a.T) @ b.T)
    assert not np.isfinite(want).any() and np.isnan(got[2]).all()
    assert np.array_equal(np.isnan(got[1]), np.isnan(want)) and np.array_equal(got[1][~np.isnan(want)], want[~np.isnan(want)])
    x[1, 7] = x[2, 7] = 0.0
    rest = np.delete(np.arange(m), [1, 2])
    fin = x.copy()
    fin[0, 7] = fin[3, 7] = 0.0
    want, tol = moe_ref.adapters(host(dev(fin, types[0])), slot, c.pairs, base, rows)
    assert (np.abs(got[rest] - want[rest]) <= tol[rest]).all()


@pytest.mark.parametrize("m", [20, 600, 4200])
@pytest.mark.parametrize("types", [("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f32")])
def test_broken_adapter(gpu, m, types):
    """Matrices with infinities and NaN in one slot do not reach the rows of other slots, or of none."""
    import torch
    rows, cols = 70, 130
    c = Case(gpu, 4, 4, rows, cols, 20, types[1])
    rng = np.random.default_rng(m)
    dt = torch.from_numpy(c.pairs[1][0]).to(getattr(torch, {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}[types[1]])).dtype
    a, b = torch.randn(20, cols).to(dt), torch.randn(rows, 20).to(dt)
    a[3, 5], a[17, 100], b[9, 2], b[50, 19] = float("inf"), float("nan"), float("-inf"), float("nan")
    c.h.set(1, a.cuda(), b.cuda(), 1.0)
    x, slot = mx4_ref.activations(rng, m, cols), slots_of(rng, m, 4, "any")
    slot[:4] = [0, 1, 2, -1]
    x = dev(x, types[0])
    base = rng.standard_normal((m, rows)).astype(np.float32)
    y = torch.empty((m, rows), device="cuda")
    c.h.linear(x, dev(slot), y, dev(base))
    torch.cuda.synchronize()
    pairs = {s: p for s, p in c.pairs.items() if s != 1}
    rest = slot != 1
    want, tol = moe_ref.adapters(host(x), slot, pairs, base, rows)
    got = host(y)
    assert (np.abs(got[rest] - want[rest]) <= tol[rest]).all() and np.isnan(got[~rest]).any(1).all()


def test_slots_are_replaced(gpu):
    """A slot takes another adapter, of another rank, and none; the others stay."""
    import torch
    rng = np.random.default_rng(9)
    for m in (4, 96, 520, 4100):
        c = Case(gpu, 1, 4, 200, 320, 32)
        other = Case(gpu, 2, 4, 200, 320, 32, ranks=[32, 3, 17])
        x, slot = dev(mx4_ref.activations(rng, m, 320)), (np.arange(m) % 4).astype(np.int32)
        y = torch.empty((m, 200), device="cuda")
        a, b, s = other.pairs[1]
        c.h.set(0, torch.from_numpy(a).to(torch.bfloat16), torch.from_numpy(b).to(torch.bfloat16), s)
        c.pairs[0] = other.pairs[1]
        c.h.clear(1)
        del c.pairs[1]
        c.h.linear(x, dev(slot), y)
        torch.cuda.synchronize()
        c.check(x, slot, y)
        c.h.clear(0)
        c.h.clear(2)
        c.h.linear(x, dev(slot), y)
        torch.cuda.synchronize()
        assert not y.any()


def test_slot_of_strided_device_matrices(gpu):
    """A and B as views of larger matrices."""
    import torch
    rng = np.random.default_rng(10)
    h = gpu.Adapters(2, 90, 70, 8, torch.float16)
    a = torch.from_numpy(rng.standard_normal((8, 100))).half().cuda()
    b = torch.from_numpy(rng.standard_normal((90, 33))).half().cuda()
    h.set(1, a[:5, 3:73], b[:, 7:12], -1.5)
    x, slot = dev(mx4_ref.activations(rng, 3, 70)), np.array([1, 0, 1], np.int32)
    y = torch.empty((3, 90), device="cuda")
    h.linear(x, dev(slot), y)
    torch.cuda.synchronize()
    want, tol = moe_ref.adapters(host(x), slot, {1: (a[:5, 3:73].double().cpu().numpy(), b[:, 7:12].double().cpu().numpy(), -1.5)}, None, 90)
    assert (np.abs(host(y) - want) <= tol).all()


@pytest.mark.parametrize("m", [3, 90, 520, 4097])
def test_far_offsets(gpu, m):
    """Slots behind 2^32 bytes, and rows of x and y behind 2^31 elements."""
    import torch
    torch.cuda.empty_cache()
    h = gpu.Adapters(300, 16000, 16000, 256, torch.bfloat16)   # 16 MB a slot
    assert h.bytes > 1 << 32
    rng = np.random.default_rng(11)
    a, b = torch.from_numpy(rng.standard_normal((2, 16000)) / 100).bfloat16(), torch.from_numpy(rng.standard_normal((16000, 2))).bfloat16()
    h.set(299, a, b, 0.75)
    ld = (1 << 31) // (m - 1) + 16
    xb = torch.zeros((m - 1) * ld + 16000, dtype=torch.bfloat16, device="cuda")
    yb = torch.zeros((m - 1) * ld + 16000, device="cuda")
    x, y = torch.as_strided(xb, (m, 16000), (ld, 1), 0), torch.as_strided(yb, (m, 16000), (ld, 1), 0)
    x.copy_(dev(mx4_ref.activations(rng, m, 16000), "bf16"))
    slot = np.full(m, 299, np.int32)
    h.linear(x, dev(slot), y)
    torch.cuda.synchronize()
    some = np.unique(np.concatenate([np.arange(min(m, 40)), np.arange(max(0, m - 40), m)]))
    at = torch.from_numpy(some).cuda()
    want, tol = moe_ref.adapters(host(x[at]), slot[some], {299: (a.double().numpy(), b.double().numpy(), 0.75)}, None, 16000)
    assert (np.abs(host(y[at]) - want) <= tol).all()
    h.close()
    del xb, yb, x, y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("m", [2, 80, 600, 4100])
def test_in_a_graph_beside_a_projection(gpu, m):
    """The shared projection (MXFP4) and the adapters on its output in place, captured and replayed on other inputs and slots."""
    import torch
    rows, cols = 192, 512
    rng = np.random.default_rng(12)
    wc, ws = mx4_ref.quantise(mx4_ref.matrix(rng, rows, cols))
    w = gpu.Mx4Weight(rows, cols, wc, ws)
    c = Case(gpu, 5, 5, rows, cols, 16)
    x, slot = torch.zeros((m, cols), device="cuda"), torch.zeros(m, dtype=torch.int32, device="cuda")
    kp = gpu.mx4_kpad(cols)
    xc, xs = (torch.zeros((m, n), dtype=torch.uint8, device="cuda") for n in (kp // 2, kp // 32))
    y, plain = torch.zeros((m, rows), device="cuda"), torch.zeros((m, rows), device="cuda")

    def step():
        gpu.mx4_quant_rows(x, xc, xs)
        w.linear(xc, xs, y)
        plain.copy_(y)
        c.h.linear(x, slot, y, y)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for i in range(4):
        x.copy_(dev(mx4_ref.activations(rng, m, cols)))
        slot.copy_(dev(slots_of(rng, m, 5, "any")))
        step()
        torch.cuda.synchronize()
        want = y.clone()
        c.check(x, host(slot), y, host(plain))
        y.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_rows_do_not_depend_on_each_other(gpu):
    """A row's result is the same bits whatever slots the other rows name, and on any stream."""
    import torch
    rng = np.random.default_rng(13)
    for m in (40, 160, 600, 4200):
        c = Case(gpu, 6, 6, 512, 768, 16)
        x = dev(mx4_ref.activations(rng, m, 768))
        a, b = slots_of(rng, m, 6, "any"), slots_of(rng, m, 6, "runs")
        a[::3] = b[::3]
        ya, yb = (torch.empty((m, 512), device="cuda") for _ in range(2))
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        ad, bd = dev(a), dev(b)
        torch.cuda.synchronize()
        c.h.linear(x, ad, ya)
        c.h.linear(x, bd, yb, stream=s)
        torch.cuda.synchronize()
        assert torch.equal(ya[::3], yb[::3])
