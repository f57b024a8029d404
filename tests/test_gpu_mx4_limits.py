"""Microscaled 4-bit rows and products on the GPU at the ends of what the calls take (include/eif_hip_mx.h)."""
import numpy as np
import pytest

import mx4_ref
from test_gpu_mx4 import dev

pytestmark = pytest.mark.gpu


def test_quant_rows_beyond_a_launch(gpu):
    """More runs of 256 columns than the threads of one launch have room for: rows that repeat give codes that repeat."""
    import torch
    torch.cuda.empty_cache()
    rows, period = (1 << 26) + 4099, 4099
    base = mx4_ref.activations(np.random.default_rng(1), period, 32)
    base = dev(base, "bf16")
    wc, ws = mx4_ref.quantise(base.float().cpu().numpy())
    times = -(-rows // period)
    x = base.repeat(times, 1)[:rows]
    codes = torch.full((times * period, 128), 0xA5, dtype=torch.uint8, device="cuda")
    scales = torch.full((times * period, 8), 0xA5, dtype=torch.uint8, device="cuda")
    gpu.mx4_quant_rows(x, codes[:rows], scales[:rows])
    torch.cuda.synchronize()
    for got, want in ((codes, dev(wc)), (scales, dev(ws))):
        assert (got[rows:] == 0xA5).all()
        tail = rows - (times - 1) * period
        got = got.view(times, period, -1)
        assert torch.equal(got[-1, :tail], want[:tail])
        for lo in range(0, times - 1, 1024):
            part = got[lo:min(lo + 1024, times - 1)]
            assert torch.equal(part, want.expand_as(part))


def test_weight_beyond_a_launch(gpu):
    """A matrix whose layout has more than 2^32 pieces of 16 bytes: rows that repeat give outputs that repeat."""
    import torch
    torch.cuda.empty_cache()
    rows, period = (1 << 29) + 4099, 4099
    rng = np.random.default_rng(2)
    wc, ws = mx4_ref.quantise(mx4_ref.matrix(rng, period, 32))
    wc, ws = dev(wc[:, :16]), dev(ws[:, :1])
    times = -(-rows // period)
    w = gpu.Mx4Weight(rows, 32, wc.repeat(times, 1)[:rows], ws.repeat(times, 1)[:rows])
    assert w.bytes > 1 << 36
    x = dev(mx4_ref.activations(rng, 1, 32))
    want = torch.full((1, period), float("nan"), device="cuda")
    gpu.Mx4Weight(period, 32, wc, ws).linear_rows(x, want)
    y = torch.full((1, times * period), float("nan"), device="cuda")
    w.linear_rows(x, y[:, :rows])
    torch.cuda.synchronize()
    w.close()
    assert y[0, rows:].isnan().all() and not want.isnan().any()
    tail = rows - (times - 1) * period
    y = y.view(times, period)
    assert torch.equal(y[:-1], want.expand(times - 1, period)) and torch.equal(y[-1, :tail], want[0, :tail])
    torch.cuda.empty_cache()


@pytest.mark.parametrize("form,n,m", [("rows", 320, 3), ("linear", 320, 12), ("linear", 640, 28), ("linear", 2208, 300), ("linear", 5760, 1101),
                                      ("linear", 19840, 600), ("grouped", 320, 60), ("grouped", 2560, 3000)])
def test_gates_far_below_zero(gpu, form, n, m):
    """SiLU(g) u where e^-g nears the end of FP32's range and passes it. The sums are zeros, so that g and u are the biases alone.
    -g log2(e) is off by two roundings, which move the exponential by |g| 2^-23; the exponential, the quotient and the products
    come to 2^-21. From e^-g = 2^126 on the quotient may be 0, where |SiLU(g)| <= 87.4 2^-126 < 2^-119; a result below the
    smallest normal number is off by half a step of its own."""
    import torch
    k, h, experts = 64, n // 2, 5 if form == "grouped" else 1
    w = gpu.Mx4Weight(n, k, np.zeros((experts * n, k // 2), np.uint8), np.zeros((experts * n, k // 32), np.uint8), experts=experts)
    rng = np.random.default_rng(n + m)
    g = np.concatenate([[-0.0, 0.0, -87.25, -87.5, -88.0, -88.75, -89.0, -92.0, -104.0, -174.0, -180.0, -190.0, -300.0, -1e9, 88.0],
                        rng.uniform(-60, -40, h // 4), rng.uniform(-200, 90, h)])[:h].astype(np.float32)
    u = rng.choice([1.0, -1e6, 1e30, -3e38, 3e-3], h).astype(np.float32)
    bias = dev(np.tile(np.concatenate([g, u]), (experts, 1)))
    y = torch.full((m, h), float("nan"), device="cuda")
    x = dev(mx4_ref.activations(rng, m, k))
    if form == "rows":
        w.linear_rows(x, y, bias[0], glu=True)
    else:
        codes = torch.zeros((m, w.kpad // 2), dtype=torch.uint8, device="cuda")
        scales = torch.zeros((m, w.kpad // 32), dtype=torch.uint8, device="cuda")
        gpu.mx4_quant_rows(x, codes, scales)
        if form == "grouped":
            w.linear_grouped(codes, scales, dev(np.linspace(0, m, experts + 1).astype(np.int32)), y, bias=bias, glu=True)
        else:
            w.linear(codes, scales, y, bias[0], glu=True)
    torch.cuda.synchronize()
    g, u = g.astype(np.float64), u.astype(np.float64)
    with np.errstate(over="ignore"):
        want = g / (1.0 + np.exp(-g)) * u
    tol = np.abs(want) * (2.0 ** -21 + np.abs(g) * 2.0 ** -23) + 2.0 ** -119 * np.abs(u) + 2.0 ** -149
    keep = np.abs(want) < 3.4e38
    got = y.cpu().numpy().astype(np.float64)
    bad = (np.abs(got - want) > tol) & keep | ~keep & ~np.isinf(got)
    assert not bad.any(), [(g[c], u[c], got[r, c], want[c]) for r, c in np.argwhere(bad)[:5]]


@pytest.mark.parametrize("n,k,m", [(2560, 6912, 24), (4864, 896, 48), (640, 2560, 30), (4096, 1024, 300), (2880, 2304, 700), (10240, 1024, 600)])
def test_order_of_sums_by_shapes_alone(gpu, n, k, m):
    """Operand rows that span 2^32 bytes give the bits of adjacent ones, on scales so wide apart that every sum rounds."""
    import torch
    torch.cuda.empty_cache()
    g = torch.Generator(device="cuda").manual_seed(n + m)

    def packed(*shape):
        c = torch.randint(0, 256, (*shape, mx4_ref.kpad(k) // 2), dtype=torch.uint8, device="cuda", generator=g)
        s = torch.randint(115, 140, (*shape, mx4_ref.kpad(k) // 32), dtype=torch.uint8, device="cuda", generator=g)
        c[..., (k + 1) // 2:], s[..., -(-k // 32):] = 0, 0
        return c, s

    w = gpu.Mx4Weight(n, k, *packed(2, n), experts=2)
    one = gpu.Mx4Weight(n, k, *packed(n))
    codes, scales = packed(m)
    stride = (5 << 30) // (m - 1) // 16 * 16
    far = torch.empty(stride * (m - 1) + codes.shape[1], dtype=torch.uint8, device="cuda").as_strided(codes.shape, (stride, 1))
    far.copy_(codes)
    offsets = dev(np.array([0, m // 3, m], np.int32))
    got = []
    for c in (codes, far):
        y = torch.full((2, m, n), float("nan"), device="cuda")
        one.linear(c, scales, y[0])
        w.linear_grouped(c, scales, offsets, y[1])
        torch.cuda.synchronize()
        got.append(y)
    assert not got[0].isnan().any() and torch.equal(got[0], got[1])


@pytest.mark.parametrize("n,m", [(96, 3), (96, 40), (4096, 300), (4130, 1100)])
def test_scale_bytes_of_the_whole_range(gpu, n, m):
    """Scale bytes that the quantiser never gives, 253 and 254, against 1 and 0: the scales' products are 1, the sums exact."""
    import torch
    k = 1024
    rng = np.random.default_rng(n + m)
    byte = rng.choice([0, 1, 2, 127, 252, 253, 254], k // 32).astype(np.uint8)
    wc, ac = (dev(rng.integers(0, 256, (r, k // 2)).astype(np.uint8)) for r in (n, m))
    w = gpu.Mx4Weight(n, k, wc, dev(np.tile(byte, (n, 1))))
    y = torch.full((m, n), float("nan"), device="cuda")
    w.linear(ac, dev(np.tile(254 - byte, (m, 1)).astype(np.uint8)), y)
    torch.cuda.synchronize()
    one = np.full(k // 32, 127, np.uint8)
    want = mx4_ref.values(ac.cpu().numpy(), np.tile(one, (m, 1)), k) @ mx4_ref.values(wc.cpu().numpy(), np.tile(one, (n, 1)), k).T
    assert np.array_equal(y.cpu().numpy().astype(np.float64), want)


def test_one_row_of_many_experts(gpu):
    """One row to the last of 4096 matrices, and none to any."""
    import torch
    experts, n, k = 4096, 48, 64
    rng = np.random.default_rng(3)
    wc, ws = mx4_ref.quantise(mx4_ref.matrix(rng, experts * n, k))
    wc, ws = wc[:, :k // 2], ws[:, :k // 32]
    w = gpu.Mx4Weight(n, k, dev(wc).reshape(experts, n, -1), dev(ws).reshape(experts, n, -1), experts=experts)
    ac, as_ = mx4_ref.quantise(mx4_ref.activations(rng, 2, k))
    want, tol = mx4_ref.product(mx4_ref.values(ac, as_, k)[1:], mx4_ref.values(wc[-n:], ws[-n:], k))
    for last in (1, 0):
        offsets = np.zeros(experts + 1, np.int32)
        offsets[-1] = last
        y = torch.full((1, n), float("nan"), device="cuda")
        w.linear_grouped(dev(ac), dev(as_), dev(offsets), y, dev(np.array([1], np.int32)))
        torch.cuda.synchronize()
        assert (np.abs(y.cpu().numpy() - want) <= tol).all() if last else y.isnan().all()
