"""Routing to experts, sorting by expert and combining on the GPU (include/eif_hip_moe.h) against the definitions in 64 bits."""
import itertools

import numpy as np
import pytest

import moe_ref
import mx4_ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}
EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def dev(a, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(getattr(torch, TYPES[dtype]))


def host(t):
    return t.float().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def ints(n, fill=-7):
    import torch
    return torch.full((n,), fill, dtype=torch.int32, device="cuda")


def logits_of(rng, tokens, experts, kind):
    """Ordinary logits, and rows where the choice can go wrong."""
    x = (1.5 * rng.standard_normal((tokens, experts)) + 0.7 * rng.standard_normal((1, experts))).astype(np.float32)
    if kind == "ties":
        return (np.round(2 * x) / 2).astype(np.float32)
    if kind == "edges":
        for t in range(tokens):
            r = x[t]
            n = t % 9
            if n == 1:
                r[:] = -np.inf
            elif n == 2:
                r[rng.random(experts) < 0.7] = -np.inf
            elif n == 3:
                r[rng.random(experts) < 0.3] = np.nan
            elif n == 4:
                r[int(rng.integers(experts))] = np.inf
                r[int(rng.integers(experts))] = np.inf
            elif n == 5:
                r[:] = -np.inf
                r[int(rng.integers(experts))] = -3e38
            elif n == 6:
                r *= np.float32(1e37)
            elif n == 7:
                r[:] = np.nan
            elif n == 8:
                r[:] = -200.0 - np.round(r)
    return x


def weight_tolerance(logits, want, spec):
    """Relative: the weight's own rounding, 2^-24; and for a softmax over all experts without a bias, whose sum is of FP32
    exponentials e^-d of d = m - l: d and its multiple are off by 2^-23 d, an exponential by 2^-23 of itself more, and each is part of at
    most 64 sums."""
    if spec.get("renormalise", True) or spec.get("score", 0) == moe_ref.SIGMOID or spec.get("bias") is not None:
        return 2.0 ** -24 * 1.01
    l = np.where(np.isnan(logits), -np.inf, np.minimum(logits.astype(np.float64), moe_ref.MOST))
    m = l.max(1, keepdims=True)
    d = np.where(l > -np.inf, np.where(m > -np.inf, m, 0.0) - l, np.inf)
    e = np.where(d < 800, np.exp(-np.minimum(d, 800.0)), 0.0)
    z = np.maximum(e.sum(1), 1e-300)
    return (2.0 ** -23 * ((e * np.minimum(d, 800.0)).sum(1) / z) + 2.0 ** -23 + 66 * 2.0 ** -24)[:, None]


def check_route(gpu, logits, top, sorted_too=True, **spec):
    import torch
    tokens, experts = logits.shape
    ids, w = ints(tokens * top).view(tokens, top), torch.full((tokens, top), float("nan"), device="cuda")
    places = {}
    if sorted_too:
        need = gpu.moe_sort_bytes(tokens, top, experts)
        places = dict(offsets=ints(experts + 1), row=ints(tokens * top), slot=ints(tokens * top),
                      work=torch.full((need,), 0x5A, dtype=torch.uint8, device="cuda") if need else None)
    b = spec.pop("bias", None)
    gpu.moe_route(logits, ids, w, bias=None if b is None else dev(b), **spec, **places)
    torch.cuda.synchronize()
    spec["bias"] = b
    lh = host(logits)
    want_ids, want = moe_ref.route(lh, top, **spec)
    got = host(ids)
    bad = np.nonzero((got != want_ids).any(1))[0]
    assert not bad.size, (bad[:5], got[bad[:3]].tolist(), want_ids[bad[:3]].tolist())
    gw = host(w).astype(np.float64)
    tol = weight_tolerance(lh, want, spec) * np.abs(want) + 2.0 ** -149
    assert (np.abs(gw - want) <= tol).all(), np.max(np.abs(gw - want) / np.maximum(tol, 1e-300))
    if sorted_too:
        for got, want, name in zip((places["offsets"], places["row"], places["slot"]), moe_ref.sort(want_ids, experts), ("offsets", "row", "slot")):
            assert np.array_equal(host(got), want), name


ROUTE = [  # tokens, experts, top, groups, kept, best
    (1, 1, 1, 1, 1, 1), (1, 32, 4, 1, 1, 1), (3, 2, 2, 2, 1, 1), (20, 8, 2, 1, 1, 1), (17, 63, 7, 1, 1, 1), (64, 256, 8, 8, 4, 2),
    (9, 65, 16, 5, 2, 2), (40, 160, 6, 8, 3, 1), (11, 256, 17, 4, 4, 1), (27, 257, 8, 1, 1, 1), (5, 384, 64, 48, 17, 2),
    (18, 512, 22, 64, 9, 1), (10, 1000, 33, 10, 3, 2), (9, 1024, 64, 1, 1, 1), (12, 1025, 3, 5, 4, 2), (10, 4096, 64, 64, 16, 2),
    (9, 4095, 5, 63, 2, 1), (27, 64, 8, 64, 12, 2), (1030, 64, 8, 1, 1, 1), (1100, 256, 16, 8, 4, 2), (1500, 96, 5, 4, 2, 1),
    (1025, 30, 3, 1, 1, 1), (1024, 16, 16, 16, 5, 2), (2000, 128, 8, 16, 4, 2), (1027, 7, 4, 7, 4, 1),
    # where the lanes of a token change, and where the sort is in the same launch
    (64, 64, 8, 1, 1, 1), (65, 64, 8, 8, 4, 2), (8, 200, 6, 8, 4, 2), (9, 256, 8, 1, 1, 1), (2049, 256, 8, 8, 4, 2), (2050, 100, 16, 5, 3, 1),
    (4100, 200, 7, 1, 1, 1), (2048, 66, 5, 6, 3, 2),
]


@pytest.mark.parametrize("tokens,experts,top,groups,kept,best", ROUTE)
def test_route(gpu, tokens, experts, top, groups, kept, best):
    rng = np.random.default_rng(tokens * 7 + experts)
    bias = (0.2 * rng.standard_normal(experts)).astype(np.float32)
    shut = bias.copy()
    shut[rng.random(experts) < 0.2] = -np.inf
    shut[rng.random(experts) < 0.1] = np.nan
    shut[rng.random(experts) < 0.1] = np.inf
    combos = list(itertools.product((moe_ref.SOFTMAX, moe_ref.SIGMOID), (None, bias, shut), (True, False)))
    for i, (score, b, renormalise) in enumerate(combos if tokens < 1000 else combos[::3]):
        kind = ("plain", "ties", "edges")[i % 3]
        x = dev(logits_of(rng, tokens, experts, kind), ("f32", "f16", "bf16")[(i // 3) % 3] if kind != "edges" else "f32")
        check_route(gpu, x, top, sorted_too=i % 2 == 0, score=score, bias=b, groups=groups, groups_kept=kept, group_best=best,
                    renormalise=renormalise, scale=(1.0, 2.5)[i % 2])


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bias", [False, True])
def test_route_strides(gpu, type, bias):
    """Rows of any stride and alignment, infinities of the narrow types among them."""
    import torch
    rng = np.random.default_rng(5)
    for tokens, experts, ld, off in ((33, 40, 41, 1), (1050, 96, 99, 3), (7, 300, 512, 5)):
        buf = dev(logits_of(rng, 1, tokens * ld + off, "plain")[0], type)
        x = torch.as_strided(buf, (tokens, experts), (ld, 1), off)
        x[1, 2], x[2, :3], x[3, 5] = float("inf"), float("-inf"), float("nan")
        b = rng.standard_normal(experts).astype(np.float32) if bias else None
        check_route(gpu, x, 6, score=moe_ref.SIGMOID if bias else moe_ref.SOFTMAX, bias=b)


def test_route_far_offsets(gpu):
    """Rows behind 2^31 elements."""
    import torch
    torch.cuda.empty_cache()
    rng = np.random.default_rng(6)
    ld = (1 << 31) // 3 + 64
    buf = torch.empty(4 * ld, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(buf, (5, 60), (ld - 64, 1), 0)
    x.copy_(dev(logits_of(rng, 5, 60, "plain"), "bf16"))
    check_route(gpu, x, 4)
    del buf, x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("experts", [64, 256, 1000])
def test_scores_near_one(gpu, experts):
    """Scores that 32 bits cannot tell apart: the logits' order without a bias, the 64-bit sums' with one."""
    l = np.zeros((4, experts), np.float32)
    l[0] = 20.0 + np.arange(experts) * 2.0 ** -10           # sigmoid: 1 - 2e-9 and less
    l[1] = 20.0 - np.arange(experts) * 2.0 ** -10
    l[2] = np.float32(1.0) + np.arange(experts) * np.float32(2.0 ** -23)
    l[3] = np.float32(1.0) - np.arange(experts) * np.float32(2.0 ** -24)
    l = np.concatenate([l, logits_of(np.random.default_rng(4), 5, experts, "plain")])
    shut = np.zeros(experts, np.float32)   # whole groups that are shut out beside near ones
    shut[:experts // 8] = -np.inf
    most = np.full(experts, -np.inf, np.float32)
    most[experts // 8 * 3:experts // 8 * 4] = 0.0
    large = (np.random.default_rng(3).integers(-3, 4, experts) * 2.0 ** 20).astype(np.float32)   # 32 bits keep an eighth of a score's range
    for bias in (None, np.zeros(experts, np.float32), np.full(experts, -1.0, np.float32), np.full(experts, 100.0, np.float32), shut, most,
                 large, np.full(experts, 1e6, np.float32)):
        for score in (moe_ref.SIGMOID, moe_ref.SOFTMAX):
            check_route(gpu, dev(l), 8, score=score, bias=bias)
            for kept in (2, 7):
                check_route(gpu, dev(l), 8, score=score, bias=bias, groups=8, groups_kept=kept, group_best=2)
                check_route(gpu, dev(l), 8, score=score, bias=bias, groups=8, groups_kept=kept, group_best=1, renormalise=False)


def test_many_equals(gpu):
    """More equals than there is room for: the lowest indices, of experts and of groups."""
    for tokens, experts in ((3, 64), (5, 256), (2100, 256), (3, 700)):
        x = np.zeros((tokens, experts), np.float32)
        x[1] = np.where(np.arange(experts) % 3 == 1, 0.5, -0.25)
        x[2, experts // 2:] = 1.0
        for score in (moe_ref.SOFTMAX, moe_ref.SIGMOID):
            for bias in (None, np.zeros(experts, np.float32), np.where(np.arange(experts) % 2, 0.25, 0.0).astype(np.float32)):
                check_route(gpu, dev(x), 16, score=score, bias=bias)
                check_route(gpu, dev(x), 7, score=score, bias=bias, groups=4, groups_kept=2, group_best=2, renormalise=False)


SORT = [(0, 4, 7), (1, 1, 1), (1, 3, 2), (33, 2, 8), (100, 7, 300), (1024, 8, 64), (1023, 8, 513), (1025, 8, 1024), (2500, 3, 1025), (7, 4096, 9),
        (2731, 3, 4096), (8193, 1, 5), (4096, 4, 128), (30001, 8, 256), (100003, 3, 2049), (131072, 8, 4096), (300000, 7, 1)]


@pytest.mark.parametrize("tokens,top,experts", SORT)
def test_sort(gpu, tokens, top, experts):
    import torch
    rng = np.random.default_rng(tokens + experts)
    p = np.exp(0.7 * rng.standard_normal(experts))
    ids = rng.choice(experts, (tokens, top), p=p / p.sum()).astype(np.int32)
    drop = rng.random((tokens, top))
    ids = np.where(drop < 0.05, rng.choice(np.array([-1, experts, -2 ** 31, 2 ** 31 - 1, -77], np.int64), (tokens, top)), ids).astype(np.int32)
    for which in (ids, np.full_like(ids, experts - 1), np.full_like(ids, -1)):
        n = tokens * top
        offsets, row, slot = ints(experts + 3), ints(n + 3), ints(n + 3)
        need = gpu.moe_sort_bytes(tokens, top, experts)
        work = torch.full((need + 8,), 0x5A, dtype=torch.uint8, device="cuda")
        if tokens:
            gpu.moe_sort(dev(which), experts, offsets, row, slot, work[:need] if need else None)
        else:
            assert gpu.load().eif_hip_moe_sort(None, 0, top, experts, gpu.ptr(offsets), None, None, None, 0, gpu.stream_ptr()) == 0
        torch.cuda.synchronize()
        wo, wr, ws = moe_ref.sort(which, experts)
        assert np.array_equal(host(offsets)[:-2], wo) and np.array_equal(host(row)[:n], wr) and np.array_equal(host(slot)[:n], ws)
        assert (host(offsets)[-2:] == -7).all() and (host(row)[n:] == -7).all() and (host(slot)[n:] == -7).all() and (host(work)[need:] == 0x5A).all()


COMBINE = [(1, 1, 1), (8, 4, 2560), (3, 7, 65), (5, 12, 1000), (100, 2, 64), (300, 8, 257), (2, 3, 8192), (17, 9, 1028), (700, 5, 20), (1, 64, 4100)]


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,top,dim", COMBINE)
def test_combine(gpu, type, tokens, top, dim):
    import torch
    rng = np.random.default_rng(tokens + dim)
    rows = tokens * top + 3
    y = rng.standard_normal((rows, dim)).astype(np.float32)
    slot = rng.permutation(tokens * top).astype(np.int32).reshape(tokens, top)
    slot[rng.random(slot.shape) < 0.1] = -1
    slot[rng.random(slot.shape) < 0.05] = rows
    slot[rng.random(slot.shape) < 0.05] = 2 ** 31 - 1
    slot[rng.random(slot.shape) < 0.05] = 1   # the same row twice
    if tokens > 2:
        slot[1] = -1
    y[rows - 1] = np.nan   # no slot names it
    w = rng.standard_normal((tokens, top)).astype(np.float32)
    w[slot < 0] = np.nan
    add = rng.standard_normal((tokens, dim)).astype(np.float32)
    for ww, aa in ((w, add), (None, None), (w, None), (None, add)):
        buf = torch.full((tokens, dim + 8), 99.0, dtype=getattr(torch, TYPES[type]), device="cuda")
        off = 0 if ww is not None else 3
        out = buf[:, off:off + dim]
        gpu.moe_combine(dev(y), dev(slot), out, None if ww is None else dev(ww), None if aa is None else dev(aa))
        torch.cuda.synchronize()
        want, mag = moe_ref.combine(y, slot, ww, aa)
        tol = (top + 1) * 2.0 ** -24 * mag + 1.001 * EPS[type] * np.abs(want) + 2.0 ** -25 * (type == "f16")
        got = host(out).astype(np.float64)
        assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) - tol)
        rest = torch.cat([buf[:, :off], buf[:, off + dim:]], 1)
        assert (rest == 99.0).all()


def test_combine_in_place_and_strides(gpu):
    """The residual is the output; rows of any stride; infinities go where their row goes."""
    import torch
    rng = np.random.default_rng(3)
    for dim, ld in ((64, 64), (64, 100), (61, 67), (1030, 1031)):
        y, slot = rng.standard_normal((40, dim)).astype(np.float32), rng.integers(-1, 40, (30, 3)).astype(np.int32)
        y[7, 5] = np.inf
        h = rng.standard_normal((30, ld)).astype(np.float32)
        d = dev(h)
        yd = torch.full((40, ld + 4), float("nan"), device="cuda")
        yd[:, :dim] = dev(y)
        gpu.moe_combine(yd[:, :dim], dev(slot), d[:, :dim], None, d[:, :dim])
        torch.cuda.synchronize()
        want, mag = moe_ref.combine(y, slot, None, h[:, :dim])
        got = host(d)
        fin = np.isfinite(want)
        assert np.array_equal(got[:, :dim][~fin], want[~fin]) and (~fin).sum() == (slot == 7).any(1).sum()
        assert (np.abs(got[:, :dim][fin] - want[fin]) <= 5 * 2.0 ** -24 * mag[fin]).all() and np.array_equal(got[:, dim:], h[:, dim:])


def test_combine_far_offsets(gpu):
    """Rows of y, of the residual and of the output behind 2^31 elements."""
    import torch
    torch.cuda.empty_cache()
    ld = (1 << 30) + 4
    buf = torch.zeros(3 * ld, device="cuda")
    y = torch.as_strided(buf, (4, 128), (ld - 256, 1), 0)
    a = torch.as_strided(buf, (4, 128), (ld - 256, 1), 256)
    o = torch.as_strided(buf, (4, 128), (ld - 256, 1), 512)
    rng = np.random.default_rng(4)
    yh, ah = rng.standard_normal((2, 4, 128)).astype(np.float32)
    y.copy_(dev(yh)), a.copy_(dev(ah))
    slot = np.array([[3, 0], [2, 3], [1, 1], [3, 3]], np.int32)
    gpu.moe_combine(y, dev(slot), o, None, a)
    torch.cuda.synchronize()
    want, mag = moe_ref.combine(yh, slot, None, ah)
    assert (np.abs(host(o) - want) <= 3 * 2.0 ** -24 * mag).all()
    del buf, y, a, o
    torch.cuda.empty_cache()


class Layer:
    """A routed feed-forward on MXFP4 experts: router, sorted rows, gated products, down products, weighted sum and residual."""

    def __init__(self, gpu, tokens, dim, hidden, experts, top, seed=1):
        import torch
        rng = np.random.default_rng(seed)
        self.gpu, self.tokens, self.dim, self.hidden, self.experts, self.top = gpu, tokens, dim, hidden, experts, top
        self.router = (rng.standard_normal((experts, dim)) * 127 / 4).clip(-127, 127).astype(np.int8)
        self.rscale = np.full(experts, 4 / 127 / np.sqrt(dim), np.float32)
        self.rw = gpu.QWeight(gpu.W_INT8, experts, dim, 0, self.router, self.rscale)
        self.bias = (0.1 * rng.standard_normal(experts)).astype(np.float32)
        gc, gs = mx4_ref.quantise(mx4_ref.matrix(rng, experts * 2 * hidden, dim))
        dc, ds = mx4_ref.quantise(mx4_ref.matrix(rng, experts * dim, hidden))
        self.gv = mx4_ref.values(gc, gs, dim).reshape(experts, 2 * hidden, dim)
        self.dv = mx4_ref.values(dc, ds, hidden).reshape(experts, dim, hidden)
        self.gu = gpu.Mx4Weight(2 * hidden, dim, gc, gs, experts=experts)
        self.down = gpu.Mx4Weight(dim, hidden, dc, ds, experts=experts)
        n, kd, kh = tokens * top, gpu.mx4_kpad(dim), gpu.mx4_kpad(hidden)
        f = lambda *s: torch.zeros(s, device="cuda")   # noqa: E731
        u = lambda *s: torch.zeros(s, dtype=torch.uint8, device="cuda")   # noqa: E731
        self.x, self.out, self.logits, self.w = f(tokens, dim), f(tokens, dim), f(tokens, experts), f(tokens, top)
        self.xq, self.xqs = torch.zeros((tokens, self.rw.kpad), dtype=torch.int8, device="cuda"), f(tokens)
        self.ids, self.slot = ints(n).view(tokens, top), ints(n).view(tokens, top)
        self.offsets, self.row = ints(experts + 1), ints(n)
        self.work = u(max(4, gpu.moe_sort_bytes(tokens, top, experts)))
        self.xc, self.xs, self.hc, self.hs = u(tokens, kd // 2), u(tokens, kd // 32), u(n, kh // 2), u(n, kh // 32)
        self.h, self.y = f(n, hidden), f(n, dim)
        self.biasd = dev(self.bias)

    def run(self):
        g = self.gpu
        g.prep_rows(self.x, self.xq, self.xqs, 0, 1.0)
        self.rw.linear(self.xq, self.xqs, self.logits)
        g.moe_route(self.logits, self.ids, self.w, score=g.SCORE_SIGMOID, bias=self.biasd, scale=1.5, offsets=self.offsets, row=self.row,
                    slot=self.slot, work=self.work)
        g.mx4_quant_rows(self.x, self.xc, self.xs)
        self.gu.linear_grouped(self.xc, self.xs, self.offsets, self.h, self.row, glu=True)
        g.mx4_quant_rows(self.h, self.hc, self.hs)
        self.down.linear_grouped(self.hc, self.hs, self.offsets, self.y)
        g.moe_combine(self.y, self.slot, self.out, self.w, self.x)

    def check(self):
        """Every step against 64 bits, on what the step before it left."""
        x, logits = host(self.x), host(self.logits)
        xq = host(self.xq)[:, :self.dim].astype(np.float64) * host(self.xqs)[:, None]
        want = xq @ (self.router.astype(np.float64) * self.rscale[:, None]).T
        assert np.allclose(logits, want, rtol=1e-5, atol=1e-6)
        ids, w = moe_ref.route(logits, self.top, moe_ref.SIGMOID, self.bias, scale=1.5)
        assert np.array_equal(host(self.ids), ids) and np.allclose(host(self.w), w, rtol=2.0 ** -23)
        o, r, s = moe_ref.sort(ids, self.experts)
        assert np.array_equal(host(self.offsets), o) and np.array_equal(host(self.row)[:o[-1]], r[:o[-1]])
        assert np.array_equal(host(self.slot).ravel(), s)
        xv = mx4_ref.values(*mx4_ref.quantise(x), self.dim)
        h, y = host(self.h), host(self.y)
        hv = mx4_ref.values(*mx4_ref.quantise(h), self.hidden)
        for e in range(self.experts):
            at = slice(o[e], o[e + 1])
            for got, (v, tol) in ((h[at], mx4_ref.product(xv[r[at]], self.gv[e], glu=True)), (y[at], mx4_ref.product(hv[at], self.dv[e]))):
                assert (np.abs(got - v) <= tol).all()
        want, mag = moe_ref.combine(y, s.reshape(ids.shape), host(self.w), x)
        assert (np.abs(host(self.out) - want) <= (self.top + 2) * 2.0 ** -24 * mag).all()


@pytest.mark.parametrize("tokens,dim,hidden,experts,top", [(1, 256, 64, 8, 2), (9, 320, 96, 32, 4), (130, 256, 128, 16, 3), (1200, 128, 64, 24, 8)])
def test_routed_feed_forward(gpu, tokens, dim, hidden, experts, top):
    import torch
    layer = Layer(gpu, tokens, dim, hidden, experts, top)
    for seed in (1, 2):
        layer.x.copy_(dev(mx4_ref.activations(np.random.default_rng(seed), tokens, dim)))
        layer.run()
        torch.cuda.synchronize()
        layer.check()


@pytest.mark.parametrize("tokens", [3, 1100])
def test_routed_feed_forward_in_a_graph(gpu, tokens):
    """Captured once, replayed on other inputs with the program's own work between: every replay is the eager result."""
    import torch
    layer = Layer(gpu, tokens, 256, 64, 16, 8)
    layer.run()   # the first call outside: the INT8 linear allocates on its first batch
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        layer.run()
    for seed in range(4):
        layer.x.copy_(dev(mx4_ref.activations(np.random.default_rng(seed), tokens, 256)))
        layer.run()
        torch.cuda.synchronize()
        want = [t.clone() for t in (layer.out, layer.w, layer.ids, layer.offsets, layer.slot)]
        for t in (layer.out, layer.w, layer.ids, layer.offsets, layer.slot):
            t.fill_(3)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, (layer.out, layer.w, layer.ids, layer.offsets, layer.slot)):
            assert torch.equal(a, b)
    layer.check()


def test_calls_at_once(gpu):
    """Calls of two streams, with outputs and workspaces of their own, on the same logits."""
    import torch
    rng = np.random.default_rng(8)
    tokens, experts, top = 9000, 200, 6
    x = dev(logits_of(rng, tokens, experts, "plain"))
    need = gpu.moe_sort_bytes(tokens, top, experts)
    assert need
    sets = []
    for i in range(2):
        st = torch.cuda.Stream()
        o = dict(offsets=ints(experts + 1), row=ints(tokens * top), slot=ints(tokens * top),
                 work=torch.empty(need, dtype=torch.uint8, device="cuda"))
        sets.append((st, ints(tokens * top).view(tokens, top), torch.zeros((tokens, top), device="cuda"), o))
    torch.cuda.synchronize()
    for _ in range(5):
        for st, ids, w, o in sets:
            gpu.moe_route(x, ids, w, stream=st, **o)
    torch.cuda.synchronize()
    want = moe_ref.sort(moe_ref.route(host(x), top)[0], experts)
    for _, ids, w, o in sets:
        for got, v in zip((o["offsets"], o["row"], o["slot"]), want):
            assert np.array_equal(host(got), v)
