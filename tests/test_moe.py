"""Routing to experts and adapters without a GPU: the references of the tests on cases worked out by hand, and what the host code
refuses or launches, on the stand-in for the HIP runtime (fakehip/fakehip.cpp)."""
import numpy as np
import pytest

import moe_ref
from test_host_launches import fake, run  # noqa: F401


def test_reference_choice():
    inf, nan = np.inf, np.nan
    l = [[0.0, 2.0, 1.0, 2.0], [nan, -inf, 0.5, -inf], [-inf] * 4, [inf, 3.0, inf, nan]]
    ids, w = moe_ref.route(l, 3)
    assert ids.tolist() == [[1, 3, 2], [2, -1, -1], [-1, -1, -1], [0, 2, 1]]
    e = np.exp([0.0, 0.0, -1.0])
    assert np.allclose(w[0], e / e.sum()) and w[1].tolist() == [1, 0, 0] and not w[2].any() and w[3].tolist() == [0.5, 0.5, 0]
    ids, w = moe_ref.route(l[:1], 2, moe_ref.SIGMOID, bias=[1.0, 0.0, -inf, 0.0], renormalise=False, scale=2.0)
    assert ids.tolist() == [[0, 1]] and np.allclose(w, [[1.0, 2 / (1 + np.exp(-2.0))]])


def test_reference_groups():
    # three groups of two; by the best one: 1, 5, 4; by the two best (scores of a sigmoid): both high in the first
    l = [[1.0, 1.0, 5.0, -9.0, 4.0, -9.0]]
    assert moe_ref.route(l, 2, moe_ref.SIGMOID, groups=3, groups_kept=1)[0].tolist() == [[2, 3]]
    assert moe_ref.route(l, 2, moe_ref.SIGMOID, groups=3, groups_kept=1, group_best=2)[0].tolist() == [[0, 1]]
    assert moe_ref.route(l, 4, moe_ref.SIGMOID, groups=3, groups_kept=1)[0].tolist() == [[2, 3, -1, -1]]


def test_reference_sort_and_combine():
    ids = np.array([[2, 0], [-1, 2], [5, 0]], np.int32)
    o, r, s = moe_ref.sort(ids, 3)
    assert o.tolist() == [0, 2, 2, 4] and r.tolist() == [0, 2, 0, 1, -7, -7] and s.tolist() == [2, 0, -1, 3, -1, 1]
    y = np.arange(8.0).reshape(4, 2)
    out, _ = moe_ref.combine(y, s.reshape(3, 2), np.full((3, 2), 0.5), np.ones((3, 2)))
    assert out.tolist() == [[3.0, 4.0], [4.0, 4.5], [2.0, 2.5]]


CALLS = """
    ARG = -1
    at = lambda n: vp(X.value + n)
    def spec_of(**kw):
        d = dict(experts=64, top_k=4, score=0, bias=None, groups=1, groups_kept=1, group_best=1, renormalise=1, scale=1.0)
        d.update(kw)
        return bh.MoeRouteSpec(**d)
    def route(logits=X, type=0, ldl=64, tokens=3, ids=X, weights=X, offsets=None, row=None, slot=None, work=None, bytes=0, spec=True, **kw):
        fake.fake_reset()
        s = spec_of(**kw) if spec else None
        rc = lib.eif_hip_moe_route(logits, type, ldl, tokens, C.byref(s) if s else None, ids, weights, offsets, row, slot, work, bytes, None)
        return rc
    def sort(ids=X, tokens=3, top=4, experts=64, offsets=X, row=X, slot=X, work=None, bytes=0):
        fake.fake_reset()
        return lib.eif_hip_moe_sort(ids, tokens, top, experts, offsets, row, slot, work, bytes, None)
    def combine(y=X, ldy=64, rows=12, slot=X, weights=X, tokens=3, top=4, add=None, lda=0, dim=64, out=X, type=0, ldo=64):
        fake.fake_reset()
        return lib.eif_hip_moe_combine(y, ldy, rows, slot, weights, tokens, top, add, lda, dim, out, type, ldo, None)
"""


def test_route_refuses(fake):  # noqa: F811
    run(fake, CALLS + """
    inf, nan = float("inf"), float("nan")
    assert route() == 0 and fake.fake_launches() == 1
    assert route(tokens=0, logits=None, ids=None, weights=None) == 0 and fake.fake_launches() == 0
    assert route(offsets=X, row=X, slot=X) == 0 and route(type=1, logits=at(2)) == 0 and route(bias=X.value) == 0
    assert route(groups=8, groups_kept=3, group_best=2) == 0 and route(scale=-2.0) == 0
    for bad in (dict(spec=False), dict(tokens=-1), dict(type=3), dict(type=-1), dict(ldl=63), dict(logits=None), dict(ids=None),
                dict(weights=None), dict(experts=0), dict(top_k=0), dict(top_k=65), dict(score=2), dict(score=-1), dict(groups=0),
                dict(groups=3), dict(groups=128), dict(groups_kept=0), dict(groups_kept=2), dict(group_best=0), dict(group_best=3),
                dict(scale=inf), dict(scale=nan), dict(bias=at(2).value), dict(logits=at(2)), dict(type=2, logits=at(1)), dict(ids=at(2)),
                dict(weights=at(1)), dict(offsets=X), dict(row=X), dict(offsets=X, row=X), dict(offsets=X, row=X, slot=at(2)),
                dict(offsets=X, row=X, slot=X, work=at(2)), dict(offsets=X, row=X, slot=X, tokens=4096)):
        assert route(**bad) == ARG and fake.fake_launches() == 0, bad
    assert route(experts=4096, top_k=64, ldl=4096) == 0 and route(experts=4097, top_k=4, ldl=5000) == LIMIT
    assert route(experts=128, top_k=65, ldl=128) == LIMIT and route(experts=128, ldl=128, groups=128, groups_kept=1) == LIMIT
    assert route(tokens=1 << 25, ldl=1 << 36) == 0 and route(tokens=(1 << 25) + 1) == LIMIT
    assert route(tokens=1 << 25, top_k=32) == 0 and route(tokens=1 << 25, top_k=33) == LIMIT
    assert route(tokens=1 << 25, experts=4096, ldl=4096, bias=X.value, groups=2, groups_kept=1) == 0
    fake.fake_reset(); fake.fake_fail_launch(0)
    s = spec_of()
    assert lib.eif_hip_moe_route(X, 0, 64, 3, C.byref(s), X, X, X, X, X, None, 0, None) == DEVICE and fake.fake_launches() == 1
    """)


def test_sort_refuses(fake):  # noqa: F811
    run(fake, CALLS + """
    size = lib.eif_hip_moe_sort_bytes
    assert sort() == 0 and fake.fake_launches() == 1 and size(3, 4, 64) == 0
    assert sort(tokens=0, ids=None, row=None, slot=None) == 0 and fake.fake_launches() == 1
    for bad in (dict(ids=None), dict(tokens=-1), dict(top=0), dict(experts=0), dict(offsets=None), dict(row=None), dict(slot=None),
                dict(ids=at(2)), dict(offsets=at(1)), dict(row=at(2)), dict(slot=at(3)), dict(work=at(2))):
        assert sort(**bad) == ARG and fake.fake_launches() == 0, bad
    assert sort(experts=4097) == LIMIT and sort(top=4097) == LIMIT and sort(tokens=(1 << 28) + 1) == LIMIT
    for tokens, top, experts in ((1 << 15, 8, 128), (1 << 28, 4, 4096), (70000, 1, 1)):
        need = size(tokens, top, experts)
        assert need > 0 and need % (4 * experts) == 0 and need <= 256 * 4 * experts
        assert sort(tokens=tokens, top=top, experts=experts) == ARG
        assert sort(tokens=tokens, top=top, experts=experts, work=X, bytes=need - 1) == ARG and fake.fake_launches() == 0
        assert sort(tokens=tokens, top=top, experts=experts, work=X, bytes=need) == 0 and fake.fake_launches() == 2
        fake.fake_fail_launch(2)
    assert [size(*a) for a in ((0, 4, 64), (-1, 4, 64), (1 << 15, 0, 64), (1 << 15, 4, 0), (1 << 15, 4, 4097), ((1 << 28) + 1, 4, 64))] == [0] * 6
    fake.fake_reset(); fake.fake_fail_launch(0)
    assert lib.eif_hip_moe_sort(X, 1 << 15, 8, 128, X, X, X, X, 1 << 20, None) == DEVICE and fake.fake_launches() == 1
    """)


def test_combine_refuses(fake):  # noqa: F811
    run(fake, CALLS + """
    assert combine() == 0 and fake.fake_launches() == 1 and combine(weights=None) == 0 and combine(rows=0, y=None) == 0
    assert combine(tokens=0, y=None, slot=None, out=None) == 0 and fake.fake_launches() == 0
    assert combine(add=X, lda=64) == 0 and combine(add=at(4), lda=64, type=2, out=at(2)) == 0
    for bad in (dict(y=None), dict(slot=None), dict(out=None), dict(tokens=-1), dict(rows=-1), dict(top=0), dict(dim=0), dict(ldy=63),
                dict(ldo=63), dict(add=X, lda=63), dict(type=3), dict(type=-1), dict(y=at(2)), dict(slot=at(2)), dict(weights=at(2)),
                dict(add=at(2), lda=64), dict(out=at(2)), dict(type=1, out=at(1)), dict(add=X, lda=64, type=1), dict(add=X, lda=128)):
        assert combine(**bad) == ARG and fake.fake_launches() == 0, bad
    big = 1 << 24
    assert combine(dim=big + 1, ldy=big + 1, ldo=big + 1) == LIMIT and combine(dim=big, ldy=big, ldo=big) == 0
    assert combine(tokens=big - 1, top=1) == 0 and combine(tokens=big, top=1) == LIMIT and combine(tokens=1 << 23, top=129) == LIMIT
    assert combine(tokens=511, top=1, dim=1 << 23, ldy=big, ldo=big) == 0 and combine(tokens=512, top=1, dim=1 << 23, ldy=big, ldo=big) == LIMIT
    assert combine(tokens=511, top=1, dim=(1 << 23) - 1, ldy=big, ldo=big, y=at(4)) == 0
    """)


@pytest.mark.parametrize("tokens,experts,top,bias,launches,grid,block", [
    (1, 32, 4, False, 1, 1, 64), (64, 64, 8, False, 1, 1, 1024), (65, 64, 8, False, 2, 17, 64), (8, 256, 8, True, 1, 1, 512),
    (9, 256, 8, True, 2, 9, 64), (2048, 256, 8, True, 3, 2048, 64), (2049, 256, 8, True, 3, 513, 64), (16001, 256, 8, True, 3, 1001, 256),
    (3, 4096, 8, False, 2, 3, 64), (5000, 4096, 64, True, 3, 5000, 64), (600, 1024, 17, False, 3, 600, 64), (4096, 64, 1, False, 2, 1024, 64),
])
def test_route_launches(fake, tokens, experts, top, bias, launches, grid, block):  # noqa: F811
    """A few tokens are chosen and sorted in one launch; up to 4096 pairs are sorted in one, more in two."""
    run(fake, CALLS + f"""
    tokens, experts, top = {tokens}, {experts}, {top}
    need = lib.eif_hip_moe_sort_bytes(tokens, top, experts)
    assert route(tokens=tokens, experts=experts, ldl=experts, top_k=top, bias=X.value if {bias} else None, score=1, offsets=X, row=X, slot=X,
                 work=X, bytes=need) == 0
    assert fake.fake_launches() == {launches} and (fake.fake_launch_grid(0), fake.fake_launch_block(0)) == ({grid}, {block})
    assert (need > 0) == (tokens * top > 4096)
    assert route(tokens=tokens, experts=experts, ldl=experts, top_k=top, bias=X.value if {bias} else None, score=1) == 0
    assert fake.fake_launches() == 1
    """)


ADAPTERS = """
    ARG, LIMIT, NOMEM, DEVICE = -1, -4, -3, -2
    at = lambda n: vp(X.value + n)
    def create(slots=3, rows=64, cols=96, rank=16, type=2, out=True):
        h = vp(1)
        rc = lib.eif_hip_adapters_create(C.byref(h) if out else None, slots, rows, cols, rank, type)
        assert not out or (rc == 0) == bool(h.value)
        return rc, h
"""


def test_adapters_create_and_give_back(fake):  # noqa: F811
    run(fake, ADAPTERS + """
    def rc(**kw):
        r, h = create(**kw)
        lib.eif_hip_adapters_destroy(h if r == 0 else None)
        return r
    assert rc() == 0 and fake.fake_live() == 0
    for bad in (dict(out=False), dict(slots=0), dict(rows=0), dict(cols=0), dict(rank=0), dict(type=3), dict(type=-1)):
        assert rc(**bad) == ARG, bad
    for big in (dict(slots=65537), dict(rows=(1 << 20) + 1), dict(cols=(1 << 20) + 1), dict(rank=257)):
        assert rc(**big) == LIMIT, big
    fake.fake_reset(); fake.fake_fail_malloc(1)
    assert rc() == NOMEM and fake.fake_live() == 0
    fake.fake_reset()
    r, h = create()
    i, b = [C.c_int() for _ in range(5)], C.c_size_t()
    assert lib.eif_hip_adapters_info(h, *map(C.byref, i), C.byref(b)) == 0 and [v.value for v in i] == [3, 64, 96, 16, 2]
    assert b.value == 3 * (16 * (96 + 64) * 2 + 8)
    assert lib.eif_hip_adapters_info(h, None, None, None, None, None, None) == 0
    assert lib.eif_hip_adapters_info(None, None, None, None, None, None, None) == ARG
    lib.eif_hip_adapters_destroy(h); lib.eif_hip_adapters_destroy(None)
    assert fake.fake_live() == 0
    """)


def test_adapters_set_refuses(fake):  # noqa: F811
    run(fake, ADAPTERS + """
    rc, h = create()
    def put(slot=1, rank=8, A=X, lda=96, B=X, ldb=8, scale=1.0, dev=1, h=h):
        fake.fake_reset()
        return lib.eif_hip_adapters_set(h, slot, rank, A, lda, B, ldb, scale, dev, None)
    live = fake.fake_live()
    assert put() == 0 and put(dev=0) == 0 and put(rank=0, A=None, B=None, lda=0, ldb=0, scale=float("nan")) == 0 and put(rank=16, ldb=16) == 0
    for bad in (dict(h=None), dict(slot=-1), dict(slot=3), dict(rank=-1), dict(rank=17, ldb=17), dict(A=None), dict(B=None), dict(lda=95),
                dict(ldb=7), dict(scale=float("inf")), dict(scale=float("nan")), dict(A=at(1)), dict(B=at(1))):
        assert put(**bad) == ARG and fake.fake_launches() == 0, bad
    assert put(lda=1 << 60) == LIMIT and put(ldb=1 << 60) == LIMIT
    fake.fake_device(1)
    assert put() == ARG
    fake.fake_device(0)
    fake.fake_fail_malloc(1)
    assert lib.eif_hip_adapters_set(h, 1, 8, X, 96, X, 8, 1.0, 0, None) == NOMEM and fake.fake_live() == live
    fake.fake_reset(); fake.fake_fail_launch(0)
    assert lib.eif_hip_adapters_set(h, 1, 8, X, 96, X, 8, 1.0, 0, None) == DEVICE and fake.fake_live() == live
    lib.eif_hip_adapters_destroy(h)
    """)


def test_adapters_linear_refuses(fake):  # noqa: F811
    run(fake, ADAPTERS + """
    rc, h = create()
    def linear(x=X, type=0, ldx=96, slot=X, base=at(64), ldbase=64, y=X, ldy=64, M=5, h=h):
        fake.fake_reset()
        return lib.eif_hip_adapters_linear(h, x, type, ldx, slot, base, ldbase, y, ldy, M, None)
    assert linear() == 0 and fake.fake_launches() == 1 and linear(base=None, ldbase=0) == 0 and linear(base=X) == 0
    assert linear(M=0, x=None, y=None, slot=None, base=None) == 0 and fake.fake_launches() == 0
    assert linear(M=1 << 24) == 0 and linear(M=(1 << 24) + 1) == LIMIT and linear(M=5000, type=1, x=at(2)) == 0
    for bad in (dict(h=None), dict(x=None), dict(slot=None), dict(y=None), dict(type=3), dict(type=-1), dict(ldx=95), dict(ldy=63),
                dict(ldbase=63), dict(M=-1), dict(base=X, ldbase=128), dict(x=at(2)), dict(type=2, x=at(1)), dict(slot=at(2)),
                dict(base=at(2)), dict(y=at(2))):
        assert linear(**bad) == ARG and fake.fake_launches() == 0, bad
    fake.fake_device(1)
    assert linear() == ARG and linear(M=0) == ARG
    fake.fake_device(0)
    fake.fake_reset(); fake.fake_fail_launch(0)
    assert lib.eif_hip_adapters_linear(h, X, 0, 96, X, None, 0, X, 64, 5, None) == DEVICE
    lib.eif_hip_adapters_destroy(h)
    """)


@pytest.mark.parametrize("M,rank,block,grid", [
    (1, 16, 1024, 8), (9, 16, 1024, 16), (512, 16, 1024, 512), (513, 16, 512, 40 * 1), (256, 64, 1024, 256), (257, 64, 512, 24), (4095, 16, 512, 256),
    (4096, 16, 512, 128), (1 << 24, 16, 512, 1 << 19),
])
def test_adapters_forms(fake, M, rank, block, grid):  # noqa: F811
    """A row a workgroup up to 512 rows of up to 16 ranks, or 256; then tiles of 16 rows, from 4096 rows on of 32."""
    run(fake, ADAPTERS + f"""
    rc, h = create(rank={rank})
    fake.fake_reset()
    assert rc == 0 and lib.eif_hip_adapters_linear(h, X, 0, 96, X, None, 0, X, 64, {M}, None) == 0
    assert fake.fake_launches() == 1 and (fake.fake_launch_grid(0), fake.fake_launch_block(0)) == ({grid}, {block})
    lib.eif_hip_adapters_destroy(h)
    """)


TENSORS = """
    import torch

    class T:   # the shape, type and strides of a tensor on the device
        def __init__(self, *shape, dtype=torch.float32, cuda=True, stride=None):
            self.t = torch.empty(shape, dtype=dtype) if stride is None else torch.empty(1 << 16, dtype=dtype).as_strided(shape, stride)
            self.is_cuda, self.dtype, self.shape = cuda, dtype, self.t.shape
        def __getattr__(self, n):
            return getattr(self.t, n)

    i32 = torch.int32
    bh.stream_ptr = lambda s=None: None
    def refused(f, *a, **k):
        try:
            f(*a, **k)
        except bh.HipError:
            return True
        return False
"""


def test_binding_looks_at_tensors(fake):  # noqa: F811
    run(fake, TENSORS + """
    def route(logits=(5, 64), ids=(5, 4), weights=(5, 4), sorted=True, tail=0, **kw):
        mk = lambda a, **d: a if isinstance(a, T) else T(*a, **d)
        places = dict(offsets=T(65, dtype=i32), row=T(20 - tail, dtype=i32), slot=T(20, dtype=i32)) if sorted else {}
        bh.moe_route(mk(logits), mk(ids, dtype=i32), mk(weights), **{**places, **kw})
    route(); route(sorted=False); route(bias=T(64)); route(logits=T(5, 64, dtype=torch.bfloat16, stride=(80, 1)))
    for bad in (dict(logits=T(5, 64, dtype=torch.float64)), dict(logits=T(5, 64, cuda=False)), dict(logits=T(5, 64, stride=(1, 5))),
                dict(ids=T(5, 4, dtype=torch.int64)), dict(ids=(4, 4)), dict(weights=(5, 3)), dict(weights=(5, 5)), dict(tail=1),
                dict(ids=T(5, 4, dtype=i32, stride=(8, 1))), dict(bias=T(63)), dict(offsets=T(64, dtype=i32)), dict(slot=None),
                dict(work=T(8, cuda=False)), dict(ids=(5, 65), weights=(5, 65)), dict(score=2)):
        assert refused(route, **bad), bad
    def sort(ids=None, experts=64, offsets=65, row=20, slot=20):
        bh.moe_sort(ids or T(5, 4, dtype=i32), experts, T(offsets, dtype=i32), T(row, dtype=i32), T(slot, dtype=i32))
    sort()
    for bad in (dict(ids=T(5, 4)), dict(ids=T(5, 4, dtype=i32, stride=(8, 1))), dict(offsets=64), dict(row=19), dict(slot=19), dict(experts=0)):
        assert refused(sort, **bad), bad
    def combine(y=None, slot=None, out=None, **kw):
        bh.moe_combine(y or T(20, 32), slot or T(5, 4, dtype=i32), out or T(5, 32), **kw)
    combine(); combine(weights=T(5, 4), add=T(5, 32)); combine(out=T(5, 32, dtype=torch.float16), y=T(20, 40))
    for bad in (dict(y=T(20, 31)), dict(y=T(20, 32, dtype=torch.float16)), dict(slot=T(4, 4, dtype=i32)), dict(slot=T(5, 4)),
                dict(weights=T(5, 3)), dict(weights=T(5, 4, stride=(8, 1))), dict(add=T(4, 32)), dict(add=T(5, 32, dtype=torch.float16)),
                dict(out=T(5, 32, dtype=torch.float64))):
        assert refused(combine, **bad), bad
    h = bh.Adapters(3, 64, 96, 16, torch.bfloat16)
    b16 = torch.bfloat16
    h.set(0, T(8, 96, dtype=b16), T(64, 8, dtype=b16)); h.set(2, T(1, 96, dtype=b16), T(64, 1, dtype=b16), 2.0); h.clear(0)
    for A, B in ((T(8, 95, dtype=b16), T(64, 8, dtype=b16)), (T(8, 96), T(64, 8)), (T(8, 96, dtype=b16), T(64, 7, dtype=b16)),
                 (T(8, 96, dtype=b16, cuda=False), T(64, 8, dtype=b16)), (T(17, 96, dtype=b16), T(64, 17, dtype=b16)),
                 (T(8, 96, dtype=b16, stride=(0, 1)), T(64, 8, dtype=b16)), (T(8, 96, dtype=b16, stride=(1, 8)), T(64, 8, dtype=b16))):
        assert refused(h.set, 0, A, B), (A.shape, B.shape)
    assert refused(h.set, 3, T(8, 96, dtype=b16), T(64, 8, dtype=b16)) and refused(bh.Adapters, 3, 64, 96, 16, torch.int8)
    def linear(x=None, slot=None, y=None, base=None):
        h.linear(x or T(5, 96), slot or T(5, dtype=i32), y or T(5, 64), base)
    linear(); linear(base=T(5, 64)); linear(x=T(5, 96, dtype=torch.float16))
    for bad in (dict(x=T(5, 95)), dict(x=T(5, 96, dtype=torch.float64)), dict(slot=T(4, dtype=i32)), dict(slot=T(5)), dict(y=T(4, 64)),
                dict(y=T(5, 63)), dict(base=T(5, 63)), dict(base=T(5, 64, dtype=b16)), dict(x=T(5, 96, cuda=False))):
        assert refused(linear, **bad), bad
    h.close(); h.close()
    """)
