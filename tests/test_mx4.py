"""The microscaled 4-bit calls without a GPU: the reference of the tests against the format's own examples, and what the
host code refuses or launches, on the stand-in for the HIP runtime (fakehip/fakehip.cpp)."""
import numpy as np
import pytest

import mx4_ref
from test_host_launches import fake, run  # noqa: F401


def test_reference_rounds_as_the_format_says():
    x = np.zeros((1, 32), np.float32)
    x[0, :16] = [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.5, 7.99, -0.25, -0.3, -0.0, 0.2, -5.0001, 0.74]
    c, s = mx4_ref.quantise(x)
    assert s[0, 0] == 127 and not s[0, 1:].any()
    v = mx4_ref.values(c, s, 32)[0, :16]
    assert v.tolist() == [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, 6.0, -0.0, -0.5, -0.0, 0.0, -6.0, 0.5]
    assert c[0, 0] == 6 and c[0, 5] == 0x98   # 4.0 beside 0; -0.25 keeps its sign beside -0.5


def test_reference_scales():
    x = np.zeros((7, 33), np.float32)
    x[:, 0] = [1.0, 1.999, 3.0e38, 1e-40, 2.0 ** -126, np.inf, np.nan]
    c, s = mx4_ref.quantise(x)
    assert s[:, 0].tolist() == [125, 125, 252, 0, 0, 255, 255] and not s[:, 1:].any()
    v = mx4_ref.values(c, s, 33)
    assert v[0, 0] == 1.0 and v[1, 0] == 1.5 and np.isnan(v[5:, :32]).all() and (v[5:, 32] == 0).all()
    assert v[3, 0] == 0.0 and v[4, 0] == 2.0 ** -126


WEIGHT = """
    u8 = C.POINTER(C.c_uint8)

    def mx4(rows, cols, experts=1):
        c = np.zeros((experts * rows, (cols + 1) // 2), np.uint8)
        s = np.zeros((experts * rows, (cols + 31) // 32), np.uint8)
        return bh.Mx4Weight(rows, cols, c, s, experts=experts)

    ARG = -1
    at = lambda n: vp(X.value + n)
"""


def test_quant_refuses(fake):  # noqa: F811
    run(fake, WEIGHT + """
    def q(x=X, type=0, ldx=64, rows=2, cols=64, codes=X, ldc=128, scales=X, lds=8, values=X, ldv=64):
        fake.fake_reset()
        rc = lib.eif_hip_mx4_quant_rows(x, type, ldx, rows, cols, codes, ldc, scales, lds, values, ldv, None)
        assert fake.fake_launches() == (1 if rc == 0 and rows else 0)
        return rc
    assert q() == 0 and q(rows=0) == 0 and q(rows=0, x=None) == 0 and q(values=None, ldv=0) == 0
    assert q(codes=None, scales=None, ldc=0, lds=0) == 0
    assert q(ldc=256) == 0 and q(cols=257, ldx=257, ldv=257, ldc=256, lds=16) == 0
    for bad in (dict(x=None), dict(type=3), dict(type=-1), dict(ldx=63), dict(rows=-1), dict(cols=0), dict(ldc=112),
                dict(ldc=136), dict(lds=0), dict(lds=12), dict(lds=7), dict(codes=None), dict(scales=None), dict(ldv=63),
                dict(codes=None, scales=None, values=None), dict(codes=at(8)), dict(scales=at(4)), dict(values=at(2)),
                dict(x=at(2)), dict(type=1, x=at(1)), dict(cols=257, ldx=257, ldv=257)):
        assert q(**bad) == ARG, bad
    assert q(type=1, x=at(2)) == 0 and q(x=at(4)) == 0
    big = 1 << 24
    assert q(cols=big + 1, ldx=big + 1, ldc=big, lds=big, ldv=big + 1) == LIMIT
    assert q(rows=1 << 30, cols=1 << 20, ldx=1 << 20, ldc=1 << 19, lds=1 << 15, ldv=1 << 20) == LIMIT
    fake.fake_reset(); fake.fake_fail_launch(0)
    assert lib.eif_hip_mx4_quant_rows(X, 0, 64, 2, 64, X, 128, X, 8, None, 0, None) == DEVICE
    assert [lib.eif_hip_mx4_kpad(c) for c in (-1, 0, 1, 256, 257, big, big + 1)] == [0, 0, 256, 256, 512, big, 0]
    """)


def test_create_refuses_and_gives_back(fake):  # noqa: F811
    run(fake, WEIGHT + """
    def create(experts=1, rows=16, cols=64, codes=X, ldc=32, scales=X, lds=2, dev=1, out=True):
        h = vp(1)
        rc = lib.eif_hip_mx4_weight_create(C.byref(h) if out else None, experts, rows, cols, codes, ldc, scales, lds, dev, None)
        assert not out or (rc == 0) == bool(h.value)
        if rc == 0:
            lib.eif_hip_mx4_weight_destroy(h)
        return rc
    assert create() == 0 and create(dev=0) == 0 and fake.fake_live() == 0
    for bad in (dict(out=False), dict(codes=None), dict(scales=None), dict(experts=0), dict(rows=0), dict(cols=0), dict(ldc=31),
                dict(lds=1), dict(cols=65, ldc=32), dict(cols=65, ldc=33)):
        assert create(**bad) == ARG, bad
    assert create(cols=65, ldc=33, lds=3) == 0
    assert create(rows=(1 << 30) + 1) == LIMIT and create(cols=(1 << 24) + 1, ldc=1 << 24, lds=1 << 20) == LIMIT and create(experts=4097) == LIMIT and create(experts=4096) == 0
    assert create(experts=4096, rows=1 << 30, cols=1, ldc=1, lds=1) == LIMIT
    for dev in (0, 1):
        fake.fake_reset(); fake.fake_fail_malloc(1)
        assert create(dev=dev) == -3 and fake.fake_live() == 0
        for i in (0, 1):
            fake.fake_reset(); fake.fake_fail_launch(i)
            assert create(dev=dev) == DEVICE and fake.fake_live() == 0
    fake.fake_reset()
    w = mx4(33, 300, 3)
    i = [C.c_int() for _ in range(4)]; b = C.c_size_t()
    assert lib.eif_hip_mx4_weight_info(w.h, *map(C.byref, i), C.byref(b)) == 0 and [v.value for v in i] == [3, 33, 300, 512]
    assert b.value == (9 + 15) * (2 * 2048 + 256)   # 15 row tiles behind the last and lib.eif_hip_mx4_weight_info(None, None, None, None, None, None) == ARG
    w.close(); w.close(); lib.eif_hip_mx4_weight_destroy(None)
    assert fake.fake_live() == 0
    """)


def test_products_refuse(fake):  # noqa: F811
    run(fake, WEIGHT + """
    w, g, odd = mx4(64, 300), mx4(64, 300, 3), mx4(48, 300)

    def linear(w=w, codes=X, ldc=256, scales=X, lds=16, bias=None, glu=0, y=X, ldy=64, M=5):
        fake.fake_reset()
        rc = lib.eif_hip_mx4_linear(w and w.h, codes, ldc, scales, lds, bias, glu, y, ldy, M, None)
        assert fake.fake_launches() == (1 if rc == 0 and M else 0)
        return rc

    def grouped(w=g, codes=X, ldc=256, scales=X, lds=16, rows_in=5, index=X, offsets=X, bias=None, glu=0, y=X, ldy=64, M=5):
        fake.fake_reset()
        rc = lib.eif_hip_mx4_linear_grouped(w and w.h, codes, ldc, scales, lds, rows_in, index, offsets, bias, glu, y, ldy, M, None)
        assert fake.fake_launches() == (1 if rc == 0 and M and rows_in else 0)
        return rc

    def rows(w=w, x=X, type=0, ldx=300, bias=None, glu=0, y=X, ldy=64, M=5):
        fake.fake_reset()
        rc = lib.eif_hip_mx4_linear_rows(w and w.h, x, type, ldx, bias, glu, y, ldy, M, None)
        assert fake.fake_launches() == (1 if rc == 0 and M else 0)
        return rc

    for f in (linear, grouped, rows):
        assert f() == 0 and f(M=0) == 0 and f(M=0, y=None) == 0 and f(bias=X) == 0
        assert f(glu=1, ldy=32) == 0 and f(glu=1, ldy=31) == ARG
        for bad in (dict(w=None), dict(M=-1), dict(ldy=63), dict(y=None)):
            assert f(**bad) == ARG, (f, bad)
        assert f(w=odd, glu=1) == LIMIT and f(M=(1 << 30) + 1) == LIMIT
        fake.fake_device(1)
        assert f() == ARG      # a weight of another device
        fake.fake_device(0)
    for f in (linear, grouped):
        for bad in (dict(codes=None), dict(scales=None), dict(ldc=240), dict(ldc=264), dict(lds=8), dict(lds=20),
                    dict(codes=at(8)), dict(scales=at(4))):
            assert f(**bad) == ARG, (f, bad)
    for f in (linear, rows):
        assert f(w=g) == ARG   # a stack is for the grouped product
    assert grouped(w=w) == 0 and grouped(rows_in=0) == 0 and grouped(rows_in=-1) == ARG and grouped(index=None) == 0
    assert grouped(offsets=None) == ARG and grouped(offsets=at(2)) == ARG and grouped(index=at(1)) == ARG
    assert rows(ldx=299) == ARG and rows(type=3) == ARG and rows(x=None) == ARG and rows(x=at(2)) == ARG
    assert rows(type=2, x=at(2)) == 0 and rows(type=2, x=at(1)) == ARG
    assert rows(M=8) == 0 and rows(M=9) == LIMIT
    wide = mx4(16, 16385)
    assert rows(w=wide, ldx=16385) == LIMIT
    for f, a in ((lib.eif_hip_mx4_linear, (w.h, X, 256, X, 16, None, 0, X, 64, 5, None)),
                 (lib.eif_hip_mx4_linear_rows, (w.h, X, 0, 300, None, 0, X, 64, 5, None)),
                 (lib.eif_hip_mx4_linear_grouped, (g.h, X, 256, X, 16, 5, X, X, None, 0, X, 64, 5, None))):
        fake.fake_reset(); fake.fake_fail_launch(0)
        assert f(*a) == DEVICE
    """)


def test_products_allocate_nothing(fake):  # noqa: F811
    """Inside and outside a capture, at every number of rows: launches on the caller's stream, no memory."""
    run(fake, WEIGHT + """
    w, g = mx4(64, 1000), mx4(64, 1000, 7)
    n = fake.fake_mallocs()
    for capturing in (0, 1):
        fake.fake_capturing(capturing)
        for M in (1, 8, 16, 17, 100, 5000):
            fake.fake_reset()
            assert lib.eif_hip_mx4_linear(w.h, X, 512, X, 32, None, 0, X, 64, M, 0x100) == 0
            assert lib.eif_hip_mx4_linear_grouped(g.h, X, 512, X, 32, M, None, X, None, 1, X, 64, M, 0x100) == 0
            assert lib.eif_hip_mx4_quant_rows(X, 1, 1000, M, 1000, X, 512, X, 32, None, 0, 0x100) == 0
            assert M > 8 or lib.eif_hip_mx4_linear_rows(w.h, X, 0, 1000, None, 0, X, 64, M, 0x100) == 0
            assert {fake.fake_launch_stream(i) for i in range(fake.fake_launches())} == {0x100}
    assert fake.fake_mallocs() == n
    """)


GRID = [  # experts, rows, cols, gated, token rows, workgroups, threads: the form that a product takes
    (0, 13824, 2560, 0, 1, 432, 512), (0, 151936, 1024, 0, 16, 1187, 512), (0, 2560, 6912, 0, 24, 160, 512),
    (0, 4864, 896, 0, 48, 456, 512), (0, 2560, 2560, 0, 100, 80, 256), (0, 1024, 1024, 0, 600, 152, 256), (0, 8192, 8192, 0, 128, 256, 256),
    (0, 4096, 4096, 0, 1024, 256, 256), (0, 13824, 2560, 1, 512, 216, 256),
    (0, 4096, 4096, 0, 512, 256, 256), (0, 8192, 8192, 0, 4096, 1024, 256),
    (64, 2816, 2048, 1, 16384, (128 + 63) * 11 + 3, 256), (32, 2816, 2560, 1, 32, (2 + 31) * 11, 512),
    (32, 2816, 2560, 1, 800, (13 + 31) * 22, 256),
    # the shapes of the GPU tests of large products
    (0, 4130, 1024, 0, 3070, 17 * 24, 256), (0, 9920, 1024, 0, 600, 78 * 5 + 2, 256), (0, 2880, 1024, 0, 1101, 23 * 18 + 2, 256),
    (0, 1100, 2304, 0, 300, 9 * 10 + 6, 256), (0, 4096, 1024, 0, 300, 160, 256), (0, 10240, 1024, 0, 600, 200, 256), (7, 2304, 1536, 0, 6000, (47 + 6) * 9 + 3, 256),
    (20, 1280, 1536, 0, 3000, (24 + 19) * 10 + 2, 256), (40, 640, 1536, 0, 3600, (57 + 39) * 5, 256),
    (9, 1100, 2304, 0, 700, (22 + 8) * 9 + 2, 256),
]


@pytest.mark.parametrize("experts,rows,cols,glu,M,blocks,threads", GRID)
def test_forms(fake, experts, rows, cols, glu, M, blocks, threads):  # noqa: F811
    """The form of a product goes by its rows, columns and token rows, and by expert its grid holds every split of the rows."""
    run(fake, WEIGHT + f"""
    experts, rows, cols, glu, M = {experts}, {rows}, {cols}, {glu}, {M}
    h = vp()
    assert lib.eif_hip_mx4_weight_create(C.byref(h), max(experts, 1), rows, cols, X, cols // 2, X, cols // 32, 1, None) == 0
    fake.fake_reset()
    kp = lib.eif_hip_mx4_kpad(cols)
    if experts:
        rc = lib.eif_hip_mx4_linear_grouped(h, X, kp // 2, X, kp // 32, M, None, X, None, glu, X, rows, M, None)
    else:
        rc = lib.eif_hip_mx4_linear(h, X, kp // 2, X, kp // 32, None, glu, X, rows, M, None)
    assert rc == 0 and fake.fake_launches() == 1
    assert (fake.fake_launch_grid(0), fake.fake_launch_block(0)) == ({blocks}, {threads})
    """)
