"""The microscaled 4-bit calls at the ends of what they take, without a GPU, on the stand-in for the HIP runtime
(fakehip/fakehip.cpp)."""
from test_host_launches import fake, run  # noqa: F401
from test_mx4 import WEIGHT

LAUNCHED = WEIGHT + """
    most = (1 << 24) - 1   # workgroups of 256 threads: a launch holds fewer than 2^32
    def launched():
        return [fake.fake_launch_grid(i) for i in range(min(fake.fake_launches(), 64))]
    def create(rows, cols, experts=1):
        h = vp()
        fake.fake_reset()
        rc = lib.eif_hip_mx4_weight_create(C.byref(h), experts, rows, cols, X, (cols + 1) // 2, X, (cols + 31) // 32, 1, None)
        return rc, h
"""


def test_quant_rows_of_several_launches(fake):  # noqa: F811
    """Rows beyond what a launch holds go out in further launches, up to the stated number of runs."""
    run(fake, LAUNCHED + """
    def q(rows, cols):
        fake.fake_reset()
        ld = -(-cols // 256) * 256
        rc = lib.eif_hip_mx4_quant_rows(X, 2, ld, rows, cols, X, ld // 2, X, ld // 32, X, ld, None)
        return rc, launched()
    assert q(4 * most, 64) == (0, [most]) and q(4 * most + 1, 64) == (0, [most, 1])
    assert q(70_000_000, 64) == (0, [most, 70_000_000 // 4 - most])
    per = 4 * most // 5    # whole rows of five runs
    assert q(2 * per + 3, 1100) == (0, [-(-5 * per // 4)] * 2 + [4])
    assert q((1 << 31) - 1, 900)[0] == 0 and fake.fake_launches() == 129
    assert q((1 << 17) - 1, 1 << 24)[0] == 0 and q(1 << 17, 1 << 24) == (LIMIT, []) and q((1 << 31) - 1, 1025) == (LIMIT, [])
    fake.fake_reset(); fake.fake_fail_launch(1)
    assert lib.eif_hip_mx4_quant_rows(X, 2, 256, 8 * most, 64, X, 128, X, 8, X, 256, None) == DEVICE and fake.fake_launches() == 2
    """)


def test_weights_of_several_launches(fake):  # noqa: F811
    """A weight is laid out by as many launches as it takes: 2^32 - 256 pieces of 16 bytes each."""
    run(fake, LAUNCHED + """
    # a row tile of one span: 128 pieces, 64 dwords of scales
    for rows, grids in ((1 << 16, [1 << 11, 1 << 10]), ((1 << 29) - 32, [most, 1 << 23]), ((1 << 29) - 16, [most, 1, 1 << 23]),
                        (1 << 30, [most, most, 2, most, 1])):
        rc, h = create(rows, 32)
        assert rc == 0 and launched() == grids, (rows, launched())
        lib.eif_hip_mx4_weight_destroy(h)
    assert fake.fake_live() == 0
    """)


def test_products_that_no_launch_holds(fake):  # noqa: F811
    run(fake, LAUNCHED + """
    def linear(h, M, ldc=128, ldy=1 << 30, glu=0):
        fake.fake_reset()
        rc = lib.eif_hip_mx4_linear(h, X, ldc, X, 8, None, glu, X, ldy, M, None)
        assert len(launched()) == (1 if rc == 0 else 0)
        return rc
    # the tiled forms: 32 token rows a workgroup (rows that span 2^32 bytes), whose number is rounded up to whole XCDs
    rc, h = create(64, 32)
    assert rc == 0 and linear(h, 32 * (most - 7)) == 0 and launched() == [most - 7] and linear(h, 32 * (most - 7) + 1) == LIMIT
    lib.eif_hip_mx4_weight_destroy(h)
    # the split form: 128 rows a workgroup of 512
    rc, h = create((1 << 30) - 128, 32)
    assert rc == 0 and linear(h, 1) == 0 and launched() == [(1 << 23) - 1]
    assert lib.eif_hip_mx4_linear_rows(h, X, 0, 32, None, 0, X, 1 << 30, 1, None) == 0
    lib.eif_hip_mx4_weight_destroy(h)
    rc, h = create((1 << 30) - 127, 32)
    fake.fake_reset()
    assert rc == 0 and linear(h, 1) == LIMIT
    assert lib.eif_hip_mx4_linear_rows(h, X, 0, 32, None, 0, X, 1 << 30, 1, None) == LIMIT and not launched()
    lib.eif_hip_mx4_weight_destroy(h)
    # by expert, a grid for every split of the rows: 4096 + 4095 groups of 16
    for rows, grid in ((131072, [8191 * 1024]), (131073, [])):
        rc, h = create(rows, 32, 4096)
        fake.fake_reset()
        want = 0 if grid else LIMIT
        assert rc == 0 and lib.eif_hip_mx4_linear_grouped(h, X, 128, X, 8, 1, X, X, None, 0, X, 1 << 18, 65536, None) == want
        assert launched() == grid
        lib.eif_hip_mx4_weight_destroy(h)
    """)


def test_strides_do_not_change_the_order_of_sums(fake):  # noqa: F811
    """Few rows that span 2^32 bytes take the form of adjacent ones, whose waves' partial sums meet in the same order."""
    run(fake, LAUNCHED + """
    for rows, cols, M in ((2560, 6912, 24), (4864, 896, 48), (64, 300, 300)):
        rc, h = create(rows, cols)
        kp, forms = lib.eif_hip_mx4_kpad(cols), []
        for ldc in (kp // 2, 1 << 30):
            fake.fake_reset()
            assert rc == 0 and lib.eif_hip_mx4_linear(h, X, ldc, X, kp // 32, None, 0, X, rows, M, None) == 0
            forms.append((launched(), fake.fake_launch_block(0)))
        assert forms[0] == forms[1] and forms[0][1] == 512, (rows, cols, M, forms)
        lib.eif_hip_mx4_weight_destroy(h)
    """)


def test_misaligned_floats(fake):  # noqa: F811
    run(fake, LAUNCHED + """
    rc, h = create(64, 256)
    def calls(bias, y, M=5):
        fake.fake_reset()
        return [lib.eif_hip_mx4_linear(h, X, 128, X, 8, bias, 0, y, 64, M, None),
                lib.eif_hip_mx4_linear_rows(h, X, 0, 256, bias, 0, y, 64, M, None),
                lib.eif_hip_mx4_linear_grouped(h, X, 128, X, 8, 5, X, X, bias, 0, y, 64, M, None)]
    assert rc == 0 and calls(at(4), at(4)) == [0] * 3 and calls(None, at(12)) == [0] * 3
    for n in (1, 2, 3):
        assert calls(X, at(n)) == [ARG] * 3 and calls(at(n), X) == [ARG] * 3 and calls(at(n), X, 0) == [ARG] * 3
        assert not launched()
    assert lib.eif_hip_mx4_quant_rows(X, 0, 256, 2, 256, None, 0, None, 0, at(2), 256, None) == ARG
    lib.eif_hip_mx4_weight_destroy(h)
    """)


def test_info_of_no_weight(fake):  # noqa: F811
    run(fake, LAUNCHED + """
    assert lib.eif_hip_mx4_weight_info(None, None, None, None, None, None) == ARG
    rc, h = create(64, 256)
    assert rc == 0 and lib.eif_hip_mx4_weight_info(h, None, None, None, None, None) == 0
    lib.eif_hip_mx4_weight_destroy(h)
    """)


def test_weight_sources_without_end(fake):  # noqa: F811
    """Strides whose product with the rows passes 64 bits are refused before anything is allocated or copied."""
    run(fake, LAUNCHED + """
    h, n = vp(), fake.fake_mallocs()
    src = np.zeros(1 << 16, np.uint8)
    src = vp(src.ctypes.data)
    for dev in (0, 1):
        for experts, rows, ldc, lds in ((1, 5, 1 << 62, 2), (1, 5, 32, 1 << 62), (4096, 1 << 12, 1 << 40, 2), (1, 2, (1 << 63) - 1, 2)):
            fake.fake_reset()
            assert lib.eif_hip_mx4_weight_create(C.byref(h), experts, rows, 64, src, ldc, src, lds, dev, None) == LIMIT, (ldc, lds)
            assert not launched() and not h.value and fake.fake_mallocs() == n
    """)


TENSORS = LAUNCHED + """
    import torch

    class T:
        \"\"\"A device tensor as far as the binding looks at one.\"\"\"
        def __init__(self, *shape, dtype=torch.float32, strides=None, cuda=True):
            self.shape, self.dtype, self.is_cuda = torch.Size(shape), dtype, cuda
            self.strides_ = strides or [int(np.prod(shape[i + 1:])) for i in range(len(shape))]
        def stride(self, i):
            return self.strides_[i]
        def data_ptr(self):
            return X.value

    class S:
        cuda_stream = 0

    u8, i32, i64, f16, f64 = torch.uint8, torch.int32, torch.int64, torch.float16, torch.float64

    def refused(f, *args, **kw):
        fake.fake_reset()
        try:
            f(*args, stream=S, **kw)
        except bh.HipError as e:
            return not launched() and "(-" not in str(e)   # by the binding, not by the library
        return False

    def taken(f, *args, **kw):
        fake.fake_reset()
        f(*args, stream=S, **kw)
        return len(launched()) == 1
"""


def test_binding_quant_rows(fake):  # noqa: F811
    run(fake, TENSORS + """
    q, x, c, s, v = bh.mx4_quant_rows, T(5, 300), T(5, 256, dtype=u8), T(5, 16, dtype=u8), T(5, 300)
    assert taken(q, x, c, s, v) and taken(q, x, c, s) and taken(q, x, values=v) and taken(q, T(5, 300, dtype=f16), T(7, 272, dtype=u8), s)
    for args in ((T(5, 300, cuda=False), c, s), (torch.zeros(5, 300), c, s), (T(5, 300, dtype=f64), c, s), (T(5, 300, strides=[1, 5]), c, s),
                 (T(300), c, s), (x, T(4, 256, dtype=u8), s), (x, T(5, 240, dtype=u8), s), (x, T(5, 256, dtype=i32), s),
                 (x, c, T(4, 16, dtype=u8)), (x, c, T(5, 8, dtype=u8)), (x, c, T(5, 16)), (x, c, s, T(4, 300)), (x, c, s, T(5, 299)),
                 (x, c, s, T(5, 300, dtype=f16)), (x, c, s, T(5, 300, cuda=False)), (x, c, s, T(5, 300, strides=[900, 3]))):
        assert refused(q, *args), [(t.shape, t.dtype) for t in args]
    """)


def test_binding_weight(fake):  # noqa: F811
    run(fake, TENSORS + """
    def W(c, s, experts=1, stream=None):
        return bh.Mx4Weight(64, 300, c, s, experts=experts, stream=S)
    for c, s, e in ((T(64, 150, dtype=u8), T(64, 10, dtype=u8), 1), (T(2, 64, 160, dtype=u8), T(2, 64, 10, dtype=u8), 2),
                    (np.zeros((64, 150), np.uint8), np.zeros((64, 10), np.uint8), 1)):
        W(c, s, e).close()
    c, s = T(64, 150, dtype=u8), T(64, 10, dtype=u8)
    for args in ((T(64, 150, dtype=u8, cuda=False), s), (c, T(64, 10, dtype=u8, cuda=False)), (torch.zeros(64, 150, dtype=u8), torch.zeros(64, 10, dtype=u8)),
                 (T(64, 150, dtype=i32), s), (c, T(64, 10)), (T(64, 149, dtype=u8, strides=[160, 1]), s), (c, T(64, 9, dtype=u8, strides=[16, 1])),
                 (T(63, 150, dtype=u8), s), (c, np.zeros((64, 10), np.uint8)), (np.zeros((64, 150), np.int8), np.zeros((64, 10), np.uint8))):
        assert refused(W, *args), args
    """)


def test_binding_products(fake):  # noqa: F811
    """Tensors that a product would read or write beyond their ends, or take for another type, never reach it."""
    run(fake, TENSORS + """
    w, g = mx4(64, 300), mx4(64, 300, 3)
    c, s, y, h = T(5, 256, dtype=u8), T(5, 16, dtype=u8), T(5, 64), T(5, 32)
    off, idx, b, bg = T(4, dtype=i32), T(5, dtype=i32), T(64), T(3, 64)
    lin, rows, grp = w.linear, w.linear_rows, lambda c, s, y, **k: g.linear_grouped(c, s, k.pop("off", off), y, **k)
    for f in (lin, grp):
        ok = b if f is lin else bg
        assert taken(f, c, s, y) and taken(f, c, s, y, bias=ok) and taken(f, c, s, h, glu=True) and taken(f, T(9, 272, dtype=u8), T(9, 24, dtype=u8), y)
        bad = [(T(5, 240, dtype=u8), s, y), (c, T(5, 8, dtype=u8), y), (c, T(4, 16, dtype=u8), y), (T(5, 256, dtype=i32), s, y), (c, T(5, 16), y),
               (T(5, 256, dtype=u8, cuda=False), s, y), (c, s, T(5, 63)), (c, s, T(5, 64, dtype=f16)), (c, s, T(5, 64, cuda=False)),
               (c, s, T(5, 64, strides=[1, 5])), (c, s, T(64))]
        for args in bad + ([(T(4, 256, dtype=u8), s, y)] if f is lin else []):
            assert refused(f, *args), [(t.shape, t.dtype) for t in args]
        assert refused(f, c, s, T(5, 31), glu=True)
    for bias in (T(63), T(64, dtype=f16), T(64, cuda=False), T(64, strides=[2])):
        assert refused(lin, c, s, y, bias=bias) and refused(rows, T(5, 300), y, bias=bias)
    for bias in (b, T(2, 64), T(3, 63), T(3, 64, strides=[80, 1]), T(191), T(3, 64, dtype=f16)):
        assert refused(grp, c, s, y, bias=bias)
    assert taken(grp, c, s, y, bias=T(192)) and taken(grp, c, s, y, row_index=idx) and taken(grp, T(2, 256, dtype=u8), T(2, 16, dtype=u8), y)
    for o in (T(4, dtype=i64), T(3, dtype=i32), T(4, dtype=i32, strides=[2]), T(4, dtype=i32, cuda=False)):
        assert refused(grp, c, s, y, off=o)
    for i in (T(5, dtype=i64), T(4, dtype=i32), T(5, dtype=i32, strides=[2]), T(5, dtype=i32, cuda=False)):
        assert refused(grp, c, s, y, row_index=i)
    assert taken(rows, T(5, 300), y) and taken(rows, T(3, 304, dtype=f16), y) and taken(rows, T(5, 300), h, glu=True)
    for args in ((T(6, 300), y), (T(5, 299), y), (T(5, 300, dtype=f64), y), (T(5, 300, cuda=False), y), (T(5, 300, strides=[1, 5]), y), (T(5, 300), T(5, 63))):
        assert refused(rows, *args), [(t.shape, t.dtype) for t in args]
    """)
