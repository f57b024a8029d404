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
