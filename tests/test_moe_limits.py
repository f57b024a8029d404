"""Routing and adapters without a GPU: tensors that the Python binding has to take, on the stand-in for the HIP runtime."""
from test_host_launches import fake, run  # noqa: F401
from test_moe import TENSORS


def test_one_row_of_any_stride(fake):  # noqa: F811
    """The stride between the rows of a single one means nothing: a column turned around, or an expanded vector, is a row."""
    run(fake, TENSORS + """
    b16 = torch.bfloat16
    for s in (0, 1, 7, 200):
        one = lambda n, dtype=torch.float32: T(1, n, dtype=dtype, stride=(s, 1))
        bh.moe_route(one(64), T(1, 4, dtype=i32), T(1, 4))
        bh.moe_route(one(64, b16), one(4, i32), one(4), bias=T(64))
        bh.moe_combine(one(32), T(1, 1, dtype=i32), one(32), add=one(32))
        bh.moe_combine(T(20, 32), one(4, i32), one(32, b16), one(4))
        h = bh.Adapters(3, 64, 96, 16, b16)
        h.linear(one(96), T(1, dtype=i32), one(64), one(64))
        h.linear(one(96, b16), T(1, dtype=i32), one(64))
        h.set(0, one(96, b16), T(64, 1, dtype=b16, stride=(s + 1, 5)))
        h.close()
    assert refused(bh.moe_route, T(2, 64, stride=(1, 1)), T(2, 4, dtype=i32), T(2, 4)) and refused(bh.moe_combine, T(20, 32), T(2, 4, dtype=i32), T(2, 32, stride=(0, 1)))
    bh.moe_route(T(0, 64), T(0, 4, dtype=i32), T(0, 4)); bh.moe_combine(T(0, 32), T(3, 4, dtype=i32), T(3, 32))
    """)
