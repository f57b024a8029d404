"""Low-rank adapters on the GPU (include/eif_hip_adapters.h) whose matrices hold infinities, and rows of the least values, in each form."""
import numpy as np
import pytest

import moe_ref
from test_gpu_adapters import Case
from test_gpu_moe import TYPES, dev, host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [9, 256, 257, 513, 4100])
@pytest.mark.parametrize("types", [("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("rank", [16, 48])
def test_infinite_elements(gpu, types, rank, m):
    """What an infinity of A or B reaches is infinite or NaN in every form, the infinity's column of x being zero or not, and x of few bits
    or of many; the other outputs and rows are as without it."""
    import torch
    rows, cols = 72, 136
    rng = np.random.default_rng(m + rank)
    c = Case(gpu, 6, 6, rows, cols, rank, types[1], ranks=[rank] * 5)
    dt = getattr(torch, TYPES[types[1]])
    x = np.where(rng.random((m, cols)) < 0.5, rng.integers(-4, 5, (m, cols)) / 2, rng.standard_normal((m, cols))).astype(np.float32)
    slot = (np.arange(m) % 6).astype(np.int32)   # the last is empty
    base = rng.standard_normal((m, rows)).astype(np.float32)
    x = host(dev(x, types[0]))

    def put(s, a_at=None, b_at=None):
        a, b, scale = (v.copy() if i < 2 else v for i, v in enumerate(c.pairs[s]))
        if a_at:
            a[a_at] = np.inf
        if b_at:
            b[b_at] = -np.inf
        c.h.set(s, torch.from_numpy(a).to(dt).cuda(), torch.from_numpy(b).to(dt).cuda(), scale)

    put(1, a_at=(rank - 1, 5))
    put(2, b_at=(9, rank - 1))
    put(3, a_at=(0, cols - 1), b_at=(rows - 1, 0))
    y = torch.full((m, rows), 7.0, device="cuda")
    c.h.linear(dev(x, types[0]), dev(slot), y, dev(base))
    torch.cuda.synchronize()
    got = host(y)
    reached = np.zeros((m, rows), bool)
    reached[(slot == 1) | (slot == 3)] = True    # all outputs of the row come from every rank
    reached[slot == 2, 9] = True
    assert not np.isfinite(got[reached]).any()
    want, tol = moe_ref.adapters(x, slot, c.pairs, base, rows)
    assert (np.abs(got - want)[~reached] <= tol[~reached]).all()


@pytest.mark.parametrize("m", [9, 600, 4100])
@pytest.mark.parametrize("types", [("f32", "bf16"), ("f32", "f16"), ("f32", "f32"), ("bf16", "bf16")])
def test_least_values(gpu, types, m):
    """Values down to the least of FP32 come through matrices of ones on the diagonal: x and A x are off by 2^-133 each at most, which is
    what bf16 parts leave out."""
    import torch
    rng = np.random.default_rng(m)
    dt = getattr(torch, TYPES[types[1]])
    h = gpu.Adapters(1, 48, 40, 16, dt)
    h.set(0, torch.eye(16, 40).to(dt).cuda(), torch.eye(48, 16).to(dt).cuda(), 1.0)
    x = (rng.standard_normal((m, 40)) * 2.0 ** rng.integers(-149, -100, (m, 1))).astype(np.float32)
    y, xd = torch.full((m, 48), 7.0, device="cuda"), dev(x, types[0])
    h.linear(xd, dev(np.zeros(m, np.int32)), y)
    torch.cuda.synchronize()
    got, x = host(y).astype(np.float64), host(xd).astype(np.float64)
    assert (np.abs(got[:, :16] - x[:, :16]) <= 2 * 2.0 ** -133 + 2.0 ** -22 * np.abs(x[:, :16])).all() and not got[:, 16:].any()
