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
