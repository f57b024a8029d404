"""Routing to experts on the GPU (include/eif_hip_moe.h) at the ends of what scores and biases hold, against the definition in 64
bits: sums of biases that 32 bits do not hold, sums over all experts, scores next to the least numbers; and in the forms of many tokens."""
import numpy as np
import pytest

import moe_ref
from test_gpu_moe import dev, host, ints, logits_of

pytestmark = pytest.mark.gpu

LOWEST, MOST = np.finfo(np.float32).min, np.finfo(np.float32).max


def check(gpu, rows, tokens, top, type="f32", sorted_too=False, **spec):
    """Logits `rows`, repeated to so many tokens. A weight is computed in 64 bits and rounded once: off by 2^-24 of it, or 2^-150, and by
    some 1e-14 of it before."""
    import torch
    few = dev(rows, type)
    at = np.arange(tokens) % rows.shape[0]
    x = few[torch.from_numpy(at).cuda()].contiguous()
    ids, w = ints(tokens * top).view(tokens, top), torch.full((tokens, top), float("nan"), device="cuda")
    places = {}
    if sorted_too:
        need = gpu.moe_sort_bytes(tokens, top, rows.shape[1])
        places = dict(offsets=ints(rows.shape[1] + 1), row=ints(tokens * top), slot=ints(tokens * top),
                      work=torch.full((need,), 0x5A, dtype=torch.uint8, device="cuda") if need else None)
    b = spec.get("bias")
    gpu.moe_route(x, ids, w, **{**spec, "bias": None if b is None else dev(b)}, **places)
    torch.cuda.synchronize()
    want_ids, want = moe_ref.route(host(few), top, **spec)
    want_ids, want = want_ids[at], want[at]
    got = host(ids)
    bad = np.nonzero((got != want_ids).any(1))[0]
    assert not bad.size, (spec, bad[:5], got[bad[:3]].tolist(), want_ids[bad[:3]].tolist())
    gw = host(w).astype(np.float64)
    off = np.abs(gw - want) / (1.01 * 2.0 ** -24 * np.abs(want) + 2.0 ** -149)
    assert (off <= 1.0).all(), (spec, np.max(off))
    if sorted_too:
        for p, v, name in zip((places["offsets"], places["row"], places["slot"]), moe_ref.sort(want_ids, rows.shape[1]), ("offsets", "row", "slot")):
            assert np.array_equal(host(p), v), name


@pytest.mark.parametrize("tokens,experts,groups", [(3, 16, 4), (5, 64, 32), (7, 64, 64), (7, 256, 8), (7, 256, 64), (2100, 256, 8), (2100, 256, 64),
                                                   (4100, 96, 48), (5, 1000, 10), (3, 1100, 11)])
def test_groups_of_lowest_biases(gpu, tokens, experts, groups):
    """Two biases whose sum 32 bits do not hold: a group of them is worth more than one that is shut out, and as much as 64 bits say."""
    rng = np.random.default_rng(experts + groups)
    rows = (1.5 * rng.standard_normal((7, experts))).astype(np.float32)
    size = experts // groups
    rows[0, :size] = -np.inf
    rows[1, rng.random(experts) < 0.5] = -np.inf
    rows[2, size:] = -np.inf
    group = np.arange(experts) // size
    worths = np.array([LOWEST, LOWEST / 2, MOST, MOST * 0.75, -np.inf, np.nan, np.inf, 0.1], np.float32)
    biases = [np.full(experts, LOWEST, np.float32), np.where(group == groups - 1, 0.25, LOWEST).astype(np.float32),
              np.where(group % 2, -np.inf, LOWEST).astype(np.float32), np.where(group % 2, MOST, np.inf).astype(np.float32)]
    biases += [worths[rng.integers(8, size=groups)][group] for _ in range(6)]
    biases += [worths[rng.integers(8, size=experts)] for _ in range(2)]
    biases += [np.where(rng.random(experts) < 0.7, LOWEST, (0.2 * rng.standard_normal(experts)).astype(np.float32))]
    for b in biases:
        for kept in sorted({1, 2, groups // 2, groups - 1}):
            for best in (1, 2):
                for score in (moe_ref.SIGMOID, moe_ref.SOFTMAX):
                    check(gpu, rows, tokens, min(8, experts), score=score, bias=b, groups=groups, groups_kept=kept, group_best=best)


@pytest.mark.parametrize("tokens,experts,groups", [(9, 7, 1), (70, 64, 1), (2051, 64, 8), (9, 200, 1), (2051, 96, 1), (4101, 256, 8), (9, 300, 1),
                                                   (4101, 512, 1), (9, 1000, 8), (9, 1025, 5)])
@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_weights_of_all_experts(gpu, tokens, experts, groups, type):
    """A softmax over all experts is summed in 64 bits, by whichever form, and a weight rounded once."""
    rng = np.random.default_rng(experts)
    rows = rng.standard_normal((13, experts)).astype(np.float32)
    rows[:4] = 1.0 + rows[:4] / 256            # near each other: each a small share of the sum
    rows[4:7] = 40.0 + 0.25 * rows[4:7]
    rows[7] *= 30.0
    rows[8, rng.random(experts) < 0.5] = -np.inf
    rows[9] = -np.inf
    rows[10, rng.integers(experts)] = np.inf
    rows[11] *= np.float32(1e37)
    for scale in (1.0, 2.5):
        check(gpu, rows, tokens, min(7, experts), type, score=moe_ref.SOFTMAX, groups=groups, groups_kept=max(1, groups // 2), renormalise=False,
              scale=scale)


@pytest.mark.parametrize("tokens,experts,groups", [(6, 16, 4), (6, 64, 1), (6, 256, 8), (2100, 256, 8), (2100, 128, 1), (6, 1000, 10), (3, 1100, 11)])
def test_least_scores(gpu, tokens, experts, groups):
    """Scores next to the least numbers of 64 bits, and of them: 1 / (1 + e^-l) down to where e^-l leaves 64 bits."""
    rng = np.random.default_rng(experts)
    rows = np.empty((6, experts), np.float32)
    rows[0] = rng.uniform(-712.0, -690.0, experts)
    rows[1] = rng.uniform(-709.79, -709.69, experts)
    rows[2] = rng.uniform(-709.0, -708.0, experts)
    rows[3] = rng.uniform(-746.0, -709.6, experts)
    rows[4] = -709.75
    rows[5] = np.where(np.arange(experts) % 3 == 1, -700.0, np.where(np.arange(experts) % 3, -709.8, -699.9))
    for b in (None, np.zeros(experts, np.float32), np.where(np.arange(experts) % 2, 0.0, -np.inf).astype(np.float32)):
        for best in (1, 2):
            for renormalise in (True, False):
                check(gpu, rows, tokens, min(8, experts), score=moe_ref.SIGMOID, bias=b, groups=groups, groups_kept=max(1, groups // 2),
                      group_best=best, renormalise=renormalise)


@pytest.mark.parametrize("tokens,experts,top,groups,kept", [
    (4999, 256, 8, 8, 4), (4999, 256, 16, 1, 1), (2300, 256, 14, 16, 9), (5001, 100, 5, 5, 3), (4097, 130, 9, 13, 6), (4113, 24, 4, 8, 3),
    (4097, 60, 6, 60, 20), (4500, 300, 8, 10, 4), (4200, 1000, 12, 20, 7), (4103, 512, 64, 1, 1), (5003, 1024, 17, 64, 30), (4099, 1030, 6, 10, 5),
])
def test_long_prompts(gpu, tokens, experts, top, groups, kept):
    """Many tokens, of workgroups with four waves, the last of them partly filled: biases that shut experts out, padding, infinities,
    equals and near groups, of every type."""
    rng = np.random.default_rng(tokens)
    n = 61
    bias = (0.2 * rng.standard_normal(experts)).astype(np.float32)
    shut = bias.copy()
    shut[rng.random(experts) < 0.2] = -np.inf
    shut[rng.random(experts) < 0.1] = np.nan
    shut[rng.integers(experts)] = np.inf
    for i, (score, b) in enumerate(((s, b) for s in (moe_ref.SOFTMAX, moe_ref.SIGMOID) for b in (None, bias, shut))):
        for j, (kind, type) in enumerate((("plain", "bf16"), ("ties", "f16"), ("edges", "f32"))):
            rows = logits_of(rng, n, experts, kind)
            check(gpu, rows, tokens, top, type, sorted_too=(i + j) % 2 == 0, score=score, bias=b, groups=groups, groups_kept=kept,
                  group_best=1 + (i + j + i // 3) % 2 if groups < experts else 1, renormalise=(i + j) % 3 != 0, scale=(1.0, 2.5)[j % 2])
    near = np.concatenate([20.0 + np.arange(experts)[None] * 2.0 ** -10 * s for s in (1.0, -1.0)] + [logits_of(rng, 3, experts, "plain")])
    large = (rng.integers(-3, 4, experts) * 2.0 ** 20).astype(np.float32)
    for b in (None, np.zeros(experts, np.float32), np.full(experts, 100.0, np.float32), large):
        check(gpu, near.astype(np.float32), tokens, top, score=moe_ref.SIGMOID, bias=b, groups=groups, groups_kept=kept, group_best=2)
