"""Microscaled 4-bit operators as measurable cases (include/eif_hip_mx.h).

Three operators, all on MXFP4 (blocks of 32 columns share a power-of-two scale, values are E2M1):

  quant    rows of f32, f16 or bf16 -> MXFP4 codes and scales, and the values they stand for (eif_hip_mx4_quant_rows).
  linear   the product of quantised token rows with a resident MXFP4 matrix, plain or gated (eif_hip_mx4_linear), and its
           form for a few tokens, which takes the rows unquantised (eif_hip_mx4_linear_rows).
  grouped  the product of token rows sorted by expert with a stack of resident matrices (eif_hip_mx4_linear_grouped).

Inputs are made from the seed alone: activations N(0,1) with 1 % outliers 20 times as large, weights N(0,1) / sqrt(K) with
a spread over rows, experts chosen with a bias of their own so that the groups are ragged.
"""
import ctypes as C
import math
import os
import random
import sys

import torch

own = False

_DEV = "cuda:0"
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_TYPE_IDS = {"f32": 0, "f16": 1, "bf16": 2}


def listed():
    return [
        # the activations of one decoded token
        dict(kind="quant", name="quant_token", type="f32", rows=1, cols=2560),
        # the activations of a long prompt in front of a down projection; an odd count of rows
        dict(kind="quant", name="quant_prompt", type="f32", rows=3001, cols=6912),
        # a weight matrix of a bf16 checkpoint on its way into the library
        dict(kind="quant", name="quant_weights", type="bf16", rows=13824, cols=2560),
        # one decoded token: the gated feed-forward input, and the vocabulary head
        dict(kind="rows", name="rows_gate_up_1", type="f32", tokens=1, rows=13824, cols=2560, glu=True, bias=False),
        dict(kind="rows", name="rows_head_1", type="f32", tokens=1, rows=151936, cols=1024, glu=False, bias=False),
        # a few users' tokens at once through a down projection
        dict(kind="linear", name="linear_down_24", tokens=24, rows=2560, cols=6912, glu=False, bias=False),
        # a short prompt on a small model with biases
        dict(kind="linear", name="linear_small_201", tokens=201, rows=1152, cols=896, glu=False, bias=True),
        # a prompt through the gated feed-forward input
        dict(kind="linear", name="linear_gate_up_512", tokens=512, rows=13824, cols=2560, glu=True, bias=False),
        # the largest: many prompts through a wide square matrix
        dict(kind="linear", name="linear_wide_4096", tokens=4096, rows=8192, cols=8192, glu=False, bias=False),
        # eight users' tokens, four experts each of 32: most experts have one row or none
        dict(kind="grouped", name="grouped_decode", tokens=8, top=4, experts=32, rows=2816, cols=2560, glu=True, bias=False,
             gather=True, spare=0),
        # a prompt, eight experts each of 64: the gated input of the experts, rows taken from the token rows
        dict(kind="grouped", name="grouped_gate_up", tokens=2048, top=8, experts=64, rows=2816, cols=2048, glu=True,
             bias=False, gather=True, spare=0),
        # the same experts' down projections on rows already sorted, in a buffer with some rows to spare
        dict(kind="grouped", name="grouped_down", tokens=2048, top=8, experts=64, rows=2048, cols=1408, glu=False,
             bias=True, gather=False, spare=37),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cols(rng, lo, hi):
    """Columns: mostly whole blocks of 32, sometimes an odd count."""
    c = _log_int(rng, lo, hi)
    return c if rng.random() < 0.25 else max(32, 32 * (c // 32))


def draw(rng: random.Random):
    kind = rng.choice(["quant", "rows", "linear", "linear", "grouped", "grouped"])
    if kind == "quant":
        cols = _cols(rng, 33, 14336)
        return dict(kind=kind, type=rng.choice(["f32", "f16", "bf16"]), rows=_log_int(rng, 1, min(16384, 35_000_000 // cols)),
                    cols=cols)
    glu = rng.random() < 0.4
    if kind == "grouped":
        experts, cols = _log_int(rng, 2, 128), _cols(rng, 256, 4096)
        rows = _log_int(rng, 128, min(8192, 64 * 2816 * 2048 // (experts * cols)))
        rows = max(32, 32 * (rows // 32)) if glu else rows
        top = rng.randint(1, min(8, experts))
        tokens = _log_int(rng, 1, max(1, min(4096, 2048 * 8 * 2816 * 2048 // (rows * cols) // top)))
        return dict(kind=kind, tokens=tokens, top=top, experts=experts, rows=rows, cols=cols, glu=glu, bias=rng.random() < 0.3,
                    gather=rng.random() < 0.5, spare=rng.choice([0, 0, 1, 50]))
    cols = _cols(rng, 256, 8192)
    rows = _log_int(rng, 64, 16384)
    if kind == "rows" and rng.random() < 0.3:
        rows, glu, cols = rng.randint(32000, 151936), False, 32 * rng.randint(16, 32)
    rows = max(32, 32 * (rows // 32)) if glu else rows
    c = dict(kind=kind, tokens=rng.randint(1, 8) if kind == "rows" else
             _log_int(rng, 1, min(4096, 4096 * 8192 * 8192 // (rows * cols))), rows=rows, cols=cols, glu=glu,
             bias=rng.random() < 0.3)
    if kind == "rows":
        c["type"] = rng.choice(["f32", "f16", "bf16"])
    return c


# ---- the format, in plain operations ----

# E2M1: value of each code (bit 3 is the sign)
_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def _blocks(x):
    """[R, K] -> float32 [R, ceil(K / 32), 32], the last block filled with zeros."""
    r, k = x.shape
    x = x.float()
    if k % 32:
        x = torch.cat([x, x.new_zeros((r, -k % 32))], 1)
    return x.reshape(r, -1, 32)


def _quantise(x):
    """Magnitude code [R, B, 32], sign, and scale byte [R, B] of rows x."""
    b = _blocks(x)
    amax = b.abs().amax(2)
    exponent = torch.frexp(amax)[1] - 3                  # floor(log2 amax) - 2
    exponent = torch.where(amax > 0, exponent, -127).clamp(min=-127)
    finite = torch.isfinite(amax)
    byte = torch.where(finite, exponent + 127, 255)
    inverse = torch.ldexp(torch.ones_like(amax), torch.where(finite, -exponent, 0))
    a = (b * inverse[:, :, None]).abs()
    # the code is the count of midpoints below |v|; a midpoint itself goes to the even code
    code = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = torch.where(finite[:, :, None], code, 0)
    return code, torch.signbit(b) & finite[:, :, None], byte


def _scale(byte):
    """The power of two that a scale byte stands for."""
    s = torch.ldexp(torch.ones_like(byte, dtype=torch.float32), byte.int() - 127)
    return torch.where(byte == 255, math.nan, s)


def _quantised_values(x):
    code, sign, byte = _quantise(x)
    v = torch.tensor(_E2M1, device=x.device)[code + 8 * sign.int()] * _scale(byte)[:, :, None]
    return v.reshape(x.shape[0], -1)[:, :x.shape[1]].contiguous()


def _packed(x, blocks=0):
    """(codes, scales) of rows x: two codes a byte (even column in the low nibble), padded to `blocks` blocks."""
    code, sign, byte = _quantise(x)
    c = (code + 8 * sign.int()).reshape(x.shape[0], -1).to(torch.uint8)
    c = (c[:, 0::2] | (c[:, 1::2] << 4)).contiguous()
    byte = byte.to(torch.uint8).contiguous()
    more = blocks - byte.shape[1]
    if more > 0:
        c, byte = torch.nn.functional.pad(c, (0, 16 * more)), torch.nn.functional.pad(byte, (0, more))
    return c, byte


def _decoded(codes, scales, cols):
    """Values [..., cols] of packed rows."""
    lut = torch.tensor(_E2M1, device=codes.device)
    v = torch.stack([lut[(codes & 15).int()], lut[(codes >> 4).int()]], -1).flatten(-2)
    v = v.unflatten(-1, (-1, 32))[..., :scales.shape[-1], :] * _scale(scales)[..., None]
    return v.flatten(-2)[..., :cols]


# ---- inputs ----

def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(int(seed) * 6151 + 29)


def _activations(g, m, k):
    x = torch.randn((m, k), generator=g, device=_DEV)
    return torch.where(torch.rand((m, k), generator=g, device=_DEV) < 0.01, 20.0 * x, x)


def _matrix(g, rows, cols):
    spread = torch.exp2(torch.randn((rows, 1), generator=g, device=_DEV))
    return torch.randn((rows, cols), generator=g, device=_DEV) * spread / math.sqrt(cols)


def _blocks_padded(cols):
    """Blocks of an operand row of the products: whole runs of 256 columns."""
    return 8 * -(-cols // 256)


def _inputs(c, seed):
    g = _gen(seed)
    if c["kind"] == "quant":
        return {"x": _activations(g, c["rows"], c["cols"]).to(_TYPES[c["type"]])}
    d = {}
    if c["kind"] == "grouped":
        e, t = c["experts"], c["tokens"]
        parts = [_packed(_matrix(g, c["rows"], c["cols"])) for _ in range(e)]
        d["w"] = torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts])
        score = torch.randn((t, e), generator=g, device=_DEV) + 0.7 * torch.randn((1, e), generator=g, device=_DEV)
        ids = score.topk(c["top"], 1)[1].flatten()
        order = torch.argsort(ids, stable=True)
        counts = torch.bincount(ids, minlength=e)
        d["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).int()
        d["most"] = int(counts.max())
        d["index"] = (order // c["top"]).int() if c["gather"] else None
        n_x = t if c["gather"] else t * c["top"]
        d["a"] = _packed(_activations(g, n_x, c["cols"]), _blocks_padded(c["cols"]))
        d["bias"] = torch.randn((e, c["rows"]), generator=g, device=_DEV) if c["bias"] else None
        return d
    d["w"] = _packed(_matrix(g, c["rows"], c["cols"]))
    x = _activations(g, c["tokens"], c["cols"])
    if c["kind"] == "rows":
        d["x"] = x.to(_TYPES[c["type"]])
    else:
        d["a"] = _packed(x, _blocks_padded(c["cols"]))
    d["bias"] = torch.randn((c["rows"],), generator=g, device=_DEV) if c["bias"] else None
    return d


def _out_rows(c):
    return c["tokens"] * c["top"] + c["spare"] if c["kind"] == "grouped" else c["tokens"]


def prepare(case, seed):
    c = case
    s = dict(_inputs(c, seed), case=c)
    if c["kind"] != "quant":
        s["y"] = torch.zeros((_out_rows(c), c["rows"] // (2 if c["glu"] else 1)), device=_DEV)
    if own:
        s["call"] = _call(c, s)
    torch.cuda.synchronize()
    return s


# ---- the framework's calls ----

def _framework():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bitllm.c_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import bitllm_hip
    return bitllm_hip


def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _call(c, s):
    """The resident weight and the arguments of the call, as a program keeps them from step to step."""
    bh = _framework()
    bh.check(bh.load().eif_hip_init(0), "eif_hip_init")
    lib, kind = bh.load(), c["kind"]
    if kind == "quant":
        r, blocks = c["rows"], _blocks_padded(c["cols"])
        s["codes"] = torch.empty((r, 16 * blocks), dtype=torch.uint8, device=_DEV)
        s["scales"] = torch.empty((r, blocks), dtype=torch.uint8, device=_DEV)
        s["values"] = torch.empty((r, c["cols"]), device=_DEV)
        return lib.eif_hip_mx4_quant_rows, (_p(s["x"]), _TYPE_IDS[c["type"]], c["cols"], r, c["cols"], _p(s["codes"]),
                                            16 * blocks, _p(s["scales"]), blocks, _p(s["values"]), c["cols"])
    experts = c.get("experts", 1)
    w = s["weight"] = bh.Mx4Weight(c["rows"], c["cols"], *s["w"], experts=experts)
    y, glu = s["y"], 1 if c["glu"] else 0
    if kind == "rows":
        return lib.eif_hip_mx4_linear_rows, (w.h, _p(s["x"]), _TYPE_IDS[c["type"]], c["cols"], _p(s["bias"]), glu, _p(y),
                                             y.stride(0), c["tokens"])
    a, b = s["a"]
    if kind == "linear":
        return lib.eif_hip_mx4_linear, (w.h, _p(a), a.stride(0), _p(b), b.stride(0), _p(s["bias"]), glu, _p(y), y.stride(0),
                                        c["tokens"])
    return lib.eif_hip_mx4_linear_grouped, (w.h, _p(a), a.stride(0), _p(b), b.stride(0), a.shape[0], _p(s["index"]),
                                            _p(s["offsets"]), _p(s["bias"]), glu, _p(y), y.stride(0), y.shape[0])


def _run_own(s):
    f, args = s["call"]
    rc = f(*args, torch.cuda.current_stream().cuda_stream)
    if rc:
        raise RuntimeError("%s: %d" % (f.__name__, rc))
    return s["values"] if s["case"]["kind"] == "quant" else s["y"]


# ---- the plain forms ----

def _gated(y):
    g, u = y.chunk(2, -1)
    return g / (1.0 + torch.exp(-g)) * u


def _plain(s):
    c = s["case"]
    if c["kind"] == "quant":
        return _quantised_values(s["x"])
    w = _decoded(*s["w"], c["cols"])
    if c["kind"] != "grouped":
        a = _quantised_values(s["x"]) if c["kind"] == "rows" else _decoded(*s["a"], c["cols"])
        y = torch.matmul(a, w.t())
        y = y if s["bias"] is None else y + s["bias"]
        return _gated(y) if c["glu"] else y
    # every group's rows in a panel of the largest group's size, one batched product
    n = c["tokens"] * c["top"]
    at = torch.arange(n, device=_DEV, dtype=torch.int32)
    e = torch.searchsorted(s["offsets"], at, right=True) - 1
    place = at - s["offsets"][e]
    a = _decoded(*s["a"], c["cols"])
    panel = torch.zeros((c["experts"], s["most"], c["cols"]), device=_DEV)
    panel[e, place] = a if s["index"] is None else a[s["index"]]
    y = torch.matmul(w, panel.transpose(1, 2).contiguous()).transpose(1, 2)[e, place]
    y = y if s["bias"] is None else y + s["bias"][e]
    out = s["y"]
    out[:n] = _gated(y) if c["glu"] else y
    return out


def run(state):
    return _run_own(state) if own else _plain(state)


# ---- what a pass cannot do without ----

def _packed_bytes(rows, cols):
    return rows * (-(-cols // 2) + -(-cols // 32))


def work(case):
    c = case
    size = {"f32": 4, "f16": 2, "bf16": 2}
    r, k = c["rows"], c["cols"]
    if c["kind"] == "quant":
        return {"bytes": r * k * size[c["type"]] + _packed_bytes(r, k) + 4 * r * k, "flops": 4 * r * k}
    outs = r // 2 if c["glu"] else r
    if c["kind"] == "grouped":
        n = c["tokens"] * c["top"]
        busy = c["experts"] * (1.0 - (1.0 - c["top"] / c["experts"]) ** c["tokens"])   # experts with rows, for even odds
        return {"bytes": busy * _packed_bytes(r, k) + _packed_bytes(c["tokens"] if c["gather"] else n, k) + 4 * n * outs,
                "flops": 2 * n * r * k}
    m = c["tokens"]
    a = m * k * size[c["type"]] if c["kind"] == "rows" else _packed_bytes(m, k)
    return {"bytes": _packed_bytes(r, k) + a + 4 * m * outs, "flops": 2 * m * r * k}


# ---- the same from the definition, in 64 bits ----

def _exact_decoded(codes, scales, cols):
    """Sign, exponent and mantissa bits of every code, in 64 bits."""
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(torch.int16)
    n = torch.nn.functional.pad(n, (0, max(0, 32 * scales.shape[-1] - n.shape[-1])))[..., :32 * scales.shape[-1]]
    exponent, mantissa = (n >> 1) & 3, (n & 1).double()
    v = torch.where(exponent == 0, 0.5 * mantissa, torch.exp2(exponent.double() - 1) * (1 + 0.5 * mantissa))
    v = torch.where(n >= 8, -v, v)
    s = torch.exp2(scales.double() - 127).masked_fill(scales == 255, math.nan)
    return (v * s.repeat_interleave(32, -1))[..., :cols]


def _exact_rows(x):
    """Every value to the nearest of its block's grid, found by distance; of two as near, the one with even mantissa."""
    k = x.shape[1]
    b = torch.nn.functional.pad(x.double(), (0, -k % 32)).unflatten(1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(amax))
    e = torch.where(torch.exp2(e) > amax, e - 1, torch.where(torch.exp2(e + 1) <= amax, e + 1, e))
    step = torch.exp2((e - 2).clamp(min=-127))
    a = b.abs() / step
    # spacing of the grid at |a|: 0.5 below 2, 1 below 4, 2 above
    unit = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / unit) * unit).clamp(max=6.0)
    v = torch.where(amax > 0, torch.copysign(a, b) * step, 0.0)
    v = torch.where(torch.isfinite(amax), v, math.nan)
    return v.flatten(1)[:, :k]


def _exact_product(a, w, bias, glu):
    y = a @ w.T
    if bias is not None:
        y = y + bias.double()
    if not glu:
        return y
    g, u = y[:, :y.shape[1] // 2], y[:, y.shape[1] // 2:]
    return g * torch.sigmoid(g) * u


def exact(case, seed):
    c, d = case, _inputs(case, seed)
    if c["kind"] == "quant":
        return _exact_rows(d["x"])
    if c["kind"] != "grouped":
        a = _exact_rows(d["x"]) if c["kind"] == "rows" else _exact_decoded(*d["a"], c["cols"])
        return _exact_product(a, _exact_decoded(*d["w"], c["cols"]), d["bias"], c["glu"])
    a = _exact_decoded(*d["a"], c["cols"])
    y = torch.zeros((_out_rows(c), c["rows"] // (2 if c["glu"] else 1)), dtype=torch.float64, device=_DEV)
    edges = d["offsets"].tolist()
    for e in range(c["experts"]):
        lo, hi = edges[e], edges[e + 1]
        if hi > lo:
            rows = a[lo:hi] if d["index"] is None else a[d["index"][lo:hi].long()]
            w = _exact_decoded(d["w"][0][e], d["w"][1][e], c["cols"])
            y[lo:hi] = _exact_product(rows, w, None if d["bias"] is None else d["bias"][e], c["glu"])
    return y
