"""What a served layer puts around the resident products, as measurable cases (include/eif_hip_moe.h, include/eif_hip_adapters.h).

Four operators:

  route     logits of a router -> the chosen experts and their weights, and the rows sorted by expert as the products by expert take
            them (eif_hip_moe_route): softmax or sigmoid scores, a bias for balance, groups of experts, renormalised weights.
  sort      chosen experts -> offsets, rows and places (eif_hip_moe_sort).
  combine   the experts' output rows -> a weighted sum per token, added to the residual (eif_hip_moe_combine).
  adapters  low-rank adapters of many requests beside a shared projection (eif_hip_adapters_linear).

Inputs are made from the seed alone. Experts have a popularity of their own, so that their groups are ragged; some tokens are padding,
whose logits are all -inf. Choices between experts are made in 64 bits: near ones differ where 32 bits round.
"""
import ctypes as C
import math
import os
import random
import sys

import numpy as np
import torch

own = False

_DEV = "cuda:0"
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_TYPE_IDS = {"f32": 0, "f16": 1, "bf16": 2}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_MOST = 3.4028234663852886e38   # what an infinite logit counts as


def listed():
    return [
        # one decoded token, 4 of 32 experts
        dict(kind="route", name="route_token", type="f32", tokens=1, experts=32, top=4, score="softmax", bias=False, groups=1, kept=1,
             best=1, renormalise=True, scale=1.0, padded=0),
        # a decode batch of 64 users: balance bias, the best 4 of 8 groups
        dict(kind="route", name="route_users", type="f32", tokens=64, experts=256, top=8, score="sigmoid", bias=True, groups=8, kept=4,
             best=2, renormalise=True, scale=2.5, padded=0),
        # a prompt whose router ran in bf16: equal logits are frequent
        dict(kind="route", name="route_prompt", type="bf16", tokens=2048, experts=64, top=8, score="softmax", bias=False, groups=1,
             kept=1, best=1, renormalise=False, scale=1.0, padded=5),
        # many prompts at once, an odd count
        dict(kind="route", name="route_long", type="f32", tokens=16001, experts=256, top=8, score="sigmoid", bias=True, groups=8, kept=4,
             best=2, renormalise=True, scale=2.5, padded=37),
        # a few users' choices made elsewhere
        dict(kind="sort", name="sort_users", tokens=33, experts=8, top=2, dropped=0.0),
        # many prompts' choices, some dropped for lack of room
        dict(kind="sort", name="sort_long", tokens=32768, experts=128, top=8, dropped=0.02),
        # eight users' tokens, the experts of the products above
        dict(kind="combine", name="combine_users", type="f32", tokens=8, top=4, dim=2560, add=True, dropped=0.0),
        # a prompt, into the next layer's bf16 rows
        dict(kind="combine", name="combine_prompt", type="bf16", tokens=2048, top=8, dim=2048, add=True, dropped=0.01),
        # one decoded token of a request with an adapter, beside a square projection
        dict(kind="adapters", name="adapters_token", type="f32", weights="bf16", tokens=1, rows=2560, cols=2560, slots=4, rank=16,
             requests=1, ragged=False),
        # 48 users, each with an adapter of its own or none, ranks of 8 to 64
        dict(kind="adapters", name="adapters_users", type="f32", weights="f16", tokens=48, rows=4096, cols=4096, slots=32, rank=64,
             requests=48, ragged=True),
        # five requests' prompts behind one another, an odd count
        dict(kind="adapters", name="adapters_prompts", type="f32", weights="bf16", tokens=1531, rows=6912, cols=2560, slots=8, rank=16,
             requests=5, ragged=False),
        # the largest: many long prompts beside a wide square projection
        dict(kind="adapters", name="adapters_long", type="bf16", weights="bf16", tokens=8192, rows=4096, cols=4096, slots=16, rank=64,
             requests=9, ragged=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng: random.Random):
    kind = rng.choice(["route", "route", "sort", "combine", "adapters", "adapters"])
    if kind in ("route", "sort"):
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log_int(rng, max(2, 8 // groups), 512 // groups)
        kept = rng.randint(1, groups)
        top = rng.randint(1, min(16, experts // groups * kept))
        if kind == "sort":
            return dict(kind=kind, tokens=_log_int(rng, 1, 32768 * 8 // top), experts=experts, top=top, dropped=rng.choice([0.0, 0.02, 0.5]))
        tokens = _log_int(rng, 1, min(16384, 16001 * 256 // experts))
        return dict(kind=kind, type=rng.choice(["f32", "f32", "f16", "bf16"]), tokens=tokens, experts=experts, top=top,
                    score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups, kept=kept,
                    best=rng.choice([1, 2]) if groups > 1 else 1, renormalise=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]),
                    padded=rng.randint(0, tokens // 4))
    if kind == "combine":
        dim, top = _log_int(rng, 64, 8192), rng.randint(1, 12)
        return dict(kind=kind, type=rng.choice(["f32", "f16", "bf16"]), tokens=_log_int(rng, 1, max(1, 2048 * 8 * 2048 // (dim * top))),
                    top=top, dim=dim, add=rng.random() < 0.7, dropped=rng.choice([0.0, 0.01, 0.3]))
    rows, cols, rank = _log_int(rng, 64, 8192), _log_int(rng, 64, 8192), rng.choice([4, 8, 16, 16, 32, 64, rng.randint(1, 64)])
    tokens = _log_int(rng, 1, min(8192, 8192 * 4096 * 2 // (rows + cols)))
    return dict(kind=kind, type=rng.choice(["f32", "f16", "bf16"]), weights=rng.choice(["f32", "f16", "bf16"]), tokens=tokens, rows=rows,
                cols=cols, slots=_log_int(rng, 1, 48), rank=rank, requests=rng.choice([1, min(5, tokens), min(tokens, 64)]),
                ragged=rng.random() < 0.4)


# ---- inputs ----

def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(int(seed) * 7411 + 83)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=_DEV)


def _chosen(g, tokens, experts, top, dropped):
    """Distinct experts of each token, by popularity, a share of them dropped."""
    score = _randn(g, tokens, experts) + 0.7 * _randn(g, 1, experts)
    ids = score.topk(top, 1)[1].int()
    return torch.where(torch.rand((tokens, top), generator=g, device=_DEV) < dropped, -1, ids)


def _places(ids, experts):
    """(key, order): pairs in order of their expert, pairs without one last."""
    flat = ids.flatten().long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    return key, torch.argsort(key, stable=True)


def _inputs(c, seed):
    g, kind = _gen(seed), c["kind"]
    t = c["tokens"]
    if kind == "route":
        logits = 1.5 * _randn(g, t, c["experts"]) + 0.7 * _randn(g, 1, c["experts"])
        if c["padded"]:
            logits[t - c["padded"]:] = -math.inf
        return {"logits": logits.to(_TYPES[c["type"]]), "bias": 0.2 * _randn(g, c["experts"]) if c["bias"] else None}
    if kind == "sort":
        return {"ids": _chosen(g, t, c["experts"], c["top"], c["dropped"])}
    if kind == "combine":
        ids = _chosen(g, t, max(8, c["top"]), c["top"], c["dropped"])
        key, order = _places(ids, max(8, c["top"]))
        slot = torch.empty_like(order)
        slot[order] = torch.arange(t * c["top"], device=_DEV)
        w = torch.rand((t, c["top"]), generator=g, device=_DEV)
        return {"y": _randn(g, t * c["top"], c["dim"]), "slot": torch.where(ids.flatten() >= 0, slot, -1).int(),
                "weights": w / w.sum(1, keepdim=True), "add": _randn(g, t, c["dim"]) if c["add"] else None}
    r = c["rank"]
    wt = _TYPES[c["weights"]]
    ranks = torch.full((c["slots"],), r, dtype=torch.int64)
    if c["ragged"]:
        ranks = torch.tensor([max(1, r >> (i % 4)) for i in range(c["slots"])])
    a = (_randn(g, c["slots"], r, c["cols"]) / math.sqrt(c["cols"])).to(wt)
    b = (_randn(g, c["slots"], c["rows"], r) / math.sqrt(r)).to(wt)
    mine = torch.arange(r)[None] < ranks[:, None]
    a, b = a * mine[:, :, None].to(_DEV), b * mine[:, None, :].to(_DEV)
    # requests of ragged lengths behind one another; where there are many, one in eight has no adapter
    cuts = torch.rand((c["requests"],), generator=g, device=_DEV).sort()[0]
    at = torch.searchsorted(cuts, torch.arange(t, device=_DEV) / t) if c["requests"] < t else torch.arange(t, device=_DEV)
    of = torch.randint(0, c["slots"], (max(t, c["requests"]) + 1,), generator=g, device=_DEV)
    of = torch.where((torch.rand(of.shape, generator=g, device=_DEV) < 0.125) & (c["requests"] > 8), -1, of)
    x = _randn(g, t, c["cols"])
    x = torch.where(torch.rand(x.shape, generator=g, device=_DEV) < 0.01, 20.0 * x, x)
    return {"x": x.to(_TYPES[c["type"]]), "a": a, "b": b, "ranks": ranks.tolist(), "of": of[at].int(),
            "scales": [0.5 + 0.25 * (i % 5) for i in range(c["slots"])], "base": _randn(g, t, c["rows"])}


def prepare(case, seed):
    c = case
    s = dict(_inputs(c, seed), case=c)
    t = c["tokens"]
    ints = lambda n: torch.full((n,), -7, dtype=torch.int32, device=_DEV)   # noqa: E731
    if c["kind"] in ("route", "sort"):
        n = t * c["top"]
        s.update(offsets=ints(c["experts"] + 1), row=ints(n), slot=ints(n))
        if c["kind"] == "route":
            s.update(ids=ints(n).view(t, c["top"]), weights=torch.zeros((t, c["top"]), device=_DEV))
    elif c["kind"] == "combine":
        s["out"] = torch.zeros((t, c["dim"]), dtype=_TYPES[c["type"]], device=_DEV)
    else:
        s["y"] = torch.zeros((t, c["rows"]), device=_DEV)
        s["scale"] = torch.tensor(s["scales"], device=_DEV)
        counts = torch.bincount((s["of"] + 1).long(), minlength=c["slots"] + 1)
        s["most"] = int(counts[1:].max())
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
    """The handle, workspace and arguments of the call, as a program keeps them from step to step."""
    bh = _framework()
    bh.check(bh.load().eif_hip_init(0), "eif_hip_init")
    lib, kind, t = bh.load(), c["kind"], c["tokens"]
    if kind in ("route", "sort"):
        need = lib.eif_hip_moe_sort_bytes(t, c["top"], c["experts"])
        s["work"] = torch.empty((max(need, 4),), dtype=torch.uint8, device=_DEV)
        places = (_p(s["offsets"]), _p(s["row"]), _p(s["slot"]), _p(s["work"]), need)
        if kind == "sort":
            return lib.eif_hip_moe_sort, (_p(s["ids"]), t, c["top"], c["experts"]) + places
        s["spec"] = bh.MoeRouteSpec(experts=c["experts"], top_k=c["top"], score={"softmax": 0, "sigmoid": 1}[c["score"]],
                                    bias=None if s["bias"] is None else s["bias"].data_ptr(), groups=c["groups"], groups_kept=c["kept"],
                                    group_best=c["best"], renormalise=int(c["renormalise"]), scale=c["scale"])
        return lib.eif_hip_moe_route, (_p(s["logits"]), _TYPE_IDS[c["type"]], c["experts"], t, C.byref(s["spec"]), _p(s["ids"]),
                                       _p(s["weights"])) + places
    if kind == "combine":
        return lib.eif_hip_moe_combine, (_p(s["y"]), c["dim"], t * c["top"], _p(s["slot"]), _p(s["weights"]), t, c["top"], _p(s["add"]),
                                         c["dim"] if c["add"] else 0, c["dim"], _p(s["out"]), _TYPE_IDS[c["type"]], c["dim"])
    h = s["adapters"] = bh.Adapters(c["slots"], c["rows"], c["cols"], c["rank"], s["a"].dtype)
    for i, r in enumerate(s["ranks"]):
        h.set(i, s["a"][i, :r], s["b"][i, :, :r], s["scales"][i])
    return lib.eif_hip_adapters_linear, (h.h, _p(s["x"]), _TYPE_IDS[c["type"]], c["cols"], _p(s["of"]), _p(s["base"]), c["rows"],
                                         _p(s["y"]), c["rows"], t)


_OUTPUTS = {"route": ("ids", "weights", "offsets", "row", "slot"), "sort": ("offsets", "row", "slot"), "combine": ("out",),
            "adapters": ("y",)}


def _run_own(s):
    f, args = s["call"]
    rc = f(*args, torch.cuda.current_stream().cuda_stream)
    if rc:
        raise RuntimeError("%s: %d" % (f.__name__, rc))
    return {k: s[k] for k in _OUTPUTS[s["case"]["kind"]]}


# ---- the plain forms ----

def _plain_route(s):
    c = s["case"]
    l = s["logits"].double().clamp(max=_MOST)
    open_ = l > -math.inf
    l = torch.where(open_, l, -math.inf)
    if c["score"] == "softmax":
        p = torch.where(open_, torch.exp(l - l.amax(1, keepdim=True)), 0.0)
        p = torch.where(open_, p / p.sum(1, keepdim=True), 0.0)
    else:
        p = 1.0 / (1.0 + torch.exp(-l))
    value = p if s["bias"] is None else p + s["bias"].double()
    by = l if s["bias"] is None else torch.where(open_, value, -math.inf)
    if c["groups"] > 1:
        split = (l.shape[0], c["groups"], -1)
        best = by.view(split).amax(2)
        if c["best"] == 2:
            two = torch.where(open_, value, -math.inf).view(split).topk(min(2, c["experts"] // c["groups"]), 2)[0]
            best = torch.where(best > -math.inf, torch.where(two > -math.inf, two, 0.0).sum(2), -math.inf)
        keep = torch.sort(best, dim=1, descending=True, stable=True)[1][:, :c["kept"]]
        kept = torch.zeros_like(best, dtype=torch.bool).scatter_(1, keep, True)
        by = torch.where(kept[:, :, None], by.view(split), -math.inf).view(l.shape)
    by, ids = torch.sort(by, dim=1, descending=True, stable=True)
    by, ids = by[:, :c["top"]], ids[:, :c["top"]]
    there = by > -math.inf
    if not c["renormalise"]:
        w = p.gather(1, ids)
    elif c["score"] == "softmax":
        w = torch.where(there, l.gather(1, ids), -math.inf)
        w = torch.exp(w - w.amax(1, keepdim=True))
        w = w / w.sum(1, keepdim=True)
    else:
        w = torch.where(there, p.gather(1, ids), 0.0)
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    return torch.where(there, ids, -1).int(), torch.where(there, w * c["scale"], 0.0).float()


def _plain_sort(ids, s):
    c = s["case"]
    key, order = _places(ids, c["experts"])
    n = key.numel()
    counts = torch.zeros(c["experts"] + 1, dtype=torch.int64, device=_DEV).scatter_add_(0, key, torch.ones_like(key))
    ends = counts.cumsum(0)[:-1]
    at = torch.arange(n, device=_DEV)
    slot = torch.empty_like(order).scatter_(0, order, at)
    return {"offsets": torch.cat([ends.new_zeros(1), ends]).int(), "row": torch.where(at < ends[-1], order // c["top"], s["row"]).int(),
            "slot": torch.where(key < c["experts"], slot, -1).int()}


def _plain_combine(s):
    c = s["case"]
    slot = s["slot"].view(c["tokens"], c["top"])
    rows = s["y"][slot.clamp(min=0).long()] * s["weights"][:, :, None]
    y = torch.where(slot[:, :, None] >= 0, rows, 0.0).sum(1)
    y = y if s["add"] is None else s["add"] + y
    return y.to(_TYPES[c["type"]])


def _plain_adapters(s):
    # every adapter's rows in a panel of the largest count, two batched products
    c, of = s["case"], s["of"].long()
    key = torch.where(of >= 0, of, c["slots"])
    order = torch.argsort(key, stable=True)
    first = torch.searchsorted(key[order], torch.arange(c["slots"] + 1, device=_DEV))
    place = torch.empty_like(order).scatter_(0, order, torch.arange(c["tokens"], device=_DEV)) - first[key]
    has = of >= 0
    panel = torch.zeros((c["slots"] + 1, max(s["most"], 1), c["cols"]), device=_DEV)
    panel[key, torch.where(has, place, 0)] = s["x"].float()
    v = torch.matmul(panel[:-1], s["a"].float().transpose(1, 2).contiguous()) * s["scale"][:, None, None]
    y = torch.matmul(v, s["b"].float().transpose(1, 2).contiguous())
    y = y[torch.where(has, of, 0), torch.where(has, place, 0)]
    return s["base"] + torch.where(has[:, None], y, 0.0)


def _plain(s):
    kind = s["case"]["kind"]
    if kind == "route":
        ids, weights = _plain_route(s)
        return dict(ids=ids, weights=weights, **_plain_sort(ids, s))
    if kind == "sort":
        return _plain_sort(s["ids"], s)
    return {"out": _plain_combine(s)} if kind == "combine" else {"y": _plain_adapters(s)}


def run(state):
    return _run_own(state) if own else _plain(state)


# ---- what a pass cannot do without ----

def work(case):
    c, t = case, case["tokens"]
    if c["kind"] == "combine":
        n = t * c["top"] * (1.0 - c["dropped"])
        return {"bytes": 4 * n * c["dim"] + t * c["dim"] * ((4 if c["add"] else 0) + _SIZE[c["type"]]) + 8 * t * c["top"],
                "flops": 2 * n * c["dim"]}
    if c["kind"] == "adapters":
        n = t * (0.875 if c["requests"] > 8 else 1.0)
        busy = c["slots"] * (1.0 - (1.0 - 1.0 / c["slots"]) ** min(c["requests"], t))   # adapters with rows, for even odds
        rank = sum(max(1, c["rank"] >> (i % 4)) for i in range(c["slots"])) / c["slots"] if c["ragged"] else c["rank"]
        return {"bytes": n * c["cols"] * _SIZE[c["type"]] + busy * rank * (c["rows"] + c["cols"]) * _SIZE[c["weights"]] + 8 * t * c["rows"],
                "flops": 2 * n * rank * (c["rows"] + c["cols"])}
    n = t * c["top"]
    if c["kind"] == "sort":
        return {"bytes": 12 * n + 4 * c["experts"], "flops": 2 * n}
    return {"bytes": t * c["experts"] * _SIZE[c["type"]] + 16 * n + 8 * c["experts"], "flops": 40 * t * c["experts"]}


# ---- the same from the definition, in 64 bits ----

def _exact_route(c, logits, bias):
    l = np.minimum(logits.double().cpu().numpy(), _MOST)
    shut = ~(l > -np.inf)
    with np.errstate(all="ignore"):
        if c["score"] == "softmax":
            e = np.exp(l - np.max(np.where(shut, -np.inf, l), 1, keepdims=True))
            e[shut] = 0.0
            p = e / e.sum(1, keepdims=True)
        else:
            p = 1.0 / (1.0 + np.exp(-l))
    p[shut] = 0.0
    value = p if bias is None else p + bias.double().cpu().numpy()
    by = np.where(shut, -np.inf, l if bias is None else value)
    size = c["experts"] // c["groups"]
    if c["groups"] > 1:
        high = np.sort(np.where(shut, -np.inf, value if c["best"] == 2 else by).reshape(len(l), c["groups"], size), 2)[:, :, ::-1]
        high = high[:, :, :c["best"]]
        of_group = np.where(high[:, :, 0] == -np.inf, -np.inf, np.where(high == -np.inf, 0.0, high).sum(2))
        rank = np.argsort(np.argsort(-of_group, 1, kind="stable"), 1)
        by = np.where(np.repeat(rank < c["kept"], size, 1), by, -np.inf)
    ids = np.argsort(-by, 1, kind="stable")[:, :c["top"]]
    there = np.take_along_axis(by, ids, 1) > -np.inf
    if c["renormalise"] and c["score"] == "softmax":   # softmax over the chosen
        z = np.where(there, np.take_along_axis(l, ids, 1), -np.inf)
        with np.errstate(all="ignore"):
            w = np.exp(z - z.max(1, keepdims=True))
    else:
        w = np.where(there, np.take_along_axis(p, ids, 1), 0.0)
    w = np.where(there, w, 0.0)
    if c["renormalise"]:
        total = w.sum(1, keepdims=True)
        w = np.divide(w, total, out=np.zeros_like(w), where=total > 0)
    return np.where(there, ids, -1).astype(np.int32), w * c["scale"]


def exact(case, seed):
    c, d = case, _inputs(case, seed)
    if c["kind"] == "route":
        ids, w = _exact_route(c, d["logits"], d["bias"])
        return {"ids": ids, "weights": w, "offsets": None, "row": None, "slot": None}
    if c["kind"] == "sort":
        return None   # whole numbers alone
    if c["kind"] == "combine":
        out = torch.zeros((c["tokens"], c["dim"]), dtype=torch.float64, device=_DEV) if d["add"] is None else d["add"].double()
        slot = d["slot"].view(c["tokens"], c["top"]).long()
        for k in range(c["top"]):
            at = torch.nonzero(slot[:, k] >= 0)[:, 0]
            out[at] += d["weights"][at, k, None].double() * d["y"][slot[at, k]].double()
        return {"out": out}
    y = d["base"].double()
    for i, r in enumerate(d["ranks"]):
        at = torch.nonzero(d["of"] == i)[:, 0]
        v = d["x"][at].double() @ d["a"][i, :r].double().T
        y[at] += d["scales"][i] * (v @ d["b"][i, :, :r].double().T)
    return {"y": y}
