"""Operators on 4-bit weights with group scales, and the selection of experts in groups, as cases that can be timed: dense
products and gated products from one token to a prompt, the experts of a layer, the router.  Sizes are those of the
benchmark's 35B-A3B-shaped transformer (model width 2048, 256 experts of 512, vocabulary 248320) and of the tests; draw()
spreads them over the ranges that the operators take.

listed() / draw(rng) give cases, prepare(case, seed) what a program holds before the call, run(state) one pass: the
framework's calls where `own` is true, plain torch operations in 32 bits (64 in the selection) where it is not."""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
VOCAB, K_MODEL = 248320, 2048
CODE_SPREAD = 2.6  # standard deviation of the codes of a normal weight whose group's largest one has the code 15 or 0
WEIGHT_SCALE = 0.02


def listed() -> list[dict]:
    return [
        # one small projection of one token, launched by itself: nothing but latency
        {"name": "mmv_small_t1", "kind": "mmv", "rows": 512, "k": 2048, "tokens": 1, "group": 128, "zeros": False, "scales": "bf16", "x": "bf16"},
        # draft copy of the output projection, one drafted token
        {"name": "mmv_head_t1", "kind": "mmv", "rows": VOCAB, "k": 2048, "tokens": 1, "group": 128, "zeros": False, "scales": "bf16", "x": "bf16"},
        # FP32 activations of three drafted tokens on a checkpoint with FP16 scales and zero points
        {"name": "mmv_f32_t3", "kind": "mmv", "rows": 8192, "k": 2048, "tokens": 3, "group": 64, "zeros": True, "scales": "f16", "x": "f32"},
        # gate / up of a shared expert, a ragged small batch, groups of 32
        {"name": "glu_t11", "kind": "glu", "rows": 1453, "k": 2560, "tokens": 11, "group": 32, "zeros": True, "scales": "bf16", "x": "bf16"},
        # qkv projection of a serving batch, and of a prompt
        {"name": "linear_t16", "kind": "linear", "rows": 5120, "k": 2048, "tokens": 16, "group": 128, "zeros": True, "scales": "f16", "x": "bf16"},
        {"name": "linear_t2048", "kind": "linear", "rows": 5120, "k": 2048, "tokens": 2048, "group": 128, "zeros": False, "scales": "bf16", "x": "bf16"},
        # the routed experts of a layer: one token, a ragged batch, a prompt
        {"name": "experts_t1", "kind": "experts", "experts": 256, "mid": 512, "k": K_MODEL, "topk": 8, "tokens": 1, "group": 128, "zeros": False, "scales": "bf16"},
        {"name": "experts_t77", "kind": "experts", "experts": 256, "mid": 512, "k": K_MODEL, "topk": 8, "tokens": 77, "group": 64, "zeros": True, "scales": "f16"},
        {"name": "experts_t2048", "kind": "experts", "experts": 256, "mid": 512, "k": K_MODEL, "topk": 8, "tokens": 2048, "group": 128, "zeros": False, "scales": "bf16"},
        # selection: one token and a prompt with sigmoid scores, a bias and four of eight groups; softmax scores, three of six groups
        {"name": "router_t1", "kind": "router", "experts": 256, "topk": 8, "tokens": 1, "groups": 8, "kept": 4, "scoring": "sigmoid", "group_score": "top2", "bias": True, "renorm": True, "scale": 2.5},
        {"name": "router_t333", "kind": "router", "experts": 96, "topk": 6, "tokens": 333, "groups": 6, "kept": 3, "scoring": "softmax", "group_score": "max", "bias": False, "renorm": False, "scale": 1.0},
        {"name": "router_t8192", "kind": "router", "experts": 256, "topk": 8, "tokens": 8192, "groups": 8, "kept": 4, "scoring": "sigmoid", "group_score": "top2", "bias": True, "renorm": True, "scale": 2.5},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    """One more case of the same kinds; no larger than the largest listed ones."""
    kind = rng.choice(("mmv", "mmv", "glu", "linear", "linear", "experts", "experts", "router", "router"))
    layout = {"group": rng.choice((32, 64, 128, 128, 256)), "zeros": rng.random() < 0.5, "scales": rng.choice(("bf16", "f16"))}
    if kind in ("mmv", "glu", "linear"):
        k = 32 * _log_int(rng, 2, 256)
        rows = _log_int(rng, 1, min(VOCAB, (1 << (28 if kind == "glu" else 29)) // k))
        most = max(1, min(4096, (1 << 34) // (rows * k)))  # products of a prompt on ordinary matrices, of a few tokens on the largest
        tokens = _log_int(rng, 1, min(most, 16)) if kind != "linear" else _log_int(rng, 1, most)
        x = "f32" if kind != "linear" and rng.random() < 0.3 else "bf16"
        return {"kind": kind, "rows": rows, "k": k, "tokens": tokens, **layout, "x": x}
    if kind == "experts":
        experts, mid = rng.choice(((256, 512), (128, 768), (64, 1024), (48, 512), (8, 1408)))
        return {"kind": kind, "experts": experts, "mid": mid, "k": 512 * rng.randint(1, 4), "topk": rng.choice((1, 2, 4, 6, 8)),
                "tokens": _log_int(rng, 1, 2048), **layout}
    groups = rng.choice((1, 1, 4, 8, 16))
    experts = groups * rng.randint(max(1, 16 // groups), 512 // groups)
    kept = rng.randint(max(1, groups // 4), groups)
    return {"kind": kind, "experts": experts, "topk": rng.randint(1, min(16, kept * (experts // groups))), "tokens": _log_int(rng, 1, 8192),
            "groups": groups, "kept": kept, "scoring": rng.choice(("softmax", "sigmoid")), "group_score": rng.choice(("max", "top2")),
            "bias": rng.random() < 0.6, "renorm": rng.random() < 0.6, "scale": rng.choice((1.0, 2.5))}


def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _matrix(g: torch.Generator, case: dict, rows: int, k: int) -> dict:
    """codes uint8 [rows, k / 2] (even column in the low half), scales [rows, groups], zeros uint8 [rows, groups] or None."""
    codes = torch.empty((rows, k // 2), dtype=torch.uint8, device=DEVICE)
    step = max(1, (1 << 27) // k)
    for r in range(0, rows, step):
        n = min(step, rows - r)
        u = (torch.randn((n, k), generator=g, device=DEVICE) * CODE_SPREAD + 8.0).round_().clamp_(0, 15).to(torch.uint8)
        codes[r: r + n] = u[:, 0::2] | (u[:, 1::2] << 4)
    groups = -(-k // case["group"])
    scales = (0.5 + torch.rand((rows, groups), generator=g, device=DEVICE)) * (WEIGHT_SCALE / CODE_SPREAD)
    zeros = torch.randint(5, 12, (rows, groups), generator=g, device=DEVICE, dtype=torch.uint8) if case["zeros"] else None
    return {"codes": codes, "scales": scales.to(torch.bfloat16 if case["scales"] == "bf16" else torch.float16), "zeros": zeros, "group": case["group"]}


def _inputs(case: dict, seed: int) -> dict:
    g = _generator(seed)
    kind = case["kind"]
    st = {"kind": kind, "case": case}
    if kind == "router":
        st["logits"] = torch.randn((case["tokens"], case["experts"]), generator=g, device=DEVICE) * 1.5
        st["bias"] = torch.randn(case["experts"], generator=g, device=DEVICE) * 0.05 if case["bias"] else None
        return st
    k, t = case["k"], case["tokens"]
    if kind == "experts":
        e, mid = case["experts"], case["mid"]
        for name, rows, cols in (("gate", mid, k), ("up", mid, k), ("down", k, mid)):
            st[name] = _matrix(g, case, e * rows, cols)
        scores = torch.randn((t, e), generator=g, device=DEVICE)
        wts, ids = torch.softmax(scores, 1).topk(case["topk"], dim=1)
        st["ids"], st["wts"] = ids.to(torch.int32), wts / wts.sum(1, keepdim=True)
        st["x"] = torch.randn((t, k), generator=g, device=DEVICE).to(torch.bfloat16)
        return st
    st["w"] = _matrix(g, case, case["rows"], k)
    if kind == "glu":
        st["up"] = _matrix(g, case, case["rows"], k)
    x = torch.randn((t, k), generator=g, device=DEVICE)
    st["x"] = x if case["x"] == "f32" else x.to(torch.bfloat16)
    return st


def prepare(case: dict, seed: int) -> dict:
    st = _inputs(case, seed)
    if own:
        from orin_qwen_lossless_amd import ops

        ops.init()
        st["ops"] = ops
        for name in ("w", "gate", "up", "down"):
            if name in st:
                m = st[name]
                st[name] = ops.Int4Weight(m["codes"], m["scales"], m["zeros"], m["group"])
    return st


# ---------------------------------------------------------------- the framework's calls

def _run_own(st: dict):
    ops, case, kind = st["ops"], st["case"], st["kind"]
    if kind == "mmv":
        return ops.int4_mmv(st["x"], st["w"])
    if kind == "glu":
        return ops.int4_mmv_glu2(st["x"], st["w"], st["up"])
    if kind == "linear":
        return ops.int4_linear(st["x"], st["w"])
    if kind == "experts":
        return ops.int4_moe_experts(st["x"], st["gate"], st["up"], st["down"], st["wts"], st["ids"], case["experts"])
    return ops.router_topk_grouped(st["logits"], case["topk"], bias=st["bias"], n_groups=case["groups"], topk_groups=case["kept"],
                                   scoring=case["scoring"], group_score=case["group_score"], renorm=case["renorm"], scale=case["scale"])


# ---------------------------------------------------------------- plain form

def _plain_weight(m: dict, rows=slice(None)) -> torch.Tensor:
    codes, scales = m["codes"][rows], m["scales"][rows].float()
    n, k = codes.shape[0], codes.shape[1] * 2
    u = torch.empty((n, k), dtype=torch.float32, device=codes.device)
    u[:, 0::2] = codes & 15
    u[:, 1::2] = codes >> 4
    zeros = m["zeros"][rows].float() if m["zeros"] is not None else torch.full_like(scales, 8.0)
    spread = lambda t: t.repeat_interleave(m["group"], 1)[:, :k]  # noqa: E731
    return u.sub_(spread(zeros)).mul_(spread(scales))


def _silu(v: torch.Tensor) -> torch.Tensor:
    return v / (1.0 + torch.exp(-v))


def _plain_experts(st: dict) -> torch.Tensor:
    case, x, ids, wts = st["case"], st["x"].float(), st["ids"], st["wts"]
    e, mid, k = case["experts"], case["mid"], case["k"]
    t, slots = ids.shape
    if t * slots <= 64:  # few: the matrices of every (token, slot)
        rows = lambda n: (ids.reshape(-1).long()[:, None] * n + torch.arange(n, device=ids.device)).reshape(-1)  # noqa: E731
        xr = x.repeat_interleave(slots, 0).unsqueeze(2)
        g = torch.matmul(_plain_weight(st["gate"], rows(mid)).view(t * slots, mid, k), xr)
        u = torch.matmul(_plain_weight(st["up"], rows(mid)).view(t * slots, mid, k), xr)
        y = torch.matmul(_plain_weight(st["down"], rows(k)).view(t * slots, k, mid), _silu(g) * u)
        return (y.view(t, slots, k) * wts[:, :, None]).sum(1).to(torch.bfloat16)
    out = torch.zeros((t, k), dtype=torch.float32, device=x.device)
    for i in range(e):
        tok, slot = (ids == i).nonzero(as_tuple=True)
        if tok.numel() == 0:
            continue
        xe = x[tok]
        h = _silu(xe @ _plain_weight(st["gate"], slice(i * mid, (i + 1) * mid)).t()) * (xe @ _plain_weight(st["up"], slice(i * mid, (i + 1) * mid)).t())
        out.index_add_(0, tok, (h @ _plain_weight(st["down"], slice(i * k, (i + 1) * k)).t()) * wts[tok, slot][:, None])
    return out.to(torch.bfloat16)


def _first(v: torch.Tensor, n: int) -> torch.Tensor:
    """Indices of the n largest along the last axis, ties to the lowest index."""
    return torch.sort(v, dim=-1, descending=True, stable=True).indices[..., :n]


def _plain_router(st: dict):
    case, logits = st["case"], st["logits"].double()  # choices are compared: 32 bits would order near ones by their rounding
    t, e, groups = case["tokens"], case["experts"], case["groups"]
    if case["scoring"] == "softmax":
        p = torch.exp(logits - logits.max(1, keepdim=True).values)
        p = p / p.sum(1, keepdim=True)
    else:
        p = 1.0 / (1.0 + torch.exp(-logits))
    choice = p + st["bias"].double() if st["bias"] is not None else p
    if case["kept"] < groups:
        per = choice.view(t, groups, e // groups)
        best = torch.sort(per, dim=2, descending=True).values
        rank = best[:, :, 0] + best[:, :, 1] if case["group_score"] == "top2" and e // groups > 1 else best[:, :, 0]
        keep = torch.zeros((t, groups), dtype=torch.bool, device=logits.device).scatter_(1, _first(rank, case["kept"]), True)
        choice = torch.where(keep[:, :, None], per, -math.inf).view(t, e)
    ids = _first(choice, case["topk"])
    w = p.gather(1, ids)
    if case["renorm"]:
        w = w / w.sum(1, keepdim=True)
    return (w * case["scale"]).float(), ids.to(torch.int32)


def run(st: dict):
    if own:
        return _run_own(st)
    kind = st["kind"]
    if kind == "router":
        return _plain_router(st)
    if kind == "experts":
        return _plain_experts(st)
    x = st["x"].float()
    y = x @ _plain_weight(st["w"]).t()
    if kind == "glu":
        return _silu(y) * (x @ _plain_weight(st["up"]).t())
    return y.to(torch.bfloat16) if kind == "linear" else y


# ---------------------------------------------------------------- from the definition, in 64 bits

def _value(m: dict, lo: int, hi: int) -> torch.Tensor:
    """w[r, c] = scale[r, c div group] * (code[r, c] - zero[r, c div group]) of rows lo..hi."""
    b = m["codes"][lo:hi].to(torch.int64)
    code = torch.stack((b % 16, b // 16), dim=2).flatten(1).double()
    of = torch.arange(code.shape[1], device=code.device) // m["group"]
    zero = m["zeros"][lo:hi].double()[:, of] if m["zeros"] is not None else 8.0
    return m["scales"][lo:hi].double()[:, of] * (code - zero)


def _times(m: dict, x: torch.Tensor) -> torch.Tensor:
    rows, k = m["codes"].shape[0], m["codes"].shape[1] * 2
    step = max(1, (1 << 26) // k)
    return torch.cat([torch.matmul(_value(m, r, min(r + step, rows)), x.t()).t() for r in range(0, rows, step)], dim=1)


def exact(case: dict, seed: int):
    st = _inputs(case, seed)
    kind = case["kind"]
    gated = lambda a, b: a * torch.sigmoid(a) * b  # noqa: E731
    if kind in ("mmv", "linear"):
        return _times(st["w"], st["x"].double())
    if kind == "glu":
        return gated(_times(st["w"], st["x"].double()), _times(st["up"], st["x"].double()))
    if kind == "experts":
        x, mid, k = st["x"].double(), case["mid"], case["k"]
        weight_of = torch.zeros((case["tokens"], case["experts"]), dtype=torch.float64, device=x.device).scatter_(1, st["ids"].long(), st["wts"].double())
        out = torch.zeros((case["tokens"], k), dtype=torch.float64, device=x.device)
        for e in torch.unique(st["ids"]).tolist():
            on = weight_of[:, e].nonzero()[:, 0]
            h = gated(x[on] @ _value(st["gate"], e * mid, e * mid + mid).t(), x[on] @ _value(st["up"], e * mid, e * mid + mid).t())
            out[on] += weight_of[on, e, None] * (h @ _value(st["down"], e * k, e * k + k).t())
        return out
    z = st["logits"].double()
    p = torch.softmax(z, 1) if case["scoring"] == "softmax" else torch.sigmoid(z)
    c = p if st["bias"] is None else p + st["bias"].double()
    t, e, n = case["tokens"], case["experts"], case["groups"]
    size = e // n
    by_group = c.view(t * n, size)
    rank = by_group.topk(min(2, size) if case["group_score"] == "top2" else 1, dim=1).values.sum(1).view(t, n)
    # a place in the order: how many come before it (larger, or as large with a lower index)
    before = (rank[:, None, :] > rank[:, :, None]).sum(2) + ((rank[:, None, :] == rank[:, :, None]) & torch.ones((n, n), dtype=torch.bool, device=z.device).tril(-1)).sum(2)
    open_ = (before < case["kept"]).repeat_interleave(size, 1)
    ids = torch.empty((t, case["topk"]), dtype=torch.int64, device=z.device)
    for j in range(case["topk"]):
        left = torch.where(open_, c, -math.inf)
        top = left.max(1, keepdim=True).values
        pick = torch.where(open_ & (left == top), torch.arange(e, device=z.device), e).min(1).values
        ids[:, j] = pick
        open_.scatter_(1, pick[:, None], False)
    w = torch.gather(p, 1, ids)
    return w * (case["scale"] / w.sum(1, keepdim=True) if case["renorm"] else case["scale"]), ids.to(torch.int32)


def _matrix_bytes(case: dict, rows: float, k: int) -> float:
    return rows * (k / 2 + -(-k // case["group"]) * (3 if case["zeros"] else 2))


def work(case: dict) -> dict:
    """Bytes (codes, scales and zeros as stored, inputs and outputs once) and operations one pass cannot do without."""
    kind = case["kind"]
    t = case["tokens"]
    if kind == "router":
        return {"bytes": t * (case["experts"] * 4 + case["topk"] * 8) + (4 * case["experts"] if case["bias"] else 0), "flops": 0}
    k = case["k"]
    if kind == "experts":
        e, mid, pairs = case["experts"], case["mid"], t * case["topk"]
        active = e * (1.0 - (1.0 - case["topk"] / e) ** t)  # experts that the tokens are expected to name
        return {"bytes": active * (2 * _matrix_bytes(case, mid, k) + _matrix_bytes(case, k, mid)) + 4.0 * t * k + 8 * pairs, "flops": 6.0 * pairs * mid * k}
    n = 2 if kind == "glu" else 1
    out = 2 if kind == "linear" else 4
    return {"bytes": n * _matrix_bytes(case, case["rows"], k) + t * (k * (4 if case["x"] == "f32" else 2) + case["rows"] * out), "flops": 2.0 * n * t * case["rows"] * k}
