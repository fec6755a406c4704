"""Operators on 8-bit floating point (e4m3) with a scale for every block of 128, as cases that can be timed: the norm that leaves its
rows in that form, dense and gated products of such rows with matrices of 128 x 128 blocks, and the routed experts of a layer,
whose lists are ragged.  Sizes are those of the benchmark's 35B-A3B-shaped transformer (model width 2048, 256 experts of 512,
vocabulary 248320) and generic ones; draw() spreads them over the ranges that the operators take.

A row's block of up to 128 values v, with m = max(max |v|, 2^-100), is held as the scale m / 448 and the codes e4m3(v * (448 / m)); both
quotients and the product are FP32.  A matrix stands for scale[r div 128, k div 128] * code[r, k].

listed() / draw(rng) give cases, prepare(case, seed) what a program holds before the call, run(state) one pass: the
framework's calls where `own` is true, plain torch operations in 32 bits where it is not."""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
VOCAB, K_MODEL = 248320, 2048
BLOCK, LARGEST, SMALLEST = 128, 448.0, 2.0 ** -100
CODE_SPREAD = 112.0  # standard deviation of the codes of a normal weight: the largest of a block of 128 x 128 is at four of it
WEIGHT_SCALE = 0.02
EXPERT_SPREAD = 0.25  # how far the experts' popularity lies apart, against the tokens' own choice
E4M3 = torch.float8_e4m3fn


def listed() -> list[dict]:
    return [
        # the residual's addition and norm ahead of a projection: one token, nothing but latency
        {"name": "norm_t1", "kind": "norm", "tokens": 1, "n": 2048, "slots": 0, "sum": True},
        # a ragged batch behind the experts of a layer: their weighted sum, the residual and the norm
        {"name": "norm_t333", "kind": "norm", "tokens": 333, "n": 2576, "slots": 8, "sum": True},
        # a long prompt
        {"name": "norm_t8192", "kind": "norm", "tokens": 8192, "n": 2048, "slots": 0, "sum": True},
        # one small projection of one token, from BF16
        {"name": "linear_small_t1", "kind": "linear", "rows": 512, "k": 2048, "tokens": 1, "x": "bf16", "scales": "f32", "out": "bf16"},
        # the output projection of one token, behind the norm
        {"name": "linear_head_t1", "kind": "linear", "rows": VOCAB, "k": 2048, "tokens": 1, "x": "rows", "scales": "f32", "out": "f32"},
        # a small ragged batch on a matrix whose last blocks are cut short, scales in BF16
        {"name": "linear_t19", "kind": "linear", "rows": 1453, "k": 2576, "tokens": 19, "x": "bf16", "scales": "bf16", "out": "bf16"},
        # qkv projection of a prompt behind the norm; a wide projection of a long one
        {"name": "linear_t2048", "kind": "linear", "rows": 5120, "k": 2048, "tokens": 2048, "x": "rows", "scales": "f32", "out": "bf16"},
        {"name": "linear_t8192", "kind": "linear", "rows": 8192, "k": 2048, "tokens": 8192, "x": "rows", "scales": "f32", "out": "bf16"},
        # gate and up of a shared expert, its hidden rows in 8 bits for the product behind it
        {"name": "glu_t300", "kind": "glu", "rows": 1408, "k": 2048, "tokens": 300, "x": "rows", "scales": "f32", "out": "rows"},
        # the routed experts of a layer: one token, a ragged batch, a prompt
        {"name": "experts_t1", "kind": "experts", "experts": 256, "mid": 512, "k": K_MODEL, "topk": 8, "tokens": 1, "x": "bf16", "scales": "f32"},
        {"name": "experts_t77", "kind": "experts", "experts": 256, "mid": 512, "k": K_MODEL, "topk": 8, "tokens": 77, "x": "bf16", "scales": "bf16"},
        {"name": "experts_t2048", "kind": "experts", "experts": 256, "mid": 512, "k": K_MODEL, "topk": 8, "tokens": 2048, "x": "rows", "scales": "f32"},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    """One more case of the same kinds; no larger than the largest listed ones."""
    kind = rng.choice(("norm", "norm", "linear", "linear", "linear", "glu", "experts", "experts"))
    if kind == "norm":
        n = 16 * _log_int(rng, 4, 512)
        slots = rng.choice((0, 0, 0, 2, 8))
        return {"kind": kind, "tokens": _log_int(rng, 1, min(8192, (1 << 24) // (n * max(1, slots)))), "n": n, "slots": slots, "sum": rng.random() < 0.7}
    how = {"x": rng.choice(("bf16", "rows", "rows")), "scales": rng.choice(("f32", "f32", "bf16"))}
    if kind in ("linear", "glu"):
        k = 16 * _log_int(rng, 4, 512)
        rows = _log_int(rng, 1, min(VOCAB, (1 << (28 if kind == "glu" else 29)) // k))
        rows += -rows % 16 if kind == "glu" else 0  # (the hidden rows are the next product's)
        tokens = _log_int(rng, 1, max(1, min(8192, (1 << 35) // (rows * k))))
        return {"kind": kind, "rows": rows, "k": k, "tokens": tokens, **how, "out": rng.choice(("bf16", "bf16", "f32") if kind == "linear" else ("rows", "rows", "bf16"))}
    experts, mid = rng.choice(((256, 512), (128, 768), (64, 1024), (48, 512), (24, 720), (8, 1408)))
    return {"kind": kind, "experts": experts, "mid": mid, "k": 512 * rng.randint(1, 4), "topk": rng.choice((1, 2, 4, 6, 8)),
            "tokens": _log_int(rng, 1, 2048), **how}


def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _matrix(g: torch.Generator, case: dict, rows: int, k: int, n_matrices: int = 1) -> dict:
    """codes e4m3 [n_matrices * rows, k], scales [n_matrices * ceil(rows / 128), ceil(k / 128)]: blocks begin anew in every matrix."""
    codes = torch.empty((n_matrices * rows, k), dtype=E4M3, device=DEVICE)
    step = max(1, (1 << 28) // k)
    for r in range(0, n_matrices * rows, step):
        m = min(step, n_matrices * rows - r)
        codes[r: r + m] = (torch.randn((m, k), generator=g, device=DEVICE) * CODE_SPREAD).clamp_(-LARGEST, LARGEST).to(E4M3)
    scales = (0.5 + torch.rand((n_matrices * -(-rows // BLOCK), -(-k // BLOCK)), generator=g, device=DEVICE)) * (WEIGHT_SCALE / CODE_SPREAD)
    return {"codes": codes, "scales": scales.to(torch.bfloat16) if case["scales"] == "bf16" else scales, "n_matrices": n_matrices}


def _rows(v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of FP32 rows [T, K], a scale for every 128 columns."""
    t, k = v.shape
    blocks = torch.nn.functional.pad(v, (0, -k % BLOCK)).view(t, -1, BLOCK)
    m = blocks.abs().amax(2).clamp_min(SMALLEST)
    q = (blocks * (torch.full_like(m, LARGEST) / m)[:, :, None]).to(E4M3)  # (a number over a tensor is a product with its reciprocal)
    return q.view(t, -1)[:, :k].contiguous(), m / LARGEST


def _activations(g: torch.Generator, case: dict, rows: int, k: int):
    """Normal activations with a few wide columns, as a transformer's have; BF16, or codes and scales that an earlier call left."""
    x = torch.randn((rows, k), generator=g, device=DEVICE) * (1.0 + 7.0 * (torch.rand(k, generator=g, device=DEVICE) < 0.01))
    return x.to(torch.bfloat16) if case["x"] == "bf16" else _rows(x)


def _scores(tokens: int, experts: int, g: torch.Generator, device: str) -> torch.Tensor:
    r = lambda *s: torch.randn(s, generator=g, device=device)  # noqa: E731
    return r(tokens, experts) + EXPERT_SPREAD * r(experts)


def _inputs(case: dict, seed: int) -> dict:
    g = _generator(seed)
    kind, t = case["kind"], case["tokens"]
    st = {"kind": kind, "case": case}
    if kind == "norm":
        n, slots = case["n"], case["slots"]
        r = lambda *s: torch.randn(s, generator=g, device=DEVICE)  # noqa: E731
        st["a"], st["b"] = (r(t, n) * 2).to(torch.bfloat16), r(t, n).to(torch.bfloat16)
        st["gamma"] = (1 + 0.2 * r(n)).to(torch.bfloat16)
        st["ys"], st["wts"] = (r(t, slots, n), torch.softmax(r(t, slots), 1)) if slots else (None, None)
        return st
    k = case["k"]
    if kind == "experts":
        e, mid = case["experts"], case["mid"]
        for name, rows, cols in (("gate", mid, k), ("up", mid, k), ("down", k, mid)):
            st[name] = _matrix(g, case, rows, cols, e)
        wts, ids = torch.softmax(_scores(t, e, g, DEVICE), 1).topk(case["topk"], dim=1)
        st["ids"], st["wts"] = ids.to(torch.int32), wts / wts.sum(1, keepdim=True)
    else:
        st["w"] = _matrix(g, case, case["rows"], k)
        if kind == "glu":
            st["up"] = _matrix(g, case, case["rows"], k)
    st["x"] = _activations(g, case, t, k)
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
                st[name] = ops.Fp8Weight(m["codes"], m["scales"], m["n_matrices"])
        if isinstance(st.get("x"), tuple):
            st["x"] = ops.Fp8Rows(*st["x"])
    return st


OUT = {"bf16": torch.bfloat16, "f32": torch.float32, "rows": E4M3}


# ---------------------------------------------------------------- the framework's calls

def _run_own(st: dict):
    ops, case, kind = st["ops"], st["case"], st["kind"]
    if kind == "norm":
        r = ops.add_rmsnorm_fp8(st["a"], st["b"], ys=st["ys"], topk_weights=st["wts"], gamma=st["gamma"], want_sum=case["sum"])
        return (r[0].codes, r[0].scales, r[1]) if case["sum"] else (r.codes, r.scales)
    if kind == "linear":
        return ops.fp8_linear(st["x"], st["w"], out_dtype=OUT[case["out"]])
    if kind == "glu":
        r = ops.fp8_linear_glu2(st["x"], st["w"], st["up"], out_dtype=OUT[case["out"]])
        return (r.codes, r.scales) if case["out"] == "rows" else r
    return ops.fp8_moe_experts(st["x"], st["gate"], st["up"], st["down"], st["wts"], st["ids"], case["experts"])


# ---------------------------------------------------------------- plain form

def _row_values(x) -> torch.Tensor:
    q, s = x if isinstance(x, tuple) else _rows(x.float())
    return q.float() * s.repeat_interleave(BLOCK, 1)[:, : q.shape[1]]


def _weight_values(m: dict, which: torch.Tensor | None = None) -> torch.Tensor:
    """[matrices, rows, k] FP32, of all matrices or of those that `which` names."""
    n = m["n_matrices"]
    codes, scales = m["codes"].view(torch.uint8).view(n, -1, m["codes"].shape[1]), m["scales"].view(n, -1, m["scales"].shape[1])
    if which is not None:
        codes, scales = codes[which], scales[which]
    rows, k = codes.shape[1:]
    return codes.view(E4M3).float().mul_(scales.float().repeat_interleave(BLOCK, 1)[:, :rows].repeat_interleave(BLOCK, 2)[:, :, :k])


def _silu(v: torch.Tensor) -> torch.Tensor:
    return v / (1.0 + torch.exp(-v))


def _plain_norm(st: dict):
    case = st["case"]
    s = st["a"].float() + st["b"].float()
    if st["ys"] is not None:
        s = s + (st["ys"] * st["wts"][:, :, None]).sum(1)
    y = s * torch.rsqrt((s * s).mean(1, keepdim=True) + 1e-6) * st["gamma"].float()
    return (*_rows(y), s.to(torch.bfloat16)) if case["sum"] else _rows(y)


def _plain_experts(st: dict) -> torch.Tensor:
    """The pairs of every expert that is named as one padded product."""
    x, ids = _row_values(st["x"]), st["ids"].long()
    t, slots = ids.shape
    named, of = torch.unique(ids.reshape(-1), return_inverse=True)
    count = torch.bincount(of, minlength=named.numel())
    order = torch.argsort(of, stable=True)
    place = torch.arange(t * slots, device=x.device) - (torch.cumsum(count, 0) - count)[of[order]]
    wide = int(count.max())
    at = torch.empty_like(of)
    at[order] = of[order] * wide + place
    xe = torch.zeros((named.numel() * wide, x.shape[1]), dtype=torch.float32, device=x.device)
    xe[at] = x.repeat_interleave(slots, 0)
    xe = xe.view(named.numel(), wide, -1).transpose(1, 2).contiguous()
    h = _silu(torch.matmul(_weight_values(st["gate"], named), xe)) * torch.matmul(_weight_values(st["up"], named), xe)
    hidden = _row_values(_rows(h.transpose(1, 2).reshape(named.numel() * wide, -1)))
    y = torch.matmul(_weight_values(st["down"], named), hidden.view(named.numel(), wide, -1).transpose(1, 2).contiguous())
    ys = y.transpose(1, 2).reshape(named.numel() * wide, -1)[at].view(t, slots, -1)
    return (ys * st["wts"][:, :, None]).sum(1).to(torch.bfloat16)


def run(st: dict):
    if own:
        return _run_own(st)
    kind = st["kind"]
    if kind == "norm":
        return _plain_norm(st)
    if kind == "experts":
        return _plain_experts(st)
    x, out = _row_values(st["x"]), st["case"]["out"]
    y = x @ _weight_values(st["w"])[0].t()
    if kind == "glu":
        y = _silu(y) * (x @ _weight_values(st["up"])[0].t())
    return _rows(y) if out == "rows" else y.to(OUT[out])


# ---------------------------------------------------------------- from the definition, in 64 bits

def _to_grid(v: torch.Tensor) -> torch.Tensor:
    """The nearest number of four significant bits from 2^-6 on, of the multiples of 2^-9 below; ties to the even one."""
    e = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(v / step) * step


def _in_blocks(v: torch.Tensor):
    """(codes' values, scales) of rows in 64 bits; the quotient and the product are FP32 by definition."""
    t, k = v.shape
    codes, scales = [], []
    for c in range(0, k, BLOCK):
        b = v[:, c: c + BLOCK]
        m = b.abs().max(1, keepdim=True).values.clamp_min(SMALLEST).float()
        codes.append(_to_grid((b.float() * torch.true_divide(torch.tensor(LARGEST, device=m.device).expand_as(m), m)).double()))
        scales.append((m / LARGEST).double())
    return torch.cat(codes, 1), torch.cat(scales, 1)


def _spread(s: torch.Tensor, k: int) -> torch.Tensor:
    return s[:, torch.arange(k, device=s.device) // BLOCK]


def _x64(st: dict) -> torch.Tensor:
    q, s = (st["x"][0].double(), st["x"][1].double()) if isinstance(st["x"], tuple) else _in_blocks(st["x"].double())
    return q * _spread(s, q.shape[1])


def _w64(m: dict, lo: int, hi: int, block_row: int) -> torch.Tensor:
    """Rows lo..hi, which begin with a block whose scales are row block_row of the scales."""
    of = block_row + torch.arange(hi - lo, device=m["codes"].device) // BLOCK
    return m["codes"][lo:hi].double() * _spread(m["scales"].double()[of], m["codes"].shape[1])


def _times(m: dict, x: torch.Tensor) -> torch.Tensor:
    rows, k = m["codes"].shape
    step = max(1, (1 << 26) // k // BLOCK) * BLOCK
    return torch.cat([x @ _w64(m, r, min(r + step, rows), r // BLOCK).t() for r in range(0, rows, step)], dim=1)


def exact(case: dict, seed: int):
    st = _inputs(case, seed)
    kind = case["kind"]
    gated = lambda a, b: a * torch.sigmoid(a) * b  # noqa: E731
    if kind == "norm":
        s = st["a"].double() + st["b"].double()
        for i in range(case["slots"]):
            s = s + st["wts"][:, i, None].double() * st["ys"][:, i].double()
        y = s / torch.sqrt(s.square().sum(1, keepdim=True) / case["n"] + 1e-6) * st["gamma"].double()
        return (*_in_blocks(y), s) if case["sum"] else _in_blocks(y)
    x = _x64(st)
    if kind == "linear":
        return _times(st["w"], x)
    if kind == "glu":
        y = gated(_times(st["w"], x), _times(st["up"], x))
        return _in_blocks(y) if case["out"] == "rows" else y
    mid, k = case["mid"], case["k"]
    weight_of = torch.zeros((case["tokens"], case["experts"]), dtype=torch.float64, device=x.device).scatter_(1, st["ids"].long(), st["wts"].double())
    out = torch.zeros((case["tokens"], k), dtype=torch.float64, device=x.device)
    per_mid, per_k = -(-mid // BLOCK), -(-k // BLOCK)
    for e in torch.unique(st["ids"]).tolist():
        on = weight_of[:, e].nonzero()[:, 0]
        h = gated(x[on] @ _w64(st["gate"], e * mid, e * mid + mid, e * per_mid).t(), x[on] @ _w64(st["up"], e * mid, e * mid + mid, e * per_mid).t())
        q, s = _in_blocks(h)
        out[on] += weight_of[on, e, None] * ((q * _spread(s, mid)) @ _w64(st["down"], e * k, e * k + k, e * per_k).t())
    return out


def _row_bytes(t: int, k: int, how: str) -> float:
    return t * {"bf16": 2 * k, "f32": 4 * k, "rows": k + 4 * -(-k // BLOCK)}[how]


def _matrix_bytes(case: dict, rows: float, k: int) -> float:
    return rows * k + -(-rows // BLOCK) * -(-k // BLOCK) * (2 if case["scales"] == "bf16" else 4)


def work(case: dict) -> dict:
    """Bytes (codes and scales as stored, inputs and outputs once) and operations one pass cannot do without."""
    kind, t = case["kind"], case["tokens"]
    if kind == "norm":
        n, slots = case["n"], case["slots"]
        return {"bytes": 2 * _row_bytes(t, n, "bf16") + t * slots * (4 * n + 4) + 2 * n + _row_bytes(t, n, "rows") + (_row_bytes(t, n, "bf16") if case["sum"] else 0),
                "flops": 6.0 * t * n + 2.0 * t * slots * n}
    k = case["k"]
    if kind == "experts":
        e, mid, pairs = case["experts"], case["mid"], t * case["topk"]
        ids = _scores(t, e, torch.Generator().manual_seed(0), "cpu").topk(case["topk"], dim=1).indices
        active = torch.unique(ids).numel()  # experts that such tokens name
        return {"bytes": active * (2 * _matrix_bytes(case, mid, k) + _matrix_bytes(case, k, mid)) + _row_bytes(t, k, case["x"]) + 2.0 * t * k + 8 * pairs, "flops": 6.0 * pairs * mid * k}
    n = 2 if kind == "glu" else 1
    return {"bytes": n * _matrix_bytes(case, case["rows"], k) + _row_bytes(t, k, case["x"]) + _row_bytes(t, case["rows"], case["out"]), "flops": 2.0 * n * t * case["rows"] * k}
