"""What the operators in front of the expert FFN are measured on: the calls that a serving program makes of them in every MoE layer.

A case is a dict of plain values.  ``kind`` names the operator:

``norm``     residual addition, RMS norm and int8 rows with a scale per token (``moe_add_rms_norm_quant``): the int8 rows and scales go to
             the experts, the normalised rows to the router, the sum on to the next layer.
``logits``   the router's product (``moe_router_logits``): hidden states of 16 or 32 bits, weights of theirs or of 32 bits, fp32 logits.
``gating``   the choice of experts (``moe_gating_top_k_grouped``): softmax or sigmoid scores, a bias for balance, groups, top-k,
             renormalised and scaled weights.

Shapes: those of ``synth.CONFIGS`` (hidden 4096 and 7168; 8, 128 and 256 experts) and generic ones off every grid.  Where ``own`` is false
``run`` computes the operators' plain forms in elementary torch operations.
"""
import math

import torch

own = False

_EPSILON = 1e-6     # of the norm
_RENORM_EPS = 1e-20
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_aclnn = None


def _operators():
    """The framework's operators; imported by the passes that call them only."""
    global _aclnn
    if _aclnn is None:
        from __graft_entry__ import load_package
        _aclnn = load_package().aclnn
    return _aclnn


def _norm(name, tokens, hidden, dtype="bf16", gamma="same", residual=True, smooth=False, rows=True):
    return {"name": name, "kind": "norm", "tokens": tokens, "hidden": hidden, "dtype": dtype, "gamma": gamma,
            "residual": residual, "smooth": smooth, "rows": rows}


def _logits(name, tokens, hidden, experts, dtype="bf16", weight="same"):
    return {"name": name, "kind": "logits", "tokens": tokens, "hidden": hidden, "experts": experts, "dtype": dtype, "weight": weight}


def _gating(name, tokens, experts, top_k, score="sigmoid", bias=True, groups=1, group_limit=1, group_mode="top2", renorm=True,
            factor=1.0, dtype="fp32", scores=False, finished=False):
    return {"name": name, "kind": "gating", "tokens": tokens, "experts": experts, "top_k": top_k, "score": score, "bias": bias,
            "groups": groups, "group_limit": group_limit, "group_mode": group_mode, "renorm": renorm, "factor": factor,
            "dtype": dtype, "scores": scores, "finished": finished}


def listed():
    return [
        # one user's next token: every launch and every host microsecond shows
        _norm("norm_1_token", 1, 4096),
        # a decode step of a serving batch, fp16, channels smoothed before they are quantised
        _norm("norm_decode_64_tokens", 64, 7168, dtype="fp16", gamma="fp32", smooth=True),
        # a ragged batch of fp32 rows off the 128 grid that had their residual added before
        _norm("norm_ragged_fp32", 301, 2880, dtype="fp32", residual=False, smooth=True),
        # a prompt
        _norm("norm_prefill", 8192, 7168),
        _logits("logits_1_token", 1, 4096, 128),
        # a decode step; the router's weights are kept in fp32, as routers are trained
        _logits("logits_decode_64_tokens", 64, 7168, 256, weight="fp32"),
        _logits("logits_ragged", 301, 2880, 60, dtype="fp16"),
        # a prompt over many experts, fp32 weights: the largest case
        _logits("logits_prefill", 8192, 7168, 256, weight="fp32"),
        # a long prompt over few experts: bound by the hidden states' bytes
        _logits("logits_few_experts", 16384, 4096, 8),
        # one token over 256 experts in eight groups, four of them kept
        _gating("gating_1_token", 1, 256, 8, groups=8, group_limit=4, factor=2.5),
        # a ragged batch with finished rows, softmax scores given back for their statistics, bf16 logits, no bias
        _gating("gating_ragged", 301, 160, 6, score="softmax", bias=False, groups=8, group_limit=3, group_mode="max", renorm=False,
                factor=16.0, dtype="bf16", scores=True, finished=True),
        # a long prompt
        _gating("gating_prefill", 16384, 256, 8, groups=8, group_limit=4, factor=2.5),
    ]


# The largest listed cases of each kind cost this much; drawn ones stay below.
_MAX_NORM = 8192 * 7168
_MAX_PRODUCT = 8192 * 7168 * 256
_MAX_HIDDEN_STATES = 16384 * 4096
_MAX_SCORES = 16384 * 256


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "logits", "gating"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    while True:
        tokens = _log_uniform(rng, 1, 16384)
        if rng.random() < 0.5:
            hidden = rng.choice([1024, 2880, 4096, 7168])
        else:
            hidden = _log_uniform(rng, 512, 8192)
            if rng.random() < 0.7:
                hidden = hidden // 32 * 32
        if kind == "norm":
            if tokens * hidden <= _MAX_NORM // (2 if dtype == "fp32" else 1):
                case = _norm("", tokens, hidden, dtype, rng.choice(["same", "same", "fp32"]), rng.random() < 0.75, rng.random() < 0.3,
                             rng.random() < 0.8)
                break
        elif kind == "logits":
            experts = rng.choice([8, 32, 64, 128, 256]) if rng.random() < 0.5 else _log_uniform(rng, 4, 512)
            if tokens * hidden * experts <= _MAX_PRODUCT and tokens * hidden <= _MAX_HIDDEN_STATES // (2 if dtype == "fp32" else 1):
                case = _logits("", tokens, hidden, experts, dtype, rng.choice(["same", "fp32"]))
                break
        else:
            experts = rng.choice([8, 16, 32, 60, 64, 72, 96, 128, 160, 192, 256, 384, 512])
            groups = rng.choice([g for g in (1, 1, 2, 4, 6, 8) if experts % g == 0 and experts // g >= 8 or g == 1])
            limit = rng.randint(1, groups)
            top_k = rng.choice([1, 2, 4, 6, 8, 8, 12])
            if tokens * experts <= _MAX_SCORES and top_k <= limit * (experts // groups):
                case = _gating("", tokens, experts, top_k, rng.choice(["softmax", "sigmoid", "sigmoid"]), rng.random() < 0.6, groups, limit,
                               rng.choice(["max", "top2"]), rng.random() < 0.7, rng.choice([1.0, 2.5]), dtype, rng.random() < 0.2,
                               rng.random() < 0.2)
                break
    del case["name"]
    return case


def prepare(case, seed):
    """Inputs, and the output buffers that a serving loop keeps."""
    device = torch.device("cuda")
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    tokens, dtype = case["tokens"], _DTYPES[case["dtype"]]
    state = {"case": case}

    def normal(*shape):
        return torch.randn(shape, device=device, generator=g)

    def empty(*shape, dtype):
        return torch.empty(shape, dtype=dtype, device=device)

    if case["kind"] == "norm":
        hidden = case["hidden"]
        # channels of unlike magnitude, as hidden states have
        state["x"] = (normal(tokens, hidden) * torch.exp(0.5 * normal(hidden))).to(dtype)
        state["residual"] = normal(tokens, hidden).to(dtype) if case["residual"] else None
        state["gamma"] = (1 + 0.2 * normal(hidden)).to(dtype if case["gamma"] == "same" else torch.float32)
        state["smooth"] = torch.exp(0.3 * normal(hidden)) if case["smooth"] else None
        state["out"] = (empty(tokens, hidden, dtype=torch.int8), empty(tokens, dtype=torch.float32),
                        empty(tokens, hidden, dtype=dtype) if case["rows"] else None,
                        empty(tokens, hidden, dtype=dtype) if case["residual"] else None)
        state["values"] = empty(tokens, hidden, dtype=torch.bfloat16)
    elif case["kind"] == "logits":
        hidden, experts = case["hidden"], case["experts"]
        state["x"] = normal(tokens, hidden).to(dtype)
        state["weight"] = (normal(experts, hidden) / math.sqrt(hidden)).to(dtype if case["weight"] == "same" else torch.float32)
        state["out"] = empty(tokens, experts, dtype=torch.float32)
    else:
        experts, top_k = case["experts"], case["top_k"]
        state["x"] = normal(tokens, experts).to(dtype)
        state["bias"] = 0.05 * normal(experts) if case["bias"] else None
        state["finished"] = (torch.rand((tokens,), device=device, generator=g) < 0.1) if case["finished"] else None
        state["out"] = (empty(tokens, top_k, dtype=dtype), empty(tokens, top_k, dtype=torch.int32),
                        empty(tokens, experts, dtype=torch.float32) if case["scores"] else None)
    return state


# ------------------------------------------------------------------------------------------------ passes
def _given(outputs):
    return {name: t for name, t in outputs.items() if t is not None}


def _norm_pass(case, s):
    if own:
        q, scale, rows, total = _operators().moe_add_rms_norm_quant(s["x"], s["gamma"], residual=s["residual"], smooth_scale=s["smooth"],
                                                                    epsilon=_EPSILON, out=s["out"])
    else:
        total = None
        x = s["x"]
        if s["residual"] is not None:
            x = total = (x.float() + s["residual"].float()).to(x.dtype)
        x = x.float()
        normed = x * torch.rsqrt(x.square().mean(dim=1, keepdim=True) + _EPSILON) * s["gamma"].float()
        rows = normed.to(s["x"].dtype) if case["rows"] else None
        v = normed if s["smooth"] is None else normed * s["smooth"]
        scale = v.abs().amax(dim=1) / 127.0
        q = torch.clamp(torch.round(v / scale[:, None]), -127, 127).to(torch.int8)
    # the int8 rows as the values they stand for
    torch.mul(q, scale[:, None], out=s["values"])
    return _given({"values": s["values"], "scale": scale, "rows": rows, "sum": total})


def _logits_pass(case, s):
    if own:
        return _operators().moe_router_logits(s["x"], s["weight"], out=s["out"])
    return s["x"].float() @ s["weight"].float().t()


def _gating_pass(case, s):
    experts, top_k, groups, limit = case["experts"], case["top_k"], case["groups"], case["group_limit"]
    if own:
        weight, idx, scores = _operators().moe_gating_top_k_grouped(
            s["x"], top_k, bias=s["bias"], finished=s["finished"], k_group=limit, group_count=groups,
            group_select_mode=1 if case["group_mode"] == "top2" else 0, score_type=1 if case["score"] == "sigmoid" else 0,
            renorm=1 if case["renorm"] else 0, routed_scaling_factor=case["factor"], eps=_RENORM_EPS, out=s["out"])
        return _given({"weight": weight, "idx": idx, "scores": scores})
    # in 64 bits: neighbouring scores decide which expert is taken
    x = s["x"].double()
    if case["score"] == "softmax":
        e = torch.exp(x - x.amax(dim=1, keepdim=True))
        p = e / e.sum(dim=1, keepdim=True)
    else:
        p = 1.0 / (1.0 + torch.exp(-x))
    t = p if s["bias"] is None else p + s["bias"].double()
    if limit < groups:
        by_group = t.view(-1, groups, experts // groups)
        best = by_group.amax(dim=2) if case["group_mode"] == "max" else by_group.topk(2, dim=2).values.sum(dim=2)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :limit]
        keep = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
        t = by_group.masked_fill(~keep[:, :, None], -math.inf).view(-1, experts)
    idx = torch.sort(t, dim=1, descending=True, stable=True).indices[:, :top_k]
    weight = torch.gather(p, 1, idx)
    if case["renorm"]:
        weight = weight / (weight.sum(dim=1, keepdim=True) + _RENORM_EPS)
    weight = (weight * case["factor"]).to(s["x"].dtype)
    idx = idx.int()
    if s["finished"] is not None:
        idx = idx.masked_fill(s["finished"][:, None], experts)
    return _given({"weight": weight, "idx": idx, "scores": p.float() if case["scores"] else None})


_PASSES = {"norm": _norm_pass, "logits": _logits_pass, "gating": _gating_pass}


def run(state):
    case = state["case"]
    return _PASSES[case["kind"]](case, state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def _size(name):
    return 4 if name == "fp32" else 2


def work(case):
    tokens, size = case["tokens"], _size(case["dtype"])
    if case["kind"] == "norm":
        hidden = case["hidden"]
        rows = 1 + case["residual"] * 2 + case["rows"]          # x, residual and sum, the normalised rows
        vectors = hidden * ((size if case["gamma"] == "same" else 4) + 4 * case["smooth"])
        return {"bytes": tokens * hidden * (size * rows + 1) + 4 * tokens + vectors, "flops": 8 * tokens * hidden}
    experts = case["experts"]
    if case["kind"] == "logits":
        hidden = case["hidden"]
        weights = experts * hidden * (size if case["weight"] == "same" else 4)
        return {"bytes": tokens * hidden * size + weights + 4 * tokens * experts, "flops": 2 * tokens * hidden * experts}
    out = tokens * case["top_k"] * (4 + size) + (4 * tokens * experts if case["scores"] else 0)
    return {"bytes": tokens * experts * size + 4 * experts * case["bias"] + tokens * case["finished"] + out,
            "flops": tokens * experts * (20 + case["top_k"])}


# ------------------------------------------------------------------------------------------------ the definitions, in 64 bits
def _exact_norm(case, s):
    x = s["x"]
    total = None
    if s["residual"] is not None:
        total = x.double() + s["residual"].double()
        x = total.to(x.dtype)               # the sum as it is kept is what is normalised
    x = x.double()
    mean_square = torch.linalg.vector_norm(x, dim=1) ** 2 / case["hidden"]
    normed = x / torch.sqrt(mean_square + _EPSILON)[:, None] * s["gamma"].double()
    v = normed * s["smooth"].double() if s["smooth"] is not None else normed
    scale = torch.maximum(v.max(dim=1).values, -v.min(dim=1).values) / 127.0
    values = torch.floor(v / scale[:, None] + 0.5) * scale[:, None]
    return _given({"values": values, "scale": scale, "rows": normed if case["rows"] else None, "sum": total})


def _exact_gating(case, s):
    import numpy as np
    x = s["x"].double().cpu().numpy()
    experts, groups = case["experts"], case["groups"]
    if case["score"] == "softmax":
        p = np.exp(x - np.logaddexp.reduce(x, axis=1)[:, None])
    else:
        p = np.exp(-np.logaddexp(0.0, -x))
    t = p.copy() if s["bias"] is None else p + s["bias"].double().cpu().numpy()
    by_group = np.sort(t.reshape(len(t), groups, -1), axis=2)
    best = by_group[:, :, -1] + (by_group[:, :, -2] if case["group_mode"] == "top2" else 0.0)
    out = np.argsort(-best, axis=1, kind="stable")[:, case["group_limit"]:]
    left = np.zeros((len(t), groups), dtype=bool)
    np.put_along_axis(left, out, True, axis=1)
    t[np.repeat(left, experts // groups, axis=1)] = -np.inf
    idx = np.argsort(-t, axis=1, kind="stable")[:, :case["top_k"]]
    weight = np.take_along_axis(p, idx, axis=1)
    if case["renorm"]:
        weight = weight / (weight.sum(axis=1)[:, None] + _RENORM_EPS)
    weight = weight * case["factor"]
    if s["finished"] is not None:
        idx = np.where(s["finished"].cpu().numpy()[:, None], experts, idx)
    return _given({"weight": weight, "idx": idx.astype(np.int32), "scores": p if case["scores"] else None})


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        return _exact_norm(case, s)
    if case["kind"] == "logits":
        return torch.matmul(s["weight"].double(), s["x"].double().t()).t().contiguous()
    return _exact_gating(case, s)
