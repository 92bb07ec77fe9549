"""What the operators for tuning a quantised model's router and norms are measured on, and the norms that close a block when it serves: the experts'
int8 weights stay as they are, the router, the gates, the norms and the residual scales around them learn.

A case is a dict of plain values.  ``kind`` names the operator:

``balance``      the balance loss of a batch's sequences with the experts' counts (``moe_balance_loss``).
``router_grad``  the gradient of the choice of experts with respect to the logits (``moe_gating_top_k_grouped_grad``): of the picked weights, of the
                 balance loss, or of both in one pass.
``close``        the norm behind a block with its gate and residual scales, the addition and the next block's norm (``moe_sandwich_norm``), as rows of
                 the stream's type, as int8 rows with scales, or both.
``close_grad``   its gradients (``moe_sandwich_norm_grad``): of the block's output, the residual, both norms' weights and the gate.

Shapes: those of ``synth.CONFIGS`` (hidden 1024, 4096 and 7168; 8, 128 and 256 experts) and generic ones off every grid.  Where ``own`` is false
``run`` computes the operators' plain forms in elementary torch operations.
"""
import math

import torch

own = False

_EPSILON = 1e-6     # of the norms
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


def _balance(name, tokens, experts, top_k, score="sigmoid", dtype="fp32", sequences=0, padded=False, finished=False):
    return {"name": name, "kind": "balance", "tokens": tokens, "experts": experts, "top_k": top_k, "score": score, "dtype": dtype,
            "sequences": sequences, "padded": padded, "finished": finished}


def _router_grad(name, tokens, experts, top_k, score="sigmoid", dtype="fp32", sequences=0, padded=False, finished=False, renorm=True, factor=1.0,
                 weights=True, balance=True):
    return {"name": name, "kind": "router_grad", "tokens": tokens, "experts": experts, "top_k": top_k, "score": score, "dtype": dtype,
            "sequences": sequences, "padded": padded, "finished": finished, "renorm": renorm, "factor": factor, "weights": weights,
            "balance": balance}


def _close(name, tokens, hidden, dtype="bf16", gamma="same", post=True, pre=True, gate="none", sigmoid=False, residual_scale=1.0,
           branch_scale=1.0, rows=True, quantise=False):
    return {"name": name, "kind": "close", "tokens": tokens, "hidden": hidden, "dtype": dtype, "gamma": gamma, "post": post, "pre": pre,
            "gate": gate, "sigmoid": sigmoid, "residual_scale": residual_scale, "branch_scale": branch_scale, "rows": rows, "quantise": quantise}


def _close_grad(name, tokens, hidden, dtype="bf16", gamma="same", post=True, pre=True, gate="none", sigmoid=False, residual_scale=1.0,
                branch_scale=1.0):
    return {"name": name, "kind": "close_grad", "tokens": tokens, "hidden": hidden, "dtype": dtype, "gamma": gamma, "post": post, "pre": pre,
            "gate": gate, "sigmoid": sigmoid, "residual_scale": residual_scale, "branch_scale": branch_scale}


def listed():
    return [
        # the load of the experts in one decode step of a serving batch
        _balance("balance_64_tokens", 64, 128, 8, score="softmax"),
        # packed sequences of unlike lengths with padding behind the last one and finished rows, bf16 logits
        _balance("balance_packed", 3011, 160, 6, score="softmax", dtype="bf16", sequences=7, padded=True, finished=True),
        # a training batch of sequences
        _balance("balance_batch", 16384, 256, 8, sequences=8),
        # a short sequence over few experts
        _router_grad("router_grad_256_tokens", 256, 8, 2, score="softmax"),
        # the packed batch's gradient, weights scaled and not renormalised
        _router_grad("router_grad_packed", 3011, 160, 6, score="softmax", dtype="bf16", sequences=7, padded=True, finished=True, renorm=False,
                     factor=16.0),
        # the training batch's: picked weights and balance in one pass
        _router_grad("router_grad_batch", 16384, 256, 8, sequences=8, factor=2.5),
        # one user's next token
        _close("close_1_token", 1, 4096),
        # a decode step of a serving batch: a gate per token (as a shared expert has), int8 rows for the next product
        _close("close_decode_64_tokens", 64, 7168, dtype="fp16", gamma="fp32", gate="row", sigmoid=True, rows=False, quantise=True),
        # a prompt, a gate per channel, residual and branch scaled
        _close("close_prefill", 8192, 7168, gate="channel", residual_scale=0.9, branch_scale=0.25),
        # a short batch's gradients, one norm only
        _close_grad("close_grad_64_rows", 64, 4096, pre=False, branch_scale=0.25),
        # a ragged batch of fp32 rows off the 128 grid, a gate for every value
        _close_grad("close_grad_ragged_fp32", 1203, 2880, dtype="fp32", gate="full", sigmoid=True),
        # a training batch: the largest case
        _close_grad("close_grad_batch", 8192, 7168, gate="channel", residual_scale=0.9, branch_scale=0.25),
    ]


# The largest listed cases of each kind cost this much; drawn ones stay below.
_MAX_SCORES = 16384 * 256
_MAX_ROWS = 8192 * 7168


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_router(rng, kind, tokens, dtype):
    while True:
        experts = rng.choice([8, 16, 32, 60, 64, 72, 96, 128, 160, 192, 256, 384, 512]) if rng.random() < 0.7 else _log_uniform(rng, 4, 600)
        top_k = rng.choice([1, 2, 4, 6, 8, 8, 12])
        sequences = 0 if rng.random() < 0.4 else _log_uniform(rng, 1, max(2, min(64, tokens)))
        if tokens * experts <= _MAX_SCORES and top_k <= experts:
            break
    score = rng.choice(["softmax", "sigmoid"])
    padded, finished = sequences > 0 and rng.random() < 0.4, rng.random() < 0.3
    if kind == "balance":
        return _balance("", tokens, experts, top_k, score, dtype, sequences, padded, finished)
    weights, balance = rng.choice([(True, True), (True, True), (True, False), (False, True)])
    renorm = top_k > 1 and rng.random() < 0.6       # a single renormalised weight is 1, and has no gradient
    return _router_grad("", tokens, experts, top_k, score, dtype, sequences, padded, finished, renorm, rng.choice([1.0, 2.5]), weights, balance)


def draw(rng):
    kind = rng.choice(["balance", "router_grad", "close", "close_grad"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind in ("balance", "router_grad"):
        case = _draw_router(rng, kind, _log_uniform(rng, 1, 16384), "fp32" if rng.random() < 0.6 else dtype)
    else:
        while True:
            tokens = _log_uniform(rng, 1, 16384)
            if rng.random() < 0.5:
                hidden = rng.choice([1024, 2880, 4096, 7168])
            else:
                hidden = _log_uniform(rng, 256, 12000)
                if rng.random() < 0.7:
                    hidden = hidden // 32 * 32
            if tokens * hidden <= _MAX_ROWS // (2 if dtype == "fp32" else 1):
                break
        post = rng.random() < 0.8
        pre = not post or rng.random() < 0.7
        gate = rng.choice(["none", "none", "channel", "row", "full"])
        shared = (tokens, hidden, dtype, rng.choice(["same", "same", "fp32"]), post, pre, gate, rng.random() < 0.5,
                  rng.choice([1.0, 1.0, 0.9]), rng.choice([1.0, 0.25]))
        if kind == "close":
            quantise = pre and rng.random() < 0.4
            case = _close("", *shared, rows=not quantise or rng.random() < 0.5, quantise=quantise)
        else:
            case = _close_grad("", *shared)
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------ inputs
def _prepare_router(case, state, normal, rand, empty):
    device = torch.device("cuda")
    tokens, experts, top_k, dtype = case["tokens"], case["experts"], case["top_k"], _DTYPES[case["dtype"]]
    popular = normal(experts)       # experts of unlike popularity, as an untrained router has
    state["x"] = (normal(tokens, experts) + 0.5 * popular).to(dtype)
    idx = torch.topk(state["x"].float() + 0.1 * normal(experts), top_k, dim=1).indices.int()
    if case["finished"]:
        idx = torch.where(rand(tokens, 1) < 0.1, torch.full_like(idx, experts), idx)
    state["idx"] = idx
    sequences = case["sequences"]
    state["offsets"] = None
    if sequences > 0:
        end = tokens - tokens // 16 if case["padded"] else tokens
        cuts = torch.sort((rand(sequences - 1) * (end + 1)).int()).values
        state["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int32, device=device), cuts, torch.full((1,), end, dtype=torch.int32, device=device)]).int()
    sequences = max(sequences, 1)
    if case["kind"] == "balance":
        state["out"] = (empty(sequences, dtype=torch.float32), empty(sequences, experts, dtype=torch.int32), empty(sequences, dtype=torch.int32),
                        empty(sequences, experts, dtype=torch.float32))
        return
    state["y_grad"] = 0.1 * normal(tokens, top_k) if case["weights"] else None
    state["loss_grad"] = state["counts"] = state["rows"] = None
    if case["balance"]:
        member, live = _sequence_of_rows(case, state)
        state["counts"], state["rows"] = _counts(case, state, member, live)
        state["loss_grad"] = 0.01 * (1 + 0.1 * rand(sequences))
    state["out"] = empty(tokens, experts, dtype=dtype)


def _prepare_close(case, state, normal, rand, empty):
    tokens, hidden, dtype = case["tokens"], case["hidden"], _DTYPES[case["dtype"]]
    weights = dtype if case["gamma"] == "same" else torch.float32
    # channels of unlike magnitude, as hidden states have
    state["x"] = (normal(tokens, hidden) * torch.exp(0.5 * normal(hidden))).to(dtype)
    state["post"] = (1 + 0.2 * normal(hidden)).to(weights) if case["post"] else None
    state["pre"] = (1 + 0.2 * normal(hidden)).to(weights) if case["pre"] else None
    state["gate"] = {"none": lambda: None, "channel": lambda: (0.5 + 0.2 * normal(hidden)).to(weights),
                     "row": lambda: normal(tokens, 1), "full": lambda: normal(tokens, hidden).to(dtype)}[case["gate"]]()
    state["residual"] = normal(tokens, hidden).to(dtype)
    if case["kind"] == "close":
        state["out"] = (empty(tokens, hidden, dtype=dtype), empty(tokens, hidden, dtype=dtype) if case["pre"] and case["rows"] else None,
                        empty(tokens, hidden, dtype=torch.int8) if case["quantise"] else None,
                        empty(tokens, dtype=torch.float32) if case["quantise"] else None, None, None)
        state["values"] = empty(tokens, hidden, dtype=torch.bfloat16) if case["quantise"] else None
        return
    # what the forward pass has left: the sum and both norms' factors
    state["sum"], _, state["post_rstd"], state["pre_rstd"] = _close_rows(case, state)
    del state["residual"]
    state["sum_grad"] = normal(tokens, hidden).to(dtype)
    state["norm_grad"] = normal(tokens, hidden).to(dtype) if case["pre"] else None
    gate = {"none": lambda: None, "channel": lambda: empty(hidden, dtype=torch.float32), "row": lambda: empty(tokens, 1, dtype=torch.float32),
            "full": lambda: empty(tokens, hidden, dtype=dtype)}[case["gate"]]()
    state["out"] = (empty(tokens, hidden, dtype=dtype), empty(tokens, hidden, dtype=dtype),
                    empty(hidden, dtype=torch.float32) if case["post"] else None, gate,
                    empty(hidden, dtype=torch.float32) if case["pre"] else None)


def prepare(case, seed):
    """Inputs, and the output buffers that a training or serving loop keeps."""
    device = torch.device("cuda")
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    state = {"case": case}
    make = _prepare_router if case["kind"] in ("balance", "router_grad") else _prepare_close
    make(case, state, lambda *shape: torch.randn(shape, device=device, generator=g), lambda *shape: torch.rand(shape, device=device, generator=g),
         lambda *shape, dtype: torch.empty(shape, dtype=dtype, device=device))
    return state


# ------------------------------------------------------------------------------------------------ passes
def _given(outputs):
    return {name: t for name, t in outputs.items() if t is not None}


def _sequence_of_rows(case, s):
    """Which sequence each row is in, as a matrix of ones and zeros [sequences, tokens], and which rows count at all."""
    live = (s["idx"][:, 0] >= 0) & (s["idx"][:, 0] < case["experts"])
    row = torch.arange(case["tokens"], device=live.device)
    if s["offsets"] is None:
        member = live[None, :]
    else:
        member = (row >= s["offsets"][:-1, None]) & (row < s["offsets"][1:, None]) & live
    return member.float(), live


def _counts(case, s, member, live):
    experts = case["experts"]
    picked = torch.zeros((case["tokens"], experts + 1), device=live.device).scatter_add_(1, s["idx"].long(), torch.ones_like(s["idx"], dtype=torch.float32))
    return (member @ picked[:, :experts]).round().int(), member.sum(1).round().int()


def _scores(case, x):
    """Softmax scores, or sigmoid scores as shares of their sum."""
    if case["score"] == "softmax":
        e = torch.exp(x - x.amax(dim=1, keepdim=True))
    else:
        e = 1.0 / (1.0 + torch.exp(-x))
    return e / e.sum(dim=1, keepdim=True)


def _balance_pass(case, s):
    if own:
        loss, counts, rows, prob = _operators().moe_balance_loss(s["x"], s["idx"], seq_offsets=s["offsets"],
                                                                 score_type=1 if case["score"] == "sigmoid" else 0, out=s["out"])
        return {"loss": loss, "counts": counts, "rows": rows, "prob": prob}
    member, live = _sequence_of_rows(case, s)
    counts, rows = _counts(case, s, member, live)
    n = rows.clamp(min=1).float()
    prob = (member @ _scores(case, s["x"].float())) / n[:, None]
    loss = (counts.float() * prob).sum(1) * (case["experts"] / case["top_k"]) / n
    return {"loss": loss, "counts": counts, "rows": rows, "prob": prob}


def _router_grad_pass(case, s):
    experts, top_k = case["experts"], case["top_k"]
    if own:
        return _operators().moe_gating_top_k_grouped_grad(
            s["x"], s["idx"], y_grad=s["y_grad"], loss_grad=s["loss_grad"], counts=s["counts"], rows=s["rows"],
            seq_offsets=None if s["loss_grad"] is None else s["offsets"],      # the sequences are the loss's
            score_type=1 if case["score"] == "sigmoid" else 0, renorm=1 if case["renorm"] else 0, routed_scaling_factor=case["factor"],
            eps=_RENORM_EPS, out=s["out"])
    x = s["x"].float()
    share = _scores(case, x)
    live = (s["idx"][:, :1] >= 0) & (s["idx"][:, :1] < experts)
    grad = torch.zeros_like(x)
    if s["y_grad"] is not None:
        p = share if case["score"] == "softmax" else 1.0 / (1.0 + torch.exp(-x))
        at = s["idx"].long().clamp(0, experts - 1)
        y_grad = torch.where(live, s["y_grad"].float(), 0.0) * case["factor"]
        if case["renorm"]:
            picked = torch.gather(p, 1, at)
            total = picked.sum(dim=1, keepdim=True) + _RENORM_EPS
            y_grad = (y_grad - (y_grad * picked / total).sum(dim=1, keepdim=True)) / total
        p_grad = torch.zeros_like(x).scatter_add_(1, at, y_grad)
        if case["score"] == "softmax":
            grad = p * (p_grad - (p_grad * p).sum(dim=1, keepdim=True))
        else:
            grad = p_grad * p * (1.0 / (1.0 + torch.exp(x)))
    if s["loss_grad"] is not None:
        member, _ = _sequence_of_rows(case, s)
        n = s["rows"].clamp(min=1).float()
        per_expert = s["counts"].float() * (s["loss_grad"] * (experts / top_k) / (n * n))[:, None]
        share_grad = member.t() @ per_expert
        balance = share * (share_grad - (share_grad * share).sum(dim=1, keepdim=True))
        if case["score"] == "sigmoid":
            balance = balance / (1.0 + torch.exp(x))
        grad = grad + balance
    return torch.where(live, grad, 0.0).to(s["x"].dtype)


def _gate_values(case, gate):
    g = gate.float()
    return 1.0 / (1.0 + torch.exp(-g)) if case["sigmoid"] else g


def _close_rows(case, s):
    """(sum, next block's rows in fp32, both norms' factors)"""
    v = s["x"].float()
    post_rstd = pre_rstd = normed = None
    if s["post"] is not None:
        post_rstd = torch.rsqrt(v.square().mean(dim=1) + _EPSILON)
        v = v * post_rstd[:, None] * s["post"].float()
    if s["gate"] is not None:
        v = v * _gate_values(case, s["gate"])
    total = (case["residual_scale"] * s["residual"].float() + case["branch_scale"] * v).to(s["x"].dtype)
    if s["pre"] is not None:
        t = total.float()
        pre_rstd = torch.rsqrt(t.square().mean(dim=1) + _EPSILON)
        normed = t * pre_rstd[:, None] * s["pre"].float()
    return total, normed, post_rstd, pre_rstd


def _close_pass(case, s):
    if own:
        total, rows, q, scale, _, _ = _operators().moe_sandwich_norm(
            s["x"], s["residual"], post_gamma=s["post"], gate=s["gate"], pre_gamma=s["pre"], gate_type=1 if case["sigmoid"] else 0,
            residual_scale=case["residual_scale"], branch_scale=case["branch_scale"], epsilon=_EPSILON, out=s["out"])
    else:
        total, normed, _, _ = _close_rows(case, s)
        rows = normed.to(total.dtype) if case["pre"] and case["rows"] else None
        if case["quantise"]:
            scale = normed.abs().amax(dim=1) / 127.0
            q = torch.clamp(torch.round(normed / scale[:, None]), -127, 127).to(torch.int8)
    if not case["quantise"]:
        return _given({"sum": total, "rows": rows})
    # the int8 rows as the values they stand for
    torch.mul(q, scale[:, None], out=s["values"])
    return _given({"sum": total, "rows": rows, "values": s["values"], "scale": scale})


def _close_grad_pass(case, s):
    if own:
        x_grad, residual_grad, post_grad, gate_grad, pre_grad = _operators().moe_sandwich_norm_grad(
            s["x"], s["sum"], sum_grad=s["sum_grad"], norm_grad=s["norm_grad"], post_gamma=s["post"], gate=s["gate"], pre_gamma=s["pre"],
            post_rstd=s["post_rstd"], pre_rstd=s["pre_rstd"], gate_type=1 if case["sigmoid"] else 0, residual_scale=case["residual_scale"],
            branch_scale=case["branch_scale"], out=s["out"])
        return _given({"x": x_grad, "residual": residual_grad, "post": post_grad, "gate": gate_grad, "pre": pre_grad})
    dtype = s["x"].dtype
    total = s["sum_grad"].float()
    post_grad = gate_grad = pre_grad = None
    if s["pre"] is not None:
        normed = s["sum"].float() * s["pre_rstd"][:, None]
        d = s["norm_grad"].float()
        pre_grad = (d * normed).sum(dim=0)
        d = d * s["pre"].float()
        total = total + (d - normed * (d * normed).mean(dim=1, keepdim=True)) * s["pre_rstd"][:, None]
    residual_grad = (case["residual_scale"] * total).to(dtype)
    v = case["branch_scale"] * total
    x = s["x"].float()
    normed = x if s["post"] is None else x * s["post_rstd"][:, None]
    u = normed if s["post"] is None else normed * s["post"].float()
    if s["gate"] is not None:
        g = _gate_values(case, s["gate"])
        gate_grad = v * u * (g * (1.0 - g)) if case["sigmoid"] else v * u
        v = v * g
        if case["gate"] == "channel":
            gate_grad = gate_grad.sum(dim=0)
        elif case["gate"] == "row":
            gate_grad = gate_grad.sum(dim=1, keepdim=True)
        else:
            gate_grad = gate_grad.to(dtype)
    if s["post"] is not None:
        post_grad = (v * normed).sum(dim=0)
        v = v * s["post"].float()
        v = (v - normed * (v * normed).mean(dim=1, keepdim=True)) * s["post_rstd"][:, None]
    return _given({"x": v.to(dtype), "residual": residual_grad, "post": post_grad, "gate": gate_grad, "pre": pre_grad})


_PASSES = {"balance": _balance_pass, "router_grad": _router_grad_pass, "close": _close_pass, "close_grad": _close_grad_pass}


def run(state):
    case = state["case"]
    return _PASSES[case["kind"]](case, state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def _size(name):
    return 4 if name == "fp32" else 2


def work(case):
    tokens, size = case["tokens"], _size(case["dtype"])
    if case["kind"] in ("balance", "router_grad"):
        experts, top_k, sequences = case["experts"], case["top_k"], max(case["sequences"], 1)
        tables = sequences * (4 * experts + 8)      # counts, rows, loss or its gradient
        if case["kind"] == "balance":
            return {"bytes": tokens * (experts * size + 4 * top_k) + tables + 4 * sequences * experts, "flops": tokens * (experts * 12 + top_k)}
        return {"bytes": tokens * (2 * experts * size + 4 * top_k + 4 * top_k * case["weights"]) + tables * case["balance"],
                "flops": tokens * (experts * 20 + 8 * top_k)}
    hidden = case["hidden"]
    weight = size if case["gamma"] == "same" else 4
    vectors = hidden * weight * (case["post"] + case["pre"] + (case["gate"] == "channel"))
    gate = {"none": 0, "channel": 0, "row": 4 * tokens, "full": tokens * hidden * size}[case["gate"]]
    if case["kind"] == "close":
        rows = 3 + (case["pre"] and case["rows"])       # x, residual and sum, the next block's rows
        return {"bytes": tokens * hidden * (size * rows + case["quantise"]) + 4 * tokens * case["quantise"] + vectors + gate,
                "flops": 16 * tokens * hidden}
    needs_x = case["post"] or case["gate"] != "none"    # without either the block's output does not show in its gradients
    rows = 3 + needs_x + 2 * case["pre"]                # the sum's gradient, both rows' gradients, x; the sum and the rows' gradient
    sums = 4 * hidden * (case["post"] + case["pre"] + (case["gate"] == "channel"))
    return {"bytes": tokens * (hidden * size * rows + 4 * (case["post"] + case["pre"])) + vectors + 2 * gate + sums, "flops": 30 * tokens * hidden}


# ------------------------------------------------------------------------------------------------ the definitions, in 64 bits
def _bounds(case, s):
    if s["offsets"] is None:
        return [(0, case["tokens"])]
    at = s["offsets"].tolist()
    return list(zip(at[:-1], at[1:]))


def _exact_shares(case, x):
    logs = torch.log_softmax(x, dim=1) if case["score"] == "softmax" else torch.nn.functional.logsigmoid(x)
    return torch.exp(logs - torch.logsumexp(logs, dim=1, keepdim=True))


def _exact_balance(case, s):
    experts, top_k = case["experts"], case["top_k"]
    shares, idx = _exact_shares(case, s["x"].double()), s["idx"].long()
    live = idx[:, 0] < experts
    loss, counts, rows, prob = [], [], [], []
    for lo, hi in _bounds(case, s):
        kept = live[lo:hi].nonzero()[:, 0] + lo
        n = len(kept)
        count = torch.bincount(idx[kept].reshape(-1), minlength=experts)
        mean = shares[kept].sum(0) / max(n, 1)
        loss.append(torch.dot(count.double() * (experts / (top_k * max(n, 1))), mean))
        counts.append(count)
        rows.append(n)
        prob.append(mean)
    return {"loss": torch.stack(loss), "counts": torch.stack(counts).int(), "rows": torch.tensor(rows, dtype=torch.int32), "prob": torch.stack(prob)}


def _exact_router_grad(case, s):
    """By differentiation of the definition."""
    experts, top_k = case["experts"], case["top_k"]
    idx = s["idx"].long()
    live = idx[:, 0] < experts
    x = s["x"].double().requires_grad_(True)
    value = x.sum() * 0.0
    if s["y_grad"] is not None:
        p = torch.softmax(x, dim=1) if case["score"] == "softmax" else torch.sigmoid(x)
        y = torch.gather(p[live], 1, idx[live])
        if case["renorm"]:
            y = y / (y.sum(1, keepdim=True) + _RENORM_EPS)
        value = value + (y * s["y_grad"].double()[live] * case["factor"]).sum()
    if s["loss_grad"] is not None:
        shares = _exact_shares(case, x)
        for i, (lo, hi) in enumerate(_bounds(case, s)):
            kept = live[lo:hi].nonzero()[:, 0] + lo
            if len(kept):
                load = s["counts"][i].double() * (experts / (top_k * len(kept)))
                value = value + s["loss_grad"][i].double() * (load * shares[kept].mean(0)).sum()
    return torch.autograd.grad(value, x)[0]


def _exact_close_parts(case, s):
    x = s["x"].double()
    u = x
    if s["post"] is not None:
        u = x / torch.sqrt(torch.linalg.vector_norm(x, dim=1) ** 2 / case["hidden"] + _EPSILON)[:, None] * s["post"].double()
    g = None
    if s["gate"] is not None:
        g = torch.sigmoid(s["gate"].double()) if case["sigmoid"] else s["gate"].double()
    return u, g


def _exact_close(case, s):
    u, g = _exact_close_parts(case, s)
    total = case["branch_scale"] * (u if g is None else g * u) + case["residual_scale"] * s["residual"].double()
    if s["pre"] is None:
        return {"sum": total}
    kept = total.to(s["x"].dtype).double()      # the sum as it is kept is what is normalised
    normed = kept / torch.sqrt(torch.linalg.vector_norm(kept, dim=1) ** 2 / case["hidden"] + _EPSILON)[:, None] * s["pre"].double()
    out = {"sum": total, "rows": normed if case["rows"] else None}
    if case["quantise"]:
        out["scale"] = torch.maximum(normed.max(dim=1).values, -normed.min(dim=1).values) / 127.0
        out["values"] = torch.floor(normed / out["scale"][:, None] + 0.5) * out["scale"][:, None]
    return _given({name: out.get(name) for name in ("sum", "rows", "values", "scale")})


def _exact_close_grad(case, s):
    hidden = case["hidden"]
    total = s["sum_grad"].double()
    post_grad = gate_grad = pre_grad = None
    if s["pre"] is not None:
        kept, r = s["sum"].double(), s["pre_rstd"].double()[:, None]
        d = s["norm_grad"].double()
        pre_grad = torch.einsum("th,th,t->h", d, kept, r[:, 0])
        d = d * s["pre"].double()
        total = total + d * r - kept * (r ** 3 / hidden * (d * kept).sum(1, keepdim=True))
    x = s["x"].double()
    r = s["post_rstd"].double()[:, None] if s["post"] is not None else 1.0
    u = x * r * s["post"].double() if s["post"] is not None else x
    v = case["branch_scale"] * total
    if s["gate"] is not None:
        raw = s["gate"].double()
        g = torch.sigmoid(raw) if case["sigmoid"] else raw
        gate_grad = v * u * (torch.sigmoid(raw) * torch.sigmoid(-raw) if case["sigmoid"] else 1.0)
        gate_grad = {"channel": lambda t: t.sum(0), "row": lambda t: t.sum(1, keepdim=True), "full": lambda t: t}[case["gate"]](gate_grad)
        v = v * g
    if s["post"] is not None:
        post_grad = (v * x * r).sum(0)
        v = v * s["post"].double()
        v = v * r - x * (r ** 3 / hidden * (v * x).sum(1, keepdim=True))
    return _given({"x": v, "residual": case["residual_scale"] * total, "post": post_grad, "gate": gate_grad, "pre": pre_grad})


def exact(case, seed):
    s = prepare(case, seed)
    return {"balance": _exact_balance, "router_grad": _exact_router_grad, "close": _exact_close, "close_grad": _exact_close_grad}[case["kind"]](case, s)
