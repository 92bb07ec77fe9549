"""The operators for tuning the router and the norms, on the GPU against their formulas in 64 bits on the CPU.

Tolerances, with u = 2^-24 (half an ulp of fp32 in relative terms) and half(t) = finfo(t).eps / 2 for the rounding of an output:
scores    an exponential is off by 4 u, and by |x - top| u of its argument's subtraction; the row's sum by (E / 64 + 10) u (a lane's terms and a tree), reciprocal,
          product and sigmoid's division by 6 u: a score's relative error is at most (spread + E / 64 + 20) u.  Below 2^-126 a score may be zero.
balance   a lane adds up to 512 scores, 8 waves and up to 6 steps of a wave follow, the rest is in 64 bits: (min(n, 512) + 14) u more.  All terms are positive.
gradient  products and sums of scores and of given numbers: each of the up to six factors and sums in a term has a score's error, taken of the terms' magnitudes.
norms     a row's sum of H terms: (H / 64 + 20) u of the terms' magnitudes (a lane's share, a tree of six, up to eight waves and what each term has); a
          gradient has two of them in a row, and 20 products.  Column sums: up to 512 terms in a lane, the rest in 64 bits.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def _on(dev, *ts):
    return [None if t is None else t.to(dev) for t in ts]


def _within(got, want, bound):
    """|got - want| <= bound element by element; where the definition has NaN, so has the operator."""
    got, want = got.cpu().double(), want.double()
    assert got.shape == want.shape
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    bad = ((got - want).abs() > bound) & ~nan
    assert not bad.any(), (int(bad.sum()), float((got - want).abs()[bad].max()), float(bound.expand_as(want)[bad].max() if torch.is_tensor(bound) else bound))


# ------------------------------------------------------------------------------------------------ the router's definitions in 64 bits
def _router_inputs(T, E, k, dtype, seed, finished=0.0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    lead = T if isinstance(T, tuple) else (T,)
    x = (spread * torch.randn(lead + (E,), generator=g)).to(dtype)
    if k <= E:
        idx = torch.topk(x.float() + 0.5 * torch.randn(E, generator=g), k, dim=-1).indices.int()
    else:
        idx = torch.randint(0, E, lead + (k,), generator=g, dtype=torch.int32)
    if finished:
        idx = torch.where(torch.rand(lead + (1,), generator=g) < finished, torch.full_like(idx, E), idx)
    return x, idx


def _offsets(T, S, seed, begin=0, end=None, dtype=torch.int32):
    g = torch.Generator().manual_seed(seed)
    end = T if end is None else end
    cuts = torch.sort(torch.randint(begin, end + 1, (S - 1,), generator=g)).values
    return torch.cat([torch.tensor([begin]), cuts, torch.tensor([end])]).to(dtype)


def _shares(x, score):
    logs = torch.log_softmax(x.double(), -1) if score == 0 else torch.nn.functional.logsigmoid(x.double())
    top = logs.amax(-1, keepdim=True)
    nothing = top == -math.inf
    e = torch.exp(logs - torch.where(nothing, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    r = e / torch.where(total == 0, torch.ones_like(total), total)
    rowless = (x == -math.inf).all(-1, keepdim=True)            # log_softmax of nothing is NaN
    return torch.where(rowless, torch.zeros_like(r), r)


def _score_error(x):
    finite = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).double()
    spread = float(finite.abs().max()) * 2 if finite.numel() else 0.0
    return (min(spread, 90.0) + x.shape[-1] / 64 + 20) * U


def _ranges(offsets, T):
    return [(0, T)] if offsets is None else list(zip(offsets.tolist()[:-1], offsets.tolist()[1:]))


def _balance_want(x, idx, offsets, score):
    E, k = x.shape[-1], idx.shape[-1]
    x, idx = x.reshape(-1, E), idx.reshape(-1, k).long()
    r = _shares(x, score)
    live = (idx[:, 0] >= 0) & (idx[:, 0] < E)
    counts, rows, prob = [], [], []
    for lo, hi in _ranges(offsets, len(x)):
        at = torch.arange(lo, max(lo, hi))[live[lo:max(lo, hi)]]
        ids = idx[at].reshape(-1)
        counts.append(torch.bincount(ids[(ids >= 0) & (ids < E)], minlength=E))
        rows.append(len(at))
        prob.append(r[at].sum(0) / max(len(at), 1))
    counts, rows, prob = torch.stack(counts), torch.tensor(rows), torch.stack(prob)
    loss = (counts * prob).sum(1) * E / (k * rows.clamp(min=1))
    return loss, counts.int(), rows.int(), prob


def _check_balance(x, idx, offsets, score, got):
    loss, counts, rows, prob = _balance_want(x, idx, offsets, score)
    assert torch.equal(got[1].cpu(), counts) and torch.equal(got[2].cpu(), rows)
    tol = _score_error(x) + (min(float(rows.max()), 512) + 14 + 3) * U
    if got[3] is not None:
        _within(got[3], prob, tol * prob + 2.0 ** -126)
    _within(got[0], loss, tol * loss + 1e-30)


BALANCE_EXPERTS = [1, 3, 4, 8, 9, 16, 33, 64, 100, 128, 160, 256, 300, 512, 777, 1024, 1500, 2048]


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("E", BALANCE_EXPERTS)
def test_balance_experts(aclnn, dev, E, score):
    for T, k, name, S in [(1, 1, "f32", None), (7, min(E, 8), "bf16", None), (70, min(E, 6), "f16", 3), (2051, min(E, 8), "f32", None), (1025, 12, "bf16", 9)]:
        x, idx = _router_inputs(T, E, k, TORCH[name], E + T, finished=0.2 if T > 7 else 0.0)
        offsets = None if S is None else _offsets(T, S, T, begin=T // 9, end=T - T // 7)
        got = aclnn.moe_balance_loss(*_on(dev, x, idx, offsets), score_type=score)
        _check_balance(x, idx, offsets, score, got)


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("T,E,k,S", [(16384, 256, 8, None), (16384, 256, 8, 8), (40000, 8, 2, None), (9000, 160, 6, 700), (300, 64, 8, 300), (3000, 2048, 64, 2),
                                     (100, 16, 2, 5000), (1, 256, 8, 4)])
def test_balance_batches(aclnn, dev, T, E, k, S, score):
    """Chunks of many sequences, sequences of many chunks, more sequences than rows."""
    x, idx = _router_inputs(T, E, k, torch.float32, T + E, finished=0.1)
    for kind in (torch.int32, torch.int64):
        offsets = None if S is None else _offsets(T, S, T + E, dtype=kind)
        _check_balance(x, idx, offsets, score, aclnn.moe_balance_loss(*_on(dev, x, idx, offsets), score_type=score))


def test_balance_of_even_choices_is_one(aclnn, dev):
    """Equal logits, every expert picked equally often."""
    T, E, k = 1024, 64, 4
    idx = (torch.arange(T * k).reshape(T, k) % E).int().to(dev)
    for score in (0, 1):
        loss, counts, rows, prob = aclnn.moe_balance_loss(torch.full((T, E), 0.5, device=dev), idx, score_type=score)
        assert abs(float(loss) - 1) <= 8 * U and torch.all(counts == T * k // E) and int(rows) == T
        assert torch.all((prob - 1 / E).abs() <= (E / 64 + 20) * U / E)


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("E", [6, 128, 500])
def test_balance_rows_of_unusual_values(aclnn, dev, E, score):
    """Masked experts, rows with nothing left, scores that fp32 loses, NaN and infinities; each in a sequence of its own."""
    T, k = 8, 2
    x, idx = _router_inputs(T, E, k, torch.float32, E, spread=3.0)
    x[0, 1:] = -math.inf                                    # one expert left
    x[1] = -math.inf                                        # none
    x[2] -= 95.0                                            # sigmoid scores below 2^-126: in the proportions of e^x
    x[3, E // 2] = math.nan
    x[4] = torch.finfo(torch.float32).min                   # masked by the type's lowest value throughout
    x[5, 2:] = torch.finfo(torch.float32).min
    x[6, 0] = 80.0
    offsets = torch.arange(T + 1, dtype=torch.int32)
    got = aclnn.moe_balance_loss(*_on(dev, x, idx, offsets), score_type=score)
    want = _balance_want(x, idx, offsets, score)
    if score == 1:
        # every score of row 4 is exactly 0, its logits equal: the definition divides 0 by 0; the operator takes the limit, equal shares
        want[3][4] = 1 / E
        want[0][4] = (want[1][4] * want[3][4]).sum() * E / k
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])
    tol = (95 * 2 + E / 64 + 40) * U
    _within(got[3], want[3], tol * want[3] + 2.0 ** -126)
    _within(got[0], want[0], tol * want[0] + E * 2.0 ** -126)
    if score == 0:
        x[7, 1] = math.inf
        assert torch.isnan(aclnn.moe_balance_loss(*_on(dev, x, idx, offsets))[3][7]).all()


def test_balance_ids_that_are_no_experts(aclnn, dev):
    """The first id says whether a row counts; the others count or not by themselves; one twice counts twice."""
    x, _ = _router_inputs(6, 8, 3, torch.float32, 1)
    idx = torch.tensor([[8, 1, 2], [-1, 3, 3], [0, 8, 2], [5, 5, 5], [1, -7, 2147483647], [-2147483648, 0, 1]], dtype=torch.int32)
    got = aclnn.moe_balance_loss(*_on(dev, x, idx))
    _check_balance(x, idx, None, 0, got)
    assert got[1].cpu().tolist() == [[1, 1, 1, 0, 0, 3, 0, 0]] and int(got[2]) == 3


def test_balance_offsets_outside_the_rows(aclnn, dev):
    """Held to the rows; falling ones give unspecified values and leave what is around the outputs alone."""
    x, idx = _router_inputs(500, 96, 4, torch.float32, 2)
    for kind in (torch.int32, torch.int64):
        wild = torch.tensor([-5, 100, 100, 700, 900], dtype=kind)
        held = torch.tensor([0, 100, 100, 500, 500], dtype=kind)
        got = aclnn.moe_balance_loss(*_on(dev, x, idx, wild))
        _check_balance(x, idx, held, 0, got)
        S = 4
        around = [torch.full((S * n + 8,), 7, dtype=t, device=dev) for n, t in [(1, torch.float32), (96, torch.int32), (1, torch.int32), (96, torch.float32)]]
        out = tuple(t[4:-4].view((S, 96) if n == 96 else (S,)) for t, n in zip(around, (1, 96, 1, 96)))
        aclnn.moe_balance_loss(*_on(dev, x, idx, torch.tensor([400, 30, 499, -1, 250], dtype=kind)), out=out)
        for t in around:
            assert torch.all(t[:4] == 7) and torch.all(t[-4:] == 7)


def test_balance_empty_batches(aclnn, dev):
    for shape, offsets in [((0, 64), None), ((0, 64), torch.zeros(4, dtype=torch.int32)), ((3, 0, 64), None)]:
        idx = torch.empty(shape[:-1] + (2,), dtype=torch.int32, device=dev)
        S = 1 if offsets is None else 3
        out = (torch.full((S,), 5.0, device=dev), torch.full((S, 64), 5, dtype=torch.int32, device=dev), torch.full((S,), 5, dtype=torch.int32, device=dev),
               torch.full((S, 64), 5.0, device=dev))
        aclnn.moe_balance_loss(torch.empty(shape, device=dev), idx, seq_offsets=None if offsets is None else offsets.to(dev), out=out)
        for t in out:
            assert not t.any()
    x, idx = _router_inputs(70, 64, 2, torch.float32, 1)
    idx[:] = 64                                                                      # every row finished
    _check_balance(x, idx, None, 0, aclnn.moe_balance_loss(*_on(dev, x, idx)))


def test_balance_strides_and_outputs(aclnn, dev):
    x, idx = _router_inputs((3, 50), 33, 3, torch.bfloat16, 4)
    want = aclnn.moe_balance_loss(*_on(dev, x, idx))
    _check_balance(x, idx, None, 0, want)
    wide = torch.zeros((3, 50, 70), dtype=torch.bfloat16, device=dev)
    wide[..., 5:38] = x.to(dev)
    ids = torch.zeros((3, 50, 6), dtype=torch.int32, device=dev)
    ids[..., ::2] = idx.to(dev)
    flat = torch.zeros(150 * 33 + 1, dtype=torch.bfloat16, device=dev)               # rows that begin on any element
    flat[1:] = x.to(dev).reshape(-1)
    for a, b in [(wide[..., 5:38], ids[..., ::2]), (flat[1:].view(3, 50, 33), idx.to(dev))]:
        for p, q in zip(aclnn.moe_balance_loss(a, b), want):
            assert torch.equal(p, q)
    none = aclnn.moe_balance_loss(*_on(dev, x, idx), output_prob=False)
    assert none[3] is None and torch.equal(none[0], want[0])


# ------------------------------------------------------------------------------------------------ gradient of the choice
def _grad_want(x, idx, dy, dl, counts, rows, offsets, score, renorm, factor, eps):
    """(gradient, magnitude of its terms) in 64 bits."""
    shape, E, k = x.shape, x.shape[-1], idx.shape[-1]
    x, idx = x.reshape(-1, E).double(), idx.reshape(-1, k).long()
    r = _shares(x, score)
    p, rest = (r, None) if score == 0 else (torch.sigmoid(x), torch.sigmoid(-x))
    grad, mass = torch.zeros_like(x), torch.zeros_like(x)
    valid = (idx >= 0) & (idx < E)
    at = idx.clamp(0, E - 1)
    if dy is not None:
        y = dy.reshape(-1, k).double() * valid
        picked = torch.gather(p, 1, at) * valid
        size = y.abs()
        if renorm:
            total = picked.sum(1, keepdim=True) + eps
            total = torch.where(picked.sum(1, keepdim=True) == 0, torch.full_like(total, math.inf), total)
            size = (size + (size * picked).sum(1, keepdim=True) / total) / total
            y = (y - (y * picked).sum(1, keepdim=True) / total) / total
        dp = torch.zeros_like(x).scatter_add(1, at, y * valid * factor)
        size = torch.zeros_like(x).scatter_add(1, at, size * valid * abs(factor))
        if score == 0:
            grad = p * (dp - (dp * p).sum(1, keepdim=True))
            mass = p * (size + (size * p).sum(1, keepdim=True))
        else:
            grad, mass = p * rest * dp, p * rest * size
    if dl is not None:
        dr = torch.zeros_like(x)
        for s, (lo, hi) in enumerate(_ranges(offsets, len(x))):
            n = int(rows[s])
            if n > 0:
                dr[lo:max(lo, hi)] = float(dl[s]) * E / (k * n * n) * counts[s].double()
        g, m = r * (dr - (dr * r).sum(1, keepdim=True)), r * (dr.abs() + (dr.abs() * r).sum(1, keepdim=True))
        grad, mass = (grad + g, mass + m) if score == 0 else (grad + g * rest, mass + m * rest)
    live = valid[:, :1]
    zero = torch.zeros_like(grad)
    return torch.where(live, grad, zero).reshape(shape), torch.where(live, mass, zero).reshape(shape)


def _check_grad(got, x, *args):
    want, mass = _grad_want(x, *args)
    tol = 6 * _score_error(x) + 10 * U
    _within(got, want, tol * mass + _half(got.dtype) * (want.abs() + tol * mass) + _tiny(got.dtype) + 2.0 ** -100 * mass)


GRADS = [(1, 8, 2, "f32", None), (7, 128, 8, "bf16", None), (70, 160, 6, "f16", 3), (1025, 256, 8, "f32", 9), (33, 60, 12, "bf16", 2)]


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("renorm", [0, 1])
@pytest.mark.parametrize("E", [1, 3, 8, 9, 16, 33, 64, 128, 160, 256, 300, 512, 777, 1024, 2048])
def test_grad_experts(aclnn, dev, E, renorm, score):
    for T, _, k, name, S in GRADS:
        k = min(k, E) if T < 1000 else k                                             # more ids than experts: some come twice
        dtype = TORCH[name]
        x, idx = _router_inputs(T, E, k, dtype, E + T, finished=0.2 if T > 7 else 0.0)
        g = torch.Generator().manual_seed(E)
        dy = torch.randn(idx.shape, generator=g)
        offsets = None if S is None else _offsets(T, S, T, begin=T // 9, end=T - T // 7)
        _, counts, rows, _ = _balance_want(x, idx, offsets, score)
        dl = torch.rand(len(rows), generator=g)
        tables = (dl, counts, rows)
        for y, t, out in [(dy, tables, dtype), (dy.to(dtype), (None,) * 3, torch.float32), (None, tables, torch.float32)]:
            off = offsets if t[0] is not None else None
            got = aclnn.moe_gating_top_k_grouped_grad(*_on(dev, x, idx, y, *t, off), score_type=score, renorm=renorm, routed_scaling_factor=2.5, eps=1e-6,
                                                      x_grad_dtype=out)
            assert got.dtype == out
            _check_grad(got, x, idx, y, *t, off, score, renorm, 2.5, 1e-6)


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("T,E,k,S", [(16384, 256, 8, 8), (30001, 8, 2, None), (9000, 160, 6, 700), (300, 64, 8, 300), (1500, 2048, 64, 2), (100, 16, 2, 5000)])
def test_grad_batches(aclnn, dev, T, E, k, S, score):
    x, idx = _router_inputs(T, E, k, torch.float32, T + E, finished=0.1)
    g = torch.Generator().manual_seed(T)
    offsets = None if S is None else _offsets(T, S, T + E)
    loss, counts, rows, _ = aclnn.moe_balance_loss(*_on(dev, x, idx, offsets), score_type=score)
    dl, dy = torch.rand(len(rows), generator=g), torch.randn(idx.shape, generator=g)
    got = aclnn.moe_gating_top_k_grouped_grad(*_on(dev, x, idx, dy, dl), counts, rows, *_on(dev, offsets), score_type=score, renorm=1)
    _check_grad(got, x, idx, dy, dl, counts.cpu(), rows.cpu(), offsets, score, 1, 1.0, 1e-20)


@pytest.mark.parametrize("score", [0, 1])
def test_grad_rows_of_unusual_values(aclnn, dev, score):
    T, E, k = 9, 96, 3
    x, idx = _router_inputs(T, E, k, torch.float32, 3, spread=2.0)
    x[0, 10:] = -math.inf
    x[0, 0] = 1.0
    idx[0] = torch.tensor([0, 50, 4])                       # a pick that was masked
    x[1] = -math.inf                                        # nothing left: all picks have p = 0
    x[2] -= 95.0                                            # sigmoid scores below 2^-126
    x[3, 40] = math.nan
    x[4] = torch.finfo(torch.float32).min
    x[5, 5] = 60.0                                          # a score of one to 26 digits
    idx[6] = torch.tensor([7, 7, 7])                        # the same index three times
    idx[7] = torch.tensor([3, -1, 96])
    idx[8] = torch.tensor([96, 1, 2])
    g = torch.Generator().manual_seed(5)
    dy = torch.randn((T, k), generator=g)
    counts = torch.randint(0, 9, (1, E), generator=g, dtype=torch.int32)
    rows, dl = torch.tensor([T], dtype=torch.int32), torch.tensor([0.7])
    for renorm in (0, 1):
        got = aclnn.moe_gating_top_k_grouped_grad(*_on(dev, x, idx, dy, dl, counts, rows), score_type=score, renorm=renorm).cpu()
        want, mass = _grad_want(x, idx, dy, dl, counts, rows, None, score, renorm, 1.0, 1e-20)
        tol = (6 * (2 * 100 + E / 64 + 20) + 10) * U
        rest = [r for r in range(T) if r not in (2, 3, 4)]
        _within(got[rest], want[rest], (tol * mass + 2.0 ** -24 * want.abs() + 2.0 ** -120)[rest])
        if score == 0:
            assert torch.isnan(got[3]).all()
            _within(got[[2, 4]], want[[2, 4]], (tol * mass + 2.0 ** -120)[[2, 4]])
        else:
            # row 2: the picks' scores are lost in fp32, the shares of the balance are not; row 4: the definition's shares are 0 / 0
            only = aclnn.moe_gating_top_k_grouped_grad(*_on(dev, x, idx, None, dl, counts, rows), score_type=1).cpu()
            w, m = _grad_want(x, idx, None, dl, counts, rows, None, 1, renorm, 1.0, 1e-20)
            _within(only[2], w[2], tol * m[2] + 2.0 ** -120)
            assert torch.isfinite(only[4]).all()
            assert torch.isnan(got[3, 40])
        assert not got[1].any() and not got[8].any()


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("T,E,k,dtype_name", [(512, 64, 4, "f32"), (300, 8, 8, "f32"), (2000, 250, 5, "bf16"), (900, 7, 3, "f16")])
def test_grad_of_nearly_even_counts(aclnn, dev, T, E, k, dtype_name, score):
    """Where a batch is spread as the loss wants it, its gradient is small, and as exact as it is small: errors are taken of the counts' distances from their
    mean, not of the counts.  Of even counts it is nothing at all."""
    x, _ = _router_inputs(T, E, k, TORCH[dtype_name], E)
    idx = (torch.arange(T * k).reshape(T, k) % E).int()
    g = torch.Generator().manual_seed(E)
    dl = torch.tensor([0.01, 3.0])
    offsets = torch.tensor([0, T // 3, T], dtype=torch.int32)
    rows = torch.tensor([T // 3, T - T // 3], dtype=torch.int32)
    even = torch.tensor([1 << 9, 1 << 19], dtype=torch.int32)[:, None].expand(2, E).contiguous()
    for counts in (even + torch.randint(-2, 3, (2, E), generator=g, dtype=torch.int32), even):
        # rows and picks such that the mean of the counts is k n / E, as it is where every id is an expert
        n = torch.tensor([(1 << 9) * E // k, (1 << 19) * E // k], dtype=torch.int32)
        got = aclnn.moe_gating_top_k_grouped_grad(*_on(dev, x, idx, None, dl, counts, n, offsets), score_type=score, x_grad_dtype=torch.float32)
        want, mass = _grad_want(x, idx, None, dl, counts.double() - counts.double().mean(1, keepdim=True), n, offsets, score, 0, 1.0, 0.0)
        size = mass if (counts != even).any() else torch.zeros_like(mass)
        # (the mean of k n / E rounded to a whole number is up to a half off)
        slack = 4 * U * (dl * E / k / n / n)[:, None].double() * torch.ones(1, E)
        slack = torch.cat([slack[:1].expand(int(rows[0]), E), slack[1:].expand(int(rows[1]), E)])
        _within(got, want, (6 * _score_error(x) + 10 * U) * size + slack)
        if (1 << 19) * E % k == 0 and (1 << 9) * E % k == 0 and not (counts != even).any():
            assert not got.any()


def test_grad_strides_and_ranks(aclnn, dev):
    """Three dimensions, views of larger tensors, rows that begin on any element; a gradient of 16 bits from picks' gradients of either type."""
    x, idx = _router_inputs((3, 50), 33, 3, torch.bfloat16, 4, finished=0.1)
    offsets = torch.tensor([0, 61, 61, 140], dtype=torch.int64)
    g = torch.Generator().manual_seed(4)
    dy, dl = torch.randn(idx.shape, generator=g), torch.rand(3, generator=g)
    _, counts, rows, _ = _balance_want(x, idx, offsets, 1)
    want = aclnn.moe_gating_top_k_grouped_grad(*_on(dev, x, idx, dy, dl, counts, rows, offsets), score_type=1, renorm=1)
    assert want.shape == x.shape
    _check_grad(want, x, idx, dy, dl, counts, rows, offsets, 1, 1, 1.0, 1e-20)
    wide = torch.zeros((3, 50, 70), dtype=torch.bfloat16, device=dev)
    wide[..., 5:38] = x.to(dev)
    flat = torch.zeros(150 * 33 + 1, dtype=torch.bfloat16, device=dev)
    flat[1:] = x.to(dev).reshape(-1)
    ids = torch.zeros((3, 50, 6), dtype=torch.int32, device=dev)
    ids[..., ::2] = idx.to(dev)
    picks = dy.to(dev).transpose(0, 2).contiguous().transpose(0, 2)
    tables = torch.stack([counts, counts], -1).to(dev)[..., 1]
    spread = torch.stack([offsets, offsets], -1).to(dev)[:, 0]
    for logits in (wide[..., 5:38], flat[1:].view(3, 50, 33)):
        out = torch.zeros(150 * 33 + 3, dtype=torch.bfloat16, device=dev)
        got = aclnn.moe_gating_top_k_grouped_grad(logits, ids[..., ::2], picks, dl.to(dev), tables, rows.to(dev), spread, score_type=1, renorm=1,
                                                  out=out[1:-2].view(3, 50, 33))
        assert torch.equal(got, want) and not out[0] and not out[-2:].any()
    dy16 = dy.to(torch.bfloat16)
    _check_grad(aclnn.moe_gating_top_k_grouped_grad(*_on(dev, x, idx, dy16)), x, idx, dy16, None, None, None, None, 0, 0, 1.0, 1e-20)


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("E", [96, 2048])
def test_grad_of_picks_with_small_scores(aclnn, dev, E, score):
    """Picks far below the row's top, with nothing added to their sum: their shares of it are ordinary numbers, though a score divided by the row's sum, or one
    divided by the sum of the scores, would leave fp32."""
    T, k = 40, 4
    x, _ = _router_inputs(T, E, k, torch.float32, 17)
    idx = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(t))[:k] for t in range(T)]).int()
    x = x.clamp(-2, 2)
    x.scatter_add_(1, idx.long(), torch.full((T, k), -82.0))        # e^(-82 - 2 - 2) is above 2^-126, and divided by the sum of a row it is below
    dy = torch.randn((T, k), generator=torch.Generator().manual_seed(18))
    for eps in (0.0, 2.0 ** -120):
        got = aclnn.moe_gating_top_k_grouped_grad(*_on(dev, x, idx, dy), score_type=score, renorm=1, eps=eps)
        _check_grad(got, x, idx, dy, None, None, None, None, score, 1, 1.0, eps)


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("E,k", [(8, 2), (16, 12), (96, 4), (256, 8), (2048, 4)])
def test_grad_of_picks_whose_scores_fp32_loses(aclnn, dev, E, k, score):
    """Weights of picks far below the row's top, or of sigmoid scores below fp32's range: the choice has their shares in 64 bits, and so has the gradient; and small
    gradients of small scores, whose products fp32 does not hold.  Every second row is an ordinary one."""
    T = 75
    x, _ = _router_inputs(T, E, k, torch.float32, 27)
    g = torch.Generator().manual_seed(28)
    idx = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).int()
    idx[4, 1], idx[6, 0], idx[9, 1] = -1, E, idx[9, 0]
    dy = torch.randn((T, k), generator=g)
    for down, size, eps in [(80.0, 1e-8, 0.0), (60.0, 1e-25, 1e-20), (95.0, 1.0, 0.0), (100.0, 1e-3, 2.0 ** -140), (95.0, 1.0, 1e-20), (400.0, 1.0, 0.0),
                            (400.0, 1.0, 1e-20), (45.0, 1.0, 1e-20)]:
        low = x.clone()
        low[::2].scatter_add_(1, idx[::2].long().clamp(0, E - 1), torch.full((T // 2 + 1, k), -down))
        low[10, idx[10].long()] = torch.finfo(torch.float32).min                     # nothing is left of these in 64 bits either
        low[12, idx[12].long()] = -math.inf
        low[14, idx[14, 0].long()] = -math.inf
        y = dy * size
        got = aclnn.moe_gating_top_k_grouped_grad(*_on(dev, low, idx, y), score_type=score, renorm=1, eps=eps)
        want, mass = _grad_want(low, idx, y, None, None, None, None, score, 1, 1.0, eps)
        kept = torch.isfinite(low) & (low > -1e30)
        tol = (6 * (2 * (down + 10) + E / 64 + 20) + 10) * U
        _within(got, want, tol * mass + U * want.abs() + 2.0 ** -126 * kept + 2.0 ** -100 * mass)
        assert not got[10].any() and not got[12].any() and not got[6].any()
        for again in range(2):
            assert torch.equal(got, aclnn.moe_gating_top_k_grouped_grad(*_on(dev, low, idx, y), score_type=score, renorm=1, eps=eps))


def test_grad_against_differences(aclnn, dev):
    """Along random directions: the definition's central differences in 64 bits (their own error: h^2 of third derivatives below 1, and 2^-53 / h of the value)."""
    T, E, k = 40, 24, 3
    g = torch.Generator().manual_seed(11)
    for score in (0, 1):
        for renorm in (0, 1):
            x, idx = _router_inputs(T, E, k, torch.float32, 20 + score)
            dy, offsets = torch.randn((T, k), generator=g), torch.tensor([0, 17, 40], dtype=torch.int32)
            _, counts, rows, _ = _balance_want(x, idx, offsets, score)
            dl = torch.tensor([0.3, 1.1])

            def value(z):
                p = torch.softmax(z, 1) if score == 0 else torch.sigmoid(z)
                y = torch.gather(p, 1, idx.long())
                if renorm:
                    y = y / (y.sum(1, keepdim=True) + 1e-20)
                total = (2.5 * y * dy.double()).sum()
                r = p / p.sum(1, keepdim=True)
                for s, (lo, hi) in enumerate(_ranges(offsets, T)):
                    total = total + dl[s].double() * E / (k * int(rows[s])) * (counts[s] * r[lo:hi].mean(0)).sum()
                return float(total)

            got = aclnn.moe_gating_top_k_grouped_grad(*_on(dev, x, idx, dy, dl, counts, rows, offsets), score_type=score, renorm=renorm,
                                                      routed_scaling_factor=2.5).cpu().double()
            _, mass = _grad_want(x, idx, dy, dl, counts, rows, offsets, score, renorm, 2.5, 1e-20)
            for _ in range(4):
                d = torch.randn((T, E), generator=g).double()
                h = 1e-5
                along = (value(x.double() + h * d) - value(x.double() - h * d)) / (2 * h)
                bound = float(((6 * _score_error(x) + 10 * U) * mass * d.abs()).sum()) + 1e-7 * float((mass * d.abs()).sum())
                assert abs(float((got * d).sum()) - along) <= bound


# ------------------------------------------------------------------------------------------------ sandwich norm
WIDTHS = [1, 3, 8, 64, 257, 1000, 1024, 2880, 4096, 5000, 7168, 8192, 8200, 12000, 16384, 16392, 20001]


def _sandwich_inputs(T, H, dtype, seed, post=True, pre=True, gate="none", wide=False):
    g = torch.Generator().manual_seed(seed)
    lead = T if isinstance(T, tuple) else (T,)
    kind = torch.float32 if wide else dtype
    x = (torch.randn(lead + (H,), generator=g) * torch.exp(0.5 * torch.randn(H, generator=g))).to(dtype)
    res = torch.randn(lead + (H,), generator=g).to(dtype)
    post = (1 + 0.3 * torch.randn(H, generator=g)).to(kind) if post else None
    pre = (1 + 0.3 * torch.randn(H, generator=g)).to(kind) if pre else None
    gate = {"none": lambda: None, "channel": lambda: (0.5 + 0.3 * torch.randn(H, generator=g)).to(kind), "row": lambda: torch.randn(lead + (1,), generator=g).to(kind),
            "each": lambda: torch.randn(lead + (H,), generator=g).to(dtype)}[gate]()
    return x, res, post, gate, pre


def _gate64(gate, gate_type):
    if gate is None:
        return 1.0
    return torch.sigmoid(gate.double()) if gate_type else gate.double()


def _norm_error(H):
    return (H / 64 + 20) * U


def _check_sandwich(x, res, post, gate, pre, got, gate_type=0, alpha=1.0, beta=1.0, eps=1e-6, smooth=None):
    total, norm, y, scale, post_rstd, pre_rstd = [None if t is None else t.cpu() for t in got]
    dtype, H = x.dtype, x.shape[-1]
    alpha, beta = [float(torch.tensor(v, dtype=torch.float32)) for v in (alpha, beta)]
    tol = _norm_error(H)
    u = x.double()
    if post is not None:
        r = 1 / torch.sqrt(u.square().mean(-1, keepdim=True) + eps)
        if post_rstd is not None:
            _within(post_rstd, r[..., 0], tol * r[..., 0])
        u = u * r * post.double()
    v, a = beta * _gate64(gate, gate_type) * u, alpha * res.double()
    bound = (tol + 10 * U) * v.abs() + 2 * U * a.abs()
    _within(total, a + v, bound + _half(dtype) * ((a + v).abs() + bound) + _tiny(dtype))
    if pre is None:
        assert norm is None and y is None and pre_rstd is None
        return
    s = total.double()                                  # the sum as it was kept
    r = 1 / torch.sqrt(s.square().mean(-1, keepdim=True) + eps)
    if pre_rstd is not None:
        _within(pre_rstd, r[..., 0], tol * r[..., 0])
    n = s * r * pre.double()
    if norm is not None:
        _within(norm, n, (tol + _half(dtype) * (1 + tol)) * n.abs() + _tiny(dtype))
    if y is not None:
        w = n if smooth is None else n * smooth.double()
        want = w.abs().amax(-1) / 127
        _within(scale, want, tol * want + 1e-44)
        assert torch.all((y.double() - w / want[..., None]).abs() <= 0.5 + 127 * 8 * U)


@pytest.mark.parametrize("dtype_name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H", WIDTHS)
def test_sandwich_widths(aclnn, dev, H, dtype_name):
    for i, (T, post, pre, gate, wide, quantise) in enumerate([(1, True, True, "none", False, False), (3, True, True, "channel", True, True),
                                                              (33, True, False, "row", True, False), ((2, 5), False, True, "each", False, True),
                                                              (9, False, False, "channel", False, False)]):
        ins = _sandwich_inputs(T, H, TORCH[dtype_name], H + i, post, pre, gate, wide)
        smooth = torch.exp(0.3 * torch.randn(H, generator=torch.Generator().manual_seed(H))) if quantise else None
        kw = dict(gate_type=i % 2, residual_scale=0.9 if i else 1.0, branch_scale=0.25 if i else 1.0, epsilon=1e-5)
        got = aclnn.moe_sandwich_norm(*_on(dev, *ins), smooth_scale=None if smooth is None else smooth.to(dev), quantise=quantise, output_rstd=True, **kw)
        _check_sandwich(*ins, got, i % 2, kw["residual_scale"], kw["branch_scale"], 1e-5, smooth)


def test_sandwich_outputs_alone_and_in_place(aclnn, dev):
    for H in (1000, 4096, 20000):
        ins = _sandwich_inputs(37, H, torch.bfloat16, 5, gate="row")
        x, res, post, gate, pre = _on(dev, *ins)
        whole = aclnn.moe_sandwich_norm(x, res, post, gate, pre, quantise=True, output_rstd=True)
        _check_sandwich(*ins, whole)
        for keep in [(1,), (2, 3), (5,), (1, 2, 3, 4), (4, 5)]:
            out = tuple(torch.zeros_like(t) if i in keep or i == 0 else None for i, t in enumerate(whole))
            if not any(i in keep for i in (1, 2, 5)):
                continue
            aclnn.moe_sandwich_norm(x, res, post, gate, pre, out=out)
            for a, b in zip(out, whole):
                assert a is None or torch.equal(a, b)
        for which in (0, 1):
            a, b = x.clone(), res.clone()
            again = aclnn.moe_sandwich_norm(a, b, post, gate, pre, out=((a, b)[which],) + tuple(torch.empty_like(t) for t in whole[1:]))
            for p, q in zip(again, whole):
                assert torch.equal(p, q)
            assert torch.equal((b, a)[which], (res, x)[which])
        twice = aclnn.moe_sandwich_norm(x, x, post, gate, pre)                       # the same tensor twice
        _check_sandwich(ins[0], ins[0], *ins[2:], twice)


@pytest.mark.parametrize("dtype_name", ["f32", "bf16"])
def test_sandwich_strides_and_offsets(aclnn, dev, dtype_name):
    dtype = TORCH[dtype_name]
    for H in (1001, 4096, 9000):
        ins = _sandwich_inputs(9, H, dtype, H, gate="each")
        x, res, post, gate, pre = _on(dev, *ins)
        want = aclnn.moe_sandwich_norm(x, res, post, gate, pre, quantise=True)
        flat = torch.zeros(9 * H + 3, dtype=dtype, device=dev)
        odd = flat[3:].view(9, H)
        odd.copy_(x)
        wide = torch.zeros((9, 2 * H), dtype=dtype, device=dev)
        wide[:, H:] = res
        gammas = torch.zeros((2, 2 * H), dtype=dtype, device=dev)
        gammas[0, ::2], gammas[1, 1:H + 1] = post, pre
        out = (torch.zeros(9 * H + 1, dtype=dtype, device=dev)[1:].view(9, H), torch.zeros(9 * H + 7, dtype=dtype, device=dev)[7:].view(9, H),
               torch.zeros(9 * H + 5, dtype=torch.int8, device=dev)[5:].view(9, H), torch.zeros(10, device=dev)[1:], None, None)
        got = aclnn.moe_sandwich_norm(odd, wide[:, H:], gammas[0, ::2], gate.t().contiguous().t(), gammas[1, 1:H + 1], out=out)
        for a, b in zip(got, want):
            assert a is None or torch.equal(a, b)


@pytest.mark.parametrize("H", [1000, 4096, 20001])
def test_sandwich_rows_of_unusual_values(aclnn, dev, H):
    x, res, post, gate, pre = _sandwich_inputs(8, H, torch.float32, H, gate="row")
    x[0] = 0                                                # u = 0: the residual alone
    x[1], res[1] = 0, 0
    x[2, H // 2] = math.nan
    x[3, H - 1] = math.inf
    x[4] *= 1e-30                                           # squares underflow: x / sqrt(eps)
    res[5, 0] = -math.inf
    gate[6] = 0
    total, norm, y, scale, post_rstd, pre_rstd = [t.cpu() for t in aclnn.moe_sandwich_norm(*_on(dev, x, res, post, gate, pre), quantise=True, output_rstd=True)]
    assert torch.equal(total[0], res[0]) and not total[1].any() and not norm[1].any() and not y[1].any() and scale[1] == 0
    assert torch.isnan(total[2]).all() and torch.isnan(norm[2]).all() and torch.isnan(scale[2]) and not y[2].any()
    assert torch.isnan(total[3, H - 1]) and torch.isnan(scale[3])                    # inf * 1 / inf; the factor of the others is 0
    assert torch.equal(total[6], res[6])
    for rows in (slice(0, 1), slice(4, 5), slice(6, 8)):
        _check_sandwich(x[rows], res[rows], post, gate[rows], pre, [t[rows] for t in (total, norm, y, scale, post_rstd, pre_rstd)])
    nothing = aclnn.moe_sandwich_norm(*_on(dev, torch.zeros(2, H), torch.zeros(2, H), post, None, pre), epsilon=0.0, output_rstd=True)
    assert not any(t.any() for t in nothing if t is not None)


def test_sandwich_in_place_beside_sums_near_the_top(aclnn, dev):
    """The sum in the residual's place where a lane's last piece reaches back over another wave's: what that one has written there already, taken for the
    residual once more, would be past the type's range, and must not come into the row's norm."""
    T, H = 600, 1031
    x = torch.full((T, H), 3e4, dtype=torch.float16)
    res = torch.full((T, H), 2.5e4, dtype=torch.float16)
    pre = torch.ones(H, dtype=torch.float16)
    for _ in range(3):
        x_dev, res_dev, pre_dev = _on(dev, x, res, pre)
        out = (res_dev, torch.empty_like(x_dev), torch.empty((T, H), dtype=torch.int8, device=dev), torch.empty(T, device=dev), None, torch.empty(T, device=dev))
        _check_sandwich(x, res, None, None, pre, aclnn.moe_sandwich_norm(x_dev, res_dev, pre_gamma=pre_dev, out=out))


# More rows than workgroups, so that workgroups go on to a second row and some to a third: one piece a lane (1280, 2048 and 768 workgroups), two on up to 512 lanes
# (512, 256), two on up to 768 and four (256; 512 off the eight).
LOOPS = [(2600, 1031), (4200, 1000), (1600, 2880), (1100, 5000), (1100, 7167), (600, 8192), (600, 8200), (600, 9001), (600, 12000), (600, 12304), (1100, 16381),
         (600, 16384)]


@pytest.mark.parametrize("dtype_name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,H", LOOPS)
def test_sandwich_more_rows_than_workgroups(aclnn, dev, T, H, dtype_name):
    """The same bits as in calls that give every row a workgroup of its own, the sum apart and in the place of either input; the last rows against the formula."""
    dtype = TORCH[dtype_name]
    smooth = torch.exp(0.3 * torch.randn(H, generator=torch.Generator().manual_seed(H)))
    for i, (post, pre, gate) in enumerate([(True, True, "row"), (False, True, "each"), (True, False, "channel")]):
        few = _sandwich_inputs(211, H, dtype, T + i, post, pre, gate, dtype_name == "f16")
        at = [(torch.arange(T) * step + 3) % 211 for step in (1, 7, 5)]             # rows a workgroup apart are others
        ins = [few[0][at[0]], few[1][at[1]], few[2], few[3] if gate == "channel" else few[3][at[2]], few[4]]
        given = _on(dev, *ins)
        kw = dict(gate_type=i % 2, residual_scale=0.9, branch_scale=0.25)
        if pre:
            kw["smooth_scale"] = smooth.to(dev)
        whole = aclnn.moe_sandwich_norm(*given, quantise=pre, output_rstd=True, **kw)
        _check_sandwich(*[t[-40:] if j in (0, 1) or j == 3 and gate != "channel" else t for j, t in enumerate(ins)],
                        [None if t is None else t[-40:] for t in whole], i % 2, 0.9, 0.25, 1e-6, smooth if pre else None)
        for begin in range(0, T, 200):
            part = slice(begin, begin + 200)
            alone = aclnn.moe_sandwich_norm(given[0][part], given[1][part], given[2], given[3] if gate == "channel" else given[3][part], given[4], quantise=pre,
                                            output_rstd=True, **kw)
            for a, b in zip(alone, whole):
                assert (a is None) == (b is None) and (a is None or torch.equal(a, b[part])), begin
        for which in (0, 1):
            pair = [given[0].clone(), given[1].clone()]
            out = (pair[which],) + tuple(None if t is None else torch.empty_like(t) for t in whole[1:])
            for a, b in zip(aclnn.moe_sandwich_norm(*pair, *given[2:], out=out, **kw), whole):
                assert (a is None) == (b is None) and (a is None or torch.equal(a, b))
            assert torch.equal(pair[1 - which], given[1 - which])


def test_sandwich_gate_of_one_row_for_all(aclnn, dev):
    """A gate with a stride of zero over the rows is read as a gate of its own for each of them."""
    T, H = 19, 1000
    x, res, post, gate, pre = _sandwich_inputs(T, H, torch.bfloat16, 8, gate="each")
    shared = gate[:1].expand(T, H)
    _check_sandwich(x, res, post, shared, pre, aclnn.moe_sandwich_norm(*_on(dev, x, res, post), gate[:1].to(dev).expand(T, H), pre.to(dev), gate_type=1), 1)
    ins = list(_grad_inputs(T, H, torch.bfloat16, 8, True, True, "each", False, 1))
    ins[5] = shared
    given = _on(dev, *ins)
    given[5] = gate[:1].to(dev).expand(T, H)
    _check_sandwich_grad(aclnn.moe_sandwich_norm_grad(*given, gate_type=1), *ins, 1, 1.0, 1.0)


@pytest.mark.parametrize("H", [1000, 20000])
def test_sandwich_gates_far_from_zero(aclnn, dev, H):
    """Sigmoid gates and their slopes from nearly shut to open, each to its own precision: |gate| + 4 units for the gate, as many for 1 less it, 6 for products."""
    T = 6
    g = torch.Generator().manual_seed(H)
    x, ds = torch.randn((T, H), generator=g), torch.randn((T, H), generator=g)
    gate = 100 * (2 * torch.rand((T, H), generator=g) - 1)
    gate[0, :6] = torch.tensor([math.inf, -math.inf, torch.finfo(torch.float32).max, torch.finfo(torch.float32).min, 0.0, -0.0])
    open_, shut = torch.sigmoid(gate.double()), torch.sigmoid(-gate.double())
    tol = (2 * gate.double().abs().clamp(max=90) + 8 + 6) * U
    lost = 2.0 ** -126 * (1 + x.double().abs()) * (1 + ds.double().abs())
    total = aclnn.moe_sandwich_norm(x.to(dev), torch.zeros((T, H), device=dev), gate=gate.to(dev), gate_type=1)[0]
    _within(total, x.double() * open_, tol * (x.double() * open_).abs() + lost)
    got = aclnn.moe_sandwich_norm_grad(x.to(dev), sum_grad=ds.to(dev), gate=gate.to(dev), gate_type=1)
    _within(got[0], ds.double() * open_, tol * (ds.double() * open_).abs() + lost)
    slope = ds.double() * x.double() * open_ * shut
    _within(got[3], slope, tol * slope.abs() + lost)
    row = gate[:, 6:7].clone()
    one = aclnn.moe_sandwich_norm(x.to(dev), torch.zeros((T, H), device=dev), gate=row.to(dev), gate_type=1)[0]
    _within(one, x.double() * open_[:, 6:7], tol[:, 6:7] * (x.double() * open_[:, 6:7]).abs() + lost)


def test_sandwich_long_batches_and_empty_ones(aclnn, dev):
    ins = _sandwich_inputs(70000, 64, torch.bfloat16, 3, gate="each")
    _check_sandwich(*ins, aclnn.moe_sandwich_norm(*_on(dev, *ins)))
    for shape in [(0, 64), (3, 0, 64)]:
        x = torch.empty(shape, dtype=torch.bfloat16, device=dev)
        got = aclnn.moe_sandwich_norm(x, x.clone(), pre_gamma=torch.ones(64, dtype=torch.bfloat16, device=dev), quantise=True)
        assert got[0].shape == shape and got[3].shape == shape[:-1]
        grads = aclnn.moe_sandwich_norm_grad(x, sum_grad=x.clone(), post_gamma=torch.ones(64, dtype=torch.bfloat16, device=dev),
                                             post_rstd=torch.empty(shape[:-1], device=dev))
        assert grads[0].shape == shape and not grads[2].any() and grads[2].shape == (64,)


# ------------------------------------------------------------------------------------------------ its gradients
def _sandwich_grad_want(x, s, ds, dn, post, gate, pre, post_rstd, pre_rstd, gate_type, alpha, beta):
    """((gradient, magnitude of its terms) ...) in 64 bits."""
    H, zero = x.shape[-1], torch.zeros(x.shape, dtype=torch.float64)
    alpha, beta = [float(torch.tensor(v, dtype=torch.float32)) for v in (alpha, beta)]
    flat = lambda t: t.reshape(-1, H).sum(0)
    d, m = (zero, zero) if ds is None else (ds.double(), ds.double().abs())
    pre_grad = None
    if pre is not None:
        r = pre_rstd.double()[..., None]
        h, g = s.double() * r, dn.double()
        pre_grad = flat(g * h), flat((g * h).abs())
        g = g * pre.double()
        d = d + r * (g - h * (g * h).mean(-1, keepdim=True))
        m = m + r.abs() * (g.abs() + h.abs() * (g * h).abs().mean(-1, keepdim=True))
    res_grad = alpha * d, abs(alpha) * m
    v, w = beta * d, abs(beta) * m
    r = 1.0 if post is None else post_rstd.double()[..., None]
    h = x.double() * r
    u = h if post is None else h * post.double()
    gate_grad = post_grad = None
    if gate is not None:
        slope = torch.sigmoid(gate.double()) * torch.sigmoid(-gate.double()) if gate_type else torch.ones_like(gate, dtype=torch.float64)
        each, size = v * u * slope, w * u.abs() * slope
        if gate.dim() == 1:
            gate_grad = flat(each), flat(size)
        elif gate.shape[-1] == 1:
            gate_grad = each.sum(-1, keepdim=True), size.sum(-1, keepdim=True)
        else:
            gate_grad = each, size
        open_ = _gate64(gate, gate_type)
        v, w = v * open_, w * open_.abs()
    if post is not None:
        post_grad = flat(v * h), flat(w * h.abs())
        v, w = v * post.double(), w * post.double().abs()
        v = r * (v - h * (v * h).mean(-1, keepdim=True))
        w = r.abs() * (w + h.abs() * (w * h.abs()).mean(-1, keepdim=True))
    return (v, w), res_grad, post_grad, gate_grad, pre_grad


def _check_sandwich_grad(got, *args):
    want = _sandwich_grad_want(*args)
    x = args[0]
    H, T = x.shape[-1], x.numel() // x.shape[-1]
    tol = 2 * _norm_error(H) + 20 * U
    for g, w in zip(got, want):
        assert (g is None) == (w is None)
        if g is None:
            continue
        value, mass = w
        columns = tol + (min(T, 512) + 2) * U if g.dim() == 1 else tol
        _within(g, value, columns * mass + _half(g.dtype) * (value.abs() + columns * mass) + _tiny(g.dtype))


def _grad_inputs(T, H, dtype, seed, post, pre, gate, wide, gate_type=0, alpha=1.0, beta=1.0):
    x, res, post, gate, pre = _sandwich_inputs(T, H, dtype, seed, post, pre, gate, wide)
    g = torch.Generator().manual_seed(seed + 1)
    ds, dn = torch.randn(x.shape, generator=g).to(dtype), torch.randn(x.shape, generator=g).to(dtype) if pre is not None else None
    u = x.double()
    post_rstd = pre_rstd = None
    if post is not None:
        post_rstd = (1 / torch.sqrt(u.square().mean(-1) + 1e-6)).float()
        u = u * post_rstd.double()[..., None] * post.double()
    s = (alpha * res.double() + beta * _gate64(gate, gate_type) * u).to(dtype)
    if pre is not None:
        pre_rstd = (1 / torch.sqrt(s.double().square().mean(-1) + 1e-6)).float()
    return x, s, ds, dn, post, gate, pre, post_rstd, pre_rstd


@pytest.mark.parametrize("dtype_name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H", WIDTHS)
def test_sandwich_grad_widths(aclnn, dev, H, dtype_name):
    for i, (T, post, pre, gate, wide) in enumerate([(1, True, True, "none", False), (3, True, True, "channel", True), (33, True, False, "row", True),
                                                    ((2, 5), False, True, "each", False), (9, False, False, "channel", False), (13, False, True, "none", True),
                                                    (300, True, True, "row", False)]):
        ins = _grad_inputs(T, H, TORCH[dtype_name], H + i, post, pre, gate, wide, i % 2, 0.9, 0.25)
        got = aclnn.moe_sandwich_norm_grad(*_on(dev, *ins), gate_type=i % 2, residual_scale=0.9, branch_scale=0.25)
        _check_sandwich_grad(got, *ins, i % 2, 0.9, 0.25)


@pytest.mark.parametrize("T,H", [(5000, 512), (2000, 4096), (1200, 7168), (700, 12288), (200000, 16)])
def test_sandwich_grad_batches(aclnn, dev, T, H):
    for gate, dtype in [("channel", torch.bfloat16), ("each", torch.float32)]:
        ins = _grad_inputs(T, H, dtype, T, True, True, gate, False, 1)
        got = aclnn.moe_sandwich_norm_grad(*_on(dev, *ins), gate_type=1)
        _check_sandwich_grad(got, *ins, 1, 1.0, 1.0)
        for a, b in zip(got, aclnn.moe_sandwich_norm_grad(*_on(dev, *ins), gate_type=1)):   # equal calls, equal bits
            assert torch.equal(a, b)


@pytest.mark.parametrize("H", [1000, 5000, 20000])
def test_sandwich_grad_outputs_alone(aclnn, dev, H):
    for gate in ("channel", "row", "each"):
        ins = _on(dev, *_grad_inputs(21, H, torch.bfloat16, 5, True, True, gate, False))
        whole = aclnn.moe_sandwich_norm_grad(*ins)
        for keep in range(5):
            out = tuple(torch.full_like(t, 3) if i == keep else None for i, t in enumerate(whole))
            aclnn.moe_sandwich_norm_grad(*ins, out=out)
            assert torch.equal(out[keep], whole[keep])
        only = list(ins)
        only[2] = None                                      # no gradient of the sum
        _check_sandwich_grad(aclnn.moe_sandwich_norm_grad(*only), *[None if t is None else t.cpu() for t in only], 0, 1.0, 1.0)


@pytest.mark.parametrize("T,H", [(1100000, 7), (1100000, 3)])
def test_sandwich_grad_columns_of_long_batches(aclnn, dev, T, H):
    """So many rows that a group of the columns' sums has 512 of them, an element at a time."""
    for gate, dtype in [("channel", torch.float32), ("row", torch.bfloat16)]:
        ins = _grad_inputs(T, H, dtype, H, True, True, gate, False, 1)
        _check_sandwich_grad(aclnn.moe_sandwich_norm_grad(*_on(dev, *ins), gate_type=1), *ins, 1, 1.0, 1.0)


def test_sandwich_grad_strides_and_offsets(aclnn, dev):
    for H in (1001, 4096, 9000):
        ins = _on(dev, *_grad_inputs(9, H, torch.bfloat16, H, True, True, "each", False))
        want = aclnn.moe_sandwich_norm_grad(*ins)

        def odd(t):
            flat = torch.zeros(t.numel() + 3, dtype=t.dtype, device=dev)
            flat[3:] = t.reshape(-1)
            return flat[3:].view(t.shape)

        out = tuple(odd(torch.zeros_like(t)) for t in want)
        for got in (aclnn.moe_sandwich_norm_grad(*map(odd, ins), out=out),
                    aclnn.moe_sandwich_norm_grad(*[torch.stack([t, t], -1)[..., 0] for t in ins])):
            for a, b in zip(got, want):
                assert torch.equal(a, b)


def test_sandwich_grad_against_differences(aclnn, dev):
    """Along random directions of every input, against the forward formula's central differences in 64 bits; the gradients take the forward's factors as
    they come in fp32 and the sum unrounded (fp32), 2^-24 of their terms each."""
    T, H, h = 12, 40, 1e-5
    g = torch.Generator().manual_seed(7)
    for gate_kind in ("channel", "row", "each"):
        for gate_type in (0, 1):
            x, res, post, gate, pre = _sandwich_inputs(T, H, torch.float32, 3, gate=gate_kind)
            ds, dn = torch.randn((T, H), generator=g), torch.randn((T, H), generator=g)

            def value(x, res, post, gate, pre):
                u = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * post
                s = 0.5 * res + 2.0 * (torch.sigmoid(gate) if gate_type else gate) * u
                n = s / torch.sqrt(s.square().mean(-1, keepdim=True) + 1e-6) * pre
                return float((s * ds.double()).sum() + (n * dn.double()).sum())

            s, n, _, _, post_rstd, pre_rstd = aclnn.moe_sandwich_norm(*_on(dev, x, res, post, gate, pre), gate_type=gate_type, residual_scale=0.5, branch_scale=2.0,
                                                                      output_rstd=True)
            got = aclnn.moe_sandwich_norm_grad(x.to(dev), s, *_on(dev, ds, dn, post, gate, pre), post_rstd, pre_rstd, gate_type=gate_type, residual_scale=0.5,
                                               branch_scale=2.0)
            mass = [m for _, m in _sandwich_grad_want(x, s.cpu(), ds, dn, post, gate, pre, post_rstd.cpu(), pre_rstd.cpu(), gate_type, 0.5, 2.0)]
            at = [t.double() for t in (x, res, post, gate, pre)]
            for i, (grad, size) in enumerate(zip(got, mass)):
                d = torch.randn(at[i].shape, generator=g).double()
                plus, minus = [t + h * d if j == i else t for j, t in enumerate(at)], [t - h * d if j == i else t for j, t in enumerate(at)]
                along = (value(*plus) - value(*minus)) / (2 * h)
                scale = float((size * d.abs()).sum())
                assert abs(float((grad.cpu().double() * d).sum()) - along) <= (4 * _norm_error(H) + 60 * U) * scale + 1e-7 * scale


# ------------------------------------------------------------------------------------------------ streams, graphs, memory
def _calls(aclnn, dev, seed):
    """One call of each operator with its outputs: (call, outputs)."""
    x, idx = _on(dev, *_router_inputs(3000, 160, 6, torch.float32, seed, finished=0.1))
    offsets = _offsets(3000, 5, seed).to(dev)
    dy, dl = torch.randn(idx.shape, device=dev), torch.rand(5, device=dev)
    counts = torch.randint(0, 50, (5, 160), device=dev, dtype=torch.int32)
    rows = torch.full((5,), 500, device=dev, dtype=torch.int32)
    balance = (torch.empty(5, device=dev), torch.empty((5, 160), dtype=torch.int32, device=dev), torch.empty(5, dtype=torch.int32, device=dev),
               torch.empty((5, 160), device=dev))
    dx = torch.empty_like(x)
    ins = _on(dev, *_sandwich_inputs(500, 4096, torch.bfloat16, seed, gate="channel"))
    total, norm = torch.empty_like(ins[0]), torch.empty_like(ins[0])
    grads_in = _on(dev, *_grad_inputs(500, 4096, torch.bfloat16, seed, True, True, "channel", False))
    grads = (torch.empty_like(total), torch.empty_like(total), torch.empty(4096, device=dev), torch.empty(4096, device=dev), torch.empty(4096, device=dev))
    return [(lambda ws: aclnn.moe_balance_loss(x, idx, offsets, out=balance, workspace=ws), balance),
            (lambda ws: aclnn.moe_gating_top_k_grouped_grad(x, idx, dy, dl, counts, rows, offsets, renorm=1, out=dx, workspace=ws), (dx,)),
            (lambda ws: aclnn.moe_sandwich_norm(*ins, out=(total, norm, None, None, None, None), workspace=ws), (total, norm)),
            (lambda ws: aclnn.moe_sandwich_norm_grad(*grads_in, out=grads, workspace=ws), grads)]


def test_graph_replays(aclnn, dev):
    """Captured once, replayed with other eager calls and synchronisations between, every replay against the eager outputs."""
    for n, (call, outputs) in enumerate(_calls(aclnn, dev, 5)):
        ws = aclnn.Workspace()
        call(ws)
        want = [t.clone() for t in outputs]
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            call(ws)
            side.synchronize()
            with torch.cuda.graph(graph, stream=side):
                call(ws)
        other = _calls(aclnn, dev, 6)[n][0]
        for replay in range(4):
            for t in outputs:
                t.fill_(3)
            if replay % 2:
                other(None)
                torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(outputs, want):
                assert torch.equal(a, b), (n, replay)


def test_two_graphs_share_a_workspace(aclnn, dev):
    """All four operators captured twice, on unlike inputs, with one workspace; replayed in turn, every replay against the eager outputs."""
    both = [_calls(aclnn, dev, seed) for seed in (9, 10)]
    want = [[t.clone() for call, outputs in calls for t in (call(None), outputs)[1]] for calls in both]
    ws = aclnn.Workspace()
    for calls in both:                                      # as large as any of them needs
        for call, _ in calls:
            call(ws)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    side = torch.cuda.Stream()
    for graph, calls in zip(graphs, both):
        with torch.cuda.graph(graph, stream=side):
            for call, _ in calls:
                call(ws)
    for which in (0, 1, 1, 0, 1, 0):
        for _, outputs in both[which]:
            for t in outputs:
                t.fill_(3)
        graphs[which].replay()
        torch.cuda.synchronize()
        for a, b in zip([t for _, outputs in both[which] for t in outputs], want[which]):
            assert torch.equal(a, b)


def test_two_streams_at_once(aclnn, dev):
    """The same operators on two streams, each with a workspace of its own."""
    first, second = _calls(aclnn, dev, 7), _calls(aclnn, dev, 8)
    want = [[t.clone() for call, outputs in calls for t in (call(None), outputs)[1]] for calls in (first, second)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    spaces = [aclnn.Workspace(), aclnn.Workspace()]
    for _ in range(5):
        for calls in (first, second):
            for _, outputs in calls:
                for t in outputs:
                    t.zero_()
        torch.cuda.synchronize()
        for i in range(4):
            for stream, space, calls in zip(streams, spaces, (first, second)):
                with torch.cuda.stream(stream):
                    calls[i][0](space)
        torch.cuda.synchronize()
        for calls, expected in zip((first, second), want):
            for a, b in zip([t for _, outputs in calls for t in outputs], expected):
                assert torch.equal(a, b)


def test_behind_two_to_the_31_elements(aclnn, dev):
    T, E, k = (1 << 20) + 5000, 2048, 2                     # 2.16e9 logits
    x = torch.zeros((T, E), dtype=torch.bfloat16, device=dev)
    idx = torch.zeros((T, k), dtype=torch.int32, device=dev)
    idx[:, 1] = 1
    tail, ids = _router_inputs(40, E, k, torch.bfloat16, 9)
    x[-40:], idx[-40:] = tail.to(dev), ids.to(dev)
    offsets = torch.tensor([0, T - 40, T], dtype=torch.int64)
    got = aclnn.moe_balance_loss(x, idx, offsets.to(dev))
    want = _balance_want(tail, ids, None, 0)
    assert torch.equal(got[1][1:].cpu(), want[1]) and got[2].tolist() == [T - 40, 40] and int(got[1][0, 0]) == T - 40
    tol = _score_error(tail) + 60 * U
    _within(got[3][1:], want[3], tol * want[3])
    _within(got[3][:1], torch.full((1, E), 1 / E, dtype=torch.float64), torch.tensor((E / 64 + 20 + 530) * U / E))
    dy = torch.randn((T, k), device=dev)
    grad = aclnn.moe_gating_top_k_grouped_grad(x, idx, dy, renorm=1)
    _check_grad(grad[-40:], tail, ids, dy[-40:].cpu(), None, None, None, None, 0, 1, 1.0, 1e-20)
    del x, grad
    T, H = 530000, 4096                                     # 2.17e9 values
    x = torch.zeros((T, H), dtype=torch.bfloat16, device=dev)
    res = torch.ones((T, H), dtype=torch.bfloat16, device=dev)
    ins = _sandwich_inputs(30, H, torch.bfloat16, 4, gate="channel")
    x[-30:], res[-30:] = ins[0].to(dev), ins[1].to(dev)
    got = aclnn.moe_sandwich_norm(x, res, *_on(dev, *ins[2:]), output_rstd=True)
    _check_sandwich(*ins, [None if t is None else t[-30:] for t in got])
    total, post_rstd, pre_rstd = got[0], got[4], got[5]
    grads = aclnn.moe_sandwich_norm_grad(x, total, res, res, *_on(dev, *ins[2:]), post_rstd, pre_rstd)
    want = _sandwich_grad_want(ins[0], total[-30:].cpu(), ins[1], ins[1], *ins[2:], post_rstd[-30:].cpu(), pre_rstd[-30:].cpu(), 0, 1.0, 1.0)
    tol = 2 * _norm_error(H) + 20 * U
    for g, (value, mass) in zip(grads[:2], want[:2]):
        _within(g[-30:], value, tol * mass + _half(g.dtype) * (value.abs() + tol * mass) + _tiny(g.dtype))


def test_column_sums_behind_two_to_the_31_elements(aclnn, dev):
    """Rows of which all but the last are alike: what they add to the columns has a closed form."""
    T, H, n = 530000, 4096, 30                              # 2.17e9 values
    x = torch.zeros((T, H), dtype=torch.bfloat16, device=dev)
    ones = torch.ones((T, H), dtype=torch.bfloat16, device=dev)
    ins = _grad_inputs(n, H, torch.bfloat16, 4, True, True, "channel", False)
    sums, norm_grad = ones.clone(), ones.clone()
    x[-n:], sums[-n:], ones[-n:], norm_grad[-n:] = [t.to(dev) for t in ins[:4]]
    post_rstd, pre_rstd = torch.full((T,), 3.0, device=dev), torch.full((T,), 0.5, device=dev)
    post_rstd[-n:], pre_rstd[-n:] = ins[7].to(dev), ins[8].to(dev)
    post, gate, pre = ins[4:7]
    out = (None, None) + tuple(torch.empty(H, device=dev) for _ in range(3))
    got = aclnn.moe_sandwich_norm_grad(x, sums, ones, norm_grad, *_on(dev, post, gate, pre), post_rstd, pre_rstd, out=out)[2:]
    want = list(_sandwich_grad_want(*ins, 0, 1.0, 1.0)[2:])
    # The rows alike have x = 0: nothing for the post norm and the gate; the pre norm gets 1 * 1 * 0.5 a row.
    want[2] = want[2][0] + (T - n) * 0.5, want[2][1] + (T - n) * 0.5
    tol = 2 * _norm_error(H) + (512 + 2 + 20) * U
    for g, (value, mass) in zip(got, want):
        _within(g, value, tol * mass + _half(g.dtype) * (value.abs() + tol * mass))
    # and with a value there: a row has v = d S = 1 + 0.5 (pre - 0.5 mean(pre) 0.5), x^ = 0.25 * 3
    x[:-n] = 0.25
    got = aclnn.moe_sandwich_norm_grad(x, sums, ones, norm_grad, *_on(dev, post, gate, pre), post_rstd, pre_rstd, out=out)[2:]
    p, o, g = pre.double(), post.double(), gate.double()
    v, m = 1 + 0.5 * (p - 0.25 * p.mean()), 1 + 0.5 * (p.abs() + 0.25 * p.abs().mean())
    first = _sandwich_grad_want(*ins, 0, 1.0, 1.0)[2:4]
    for got_, (value, mass), one, size in zip(got[:2], first, [v * g * 0.75, v * 0.75 * o], [m * g.abs() * 0.75, m * 0.75 * o.abs()]):
        value, mass = value + (T - n) * one, mass + (T - n) * size
        _within(got_, value, tol * mass + _half(got_.dtype) * (value.abs() + tol * mass))


# ------------------------------------------------------------------------------------------------ together
def test_a_router_is_tuned_over_frozen_experts(aclnn, pkg, dev):
    """Norm and int8 rows, router, choice, balance, int8 experts, closing norm; then back to the router's weights, the gammas and the gate, against
    differentiation in 64 bits with what the experts answered as it came."""
    T, H, I, E, k = 66, 256, 128, 16, 4
    g = torch.Generator().manual_seed(21)
    residual = torch.randn((T, H), generator=g).to(torch.bfloat16)
    gamma, post, pre = [(1 + 0.2 * torch.randn(H, generator=g)) for _ in range(3)]
    gate = (0.5 + 0.1 * torch.randn(H, generator=g))
    router = torch.randn((E, H), generator=g) / H ** 0.5
    w13 = torch.randint(-127, 128, (E, 2 * I, H), generator=g, dtype=torch.int8).to(dev)
    w2 = torch.randint(-127, 128, (E, H, I), generator=g, dtype=torch.int8).to(dev)
    s13, s2 = torch.full((E, 2 * I), 0.001, device=dev), torch.full((E, H), 0.002, device=dev)
    offsets = torch.tensor([0, 40, 60], dtype=torch.int32)          # the last six rows are padding

    q, x_scale, norm, _ = aclnn.moe_add_rms_norm_quant(*_on(dev, residual, gamma))
    logits = aclnn.moe_router_logits(norm, router.to(dev))
    weight, idx, _ = aclnn.moe_gating_top_k_grouped(logits, k, score_type=1, renorm=1, routed_scaling_factor=2.5)
    loss, counts, rows, prob = aclnn.moe_balance_loss(logits, idx, offsets.to(dev), score_type=1)
    ffn = pkg.MoeFfnW8A8(w13, s13, w2, s2)
    out = ffn.forward(q, x_scale, idx, weight).clone()              # its own buffer, written again below
    # what each pick's expert answers by itself
    answers = torch.stack([ffn.forward(q, x_scale, idx, torch.nn.functional.one_hot(torch.full((T,), j), k).float().to(dev)).clone() for j in range(k)], 1)
    total, closed, _, _, post_rstd, pre_rstd = aclnn.moe_sandwich_norm(out, residual.to(dev), post.to(dev), gate.to(dev), pre.to(dev), branch_scale=0.5,
                                                                       output_rstd=True)
    d_total, d_closed = [torch.randn((T, H), generator=g).to(torch.bfloat16) for _ in range(2)]
    d_loss = torch.tensor([0.8, 1.3])
    out_grad, residual_grad, post_grad, gate_grad, pre_grad = aclnn.moe_sandwich_norm_grad(
        out, total, *_on(dev, d_total, d_closed, post, gate, pre), post_rstd, pre_rstd, branch_scale=0.5)
    y_grad = (answers.float() * out_grad.float()[:, None]).sum(-1)
    logits_grad = aclnn.moe_gating_top_k_grouped_grad(logits, idx, y_grad, d_loss.to(dev), counts, rows, offsets.to(dev), score_type=1, renorm=1,
                                                      routed_scaling_factor=2.5)
    router_grad = logits_grad.t() @ norm.float()

    leaves = [t.double().requires_grad_(True) for t in (router, post, gate, pre)]
    r, p, ga, pr = leaves
    x = norm.cpu().double()
    scores = torch.sigmoid(x @ r.t())
    picked = torch.gather(scores, 1, idx.cpu().long())
    picked = 2.5 * picked / picked.sum(1, keepdim=True)
    _within(weight, picked.detach(), 1e-5 * picked.detach())
    mixed = (picked[:, :, None] * answers.cpu().double()).sum(1)
    # each answer was rounded by itself, their sum once
    _within(out, mixed.detach(), 2 * 2.0 ** -8 * (picked.detach()[:, :, None] * answers.cpu().double().abs()).sum(1))
    rms = lambda t: t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6)
    s = residual.double() + 0.5 * ga * rms(mixed) * p
    n = rms(s) * pr
    value = (s * d_total.double()).sum() + (n * d_closed.double()).sum()
    shares = scores / scores.sum(1, keepdim=True)
    want_loss = torch.stack([(counts[i].cpu().double() * shares[lo:hi].mean(0)).sum() * E / (k * (hi - lo)) for i, (lo, hi) in enumerate([(0, 40), (40, 60)])])
    _within(loss, want_loss.detach(), 1e-5 * want_loss.detach())
    value = value + (want_loss * d_loss.double()).sum()
    wants = torch.autograd.grad(value, leaves)
    # bf16 roundings on the way (experts' mix, sum, both rows' gradients): 2^-8 each, in the 2-norm of sums of many terms of either sign
    for got, want in zip((router_grad, post_grad, gate_grad, pre_grad), wants):
        assert float((got.cpu().double() - want).norm()) <= 4 * 2.0 ** -8 * float(want.norm())
