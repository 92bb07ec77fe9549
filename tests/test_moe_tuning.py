"""What the operators for tuning the router and the norms refuse, and what they ask for, without a GPU: aclnnMoeBalanceLoss,
aclnnMoeGatingTopKGroupedGrad, aclnnMoeSandwichNorm, aclnnMoeSandwichNormGrad.  First phases never touch device memory, so fake addresses suffice."""
import ctypes

import pytest
import torch

from test_moe_front import BF16, BOOL, F16, F32, I8, I32, I64, INVALID, NULLPTR, _handles, _status, _T


def _maker(aclnn, over):
    """Tensors by name: ``name`` (extents, None for an absent one), ``name_dtype``, ``name_strides`` and ``name_at`` override what is given."""
    def make(name, shape, dtype):
        shape = over.get(name, shape)
        if shape is None:
            return None
        return _T(aclnn, shape, over.get(name + "_dtype", dtype), over.get(name + "_strides"), over.get(name + "_at"))
    return make


def _check_invalid(aclnn, api, args, fragment):
    code, msg = _status(aclnn, api, args)
    assert code == INVALID and fragment in msg, (code, msg)


# ------------------------------------------------------------------------------------------------ balance
def _balance(aclnn, shape=(6, 16), k=4, score=0, dtype=F32, sequences=None, **over):
    make = _maker(aclnn, over)
    S = 1 if sequences is None else sequences
    x, idx = make("x", shape, dtype), make("idx", tuple(shape[:-1]) + (k,), I32)
    off = make("off", None if sequences is None else (sequences + 1,), I32)
    return _handles(x, idx, off) + [score] + _handles(make("loss", (S,), F32), make("counts", (S, shape[-1]), I32), make("rows", (S,), I32),
                                                     make("prob", (S, shape[-1]), F32))


def test_balance_valid(aclnn):
    for kw in [dict(), dict(score=1), dict(dtype=BF16), dict(dtype=F16), dict(prob=None), dict(sequences=3), dict(sequences=3, off_dtype=I64),
               dict(shape=(2, 3, 16)), dict(shape=(0, 16)), dict(shape=(1, 1), k=1), dict(shape=(5, 2048), k=64), dict(sequences=1),
               dict(shape=(0, 16), sequences=2), dict(shape=(6, 4), k=9)]:
        assert _status(aclnn, "aclnnMoeBalanceLoss", _balance(aclnn, **kw))[0] == 0, kw


def test_balance_workspace(aclnn):
    """A short batch of one sequence needs none; otherwise a table of a piece per chunk and sequence, not of a row each."""
    assert _status(aclnn, "aclnnMoeBalanceLoss", _balance(aclnn, shape=(64, 256))) == (0, 0)
    need = _status(aclnn, "aclnnMoeBalanceLoss", _balance(aclnn, shape=(16384, 256), sequences=8))[1]
    assert 8 * 256 * 8 <= need <= 8 * 300 * 300
    need = _status(aclnn, "aclnnMoeBalanceLoss", _balance(aclnn, shape=(1 << 26, 8)))[1]
    assert need <= (1 << 26) // 4096 * 8 * 16


@pytest.mark.parametrize("kw,fragment", [
    (dict(dtype=I8), "FLOAT, FLOAT16 or BF16"),
    (dict(shape=(16,), idx=(4,)), "rank 2 or 3"),
    (dict(shape=(6, 0), counts=(1, 0), prob=(1, 0)), "1 to 2048 experts"),
    (dict(shape=(6, 2049)), "1 to 2048 experts"),
    (dict(shape=(-6, 16)), "negative extent"),
    (dict(shape=(65536, 1025, 8)), "more than 67108864 rows"),
    (dict(idx_dtype=I64), "expertIdx"),
    (dict(idx=(5, 4)), "expertIdx [5,4]"),
    (dict(idx=(6,)), "expertIdx [6]"),
    (dict(k=0), "1 to 64"),
    (dict(k=65), "1 to 64"),
    (dict(score=2), "scoreType (=2)"),
    (dict(score=-1), "scoreType (=-1)"),
    (dict(sequences=3, off_dtype=F32), "seqOffsets must be INT32 or INT64"),
    (dict(sequences=3, off=(4, 1)), "seqOffsets [4,1]"),
    (dict(off=(1,)), "seqOffsets [1]"),
    (dict(off=((1 << 20) + 2,)), "1 to 1048576 sequences"),
    (dict(sequences=3, loss=(1,)), "lossOut [1]"),
    (dict(loss=()), "lossOut []"),
    (dict(loss_dtype=BF16), "lossOut"),
    (dict(rows_dtype=I64), "rowsOut"),
    (dict(rows=(2,)), "rowsOut [2]"),
    (dict(counts_dtype=I64), "countsOut"),
    (dict(counts=(16,)), "countsOut [16]"),
    (dict(prob_dtype=BF16), "probOut"),
    (dict(prob=(1, 15)), "probOut [1,15]"),
    (dict(counts_strides=[16, 2]), "outputs must be contiguous"),
    (dict(x_strides=[16, -1]), "negative strides"),
    (dict(counts_at=0x77000000, prob_at=0x77000000), "two outputs share memory"),
    (dict(x_at=0x77000000, prob_at=0x77000010), "shares memory with an input"),
    (dict(idx_at=0x77000000, counts_at=0x77000000), "shares memory with an input"),
    (dict(sequences=3, off_at=0x77000000, rows_at=0x77000004), "shares memory with an input"),
])
def test_balance_invalid(aclnn, kw, fragment):
    _check_invalid(aclnn, "aclnnMoeBalanceLoss", _balance(aclnn, **kw), fragment)


def test_balance_counts_fit_their_type(aclnn):
    """One expert may be every id of every row: as many as INT32 holds are taken, no more."""
    for rows, k in [((1 << 25) - 1, 64), (1 << 26, 31)]:
        assert _status(aclnn, "aclnnMoeBalanceLoss", _balance(aclnn, shape=(rows, 4), k=k, x_at=1 << 45, idx_at=1 << 46))[0] == 0
    for rows, k in [(1 << 25, 64), (1 << 26, 32), ((1 << 31) // 63 + 1, 63)]:
        _check_invalid(aclnn, "aclnnMoeBalanceLoss", _balance(aclnn, shape=(rows, 4), k=k, sequences=3), "2147483647 ids")


def test_balance_nulls(aclnn):
    for pos in (0, 1, 4, 5, 6):
        args = _balance(aclnn)
        args[pos] = None
        assert _status(aclnn, "aclnnMoeBalanceLoss", args)[0] == NULLPTR, pos
    for kw in [dict(x_at=0), dict(loss_at=0), dict(sequences=2, off_at=0)]:
        assert _status(aclnn, "aclnnMoeBalanceLoss", _balance(aclnn, **kw))[0] == NULLPTR, kw


# ------------------------------------------------------------------------------------------------ gradient of the choice
def _grad(aclnn, shape=(6, 16), k=4, score=0, renorm=1, factor=2.5, eps=1e-20, dtype=F32, sequences=None, weights=True, balance=True, **over):
    make = _maker(aclnn, over)
    S = 1 if sequences is None else sequences
    picked = tuple(shape[:-1]) + (k,)
    x, idx = make("x", shape, dtype), make("idx", picked, I32)
    dy = make("dy", picked if weights else None, dtype)
    tables = [make(name, extents if balance else None, kind) for name, extents, kind in [("dl", (S,), F32), ("counts", (S, shape[-1]), I32), ("rows", (S,), I32)]]
    off = make("off", None if sequences is None else (sequences + 1,), I32)
    return _handles(x, idx, dy, *tables, off) + [score, renorm, factor, eps] + _handles(make("dx", shape, dtype))


def test_grad_valid(aclnn):
    for kw in [dict(), dict(weights=False), dict(balance=False), dict(score=1, renorm=0), dict(dtype=BF16), dict(dtype=BF16, dy_dtype=F32), dict(dtype=F16, dx_dtype=F32),
               dict(sequences=3), dict(sequences=3, off_dtype=I64), dict(shape=(2, 3, 16)), dict(shape=(0, 16)), dict(shape=(3, 2048), k=64),
               dict(factor=-1.0, eps=0.0)]:
        assert _status(aclnn, "aclnnMoeGatingTopKGroupedGrad", _grad(aclnn, **kw)) == (0, 0), kw
    assert _status(aclnn, "aclnnMoeGatingTopKGroupedGrad", _grad(aclnn, x_strides=[32, 1], dy_strides=[1, 6])) == (0, 768)


@pytest.mark.parametrize("kw,fragment", [
    (dict(dtype=I32), "FLOAT, FLOAT16 or BF16"),
    (dict(shape=(6, 2049)), "1 to 2048 experts"),
    (dict(idx_dtype=I64), "expertIdx"),
    (dict(k=65), "1 to 64"),
    (dict(score=3), "scoreType (=3)"),
    (dict(renorm=2), "renorm (=2)"),
    (dict(factor=float("nan")), "routedScalingFactor"),
    (dict(factor=1e39), "routedScalingFactor"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(dy=(6, 5)), "yGrad [6,5]"),
    (dict(dy_dtype=F16), "yGrad"),
    (dict(dl=(2,)), "lossGrad [2]"),
    (dict(dl_dtype=F16), "lossGrad"),
    (dict(counts=(1, 15)), "counts [1,15]"),
    (dict(counts_dtype=I64), "counts"),
    (dict(rows=(1, 1)), "rows [1,1]"),
    (dict(sequences=3, rows=(1,)), "rows [1]"),
    (dict(sequences=3, balance=False), "seqOffsets belongs to lossGrad"),
    (dict(dx=(6, 15)), "xGradOut [6,15]"),
    (dict(dx_dtype=BF16), "xGradOut"),
    (dict(dx_strides=[1, 6]), "outputs must be contiguous"),
    (dict(x_at=0x77000000, dx_at=0x77000000), "shares memory with an input"),
    (dict(dy_at=0x77000000, dx_at=0x77000000), "shares memory with an input"),
])
def test_grad_invalid(aclnn, kw, fragment):
    _check_invalid(aclnn, "aclnnMoeGatingTopKGroupedGrad", _grad(aclnn, **kw), fragment)


def test_grad_nulls(aclnn):
    for pos in (0, 1, 11):
        args = _grad(aclnn)
        args[pos] = None
        assert _status(aclnn, "aclnnMoeGatingTopKGroupedGrad", args)[0] == NULLPTR, pos
    for kw in [dict(dl=None), dict(counts=None), dict(rows=None), dict(weights=False, balance=False), dict(x_at=0), dict(dx_at=0)]:
        assert _status(aclnn, "aclnnMoeGatingTopKGroupedGrad", _grad(aclnn, **kw))[0] == NULLPTR, kw


# ------------------------------------------------------------------------------------------------ sandwich norm
GATES = {"none": lambda shape: None, "channel": lambda shape: shape[-1:], "row": lambda shape: tuple(shape[:-1]) + (1,), "each": lambda shape: shape}


def _sandwich(aclnn, shape=(6, 24), dtype=BF16, post=True, pre=True, gate="none", smooth=False, gate_type=0, alpha=1.0, beta=1.0, eps=1e-6, quantise=True,
              **over):
    make = _maker(aclnn, over)
    rows = shape[:-1]
    ins = [make("x", shape, dtype), make("res", shape, dtype), make("post_gamma", shape[-1:] if post else None, dtype), make("g", GATES[gate](shape), dtype),
           make("pre_gamma", shape[-1:] if pre else None, dtype), make("sm", shape[-1:] if smooth else None, F32)]
    quantise = quantise and pre
    outs = [make("sum", shape, dtype), make("norm", shape if pre else None, dtype), make("y", shape if quantise else None, I8),
            make("scale", rows if quantise else None, F32), make("post_rstd", rows if post else None, F32), make("pre_rstd", rows if pre else None, F32)]
    return _handles(*ins) + [gate_type, alpha, beta, eps] + _handles(*outs)


def test_sandwich_valid(aclnn):
    for kw in [dict(), dict(dtype=F32), dict(dtype=F16, post_gamma_dtype=F32, pre_gamma_dtype=F32), dict(post=False), dict(pre=False), dict(pre=False, post=False),
               dict(gate="channel"), dict(gate="row"), dict(gate="row", g_dtype=F32), dict(gate="each", gate_type=1), dict(smooth=True), dict(quantise=False),
               dict(post=False, pre=False, gate="channel", g_dtype=F32), dict(norm=None), dict(post_rstd=None, pre_rstd=None), dict(shape=(2, 3, 24), gate="row"),
               dict(shape=(0, 24)), dict(shape=(1, 1), gate="each"), dict(x_at=0x77000000, sum_at=0x77000000), dict(res_at=0x77000000, sum_at=0x77000000),
               dict(alpha=0.0, beta=-2.0, eps=0.0), dict(shape=(24, 24), gate="channel")]:
        assert _status(aclnn, "aclnnMoeSandwichNorm", _sandwich(aclnn, **kw)) == (0, 0), kw
    assert _status(aclnn, "aclnnMoeSandwichNorm", _sandwich(aclnn, x_strides=[48, 1], gate="channel", g_strides=[2])) == (0, 768)


@pytest.mark.parametrize("kw,fragment", [
    (dict(dtype=I8), "FLOAT, FLOAT16 or BF16"),
    (dict(shape=(24,)), "rank 2 or 3"),
    (dict(shape=(6, 0)), "last extent of x is zero"),
    (dict(shape=(-6, 24)), "negative extent"),
    (dict(res=(5, 24)), "residual [5,24]"),
    (dict(res_dtype=F32), "residual"),
    (dict(post_gamma=(23,)), "postGamma [23]"),
    (dict(pre_gamma=(24, 1)), "preGamma [24,1]"),
    (dict(pre_gamma_dtype=F16), "of x's type or FLOAT"),
    (dict(pre_gamma_dtype=F32), "must have one type"),
    (dict(gate="channel", g_dtype=F32), "of the gammas' type"),
    (dict(gate="channel", post=False, pre=False, g_dtype=F16), "of x's type or FLOAT"),
    (dict(gate="row", g_dtype=I32), "of x's type or FLOAT"),
    (dict(gate="each", g_dtype=F32), "gate [6,24]"),
    (dict(gate="each", g=(6, 23)), "gate [6,23]"),
    (dict(gate="each", g=(6,)), "gate [6]"),
    (dict(gate_type=2), "gateType (=2)"),
    (dict(alpha=float("inf")), "residualScale"),
    (dict(beta=float("nan")), "branchScale"),
    (dict(eps=-1.0), "epsilon"),
    (dict(smooth=True, sm=(25,)), "smoothScale must be FLOAT [24]"),
    (dict(smooth=True, sm_dtype=BF16), "smoothScale must be FLOAT [24]"),
    (dict(smooth=True, quantise=False), "smoothScale goes into yOut"),
    (dict(sum_dtype=F32), "sumOut"),
    (dict(norm=(6, 25)), "normOut [6,25]"),
    (dict(y_dtype=BF16), "yOut"),
    (dict(scale=(6, 1)), "scaleOut [6,1]"),
    (dict(post_rstd=(5,)), "postRstdOut [5]"),
    (dict(pre_rstd_dtype=BF16), "preRstdOut"),
    (dict(pre=False, norm=(6, 24)), "the norm with preGamma"),
    (dict(pre=False, pre_rstd=(6,)), "the norm with preGamma"),
    (dict(post=False, post_rstd=(6,)), "the norm with postGamma"),
    (dict(sum_strides=[48, 1]), "outputs must be contiguous"),
    (dict(norm_strides=[48, 1]), "outputs must be contiguous"),
    (dict(x_at=0x77000000, sum_at=0x77000030), "shares memory with an input"),
    (dict(x_at=0x77000000, norm_at=0x77000000), "shares memory with an input"),
    (dict(gate="each", g_at=0x77000000, sum_at=0x77000000), "shares memory with an input"),
    (dict(sum_at=0x77000000, norm_at=0x77000000), "two outputs share memory"),
    (dict(scale_at=0x77000000, pre_rstd_at=0x77000004), "two outputs share memory"),
])
def test_sandwich_invalid(aclnn, kw, fragment):
    _check_invalid(aclnn, "aclnnMoeSandwichNorm", _sandwich(aclnn, **kw), fragment)


def test_sandwich_nulls(aclnn):
    for pos in (0, 1, 10):
        args = _sandwich(aclnn)
        args[pos] = None
        assert _status(aclnn, "aclnnMoeSandwichNorm", args)[0] == NULLPTR, pos
    for kw in [dict(y=None), dict(scale=None), dict(norm=None, y=None, scale=None, pre_rstd=None), dict(x_at=0), dict(sum_at=0), dict(post_rstd_at=0)]:
        assert _status(aclnn, "aclnnMoeSandwichNorm", _sandwich(aclnn, **kw))[0] == NULLPTR, kw


def _sandwich_grad(aclnn, shape=(6, 24), dtype=BF16, post=True, pre=True, gate="none", gate_type=0, alpha=1.0, beta=1.0, **over):
    make = _maker(aclnn, over)
    rows, H = shape[:-1], shape[-1:]
    ins = [make("x", shape, dtype), make("sum", shape if pre else None, dtype), make("ds", shape, dtype), make("dn", shape if pre else None, dtype),
           make("post_gamma", H if post else None, dtype), make("g", GATES[gate](shape), dtype), make("pre_gamma", H if pre else None, dtype),
           make("post_rstd", rows if post else None, F32), make("pre_rstd", rows if pre else None, F32)]
    outs = [make("dx", shape, dtype), make("dres", shape, dtype), make("dpost", H if post else None, F32),
            make("dg", GATES[gate](shape), dtype if gate == "each" else F32), make("dpre", H if pre else None, F32)]
    return _handles(*ins) + [gate_type, alpha, beta] + _handles(*outs)


def test_sandwich_grad_valid(aclnn):
    for kw in [dict(), dict(dtype=F32), dict(dtype=F16, post_gamma_dtype=F32, pre_gamma_dtype=F32), dict(post=False), dict(pre=False), dict(pre=False, sum=(6, 24)),
               dict(gate="channel"), dict(gate="row", g_dtype=F32), dict(gate="each", gate_type=1), dict(ds=None), dict(dx=None, dres=None), dict(dpost=None, dpre=None),
               dict(gate="row", dg=None), dict(shape=(2, 3, 24), gate="row"), dict(shape=(0, 24)), dict(post=False, pre=False, gate="channel", g_dtype=F32)]:
        assert _status(aclnn, "aclnnMoeSandwichNormGrad", _sandwich_grad(aclnn, **kw))[0] == 0, kw
    assert _status(aclnn, "aclnnMoeSandwichNormGrad", _sandwich_grad(aclnn, post=False, pre=False)) == (0, 0)
    need = _status(aclnn, "aclnnMoeSandwichNormGrad", _sandwich_grad(aclnn, shape=(8192, 7168)))[1]
    assert 2 * 256 * 7168 * 4 <= need <= 2 * 1024 * 7168 * 4


@pytest.mark.parametrize("kw,fragment", [
    (dict(dtype=I8), "FLOAT, FLOAT16 or BF16"),
    (dict(shape=(6, 0)), "last extent of x is zero"),
    (dict(shape=(6, (1 << 24) + 1)), "up to 16777216"),
    (dict(sum=(5, 24)), "sum [5,24]"),
    (dict(ds_dtype=F32), "sumGrad"),
    (dict(dn=(6, 23)), "normGrad [6,23]"),
    (dict(post_rstd=(5,)), "postRstd [5]"),
    (dict(pre_rstd_dtype=BF16), "preRstd"),
    (dict(gate="channel", g_dtype=F32), "of the gammas' type"),
    (dict(gate_type=-1), "gateType (=-1)"),
    (dict(alpha=float("nan")), "residualScale"),
    (dict(dx=(6, 25)), "xGradOut [6,25]"),
    (dict(dres_dtype=F32), "residualGradOut"),
    (dict(post=False, dpost=(24,)), "postGammaGradOut is given without postGamma"),
    (dict(pre=False, dpre=(24,)), "preGammaGradOut is given without preGamma"),
    (dict(dg=(24,)), "gateGradOut is given without a gate"),
    (dict(dpost_dtype=BF16), "postGammaGradOut"),
    (dict(dpre=(23,)), "preGammaGradOut [23]"),
    (dict(gate="channel", dg_dtype=BF16), "gateGradOut"),
    (dict(gate="row", dg=(6,)), "gateGradOut [6]"),
    (dict(gate="each", dg_dtype=F32), "gateGradOut"),
    (dict(dx_strides=[48, 1]), "outputs must be contiguous"),
    (dict(ds_at=0x77000000, dres_at=0x77000000), "shares memory with an input"),
    (dict(dx_at=0x77000000, dres_at=0x77000000), "two outputs share memory"),
])
def test_sandwich_grad_invalid(aclnn, kw, fragment):
    _check_invalid(aclnn, "aclnnMoeSandwichNormGrad", _sandwich_grad(aclnn, **kw), fragment)


def test_sandwich_grad_nulls(aclnn):
    args = _sandwich_grad(aclnn)
    args[0] = None
    assert _status(aclnn, "aclnnMoeSandwichNormGrad", args)[0] == NULLPTR
    for kw in [dict(dn=None), dict(sum=None), dict(pre_gamma=None, dpre=None), dict(pre_rstd=None), dict(post_rstd=None), dict(post_gamma=None, dpost=None),
               dict(pre=False, ds=None), dict(dx=None, dres=None, dpost=None, dpre=None), dict(x_at=0), dict(dx_at=0)]:
        assert _status(aclnn, "aclnnMoeSandwichNormGrad", _sandwich_grad(aclnn, **kw))[0] == NULLPTR, kw


# ------------------------------------------------------------------------------------------------ all
def test_second_phases_check_their_workspace(aclnn):
    lib = aclnn.lib()
    for api, args in [("aclnnMoeBalanceLoss", _balance(aclnn, sequences=2)), ("aclnnMoeGatingTopKGroupedGrad", _grad(aclnn, x_strides=[48, 1])),
                      ("aclnnMoeSandwichNorm", _sandwich(aclnn, x_strides=[48, 1])), ("aclnnMoeSandwichNormGrad", _sandwich_grad(aclnn))]:
        for workspace, short in [(None, 0), (0x1000, 1)]:
            ws, ex = ctypes.c_uint64(0), ctypes.c_void_p(None)
            assert getattr(lib, api + "GetWorkspaceSize")(*args, ctypes.byref(ws), ctypes.byref(ex)) == 0 and ws.value > 0
            assert getattr(lib, api)(workspace, ws.value - short, ex, None) == (NULLPTR if workspace is None else INVALID), api
        assert getattr(lib, api)(None, 0, None, None) == NULLPTR
    for api, args in [("aclnnMoeBalanceLoss", _balance(aclnn, sequences=2)), ("aclnnMoeSandwichNormGrad", _sandwich_grad(aclnn))]:
        ws, ex = ctypes.c_uint64(0), ctypes.c_void_p(None)
        assert getattr(lib, api + "GetWorkspaceSize")(*args, ctypes.byref(ws), ctypes.byref(ex)) == 0
        assert getattr(lib, api)(0x1008, ws.value, ex, None) == INVALID and "16-byte" in aclnn.last_error()


def test_host_tensors_are_refused(aclnn):
    x, idx = torch.zeros((2, 16)), torch.zeros((2, 2), dtype=torch.int32)
    for call in [lambda: aclnn.moe_balance_loss(x, idx), lambda: aclnn.moe_gating_top_k_grouped_grad(x, idx, y_grad=torch.zeros(2, 2)),
                 lambda: aclnn.moe_sandwich_norm(x, x, post_gamma=torch.ones(16)), lambda: aclnn.moe_sandwich_norm_grad(x, sum_grad=x)]:
        with pytest.raises(aclnn.AclnnError, match="not on the current GPU") as e:
            call()
        assert e.value.code == INVALID
