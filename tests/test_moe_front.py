"""What the operators in front of the expert FFN refuse, and what they ask for, without a GPU: aclnnMoeAddRmsNormQuant,
aclnnMoeRouterLogits, aclnnMoeGatingTopKGrouped.  First phases never touch device memory, so fake addresses suffice."""
import ctypes
import math
import random
import struct

import pytest
import torch

NULLPTR, INVALID = 161001, 161002
F32, F16, I8, I32, I64, BOOL, BF16 = 0, 1, 2, 3, 9, 12, 27


class _T:
    """Descriptor over a fake device address, far from every other one's."""
    _next = 0x100000000

    def __init__(self, aclnn, shape, dtype, strides=None, at=None):
        if at is None:
            _T._next += 0x100000000
            at = _T._next
        self.at = at
        self.h = aclnn.create_tensor(list(shape), dtype, at, strides)


def _status(aclnn, api, args):
    try:
        return 0, aclnn.workspace_size(api, args)
    except aclnn.AclnnError as e:
        assert e.message, "an error status must come with a message"
        return e.code, e.message


def _handles(*tensors):
    return [t.h if t is not None else None for t in tensors]


# ------------------------------------------------------------------------------------------------ norm
def _norm(aclnn, shape=(6, 24), dtype=BF16, residual=True, smooth=False, eps=1e-6, **over):
    make = lambda name, default, kind: None if over.get(name, ()) is None else _T(
        aclnn, over.get(name, default), over.get(name + "_dtype", kind), over.get(name + "_strides"), over.get(name + "_at"))
    x = make("x", shape, dtype)
    res = make("res", shape, dtype) if residual else None
    gamma = make("gamma", shape[-1:], dtype)
    sm = make("sm", shape[-1:], F32) if smooth else None
    y, scale = make("y", shape, I8), make("scale", shape[:-1], F32)
    norm, total = make("norm", shape, dtype), make("sum", shape, dtype)
    return _handles(x, res, gamma, sm) + [eps] + _handles(y, scale, norm, total)


def test_norm_valid(aclnn):
    for kw in [dict(), dict(dtype=F32), dict(dtype=F16, gamma_dtype=F32), dict(residual=False), dict(smooth=True), dict(norm=None),
               dict(sum=None), dict(y=None, scale=None), dict(shape=(2, 3, 24)), dict(shape=(0, 24)), dict(shape=(1, 1)), dict(eps=0.0),
               dict(shape=(2, 0, 24)), dict(x_at=0x77000000, sum_at=0x77000000), dict(res_at=0x77000000, sum_at=0x77000000)]:
        assert _status(aclnn, "aclnnMoeAddRmsNormQuant", _norm(aclnn, **kw)) == (0, 0), kw


@pytest.mark.parametrize("kw,fragment", [
    (dict(dtype=I8), "FLOAT, FLOAT16 or BF16"),
    (dict(shape=(24,)), "rank 2 or 3"),
    (dict(shape=(2, 2, 2, 24)), "rank 2 or 3"),
    (dict(shape=(6, 0)), "last extent of x is zero"),
    (dict(shape=(-6, 24)), "negative extent"),
    (dict(shape=(65536, 1025, 1)), "more than 67108864 rows"),
    (dict(gamma=(23,)), "gamma must be [24]"),
    (dict(gamma_dtype=F16), "of x's type or FLOAT"),
    (dict(gamma=(24, 1)), "gamma must be [24]"),
    (dict(smooth=True, sm=(25,)), "smoothScale must be FLOAT [24]"),
    (dict(smooth=True, sm_dtype=BF16), "smoothScale must be FLOAT [24]"),
    (dict(eps=-1e-6), "epsilon"),
    (dict(eps=float("nan")), "epsilon"),
    (dict(eps=float("inf")), "epsilon"),
    (dict(res=(5, 24)), "residual [5,24]"),
    (dict(res_dtype=F32), "residual"),
    (dict(norm=(6, 25)), "normOut [6,25]"),
    (dict(norm_dtype=F32), "normOut"),
    (dict(sum=(6, 25)), "sumOut [6,25]"),
    (dict(y_dtype=BF16), "yOut"),
    (dict(y=(6, 23)), "yOut [6,23]"),
    (dict(scale=(6, 1)), "scaleOut [6,1]"),
    (dict(scale_dtype=F16), "scaleOut"),
    (dict(y=None, scale=None, smooth=True), "smoothScale goes into yOut"),
    (dict(norm_strides=[48, 1]), "outputs must be contiguous"),
    (dict(y_strides=[1, 6]), "outputs must be contiguous"),
    (dict(x_strides=[24, -1]), "negative strides"),
    (dict(x_at=0x77000000, norm_at=0x77000000), "shares memory with an input"),      # only the sum may be in place
    (dict(x_at=0x77000000, sum_at=0x77000030), "shares memory with an input"),       # one row further on
    (dict(gamma_at=0x77000000, scale_at=0x77000004), "shares memory with an input"),
    (dict(norm_at=0x77000000, sum_at=0x77000000), "two outputs share memory"),
])
def test_norm_invalid(aclnn, kw, fragment):
    code, msg = _status(aclnn, "aclnnMoeAddRmsNormQuant", _norm(aclnn, **kw))
    assert code == INVALID and fragment in msg, (code, msg)


def test_norm_nulls(aclnn):
    for pos in (0, 2):
        args = _norm(aclnn)
        args[pos] = None
        assert _status(aclnn, "aclnnMoeAddRmsNormQuant", args)[0] == NULLPTR, pos
    for kw in [dict(y=None), dict(scale=None), dict(y=None, scale=None, norm=None), dict(x_at=0), dict(norm_at=0)]:
        assert _status(aclnn, "aclnnMoeAddRmsNormQuant", _norm(aclnn, **kw))[0] == NULLPTR, kw


def test_norm_stages_strided_inputs(aclnn):
    assert _status(aclnn, "aclnnMoeAddRmsNormQuant", _norm(aclnn, x_strides=[48, 1])) == (0, 512)
    assert _status(aclnn, "aclnnMoeAddRmsNormQuant", _norm(aclnn, x_strides=[48, 1], gamma_strides=[2])) == (0, 768)


# ------------------------------------------------------------------------------------------------ logits
def _logits(aclnn, shape=(6, 24), experts=5, dtype=BF16, **over):
    make = lambda name, default, kind: _T(aclnn, over.get(name, default), over.get(name + "_dtype", kind), over.get(name + "_strides"),
                                          over.get(name + "_at"))
    return _handles(make("x", shape, dtype), make("w", (experts, shape[-1]), dtype), make("out", tuple(shape[:-1]) + (experts,), F32))


def test_logits_valid(aclnn):
    for kw in [dict(), dict(dtype=F32), dict(dtype=F16), dict(w_dtype=F32), dict(dtype=F16, w_dtype=F32), dict(shape=(2, 3, 24)),
               dict(shape=(0, 24)), dict(shape=(1, 1), experts=1), dict(shape=(4096, 7168), experts=256), dict(experts=4096)]:
        assert _status(aclnn, "aclnnMoeRouterLogits", _logits(aclnn, **kw))[0] == 0, kw


@pytest.mark.parametrize("kw,fragment", [
    (dict(dtype=I8), "FLOAT, FLOAT16 or BF16"),
    (dict(shape=(24,)), "rank 2 or 3"),
    (dict(shape=(6, 0)), "last extent of x is zero"),
    (dict(shape=(-6, 24)), "negative extent"),
    (dict(w_dtype=F16), "weight must be of x's type or FLOAT"),
    (dict(w=(5, 23)), "weight [5,23]"),
    (dict(w=(24,)), "weight [24]"),
    (dict(experts=0), "takes 1 to 4096"),
    (dict(experts=4097), "takes 1 to 4096"),
    (dict(out=(6, 6)), "logitsOut [6,6]"),
    (dict(out_dtype=BF16), "logitsOut"),
    (dict(out_strides=[1, 6]), "outputs must be contiguous"),
    (dict(x_at=0x77000000, out_at=0x77000008), "shares memory with an input"),
])
def test_logits_invalid(aclnn, kw, fragment):
    code, msg = _status(aclnn, "aclnnMoeRouterLogits", _logits(aclnn, **kw))
    assert code == INVALID and fragment in msg, (code, msg)


def test_logits_nulls(aclnn):
    for pos in range(3):
        args = _logits(aclnn)
        args[pos] = None
        assert _status(aclnn, "aclnnMoeRouterLogits", args)[0] == NULLPTR, pos
    assert _status(aclnn, "aclnnMoeRouterLogits", _logits(aclnn, w_at=0))[0] == NULLPTR


# ------------------------------------------------------------------------------------------------ gating
def _gating(aclnn, shape=(6, 16), k=4, k_group=2, groups=4, mode=1, score=1, renorm=1, factor=2.5, eps=1e-20, dtype=F32, bias=True,
            finished=False, scores=False, **over):
    make = lambda name, default, kind: _T(aclnn, over.get(name, default), over.get(name + "_dtype", kind), over.get(name + "_strides"),
                                          over.get(name + "_at"))
    x = make("x", shape, dtype)
    b = make("b", shape[-1:], F32) if bias else None
    fin = make("fin", shape[:-1], BOOL) if finished else None
    picked = tuple(shape[:-1]) + (max(k, 0),)
    y, idx = make("y", picked, dtype), make("idx", picked, I32)
    sc = make("scores", shape, F32) if scores else None
    return _handles(x, b, fin) + [k, k_group, groups, mode, score, renorm, factor, eps] + _handles(y, idx, sc)


def test_gating_valid(aclnn):
    for kw in [dict(), dict(bias=False), dict(score=0), dict(renorm=0), dict(mode=0), dict(dtype=BF16), dict(dtype=F16, y_dtype=F32),
               dict(finished=True, scores=True), dict(shape=(2, 3, 16), finished=True), dict(shape=(0, 16)), dict(k=8), dict(groups=1, k_group=1, k=16),
               dict(groups=16, k_group=4, mode=0), dict(groups=16, k_group=16), dict(shape=(3, 2048), groups=1, k_group=1, k=64),
               dict(factor=-1.0, eps=0.0)]:
        assert _status(aclnn, "aclnnMoeGatingTopKGrouped", _gating(aclnn, **kw)) == (0, 0), kw


@pytest.mark.parametrize("kw,fragment", [
    (dict(dtype=I8), "FLOAT, FLOAT16 or BF16"),
    (dict(shape=(16,)), "rank 2 or 3"),
    (dict(shape=(6, 0), groups=1, k_group=1), "1 to 2048 experts"),
    (dict(shape=(2, 2049), groups=1, k_group=1), "1 to 2048 experts"),
    (dict(shape=(-6, 16)), "negative extent"),
    (dict(groups=5), "must divide the 16 experts"),
    (dict(groups=0), "must divide the 16 experts"),
    (dict(groups=32), "must divide the 16 experts"),
    (dict(k_group=0), "kGroup (=0)"),
    (dict(k_group=5), "kGroup (=5)"),
    (dict(mode=2), "groupSelectMode (=2)"),
    (dict(groups=16, k_group=4, mode=1), "a group, which has one"),
    (dict(score=2), "scoreType (=2)"),
    (dict(renorm=2), "renorm (=2)"),
    (dict(k=0), "k (=0)"),
    (dict(k=9), "at most the 8 experts of the groups that stay"),
    (dict(shape=(2, 128), groups=1, k_group=1, k=65), "k (=65) must be 1 to 64"),
    (dict(factor=float("inf")), "routedScalingFactor"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(b_dtype=BF16), "bias must be FLOAT [16]"),
    (dict(b=(15,)), "bias must be FLOAT [16]"),
    (dict(finished=True, fin_dtype=I8), "finished must be BOOL"),
    (dict(finished=True, fin=(6, 1)), "finished must be BOOL"),
    (dict(y=(6, 5)), "yOut [6,5]"),
    (dict(y_dtype=F16), "yOut"),
    (dict(idx_dtype=I64), "expertIdxOut"),
    (dict(idx=(5, 4)), "expertIdxOut [5,4]"),
    (dict(scores=True, scores_dtype=F16), "scoresOut"),
    (dict(y_strides=[1, 6]), "outputs must be contiguous"),
    (dict(x_at=0x77000000, y_at=0x77000000), "shares memory with an input"),
    (dict(idx_at=0x77000000, y_at=0x77000010), "two outputs share memory"),
])
def test_gating_invalid(aclnn, kw, fragment):
    code, msg = _status(aclnn, "aclnnMoeGatingTopKGrouped", _gating(aclnn, **kw))
    assert code == INVALID and fragment in msg, (code, msg)


def test_gating_nulls(aclnn):
    for pos in (0, 11, 12):
        args = _gating(aclnn)
        args[pos] = None
        assert _status(aclnn, "aclnnMoeGatingTopKGrouped", args)[0] == NULLPTR, pos
    assert _status(aclnn, "aclnnMoeGatingTopKGrouped", _gating(aclnn, x_at=0))[0] == NULLPTR


# ------------------------------------------------------------------------------------------------ both
def test_second_phases_check_their_workspace(aclnn):
    lib = aclnn.lib()
    for api, args in [("aclnnMoeAddRmsNormQuant", _norm(aclnn, x_strides=[48, 1])), ("aclnnMoeRouterLogits", _logits(aclnn, x_strides=[48, 1])),
                      ("aclnnMoeGatingTopKGrouped", _gating(aclnn, x_strides=[48, 1]))]:
        for workspace, short in [(None, 0), (0x1000, 1)]:
            ws, ex = ctypes.c_uint64(0), ctypes.c_void_p(None)
            assert getattr(lib, api + "GetWorkspaceSize")(*args, ctypes.byref(ws), ctypes.byref(ex)) == 0 and ws.value > 0
            assert getattr(lib, api)(workspace, ws.value - short, ex, None) == (NULLPTR if workspace is None else INVALID), api
        assert getattr(lib, api)(None, 0, None, None) == NULLPTR


def _packed_logits(T, K, E, address=0x100000000):
    shapes = [(T, K), (E, K), (T, E)]
    packed = [8]
    for i, (rows, cols) in enumerate(shapes):
        packed += [2, BF16 if i < 2 else F32, address * (i + 1), rows, cols, cols, 1]
    return packed


def test_one_call_of_both_phases_enqueues_nothing_without_its_workspace(aclnn):
    packed = _packed_logits(8192, 7168, 256)
    data, needed = struct.pack("%dq" % len(packed), *packed), ctypes.c_uint64(0)
    run = aclnn.lib().opapiRunPacked
    for size in (0, 1 << 20):
        assert run(data, len(packed), 0x1000, size, None, ctypes.byref(needed)) == 0
        assert needed.value >= 2 * 8192 * 256 * 4 and needed.value > size
    assert run(data, len(packed), None, 0, None, None) == NULLPTR
    assert run(None, 0, None, 0, None, ctypes.byref(needed)) == NULLPTR
    assert run(data, len(packed) - 1, None, 0, None, ctypes.byref(needed)) == INVALID
    # the workspace's own second phase: what it asks for has to be there, and on 16 bytes
    ws, ex = ctypes.c_uint64(0), ctypes.c_void_p(None)
    lib = aclnn.lib()
    args = _logits(aclnn, shape=(8192, 7168), experts=256)
    assert lib.aclnnMoeRouterLogitsGetWorkspaceSize(*args, ctypes.byref(ws), ctypes.byref(ex)) == 0
    assert lib.aclnnMoeRouterLogits(0x1008, ws.value, ex, None) == INVALID and "16-byte" in aclnn.last_error()


def test_host_tensors_are_refused(aclnn):
    x, w = torch.zeros((2, 16)), torch.zeros((4, 16))
    for call in [lambda: aclnn.moe_add_rms_norm_quant(x, torch.ones(16)), lambda: aclnn.moe_router_logits(x, w),
                 lambda: aclnn.moe_gating_top_k_grouped(x, 2)]:
        with pytest.raises(aclnn.AclnnError, match="not on the current GPU") as e:
            call()
        assert e.value.code == INVALID


def test_the_module_that_reads_tensors_checks_what_it_is_given(aclnn):
    run, function = aclnn._binding()
    x = torch.zeros((2, 4))
    assert run(function, 0, 0, 0, 0, (8,), (x, x, x)) is x                       # not on the device
    assert run(function, 0, 0, 0, 0, (8,), (None, None, None)) == -NULLPTR
    assert run(function, 0, 0, 0, 0, (99,), ()) == -INVALID
    for args in [(function, 0, 0, 0, 0, (8,), (1, x, x)), (function, 0, 0, 0, 0, ("8",), (x,)), (function, 0, 0, 0, 0, [8], (x,)), (function,),
                 (function, 0, 0, 0, 0, (8,) * 17, ()), (function, 0, 0, 0, 0, (8,), (None,) * 17), ("f", 0, 0, 0, 0, (8,), ())]:
        with pytest.raises(TypeError):
            run(*args)
    with pytest.raises(OverflowError):
        run(function, 0, 0, 0, 0, (1 << 64,), ())


def test_a_workspace_follows_the_device(aclnn):
    """What was reserved on one device is no memory for a call on another one, however large it is."""
    space = aclnn.Workspace()
    first = space.reserve(64, torch.device("cpu"))
    assert space.reserve(16, "cpu") is first and space.reserve(64, first.device) is first
    moved = space.reserve(16, torch.device("meta"))
    assert moved.device.type == "meta" and space.tensor is moved
    assert space.reserve(32, "meta").numel() == 32
    assert space.reserve(16, "cpu").device.type == "cpu"


# ------------------------------------------------------------------------------------------------ which kernel a router product takes
ROUTER_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ROUTER_TYPES = [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32"), ("f32", "f32")]
ROUTER_SHAPES = 11        # 0 to 5 without LDS tiles, 6 to 10 with; 9 and 10 take rows of one part only

# Rows, columns and experts that between them take every kernel there is, with the columns split and whole.  Which size takes which goes by fitted costs:
# the tests below fail when a change of theirs leaves a kernel out, and the sizes are then chosen again.
ROUTER_SIZES = [(1, 130, 1), (1, 134, 2524), (1, 136, 1), (1, 136, 2127), (1, 162, 1069), (1, 184, 1033), (3, 130, 171), (3, 136, 173), (3, 24259, 505),
                (7, 22789, 131), (9, 30808, 359), (10, 26456, 77), (12, 135, 1032), (17, 7216, 2739), (20, 552, 209), (25, 152, 569), (28, 438, 154),
                (41, 17808, 432), (43, 22197, 12), (1195, 14928, 10), (2018, 503, 517), (2181, 4561, 1), (2336, 544, 3205), (2879, 820, 2724), (3286, 518, 1179),
                (5725, 512, 141), (8440, 3497, 68), (11041, 544, 272), (11180, 504, 332), (11429, 507, 133), (11753, 3536, 66), (11783, 504, 138),
                (11928, 512, 593), (12326, 530, 530), (13226, 519, 274)]


def _router_kernel(aclnn, xt, wt, rows, cols, experts):
    """(types, shape, whether rows and weights lie on 16 bytes, whether columns are split)."""
    x, w = ROUTER_DTYPES[xt], ROUTER_DTYPES[wt]
    shape, splits = aclnn.router_logits_plan(x, w, rows, cols, experts)
    return xt, wt, shape, cols * x.itemsize % 16 == 0 and cols * w.itemsize % 16 == 0, splits > 1


def test_the_router_sizes_take_every_kernel(aclnn):
    ran = {_router_kernel(aclnn, xt, wt, *size)[:4] for size in ROUTER_SIZES for xt, wt in ROUTER_TYPES}
    there = {(xt, wt, shape, grid) for xt, wt in ROUTER_TYPES for shape in range(ROUTER_SHAPES) for grid in (False, True)
             if shape < 9 or xt == "bf16" or (xt, wt) == ("f16", "f16")}
    assert ran == there


def test_the_router_sizes_take_what_other_sizes_take(aclnn):
    ran = {_router_kernel(aclnn, xt, wt, *size) for size in ROUTER_SIZES for xt, wt in ROUTER_TYPES}
    rng = random.Random(11)
    spread = lambda least, most: int(round(math.exp(rng.uniform(math.log(least), math.log(most)))))
    for _ in range(20000):
        size = [spread(1, 16384), spread(1, 32768), spread(1, 4096 if rng.random() < 0.1 else 512)]
        if rng.random() < 0.5:
            size[1] = max(8, size[1] // 8 * 8)
        kernel = _router_kernel(aclnn, *rng.choice(ROUTER_TYPES), *size)
        assert kernel in ran, (size, kernel)


def test_router_plan_refuses_what_the_operator_refuses(aclnn):
    f32, f16, bf16 = torch.float32, torch.float16, torch.bfloat16
    for args, fragment in [((torch.int8, f32, 1, 1, 1), "x must be"), ((f16, bf16, 1, 1, 1), "weight of x's type"), ((f32, f16, 1, 1, 1), "weight of x's type"),
                           ((f32, f32, 0, 1, 1), "out of range"), ((f32, f32, (1 << 26) + 1, 1, 1), "out of range"), ((f32, f32, 1, 0, 1), "out of range"),
                           ((f32, f32, 1, 1 << 31, 1), "out of range"), ((f32, f32, 1, 1, 4097), "out of range")]:
        with pytest.raises(aclnn.AclnnError, match=fragment) as e:
            aclnn.router_logits_plan(*args)
        assert e.value.code == INVALID
    null = ctypes.POINTER(ctypes.c_int)()
    assert aclnn.lib().opapiRouterLogitsPlan(F32, F32, 1, 1, 1, null, null) == NULLPTR
    assert aclnn.router_logits_plan(f32, f32, 1, 1, 1)[1] == 1
