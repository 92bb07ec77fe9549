"""The operators in front of the expert FFN on the GPU against their formulas in 64 bits on the CPU.

Tolerances, with u = 2^-24 (half an ulp of fp32 in relative terms) and half(t) = finfo(t).eps / 2 for the rounding of an output:
norm    the sum is the same bits.  r = 1/sqrt(mean + eps): the sum of H squares in one lane's share (at most H / 64 terms in a row) and a tree
        of 10 more is off by (H / 64 + 10) u, the root halves that; division, root, addition and the two products add 6 u.
        scale: the maximum's two products, r and a division, the same count.
int8    v / scale = 127 w / max w has eight roundings of fp32 in it: |y - v / scale| <= 1/2 + 127 * 8 u.
logits  a sum of K products in any order is off by at most K u sum |x w|; where both sides are split into parts of 8 bits, the three products
        that are left out are at most 2^-24 of |x w| each.  As a whole the roundings walk at random: 2 sqrt(K) u in the 2-norm.
gating  choices are exact: they are made in 64 bits.  p, the weights and their sum: fp32's rounding at most, four times u.
"""
import numpy as np
import pytest
import torch

from test_moe_front import ROUTER_SIZES

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


# ------------------------------------------------------------------------------------------------ norm
def _norm_inputs(T, H, dtype, seed, gamma32=False, residual=True, smooth=False):
    g = torch.Generator().manual_seed(seed)
    lead = T if isinstance(T, tuple) else (T,)
    x = (torch.randn(lead + (H,), generator=g) * torch.exp(torch.randn(H, generator=g))).to(dtype)
    res = torch.randn(lead + (H,), generator=g).to(dtype) if residual else None
    gamma = (1 + 0.3 * torch.randn(H, generator=g)).to(torch.float32 if gamma32 else dtype)
    sm = torch.exp(0.3 * torch.randn(H, generator=g)) if smooth else None
    return x, res, gamma, sm


def _on(dev, *ts):
    return [None if t is None else t.to(dev) for t in ts]


def _check_norm(x, res, gamma, sm, eps, got):
    y, scale, norm, total = [None if t is None else t.cpu() for t in got]
    dtype, H = x.dtype, x.shape[-1]
    s = x if res is None else (x.float() + res.float()).to(dtype)
    if total is not None:
        assert torch.equal(total, s)
    s64 = s.double()
    tol = ((H / 64 + 10) / 2 + 6) * U
    n = s64 / torch.sqrt(s64.square().mean(-1, keepdim=True) + eps) * gamma.double()
    if norm is not None:
        assert torch.all((norm.double() - n).abs() <= (tol + _half(dtype) * (1 + tol)) * n.abs() + _tiny(dtype))
    if y is None:
        return
    v = n if sm is None else n * sm.double()
    want = v.abs().amax(-1) / 127
    assert torch.all((scale.double() - want).abs() <= tol * want + 1e-44)
    q = v / want[..., None]
    assert torch.all((y.double() - q).abs() <= 0.5 + 127 * 8 * U)
    assert torch.all(y.int().abs().amax(-1) == 127)


@pytest.mark.parametrize("H", [1, 3, 8, 64, 257, 1000, 1024, 2880, 4096, 7168, 8192, 16384, 20001, 40000])
@pytest.mark.parametrize("dtype_name", ["f32", "f16", "bf16"])
def test_norm_widths(aclnn, dev, H, dtype_name):
    for T, gamma32, residual, smooth in [(1, False, True, False), (3, True, False, True), (65, True, True, True), ((2, 5), False, False, False)]:
        x, res, gamma, sm = _norm_inputs(T, H, TORCH[dtype_name], H + 7 * smooth, gamma32, residual, smooth)
        got = aclnn.moe_add_rms_norm_quant(*_on(dev, x, gamma, res, sm), epsilon=1e-5)
        assert got[3] is None or residual
        _check_norm(x, res, gamma, sm, 1e-5, got)


@pytest.mark.parametrize("H", [1000, 1024])
def test_norm_outputs_alone_and_in_place(aclnn, dev, H):
    """Every set of outputs gives the same bits; the sum may take x's or the residual's place."""
    x, res, gamma, sm = _norm_inputs(37, H, torch.bfloat16, 5)
    xd, rd, gd = _on(dev, x, res, gamma)
    y, scale, norm, total = aclnn.moe_add_rms_norm_quant(xd, gd, residual=rd)
    _check_norm(x, res, gamma, None, 1e-6, (y, scale, norm, total))
    for out in [(y.clone(), scale.clone(), None, None), (None, None, norm.clone(), None), (None, None, norm.clone(), total.clone()),
                (y.clone(), scale.clone(), norm.clone(), None), (y.clone(), scale.clone(), None, total.clone())]:
        for t in out:
            if t is not None:
                t.zero_()
        aclnn.moe_add_rms_norm_quant(xd, gd, residual=rd, out=out)
        for got, want in zip(out, (y, scale, norm, total)):
            assert got is None or torch.equal(got, want)
    for which in (0, 1):
        a, b = xd.clone(), rd.clone()
        again = aclnn.moe_add_rms_norm_quant(a, gd, residual=b, out=(torch.empty_like(y), torch.empty_like(scale), torch.empty_like(norm), (a, b)[which]))
        for got, want in zip(again, (y, scale, norm, total)):
            assert torch.equal(got, want)
        assert torch.equal((b, a)[which], (rd, xd)[which])
    both = aclnn.moe_add_rms_norm_quant(xd, gd, residual=xd)    # the same tensor twice
    _check_norm(x, x, gamma, None, 1e-6, both)
    copied = aclnn.moe_add_rms_norm_quant(xd, gd, out=(torch.empty_like(y), torch.empty_like(scale), None, total))  # a sum of one
    assert torch.equal(copied[3], xd)


@pytest.mark.parametrize("dtype_name", ["f32", "f16", "bf16"])
def test_norm_strides_and_offsets(aclnn, dev, dtype_name):
    """Views at odd places: rows that do not start on 16 bytes, slices of wider tensors, a transposed pair, outputs at an offset."""
    dtype = TORCH[dtype_name]
    for H in (1001, 1024, 4096):
        x, res, gamma, sm = _norm_inputs(9, H, dtype, H, True, True, True)
        want = aclnn.moe_add_rms_norm_quant(*_on(dev, x, gamma, res, sm))
        flat = torch.zeros(9 * H + 3, dtype=dtype, device=dev)
        odd = flat[3:].view(9, H)
        odd.copy_(x)
        wide = torch.zeros((9, 2 * H), dtype=dtype, device=dev)
        wide[:, H:] = res.to(dev)
        g2 = torch.zeros(2 * H, device=dev)
        g2[::2] = gamma.to(dev)
        s2 = torch.zeros(H + 1, device=dev)
        s2[1:] = sm.to(dev)
        out = (torch.zeros(9 * H + 5, dtype=torch.int8, device=dev)[5:].view(9, H), torch.zeros(10, device=dev)[1:],
               torch.zeros(9 * H + 1, dtype=dtype, device=dev)[1:].view(9, H), torch.zeros(9 * H + 7, dtype=dtype, device=dev)[7:].view(9, H))
        got = aclnn.moe_add_rms_norm_quant(odd, g2[::2], residual=wide[:, H:], smooth_scale=s2[1:], out=out)
        _check_norm(x, res, gamma, sm, 1e-6, got)
        assert torch.equal(got[3], want[3])
        t = aclnn.moe_add_rms_norm_quant(x.to(dev).t().contiguous().t(), gamma.to(dev), residual=res.to(dev), smooth_scale=sm.to(dev))
        for a, b in zip(t, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("H", [1000, 4096, 20001])
def test_norm_rows_of_unusual_values(aclnn, dev, H):
    """Zeros, NaN, infinities, squares past fp32, values at its lower end, and their neighbours left alone."""
    x, _, gamma, _ = _norm_inputs(8, H, torch.float32, H, True, False)
    x[0] = 0
    x[1, H // 2] = float("nan")
    x[2, H - 1] = float("inf")
    x[3] *= 1e30
    x[4] *= 1e-41          # squares underflow: the norm is x / sqrt(eps)
    x[5] *= 1e-20
    y, scale, norm, _ = [t if t is None else t.cpu() for t in aclnn.moe_add_rms_norm_quant(*_on(dev, x, gamma), epsilon=1e-6)]
    assert not y[:4].any() and scale[0] == 0 and torch.isnan(scale[1:3]).all() and scale[3] == 0
    assert not norm[0].any() and torch.isnan(norm[1]).all() and torch.isnan(norm[2, H - 1]) and not norm[3].any()
    for rows in (slice(5, 6), slice(6, 8)):
        _check_norm(x[rows], None, gamma, None, 1e-6, (y[rows], scale[rows], norm[rows], None))
    # row 4 holds multiples of 2^-149; its int8 row is still the nearest to 127 w / max w
    w = x[4].double() * gamma.double()
    q = 127 * w / w.abs().max()
    step = 127 * 2.0 ** -149 / float(w.abs().max())              # w itself is rounded to a multiple of 2^-149, and so is the maximum
    assert torch.all((y[4].double() - q).abs() <= 0.5 + 1.1 * step + 127 * 8 * U)
    z, zs, zn, _ = aclnn.moe_add_rms_norm_quant(*_on(dev, torch.zeros(2, H), gamma), epsilon=0.0)
    assert not z.any() and not zs.any() and not zn.any()


@pytest.mark.parametrize("dtype_name", ["f32", "bf16"])
@pytest.mark.parametrize("H", [1 << 20, (1 << 22) + 3])
def test_norm_of_very_long_rows(aclnn, dev, H, dtype_name):
    """The error does not grow with the row.  Of squares that are added up in 64 bits the sum's rounding to fp32 is what is left: that, the division by H
    and the addition of epsilon under the root, 3/2 u; the root, its reciprocal and two products 4 u."""
    dtype = TORCH[dtype_name]
    tol = 5.5 * U
    g = torch.Generator().manual_seed(H)
    x = (torch.tensor([[0.7], [1.1]]) * (1 + 2.0 ** -10 * torch.rand((2, H), generator=g))).to(dtype)   # nearly equal: roundings of one sign in long runs
    gamma = (1 + 0.3 * torch.randn(H, generator=g)).to(dtype)
    y, scale, norm, _ = [t if t is None else t.cpu() for t in aclnn.moe_add_rms_norm_quant(*_on(dev, x, gamma), epsilon=1e-6)]
    n = x.double() / torch.sqrt(x.double().square().mean(-1, keepdim=True) + 1e-6) * gamma.double()
    assert torch.all((norm.double() - n).abs() <= (tol + _half(dtype) * (1 + tol)) * n.abs())
    want = n.abs().amax(-1) / 127
    assert torch.all((scale.double() - want).abs() <= (tol + U) * want)     # a division more
    assert torch.all((y.double() - n / want[:, None]).abs() <= 0.5 + 127 * 8 * U)


@pytest.mark.parametrize("dtype_name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H", [1000, 1001, 4096, 20001])
def test_norm_values_in_the_middle_go_to_the_even_step(aclnn, dev, H, dtype_name):
    """Rows of whole numbers up to 254 times one gamma: 127 w / max w is half the number whatever gamma is, and every odd one lies in the middle."""
    dtype = TORCH[dtype_name]
    g = torch.Generator().manual_seed(H)
    s = torch.randint(-253, 254, (34, H), generator=g)
    s[:, 0] = torch.where(torch.arange(34) % 2 == 0, 254, -254)
    s[:, -1] = -s[:, 0]
    want = torch.round(s.double() / 2).to(torch.int8)                      # half to even
    x = (s.double() * torch.exp2(torch.arange(34) % 17 - 10.0)[:, None]).to(dtype)
    for value in (7, 13, 51, 253, 201):
        y, _, _, _ = aclnn.moe_add_rms_norm_quant(*_on(dev, x, torch.full((H,), float(value), dtype=dtype)))
        assert torch.equal(y.cpu(), want)


def test_norm_long_batches_and_empty_ones(aclnn, dev):
    x, res, gamma, _ = _norm_inputs(70000, 64, torch.bfloat16, 3)     # more rows than a grid of one dimension had in 16 bits
    _check_norm(x, res, gamma, None, 1e-6, aclnn.moe_add_rms_norm_quant(*_on(dev, x, gamma, res)))
    for shape in [(0, 64), (3, 0, 64)]:
        y, scale, norm, total = aclnn.moe_add_rms_norm_quant(torch.empty(shape, dtype=torch.bfloat16, device=dev), gamma.to(dev))
        assert y.shape == shape and scale.shape == shape[:-1] and total is None


# ------------------------------------------------------------------------------------------------ logits
def _check_logits(x, w, got):
    K = x.shape[-1]
    x64, w64 = x.double().reshape(-1, K), w.double()
    want, mass = x64 @ w64.t(), x64.abs() @ w64.abs().t()
    got = got.cpu().double().reshape(want.shape)
    assert torch.all((got - want).abs() <= (K + 4) * U * mass)
    assert (got - want).norm() <= 2 * K ** 0.5 * U * max(float(want.norm()), float(mass.norm()) / K ** 0.5)


TYPES = [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32"), ("f32", "f32")]


@pytest.mark.parametrize("xt,wt", TYPES)
@pytest.mark.parametrize("T,K,E", [(1, 1, 1), (1, 4096, 128), (1, 7168, 256), (2, 31, 3), (3, 257, 8), (4, 1024, 60), (5, 8192, 17), (16, 2880, 32),
                                   (17, 512, 500), (33, 1000, 64), (64, 7168, 256), (65, 33, 130), (100, 2049, 16), (128, 96, 96), (301, 2880, 60),
                                   (513, 576, 257), (1200, 640, 8), (2047, 1536, 128)])
def test_logits_sizes(aclnn, dev, xt, wt, T, K, E):
    g = torch.Generator().manual_seed(T + K + E)
    x = torch.randn((T, K), generator=g).to(TORCH[xt])
    w = (torch.randn((E, K), generator=g) / K ** 0.5).to(TORCH[wt])
    _check_logits(x, w, aclnn.moe_router_logits(*_on(dev, x, w)))


@pytest.mark.parametrize("T,K,E,types", [(16, 200, 300, TYPES), (16, 520, 300, TYPES), (1500, 200, 20, TYPES), (16000, 200, 33, TYPES), (16000, 203, 300, TYPES),
                                         (10000, 200, 200, TYPES), (10000, 1001, 33, TYPES), (3000, 7168, 20, TYPES[:1]), (3000, 6001, 20, TYPES[2:3]),
                                         (6500, 2049, 200, TYPES[1:2]), (6500, 2056, 200, TYPES), (13000, 4096, 100, TYPES[:3:2]), (5000, 7168, 8, TYPES[2:3])])
def test_logits_of_many_rows(aclnn, dev, T, K, E, types):
    """Sizes that every tile is chosen for, on and off the 16-byte grid, with and without the columns split."""
    for xt, wt in types:
        g = torch.Generator().manual_seed(T + K + E)
        x = torch.randn((T, K), generator=g).to(TORCH[xt])
        w = (torch.randn((E, K), generator=g) / K ** 0.5).to(TORCH[wt])
        _check_logits(x, w, aclnn.moe_router_logits(*_on(dev, x, w)))


@pytest.mark.parametrize("xt,wt", TYPES)
@pytest.mark.parametrize("T", [1, 3, 16, 70, 300, 1100])
def test_logits_keep_every_bit(aclnn, dev, xt, wt, T):
    """Rows of a single one pick weights out: not one bit of theirs may be lost, over the whole range of exponents; and the other way round."""
    g = torch.Generator().manual_seed(T)
    K, E = 200, 24
    spread = torch.exp2(torch.randint(-13, 14, (E, K), generator=g).float())
    w = (torch.randn((E, K), generator=g) * spread).to(TORCH[wt])
    at = torch.randint(0, K, (T,), generator=g)
    x = torch.zeros((T, K), dtype=TORCH[xt])
    x[torch.arange(T), at] = 1
    assert torch.equal(aclnn.moe_router_logits(*_on(dev, x, w)).cpu(), w.float().t()[at])
    x = (torch.randn((T, K), generator=g) * spread[0]).to(TORCH[xt])
    pick = torch.randint(0, K, (E,), generator=g)
    w = torch.zeros((E, K), dtype=TORCH[wt])
    w[torch.arange(E), pick] = 1
    assert torch.equal(aclnn.moe_router_logits(*_on(dev, x, w)).cpu(), x.float()[:, pick])


@pytest.mark.parametrize("xt,wt", TYPES)
@pytest.mark.parametrize("T", [30, 3000])
@pytest.mark.parametrize("K", [1, 2, 3, 4, 9])
def test_logits_of_few_columns(aclnn, dev, xt, wt, T, K):
    """Of a few products each one's own rounding shows, and what is left out of those of parts."""
    g = torch.Generator().manual_seed(T + K)
    x, w = torch.randn((T, K), generator=g), torch.randn((393, K), generator=g)
    x[::2] = torch.sign(x[::2]) * (1 + 2.0 ** -8 - 2.0 ** -16 - 2.0 ** -23)    # remainders as large as they get
    w[::3] = torch.sign(w[::3]) * (1 + 2.0 ** -7 - 2.0 ** -16 - 2.0 ** -22)
    x, w = x.to(TORCH[xt]), w.to(TORCH[wt])
    _check_logits(x, w, aclnn.moe_router_logits(*_on(dev, x, w)))


@pytest.mark.parametrize("T,K,E", ROUTER_SIZES)
def test_logits_of_every_kernel(aclnn, dev, T, K, E):
    """Every shape there is, as planned and, with rows and weights an element further on, by the kernel for those off the 16-byte grid."""
    g = torch.Generator().manual_seed(T + K + E)
    x, w = torch.randn((T, K), generator=g), torch.randn((E, K), generator=g) / K ** 0.5
    for xt, wt in TYPES:
        xs, ws = x.to(TORCH[xt]), w.to(TORCH[wt])
        room = torch.full((T * E + 4096,), 7.0, device=dev)
        _check_logits(xs, ws, aclnn.moe_router_logits(*_on(dev, xs, ws), out=room[:T * E].view(T, E)))
        assert torch.all(room[T * E:] == 7.0)
        if K * xs.element_size() % 16 == 0 and K * ws.element_size() % 16 == 0:
            odd = [torch.zeros(t.numel() + 1, dtype=t.dtype, device=dev)[1:].view(t.shape) for t in (xs, ws)]
            _check_logits(xs, ws, aclnn.moe_router_logits(odd[0].copy_(xs), odd[1].copy_(ws), out=room[:T * E].view(T, E)))
            assert torch.all(room[T * E:] == 7.0)


def test_logits_strides_offsets_and_extents(aclnn, dev):
    g = torch.Generator().manual_seed(2)
    for T, K, E in [(1, 1024, 60), (7, 1000, 16), (130, 1024, 60), (600, 513, 32)]:
        for xt, wt in TYPES:
            x, w = torch.randn((T, K), generator=g).to(TORCH[xt]), torch.randn((E, K), generator=g).to(TORCH[wt])
            want = aclnn.moe_router_logits(*_on(dev, x, w))
            flat = torch.zeros(T * K + 1, dtype=x.dtype, device=dev)
            odd = flat[1:].view(T, K)
            odd.copy_(x)
            wide = torch.zeros((E, K + 5), dtype=w.dtype, device=dev)
            wide[:, 2:K + 2] = w.to(dev)
            wodd = torch.zeros(E * K + 3, dtype=w.dtype, device=dev)[3:].view(E, K)
            wodd.copy_(w)
            out = torch.zeros(T * E + 1, device=dev)[1:].view(T, E)
            _check_logits(x, w, aclnn.moe_router_logits(odd, wide[:, 2:K + 2], out=out))
            _check_logits(x, w, aclnn.moe_router_logits(odd, wodd))
            assert torch.equal(aclnn.moe_router_logits(x.to(dev), w.to(dev).t().contiguous().t()), want)
    x3 = torch.randn((2, 3, 64), generator=g)
    w = torch.randn((5, 64), generator=g)
    out = aclnn.moe_router_logits(*_on(dev, x3, w))
    assert out.shape == (2, 3, 5)
    _check_logits(x3, w, out)
    assert aclnn.moe_router_logits(torch.empty((0, 64), device=dev), w.to(dev)).shape == (0, 5)


def test_logits_rows_apart(aclnn, dev):
    """A row with a NaN or an infinity leaves the others as they are, and memory behind the last row and expert is left alone."""
    g = torch.Generator().manual_seed(4)
    for xt, wt in TYPES:
        for T, E in [(5, 20), (90, 40), (700, 24)]:
            x, w = torch.randn((T, 640), generator=g).to(TORCH[xt]), torch.randn((E, 640), generator=g).to(TORCH[wt])
            want = aclnn.moe_router_logits(*_on(dev, x, w))
            bad = x.clone()
            bad[1, 7] = float("nan")
            bad[3, 600] = float("inf")
            room = torch.full((T * E + 4096,), 7.0, device=dev)
            got = aclnn.moe_router_logits(*_on(dev, bad, w), out=room[:T * E].view(T, E))
            keep = [r for r in range(T) if r not in (1, 3)]
            assert torch.equal(got[keep], want[keep]) and torch.isnan(got[1]).all() and not torch.isfinite(got[3]).any()
            assert torch.equal(room[T * E:], torch.full((4096,), 7.0, device=dev))


def test_logits_of_few_columns_and_very_many_rows(aclnn, dev):
    """2^26 rows of four columns: offsets behind 2^31 in the logits, and launches of fewer than 2^32 threads."""
    T, K, E = 1 << 26, 4, 36
    x = torch.randn((T, K), device=dev, generator=torch.Generator(device=dev).manual_seed(5)).bfloat16()
    w = torch.randn((E, K), generator=torch.Generator().manual_seed(6)).bfloat16()
    out = aclnn.moe_router_logits(x, w.to(dev))
    for at in (0, T // 2 - 500, (1 << 31) // E - 500, (1 << 31) // E + 500, T - 1000):
        _check_logits(x[at:at + 1000].cpu(), w, out[at:at + 1000])


@pytest.mark.parametrize("dtype_name", ["f16", "bf16"])
@pytest.mark.parametrize("T", [2, 40, 2000])
def test_logits_of_subnormal_values(aclnn, dev, dtype_name, T):
    """Values below the type's normal range are values like others; for bf16 those are fp32's own, so the weights are large."""
    dtype = TORCH[dtype_name]
    g = torch.Generator().manual_seed(T)
    x = (torch.randn((T, 256), generator=g) * (torch.finfo(dtype).smallest_normal / 8)).to(dtype)
    w = (torch.randn((40, 256), generator=g) * (1.0 if dtype_name == "f16" else 1e20)).to(dtype)
    assert int((x != 0).sum()) > x.numel() // 2
    _check_logits(x, w, aclnn.moe_router_logits(*_on(dev, x, w)))


@pytest.mark.parametrize("K", [2048, 7168])
def test_logits_of_prompts_in_graphs(aclnn, dev, K):
    """Two captured calls over a workspace each (the longer columns are split), replayed in turn with eager calls between them."""
    g = torch.Generator().manual_seed(7)
    w = (torch.randn((256, K), generator=g) / 45).to(dev)
    graphs = []
    for T in (600, 700):
        x, out, space = torch.randn((T, K), generator=g).bfloat16().to(dev), torch.empty((T, 256), device=dev), aclnn.Workspace()
        aclnn.moe_router_logits(x, w, out=out, workspace=space)
        assert K == 2048 or space.tensor is not None
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            aclnn.moe_router_logits(x, w, out=out, workspace=space)
        graphs.append((x, out, space, graph))
    for step in range(4):
        for x, out, _, graph in graphs:
            x.copy_(torch.randn(x.shape, generator=g).bfloat16())
            graph.replay()
            got = out.clone()
            assert torch.equal(got, aclnn.moe_router_logits(x, w))


# ------------------------------------------------------------------------------------------------ gating
def _gating_reference(x, k, bias=None, k_group=1, group_count=1, group_select_mode=0, score_type=0, renorm=0, routed_scaling_factor=1.0, eps=1e-20):
    x = x.double().numpy()
    rows, E = x.shape
    masked = x == -np.inf
    with np.errstate(all="ignore"):
        if score_type == 1:
            p = 1 / (1 + np.exp(-x))
        else:
            top = x.max(-1, keepdims=True)
            e = np.where(masked, 0, np.exp(x - top))
            p = np.where(masked, 0, e / e.sum(-1, keepdims=True))
        t = np.where(masked, -np.inf, p if bias is None else p + bias.double().numpy())
    key = x if bias is None else t               # p is a monotone function of the logit: without a bias logits are compared
    order_of = lambda v: np.argsort(-np.nan_to_num(v, nan=np.inf, neginf=-np.inf), axis=-1, kind="stable")  # NaN ahead of all
    out = np.zeros((rows, E), dtype=bool)
    if k_group < group_count:
        g = (t if group_select_mode == 1 else key).reshape(rows, group_count, -1)
        desc = -np.sort(-np.nan_to_num(g, nan=np.inf, neginf=-np.inf), axis=-1)
        best = desc[:, :, 0]
        if group_select_mode == 1:
            best = np.where(desc[:, :, 1] == -np.inf, best, best + desc[:, :, 1])
        gone = order_of(best)[:, k_group:]
        left = np.zeros((rows, group_count), dtype=bool)
        np.put_along_axis(left, gone, True, -1)
        out = np.repeat(left, E // group_count, axis=-1)
    idx = np.empty((rows, k), dtype=np.int64)
    for r in range(rows):
        kept = np.flatnonzero(~out[r])
        idx[r] = kept[order_of(key[r:r + 1, kept])[0][:k]]
    y = np.take_along_axis(p, idx, -1)
    if renorm:
        total = y.sum(-1, keepdims=True) + eps
        with np.errstate(all="ignore"):
            y = np.where(total == 0, 0, y / total)
    return y * routed_scaling_factor, idx, p


def _check_gating(aclnn, dev, x, k, y_dtype=None, **kw):
    bias = kw.get("bias")
    call = dict(kw, bias=None if bias is None else bias.to(dev))
    y, idx, scores = aclnn.moe_gating_top_k_grouped(x.to(dev), k, y_dtype=y_dtype, output_scores=True, **call)
    yr, ir, pr = _gating_reference(x, k, **kw)
    assert y.dtype == (x.dtype if y_dtype is None else y_dtype)
    assert np.array_equal(idx.cpu().numpy(), ir)
    tol = 4 * U + (_half(y.dtype) if y.dtype != torch.float32 else 0)
    np.testing.assert_allclose(y.cpu().double().numpy(), yr, rtol=tol, atol=float(_tiny(y.dtype)))
    np.testing.assert_allclose(scores.cpu().double().numpy(), pr, rtol=4 * U, atol=1e-44)
    again = aclnn.moe_gating_top_k_grouped(x.to(dev), k, y_dtype=y_dtype, **call)     # without the scores: the same bits
    assert torch.equal(again[0], y) and torch.equal(again[1], idx) and again[2] is None


SHAPES = [(1, 1, 1, 1, 1), (3, 2, 1, 1, 1), (2, 8, 2, 1, 1), (7, 8, 4, 4, 2), (1, 256, 8, 8, 4), (64, 256, 8, 8, 4), (5, 60, 6, 6, 3), (33, 64, 64, 1, 1), (9, 65, 5, 5, 2),
          (301, 160, 6, 8, 3), (17, 96, 12, 2, 1), (4, 72, 7, 8, 8), (6, 384, 8, 4, 2), (11, 512, 8, 16, 5), (3, 500, 10, 10, 3), (2, 513, 8, 3, 1),
          (5, 1024, 20, 32, 16), (3, 2048, 64, 64, 9), (2, 2047, 33, 1, 1), (2000, 128, 8, 1, 1), (3, 144, 3, 144, 72), (2, 192, 64, 3, 2)]


@pytest.mark.parametrize("T,E,k,groups,k_group", SHAPES)
@pytest.mark.parametrize("score_type", [0, 1])
def test_gating_against_formula(aclnn, dev, T, E, k, groups, k_group, score_type):
    g = torch.Generator().manual_seed(T * E + k)
    x = torch.randn((T, E), generator=g)
    bias = 0.1 * torch.randn(E, generator=g)
    for b in (None, bias):
        for mode in (0, 1):
            if mode == 1 and E // groups < 2 and k_group < groups:
                continue
            _check_gating(aclnn, dev, x, k, bias=b, k_group=k_group, group_count=groups, group_select_mode=mode, score_type=score_type,
                          renorm=mode, routed_scaling_factor=2.5)


@pytest.mark.parametrize("dtype_name", ["f16", "bf16"])
def test_gating_sixteen_bits(aclnn, dev, dtype_name):
    g = torch.Generator().manual_seed(9)
    for T, E, k, groups, k_group in [(50, 256, 8, 8, 4), (301, 160, 6, 8, 3), (5, 1000, 33, 1, 1), (3, 63, 9, 7, 5)]:
        x = torch.randn((T, E), generator=g).to(TORCH[dtype_name])
        bias = 0.1 * torch.randn(E, generator=g)
        for y_dtype in (None, torch.float32):
            for score_type, renorm in [(0, 0), (0, 1), (1, 1)]:
                _check_gating(aclnn, dev, x, k, y_dtype=y_dtype, bias=bias, k_group=k_group, group_count=groups, score_type=score_type, renorm=renorm,
                              routed_scaling_factor=16.0, eps=1e-6)


@pytest.mark.parametrize("E,groups", [(8, 4), (64, 1), (64, 8), (65, 5), (256, 8), (255, 5), (512, 2), (768, 8), (2048, 4)])
def test_gating_equal_values_take_the_lower_index(aclnn, dev, E, groups):
    rng = np.random.default_rng(E + groups)
    x = torch.from_numpy(rng.integers(0, 5, (12, E)).astype(np.float32))   # one sign: sums of two never meet
    x[0] = 0.25
    x[1] = 0.0
    x[1, E - 1] = 1.0
    for k_group in sorted({1, (groups + 1) // 2, groups}):
        for k in sorted({1, min(8, E // groups * k_group), min(64, E // groups * k_group)}):
            for mode in (0, 1):
                _check_gating(aclnn, dev, x, k, k_group=k_group, group_count=groups, group_select_mode=mode, score_type=1, renorm=1)
            _check_gating(aclnn, dev, x, k, bias=torch.full((E,), -3.0), k_group=k_group, group_count=groups, score_type=0)  # t below zero


@pytest.mark.parametrize("E", [16, 96, 256, 640])
@pytest.mark.parametrize("score_type", [0, 1])
def test_gating_masked_and_unusual_logits(aclnn, dev, E, score_type):
    """Logits of -inf (some, all of a group, all but one of a group, whole rows), the types' lowest values, saturated ones, NaN."""
    g = torch.Generator().manual_seed(E)
    x = torch.randn((10, E), generator=g)
    bias = torch.randn(E, generator=g)                                # larger than the scores: masks have to win against it
    size = E // 4
    x[0, ::3] = -float("inf")
    x[1] = -float("inf")
    x[2, :size] = -float("inf")
    x[3, size + 1:2 * size] = -float("inf")
    x[4, 1:] = -float("inf")
    x[5, ::2] = torch.finfo(torch.float32).min
    x[6] = torch.finfo(torch.float32).min
    x[7, E // 2] = 1e4
    x[8] *= 200
    k = min(8, E // 4)
    for k_group in (1, 2, 4):
        for mode in (0, 1):
            for b in (None, bias):
                _check_gating(aclnn, dev, x, k, bias=b, k_group=k_group, group_count=4, group_select_mode=mode, score_type=score_type, renorm=1)
    _check_gating(aclnn, dev, x, k, k_group=2, group_count=4, score_type=score_type, renorm=1, eps=0.0)
    x[9, E // 3] = float("nan")
    y, idx, scores = aclnn.moe_gating_top_k_grouped(x.to(dev), k, bias=bias.to(dev), k_group=2, group_count=4, group_select_mode=1,
                                                    score_type=score_type, output_scores=True)
    _, ir, _ = _gating_reference(x, k, bias, 2, 4, 1, score_type)
    assert np.array_equal(idx.cpu().numpy()[:9], ir[:9])
    row = idx[9].cpu().tolist()
    assert len(set(row)) == k and min(row) >= 0 and max(row) < E
    assert (row[0] == E // 3) if score_type == 1 else torch.isnan(y[9]).all()
    assert torch.isnan(scores[9]).all() if score_type == 0 else int(torch.isnan(scores[9]).sum()) == 1


def test_gating_close_scores_are_told_apart(aclnn, dev):
    """Sums p + bias that agree in fp32 and differ in 64 bits: the larger one is picked, wherever it stands."""
    E = 128
    x = torch.zeros((4, E))
    bias = torch.linspace(0.0, 0.25, E)
    x[0] = torch.log((0.5 + 0.25 - bias).double() / (0.5 - 0.25 + bias).double()).float()   # sigmoid(x) + bias = 0.75 up to rounding
    x[1] = x[0].flip(0)
    x[2] = x[0] + 1e-7
    x[3] = x[0]
    x[3, 5:9] += 2e-7
    for kw in [dict(), dict(k_group=2, group_count=8, group_select_mode=1), dict(k_group=3, group_count=4)]:
        _check_gating(aclnn, dev, x, 8, bias=bias, score_type=1, renorm=1, **kw)


def test_gating_finished_strided_and_ranked_inputs(aclnn, dev):
    g = torch.Generator().manual_seed(1)
    x = torch.randn((4, 6, 96), generator=g)
    bias = 0.1 * torch.randn(96, generator=g)
    fin = torch.rand((4, 6), generator=g) < 0.5
    kw = dict(k_group=2, group_count=4, group_select_mode=1, score_type=1, renorm=1)
    y, idx, _ = aclnn.moe_gating_top_k_grouped(x.to(dev), 5, bias=bias.to(dev), finished=fin.to(dev), **kw)
    yr, ir, _ = _gating_reference(x.view(24, 96), 5, bias, **kw)
    assert np.array_equal(idx.cpu().numpy().reshape(24, 5), np.where(fin.view(24, 1).numpy(), 96, ir))
    np.testing.assert_allclose(y.cpu().numpy().reshape(24, 5), yr, rtol=4 * U)
    wide = torch.zeros((4, 6, 200), device=dev)
    wide[..., 100:196] = x.to(dev)
    b2 = torch.zeros(192, device=dev)
    b2[::2] = bias.to(dev)
    f2 = fin.t().contiguous().to(dev).t()
    out = (torch.zeros(24 * 5 + 1, device=dev)[1:].view(4, 6, 5), torch.zeros(24 * 5 + 3, dtype=torch.int32, device=dev)[3:].view(4, 6, 5),
           torch.zeros(24 * 96 + 1, device=dev)[1:].view(4, 6, 96))
    again = aclnn.moe_gating_top_k_grouped(wide[..., 100:196], 5, bias=b2[::2], finished=f2, out=out, **kw)
    assert torch.equal(again[0], y) and torch.equal(again[1], idx)
    for dtype in (torch.float32, torch.bfloat16):                    # rows off the 16-byte grid
        for E in (96, 97):
            flat = torch.zeros(7 * E + 1, dtype=dtype, device=dev)
            odd = flat[1:].view(7, E)
            odd.copy_(torch.randn((7, E), generator=g))
            a, b = aclnn.moe_gating_top_k_grouped(odd, 5, **dict(kw, k_group=1, group_count=1)), aclnn.moe_gating_top_k_grouped(odd.clone(), 5, **dict(kw, k_group=1, group_count=1))
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert aclnn.moe_gating_top_k_grouped(torch.empty((0, 96), device=dev), 5, **kw)[1].shape == (0, 5)


# Rows by the thousand are chosen sixteen lanes each: the cases above again at such lengths.
LONG = 4003


def _long_rows(E, seed):
    """Twelve rows, of which ten are where a choice can go wrong, and the order they are repeated in."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((12, E), generator=g)
    x[0, ::3] = -float("inf")
    x[1] = -float("inf")
    x[2, :E // 4] = -float("inf")
    x[3, E // 4 + 1:E // 2] = -float("inf")
    x[4, 1:] = -float("inf")
    x[5, ::2] = torch.finfo(torch.float32).min
    x[6] = torch.finfo(torch.float32).min
    x[7, E // 2] = 1e4
    x[8] *= 200
    x[9] = torch.randint(0, 5, (E,), generator=g).float()
    return x, torch.randint(0, 12, (LONG,), generator=g)


def _check_long(aclnn, dev, x, order, k, **kw):
    bias = kw.get("bias")
    yr, ir, pr = _gating_reference(x, k, **kw)
    y, idx, scores = aclnn.moe_gating_top_k_grouped(x[order].to(dev), k, output_scores=True, **dict(kw, bias=None if bias is None else bias.to(dev)))
    assert np.array_equal(idx.cpu().numpy(), ir[order])
    tol = 4 * U + (_half(y.dtype) if y.dtype != torch.float32 else 0)
    np.testing.assert_allclose(y.cpu().double().numpy(), yr[order], rtol=tol, atol=float(_tiny(y.dtype)))
    np.testing.assert_allclose(scores.cpu().double().numpy(), pr[order], rtol=4 * U, atol=1e-44)


@pytest.mark.parametrize("E,groups", [(8, 4), (16, 4), (20, 4), (48, 3), (96, 4), (128, 16), (255, 5), (256, 8), (500, 10), (512, 16)])
@pytest.mark.parametrize("score_type", [0, 1])
def test_gating_long_batches(aclnn, dev, E, groups, score_type):
    x, order = _long_rows(E, E + groups)
    bias = torch.randn(E, generator=torch.Generator().manual_seed(E))
    for k_group in sorted({1, (groups + 1) // 2, groups}):
        k = min(16, E // groups * k_group)
        for mode in (0, 1):
            for b in (None, bias, 1e-3 * bias):
                _check_long(aclnn, dev, x, order, k, bias=b, k_group=k_group, group_count=groups, group_select_mode=mode, score_type=score_type, renorm=mode)
    for dtype in (torch.float16, torch.bfloat16):
        short = x.clamp(min=torch.finfo(dtype).min).to(dtype)
        short[x == -float("inf")] = -float("inf")
        _check_long(aclnn, dev, short, order, min(8, E // groups), bias=bias, k_group=1, group_count=groups, score_type=score_type)
        _check_long(aclnn, dev, short, order, min(8, E), score_type=score_type)


@pytest.mark.parametrize("T", [7, LONG])
@pytest.mark.parametrize("E", [16, 24, 60, 100, 160, 256, 384])
def test_gating_rows_off_the_grid(aclnn, dev, T, E):
    """Rows and a bias that start between the boundaries of the lanes' packets: the same bits as those on them."""
    g = torch.Generator().manual_seed(E)
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.randn((T, E), generator=g).to(dtype).to(dev)
        bias = (0.1 * torch.randn(E, generator=g)).to(dev)
        odd = torch.zeros(T * E + 1, dtype=dtype, device=dev)[1:].view(T, E)
        odd.copy_(x)
        shifted = torch.zeros(E + 1, device=dev)[1:]
        shifted.copy_(bias)
        for kw in [dict(), dict(k_group=2, group_count=4, group_select_mode=1)]:
            for b, o in [(None, None), (bias, shifted)]:
                want = aclnn.moe_gating_top_k_grouped(x, 4, bias=b, score_type=1, renorm=1, output_scores=True, **kw)
                got = aclnn.moe_gating_top_k_grouped(odd, 4, bias=o, score_type=1, renorm=1, output_scores=True, **kw)
                assert all(torch.equal(p, q) for p, q in zip(want, got))


@pytest.mark.parametrize("T", [3, LONG])
@pytest.mark.parametrize("E,groups", [(16, 4), (96, 4), (640, 4)])
def test_gating_zeros_of_either_sign_are_equal(aclnn, dev, T, E, groups):
    x = torch.full((1, E), -1.0)
    x[0, 1::2] = 0.0
    x[0, 3::4] = -0.0
    order = torch.zeros(T, dtype=torch.int64)
    for score_type in (0, 1):
        for mode in (0, 1):
            _check_long(aclnn, dev, x, order, 4, score_type=score_type, k_group=2, group_count=groups, group_select_mode=mode)
    x[0, ::2] = torch.finfo(torch.float32).min    # first in their lanes: what is compared is zeros of one lane and of others
    _check_long(aclnn, dev, x, order, min(8, E // 2), score_type=1)


@pytest.mark.parametrize("T", [12, LONG])
@pytest.mark.parametrize("E", [16, 96, 256, 640])
@pytest.mark.parametrize("low", [-float("inf"), torch.finfo(torch.float32).min])
def test_gating_biases_that_mask_experts(aclnn, dev, T, E, low):
    """A bias of -inf, or of the lowest value, puts an expert behind those that have none; its score stays what it is."""
    x, order = _long_rows(E, E)
    g = torch.Generator().manual_seed(E + 1)
    for share in (0.25, 0.9):
        bias = 0.1 * torch.randn(E, generator=g)
        bias[torch.rand(E, generator=g) < share] = low
        for score_type in (0, 1):
            for kw in [dict(), dict(k_group=2, group_count=4), dict(k_group=2, group_count=4, group_select_mode=1)]:
                _check_long(aclnn, dev, x, order[:T], min(8, E // 4), bias=bias, score_type=score_type, **kw)


@pytest.mark.parametrize("T", [12, LONG])
@pytest.mark.parametrize("E", [8, 16, 60, 96, 256, 384, 640])
def test_gating_biases_that_are_all_equal(aclnn, dev, T, E):
    """One bias for all, from zero to those beside which no score shows in 32 bits, and every expert masked: the choice is the one in 64 bits, however many
    rows there are."""
    x, order = _long_rows(E, E)
    for value in (0.0, -3.0, 2.0 ** 18, 2.0 ** 24, -2.0 ** 24, 2.0 ** 25, 1e9, -1e9, torch.finfo(torch.float32).max, torch.finfo(torch.float32).min, -float("inf")):
        bias = torch.full((E,), value)
        for score_type in (0, 1):
            for kw in [dict(), dict(k_group=2, group_count=4), dict(k_group=2, group_count=4, group_select_mode=1)]:
                _check_long(aclnn, dev, x, order[:T], min(8, E // 4), bias=bias, score_type=score_type, **kw)
    flat = 1e-3 * torch.randn((12, E), generator=torch.Generator().manual_seed(E))   # softmax scores of 1 / E: 2^16 hides them
    for value in (2.0 ** 14, 2.0 ** 16, -2.0 ** 17):
        _check_long(aclnn, dev, flat, order[:T], min(8, E // 4), bias=torch.full((E,), value), score_type=0)


@pytest.mark.parametrize("T", [12, LONG])
@pytest.mark.parametrize("E", [16, 640])
def test_gating_factors_that_only_64_bits_hold(aclnn, dev, T, E):
    """The factor is a double, and what counts is whether the weights fit: 2^130 passes fp32, times a weight below 1/4 it does not."""
    g = torch.Generator().manual_seed(E)
    x, order = 0.01 * torch.randn((12, E), generator=g), torch.randint(0, 12, (T,), generator=g)
    for factor in (2.0 ** 130, -2.0 ** 130, 0.1, 2.0 ** -160):
        _check_long(aclnn, dev, x, order, 4, routed_scaling_factor=factor)
        _check_long(aclnn, dev, x, order, 4, bias=torch.randn(E, generator=g), routed_scaling_factor=factor)


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("H", [37, 40])
def test_elements_behind_2_to_the_31(aclnn, dev, H):
    """The most rows there may be, of 2.5 and 2.7 thousand million elements: norm and choice of experts at the start, the middle and the end."""
    T = 1 << 26
    g = torch.Generator(device=dev).manual_seed(H)
    x = torch.empty((T, H), dtype=torch.bfloat16, device=dev).normal_(generator=g)
    gamma = torch.ones(H, dtype=torch.bfloat16)
    y, scale, norm, total = aclnn.moe_add_rms_norm_quant(x, gamma.to(dev))
    bias = 0.1 * torch.randn(H, generator=torch.Generator().manual_seed(H))
    weight, idx, _ = aclnn.moe_gating_top_k_grouped(x, 2, bias=bias.to(dev), score_type=1, renorm=1, y_dtype=torch.float32)
    assert total is None
    for at in (0, T // 2, (1 << 31) // H - 500, T - 1000):
        rows = x[at:at + 1000].cpu()
        _check_norm(rows, None, gamma, None, 1e-6, (y[at:at + 1000], scale[at:at + 1000], norm[at:at + 1000], None))
        yr, ir, _ = _gating_reference(rows, 2, bias, score_type=1, renorm=1)
        assert np.array_equal(idx[at:at + 1000].cpu().numpy(), ir)
        np.testing.assert_allclose(weight[at:at + 1000].cpu().numpy(), yr, rtol=4 * U)


def _block(pkg, dev, tokens, H=1024, I=512, E=16, seed=3, weight32=True):
    g = torch.Generator().manual_seed(seed)
    x, res, gamma, _ = _norm_inputs(tokens, H, torch.bfloat16, seed)
    router = (torch.randn((E, H), generator=g) / H ** 0.5).to(torch.float32 if weight32 else torch.bfloat16)
    bias = 0.05 * torch.randn(E, generator=g)
    w13 = torch.randint(-127, 128, (E, 2 * I, H), generator=g, dtype=torch.int8)
    w2 = torch.randint(-127, 128, (E, H, I), generator=g, dtype=torch.int8)
    w13s, w2s = 1e-3 + 1e-3 * torch.rand((E, 2 * I), generator=g), 1e-3 + 1e-3 * torch.rand((E, H), generator=g)
    ffn = pkg.MoeFfnW8A8(*_on(dev, w13, w13s, w2, w2s))
    return _on(dev, x, res, gamma, router, bias), ffn, (w13, w13s, w2, w2s)


def _run_block(aclnn, ffn, x, res, gamma, router, bias, out=None):
    q, scale, norm, total = aclnn.moe_add_rms_norm_quant(x, gamma, residual=res)
    logits = aclnn.moe_router_logits(norm, router)
    wgt, idx, _ = aclnn.moe_gating_top_k_grouped(logits, 4, bias=bias, k_group=2, group_count=4, group_select_mode=1, score_type=1, renorm=1,
                                                 routed_scaling_factor=2.5)
    return total, q, scale, norm, logits, wgt, idx, ffn.forward(q, scale, idx, wgt)


@pytest.mark.parametrize("tokens", [1, 23, 300])
def test_block_from_hidden_states_to_expert_output(pkg, aclnn, oracle, dev, tokens):
    """Norm, router product, choice of experts and the expert FFN chained, every stage against its formula on what the one before gave."""
    ins, ffn, (w13, w13s, w2, w2s) = _block(pkg, dev, tokens)
    total, q, scale, norm, logits, wgt, idx, out = _run_block(aclnn, ffn, *ins)
    torch.cuda.synchronize()
    x, res, gamma, router, bias = [t.cpu() for t in ins]
    _check_norm(x, res, gamma, None, 1e-6, (q, scale, norm, total))
    _check_logits(norm.cpu(), router, logits)
    yr, ir, _ = _gating_reference(logits.cpu(), 4, bias, k_group=2, group_count=4, group_select_mode=1, score_type=1, renorm=1, routed_scaling_factor=2.5)
    assert np.array_equal(idx.cpu().numpy(), ir)
    np.testing.assert_allclose(wgt.cpu().numpy(), yr, rtol=4 * U)
    E = router.shape[0]
    ex, row_idx, cumsum, xs = oracle.moe_init_routing_v3(q.cpu().numpy(), ir.astype(np.int32), scale.cpu().numpy(), E, None, 0, 1)
    gl = cumsum.astype(np.int64)
    h, hs = oracle.grouped_matmul_swiglu_quant(ex, w13.numpy(), w13s.numpy(), xs.reshape(-1), gl, w_trans=True)
    y = oracle.grouped_matmul_dequant(h, w2.numpy(), w2s.numpy(), hs, gl, w_trans=True, out_dtype=oracle.DT_BF16)
    ref = oracle.bf16_bits_to_f32(oracle.moe_finalize_routing_v2(y, row_idx, scales=wgt.cpu().numpy(), drop_pad_mode=2, dtype=oracle.DT_BF16,
                                                                scale_dtype=oracle.DT_F32))
    got = out.float().cpu().numpy()
    # the FFN's own bar: its int8 intermediate may be one unit off, 1 / 127 of a term
    rel = np.abs(got - ref) / np.maximum(np.abs(ref), 1e-3 * np.abs(ref).max())
    assert np.median(rel) < 1e-2 and np.quantile(rel, 0.999) < 5e-2


@pytest.mark.parametrize("tokens", [1, 40])
def test_block_in_a_graph_and_on_another_stream(pkg, aclnn, dev, tokens):
    """Two captured blocks over different inputs, replayed in turn with eager work between them, and eager calls on a stream of their own."""
    blocks = []
    for seed in (3, 4):
        ins, ffn, _ = _block(pkg, dev, tokens, seed=seed)
        _run_block(aclnn, ffn, *ins)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = _run_block(aclnn, ffn, *ins)
        blocks.append((ins, ffn, graph, outs))
    for step in range(4):
        for ins, ffn, graph, outs in blocks:
            g = torch.Generator().manual_seed(100 + step)
            ins[0].copy_(torch.randn(ins[0].shape, generator=g).to(torch.bfloat16))
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in outs]
            want = _run_block(aclnn, ffn, *ins)
            for a, b in zip(got, want):
                assert torch.equal(a, b)
    ins, ffn, _, _ = blocks[0]
    want = [t.clone() for t in _run_block(aclnn, ffn, *ins)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [t.clone() for t in _run_block(aclnn, ffn, *ins)]
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_tensors_that_do_not_fit_are_refused(aclnn, dev):
    x, gamma = torch.ones((2, 64), dtype=torch.bfloat16, device=dev), torch.ones(64, dtype=torch.bfloat16)
    with pytest.raises(aclnn.AclnnError, match="on cuda:0 and cpu"):
        aclnn.moe_add_rms_norm_quant(x, gamma)
    with pytest.raises(TypeError, match="not one the operators know"):
        aclnn.moe_router_logits(x, torch.ones((3, 64), dtype=torch.float64, device=dev))
    with pytest.raises(aclnn.AclnnError, match="must be"):
        aclnn.moe_router_logits(x, torch.ones((3, 63), dtype=torch.bfloat16, device=dev))
    with pytest.raises(TypeError):
        aclnn.moe_router_logits(x, torch.ones((1,) * 9, device=dev), out=torch.ones((2, 1), device=dev))
    y, scale, norm, _ = aclnn.moe_add_rms_norm_quant(x, gamma.to(dev), epsilon=0)  # a whole number for a double
    assert torch.equal(norm, x) and int(y.min()) == 127


def test_calls_at_once_on_two_streams(aclnn, dev):
    """Calls of the same sizes side by side: without a workspace of the caller's every call has its own."""
    g = torch.Generator().manual_seed(8)
    w = torch.randn((256, 4096), generator=g).to(dev)
    xs = [torch.randn((48, 4096), generator=g).bfloat16().to(dev) for _ in range(2)]
    want = [aclnn.moe_router_logits(x, w) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(aclnn.moe_router_logits(xs[i], w))
    torch.cuda.synchronize()
    for i in range(2):
        for t in got[i]:
            assert torch.equal(t, want[i])


@pytest.mark.parametrize("kept", [False, True])
def test_split_products_at_once_on_two_streams(aclnn, dev, kept):
    """Products whose columns are split over workgroups, and so need room for their parts, side by side: each call has room of its own, or each stream has
    (kept)."""
    T, K, E = 600, 7168, 256
    assert aclnn.router_logits_plan(torch.bfloat16, torch.float32, T, K, E)[1] > 1
    g = torch.Generator().manual_seed(9)
    w = (torch.randn((E, K), generator=g) / K ** 0.5).to(dev)
    xs = [torch.randn((T, K), generator=g).bfloat16().to(dev) for _ in range(2)]
    spaces = [aclnn.Workspace() for _ in xs]
    want = [aclnn.moe_router_logits(x, w, workspace=space) for x, space in zip(xs, spaces)]
    for x, space, t in zip(xs, spaces, want):
        assert space.requested["aclnnMoeRouterLogits"] >= 2 * T * E * 4
        _check_logits(x.cpu(), w.cpu(), t)
    assert spaces[0].tensor.data_ptr() != spaces[1].tensor.data_ptr()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(aclnn.moe_router_logits(xs[i], w, workspace=spaces[i] if kept else None))
    torch.cuda.synchronize()
    for i in range(2):
        for t in got[i]:
            assert torch.equal(t, want[i])
