"""GPU: the operators on rows of channels against their formulas in 64 bits.

Tolerances are elementwise bounds: u is half a step of the type (eps / 2), B = 2^-24 that of the fp32 sums.  Products are
also tested with small integers, for which every intermediate is exact in every type, so that results have to be equal:
what a wrong index would change there no tolerance hides."""
import math

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from super_resolution_amd import conv_core as cc
from super_resolution_amd import token_ops, tokens

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
B = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]
ACTS = {"silu": F.silu, "gelu": F.gelu, "relu": torch.relu, "sigmoid": torch.sigmoid}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rnd(*shape, seed=0, scale=1.0, shift=0.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype).to(DEV)


def within(got, want, tol, what=""):
    got, want = got.double(), want.double()
    bad = (got - want).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got - want).abs() / tol).max().item():.3g} x the bound"


# ---- layer norm -----------------------------------------------------------------------------------------------------
def norm_bounds(x, w, b, dy, eps, u):
    """Formula and bounds, in 64 bits, of y, dx, dw, db."""
    x, dy = x.double(), dy.double()
    rows, c = x.shape
    w = torch.ones(c, dtype=torch.float64, device=DEV) if w is None else w.double()
    b = torch.zeros(c, dtype=torch.float64, device=DEV) if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    xh = (x - mean) * rstd
    y = xh * w + b
    d = dy * w
    s, q = d.mean(1, keepdim=True), (d * xh).mean(1, keepdim=True)
    dx = rstd * (d - s - xh * q)
    # a sum of n terms held by 64 lanes and more, added pairwise over the lanes: fewer than n / 64 + 16 roundings deep
    deep = c / 64 + 24
    e_xh = B * deep * (x.abs().amax(1, keepdim=True) * rstd + xh.abs()) * 1.5
    t_y = u * y.abs() + 1.01 * w.abs() * e_xh + 4 * B * (xh.abs() * w.abs() + b.abs())
    e_q = (d.abs() * e_xh).mean(1, keepdim=True) + B * deep * (d * xh).abs().mean(1, keepdim=True)
    e_s = B * deep * d.abs().mean(1, keepdim=True)
    t_dx = u * dx.abs() + 1.01 * rstd * (e_s + xh.abs() * e_q + e_xh * q.abs() + 8 * B * (d.abs() + s.abs() + (xh * q).abs())) + B * deep * dx.abs()
    dw, db = (dy * xh).sum(0), dy.sum(0)
    rdeep = rows + 24
    t_dw = (dy.abs() * e_xh).sum(0) + B * rdeep * (dy * xh).abs().sum(0)
    t_db = B * rdeep * dy.abs().sum(0)
    return (y, dx, dw, db), (t_y, t_dx, t_dw, t_db)


NORM_SHAPES = [(1, 1), (3, 1), (1, 2), (5, 7), (64, 8), (33, 60), (100, 64), (7, 96), (50, 129), (19, 256), (9, 500), (6, 512), (40, 1000),
               (1030, 1024), (5, 1500), (4, 2048), (3, 4096), (2, 4100), (3, 5001), (2, 8192), (2, 8200), (3, 9001), (1, 20000), (5000, 24)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", NORM_SHAPES)
def test_layer_norm_matches_the_formula(shape, dtype):
    rows, c = shape
    x = rnd(rows, c, seed=1, scale=2.0, shift=3.0, dtype=dtype)
    for wt in {dtype, torch.float32}:
        w, b = rnd(c, seed=2, scale=0.3, shift=1.0, dtype=wt), rnd(c, seed=3, dtype=wt)
        dy = rnd(rows, c, seed=4, dtype=dtype)
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        y = tokens.layer_norm(*leaves, 1e-5)
        grads = torch.autograd.grad(y, leaves, dy)
        want, tol = norm_bounds(x, w, b, dy, 1e-5, half_step(dtype))
        tiny = torch.finfo(dtype).tiny
        within(y, want[0], tol[0] + tiny, "y")
        within(grads[0], want[1], tol[1] + tiny, "dx")
        uw = half_step(wt)
        within(grads[1], want[2], tol[2] + uw * want[2].abs() + 1e-30, "dw")
        within(grads[2], want[3], tol[3] + uw * want[3].abs() + 1e-30, "db")
        assert grads[1].dtype == wt and y.dtype == dtype
        assert torch.equal(tokens.layer_norm(x, w, b), y)                      # the unrecorded call
        assert torch.equal(torch.autograd.grad(tokens.layer_norm(*leaves, 1e-5), leaves, dy)[1], grads[1])   # a fixed order


@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_without_parameters_and_single_gradients(dtype):
    x, dy = rnd(37, 72, seed=5, dtype=dtype), rnd(37, 72, seed=6, dtype=dtype)
    w = rnd(72, seed=7, dtype=dtype)
    want, tol = norm_bounds(x, None, None, dy, 1e-3, half_step(dtype))
    xg = x.clone().requires_grad_()
    y = tokens.layer_norm(xg, eps=1e-3)
    within(y, want[0], tol[0] + 1e-30)
    within(torch.autograd.grad(y, xg, dy)[0], want[1], tol[1] + 1e-30)
    want, tol = norm_bounds(x, w, None, dy, 1e-5, half_step(dtype))
    wg = w.clone().requires_grad_()                                            # the weight alone
    y = tokens.layer_norm(x, wg)
    within(y, want[0], tol[0] + 1e-30)
    within(torch.autograd.grad(y, wg, dy)[0], want[2], tol[2] + half_step(dtype) * want[2].abs() + 1e-30)
    bg = w.clone().requires_grad_()                                            # a bias alone
    y = tokens.layer_norm(x, None, bg)
    within(torch.autograd.grad(y, bg, dy)[0], dy.double().sum(0), tol[3] + half_step(dtype) * dy.double().sum(0).abs() + 1e-30)


def test_layer_norm_of_rows_with_more_columns_than_a_grid_axis_has_blocks():
    rows, c = 2, (1 << 24) + 5
    x, dy = rnd(rows, c, seed=16), rnd(rows, c, seed=17)
    w, b = rnd(c, seed=18), rnd(c, seed=19)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = tokens.layer_norm(*leaves)
    got = (y, *torch.autograd.grad(y, leaves, dy))
    for g, want, tol in zip(got, *norm_bounds(x.detach(), w.detach(), b.detach(), dy, 1e-5, B)):
        within(g.detach(), want, tol + B * want.abs() + 1e-30)


def test_layer_norm_strides_alignment_and_odd_rows():
    big = rnd(40, 300, seed=8)
    ref = lambda t: tokens.layer_norm(t.contiguous().clone())
    for view in (big[:, :64], big[:, 1:65], big[::3, 4:260], big.t(), big[:, ::2], big[:1].expand(9, 300), big.view(5, 8, 300)[:, ::2],
                 big.view(5, 8, 300).transpose(0, 1), big[3], big[:, 7:8]):
        assert torch.equal(tokens.layer_norm(view), ref(view)) or torch.allclose(tokens.layer_norm(view), ref(view), atol=1e-5)
        v = view.detach().clone(memory_format=torch.preserve_format).requires_grad_()
        g = rnd(*view.shape, seed=9)
        a = torch.autograd.grad(tokens.layer_norm(v), v, g)[0]
        c = view.contiguous().clone().requires_grad_()
        b = torch.autograd.grad(tokens.layer_norm(c), c, g)[0]
        assert torch.allclose(a, b, atol=1e-4)
    # an expanded gradient, as sum() makes it
    x = rnd(6, 48, seed=10).requires_grad_()
    w = rnd(48, seed=11).requires_grad_()
    gx, gw = torch.autograd.grad(tokens.layer_norm(x, w).sum(), (x, w))
    x2, w2 = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    ex, ew = torch.autograd.grad(F.layer_norm(x2, (48,), w2).sum(), (x2, w2))
    assert torch.allclose(gx.double(), ex, atol=1e-5) and torch.allclose(gw.double(), ew, atol=1e-5)


def test_layer_norm_empty_constant_and_non_finite_rows():
    w = rnd(16, seed=12).requires_grad_()
    b = rnd(16, seed=13).requires_grad_()
    x = torch.empty(0, 16, device=DEV, requires_grad=True)
    y = tokens.layer_norm(x, w, b)
    assert y.shape == (0, 16)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.empty(0, 16, device=DEV))
    assert gx.shape == (0, 16) and (gw == 0).all() and (gb == 0).all()
    assert torch.equal(tokens.layer_norm(torch.full((3, 16), 7.0, device=DEV), w, b), b.detach().expand(3, 16))
    # a large mean: the variance survives
    x = rnd(4, 512, seed=14, shift=1000.0)
    want = F.layer_norm(x.double(), (512,))
    assert (tokens.layer_norm(x).double() - want).abs().max() < 2e-2 * 1000 * 2.0 ** -13
    x = rnd(5, 40, seed=15)
    x[1, 3], x[3, 0] = float("nan"), float("inf")
    y = tokens.layer_norm(x)
    assert y[1].isnan().all() and y[3].isnan().all() and y[[0, 2, 4]].isfinite().all()


# ---- dropout --------------------------------------------------------------------------------------------------------
def keep_mask(n, p, seed, step, site, first=0):
    """Which elements stay, on the CPU, from the generator's definition."""
    m = 0xFFFFFFFF
    c = np.zeros(((n + 7) // 8, 4), np.uint64)
    c[:, 0] = np.arange(len(c), dtype=np.uint64) + np.uint64(first // 8)
    c[:, 2], c[:, 3] = step & m, site
    k0, k1 = seed & m, (seed >> 32) & m
    for _ in range(7):
        a, b = c[:, 0] * np.uint64(0xD2511F53), c[:, 2] * np.uint64(0xCD9E8D57)
        s = np.uint64(32)
        c = np.stack([(b >> s) ^ c[:, 1] ^ np.uint64(k0), b & np.uint64(m), (a >> s) ^ c[:, 3] ^ np.uint64(k1), a & np.uint64(m)], 1)
        k0, k1 = (k0 + 0x9E3779B9) & m, (k1 + 0xBB67AE85) & m
    bits = np.stack([c & np.uint64(0xFFFF), c >> np.uint64(16)], 2).reshape(-1)[:n]
    return torch.from_numpy(bits >= np.uint64(math.floor(p * 65536 + 0.5))).to(DEV)


def state(seed=-12345678901234567, step=3):
    return torch.tensor([seed, step], dtype=torch.int64, device=DEV)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 1000, 4096, 100003])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0, 1e-7])
def test_dropout_and_its_gradient(n, p, dtype):
    x, skip, dy = rnd(n, seed=20, dtype=dtype), rnd(n, seed=21, dtype=dtype), rnd(n, seed=22, dtype=dtype)
    keep = keep_mask(n, p, -12345678901234567, 3, 5)
    t = math.floor(p * 65536 + 0.5)
    scale = 65536 / (65536 - t) if t < 65536 else 0.0
    u = half_step(dtype)
    # under the smallest normal number the type's steps stay those at it: a rounding is off by up to tiny * u there
    # (fp16: 2^-14 * 2^-11 = 2^-25, half of its smallest subnormal 2^-24)
    low = torch.finfo(dtype).tiny * u
    for s in (None, skip):
        xg, sg = x.clone().requires_grad_(), (None if s is None else s.clone().requires_grad_())
        y = tokens.dropout(xg, p, state(), site=5, residual=sg)
        kept = torch.where(keep, x.double() * scale, 0.0)
        want = kept if s is None else kept + s.double()
        # the scale is fp32, the product and the sum round once each in fp32, the result once in its type
        within(y, want, u * want.abs() + 4 * B * (kept.abs() + want.abs()) + low)
        grads = torch.autograd.grad(y, [xg] if s is None else [xg, sg], dy)
        want = torch.where(keep, dy.double() * scale, 0.0)
        within(grads[0], want, u * want.abs() + 4 * B * want.abs() + low)
        if s is not None:
            assert torch.equal(grads[1], dy)
    if p == 0.0:
        assert torch.equal(tokens.dropout(x, p, state()), x)


def test_dropout_masks_depend_on_seed_step_and_site_and_hold_their_probability():
    x = torch.ones(1 << 20, device=DEV)
    masks = [tokens.dropout(x, 0.3, state(*s), site=site) != 0 for s, site in
             (((1, 0), 0), ((2, 0), 0), ((1, 1), 0), ((1, 0), 1), ((1 + (1 << 32), 0), 0))]
    n = x.numel()
    for i, m in enumerate(masks):
        # five standard deviations of a binomial count
        assert abs(int(m.sum()) - 0.7 * n) < 5 * math.sqrt(n * 0.21)
        for o in masks[:i]:
            assert abs(int((m & o).sum()) - 0.49 * n) < 5 * math.sqrt(n * 0.49 * 0.51)
    assert torch.equal(masks[0], tokens.dropout(x, 0.3, state(1, 0)) != 0)
    assert torch.equal(masks[0], tokens.dropout(x, 0.3, state(1, 1 << 32)) != 0)        # the step counts modulo 2^32


def test_dropout_strides_alignment_and_non_finite_values():
    base = rnd(33, 40, seed=23)
    for dtype in TYPES:
        flat = rnd(1001, seed=24, dtype=dtype)
        assert torch.equal(tokens.dropout(flat[1:], 0.4, state()), tokens.dropout(flat[1:].clone(), 0.4, state()))
        assert torch.equal(tokens.dropout(flat[:-1], 0.4, state(), residual=flat[1:]),
                           tokens.dropout(flat[:-1].clone(), 0.4, state(), residual=flat[1:].clone()))
    assert torch.equal(tokens.dropout(base.t(), 0.4, state()), tokens.dropout(base.t().contiguous(), 0.4, state()))
    x = torch.full((64,), float("nan"), device=DEV)
    y = tokens.dropout(x, 0.5, state())
    keep = keep_mask(64, 0.5, -12345678901234567, 3, 0)
    assert y[keep].isnan().all() and (y[~keep] == 0).all()
    assert tokens.dropout(torch.empty(0, 8, device=DEV), 0.5, state()).shape == (0, 8)
    # changing the state in place before the backward pass is reported
    s, xg = state(), base.clone().requires_grad_()
    y = tokens.dropout(xg, 0.5, s)
    s.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# ---- gated feed-forward ---------------------------------------------------------------------------------------------
def ffn_inputs(t, c, f, dtype, biases, seed):
    x, dy = rnd(t, c, seed=seed, dtype=dtype), rnd(t, c, seed=seed + 1, dtype=dtype)
    ws = [rnd(f, c, seed=seed + 2, scale=c ** -0.5, dtype=dtype), rnd(f, c, seed=seed + 3, scale=c ** -0.5, dtype=dtype),
          rnd(c, f, seed=seed + 4, scale=f ** -0.5, dtype=dtype)]
    bs = [rnd(n, seed=seed + 5 + i, scale=0.2, dtype=dtype) if biases else None for i, n in enumerate((f, f, c))]
    return x, dy, ws, bs


def sparse_ints(rows, cols, per_row, seed, dtype, values=(-1, 1)):
    """Rows with a few small integers: every product and sum of the block stays an integer that all types hold."""
    g = torch.Generator().manual_seed(seed)
    m = torch.zeros(rows, cols)
    at = torch.randint(0, cols, (rows, per_row), generator=g)
    v = torch.tensor(values, dtype=torch.float32)[torch.randint(0, len(values), (rows, per_row), generator=g)]
    return m.scatter_(1, at, v).to(dtype).to(DEV)


def ternary(rows, cols, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(-1, 2, (rows, cols), generator=g)).to(dtype).to(DEV)


FFN_SHAPES = [(1, 1, 1), (1, 8, 8), (2, 7, 5), (3, 64, 256), (15, 33, 70), (16, 64, 64), (17, 24, 40), (31, 100, 36), (32, 129, 257),
              (33, 256, 512), (40, 1027, 2101), (64, 60, 130), (64, 2048, 1032), (65, 512, 72), (127, 64, 128), (128, 96, 1000), (129, 1000, 96), (257, 180, 360), (300, 136, 264),
              (1000, 65, 129), (2049, 64, 256), (16385, 72, 520), (700, 1024, 2056), (513, 520, 8200)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", FFN_SHAPES)
def test_gated_ffn_is_exact_on_small_integers(shape, dtype):
    """relu on integers: g, u in [-4, 4], h in [-12, 12], dg, du in [-48, 48] are exact in every type, the fp32 sums are
    (below 2^24), and the results are the exact values rounded once."""
    t, c, f = shape
    x, dy = sparse_ints(t, c, 3, 1, dtype), sparse_ints(t, c, 3, 2, dtype)
    ws = [ternary(f, c, 3, dtype), ternary(f, c, 4, dtype), ternary(c, f, 5, dtype)]
    bs = [ternary(1, n, 6 + i, dtype)[0] for i, n in enumerate((f, f, c))]
    leaves = [v.clone().requires_grad_() for v in (x, *ws, *bs)]
    y = tokens.gated_ffn(*leaves, activation="relu")
    grads = torch.autograd.grad(y, leaves, dy)
    # (float64 products of these integers are exact whatever their order)
    xd, dyd, wg, wu, wd, bg, bu, bd = (v.double() for v in (x, dy, *ws, *bs))
    g, u = xd @ wg.t().contiguous() + bg, xd @ wu.t().contiguous() + bu
    h = g.clamp_min(0) * u
    dh = dyd @ wd
    dg, du = dh * u * (g > 0), dh * g.clamp_min(0)
    want = [h @ wd.t().contiguous() + bd, dg @ wg + du @ wu, dg.t().contiguous() @ xd, du.t().contiguous() @ xd,
            dyd.t().contiguous() @ h, dg.sum(0), du.sum(0), dyd.sum(0)]
    assert max(float(v.abs().max()) for v in (g, u)) <= 4 and max(float(v.abs().max()) for v in want) < 2 ** 24
    for name, a, b in zip(("y", "dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down"), (y, *grads), want):
        assert torch.equal(a, b.to(dtype)), (name, int((a != b.to(dtype)).sum()), a.numel())
    with torch.no_grad():
        assert torch.equal(tokens.gated_ffn(x, *ws, *bs, activation="relu"), y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(16384, 64, 256), (16500, 1, 1), (16400, 33, 70), (20001, 128, 96), (16384, 72, 520), (16391, 8, 1000),
                                   (16640, 96, 31)])
def test_gated_ffn_unrecorded_on_many_narrow_rows_is_exact_on_small_integers(shape, dtype):
    """Forward only, up to 128 channels (16-bit types: one launch that keeps the hidden channels in registers)."""
    t, c, f = shape
    x = sparse_ints(t, c, 3, 11, dtype)
    ws = [ternary(f, c, 12, dtype), ternary(f, c, 13, dtype), ternary(c, f, 14, dtype)]
    bs = [ternary(1, n, 15 + i, dtype)[0] for i, n in enumerate((f, f, c))]
    xd, wg, wu, wd, bg, bu, bd = (v.double() for v in (x, *ws, *bs))
    for biases in (True, False):
        g, u = xd @ wg.t().contiguous(), xd @ wu.t().contiguous()
        if biases:
            g, u = g + bg, u + bu
        want = (g.clamp_min(0) * u) @ wd.t().contiguous() + (bd if biases else 0)
        y = tokens.gated_ffn(x, *ws, *(bs if biases else ()), activation="relu")
        assert torch.equal(y, want.to(dtype)), (biases, int((y != want.to(dtype)).sum()))
    wide = torch.full((t, c + 5), float("nan"), dtype=dtype, device=DEV)       # rows of another stride, at an odd address
    wide[:, 3:3 + c] = x
    assert torch.equal(tokens.gated_ffn(wide[:, 3:3 + c], *ws, activation="relu"), y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", list(ACTS))
def test_gated_ffn_unrecorded_on_many_narrow_rows_matches_the_formula(act, dtype):
    for c, f in ((64, 96), (100, 40)):
        x, dy, ws, bs = ffn_inputs(16400, c, f, dtype, True, 35)
        want, tol = ffn_bounds(x, dy, ws, bs, act, half_step(dtype))
        within(tokens.gated_ffn(x, *ws, *bs, activation=act), want[0], tol[0] + torch.finfo(dtype).tiny * (1 + f), "y")
        x[7, 3] = float("nan")
        y = tokens.gated_ffn(x, *ws, *bs, activation=act)
        assert y[7].isnan().all() and y[:7].isfinite().all() and y[8:].isfinite().all()


def ffn_bounds(x, dy, ws, bs, act, u, uh=None):
    """Results and bounds in 64 bits.  Per sum of n products: n B of the sum of magnitudes; u per rounding to the type (uh: of
    h, dg and du, where that is another)."""
    uh = u if uh is None else uh
    t, c = x.shape
    f = ws[0].shape[0]
    xd, dyd = x.double(), dy.double()
    wg, wu, wd = (w.double() for w in ws)
    bg, bu, bd = (torch.zeros(n, dtype=torch.float64, device=DEV) if b is None else b.double() for b, n in zip(bs, (f, f, c)))
    T = lambda m: m.t().contiguous()
    g, uu = xd @ T(wg) + bg, xd @ T(wu) + bu
    gl = g.clone().requires_grad_()
    a = ACTS[act](gl)
    (da,) = torch.autograd.grad(a.sum(), gl)
    a = a.detach()
    h, dh = a * uu, dyd @ wd
    dg, du = dh * uu * da, dh * a
    # slopes: |act'| <= 1.13, |act''| <= 0.8 for every activation (relu's kink aside, where g's sign is exact enough: below)
    e_g = (c + 4) * B * (xd.abs() @ T(wg.abs()) + bg.abs()) + 4 * B * g.abs()
    e_u = (c + 4) * B * (xd.abs() @ T(wu.abs()) + bu.abs()) + 4 * B * uu.abs()
    fn = 2.0 ** -20                                            # the activations' own error, relative to max(|a|, |a'|)
    e_a = 1.13 * e_g + fn * a.abs()
    e_h = e_a * uu.abs() + a.abs() * e_u + 2 * uh * h.abs()
    y = h @ T(wd) + bd
    t_y = e_h @ T(wd.abs()) + (f + 4) * B * (h.abs() @ T(wd.abs()) + bd.abs()) + u * y.abs()
    # the backward pass multiplies dh with act(g) and u act'(g), kept as the upper 24 bits of fp32 (cut: off by less than
    # 2^-15): |a~ - a| <= e_a + 2^-15 |a| and, with d = u act'(g), |d~ - d| <= (e_u |act'| + |u| e_act') (1 + ..) + 2^-15 |d|
    cut = 0.0 if u < 2.0 ** -20 else 2.0 ** -15
    e_dh = (c + 4) * B * (dyd.abs() @ wd.abs())
    e_da = 0.8 * e_g + fn * (1 + da.abs())
    if act == "relu":
        e_da = (g.abs() <= 2 * e_g).double()
    e_as = e_a + 1.01 * cut * a.abs()
    e_d = e_u * (da.abs() + e_da) + uu.abs() * e_da + 1.01 * cut * (uu * da).abs() + 4 * B * (uu * da).abs()
    grow = 1.01
    e_dg = grow * (e_dh * (uu * da).abs() + dh.abs() * e_d + 4 * B * dg.abs()) + 1.01 * uh * dg.abs()
    e_du = grow * (e_dh * a.abs() + dh.abs() * e_as + 4 * B * du.abs()) + 1.01 * uh * du.abs()
    dx = dg @ wg + du @ wu
    t_dx = e_dg @ wg.abs() + e_du @ wu.abs() + (2 * f + 4) * B * (dg.abs() @ wg.abs() + du.abs() @ wu.abs()) + u * dx.abs()
    out, tol = [y, dx], [t_y, t_dx]
    for d, e in ((dg, e_dg), (du, e_du)):
        out.append(T(d) @ xd)
        tol.append(T(e) @ xd.abs() + (t + 4) * B * (T(d.abs()) @ xd.abs()) + u * out[-1].abs())
    out.append(T(dyd) @ h)
    tol.append(T(dyd.abs()) @ e_h + (t + 4) * B * (T(dyd.abs()) @ h.abs()) + u * out[-1].abs())
    for d, e in ((dg, e_dg), (du, e_du), (dyd, torch.zeros_like(dyd))):
        out.append(d.sum(0))
        tol.append(e.sum(0) + (t + 4) * B * d.abs().sum(0) + u * out[-1].abs())
    return out, tol


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("shape", [(1, 64, 96), (5, 20, 33), (70, 128, 136), (333, 65, 200)])
def test_gated_ffn_matches_the_formula(shape, act, dtype):
    t, c, f = shape
    for biases in (False, True):
        x, dy, ws, bs = ffn_inputs(t, c, f, dtype, biases, 30)
        leaves = [v.clone().requires_grad_() for v in (x, *ws, *bs) if v is not None]
        y = tokens.gated_ffn(*leaves, activation=act)
        grads = torch.autograd.grad(y, leaves, dy)
        want, tol = ffn_bounds(x, dy, ws, bs, act, half_step(dtype))
        # below the smallest normal number a rounding is absolute
        tiny = torch.finfo(dtype).tiny * (1 + f)
        for name, a, b, e in zip(("y", "dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down"), (y, *grads), want, tol):
            within(a, b, e + tiny, name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 20, 1700), (5, 33, 96), (16, 40, 640), (20, 24, 500), (61, 16, 520)])
def test_gated_ffn_of_a_small_block_rounds_once(shape, dtype):
    """Few rows of few channels: h is a sum of two numbers of the type, whose rounding is u^2 (fp16: half a smallest subnormal at least,
    2^-25).  Bias gradients of gate and up, of any rows: dg and du are summed in fp32."""
    t, c, f = shape
    x, dy, ws, bs = ffn_inputs(t, c, f, dtype, True, 40)
    leaves = [v.clone().requires_grad_() for v in (x, *ws, *bs)]
    y = tokens.gated_ffn(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    u = half_step(dtype)
    want, tol = ffn_bounds(x, dy, ws, bs, "silu", u, 1.01 * u * u)
    low = 2.0 ** -25 if dtype == torch.float16 else 1e-30
    tiny = torch.finfo(dtype).tiny
    within(y, want[0], tol[0] + low * ws[2].double().abs().sum(1) + tiny, "y")
    within(tokens.gated_ffn(x, *ws, *bs), want[0], tol[0] + low * ws[2].double().abs().sum(1) + tiny, "y unrecorded")
    for k in (5, 6):
        within(grads[k - 1], want[k], tol[k] + tiny * (1 + t), k)
    x[0, 0] = float("inf")
    assert tokens.gated_ffn(x, *ws, *bs)[0].isnan().any() and tokens.gated_ffn(x, *ws, *bs)[1:].isfinite().all()
    huge = torch.full((1, c), 200.0, dtype=dtype, device=DEV)       # h is infinite in fp16, and so is y, without a NaN
    ones = [torch.ones_like(w) for w in ws]
    out = tokens.gated_ffn(huge, *ones, activation="relu")
    assert not out.isnan().any() and (out.isinf().all() if dtype == torch.float16 else out.isfinite().all())


def test_gated_ffn_gradients_against_differences():
    t, c, f = 9, 24, 40
    for act in ("silu", "gelu", "sigmoid"):
        x, dy, ws, bs = ffn_inputs(t, c, f, torch.float32, True, 50)
        leaves = [v.clone().requires_grad_() for v in (x, *ws, *bs)]
        grads = torch.autograd.grad(tokens.gated_ffn(*leaves, activation=act), leaves, dy)
        for i, (v, g) in enumerate(zip((x, *ws, *bs), grads)):
            d = rnd(*v.shape, seed=60 + i)
            d = d / d.norm()
            step = 0.02
            up, down = ([w if k != i else w + s * step * d for k, w in enumerate((x, *ws, *bs))] for s in (1, -1))
            loss = [(tokens.gated_ffn(*p, activation=act).double() * dy.double()).sum() for p in (up, down)]
            # the third derivative along a unit direction is O(|dy|) here; fp32 noise of the two losses over 2 steps
            size = (dy.double().norm() * 4).item()
            assert abs(((loss[0] - loss[1]) / (2 * step) - (g.double() * d.double()).sum()).item()) < size * (step ** 2 + 64 * B / step)


def test_layer_norm_gradient_against_differences():
    x, w, dy = rnd(5, 40, seed=70), rnd(40, seed=71), rnd(5, 40, seed=72)
    xg = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(tokens.layer_norm(xg, w), xg, dy)
    d = rnd(5, 40, seed=73)
    d = d / d.norm()
    step = 0.02
    loss = [(tokens.layer_norm(x + s * step * d, w).double() * dy.double()).sum() for s in (1, -1)]
    size = (dy.double().norm() * w.double().abs().max() * 4).item()
    assert abs(((loss[0] - loss[1]) / (2 * step) - (g.double() * d.double()).sum()).item()) < size * (step ** 2 + 64 * B / step)


@pytest.mark.parametrize("dtype", TYPES)
def test_gated_ffn_strides_alignment_and_leading_dimensions(dtype):
    t, c, f = 21, 40, 56
    x, dy, ws, bs = ffn_inputs(t, c, f, dtype, True, 80)

    def both(x, ws, dy):
        leaves = [v.detach().requires_grad_() for v in (x, *ws)]
        y = tokens.gated_ffn(*leaves, *bs)
        return [y, *torch.autograd.grad(y, leaves, dy)]

    want = both(x, ws, dy)
    wide = torch.full((t, c + 24), float("nan"), dtype=dtype, device=DEV)
    for off in (0, 8, 3):                                          # a view of wider rows: aligned, aligned, unaligned
        wide[:, off:off + c] = x
        wide2 = wide.clone()
        wide2[:, off:off + c] = dy
        got = both(wide[:, off:off + c], ws, wide2[:, off:off + c])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = both(x.t().contiguous().t(), [w.t().contiguous().t() for w in ws], dy.t().contiguous().t())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    flat = [torch.zeros(w.numel() + 1, dtype=dtype, device=DEV) for w in ws]
    for m, w in zip(flat, ws):
        m[1:] = w.reshape(-1)
    got = both(x, [m[1:].view(w.shape) for m, w in zip(flat, ws)], dy)   # weights at an odd address
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = both(x.view(3, 7, 1, c), ws, dy.view(3, 7, 1, c))
    assert got[0].shape == (3, 7, 1, c) and all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, want))
    got = both(x[4], ws, dy[4])
    assert got[0].shape == (c,)
    ones = both(x, ws, torch.ones((), dtype=dtype, device=DEV).expand(t, c))
    assert all(torch.equal(a, b) for a, b in zip(ones, both(x, ws, torch.ones_like(dy))))
    # one tensor as gate and up weight: its gradient is the sum
    w = ws[0].clone().requires_grad_()
    (g,) = torch.autograd.grad(tokens.gated_ffn(x, w, w, ws[2], *bs), w, dy)
    split = [ws[0].clone().requires_grad_() for _ in range(2)]
    pair = torch.autograd.grad(tokens.gated_ffn(x, *split, ws[2], *bs), split, dy)
    assert torch.equal(g, pair[0] + pair[1])


def test_gated_ffn_empty_rows_single_gradients_and_non_finite_rows():
    c, f = 24, 40
    _, _, ws, bs = ffn_inputs(4, c, f, torch.float32, True, 90)
    x = torch.empty(0, c, device=DEV, requires_grad=True)
    leaves = [x, *(v.clone().requires_grad_() for v in (*ws, *bs))]
    y = tokens.gated_ffn(*leaves)
    assert y.shape == (0, c)
    grads = torch.autograd.grad(y, leaves, torch.empty(0, c, device=DEV))
    assert grads[0].shape == (0, c) and all((g == 0).all() for g in grads[1:])
    x, dy, ws, bs = ffn_inputs(77, c, f, torch.bfloat16, True, 91)
    full = [v.clone().requires_grad_() for v in (x, *ws, *bs)]
    want = torch.autograd.grad(tokens.gated_ffn(*full), full, dy)
    for i in range(7):                                             # each gradient alone
        one = [v.clone().requires_grad_(k == i) for k, v in enumerate((x, *ws, *bs))]
        assert torch.equal(torch.autograd.grad(tokens.gated_ffn(*one), one[i], dy)[0], want[i])
    x = x.clone()
    clean = tokens.gated_ffn(x, *ws, *bs)
    x[5, 3] = float("nan")
    y = tokens.gated_ffn(x, *ws, *bs)
    rows = torch.arange(77, device=DEV) != 5
    assert y[5].isnan().all() and torch.equal(y[rows], clean[rows])


# ---- together, streams, graphs --------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
def test_block_in_a_network_trains(dtype):
    """norm -> feed-forward -> dropout onto the skip, on the pixels between two 3x3 convs: against the same in 64 bits with
    the mask of the generator's definition (gradients of the normalisation's weight, relative norm)."""
    N, H, W, c, f = 2, 6, 9, 24, 56
    torch.manual_seed(3)
    block = tokens.FeedForwardBlock(c, f, dropout=0.25, activation="gelu").to(DEV)
    block.seed(77)
    x, dy = rnd(N, H, W, c, seed=100, dtype=dtype), rnd(N, H, W, c, seed=101, dtype=dtype)
    xg = x.clone().requires_grad_()
    y = block(xg)
    y.backward(dy)
    assert block.rng_state.tolist() == [77, 1] and y.dtype == dtype
    p = {k: v.detach().double().requires_grad_() for k, v in block.named_parameters()}
    xd = x.double().requires_grad_()
    h = F.layer_norm(xd, (c,), p["norm.weight"], p["norm.bias"])
    h = F.gelu(F.linear(h, p["gate.weight"], p["gate.bias"])) * F.linear(h, p["up.weight"], p["up.bias"])
    h = F.linear(h, p["down.weight"], p["down.bias"])
    keep = keep_mask(x.numel(), 0.25, 77, 0, 0).view(x.shape)
    (xd + torch.where(keep, h / 0.75, 0.0)).backward(dy.double())
    # at most eight roundings to the type on any path from an input to a gradient
    tol = 8 * half_step(dtype) + 1e-5
    for a, b in [(xg.grad, xd.grad), *((v.grad, p[k].grad) for k, v in block.named_parameters())]:
        assert a is not None and (a.double() - b).norm() <= tol * b.norm()
    block.eval()
    assert torch.equal(block(x), block(x)) and block.rng_state.tolist() == [77, 1]


def test_block_between_convs():
    """The conv core's activations through rows and back: gradients reach every parameter, and equal runs are equal."""
    torch.manual_seed(4)
    block = tokens.FeedForwardBlock(32, 64, dropout=0.1).to(DEV)
    w = [(torch.randn(32, 32, 3, 3) * 0.05).to(DEV).requires_grad_() for _ in range(2)]
    b = [torch.zeros(32, device=DEV, requires_grad=True) for _ in range(2)]
    x = rnd(2, 32, 10, 13, seed=110)

    def run():
        block.seed(5)
        h = cc.conv3x3(cc.to_blocked(x), w[0], b[0], 0.2)
        h = tokens.blocked_from_rows(block(tokens.rows_from_blocked(h, 32)))
        y = cc.from_blocked(cc.conv3x3(h, w[1], b[1]), 32)
        return [y, *torch.autograd.grad(y.square().mean(), [*w, *b, *block.parameters()])]

    first, second = run(), run()
    assert all(torch.equal(a, c) for a, c in zip(first, second))
    assert all(g.abs().max() > 0 for g in first)


FAR = (1 << 20) + 3                                                # rows of 2056 channels pass 2^31 elements


def first_and_last_rows():
    return torch.cat([torch.arange(40), torch.arange(FAR - 40, FAR)]).to(DEV)


def test_gated_ffn_offsets_past_32_bits():
    """All rows but the first and the last are zeros, which add nothing."""
    c, f, dtype = 8, 2056, torch.bfloat16
    at = first_and_last_rows()
    x, dy = (torch.zeros(FAR, c, dtype=dtype, device=DEV) for _ in range(2))
    x[at], dy[at] = sparse_ints(80, c, 3, 170, dtype), sparse_ints(80, c, 3, 171, dtype)
    leaves = [v.requires_grad_() for v in (x, ternary(f, c, 172, dtype), ternary(f, c, 173, dtype), ternary(c, f, 174, dtype))]
    y = tokens.gated_ffn(*leaves, activation="relu")
    dx, *dws = torch.autograd.grad(y, leaves, dy)
    xd, dyd, wg, wu, wd = (v.detach().double() for v in (x[at], dy[at], *leaves[1:]))
    g, u = xd @ wg.t().contiguous(), xd @ wu.t().contiguous()
    h = g.clamp_min(0) * u
    dh = dyd @ wd
    dg, du = dh * u * (g > 0), dh * g.clamp_min(0)
    for got, want in zip((y.detach()[at], dx[at], *dws), (h @ wd.t().contiguous(), dg @ wg + du @ wu, dg.t().contiguous() @ xd,
                                                          du.t().contiguous() @ xd, dyd.t().contiguous() @ h)):
        assert torch.equal(got, want.to(dtype))
    assert not y.detach()[40:-40].any() and not dx[40:-40].any()


def test_layer_norm_and_dropout_offsets_past_32_bits():
    c, dtype = 2056, torch.bfloat16
    at = first_and_last_rows()
    x = torch.randn(FAR, c, dtype=dtype, device=DEV, generator=torch.Generator(DEV).manual_seed(180)).requires_grad_()
    w = rnd(c, seed=181).requires_grad_()
    dy = torch.zeros(FAR, c, dtype=dtype, device=DEV)
    dy[at] = rnd(80, c, seed=182, dtype=dtype)
    y = tokens.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    want, tol = norm_bounds(x.detach()[at], w.detach(), None, dy[at], 1e-5, half_step(dtype))
    for got, k in ((y.detach()[at], 0), (dx[at], 1), (dw, 2)):
        within(got, want[k], tol[k] + B * want[k].abs() + 1e-30)
    del y, dx, dy
    last = FAR * c - 4096
    x = x.detach()
    y = tokens.dropout(x, 0.5, state())
    for first in (0, last):
        part = x.view(-1)[first:first + 4096]
        keep = keep_mask(4096, 0.5, -12345678901234567, 3, 0, first)
        assert torch.equal(y.view(-1)[first:first + 4096], torch.where(keep, part * 2, torch.zeros_like(part)))


def test_tied_weights_and_a_skip_from_the_input():
    """w_gate is w_up and also, transposed by the caller, w_down; dropout's skip is its own input."""
    x, w, dy = sparse_ints(50, 24, 3, 190, torch.float32), ternary(40, 24, 191, torch.float32), sparse_ints(50, 24, 3, 192, torch.float32)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    grads = torch.autograd.grad(tokens.gated_ffn(xg, wg, wg, wg.t(), activation="relu"), (xg, wg), dy)
    apart = [x.clone().requires_grad_(), w.clone().requires_grad_(), w.clone().requires_grad_(), w.t().clone().requires_grad_()]
    a = torch.autograd.grad(tokens.gated_ffn(*apart, activation="relu"), apart, dy)
    assert torch.equal(grads[0], a[0]) and torch.equal(grads[1], a[1] + a[2] + a[3].t())
    xg = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(tokens.dropout(xg, 0.5, state(), residual=xg), xg, dy)
    assert torch.equal(g, tokens.dropout(dy, 0.5, state(), residual=dy))


def chain(x, ws, rng, dy):
    leaves = [v.detach().requires_grad_() for v in (x, *ws)]
    h = tokens.layer_norm(leaves[0])
    y = tokens.dropout(tokens.gated_ffn(h, *leaves[1:]), 0.2, rng, residual=leaves[0])
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


@pytest.mark.parametrize("shape", [(40, 64, 96), (3, 33, 50), (1000, 64, 256)])
def test_on_a_side_stream_and_in_a_replayed_graph(shape):
    t, c, f = shape
    x, dy, ws, _ = ffn_inputs(t, c, f, torch.bfloat16, False, 120)
    rng = state(9, 0)
    want = chain(x, ws, rng, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        busy = torch.randn(2048, 2048, device=DEV)
        for _ in range(10):
            busy = busy @ busy * 1e-3
        late = x * 1.0                                             # written behind the busy work
        got = chain(late, ws, rng, dy)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    sx = x.clone()
    with torch.cuda.graph(graph):
        out = chain(sx, ws, rng, dy)
        rng[1].add_(1)
    rng.copy_(state(9, 0))
    for step in range(4):
        fresh = rnd(t, c, seed=130 + step, dtype=torch.bfloat16)
        sx.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        eager = chain(fresh, ws, state(9, step), dy)               # eager work between the replays
        assert rng.tolist() == [9, step + 1]
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), step


def test_two_graphs_do_not_share_memory():
    x, dy, ws, _ = ffn_inputs(200, 64, 128, torch.bfloat16, False, 140)
    rng, graphs, outs, ins = state(), [], [], []
    for k in range(2):
        ins.append(x * (k + 1))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(chain(ins[k], ws, rng, dy))
        graphs.append(g)
    for g in (graphs[0], graphs[1], graphs[0]):
        g.replay()
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(a, b) for a, b in zip(outs[k], chain(x * (k + 1), ws, rng, dy)))


def test_a_capture_refuses_leaves_of_a_live_graph_of_the_default_stream():
    x, w = rnd(20, 16, seed=160).requires_grad_(), rnd(16, seed=161).requires_grad_()
    block = tokens.FeedForwardBlock(16, 40).to(DEV)
    params = list(block.parameters())
    h = rnd(20, 16, seed=162, dtype=torch.bfloat16)
    want = [*torch.autograd.grad(tokens.layer_norm(x, w).sum(), (x, w)), *torch.autograd.grad(block(h).sum(), params)]
    live = [tokens.layer_norm(x, w), block(h)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="recorded on the default stream"):
            tokens.layer_norm(x, w)
        with pytest.raises(RuntimeError, match="recorded on the default stream"):
            block(h)
        with torch.no_grad():                                      # (nothing is recorded)
            unrecorded = tokens.layer_norm(x, w)
    graph.replay()
    assert torch.equal(unrecorded, live[0])
    live.clear()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [*torch.autograd.grad(tokens.layer_norm(x, w).sum(), (x, w)), *torch.autograd.grad(block(h).sum(), params)]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_opcheck():
    utils = ("test_schema", "test_faketensor")
    x, dy, ws, bs = ffn_inputs(10, 24, 40, torch.bfloat16, True, 150)
    w = rnd(24, seed=151)
    check = torch.library.opcheck
    check(torch.ops.sr355.layer_norm_fwd, (x, w, w, 1e-5, True), test_utils=utils)
    stats = token_ops.layer_norm_fwd(x, w, w, 1e-5, True)[1]
    check(torch.ops.sr355.layer_norm_bwd, (dy, x, w, stats, torch.float32, [True, False, True]), test_utils=utils)
    check(torch.ops.sr355.dropout, (x, dy, 0.3, state(), 1), test_utils=utils)
    check(torch.ops.sr355.gated_ffn_fwd, (x, *ws, *bs, 0, True), test_utils=utils)
    saved = token_ops.gated_ffn_fwd(x, *ws, *bs, 0, True)[1]
    check(torch.ops.sr355.gated_ffn_bwd, (dy, x, *ws, saved, 0, [True] * 7), test_utils=utils)


def test_refusals():
    x = rnd(4, 8)
    w, wd = rnd(16, 8), rnd(8, 16)
    rng = state()
    bad = [
        (lambda: tokens.layer_norm(x.double()), "float32"),
        (lambda: tokens.layer_norm(x, rnd(9)), "weight"),
        (lambda: tokens.layer_norm(x, rnd(8).to(torch.bfloat16)), "weight"),
        (lambda: tokens.layer_norm(x.bfloat16(), rnd(8), rnd(8).bfloat16()), "types"),
        (lambda: tokens.layer_norm(x, torch.ones(8)), "tensors on"),
        (lambda: tokens.layer_norm(x, eps=-1.0), "eps"),
        (lambda: tokens.layer_norm(torch.empty(3, 0, device=DEV)), "at least one channel"),
        (lambda: tokens.layer_norm(torch.tensor(1.0, device=DEV)), "at least one channel"),
        (lambda: tokens.gated_ffn(x, w, w, w), "w_down"),
        (lambda: tokens.gated_ffn(x, w[:, :7], w, wd), "w_gate"),
        (lambda: tokens.gated_ffn(x, w, w[:15], wd), "w_up"),
        (lambda: tokens.gated_ffn(x, w.bfloat16(), w, wd), "w_gate"),
        (lambda: tokens.gated_ffn(x, w[:0], w[:0], wd[:, :0]), "w_gate"),
        (lambda: tokens.gated_ffn(x, w[0], w, wd), "w_gate"),
        (lambda: tokens.gated_ffn(x, w, w, wd, rnd(8)), "b_gate"),
        (lambda: tokens.gated_ffn(x, w, w, wd, None, rnd(16).bfloat16()), "b_up"),
        (lambda: tokens.gated_ffn(x, w, w, wd.cpu()), "tensors on"),
        (lambda: tokens.gated_ffn(x, w, w, wd, activation="swish"), "activation"),
        (lambda: tokens.gated_ffn(x.long(), w, w, wd), "float32"),
        (lambda: tokens.dropout(x, 1.5, rng), "probability"),
        (lambda: tokens.dropout(x, float("nan"), rng), "probability"),
        (lambda: tokens.dropout(x, 0.5, rng.int()), "int64"),
        (lambda: tokens.dropout(x, 0.5, rng[:1]), "int64"),
        (lambda: tokens.dropout(x, 0.5, rng.cpu()), "tensors on"),
        (lambda: tokens.dropout(x, 0.5, rng, site=-1), "site"),
        (lambda: tokens.dropout(x, 0.5, rng, residual=x[:3]), "skip"),
        (lambda: tokens.dropout(x, 0.5, rng, residual=x.bfloat16()), "skip"),
    ]
    for k, (call, match) in enumerate(bad):
        with pytest.raises(RuntimeError, match=match):
            call()
            pytest.fail(f"call {k} was not refused")
    saved = token_ops.gated_ffn_fwd(x, w, w, wd, None, None, None, 0, True)[1]
    for s in (saved[:1].expand(saved.numel()), saved.float(), saved[:-512], saved[8:]):
        with pytest.raises(RuntimeError, match="saved"):
            token_ops.gated_ffn_bwd(x, x, w, w, wd, s, 0, [True] * 7)
    # gradients are once differentiable, and say so
    xg = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(tokens.layer_norm(xg).square().sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), xg)
