"""GPU: the operators on rows of channels where one argument differs from what the others are like, and on rows and values at
the ends of their ranges.  Products of small integers are exact, so results have to be equal."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from super_resolution_amd import tokens

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def rnd(*shape, seed=0, scale=1.0, shift=0.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype).to(DEV)


def sparse_ints(rows, cols, per_row, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    at = torch.randint(0, cols, (rows, per_row), generator=g)
    return torch.zeros(rows, cols).scatter_(1, at, torch.randint(0, 2, (rows, per_row), generator=g) * 2.0 - 1).to(dtype).to(DEV)


def ternary(rows, cols, seed, dtype):
    return torch.randint(-1, 2, (rows, cols), generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def T(m):
    return m.t().contiguous()


def relu_block(x, dy, wg, wu, wd):
    """y and the gradients of x and the weights in 64 bits."""
    x, dy, wg, wu, wd = (v.double() for v in (x, dy, wg, wu, wd))
    g, u = x @ T(wg), x @ T(wu)
    h, dh = g.clamp_min(0) * u, dy @ wd
    dg, du = dh * u * (g > 0), dh * g.clamp_min(0)
    return h @ T(wd), dg @ wg + du @ wu, T(dg) @ x, T(du) @ x, T(dy) @ h


@pytest.mark.parametrize("dtype,c", [(torch.bfloat16, 264), (torch.float16, 1000), (torch.float32, 20), (torch.float32, 132)])
@pytest.mark.parametrize("rows", [1, 33, 70, 300])
def test_one_weight_at_an_odd_address(rows, c, dtype):
    """As a view into one flat buffer of parameters has it.  |g|, |u| <= 3, |dh| <= 3: every intermediate is exact in every type."""
    f = 56
    x, dy = sparse_ints(rows, c, 3, 1, dtype), sparse_ints(rows, c, 3, 2, dtype)
    ws = [ternary(f, c, 3, dtype), ternary(f, c, 4, dtype), ternary(c, f, 5, dtype)]
    want = [v.to(dtype) for v in relu_block(x, dy, *ws)]
    for moved in range(3):
        args = list(ws)
        args[moved] = torch.empty(ws[moved].numel() + 1, dtype=dtype, device=DEV)[1:].view(ws[moved].shape).copy_(ws[moved])
        leaves = [v.detach().requires_grad_() for v in (x, *args)]
        y = tokens.gated_ffn(*leaves, activation="relu")
        for got, w in zip((y, *torch.autograd.grad(y, leaves, dy)), want):
            assert torch.equal(got, w), moved
        with torch.no_grad():
            assert torch.equal(tokens.gated_ffn(x, *args, activation="relu"), y), moved


# ---- layer norm around a large value -----------------------------------------------------------------------------------
NORM_WIDTHS = [1, 3, 8, 50, 77, 129, 500, 999, 1000, 2048, 5001, 8192, 9001, 20000]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", NORM_WIDTHS)
@pytest.mark.parametrize("value", [1000.1, 12345.6, -0.3, 7.0, 1e-30, 3e29])
def test_layer_norm_of_equal_channels_is_the_bias(value, c, dtype):
    if value == 3e29 and dtype == torch.float16:
        value = 65504.0
    x = torch.full((5, c), value, dtype=dtype, device=DEV).requires_grad_()
    w, b = rnd(c, seed=20, dtype=dtype).requires_grad_(), rnd(c, seed=21, dtype=dtype).requires_grad_()
    y = tokens.layer_norm(x, w, b)
    assert torch.equal(y, b.detach().expand(5, c))
    assert (tokens.layer_norm(x.detach()) == 0).all()
    (dw,) = torch.autograd.grad(y, w, rnd(5, c, seed=22, dtype=dtype))
    assert (dw == 0).all()


@pytest.mark.parametrize("c", [c for c in NORM_WIDTHS if c > 1])
@pytest.mark.parametrize("shift,scale", [(1000.1, 0.01), (12345.6, 0.5), (-3e5, 2.0), (0.5, 1.0)])
def test_layer_norm_far_from_zero_keeps_its_precision(shift, scale, c):
    """The rounding errors of y are those of the channels' distances from the row's first one, whatever is common to them: a sum
    of n terms over 64 lanes and more is fewer than n / 64 + 24 roundings deep."""
    rows, u = 6, 2.0 ** -24
    x = rnd(rows, c, seed=23, scale=scale, shift=shift)
    x[3] = 0.0
    x[3, c // 2] = shift                                        # one channel apart, and its mirror: the first one apart
    x[4] = 0.0
    x[4, 0] = shift
    y = tokens.layer_norm(x)
    d = x.double()
    rstd = 1 / (d.var(1, unbiased=False, keepdim=True) + 1e-5).sqrt()
    xh = (d - d.mean(1, keepdim=True)) * rstd
    far = (d - d[:, :1]).abs().amax(1, keepdim=True)
    tol = u * (c / 64 + 24) * (far * rstd + xh.abs()) * 1.5 + 5 * u * xh.abs()
    bad = (y.double() - xh).abs() > tol
    assert not bad.any(), ((y.double() - xh).abs() / tol).max()


# ---- infinities ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c,f", [(24, 5), (24, 13), (8, 40), (100, 44), (24, 56), (264, 33)])
@pytest.mark.parametrize("rows", [3, 70, 300, 16500])
def test_an_infinity_beside_no_hidden_channels(rows, c, f, dtype):
    """Hidden channels behind the last one, up to whole units and tiles, count for nothing: where the formula gives an infinity, it
    is one.  All values are positive, so that the formula has no NaN."""
    x = torch.ones(rows, c, dtype=dtype, device=DEV)
    x[1, 2] = float("inf")
    dy = torch.ones(rows, c, dtype=dtype, device=DEV)
    ws = [torch.full(s, 0.125, dtype=dtype, device=DEV) for s in ((f, c), (f, c), (c, f))]
    leaves = [v.detach().requires_grad_() for v in (x, *ws)]
    y = tokens.gated_ffn(*leaves, activation="relu")
    got = [y, *torch.autograd.grad(y, leaves, dy)]
    with torch.no_grad():
        got.append(tokens.gated_ffn(x, *ws, activation="relu"))
    want = relu_block(x, dy, *ws)
    u = torch.finfo(dtype).eps / 2
    for k, (a, b) in enumerate(zip(got, (*want, want[0]))):
        assert torch.equal(a.isinf(), b.to(dtype).isinf()) and not a.isnan().any(), k       # (fp16 ends at 65504)
        ok = ~b.to(dtype).isinf()
        assert ((a[ok].double() - b[ok]).abs() <= (3 * u + 2.0 ** -15) * b[ok]).all(), k
    x[1, 2] = 1.0
    dy[2, 1] = float("inf")
    leaves = [v.detach().requires_grad_() for v in (x, *ws)]
    got = torch.autograd.grad(tokens.gated_ffn(*leaves, activation="relu"), leaves, dy)
    for k, (a, b) in enumerate(zip(got, relu_block(x, dy, *ws)[1:])):
        assert torch.equal(a.isinf(), b.to(dtype).isinf()) and not a.isnan().any(), k


# ---- the activations far from zero ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [40, 300, 16500])
def test_gelu_keeps_its_precision_where_it_is_small(rows, dtype):
    """One channel and one hidden channel: y = gelu(x) * 4096 (fp16: 1024), its derivative beside it.  h is rounded to the type and taken over by
    y, or y is rounded once; act' is kept with 16 bits; the normal integral itself is good to 2^-17 of its value."""
    lo = -5.5 if dtype == torch.float16 else -12.0               # fp16: where 1024 gelu(x) is a normal number
    x = torch.linspace(lo, 6.0, rows).to(dtype).to(DEV)[:, None].requires_grad_()
    one = torch.ones(1, 1, dtype=dtype, device=DEV)
    up = torch.full((1,), 4096.0 if dtype != torch.float16 else 1024.0, dtype=dtype, device=DEV)
    d = x.detach().double()
    cdf, density = 0.5 * torch.erfc(-d * 0.5 ** 0.5), torch.exp(-0.5 * d * d) / (2 * torch.pi) ** 0.5
    want, slope = d * cdf * up.item(), (cdf + d * density) * up.item()
    u = torch.finfo(dtype).eps / 2
    # the exponent g^2 / 2 is rounded to fp32: relative to the result that is g^2 / 2 of its steps, twice
    own = 2.0 ** -17 + 2.0 ** -23 * d * d
    y = tokens.gated_ffn(x, one, torch.zeros_like(one), one, None, up, None, activation="gelu")
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    with torch.no_grad():
        alone = tokens.gated_ffn(x, one, torch.zeros_like(one), one, None, up, None, activation="gelu")
    for got in (y, alone):
        bad = (got.double() - want).abs() > (2 * u + own) * want.abs()
        assert not bad.any(), (x[bad][0].item(), got[bad][0].item(), want[bad][0].item())
    size = (cdf + (d * density).abs()) * up.item()
    bad = (dx.double() - slope).abs() > 2 * u * slope.abs() + (own + (2.0 ** -15 if u > 2.0 ** -20 else 0.0)) * size
    assert not bad.any(), (x[bad][0].item(), dx[bad][0].item(), slope[bad][0].item())


# ---- blocks ----------------------------------------------------------------------------------------------------------------
def test_stacked_blocks_drop_different_elements():
    """A dropped element is its skip.  Two masks of independent draws agree on 0.36 + 0.16 of n elements: five standard deviations."""
    torch.manual_seed(31)
    blocks = [tokens.FeedForwardBlock(64, 32, dropout=0.4).to(DEV) for _ in range(2)]
    x, n = rnd(500, 64, seed=32), 500 * 64
    drops = [b(x) == x for b in blocks] + [blocks[0](x) == x]
    for k, a in enumerate(drops):
        assert abs(int(a.sum()) - 0.4 * n) < 5 * (n * 0.24) ** 0.5
        for b in drops[:k]:
            assert abs(int((a == b).sum()) - 0.52 * n) < 5 * (n * 0.52 * 0.48) ** 0.5


def test_forward_mode_derivatives_are_refused():
    x, w, wd, v, rng = rnd(4, 8), rnd(16, 8), rnd(8, 16), rnd(8), torch.zeros(2, dtype=torch.int64, device=DEV)
    dual = lambda t: fwd.make_dual(t, torch.ones_like(t))
    calls = (lambda: tokens.layer_norm(dual(x)), lambda: tokens.layer_norm(x, dual(v)), lambda: tokens.layer_norm(x, v, dual(v)),
             lambda: tokens.layer_norm(dual(x.clone().requires_grad_())), lambda: tokens.gated_ffn(dual(x), w, w, wd),
             lambda: tokens.gated_ffn(x, dual(w), w, wd), lambda: tokens.gated_ffn(x, w, dual(w), wd),
             lambda: tokens.gated_ffn(x, w, w, dual(wd)), lambda: tokens.gated_ffn(x, w, w, wd, None, None, dual(v)),
             lambda: tokens.dropout(dual(x), 0.5, rng), lambda: tokens.dropout(x, 0.5, rng, 0, dual(x)),
             lambda: tokens.FeedForwardBlock(8, 16).to(DEV)(dual(x)), lambda: torch.ops.sr355.dropout(dual(x), None, 0.5, rng, 0))
    for k, call in enumerate(calls):
        with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            call()
            pytest.fail(f"call {k} was not refused")


# ---- layer norm of very long rows ------------------------------------------------------------------------------------------
def test_layer_norm_of_a_row_of_more_than_2_28_channels():
    """One row, so that db is dy and dw one product; the two row means are sums of 2^20 terms a lane."""
    c, u, step = (1 << 28) + 70, 2.0 ** -8, 2.0 ** -24
    g = torch.Generator(DEV).manual_seed(40)
    x, dy, w = (torch.randn(c, device=DEV, generator=g).to(torch.bfloat16) for _ in range(3))
    leaves = [x[None].requires_grad_(), w.requires_grad_(), torch.zeros(c, dtype=torch.bfloat16, device=DEV, requires_grad=True)]
    y = tokens.layer_norm(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dy[None])
    assert torch.equal(db, dy)
    deep = step * (c / 256 + 24)
    with torch.no_grad():
        d = x.double()
        d -= d.mean()
        rstd = (d.square().mean() + 1e-5).rsqrt()
        d *= rstd                                                  # xh: of size one, its mean and scale off by `deep` at most
        want = d * w.double()
        assert ((y[0].double() - want).abs() <= (u + 4 * deep) * want.abs() + 4 * deep * w.double().abs()).all()
        want = d * dy.double()
        assert ((dw.double() - want).abs() <= (u + 4 * deep) * want.abs() + 4 * deep * dy.double().abs()).all()
        t = dy.double() * w.double()
        s, q, size = t.mean(), (t * d).mean(), t.abs().mean()
        want = rstd * (t - s - d * q)
        assert ((dx[0].double() - want).abs() <= (u + 4 * deep) * want.abs() + 8 * deep * size * (1 + d.abs())).all()


def test_layer_norm_refuses_more_channels_than_an_int_counts():
    x, stats = torch.zeros(1, 1, device=DEV).expand(1, (1 << 32) + 8), torch.zeros(2, 1, device=DEV)
    with pytest.raises(RuntimeError, match="channels"):
        tokens.layer_norm(x)
    with pytest.raises(RuntimeError, match="channels"):
        torch.ops.sr355.layer_norm_bwd(x, x, None, stats, torch.float32, [True, False, False])


# ---- captures ----------------------------------------------------------------------------------------------------------------
def test_a_capture_sees_leaves_behind_other_operations():
    """Parameters that are cast for the call, or an input that other layers made: their leaves' gradients are added up by PyTorch,
    too, on the stream of the graph that lives."""
    x, w = rnd(20, 16, seed=50, dtype=torch.bfloat16), rnd(16, seed=51, shift=1.0).requires_grad_()
    ws = [rnd(*s, seed=52 + k, scale=0.2).requires_grad_() for k, s in enumerate(((40, 16), (40, 16), (16, 40)))]
    rng = torch.zeros(2, dtype=torch.int64, device=DEV)
    half = lambda t: t.to(torch.bfloat16)
    calls = (lambda: tokens.layer_norm(x, half(w)), lambda: tokens.gated_ffn(x, *map(half, ws)),
             lambda: tokens.layer_norm(x * half(w) + 1.0), lambda: tokens.dropout(x * half(w), 0.5, rng))
    leaves = ([w], ws, [w], [w])
    want = [torch.autograd.grad(c().float().sum(), v) for c, v in zip(calls, leaves)]
    live = [c() for c in calls]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in calls:
            with pytest.raises(RuntimeError, match="recorded on the default stream"):
                call()
        out = x * 2
    graph.replay()
    assert torch.equal(out, x * 2)
    live.clear()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [torch.autograd.grad(c().float().sum(), v) for c, v in zip(calls, leaves)]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
        torch.cuda.synchronize()
