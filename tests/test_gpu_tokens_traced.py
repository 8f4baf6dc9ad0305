"""GPU: the operators on rows of channels in compiled code and as registered ops: the results and gradients of the eager calls."""
import pytest
import torch
from torch import nn
from torch.fx.experimental.proxy_tensor import make_fx

from super_resolution_amd import tokens

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rnd(*shape, seed=0, scale=1.0, shift=0.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype).to(DEV)


def arguments(dtype, rows=37, c=24, f=40):
    x, w, b = rnd(rows, c, seed=1, dtype=dtype), rnd(c, seed=2, shift=1.0), rnd(c, seed=3)
    ws = [rnd(*s, seed=4 + k, scale=0.2, dtype=dtype) for k, s in enumerate(((f, c), (f, c), (c, f)))]
    bs = [rnd(n, seed=7 + k, dtype=dtype) for k, n in enumerate((f, f, c))]
    return [v.requires_grad_() for v in (x, w, b, *ws, *bs)], torch.tensor([5, 6], device=DEV), rnd(rows, c, seed=10, dtype=dtype)


def step(rng, x, w, b, wg, wu, wd, bg, bu, bd):
    h = tokens.gated_ffn(tokens.layer_norm(x, w, b), wg, wu, wd, bg, bu, bd, activation="gelu")
    return tokens.dropout(h, 0.25, rng, 2, x)


def same(a, b):
    return all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_compiled_in_one_graph(dtype, backend):
    torch._dynamo.reset()
    compiled = torch.compile(step, fullgraph=True, backend=backend)
    for rows in (37, 50, 1):                                       # (the second number of rows makes it symbolic)
        leaves, rng, dy = arguments(dtype, rows)
        want = step(rng, *leaves)
        got = compiled(rng, *leaves)
        assert torch.equal(got, want)
        assert same(torch.autograd.grad(got, leaves, dy), torch.autograd.grad(want, leaves, dy))
        with torch.no_grad():
            assert torch.equal(compiled(rng, *leaves), want)


def test_a_compiled_block_trains():
    torch._dynamo.reset()
    torch.manual_seed(3)
    net = nn.Sequential(tokens.FeedForwardBlock(24, 40, dropout=0.2), tokens.FeedForwardBlock(24, 40, dropout=0.2)).to(DEV)
    state = {k: v.clone() for k, v in net.state_dict().items()}
    x, dy = rnd(30, 24, seed=20, dtype=torch.bfloat16), rnd(30, 24, seed=21, dtype=torch.bfloat16)

    def run(f):
        net.load_state_dict(state)
        out = []
        for _ in range(3):
            y = f(x)
            out += [y.detach(), *torch.autograd.grad(y, list(net.parameters()), dy)]
        return out + [b.rng_state.clone() for b in net]

    assert same(run(torch.compile(net, fullgraph=True, backend="aot_eager")), run(net))


def test_the_registered_ops_have_gradients():
    """Also where their caller did not ask for what the backward pass reads."""
    leaves, rng, dy = arguments(torch.bfloat16)
    x, w, b, *ws = leaves
    ops = torch.ops.sr355
    for keep in (True, False):
        pairs = ((ops.layer_norm_fwd(x, w, b, 1e-5, keep)[0], tokens.layer_norm(x, w, b), [x, w, b]),
                 (ops.layer_norm_fwd(x, None, b, 1e-5, keep)[0], tokens.layer_norm(x, None, b), [b]),
                 (ops.gated_ffn_fwd(x, *ws, 0, keep)[0], tokens.gated_ffn(x, *ws), [x, *ws]),
                 (ops.dropout(x, x, 0.3, rng, 1), tokens.dropout(x, 0.3, rng, 1, x), [x]))
        for got, want, vs in pairs:
            assert torch.equal(got, want)
            assert same(torch.autograd.grad(got, vs, dy), torch.autograd.grad(want, vs, dy))


def test_functional_transforms_are_refused():
    """(Through a registered op a tangent would be lost without a word.)"""
    leaves, rng, dy = arguments(torch.float32)
    loss = lambda *a: (step(rng, *a) * dy).sum()
    values = tuple(v.detach() for v in leaves)
    for transform in (lambda: torch.func.grad(loss)(*values), lambda: torch.func.jvp(loss, values, values),
                      lambda: torch.func.vjp(tokens.layer_norm, values[0])[1](dy), lambda: torch.vmap(tokens.layer_norm)(values[0]),
                      lambda: torch.func.jvp(tokens.layer_norm, (values[0],), (dy,)),
                      lambda: torch.func.jvp(lambda t: tokens.dropout(t, 0.5, rng), (values[0],), (dy,))):
        with pytest.raises(RuntimeError, match="torch.func"):
            transform()


def test_a_training_step_is_traced():
    leaves, rng, dy = arguments(torch.bfloat16)
    values = [v.detach() for v in leaves]

    def train(*a):
        vs = [v.detach().requires_grad_() for v in a]
        return torch.autograd.grad(step(rng, *vs), vs, dy)

    graph = make_fx(train, tracing_mode="real")(*values)
    ops = sorted(n.target.name().split("::")[1] for n in graph.graph.nodes if n.op == "call_function" and "sr355" in str(n.target))
    assert ops == ["dropout", "dropout", "gated_ffn_bwd", "gated_ffn_fwd", "layer_norm_bwd", "layer_norm_fwd"]
    assert same(graph(*values), train(*values))
