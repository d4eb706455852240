"""The differentiable functions' dealings with autograd, on the CPU: the
operators behind them are stood in for by torch operations, which also note
what they were asked for."""
import pytest
import torch

from warchest_b200 import SolveError
from warchest_b200 import train_layers as layers
from warchest_b200 import train_ops as ops


@pytest.fixture
def asked(monkeypatch):
    """Stand-ins for the operators; the list of what was called."""
    calls = []

    def note(f):
        def g(*args, **options):
            calls.append(f.__name__)
            return f(*args, **options)

        monkeypatch.setattr(ops, f.__name__, g)

    @note
    def act8_pack(x):
        return ops.Act8(x.detach().clone(), torch.zeros(len(x), 1), x.shape[1])

    @note
    def gelu8(z, bias=None):
        s = z if bias is None else z + bias
        return torch.nn.functional.gelu(s, approximate="tanh"), ops.Act8(s.detach().clone(), torch.zeros(len(z), 1), z.shape[1])

    @note
    def gelu8_backward(da, z8, want_bias=True):
        with torch.enable_grad():
            z = z8.q.detach().clone().requires_grad_()
            dz, = torch.autograd.grad(torch.nn.functional.gelu(z, approximate="tanh"), z, da)
        return dz, dz.sum(0) if want_bias else None

    @note
    def act8_wgrad(x8, dy, *, dtype=torch.float32, want_bias=True):
        return x8.q.t() @ dy, dy.sum(0) if want_bias else None

    @note
    def block_norm(x, h, *, gate=None, rows_per_gate=None, residual_scale=1.0, post=None, pre=None, kind="layer", eps=1e-5, pack=False):
        y = residual_scale * x + h * (1 if post is None else post[0])
        n = None if pre is None else y * y * pre[0]
        return ops.BlockNorm(y, n, act8_pack(n) if pack else None, torch.zeros(len(x), 4))

    @note
    def block_norm_backward(dy, dn, x, h, stats, *, gate=None, rows_per_gate=None, residual_scale=1.0, post=None, pre=None, kind="layer",
                            eps=1e-5, want=None):
        calls.append(want)
        y = residual_scale * x + h * (1 if post is None else post[0])
        d = (0 if dy is None else dy) + (0 if dn is None else 2 * dn * y * pre[0])
        return ops.BlockNormGrads(residual_scale * d, d * (1 if post is None else post[0]), None, None if post is None else (d * h).sum(0), None,
                                  None if pre is None else (dn * y * y).sum(0), None)

    @note
    def policy_loss(logits, actions, old_logp, advantages, *, weights=None, ref_logp=None, legal=None, upstream=None, want_grad=True, **unused):
        p = torch.softmax(logits.detach(), 1)
        hit = torch.nn.functional.one_hot(actions, logits.shape[1])
        logp = (p * hit).sum(1).log()
        up = 1.0 if upstream is None else upstream
        return ops.PolicyLoss(-(logp * advantages).sum(), logp, logp.clone(), logp.clone(), logp.clone(),
                              up * advantages[:, None] * (p - hit) if want_grad else None)

    return calls


def leaf(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).requires_grad_()


def losses():
    """Each function as a scalar of some leaves."""
    x, h, w, b = leaf(5, 4, seed=1), leaf(5, 4, seed=2), leaf(4, 3, seed=3), leaf(3, seed=4)
    post, pre = leaf(4, seed=5), leaf(4, seed=6)
    a = torch.tensor([0, 3, 2, 1, 0])
    return {"policy_loss": (lambda: layers.policy_loss(x, a, x[:, 0].detach(), x[:, 1].detach()).loss, [x]),
            "block_norm": (lambda: sum(v.sum() for v in layers.block_norm(x, h, post=post, pre=pre)), [x, h, post, pre]),
            "gelu8": (lambda: layers.gelu8(x).sum(), [x]), "gelu8 bias": (lambda: layers.gelu8(x[:, :3], b).sum(), [x, b]),
            "linear8": (lambda: layers.linear8(x, w, b).sum(), [x, w, b])}


@pytest.mark.parametrize("name", ["policy_loss", "block_norm", "gelu8", "gelu8 bias", "linear8"])
def test_second_derivatives_raise(asked, name):
    f, leaves = losses()[name]
    first = torch.autograd.grad(f(), leaves)
    graph = torch.autograd.grad(f(), leaves, create_graph=True)
    for a, b in zip(first, graph):
        assert torch.equal(a, b) and not a.requires_grad
        # alone, and beside a term that has a derivative
        for penalty in (b.square().sum(), b.square().sum() + leaves[0].sum()):
            with pytest.raises(SolveError, match="second derivative"):
                torch.autograd.grad(penalty, leaves, retain_graph=True, allow_unused=True)


def test_a_gradient_penalty_through_several_raises(asked):
    w1, w2, x = leaf(4, 6, seed=7), leaf(6, 2, seed=8), leaf(5, 4, seed=9)
    y = layers.linear8(layers.gelu8(layers.linear8(x, w1)), w2)
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(SolveError, match="second derivative"):
        (y.sum() + g.square().sum()).backward(retain_graph=True)
    for leaf_of in (w1, w2, x):
        with pytest.raises(SolveError, match="second derivative"):
            torch.autograd.grad(g.square().sum() + leaf_of.sum(), leaf_of, retain_graph=True)


def test_gradients_under_create_graph_reach_the_leaves(asked):
    for f, leaves in losses().values():
        want = torch.autograd.grad(f(), leaves)
        f().backward(create_graph=True)
        for t, g in zip(leaves, want):
            assert torch.equal(t.grad, g)
            t.grad = None


def test_linear8_keeps_its_input_only_for_a_weight_gradient(asked):
    x, w, b = leaf(5, 4, seed=1), leaf(4, 3, seed=3), leaf(3, seed=4)
    want = torch.autograd.grad(layers.linear8(x, w, b).square().sum(), (x, b))
    assert asked == ["act8_pack", "act8_wgrad"]
    del asked[:]
    frozen = w.detach()
    for a, g in zip(want, torch.autograd.grad(layers.linear8(x, frozen, b).square().sum(), (x, b))):
        assert torch.equal(a, g)
    with torch.no_grad():
        assert torch.equal(layers.linear8(x, w, b), x @ w + b)
    assert layers.linear8(x.detach(), frozen).shape == (5, 3)
    assert asked == []
    g, = torch.autograd.grad(layers.linear8(x.detach(), w, b.detach(), x8=ops.Act8(x.detach(), torch.zeros(5, 1), 4)).sum(), w)
    assert torch.equal(g, x.detach().t() @ torch.ones(5, 3)) and asked == ["act8_wgrad"]


def test_block_norm_forms_the_gradients_that_are_wanted(asked):
    x, h, post, pre = leaf(5, 4, seed=1), leaf(5, 4, seed=2), leaf(4, seed=5), leaf(4, seed=6)
    for some in ((x,), (h, pre), (post,), (x, h, post, pre)):
        del asked[:]
        on = lambda t: t if any(t is s for s in some) else t.detach()  # noqa: E731
        y, n = layers.block_norm(on(x), on(h), post=on(post), pre=on(pre))
        torch.autograd.grad(y.sum() + n.sum(), some)
        assert asked[1:] == ["block_norm_backward", tuple(any(t is s for s in some) for t in (x, h, None, post, None, pre, None))]


def test_gelu8_sums_its_bias_only_for_a_gradient(asked, monkeypatch):
    z, b = leaf(5, 4, seed=1), leaf(4, seed=2)
    seen, real = [], ops.gelu8_backward
    monkeypatch.setattr(ops, "gelu8_backward", lambda da, z8, want_bias=True: (seen.append(want_bias), real(da, z8, want_bias=want_bias))[1])
    torch.autograd.grad(layers.gelu8(z, b).sum(), (z, b))
    torch.autograd.grad(layers.gelu8(z, b.detach()).sum(), z)
    assert seen == [True, False]


@pytest.mark.parametrize("rows,width", [(4, 4), (5, 3), (6, 4)])
def test_linear8_refuses_the_8_bits_of_another_input(asked, rows, width):
    """Before the forward pass, and also where the blocks are as many (a width of 3 for 4)."""
    x, w = leaf(5, 4, seed=1), leaf(4, 3, seed=3)
    with pytest.raises(SolveError, match="differ in shape") as e:
        layers.linear8(x, w, x8=ops.Act8(torch.zeros(rows, 32, dtype=torch.int8), torch.zeros(rows, 1, dtype=torch.uint8), width))
    assert e.value.code == 1
