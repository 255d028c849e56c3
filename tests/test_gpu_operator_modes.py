"""GPU: the embedding, the adapters, the distillation loss and the latent MLPs under what torch puts around calls: forward mode, tracing, function
transforms, second derivatives.  What an operator has no rule for is refused, never answered wrongly."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


def _calls():
    """name -> (function of its differentiable inputs alone, those inputs)"""
    from unet_amd import adapter_linear, distillation_loss, scaled_embedding
    from unet_amd.latent import ParamToZ
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).cuda()
    ids = torch.randint(-1, 6, (11,), generator=g).cuda()
    w, b, A, B, who = r(9, 8), r(9), r(3, 2, 8), r(3, 9, 2), torch.randint(-1, 3, (11,), generator=g).cuda()
    top, idx = r(11, 4), torch.randint(0, 30, (11, 4), generator=g).cuda()
    torch.manual_seed(2)
    mlp = ParamToZ(4, 6, hidden=(16, 8)).cuda().eval()
    for p in mlp.parameters():
        p.requires_grad_(False)
    return {
        "scaled_embedding": (lambda t: scaled_embedding(ids, t, 2.0), (r(6, 5),)),
        "adapter_linear": (lambda x, a, c: adapter_linear(x, w, b, a, c, who), (r(11, 8), A, B)),
        "adapter_linear, many rows": (lambda x, a, c: adapter_linear(x, w, b, a, c, who.repeat(9)), (r(99, 8), A, B)),
        "distillation_loss": (lambda z: distillation_loss(z, top, idx), (r(11, 30),)),
        "distillation_loss, per row": (lambda z: distillation_loss(z, top, idx, weights=torch.ones(11, device="cuda"), reduction="none"), (r(11, 30),)),
        "latent MLP": (mlp, (r(11, 4),)),
    }


NAMES = ["scaled_embedding", "adapter_linear", "adapter_linear, many rows", "distillation_loss", "distillation_loss, per row", "latent MLP"]


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused_not_dropped(name):
    fn, args = _calls()[name]
    for at in range(len(args)):
        with forward_ad.dual_level():
            dual = [forward_ad.make_dual(a, torch.ones_like(a)) if i == at else a for i, a in enumerate(args)]
            with pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
                fn(*dual)
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(fn, args, tuple(torch.ones_like(a) for a in args))
    with forward_ad.dual_level():
        a = fn(*args)                                     # no tangent anywhere: the value
    assert torch.equal(a, fn(*args))


@pytest.mark.parametrize("name", NAMES)
def test_a_trace_computes(name):
    """Traced without gradients, replayed on other inputs."""
    fn, args = _calls()[name]
    with torch.no_grad():
        traced = torch.jit.trace(fn, args, check_trace=False)
        for k in (1.0, -0.5, 3.0):
            other = tuple(a * k for a in args)
            torch.full((1 << 16,), float("nan"), device="cuda")      # what a reused allocation may hold
            assert torch.equal(traced(*other), fn(*other))


@pytest.mark.parametrize("name", NAMES)
def test_batched_transforms_are_refused(name):
    fn, args = _calls()[name]
    with pytest.raises(RuntimeError):
        torch.func.vmap(fn)(*(a.unsqueeze(0).repeat(2, *([1] * a.dim())) for a in args))
@pytest.mark.parametrize("name", NAMES[:5])
def test_second_derivatives_are_refused_where_they_are_taken(name):
    """Under create_graph the first derivatives are what they are without it, beside a penalty on other gradients of the same graph; differentiating
    them raises."""
    fn, args = _calls()[name]
    for wanted in range(len(args)):                       # one input at a time, then its gradients with all of them
        leaves = [a.clone().requires_grad_(i == wanted or wanted == 0) for i, a in enumerate(args)]
        live = [t for t in leaves if t.requires_grad]
        plain = torch.autograd.grad(fn(*leaves).square().sum(), live)
        grads = torch.autograd.grad(fn(*leaves).square().sum(), live, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(plain, grads))
        for g in grads:
            assert g.requires_grad
            with pytest.raises(RuntimeError, match="not differentiable twice"):
                torch.autograd.grad(g.sum(), live, retain_graph=True, allow_unused=True)
    # a gradient penalty elsewhere in the graph
    u = torch.randn(5, device="cuda", requires_grad=True)
    leaves = [a.clone().requires_grad_(True) for a in args]
    total = fn(*leaves).sum() + (u ** 3).sum()
    gu, *rest = torch.autograd.grad(total, (u, *leaves), create_graph=True)
    (gu.square().sum() + total).backward()
    # 9 u^4 and u^3, each product and sum rounded
    want = 36 * u.detach() ** 3 + 3 * u.detach() ** 2
    assert bool(((u.grad - want).abs() <= 1e-5 * (36 * u.detach().abs() ** 3 + 3 * u.detach() ** 2)).all())
    for leaf, g in zip(leaves, rest):
        assert torch.equal(leaf.grad, g.detach())


def test_a_first_derivative_of_the_distillation_depends_on_its_logits():
    """The upstream gradient of a plain .backward(create_graph=True) needs no gradient itself, the result does: a penalty on it must not lose its
    term in silence."""
    from unet_amd import distillation_loss
    z = torch.randn(3, 20, device="cuda", requires_grad=True)
    top, idx = torch.randn(3, 2, device="cuda"), torch.zeros(3, 2, dtype=torch.int64, device="cuda")
    (g,) = torch.autograd.grad(distillation_loss(z, top, idx), (z,), create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable twice"):
        (distillation_loss(z, top, idx) + g.square().sum()).backward()


def test_gradients_that_depend_on_nothing_are_constants():
    """The table's gradient is linear in the upstream one alone: with a constant one there is nothing to differentiate."""
    from unet_amd import scaled_embedding
    t = torch.randn(4, 3, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(scaled_embedding(torch.tensor([0, 2, 2], device="cuda"), t).sum(), (t,), create_graph=True)
    assert not g.requires_grad and torch.equal(g[2], torch.full((3,), 2.0, device="cuda"))


def test_sizes_beyond_a_c_int_are_refused():
    """2^32 + 8 columns must not become 8 on their way into the library.  Views of one element: nothing of that size is allocated."""
    from unet_amd import adapter_linear, distillation_loss, scaled_embedding
    w = (1 << 32) + 8
    one, zero = torch.ones(1, 1, device="cuda"), torch.zeros(1, 1, dtype=torch.int64, device="cuda")
    before = torch.cuda.memory_allocated()
    with pytest.raises(ValueError, match="too long"):
        scaled_embedding(zero[0], one.expand(1, w))
    with pytest.raises(ValueError, match="too large"):
        adapter_linear(one.expand(1, w), one.expand(1, w), None, one[None].expand(1, 1, w), one[None], zero[0])
    with pytest.raises(ValueError, match="too large"):
        adapter_linear(one, one.expand(w, 1), None, one[None], one[None].expand(1, w, 1), zero[0])
    with pytest.raises(ValueError, match="at most"):
        adapter_linear(one, one, None, one[None].expand(w, 1, 1), one[None].expand(w, 1, 1), zero[0])
    with pytest.raises(ValueError, match="too long"):
        distillation_loss(one.expand(1, w), one, zero)
    with pytest.raises(ValueError, match="too long"):
        distillation_loss(one, one.expand(1, w), zero.expand(1, w))
    assert torch.cuda.memory_allocated() == before


@pytest.mark.parametrize("name", NAMES[:5])
def test_recomputed_forward_passes(name):
    """Non-reentrant checkpoints hand each saved tensor out once, with and without create_graph; all through offloaded ones too."""
    from torch.utils.checkpoint import checkpoint
    fn, args = _calls()[name]
    leaves = [a.clone().requires_grad_(True) for a in args]
    want = torch.autograd.grad(fn(*leaves).square().sum(), leaves)
    for create in (False, True):
        y = checkpoint(fn, *leaves, use_reentrant=False)
        got = torch.autograd.grad(y.square().sum(), leaves, create_graph=create)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        with torch.autograd.graph.save_on_cpu():
            y = fn(*leaves)
        got = torch.autograd.grad(y.square().sum(), leaves, create_graph=create)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
