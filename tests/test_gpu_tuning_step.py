"""GPU: a tuning step as its parts are used together -- ids -> scaled embedding -> shared projection with adapters -> distillation from a
teacher's top logits -> gradients -> clip and AdamW -- against the same step in 64 bits, and the adapters inside the latent MLPs.

Tolerance of a gradient, u = 2^-24: the logits z are off by dz = (K + r + 8) u (|W||e| + |b| + 2 |B||h|), which changes q by at most
4 dz / tau of itself; the loss's own gradient is off by E = (6 A + V / 64 + 64) u of (q + p) (tests/test_gpu_distill.py); every later sum of n
terms adds n u of its sum of absolute values.  So each gradient is within (E + 4 max dz / tau + (T + K + V + 64) u) of the same chain with
every factor replaced by its absolute value."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _case():
    g = torch.Generator().manual_seed(3)
    T, M, K, V, r, G, Kt, tau, scale = 150, 40, 48, 300, 6, 5, 12, 2.0, 6.0
    d = dict(ids=torch.randint(-1, M, (T,), generator=g), who=torch.randint(-1, G, (T,), generator=g), E=torch.randn(M, K, generator=g) / scale,
             W=torch.randn(V, K, generator=g) / K ** 0.5, b=torch.randn(V, generator=g), A=torch.randn(G, r, K, generator=g) / K ** 0.5,
             B=torch.randn(G, V, r, generator=g) / r ** 0.5, sc=0.5 + torch.rand(G, generator=g), top=torch.randn(T, Kt, generator=g) + 4,
             idx=torch.randint(-1, V, (T, Kt), generator=g), w=(torch.rand(T, generator=g) < 0.8).float())
    return d, tau, scale


def _reference(d, tau, scale):
    """Loss and gradients in 64 bits, and the bounds of the gradients."""
    x = {k: v.double() if v.is_floating_point() else v for k, v in d.items()}
    ok = x["ids"] >= 0
    e = torch.where(ok[:, None], scale * x["E"][x["ids"].clamp(min=0)], torch.zeros(1, dtype=torch.float64))
    has = (x["who"] >= 0)[:, None]
    a = x["who"].clamp(min=0)
    s = torch.where(has[:, 0], x["sc"][a], torch.zeros(1, dtype=torch.float64))[:, None]
    Aa, Ba = x["A"][a], x["B"][a]
    h = s * torch.matmul(Aa, e[:, :, None])[:, :, 0]
    ha = s * torch.matmul(Aa.abs(), e.abs()[:, :, None])[:, :, 0]
    z = e @ x["W"].t() + x["b"] + torch.matmul(Ba, h[:, :, None])[:, :, 0]
    K, V, r, T = e.shape[1], z.shape[1], h.shape[1], z.shape[0]
    dz = (K + r + 8) * U * (e.abs() @ x["W"].abs().t() + x["b"].abs() + 2 * torch.matmul(Ba.abs(), ha[:, :, None])[:, :, 0])
    logq = torch.log_softmax(z / tau, 1)
    live = x["idx"] >= 0
    t = torch.where(live, x["top"] / tau, torch.full_like(x["top"], -1e300))
    logp = torch.log_softmax(t, 1)
    p = torch.where(live, logp.exp(), torch.zeros_like(logp))
    some = live.any(1).double() * x["w"]
    den = x["w"].sum()
    at = x["idx"].clamp(min=0)
    loss = ((p * (logp - torch.gather(logq, 1, at))).nan_to_num(0.0).sum(1) * tau * tau * some).sum() / den
    c = (tau * some / den)[:, None]
    sp = torch.zeros_like(z).scatter_add_(1, at, p)
    q = logq.exp()
    g, ga = c * (q - sp), c * (q + sp)

    def chain(g, e, h, W, A, B):
        dh = s * torch.matmul(B.transpose(1, 2), g[:, :, None])[:, :, 0]
        de = g @ W + torch.matmul(A.transpose(1, 2), dh[:, :, None])[:, :, 0]
        dE = torch.zeros_like(x["E"]).index_add_(0, x["ids"].clamp(min=0), torch.where(ok[:, None], de, torch.zeros_like(de))) * scale
        G = x["A"].shape[0]
        dA, dB = torch.zeros_like(x["A"]), torch.zeros_like(x["B"])
        for i in range(G):
            m = x["who"] == i
            dA[i], dB[i] = dh[m].t() @ e[m], g[m].t() @ h[m]
        return dE, dA, dB
    spread = max(float((z.max(1).values - z.min(1).values).max()), 10.0) / tau
    rel = (6 * spread + V / 64 + 64) * U + 4 * float(dz.max()) / tau + (T + K + V + 64) * U
    grads = chain(g, e, h, x["W"], Aa, Ba)
    sizes = chain(ga, e.abs(), ha, x["W"].abs(), Aa.abs(), Ba.abs())
    return float(loss), grads, [rel * v for v in sizes], rel


def test_one_step_through_all_of_it():
    from unet_amd import AdapterLinear, ScaledEmbedding, _lib as L, distillation_loss
    d, tau, scale = _case()
    emb = ScaledEmbedding(*d["E"].shape, scale=scale).cuda()
    lin = torch.nn.Linear(d["W"].shape[1], d["W"].shape[0]).cuda()
    with torch.no_grad():
        emb.weight.copy_(d["E"]), lin.weight.copy_(d["W"]), lin.bias.copy_(d["b"])
    head = AdapterLinear(lin, d["A"].shape[0], d["A"].shape[1])
    with torch.no_grad():
        head.A.copy_(d["A"]), head.B.copy_(d["B"]), head.scales.copy_(d["sc"])
    logits = head(emb(d["ids"].cuda()), d["who"].cuda())
    loss = distillation_loss(logits, d["top"].cuda(), d["idx"].cuda(), temperature=tau, weights=d["w"].cuda())
    loss.backward()
    ref, grads, tols, rel = _reference(d, tau, scale)
    assert abs(float(loss.detach()) - ref) <= 20 * rel * max(1.0, abs(ref)) * tau * tau
    params = (emb.weight, head.A, head.B)
    for p, g, t in zip(params, grads, tols):
        assert ((p.grad.double().cpu() - g).abs() <= t + 1e-30).all()
    assert lin.weight.grad is None and lin.bias.grad is None
    # clip + AdamW over one arena, as the framework's trainers do; the first step moves every parameter with a gradient by about lr
    flat = torch.cat([p.detach().reshape(-1) for p in params])
    grad = torch.cat([p.grad.reshape(-1) for p in params])
    before, m, v = flat.clone(), torch.zeros_like(flat), torch.zeros_like(flat)
    parts, norm = torch.zeros(256, device="cuda"), torch.zeros(1, device="cuda")
    n = L.check(L.lib().sx_grad_sumsq_partial(L.ptr(grad), grad.numel(), L.ptr(parts), L.stream_ptr()))
    L.check(L.lib().sx_adamw_step_fused(L.ptr(flat), L.ptr(grad), L.ptr(m), L.ptr(v), flat.numel(), 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1e9, L.ptr(parts), n,
                                        1.0, L.ptr(norm), L.stream_ptr()))
    want = torch.cat([g.reshape(-1) for g in grads])
    assert abs(float(norm) - float(want.norm())) <= 1e-4 * float(want.norm())
    moved = (flat - before).cpu()
    big = want.abs() > 1e-3 * want.abs().max()
    assert ((moved + 1e-3 * want.sign().float()).abs()[big] <= 2e-5).all()      # lr * g / (|g| + eps), eps = 1e-8 against |g| above 1e-5


def test_step_captured_in_a_graph():
    from unet_amd import adapter_linear, distillation_loss, scaled_embedding
    d, tau, scale = _case()
    t = {k: v.cuda() for k, v in d.items()}
    for k in ("E", "A", "B"):
        t[k].requires_grad_(True)

    def step():
        z = adapter_linear(scaled_embedding(t["ids"], t["E"], scale), t["W"], t["b"], t["A"], t["B"], t["who"], scales=t["sc"])
        loss = distillation_loss(z, t["top"], t["idx"], temperature=tau, weights=t["w"])
        return (loss.detach(), *torch.autograd.grad(loss, (t["E"], t["A"], t["B"])))
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    g = torch.Generator().manual_seed(9)
    for _ in range(3):
        with torch.no_grad():
            t["ids"].copy_(torch.randint(-1, 40, (150,), generator=g)), t["who"].copy_(torch.randint(-1, 5, (150,), generator=g))
            t["A"].add_(0.01), t["top"].mul_(1.1)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("layernorm", [False, True])
def test_adapted_latent_mlp(layernorm):
    """The latent MLPs with adapters: B = 0 gives the shared MLP's own output, and a step's gradients agree with the same network in 64 bits
    up to 1e-4 of their norm (fp32 sums of at most 48 terms through three layers: 3 * 2 * 60 * 2^-24 ~ 2e-5 per factor)."""
    from unet_amd import AdaptedMLP
    from unet_amd.latent import ZToParam
    torch.manual_seed(5)
    mlp = ZToParam(24, 5, hidden=(48, 32), use_layernorm=layernorm).cuda().eval()
    x, ids = torch.randn(37, 24, device="cuda"), torch.randint(-1, 3, (37,), device="cuda")
    with torch.no_grad():
        shared = mlp(x)
    m = AdaptedMLP(mlp, 3, 4)
    with torch.no_grad():
        assert (m(x, ids) - shared).abs().max() <= 1e-5
    for l in m.net:
        if hasattr(l, "B"):
            torch.nn.init.normal_(l.B, std=0.2)
    tgt = torch.randn(37, 5, device="cuda")
    (m(x, ids) - tgt).square().mean().backward()
    h, leaves = x.double().cpu(), []
    for l in m.net:
        if hasattr(l, "B"):
            A, B = l.A.detach().double().cpu().requires_grad_(True), l.B.detach().double().cpu().requires_grad_(True)
            leaves += [(l.A, A), (l.B, B)]
            y = h @ l.linear.weight.detach().double().cpu().t() + l.linear.bias.detach().double().cpu()
            on = (ids.cpu() >= 0)[:, None]
            a = ids.cpu().clamp(min=0)
            low = torch.matmul(B[a], torch.matmul(A[a], h[:, :, None]))[:, :, 0] * l.scales.double().cpu()[a][:, None]
            h = y + torch.where(on, low, torch.zeros_like(low))
        elif isinstance(l, torch.nn.LayerNorm):
            h = torch.nn.functional.layer_norm(h, (h.shape[1],), l.weight.detach().double().cpu(), l.bias.detach().double().cpu(), l.eps)
        else:
            h = torch.nn.functional.silu(h)
    (h - tgt.double().cpu()).square().mean().backward()
    for p, q in leaves:
        assert float((p.grad.double().cpu() - q.grad).norm()) <= 1e-4 * float(q.grad.norm())
    assert all(q.grad is None for n, q in m.named_parameters() if not n.endswith((".A", ".B")))
