"""GPU: distillation_loss and its gradient against a plain implementation in 64 bits.

Tolerances, u = 2^-24.  With |z - max| / tau <= A and |top - max| / tau <= A, an argument of exp is off by 3 u A (difference, 1 / tau,
product), an exponential by (3 A + 4) u of itself, a sum of n of them by at most n u more (n = additions in a thread's chain plus the joins,
<= V / 64 + 32), so q and p are off by E = (6 A + V / 64 + 64) u of themselves and each logarithm by as much in absolute terms plus 2 u of its
own size <= 2 u (A + log V).  The row's loss, tau^2 sum p (log p - log q), is off by tau^2 * (2 E + E * max|log p - log q| + 8 u (A + log V)),
the gradient by c (E q + E p) + half a step of its type of itself (plus u for its products, in E)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def _inputs(lead, V, K, dtype=torch.float32, tdtype=torch.float32, idt=torch.int64, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(*lead, V, generator=g) * spread).to(dtype)
    top = (torch.randn(*lead, K, generator=g) * 2.0 + 5.0).to(tdtype)
    idx = torch.randint(0, V, (*lead, K), generator=g).to(idt)               # with entries that name the same index
    return z.cuda().requires_grad_(True), top.cuda(), idx.cuda()


def _ref(z, top, idx, tau, weights, reduction, g=None):
    V = z.shape[-1]
    z, top, idx = z.detach().double().cpu().reshape(-1, V), top.double().cpu().reshape(-1, top.shape[-1]), idx.long().cpu().reshape(-1, idx.shape[-1])
    N = z.shape[0]
    w = torch.ones(N, dtype=torch.float64) if weights is None else weights.double().cpu().reshape(-1)
    den = max(float(w.sum()), 1e-8) if reduction == "mean" else 1.0
    ok = (idx >= 0) & (idx < V)
    loss, grad = torch.zeros(N, dtype=torch.float64), torch.zeros(N, V, dtype=torch.float64)
    etol, ltol = torch.zeros(N, V, dtype=torch.float64), torch.zeros(N, dtype=torch.float64)
    up = torch.ones(N, dtype=torch.float64) if g is None else (g.double().cpu().reshape(-1) if g.dim() or reduction == "none" else g.double().cpu().expand(N))
    for r in range(N):
        if not ok[r].any() or w[r] == 0:
            continue
        logq = torch.log_softmax(z[r] / tau, 0)
        t, i = top[r][ok[r]] / tau, idx[r][ok[r]]
        logp = torch.log_softmax(t, 0)
        p = logp.exp()
        d = torch.where(p > 0, logp - logq[i], torch.zeros_like(p))
        loss[r] = tau * tau * w[r] * (p * d).sum()
        q = logq.exp()
        sp = torch.zeros(V, dtype=torch.float64).index_add_(0, i, p)
        c = up[r] * w[r] * tau / den
        grad[r] = c * (q - sp)
        zf, tf = z[r][torch.isfinite(z[r])], t[torch.isfinite(t)]
        A = max(float((zf.max() - zf.min()) / tau), float(tf.max() - tf.min()))
        A = min(A, 200.0)                                                     # beyond it every exponential is 0 on both sides
        E = (6 * A + V / 64 + 64) * U
        etol[r] = abs(c) * E * (q + sp)
        ltol[r] = tau * tau * abs(w[r]) * (2 * E + E * float(d[torch.isfinite(d)].abs().max() if torch.isfinite(d).any() else 0) + 8 * U * (A + math.log(V)))
    if reduction != "none":
        ltol = (ltol.sum() + N * U * loss.abs().sum()) / den
        loss = loss.sum() / den
    return loss, grad, ltol, etol


def _check(z, top, idx, tau=1.0, weights=None, reduction="mean", g=None):
    from unet_amd.losses import distillation_loss
    loss = distillation_loss(z, top, idx, temperature=tau, weights=weights, reduction=reduction)
    (grad,) = torch.autograd.grad(loss, (z,), g if g is not None else torch.ones_like(loss))
    rl, rg, lt, gt = _ref(z, top, idx, tau, weights, reduction, g)
    assert loss.dtype == torch.float32 and grad.dtype == z.dtype and grad.shape == z.shape
    got = loss.detach().double().cpu().reshape(rl.shape)
    inf = torch.isinf(rl)
    assert torch.equal(torch.isinf(got), inf) and ((got - rl).abs() <= lt + U * rl.abs())[~inf].all(), (got - rl).abs().max()
    gg = grad.double().cpu().reshape(rg.shape)
    assert ((gg - rg).abs() <= gt + 1.01 * (HALF[z.dtype] + U) * rg.abs() + 1e-38).all(), ((gg - rg).abs() - gt).max()
    return loss, grad


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lead,V,K", [((1,), 1, 1), ((3,), 2, 5), ((2, 3), 17, 3), ((5,), 255, 16), ((4,), 256, 1), ((3,), 1024, 64), ((2,), 1025, 128),
                                      ((3,), 4099, 33), ((2,), 8192, 300), ((2,), 33001, 20), ((2,), 65536, 64), ((1,), 131071, 8), ((1,), 140000, 8)])
def test_loss_and_gradient(lead, V, K, dtype):
    for i, (tau, red, tdt, idt) in enumerate(((1.0, "mean", torch.float32, torch.int64), (2.0, "sum", torch.bfloat16, torch.int32), (1.5, "none", torch.float32, torch.int32))):
        z, top, idx = _inputs(lead, V, K, dtype, tdt, idt, seed=i)
        g = torch.randn(lead, generator=torch.Generator().manual_seed(9)).cuda() if red == "none" else None
        _check(z, top, idx, tau, None, red, g)


def test_upstream_gradients_other_than_one_and_a_second_backward():
    from unet_amd.losses import distillation_loss
    for dtype in (torch.float32, torch.bfloat16):
        z, top, idx = _inputs((6,), 777, 9, dtype)
        for red, g in (("mean", torch.tensor(0.3)), ("sum", torch.tensor(1.0)), ("none", torch.tensor([1.0, 0.0, -2.0, 1.0, 0.5, 3.0]))):
            _check(z, top, idx, 2.0, None, red, g.cuda())
        loss = distillation_loss(z, top, idx)
        (a,) = torch.autograd.grad(loss, (z,), retain_graph=True)
        keep = a.clone()
        (b,) = torch.autograd.grad(loss, (z,), torch.tensor(1.0, device="cuda"), retain_graph=True)
        assert torch.equal(a, keep) and torch.equal(a, b) and a.data_ptr() != b.data_ptr()
        loss2 = distillation_loss(z, top, idx)
        loss2 /= 4                                     # gradient accumulation's usual form
        (c,) = torch.autograd.grad(loss2, (z,))
        rg = _ref(z, top, idx, 1.0, None, "mean", torch.tensor(0.25))[1]
        assert ((c.double().cpu() - rg).abs() <= 1e-5 * rg.abs().max() + HALF[dtype] * 1.01 * rg.abs()).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("red", ["mean", "sum", "none"])
def test_masked_rows_hold_nothing_back(dtype, red):
    """Rows of weight 0 and rows whose entries are all padding: loss 0 and gradient 0, with NaN and infinities in their logits."""
    z, top, idx = _inputs((7,), 300, 6, dtype)
    w = torch.tensor([1.0, 0.0, 2.5, 0.0, 1.0, 1.0, 0.5]).cuda()
    with torch.no_grad():
        z[1] = float("nan")
        z[3, 5] = float("inf")
        idx[4] = -1
        z[4, :7] = float("nan")
        top[4] = float("nan")
        idx[5, ::2] = 300                              # outside on the other side
        top[5, ::2] = float("inf")
        top[1] = float("nan")
    from unet_amd.losses import distillation_loss
    loss = distillation_loss(z, top, idx, temperature=1.5, weights=w, reduction=red)
    g = torch.ones_like(loss)
    (grad,) = torch.autograd.grad(loss, (z,), g)
    assert torch.isfinite(loss).all() and torch.isfinite(grad).all()
    assert not grad[[1, 3, 4]].any()
    if red == "none":
        assert not loss.detach()[[1, 3, 4]].any()
    live = [0, 2, 5, 6]
    z2, t2 = z.detach().clone(), top.clone()
    z2[[1, 3, 4]] = 0.0
    t2[[1, 4]] = 0.0
    t2[5, ::2] = 0.0
    rl, rg, lt, gt = _ref(z2, t2, idx, 1.5, w, red)
    assert ((loss.detach().double().cpu() - rl).abs() <= lt + U * rl.abs()).all()
    assert ((grad.double().cpu() - rg).abs() <= gt + 1.01 * (HALF[dtype] + U) * rg.abs())[live].all()


def test_all_rows_masked():
    z, top, idx = _inputs((3,), 50, 4)
    loss, grad = _check(z, top, idx, 1.0, torch.zeros(3).cuda(), "mean")
    assert float(loss) == 0.0 and not grad.any()
    from unet_amd.losses import distillation_loss
    loss, grad = _check(z, top, torch.full_like(idx, -1), 1.0, None, "mean")
    assert float(loss) == 0.0 and not grad.any()
    e = torch.empty(0, 50, device="cuda", requires_grad=True)
    loss = distillation_loss(e, torch.empty(0, 4, device="cuda"), torch.empty(0, 4, dtype=torch.int64, device="cuda"))
    assert float(loss) == 0.0 and torch.autograd.grad(loss, (e,))[0].shape == (0, 50)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lowest_values_and_infinities_in_the_vocabulary(dtype):
    """A masked vocabulary (the type's lowest value or -inf) next to live logits; a teacher entry of -inf has no mass; a teacher entry with
    mass on a -inf logit makes the loss infinite, its gradient stays finite; far offsets cancel."""
    low = torch.finfo(dtype).min
    for fill in (low, float("-inf")):
        z, top, idx = _inputs((4,), 500, 8, dtype)
        idx = idx % 250
        with torch.no_grad():
            z[:, 250:] = fill
            top[0, 3] = float("-inf")
            z[1] += 1000.0
            idx[2, :] = idx[2, 0]
        _check(z, top, idx, 1.0)
    z, top, idx = _inputs((2,), 500, 8, dtype)
    with torch.no_grad():
        z[0, idx[0, 2]] = float("-inf")
    loss, grad = _check(z, top, idx, 1.0, None, "none")
    assert math.isinf(float(loss[0].detach())) and torch.isfinite(grad).all()
    z = torch.full((2, 300), low, dtype=dtype, device="cuda", requires_grad=True)
    _check(z, top, idx % 300, 1.0)


@pytest.mark.parametrize("K", [5, 300])
def test_teacher_rows_without_mass(K):
    """A row whose teacher logits are all -inf has no entry left, also next to padding; one finite entry among them takes all the mass."""
    z, top, idx = _inputs((5,), 700, K)
    with torch.no_grad():
        top[0] = float("-inf")
        top[1] = float("-inf")
        idx[1, ::2] = -1
        top[2, 1:] = float("-inf")
        z[0, 3] = float("nan")
    from unet_amd.losses import distillation_loss
    for red in ("mean", "none"):
        loss = distillation_loss(z, top, idx, reduction=red)
        (grad,) = torch.autograd.grad(loss, (z,), torch.full_like(loss, 2.0))
        assert torch.isfinite(loss).all() and torch.isfinite(grad).all() and not grad[:2].any()
    assert not loss.detach()[:2].any()
    z2 = z.detach().clone()
    z2[0] = 0.0
    idx[:2] = -1
    top[:2] = 0.0
    rl, rg, lt, gt = _ref(z2, top, idx, 1.0, None, "none", torch.full((5,), 2.0))
    assert ((loss.detach().double().cpu() - rl).abs() <= lt + U * rl.abs()).all()
    assert ((grad.double().cpu() - rg).abs() <= gt + 1.01 * 2 * U * rg.abs() + 1e-38).all()


def test_strided_and_misaligned_logits():
    g = torch.Generator().manual_seed(1)
    for dtype in (torch.float32, torch.bfloat16):
        wide = (torch.randn(6, 2100, generator=g) * 3).to(dtype).cuda()
        _, top, idx = _inputs((6,), 2000, 12)
        for c0 in (0, 1, 3, 8):
            _check(wide[:, c0:c0 + 2000].detach().requires_grad_(True), top, idx)
        col = wide.t()[:2000].contiguous().t().detach().requires_grad_(True)       # rows that are not contiguous
        _check(col, top, idx)
        _check(wide[::2, :2000].detach().requires_grad_(True), top[:3], idx[:3])
        odd = wide.reshape(-1)[5:5 + 6 * 1999].view(6, 1999).detach().requires_grad_(True)
        _check(odd, top, idx % 1999)


def test_same_bits_on_every_run_other_stream_and_graph_replays():
    from unet_amd.losses import distillation_loss
    z, top, idx = _inputs((50,), 3001, 10, torch.bfloat16)
    w = (torch.rand(50, generator=torch.Generator().manual_seed(2)) < 0.7).cuda()

    def step():
        loss = distillation_loss(z, top, idx, temperature=2.0, weights=w)
        return loss.detach(), torch.autograd.grad(loss, (z,))[0]
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        z2, top2, idx2 = _inputs((50,), 3001, 10, torch.bfloat16, seed=seed + 20)
        with torch.no_grad():
            z.copy_(z2), top.copy_(top2), idx.copy_(idx2)
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_gradient_against_differences():
    """Central differences of the loss in 64 bits would be the reference's own; here the kernel's loss is differenced.  Step 1/16 at an fp32
    loss of size ~10: the loss's rounding gives 10 * 2^-22 * 8 ~ 2e-5, the third derivative (<= tau^2 / tau^3 = 1) h^2 / 6 = 6.5e-4."""
    from unet_amd.losses import distillation_loss
    z, top, idx = _inputs((3,), 40, 5)
    (grad,) = torch.autograd.grad(distillation_loss(z, top, idx, reduction="sum"), (z,))
    with torch.no_grad():
        for r, v in ((0, 0), (1, int(idx[1, 0])), (2, 39)):
            hi, lo = z.clone(), z.clone()
            hi[r, v] += 1 / 16
            lo[r, v] -= 1 / 16
            d = (float(distillation_loss(hi, top, idx, reduction="sum")) - float(distillation_loss(lo, top, idx, reduction="sum"))) * 8
            assert abs(d - float(grad[r, v])) <= 8e-4


def test_no_gradient_wanted():
    from unet_amd.losses import distillation_loss
    z, top, idx = _inputs((5,), 600, 7)
    a = distillation_loss(z.detach(), top, idx)
    with torch.no_grad():
        b = distillation_loss(z, top, idx)
    assert not a.requires_grad and not b.requires_grad and torch.equal(a, b)
    assert torch.equal(a, distillation_loss(z, top, idx).detach())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_highest_values(dtype):
    """Rows whose logits lie near the type's largest value: their product with log2 e has no room in 32 bits, their differences do."""
    top_value = torch.finfo(dtype).max
    z, top, idx = _inputs((3,), 600, 8, dtype)
    with torch.no_grad():
        z[0] = top_value
        z[1] = top_value
        z[1, 300:] = top_value / 2
        z[2] = torch.finfo(dtype).min
        z[2, :300] = top_value
    _check(z, top, idx % 300, 1.0)
    _check(z, top, idx % 300, 2.0, None, "none")


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("wanted", [False, True])
def test_more_rows_than_blocks(reduction, wanted):
    """Several rows per block, rows of weight 0 (with NaN logits) among them, so that a row's loads pass over them; with and without
    a gradient."""
    from unet_amd.losses import distillation_loss
    N = 2048 * 2 + 77
    z, top, idx = _inputs((N,), 301, 4, torch.bfloat16)
    w = torch.rand(N, generator=torch.Generator().manual_seed(5)).cuda() + 0.5
    w[::3] = 0.0
    w[2048:2060] = 0.0
    with torch.no_grad():
        z[::3] = float("nan")
    if wanted:
        _check(z, top, idx, 1.5, w, reduction)
        return
    want, _, ltol, _ = _ref(z, top, idx, 1.5, w, reduction)
    got = distillation_loss(z.detach(), top, idx, temperature=1.5, weights=w, reduction=reduction)
    assert bool(((got.double().cpu() - want).abs() <= ltol).all())


@pytest.mark.parametrize("V,K", [(301, 4), (9000, 70), (9000, 300)])
def test_upstream_gradients_of_many_rows(V, K):
    """Several rows per block in the gradient for other upstream factors than 1; pairs that fill more than one round of the threads."""
    N = 8192 + 3 if V < 1000 else 1100
    z, top, idx = _inputs((N,), V, K)
    with torch.no_grad():
        top[1], idx[2] = float("-inf"), -1
    w = torch.rand(N, generator=torch.Generator().manual_seed(6)).cuda()
    w[5::7] = 0.0
    g = torch.randn(N, generator=torch.Generator().manual_seed(7)).cuda()
    _check_rows(z, top, idx, w, g)


def _check_rows(z, top, idx, w, g):
    """As _check with reduction "none", in 64 bits on the GPU."""
    from unet_amd.losses import distillation_loss
    loss = distillation_loss(z, top, idx, weights=w, reduction="none")
    (grad,) = torch.autograd.grad(loss, (z,), g)
    zd, td = z.detach().double(), top.double()
    ok = (idx >= 0) & (idx < z.shape[1]) & ~torch.isneginf(td)
    p = torch.softmax(td.masked_fill(~ok, float("-inf")), 1).masked_fill(~ok.any(1, keepdim=True), 0.0)
    q = torch.softmax(zd, 1)
    sp = torch.zeros_like(zd).scatter_add_(1, idx.clamp_min(0).long(), p)
    c = (g * w).double().unsqueeze(1) * ok.any(1, keepdim=True)
    d = (torch.log(p) - torch.log(q).gather(1, idx.clamp_min(0).long())).masked_fill(~ok, 0.0)
    want = (w.double() * (p * d).sum(1)) * ok.any(1)
    A = 60.0                                              # logits within +-3 * 6 of one another and the teacher's within +-2 * 6
    E = (6 * A + z.shape[1] / 64 + 64) * U
    assert bool(((grad.double() - c * (q - sp)).abs() <= c.abs() * E * (q + sp) + 1.01 * 2 * U * (c * (q - sp)).abs() + 1e-38).all())
    assert bool(((loss.detach().double() - want).abs() <= w.double() * (2 * E + E * d.abs().amax(1) + 8 * U * (A + math.log(z.shape[1]))) + U * want.abs()).all())


@pytest.mark.parametrize("tau", [1e-4, 1e-20])
def test_temperatures_near_zero(tau):
    """Both distributions are one-hot: the loss is tau * (z_max - z at the teacher's best), the gradient tau * (one-hot - one-hot) / rows.  Each is a
    difference, a product by 1 / tau and two by tau: at most 8 u of itself."""
    z, top, idx = _inputs((4,), 300, 5)
    with torch.no_grad():
        z.mul_(16).round_()                                # gaps of whole numbers, not ties
        z[:, 7] = 200.0
        top.copy_(torch.arange(5.0).expand(4, 5))
    from unet_amd.losses import distillation_loss
    loss = distillation_loss(z, top, idx, temperature=tau)
    (grad,) = torch.autograd.grad(loss, (z,))
    zd, best = z.detach().double().cpu(), idx[:, 4].cpu()
    t = float(torch.tensor(tau, dtype=torch.float32))
    want = (t * (200.0 - zd.gather(1, best[:, None])[:, 0])).mean()
    wg = torch.zeros(4, 300, dtype=torch.float64)
    wg[:, 7] += t / 4
    wg.scatter_add_(1, best[:, None], torch.full((4, 1), -t / 4, dtype=torch.float64))
    assert abs(float(loss.detach()) - float(want)) <= 8 * U * float(want)
    assert bool(((grad.cpu().double() - wg).abs() <= 8 * U * wg.abs()).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,K", [(700, 65), (3000, 100), (6000, 128), (40, 129), (1500, 200), (2500, 256), (5000, 256), (12000, 200), (20000, 64), (30000, 257)])
def test_pairs_per_thread(V, K, dtype):
    """Every size of block that the pairs can ask for, with rows that fill one to sixteen vectors a thread."""
    for red, g in (("mean", None), ("none", torch.tensor([0.5, 1.0, -3.0]).cuda())):
        z, top, idx = _inputs((3,), V, K, dtype, torch.bfloat16, torch.int32, seed=K)
        idx[1, ::3] = -1
        _check(z, top, idx, 1.25, None, red, g)


@pytest.mark.parametrize("V", [100, 900, 1800, 3700, 7000, 15000, 30000, 60000, 120000])
def test_loss_without_a_gradient(V):
    """The loss alone is what it is beside a gradient, for rows of every size class and more rows than blocks hold at once."""
    from unet_amd.losses import distillation_loss
    N = 600 if V > 5000 else 9000
    z, top, idx = _inputs((N,), V, 8, torch.bfloat16, seed=V) if V <= 5000 else (torch.randn(N, V, device="cuda").to(torch.bfloat16).requires_grad_(True),
                                                                                 torch.randn(N, 8, device="cuda"), torch.randint(0, V, (N, 8), device="cuda"))
    alone = distillation_loss(z.detach(), top, idx, reduction="none")
    q = torch.log_softmax(z.detach().double(), 1)
    p = torch.softmax(top.double(), 1)
    d = torch.log(p) - q.gather(1, idx)
    E = (6 * 60.0 + V / 64 + 64) * U
    tol = 2 * E + E * d.abs().amax(1) + 8 * U * (60.0 + math.log(V))
    want = (p * d).sum(1)
    assert bool(((alone.double() - want).abs() <= tol + U * want.abs()).all())
    total = distillation_loss(z, top, idx, reduction="sum")
    assert abs(float(total.detach()) - float(want.sum())) <= float(tol.sum() + N * U * want.abs().sum())


@pytest.mark.parametrize("N", [1, 3, 4097, 20001, 300007])
@pytest.mark.parametrize("shift", [0, 1])
def test_sums_over_many_rows(N, shift):
    """The mean's two sums, from 16-byte boundaries and off them: the same as of the rows' losses and of the weights."""
    from unet_amd.losses import distillation_loss
    z, top, idx = _inputs((N,), 9, 2, seed=N)
    w = torch.rand(N + shift, generator=torch.Generator().manual_seed(N)).cuda()[shift:]
    rows = distillation_loss(z.detach(), top, idx, weights=w, reduction="none").double()
    for red, want in (("mean", rows.sum() / w.double().sum()), ("sum", rows.sum())):
        got = distillation_loss(z.detach(), top, idx, weights=w, reduction=red)
        # a thread adds n / 4096 terms, ten joins and a division behind them, in either sum; all terms are positive
        assert abs(float(got) - float(want)) <= 2 * (N / 4096 + 16) * U * float(want)
        assert torch.equal(got, distillation_loss(z.detach(), top, idx, weights=w, reduction=red))


FILLS = [-1e4, -1e9, -1e10, -1e12, -1e20, -1e29, -1e30, -3e38]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,K", [(257, 6), (500, 9), (2001, 70), (500, 300), (9001, 300)])
@pytest.mark.parametrize("fill", FILLS)
def test_masked_vocabulary_of_any_fill(fill, V, K, dtype):
    """Logits masked by a large negative number, at the head, at the tail, scattered, and all but one, so that threads meet only such
    numbers, first, last or throughout; rows of a length that leaves loose elements; rows in registers and rows read twice (K = 300).  A
    thread's maximum is then the fill, and the product with log2 e / tau has a rounding error of many powers of 2."""
    for tau in (0.5, 1.0, 2.0, 1e-5):
        z, top, idx = _inputs((5,), V, K, dtype)
        live = torch.zeros(5, V, dtype=torch.bool)
        live[0, V // 2:] = True
        live[1, :V // 3] = True
        live[2, torch.randperm(V, generator=torch.Generator().manual_seed(V))[:V // 10]] = True
        live[3, V - 1] = True
        live[4] = True
        with torch.no_grad():
            z[~live.cuda()] = fill
            for r in range(5):
                at = live[r].nonzero().view(-1).cuda()
                idx[r] = at[idx[r] % at.numel()]
        _check(z, top, idx, tau)
        _check(z, top, idx, tau, None, "none", torch.tensor([0.5, -1.0, 1.0, 2.0, 3.0]).cuda())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [6, 300])
def test_rows_of_one_far_value_and_teachers_on_masked_entries(K, dtype):
    """Whole rows at a far value, whose softmax is flat, and a teacher whose mass lies on masked entries: a large loss, no NaN."""
    for V in (257, 4003):
        z, top, idx = _inputs((8,), V, K, dtype)
        with torch.no_grad():
            for r, v in enumerate((1e7, -1e7, 1e10, -1e10, 1e20, -1e20)):
                z[r] = v
            z[6, 1:] = -1e10
            z[7, :V // 2] = -1e20
            idx[6], idx[7] = 1 + idx[6] % (V - 1), idx[7] % (V // 2)
        for tau in (0.5, 1.0, 1.5):
            _check(z, top, idx, tau, None, "none")
            _check(z, top, idx, tau)
    z, top, idx = _inputs((3,), 700, K, dtype)
    with torch.no_grad():
        z.mul_(1000.0)                                    # logits in the thousands at a temperature near zero
    _check(z, top, idx, 1e-6)


def test_saved_tensor_hooks_see_the_gradient_buffer():
    """The N x V gradient that the forward pass leaves is saved where hooks see it (offloading), a recomputed forward pass (checkpoint) works, and
    a gradient that was changed in place does not keep a second backward pass from its own."""
    from torch.utils.checkpoint import checkpoint
    from unet_amd.losses import distillation_loss
    for dtype in (torch.float32, torch.bfloat16):
        z, top, idx = _inputs((6,), 777, 9, dtype)
        (want,) = torch.autograd.grad(distillation_loss(z, top, idx), (z,))
        big = []

        def pack(t):
            big.append(t.shape == z.shape and t.data_ptr() != z.data_ptr())
            return t.cpu()
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.cuda()):
            loss = distillation_loss(z, top, idx)
        assert sum(big) == 1
        (a,) = torch.autograd.grad(loss, (z,), retain_graph=True)
        assert torch.equal(a, want)
        (b,) = torch.autograd.grad(loss, (z,), torch.tensor(2.0, device="cuda"))
        assert bool(((b.float() - 2 * want.float()).abs() <= 2.02 * HALF[dtype] * 2 * want.float().abs() + 1e-9).all())
        loss = checkpoint(lambda t: distillation_loss(t, top, idx), z, use_reentrant=False)
        assert torch.equal(torch.autograd.grad(loss, (z,))[0], want)
        loss = distillation_loss(z, top, idx)
        (a,) = torch.autograd.grad(loss, (z,), retain_graph=True)
        assert torch.equal(a, want)
        a.zero_()
        (b,) = torch.autograd.grad(loss, (z,))
        assert not a.any() and bool(((b.float() - want.float()).abs() <= 2.02 * HALF[dtype] * want.float().abs() + 1e-9).all())


def test_a_captured_backward_pass_takes_every_factor():
    """The gradient pass alone in a graph, of a loss that was computed before on the stream of the capture (an autograd node runs on its
    forward pass's stream): replays with other upstream gradients, and after the gradient of the replay before was changed in place."""
    from unet_amd.losses import distillation_loss
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        z, top, idx = _inputs((20,), 901, 7)
        g = torch.ones((), device="cuda")
        want = torch.autograd.grad(distillation_loss(z, top, idx), (z,))[0].clone()
        loss = distillation_loss(z, top, idx)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            (grad,) = torch.autograd.grad(loss, (z,), g, retain_graph=True)
        for f in (1.0, 2.0, 1.0, 0.0, 1.0):
            g.fill_(f)
            graph.replay()
            torch.cuda.synchronize()
            # both round gs * exp2(.) and, at the teacher's indices, gs * exp2(.) - gc * p: a factor of 1, 2 or 0 scales every term exactly
            assert bool(((grad - f * want).abs() <= 8 * U * (f * want).abs() + 1e-9).all()), f
            grad.zero_()


def test_forward_and_backward_captured_in_graphs_of_their_own():
    from unet_amd import _lib as L
    from unet_amd.losses import distillation_loss
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        z, top, idx = _inputs((20,), 901, 7)
        g = torch.ones((), device="cuda")
        torch.autograd.grad(distillation_loss(z, top, idx), (z,), g)      # (first launches outside of a capture)
        one, two, both = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        ids = [L.capture_id(z.device)]
        with torch.cuda.graph(one, stream=side):
            ids.append(L.capture_id(z.device))
            loss = distillation_loss(z, top, idx)
        with torch.cuda.graph(two, stream=side):
            ids.append(L.capture_id(z.device))
            (grad,) = torch.autograd.grad(loss, (z,), g)
        with torch.cuda.graph(both, stream=side):
            ids.append(L.capture_id(z.device))
            (grad2,) = torch.autograd.grad(distillation_loss(z, top, idx), (z,), g)
            assert L.capture_id(z.device) == ids[3]
        assert ids[0] == 0 == L.capture_id(z.device) and len(set(ids)) == 4 and min(ids) == 0
        for seed in range(3):
            with torch.no_grad():
                z.copy_(_inputs((20,), 901, 7, seed=seed + 3)[0])
            for f in (1.0, 3.0, 1.0):
                g.fill_(f)
                want = torch.autograd.grad(distillation_loss(z, top, idx), (z,), g)[0]
                if f == 1.0:
                    one.replay()
                two.replay()
                both.replay()
                torch.cuda.synchronize()
                assert bool(((grad - want).abs() <= 8 * U * want.abs() + 1e-9).all()) and torch.equal(grad2, want), (seed, f)
                grad.zero_()


@pytest.mark.parametrize("V,K", [(300, 4), (300, 300), (9000, 4)])
@pytest.mark.parametrize("N", [5, 5000])
def test_a_nan_weight_reaches_the_mean(N, V, K):
    """A NaN among the weights: their sum is NaN and with it the mean and every gradient of a live row, as in 64 bits; rows of weight 0 keep
    theirs, and "sum" and "none" keep it in its row."""
    from unet_amd.losses import distillation_loss
    if N * V > 10_000_000:
        N = 1000
    z, top, idx = _inputs((N,), V, K)
    w = torch.ones(N, device="cuda")
    w[1], w[3] = float("nan"), 0.0
    live = torch.ones(N, dtype=torch.bool, device="cuda")
    live[3] = False
    loss = distillation_loss(z, top, idx, weights=w)
    (grad,) = torch.autograd.grad(loss, (z,))
    assert torch.isnan(loss) and torch.isnan(grad[live]).all() and not grad[3].any()
    (grad,) = torch.autograd.grad(distillation_loss(z, top, idx, weights=w), (z,), torch.tensor(0.5, device="cuda"))
    assert torch.isnan(grad[live]).all() and not grad[3].any()
    live[1] = False
    for red in ("sum", "none"):
        loss = distillation_loss(z, top, idx, weights=w, reduction=red)
        (grad,) = torch.autograd.grad(loss, (z,), torch.ones_like(loss))
        assert torch.isnan(grad[1]).all() and torch.isfinite(grad[live]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,K", [(700, 513), (3000, 768), (3000, 2500), (40, 1500), (9001, 1025)])
def test_very_many_pairs(V, K, dtype):
    """More pairs than a block has threads, most of them naming an index that others name too."""
    for red, g in (("mean", None), ("none", torch.tensor([0.5, 1.0, -3.0, 2.0]).cuda())):
        z, top, idx = _inputs((4,), V, K, dtype, torch.float32, torch.int32, seed=K)
        idx[1, ::3] = -1
        idx[2] = idx[2] % 7
        _check(z, top, idx, 1.25, None, red, g)
    z, top, idx = _inputs((4100,), 33, 600, dtype, seed=3)
    _check_rows_bf16_or_fp32(z, top, idx)


def _check_rows_bf16_or_fp32(z, top, idx):
    """Rows enough for a wave each: against the same loss of a few of them."""
    from unet_amd.losses import distillation_loss
    loss = distillation_loss(z, top, idx, reduction="none")
    (grad,) = torch.autograd.grad(loss, (z,), torch.ones_like(loss))
    for a in (0, 2000, 4096):
        zs = z.detach()[a:a + 4].clone().requires_grad_(True)
        rl, rg, lt, gt = _ref(zs, top[a:a + 4], idx[a:a + 4], 1.0, None, "none", torch.ones(4))
        assert bool(((loss.detach()[a:a + 4].double().cpu() - rl).abs() <= lt + U * rl.abs()).all())
        assert bool(((grad[a:a + 4].double().cpu() - rg).abs() <= gt + 1.01 * (HALF[z.dtype] + U) * rg.abs() + 1e-38).all())
