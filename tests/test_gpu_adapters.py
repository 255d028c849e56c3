"""GPU: adapter_linear and its gradients against a plain implementation in 64 bits.

Tolerances, u = 2^-24 (fp32 sums: at most u of a partial sum per addition, so n additions are off by n u of the sum of absolute values),
s = 2^-17 (what a factor split into two bf16 parts loses; 0 in fp32), h = half a step of the output type.  With |h| = |s_a| |A||x| the
sums of absolute values: h is off by (K + 3) u |h|; y by (K + r + 3) u (|W||x| + |b|) + ((2 K + 2 r + 8) u + s) |B||h|; the
gradients alike with N for K, and those of A and B by (n + K + N + 8) u + s of their sum over n rows.  Then h |ref|."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
SPLIT = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -17}


def _inputs(T, K, N, r, G, dtype, kind="random", bias=True, scales=True, seed=0, idt=torch.int64):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, K, generator=g).to(dtype)
    w = (torch.randn(N, K, generator=g) / K ** 0.5).to(dtype)
    b = torch.randn(N, generator=g).to(dtype) if bias else None
    A = (torch.randn(G, r, K, generator=g) / K ** 0.5).to(dtype)
    B = (torch.randn(G, N, r, generator=g) / r ** 0.5).to(dtype)
    sc = 0.25 + torch.rand(G, generator=g) if scales else None
    if kind == "none":
        ids = torch.full((T,), -1)
    elif kind == "one":
        ids = torch.full((T,), G - 1)
    elif kind == "segments":
        ids = (torch.arange(T) * (G + 1) // max(T, 1))             # the last segment has no adapter
    else:
        ids = torch.randint(-1, G + 1, (T,), generator=g)          # -1 and G: none
    dy = torch.randn(T, N, generator=g).to(dtype)
    c = lambda t: None if t is None else t.cuda()
    return dict(x=c(x).requires_grad_(True), w=c(w), b=c(b), A=c(A).requires_grad_(True), B=c(B).requires_grad_(True), ids=c(ids.to(idt)), sc=c(sc), dy=c(dy))


def _ref(i):
    d = lambda t: t.detach().double().cpu()
    x, w, A, B, dy, ids = d(i["x"]), d(i["w"]), d(i["A"]), d(i["B"]), d(i["dy"]), i["ids"].long().cpu()
    dt = i["x"].dtype
    T, K = x.shape
    N, (G, r) = w.shape[0], A.shape[:2]
    sc = torch.ones(G, dtype=torch.float64) if i["sc"] is None else d(i["sc"])
    b = torch.zeros(N, dtype=torch.float64) if i["b"] is None else d(i["b"])
    y, dx = x @ w.t() + b, dy @ w
    ty, tx = (K + r + 3) * U * (x.abs() @ w.abs().t() + b.abs()), (N + r + 3) * U * (dy.abs() @ w.abs())
    dA, dB, tA, tB = (torch.zeros_like(t) for t in (A, B, A, B))
    s, h = SPLIT[dt], HALF[dt]
    for a in range(G):
        t = (ids == a).nonzero().view(-1)
        xa, da = x[t], dy[t]
        hh, ha = sc[a] * xa @ A[a].t(), sc[a].abs() * xa.abs() @ A[a].abs().t()
        dh, dha = sc[a] * da @ B[a], sc[a].abs() * da.abs() @ B[a].abs()
        y[t] += hh @ B[a].t()
        dx[t] += dh @ A[a]
        dA[a], dB[a] = dh.t() @ xa, da.t() @ hh
        ty[t] += ((2 * K + 2 * r + 8) * U + s) * (ha @ B[a].abs().t())
        tx[t] += ((2 * N + 2 * r + 8) * U + s) * (dha @ A[a].abs())
        e = (t.numel() + K + N + 8) * U + s
        tA[a], tB[a] = e * (dha.t() @ xa.abs()), e * (da.abs().t() @ ha)
    return [(v, t + 1.01 * h * v.abs()) for v, t in ((y, ty), (dx, tx), (dA, tA), (dB, tB))]


def _call(i):
    from unet_amd.adapters import adapter_linear
    y = adapter_linear(i["x"], i["w"], i["b"], i["A"], i["B"], i["ids"], scales=i["sc"])
    return (y.detach(), *torch.autograd.grad(y, (i["x"], i["A"], i["B"]), i["dy"]))


def _check(i):
    got = _call(i)
    for name, v, (ref, tol) in zip(("y", "dx", "dA", "dB"), got, _ref(i)):
        assert v.dtype == i["x"].dtype and v.shape == ref.shape, name
        err = (v.double().cpu() - ref).abs()
        assert (err <= tol).all(), (name, float((err - tol).max()), float(err.max()))
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K,N,r,G", [(1, 1, 1, 1, 1), (1, 64, 48, 4, 3), (2, 17, 5, 3, 2), (15, 256, 64, 8, 4), (16, 256, 256, 16, 16), (17, 100, 65, 17, 5),
                                       (64, 512, 520, 16, 64), (65, 72, 130, 33, 7), (128, 128, 256, 64, 2), (200, 333, 97, 128, 3), (300, 64, 1000, 5, 300),
                                       (129, 1032, 40, 100, 1)])
def test_forward_and_gradients(T, K, N, r, G, dtype):
    for n, kind in enumerate(("random", "segments", "one")):
        _check(_inputs(T, K, N, r, G, dtype, kind, bias=n != 1, scales=n != 2, seed=n, idt=torch.int32 if n == 1 else torch.int64))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K,N,r,G,kind", [(512, 512, 512, 16, 4, "segments"), (700, 520, 584, 8, 3, "random"), (1030, 517, 611, 5, 7, "random"),
                                            (2050, 256, 768, 32, 2, "segments"), (640, 1024, 512, 24, 9, "random")])
def test_larger_tiles(T, K, N, r, G, kind, dtype):
    _check(_inputs(T, K, N, r, G, dtype, kind))


@pytest.mark.parametrize("T,K,N,r,G,kind", [(4100, 72, 4096, 20, 3, "random"), (4100, 4096, 72, 20, 3, "segments"), (4100, 264, 2048, 8, 40, "random"),
                                            (4100, 2048, 264, 8, 40, "segments"), (4100, 328, 4096, 128, 2, "segments")])
def test_largest_tiles(T, K, N, r, G, kind):
    _check(_inputs(T, K, N, r, G, torch.bfloat16, kind))


@pytest.mark.parametrize("T,K,N,r,G,kind", [(4100, 36, 4096, 20, 3, "random"), (4100, 2048, 132, 5, 40, "segments")])
def test_largest_tiles_fp32(T, K, N, r, G, kind):
    _check(_inputs(T, K, N, r, G, torch.float32, kind))


def test_operands_beyond_two_gib():
    """x of 2.2 GB (offsets that pass 32 bits): the rows of its end against a call on them alone."""
    from unet_amd.adapters import adapter_linear
    T, K, N, r, G = 1 << 20, 1048, 24, 4, 3
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(T, K, generator=g, device="cuda", dtype=torch.bfloat16)
    i = _inputs(8, K, N, r, G, torch.bfloat16)
    ids = torch.randint(-1, G, (T,), generator=g, device="cuda")
    with torch.no_grad():
        y = adapter_linear(x, i["w"], i["b"], i["A"], i["B"], ids)
        assert y.shape == (T, N)
        for a in (0, 500000, T - 200):
            i["x"], i["ids"], i["sc"] = x[a:a + 200], ids[a:a + 200], None
            ref, tol = _ref({**i, "dy": torch.zeros(200, N)})[0]
            assert ((y[a:a + 200].double().cpu() - ref).abs() <= tol).all()


def test_rows_without_an_adapter():
    for dtype in (torch.float32, torch.bfloat16):
        y, dx, dA, dB = _check(_inputs(70, 40, 33, 6, 4, dtype, "none"))
        assert not dA.any() and not dB.any()


def test_adapters_without_a_row_get_zeros():
    i = _inputs(40, 64, 64, 8, 12, torch.float32)
    i["ids"] = i["ids"].clamp(-1, 2)
    _, _, dA, dB = _check(i)
    assert not dA[3:].any() and not dB[3:].any()


def test_nan_stays_in_its_row_and_adapter():
    """A NaN adapter touches its own rows alone (and, through them, its own gradients); a NaN row its own row and adapter."""
    for dtype in (torch.float32, torch.bfloat16):
        i = _inputs(90, 96, 80, 8, 5, dtype)
        with torch.no_grad():
            i["A"][3] = float("nan")
            i["B"][3] = float("nan")
        y, dx, dA, dB = _call(i)
        other = i["ids"] != 3
        assert torch.isfinite(y[other]).all() and torch.isfinite(dx[other]).all() and torch.isnan(y[~other]).all()
        keep = [0, 1, 2, 4]
        assert torch.isfinite(dA[keep]).all() and torch.isfinite(dB[keep]).all()
        i = _inputs(90, 96, 80, 8, 5, dtype)
        with torch.no_grad():
            i["ids"][7] = -1
            i["x"][7] = float("nan")
            i["dy"][7] = float("inf")
        y, dx, dA, dB = _call(i)
        rest = torch.arange(90) != 7
        assert torch.isfinite(y[rest]).all() and torch.isfinite(dx[rest]).all() and torch.isfinite(dA).all() and torch.isfinite(dB).all()


def test_empty_batch():
    from unet_amd.adapters import adapter_linear
    i = _inputs(4, 24, 16, 3, 2, torch.bfloat16)
    x = i["x"].detach()[:0].requires_grad_(True)
    y = adapter_linear(x, i["w"], i["b"], i["A"], i["B"], i["ids"][:0])
    dx, dA, dB = torch.autograd.grad(y, (x, i["A"], i["B"]), i["dy"][:0])
    assert y.shape == (0, 16) and dx.shape == (0, 24) and not dA.any() and not dB.any()


def test_strided_and_misaligned_operands():
    g = torch.Generator().manual_seed(4)
    for dtype in (torch.float32, torch.bfloat16):
        for T, K, N, off in ((33, 64, 80, 0), (33, 64, 80, 3), (600, 512, 512, 8), (600, 512, 512, 1)):
            i = _inputs(T, K, N, 8, 3, dtype)
            wide = torch.randn(T, K + 16, generator=g).to(dtype).cuda()
            i["x"] = wide[:, off:off + K].detach().requires_grad_(True)
            ww = (torch.randn(N, K + 24, generator=g) / K ** 0.5).to(dtype).cuda()
            i["w"] = ww[:, off:off + K]
            i["dy"] = torch.randn(T, N + 7, generator=g).to(dtype).cuda()[:, 2:2 + N]
            i["A"] = i["A"].detach().transpose(1, 2).contiguous().transpose(1, 2).requires_grad_(True)
            _check(i)


def test_shapes_of_requests():
    """(requests, tokens, K) with one id per request, and with one per token; broadcast upstream gradients."""
    from unet_amd.adapters import adapter_linear
    i = _inputs(4 * 9, 40, 24, 4, 3, torch.float32)
    x3 = i["x"].detach().view(4, 9, 40)
    ids = torch.tensor([2, -1, 0, 2], device="cuda")
    y3 = adapter_linear(x3, i["w"], i["b"], i["A"], i["B"], ids, scales=i["sc"])
    i["ids"] = ids.repeat_interleave(9)
    assert y3.shape == (4, 9, 24)
    assert torch.equal(y3.view(36, 24), _check(i)[0])
    assert torch.equal(y3, adapter_linear(x3, i["w"], i["b"], i["A"], i["B"], i["ids"].view(4, 9), scales=i["sc"]))
    i["dy"] = torch.ones(1, 1, device="cuda").expand(36, 24)
    _check(i)
    y1 = adapter_linear(x3[0, 0], i["w"], i["b"], i["A"], i["B"], ids[0], scales=i["sc"])
    assert y1.shape == (24,)


def test_gradients_not_wanted():
    from unet_amd.adapters import adapter_linear
    i = _inputs(50, 64, 48, 8, 3, torch.bfloat16)
    want = _call(i)
    for k, (nx, na, nb) in enumerate(((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1))):
        x, A, B = (t.detach().requires_grad_(bool(f)) for t, f in ((i["x"], nx), (i["A"], na), (i["B"], nb)))
        y = adapter_linear(x, i["w"], i["b"], A, B, i["ids"], scales=i["sc"])
        ts = [t for t in (x, A, B) if t.requires_grad]
        for got, ref in zip(torch.autograd.grad(y, ts, i["dy"]), [w for w, f in zip(want[1:], (nx, na, nb)) if f]):
            assert torch.equal(got, ref)
    with torch.no_grad():                       # another path: one launch less order, the same result up to the roundings of the sums
        y = adapter_linear(i["x"], i["w"], i["b"], i["A"], i["B"], i["ids"], scales=i["sc"])
    ref, tol = _ref(i)[0]
    assert ((y.double().cpu() - ref).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K,N,r,G", [(1, 1, 1, 1, 1), (1, 2048, 2048, 8, 4), (1, 40, 17, 128, 2), (2, 96, 256, 16, 1), (15, 517, 100, 5, 3), (16, 256, 300, 24, 16),
                                       (17, 1000, 33, 33, 9), (32, 512, 512, 16, 40), (33, 64, 2000, 128, 33), (48, 129, 130, 3, 7), (63, 4096, 272, 16, 64),
                                       (64, 1032, 1001, 64, 64), (64, 512, 512, 8, 300), (65, 96, 80, 8, 3), (200, 100, 64, 7, 5)])
def test_forward_alone(T, K, N, r, G, dtype):
    """Without a gradient: single tokens of up to 64 requests in two launches, more rows as before."""
    from unet_amd.adapters import adapter_linear
    for n, kind in enumerate(("random", "one", "none")):
        i = _inputs(T, K, N, r, G, dtype, kind, bias=n != 1, scales=n != 2, seed=n, idt=torch.int32 if n == 1 else torch.int64)
        with torch.no_grad():
            y = adapter_linear(i["x"], i["w"], i["b"], i["A"], i["B"], i["ids"], scales=i["sc"])
            again = adapter_linear(i["x"], i["w"], i["b"], i["A"], i["B"], i["ids"], scales=i["sc"])
        ref, tol = _ref(i)[0]
        assert y.dtype == dtype and ((y.double().cpu() - ref).abs() <= tol).all() and torch.equal(y, again)


def test_forward_alone_keeps_nan_in_its_rows():
    from unet_amd.adapters import adapter_linear
    for dtype in (torch.float32, torch.bfloat16):
        i = _inputs(40, 96, 80, 8, 5, dtype)
        with torch.no_grad():
            i["A"][3] = float("nan")
            i["B"][3] = float("inf")
            i["x"][7] = float("nan")
            y = adapter_linear(i["x"], i["w"], i["b"], i["A"], i["B"], i["ids"], scales=i["sc"])
        clean = (i["ids"] != 3) & (torch.arange(40, device="cuda") != 7)
        assert torch.isfinite(y[clean]).all() and torch.isnan(y[~clean]).all()


def test_forward_alone_in_a_graph():
    from unet_amd.adapters import adapter_linear
    i = _inputs(20, 256, 320, 16, 6, torch.bfloat16)
    f = lambda: adapter_linear(i["x"], i["w"], i["b"], i["A"], i["B"], i["ids"], scales=i["sc"])
    with torch.no_grad():
        f()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f()
        for seed in range(3):
            j = _inputs(20, 256, 320, 16, 6, torch.bfloat16, seed=seed + 50)
            for k in ("x", "A", "B", "ids"):
                i[k].copy_(j[k])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, f())


@pytest.mark.parametrize("T,K,N", [(40, 96, 64), (520, 512, 512)])
def test_same_bits_on_every_run_other_stream_and_graph_replays(T, K, N):
    i = _inputs(T, K, N, 8, 4, torch.bfloat16)
    want = _call(i)
    for a, b in zip(_call(i), want):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _call(i)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _call(i)
    for seed in range(3):
        j = _inputs(T, K, N, 8, 4, torch.bfloat16, seed=seed + 30)
        with torch.no_grad():
            for k in ("x", "A", "B", "ids", "dy"):
                i[k].copy_(j[k])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, _call(i)):
            assert torch.equal(a, b)


def test_refusals():
    from unet_amd.adapters import adapter_linear
    i = _inputs(6, 16, 8, 4, 3, torch.float32)
    a = dict(x=i["x"], weight=i["w"], bias=i["b"], A=i["A"], B=i["B"], ids=i["ids"], scales=i["sc"])

    def bad(**kw):
        with pytest.raises(ValueError):
            adapter_linear(**{**a, **kw})
    bad(x=i["x"].detach().half(), weight=i["w"].half(), bias=None, A=i["A"].detach().half(), B=i["B"].detach().half())
    bad(x=i["x"].detach().bfloat16())
    bad(x=i["x"][:, :15]), bad(A=i["A"][:, :3]), bad(B=i["B"][:2]), bad(bias=i["b"][:7]), bad(scales=i["sc"][:2])
    bad(ids=i["ids"][:5]), bad(ids=i["ids"].float()), bad(ids=i["ids"][0]), bad(ids=i["ids"].cpu().short().cuda())
    bad(weight=i["w"].clone().requires_grad_(True)), bad(bias=i["b"].clone().requires_grad_(True)), bad(scales=i["sc"].clone().requires_grad_(True))
    bad(A=torch.zeros(3, 129, 16, device="cuda"), B=torch.zeros(3, 8, 129, device="cuda"))
    bad(A=torch.zeros(0, 4, 16, device="cuda"), B=torch.zeros(0, 8, 4, device="cuda"))
    with pytest.raises(RuntimeError):
        adapter_linear(**{**a, "ids": i["ids"].cpu()})


def test_gradients_against_differences():
    """The projection is linear in x, A and B each, so a central difference is exact but for fp32 roundings: y is off by about
    (K + r) 2^-24 * 5 ~ 1e-5 per value, 24 x 20 of them against |dy| ~ 1, divided by the step of 2: under 3e-3 even if all had one sign."""
    from unet_amd.adapters import adapter_linear
    i = _inputs(24, 32, 20, 4, 3, torch.float32)
    _, dx, dA, dB = _call(i)
    f = lambda **kw: (adapter_linear(kw.get("x", i["x"]), i["w"], i["b"], kw.get("A", i["A"]), kw.get("B", i["B"]), i["ids"], scales=i["sc"]).double() * i["dy"].double()).sum()
    with torch.no_grad():
        for name, grad, at in (("x", dx, (3, 5)), ("x", dx, (23, 31)), ("A", dA, (1, 2, 7)), ("B", dB, (2, 19, 3))):
            hi, lo = i[name].clone(), i[name].clone()
            hi[at] += 1.0
            lo[at] -= 1.0
            assert abs(float(f(**{name: hi}) - f(**{name: lo})) / 2 - float(grad[at])) <= 3e-3


def test_module_starts_as_the_shared_projection_and_trains_its_adapters_alone():
    from unet_amd import AdapterLinear
    torch.manual_seed(1)
    lin = torch.nn.Linear(48, 40).cuda()
    m = AdapterLinear(lin, 3, 4, alpha=8)
    x, ids = torch.randn(30, 48, device="cuda"), torch.randint(0, 3, (30,), device="cuda")
    ref = x.double() @ lin.weight.detach().double().t() + lin.bias.detach().double()
    y = m(x, ids)
    assert (y.detach().double() - ref).abs().max() <= 52 * U * (x.abs().double() @ lin.weight.detach().abs().double().t() + 1).max()
    y.square().sum().backward()
    assert m.B.grad.abs().max() > 0 and not m.A.grad.any() and lin.weight.grad is None and lin.bias.grad is None


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K,N,r,G,kind", [(84, 2880, 128, 8, 1, "segments"), (399, 64, 2112, 24, 36, "random"), (250, 4000, 100, 33, 20, "random"),
                                            (1022, 1300, 136, 5, 2, "random"), (70, 19, 20, 19, 118, "random"), (1500, 200, 1950, 40, 90, "random"),
                                            (530, 2050, 330, 128, 33, "segments")])
def test_reductions_in_parts_and_seldom_shared_adapters(T, K, N, r, G, kind, dtype):
    """Few tiles with a long reduction in either direction, fragments of many adapters, rows that come one by one."""
    _check(_inputs(T, K, N, r, G, dtype, kind))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K,N,G", [(96, 80, 12), (3200, 64, 2), (64, 3200, 30)])
def test_nan_stays_in_its_row_and_adapter_in_parts_too(K, N, G, dtype):
    from unet_amd.adapters import adapter_linear
    i = _inputs(100, K, N, 8, G, dtype)
    ids = i["ids"].cpu()
    with torch.no_grad():
        i["A"][1] = float("nan")
        i["B"][1, :, 3] = float("inf")
        row = int((ids != 1).nonzero()[5])
        i["x"][row] = float("nan")
    y, dx, dA, dB = _call(i)
    bad = (ids == 1)
    bad[row] = True
    assert torch.isnan(y.cpu()[bad]).all() and torch.isfinite(y.cpu()[~bad]).all()
    bad[row] = False                                       # dx of the NaN row does not depend on it
    assert torch.isfinite(dx.cpu()[~bad]).all()
    sound = torch.ones(G, dtype=torch.bool)
    sound[1] = False
    if ids[row] >= 0 and ids[row] < G:
        sound[ids[row]] = False
    assert torch.isfinite(dA.cpu()[sound]).all() and torch.isfinite(dB.cpu()[sound]).all()


@pytest.mark.parametrize("K,N,G", [(2816, 128, 1), (256, 256, 16)])
def test_parts_have_the_same_bits_in_a_replayed_graph(K, N, G):
    from unet_amd.adapters import adapter_linear
    i = _inputs(200, K, N, 8, G, torch.float32)
    a = {k: (v.detach() if torch.is_tensor(v) else v) for k, v in i.items()}
    with torch.no_grad():
        want = adapter_linear(a["x"], a["w"], a["b"], a["A"], a["B"], a["ids"], scales=a["sc"])
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            adapter_linear(a["x"], a["w"], a["b"], a["A"], a["B"], a["ids"], scales=a["sc"])
        torch.cuda.current_stream().wait_stream(side)
        with torch.cuda.graph(graph):
            y = adapter_linear(a["x"], a["w"], a["b"], a["A"], a["B"], a["ids"], scales=a["sc"])
        for _ in range(3):
            y.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want)
            torch.randn(1 << 20, device="cuda").sum()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K,N,r,used", [(5, 96, 80, 4, 2), (64, 260, 128, 8, 5), (300, 517, 65, 8, 1), (2100, 520, 264, 8, 5), (700, 64, 1100, 20, 40)])
def test_many_registered_adapters_few_of_them_in_the_batch(T, K, N, r, used, dtype):
    """1500 adapters, rows of a few of them together or mixed: the same results whatever is registered besides; zeros for the others."""
    from unet_amd.adapters import adapter_linear
    i = _inputs(T, K, N, r, 1500, dtype, seed=T)
    g = torch.Generator().manual_seed(used)
    some = torch.randperm(1500, generator=g)[:used]
    for ids in (some[torch.arange(T) * used // T], some[torch.randint(0, used, (T,), generator=g)]):
        i["ids"] = ids.cuda()
        y, _, dA, dB = _check(i)
        others = torch.ones(1500, dtype=torch.bool)
        others[some] = False
        assert not dA[others.cuda()].any() and not dB[others.cuda()].any()
        with torch.no_grad():
            alone = adapter_linear(i["x"], i["w"], i["b"], i["A"], i["B"], i["ids"], scales=i["sc"])
        ref, tol = _ref(i)[0]
        assert bool(((alone.double().cpu() - ref).abs() <= tol).all())


@pytest.mark.parametrize("dtype,K,N", [(torch.float32, 23304, 23205), (torch.bfloat16, 32872, 32801)])
def test_a_projection_beyond_two_gib(dtype, K, N):
    """W (and its transpose in the backward pass) of 2 GiB and more: 32-bit offsets end inside of it.  References in 64 bits by pieces of W, the
    tolerances of the top of this file."""
    T, r, G = 70, 3, 2
    i = _inputs(T, 8, 8, r, G, dtype, "random")
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.empty(N, K, dtype=dtype, device="cuda")
    assert w.numel() * w.element_size() >= 1 << 31
    for a in range(0, N, 4096):
        w[a:a + 4096] = (torch.randn(min(4096, N - a), K, generator=g, device="cuda") / K ** 0.5).to(dtype)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
    i.update(w=w, x=rand(T, K).to(dtype).requires_grad_(True), b=rand(N).to(dtype), dy=rand(T, N).to(dtype),
             A=(rand(G, r, K) / K ** 0.5).to(dtype).requires_grad_(True), B=(rand(G, N, r) / r ** 0.5).to(dtype).requires_grad_(True))
    y, dx, dA, dB = _call(i)
    d = lambda t: t.detach().double()
    x, dy, A, B, sc, ids = d(i["x"]), d(i["dy"]), d(i["A"]), d(i["B"]), d(i["sc"]), i["ids"]
    ry, by = torch.empty(T, N, dtype=torch.float64, device="cuda"), torch.empty(T, N, dtype=torch.float64, device="cuda")
    rx, bx = torch.zeros(T, K, dtype=torch.float64, device="cuda"), torch.zeros(T, K, dtype=torch.float64, device="cuda")
    for a in range(0, N, 4096):
        wa = w[a:a + 4096].double()
        ry[:, a:a + 4096], by[:, a:a + 4096] = x @ wa.t(), x.abs() @ wa.abs().t()
        rx += dy[:, a:a + 4096] @ wa
        bx += dy[:, a:a + 4096].abs() @ wa.abs()
    b = d(i["b"])
    ry, ty, tx = ry + b, (K + r + 3) * U * (by + b.abs()), (N + r + 3) * U * bx
    rA, rB, tA, tB = (torch.zeros_like(t) for t in (A, B, A, B))
    s = SPLIT[dtype]
    for k in range(G):
        t = (ids == k).nonzero().view(-1)
        Ak, Bk, xa, da = A[k], B[k], x[t], dy[t]
        hh, ha = sc[k] * (xa @ Ak.t()), sc[k] * (xa.abs() @ Ak.abs().t())
        dh, dha = sc[k] * (da @ Bk), sc[k] * (da.abs() @ Bk.abs())
        ry[t] += hh @ Bk.t()
        rx[t] += dh @ Ak
        rA[k], rB[k] = dh.t() @ xa, da.t() @ hh
        ty[t] += ((2 * K + 2 * r + 8) * U + s) * (ha @ Bk.abs().t())
        tx[t] += ((2 * N + 2 * r + 8) * U + s) * (dha @ Ak.abs())
        e = (t.numel() + K + N + 8) * U + s
        tA[k], tB[k] = e * (dha.t() @ xa.abs()), e * (da.abs().t() @ ha)
    for name, got, ref, tol in (("y", y, ry, ty), ("dx", dx, rx, tx), ("dA", dA, rA, tA), ("dB", dB, rB, tB)):
        assert bool(((got.double() - ref).abs() <= tol + 1.01 * HALF[dtype] * ref.abs()).all()), name
