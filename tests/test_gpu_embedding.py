"""GPU: scaled_embedding and its gradient against a plain implementation in 64 bits.

Tolerances (u = 2^-24, h = half a step of the output type: 2^-24 fp32, 2^-8 bf16): the lookup is one fp32 product and one rounding,
so |err| <= (u + h) |ref| (1 + u) -> 1.01 * (u + h) |ref|.  The gradient adds n rows in fp32 (each addition off by u of a partial sum
that never exceeds sum |d|), multiplies by the scale and rounds: |err| <= 1.01 * (n u scale sum|d| + (u + h) |ref|)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def _ref(ids, table, scale, dout):
    i, t, d = ids.long().cpu().reshape(-1), table.detach().double().cpu(), dout.double().cpu().reshape(-1, table.shape[1])
    ok = (i >= 0) & (i < t.shape[0])
    out = torch.zeros(i.numel(), t.shape[1], dtype=torch.float64)
    out[ok] = t[i[ok]] * scale
    grad = torch.zeros_like(t).index_add_(0, i[ok], d[ok]) * scale
    size = torch.zeros_like(t).index_add_(0, i[ok], d[ok].abs()) * scale
    count = torch.zeros(t.shape[0], dtype=torch.float64).index_add_(0, i[ok], torch.ones(int(ok.sum()), dtype=torch.float64))
    return out.view(*ids.shape, t.shape[1]), grad, size, count


def _check(ids, table, scale, dout):
    from unet_amd.embedding import scaled_embedding
    out = scaled_embedding(ids, table, scale)
    (grad,) = torch.autograd.grad(out, (table,), dout)
    ro, rg, size, count = _ref(ids, table, scale, dout)
    h = HALF[table.dtype]
    assert out.dtype == table.dtype and grad.dtype == table.dtype and out.shape == (*ids.shape, table.shape[1])
    assert ((out.detach().double().cpu() - ro).abs() <= 1.01 * (U + h) * ro.abs()).all()
    assert ((grad.double().cpu() - rg).abs() <= 1.01 * (count[:, None] * U * size + (U + h) * rg.abs())).all()
    return out, grad


def _inputs(shape, V, D, dtype, idt, kind, seed=0):
    g = torch.Generator().manual_seed(seed)
    if kind == "one":
        ids = torch.full(shape, V // 2)
    elif kind == "none":
        ids = torch.full(shape, -1)
    elif kind == "hot":                          # one row takes most of the tokens, the others few
        ids = torch.where(torch.rand(shape, generator=g) < 0.7, torch.tensor(V - 1), torch.randint(0, V, shape, generator=g))
    else:                                        # with ids outside the table on both sides
        ids = torch.randint(-3, V + 3, shape, generator=g)
    table = torch.randn(V, D, generator=g).to(dtype)
    dout = torch.randn(*shape, D, generator=g).to(dtype)
    return ids.to(idt).cuda(), table.cuda().requires_grad_(True), dout.cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,V,D", [((1,), 1, 1), ((1,), 5, 8), ((7,), 3, 7), ((63,), 50, 33), ((64,), 64, 64), ((65,), 11, 128), ((3, 43), 17, 331),
                                       ((129,), 2, 1030), ((1000,), 2050, 16), ((4, 5, 13), 1500, 72), ((2049,), 9, 264)])
def test_lookup_and_gradient(shape, V, D, dtype):
    for kind, idt, scale in (("any", torch.int64, 1.0), ("hot", torch.int32, 32.0), ("one", torch.int64, 0.375)):
        _check(*_inputs(shape, V, D, dtype, idt, kind)[:2], scale, _inputs(shape, V, D, dtype, idt, kind)[2])


def test_rows_that_several_runs_share():
    """Rows with exactly 64, 65, 128 and 1000 tokens next to each other: a run of 64 sorted entries that ends on a row's border, inside it
    and that lies in one row entirely."""
    counts = [3, 64, 65, 0, 128, 1000, 1, 63, 192, 0]
    ids = torch.cat([torch.full((c,), v) for v, c in enumerate(counts)])
    ids = ids[torch.randperm(ids.numel(), generator=torch.Generator().manual_seed(3))].cuda()
    for D in (20, 256, 2000):
        g = torch.Generator().manual_seed(D)
        table = torch.randn(len(counts), D, generator=g).cuda().requires_grad_(True)
        _check(ids, table, 2.0, torch.randn(ids.numel(), D, generator=g).cuda())


def test_gradient_has_the_same_bits_on_every_run_and_writes_every_row():
    from unet_amd.embedding import scaled_embedding
    ids, table, dout = _inputs((3000,), 400, 96, torch.float32, torch.int64, "hot")
    grads = []
    for i in range(3):
        torch.full((400, 96), float("nan"), device="cuda")          # what a reused allocation may hold
        grads.append(torch.autograd.grad(scaled_embedding(ids, table, 1.5), (table,), dout)[0])
    assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[2]) and torch.isfinite(grads[0]).all()


def test_padding_only_and_empty_batches():
    from unet_amd.embedding import scaled_embedding
    ids, table, dout = _inputs((70,), 30, 24, torch.bfloat16, torch.int32, "none")
    out, grad = _check(ids, table, 1.0, dout)
    assert not out.any() and not grad.any()
    e = torch.empty(0, 4, dtype=torch.int64, device="cuda")
    out = scaled_embedding(e, table)
    assert out.shape == (0, 4, 24)
    (grad,) = torch.autograd.grad(out, (table,), torch.empty(0, 4, 24, dtype=torch.bfloat16, device="cuda"))
    assert grad.shape == table.shape and not grad.any()


def test_padding_keeps_nan_rows_out():
    """NaN gradients of padded tokens and NaN rows of the table that no id names stay where they are."""
    ids, table, dout = _inputs((200,), 40, 16, torch.float32, torch.int64, "any")
    bad = (ids < 0) | (ids >= 40)
    assert bad.any()
    with torch.no_grad():
        ids[ids == 7] = 8
        table[7] = float("nan")
    from unet_amd.embedding import scaled_embedding
    dout[bad] = float("nan")
    out = scaled_embedding(ids, table, 2.0)
    (grad,) = torch.autograd.grad(out, (table,), dout)
    assert torch.isfinite(out).all() and torch.isfinite(grad).all()


def test_strided_and_misaligned_operands():
    """A table that is a column range of a wider one, a transposed id tensor, a gradient that is a slice or broadcast."""
    g = torch.Generator().manual_seed(5)
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.randn(50, 90, generator=g).to(dtype).cuda()
        ids = torch.randint(0, 50, (9, 21), generator=g).cuda().t()
        for c0, D in ((0, 64), (1, 64), (8, 80), (3, 87)):
            table = wide[:, c0:c0 + D].detach().requires_grad_(True)
            big = torch.randn(21, 9, D + 5, generator=g).to(dtype).cuda()
            _check(ids, table, 0.5, big[..., 2:2 + D])
            _check(ids, table, 0.5, big[:1, :1, :D].expand(21, 9, D))


def test_other_stream_and_graph_replays():
    from unet_amd.embedding import scaled_embedding
    ids, table, dout = _inputs((500,), 60, 128, torch.float32, torch.int64, "hot")
    want = torch.autograd.grad(scaled_embedding(ids, table, 2.0), (table,), dout)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = torch.autograd.grad(scaled_embedding(ids, table, 2.0), (table,), dout)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = scaled_embedding(ids, table, 2.0)
        grad = torch.autograd.grad(out, (table,), dout)[0]
    for seed in range(3):
        ids2, _, dout2 = _inputs((500,), 60, 128, torch.float32, torch.int64, "any", seed=seed + 10)
        ids.copy_(ids2), dout.copy_(dout2)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, torch.autograd.grad(scaled_embedding(ids, table, 2.0), (table,), dout)[0])
        assert torch.equal(out, scaled_embedding(ids, table, 2.0))


def test_gradient_against_differences():
    from unet_amd.embedding import scaled_embedding
    ids, table, dout = _inputs((40,), 12, 8, torch.float32, torch.int64, "any")
    (grad,) = torch.autograd.grad(scaled_embedding(ids, table, 2.0), (table,), dout)
    with torch.no_grad():
        for v, c in ((0, 0), (5, 3), (11, 7)):
            hi, lo = table.clone(), table.clone()
            hi[v, c] += 0.5
            lo[v, c] -= 0.5
            diff = ((scaled_embedding(ids, hi, 2.0).double() - scaled_embedding(ids, lo, 2.0).double()) * dout.double()).sum()
            assert abs(float(diff) - float(grad[v, c])) <= 1e-4           # linear: only fp32 roundings of ~40 terms of size ~4 differ


def test_module_feeds_film_parameters():
    """The lookup as the network's conditions: UNet params from a learned table, trained through the U-Net's backward pass."""
    from unet_amd import ScaledEmbedding, UNet
    torch.manual_seed(0)
    net, emb = UNet(1, 2, 8, P=5, film_hidden=16, depth=2).cuda().train(), ScaledEmbedding(7, 5).cuda()
    for m in net.modules():
        if hasattr(m, "n_channels"):
            torch.nn.init.normal_(m.net[-1].weight, std=0.1)
    ids = torch.tensor([2, 6, 2], device="cuda")
    net(torch.randn(3, 1, 16, 8, device="cuda"), params=emb(ids)).square().sum().backward()
    g = emb.weight.grad
    assert torch.isfinite(g).all() and g[2].abs().max() > 0 and g[6].abs().max() > 0
    assert not g[[0, 1, 3, 4, 5]].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D,offset,extra", [(500, 0, 0), (500, 4, 0), (634, 0, 6), (634, 2, 10), (96, 2, 8), (96, 1, 7), (1028, 0, 4), (2054, 0, 2)])
def test_every_width_of_loads(D, offset, extra, dtype):
    """Row lengths, strides and starts that allow loads of 16 bytes, of half, a quarter, an eighth of that, in tables and in upstream
    gradients that are views of wider ones."""
    ids, _, _ = _inputs((700,), 90, 8, dtype, torch.int64, "any")
    g = torch.Generator().manual_seed(D + offset)
    wide = torch.randn(90, D + offset + extra, generator=g).to(dtype).cuda()
    table = wide[:, offset:offset + D].requires_grad_(True)
    dout = torch.randn(700, D + offset + extra, generator=g).to(dtype).cuda()[:, offset:offset + D]
    _check(ids, table, 3.0, dout)


def test_padding_is_zero_whatever_the_scale():
    from unet_amd.embedding import scaled_embedding
    table = torch.ones(3, 40, device="cuda", requires_grad=True)
    out = scaled_embedding(torch.tensor([-1, 1, 3], device="cuda"), table, float("inf"))
    assert torch.equal(out[0], torch.zeros(40, device="cuda")) and torch.equal(out[2], out[0]) and torch.isinf(out[1]).all()
    (grad,) = torch.autograd.grad(out, (table,), torch.ones_like(out))
    assert torch.equal(grad[0], torch.zeros(40, device="cuda")) and torch.equal(grad[2], grad[0]) and torch.isinf(grad[1]).all()


@pytest.mark.parametrize("n,V", [(16384, 1), (50000, 20), (50000, 300000), (300001, 70), (17_000_000, 5)])
def test_many_ids(n, V):
    """More ids of one row than a block's list holds, on its own or beside rare ones; more than an entry of a list can number.  Gradients of
    ones are counts: whole numbers below 2^24, exact."""
    from unet_amd.embedding import scaled_embedding
    g = torch.Generator().manual_seed(n)
    ids = torch.where(torch.rand(n, generator=g) < 0.8, torch.tensor(V // 2), torch.randint(-1, V + 1, (n,), generator=g)).to(torch.int32)
    table = torch.zeros(V, 1, device="cuda", requires_grad=True)
    out = scaled_embedding(ids.cuda(), table)
    (grad,) = torch.autograd.grad(out, (table,), torch.ones_like(out))
    ok = (ids >= 0) & (ids < V)
    assert torch.equal(grad[:, 0].cpu().double(), torch.bincount(ids[ok].long(), minlength=V).double())
    if n < 10 ** 6:
        w = torch.randn(n, 1, generator=g)
        a, b = (torch.autograd.grad(scaled_embedding(ids.cuda(), table), (table,), w.cuda())[0] for _ in range(2))
        want = torch.zeros(V, 1, dtype=torch.float64).index_add_(0, ids[ok].long(), w[ok].double())
        size = torch.zeros(V, 1, dtype=torch.float64).index_add_(0, ids[ok].long(), w[ok].double().abs())
        assert torch.equal(a, b) and bool(((a.cpu().double() - want).abs() <= 1.01 * (n * U * size + U * want.abs()) + 1e-38).all())
