"""CPU: what the scaled embedding, the adapter projection, the distillation loss and their C entry points refuse, before anything reaches a GPU."""
import ctypes

import pytest
import torch


def test_embedding_refusals():
    from unet_amd.embedding import scaled_embedding
    ids = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        scaled_embedding(ids, torch.zeros(4, 8))


def test_distillation_refusals():
    from unet_amd.losses import distillation_loss
    z, top, idx = torch.zeros(3, 10), torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        distillation_loss(z, top, idx)
    with pytest.raises(ValueError, match="reduction"):
        distillation_loss(z, top, idx, reduction="median")
    for t in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            distillation_loss(z, top, idx, temperature=t)


P = ctypes.c_void_p(4096)          # an address that a refused call never reads


def _bad(rc):
    from unet_amd import _lib as L
    with pytest.raises(ValueError):
        L.check(rc)


def test_embedding_c_entry_refusals():
    from unet_amd import _lib as L
    lib = L.lib()
    need = lib.sx_embedding_workspace_bytes(100, 50, 16)
    assert need > 0
    for n, rows, dim in ((-1, 5, 4), (1, 0, 4), (1, 5, 0), (1, (1 << 24) + 1, 4), (1 << 31, 5, 4)):
        _bad(lib.sx_embedding_workspace_bytes(n, rows, dim))
    _bad(lib.sx_embedding_forward(7, 10, 5, 4, P, 4, P, 1, 1.0, P, None))
    _bad(lib.sx_embedding_forward(0, 10, 5, 4, P, 3, P, 1, 1.0, P, None))
    _bad(lib.sx_embedding_forward(0, 10, 5, 4, None, 4, P, 1, 1.0, P, None))
    _bad(lib.sx_embedding_forward(0, 10, 5, 4, P, 4, None, 1, 1.0, P, None))
    _bad(lib.sx_embedding_backward(0, 100, 50, 16, P, 16, P, 1, 1.0, P, P, need - 1, None))
    _bad(lib.sx_embedding_backward(0, 100, 50, 16, P, 16, P, 1, 1.0, P, ctypes.c_void_p(4100), need, None))
    _bad(lib.sx_embedding_backward(0, 100, 50, 16, P, 16, P, 1, 1.0, None, P, need, None))
    _bad(lib.sx_embedding_backward(0, 100, 50, 16, P, 15, P, 1, 1.0, P, P, need, None))
    assert lib.sx_embedding_forward(0, 0, 5, 4, None, 4, None, 1, 1.0, None, None) == 0


def test_distill_c_entry_refusals():
    from unet_amd import _lib as L
    lib = L.lib()

    def fwd(dt=0, N=3, V=10, K=2, z=P, ld=10, tdt=0, top=P, idx=P, tau=1.0, w=None, mean=1, rows=P, den=P, d=None, ldd=10):
        return lib.sx_distill_forward(dt, N, V, K, z, ld, tdt, top, idx, 1, tau, w, mean, rows, None, den, None, d, ldd, None)
    for kw in (dict(dt=3), dict(tdt=2), dict(N=-1), dict(N=1 << 22), dict(V=0), dict(K=0), dict(ld=9), dict(tau=0.0), dict(tau=float("nan")),
               dict(tau=float("inf")), dict(z=None), dict(top=None), dict(idx=None), dict(rows=None), dict(d=P, ldd=9), dict(w=P, den=None)):
        _bad(fwd(**kw))

    def bwd(dt=0, V=10, ld=10, tau=1.0, stats=P, g=P, d=P, ldd=10, w=None, den=None):
        return lib.sx_distill_backward(dt, 3, V, 2, P, ld, 0, P, P, 1, tau, w, 1, stats, den, g, 0, 0, d, ldd, None)
    for kw in (dict(dt=5), dict(V=-1), dict(ld=9), dict(tau=-1.0), dict(stats=None), dict(g=None), dict(d=None), dict(ldd=9), dict(w=P)):
        _bad(bwd(**kw))


def test_adapter_refusals():
    from unet_amd.adapters import adapter_linear
    with pytest.raises(RuntimeError, match="no CPU path"):
        adapter_linear(torch.zeros(2, 8), torch.zeros(4, 8), None, torch.zeros(1, 2, 8), torch.zeros(1, 4, 2), torch.zeros(2, dtype=torch.int64))


def test_adapter_c_entry_refusals():
    from unet_amd import _lib as L
    lib = L.lib()
    nk, nw, nb = lib.sx_adapter_kept_bytes(0, 10, 4, 3), lib.sx_adapter_workspace_bytes(0, 10, 16, 8, 4, 3, 0), lib.sx_adapter_workspace_bytes(0, 10, 16, 8, 4, 3, 1)
    na = lib.sx_adapter_workspace_bytes(0, 10, 16, 8, 4, 3, 2)
    assert nk > 0 and nw > 0 and nb > 0
    for T, r, G in ((-1, 4, 3), ((1 << 24) + 1, 4, 3), (1, 0, 3), (1, 129, 3), (1, 4, 0), (1, 4, 65536)):
        _bad(lib.sx_adapter_kept_bytes(0, T, r, G))
        _bad(lib.sx_adapter_workspace_bytes(0, T, 16, 8, r, G, 0))
    _bad(lib.sx_adapter_kept_bytes(4, 10, 4, 3))
    _bad(lib.sx_adapter_workspace_bytes(0, 10, 16, 8, 4, 3, 3))
    _bad(lib.sx_adapter_workspace_bytes(1, 10, 1 << 20, 8, 4, 1000, 1))
    for dt, K, N in ((2, 16, 8), (0, 0, 8), (0, 16, 0), (0, (1 << 20) + 1, 8), (1, 16, (1 << 20) + 1)):
        _bad(lib.sx_adapter_workspace_bytes(dt, 10, K, N, 4, 3, 1))

    def fwd(dt=0, T=10, r=4, G=3, x=P, ldx=16, w=P, ldw=16, A=P, B=P, ids=P, y=P, ldy=8, kept=P, nk=nk, ws=P, nw=nw):
        return lib.sx_adapter_forward(dt, T, 16, 8, r, G, x, ldx, w, ldw, None, A, B, None, ids, 1, y, ldy, kept, nk, ws, nw, None)
    odd = ctypes.c_void_p(4100)
    for kw in (dict(dt=9), dict(T=-5), dict(r=0), dict(r=200), dict(G=0), dict(x=None), dict(w=None), dict(A=None), dict(B=None), dict(ids=None),
               dict(y=None), dict(ws=None), dict(kept=None, nk=0, nw=na - 1), dict(ldx=15), dict(ldw=15), dict(ldy=7), dict(nk=nk - 1), dict(nw=nw - 1), dict(kept=odd),
               dict(ws=odd), dict(x=odd), dict(w=odd), dict(A=odd), dict(B=odd), dict(ldx=18), dict(ldw=17)):
        _bad(fwd(**kw))
    assert fwd(T=0) == 0

    def bwd(dt=0, T=10, x=P, ldx=16, w=P, ldw=16, A=P, B=P, dy=P, ldd=8, kept=P, nk=nk, ws=P, nw=nb):
        return lib.sx_adapter_backward(dt, T, 16, 8, 4, 3, x, ldx, w, ldw, A, B, None, dy, ldd, kept, nk, P, P, P, ws, nw, None)
    for kw in (dict(dt=9), dict(T=0), dict(x=None), dict(w=None), dict(A=None), dict(B=None), dict(dy=None), dict(kept=None), dict(ws=None), dict(ldx=15),
               dict(ldw=15), dict(ldd=7), dict(ldd=9), dict(dy=odd), dict(nk=nk - 1), dict(nw=nb - 1), dict(kept=odd), dict(ws=odd)):
        _bad(bwd(**kw))


def test_temperatures_and_sizes_out_of_reach_are_refused():
    """A temperature whose reciprocal is infinite in 32 bits, or that is infinite there itself; rows that 32-bit positions cannot number."""
    from unet_amd import _lib as L
    from unet_amd.losses import distillation_loss
    z = torch.zeros(2, 5)
    for t in (1e-40, 1e39):
        with pytest.raises(ValueError, match="temperature"):
            distillation_loss(z, z, torch.zeros(2, 5, dtype=torch.int64), temperature=t)
    lib, P = L.lib(), 4096
    for kw in (dict(V=(1 << 30) + 1), dict(K=(1 << 30) + 1), dict(tau=1e-40)):
        a = dict(V=10, K=2, tau=1.0)
        a.update(kw)
        assert lib.sx_distill_forward(0, 3, a["V"], a["K"], P, 1 << 31, 0, P, P, 1, a["tau"], None, 1, P, None, P, None, None, 10, None) < 0


def test_what_looks_into_calls_is_seen():
    """A direct call of the kernels would drop a tangent and leave nothing in a trace: forward mode, traces and function transforms are noticed."""
    from torch.autograd import forward_ad
    from unet_amd import _lib as L
    t, p, seen = torch.ones(3), torch.ones(3, requires_grad=True), []

    def f(x):
        seen.append(L.by_autograd(x))
        return x * 2
    f(t)
    f(p)
    with torch.no_grad():
        f(p)
        torch.jit.trace(f, (t,), check_trace=False)
    with forward_ad.dual_level():
        f(t)
    torch.func.vmap(f)(t)
    torch.func.jvp(f, (t,), (t,))
    f(t)
    assert seen == [False, True, False, True, True, True, True, False]


def test_embedding_workspace_holds_the_runs_there_are():
    """Two partial rows for each run of sorted ids, of which there are 1024 at most (4096 of rows that groups of 16 threads may take), however
    many ids; beside them a place and a bucket per id and two numbers per row of the table."""
    from unet_amd import _lib as L
    lib = L.lib()
    for n in (0, 16, 17, 1000, 65536, 70000, 1 << 24, (1 << 31) - 2048):
        for rows, dim in ((50, 1), (50, 128), (50, 129), (1 << 24, 1024), (7, 5000)):
            need, base, runs = lib.sx_embedding_workspace_bytes(n, rows, dim), 8 * n + 8 * (rows + 1), 4096 if dim <= 128 else 1024
            assert base <= need <= base + runs * 8 * dim + 5 * 256, (n, rows, dim)
            if n > 16:
                used = 16
                while used * runs < n:
                    used *= 2
                assert need >= base + (8 * dim * -(-n // used) if n > used else 0), (n, rows, dim)
