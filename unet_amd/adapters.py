"""Low-rank adapters of many requests at once beside one shared (frozen) projection, on the HIP kernels of `csrc/adapters.hip`.

One set of trained weights serves many machines or scenarios, each with a small correction of its own: row t of a batch is
projected by the shared weight and by the adapter that its id names,

    y[t] = W x[t] + b + s_a B_a (A_a x[t]),   a = ids[t].

No counterpart in the reference (its models are trained whole, per machine).  No CPU fallback."""
from __future__ import annotations

import torch
from torch import nn

from . import _lib as L

MAX_RANK = 128


class _AdapterFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, A, B, ids, scales):
        lib = L.lib()
        N, K = weight.shape
        G, r = A.shape[:2]
        dt = L.dtype_code(x, "adapter_linear")
        x2, ldx = L.rows_2d(x.detach(), K, aligned=True)
        w, ldw = L.rows_2d(weight.detach(), K, aligned=True)
        T, dev = x2.shape[0], x.device
        i64 = L.ids_flag(ids, "adapter_linear")
        Ad, Bd = L.rows_2d(A.detach().contiguous(), K, aligned=True)[0], L.rows_2d(B.detach().contiguous(), r, aligned=True)[0]
        y = torch.empty(*x.shape[:-1], N, dtype=x.dtype, device=dev)
        nk = L.check(lib.sx_adapter_kept_bytes(dt, T, r, G), "sx_adapter_kept_bytes")
        nw = L.check(lib.sx_adapter_workspace_bytes(dt, T, K, N, r, G, 0), "sx_adapter_workspace_bytes")
        kept = torch.empty(nk, dtype=torch.uint8, device=dev)
        ws = torch.empty(nw, dtype=torch.uint8, device=dev)
        with torch.cuda.device(dev):
            L.check(lib.sx_adapter_forward(dt, T, K, N, r, G, L.ptr(x2), ldx, L.ptr(w), ldw, L.ptr(bias), L.ptr(Ad), L.ptr(Bd), L.ptr(scales),
                                           L.ptr(ids), i64, L.ptr(y), N, L.ptr(kept), nk, L.ptr(ws), nw, L.stream_ptr()), "sx_adapter_forward")
        if any(ctx.needs_input_grad):
            ctx.save_for_backward(x, weight, A, B, scales, kept)
            ctx.meta = (dt, T, K, N, r, G)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        lib = L.lib()
        x, weight, A, B, scales, kept = ctx.saved_tensors
        dt, T, K, N, r, G = ctx.meta
        need_x, need_a, need_b = ctx.needs_input_grad[0], ctx.needs_input_grad[3], ctx.needs_input_grad[4]
        dev = x.device
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
        dA = torch.empty(A.shape, dtype=A.dtype, device=dev) if need_a else None
        dB = torch.empty(B.shape, dtype=B.dtype, device=dev) if need_b else None
        if T == 0:
            for g in (dA, dB):
                if g is not None:
                    g.zero_()
            return dx, None, None, dA, dB, None, None
        x2, ldx = L.rows_2d(x.detach(), K)
        w, ldw = L.rows_2d(weight.detach(), K)
        d2, ldd = L.rows_2d(dy, N, aligned=True)
        Ad, Bd = A.detach().contiguous(), B.detach().contiguous()
        nw = L.check(lib.sx_adapter_workspace_bytes(dt, T, K, N, r, G, 1), "sx_adapter_workspace_bytes")
        ws = torch.empty(nw, dtype=torch.uint8, device=dev)
        with torch.cuda.device(dev):
            L.check(lib.sx_adapter_backward(dt, T, K, N, r, G, L.ptr(x2), ldx, L.ptr(w), ldw, L.ptr(Ad), L.ptr(Bd), L.ptr(scales), L.ptr(d2), ldd,
                                            L.ptr(kept), kept.numel(), L.ptr(dx), L.ptr(dA), L.ptr(dB), L.ptr(ws), nw, L.stream_ptr()),
                    "sx_adapter_backward")
        return dx, None, None, dA, dB, None, None


def adapter_linear(x, weight, bias, A, B, ids, *, scales=None):
    """y = x W^T + bias + scales[a] * (x A_a^T) B_a^T for every row of x, a being the row's adapter.

    x (..., K); weight (N, K) and bias (N,) or None: the shared projection, frozen (neither may require a gradient); A (G, r, K) and
    B (G, N, r): the adapters, 1 <= r <= 128; all of one dtype, fp32 or bf16.  scales (G,) fp32 or None = 1.  ids: int64 / int32, one
    per row (x.shape[:-1]) or one per leading index of x (x.shape[:k], k >= 1: e.g. one per request of (requests, tokens, K)); an id
    outside [0, G) -- -1 by convention -- means the shared projection alone.  Sums in fp32, one rounding at the end; the same bits on every
    run.  Gradients go to x, A and B (zeros for an adapter no row names).  Not differentiable twice."""
    who = "adapter_linear"
    for t in (x, weight, A, B, ids):
        if not t.is_cuda:
            raise RuntimeError(f"{who}: the HIP path needs CUDA (ROCm) tensors; this build has no CPU path")
    if weight.dim() != 2 or x.dim() < 1 or weight.shape[1] < 1 or weight.shape[0] < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"{who}: x must be (..., K) and weight (N, K), got {tuple(x.shape)} / {tuple(weight.shape)}")
    N, K = weight.shape
    if A.dim() != 3 or B.dim() != 3 or A.shape[2] != K or tuple(B.shape) != (A.shape[0], N, A.shape[1]):
        raise ValueError(f"{who}: A must be (G, r, {K}) and B (G, {N}, r), got {tuple(A.shape)} / {tuple(B.shape)}")
    G, r = A.shape[:2]
    if not (1 <= r <= MAX_RANK and G >= 1):
        raise ValueError(f"{who}: rank {r} must be 1..{MAX_RANK} and there must be an adapter, got {G}")
    if bias is not None and tuple(bias.shape) != (N,):
        raise ValueError(f"{who}: bias must be ({N},), got {tuple(bias.shape)}")
    if scales is not None and tuple(scales.shape) != (G,):
        raise ValueError(f"{who}: scales must be ({G},), got {tuple(scales.shape)}")
    L.dtype_code(x, who), L.ids_flag(ids, who)
    for t in (weight, A, B) + (() if bias is None else (bias,)):
        if t.dtype != x.dtype:
            raise ValueError(f"{who}: weight, bias, A and B must have x's dtype {x.dtype}, got {t.dtype}")
    for t in (weight, A, B, ids) + tuple(t for t in (bias, scales) if t is not None):
        if t.device != x.device:
            raise ValueError(f"{who}: all tensors must be on {x.device}, got one on {t.device}")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (weight, bias, scales)):
        raise ValueError(f"{who}: the shared projection and the scales are frozen; pass them without requires_grad")
    lead = tuple(x.shape[:-1])
    if ids.dim() < (1 if lead else 0) or tuple(ids.shape) != lead[:ids.dim()]:
        raise ValueError(f"{who}: ids must be {lead} or one per leading index of it, got {tuple(ids.shape)}")
    if ids.dim() < len(lead):
        ids = ids.reshape(tuple(ids.shape) + (1,) * (len(lead) - ids.dim())).expand(lead)
    if scales is not None:
        scales = scales.detach().float().contiguous()
    return _AdapterFn.apply(x, weight, None if bias is None else bias.contiguous(), A, B, ids.contiguous(), scales)


class AdapterLinear(nn.Module):
    """An `nn.Linear` kept frozen, with `num` adapters of rank `rank` beside it: `A` ~ N(0, 1 / in_features), `B` = 0 (the projection
    starts as the shared one), every adapter scaled by alpha / rank.  `forward(x, ids)` is `adapter_linear`."""

    def __init__(self, linear, num, rank, alpha=None):
        super().__init__()
        self.linear = linear
        for p in linear.parameters():
            p.requires_grad_(False)
        N, K = linear.weight.shape
        kw = dict(dtype=linear.weight.dtype, device=linear.weight.device)
        self.A = nn.Parameter(torch.randn(num, rank, K, **kw) / K ** 0.5)
        self.B = nn.Parameter(torch.zeros(num, N, rank, **kw))
        self.register_buffer("scales", torch.full((num,), float(rank if alpha is None else alpha) / rank, device=linear.weight.device))

    def forward(self, x, ids):
        return adapter_linear(x, self.linear.weight, self.linear.bias, self.A, self.B, ids, scales=self.scales)
