"""Low-rank adapters of many requests at once beside one shared (frozen) projection, on the HIP kernels of `csrc/adapters.hip`.

One set of trained weights serves many machines or scenarios, each with a small correction of its own: row t of a batch is
projected by the shared weight and by the adapter that its id names,

    y[t] = W x[t] + b + s_a B_a (A_a x[t]),   a = ids[t].

No counterpart in the reference (its models are trained whole, per machine).  No CPU fallback."""
from __future__ import annotations

import torch
from torch import nn

from . import _lib as L

MAX_RANK, MAX_ADAPTERS = 128, 65535


def _project(x, weight, bias, A, B, ids, scales, keep):
    """(y, what the backward pass needs of it if `keep`)"""
    N, K = weight.shape
    G, r = A.shape[:2]
    dt, dev = L.dtype_code(x, "adapter_linear"), x.device
    x2, ldx = L.rows_2d(x, K, aligned=True)
    w, ldw = L.rows_2d(weight, K, aligned=True)
    T = x2.shape[0]
    Ad, Bd = L.packed(A, aligned=True), L.packed(B, aligned=True)
    y = torch.empty(*x.shape[:-1], N, dtype=x.dtype, device=dev)
    nk = L.size_of("sx_adapter_kept_bytes", dt, T, r, G) if keep else 0
    nw = L.size_of("sx_adapter_workspace_bytes", dt, T, K, N, r, G, L.SX_ADAPTER_FORWARD if keep else L.SX_ADAPTER_ALONE)
    kept = torch.empty(nk, dtype=torch.uint8, device=dev) if keep else None
    ws = torch.empty(nw, dtype=torch.uint8, device=dev)
    L.launch("sx_adapter_forward", dev, dt, T, K, N, r, G, L.addr(x2), ldx, L.addr(w), ldw, L.addr(bias), L.addr(Ad), L.addr(Bd), L.addr(scales),
             L.addr(ids), L.ids_flag(ids, "adapter_linear"), L.addr(y), N, L.addr(kept), nk, L.addr(ws), nw)
    return y, kept


class _AdapterFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, A, B, ids, scales):
        y, kept = _project(x, weight, bias, A, B, ids, scales, any(ctx.needs_input_grad))
        ctx.save_for_backward(x, weight, A, B, scales, kept)
        return y

    @staticmethod
    def backward(ctx, dy):
        saved = ctx.saved_tensors                  # once: recomputed ones are handed out a single time
        if not torch.is_grad_enabled():
            dx, dA, dB = _AdapterFn.gradients(ctx, saved, dy)
        else:
            who, (x, _, A, B, _, _) = "adapter_linear", saved
            with torch.no_grad():
                dx, dA, dB = _AdapterFn.gradients(ctx, saved, dy)
            dx, dA, dB = L.not_twice(who, dx, dy, A, B), L.not_twice(who, dA, dy, x, B), L.not_twice(who, dB, dy, x, A)
        return dx, None, None, dA, dB, None, None

    @staticmethod
    def gradients(ctx, saved, dy):
        x, weight, A, B, scales, kept = saved
        need_x, _, _, need_a, need_b = ctx.needs_input_grad[:5]
        N, K = weight.shape
        G, r = A.shape[:2]
        dt, dev = L.dtype_code(x, "adapter_linear"), x.device
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
        dA = torch.empty(A.shape, dtype=A.dtype, device=dev) if need_a else None
        dB = torch.empty(B.shape, dtype=B.dtype, device=dev) if need_b else None
        x2, ldx = L.rows_2d(x, K)
        T = x2.shape[0]
        if T == 0:
            for g in (dA, dB):
                if g is not None:
                    g.zero_()
            return dx, dA, dB
        w, ldw = L.rows_2d(weight, K)
        d2, ldd = L.rows_2d(dy, N, aligned=True)
        Ad, Bd = L.packed(A), L.packed(B)
        nw = L.size_of("sx_adapter_workspace_bytes", dt, T, K, N, r, G, L.SX_ADAPTER_BACKWARD)
        ws = torch.empty(nw, dtype=torch.uint8, device=dev)
        L.launch("sx_adapter_backward", dev, dt, T, K, N, r, G, L.addr(x2), ldx, L.addr(w), ldw, L.addr(Ad), L.addr(Bd), L.addr(scales), L.addr(d2), ldd,
                 L.addr(kept), kept.numel(), L.addr(dx), L.addr(dA), L.addr(dB), L.addr(ws), nw)
        return dx, dA, dB


def adapter_linear(x, weight, bias, A, B, ids, *, scales=None):
    """y = x W^T + bias + scales[a] * (x A_a^T) B_a^T for every row of x, a being the row's adapter.

    x (..., K); weight (N, K) and bias (N,) or None: the shared projection, frozen (neither may require a gradient); A (G, r, K) and
    B (G, N, r): the adapters, 1 <= r <= 128; all of one dtype, fp32 or bf16.  scales (G,) fp32 or None = 1.  ids: int64 / int32, one
    per row (x.shape[:-1]) or one per leading index of x (x.shape[:k], k >= 1: e.g. one per request of (requests, tokens, K)); an id
    outside [0, G) -- -1 by convention -- means the shared projection alone.  Sums in fp32, one rounding at the end; the same bits on every
    run.  Gradients go to x, A and B (zeros for an adapter no row names).  Not differentiable twice."""
    who = "adapter_linear"
    if not (x.is_cuda and weight.is_cuda and A.is_cuda and B.is_cuda and ids.is_cuda):
        raise RuntimeError(f"{who}: the HIP path needs CUDA (ROCm) tensors; this build has no CPU path")
    if weight.dim() != 2 or x.dim() < 1 or weight.shape[1] < 1 or weight.shape[0] < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"{who}: x must be (..., K) and weight (N, K), got {tuple(x.shape)} / {tuple(weight.shape)}")
    N, K = weight.shape
    if A.dim() != 3 or B.dim() != 3 or A.shape[2] != K or tuple(B.shape) != (A.shape[0], N, A.shape[1]):
        raise ValueError(f"{who}: A must be (G, r, {K}) and B (G, {N}, r), got {tuple(A.shape)} / {tuple(B.shape)}")
    G, r = A.shape[:2]
    if not (1 <= r <= MAX_RANK and 1 <= G <= MAX_ADAPTERS):
        raise ValueError(f"{who}: rank {r} must be 1..{MAX_RANK} and there must be an adapter, at most {MAX_ADAPTERS}, got {G}")
    if max(N, K) > L.MAX_WIDTH:
        raise ValueError(f"{who}: a projection of {K} to {N} is too large")
    if bias is not None and tuple(bias.shape) != (N,):
        raise ValueError(f"{who}: bias must be ({N},), got {tuple(bias.shape)}")
    if scales is not None and tuple(scales.shape) != (G,):
        raise ValueError(f"{who}: scales must be ({G},), got {tuple(scales.shape)}")
    L.dtype_code(x, who), L.ids_flag(ids, who)
    dtype, dev = x.dtype, x.device
    if not (weight.dtype == A.dtype == B.dtype == dtype and (bias is None or bias.dtype == dtype)):
        raise ValueError(f"{who}: weight, bias, A and B must have x's dtype {dtype}")
    if not (weight.device == A.device == B.device == ids.device == dev and (bias is None or bias.device == dev) and (scales is None or scales.device == dev)):
        raise ValueError(f"{who}: all tensors must be on x's device {dev}")
    if L.wants_grad(weight, bias, scales):
        raise ValueError(f"{who}: the shared projection and the scales are frozen; pass them without requires_grad")
    lead = tuple(x.shape[:-1])
    if ids.dim() < (1 if lead else 0) or tuple(ids.shape) != lead[:ids.dim()]:
        raise ValueError(f"{who}: ids must be {lead} or one per leading index of it, got {tuple(ids.shape)}")
    if ids.dim() < len(lead):
        ids = ids.reshape(tuple(ids.shape) + (1,) * (len(lead) - ids.dim())).expand(lead)
    args = (x, weight, None if bias is None else L.packed(bias), A, B, L.packed(ids), None if scales is None else L.plain_f32(scales))
    return _AdapterFn.apply(*args) if L.by_autograd(x, A, B) else _project(*args, False)[0]


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
