"""Learned rows for discrete conditions (machine, scenario, parameter bin): a scaled table lookup and its gradient on the HIP
kernels of `csrc/embedding.hip`.  No counterpart in the reference, whose conditions are all continuous (`params`); the rows
feed the same places, e.g. `UNet(..., P=dim)(x, params=scaled_embedding(ids, table))` with dim <= 64, the most that the U-Net
takes, or the latent MLPs' input.  No CPU fallback."""
from __future__ import annotations

import torch
from torch import nn

from . import _lib as L


def _lookup(ids, table, scale):
    """(flat ids, output)"""
    V, D = table.shape
    i = L.packed(ids)
    t, ld = L.rows_2d(table, D)
    out = torch.empty(*ids.shape, D, dtype=table.dtype, device=table.device)
    L.launch("sx_embedding_forward", table.device, L.dtype_code(table, "scaled_embedding"), i.numel(), V, D, L.addr(t), ld, L.addr(i),
             L.ids_flag(i, "scaled_embedding"), scale, L.addr(out))
    return i, out


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale):
        i, out = _lookup(ids, table, scale)
        ctx.save_for_backward(i)
        ctx.meta = (*table.shape, scale, table.dtype)
        return out

    @staticmethod
    def backward(ctx, dout):
        if torch.is_grad_enabled():
            with torch.no_grad():
                grads = _EmbeddingFn.backward(ctx, dout)
            return None, L.not_twice("scaled_embedding", grads[1], dout), None
        (i,) = ctx.saved_tensors
        V, D, scale, dtype = ctx.meta
        n, dev = i.numel(), dout.device
        d, ld = L.rows_2d(dout, D)
        grad = torch.empty(V, D, dtype=dtype, device=dev)
        nb = L.size_of("sx_embedding_workspace_bytes", n, V, D)
        ws = torch.empty(nb, dtype=torch.uint8, device=dev)
        L.launch("sx_embedding_backward", dev, L.dtype_code(grad, "scaled_embedding"), n, V, D, L.addr(d), ld, L.addr(i),
                 L.ids_flag(i, "scaled_embedding"), scale, L.addr(grad), L.addr(ws), nb)
        return None, grad, None


def scaled_embedding(ids, table, scale=1.0):
    """out[..., :] = scale * table[ids[...], :] in the table's dtype (fp32 or bf16; one rounding).

    table (rows, dim), at most 2^24 rows.  ids: int64 / int32 of any shape, on the table's device.  An id outside [0, rows) -- -1 by convention -- is padding: a row of
    zeros, no gradient.  The table's gradient sums the tokens of a row in their order, in fp32: the same bits on every run.
    Not differentiable twice.  `scale` is a number."""
    who = "scaled_embedding"
    if not table.is_cuda or not ids.is_cuda:
        raise RuntimeError(f"{who}: the HIP path needs CUDA (ROCm) tensors; this build has no CPU path")
    if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1:
        raise ValueError(f"{who}: table must be (rows, dim) with at least one of each, got {tuple(table.shape)}")
    if table.shape[1] > L.MAX_WIDTH:
        raise ValueError(f"{who}: rows of {table.shape[1]} are too long")
    if ids.device != table.device:
        raise ValueError(f"{who}: ids are on {ids.device}, the table on {table.device}")
    L.ids_flag(ids, who)
    L.dtype_code(table, who)
    return _EmbeddingFn.apply(ids, table, float(scale)) if L.by_autograd(table) else _lookup(ids, table, float(scale))[1]


class ScaledEmbedding(nn.Module):
    """`scaled_embedding` with its table as the parameter `weight` (num, dim), initialised N(0, 1) / scale."""

    def __init__(self, num, dim, scale=1.0):
        super().__init__()
        self.scale = float(scale)
        self.weight = nn.Parameter(torch.empty(num, dim))
        nn.init.normal_(self.weight, std=1.0 / abs(self.scale) if self.scale else 1.0)

    def forward(self, ids):
        return scaled_embedding(ids, self.weight, self.scale)
