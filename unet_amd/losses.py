"""MI355X-native mirror of `solpex.losses` (reference: solpex/losses.py).

`masked_weighted_loss`, `mae_norm` and `batch_error_sums_ev` keep the reference signatures and error
behaviour; on device they run the fused HIP kernels of libsolpex_hip.so (loss forward AND its
gradient in one pass).  `edge_weights` stays host-side scipy exactly as in the reference (called once
per run, solpex/train.py:132-134).
"""
from __future__ import annotations

import numpy as np
import torch

from . import _lib as L

_BASES = ("huber", "l1", "mse")


def _require_cuda(t, who):
    if not t.is_cuda:
        raise RuntimeError(f"{who}: the HIP path needs CUDA (ROCm) tensors; this build has no CPU path")


def _nhwc(t):
    """(B,C,H,W) tensor -> (tensor, ld, sx dtype) readable by the NHWC kernels without a copy if possible."""
    B, Cc, H, W = t.shape
    sb, sc, sh, sw = t.stride()
    ok = (t.dtype in (torch.float32, torch.bfloat16) and (sc == 1 or Cc == 1) and sh == W * sw and sb == H * W * sw
          and sw >= Cc)
    if not ok:
        if t.dtype not in (torch.float32, torch.bfloat16):
            t = t.float()
        t = t.contiguous(memory_format=torch.channels_last)
        if Cc == 1:
            t = t.contiguous()
        sw = Cc
    return t, int(sw), (L.SX_BF16 if t.dtype == torch.bfloat16 else L.SX_F32)


def _prep_mask(mask, B, H, W, who):
    if mask.dim() != 4 or mask.shape[0] != B or mask.shape[1] != 1 or tuple(mask.shape[2:]) != (H, W):
        raise ValueError(f"{who}: mask must be (B,1,H,W) = ({B},1,{H},{W}), got {tuple(mask.shape)}")
    return mask.float().contiguous()


def _prep_w(w, H, W, device, who):
    if w is None:
        return None
    if not torch.is_tensor(w):
        w = torch.as_tensor(w)
    if w.numel() != H * W:
        raise ValueError(f"{who}: w must broadcast from (H,W) = ({H},{W}); per-sample weight maps are not supported, "
                         f"got {tuple(w.shape)}")
    return w.to(device=device, dtype=torch.float32).reshape(H, W).contiguous()


def _prep_cw(cw, Cc, device):
    if cw is None:
        return None
    if not torch.is_tensor(cw):
        cw = torch.as_tensor(np.asarray(cw, dtype=np.float32))
    cw = cw.to(device=device, dtype=torch.float32).reshape(-1).contiguous()
    if cw.numel() == 1 and Cc != 1:
        cw = cw.expand(Cc).contiguous()
    if cw.numel() != Cc:
        raise ValueError(f"channel_weights length={cw.numel()} but C={Cc}")
    return cw


class LossBuffers:
    """Device scratch for one loss shape (workspace, denominators, outputs)."""

    def __init__(self, B, Cc, H, W, multiscale, grad_ds, device):
        lib = L.lib()
        nbytes = L.check(lib.sx_loss_workspace_bytes(B, Cc, H, W, int(multiscale), int(grad_ds)))
        self.ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)
        self.den = torch.empty(9, dtype=torch.float32, device=device)
        self.out = torch.empty(4, dtype=torch.float32, device=device)    # loss, sum|p-t|*m, sum m, sum m


def loss_prepare(bufs, B, Cc, H, W, mask, w, multiscale, grad_ds, lam_grad):
    L.check(L.lib().sx_loss_prepare(B, Cc, H, W, L.ptr(mask), L.ptr(w), int(multiscale), int(grad_ds), float(lam_grad),
                                    L.ptr(bufs.ws), L.ptr(bufs.den), L.stream_ptr()), "sx_loss_prepare")


def loss_forward_backward(bufs, sx_dtype, B, Cc, H, W, pred, pred_ld, target, mask, w, cw, base, huber_beta, lam_w, lam_grad,
                          grad_mode, grad_base, multiscale, ms_weight, grad_ds, d_pred, dpred_ld, grad_scale=1.0, out=None,
                          bias_sums=None):
    """`bias_sums` (optional, zeroed [SX_HEAD_BIAS_SLOTS][C] fp32): also form the output head's bias gradient from d_pred;
    returns True when the kernels took it (then nothing may add to d_pred afterwards)."""
    import ctypes
    done = ctypes.c_int(0)
    L.check(L.lib().sx_loss_forward_backward_bias(
        sx_dtype, B, Cc, H, W, L.ptr(pred), pred_ld, L.ptr(target), L.ptr(mask), L.ptr(w), L.ptr(cw),
        L.PX_KINDS[base], float(huber_beta), float(lam_w), float(lam_grad), 1 if grad_mode == "magnitude" else 0,
        L.PX_KINDS[grad_base], int(multiscale), float(ms_weight), int(grad_ds), L.ptr(bufs.den), L.ptr(bufs.ws),
        L.ptr(bufs.out if out is None else out), L.ptr(d_pred), dpred_ld, float(grad_scale),
        L.ptr(bias_sums), ctypes.cast(ctypes.byref(done), ctypes.c_void_p) if bias_sums is not None else None, L.stream_ptr()),
        "sx_loss_forward_backward")
    return bool(done.value)


class _LossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, pred, target, mask, w, cw, opts):
        B, Cc, H, W = pred.shape
        p, ld, dt = _nhwc(pred.detach())
        need_grad = ctx.needs_input_grad[0]
        bufs = LossBuffers(B, Cc, H, W, opts["multiscale"], opts["grad_ds"], pred.device)
        loss_prepare(bufs, B, Cc, H, W, mask, w, opts["multiscale"], opts["grad_ds"], opts["lam_grad"])
        d_pred = None
        if need_grad:
            sess = getattr(pred, "_sx_sess", None)
            if sess is not None and sess.view(L.SX_T_PRED).data_ptr() == pred.data_ptr() and ld == sess.view(L.SX_T_PRED).stride(3):
                d_pred = sess.view(L.SX_T_DPRED)        # written in place: decode backward reads it without a copy
            else:
                d_pred = torch.empty_strided(p.shape, p.stride(), dtype=p.dtype, device=p.device)
        loss_forward_backward(bufs, dt, B, Cc, H, W, p, ld, target, mask, w, cw, opts["base"], opts["huber_beta"],
                              opts["lam_w"], opts["lam_grad"], opts["grad_mode"], opts["grad_base"], opts["multiscale"],
                              opts["ms_weight"], opts["grad_ds"], d_pred, ld)
        ctx.d_pred = d_pred
        ctx.pred_dtype = pred.dtype
        return bufs.out[0].clone()

    @staticmethod
    def backward(ctx, g):
        d = ctx.d_pred
        d.mul_(g.to(d.dtype))      # in place: keeps the zero-copy hand-off to the decoder's backward
        if d.dtype != ctx.pred_dtype:
            d = d.to(ctx.pred_dtype)
        return d, None, None, None, None, None


def masked_weighted_loss(pred, target, mask, *, w=None, lam_grad=0.2, lam_w=1.0, base="huber", huber_beta=0.05,
                         grad_mode="vector", grad_base="l1", multiscale=0, ms_weight=0.5, grad_ds: int = 1,
                         channel_weights=None):
    """Reference: solpex/losses.py:82-213 (same arguments, same ValueErrors)."""
    if base not in _BASES:
        raise ValueError(f"Unknown base={base}")
    if lam_grad != 0.0 and grad_base not in _BASES:
        raise ValueError(f"Unknown grad_base={grad_base}")
    _require_cuda(pred, "masked_weighted_loss")
    if pred.dim() != 4 or tuple(target.shape) != tuple(pred.shape):
        raise ValueError(f"masked_weighted_loss: pred/target must both be (B,C,H,W), got {tuple(pred.shape)} / {tuple(target.shape)}")
    B, Cc, H, W = pred.shape
    if grad_ds is None or grad_ds < 1:
        grad_ds = 1
    opts = dict(lam_grad=float(lam_grad), lam_w=float(lam_w), base=base, huber_beta=float(huber_beta),
                grad_mode="magnitude" if grad_mode == "magnitude" else "vector",
                grad_base=grad_base if grad_base in _BASES else "l1",
                multiscale=int(min(max(int(multiscale or 0), 0), 2)), ms_weight=float(ms_weight), grad_ds=int(grad_ds))
    m = _prep_mask(mask, B, H, W, "masked_weighted_loss")
    wt = _prep_w(w, H, W, pred.device, "masked_weighted_loss")
    cw = _prep_cw(channel_weights, Cc, pred.device)
    tgt = target.detach().float().contiguous()
    return _LossFn.apply(pred, tgt, m, wt, cw, opts)


def _distill(logits, top, idx, weights, tau, reduction, need):
    """(loss, sum of the weights and row statistics, d loss / d logits), the last two only if `need`.  The gradient is formed here for the
    losses whose upstream gradient is mostly 1; that of a loss per row waits for its upstream gradient."""
    who = "distillation_loss"
    V, K = logits.shape[-1], top.shape[-1]
    z, ld = L.rows_2d(logits, V)
    N, dev = z.shape[0], logits.device
    rows = torch.empty(logits.shape[:-1], dtype=torch.float32, device=dev)
    loss = None if reduction == "none" else torch.empty((), dtype=torch.float32, device=dev)
    keep = torch.empty(1 + (4 * N if need else 0), dtype=torch.float32, device=dev)
    d = torch.empty(logits.shape, dtype=logits.dtype, device=dev) if need and reduction != "none" else None
    L.launch("sx_distill_forward", dev, L.dtype_code(logits, who), N, V, K, L.addr(z), ld, L.dtype_code(top, who), L.addr(top), L.addr(idx),
             L.ids_flag(idx, who), tau, L.addr(weights), 1 if reduction == "mean" else 0, L.addr(rows), L.addr(keep) + 4 if need else None, L.addr(keep),
             L.addr(loss), L.addr(d), V)
    return (rows if loss is None else loss), keep, d


class _DistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top, idx, weights, tau, reduction):
        loss, keep, d = _distill(logits, top, idx, weights, tau, reduction, ctx.needs_input_grad[0])
        ctx.save_for_backward(logits, top, idx, weights, keep, d)
        ctx.meta = (tau, reduction)
        ctx.made = None if d is None else L.capture_id(d.device)
        return loss

    @staticmethod
    def backward(ctx, g):
        saved = ctx.saved_tensors                  # once: recomputed ones are handed out a single time
        if not torch.is_grad_enabled():
            d = _DistillFn.gradient(ctx, saved, g)
        else:
            with torch.no_grad():
                d = _DistillFn.gradient(ctx, saved, g)
            d = L.not_twice("distillation_loss", d, g, saved[0])
        return d, None, None, None, None, None

    @staticmethod
    def gradient(ctx, saved, g):
        """Where the forward pass left the gradient for an upstream gradient of 1, that is it; for another one the gradient is computed
        again from the logits (one rounding), not scaled after its own."""
        who = "distillation_loss"
        logits, top, idx, weights, keep, d = saved
        tau, reduction = ctx.meta
        V, K = logits.shape[-1], top.shape[-1]
        # The buffer is the caller's from here on, who may change it: a second backward pass fills one of its own (and does not mind the
        # change: what goes out counts its versions for itself).  So does one in a graph of its own: replayed without the forward pass, it
        # would find what the replay before or the caller left.
        made, ctx.made = ctx.made, None
        ready = made is not None and made >= 0 and made == L.capture_id(logits.device)
        d = d.data if ready else torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        z, ld = L.rows_2d(logits, V)
        g = L.plain_f32(g)
        L.launch("sx_distill_backward", logits.device, L.dtype_code(logits, who), z.shape[0], V, K, L.addr(z), ld, L.dtype_code(top, who), L.addr(top),
                 L.addr(idx), L.ids_flag(idx, who), tau, L.addr(weights), 1 if reduction == "mean" else 0, L.addr(keep) + 4, L.addr(keep), L.addr(g),
                 1 if reduction == "none" else 0, 1 if ready else 0, L.addr(d), V)
        return d


def distillation_loss(logits, top_logits, top_idx, *, temperature=1.0, weights=None, reduction="mean"):
    """Distillation of `logits` (..., V) from a teacher's top logits: `top_logits` (..., K) at the indices `top_idx` (..., K).

    loss = tau^2 * sum_k p_k (log p_k - log q_k) with p = softmax(top_logits / tau) over the row's K entries and q = softmax(logits /
    tau) over all V.  An entry whose index is outside [0, V) (-1 by convention) or whose logit is -inf is ignored; a row without any
    entry left or of weight 0 has loss 0 and gradient 0, whatever its logits hold.  `weights` (...): per row, or a mask.  reduction: "mean" =
    sum / max(sum weights, 1e-8), "sum", or "none" (a loss per row, weights included).  fp32 / bf16 logits, fp32 arithmetic, an fp32
    loss; the gradient has the logits' dtype and only goes to the logits.  Not differentiable twice.  Made for a teacher's top entries:
    beyond 512 of them the time grows with K^2 (512 rows: 0.17 ms with 1000, 8.5 ms with 8000)."""
    who = "distillation_loss"
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"Unknown reduction={reduction}")
    tau = float(temperature)
    if not 2.0 ** -126 <= tau < 2.0 ** 128:
        raise ValueError(f"{who}: temperature must be positive and finite (normal in 32 bits), got {temperature}")
    for t in (logits, top_logits, top_idx):
        _require_cuda(t, who)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{who}: logits must be (..., V), got {tuple(logits.shape)}")
    lead = tuple(logits.shape[:-1])
    if top_logits.dim() < 1 or top_logits.shape[-1] < 1 or tuple(top_logits.shape) != tuple(top_idx.shape) or tuple(top_logits.shape[:-1]) != lead:
        raise ValueError(f"{who}: top_logits and top_idx must both be {lead + ('K',)}, got {tuple(top_logits.shape)} / {tuple(top_idx.shape)}")
    if max(logits.shape[-1], top_logits.shape[-1]) > L.MAX_WIDTH:
        raise ValueError(f"{who}: rows of {logits.shape[-1]} logits with {top_logits.shape[-1]} of the teacher's are too long")
    if top_logits.device != logits.device or top_idx.device != logits.device:
        raise ValueError(f"{who}: logits, top_logits and top_idx must be on one device")
    L.dtype_code(logits, who), L.dtype_code(top_logits, who), L.ids_flag(top_idx, who)
    if weights is not None:
        if tuple(weights.shape) != lead:
            raise ValueError(f"{who}: weights must be {lead}, got {tuple(weights.shape)}")
        weights = L.plain_f32(weights if weights.device == logits.device else weights.to(logits.device))
    top, idx = L.packed(top_logits.detach() if top_logits.requires_grad else top_logits), L.packed(top_idx)
    if L.by_autograd(logits):
        return _DistillFn.apply(logits, top, idx, weights, tau, reduction)
    return _distill(logits, top, idx, weights, tau, reduction, False)[0]


def edge_weights(mask_np: np.ndarray, sigma_px: float = 3.0) -> np.ndarray:
    """Reference: solpex/losses.py:215-224.  Host-side (scipy), once per run."""
    from scipy.ndimage import binary_erosion, distance_transform_edt
    inside = np.asarray(mask_np).astype(bool)
    if not inside.any():
        return np.zeros_like(mask_np, dtype=np.float32)
    rim = inside & ~binary_erosion(inside, iterations=1, border_value=0)
    dist = distance_transform_edt(~rim)
    return (np.exp(-(dist ** 2) / (2.0 * sigma_px ** 2)) * inside).astype(np.float32)


def _err_sums(pred, target, mask, table):
    _require_cuda(pred, "masked metrics")
    B, Cc, H, W = pred.shape
    p = pred.detach()
    if p.dtype not in (torch.float32, torch.bfloat16):
        p = p.float()
    dt = L.SX_BF16 if p.dtype == torch.bfloat16 else L.SX_F32
    sb, sc, sh, sw = p.stride()
    tgt = target.detach().float().contiguous()
    m = _prep_mask(mask, B, H, W, "masked metrics")
    out = torch.zeros(3, dtype=torch.float32, device=p.device)
    if table is None:
        args = (None, None, None, None, None)
        denorm = 0
    else:
        args = table.c_args()
        denorm = 1
    L.check(L.lib().sx_masked_err_sums(dt, denorm, B, Cc, H, W, L.ptr(p), sb, sc, sh, sw, L.ptr(tgt), L.ptr(m), *args,
                                       L.ptr(out), L.stream_ptr()), "sx_masked_err_sums")
    return out


def mae_norm(pred, target, mask):
    """Reference: solpex/losses.py:226-227 (sum over channels / number of masked PIXELS)."""
    s = _err_sums(pred, target, mask, None)
    return s[0] / s[2].clamp_min(1e-8)


def batch_error_sums_ev(pred, target, mask, norm):
    """Reference: solpex/losses.py:229-253.  Returns (abs_sum, sq_sum, px) device scalars."""
    from .data import norm_table
    with torch.no_grad():
        s = _err_sums(pred, target, mask, norm_table(norm, pred.shape[1]))
        return s[0], s[1], s[2]
