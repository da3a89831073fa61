"""Distillation from a teacher's top logits: class or codebook scores trained per pixel.

A semantic scene renders class scores per pixel and trains them against a 2-D teacher. Whole
distributions of every view do not fit, so the teacher's side keeps the k largest logits of each
pixel, their classes and the log-sum-exp of all (``top_logits``); ``distill_loss`` takes the
divergence of the student's softmax from them, with its gradient. No counterpart in the reference,
whose losses are photometric. One read of the logits per call; there is no CPU fallback.
"""

from __future__ import annotations

import contextlib
import ctypes
import math
import operator

import torch
from torch.autograd.function import once_differentiable

from splax_b200 import _lib

MAX_CLASSES = 262144  # SPLAX_DISTILL_MAX_CLASSES
MAX_K = 128  # SPLAX_DISTILL_MAX_K
WORKSPACE = 65536  # SPLAX_DISTILL_WORKSPACE, bytes

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _check_logits(logits: torch.Tensor, temperature: float) -> float:
    if logits.dtype not in _DTYPES:
        raise ValueError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= MAX_CLASSES:
        raise ValueError(f"logits {tuple(logits.shape)} must have 1 to {MAX_CLASSES} classes on "
                         "their last axis")
    t = float(temperature)
    if not 1e-30 <= t <= 1e30:
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    return t


def _rows(logits: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """(tensor, rows, row stride) with the classes contiguous; a copy only where the strides do
    not give that (rows of a wider array are taken in place)."""
    classes = logits.shape[-1]
    flat = logits.detach()
    if flat.dim() != 2:
        flat = flat.reshape(-1, classes)
    rows = flat.shape[0]
    stride, inner = flat.stride()
    if (classes > 1 and inner != 1) or (rows > 1 and stride < classes):
        flat = flat.contiguous()
        stride = classes
    return flat, rows, (stride if rows > 1 else classes)


def _on(dev: torch.device):
    """The device as the current one; nothing to do where it is."""
    if torch.cuda.current_device() == dev.index:
        return contextlib.nullcontext()
    return torch.cuda.device(dev)


def _stream(dev: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(dev.index)


def top_logits(logits: torch.Tensor, k: int, *, temperature: float = 1.0
               ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``k`` largest of the (..., C) logits along the last axis: ``values`` (..., k) in their
    type, ``ids`` (..., k) int32 and ``lse`` (...) float32, the log-sum-exp of
    ``logits / temperature`` over all C classes. Largest first, equal values in ascending class
    order; NaN ranks above every number. A row that holds a NaN or +inf has no softmax: its
    ``lse`` is NaN, which a loss shows. Not differentiable (a teacher's side). 1 <= k <=
    min(C, 128), C <= 262144; the rows may be strided."""
    t = _check_logits(logits, temperature)
    classes, k = logits.shape[-1], operator.index(k)
    if not 1 <= k <= min(classes, MAX_K):
        raise ValueError(f"k={k} must be between 1 and min({classes} classes, {MAX_K})")
    dev = _lib.require_cuda(logits)
    with _on(dev):
        z, rows, stride = _rows(logits)
        lead = logits.shape[:-1]
        values = torch.empty((*lead, k), device=dev, dtype=logits.dtype)
        ids = torch.empty((*lead, k), device=dev, dtype=torch.int32)
        lse = torch.empty(lead, device=dev, dtype=torch.float32)
        rc = _lib.load().splax_top_logits(
            z.data_ptr(), _DTYPES[z.dtype], rows, classes, stride, k, t, values.data_ptr(),
            ids.data_ptr(), lse.data_ptr(), _stream(dev))
    if rc:
        _lib.check(rc)
    return values, ids, lse


def _capture_id(dev: torch.device) -> int:
    if not torch.cuda.is_current_stream_capturing():
        return 0
    out = ctypes.c_uint64(0)
    _lib.check(_lib.load().splax_capture_id(_stream(dev), ctypes.byref(out)))
    return out.value


def _address(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _fp32(t: torch.Tensor | None) -> torch.Tensor | None:
    return None if t is None else t.detach().to(torch.float32).contiguous()


class _DistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_values, top_ids, top_lse, weights, temperature, denom, trains):
        dev = logits.device
        lib = _lib.load()
        with _on(dev):
            z, ctx.rows, _ = _rows(logits)
            v, i = top_values.detach().contiguous(), top_ids.detach().contiguous()
            saved = (z, v, i, _fp32(top_lse), _fp32(weights))
            ctx.scalars = (temperature, denom)
            args = _DistillFn._args(ctx, *saved)
            loss = torch.empty((), device=dev, dtype=torch.float32)
            work = torch.empty(WORKSPACE, device=dev, dtype=torch.uint8)
            # a training step takes the gradient next: compute it with the loss from one read of
            # the logits (for a unit cotangent; backward scales it)
            ctx.grad = None
            if trains:
                ctx.grad = torch.empty(logits.shape, device=dev, dtype=logits.dtype)
                rc = lib.splax_distill_loss_and_grad(*args, work.data_ptr(), loss.data_ptr(),
                                                     ctx.grad.data_ptr(), _stream(dev))
                ctx.capture = _capture_id(dev)
            else:
                rc = lib.splax_distill_loss(*args, work.data_ptr(), loss.data_ptr(), _stream(dev))
        if rc:
            _lib.check(rc)
        ctx.save_for_backward(*saved)
        ctx.shape = logits.shape
        return loss

    @staticmethod
    def _args(ctx, z, v, i, lse, w):
        """What the library's calls have in common."""
        return (z.data_ptr(), _DTYPES[z.dtype], ctx.rows, z.shape[1],
                z.stride(0) if ctx.rows > 1 else z.shape[1], v.data_ptr(), _DTYPES[v.dtype],
                i.data_ptr(), 64 if i.dtype == torch.int64 else 32, _address(lse), v.shape[-1],
                _address(w), *ctx.scalars)

    @staticmethod
    def backward(ctx, v_loss):
        if torch.is_grad_enabled():  # a graph of the backward is asked for: marked as having none
            g = _DistillFn._again(ctx, v_loss)
            g = g[0] if isinstance(g, tuple) else g
        else:
            g = _DistillFn._gradient(ctx, v_loss)
        return g, None, None, None, None, None, None, None

    @staticmethod
    def _gradient(ctx, v_loss):
        saved = ctx.saved_tensors  # refuses logits that were changed since
        z = saved[0]
        dev = z.device
        lib = _lib.load()
        cot = v_loss.detach()
        if cot.dtype != torch.float32:
            cot = cot.to(torch.float32)
        # The gradient of the forward pass is handed out once, for a unit cotangent as it stands. For
        # another, fp32 is scaled in place; 16 bits, which may have lost what the cotangent would
        # have lifted into their range, are computed again. So is the gradient of a later backward,
        # or of one that is replayed apart from its forward.
        g, ctx.grad = ctx.grad, None
        with _on(dev):
            if g is None or ctx.capture != _capture_id(dev):
                g = torch.empty(ctx.shape, device=dev, dtype=z.dtype)
                rc = lib.splax_distill_loss_bwd(*_DistillFn._args(ctx, *saved), cot.data_ptr(),
                                                g.data_ptr(), _stream(dev))
            elif g.dtype == torch.float32:
                rc = lib.splax_distill_scale_grad(g.data_ptr(), _DTYPES[g.dtype], g.numel(),
                                                  cot.data_ptr(), _stream(dev))
            else:
                rc = lib.splax_distill_rescale_grad(*_DistillFn._args(ctx, *saved),
                                                    cot.data_ptr(), g.data_ptr(), _stream(dev))
        if rc:
            _lib.check(rc)
        return g

    _again = staticmethod(once_differentiable(_gradient.__func__))


def distill_loss(logits: torch.Tensor, top_values: torch.Tensor, top_ids: torch.Tensor,
                 top_lse: torch.Tensor | None = None, *, temperature: float = 1.0,
                 weights: torch.Tensor | None = None, denom: float | None = None
                 ) -> torch.Tensor:
    """Divergence of ``softmax(logits / temperature)`` from a teacher's distribution given by its
    top logits, as a 0-d tensor: ``temperature**2 * sum_r weights_r KL_r / denom``.

    ``logits`` (..., C) are the student's (fp32, bf16 or fp16; the rows may be strided);
    ``top_values`` and ``top_ids`` (..., K) the teacher's logits and their classes (int32 or
    int64), K <= 128. An entry whose class lies outside [0, C) is empty. Without ``top_lse`` the
    entries are renormalised among themselves; with it (``top_logits`` at the same temperature)
    they keep their probabilities and the teacher's remaining mass is compared with the student's
    mass on all classes that no entry names. ``weights`` (...) scale the rows; a row adds nothing
    where its weight is 0, where all its entries are empty or all its logits are -inf. ``denom``
    defaults to the number of rows (of none it has to be given); pass the global one when each rank holds a shard, and fold a
    constant factor of the loss into it: a backward whose cotangent is not one costs a pass over
    the gradient, or in 16 bits another computation of it. The gradient is in the logits' type,
    rounded with the cotangent in it: for fp16 scale the loss, or choose ``denom``, so that it does
    not vanish there. Logits of any finite size count by their differences, in the loss in 64 bits.
    Differentiable once, with respect to the logits; the teacher and the weights
    get no gradient."""
    t = _check_logits(logits, temperature)
    lead = logits.shape[:-1]
    if top_values.dtype not in _DTYPES:
        raise ValueError("top_values must be float32, bfloat16 or float16, got "
                         f"{top_values.dtype}")
    if top_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"top_ids must be int32 or int64, got {top_ids.dtype}")
    if top_values.shape != top_ids.shape or top_values.shape[:-1] != lead or \
            top_values.dim() != logits.dim() or not 1 <= top_values.shape[-1] <= MAX_K:
        raise ValueError(f"top_values {tuple(top_values.shape)} and top_ids "
                         f"{tuple(top_ids.shape)} must be {tuple(lead)} + (K,), 1 <= K <= {MAX_K}")
    for name, x in (("top_lse", top_lse), ("weights", weights)):
        if x is not None and (x.shape != lead or not x.dtype.is_floating_point):
            raise ValueError(f"{name} must be floating-point of shape {tuple(lead)}, got "
                             f"{x.dtype} {tuple(x.shape)}")
    d = float(math.prod(lead) if denom is None else denom)
    if not 1e-30 <= d <= 1e30:
        raise ValueError(f"denom must be positive and finite, got {d}")
    _lib.require_cuda(logits, top_values, top_ids, top_lse, weights)
    return _DistillFn.apply(logits, top_values, top_ids, top_lse, weights, t, d,
                            logits.requires_grad and torch.is_grad_enabled())
