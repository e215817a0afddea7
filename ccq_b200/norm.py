"""Layer norm, RMS norm and the gated RMS norm of a mixer block, forward and backward.

    h = x (+ residual);   n = (h - mean) / sqrt(var + eps)      (RMS: mean = 0, var = mean of h^2)
    y = n weight (+ bias);   gated: y = n weight gate sigmoid(gate)

The sums are fp32, the outputs are rounded once.  Gradients are of first order, in reverse mode; others raise.  Every call goes to the sm_100a kernels in
``libccq_b200.so``; there is no CPU or eager fallback.
"""
from __future__ import annotations

import torch

from . import _lib
from ._call import cuda_index, first_derivative, invoke, ptr, wants_grad
from .ops import _dtype_code


def _param(t, D, name):
    if t is None:
        return None
    if t.shape != (D,):
        raise ValueError(f'{name} has shape {tuple(t.shape)}, expected {(D,)}')
    return t.contiguous() if t.dtype == torch.float32 else t.float()


def _like(t, x, name):
    if t is None:
        return None
    if t.shape != x.shape:
        raise ValueError(f'{name} has shape {tuple(t.shape)}, expected {tuple(x.shape)}')
    return (t if t.dtype == x.dtype else t.to(x.dtype)).contiguous()


def _forward(x, weight, bias, residual, gate, eps, form, need_stats):
    """One ccq_layer_norm_fwd call; returns (y, h or None, what a backward needs)."""
    index = cuda_index(x, weight, bias, residual, gate)
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f'x must have a last axis of at least one element, got {tuple(x.shape)}')
    D = x.shape[-1]
    x = x.contiguous()
    weight, bias = _param(weight, D, 'weight'), _param(bias, D, 'bias')
    residual, gate = _like(residual, x, 'residual'), _like(gate, x, 'gate')
    rows = x.numel() // D
    y = torch.empty_like(x)
    h = torch.empty_like(x) if residual is not None else None
    stats = torch.empty(rows, 2, device=x.device, dtype=torch.float32) if need_stats else None
    invoke(_lib.load().ccq_layer_norm_fwd, index, _dtype_code(x), form, rows, D, eps, x.data_ptr(), ptr(residual),
           ptr(weight), ptr(bias), ptr(gate), y.data_ptr(), ptr(h), ptr(stats))
    return y, h, (x, residual, weight, bias, gate, stats)


class LayerNorm(torch.autograd.Function):
    """The three forms as one autograd function: returns (y, h or None)."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, gate, eps, form):
        ctx.types = tuple(t.dtype if t is not None else None for t in (weight, bias, residual, gate))
        y, h, kept = _forward(x, weight, bias, residual, gate, eps, form, True)
        ctx.save_for_backward(*kept)
        ctx.form = form
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @first_derivative
    def backward(ctx, dy, dh):
        x, residual, weight, bias, gate, stats = ctx.saved_tensors
        D = x.shape[-1]
        rows = x.numel() // D
        dy = torch.zeros_like(x) if dy is None else _like(dy, x, 'the gradient of y')
        dh = _like(dh, x, 'the gradient of h')
        dx = torch.empty_like(x)
        dgate = torch.empty_like(gate) if gate is not None else None
        dw = torch.empty_like(weight) if weight is not None and ctx.needs_input_grad[1] else None
        db = torch.empty_like(bias) if bias is not None and ctx.needs_input_grad[2] else None
        lib = _lib.load()
        nbytes = lib.ccq_layer_norm_workspace_size(_lib.CCQ_OP_BWD, rows, D)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
        invoke(lib.ccq_layer_norm_bwd, x.device.index, _dtype_code(x), ctx.form, rows, D, x.data_ptr(), ptr(residual),
               ptr(weight), ptr(bias), ptr(gate), stats.data_ptr(), dy.data_ptr(), ptr(dh), dx.data_ptr(), ptr(dgate),
               ptr(dw), ptr(db), ptr(ws), nbytes)
        tw, tb, tr, tg = ctx.types
        return (dx, dw.to(tw) if dw is not None else None, db.to(tb) if db is not None else None,
                dx.to(tr) if residual is not None else None, dgate.to(tg) if gate is not None else None, None, None)


def _norm(x, weight, bias, residual, gate, eps, form):
    if residual is not None and residual.dtype != x.dtype and x.dtype in (torch.bfloat16, torch.float16) \
            and torch.promote_types(x.dtype, residual.dtype) != x.dtype:
        # a residual stream that x's type cannot hold is not rounded to it
        y, h = _norm(x.float(), weight, bias, residual, gate, eps, form)
        return y.to(x.dtype), h
    if wants_grad(x, weight, bias, residual, gate):
        return LayerNorm.apply(x, weight, bias, residual, gate, float(eps), form)
    return _forward(x, weight, bias, residual, gate, float(eps), form, False)[:2]


def layer_norm(x, weight=None, bias=None, *, eps=1e-5, residual=None):
    """Layer norm over the last axis (at most 16384 elements).

    weight and bias: [D] or None.  With ``residual`` (x's shape) the norm reads h = x + residual, and the
    call returns (y, h): h is the stream the next block adds to.  y has x's dtype, and so has h unless residual's
    is wider: a float32 stream stays one, and the call then runs in float32 (its casts are passes of their own).
    """
    y, h = _norm(x, weight, bias, residual, None, eps, _lib.CCQ_NORM_LAYER)
    return (y, h) if residual is not None else y


def rms_norm(x, weight=None, *, eps=1e-5, residual=None):
    """``layer_norm`` without the mean and the bias."""
    y, h = _norm(x, weight, None, residual, None, eps, _lib.CCQ_NORM_RMS)
    return (y, h) if residual is not None else y


def gated_rms_norm(x, gate, weight=None, *, eps=1e-5):
    """rms_norm(x) * gate * sigmoid(gate): the norm a GDN layer applies to each head's output
    (ccq/gdn/layer.py, o_norm); gate has x's shape and is taken in its dtype."""
    return _norm(x, weight, None, None, gate, eps, _lib.CCQ_NORM_RMS)[0]
