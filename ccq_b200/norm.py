"""Layer norm, RMS norm and the gated RMS norm of a mixer block, forward and backward.

    h = x (+ residual);   n = (h - mean) / sqrt(var + eps)      (RMS: mean = 0, var = mean of h^2)
    y = n weight (+ bias);   gated: y = n weight gate sigmoid(gate)

The sums are fp32, the outputs are rounded once.  Every call goes to the sm_100a kernels in
``libccq_b200.so``; there is no CPU or eager fallback.
"""
from __future__ import annotations

import torch

from . import _lib
from .ops import _check_cuda, _dtype_code, _p, _stream


def _param(t, D, name):
    if t is None:
        return None
    if tuple(t.shape) != (D,):
        raise ValueError(f'{name} has shape {tuple(t.shape)}, expected {(D,)}')
    return t.detach().float().contiguous()


def _like(t, x, name):
    if t is None:
        return None
    if t.shape != x.shape:
        raise ValueError(f'{name} has shape {tuple(t.shape)}, expected {tuple(x.shape)}')
    return t.detach().to(x.dtype).contiguous()


class LayerNorm(torch.autograd.Function):
    """The three forms as one autograd function: returns (y, h or None)."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, gate, eps, form):
        _check_cuda(x, weight, bias, residual, gate)
        if x.ndim < 1 or x.shape[-1] < 1:
            raise ValueError(f'x must have a last axis of at least one element, got {tuple(x.shape)}')
        D = x.shape[-1]
        ctx.types = tuple(t.dtype if t is not None else None for t in (weight, bias, residual, gate))
        x = x.detach().contiguous()
        weight, bias = _param(weight, D, 'weight'), _param(bias, D, 'bias')
        residual, gate = _like(residual, x, 'residual'), _like(gate, x, 'gate')
        rows = x.numel() // D
        y = torch.empty_like(x)
        h = torch.empty_like(x) if residual is not None else None
        need = any(ctx.needs_input_grad[:5])
        stats = torch.empty(rows, 2, device=x.device, dtype=torch.float32) if need else None
        with torch.cuda.device(x.device):
            st = _lib.load().ccq_layer_norm_fwd(_dtype_code(x), form, rows, D, float(eps), _p(x), _p(residual),
                                                _p(weight), _p(bias), _p(gate), _p(y), _p(h), _p(stats),
                                                _stream(x.device))
        _lib.check(st)
        ctx.save_for_backward(x, residual, weight, bias, gate, stats)
        ctx.form = form
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    def backward(ctx, dy, dh):
        x, residual, weight, bias, gate, stats = ctx.saved_tensors
        D = x.shape[-1]
        rows = x.numel() // D
        dy = torch.zeros_like(x) if dy is None else dy.to(x.dtype).contiguous()
        dh = dh.to(x.dtype).contiguous() if dh is not None else None
        dx = torch.empty_like(x)
        dgate = torch.empty_like(gate) if gate is not None else None
        dw = torch.empty_like(weight) if weight is not None and ctx.needs_input_grad[1] else None
        db = torch.empty_like(bias) if bias is not None and ctx.needs_input_grad[2] else None
        lib = _lib.load()
        nbytes = lib.ccq_layer_norm_workspace_size(_lib.CCQ_OP_BWD, rows, D)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
        with torch.cuda.device(x.device):
            st = lib.ccq_layer_norm_bwd(_dtype_code(x), ctx.form, rows, D, _p(x), _p(residual), _p(weight), _p(bias),
                                        _p(gate), _p(stats), _p(dy), _p(dh), _p(dx), _p(dgate), _p(dw), _p(db), _p(ws),
                                        nbytes, _stream(x.device))
        _lib.check(st)
        tw, tb, tr, tg = ctx.types
        return (dx, dw.to(tw) if dw is not None else None, db.to(tb) if db is not None else None,
                dx.to(tr) if residual is not None else None, dgate.to(tg) if gate is not None else None, None, None)


def layer_norm(x, weight=None, bias=None, *, eps=1e-5, residual=None):
    """Layer norm over the last axis (at most 16384 elements).

    weight and bias: [D] or None.  With ``residual`` (x's shape) the norm reads h = x + residual, and the
    call returns (y, h): h, rounded to x's dtype, is the stream the next block adds to.
    """
    y, h = LayerNorm.apply(x, weight, bias, residual, None, eps, _lib.CCQ_NORM_LAYER)
    return (y, h) if residual is not None else y


def rms_norm(x, weight=None, *, eps=1e-5, residual=None):
    """``layer_norm`` without the mean and the bias."""
    y, h = LayerNorm.apply(x, weight, None, residual, None, eps, _lib.CCQ_NORM_RMS)
    return (y, h) if residual is not None else y


def gated_rms_norm(x, gate, weight=None, *, eps=1e-5):
    """rms_norm(x) * gate * sigmoid(gate): the norm a GDN layer applies to each head's output
    (ccq/gdn/layer.py, o_norm); gate has x's shape."""
    y, _ = LayerNorm.apply(x, weight, None, None, gate, eps, _lib.CCQ_NORM_RMS)
    return y
