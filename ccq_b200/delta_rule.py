"""Gated delta rule: the token mixer behind the cleaned queries, chunked with gradients and token by token.

Per (document, value head), with a state S [K, V] in fp32:

    S <- exp(g_t) S;   u_t = beta_t (v_t - S^T k_t);   S <- S + k_t u_t^T;   o_t = scale S^T q_t

``gated_delta_rule`` computes what the reference's GDN path takes from its backbone for training and
prefill (ccq/ops/ccq_gdn/fused_chunk.py:54), ``gated_delta_step`` what it takes for generation
(ccq/ops/ccq_gdn/fused_recurrent.py:66).  Every call goes to the sm_100a kernels in ``libccq_b200.so``;
there is no CPU or eager fallback.
"""
from __future__ import annotations

import torch

from . import _lib
from .ops import _check_cuda, _dtype_code, _p, _seqs, _state, _stream


def _inputs(q, k, v, g, beta):
    """The five inputs detached, contiguous and checked; k and v in q's dtype, g and beta in their own
    (another type than float32, bfloat16 or float16 is an error)."""
    if q.ndim != 4 or v.ndim != 4:
        raise ValueError(f'q, k must be [B, T, H, K] and v [B, T, HV, V], got {tuple(q.shape)} and {tuple(v.shape)}')
    B, T, H, K = q.shape
    HV, V = v.shape[2:]
    if tuple(k.shape) != (B, T, H, K):
        raise ValueError(f'k has shape {tuple(k.shape)}, expected {(B, T, H, K)}')
    if tuple(v.shape[:2]) != (B, T):
        raise ValueError(f'v has shape {tuple(v.shape)}, expected {(B, T)} + (HV, V)')
    for name, t in (('g', g), ('beta', beta)):
        if tuple(t.shape) != (B, T, HV):
            raise ValueError(f'{name} has shape {tuple(t.shape)}, expected {(B, T, HV)}')
    if HV % H != 0:
        raise ValueError(f'the number of value heads ({HV}) must be a multiple of the number of key heads ({H})')
    q, k, v, g, beta = (t.detach() for t in (q, k, v, g, beta))
    return _aligned(q), _aligned(k.to(q.dtype)), _aligned(v.to(q.dtype)), g.contiguous(), beta.contiguous()


def _aligned(t):
    """t contiguous and on a 16-byte boundary, as the tensor-core path reads it (a copy of a view that is not)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _workspace(op, q, v, N, cu, have_fwd=False):
    B, T, H, K = q.shape
    HV, V = v.shape[2:]
    flags = (_lib.CCQ_GDR_VARLEN if cu is not None else 0) | (_lib.CCQ_GDR_HAVE_FWD if have_fwd else 0)
    nbytes = _lib.load().ccq_gdr_workspace_size(op, _dtype_code(q), B, T, H, HV, K, V, N, flags)
    return (torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None), nbytes


def _head(q, k, v, g, beta, scale, cu, N, h0):
    """The arguments the C entry points share."""
    B, T, H, K = q.shape
    HV, V = v.shape[2:]
    return (_dtype_code(q), B, T, H, HV, K, V, _p(q), _p(k), _p(v), _dtype_code(g), _p(g), _dtype_code(beta), _p(beta),
            float(scale), _p(cu), N, _p(h0))


def _fwd_raw(q, k, v, g, beta, scale, h0, want_state, cu, N):
    o = torch.empty_like(v)
    state = torch.empty(N, *v.shape[2:3], q.shape[3], v.shape[3], device=q.device,
                        dtype=torch.float32) if want_state else None
    ws, nbytes = _workspace(_lib.CCQ_OP_FWD, q, v, N, cu)
    with torch.cuda.device(q.device):
        st = _lib.load().ccq_gdr_fwd(*_head(q, k, v, g, beta, scale, cu, N, h0), _p(o), _p(state), _p(ws), nbytes,
                                     _stream(q.device))
    _lib.check(st)
    return o, state, ws


class GatedDeltaRule(torch.autograd.Function):
    """``gated_delta_rule`` as an autograd function.  A call that needs gradients keeps the forward's workspace
    (540 bytes per token and value head on the tensor-core path); the backward recomputes the chunk states."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta, scale, initial_state, output_final_state, cu_seqlens):
        _check_cuda(q, k, v, g, beta, initial_state, cu_seqlens)
        types = (k.dtype, v.dtype)
        q, k, v, g, beta = _inputs(q, k, v, g, beta)
        cu, N = _seqs(q.shape[0], cu_seqlens, q.shape[1])
        h0 = _state(initial_state, (N, v.shape[2], q.shape[3], v.shape[3]))
        o, state, ws = _fwd_raw(q, k, v, g, beta, scale, h0, output_final_state, cu, N)
        ctx.save_for_backward(q, k, v, g, beta, h0, cu, ws if any(ctx.needs_input_grad) else None)
        ctx.scale, ctx.N, ctx.types = scale, N, types
        ctx.state_dtype = initial_state.dtype if initial_state is not None else None
        ctx.set_materialize_grads(False)
        return o, state

    @staticmethod
    def backward(ctx, do, dstate):
        q, k, v, g, beta, h0, cu, fwd_ws = ctx.saved_tensors
        do = torch.zeros_like(v) if do is None else _aligned(do.to(v.dtype))
        dstate = dstate.float().contiguous() if dstate is not None else None
        dq, dk, dv, dg, dbeta = (torch.empty_like(t) for t in (q, k, v, g, beta))
        dh0 = torch.empty_like(h0) if h0 is not None else None
        ws, nbytes = _workspace(_lib.CCQ_OP_BWD, q, v, ctx.N, cu, fwd_ws is not None)
        with torch.cuda.device(q.device):
            st = _lib.load().ccq_gdr_bwd_from(*_head(q, k, v, g, beta, ctx.scale, cu, ctx.N, h0), _p(do), _p(dstate),
                                              _p(dq), _p(dk), _p(dv), _p(dg), _p(dbeta), _p(dh0), _p(fwd_ws), _p(ws),
                                              nbytes, _stream(q.device))
        _lib.check(st)
        if dh0 is not None:
            dh0 = dh0.to(ctx.state_dtype)
        return dq, dk.to(ctx.types[0]), dv.to(ctx.types[1]), dg, dbeta, None, dh0, None, None


def gated_delta_rule(q, k, v, g, beta, *, scale=None, initial_state=None, output_final_state=False, cu_seqlens=None):
    """Gated delta rule over whole sequences, with gradients.

    q, k: [B, T, H, K]; v: [B, T, HV, V] with HV a multiple of H (value head h reads key head
    h // (HV // H)); g: [B, T, HV] log decay; beta: [B, T, HV] write strength; scale defaults to
    K ** -0.5; initial_state: [N, HV, K, V].  With ``cu_seqlens`` (B = 1) the T tokens hold N packed
    documents.  K is at most 256.  Returns (o [B, T, HV, V], final state [N, HV, K, V] fp32 or None).

    g and beta may be float32, bfloat16 or float16; their gradients come in the same types.  Inputs must be
    finite, except that g = -inf empties the state before its token.
    """
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    return GatedDeltaRule.apply(q, k, v, g, beta, scale, initial_state, bool(output_final_state), cu_seqlens)


def gated_delta_step(q, k, v, g, beta, state=None, *, scale=None, cu_seqlens=None, inplace=False):
    """The same recurrence token by token over a cache (inference; no autograd), meant for one token or
    a few per sequence.

    Returns (o, state after [N, HV, K, V] fp32).  ``inplace=True`` updates the given state, which must
    then be a contiguous float32 tensor.
    """
    _check_cuda(q, k, v, g, beta, state, cu_seqlens)
    q, k, v, g, beta = _inputs(q, k, v, g, beta)
    cu, N = _seqs(q.shape[0], cu_seqlens, q.shape[1])
    shape = (N, v.shape[2], q.shape[3], v.shape[3])
    if inplace and (state is None or state.dtype != torch.float32 or not state.is_contiguous()):
        raise ValueError('inplace needs a contiguous float32 state')
    h0 = _state(state, shape)
    out = h0 if inplace else torch.empty(shape, device=q.device, dtype=torch.float32)
    o = torch.empty_like(v)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    with torch.cuda.device(q.device):
        st = _lib.load().ccq_gdr_step(*_head(q, k, v, g, beta, scale, cu, N, h0), _p(out), _p(o), _stream(q.device))
    _lib.check(st)
    return o, (state if inplace else out)
