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
from ._call import cuda_index, first_derivative, invoke, ptr, wants_grad, written
from .ops import _dtype_code, _seqs, _state


def _check(q, k, v, g, beta):
    if q.ndim != 4 or v.ndim != 4:
        raise ValueError(f'q, k must be [B, T, H, K] and v [B, T, HV, V], got {tuple(q.shape)} and {tuple(v.shape)}')
    B, T, H, K = q.shape
    HV = v.shape[2]
    if k.shape != q.shape:
        raise ValueError(f'k has shape {tuple(k.shape)}, expected {(B, T, H, K)}')
    if v.shape[0] != B or v.shape[1] != T:
        raise ValueError(f'v has shape {tuple(v.shape)}, expected {(B, T)} + (HV, V)')
    gates = (B, T, HV)
    if g.shape != gates:
        raise ValueError(f'g has shape {tuple(g.shape)}, expected {gates}')
    if beta.shape != gates:
        raise ValueError(f'beta has shape {tuple(beta.shape)}, expected {gates}')
    if HV % H != 0:
        raise ValueError(f'the number of value heads ({HV}) must be a multiple of the number of key heads ({H})')


def _inputs(q, k, v, g, beta):
    """The five inputs checked, contiguous and aligned; k and v in q's dtype, g and beta in their own
    (another type than float32, bfloat16 or float16 is an error)."""
    _check(q, k, v, g, beta)
    dt = q.dtype
    return (_aligned(q), _aligned(k if k.dtype == dt else k.to(dt)), _aligned(v if v.dtype == dt else v.to(dt)),
            g.contiguous(), beta.contiguous())


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
    return (_dtype_code(q), B, T, H, HV, K, V, q.data_ptr(), k.data_ptr(), v.data_ptr(), _dtype_code(g), g.data_ptr(),
            _dtype_code(beta), beta.data_ptr(), scale, ptr(cu), N, ptr(h0))


def _forward(q, k, v, g, beta, scale, initial_state, output_final_state, cu_seqlens):
    """One ccq_gdr_fwd call; returns (o, final state or None, what a backward needs).  Only the tensor-core path's
    workspace is of use to a backward; the exact path's is let go."""
    index = cuda_index(q, k, v, g, beta, initial_state, cu_seqlens)
    q, k, v, g, beta = _inputs(q, k, v, g, beta)
    cu, N = _seqs(q.shape[0], cu_seqlens, q.shape[1])
    shape = (N, v.shape[2], q.shape[3], v.shape[3])
    h0 = _state(initial_state, shape)
    o = torch.empty_like(v)
    state = torch.empty(shape, device=q.device, dtype=torch.float32) if output_final_state else None
    ws, nbytes = _workspace(_lib.CCQ_OP_FWD, q, v, N, cu)
    lib = _lib.load()
    invoke(lib.ccq_gdr_fwd, index, *_head(q, k, v, g, beta, scale, cu, N, h0), o.data_ptr(), ptr(state), ptr(ws), nbytes)
    if lib.ccq_last_path() != _lib.CCQ_PATH_TCGEN05:
        ws = None
    return o, state, (q, k, v, g, beta, h0, cu, ws)


class GatedDeltaRule(torch.autograd.Function):
    """``gated_delta_rule`` as an autograd function.  A call that needs gradients keeps the forward's workspace
    (540 bytes per token and value head on the tensor-core path, 800 in float16); the backward recomputes the chunk states."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta, scale, initial_state, output_final_state, cu_seqlens):
        ctx.types = (k.dtype, v.dtype)
        ctx.state_dtype = initial_state.dtype if initial_state is not None else None
        o, state, kept = _forward(q, k, v, g, beta, scale, initial_state, output_final_state, cu_seqlens)
        ctx.save_for_backward(*kept)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, state

    @staticmethod
    @first_derivative
    def backward(ctx, do, dstate):
        q, k, v, g, beta, h0, cu, fwd_ws = ctx.saved_tensors
        do = torch.zeros_like(v) if do is None else _aligned(do if do.dtype == v.dtype else do.to(v.dtype))
        dstate = dstate.float().contiguous() if dstate is not None else None
        dq, dk, dv, dg, dbeta = (torch.empty_like(t) for t in (q, k, v, g, beta))
        dh0 = torch.empty_like(h0) if h0 is not None else None
        N = cu.numel() - 1 if cu is not None else q.shape[0]
        ws, nbytes = _workspace(_lib.CCQ_OP_BWD, q, v, N, cu, fwd_ws is not None)
        invoke(_lib.load().ccq_gdr_bwd_from, q.device.index, *_head(q, k, v, g, beta, ctx.scale, cu, N, h0), do.data_ptr(),
               ptr(dstate), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dg.data_ptr(), dbeta.data_ptr(), ptr(dh0),
               ptr(fwd_ws), ptr(ws), nbytes)
        if dh0 is not None:
            dh0 = dh0.to(ctx.state_dtype)
        return dq, dk.to(ctx.types[0]), dv.to(ctx.types[1]), dg, dbeta, None, dh0, None, None


def gated_delta_rule(q, k, v, g, beta, *, scale=None, initial_state=None, output_final_state=False, cu_seqlens=None):
    """Gated delta rule over whole sequences, with gradients (of first order, in reverse mode; others raise).

    q, k: [B, T, H, K]; v: [B, T, HV, V] with HV a multiple of H (value head h reads key head
    h // (HV // H)); g: [B, T, HV] log decay; beta: [B, T, HV] write strength; scale defaults to
    K ** -0.5; initial_state: [N, HV, K, V].  With ``cu_seqlens`` (B = 1) the T tokens hold N packed
    documents.  K is at most 256.  Returns (o [B, T, HV, V], final state [N, HV, K, V] fp32 or None).

    g and beta may be float32, bfloat16 or float16; their gradients come in the same types.  Inputs must be
    finite, except that g = -inf empties the state before its token.

    16-bit inputs with K a multiple of 8 up to 128 and V a multiple of 8 run on the tensor cores, where the
    state and its gradient keep fp32 accuracy (about 4e-6) and dq, dk and dbeta that of the 16-bit type;
    everything else, fp32 inputs among it, runs in fp32 on the CUDA cores.  k and v are taken in q's dtype.  States
    and their gradients may have any size that fp32 holds, with float16 inputs too; what is returned in float16
    has that type's range.
    """
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if wants_grad(q, k, v, g, beta, initial_state):
        return GatedDeltaRule.apply(q, k, v, g, beta, scale, initial_state, bool(output_final_state), cu_seqlens)
    return _forward(q, k, v, g, beta, scale, initial_state, output_final_state, cu_seqlens)[:2]


def check_step(q, k, v, g, beta, state, inplace):
    """Raises what ``gated_delta_step`` of a dense batch would, before anything is written."""
    cuda_index(q, k, v, g, beta, state)
    _check(q, k, v, g, beta)
    for t in (q, g, beta):
        _dtype_code(t)
    _check_state(state, (q.shape[0], v.shape[2], q.shape[3], v.shape[3]), inplace)


def _check_state(state, shape, inplace):
    if inplace and (state is None or state.dtype != torch.float32 or not state.is_contiguous()):
        raise ValueError('inplace needs a contiguous float32 state')
    if state is not None and tuple(state.shape) != shape:
        raise ValueError(f'state has shape {tuple(state.shape)}, expected {shape}')


def gated_delta_step(q, k, v, g, beta, state=None, *, scale=None, cu_seqlens=None, inplace=False):
    """The same recurrence token by token over a cache (inference; no autograd), meant for one token or
    a few per sequence.

    Returns (o, state after [N, HV, K, V] fp32).  ``inplace=True`` updates the given state, which must
    then be a contiguous float32 tensor.
    """
    index = cuda_index(q, k, v, g, beta, state, cu_seqlens)
    q, k, v, g, beta = _inputs(q, k, v, g, beta)
    cu, N = _seqs(q.shape[0], cu_seqlens, q.shape[1])
    shape = (N, v.shape[2], q.shape[3], v.shape[3])
    _check_state(state, shape, inplace)
    h0 = state if inplace else _state(state, shape)  # in place it is as the kernel takes it
    out = state if inplace else torch.empty(shape, device=q.device, dtype=torch.float32)
    o = torch.empty_like(v, requires_grad=False)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    invoke(_lib.load().ccq_gdr_step, index, *_head(q, k, v, g, beta, scale, cu, N, h0), out.data_ptr(), o.data_ptr())
    if inplace:
        written(out)
    return o, out
