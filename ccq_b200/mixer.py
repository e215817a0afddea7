"""The CCQ gated-delta-rule mixer end to end on this framework's kernels: l2norm of q and k, the cleaning read, the
gated delta rule, over whole sequences (training, prefill) and token by token over the generation cache.

The cache is the reference's 4-tuple (ccq/gdn/layer.py:318-336, :394-400): (recurrent state [N, HV, K, V],
covariance state [N, H, K, K], mean state [N, H, K] or None, position offset), the states fp32.  The offset is an
int, the position all of them have reached; after packed documents, which end at positions of their own, it is
a tensor [N].  The cleaning read divides by one position for the whole call, so such a cache is continued
document by document: (state[n:n + 1], cov[n:n + 1], mean[n:n + 1], int(offset[n])).
"""
from __future__ import annotations

import torch

from .delta_rule import check_step, gated_delta_rule, gated_delta_step
from .ops import decode_step_l2norm, fused_ccq_clean_read_l2norm


def _unpack(cache):
    if cache is None:
        return None, None, None, 0
    if isinstance(cache[3], torch.Tensor) and cache[3].numel() != 1:
        raise ValueError(f'the cache holds {cache[3].numel()} documents that ended at positions of their own, and one call has one '
                         'position: continue them one by one, with the rows of the states and int(offset) of each')
    return cache


def _after(offset, T, cu_seqlens):
    """The position offset after T tokens; one for each of several packed documents."""
    if cu_seqlens is None or cu_seqlens.numel() == 2:
        return offset + T
    return offset + (cu_seqlens[1:] - cu_seqlens[:-1]).to(torch.int64)


def ccq_gated_delta_rule(q, k, v, lambda_h, g, beta, *, scale=None, cache=None, output_cache=False, cu_seqlens=None,
                         subtract_mean=True):
    """What the reference's fused_chunk path computes for a GDN layer (ccq/ops/ccq_gdn/fused_chunk.py:16-59 with
    the l2norm on), with gradients.

    q, k: [B, T, H, K] raw; v: [B, T, HV, V]; lambda_h: as ``fused_ccq_clean_read``; g, beta: [B, T, HV].
    Returns (o [B, T, HV, V], the cache after the last token or None).
    """
    state, cov, mean, offset = _unpack(cache)
    q_clean, k_norm, cov, mean = fused_ccq_clean_read_l2norm(
        q, k, lambda_h, position_offset=offset, initial_cov_state=cov,
        initial_mean_state=mean if subtract_mean else None, output_final_state=output_cache,
        subtract_mean=subtract_mean, cu_seqlens=cu_seqlens)
    o, state = gated_delta_rule(q_clean, k_norm, v, g, beta, scale=scale, initial_state=state,
                                output_final_state=output_cache, cu_seqlens=cu_seqlens)
    return o, (state, cov, mean, _after(offset, q.shape[1], cu_seqlens)) if output_cache else None


def ccq_gated_delta_step(q, k, v, lambda_h, g, beta, cache, *, scale=None, subtract_mean=True, inplace=True):
    """The same for one token, or a few, of each sequence over its cache (inference; no autograd; K a
    multiple of 4).  ``inplace=True`` updates the cache's tensors.  Returns (o, cache after).
    """
    state, cov, mean, offset = _unpack(cache)
    inplace = inplace and cache is not None
    check_step(q, k, v, g, beta, state, inplace)  # the cleaning read writes its states before the rule is called
    q_clean, k_norm, cov, mean = decode_step_l2norm(q, k, lambda_h, cov, mean, position_offset=offset,
                                                    subtract_mean=subtract_mean, inplace=inplace)
    o, state = gated_delta_step(q_clean, k_norm, v, g, beta, state, scale=scale, inplace=inplace)
    return o, (state, cov, mean, offset + q.shape[1])
