"""The operators together as a layer uses them: the mixer over whole sequences and over its cache, the example
block, and the GDN orchestrators on this framework's backbone.

The mixer is compared with its parts in float64 (oracle: l2norm, cleaning, gated delta rule) at the bfloat16 bar
of the cleaning operator, 2e-2 max-abs, relative to the largest output.
"""
import os
import sys

import numpy as np
import pytest
import torch

from oracle import ccq_oracle as O
from oracle import delta_rule_oracle as D

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'examples'))


@pytest.fixture(scope='module', autouse=True)
def _lib():
    if not torch.cuda.is_available():
        pytest.skip('no CUDA device')
    from ccq_b200 import _lib as L
    L.load()


def inputs(B, T, H, HV, K, V, dtype=torch.bfloat16, seed=0):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device='cuda')  # noqa: E731
    g = -torch.nn.functional.softplus(r(B, T, HV) - 2.0)
    return [t.to(dtype) for t in (r(B, T, H, K), r(B, T, H, K), r(B, T, HV, V), torch.rand(B, T, H, generator=gen, device='cuda'))] \
        + [g, torch.sigmoid(r(B, T, HV)).to(dtype)]


def expected(q, k, v, lam, g, beta):
    n = lambda t: t.detach().double().cpu().numpy()  # noqa: E731
    unit = lambda t: torch.nn.functional.normalize(t.double(), dim=-1, eps=1e-12).to(t.dtype)  # noqa: E731
    qn, kn = unit(q), unit(k)
    qc, _, _ = O.clean_read_fwd(n(qn), n(kn), n(lam))
    qc = torch.tensor(np.asarray(qc), device='cuda').to(q.dtype)
    return D.delta_rule(qc, kn, v, g, beta, q.shape[-1] ** -0.5)


@pytest.mark.parametrize('H,HV', [(2, 2), (2, 4)])
def test_mixer_against_its_parts(H, HV):
    import ccq_b200
    x = inputs(2, 150, H, HV, 128, 128)
    ref = expected(*x)
    o, cache = ccq_b200.ccq_gated_delta_rule(*x, output_cache=True)
    assert (o.double() - ref['o']).abs().max() <= 2e-2 * max(1.0, ref['o'].abs().max().item())
    assert cache[3] == 150 and cache[0].shape == (2, HV, 128, 128) and cache[1].shape == (2, H, 128, 128)
    assert (cache[0].double() - ref['state']).abs().max() <= 2e-2 * max(1.0, ref['state'].abs().max().item())


def test_generation_follows_prefill():
    import ccq_b200
    x = inputs(3, 90, 2, 4, 128, 64, seed=2)
    whole, end = ccq_b200.ccq_gated_delta_rule(*x, output_cache=True)
    _, cache = ccq_b200.ccq_gated_delta_rule(*(t[:, :70] for t in x), output_cache=True)
    for t in (70, 71, 72):
        state = cache[0]
        o, cache = ccq_b200.ccq_gated_delta_step(*(y[:, t:t + 1] for y in x), cache)
        assert cache[0] is state and cache[3] == t + 1
        assert (o - whole[:, t:t + 1]).abs().max() <= 2e-2
    o, cache = ccq_b200.ccq_gated_delta_step(*(y[:, 73:] for y in x), cache, inplace=False)  # several drafted tokens
    assert cache[0] is not state and (o - whole[:, 73:]).abs().max() <= 2e-2
    assert (cache[0] - end[0]).abs().max() <= 2e-2 * max(1.0, end[0].abs().max().item())


def test_gradients_reach_every_input():
    import ccq_b200
    x = [t.requires_grad_(True) for t in inputs(1, 100, 2, 2, 128, 128, seed=3)]
    o, _ = ccq_b200.ccq_gated_delta_rule(*x)
    grads = torch.autograd.grad(o.float().square().sum(), x)
    for t, d in zip(x, grads):
        assert d.shape == t.shape and d.dtype == t.dtype and torch.isfinite(d).all() and (d != 0).any()


def test_example_block():
    import gdn_block
    torch.manual_seed(0)
    block = gdn_block.GDNBlock(256, 2, 4).cuda()
    losses = gdn_block.train(block, steps=4, T=130, width=256)
    assert all(np.isfinite(losses)) and losses[-1] < losses[0]
    assert gdn_block.generate(block, prompt=70, tokens=3, width=256) <= 2e-2


def test_orchestrators_on_the_b200_backbone():
    """What install(backbone='b200') routes the two GDN orchestrators to, without the reference installed."""
    import ccq_b200
    from ccq_b200 import integration
    q, k, v, lam, g, beta = inputs(2, 100, 2, 2, 128, 128, seed=4)
    want, cache = ccq_b200.ccq_gated_delta_rule(q, k, v, lam, g, beta, output_cache=True)
    integration._backbone = 'b200'
    try:
        for f in (integration.fused_chunk_ccq_gdn, integration.chunk_ccq_gdn):
            o, S, cov, mean = f(q, k, v, lam, g, beta, output_final_state=True, use_qk_l2norm_in_kernel=True)
            assert torch.equal(o, want) and torch.equal(S, cache[0]) and torch.equal(cov, cache[1])
            o, S, cov, mean = f(q, k, v, lam, g, beta, use_qk_l2norm_in_kernel=True, enable_ccq=False)
            assert o.shape == want.shape and cov is None and torch.isfinite(o).all()
        with pytest.raises(ValueError, match='cp_context'):
            integration.chunk_ccq_gdn(q, k, v, lam, g, beta, transpose_state_layout=True)
    finally:
        integration._backbone = 'fla'
    with pytest.raises(ValueError, match='backbone'):
        integration.install(backbone='other')


def test_backward_without_the_forward_workspace():
    """ccq_gdr_bwd forms the inverses and scores again and gives the same bits as the call that is handed them."""
    from ccq_b200 import _lib
    from ccq_b200 import delta_rule as R
    lib = _lib.load()
    q, k, v, _, g, beta = inputs(2, 200, 2, 4, 128, 128, seed=5)
    q, k = (torch.nn.functional.normalize(t.float(), dim=-1).bfloat16() for t in (q, k))
    do = torch.randn_like(v)
    head = R._head(q, k, v, g, beta, 0.1, None, 2, None)
    stream = torch.cuda.current_stream().cuda_stream
    fws, n = R._workspace(_lib.CCQ_OP_FWD, q, v, 2, None)
    o = torch.empty_like(v)
    _lib.check(lib.ccq_gdr_fwd(*head, o.data_ptr(), None, fws.data_ptr(), n, stream))
    outs = []
    for have in (False, True):
        d = [torch.empty_like(t) for t in (q, k, v, g, beta)]
        ws, n = R._workspace(_lib.CCQ_OP_BWD, q, v, 2, None, have)
        args = (*head, do.data_ptr(), None, *(t.data_ptr() for t in d), None)
        if have:
            st = lib.ccq_gdr_bwd_from(*args, fws.data_ptr(), ws.data_ptr(), n, stream)
        else:
            st = lib.ccq_gdr_bwd(*args, ws.data_ptr(), n, stream)
        _lib.check(st)
        outs.append(d)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*outs))
