"""The mixer's generation cache after packed documents: every document goes on from its own position.

Compared with one pass over the whole document at the bar of the mixer's other tests, 2e-2 max-abs (the cleaning
operator's bfloat16 bar)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
LENS = [70, 1, 0, 33, 128]


@pytest.fixture(scope='module', autouse=True)
def _lib():
    if not torch.cuda.is_available():
        pytest.skip('no CUDA device')
    from ccq_b200 import _lib as L
    L.load()


def inputs(T, H=2, HV=4, K=128, V=64, seed=0):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device='cuda')  # noqa: E731
    x = [r(1, T, H, K), r(1, T, H, K), r(1, T, HV, V), torch.rand(1, T, H, generator=gen, device='cuda')]
    return [t.bfloat16() for t in x] + [-torch.nn.functional.softplus(r(1, T, HV) - 2.0), r(1, T, HV).sigmoid().bfloat16()]


def packed(n_more, subtract_mean=True):
    """Documents of LENS + n_more tokens: whole, and the cache after the first LENS of each, packed."""
    import ccq_b200
    docs = [inputs(n + n_more, seed=i) for i, n in enumerate(LENS)]
    cu = torch.tensor([0] + LENS, device='cuda').cumsum(0)
    x = [torch.cat([d[j][:, :n] for d, n in zip(docs, LENS)], 1) for j in range(6)]
    o, cache = ccq_b200.ccq_gated_delta_rule(*x, output_cache=True, cu_seqlens=cu, subtract_mean=subtract_mean)
    return docs, cache


@pytest.mark.parametrize('subtract_mean', [True, False])
def test_generation_follows_a_packed_prefill(subtract_mean):
    import ccq_b200
    docs, cache = packed(3, subtract_mean)
    assert cache[3].tolist() == LENS
    for n, (doc, length) in enumerate(zip(docs, LENS)):
        whole, _ = ccq_b200.ccq_gated_delta_rule(*doc, subtract_mean=subtract_mean)
        one = tuple(t[n:n + 1].clone() if t is not None else None for t in cache[:3]) + (int(cache[3][n]),)
        for t in range(length, length + 3):
            o, one = ccq_b200.ccq_gated_delta_step(*(y[:, t:t + 1] for y in doc), one, subtract_mean=subtract_mean)
            assert (o - whole[:, t:t + 1]).abs().max() <= 2e-2
        assert one[3] == length + 3


def test_documents_of_different_lengths_take_no_common_step():
    import ccq_b200
    docs, cache = packed(1)
    token = [torch.cat([d[j][:, n:n + 1] for d, n in zip(docs, LENS)]) for j in range(6)]
    kept = [t.clone() for t in cache[:3]]
    with pytest.raises(ValueError, match='positions of their own'):
        ccq_b200.ccq_gated_delta_step(*token, cache)
    with pytest.raises(ValueError, match='positions of their own'):
        ccq_b200.ccq_gated_delta_rule(*token, cache=cache)
    assert all(torch.equal(a, b) for a, b in zip(kept, cache[:3]))


def test_one_packed_document_keeps_an_int_offset():
    import ccq_b200
    x = inputs(40)
    _, cache = ccq_b200.ccq_gated_delta_rule(*x, output_cache=True, cu_seqlens=torch.tensor([0, 40], device='cuda'))
    assert cache[3] == 40 and isinstance(cache[3], int)


@pytest.mark.parametrize('edit', ['half state', 'transposed state', 'state shape', 'value batch', 'gate type', 'beta shape', 'no state'])
def test_a_refused_step_leaves_the_cache_as_it_was(edit):
    """The cleaning read and the rule update the cache one after the other: what the rule refuses, neither may do."""
    import ccq_b200
    x = inputs(30)
    _, cache = ccq_b200.ccq_gated_delta_rule(*x, output_cache=True)
    q, k, v, lam, g, beta = inputs(1, seed=9)
    state = cache[0]
    if edit == 'half state':
        state = state.half()
    elif edit == 'transposed state':
        state = state.transpose(2, 3).contiguous().transpose(2, 3)
    elif edit == 'state shape':
        state = state[:, :1].contiguous()
    elif edit == 'value batch':
        v = torch.cat([v, v])
    elif edit == 'gate type':
        g = g.double()
    elif edit == 'beta shape':
        beta = beta[..., :1]
    else:
        state = None
    cache = (state, *cache[1:])
    kept = [t.clone() for t in cache[1:3]]
    with pytest.raises((ValueError, TypeError)):
        ccq_b200.ccq_gated_delta_step(q, k, v, lam, g, beta, cache)
    assert all(torch.equal(a, b) for a, b in zip(kept, cache[1:3]))
