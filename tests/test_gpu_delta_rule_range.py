"""The gated delta rule in float16 away from the scale of one, against the float64 statement.

The inputs q, k, v and d_o are float16 values; states, their gradients, dg and dbeta are float32 of any size.  Bars as in
the operator's other tests (2-norm of the difference over that of the value): 2e-5 for the states, 1e-3 for the rest,
and for what is rounded to float16 half of its smallest step, 2^-25 an element, which is all that is left of values near it.
The state's gradient has to hold the state's bar too."""
import pytest
import torch

from oracle import delta_rule_oracle as O

pytestmark = pytest.mark.gpu
NAMES = ('q', 'k', 'v', 'g', 'beta')


@pytest.fixture(scope='module', autouse=True)
def _lib():
    if not torch.cuda.is_available():
        pytest.skip('no CUDA device')
    from ccq_b200 import _lib as L
    L.load()


def check(B, T, H, HV, K, V, v=1.0, state=1.0, do=1.0, dstate=1.0, scale=None, lens=None, dtype=torch.float16, keys=1.0, write=1.0, column=None, gate=None):
    """One forward and backward; the arguments after the sizes are those of the values."""
    import ccq_b200
    gen = torch.Generator(device='cuda').manual_seed(T + V)
    r = lambda *s: torch.randn(*s, generator=gen, device='cuda')  # noqa: E731
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
    N = len(lens) if lens else B
    x = dict(q=(keys * unit(r(B, T, H, K))).to(dtype), k=unit(r(B, T, H, K)).to(dtype), v=(v * r(B, T, HV, V)).to(dtype),
             g=-torch.nn.functional.softplus(r(B, T, HV) * 2 - 3.0), beta=write * torch.sigmoid(r(B, T, HV)))
    if gate:
        x['g'] = gate(x['g'])
    d_o, h0, dh = (do * r(B, T, HV, V)).to(dtype), state * r(N, HV, K, V), dstate * r(N, HV, K, V)
    if column is not None:
        h0[..., column] *= 1e4
    for t in (*x.values(), h0):
        t.requires_grad_(True)
    cu = torch.tensor([0] + list(lens), device='cuda').cumsum(0) if lens else None
    o, S = ccq_b200.gated_delta_rule(*(x[n] for n in NAMES), scale=scale, initial_state=h0, output_final_state=True, cu_seqlens=cu)
    assert ccq_b200.last_path() == 'tcgen05'
    grads = torch.autograd.grad([o, S], [*(x[n] for n in NAMES), h0], [d_o, dh])
    ref = O.delta_rule(*(x[n] for n in NAMES), K ** -0.5 if scale is None else scale, h0, lens, d_o, dh)
    got = dict(zip(['d' + n for n in NAMES] + ['dstate'], grads), o=o, state=S)
    for name, t in got.items():
        want = ref[name]
        if t.dtype == torch.float16:
            assert want.abs().max() < 65504, f'{name}: the test asks for more than float16 holds'
        assert torch.isfinite(t).all(), name
        bar = (2e-5 if 'state' in name else 1e-3) * want.norm().item()
        if t.dtype == torch.float16:
            bar += 2.0 ** -25 * t.numel() ** 0.5
        off = (t.detach().double() - want).norm().item()
        assert off <= bar, f'{name}: {off / max(want.norm().item(), 1e-300):.2e} of {want.norm().item():.2e}, bar {bar:.2e}'
    return got


SIZES = [(2, 130, 2, 2, 128, 128, None), (1, 200, 1, 2, 64, 72, [70, 0, 1, 129]), (1, 100, 2, 4, 128, 256, None)]


@pytest.mark.parametrize('B,T,H,HV,K,V,lens', SIZES)
@pytest.mark.parametrize('size', [1e-5, 1e-3, 1.0, 1e3])
def test_values_and_states(B, T, H, HV, K, V, lens, size):
    check(B, T, H, HV, K, V, v=size, state=size, lens=lens)


@pytest.mark.parametrize('B,T,H,HV,K,V,lens', SIZES)
@pytest.mark.parametrize('size', [1e-5, 1e-3, 1e2])
def test_gradients(B, T, H, HV, K, V, lens, size):
    check(B, T, H, HV, K, V, do=size, dstate=size, lens=lens)


@pytest.mark.parametrize('B,T,H,HV,K,V,lens', SIZES)
@pytest.mark.parametrize('kw', [
    dict(state=1e6, scale=1e-4, do=1e-2, dstate=1e-4),     # a state that float16 does not hold
    dict(state=1e12, scale=1e-9, do=1e-2, dstate=1e-10),
    dict(dstate=1e6, do=1e-3, state=1e-2, v=1e-2, write=1e-2),  # its gradient (dv = beta dS k has to fit)
    dict(state=1e-12, v=1e-3),                             # a state that vanishes beside the values, and before them
    dict(dstate=1e-12, do=1e-3),
    dict(v=1e3, do=1e-5, state=1e3, dstate=1e-5),
    dict(v=1e-5, do=1e3, state=1e-5, dstate=1e3),
])
def test_far_apart(B, T, H, HV, K, V, lens, kw):
    check(B, T, H, HV, K, V, lens=lens, **kw)


def test_one_large_column():
    check(2, 130, 2, 2, 128, 128, column=5, scale=1e-2, do=1e-2, dstate=1e-2)


@pytest.mark.parametrize('keys', [1e-4, 30.0])
def test_scores(keys):
    """q of another size: the scores P go with it."""
    check(2, 130, 2, 2, 128, 128, keys=keys)


@pytest.mark.parametrize('kw', [dict(v=1e-5, state=1e-5, do=1e-5, dstate=1e-5), dict(state=1e6, scale=1e-4, do=1e-2, dstate=1e-4)])
def test_segments(kw):
    check(1, 1601, 1, 1, 128, 128, **kw)


@pytest.mark.parametrize('gate', [lambda g: 40 * g, lambda g: -0.2 * g, lambda g: 40 * g * (g < -0.05) - 0.1 * g], ids=['falls', 'grows', 'both'])
@pytest.mark.parametrize('kw', [dict(), dict(v=1e-3, state=1e-3, do=1e-3, dstate=1e-3), dict(state=1e5, scale=1e-4, do=1e-4, dstate=1e-5)])
def test_decay(gate, kw):
    """Decay that empties the state within a few tokens, growth, and one after the other: factors from bounds follow."""
    check(2, 200, 2, 2, 128, 128, gate=gate, **kw)


def test_nothing_at_all():
    """All values, states and gradients zero, and beta zero: exact zeros, no factor of nothing."""
    got = check(1, 70, 2, 2, 128, 128, v=0.0, state=0.0, do=0.0, dstate=0.0)
    assert all((t == 0).all() for t in got.values())


@pytest.mark.parametrize('chunk', [0, 1])
def test_empty_chunks(chunk):
    """A chunk without write strength or without a gradient, beside one with both, and states of 1e9."""
    import ccq_b200
    r = lambda *s: torch.randn(*s, device='cuda')  # noqa: E731
    q, k = (torch.nn.functional.normalize(r(1, 128, 2, 128), dim=-1).half() for _ in range(2))
    v, d_o, g, beta = r(1, 128, 2, 256).half(), 1e-2 * r(1, 128, 2, 256).half(), -torch.rand(1, 128, 2, device='cuda'), r(1, 128, 2).sigmoid()
    beta[:, 64 * chunk:64 * chunk + 64] = 0
    d_o[:, 64 - 64 * chunk:128 - 64 * chunk] = 0
    h0 = 1e9 * r(1, 2, 128, 256)
    x = [t.requires_grad_(True) for t in (q, k, v, g, beta, h0)]
    o, S = ccq_b200.gated_delta_rule(*x[:5], scale=1e-6, initial_state=h0, output_final_state=True)
    grads = torch.autograd.grad(o, x, d_o)
    ref = O.delta_rule(*x[:5], 1e-6, h0, None, d_o)
    for name, t in zip(['o', 'state', 'dq', 'dk', 'dv', 'dg', 'dbeta', 'dstate'], [o, S, *grads]):
        want = ref[name]
        if want.abs().max() >= 65504 and t.dtype == torch.float16:
            continue
        bar = (2e-5 if 'state' in name else 1e-3) * want.norm().item() + (2.0 ** -25 * t.numel() ** 0.5 if t.dtype == torch.float16 else 0)
        assert torch.isfinite(t).all() and (t.double() - want).norm().item() <= bar, name


def test_step_and_rule_agree_on_a_large_state():
    """Prefill onto a state of 1e6, token by token and in chunks."""
    import ccq_b200
    r = lambda *s: torch.randn(*s, device='cuda')  # noqa: E731
    q, k = (torch.nn.functional.normalize(r(2, 70, 2, 128), dim=-1).half() for _ in range(2))
    v, g, beta, h0 = r(2, 70, 2, 64).half(), -torch.rand(2, 70, 2, device='cuda') / 8, r(2, 70, 2).sigmoid(), 1e6 * r(2, 2, 128, 64)
    a, S = ccq_b200.gated_delta_rule(q, k, v, g, beta, scale=1e-4, initial_state=h0, output_final_state=True)
    b, T = ccq_b200.gated_delta_step(q, k, v, g, beta, h0, scale=1e-4)
    assert torch.isfinite(a).all() and (a.double() - b.double()).norm() <= 1e-3 * b.double().norm()
    assert (S - T).norm() <= 3e-5 * T.norm()


@pytest.mark.parametrize('bad', [float('nan'), float('inf'), 6e4])
def test_factors_stay_in_their_document(bad):
    """A document of NaN, infinities or values near float16's end between two others: theirs are the same, bit for bit."""
    import ccq_b200
    lens, r = [70, 33, 90], lambda *s: torch.randn(*s, device='cuda')
    cu = torch.tensor([0] + lens, device='cuda').cumsum(0)
    T = sum(lens)
    x = [torch.nn.functional.normalize(r(1, T, 2, 128), dim=-1).half() for _ in range(2)]
    x += [r(1, T, 4, 256).half(), -torch.rand(1, T, 4, device='cuda'), r(1, T, 4).sigmoid()]
    d_o = r(1, T, 4, 256).half()

    def run():
        y = [t.clone().requires_grad_(True) for t in x]
        o, S = ccq_b200.gated_delta_rule(*y, output_final_state=True, cu_seqlens=cu)
        return [o, *torch.autograd.grad(o, y, d_o)], S

    clean, S0 = run()
    for t in x[:3] + [d_o]:
        t[:, 70:103] = bad
    dirty, S1 = run()
    again, _ = run()
    for a, b, c in zip(clean, dirty, again):
        assert torch.equal(a[:, :70], b[:, :70]) and torch.equal(a[:, 103:], b[:, 103:])
        assert torch.equal(b[:, :70], c[:, :70]) and torch.equal(b[:, 103:], c[:, 103:])
    assert torch.equal(S0[[0, 2]], S1[[0, 2]])
