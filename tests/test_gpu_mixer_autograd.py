"""What the mixer operators tell autograd."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module', autouse=True)
def _lib():
    if not torch.cuda.is_available():
        pytest.skip('no CUDA device')
    from ccq_b200 import _lib as L
    L.load()


def inputs(T=40, B=2, H=2, HV=2, K=128, V=64, dtype=torch.bfloat16):
    r = lambda *s: torch.randn(*s, device='cuda')  # noqa: E731
    unit = lambda t: torch.nn.functional.normalize(t, dim=-1)  # noqa: E731
    x = [unit(r(B, T, H, K)), unit(r(B, T, H, K)), r(B, T, HV, V)]
    return [t.to(dtype) for t in x] + [-torch.rand(B, T, HV, device='cuda'), r(B, T, HV).sigmoid()]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('leaf', ['q', 'state'])
def test_a_step_on_a_saved_state_is_seen(dtype, leaf):
    """A backward that saved the state raises once a step has written to it, as after an in-place operation of torch."""
    import ccq_b200
    x, token = inputs(dtype=dtype), inputs(1, dtype=dtype)
    state = torch.randn(2, 2, 128, 64, device='cuda')
    (x[0] if leaf == 'q' else state).requires_grad_(True)
    loss = ccq_b200.gated_delta_rule(*x, initial_state=state)[0].float().sum()
    with torch.no_grad():
        ccq_b200.gated_delta_step(*token, state)                     # a new state: nothing is written
        loss.backward(retain_graph=True)
        ccq_b200.gated_delta_step(*token, state, inplace=True)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()


@pytest.mark.parametrize('which', [1, 2])
def test_a_step_on_a_saved_covariance_or_mean_is_seen(which):
    import ccq_b200
    q, k, _, _, _ = inputs()
    cov, mean = torch.randn(2, 2, 128, 128, device='cuda'), torch.randn(2, 2, 128, device='cuda')
    one = lambda t, i: t.clone() if i != which else t  # noqa: E731
    loss = ccq_b200.fused_ccq_clean_read(q.requires_grad_(True), k, 0.5, initial_cov_state=cov,
                                         initial_mean_state=mean)[0].float().sum()
    with torch.no_grad():
        ccq_b200.decode_step(q[:, :1], k[:, :1], 0.5, cov, mean)
        loss.backward(retain_graph=True)
        ccq_b200.decode_step(q[:, :1], k[:, :1], 0.5, one(cov, 1), one(mean, 2), inplace=True)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()


def test_steps_in_inference_mode():
    import ccq_b200
    with torch.inference_mode():
        state = torch.zeros(2, 2, 128, 64, device='cuda')
        o, S = ccq_b200.gated_delta_step(*inputs(1), state, inplace=True)
        assert S is state and torch.isfinite(o).all() and (state != 0).any()


def _calls():
    import ccq_b200
    x = inputs(dtype=torch.float32)
    rows, w = torch.randn(5, 64, device='cuda'), torch.ones(64, device='cuda')
    yield 'rule', x, lambda *t: ccq_b200.gated_delta_rule(*t)[0]
    yield 'rule with a state', [*x, torch.randn(2, 2, 128, 64, device='cuda')], lambda *t: ccq_b200.gated_delta_rule(*t[:5], initial_state=t[5])[0]
    yield 'layer norm', [rows, w, w], ccq_b200.layer_norm
    yield 'rms norm', [rows, w, rows], lambda a, b, c: ccq_b200.rms_norm(a, b, residual=c)[0]
    yield 'gated', [rows, rows, w], ccq_b200.gated_rms_norm


@pytest.mark.parametrize('grad', [True, False])
def test_forward_mode_is_refused(grad):
    """There is no forward-mode derivative: an input that carries a tangent raises, whichever it is, and does not
    come out as a constant."""
    from torch.autograd import forward_ad
    for name, x, f in _calls():
        for i in range(len(x)):
            with torch.set_grad_enabled(grad), forward_ad.dual_level():
                y = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(x)]
                with pytest.raises((RuntimeError, NotImplementedError), match='jvp|forward mode'):
                    f(*y)
                assert torch.isfinite(f(*x)).all(), name     # no tangent: an ordinary call


def test_a_second_derivative_is_refused():
    """A penalty on a gradient raises; without the refusal its part through the operators would be left out."""
    for name, x, f in _calls():
        x = [t.detach().clone().requires_grad_(True) for t in x]
        seed = torch.randn_like(f(*x))
        plain = torch.autograd.grad(f(*x), x, seed)
        graph = torch.autograd.grad(f(*x), x, seed, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(plain, graph)), name
        for d in graph:
            with pytest.raises(RuntimeError, match='second derivative'):
                (d.square().sum() + sum(t.square().sum() for t in x)).backward()
