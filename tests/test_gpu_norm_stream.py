"""The norms with a residual stream in a wider type than x's, against their float64 statement.

Bars as in the norms' other tests: fp32 arithmetic to 1e-5 of the value (of the largest term for the input gradient),
and one rounding of what has a 16-bit type, at most 2^-8 (bfloat16) or 2^-11 (float16) of it."""
import pytest
import torch

from oracle import delta_rule_oracle as O

pytestmark = pytest.mark.gpu
ROUND = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope='module', autouse=True)
def _lib():
    if not torch.cuda.is_available():
        pytest.skip('no CUDA device')
    from ccq_b200 import _lib as L
    L.load()


@pytest.mark.parametrize('x_type,stream', [(torch.bfloat16, torch.float32), (torch.float16, torch.float32),
                                           (torch.bfloat16, torch.float16), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize('form', ['layer', 'rms'])
@pytest.mark.parametrize('R,D', [(1, 64), (37, 250), (300, 2048)])
def test_mixed_types(x_type, stream, form, R, D):
    import ccq_b200
    r = lambda *s: torch.randn(*s, device='cuda')  # noqa: E731
    wide = torch.promote_types(x_type, stream)
    x, res = r(R, D).to(x_type).requires_grad_(True), (20 * r(R, D)).to(stream).requires_grad_(True)
    w = (1 + 0.1 * r(D)).requires_grad_(True)
    dy, dh = r(R, D).to(x_type), r(R, D).to(wide)
    f = ccq_b200.layer_norm if form == 'layer' else ccq_b200.rms_norm
    y, h = f(x, w, residual=res)
    assert y.dtype == x_type and h.dtype == wide
    grads = torch.autograd.grad([y, h], [x, res, w], [dy, dh])
    ref = O.norm(x, w, residual=res, center=form == 'layer', dy=dy, dh=dh)
    got = dict(y=y, h=h, dx=grads[0], dresidual=grads[1], dweight=grads[2])
    ref['dresidual'] = ref['dx']
    for name, t in got.items():
        size = ref[name].norm().item()
        terms = ref['terms'] if name in ('dx', 'dresidual') else size
        off = (t.detach().double() - ref[name]).norm().item()
        assert off <= ROUND[t.dtype] * size + 1e-5 * terms, f'{name}: {off:.2e} of {size:.2e}'


def test_a_float32_stream_keeps_small_additions():
    """64 blocks that each add 1/64 of a stream's last bfloat16 place: rounding on the way would lose them all."""
    import ccq_b200
    x = torch.full((4, 128), 2.0 ** -8 / 64, dtype=torch.bfloat16, device='cuda')
    h = torch.ones(4, 128, device='cuda')
    for _ in range(64):
        _, h = ccq_b200.rms_norm(x, residual=h)
    assert h.dtype == torch.float32 and torch.equal(h, torch.full_like(h, 1 + 2.0 ** -8))
