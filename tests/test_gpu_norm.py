"""Layer norm, RMS norm and the gated RMS norm on the GPU against their float64 statement.

Bars, on the 2-norm of the difference.  Arithmetic in fp32, the weight gradients' sums over the rows among
it: 1e-5 of the value; for the input gradient, whose terms cancel where a row has few elements or little
variance, 1e-5 of its largest term r dn (and of dh).  Values in a 16-bit type are rounded once after
that: at most the unit rounding of the value, 2^-8 for bfloat16 (8 significant bits) and 2^-11 for float16.
"""
import pytest
import torch

from oracle import delta_rule_oracle as O

pytestmark = pytest.mark.gpu

DT = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
ROUND = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BAR = {d: u + 1e-5 for d, u in ROUND.items()}


@pytest.fixture(scope='module', autouse=True)
def _lib():
    if not torch.cuda.is_available():
        pytest.skip('no CUDA device')
    from ccq_b200 import _lib as L
    L.load()


def rel(x, y):
    x, y = x.detach().double(), y.double()
    assert x.shape == y.shape and torch.isfinite(x).all()
    n, d = y.norm().item(), (x - y).norm().item()
    return d / n if n > 0 else d


def make(R, D, dtype, seed=0):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device='cuda')  # noqa: E731
    return dict(x=(r(R, D) * 2 + 0.5).to(dtype), weight=1 + 0.2 * r(D), bias=0.3 * r(D), residual=r(R, D).to(dtype),
                gate=r(R, D).to(dtype), dy=r(R, D).to(dtype), dh=r(R, D).to(dtype))


def check(form, R, D, dtype, residual=False, weight=True, bias=True, dh=True, t=None, eps=1e-5):
    import ccq_b200
    t = t or make(R, D, dtype)
    leaf = {n: t[n].detach().clone().requires_grad_(True) for n in ('x', 'weight', 'bias', 'residual', 'gate')}
    w = leaf['weight'] if weight else None
    if form == 'gated':
        y, h = ccq_b200.gated_rms_norm(leaf['x'], leaf['gate'], w, eps=eps), None
        kw = dict(weight=w, gate=leaf['gate'], center=False)
    else:
        res = leaf['residual'] if residual else None
        b = leaf['bias'] if bias and form == 'layer' else None
        f = ccq_b200.layer_norm if form == 'layer' else ccq_b200.rms_norm
        y = f(leaf['x'], w, *([b] if form == 'layer' else []), eps=eps, residual=res)
        y, h = y if residual else (y, None)
        kw = dict(weight=w, bias=b, residual=res, center=form == 'layer')
    names = ['x'] + (['weight'] if weight else []) + (['bias'] if kw.get('bias') is not None else [])
    names += (['residual'] if residual else []) + (['gate'] if form == 'gated' else [])
    outs, seen = [y], [t['dy']]
    if residual and dh:
        outs, seen = [y, h], [t['dy'], t['dh']]
    grads = dict(zip(names, torch.autograd.grad(outs, [leaf[n] for n in names], seen)))
    ref = O.norm(leaf['x'], eps=eps, dy=t['dy'], dh=t['dh'] if residual and dh else None, **kw)
    got = {'y': y, **{'d' + n: g for n, g in grads.items()}}
    if residual:
        got['h'] = h
        ref['dresidual'] = ref['dx']
    for name, v in got.items():
        assert v.dtype == (torch.float32 if name in ('dweight', 'dbias') else dtype)
        size = ref[name].norm().item()
        terms = ref['terms'] if name in ('dx', 'dresidual') else size
        off = (v.detach().double() - ref[name]).norm().item()
        assert v.shape == ref[name].shape and torch.isfinite(v).all()
        assert off <= ROUND[v.dtype] * size + 1e-5 * terms, f'{name}: {off:.2e} of {size:.2e}'
    return got


@pytest.mark.parametrize('D', [1, 2, 7, 8, 33, 64, 96, 127, 128, 136, 256, 257, 512, 1000, 1024, 1531, 2048, 4096, 5000,
                               8192, 8200, 16384])
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_widths(D, dtype):
    check('layer' if D > 1 else 'rms', 37, D, DT[dtype])


@pytest.mark.parametrize('form,residual', [('layer', False), ('layer', True), ('rms', False), ('rms', True), ('gated', False)])
@pytest.mark.parametrize('R', [1, 3, 65, 2500])
@pytest.mark.parametrize('D', [64, 100, 640])
def test_forms(form, residual, R, D):
    check(form, R, D, torch.bfloat16, residual)


@pytest.mark.parametrize('form', ['layer', 'rms', 'gated'])
def test_without_parameters(form):
    check(form, 50, 128, torch.float32, weight=False, bias=False)
    check(form, 50, 128, torch.bfloat16, residual=form != 'gated', bias=False, dh=False)


def test_constant_and_zero_rows():
    """Rows without variance: eps alone keeps the result finite."""
    t = make(6, 64, torch.float32)
    t['x'][0], t['x'][1], t['residual'][0], t['residual'][1] = 0.0, 3.0, 0.0, 0.0
    check('layer', 6, 64, torch.float32, residual=True, t=t)
    check('rms', 6, 64, torch.float32, t=t)


def test_rows_do_not_touch_each_other():
    import ccq_b200
    t = make(40, 256, torch.bfloat16)
    want = ccq_b200.layer_norm(t['x'], t['weight'], t['bias'])
    t['x'][7] = float('nan')
    t['x'][8] = float('inf')
    got = ccq_b200.layer_norm(t['x'], t['weight'], t['bias'])
    keep = [i for i in range(40) if i not in (7, 8)]
    assert torch.equal(got[keep], want[keep])


def test_leading_axes_strides_and_no_rows():
    import ccq_b200
    t = make(24, 96, torch.float16)
    want = ccq_b200.layer_norm(t['x'], t['weight'], t['bias'])
    wide = torch.zeros(24, 97, dtype=torch.float16, device='cuda')
    wide[:, 1:] = t['x']
    assert torch.equal(ccq_b200.layer_norm(wide[:, 1:], t['weight'], t['bias']), want)
    got = ccq_b200.layer_norm(t['x'].view(2, 3, 4, 96), t['weight'], t['bias'])
    assert torch.equal(got.view(24, 96), want)
    x = torch.zeros(0, 96, device='cuda', requires_grad=True)
    w = t['weight'].clone().requires_grad_(True)
    y = ccq_b200.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, [x, w], torch.zeros_like(y))
    assert y.shape == dx.shape == (0, 96) and (dw == 0).all()


def test_unaligned():
    """A contiguous row view that starts off a 16-byte boundary takes the scalar loads."""
    import ccq_b200
    t = make(9, 128, torch.bfloat16)
    buf = torch.empty(9 * 128 + 1, dtype=torch.bfloat16, device='cuda')
    buf[1:] = t['x'].reshape(-1)
    got = ccq_b200.layer_norm(buf[1:].view(9, 128), t['weight'], t['bias'])
    assert rel(got, O.norm(t['x'], t['weight'], t['bias'])['y']) <= BAR[torch.bfloat16]


def test_same_bits_and_another_stream():
    import ccq_b200
    t = make(3000, 512, torch.bfloat16)
    leaf = [t[n].requires_grad_(True) for n in ('x', 'weight', 'bias')]

    def run():
        y = ccq_b200.layer_norm(*leaf)
        return [y, *torch.autograd.grad(y, leaf, t['dy'])]

    one = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        two = run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(one, two))


@pytest.mark.parametrize('form', ['layer', 'gated'])
def test_gradients_against_differences(form):
    """Central differences of the fp32 forward along one direction in every input at once; a loss error of
    about 1e-6 |y| over a step of 1e-2 and the third derivative leave about 1e-3 of the slope's scale."""
    import ccq_b200
    t = make(11, 75, torch.float32, seed=3)
    names = ['x', 'weight', 'gate'] if form == 'gated' else ['x', 'weight', 'bias', 'residual']

    def call(v):
        if form == 'gated':
            return ccq_b200.gated_rms_norm(v['x'], v['gate'], v['weight'])
        return ccq_b200.layer_norm(v['x'], v['weight'], v['bias'], residual=v['residual'])[0]

    leaf = {n: t[n].clone().requires_grad_(True) for n in names}
    grads = torch.autograd.grad(call(leaf), [leaf[n] for n in names], t['dy'])
    gen = torch.Generator(device='cuda').manual_seed(1)
    for n, g in zip(names, grads):
        d = torch.randn(t[n].shape, generator=gen, device='cuda')
        d = d / d.norm()
        up, down = ((call({**t, n: t[n] + s * d}).double() * t['dy'].double()).sum() for s in (1e-2, -1e-2))
        want = ((up - down) / 2e-2).item()
        assert abs((g.double() * d.double()).sum().item() - want) <= 3e-3 * max(1.0, g.norm().item() / g.numel() ** 0.5 * 3)


def test_refusals():
    import ccq_b200
    t = make(4, 32, torch.float32)
    with pytest.raises(ValueError, match='weight has shape'):
        ccq_b200.layer_norm(t['x'], t['weight'][:5])
    with pytest.raises(ValueError, match='bias has shape'):
        ccq_b200.layer_norm(t['x'], t['weight'], t['bias'][:5])
    with pytest.raises(ValueError, match='residual has shape'):
        ccq_b200.rms_norm(t['x'], residual=t['residual'][:2])
    with pytest.raises(ValueError, match='gate has shape'):
        ccq_b200.gated_rms_norm(t['x'], t['gate'][:2])
    with pytest.raises(TypeError, match='dtype'):
        ccq_b200.layer_norm(t['x'].double())
    with pytest.raises(RuntimeError, match='CUDA'):
        ccq_b200.layer_norm(t['x'].cpu())
    with pytest.raises(ccq_b200.CCQError, match='eps'):
        ccq_b200.layer_norm(t['x'], eps=-1.0)
    with pytest.raises(ccq_b200.CCQError, match='D=16385'):
        ccq_b200.layer_norm(torch.zeros(1, 16385, device='cuda'))
