"""The gated delta rule on the GPU against its float64 statement (oracle/delta_rule_oracle.py).

Bars, as the 2-norm of the difference over that of the value.  float32: 1e-5, the bar of the other
operators (sums of at most 256 products, about 2^-24 sqrt(256) each, and a few of them in a row).  16-bit
types: one rounding to nearest is off by about 0.42 u in the 2-norm, u = 2^-8 for bfloat16 and 2^-11 for
float16; the output's own and up to seven of operands along a path, independent, make 1.2 u: 5e-3 and
(with float16's subnormals) 1e-3.  The states, float32 outputs of 16-bit calls: 2e-5.
"""
import pytest
import torch

from oracle import delta_rule_oracle as O

pytestmark = pytest.mark.gpu

BAR = {torch.float32: 1e-5, torch.bfloat16: 5e-3, torch.float16: 1e-3}
DT = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


@pytest.fixture(scope='module', autouse=True)
def _lib():
    if not torch.cuda.is_available():
        pytest.skip('no CUDA device')
    from ccq_b200 import _lib as L
    L.load()


def rel(x, y):
    x, y = x.detach().double(), y.double()
    assert x.shape == y.shape
    assert torch.isfinite(x).all()
    n = y.norm().item()
    d = (x - y).norm().item()
    return d / n if n > 0 else d


def inputs(B, T, H, HV, K, V, dtype, N=None, seed=0, strong=False):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device='cuda')  # noqa: E731
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
    q, k = unit(r(B, T, H, K)).to(dtype), unit(r(B, T, H, K)).to(dtype)
    v, do = r(B, T, HV, V).to(dtype), r(B, T, HV, V).to(dtype)
    g = -torch.nn.functional.softplus(r(B, T, HV) * 2 - (0.0 if strong else 3.0)) * (8.0 if strong else 1.0)
    beta = torch.sigmoid(r(B, T, HV))
    N = N or B
    return dict(q=q, k=k, v=v, g=g, beta=beta), do, 0.5 * r(N, HV, K, V), 0.1 * r(N, HV, K, V)


NAMES = ('q', 'k', 'v', 'g', 'beta')


def check(B, T, H, HV, K, V, dtype, lens=None, states=True, gate=torch.float32, scale=None, seed=0, strong=False,
          edit=None):
    """One forward and backward against the oracle; returns the framework's outputs."""
    import ccq_b200
    N = len(lens) if lens else B
    x, do, h0, dh = inputs(B, T, H, HV, K, V, dtype, N, seed, strong)
    x['g'], x['beta'] = x['g'].to(gate), x['beta'].to(gate)
    if edit:
        edit(x)
    for n in NAMES:
        x[n].requires_grad_(True)
    h0 = h0.requires_grad_(True) if states else None
    cu = torch.tensor([0] + list(lens), device='cuda').cumsum(0) if lens else None
    o, S = ccq_b200.gated_delta_rule(*(x[n] for n in NAMES), scale=scale, initial_state=h0, output_final_state=True,
                                     cu_seqlens=cu)
    outs, seen = ([o, S], [do, dh]) if states else ([o], [do])
    wrt = [x[n] for n in NAMES] + ([h0] if states else [])
    grads = torch.autograd.grad(outs, wrt, seen)
    ref = O.delta_rule(*(x[n] for n in NAMES), K ** -0.5 if scale is None else scale, h0, lens, do,
                       dh if states else None)
    got = dict(zip(['d' + n for n in NAMES] + ['dstate'], grads), o=o, state=S)
    for name, t in got.items():
        assert t.dtype == (torch.float32 if 'state' in name else gate if name in ('dg', 'dbeta') else dtype)
        bar = BAR[dtype] if name not in ('state',) else (1e-5 if dtype == torch.float32 else 2e-5)
        if gate != torch.float32 and name in ('dg', 'dbeta'):
            bar = max(bar, BAR[gate])
        assert rel(t, ref[name]) <= bar, f'{name}: {rel(t, ref[name]):.2e} over {bar:.1e}'
    return got


@pytest.mark.parametrize('T', [1, 2, 31, 32, 33, 64, 65, 127, 200])
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_lengths(T, dtype):
    check(2, T, 2, 2, 128, 128, DT[dtype], states=T % 2 == 1)


@pytest.mark.parametrize('K,V', [(1, 1), (4, 3), (20, 33), (64, 64), (64, 128), (96, 160), (100, 48), (128, 8), (128, 72),
                                 (128, 256), (72, 128), (192, 128), (256, 256), (255, 31)])
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_head_sizes(K, V, dtype):
    check(1, 90, 2, 2, K, V, DT[dtype])


@pytest.mark.parametrize('H,HV', [(1, 1), (1, 4), (2, 6), (3, 3)])
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_shared_key_heads(H, HV, dtype):
    check(2, 100, H, HV, 128, 128, DT[dtype], states=False)


@pytest.mark.parametrize('lens', [[5], [0, 7], [64, 1, 0, 63, 65, 128], [1, 1, 1, 0, 0, 200], [130, 130]])
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('states', [True, False])
def test_packed_documents(lens, dtype, states):
    check(1, sum(lens), 2, 4, 128, 128, DT[dtype], lens=lens, states=states)


@pytest.mark.parametrize('dtype,gate', [('bf16', 'bf16'), ('f16', 'f16'), ('bf16', 'f32'), ('f32', 'bf16')])
def test_gate_types(dtype, gate):
    check(2, 70, 2, 2, 128, 128, DT[dtype], gate=DT[gate])


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_strong_decay_and_scale(dtype):
    check(2, 150, 2, 2, 128, 128, DT[dtype], strong=True, scale=0.5)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_gates_at_their_ends(dtype):
    """beta of 0 and 1, no decay, resets (g of -inf and of the type's lowest value)."""
    def edit(x):
        x['beta'][:, ::3] = 0.0
        x['beta'][:, 1::3] = 1.0
        x['g'][:, ::5] = 0.0
        x['g'][:, 40] = float('-inf')
        x['g'][:, 71] = torch.finfo(torch.float32).min
    check(2, 150, 2, 2, 128, 128, DT[dtype], edit=edit)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_first_token_without_state_has_no_decay_gradient(dtype):
    got = check(1, 130, 2, 2, 128, 128, DT[dtype], lens=[1, 65, 0, 64], states=False)
    assert (got['dg'][0, [0, 1, 66]] == 0).all()


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
def test_documents_do_not_touch_each_other(dtype, bad):
    """A document of NaN or infinities between two others: theirs are the same, bit for bit."""
    import ccq_b200
    lens = [70, 33, 90]
    cu = torch.tensor([0] + lens, device='cuda').cumsum(0)
    x, do, _, _ = inputs(1, sum(lens), 2, 2, 128, 128, DT[dtype])

    def run():
        y = {n: t.clone().requires_grad_(True) for n, t in x.items()}
        o, S = ccq_b200.gated_delta_rule(*(y[n] for n in NAMES), output_final_state=True, cu_seqlens=cu)
        return [o, *torch.autograd.grad(o, [y[n] for n in NAMES], do)], S

    clean, S0 = run()
    for n in NAMES:
        x[n][:, 70:103] = bad
    dirty, S1 = run()
    for a, b in zip(clean, dirty):
        assert torch.equal(a[:, :70], b[:, :70]) and torch.equal(a[:, 103:], b[:, 103:])
    assert torch.equal(S0[[0, 2]], S1[[0, 2]])


def test_long_document():
    check(1, 3000, 1, 1, 128, 128, torch.bfloat16, states=False)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_same_inputs_same_bits_and_another_stream(dtype):
    import ccq_b200
    x, do, h0, _ = inputs(2, 300, 2, 4, 128, 128, DT[dtype])
    y = [x[n].requires_grad_(True) for n in NAMES]

    def run():
        o, S = ccq_b200.gated_delta_rule(*y, initial_state=h0, output_final_state=True)
        return [o, S, *torch.autograd.grad(o, y, do)]

    one = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        two = run()
    side.synchronize()
    for a, b in zip(one, two):
        assert torch.equal(a, b)


def test_strided_inputs():
    import ccq_b200
    x, _, h0, _ = inputs(2, 70, 2, 2, 128, 128, torch.bfloat16)
    want = ccq_b200.gated_delta_rule(*(x[n] for n in NAMES), initial_state=h0)[0]
    odd = [x[n].transpose(0, 1).contiguous().transpose(0, 1) for n in NAMES]
    wide = torch.zeros(2, 70, 2, 129, dtype=torch.bfloat16, device='cuda')
    wide[..., 1:] = x['q']
    odd[0] = wide[..., 1:]
    got = ccq_b200.gated_delta_rule(*odd, initial_state=h0.transpose(2, 3).contiguous().transpose(2, 3))[0]
    assert torch.equal(got, want)


def test_unaligned_views():
    """Contiguous tensors that do not start on a 16-byte boundary."""
    import ccq_b200
    x, do, _, _ = inputs(1, 70, 2, 2, 128, 128, torch.bfloat16)

    def shift(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device='cuda')
        buf[1:] = t.reshape(-1)
        return buf[1:].reshape(t.shape)

    y = [shift(x[n]).requires_grad_(True) for n in NAMES]
    o, _ = ccq_b200.gated_delta_rule(*y)
    grads = torch.autograd.grad(o, y, shift(do))
    ref = O.delta_rule(*y, 128 ** -0.5, do=do)
    for n, t in zip(['o'] + ['d' + n for n in NAMES], [o, *grads]):
        assert rel(t, ref[n]) <= BAR[torch.bfloat16]


def test_no_tokens():
    import ccq_b200
    x, _, h0, dh = inputs(2, 0, 2, 2, 16, 16, torch.float32, N=2)
    h0.requires_grad_(True)
    o, S = ccq_b200.gated_delta_rule(*(x[n].requires_grad_(True) for n in NAMES), initial_state=h0,
                                     output_final_state=True)
    assert o.shape == (2, 0, 2, 16) and torch.equal(S, h0)
    assert torch.equal(torch.autograd.grad(S, h0, dh)[0], dh)


@pytest.mark.parametrize('name', NAMES + ('state',))
def test_gradients_against_differences(name):
    """Central differences of the fp32 forward along a random direction.  The loss is summed in float64; an
    output error of 1e-6 |o| over a step of 1e-2 and a third derivative of order one leave about 1e-3."""
    import ccq_b200
    x, do, h0, dh = inputs(1, 75, 2, 4, 48, 40, torch.float32, seed=5)
    x['state'] = h0

    def loss(y):
        o, S = ccq_b200.gated_delta_rule(*(y[n] for n in NAMES), initial_state=y['state'], output_final_state=True)
        return (o.double() * do.double()).sum() + (S.double() * dh.double()).sum()

    y = {n: t.clone() for n, t in x.items()}
    y[name].requires_grad_(True)
    o, S = ccq_b200.gated_delta_rule(*(y[n] for n in NAMES), initial_state=y['state'], output_final_state=True)
    grad = torch.autograd.grad([o, S], y[name], [do, dh])[0].double()
    gen = torch.Generator(device='cuda').manual_seed(9)
    d = torch.randn(x[name].shape, generator=gen, device='cuda')
    d = d / d.norm()
    step = 1e-2
    up, down = (loss({**x, name: x[name] + s * d}) for s in (step, -step))
    want = ((up - down) / (2 * step)).item()
    assert abs((grad * d.double()).sum().item() - want) <= 3e-3 * max(1.0, grad.norm().item() / grad.numel() ** 0.5 * 3)


# ------------------------------------------------------------------------------------------------
# token by token
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('K,V', [(1, 1), (7, 5), (64, 64), (64, 20), (128, 128), (96, 160), (128, 130), (256, 256), (200, 96)])
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('B,T', [(1, 1), (3, 4), (80, 1)])
def test_step(K, V, dtype, B, T):
    import ccq_b200
    x, _, h0, _ = inputs(B, T, 2, 4, K, V, DT[dtype])
    ref = O.delta_rule(*(x[n] for n in NAMES), K ** -0.5, h0)
    o, S = ccq_b200.gated_delta_step(*(x[n] for n in NAMES), h0)
    assert rel(o, ref['o']) <= BAR[DT[dtype]] and rel(S, ref['state']) <= 1e-5
    keep = h0.clone()
    o2, S2 = ccq_b200.gated_delta_step(*(x[n] for n in NAMES), keep, inplace=True)
    assert S2 is keep and torch.equal(S2, S) and torch.equal(o2, o)


def test_step_packed_and_without_state():
    import ccq_b200
    lens = [1, 0, 5, 2]
    x, _, h0, _ = inputs(1, sum(lens), 2, 2, 128, 128, torch.bfloat16, N=len(lens))
    cu = torch.tensor([0] + lens, device='cuda').cumsum(0)
    for state in (h0, None):
        ref = O.delta_rule(*(x[n] for n in NAMES), 128 ** -0.5, state, lens)
        o, S = ccq_b200.gated_delta_step(*(x[n] for n in NAMES), state, cu_seqlens=cu)
        assert rel(o, ref['o']) <= 5e-3 and rel(S, ref['state']) <= 1e-5


def test_step_follows_prefill():
    """Prefill of 100 tokens, then 5 steps, against all 105 at once."""
    import ccq_b200
    x, _, _, _ = inputs(2, 105, 2, 2, 128, 128, torch.bfloat16)
    whole, S = ccq_b200.gated_delta_rule(*(x[n] for n in NAMES), output_final_state=True)
    _, cache = ccq_b200.gated_delta_rule(*(x[n][:, :100] for n in NAMES), output_final_state=True)
    for t in range(100, 105):
        o, cache = ccq_b200.gated_delta_step(*(x[n][:, t:t + 1] for n in NAMES), cache, inplace=True)
        assert rel(o, whole[:, t:t + 1].double()) <= 5e-3
    assert rel(cache, S.double()) <= 4e-5


# ------------------------------------------------------------------------------------------------
# refusals
# ------------------------------------------------------------------------------------------------
def test_refusals():
    import ccq_b200
    x, _, h0, _ = inputs(2, 8, 2, 4, 16, 16, torch.float32)
    args = [x[n] for n in NAMES]

    def swap(i, t):
        return [t if j == i else y for j, y in enumerate(args)]

    for f in (ccq_b200.gated_delta_rule, ccq_b200.gated_delta_step):
        with pytest.raises(ValueError, match='k has shape'):
            f(*swap(1, args[1][:, :4]))
        with pytest.raises(ValueError, match='v has shape'):
            f(*swap(2, args[2][:1]))
        with pytest.raises(ValueError, match='multiple'):
            f(args[0], args[1], args[2][:, :, :3], args[3][..., :3], args[4][..., :3])
        with pytest.raises(ValueError, match='g has shape'):
            f(*swap(3, args[3][..., :2]))
        with pytest.raises(TypeError, match='dtype'):
            f(*swap(0, args[0].double()))
        with pytest.raises(TypeError, match='dtype'):
            f(*swap(4, args[4].double()))
        with pytest.raises(RuntimeError, match='CUDA'):
            f(*swap(0, args[0].cpu()))
        with pytest.raises(ValueError, match='batch size 1'):
            f(*args, cu_seqlens=torch.tensor([0, 16], device='cuda'))
    with pytest.raises(ValueError, match='state has shape'):
        ccq_b200.gated_delta_rule(*args, initial_state=h0[:1])
    with pytest.raises(ValueError, match='inplace'):
        ccq_b200.gated_delta_step(*args, h0.double(), inplace=True)
    with pytest.raises(ValueError, match='inplace'):
        ccq_b200.gated_delta_step(*args, inplace=True)
    big = inputs(1, 4, 1, 1, 257, 16, torch.float32)[0]
    with pytest.raises(ccq_b200.CCQError, match='K=257'):
        ccq_b200.gated_delta_rule(*(big[n] for n in NAMES))


# ------------------------------------------------------------------------------------------------
# few heads, a long axis: documents in segments that run side by side
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
@pytest.mark.parametrize('B,T,H,HV,K,V,lens', [
    (1, 1601, 1, 1, 128, 128, None),
    (2, 1100, 1, 2, 128, 256, None),
    (1, 2048, 2, 2, 64, 72, None),
    (1, 1500, 1, 2, 96, 128, [700, 0, 733, 64, 3]),
    (1, 1700, 1, 1, 128, 128, [5, 1695]),
])
@pytest.mark.parametrize('states', [True, False])
def test_segments(B, T, H, HV, K, V, lens, states, dtype):
    check(B, T, H, HV, K, V, DT[dtype], lens=lens, states=states)


def test_segments_with_gates_at_their_ends():
    def edit(x):
        x['beta'][:, ::3] = 0.0
        x['g'][:, 700] = float('-inf')
        x['g'][:, 511:513] = float('-inf')
        x['g'][:, 800:1400] = 0.0
    check(1, 1600, 1, 1, 128, 128, torch.bfloat16, edit=edit)


# ------------------------------------------------------------------------------------------------
# the exact path: key sizes around its shared-memory steps, and many heads (wider tiles of V)
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('K', [132, 149, 160, 176, 185, 188, 189, 224])
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_key_sizes_past_128(K, dtype):
    check(1, 70, 1, 1, K, 40, DT[dtype])


@pytest.mark.parametrize('B,T,H,HV,K,V,lens', [
    (3, 100, 26, 26, 64, 32, None),
    (2, 65, 10, 20, 160, 72, None),
    (1, 130, 8, 16, 33, 47, [1, 0, 64, 65]),
    (1, 40, 40, 80, 256, 8, None),
])
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_exact_path_with_many_heads(B, T, H, HV, K, V, lens, dtype):
    check(B, T, H, HV, K, V, DT[dtype], lens=lens, states=lens is None)
