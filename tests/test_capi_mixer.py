"""The C entry points of the gated delta rule and of layer norm refuse bad arguments before touching a GPU."""
import ctypes

import pytest


@pytest.fixture(scope='module')
def lib():
    from ccq_b200 import _lib
    from ccq_b200.build import build
    build()
    return _lib.load()


def P(x):
    return None if x is None else ctypes.c_void_p(x)


def gdr(dtype=1, B=2, T=8, H=2, HV=4, K=64, V=64, q=16, v=16, g=16, g_dtype=0, cu=None, n=2):
    return (dtype, B, T, H, HV, K, V, P(q), P(16), P(v), g_dtype, P(g), 0, P(16), 1.0, P(cu), n, None)


@pytest.mark.parametrize('kw,status,msg', [
    (dict(dtype=7), 1, 'dtype'),
    (dict(g_dtype=5), 1, 'gate dtypes'),
    (dict(V=0), 1, 'bad sizes'),
    (dict(HV=3), 1, 'multiple'),
    (dict(K=257), 2, 'K=257'),
    (dict(V=70000), 2, 'V=70000'),
    (dict(g=None), 1, 'required'),
    (dict(v=None), 1, 'required'),
    (dict(n=3), 1, 'n_seqs'),
    (dict(cu=64), 1, 'B == 1'),
])
def test_gdr_refusals(lib, kw, status, msg):
    a = gdr(**kw)
    for st in (lib.ccq_gdr_fwd(*a, P(16), None, None, 0, None),
               lib.ccq_gdr_bwd(*a, P(16), None, P(16), P(16), P(16), P(16), P(16), None, None, 0, None),
               lib.ccq_gdr_step(*a, P(16), P(16), None)):
        assert st == status
        assert msg in lib.ccq_last_error().decode()


def test_gdr_outputs_and_workspace(lib):
    need = lib.ccq_gdr_workspace_size(0, 1, 2, 8, 2, 4, 64, 64, 2, 0)
    assert need > 0
    assert lib.ccq_gdr_fwd(*gdr(), None, None, P(16), need, None) == 1
    assert lib.ccq_gdr_fwd(*gdr(), P(16), None, P(16), need - 1, None) == 4
    assert 'workspace' in lib.ccq_last_error().decode()
    assert lib.ccq_gdr_bwd(*gdr(), P(16), None, P(16), None, P(16), P(16), P(16), None, P(16), 1 << 40, None) == 1
    assert lib.ccq_gdr_bwd(*gdr(), P(16), None, P(16), P(16), P(16), P(16), P(16), None, P(16), 64, None) == 4
    assert lib.ccq_gdr_step(*gdr(), None, P(16), None) == 1
    assert 'state_out' in lib.ccq_last_error().decode()
    assert lib.ccq_gdr_workspace_size(0, 1, 2, 8, 2, 4, 300, 64, 2, 0) == 0


@pytest.mark.parametrize('kw,status,msg', [
    (dict(dtype=4), 1, 'dtype'),
    (dict(form=2), 1, 'form'),
    (dict(D=0), 1, 'bad sizes'),
    (dict(D=16385), 2, 'D=16385'),
    (dict(eps=-1.0), 1, 'eps'),
    (dict(x=None), 1, 'x is required'),
    (dict(y=None), 1, 'y is required'),
    (dict(residual=16), 1, 'h is required'),
    (dict(stats=20), 1, 'aligned'),
])
def test_layer_norm_refusals(lib, kw, status, msg):
    a = dict(dtype=1, form=0, rows=4, D=64, eps=1e-5, x=16, residual=None, y=16, stats=None)
    a.update(kw)
    st = lib.ccq_layer_norm_fwd(a['dtype'], a['form'], a['rows'], a['D'], a['eps'], P(a['x']), P(a['residual']), None,
                                None, None, P(a['y']), None, P(a['stats']), None)
    assert st == status and msg in lib.ccq_last_error().decode()


def test_layer_norm_bwd_refusals(lib):
    need = lib.ccq_layer_norm_workspace_size(1, 4, 64)
    assert need > 0 and lib.ccq_layer_norm_workspace_size(0, 4, 64) == 0
    args = lambda stats=16, gate=None, ws=16, n=need: (  # noqa: E731
        1, 0, 4, 64, P(16), None, None, None, P(gate), P(stats), P(16), None, P(16), None, None, None, P(ws), n, None)
    assert lib.ccq_layer_norm_bwd(*args(stats=None)) == 1
    assert lib.ccq_layer_norm_bwd(*args(gate=16)) == 1 and 'dgate' in lib.ccq_last_error().decode()
    assert lib.ccq_layer_norm_bwd(*args(n=need - 1)) == 4
    assert lib.ccq_layer_norm_bwd(*args(ws=None)) == 4


def test_layer_norm_combinations(lib):
    need = lib.ccq_layer_norm_workspace_size(1, 4, 64)
    for form, residual, bias, gate in ((1, None, 16, None), (0, None, None, 16), (1, 16, None, 16)):
        st = lib.ccq_layer_norm_fwd(1, form, 4, 64, 1e-5, P(16), P(residual), None, P(bias), P(gate), P(16), P(16), None, None)
        assert st == 2 and lib.ccq_last_error()
        st = lib.ccq_layer_norm_bwd(1, form, 4, 64, P(16), P(residual), None, P(bias), P(gate), P(16), P(16), None, P(16), P(16),
                                    None, None, P(16), need, None)
        assert st == 2 and lib.ccq_last_error()


def test_gdr_workspace_flags(lib):
    size = lambda op, flags: lib.ccq_gdr_workspace_size(op, 1, 1, 1000, 2, 4, 128, 128, 1, flags)  # noqa: E731
    assert size(0, 1) > 0 and size(1, 0) > size(1, 2) > 0       # without the forward's workspace the backward needs more
    assert size(1, 4) > 0 and size(0, 4) != size(0, 0)          # an unaligned call takes the exact path
