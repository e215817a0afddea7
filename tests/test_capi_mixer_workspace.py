"""A workspace that does not start where the kernels' widest access needs it is refused before any launch, on every path."""
import pytest

from test_capi_mixer import P, gdr, lib  # noqa: F401

MANY = 1 << 40


@pytest.mark.parametrize('dtype', [0, 1, 2])
@pytest.mark.parametrize('at', [17, 20, 24])
def test_gdr_workspace_alignment(lib, dtype, at):  # noqa: F811
    a = gdr(dtype=dtype)
    bwd = (*a, P(16), None, P(16), P(16), P(16), P(16), P(16), None)
    for st in (lib.ccq_gdr_fwd(*a, P(16), None, P(at), MANY, None),
               lib.ccq_gdr_bwd(*bwd, P(at), MANY, None),
               lib.ccq_gdr_bwd_from(*bwd, P(16), P(at), MANY, None),
               lib.ccq_gdr_bwd_from(*bwd, P(at), P(16), MANY, None)):
        assert st == 1 and '16-byte aligned' in lib.ccq_last_error().decode()


def test_layer_norm_workspace_alignment(lib):  # noqa: F811
    st = lib.ccq_layer_norm_bwd(1, 0, 4, 64, P(16), None, None, None, None, P(16), P(16), None, P(16), None, None, None,
                                P(18), MANY, None)
    assert st == 1 and '4-byte aligned' in lib.ccq_last_error().decode()
