"""The gated delta rule's path is the same in a forward and in the backward that reads its workspace: it does not
depend on the forward's o, nor on the environment once a call has been made.  Decided on the host, before any launch."""
import pytest

from test_capi_mixer import P, gdr, lib  # noqa: F401

SIZES = (1, 2, 8, 2, 4, 64, 64, 2)  # dtype, B, T, H, HV, K, V, n_seqs of gdr()


def size(lib, op, flags=0):  # noqa: F811
    return lib.ccq_gdr_workspace_size(op, *SIZES, flags)


@pytest.mark.parametrize('o', [16, 18, 24])
def test_output_alignment_does_not_choose_the_path(lib, o):  # noqa: F811
    """Whatever o is, the forward asks for the tensor-core path's workspace, which is what the backward reads."""
    need = size(lib, 0)
    assert lib.ccq_gdr_fwd(*gdr(), P(o), None, P(16), need - 1, None) == 4
    assert f'{need} bytes' in lib.ccq_last_error().decode()


def test_environment_does_not_change_the_path(lib, monkeypatch):  # noqa: F811
    sizes = [size(lib, op) for op in (0, 1)]
    monkeypatch.setenv('CCQ_B200_FORCE_SIMT', '1')
    assert [size(lib, op) for op in (0, 1)] == sizes


def test_unaligned_size_is_enough_for_either_path(lib):  # noqa: F811
    for op in (0, 1):
        assert size(lib, op, 4) > size(lib, op)
