"""The gated delta rule through its C entry points where the forward's o is off a 16-byte boundary: the same path, the
same bits, and a workspace the backward can start from."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def lib():
    if not torch.cuda.is_available():
        pytest.skip('no CUDA device')
    from ccq_b200 import _lib
    return _lib.load()


@pytest.mark.parametrize('T,HV,V,lens', [(1, 2, 128, None), (64, 2, 128, None), (200, 4, 72, None), (131, 2, 256, [3, 0, 128])])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_unaligned_output(lib, T, HV, V, lens, dtype):
    from ccq_b200 import _lib
    from ccq_b200 import delta_rule as R
    gen = torch.Generator(device='cuda').manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=gen, device='cuda')  # noqa: E731
    B, H, K = (1 if lens else 2), 2, 128
    N = len(lens) if lens else B
    cu = torch.tensor([0] + lens, device='cuda').cumsum(0) if lens else None
    q, k = (torch.nn.functional.normalize(r(B, T, H, K), dim=-1).to(dtype) for _ in range(2))
    v, do, g, beta = r(B, T, HV, V).to(dtype), r(B, T, HV, V).to(dtype), -torch.rand(B, T, HV, device='cuda'), r(B, T, HV).sigmoid()
    head = R._head(q, k, v, g, beta, 0.1, cu, N, None)
    stream = torch.cuda.current_stream().cuda_stream
    outs = []
    for shift in (0, 1, 4):
        buf = torch.full((v.numel() + 16,), 7.0, dtype=dtype, device='cuda')
        fws, n = R._workspace(_lib.CCQ_OP_FWD, q, v, N, cu)
        _lib.check(lib.ccq_gdr_fwd(*head, buf[8 + shift:].data_ptr(), None, fws.data_ptr(), n, stream))
        assert _lib.last_path() == 'tcgen05'
        d = [torch.empty_like(t) for t in (q, k, v, g, beta)]
        ws, n = R._workspace(_lib.CCQ_OP_BWD, q, v, N, cu, True)
        _lib.check(lib.ccq_gdr_bwd_from(*head, do.data_ptr(), None, *(t.data_ptr() for t in d), None, fws.data_ptr(),
                                        ws.data_ptr(), n, stream))
        o = buf[8 + shift:8 + shift + v.numel()].reshape(v.shape)
        assert (buf[:8 + shift] == 7).all() and (buf[8 + shift + v.numel():] == 7).all()
        outs.append([o, *d])
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


@pytest.mark.parametrize('dtype,K,kept', [(torch.float32, 64, False), (torch.bfloat16, 136, False), (torch.bfloat16, 64, True)])
def test_only_a_workspace_the_backward_reads_is_kept(lib, dtype, K, kept):
    """Between forward and backward a call holds its inputs, o and, on the tensor-core path alone, the forward's
    workspace (on the exact path 268 bytes a token and head that nobody reads)."""
    import ccq_b200
    B, T, H, V = 1, 2048, 4, 64
    x = [torch.nn.functional.normalize(torch.randn(B, T, H, n, device='cuda'), dim=-1).to(dtype) for n in (K, K, V)]
    x = [t.requires_grad_(True) for t in (*x, -torch.rand(B, T, H, device='cuda'), torch.rand(B, T, H, device='cuda'))]
    before = torch.cuda.memory_allocated()
    o, _ = ccq_b200.gated_delta_rule(*x)
    more = torch.cuda.memory_allocated() - before - o.numel() * o.element_size()
    assert (more > 100 * B * T * H) == kept, more
    assert all(torch.isfinite(d).all() for d in torch.autograd.grad(o.float().sum(), x))
