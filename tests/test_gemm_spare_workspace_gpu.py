"""Products that are handed more device memory than they ask for: the tiles that need none leave it alone and give the result."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K,trans_b", [(384, 14336, 512, True), (384, 14336, 512, False), (1024, 4608, 640, True), (2048, 2496, 1024, False), (300, 1000, 768, True)])
def test_more_workspace_than_asked_for(M, N, K, trans_b):
    """A result is off by its rounding to bfloat16 (half a step, 2^-8) and K additions in fp32 at most."""
    from metalhlo_amd import _lib, kernels
    lib = _lib.load()
    rng = np.random.default_rng(M)
    a = torch.from_numpy(rng.standard_normal((M, K)).astype(np.float32)).to(torch.bfloat16).cuda()
    b = torch.from_numpy(rng.standard_normal((N, K) if trans_b else (K, N)).astype(np.float32)).to(torch.bfloat16).cuda()
    room = torch.full((64 << 20,), 0xA5, dtype=torch.uint8, device="cuda")
    c = torch.full((M, N), 7, dtype=torch.bfloat16, device="cuda")
    dt = kernels.DTYPE_CODE[a.dtype]
    asked = lib.mhip_gemm_workspace(M, N, K, 1, 0, int(trans_b), dt)
    assert asked < room.numel()
    _lib.check(lib.mhip_gemm_ws(torch.cuda.current_stream().cuda_stream, a.data_ptr(), b.data_ptr(), None, None, c.data_ptr(), M, N, K, 1, 0, 0, M * N, 0, int(trans_b), 0, dt, room.data_ptr(), room.numel()))
    w = b.double().t() if trans_b else b.double()
    want, size = a.double() @ w, a.double().abs() @ w.abs()
    assert ((c.double() - want).abs() <= 2.0 ** -8 * want.abs() + K * 2.0 ** -24 * size + 1e-30).all()
    assert (room[asked:] == 0xA5).all()
