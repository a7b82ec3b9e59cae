"""The GEMM that dequantises inside the CTA pairs gives the same bits each time, and those of the weight panel's
form, which has no dequantising warps: its rows are sums of the same products in the same order."""
import pytest
import torch

from mes_b200 import _C
from oracle import awq as oawq

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _weights(K, N):
    qw, qz, sc = oawq.random_awq(K, N, seed=K + N)
    return _C.awq_repack(torch.from_numpy(qw).to(DEV)), torch.from_numpy(qz).to(DEV), torch.from_numpy(sc).view(torch.int16).to(DEV)


@pytest.mark.parametrize("M,K,N", [(5000, 1024, 6144), (1300, 3584, 512), (300, 4096, 6144), (1000, 1024, 2048), (700, 8960, 1536)])
def test_fused_pair_repeats(M, K, N):
    w = _weights(K, N)
    panel = torch.empty(N, K, dtype=torch.bfloat16, device=DEV)
    _C.awq_panels([w], [panel])
    g = torch.Generator().manual_seed(M)
    x = torch.randn(max(M, 1300), K, generator=g).to(torch.bfloat16).to(DEV)
    # above 1024 rows this takes the panel, whose rows do not depend on the batch
    want = torch.zeros(x.shape[0], N, device=DEV)
    _C.awq_gemm_residual(x, *w, want, panel=panel)
    want = want[:M]
    if M > 1024:
        _C.use_gemm_workspace = False
    try:
        for i in range(60):
            got = torch.zeros(M, N, device=DEV)
            _C.awq_gemm_residual(x[:M], *w, got)
            assert torch.equal(got, want), i
    finally:
        _C.use_gemm_workspace = True
    assert _C.take_device_error() == 0
