"""The 8-bit cache's operators at the calls that are easily missed: operands that lie where nobody expects them, numbers at the ends of
their range, weights that are small beside their row's largest."""

from __future__ import annotations

import pytest
import torch

from test_kv8 import Cache, write

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [3, 600])
@pytest.mark.parametrize("D", [64, 128])
def test_norm_weights_may_begin_at_any_float(D, T, dtype):
    """Contiguous float32 vectors 4, 8 and 12 bytes behind a 16-byte address: the same bits as from vectors of their own."""
    G, H, P = 2, 4, 16
    g = torch.Generator().manual_seed(D + T)
    x = torch.randn(T, (H + 2 * G) * D, generator=g).to(dtype).cuda()
    w = (torch.rand(2, D, generator=g) + 0.5).cuda()
    freq = torch.exp(-torch.arange(D // 2) * 0.2).cuda()
    want = Cache([T], G, D, P)
    q, _ = write(want, [(0, 0, x)], H, w[0].clone(), w[1].clone(), 1e-6, freq)
    for at_q, at_k in ((1, 0), (0, 3), (2, 1)):
        wide = torch.zeros(2, D + 4, device="cuda")
        wq, wk = wide[0, at_q:at_q + D], wide[1, at_k:at_k + D]
        wq.copy_(w[0])
        wk.copy_(w[1])
        got = Cache([T], G, D, P)
        q2, _ = write(got, [(0, 0, x)], H, wq, wk, 1e-6, freq)
        assert torch.equal(q, q2) and torch.equal(got.scales.view(torch.int32), want.scales.view(torch.int32))
        assert torch.equal(got.pool.view(torch.uint8), want.pool.view(torch.uint8))
