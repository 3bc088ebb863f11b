"""Layers on an 8-bit cache in the forms that a declaration may ask for: a cache that another layer wrote, interleaved and scaled rotations,
chunks, a sink, gates; and what such a layer refuses when it is built."""

from __future__ import annotations

import pytest
import torch

from test_kv8 import Cache, i32, write
from tokenomos_b200 import ops
from tokenomos_b200.ops import KernelError

gpu = pytest.mark.gpu


def attention(H, G, D, d, rope, norms=None, source=None, seed=0, dtype=torch.bfloat16, device="cuda", **kw):
    """An attention layer with random weights on an 8-bit cache (``source``: on that entry's)."""
    from tokenomos_b200.parts.attention import Attention
    from tokenomos_b200.parts.linear import Linear

    g = torch.Generator().manual_seed(seed)
    wq, wk, wv, wo = ((torch.randn(n, m, generator=g) * m ** -0.5).to(dtype).to(device) for n, m in ((H * D, d), (G * D, d), (G * D, d), (d, H * D)))
    qn, kn = norms if norms is not None else (None, None)
    mats = [wq] if source is not None else [wq, wk, wv]
    return Attention(Linear.fused(mats), Linear(wo), H, G, D, rope, 1e-5, qn, kn if source is None else None, kv_source=source, cache8=True, **kw)


# ---- a cache that another layer wrote ----

@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D, R, interleaved, norm, start", [(64, 64, False, True, 0), (128, 20, False, False, 0), (64, 32, True, True, 90000), (128, 128, False, True, 31000)])
def test_queries_without_keys_are_the_queries_of_the_whole_write(dtype, D, R, interleaved, norm, start):
    H, G, P = 6, 2, 16
    g = torch.Generator().manual_seed(D + R)
    w = (torch.rand(2, D, generator=g) + 0.5).cuda() if norm else (None, None)
    freq = torch.exp(-torch.arange(R // 2) * 0.3).cuda()
    for T in (1, 5, 700):
        x = torch.randn(T, (H + 2 * G) * D, generator=g).to(dtype).cuda()
        cache = Cache([T], G, D, P)
        wide = torch.zeros(1, (start + T) // P + 2, dtype=torch.int32)
        wide[0, start // P:start // P + cache.table.shape[1]] = cache.table[0]
        wide[0, start // P + cache.table.shape[1]:] = cache.table[0, -1]
        cache.table_dev = wide.cuda()
        want, pos = write(cache, [(0, start, x)], H, w[0], w[1], 1e-6, freq, 1.25, interleaved)
        rows = x[:, :H * D]
        for qkv in (rows, rows.contiguous()):
            got = ops.qk_norm_rope_write8(qkv, None, None, w[0], None, 1e-6, freq, pos, pos, None, H, 0, D, P, 1.25, interleaved)
            assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("position", ["rope", "interleaved"])
def test_a_layer_that_reads_another_ones_cache_asks_as_that_one_does(position, dtype):
    """Two layers of the same query weights over one cache: the same bits, in a prompt, a portion behind it and single tokens."""
    from test_parts import _ctx_for
    from tokenomos_b200.engine.step import StepEntry
    from tokenomos_b200.parts.contract import SharedState
    from tokenomos_b200.parts.rope import Rope, Rotary

    H, G, D, d = 4, 2, 64, 48
    if position == "rope":
        rope, norms = Rope(D, D // 2, 1e4, "cuda"), tuple((torch.rand(2, D) + 0.5).cuda())
    else:
        rope, norms = Rotary(D, 48, 1e4, "interleaved", {"kind": "yarn", "factor": 4.0, "original": 64, "fast": 16.0, "slow": 2.0}, "cuda"), None
    owner, reader = (attention(H, G, D, d, rope, norms, source, seed=3, dtype=dtype) for source in (None, 0))
    assert reader.state_specs() == {"kv": SharedState(0, "kv"), "kv_scale": SharedState(0, "kv_scale")}
    specs = {(i, name): s for i, layer in enumerate((owner, reader)) for name, s in layer.state_specs().items()}
    ctx, cache, step = _ctx_for(specs, 16, [70, 2, 1], dtype)
    for n in (73, 31, 3):
        x = torch.randn(n, d).to(dtype).cuda()
        want = owner.forward(x, ctx, 0)
        assert torch.isfinite(want).all() and want.abs().max() > 0
        assert torch.equal(reader.forward(x, ctx, 1), want)
        for rid, m in zip((0, 1, 2), {73: (70, 2, 1), 31: (1, 29, 1), 3: (1, 1, 1)}[n]):
            cache.commit(rid, m)
        if n != 3:
            ctx, _, _ = step.layout([StepEntry(rid, [0] * m, []) for rid, m in zip((0, 1, 2), {73: (1, 29, 1), 31: (1, 1, 1)}[n])])


@gpu
def test_keys_without_a_cache_are_refused():
    x, f, one = torch.zeros(1, 4 * 64, device="cuda"), torch.zeros(0, device="cuda"), i32([0])
    with pytest.raises(KernelError, match="need a cache"):
        ops.qk_norm_rope_write8(x, None, None, None, None, 0.0, f, one, one, None, 2, 1, 64, 16)
    with pytest.raises(KernelError, match="shorter"):
        ops.qk_norm_rope_write8(x, None, None, None, None, 0.0, f, one[:0], one, None, 4, 0, 64, 16)


# ---- what is refused when a layer is built ----

@pytest.mark.parametrize("scale", [0.0, -0.125, float("nan")])
def test_a_factor_of_the_scores_that_is_not_positive_is_refused(scale):
    from tokenomos_b200.parts.rope import Rope

    rope = Rope(64, 32, 1e4, "cpu")
    assert attention(4, 2, 64, 16, rope, device="cpu", scale=0.5).scale == 0.5
    with pytest.raises(ValueError, match="positive"):
        attention(4, 2, 64, 16, rope, device="cpu", scale=scale)


@pytest.mark.parametrize("which", ["q", "k", "both"])
def test_rotary_refuses_norms_over_either_cache(which):
    """(Nothing is launched: the check comes first.)"""
    from tokenomos_b200.parts.contract import HeadLayout
    from tokenomos_b200.parts.rope import Rotary

    w = torch.ones(64)
    heads = HeadLayout(4, 2, 64, w if which != "k" else None, w if which != "q" else None, 1e-5)
    rotary = Rotary(64, 64, 1e4, "half", None, "cpu")
    with pytest.raises(ValueError, match="norms"):
        rotary.encode_qk(torch.zeros(1, 8 * 64), None, heads, None, None)
    with pytest.raises(ValueError, match="norms"):
        rotary.encode_qk8(torch.zeros(1, 8 * 64), None, heads, None, None, None)
