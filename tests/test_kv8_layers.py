"""Layers on an 8-bit cache in the forms that a declaration may ask for: a cache that another layer wrote, interleaved and scaled rotations,
chunks, a sink, gates; and what such a layer refuses when it is built."""

from __future__ import annotations

import pytest
import torch

from test_kv8 import Cache, attend, i32, norm_rope, write
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


# ---- a layer alone, over steps as a model makes them ----

YARN = {"kind": "yarn", "factor": 4.0, "original": 64, "fast": 16.0, "slow": 2.0}
ROPE = {"kind": "rope", "params": {"head_dim": 64, "angles": 24, "theta": 1e4}}


def rotary(dim, dims, layout, scaling=None):
    return {"kind": "rotary", "params": {"head_dim": dim, "dims": dims, "base": 1e4, "layout": layout, "scaling": scaling}}


LAYERS = {
    "interleaved, yarn, window, sink, gate an element": dict(dim=64, position=rotary(64, 64, "interleaved", YARN), window=24, sink=True, gate="element"),
    "half, linear, partial, sink": dict(dim=128, position=rotary(128, 96, "half", {"kind": "linear", "factor": 3.0}), sink=True),
    "chunks, sink": dict(dim=64, position=rotary(64, 32, "interleaved"), chunk=20, sink=True),
    "chunks of a page, norms, gate a head": dict(dim=64, position=ROPE, norms=True, chunk=16, gate="head"),
    "chunks longer than any request": dict(dim=128, position=rotary(128, 128, "half"), chunk=1000),
    "norms, a factor of its own": dict(dim=64, position=ROPE, norms=True, scale=0.31, gate="element"),
}


def reference(layer_def, w, x, kv, pos):
    """One sequence's outputs in 64 bits: rows x [n, d] at positions pos over what the cache holds, kv [2, G, L, D]."""
    from tokenomos_b200.parts.rope import Rope, Rotary

    D, H, p = layer_def["dim"], 6, layer_def["position"]["params"]
    if layer_def["position"]["kind"] == "rope":
        freq, mult, inter = Rope(D, p["angles"], p["theta"], "cuda").inv_freq, 1.0, False
    else:
        freq, mult, inter = Rotary(D, p["dims"], p["base"], p["layout"], p["scaling"], "cuda").plain_rotation()
    q = (x.double() @ w["q"].double().T).view(-1, H, D)
    q = norm_rope(q, w.get("q_norm"), 1e-5, freq, pos, mult, inter)
    reach = -layer_def["chunk"] if layer_def.get("chunk") else layer_def.get("window")
    ones = torch.ones(kv.shape[1], kv.shape[2], device="cuda")
    o, _, _ = attend(q, kv, pos, reach, layer_def.get("scale") or D ** -0.5, ones, layer_def.get("sink", False))
    if "gate" in w:
        gate = torch.sigmoid(x.double() @ w["gate"].double().T)
        o = o * (gate[..., None] if layer_def["gate"] == "head" else gate.view(-1, H, D))
    return o.reshape(-1, H * D) @ w["o"].double().T


@gpu
@pytest.mark.parametrize("P", [16, 8, 12])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("name", LAYERS)
def test_layers_of_every_form_over_prompts_portions_and_tokens(name, dtype, P):
    """Built as a declaration builds them, on pools whose other pages are NaN. Against 64 bits over what the cache holds after the step's write, and the cache
    against the keys and values in 64 bits: half a step of e4m3 (2^-4) and a second rounding below its normal numbers (test_kv8), and in bfloat16 the projection's
    rounding, 2^-8 of an element, which norm and rotation spread over a pair. In 32 bits an output is off by sums of 48 to 768 products and a weight's 2^-18 at
    scores of up to 20: 2e-5 of the largest, as other layers' tests ask; in bfloat16 rows, weights and sums of rounded numbers: 3e-2."""
    from tokenomos_b200.cache.manager import CacheManager
    from tokenomos_b200.engine.step import StepEntry, StepFunction
    from tokenomos_b200.parts.attention import build_attention
    from tokenomos_b200.parts.registry import Runtime

    layer_def = LAYERS[name]
    H, G, D, d = 6, 2, layer_def["dim"], 48
    g = torch.Generator().manual_seed(P)
    w = {n: (torch.randn(rows, cols, generator=g) * cols ** -0.5).to(dtype).cuda() for n, rows, cols in (
        ("q", H * D, d), ("k", G * D, d), ("v", G * D, d), ("o", d, H * D))}
    if layer_def.get("norms"):
        w["q_norm"], w["k_norm"] = (torch.rand(2, D, generator=g) + 0.5).cuda()
    if "gate" in layer_def:
        w["gate"] = torch.randn(H if layer_def["gate"] == "head" else H * D, d, generator=g).to(dtype).cuda()
    params = {"heads": H, "kv_heads": G, "head_dim": D, "eps": 1e-5, "window": layer_def.get("window"), "chunk": layer_def.get("chunk"),
              "scale": layer_def.get("scale"), "sink": layer_def.get("sink", False), "gate_kind": layer_def.get("gate", "head"), "position": layer_def["position"]}
    layer = build_attention(params, dict(w), Runtime(dtype, torch.device("cuda"), cache8=True))
    specs = {(0, k): v for k, v in layer.state_specs().items()}
    cache = CacheManager(specs, P, 60, 4, dtype, "cuda", max_len=512, poison=True)
    step = StepFunction(type("M", (), {"vocab": 1 << 30}), cache)
    lens = {"a": [70, 1, 1, 30, 1], "b": [2, 40, 1, 1, 1], "c": [1, 1, 33, 1, 0]}
    for rid in lens:
        cache.admit(rid)
    done, rows = dict.fromkeys(lens, 0), {rid: torch.zeros(0, d, dtype=dtype, device="cuda") for rid in lens}
    tol = 2e-5 if dtype == torch.float32 else 3e-2
    for i in range(5):
        now = [(rid, n[i]) for rid, n in lens.items() if n[i]]
        ctx, _, _ = step.layout([StepEntry(rid, [0] * n, []) for rid, n in now])
        x = torch.randn(sum(n for _, n in now), d, generator=g).to(dtype).cuda()
        out = layer.forward(x, ctx, 0).double()
        at = 0
        for rid, n in now:
            xs, got = x[at:at + n], out[at:at + n]
            at += n
            rows[rid] = torch.cat((rows[rid], xs))
            end = done[rid] + n
            table = torch.tensor(cache.block_table(rid, specs[(0, "kv")].group), device="cuda")[:-(-end // P)]
            pool, scales = cache.states[(0, "kv")], cache.states[(0, "kv_scale")]
            kv = pool.view(torch.uint8)[table].view(torch.float8_e4m3fn).double() * scales[table].double()[..., None, None]
            kv = kv.permute(1, 2, 0, 3, 4).reshape(2, G, -1, D)[:, :, :end]
            want = reference(layer_def, w, xs, kv, torch.arange(done[rid], end, device="cuda"))
            assert torch.isfinite(got).all()
            assert (got - want).abs().max() <= tol * want.abs().max(), (rid, i, ((got - want).abs().max() / want.abs().max()).item())
            # the cached values of the pages that are still held
            v = (rows[rid].double() @ w["v"].double().T).view(-1, G, D).permute(1, 0, 2)
            per = scales[table, 1].double().t().repeat_interleave(P, 1)[:, :end, None]
            held = table.repeat_interleave(P)[:end] > 0
            off = (kv[1] - v).abs() <= v.abs() * (2.0 ** -4 + (2.0 ** -8 if dtype == torch.bfloat16 else 0)) * (1 + 2.0 ** -10) + per * 2.0 ** -9 + v.abs().max() * 2.0 ** -18
            assert off[:, held].all()
            done[rid] = end
            cache.commit(rid, n)
            cache.check()


# ---- a model whose mixers have a sink, scaled rotations and a gate an element ----

@pytest.fixture(scope="module")
def darizen(tmp_path_factory):
    import part_rig
    from test_darizen import att2, make_tensors, mlp

    config = {"architecture": "Darizen", "vocab": 300, "width": 96, "norm": {"eps": 1e-5},
              "layers": [dict(att2(6, 2, 64, 64, 40, factor=4.0), mlp=mlp(96, 1.5)), dict(att2(4, 1, 128, 128, 500, dims=64), mlp=mlp(80, 1.5))],
              "loop": {"start": 0, "stop": 1, "times": 2}}
    tensors = make_tensors(config, 21)
    for name in tensors:
        if name.endswith((".mix.q", ".mix.k")):          # (scores of about one: a number next to the middle of two e4m3 ones moves little)
            tensors[name] = (tensors[name].float() * 0.4).to(torch.bfloat16)
    folder = tmp_path_factory.mktemp("kv8_darizen")
    part_rig.write_folder(folder, config, tensors)
    return config, {k: v.double() for k, v in tensors.items()}, folder


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("page", [16, 12])
def test_darizen_on_an_8_bit_cache_however_its_tokens_are_cut(darizen, dtype, page, monkeypatch):
    """The bounds are those of ``test_kv8_model``: in 32 bits a few of 10^5 cached numbers next to the middle of two e4m3 ones, in bfloat16 the 16-bit cache's
    error and what rounding keys and values moves the oracle's logits by."""
    import plain_darizen as plain
    import trace_util
    from test_kv8_model import TOL_F32, engine_of, replay, round8

    config, w, folder = darizen
    g = torch.Generator().manual_seed(3)
    requests = {f"r{i}": torch.randint(0, config["vocab"], (n,), generator=g).tolist() for i, n in enumerate((2, 31, 150, 65, 200, 90))}
    unrounded = {rid: plain.forward(config, w, ids)[0] for rid, ids in requests.items()}
    attention64 = plain.sink_softmax_attention
    monkeypatch.setattr(plain, "sink_softmax_attention", lambda q, k, v, scale, mask: attention64(q, round8(k, page), round8(v, page), scale, mask))
    want = {rid: plain.forward(config, w, ids)[0] for rid, ids in requests.items()}
    mixed = trace_util.mixed(requests, live=4, seed=7)
    pages = -(-max(trace_util.max_live_tokens(mixed, page), 200 + page) // page) + 3
    for name, steps in (("mixed", mixed), ("tail", trace_util.tail_decoded(requests, 32))):
        got = replay(*engine_of(folder, dtype, page, pages)[:0:-1], steps)
        wide = replay(*engine_of(folder, dtype, page, pages, kind=None)[:0:-1], steps) if dtype == "bfloat16" else None
        for rid, ref in want.items():
            err, bound = (got[rid] - ref).abs().max(), TOL_F32 * ref.abs().max()
            if wide is not None:
                bound = (wide[rid] - unrounded[rid]).abs().max() + (ref - unrounded[rid]).abs().max()
            assert torch.isfinite(got[rid]).all() and err <= bound, (name, rid, (err / ref.abs().max()).item(), (bound / ref.abs().max()).item())


@gpu
def test_darizen_generates_on_an_8_bit_cache_with_and_without_graphs(darizen):
    """Recorded and eager steps cut the same tokens alike: the same replies. (The same kernels, sizes and bits.)"""
    from tokenomos_b200 import LLM, SamplingParams

    _, _, folder = darizen
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 300, (n,), generator=g).tolist() for n in (37, 5, 64, 18, 51)]
    for prompt in prompts:
        outs = []
        for graphs in (False, True):
            with LLM(str(folder), graphs=graphs, work="fp32", cache="fp8", page=16, max_len=128, slots=2, pages=20, poison=True) as llm:
                outs.append(llm.generate([prompt], SamplingParams(max_tokens=12))[0].token_ids)
        assert outs[0] == outs[1] and len(outs[0]) == 12


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
