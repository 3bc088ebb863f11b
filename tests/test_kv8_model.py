"""Models on an 8-bit cache through the framework's own entry points: trace replay however the tokens are cut, generation through
eager and recorded steps, against the plain implementation with its keys and values rounded the same way; and what has no 8-bit form."""

from __future__ import annotations

import pytest
import torch

import plain_lfm3
import trace_util
from conftest import TINY, TINY_D

gpu = pytest.mark.gpu

# heads of 128, a window and a partial rotation, the per-head gate, sandwich norms, pages that are no power of two
TINY_E = {
    "architectures": ["Lfm3ForCausalLM"], "hidden_size": 96, "num_hidden_layers": 4,
    "layer_types": ["sliding_attention", "conv", "full_attention", "sliding_attention"],
    "num_attention_heads": 6, "num_key_value_heads": 2, "head_dim": 128,
    "intermediate_size": 112, "vocab_size": 300, "norm_eps": 1e-5, "conv_L_cache": 2,
    "conv_bias": True, "tie_word_embeddings": True, "sliding_window": 21,
    "use_sandwich_norm": True, "attention_gate": True,
    "rope_parameters": {
        "full_attention": {"rope_type": "default", "rope_theta": 50000.0},
        "sliding_attention": {"rope_type": "default", "rope_theta": 10000.0, "partial_rotary_factor": 0.5},
    },
}
CASES = {"D16": (TINY_D, 16, 0.06), "D64": (TINY_D, 64, 0.06), "E12": (TINY_E, 12, 0.07), "E16": (TINY_E, 16, 0.07)}

# Of the largest |logit|, in 32-bit. The oracle rounds the same numbers to e4m3 as the engine, formed in 64 bits: a number next to the middle of two e4m3
# ones may go to the other, a step of 2^-3 of it. That is one number in about 2^17 (2^-21 of error in a number against its step), a few of the
# 10^5 cached here, each 2^-3 of one of 64 or 128 terms of a score or one of a hundred of an output.
TOL_F32 = 5e-3
# In bfloat16 a model's logits are off by what its 16-bit activations do (E: as much as the 16-bit cache's engine is, which the test measures beside it),
# and the numbers that are rounded to e4m3 differ by d = 2^-9 or a few: a share d / step of them, 2^-9 / 2^-3 to 2^-7 / 2^-3, goes one step the other
# way. That noise's variance is at most step^2 / 16 against the rounding's own step^2 / 12, and it enters the logits the same way, so it is no more
# than what rounding keys and values moves the oracle's logits by. Hence the bound: the 16-bit cache's error plus that.


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    from tokenomos_b200.weights import write_model_folder

    out = {}
    for name, config in (("D", TINY_D), ("E", TINY_E)):
        out[name] = tmp_path_factory.mktemp(f"kv8_{name}")
        write_model_folder(out[name], config, 5, CASES[f"{name}16"][2], 0.1, torch.bfloat16)
    return out


def round8(x: torch.Tensor, page: int) -> torch.Tensor:
    """x [T, heads, D] as the 8-bit cache holds it: e4m3 of x / s, s the smallest power of two with which the block's largest is at most
    448 (a block: the positions of a page, one head)."""
    out = x.clone()
    for a in range(0, x.shape[0], page):
        block = x[a:a + page]
        s = torch.exp2(torch.ceil(torch.log2(block.abs().amax((0, 2), keepdim=True) / 448)).clamp(-40, 40))
        y = block / s
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        out[a:a + page] = torch.round(y / step) * step * s
    return out


def attention8(page):
    """``plain_lfm3.attention`` over keys and values rounded to 8 bits."""
    def fn(x, w, prefix, s, kind, dtype):
        T, H, G, D = x.shape[0], s["heads"], s["kv_heads"], s["head_dim"]
        q, k, v = ((x @ w[f"{prefix}{n}_proj.weight"].to(dtype).T).view(T, h, D) for n, h in (("q", H), ("k", G), ("v", G)))
        q = plain_lfm3.rmsnorm(q, w[f"{prefix}q_norm.weight"], s["eps"])
        k = plain_lfm3.rmsnorm(k, w[f"{prefix}k_norm.weight"], s["eps"])
        theta, angles = s["ropes"][kind]
        cos, sin = plain_lfm3.rope_tables(torch.arange(T), D, angles, theta, dtype)
        q, k = plain_lfm3.rotate(q, cos, sin), plain_lfm3.rotate(k, cos, sin)
        k, v = (round8(t, page).repeat_interleave(H // G, 1) for t in (k, v))
        i = torch.arange(T)
        see = i[None] <= i[:, None]
        if kind == "sliding_attention":
            see = see & (i[:, None] - i[None] < s["window"])
        p = torch.softmax((torch.einsum("ihd,jhd->hij", q, k) * D ** -0.5).masked_fill(~see, float("-inf")), -1)
        out = torch.einsum("hij,jhd->ihd", p, v)
        if f"{prefix}gate_proj.weight" in w:
            out = out * torch.sigmoid(x @ w[f"{prefix}gate_proj.weight"].to(dtype).T)[..., None]
        return out.reshape(T, H * D) @ w[f"{prefix}o_proj.weight"].to(dtype).T
    return fn


def engine_of(folder, dtype, page, pages, slots=6, kind="fp8"):
    from tokenomos_b200 import models
    from tokenomos_b200.cache.manager import CacheManager
    from tokenomos_b200.engine.step import StepFunction

    conf = models.configure(folder, work=dtype, cache=kind)
    model = models.load(folder, "cuda", conf)
    cache = CacheManager(model.state_specs(), page, pages, slots, conf.work, "cuda", max_len=(pages - 1) * page, poison=True)
    return model, cache, StepFunction(model, cache)


def replay(step_fn, cache, steps):
    from tokenomos_b200.engine.step import StepEntry

    out = {}
    for s in steps:
        for e in s["entries"]:
            if e["id"] not in cache.requests:
                cache.admit(e["id"])
        logits = step_fn.run([StepEntry(e["id"], e["tokens"], e["want"]) for e in s["entries"]])
        if logits is not None:
            out[s["step"]] = logits.double().cpu()
        for rid in s["end"]:
            cache.release(rid)
        cache.check()
    return trace_util.collect(steps, out)


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("case", CASES)
def test_replay_however_the_tokens_are_cut(case, dtype, folders, monkeypatch):
    config, page, _ = CASES[case]
    folder = folders[case[0]]
    g = torch.Generator().manual_seed(3)
    requests = {f"r{i}": torch.randint(0, config["vocab_size"], (n,), generator=g).tolist() for i, n in enumerate((2, 31, 150, 65, 200, 90))}
    conf, w = plain_lfm3.read_folder(folder)
    unrounded = {rid: plain_lfm3.forward_logits(conf, w, ids) for rid, ids in requests.items()}
    monkeypatch.setattr(plain_lfm3, "attention", attention8(page))
    want = {rid: plain_lfm3.forward_logits(conf, w, ids) for rid, ids in requests.items()}
    mixed = trace_util.mixed(requests, live=4, seed=7)
    pages = -(-max(trace_util.max_live_tokens(mixed, page), 200 + page) // page) + 3
    for name, steps in (("mixed", mixed), ("tail", trace_util.tail_decoded(requests, 32))):
        model, cache, step_fn = engine_of(folder, dtype, page, pages)
        got = replay(step_fn, cache, steps)
        wide = replay(*engine_of(folder, dtype, page, pages, kind=None)[:0:-1], steps) if dtype == "bfloat16" else None
        for rid, ref in want.items():
            assert torch.isfinite(got[rid]).all(), (name, rid)
            err = (got[rid] - ref).abs().max()
            bound = TOL_F32 * ref.abs().max()
            if wide is not None:
                bound = (wide[rid] - unrounded[rid]).abs().max() + (ref - unrounded[rid]).abs().max()
            assert err <= bound, (name, rid, (err / ref.abs().max()).item(), (bound / ref.abs().max()).item())


@gpu
@pytest.mark.parametrize("case", ["D16", "E16"])
def test_generation_through_recorded_and_eager_steps(case, folders, monkeypatch):
    """The same prompts through eager steps, recorded mixed steps and recorded decode steps: every greedy token is the rounded oracle's best
    given the same history, or within the noise of its logits (what rounding keys and values moves them by, twice: two logits are compared)."""
    from tokenomos_b200 import LLM, SamplingParams

    config, page, _ = CASES[case]
    folder = folders[case[0]]
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, config["vocab_size"], (n,), generator=g).tolist() for n in (37, 5, 64, 18, 51, 9, 70, 26)]
    conf, w = plain_lfm3.read_folder(folder)
    plain_attention = plain_lfm3.attention
    kw = dict(work="bf16", cache="fp8", page=page, max_len=128, slots=5, pages=60, prefill_budget=24, poison=True)
    for graphs in (False, True):
        with LLM(str(folder), graphs=graphs, **kw) as llm:
            assert llm.engine.cache.states[(0, "kv")].dtype == torch.float8_e4m3fn
            llm.engine.step_fn.capture_after = 0
            outs = llm.generate(prompts, SamplingParams(max_tokens=16))
            assert not graphs or llm.engine.stats.graph_steps > 5
            llm.engine.cache.check()
        for prompt, out in zip(prompts, outs):
            monkeypatch.setattr(plain_lfm3, "attention", plain_attention)
            unrounded = plain_lfm3.forward_logits(conf, w, prompt + out.token_ids)
            monkeypatch.setattr(plain_lfm3, "attention", attention8(page))
            logits = plain_lfm3.forward_logits(conf, w, prompt + out.token_ids)
            noise = (logits - unrounded).abs().max() + 0.03 * logits.abs().max()
            for i, tok in enumerate(out.token_ids):
                row = logits[len(prompt) + i - 1]
                assert row.max() - row[tok] <= 2 * noise, (graphs, i)


@gpu
def test_an_8_bit_page_costs_half_and_a_little(folders):
    from tokenomos_b200 import models
    from tokenomos_b200.cache.manager import CacheManager

    size = {}
    for kind in (None, "fp8"):
        model = models.load(folders["D"], "cuda", models.configure(folders["D"], cache=kind))
        size[kind] = CacheManager(model.state_specs(), 16, 8, 2, torch.bfloat16, "meta").bytes_per_page()
    # a byte instead of two for each element, and four for each block of 16 x 64
    assert size["fp8"] == size[None] // 2 + size[None] // 2 // (16 * 64) * 4


def test_models_and_layers_without_an_8_bit_form_are_refused(tmp_path):
    from tokenomos_b200 import models
    from tokenomos_b200.weights import write_model_folder

    folder = tmp_path / "a"
    write_model_folder(folder, TINY["A"]["config"], 0, 0.02, 0.0, torch.bfloat16)        # heads of 16
    with pytest.raises(ValueError, match="heads of 64 or 128"):
        models.load(folder, "cpu", models.configure(folder, cache="fp8"))
    with pytest.raises(ValueError, match="known"):
        models.configure(folder, cache="int4")


def test_a_cache_type_beside_a_configured_model_is_refused(tmp_path):
    from tokenomos_b200 import LLM, models
    from tokenomos_b200.weights import write_model_folder

    write_model_folder(tmp_path / "d", TINY_D, 0, 0.02, 0.0, torch.bfloat16)
    with pytest.raises(ValueError, match="configured already"):
        LLM(tmp_path / "d", "cpu", models.configure(tmp_path / "d"), cache="fp8")


@pytest.mark.parametrize("option, value", [("keep_first", 2), ("v_is_k", True), ("v_dim", 32), ("pointwise", {}), ("value_mix", {"source": None})])
def test_attention_options_without_an_8_bit_form_are_refused(option, value):
    from tokenomos_b200.parts.attention import build_attention
    from tokenomos_b200.parts.registry import Runtime

    params = {"heads": 2, "kv_heads": 1, "head_dim": 64, "window": 8,
              "position": {"kind": "rotary", "params": {"head_dim": 64, "dims": 64, "base": 1e4, "layout": "half"}}, option: value}
    v = 64 if option != "v_dim" else 32
    tensors = {"q": torch.zeros(128, 32), "k": torch.zeros(64, 32), "v": torch.zeros(v, 32), "o": torch.zeros(32, 2 * v)}
    if option == "v_is_k":
        del tensors["v"]
    with pytest.raises(ValueError, match="8-bit cache|position part"):
        build_attention(params, tensors, Runtime(torch.float32, torch.device("cpu"), cache8=True))


def test_a_mixer_that_keeps_latents_is_refused():
    """(A model whose layers keep a paged state of another kind says so when it is built.)"""
    from tokenomos_b200.parts import build as b
    from tokenomos_b200.parts.contract import BlockScales, LatentKV, PagedKV
    from tokenomos_b200.parts.registry import Runtime

    class Stack:
        def __init__(self, specs):
            self.specs = specs

        def state_specs(self):
            return self.specs

    kv = PagedKV(1, 64, torch.float8_e4m3fn)
    b.check_cache8(Stack({(0, "kv"): kv, (0, "kv_scale"): BlockScales(kv)}), Runtime(torch.float32, torch.device("cpu"), cache8=True))
    with pytest.raises(ValueError, match="no 8-bit form"):
        b.check_cache8(Stack({(0, "kv"): LatentKV(80)}), Runtime(torch.float32, torch.device("cpu"), cache8=True))
    b.check_cache8(Stack({(0, "kv"): LatentKV(80)}), Runtime(torch.float32, torch.device("cpu")))


CHECKED = """
import sys
sys.path.insert(0, "tests")
import torch
import test_kv8_model, trace_util
from tokenomos_b200 import ops
folder, dtype = sys.argv[1], sys.argv[2]
assert ops.checks_enabled()
g = torch.Generator().manual_seed(3)
reqs = {f"r{i}": torch.randint(0, 400, (n,), generator=g).tolist() for i, n in enumerate((2, 31, 150, 65, 200))}
steps = trace_util.mixed(reqs, live=4, seed=7)
pages = -(-trace_util.max_live_tokens(steps, 16) // 16) + 1
got = test_kv8_model.replay(*test_kv8_model.engine_of(folder, dtype, 16, pages)[:0:-1], steps)
assert all(torch.isfinite(v).all() for v in got.values())
assert ops.checks_status() is None, ops.checks_status()
print("clean")
"""


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_replay_under_the_index_checks_finds_nothing(dtype, folders):
    from test_checks import run_checked

    assert run_checked(CHECKED, str(folders["D"]), dtype).startswith("clean")
