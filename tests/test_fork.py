"""Several replies of one prompt: forks in the cache manager's books and tensors, in the scheduler's plans, and through the entry points."""

from __future__ import annotations

import random

import pytest
import torch

import plain_lfm3
from conftest import TINY
from test_generate import MARGIN_BF16, prompts_for, teacher_forced_ok
from test_scheduler import FakeDevice, drive, expected
from tokenomos_b200.cache.manager import CacheError, CacheManager, OutOfPages
from tokenomos_b200.engine.scheduler import Request, Scheduler
from tokenomos_b200.parts.contract import BlockScales, ChunkKV, PagedKV, SharedState, SlotState, WindowKV
from tokenomos_b200.sampling.params import SamplingParams

gpu = pytest.mark.gpu
KV8 = PagedKV(2, 16, torch.float8_e4m3fn)
SPECS = {(0, "conv"): SlotState((2, 8)), (1, "kv"): KV8, (1, "kv_scale"): BlockScales(KV8), (2, "kv"): WindowKV(2, 16, 10),
         (3, "kv"): SharedState(1, "kv"), (4, "kv"): ChunkKV(1, 8, 6), (5, "sum"): SlotState((3,), torch.float32)}


def make(pages=40, page=4, slots=6, device="meta", poison=False, max_len=None):
    return CacheManager(SPECS, page, pages, slots, torch.float32, device, max_len, poison)


def grow(c, rid, n):
    c.extend(rid, n)
    c.commit(rid, n)


# ---- the books ----

@pytest.mark.parametrize("length", [0, 3, 4, 9, 16, 25])
def test_a_fork_shares_full_pages_and_copies_the_one_being_filled(length):
    c = make(device="cpu", poison=True)
    c.admit("a")
    if length:
        grow(c, "a", length)
    for key, t in c.states.items():
        t.copy_(torch.randn(t.shape).to(t.dtype))
    a = c.requests["a"]
    before = {k: c.free_pages(k) for k in c.groups}
    children = c.fork("a", ["b", "c"])
    c.check()
    full, part = divmod(length, 4)
    for new in children:
        assert new.length == length and new.slot not in (0, a.slot)
        for k, g in c.groups.items():
            table = new.tables[k]
            assert len(table) == full + (part > 0) and table[:full] == a.tables[k][:full]
            if part:
                assert table[full] not in (0, a.tables[k][full])
                for m in g.members:
                    raw = c.states[m].view(torch.uint8)
                    assert torch.equal(raw[table[full]], raw[a.tables[k][full]])
        if length:
            assert torch.equal(c.states[(0, "conv")][new.slot], c.states[(0, "conv")][a.slot])
            assert torch.equal(c.states[(5, "sum")][new.slot], c.states[(5, "sum")][a.slot])
    for k in c.groups:
        assert before[k] - c.free_pages(k) == (2 if part else 0)
    assert c.fork_pages("a") == (1 if part else 0)
    # the shared pages go back with the last that holds them, in any order
    for rid in ("b", "a", "c"):
        c.release(rid)
        c.check()
    assert all(c.free_pages(k) == 39 for k in c.groups) and c.free_slots() == 6


def test_a_shared_page_is_poisoned_when_the_last_holder_lets_it_go():
    c = make(device="cpu", poison=True)
    c.admit("a")
    grow(c, "a", 8)
    page = c.block_table("a", ("full",))[0]
    for key in c.groups[("full",)].members:
        c.states[key].view(torch.uint8)[page] = 0
    c.fork("a", ["b"])
    c.release("a")
    assert (c.states[(1, "kv")].view(torch.uint8)[page] == 0).all() and (c.states[(1, "kv_scale")][page] == 0).all()
    c.release("b")
    assert c.states[(1, "kv")][page].float().isnan().all() and c.states[(1, "kv_scale")][page].isnan().all()


def test_windows_give_shared_pages_back_one_holder_at_a_time():
    c = make()
    c.admit("a")
    grow(c, "a", 9)
    c.fork("a", ["b"])
    shared = c.block_table("a", ("window", 10))[0]
    assert shared and shared == c.block_table("b", ("window", 10))[0]
    grow(c, "a", 8)                          # a's window has passed the first page
    c.check()
    assert c.block_table("a", ("window", 10))[0] == 0 and c.block_table("b", ("window", 10))[0] == shared
    assert c.groups[("window", 10)].pages.holders(shared) == 1
    grow(c, "b", 8)
    c.check()
    assert c.groups[("window", 10)].pages.holders(shared) == 0


def test_a_fork_is_all_or_nothing():
    c = make(pages=5, slots=3)
    c.admit("a")
    grow(c, "a", 9)                          # three pages of four, the last one partly filled
    with pytest.raises(OutOfPages, match="2 forks"):
        c.fork("a", ["b", "c"])
    c.check()
    assert set(c.requests) == {"a"} and c.free_slots() == 2
    c.fork("a", ["b"])
    with pytest.raises(CacheError, match="already live"):
        c.fork("a", ["b"])
    with pytest.raises(CacheError, match="already live"):
        c.fork("a", ["x", "x"])
    with pytest.raises(CacheError, match="not live"):
        c.fork("nobody", ["x"])
    c.check()


@pytest.mark.parametrize("seed", range(6))
def test_random_orders_with_forks_keep_the_books(seed):
    rng = random.Random(seed)
    c = make(pages=rng.choice([15, 40]), page=rng.choice([1, 4, 8]), slots=5, max_len=120)
    live, next_id = [], 0
    for _ in range(400):
        op = rng.random()
        if op < 0.15 and c.free_slots():
            c.admit(next_id)
            live.append(next_id)
            next_id += 1
        elif op < 0.35 and live:
            rid, n = rng.choice(live), rng.randint(1, 3)
            try:
                c.fork(rid, list(range(next_id, next_id + n)))
                live += range(next_id, next_id + n)
            except OutOfPages:
                assert c.free_slots() < n or c.free_pages() < n
            next_id += n
        elif op < 0.8 and live:
            rid, n = rng.choice(live), rng.choice([1, 1, 2, 5, 17])
            if c.try_extend(rid, n):
                # what a step writes is nobody else's
                st = c.requests[rid]
                for k, g in c.groups.items():
                    for b in range(st.length // c.page_size, -(-(st.length + n) // c.page_size)):
                        assert g.pages.holders(st.tables[k][b]) == 1
                c.commit(rid, n)
        elif live:
            c.release(live.pop(rng.randrange(len(live))))
        c.check()
    for rid in live:
        c.release(rid)
    c.check()
    assert all(c.free_pages(k) == c.num_pages - 1 for k in c.groups)


# ---- the scheduler ----

def scheduler(pages=200, page=4, slots=8, budget=16, max_len=400):
    return Scheduler(make(pages, page, slots, max_len=max_len), budget)


def group(prompt, n, max_new):
    reqs = [Request(list(prompt), max_new=max_new, seed=i) for i in range(n)]
    reqs[0].siblings = reqs[1:]
    return reqs


def test_the_prompt_is_read_once_and_its_last_token_by_each():
    s = scheduler()
    reqs = group(range(40), 3, 3)
    s.add(reqs[0])
    log = []
    drive(s, log)
    assert [[p[1:] for p in step] for step in log] == (
        [[(0, 16, False)], [(16, 16, False)], [(32, 7, False)]] + [[(39 + i, 1, True)] * 3 for i in range(3)])
    assert all(r.output == expected(r.prompt, 3) and r.finish == "length" for r in reqs)
    assert s.stats["forked"] == 2 and s.cache.free_pages() == 199 and s.cache.free_slots() == 8


@pytest.mark.parametrize("prompt", [1, 2, 5])
def test_short_prompts(prompt):
    s = scheduler()
    reqs = group(range(prompt), 4, 2)
    s.add(reqs[0])
    drive(s, [])
    assert all(r.output == expected(r.prompt, 2) for r in reqs) and s.idle()
    assert s.stats["forked"] == (3 if prompt > 1 else 0)


def test_siblings_beyond_the_slots_wait_and_read_the_prompt_themselves():
    s = scheduler(slots=2)
    reqs = group(range(20), 5, 3)
    s.add(reqs[0])
    other = Request(list(range(7)), max_new=2)
    s.add(other)
    drive(s, [])
    assert all(r.output == expected(r.prompt, 3) for r in reqs) and other.output == expected(other.prompt, 2)
    assert s.stats["forked"] <= 1 and s.cache.free_slots() == 2
    s.cache.check()


@pytest.mark.parametrize("seed", range(8))
def test_random_groups_with_preemptions_and_a_step_in_flight(seed):
    """The engine's order of calls (a step is delivered after the next one is launched) with few pages: every reply is what the prompt
    gives, whatever was forked, preempted and computed again."""
    from tokenomos_b200.engine.scheduler import NeedsDrain

    rng = random.Random(seed)
    s = scheduler(pages=rng.choice([14, 30]), slots=rng.choice([3, 6]), budget=rng.choice([5, 16]), max_len=48)
    reqs = []
    for _ in range(6):
        g = group([rng.randrange(50) for _ in range(rng.randint(1, 24))], rng.randint(1, 4), rng.randint(1, 9))
        s.add(g[0])
        reqs += g
    device, flying = FakeDevice(), []
    seen = device.seen

    def forked():
        # what a fork copies: the history of the request that read the prompt
        for r in s.running:
            if r.computed and r.rid not in seen:
                lead = next(x for x in s.running + reqs if x is not r and x.prompt == r.prompt and x.rid in seen)
                seen[r.rid] = list(r.prompt[:r.computed])
                assert seen[lead.rid][:r.computed] == seen[r.rid]

    for _ in range(2000):
        if s.idle():
            break
        try:
            planned = s.plan()
        except NeedsDrain:
            while flying:
                s.deliver(*flying.pop(0))
            continue
        forked()
        sampled = device.run(planned)
        s.launch(planned)
        flying.append((planned, sampled))
        if len(flying) > 1:
            s.deliver(*flying.pop(0))
        s.cache.check()
    while flying:
        s.deliver(*flying.pop(0))
    assert s.idle() and all(r.output == expected(r.prompt, r.max_new) for r in reqs)
    assert s.cache.free_pages() == s.cache.num_pages - 1


def test_what_is_refused():
    s = scheduler()
    a, b = Request([1, 2]), Request([1, 3])
    a.siblings = [b]
    with pytest.raises(ValueError, match="siblings"):
        s.add(a)
    b.prompt, b.max_new = [1, 2], 1000
    with pytest.raises(ValueError, match="too long"):
        s.add(a)
    with pytest.raises(ValueError, match="at least one reply"):
        SamplingParams(n=0).validate()


# ---- the engine ----

@gpu
@pytest.mark.parametrize("name, work, cache", [("B", "fp32", None), ("C", "fp32", None), ("D", "bf16", None), ("D", "bf16", "fp8"), ("D", "fp32", "fp8")])
@pytest.mark.parametrize("graphs", [False, True])
def test_replies_of_one_prompt_through_llm(name, work, cache, graphs, model_folders):
    """Greedy replies of a prompt are one and the same, and the plain implementation's (16-bit: within the margin; 8-bit: those of an engine that
    reads the prompt for each); sampled ones are those of as many requests with their seeds."""
    from tokenomos_b200 import LLM

    folder = model_folders[name][torch.bfloat16]
    config, w = plain_lfm3.read_folder(folder)
    prompts = prompts_for(name, [37, 1, 16, 50], seed=4)
    kw = dict(work=work, cache=cache, page=TINY[name]["page"], max_len=96, slots=6, pages=70, prefill_budget=24, poison=True, graphs=graphs)
    with LLM(str(folder), **kw) as llm:
        llm.engine.step_fn.capture_after = 0
        outs = llm.generate(prompts, SamplingParams(max_tokens=10, n=4))
        assert llm.engine.scheduler.stats["forked"] >= 3
        llm.engine.cache.check()
        sampled = llm.generate(prompts, SamplingParams(max_tokens=10, n=3, temperature=0.9, top_p=0.9, seed=11))
        apart = [[llm.generate([p], SamplingParams(max_tokens=10, temperature=0.9, top_p=0.9, seed=11 + i))[0] for i in range(3)] for p in prompts]
    assert len(outs) == 16 and len(sampled) == 12
    for i, prompt in enumerate(prompts):
        mine = outs[4 * i:4 * i + 4]
        assert all(o.token_ids == mine[0].token_ids and o.prompt_tokens == len(prompt) for o in mine)
        if cache is None:
            teacher_forced_ok(config, w, prompt, mine[0].token_ids, 1e-4 if work == "fp32" else MARGIN_BF16[name])
        if work == "fp32":
            assert [o.token_ids for o in sampled[3 * i:3 * i + 3]] == [o.token_ids for o in apart[i]]
        assert len({tuple(o.token_ids) for o in sampled[3 * i:3 * i + 3]}) > 1


@gpu
def test_stream_takes_one_reply(model_folders):
    from tokenomos_b200 import LLM

    with LLM(str(model_folders["A"][torch.bfloat16]), page=16, max_len=64, slots=2, pages=12) as llm:
        with pytest.raises(ValueError, match="one reply"):
            next(llm.stream([1, 2], SamplingParams(n=2)))
