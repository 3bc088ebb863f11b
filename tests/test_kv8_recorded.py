"""The 8-bit cache's operators recorded, replayed side by side and repeated: every form of the attention, those whose shares meet in
scratch memory above all."""

from __future__ import annotations

import pytest
import torch

from test_kv8 import Cache, attend, i32, within, write
from tokenomos_b200 import ops
from tokenomos_b200.ops import _lib, kv8

gpu = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
# (type, page, whether the shares meet in scratch memory); bfloat16 over whole pages joins its shares in clusters
FORMS = [(BF16, 16, False), (BF16, 8, False), (F32, 16, True), (F32, 8, True), (BF16, 12, True), (F32, 5, True)]


class Call:
    """One call of either form over a cache of its own: sequences of up to `longest` positions, their last `new` tokens."""

    def __init__(self, dtype, P, new, D, seed, lens=(2600, 1900), H=4):
        self.H, self.G, self.D, self.P, self.new, self.lens = H, 1, D, P, new, list(lens)
        self.cache = Cache(self.lens, self.G, D, P, seed=seed).fill(seed)
        gen = torch.Generator().manual_seed(seed)
        T = new * len(self.lens)
        self.q = torch.randn(T, self.H, D, generator=gen).to(dtype).cuda()
        self.out = torch.full_like(self.q, 7.0)
        self.positions = i32([n - new + i for n in self.lens for i in range(new)])
        self.tok_seq = i32([s for s in range(len(self.lens)) for _ in range(new)])
        size = ops.attention_kv8_tokens(self.H, self.G, D, P, dtype)
        tiles = [(s * new + o, min(size, new - o)) for s in range(len(self.lens)) for o in range(0, new, size)]
        self.tok0, self.ntok = i32([a for a, _ in tiles]), i32([b for _, b in tiles])
        self.items = T if new == 1 else len(tiles)
        self.dtype, self.scale = dtype, D ** -0.5

    def shares(self):
        """How many CTAs share a row's keys."""
        code, longest = _lib.F32 if self.dtype == F32 else _lib.BF16, max(self.lens)
        sms = torch.cuda.get_device_properties(0).multi_processor_count
        if self.new == 1:
            if kv8._decode_chooses(self.P, code):
                return _lib.lib().tk_attn_kv8_tc_splits(self.items, self.H, self.G, self.D, self.P, longest, longest)
        elif kv8._prefill_chooses(self.H, self.G, self.D, self.P, code):
            return _lib.lib().tk_attn_kv8_prefill_splits(len(self.q), self.items, self.H, self.G, self.D, self.P, longest, sms)
        return _lib.call("tk_attn_kv8_splits", self.items, self.H, self.G, self.D, self.P, code, longest, longest, int(self.new == 1), sms)

    def __call__(self):
        c, longest = self.cache, max(self.lens)
        if self.new == 1:
            ops.attention_kv8_decode(self.q, c.pool, c.scales, self.out, self.positions, self.tok_seq, c.table_dev, None, None, self.scale, longest)
        else:
            ops.attention_kv8_prefill(self.q, c.pool, c.scales, self.out, self.positions, self.tok_seq, c.table_dev, self.tok0, self.ntok, None, self.scale,
                                      longest)

    def check(self):
        for s, n in enumerate(self.positions[self.new - 1::self.new].tolist()):
            rows = slice(s * self.new, (s + 1) * self.new)
            want, size, reach = attend(self.q[rows].double(), self.cache.of(s, n + 1), self.positions[rows], None, self.scale, self.cache.value_scales(s, n + 1))
            within(self.out[rows], want, size, reach, n + 1, self.dtype)


def record(call):
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    return g


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [1, 30])
@pytest.mark.parametrize("dtype, P, scratch", FORMS)
def test_recorded_calls_side_by_side_keep_their_workspaces_apart(dtype, P, scratch, new, D):
    """Two recorded calls replayed on two streams again and again, with eager calls on a third: new contents and positions come through, nobody's
    shares are another's."""
    calls = [Call(dtype, P, new, D, seed) for seed in range(3)]
    assert all(c.shares() > 1 for c in calls)
    assert scratch == (kv8._decode_chooses(P, _lib.F32 if dtype == F32 else _lib.BF16) is False)
    graphs = [record(c) for c in calls[:2]]
    for c in calls:
        c.q.copy_(torch.randn_like(c.q))
        c.positions -= i32([300] * new + [41] * new)
        c.out.fill_(7.0)
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, run in zip(streams, [g.replay for g in graphs] + [calls[2]]):
            with torch.cuda.stream(s):
                run()
    torch.cuda.synchronize()
    for c in calls:
        c.check()


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [1, 30])
@pytest.mark.parametrize("dtype, P, scratch", FORMS)
def test_the_same_call_gives_the_same_bits_in_every_form(dtype, P, scratch, new, D):
    call = Call(dtype, P, new, D, 5)
    call()
    first = call.out.clone()
    call.check()
    g = record(call)
    for i in range(8):
        call.out.fill_(float(i))
        g.replay() if i % 2 else call()
        assert torch.equal(first, call.out)


@gpu
@pytest.mark.parametrize("T", [9, 600])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_recorded_write_follows_its_inputs(dtype, T):
    """Recorded once, replayed over other rows, positions and pages: the bits of an eager call, and a page that grows keeps growing."""
    H, G, D, P = 4, 2, 64, 16
    gen = torch.Generator().manual_seed(T)
    w = (torch.rand(2, D, generator=gen) + 0.5).cuda()
    freq = torch.exp(-torch.arange(D // 2) * 0.2).cuda()
    a, b = Cache([2 * T + 7], G, D, P), Cache([2 * T + 7], G, D, P)
    x, pos, seq = torch.zeros(T, (H + 2 * G) * D, dtype=dtype, device="cuda"), i32([0] * T), i32([0] * T)
    run = lambda c: ops.qk_norm_rope_write8(x, c.pool, c.scales, w[0], w[1], 1e-6, freq, pos, seq, c.table_dev, H, G, D, P)  # noqa: E731
    pos.copy_(torch.arange(T))
    g = torch.cuda.CUDAGraph()
    keep = a.pool.view(torch.uint8).clone(), a.scales.clone()
    with torch.cuda.graph(g):
        q = run(a)
    a.pool.view(torch.uint8).copy_(keep[0])
    a.scales.copy_(keep[1])
    for start, size in ((0, 1.0), (T, 30.0)):
        x.copy_((torch.randn(x.shape, generator=gen) * size).to(dtype))
        pos.copy_(torch.arange(start, start + T))
        g.replay()
        want = run(b)
        assert torch.equal(q, want) and torch.equal(a.pool.view(torch.uint8), b.pool.view(torch.uint8))
        assert torch.equal(a.scales.view(torch.int32), b.scales.view(torch.int32))


FIRST = """
import sys
sys.path.insert(0, "tests")
import torch
from test_kv8_recorded import Call
call = Call(torch.bfloat16, 16, int(sys.argv[1]), 128, 0, H=16)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    call()
g.replay()
torch.cuda.synchronize()
call.check()
print("fine")
"""


@gpu
@pytest.mark.parametrize("new", [1, 30])
def test_a_process_may_record_its_first_call(new):
    """What the entry points ask of the device once (attributes, places) may be asked while a stream is being recorded."""
    import subprocess
    import sys
    from pathlib import Path

    done = subprocess.run([sys.executable, "-c", FIRST, str(new)], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip() == "fine", done.stdout + done.stderr
