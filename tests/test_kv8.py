"""The 8-bit cache's operators against their definitions in 64 bits: the quantised write (norm, rotation, block scales, blocks that
grow), attention over what it leaves (single tokens and prompt portions), the copying of rows, and what they refuse."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from tokenomos_b200 import ops
from tokenomos_b200.ops import KernelError, _lib

gpu = pytest.mark.gpu
F8 = torch.float8_e4m3fn
NAN_BYTE = 0x7F


# ---- definitions in 64 bits ----

def values(pool, scales):
    return pool.double() * scales.double()[..., None, None]


def norm_rope(x, w, eps, freq, pos, mult, interleaved):
    """x [T, heads, D] in float64."""
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    R = 2 * freq.numel()
    a = pos.double()[:, None, None] * freq.double()
    c, s = a.cos() * mult, a.sin() * mult
    out = x.clone()
    if interleaved:
        u, v = x[..., 0:R:2], x[..., 1:R:2]
        out[..., 0:R:2], out[..., 1:R:2] = u * c - v * s, v * c + u * s
    else:
        u, v = x[..., :R // 2], x[..., R // 2:R]
        out[..., :R // 2], out[..., R // 2:R] = u * c - v * s, v * c + u * s
    return out


def attend(q, kv, pos, window, scale, sv, sink=False):
    """q [T, H, D], kv [2, G, L, D] (float64, one sequence's cache), pos [T], sv [G, L] (the values' scales): (outputs, sum of p |v| per output,
    and for the bounds the largest sum |q k| scale of a row and what 8-bit terms leave)."""
    T, H, D = q.shape
    G, L = kv.shape[1], kv.shape[2]
    k, v = kv.repeat_interleave(H // G, 1)
    s = torch.einsum("thd,hld->htl", q, k) * scale
    j, i = torch.arange(L, device=q.device), pos[:, None]
    see = j <= i
    if window and window > 0:
        see = see & (j > i - window)
    elif window:
        see = see & (j >= i - i % -window)
    s = s.masked_fill(~see, -math.inf)
    if sink:
        s = torch.cat((s, torch.zeros(H, T, 1, dtype=s.dtype, device=s.device)), -1)
    p = torch.softmax(s, -1)[..., :L]
    # (a value that a row does not see takes no part, whatever it is)
    seen_v = torch.where(see.any(0)[None, :, None], v, 0.0)
    o = torch.einsum("htl,hld->thd", p, seen_v)
    size = torch.einsum("htl,hld->thd", p, seen_v.abs())
    seen_k = torch.where(see.any(0)[None, :, None], k, 0.0).abs()
    reach = torch.einsum("thd,hld->htl", q.abs(), seen_k).amax(-1).t() * abs(scale)
    # what the terms of q and of the weights leave: 2^-18 of q's largest element beside every key element; 2^-24 of the row's largest weight of a
    # value's byte beside every byte
    left = q.abs().amax(-1) * seen_k.sum(-1).amax(-1)[None] * abs(scale) * 2.0 ** -18
    sv = sv.double().repeat_interleave(H // G, 0)
    rest = (p * sv[:, None]).amax(-1).t()[..., None] * (seen_v.abs() / sv[..., None]).sum(1)[None] * 2.0 ** -24
    return o, size, (reach, left, rest)


def within(got, want, size, reach, keys, dtype, least=0.0):
    """The kernel's bound. A weight's relative error: its score (D products in 32-bit sums, a few roundings of a number of at most
    `reach` log2(e): (D + 8) 2^-24 of it, and for 32-bit q 2^-22 from its two halves), the exponential's 2^-22, its rounding to
    float16 (2^-11; as two float16 2^-22; as four e4m3 terms 2^-16) and, in terms, what they leave (``attend``); the same for the sum; sums over
    keys in 32 bits, each term's products their own; one rounding of the result. `least`: of the row's largest weight, what a 32-bit row's weights
    are rounded to where that is more."""
    D = want.shape[-1]
    unit = torch.finfo(dtype).eps / 2
    reach, left, rest = reach
    eps = reach[..., None] * ((2 * D + 8) * 2.0 ** -24 + (2.0 ** -22 if dtype == torch.float32 else 0)) + 2.0 ** -22
    half = 2.0 ** -22
    if dtype == torch.bfloat16:
        eps, half = eps + left[..., None], 2.0 ** -11
    bound = unit * want.abs() * 1.01 + size * (2 * eps + half + 8 * (keys + 64) * 2.0 ** -24) + 2.0 ** -120
    if dtype == torch.bfloat16:
        bound = bound + rest
    else:
        bound = bound + rest * 2.0 ** 24 * least
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= bound).all(), ((off / bound).max().item(), off.max().item())


# ---- a cache and sequences in it ----

class Cache:
    """Sequences in an 8-bit cache whose pages come in no order; everything that nobody writes is NaN."""

    def __init__(self, lens, G, D, P, seed=0, pages=None):
        gen = torch.Generator().manual_seed(seed)
        blocks = [-(-n // P) for n in lens]
        pages = pages or sum(blocks) + 3
        order = (torch.randperm(pages - 1, generator=gen) + 1).tolist()
        self.table = torch.zeros(len(lens), max(blocks), dtype=torch.int32)
        for s, b in enumerate(blocks):
            self.table[s, :b] = torch.tensor([order.pop() for _ in range(b)], dtype=torch.int32)
        self.lens, self.G, self.D, self.P = lens, G, D, P
        self.table_dev = self.table.cuda()
        self.pool = torch.full((pages, 2, G, P, D), NAN_BYTE, dtype=torch.uint8, device="cuda").view(F8)
        self.scales = torch.full((pages, 2, G), math.nan, device="cuda")

    def fill(self, seed=0, spread=0):
        """Random bytes and scales at the positions that there are."""
        gen = torch.Generator().manual_seed(seed)
        for s, n in enumerate(self.lens):
            for b in range(-(-n // self.P)):
                page, here = int(self.table[s, b]), min(self.P, n - b * self.P)
                x = (torch.randn(2, self.G, here, self.D, generator=gen) * 110).clamp(-448, 448).to(F8)
                self.pool.view(torch.uint8)[page, :, :, :here] = x.view(torch.uint8).cuda()
                e = torch.randint(-8, -5, (2, self.G), generator=gen)
                e[1] += torch.randint(-spread, spread + 1, (self.G,), generator=gen)
                self.scales[page] = torch.exp2(e.float()).cuda()
        return self

    def of(self, s, upto=None):
        """[2, G, n, D] float64: sequence s's keys and values."""
        n = self.lens[s] if upto is None else upto
        rows = self.table[s, :-(-n // self.P)].long().cuda()
        raw = self.pool.view(torch.uint8)[rows].view(F8).double() * self.scales[rows].double()[..., None, None]
        return raw.permute(1, 2, 0, 3, 4).reshape(2, self.G, -1, self.D)[:, :, :n]


    def value_scales(self, s, upto=None):
        """[G, n]: of each position of sequence s."""
        n = self.lens[s] if upto is None else upto
        return self.scales[self.table[s, :-(-n // self.P)].long().cuda(), 1].t().repeat_interleave(self.P, 1)[:, :n]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def write(cache, rows, H, wq, wk, eps, freq, mult=1.0, interleaved=False):
    """``rows``: (sequence, first position, [n, (H + 2 G) D] rows) of one step."""
    pos = i32([p + i for _, p, x in rows for i in range(len(x))])
    seq = i32([s for s, _, x in rows for _ in range(len(x))])
    return ops.qk_norm_rope_write8(torch.cat([x for _, _, x in rows]), cache.pool, cache.scales, wq, wk, eps, freq, pos, seq, cache.table_dev,
                                   H, cache.G, cache.D, cache.P, mult, interleaved), pos


def half_step(x, s):
    """Half the distance of the e4m3 numbers around x / s, in x's units."""
    y = (x / s).abs().clamp(min=2.0 ** -6)
    return torch.exp2(torch.floor(torch.log2(y)) - 4) * s


# ---- the write ----

@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H, G, D, P, R, interleaved, norm", [
    (4, 2, 64, 16, 64, False, True), (3, 1, 64, 5, 32, False, True), (16, 8, 64, 16, 64, True, False), (5, 5, 128, 1, 128, False, True),
    (2, 1, 128, 64, 20, False, False), (6, 2, 128, 40, 128, True, True), (1, 1, 64, 16, 0, False, True), (4, 2, 64, 7, 6, True, False),
])
def test_write_follows_the_definition_however_the_tokens_are_cut(dtype, H, G, D, P, R, interleaved, norm):
    g = torch.Generator().manual_seed(H * 7 + P)
    lens = [97, 1, 40]
    x = [torch.randn(n, (H + 2 * G) * D, generator=g) * torch.exp2(torch.randint(-9, 9, (n, 1), generator=g).float()) for n in lens]
    x = [v.cuda().to(dtype) for v in x]
    wq, wk = (torch.rand(2, D, generator=g) + 0.5).cuda() if norm else (None, None)
    freq = torch.exp(-torch.arange(R // 2) * 0.3).cuda()
    mult, eps = 1.25, 1e-5
    exact = [norm_rope(v.double().view(-1, H + 2 * G, D)[:, :H + G], None, eps, freq, torch.arange(len(v), device="cuda"), mult, interleaved)
             for v in x]
    for v, e in zip(x, exact):
        heads = v.double().view(-1, H + 2 * G, D)
        at = torch.arange(len(v), device="cuda")
        e[:, :H] = norm_rope(heads[:, :H], wq, eps, freq, at, mult, interleaved)
        e[:, H:] = norm_rope(heads[:, H:H + G], wk, eps, freq, at, mult, interleaved)
    cuts = {"whole": [[(s, 0, n) for s, n in enumerate(lens)]],
            "cut": [[(0, 0, 3), (2, 0, 17)], [(0, 3, 4), (1, 0, 1), (2, 17, 18)], [(0, 4, 60)], [(0, 60, 61), (2, 18, 40)], [(0, 61, 97)]]}
    left = {}
    for name, steps in cuts.items():
        cache = Cache(lens, G, D, P)
        for step in steps:
            q, pos = write(cache, [(s, a, x[s][a:b]) for s, a, b in step], H, wq, wk, eps, freq, mult, interleaved)
            want = torch.cat([exact[s][a:b, :H] for s, a, b in step])
            # (a few 32-bit roundings of numbers of the head's size, then the result's own)
            bound = want.abs() * torch.finfo(dtype).eps / 2 * 1.01 + want.abs().amax(-1, keepdim=True) * 2.0 ** -20
            assert ((q.double() - want).abs() <= bound).all()
        left[name] = cache
        for s, n in enumerate(lens):
            kv = torch.stack((exact[s][:, H:], x[s].double().view(n, -1, D)[:, H + G:])).permute(0, 2, 1, 3)         # [2, G, n, D]
            got = cache.of(s)
            blocks = cache.table[s, :-(-n // P)].long().cuda()
            sc = cache.scales[blocks].permute(1, 2, 0).double()                                                     # [2, G, blocks]
            assert (torch.frexp(sc)[0] == 0.5).all()
            most = torch.stack([kv[:, :, b * P:(b + 1) * P].abs().amax((2, 3)) for b in range(len(blocks))], -1)
            # the smallest power of two that holds the block's largest (32-bit roundings may move a largest that is next to the border)
            assert (most <= 448 * sc * (1 + 2.0 ** -20)).all() and (most >= 224 * sc * (1 - 2.0 ** -20)).all()
            per = sc.repeat_interleave(P, -1)[:, :, :n, None]
            # one rounding to e4m3, a second one below its smallest normal number when the block grew, and the 32-bit arithmetic before
            bound = half_step(kv, per) * (1 + 2.0 ** -20) + per * 2.0 ** -10 + kv.abs().amax(-1, keepdim=True) * 2.0 ** -20
            assert ((got - kv).abs() <= bound).all()
    # the same values above the smallest normal number (queries and keys do not depend on the cut, so neither do largest values)
    a, b = left["whole"], left["cut"]
    for s in range(len(lens)):
        rows = a.table[s, :-(-lens[s] // P)].long()
        assert torch.equal(a.scales[rows.cuda()], b.scales[rows.cuda()])
        va, vb = a.of(s), b.of(s)
        per = a.scales[rows.cuda()].permute(1, 2, 0).double().repeat_interleave(P, -1)[:, :, :lens[s], None]
        # From the smallest normal number N = 2^-6 s' up a byte's spacing is the same relative to its binade under the old scale and the new
        # one, so rounding twice is rounding once. Below N the second rounding is coarser, and N itself can come from there: x = 0.9374 N
        # goes to 0.9375 N first (spacing N / 16), a tie of the second rounding (spacing N / 8) that goes to N, while x alone goes to 0.875 N.
        normal = (va.abs() > per * 2.0 ** -6) | (vb.abs() > per * 2.0 ** -6)
        assert torch.equal(va[normal], vb[normal]) and ((va - vb).abs() <= per * 2.0 ** -9).all()
    # nothing behind the last positions, and no other page, was written
    held = torch.zeros(a.pool.shape[0], P, dtype=torch.bool)
    for s, n in enumerate(lens):
        for t in range(n):
            held[int(a.table[s, t // P]), t % P] = True
    raw = a.pool.view(torch.uint8).permute(0, 3, 1, 2, 4)
    assert (raw[~held.cuda()] == NAN_BYTE).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H, G, D, P", [(2, 1, 64, 16), (16, 8, 64, 16), (9, 3, 128, 7), (8, 8, 64, 64)])
def test_a_large_step_writes_what_small_ones_write(dtype, H, G, D, P):
    """Steps of 512 tokens and more look for their runs and share their heads out otherwise: the same bits all the same, in pages that are new and
    in pages that hold earlier tokens, whatever the runs' lengths and places."""
    g = torch.Generator().manual_seed(D + P)
    firsts = torch.randint(0, 40, (70,), generator=g).tolist()
    counts = (torch.randint(1, 4, (70,), generator=g) ** 4).tolist()          # 1, 16 and 81
    counts[5], counts[41] = 700, 333
    lens = [a + n for a, n in zip(firsts, counts)]
    freq = torch.exp(-torch.arange(D // 2) * 0.2).cuda()
    wq, wk = (torch.rand(2, D, generator=g) + 0.5).cuda()
    before = [torch.randn(a, (H + 2 * G) * D, generator=g).cuda().to(dtype) for a in firsts]
    rows = [(torch.randn(n, (H + 2 * G) * D, generator=g) * 4).cuda().to(dtype) for n in counts]
    assert sum(counts) >= 512 and sum(firsts) >= 512
    large, small = Cache(lens, G, D, P), Cache(lens, G, D, P)
    for part, at in ((before, [0] * 70), (rows, firsts)):
        step = [(s, a, x) for s, (a, x) in enumerate(zip(at, part)) if len(x)]
        q, _ = write(large, step, H, wq, wk, 1e-6, freq)
        got = []
        for s, a, x in step:                                                   # (whole pages' runs, fewer than 512 tokens)
            i = 0
            while i < len(x):
                n = min(len(x) - i, (P - (a + i) % P) + 400 // P * P)
                got.append(write(small, [(s, a + i, x[i:i + n])], H, wq, wk, 1e-6, freq)[0])
                i += n
        assert torch.equal(q, torch.cat(got))
        assert torch.equal(large.pool.view(torch.uint8), small.pool.view(torch.uint8))
        assert torch.equal(large.scales.view(torch.int32), small.scales.view(torch.int32))


@gpu
def test_a_block_that_grows_rescales_what_it_holds():
    """Tokens of rising size, one a step: the earlier bytes follow the scale exactly while they are normal numbers."""
    G, D, P = 2, 64, 16
    cache = Cache([16], G, D, P)
    g = torch.Generator().manual_seed(3)
    freq = torch.zeros(0, device="cuda")
    sizes = [-12, -20, -3, -3, 4, 4, 9, 2, 13]
    before = None
    for t, e in enumerate(sizes):
        x = (torch.randn(1, 3 * G * D, generator=g) * 2.0 ** e).cuda()
        write(cache, [(0, t, x)], G, None, None, 0.0, freq)
        now = cache.of(0, t + 1)
        if before is not None:
            per = cache.scales[int(cache.table[0, 0])].double()[:, :, None, None]
            assert ((now[:, :, :t] - before).abs() <= per * 2.0 ** -10).all()          # half the smallest step
            same = before.abs() >= per * 2.0 ** -6
            assert torch.equal(now[:, :, :t][same], before[same])
        before = now.clone()
    page = int(cache.table[0, 0])
    assert (cache.scales[page] >= 2.0 ** 4).all()          # 2^13 / 448 and more


@gpu
def test_a_page_used_again_does_not_keep_the_last_ones_scale():
    cache = Cache([16], 1, 64, 16)
    freq = torch.zeros(0, device="cuda")
    big = torch.full((16, 3 * 64), 1000.0, device="cuda")
    write(cache, [(0, 0, big)], 1, None, None, 0.0, freq)
    small = torch.full((1, 3 * 64), 0.01, device="cuda")
    write(cache, [(0, 0, small)], 1, None, None, 0.0, freq)
    assert (cache.scales[int(cache.table[0, 0])] < 1e-4).all()
    assert ((cache.of(0, 1) - 0.01).abs() <= 0.01 / 16).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_what_is_not_finite_marks_its_token_and_no_other(dtype):
    G, D, P, n = 3, 64, 8, 20
    x = torch.randn(n, 3 * G, D, generator=torch.Generator().manual_seed(0)).cuda().to(dtype)
    x[3, G + 1, 5] = math.nan               # a key of head 1
    x[9, 2 * G + 0, 63] = math.inf          # a value of head 0
    x[10, 2 * G + 2, 0] = -1e30             # a value beyond the format's reach, head 2
    x[11] = 0                               # zeros are values like others
    marked = {(3, 1), (9, 0), (10, 2)}
    cache = Cache([n], G, D, P)
    write(cache, [(0, 0, x.view(n, -1))], G, None, None, 0.0, torch.zeros(0, device="cuda"))
    got = cache.of(0)
    for t in range(n):
        for h in range(G):
            if (t, h) in marked:
                assert got[0, h, t].isnan().all() and (got[1, h, t] == 0).all()
            else:
                assert ((got[:, h, t] - x[t, [G + h, 2 * G + h]].double()).abs() <= x[t, [G + h, 2 * G + h]].double().abs() / 16 + 2.0 ** -14).all()


@gpu
def test_tiny_and_huge_blocks_stay_within_the_scales_bounds():
    cache = Cache([8, 8, 8], 1, 64, 8)
    for s, v in enumerate((0.0, 2.0 ** -60, 2.0 ** 48)):
        write(cache, [(s, 0, torch.full((8, 192), v, device="cuda"))], 1, None, None, 0.0, torch.zeros(0, device="cuda"))
        want = {0: 2.0 ** -40, 1: 2.0 ** -40, 2: 2.0 ** 40}[s]
        assert (cache.scales[int(cache.table[s, 0])] == want).all()
        assert (cache.of(s) == (v if s != 1 else 0.0)).all()


@gpu
def test_write_far_positions_turn_by_the_exact_angle():
    G, D, P = 1, 64, 16
    start = 131000
    cache = Cache([16], G, D, P)
    wide = torch.zeros(1, start // P + 2, dtype=torch.int32)
    wide[0, start // P:] = cache.table[0, 0]
    cache.table_dev = wide.cuda()
    freq = (1e6 ** (-torch.arange(32) / 32)).float().cuda()
    x = torch.randn(4, 3 * D, generator=torch.Generator().manual_seed(0)).cuda()
    q, pos = write(cache, [(0, start, x)], G, None, None, 0.0, freq)
    want = norm_rope(x.double().view(4, 3, D)[:, :1], None, 0.0, freq, pos, 1.0, False)
    assert ((q.double() - want).abs() <= 2.0 ** -20 * want.abs().amax(-1, keepdim=True)).all()


# ---- attention ----

def run_attention(cache, q, new, window, scale, gate=None, sink=False):
    """Every sequence's last ``new`` tokens as one step: single tokens through the decode form, portions through the other."""
    T, H, _ = q.shape
    pos = i32([cache.lens[s] - n + i for s, n in enumerate(new) for i in range(n)])
    seq = i32([s for s, n in enumerate(new) for _ in range(n)])
    out = torch.full_like(q, 7.0)
    start, tiles, singles = 0, [], []
    size = ops.attention_kv8_tokens(H, cache.G, cache.D, cache.P, q.dtype)
    for n in new:
        if n == 1:
            singles.append(start)
        else:
            tiles += [(start + o, min(size, n - o)) for o in range(0, n, size)]
        start += n
    longest = max(cache.lens)
    if singles:
        ops.attention_kv8_decode(q, cache.pool, cache.scales, out, pos, seq, cache.table_dev, i32(singles + [-1]), window, scale, longest, gate, sink)
    if tiles:
        tiles.append((0, 0))
        ops.attention_kv8_prefill(q, cache.pool, cache.scales, out, pos, seq, cache.table_dev, i32([a for a, _ in tiles]), i32([b for _, b in tiles]),
                                  window, scale, longest, gate, sink)
    return out, pos


def check_attention(cache, new, H, dtype, window=None, scale=None, sink=False, seed=0, size=1.0):
    D = cache.D
    scale = D ** -0.5 if scale is None else scale
    q = (torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(seed)) * size).to(dtype).cuda()
    out, pos = run_attention(cache, q, new, window, scale, sink=sink)
    start = 0
    for s, n in enumerate(new):
        want, sz, reach = attend(q[start:start + n].double(), cache.of(s), pos[start:start + n], window, scale, cache.value_scales(s), sink)
        within(out[start:start + n], want, sz, reach, cache.lens[s], dtype)
        start += n


SHAPES = [(1, 1, 64, 16), (4, 2, 64, 16), (32, 8, 64, 16), (6, 2, 64, 16), (5, 1, 64, 5), (16, 1, 64, 64), (8, 8, 64, 1), (4, 1, 128, 16),
          (12, 4, 128, 12), (16, 1, 128, 8), (2, 2, 128, 32), (9, 1, 64, 48), (4, 2, 64, 128), (8, 1, 64, 256), (4, 1, 128, 256), (8, 4, 64, 32)]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H, G, D, P", SHAPES)
def test_attention_of_single_tokens(dtype, H, G, D, P):
    lens = [1, 2, 15, 16, 17, 33, 300, 64, 129]
    check_attention(Cache(lens, G, D, P).fill(), [1] * len(lens), H, dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H, G, D, P", SHAPES)
def test_attention_of_portions_and_single_tokens_in_one_step(dtype, H, G, D, P):
    lens = [2, 77, 40, 300, 129, 16]
    check_attention(Cache(lens, G, D, P).fill(), [2, 77, 1, 45, 128, 3], H, dtype)


@gpu
@pytest.mark.parametrize("window", [None, 7, 8, 100, -24])
@pytest.mark.parametrize("H, G, D, P", [(4, 2, 64, 8), (3, 1, 64, 8), (32, 8, 128, 8), (14, 2, 64, 8), (16, 1, 128, 8), (6, 2, 64, 16), (5, 1, 128, 32), (22, 2, 64, 16),
                                        (39, 3, 64, 64), (7, 1, 64, 8)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_over_pages_of_8_and_of_groups_that_do_not_divide_a_tile(dtype, H, G, D, P, window):
    lens = [1, 8, 9, 63, 64, 65, 257, 1500, 130, 700, 2300]
    new = [1, 8, 2, 63, 1, 40, 200, 1, 129, 700, 45]
    check_attention(Cache(lens, G, D, P, seed=P).fill(seed=H, spread=4), new, H, dtype, window=window)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window", [1, 7, 16, 50, 1000, -1, -16, -50, -1000])
@pytest.mark.parametrize("sink", [False, True])
def test_attention_windows_chunks_and_a_sink(dtype, window, sink):
    lens = [1, 5, 64, 200, 150, 49, 51, 160]
    check_attention(Cache(lens, 2, 64, 16).fill(), [1, 5, 1, 130, 1, 1, 51, 160], 8, dtype, window, sink=sink)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_shares_long_contexts_out_and_joins_them(dtype, D):
    lens = [2500, 900, 3]
    check_attention(Cache(lens, 2, D, 16).fill(), [1, 1, 1], 8, dtype)
    check_attention(Cache(lens, 1, D, 16).fill(), [20, 300, 1], 4, dtype)
    check_attention(Cache(lens, 1, D, 16).fill(), [1, 17, 3], 4, dtype, window=700, sink=True)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_with_peaked_scores_and_scales_far_apart(dtype):
    """Scores of hundreds (one key takes all), and value blocks 2^60 apart."""
    lens = [200, 65]
    check_attention(Cache(lens, 1, 64, 16).fill(), [1, 65], 4, dtype, size=40.0)
    check_attention(Cache(lens, 1, 64, 16).fill(spread=30), [1, 65], 4, dtype)
    check_attention(Cache(lens, 1, 64, 16).fill(), [50, 1], 4, dtype, size=1e-12)
    check_attention(Cache(lens, 1, 64, 16).fill(), [1, 1], 4, dtype, scale=1e-30)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_small_weights_beside_a_large_one(dtype):
    """The first key takes half of the weight and its value is 0: what comes out is the other thousands' (each about 2^-13 of it)."""
    n = 8000
    cache = Cache([n], 1, 64, 16).fill()
    page, page1 = int(cache.table[0, 0]), cache.table[0, 1:].long().cuda()
    cache.pool[page, :, :, 0] = torch.zeros(64, device="cuda").to(F8)
    cache.pool[page, 0, 0, 0, 0] = torch.tensor(256.0).to(F8)
    cache.scales[:] = 2.0 ** -7
    q = torch.zeros(1, 4, 64, device="cuda", dtype=dtype)
    q[0, :, 0] = 4.0
    cache.pool.view(torch.uint8)[page1, 0, :, :, 0] = 0
    cache.pool.view(torch.uint8)[page, 0, :, 1:, 0] = 0
    scale = math.log(n) / (4.0 * 2.0)
    out, pos = run_attention(cache, q, [1], None, scale)
    want, sz, reach = attend(q.double(), cache.of(0), pos, None, scale, cache.value_scales(0))
    within(out, want, sz, reach, n, dtype)
    # (a tenth of the weights lost would move the mean of 8,000 random values by about as much)
    assert ((out.double() - want).norm() / want.norm()).item() < 0.01


@gpu
@pytest.mark.parametrize("new", [1, 30])
@pytest.mark.parametrize("P", [16, 12])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("below", [8, 20, 30, 45])
def test_weights_far_below_one_that_meets_zero_bytes(dtype, P, new, below):
    """The first key's weight is 2^below times any other's and its value is 0. Two float16 terms of a weight end at half of float16's smallest step,
    2^-25, while the row's largest weight is 2^7 at least: what is lost of a 32-bit row's weight is 2^-22 of it (`within`) or 2^-32 of the largest."""
    n = 300
    cache = Cache([n], 1, 64, P).fill(seed=below)
    raw = cache.pool.view(torch.uint8)
    raw[cache.table[0].long().cuda(), 0, 0] = 0
    raw[int(cache.table[0, 0]), :, 0, 0] = 0
    cache.pool[int(cache.table[0, 0]), 0, 0, 0, 0] = torch.tensor(256.0).to(F8)
    cache.scales[:] = 2.0 ** -7
    q = torch.zeros(new, 4, 64, device="cuda", dtype=dtype)
    q[:, :, 0] = 4.0
    scale = below * math.log(2.0) / (4.0 * 2.0)
    out, pos = run_attention(cache, q, [new], None, scale)
    want, sz, reach = attend(q.double(), cache.of(0), pos, None, scale, cache.value_scales(0))
    within(out, want, sz, reach, n, dtype, least=2.0 ** -32)


@gpu
@pytest.mark.parametrize("P", [16, 5])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_marked_token_reaches_only_the_rows_that_see_it(dtype, P):
    lens, new, H, G, D = [150, 40], [150, 1], 4, 2, 64
    cache = Cache(lens, G, D, P).fill()
    q = torch.randn(151, H, D, generator=torch.Generator().manual_seed(0)).to(dtype).cuda()
    clean, _ = run_attention(cache, q, new, 30, D ** -0.5)
    page, at = int(cache.table[0, 70 // P]), 70 % P
    raw = cache.pool.view(torch.uint8)
    raw[page, 0, 1, at], raw[page, 1, 1, at] = NAN_BYTE, 0
    out, _ = run_attention(cache, q, new, 30, D ** -0.5)
    hit = torch.zeros(151, H, dtype=torch.bool)
    hit[70:100, 2:] = True                    # the window's queries, the head's group
    assert out[hit.cuda()].isnan().all()
    assert torch.equal(out[~hit.cuda()], clean[~hit.cuda()])


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_applies_a_gate_per_head_and_leaves_other_rows_alone(dtype):
    lens, new, H, G, D = [90, 20, 300], [33, 1, 1], 6, 2, 64
    cache = Cache(lens, G, D, 16).fill()
    gen = torch.Generator().manual_seed(0)
    q = torch.randn(35, H, D, generator=gen).to(dtype).cuda()
    wide = torch.randn(35, 3 * H, generator=gen).to(dtype).cuda()
    gate = wide[:, H:2 * H]
    plain, pos = run_attention(cache, q, new, None, 0.125)
    gated, _ = run_attention(cache, q, new, None, 0.125, gate=gate)
    want = plain.float() * torch.sigmoid(gate.float()).to(dtype).float()[..., None]
    # the product's rounding, and a sigmoid next to the middle of two numbers
    assert ((gated.float() - want).abs() <= want.abs() * 3 * torch.finfo(dtype).eps).all()
    out = torch.full_like(q, 7.0)
    seq = i32([0] * 33 + [1, 2])
    ops.attention_kv8_decode(q, cache.pool, cache.scales, out, pos, seq, cache.table_dev, i32([33]), None, 0.125, 300)
    assert torch.equal(out[33], plain[33]) and (out[:33] == 7).all() and (out[34] == 7).all()


@gpu
def test_a_row_that_sees_nothing_is_zero():
    cache = Cache([40], 1, 64, 16).fill()
    q = torch.randn(2, 4, 64, device="cuda").to(torch.bfloat16)
    out = torch.full_like(q, 7.0)
    for sink in (False, True):
        ops.attention_kv8_decode(q, cache.pool, cache.scales, out, i32([-1, 39]), i32([0, 0]), cache.table_dev, None, None, 0.125, 40, None, sink)
        assert (out[0] == 0).all() and torch.isfinite(out[1]).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_tile_longer_than_it_may_be_writes_only_its_own_rows(dtype):
    lens, H, G, D = [300], 4, 2, 64
    cache = Cache(lens, G, D, 16).fill()
    q = torch.randn(300, H, D, generator=torch.Generator().manual_seed(0)).to(dtype).cuda()
    size = ops.attention_kv8_tokens(H, G, D, 16, dtype)
    want, pos = run_attention(cache, q, [300], None, 0.125)
    out = torch.full_like(q, 7.0)
    ops.attention_kv8_prefill(q, cache.pool, cache.scales, out, pos, i32([0] * 300), cache.table_dev, i32([0]), i32([size + 40]), None, 0.125, 300)
    assert ((out[:size].float() - want[:size].float()).abs() <= 1e-2).all() and (out[size:] == 7).all()


@gpu
def test_tokens_without_a_position_write_nothing():
    cache = Cache([16], 2, 64, 16)
    x = torch.randn(3, 6 * 64, device="cuda")
    q = ops.qk_norm_rope_write8(x, cache.pool, cache.scales, None, None, 0.0, torch.zeros(0, device="cuda"), i32([-1, 0, 1]), i32([0, 0, 0]), cache.table_dev,
                                2, 2, 64, 16)
    assert torch.equal(q, x.view(3, 6, 64)[:, :2])
    raw = cache.pool.view(torch.uint8)
    page = int(cache.table[0, 0])
    assert (raw[page, :, :, :2] != NAN_BYTE).any() and (raw[page, :, :, 2:] == NAN_BYTE).all()
    assert all((raw[p] == NAN_BYTE).all() for p in range(raw.shape[0]) if p != page)


@gpu
def test_offsets_past_32_bits():
    """A pool of 4.5 GB: the pages that are used lie at its end."""
    pages = 280000
    cache = Cache([100, 33], 8, 64, 16, pages=pages)
    count = int((cache.table > 0).sum())
    used = torch.arange(pages - count, pages, dtype=torch.int32)
    cache.table[cache.table > 0] = used
    cache.table_dev = cache.table.cuda()
    assert cache.pool.numel() > 1 << 32 and int(used.min()) * 2 * 8 * 16 * 64 > 1 << 32
    cache.fill()
    check_attention(cache, [60, 1], 16, torch.bfloat16)
    x = torch.randn(100, 32 * 64, device="cuda").to(torch.bfloat16)
    write(cache, [(0, 0, x)], 16, None, None, 0.0, torch.zeros(0, device="cuda"))
    v = x.double().view(100, 32, 64)[:, 24:].permute(1, 0, 2)
    assert ((cache.of(0)[1] - v).abs() <= v.abs() / 16 + 2.0 ** -12).all()
    ops.copy_rows([cache.pool, cache.scales], [pages - 1], [3])
    assert torch.equal(cache.pool[3].view(torch.uint8), cache.pool[pages - 1].view(torch.uint8))
    ops.copy_rows([cache.pool], [3], [pages - 2])
    assert torch.equal(cache.pool[pages - 2].view(torch.uint8), cache.pool[3].view(torch.uint8))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_run_of_steps_as_a_model_makes_them(dtype):
    """Prompt, portions, single tokens: each step writes and attends; every output against attention in 64 bits over what the cache holds
    after its write."""
    H, G, D, P = 8, 2, 64, 16
    lens = [90, 60, 31]
    cache = Cache(lens, G, D, P)
    gen = torch.Generator().manual_seed(0)
    freq = (1e4 ** (-torch.arange(32) / 32)).float().cuda()
    w = torch.ones(D, device="cuda")
    have = [0, 0, 0]
    for step in [(70, 30, 0), (18, 1, 30), (1, 28, 1), (1, 1, 0)]:
        rows, before = [], list(have)
        for s, n in enumerate(step):
            if n:
                rows.append((s, have[s], torch.randn(n, (H + 2 * G) * D, generator=gen).to(dtype).cuda()))
                have[s] += n
        q, pos = write(cache, rows, H, w, w, 1e-6, freq)
        live = [s for s, n in enumerate(step) if n]
        view = Cache.__new__(Cache)
        view.__dict__.update(cache.__dict__)
        view.lens = [have[s] for s in live]
        view.table, view.table_dev = cache.table[live], cache.table_dev[live].contiguous()
        out, _ = run_attention(view, q, [step[s] for s in live], None, D ** -0.5)
        start = 0
        for k, s in enumerate(live):
            n = step[s]
            want, sz, reach = attend(q[start:start + n].double(), view.of(k), pos[start:start + n], None, D ** -0.5, view.value_scales(k))
            within(out[start:start + n], want, sz, reach, have[s], dtype)
            start += n


@gpu
def test_two_recorded_calls_share_no_workspace_and_replay_on_new_contents():
    lens = [2000, 1500]
    caches = [Cache(lens, 1, 64, 16, seed=s).fill(s) for s in (0, 1)]
    q = [torch.randn(2, 4, 64, device="cuda").to(torch.bfloat16) for _ in range(2)]
    out = [torch.zeros_like(t) for t in q]
    pos, seq = i32([1999, 1499]), i32([0, 1])
    call = [lambda k=k: ops.attention_kv8_decode(q[k], caches[k].pool, caches[k].scales, out[k], pos, seq, caches[k].table_dev, None, None, 0.125, 2000)
            for k in (0, 1)]
    for c in call:
        c()
    torch.cuda.synchronize()
    graphs = []
    for c in call:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c()
        graphs.append(g)
    for t in q:
        t.copy_(torch.randn_like(t))
    pos.copy_(i32([700, 1400]))
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, sides):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for k in (0, 1):
        for s, p in enumerate((700, 1400)):
            want, sz, reach = attend(q[k][s:s + 1].double(), caches[k].of(s, p + 1), pos[s:s + 1], None, 0.125, caches[k].value_scales(s, p + 1))
            within(out[k][s:s + 1], want, sz, reach, p + 1, torch.bfloat16)


@gpu
def test_the_same_call_gives_the_same_bits():
    lens = [1800, 70]
    cache = Cache(lens, 2, 64, 16).fill()
    q = torch.randn(31, 8, 64, device="cuda").to(torch.bfloat16)
    first, _ = run_attention(cache, q, [1, 30], None, 0.125)
    for _ in range(3):
        again, _ = run_attention(cache, q, [1, 30], None, 0.125)
        assert torch.equal(first, again)


# ---- copies ----

@gpu
@pytest.mark.parametrize("pairs", [1, 2, 16, 17, 300, 1100])
def test_copy_rows_of_tensors_of_all_kinds(pairs):
    rows = 2 * pairs + 3
    gen = torch.Generator().manual_seed(pairs)
    ts = [torch.randn(rows, 2, 3, 5, generator=gen).cuda(), torch.randint(0, 255, (rows, 7), generator=gen, dtype=torch.uint8).cuda(),
          torch.randn(rows, 4 * 2049, generator=gen).cuda(), torch.randn(rows, 2, 64, generator=gen).to(torch.bfloat16).cuda(),
          torch.randn(rows, 2, 2, 16, 64, generator=gen).cuda().to(F8), torch.randint(0, 9, (rows,), generator=gen, dtype=torch.int64).cuda(),
          torch.randint(0, 255, (rows * 16 + 1,), generator=gen, dtype=torch.uint8).cuda()[1:].view(rows, 16)]
    order = torch.randperm(rows, generator=gen).tolist()
    src, dst = [order[0]] + order[2:pairs + 1], order[pairs + 1:2 * pairs + 1]
    want = [t.clone() for t in ts]
    for w in want:
        w.view(torch.uint8)[dst] = w.view(torch.uint8)[src] if w.dim() > 1 else w.view(torch.uint8)[src]
    want = []
    for t in ts:
        w = t.clone()
        flat = w.view(torch.uint8).view(rows, -1) if w.dim() > 1 or w.element_size() == 1 else w.view(rows, 1).view(torch.uint8).view(rows, -1)
        flat[dst] = flat[src].clone()
        want.append(w)
    ops.copy_rows(ts, src, dst)
    for t, w in zip(ts, want):
        assert torch.equal(t.view(torch.uint8) if t.dim() > 1 else t, w.view(torch.uint8) if w.dim() > 1 else w)


@gpu
def test_one_source_for_several_destinations_and_many_tensors():
    ts = [torch.randn(9, 40 + k, device="cuda") for k in range(70)]
    want = [t.clone() for t in ts]
    for w in want:
        w[[1, 5, 8]] = w[2].clone()
    ops.copy_rows(ts, [2, 2, 2], [1, 5, 8])
    assert all(torch.equal(t, w) for t, w in zip(ts, want))
    ops.copy_rows([], [1], [2])
    ops.copy_rows(ts, [], [])


@gpu
def test_copy_rows_follows_the_stream_and_is_recorded():
    a = torch.zeros(4, 1 << 16, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        a[0].fill_(3.0)
        ops.copy_rows([a], [0], [2])
        got = a[2].clone()
    s.synchronize()
    assert (got == 3).all()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.copy_rows([a], [2, 2], [1, 3])
    a[2].fill_(5.0)
    g.replay()
    torch.cuda.synchronize()
    assert (a[1] == 5).all() and (a[3] == 5).all()


# ---- what is refused ----

def c_ints(*v):
    return (ctypes.c_int * len(v))(*v)


@pytest.mark.parametrize("src, dst, says", [
    ((1, 2), (3, 3), "destination twice"), ((1, 2), (2, 3), "both a source"), ((4,), (4,), "both a source"), ((1,), (10,), "outside"),
    ((-1,), (2,), "outside"), ((10,), (2,), "outside"), ((1,), (-5,), "outside"),
])
def test_copy_rows_refuses_rows_that_would_race_or_lie_outside(src, dst, says):
    """(The entry point's own checks, on the host: nothing is launched.)"""
    base, row, rows = (ctypes.c_void_p * 1)(256), (ctypes.c_int64 * 1)(16), c_ints(10)
    with pytest.raises(KernelError, match=says):
        _lib.call("tk_copy_rows", base, row, rows, 1, c_ints(*src), c_ints(*dst), len(src), None)


def test_entry_points_refuse_shapes_that_are_not_built():
    with pytest.raises(KernelError, match="heads of 96"):
        _lib.call("tk_qk_norm_rope_write8", 256, 96 * 3, 256, 256, 256, None, None, 0.0, None, 1.0, 0, 256, 256, 256, 1, 1, 1, 1, 96, 0, 16, 1, None)
    with pytest.raises(KernelError, match="rotary width"):
        _lib.call("tk_qk_norm_rope_write8", 256, 64 * 3, 256, 256, 256, None, None, 0.0, None, 1.0, 0, 256, 256, 256, 1, 1, 1, 1, 64, 66, 16, 1, None)
    with pytest.raises(KernelError, match="come together"):
        _lib.call("tk_qk_norm_rope_write8", 256, 64 * 3, 256, 256, 256, 256, None, 0.0, None, 1.0, 0, 256, 256, 256, 1, 1, 1, 1, 64, 0, 16, 1, None)
    with pytest.raises(KernelError, match="16 bytes"):
        _lib.call("tk_qk_norm_rope_write8", 264, 64 * 3, 256, 256, 256, None, None, 0.0, None, 1.0, 0, 256, 256, 256, 1, 1, 1, 1, 64, 0, 16, 1, None)
    for H, G, D in ((4, 3, 64), (17, 1, 64), (4, 2, 96), (4, 0, 64)):
        assert not ops.kv8_supported(H, G, D)
        with pytest.raises(KernelError, match="not taken"):
            _lib.call("tk_attn_kv8", 256, 256, 256, 256, 256, 256, 256, 1, None, None, 1, H, G, D, 16, 0, 1.0, 1, 99, 1, None, None, 0, 0, 1, None)
    with pytest.raises(KernelError, match="positive"):
        _lib.call("tk_attn_kv8", 256, 256, 256, 256, 256, 256, 256, 1, None, None, 1, 4, 2, 64, 16, 0, 0.0, 1, 99, 1, None, None, 0, 0, 1, None)
    with pytest.raises(KernelError, match="bad sizes"):
        _lib.call("tk_attn_kv8", 256, 256, 256, 256, 256, 256, 256, 1, None, None, 1, 4, 2, 64, 16, 0, 1.0, 4, 99, 1, None, None, 0, 0, 0, None)
    with pytest.raises(KernelError, match="at most 16"):
        _lib.call("tk_attn_kv8", 256, 256, 256, 256, 256, 256, 256, 1, None, None, 1, 4, 2, 64, 16, 0, 1.0, 17, 99, 1, None, None, 0, 0, 1, None)


def test_tensors_of_the_host_are_refused():
    t = torch.zeros(4, 4)
    with pytest.raises(KernelError, match="CUDA tensors only"):
        ops.copy_rows([t], [0], [1])
    pool, scales = torch.zeros(2, 2, 1, 16, 64, dtype=torch.uint8).view(F8), torch.ones(2, 2, 1)
    i = torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 1, 64)
    with pytest.raises(KernelError, match="CUDA tensors only"):
        ops.attention_kv8_decode(q, pool, scales, q, i, i, i.view(1, 1), None, None, 1.0, 1)
    with pytest.raises(KernelError, match="CUDA tensors only"):
        ops.qk_norm_rope_write8(torch.zeros(1, 192), pool, scales, None, None, 0.0, torch.zeros(0), i, i, i.view(1, 1), 1, 1, 64, 16)


@gpu
def test_tensors_that_do_not_match_are_refused():
    cache = Cache([16], 2, 64, 16).fill()
    q = torch.zeros(1, 4, 64, device="cuda", dtype=torch.bfloat16)
    one = i32([0])

    def decode(**change):
        a = dict(q=q, pool=cache.pool, scales=cache.scales, out=torch.empty_like(q), positions=one, tok_seq=one, block_table=cache.table_dev,
                 tok_index=None, window=None, scale=1.0, longest=16) | change
        ops.attention_kv8_decode(**a)

    for change, says in ((dict(pool=cache.pool.view(torch.uint8)), "float8"), (dict(scales=cache.scales.double()), "float32"),
                         (dict(scales=cache.scales[1:]), "float32"), (dict(q=q.half(), out=q.half()), "not built"),
                         (dict(out=q.float()), "one type"), (dict(q=q[:, :3], out=q[:, :3]), "multiple"),
                         (dict(positions=one[:0]), "shorter"), (dict(tok_seq=one.long()), "int32"), (dict(block_table=one), "block_table"),
                         (dict(gate=torch.zeros(1, 4, device="cuda")), "gate"), (dict(tok_index=one.long()), "int32")):
        with pytest.raises(KernelError, match=says):
            decode(**change)
    with pytest.raises(KernelError, match="first tokens"):
        ops.attention_kv8_prefill(q, cache.pool, cache.scales, q.clone(), one, one, cache.table_dev, one, i32([1, 1]), None, 1.0, 16)
    x, f = torch.zeros(1, 8 * 64, device="cuda"), torch.zeros(0, device="cuda")
    with pytest.raises(KernelError, match="heads of 64"):
        ops.qk_norm_rope_write8(x[:, 1:], cache.pool, cache.scales, None, None, 0.0, f, one, one, cache.table_dev, 4, 2, 64, 16)
    with pytest.raises(KernelError, match="does not match"):
        ops.qk_norm_rope_write8(x, cache.pool, cache.scales, None, None, 0.0, f, one, one, cache.table_dev, 4, 2, 64, 8)
    with pytest.raises(KernelError, match="contiguous"):
        ops.copy_rows([torch.zeros(4, 4, device="cuda").t()], [0], [1])
    with pytest.raises(KernelError, match="sources"):
        ops.copy_rows([x], [0], [])
    with pytest.raises(KernelError, match="32-bit"):
        ops.copy_rows([x], [0.5], [1])
