"""The 8-bit cache's operators at the calls that are easily missed: operands that lie where nobody expects them, numbers at the ends of
their range, weights that are small beside their row's largest."""

from __future__ import annotations

import math

import pytest
import torch

from test_kv8 import Cache, attend, i32, run_attention, within, write
from tokenomos_b200 import ops
from tokenomos_b200.ops import _lib

gpu = pytest.mark.gpu


def shares_of_tokens(T, H, G, D, P, n):
    """How many CTAs share each of T single tokens' keys in the tcgen05 form, behind n positions each."""
    return _lib.lib().tk_attn_kv8_tc_splits(T, H, G, D, P, n, n)


# ---- operands that lie where nobody expects them ----

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


# ---- weights that are small beside their row's largest ----

def rows_with_one_large_weight(n, H, G, D, P, share, T, seed=0):
    """A sequence of n positions whose first key takes `share` of every row's weight and has values of 0; the others' weights are log-normal, their
    values random. (cache, q [T, H, D], scale): all that q asks of a key are its first two elements, which both terms of q hold exactly."""
    gen = torch.Generator().manual_seed(seed)
    cache = Cache([n], G, D, P, seed=seed)
    pages = cache.table[0].long().cuda()
    kv = (torch.randn(len(pages), 2, G, P, D, generator=gen) * 60).to(torch.float8_e4m3fn)
    score = torch.randn(len(pages), G, P, generator=gen)
    kv.view(torch.uint8)[:, 0, :, :, 0] = (score * 64).to(torch.float8_e4m3fn).view(torch.uint8)
    kv.view(torch.uint8)[:, 0, :, :, 1] = 0
    kv.view(torch.uint8)[0, :, :, 0, :2] = 0
    kv.view(torch.uint8)[0, 1, :, 0] = 0
    kv[0, 0, :, 0, 1] = torch.tensor(256.0).to(torch.float8_e4m3fn)
    cache.pool.view(torch.uint8)[pages] = kv.view(torch.uint8).cuda()
    cache.scales[pages] = 2.0 ** -6
    first = math.log(share / (1 - share) * n * math.exp(0.5))               # (the mean of a log-normal number is e^(1/2))
    q = torch.zeros(T, H, D)
    q[..., 0], q[..., 1] = 1.0, first / 4
    return cache, q.to(torch.bfloat16).cuda(), 1.0


@gpu
@pytest.mark.parametrize("share", [0.5, 0.99, 0.999])
@pytest.mark.parametrize("n, H, G, D, P, T", [(3000, 32, 8, 64, 16, 64), (3000, 8, 8, 64, 8, 64), (2000, 64, 8, 64, 16, 40), (3000, 128, 8, 128, 16, 38), (2500, 16, 8, 128, 32, 64),
                                              (32000, 8, 2, 64, 16, 2), (32000, 4, 1, 128, 16, 1)])
def test_small_weights_beside_a_large_one_keep_their_bits(n, H, G, D, P, T, share):
    """Single tokens, unshared (T G CTAs and more fill the GPU) and shared out. The errors are independent of each other: the output's rounding (half a
    step, 2^-8 of an element), each weight's to float16's eleven bits (2^-11 of it) or to half of float16's smallest step, 2^-25 beside a largest
    weight of 2^6 at least; uniform ones, whose root mean square is their largest over sqrt(3). A quarter is left for the samples, 64 elements a
    row and more. (With q's two elements and powers of two as scales, scores are exact to 32-bit rounding: 2^-21 of a weight.)"""
    cache, q, scale = rows_with_one_large_weight(n, H, G, D, P, share, T)
    if n < 4000:
        assert shares_of_tokens(T, H, G, D, P, n) == 1
    pos, seq = i32([n - 1] * T), i32([0] * T)
    out = torch.full_like(q, 7.0)
    ops.attention_kv8_decode(q, cache.pool, cache.scales, out, pos, seq, cache.table_dev, None, None, scale, n)
    k, v = cache.of(0)
    p = torch.softmax(torch.einsum("hd,gnd->hgn", q[0, :1].double(), k)[0] * scale, -1)          # [G, n]
    assert ((p[:, 0] - share).abs() <= 0.15 * (1 - share)).all()
    want = torch.einsum("gn,gnd->gd", p, v)
    fine = torch.einsum("gn,gnd->gd", p.square(), v.square())
    coarse = p[:, :1].square() * v.square().sum(1)
    mean = (want.square() * 2.0 ** -16 + fine * 2.0 ** -22 + coarse * 2.0 ** -62).sum() / 3
    got = out.double().view(T, G, H // G, D)
    for t in range(T):
        for r in range(H // G):
            off = (got[t, :, r] - want).norm()
            assert off <= 1.25 * mean.sqrt(), (t, r, (off / want.norm()).item(), (mean.sqrt() / want.norm()).item())


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("share", [0.5, 0.999])
def test_a_prompts_last_row_and_the_same_token_decoded_agree(share, dtype):
    """A row of a portion and the same row as a single token: both within the bound above of the definition, so within twice it of each other. A 32-bit
    weight is off by its score's roundings: four of numbers of up to 40, as logarithms of 2 (2^-17 of the weight)."""
    n, H, G, D = 3000, 8, 2, 64
    cache, q, scale = rows_with_one_large_weight(n, H, G, D, 16, share, 40, seed=1)
    q = q.to(dtype)
    outs = [run_attention(cache, q[:new], [new], None, scale)[0][-1].double().view(G, H // G, D) for new in (1, 40)]
    k, v = cache.of(0)
    p = torch.softmax(torch.einsum("hd,gnd->hgn", q[0, :1].double(), k)[0] * scale, -1)
    want = torch.einsum("gn,gnd->gd", p, v)
    fine = torch.einsum("gn,gnd->gd", p.square(), v.square())
    coarse = p[:, :1].square() * v.square().sum(1)
    unit, each = torch.finfo(dtype).eps / 2, 2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -17
    mean = (want.square() * (unit ** 2 + each ** 2) + fine * each ** 2 + coarse * 2.0 ** -62).sum() / 3
    for out in outs:
        for r in range(H // G):
            assert (out[:, r] - want).norm() <= 1.25 * mean.sqrt()


# ---- queries that are not finite ----

@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("P", [16, 8, 12])
@pytest.mark.parametrize("new", [1, 20])
@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan])
def test_a_row_whose_query_is_not_finite_is_nan_and_no_other(what, new, P, dtype):
    """Keys whose first element is negative (none is 0): an infinite query element makes minus infinity of every score, and a softmax of those is no
    number."""
    H, G, D, n = 4, 2, 64, 90
    cache = Cache([n], G, D, P).fill()
    pages = cache.table[0].long().cuda()
    cache.pool.view(torch.uint8)[pages, 0, :, :, 0] = torch.tensor(-64.0).to(torch.float8_e4m3fn).view(torch.uint8).item()
    q = torch.randn(new, H, D, generator=torch.Generator().manual_seed(0)).to(dtype).cuda()
    clean, _ = run_attention(cache, q, [new], None, 0.125)
    bad = q.clone()
    bad[-1, 2, 0] = what
    out, _ = run_attention(cache, bad, [new], None, 0.125)
    assert out[-1, 2].isnan().all()
    out[-1, 2] = clean[-1, 2]
    assert torch.equal(out, clean) and torch.isfinite(clean).all()


# ---- norms ----

@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
def test_a_head_whose_squares_overflow_is_zero_as_in_the_16_bit_write(D, dtype):
    """Elements of 1e25: their squares' mean is infinite in 32 bits, what is divided by its root is 0, in the query, in the cached key, and in
    ``qk_norm_rope_write``; the token is not marked. One infinite element makes NaN of the head and marks the token in its KV head."""
    H, G, P = 2, 2, 16
    g = torch.Generator().manual_seed(D)
    x = torch.randn(4, H + 2 * G, D, generator=g)
    x[1, :H + G] *= 1e25
    x[2, 0, 5] = math.inf
    x[2, H + 1, 7] = math.inf
    x = x.to(dtype).cuda()
    w = (torch.rand(2, D, generator=g) + 0.5).cuda()
    freq = torch.exp(-torch.arange(D // 2) * 0.2).cuda()
    cache = Cache([4], G, D, P)
    q, pos = write(cache, [(0, 0, x.view(4, -1))], H, w[0].contiguous(), w[1].contiguous(), 1e-6, freq)
    wide = torch.zeros(cache.pool.shape, dtype=dtype, device="cuda")
    q16 = ops.qk_norm_rope_write(x.view(4, -1), wide, w[0].contiguous(), w[1].contiguous(), 1e-6, freq, pos, i32([0] * 4), cache.table_dev, H, G, D, P)
    page = int(cache.table[0, 0])
    assert (q16[1] == 0).all() and (wide[page, 0, :, 1] == 0).all()
    assert (q[1] == 0).all() and (cache.of(0)[0, :, 1] == 0).all()
    assert torch.isfinite(q[[0, 1, 3]].float()).all() and torch.isfinite(cache.of(0)[:, :, [0, 1, 3]]).all()
    assert q[2, 0].isnan().any() and torch.isfinite(q[2, 1].float()).all()
    assert cache.of(0)[0, 1, 2].isnan().all() and torch.isfinite(cache.of(0)[0, 0, 2]).all()
    # (values are not normed)
    v = x[1, H + G:].double()
    assert ((cache.of(0)[1, :, 1] - v).abs() <= v.abs() / 16 + cache.value_scales(0)[:, 1:2] * 2.0 ** -10).all()


# ---- how many CTAs share a row's keys ----

@gpu
@pytest.mark.parametrize("P", [8, 16, 64])
@pytest.mark.parametrize("H, G, D, places", [(8, 8, 64, 4), (32, 8, 64, 4), (4, 1, 64, 4), (8, 1, 64, 2), (16, 1, 64, 2), (2, 2, 128, 2), (32, 4, 128, 2), (9, 1, 128, 1),
                                              (16, 1, 128, 1), (64, 4, 128, 1)])
def test_single_tokens_keys_are_shared_by_as_many_ctas_as_are_resident(H, G, D, places, P):
    """`places`: CTAs of the kernel that an SM holds, by its shared memory of up to 228 KB (a KV head of 128 with more than eight query heads: 119 KB a
    CTA, so one) and its registers."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    for T in (1, 2, 4, 9, 18, 36, 37, 64, 100, 148, 200, 600):
        for n in (1, 128, 500, 2048, 9000, 30000):
            shares = shares_of_tokens(T, H, G, D, P, n)
            assert 1 <= shares <= 16 and (shares == 1 or shares * T * G <= places * sms), (T, n, shares)
            assert shares <= max(1, -(-n // 128))
    assert shares_of_tokens(1, H, G, D, P, 2048) == 8


# the most clusters of 3, 4, ... CTAs that ran together on a B200's 148 SMs, by CTAs an SM (one more, and a launch took half as long again)
TOGETHER = {1: {2: 74, 3: 45, 4: 33, 5: 26, 6: 22, 7: 15, 8: 15, 16: 7}, 2: {2: 148, 3: 92, 4: 70, 5: 56, 6: 45, 7: 37, 8: 33, 16: 14},
            4: {2: 296, 3: 185, 4: 140, 5: 112, 6: 92, 7: 76, 8: 66, 16: 28}}


@gpu
@pytest.mark.parametrize("H, G, D, places", [(4, 1, 64, 4), (4, 2, 64, 4), (8, 1, 64, 2), (16, 1, 64, 2), (8, 2, 128, 2), (16, 1, 128, 1)])
def test_clusters_of_single_tokens_leave_the_places_empty_that_they_cannot_fill(H, G, D, places):
    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("counted on 148 SMs")
    for T in range(1, 310 // G):
        for n in (500, 900, 2000, 4000, 9000, 30000):
            shares = shares_of_tokens(T, H, G, D, 16, n)
            assert shares == 1 or T * G <= TOGETHER[places][shares], (T, n, shares)
    # and those that they can
    for want, n in ((4, 500), (8, 4000), (16, 9000)):
        assert shares_of_tokens(TOGETHER[places][want] * 9 // 10 // G, H, G, D, 16, n) == want


@gpu
@pytest.mark.parametrize("T, n", [(18, 2100), (36, 1500), (64, 900), (160, 300)])
def test_a_kv_head_of_128_with_16_query_heads_whatever_its_shares(T, n):
    """(Rows of one sequence at the same position: what each asks differs.)"""
    H, G, D = 16, 1, 128
    cache = Cache([n], G, D, 16).fill()
    q = torch.randn(T, H, D, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16).cuda()
    out = torch.full_like(q, 7.0)
    pos = i32([n - 1] * T)
    ops.attention_kv8_decode(q, cache.pool, cache.scales, out, pos, i32([0] * T), cache.table_dev, None, None, D ** -0.5, n)
    want, sz, reach = attend(q.double(), cache.of(0), pos, None, D ** -0.5, cache.value_scales(0))
    within(out, want, sz, reach, n, torch.bfloat16)


@gpu
@pytest.mark.parametrize("H, G, D", [(16, 4, 128), (8, 8, 128), (32, 1, 128), (16, 4, 64), (32, 8, 64)])
def test_portions_keys_are_shared_by_as_many_ctas_as_are_resident(H, G, D):
    """Heads of 128 have one CTA an SM, and an eighth of the SMs or so has no room for clusters of four, nearly a fifth none for clusters of eight;
    heads of 64 have two, and 16 of those places no room."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    for tokens in (40, 100, 128, 144, 250, 288, 544, 560, 1200, 5000):
        tiles = -(-tokens // (128 // (H // G)))
        for P in (8, 16):
            for n in (300, 2500, 4200, 8300, 16000, 30000):
                shares = _lib.lib().tk_attn_kv8_prefill_splits(tokens, tiles, H, G, D, P, n, sms)
                ctas = shares * tiles * G
                assert shares in (1, 2, 4, 8)
                if D == 128:
                    assert shares == 1 or ctas <= {2: 148, 4: 136, 8: 128}[shares], (tokens, n, shares)
                else:
                    assert shares == 1 or ctas <= 296 - 16 * (shares > 2) or (shares == 8 and ctas <= 296 and n >= 16384), (tokens, n, shares)
    assert _lib.lib().tk_attn_kv8_prefill_splits(H // G, 1, H, G, D, 16, 8300, sms) == 8


@pytest.mark.parametrize("dtype, P, D, places", [("f32", 16, 64, 3), ("f32", 8, 64, 3), ("f32", 12, 64, 2), ("f32", 4, 64, 2), ("f32", 16, 128, 2), ("bf16", 12, 64, 2),
                                                  ("bf16", 4, 64, 2), ("bf16", 5, 128, 2)])
def test_the_other_forms_keys_are_shared_by_what_its_kernels_leave_room_for(dtype, P, D, places):
    """(The rule on the host, for 148 SMs.) Beyond what is resident only threes, where fewer than two would be and the sequences are long."""
    code = _lib.F32 if dtype == "f32" else _lib.BF16
    for items in (1, 3, 8, 11, 14, 20, 25, 31, 37, 42, 64, 300):
        for n in (1, 512, 513, 1200, 2500, 30000):
            for single in (0, 1):
                shares = _lib.call("tk_attn_kv8_splits", items, 16, 8, D, P, code, n, n, single, 148)
                assert shares >= 1 and (n > 512 or shares == 1) and shares <= -(-n // 256)
                fit = places * 148 // (items * 8)
                assert shares <= max(1, fit) or (shares == 3 and fit <= 1 and n >= 1024), (items, n, shares)
    assert _lib.call("tk_attn_kv8_splits", 8, 16, 8, D, P, code, 4000, 4000, 1, 148) == (6 if places == 3 else 4)
