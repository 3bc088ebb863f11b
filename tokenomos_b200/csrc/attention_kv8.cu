// Attention over the 8-bit cache (kv8.cuh) on mma.sync.m16n8k16, with float16 operands and 32-bit sums: all of the 32-bit
// models, and pages that the tcgen05 kernels (attention_kv8_tc.cu, attention_kv8_prefill.cu) do not take.
//
//   o[r] = sum_j p_rj v_j / sum_j p_rj,   p_rj = exp(scale * q_r . k_j),   k_j = s_K kb_j,  v_j = s_V vb_j   (bytes kb, vb)
//
// A CTA takes 16 rows (tokens of one sequence x the query heads of one KV head; one token when it decodes) and a share of their
// keys; its warps walk groups of 32 (16 for heads of 128) keys in turn and are joined through shared memory, the CTAs of a
// row through scratch memory and a second kernel.
//
// Pages of a power of two of 8 positions and more come by bulk copies (32-bit), up to three units of 32 keys (heads of 128: 16) a warp in shared memory or on their way; smaller or odd ones are read by
// each lane. From bytes to operands nothing is moved between lanes: the order of a product's inner index is free as long as both operands follow it, and the order of the output's columns is
// too: a lane reads D / 4 bytes side by side of one key's row (16 bytes for D = 64; four lanes a row) and uses them as its fragments of all the D / 16
// steps of q . k, with q's fragments laid out to match; and of a value row it reads D / 8 bytes, one for each of the D / 8 column tiles, so that two rows' bytes
// interleave (prmt) into the pairs that a fragment holds. e4m3 is exact in float16.
//
// What is rounded: q (bfloat16: not at all, 32-bit: to 22 bits, as two float16 with two products) after division by a power of two that brings its row
// to [2^14, 2^15), so that its small elements keep their bits; the weights (of the bytes) to float16's 11 bits (32-bit: 22,
// as two) or, where that is more, to 2^-32 of the row's largest: half of float16's smallest step against 2^7, which that one has at least. Scores, the running
// maximum, sums and outputs are 32-bit; the output is rounded once.
//
// A value block's scale joins the exponent: with x_j = log2(p_j) + log2(s_V), w_j = 2^(x_j - m + 7) are the weights of the bytes, m following their
// running maximum lazily (it is raised when a row exceeds it by 8, so w <= 2^15), and the softmax's sum is of w_j / s_V. A weight
// then loses bits to float16's range only beside one that gives the output that much more a byte, however far apart the blocks' scales are.
//
// Masked keys and values are never read (their bytes are zero in the products), so what an unwritten part of a page holds does not
// matter. A row that sees no key is 0.
//
// Measured (32-bit, 16 heads over 8 of 64, one B200): two prompts of up to 301 tokens 15.6 us, 1,000 tokens 31.4, 8 single tokens behind up to 4,000 positions 17.0 (1.7 TB/s), one
// behind 2,000 9.4. Keys that each lane looks up (bfloat16, 32 heads over 8 of 64, pages of 12): 1,000 tokens 166, 256 behind 4,000 304, 8 single tokens behind up to 4,000 42.7; 64 behind up to 1,000, pages
// of 4, 70.5. Bound by latency: 168 registers leave three CTAs an SM (the two prompts in two shares each 23.9 us, with two CTAs 27.3; units of 16 keys allow four: 12.9 for the two prompts, but 34.6 for the
// 1,000 tokens and 49.5 for 34.5 unshared single tokens). A warp a row tile instead of a share of a CTA's keys was slower for prompts.
#include <math.h>

#include <type_traits>

#include "kv8_attn.cuh"

namespace {

constexpr int K8_ROWS = 16;
constexpr int K8_WARPS = 4, K8_THREADS = K8_WARPS * 32;
constexpr int K8_DEPTH = 3;                       // units of keys and values a warp has in shared memory or on their way
constexpr float K8_LAZY = 8.0f, K8_LIFT = 7.0f;

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// T: type of q and the output. D: head size. KG: 16 where pages are a power of two of 16 positions or more, so 16 keys that begin at a multiple of 16 lie in
// one page, 8 for pages of 8; 0: every lane looks its own keys' pages up.
template <typename T, int D, int KG>
__global__ void __launch_bounds__(K8_THREADS, D == 64 && KG > 0 ? 3 : 2)
attn_kv8_kernel(const T* q, const uint8_t* pool, const float* scales, T* out, const K8Args a) {
    constexpr bool WIDE = sizeof(T) == 4;                // q and the weights as two float16
    constexpr int U = D == 64 ? 2 : 1;                   // groups of 16 keys a warp takes at a time
    constexpr int KS = D / 16, NT = D / 8;               // steps of q . k, column tiles of the output
    constexpr int KW = D / 64;                           // 16-byte words a lane reads of a key
    constexpr int VW = D / 32;                           // 4-byte words a lane reads of a value row
    constexpr int UNIT = U * 32 * D;                     // a unit's bytes
    constexpr bool BULK = KG > 0;
    constexpr int HALVES = KG == 8 ? 2 : 1, PIECES = U * HALVES;      // pages' pieces (of KG keys) of a group, of a unit
    extern __shared__ __align__(128) float smem[];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, c = lane & 3;
    const int split = blockIdx.x % a.nsplit, kvh = (blockIdx.x / a.nsplit) % a.Hkv, item = blockIdx.x / (a.nsplit * a.Hkv);
    const int tok0 = a.item_tok0 != nullptr ? a.item_tok0[item] : item;
    const int ntok = a.item_ntok != nullptr ? min(a.item_ntok[item], K8_ROWS / (a.H / a.Hkv)) : 1;       // (a longer tile's rest is left alone)
    if (tok0 < 0 || ntok <= 0) return;                   // a padded entry of a recorded step
    const int G = a.H / a.Hkv, rows = ntok * G;
    const int* bt = a.block_table + (size_t)a.tok_seq[tok0] * a.bt_stride;
    const int pos_first = a.positions[tok0], pos_last = pos_first + ntok - 1;
    const int lo = first_seen(pos_first, a.window), lo_last = first_seen(pos_last, a.window);
    // groups of 16 keys, from the one that holds `lo`; this CTA's are [g_begin, g_end), its warps take U of them in turn
    const int g_lo = lo >> 4, g_all = (pos_last >> 4) - g_lo + 1;
    const int all_units = (g_all + U - 1) / U;
    const int g_begin = g_lo + (int)((int64_t)all_units * split / a.nsplit) * U;
    const int g_end = min(g_lo + (int)((int64_t)all_units * (split + 1) / a.nsplit) * U, g_lo + g_all);

    // ---- q: rows g and g + 8, columns [c D / 4, (c + 1) D / 4) ----
    uint32_t qa[KS][4], qb[WIDE ? KS : 1][4];
    float row_c[2];
    int row_pos[2];
#pragma unroll
    for (int hrow = 0; hrow < 2; ++hrow) {
        const int r = g + 8 * hrow;
        const bool valid = r < rows;
        const T* src = q + ((size_t)(tok0 + (valid ? r / G : 0)) * a.H + kvh * G + (valid ? r % G : 0)) * D + c * (D / 4);
        float x[D / 4];
        float most = 0.f;
#pragma unroll
        for (int e = 0; e < D / 4; e += 4) {
            const float4 v = Quad<T>::load(src + e);
            x[e] = v.x, x[e + 1] = v.y, x[e + 2] = v.z, x[e + 3] = v.w;
        }
#pragma unroll
        for (int e = 0; e < D / 4; ++e) {
            if (!valid) x[e] = 0.f;
            most = fmaxf(most, fabsf(x[e]));
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // a row's largest element to [2^14, 2^15); of a row with an infinite element every score is NaN (minus infinities alone would pass for a row that
        // sees nothing), as one NaN makes it by itself
        int e2 = (__float_as_int(most) >> 23) - 127;
        const bool fine = e2 <= 127;
        e2 = !fine || most == 0.f ? 14 : max(e2, -100);
        const float up = fine ? exp2i(14 - e2) : NAN;
        row_c[hrow] = a.scale * K8_LOG2E * exp2i(e2 - 14);
        row_pos[hrow] = valid ? pos_first + r / G : -1;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const float u = x[4 * ks + 2 * half] * up, v = x[4 * ks + 2 * half + 1] * up;
                qa[ks][hrow + 2 * half] = half2_bits(u, v);
                if constexpr (WIDE) {
                    const float2 hi = half2_floats(qa[ks][hrow + 2 * half]);
                    qb[ks][hrow + 2 * half] = half2_bits(u - hi.x, v - hi.y);
                }
            }
    }

    // ---- where keys and values come from ----
    const int P = a.P;
    const size_t v_delta = (size_t)a.Hkv * P * D, page_bytes = 2 * v_delta;
    const uint8_t* head = pool + (size_t)kvh * P * D;
    const int units = (g_end - g_begin + U - 1) / U;
    const int mine = units > warp ? (units - warp + K8_WARPS - 1) / K8_WARPS : 0;         // this warp's: unit warp, warp + K8_WARPS, ...
    auto group_of = [&](int k, int u) { return g_begin + (warp + k * K8_WARPS) * U + u; };
    // lane i knows the page and, from when its bytes are asked for, the scales of piece i of a block of 32 pieces
    constexpr int BLOCK = 32 / PIECES;
    int page_now = 0, page_then = 0;
    float sk_now = 1.f, sv_now = 1.f, sk_then = 1.f, sv_then = 1.f;
    const int p_end = BULK ? min(g_end * HALVES, pos_last / (BULK ? KG : 16) + 1) : 0;       // (the last group's second page may not be there)
    auto piece_of = [&](int k, int i) { return group_of(k, 0) * HALVES + i; };
    auto page_of_block = [&](int block) {
        const int pc = piece_of(block * BLOCK + lane / PIECES, lane % PIECES);
        return pc < p_end ? TK_PAGE(TK_K_KV8_ATTN, bt[(pc * KG) >> a.p_shift]) : -1;
    };
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + (uint32_t)warp * (K8_DEPTH * UNIT);
    const uint32_t bars = (uint32_t)__cvta_generic_to_shared(smem) + K8_WARPS * K8_DEPTH * UNIT + (uint32_t)warp * (K8_DEPTH * 8);
    const uint8_t* stage = reinterpret_cast<const uint8_t*>(smem) + warp * (K8_DEPTH * UNIT);
    auto issue = [&](int k) {
        if (k >= mine) return;
        if (k % BLOCK == 0) {
            page_now = k == 0 ? page_of_block(0) : page_then;
            page_then = page_of_block(k / BLOCK + 1);
            const float* sc = scales + (size_t)max(page_now, 0) * (2 * a.Hkv) + kvh;
            sk_then = page_now >= 0 ? sc[0] : 1.f;
            sv_then = page_now >= 0 ? sc[a.Hkv] : 1.f;
        }
        const int first = piece_of(k, 0), n = min(PIECES, p_end - first);
        const uint32_t bar = bars + (uint32_t)(k % K8_DEPTH) * 8;
        const int page = __shfl_sync(0xffffffffu, page_now, (k % BLOCK) * PIECES + (lane >> 1) % PIECES);
        if (lane == 0)
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(n * 2 * KG * D) : "memory");
        __syncwarp();
        if (lane < 2 * n) {
            const int i = lane >> 1, which = lane & 1;
            const uint8_t* src = head + (size_t)page * page_bytes + which * v_delta + (uint32_t)((((first + i) * KG) & (P - 1)) * D);
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                             ring + (uint32_t)(k % K8_DEPTH) * UNIT + (uint32_t)(i / HALVES * 32 * D + which * 16 * D + i % HALVES * KG * D)),
                         "l"(src), "r"(KG * D), "r"(bar)
                         : "memory");
        }
    };
    if constexpr (BULK) {
        if (lane == 0) {
            for (int i = 0; i < K8_DEPTH; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bars + i * 8) : "memory");
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        __syncwarp();
        for (int k = 0; k < K8_DEPTH - 1; ++k) issue(k);
    }
    // A key's place among a group's 16: tile t, column n holds key 8 t + order(n); with it the value rows that the four lanes of a column read lie
    // on both halves of the banks, and so do two neighbouring columns' keys.
    auto order = [](int n) { return n ^ ((n >> 1) & 1); };
    const int k_row = order(g), v_row0 = order(2 * c), v_row1 = order(2 * c + 1);
    auto key_in_group = [&](int t, int e) { return 8 * t + (e ? v_row1 : v_row0); };       // of this lane's columns 2c + e
    bool waited = true;

    float o[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    for (int k = 0; k < mine; ++k) {
        const int gr = group_of(k, 0);
        const bool inner = (gr << 4) >= lo && ((gr + U) << 4) <= min(pos_last + 1, g_end << 4);      // all of its keys are read
        const uint8_t* here = stage + (k % K8_DEPTH) * UNIT;
        constexpr int NS = BULK ? HALVES : 4;            // scales a group has for a lane: one, two (its tiles'), or one for each of its four keys
        auto scale_at = [](int t, int e) { return NS == 1 ? 0 : NS == 2 ? t : 2 * t + e; };
        float ksc[U][NS], vsc[U][NS];
        uint4 kw[U][2][KW];
        if constexpr (BULK) {
            issue(k + K8_DEPTH - 1);
            if (k % BLOCK == 0) {                        // (asked for when the first of the block's bytes were)
                sk_now = sk_then;
                sv_now = sv_then;
            }
            waited = waited && k8_wait(bars + (uint32_t)(k % K8_DEPTH) * 8, (uint32_t)((k / K8_DEPTH) & 1));
            if (!__all_sync(0xffffffffu, waited)) break;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int w = 0; w < KW; ++w)
                        kw[u][t][w] = *reinterpret_cast<const uint4*>(here + u * 32 * D + (8 * t + k_row) * D + c * (D / 4) + 16 * w);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int j = ((gr + u) << 4) + 8 * t + k_row;
                    const bool there = gr + u < g_end && j >= lo && j <= pos_last;
#pragma unroll
                    for (int w = 0; w < KW; ++w) kw[u][t][w] = make_uint4(0u, 0u, 0u, 0u);
                    if (there) {
                        const uint8_t* src = head + (size_t)TK_PAGE(TK_K_KV8_ATTN, bt[j / P]) * page_bytes + (size_t)(j % P) * D + c * (D / 4);
#pragma unroll
                        for (int w = 0; w < KW; ++w) kw[u][t][w] = *reinterpret_cast<const uint4*>(src + 16 * w);
                    }
                }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = ((gr + u) << 4) + key_in_group(i >> 1, i & 1);
                    const bool there = gr + u < g_end && j >= lo && j <= pos_last;
                    const float* sc = scales + (size_t)(there ? TK_PAGE(TK_K_KV8_ATTN, bt[j / P]) : 0) * (2 * a.Hkv) + kvh;
                    ksc[u][i] = there ? sc[0] : 1.f;
                    vsc[u][i] = there ? sc[a.Hkv] : 1.f;
                }
        }
        // products of keys 2c, 2c + 1 of tile t with rows g and g + 8; a key's logarithm is x * kc + ev, with the value block's exponent in it
        float x[U][2][4], kc[U][NS][2], ev[U][NS], inv_vs[U][NS];
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[u][t][e] = 0.f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const uint4 w4 = kw[u][t][ks >> 2];
                    const uint32_t w = (ks & 3) == 0 ? w4.x : (ks & 3) == 1 ? w4.y : (ks & 3) == 2 ? w4.z : w4.w;
                    const uint32_t b0 = e4m3x2_to_half2((uint16_t)w), b1 = e4m3x2_to_half2((uint16_t)(w >> 16));
                    mma_f16(x[u][t], qa[ks], b0, b1);
                    if constexpr (WIDE) mma_f16(x[u][t], qb[ks], b0, b1);
                }
            }
            if constexpr (BULK) {
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    ksc[u][i] = __shfl_sync(0xffffffffu, sk_now, (k % BLOCK) * PIECES + u * HALVES + i);
                    vsc[u][i] = __shfl_sync(0xffffffffu, sv_now, (k % BLOCK) * PIECES + u * HALVES + i);
                }
            }
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                // of a power of two: its exponent as a number, and its inverse
                const int bits = __float_as_int(vsc[u][i]);
                ev[u][i] = __int_as_float(0x4b000000 | (bits >> 23)) - 8388735.0f;
                inv_vs[u][i] = __int_as_float((254 << 23) - bits);
                // (never 0: what is hidden is minus infinity before it is multiplied)
                kc[u][i][0] = fmaxf(ksc[u][i] * row_c[0], 1.2e-38f);
                kc[u][i][1] = fmaxf(ksc[u][i] * row_c[1], 1.2e-38f);
            }
            const int j0 = (gr + u) << 4;
            if (j0 + 15 > pos_first || j0 < lo_last || gr + u >= g_end) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = j0 + key_in_group(t, e & 1), p = row_pos[e >> 1];
                        if (j > p || j < first_seen(p, a.window) || gr + u >= g_end) x[u][t][e] = -INFINITY;
                    }
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                if constexpr (NS == 1) {
                    const float most = fmaxf(fmaxf(x[u][0][2 * r], x[u][0][2 * r + 1]), fmaxf(x[u][1][2 * r], x[u][1][2 * r + 1]));
                    top[r] = fmaxf(top[r], fmaf(most, kc[u][0][r], ev[u][0]));
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        top[r] = fmaxf(top[r], fmaf(x[u][i >> 1][2 * r + (i & 1)], kc[u][scale_at(i >> 1, i & 1)][r], ev[u][scale_at(i >> 1, i & 1)]));
                }
            }
        }
        if (__any_sync(0xffffffffu, top[0] > m[0] + K8_LAZY || top[1] > m[1] + K8_LAZY)) {
#pragma unroll
            for (int hrow = 0; hrow < 2; ++hrow) {
                float t = fmaxf(top[hrow], __shfl_xor_sync(0xffffffffu, top[hrow], 1));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
                const float m_new = fmaxf(m[hrow], t);
                const float f = m_new == -INFINITY ? 1.f : k8_exp2(m[hrow] - m_new);
                m[hrow] = m_new;
                l[hrow] *= f;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    o[j][2 * hrow] *= f;
                    o[j][2 * hrow + 1] *= f;
                }
            }
        }
        const float base[2] = {m[0] == -INFINITY ? 0.f : K8_LIFT - m[0], m[1] == -INFINITY ? 0.f : K8_LIFT - m[1]};
#pragma unroll
        for (int u = 0; u < U; ++u) {
            uint32_t pa[4], pb[4];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int hrow = 0; hrow < 2; ++hrow) {
                    const int i0 = scale_at(t, 0), i1 = scale_at(t, 1);
                    const float w0 = k8_exp2(fmaf(x[u][t][2 * hrow], kc[u][i0][hrow], ev[u][i0] + base[hrow]));
                    const float w1 = k8_exp2(fmaf(x[u][t][2 * hrow + 1], kc[u][i1][hrow], ev[u][i1] + base[hrow]));
                    l[hrow] = fmaf(w0, inv_vs[u][i0], l[hrow]);
                    l[hrow] = fmaf(w1, inv_vs[u][i1], l[hrow]);
                    pa[hrow + 2 * t] = half2_bits(w0, w1);
                    if constexpr (WIDE) {
                        const float2 hi = half2_floats(pa[hrow + 2 * t]);
                        pb[hrow + 2 * t] = half2_bits(w0 - hi.x, w1 - hi.y);
                    }
                }
            uint32_t vw[4][VW];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = key_in_group(i >> 1, i & 1), j = ((gr + u) << 4) + row;
                const bool there = inner || (gr + u < g_end && j >= lo && j <= pos_last);
                const uint8_t* src = here + u * 32 * D + 16 * D + row * D + g * (D / 8);
                if constexpr (!BULK)
                    if (there) src = head + (size_t)TK_PAGE(TK_K_KV8_ATTN, bt[j / P]) * page_bytes + v_delta + (size_t)(j % P) * D + g * (D / 8);
                // (what is not to be read is in shared memory all the same where a page's bytes came as one, and never matters)
                if constexpr (VW == 2) {
                    uint2 v = make_uint2(0u, 0u);
                    if (there) v = *reinterpret_cast<const uint2*>(src);
                    vw[i][0] = v.x, vw[i][1] = v.y;
                } else {
                    uint4 v = make_uint4(0u, 0u, 0u, 0u);
                    if (there) v = *reinterpret_cast<const uint4*>(src);
                    vw[i][0] = v.x, vw[i][1] = v.y, vw[i][2] = v.z, vw[i][3] = v.w;
                }
            }
#pragma unroll
            for (int w = 0; w < VW; ++w)
#pragma unroll
                for (int pair = 0; pair < 2; ++pair) {
                    const uint32_t sel = pair ? 0x7362 : 0x5140;
                    const uint32_t y0 = __byte_perm(vw[0][w], vw[1][w], sel), y1 = __byte_perm(vw[2][w], vw[3][w], sel);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int j = 4 * w + 2 * pair + e;
                        const uint32_t b0 = e4m3x2_to_half2((uint16_t)(y0 >> (16 * e))), b1 = e4m3x2_to_half2((uint16_t)(y1 >> (16 * e)));
                        mma_f16(o[j], pa, b0, b1);
                        if constexpr (WIDE) mma_f16(o[j], pb, b0, b1);
                    }
                }
        }
    }
#pragma unroll
    for (int hrow = 0; hrow < 2; ++hrow) {
        l[hrow] += __shfl_xor_sync(0xffffffffu, l[hrow], 1);
        l[hrow] += __shfl_xor_sync(0xffffffffu, l[hrow], 2);
        float t = fmaxf(m[hrow], __shfl_xor_sync(0xffffffffu, m[hrow], 1));       // (equal in the four already)
        m[hrow] = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
    }

    __syncthreads();                                     // (the ring's place is used again)
    // ---- the warps' shares joined: [warp][row] D floats (4 apart from a power of two) and [warp][row] (m, l) ----
    constexpr int LD = D + 4;
    float* share = smem;
    float2* ml = reinterpret_cast<float2*>(smem + K8_WARPS * K8_ROWS * LD);
#pragma unroll
    for (int hrow = 0; hrow < 2; ++hrow) {
        float* dst = share + (warp * K8_ROWS + g + 8 * hrow) * LD + c * (D / 4);
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int j = 0; j < NT; j += 4)
                *reinterpret_cast<float4*>(dst + e * NT + j) = make_float4(o[j][2 * hrow + e], o[j + 1][2 * hrow + e], o[j + 2][2 * hrow + e], o[j + 3][2 * hrow + e]);
        if (c == 0) ml[warp * K8_ROWS + g + 8 * hrow] = make_float2(m[hrow], l[hrow]);
    }
    __syncthreads();
    for (int i = tid; i < rows * (D / 4); i += K8_THREADS) {
        const int r = i / (D / 4), col = (i % (D / 4)) * 4;
        float m_all = -INFINITY, l_all = 0.f;
#pragma unroll
        for (int w = 0; w < K8_WARPS; ++w) m_all = fmaxf(m_all, ml[w * K8_ROWS + r].x);
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < K8_WARPS; ++w) {
            const float2 s = ml[w * K8_ROWS + r];
            const float f = k8_factor(s.x, s.y, m_all);
            l_all = fmaf(s.y, f, l_all);
            const float4 p = *reinterpret_cast<const float4*>(share + (w * K8_ROWS + r) * LD + col);
            v[0] = fmaf(p.x, f, v[0]), v[1] = fmaf(p.y, f, v[1]), v[2] = fmaf(p.z, f, v[2]), v[3] = fmaf(p.w, f, v[3]);
        }
        const int tok = tok0 + r / G, hd = kvh * G + r % G;
        if (a.nsplit == 1) {
            if (a.sink && m_all > -INFINITY) l_all += k8_exp2(K8_LIFT - m_all);
            const float inv = l_all == 0.f ? 0.f : 1.f / l_all;
            float4 y;
            const float gate = k8_gate<T>(a, tok, hd);
            y.x = k8_apply<T>(v[0] * inv, a, gate), y.y = k8_apply<T>(v[1] * inv, a, gate);
            y.z = k8_apply<T>(v[2] * inv, a, gate), y.w = k8_apply<T>(v[3] * inv, a, gate);
            Quad<T>::store(out + ((size_t)tok * a.H + hd) * D + col, y);
        } else {
            float* part = a.scratch + ((((size_t)item * a.Hkv + kvh) * a.nsplit + split) * a.rows_most + r) * (D + 4);
            *reinterpret_cast<float4*>(part + col) = make_float4(v[0], v[1], v[2], v[3]);
            if (col == 0) *reinterpret_cast<float2*>(part + D) = make_float2(m_all, l_all);
        }
    }
}

template <typename T, int D, int KG>
cudaError_t k8_launch(const void* q, const void* pool, const float* scales, void* out, const K8Args& a, cudaStream_t stream) {
    constexpr int shares = (K8_WARPS * K8_ROWS * (D + 4) + 2 * K8_WARPS * K8_ROWS) * 4;
    constexpr int ring = KG > 0 ? K8_WARPS * K8_DEPTH * (4096 + 8) : 0;
    constexpr int smem = ring > shares ? ring : shares;
    if (smem > 48 * 1024) {
        static std::atomic<uint64_t> done{0};
        const cudaError_t e = k8_allow(attn_kv8_kernel<T, D, KG>, smem, false, done);
        if (e != cudaSuccess) return e;
    }
    return tk_launch(attn_kv8_kernel<T, D, KG>, dim3((unsigned)(a.items * a.Hkv * a.nsplit)), dim3(K8_THREADS), smem, stream, (const T*)q,
                     (const uint8_t*)pool, scales, (T*)out, a);
}

// (bfloat16 comes here for pages that the tcgen05 kernels do not take)
template <typename T, int D>
cudaError_t k8_pages(const void* q, const void* pool, const float* scales, void* out, const K8Args& a, cudaStream_t stream) {
    if constexpr (sizeof(T) == 4) {
        if (a.p_shift >= 4) return k8_launch<T, D, 16>(q, pool, scales, out, a, stream);
        if (a.p_shift == 3) return k8_launch<T, D, 8>(q, pool, scales, out, a, stream);
    }
    return k8_launch<T, D, 0>(q, pool, scales, out, a, stream);
}

template <typename T>
cudaError_t k8_dispatch(const void* q, const void* pool, const float* scales, void* out, const K8Args& a, int D, cudaStream_t stream) {
    const cudaError_t e = D == 64 ? k8_pages<T, 64>(q, pool, scales, out, a, stream) : k8_pages<T, 128>(q, pool, scales, out, a, stream);
    if (e != cudaSuccess || a.nsplit == 1) return e;
    const unsigned grid = (unsigned)(((int64_t)a.items * a.Hkv * a.rows_most + 3) / 4);
    return D == 64 ? tk_launch(attn_kv8_merge_kernel<T, 64>, dim3(grid), dim3(128), 0, stream, (T*)out, a, K8_LIFT)
                   : tk_launch(attn_kv8_merge_kernel<T, 128>, dim3(grid), dim3(128), 0, stream, (T*)out, a, K8_LIFT);
}

}  // namespace

// Whether the 8-bit cache's kernels take a layer: heads of 64 or 128, up to 16 query heads a KV head.
TK_API int tk_attn_kv8_supported(int H, int Hkv, int D) {
    return Hkv > 0 && H > 0 && H % Hkv == 0 && H / Hkv <= K8_ROWS && (D == 64 || D == 128);
}

// Whether prompt portions of this shape take the tcgen05 kernel: 16-bit, pages that are a power of two and 8 or more positions.
TK_API int tk_attn_kv8_prefill_supported(int H, int Hkv, int D, int P, int dtype) {
    return tk_attn_kv8_supported(H, Hkv, D) && dtype == TK_BF16 && P >= 8 && (P & (P - 1)) == 0;
}

int tk_attn_kv8_prefill_clusters(int D, int P, int n, int sm_count);

// Tokens of one sequence a tile of tk_attn_kv8 has.
TK_API int tk_attn_kv8_tokens(int H, int Hkv, int D, int P, int dtype) {
    return (tk_attn_kv8_prefill_supported(H, Hkv, D, P, dtype) ? 128 : K8_ROWS) / (H / Hkv);
}

// The most CTAs (1, 2, 4 or 8, a cluster) that may share one tile's keys in the tcgen05 kernel for portions, for a step of `tokens` tokens in tiles of
// 128 / G whose list has `items` entries (a captured step's is longer than what it uses): doubled while each keeps 8 key tiles, all CTAs are resident (heads of
// 64: two an SM, 128: one), and from two on, beyond one an SM, only where each keeps 32 (two CTAs of an SM walk at 0.7 of one's pace). Eight of heads of 64 pay behind 16,384
// positions even if the last of them wait. (us; 16 heads over 4 of 128: 128 tokens behind 8,000 39.4 by 4, 55.4 by 8, which are not resident; 288 behind 4,000 36.5 by 2, 53.8 by
// 4. Of 64: 544 behind 7,000 44.9 by 2, 41.9 by 4; 560, of which not all are, 45.0 by 2, 60.1 by 4; 288 behind 12,000 54.9 by 4, 56.7 by 8, behind 30,000 118.7 and 106.3.)
TK_API int tk_attn_kv8_prefill_splits(int tokens, int items, int H, int Hkv, int D, int P, int longest, int sm_count) {
    const int per_tile = 128 / (H / Hkv);
    const int64_t ctas = (int64_t)((tokens + per_tile - 1) / per_tile) * Hkv, launched = (int64_t)items * Hkv;
    auto pays = [&](int n) {
        return n * ctas <= (D == 64 ? 2 : 1) * (int64_t)sm_count && n * launched <= 2048 && longest >= n * 480 &&
               (n == 2 || n * ctas <= sm_count || longest >= n * 1024) &&
               (ctas <= tk_attn_kv8_prefill_clusters(D, P, n, sm_count) || (D == 64 && n == 8 && longest >= 16384));
    };
    int split = 1;
    while (split < 8 && pays(2 * split)) split *= 2;
    return split;
}

// Ways the mma.sync kernel shares the keys of each of `items` tiles out over CTAs, when no sequence holds more than `longest` positions and a query sees at most
// `reach` of them; single: single tokens, whose sequences differ in length. The shares meet in scratch memory and cost a second launch: none up to 512 keys, then 256 keys
// each at least, and as many as keep every CTA resident (three an SM for 32-bit heads of 64 whose pages come by bulk copies, else two: k8_launch's kernels have
// 168 registers there and up to 250 elsewhere). Where two would not be resident, but a quarter of the places is free, three of long contexts all the same (us, 32-bit,
// 8 KV heads of 64 with two query heads each: 2 prompts of up to 301 tokens 15.5 unshared, 24.0 by 2; 60 tokens behind 200 6.4 and 9.0; 256 behind 4,000 59.3, 52.1 by
// 2, 48.7 by 3; 8 single tokens behind 4,000 34.5, 19.6 by 4, 16.8 by 6, 19.7 by 8; 64 behind 1,000 23.6, 26.8 by 2). Keys that each lane looks up take four times as long, so
// there it pays for single tokens from 1,024 keys, and up to an eighth more of them than the places (us, bfloat16, pages of 12: 8 behind 4,000 42.6 by 4, 52.8 by 6, which are
// not all resident; 11 behind 1,200 24.4 by 3, 27.2 by 5; 20 behind 1,200 46.3 unshared, 43.6 by 2, 36.0 by 3; 37 behind 5,000 241 and 218 by 3; 100 tokens behind 1,000
// 44.1 unshared, 50.5 by 2, 60.1 by 3).
TK_API int tk_attn_kv8_splits(int items, int H, int Hkv, int D, int P, int dtype, int longest, int reach, int single, int sm_count) {
    const int64_t ctas = (int64_t)items * Hkv;
    if (ctas <= 0) return 1;
    const int64_t keys = longest < reach ? longest : reach;
    const bool bulk = dtype == TK_F32 && P >= 8 && (P & (P - 1)) == 0;
    const int64_t places = (int64_t)sm_count * (D == 64 && bulk ? 3 : 2);
    int64_t n = places / ctas;
    if (n <= 1 && (4 * ctas <= 3 * places ? keys >= (bulk || !single ? 2048 : 1024) : !bulk && single && keys >= 2048 && 8 * ctas <= 9 * places)) n = 3;
    if (n > (keys + 255) / 256) n = (keys + 255) / 256;
    return (int)(n < 1 || keys <= 512 ? 1 : n > 128 ? 128 : n);
}

// Whether single tokens of this shape take the tcgen05 kernel: 16-bit queries, pages that are a power of two and 8 or more positions.
TK_API int tk_attn_kv8_single_tc(int P, int dtype) { return dtype == TK_BF16 && P >= 8 && (P & (P - 1)) == 0; }

int tk_attn_kv8_tc(const void* q, const void* pool, const float* scales, void* out, const void* args, int D, cudaStream_t stream);
int tk_attn_kv8_tc_status();
TK_API int tk_attn_kv8_tc_splits(int items, int H, int Hkv, int D, int P, int longest, int reach);
int tk_attn_kv8_prefill_tc(const void* q, const void* pool, const float* scales, void* out, const void* args, int D, cudaStream_t stream);
int tk_attn_kv8_prefill_tc_status();

// 0, or 1 if a warp gave up waiting for its keys since the last call. Resets the word.
TK_API int tk_attn_kv8_status() {
    const int found[3] = {k8_take_status(), tk_attn_kv8_tc_status(), tk_attn_kv8_prefill_tc_status()};
    for (int v : found)
        if (v != 0) return v;
    return 0;
}

// tokens: rows of q. q, out: [T, H, D]; pool: [pages, 2, Hkv, P, D] bytes, scales: [pages, 2, Hkv]. item_tok0 / item_ntok: tiles of at most tk_attn_kv8_tokens tokens of one
// sequence at consecutive positions (0 tokens: skipped); item_ntok null: single tokens' rows (negative: skipped; item_tok0 null too: rows 0, 1, ...).
// nsplit 0: chosen here, for sequences of at most `longest` positions (the tcgen05 kernels, which need no scratch). window: see first_seen. scratch: items * H * (tokens a tile, or 1) * nsplit * (D + 4) floats when nsplit > 1. gate: [T, >= H], the per-head output gate.
TK_API int tk_attn_kv8(const void* q, const void* pool, const float* scales, void* out, const int* positions, const int* tok_seq,
                       const int* block_table, int bt_stride, const int* item_tok0, const int* item_ntok, int items, int H, int Hkv, int D,
                       int P, int window, float scale, int nsplit, int longest, int tokens, float* scratch, const void* gate, int64_t ldg, int sink,
                       int dtype, cudaStream_t stream) {
    TK_CHECK_ARG(tk_attn_kv8_supported(H, Hkv, D), "attn_kv8: shape H=%d Hkv=%d D=%d is not taken (heads of 64 or 128, up to %d a KV head)", H,
                 Hkv, D, K8_ROWS);
    const bool meets_in_scratch = item_ntok == nullptr ? !tk_attn_kv8_single_tc(P, dtype) : !tk_attn_kv8_prefill_supported(H, Hkv, D, P, dtype);
    TK_CHECK_ARG(items >= 0 && P > 0 && nsplit >= (meets_in_scratch ? 1 : 0) && (nsplit <= 1 || scratch != nullptr || !meets_in_scratch), "attn_kv8: bad sizes");
    TK_CHECK_ARG(item_ntok == nullptr || item_tok0 != nullptr, "attn_kv8: tiles have first tokens");
    TK_CHECK_ARG((int64_t)items * Hkv * nsplit < 0x7fffffff, "attn_kv8: %d splits of %d items", nsplit, items);
    TK_CHECK_ARG(scale > 0.f, "attn_kv8: the scores' factor is positive");
    TK_CHECK_ARG(dtype == TK_F32 || dtype == TK_BF16, "attn_kv8: unknown dtype %d", dtype);
    TK_CHECK_ARG((uintptr_t)q % 16 == 0 && (uintptr_t)pool % 16 == 0 && (uintptr_t)out % 16 == 0, "attn_kv8: 16-byte aligned tensors");
    if (items == 0) return 0;
    if (nsplit == 0) {
        int device = 0, sms = 0;
        if (cudaGetDevice(&device) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
            tk_set_error("attn_kv8: no device");
            return -1;
        }
        const int64_t reach = window == 0 ? longest : (int64_t)(window < 0 ? -window : window) + (item_ntok != nullptr ? tokens : 0);
        const int most = (int)(reach < longest ? reach : longest);
        nsplit = item_ntok != nullptr ? tk_attn_kv8_prefill_splits(tokens, items, H, Hkv, D, P, most, sms) : tk_attn_kv8_tc_splits(items, H, Hkv, D, P, longest, most);
    }
    int shift = -1;
    if ((P & (P - 1)) == 0)
        for (shift = 0; (1 << shift) < P;) ++shift;
    const int G = H / Hkv;
    K8Args a{positions, tok_seq, block_table, item_tok0, item_ntok, gate, scratch, ldg, bt_stride, items, H, Hkv, P, shift, window, nsplit, sink,
             item_ntok != nullptr ? (K8_ROWS / G) * G : G, scale};
    if (item_ntok != nullptr && tk_attn_kv8_prefill_supported(H, Hkv, D, P, dtype)) {
        TK_CHECK_ARG(nsplit == 1 || nsplit == 2 || nsplit == 4 || nsplit == 8, "attn_kv8: %d shares of a tile's keys (1, 2, 4 or 8)", nsplit);
        return tk_attn_kv8_prefill_tc(q, pool, scales, out, &a, D, stream);
    }
    if (item_ntok == nullptr && tk_attn_kv8_single_tc(P, dtype)) {
        TK_CHECK_ARG(nsplit <= 16, "attn_kv8: %d shares of a token's keys (at most 16)", nsplit);
        return tk_attn_kv8_tc(q, pool, scales, out, &a, D, stream);
    }
    const cudaError_t e = dtype == TK_F32 ? k8_dispatch<float>(q, pool, scales, out, a, D, stream)
                                          : k8_dispatch<__nv_bfloat16>(q, pool, scales, out, a, D, stream);
    if (e != cudaSuccess) {
        tk_set_error("attn_kv8: launch failed: %s", cudaGetErrorString(e));
        cudaGetLastError();
        return -2;
    }
    return 0;
}
