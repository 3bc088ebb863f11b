// Single tokens' attention over the 8-bit cache (kv8.cuh) on the fifth-generation tensor cores, for bfloat16: the cache's bytes are the products'
// operands as they lie in memory, no instruction ever touches them.
//
//   S^T = K q^T      tcgen05.mma kind::f8f6f4, M = 128 keys, a column a query head: a thread owns a key and reads its scores
//   O^T += V^T P^T   M = D, the same columns: V's [key][d] is the M-major operand as it lands
//
// What is not 8-bit is a sum of 8-bit terms, a column each, added up when they are read: e4m3 has four significant bits, so q (after
// division by a power of two that brings its row's largest to [128, 256)) is two terms, exactly for elements down to 2^-12 of the row's
// largest and to 2^-18 of that below. A weight is rounded to float16 and is four terms, each the e4m3 of what those before it leave times 2^5: of a weight of at
// most 2^8 a term leaves at most 2^3, so 2^8 again goes into the next one, and the last one's smallest step, 2^-9 2^-15, is float16's: the four are the
// float16 weight exactly. The weights' reference maximum follows lazily (raised when a row exceeds it by 2^2) and weights are lifted by 2^6 (at most 256, of
// 448): a weight is off by at most 2^-11 of itself or, where that is more, by 2^-31 of the row's largest (half of float16's smallest step against 2^6), as in the form for portions. (Terms
// of one size lose the many small weights beside a large one: with factors of 1, 1, 2^8 and 2^8, 3,000 keys that have a thousandth of a row's weight between
// them, beside one that has the rest and a value of 0, came out 6 % off; now 0.2 %, the output's own rounding.) A value block's scale is in the
// exponent, as in attention_kv8.cu. Columns cost nothing here: a product's time is that of reading its 128 x 32 or D x 32 bytes of the first operand
// from shared memory. (With the heads as the M side of the second product, 32 rows of 128, and the terms one after the other, the products
// alone took 575 cycles a tile of 128 keys, and 8 tokens behind 32,000 positions 71 us.)
//
// A CTA takes the query heads of one KV head of one token and a share of its keys, in tiles of 128 (up to 16 CTAs, a cluster, share them and join
// their shares through each other's shared memory):
//   warps 4, 5  bring K and V by TMA, a page (or 128 positions of one) a load, up to three tiles ahead
//   warp 6      issues the products
//   warps 0-3   thread = key: masks, reference maximum (one vote of the four warps a tile), weights, their terms into shared memory
//               ([term and head][key], the second product's other operand); positions that are not to be seen have their value rows zeroed there
//
// Measured (one B200, pages of 16): one token behind 2,048 positions 7.7 us and 64 behind up to 3,000 32.3 (32 heads over 8 of 64; 9.9 and 69 on mma.sync), 8
// behind 32,000 45.2 (16 heads over 8: 5.7 TB/s; 109), 16 behind a window of 1,024 9.2 (16 heads over 4 of 128; 16.3), 64 behind up to 3,000 of one KV head of 128 with
// 16 query heads 24.7 (floor 5.8: one CTA an SM, 128 registers a thread and what they spill). HBM bounds long contexts (7 TB/s while all of
// the 64's CTAs work, 2,240 cycles a tile; then the longest ones end alone); below
// some 8 MB of cache the launch, the chain of a tile's products and weights and the shares' joining are what there is. Tried and slower or no faster: two or four to six tiles
// ahead, four copying warps or one (65-100 cycles a load, one after the other within a warp), the shares joined through global memory,
// CTAs that stay and take one unshared token and KV head after the other, their loads and q running ahead (512 behind up to 300: 59 became 49, but 128 behind up
// to 4,000 75 became 81 and 128 behind up to 500 18.3 became 20.5).
//
// Masking and sums are those of attention_kv8.cu; every wait is bounded (about a second), the kernel then frees its tensor memory and
// returns, and tk_attn_kv8_status() says so.
#include <cooperative_groups.h>
#include <math.h>

#include "kv8_attn.cuh"
#include "kv8_tc.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int K8T_KEYS = 128;
constexpr int K8T_COPIERS = 2;                             // warps that bring keys, and values
constexpr int K8T_MMA_WARP = 4 + K8T_COPIERS, K8T_THREADS = (K8T_MMA_WARP + 1) * 32;
constexpr int K8T_PTERMS = 4;
constexpr float K8T_LAZY = 2.0f, K8T_LIFT = 6.0f, K8T_FINER = 32.0f;       // (a term's factor over the one before)

// eight columns of this thread's lane; the loads of several calls are waited for together
__device__ __forceinline__ void tmem_ld8_start(uint32_t addr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr));
}
template <int N>
__device__ __forceinline__ void tmem_ld_n(uint32_t addr, float (&v)[N]) {
    uint32_t r[N];
#pragma unroll
    for (int i = 0; i < N; i += 8) tmem_ld8_start(addr + i, r + i);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __uint_as_float(r[i]);
}
template <int N>
__device__ __forceinline__ void tmem_st_n(uint32_t addr, const float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 8)
        asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr + i), "f"(v[i]), "f"(v[i + 1]),
                     "f"(v[i + 2]), "f"(v[i + 3]), "f"(v[i + 4]), "f"(v[i + 5]), "f"(v[i + 6]), "f"(v[i + 7])
                     : "memory");
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// whether `mine` holds for any of the 128 threads of the weights' warps
__device__ __forceinline__ bool any_of_128(bool mine) {
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %1, 0;\n\t"
        "bar.red.or.pred q, 1, 128, p;\n\t"
        "selp.b32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"((uint32_t)mine)
        : "memory");
    return any != 0;
}
__device__ __forceinline__ void sync_128() { asm volatile("bar.sync 2, 128;" ::: "memory"); }

// tiles of keys and values in shared memory (they leave room for four CTAs an SM where a KV head of 64 has up to four query heads, else for two, and for one of
// heads of 128 with more than eight)
constexpr int K8T_STAGES = 3;

template <int D, int NR, int KG>
struct K8tSmem {
    static constexpr int GROUPS = K8T_KEYS / KG;                                   // that share scales: 16 keys, or 8 where a page has no more
    static constexpr int STAGES = K8T_STAGES;
    static constexpr int S_COLS = 2 * NR < 16 ? 16 : 2 * NR;                       // scores' columns: term, head
    static constexpr int O_COLS = 4 * NR < 16 ? 16 : 4 * NR;                       // outputs' columns: term, head
    static constexpr int P_BYTES = O_COLS * K8T_KEYS;                              // [term, head / 16][key][16]
    static constexpr int P = 0;                                                    // two of them
    static constexpr int Q = 2 * P_BYTES;                                          // [term, head][d]
    static constexpr int KV = Q + (S_COLS * D < 1024 ? 1024 : S_COLS * D);         // stages: K tile, V tile
    static constexpr int STAGE = 2 * K8T_KEYS * D;
    static constexpr int BARS = KV + STAGES * STAGE;
    static constexpr int SCALES = BARS + (2 * STAGES + 6) * 8 + 16;                // of a tile's groups of keys: (key's, value's)
    static constexpr int MISC = SCALES + STAGES * GROUPS * 8;
    static constexpr int BYTES = MISC + (16 * 4 + 4 * 16 * 4);                     // row factors, warps' maxima or sums
    static constexpr int BOUND = D == 64 && NR <= 4 ? 4 : 2;                       // CTAs an SM that registers are kept for
    static constexpr int FIT = 233472 / (BYTES + 1024);                            // and that its shared memory holds (1 KB of each CTA's is the system's)
    static constexpr int PER_SM = FIT < BOUND ? FIT : BOUND;
    static_assert(SCALES % 8 == 0 && MISC % 8 == 0, "pairs");
    // a share of the keys, for the CTAs that join theirs: [head][d] and the heads' maxima and sums, where the first tiles were
    static_assert(NR * (D + 2) * 4 <= STAGES * STAGE, "a share");
    static_assert(Q % 1024 == 0 && KV % 1024 == 0, "swizzled tiles");
};

// The weights' terms as the second product's other operand: 16 of them (bytes) a key, keys one after the other, further ones K8T_KEYS keys on. MN-major
// without swizzle: eight keys are 128 bytes, the next eight follow.
__device__ __forceinline__ uint64_t desc_keys16(uint32_t at) {
    return (uint64_t)((at & 0x3FFFF) >> 4) | (uint64_t)(128 >> 4) << 16 | (uint64_t)(16 * K8T_KEYS >> 4) << 32 | (uint64_t)1 << 46;
}

// D: head size; NR: query heads a KV head has, rounded up to 2, 4, 8 or 16
template <int D, int NR, int KG>
__global__ void __launch_bounds__(K8T_THREADS, K8tSmem<D, NR, KG>::BOUND)
attn_kv8_tc_kernel(const __nv_bfloat16* q, const float* scales, __nv_bfloat16* out, const __grid_constant__ CUtensorMap map, const K8Args a) {
    using L = K8tSmem<D, NR, KG>;
    constexpr int GROUPS = L::GROUPS, AHEAD = 32 / GROUPS;                         // tiles whose pages and scales a copying warp's lanes know
    constexpr int STAGES = L::STAGES;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 128) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map)) : "memory");
    const uint32_t base = smem_u32(smem_raw);
    const uint32_t bars = base + L::BARS;
    auto kv_full = [&](int s) { return bars + (uint32_t)s * 8; };
    auto kv_empty = [&](int s) { return bars + (uint32_t)(STAGES + s) * 8; };
    auto s_full = [&](int b) { return bars + (uint32_t)(2 * STAGES + b) * 8; };
    auto p_full = [&](int b) { return bars + (uint32_t)(2 * STAGES + 2 + b) * 8; };
    auto pv_full = [&](int b) { return bars + (uint32_t)(2 * STAGES + 4 + b) * 8; };
    const uint32_t tmem_slot = bars + (2 * STAGES + 6) * 8;
    float* row_factor = reinterpret_cast<float*>(smem_raw + L::MISC);             // [16]
    float* by_warp = row_factor + 16;                                             // [4][16]
    float* share = reinterpret_cast<float*>(smem_raw + L::KV);                    // [head][d]
    float2* share_ml = reinterpret_cast<float2*>(share + NR * D);
    constexpr uint32_t COLS = 128;                                                // tensor memory: two of up to 32 columns for scores, up to 64 for outputs

    if (tid == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(kv_full(i), K8T_COPIERS);
            mbar_init(kv_empty(i), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full(i), 1);
            mbar_init(p_full(i), 4);
            mbar_init(pv_full(i), 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == K8T_MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_wait();
    const int split = blockIdx.x % a.nsplit, kvh = (blockIdx.x / a.nsplit) % a.Hkv, item = blockIdx.x / (a.nsplit * a.Hkv);
    const int tok = a.item_tok0 != nullptr ? a.item_tok0[item] : item;
    const int G = a.H / a.Hkv, P = a.P;
    const int* bt = tok >= 0 ? a.block_table + (size_t)a.tok_seq[tok] * a.bt_stride : nullptr;
    const int pos = tok >= 0 ? a.positions[tok] : -1;             // (a padded entry of a recorded step has no tiles)
    const int lo = first_seen(pos, a.window), t_lo = lo / K8T_KEYS;
    const int all_tiles = pos >= lo ? pos / K8T_KEYS - t_lo + 1 : 0;
    const int t_begin = t_lo + (int)((int64_t)all_tiles * split / a.nsplit);
    const int n_tiles = t_lo + (int)((int64_t)all_tiles * (split + 1) / a.nsplit) - t_begin;

    // ---- q's terms: 8 lanes a row ----
    if (warp < 4) {
        const int r = tid >> 3, c0 = (tid & 7) * (D / 8);
        float x[D / 8], most = 0.f;
#pragma unroll
        for (int e = 0; e < D / 8; ++e) x[e] = 0.f;
        if (r < G && tok >= 0) {
            const __nv_bfloat16* src = q + ((size_t)tok * a.H + kvh * G + r) * D + c0;
#pragma unroll
            for (int e = 0; e < D / 8; e += 4) {
                const float4 v = Quad<__nv_bfloat16>::load(src + e);
                x[e] = v.x, x[e + 1] = v.y, x[e + 2] = v.z, x[e + 3] = v.w;
            }
        }
        bool fine = true;
#pragma unroll
        for (int e = 0; e < D / 8; ++e) {
            most = fmaxf(most, fabsf(x[e]));
            fine = fine && fabsf(x[e]) <= 3.4e38f;
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        fine = (__ballot_sync(0xffffffffu, !fine) >> (lane & 24) & 255u) == 0;
        int e2 = (__float_as_int(most) >> 23) - 127;
        e2 = most == 0.f ? 7 : min(max(e2, -100), 127);
        const float up = exp2i(7 - e2);
        // (a row that is not finite has no scores that are)
        if ((tid & 7) == 0) row_factor[r] = fine ? a.scale * K8_LOG2E * exp2i(e2 - 7) : NAN;
#pragma unroll
        for (int e = 0; e < D / 8; e += 8) {
            uint32_t t1[2], t2[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                t1[h] = t2[h] = 0;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float u = x[e + 4 * h + 2 * k] * up, v = x[e + 4 * h + 2 * k + 1] * up;
                    const uint16_t first = to_e4m3x2(u, v);
                    const float2 back = half2_floats(e4m3x2_to_half2(first));
                    t1[h] |= (uint32_t)first << (16 * k);
                    t2[h] |= (uint32_t)to_e4m3x2(u - back.x, v - back.y) << (16 * k);
                }
            }
            if (r < NR) {
                unsigned char* at = smem_raw + L::Q + ((c0 + e) & 8);
                *reinterpret_cast<uint2*>(at + swizzled<D>(r, (c0 + e) >> 4)) = make_uint2(t1[0], t1[1]);
                *reinterpret_cast<uint2*>(at + swizzled<D>(NR + r, (c0 + e) >> 4)) = make_uint2(t2[0], t2[1]);
            }
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem_raw + (tmem_slot - base));
    const uint32_t tmem_o = tmem + 64;

    if (warp >= 4 && warp < K8T_MMA_WARP) {
        // ---- K and V: lane i knows the page and the scales of KG positions of one of four tiles (KG = 8: two), and brings the page (or 128 positions of it)
        // if they are its first of the tile: keys one warp, values the other. (A warp's loads go out one after the other, 65 to 100 cycles
        // each however they are issued: one warp for a tile's 16 set the pace at 1,450 cycles a tile.) The pages of four (two) tiles are asked for
        // eight (four) tiles ahead, their scales half as many: no trip is waited for. ----
        const int which = warp - 4, per = 1 << min(a.p_shift, 7);
        const int group = lane & (GROUPS - 1), at_row = (group * KG) & (per - 1);        // (of a page, as far as a tile reaches)
        bool ok = true;
        auto page_of = [&](int block) {
            const int it = block * AHEAD + lane / GROUPS, j = (t_begin + it) * K8T_KEYS + group * KG - at_row;
            return it < n_tiles && j <= pos && j + per > lo ? TK_PAGE(TK_K_KV8_ATTN, bt[j >> a.p_shift]) : -1;
        };
        auto scales_of = [&](int pg) {
            const float* from = scales + (size_t)max(pg, 0) * (2 * a.Hkv) + kvh;
            return pg >= 0 ? make_float2(from[0], from[a.Hkv]) : make_float2(1.f, 1.f);
        };
        int page = -1, page_next = page_of(0), page_after = page_of(1);
        float2 scale = make_float2(1.f, 1.f), scale_next = scales_of(page_next);
        float2* sc = reinterpret_cast<float2*>(smem_raw + L::SCALES);
        for (int it = 0; it < n_tiles; ++it) {
            const int s = it % STAGES;
            if (it % AHEAD == 0) {
                page = page_next;
                scale = scale_next;
                page_next = page_after;
                scale_next = scales_of(page_next);
                page_after = page_of(it / AHEAD + 2);
            }
            if (it >= STAGES) ok = k8_wait(kv_empty(s), (uint32_t)((it / STAGES - 1) & 1));
            if (!__all_sync(0xffffffffu, ok)) break;
            const bool ours = lane / GROUPS == it % AHEAD, mine = ours && page >= 0 && at_row == 0;
            const int loads = __popc(__ballot_sync(0xffffffffu, mine));
            if (mine) {
                const int row = ((page * 2 + which) * a.Hkv + kvh) * P + (((t_begin + it) * K8T_KEYS + group * KG) & (P - 1));
                tma_load_2d(base + L::KV + (uint32_t)s * L::STAGE + (uint32_t)((which * K8T_KEYS + group * KG) * D), &map, 0, row, kv_full(s));
            }
            if (which == 0 && ours) sc[s * GROUPS + group] = scale;
            __syncwarp();
            // (the phase ends with this arrival and the bytes, whichever come last)
            if (lane == 0) mbar_expect_tx(kv_full(s), (uint32_t)(loads * per * D));
        }
    } else if (warp == K8T_MMA_WARP) {
        // ---- the products ----
        constexpr uint32_t id_s = idesc8(K8T_KEYS, L::S_COLS, false), id_o = idesc8(D, L::O_COLS, true) | 1u << 16;
        const uint64_t qd = desc8<D>(base + L::Q);
        auto wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, k8_wait(bar, parity)) != 0; };
        bool ok = true;
        auto scores = [&](int j) {
            const int s = j % STAGES;
            ok = ok && wait(kv_full(s), (uint32_t)((j / STAGES) & 1));
            if (!ok) return;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint64_t kd = desc8<D>(base + L::KV + (uint32_t)s * L::STAGE);
            if (elect_lane()) {
#pragma unroll
                for (int k = 0; k < D / 32; ++k) umma_f8(tmem + (uint32_t)(j & 1) * 32, kd + 2 * k, qd + 2 * k, id_s, k > 0 ? 1u : 0u);
                umma_commit(s_full(j & 1));
            }
            __syncwarp();
        };
        if (n_tiles > 0) scores(0);
        for (int j = 0; j < n_tiles && ok; ++j) {
            // (the scores of tile j - 1 have been read: its weights were waited for)
            if (j + 1 < n_tiles) scores(j + 1);
            if (!ok) break;
            const int s = j % STAGES, b = j & 1;
            ok = wait(p_full(b), (uint32_t)((j >> 1) & 1));
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint64_t vd = desc8<D>(base + L::KV + (uint32_t)s * L::STAGE + K8T_KEYS * D);
            const uint64_t pd = desc_keys16(base + L::P + b * L::P_BYTES);
            if (elect_lane()) {
#pragma unroll
                for (int k = 0; k < K8T_KEYS / 32; ++k)
                    umma_f8(tmem_o, vd + (uint64_t)(k * 32 * D / 16), pd + 32 * k, id_o, j + k > 0 ? 1u : 0u);
                umma_commit(pv_full(b));
                umma_commit(kv_empty(s));
            }
            __syncwarp();
        }
    } else {
        // ---- the weights ----
        float c[NR], m[NR], l[NR], up[NR], limit[NR];         // (of a row without a maximum yet: nothing above is small enough)
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            c[r] = row_factor[r];
            m[r] = limit[r] = -INFINITY;
            l[r] = up[r] = 0.f;
        }
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        bool ok = true;
        for (int it = 0; it < n_tiles; ++it) {
            const int b = it & 1, turn = it >> 1, j = (t_begin + it) * K8T_KEYS + tid;
            const bool seen = j >= lo && j <= pos;
            // (after a failed wait the loop runs to its end without waiting: every thread meets every barrier)
            if (ok) ok = k8_wait(s_full(b), (uint32_t)(turn & 1)) && k8_wait(kv_full(it % STAGES), (uint32_t)((it / STAGES) & 1));
            ok = __all_sync(0xffffffffu, ok);
            const float2 sc = reinterpret_cast<const float2*>(smem_raw + L::SCALES)[(it % STAGES) * GROUPS + tid / KG];
            const int bits = __float_as_int(sc.y);
            const float ev = __int_as_float(0x4b000000 | (bits >> 23)) - 8388735.0f, inv_v = __int_as_float((254 << 23) - bits);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            float x[NR], y[NR];
            {
                constexpr int N = 2 * NR < 8 ? 8 : 2 * NR;
                float sum[N];
                tmem_ld_n<N>(tmem + lanes + (uint32_t)b * 32, sum);
#pragma unroll
                for (int r = 0; r < NR; ++r) x[r] = sum[r] + sum[NR + r];
            }
            // the weights' logarithms
            auto weigh = [&](int r) { y[r] = seen ? fmaf(x[r], sc.x * c[r], ev + up[r]) : -INFINITY; };
            bool above = false;
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                weigh(r);
                above = above || y[r] > limit[r];
            }
            if (any_of_128(above)) {
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    const float top = warp_max(y[r] - up[r]);
                    if (lane == 0) by_warp[warp * 16 + r] = top;
                }
                sync_128();
                float f[NR];
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    const float top = fmaxf(fmaxf(by_warp[r], by_warp[16 + r]), fmaxf(by_warp[32 + r], by_warp[48 + r]));
                    const float m_new = fmaxf(m[r], top);
                    f[r] = m_new == -INFINITY ? 1.f : k8_exp2(m[r] - m_new);
                    m[r] = m_new;
                    l[r] *= f[r];
                    up[r] = m_new == -INFINITY ? 0.f : K8T_LIFT - m_new;
                    limit[r] = m_new == -INFINITY ? -INFINITY : K8T_LIFT + K8T_LAZY;
                    weigh(r);
                }
                if (it > 0) {
                    // what this warp's lanes have accumulated (no product is under way once the last tile's is done)
                    if (ok) ok = k8_wait(pv_full(b ^ 1), (uint32_t)(((it - 1) >> 1) & 1));
                    ok = __all_sync(0xffffffffu, ok);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    float v[L::O_COLS];
                    tmem_ld_n<L::O_COLS>(tmem_o + lanes, v);
#pragma unroll
                    for (int i = 0; i < K8T_PTERMS * NR; ++i) v[i] *= f[i % NR];
                    tmem_st_n<L::O_COLS>(tmem_o + lanes, v);
                }
                sync_128();                              // (the warps' maxima are read; they are written again at the next raise)
            }
            // the terms of tile it - 2 have been read
            if (ok && it >= 2) ok = k8_wait(pv_full(b), (uint32_t)((turn - 1) & 1));
            constexpr int WORDS = L::O_COLS / 4;
            uint32_t terms[WORDS];
#pragma unroll
            for (int i = 0; i < WORDS; ++i) terms[i] = 0;
#pragma unroll
            for (int r = 0; r < NR; r += 2) {
                float w[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    w[h] = k8_exp2(y[r + h]);
                    l[r + h] = fmaf(w[h], inv_v, l[r + h]);
                }
                __half2 left = __floats2half2_rn(w[0], w[1]);        // (what a term leaves of a float16 is one, and so is 2^5 times that)
#pragma unroll
                for (int t = 0; t < K8T_PTERMS; ++t) {
                    uint16_t two;
                    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(two) : "r"(*reinterpret_cast<const uint32_t*>(&left)));
                    terms[(t * NR + r) / 4] |= (uint32_t)two << (8 * ((t * NR + r) & 2));
                    const uint32_t back = e4m3x2_to_half2(two);
                    left = __hmul2(__hsub2(left, *reinterpret_cast<const __half2*>(&back)), __float2half2_rn(K8T_FINER));
                }
            }
            unsigned char* p = smem_raw + L::P + b * L::P_BYTES + tid * 16;
#pragma unroll
            for (int i = 0; i < WORDS; i += 4) *reinterpret_cast<uint4*>(p + i * 4 * K8T_KEYS) = make_uint4(terms[i], terms[i + 1], terms[i + 2], terms[i + 3]);
            if (!seen) {
                // whatever the cache (or an earlier tile) has left there
                uint4* row = reinterpret_cast<uint4*>(smem_raw + L::KV + (it % STAGES) * L::STAGE + K8T_KEYS * D + tid * D);
#pragma unroll
                for (int e = 0; e < D / 16; ++e) row[e] = make_uint4(0u, 0u, 0u, 0u);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full(b));
        }
        // ---- the sums over keys, then a column of the head a lane (D = 64: the products leave 16 in each warp's lanes) ----
        sync_128();
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const float sum = warp_sum(l[r]);
            if (lane == 0) by_warp[warp * 16 + r] = sum;
        }
        if (ok && n_tiles > 0) ok = k8_wait(pv_full((n_tiles - 1) & 1), (uint32_t)(((n_tiles - 1) >> 1) & 1));
        ok = __all_sync(0xffffffffu, ok);
        sync_128();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        float v[L::O_COLS];
#pragma unroll
        for (int i = 0; i < L::O_COLS; ++i) v[i] = 0.f;
        if (n_tiles > 0) tmem_ld_n<L::O_COLS>(tmem_o + lanes, v);
        constexpr int PER = D / 4;
        const int d = warp * PER + lane;
        if (tok >= 0 && lane < PER) {
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                if (r >= G) continue;
                float o = v[3 * NR + r];
#pragma unroll
                for (int t = K8T_PTERMS - 2; t >= 0; --t) o = fmaf(o, 1.f / K8T_FINER, v[t * NR + r]);
                float l_r = (by_warp[r] + by_warp[16 + r]) + (by_warp[32 + r] + by_warp[48 + r]);
                const int head = kvh * G + r;
                if (a.nsplit == 1) {
                    if (a.sink && m[r] > -INFINITY) l_r += k8_exp2(K8T_LIFT - m[r]);
                    o = l_r == 0.f ? 0.f : o / l_r;
                    out[((size_t)tok * a.H + head) * D + d] = __float2bfloat16_rn(k8_apply<__nv_bfloat16>(o, a, k8_gate<__nv_bfloat16>(a, tok, head)));
                } else {
                    share[r * D + d] = o;
                    if (d == 0) share_ml[r] = make_float2(m[r], l_r);
                }
            }
        }
    }
    if (a.nsplit > 1) {
        // each CTA forms an equal part of the outputs from all shares, through the cluster's shared memory
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        if (tok >= 0) {
            for (int i = split * K8T_THREADS + tid; i < G * D; i += a.nsplit * K8T_THREADS) {
                const int r = i / D, d = i % D, head = kvh * G + r;
                float m_all = -INFINITY, l_all = 0.f, o = 0.f;
                for (int sp = 0; sp < a.nsplit; ++sp) m_all = fmaxf(m_all, cluster.map_shared_rank(share_ml, sp)[r].x);
#pragma unroll 4
                for (int sp = 0; sp < a.nsplit; ++sp) {
                    const float2 ml = cluster.map_shared_rank(share_ml, sp)[r];
                    const float f = k8_factor(ml.x, ml.y, m_all);
                    l_all = fmaf(ml.y, f, l_all);
                    o = fmaf(cluster.map_shared_rank(share, sp)[r * D + d], f, o);
                }
                if (a.sink && m_all > -INFINITY) l_all += k8_exp2(K8T_LIFT - m_all);
                o = l_all == 0.f ? 0.f : o / l_all;
                out[((size_t)tok * a.H + head) * D + d] = __float2bfloat16_rn(k8_apply<__nv_bfloat16>(o, a, k8_gate<__nv_bfloat16>(a, tok, head)));
            }
        }
        cluster.sync();                                  // nobody leaves while its share is read
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == K8T_MMA_WARP) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS) : "memory");
    }
}

template <int D, int NR, int KG>
cudaError_t k8t_config(cudaLaunchConfig_t& cfg, cudaLaunchAttribute* attr, int64_t ctas, int nsplit, cudaStream_t stream) {
    constexpr int smem = K8tSmem<D, NR, KG>::BYTES;
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = k8_allow(attn_kv8_tc_kernel<D, NR, KG>, smem, true, done);
    if (e != cudaSuccess) return e;
    cfg = {};
    cfg.gridDim = dim3((unsigned)(ctas * nsplit));
    cfg.blockDim = dim3(K8T_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = k8_attributes(attr, nsplit);
    return cudaSuccess;
}

struct K8tLaunch {
    const void* q;
    const float* scales;
    void* out;
    const CUtensorMap& map;
    const K8Args& a;
    cudaStream_t stream;

    template <int D, int NR, int KG>
    cudaError_t run() const {
        cudaLaunchConfig_t cfg;
        cudaLaunchAttribute attr[2];
        const cudaError_t e = k8t_config<D, NR, KG>(cfg, attr, (int64_t)a.items * a.Hkv, a.nsplit, stream);
        if (e != cudaSuccess) return e;
        return cudaLaunchKernelEx(&cfg, attn_kv8_tc_kernel<D, NR, KG>, (const __nv_bfloat16*)q, scales, (__nv_bfloat16*)out, map, a);
    }
};

// How many clusters of `n` CTAs the device holds at once, asked for once. Where an SM holds one CTA, clusters lie in whole parts of the device, 15 of 8 or 33 of 4, not 148
// SMs' worth, and the occupancy calculator knows.
struct K8tPlaces {
    int n;
    int* clusters;

    template <int D, int NR, int KG>
    cudaError_t run() const {
        static std::atomic<int> known[16][17];
        int device = 0, sms = 0;
        cudaError_t e = cudaGetDevice(&device);
        if (e != cudaSuccess) return e;
        if (device < 16 && (*clusters = known[device][n].load(std::memory_order_relaxed)) > 0) return e;
        if constexpr (K8tSmem<D, NR, KG>::PER_SM > 1) {
            e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
            *clusters = k8_clusters(K8tSmem<D, NR, KG>::PER_SM, sms, n);
        } else {
            cudaLaunchConfig_t cfg;
            cudaLaunchAttribute attr[2];
            e = k8t_config<D, NR, KG>(cfg, attr, 1, n, nullptr);
            if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(clusters, attn_kv8_tc_kernel<D, NR, KG>, &cfg);
        }
        if (e == cudaSuccess && device < 16) known[device][n].store(*clusters, std::memory_order_relaxed);
        return e;
    }
};

template <int D, int KG, typename F>
cudaError_t k8t_rows(int G, const F& f) {
    return G <= 2 ? f.template run<D, 2, KG>() : G <= 4 ? f.template run<D, 4, KG>() : G <= 8 ? f.template run<D, 8, KG>() : f.template run<D, 16, KG>();
}

// f.run<D, NR, KG>() for the kernel of a layer
template <typename F>
cudaError_t k8t_pick(int G, int D, int P, const F& f) {
    return P == 8 ? (D == 64 ? k8t_rows<64, 8>(G, f) : k8t_rows<128, 8>(G, f)) : (D == 64 ? k8t_rows<64, 16>(G, f) : k8t_rows<128, 16>(G, f));
}

}  // namespace

// How many CTAs share each of `items` tokens' keys, when no sequence holds more than `longest` positions and a query sees at most `reach` of them: as many as keep
// every CTA resident (one CTA more and the launch runs in two waves), in clusters of at most eight with two tiles of 128 keys each, or of 16 with four (us by
// shares, 8 KV heads of 64: a token behind 2,048 positions 14.9 unshared, 8.7 by 4, 7.6 by 8, 8.5 by 16; behind 30,000 136, 40, 24.7, 20.8; 8 tokens behind 32,000 49.0
// by 6, 45.7 by 8, 61.7 by 10; 16 behind 4,000 15.3 by 4, 20.3 by 5; 64 behind up to 3,000 33.1 unshared, 38.9 by 2; one KV head: 30 tokens behind 9,000 14.7 by 8, 20.9 by 16, 72 behind
// 4,000 13.5 by 7, 18.4 by 8. One KV head of 128 with 16 query heads, whose CTA fills
// an SM: 18 tokens behind 30,000 51.2 by 6, 76.8 by 8, 82.2 by 16; 64 behind 3,000 33.0 unshared, 24.7 by 2, 33.6 by 4).
TK_API int tk_attn_kv8_tc_splits(int items, int H, int Hkv, int D, int P, int longest, int reach) {
    const int64_t ctas = (int64_t)items * Hkv, keys = longest < reach ? longest : reach, tiles = (keys + 127) / 128 + (reach < longest ? 1 : 0);
    auto resident = [&](int n) {
        int clusters = 0;
        if (k8t_pick(H / Hkv, D, P, K8tPlaces{n, &clusters}) != cudaSuccess) {
            cudaGetLastError();
            return false;
        }
        return ctas <= clusters;
    };
    if (tiles >= 64 && resident(16)) return 16;
    int n = (int)(tiles >= 16 ? 8 : (tiles + 1) / 2);
    if (n < 4) n = tiles < 4 ? (int)tiles : 4;
    while (n > 1 && !resident(n)) --n;
    return n < 1 ? 1 : n;
}

// The arguments of tk_attn_kv8 for single tokens (attention_kv8.cu checks them): bfloat16, pages that are a power of two and 8 or more.
int tk_attn_kv8_tc(const void* q, const void* pool, const float* scales, void* out, const void* args, int D, cudaStream_t stream) {
    const K8Args& a = *static_cast<const K8Args*>(args);
    CUtensorMap map = {};
    TK_CHECK_ARG(k8_map(&map, pool, D, a.P < K8T_KEYS ? a.P : K8T_KEYS), "attn_kv8: cuTensorMapEncodeTiled failed");
    const cudaError_t e = k8t_pick(a.H / a.Hkv, D, a.P, K8tLaunch{q, scales, out, map, a, stream});
    if (e != cudaSuccess) {
        tk_set_error("attn_kv8: launch failed: %s", cudaGetErrorString(e));
        cudaGetLastError();
        return -2;
    }
    return 0;
}

int tk_attn_kv8_tc_status() { return k8_take_status(); }
