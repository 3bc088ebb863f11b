// Prompt portions' attention over the 8-bit cache (kv8.cuh) on the fifth-generation tensor cores, for bfloat16.
//
//   S  = q K^T     tcgen05.mma kind::f8f6f4, M = 128 rows, N = 64 keys: K's bytes as they land, q as two e4m3 terms (attention_kv8_tc.cu)
//                  multiplied one after the other into the same accumulator
//   O += P V       kind::f16, P float16 in tensor memory where S was, V's bytes turned into float16 on the way (e4m3 is exact in it)
//
// A CTA takes up to 128 rows: 128 / G tokens (rounded down) of one sequence with the G query heads that share one KV head (row = token * G + head), and walks the keys
// in tiles of 64, this step's own included. Warps coupled by mbarriers only:
//
//   warp 0      brings K and V by TMA, a page (or 64 positions of one) a load, up to five tiles ahead, and the tiles' scales
//   warps 1, 2  turn V into float16 tiles; positions that nobody may read become zeros there, whatever the cache holds
//   warp 3      one lane issues the products: S_j, and P_j V_j into one of two outputs that live in tensor memory for the whole walk
//   warps 4-11  bring q's terms, then are two groups of 128 threads that take the key tiles in turn, each with scores, weights and an output of
//               its own, so that one's chain runs under the other's; thread r owns row r of its group's tiles
//
// A tile's 64 keys lie in four groups of 16 (or eight of 8, for pages of 8) with one scale for keys and one for values each. With c = scale log2(e)
// and x_j = s_K c (q . kb_j) + log2(s_V), the weight of a value's bytes is 2^(x_j - m + 7) and the softmax's sum adds those weights over s_V, a group at a
// time: a score costs one multiply-add and one exponential, as without scales. m follows the running maximum lazily (raised when a row exceeds it
// by 8: weights stay below 2^15 of float16's 65,504, and reach down to 2^-31 of the row's largest); only then is the output read, scaled and
// written back. At the end the first group merges both outputs, and up to eight CTAs (a cluster) that share a tile's keys merge theirs.
//
// Measured (32 heads over 8 of 64, one B200): a prompt of 2,048 tokens 41.6 us (the mma.sync kernel 124), 512 tokens behind 8,192 positions 71.1 (205), 512 behind
// 30,000 224; heads of 128, 16 over 4: 1,000 tokens 18.4 (52), 256 behind 4,000 28.9 (75). Bound by each group's chain (scores, maximum, exponentials, weights
// back, products), four groups an SM as tensor memory allows: exponentials' unit 49 % busy, ALU 42 %, tensor cores 24 %, 2.1 of 4 instructions a cycle.
// Tried and slower: a warp a group for the products (71.1 became 79.6, 83.1 when those warps brought the tiles too: one warp keeps the groups out of step),
// weights through shared memory so that the next scores need not wait for their product (86.8), the first half of a row's scores read twice instead of kept
// (71.2, heads of 128 3 % slower), sums and products one by one instead of in pairs (74.0).
//
// Masking, sums, gate, sink and bounded waits are those of the other kernels of this cache; tk_attn_kv8_status() says where a wait gave up.
#include <cooperative_groups.h>
#include <math.h>

#include <type_traits>

#include "kv8_attn.cuh"
#include "kv8_tc.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int KP_ROWS = 128, KP_KEYS = 64;
constexpr int KP_THREADS = 384;
constexpr int KP_STAGES = 5;
constexpr int KP_SPLIT_TILES = 8;                          // key tiles a CTA should have before a tile's keys are shared out
constexpr float KP_LAZY = 8.0f, KP_LIFT = 7.0f;

// shared memory of a CTA: two fit an SM for heads of 64, one for heads of 128. KG: keys that share scales, 16, or 8 where a page has no more.
template <int D, int KG>
struct KpSmem {
    static constexpr int GROUPS = KP_KEYS / KG;
    static constexpr int Q_BYTES = KP_ROWS * D;            // of a term
    static constexpr int RAW = KP_KEYS * D;                // keys' or values' bytes of a tile
    static constexpr int HALF = KP_KEYS * 128;             // float16 values of a tile, 64 columns
    static constexpr int V16 = HALF * (D / 64);
    static constexpr int Q = 0, K = 2 * Q_BYTES, V = K + KP_STAGES * RAW, H = V + KP_STAGES * RAW;
    static constexpr int SCALES = H + KP_STAGES * V16;     // [stage][group] (key's, value's)
    static constexpr int FACTOR = SCALES + KP_STAGES * GROUPS * 8;
    static constexpr int BARS = FACTOR + KP_ROWS * 4;
    static constexpr int BYTES = BARS + (3 * KP_STAGES + 7) * 8 + 16;
    static constexpr int SHARE_LD = D + 4;
    static_assert(K % 1024 == 0 && V % 1024 == 0 && H % 1024 == 0 && SCALES % 8 == 0, "swizzled tiles");
    static_assert(KP_ROWS * (SHARE_LD + 2) * 4 <= SCALES - K, "a share of the keys lies where the tiles were");
};

// the largest of three that are numbers
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// D += A B with A (float16, two to a 32-bit column) in tensor memory
__device__ __forceinline__ void umma_f16_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

template <int D, int KG>
__global__ void __launch_bounds__(KP_THREADS, D == 64 ? 2 : 1)
attn_kv8_prefill_kernel(const __nv_bfloat16* q, const float* scales, __nv_bfloat16* out, const __grid_constant__ CUtensorMap map, const K8Args a) {
    using L = KpSmem<D, KG>;
    constexpr int GROUPS = L::GROUPS, AHEAD = 32 / GROUPS;         // tiles whose pages and scales the copying warp's lanes know
    constexpr uint32_t COLS = D == 64 ? 256 : 512;         // tensor memory: two of 64 columns for scores, two of D for outputs
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map)) : "memory");
    pdl_wait();
    const uint32_t base = smem_u32(smem_raw);
    const uint32_t bars = base + L::BARS;
    auto kv_full = [&](int s) { return bars + (uint32_t)s * 8; };
    auto v_full = [&](int s) { return bars + (uint32_t)(KP_STAGES + s) * 8; };
    auto kv_empty = [&](int s) { return bars + (uint32_t)(2 * KP_STAGES + s) * 8; };
    auto s_full = [&](int b) { return bars + (uint32_t)(3 * KP_STAGES + b) * 8; };
    auto p_full = [&](int b) { return bars + (uint32_t)(3 * KP_STAGES + 2 + b) * 8; };
    auto pv_full = [&](int b) { return bars + (uint32_t)(3 * KP_STAGES + 4 + b) * 8; };
    const uint32_t q_full = bars + (3 * KP_STAGES + 6) * 8, tmem_slot = q_full + 8;
    float* row_factor = reinterpret_cast<float*>(smem_raw + L::FACTOR);
    float* share_o = reinterpret_cast<float*>(smem_raw + L::K);
    float2* share_ml = reinterpret_cast<float2*>(share_o + KP_ROWS * L::SHARE_LD);

    const int max_split = a.nsplit, Hkv = a.Hkv, H = a.H, P = a.P, G = H / Hkv;
    // the KV head fastest and the tiles in reverse: a causal tile late in its sequence reads the most keys, so the longest CTAs start first
    const int which = blockIdx.x / max_split, kvh = which % Hkv;
    const int tile = gridDim.x / (max_split * Hkv) - 1 - which / Hkv;
    const int tok0 = a.item_tok0[tile], ntok = min(a.item_ntok[tile], KP_ROWS / G);      // (a longer tile's rest is left alone)
    if (ntok <= 0) return;       // an unused entry of a fixed-length tile list (captured steps); the whole cluster's
    const int rows = ntok * G;
    const int* bt_row = a.block_table + (size_t)a.tok_seq[tok0] * a.bt_stride;
    const int pos_first = a.positions[tok0], pos_last = pos_first + ntok - 1;
    const int lo = first_seen(pos_first, a.window);
    const int j_begin = (lo / KP_KEYS) * KP_KEYS;
    // as many CTAs (a power of two) share the tile's keys as leave each KP_SPLIT_TILES key tiles; the others have nothing to do
    const int split = blockIdx.x % max_split;
    const int all_tiles = (pos_last - j_begin) / KP_KEYS + 1;
    const int most = min(max_split, max(1, all_tiles / KP_SPLIT_TILES)), nsplit = most >= 8 ? 8 : most >= 4 ? 4 : most >= 2 ? 2 : 1;
    if (split >= nsplit) return;                         // (a cluster's barrier waits for nobody who has left)
    const int n_tiles = (all_tiles - split + nsplit - 1) / nsplit;       // at least one
    auto tile_j0 = [&](int it) { return j_begin + (split + it * nsplit) * KP_KEYS; };

    if (tid == 0) {
        for (int i = 0; i < KP_STAGES; ++i) {
            mbar_init(kv_full(i), 1);
            mbar_init(v_full(i), 2);
            mbar_init(kv_empty(i), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full(i), 1);
            mbar_init(p_full(i), 4);
            mbar_init(pv_full(i), 1);
        }
        mbar_init(q_full, 8);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 3) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem_raw + (tmem_slot - base));
    const uint32_t tmem_pv = tmem + 2 * KP_KEYS;         // outputs at columns 128 + 64 b; S_b at [64 b, 64 b + 64)

    // the first four warps give registers up and the softmax warps (a whole row of scores each) take them: 128 x 48 + 256 x 96 of 384 x 80
    // (heads of 128: one CTA an SM has registers for all)
    if (warp < 4) {
        if constexpr (D == 64) asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        if (warp == 0) {
            // lane i knows the page and the scales of KG positions of one of eight tiles (KG = 8: four), and brings the page (or 64 positions of it) if
            // they are its first of the tile; asked for 16 and 8 (8 and 4) tiles ahead
            const int per = 1 << min(a.p_shift, 6), group = lane & (GROUPS - 1), at_row = (group * KG) & (per - 1);
            bool ok = true;
            auto page_of = [&](int block) {
                const int it = block * AHEAD + lane / GROUPS, j = tile_j0(it) + group * KG - at_row;
                return it < n_tiles && j <= pos_last && j + per > lo ? TK_PAGE(TK_K_KV8_ATTN, bt_row[j >> a.p_shift]) : -1;
            };
            auto scales_of = [&](int pg) {
                const float* from = scales + (size_t)max(pg, 0) * (2 * Hkv) + kvh;
                return pg >= 0 ? make_float2(from[0], from[Hkv]) : make_float2(1.f, 1.f);
            };
            int page = -1, page_next = page_of(0), page_after = page_of(1);
            float2 scale = make_float2(1.f, 1.f), scale_next = scales_of(page_next);
            float2* sc = reinterpret_cast<float2*>(smem_raw + L::SCALES);
            for (int it = 0; it < n_tiles; ++it) {
                const int s = it % KP_STAGES;
                if (it % AHEAD == 0) {
                    page = page_next;
                    scale = scale_next;
                    page_next = page_after;
                    scale_next = scales_of(page_next);
                    page_after = page_of(it / AHEAD + 2);
                }
                if (it >= KP_STAGES) ok = k8_wait(kv_empty(s), (uint32_t)((it / KP_STAGES - 1) & 1));
                if (!__all_sync(0xffffffffu, ok)) break;
                const bool ours = lane / GROUPS == it % AHEAD, mine = ours && page >= 0 && at_row == 0;
                const int loads = __popc(__ballot_sync(0xffffffffu, mine));
                if (mine) {
                    const int row = (page * 2 * Hkv + kvh) * P + ((tile_j0(it) + group * KG) & (P - 1));
                    const uint32_t at = base + (uint32_t)(s * L::RAW + group * KG * D);
                    tma_load_2d(at + L::K, &map, 0, row, kv_full(s));
                    tma_load_2d(at + L::V, &map, 0, row + Hkv * P, kv_full(s));
                }
                if (ours) sc[s * GROUPS + group] = scale;
                __syncwarp();
                // (the phase ends with this arrival and the bytes, whichever come last)
                if (lane == 0) mbar_expect_tx(kv_full(s), (uint32_t)(loads * 2 * per * D));
            }
        } else if (warp < 3) {
            // ---- V in float16, 64 columns a tile: a thread turns four or eight chunks of 16 bytes ----
            const int t = tid - 32;
            bool ok = true;
            for (int it = 0; it < n_tiles; ++it) {
                const int s = it % KP_STAGES, j0 = tile_j0(it);
                ok = k8_wait(kv_full(s), (uint32_t)((it / KP_STAGES) & 1));
                if (!__all_sync(0xffffffffu, ok)) break;
                const unsigned char* raw = smem_raw + L::V + s * L::RAW;
                unsigned char* wide = smem_raw + L::H + s * L::V16;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    const int at = t + 64 * i, key = at / (D / 16), chunk = at % (D / 16), j = j0 + key;
                    uint4 v = *reinterpret_cast<const uint4*>(raw + swizzled<D>(key, chunk));
                    if (j < lo || j > pos_last) v = make_uint4(0u, 0u, 0u, 0u);
                    uint4 x, y;
                    x.x = e4m3x2_to_half2((uint16_t)v.x), x.y = e4m3x2_to_half2((uint16_t)(v.x >> 16));
                    x.z = e4m3x2_to_half2((uint16_t)v.y), x.w = e4m3x2_to_half2((uint16_t)(v.y >> 16));
                    y.x = e4m3x2_to_half2((uint16_t)v.z), y.y = e4m3x2_to_half2((uint16_t)(v.z >> 16));
                    y.z = e4m3x2_to_half2((uint16_t)v.w), y.w = e4m3x2_to_half2((uint16_t)(v.w >> 16));
                    unsigned char* to = wide + (chunk >> 2) * L::HALF;
                    *reinterpret_cast<uint4*>(to + swizzled<128>(key, 2 * (chunk & 3))) = x;
                    *reinterpret_cast<uint4*>(to + swizzled<128>(key, 2 * (chunk & 3) + 1)) = y;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(v_full(s));
            }
        } else {
            // ---- the products: the warp walks the tiles together, one elected lane issues ----
            constexpr uint32_t id_s = idesc8(KP_ROWS, KP_KEYS, false);
            constexpr uint32_t id_pv = (1u << 4) | (1u << 16) | ((uint32_t)(64 >> 3) << 17) | ((uint32_t)(KP_ROWS >> 4) << 24);   // f16, 64 columns, V [key][d]: MN-major
            const uint64_t qd = desc8<D>(base + L::Q);
            auto wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, k8_wait(bar, parity)) != 0; };
            auto keys_of = [&](int j) { return j >= n_tiles || wait(kv_full(j % KP_STAGES), (uint32_t)((j / KP_STAGES) & 1)); };
            bool ok = n_tiles > 0 && wait(q_full, 0);
            auto issue_s = [&](int j) {                  // (one lane)
                const int b = j & 1;
                const uint64_t kd = desc8<D>(base + L::K + (uint32_t)(j % KP_STAGES) * L::RAW);
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int k = 0; k < D / 32; ++k)
                        umma_f8(tmem + (uint32_t)b * KP_KEYS, qd + (uint64_t)(t * L::Q_BYTES / 16 + 2 * k), kd + 2 * k, id_s, t + k > 0 ? 1u : 0u);
                umma_commit(s_full(b));
            };
            for (int j = 0; j < 2 && j < n_tiles && ok; ++j) {
                ok = keys_of(j);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (ok && elect_lane()) issue_s(j);
                __syncwarp();
            }
            for (int j = 0; j < n_tiles && ok; ++j) {
                const int s = j % KP_STAGES, b = j & 1;
                // (what came long ago is waited for first: a group's weights are followed by its product at once)
                ok = wait(v_full(s), (uint32_t)((j / KP_STAGES) & 1)) && keys_of(j + 2) && wait(p_full(b), (uint32_t)((j >> 1) & 1));
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t vd = desc8<128>(base + L::H + (uint32_t)s * L::V16);
                if (elect_lane()) {
#pragma unroll
                    for (int h = 0; h < D / 64; ++h)
#pragma unroll
                        for (int k = 0; k < KP_KEYS / 16; ++k)       // 16 keys: 8 columns of P, 16 rows of V
                            umma_f16_ta(tmem_pv + (uint32_t)(b * D + 64 * h), tmem + (uint32_t)(b * KP_KEYS + 8 * k), vd + (uint64_t)(h * L::HALF / 16 + 128 * k),
                                        id_pv, (j > 1 || k > 0) ? 1u : 0u);
                    // (in order behind the product that reads P_j, where S_{j+2} goes; the group's next wait is for it, and for that product)
                    if (j + 2 < n_tiles) issue_s(j + 2);
                    // (one phase of pv_full: a group that skipped phases could not tell by a phase's one bit which is open)
                    else umma_commit(pv_full(b));
                    umma_commit(kv_empty(s));
                }
                __syncwarp();
            }
        }
        __syncwarp();
    } else {
        if constexpr (D == 64) asm volatile("setmaxnreg.inc.sync.aligned.u32 96;");
        {
            // ---- q's terms: a row two threads (rows past the tile are zero) ----
            const int rr = (tid - 128) >> 1, c0 = (tid & 1) * (D / 2);
            uint4 raw[D / 16];
            float big = 0.f;
            bool fine = true;
            const __nv_bfloat16* src = q + ((size_t)(tok0 + rr / G) * H + kvh * G + rr % G) * D + c0;
#pragma unroll
            for (int e = 0; e < D / 16; ++e) {
                raw[e] = make_uint4(0u, 0u, 0u, 0u);
                if (rr < rows) raw[e] = *reinterpret_cast<const uint4*>(src + 8 * e);
            }
#pragma unroll
            for (int e = 0; e < D / 16; ++e)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t w = (&raw[e].x)[k];
                    const float u = fabsf(__uint_as_float(w << 16)), v = fabsf(__uint_as_float(w & 0xffff0000u));
                    big = fmaxf(big, fmaxf(u, v));
                    fine = fine && u <= 3.4e38f && v <= 3.4e38f;
                }
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
            fine = __shfl_xor_sync(0xffffffffu, (int)fine, 1) != 0 && fine;
            int e2 = (__float_as_int(big) >> 23) - 127;
            e2 = big == 0.f ? 7 : min(max(e2, -100), 127);
            const float up = exp2i(7 - e2);
            if ((tid & 1) == 0) row_factor[rr] = fine ? a.scale * K8_LOG2E * exp2i(e2 - 7) : NAN;        // (no score of a row that is not finite is)
#pragma unroll
            for (int e = 0; e < D / 2; e += 16) {
                uint32_t t1[4], t2[4];
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    t1[w] = t2[w] = 0;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint32_t two = (&raw[(e + 4 * w) >> 3].x)[((e + 4 * w) & 7) / 2 + k];
                        const float u = __uint_as_float(two << 16) * up, v = __uint_as_float(two & 0xffff0000u) * up;
                        const uint16_t first = to_e4m3x2(u, v);
                        const float2 back = half2_floats(e4m3x2_to_half2(first));
                        t1[w] |= (uint32_t)first << (16 * k);
                        t2[w] |= (uint32_t)to_e4m3x2(u - back.x, v - back.y) << (16 * k);
                    }
                }
                unsigned char* at = smem_raw + L::Q + swizzled<D>(rr, (c0 + e) >> 4);
                *reinterpret_cast<uint4*>(at) = make_uint4(t1[0], t1[1], t1[2], t1[3]);
                *reinterpret_cast<uint4*>(at + L::Q_BYTES) = make_uint4(t2[0], t2[1], t2[2], t2[3]);
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
        asm volatile("bar.sync 5, 256;" ::: "memory");                   // (the rows' factors)
        // ---- the weights ----
        const int grp = (warp - 4) >> 2, r = (tid - 128) & 127, quarter = warp & 3;
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        const uint32_t out_addr = tmem_pv + (uint32_t)grp * D + lane_base;
        const int pos_r = r < rows ? pos_first + r / G : -1;
        const int lo_r = first_seen(pos_r, a.window), lo_last = first_seen(pos_last, a.window);
        const float c_row = row_factor[r];
        const uint32_t s_addr = tmem + lane_base + (uint32_t)grp * KP_KEYS;
        float m_ref = -INFINITY, l_row = 0.f;
        bool ok = true;
        for (int j = grp; j < n_tiles; j += 2) {
            const int turn = j >> 1, j0 = tile_j0(j), s = j % KP_STAGES;
            // (after a failed wait the loop still runs to its end, without waiting: every thread meets the barrier behind it)
            if (ok) ok = k8_wait(kv_full(s), (uint32_t)((j / KP_STAGES) & 1));
            // (a group's scales are read when they are used, twice: the scores leave no registers to keep them in)
            const uint32_t sc = base + L::SCALES + (uint32_t)(s * GROUPS * 8);
            auto scale_of = [&](int g) {
                float2 f;
                asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(f.x), "=f"(f.y) : "r"(sc + 8u * g) : "memory");
                const float k = f.x * c_row;
                const int bits = __float_as_int(f.y);
                // (never 0: what is hidden is minus infinity before it is multiplied; NaN stays)
                return make_float3(k < 1.2e-38f ? 1.2e-38f : k, __int_as_float(0x4b000000 | (bits >> 23)) - 8388735.0f, __int_as_float((254 << 23) - bits));
            };
            if (ok) ok = k8_wait(s_full(grp), (uint32_t)(turn & 1));
            ok = __all_sync(0xffffffffu, ok);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            float x[2][32];                              // the row's 64 products stay in registers
            tmem_ld32(s_addr, x[0]);
            tmem_ld32(s_addr + 32u, x[1]);
            // a tile every row of the CTA sees whole needs no comparisons
            if (j0 + KP_KEYS - 1 > pos_first || j0 < lo_last) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const int key = j0 + 32 * h + e;
                        if (key > pos_r || key < lo_r) x[h][e] = -INFINITY;
                    }
            }
            float top = -INFINITY;
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                const float* v = &x[g * KG / 32][g * KG % 32];
                float most = fmaxf(max3(v[0], v[1], v[2]), max3(v[3], v[4], v[5]));
                most = max3(most, v[6], v[7]);
                if constexpr (KG == 16) most = max3(most, max3(max3(v[8], v[9], v[10]), v[14], v[15]), max3(v[11], v[12], v[13]));
                const float3 f = scale_of(g);
                top = fmaxf(top, fmaf(most, f.x, f.y));
            }
            if (__any_sync(0xffffffffu, top > m_ref + KP_LAZY)) {
                const float m_new = fmaxf(m_ref, top);
                if (turn >= 1) {
                    // (the product of the group's tile before has landed: it was issued ahead of these scores, whose commit covers both)
                    const float f = m_new == -INFINITY ? 1.0f : k8_exp2(m_ref - m_new);
#pragma unroll
                    for (int c = 0; c < D; c += 16) {          // (narrow: the scores stay in registers)
                        float part[16];
                        tmem_ld16(out_addr + (uint32_t)c, part);
#pragma unroll
                        for (int e = 0; e < 16; ++e) part[e] *= f;
                        tmem_st16(out_addr + (uint32_t)c, part);
                    }
                    l_row *= f;
                }
                m_ref = m_new;
            }
            const float up = m_ref == -INFINITY ? 0.f : KP_LIFT - m_ref;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t packed[16];
#pragma unroll
                for (int gg = 0; gg < 32 / KG; ++gg) {
                    const int g = 32 / KG * h + gg;
                    const float3 f = scale_of(g);
                    const float2 k2 = make_float2(f.x, f.x), b2 = make_float2(f.y + up, f.y + up);
                    float2 sum = make_float2(0.f, 0.f), alt = sum;
#pragma unroll
                    for (int e = 0; e < KG; e += 2) {
                        const float2 y = __ffma2_rn(make_float2(x[h][KG * gg + e], x[h][KG * gg + e + 1]), k2, b2);
                        const float2 w = make_float2(k8_exp2(y.x), k8_exp2(y.y));
                        if (e & 2) alt = __fadd2_rn(alt, w);
                        else sum = __fadd2_rn(sum, w);
                        const __half2 p = __floats2half2_rn(w.x, w.y);
                        packed[KG / 2 * gg + (e >> 1)] = *reinterpret_cast<const uint32_t*>(&p);
                    }
                    l_row = fmaf((sum.x + sum.y) + (alt.x + alt.y), f.z, l_row);
                }
                asm volatile(
                    "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                    ::"r"(s_addr + (uint32_t)(16 * h)), "r"(packed[0]), "r"(packed[1]), "r"(packed[2]), "r"(packed[3]), "r"(packed[4]),
                      "r"(packed[5]), "r"(packed[6]), "r"(packed[7]), "r"(packed[8]), "r"(packed[9]), "r"(packed[10]), "r"(packed[11]),
                      "r"(packed[12]), "r"(packed[13]), "r"(packed[14]), "r"(packed[15])
                    : "memory");
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full(grp));
        }
        if (ok && n_tiles > grp) ok = k8_wait(pv_full(grp), 0);
        ok = __all_sync(0xffffffffu, ok);
        // the second group's maximum and sum of each row go to q's first term, which no product reads any more: the last S of either group was issued
        // before the P V waited for above
        float2* other = reinterpret_cast<float2*>(smem_raw + L::Q) + r;
        if (grp == 1 && n_tiles > 1) *other = make_float2(m_ref, l_row);
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        asm volatile("bar.sync 5, 256;" ::: "memory");
        if (grp == 0 && n_tiles > 0) {
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            // both outputs under one reference: o = f0 o0 + f1 o1
            const bool two = n_tiles > 1;
            const float2 theirs = two ? *other : make_float2(-INFINITY, 0.f);
            const float m_all = fmaxf(m_ref, theirs.x);
            const float f0 = k8_factor(m_ref, l_row, m_all), f1 = k8_factor(theirs.x, theirs.y, m_all);
            l_row = two ? fmaf(l_row, f0, theirs.y * f1) : l_row;
            m_ref = m_all;
            const int tok = tok0 + r / G, head = kvh * G + r % G;
            __nv_bfloat16* dst = out + ((size_t)tok * H + head) * D;
            float inv = 1.f, gate = 1.f;
            if (nsplit == 1) {
                if (a.sink && m_ref > -INFINITY) l_row += k8_exp2(KP_LIFT - m_ref);
                inv = l_row == 0.f ? 0.f : 1.0f / l_row;
                if (r < rows) gate = k8_gate<__nv_bfloat16>(a, tok, head);
            }
#pragma unroll
            for (int c = 0; c < D; c += 16) {
                float v[16], more[16];
                tmem_ld16(out_addr + (uint32_t)c, v);
                if (two) tmem_ld16(out_addr + (uint32_t)(D + c), more);
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = two ? fmaf(v[e], f0, more[e] * f1) : v[e];
                if (nsplit > 1) {
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        *reinterpret_cast<float4*>(share_o + r * L::SHARE_LD + c + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
                } else if (r < rows) {
                    uint32_t packed[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const __nv_bfloat162 y = __floats2bfloat162_rn(k8_apply<__nv_bfloat16>(v[2 * e] * inv, a, gate),
                                                                       k8_apply<__nv_bfloat16>(v[2 * e + 1] * inv, a, gate));
                        packed[e] = *reinterpret_cast<const uint32_t*>(&y);
                    }
                    *reinterpret_cast<uint4*>(dst + c) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
                    *reinterpret_cast<uint4*>(dst + c + 8) = make_uint4(packed[4], packed[5], packed[6], packed[7]);
                }
            }
            if (nsplit > 1) share_ml[r] = make_float2(m_ref, l_row);
        }
    }
    if (nsplit > 1) {
        // every CTA forms an equal part of the columns from all shares, through the cluster's shared memory
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        if (warp >= 4) {
            const int r = (tid - 128) & 127;
            const int tok = tok0 + r / G, head = kvh * G + r % G;
            auto merge = [&](auto shares) {
                // eight reads of four columns a thread, whatever the number of shares, all in flight together
                constexpr int NS = decltype(shares)::value, PER = D / 2 / NS;
                const int c0 = split * 2 * PER + ((tid - 128) >> 7) * PER;
                float2 ml[NS];
                float4 o[NS][PER / 4];
#pragma unroll
                for (int sp = 0; sp < NS; ++sp) {
                    ml[sp] = cluster.map_shared_rank(share_ml, sp)[r];
                    const float* from = cluster.map_shared_rank(share_o, sp) + r * L::SHARE_LD + c0;
#pragma unroll
                    for (int k = 0; k < PER / 4; ++k) o[sp][k] = *reinterpret_cast<const float4*>(from + 4 * k);
                }
                float m_all = -INFINITY, l_all = 0.f;
#pragma unroll
                for (int sp = 0; sp < NS; ++sp) m_all = fmaxf(m_all, ml[sp].x);
#pragma unroll
                for (int sp = 0; sp < NS; ++sp) {
                    ml[sp].x = k8_factor(ml[sp].x, ml[sp].y, m_all);
                    l_all = fmaf(ml[sp].y, ml[sp].x, l_all);
                }
                if (a.sink && m_all > -INFINITY) l_all += k8_exp2(KP_LIFT - m_all);
                const float inv = l_all == 0.f ? 0.f : 1.0f / l_all;
                if (r >= rows) return;
                const float gate = k8_gate<__nv_bfloat16>(a, tok, head);
#pragma unroll
                for (int k = 0; k < PER / 4; ++k) {
                    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int sp = 0; sp < NS; ++sp)
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = fmaf((&o[sp][k].x)[e], ml[sp].x, v[e]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = k8_apply<__nv_bfloat16>(v[e] * inv, a, gate);
                    Quad<__nv_bfloat16>::store(out + ((size_t)tok * H + head) * D + c0 + 4 * k, make_float4(v[0], v[1], v[2], v[3]));
                }
            };
            if (nsplit == 2) merge(std::integral_constant<int, 2>());
            else if (nsplit == 4) merge(std::integral_constant<int, 4>());
            else merge(std::integral_constant<int, 8>());
        }
        cluster.sync();                                  // nobody leaves while its share is read
    }
    // ---- teardown: the tensor memory goes back whatever happened above ----
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 3) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS) : "memory");
    }
}

template <int D, int KG>
cudaError_t kp_config(cudaLaunchConfig_t& cfg, cudaLaunchAttribute* attr, int64_t ctas, int nsplit, cudaStream_t stream) {
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = k8_allow(attn_kv8_prefill_kernel<D, KG>, KpSmem<D, KG>::BYTES, false, done);
    if (e != cudaSuccess) return e;
    cfg = {};
    cfg.gridDim = dim3((unsigned)(ctas * nsplit));
    cfg.blockDim = dim3(KP_THREADS);
    cfg.dynamicSmemBytes = KpSmem<D, KG>::BYTES;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = k8_attributes(attr, nsplit);
    return cudaSuccess;
}

template <int D, int KG>
cudaError_t kp_launch(const void* q, const float* scales, void* out, const CUtensorMap& map, const K8Args& a, cudaStream_t stream) {
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[2];
    const cudaError_t e = kp_config<D, KG>(cfg, attr, (int64_t)a.items * a.Hkv, a.nsplit, stream);
    if (e != cudaSuccess) return e;
    return cudaLaunchKernelEx(&cfg, attn_kv8_prefill_kernel<D, KG>, (const __nv_bfloat16*)q, scales, (__nv_bfloat16*)out, map, a);
}

// clusters of n CTAs that a device with one CTA an SM holds, asked for once (n: 2, 4 or 8)
template <int D, int KG>
cudaError_t kp_clusters(int n, int* clusters) {
    static std::atomic<int> known[16][9];
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess || (device < 16 && (*clusters = known[device][n].load(std::memory_order_relaxed)) > 0)) return e;
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[2];
    e = kp_config<D, KG>(cfg, attr, 1, n, nullptr);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(clusters, attn_kv8_prefill_kernel<D, KG>, &cfg);
    if (e == cudaSuccess && device < 16) known[device][n].store(*clusters, std::memory_order_relaxed);
    return e;
}

}  // namespace

// How many clusters of n CTAs (2, 4 or 8) are resident at once. Heads of 128 fill an SM's tensor memory with one CTA, and clusters lie in whole parts of the device: the
// occupancy calculator says 74 of 2, 33 of 4, 15 of 8 for 148 SMs. Heads of 64 have two CTAs an SM.
int tk_attn_kv8_prefill_clusters(int D, int P, int n, int sm_count) {
    if (D == 64) return k8_clusters(2, sm_count, n);
    int clusters = 0;
    if ((P == 8 ? kp_clusters<128, 8>(n, &clusters) : kp_clusters<128, 16>(n, &clusters)) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return clusters;
}

// The arguments of tk_attn_kv8 for tiles (attention_kv8.cu checks them): bfloat16, pages that are a power of two and 8 or more.
int tk_attn_kv8_prefill_tc(const void* q, const void* pool, const float* scales, void* out, const void* args, int D, cudaStream_t stream) {
    const K8Args& a = *static_cast<const K8Args*>(args);
    CUtensorMap map = {};
    TK_CHECK_ARG(k8_map(&map, pool, D, a.P < KP_KEYS ? a.P : KP_KEYS), "attn_kv8: cuTensorMapEncodeTiled failed");
    const cudaError_t e = a.P == 8 ? (D == 64 ? kp_launch<64, 8>(q, scales, out, map, a, stream) : kp_launch<128, 8>(q, scales, out, map, a, stream))
                                   : (D == 64 ? kp_launch<64, 16>(q, scales, out, map, a, stream) : kp_launch<128, 16>(q, scales, out, map, a, stream));
    if (e != cudaSuccess) {
        tk_set_error("attn_kv8: launch failed: %s", cudaGetErrorString(e));
        cudaGetLastError();
        return -2;
    }
    return 0;
}

int tk_attn_kv8_prefill_tc_status() { return k8_take_status(); }
