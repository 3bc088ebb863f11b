// Single tokens' attention over the 8-bit cache (kv8.cuh) on the fifth-generation tensor cores, for bfloat16: the cache's bytes are the products'
// operands as they lie in memory, no instruction ever touches them.
//
//   S^T = K q^T      tcgen05.mma kind::f8f6f4, M = 128 keys, a column a query head: a thread owns a key and reads its scores
//   O^T += V^T P^T   M = D, the same columns: V's [key][d] is the M-major operand as it lands
//
// What is not 8-bit is a sum of 8-bit terms, a column each, added up when they are read: e4m3 has four significant bits, so q (after
// division by a power of two that brings its row's largest to [128, 256)) is two terms, exactly for elements down to 2^-12 of the row's
// largest and to 2^-18 of that below. A weight is four: two that leave 2^-8 of it or 2^-10 (e4m3's smallest steps), and two of what they leave times
// 2^8. The weights' reference maximum follows lazily (raised when a row exceeds it by 2^2) and weights are lifted by 2^6 (at most 256, of 448): a
// weight is off by at most 2^-16 of itself or 2^-24 of the row's largest. (Two terms alone lose the many small weights beside a large one: 30,000
// keys that share half of a row's weight with one that has the other half would be off by a tenth.) A value block's scale is in the
// exponent, as in attention_kv8.cu. Columns cost nothing here: a product's time is that of reading its 128 x 32 or D x 32 bytes of the first operand
// from shared memory. (With the heads as the M side of the second product, 32 rows of 128, and the terms one after the other, the products
// alone took 575 cycles a tile of 128 keys, and 8 tokens behind 32,000 positions 71 us.)
//
// A CTA takes the query heads of one KV head of one token and a share of its keys, in tiles of 128:
//   warp 4      brings K and V by TMA, a page (or 128 positions of one) a load, two or three tiles ahead
//   warp 5      issues the products
//   warps 0-3   thread = key: masks, reference maximum (one vote of the four warps a tile), weights, their terms into shared memory
//               ([term and head][key], the second product's other operand); positions that are not to be seen have their value rows zeroed there
//
// Masking and sums are those of attention_kv8.cu; every wait is bounded (about a second), the kernel then frees its tensor memory and
// returns, and tk_attn_kv8_status() says so.
#include <math.h>

#include "kv8.cuh"
#include "kv8_attn.cuh"
#include "tcgen05.cuh"

namespace {

constexpr int K8T_KEYS = 128, K8T_ROWS = 16;
constexpr int K8T_THREADS = 192;
constexpr int K8T_QTERMS = 2, K8T_PTERMS = 4;
constexpr float K8T_LAZY = 2.0f, K8T_LIFT = 6.0f, K8T_FINE = 256.0f;

// K-major or MN-major operand whose rows are D = 64 (64-byte swizzle) or 128 bytes (128-byte swizzle), groups of eight rows one after the other
template <int BYTES>
__device__ __forceinline__ uint64_t desc8(uint32_t at) {
    uint64_t d = 0;
    d |= (uint64_t)((at & 0x3FFFF) >> 4);
    d |= (uint64_t)1 << 16;
    d |= (uint64_t)((8 * BYTES) >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)(BYTES == 64 ? 4 : 2) << 61;
    return d;
}
// byte offset of 16-byte chunk `chunk` of row `row`
template <int BYTES>
__device__ __forceinline__ uint32_t swizzled(int row, int chunk) {
    return (uint32_t)(row * BYTES + ((BYTES == 64 ? chunk ^ ((row >> 1) & 3) : chunk ^ (row & 7)) << 4));
}

// e4m3 x e4m3 -> f32
__host__ __device__ constexpr uint32_t idesc8(int m, int n, bool a_m_major) {
    return (1u << 4) | (a_m_major ? 1u << 15 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ bool elect_lane() {
    uint32_t mine;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(mine));
    return mine != 0;
}

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

// tiles of keys and values in shared memory: as many as leave room for three CTAs an SM (D = 64), or two
template <int D>
constexpr int k8t_stages = D == 64 ? 3 : 2;

template <int D, int NR>
struct K8tSmem {
    static constexpr int STAGES = k8t_stages<D>;
    static constexpr int S_COLS = 2 * NR < 16 ? 16 : 2 * NR;                       // scores' columns: term, head
    static constexpr int O_COLS = 4 * NR < 16 ? 16 : 4 * NR;                       // outputs' columns: term, head
    static constexpr int P_BYTES = O_COLS * K8T_KEYS;                              // [term, head][key], 128-byte swizzle
    static constexpr int P = 0;                                                    // two of them
    static constexpr int Q = 2 * P_BYTES;                                          // [term, head][d]
    static constexpr int KV = Q + (S_COLS * D < 1024 ? 1024 : S_COLS * D);         // stages: K tile, V tile
    static constexpr int STAGE = 2 * K8T_KEYS * D;
    static constexpr int BARS = KV + STAGES * STAGE;
    static constexpr int MISC = BARS + (2 * STAGES + 6) * 8 + 16;
    static constexpr int BYTES = MISC + (16 * 4 + 4 * 16 * 4);                     // row factors, warps' maxima or sums
    static_assert(Q % 1024 == 0 && KV % 1024 == 0, "swizzled tiles");
};

// D: head size; NR: query heads a KV head has, rounded up to 2, 4, 8 or 16
template <int D, int NR>
__global__ void __launch_bounds__(K8T_THREADS)
attn_kv8_tc_kernel(const __nv_bfloat16* q, const float* scales, __nv_bfloat16* out, const __grid_constant__ CUtensorMap map, const K8Args a) {
    using L = K8tSmem<D, NR>;
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
    constexpr uint32_t COLS = 128;                                                // tensor memory: two of up to 32 columns for scores, up to 64 for outputs

    if (tid == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(kv_full(i), 1);
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
    if (warp == 5) {
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

    if (warp == 4) {
        // ---- K and V: lane i brings positions [i per, (i + 1) per) of a tile, if any of them may be read ----
        const int per_log = min(a.p_shift, 7), per = 1 << per_log;
        bool ok = true;
        for (int it = 0; it < n_tiles; ++it) {
            const int s = it % STAGES, j = (t_begin + it) * K8T_KEYS + lane * per;
            const bool mine = lane < (K8T_KEYS >> per_log) && j <= pos && j + per > lo;
            int page = 0;
            if (mine) page = TK_PAGE(TK_K_KV8_ATTN, bt[j >> a.p_shift]);
            if (it >= STAGES) ok = k8_wait(kv_empty(s), (uint32_t)((it / STAGES - 1) & 1));
            if (!__all_sync(0xffffffffu, ok)) break;
            const int loads = __popc(__ballot_sync(0xffffffffu, mine));
            if (lane == 0) mbar_expect_tx(kv_full(s), (uint32_t)(loads * 2 * per * D));
            __syncwarp();
            if (mine) {
                const int row = ((page * 2) * a.Hkv + kvh) * P + (j & (P - 1));
                const uint32_t at = base + L::KV + (uint32_t)s * L::STAGE + (uint32_t)(lane * per * D);
                tma_load_2d(at, &map, 0, row, kv_full(s));
                tma_load_2d(at + K8T_KEYS * D, &map, 0, row + a.Hkv * P, kv_full(s));
            }
        }
    } else if (warp == 5) {
        // ---- the products ----
        constexpr uint32_t id_s = idesc8(K8T_KEYS, L::S_COLS, false), id_o = idesc8(D, L::O_COLS, true);
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
            const uint64_t pd = desc8<128>(base + L::P + b * L::P_BYTES);
            if (elect_lane()) {
#pragma unroll
                for (int k = 0; k < K8T_KEYS / 32; ++k)
                    umma_f8(tmem_o, vd + (uint64_t)(k * 32 * D / 16), pd + 2 * k, id_o, j + k > 0 ? 1u : 0u);
                umma_commit(pv_full(b));
                umma_commit(kv_empty(s));
            }
            __syncwarp();
        }
    } else {
        // ---- the weights ----
        float c[NR], m[NR], l[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            c[r] = row_factor[r];
            m[r] = -INFINITY;
            l[r] = 0.f;
        }
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        bool ok = true;
        // a key's page is looked up two tiles ahead of its use, its scales one
        auto page_of = [&](int it) {
            const int j = (t_begin + it) * K8T_KEYS + tid;
            return it < n_tiles && j >= lo && j <= pos ? TK_PAGE(TK_K_KV8_ATTN, bt[j >> a.p_shift]) : -1;
        };
        int page = page_of(0);
        float ks = 1.f, vs = 1.f;
        auto scales_of = [&](int pg) {
            const float* sc = scales + (size_t)max(pg, 0) * (2 * a.Hkv) + kvh;
            ks = pg >= 0 ? sc[0] : 1.f;
            vs = pg >= 0 ? sc[a.Hkv] : 1.f;
        };
        scales_of(page);
        page = page_of(1);
        for (int it = 0; it < n_tiles; ++it) {
            const int b = it & 1, turn = it >> 1, j = (t_begin + it) * K8T_KEYS + tid;
            const bool seen = j >= lo && j <= pos;
            const float k_now = ks;
            const int bits = __float_as_int(vs);
            const float ev = __int_as_float(0x4b000000 | (bits >> 23)) - 8388735.0f, inv_v = __int_as_float((254 << 23) - bits);
            scales_of(page);
            page = page_of(it + 2);
            // (after a failed wait the loop runs to its end without waiting: every thread meets every barrier)
            if (ok) ok = k8_wait(s_full(b), (uint32_t)(turn & 1));
            ok = __all_sync(0xffffffffu, ok);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            float x[NR];
            {
                constexpr int N = 2 * NR < 8 ? 8 : 2 * NR;
                float sum[N];
                tmem_ld_n<N>(tmem + lanes + (uint32_t)b * 32, sum);
#pragma unroll
                for (int r = 0; r < NR; ++r) x[r] = sum[r] + sum[NR + r];
            }
            bool above = false;
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                x[r] = seen ? fmaf(x[r], k_now * c[r], ev) : -INFINITY;
                above = above || x[r] > m[r] + K8T_LAZY;
            }
            if (any_of_128(above)) {
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    const float top = warp_max(x[r]);
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
            unsigned char* p = smem_raw + L::P + b * L::P_BYTES + (tid & 15);
#pragma unroll
            for (int r = 0; r < NR; r += 2) {
                float w[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    w[h] = k8_exp2(x[r + h] + (m[r + h] == -INFINITY ? 0.f : K8T_LIFT - m[r + h]));
                    l[r + h] = fmaf(w[h], inv_v, l[r + h]);
                }
#pragma unroll
                for (int t = 0; t < K8T_PTERMS; ++t) {
                    const uint16_t two = to_e4m3x2(w[0], w[1]);
                    p[swizzled<128>(t * NR + r, tid >> 4)] = (unsigned char)two;
                    p[swizzled<128>(t * NR + r + 1, tid >> 4)] = (unsigned char)(two >> 8);
                    const float2 back = half2_floats(e4m3x2_to_half2(two));
                    w[0] -= back.x;
                    w[1] -= back.y;
                    if (t == 1) {
                        w[0] *= K8T_FINE;
                        w[1] *= K8T_FINE;
                    }
                }
            }
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
                float o = fmaf(v[2 * NR + r] + v[3 * NR + r], 1.f / K8T_FINE, v[r] + v[NR + r]);
                float l_r = (by_warp[r] + by_warp[16 + r]) + (by_warp[32 + r] + by_warp[48 + r]);
                const int head = kvh * G + r;
                if (a.nsplit == 1) {
                    if (a.sink && m[r] > -INFINITY) l_r += k8_exp2(K8T_LIFT - m[r]);
                    o = l_r == 0.f ? 0.f : o / l_r;
                    out[((size_t)tok * a.H + head) * D + d] = __float2bfloat16_rn(k8_apply<__nv_bfloat16>(o, a, k8_gate<__nv_bfloat16>(a, tok, head)));
                } else {
                    float* part = a.scratch + ((((size_t)item * a.Hkv + kvh) * a.nsplit + split) * a.rows_most + r) * (D + 4);
                    part[d] = o;
                    if (d == 0) *reinterpret_cast<float2*>(part + D) = make_float2(m[r], l_r);
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 5) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS) : "memory");
    }
}

// the cache as rows of D bytes, boxes of a page or of 128 positions of one
bool k8t_map(CUtensorMap* map, const void* pool, int D, int P) {
    EncodeTiled fn = encode_fn();
    if (fn == nullptr) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)D, 0x7fffffffu};
    const cuuint64_t strides[1] = {(cuuint64_t)D};
    const cuuint32_t box[2] = {(cuuint32_t)D, (cuuint32_t)(P < K8T_KEYS ? P : K8T_KEYS)};
    const cuuint32_t estr[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(pool), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int NR>
cudaError_t k8t_launch(const void* q, const float* scales, void* out, const CUtensorMap& map, const K8Args& a, cudaStream_t stream) {
    constexpr int smem = K8tSmem<D, NR>::BYTES;
    cudaError_t e = cudaFuncSetAttribute(attn_kv8_tc_kernel<D, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    return tk_launch(attn_kv8_tc_kernel<D, NR>, dim3((unsigned)(a.items * a.Hkv * a.nsplit)), dim3(K8T_THREADS), smem, stream, (const __nv_bfloat16*)q,
                     scales, (__nv_bfloat16*)out, map, a);
}

template <int D>
cudaError_t k8t_rows(const void* q, const float* scales, void* out, const CUtensorMap& map, const K8Args& a, cudaStream_t stream) {
    const int G = a.H / a.Hkv;
    cudaError_t e = G <= 2   ? k8t_launch<D, 2>(q, scales, out, map, a, stream)
                    : G <= 4 ? k8t_launch<D, 4>(q, scales, out, map, a, stream)
                    : G <= 8 ? k8t_launch<D, 8>(q, scales, out, map, a, stream)
                             : k8t_launch<D, 16>(q, scales, out, map, a, stream);
    if (e != cudaSuccess || a.nsplit == 1) return e;
    const unsigned grid = (unsigned)(((int64_t)a.items * a.Hkv * a.rows_most + 3) / 4);
    return tk_launch(attn_kv8_merge_kernel<__nv_bfloat16, D>, dim3(grid), dim3(128), 0, stream, (__nv_bfloat16*)out, a, K8T_LIFT);
}

}  // namespace

// The arguments of tk_attn_kv8 for single tokens (attention_kv8.cu checks them): bfloat16, pages that are a power of two and 16 or more.
int tk_attn_kv8_tc(const void* q, const void* pool, const float* scales, void* out, const void* args, int D, cudaStream_t stream) {
    const K8Args& a = *static_cast<const K8Args*>(args);
    CUtensorMap map = {};
    TK_CHECK_ARG(k8t_map(&map, pool, D, a.P), "attn_kv8: cuTensorMapEncodeTiled failed");
    const cudaError_t e = D == 64 ? k8t_rows<64>(q, scales, out, map, a, stream) : k8t_rows<128>(q, scales, out, map, a, stream);
    if (e != cudaSuccess) {
        tk_set_error("attn_kv8: launch failed: %s", cudaGetErrorString(e));
        cudaGetLastError();
        return -2;
    }
    return 0;
}

int tk_attn_kv8_tc_status() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_k8_error, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) cudaMemcpyToSymbol(g_k8_error, &zero, sizeof(int));
    return v;
}
