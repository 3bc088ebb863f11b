// Attention over the 8-bit cache (kv8.cuh) on mma.sync.m16n8k16, with float16 operands and 32-bit sums: single tokens of any
// model, and prompt portions of the sizes that the tcgen05 kernel (attention_kv8_tc.cu) does not take.
//
//   o[r] = sum_j p_rj v_j / sum_j p_rj,   p_rj = exp(scale * q_r . k_j),   k_j = s_K kb_j,  v_j = s_V vb_j   (bytes kb, vb)
//
// A CTA takes 16 rows (tokens of one sequence x the query heads of one KV head; one token when it decodes) and a share of their
// keys; its warps walk groups of 32 (16 for heads of 128) keys in turn and are joined through shared memory, the CTAs of a
// row through scratch memory and a second kernel.
//
// Bytes to operands without shared memory. The order of a product's inner index is free as long as both operands follow it, and the order of the output's columns is
// too: a lane reads D / 4 bytes side by side of one key's row (16 bytes for D = 64; four lanes a row) and uses them as its fragments of all the D / 16
// steps of q . k, with q's fragments laid out to match; and of a value row it reads D / 8 bytes, one for each of the D / 8 column tiles, so that two rows' bytes
// interleave (prmt) into the pairs that a fragment holds. e4m3 is exact in float16.
//
// What is rounded: q (bfloat16: not at all, 32-bit: to 22 bits, as two float16 with two products) after division by a power of two that brings its row
// to [2^14, 2^15), so that its small elements keep their bits; the weights to float16's 11 bits (32-bit: 22, as two). Scores, the running
// maximum, sums and outputs are 32-bit; the output is rounded once.
//
// A value block's scale joins the exponent: with x_j = log2(p_j) + log2(s_V), w_j = 2^(x_j - m + 7) are the weights of the bytes, m following their
// running maximum lazily (it is raised when a row exceeds it by 8, so w <= 2^15), and the softmax's sum is of w_j / s_V. No weight then
// loses bits to float16's range against a larger one, however far apart the blocks' scales are.
//
// Masked keys and values are never read (their bytes are zero in the products), so what an unwritten part of a page holds does not
// matter. A row that sees no key is 0.
//
// Bound by HBM for long contexts; measured figures stand with the entry points.
#include <math.h>

#include <type_traits>

#include "kv8.cuh"

namespace {

constexpr int K8_ROWS = 16;
constexpr int K8_WARPS = 4, K8_THREADS = K8_WARPS * 32;
constexpr float K8_LOG2E = 1.4426950408889634f;
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
__device__ __forceinline__ float2 half2_floats(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }

__device__ __forceinline__ float k8_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct K8Args {
    const int* positions;
    const int* tok_seq;
    const int* block_table;
    const int* item_tok0;        // tiles' first tokens, or rows of single tokens (null: item i is row i)
    const int* item_ntok;        // tiles' tokens (null: one each)
    const void* gate;
    float* scratch;              // [item, KV head, split, row] D + 2 floats, when nsplit > 1
    int64_t ldg;
    int bt_stride, items, H, Hkv, P, p_shift, window, nsplit, sink, rows_most;
    float scale;
};

// The share of a row's keys that one CTA or warp has seen, under reference m: o = sum w v, l = sum w / s_V.
__device__ __forceinline__ float k8_factor(float m, float l, float m_all) {
    // (nothing seen: left out; a sum that is not a number under no maximum: every score was one)
    return m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : k8_exp2(m - m_all);
}

template <typename T>
__device__ __forceinline__ float k8_gated(float o, const K8Args& a, int tok, int head) {
    o = round_as<T>(o);
    if (a.gate == nullptr) return o;
    const float g = to_f<T>(reinterpret_cast<const T*>(a.gate)[(size_t)tok * a.ldg + head]);
    return o * round_as<T>(1.0f / (1.0f + expf(-g)));
}

// T: type of q and the output. D: head size. PAGE16: pages are a multiple of 16 positions and a power of two, so 16 keys that begin at a multiple of
// 16 lie in one page; otherwise every lane looks its own keys' pages up.
template <typename T, int D, bool PAGE16>
__global__ void __launch_bounds__(K8_THREADS)
attn_kv8_kernel(const T* q, const uint8_t* pool, const float* scales, T* out, const K8Args a) {
    constexpr bool WIDE = sizeof(T) == 4;                // q and the weights as two float16
    constexpr int U = D == 64 ? 2 : 1;                   // groups of 16 keys a warp takes at a time
    constexpr int KS = D / 16, NT = D / 8;               // steps of q . k, column tiles of the output
    constexpr int KW = D / 64;                           // 16-byte words a lane reads of a key
    constexpr int VW = D / 32;                           // 4-byte words a lane reads of a value row
    extern __shared__ float smem[];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, c = lane & 3;
    const int split = blockIdx.x % a.nsplit, kvh = (blockIdx.x / a.nsplit) % a.Hkv, item = blockIdx.x / (a.nsplit * a.Hkv);
    const int tok0 = a.item_tok0 != nullptr ? a.item_tok0[item] : item;
    const int ntok = a.item_ntok != nullptr ? a.item_ntok[item] : 1;
    if (tok0 < 0 || ntok <= 0) return;                   // a padded entry of a recorded step
    const int G = a.H / a.Hkv, rows = ntok * G;
    const int* bt = a.block_table + (size_t)a.tok_seq[tok0] * a.bt_stride;
    const int pos_first = a.positions[tok0], pos_last = pos_first + ntok - 1;
    const int lo = first_seen(pos_first, a.window), lo_last = first_seen(pos_last, a.window);
    // groups of 16 keys, from the one that holds `lo`; this CTA's are [g_begin, g_end), its warps take U of them in turn
    const int g_lo = lo >> 4, g_all = (pos_last >> 4) - g_lo + 1;
    const int units = (g_all + U - 1) / U;
    const int g_begin = g_lo + (int)((int64_t)units * split / a.nsplit) * U;
    const int g_end = min(g_lo + (int)((int64_t)units * (split + 1) / a.nsplit) * U, g_lo + g_all);

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
        // a row's largest element to [2^14, 2^15) (a row that is not finite stays as it is)
        int e2 = (__float_as_int(most) >> 23) - 127;
        e2 = e2 > 127 || most == 0.f ? 14 : max(e2, -100);
        const float up = exp2i(14 - e2);
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

    // ---- keys and values: the next groups' bytes and scales are on their way while these are used ----
    const int P = a.P;
    const size_t head = (size_t)kvh * P * D, v_delta = (size_t)a.Hkv * P * D, page_bytes = 2 * v_delta;
    uint4 kw[U][2][KW];
    uint32_t vw[U][4][VW];
    constexpr int NS = PAGE16 ? 1 : 4;                   // scales a group has for a lane: one, or one for each of its four keys
    float ks_[U][NS], vs_[U][NS];
    int page_next[U];
    auto look_up = [&](int gr) {
        if constexpr (PAGE16) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                page_next[u] = gr + u < g_end ? TK_PAGE(TK_K_KV8_ATTN, bt[((gr + u) << 4) >> a.p_shift]) : 0;
        }
    };
    auto load = [&](int gr) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j0 = (gr + u) << 4;
            const bool whole = gr + u < g_end;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int j = j0 + 8 * t + g;
                const bool there = whole && j >= lo && j <= pos_last;
                const uint8_t* src = nullptr;
                if (there) {
                    const int page = PAGE16 ? page_next[u] : TK_PAGE(TK_K_KV8_ATTN, bt[j / P]);
                    src = pool + (size_t)page * page_bytes + head + (size_t)(PAGE16 ? j & (P - 1) : j % P) * D + c * (D / 4);
                }
#pragma unroll
                for (int w = 0; w < KW; ++w) kw[u][t][w] = there ? *reinterpret_cast<const uint4*>(src + 16 * w) : make_uint4(0u, 0u, 0u, 0u);
            }
            if constexpr (PAGE16) {
                const float* s = scales + (size_t)page_next[u] * 2 * a.Hkv + kvh;
                ks_[u][0] = whole ? s[0] : 1.f;
                vs_[u][0] = whole ? s[a.Hkv] : 1.f;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = j0 + 2 * c + (i & 1) + 8 * (i >> 1);
                const bool there = whole && j >= lo && j <= pos_last;
                const uint8_t* src = nullptr;
                int page = 0;
                if (there) {
                    page = PAGE16 ? page_next[u] : TK_PAGE(TK_K_KV8_ATTN, bt[j / P]);
                    src = pool + (size_t)page * page_bytes + head + v_delta + (size_t)(PAGE16 ? j & (P - 1) : j % P) * D + g * (D / 8);
                }
                if constexpr (!PAGE16) {
                    const float* s = scales + (size_t)page * 2 * a.Hkv + kvh;
                    ks_[u][i] = there ? s[0] : 1.f;
                    vs_[u][i] = there ? s[a.Hkv] : 1.f;
                }
                if constexpr (VW == 2) {
                    const uint2 w = there ? *reinterpret_cast<const uint2*>(src) : make_uint2(0u, 0u);
                    vw[u][i][0] = w.x, vw[u][i][1] = w.y;
                } else {
                    const uint4 w = there ? *reinterpret_cast<const uint4*>(src) : make_uint4(0u, 0u, 0u, 0u);
                    vw[u][i][0] = w.x, vw[u][i][1] = w.y, vw[u][i][2] = w.z, vw[u][i][3] = w.w;
                }
            }
        }
    };

    float o[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    constexpr int STEP = K8_WARPS * U;
    int gr = g_begin + warp * U;
    if (gr < g_end) {
        look_up(gr);
        load(gr);
        look_up(gr + STEP);
    }
    for (; gr < g_end; gr += STEP) {
        // scores in base-2 logarithms with the value blocks' exponents in them: x[u][t] of keys 2c, 2c + 1 of tile t, rows g and g + 8
        float x[U][2][4], inv_vs[U][NS];
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
            float ksc[NS], ev[NS];
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                const int be = (__float_as_int(vs_[u][i]) >> 23) & 255;
                ev[i] = (float)(be - 127);
                inv_vs[u][i] = __int_as_float((254 - be) << 23);
                ksc[i] = ks_[u][i];
            }
            const int j0 = (gr + u) << 4;
            const bool masked = j0 + 15 > pos_first || j0 < lo_last || gr + u >= g_end;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = PAGE16 ? 0 : 2 * t + (e & 1);
                    x[u][t][e] = fmaf(x[u][t][e], ksc[i] * row_c[e >> 1], ev[i]);
                    if (masked) {
                        const int j = j0 + 8 * t + 2 * c + (e & 1), p = row_pos[e >> 1];
                        if (j > p || j < first_seen(p, a.window) || gr + u >= g_end) x[u][t][e] = -INFINITY;
                    }
                }
        }
        // the values' bytes leave their registers before the next groups' arrive
        uint32_t vc[U][4][VW];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int w = 0; w < VW; ++w) vc[u][i][w] = vw[u][i][w];
        if (gr + STEP < g_end) {
            load(gr + STEP);
            look_up(gr + 2 * STEP);
        }
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) top[e >> 1] = fmaxf(top[e >> 1], x[u][t][e]);
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
                    const float w0 = k8_exp2(x[u][t][2 * hrow] + base[hrow]), w1 = k8_exp2(x[u][t][2 * hrow + 1] + base[hrow]);
                    l[hrow] = fmaf(w0, inv_vs[u][PAGE16 ? 0 : 2 * t], l[hrow]);
                    l[hrow] = fmaf(w1, inv_vs[u][PAGE16 ? 0 : 2 * t + 1], l[hrow]);
                    pa[hrow + 2 * t] = half2_bits(w0, w1);
                    if constexpr (WIDE) {
                        const float2 hi = half2_floats(pa[hrow + 2 * t]);
                        pb[hrow + 2 * t] = half2_bits(w0 - hi.x, w1 - hi.y);
                    }
                }
#pragma unroll
            for (int w = 0; w < VW; ++w)
#pragma unroll
                for (int pair = 0; pair < 2; ++pair) {
                    const uint32_t sel = pair ? 0x7362 : 0x5140;
                    const uint32_t y0 = __byte_perm(vc[u][0][w], vc[u][1][w], sel), y1 = __byte_perm(vc[u][2][w], vc[u][3][w], sel);
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
            y.x = k8_gated<T>(v[0] * inv, a, tok, hd), y.y = k8_gated<T>(v[1] * inv, a, tok, hd);
            y.z = k8_gated<T>(v[2] * inv, a, tok, hd), y.w = k8_gated<T>(v[3] * inv, a, tok, hd);
            Quad<T>::store(out + ((size_t)tok * a.H + hd) * D + col, y);
        } else {
            float* part = a.scratch + ((((size_t)item * a.Hkv + kvh) * a.nsplit + split) * a.rows_most + r) * (D + 4);
            *reinterpret_cast<float4*>(part + col) = make_float4(v[0], v[1], v[2], v[3]);
            if (col == 0) *reinterpret_cast<float2*>(part + D) = make_float2(m_all, l_all);
        }
    }
}

// The CTAs' shares of a row joined: a warp a row, D / 32 columns a lane.
template <typename T, int D>
__global__ void __launch_bounds__(128)
attn_kv8_merge_kernel(T* out, const K8Args a) {
    constexpr int C = D / 32;
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, G = a.H / a.Hkv;
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int r = (int)(at % a.rows_most), kvh = (int)(at / a.rows_most % a.Hkv);
    const int64_t item = at / ((int64_t)a.rows_most * a.Hkv);
    if (item >= a.items) return;
    const int tok0 = a.item_tok0 != nullptr ? a.item_tok0[item] : (int)item;
    const int ntok = a.item_ntok != nullptr ? a.item_ntok[item] : 1;
    if (tok0 < 0 || r >= ntok * G) return;
    const float* part = a.scratch + ((item * a.Hkv + kvh) * a.nsplit * a.rows_most + r) * (D + 4);
    const size_t step = (size_t)a.rows_most * (D + 4);
    float m_all = -INFINITY;
    for (int s = lane; s < a.nsplit; s += 32) m_all = fmaxf(m_all, part[s * step + D]);
    m_all = warp_max(m_all);
    float v[C], l_all = 0.f;
#pragma unroll
    for (int e = 0; e < C; ++e) v[e] = 0.f;
#pragma unroll 4
    for (int s = 0; s < a.nsplit; ++s) {
        const float2 ml = *reinterpret_cast<const float2*>(part + s * step + D);
        const float f = k8_factor(ml.x, ml.y, m_all);
        l_all = fmaf(ml.y, f, l_all);
#pragma unroll
        for (int e = 0; e < C; ++e) v[e] = fmaf(part[s * step + lane * C + e], f, v[e]);
    }
    if (a.sink && m_all > -INFINITY) l_all += k8_exp2(K8_LIFT - m_all);
    const float inv = l_all == 0.f ? 0.f : 1.f / l_all;
    const int tok = tok0 + r / G, hd = kvh * G + r % G;
#pragma unroll
    for (int e = 0; e < C; ++e) out[((size_t)tok * a.H + hd) * D + lane * C + e] = from_f<T>(k8_gated<T>(v[e] * inv, a, tok, hd));
}

template <typename T, int D, bool PAGE16>
cudaError_t k8_launch(const void* q, const void* pool, const float* scales, void* out, const K8Args& a, cudaStream_t stream) {
    constexpr int smem = (K8_WARPS * K8_ROWS * (D + 4) + 2 * K8_WARPS * K8_ROWS) * 4;
    static_assert(smem <= 48 * 1024, "within what a kernel has without asking");
    return tk_launch(attn_kv8_kernel<T, D, PAGE16>, dim3((unsigned)(a.items * a.Hkv * a.nsplit)), dim3(K8_THREADS), smem, stream, (const T*)q,
                     (const uint8_t*)pool, scales, (T*)out, a);
}

template <typename T>
cudaError_t k8_dispatch(const void* q, const void* pool, const float* scales, void* out, const K8Args& a, int D, cudaStream_t stream) {
    const bool page16 = a.p_shift >= 4;
    cudaError_t e = D == 64 ? (page16 ? k8_launch<T, 64, true>(q, pool, scales, out, a, stream) : k8_launch<T, 64, false>(q, pool, scales, out, a, stream))
                            : (page16 ? k8_launch<T, 128, true>(q, pool, scales, out, a, stream) : k8_launch<T, 128, false>(q, pool, scales, out, a, stream));
    if (e != cudaSuccess || a.nsplit == 1) return e;
    const unsigned grid = (unsigned)(((int64_t)a.items * a.Hkv * a.rows_most + 3) / 4);
    return D == 64 ? tk_launch(attn_kv8_merge_kernel<T, 64>, dim3(grid), dim3(128), 0, stream, (T*)out, a)
                   : tk_launch(attn_kv8_merge_kernel<T, 128>, dim3(grid), dim3(128), 0, stream, (T*)out, a);
}

}  // namespace

// Whether the 8-bit cache's kernels take a layer: heads of 64 or 128, up to 16 query heads a KV head.
TK_API int tk_attn_kv8_supported(int H, int Hkv, int D) {
    return Hkv > 0 && H > 0 && H % Hkv == 0 && H / Hkv <= K8_ROWS && (D == 64 || D == 128);
}

// Tokens of one sequence a tile of tk_attn_kv8 has.
TK_API int tk_attn_kv8_tokens(int H, int Hkv) { return K8_ROWS / (H / Hkv); }

// Ways to share the keys of each of `items` rows' tiles out over CTAs, when no sequence holds more than `longest` positions.
TK_API int tk_attn_kv8_splits(int items, int Hkv, int longest, int sm_count) {
    const int64_t ctas = (int64_t)items * Hkv;
    if (ctas <= 0) return 1;
    const int64_t fill = (4 * (int64_t)sm_count + ctas - 1) / ctas, keys = (longest + 255) / 256;
    const int64_t n = fill < keys ? fill : keys;
    return (int)(n < 1 ? 1 : n > 128 ? 128 : n);
}

// q, out: [T, H, D]; pool: [pages, 2, Hkv, P, D] bytes, scales: [pages, 2, Hkv]. item_tok0 / item_ntok: tiles of at most tk_attn_kv8_tokens tokens of one
// sequence at consecutive positions (0 tokens: skipped); item_ntok null: single tokens' rows (negative: skipped; item_tok0 null too: rows 0, 1, ...).
// window: see first_seen. scratch: items * H * (tokens a tile, or 1) * nsplit * (D + 4) floats when nsplit > 1. gate: [T, >= H], the per-head output gate.
TK_API int tk_attn_kv8(const void* q, const void* pool, const float* scales, void* out, const int* positions, const int* tok_seq,
                       const int* block_table, int bt_stride, const int* item_tok0, const int* item_ntok, int items, int H, int Hkv, int D,
                       int P, int window, float scale, int nsplit, float* scratch, const void* gate, int64_t ldg, int sink, int dtype,
                       cudaStream_t stream) {
    TK_CHECK_ARG(tk_attn_kv8_supported(H, Hkv, D), "attn_kv8: shape H=%d Hkv=%d D=%d is not taken (heads of 64 or 128, up to %d a KV head)", H,
                 Hkv, D, K8_ROWS);
    TK_CHECK_ARG(items >= 0 && P > 0 && nsplit >= 1 && (nsplit == 1 || scratch != nullptr), "attn_kv8: bad sizes");
    TK_CHECK_ARG(item_ntok == nullptr || item_tok0 != nullptr, "attn_kv8: tiles have first tokens");
    TK_CHECK_ARG((int64_t)items * Hkv * nsplit < 0x7fffffff, "attn_kv8: %d splits of %d items", nsplit, items);
    TK_CHECK_ARG(dtype == TK_F32 || dtype == TK_BF16, "attn_kv8: unknown dtype %d", dtype);
    TK_CHECK_ARG((uintptr_t)q % 16 == 0 && (uintptr_t)pool % 16 == 0 && (uintptr_t)out % 16 == 0, "attn_kv8: 16-byte aligned tensors");
    if (items == 0) return 0;
    int shift = -1;
    if ((P & (P - 1)) == 0)
        for (shift = 0; (1 << shift) < P;) ++shift;
    const int G = H / Hkv;
    K8Args a{positions, tok_seq, block_table, item_tok0, item_ntok, gate, scratch, ldg, bt_stride, items, H, Hkv, P, shift, window, nsplit, sink,
             item_ntok != nullptr ? (K8_ROWS / G) * G : G, scale};
    const cudaError_t e = dtype == TK_F32 ? k8_dispatch<float>(q, pool, scales, out, a, D, stream)
                                          : k8_dispatch<__nv_bfloat16>(q, pool, scales, out, a, D, stream);
    if (e != cudaSuccess) {
        tk_set_error("attn_kv8: launch failed: %s", cudaGetErrorString(e));
        cudaGetLastError();
        return -2;
    }
    return 0;
}
