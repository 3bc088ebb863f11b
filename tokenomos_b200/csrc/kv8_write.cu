// One step's queries, keys and values of an attention layer with an 8-bit cache (kv8.cuh): per-head q/k RMSNorm, rotation,
// and the quantised write, in one kernel from the projection's rows.
//
//   y = x / sqrt(mean(x^2) + eps) * w                                 (q and k heads, if the layer has the norms)
//   (u, v) -> (u cos - v sin, v cos + u sin) * cs_mult                (columns i and i + R/2, or 2i and 2i + 1, of the first R)
//   s' = max(s if the block holds earlier tokens, 2^ceil(log2(max|x| / 448)) over the step's tokens of the block)
//   byte = e4m3(x / s');  earlier bytes of the block: e4m3(b * s / s')
//
// All of it in 32 bits and rounded once; the angle position * frequency is formed and reduced in 64 bits, since at position
// 32,000 its 32-bit product is off by 1e-3.
//
// A block (page, K|V, head) has one writer: the tokens of a sequence that fall into one page within a step form a run, and the run's first
// token's warp takes all of it, head by head (a block's maximum then needs no atomics, and the bytes do not depend on
// which warp came first). It walks the run twice, for the maximum and for the bytes, the second time from L1. A token that
// follows another one of its run has no keys and values to write: its CTAs for those leave at once. Queries need no run:
// grid.y's first CTAs take a token's query heads, the others its KV heads, a warp each.
//
// Bound by its chain of loads at decode sizes and by HBM for prompts; measured figures stand with the entry point.
#include <math.h>

#include "kv8.cuh"

namespace {

constexpr int W8_THREADS = 128, W8_WARPS = W8_THREADS / 32;
constexpr int W8_CHUNK = 16;                 // tokens whose cos and sin are in shared memory at a time

// eight neighbouring elements as 32-bit values
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]);
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&v)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
template <>
__device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float (&v)[8]) {
    uint4 raw;
    uint32_t* w = &raw.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 two = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&two);
    }
    *reinterpret_cast<uint4*>(p) = raw;
}

// cos and sin of position * freq, times `mult`
__device__ __forceinline__ float2 turn_of(int pos, float freq, float mult) {
    const double a = (double)pos * (double)freq;
    const double k = rint(a * 0.15915494309189535);
    const float r = (float)fma(-k, 2.4492935982947064e-16, fma(-k, 6.283185307179586, a));
    float s, c;
    sincosf(r, &s, &c);
    return make_float2(c * mult, s * mult);
}

struct W8Args {
    int H, Hkv, R, P;
    float eps, cs_mult;
    int interleaved, q_ctas;
};

// The norm and rotation of a head that LPH lanes hold, eight columns each (`c`: this lane's first one). `turns`: its
// token's [R / 2] (cos, sin).
template <int LPH>
__device__ __forceinline__ void norm_rotate(float (&x)[8], const float* __restrict__ w, const float2* turns, int c, const W8Args& a) {
    if (w != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float rstd = 1.0f / sqrtf(ss / (float)(LPH * 8) + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * rstd * w[c + i];
    }
    const int half = a.R >> 1;
    if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            if (c + i < a.R) {
                const float2 t = turns[(c + i) >> 1];
                const float u = x[i], v = x[i + 1];
                x[i] = u * t.x - v * t.y;
                x[i + 1] = v * t.x + u * t.y;
            }
        }
        return;
    }
    if (half == LPH * 4) {            // the whole head turns: a column's partner lies half the lanes away
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = __shfl_xor_sync(0xffffffffu, x[i], LPH / 2);
        const bool first = c < half;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 t = turns[first ? c + i : c + i - half];
            x[i] = first ? x[i] * t.x - p[i] * t.y : x[i] * t.x + p[i] * t.y;
        }
        return;
    }
    // part of the head, of any even width: column by column from the lane that holds the partner
    const int lane = threadIdx.x & 31, row0 = lane & ~(LPH - 1);
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int col = c + i, mate = col < half ? col + half : (col < a.R ? col - half : col);
        // (every lane asks for one register of one lane: eight exchanges pick the one that is meant)
        float got = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float y = __shfl_sync(0xffffffffu, x[k], row0 + (mate >> 3));
            if ((mate & 7) == k) got = y;
        }
        p[i] = got;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int col = c + i;
        if (col < a.R) {
            const float2 t = turns[col < half ? col : col - half];
            x[i] = col < half ? x[i] * t.x - p[i] * t.y : x[i] * t.x + p[i] * t.y;
        }
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(W8_THREADS)
qk_norm_rope_write8_kernel(const T* qkv, int64_t qkv_stride, T* q_out, uint8_t* pool, float* scales, const float* __restrict__ wq,
                           const float* __restrict__ wk, const float* __restrict__ freq, const int* positions, const int* tok_seq,
                           const int* block_table, int bt_stride, int T_, const W8Args a) {
    constexpr int LPH = D / 8, RPW = 32 / LPH;           // lanes of a head row, rows a warp holds at a time
    __shared__ float2 turns[W8_CHUNK * D / 2];
    pdl_launch_dependents();
    pdl_wait();
    const int t = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int sub = lane / LPH, c = (lane % LPH) * 8, half = a.R >> 1;
    const int pos = positions[t];
    if ((int)blockIdx.y < a.q_ctas) {
        // ---- the query heads of token t ----
        const T* row = qkv + (size_t)t * qkv_stride;
        const int h0 = (blockIdx.y * W8_WARPS + warp) * RPW + sub, step = a.q_ctas * W8_WARPS * RPW;
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (h0 < a.H) load8(row + (size_t)h0 * D + c, x);             // (asked for before the angles are formed)
        for (int i = tid; i < half; i += W8_THREADS) turns[i] = turn_of(pos, freq[i], a.cs_mult);
        __syncthreads();
        for (int h = h0; h - sub < a.H; h += step) {
            if (h != h0 && h < a.H) load8(row + (size_t)h * D + c, x);
            norm_rotate<LPH>(x, wq, turns, c, a);
            if (h < a.H) store8(q_out + ((size_t)t * a.H + h) * D + c, x);
        }
        return;
    }
    // ---- the keys and values of the run that begins with token t, if one does ----
    const int seq = tok_seq[t], off = pos % a.P;
    if (t > 0 && off > 0 && tok_seq[t - 1] == seq && positions[t - 1] == pos - 1) return;
    int n = 1;                                            // the run's tokens
    for (bool more = true; more;) {
        const int i = n + lane;
        const bool mine = off + i < a.P && t + i < T_ && tok_seq[t + i] == seq && positions[t + i] == pos + i;
        const uint32_t vote = __ballot_sync(0xffffffffu, mine);
        more = vote == 0xffffffffu;
        n += more ? 32 : __ffs(~vote) - 1;
    }
    const int page = TK_PAGE(TK_K_KV8_WRITE, block_table[(size_t)seq * bt_stride + pos / a.P]);
    const int h = (blockIdx.y - a.q_ctas) * W8_WARPS + warp;
    const bool live = h < a.Hkv;
    const T* krow = qkv + (size_t)t * qkv_stride + (size_t)(a.H + (live ? h : 0)) * D + c;
    const size_t v_off = (size_t)a.Hkv * D;
    float k[8], v[8];
    bool bad = false;
    // rows i of the run (one a group of LPH lanes): key and value as they are to be cached
    auto load = [&](int first, int i) {
        const bool there = i < n;
        const T* p = krow + (size_t)(there ? i : 0) * qkv_stride;
        load8(p, k);
        load8(p + v_off, v);
        norm_rotate<LPH>(k, wk, turns + (i - first) * half, c, a);
        bool fine = true;
#pragma unroll
        for (int e = 0; e < 8; ++e) fine = fine && fabsf(k[e]) <= KV8_MOST && fabsf(v[e]) <= KV8_MOST;
        const uint32_t group = (LPH == 32 ? 0xffffffffu : ((1u << LPH) - 1)) << (sub * LPH);
        bad = (__ballot_sync(0xffffffffu, !fine) & group) != 0;
    };
    auto turns_of = [&](int first) {
        __syncthreads();
        for (int i = tid; i < W8_CHUNK * half; i += W8_THREADS)
            if (first + i / half < n) turns[i] = turn_of(pos + first + i / half, freq[i % half], a.cs_mult);
        __syncthreads();
    };
    // first pass: the largest magnitudes
    float most_k = 0.f, most_v = 0.f;
    for (int first = 0; first < n; first += W8_CHUNK) {
        turns_of(first);
        for (int i = first; i < min(n, first + W8_CHUNK); i += RPW) {
            load(first, i + sub);
            if (i + sub < n && !bad) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    most_k = fmaxf(most_k, fabsf(k[e]));
                    most_v = fmaxf(most_v, fabsf(v[e]));
                }
            }
        }
    }
    most_k = warp_max(most_k);
    most_v = warp_max(most_v);
    float* scale = scales + (size_t)page * 2 * a.Hkv + (live ? h : 0);
    uint8_t* block = pool + ((size_t)page * 2 * a.Hkv + (live ? h : 0)) * a.P * D;
    const size_t v_block = (size_t)a.Hkv * a.P * D;
    float s_k = exp2i(kv8_exponent(most_k)), s_v = exp2i(kv8_exponent(most_v));
    if (off > 0) {
        // the block holds earlier tokens: its scale only grows, and then their bytes follow
        const float old_k = scale[0], old_v = scale[a.Hkv];
        __syncwarp();
        s_k = fmaxf(s_k, old_k);
        s_v = fmaxf(s_v, old_v);
        for (int which = 0; which < 2; ++which) {
            const float ratio = which ? old_v / s_v : old_k / s_k;
            if (ratio == 1.0f || !live) continue;
            uint4* bytes = reinterpret_cast<uint4*>(block + which * v_block);
            for (int i = lane; i < off * D / 16; i += 32) {
                uint4 raw = bytes[i];
                uint32_t* w = &raw.x;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t lo = e4m3x2_to_half2((uint16_t)w[e]), hi = e4m3x2_to_half2((uint16_t)(w[e] >> 16));
                    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&lo));
                    const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                    w[e] = to_e4m3x2(x.x * ratio, x.y * ratio) | ((uint32_t)to_e4m3x2(y.x * ratio, y.y * ratio) << 16);
                }
                bytes[i] = raw;
            }
        }
    }
    if (live && lane == 0) {
        scale[0] = s_k;
        scale[a.Hkv] = s_v;
    }
    // second pass: the bytes (a run that the warp holds at once is in registers still)
    const float inv_k = 1.0f / s_k, inv_v = 1.0f / s_v;      // (powers of two: exact)
    for (int first = 0; first < n; first += W8_CHUNK) {
        if (n > W8_CHUNK) turns_of(first);
        for (int i = first; i < min(n, first + W8_CHUNK); i += RPW) {
            if (n > RPW) load(first, i + sub);
            if (i + sub >= n || !live) continue;
            uint32_t kb[2], vb[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                kb[e] = to_e4m3x2(k[4 * e] * inv_k, k[4 * e + 1] * inv_k) | ((uint32_t)to_e4m3x2(k[4 * e + 2] * inv_k, k[4 * e + 3] * inv_k) << 16);
                vb[e] = to_e4m3x2(v[4 * e] * inv_v, v[4 * e + 1] * inv_v) | ((uint32_t)to_e4m3x2(v[4 * e + 2] * inv_v, v[4 * e + 3] * inv_v) << 16);
                if (bad) kb[e] = 0x7f7f7f7fu, vb[e] = 0u;
            }
            uint8_t* at = block + (size_t)(off + i + sub) * D + c;
            *reinterpret_cast<uint2*>(at) = make_uint2(kb[0], kb[1]);
            *reinterpret_cast<uint2*>(at + v_block) = make_uint2(vb[0], vb[1]);
        }
    }
}

}  // namespace

// qkv: [T, (H + 2 Hkv) D] with row stride `qkv_stride`, 16-byte aligned rows; pool: [pages, 2, Hkv, P, D] bytes, scales: [pages, 2, Hkv]. wq / wk:
// both or neither. freq: [R / 2]. The tokens of a sequence lie side by side in the step, at consecutive positions.
TK_API int tk_qk_norm_rope_write8(const void* qkv, int64_t qkv_stride, void* q_out, void* pool, float* scales, const float* wq,
                                  const float* wk, float eps, const float* freq, float cs_mult, int interleaved, const int* positions,
                                  const int* tok_seq, const int* block_table, int bt_stride, int T_, int H, int Hkv, int D, int R, int P,
                                  int dtype, cudaStream_t stream) {
    TK_CHECK_ARG(T_ >= 0 && H > 0 && Hkv > 0 && P > 0 && bt_stride >= 0, "qk_norm_rope_write8: bad sizes");
    TK_CHECK_ARG(D == 64 || D == 128, "qk_norm_rope_write8: heads of %d (64 and 128 are built)", D);
    TK_CHECK_ARG(R >= 0 && R <= D && R % 2 == 0, "qk_norm_rope_write8: rotary width %d of head %d", R, D);
    TK_CHECK_ARG((wq == nullptr) == (wk == nullptr), "qk_norm_rope_write8: q and k norms come together");
    TK_CHECK_ARG(dtype == TK_F32 || dtype == TK_BF16, "qk_norm_rope_write8: unknown dtype %d", dtype);
    const int vec = dtype == TK_F32 ? 4 : 8;
    TK_CHECK_ARG(qkv_stride % vec == 0 && (uintptr_t)qkv % 16 == 0 && (uintptr_t)q_out % 16 == 0 && (uintptr_t)pool % 16 == 0,
                 "qk_norm_rope_write8: rows are read 16 bytes at a time: 16-byte aligned, whole 16 bytes apart");
    if (T_ == 0) return 0;
    // few tokens: the query heads spread over CTAs, a pass each; many: one CTA takes a token's and forms its angles once
    const int per_pass = W8_WARPS * 32 / (D / 8);
    W8Args a{H, Hkv, R, P, eps, cs_mult, interleaved, T_ >= 512 ? 1 : ceil_div(H, per_pass)};
    const dim3 grid(T_, a.q_ctas + ceil_div(Hkv, W8_WARPS));
#define TK_W8(T, DD)                                                                                                                 \
    tk_launch(qk_norm_rope_write8_kernel<T, DD>, grid, dim3(W8_THREADS), 0, stream, (const T*)qkv, qkv_stride, (T*)q_out, (uint8_t*)pool, \
              scales, wq, wk, freq, positions, tok_seq, block_table, bt_stride, T_, a)
    if (dtype == TK_F32) {
        if (D == 64) TK_W8(float, 64);
        else TK_W8(float, 128);
    } else {
        if (D == 64) TK_W8(__nv_bfloat16, 64);
        else TK_W8(__nv_bfloat16, 128);
    }
#undef TK_W8
    TK_CHECK_LAUNCH("qk_norm_rope_write8");
    return 0;
}
