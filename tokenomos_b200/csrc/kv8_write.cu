// One step's queries, keys and values of an attention layer with an 8-bit cache (kv8.cuh): per-head q/k RMSNorm, rotation,
// and the quantised write, in one kernel from the projection's rows.
//
//   y = x / sqrt(mean(x^2) + eps) * w                                 (q and k heads, if the layer has the norms)
//   (u, v) -> (u cos - v sin, v cos + u sin) * cs_mult                (columns i and i + R/2, or 2i and 2i + 1, of the first R)
//   s' = max(s if the block holds earlier tokens, 2^ceil(log2(max|x| / 448)) over the step's tokens of the block)
//   byte = e4m3(x / s');  earlier bytes of the block: e4m3(b * s / s')
//
// All of it in 32 bits and rounded once; the angle position * frequency is formed and reduced as a sum of two 32-bit numbers (at position 32,000 one
// 32-bit product is off by 1e-3).
//
// A block (page, K|V, head) has one writer: the tokens of a sequence that fall into one page within a step form a run, and four warps of one CTA take a
// run's keys and values of one KV head (a block's maximum then needs no atomics, and the bytes do not depend on which warp came first). They hold 16
// tokens in registers (8 for heads of 128) between the maximum and the bytes; a longer run is read again, from L1. Runs begin where the CTAs
// look for them, among `look` tokens in a row each: one of a small step, 4 to 16 of a large one. Queries need no run: CTAs
// of their own take the heads of one token, or of four where there are many. Large steps take CTAs of 8 warps (two KV heads each).
//
// Measured (one B200, 32 heads over 8 of 64): 8 single tokens 3.0 us, a prompt of 2,048 tokens 11.4 (3.5 us of them its bytes' at HBM's rate), three portions of 333 tokens of the
// 32-bit model (16 heads over 8) 5.5. Bound by its chain of dependent loads (tokens, page, rows) at decode sizes, by instructions in long prompts (2.3 of 4 a cycle).
#include <math.h>

#include <algorithm>

#include "kv8.cuh"

namespace {


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

// cos and sin of position * freq, times `mult`: the product as hi + lo exactly, over pi as a_hi + a_lo, whole turns taken off a_hi exactly
__device__ __forceinline__ float2 turn_of(int pos, float freq, float mult) {
    constexpr float INV_PI = 0.318309886f, INV_PI_LO = 1.28412766e-8f;
    const float p = (float)pos, hi = p * freq, lo = fmaf(p, freq, -hi);
    const float a_hi = hi * INV_PI, a_lo = fmaf(hi, INV_PI, -a_hi) + fmaf(hi, INV_PI_LO, lo * INV_PI);
    float s, c;
    sincospif(fmaf(-2.0f, rintf(0.5f * a_hi), a_hi) + a_lo, &s, &c);
    return make_float2(c * mult, s * mult);
}

struct W8Args {
    int H, Hkv, R, P;
    float eps, cs_mult;
    int interleaved, q_ctas, q_tokens, kv_blocks, look;
};

// The norm and rotation of a head that LPH lanes hold, eight columns each (`c`: this lane's first one). `w`: the norm's weights of its columns,
// `turns`: its token's [R / 2] (cos, sin).
template <int LPH>
__device__ __forceinline__ void norm_rotate(float (&x)[8], bool norm, const float (&w)[8], const float2* turns, int c, const W8Args& a) {
    if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float mean = fmaf(ss, 1.0f / (LPH * 8), a.eps);
        float rstd = rsqrtf(mean);
        // a Newton step: to the last bit or two. (Of an infinite mean the root's inverse is 0 and stays so: the step would make NaN of 0 x infinity, and
        // mark a token whose elements are all finite)
        if (rstd != 0.f) rstd = rstd * fmaf(-0.5f * mean * rstd, rstd, 1.5f);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * rstd * w[i];
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
        const bool first = c < half;
        const float4* t4 = reinterpret_cast<const float4*>(turns + (first ? c : c - half));
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float4 t = t4[i >> 1];
            const float p0 = __shfl_xor_sync(0xffffffffu, x[i], LPH / 2), p1 = __shfl_xor_sync(0xffffffffu, x[i + 1], LPH / 2);
            x[i] = fmaf(x[i], t.x, first ? -p0 * t.y : p0 * t.y);
            x[i + 1] = fmaf(x[i + 1], t.z, first ? -p1 * t.w : p1 * t.w);
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

template <typename T, int D, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, WARPS == 8 ? 4 : 1)
qk_norm_rope_write8_kernel(const T* qkv, int64_t qkv_stride, T* q_out, uint8_t* pool, float* scales, const float* __restrict__ wq,
                           const float* __restrict__ wk, const float* __restrict__ freq, const int* positions, const int* tok_seq,
                           const int* block_table, int bt_stride, int T_, const W8Args a) {
    constexpr int THREADS = WARPS * 32, LPH = D / 8, RPW = 32 / LPH;      // lanes of a head row, rows a warp holds at a time
    constexpr int SHARE = 4, CHUNK = SHARE * RPW, HEADS = WARPS / SHARE;  // warps of a KV head, tokens they hold, KV heads of a CTA
    constexpr int HALF = D / 2;                                           // a token's place in the table of angles
    __shared__ __align__(16) float2 turns[CHUNK * HALF];
    __shared__ float2 most_of[WARPS];
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int sub = lane / LPH, c = (lane % LPH) * 8, half = a.R >> 1;
    const bool queries = (int)blockIdx.x >= a.kv_blocks, norm = wq != nullptr;
    float w[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
    if (norm) {                                          // (nobody writes them: asked for while the kernel before ends)
        const float* from = (queries ? wq : wk) + c;
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = from[e];      // (a vector of floats may begin at any of them; 16 bytes at a time is no faster)
    }
    const float f_mine = tid % HALF < half ? freq[tid % HALF] : 0.f;
    pdl_wait();
    // the angles of `count` tokens, a frequency a thread
    auto turns_of = [&](int count, auto pos_of) {
        for (int tt = tid / HALF; tt < count; tt += THREADS / HALF)
            if (tid % HALF < half) turns[tt * HALF + tid % HALF] = turn_of(pos_of(tt), f_mine, a.cs_mult);
    };
    if (queries) {
        // ---- query heads of `q_tokens` tokens, RPW of a token's at a time ----
        const int at = blockIdx.x - a.kv_blocks, t0 = at / a.q_ctas * a.q_tokens, tokens = min(a.q_tokens, T_ - t0), groups = (a.H + RPW - 1) / RPW;
        int tt = 0, hg = at % a.q_ctas * WARPS + warp;
        const int step = a.q_ctas * WARPS;
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        auto next = [&] {
            hg += step;
            while (hg >= groups && tt < tokens) hg -= groups, ++tt;
        };
        auto load = [&](float (&v)[8]) {
            if (tt < tokens && hg * RPW + sub < a.H) load8(qkv + (size_t)(t0 + tt) * qkv_stride + (size_t)(hg * RPW + sub) * D + c, v);
        };
        hg -= step;
        next();
        load(x);                                          // (asked for before the angles are formed)
        turns_of(tokens, [&](int i) { return positions[t0 + i]; });
        __syncthreads();
        while (tt < tokens) {
            const int h = hg * RPW + sub, t = tt;
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = x[e];
            next();
            load(x);
            norm_rotate<LPH>(y, norm, w, turns + t * HALF, c, a);
            if (h < a.H) store8(q_out + ((size_t)(t0 + t) * a.H + h) * D + c, y);
        }
        return;
    }
    // ---- the keys and values of KV head h, four warps, in the runs that begin among `look` tokens ----
    const int kv_ctas = (a.Hkv + HEADS - 1) / HEADS, t_first = blockIdx.x / kv_ctas * a.look;
    const int h_mine = blockIdx.x % kv_ctas * HEADS + warp / SHARE, part = warp % SHARE;
    const bool live = h_mine < a.Hkv;
    const int h = live ? h_mine : 0;
    const size_t v_off = (size_t)a.Hkv * D, v_block = (size_t)a.Hkv * a.P * D;
    // lane i: token t_first - 1 + i, and whether it goes on with the run of the one before
    const int t_mine = t_first - 1 + lane;
    const bool there = t_mine >= 0 && t_mine < T_;
    const int pos_mine = there ? positions[t_mine] : 0, seq_mine = there ? tok_seq[t_mine] : -1, off_mine = pos_mine % a.P;
    const int pos_prev = __shfl_up_sync(0xffffffffu, pos_mine, 1), seq_prev = __shfl_up_sync(0xffffffffu, seq_mine, 1);
    const uint32_t on = __ballot_sync(0xffffffffu, there && lane > 0 && seq_mine == seq_prev && pos_mine == pos_prev + 1 && off_mine > 0);
    for (int j = 1; j <= a.look && t_first + j - 1 < T_; ++j) {
        if (on >> j & 1) continue;
        const int t = t_first + j - 1;
        const int pos = __shfl_sync(0xffffffffu, pos_mine, j), seq = __shfl_sync(0xffffffffu, seq_mine, j), off = pos % a.P;
        if (pos < 0) continue;                            // (no position: nothing is written)
        int n = j < 31 ? __ffs(~(on >> (j + 1))) : 1;     // the run's tokens, as far as these lanes reach
        for (bool more = j + n == 32; more;) {
            const int i = n + lane;
            const bool mine = off + i < a.P && t + i < T_ && tok_seq[t + i] == seq && positions[t + i] == pos + i;
            const uint32_t vote = __ballot_sync(0xffffffffu, mine);
            more = vote == 0xffffffffu;
            n += more ? 32 : __ffs(~vote) - 1;
        }
        const T* krow = qkv + (size_t)t * qkv_stride + (size_t)(a.H + h) * D + c;
        float k[8], v[8];
        bool bad = false;
        // token i of the run (one a group of LPH lanes): key and value as they are to be cached
        auto load = [&](int first, int i) {
            const T* row = krow + (size_t)(i < n ? i : 0) * qkv_stride;
            load8(row, k);
            load8(row + v_off, v);
            __syncthreads();                              // (what the angles before were for is done)
            turns_of(min(CHUNK, n - first), [&](int tt) { return pos + first + tt; });
            __syncthreads();
            norm_rotate<LPH>(k, norm, w, turns + (i - first) * HALF, c, a);
            bool fine = true;
#pragma unroll
            for (int e = 0; e < 8; ++e) fine = fine && fabsf(k[e]) <= KV8_MOST && fabsf(v[e]) <= KV8_MOST;
            const uint32_t group = (LPH == 32 ? 0xffffffffu : ((1u << LPH) - 1)) << (sub * LPH);
            bad = (__ballot_sync(0xffffffffu, !fine) & group) != 0;
        };
        const int page = TK_PAGE(TK_K_KV8_WRITE, block_table[(size_t)seq * bt_stride + pos / a.P]);
        float* scale = scales + (size_t)page * 2 * a.Hkv + h;
        uint8_t* block = pool + ((size_t)page * 2 * a.Hkv + h) * a.P * D;
        float old_k = 0.f, old_v = 0.f;
        if (off > 0) old_k = scale[0], old_v = scale[a.Hkv];
        // the largest magnitudes
        float most_k = 0.f, most_v = 0.f;
        for (int first = 0; first < n; first += CHUNK) {
            const int i = first + part * RPW + sub;
            load(first, i);
            if (i < n && !bad) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    most_k = fmaxf(most_k, fabsf(k[e]));
                    most_v = fmaxf(most_v, fabsf(v[e]));
                }
            }
        }
        most_k = warp_max(most_k);
        most_v = warp_max(most_v);
        if (lane == 0) most_of[warp] = make_float2(most_k, most_v);
        __syncthreads();                                  // (and every thread has read the old scales)
#pragma unroll
        for (int p = 0; p < SHARE; ++p) {
            const float2 m = most_of[warp - part + p];
            most_k = fmaxf(most_k, m.x);
            most_v = fmaxf(most_v, m.y);
        }
        float s_k = exp2i(kv8_exponent(most_k)), s_v = exp2i(kv8_exponent(most_v));
        if (off > 0) {
            // the block holds earlier tokens: its scale only grows, and then their bytes follow
            s_k = fmaxf(s_k, old_k);
            s_v = fmaxf(s_v, old_v);
            for (int which = 0; which < 2; ++which) {
                const float ratio = which ? old_v / s_v : old_k / s_k;
                if (ratio == 1.0f || !live) continue;
                uint4* bytes = reinterpret_cast<uint4*>(block + which * v_block);
                for (int i = part * 32 + lane; i < off * D / 16; i += SHARE * 32) {
                    uint4 raw = bytes[i];
                    uint32_t* b = &raw.x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t lo = e4m3x2_to_half2((uint16_t)b[e]), hi = e4m3x2_to_half2((uint16_t)(b[e] >> 16));
                        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&lo));
                        const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                        b[e] = to_e4m3x2(x.x * ratio, x.y * ratio) | ((uint32_t)to_e4m3x2(y.x * ratio, y.y * ratio) << 16);
                    }
                    bytes[i] = raw;
                }
            }
        }
        if (live && part == 0 && lane == 0) {
            scale[0] = s_k;
            scale[a.Hkv] = s_v;
        }
        // the bytes
        const float inv_k = 1.0f / s_k, inv_v = 1.0f / s_v;      // (powers of two: exact)
        for (int first = 0; first < n; first += CHUNK) {
            const int i = first + part * RPW + sub;
            if (n > CHUNK) load(first, i);
            if (i >= n || !live) continue;
            uint32_t kb[2], vb[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                kb[e] = to_e4m3x2(k[4 * e] * inv_k, k[4 * e + 1] * inv_k) | ((uint32_t)to_e4m3x2(k[4 * e + 2] * inv_k, k[4 * e + 3] * inv_k) << 16);
                vb[e] = to_e4m3x2(v[4 * e] * inv_v, v[4 * e + 1] * inv_v) | ((uint32_t)to_e4m3x2(v[4 * e + 2] * inv_v, v[4 * e + 3] * inv_v) << 16);
                if (bad) kb[e] = 0x7f7f7f7fu, vb[e] = 0u;
            }
            uint8_t* dst = block + (size_t)(off + i) * D + c;
            *reinterpret_cast<uint2*>(dst) = make_uint2(kb[0], kb[1]);
            *reinterpret_cast<uint2*>(dst + v_block) = make_uint2(vb[0], vb[1]);
        }
    }
}

}  // namespace

// qkv: [T, (H + 2 Hkv) D] with row stride `qkv_stride`, 16-byte aligned rows; pool: [pages, 2, Hkv, P, D] bytes, scales: [pages, 2, Hkv]. wq / wk:
// both or neither, D floats at any float's address. Hkv 0: queries only (no pool, scales, tables nor wk). freq: [R / 2]. The tokens of a sequence lie side by side in the step, at consecutive positions.
TK_API int tk_qk_norm_rope_write8(const void* qkv, int64_t qkv_stride, void* q_out, void* pool, float* scales, const float* wq,
                                  const float* wk, float eps, const float* freq, float cs_mult, int interleaved, const int* positions,
                                  const int* tok_seq, const int* block_table, int bt_stride, int T_, int H, int Hkv, int D, int R, int P,
                                  int dtype, cudaStream_t stream) {
    TK_CHECK_ARG(T_ >= 0 && H > 0 && Hkv >= 0 && P > 0 && bt_stride >= 0, "qk_norm_rope_write8: bad sizes");
    TK_CHECK_ARG(D == 64 || D == 128, "qk_norm_rope_write8: heads of %d (64 and 128 are built)", D);
    TK_CHECK_ARG(R >= 0 && R <= D && R % 2 == 0, "qk_norm_rope_write8: rotary width %d of head %d", R, D);
    TK_CHECK_ARG(Hkv == 0 || (wq == nullptr) == (wk == nullptr), "qk_norm_rope_write8: q and k norms come together");
    TK_CHECK_ARG(dtype == TK_F32 || dtype == TK_BF16, "qk_norm_rope_write8: unknown dtype %d", dtype);
    const int vec = dtype == TK_F32 ? 4 : 8;
    TK_CHECK_ARG(qkv_stride % vec == 0 && (uintptr_t)qkv % 16 == 0 && (uintptr_t)q_out % 16 == 0 && (uintptr_t)pool % 16 == 0,
                 "qk_norm_rope_write8: rows are read 16 bytes at a time: 16-byte aligned, whole 16 bytes apart");
    if (T_ == 0) return 0;
    // (a prompt of 2,048 tokens, 32 heads over 8 of 64, us by warps a CTA: 15.7 with 4, 13.2 with 8, 13.9 with 16; three portions of 333 of the 32-bit
    // model 6.9, 6.1, 6.8; eight single tokens 3.0 with 4)
    const bool many = T_ >= 512;
    // Of a large step's keys and values a CTA takes as many tokens as leave about four CTAs an SM, but 4 at least (a step of single tokens has a run each) and 16 at
    // most (a page; us with 4 tokens, 16, and so: the prompt of 2,048 13.3, 10.8, 11.4; 8,192 49.9, 41.0, 41.0; three portions of 333 6.2, 6.8, 5.4; 600 single tokens 18.7,
    // 38.7, 16.8).
    const int warps = many ? 8 : 4, q_tokens = many ? 4 : 1;
    const int look = many ? (int)std::clamp<int64_t>((int64_t)T_ * ceil_div(Hkv, warps / 4) / (4 * 148) + 1, 4, 16) : 1;
    const int q_ctas = many ? 1 : ceil_div(H, warps * 32 / (D / 8));
    const int64_t kv_blocks = (int64_t)ceil_div(T_, look) * ceil_div(Hkv, warps / 4), blocks = kv_blocks + (int64_t)ceil_div(T_, q_tokens) * q_ctas;
    TK_CHECK_ARG(blocks < 0x7fffffff, "qk_norm_rope_write8: %d tokens are too many", T_);
    const W8Args a{H, Hkv, R, P, eps, cs_mult, interleaved, q_ctas, q_tokens, (int)kv_blocks, look};
#define TK_W8(T, DD, WARPS)                                                                                                                       \
    tk_launch(qk_norm_rope_write8_kernel<T, DD, WARPS>, dim3((unsigned)blocks), dim3(WARPS * 32), 0, stream, (const T*)qkv, qkv_stride, (T*)q_out, \
              (uint8_t*)pool, scales, wq, wk, freq, positions, tok_seq, block_table, bt_stride, T_, a)
#define TK_W8_STEP(T, DD)               \
    do {                                \
        if (many) TK_W8(T, DD, 8);     \
        else TK_W8(T, DD, 4);           \
    } while (0)
    if (dtype == TK_F32) {
        if (D == 64) TK_W8_STEP(float, 64);
        else TK_W8_STEP(float, 128);
    } else {
        if (D == 64) TK_W8_STEP(__nv_bfloat16, 64);
        else TK_W8_STEP(__nv_bfloat16, 128);
    }
#undef TK_W8_STEP
#undef TK_W8
    TK_CHECK_LAUNCH("qk_norm_rope_write8");
    return 0;
}
