// What the kernels of attention over the 8-bit cache share: their arguments, bounded waits, the per-head gate, and the joining of the shares of
// a row's keys that several CTAs have seen.
#pragma once

#include <atomic>

#include "kv8.cuh"

namespace {

constexpr float K8_LOG2E = 1.4426950408889634f;
constexpr long long K8_WAIT_CYCLES = 2000000000LL;

__device__ __forceinline__ float2 half2_floats(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }

__device__ __forceinline__ float k8_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

static __device__ int g_k8_error = 0;                       // (each file that includes this has its own)

// Whether the barrier's phase completed; a wait ends after about a second, or once another thread has given up.
__device__ __forceinline__ bool k8_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
__device__ __forceinline__ bool k8_wait(uint32_t bar, uint32_t parity) {
    if (k8_try(bar, parity)) return true;
    const long long start = clock64();
    int it = 0;
    while (!k8_try(bar, parity)) {
        if ((++it & 255) == 0) {
            if (*(volatile int*)&g_k8_error != 0) return false;
            if (clock64() - start > K8_WAIT_CYCLES) {
                atomicCAS(&g_k8_error, 0, 1);
                return false;
            }
        }
    }
    return true;
}

// 0, or 1 if a wait of this file's kernels gave up since the last call; -1: the word could not be read
inline int k8_take_status() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_k8_error, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) cudaMemcpyToSymbol(g_k8_error, &zero, sizeof(int));
    return v;
}

// Dynamic shared memory (and clusters of more than eight CTAs) that a kernel may have, asked for once a device: `done` holds a bit a device.
template <typename K>
inline cudaError_t k8_allow(K kernel, int smem, bool wide, std::atomic<uint64_t>& done) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess || (device < 64 && done.load(std::memory_order_relaxed) >> device & 1)) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess && wide) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && device < 64) done.fetch_or(1ull << device, std::memory_order_relaxed);
    return e;
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

// The per-head output gate, round(sigmoid(gate)), of a row's output, round(o) * gate.
template <typename T>
__device__ __forceinline__ float k8_gate(const K8Args& a, int tok, int head) {
    if (a.gate == nullptr) return 1.f;
    const float g = to_f<T>(reinterpret_cast<const T*>(a.gate)[(size_t)tok * a.ldg + head]);
    return round_as<T>(1.0f / (1.0f + expf(-g)));
}
template <typename T>
__device__ __forceinline__ float k8_apply(float o, const K8Args& a, float gate) {
    return a.gate == nullptr ? o : round_as<T>(o) * gate;
}

// The share of a row's keys that one CTA or warp has seen, under reference m: o = sum w v, l = sum w / s_V.
__device__ __forceinline__ float k8_factor(float m, float l, float m_all) {
    // (nothing seen: left out; a sum that is not a number under no maximum: every score was one)
    return m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : k8_exp2(m - m_all);
}

// The CTAs' shares of a row joined: a warp a row, D / 32 columns a lane.
template <typename T, int D>
__global__ void __launch_bounds__(128)
attn_kv8_merge_kernel(T* out, const K8Args a, float lift) {
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
    if (tok0 < 0 || r >= ntok * G) return;               // (r is below a tile's most rows)
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
    if (a.sink && m_all > -INFINITY) l_all += k8_exp2(lift - m_all);
    const float inv = l_all == 0.f ? 0.f : 1.f / l_all;
    const int tok = tok0 + r / G, hd = kvh * G + r % G;
    const float gate = k8_gate<T>(a, tok, hd);
#pragma unroll
    for (int e = 0; e < C; ++e) out[((size_t)tok * a.H + hd) * D + lane * C + e] = from_f<T>(k8_apply<T>(v[e] * inv, a, gate));
}

}  // namespace
