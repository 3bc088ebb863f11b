// Rows (pages of a cache, state rows of requests) of several tensors copied to other rows of the same tensors, in one launch:
// what forking a request's cache takes. dst[i] <- src[i] in every tensor; no row is a destination twice, and none is both a
// source and a destination, so the copies need no order.
//
// Tensors and pairs travel in the launch's own arguments: no upload, no buffer that a later call would have to wait for, and a
// recorded launch keeps what it was recorded with. Bound by HBM (each byte read and written once) or, for a few pages, by
// the launch; a CTA moves 16 KB, four 16-byte loads of a thread in flight. Measured (one B200): a page of six layers (8 KV heads of 64, 16 positions, 8 bits)
// 1.95 us, 512 pages of six layers in 16 bits 33.1 us (201 MB moved: 6.1 TB/s).
#include <algorithm>
#include <memory>
#include <new>

#include "common.cuh"

namespace {

constexpr int CR_THREADS = 256, CR_CHUNK = CR_THREADS * 64;

struct CrTensor {
    unsigned char* base;
    int64_t row;               // bytes
    int chunk0, width;         // first of its chunks among a pair's; bytes an access
};

template <int TENSORS, int PAIRS>
struct CrArgs {
    CrTensor tensor[TENSORS];
    int2 pair[PAIRS];
    int tensors, chunks;
};

template <typename V>
__device__ __forceinline__ void copy_part(unsigned char* to, const unsigned char* from, int64_t bytes) {
    const V* a = reinterpret_cast<const V*>(from);
    V* b = reinterpret_cast<V*>(to);
    const int n = (int)(bytes / sizeof(V));
    int i = threadIdx.x;
    for (; i + 3 * CR_THREADS < n; i += 4 * CR_THREADS) {
        V v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = a[i + u * CR_THREADS];
#pragma unroll
        for (int u = 0; u < 4; ++u) b[i + u * CR_THREADS] = v[u];
    }
    for (; i < n; i += CR_THREADS) b[i] = a[i];
}

template <int TENSORS, int PAIRS>
__global__ void __launch_bounds__(CR_THREADS) copy_rows_kernel(const __grid_constant__ CrArgs<TENSORS, PAIRS> a) {
    pdl_launch_dependents();
    pdl_wait();
    const int pair = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    int k = 0;
    while (k + 1 < a.tensors && a.tensor[k + 1].chunk0 <= chunk) ++k;
    const int64_t row = a.tensor[k].row, at = (int64_t)(chunk - a.tensor[k].chunk0) * CR_CHUNK;
    const int64_t bytes = row - at < CR_CHUNK ? row - at : CR_CHUNK;
    const int2 p = a.pair[pair];
    const unsigned char* from = a.tensor[k].base + (int64_t)p.x * row + at;
    unsigned char* to = a.tensor[k].base + (int64_t)p.y * row + at;
    if (a.tensor[k].width == 16) copy_part<uint4>(to, from, bytes);
    else if (a.tensor[k].width == 4) copy_part<uint32_t>(to, from, bytes);
    else copy_part<unsigned char>(to, from, bytes);
}

template <int TENSORS, int PAIRS>
int copy_some(void* const* base, const int64_t* row, int tensors, const int* src, const int* dst, int pairs, cudaStream_t stream) {
    for (int t0 = 0; t0 < tensors; t0 += TENSORS) {
        CrArgs<TENSORS, PAIRS> a;
        a.tensors = std::min(TENSORS, tensors - t0);
        int64_t chunks = 0;
        for (int k = 0; k < a.tensors; ++k) {
            const uintptr_t p = (uintptr_t)base[t0 + k];
            const int64_t r = row[t0 + k];
            a.tensor[k] = CrTensor{(unsigned char*)p, r, (int)chunks, (p | r) % 16 == 0 ? 16 : (p | r) % 4 == 0 ? 4 : 1};
            chunks += (r + CR_CHUNK - 1) / CR_CHUNK;
            TK_CHECK_ARG(chunks * PAIRS < 0x7fffffff, "copy_rows: rows of %lld bytes are too long", (long long)r);
        }
        a.chunks = (int)chunks;
        for (int i = 0; i < pairs; i += PAIRS) {
            const int n = std::min(PAIRS, pairs - i);
            for (int j = 0; j < n; ++j) a.pair[j] = make_int2(src[i + j], dst[i + j]);
            tk_launch(copy_rows_kernel<TENSORS, PAIRS>, dim3((unsigned)(n * a.chunks)), dim3(CR_THREADS), 0, stream, a);
            TK_CHECK_LAUNCH("copy_rows");
        }
    }
    return 0;
}

}  // namespace

// base, row, rows: host arrays, one entry a tensor (its first byte, its rows' bytes, how many rows it has); src, dst: host arrays of row numbers.
TK_API int tk_copy_rows(void* const* base, const int64_t* row, const int* rows, int tensors, const int* src, const int* dst, int pairs,
                        cudaStream_t stream) {
    TK_CHECK_ARG(tensors >= 0 && pairs >= 0, "copy_rows: bad sizes");
    if (tensors == 0 || pairs == 0) return 0;
    int least = 0x7fffffff;
    for (int k = 0; k < tensors; ++k) {
        TK_CHECK_ARG(base[k] != nullptr && row[k] > 0, "copy_rows: tensor %d has no rows", k);
        least = std::min(least, rows[k]);
    }
    for (int i = 0; i < pairs; ++i)
        TK_CHECK_ARG(src[i] >= 0 && src[i] < least && dst[i] >= 0 && dst[i] < least, "copy_rows: row %d to %d, outside 0..%d", src[i],
                     dst[i], least - 1);
    // no destination twice, none that is a source: a bit a row (a few pairs are compared with each other)
    int twice = -1, both = -1;
    if (pairs <= 16) {
        for (int i = 0; i < pairs; ++i)
            for (int j = 0; j < pairs; ++j) {
                if (j < i && dst[i] == dst[j]) twice = dst[i];
                if (src[i] == dst[j]) both = src[i];
            }
    } else {
        std::unique_ptr<uint64_t[]> seen(new (std::nothrow) uint64_t[(size_t)least / 64 + 1]());
        if (!seen) {
            tk_set_error("copy_rows: no memory to check %d pairs", pairs);
            return -3;
        }
        for (int i = 0; i < pairs; ++i) {
            if (seen[dst[i] >> 6] >> (dst[i] & 63) & 1) twice = dst[i];
            seen[dst[i] >> 6] |= 1ull << (dst[i] & 63);
        }
        for (int i = 0; i < pairs; ++i)
            if (seen[src[i] >> 6] >> (src[i] & 63) & 1) both = src[i];
    }
    TK_CHECK_ARG(twice < 0, "copy_rows: row %d is a destination twice", twice);
    TK_CHECK_ARG(both < 0, "copy_rows: row %d is both a source and a destination", both);
    if (pairs <= 16) return copy_some<32, 16>(base, row, tensors, src, dst, pairs, stream);
    return copy_some<32, 1024>(base, row, tensors, src, dst, pairs, stream);
}
