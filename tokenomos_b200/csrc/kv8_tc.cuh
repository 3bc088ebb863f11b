// What the tcgen05 kernels of the 8-bit cache share: descriptors of 8-bit tiles, the product of two, the tensor map of a cache, launch attributes.
#pragma once

#include "kv8.cuh"
#include "tcgen05.cuh"

namespace {

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

// the cache as rows of D bytes, boxes of `box_rows` positions of a page; its extent is not known here, and no row is asked for but those of pages that
// block_table names
inline bool k8_map(CUtensorMap* map, const void* pool, int D, int box_rows) {
    EncodeTiled fn = encode_fn();
    if (fn == nullptr) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)D, 0x7fffffffu};
    const cuuint64_t strides[1] = {(cuuint64_t)D};
    const cuuint32_t box[2] = {(cuuint32_t)D, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(pool), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How many clusters of n CTAs are resident at once where an SM holds per_sm of them, two or more. Pairs fill the device; larger clusters leave places empty, by measurement (148 SMs; the time of a
// launch jumps by half where one cluster more has to wait): with two CTAs an SM 92 clusters of 3 run together, 70 of 4, 56 of 5, 45 of 6, 37 of 7, 33 of 8, 14 of 16; with four 185, 140, 112, 92, 76, 66
// and 28. (The occupancy calculator cannot be asked: it answers one CTA an SM for every kernel that allocates tensor memory, and is exact for those that have no more.)
inline int k8_clusters(int per_sm, int sm_count, int n) {
    constexpr int EMPTY[9] = {0, 0, 0, 10, 8, 10, 13, 18, 16};             // SMs' worth, by cluster size
    return per_sm * (sm_count - (n <= 8 ? EMPTY[n] : 36)) / n;
}

// programmatic dependent launch and, for more than one share, a cluster of that many CTAs; returns how many attributes
inline int k8_attributes(cudaLaunchAttribute* attr, int cluster) {
    int n = 0;
    if (tk_pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = (unsigned)cluster;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    return n;
}

}  // namespace
