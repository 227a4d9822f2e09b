// forward_few.cuh -- the few-rows product of the forward kernels: up to 8 G rows of
// activations times a 128-column block of an EXL3 tensor, decoded on the fly.
//
// Eight warps, one 16-column tile column each, walk the CTA's share of k in blocks
// of 128 (the Hadamard block).  A warp streams its own tiles through a private
// cp.async ring in shared memory (no barrier between warps, nothing to wait for but
// its own copies) and multiplies them with mma.sync: at 8 to 16 rows the product is
// bound by the decode's instruction issue and by the trellis' bytes, not by the
// matrix unit, and mma.sync takes the decoded operand from the registers it was
// decoded into, without the trip through tensor memory that tcgen05 would need.
#pragma once
#include <cooperative_groups.h>

#include "trellis_mma.cuh"

namespace exl3b {

constexpr int kFewWarps = 8;
constexpr int kFewStages = 4;         // ring depth in blocks of 128 k
constexpr int kPartPitch = 132;       // floats per row of a partial block

// element types of activations (the ABI's dtype values)
enum XType : int { X_BF16 = 1, X_FP16 = 2 };

__device__ __forceinline__ void load4x(const void* p, size_t i, int dtype, float (&v)[4]) {
    if (dtype == X_BF16) load4(static_cast<const __nv_bfloat16*>(p) + i, v);
    else load4(static_cast<const __half*>(p) + i, v);
}

__device__ __forceinline__ void store4x(void* p, size_t i, int dtype, const float (&v)[4]) {
    if (dtype == X_BF16) store4(static_cast<__nv_bfloat16*>(p) + i, v);
    else store4(static_cast<__half*>(p) + i, v);
}

__host__ __device__ inline int few_ring_bytes(int K) { return kFewStages * 256 * K; }   // per warp
// One row of rotated activations in shared memory: fp16, plus 64 bytes so that the
// two rows a quarter-warp reads at once fall into different banks.
__host__ __device__ inline int few_row_bytes(int nblk) { return nblk * 256 + 64; }

// Issue the copies of one k block of a warp's tile column into a ring stage.
__device__ __forceinline__ void few_issue(const uint8_t* src, size_t kt_bytes, int K, uint8_t* stage,
                                          int lane) {
    const uint32_t dst = (uint32_t)__cvta_generic_to_shared(stage);
    const int per = 2 * K;                                  // 16-byte pieces of a tile
    for (int c = lane; c < 8 * per; c += 32) {
        const int kt = c / per;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                     :: "r"(dst + 16 * c), "l"(src + kt * kt_bytes + 16 * (c - kt * per)) : "memory");
    }
}

// Rotate one 128-block of a row held by a warp (element 4 lane + j in v[j], suh
// already applied) and store it as the product's B operand: fp16 times a power of
// two (block_scale; its reciprocal goes to *inv_scale).  The 16 k of a tile are
// stored so that a lane's four values, and those of the next tile, are 16 bytes.
// Rounding to fp16 (2^-11 relative at most) matches the weights' type, which a
// matrix instruction needs; bf16 would cost three bits of the activations.
__device__ __forceinline__ void few_put_block(float (&v)[4], uint8_t* dst, float* inv_scale,
                                              int lane) {
    float m = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float inv;
    const float s = block_scale(m, inv) * kInvSqrt128;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] *= s;
    had128_warp(v, lane);
    // k = 4 lane: pair of tiles k / 32, tile (k / 16) & 1, inside it q = (k % 8) / 2
    const int k = 4 * lane;
    const int off = (k >> 5) * 32 + ((k & 7) >> 1) * 8 + ((k >> 4) & 1) * 4 + ((k >> 3) & 1) * 2;
    const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
    *reinterpret_cast<__half2*>(dst + 2 * off) = a;
    *reinterpret_cast<__half2*>(dst + 2 * off + 16) = b;
    if (lane == 0) *inv_scale = inv;
}

// acc[g][..] += the warp's 16 columns of `nblk` k blocks, rows 8 g .. 8 g + 7.
//   src       first tile of the warp's column in the CTA's share
//   xh        rows of few_put_block blocks, row pitch `xpitch` bytes
//   inv       [nblk][8 G] reciprocal block scales
// The first kFewStages - 1 blocks were issued (and committed) by the caller.
template <int K, int CODE, int G>
__device__ __forceinline__ void few_product(const uint8_t* src, size_t kt_bytes, int nblk,
                                            uint8_t* ring, const uint8_t* xh, int xpitch,
                                            const float* inv, float (&acc)[G][4], int lane) {
    const LaneWindow<K> lw(lane);
    const uint8_t* xrow = xh + (lane >> 2) * xpitch + (lane & 3) * 16;
    const float* irow = inv + (lane & 3) * 2;
    for (int b = 0; b < nblk; ++b) {
        const int nxt = b + kFewStages - 1;
        if (nxt < nblk)
            few_issue(src + (size_t)nxt * 8 * kt_bytes, kt_bytes, K,
                      ring + (nxt % kFewStages) * 256 * K, lane);
        asm volatile("cp.async.commit_group;" ::: "memory");
        asm volatile("cp.async.wait_group %0;" :: "n"(kFewStages - 1) : "memory");
        __syncwarp();
        const uint32_t* tiles = reinterpret_cast<const uint32_t*>(ring + (b % kFewStages) * 256 * K);
        float blk[G][4];
#pragma unroll
        for (int g = 0; g < G; ++g) blk[g][0] = blk[g][1] = blk[g][2] = blk[g][3] = 0.0f;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            uint4 x[G];
#pragma unroll
            for (int g = 0; g < G; ++g)
                x[g] = *reinterpret_cast<const uint4*>(xrow + g * 8 * xpitch + b * 256 + p * 64);
            uint32_t a[4];
            decode_tile<K, CODE>(tiles + (2 * p) * 8 * K, lw, a);
#pragma unroll
            for (int g = 0; g < G; ++g) mma_16816(blk[g], a, x[g].x, x[g].y);
            decode_tile<K, CODE>(tiles + (2 * p + 1) * 8 * K, lw, a);
#pragma unroll
            for (int g = 0; g < G; ++g) mma_16816(blk[g], a, x[g].z, x[g].w);
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const float2 f = *reinterpret_cast<const float2*>(irow + b * 8 * G + g * 8);
            acc[g][0] = fmaf(blk[g][0], f.x, acc[g][0]);
            acc[g][1] = fmaf(blk[g][1], f.y, acc[g][1]);
            acc[g][2] = fmaf(blk[g][2], f.x, acc[g][2]);
            acc[g][3] = fmaf(blk[g][3], f.y, acc[g][3]);
        }
        __syncwarp();      // every lane has read the stage before it is refilled
    }
}

template <int CODE, int G>
__device__ __forceinline__ void few_product_k(int K, const uint8_t* src, size_t kt_bytes, int nblk,
                                              uint8_t* ring, const uint8_t* xh, int xpitch,
                                              const float* inv, float (&acc)[G][4], int lane) {
    switch (K) {
        case 2: few_product<2, CODE, G>(src, kt_bytes, nblk, ring, xh, xpitch, inv, acc, lane); break;
        case 3: few_product<3, CODE, G>(src, kt_bytes, nblk, ring, xh, xpitch, inv, acc, lane); break;
        case 4: few_product<4, CODE, G>(src, kt_bytes, nblk, ring, xh, xpitch, inv, acc, lane); break;
        case 5: few_product<5, CODE, G>(src, kt_bytes, nblk, ring, xh, xpitch, inv, acc, lane); break;
        case 6: few_product<6, CODE, G>(src, kt_bytes, nblk, ring, xh, xpitch, inv, acc, lane); break;
        default: few_product<7, CODE, G>(src, kt_bytes, nblk, ring, xh, xpitch, inv, acc, lane); break;
    }
}

// First blocks of the ring (kFewStages - 1 groups, empty ones past the end).
__device__ __forceinline__ void few_prologue(const uint8_t* src, size_t kt_bytes, int K, int nblk,
                                             uint8_t* ring, int lane) {
#pragma unroll
    for (int s = 0; s < kFewStages - 1; ++s) {
        if (s < nblk) few_issue(src + (size_t)s * 8 * kt_bytes, kt_bytes, K, ring + s * 256 * K, lane);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
}

// A warp's accumulators -> the CTA's partial block [8 G rows][128 columns].
template <int G>
__device__ __forceinline__ void few_store_part(float* part, const float (&acc)[G][4], int tile,
                                               int lane) {
    const int n = tile * 16 + (lane >> 2), r = (lane & 3) * 2;
#pragma unroll
    for (int g = 0; g < G; ++g) {
        float* p = part + (g * 8 + r) * kPartPitch + n;
        p[0] = acc[g][0];
        p[kPartPitch] = acc[g][1];
        p[8] = acc[g][2];
        p[kPartPitch + 8] = acc[g][3];
    }
}

// Sum of one row of the cluster's partial blocks, in rank order, elements
// 4 lane .. 4 lane + 3, then the output rotation (normalised).
__device__ __forceinline__ void few_sum_row(const float* part, int row, int nrank, int lane,
                                            float (&v)[4]) {
    namespace cg = cooperative_groups;
    const float* own = part + row * kPartPitch + 4 * lane;
    v[0] = v[1] = v[2] = v[3] = 0.0f;
    if (nrank == 1) {
        const float4 f = *reinterpret_cast<const float4*>(own);
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
        cg::cluster_group cl = cg::this_cluster();
        for (int r = 0; r < nrank; ++r) {
            const float4 f = *reinterpret_cast<const float4*>(
                cl.map_shared_rank(const_cast<float*>(own), r));
            v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] *= kInvSqrt128;
    had128_warp(v, lane);
}

}  // namespace exl3b
