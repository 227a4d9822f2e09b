// forward_few.cuh -- the few-rows product of the forward kernels: up to 8 G rows of
// activations times a 128-column block of an EXL3 tensor, decoded on the fly.
//
// Two groups of eight warps, one 16-column tile column each, walk the CTA's share of
// k in blocks of 128 (the Hadamard block), taking blocks in turn.  A warp streams its own tiles through a private
// cp.async ring in shared memory (no barrier between warps, nothing to wait for but
// its own copies) and multiplies them with mma.sync: at 8 to 16 rows the product is
// bound by the decode's instruction issue and by the trellis' bytes, not by the
// matrix unit, and mma.sync takes the decoded operand from the registers it was
// decoded into, without the trip through tensor memory that tcgen05 would need.
#pragma once
#include "exl3b_internal.h"
#include "trellis_mma.cuh"

namespace exl3b {

constexpr int kFewGroups = 2;         // groups of eight warps, taking k blocks in turn
constexpr int kFewWarps = 8 * kFewGroups;
constexpr int kFewStages = 3;         // ring depth in blocks of 128 k

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
// Rotated activations in shared memory: [block][8 G rows][256 bytes], the two halves
// of each 128-byte group exchanged in odd rows so that the two rows a quarter-warp
// reads at once fall into different banks.
constexpr int kRowBytes = 256;
__device__ __forceinline__ int few_swizzle(int row, int byte) { return byte ^ ((row & 1) << 6); }

// A warp's stream of k blocks: 16 K pieces of 16 bytes a block, piece c by lane
// c mod 32 in turn.  Where a lane's pieces lie inside a block does not change, so
// they are found once.
template <int K>
struct FewStream {
    static constexpr int kPieces = (16 * K + 31) / 32;         // per lane
    uint32_t kt[kPieces], off[kPieces];    // k tile of a piece and its place in the tile
    int lane;

    __device__ __forceinline__ explicit FewStream(int lane_) : lane(lane_) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int c = lane + 32 * i;
            kt[i] = c / (2 * K);
            off[i] = 16 * (c - kt[i] * 2 * K);
        }
    }
    // Copy the block whose first tile is at `src` into stage `stage` of the ring.
    __device__ __forceinline__ void issue(const uint8_t* src, uint32_t kt_bytes, uint8_t* ring,
                                          int stage) {
        const uint32_t dst = (uint32_t)__cvta_generic_to_shared(ring) + stage * 256 * K + 16 * lane;
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
            if (16 * K % 32 == 0 || i + 1 < kPieces || lane + 32 * i < 16 * K)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                             :: "r"(dst + 512 * i), "l"(src + (kt[i] * kt_bytes + off[i])) : "memory");
    }
};

__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory");
}

// Programmatic dependent launch: let the next kernel of the stream start its
// prologue; wait for the previous kernel's results.
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Rotate one 128-block of a row held by a warp (element 4 lane + j in v[j], suh
// already applied) and store it as the product's B operand: fp16 times a power of
// two (block_scale; its reciprocal goes to *inv_scale).  The 16 k of a tile are
// stored so that a lane's four values, and those of the next tile, are 16 bytes.
// Rounding to fp16 (2^-11 relative at most) matches the weights' type, which a
// matrix instruction needs; bf16 would cost three bits of the activations.
__device__ __forceinline__ void few_put_block(float (&v)[4], uint8_t* dst, float* inv_scale,
                                              int lane, int swz) {
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
    *reinterpret_cast<__half2*>(dst + ((2 * off) ^ swz)) = a;
    *reinterpret_cast<__half2*>(dst + ((2 * off + 16) ^ swz)) = b;
    if (lane == 0) *inv_scale = inv;
}

// acc[g][..] += one k block: the warp's eight tiles at `tiles`, rows 8 g .. 8 g + 7 of
// the block at `xh`, reciprocal scales inv [8 G].
template <int K, int CODE, int G>
__device__ __forceinline__ void few_block(const LaneWindow<K>& lw, const uint8_t* tiles_,
                                          const uint8_t* xh, const float* inv, float (&acc)[G][4],
                                          int lane) {
    const uint32_t* tiles = reinterpret_cast<const uint32_t*>(tiles_);
    const int row = lane >> 2, swz = (row & 1) << 6;
    const uint8_t* even = xh + row * kRowBytes + (lane & 3) * 16 + swz;      // p even: p * 64 ^ swz
    const uint8_t* odd = even - 2 * swz;                                     // p odd
    float blk[G][4];
#pragma unroll
    for (int g = 0; g < G; ++g) blk[g][0] = blk[g][1] = blk[g][2] = blk[g][3] = 0.0f;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        uint4 x[G];
#pragma unroll
        for (int g = 0; g < G; ++g)
            x[g] = *reinterpret_cast<const uint4*>((p & 1 ? odd : even) + g * 8 * kRowBytes + p * 64);
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
        const float2 f = *reinterpret_cast<const float2*>(inv + g * 8 + (lane & 3) * 2);
        acc[g][0] = fmaf(blk[g][0], f.x, acc[g][0]);
        acc[g][1] = fmaf(blk[g][1], f.y, acc[g][1]);
        acc[g][2] = fmaf(blk[g][2], f.x, acc[g][2]);
        acc[g][3] = fmaf(blk[g][3], f.y, acc[g][3]);
    }
}

// f(BitWidth<K>()) for a runtime K: one copy of the streaming loop
// per bit width, chosen once per warp.
template <int K> struct BitWidth { static constexpr int value = K; };
template <typename F>
__device__ __forceinline__ void with_bits(int K, const F& f) {
    switch (K) {
        case 2: f(BitWidth<2>()); break;
        case 3: f(BitWidth<3>()); break;
        case 4: f(BitWidth<4>()); break;
        case 5: f(BitWidth<5>()); break;
        case 6: f(BitWidth<6>()); break;
        default: f(BitWidth<7>()); break;
    }
}

// ------------------------------------------------------------------ the product
// The work is a sequence of units, each a column block (128 columns) of one tensor
// times up to 8 G rows: kb blocks of 128 x 128.  The decode, equal in every block,
// bounds it, so each CTA (one per SM) takes an equal run of the sequence's blocks,
// wherever it starts and ends, and parks the sums of every unit that it touches; a
// second kernel, launched early and waiting, adds them up in the order of the CTAs and
// their groups.  Measured on one row of 5120 x 5120 at K = 4: 11.9 us; with k split over
// clusters that join through distributed shared memory 11.3 at the one cluster size
// that fits the 40 column blocks and 14 to 16 at the others (row of 17408 x 5120: 31 to
// 37 and up); with the last CTA of a unit to arrive adding the sums 14.7.
struct FewRun {
    int kb, units, ctas;
    int least, longer;         // blocks of a CTA's run; the first `longer` have one more
    __host__ __device__ FewRun(int kb_, int units_, int sms) : kb(kb_), units(units_) {
        const int total = kb * units;
        ctas = total < sms ? total : sms;
        least = ctas ? total / ctas : 0;
        longer = ctas ? total % ctas : 0;
    }
    __host__ __device__ int start(int cta) const { return cta * least + (cta < longer ? cta : longer); }
    // the CTA whose run holds block g
    __host__ __device__ int owner(int g) const {
        const int head = longer * (least + 1);
        return g < head ? g / (least + 1) : longer + (g - head) / least;
    }
    __host__ __device__ int first(int u) const { return owner(u * kb); }
    __host__ __device__ int last(int u) const { return owner(u * kb + kb - 1); }
};

// Parked sums: CTA c's of unit u at slot u + c (along the sequence u or c grows, so
// the slots differ), per group [8 G rows][128 columns].
__host__ __device__ inline size_t few_park_bytes(int units, int ctas, int G) {
    return (size_t)(units + ctas) * kFewGroups * 8 * G * 512;
}

// Rows are in shared memory for a chunk of blocks at a time (two buffers of 16 / G).
// A group of warps issues at least kFewStages copies per chunk, which is what makes
// the next chunk's rows older than any copy in flight when the chunk ends.
template <int G> struct FewChunk { static constexpr int value = 16 / G; };

__host__ __device__ inline int few_smem(int Kmax) {
    return kFewWarps * few_ring_bytes(Kmax) + 2 * 16 * 8 * (kRowBytes + 4);
}

// A job tells what the units are:
//   unit(u)      -> FewUnit, the weight
//   rows(u)      -> its rows, at most 8 G
//   row(u, r, b) -> index of the rotated block b of row r (blocks of 256 bytes at
//                   xh(), reciprocal scales at inv()); or, where kRotate is set,
//   rotate(u, r, b, dst, inv, swz)  puts the block itself (a warp)
//   wait()       -> returns once the rows are there
struct FewUnit {
    const uint8_t* tiles;      // first tile of the column block
    uint32_t kt_bytes;         // to the next k tile
    int K;
};

// Multiply this CTA's run and park the sums.  All threads.
template <int CODE, int G, typename Job>
__device__ __forceinline__ void few_run(const Job& job, const FewRun& run, int Kmax, uint8_t* sm,
                                        float* park) {
    constexpr int kChunk = FewChunk<G>::value;
    static_assert(kChunk / kFewGroups > kFewStages, "a chunk outlasts the ring");
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31, grp = warp >> 3, col = warp & 7;
    const int cta = blockIdx.x, g0 = run.start(cta), count = run.start(cta + 1) - g0;
    uint8_t* ring = sm + warp * few_ring_bytes(Kmax);
    uint8_t* xh = sm + kFewWarps * few_ring_bytes(Kmax);
    float* inv = reinterpret_cast<float*>(xh + 2 * kChunk * 8 * G * kRowBytes);
    const int kb = run.kb, u0 = g0 / kb, b0 = g0 - u0 * kb;

    // Rows of a chunk's blocks.  Rows past the unit's last stay unwritten: a row is a
    // column of the matrix instruction, and only rows that exist are read back.
    auto load_rows = [&](int c) {
        const int lo = c * kChunk, n = min(kChunk, count - lo);
        uint8_t* x = xh + (c & 1) * kChunk * 8 * G * kRowBytes;
        float* s = inv + (c & 1) * kChunk * 8 * G;
        if constexpr (Job::kRotate) {
            const int rows = job.rows(u0);                    // of every unit
            for (int j = warp; j < n * rows; j += kFewWarps) {
                const int blk = j / rows, r = j - blk * rows, f = b0 + lo + blk, u = u0 + f / kb;
                job.rotate(u, r, f - f / kb * kb, x + (blk * 8 * G + r) * kRowBytes, s + blk * 8 * G + r,
                           (r & 1) << 6);
            }
        } else {
            // 16 lanes copy four rows of one block
            const int half = t >> 4, blk = half / (2 * G), q = t & 15, r0 = half % (2 * G) * 4;
            if (blk < n) {
                const int f = b0 + lo + blk, u = u0 + f / kb, b = f - f / kb * kb, rows = job.rows(u);
                const uint32_t dst = (uint32_t)__cvta_generic_to_shared(x) + blk * 8 * G * kRowBytes;
                const uint32_t dsi = (uint32_t)__cvta_generic_to_shared(s + blk * 8 * G);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = r0 + e;
                    if (r >= rows) break;
                    const size_t from = job.row(u, r, b);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                                 :: "r"(dst + r * kRowBytes + few_swizzle(r, 16 * q)),
                                    "l"(job.xh() + from * kRowBytes + 16 * q) : "memory");
                    if (q == 0)
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;"
                                     :: "r"(dsi + 4 * r), "l"(job.inv() + from) : "memory");
                }
            }
        }
    };

    float acc[G][4];
#pragma unroll
    for (int g = 0; g < G; ++g) acc[g][0] = acc[g][1] = acc[g][2] = acc[g][3] = 0.0f;
    int i = grp;                              // this group's next block of the run
    int chunk = 0;                            // chunk whose rows are ready, once i >= 0
    bool rows_ready = false;
    // Stretches of equal bit width: the ring restarts where it changes.
    while (i < count) {
        const int K0 = job.unit(u0 + (b0 + i) / kb).K;
        with_bits(K0, [&](auto bits) {
            constexpr int K = decltype(bits)::value;
            int u = u0 + (b0 + i) / kb, b = (b0 + i) % kb;
            // the issuing side runs kFewStages - 1 of the group's blocks ahead
            FewUnit to = job.unit(u);
            int iu = u, ib = b, ii = i;
            bool more = true;                 // the next block to issue has this width
            FewStream<K> st(lane);
            auto issue = [&](int stage) {
                if (more && ii < count) {
                    st.issue(to.tiles + (size_t)ib * 8 * to.kt_bytes + (size_t)col * 32 * K, to.kt_bytes,
                             ring, stage);
                    ii += kFewGroups;
                    ib += kFewGroups;
                    if (ib >= kb && ii < count) {
                        while (ib >= kb) { ib -= kb; ++iu; }
                        to = job.unit(iu);
                        more = to.K == K;
                    }
                }
                cp_commit();
            };
#pragma unroll
            for (int s = 0; s < kFewStages - 1; ++s) issue(s);
            if (!rows_ready) {
                job.wait();                   // the rows come from the kernel before
                load_rows(0);
                cp_commit();
                cp_wait<0>();
                __syncthreads();
                rows_ready = true;
                if (kChunk < count) load_rows(1);     // joins the next commit
            }
            const LaneWindow<K> lw(lane);
            int cur = 0, fill = kFewStages - 1;
            while (true) {
                if (i / kChunk != chunk) {
                    // the next chunk's rows were issued a chunk ago: older than every
                    // copy still in flight
                    cp_wait<kFewStages - 1>();
                    __syncthreads();
                    ++chunk;
                    if ((chunk + 1) * kChunk < count) load_rows(chunk + 1);
                }
                issue(fill);
                cp_wait<kFewStages - 1>();
                __syncwarp();
                const int slot = (chunk & 1) * kChunk + (i - chunk * kChunk);
                few_block<K, CODE, G>(lw, ring + cur * 256 * K, xh + slot * 8 * G * kRowBytes,
                                      inv + slot * 8 * G, acc, lane);
                fill = cur;
                cur = cur + 1 == kFewStages ? 0 : cur + 1;
                __syncwarp();      // every lane has read the stage before it is refilled
                i += kFewGroups;
                b += kFewGroups;
                if (b < kb && i < count) continue;
                // the group's last block of this unit here: park the sums
                const int rows = job.rows(u);
                float* out = park + ((size_t)(u + cta) * kFewGroups + grp) * 8 * G * 128 + col * 16 +
                             (lane >> 2);
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const int r = g * 8 + (lane & 3) * 2;
                    if (r < rows) {
                        out[r * 128] = acc[g][0];
                        out[r * 128 + 8] = acc[g][2];
                    }
                    if (r + 1 < rows) {
                        out[r * 128 + 128] = acc[g][1];
                        out[r * 128 + 136] = acc[g][3];
                    }
                    acc[g][0] = acc[g][1] = acc[g][2] = acc[g][3] = 0.0f;
                }
                if (i >= count) break;
                while (b >= kb) { b -= kb; ++u; }
                if (job.unit(u).K != K) break;
            }
            cp_wait<0>();
            __syncwarp();
        });
    }
    // every warp takes part in every chunk's barrier
    if (!rows_ready) { job.wait(); load_rows(0); cp_commit(); cp_wait<0>(); __syncthreads(); if (kChunk < count) load_rows(1); }
    while ((chunk + 1) * kChunk < count) {
        cp_commit();
        cp_wait<0>();
        __syncthreads();
        ++chunk;
        if ((chunk + 1) * kChunk < count) load_rows(chunk + 1);
    }
}

// Sum of unit u's parked sums of row r, elements 4 lane .. 4 lane + 3: the ones at
// `part`, part + parts, ... in the order of the CTAs and their groups.  A warp.
template <int G>
__device__ __forceinline__ void few_sum(const float* park, const FewRun& run, int u, int r, int lane,
                                        int part, int parts, float (&v)[4]) {
    const int lo = u * run.kb, hi = lo + run.kb;
    const int c0 = run.first(u), n = (run.last(u) - c0 + 1) * kFewGroups;
    const float* from = park + (size_t)(u + c0) * kFewGroups * 8 * G * 128 + r * 128 + 4 * lane;
    v[0] = v[1] = v[2] = v[3] = 0.0f;
#pragma unroll 4
    for (int i = part; i < n; i += parts) {
        const int c = c0 + i / kFewGroups, g = i % kFewGroups;
        const int s = run.start(c), e = run.start(c + 1);
        const int f = s > lo ? s : lo, l = e < hi ? e : hi;      // the CTA's blocks of u
        // a group takes every other block of the run: none of a single one, maybe
        if (l - f >= kFewGroups || ((f - s) & 1) == g) {
            const float4 q = __ldcg(reinterpret_cast<const float4*>(from + (size_t)i * 8 * G * 128));
            v[0] += q.x; v[1] += q.y; v[2] += q.z; v[3] += q.w;
        }
    }
}

__device__ __forceinline__ void add4(float (&v)[4], const float4& q) {
    v[0] += q.x; v[1] += q.y; v[2] += q.z; v[3] += q.w;
}

// The output rotation (normalised) of a block held by a warp.
__device__ __forceinline__ void few_rotate_back(float (&v)[4], int lane) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] *= kInvSqrt128;
    had128_warp(v, lane);
}

template <typename... P, typename... A>
int launch_kernel(void (*kern)(P...), const char* what, dim3 grid, int threads, size_t smem, bool pdl,
                  cudaStream_t stream, A... args) {
    if (smem > 48 * 1024 &&
        check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
                   what))
        return RC_DEVICE_ERROR;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = pdl ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
    note_launch();
    return check_cuda(e, what) ? RC_DEVICE_ERROR : RC_OK;
}

}  // namespace exl3b
