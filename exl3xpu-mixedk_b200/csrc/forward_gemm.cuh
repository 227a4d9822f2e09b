// forward_gemm.cuh -- the product for long prompts: the weight is decoded once into
// fp16 (its code values are fp16 numbers, so nothing is lost) and multiplied by a
// tcgen05 GEMM whose epilogue rotates the sums back in registers.
//
// A pair of CTAs (cta_group::2) owns 256 rows x 256 columns of the output: each loads
// its 128 rows and 128 of the columns, and holds its rows' 256 sums in tensor memory,
// twice, so that the epilogue of a tile overlaps the next one's MMAs.  In tensor memory
// a lane is a row, so a thread has all 128 columns of a Hadamard block in registers
// and no lane needs another's.  Decoding in the product instead (forward_mid.cuh) reads the
// rows' operand once per 128 columns rather than per 256 and is bound by that: 1044 us in
// all against 600 at 4096 rows of 5120 x 17408 without activation.
//
// Measured there (K = 5, silu and multiply): 553 to 585 us, the matrix pipe busy 79% of
// the cycles at 1.41 GHz, to which the power limit takes the clock at once (602 thousand
// cycles of MMAs); a library GEMM of the same shape, without decode or epilogue, 490.  The
// time does not depend on a sixth stage (four: 3% more); L2 delivers 13 TB/s.
#pragma once
#include "forward_mid.cuh"

namespace exl3b {

constexpr int kGemmTile = 256;                      // rows and columns of a pair's tile
constexpr int kGemmBox = 128 * 128;                 // 128 rows of 64 k: 16 KB
constexpr int kGemmStage = 2 * kGemmBox;            // rows | columns
constexpr int kGemmPitch = 36;                      // floats: 32 columns of a row in the epilogue
constexpr int kGemmPatch = 32 * kGemmPitch * 4;     // a warp's 32 rows of them
constexpr int kGemmEpilogue = 8;                    // warps: a quarter of the rows, a half of the columns
constexpr int kGemmStages = 5;
constexpr int kGemmBytes = kGemmStages * kGemmStage + kGemmEpilogue * kGemmPatch + 256 + 1024;
constexpr int kGemmThreadsAll = 64 + 32 * kGemmEpilogue;      // loader, MMA, epilogue

// W_inner^T as fp16 [n][k]; the k of a pair of tiles in few_put_block's order, in which
// a lane's values of two tiles are 16 bytes of a row.  A warp per tile column and 128 k.
// 45 us at 5120 x 17408, K = 5, where the bytes read and written take 36; a warp that walks
// a column with its tiles copied ahead gains nothing.
template <int K, int CODE>
__device__ __forceinline__ void expand_block(const uint8_t* src, size_t kt_bytes, __half* out, int k,
                                             int lane) {
    const LaneWindow<K> lw(lane);
    uint8_t* to = reinterpret_cast<uint8_t*>(out + (size_t)(lane >> 2) * k) + (lane & 3) * 16;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        uint32_t a[4], b[4];
        decode_tile<K, CODE>(reinterpret_cast<const uint32_t*>(src + (2 * p) * kt_bytes), lw, a);
        decode_tile<K, CODE>(reinterpret_cast<const uint32_t*>(src + (2 * p + 1) * kt_bytes), lw, b);
        *reinterpret_cast<uint4*>(to + 64 * p) = make_uint4(a[0], a[2], b[0], b[2]);
        *reinterpret_cast<uint4*>(to + 64 * p + (size_t)16 * k) = make_uint4(a[1], a[3], b[1], b[3]);
    }
}

template <int CODE>
__global__ void __launch_bounds__(256)
linear_expand_kernel(const uint8_t* trellis, int K, int k, int n, __half* w) {
    const int lane = threadIdx.x & 31, col = blockIdx.x * 8 + (threadIdx.x >> 5), b = blockIdx.y;
    pdl_launch();
    const size_t kt_bytes = (size_t)(n >> 4) * 32 * K;
    const uint8_t* src = trellis + (size_t)b * 8 * kt_bytes + (size_t)col * 32 * K;
    __half* out = w + (size_t)col * 16 * k + b * 128;
    with_bits(K, [&](auto bits) {
        expand_block<decltype(bits)::value, CODE>(src, kt_bytes, out, k, lane);
    });
    pdl_wait();                // this kernel's end stands for the rotation's, too
}

struct GemmArgs {
    int M, k, n;
    int parts;                 // of the rows' values: 2 with the remainders, M rows on
    const float* inv;          // [M] reciprocal row scales
    int* err;
    WaitLimit limit;
};

// 128-point Hadamard transform of a thread's values, not normalised.
__device__ __forceinline__ void had128_thread(float (&v)[128]) {
#pragma unroll
    for (int h = 1; h < 128; h <<= 1)
#pragma unroll
        for (int i = 0; i < 128; ++i)
            if (!(i & h)) {
                const float a = v[i], b = v[i + h];
                v[i] = a + b;
                v[i + h] = a - b;
            }
}

// Tile t: groups of up to 16 row tiles, columns slowest inside a group, so that the
// tiles in flight share their operands in L2.
__device__ __forceinline__ void gemm_place(int t, int mt, int nt, int& m, int& n) {
    const int per = 16 * nt, g = t / per, first = g * 16, rows = min(16, mt - first), in = t - g * per;
    n = in / rows;
    m = first + in - n * rows;
}

template <typename Epilogue>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGemmThreadsAll, 1)
linear_gemm_kernel(const __grid_constant__ CUtensorMap rows, const __grid_constant__ CUtensorMap cols,
                   const GemmArgs g, const Epilogue ep) {
    extern __shared__ __align__(1024) uint8_t sm_raw[];
    __shared__ int fail, peer_fail, sent[2];    // sent: chunks that each CTA has asked for
    __shared__ uint32_t tmem_slot;
    uint8_t* sm = (uint8_t*)(((uintptr_t)sm_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + kGemmStages * kGemmStage + kGemmEpilogue * kGemmPatch);
    const uint32_t full = shared_addr(bars), empty = full + 8 * kGemmStages,
                   afull = empty + 8 * kGemmStages, aempty = afull + 16, done = aempty + 16;
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const int rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int mt = (g.M + kGemmTile - 1) / kGemmTile, nt = (g.n + kGemmTile - 1) / kGemmTile;
    const int tiles = mt * nt, kchunks = g.k >> 6, chunks = g.parts * kchunks;
    if (t == 0) {
        for (int i = 0; i < kGemmStages; ++i) {
            bar_init(full + 8 * i, 1);
            bar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(afull + 8 * i, 1);
            bar_init(aempty + 8 * i, 2 * kGemmEpilogue);
        }
        bar_init(done, 1);
        fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tc_alloc_pair(shared_addr(&tmem_slot));
    tc_fence_before();
    __syncthreads();
    cluster_meet();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_wait();

    if (t == 0) {
        // loader: this CTA's rows and columns of every chunk, counted at the leader
        asm volatile("fence.proxy.async.global;" ::: "memory");
        int s = 0, r = 0, issued = 0;
        bool ok = true;
        for (int tile = pair; tile < tiles && ok; tile += pairs) {
            int m, n;
            gemm_place(tile, mt, nt, m, n);
            for (int c = 0; c < chunks; ++c) {
                if (r > 0) ok = bar_wait(empty + 8 * s, (r - 1) & 1, &fail, g.limit);
                if (!ok) break;
                const uint32_t dst = shared_addr(sm) + s * kGemmStage, bar = cluster_addr(full + 8 * s, 0);
                if (rank == 0) bar_expect(full + 8 * s, 2 * kGemmStage);
                // (rows past the last of the values are remainders, or zeros; their sums
                // are not stored)
                const int x = c < kchunks ? c : c - kchunks;
                tma_load_pair(dst, &rows, x * 64, m * kGemmTile + rank * 128 + (x == c ? 0 : g.M), bar);
                tma_load_pair(dst + kGemmBox, &cols, x * 64, n * kGemmTile + rank * 128, bar);
                ++issued;
                if (++s == kGemmStages) { s = 0; ++r; }
            }
        }
        if (!ok) atomicExch(&fail, 1);
        cluster_store(cluster_addr(shared_addr(&sent[rank]), 0), issued);
    } else if (t == 32) {
        if (rank == 0) {
            const uint32_t idesc = mma_desc_f16(256, 256);
            int s = 0, r = 0, lt = 0;
            bool ok = true;
            for (int tile = pair; tile < tiles && ok; tile += pairs, ++lt) {
                const int acc = lt & 1, use = lt >> 1;
                if (use > 0) ok = bar_wait(aempty + 8 * acc, (use - 1) & 1, &fail, g.limit);
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = tmem + acc * 256;
                for (int c = 0; c < chunks; ++c) {
                    ok = bar_wait(full + 8 * s, r & 1, &fail, g.limit);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t base = shared_addr(sm) + s * kGemmStage;
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        asm volatile(
                            "{\n\t.reg .pred p;\n\t"
                            "setp.ne.b32 p, %4, 0;\n\t"
                            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                            :: "r"(d), "l"(operand_desc(base + 32 * q)),
                               "l"(operand_desc(base + kGemmBox + 32 * q)), "r"(idesc),
                               "r"((uint32_t)(c > 0 || q > 0)) : "memory");
                    tc_commit_pair(empty + 8 * s);
                    if (++s == kGemmStages) { s = 0; ++r; }
                }
                if (ok) tc_commit_pair(afull + 8 * acc);
            }
            if (!ok) atomicExch(&fail, 1);
            tc_commit_pair(done);
            if (!bar_drain(done, 0)) atomicExch(&fail, 1);
        }
    } else if (warp >= 2) {
        // epilogue: lane = row up to the rotation; then, 32 columns at a time through
        // shared memory, eight lanes a row, so that global memory sees 64-byte pieces and
        // the code stays small (unrolled over a thread's 128 columns it missed the
        // instruction cache: 1.74 ms with silu).  Operands are asked for before the
        // exchange: a warp has little else to hide their latency.
        const int quad = warp & 3, half = (warp - 2) >> 2;
        float* patch = reinterpret_cast<float*>(sm + kGemmStages * kGemmStage + (warp - 2) * kGemmPatch);
        int lt = 0;
        for (int tile = pair; tile < tiles; tile += pairs, ++lt) {
            const int acc = lt & 1, use = lt >> 1;
            int m, n;
            gemm_place(tile, mt, nt, m, n);
            const int row0 = m * kGemmTile + rank * 128 + 32 * quad, row = row0 + lane;
            const int col = n * kGemmTile + half * 128, have = col < g.n ? min(32, g.M - row0) : 0;
            const float f = row < g.M ? g.inv[row] * kInvSqrt128 : 0.0f;
            const bool ok = __all_sync(0xffffffffu, bar_wait(afull + 8 * acc, use & 1, &fail, g.limit));
            if (!ok) {
                if (lane == 0) atomicExch(&fail, 1);
                break;
            }
            tc_fence_after();
            float v[128];
#pragma unroll
            for (int c = 0; c < 4; ++c)
                tc_load32(tmem + ((uint32_t)(32 * quad) << 16) + acc * 256 + half * 128 + c * 32,
                          *reinterpret_cast<uint32_t(*)[32]>(&v[c * 32]));
            tc_wait_ld();
            tc_fence_before();                 // read out: the leader may use it again
            __syncwarp();
            if (lane == 0) bar_arrive_cluster(cluster_addr(aempty + 8 * acc, 0));
            if (have <= 0) continue;
            had128_thread(v);
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
                typename Epilogue::Operands op;
                ep.fetch(op, row0, have, col + c * 32, lane);
                float4* to = reinterpret_cast<float4*>(patch + lane * kGemmPitch);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e == c) {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            to[j] = make_float4(v[e * 32 + 4 * j] * f, v[e * 32 + 4 * j + 1] * f,
                                                v[e * 32 + 4 * j + 2] * f, v[e * 32 + 4 * j + 3] * f);
                    }
                __syncwarp();
                ep.finish(op, row0, have, col + c * 32, patch, lane);
                __syncwarp();
            }
        }
        // the leader's last arrival here, so that none comes after this CTA has ended
        if (rank == 1 && !bar_drain(done, 0) && lane == 0) atomicExch(&fail, 1);
    }
    // Without a failure every load has been multiplied by now.  After one the leader,
    // at whose barriers both CTAs' loads are counted, sees to it that they have landed
    // before either's shared memory is released.
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (t == 0) cluster_store(cluster_addr(shared_addr(&peer_fail), rank ^ 1), fail);
    cluster_meet();
    if (fail || peer_fail) {
        if (t == 0) *(volatile int*)g.err = 1;
        if (t == 0 && rank == 0) {
            const int both = min(sent[0], sent[1]), all = max(sent[0], sent[1]);
            for (int i = max(0, both - kGemmStages); i < all; ++i) {
                const uint32_t bar = full + 8 * (i % kGemmStages);
                if (i >= sent[1]) bar_forgo(bar, kGemmStage);       // the other will not ask
                if (i >= sent[0]) bar_expect(bar, kGemmStage);      // the other has asked ahead
                bar_drain(bar, (i / kGemmStages) & 1);
            }
        }
        if (t == 0 && rank == 1) bar_drain(done, 0);
        cluster_meet();
    }
    if (warp == 1) tc_free_pair(tmem);
}

}  // namespace exl3b
