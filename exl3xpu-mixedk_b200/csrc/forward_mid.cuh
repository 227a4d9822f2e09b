// forward_mid.cuh -- the product for a few dozen to a few hundred rows: decoded weights
// go from registers to tensor memory as the A operand of tcgen05.mma, the rotated rows
// are the B operand in shared memory.
//
// D (128 columns of W x N rows) += W_inner^T (128 x 128, TMEM) . rows^T.  A decoded
// tile is the 16 x 128-bit store pattern of tensor memory as it is, so it reaches the
// matrix unit without passing through shared memory, and one decode serves up to 256
// rows (mma.sync takes 16 and is bound by its own issue beyond).  A block takes the two
// decoding groups about 830 cycles and the matrix unit 4 N, so the decode bounds the
// kernel up to some 200 rows.  203 rows of 5120 x 6144 at K = 3: 21.4 us; without the decode
// 17.1, with one MMA a block of eight 17.1, with neither 14.5, which is the wait for the
// rows' rotation, their copies and the parking of the sums (37 rows of 6144 x 5120, MCG, K =
// 6, without remainders: 18.1, 12.8, 15.9, 9.7).
//
// 18 warps: 16 decode (two groups, blocks in turn; warp w writes the TMEM lanes
// 32 (w mod 4) .. it may), one issues the MMAs, one loads the rows by TMA.  A group has two A
// buffers, so it decodes a block while the one before is multiplied.  The blocks are
// spread over the SMs as in forward_few.cuh, and the sums of a unit parked per CTA.
#pragma once
#include "forward_few.cuh"
#include "tc.cuh"

namespace exl3b {

constexpr int kMidThreads = 32 * (kFewWarps + 2);
constexpr int kMidRows = 256;             // of one pass
constexpr int kMidAcc = 0, kMidA = 256;   // TMEM columns of D and of the four A buffers

struct MidArgs {
    const uint8_t* trellis;
    int K, nbn;                           // column blocks
    int M, N;                             // rows; rows of a pass (multiple of 16)
    int stages;                           // of the rows' ring
    FewRun run;                           // units: (pass, column block)
    float* park;                          // [units + ctas][N][128]
    int* err;
    WaitLimit limit;
};

__host__ __device__ inline int mid_smem(int K, int N, int stages) {
    return kFewWarps * few_ring_bytes(K) + stages * N * 256 + 256 + 1024;
}

// Decode four k tiles and store them as 64 k of this warp's 16 lanes of A.
template <int K, int CODE>
__device__ __forceinline__ void mid_decode4(const uint32_t* tiles, const LaneWindow<K>& lw,
                                            uint32_t (&r)[16]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t a[4];
        decode_tile<K, CODE>(tiles + j * 8 * K, lw, a);
        r[4 * j] = a[0]; r[4 * j + 1] = a[1]; r[4 * j + 2] = a[2]; r[4 * j + 3] = a[3];
    }
}

__device__ __forceinline__ void mid_store(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
           "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
           "r"(r[15]) : "memory");
}

template <int CODE>
__global__ void __launch_bounds__(kMidThreads, 1)
linear_mid_kernel(const __grid_constant__ CUtensorMap rows, const MidArgs a) {
    extern __shared__ __align__(1024) uint8_t sm_raw[];
    __shared__ int fail;
    __shared__ uint32_t tmem_slot;
    uint8_t* sm = (uint8_t*)(((uintptr_t)sm_raw + 1023) & ~(uintptr_t)1023);
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    uint8_t* xs = sm;                                           // [stages][2][N][128 bytes]
    uint8_t* rings = sm + a.stages * a.N * 256;
    uint64_t* bars = reinterpret_cast<uint64_t*>(rings + kFewWarps * few_ring_bytes(a.K));
    const uint32_t xfull = shared_addr(bars), xempty = xfull + 32, afull = xfull + 64,
                   aempty = xfull + 96, dfull = xfull + 128, dempty = xfull + 136, done = xfull + 144;
    const int cta = blockIdx.x, kb = (int)a.run.kb.d;
    const int g0 = a.run.start(cta), count = a.run.start(cta + 1) - g0;
    int u0;
    const int b0 = a.run.kb.mod(g0, u0);
    if (t == 0) {
        for (int i = 0; i < 4; ++i) {
            bar_init(xfull + 8 * i, 1);
            bar_init(xempty + 8 * i, 1);
            bar_init(afull + 8 * i, 8);
            bar_init(aempty + 8 * i, 1);
        }
        bar_init(dfull, 1);
        bar_init(dempty, kFewWarps);
        bar_init(done, 1);
        fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kFewWarps) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;"
                     :: "r"(shared_addr(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_launch();

    if (warp < kFewWarps) {
        // ------------------------------------------------------------ decode
        const int grp = warp >> 3, quad = warp & 3, col = 2 * quad + ((warp >> 2) & 1);
        uint8_t* ring = rings + warp * few_ring_bytes(a.K);
        const uint32_t lanes = tmem + ((uint32_t)(16 * col) << 16);
        const uint32_t kt_bytes = (uint32_t)a.nbn * 256 * a.K;
        with_bits(a.K, [&](auto bits) {
            constexpr int K = decltype(bits)::value;
            FewStream<K> st(ring, lane);
            // issuing side: unit column and block of the group's next block to copy
            int iu = u0, ib = b0 + grp, ii = grp;
            auto settle = [&]() {
                while (ib >= kb) { ib -= kb; ++iu; }
                st.seek(a.trellis + (size_t)(iu % a.nbn) * 256 * K + (size_t)ib * 8 * kt_bytes +
                            (size_t)col * 32 * K, kt_bytes);
            };
            auto issue = [&](int stage) {
                if (ii < count) {
                    st.issue(stage);
                    ib += kFewGroups;
                    ii += kFewGroups;
                    if (ib >= kb) settle();
                    else st.src += (size_t)kFewGroups * 8 * kt_bytes;
                }
                cp_commit();
            };
            if (ii < count) settle();
#pragma unroll
            for (int s = 0; s < kFewStages - 1; ++s) issue(s);
            const LaneWindow<K> lw(lane);
            int cur = 0, fill = kFewStages - 1, i = grp, left = b0, unit = 0;
            bool ok = true;
            for (int lo = 0; lo < count && ok; ++unit) {       // units of this CTA
                const int hi = min(lo + kb - left, count);
                left = 0;
                for (; i < hi; i += kFewGroups) {
                    issue(fill);
                    cp_wait<kFewStages - 1>();
                    __syncwarp();
                    const uint32_t* tiles = reinterpret_cast<const uint32_t*>(ring + cur * 256 * K);
                    const int buf = i & 3, use = i >> 2;
                    const uint32_t to = lanes + kMidA + buf * 64;
                    uint32_t r[16];
                    mid_decode4<K, CODE>(tiles, lw, r);
                    if (use > 0) ok = bar_wait(aempty + 8 * buf, (use - 1) & 1, &fail, a.limit);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_fence_after();
                    mid_store(to, r);
                    mid_decode4<K, CODE>(tiles + 32 * K, lw, r);
                    mid_store(to + 32, r);
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(afull + 8 * buf);
                    fill = cur;
                    cur = cur + 1 == kFewStages ? 0 : cur + 1;
                }
                if (!ok) break;
                // the unit's sums: this warp's 32 columns, every fourth group of 32 rows
                ok = __all_sync(0xffffffffu, bar_wait(dfull, unit & 1, &fail, a.limit));
                if (!ok) break;
                tc_fence_after();
                const int u = u0 + unit, pass = u / a.nbn;
                const int have = min(a.N, a.M - pass * a.N);
                float* out = a.park + (size_t)(u + cta) * a.N * 128 + 32 * quad + lane;
                for (int r0 = (warp >> 2) * 32; r0 < have; r0 += 128) {
                    uint32_t d[32];
                    tc_load32(tmem + ((uint32_t)(32 * quad) << 16) + kMidAcc + r0, d);
                    tc_wait_ld();
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (r0 + j < have) out[(size_t)(r0 + j) * 128] = __uint_as_float(d[j]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(dempty);
                lo = hi;
            }
            cp_wait<0>();
            if (!ok && lane == 0) atomicExch(&fail, 1);
        });
    } else if (warp == kFewWarps) {
        // ------------------------------------------------------------ multiply
        if (lane == 0) {
            const uint32_t idesc = mma_desc_f16(128, a.N);
            const uint32_t xb = shared_addr(xs);
            bool ok = true;
            int left = b0, unit = 0, i = 0, xs_i = 0, xs_n = 0;
            for (int lo = 0; lo < count && ok; ++unit) {
                const int hi = min(lo + kb - left, count);
                left = 0;
                if (unit > 0) ok = bar_wait(dempty, (unit - 1) & 1, &fail, a.limit);
                for (; i < hi && ok; ++i) {
                    ok = bar_wait(xfull + 8 * xs_i, xs_n & 1, &fail, a.limit) &&
                         bar_wait(afull + 8 * (i & 3), (i >> 2) & 1, &fail, a.limit);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t at = tmem + kMidA + (i & 3) * 64, bt = xb + xs_i * a.N * 256;
#pragma unroll
                    for (int s = 0; s < 8; ++s) {
                        const uint64_t bd = operand_desc(bt + (s >> 2) * a.N * 128 + (s & 3) * 32);
                        asm volatile(
                            "{\n\t.reg .pred p;\n\t"
                            "setp.ne.b32 p, %4, 0;\n\t"
                            "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                            :: "r"(tmem + kMidAcc), "r"(at + 8 * s), "l"(bd), "r"(idesc),
                               "r"((uint32_t)(i > lo || s > 0)) : "memory");
                    }
                    tc_commit(aempty + 8 * (i & 3));
                    tc_commit(xempty + 8 * xs_i);
                    if (++xs_i == a.stages) { xs_i = 0; ++xs_n; }
                }
                if (ok) tc_commit(dfull);
                lo = hi;
            }
            if (!ok) atomicExch(&fail, 1);
            tc_commit(done);                   // tracks every MMA issued
            if (!bar_drain(done, 0)) atomicExch(&fail, 1);
        }
    } else if (lane == 0) {
        // ------------------------------------------------------------ load rows
        pdl_wait();                            // written by the kernel before,
        asm volatile("fence.proxy.async.global;" ::: "memory");    // through the generic proxy
        bool ok = true;
        int b = b0, u = u0, s = 0, n = 0, issued = 0;
        for (int i = 0; i < count; ++i) {
            if (n > 0) ok = bar_wait(xempty + 8 * s, (n - 1) & 1, &fail, a.limit);
            if (!ok) break;
            const uint32_t dst = shared_addr(xs) + s * a.N * 256, bar = xfull + 8 * s;
            const int y = u / a.nbn * a.N;
            bar_expect(bar, a.N * 256);
            tma_load(dst, &rows, b * 128, y, bar);
            tma_load(dst + a.N * 128, &rows, b * 128 + 64, y, bar);
            issued = i + 1;
            if (++b == kb) { b = 0; ++u; }
            if (++s == a.stages) { s = 0; ++n; }
        }
        if (!ok) atomicExch(&fail, 1);
        // every issued load lands before the shared memory is released
        for (int i = max(0, issued - a.stages); i < issued; ++i)
            bar_drain(xfull + 8 * (i % a.stages), (i / a.stages) & 1);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (t == 0 && fail) *(volatile int*)a.err = 1;
    if (warp == kFewWarps)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" :: "r"(tmem) : "memory");
}

}  // namespace exl3b
