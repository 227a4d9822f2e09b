// forward_few.cuh -- the few-rows product of the forward kernels: up to 8 G rows of
// activations times a 128-column block of an EXL3 tensor, decoded on the fly.
//
// Two groups of eight warps, one 16-column tile column each, walk the CTA's share of
// k in blocks of 128 (the Hadamard block), taking blocks in turn.  A warp streams its own tiles through a private
// cp.async ring in shared memory (no barrier between warps, nothing to wait for but
// its own copies) and multiplies them with mma.sync: up to 16 rows the product is
// bound by the decode's instruction issue (2.7 to 2.9 of 4 a cycle and SM; one row of 5120
// x 17408 at K = 5 27.5 us, of which the decode's issue is 18 and the trellis' bytes 9), not
// by the matrix unit, and mma.sync takes the decoded operand from the registers it was
// decoded into, without the trip through tensor memory that tcgen05 would need.
#pragma once
#include <atomic>

#include "exl3b_internal.h"
#include "trellis_mma.cuh"

namespace exl3b {

constexpr int kFewGroups = 2;         // groups of eight warps, taking k blocks in turn
constexpr int kFewWarps = 8 * kFewGroups;
constexpr int kFewStages = 3;         // weight ring of a warp, in blocks of 128 k
constexpr int kRowStages = 4;         // row ring of a group: one more, see few_run

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
// c mod 32 in turn.
template <int K>
struct FewStream {
    static constexpr int kPieces = (16 * K + 31) / 32;         // per lane
    const uint8_t* src;        // the next block's first tile, plus this lane's first piece
    uint32_t off[kPieces];     // its other pieces from there
    uint32_t dst;              // its place in the ring
    int lane;

    __device__ __forceinline__ FewStream(uint8_t* ring, int lane_) : lane(lane_) {
        dst = (uint32_t)__cvta_generic_to_shared(ring) + 16 * lane;
    }
    // Go on at the block whose first tile is at `tile`, `kt_bytes` between k tiles.
    __device__ __forceinline__ void seek(const uint8_t* tile, uint32_t kt_bytes) {
        uint32_t first = 0;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int c = lane + 32 * i, kt = c / (2 * K);
            const uint32_t o = kt * kt_bytes + 16 * (c - kt * 2 * K);
            if (i == 0) first = o;
            off[i] = o - first;
        }
        src = tile + first;
    }
    // Copy that block into stage `stage` of the ring.
    __device__ __forceinline__ void issue(int stage) const {
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
            if (16 * K % 32 == 0 || i + 1 < kPieces || lane + 32 * i < 16 * K)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                             :: "r"(dst + stage * 256 * K + 512 * i), "l"(src + off[i]) : "memory");
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
// matrix instruction needs; bf16 would cost three bits of the activations.  With LO,
// what the rounding left is stored as well, at dst + lo, rounded to fp16 itself: the
// pair holds 22 bits of the values (to 2^-25 of the block's largest).
template <bool LO = false>
__device__ __forceinline__ void few_put_block(float (&v)[4], uint8_t* dst, float* inv_scale,
                                              int lane, int swz, size_t lo = 0) {
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
    if constexpr (LO) {
        const float2 fa = __half22float2(a), fb = __half22float2(b);
        *reinterpret_cast<__half2*>(dst + lo + ((2 * off) ^ swz)) =
            __floats2half2_rn(v[0] - fa.x, v[1] - fa.y);
        *reinterpret_cast<__half2*>(dst + lo + ((2 * off + 16) ^ swz)) =
            __floats2half2_rn(v[2] - fb.x, v[3] - fb.y);
    }
    if (lane == 0) *inv_scale = inv;
}

// acc[g][..] += one k block: the warp's eight tiles at `tiles`, rows 8 g .. 8 g + 7 of
// the block at `xh` (with LO, their remainders 8 G rows on), reciprocal scales inv [8 G].
template <int K, int CODE, int G, bool LO>
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
        constexpr int N = LO ? 2 * G : G;
        uint4 x[N];
#pragma unroll
        for (int g = 0; g < N; ++g)
            x[g] = *reinterpret_cast<const uint4*>((p & 1 ? odd : even) + g * 8 * kRowBytes + p * 64);
        uint32_t a[4];
        decode_tile<K, CODE>(tiles + (2 * p) * 8 * K, lw, a);
#pragma unroll
        for (int g = 0; g < N; ++g) mma_16816(blk[g % G], a, x[g].x, x[g].y);
        decode_tile<K, CODE>(tiles + (2 * p + 1) * 8 * K, lw, a);
#pragma unroll
        for (int g = 0; g < N; ++g) mma_16816(blk[g % G], a, x[g].z, x[g].w);
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

// Division of an int >= 0 by a divisor known ahead: q = mulhi and shifts (the
// round-up method of Granlund and Montgomery, exact for all 32-bit dividends).
struct FastDiv {
    uint32_t d, mul, sh1, sh2;
    __host__ __device__ FastDiv() {}
    __host__ __device__ explicit FastDiv(uint32_t d_) : d(d_) {
        uint32_t l = 0;
        while (l < 32 && (1ull << l) < d) ++l;
        mul = (uint32_t)((((1ull << l) - d) << 32) / d) + 1;
        sh1 = l < 1 ? l : 1;
        sh2 = l > 1 ? l - 1 : 0;
    }
    __device__ __forceinline__ int div(int n) const {
        const uint32_t t = __umulhi(mul, (uint32_t)n);
        return (int)((t + (((uint32_t)n - t) >> sh1)) >> sh2);
    }
    // n = q * d + returned remainder
    __device__ __forceinline__ int mod(int n, int& q) const {
        q = div(n);
        return n - q * (int)d;
    }
};

struct FewRun {
    int units, ctas;
    int least, longer;         // blocks of a CTA's run; the first `longer` have one more
    FastDiv kb;                // blocks of a unit
    __host__ __device__ FewRun() {}
    __host__ __device__ FewRun(const FastDiv& kb_, int units_, int sms) : units(units_), kb(kb_) {
        const int total = (int)kb.d * units;
        ctas = total < sms ? total : sms;
        least = ctas ? total / ctas : 0;
        longer = ctas ? total % ctas : 0;
    }
    __host__ __device__ int start(int cta) const { return cta * least + (cta < longer ? cta : longer); }
};

// A run as the joining kernels see it: which CTA's run holds block g.
struct FewJoin {
    FewRun run;
    FastDiv least, more;       // by the blocks of the short runs and of the longer ones
    __host__ __device__ FewJoin() {}
    __host__ explicit FewJoin(const FewRun& r)
        : run(r), least(r.least ? r.least : 1), more(r.least + 1) {}
    __device__ __forceinline__ int owner(int g) const {
        const int head = run.longer * (run.least + 1);
        return g < head ? more.div(g) : run.longer + least.div(g - head);
    }
};

// Parked sums: CTA c's of unit u at slot u + c (along the sequence u or c grows, so
// the slots differ), per group [8 G rows][128 columns].
__host__ __device__ inline size_t few_park_bytes(int units, int ctas, int G) {
    return (size_t)(units + ctas) * kFewGroups * 8 * G * 512;
}

// Shared memory of the product: weight rings, then the rows -- rings of kRowStages
// blocks per group, or (rotated in place) all `blocks` of the run.
constexpr int kFewRoom = 222 * 1024;      // of the 227 KB a CTA may have
__host__ __device__ inline int few_smem(int Kmax, int G, int blocks, bool lo = false) {
    return kFewWarps * few_ring_bytes(Kmax) + blocks * 8 * G * ((lo ? 2 : 1) * kRowBytes + 4);
}

// A job tells what the units are.  Its Cursor stands at one unit: tiles (first tile of
// the column block), kt_bytes (to the next k tile), K.
//   cursor(u), next(cursor)   the weight of unit u, of the one after it
//   rows(u)                   its rows, at most 8 G
// and, unless kRotate,
//   row(u, r) -> index of block 0 of the unit's row r among the rotated blocks (256
//                bytes each at xh(), reciprocal scales at inv()); block b is b * kRowStep on
//   lo()      with kLo, bytes from a rotated block to its remainders
//   wait()    -> returns once the rows are there
// or, with kRotate (every unit has the same rows),
//   rotate(r, b, dst, inv, swz)   puts block b of row r itself (a warp), with kLo its
//                                 remainders 8 G rows on

// Multiply this CTA's run and park the sums.  All threads.
//
// Each iteration of a group is one block: every warp copies its tiles of the block two
// ahead into its own ring and the group's warps share the copy of that block's rows;
// then the group meets at a barrier, which makes the rows of the present block visible
// to all and tells that the block before is read, so that its place may be refilled in
// the next iteration -- hence a row ring one deeper than the distance needs.
template <int CODE, int G, typename Job>
__device__ __forceinline__ void few_run(const Job& job, const FewRun& run, int Kmax, uint8_t* sm,
                                        float* park) {
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31, grp = warp >> 3, col = warp & 7;
    const int cta = blockIdx.x, g0 = run.start(cta), count = run.start(cta + 1) - g0;
    const int kb = (int)run.kb.d;
    uint8_t* ring = sm + warp * few_ring_bytes(Kmax);
    const int blocks = Job::kRotate ? count : kFewGroups * kRowStages;
    constexpr bool LO = Job::kLo;
    constexpr int kBlockBytes = 8 * G * (LO ? 2 : 1) * kRowBytes;
    uint8_t* xh = sm + kFewWarps * few_ring_bytes(Kmax);
    float* inv = reinterpret_cast<float*>(xh + blocks * kBlockBytes);
    const int mine = Job::kRotate ? 0 : grp * kRowStages;      // the group's first row stage
    int u0;
    const int b0 = run.kb.mod(g0, u0);
    float acc[G][4];
#pragma unroll
    for (int g = 0; g < G; ++g) acc[g][0] = acc[g][1] = acc[g][2] = acc[g][3] = 0.0f;
    int i = grp;                              // this group's next block of the run
    int u;                                    // its unit and block there
    int b = run.kb.mod(b0 + i, u);
    u += u0;
    auto at = job.cursor(u);
    bool waited = false;
    // this warp's rows of a block: G, sixteen lanes each; a single row's remainders by
    // the other sixteen
    constexpr bool kHalves = LO && G == 1;
    const int rr = G == 1 ? col : 2 * col + (lane >> 4);
    const uint32_t rdst = (uint32_t)__cvta_generic_to_shared(xh) + mine * kBlockBytes + rr * kRowBytes +
                          few_swizzle(rr, 16 * (lane & 15)) + (kHalves ? (lane >> 4) * 8 * kRowBytes : 0);
    const uint32_t idst = (uint32_t)__cvta_generic_to_shared(inv) + 4 * (mine * 8 * G + rr);
    // Stretches of equal bit width: the weight ring restarts where it changes.
    while (i < count) {
        with_bits(at.K, [&](auto bits) {
            constexpr int K = decltype(bits)::value;
            // the issuing side runs kFewStages - 1 of the group's blocks ahead: `left`
            // blocks of unit `to`, 0 once there are no more of this width
            auto to = at;
            int iu = u, ib = b, ii = i, left = 0;
            size_t step = 0;
            [[maybe_unused]] size_t xstep = 0;
            [[maybe_unused]] const uint8_t* xsrc = nullptr;    // this lane's piece of its row there
            [[maybe_unused]] const float* isrc = nullptr;
            [[maybe_unused]] bool has = false;
            FewStream<K> st(ring, lane);
            auto seek = [&]() {
                left = (min(kb - ib, count - ii) + kFewGroups - 1) / kFewGroups;
                st.seek(to.tiles + (size_t)ib * 8 * to.kt_bytes + (size_t)col * 32 * K, to.kt_bytes);
                step = (size_t)kFewGroups * 8 * to.kt_bytes;
                if constexpr (!Job::kRotate) {
                    has = rr < job.rows(iu) && (G == 2 || LO || lane < 16);
                    if (has) {
                        const size_t from = job.row(iu, rr) + (size_t)ib * job.row_step();
                        xsrc = job.xh() + from * kRowBytes + 16 * (lane & 15);
                        if constexpr (kHalves) xsrc += lane < 16 ? 0 : job.lo();
                        isrc = job.inv() + from;
                    }
                    xstep = (size_t)kFewGroups * job.row_step();
                }
            };
            // rows past the unit's last stay unwritten: a row is a column of the matrix
            // instruction, and only rows that exist are read back
            auto issue_rows = [&](int stage) {
                if constexpr (!Job::kRotate) {
                    if (has) {
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                                     :: "r"(rdst + stage * kBlockBytes), "l"(xsrc) : "memory");
                        if constexpr (LO && G == 2)
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                                         :: "r"(rdst + stage * kBlockBytes + 8 * G * kRowBytes),
                                            "l"(xsrc + job.lo()) : "memory");
                        if (kHalves ? lane == 0 : (lane & 15) == 0)
                            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;"
                                         :: "r"(idst + stage * 32 * G), "l"(isrc) : "memory");
                        xsrc += xstep * kRowBytes;
                        isrc += xstep;
                    }
                }
            };
            auto issued = [&](int n) {
                left -= n;
                ib += n * kFewGroups;
                ii += n * kFewGroups;
                if (left > 0 || ii >= count) return;
                while (ib >= kb) { ib -= kb; ++iu; job.next(to); }
                if (to.K != K) { ii = count; return; }
                seek();
            };
            seek();
            if (!waited) {
                // the weights do not depend on the kernel before; the rows do
                st.issue(0);
                if constexpr (Job::kRotate) {
                    for (int j = warp; j < count * job.rows(0); j += kFewWarps) {
                        const int rows = job.rows(0), blk = rows == 1 ? j : j >> 1, r = j - blk * rows;
                        int q;
                        const int kblk = run.kb.mod(b0 + blk, q);
                        job.rotate(r, kblk, xh + blk * kBlockBytes + r * kRowBytes, inv + blk * 8 * G + r,
                                   (r & 1) << 6);
                    }
                    __syncthreads();
                } else {
                    job.wait();
                }
            } else {
                // the group's warps have all read the last block of the stretch before
                asm volatile("bar.sync %0, 256;" :: "r"(1 + grp) : "memory");
            }
#pragma unroll
            for (int s = 0; s < kFewStages - 1; ++s) {
                if (left > 0) {
                    if (s > 0 || waited) st.issue(s);
                    issue_rows(s);
                    st.src += step;
                    issued(1);
                }
                cp_commit();
            }
            waited = true;
            const LaneWindow<K> lw(lane);
            int cur = 0, fill = kFewStages - 1, rcur = 0;
            while (true) {
                // blocks until the unit, the run or the issued unit ends
                int n = (min(kb - b, count - i) + kFewGroups - 1) / kFewGroups;
                const bool feed = left > 0;
                if (feed) n = min(n, left);
                const int from = Job::kRotate ? i : mine;
                const uint8_t* x = xh + from * kBlockBytes;
                const float* f = inv + from * 8 * G;
#pragma unroll 1
                for (int j = 0; j < n; ++j) {
                    if (feed) {
                        st.issue(fill);
                        st.src += step;
                        issue_rows((rcur + kFewStages - 1) & (kRowStages - 1));
                    }
                    cp_commit();
                    cp_wait<kFewStages - 1>();
                    if constexpr (Job::kRotate) {
                        __syncwarp();
                        few_block<K, CODE, G, LO>(lw, ring + cur * 256 * K, x, f, acc, lane);
                        x += kFewGroups * kBlockBytes;
                        f += kFewGroups * 8 * G;
                        __syncwarp();      // every lane has read the stage before it is refilled
                    } else {
                        asm volatile("bar.sync %0, 256;" :: "r"(1 + grp) : "memory");
                        few_block<K, CODE, G, LO>(lw, ring + cur * 256 * K, x + rcur * kBlockBytes,
                                                  f + rcur * 8 * G, acc, lane);
                        rcur = (rcur + 1) & (kRowStages - 1);
                        __syncwarp();
                    }
                    fill = cur;
                    cur = cur + 1 == kFewStages ? 0 : cur + 1;
                }
                if (feed) issued(n);
                i += n * kFewGroups;
                b += n * kFewGroups;
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
                while (b >= kb) { b -= kb; ++u; job.next(at); }
                if (at.K != K) break;
            }
            cp_wait<0>();
            __syncwarp();
        });
    }
    // a group without a block meets the others all the same
    if (Job::kRotate && !waited) {
        __syncthreads();
    }
}

// The parked sums of unit u: GROUPS per CTA of its run.
template <int GROUPS>
struct FewParts {
    int lo, hi, c0, n;
    __device__ __forceinline__ FewParts(const FewJoin& j, int u) {
        lo = u * (int)j.run.kb.d;
        hi = lo + (int)j.run.kb.d;
        c0 = j.owner(lo);
        n = (j.owner(hi - 1) - c0 + 1) * GROUPS;
    }
};

// Sum of unit u's parked sums of row r (of `rows` a slot), elements 4 lane ..
// 4 lane + 3: the ones at `part`, part + parts, ... in the order of the CTAs and their
// groups.  A warp.
template <int GROUPS>
__device__ __forceinline__ void few_sum(const float* park, const FewJoin& join, const FewParts<GROUPS>& p,
                                        int u, int rows, int r, int lane, int part, int parts,
                                        float (&v)[4]) {
    const size_t slot = (size_t)rows * 128;
    const float* from = park + (size_t)(u + p.c0) * GROUPS * slot + r * 128 + 4 * lane;
    v[0] = v[1] = v[2] = v[3] = 0.0f;
#pragma unroll 4
    for (int i = part; i < p.n; i += parts) {
        if (GROUPS > 1) {
            const int c = p.c0 + i / GROUPS, g = i % GROUPS;
            const int s = join.run.start(c), e = join.run.start(c + 1);
            const int f = s > p.lo ? s : p.lo, l = e < p.hi ? e : p.hi;      // the CTA's blocks of u
            // a group takes every other block of the run: none of a single one, maybe
            if (l - f < GROUPS && ((f - s) & 1) != g) continue;
        }
        const float4 q = __ldcg(reinterpret_cast<const float4*>(from + i * slot));
        v[0] += q.x; v[1] += q.y; v[2] += q.z; v[3] += q.w;
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

// The kernel attributes of a launch, set once per kernel and device: shared memory up to
// what a CTA may have, and the same split of L1 for all, since a kernel that wants
// another waits for the SM to empty.  (Setting them again is harmless: two threads may.)
template <typename... P>
int prepare_kernel(void (*kern)(P...), const char* what, std::atomic<uint64_t>& done) {
    int dev = 0;
    if (check_cuda(cudaGetDevice(&dev), what)) return RC_DEVICE_ERROR;
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_acquire) & bit) return RC_OK;
    cudaFuncAttributes fa;
    if (check_cuda(cudaFuncGetAttributes(&fa, kern), what) ||
        check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        227 * 1024 - (int)fa.sharedSizeBytes), what) ||
        check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout,
                                        cudaSharedmemCarveoutMaxShared), what))
        return RC_DEVICE_ERROR;
    done.fetch_or(bit, std::memory_order_release);
    return RC_OK;
}

template <auto Kern, typename... A>
int launch_kernel(const char* what, dim3 grid, int threads, size_t smem, bool pdl, cudaStream_t stream,
                  A... args) {
    static std::atomic<uint64_t> done{0};
    if (prepare_kernel(Kern, what, done)) return RC_DEVICE_ERROR;
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
    const cudaError_t e = cudaLaunchKernelEx(&cfg, Kern, args...);
    note_launch();
    return check_cuda(e, what) ? RC_DEVICE_ERROR : RC_OK;
}

}  // namespace exl3b
