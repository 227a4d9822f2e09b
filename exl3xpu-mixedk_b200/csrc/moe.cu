// moe.cu -- mixture-of-experts layer for a few tokens, experts held as EXL3 tensors:
//   l = x R^T;  S = the top_k largest l (ties: lowest index);  p = softmax(l)
//   y = sum_{e in S} w_e ((silu(x Wg_e) * (x Wu_e)) Wd_e) + residual,  w = p or p / sum_S p
//
// Six launches, every one but the first started while the one before still runs: the
// router (logits, choice, weights); the chosen experts' rotations of the tokens, and
// the plan of the products; the gate and up products of every chosen expert; their
// join, to the down projection's rotated rows; the down products; their join, to the
// weighted sum.  Each chosen expert's tensors are read once for 8 G of its tokens; the work is
// bound by their decode, spread evenly over the SMs as in forward_few.cuh.  Nothing depends on
// the order in which CTAs run: partial sums are added in a fixed order, and a token's
// experts in the order of their choice.
#include <cooperative_groups.h>
#include <string.h>

#include <utility>

#include "forward_few.cuh"
#include "../../include/exl3b200.h"

namespace cg = cooperative_groups;

namespace exl3b {

constexpr int kMaxExperts = 1024;
constexpr int kMaxTokens = 256;
constexpr int kMaxTopK = 32;
constexpr int kMaxPairs = 2048;           // (token, choice) pairs of one call
constexpr int kMaxWidth = 1 << 16;        // D and F: blocks are counted in 32 bits

// What the later kernels need of a chosen expert.
struct Chosen {
    const uint8_t* tiles[3];              // gate, up, down
    const __half* svh[3];
    const __half* suh[3];
    int K[3];
    int expert;
};

struct MoeArgs {
    const void* x;
    int64_t ldx;
    int dtype;
    int T, D, F, E, top_k, normalize;
    FastDiv kd, kf;                       // blocks of D and of F
    const void* router;
    int64_t ldr;
    int router_dtype;                     // 0 fp32, else XType
    const exl3b_expert* experts;          // [3][E] gate, up, down
    int Kmax[3];
    const void* residual;
    int64_t ldres;
    void* out;
    int64_t ldo;
    // workspace
    int slots_max;                        // experts x groups of 8 G rows at most
    Chosen* chosen;                       // [T * top_k]
    float* wts;                           // [T * top_k]
    int* place;                           // [T * top_k] slot << 8 | row of a pair
    uint8_t* plan;                        // PlanHead and arrays
    int ctas1, ctas2;                     // of the products
    uint8_t* xh1;                         // [2][T * top_k][D / 128][256], few_put_block order, and
    float* inv1;                          //   as much again for the remainders (LO)
    uint8_t* xh2;                         // [T * top_k][F / 128][256], and the remainders
    float* inv2;
    float* park;
};

// The line of p to L2: any address will do (a bulk prefetch would want 16-byte ones,
// and suh and svh are 8-byte aligned).
__device__ __forceinline__ void prefetch_line(const void* p) {
    asm volatile("prefetch.global.L2 [%0];" :: "l"(p));
}

// ------------------------------------------------------------------ router
constexpr int kRouterRanks = 4;            // CTAs of a cluster
constexpr int kRouterWarps = 16;
constexpr int kRouterThreads = 32 * kRouterWarps;

// A sum kept as a pair of fp32 (its value and the rounding errors' sum).  The choice of
// experts must not hang on the batch, so a logit is always summed in the same order,
// nor on how long a row is: eight products at a time are summed in fp32, those sums
// without loss.  What is left are the eights' own roundings, as a root of mean squares
// 2^-26 of the logits' for bf16 tensors and 2^-24.4 for fp16 ones or an fp32 router, at
// any D.  (fp64 additions and conversions run at a 1/64 of the fp32 rate here: 7 us a
// token; the lossless sum of every product cost 3 us more than this at 64 tokens.)
struct PairSum {
    float s = 0.0f, c = 0.0f;
    __device__ __forceinline__ void add(float p) {      // two-sum (Knuth)
        const float t = s + p, q = t - s;
        c += (s - (t - q)) + (p - q);
        s = t;
    }
    // (an infinite sum has no meaningful error term)
    __device__ __forceinline__ double value() const { return c != c ? (double)s : (double)s + (double)c; }
};

__device__ __forceinline__ void unpack8(const uint4& v, int dtype, float (&x)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t u = (&v.x)[j];
        if (dtype == X_BF16) {
            x[2 * j] = __uint_as_float(u << 16);
            x[2 * j + 1] = __uint_as_float(u & 0xFFFF0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
            x[2 * j] = f.x;
            x[2 * j + 1] = f.y;
        }
    }
}

// Eight elements of a router row, as stored.
template <bool F32> struct RouterPiece { uint4 v[F32 ? 2 : 1]; };

template <bool F32>
__device__ __forceinline__ RouterPiece<F32> load_router(const MoeArgs& a, size_t off) {
    RouterPiece<F32> p;
    const uint4* from = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.router) +
                                                       off * (F32 ? 4 : 2));
    p.v[0] = __ldg(from);
    if (F32) p.v[F32] = __ldg(from + 1);
    return p;
}

// acc += 8 products of x and a router row.
template <bool F32>
__device__ __forceinline__ void dot8(const MoeArgs& a, const float (&x)[8], const RouterPiece<F32>& p,
                                     PairSum& acc) {
    float r[8];
    if (F32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = __uint_as_float((&p.v[F32 ? j >> 2 : 0].x)[j & 3]);
    } else {
        unpack8(p.v[0], a.dtype, r);
    }
    float q0 = x[0] * r[0], q1 = x[1] * r[1];
#pragma unroll
    for (int j = 2; j < 8; j += 2) {
        q0 = fmaf(x[j], r[j], q0);
        q1 = fmaf(x[j + 1], r[j + 1], q1);
    }
    acc.add(q0 + q1);
}

// Logits of TT tokens (x rows at xr, pitch ldx elements) for experts e0 and, with EE = 2
// and `two`, e1.  A warp.  The router's rows come from memory, so kBatch pieces of 256
// columns are asked for before the first is used.
template <bool F32, int TT, int EE>
__device__ __forceinline__ void logits(const MoeArgs& a, const uint16_t* xr, int tokens, int e0, int e1,
                                       bool two, double (&out)[EE][TT]) {
    constexpr int kBatch = F32 ? 4 : 8;
    const int lane = threadIdx.x & 31, n = a.D >> 3;
    PairSum sum[EE][TT];
    for (int c0 = lane; c0 < n; c0 += 32 * kBatch) {
        RouterPiece<F32> r[EE][kBatch];
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
            const int c = c0 + 32 * q;
            if (c < n) {
                r[0][q] = load_router<F32>(a, (size_t)e0 * a.ldr + 8 * c);
                if (EE == 2 && two) r[EE - 1][q] = load_router<F32>(a, (size_t)e1 * a.ldr + 8 * c);
            }
        }
#pragma unroll
        for (int k = 0; k < TT; ++k) {
            if (k >= tokens) break;
            uint4 xv[kBatch];
#pragma unroll
            for (int q = 0; q < kBatch; ++q)
                if (c0 + 32 * q < n)
                    xv[q] = __ldg(reinterpret_cast<const uint4*>(xr + (size_t)k * a.ldx) + c0 + 32 * q);
#pragma unroll
            for (int q = 0; q < kBatch; ++q) {
                if (c0 + 32 * q < n) {
                    float x[8];
                    unpack8(xv[q], a.dtype, x);
                    dot8<F32>(a, x, r[0][q], sum[0][k]);
                    if (EE == 2 && two) dot8<F32>(a, x, r[EE - 1][q], sum[EE - 1][k]);
                }
            }
        }
    }
#pragma unroll
    for (int e = 0; e < EE; ++e)
#pragma unroll
        for (int k = 0; k < TT; ++k) {
            out[e][k] = sum[e][k].value();
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) out[e][k] += __shfl_xor_sync(0xffffffffu, out[e][k], o);
        }
}

// An order on fp64 values as integers; NaN counts as largest (its weights are NaN
// whatever is chosen), -0 as 0.
__device__ __forceinline__ long long order_key(long long bits) {
    const long long mag = bits & 0x7FFFFFFFFFFFFFFFLL;
    if (mag > 0x7FF0000000000000LL) return 0x7FFFFFFFFFFFFFFFLL;
    return bits < 0 ? -mag : mag;
}

__device__ __forceinline__ uint32_t peer(const void* p, int rank) {
    uint32_t addr;
    asm("mapa.shared::cluster.u32 %0, %1, %2;"
        : "=r"(addr) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return addr;
}

// Cluster (4 CTAs) per TT tokens.  Its 64 warps share the experts' logits, which go to
// every CTA; the CTAs share the experts again to find their places in the order (the
// number of larger logits, and of equal ones before); an expert placed below top_k is
// chosen.
template <bool F32, int TT>
__global__ void __cluster_dims__(kRouterRanks, 1, 1) __launch_bounds__(kRouterThreads, 1)
moe_router_kernel(const MoeArgs a) {
    __shared__ long long logit[TT][kMaxExperts];      // fp64 bits
    __shared__ int chosen[TT][kMaxTopK];
    __shared__ float share[TT][kMaxTopK];
    __shared__ double largest[TT];
    __shared__ float total[TT];
    pdl_launch();
    cg::cluster_group cl = cg::this_cluster();
    auto started = cl.barrier_arrive();
    const int rank = cl.block_rank(), token0 = blockIdx.y * TT, t = threadIdx.x;
    const int warp = t >> 5, lane = t & 31, tokens = min(TT, a.T - token0);
    const uint16_t* xr = static_cast<const uint16_t*>(a.x) + (size_t)token0 * a.ldx;
    constexpr int EE = TT == 1 ? 2 : 1, kWarps = kRouterRanks * kRouterWarps;
    // the experts' table is wanted soon, and has left the cache since the last call
    for (int i = t * 128; i < 3 * a.E * (int)sizeof(exl3b_expert); i += kRouterThreads * 128)
        prefetch_line(reinterpret_cast<const uint8_t*>(a.experts) + i);
    bool wait = true;
    for (int e0 = rank * kRouterWarps + warp; e0 < a.E; e0 += EE * kWarps) {
        const int e1 = e0 + kWarps;
        const bool two = EE == 2 && e1 < a.E;
        double l[EE][TT];
        logits<F32, TT, EE>(a, xr, tokens, e0, e1, two, l);
        if (wait) { cl.barrier_wait(std::move(started)); wait = false; }   // the others run
        if (lane < kRouterRanks) {
#pragma unroll
            for (int k = 0; k < TT; ++k) {
                asm volatile("st.shared::cluster.f64 [%0], %1;"
                             :: "r"(peer(&logit[k][e0], lane)), "d"(l[0][k]) : "memory");
                if (two)
                    asm volatile("st.shared::cluster.f64 [%0], %1;"
                                 :: "r"(peer(&logit[k][e1], lane)), "d"(l[EE - 1][k]) : "memory");
            }
        }
    }
    if (wait) cl.barrier_wait(std::move(started));
    cl.sync();
    if (warp < tokens) {       // largest logit and softmax sum
        double m = -INFINITY;
        for (int e = lane; e < a.E; e += 32) m = fmax(m, __longlong_as_double(logit[warp][e]));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
        float sum = 0.0f;
        for (int e = lane; e < a.E; e += 32)
            sum += expf((float)(__longlong_as_double(logit[warp][e]) - m));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) { largest[warp] = m; total[warp] = sum; }
    }
    // 16 lanes count for one expert
    const int q = t & 15, shared = (a.E + kRouterRanks - 1) / kRouterRanks;
    for (int k = 0; k < tokens; ++k) {
        for (int i0 = 0; i0 < shared; i0 += 2 * kRouterWarps) {
            const int e = (i0 + (t >> 4)) * kRouterRanks + rank;
            int place = 0;
            if (e < a.E) {
                const long long mine = order_key(logit[k][e]);
                for (int o = q; o < a.E; o += 16) {
                    const long long key = order_key(logit[k][o]);
                    place += key > mine || (key == mine && o < e);
                }
            }
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
            if (e < a.E && place < a.top_k && q < kRouterRanks)
                asm volatile("st.shared::cluster.s32 [%0], %1;"
                             :: "r"(peer(&chosen[k][place], q)), "r"(e) : "memory");
        }
    }
    cl.sync();
    // what is kept of token `rank`: a warp
    for (int k = rank; k < tokens; k += kRouterRanks) {
        if (warp != k / kRouterRanks || lane >= a.top_k) continue;
        const int e = chosen[k][lane], to = (token0 + k) * a.top_k + lane;
        Chosen c;
#pragma unroll
        for (int m = 0; m < 3; ++m) {
            const exl3b_expert w = a.experts[(size_t)m * a.E + e];
            c.tiles[m] = static_cast<const uint8_t*>(w.trellis);
            c.svh[m] = static_cast<const __half*>(w.svh);
            c.suh[m] = static_cast<const __half*>(w.suh);
            c.K[m] = min(max(w.K, 2), a.Kmax[m]);
        }
        c.expert = e;
        a.chosen[to] = c;
        const float p = expf((float)(__longlong_as_double(logit[k][e]) - largest[k])) / total[k];
        float sum = p;
        if (a.normalize) {
            share[k][lane] = p;
            __syncwarp(a.top_k == 32 ? 0xffffffffu : (1u << a.top_k) - 1);
            sum = 0.0f;
            for (int j = 0; j < a.top_k; ++j) sum += share[k][j];
        }
        a.wts[to] = a.normalize ? p / sum : p;
    }
}

// ------------------------------------------------------------------ experts
// The chosen experts in ascending order, each cut into slots of up to 8 G of its
// (token, choice) pairs, which are in ascending order too; with the tensors of the
// slots' experts.  Made once, in device memory; the products copy it to shared memory.
struct PlanHead {
    FewJoin join[2];           // the products' runs
    int slots;
};

struct Plan {
    const PlanHead* head;
    int* pair;                 // [P]
    int2* slot;                // [slots_max] {expert, first pair << 8 | rows}
    const uint8_t** tiles;     // [3][slots_max + 1]
    int* K;                    // [3][slots_max + 1]
};

__host__ __device__ inline int up16(int b) { return (b + 15) & ~15; }
__host__ __device__ inline int plan_bytes(int P, int slots_max) {
    return up16(sizeof(PlanHead)) + up16(P * 4) + up16(slots_max * 8) + up16(36 * (slots_max + 1));
}
__device__ __forceinline__ Plan plan_at(uint8_t* where, int P, int slots_max) {
    Plan p;
    p.head = reinterpret_cast<const PlanHead*>(where);
    where += up16(sizeof(PlanHead));
    p.pair = reinterpret_cast<int*>(where);
    where += up16(P * 4);
    p.slot = reinterpret_cast<int2*>(where);
    where += up16(slots_max * 8);
    p.tiles = reinterpret_cast<const uint8_t**>(where);
    p.K = reinterpret_cast<int*>(where + 24 * (slots_max + 1));
    return p;
}

constexpr int kPlanThreads = 512;

// Shared memory of make_plan, each part from a 16-byte boundary to the next.
struct PlanScratch {
    int from, before, bytes;   // `where` begins at 0
    __host__ __device__ PlanScratch(int P, int E)
        : from(up16(P * 4)), before(from + up16(E * 8)), bytes(before + up16((P + 31) / 32 * E)) {}
};

// One CTA of kPlanThreads; `tmp`: PlanScratch::bytes of shared memory.
template <int G>
__device__ __forceinline__ void make_plan(const MoeArgs& a, uint8_t* tmp) {
    __shared__ int totals[kPlanThreads / 32];
    constexpr int kWarps = kPlanThreads / 32;
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31, P = a.T * a.top_k, chunks = (P + 31) / 32;
    const Plan p = plan_at(a.plan, P, a.slots_max);
    const PlanScratch at(P, a.E);
    int* where = reinterpret_cast<int*>(tmp);                   // [P] expert << 8 | place in its chunk
    int* from = reinterpret_cast<int*>(tmp + at.from);          // [E] an expert's first pair and slot
    int* count = from + a.E;                                    // [E] its pairs
    uint8_t* before = tmp + at.before;                          // [chunks][E] then running
    Chosen own;
    if (t < P) own = a.chosen[t];
    for (int i = at.before + 16 * t; i < at.bytes; i += 16 * kPlanThreads)
        *reinterpret_cast<uint4*>(tmp + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    // 32 pairs a warp: how many of the same expert come before a pair there
    for (int c = warp; c < chunks; c += kWarps) {
        const int i = c * 32 + lane;
        const int e = i >= P ? -1 : i == t ? own.expert : a.chosen[i].expert;
        const uint32_t same = __match_any_sync(0xffffffffu, e);
        if (e >= 0) {
            where[i] = e << 8 | __popc(same & ((1u << lane) - 1));
            if ((same >> lane) == 1) before[c * a.E + e] = (uint8_t)__popc(same);
        }
    }
    __syncthreads();
    // and how many in the chunks before; a count of more than 255 lies in the last sum
    // only, since an expert has at most T pairs, T <= 256, and the last chunk's is not added
    const int e0 = 2 * t;
    int c2[2] = {0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (e0 + h < a.E) {
            int sum = 0;
            for (int c = 0; c < chunks; ++c) {
                const int x = before[c * a.E + e0 + h];
                before[c * a.E + e0 + h] = (uint8_t)sum;
                sum += x;
            }
            c2[h] = sum;
            count[e0 + h] = sum;
        }
    // running sums over two experts a thread: pairs in the low half, slots in the high
    const int m0 = c2[0] | (c2[0] + 8 * G - 1) / (8 * G) << 16, m1 = c2[1] | (c2[1] + 8 * G - 1) / (8 * G) << 16;
    int sum = m0 + m1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
    }
    if (lane == 31) totals[warp] = sum;
    __syncthreads();
    int base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        const int x = totals[w];
        if (w < warp) base += x;
        all += x;
    }
    const int slots = all >> 16, at0 = base + sum - m0 - m1;
    if (e0 < a.E) from[e0] = at0;
    if (e0 + 1 < a.E) from[e0 + 1] = at0 + m0;
    if (warp == kWarps - 1 && lane < 4) {      // the products' runs: a divisor a lane
        const bool down = lane >= 2;
        const FewRun run = down ? FewRun(a.kf, slots * (int)a.kd.d, a.ctas2)
                                : FewRun(a.kd, 2 * slots * (int)a.kf.d, a.ctas1);
        const FastDiv d(lane & 1 ? run.least + 1 : run.least);
        PlanHead* h = const_cast<PlanHead*>(p.head);
        FewJoin* join = h->join + (down ? 1 : 0);
        if (lane & 1) join->more = d;
        else { join->run = run; join->least = d; }
        if (lane == 0) h->slots = slots;
    }
    __syncthreads();
    for (int i = t; i < P; i += kPlanThreads) {
        const int e = where[i] >> 8, f = from[e], r = before[(i >> 5) * a.E + e] + (where[i] & 0xFF);
        const int slot = (f >> 16) + r / (8 * G);
        p.pair[(f & 0xFFFF) + r] = i;
        a.place[i] = slot << 8 | r % (8 * G);
        if (r % (8 * G)) continue;
        p.slot[slot] = make_int2(e, ((f & 0xFFFF) + r) << 8 | min(8 * G, count[e] - r));
#pragma unroll
        for (int m = 0; m < 3; ++m) {
            p.tiles[m * (a.slots_max + 1) + slot] = i == t ? own.tiles[m] : a.chosen[i].tiles[m];
            p.K[m * (a.slots_max + 1) + slot] = i == t ? own.K[m] : a.chosen[i].K[m];
        }
    }
}

// Rotate the tokens for gate and up of every chosen expert (a warp a block); the last
// CTA makes the plan.  What the joins will want of the experts is brought into L2
// meanwhile.  (Bringing the tensors, too, delayed the rotation itself: one token 35 -> 43
// us, nine tokens through large experts 104 -> 140.)
template <int G, bool LO>
__global__ void __launch_bounds__(kPlanThreads)
moe_rotate_kernel(const MoeArgs a, const FastDiv top_k) {
    extern __shared__ __align__(16) uint8_t sm[];
    pdl_wait();
    pdl_launch();
    if (blockIdx.x == gridDim.x - 1) {
        make_plan<G>(a, sm);
        return;
    }
    const int lane = threadIdx.x & 31, P = a.T * a.top_k, kd = (int)a.kd.d;
    const int i = blockIdx.x * (kPlanThreads / 32) + (threadIdx.x >> 5);      // (pair, block)
    int pair;
    const int b = a.kd.mod(i, pair), k = b * 128 + 4 * lane;
    if (pair >= P) return;
    const Chosen& ch = a.chosen[pair];
    float x[4], s[2][4];
    load4x(a.x, (size_t)top_k.div(pair) * a.ldx + k, a.dtype, x);
    load4(ch.suh[0] + k, s[0]);
    load4(ch.suh[1] + k, s[1]);
    if (lane < 8) {            // block b of svh down; the others of F are shared out; two lanes each
        const int w = lane >> 1;
        const __half* v = w == 0 ? ch.svh[2] : w == 1 ? ch.svh[0] : w == 2 ? ch.svh[1] : ch.suh[2];
        const int n = w == 0 ? kd : (int)a.kf.d;
        for (int f = b; f < n; f += kd) prefetch_line(v + f * 128 + (lane & 1) * 64);
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        float v[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = x[c] * s[m][c];
        const size_t to = ((size_t)m * P + pair) * kd + b;
        few_put_block<LO>(v, a.xh1 + to * kRowBytes, a.inv1 + to, lane, 0, (size_t)2 * P * kd * kRowBytes);
    }
}

// The plan, copied to shared memory at `where`.  All threads.
__device__ __forceinline__ Plan copy_plan(const MoeArgs& a, uint8_t* where) {
    const int P = a.T * a.top_k, n = plan_bytes(P, a.slots_max) / 16;
    const uint4* from = reinterpret_cast<const uint4*>(a.plan);
    for (int i = threadIdx.x; i < n; i += blockDim.x) reinterpret_cast<uint4*>(where)[i] = __ldcg(from + i);
    __syncthreads();
    return plan_at(where, P, a.slots_max);
}

// Units: (tensor, slot, column block); rows: rotated rows of the pairs.
template <int G, bool LO>
struct ExpertJob {
    static constexpr bool kRotate = false, kLo = LO;
    const MoeArgs& a;
    const Plan& p;
    const uint8_t* x;          // [kinds][P][kb][256]
    const float* s;
    int kb;                    // blocks of a row
    const FastDiv& cols;       // column blocks
    bool early;                // the rows are there already
    int first, slots;          // the first unit's tensor; slots of each
    size_t remainders;
    struct Cursor {
        const uint8_t* tiles;
        uint32_t kt_bytes;
        int K, m, s, left;         // tensor, slot; column blocks from here to the last
    };
    __device__ __forceinline__ void load(Cursor& c) const {
        const int v = c.m * (a.slots_max + 1) + c.s;
        c.K = p.K[v];
        c.tiles = p.tiles[v];
        c.kt_bytes = cols.d * 256 * c.K;
        c.left = (int)cols.d;
    }
    __device__ __forceinline__ Cursor cursor(int u) const {
        Cursor c;
        int v;
        const int nb = cols.mod(u, v);
        c.m = first + (v >= slots);
        c.s = v >= slots ? v - slots : v;
        load(c);
        c.tiles += (size_t)nb * 256 * c.K;
        c.left -= nb;
        return c;
    }
    __device__ __forceinline__ void next(Cursor& c) const {
        c.tiles += 256 * c.K;
        if (--c.left == 0) {
            if (++c.s == slots) { c.s = 0; ++c.m; }
            if (c.m < 3) load(c);      // else past the last: not used
        }
    }
    __device__ __forceinline__ int rows(int u) const {
        const int v = cols.div(u);
        return p.slot[v >= slots ? v - slots : v].y & 0xFF;
    }
    __device__ __forceinline__ size_t row(int u, int r) const {
        const int v = cols.div(u), m = v >= slots;
        return ((size_t)m * a.T * a.top_k + p.pair[(p.slot[m ? v - slots : v].y >> 8) + r]) * kb;
    }
    __device__ __forceinline__ int row_step() const { return 1; }
    __device__ __forceinline__ const uint8_t* xh() const { return x; }
    __device__ __forceinline__ const float* inv() const { return s; }
    __device__ __forceinline__ size_t lo() const { return remainders; }
    __device__ __forceinline__ void wait() const { if (!early) pdl_wait(); }
};

template <int CODE, int G, bool LO>
__global__ void __launch_bounds__(32 * kFewWarps, 1) moe_gate_up_kernel(const MoeArgs a, int plan) {
    extern __shared__ __align__(16) uint8_t sm[];
    pdl_wait();
    pdl_launch();              // from here on the plan is there for everyone
    const Plan p = copy_plan(a, sm + plan);
    const FewRun run = p.head->join[0].run;
    if (blockIdx.x >= run.ctas) return;
    const ExpertJob<G, LO> job = {a, p, a.xh1, a.inv1, (int)a.kd.d, a.kf, true, 0, p.head->slots,
                                  (size_t)2 * a.T * a.top_k * a.kd.d * kRowBytes};
    few_run<CODE, G>(job, run, max(a.Kmax[0], a.Kmax[1]), sm, a.park);
}

template <int CODE, int G, bool LO>
__global__ void __launch_bounds__(32 * kFewWarps, 1) moe_down_kernel(const MoeArgs a, int plan) {
    extern __shared__ __align__(16) uint8_t sm[];
    pdl_launch();
    const Plan p = copy_plan(a, sm + plan);
    const FewRun run = p.head->join[1].run;
    if (blockIdx.x >= run.ctas) return;
    const ExpertJob<G, LO> job = {a, p, a.xh2, a.inv2, (int)a.kf.d, a.kd, false, 2, p.head->slots,
                                  (size_t)a.T * a.top_k * a.kf.d * kRowBytes};
    few_run<CODE, G>(job, run, a.Kmax[2], sm, a.park);
}

// h = silu(gate) * up of a (pair, column block of F), and the down projection's rotated
// row: a warp each.
template <int G, bool LO>
__global__ void __launch_bounds__(128) moe_gate_up_finish_kernel(const MoeArgs a) {
    const int lane = threadIdx.x & 31, i = blockIdx.x * 4 + (threadIdx.x >> 5);
    const int fbn = (int)a.kf.d;
    int pair;
    const int fb = a.kf.mod(i, pair), f = fb * 128 + 4 * lane;
    pdl_wait();
    pdl_launch();
    if (pair >= a.T * a.top_k) return;
    const Chosen c = a.chosen[pair];
    const int at = a.place[pair];
    const FewJoin join = reinterpret_cast<const PlanHead*>(a.plan)->join[0];
    float sg[4], su[4], sd[4], v[4], h[4];
    load4(c.svh[0] + f, sg);
    load4(c.svh[1] + f, su);
    load4(c.suh[2] + f, sd);
    const int ug = (at >> 8) * fbn + fb, uu = ug + join.run.units / 2;
    const FewParts<kFewGroups> pg(join, ug), pu(join, uu);
    few_sum(a.park, join, pg, ug, 8 * G, at & 0xFF, lane, 0, 1, v);
    few_sum(a.park, join, pu, uu, 8 * G, at & 0xFF, lane, 0, 1, h);
    few_rotate_back(v, lane);
    few_rotate_back(h, lane);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = silu_f(v[j] * sg[j]) * (h[j] * su[j]) * sd[j];
    const size_t to = (size_t)pair * fbn + fb;
    few_put_block<LO>(v, a.xh2 + to * kRowBytes, a.inv2 + to, lane, 0,
                      (size_t)a.T * a.top_k * fbn * kRowBytes);
}

// Weighted sum over a token's experts of one column block, and the residual: a CTA
// each, whose four warps take every fourth expert in the order of choice.
template <int G>
__global__ void __launch_bounds__(128) moe_down_finish_kernel(const MoeArgs a) {
    __shared__ float4 sum[3][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int nb = blockIdx.x, token = blockIdx.y, n = nb * 128 + 4 * lane, nbn = gridDim.x;
    float res[4] = {0.0f, 0.0f, 0.0f, 0.0f}, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (warp == 0 && a.residual) load4x(a.residual, (size_t)token * a.ldres + n, a.dtype, res);
    pdl_wait();
    const FewJoin join = reinterpret_cast<const PlanHead*>(a.plan)->join[1];
    for (int j = warp; j < a.top_k; j += 4) {
        const int pair = token * a.top_k + j, at = a.place[pair], u = (at >> 8) * nbn + nb;
        float v[4], s[4];
        load4(a.chosen[pair].svh[2] + n, s);
        const float wt = a.wts[pair];
        const FewParts<kFewGroups> parts(join, u);
        few_sum(a.park, join, parts, u, 8 * G, at & 0xFF, lane, 0, 1, v);
        few_rotate_back(v, lane);
#pragma unroll
        for (int c = 0; c < 4; ++c) y[c] = fmaf(v[c], s[c] * wt, y[c]);
    }
    if (warp) sum[warp - 1][lane] = make_float4(y[0], y[1], y[2], y[3]);
    __syncthreads();
    if (warp) return;
#pragma unroll
    for (int i = 0; i < 3; ++i) add4(y, sum[i][lane]);
#pragma unroll
    for (int c = 0; c < 4; ++c) y[c] += res[c];
    store4x(a.out, (size_t)token * a.ldo + n, a.dtype, y);
}

// ------------------------------------------------------------------ host side
static size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }

// Groups of 16 rows where an expert has more than 8 tokens on average; below that the
// few experts with more are read twice, which costs less than twice the rows for all.
static int moe_groups(int T, int E, int top_k) { return T * top_k > 8 * E ? 2 : 1; }

// Slots at most: every pair's expert its own, plus the full groups beyond the first.
static int moe_slots(int T, int E, int top_k) {
    const int P = T * top_k, rows = 8 * moe_groups(T, E, top_k);
    return (P < E ? P : E) + P / rows;
}

static size_t moe_layout(MoeArgs* a, int T, int D, int F, int E, int top_k, int sms, uint8_t* ws) {
    const size_t P = (size_t)T * top_k, kd = D / 128, kf = F / 128;
    const int slots = moe_slots(T, E, top_k), G = moe_groups(T, E, top_k);
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t o = off; off += up256(bytes); return ws + o; };
    const size_t park1 = few_park_bytes((int)(2 * slots * kf), sms, G);
    const size_t park2 = few_park_bytes((int)(slots * kd), sms, G);
    uint8_t* chosen = take(P * sizeof(Chosen));
    uint8_t* wts = take(P * 4);
    uint8_t* place = take(P * 4);
    uint8_t* plan = take(plan_bytes((int)P, slots));
    uint8_t* xh1 = take(4 * P * kd * kRowBytes);       // with the remainders' half
    uint8_t* inv1 = take(2 * P * kd * 4);
    uint8_t* xh2 = take(2 * P * kf * kRowBytes);
    uint8_t* inv2 = take(P * kf * 4);
    uint8_t* park = take(park1 > park2 ? park1 : park2);
    if (a) {
        a->slots_max = slots;
        a->chosen = reinterpret_cast<Chosen*>(chosen);
        a->wts = reinterpret_cast<float*>(wts);
        a->place = reinterpret_cast<int*>(place);
        a->plan = plan;
        const long long t1 = 2LL * slots * kd * kf, t2 = t1 / 2;
        a->ctas1 = (int)(t1 < sms ? t1 : sms);
        a->ctas2 = (int)(t2 < sms ? t2 : sms);
        a->xh1 = xh1;
        a->inv1 = reinterpret_cast<float*>(inv1);
        a->xh2 = xh2;
        a->inv2 = reinterpret_cast<float*>(inv2);
        a->park = reinterpret_cast<float*>(park);
    }
    return off;
}

template <bool F32, int TT>
static int router_launch(const MoeArgs& a, cudaStream_t stream) {
    return launch_kernel<moe_router_kernel<F32, TT>>("moe_router launch", dim3(kRouterRanks, (a.T + TT - 1) / TT),
                                                     kRouterThreads, 0, false, stream, a);
}

template <int CODE, int G, bool LO>
static int moe_run(const MoeArgs& a, int sms, cudaStream_t stream) {
    const int P = a.T * a.top_k, kd = a.D >> 7, kf = a.F >> 7;
    // tokens of a cluster: as many as it takes for all clusters to run at once
    const int most = sms / kRouterRanks, tt = a.T <= most ? 1 : a.T <= 2 * most ? 2 : 4;
    int rc = a.router_dtype == 0
                 ? (tt == 1 ? router_launch<true, 1>(a, stream) :
                    tt == 2 ? router_launch<true, 2>(a, stream) : router_launch<true, 4>(a, stream))
                 : (tt == 1 ? router_launch<false, 1>(a, stream) :
                    tt == 2 ? router_launch<false, 2>(a, stream) : router_launch<false, 4>(a, stream));
    if (rc) return rc;
    constexpr int kWarps = kPlanThreads / 32;
    rc = launch_kernel<moe_rotate_kernel<G, LO>>("moe_rotate launch", dim3((P * kd + kWarps - 1) / kWarps + 1),
                       kPlanThreads, PlanScratch(P, a.E).bytes, true, stream, a, FastDiv(a.top_k));
    if (rc) return rc;
    const int K1 = a.Kmax[0] > a.Kmax[1] ? a.Kmax[0] : a.Kmax[1], plan = plan_bytes(P, a.slots_max);
    const int at1 = up16(few_smem(K1, G, kFewGroups * kRowStages, LO));
    const int at2 = up16(few_smem(a.Kmax[2], G, kFewGroups * kRowStages, LO));
    rc = launch_kernel<moe_gate_up_kernel<CODE, G, LO>>("moe_gate_up launch", dim3(a.ctas1), 32 * kFewWarps,
                       at1 + plan, true, stream, a, at1);
    if (rc) return rc;
    rc = launch_kernel<moe_gate_up_finish_kernel<G, LO>>("moe_gate_up_finish launch", dim3((P * kf + 3) / 4),
                       128, 0, true, stream, a);
    if (rc) return rc;
    rc = launch_kernel<moe_down_kernel<CODE, G, LO>>("moe_down launch", dim3(a.ctas2), 32 * kFewWarps,
                       at2 + plan, true, stream, a, at2);
    if (rc) return rc;
    return launch_kernel<moe_down_finish_kernel<G>>("moe_down_finish launch", dim3(kd, a.T), 128, 0, true,
                         stream, a);
}

}  // namespace exl3b

using namespace exl3b;

namespace {

bool aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

bool moe_dims(int T, int D, int F, int E, int top_k) {
    return T >= 0 && T <= kMaxTokens && D > 0 && D % 128 == 0 && D <= kMaxWidth && F > 0 &&
           F % 128 == 0 && F <= kMaxWidth && E > 0 &&
           E <= kMaxExperts && top_k > 0 && top_k <= kMaxTopK && top_k <= E && T * top_k <= kMaxPairs;
}

}  // namespace

extern "C" {

size_t exl3b_moe_workspace_bytes(int T, int D, int F, int E, int top_k) {
    if (T <= 0 || !moe_dims(T, D, F, E, top_k)) return 0;
    const int sms = device_sms();
    return sms > 0 ? moe_layout(nullptr, T, D, F, E, top_k, sms, nullptr) : 0;
}

int exl3b_moe(const void* dX, int dtype, int64_t ldx, int T, int D, int F, int E, int top_k,
              int normalize, const void* dRouter, int router_dtype, int64_t ldr,
              const exl3b_expert* dExperts, int Kmax_gate, int Kmax_up, int Kmax_down, int code,
              const void* d_residual, int64_t ldres, void* dOut, int64_t ldo, void* ws,
              size_t ws_bytes, void* stream) {
    for (int K : {Kmax_gate, Kmax_up, Kmax_down})
        if (K < 2 || K > 7) { set_error("K=%d outside 2..7", K); return RC_BAD_K; }
    if (code < 0 || code > 2 || (dtype != X_BF16 && dtype != X_FP16) ||
        (router_dtype != 0 && router_dtype != dtype)) {
        set_error("moe: code %d, dtype %d, router dtype %d", code, dtype, router_dtype);
        return RC_BAD_REQUEST;
    }
    if (!moe_dims(T, D, F, E, top_k)) {
        set_error("moe: %d tokens (at most %d), hidden %d and expert width %d (multiples of 128, at most 65536), "
                  "%d experts (at most %d), top_k %d (at most %d; tokens x top_k at most %d)", T,
                  kMaxTokens, D, F, E, kMaxExperts, top_k, kMaxTopK, kMaxPairs);
        return RC_BAD_REQUEST;
    }
    if (T == 0) return RC_OK;
    if (!dX || !aligned(dX, 16) || (T > 1 && (ldx < D || ldx % 8)) || !dRouter ||
        !aligned(dRouter, 16) || (E > 1 && (ldr < D || ldr % 8)) || !dExperts ||
        !aligned(dExperts, 8)) {
        set_error("moe: x and router need 16-byte aligned rows (pitches %lld, %lld)",
                  (long long)ldx, (long long)ldr);
        return RC_BAD_REQUEST;
    }
    if (!dOut || !aligned(dOut, 8) || (T > 1 && (ldo < D || ldo % 4)) ||
        (d_residual && (!aligned(d_residual, 8) || (T > 1 && (ldres < D || ldres % 4))))) {
        set_error("moe: out and residual need 8-byte aligned rows (pitches %lld, %lld)",
                  (long long)ldo, (long long)ldres);
        return RC_BAD_REQUEST;
    }
    if (!ws || !aligned(ws, 256)) {
        set_error("moe: workspace missing or misaligned");
        return RC_WORKSPACE;
    }
    DeviceState* st;
    if (device_state(&st)) { set_error("no usable CUDA device"); return RC_NO_DEVICE; }
    const size_t need = exl3b_moe_workspace_bytes(T, D, F, E, top_k);
    if (!ws || ws_bytes < need || !aligned(ws, 256)) {
        set_error("moe: workspace %zu < %zu bytes or misaligned", ws_bytes, need);
        return RC_WORKSPACE;
    }
    const int rc = forward_status(st);
    if (rc) return rc;
    MoeArgs a;
    memset(&a, 0, sizeof(a));
    a.kd = FastDiv(D / 128);
    a.kf = FastDiv(F / 128);
    a.x = dX; a.ldx = ldx; a.dtype = dtype;
    a.T = T; a.D = D; a.F = F; a.E = E; a.top_k = top_k; a.normalize = normalize;
    a.router = dRouter; a.ldr = ldr; a.router_dtype = router_dtype;
    a.experts = dExperts;
    a.Kmax[0] = Kmax_gate; a.Kmax[1] = Kmax_up; a.Kmax[2] = Kmax_down;
    a.residual = d_residual; a.ldres = ldres; a.out = dOut; a.ldo = ldo;
    moe_layout(&a, T, D, F, E, top_k, st->sms, static_cast<uint8_t*>(ws));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    // fp16: the operands of the products keep what their rounding leaves (LO)
#define EXL3B_MOE(C) \
    (moe_groups(T, E, top_k) == 2 \
         ? dtype == X_FP16 ? moe_run<C, 2, true>(a, st->sms, s) : moe_run<C, 2, false>(a, st->sms, s) \
         : dtype == X_FP16 ? moe_run<C, 1, true>(a, st->sms, s) : moe_run<C, 1, false>(a, st->sms, s))
    switch (code) {
        case CODE_MUL1: return EXL3B_MOE(CODE_MUL1);
        case CODE_3INST: return EXL3B_MOE(CODE_3INST);
        default: return EXL3B_MOE(CODE_MCG);
    }
#undef EXL3B_MOE
}

}  // extern "C"
