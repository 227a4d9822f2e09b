// moe.cu -- mixture-of-experts layer for a few tokens, experts held as EXL3 tensors:
//   l = x R^T;  S = the top_k largest l (ties: lowest index);  p = softmax(l)
//   y = sum_{e in S} w_e ((silu(x Wg_e) * (x Wu_e)) Wd_e) + residual,  w = p or p / sum_S p
//
// The router (logits, choice, weights, and the chosen experts' rotations of the
// token), then the gate and up products of every chosen expert, the down products, and
// after each a kernel that joins the parked sums: to the down projection's rotated
// rows, and to the weighted sum.  Every launch but the first overlaps the one before
// it.  Each chosen expert's tensors are read once for 8 G of its tokens; the work is
// bound by their decode, spread evenly over the SMs as in forward_few.cuh.  Nothing depends on
// the order in which CTAs run: partial sums are added in a fixed order, and a token's
// experts in the order of their choice.
#include <cooperative_groups.h>
#include <utility>

#include "forward_few.cuh"
#include "../../include/exl3b200.h"

namespace cg = cooperative_groups;

namespace exl3b {

constexpr int kMaxExperts = 1024;
constexpr int kMaxTokens = 256;
constexpr int kMaxTopK = 32;
constexpr int kMaxPairs = 2048;           // (token, choice) pairs of one call

struct MoeArgs {
    const void* x;
    int64_t ldx;
    int dtype;
    int T, D, F, E, top_k, normalize;
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
    int* ids;                             // [T * top_k]
    float* wts;                           // [T * top_k]
    int* place;                           // [1 + T * top_k]: slots, then slot << 8 | row of a pair
    uint8_t* xh1;                         // [2][T * top_k][D / 128][256], few_put_block order
    float* inv1;
    uint8_t* xh2;                         // [T * top_k][F / 128][256]
    float* inv2;
    float* park;
};

// ------------------------------------------------------------------ router
constexpr int kRouterRanks = 8;

// 8 products of a router row and x, summed in fp64.  bf16 and fp16 products are
// exact in fp32; the choice of experts must not hang on the order of a sum, and a
// conversion and an fp64 addition per product cost a microsecond at most.
__device__ __forceinline__ double dot8(const MoeArgs& a, const uint4& xv, size_t off) {
    float x[8];
    if (a.dtype == X_BF16) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t u = (&xv.x)[j];
            x[2 * j] = __uint_as_float(u << 16);
            x[2 * j + 1] = __uint_as_float(u & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&(&xv.x)[j]));
            x[2 * j] = f.x;
            x[2 * j + 1] = f.y;
        }
    }
    double s = 0.0;
    if (a.router_dtype == 0) {
        const float4* r = reinterpret_cast<const float4*>(static_cast<const float*>(a.router) + off);
        const float4 r0 = r[0], r1 = r[1];
        const float f[8] = {r0.x, r0.y, r0.z, r0.w, r1.x, r1.y, r1.z, r1.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) s = fma((double)x[j], (double)f[j], s);
    } else {
        float r[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            load4x(a.router, off + 4 * h, a.router_dtype, r);
#pragma unroll
            for (int j = 0; j < 4; ++j) s += (double)(x[4 * h + j] * r[j]);
        }
    }
    return s;
}

// An order on fp64 values as integers; NaN counts as largest (its weights are NaN
// whatever is chosen).
__device__ __forceinline__ long long order_key(double v) {
    if (v != v) return 0x7FFFFFFFFFFFFFFFLL;
    const long long b = __double_as_longlong(v == 0.0 ? 0.0 : v);
    return b < 0 ? b ^ 0x7FFFFFFFFFFFFFFFLL : b;
}

__device__ __forceinline__ uint32_t peer(const void* p, int rank) {
    uint32_t addr;
    asm("mapa.shared::cluster.u32 %0, %1, %2;"
        : "=r"(addr) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return addr;
}

// Cluster (8 CTAs) per token.  Its 64 warps share the experts' logits, which go to
// every CTA; the CTAs share the experts again to find their place in the order (the
// number of larger logits, and of equal ones before); an expert placed below top_k is
// chosen.  Then all rotate the token for the chosen experts.
__global__ void __cluster_dims__(kRouterRanks, 1, 1) __launch_bounds__(256)
moe_router_kernel(const MoeArgs a) {
    __shared__ double logit[kMaxExperts];
    __shared__ int chosen[kMaxTopK];
    __shared__ float share[kMaxTopK];
    pdl_launch();
    cg::cluster_group cl = cg::this_cluster();
    auto started = cl.barrier_arrive();
    const int rank = cl.block_rank(), token = blockIdx.y, t = threadIdx.x;
    const int warp = t >> 5, lane = t & 31;
    const uint4* xr = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x) + token * a.ldx);
    bool wait = true;
    for (int e0 = rank * 8 + warp; e0 < a.E; e0 += 16 * kRouterRanks) {
        const int e1 = e0 + 8 * kRouterRanks;
        const bool two = e1 < a.E;
        double s0 = 0.0, s1 = 0.0;
#pragma unroll 4
        for (int c = lane; c < a.D / 8; c += 32) {
            const uint4 xv = xr[c];
            s0 += dot8(a, xv, (size_t)e0 * a.ldr + 8 * c);
            if (two) s1 += dot8(a, xv, (size_t)e1 * a.ldr + 8 * c);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            s0 += __shfl_xor_sync(0xffffffffu, s0, o);
            s1 += __shfl_xor_sync(0xffffffffu, s1, o);
        }
        if (wait) { cl.barrier_wait(std::move(started)); wait = false; }   // the others run
        if (lane < kRouterRanks) {
            asm volatile("st.shared::cluster.f64 [%0], %1;" :: "r"(peer(logit + e0, lane)), "d"(s0) : "memory");
            if (two)
                asm volatile("st.shared::cluster.f64 [%0], %1;" :: "r"(peer(logit + e1, lane)), "d"(s1) : "memory");
        }
    }
    if (wait) cl.barrier_wait(std::move(started));
    cl.sync();
    // largest logit and softmax sum, in every warp
    double m = -INFINITY;
    for (int e = lane; e < a.E; e += 32) m = fmax(m, logit[e]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
    float sum = 0.0f;
    for (int e = lane; e < a.E; e += 32) sum += expf((float)(logit[e] - m));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    // 8 lanes count for one expert
    for (int e = rank * 32 + (t >> 3); e - (t >> 3) < a.E; e += 32 * kRouterRanks) {
        int place = 0;
        if (e < a.E) {
            const long long mine = order_key(logit[e]);
            for (int o = t & 7; o < a.E; o += 8) {
                const long long k = order_key(logit[o]);
                place += k > mine || (k == mine && o < e);
            }
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
        if (e < a.E && place < a.top_k) {
            const float p = expf((float)(logit[e] - m)) / sum;
            asm volatile("st.shared::cluster.s32 [%0], %1;" :: "r"(peer(chosen + place, t & 7)), "r"(e) : "memory");
            asm volatile("st.shared::cluster.f32 [%0], %1;" :: "r"(peer(share + place, t & 7)), "f"(p) : "memory");
        }
    }
    cl.sync();
    if (rank == 0 && t < a.top_k) {
        float all = 0.0f;
        for (int j = 0; j < a.top_k; ++j) all += share[j];
        a.ids[token * a.top_k + t] = chosen[t];
        a.wts[token * a.top_k + t] = a.normalize ? share[t] / all : share[t];
    }
    // rotate the token for gate and up of every chosen expert
    const int kd = a.D >> 7, P = a.T * a.top_k;
#pragma unroll 2
    for (int i = rank * 8 + warp; i < 2 * a.top_k * kd; i += 8 * kRouterRanks) {
        const int m2 = i & 1, j = (i >> 1) % a.top_k, b = (i >> 1) / a.top_k, k = b * 128 + 4 * lane;
        const exl3b_expert* w = a.experts + (size_t)m2 * a.E + chosen[j];
        float v[4], s[4];
        load4x(a.x, (size_t)token * a.ldx + k, a.dtype, v);
        load4(static_cast<const __half*>(w->suh) + k, s);
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] *= s[c];
        const size_t to = ((size_t)m2 * P + token * a.top_k + j) * kd + b;
        few_put_block(v, a.xh1 + to * kRowBytes, a.inv1 + to, lane, 0);
    }
}

// ------------------------------------------------------------------ experts
// The chosen experts in ascending order, each cut into slots of up to 8 G of its
// (token, choice) pairs, which are in ascending order too; with the tensors of the
// slots' experts, so that the product need not fetch them.
struct Plan {
    int* pair;                 // [P]
    int2* slot;                // {expert, first pair << 8 | rows}
    const uint8_t** tiles;     // [kinds][slots]
    int* K;                    // [kinds][slots]
    int slots;
};

__host__ __device__ inline int plan_bytes(int P, int slots_max, int kinds) {
    return (P * 4 + 7) / 8 * 8 + slots_max * (8 + 12 * kinds);
}

// For tensors `first` .. first + kinds - 1 of every expert.  `tmp`: room for P + E ints.
// `place`: where to note the pairs' slots (nullable).  All threads.
template <int G>
__device__ __forceinline__ Plan make_plan(const MoeArgs& a, int first, int kinds, uint8_t* where,
                                          int* tmp, int* place) {
    __shared__ int nslots;
    const int t = threadIdx.x, P = a.T * a.top_k;
    Plan p;
    p.pair = reinterpret_cast<int*>(where);
    p.slot = reinterpret_cast<int2*>(where + (P * 4 + 7) / 8 * 8);
    p.tiles = reinterpret_cast<const uint8_t**>(p.slot + a.slots_max);
    p.K = reinterpret_cast<int*>(p.tiles + kinds * a.slots_max);
    int* count = tmp + P;
    for (int i = t; i < P; i += blockDim.x) tmp[i] = a.ids[i];
    __syncthreads();
    for (int e = t; e < a.E; e += blockDim.x) {
        int c = 0;
        for (int i = 0; i < P; ++i) c += tmp[i] == e;
        count[e] = c;
    }
    __syncthreads();
    if (t < 32) {              // running sums of pairs (low half) and slots (high half)
        int sum = 0;
        for (int base = 0; base < a.E; base += 32) {
            const int c = base + t < a.E ? count[base + t] : 0;
            const int mine = c | ((c + 8 * G - 1) / (8 * G)) << 16;
            int run = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, run, o);
                if (t >= o) run += up;
            }
            if (base + t < a.E) count[base + t] = sum + run - mine;
            sum += __shfl_sync(0xffffffffu, run, 31);
        }
        if (t == 0) {
            nslots = sum >> 16;
            if (place) place[0] = nslots;
        }
    }
    __syncthreads();
    p.slots = nslots;
    for (int e = t; e < a.E; e += blockDim.x) {
        const int from = count[e] & 0xFFFF;
        int at = from, slot = count[e] >> 16;
        for (int i = 0; i < P; ++i)
            if (tmp[i] == e) {
                if (place) place[1 + i] = (slot + (at - from) / (8 * G)) << 8 | (at - from) % (8 * G);
                p.pair[at++] = i;
            }
        for (int r = from; r < at; r += 8 * G, ++slot) {
            p.slot[slot] = make_int2(e, r << 8 | min(8 * G, at - r));
            for (int m = 0; m < kinds; ++m) {
                const exl3b_expert* w = a.experts + (size_t)(first + m) * a.E + e;
                p.tiles[m * p.slots + slot] = static_cast<const uint8_t*>(w->trellis);
                p.K[m * p.slots + slot] = min(max(w->K, 2), a.Kmax[first + m]);
            }
        }
    }
    __syncthreads();
    return p;
}

// Units: (tensor, slot, column block); rows: rotated rows of the pairs.
template <int G>
struct ExpertJob {
    static constexpr bool kRotate = false;
    const MoeArgs& a;
    const Plan& p;
    const uint8_t* x;          // [kinds][P][kb][256]
    const float* s;
    int kb, cols;              // blocks of a row, column blocks
    bool early;                // the rows are there already
    __device__ __forceinline__ FewUnit unit(int u) const {
        const int v = u / cols, K = p.K[v];
        return {p.tiles[v] + (size_t)(u - v * cols) * 256 * K, (uint32_t)cols * 256 * K, K};
    }
    __device__ __forceinline__ int rows(int u) const { return p.slot[u / cols % p.slots].y & 0xFF; }
    __device__ __forceinline__ size_t row(int u, int r, int b) const {
        const int v = u / cols, m = v / p.slots;
        return ((size_t)m * a.T * a.top_k + p.pair[(p.slot[v - m * p.slots].y >> 8) + r]) * kb + b;
    }
    __device__ __forceinline__ const uint8_t* xh() const { return x; }
    __device__ __forceinline__ const float* inv() const { return s; }
    __device__ __forceinline__ void wait() const { if (!early) pdl_wait(); }
};

template <int CODE, int G>
__global__ void __launch_bounds__(32 * kFewWarps, 1) moe_gate_up_kernel(const MoeArgs a) {
    extern __shared__ __align__(16) uint8_t sm[];
    const int Kmax = max(a.Kmax[0], a.Kmax[1]);
    pdl_wait();
    pdl_launch();              // from here on the router's results are there for everyone
    const Plan p = make_plan<G>(a, 0, 2, sm + few_smem(Kmax), reinterpret_cast<int*>(sm),
                                blockIdx.x == 0 ? a.place : nullptr);
    const FewRun run(a.D >> 7, 2 * p.slots * (a.F >> 7), gridDim.x);
    if (blockIdx.x >= run.ctas) return;
    const ExpertJob<G> job = {a, p, a.xh1, a.inv1, a.D >> 7, a.F >> 7, true};
    few_run<CODE, G>(job, run, Kmax, sm, a.park);
}

template <int CODE, int G>
__global__ void __launch_bounds__(32 * kFewWarps, 1) moe_down_kernel(const MoeArgs a) {
    extern __shared__ __align__(16) uint8_t sm[];
    pdl_launch();
    const Plan p = make_plan<G>(a, 2, 1, sm + few_smem(a.Kmax[2]), reinterpret_cast<int*>(sm), nullptr);
    const FewRun run(a.F >> 7, p.slots * (a.D >> 7), gridDim.x);
    if (blockIdx.x >= run.ctas) return;
    const ExpertJob<G> job = {a, p, a.xh2, a.inv2, a.F >> 7, a.D >> 7, false};
    few_run<CODE, G>(job, run, a.Kmax[2], sm, a.park);
}

// h = silu(gate) * up of a (pair, column block of F), and the down projection's rotated
// row: a CTA each; two warps add the gate's parked sums, two those of up.
template <int G>
__global__ void __launch_bounds__(128) moe_gate_up_finish_kernel(const MoeArgs a, int ctas) {
    __shared__ float4 sum[3][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int fb = blockIdx.x, pair = blockIdx.y, f = fb * 128 + 4 * lane, fbn = gridDim.x;
    pdl_wait();
    pdl_launch();
    const int e = a.ids[pair], slots = a.place[0], at = a.place[1 + pair];
    float sg[4], su[4], sd[4], v[4];
    if (warp == 0) {
        load4(static_cast<const __half*>(a.experts[e].svh) + f, sg);
        load4(static_cast<const __half*>(a.experts[a.E + e].svh) + f, su);
        load4(static_cast<const __half*>(a.experts[2 * a.E + e].suh) + f, sd);
    }
    const FewRun run(a.D >> 7, 2 * slots * fbn, ctas);
    few_sum<G>(a.park, run, ((warp >> 1) * slots + (at >> 8)) * fbn + fb, at & 0xFF, lane, warp & 1, 2, v);
    if (warp) sum[warp - 1][lane] = make_float4(v[0], v[1], v[2], v[3]);
    __syncthreads();
    if (warp) return;
    add4(v, sum[0][lane]);
    float h[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    add4(h, sum[1][lane]);
    add4(h, sum[2][lane]);
    few_rotate_back(v, lane);
    few_rotate_back(h, lane);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = silu_f(v[j] * sg[j]) * (h[j] * su[j]) * sd[j];
    const size_t to = (size_t)pair * fbn + fb;
    few_put_block(v, a.xh2 + to * kRowBytes, a.inv2 + to, lane, 0);
}

// Weighted sum over a token's experts of one column block, and the residual: a CTA
// each, whose four warps take every fourth expert in the order of choice.
template <int G>
__global__ void __launch_bounds__(128) moe_down_finish_kernel(const MoeArgs a, int ctas) {
    __shared__ float4 sum[3][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int nb = blockIdx.x, token = blockIdx.y, n = nb * 128 + 4 * lane, nbn = gridDim.x;
    float res[4] = {0.0f, 0.0f, 0.0f, 0.0f}, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (warp == 0 && a.residual) load4x(a.residual, (size_t)token * a.ldres + n, a.dtype, res);
    pdl_wait();
    const FewRun run(a.F >> 7, a.place[0] * nbn, ctas);
    for (int j = warp; j < a.top_k; j += 4) {
        const int pair = token * a.top_k + j, at = a.place[1 + pair];
        float v[4], s[4];
        load4(static_cast<const __half*>(a.experts[2 * a.E + a.ids[pair]].svh) + n, s);
        const float wt = a.wts[pair];
        few_sum<G>(a.park, run, (at >> 8) * nbn + nb, at & 0xFF, lane, 0, 1, v);
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
    uint8_t* ids = take(P * 4);
    uint8_t* wts = take(P * 4);
    uint8_t* place = take((1 + P) * 4);
    uint8_t* xh1 = take(2 * P * kd * kRowBytes);
    uint8_t* inv1 = take(2 * P * kd * 4);
    uint8_t* xh2 = take(P * kf * kRowBytes);
    uint8_t* inv2 = take(P * kf * 4);
    uint8_t* park = take(park1 > park2 ? park1 : park2);
    if (a) {
        a->slots_max = slots;
        a->ids = reinterpret_cast<int*>(ids);
        a->wts = reinterpret_cast<float*>(wts);
        a->place = reinterpret_cast<int*>(place);
        a->xh1 = xh1;
        a->inv1 = reinterpret_cast<float*>(inv1);
        a->xh2 = xh2;
        a->inv2 = reinterpret_cast<float*>(inv2);
        a->park = reinterpret_cast<float*>(park);
    }
    return off;
}

template <int CODE, int G>
static int moe_run(const MoeArgs& a, int sms, cudaStream_t stream) {
    int rc = launch_kernel(moe_router_kernel, "moe_router launch", dim3(kRouterRanks, a.T), 256, 0, false,
                           stream, a);
    if (rc) return rc;
    const int P = a.T * a.top_k, kd = a.D >> 7, kf = a.F >> 7;
    const int K1 = a.Kmax[0] > a.Kmax[1] ? a.Kmax[0] : a.Kmax[1];
    const long long t1 = 2LL * a.slots_max * kf * kd, t2 = t1 / 2;
    const int c1 = (int)(t1 < sms ? t1 : sms), c2 = (int)(t2 < sms ? t2 : sms);
    rc = launch_kernel(moe_gate_up_kernel<CODE, G>, "moe_gate_up launch", dim3(c1), 32 * kFewWarps,
                       few_smem(K1) + plan_bytes(P, a.slots_max, 2), true, stream, a);
    if (rc) return rc;
    rc = launch_kernel(moe_gate_up_finish_kernel<G>, "moe_gate_up_finish launch", dim3(kf, P), 128, 0,
                       true, stream, a, c1);
    if (rc) return rc;
    rc = launch_kernel(moe_down_kernel<CODE, G>, "moe_down launch", dim3(c2), 32 * kFewWarps,
                       few_smem(a.Kmax[2]) + plan_bytes(P, a.slots_max, 1), true, stream, a);
    if (rc) return rc;
    return launch_kernel(moe_down_finish_kernel<G>, "moe_down_finish launch", dim3(kd, a.T), 128, 0, true,
                         stream, a, c2);
}

}  // namespace exl3b

using namespace exl3b;

namespace {

bool aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

bool moe_dims(int T, int D, int F, int E, int top_k) {
    return T >= 0 && T <= kMaxTokens && D > 0 && D % 128 == 0 && F > 0 && F % 128 == 0 && E > 0 &&
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
        set_error("moe: %d tokens (at most %d), hidden %d and expert width %d (multiples of 128), "
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
    MoeArgs a = {};
    a.x = dX; a.ldx = ldx; a.dtype = dtype;
    a.T = T; a.D = D; a.F = F; a.E = E; a.top_k = top_k; a.normalize = normalize;
    a.router = dRouter; a.ldr = ldr; a.router_dtype = router_dtype;
    a.experts = dExperts;
    a.Kmax[0] = Kmax_gate; a.Kmax[1] = Kmax_up; a.Kmax[2] = Kmax_down;
    a.residual = d_residual; a.ldres = ldres; a.out = dOut; a.ldo = ldo;
    moe_layout(&a, T, D, F, E, top_k, st->sms, static_cast<uint8_t*>(ws));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
#define EXL3B_MOE(C) (moe_groups(T, E, top_k) == 2 ? moe_run<C, 2>(a, st->sms, s) : moe_run<C, 1>(a, st->sms, s))
    switch (code) {
        case CODE_MUL1: return EXL3B_MOE(CODE_MUL1);
        case CODE_3INST: return EXL3B_MOE(CODE_3INST);
        default: return EXL3B_MOE(CODE_MCG);
    }
#undef EXL3B_MOE
}

}  // extern "C"
