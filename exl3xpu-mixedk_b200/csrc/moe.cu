// moe.cu -- mixture-of-experts layer for a few tokens, experts held as EXL3 tensors:
//   l = x R^T;  S = the top_k largest l (ties: lowest index);  p = softmax(l)
//   y = sum_{e in S} w_e ((silu(x Wg_e) * (x Wu_e)) Wd_e) + residual,  w = p or p / sum_S p
//
// Three launches: the router (logits, choice, weights), gate and up of every chosen
// expert down to the down projection's rotated operand, and the down projection with
// the weighted sum.  Each chosen expert's tensors are read once for all of its tokens
// (up to 8 G at a time); the work is bound by their decode, as in forward_few.cuh.
// Nothing depends on the order in which CTAs run: partial sums are joined in rank
// order and a token's experts in the order of their choice.
#include <cooperative_groups.h>

#include "exl3b_internal.h"
#include "forward_few.cuh"
#include "../../include/exl3b200.h"

namespace cg = cooperative_groups;

namespace exl3b {

constexpr int kMaxExperts = 1024;
constexpr int kMaxTokens = 256;           // of one call: bounds the token list of an expert
constexpr int kMaxTopK = 32;

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
    int* ids;                             // [T * top_k]
    float* wts;                           // [T * top_k]
    int* arrived;                         // [T][D / 128]
    uint8_t* xh;                          // [T * top_k][F] fp16, few_put_block order
    float* inv;                           // [T * top_k][F / 128]
    float* part;                          // [T * top_k][D]
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

// Cluster (8 CTAs) per token: 64 warps share the experts, rank 0 chooses.
__global__ void __cluster_dims__(kRouterRanks, 1, 1) __launch_bounds__(256)
moe_router_kernel(const MoeArgs a) {
    __shared__ double logit[kMaxExperts];
    cg::cluster_group cl = cg::this_cluster();
    const int rank = cl.block_rank(), token = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    cl.sync();                               // rank 0 runs: its shared memory may be written
    double* l0 = cl.map_shared_rank(logit, 0);
    const uint4* xr = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x) + token * a.ldx);
    for (int e = rank * 8 + warp; e < a.E; e += 8 * kRouterRanks) {
        double s = 0.0;
        for (int c = lane; c < a.D / 8; c += 32) s += dot8(a, xr[c], (size_t)e * a.ldr + 8 * c);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) l0[e] = s;
    }
    for (int i = rank * 256 + threadIdx.x; i < a.D / 128; i += 256 * kRouterRanks)
        a.arrived[(size_t)token * (a.D / 128) + i] = 0;
    cl.sync();
    if (rank != 0 || warp != 0) return;
    // largest logit, softmax sum
    double m = -INFINITY;
    for (int e = lane; e < a.E; e += 32) m = fmax(m, logit[e]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
    float sum = 0.0f;
    for (int e = lane; e < a.E; e += 32) sum += expf((float)(logit[e] - m));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    // top_k rounds of (largest value, then lowest index); a NaN counts as largest (its
    // weights are NaN whatever is chosen), a chosen entry is marked by its lane
    uint32_t taken = 0;                      // bit i: entry lane + 32 i
    float my_w = 0.0f, picked = 0.0f;
    int my_id = 0;
    for (int j = 0; j < a.top_k; ++j) {
        double best = -INFINITY;
        int bi = kMaxExperts;
        for (int i = 0; lane + 32 * i < a.E; ++i) {
            if (taken >> i & 1) continue;
            const double v = logit[lane + 32 * i];
            const double key = v != v ? INFINITY : v;
            if (bi == kMaxExperts || key > best) { best = key; bi = lane + 32 * i; }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const double ov = __shfl_xor_sync(0xffffffffu, best, o);
            const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
            if (oi != kMaxExperts && (bi == kMaxExperts || ov > best || (ov == best && oi < bi))) {
                best = ov;
                bi = oi;
            }
        }
        if ((bi & 31) == lane) taken |= 1u << (bi >> 5);
        const float p = expf((float)(logit[bi] - m)) / sum;
        picked += p;
        if (lane == j) { my_w = p; my_id = bi; }
    }
    if (lane < a.top_k) {
        a.ids[token * a.top_k + lane] = my_id;
        a.wts[token * a.top_k + lane] = a.normalize ? my_w / picked : my_w;
    }
}

// ------------------------------------------------------------------ experts
// The slot-th chosen expert (ascending), and its (token, choice) pairs in order.
struct ExpertTokens {
    uint32_t bits[kMaxExperts / 32];
    int pair[kMaxTokens];
    int count;
};

// Returns the expert, or -1 when fewer than slot + 1 were chosen.  All threads.
__device__ __forceinline__ int find_expert(const MoeArgs& a, int slot, ExpertTokens& s) {
    const int t = threadIdx.x, P = a.T * a.top_k;
    if (t < kMaxExperts / 32) s.bits[t] = 0;
    __syncthreads();
    for (int i = t; i < P; i += blockDim.x) {
        const int e = a.ids[i];
        atomicOr(&s.bits[e >> 5], 1u << (e & 31));
    }
    __syncthreads();
    int e = -1, left = slot;
    for (int w = 0; w < kMaxExperts / 32; ++w) {
        const uint32_t b = s.bits[w];
        const int c = __popc(b);
        if (left < c) {
            uint32_t r = b;
            for (int i = 0; i < left; ++i) r &= r - 1;
            e = 32 * w + __ffs(r) - 1;
            break;
        }
        left -= c;
    }
    if (e < 0) return -1;
    if (t < 32) {
        int n = 0;
        for (int base = 0; base < P; base += 32) {
            const bool hit = base + t < P && a.ids[base + t] == e;
            const uint32_t m = __ballot_sync(0xffffffffu, hit);
            if (hit) s.pair[n + __popc(m & ((1u << t) - 1))] = base + t;
            n += __popc(m);
        }
        if (t == 0) s.count = n;
    }
    __syncthreads();
    return e;
}

struct MoeShare { int b0, nblk, maxblk; };

__device__ __forceinline__ MoeShare share_of(int kb, int rank, int nrank) {
    MoeShare s;
    s.b0 = (int)((long long)kb * rank / nrank);
    s.nblk = (int)((long long)kb * (rank + 1) / nrank) - s.b0;
    s.maxblk = (kb + nrank - 1) / nrank;
    return s;
}

// gate and up of one expert, 128 columns of F, the share of D of this rank; then
// h = silu(g) * u and the down projection's operand, rotated and rounded.
template <int CODE, int G>
__global__ void __launch_bounds__(32 * kFewWarps, 2) moe_gate_up_kernel(const MoeArgs a) {
    extern __shared__ __align__(16) uint8_t sm[];
    __shared__ ExpertTokens et;
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const int nrank = gridDim.x, rank = blockIdx.x, fb = blockIdx.y;
    const int e = find_expert(a, blockIdx.z, et);
    if (e < 0) return;                        // the whole cluster
    const exl3b_expert w[2] = {a.experts[e], a.experts[a.E + e]};
    const exl3b_expert down = a.experts[2 * a.E + e];
    if (w[0].K < 2 || w[0].K > a.Kmax[0] || w[1].K < 2 || w[1].K > a.Kmax[1]) return;
    const MoeShare sh = share_of(a.D >> 7, rank, nrank);
    const int xpitch = few_row_bytes(sh.maxblk);
    uint8_t* ring[2];
    ring[0] = sm + warp * few_ring_bytes(a.Kmax[0]);
    uint8_t* p = sm + kFewWarps * few_ring_bytes(a.Kmax[0]);
    ring[1] = p + warp * few_ring_bytes(a.Kmax[1]);
    p += kFewWarps * few_ring_bytes(a.Kmax[1]);
    uint8_t* xh = p;                                            // [2][8 G] rows
    float* inv = reinterpret_cast<float*>(xh + 16 * G * xpitch);     // [2][maxblk][8 G]
    float* part = inv + 16 * G * sh.maxblk;                     // [2][8 G][kPartPitch]
    const int tn = a.F >> 4;
    const int count = et.count;
    for (int r0 = 0; r0 < count; r0 += 8 * G) {
        const int rows = min(8 * G, count - r0);
        const uint8_t* src[2];
        size_t kt_bytes[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            kt_bytes[m] = (size_t)tn * 32 * w[m].K;
            src[m] = static_cast<const uint8_t*>(w[m].trellis) + (size_t)sh.b0 * 8 * kt_bytes[m] +
                     (size_t)(fb * 8 + warp) * 32 * w[m].K;
            few_prologue(src[m], kt_bytes[m], w[m].K, sh.nblk, ring[m], lane);
        }
        for (int i = warp; i < sh.nblk * 8 * G; i += kFewWarps) {
            const int r = i % (8 * G), b = i / (8 * G);
            float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            const int k = (sh.b0 + b) * 128 + 4 * lane;
            if (r < rows)
                load4x(a.x, (size_t)(et.pair[r0 + r] / a.top_k) * a.ldx + k, a.dtype, x);
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                float v[4], s[4];
                load4(static_cast<const __half*>(w[m].suh) + k, s);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = x[j] * s[j];
                few_put_block(v, xh + (m * 8 * G + r) * xpitch + b * 256,
                              inv + m * 8 * G * sh.maxblk + i, lane);
            }
        }
        __syncthreads();
        float acc[G][4];
        // the up ring's first blocks were issued before the gate's later ones, so the
        // group count that few_product waits for covers both
        for (int m = 0; m < 2; ++m) {
#pragma unroll
            for (int g = 0; g < G; ++g) acc[g][0] = acc[g][1] = acc[g][2] = acc[g][3] = 0.0f;
            few_product_k<CODE, G>(w[m].K, src[m], kt_bytes[m], sh.nblk, ring[m],
                                   xh + m * 8 * G * xpitch, xpitch, inv + m * 8 * G * sh.maxblk, acc,
                                   lane);
            few_store_part<G>(part + m * 8 * G * kPartPitch, acc, warp, lane);
        }
        if (nrank > 1) cg::this_cluster().sync();
        else __syncthreads();
        for (int r = rank + nrank * warp; r < rows; r += nrank * kFewWarps) {
            float g[4], u[4], s[4];
            const int f = fb * 128 + 4 * lane;
            few_sum_row(part, r, nrank, lane, g);
            few_sum_row(part + 8 * G * kPartPitch, r, nrank, lane, u);
            load4(static_cast<const __half*>(w[0].svh) + f, s);
#pragma unroll
            for (int j = 0; j < 4; ++j) g[j] = silu_f(g[j] * s[j]);
            load4(static_cast<const __half*>(w[1].svh) + f, s);
#pragma unroll
            for (int j = 0; j < 4; ++j) g[j] *= u[j] * s[j];
            load4(static_cast<const __half*>(down.suh) + f, s);
#pragma unroll
            for (int j = 0; j < 4; ++j) g[j] *= s[j];
            const size_t pair = et.pair[r0 + r];
            few_put_block(g, a.xh + (pair * (a.F >> 7) + fb) * 256,
                          a.inv + pair * (a.F >> 7) + fb, lane);
        }
        if (nrank > 1) cg::this_cluster().sync();
        else __syncthreads();
    }
}

// down of one expert, 128 columns of D, the share of F of this rank.  A finished
// (token, choice) row is weighted and parked; whoever parks a token's last row adds
// them up in the order of choice and writes the output.
template <int CODE, int G>
__global__ void __launch_bounds__(32 * kFewWarps, 2) moe_down_kernel(const MoeArgs a) {
    extern __shared__ __align__(16) uint8_t sm[];
    __shared__ ExpertTokens et;
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const int nrank = gridDim.x, rank = blockIdx.x, nb = blockIdx.y;
    const int e = find_expert(a, blockIdx.z, et);
    if (e < 0) return;
    const exl3b_expert w = a.experts[2 * a.E + e];
    if (w.K < 2 || w.K > a.Kmax[2]) return;
    const MoeShare sh = share_of(a.F >> 7, rank, nrank);
    const int xpitch = few_row_bytes(sh.maxblk), fbn = a.F >> 7, nbn = a.D >> 7;
    uint8_t* ring = sm + warp * few_ring_bytes(a.Kmax[2]);
    uint8_t* xh = sm + kFewWarps * few_ring_bytes(a.Kmax[2]);
    float* inv = reinterpret_cast<float*>(xh + 8 * G * xpitch);
    float* part = inv + 8 * G * sh.maxblk;
    const int tn = a.D >> 4;
    const size_t kt_bytes = (size_t)tn * 32 * w.K;
    const uint8_t* src = static_cast<const uint8_t*>(w.trellis) + (size_t)sh.b0 * 8 * kt_bytes +
                         (size_t)(nb * 8 + warp) * 32 * w.K;
    const int count = et.count;
    for (int r0 = 0; r0 < count; r0 += 8 * G) {
        const int rows = min(8 * G, count - r0);
        few_prologue(src, kt_bytes, w.K, sh.nblk, ring, lane);
        // 16 lanes copy one block of one row
        for (int i = t >> 4; i < sh.nblk * 8 * G; i += 2 * kFewWarps) {
            const int r = i % (8 * G), b = i / (8 * G), c = t & 15;
            uint4 v = {0u, 0u, 0u, 0u};
            float s = 1.0f;
            if (r < rows) {
                const size_t blk = (size_t)et.pair[r0 + r] * fbn + sh.b0 + b;
                v = *reinterpret_cast<const uint4*>(a.xh + blk * 256 + 16 * c);
                s = a.inv[blk];
            }
            *reinterpret_cast<uint4*>(xh + r * xpitch + b * 256 + 16 * c) = v;
            if (c == 0) inv[i] = s;
        }
        __syncthreads();
        float acc[G][4];
#pragma unroll
        for (int g = 0; g < G; ++g) acc[g][0] = acc[g][1] = acc[g][2] = acc[g][3] = 0.0f;
        few_product_k<CODE, G>(w.K, src, kt_bytes, sh.nblk, ring, xh, xpitch, inv, acc, lane);
        few_store_part<G>(part, acc, warp, lane);
        if (nrank > 1) cg::this_cluster().sync();
        else __syncthreads();
        for (int r = rank + nrank * warp; r < rows; r += nrank * kFewWarps) {
            float v[4], s[4];
            const int col = nb * 128 + 4 * lane, pair = et.pair[r0 + r], token = pair / a.top_k;
            few_sum_row(part, r, nrank, lane, v);
            load4(static_cast<const __half*>(w.svh) + col, s);
            const float wt = a.wts[pair];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] *= s[j] * wt;
            __stcg(reinterpret_cast<float4*>(a.part + (size_t)pair * a.D + col),
                   make_float4(v[0], v[1], v[2], v[3]));
            __threadfence();
            __syncwarp();
            int n = 0;
            if (lane == 0) n = atomicAdd(a.arrived + (size_t)token * nbn + nb, 1) + 1;
            n = __shfl_sync(0xffffffffu, n, 0);
            if (n != a.top_k) continue;
            __threadfence();
            v[0] = v[1] = v[2] = v[3] = 0.0f;
            for (int j = 0; j < a.top_k; ++j) {
                const float4 f = __ldcg(reinterpret_cast<const float4*>(
                    a.part + ((size_t)token * a.top_k + j) * a.D + col));
                v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
            }
            if (a.residual) {
                load4x(a.residual, (size_t)token * a.ldres + col, a.dtype, s);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] += s[j];
            }
            store4x(a.out, (size_t)token * a.ldo + col, a.dtype, v);
        }
        if (nrank > 1) cg::this_cluster().sync();
        else __syncthreads();
    }
}

// ------------------------------------------------------------------ host side
static size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }

static size_t moe_layout(MoeArgs* a, int T, int D, int F, int top_k, uint8_t* ws) {
    const size_t P = (size_t)T * top_k;
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t o = off; off += up256(bytes); return ws + o; };
    uint8_t* ids = take(P * 4);
    uint8_t* wts = take(P * 4);
    uint8_t* arrived = take((size_t)T * (D / 128) * 4);
    uint8_t* xh = take(P * F * 2);
    uint8_t* inv = take(P * (F / 128) * 4);
    uint8_t* part = take(P * D * 4);
    if (a) {
        a->ids = reinterpret_cast<int*>(ids);
        a->wts = reinterpret_cast<float*>(wts);
        a->arrived = reinterpret_cast<int*>(arrived);
        a->xh = xh;
        a->inv = reinterpret_cast<float*>(inv);
        a->part = reinterpret_cast<float*>(part);
    }
    return off;
}

static size_t moe_smem(int nmat, int K0, int K1, int G, int kb, int S) {
    const int blk = (kb + S - 1) / S;
    size_t b = (size_t)kFewWarps * few_ring_bytes(K0);
    if (nmat == 2) b += (size_t)kFewWarps * few_ring_bytes(K1);
    return b + (size_t)nmat * 8 * G * (few_row_bytes(blk) + 4 * blk + 4 * kPartPitch);
}

// Ranks k is split over: enough CTAs to fill the SMs twice, and a share that fits.
static int moe_split(int nmat, int K0, int K1, int G, int kb, double units, int sms) {
    int S = 1;
    while (S < 8 && 2 * S <= kb &&
           (units * S < 2.0 * sms || moe_smem(nmat, K0, K1, G, kb, S) > 112 * 1024))
        S *= 2;
    return S;
}

template <typename Kern>
static int launch_cluster(Kern kern, const char* what, dim3 grid, size_t smem, const MoeArgs& a,
                          cudaStream_t stream) {
    if (check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        220 * 1024), what))
        return RC_DEVICE_ERROR;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(32 * kFewWarps);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = grid.x;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
    note_launch();
    return check_cuda(e, what) ? RC_DEVICE_ERROR : RC_OK;
}

template <int CODE, int G>
static int moe_run(const MoeArgs& a, int sms, cudaStream_t stream) {
    const int P = a.T * a.top_k;
    const int slots = P < a.E ? P : a.E;
    // chosen experts if every token chose at random; only balances the split
    double miss = 1.0;
    for (int t = 0; t < a.T; ++t) miss *= 1.0 - (double)a.top_k / a.E;
    double active = a.E * (1.0 - miss);
    if (active < 1.0) active = 1.0;
    const int kd = a.D >> 7, kf = a.F >> 7;
    const int S1 = moe_split(2, a.Kmax[0], a.Kmax[1], G, kd, active * kf, sms);
    const int S2 = moe_split(1, a.Kmax[2], 0, G, kf, active * kd, sms);
    const size_t m1 = moe_smem(2, a.Kmax[0], a.Kmax[1], G, kd, S1);
    const size_t m2 = moe_smem(1, a.Kmax[2], 0, G, kf, S2);
    if (m1 > 220 * 1024 || m2 > 220 * 1024) {
        set_error("moe: hidden %d / expert width %d too long", a.D, a.F);
        return RC_BAD_REQUEST;
    }
    moe_router_kernel<<<dim3(kRouterRanks, a.T), 256, 0, stream>>>(a);
    note_launch();
    if (check_cuda(cudaGetLastError(), "moe_router launch")) return RC_DEVICE_ERROR;
    int rc = launch_cluster(moe_gate_up_kernel<CODE, G>, "moe_gate_up launch", dim3(S1, kf, slots), m1,
                            a, stream);
    if (rc) return rc;
    return launch_cluster(moe_down_kernel<CODE, G>, "moe_down launch", dim3(S2, kd, slots), m2, a,
                          stream);
}

}  // namespace exl3b

using namespace exl3b;

namespace {

bool aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

bool moe_dims(int T, int D, int F, int E, int top_k) {
    return T >= 0 && T <= kMaxTokens && D > 0 && D % 128 == 0 && F > 0 && F % 128 == 0 && E > 0 &&
           E <= kMaxExperts && top_k > 0 && top_k <= kMaxTopK && top_k <= E;
}

}  // namespace

extern "C" {

size_t exl3b_moe_workspace_bytes(int T, int D, int F, int E, int top_k) {
    if (T <= 0 || !moe_dims(T, D, F, E, top_k)) return 0;
    return moe_layout(nullptr, T, D, F, top_k, nullptr);
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
                  "%d experts (at most %d), top_k %d (at most %d)", T, kMaxTokens, D, F, E,
                  kMaxExperts, top_k, kMaxTopK);
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
    const size_t need = exl3b_moe_workspace_bytes(T, D, F, E, top_k);
    if (!ws || ws_bytes < need || !aligned(ws, 256)) {
        set_error("moe: workspace %zu < %zu bytes or misaligned", ws_bytes, need);
        return RC_WORKSPACE;
    }
    DeviceState* st;
    if (device_state(&st)) { set_error("no usable CUDA device"); return RC_NO_DEVICE; }
    MoeArgs a = {};
    a.x = dX; a.ldx = ldx; a.dtype = dtype;
    a.T = T; a.D = D; a.F = F; a.E = E; a.top_k = top_k; a.normalize = normalize;
    a.router = dRouter; a.ldr = ldr; a.router_dtype = router_dtype;
    a.experts = dExperts;
    a.Kmax[0] = Kmax_gate; a.Kmax[1] = Kmax_up; a.Kmax[2] = Kmax_down;
    a.residual = d_residual; a.ldres = ldres; a.out = dOut; a.ldo = ldo;
    moe_layout(&a, T, D, F, top_k, static_cast<uint8_t*>(ws));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    // groups of 16 rows once an expert may have more than 8 tokens
#define EXL3B_MOE(C) (T > 8 ? moe_run<C, 2>(a, st->sms, s) : moe_run<C, 1>(a, st->sms, s))
    switch (code) {
        case CODE_MUL1: return EXL3B_MOE(CODE_MUL1);
        case CODE_3INST: return EXL3B_MOE(CODE_3INST);
        default: return EXL3B_MOE(CODE_MCG);
    }
#undef EXL3B_MOE
}

}  // extern "C"
