// forward.cu -- linear layers on EXL3 tensors: y = act(x W + bias) * mul + residual with
// W = diag(suh) B W_inner B diag(svh), W_inner decoded from its trellis on the fly.
//
// x W = (((x suh) B) W_inner) B svh: the activations are rotated instead of the
// weights, so the weight is only ever read as its trellis (K / 8 bytes per weight).

#include "exl3b_internal.h"
#include "forward_gemm.cuh"
#include "../../include/exl3b200.h"

namespace exl3b {

struct LinearArgs {
    const void* x;
    int64_t ldx;
    int dtype;                 // XType of x, bias, mul, residual and out
    int M, k, n;
    const uint8_t* trellis;
    int K, code;
    const __half* suh;
    const __half* svh;
    const void* bias;          // [n], nullable
    int act;
    const void* mul;           // [M][ldmul], nullable
    int64_t ldmul;
    const void* residual;      // [M][ldres], nullable
    int64_t ldres;
    void* out;
    int64_t ldo;
};

// Epilogue operands of four columns of one row, loaded ahead of the product's sums.
struct LinearEpilogue {
    float svh[4], bias[4], mul[4], res[4];
    __device__ __forceinline__ void load(const LinearArgs& a, int row, int col) {
        load4(a.svh + col, svh);
        if (a.bias) load4x(a.bias, col, a.dtype, bias);
        if (a.mul) load4x(a.mul, (size_t)row * a.ldmul + col, a.dtype, mul);
        if (a.residual) load4x(a.residual, (size_t)row * a.ldres + col, a.dtype, res);
    }
    // act(v * svh + bias) * mul + residual, rounded once
    __device__ __forceinline__ void finish(const LinearArgs& a, int row, int col, float (&v)[4]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] *= svh[j];
            if (a.bias) v[j] += bias[j];
            if (a.act != ACT_NONE) v[j] = activate(v[j], a.act);
            if (a.mul) v[j] *= mul[j];
            if (a.residual) v[j] += res[j];
        }
        store4x(a.out, (size_t)row * a.ldo + col, a.dtype, v);
    }
};

// ------------------------------------------------------------------ few rows
struct FewScratch {
    uint8_t* xh;               // [kb][M][256] rotated rows, and as much for the remainders
    float* inv;                // [kb][M] reciprocal scales
    float* park;
};

// suh, rotation and rounding of block b of row r; with LO, which fp16 tensors have, the
// remainders at dst + lo.  (The rounding of the operand is as large as that of an fp16
// result: one row with loud channels came out at 0.33e-3 for the 0.21e-3 of the result's
// rounding alone; eight times finer than that of bf16 it does not show there.)  A warp.
template <bool LO>
__device__ __forceinline__ void linear_rotate(const LinearArgs& a, int r, int b, uint8_t* dst,
                                              float* inv, int swz, size_t lo) {
    const int lane = threadIdx.x & 31, k = b * 128 + 4 * lane;
    float v[4], s[4];
    load4x(a.x, (size_t)r * a.ldx + k, a.dtype, v);
    load4(a.suh + k, s);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] *= s[j];
    few_put_block<LO>(v, dst, inv, lane, swz, lo);
}

template <bool LO>
__global__ void __launch_bounds__(128) linear_rotate_kernel(const LinearArgs a, const FewScratch w) {
    pdl_launch();
    const int i = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (i >= (a.k >> 7) * a.M) return;
    linear_rotate<LO>(a, i % a.M, i / a.M, w.xh + (size_t)i * kRowBytes, w.inv + i, 0,
                      (size_t)(a.k >> 7) * a.M * kRowBytes);
}

// Units: the column blocks; every one has all of the rows, at most 8 G.
template <int G, bool ROTATE, bool LO>
struct LinearJob {
    static constexpr bool kRotate = ROTATE, kLo = LO;
    const LinearArgs& a;
    const FewScratch& w;
    struct Cursor {
        const uint8_t* tiles;
        uint32_t kt_bytes;
        int K;
    };
    __device__ __forceinline__ Cursor cursor(int u) const {
        return {a.trellis + (size_t)u * 256 * a.K, (uint32_t)(a.n >> 7) * 256 * a.K, a.K};
    }
    __device__ __forceinline__ void next(Cursor& c) const { c.tiles += 256 * a.K; }
    __device__ __forceinline__ int rows(int) const { return a.M; }
    __device__ __forceinline__ size_t row(int, int r) const { return r; }
    __device__ __forceinline__ int row_step() const { return a.M; }
    __device__ __forceinline__ const uint8_t* xh() const { return w.xh; }
    __device__ __forceinline__ const float* inv() const { return w.inv; }
    __device__ __forceinline__ size_t lo() const { return (size_t)(a.k >> 7) * a.M * kRowBytes; }
    __device__ __forceinline__ void wait() const { if (!ROTATE) pdl_wait(); }
    __device__ __forceinline__ void rotate(int r, int b, uint8_t* dst, float* inv, int swz) const {
        linear_rotate<LO>(a, r, b, dst, inv, swz, 8 * G * kRowBytes);
    }
};

template <int CODE, int G, bool ROTATE, bool LO>
__global__ void __launch_bounds__(32 * kFewWarps, 1)
linear_few_kernel(const LinearArgs a, const FewScratch w, const FewRun run) {
    extern __shared__ __align__(16) uint8_t sm[];
    pdl_launch();
    const LinearJob<G, ROTATE, LO> job = {a, w};
    few_run<CODE, G>(job, run, a.K, sm, w.park);
}

// Sum of a unit's parked sums of one row, output rotation and epilogue: a CTA each,
// whose four warps take every fourth parked sum.
template <int G>
__global__ void __launch_bounds__(128)
linear_finish_kernel(const LinearArgs a, const FewScratch w, const FewJoin join) {
    __shared__ float4 sum[3][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int nb = blockIdx.x, row = blockIdx.y, col = nb * 128 + 4 * lane;
    LinearEpilogue ep;
    if (warp == 0) ep.load(a, row, col);
    const FewParts<kFewGroups> parts(join, nb);
    pdl_wait();
    float v[4];
    few_sum(w.park, join, parts, nb, 8 * G, row, lane, warp, 4, v);
    if (warp) sum[warp - 1][lane] = make_float4(v[0], v[1], v[2], v[3]);
    __syncthreads();
    if (warp) return;
#pragma unroll
    for (int i = 0; i < 3; ++i) add4(v, sum[i][lane]);
    few_rotate_back(v, lane);
    ep.finish(a, row, col, v);
}

static size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }

static FewRun linear_run(int k, int n, int sms) { return FewRun(FastDiv(k >> 7), n >> 7, sms); }

// Workspace of the few-rows path, laid out at ws.
static size_t few_layout(FewScratch* w, int M, int k, int n, int G, int sms, uint8_t* ws) {
    const FewRun run = linear_run(k, n, sms);
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t o = off; off += up256(bytes); return ws + o; };
    w->park = reinterpret_cast<float*>(take(few_park_bytes(run.units, run.ctas, G)));
    w->xh = take((size_t)(k >> 7) * M * 2 * kRowBytes);
    w->inv = reinterpret_cast<float*>(take((size_t)(k >> 7) * M * 4));
    return off;
}

template <int CODE, int G, bool LO>
static int few_launch(const LinearArgs& a, int sms, uint8_t* ws, cudaStream_t stream) {
    FewScratch w;
    few_layout(&w, a.M, a.k, a.n, G, sms, ws);
    const FewRun run = linear_run(a.k, a.n, sms);
    const dim3 fin(a.n >> 7, a.M);
    const int most = run.least + (run.longer ? 1 : 0), ring = kFewGroups * kRowStages;
    int rc = RC_OK;
    bool done = false;
    if constexpr (G == 1) {
        // one or two rows are rotated where they are used, cheaper than a launch (5120 x
        // 5120, K = 4: 12.2 us against 12.9), if a CTA's share of them fits
        if (a.M <= 2 && few_smem(a.K, G, most, LO) <= kFewRoom) {
            rc = launch_kernel<linear_few_kernel<CODE, G, true, LO>>("linear_few launch", dim3(run.ctas),
                               32 * kFewWarps, few_smem(a.K, G, most, LO), false, stream, a, w, run);
            done = true;
        }
    }
    if (!done) {
        rc = launch_kernel<linear_rotate_kernel<LO>>("linear_rotate launch",
                           dim3(((a.k >> 7) * a.M + 3) / 4), 128, 0, false, stream, a, w);
        if (rc) return rc;
        rc = launch_kernel<linear_few_kernel<CODE, G, false, LO>>("linear_few launch", dim3(run.ctas),
                           32 * kFewWarps, few_smem(a.K, G, ring, LO), true, stream, a, w, run);
    }
    if (rc) return rc;
    return launch_kernel<linear_finish_kernel<G>>("linear_finish launch", fin, 128, 0, true, stream, a,
                         w, FewJoin(run));
}

static int few_groups(int M) { return M > 8 ? 2 : 1; }

static int few_dispatch(const LinearArgs& a, int sms, uint8_t* ws, cudaStream_t stream) {
    const int G = few_groups(a.M);
    const bool lo = a.dtype == X_FP16;
#define EXL3B_FEW(C) \
    (G == 1 ? lo ? few_launch<C, 1, true>(a, sms, ws, stream) : few_launch<C, 1, false>(a, sms, ws, stream) \
            : lo ? few_launch<C, 2, true>(a, sms, ws, stream) : few_launch<C, 2, false>(a, sms, ws, stream))
    switch (a.code) {
        case CODE_MUL1: return EXL3B_FEW(CODE_MUL1);
        case CODE_3INST: return EXL3B_FEW(CODE_3INST);
        default: return EXL3B_FEW(CODE_MCG);
    }
#undef EXL3B_FEW
}

// ------------------------------------------------------------------ more rows
// suh, rotation and rounding of whole rows, a CTA each: fp16 [M][k] in the order of k
// (PAIRED: each 32 k in few_put_block's order, as linear_expand_kernel's), times one power of two a row (its reciprocal in inv [M]), since the matrix unit sums
// over all of k.  The largest magnitude of the row sets it as in block_scale: entries
// 2^-25 of it and below lose bits, which is below the rounding of the sum.  With LO the
// remainders follow as M rows more.
template <bool PAIRED, bool LO>
__global__ void __launch_bounds__(256) linear_rotate_rows_kernel(const LinearArgs a, __half* xh, float* inv) {
    __shared__ float part[8];
    constexpr int kHold = 6;                  // blocks a warp keeps in registers; others are read twice
    pdl_launch();
    const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kb = a.k >> 7;
    const size_t at = (size_t)row * a.ldx + 4 * lane;
    auto load = [&](int b, float (&v)[4]) {
        float s[4];
        load4x(a.x, at + b * 128, a.dtype, v);
        load4(a.suh + b * 128 + 4 * lane, s);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] *= s[j];
    };
    float held[kHold][4], m = 0.0f;
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
        const int b = warp + 8 * i;
        if (b < kb) load(b, held[i]);
    }
#pragma unroll
    for (int i = 0; i < kHold; ++i)
        if (warp + 8 * i < kb)
#pragma unroll
            for (int j = 0; j < 4; ++j) m = fmaxf(m, fabsf(held[i][j]));
#pragma unroll 4
    for (int b = warp + 8 * kHold; b < kb; b += 8) {
        float v[4];
        load(b, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) m = fmaxf(m, fabsf(v[j]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) part[warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) m = fmaxf(m, part[w]);
    float back;
    const float scale = block_scale(m, back) * kInvSqrt128;
    if (threadIdx.x == 0) inv[row] = back;
    auto store = [&](int b, float (&v)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] *= scale;
        had128_warp(v, lane);
        __half* to = xh + (size_t)row * a.k + b * 128;
        auto put = [&](__half* at) {
            if (PAIRED) {
                const int k = 4 * lane;
                at += (k >> 5) * 32 + ((k & 7) >> 1) * 8 + ((k >> 4) & 1) * 4 + ((k >> 3) & 1) * 2;
                *reinterpret_cast<__half2*>(at) = __floats2half2_rn(v[0], v[1]);
                *reinterpret_cast<__half2*>(at + 8) = __floats2half2_rn(v[2], v[3]);
            } else {
                store4(at + 4 * lane, v);
            }
        };
        put(to);
        if constexpr (LO) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] -= __half2float(__float2half_rn(v[j]));
            put(to + (size_t)a.M * a.k);
        }
    };
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
        const int b = warp + 8 * i;
        if (b < kb) store(b, held[i]);
    }
#pragma unroll 4
    for (int b = warp + 8 * kHold; b < kb; b += 8) {
        float v[4];
        load(b, v);
        store(b, v);
    }
}

// Sum of a unit's parked sums of one row (with LO, and of its remainders' row), output
// rotation and epilogue: a warp each.
template <bool LO>
__global__ void __launch_bounds__(128)
linear_mid_finish_kernel(const LinearArgs a, const MidArgs w, const FewJoin join, const float* inv) {
    const int lane = threadIdx.x & 31, nb = blockIdx.y, row = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= a.M) return;
    const int col = nb * 128 + 4 * lane, pass = row / w.N, u = pass * w.nbn + nb;
    LinearEpilogue ep;
    ep.load(a, row, col);
    const FewParts<1> parts(join, u);
    pdl_wait();
    float v[4];
    few_sum(w.park, join, parts, u, w.N, row - pass * w.N, lane, 0, 1, v);
    if constexpr (LO) {
        const int rest = row + a.M, pass2 = rest / w.N, u2 = pass2 * w.nbn + nb;
        const FewParts<1> parts2(join, u2);
        float v2[4];
        few_sum(w.park, join, parts2, u2, w.N, rest - pass2 * w.N, lane, 0, 1, v2);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += v2[j];
    }
    const float f = inv[row];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] *= f;
    few_rotate_back(v, lane);
    ep.finish(a, row, col, v);
}

// cuTensorMapEncodeTiled is a driver-API entry point, resolved at run time through the
// runtime: the library has no link dependency on libcuda.
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                CUtensorMapFloatOOBfill);

// Boxes of 64 x box_rows of a row-major fp16 matrix [rows][k], 128-byte swizzle.
static int encode_rows(CUtensorMap* map, const void* base, int k, int rows, int box_rows) {
    static EncodeTiled fn = nullptr;
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            set_error("cuTensorMapEncodeTiled unavailable from the driver");
            return RC_DEVICE_ERROR;
        }
        fn = reinterpret_cast<EncodeTiled>(p);
    }
    const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)k * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, one[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base), dims, strides, box,
                          one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("cuTensorMapEncodeTiled failed (%d)", (int)r);
        return RC_DEVICE_ERROR;
    }
    return RC_OK;
}

static WaitLimit forward_wait_limit() {
    return WaitLimit((long long)(sweep_wait_ns() * 2.0));   // at 2 cycles a ns, as the sweep's
}

struct MidScratch {
    __half* xh;                // [M][k], M the rows of the product: with LO twice the call's
    float* inv;                // [M]
    float* park;
};

// Passes of equal size, rows rounded up to what the matrix unit takes.
static int mid_rows(int M) {
    const int passes = (M + kMidRows - 1) / kMidRows;
    return ((M + passes - 1) / passes + 15) / 16 * 16;
}

static FewRun mid_run(int M, int k, int n, int sms) {
    const int N = mid_rows(M);
    return FewRun(FastDiv(k >> 7), (n >> 7) * ((M + N - 1) / N), sms);
}

static size_t mid_layout(MidScratch* w, int M, int k, int n, int sms, uint8_t* ws) {
    const FewRun run = mid_run(M, k, n, sms);
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t o = off; off += up256(bytes); return ws + o; };
    w->xh = reinterpret_cast<__half*>(take((size_t)M * k * 2));
    w->inv = reinterpret_cast<float*>(take((size_t)M * 4));
    w->park = reinterpret_cast<float*>(take((size_t)(run.units + run.ctas) * mid_rows(M) * 512));
    return off;
}

template <int CODE, bool LO>
static int mid_launch(const LinearArgs& a, DeviceState* st, uint8_t* ws, cudaStream_t stream) {
    MidScratch w;
    const int M = LO ? 2 * a.M : a.M;
    mid_layout(&w, M, a.k, a.n, st->sms, ws);
    MidArgs m;
    m.trellis = a.trellis;
    m.K = a.K;
    m.nbn = a.n >> 7;
    m.M = M;
    m.N = mid_rows(M);
    m.run = mid_run(M, a.k, a.n, st->sms);
    m.park = w.park;
    m.err = st->fwd_err;
    m.limit = forward_wait_limit();
    const int fit = (kFewRoom - mid_smem(a.K, m.N, 0)) / (m.N * 256);
    m.stages = fit < 4 ? fit : 4;
    CUtensorMap rows;
    int rc = encode_rows(&rows, w.xh, a.k, M, m.N);
    if (rc) return rc;
    rc = launch_kernel<linear_rotate_rows_kernel<false, LO>>("linear_rotate_rows launch", dim3(a.M), 256, 0, false,
                       stream, a, w.xh, w.inv);
    if (rc) return rc;
    rc = launch_kernel<linear_mid_kernel<CODE>>("linear_mid launch", dim3(m.run.ctas), kMidThreads,
                       mid_smem(a.K, m.N, m.stages), true, stream, rows, m);
    if (rc) return rc;
    return launch_kernel<linear_mid_finish_kernel<LO>>("linear_mid_finish launch",
                         dim3((a.M + 3) / 4, m.nbn), 128, 0, true, stream, a, m, FewJoin(m.run),
                         (const float*)w.inv);
}

// ------------------------------------------------------------------ long prompts
__device__ __forceinline__ void widen4(uint2 u, int dtype, float (&v)[4]) {
    if (dtype == X_BF16) {
        v[0] = __uint_as_float(u.x << 16); v[1] = __uint_as_float(u.x & 0xFFFF0000u);
        v[2] = __uint_as_float(u.y << 16); v[3] = __uint_as_float(u.y & 0xFFFF0000u);
    } else {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
        v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
    }
}

// The GEMM's epilogue on 32 columns from `col` of `rows` rows from row0, whose scaled
// and rotated sums are in `patch` (kGemmPitch floats a row).  A warp, eight lanes a row.
struct LinearRows {
    LinearArgs a;
    struct Operands { uint2 mul[8], res[8], svh, bias; };
    __device__ __forceinline__ static uint2 piece(const void* p, size_t i) {
        return *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
    }
    __device__ __forceinline__ void fetch(Operands& o, int row0, int rows, int col, int lane) const {
        const int c = col + (lane & 7) * 4;
        o.svh = piece(a.svh, c);
        if (a.bias) o.bias = piece(a.bias, c);
        if (a.mul) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (4 * i + (lane >> 3) < rows)
                    o.mul[i] = piece(a.mul, (size_t)(row0 + 4 * i + (lane >> 3)) * a.ldmul + c);
        }
        if (a.residual) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (4 * i + (lane >> 3) < rows)
                    o.res[i] = piece(a.residual, (size_t)(row0 + 4 * i + (lane >> 3)) * a.ldres + c);
        }
    }
    __device__ __forceinline__ void finish(const Operands& o, int row0, int rows, int col, float* patch,
                                           int lane) const {
        const int c = col + (lane & 7) * 4;
        float4* at = reinterpret_cast<float4*>(patch + (lane >> 3) * kGemmPitch + (lane & 7) * 4);
        constexpr int kStep = kGemmPitch;          // float4 between a lane's rows
        float svh[4], bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        widen4(o.svh, X_FP16, svh);
        if (a.bias) widen4(o.bias, a.dtype, bias);
        if (a.act != ACT_NONE) {                   // a loop of its own: its code is long
#pragma unroll 1
            for (int i = 0; i < 8; ++i) {
                const float4 q = at[i * kStep];
                at[i * kStep] = make_float4(activate(fmaf(q.x, svh[0], bias[0]), a.act),
                                            activate(fmaf(q.y, svh[1], bias[1]), a.act),
                                            activate(fmaf(q.z, svh[2], bias[2]), a.act),
                                            activate(fmaf(q.w, svh[3], bias[3]), a.act));
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) { svh[j] = 1.0f; bias[j] = 0.0f; }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = 4 * i + (lane >> 3);
            if (r >= rows) break;
            const float4 q = at[i * kStep];
            float v[4] = {fmaf(q.x, svh[0], bias[0]), fmaf(q.y, svh[1], bias[1]),
                          fmaf(q.z, svh[2], bias[2]), fmaf(q.w, svh[3], bias[3])}, t[4];
            if (a.mul) {
                widen4(o.mul[i], a.dtype, t);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] *= t[j];
            }
            if (a.residual) {
                widen4(o.res[i], a.dtype, t);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] += t[j];
            }
            store4x(a.out, (size_t)(row0 + r) * a.ldo + c, a.dtype, v);
        }
    }
};

struct GemmScratch {
    __half* xh;                // [M][k], with LO [2 M][k]
    float* inv;                // [M]
    __half* w;                 // [n][k]
};

static size_t gemm_layout(GemmScratch* w, int M, int k, int n, bool lo, uint8_t* ws) {
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t o = off; off += up256(bytes); return ws + o; };
    w->xh = reinterpret_cast<__half*>(take((size_t)M * k * (lo ? 4 : 2)));
    w->inv = reinterpret_cast<float*>(take((size_t)M * 4));
    w->w = reinterpret_cast<__half*>(take((size_t)n * k * 2));
    return off;
}

template <int CODE, bool LO>
static int gemm_launch(const LinearArgs& a, DeviceState* st, uint8_t* ws, cudaStream_t stream) {
    GemmScratch w;
    gemm_layout(&w, a.M, a.k, a.n, LO, ws);
    CUtensorMap rows, cols;
    int rc = encode_rows(&rows, w.xh, a.k, LO ? 2 * a.M : a.M, 128);
    if (!rc) rc = encode_rows(&cols, w.w, a.k, a.n, 128);
    if (rc) return rc;
    rc = launch_kernel<linear_rotate_rows_kernel<true, LO>>("linear_rotate_rows launch", dim3(a.M), 256, 0, false,
                       stream, a, w.xh, w.inv);
    if (rc) return rc;
    rc = launch_kernel<linear_expand_kernel<CODE>>("linear_expand launch", dim3(a.n >> 7, a.k >> 7), 256, 0,
                       true, stream, a.trellis, a.K, a.k, a.n, w.w);
    if (rc) return rc;
    const LinearRows e = {a};
    const GemmArgs g = {a.M, a.k, a.n, LO ? 2 : 1, w.inv, st->fwd_err, forward_wait_limit()};
    const int tiles = ((a.M + kGemmTile - 1) / kGemmTile) * ((a.n + kGemmTile - 1) / kGemmTile);
    const int pairs = tiles < st->sms / 2 ? tiles : st->sms / 2;
    return launch_kernel<linear_gemm_kernel<LinearRows>>("linear_gemm launch", dim3(2 * pairs),
                         kGemmThreadsAll, kGemmBytes, true, stream, rows, cols, g, e);
}

// ------------------------------------------------------------------ which path
// Sizes whose tiles, blocks and grids are counted in 32 bits: more than a device holds.
constexpr int kMostRows = 1 << 24, kMostCols = 1 << 22;
static bool sizes_fit(int M, int k, int n) {
    return M <= kMostRows && k <= kMostCols && n <= kMostCols &&
           (int64_t)M * (k > n ? k : n) <= (int64_t)1 << 38;
}

constexpr int kFewMost = 16;

// Up to 16 rows mma.sync (one decode serves them); beyond, tensor memory.  There the
// product that decodes as it goes repeats the decode per 256 rows and parks its sums,
// and the decoded copy costs its way to memory and back but leaves a plain GEMM of whole
// 256 x 256 tiles.  The estimates are fits in microseconds, without the rotation that
// both need, closest where the two are near each other.  Measured in all, decoding /
// copying (in x out, rows; bf16, K = 4): 5120 x 5120, 512 44 / 52, 768 60 / 57, 1024 77 / 83,
// 1300 92 / 84; 5120 x 17408, 512 114 / 121, 768 172 / 154, 4096 1044 / 600; 17408 x 5120,
// 1024 206 / 264, 1300 259 / 271, 2048 448 / 412; 5120 x 1024, 2048 49 / 54, 3000 67 / 60; 2048 x
// 8192, 400 34 / 32, 512 39 / 33; 640 x 2048, 1024 26 / 23; fp16: 5120 x 17408, 160 97 / 129, 400
// 175 / 184, 512 213 / 186; 5120 x 5120, 768 98 / 83, 1024 130 / 132.  (It does go to and fro: a row
// more than 768 is another wave of the GEMM there.)  The slower one is taken, by more than
// 3%, at 5 of 240 sizes (10 shapes, 96 to 4096 rows, both types; 16% at 640 x 2048 with 1024
// rows, 7% at most elsewhere) and at 4 of 60 others drawn over all sizes and K (5%).
//
// With fp16 tensors (`lo`) both multiply the remainders of the rows as well, whatever the
// number of rows: an error must not hang on who shares a batch.  Without them the GEMM
// would take half the time, for an error of the result of 1.4 to 1.6 times its rounding's.
static bool copy_pays(int M, int k, int n, bool lo, int sms) {
    const double kb = k >> 7, nb = n >> 7;
    const int rows = lo ? 2 * M : M, N = mid_rows(rows), passes = (rows + N - 1) / N;
    if (passes * nb * kb > 1e9) return true;           // blocks are counted in 32 bits
    const double mid = 12.4 + 1.05 * passes * nb * kb / sms * (N > 216 ? N : 216) / 256.0 +
                       2.65e-6 * rows * (double)n;
    const int tiles = ((M + kGemmTile - 1) / kGemmTile) * ((n + kGemmTile - 1) / kGemmTile);
    const int waves = (tiles + sms / 2 - 1) / (sms / 2);
    const double wave = (lo ? 1.22 : 0.61) * kb + 1.7; // at least its epilogue, 8.4 us
    return 12.7 + 6.0e-7 * k * (double)n + waves * (wave > 8.4 ? wave : 8.4) < mid;
}

// The products, by the numbers of exl3b_linear_product.
enum Product : int { FEW_ROWS = 1, MID_ROWS = 2, LONG_PROMPT = 3 };

static int product_of(int M, int k, int n, bool lo, int sms) {
    return M <= kFewMost ? FEW_ROWS : copy_pays(M, k, n, lo, sms) ? LONG_PROMPT : MID_ROWS;
}

// Of either type of tensors.
static size_t linear_bytes(int M, int k, int n, int sms) {
    if (M <= kFewMost) {
        FewScratch w;
        return few_layout(&w, M, k, n, few_groups(M), sms, nullptr);
    }
    size_t most = 0;
    for (int lo = 0; lo < 2; ++lo) {
        MidScratch w;
        GemmScratch g;
        const size_t bytes = product_of(M, k, n, lo, sms) == LONG_PROMPT
                                 ? gemm_layout(&g, M, k, n, lo, nullptr)
                                 : mid_layout(&w, lo ? 2 * M : M, k, n, sms, nullptr);
        if (bytes > most) most = bytes;
    }
    return most;
}

static int linear_run_all(const LinearArgs& a, DeviceState* st, uint8_t* ws, cudaStream_t stream) {
    const bool lo = a.dtype == X_FP16;
    const int product = product_of(a.M, a.k, a.n, lo, st->sms);
    if (product == FEW_ROWS) return few_dispatch(a, st->sms, ws, stream);
#define EXL3B_ROWS(C) \
    (product == LONG_PROMPT ? lo ? gemm_launch<C, true>(a, st, ws, stream) : gemm_launch<C, false>(a, st, ws, stream) \
          : lo ? mid_launch<C, true>(a, st, ws, stream) : mid_launch<C, false>(a, st, ws, stream))
    switch (a.code) {
        case CODE_MUL1: return EXL3B_ROWS(CODE_MUL1);
        case CODE_3INST: return EXL3B_ROWS(CODE_3INST);
        default: return EXL3B_ROWS(CODE_MCG);
    }
#undef EXL3B_ROWS
}

// A forward kernel's bounded wait ran out in an earlier call: told once.
int forward_status(DeviceState* st) {
    volatile int* e = st->fwd_err;
    if (*e == 0) return RC_OK;
    *e = 0;
    set_error("a wait inside an earlier forward kernel ran out; its results are not valid");
    return RC_DEVICE_ERROR;
}

}  // namespace exl3b

using namespace exl3b;

namespace {

bool aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

// rows of `cols` 2-byte elements at pitch ld, read four at a time
int check_rows(const char* what, const void* p, int64_t ld, int rows, int cols) {
    if (!p || !aligned(p, 8) || (rows > 1 && (ld < cols || ld % 4))) {
        set_error("%s: needs 8-byte aligned rows, pitch >= %d and a multiple of 4 (got %lld)", what,
                  cols, (long long)ld);
        return RC_BAD_REQUEST;
    }
    return RC_OK;
}

}  // namespace

extern "C" {

int exl3b_forward_status(void) {
    DeviceState* st;
    if (device_state(&st)) { set_error("no usable CUDA device"); return RC_NO_DEVICE; }
    return forward_status(st);
}

size_t exl3b_linear_workspace_bytes(int M, int k, int n) {
    if (M <= 0 || k <= 0 || n <= 0 || k % 128 || n % 128 || !sizes_fit(M, k, n)) return 0;
    const int sms = device_sms();
    if (sms <= 0) return 0;
    return linear_bytes(M, k, n, sms);
}

int exl3b_linear_product(int M, int k, int n, int dtype) {
    if (M <= 0 || k <= 0 || n <= 0 || k % 128 || n % 128 || !sizes_fit(M, k, n) ||
        (dtype != X_BF16 && dtype != X_FP16))
        return 0;
    const int sms = device_sms();
    return sms > 0 ? product_of(M, k, n, dtype == X_FP16, sms) : 0;
}

int exl3b_linear(const void* dX, int dtype, int64_t ldx, int M, int k, int n,
                 const int16_t* dTrellis, int K, int code, const void* d_suh_f16,
                 const void* d_svh_f16, const void* d_bias, int act, const void* d_mul,
                 int64_t ldmul, const void* d_residual, int64_t ldres, void* dOut, int64_t ldo,
                 void* ws, size_t ws_bytes, void* stream) {
    if (K < 2 || K > 7) { set_error("K=%d outside 2..7", K); return RC_BAD_K; }
    if (code < 0 || code > 2 || (dtype != X_BF16 && dtype != X_FP16) || act < ACT_NONE ||
        act > ACT_GELU_TANH) {
        set_error("linear: code %d, dtype %d, activation %d", code, dtype, act);
        return RC_BAD_REQUEST;
    }
    if (M < 0 || k <= 0 || n <= 0 || k % 128 || n % 128) {
        set_error("linear: [%d, %d] x [%d, %d]: in and out must be multiples of 128", M, k, k, n);
        return RC_BAD_REQUEST;
    }
    if (!sizes_fit(M, k, n)) {
        set_error("linear: [%d, %d] x [%d, %d]: at most %d rows, in and out at most %d, 2^38 elements",
                  M, k, k, n, kMostRows, kMostCols);
        return RC_BAD_REQUEST;
    }
    if (M == 0) return RC_OK;
    if (!dTrellis || !aligned(dTrellis, 16) || !d_suh_f16 || !aligned(d_suh_f16, 8) || !d_svh_f16 ||
        !aligned(d_svh_f16, 8) || (d_bias && !aligned(d_bias, 8))) {
        set_error("linear: trellis must be 16-byte, suh / svh / bias 8-byte aligned");
        return RC_BAD_REQUEST;
    }
    if (check_rows("linear: x", dX, ldx, M, k) || check_rows("linear: out", dOut, ldo, M, n) ||
        (d_mul && check_rows("linear: mul", d_mul, ldmul, M, n)) ||
        (d_residual && check_rows("linear: residual", d_residual, ldres, M, n)))
        return RC_BAD_REQUEST;
    DeviceState* st;
    if (device_state(&st)) { set_error("no usable CUDA device"); return RC_NO_DEVICE; }
    const size_t need = exl3b_linear_workspace_bytes(M, k, n);
    if (need && (!ws || ws_bytes < need || !aligned(ws, 256))) {
        set_error("linear: workspace %zu < %zu bytes or misaligned", ws_bytes, need);
        return RC_WORKSPACE;
    }
    LinearArgs a = {dX, ldx, dtype, M, k, n, reinterpret_cast<const uint8_t*>(dTrellis), K, code,
                    static_cast<const __half*>(d_suh_f16), static_cast<const __half*>(d_svh_f16),
                    d_bias, act, d_mul, ldmul, d_residual, ldres, dOut, ldo};
    const int rc = forward_status(st);
    if (rc) return rc;
    return linear_run_all(a, st, static_cast<uint8_t*>(ws), static_cast<cudaStream_t>(stream));
}

}  // extern "C"
