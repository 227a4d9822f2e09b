// forward.cu -- linear layers on EXL3 tensors: y = act(x W + bias) * mul + residual with
// W = diag(suh) B W_inner B diag(svh), W_inner decoded from its trellis on the fly.
//
// x W = (((x suh) B) W_inner) B svh: the activations are rotated instead of the
// weights, so the weight is only ever read as its trellis (K / 8 bytes per weight).
#include <cooperative_groups.h>

#include "exl3b_internal.h"
#include "forward_few.cuh"
#include "../../include/exl3b200.h"

namespace cg = cooperative_groups;

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

// act(v * svh + bias) * mul + residual of four columns of one row, rounded once.
__device__ __forceinline__ void linear_finish(const LinearArgs& a, int row, int col, float (&v)[4]) {
    float t[4];
    load4(a.svh + col, t);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] *= t[j];
    if (a.bias) {
        load4x(a.bias, col, a.dtype, t);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += t[j];
    }
    if (a.act != ACT_NONE) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = activate(v[j], a.act);
    }
    if (a.mul) {
        load4x(a.mul, (size_t)row * a.ldmul + col, a.dtype, t);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] *= t[j];
    }
    if (a.residual) {
        load4x(a.residual, (size_t)row * a.ldres + col, a.dtype, t);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += t[j];
    }
    store4x(a.out, (size_t)row * a.ldo + col, a.dtype, v);
}

// Few rows: CTA (128-column block, row group of 8 G), k split over the CTAs of a
// cluster, whose partial sums meet through distributed shared memory in rank order.
template <int CODE, int G>
__global__ void __launch_bounds__(32 * kFewWarps, 2) linear_few_kernel(const LinearArgs a) {
    extern __shared__ __align__(16) uint8_t sm[];
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const int nrank = gridDim.x, rank = blockIdx.x;        // cluster = x dimension
    const int nb = blockIdx.y, r0 = blockIdx.z * 8 * G;
    const int rows = min(8 * G, a.M - r0);
    const int kb = a.k >> 7;
    const int b0 = (int)((long long)kb * rank / nrank), b1 = (int)((long long)kb * (rank + 1) / nrank);
    const int nblk = b1 - b0;
    const int maxblk = (kb + nrank - 1) / nrank;
    const int xpitch = few_row_bytes(maxblk);
    uint8_t* ring = sm + warp * few_ring_bytes(a.K);
    uint8_t* xh = sm + kFewWarps * few_ring_bytes(a.K);
    float* inv = reinterpret_cast<float*>(xh + 8 * G * xpitch);
    float* part = inv + maxblk * 8 * G;

    const int tn = a.n >> 4;
    const size_t kt_bytes = (size_t)tn * 32 * a.K;
    const uint8_t* src = a.trellis + (size_t)b0 * 8 * kt_bytes + (size_t)(nb * 8 + warp) * 32 * a.K;
    few_prologue(src, kt_bytes, a.K, nblk, ring, lane);
    // rotate this CTA's share of the rows; rows past the last are zero
    for (int i = warp; i < nblk * 8 * G; i += kFewWarps) {
        const int r = i % (8 * G), b = i / (8 * G);
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (r < rows) {
            const int k = (b0 + b) * 128 + 4 * lane;
            float s[4];
            load4x(a.x, (size_t)(r0 + r) * a.ldx + k, a.dtype, v);
            load4(a.suh + k, s);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] *= s[j];
        }
        few_put_block(v, xh + r * xpitch + b * 256, inv + i, lane);
    }
    __syncthreads();
    float acc[G][4];
#pragma unroll
    for (int g = 0; g < G; ++g) acc[g][0] = acc[g][1] = acc[g][2] = acc[g][3] = 0.0f;
    few_product_k<CODE, G>(a.K, src, kt_bytes, nblk, ring, xh, xpitch, inv, acc, lane);
    few_store_part<G>(part, acc, warp, lane);
    if (nrank > 1) cg::this_cluster().sync();
    else __syncthreads();
    for (int r = rank + nrank * warp; r < rows; r += nrank * kFewWarps) {
        float v[4];
        few_sum_row(part, r, nrank, lane, v);
        linear_finish(a, r0 + r, nb * 128 + 4 * lane, v);
    }
    if (nrank > 1) cg::this_cluster().sync();       // partial blocks are read by the others
}

static size_t few_smem(int K, int G, int kb, int S) {
    const int blk = (kb + S - 1) / S;
    return (size_t)kFewWarps * few_ring_bytes(K) + (size_t)8 * G * few_row_bytes(blk) +
           (size_t)blk * 8 * G * 4 + (size_t)8 * G * kPartPitch * 4;
}

template <int CODE, int G>
static int launch_few(const LinearArgs& a, int S, cudaStream_t stream) {
    const size_t smem = few_smem(a.K, G, a.k >> 7, S);
    auto kern = linear_few_kernel<CODE, G>;
    if (check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        227 * 1024), "cudaFuncSetAttribute(linear_few)"))
        return RC_DEVICE_ERROR;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(S, a.n >> 7, (a.M + 8 * G - 1) / (8 * G));
    cfg.blockDim = dim3(32 * kFewWarps);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = S;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
    note_launch();
    return check_cuda(e, "linear_few launch") ? RC_DEVICE_ERROR : RC_OK;
}

static int few_run(const LinearArgs& a, int sms, cudaStream_t stream) {
    const int G = a.M > 8 ? 2 : 1;
    const int kb = a.k >> 7, units = (a.n >> 7) * ((a.M + 8 * G - 1) / (8 * G));
    int S = 1;
    while (S < 8 && 2 * S <= kb && units * S < 2 * sms) S *= 2;
    while (S < 8 && S < kb && few_smem(a.K, G, kb, S) > 200 * 1024) S *= 2;
    if (S > kb) S = kb;
    if (few_smem(a.K, G, kb, S) > 227 * 1024) {
        set_error("linear: in = %d is too long for %d rows", a.k, a.M);
        return RC_BAD_REQUEST;
    }
#define EXL3B_FEW(C) (G == 1 ? launch_few<C, 1>(a, S, stream) : launch_few<C, 2>(a, S, stream))
    switch (a.code) {
        case CODE_MUL1: return EXL3B_FEW(CODE_MUL1);
        case CODE_3INST: return EXL3B_FEW(CODE_3INST);
        default: return EXL3B_FEW(CODE_MCG);
    }
#undef EXL3B_FEW
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

size_t exl3b_linear_workspace_bytes(int M, int k, int n) {
    (void)n;
    if (M <= 0 || k <= 0) return 0;
    return 0;
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
    const size_t need = exl3b_linear_workspace_bytes(M, k, n);
    if (need && (!ws || ws_bytes < need || !aligned(ws, 256))) {
        set_error("linear: workspace %zu < %zu bytes or misaligned", ws_bytes, need);
        return RC_WORKSPACE;
    }
    DeviceState* st;
    if (device_state(&st)) { set_error("no usable CUDA device"); return RC_NO_DEVICE; }
    LinearArgs a = {dX, ldx, dtype, M, k, n, reinterpret_cast<const uint8_t*>(dTrellis), K, code,
                    static_cast<const __half*>(d_suh_f16), static_cast<const __half*>(d_svh_f16),
                    d_bias, act, d_mul, ldmul, d_residual, ldres, dOut, ldo};
    return few_run(a, st->sms, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
