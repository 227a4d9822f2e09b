// trellis_mma.cuh -- decode of EXL3 trellis tiles straight into tensor-core
// operand registers, shared by the forward kernels.
//
// A tile is 16 (k) x 16 (n) weights, a circular stream of 256 K bits; state t is
// the 16-bit window ending at bit (t + 1) K, and its value a code formula.  The
// sequence order (tensor_core_perm, quantize.py:101-118) is the operand order of
// a 16 x 16 x 8 matrix instruction: steps 8 lane .. 8 lane + 7 are the eight
// values that lane holds of W_inner^T as the 16 (n) x 16 (k) A operand.  So a
// warp decodes a tile with no exchange between lanes, and no value passes through
// shared memory.
//
// The decode is bound by instruction issue, not by the trellis' bytes: per weight
// about 1.3 to 2 to cut the window out, then (mul1) one multiply, one byte sum and
// a half of each of a pack and a packed fp16 multiply-add.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "exl3b_common.cuh"

namespace exl3b {

// Values of two states, packed in fp16 (lo: s0).  The formulas are those of
// build_code_lut; each value is one rounding to fp16 of an exact expression, as
// the table's.  Integer multiplies, dp4a and packed fp16 share one pipe at half rate,
// logic, shifts and byte permutes the other (mul1, K = 4: 54 cycles a tile and scheduler;
// the sums apart, packed by a permute, 58; one of them by an absolute difference from zero
// 53, but 1% more in whole products at K = 4; by an 8-bit matrix instruction 60).
template <int CODE>
__device__ __forceinline__ uint32_t code_pair(uint32_t s0, uint32_t s1) {
    uint32_t r;
    if constexpr (CODE == CODE_MUL1) {
        // 0x6400 | b is 1024 + b in fp16 for b < 1024: the byte sum (<= 1020) lands
        // in the mantissa, and one fused multiply-add gives the value.  The second sum
        // is added to the word that holds the first in its upper half.
        const uint32_t h1 = __dp4a(s1 * 0x83DCD12Du, 0x01010101u, 0x6400u);
        const uint32_t p = __dp4a(s0 * 0x83DCD12Du, 0x01010101u, h1 * 65536u + 0x6400u);
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(p), "r"(0x1EEE1EEEu), "r"(0xC931C931u));
    } else {
        uint32_t x0, x1;
        if constexpr (CODE == CODE_3INST) {
            x0 = s0 * 89226354u + 64248484u;
            x1 = s1 * 89226354u + 64248484u;
        } else {
            x0 = s0 * 0xCBAC1FEDu;
            x1 = s1 * 0xCBAC1FEDu;
        }
        // (x & m) ^ c as one instruction (0x6a = 0xf0 & 0xcc ^ 0xaa, by its definition);
        // left to the compiler it is two: 8 rows of 5120 x 17408, MCG, 29.7 -> 34.1 us
        asm("lop3.b32 %0, %0, %1, %2, 0x6a;" : "+r"(x0) : "r"(0x8FFF8FFFu), "r"(0x3B603B60u));
        asm("lop3.b32 %0, %0, %1, %2, 0x6a;" : "+r"(x1) : "r"(0x8FFF8FFFu), "r"(0x3B603B60u));
        const __half2 y0 = *reinterpret_cast<const __half2*>(&x0);
        const __half2 y1 = *reinterpret_cast<const __half2*>(&x1);
        const __half2 v = __halves2half2(__hadd_rn(__low2half(y0), __high2half(y0)),
                                         __hadd_rn(__low2half(y1), __high2half(y1)));
        r = *reinterpret_cast<const uint32_t*>(&v);
    }
    return r;
}

// 16 bits at bit POS (from the top) of the 96-bit string v0 : v1 : v2.
template <int POS>
__device__ __forceinline__ uint32_t window16(uint32_t v0, uint32_t v1, uint32_t v2) {
    const uint32_t a = POS < 32 ? v0 : v1, b = POS < 32 ? v1 : v2;
    constexpr int o = POS & 31;
    if constexpr (o == 0) return a >> 16;
    else if constexpr (o == 8) return __byte_perm(a, 0, 0x4421);
    else if constexpr (o == 16) return a & 0xFFFFu;
    else if constexpr (o < 16) return (a >> (16 - o)) & 0xFFFFu;
    else return __funnelshift_l(b, a, o - 16) & 0xFFFFu;
}

// One lane's place in a tile's stream: its eight windows are the bits
// [8 K lane + K - 16, 8 K lane + 8 K), circularly; they start `shift` bits into
// word `w0` and span at most three 32-bit words.
template <int K>
struct LaneWindow {
    static constexpr int kWords = 8 * K;                       // words of a tile
    static constexpr bool kThree = K >= 5;                     // third word needed
    int w0, w1, w2;
    uint32_t shift;
    __device__ __forceinline__ explicit LaneWindow(int lane) {
        int b = 8 * K * lane + K - 16;
        if (b < 0) b += 256 * K;
        w0 = b >> 5;
        shift = b & 31;
        w1 = w0 + 1 == kWords ? 0 : w0 + 1;
        w2 = w1 + 1 == kWords ? 0 : w1 + 1;
    }
};

// Decode one tile (its words at `tile`, shared or global memory) into this
// lane's A operand of the 16 x 8 x 16 matrix instruction: W_inner^T, rows n.
// a[0] (n, k lo), a[1] (n + 8, k lo), a[2] (n, k hi), a[3] (n + 8, k hi).
template <int K, int CODE>
__device__ __forceinline__ void decode_tile(const uint32_t* __restrict__ tile,
                                            const LaneWindow<K>& lw, uint32_t (&a)[4]) {
    const uint32_t x0 = tile[lw.w0], x1 = tile[lw.w1];
    uint32_t s[8];
    if (K == 4) {          // a lane's word and the one before it, at fixed places
        const uint32_t u = x1 << 4;
        s[0] = window16<20>(x0, x1, 0u);
        s[1] = window16<24>(x0, x1, 0u);
        s[2] = window16<28>(x0, x1, 0u);
        s[3] = x1 >> 16;
        s[4] = u >> 16;
        s[5] = __byte_perm(x1, 0, 0x4421);
        s[6] = __byte_perm(u, 0, 0x4421);
        s[7] = x1 & 0xFFFFu;
    } else {
        const uint32_t x2 = LaneWindow<K>::kThree ? tile[lw.w2] : 0u;
        const uint32_t v0 = __funnelshift_l(x1, x0, lw.shift);
        if (K == 2) {      // windows 8 bits apart share a shift
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t u = v0 << (2 * r);
                s[r] = u >> 16;
                s[r + 4] = __byte_perm(u, 0, 0x4421);
            }
        } else {
            const uint32_t v1 = __funnelshift_l(x2, x1, lw.shift);
            const uint32_t v2 = K == 7 ? x2 << lw.shift : 0u;
            s[0] = window16<0>(v0, v1, v2);
            s[1] = window16<K>(v0, v1, v2);
            s[2] = window16<2 * K>(v0, v1, v2);
            s[3] = window16<3 * K>(v0, v1, v2);
            s[4] = window16<4 * K>(v0, v1, v2);
            s[5] = window16<5 * K>(v0, v1, v2);
            s[6] = window16<6 * K>(v0, v1, v2);
            s[7] = window16<7 * K>(v0, v1, v2);
        }
    }
    a[0] = code_pair<CODE>(s[0], s[1]);
    a[2] = code_pair<CODE>(s[2], s[3]);
    a[1] = code_pair<CODE>(s[4], s[5]);
    a[3] = code_pair<CODE>(s[6], s[7]);
}

// acc[16 n][8 rows] += A (16 n x 16 k) . B (16 k x 8 rows)
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ------------------------------------------------------------ elementwise pieces
// Four consecutive elements of a bf16 / fp16 row as fp32 (8-byte aligned).
template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&v)[4]);
template <>
__device__ __forceinline__ void load4<__half>(const __half* p, float (&v)[4]) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}
template <>
__device__ __forceinline__ void load4<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[4]) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(u.x << 16); v[1] = __uint_as_float(u.x & 0xFFFF0000u);
    v[2] = __uint_as_float(u.y << 16); v[3] = __uint_as_float(u.y & 0xFFFF0000u);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&v)[4]);
template <>
__device__ __forceinline__ void store4<__half>(__half* p, const float (&v)[4]) {
    const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
    uint2 u;
    u.x = *reinterpret_cast<const uint32_t*>(&a);
    u.y = *reinterpret_cast<const uint32_t*>(&b);
    *reinterpret_cast<uint2*>(p) = u;
}
template <>
__device__ __forceinline__ void store4<__nv_bfloat16>(__nv_bfloat16* p, const float (&v)[4]) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    uint2 u;
    u.x = *reinterpret_cast<const uint32_t*>(&a);
    u.y = *reinterpret_cast<const uint32_t*>(&b);
    *reinterpret_cast<uint2*>(p) = u;
}

// 128-point Hadamard transform of a block held by one warp, element 4 lane + j
// in v[j]; not normalised (the caller folds 1 / sqrt(128) into a multiply).
__device__ __forceinline__ void had128_warp(float (&v)[4], int lane) {
    const float a = v[0] + v[1], b = v[0] - v[1], c = v[2] + v[3], d = v[2] - v[3];
    v[0] = a + c; v[1] = b + d; v[2] = a - c; v[3] = b - d;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const float sgn = (lane & m) ? -1.0f : 1.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            v[j] = fmaf(sgn, v[j], __shfl_xor_sync(0xffffffffu, v[j], m));
    }
}

constexpr float kInvSqrt128 = 0.08838834764831845f;

// Exact power of two that brings a block of magnitude `amax` to [2^10, 2^11):
// its transform (at most sqrt(128) times larger) then fits fp16 with 2^25 of
// range below it, so rounding the block to fp16 neither overflows nor loses
// bits to subnormals whatever the activations' range.  1 for an all-zero block;
// an infinite or NaN block keeps its values (the result is NaN either way).
// `inv` is the reciprocal, also exact.
__device__ __forceinline__ float block_scale(float amax, float& inv) {
    int e = (int)(__float_as_uint(amax) >> 23) - 127;          // floor(log2), -127 for subnormals
    if (amax == 0.0f || e == 128) { inv = 1.0f; return 1.0f; }
    e = 10 - e;
    e = e > 120 ? 120 : e;                                      // keep both factors normal
    inv = __uint_as_float((uint32_t)(127 - e) << 23);
    return __uint_as_float((uint32_t)(127 + e) << 23);
}

enum Act : int { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_GELU_TANH = 4 };

__device__ __forceinline__ float silu_f(float v) { return v / (1.0f + __expf(-v)); }

__device__ __forceinline__ float activate(float v, int act) {
    switch (act) {
        case ACT_RELU: return v > 0.0f ? v : (v != v ? v : 0.0f);
        case ACT_SILU: return silu_f(v);
        case ACT_GELU: return 0.5f * v * erfcf(-0.70710678f * v);
        case ACT_GELU_TANH: {
            const float u = 0.7978845608f * (v + 0.044715f * v * v * v);
            return v / (1.0f + __expf(-2.0f * u));
        }
        default: return v;
    }
}

}  // namespace exl3b
