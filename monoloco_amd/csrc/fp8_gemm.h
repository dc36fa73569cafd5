// fp8_gemm.h -- c[i, j] = bias[j] + sum over blocks b of 2^(ea[i, b] + eb[j, b]) * sum over k in b of a[i, k] b[j, k]
// for e4m3 operands in blocks of 128 (block8.h), a (m, k) and b (n, k) both contiguous along k, c in fp32 / bf16 / fp16.
//
// The matrix instruction is v_mfma_scale_f32_32x32x64_f8f6f4: 32 x 32 x 64 with an e8m0 scale for every row and 32 values of k,
// applied inside -- a block of 128 is two of them with the same scale byte, so that neither the scales of rows (both operands may
// have them) nor those of tiles cost a vector instruction.  Operand layout: lane l holds row l & 31, 32 bytes of k; which 32 of the
// 64 does not matter as long as both operands agree (all 128 share one scale).  The first operand is b (its rows become the rows of
// the result), so that a lane's 16 results are 4 x 4 consecutive columns j of one row i of c.
//
// Precision: measured, the 8-bit matrix instructions (scaled or not) align the products of 8 neighbouring k to the largest of them and
// keep 13 bits below it before they reach the fp32 accumulator: 1.5e-5 of the result's norm for normal data, the same for every k.
// That is a hundredth of bf16's rounding and a twentieth of fp16's, so results of those types use them.  fp32 results do not: there the
// codes become bf16 in registers (exact: 4 significant bits; the scale is applied in the same conversion, exact as a power of two)
// and v_mfma_f32_32x32x16_bf16 sums them -- half the rate, 4e-8 of the norm.
#pragma once
#include "block8.h"

namespace mlk {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct GemmParams {
    const uint8_t* a;
    const uint8_t* b;
    const uint8_t* sa;      // (m, kb), or (ceil(m / 128), kb) with a_tile
    const uint8_t* sb;
    long lda, ldb, ldsa, ldsb;
    int a_tile, b_tile;
    const void* bias;       // (n) of bias_dtype, or null
    int bias_dtype;
    void* c;
    long m, n, k, ldc;
    int fast_a, fast_b;     // rows are 16-byte aligned: whole 16-byte pieces inside a row are loaded as such
    int vec_c;              // rows of c are 16-byte aligned
};

// 16 bytes of row `row` at column `col`; what lies behind the matrix is 0 (codes 0 = value 0)
__device__ __forceinline__ u32x4 load16(const uint8_t* p, long ld, long rows, long k, bool fast, long row, long col) {
    u32x4 v = {0, 0, 0, 0};
    if (row < rows && col < k) {
        const uint8_t* const at = p + row * ld + col;
        if (fast && col + 16 <= k) {
            v = *(const u32x4*)at;
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (col + i < k) v[i >> 2] |= (unsigned)at[i] << (8 * (i & 3));
        }
    }
    return v;
}

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// 8 codes times 2^(byte - 127) in bf16
__device__ __forceinline__ bf16x8 to_bf16(int c0, int c1, unsigned byte) {
    if (byte == 255) {
        const __bf16 nan = __builtin_bit_cast(__bf16, (unsigned short)0x7fc0);
        return bf16x8{nan, nan, nan, nan, nan, nan, nan, nan};
    }
    const float scale = scale_value(byte);
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)c0, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)c0, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)c1, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)c1, scale, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// one 32 x 32 x 64 step for a result of type T: 8-bit products, or exact ones
template <typename T>
__device__ __forceinline__ f32x16 mfma64(i32x8 a, i32x8 b, f32x16 c, unsigned sa, unsigned sb) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int s = 0; s < 4; ++s)
            c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(to_bf16(a[2 * s], a[2 * s + 1], sa), to_bf16(b[2 * s], b[2 * s + 1], sb), c, 0, 0, 0);
        return c;
    } else {
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, (int)sa, 0, (int)sb);
    }
}

__device__ __forceinline__ float bias_at(const GemmParams& p, long j) {
    if (!p.bias || j >= p.n) return 0.0f;
    return p.bias_dtype == ML_F32 ? ((const float*)p.bias)[j] : p.bias_dtype == ML_BF16 ? (float)((const bf16_t*)p.bias)[j] : (float)((const f16_t*)p.bias)[j];
}

// 4 consecutive columns of one row of c
template <typename T>
__device__ __forceinline__ void store4(const GemmParams& p, long i, long j, const float (&v)[4]) {
    if (i >= p.m || j >= p.n) return;
    T* const at = (T*)p.c + i * p.ldc + j;
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = v[e] + bias_at(p, j + e);
    if (p.vec_c && j + 4 <= p.n) {
        typedef T t4 __attribute__((ext_vector_type(4)));
        *(t4*)at = t4{(T)x[0], (T)x[1], (T)x[2], (T)x[3]};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (j + e < p.n) at[e] = (T)x[e];
    }
}

// 64 x 64 of c per workgroup, 32 x 32 per wave, one block of 128 in LDS at a time: right for every size, stride and alignment
template <typename T>
__global__ __launch_bounds__(256) void fp8_gemm64_kernel(GemmParams p) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[2][64 * QB];
    const long nt = (p.n + 63) / 64, kb = (p.k + QB - 1) / QB;
    const long m0 = blockIdx.x / nt * 64, n0 = blockIdx.x % nt * 64;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, wm = w >> 1, wn = w & 1, lr = lane & 31, lh = lane >> 5;
    f32x16 acc = {};
    const long arow = min(m0 + wm * 32 + lr, p.m - 1), brow = min(n0 + wn * 32 + lr, p.n - 1);
    const uint8_t* const sa = p.sa + (p.a_tile ? arow / QB : arow) * p.ldsa;
    const uint8_t* const sb = p.sb + (p.b_tile ? brow / QB : brow) * p.ldsb;
    for (long t = 0; t < kb; ++t) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = (threadIdx.x >> 3) + 32 * i, ch = threadIdx.x & 7;
            *(u32x4*)(lds[0] + r * QB + ((ch ^ (r & 7)) * 16)) = load16(p.a, p.lda, p.m, p.k, p.fast_a, m0 + r, t * QB + ch * 16);
            *(u32x4*)(lds[1] + r * QB + ((ch ^ (r & 7)) * 16)) = load16(p.b, p.ldb, p.n, p.k, p.fast_b, n0 + r, t * QB + ch * 16);
        }
        __syncthreads();
        const unsigned xa = sa[t], xb = sb[t];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            i32x8 fa, fb;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int ch = s * 4 + lh * 2 + h;
                const u32x4 va = *(const u32x4*)(lds[0] + (wm * 32 + lr) * QB + ((ch ^ (lr & 7)) * 16));
                const u32x4 vb = *(const u32x4*)(lds[1] + (wn * 32 + lr) * QB + ((ch ^ (lr & 7)) * 16));
#pragma unroll
                for (int e = 0; e < 4; ++e) fa[h * 4 + e] = (int)va[e], fb[h * 4 + e] = (int)vb[e];
            }
            acc = mfma64<T>(fb, fa, acc, xb, xa);
        }
        __syncthreads();
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const float v[4] = {acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
        store4<T>(p, m0 + wm * 32 + lr, n0 + wn * 32 + 8 * g + 4 * lh, v);
    }
}

}  // namespace mlk
