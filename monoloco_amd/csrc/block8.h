// block8.h -- the 8-bit format of the residual-block operators (fp8.hip, adamw.hip) and the element types around it.
//
// A block is 128 values that share one scale: codes are OCP e4m3 (largest magnitude 448, no infinity, 0x7f = NaN), the scale is an
// e8m0 byte b = the power of two 2^(b - 127), the smallest one with which the block's largest magnitude fits into 448.  Powers of two
// because gfx950's scaled matrix instructions multiply by an e8m0 scale themselves (no vector instruction per accumulator and
// block), because x * 2^-e is exact (ONE rounding, to e4m3: half a step of 2^-4 relative), and because the scale then takes integer
// arithmetic on the bits of the block's maximum -- no division, the same on every machine.
//   zeros only       -> scale 1 (byte 127), codes 0
//   a NaN or infinity -> scale NaN (byte 255), every code NaN: a product with that block is NaN, nothing is silently clipped
//   byte >= 1 (2^-126): fp32 subnormal blocks keep fewer bits
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <cstdarg>
#include <cstdio>
#include <type_traits>

#include "../../include/monoloco_hip.h"

namespace mlk {

// ---- error text of the entry points in fp8.hip and adamw.hip (ml_ops_last_error)
inline thread_local char g_ops_err[256] = "";
inline int ops_fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_ops_err, sizeof(g_ops_err), fmt, ap);
    va_end(ap);
    return code;
}
inline int ops_launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? ML_OK : ops_fail(ML_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

constexpr int QB = 128;   // values per scale

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T> struct Vec8;   // 8 consecutive elements, moved with 16-byte accesses
template <> struct Vec8<float> { f32x4 v[2]; };
template <> struct Vec8<bf16_t> { typedef __bf16 t __attribute__((ext_vector_type(8))); t v; };
template <> struct Vec8<f16_t> { typedef _Float16 t __attribute__((ext_vector_type(8))); t v; };

__device__ __forceinline__ float vget(const Vec8<float>& a, int i) { return a.v[i >> 2][i & 3]; }
__device__ __forceinline__ float vget(const Vec8<bf16_t>& a, int i) { return (float)a.v[i]; }
__device__ __forceinline__ float vget(const Vec8<f16_t>& a, int i) { return (float)a.v[i]; }
__device__ __forceinline__ void vset(Vec8<float>& a, int i, float x) { a.v[i >> 2][i & 3] = x; }
__device__ __forceinline__ void vset(Vec8<bf16_t>& a, int i, float x) { a.v[i] = (__bf16)x; }
__device__ __forceinline__ void vset(Vec8<f16_t>& a, int i, float x) { a.v[i] = (_Float16)x; }

// Rows need no alignment: compute kernels run with unaligned access enabled, and hipcc turns a copy of 16 bytes from any address into one
// 16-byte access.  (Element by element, 32768 rows of 1023 bf16 took 137 us through the norm; so 46, as rows of 1024 do.)
template <typename V> __device__ __forceinline__ V load_any(const void* p) {
    V v;
    __builtin_memcpy(&v, p, sizeof(V));
    return v;
}
template <typename V> __device__ __forceinline__ void store_any(void* p, const V& v) { __builtin_memcpy(p, &v, sizeof(V)); }

// 8 elements at p as they are: `left` of them exist (<= 0: none), the others are 0
template <typename T>
__device__ __forceinline__ Vec8<T> load_raw8(const T* p, long left) {
    Vec8<T> v;
    if (left >= 8) {
        v = load_any<Vec8<T>>(p);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) vset(v, i, i < left ? (float)p[i] : 0.0f);
    }
    return v;
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, long left, float (&x)[8]) {
    const Vec8<T> v = load_raw8(p, left);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = vget(v, i);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, long left, const float (&x)[8]) {
    if (left >= 8) {
        Vec8<T> v;
#pragma unroll
        for (int i = 0; i < 8; ++i) vset(v, i, x[i]);
        store_any(p, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) p[i] = (T)x[i];
    }
}

// the largest of 16 neighbouring lanes' values, in all of them (four rotations inside a row of 16 lanes, no LDS)
__device__ __forceinline__ unsigned max16(unsigned x) {
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xf, 0xf, false));   // row_ror:8
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xf, 0xf, false));   // row_ror:4
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xf, 0xf, false));   // row_ror:2
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xf, 0xf, false));   // row_ror:1
    return x;
}

// magnitudes are compared as bits: an infinity or a NaN is larger than every number, and nothing drops a NaN
__device__ __forceinline__ unsigned absbits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// the block's largest magnitude (bits) -> e8m0 byte: amax = 1.f * 2^x <= 448 * 2^e = 1.75 * 2^(8 + e)
__device__ __forceinline__ unsigned scale_byte(unsigned amax) {
    if (amax == 0) return 127;
    if (amax >= 0x7f800000u) return 255;
    const int b = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (unsigned)max(b, 1);
}
// 2^-(byte - 127), byte 1 .. 247
__device__ __forceinline__ float scale_inverse(unsigned byte) { return __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ float scale_value(unsigned byte) {
    return __uint_as_float(byte == 255 ? 0x7fc00000u : byte == 0 ? 0x00400000u : byte << 23);
}

// 4 values, already divided by the scale, -> 4 codes (round to nearest, ties to even; |x| <= 448)
__device__ __forceinline__ unsigned codes4(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
// 8 values -> 8 codes under the scale byte
__device__ __forceinline__ u32x2 codes8(const float (&x)[8], unsigned byte) {
    u32x2 r;
    if (byte == 255) {
        r[0] = r[1] = 0x7f7f7f7fu;
    } else {
        const float inv = scale_inverse(byte);
        r[0] = codes4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
        r[1] = codes4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
    }
    return r;
}
// 8 codes to memory: `left` of them exist
__device__ __forceinline__ void store_codes8(uint8_t* p, long left, u32x2 c) {
    if (left >= 8) {
        store_any(p, c);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) p[i] = (uint8_t)(c[i >> 2] >> (8 * (i & 3)));
    }
}

// the sum over a wave's 64 lanes, in all of them: four rotations inside rows of 16, then the rows by lane swaps (no LDS)
__device__ __forceinline__ float wave_sum(float x) {
    auto ror = [](float v, auto ctrl) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, false)); };
    x += ror(x, std::integral_constant<int, 0x128>{});
    x += ror(x, std::integral_constant<int, 0x124>{});
    x += ror(x, std::integral_constant<int, 0x122>{});
    x += ror(x, std::integral_constant<int, 0x121>{});
    const auto y = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(y[0]) + __uint_as_float(y[1]);
    const auto z = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(z[0]) + __uint_as_float(z[1]);
}

// 16 codes to memory: `left` of them exist
__device__ __forceinline__ void store_codes16(uint8_t* p, long left, u32x4 c) {
    if (left >= 16) {
        store_any(p, c);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < left) p[i] = (uint8_t)(c[i >> 2] >> (8 * (i & 3)));
    }
}

}  // namespace mlk
