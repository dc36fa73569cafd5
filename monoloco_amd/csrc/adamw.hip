// adamw.hip -- one AdamW step over many tensors at once, moments in 32 bits or in e4m3 blocks of 128 (block8.h).
//
//   m' = b1 m + (1 - b1) g;  v' = b2 v + (1 - b2) g^2;  p' = p (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// (the reference's optimizer is torch.optim.Adam, monoloco/train/trainer.py:128; AdamW decays the weights apart from the gradient.)
// Bound by memory: per element 3 parameter / gradient accesses and 4 of the moments (28 bytes with fp32 parameters and moments, 10
// with bf16 parameters and 8-bit moments).  One launch takes up to 64 tensors: their pointers ride in the kernel's arguments (no table
// to upload, nothing kept between calls), and a workgroup finds its tensor with one load per lane and a ballot.
//
// 8-bit moments: m and r = sqrt(v) as codes (r, not v: its range is half as many powers of two).  With b2 = 0.999 a step changes r by
// less than a code's half step, so rounding to nearest would never move it: both are rounded STOCHASTICALLY, up with the probability
// of the distance, from 16 + 16 random bits per element that depend on the seed, the step, the tensor's place in the call and the
// element alone (rng.h's generator).  The update itself uses the unrounded m' and r'.  r' > 0 keeps at least the smallest code: a
// second moment that vanished would let the next step divide by eps.  (eps = 0 and a second moment below fp32's normal range: the divisor
// is taken as the smallest normal number.)
#include <algorithm>
#include <new>
#include <vector>

#include "block8.h"
#include "rng.h"

using namespace mlk;

namespace {

constexpr int MAX_TENSORS = 64;   // lanes of a wave; the table has to fit into the 4 KiB of kernel arguments

struct AdamTable {
    void* p[MAX_TENSORS];
    const void* g[MAX_TENSORS];
    void* m[MAX_TENSORS];
    void* v[MAX_TENSORS];
    uint8_t* s[MAX_TENSORS];        // 8-bit moments: scales of m, then of r (blocks each)
    long numel[MAX_TENSORS];
    unsigned first[MAX_TENSORS];    // first workgroup of the tensor; behind the last tensor: the grid
    unsigned key[MAX_TENSORS];      // random key of the tensor
};
static_assert(sizeof(AdamTable) <= 3700, "kernel arguments");

struct AdamScalars {
    float b1, c1, b2, c2, size, root, eps, keep;   // c = 1 - b; size = lr / (1 - b1^t); root = sqrt(1 - b2^t); keep = 1 - lr wd
};

constexpr int WG_ELEMS = 4096;   // elements per workgroup: 256 threads, 4 chunks of 4 (8-bit moments: 2 of 8) each

__device__ __forceinline__ float adam_update(float p, float m, float r, const AdamScalars& a) {
    return p * a.keep - a.size * m / (r / a.root + a.eps);
}

// the tensor of this workgroup: the number of tensors that start at or before it, minus one
__device__ __forceinline__ int tensor_of(const AdamTable& t, unsigned block) {
    const unsigned f = t.first[threadIdx.x & 63];
    return __builtin_amdgcn_readfirstlane(__popcll(__ballot(f <= block)) - 1);
}

template <typename T>
__global__ __launch_bounds__(256) void adamw32_kernel(AdamTable t, AdamScalars a) {
    const int k = tensor_of(t, blockIdx.x);
    const long n = t.numel[k], base = (long)(blockIdx.x - t.first[k]) * WG_ELEMS;
    T* const P = (T*)t.p[k];
    const T* const G = (const T*)t.g[k];
    float* const M = (float*)t.m[k];
    float* const V = (float*)t.v[k];
    // 4 elements a lane: 16 contiguous bytes of every fp32 array (8 of them, two accesses 32 bytes apart, cost 56 instead of 47 us for 8.4 M
    // parameters); all loads of the four chunks in flight
    constexpr int CHUNKS = WG_ELEMS / 1024;
    typedef T t4 __attribute__((ext_vector_type(4)));
    t4 p[CHUNKS], g[CHUNKS];
    f32x4 m[CHUNKS], v[CHUNKS];
    auto fetch = [&](auto& x, const auto* from, long i) {
        if (i + 4 <= n) {
            x = load_any<std::remove_reference_t<decltype(x)>>(from + i);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < n) x[e] = from[i + e];
        }
    };
    auto keep = [&](const auto& x, auto* to, long i) {
        if (i + 4 <= n) {
            store_any(to + i, x);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < n) to[i + e] = x[e];
        }
    };
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) {
        const long i = base + j * 1024 + threadIdx.x * 4;
        p[j] = g[j] = t4{}, m[j] = v[j] = f32x4{};
        fetch(p[j], P, i), fetch(g[j], G, i), fetch(m[j], (const float*)M, i), fetch(v[j], (const float*)V, i);
    }
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) {
        const long i = base + j * 1024 + threadIdx.x * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float ge = (float)g[j][e];
            m[j][e] = m[j][e] * a.b1 + ge * a.c1;
            v[j][e] = v[j][e] * a.b2 + ge * ge * a.c2;
            p[j][e] = (T)adam_update((float)p[j][e], m[j][e], sqrtf(v[j][e]), a);
        }
        keep(p[j], P, i), keep(m[j], M, i), keep(v[j], V, i);
    }
}

__device__ __forceinline__ void decode8(u32x2 c, float scale, float (&x)[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[h], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[h], true);
        x[h * 4] = lo[0] * scale, x[h * 4 + 1] = lo[1] * scale, x[h * 4 + 2] = hi[0] * scale, x[h * 4 + 3] = hi[1] * scale;
    }
}
__device__ __forceinline__ u32x2 load_codes8(const uint8_t* p, long left) {
    if (left >= 8) return load_any<u32x2>(p);
    u32x2 c = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < left) c[i >> 2] |= (unsigned)p[i] << (8 * (i & 3));
    return c;
}
// 8 new values of a moment -> codes and the block's scale (16 lanes = 128 values).  A value of t steps becomes floor(t + u / 2^16): gfx950's
// stochastic conversion does exactly that with u in the upper half of its random operand, subnormal codes included.  POSITIVE: from one
// step on (a code of at least 1) unless it is 0.
template <bool POSITIVE>
__device__ __forceinline__ u32x2 encode8(const float (&x)[8], const unsigned (&u)[8], unsigned& byte) {
    unsigned a = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) a = max(a, absbits(x[e]));
    byte = scale_byte(max16(a));
    if (byte == 255) return u32x2{0x7f7f7f7fu, 0x7f7f7f7fu};
    const float inv = scale_inverse(byte);
    int c[2] = {0, 0};
    auto put = [&](int& to, float y, float v, unsigned r, auto sel) {
        if (POSITIVE && v > 0.0f) y = fmaxf(y, 0.001953125f);
        to = __builtin_amdgcn_cvt_sr_fp8_f32(y, (int)(POSITIVE ? r & 0xffff0000u : r << 16), to, decltype(sel)::value);
    };
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        put(c[h], x[4 * h] * inv, x[4 * h], u[4 * h], std::integral_constant<int, 0>{});
        put(c[h], x[4 * h + 1] * inv, x[4 * h + 1], u[4 * h + 1], std::integral_constant<int, 1>{});
        put(c[h], x[4 * h + 2] * inv, x[4 * h + 2], u[4 * h + 2], std::integral_constant<int, 2>{});
        put(c[h], x[4 * h + 3] * inv, x[4 * h + 3], u[4 * h + 3], std::integral_constant<int, 3>{});
    }
    return u32x2{(unsigned)c[0], (unsigned)c[1]};
}

template <typename T>
__global__ __launch_bounds__(256) void adamw8_kernel(AdamTable t, AdamScalars a) {
    const int k = tensor_of(t, blockIdx.x);
    const long n = t.numel[k], base = (long)(blockIdx.x - t.first[k]) * WG_ELEMS, blocks = (n + QB - 1) / QB;
    T* const P = (T*)t.p[k];
    const T* const G = (const T*)t.g[k];
    uint8_t* const M = (uint8_t*)t.m[k];
    uint8_t* const R = (uint8_t*)t.v[k];
    uint8_t* const SM = t.s[k];
    uint8_t* const SR = SM + blocks;
    const unsigned key = t.key[k];
    const float inv_root = 1.0f / a.root;
#pragma unroll
    for (int j = 0; j < WG_ELEMS / 2048; ++j) {
        const long i = base + j * 2048 + threadIdx.x * 8, b = i / QB;
        if (b >= blocks) break;   // (16 lanes together)
        float p[8], g[8], m[8], r[8];
        load8(P + i, n - i, p);
        load8(G + i, n - i, g);
        decode8(load_codes8(M + i, n - i), scale_value(SM[b]), m);
        decode8(load_codes8(R + i, n - i), scale_value(SR[b]), r);
        const unsigned bk = mix32(key + (unsigned)b * 0x9e3779b9u) + (unsigned)(i & 127) * 0x85ebca6bu;
        unsigned u[8];
        // (the moments in the 32-bit kernel's operations; root and reciprocal are the hardware's, off by one last place: with the correctly
        // rounded root and two divisions arithmetic was the bound, 355 us for 134 M bf16 parameters)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            u[e] = mix32(bk + (unsigned)e * 0x85ebca6bu);
            m[e] = m[e] * a.b1 + g[e] * a.c1;
            r[e] = __builtin_amdgcn_sqrtf(r[e] * r[e] * a.b2 + g[e] * g[e] * a.c2);
            float den = fmaf(r[e], inv_root, a.eps);
            den = den < 1.17549435e-38f ? 1.17549435e-38f : den;   // (the reciprocal of a subnormal would be infinite; a NaN stays)
            p[e] = fmaf(p[e], a.keep, -(a.size * m[e]) * __builtin_amdgcn_rcpf(den));
        }
        unsigned bm, br;
        const u32x2 cm = encode8<false>(m, u, bm), cr = encode8<true>(r, u, br);
        if (i < n) {
            store8(P + i, n - i, p);
            store_codes8(M + i, n - i, cm);
            store_codes8(R + i, n - i, cr);
        }
        if ((threadIdx.x & 15) == 0) SM[b] = (uint8_t)bm, SR[b] = (uint8_t)br;
    }
}

uint32_t host_mix32(uint32_t x) {
    x ^= x >> 16;
    x *= 0x7feb352dU;
    x ^= x >> 15;
    x *= 0x846ca68bU;
    return x ^ (x >> 16);
}

// All tensors of a call are written side by side: memory that two of them share, in whole or in part, would be a race.  A gradient may be
// one of its own tensor's arrays (every element is read before it is written), nothing else that is written.  (152 arrays: 4 us.)
int check_apart(int n, const int64_t* numel, void* const* p, const void* const* g, int es, void* const* m, void* const* v, int ms, uint8_t* const* scales) {
    struct Span { uintptr_t from, to; int tensor; };
    std::vector<Span> w;
    w.reserve((size_t)n * 4);
    for (int i = 0; i < n; ++i) {
        if (numel[i] == 0) continue;
        auto add = [&](const void* at, int64_t bytes) { w.push_back({(uintptr_t)at, (uintptr_t)at + (uintptr_t)bytes, i}); };
        add(p[i], numel[i] * es), add(m[i], numel[i] * ms), add(v[i], numel[i] * ms);
        if (scales) add(scales[i], (numel[i] + QB - 1) / QB * 2);
    }
    std::sort(w.begin(), w.end(), [](const Span& a, const Span& b) { return a.from < b.from; });
    for (size_t i = 1; i < w.size(); ++i)
        if (w[i].from < w[i - 1].to) return ops_fail(ML_ERR_ARG, "ml_adamw_step: a tensor is given twice, or tensors share memory (%d and %d)", std::min(w[i - 1].tensor, w[i].tensor),
                                                         std::max(w[i - 1].tensor, w[i].tensor));
    for (int i = 0; i < n; ++i) {
        if (numel[i] == 0) continue;
        const uintptr_t from = (uintptr_t)g[i], to = from + (uintptr_t)numel[i] * es;
        const auto at = std::upper_bound(w.begin(), w.end(), from, [](uintptr_t x, const Span& b) { return x < b.to; });
        if (at != w.end() && at->from < to && !(at->tensor == i && at->from == from && at->to == to))
            return ops_fail(ML_ERR_ARG, "ml_adamw_step: gradient %d shares memory with what the step writes of tensor %d", i, at->tensor);
    }
    return ML_OK;
}

}  // namespace

extern "C" int ml_adamw_step(int n_tensors, const int64_t* numel, void* const* params, const void* const* grads, int dtype, void* const* exp_avgs,
                             void* const* exp_avg_sqs, uint8_t* const* scales, int64_t step, double lr, double beta1, double beta2, double eps,
                             double weight_decay, uint32_t seed, void* stream) {
    if (n_tensors < 0 || (dtype != ML_F32 && dtype != ML_BF16 && dtype != ML_F16)) return ops_fail(ML_ERR_ARG, "ml_adamw_step: bad type %d or count %d", dtype, n_tensors);
    if (n_tensors == 0) return ML_OK;
    if (!numel || !params || !grads || !exp_avgs || !exp_avg_sqs) return ops_fail(ML_ERR_ARG, "ml_adamw_step: null pointer");
    if (step < 1) return ops_fail(ML_ERR_ARG, "ml_adamw_step: steps are counted from 1, got %lld", (long long)step);
    if (!(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0)) return ops_fail(ML_ERR_ARG, "ml_adamw_step: betas are in [0, 1), eps is not negative");
    for (int i = 0; i < n_tensors; ++i) {
        if (numel[i] < 0 || numel[i] > (1LL << 35)) return ops_fail(ML_ERR_SHAPE, "ml_adamw_step: tensor %d has %lld elements", i, (long long)numel[i]);
        if (numel[i] && (!params[i] || !grads[i] || !exp_avgs[i] || !exp_avg_sqs[i] || (scales && !scales[i]))) return ops_fail(ML_ERR_ARG, "ml_adamw_step: tensor %d has a null pointer", i);
    }
    try {
        const int rc = check_apart(n_tensors, numel, params, grads, dtype == ML_F32 ? 4 : 2, exp_avgs, exp_avg_sqs, scales ? 1 : 4, scales);
        if (rc) return rc;
    } catch (const std::bad_alloc&) {
        return ops_fail(ML_ERR_STATE, "ml_adamw_step: no host memory for %d tensors", n_tensors);
    }
    const hipStream_t s = (hipStream_t)stream;
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    const hipError_t ce = hipStreamIsCapturing(s, &cap);
    if (ce != hipSuccess) return ops_fail(ML_ERR_HIP, "ml_adamw_step: %s", hipGetErrorString(ce));
    if (cap != hipStreamCaptureStatusNone) return ops_fail(ML_ERR_STATE, "ml_adamw_step: the step's number is part of the launch; a captured one would repeat it");
    const AdamScalars a{(float)beta1, (float)(1 - beta1), (float)beta2, (float)(1 - beta2), (float)(lr / (1 - pow(beta1, (double)step))),
                        (float)sqrt(1 - pow(beta2, (double)step)), (float)eps, (float)(1 - lr * weight_decay)};
    for (int i = 0; i < n_tensors;) {
        AdamTable t;
        unsigned grid = 0;
        int k = 0;
        for (; i < n_tensors && k < MAX_TENSORS; ++i) {
            if (numel[i] == 0) continue;
            const int64_t wgs = (numel[i] + WG_ELEMS - 1) / WG_ELEMS;
            if (k > 0 && grid + wgs > 0xffffffLL) break;   // (a launch has fewer than 2^32 threads; one tensor alone always fits: 2^23 workgroups)
            t.p[k] = params[i], t.g[k] = grads[i], t.m[k] = exp_avgs[i], t.v[k] = exp_avg_sqs[i], t.s[k] = scales ? scales[i] : nullptr;
            t.numel[k] = numel[i], t.first[k] = grid;
            t.key[k] = host_mix32(seed + 0x9e3779b9U * host_mix32((uint32_t)step + 0x85ebca6bU * (uint32_t)(i + 1)));
            grid += (unsigned)wgs;
            ++k;
        }
        if (k == 0) break;
        for (; k < MAX_TENSORS; ++k) t.first[k] = 0xffffffffu;
        const bool eight = scales != nullptr;
        if (dtype == ML_F32) { if (eight) adamw8_kernel<float><<<grid, 256, 0, s>>>(t, a); else adamw32_kernel<float><<<grid, 256, 0, s>>>(t, a); }
        else if (dtype == ML_BF16) { if (eight) adamw8_kernel<bf16_t><<<grid, 256, 0, s>>>(t, a); else adamw32_kernel<bf16_t><<<grid, 256, 0, s>>>(t, a); }
        else { if (eight) adamw8_kernel<f16_t><<<grid, 256, 0, s>>>(t, a); else adamw32_kernel<f16_t><<<grid, 256, 0, s>>>(t, a); }
        const int rc = ops_launched("ml_adamw_step");
        if (rc) return rc;
    }
    return ML_OK;
}
