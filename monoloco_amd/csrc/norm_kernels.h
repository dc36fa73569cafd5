// norm_kernels.h -- root-mean-square norm over the last axis, with the residual's addition, forward and backward.
//
//   h = x + residual;  rstd = 1 / sqrt(mean_j h_j^2 + eps);  y_j = h_j rstd w_j          (y, statistics from h before its rounding)
//   g = dy * w;  dx_j = rstd (g_j - h_j rstd^2 mean_i(g_i h_i)) + dh_j;   dw_j = sum over rows of dy_j h_j rstd
//
// Bound by memory: forward 2 reads + 2 writes per element (8-bit output: one byte instead of the last), backward 3 reads + 1 write.
// A row stays in registers between its reduction and its output, so everything is read once.  A lane owns chunks of 8 consecutive
// elements (one 16-byte access of a 2-byte type; 16 neighbouring lanes = one block of 128 of the 8-bit output, whose maximum is
// four DPP rotations).  WPR = waves per row, NV = chunks per lane: a row of up to 2048 elements is one wave's (no LDS, no barrier;
// four rows per workgroup), longer ones take 4, 8 or 16 waves; NV = 0 streams rows beyond 32768
// elements (backward: 16384) from memory twice.
#pragma once
#include "block8.h"

namespace mlk {

struct NormParams {
    const void* x;          // (m, n), row stride ldx
    const void* residual;   // or null
    const void* w;          // (n)
    int w_f32;              // w is fp32 (else x's type)
    long m, n, ldx, ldr, ldy, ldh;
    float eps;
    void* y;                // (m, n) in x's type, or null
    void* h;                // (m, n) in x's type, or null
    uint8_t* q;             // (m, n) codes, or null
    uint8_t* scale;         // (m, blocks), row stride lds
    long lds;
};

template <int WPR>
__device__ __forceinline__ float row_sum(float x, float* red) {
    x = wave_sum(x);
    if (WPR == 1) return x;
    __syncthreads();   // (the previous reduction's readers are done)
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < WPR; ++i) s += red[i];
    return s;
}

// 1 / sqrt(ss / n + eps), once per row, in 64 bits: what the row shares should not add to its elements' own roundings (8-bit codes next to a
// border would follow it)
__device__ __forceinline__ float row_rstd(float ss, long n, float eps) { return (float)(1.0 / sqrt((double)ss / (double)n + (double)eps)); }

template <typename T>
__device__ __forceinline__ void load_weight8(const void* w, int w_f32, long c, long n, float (&x)[8]) {
    if (w_f32) load8((const float*)w + c, n - c, x);
    else load8((const T*)w + c, n - c, x);
}

// one chunk's output
template <typename T, bool OUT8>
__device__ __forceinline__ void norm_out(const NormParams& p, long row, long c, const float (&h)[8], float rstd) {
    float wv[8], y[8];
    load_weight8<T>(p.w, p.w_f32, c, p.n, wv);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = h[i] * rstd * wv[i];
    if (OUT8) {
        unsigned a = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) a = max(a, c + i < p.n ? absbits(y[i]) : 0u);
        const unsigned byte = scale_byte(max16(a));
        if (c < p.n) {
            store_codes8(p.q + row * p.ldy + c, p.n - c, codes8(y, byte));
            if ((threadIdx.x & 15) == 0) p.scale[row * p.lds + c / QB] = (uint8_t)byte;
        }
    } else if (c < p.n) {
        store8((T*)p.y + row * p.ldy + c, p.n - c, y);
    }
}

template <typename T>
__device__ __forceinline__ void norm_in(const NormParams& p, long row, long c, float (&h)[8]) {
    load8((const T*)p.x + row * p.ldx + c, p.n - c, h);
    if (p.residual) {
        float r[8];
        load8((const T*)p.residual + row * p.ldr + c, p.n - c, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] += r[i];
    }
}

template <typename T, bool OUT8, int WPR, int NV>
__global__ __launch_bounds__(WPR == 1 ? 256 : WPR * 64) void rms_norm_kernel(NormParams p) {
    __shared__ float red[WPR];
    const int lane = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;   // place in the row's team
    const long row = WPR == 1 ? (long)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    if (row >= p.m) return;   // (WPR > 1: never taken, the grid is m)
    constexpr long STEP = WPR * 64 * 8;
    float ss = 0.0f;
    if constexpr (NV > 0) {
        float h[NV][8];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            norm_in<T>(p, row, lane * 8 + j * STEP, h[j]);
#pragma unroll
            for (int i = 0; i < 8; ++i) ss += h[j][i] * h[j][i];
        }
        const float rstd = row_rstd(row_sum<WPR>(ss, red), p.n, p.eps);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const long c = lane * 8 + j * STEP;
            if (p.h && c < p.n) store8((T*)p.h + row * p.ldh + c, p.n - c, h[j]);
            norm_out<T, OUT8>(p, row, c, h[j], rstd);
        }
    } else {   // long rows: once for the sum, once for the output
        const long end = (p.n + STEP - 1) / STEP * STEP;   // (whole teams: the block maximum needs its 16 lanes)
        float h[8];
        for (long c = lane * 8; c < end; c += STEP) {
            norm_in<T>(p, row, c, h);
#pragma unroll
            for (int i = 0; i < 8; ++i) ss += h[i] * h[i];
        }
        const float rstd = row_rstd(row_sum<WPR>(ss, red), p.n, p.eps);
        for (long c = lane * 8; c < end; c += STEP) {
            norm_in<T>(p, row, c, h);
            if (p.h && c < p.n) store8((T*)p.h + row * p.ldh + c, p.n - c, h);
            norm_out<T, OUT8>(p, row, c, h, rstd);
        }
    }
}

struct NormBackParams {
    const void* dy;   // (m, n)
    const void* h;    // (m, n): what the forward pass wrote (or its input, without a residual)
    const void* w;
    const void* dh;   // or null
    int w_f32;
    long m, n, ldy, ldh, ldd, ldx;
    float eps;
    void* dx;         // (m, n)
    float* part;      // (groups, n) partial sums of dw
};

// A workgroup takes rows g, g + groups, ...; a lane keeps its columns' part of dw in registers over all of them.  The partial sums
// are joined by reduce_rows_kernel in a fixed order: no atomics, the same bits every time.
template <typename T, int WPR, int NV>
__global__ __launch_bounds__(WPR == 1 ? 256 : WPR * 64) void rms_norm_back_kernel(NormBackParams p) {
    constexpr int TEAMS = WPR == 1 ? 4 : 1;
    constexpr long STEP = WPR * 64 * 8;
    __shared__ float red[WPR];
    __shared__ float sums[TEAMS == 1 ? 1 : 3 * STEP * (NV ? NV : 1)];
    const int team = WPR == 1 ? threadIdx.x >> 6 : 0;
    const int lane = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
    const float inv_n = 1.0f / (float)p.n;
    float* const part = p.part + (long)blockIdx.x * p.n;
    if constexpr (NV > 0) {
        // the weight in registers for all rows; the next row's operands are on their way while a row is reduced (65.6 -> 50 us for 32768 x
        // 1024 in bf16: 4 waves per SIMD alone do not cover the latency), as far as the registers go
        constexpr bool AHEAD = NV * (int)sizeof(T) <= 4;
        float dw[NV][8] = {}, wv[NV][8];
#pragma unroll
        for (int j = 0; j < NV; ++j) load_weight8<T>(p.w, p.w_f32, lane * 8 + j * STEP, p.n, wv[j]);
        struct Row { Vec8<T> h[NV], g[NV], d[NV]; };
        auto fetch = [&](Row& r, long row) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const long c = lane * 8 + j * STEP;
                r.h[j] = load_raw8((const T*)p.h + row * p.ldh + c, p.n - c);
                r.g[j] = load_raw8((const T*)p.dy + row * p.ldy + c, p.n - c);
                if (p.dh) r.d[j] = load_raw8((const T*)p.dh + row * p.ldd + c, p.n - c);
            }
        };
        Row now;
        const long by = (long)gridDim.x * TEAMS;
        long row = (long)blockIdx.x * TEAMS + team;
        if (AHEAD && row < p.m) fetch(now, row);
        for (; row < p.m; row += by) {
            Row next;
            if (AHEAD) {
                if (row + by < p.m) fetch(next, row + by);
            } else {
                fetch(now, row);
            }
            float ss = 0.0f, gh = 0.0f;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float h = vget(now.h[j], i);
                    ss += h * h;
                    gh += vget(now.g[j], i) * wv[j][i] * h;
                }
            ss = row_sum<WPR>(ss, red);
            gh = row_sum<WPR>(gh, red);
            const float rstd = row_rstd(ss, p.n, p.eps);
            const float k = rstd * rstd * (gh * inv_n);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const long c = lane * 8 + j * STEP;
                float d[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float h = vget(now.h[j], i), g = vget(now.g[j], i);
                    dw[j][i] += g * (h * rstd);
                    d[i] = rstd * (g * wv[j][i] - h * k);
                    if (p.dh) d[i] += vget(now.d[j], i);
                }
                if (c < p.n) store8((T*)p.dx + row * p.ldx + c, p.n - c, d);
            }
            if (AHEAD) now = next;
        }
        if (TEAMS > 1) {
            if (team > 0) {
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int i = 0; i < 8; ++i) sums[(team - 1) * STEP * NV + (j * 8 + i) * 64 + lane] = dw[j][i];
            }
            __syncthreads();
            if (team > 0) return;
#pragma unroll
            for (int t = 0; t < TEAMS - 1; ++t)
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int i = 0; i < 8; ++i) dw[j][i] += sums[t * STEP * NV + (j * 8 + i) * 64 + lane];
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (lane * 8 + j * STEP + i < p.n) part[lane * 8 + j * STEP + i] = dw[j][i];
    } else {
        bool first = true;   // (the workgroup's own row of `part` carries the sums: no other workgroup touches it)
        for (long row = blockIdx.x; row < p.m; row += gridDim.x, first = false) {
            float h[8], g[8], wv[8], ss = 0.0f, gh = 0.0f;
            for (long c = lane * 8; c < p.n; c += STEP) {
                load8((const T*)p.h + row * p.ldh + c, p.n - c, h);
                load8((const T*)p.dy + row * p.ldy + c, p.n - c, g);
                load_weight8<T>(p.w, p.w_f32, c, p.n, wv);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    ss += h[i] * h[i];
                    gh += g[i] * wv[i] * h[i];
                }
            }
            ss = row_sum<WPR>(ss, red);
            gh = row_sum<WPR>(gh, red);
            const float rstd = row_rstd(ss, p.n, p.eps);
            const float k = rstd * rstd * (gh * inv_n);
            for (long c = lane * 8; c < p.n; c += STEP) {
                float d[8];
                load8((const T*)p.h + row * p.ldh + c, p.n - c, h);
                load8((const T*)p.dy + row * p.ldy + c, p.n - c, g);
                load_weight8<T>(p.w, p.w_f32, c, p.n, wv);
                if (p.dh) load8((const T*)p.dh + row * p.ldd + c, p.n - c, d);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (c + i < p.n) part[c + i] = (first ? 0.0f : part[c + i]) + g[i] * (h[i] * rstd);
                    const float v = rstd * (g[i] * wv[i] - h[i] * k);
                    d[i] = p.dh ? v + d[i] : v;
                }
                store8((T*)p.dx + row * p.ldx + c, p.n - c, d);
            }
        }
    }
}

// out[c] = sum over g of part[g * n + c] in 64 bits (in 32 the join alone rounded as often as all sums before it), in a fixed order: COLS
// columns per workgroup, 1024 / COLS teams take g = t, t + teams, ..., eight loads of each in flight (one after the other: 11 us for 1024 x
// 1024).  32 columns (whole 128-byte lines) where those give every CU a workgroup, else 16: 1024 x 1024 3.4 us (with 32: 5.0), 512 x 4096 2.8
// (3.5), 512 x 8192 3.6 (with 16: 4.0).
template <typename T, int COLS>
__global__ __launch_bounds__(1024) void reduce_rows_kernel(const float* __restrict__ part, long groups, long n, T* __restrict__ out) {
    constexpr int TEAMS = 1024 / COLS;
    __shared__ double s[16][COLS];
    const int cx = threadIdx.x % COLS, t = threadIdx.x / COLS;
    const long c = (long)blockIdx.x * COLS + cx;
    double a = 0.0;
    if (c < n)
        for (long g = t; g < groups; g += 8 * TEAMS) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = part[min(g + TEAMS * u, groups - 1) * n + c];   // (no branch: hipcc would put the conversions into it)
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = g + TEAMS * u < groups ? v[u] : 0.0f;
            a += (((double)v[0] + v[1]) + ((double)v[2] + v[3])) + (((double)v[4] + v[5]) + ((double)v[6] + v[7]));
        }
#pragma unroll
    for (int d = COLS; d < 64; d *= 2) a += __shfl_xor(a, d);   // the wave's teams
    if ((threadIdx.x & 63) < COLS) s[threadIdx.x >> 6][cx] = a;
    __syncthreads();
    if (t == 0 && c < n) {
        double v[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i & 3] += s[i][cx];
        out[c] = (T)((v[0] + v[1]) + (v[2] + v[3]));
    }
}

}  // namespace mlk
