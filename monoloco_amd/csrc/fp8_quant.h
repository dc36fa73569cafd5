// fp8_quant.h -- fp32 / bf16 / fp16 matrices -> e4m3 blocks of 128 (block8.h): along rows (1 x 128), as 128 x 128 tiles, and the
// transposed matrix in the same pass (a backward product reduces over the other axis, and the matrix instruction wants both
// operands contiguous along the reduction).  Bound by memory: every element is read once, also where two forms are written.
#pragma once
#include "block8.h"

namespace mlk {

struct QuantParams {
    const void* x;      // (m, n), row stride ldx
    long m, n, ldx;
    int tile;           // one scale per 128 x 128 instead of 1 x 128
    uint8_t* q;         // (m, n), row stride ldq, or null
    uint8_t* scale;     // (m, nb) or (mb, nb), row stride lds
    long ldq, lds;
    uint8_t* qt;        // (n, m), row stride ldqt, or null
    uint8_t* scale_t;   // (n, mb) or (nb, mb), row stride ldst
    long ldqt, ldst;
    float* colsum;      // (mb, n): column sums of every 128 rows, or null
};

// rows only: 16 lanes per block of 128, no LDS
template <typename T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantParams p) {
    const long nb = (p.n + QB - 1) / QB, units = p.m * nb;
    const long u = (long)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (u >= units) return;   // (whole groups of 16 lanes)
    const long row = u / nb, b = u - row * nb, c = b * QB + (threadIdx.x & 15) * 8;
    float x[8];
    load8((const T*)p.x + row * p.ldx + c, p.n - c, x);
    unsigned a = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) a = max(a, absbits(x[i]));
    const unsigned byte = scale_byte(max16(a));
    if (c < p.n) store_codes8(p.q + row * p.ldq + c, p.n - c, codes8(x, byte));
    if ((threadIdx.x & 15) == 0) p.scale[row * p.lds + b] = (uint8_t)byte;
}

// a 128 x 128 tile per workgroup of 256 threads: thread (tr, tc) = (t / 16, t % 16) holds rows 8 tr .. + 7, columns 8 tc .. + 7 as they
// came (fp32 copies of them would cost half the occupancy).  Rows are stored 16 bytes a lane (two lanes trade rows for columns); the
// transposed tile goes through LDS, its 16-byte pieces exchanged by row / 8 against bank conflicts.  Three waves per SIMD: four would spill
// (16384 x 4096 bf16, both forms: 70.6 us with four, 52.0 with three = 5.2 TB/s).
template <typename T>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(3))) void quantize_tile_kernel(QuantParams p) {
    __shared__ unsigned cmax[4][QB];
    __shared__ float csum[4][QB];
    __shared__ __attribute__((aligned(16))) uint8_t tq[QB * QB];
    const int tc = threadIdx.x & 15, tr = threadIdx.x >> 4, wave = threadIdx.x >> 6;
    const long nb = (p.n + QB - 1) / QB;
    const long bi = blockIdx.x / nb, bj = blockIdx.x - bi * nb;
    const long r0 = bi * QB + tr * 8, c0 = bj * QB + tc * 8;
    Vec8<T> x[8];
    unsigned rmax[8], colmax[8] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = load_raw8((const T*)p.x + (r0 + i) * p.ldx + c0, r0 + i < p.m ? p.n - c0 : 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        rmax[i] = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const unsigned a = absbits(vget(x[i], j));
            rmax[i] = max(rmax[i], a);
            colmax[j] = max(colmax[j], a);
        }
        rmax[i] = max16(rmax[i]);
    }
    // columns (and sums): over the four row groups of a wave, then over the four waves
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const auto y = __builtin_amdgcn_permlane16_swap(colmax[j], colmax[j], false, false);
        const unsigned h = max((unsigned)y[0], (unsigned)y[1]);
        const auto z = __builtin_amdgcn_permlane32_swap(h, h, false, false);
        if ((threadIdx.x & 48) == 0) cmax[wave][tc * 8 + j] = max((unsigned)z[0], (unsigned)z[1]);
        if (p.colsum) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) s += vget(x[i], j);
            s += __shfl_xor(s, 16);
            s += __shfl_xor(s, 32);
            if ((threadIdx.x & 48) == 0) csum[wave][tc * 8 + j] = s;
        }
    }
    __syncthreads();
    unsigned tb = 0;
    if (p.tile) {
        unsigned a = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) a = max(a, max(max(cmax[0][tc * 8 + j], cmax[1][tc * 8 + j]), max(cmax[2][tc * 8 + j], cmax[3][tc * 8 + j])));
        tb = scale_byte(max16(a));
    }
    if (p.colsum && threadIdx.x < QB && bj * QB + threadIdx.x < p.n) {
        const int c = threadIdx.x;
        p.colsum[bi * p.n + bj * QB + c] = (csum[0][c] + csum[1][c]) + (csum[2][c] + csum[3][c]);
    }
    if (p.q) {
        const bool odd = tc & 1;
        const long cc = c0 - (odd ? 8 : 0);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            u32x2 own[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const unsigned byte = p.tile ? tb : scale_byte(rmax[i + e]);
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = vget(x[i + e], j);
                own[e] = codes8(v, byte);
                if (!p.tile && tc == 0 && r0 + i + e < p.m) p.scale[(r0 + i + e) * p.lds + bj] = (uint8_t)byte;
            }
            // even lanes keep row i and get the odd neighbour's 8 columns of it; odd lanes row i + 1
            u32x4 v;
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                const unsigned give = odd ? own[0][d] : own[1][d], keep = odd ? own[1][d] : own[0][d];
                const unsigned got = (unsigned)__builtin_amdgcn_update_dpp(0, (int)give, 0xb1, 0xf, 0xf, false);   // quad_perm 1 0 3 2
                v[d] = odd ? got : keep;
                v[2 + d] = odd ? keep : got;
            }
            const long row = r0 + i + (odd ? 1 : 0);
            if (row < p.m && cc < p.n) store_codes16(p.q + row * p.ldq + cc, p.n - cc, v);
        }
        if (p.tile && threadIdx.x == 0) p.scale[bi * p.lds + bj] = (uint8_t)tb;
    }
    if (p.qt) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = tc * 8 + j;
            const unsigned byte = p.tile ? tb : scale_byte(max(max(cmax[0][c], cmax[1][c]), max(cmax[2][c], cmax[3][c])));
            float col[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) col[i] = vget(x[i], j);
            *(u32x2*)(tq + c * QB + (((tr >> 1) ^ (tc & 7)) * 16) + (tr & 1) * 8) = codes8(col, byte);
            if (!p.tile && tr == 0 && c0 + j < p.n) p.scale_t[(c0 + j) * p.ldst + bi] = (uint8_t)byte;
        }
        if (p.tile && threadIdx.x == 0) p.scale_t[bj * p.ldst + bi] = (uint8_t)tb;
        __syncthreads();
        // row c of the transposed tile: 8 lanes x 16 bytes
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int c = (threadIdx.x >> 3) + 32 * k, ch = threadIdx.x & 7;
            const long rt = bj * QB + c, ct = bi * QB + ch * 16;
            if (rt < p.n && ct < p.m) store_codes16(p.qt + rt * p.ldqt + ct, p.m - ct, *(const u32x4*)(tq + c * QB + ((ch ^ ((c >> 3) & 7)) * 16)));
        }
    }
}

}  // namespace mlk
