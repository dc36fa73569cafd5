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
// That is a hundredth of bf16's rounding and a twentieth of fp16's, so results of those types use them: 1.5 % of the bf16 results round to
// the other neighbour than an fp32 product's (2.6e-4 of the norm between the two), both are 1.66e-3 from the exact result.  What it is small
// against is the norm, not each result: where the terms cancel to less than 1e-5 of it, the 16-bit result keeps no digits.  fp32 results do
// not use them: there the codes become bf16 in registers (exact: 4 significant bits; the scale is applied in the same conversion, exact as a
// power of two) and v_mfma_f32_32x32x16_bf16 sums them -- half the rate, 6e-8 of the norm with the result's own rounding.  (The kernel of
// few rows could do that for 16-bit results, too: 1 x 4096 x 4096 5.7 -> 6.3 us, 1 x 1024 x 1024 2.7 -> 3.5; left to who asks for fp32.)
#pragma once
#include <type_traits>

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
    int fast_a, fast_b;     // rows start on 16 bytes: what the LDS-DMA of the ring wants
};

// 16 bytes of row `row` at column `col`; what lies behind the matrix is 0 (codes 0 = value 0)
__device__ __forceinline__ u32x4 load16(const uint8_t* p, long ld, long rows, long k, long row, long col) {
    u32x4 v = {0, 0, 0, 0};
    if (row < rows && col < k) {
        const uint8_t* const at = p + row * ld + col;
        if (col + 16 <= k) {
            v = load_any<u32x4>(at);
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

// 8 codes times 2^(byte - 127) in bf16; a NaN scale makes NaN codes of all of them
__device__ __forceinline__ bf16x8 to_bf16(int c0, int c1, unsigned byte) {
    const unsigned poison = byte == 255 ? 0x7f7f7f7fu : 0u;
    const float scale = __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x3f800000u : byte << 23);
    const unsigned d0 = (unsigned)c0 | poison, d1 = (unsigned)c1 | poison;
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d0, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d0, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d1, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d1, scale, true);
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
    if (j + 4 <= p.n) {
        typedef T t4 __attribute__((ext_vector_type(4)));
        store_any(at, t4{(T)x[0], (T)x[1], (T)x[2], (T)x[3]});
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
            *(u32x4*)(lds[0] + r * QB + ((ch ^ (r & 7)) * 16)) = load16(p.a, p.lda, p.m, p.k, m0 + r, t * QB + ch * 16);
            *(u32x4*)(lds[1] + r * QB + ((ch ^ (r & 7)) * 16)) = load16(p.b, p.ldb, p.n, p.k, n0 + r, t * QB + ch * 16);
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

// ---- the ring kernel: (64 NJ) x (64 NI) of c per workgroup of 4 waves, 32 NJ x 32 NI per wave -----------------------------------
// One wave per SIMD with 4 x 4 matrix tiles (256 accumulators) for large products, 2 x 2 and 1 x 1 (two and four workgroups per CU)
// where the large tiles would be fewer than the CUs.  K runs in steps of 64 through a ring of four LDS slots (rows of 64 bytes, b then a)
// that is filled by LDS-DMA four steps ahead: while step s multiplies, the fragments of s + 1 move into the other register set,
// s + 2 and s + 3 are on their way, and s + 4 is requested into the slot whose fragments were read during s - 1.  One barrier per step;
// the wait in front of it is counted (vmcnt(2 groups): s + 1 has landed).  The compiler does not know the DMA's instructions (inline
// asm without outputs), so no ordinary vector load stands between the first request and the last wait except where a drain is meant
// (the scales of the next 32 blocks).  The scales of 32 blocks of 128 for all rows of both operands lie in LDS behind the ring.
// The last, partial block of 128 comes first, through registers, byte by byte where it must: pieces behind k become 0.
// Rows behind m or n repeat the last one and are not stored.
constexpr int G8_CHUNK = 32;              // blocks of 128 whose scales are in LDS at a time
constexpr int G8_REQ0 = 8;               // streaming kernel: the product of a step behind which its requests begin
constexpr int G8_SPITCH = G8_CHUNK + 4;   // bytes per row of them: 32 rows fall into different banks

// SPLIT: gridDim.y workgroups share the blocks of k of one tile; each stores its part of the sum in fp32 (part y at c + y m n floats, no bias),
// join_splits_kernel adds them in order.
template <typename T, int NI, int NJ, bool SPLIT = false>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(NI * NJ == 16 ? 1 : NI * NJ == 4 ? 2 : 4))) void fp8_gemm_ring_kernel(GemmParams p, int mt, int nt) {
    using OT = std::conditional_t<SPLIT, float, T>;   // what is stored
    constexpr int BN = 64 * NI, BM = 64 * NJ, ROWS = BN + BM, SLOT = ROWS * 64, RING = 4 * SLOT, NQ = NI + NJ;
    __shared__ __attribute__((aligned(16))) char smem[RING + ROWS * G8_SPITCH + BN * 4];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), wn = w & 1, wm = w >> 1;
    const int ml = lane & 31, hh = lane >> 5;

    // workgroup -> tile: consecutive workgroups go round the 8 XCDs; each XCD takes a contiguous run of tiles, in groups of 4 rows of
    // tiles walked column by column, so that the tiles it works on at a time share operands in its L2
    const int tiles = mt * nt, q8 = tiles >> 3, r8 = tiles & 7, xcd = blockIdx.x & 7;
    const int tile = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (blockIdx.x >> 3);
    const int grp = tile / (4 * nt), rem = tile - grp * 4 * nt, gm = min(4, mt - grp * 4);
    const long m0 = (long)(grp * 4 + rem % gm) * BM, n0 = (long)(rem / gm) * BN;

    if constexpr (SPLIT) {   // this workgroup's blocks of k (the last one's may end in a partial block)
        const long kb = (p.k + QB - 1) / QB, each = (kb + gridDim.y - 1) / gridDim.y, b0 = min(each * blockIdx.y, kb), b1 = min(b0 + each, kb);
        p.a += b0 * QB, p.b += b0 * QB, p.sa += b0, p.sb += b0;
        p.k = min(b1 * QB, p.k) - min(b0 * QB, p.k);
        p.c = (float*)p.c + blockIdx.y * p.m * p.n;
        p.ldc = p.n;
        p.bias = nullptr;
    }
    const int nkb = (int)(p.k / QB);                  // whole blocks of 128
    const int nst = 2 * nkb;                          // steps of 64 in the ring
    // ---- DMA: instruction q of this wave fetches 16 rows x 64 bytes; lane = row * 4 + piece, LDS linear, bank swizzle on the source
    unsigned goff[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const bool isb = q < NI;
        const int r = (isb ? (w * NI + q) : (w * NJ + q - NI)) * 16 + (lane >> 2);
        const long last = (isb ? p.n - n0 : p.m - m0) - 1;
        goff[q] = (unsigned)(min((long)r, last) * (isb ? p.ldb : p.lda)) + (((lane & 3) ^ ((r >> 2) & 3)) * 16);
    }
    const uint8_t* rqb = p.b + n0 * p.ldb;   // the next step's first row of each operand (wave-uniform)
    const uint8_t* rqa = p.a + m0 * p.lda;
    const int lds0 = (int)(size_t)(__attribute__((address_space(3))) char*)smem;
    auto request = [&](int slot, int q) {
        const int at = lds0 + slot * SLOT + (q < NI ? (w * NI + q) * 1024 : BN * 64 + (w * NJ + q - NI) * 1024);
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(goff[q]), "s"(q < NI ? rqb : rqa), "s"(at) : "memory");
    };

    // ---- fragments: row (lane & 31) of a 32-row tile, two 16-byte pieces of its 64 (the same two of both operands)
    const int swz = (ml >> 2) & 3;
    const int boff = (wn * 32 * NI + ml) * 64, aoff = BN * 64 + (wm * 32 * NJ + ml) * 64;
    const int c0 = (hh ^ swz) * 16, c1 = ((2 + hh) ^ swz) * 16;
    struct Frag { i32x8 b[NI], a[NJ]; };
    auto join = [](u32x4 x, u32x4 y) { return i32x8{(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]}; };
    auto read_one = [&](Frag& f, const char* slot, int q) {
        if (q < NI) f.b[q] = join(*(const u32x4*)(slot + boff + q * 2048 + c0), *(const u32x4*)(slot + boff + q * 2048 + c1));
        else f.a[q - NI] = join(*(const u32x4*)(slot + aoff + (q - NI) * 2048 + c0), *(const u32x4*)(slot + aoff + (q - NI) * 2048 + c1));
    };
    // scale bytes of this lane's rows
    unsigned sb[NI], sa[NJ], sbn[NI], san[NJ];
    char* const slds = smem + RING;
    auto read_scales = [&](int kb) {
        const char* const at = slds + (kb & (G8_CHUNK - 1));
#pragma unroll
        for (int i = 0; i < NI; ++i) sbn[i] = *(const uint8_t*)(at + (wn * 32 * NI + i * 32 + ml) * G8_SPITCH);
#pragma unroll
        for (int j = 0; j < NJ; ++j) san[j] = *(const uint8_t*)(at + (BN + wm * 32 * NJ + j * 32 + ml) * G8_SPITCH);
    };
    auto scale_row = [&](int r) {   // r < BN: of b, else of a
        if (r < BN) {
            const long row = min(n0 + r, p.n - 1);
            return p.sb + (p.b_tile ? row / QB : row) * p.ldsb;
        }
        const long row = min(m0 + r - BN, p.m - 1);
        return p.sa + (p.a_tile ? row / QB : row) * p.ldsa;
    };
    // blocks kb0 .. kb0 + 31 of the whole ones; a thread takes whole rows and issues all its loads before the first wait (a loop of single
    // loads cost 10 us in front of every tile)
    auto fill_scales = [&](int kb0) {
        constexpr int RT = (ROWS + 255) / 256;
        unsigned v[RT][G8_CHUNK / 4];
        const int have = min(nkb - kb0, G8_CHUNK);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int r = tid + 256 * i;
            const uint8_t* const src = scale_row(r < ROWS ? r : 0) + kb0;
#pragma unroll
            for (int j = 0; j < G8_CHUNK / 4; ++j) {
                v[i][j] = 0;
                if (4 * j + 4 <= have) {
                    __builtin_memcpy(&v[i][j], src + 4 * j, 4);
                } else {
#pragma unroll
                    for (int e = 0; e < 3; ++e)
                        if (4 * j + e < have) v[i][j] |= (unsigned)src[4 * j + e] << (8 * e);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < G8_CHUNK / 4; ++j)
                if (tid + 256 * i < ROWS && 4 * j < have) *(unsigned*)(slds + (tid + 256 * i) * G8_SPITCH + 4 * j) = v[i][j];
    };

    // everything outstanding, by the builtin: hipcc has to know that fill_scales' loads are done (threads without a row never use theirs, and
    // it would wait for them, and with them for every request, inside the steps)
    auto drain = [] {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0);
        asm volatile("" ::: "memory");
    };

    f32x16 acc[NI][NJ];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = f32x16{};

    // one step's products (with fp32 results: through bf16, the codes of one 16-wide k piece at a time)
    auto mul_row = [&](const Frag& f, int i) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = mfma64<T>(f.b[i], f.a[j], acc[i][j], sb[i], sa[j]);
    };

    Frag f0, f1;
    if (p.k > (long)nkb * QB) {   // the partial block
        const long k0 = (long)nkb * QB;
        for (int u = tid; u < ROWS * 8; u += 256) {
            const int half = u / (ROWS * 4), v = u - half * ROWS * 4, r = v >> 2, ch = v & 3;
            const long col = k0 + half * 64 + ch * 16;
            const u32x4 x = r < BN ? load16(p.b, p.ldb, p.n, p.k, n0 + r, col) : load16(p.a, p.lda, p.m, p.k, m0 + r - BN, col);
            *(u32x4*)(smem + half * SLOT + r * 64 + ((ch ^ ((r >> 2) & 3)) * 16)) = x;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NI; ++i) sb[i] = scale_row(wn * 32 * NI + i * 32 + ml)[nkb];
#pragma unroll
        for (int j = 0; j < NJ; ++j) sa[j] = scale_row(BN + wm * 32 * NJ + j * 32 + ml)[nkb];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int q = 0; q < NQ; ++q) read_one(f0, smem + half * SLOT, q);
#pragma unroll
            for (int i = 0; i < NI; ++i) mul_row(f0, i);
        }
        __syncthreads();
    }

    float* const bias = (float*)(slds + ROWS * G8_SPITCH);   // this workgroup's columns
    if (nst > 0) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int st = 0; st < 4; ++st) {
            if (st < nst) {
#pragma unroll
                for (int q = 0; q < NQ; ++q) request(st, q);
                rqb += 64, rqa += 64;
                asm volatile("s_nop 4" ::: "memory");
            }
        }
        const float b = tid < BN ? bias_at(p, n0 + tid) : 0.0f;
        fill_scales(0);   // (its wait is the first steps', too: their latencies overlap)
        if (tid < BN) bias[tid] = b;
        drain();
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < NQ; ++q) read_one(f0, smem, q);
        read_scales(0);

        // One step with the fragments FH; FN receives those of s + 1 (behind the last step: stale ones that nothing uses).  ODD: second
        // half of a block, the next block's scales are read.  WAIT: requests that may be outstanding (-1: no wait).  No branch inside:
        // the compiler would move the products behind it.
        auto step = [&](int s, Frag& FH, Frag& FN, auto odd, auto request4, auto wait) {
            constexpr bool ODD = decltype(odd)::value, MORE = decltype(request4)::value;
            constexpr int WAIT = decltype(wait)::value;
            if constexpr (WAIT >= 0) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(WAIT < 0 ? 0 : WAIT) : "memory");
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (!ODD) {
#pragma unroll
                for (int i = 0; i < NI; ++i) sb[i] = sbn[i];
#pragma unroll
                for (int j = 0; j < NJ; ++j) sa[j] = san[j];
            }
            const char* const next = smem + ((s + 1) & 3) * SLOT;
            // requests and reads behind the first half of the products: the second half covers the last reads' latency in front of the
            // next barrier (spread over all of them, every step waited ~400 of its 1440 cycles there)
            constexpr int NM = NI * NJ, HALF = NM > 1 ? NM / 2 : 1;
#pragma unroll
            for (int x = 0; x < NM; ++x) {
                const int i = x / NJ, j = x % NJ;
                __builtin_amdgcn_sched_barrier(0);
                acc[i][j] = mfma64<T>(FH.b[i], FH.a[j], acc[i][j], sb[i], sa[j]);
                __builtin_amdgcn_sched_barrier(0);
                if (x < HALF) {
#pragma unroll
                    for (int q = x * NQ / HALF; q < (x + 1) * NQ / HALF; ++q) {
                        if constexpr (MORE) request(s & 3, q);
                        read_one(FN, next, q);
                    }
                    if (ODD && x == HALF - 1) read_scales((s + 1) >> 1);
                }
            }
            if constexpr (MORE) rqb += 64, rqa += 64;
        };
        auto chunk = [&](int s) {   // in front of the first step of the next 32 blocks: nobody reads the last ones' scales any more
            if ((s & (2 * G8_CHUNK - 1)) == 0 && s > 0) {
                fill_scales(s >> 1);
                drain();
                __builtin_amdgcn_s_barrier();
                read_scales(s >> 1);
            }
        };
        constexpr std::integral_constant<bool, false> no{};
        constexpr std::integral_constant<bool, true> yes{};
        constexpr std::integral_constant<int, 2 * NQ> two{};
        constexpr std::integral_constant<int, NQ> one{};
        constexpr std::integral_constant<int, 0> all{};
        constexpr std::integral_constant<int, -1> none{};
        int s = 0;
#pragma clang loop unroll(disable)
        for (; s < nst - 4; s += 2) {
            chunk(s);
            step(s, f0, f1, no, yes, two);
            step(s + 1, f1, f0, yes, yes, two);
        }
        if (s < nst - 2) {
            chunk(s);
            step(s, f0, f1, no, no, two);
            step(s + 1, f1, f0, yes, no, one);
            s += 2;
        }
        chunk(s);
        step(s, f0, f1, no, no, all);
        step(s + 1, f1, f0, yes, no, none);
    } else if (tid < BN) {
        bias[tid] = bias_at(p, n0 + tid);
    }

    // ---- epilogue: this wave's rows of c through LDS (the ring and the scales are done with), then whole rows with 16-byte stores.
    // PASS matrix tiles along m at a time, as many as fit; a tile inside c takes straight-line code, eight stores in flight.
    // The lane's number is asked for anew: nothing that depends on it stays in registers through the steps.
    __syncthreads();
    const int el = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)), em = el & 31, eh = el >> 5;
    constexpr int ES = (int)sizeof(OT), ROWB = 32 * NI * ES, PITCH = ROWB + 16, PIECES = ROWB / 16, EV = 16 / ES;
    constexpr int PASS = NJ * 4 * 32 * PITCH <= RING + ROWS * G8_SPITCH ? NJ : NJ / 2;
    static_assert(BN <= 256 && PASS * 4 * 32 * PITCH <= RING + ROWS * G8_SPITCH, "epilogue scratch");
    char* const scr = smem + w * PASS * 32 * PITCH;
    typedef OT t4 __attribute__((ext_vector_type(4)));
    typedef OT tv __attribute__((ext_vector_type(EV)));
    const bool inside = m0 + BM <= p.m && n0 + BN <= p.n;
    const long row0 = m0 + wm * 32 * NJ, col0 = n0 + wn * 32 * NI;
#pragma unroll
    for (int j0 = 0; j0 < NJ; j0 += PASS) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int col = i * 32 + 8 * g + 4 * eh;
                const f32x4 b4 = *(const f32x4*)(bias + wn * 32 * NI + col);
#pragma unroll
                for (int j = 0; j < PASS; ++j) {
                    t4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = (OT)(acc[i][j0 + j][4 * g + e] + b4[e]);
                    *(t4*)(scr + (j * 32 + em) * PITCH + col * ES) = v;
                }
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (a wave's own scratch: no barrier)
        constexpr int UNITS = PASS * 32 * PIECES / 64, STEP = 64 / PIECES;   // a unit: STEP rows
        const int r = el / PIECES, c = el % PIECES;
        const char* const from = scr + r * PITCH + c * 16;
        if (inside) {
            OT* out = (OT*)p.c + (row0 + j0 * 32 + r) * p.ldc + col0 + c * EV;
            const long by = (long)STEP * p.ldc;
#pragma unroll
            for (int u = 0; u < UNITS; u += 8) {
                tv v[8];
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    if (u + x < UNITS) v[x] = *(const tv*)(from + (u + x) * STEP * PITCH);
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    if (u + x < UNITS) {
                        store_any(out, v[x]);
                        out += by;
                    }
            }
        } else {
            const long col = col0 + c * EV;
#pragma clang loop unroll(disable)
            for (int u = 0; u < UNITS; ++u) {
                const long row = row0 + j0 * 32 + r + u * STEP;
                const tv v = *(const tv*)(from + u * STEP * PITCH);
                if (row < p.m && col < p.n) {
                    OT* const out = (OT*)p.c + row * p.ldc + col;
                    if (col + EV <= p.n) {
                        store_any(out, v);
                    } else {
#pragma unroll
                        for (int e = 0; e < EV; ++e)
                            if (col + e < p.n) out[e] = v[e];
                    }
                }
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// c = the sum of the parts, in order, + bias; a part is (m, n) without gaps
template <typename T>
__global__ __launch_bounds__(256) void join_splits_kernel(GemmParams p, const float* __restrict__ part, int splits) {
    const long mn = p.m * p.n, i0 = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i0 >= mn) return;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (i0 + 4 <= mn) {
#pragma unroll 4
        for (int s = 0; s < splits; ++s) v += load_any<f32x4>(part + s * mn + i0);
    } else {
        for (int s = 0; s < splits; ++s)
            for (int e = 0; e < 4; ++e)
                if (i0 + e < mn) v[e] += part[s * mn + i0 + e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const long i = i0 + e, row = i / p.n, col = i - row * p.n;
        if (i < mn) ((T*)p.c)[row * p.ldc + col] = (T)(v[e] + bias_at(p, col));
    }
}

// one accumulator, AGPR -> VGPR, where it is consumed (hipcc by itself copies a hundred of them up front and spills)
__device__ __forceinline__ float from_acc(float a) {
    float v;
    asm("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(a));
    return v;
}

// ---- the streaming kernel: 256 x 256 tiles, 16-bit results, a workgroup per CU that walks tiles without a pause ----------------------
// The ring kernel's steps with 4 x 4 matrix tiles per wave, for k a multiple of 128, n a multiple of 8 (the launch asks for k >= 1024).  There a tile of 16 steps spent 17000 of
// its 38000 cycles outside its products (start and addresses 5000, first latency 3600, epilogue 8000).  Here the last four steps of a tile
// already request the first four of the next one; the next tile's scales and bias are loaded in front of the epilogue and written to LDS
// behind it; and the epilogue needs no LDS: v_permlane32_swap joins the 4 + 4 columns of two lanes into 16 bytes of a row, stored
// straight from registers.  The wait for those loads (younger than the four steps' requests, same counter) also covers the requests, so
// steps 0 .. 2 of a tile wait for nothing and its predecessor's stores retire behind them.
template <typename T>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1))) void fp8_gemm_stream_kernel(GemmParams p, int mt, int nt) {
    static_assert(sizeof(T) == 2, "16-bit results");
    constexpr int NI = 4, NJ = 4, BN = 256, BM = 256, ROWS = 512, SLOT = ROWS * 64, RING = 4 * SLOT, NQ = 8;
    __shared__ __attribute__((aligned(16))) char smem[RING + ROWS * G8_SPITCH + 2 * BN * 4];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), wn = w & 1, wm = w >> 1;
    const int ml = lane & 31, hh = lane >> 5;
    const int nkb = (int)(p.k / QB), nst = 2 * nkb;

    // workgroup -> its tiles: the ring kernel's order, cut into a run per workgroup of an XCD: tile number v, v + grid, ...
    const int tiles = mt * nt, q8 = tiles >> 3, r8 = tiles & 7;
    auto place = [&](int v, long& m0, long& n0) {
        const int xcd = v & 7;
        const int tile = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (v >> 3);
        const int grp = tile / (4 * nt), rem = tile - grp * 4 * nt, gm = min(4, mt - grp * 4);
        m0 = (long)(grp * 4 + rem % gm) * BM, n0 = (long)(rem / gm) * BN;
    };
    long m0, n0;
    place(blockIdx.x, m0, n0);

    unsigned goff[NQ];
    const uint8_t *rqb, *rqa;
    auto aim = [&](long tm, long tn) {   // the request stream to the first step of a tile
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            const bool isb = q < NI;
            const int r = (isb ? (w * NI + q) : (w * NJ + q - NI)) * 16 + (lane >> 2);
            const int last = (int)min((isb ? p.n - tn : p.m - tm) - 1, 255L);
            goff[q] = (unsigned)min(r, last) * (unsigned)(isb ? p.ldb : p.lda) + (((lane & 3) ^ ((r >> 2) & 3)) * 16);
        }
        rqb = p.b + tn * p.ldb;
        rqa = p.a + tm * p.lda;
    };
    const int lds0 = (int)(size_t)(__attribute__((address_space(3))) char*)smem;
    auto request = [&](int slot, int q) {
        const int at = lds0 + slot * SLOT + (q < NI ? (w * NI + q) * 1024 : BN * 64 + (w * NJ + q - NI) * 1024);
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(goff[q]), "s"(q < NI ? rqb : rqa), "s"(at) : "memory");
    };

    const int swz = (ml >> 2) & 3;
    const int boff = (wn * 128 + ml) * 64, aoff = BN * 64 + (wm * 128 + ml) * 64;
    const int c0 = (hh ^ swz) * 16, c1 = ((2 + hh) ^ swz) * 16;
    struct Frag { i32x8 b[NI], a[NJ]; };
    auto join = [](u32x4 x, u32x4 y) { return i32x8{(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]}; };
    auto read_one = [&](Frag& f, const char* slot, int q) {
        if (q < NI) f.b[q] = join(*(const u32x4*)(slot + boff + q * 2048 + c0), *(const u32x4*)(slot + boff + q * 2048 + c1));
        else f.a[q - NI] = join(*(const u32x4*)(slot + aoff + (q - NI) * 2048 + c0), *(const u32x4*)(slot + aoff + (q - NI) * 2048 + c1));
    };
    unsigned sb[NI], sa[NJ], sbn[NI], san[NJ];
    char* const slds = smem + RING;
    float* const bias = (float*)(slds + ROWS * G8_SPITCH);   // of this tile and of the next one, by turns
    int turn = 0;
    auto read_scales = [&](int kb) {
        const char* const at = slds + (kb & (G8_CHUNK - 1));
#pragma unroll
        for (int i = 0; i < NI; ++i) sbn[i] = *(const uint8_t*)(at + (wn * 128 + i * 32 + ml) * G8_SPITCH);
#pragma unroll
        for (int j = 0; j < NJ; ++j) san[j] = *(const uint8_t*)(at + (BN + wm * 128 + j * 32 + ml) * G8_SPITCH);
    };
    // scales of blocks kb0 .. kb0 + 31: a thread has one row of b and one of a
    struct Scales { unsigned v[2][G8_CHUNK / 4]; float bias; };
    auto load_scales = [&](Scales& t, long tm, long tn, int kb0) {
        const int have = min(nkb - kb0, G8_CHUNK);
        const long rb = min(tn + tid, p.n - 1), ra = min(tm + tid, p.m - 1);
        const uint8_t* const src[2] = {p.sb + (p.b_tile ? rb / QB : rb) * p.ldsb + kb0, p.sa + (p.a_tile ? ra / QB : ra) * p.ldsa + kb0};
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < G8_CHUNK / 4; ++j) {
                t.v[i][j] = 0;
                if (4 * j + 4 <= have) {
                    __builtin_memcpy(&t.v[i][j], src[i] + 4 * j, 4);
                } else {
#pragma unroll
                    for (int e = 0; e < 3; ++e)
                        if (4 * j + e < have) t.v[i][j] |= (unsigned)src[i][4 * j + e] << (8 * e);
                }
            }
        t.bias = bias_at(p, tn + tid);
    };
    auto write_scales = [&](const Scales& t, int turn) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < G8_CHUNK / 4; ++j) *(unsigned*)(slds + (tid + 256 * i) * G8_SPITCH + 4 * j) = t.v[i][j];
        bias[turn * BN + tid] = t.bias;
    };

    f32x16 acc[NI][NJ];
    int s0 = 0;   // steps of the tiles before this one: the ring goes on
    // as in the ring kernel; FIRST: the products start from 0, and nothing is waited for in steps 0 .. 2
    auto step = [&](int s, Frag& FH, Frag& FN, auto odd, auto first, auto wait) {
        constexpr bool ODD = decltype(odd)::value, FIRST = decltype(first)::value;
        constexpr int WAIT = decltype(wait)::value;
        if constexpr (WAIT >= 0) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(WAIT < 0 ? 0 : WAIT) : "memory");
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!ODD) {
#pragma unroll
            for (int i = 0; i < NI; ++i) sb[i] = sbn[i];
#pragma unroll
            for (int j = 0; j < NJ; ++j) sa[j] = san[j];
        }
        const char* const next = smem + ((s0 + s + 1) & 3) * SLOT;
        const int slot = (s0 + s) & 3;
#pragma unroll
        for (int x = 0; x < NI * NJ; ++x) {
            const int i = x / NJ, j = x % NJ;
            __builtin_amdgcn_sched_barrier(0);
            acc[i][j] = mfma64<T>(FH.b[i], FH.a[j], FIRST ? f32x16{} : acc[i][j], sb[i], sa[j]);
            __builtin_amdgcn_sched_barrier(0);
            if (x < NQ) read_one(FN, next, x);
            if (ODD && x == NQ) read_scales((s + 1) >> 1);
            if (x >= G8_REQ0 && x < G8_REQ0 + NQ) request(slot, x - G8_REQ0);
        }
        rqb += 64, rqa += 64;
    };
    constexpr std::integral_constant<bool, false> no{};
    constexpr std::integral_constant<bool, true> yes{};
    constexpr std::integral_constant<int, 2 * NQ> two{};
    constexpr std::integral_constant<int, -1> none{};

    Frag f0, f1;
    aim(m0, n0);
#pragma unroll
    for (int st = 0; st < 4; ++st) {
        asm volatile("s_nop 4" ::: "memory");
#pragma unroll
        for (int q = 0; q < NQ; ++q) request(st, q);
        rqb += 64, rqa += 64;
    }
    {
        Scales t;
        load_scales(t, m0, n0, 0);
        write_scales(t, 0);
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int q = 0; q < NQ; ++q) read_one(f0, smem, q);
    read_scales(0);

    for (int v = blockIdx.x;;) {
        const int vn = v + (int)gridDim.x;
        const bool more = vn < tiles;   // (the same for the whole workgroup)
        long mn = m0, nn = n0;
        // (16 steps at least: the last four, which request the next tile's first ones, are in the loop)
        step(0, f0, f1, no, yes, none);
        step(1, f1, f0, yes, no, none);
        step(2, f0, f1, no, no, none);
        step(3, f1, f0, yes, no, two);
#pragma clang loop unroll(disable)
        for (int s = 4; s < nst; s += 2) {
            if (s == nst - 4) {   // from here on the next tile's steps (behind the last tile: its own first ones again, which nothing reads)
                if (more) place(vn, mn, nn);
                aim(mn, nn);
                asm volatile("s_nop 4" ::: "memory");
            }
            if ((s & (2 * G8_CHUNK - 1)) == 0) {   // the next 32 blocks' scales; nobody reads the last ones' any more
                Scales t;
                load_scales(t, m0, n0, s >> 1);
                write_scales(t, turn);
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                read_scales(s >> 1);
            }
            step(s, f0, f1, no, no, two);
            step(s + 1, f1, f0, yes, no, two);   // (the last one: f0 = the next tile's first fragments)
        }

        // ---- epilogue, with the next tile's scales on their way (the accumulators are read by asm, for which hipcc pads nothing: a
        // matrix instruction's result may be read 18 wait states behind it)
        asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        Scales t;
        load_scales(t, mn, nn, 0);
        // (a lane's 8 columns are wholly inside or outside: n is a multiple of 8)
        T* const out0 = (T*)p.c + (m0 + wm * 128 + ml) * p.ldc + n0 + wn * 128 + 8 * hh;
        const int rows = (int)min(p.m - (m0 + wm * 128 + ml), 128L), cols = (int)min(p.n - (n0 + wn * 128 + 8 * hh), 128L);
        auto columns = [&](auto edge) {   // EDGE: a branch around every store
            constexpr bool EDGE = decltype(edge)::value;
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                f32x4 b4[4];
#pragma unroll
                for (int g = 0; g < 4; ++g) b4[g] = *(const f32x4*)(bias + turn * BN + wn * 128 + i * 32 + 8 * g + 4 * hh);
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {   // columns 16 h .. 16 h + 15 of the matrix tile: lanes below 32 get the first 8, the others the last
                        typedef T t2 __attribute__((ext_vector_type(2)));
                        unsigned d[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int g = 2 * h + (e >> 1), k = 4 * g + 2 * (e & 1);
                            d[e] = __builtin_bit_cast(unsigned, t2{(T)(from_acc(acc[i][j][k]) + b4[g][2 * (e & 1)]), (T)(from_acc(acc[i][j][k + 1]) + b4[g][2 * (e & 1) + 1])});
                        }
                        const auto x = __builtin_amdgcn_permlane32_swap(d[0], d[2], false, false), y = __builtin_amdgcn_permlane32_swap(d[1], d[3], false, false);
                        const u32x4 q = {(unsigned)x[0], (unsigned)y[0], (unsigned)x[1], (unsigned)y[1]};
                        if (!EDGE || (j * 32 < rows && i * 32 + h * 16 < cols)) store_any(out0 + (long)j * 32 * p.ldc + i * 32 + h * 16, q);
                    }
            }
        };
        if (m0 + BM <= p.m && n0 + BN <= p.n) columns(no);
        else columns(yes);
        turn ^= 1;
        write_scales(t, turn);   // (nobody reads the last scales any more; the bias has its own place)
        // (its wait: everything older than these loads has landed, the next tile's four steps among it)
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        if (!more) break;
        read_scales(0);
        s0 += nst, v = vn, m0 = mn, n0 = nn;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (no LDS-DMA is under way when the workgroup gives its LDS back)
}

// ---- few rows of a: 16 MT x 16 of c per workgroup of 8 waves, which share the blocks of k --------------------------------------
// Bound by reading b once (for one row: 16 MB of a 4096 x 4096 weight), so every CU pulls on it: n / 16 workgroups, each wave takes every
// eighth block of 128 straight into fragments (16 rows x 128 contiguous bytes per load pair, no LDS), U blocks in flight; the eight partial
// results meet in LDS in a fixed order.  Right for every stride and alignment.
template <typename T>
__device__ __forceinline__ f32x4 mfma128(i32x8 a, i32x8 b, f32x4 c, unsigned sa, unsigned sb) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int s = 0; s < 4; ++s)
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16(a[2 * s], a[2 * s + 1], sa), to_bf16(b[2 * s], b[2 * s + 1], sb), c, 0, 0, 0);
        return c;
    } else {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, (int)sa, 0, (int)sb);
    }
}

template <typename T, int MT, int U>
__global__ __launch_bounds__(512) void fp8_gemm_rows_kernel(GemmParams p) {
    constexpr int WAVES = 8;
    __shared__ __attribute__((aligned(16))) float part[WAVES][MT][64][4];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, lr = lane & 15, lg = lane >> 4;
    const long n0 = (long)blockIdx.x * 16, kb = (p.k + QB - 1) / QB;
    const long brow = min(n0 + lr, p.n - 1);
    const uint8_t* const sb = p.sb + (p.b_tile ? brow / QB : brow) * p.ldsb;
    const uint8_t* sa[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const long r = min((long)(i * 16 + lr), p.m - 1);
        sa[i] = p.sa + (p.a_tile ? r / QB : r) * p.ldsa;
    }
    auto frag = [&](const uint8_t* x, long ld, long rows, long row, long col) {
        const u32x4 u = load16(x, ld, rows, p.k, row, col), v = load16(x, ld, rows, p.k, row, col + 16);
        return i32x8{(int)u[0], (int)u[1], (int)u[2], (int)u[3], (int)v[0], (int)v[1], (int)v[2], (int)v[3]};
    };
    f32x4 acc[MT] = {};
    for (long t = w; t < kb; t += WAVES * U) {
        i32x8 fb[U], fa[U][MT];
        unsigned xb[U], xa[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long b = t + u * WAVES, col = b * QB + lg * 32;    // (behind the last block: zeros, scale 1)
            fb[u] = frag(p.b, p.ldb, p.n, n0 + lr, col);
            xb[u] = b < kb ? sb[b] : 127;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                fa[u][i] = frag(p.a, p.lda, p.m, i * 16 + lr, col);
                xa[u][i] = b < kb ? sa[i][b] : 127;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i] = mfma128<T>(fb[u], fa[u][i], acc[i], xb[u], xa[u][i]);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) *(f32x4*)part[w][i][lane] = acc[i];
    __syncthreads();
    for (int e = threadIdx.x; e < MT * 256; e += 512) {    // element (row i * 16 + r, column c): neighbouring threads, neighbouring columns
        const int c = e & 15, r = (e >> 4) & 15, i = e >> 8;
        const long row = i * 16 + r, col = n0 + c;
        if (row >= p.m || col >= p.n) continue;
        float v = 0.0f;
#pragma unroll
        for (int x = 0; x < WAVES; ++x) v += part[x][i][(c >> 2) * 16 + r][c & 3];
        ((T*)p.c)[row * p.ldc + col] = (T)(v + bias_at(p, col));
    }
}

}  // namespace mlk
