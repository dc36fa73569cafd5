// fp8.hip -- C entry points of the 8-bit residual-block operators: quantisation into e4m3 blocks of 128, the block-scaled product,
// root-mean-square norm with residual (8-bit or plain output) and its backward pass.  All are asynchronous on the caller's stream,
// allocate nothing and keep nothing between calls (a workspace is an argument), so they may be captured into a graph.
#include <algorithm>

#include "fp8_gemm.h"
#include "fp8_quant.h"
#include "norm_kernels.h"

using namespace mlk;

namespace {

// a launch has fewer than 2^32 threads
bool fits(long workgroups, int threads) { return workgroups <= 0xffffffffL / threads; }

// a matrix that memory could hold (2^46 elements, 2^40 along an axis); beyond it, sums and products of sizes would leave 64 bits
bool holds(int64_t rows, int64_t cols) { return rows <= 1LL << 40 && cols <= 1LL << 40 && (rows == 0 || cols <= (1LL << 46) / rows); }
bool holds(int64_t m, int64_t n, int64_t k) { return holds(m, n) && holds(m, k) && holds(n, k); }

int elem_size(int dtype) { return dtype == ML_F32 ? 4 : dtype == ML_BF16 || dtype == ML_F16 ? 2 : 0; }

bool rows_aligned(const void* p, long ld, int es, int to) { return !p || (((uintptr_t)p % to) == 0 && (ld * es) % to == 0); }

// `rows` runs of `width` bytes, `pitch` apart
struct Area { int64_t at, pitch, width, rows; };
// Do a result and an operand share no byte?  Exact where the operand is one run or both have the same pitch (columns of one buffer); runs
// of different pitches that interleave count as shared.
bool apart(const Area& c, const Area& t) {
    if (c.rows <= 0 || c.width <= 0 || t.rows <= 0 || t.width <= 0) return true;
    auto end = [](const Area& x) { return (__int128)x.at + (__int128)(x.rows - 1) * x.pitch + x.width; };
    if (end(c) <= t.at || end(t) <= c.at) return true;
    const int64_t d = t.at - c.at;
    if (t.rows == 1) {   // the first run of c that ends behind t's start: does it start behind t's end?
        const int64_t r = c.rows == 1 || d < c.width ? 0 : (d - c.width) / c.pitch + 1;
        return r >= c.rows || (__int128)r * c.pitch >= (__int128)d + t.width;
    }
    if (c.rows == 1) return apart(t, c);
    if (c.pitch != t.pitch) return false;
    const int64_t x = (d % c.pitch + c.pitch) % c.pitch;
    return x >= c.width && x + t.width <= c.pitch;
}

// f(T{}) for the element type
template <typename F>
void with_type(int dtype, F f) {
    if (dtype == ML_F32) f(float{});
    else if (dtype == ML_BF16) f(bf16_t{});
    else f(f16_t{});
}

template <typename T, bool OUT8>
void launch_norm(const NormParams& p, hipStream_t s) {
    const unsigned g4 = (unsigned)((p.m + 3) / 4), g1 = (unsigned)p.m;
    if (p.n <= 512) rms_norm_kernel<T, OUT8, 1, 1><<<g4, 256, 0, s>>>(p);
    else if (p.n <= 1024) rms_norm_kernel<T, OUT8, 1, 2><<<g4, 256, 0, s>>>(p);
    else if (p.n <= 2048) rms_norm_kernel<T, OUT8, 1, 4><<<g4, 256, 0, s>>>(p);
    else if (p.n <= 4096) rms_norm_kernel<T, OUT8, 4, 2><<<g1, 256, 0, s>>>(p);
    else if (p.n <= 8192) rms_norm_kernel<T, OUT8, 4, 4><<<g1, 256, 0, s>>>(p);
    else if (p.n <= 16384) rms_norm_kernel<T, OUT8, 8, 4><<<g1, 512, 0, s>>>(p);
    else if (p.n <= 32768) rms_norm_kernel<T, OUT8, 16, 4><<<g1, 1024, 0, s>>>(p);
    else rms_norm_kernel<T, OUT8, 16, 0><<<g1, 1024, 0, s>>>(p);
}

template <typename T>
void launch_norm_back(const NormBackParams& p, unsigned g, hipStream_t s) {
    if (p.n <= 512) rms_norm_back_kernel<T, 1, 1><<<g, 256, 0, s>>>(p);
    else if (p.n <= 1024) rms_norm_back_kernel<T, 1, 2><<<g, 256, 0, s>>>(p);
    else if (p.n <= 2048) rms_norm_back_kernel<T, 1, 4><<<g, 256, 0, s>>>(p);
    else if (p.n <= 4096) rms_norm_back_kernel<T, 4, 2><<<g, 256, 0, s>>>(p);
    else if (p.n <= 8192) rms_norm_back_kernel<T, 4, 4><<<g, 256, 0, s>>>(p);
    else if (p.n <= 16384) rms_norm_back_kernel<T, 8, 4><<<g, 512, 0, s>>>(p);   // (16 waves leave 128 registers each: spills)
    else rms_norm_back_kernel<T, 16, 0><<<g, 1024, 0, s>>>(p);
}

// Which product kernel (us measured on both sides of each border, bf16 results unless said):
//   m <= 32 rows (fp32 results: 64): the waves of a workgroup share k.  4096 x 4096, m = 32: 10.5 against 12.9 with 64 x 64 tiles; m = 64:
//     16.4 against 13.1, fp32 18.1 against 24.6.
//   The ring wants rows that start on 16 bytes and offsets inside a tile below 2^32; everything else takes the plain 64 x 64 kernel.
//   64 x 64 tiles while they fit the CUs once (or, k <= 2048, twice): 512 x 1024 x 1024 5.7 against 7.9 with 128 x 128; 2048 x 1024 x 1024
//     7.0 against 8.4; 384 x 4096 x 4096 (384 tiles) 22.4 against 18.5.  fp32: while the 128 x 128 tiles are fewer than the CUs.
//   256 x 256 tiles once they are more than the CUs, or k >= 2048 and 160 of them: 16384 x 1024 x 1024 (256 tiles) 26.9
//     against 24.6 with 128 x 128, 32768 x 1024 x 1024 44.7 against 48.9; 2048 x 4096 x 4096 (128) 47.1 against 40.9, 4096^3 (256) 59.7
//     against 77.9; below k = 1024 a tile's start and end outweigh its steps.  fp32: 2560 x 4096 x 4096 (160) 97 against 98, 4096^3 114 against
//     133, 8192^3 856 against 986.
//   Few tiles and a long k (the weight gradient of a large batch): 128 x 128 tiles whose blocks of k are shared by several workgroups, where
//     that is estimated to be faster than the kernels above: gemm_splits.
struct Tiles {
    long t256, t128, t64;
    Tiles(long m, long n) {
        auto across = [&](long t) { return (m + t - 1) / t * ((n + t - 1) / t); };
        t256 = across(256), t128 = across(128), t64 = across(64);
    }
};

// In how many parts k is cut, 1: not at all.  Estimates in us, from products of 9 .. 2048 rows and k = 4096 .. 65536: a step of 64 takes a
// 128 x 128 tile 0.29 (fp32 results: 0.55) alone on its CU and 0.55 (0.95) beside another one, a lone 64 x 64 tile 0.17 (0.29), the kernels of
// few rows 0.068 (m <= 16), 0.11 (m <= 32) and 0.2 (fp32, m <= 64); the operands come at 5.2 TB/s at best, the parts are written and read at
// 4.5 and joined by a launch of 4. Cut where that says 18 % less, into the parts with the least.  Uncut against cut, bf16 (fp32): 1024 x 1024 x
// 65536 171 against 86 (292, 149), x 16384 44 against 32 (75, 51); 1024 x 2048 x 8192 36.5 against 32.0 (left: 65, 58); 256 x 256 x 65536 156
// against 23 (287, 27); 512 x 512 x 8192 19.7 against 15.9 (38, 21); 128 x 4096 x 16384 41 against 24 (75, 34); 9 x 1024 x 65536 72 against 21
// (74, 31), x 16384 19.9 against 13.0 (20.9, 18.5); 32 x 1024 x 8192 18.6 against 12.3 (left: 19.0, 17.5); fp32 1920 x 1920 x 16384 195 against
// 141.  Left uncut in bf16: 9 x 1024 x 8192 10.9 against 11.5, 1 x 4096 x 16384 17.8 against 18.8, 256 x 256 x 4096 11.1 against 11.2, 1920 x
// 1920 x 16384 73 against 92 in two parts.
int gemm_splits(long m, long n, long k, bool half) {
    const Tiles t(m, n);
    const long kb = (k + QB - 1) / QB;
    if (t.t128 >= 256 || kb < 16) return 1;
    const double steps = 2.0 * kb, bytes = (double)(m + n) * k, lone = half ? 0.29 : 0.55, pair = half ? 0.55 : 0.95;
    const double uncut = m <= 16 ? 0.068 : m <= 32 ? 0.11 : half ? (t.t64 <= 256 ? 0.17 : 0.29) : m <= 64 ? 0.2 : 0.29 * std::max(1.0, 0.75 * t.t64 / 256);
    const long most = std::min({512 / t.t128, kb / 8, 64L});
    int best = 1;
    double least = 0.82 * steps * uncut;
    for (long s = 2; s <= most; ++s) {
        const double us = std::max(steps / s * (s * t.t128 <= 256 ? lone : pair), bytes / 5.2e6) + s * (double)(m * n) * 8.0 / 4.5e6 + 4.0;
        if (us < least) least = us, best = (int)s;
    }
    return best;
}

int64_t gemm_work_bytes(long m, long n, long k, bool half) {
    const int s = gemm_splits(m, n, k, half);
    return s > 1 ? (int64_t)s * m * n * 4 : 0;
}

template <typename T>
void launch_gemm(const GemmParams& p, float* work, int64_t work_bytes, hipStream_t s) {
    constexpr bool HALF = sizeof(T) == 2;
    const bool ring = p.fast_a && p.fast_b && p.lda < (1L << 23) && p.ldb < (1L << 23);
    const Tiles t(p.m, p.n);
    const long t256 = t.t256, t128 = t.t128, t64 = t.t64;
    const int splits = ring && work && (uintptr_t)work % 16 == 0 && work_bytes >= gemm_work_bytes(p.m, p.n, p.k, HALF) ? gemm_splits(p.m, p.n, p.k, HALF) : 1;
    auto tiles = [](long size, int t) { return (int)((size + t - 1) / t); };
    const long g16 = (p.n + 15) / 16;
    if (splits > 1) {
        GemmParams q = p;
        q.c = work;
        fp8_gemm_ring_kernel<T, 2, 2, true><<<dim3((unsigned)t128, (unsigned)splits), 256, 0, s>>>(q, tiles(p.m, 128), tiles(p.n, 128));
        join_splits_kernel<T><<<(unsigned)((p.m * p.n + 1023) / 1024), 256, 0, s>>>(p, work, splits);
    } else if (p.m <= 16 && fits(g16, 512)) {
        fp8_gemm_rows_kernel<T, 1, 4><<<(unsigned)g16, 512, 0, s>>>(p);
    } else if (p.m <= 32 && fits(g16, 512)) {
        fp8_gemm_rows_kernel<T, 2, 2><<<(unsigned)g16, 512, 0, s>>>(p);
    } else if (!HALF && p.m <= 64 && fits(g16, 512)) {
        if constexpr (!HALF) fp8_gemm_rows_kernel<T, 4, 2><<<(unsigned)g16, 512, 0, s>>>(p);
    } else if (!ring) {
        fp8_gemm64_kernel<T><<<(unsigned)t64, 256, 0, s>>>(p);
    } else if (p.k >= 1024 && (t256 > 256 || (t256 >= 160 && p.k >= 2048))) {
        bool streamed = false;
        if constexpr (HALF) {
            streamed = p.k % QB == 0 && p.n % 8 == 0;
            if (streamed) fp8_gemm_stream_kernel<T><<<(unsigned)(t256 < 256 ? t256 : 256), 256, 0, s>>>(p, tiles(p.m, 256), tiles(p.n, 256));
        }
        if (!streamed) fp8_gemm_ring_kernel<T, 4, 4><<<(unsigned)t256, 256, 0, s>>>(p, tiles(p.m, 256), tiles(p.n, 256));
    } else if (HALF ? t64 <= (p.k <= 2048 ? 512 : 256) : t128 < 256) {
        fp8_gemm_ring_kernel<T, 1, 1><<<(unsigned)t64, 256, 0, s>>>(p, tiles(p.m, 64), tiles(p.n, 64));
    } else {
        fp8_gemm_ring_kernel<T, 2, 2><<<(unsigned)t128, 256, 0, s>>>(p, tiles(p.m, 128), tiles(p.n, 128));
    }
}

// workgroups of the backward pass = rows of its partial sums: enough to fill 256 CUs with 16 waves, few enough that writing and
// joining their sums stays below a thirtieth of the traffic from 32768 rows on
long norm_groups(long m, long n) {
    const long teams = n <= 2048 ? 4 : 1, most = n <= 8192 ? 1024 : 512;
    const long g = (m + teams - 1) / teams;
    return g < most ? g : most;
}

template <typename T>
void launch_reduce(const float* part, long groups, long n, T* out, hipStream_t s) {
    if (n >= 256 * 32) reduce_rows_kernel<T, 32><<<(unsigned)((n + 31) / 32), 1024, 0, s>>>(part, groups, n, out);
    else reduce_rows_kernel<T, 16><<<(unsigned)((n + 15) / 16), 1024, 0, s>>>(part, groups, n, out);
}

// the bias gradient alone: the tile kernel without either form of codes
int column_sums(const void* x, int dtype, int64_t m, int64_t n, int64_t ldx, float* out, hipStream_t s) {
    const int es = elem_size(dtype);
    if (!es || (m && n && ldx < n)) return ops_fail(ML_ERR_ARG, "column sums: bad type %d or row stride", dtype);
    if (m == 0 || n == 0) return ML_OK;
    QuantParams p{};
    p.x = x, p.m = m, p.n = n, p.ldx = ldx, p.colsum = out;
    const long grid = ((n + QB - 1) / QB) * ((m + QB - 1) / QB);
    if (!fits(grid, 256)) return ops_fail(ML_ERR_SHAPE, "column sums: %lld x %lld is too large", (long long)m, (long long)n);
    with_type(dtype, [&](auto t) { quantize_tile_kernel<decltype(t)><<<(unsigned)grid, 256, 0, s>>>(p); });
    return ops_launched("column sums");
}

}  // namespace

extern "C" {

const char* ml_ops_last_error(void) { return g_ops_err; }

int ml_fp8_quantize(const void* x_dev, int dtype, int64_t m, int64_t n, int64_t ldx, int tile, uint8_t* q_dev, int64_t ldq,
                    uint8_t* scale_dev, int64_t lds, uint8_t* qt_dev, int64_t ldqt, uint8_t* scale_t_dev, int64_t ldst,
                    float* colsum_dev, void* stream) {
    const int es = elem_size(dtype);
    if (!es || m < 0 || n < 0) return ops_fail(ML_ERR_ARG, "ml_fp8_quantize: bad type %d or size %lld x %lld", dtype, (long long)m, (long long)n);
    if (m == 0 || n == 0) return ML_OK;
    if (!x_dev || (!q_dev && !qt_dev) || (q_dev && !scale_dev) || (qt_dev && !scale_t_dev)) return ops_fail(ML_ERR_ARG, "ml_fp8_quantize: null pointer");
    if (!holds(m, n)) return ops_fail(ML_ERR_SHAPE, "ml_fp8_quantize: %lld x %lld is too large", (long long)m, (long long)n);
    const long nb = (n + QB - 1) / QB, mb = (m + QB - 1) / QB;
    if (ldx < n || (q_dev && (ldq < n || lds < nb)) || (qt_dev && (ldqt < m || ldst < mb)))
        return ops_fail(ML_ERR_ARG, "ml_fp8_quantize: a row stride is shorter than its row");
    QuantParams p{};
    p.x = x_dev, p.m = m, p.n = n, p.ldx = ldx, p.tile = tile != 0;
    p.q = q_dev, p.scale = scale_dev, p.ldq = ldq, p.lds = lds;
    p.qt = qt_dev, p.scale_t = scale_t_dev, p.ldqt = ldqt, p.ldst = ldst, p.colsum = colsum_dev;
    const hipStream_t s = (hipStream_t)stream;
    const bool rows = !qt_dev && !tile && !colsum_dev;
    const long grid = rows ? (m * nb + 15) / 16 : mb * nb;
    if (!fits(grid, 256)) return ops_fail(ML_ERR_SHAPE, "ml_fp8_quantize: %lld x %lld is too large", (long long)m, (long long)n);
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (rows) quantize_rows_kernel<T><<<(unsigned)grid, 256, 0, s>>>(p);
        else quantize_tile_kernel<T><<<(unsigned)grid, 256, 0, s>>>(p);
    });
    return ops_launched("ml_fp8_quantize");
}

int64_t ml_fp8_matmul_work(int64_t m, int64_t n, int64_t k, int c_dtype) {
    return m <= 0 || n <= 0 || k <= 0 || !holds(m, n, k) ? 0 : gemm_work_bytes(m, n, k, c_dtype != ML_F32);
}

int ml_fp8_matmul(const uint8_t* a_dev, int64_t lda, const uint8_t* a_scale_dev, int64_t ldsa, int a_tile, const uint8_t* b_dev, int64_t ldb,
                  const uint8_t* b_scale_dev, int64_t ldsb, int b_tile, const void* bias_dev, int bias_dtype, void* c_dev, int c_dtype,
                  int64_t ldc, int64_t m, int64_t n, int64_t k, void* work_dev, int64_t work_bytes, void* stream) {
    const int es = elem_size(c_dtype);
    if (!es || (bias_dev && !elem_size(bias_dtype)) || m < 0 || n < 0 || k < 0) return ops_fail(ML_ERR_ARG, "ml_fp8_matmul: bad type %d, %d or size", c_dtype, bias_dtype);
    if (m == 0 || n == 0) return ML_OK;
    if (!c_dev || (k > 0 && (!a_dev || !b_dev || !a_scale_dev || !b_scale_dev))) return ops_fail(ML_ERR_ARG, "ml_fp8_matmul: null pointer");
    if (!holds(m, n, k)) return ops_fail(ML_ERR_SHAPE, "ml_fp8_matmul: %lld x %lld x %lld is too large", (long long)m, (long long)n, (long long)k);
    const long kb = (k + QB - 1) / QB;
    if (lda < k || ldb < k || ldc < n || ldsa < kb || ldsb < kb) return ops_fail(ML_ERR_ARG, "ml_fp8_matmul: a row stride is shorter than its row");
    const long grid = ((m + 63) / 64) * ((n + 63) / 64);
    if (!fits(grid, 256)) return ops_fail(ML_ERR_SHAPE, "ml_fp8_matmul: %lld x %lld is too large", (long long)m, (long long)n);
    const Area c{(int64_t)(uintptr_t)c_dev, ldc * es, n * es, m};
    auto area = [](const void* at, int64_t ld, int64_t width, int64_t rows) { return Area{(int64_t)(uintptr_t)at, ld, width, rows}; };
    const char* const shared = !apart(c, area(a_dev, lda, k, m)) ? "a" : !apart(c, area(b_dev, ldb, k, n)) ? "b"
                               : !apart(c, area(a_scale_dev, ldsa, kb, a_tile ? (m + QB - 1) / QB : m)) || !apart(c, area(b_scale_dev, ldsb, kb, b_tile ? (n + QB - 1) / QB : n)) ? "scales"
                               : bias_dev && !apart(c, area(bias_dev, 0, n * elem_size(bias_dtype), 1)) ? "bias" : nullptr;
    if (shared) return ops_fail(ML_ERR_ARG, "ml_fp8_matmul: the result shares memory with %s", shared);
    // (the stride of a single row is never taken: whatever it is, it must not decide which kernel runs)
    const long la = m > 1 ? lda : 0, lb = n > 1 ? ldb : 0;
    GemmParams p{a_dev, b_dev, a_scale_dev, b_scale_dev, la, lb, (long)ldsa, (long)ldsb, a_tile != 0, b_tile != 0, bias_dev, bias_dtype, c_dev,
                 (long)m, (long)n, (long)k, (long)ldc, 0, 0};
    p.fast_a = rows_aligned(a_dev, la, 1, 16), p.fast_b = rows_aligned(b_dev, lb, 1, 16);
    const hipStream_t s = (hipStream_t)stream;
    with_type(c_dtype, [&](auto t) { launch_gemm<decltype(t)>(p, (float*)work_dev, work_bytes, s); });
    return ops_launched("ml_fp8_matmul");
}

int ml_debug_areas_apart(int64_t at, int64_t pitch, int64_t width, int64_t rows, int64_t at2, int64_t pitch2, int64_t width2, int64_t rows2) {
    if ((rows > 1 && pitch < width) || (rows2 > 1 && pitch2 < width2)) return 0;
    return apart(Area{at, pitch, width, rows}, Area{at2, pitch2, width2, rows2});
}

// ---- a linear layer in one call: buffers at multiples of 256 bytes inside two workspaces
static int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

namespace {
struct LinearPlan {
    int64_t kb, nb, mb, ldk, ldn, ldm;                  // blocks; row strides of codes along k, n, m
    int64_t qx, sx, qw, sw, fsplit, forward;            // forward's workspace (fsplit, bsplit: parts of a product whose k is cut)
    int64_t qxt, sxt, qwt, swt, saved;                  // what the backward pass needs
    int64_t qd, sd, qdt, sdt, part, bsplit, backward;   // backward's workspace
    LinearPlan(int64_t m, int64_t n, int64_t k, bool need_dx, bool need_dw, bool need_db) {
        kb = (k + QB - 1) / QB, nb = (n + QB - 1) / QB, mb = (m + QB - 1) / QB;
        ldk = round_up(k, 16), ldn = round_up(n, 16), ldm = round_up(m, 16);
        auto most = [](int64_t a, int64_t b, int64_t c) { return std::max(ml_fp8_matmul_work(a, b, c, ML_BF16), ml_fp8_matmul_work(a, b, c, ML_F32)); };
        int64_t at = 0;
        auto take = [&](int64_t bytes) { const int64_t r = at; at += round_up(bytes, 256); return r; };
        qx = take(m * ldk), sx = take(m * kb), qw = take(n * ldk), sw = take(nb * kb);
        fsplit = take(most(m, n, k)), forward = at;
        at = 0;
        qxt = take(need_dw ? k * ldm : 0), sxt = take(need_dw ? k * mb : 0);
        qwt = take(need_dx ? k * ldn : 0), swt = take(need_dx ? kb * nb : 0), saved = at;
        at = 0;
        qd = take(need_dx ? m * ldn : 0), sd = take(need_dx ? m * nb : 0);
        qdt = take(need_dw ? n * ldm : 0), sdt = take(need_dw ? n * mb : 0);
        part = take(need_db ? mb * n * 4 : 0);
        const int64_t dx = need_dx ? most(m, k, n) : 0, dw = need_dw ? most(n, k, m) : 0;   // (one after the other)
        bsplit = take(dx > dw ? dx : dw), backward = at;
    }
};
}  // namespace

int ml_fp8_linear_sizes(int64_t m, int64_t n, int64_t k, int need_dx, int need_dw, int need_db, int64_t* bytes3) {
    if (m < 0 || n < 0 || k < 0 || !bytes3) return ops_fail(ML_ERR_ARG, "ml_fp8_linear_sizes: bad size or null pointer");
    if (!holds(m, n, k)) return ops_fail(ML_ERR_SHAPE, "ml_fp8_linear_sizes: %lld x %lld x %lld is too large", (long long)m, (long long)n, (long long)k);
    const LinearPlan l(m, n, k, need_dx, need_dw, need_db);
    bytes3[0] = l.forward, bytes3[1] = l.saved, bytes3[2] = l.backward;
    return ML_OK;
}

int ml_fp8_linear(const void* x_dev, int x_dtype, int64_t ldx, const void* w_dev, int w_dtype, int64_t ldw, const void* bias_dev, int bias_dtype, void* y_dev,
                  int64_t ldy, int64_t m, int64_t n, int64_t k, int need_dx, int need_dw, void* work_dev, void* saved_dev, void* stream) {
    if (m < 0 || n < 0 || k < 1) return ops_fail(ML_ERR_ARG, "ml_fp8_linear: bad size");
    if (!holds(m, n, k)) return ops_fail(ML_ERR_SHAPE, "ml_fp8_linear: %lld x %lld x %lld is too large", (long long)m, (long long)n, (long long)k);
    if ((m && n && !work_dev) || ((need_dx || need_dw) && n && !saved_dev)) return ops_fail(ML_ERR_ARG, "ml_fp8_linear: null workspace");
    const LinearPlan l(m, n, k, need_dx, need_dw, false);
    uint8_t *const wk = (uint8_t*)work_dev, *const sv = (uint8_t*)saved_dev;
    int rc = ml_fp8_quantize(x_dev, x_dtype, m, k, ldx, 0, wk + l.qx, l.ldk, wk + l.sx, l.kb, need_dw ? sv + l.qxt : nullptr, l.ldm, need_dw ? sv + l.sxt : nullptr,
                             l.mb, nullptr, stream);
    if (!rc)
        rc = ml_fp8_quantize(w_dev, w_dtype, n, k, ldw, 1, wk + l.qw, l.ldk, wk + l.sw, l.kb, need_dx ? sv + l.qwt : nullptr, l.ldn, need_dx ? sv + l.swt : nullptr,
                             l.nb, nullptr, stream);
    if (!rc) rc = ml_fp8_matmul(wk + l.qx, l.ldk, wk + l.sx, l.kb, 0, wk + l.qw, l.ldk, wk + l.sw, l.kb, 1, bias_dev, bias_dtype, y_dev, x_dtype, ldy, m, n, k, wk + l.fsplit,
                              l.forward - l.fsplit, stream);
    return rc;
}

int ml_fp8_linear_backward(const void* dy_dev, int dy_dtype, int64_t ldy, const void* saved_dev, void* dx_dev, int dx_dtype, void* dw_dev, int dw_dtype, void* db_dev,
                           int db_dtype, int64_t m, int64_t n, int64_t k, int need_dx, int need_dw, void* work_dev, void* stream) {
    if (m < 0 || n < 0 || k < 1) return ops_fail(ML_ERR_ARG, "ml_fp8_linear_backward: bad size");
    if (!holds(m, n, k)) return ops_fail(ML_ERR_SHAPE, "ml_fp8_linear_backward: %lld x %lld x %lld is too large", (long long)m, (long long)n, (long long)k);
    // (the layout of `saved` goes by what the forward pass was asked for, the work by what is asked for now)
    const LinearPlan l(m, n, k, need_dx, need_dw, db_dev != nullptr);
    const bool dx = dx_dev != nullptr, dw = dw_dev != nullptr;
    if ((dx && !need_dx) || (dw && !need_dw)) return ops_fail(ML_ERR_ARG, "ml_fp8_linear_backward: a gradient that the forward pass did not prepare");
    if (m && n && (!dy_dev || !work_dev || ((dx || dw) && !saved_dev))) return ops_fail(ML_ERR_ARG, "ml_fp8_linear_backward: null pointer");
    uint8_t *const wk = (uint8_t*)work_dev, *const sv = (uint8_t*)saved_dev;
    int rc = 0;
    if (dx || dw)
        rc = ml_fp8_quantize(dy_dev, dy_dtype, m, n, ldy, 0, dx ? wk + l.qd : nullptr, l.ldn, dx ? wk + l.sd : nullptr, l.nb, dw ? wk + l.qdt : nullptr, l.ldm,
                             dw ? wk + l.sdt : nullptr, l.mb, db_dev ? (float*)(wk + l.part) : nullptr, stream);
    else if (db_dev)
        rc = column_sums(dy_dev, dy_dtype, m, n, ldy, (float*)(wk + l.part), (hipStream_t)stream);
    if (!rc && dx) rc = ml_fp8_matmul(wk + l.qd, l.ldn, wk + l.sd, l.nb, 0, sv + l.qwt, l.ldn, sv + l.swt, l.nb, 1, nullptr, 0, dx_dev, dx_dtype, k, m, k, n, wk + l.bsplit, l.backward - l.bsplit,
                                     stream);
    if (!rc && dw) rc = ml_fp8_matmul(wk + l.qdt, l.ldm, wk + l.sdt, l.mb, 0, sv + l.qxt, l.ldm, sv + l.sxt, l.mb, 0, nullptr, 0, dw_dev, dw_dtype, k, n, k, m, wk + l.bsplit, l.backward - l.bsplit,
                                     stream);
    if (!rc && db_dev) rc = ml_sum_rows((const float*)(wk + l.part), m ? l.mb : 0, n, db_dev, db_dtype, stream);
    return rc;
}

int ml_rms_norm(const void* x_dev, int64_t ldx, const void* residual_dev, int64_t ldr, int dtype, const void* w_dev, int w_dtype, int64_t m,
                int64_t n, float eps, void* h_dev, int64_t ldh, void* y_dev, int64_t ldy, uint8_t* q_dev, int64_t ldq, uint8_t* scale_dev,
                int64_t lds, void* stream) {
    const int es = elem_size(dtype);
    if (!es || (w_dtype != dtype && w_dtype != ML_F32) || m < 0 || n < 0) return ops_fail(ML_ERR_ARG, "ml_rms_norm: bad types %d, %d or size", dtype, w_dtype);
    if (m == 0 || n == 0) return ML_OK;
    if (!x_dev || !w_dev || (!y_dev == !q_dev) || (q_dev && !scale_dev)) return ops_fail(ML_ERR_ARG, "ml_rms_norm: null pointer, or not one of y and q");
    const long nb = (n + QB - 1) / QB;
    if (ldx < n || (residual_dev && ldr < n) || (h_dev && ldh < n) || (y_dev && ldy < n) || (q_dev && (ldq < n || lds < nb)))
        return ops_fail(ML_ERR_ARG, "ml_rms_norm: a row stride is shorter than its row");
    if (!(n <= 2048 ? fits((m + 3) / 4, 256) : fits(m, n <= 8192 ? 256 : n <= 16384 ? 512 : 1024))) return ops_fail(ML_ERR_SHAPE, "ml_rms_norm: %lld rows of %lld are too many", (long long)m, (long long)n);
    NormParams p{};
    p.x = x_dev, p.residual = residual_dev, p.w = w_dev, p.w_f32 = w_dtype == ML_F32;
    p.m = m, p.n = n, p.ldx = ldx, p.ldr = ldr, p.ldy = q_dev ? ldq : ldy, p.ldh = ldh, p.eps = eps;
    p.y = y_dev, p.h = h_dev, p.q = q_dev, p.scale = scale_dev, p.lds = lds;
    const hipStream_t s = (hipStream_t)stream;
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (q_dev) launch_norm<T, true>(p, s);
        else launch_norm<T, false>(p, s);
    });
    return ops_launched("ml_rms_norm");
}

int64_t ml_rms_norm_backward_groups(int64_t m, int64_t n) { return m <= 0 || n <= 0 ? 0 : norm_groups(m, n); }

int ml_rms_norm_backward(const void* dy_dev, int64_t ldy, const void* h_dev, int64_t ldh, const void* dh_dev, int64_t ldd, int dtype,
                         const void* w_dev, int w_dtype, int64_t m, int64_t n, float eps, void* dx_dev, int64_t ldx, void* dw_dev,
                         float* work_dev, void* stream) {
    const int es = elem_size(dtype);
    if (!es || (w_dtype != dtype && w_dtype != ML_F32) || m < 0 || n < 0) return ops_fail(ML_ERR_ARG, "ml_rms_norm_backward: bad types %d, %d or size", dtype, w_dtype);
    if (n == 0) return ML_OK;
    if (!dw_dev || (m > 0 && (!dy_dev || !h_dev || !w_dev || !dx_dev || !work_dev))) return ops_fail(ML_ERR_ARG, "ml_rms_norm_backward: null pointer");
    if (m > 0 && (ldy < n || ldh < n || (dh_dev && ldd < n) || ldx < n)) return ops_fail(ML_ERR_ARG, "ml_rms_norm_backward: a row stride is shorter than its row");
    if (!fits((n + 31) / 32, 1024)) return ops_fail(ML_ERR_SHAPE, "ml_rms_norm_backward: %lld columns are too many", (long long)n);
    const hipStream_t s = (hipStream_t)stream;
    const long groups = m ? norm_groups(m, n) : 0;
    if (m > 0) {
        NormBackParams p{};
        p.dy = dy_dev, p.h = h_dev, p.w = w_dev, p.dh = dh_dev, p.w_f32 = w_dtype == ML_F32;
        p.m = m, p.n = n, p.ldy = ldy, p.ldh = ldh, p.ldd = ldd, p.ldx = ldx, p.eps = eps, p.dx = dx_dev, p.part = work_dev;
        with_type(dtype, [&](auto t) { launch_norm_back<decltype(t)>(p, (unsigned)groups, s); });
        const int rc = ops_launched("ml_rms_norm_backward");
        if (rc) return rc;
    }
    with_type(w_dtype, [&](auto t) { launch_reduce(work_dev, groups, n, (decltype(t)*)dw_dev, s); });
    return ops_launched("ml_rms_norm_backward");
}

int ml_sum_rows(const float* part_dev, int64_t rows, int64_t n, void* out_dev, int dtype, void* stream) {
    if (!elem_size(dtype) || rows < 0 || n < 0) return ops_fail(ML_ERR_ARG, "ml_sum_rows: bad type %d or size", dtype);
    if (n == 0) return ML_OK;
    if (!out_dev || (rows > 0 && !part_dev)) return ops_fail(ML_ERR_ARG, "ml_sum_rows: null pointer");
    if (!fits((n + 31) / 32, 1024)) return ops_fail(ML_ERR_SHAPE, "ml_sum_rows: %lld columns are too many", (long long)n);
    with_type(dtype, [&](auto t) { launch_reduce(part_dev, rows, n, (decltype(t)*)out_dev, (hipStream_t)stream); });
    return ops_launched("ml_sum_rows");
}

}  // extern "C"
