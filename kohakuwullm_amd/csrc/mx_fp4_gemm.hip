// Products with a B operand of e2m1 codes, for gfx950: C (M,N) = deq(A) deq(B)^T, A (M,K) in e4m3 or e2m1, B (N,K) in e2m1, a UE8M0 byte per
// 32 of K on both sides, fp32 sums, 16- or 32-bit results; and the same per expert, for rows sorted by expert (offsets), optionally
// gathered (index).  The instruction takes e4m3 on one side and e2m1 on the other, so codes go into it as they lie in memory.
//
// Operand layout of v_mfma_scale_f32_16x16x128_f8f6f4 for lane (r = l % 16, g = l / 16) and row r: e2m1, the 32 codes of block g, 16 bytes;
// e4m3, codes 16 g .. 16 g + 15 and 64 + 16 g .. 64 + 16 g + 15; the scale of (row r, block b) comes from lane r + 16 b.
#include <cmath>

#include "mx_fp4_gemm.h"

namespace mx {

// Whatever the tiled kernels do not take.  A wave takes 16 rows of one group and 64 columns.
template <int CDT, int ABITS>
__global__ __launch_bounds__(64) void fp4_gemm_simple_kernel(Fp4GemmArgs a) {
    const int lane = threadIdx.x, r = lane & 15, g = lane >> 4;
    int row0 = 0, end = a.M, expert = 0;
    int tile = blockIdx.x;
    if (a.offsets) {
        for (; expert < a.E; expert++) {
            row0 = group_bound(a, expert), end = group_bound(a, expert + 1);
            const int tiles = end > row0 ? (end - row0 + 15) >> 4 : 0;
            if (tile < tiles) break;
            tile -= tiles;
        }
        if (expert == a.E) return;
    }
    row0 += 16 * tile;
    const int n0 = blockIdx.y * 64;
    const int m = row0 + r < end ? row0 + r : end - 1;
    const int64_t src = source_row(a, m);
    const uint8_t *const pa = a.aq + src * a.lda, *const sa = a.as + src * a.ldas;
    const uint8_t *pb[4], *sb[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int64_t n = n0 + 16 * j + r < a.N ? n0 + 16 * j + r : a.N - 1;
        pb[j] = a.bq + expert * a.stride_be + n * a.ldb;
        sb[j] = a.bs + expert * a.stride_bse + n * a.ldbs;
    }
    v4f acc[4];
#pragma unroll
    for (int j = 0; j < 4; j++) acc[j] = v4f{0.f, 0.f, 0.f, 0.f};
    const v4i none = {0, 0, 0, 0};
    for (int k = 0; k < a.K; k += 128) {
        const int blocks = (a.K - k) >> 5;  // left; codes of blocks past the end are zero
        v4i lo = none, hi = none;
        if (ABITS == 8) {
            if ((g >> 1) < blocks) lo = *(const v4i *)(pa + k + 16 * g);
            if (2 + (g >> 1) < blocks) hi = *(const v4i *)(pa + k + 64 + 16 * g);
        } else if (g < blocks) {
            lo = *(const v4i *)(pa + k / 2 + 16 * g);
        }
        const int as = g < blocks ? sa[(k >> 5) + g] : 0;
        const v8i fa = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const v4i b = g < blocks ? *(const v4i *)(pb[j] + k / 2 + 16 * g) : none;
            const int bs = g < blocks ? sb[j][(k >> 5) + g] : 0;
            const v8i fb = __builtin_shufflevector(b, none, 0, 1, 2, 3, 4, 5, 6, 7);
            acc[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fa, fb, acc[j], ABITS == 8 ? 0 : 4, 4, 0, as, 0, bs);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const int row = row0 + 4 * g + v, n = n0 + 16 * j + r;
            if (row < end && n < a.N) store_value<CDT>(a.c, (int64_t)row * a.ldc + n, acc[j][v]);
        }
}

}  // namespace mx

using namespace mx;

static inline bool aligned(const void *p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// What the tiled kernels take: tables of experts that fit, and byte offsets from a tile's rows (gathered rows: from the matrix) of 32 bits.
static bool tiles_take(const Fp4GemmArgs &a) {
    const int64_t limit = (int64_t)1 << 31;
    return (!a.offsets || a.E <= FP4_EXPERTS) && 256 * a.ldb < limit && (a.index ? (int64_t)a.x_rows * a.lda < 2 * limit - 4096 : 256 * a.lda < limit);
}

// What the stream of stages takes besides: few enough tiles, whole groups of scale bytes, 16-byte runs of results, 32-bit offsets of scale rows.
static bool stream_takes(const Fp4GemmArgs &a, int c_dtype) {
    const int64_t limit = (int64_t)1 << 31, row_tiles = ((int64_t)a.M + 127) / 128 + (a.offsets ? a.E : 0);
    if (row_tiles * (((int64_t)a.N + 127) / 128) > FP4_STREAM_TILES) return false;
    return a.K % 512 == 0 && a.N % 8 == 0 && aligned(a.c, 16) && a.ldc * (c_dtype == MX_FP32 ? 4 : 2) % 16 == 0 && aligned(a.as, 16) && aligned(a.bs, 16) &&
           a.ldas % 16 == 0 && a.ldbs % 16 == 0 && a.stride_bse % 16 == 0 && (a.index ? a.x_rows : 128) * a.ldas < limit && 128 * a.ldbs < limit;
}

// Large tiles or small ones, by what rounds of them take: us per stage (128 of K, 256 with e2m1 on both sides) and per tile, its stores
// mostly, 1.5 (1.75) and 6 for 256 x 256 on every CU, 0.5 (0.65) and 1.4 for the stream of 128 x 128.  An expert with rows has half a row
// tile more than its rows fill.  us large / stream / 128 x 128 two per CU, A in 8 bits and in 4:
//   16384 x 8192 x 1536   184 / 270 / 269   119 / 163 / 178      2048 x 2048 x 2048   25.9 / 12.7 / 15.7   17.7 / 11.5 / 12.5
//   16384 x 4096 x 4096   229 / 267 / 279   141 / 172 / 189      1000 x 2048 x 2048   26.2 / 12.5 / 14.8   17.6 / 9.8 / 12.0
//   8192 x 8192 x 8192    410 / 496 / 510   255 / 321 / 337      301 x 8192 x 1536    20.8 / 10.1 / 12.7   14.6 / 9.2 / 11.2
//   5003 x 1536 x 4096   49.7 / 33.8 / 36  32.8 / 24.8 / 26.4    301 x 1536 x 4096    26.7 / 16.8 / 18.4   26.9 / 12.4 / 16.0
//   5003 x 4096 x 1536   42.5 / 35.3 / 37  30.2 / 27.0 / 28.6    16384 x 1536 x 512   21.8 / 22.0 / 22.1   17.8 / 17.7 / 19.4
//   in 64 experts of 1024 columns: 98304 rows, K = 1024  109 / 123 / 147   79 / 87 / 117;  K = 512  79 / 91 / 91   60 / 56 / 72
//   16384 rows, K = 1024  35.3 / 32.9 / 35.4   27.6 / 25.4 / 28.7;  4662 rows, K = 512  13.8 / 13.2 / 15.4   12.0 / 12.4 / 13.8
//
// Where the stream does not take the operands, K % 512 mostly, scales come by the dword or the byte: large tiles take 2 us (2.75) a stage then,
// 128 x 128 two per CU 0.75 (1.2) and 1.8 (1.3) a tile, in pairs as soon as there are more tiles than CUs.  us large / small, A in 8 bits and in 4:
//   124 x 1936 x 2784   24.9 / 16.4   29.9 / 19.2     1557 x 7424 x 3488  76.3 / 92.8   61.8 / 75.2
//   2000 x 2000 x 2016  33.9 / 23.3   25.0 / 17.8     4096 x 4096 x 1056  26.3 / 35.1   23.0 / 29.7
//   1186 x 3064 x 3840  45.5 / 31.0   31.3 / 21.5     8000 x 4096 x 1952  74.5 / 111    57.2 / 83.2
//   597 x 6936 x 2528   40.2 / 37.3   32.9 / 28.6     13012 x 656 x 1856  34.0 / 45.7   27.2 / 35.2
//   64 experts of 1024 x 736: 4662 rows 19.9 / 27.5, 16.7 / 22.1; 49152 rows 68.2 / 90.4, 55.6 / 74.9
static double tiles_us(const Fp4GemmArgs &a, int bits, int edge, bool stream) {
    const double live = a.offsets ? (a.E < a.M ? a.E : a.M) : 0;
    const double rows = a.offsets ? (double)a.M / edge + live / 2 : ceil((double)a.M / edge), cols = ceil((double)a.N / edge);
    const double stages = ceil(a.K / (bits == 8 ? 128.0 : 256.0)), rounds = ceil(rows * cols / num_cus());
    if (!stream) {
        if (edge == 256) return rounds * (stages * (bits == 8 ? 2 : 2.75) + 6);
        return (rounds > 1 ? 2 * ceil(rounds / 2) : 1) * (bits == 8 ? stages * 0.75 + 1.8 : stages * 1.2 + 1.3) + 4;
    }
    return edge == 256 ? rounds * (stages * (bits == 8 ? 1.5 : 1.75) + 6) : rounds * (stages * (bits == 8 ? 0.5 : 0.65) + 1.4);
}

template <int CDT, int ABITS>
static int launch_product(const Fp4GemmArgs &a, const Fp4Workspace &ws, hipStream_t st) {
    if (fp4_few_pays(a)) return launch_fp4_few(a, ABITS, CDT, st);
    if (tiles_take(a)) {
        const bool stream = stream_takes(a, CDT), big = tiles_us(a, ABITS, 256, stream) < tiles_us(a, ABITS, 128, stream);
        const Fp4Way way = big ? FP4_BIG : stream ? FP4_STREAM : FP4_SLIM;
        return launch_fp4_tiles<ABITS == 8 ? CODES_84 : CODES_44, CDT>(a, way, ws, st);
    }
    const int64_t rows = a.offsets ? (int64_t)(a.M + 15) / 16 + a.E : (a.M + 15) / 16, cols = (a.N + 63) / 64;
    if (cols > 65535 || rows >= 1 << 26) return MX_EUNSUPPORTED;  // 2^32 threads
    fp4_gemm_simple_kernel<CDT, ABITS><<<dim3((unsigned)rows, (unsigned)cols), dim3(64), 0, st>>>(a);
    return hipGetLastError() == hipSuccess ? MX_OK : MX_ELAUNCH;
}

static int product(const Fp4GemmArgs &a, int a_format, int c_dtype, const Fp4Workspace &ws, hipStream_t st) {
    auto typed = [&](auto cdt) { return a_format == MX_E4M3 ? launch_product<cdt.value, 8>(a, ws, st) : launch_product<cdt.value, 4>(a, ws, st); };
    switch (c_dtype) {
    case MX_BF16: return typed(std::integral_constant<int, MX_BF16>{});
    case MX_FP16: return typed(std::integral_constant<int, MX_FP16>{});
    default: return typed(std::integral_constant<int, MX_FP32>{});
    }
}

static bool formats_ok(int a_format, int c_dtype) {
    return (a_format == MX_E4M3 || a_format == MX_E2M1) && (c_dtype == MX_BF16 || c_dtype == MX_FP16 || c_dtype == MX_FP32);
}

// Rows of codes that can be fetched 16 bytes at a time.
static bool codes_ok(const uint8_t *q, int64_t ld) { return aligned(q, 16) && ld % 16 == 0; }

// Zeros in the rows of C inside every group (an empty contraction) or outside (rows that belong to no expert).  A workgroup takes
// every gridDim.x-th row.
template <int CDT>
__global__ __launch_bounds__(256) static void fp4_zero_kernel(Fp4GemmArgs a, int inside) {
    const int first = a.offsets ? group_bound(a, 0) : 0, last = a.offsets ? group_bound(a, a.E) : a.M;
    const int before = inside ? 0 : first, count = inside ? last - first : before + a.M - last;
    for (int i = blockIdx.x; i < count; i += gridDim.x) {
        const int64_t m = inside ? first + i : i < before ? i : last + (i - before);
        for (int n = threadIdx.x; n < a.N; n += 256) store_value<CDT>(a.c, m * a.ldc + n, 0.0f);
    }
}

static int zeros(const Fp4GemmArgs &a, int c_dtype, bool inside, hipStream_t st) {
    const dim3 grid((unsigned)(a.M < 1024 ? a.M : 1024)), block(256);
    if (c_dtype == MX_BF16) fp4_zero_kernel<MX_BF16><<<grid, block, 0, st>>>(a, inside);
    else if (c_dtype == MX_FP16) fp4_zero_kernel<MX_FP16><<<grid, block, 0, st>>>(a, inside);
    else fp4_zero_kernel<MX_FP32><<<grid, block, 0, st>>>(a, inside);
    return hipGetLastError() == hipSuccess ? MX_OK : MX_ELAUNCH;
}

extern "C" int mx_fp4_gemm_nt(const uint8_t *aq, const uint8_t *a_scale, int a_format, const uint8_t *bq, const uint8_t *b_scale, void *c,
                              int c_dtype, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldas, int64_t ldb, int64_t ldbs,
                              int64_t ldc, void *workspace, int64_t workspace_bytes, void *stream) {
    if (!formats_ok(a_format, c_dtype) || M < 0 || N < 0 || K < 0 || K % MX_BLOCK || M > 0x7FFFFFFF || N > 0x7FFFFFFF || K > 0x7FFFFFFF ||
        lda < (a_format == MX_E4M3 ? K : K / 2) || ldb < K / 2 || ldas < K / MX_BLOCK || ldbs < K / MX_BLOCK || ldc < N || workspace_bytes < 0)
        return MX_EINVAL;
    if (M == 0 || N == 0) return MX_OK;
    if (!c || (K && (!aq || !a_scale || !bq || !b_scale))) return MX_EINVAL;
    if (M > FP4_EXTENT || N > FP4_EXTENT || K > FP4_EXTENT || (K && (!codes_ok(aq, lda) || !codes_ok(bq, ldb)))) return MX_EUNSUPPORTED;
    hipStream_t st = (hipStream_t)stream;
    if (mx::stream_is_capturing(st)) return MX_ECAPTURE;
    const Fp4GemmArgs a = {aq, a_scale, bq, b_scale, nullptr, nullptr, c, lda, ldas, 0, ldb, 0, ldbs, ldc, (int)M, (int)N, (int)K, 1, (int)M};
    return K ? product(a, a_format, c_dtype, {(float *)workspace, workspace_bytes}, st) : zeros(a, c_dtype, true, st);
}

extern "C" int mx_fp4_grouped_gemm_nt(const uint8_t *xq, const uint8_t *x_scale, int x_format, int64_t x_rows, int64_t ldx, int64_t ldxs,
                                      const int32_t *index, const uint8_t *wq, const uint8_t *w_scale, int64_t stride_we, int64_t ldw,
                                      int64_t stride_wse, int64_t ldws, const int32_t *offsets, int64_t E, void *out, int out_dtype,
                                      int64_t ldo, int64_t M, int64_t N, int64_t K, int zero_rest, void *stream) {
    if (!formats_ok(x_format, out_dtype) || E <= 0 || E >= (1 << 20) || M < 0 || N < 0 || K < 0 || K % MX_BLOCK || M >= 0x7FFFFFFF ||
        N > 0x7FFFFFFF || K > 0x7FFFFFFF || x_rows < 0 || x_rows > 0x7FFFFFFF || ldx < (x_format == MX_E4M3 ? K : K / 2) || ldxs < K / MX_BLOCK || ldw < K / 2 ||
        ldws < K / MX_BLOCK || stride_we < 0 || stride_wse < 0 || ldo < N)
        return MX_EINVAL;
    if (M == 0 || N == 0) return MX_OK;
    if (!offsets || !out || (K && (!xq || !x_scale || !wq || !w_scale))) return MX_EINVAL;
    if ((!index && x_rows < M) || x_rows == 0) return MX_EINVAL;
    if (M > FP4_EXTENT || N > FP4_EXTENT || K > FP4_EXTENT || (K && (!codes_ok(xq, ldx) || !codes_ok(wq, ldw) || stride_we % 16)))
        return MX_EUNSUPPORTED;
    hipStream_t st = (hipStream_t)stream;
    if (mx::stream_is_capturing(st)) return MX_ECAPTURE;
    const Fp4GemmArgs a = {xq, x_scale, wq, w_scale, index, offsets, out, ldx, ldxs, stride_we, ldw, stride_wse, ldws, ldo, (int)M, (int)N, (int)K, (int)E, (int)x_rows};
    const int rc = zero_rest ? zeros(a, out_dtype, false, st) : MX_OK;
    if (rc != MX_OK) return rc;
    return K ? product(a, x_format, out_dtype, {nullptr, 0}, st) : zeros(a, out_dtype, true, st);
}
