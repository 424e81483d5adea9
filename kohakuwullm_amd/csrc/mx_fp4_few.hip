// Launching the product with 4-bit weights for a few rows (mx_fp4_few.h): quantized rows, experts' rows, and activations.
#include "mx_fp4_few.h"

namespace mx {

static inline bool few_aligned(const void *p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

template <int CDT, int MT, int WK, int SRC>
static int launch_few(Fp4GemmArgs a, hipStream_t st) {
    constexpr int WN = FEW_WAVES / WK;
    a.tiles_n = (a.N + 16 * WN - 1) / (16 * WN);
    const int64_t blocks = (int64_t)a.tiles_n * (a.offsets ? a.E : 1);
    if (blocks >= 1 << 23) return MX_EUNSUPPORTED;  // 2^32 threads
    const bool dwords = few_aligned(a.as, 4) && few_aligned(a.bs, 4) && a.ldas % 4 == 0 && a.ldbs % 4 == 0 && a.stride_bse % 4 == 0;
    const dim3 grid((unsigned)blocks), block(FEW_WAVES * 64);
    const int rc = a.K % 128 == 0 && dwords ? launch_with_lds<&fp4_few_kernel<CDT, MT, WK, SRC, CDT, false>>(grid, block, few_lds_bytes(SRC, MT), st, a)
                                            : launch_with_lds<&fp4_few_kernel<CDT, MT, WK, SRC, CDT, true>>(grid, block, few_lds_bytes(SRC, MT), st, a);
    if (rc != MX_OK) return rc;
    return hipGetLastError() == hipSuccess ? MX_OK : MX_ELAUNCH;
}

// Parts of K by the workgroups of 16 columns there would be: see mx_fp4_few.h.  Rows of experts: two for short contractions, else four.
// Activations are the same product with the same parts, of fewer columns (activations_pay).
template <int CDT, int MT, int SRC>
static int launch_few_parts(const Fp4GemmArgs &a, hipStream_t st) {
    const int64_t blocks = (a.N + 15) / 16, cus = num_cus();
    if (blocks <= 2 * cus) return launch_few<CDT, MT, 8, SRC>(a, st);
    if constexpr (MT <= (few_codes(SRC) ? 2 : 1)) {  // a wave stores one sub-tile
        if constexpr (few_codes(SRC))
            if (blocks > 8 * cus) return launch_few<CDT, MT, 2, SRC>(a, st);
        return launch_few<CDT, MT, 4, SRC>(a, st);
    } else {
        return launch_few<CDT, MT, 8, SRC>(a, st);
    }
}

template <int CDT, int SRC>
static int launch_few_rows(const Fp4GemmArgs &a, hipStream_t st) {
    if constexpr (few_codes(SRC))
        if (a.offsets) return a.K <= 2048 ? launch_few<CDT, 1, 2, SRC>(a, st) : launch_few<CDT, 1, 4, SRC>(a, st);
    if (a.M <= 16) return launch_few_parts<CDT, 1, SRC>(a, st);
    if (a.M <= 32) return launch_few_parts<CDT, 2, SRC>(a, st);
    if constexpr (few_codes(SRC)) return launch_few_parts<CDT, 4, SRC>(a, st);
    return MX_EUNSUPPORTED;
}

// Whether a few rows go here and not to 128 x 128 tiles, by the stages of 256 of K that a CU's workgroups of 16 columns walk together.
// us on tiles / here, weights from HBM, with those stages:
//            4096 -> 1536 (6)  1536 -> 8192 (12)  8192 -> 8192 (64)  1536 -> 65536 (96)  16384 -> 16384 (256)  4096 -> 131072 (512)
//   M = 1      14.8 / 4.6        13.1 / 4.4          25.0 / 10.7         18.6 / 12.7         56.0 / 34.1            77.2 / 58.7
//   16         14.4 / 5.7        12.8 / 4.9          25.3 / 16.0         19.1 / 16.4         59.2 / 51.2            77.4 / 94.2
//   32         14.2 / 7.4        12.6 / 5.8          25.1 / 20.9         19.5 / 24.0         57.1 / 77.1            78.7 / 145
//   64         14.4 / 10.3       13.1 / 9.7          25.1 / 34.8         20.6 / 71.6         58.2 / 125             81.6 / 291
// 64 rows besides: 8192 -> 4096 22.8 / 18.1, 16384 -> 1536 21.4 / 31.0, 2048 -> 16384 17.0 / 23.4; one workgroup fits a CU then.
// Experts' rows, by rows per expert: 64 of 1024 x 1024, 3 13.3 / 9.8, 4 14.0 / 11.1, 6 14.3 / 14.9, 12 15.1 / 22.7; of 1024 x 512, 6 10.1 /
// 9.4, 12 11.3 / 12.8; 16 of 4096 x 4096, 3 39.2 / 32.0, 6 42.0 / 40.4, 12 42.7 / 51.8; of 256 x 256, 12 7.5 / 5.0.
bool fp4_few_pays(const Fp4GemmArgs &a) {
    if (((int64_t)a.N + 15) / 16 * (a.offsets ? a.E : 1) >= 1 << 23) return false;  // 2^32 threads
    if (a.offsets) return a.M <= 6 * (int64_t)a.E;
    const int64_t cus = num_cus(), blocks = (a.N + 15) / 16, stages = blocks * ((a.K + 255) / 256);
    if (a.M <= 16) return a.M <= 4 || stages <= 256 * cus;
    if (a.M <= 32) return stages <= 64 * cus;
    return a.M <= 64 && stages <= 32 * cus && blocks <= 2 * cus && a.K <= 8192;
}

int launch_fp4_few(Fp4GemmArgs a, int bits, int c_dtype, hipStream_t st) {
    auto typed = [&](auto cdt) { return bits == 8 ? launch_few_rows<cdt.value, SRC_E4M3>(a, st) : launch_few_rows<cdt.value, SRC_E2M1>(a, st); };
    switch (c_dtype) {
    case MX_BF16: return typed(std::integral_constant<int, MX_BF16>{});
    case MX_FP16: return typed(std::integral_constant<int, MX_FP16>{});
    default: return typed(std::integral_constant<int, MX_FP32>{});
    }
}

}  // namespace mx

using namespace mx;

// Which activations are quantized inside the product: every workgroup does it again, which with more rows or more workgroups costs more than
// the launch it saves; and only those whose codes would come here too, so that the sums over K are the same ones.  Kernels' us in two
// launches / in one, weights from HBM, without the 1 to 10 us that lie between two launches:
//             512 -> 4096   1536 -> 4096   1536 -> 8192   2048 -> 16384   8192 -> 8192   1536 -> 65536   4096 -> 131072
//   M = 1       4.9 / 3.2      5.6 / 3.8      6.3 / 4.7      8.8 / 7.6     13.0 / 13.6     15.2 / 18.5     63.3 / 80.5
//   8           5.3 / 3.6      5.8 / 4.3      6.6 / 5.2      9.7 / 8.6     16.2 / 15.4     19.0 / 19.0     67.0 / 84.9
//   16          5.6 / 4.1      6.6 / 5.0      7.3 / 6.2     11.0 / 9.8     19.5 / 17.6     21.8 / 22.7     68.2 / 103
//   32          6.1 / 5.4      7.3 / 6.9      8.4 / 11.8    14.0 / 18.0                    21.9 / 47.1
static bool activations_pay(const Fp4GemmArgs &a) {
    const int64_t cus = num_cus(), blocks = ((int64_t)a.N + 15) / 16;
    return fp4_few_pays(a) && (a.M <= 16 ? a.K <= 8192 && blocks <= 4 * cus : a.M <= 32 && a.K <= 2048 && blocks <= cus);
}

extern "C" int mx_fp4_activation_gemm_nt(const void *x, int x_dtype, int64_t ldx, const uint8_t *bq, const uint8_t *b_scale, void *c, int c_dtype,
                                         int64_t M, int64_t N, int64_t K, int64_t ldb, int64_t ldbs, int64_t ldc, void *stream) {
    if (M < 0 || N < 0 || K < 0 || K % MX_BLOCK || M > 0x7FFFFFFF || N > 0x7FFFFFFF || K > 0x7FFFFFFF || ldx < K || ldb < K / 2 || ldbs < K / MX_BLOCK ||
        ldc < N)
        return MX_EINVAL;
    if ((c_dtype != MX_BF16 && c_dtype != MX_FP16) || (x_dtype != c_dtype && x_dtype != MX_FP32)) return MX_EUNSUPPORTED;
    if (M == 0 || N == 0) return MX_OK;
    if (!c || (K && (!x || !bq || !b_scale))) return MX_EINVAL;
    if (K == 0 || M > 32 || N > FP4_EXTENT || K > FP4_EXTENT || !few_aligned(x, 16) || ldx * (x_dtype == MX_FP32 ? 4 : 2) % 16 || !few_aligned(bq, 16) || ldb % 16)
        return MX_EUNSUPPORTED;
    hipStream_t st = (hipStream_t)stream;
    if (stream_is_capturing(st)) return MX_ECAPTURE;
    const Fp4GemmArgs a = {(const uint8_t *)x, nullptr, bq, b_scale, nullptr, nullptr, c, ldx, 0, 0, ldb, 0, ldbs, ldc, (int)M, (int)N, (int)K, 1, (int)M};
    if (!activations_pay(a)) return MX_EUNSUPPORTED;
    if (x_dtype == MX_FP32) return c_dtype == MX_BF16 ? launch_few_rows<MX_BF16, MX_FP32>(a, st) : launch_few_rows<MX_FP16, MX_FP32>(a, st);
    return c_dtype == MX_BF16 ? launch_few_rows<MX_BF16, MX_BF16>(a, st) : launch_few_rows<MX_FP16, MX_FP16>(a, st);
}
