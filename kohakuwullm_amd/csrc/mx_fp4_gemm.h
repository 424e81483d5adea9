// Products with a B operand of e2m1 codes: the arguments that every kernel of the family takes, and the tiled kernels' problem policy.
#pragma once

#include "mx_fp4.h"
#include "mx_gemm_core.h"

namespace mx {

struct Fp4GemmArgs {
    const uint8_t *aq, *as, *bq, *bs;
    const int32_t *index, *offsets;  // offsets NULL: one group of M rows
    void *c;
    int64_t lda, ldas, stride_be, ldb, stride_bse, ldbs, ldc;
    int M, N, K, E;
    int x_rows;  // of A, where it is gathered
    // the tiled kernels
    int tiles_m, tiles_n;  // row tiles: of the one group, or at most
    int c_vec;             // whether a lane's run of columns can be stored as one
    int dp_tiles;          // tiles that are computed whole; the others in split_k slices of K, whose fp32 tiles go to slice_ws
    int split_k;
    float *slice_ws;
};

// The longest M, N and K: the kernels add a stage, a tile or a loop's stride (1024 at most) to a row, column or place in K in 32 bits.
constexpr int64_t FP4_EXTENT = ((int64_t)1 << 31) - 1024;

// Where expert e's rows begin (e = E: end): inside the matrix whatever the table says.
__device__ __forceinline__ int group_bound(const Fp4GemmArgs &a, int e) {
    const int at = a.offsets[e];
    return at < 0 ? 0 : at < a.M ? at : a.M;
}

// The row of A that sorted position m takes.
__device__ __forceinline__ int source_row(const Fp4GemmArgs &a, int m) {
    if (!a.index) return m;
    const int at = a.index[m];
    return at < 0 ? 0 : at < a.x_rows ? at : a.x_rows - 1;
}

template <int CDT>
__device__ __forceinline__ void store_value(void *c, int64_t at, float v) {
    if (CDT == MX_FP32) ((float *)c)[at] = v;
    else if (CDT == MX_BF16) ((uint16_t *)c)[at] = (uint16_t)pack2_bf16(v, 0.f);
    else ((_Float16 *)c)[at] = (_Float16)v;
}

// Stages of a slice of K where KT of them are cut into `slices`: whole groups of scale bytes, four stages at most.
__host__ __device__ __forceinline__ int fp4_slice_stages(int KT, int slices) { return ((KT + slices - 1) / slices + 3) & ~3; }

// Row tiles of the experts before e, for e in [0, E]: a workgroup's first wave builds them once, so that the expert of a row tile is a
// search in LDS instead of a walk over the offsets in memory.  Offsets that never decrease make tiles_m of them at most, and what numbers
// tiles counts on that (plan_fp4_tiles, stream_takes): the table ends there whatever the offsets say.
constexpr int FP4_EXPERTS = 1024;  // more go to the kernel without tables
__device__ __forceinline__ void build_tile_table(int *table, const Fp4GemmArgs &a, int rows) {
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        int before = 0;
        for (int e0 = 0; e0 < a.E; e0 += 64) {
            const int e = e0 + lane;
            const int n = e < a.E ? group_bound(a, e + 1) - group_bound(a, e) : 0;
            const int tiles = n > 0 ? (n + rows - 1) / rows : 0;
            const int upto = wave_incl_scan(tiles, lane);
            if (e < a.E) table[e] = min(before + upto - tiles, a.tiles_m);
            before = min(before + __shfl(upto, 63, 64), a.tiles_m);
        }
        if (lane == 0) table[a.E] = before;
    }
    __syncthreads();
}
// The last expert that begins at or before row tile rt: the one that owns it.
typedef __attribute__((address_space(3))) const int lds_int;
__device__ __forceinline__ int expert_of_tile(lds_int *table, int E, int rt) {
    int lo = 0, hi = E;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (table[mid] <= rt) lo = mid;
        else hi = mid;
    }
    return lo;
}

// What persistent_gemm asks of a problem (mx_gemm_core.h), for both forms: one group of rows, whose last, partial round of tiles may be
// cut along K, or the rows of experts.
template <typename S, int CDT>
struct Fp4Problem {
    struct Tile {
        int row0, n0, end, expert, kt0, kt1;
        int slot;  // of slice_ws, or -1
    };
    static constexpr int NST = S::MT * 4 * (CDT == MX_FP32 && S::NT == 8 ? 2 : 1);
    static constexpr bool EARLY_WAIT = false;
    static constexpr bool REUSE_CONTEXT = true;  // context() may read row indices

    const Fp4GemmArgs p;
    int next_id;
    const int kb_end;
    lds_int *const table;  // with offsets

    __device__ Fp4Problem(const Fp4GemmArgs &a, lds_int *t) : p(a), next_id(blockIdx.x), kb_end(a.K >> 5), table(t) {}

    __device__ __forceinline__ int row_bytes() const { return S::CODES == CODES_44 ? p.K >> 1 : p.K; }  // of A

    __device__ __forceinline__ bool next(Tile &t) {
        const int KT = (row_bytes() + 127) >> 7;
        if (p.offsets) {
            // each XCD takes a contiguous range of the tiles there are: those of one row tile share its rows and their expert's weights
            const int total = p.tiles_n * table[p.E], per_xcd = total >> 3;
            if (next_id >= total) return false;
            int id = next_id;
            next_id += gridDim.x;
            if (id < (per_xcd << 3)) id = (id & 7) * per_xcd + (id >> 3);
            const int rt = id / p.tiles_n;
            t.expert = expert_of_tile(table, p.E, rt);
            t.row0 = group_bound(p, t.expert) + (rt - table[t.expert]) * S::BM;
            t.end = group_bound(p, t.expert + 1);
            t.n0 = (id - rt * p.tiles_n) * S::BN;
            t.kt0 = 0, t.kt1 = KT, t.slot = -1;
            return true;
        }
        const int tiles = p.tiles_m * p.tiles_n, cut = tiles - p.dp_tiles;
        const int per = fp4_slice_stages(KT, p.split_k);
        while (next_id < p.dp_tiles + cut * p.split_k) {
            const bool whole = next_id < p.dp_tiles;
            const int slice = whole ? 0 : (next_id - p.dp_tiles) / cut, index = next_id - slice * cut;
            next_id += gridDim.x;
            t.kt0 = whole ? 0 : slice * per;
            t.kt1 = whole || t.kt0 + per > KT ? KT : t.kt0 + per;
            if (t.kt0 >= t.kt1) continue;  // an empty last slice: the sum leaves it out
            int tm, tn;
            tile_of(index, p.tiles_m, p.tiles_n, tm, tn, KT <= 64, 8);
            t.row0 = tm * S::BM, t.n0 = tn * S::BN, t.end = p.M, t.expert = 0;
            t.slot = whole ? -1 : (index - p.dp_tiles) * p.split_k + slice;
            return true;
        }
        return false;
    }

    __device__ __forceinline__ int a_row(const Tile &t, int r) const {
        const int m = t.row0 + r;
        return source_row(p, m < t.end ? m : t.end - 1);  // rows past the group's end repeat its last one; never stored
    }
    __device__ __forceinline__ int b_row(const Tile &t, int r) const {  // kept in LDS row r of the B tile
        const int n = t.n0 + b_row_of_lds<S>(r);
        return n < p.N ? n : p.N - 1;
    }

    __device__ __forceinline__ void context(const Tile &t, const Lane &L0, IssueCtx<S> &c) const {
        const Lane L = opaque(L0);
        const int first = p.index ? 0 : t.row0;  // gathered rows are offset from the matrix, others from the tile
        c.a_base = p.aq + (int64_t)first * p.lda;
        c.b_base = p.bq + (int64_t)t.expert * p.stride_be + (int64_t)t.n0 * p.ldb;
        c.a_ks = 128, c.b_ks = S::BKB;
        c.kt0 = t.kt0, c.kt1 = t.kt1;
        c.tail_bytes = row_bytes() & 127;
        c.tail_kt = c.tail_bytes ? row_bytes() >> 7 : -1;
#pragma unroll
        for (int q = 0; q < S::QA; q++) {
            const int row = dma_row<S>(L, q);
            c.a_voff[q] = (uint32_t)((a_row(t, row) - first) * p.lda) + (((L.lane & 7) ^ swz_a(row)) << 4) + copy_bias(q);
        }
#pragma unroll
        for (int q = 0; q < S::QB; q++) {
            const int row = dma_row_b<S>(L, q);
            c.b_voff[q] = (uint32_t)((b_row(t, row) - t.n0) * p.ldb) + (dma_chunk_b<S>(L, row) << 4) + copy_bias(q);
        }
        auto scales = [&](int r) -> const uint8_t * {
            if (r < S::BM) return p.as + (int64_t)a_row(t, r) * p.ldas;
            return p.bs + (int64_t)t.expert * p.stride_bse + (int64_t)b_row(t, r - S::BM) * p.ldbs;
        };
        static_assert(!S::TWO_ROWS && S::NTHR == S::BM + S::BN, "one row of scales per thread");
        c.srow0 = scales(L.tid);
        c.srow1 = nullptr;
        c.sa_base = p.as, c.sb_base = p.bs;
        c.s_voff = (uint32_t)(c.srow0 - (L.tid < S::BM ? p.as : p.bs));
    }

    __device__ __forceinline__ int epilogue(const Tile &t, const Lane &L, v4f (&acc)[S::MT][S::NT], const LdsScratch &) const {
        if (t.slot >= 0) {
            v4f *const dst = (v4f *)p.slice_ws + (int64_t)t.slot * (S::BM * S::BN / 4);
#pragma unroll
            for (int i = 0; i < S::MT; i++)
#pragma unroll
                for (int j = 0; j < S::NT; j++) dst[(i * S::NT + j) * S::NTHR + L.tid] = acc[i][j];
            return -1;
        }
        const bool interior = t.row0 + S::BM <= t.end && t.n0 + S::BN <= p.N && p.c_vec;
        const int n = t.n0 + L.wn * S::WTN + S::NT * L.r16;
#pragma unroll
        for (int i = 0; i < S::MT; i++) {
#pragma unroll
            for (int v = 0; v < 4; v++) {
                const int m = t.row0 + L.wm * S::WTM + 16 * i + 4 * L.g + v;
                const int64_t off = (int64_t)m * p.ldc + n;
                float run[S::NT];
#pragma unroll
                for (int j = 0; j < S::NT; j++) run[j] = acc[i][j][v];
                if (interior) store_run<CDT, S::NT>(p.c, off, run, S::NT, true);
                else if (m < t.end && n < p.N) store_run<CDT, S::NT>(p.c, off, run, p.N - n < S::NT ? p.N - n : S::NT, p.c_vec != 0);
            }
        }
        return interior ? NST : -1;
    }
};

// 256 x 256 tiles on eight waves, a workgroup per CU: the most products for a byte from L2, 1.5 us a stage of 128 with e4m3 A rows, 1.75 of
// 256 with e2m1 ones, and 6 us of stores between tiles, since a wave's next copies retire behind its stores.  8192 x 8192 x 8192 410 us
// (2.7 PFLOP/s) and 255 (4.3); 16384 x 8192 x 1536 184 and 119 to 138; the matrix pipe is busy for 0.44 of that.
// 128 x 128 on four waves, two workgroups per CU: what the stream of stages does not take.
template <int CODES>
using Fp4Big = GemmShape<256, 256, 4, 2, CODES>;
template <int CODES>
using Fp4Slim = GemmShape<128, 128, 2, 2, CODES>;

// LDS of a workgroup in front of the experts' table, which is as long as there are experts: 64 leave room for two slim ones on a CU.
template <typename S>
__host__ __device__ constexpr int fp4_lds_bytes(int mode) {
    return mode == SCALES_COPY ? S::LDS_BYTES_AHEAD : S::LDS_BYTES;
}

template <typename S, int CDT, int MODE>
__device__ __forceinline__ void fp4_tiles(const Fp4GemmArgs &a) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    int *const table = (int *)(smem + fp4_lds_bytes<S>(MODE));
    if (a.offsets) build_tile_table(table, a, S::BM);
    Fp4Problem<S, CDT> prob(a, (lds_int *)table);
    persistent_gemm<S, MODE, Fp4Problem<S, CDT>, MODE == SCALES_COPY>(prob, smem);
}
template <typename S, int CDT, int MODE>
__global__ __launch_bounds__(S::NTHR) void fp4_big_kernel(Fp4GemmArgs a) {
    fp4_tiles<S, CDT, MODE>(a);
}
template <typename S, int CDT, int MODE>
__global__ __launch_bounds__(S::NTHR) __attribute__((amdgpu_waves_per_eu(2, 2))) void fp4_slim_kernel(Fp4GemmArgs a) {
    fp4_tiles<S, CDT, MODE>(a);
}

// Adds the slices of the tiles that were cut along K, in slice order.  A block per tile and row of sub-tiles.
template <typename S, int CDT>
__global__ __launch_bounds__(S::NTHR) void fp4_slices_kernel(Fp4GemmArgs p) {
    const int local = blockIdx.x / S::MT, i = blockIdx.x % S::MT, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int KT = ((S::CODES == CODES_44 ? p.K >> 1 : p.K) + 127) >> 7;
    const int per = fp4_slice_stages(KT, p.split_k), slices = (KT + per - 1) / per;
    v4f sum[S::NT];
#pragma unroll
    for (int j = 0; j < S::NT; j++) sum[j] = v4f{0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < slices; s++) {
        const v4f *const src = (const v4f *)p.slice_ws + (int64_t)(local * p.split_k + s) * (S::BM * S::BN / 4);
#pragma unroll
        for (int j = 0; j < S::NT; j++) sum[j] += src[(i * S::NT + j) * S::NTHR + tid];
    }
    int tm, tn;
    tile_of(p.dp_tiles + local, p.tiles_m, p.tiles_n, tm, tn, KT <= 64, 8);
    const int n = tn * S::BN + (wave % S::WGN) * S::WTN + S::NT * (lane & 15);
#pragma unroll
    for (int v = 0; v < 4; v++) {
        const int m = tm * S::BM + (wave / S::WGN) * S::WTM + 16 * i + 4 * (lane >> 4) + v;
        if (m >= p.M || n >= p.N) continue;
        float run[S::NT];
#pragma unroll
        for (int j = 0; j < S::NT; j++) run[j] = sum[j][v];
        store_run<CDT, S::NT>(p.c, (int64_t)m * p.ldc + n, run, p.N - n < S::NT ? p.N - n : S::NT, p.c_vec != 0);
    }
}

// mx_fp4_few.hip, the product for a few rows of A: whether it takes the operands and is the quicker way, and its launch.  bits: of A's codes.
bool fp4_few_pays(const Fp4GemmArgs &a);
int launch_fp4_few(Fp4GemmArgs a, int bits, int c_dtype, hipStream_t st);

// mx_fp4_tiles_*.hip, a file per output type and A format: the product on 256 x 256 tiles, on 128 x 128 ones, two workgroups per CU, or on
// 128 x 128 ones as a stream of K stages.
struct Fp4Workspace {
    float *at;
    int64_t bytes;
};
constexpr int FP4_STREAM_TILES = 1 << 19;  // the stream divides numbers of tiles, and eight times them, in 22 bits
enum Fp4Way { FP4_BIG, FP4_SLIM, FP4_STREAM };
template <int CODES, int CDT>
int launch_fp4_tiles(Fp4GemmArgs a, Fp4Way way, const Fp4Workspace &ws, hipStream_t st);

}  // namespace mx
