// Block-scaled 8-bit products grouped by expert (fp8_gemm.hip has the dense one), gfx950.
//
//   rows form   D[rows of e] = A[rows of e] B[e]^T           rows of e: COUNTS[e] consecutive expert-sorted rows
//   wgrad form  D[e] = A_e B_e^T + C[e]                      A_e, B_e: the columns of expert e of transposed operands,
//                                                            every expert starting at a multiple of 128
// One launch each; the counts stay on the device.  A workgroup finds its tiles from the counts themselves (a scan
// over 64 experts per wave step), so there is no plan to make, keep or share.
#include "fp8_core.h"
#include "flexhip.h"

namespace fx {

template <typename TD, int SHIFT, int BN>
struct Fp8GroupedRows {
    Fp8View A, B;
    int64_t b_expert, sb_expert;
    const int32_t* COUNTS;
    const int32_t* MAP;
    TD* D;
    int64_t ldc, ldd, total_rows;
    int E, src_rows, K, tiles_n;
    struct Where { int row0, e, rows, m0, n0; };
    FX_DEV int total(int lane) const { return count_group_tiles<SHIFT>(COUNTS, E, total_rows, lane) * tiles_n; }
    FX_DEV Where locate(int id, int total, int lane) const {
        // expert-major, column tile fastest; each XCD (own L2) takes a contiguous band of that order
        const int p = xcd_band(id, total);
        const GroupTile t = find_group_tile<SHIFT>(COUNTS, E, p / tiles_n, total_rows, lane);
        return Where{t.row0, t.e, t.rows, t.m0, (p % tiles_n) * BN};
    }
    FX_DEV bool locate_one(int id, int lane, Where& w) const {
        const GroupTile t = find_group_tile<SHIFT>(COUNTS, E, id / tiles_n, total_rows, lane);
        w = Where{t.row0, t.e, t.rows, t.m0, (id % tiles_n) * BN};
        return t.e >= 0;
    }
    FX_DEV Fp8Job<TD> job(const Where& w) const {
        Fp8Job<TD> j{A, B, w.m0, w.n0, K, nullptr, src_rows, nullptr, D + (int64_t)w.row0 * ldd};
        j.A.ext = w.rows;
        if (MAP != nullptr) {
            j.row_map = MAP + w.row0;
        } else {
            j.A.p += (int64_t)w.row0 * A.ld;
            j.A.s += (int64_t)w.row0 * A.s_row;
        }
        j.B.p += w.e * b_expert;
        j.B.s += w.e * sb_expert;
        return j;
    }
};

template <typename TD, int BM, int BN>
struct Fp8GroupedWgrad {
    Fp8View A, B;
    const int32_t* COUNTS;
    const TD* C;
    TD* D;
    int64_t ldc, ldd, c_expert, d_expert, capacity;
    int E, tiles_m, tiles_n;
    struct Where { int padded0, e, rows, m0, n0; };
    FX_DEV int total(int) const { return E * tiles_m * tiles_n; }
    FX_DEV Where locate(int id, int total, int lane) const {
        const int p = xcd_band(id, total), per = tiles_m * tiles_n;
        const int e = p / per, q = p % per;
        const GroupSpan s = find_group_span(COUNTS, E, e, capacity, lane);
        return Where{s.padded0, e, s.rows, (q / tiles_n) * BM, (q % tiles_n) * BN};
    }
    FX_DEV Fp8Job<TD> job(const Where& w) const {
        // the places behind an expert's rows hold zeros: whole K-steps
        Fp8Job<TD> j{A, B, w.m0, w.n0, (w.rows + 127) & ~127, nullptr, 0, C ? C + (int64_t)w.e * c_expert : nullptr, D + (int64_t)w.e * d_expert};
        j.A.p += w.padded0;
        j.B.p += w.padded0;
        j.A.s += (int64_t)(w.padded0 >> 7) * A.s_k;
        j.B.s += (int64_t)(w.padded0 >> 7) * B.s_k;
        return j;
    }
};

struct Fp8RowsPlan { int shift, small; };      // tile rows (their logarithm): 8, 7, or 4 .. 6 with the small kernel's form `small`

// The fastest form by the times of fp8_core.h for rows split evenly over the experts that have any, half a tile of padding
// each (the split itself is on the device; what that costs stands there).  Measured on 128 experts, N 1536, K 2048,
// routed counts: 8 rows an expert small 1 x 4 73 us, 128 81; 16 rows 94, 82; 64 rows 128 92, 256 100; 128 rows 125, 116;
// 512 rows 310, 269.
static Fp8RowsPlan fp8_rows_plan(int64_t rows, int E, int N, int K) {
    const double live = (double)(E < rows ? E : rows), avg = (double)rows / live;
    const int steps = fp8_cdiv(K, FP8_BK);
    auto tiles = [&](int bm) { const double t = avg / bm + 0.5; return live * (avg <= 1.0 || t < 1.0 ? 1.0 : t); };
    Fp8RowsPlan best{4, 0};
    double t_best = 1e30;
    for (int i = 0; i < kFp8Smalls; ++i) {
        const Fp8Small& c = kFp8Small[i];
        if (c.mt > 1 && 16 * c.mt >= 2 * avg) continue;
        const double t = fp8_time_small(c, tiles(16 * c.mt), (double)rows, N, steps);
        if (t < t_best) { t_best = t; best = Fp8RowsPlan{c.mt == 1 ? 4 : c.mt == 2 ? 5 : 6, i}; }
    }
    const double t128 = fp8_time_128(tiles(128) * fp8_cdiv(N, 128), steps > 1 ? steps : 2);
    if (t128 < t_best) { t_best = t128; best = Fp8RowsPlan{7, 0}; }
    if (K >= FP8_BK && fp8_time_256(tiles(256) * fp8_cdiv(N, 256), steps > 1 ? steps : 2) < t_best) best = Fp8RowsPlan{8, 0};
    return best;
}

template <typename TD>
struct Fp8RowsArgs {
    Fp8View a, b;
    int64_t b_expert, sb_expert;
    const int32_t *counts, *map;
    int a_rows;
    TD* D;
    int64_t ldd, rows;
    int E, K;
    template <typename Source> Source source(int tiles_n) const {
        return Source{a, b, b_expert, sb_expert, counts, map, D, 0, ldd, rows, E, a_rows, K, tiles_n};
    }
    // at most this many row tiles, whatever the split over the experts
    int64_t most(int shift) const { return (rows >> shift) + (E < rows ? E : rows); }
};

template <int AF, typename TD, int MT, int NT>
static int launch_rows_small(const Fp8RowsArgs<TD>& g, hipStream_t stream) {
    constexpr int SHIFT = MT == 1 ? 4 : MT == 2 ? 5 : 6;
    typedef Fp8GroupedRows<TD, SHIFT, 16 * NT> Source;
    typedef Fp8SmallShape<MT, NT> Shape;
    const int tiles_n = fp8_cdiv(g.b.ext, 16 * NT);
    if (!grid_fits(g.most(SHIFT) * tiles_n, Shape::NW * 64)) FX_FAIL("fx_fp8_grouped_gemm: too many tiles");
    fp8_small_kernel<AF, TD, MT, NT, Shape::NW, Shape::U, Source><<<dim3((unsigned)(g.most(SHIFT) * tiles_n)), Shape::NW * 64, 0, stream>>>(g.template source<Source>(tiles_n));
    return 0;
}

template <int AF, typename TD>
static int launch_rows_walk(const Fp8RowsArgs<TD>& g, hipStream_t stream) {
    typedef Fp8GroupedRows<TD, 8, 256> Source;
    const int tiles_n = fp8_cdiv(g.b.ext, 256);
    const int64_t total = g.most(8) * tiles_n;
    if (total > 0x7fffffff) FX_FAIL("fx_fp8_grouped_gemm: too many tiles");
    const unsigned grid = (unsigned)(total < fp8_walk_grid() ? total : fp8_walk_grid());
    if ((size_t)g.rows * (size_t)g.b.ext * sizeof(TD) >= kFp8OnceBytes) {
        auto kern = fp8_walk_kernel<AF, TD, true, Source>;
        FX_ENSURE_DYNAMIC_LDS(kern, kFp8WalkLds);
        kern<<<dim3(grid), 512, kFp8WalkLds, stream>>>(g.template source<Source>(tiles_n));
    } else {
        auto kern = fp8_walk_kernel<AF, TD, false, Source>;
        FX_ENSURE_DYNAMIC_LDS(kern, kFp8WalkLds);
        kern<<<dim3(grid), 512, kFp8WalkLds, stream>>>(g.template source<Source>(tiles_n));
    }
    return 0;
}

template <int AF, typename TD>
static int launch_rows(const Fp8RowsArgs<TD>& g, hipStream_t stream) {
    const Fp8RowsPlan p = fp8_rows_plan(g.rows, g.E, g.b.ext, g.K);
    int rc = 0;
    if (p.shift == 8) {
        rc = launch_rows_walk<AF, TD>(g, stream);
    } else if (p.shift == 7) {
        typedef Fp8GroupedRows<TD, 7, 128> Source;
        const int tiles_n = fp8_cdiv(g.b.ext, 128);
        if (!grid_fits(g.most(7) * tiles_n, 256)) FX_FAIL("fx_fp8_grouped_gemm: too many tiles");
        auto kern = fp8_tile_kernel128<AF, TD, Source>;
        FX_ENSURE_DYNAMIC_LDS(kern, kFp8Tile128Lds);
        kern<<<dim3((unsigned)(g.most(7) * tiles_n)), 256, kFp8Tile128Lds, stream>>>(g.template source<Source>(tiles_n));
    } else {
        switch (p.small) {
            case 0: rc = launch_rows_small<AF, TD, 1, 1>(g, stream); break;
            case 1: rc = launch_rows_small<AF, TD, 1, 2>(g, stream); break;
            case 2: rc = launch_rows_small<AF, TD, 1, 4>(g, stream); break;
            case 3: rc = launch_rows_small<AF, TD, 2, 2>(g, stream); break;
            case 4: rc = launch_rows_small<AF, TD, 2, 4>(g, stream); break;
            case 5: rc = launch_rows_small<AF, TD, 4, 2>(g, stream); break;
            default: rc = launch_rows_small<AF, TD, 4, 4>(g, stream); break;
        }
    }
    if (rc != 0) return rc;
    FX_CHECK_LAUNCH("fx_fp8_grouped_gemm");
    return 0;
}

template <int AF, typename TD>
static int launch_wgrad(const Fp8View& a, const Fp8View& b, const int32_t* counts, int E, int64_t capacity, const TD* C, int64_t ldc,
                        int64_t c_expert, TD* D, int64_t ldd, int64_t d_expert, hipStream_t stream) {
    const int M = a.ext, N = b.ext;
    // 256 x 256 tiles from three quarters of a round of the 256 CUs on.  Their time against 128 x 128 ones (5 shapes of 256 x 256 to
    // 1536 x 2048, 1 .. 128 experts of 32 .. 8192 rows on average): up to 64 tiles 1.5 .. 2.3, 96 and 128 tiles 1.4 .. 1.7, 192 tiles
    // 0.76 .. 1.18 (long contractions gain), whole rounds (256, 512, 768 tiles) 0.82 .. 1.03, a last round that is half full or
    // less (384, 576) 1.00 .. 1.18.
    const int64_t big = (int64_t)E * fp8_cdiv(M, 256) * fp8_cdiv(N, 256);
    if (big >= 192) {
        typedef Fp8GroupedWgrad<TD, 256, 256> Source;
        const Source src{a, b, counts, C, D, ldc, ldd, c_expert, d_expert, capacity, E, fp8_cdiv(M, 256), fp8_cdiv(N, 256)};
        const unsigned grid = (unsigned)(big < fp8_walk_grid() ? big : fp8_walk_grid());
        if ((size_t)E * (size_t)M * (size_t)N * sizeof(TD) >= kFp8OnceBytes) {
            auto kern = fp8_walk_kernel<AF, TD, true, Source>;
            FX_ENSURE_DYNAMIC_LDS(kern, kFp8WalkLds);
            kern<<<dim3(grid), 512, kFp8WalkLds, stream>>>(src);
        } else {
            auto kern = fp8_walk_kernel<AF, TD, false, Source>;
            FX_ENSURE_DYNAMIC_LDS(kern, kFp8WalkLds);
            kern<<<dim3(grid), 512, kFp8WalkLds, stream>>>(src);
        }
    } else {
        const int64_t tiles = (int64_t)E * fp8_cdiv(M, 128) * fp8_cdiv(N, 128);
        typedef Fp8GroupedWgrad<TD, 128, 128> Source;
        const Source src{a, b, counts, C, D, ldc, ldd, c_expert, d_expert, capacity, E, fp8_cdiv(M, 128), fp8_cdiv(N, 128)};
        auto kern = fp8_tile_kernel128<AF, TD, Source>;
        FX_ENSURE_DYNAMIC_LDS(kern, kFp8Tile128Lds);
        kern<<<dim3((unsigned)tiles), 256, kFp8Tile128Lds, stream>>>(src);
    }
    FX_CHECK_LAUNCH("fx_fp8_grouped_wgrad");
    return 0;
}

}  // namespace fx

using namespace fx;

extern "C" int fx_fp8_grouped_gemm(const void* A, int64_t lda, int a_dt, const void* SA, int64_t sa_row, int64_t sa_k,
                                   const int32_t* row_map, int64_t a_rows, const void* B, int64_t ldb, int64_t b_expert,
                                   const void* SB, int64_t sb_row, int64_t sb_k, int64_t sb_expert, int b_tiles,
                                   const int32_t* counts, int E, int64_t total_rows, void* D, int64_t ldd, int N, int K, int d_dt,
                                   hipStream_t stream) {
    if (E <= 0 || total_rows < 0 || N < 0 || K < 0) FX_FAIL("fx_fp8_grouped_gemm: bad shape");
    if (!is_fp8_dt(a_dt)) FX_FAIL("fx_fp8_grouped_gemm: unsupported 8-bit dtype enum %d", a_dt);
    if (d_dt != DT_F32 && d_dt != DT_F16 && d_dt != DT_BF16) FX_FAIL("fx_fp8_grouped_gemm: unsupported output dtype enum %d", d_dt);
    if (total_rows > (1 << 24)) FX_FAIL("fx_fp8_grouped_gemm: at most 2^24 expert rows");
    if (N > kFp8MaxExtent) FX_FAIL("fx_fp8_grouped_gemm: too many rows of B");
    if (total_rows == 0 || N == 0) return 0;
    if (!counts || !D || (K > 0 && (!A || !B || !SA || !SB))) FX_FAIL("fx_fp8_grouped_gemm: null pointer");
    if (K > 0 && (fp8_bad_rows(A, lda) || fp8_bad_rows(B, ldb) || (b_expert & 15))) FX_FAIL("fx_fp8_grouped_gemm: rows of A and B must start at 16-byte addresses");
    if ((K > 0 && (lda < K || ldb < K)) || ldd < N) FX_FAIL("fx_fp8_grouped_gemm: a row stride is shorter than the row");
    if (lda >= kFp8MaxLd || ldb >= kFp8MaxLd) FX_FAIL("fx_fp8_grouped_gemm: row strides must be below 2^23 bytes");
    if (row_map ? (a_rows <= 0 || a_rows > 0x7fffffff) : a_rows < total_rows) FX_FAIL("fx_fp8_grouped_gemm: A has %lld rows", (long long)a_rows);
    if (row_map && (uint64_t)a_rows * (uint64_t)lda >= (1ull << 32)) FX_FAIL("fx_fp8_grouped_gemm: a gathered A must stay below 4 GB");
    const int kb = fp8_cdiv(K, FP8_BK);
    if (!fp8_scales_fit(a_rows, sa_row, kb, sa_k) || !fp8_scales_fit(b_tiles ? fp8_cdiv(N, 128) : N, sb_row, kb, sb_k) || sb_expert < 0 || b_expert < 0)
        FX_FAIL("fx_fp8_grouped_gemm: the scales of A, and those of an expert's B, must span less than 2 GB, with no negative stride");
    const Fp8View a{(const uint8_t*)A, (const uint8_t*)SA, (int)lda, (int)sa_row, (int)sa_k, 0, 0};
    const Fp8View b{(const uint8_t*)B, (const uint8_t*)SB, (int)ldb, (int)sb_row, (int)sb_k, b_tiles ? 7 : 0, N};
    int rc = -1;
    FX_DISPATCH_FP8(a_dt, AF, FX_DISPATCH_DTYPE(d_dt, TD, rc = launch_rows<AF, TD>(Fp8RowsArgs<TD>{a, b, b_expert, sb_expert, counts, row_map, (int)a_rows, (TD*)D, ldd, total_rows, E, K}, stream)));
    return rc;
}

extern "C" int fx_fp8_grouped_wgrad(const void* A, int64_t lda, int a_dt, const void* SA, int64_t sa_row, int64_t sa_k, const void* B,
                                    int64_t ldb, const void* SB, int64_t sb_row, int64_t sb_k, const int32_t* counts, int E,
                                    int64_t capacity, const void* C, int64_t ldc, int64_t c_expert, void* D, int64_t ldd,
                                    int64_t d_expert, int M, int N, int d_dt, hipStream_t stream) {
    if (E <= 0 || capacity < 0 || (capacity & 127) || M < 0 || N < 0) FX_FAIL("fx_fp8_grouped_wgrad: bad shape");
    if (!is_fp8_dt(a_dt)) FX_FAIL("fx_fp8_grouped_wgrad: unsupported 8-bit dtype enum %d", a_dt);
    if (d_dt != DT_F32 && d_dt != DT_F16 && d_dt != DT_BF16) FX_FAIL("fx_fp8_grouped_wgrad: unsupported output dtype enum %d", d_dt);
    if (capacity >= kFp8MaxLd) FX_FAIL("fx_fp8_grouped_wgrad: at most 2^23 expert rows");
    if (M > kFp8MaxExtent || N > kFp8MaxExtent) FX_FAIL("fx_fp8_grouped_wgrad: too many rows");
    if (M == 0 || N == 0) return 0;
    if (!counts || !D || (capacity > 0 && (!A || !B || !SA || !SB))) FX_FAIL("fx_fp8_grouped_wgrad: null pointer");
    if (capacity > 0 && (fp8_bad_rows(A, lda) || fp8_bad_rows(B, ldb))) FX_FAIL("fx_fp8_grouped_wgrad: rows of A and B must start at 16-byte addresses");
    if (lda < capacity || ldb < capacity || ldd < N || (C && ldc < N)) FX_FAIL("fx_fp8_grouped_wgrad: a row stride is shorter than the row");
    if (lda >= kFp8MaxLd || ldb >= kFp8MaxLd) FX_FAIL("fx_fp8_grouped_wgrad: row strides must be below 2^23 bytes");
    if (!fp8_scales_fit(M, sa_row, capacity / 128, sa_k) || !fp8_scales_fit(N, sb_row, capacity / 128, sb_k))
        FX_FAIL("fx_fp8_grouped_wgrad: a scale tensor must span less than 2 GB, with no negative stride");
    if ((double)E * fp8_cdiv(M, 128) * fp8_cdiv(N, 128) > 2147483647.0) FX_FAIL("fx_fp8_grouped_wgrad: too many tiles");
    const Fp8View a{(const uint8_t*)A, (const uint8_t*)SA, (int)lda, (int)sa_row, (int)sa_k, 0, M};
    const Fp8View b{(const uint8_t*)B, (const uint8_t*)SB, (int)ldb, (int)sb_row, (int)sb_k, 0, N};
    int rc = -1;
    FX_DISPATCH_FP8(a_dt, AF, FX_DISPATCH_DTYPE(d_dt, TD, rc = launch_wgrad<AF, TD>(a, b, counts, E, capacity, (const TD*)C, ldc, c_expert, (TD*)D, ldd, d_expert, stream)));
    return rc;
}
