// Matrix products of 8-bit operands with a power-of-two scale per block of 128 (fp8.h), gfx950.
//
//   D[M,N] = sum over k blocks of 2^(ea[m,kb] + eb[n,kb]) * (A[M,kb] B[N,kb]^T)  + C          fp32 accumulate
//
// Both operands have the contraction contiguous (A (M,K), B (N,K)), which the quantiser's row and transposed
// outputs provide for the forward product, the input gradient and the weight gradient alike.
// v_mfma_scale_f32_32x32x64_f8f6f4 takes one e8m0 byte per operand row and 32 k, so the scales cost no vector
// instructions.  A may be e4m3 or e5m2 (gradients), B is e4m3.
#include "fp8.h"
#include "gemm_core.h"
#include "flexhip.h"

namespace fx {

typedef int i32x8_t __attribute__((ext_vector_type(8)));

// One operand: rows of 8-bit values, and the scale of (row, k block) at s[(row >> s_shift) * s_row + kb * s_k].
struct Fp8View {
    const uint8_t* p;
    int64_t ld;
    const uint8_t* s;
    int64_t s_row, s_k;
    int s_shift;      // 0: a scale per row, 7: per 128 rows
    int ext;          // rows
};

template <int AF>
FX_DEV f32x16_t mfma_fp8(i32x8_t b, i32x8_t a, f32x16_t c, int sb, int sa) {
    // the B fragment first: the accumulator then holds the transposed tile, a lane four consecutive columns of D
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b, a, c, 0, AF == DT_E4M3 ? 0 : 1, 0, sb, 0, sa);
}

// 32 consecutive k values of a row; 0 behind K.  Rows start at 16-byte addresses; a 16-byte chunk that K ends
// inside is read byte by byte (what lies behind K in memory is not the operand's).
FX_DEV i32x8_t load_frag(const uint8_t* row, int k, int K) {
    union { i32x8_t f; u32x4_t q[2]; uint8_t b[32]; } u;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int kc = k + 16 * c;
        if (kc + 16 <= K) {
            u.q[c] = ldg16(row + kc);
        } else {
            const u32x4_t zero = {0u, 0u, 0u, 0u};
            u.q[c] = zero;
            for (int j = 0; j < 16; ++j)
                if (kc + j < K) u.b[16 * c + j] = row[kc + j];
        }
    }
    return u.f;
}

// 64 x 64 tile, four waves of 32 x 32, operands straight from memory into registers.
template <int AF, typename TD>
FX_DEV void simple_tile(const Fp8View& A, const Fp8View& B, int m0, int n0, int K, const int32_t* row_map, int src_rows,
                        const TD* C, int64_t ldc, TD* D, int64_t ldd) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int half = lane >> 5;
    const int m = m0 + (wave >> 1) * 32 + (lane & 31), n = n0 + (wave & 1) * 32 + (lane & 31);
    int64_t am = min(m, A.ext - 1);
    if (row_map != nullptr) am = min(max(row_map[am], 0), src_rows - 1);
    const int64_t bn = min(n, B.ext - 1);
    const uint8_t *pa = A.p + am * A.ld, *pb = B.p + bn * B.ld;
    const uint8_t *sa = A.s + (am >> A.s_shift) * A.s_row, *sb = B.s + (bn >> B.s_shift) * B.s_row;
    f32x16_t acc;
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[v] = 0.f;
    for (int k = 0; k < K; k += 64) {
        const i32x8_t fa = load_frag(pa, k + 32 * half, K), fb = load_frag(pb, k + 32 * half, K);
        acc = mfma_fp8<AF>(fb, fa, acc, sb[(k >> 7) * B.s_k], sa[(k >> 7) * A.s_k]);
    }
    if (m >= A.ext) return;
    const int col0 = n0 + (wave & 1) * 32 + 4 * half;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
        const int col = col0 + 8 * (v >> 2) + (v & 3);
        if (col < B.ext) {
            float o = acc[v];
            if (C != nullptr) o += (float)C[(int64_t)m * ldc + col];
            D[(int64_t)m * ldd + col] = (TD)o;
        }
    }
}

template <int AF, typename TD>
__global__ __launch_bounds__(256) void fp8_gemm_simple_kernel(Fp8View A, Fp8View B, int K, const TD* C, int64_t ldc, TD* D,
                                                              int64_t ldd, int tiles_n) {
    simple_tile<AF, TD>(A, B, (blockIdx.x / tiles_n) * 64, (blockIdx.x % tiles_n) * 64, K, nullptr, 0, C, ldc, D, ldd);
}

template <int AF, typename TD>
__global__ __launch_bounds__(256) void fp8_grouped_simple_kernel(Fp8View A, Fp8View B, int64_t b_expert, int64_t sb_expert,
                                                                 const int32_t* __restrict__ COUNTS, int E, int64_t total_rows,
                                                                 const int32_t* __restrict__ MAP, int src_rows, int K, TD* D,
                                                                 int64_t ldd, int tiles_n) {
    const GroupTile t = find_group_tile<6>(COUNTS, E, blockIdx.x / tiles_n, total_rows, threadIdx.x & 63);
    if (t.e < 0 || t.rows <= t.m0) return;
    if (MAP == nullptr) { A.p += t.row0 * A.ld; A.s += t.row0 * A.s_row; }
    A.ext = t.rows;
    B.p += t.e * b_expert;
    B.s += t.e * sb_expert;
    simple_tile<AF, TD>(A, B, t.m0, (blockIdx.x % tiles_n) * 64, K, MAP ? MAP + t.row0 : nullptr, src_rows, (const TD*)nullptr,
                        0, D + t.row0 * ldd, ldd);
}

template <int AF, typename TD>
__global__ __launch_bounds__(256) void fp8_wgrad_simple_kernel(Fp8View A, Fp8View B, const int32_t* __restrict__ COUNTS, int E,
                                                               int64_t capacity, const TD* C, int64_t ldc, int64_t c_expert,
                                                               TD* D, int64_t ldd, int64_t d_expert, int tiles_m, int tiles_n) {
    const int e = blockIdx.x / (tiles_m * tiles_n), q = blockIdx.x % (tiles_m * tiles_n);
    const GroupSpan s = find_group_span(COUNTS, E, e, capacity, threadIdx.x & 63);
    A.p += s.padded0; A.s += (s.padded0 >> 7) * A.s_k;
    B.p += s.padded0; B.s += (s.padded0 >> 7) * B.s_k;
    simple_tile<AF, TD>(A, B, (q / tiles_n) * 64, (q % tiles_n) * 64, (s.rows + 127) & ~127, nullptr, 0, C ? C + e * c_expert : nullptr, ldc,
                        D + e * d_expert, ldd);
}

static int cdiv_i(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

}  // namespace fx

using namespace fx;

// Rows of an operand start at 16-byte addresses.
static bool bad_rows(const void* p, int64_t ld) { return !aligned16(p) || (ld & 15) != 0; }

#define FX_FP8_OUT(a_dt, d_dt, ...)                                                                     \
    FX_DISPATCH_FP8(a_dt, AF, FX_DISPATCH_DTYPE(d_dt, TD, __VA_ARGS__))

extern "C" size_t fx_fp8_gemm_ws_bytes(int M, int N, int K) {
    (void)M; (void)N; (void)K;
    return 0;
}

extern "C" int fx_fp8_gemm(const void* A, int64_t lda, int a_dt, const void* SA, int64_t sa_row, int64_t sa_k, int a_tiles,
                           const void* B, int64_t ldb, const void* SB, int64_t sb_row, int64_t sb_k, int b_tiles, const void* C,
                           int64_t ldc, void* D, int64_t ldd, int M, int N, int K, int d_dt, void* ws, size_t ws_bytes,
                           hipStream_t stream) {
    if (M < 0 || N < 0 || K < 0) FX_FAIL("fx_fp8_gemm: bad shape %d x %d x %d", M, N, K);
    if (!is_fp8_dt(a_dt)) FX_FAIL("fx_fp8_gemm: unsupported 8-bit dtype enum %d", a_dt);
    if (M == 0 || N == 0) return 0;
    if (!D || (K > 0 && (!A || !B || !SA || !SB))) FX_FAIL("fx_fp8_gemm: null pointer");
    if (K > 0 && (bad_rows(A, lda) || bad_rows(B, ldb))) FX_FAIL("fx_fp8_gemm: rows of A and B must start at 16-byte addresses");
    if ((K > 0 && (lda < K || ldb < K)) || ldd < N || (C && ldc < N)) FX_FAIL("fx_fp8_gemm: a row stride is shorter than the row");
    if (ws_bytes < fx_fp8_gemm_ws_bytes(M, N, K)) FX_FAIL("fx_fp8_gemm: workspace too small");
    (void)ws;
    const Fp8View a{(const uint8_t*)A, lda, (const uint8_t*)SA, sa_row, sa_k, a_tiles ? 7 : 0, M};
    const Fp8View b{(const uint8_t*)B, ldb, (const uint8_t*)SB, sb_row, sb_k, b_tiles ? 7 : 0, N};
    const int tiles_n = cdiv_i(N, 64);
    if ((int64_t)tiles_n * cdiv_i(M, 64) > 0x7fffffff) FX_FAIL("fx_fp8_gemm: too many tiles");
    FX_FP8_OUT(a_dt, d_dt, fp8_gemm_simple_kernel<AF, TD><<<dim3((unsigned)(cdiv_i(M, 64) * tiles_n)), 256, 0, stream>>>(
        a, b, K, (const TD*)C, ldc, (TD*)D, ldd, tiles_n));
    FX_CHECK_LAUNCH("fx_fp8_gemm");
    return 0;
}

extern "C" int fx_fp8_grouped_gemm(const void* A, int64_t lda, int a_dt, const void* SA, int64_t sa_row, int64_t sa_k,
                                   const int32_t* row_map, int64_t a_rows, const void* B, int64_t ldb, int64_t b_expert,
                                   const void* SB, int64_t sb_row, int64_t sb_k, int64_t sb_expert, int b_tiles,
                                   const int32_t* counts, int E, int64_t total_rows, void* D, int64_t ldd, int N, int K, int d_dt,
                                   hipStream_t stream) {
    if (E <= 0 || total_rows < 0 || N < 0 || K < 0) FX_FAIL("fx_fp8_grouped_gemm: bad shape");
    if (!is_fp8_dt(a_dt)) FX_FAIL("fx_fp8_grouped_gemm: unsupported 8-bit dtype enum %d", a_dt);
    if (total_rows > (1 << 24)) FX_FAIL("fx_fp8_grouped_gemm: at most 2^24 expert rows");
    if (total_rows == 0 || N == 0) return 0;
    if (!counts || !D || (K > 0 && (!A || !B || !SA || !SB))) FX_FAIL("fx_fp8_grouped_gemm: null pointer");
    if (K > 0 && (bad_rows(A, lda) || bad_rows(B, ldb) || (b_expert & 15))) FX_FAIL("fx_fp8_grouped_gemm: rows of A and B must start at 16-byte addresses");
    if ((K > 0 && (lda < K || ldb < K)) || ldd < N) FX_FAIL("fx_fp8_grouped_gemm: a row stride is shorter than the row");
    if (row_map ? (a_rows <= 0 || a_rows > 0x7fffffff) : a_rows < total_rows) FX_FAIL("fx_fp8_grouped_gemm: A has %lld rows", (long long)a_rows);
    const Fp8View a{(const uint8_t*)A, lda, (const uint8_t*)SA, sa_row, sa_k, 0, 0};
    const Fp8View b{(const uint8_t*)B, ldb, (const uint8_t*)SB, sb_row, sb_k, b_tiles ? 7 : 0, N};
    const int tiles_n = cdiv_i(N, 64);
    const int64_t most = total_rows / 64 + (E < total_rows ? E : total_rows);
    if (most * tiles_n > 0x7fffffff) FX_FAIL("fx_fp8_grouped_gemm: too many tiles");
    FX_FP8_OUT(a_dt, d_dt, fp8_grouped_simple_kernel<AF, TD><<<dim3((unsigned)(most * tiles_n)), 256, 0, stream>>>(
        a, b, b_expert, sb_expert, counts, E, total_rows, row_map, (int)a_rows, K, (TD*)D, ldd, tiles_n));
    FX_CHECK_LAUNCH("fx_fp8_grouped_gemm");
    return 0;
}

extern "C" int fx_fp8_grouped_wgrad(const void* A, int64_t lda, int a_dt, const void* SA, int64_t sa_row, int64_t sa_k, const void* B,
                                    int64_t ldb, const void* SB, int64_t sb_row, int64_t sb_k, const int32_t* counts, int E,
                                    int64_t capacity, const void* C, int64_t ldc, int64_t c_expert, void* D, int64_t ldd,
                                    int64_t d_expert, int M, int N, int d_dt, hipStream_t stream) {
    if (E <= 0 || capacity < 0 || (capacity & 127) || M < 0 || N < 0) FX_FAIL("fx_fp8_grouped_wgrad: bad shape");
    if (!is_fp8_dt(a_dt)) FX_FAIL("fx_fp8_grouped_wgrad: unsupported 8-bit dtype enum %d", a_dt);
    if (capacity > (1 << 24)) FX_FAIL("fx_fp8_grouped_wgrad: at most 2^24 expert rows");
    if (M == 0 || N == 0) return 0;
    if (!counts || !D || (capacity > 0 && (!A || !B || !SA || !SB))) FX_FAIL("fx_fp8_grouped_wgrad: null pointer");
    if (capacity > 0 && (bad_rows(A, lda) || bad_rows(B, ldb))) FX_FAIL("fx_fp8_grouped_wgrad: rows of A and B must start at 16-byte addresses");
    if (lda < capacity || ldb < capacity || ldd < N || (C && ldc < N)) FX_FAIL("fx_fp8_grouped_wgrad: a row stride is shorter than the row");
    const Fp8View a{(const uint8_t*)A, lda, (const uint8_t*)SA, sa_row, sa_k, 0, M};
    const Fp8View b{(const uint8_t*)B, ldb, (const uint8_t*)SB, sb_row, sb_k, 0, N};
    const int tiles_m = cdiv_i(M, 64), tiles_n = cdiv_i(N, 64);
    if ((int64_t)tiles_m * tiles_n * E > 0x7fffffff) FX_FAIL("fx_fp8_grouped_wgrad: too many tiles");
    FX_FP8_OUT(a_dt, d_dt, fp8_wgrad_simple_kernel<AF, TD><<<dim3((unsigned)(tiles_m * tiles_n * E)), 256, 0, stream>>>(
        a, b, counts, E, capacity, (const TD*)C, ldc, c_expert, (TD*)D, ldd, d_expert, tiles_m, tiles_n));
    FX_CHECK_LAUNCH("fx_fp8_grouped_wgrad");
    return 0;
}
