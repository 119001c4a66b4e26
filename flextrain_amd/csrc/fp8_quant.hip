// Block quantiser: bf16 / fp16 / fp32 matrices to 8-bit values with one scale per block of 128 (fp8.h), gfx950.
//
//   rows     block = 1 row x 128 columns:  q (R, C),  s (R, ceil(C / 128))
//   columns  block = 128 rows x 1 column, written transposed:  qt (C, R),  st (C, ceil(R / 128))
//   tiles    block = 128 x 128:  q (R, C) and qt (C, R) with one scale between them
// Row scales serve a product that contracts over the columns (forward, input gradient), column scales one that
// contracts over the rows (weight gradient).  Both products then read operands whose contraction axis is
// contiguous, so one form of the matrix kernel serves them all.
// Scales are stored with the block index of the contraction outermost (row index contiguous): the tile loader
// of the product reads the scales of 32 consecutive rows at one k block as 32 consecutive bytes.
#include "fp8.h"
#include "flexhip.h"

namespace fx {

// Distances between the matrices of a batch (blockIdx.y).
struct QuantBatch {
    int64_t x, q, s, qt, st;
};

// Rows form.  A workgroup takes 16 rows x 512 columns: a wave 4 rows, one after the other, its 64 lanes
// covering 4 blocks of 128 columns (1 KB of bf16 per load instruction).  A 16-lane group ends with the scale
// bytes of 4 consecutive rows, which leave as one 4-byte store.
template <typename T, int FMT, bool VEC>
__global__ __launch_bounds__(256) void fp8_rows_kernel(const T* __restrict__ X, int64_t ldx, uint8_t* __restrict__ Q,
                                                       int64_t ldq, uint8_t* __restrict__ S, int64_t lds, int64_t rows,
                                                       int64_t cols, unsigned tiles_c, QuantBatch batch) {
    X += blockIdx.y * batch.x;
    Q += blockIdx.y * batch.q;
    S += blockIdx.y * batch.s;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int64_t tr = blockIdx.x / tiles_c, tc = blockIdx.x % tiles_c;
    const int64_t row0 = tr * 16 + wave * 4, col = tc * 512 + lane * 8;
    float x[4][8];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int64_t r = row0 + u;
        load8_or_zero<T, VEC>(X + (r < rows ? r : 0) * ldx, col, r < rows ? cols : 0, x[u]);
    }
    unsigned bytes = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        unsigned m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, finite_mag(x[u][j]));
        const int b = scale_byte<FMT>(group_umax<16>(m));
        bytes |= (unsigned)b << (8 * u);
        const float inv = inverse_scale(b);
        if (row0 + u < rows && col < ldq) {
            uint2 o;
            o.x = pack_fp8x4<FMT>(x[u][0] * inv, x[u][1] * inv, x[u][2] * inv, x[u][3] * inv);
            o.y = pack_fp8x4<FMT>(x[u][4] * inv, x[u][5] * inv, x[u][6] * inv, x[u][7] * inv);
            *reinterpret_cast<uint2*>(Q + (row0 + u) * ldq + col) = o;
        }
    }
    if ((lane & 15) == 0 && col < cols) {
        uint8_t* s = S + (col >> 7) * lds + row0;
        if (row0 + 4 <= rows && ((reinterpret_cast<uintptr_t>(s)) & 3) == 0) {
            *reinterpret_cast<unsigned*>(s) = bytes;
        } else {
            for (int u = 0; u < 4; ++u)
                if (row0 + u < rows) s[u] = (uint8_t)(bytes >> (8 * u));
        }
    }
}

// 128 x 128 tile per workgroup of 256 lanes; lane (g, c) = (tid / 16, tid % 16) holds rows 8 g .. 8 g + 7 of
// columns 8 c .. 8 c + 7 in registers, so both directions are quantised from one read.
//   row maxima     over the 16 lanes of a g
//   column maxima  over a lane's 8 rows, the 4 g of its wave, then the 4 waves through LDS
//   transposed     a lane packs 8 consecutive rows of a column into 8 bytes, staged in LDS (pitch 136 bytes),
//                  and full 128-byte runs of a transposed row leave 16 bytes per lane
// ROWS / COLS: which outputs are written; TILE: one scale for all 128 x 128 values.
// GROUPED: the row axis is the expert-padded order (find_group_tile), optionally gathered through MAP.
template <typename T, int FMT, bool VEC, bool ROWS, bool COLS, bool TILE, bool GROUPED>
__global__ __launch_bounds__(256) void fp8_tile_kernel(
    const T* __restrict__ X, int64_t ldx, uint8_t* __restrict__ Q, int64_t ldq, uint8_t* __restrict__ S, int64_t lds,
    uint8_t* __restrict__ QT, int64_t ldt, uint8_t* __restrict__ ST, int64_t ldst, int64_t rows, int64_t cols,
    unsigned tiles_c, const int32_t* __restrict__ COUNTS, int E, const int32_t* __restrict__ MAP, int64_t src_rows,
    QuantBatch batch) {
    X += blockIdx.y * batch.x;
    if (ROWS) { Q += blockIdx.y * batch.q; S += blockIdx.y * batch.s; }
    if (COLS) { QT += blockIdx.y * batch.qt; ST += blockIdx.y * batch.st; }
    constexpr int PITCH = 136;
    __shared__ __align__(16) uint8_t stage[COLS ? 128 * PITCH : 16];
    __shared__ unsigned colmax[4][128];
    __shared__ unsigned tilemax[4];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int g = tid >> 4, c = tid & 15;
    const int64_t tr = blockIdx.x / tiles_c, tc = blockIdx.x % tiles_c;
    int64_t first = tr * 128;
    int live = (int)min((int64_t)128, rows - first);
    if (GROUPED) {
        // every expert's rows start at a multiple of 128 of the row axis written here
        const GroupTile t = find_group_tile<7>(COUNTS, E, (int)tr, rows, lane);
        first = (int64_t)t.row0 + t.m0;
        live = max(0, min(128, t.rows - t.m0));
    }
    const int64_t col = tc * 128 + c * 8;
    float x[8][8];
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        const int r = g * 8 + p;
        const bool ok = r < live;
        int64_t src = ok ? first + r : 0;
        // a map entry outside the source must not turn into an address outside it
        if (GROUPED && MAP != nullptr && ok) src = min(max((int64_t)MAP[src], (int64_t)0), src_rows - 1);
        load8_or_zero<T, VEC>(X + src * ldx, col, ok ? cols : 0, x[p]);
    }
    unsigned rmax[8], cmax[8];
#pragma unroll
    for (int p = 0; p < 8; ++p) rmax[p] = cmax[p] = 0;
#pragma unroll
    for (int p = 0; p < 8; ++p)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const unsigned m = finite_mag(x[p][j]);
            rmax[p] = max(rmax[p], m);
            cmax[j] = max(cmax[j], m);
        }
    int tile_b = 0;
    if (TILE) {
        unsigned m = 0;
#pragma unroll
        for (int p = 0; p < 8; ++p) m = max(m, rmax[p]);
        m = group_umax<64>(m);
        if (lane == 0) tilemax[wave] = m;
        __syncthreads();
        tile_b = scale_byte<FMT>(max(max(tilemax[0], tilemax[1]), max(tilemax[2], tilemax[3])));
        if (tid == 0) {
            S[tc * lds + tr] = (uint8_t)tile_b;
            if (COLS) ST[tr * ldst + tc] = (uint8_t)tile_b;
        }
    }
    if (COLS && !TILE) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            unsigned m = cmax[j];
            m = max(m, (unsigned)__shfl_xor((int)m, 16, 64));
            m = max(m, (unsigned)__shfl_xor((int)m, 32, 64));
            cmax[j] = m;
        }
        if (lane < 16)
#pragma unroll
            for (int j = 0; j < 8; ++j) colmax[wave][c * 8 + j] = cmax[j];
        __syncthreads();
    }
    if (ROWS) {
        unsigned lo = 0, hi = 0;
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            const int b = TILE ? tile_b : scale_byte<FMT>(group_umax<16>(rmax[p]));
            (p < 4 ? lo : hi) |= (unsigned)b << (8 * (p & 3));
            const float inv = inverse_scale(b);
            if (g * 8 + p < live && col < ldq) {
                uint2 o;
                o.x = pack_fp8x4<FMT>(x[p][0] * inv, x[p][1] * inv, x[p][2] * inv, x[p][3] * inv);
                o.y = pack_fp8x4<FMT>(x[p][4] * inv, x[p][5] * inv, x[p][6] * inv, x[p][7] * inv);
                *reinterpret_cast<uint2*>(Q + (first + g * 8 + p) * ldq + col) = o;
            }
        }
        if (!TILE && c == 0) {
            uint8_t* s = S + tc * lds + first + g * 8;
            if (g * 8 + 8 <= live && (reinterpret_cast<uintptr_t>(s) & 7) == 0) {
                *reinterpret_cast<uint2*>(s) = make_uint2(lo, hi);
            } else {
                for (int p = 0; p < 8; ++p)
                    if (g * 8 + p < live) s[p] = (uint8_t)((p < 4 ? lo : hi) >> (8 * (p & 3)));
            }
        }
    }
    if (COLS) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            int b = tile_b;
            if (!TILE) {
                const int k = c * 8 + j;
                b = scale_byte<FMT>(max(max(colmax[0][k], colmax[1][k]), max(colmax[2][k], colmax[3][k])));
                if (g == 0 && col + j < cols) ST[tr * ldst + col + j] = (uint8_t)b;
            }
            const float inv = inverse_scale(b);
            uint2 o;
            o.x = pack_fp8x4<FMT>(x[0][j] * inv, x[1][j] * inv, x[2][j] * inv, x[3][j] * inv);
            o.y = pack_fp8x4<FMT>(x[4][j] * inv, x[5][j] * inv, x[6][j] * inv, x[7][j] * inv);
            *reinterpret_cast<uint2*>(stage + (c * 8 + j) * PITCH + g * 8) = o;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int id = i * 256 + tid, k = id >> 3, ch = id & 7;
            const int64_t cc = tc * 128 + k, at = tr * 128 + ch * 16;
            if (cc < cols && at < ldt) {
                const uint2 a = *reinterpret_cast<const uint2*>(stage + k * PITCH + ch * 16);
                const uint2 b = *reinterpret_cast<const uint2*>(stage + k * PITCH + ch * 16 + 8);
                uint4 o;
                o.x = a.x; o.y = a.y; o.z = b.x; o.w = b.y;
                *reinterpret_cast<uint4*>(QT + cc * ldt + at) = o;
            }
        }
    }
}

// 16-byte packs: every row of x starts at a 16-byte address and its length is a whole number of 8-value packs
static bool vec_rows(const void* x, int64_t ldx, int64_t cols, int x_dt) {
    return aligned16(x) && (ldx * elem_size(x_dt)) % 16 == 0 && cols % 8 == 0;
}

}  // namespace fx

using namespace fx;

static int check_quant(const char* what, const void* x, int64_t ldx, int64_t rows, int64_t cols, int x_dt, int q_dt) {
    if (rows < 0 || cols <= 0) FX_FAIL("%s: bad shape rows=%lld cols=%lld", what, (long long)rows, (long long)cols);
    if (x_dt != DT_F32 && x_dt != DT_F16 && x_dt != DT_BF16) FX_FAIL("%s: unsupported input dtype enum %d", what, x_dt);
    if (!is_fp8_dt(q_dt)) FX_FAIL("%s: unsupported 8-bit dtype enum %d", what, q_dt);
    if (ldx < cols) FX_FAIL("%s: a row of x holds %lld values, its stride is %lld", what, (long long)cols, (long long)ldx);
    if (rows > 0 && !x) FX_FAIL("%s: null pointer", what);
    return 0;
}

extern "C" int fx_fp8_quantize(const void* x, int64_t ldx, int64_t x_batch, int batch, int64_t rows, int64_t cols, int x_dt,
                               int q_dt, int tiles, void* q, int64_t ldq, int64_t q_batch, void* s, int64_t lds, int64_t s_batch,
                               void* qt, int64_t ldt, int64_t qt_batch, void* st, int64_t ldst, int64_t st_batch,
                               hipStream_t stream) {
    if (check_quant("fx_fp8_quantize", x, ldx, rows, cols, x_dt, q_dt) != 0) return -1;
    if (batch < 0 || batch > 65535) FX_FAIL("fx_fp8_quantize: a batch holds at most 65535 matrices");
    if (rows == 0 || batch == 0) return 0;
    if (!q || !s || (!qt) != (!st)) FX_FAIL("fx_fp8_quantize: null pointer");
    const int64_t rb = (rows + 127) / 128, cb = (cols + 127) / 128;
    if ((ldq & 15) || ldq < cols || !aligned16(q)) FX_FAIL("fx_fp8_quantize: rows of q must start at 16-byte addresses and hold %lld values", (long long)cols);
    if (lds < (tiles ? rb : rows)) FX_FAIL("fx_fp8_quantize: scale stride too small");
    if (qt && ((ldt & 15) || ldt < rows || !aligned16(qt) || ldst < (tiles ? cb : cols)))
        FX_FAIL("fx_fp8_quantize: rows of qt must start at 16-byte addresses and hold %lld values, its scales %lld", (long long)rows, (long long)cols);
    if (ldq - cols >= 16 || (qt && ldt - rows >= 16)) FX_FAIL("fx_fp8_quantize: the rows of q and qt are padded to the next multiple of 16, not further");
    if (batch > 1 && ((q_batch & 15) || (qt && (qt_batch & 15)))) FX_FAIL("fx_fp8_quantize: matrices of a batch must start at 16-byte addresses");
    const bool vec = vec_rows(x, ldx, cols, x_dt) && (batch == 1 || (x_batch * elem_size(x_dt)) % 16 == 0);
    const QuantBatch qb{x_batch, q_batch, s_batch, qt_batch, st_batch};
    uint8_t *Q = (uint8_t*)q, *S = (uint8_t*)s, *QT = (uint8_t*)qt, *ST = (uint8_t*)st;
    if (!qt && !tiles) {
        const int64_t tc = (cols + 511) / 512, blocks = (rows + 15) / 16 * tc;
        if (blocks > 0x7fffffff) FX_FAIL("fx_fp8_quantize: too many blocks");
        FX_DISPATCH_DTYPE(x_dt, T, FX_DISPATCH_FP8(q_dt, FMT, {
            if (vec) fp8_rows_kernel<T, FMT, true><<<dim3((unsigned)blocks, (unsigned)batch), 256, 0, stream>>>((const T*)x, ldx, Q, ldq, S, lds, rows, cols, (unsigned)tc, qb);
            else fp8_rows_kernel<T, FMT, false><<<dim3((unsigned)blocks, (unsigned)batch), 256, 0, stream>>>((const T*)x, ldx, Q, ldq, S, lds, rows, cols, (unsigned)tc, qb);
        }));
        FX_CHECK_LAUNCH("fx_fp8_quantize");
        return 0;
    }
    if (rb * cb > 0x7fffffff) FX_FAIL("fx_fp8_quantize: too many blocks");
    const unsigned blocks = (unsigned)(rb * cb);
#define FX_TILE(VEC_, COLS_, TILE_)                                                                           \
    fp8_tile_kernel<T, FMT, VEC_, true, COLS_, TILE_, false><<<dim3(blocks, (unsigned)batch), 256, 0, stream>>>( \
        (const T*)x, ldx, Q, ldq, S, lds, QT, ldt, ST, ldst, rows, cols, (unsigned)cb, nullptr, 0, nullptr, (int64_t)0, qb)
    FX_DISPATCH_DTYPE(x_dt, T, FX_DISPATCH_FP8(q_dt, FMT, {
        if (!qt) { if (vec) FX_TILE(true, false, true); else FX_TILE(false, false, true); }
        else if (tiles) { if (vec) FX_TILE(true, true, true); else FX_TILE(false, true, true); }
        else { if (vec) FX_TILE(true, true, false); else FX_TILE(false, true, false); }
    }));
#undef FX_TILE
    FX_CHECK_LAUNCH("fx_fp8_quantize");
    return 0;
}

extern "C" int64_t fx_fp8_grouped_capacity(int64_t rows, int E) {
    return rows < 0 || E <= 0 ? -1 : (rows + 127 * (int64_t)E) / 128 * 128;
}

extern "C" int fx_fp8_quantize_grouped_cols(const void* x, int64_t ldx, int64_t src_rows, int64_t rows, int64_t cols, int x_dt,
                                            int q_dt, const int32_t* counts, int E, const int32_t* row_map, void* qt, int64_t ldt,
                                            void* st, int64_t ldst, hipStream_t stream) {
    if (check_quant("fx_fp8_quantize_grouped_cols", x, ldx, src_rows, cols, x_dt, q_dt) != 0) return -1;
    if (rows < 0 || E <= 0) FX_FAIL("fx_fp8_quantize_grouped_cols: bad shape rows=%lld E=%d", (long long)rows, E);
    const int64_t cap = fx_fp8_grouped_capacity(rows, E);
    if (cap == 0) return 0;
    if (!counts || !qt || !st) FX_FAIL("fx_fp8_quantize_grouped_cols: null pointer");
    if (rows > 0 && src_rows == 0) FX_FAIL("fx_fp8_quantize_grouped_cols: the source has no rows");
    if (!row_map && src_rows < rows) FX_FAIL("fx_fp8_quantize_grouped_cols: x has fewer rows than the experts");
    if (rows > (1 << 24) || src_rows > 0x7fffffff) FX_FAIL("fx_fp8_quantize_grouped_cols: at most 2^24 expert rows");
    if ((ldt & 15) || ldt != cap || !aligned16(qt) || ldst < cols)
        FX_FAIL("fx_fp8_quantize_grouped_cols: qt holds %lld values a row, at 16-byte addresses, and its scales %lld", (long long)cap, (long long)cols);
    const int64_t cb = (cols + 127) / 128;
    if (cap / 128 * cb > 0x7fffffff) FX_FAIL("fx_fp8_quantize_grouped_cols: too many blocks");
    const unsigned blocks = (unsigned)(cap / 128 * cb);
    const bool vec = vec_rows(x, ldx, cols, x_dt);
#define FX_TILE(VEC_)                                                                                         \
    fp8_tile_kernel<T, FMT, VEC_, false, true, false, true><<<dim3(blocks), 256, 0, stream>>>(                \
        (const T*)x, ldx, nullptr, (int64_t)0, nullptr, (int64_t)0, (uint8_t*)qt, ldt, (uint8_t*)st, ldst, rows, cols,  \
        (unsigned)cb, counts, E, row_map, src_rows, QuantBatch{0, 0, 0, 0, 0})
    FX_DISPATCH_DTYPE(x_dt, T, FX_DISPATCH_FP8(q_dt, FMT, { if (vec) FX_TILE(true); else FX_TILE(false); }));
#undef FX_TILE
    FX_CHECK_LAUNCH("fx_fp8_quantize_grouped_cols");
    return 0;
}
