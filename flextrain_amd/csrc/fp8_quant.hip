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
#include <type_traits>

#include "fp8.h"
#include "flexhip.h"

namespace fx {

// Distances between the matrices of a batch (blockIdx.y).
struct QuantBatch {
    int64_t x, q, s, qt, st;
};

// A lane's 8 consecutive values of a row: maximum magnitude (as fp32 bits, finite values only), and the 8 bytes they become.
template <typename T, int FMT>
struct Lane8 {            // 4-byte types
    float x[8];
    template <bool WHOLE, bool NT> FX_DEV void load(const T* row, int64_t col, int64_t cols) { load8<WHOLE, NT>(row, col, cols, x); }
    FX_DEV unsigned mag() const {
        unsigned m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, finite_mag(x[j]));
        return m;
    }
    // largest of a 16-lane row, as fp32 bits
    FX_DEV unsigned block_mag() const { return row16_umax(mag()); }
    FX_DEV uint2 bytes(int b) const {
        const float inv = inverse_scale(b);
        return make_uint2(pack_fp8x4<FMT>(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv),
                          pack_fp8x4<FMT>(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv));
    }
};
template <typename T, int FMT>
struct Lane8Pairs {       // 2-byte types
    unsigned x[4];
    template <bool WHOLE, bool NT> FX_DEV void load(const T* row, int64_t col, int64_t cols) { load8<T, WHOLE, NT>(row, col, cols, x); }
    FX_DEV unsigned block_mag() const {
        unsigned m = pk_umax(pk_umax(x[0] & 0x7fff7fffu, x[1] & 0x7fff7fffu), pk_umax(x[2] & 0x7fff7fffu, x[3] & 0x7fff7fffu));
        m = max(m & 0xffffu, m >> 16);
        if (__any(m >= Half<T>::INF)) {
            m = pk_umax(pk_umax(pk_finite<T>(x[0]), pk_finite<T>(x[1])), pk_umax(pk_finite<T>(x[2]), pk_finite<T>(x[3])));
            m = max(m & 0xffffu, m >> 16);
        }
        return Half<T>::f32_bits(row16_umax(m));
    }
    FX_DEV uint2 bytes(int b) const { return make_uint2(cvt_pairs<T, FMT>(x[0], x[1], b), cvt_pairs<T, FMT>(x[2], x[3], b)); }
};
template <typename T, int FMT> struct LaneOf { typedef Lane8Pairs<T, FMT> type; };
template <int FMT> struct LaneOf<float, FMT> { typedef Lane8<float, FMT> type; };

// Rows form.  A workgroup takes 16 rows x 512 columns: a wave 4 rows, one after the other, its 64 lanes
// covering 4 blocks of 128 columns (1 KB of bf16 per load instruction).  A 16-lane group ends with the scale
// bytes of 4 consecutive rows, which leave as one 4-byte store.  Bound by memory: 8192 x 14336 bf16 62 us, 5.7 TB/s.
template <typename T, int FMT>
__global__ __launch_bounds__(256) void fp8_rows_kernel(const T* __restrict__ X, int64_t ldx, uint8_t* __restrict__ Q,
                                                       int64_t ldq, uint8_t* __restrict__ S, int64_t lds, int64_t rows,
                                                       int64_t cols, unsigned tiles_c, QuantBatch batch) {
    X += blockIdx.y * batch.x;
    Q += blockIdx.y * batch.q;
    S += blockIdx.y * batch.s;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int64_t tr = blockIdx.x / tiles_c, tc = blockIdx.x % tiles_c;
    const int64_t row0 = tr * 16 + wave * 4, col = tc * 512 + lane * 8;
    typename LaneOf<T, FMT>::type x[4];
    // (the last columns of rows whose length is no multiple of 8 are read one by one)
    auto load = [&](auto whole) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t r = row0 + u;
            x[u].template load<decltype(whole)::value, false>(X + (r < rows ? r : 0) * ldx, col, r < rows ? cols : 0);
        }
    };
    if (tc * 512 + 512 <= cols || (cols & 7) == 0) load(std::true_type());
    else load(std::false_type());
    unsigned bytes = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int b = scale_byte<FMT>(x[u].block_mag());
        bytes |= (unsigned)b << (8 * u);
        if (row0 + u < rows && col < ldq) *reinterpret_cast<uint2*>(Q + (row0 + u) * ldq + col) = x[u].bytes(b);
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
// Bound by memory: 8192 x 14336 bf16 tiles 67 us (5.3 TB/s), both ways 96 us (4.9); 65536 x 1536 by expert 63 us (4.8).
template <typename T, int FMT, bool ROWS, bool COLS, bool TILE, bool GROUPED, bool NT>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 6 : 3) void fp8_tile_kernel(
    const T* __restrict__ X, int64_t ldx, uint8_t* __restrict__ Q, int64_t ldq, uint8_t* __restrict__ S, int64_t lds,
    uint8_t* __restrict__ QT, int64_t ldt, uint8_t* __restrict__ ST, int64_t ldst, int64_t rows, int64_t cols,
    unsigned tiles_c, const int32_t* __restrict__ COUNTS, int E, const int32_t* __restrict__ MAP, int64_t src_rows,
    QuantBatch batch) {
    X += blockIdx.y * batch.x;
    if (ROWS) { Q += blockIdx.y * batch.q; S += blockIdx.y * batch.s; }
    if (COLS) { QT += blockIdx.y * batch.qt; ST += blockIdx.y * batch.st; }
    constexpr int PITCH = 136;
    __shared__ __align__(16) uint8_t stage[COLS ? 128 * PITCH : 16];
    __shared__ unsigned colmax[4][sizeof(T) == 2 ? 64 : 128];
    __shared__ unsigned tilemax[4];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int g = tid >> 4, c = tid & 15;
    // Neighbouring tiles of a row on one XCD: 8192 x 14336 bf16 both ways 101 -> 95 us.  Expert columns are better off
    // without (65536 x 1536: 63 us, in bands 69).
    const int id = GROUPED ? (int)blockIdx.x : xcd_band((int)blockIdx.x, (int)gridDim.x);
    const int64_t tr = id / (int)tiles_c, tc = id % (int)tiles_c;
    int64_t first = tr * 128;
    int live = (int)min((int64_t)128, rows - first);
    if (GROUPED) {
        // every expert's rows start at a multiple of 128 of the row axis written here
        const GroupTile t = find_group_tile<7>(COUNTS, E, (int)tr, rows, lane);
        first = (int64_t)t.row0 + t.m0;
        live = max(0, min(128, t.rows - t.m0));
    }
    const int64_t col = tc * 128 + c * 8;
    typedef typename LaneOf<T, FMT>::type Lane;
    constexpr bool PAIRS = sizeof(T) == 2;
    Lane x[8];
    auto load = [&](auto whole) {
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            const int r = g * 8 + p;
            const bool ok = r < live;
            int64_t src = ok ? first + r : 0;
            // a map entry outside the source must not turn into an address outside it
            if (GROUPED && MAP != nullptr && ok) src = min(max((int64_t)MAP[src], (int64_t)0), src_rows - 1);
            x[p].template load<decltype(whole)::value, NT>(X + src * ldx, col, ok ? cols : 0);
        }
    };
    if (tc * 128 + 128 <= cols || (cols & 7) == 0) load(std::true_type());
    else load(std::false_type());
    int tile_b = 0;
    if (TILE) {
        unsigned m = 0;
#pragma unroll
        for (int p = 0; p < 8; ++p) m = max(m, x[p].block_mag());
        m = rows4_umax(m);
        if (lane == 0) tilemax[wave] = m;
        __syncthreads();
        tile_b = scale_byte<FMT>(max(max(tilemax[0], tilemax[1]), max(tilemax[2], tilemax[3])));
        if (tid == 0) {
            S[tc * lds + tr] = (uint8_t)tile_b;
            if (COLS) ST[tr * ldst + tc] = (uint8_t)tile_b;
        }
    }
    if (COLS && !TILE) {
        // maxima of this lane's 8 columns over its 8 rows, then over the wave's four rows of lanes
        if constexpr (PAIRS) {
            unsigned m[4];
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                m[d] = x[0].x[d] & 0x7fff7fffu;
#pragma unroll
                for (int p = 1; p < 8; ++p) m[d] = pk_umax(m[d], x[p].x[d] & 0x7fff7fffu);
            }
            const unsigned top = pk_umax(pk_umax(m[0], m[1]), pk_umax(m[2], m[3]));
            if (__any(max(top & 0xffffu, top >> 16) >= Half<T>::INF)) {
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    m[d] = 0;
#pragma unroll
                    for (int p = 0; p < 8; ++p) m[d] = pk_umax(m[d], pk_finite<T>(x[p].x[d]));
                }
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const auto a = __builtin_amdgcn_permlane16_swap(m[d], m[d], false, false);
                m[d] = pk_umax(a[0], a[1]);
                const auto b = __builtin_amdgcn_permlane32_swap(m[d], m[d], false, false);
                m[d] = pk_umax(b[0], b[1]);
                if (lane < 16) colmax[wave][c * 4 + d] = m[d];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                unsigned m = 0;
#pragma unroll
                for (int p = 0; p < 8; ++p) m = max(m, finite_mag(x[p].x[j]));
                m = rows4_umax(m);
                if (lane < 16) colmax[wave][c * 8 + j] = m;
            }
        }
        __syncthreads();
    }
    if (ROWS) {
        unsigned lo = 0, hi = 0;
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            const int b = TILE ? tile_b : scale_byte<FMT>(x[p].block_mag());
            (p < 4 ? lo : hi) |= (unsigned)b << (8 * (p & 3));
            if (g * 8 + p < live && col < ldq) *reinterpret_cast<uint2*>(Q + (first + g * 8 + p) * ldq + col) = x[p].bytes(b);
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
        unsigned cm[8];          // fp32 bits of the 8 columns' maxima
        if (!TILE) {
            if constexpr (PAIRS) {
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const int k = c * 4 + d;
                    const unsigned m = pk_umax(pk_umax(colmax[0][k], colmax[1][k]), pk_umax(colmax[2][k], colmax[3][k]));
                    cm[2 * d] = Half<T>::f32_bits(m & 0xffffu);
                    cm[2 * d + 1] = Half<T>::f32_bits(m >> 16);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int k = c * 8 + j;
                    cm[j] = max(max(colmax[0][k], colmax[1][k]), max(colmax[2][k], colmax[3][k]));
                }
            }
        }
        unsigned blo = 0, bhi = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int b = TILE ? tile_b : scale_byte<FMT>(cm[j]);
            (j < 4 ? blo : bhi) |= (unsigned)b << (8 * (j & 3));
            uint2 o;
            if constexpr (PAIRS) {
                // values of one column from two rows, side by side
                constexpr unsigned sel_lo = 0x05040100u, sel_hi = 0x07060302u;
                const unsigned sel = (j & 1) ? sel_hi : sel_lo;
                const int d = j >> 1;
                o.x = cvt_pairs<T, FMT>(__builtin_amdgcn_perm(x[1].x[d], x[0].x[d], sel), __builtin_amdgcn_perm(x[3].x[d], x[2].x[d], sel), b);
                o.y = cvt_pairs<T, FMT>(__builtin_amdgcn_perm(x[5].x[d], x[4].x[d], sel), __builtin_amdgcn_perm(x[7].x[d], x[6].x[d], sel), b);
            } else {
                const float inv = inverse_scale(b);
                o.x = pack_fp8x4<FMT>(x[0].x[j] * inv, x[1].x[j] * inv, x[2].x[j] * inv, x[3].x[j] * inv);
                o.y = pack_fp8x4<FMT>(x[4].x[j] * inv, x[5].x[j] * inv, x[6].x[j] * inv, x[7].x[j] * inv);
            }
            *reinterpret_cast<uint2*>(stage + (c * 8 + j) * PITCH + g * 8) = o;
        }
        if (!TILE && g == 0) {
            uint8_t* s = ST + tr * ldst + col;
            if (col + 8 <= cols && (reinterpret_cast<uintptr_t>(s) & 7) == 0) {
                *reinterpret_cast<uint2*>(s) = make_uint2(blo, bhi);
            } else {
                for (int j = 0; j < 8; ++j)
                    if (col + j < cols) s[j] = (uint8_t)((j < 4 ? blo : bhi) >> (8 * (j & 3)));
            }
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
    const QuantBatch qb{x_batch, q_batch, s_batch, qt_batch, st_batch};
    uint8_t *Q = (uint8_t*)q, *S = (uint8_t*)s, *QT = (uint8_t*)qt, *ST = (uint8_t*)st;
    if (!qt && !tiles) {
        const int64_t tc = (cols + 511) / 512, blocks = (rows + 15) / 16 * tc;
        if (!grid_fits(blocks, 256)) FX_FAIL("fx_fp8_quantize: too many blocks");
        FX_DISPATCH_DTYPE(x_dt, T, FX_DISPATCH_FP8(q_dt, FMT, {
            fp8_rows_kernel<T, FMT><<<dim3((unsigned)blocks, (unsigned)batch), 256, 0, stream>>>((const T*)x, ldx, Q, ldq, S, lds, rows, cols, (unsigned)tc, qb);
        }));
        FX_CHECK_LAUNCH("fx_fp8_quantize");
        return 0;
    }
    if (!grid_fits(rb * cb, 256)) FX_FAIL("fx_fp8_quantize: too many blocks");
    const unsigned blocks = (unsigned)(rb * cb);
    // read past the caches, which then hold the bytes being written: 8192 x 14336 bf16 both ways 111 -> 105 us, 65536 x 1536
    // columns by expert 72 -> 62 us
    const bool nt = (size_t)batch * (size_t)rows * (size_t)cols * elem_size(x_dt) >= kStreamingBytes;
#define FX_TILE(COLS_, TILE_, NT_)                                                                                 \
    fp8_tile_kernel<T, FMT, true, COLS_, TILE_, false, NT_><<<dim3(blocks, (unsigned)batch), 256, 0, stream>>>(    \
        (const T*)x, ldx, Q, ldq, S, lds, QT, ldt, ST, ldst, rows, cols, (unsigned)cb, nullptr, 0, nullptr, (int64_t)0, qb)
    FX_DISPATCH_DTYPE(x_dt, T, FX_DISPATCH_FP8(q_dt, FMT, {
        if (!qt) FX_TILE(false, true, false);
        else if (tiles) FX_TILE(true, true, false);
        else if (nt) FX_TILE(true, false, true);
        else FX_TILE(true, false, false);
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
    // rows of qt are operands of fx_fp8_grouped_wgrad, which takes strides below 2^23
    if (cap >= (1 << 23)) FX_FAIL("fx_fp8_quantize_grouped_cols: a capacity of %lld rows is not below 2^23", (long long)cap);
    if (!counts || !qt || !st) FX_FAIL("fx_fp8_quantize_grouped_cols: null pointer");
    if (rows > 0 && src_rows == 0) FX_FAIL("fx_fp8_quantize_grouped_cols: the source has no rows");
    if (!row_map && src_rows < rows) FX_FAIL("fx_fp8_quantize_grouped_cols: x has fewer rows than the experts");
    if (src_rows > 0x7fffffff) FX_FAIL("fx_fp8_quantize_grouped_cols: the source has too many rows");
    if ((ldt & 15) || ldt != cap || !aligned16(qt) || ldst < cols)
        FX_FAIL("fx_fp8_quantize_grouped_cols: qt holds %lld values a row, at 16-byte addresses, and its scales %lld", (long long)cap, (long long)cols);
    const int64_t cb = (cols + 127) / 128;
    if (!grid_fits(cap / 128 * cb, 256)) FX_FAIL("fx_fp8_quantize_grouped_cols: too many blocks");
    const unsigned blocks = (unsigned)(cap / 128 * cb);
    // rows read once (gathered ones belong to several experts) pass the caches, which hold the bytes being written instead
    const bool nt = row_map == nullptr && (size_t)rows * (size_t)cols * elem_size(x_dt) >= kStreamingBytes;
#define FX_TILE(NT_)                                                                                               \
    fp8_tile_kernel<T, FMT, false, true, false, true, NT_><<<dim3(blocks), 256, 0, stream>>>(                      \
        (const T*)x, ldx, nullptr, (int64_t)0, nullptr, (int64_t)0, (uint8_t*)qt, ldt, (uint8_t*)st, ldst, rows, cols,  \
        (unsigned)cb, counts, E, row_map, src_rows, QuantBatch{0, 0, 0, 0, 0})
    FX_DISPATCH_DTYPE(x_dt, T, FX_DISPATCH_FP8(q_dt, FMT, { if (nt) FX_TILE(true); else FX_TILE(false); }));
#undef FX_TILE
    FX_CHECK_LAUNCH("fx_fp8_quantize_grouped_cols");
    return 0;
}
