// 8-bit floating point with one power-of-two scale per block of 128 values, gfx950.
//
// Values are OCP e4m3 (largest 448) or e5m2 (largest 57344).  A block's scale is 2^e with the smallest
// integer e that brings the block's largest finite magnitude to at most the type's largest number; it is
// held as the byte e + 127 (e8m0), the form v_mfma_scale_f32_*_f8f6f4 takes, so the matrix instruction
// applies it at no cost.  Why a power of two and not amax / 448 in fp32: dividing by it is exact, so the one
// rounding of a value is the one to its 3 (2) mantissa bits, whose relative size does not depend on the
// scale; what it gives up is at most one of the type's 18 (32) binades.  With fp32 scales the product of
// two scales would have to be applied to every accumulator after every block of 128 k (one vector
// instruction per two matrix passes, and a second set of accumulators).
// A block of zeros has e = 0.  Infinities and NaN do not count towards the largest magnitude: they stay
// (e4m3 has no infinity: NaN) and spoil only the sums that read them.
#pragma once
#include "common.h"

namespace fx {

enum : int { DT_E4M3 = 3, DT_E5M2 = 4 };

constexpr int FP8_BLOCK = 128;

inline bool is_fp8_dt(int dt) { return dt == DT_E4M3 || dt == DT_E5M2; }

// Bits of |v| when v is finite, else 0: unsigned comparison of such bits orders the magnitudes.
FX_DEV unsigned finite_mag(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v) & 0x7fffffffu;
    return u < 0x7f800000u ? u : 0u;
}

// e + 127 of a block whose largest finite magnitude has these bits.  Both largest numbers are 1.75 times a
// power of two (1.75 * 2^8, 1.75 * 2^15), so e is the exponent of amax less 8 (15), plus one when the
// mantissa exceeds 1.75: adding 0x1fffff carries into the exponent field for exactly those.
template <int FMT>
FX_DEV int scale_byte(unsigned amax_bits) {
    constexpr int top = FMT == DT_E4M3 ? 8 : 15;
    const int b = (int)((amax_bits + 0x1fffffu) >> 23) - top;
    return amax_bits == 0u ? 127 : (b < 0 ? 0 : b);
}

// 2^-e for the byte e + 127 (at most 247, so this is a normal number)
FX_DEV float inverse_scale(int byte) { return __builtin_bit_cast(float, (unsigned)(254 - byte) << 23); }

// Four values, already divided by their scale, to four bytes (nearest even).
template <int FMT>
FX_DEV unsigned pack_fp8x4(float a, float b, float c, float d) {
    int w = 0;
    if constexpr (FMT == DT_E4M3) {
        w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    } else {
        w = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, w, false);
        w = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, w, true);
    }
    return (unsigned)w;
}

// Largest of W contiguous lanes, as unsigned.
template <int W>
FX_DEV unsigned group_umax(unsigned v) {
#pragma unroll
    for (int off = W / 2; off > 0; off >>= 1) {
        const unsigned o = (unsigned)__shfl_xor((int)v, off, 64);
        v = v > o ? v : o;
    }
    return v;
}

// Largest of the 16 lanes of a row of the wave (rotations within the row: no LDS round trips), and of the four rows.
FX_DEV unsigned row16_umax(unsigned v) {
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));     // row_ror:8
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
    return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
}
FX_DEV unsigned rows4_umax(unsigned v) {
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);      // rows 0 and 2 twice / rows 1 and 3 twice
    v = max((unsigned)a[0], (unsigned)a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max((unsigned)b[0], (unsigned)b[1]);
}

// ---------------------------------------------------------------- 2-byte inputs, two to a register
// Magnitudes of bf16 / fp16 values order like their low 15 bits, so maxima are taken on pairs as they come from memory, and
// v_cvt_scalef32_pk_{fp8,bf8}_{bf16,f16} divides a pair by its scale and rounds it in one instruction (checked over all
// 65,536 inputs of either type: nearest even, subnormals kept).
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
typedef short s16x2_t __attribute__((ext_vector_type(2)));

FX_DEV unsigned pk_umax(unsigned a, unsigned b) {
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a), __builtin_bit_cast(u16x2_t, b)));
}
template <typename T> struct Half;
template <> struct Half<bf16> {
    static constexpr unsigned INF = 0x7f80u;                 // magnitude bits from here on are not finite
    static FX_DEV unsigned f32_bits(unsigned m) { return m << 16; }
};
template <> struct Half<f16> {
    static constexpr unsigned INF = 0x7c00u;
    static FX_DEV unsigned f32_bits(unsigned m) {
        const unsigned short h = (unsigned short)m;
        const float f = (float)__builtin_bit_cast(f16, h);
        return __builtin_bit_cast(unsigned, f);
    }
};
// Magnitude bits of a pair, 0 in the place of a value that is not finite.
template <typename T>
FX_DEV unsigned pk_finite(unsigned x) {
    unsigned lo = x & 0x7fffu, hi = (x >> 16) & 0x7fffu;
    lo = lo < Half<T>::INF ? lo : 0u;
    hi = hi < Half<T>::INF ? hi : 0u;
    return lo | (hi << 16);
}
// Two pairs, divided by 2^(byte - 127), to four bytes.
template <typename T, int FMT>
FX_DEV unsigned cvt_pairs(unsigned p0, unsigned p1, int byte) {
    const unsigned sb = (unsigned)byte << 23;
    const float scale = __builtin_bit_cast(float, sb);
    s16x2_t w = {0, 0};
    typedef T pair_t __attribute__((ext_vector_type(2)));
    const pair_t a = __builtin_bit_cast(pair_t, p0), b = __builtin_bit_cast(pair_t, p1);
    if constexpr (__is_same(T, bf16) && FMT == DT_E4M3) {
        w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, a, scale, false);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, b, scale, true);
    } else if constexpr (__is_same(T, bf16)) {
        w = __builtin_amdgcn_cvt_scalef32_pk_bf8_bf16(w, a, scale, false);
        w = __builtin_amdgcn_cvt_scalef32_pk_bf8_bf16(w, b, scale, true);
    } else if constexpr (FMT == DT_E4M3) {
        w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w, a, scale, false);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w, b, scale, true);
    } else {
        w = __builtin_amdgcn_cvt_scalef32_pk_bf8_f16(w, a, scale, false);
        w = __builtin_amdgcn_cvt_scalef32_pk_bf8_f16(w, b, scale, true);
    }
    return __builtin_bit_cast(unsigned, w);
}
typedef unsigned u32x4_any_t __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_any_t __attribute__((ext_vector_type(4), aligned(4)));

// Eight consecutive 2-byte values of a row that has `cols` of them as four pairs, 0 behind its end.  WHOLE: a lane's eight
// lie in the row or behind its end together.
template <typename T, bool WHOLE, bool NT>
FX_DEV void load8(const T* row, int64_t col, int64_t cols, unsigned (&o)[4]) {
    if constexpr (WHOLE) {
        u32x4_any_t v = {0u, 0u, 0u, 0u};
        if (col < cols) {
            const u32x4_any_t* p = reinterpret_cast<const u32x4_any_t*>(row + col);
            v = NT ? __builtin_nontemporal_load(p) : *p;
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) o[d] = v[d];
    } else {
        const unsigned short* p = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const unsigned lo = col + 2 * d < cols ? p[col + 2 * d] : 0u, hi = col + 2 * d + 1 < cols ? p[col + 2 * d + 1] : 0u;
            o[d] = lo | (hi << 16);
        }
    }
}
// The same of 4-byte values.
template <bool WHOLE, bool NT>
FX_DEV void load8(const float* row, int64_t col, int64_t cols, float (&o)[8]) {
    if constexpr (WHOLE) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            f32x4_any_t v = {0.f, 0.f, 0.f, 0.f};
            if (col < cols) {
                const f32x4_any_t* p = reinterpret_cast<const f32x4_any_t*>(row + col + 4 * u);
                v = NT ? __builtin_nontemporal_load(p) : *p;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) o[4 * u + e] = v[e];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = col + j < cols ? row[col + j] : 0.f;
    }
}

// ---------------------------------------------------------------- experts
// Expert-sorted rows: expert e owns COUNTS[e] consecutive rows.  The counts stay on the device, so a workgroup
// finds its place itself: the 64 lanes of a wave look at 64 experts at a time (a scan over the lanes for the rows, one
// for the tiles).  The counts may promise more rows than there are (the host cannot check them): a count is cut to
// the rows that are left, so every tile that exists has rows and no address leaves the buffers.  total_rows is at
// most 2^24, 64 counts fit 32 bits.

// A value that all lanes hold alike, in a scalar register.
FX_DEV int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Inclusive sum over the lanes of a wave: within rows of 16 by shifts, then across rows by broadcasts of a row's last
// lane (six additions with a data-parallel operand; shuffles through the LDS unit take ten times as long, and a
// small product waits for this before it can load anything).
FX_DEV int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);      // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);      // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);      // row_bcast:31 into rows 2 and 3
    return v;
}
FX_DEV int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// Expert e0 + lane of a step over 64 experts: its first row and its rows (cut to what is left), given the rows before
// the step; moves row_base behind the step.
FX_DEV void group_rows(const int32_t* COUNTS, int E, int e0, int total_rows, int lane, int& row_base, int& row0, int& rows) {
    const int c = e0 + lane < E ? min(max(COUNTS[e0 + lane], 0), total_rows) : 0;
    const int sum = wave_scan(c);
    row0 = min(row_base + sum - c, total_rows);
    rows = min(c, total_rows - row0);
    row_base = min(row_base + lane_value(sum, 63), total_rows);
}

struct GroupTile {     // (the same in every lane, and held in scalar registers)
    int e;             // expert, -1: the tile belongs to none
    int row0;          // its first row
    int rows;          // its rows
    int m0;            // first row of the tile within the expert, below `rows`
};

// Tile `tile` of the list of all experts' tiles of 2^SHIFT rows (an expert without rows has no tile).
template <int SHIFT>
FX_DEV GroupTile find_group_tile(const int32_t* COUNTS, int E, int tile, int64_t total_rows, int lane) {
    int row_base = 0, tile_base = 0;
    for (int e0 = 0; e0 < E; e0 += 64) {
        int row0, rows;
        group_rows(COUNTS, E, e0, (int)total_rows, lane, row_base, row0, rows);
        const int nt = (rows + (1 << SHIFT) - 1) >> SHIFT;
        const int it = tile_base + wave_scan(nt);
        const unsigned long long who = __ballot(tile >= it - nt && tile < it);
        if (who != 0ull) {
            const int src = uniform((int)__builtin_ctzll(who));
            GroupTile t;
            t.e = e0 + src;
            t.row0 = lane_value(row0, src);
            t.rows = lane_value(rows, src);
            t.m0 = (tile - lane_value(it - nt, src)) << SHIFT;
            return t;
        }
        tile_base = lane_value(it, 63);
    }
    return GroupTile{-1, 0, 0, 0};
}

// Number of such tiles.
template <int SHIFT>
FX_DEV int count_group_tiles(const int32_t* COUNTS, int E, int64_t total_rows, int lane) {
    int n = 0, row_base = 0;
    for (int e0 = 0; e0 < E; e0 += 64) {
        int row0, rows;
        group_rows(COUNTS, E, e0, (int)total_rows, lane, row_base, row0, rows);
        n += (rows + (1 << SHIFT) - 1) >> SHIFT;
    }
    return lane_value(wave_scan(n), 63);
}

// Rows of expert e, and where they start when every expert's rows begin at a multiple of 128.
struct GroupSpan {
    int padded0, rows;
};
FX_DEV GroupSpan find_group_span(const int32_t* COUNTS, int E, int e, int64_t capacity, int lane) {
    int padded0 = 0;
    int mine = 0;
    for (int e0 = 0; e0 <= e; e0 += 64) {
        const int i = e0 + lane;
        const int c = i < E ? min(max(COUNTS[i], 0), (int)capacity) : 0;
        const int p = i < e ? (c + 127) & ~127 : 0;
        padded0 = min(padded0 + lane_value(wave_scan(p), 63), (int)capacity);
        if (e < e0 + 64) mine = lane_value(c, e - e0);
    }
    GroupSpan s;
    s.padded0 = padded0;
    s.rows = padded0 + ((mine + 127) & ~127) <= (int)capacity ? mine : 0;
    return s;
}

// A launch has fewer than 2^32 threads along an axis.
static inline bool grid_fits(int64_t blocks, int threads) { return blocks * threads < ((int64_t)1 << 32); }

#define FX_DISPATCH_FP8(dt, FMT, ...)                                                \
    switch (dt) {                                                                    \
        case fx::DT_E4M3: { constexpr int FMT = fx::DT_E4M3; __VA_ARGS__; break; }   \
        case fx::DT_E5M2: { constexpr int FMT = fx::DT_E5M2; __VA_ARGS__; break; }   \
        default: FX_FAIL("unsupported 8-bit dtype enum %d", (int)(dt));              \
    }

}  // namespace fx
