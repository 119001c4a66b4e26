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

// Eight consecutive values of a row that has `cols` of them, 0 behind its end.  VEC: the address is 16-byte
// aligned and a pack never straddles the end.
template <typename T, bool VEC, bool NT = false>
FX_DEV void load8_or_zero(const T* row, int64_t col, int64_t cols, float (&o)[8]) {
    if (VEC && col < cols) {
        load_f32<T, 8, NT>(row + col, o);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = (!VEC && col + j < cols) ? (float)row[col + j] : 0.f;
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

FX_DEV int wave_scan(int v, int lane) {          // inclusive
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int a = __shfl_up(v, off, 64);
        if (lane >= off) v += a;
    }
    return v;
}

// Expert e0 + lane of a step over 64 experts: its first row and its rows (cut to what is left), given the rows before
// the step; moves row_base behind the step.
FX_DEV void group_rows(const int32_t* COUNTS, int E, int e0, int total_rows, int lane, int& row_base, int& row0, int& rows) {
    const int c = e0 + lane < E ? min(max(COUNTS[e0 + lane], 0), total_rows) : 0;
    const int sum = wave_scan(c, lane);
    row0 = min(row_base + sum - c, total_rows);
    rows = min(c, total_rows - row0);
    row_base = min(row_base + uniform(__shfl(sum, 63, 64)), total_rows);
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
        const int it = tile_base + wave_scan(nt, lane);
        const unsigned long long who = __ballot(tile >= it - nt && tile < it);
        if (who != 0ull) {
            const int src = (int)__builtin_ctzll(who);
            GroupTile t;
            t.e = uniform(e0 + src);
            t.row0 = uniform(__shfl(row0, src, 64));
            t.rows = uniform(__shfl(rows, src, 64));
            t.m0 = uniform((tile - __shfl(it - nt, src, 64)) << SHIFT);
            return t;
        }
        tile_base = uniform(__shfl(it, 63, 64));
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
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, 64);
    return uniform(n);
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
        int p = i < e ? (c + 127) & ~127 : 0;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) p += __shfl_xor(p, off, 64);
        padded0 = min(padded0 + uniform(p), (int)capacity);
        if (e < e0 + 64) mine = uniform(__shfl(c, e - e0, 64));
    }
    GroupSpan s;
    s.padded0 = padded0;
    s.rows = padded0 + ((mine + 127) & ~127) <= (int)capacity ? mine : 0;
    return s;
}

#define FX_DISPATCH_FP8(dt, FMT, ...)                                                \
    switch (dt) {                                                                    \
        case fx::DT_E4M3: { constexpr int FMT = fx::DT_E4M3; __VA_ARGS__; break; }   \
        case fx::DT_E5M2: { constexpr int FMT = fx::DT_E5M2; __VA_ARGS__; break; }   \
        default: FX_FAIL("unsupported 8-bit dtype enum %d", (int)(dt));              \
    }

}  // namespace fx
