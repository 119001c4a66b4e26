// Tile code of the 8-bit products (see fp8_gemm.hip for what they compute), gfx950.
//
// A workgroup of WAVES_M x WAVES_N waves owns a BM x BN tile of D and walks K in steps of 128 bytes, one scale
// block.  Both operands go from memory straight into LDS (global_load_lds_dwordx4), two LDS stages alternate, one
// barrier per K-step.  LDS row r holds its 128 k-values as eight 16-byte chunks, chunk c at position
// c ^ ((r >> 1) & 7): 16 lanes of a fragment read (16 consecutive rows, one chunk) then touch all 64 banks once.
// The matrix instruction takes 32 consecutive k of a row per lane: two 16-byte LDS reads a fragment.  It runs for
// 64 cycles, twice as long as the 16-bit one on the same number of bytes, so a K-step costs the matrix pipe and the
// LDS exactly what a 64-wide K-step of the 16-bit core costs them, for twice the arithmetic.
#pragma once
#include <math.h>

#include "fp8.h"
#include "gemm_core2.h"

namespace fx {

typedef int i32x8_t __attribute__((ext_vector_type(8)));

constexpr int FP8_BK = 128;

// The compiler sees a new value (no instruction): what is computed from it stays where it is written.
#define FX_OPAQUE(x) asm volatile("" : "+v"(x))

// A wave-uniform pointer to global memory held in scalar registers (a no-op where the compiler knows).
typedef const __attribute__((address_space(1))) uint8_t* global_bytes;
FX_DEV global_bytes uniform_ptr(const uint8_t* p) {
    const uint64_t u = reinterpret_cast<uint64_t>(p);
    return reinterpret_cast<global_bytes>(((uint64_t)(unsigned)uniform((int)(u >> 32)) << 32) | (uint64_t)(unsigned)uniform((int)(unsigned)u));
}

// One operand: rows of 8-bit values, and the scale of (row, k block) at s[(row >> s_shift) * s_row + kb * s_k].
// A scale tensor spans less than 2^31 bytes, a row 2^23 (the host checks): lane offsets are 32 bits wide.
struct Fp8View {
    const uint8_t* p;
    const uint8_t* s;
    int ld, s_row, s_k;
    int s_shift;      // 0: a scale per row, 7: per 128 rows
    int ext;          // rows
};

// What a workgroup does next: D rows [m0, m0 + BM), columns [n0, n0 + BN) of one product.
template <typename TD>
struct Fp8Job {
    Fp8View A, B;
    int m0, n0, K;
    const int32_t* row_map;       // A row r of this product is source row row_map[r] (A.p, A.s: the whole source), or null
    int src_rows;
    const TD* C;
    TD* D;
};

// The B fragment goes first: the accumulator then holds the transposed tile, a lane four consecutive columns of D.
// SB / SA: which byte of the packed scales belongs to the fragment.
template <int AF, int SB, int SA>
FX_DEV f32x16_t mfma_fp8(const i32x8_t& b, const i32x8_t& a, f32x16_t c, int sb, int sa) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b, a, c, 0, AF == DT_E4M3 ? 0 : 1, SB, sb, SA, sa);
}

// 16 k-values of a row from k on, 0 behind K.  Rows start at 16-byte addresses; a chunk that K ends inside is read
// byte by byte (what lies behind K in memory is not the operand's).
FX_DEV u32x4_t load_chunk(const uint8_t* row, int k, int K) {
    union { u32x4_t q; uint8_t b[16]; } u;
    if (k + 16 <= K) return ldg16(row + k);
    const u32x4_t zero = {0u, 0u, 0u, 0u};
    u.q = zero;
    for (int j = 0; j < 16; ++j)
        if (k + j < K) u.b[j] = row[k + j];
    return u.q;
}

template <int AF, typename TD, int BM, int BN, int WAVES_M, int WAVES_N>
struct Fp8Loop {
    static constexpr int NW = WAVES_M * WAVES_N, NT = NW * 64;
    static constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N;
    static constexpr int TM = WM / 32, TN = WN / 32, MFMAS = TM * TN;
    static constexpr int NA = BM / 8 / NW, NB = BN / 8 / NW, LD = NA + NB;      // 1 KB load instructions per wave and K-step
    static constexpr int STAGE = (BM + BN) * FP8_BK;                            // bytes
    static constexpr int HI = TM / 2;                                           // A fragments with two register sets
    static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0, "tile rows must split evenly over the waves");
    static_assert((TM == 2 || TM == 4) && TN == 2, "fragment schedule below");
    static constexpr int PER = (LD + MFMAS - 1) / MFMAS;

    // fragments: a sub-step (64 k) needs TM of A and TN of B.  B and the upper half of A have two register sets that
    // alternate between the two sub-steps of a K-step; the lower half of A is read again as soon as its last MFMA
    // is issued.  All reads of a sub-step are then out two MFMAs before its end.
    i32x8_t alo[TM - HI], ahi[2][HI], bf[2][TN];
    unsigned aoff[NA], boff[NB];          // lane byte offsets of the tile loads
    const uint8_t *abase, *bbase;
    unsigned soa[TM / 2], sob[TN / 2];    // lane offsets of the scales: lane l fetches rows l, 64 + l, .. of its wave's
    const uint8_t *sabase, *sbbase;
    int sak, sbk;
    int rawa[TM / 2], rawb[TN / 2];       // scale bytes requested for the next K-step
    int sca, scb;                         // packed scales of the current one
    int wave, lane;
    unsigned lds_lane;

    // source row of tile row r of A (clamped to the last one; its products are never stored)
    static FX_DEV int64_t a_row(const Fp8Job<TD>& j, int r) {
        const int g = min(j.m0 + r, j.A.ext - 1);
        // a map entry outside the source must not turn into an address outside it
        return j.row_map != nullptr ? (int64_t)min(max(j.row_map[g], 0), j.src_rows - 1) : (int64_t)g;
    }

    // one instruction of a K-step's loads
    template <int IDX>
    FX_DEV void issue_one(uint8_t* buf) {
        if constexpr (IDX < NA) {
            load_to_lds16_s(aoff[IDX], abase, (unsigned)(uintptr_t)(buf + (IDX * NW + wave) * 1024));
            if (IDX == NA - 1) abase += FP8_BK;
        } else if constexpr (IDX < LD) {
            load_to_lds16_s(boff[IDX - NA], bbase, (unsigned)(uintptr_t)(buf + BM * FP8_BK + ((IDX - NA) * NW + wave) * 1024));
            if (IDX == LD - 1) bbase += FP8_BK;
        }
    }
    FX_DEV void move(int bytes) { abase += bytes; bbase += bytes; }
    FX_DEV void issue(uint8_t* buf) { static_for<0, LD>([&](auto i) { issue_one<decltype(i)::value>(buf); }); }

    FX_DEV void fetch_scales() {
#pragma unroll
        for (int i = 0; i < TM / 2; ++i) {
            unsigned o = soa[i];
            FX_OPAQUE(o);             // a 32-bit offset here, not a 64-bit one kept in a register pair
            rawa[i] = uniform_ptr(sabase)[o];
        }
#pragma unroll
        for (int i = 0; i < TN / 2; ++i) {
            unsigned o = sob[i];
            FX_OPAQUE(o);
            rawb[i] = uniform_ptr(sbbase)[o];
        }
        sabase += sak;
        sbbase += sbk;
    }
    // Byte i of the packed scales belongs to fragment i, whose row in lane l is 32 i + l % 32; lane l has fetched the
    // bytes of rows 64 u + l.  Exchanging the upper half of one copy with the lower half of another leaves the bytes of
    // rows 64 u + l % 32 in the first and those of rows 64 u + 32 + l % 32 in the second.
    template <int T>
    static FX_DEV int pack(const int (&raw)[T]) {
        unsigned w = (unsigned)raw[0];
        if constexpr (T == 2) w |= (unsigned)raw[1] << 16;
        const auto x = __builtin_amdgcn_permlane32_swap(w, w, false, false);
        return (int)(x[0] | (x[1] << 8));
    }
    FX_DEV void pack_scales(int& a, int& b) const {
        a = pack(rawa);
        b = pack(rawb);
    }

    FX_DEV void init() {
        lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int r = lane & 31, h = lane >> 5;
        lds_lane = (unsigned)(r * FP8_BK + (((2 * h) ^ swz(r)) << 4));
    }

    // A contraction is walked in steps(K) >= 2 K-steps.  When K is no multiple of 128 the last
    // step starts back(K) bytes early, so that it ends where the row's last 16-byte chunk ends and no load leaves the
    // row; patch() then zeroes the bytes that belong to the step before and those behind K (a K that ends inside the last
    // chunk of its 128 needs no step back, and still has bytes behind it).  A contraction of 128 or less
    // has a second step made of such bytes only; of one below 128, start<true>() zeroes what lies behind K in the first as well,
    // and the chunks behind its last one are requested from there.
    static FX_DEV int steps(int K) { return max(2, (K + FP8_BK - 1) / FP8_BK); }
    static FX_DEV int back(int K) { return steps(K) * FP8_BK - max(FP8_BK, (K + 15) & ~15); }
    // Zero what lies outside bytes [lo, hi) of the landed K-step in `buf`: every lane mends the chunks it loaded itself (its
    // loads have been waited for; a barrier follows).  lo is a multiple of 16.
    FX_DEV void patch(uint8_t* buf, int lo, int hi) const {
        const int rr = lane >> 3, pos = lane & 7;
#pragma unroll 1
        for (int i = 0; i < NA + NB; ++i) {
            const bool is_a = i < NA;
            const int q = (is_a ? i : i - NA) * NW + wave;
            const int c = pos ^ swz(q * 8 + rr);
            if (c * 16 < lo || c * 16 + 16 > hi) {
                uint8_t* p = buf + (is_a ? 0 : BM * FP8_BK) + q * 1024 + lane * 16;
                u32x4_t x = *reinterpret_cast<const u32x4_t*>(p);
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const int left = c * 16 < lo ? 0 : hi - c * 16 - d * 4;          // bytes of this word that stay
                    x[d] = left >= 4 ? x[d] : left <= 0 ? 0u : x[d] & (0xffffffffu >> (8 * (4 - left)));
                }
                *reinterpret_cast<u32x4_t*>(p) = x;
            }
        }
    }

    // Loads and scales of tile j (K > 0) from here on.
    FX_DEV void setup(const Fp8Job<TD>& j) {
        int lane = this->lane;
        FX_OPAQUE(lane);          // keeps the pieces of the offsets from being carried through the K loop in registers
        const int wm = wave / WAVES_N, wn = wave % WAVES_N;
        const int rr = lane >> 3, pos = lane & 7;
        const bool gathered = j.row_map != nullptr;
        const int last = min(FP8_BK, (j.K + 15) & ~15) - 16;        // offset of a row's last chunk within a K-step
        // offsets are taken from the tile's first row (gathered: from the source's, which is below 4 GB)
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int r = (i * NW + wave) * 8 + rr;
            const int64_t row = a_row(j, r) - (gathered ? 0 : j.m0);
            aoff[i] = (unsigned)(row * j.A.ld + min((pos ^ swz(r)) << 4, last));
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int r = (i * NW + wave) * 8 + rr;
            boff[i] = (unsigned)((int64_t)(min(j.n0 + r, j.B.ext - 1) - j.n0) * j.B.ld + min((pos ^ swz(r)) << 4, last));
        }
        abase = j.A.p + (gathered ? 0 : (int64_t)j.m0 * j.A.ld);
        bbase = j.B.p + (int64_t)j.n0 * j.B.ld;
#pragma unroll
        for (int i = 0; i < TM / 2; ++i) soa[i] = (unsigned)((int)a_row(j, wm * WM + i * 64 + lane) >> j.A.s_shift) * (unsigned)j.A.s_row;
#pragma unroll
        for (int i = 0; i < TN / 2; ++i) sob[i] = (unsigned)(min(j.n0 + wn * WN + i * 64 + lane, j.B.ext - 1) >> j.B.s_shift) * (unsigned)j.B.s_row;
        sabase = j.A.s;
        sbbase = j.B.s;
        sak = j.K > FP8_BK ? j.A.s_k : 0;         // (a contraction of one block has one scale)
        sbk = j.K > FP8_BK ? j.B.s_k : 0;
    }

    // First tile of a workgroup: its first two K-steps requested, the first landed and readable by everyone.  SHORT: the
    // contraction may be below 128.
    template <bool SHORT>
    FX_DEV void start(const Fp8Job<TD>& j, uint8_t* buf0, uint8_t* buf1) {
        setup(j);
        fetch_scales();
        issue(buf0);
        move(steps(j.K) == 2 ? -back(j.K) : 0);
        issue(buf1);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LD) : "memory");
        if constexpr (SHORT) {
            if (j.K < FP8_BK) patch(buf0, 0, j.K);
        }
        __syncthreads();
    }

    // The 32 k-values of this lane in tile row row0 + (lane & 31), sub-step ks: chunks c = 4 ks + 2 h and c + 1 of that row,
    // at positions c ^ swz(row).  lds_lane is the byte offset of chunk 2 h; the others differ from it in bits 4 and 6.
    // (row0 is a multiple of 32: swz(row0 + r) = swz(r).)
    FX_DEV i32x8_t read_frag(const uint8_t* tile, int row0, int ks) const {
        union { i32x8_t f; u32x4_t q[2]; } u;
        const unsigned o = lds_lane ^ (unsigned)(ks * 64);
        u.q[0] = *reinterpret_cast<const u32x4_t*>(tile + row0 * FP8_BK + o);
        u.q[1] = *reinterpret_cast<const u32x4_t*>(tile + row0 * FP8_BK + (o ^ 16u));
        return u.f;
    }
    template <int I, int P>
    FX_DEV void read_a(const uint8_t* buf, int ks) {
        const int row0 = (wave / WAVES_N) * WM + I * 32;
        if constexpr (I < TM - HI) alo[I] = read_frag(buf, row0, ks);
        else ahi[P][I - (TM - HI)] = read_frag(buf, row0, ks);
    }
    template <int J, int P>
    FX_DEV void read_b(const uint8_t* buf, int ks) {
        bf[P][J] = read_frag(buf + BM * FP8_BK, (wave % WAVES_N) * WN + J * 32, ks);
    }

    // MFMAs of the sub-step whose fragments are in register set P; with FETCH the fragments of sub-step ks_f in `buf`
    // are read into set 1 - P meanwhile.  after(IntC<M>) runs in the shadow of MFMA M.
    template <int P, bool FETCH, int M = 0, typename After>
    FX_DEV void sub(f32x16_t (&acc)[TM][TN], const uint8_t* buf, int ks_f, After&& after) {
        if constexpr (M < MFMAS) {
            constexpr int i = M / TN, j = M % TN, Q = 1 - P;
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (i < TM - HI) acc[i][j] = mfma_fp8<AF, j, i>(bf[P][j], alo[i], acc[i][j], scb, sca);
            else acc[i][j] = mfma_fp8<AF, j, i>(bf[P][j], ahi[P][i - (TM - HI)], acc[i][j], scb, sca);
            if constexpr (FETCH) {
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (TM == 4) {
                    if constexpr (M == 0) read_b<0, Q>(buf, ks_f);
                    if constexpr (M == 1) read_b<1, Q>(buf, ks_f);
                    if constexpr (M == 2) read_a<0, Q>(buf, ks_f);     // its last MFMA was M == 1
                    if constexpr (M == 3) read_a<2, Q>(buf, ks_f);
                    if constexpr (M == 4) read_a<1, Q>(buf, ks_f);     // its last MFMA was M == 3
                    if constexpr (M == 5) read_a<3, Q>(buf, ks_f);
                } else {
                    if constexpr (M == 0) read_b<0, Q>(buf, ks_f);
                    if constexpr (M == 1) { read_b<1, Q>(buf, ks_f); read_a<0, Q>(buf, ks_f); }
                    if constexpr (M == 2) read_a<1, Q>(buf, ks_f);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            after(IntC<M>());
            sub<P, FETCH, M + 1>(acc, buf, ks_f, after);
        } else {
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    struct Nothing { template <typename I> FX_DEV void operator()(I) const {} };

    // One K-step from `cur` whose successor, of which bytes [lo, hi) count, is in (or on its way to) `nxt`; the caller has called
    // fetch_scales() for the successor.  With MORE the K-step that the loader stands at is requested into `cur`.
    template <bool MORE, bool SHORT>
    FX_DEV void step(f32x16_t (&acc)[TM][TN], uint8_t* cur, uint8_t* nxt, int lo, int hi) {
        sub<0, true>(acc, cur, 1, Nothing());
        // every read of `cur` is out.  Once they and this wave's loads into `nxt` have landed, the barrier makes `nxt`
        // readable and `cur` writable for everyone; the second half's MFMAs run after it, while the first fragments
        // of the next K-step are read and the loads of the one after go out.
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        if constexpr (SHORT) {
            if (lo > 0 || hi < FP8_BK) patch(nxt, lo, hi);
        }
        __syncthreads();
        // packed here, where nothing is in flight: a use further down would wait for the tile loads issued since
        int na, nb;
        pack_scales(na, nb);
        sub<1, true>(acc, nxt, 0, [&](auto m) {
            constexpr int M = decltype(m)::value;
            if constexpr (MORE) static_for<M * PER, (M + 1) * PER>([&](auto i) { issue_one<decltype(i)::value>(cur); });
        });
        sca = na;
        scb = nb;
    }
    // The last K-step; with MORE the next tile's second K-step goes into `cur` once everyone has read it.
    template <bool MORE>
    FX_DEV void last_step(f32x16_t (&acc)[TM][TN], uint8_t* cur) {
        sub<0, true>(acc, cur, 1, Nothing());
        if constexpr (MORE) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __syncthreads();
        }
        sub<1, false>(acc, cur, 0, [&](auto m) {
            constexpr int M = decltype(m)::value;
            if constexpr (MORE) static_for<M * PER, (M + 1) * PER>([&](auto i) { issue_one<decltype(i)::value>(cur); });
        });
    }

    // K loop of tile `job` (K > 0), whose first K-step is readable in buf[par] and whose second is landed in or on its way
    // to buf[1 - par], scales of the first requested.  Leaves the (transposed) accumulators.
    // AHEAD: the stages go on without a gap into tile `next`: its first K-step is requested while the last but one of this
    // tile is multiplied, its second during the last, so both arrive under MFMAs and the epilogue; par moves on to where
    // its first K-step is.  (Behind a workgroup's last tile `next` is that tile again: a condition around MFMAs
    // would cost registers, two K-steps fetched for nothing cost nothing.)
    template <bool AHEAD>
    FX_DEV void run(const Fp8Job<TD>& job, const Fp8Job<TD>& next, uint8_t* buf0, uint8_t* buf1, int& par, f32x16_t (&acc)[TM][TN]) {
        const int wm = wave / WAVES_N, wn = wave % WAVES_N;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;
        const int K = job.K, n = steps(K);
        const int lo = back(K), hi = lo + K - (n - 1) * FP8_BK;         // what counts of the last step
        // wave-uniform: does any element of this wave's sub-tile exist?
        const bool live = __builtin_amdgcn_readfirstlane((job.m0 + wm * WM < job.A.ext) && (job.n0 + wn * WN < job.B.ext));
        const int p0 = par;
        par = (p0 + n) & 1;
        auto stage = [&](int kt) { return ((kt + p0) & 1) ? buf1 : buf0; };
        const int next_back = steps(next.K) == 2 ? back(next.K) : 0;
        if (live) {
            pack_scales(sca, scb);
            static_for<0, TN>([&](auto j) { read_b<decltype(j)::value, 0>(stage(0), 0); });
            static_for<0, TM>([&](auto i) { read_a<decltype(i)::value, 0>(stage(0), 0); });
            // straight-line K-steps: a branch between the MFMAs lets the compiler sink them all behind the loads
            for (int kt = 0; kt < n - 2; ++kt) {
                move(kt == n - 3 ? -lo : 0);
                fetch_scales();
                step<true, false>(acc, stage(kt), stage(kt + 1), 0, FP8_BK);
            }
            fetch_scales();
            if (AHEAD) setup(next);
            step<AHEAD, true>(acc, stage(n - 2), stage(n - 1), lo, hi);
            if (AHEAD) { move(-next_back); fetch_scales(); }
            last_step<AHEAD>(acc, stage(n - 1));
        } else {
            // this wave loads its share of the stages, meets every barrier of the other branch and leaves the matrix
            // pipe to the wave it shares a SIMD with
            for (int kt = 0; kt < n - 2; ++kt) {
                move(kt == n - 3 ? -lo : 0);
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
                issue(stage(kt));
            }
            if (AHEAD) setup(next);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (lo > 0 || hi < FP8_BK) patch(stage(n - 1), lo, hi);
            __syncthreads();
            if (AHEAD) {
                issue(stage(n - 2));
                move(-next_back);
                fetch_scales();
                __syncthreads();
                issue(stage(n - 1));
            }
        }
    }
};

// What the lanes of a wave have written to LDS, its other lanes may read from here on (and overwrite what was read).  The LDS
// serves a wave's accesses in their order, so this is no instruction: it keeps the compiler, which sees one lane's
// addresses, from exchanging them.
FX_DEV void wave_exchange() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// D (+ C) of one wave from its accumulators, a band of 32 rows at a time through 4 KB of LDS of its own (`st`), so that a
// load or store instruction of a wave covers eight whole 128-byte pieces of rows.
//   accumulator side  lane (r, h) = (lane % 32, lane / 32) holds of row 32 i + r the columns 32 j + 8 g + 4 h .. + 3
//                     (g = 0 .. 3); swapping the upper half-wave of group 2 q with the lower one of group 2 q + 1 leaves
//                     it 8 consecutive columns
//   memory side       lane l holds 16-byte chunk l % 8 of rows l / 8, l / 8 + 8, ..
// Chunk c of staged row r sits at c ^ ((r >> 1) & 7): 16 lanes of either side touch every bank once.  C comes in on the
// memory side (all bands of a 2-byte type requested at once), is added in fp32 on the accumulator side, and the sum is
// rounded once.  Straight 16-byte stores from the accumulator side (32 bytes of each of 32 rows per instruction) took
// 593 us for the expert weight gradients, which move 1.6 GB of C and D.
// LAND: before the first store, everything this wave has requested so far must have landed (loads and stores share one
// counter: a wait placed after the stores would also wait for them to drain).
// Rows of C and D may start at any address of their type (an output of 919 columns): the card takes 16-byte accesses there,
// and the element by element form is left to a row's last chunk (10736 x 5921 x 1723 202 -> 123 us, against 8 two-byte stores a chunk).
constexpr int FP8_STAGE_BYTES = 4096;      // per wave

template <typename TD, int TM, int TN, bool LAND, bool NT>
FX_DEV void fp8_epilogue(const f32x16_t (&acc)[TM][TN], const TD* C, int64_t ldc, TD* D, int64_t ldd, int row_base, int col_base,
                         int M, int N, uint8_t* st, int lane) {
    typedef typename VecOf<TD>::type Pack;
    static_assert(TN == 2, "a staged row holds 64 columns of a 2-byte type or 32 of a 4-byte one");
    constexpr int CE = VecOf<TD>::N;                         // values of a 16-byte chunk
    constexpr int JP = sizeof(TD) == 2 ? TN : 1, PASS = TN / JP;
    constexpr int CB = sizeof(TD) == 2 ? TM : (TM + 1) / 2;  // bands whose C is requested together
    const int r = lane & 31, h = lane >> 5, rr = lane >> 3, ch = lane & 7;
    typedef typename AnyPack<TD>::type Any;                  // rows of C and D start anywhere
    auto at = [&](int row, int c) { return reinterpret_cast<Pack*>(st + row * 128 + ((c ^ ((row >> 1) & 7)) << 4)); };
    Pack c[CB][PASS][4];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        if (C != nullptr && i % CB == 0) {
#pragma unroll
            for (int b = 0; b < CB; ++b)
#pragma unroll
                for (int s = 0; s < PASS; ++s)
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const int row = row_base + (i + b) * 32 + t * 8 + rr, col = col_base + s * 32 + ch * CE;
                        if (row < M) {
                            const TD* src = C + (int64_t)row * ldc + col;
                            if (col + CE <= N) {
                                c[b][s][t] = NT ? __builtin_nontemporal_load(reinterpret_cast<const Any*>(src)) : *reinterpret_cast<const Any*>(src);
                            } else {
#pragma unroll
                                for (int e = 0; e < CE; ++e)
                                    if (col + e < N) c[b][s][t][e] = src[e];
                            }
                        }
                    }
        }
        if (LAND && i == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int s = 0; s < PASS; ++s) {
            wave_exchange();          // the previous band has been read back before this one is staged
            if (C != nullptr) {
#pragma unroll
                for (int t = 0; t < 4; ++t) *at(t * 8 + rr, ch) = c[i % CB][s][t];
            }
            wave_exchange();
#pragma unroll
            for (int jj = 0; jj < JP; ++jj)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int j = s * JP + jj;
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float lo = acc[i][j][8 * q + e], hi = acc[i][j][8 * q + 4 + e];
                        const auto x = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, lo), __builtin_bit_cast(unsigned, hi), false, false);
                        v[e] = __builtin_bit_cast(float, (unsigned)x[0]);
                        v[4 + e] = __builtin_bit_cast(float, (unsigned)x[1]);
                    }
#pragma unroll
                    for (int u = 0; u < 8 / CE; ++u) {
                        Pack* p = at(r, jj * 4 + (q * 2 + h) * (8 / CE) + u);
                        Pack o;
                        if (C != nullptr) {
                            const Pack add = *p;
#pragma unroll
                            for (int e = 0; e < CE; ++e) v[u * CE + e] += (float)add[e];
                        }
#pragma unroll
                        for (int e = 0; e < CE; ++e) o[e] = (TD)v[u * CE + e];
                        *p = o;
                    }
                }
            wave_exchange();
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const Pack o = *at(t * 8 + rr, ch);
                const int row = row_base + i * 32 + t * 8 + rr, col = col_base + s * 32 + ch * CE;
                if (row < M && col < N) {
                    TD* d = D + (int64_t)row * ldd + col;
                    if (col + CE <= N) {
                        if (NT) __builtin_nontemporal_store((Any)o, reinterpret_cast<Any*>(d));
                        else *reinterpret_cast<Any*>(d) = o;
                    } else {
#pragma unroll
                        for (int e = 0; e < CE; ++e)
                            if (col + e < N) d[e] = o[e];
                    }
                }
            }
        }
    }
}

// ---------------------------------------------------------------- kernels over a list of tiles
// A Source names the tiles of a launch: total(lane) how many there are, locate(id, lane) where tile `id` lies (a small
// struct), locate_one(id, lane, where) the same without the total (false: no such tile), job(where) its operands.  Counts of experts are read by whole waves (find_group_tile), so every lane calls.

// 256 x 256 tiles, eight waves of 128 x 64, one workgroup per CU that walks the list with the grid as stride (Fp8Loop::run
// keeps its loads going over the tile boundaries).  LDS: two stages of 64 KB, and what the epilogue stages through.
// Bound by the matrix unit at the clock that power allows (8192 x 14336 x 4096 363 us, 2.65 PFLOP/s) while operands are in the
// caches, by their way from memory, one K-step ahead, when they are not (402 us).  Per tile about 1.4 us a K-step and 5.
constexpr int FP8_WALK_BM = 256, FP8_WALK_BN = 256;
constexpr size_t kFp8WalkStages = 128 * 1024, kFp8WalkLds = kFp8WalkStages + 8 * FP8_STAGE_BYTES;     // all 160 KB

// An output larger than the cache in front of the memory goes past it (NT; C as well), so that the operands keep their place:
// weight gradients of 128 experts, 805 MB, 558 -> 517 us.  Smaller ones stay in it for their reader and lose by passing it
// (8192 x 8192 x 8192, 134 MB: 387 -> 402 us; 8192 x 14336 x 4096, 235 MB: 363 -> 375 us).
constexpr size_t kFp8OnceBytes = (size_t)256 << 20;

// A tile whose contraction is empty: C (nothing to do where D is C), or zeros.  16 bytes a lane, all of C requested before the
// first store: 93 experts of 720 x 280, 8 of them with a row, 116 us element by element, 27 like this.
template <typename TD, int BM, int BN, int NT>
FX_DEV void fp8_empty_tile(const Fp8Job<TD>& j, int64_t ldc, int64_t ldd) {
    if (j.C == j.D && ldc == ldd) return;
    typedef typename AnyPack<TD>::type Any;
    constexpr int CE = 16 / (int)sizeof(TD), ROW = BN / CE, STEP = NT / ROW, BATCH = 8;
    static_assert(NT % ROW == 0 && BM % (STEP * BATCH) == 0, "whole batches");
    const int col = j.n0 + (threadIdx.x % ROW) * CE, row0 = j.m0 + threadIdx.x / ROW;
    const bool whole = col + CE <= j.B.ext;
    for (int r = 0; r < BM; r += STEP * BATCH) {
        Any v[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
            const int64_t row = row0 + r + u * STEP;
#pragma unroll
            for (int e = 0; e < CE; ++e) v[u][e] = (TD)0.f;
            if (j.C != nullptr && row < j.A.ext && whole) v[u] = *reinterpret_cast<const Any*>(j.C + row * ldc + col);
        }
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
            const int64_t row = row0 + r + u * STEP;
            if (row >= j.A.ext) continue;
            if (whole) {
                *reinterpret_cast<Any*>(j.D + row * ldd + col) = v[u];
            } else {
                for (int e = 0; col + e < j.B.ext; ++e) j.D[row * ldd + col + e] = j.C != nullptr ? j.C[row * ldc + col + e] : (TD)0.f;
            }
        }
    }
}

template <int AF, typename TD, bool NT, typename Source>
__global__ __launch_bounds__(512) void fp8_walk_kernel(Source src) {
    extern __shared__ __align__(16) unsigned char smem[];
    typedef Fp8Loop<AF, TD, FP8_WALK_BM, FP8_WALK_BN, 2, 4> Loop;
    static_assert(2 * Loop::STAGE == (int)kFp8WalkStages, "two stages");
    uint8_t *buf0 = smem, *buf1 = smem + Loop::STAGE;
    Loop loop;
    loop.init();
    const int total = src.total(loop.lane);
    // the next tile from `id` on that has a contraction; those without are written on the way
    auto find = [&](int& id, typename Source::Where& w) {
        for (; id < total; id += (int)gridDim.x) {
            w = src.locate(id, total, loop.lane);
            const Fp8Job<TD> j = src.job(w);
            if (j.K > 0) return true;
            fp8_empty_tile<TD, FP8_WALK_BM, FP8_WALK_BN, 512>(j, src.ldc, src.ldd);
        }
        return false;
    };
    int id = blockIdx.x;
    typename Source::Where cur;
    if (!find(id, cur)) return;
    loop.template start<false>(src.job(cur), buf0, buf1);
    int par = 0;
    for (;;) {
        typename Source::Where nxt = cur;
        id += (int)gridDim.x;
        const bool more = find(id, nxt);
        if (!more) nxt = cur;
        f32x16_t acc[Loop::TM][Loop::TN];
        loop.template run<true>(src.job(cur), src.job(nxt), buf0, buf1, par, acc);
        const Fp8Job<TD> j = src.job(cur);
        fp8_epilogue<TD, Loop::TM, Loop::TN, true, NT>(acc, j.C, src.ldc, j.D, src.ldd, j.m0 + (loop.wave / 4) * Loop::WM,
                                                   j.n0 + (loop.wave % 4) * Loop::WN, j.A.ext, j.B.ext,
                                                   smem + kFp8WalkStages + loop.wave * FP8_STAGE_BYTES, loop.lane);
        if (!more) break;
        __syncthreads();          // everyone's share of the next tile's first K-steps has landed
        cur = nxt;
    }
}

// 128 x 128 tiles, four waves of 64 x 64, one tile per workgroup; 80 KB of LDS, so two workgroups share a CU and one's
// epilogue and first loads run under the other's K loop.  Bound by the latency of a K-step's loads (0.6 us alone on its CU):
// 512 x 4096 x 4096 24 us, 2048 x 2048 x 2048 16 us.
constexpr size_t kFp8Tile128Stages = 64 * 1024, kFp8Tile128Lds = kFp8Tile128Stages + 4 * FP8_STAGE_BYTES;

template <int AF, typename TD, typename Source>
__global__ __launch_bounds__(256, 2) void fp8_tile_kernel128(Source src) {
    extern __shared__ __align__(16) unsigned char smem[];
    typedef Fp8Loop<AF, TD, 128, 128, 2, 2> Loop;
    static_assert(2 * Loop::STAGE == (int)kFp8Tile128Stages, "two stages");
    Loop loop;
    loop.init();
    const int total = src.total(loop.lane);
    if ((int)blockIdx.x >= total) return;
    const Fp8Job<TD> j = src.job(src.locate(blockIdx.x, total, loop.lane));
    if (j.K == 0) {
        fp8_empty_tile<TD, 128, 128, 256>(j, src.ldc, src.ldd);
        return;
    }
    loop.template start<true>(j, smem, smem + Loop::STAGE);
    f32x16_t acc[Loop::TM][Loop::TN];
    int par = 0;
    loop.template run<false>(j, j, smem, smem + Loop::STAGE, par, acc);
    fp8_epilogue<TD, Loop::TM, Loop::TN, false, false>(acc, j.C, src.ldc, j.D, src.ldd, j.m0 + (loop.wave / 2) * Loop::WM,
                                                j.n0 + (loop.wave % 2) * Loop::WN, j.A.ext, j.B.ext,
                                                smem + kFp8Tile128Stages + loop.wave * FP8_STAGE_BYTES, loop.lane);
}

// Small products: one workgroup per tile of 16 MT x 16 NT, its NW waves share the contraction (wave w takes K-steps
// w, w + NW, ..) and add up through LDS in ascending order.  Operands go straight from memory into registers: with
// few rows nothing is used twice by a workgroup, so LDS staging and its barriers would only add latency, and with one
// launch and one pass a single token costs the weight's bytes (1 x 14336 x 4096 11.1 us, 5.3 TB/s).  The matrix instruction is the 16 x 16 x 128 one.
// A lane takes bytes [16 h, 16 h + 16) and [64 + 16 h, ..) of its row's 128 (h = lane / 16), so one load instruction
// of a wave covers 64 contiguous bytes of each of 16 rows; A and B use the same order of k, which is all that matters.
typedef float f32x4v_t __attribute__((ext_vector_type(4)));

template <int AF>
FX_DEV f32x4v_t mfma_fp8_16(const i32x8_t& b, const i32x8_t& a, f32x4v_t c, int sb, int sa) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, c, 0, AF == DT_E4M3 ? 0 : 1, 0, sb, 0, sa);
}

template <int AF, typename TD, int MT, int NT, int NW, int U, typename Source>
__global__ __launch_bounds__(NW * 64) void fp8_small_kernel(Source src) {
    __shared__ f32x4v_t red[NW][MT * NT][64];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    typename Source::Where where;
    if (!src.locate_one(blockIdx.x, lane, where)) return;
    const Fp8Job<TD> j = src.job(where);
    const int r = lane & 15, h = lane >> 4;
    const uint8_t *pa[MT], *pb[NT], *sa[MT], *sb[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int g = min(j.m0 + i * 16 + r, j.A.ext - 1);
        const int row = j.row_map != nullptr ? min(max(j.row_map[g], 0), j.src_rows - 1) : g;
        pa[i] = j.A.p + (int64_t)row * j.A.ld + h * 16;
        sa[i] = j.A.s + (int64_t)(row >> j.A.s_shift) * j.A.s_row;
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int row = min(j.n0 + i * 16 + r, j.B.ext - 1);
        pb[i] = j.B.p + (int64_t)row * j.B.ld + h * 16;
        sb[i] = j.B.s + (int64_t)(row >> j.B.s_shift) * j.B.s_row;
    }
    f32x4v_t acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[i][n] = f32x4v_t{0.f, 0.f, 0.f, 0.f};
    union Frag { i32x8_t f; u32x4_t q[2]; };
    const int K = j.K, nfull = K / FP8_BK;
    auto load = [&](Frag (&fa)[MT], Frag (&fb)[NT], int (&ca)[MT], int (&cb)[NT], int kb) {
        const int64_t k = (int64_t)kb * FP8_BK;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            fb[n].q[0] = ldg16(pb[n] + k);
            fb[n].q[1] = ldg16(pb[n] + k + 64);
            cb[n] = sb[n][(int64_t)kb * j.B.s_k];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            fa[i].q[0] = ldg16(pa[i] + k);
            fa[i].q[1] = ldg16(pa[i] + k + 64);
            ca[i] = sa[i][(int64_t)kb * j.A.s_k];
        }
    };
    auto multiply = [&](const Frag (&fa)[MT], const Frag (&fb)[NT], const int (&ca)[MT], const int (&cb)[NT]) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[i][n] = mfma_fp8_16<AF>(fb[n].f, fa[i].f, acc[i][n], cb[n], ca[i]);
    };
    Frag fa[U][MT], fb[U][NT];
    int ca[U][MT], cb[U][NT];
    int kb = wave;
    for (; kb + (U - 1) * NW < nfull; kb += U * NW) {       // U K-steps in flight
#pragma unroll
        for (int u = 0; u < U; ++u) load(fa[u], fb[u], ca[u], cb[u], kb + u * NW);
#pragma unroll
        for (int u = 0; u < U; ++u) multiply(fa[u], fb[u], ca[u], cb[u]);
    }
#pragma unroll
    for (int u = 0; u < U - 1; ++u)
        if (kb + u * NW < nfull) load(fa[u], fb[u], ca[u], cb[u], kb + u * NW);
#pragma unroll
    for (int u = 0; u < U - 1; ++u)
        if (kb + u * NW < nfull) multiply(fa[u], fb[u], ca[u], cb[u]);
    if (nfull * FP8_BK < K && nfull % NW == wave) {         // last partial K-step: zero behind K
        const int k = nfull * FP8_BK;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            fb[0][n].q[0] = load_chunk(pb[n] - h * 16, k + h * 16, K);
            fb[0][n].q[1] = load_chunk(pb[n] - h * 16, k + 64 + h * 16, K);
            cb[0][n] = sb[n][(int64_t)nfull * j.B.s_k];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            fa[0][i].q[0] = load_chunk(pa[i] - h * 16, k + h * 16, K);
            fa[0][i].q[1] = load_chunk(pa[i] - h * 16, k + 64 + h * 16, K);
            ca[0][i] = sa[i][(int64_t)nfull * j.A.s_k];
        }
        multiply(fa[0], fb[0], ca[0], cb[0]);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) red[wave][i * NT + n][lane] = acc[i][n];
    __syncthreads();
    // lane holds D[m = lane % 16][n = 4 (lane / 16) .. + 3] of a 16 x 16 block; wave t % NW finishes block t
    for (int t = wave; t < MT * NT; t += NW) {
        f32x4v_t s = red[0][t][lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) s += red[w][t][lane];
        const int m = j.m0 + (t / NT) * 16 + r, n = j.n0 + (t % NT) * 16 + h * 4;
        if (m >= j.A.ext) continue;
        typedef TD t4_t __attribute__((ext_vector_type(4), aligned(sizeof(TD))));       // (rows start anywhere)
        TD* d = j.D + (int64_t)m * src.ldd + n;
        const TD* c = j.C != nullptr ? j.C + (int64_t)m * src.ldc + n : nullptr;
        if (n + 4 <= j.B.ext) {
            if (c != nullptr) {
                const t4_t cv = *reinterpret_cast<const t4_t*>(c);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[e] += (float)cv[e];
            }
            const t4_t o = {(TD)s[0], (TD)s[1], (TD)s[2], (TD)s[3]};
            *reinterpret_cast<t4_t*>(d) = o;
        } else {
            for (int e = 0; e < 4 && n + e < j.B.ext; ++e) d[e] = (TD)(c != nullptr ? s[e] + (float)c[e] : s[e]);
        }
    }
}

// ---------------------------------------------------------------- which kernel
// Times in microseconds, fitted to sweeps of M in 1 .. 2048, N and K in 1000 .. 14336 (dense) and of 8 .. 65536 rows over
// 128 experts.  They are for choosing, and good to a factor of 1.5 either way, not better: over 241 dense products (M 16 ..
// 6373, N 128 .. 14336, K 256 .. 11915) the measured time is 0.76 to 1.51 of the fit in nine of ten, within 15 % in 60 of 100;
// over 179 by expert (8 .. 128 experts of 1 .. 512 rows on average) 0.85 to 1.49, within 15 % in 44 of 100.  Operands that the
// caches do not hold (6373 x 344 x 11915: 84 measured, 52 fitted; 333 x 14336 x 11915: 122, 72) and 128-row tiles at two
// and more to a CU are slower than fitted, the smallest launches faster.  What the choice costs against the fastest of the three
// forms: nothing in half of the dense products, up to 6 % in nine of ten, at worst 1.6 times (333 x 579 x 256: 6.0 us in 128 x 128
// tiles, 3.7 small; 1024 x 579 x 4096: 25.6 small, 19.1 in tiles); by expert up to 9 % in nine of ten, at worst 1.5
// times (32 experts of 128 rows, N 2048, K 768: 29.9 us in 256-row tiles, 19.6 in 128-row ones: the rows are not split evenly).
//   small   4 + max(1, workgroups / 256) * steps * (MT + NT) * 0.05 + 5 for every million outputs      a CU takes in 40 KB of
//           operands per us; its stores are 8 bytes a lane
//   128     4 + steps * 0.62 up to one workgroup per CU, 0.95 at two, then steps * 1.1 + 3 for every further 512
//   256     4 + rounds of 256 * (steps * 1.5 + 5)
// steps: 128-long K-steps.  Examples (measured): 64 x 4096 x 4096 small 2 x 2 10.2, 128 15.4; 512 x 4096 x 4096 small 32.9,
// 128 23.9, 256 41.5; 1024 x 14336 x 4096 128 76.6, 256 59.4.
struct Fp8Small { int mt, nt; };
constexpr Fp8Small kFp8Small[] = {{1, 1}, {1, 2}, {1, 4}, {2, 2}, {2, 4}, {4, 2}, {4, 4}};
constexpr int kFp8Smalls = sizeof(kFp8Small) / sizeof(kFp8Small[0]);

static inline double fp8_time_small(const Fp8Small& c, double tiles_m, double rows, int N, int steps) {
    const double w = tiles_m * (double)((N + 16 * c.nt - 1) / (16 * c.nt)) / 256.0;
    return 4.0 + (w > 1.0 ? w : 1.0) * steps * (c.mt + c.nt) * 0.05 + rows * (double)N * 5e-6;
}
static inline double fp8_time_128(double workgroups, double steps) {
    if (workgroups <= 256.0) return 4.0 + steps * 0.62;
    if (workgroups <= 512.0) return 4.0 + steps * (0.62 + 0.33 * (workgroups / 256.0 - 1.0));
    return 4.0 + ceil(workgroups / 512.0) * (steps * 1.1 + 3.0);
}
static inline double fp8_time_256(double tiles, double steps) { return 4.0 + ceil(tiles / 256.0) * (steps * 1.5 + 5.0); }

// Waves that share a tile's contraction (4 or 8) and K-steps each has in flight (1, 2 or 4) in the small kernel.  Few operands per step
// leave registers for more of them in flight; the 64 KB of sums of a 4 x 4 tile leave room for 4 waves.  Measured over the
// products for which a tile is within 25 % of the fastest (M 1 .. 1000, N 579 .. 14336, K 1000 .. 4096; 8 x 2: 8 waves, 2 in
// flight), the other settings against the one taken, on average: 1 x 1 (8 x 4) 0.97 .. 1.01;  1 x 2 (8 x 2) 1.02 .. 1.11;
// 1 x 4 (8 x 2) 1.00 .. 1.08;  2 x 2 (4 x 2) 0.98 .. 1.24;  2 x 4 (4 x 2) 0.98 .. 1.41;  4 x 2 (8 x 1) 0.99 .. 1.38;
// 4 x 4 (4 x 1) 1.24.
template <int MT, int NT> struct Fp8SmallShape { static constexpr int NW = (MT == 2 || NT * MT == 16) ? 4 : 8, U = MT * NT == 1 ? 4 : MT == 4 ? 1 : 2; };

static inline int fp8_cdiv(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// One workgroup per CU for the kernels that walk their tiles.
static inline int fp8_walk_grid() {
    int dev = 0, n = 0;
    (void)hipGetDevice(&dev);
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    return n;
}

// Bytes a scale tensor spans (0: none), and whether lane offsets of 32 bits cover an operand.
static inline bool fp8_scales_fit(int64_t rows, int64_t s_row, int64_t blocks, int64_t s_k) {
    if (rows <= 0 || blocks <= 0) return true;
    if (s_row < 0 || s_k < 0) return false;
    const double span = (double)(rows - 1) * (double)s_row + (double)(blocks - 1) * (double)s_k;
    return span < 2147483647.0;
}
constexpr int64_t kFp8MaxLd = (int64_t)1 << 23;
constexpr int kFp8MaxExtent = 0x7fffffff - 512;      // a row number behind an edge tile stays an int

// Rows of an operand start at 16-byte addresses.
static inline bool fp8_bad_rows(const void* p, int64_t ld) { return !aligned16(p) || (ld & 15) != 0; }

}  // namespace fx
