// Residual addition + RMSNorm with the output in 8 bits (or in the input's type), gfx950.
//
//   h = T(x + residual)      rstd = (mean(h^2) + eps)^-1/2      y = h * rstd * w
//   (q, s) = y in blocks of 1 x 128 (fp8.h), or y rounded to T
//
// One pass: a row stays in registers from its load to its last store, so x and residual are read once, h and
// the 8-bit row written once (7 bytes an element for 2-byte types; a norm followed by a quantiser moves 11).
// The sum h is rounded to T before anything uses it: the backward pass starts from the stored h, and the
// statistics must be those of the row it sees.  With an 8-bit output y is NOT rounded to T on the way (one
// rounding, from the exact value); with output type T the product is rounded as flextrain_rmsnorm_fwd rounds it
// (T(h * rstd) * w): the same rstd as that op on h where it takes its vector kernel (ncols % 8 == 0, at most 16384, 16-byte
// addresses; its other kernel adds the squares in another order), and the same y in bf16 and fp32.  In fp16 the compiler
// turns a product and its conversion into one v_fma_mix, which rounds once, in some places of either kernel and not in
// others: with a weight up to 5 values of 100,000 are a step apart.
// Thread mapping: that of rmsnorm.hip (LPR lanes a row, pack v of lane l holds columns (v * LPR + l) * 8 .. + 7),
// so the 128 columns of a block lie in one pack of 16 consecutive lanes.
// Bound by memory: 8192 x 4096 bf16 with a residual 51 us, 4.6 TB/s; one row 4 us, which is latency.
#include "fp8.h"
#include "flexhip.h"

namespace fx {

enum : int { OUT_SAME = -1 };      // output in the input's type; otherwise DT_E4M3 / DT_E5M2

FX_DEV float norm_w1(const void* w, int w_dt, int64_t c) {
    return w_dt == DT_F32 ? reinterpret_cast<const float*>(w)[c]
           : w_dt == DT_BF16 ? (float)reinterpret_cast<const bf16*>(w)[c] : (float)reinterpret_cast<const f16*>(w)[c];
}
// With an 8-bit output every value is that of the exact y, rounded once: the statistics are 64-bit, and y = h * rstd * w comes as a
// sum of two fp32 numbers.  (An fp32 y that is off by an ulp falls on the wrong side of the middle between two 8-bit values once
// in a few million, so that two programs which add a row's squares in another order differ by whole steps of 2^-3 there.)
// 8192 x 4096 bf16 take 45 us in fp32, 51 like this and 55 with 64-bit products.  eps comes in 64 bits too: 1e-5 rounded to fp32
// moves rstd by 6e-9 where the mean square is as small as that.  An output in the input's type keeps the fp32 arithmetic
// (eps with it) of flextrain_rmsnorm_fwd.
template <int OUT> struct NormMath { typedef double type; };
template <> struct NormMath<OUT_SAME> { typedef float type; };

template <int W>
FX_DEV double group_sum(double v) {
#pragma unroll
    for (int off = W / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}
FX_DEV float mean_of(float ss, int n, double) { return ss / (float)n; }
FX_DEV double mean_of(double ss, int, double inv_n) { return ss * inv_n; }
FX_DEV float inverse_root(float m) { return rsqrtf(m); }
// The instruction's estimate (22 bits or more) and two Newton steps; 0 and infinity have none.
FX_DEV double inverse_root(double m) {
    double r = __builtin_amdgcn_rsq(m);
    if (m > 0.0 && m < __builtin_huge_val()) {
        r = r * (1.5 - 0.5 * m * r * r);
        r = r * (1.5 - 0.5 * m * r * r);
    }
    return r;
}
// h * (hi + lo) * w to fp32 by rounding to odd (Boldo and Melquiond, IEEE Trans. Computers 57, 2008): of the two neighbours of
// a value between them the one whose last bit is 1.  It lies on the same side of every 8-bit value, and of every middle
// between two, as the value itself, so rounding it again gives what rounding the value gives.  Products and their
// remainders by fma: off by 2^-45 of the value or less (while it is far from fp32's subnormals).
FX_DEV float product_odd(float h, float hi, float lo, float w) {
#pragma clang fp contract(off)
    const float p = h * hi, pe = fmaf(h, lo, fmaf(h, hi, -p));
    const float y = p * w, ye = fmaf(pe, w, fmaf(p, w, -y));
    const float s = y + ye, t = (y - s) + ye;
    unsigned b = __builtin_bit_cast(unsigned, s);
    const unsigned other = (b ^ __builtin_bit_cast(unsigned, t)) >> 31;          // 1: the value is nearer to 0 than s
    if (t != 0.f && (b & 1u) == 0u) b += 1u - 2u * other;
    return finite_mag(y) == 0u ? y : __builtin_bit_cast(float, b);               // (0, infinite, NaN)
}
FX_DEV float low_part(float, float) { return 0.f; }
FX_DEV float low_part(double r, float hi) { return hi > 0.f && hi < __builtin_huge_valf() ? (float)(r - (double)hi) : 0.f; }
template <typename T, int OUT>
FX_DEV float normed(float h, float hi, float lo, float w, bool has_w) {
    if constexpr (OUT != OUT_SAME) return product_odd(h, hi, lo, has_w ? w : 1.f);
    else return has_w ? round_to<T>(h * hi) * w : h * hi;
}

template <typename T, int LPR, int MAXV, int OUT, bool TAIL>
__global__ __launch_bounds__(256) void add_rmsnorm_kernel(const T* X, const T* R, const void* __restrict__ W, int w_dt,
                                                          T* H /* may alias X or R */, void* Y, int64_t ldy,
                                                          uint8_t* __restrict__ S, int64_t lds, float* __restrict__ RSTD,
                                                          int64_t rows, int ncols, double inv_n, typename NormMath<OUT>::type eps) {
    constexpr int G = 256 / LPR;
    typedef typename NormMath<OUT>::type M;
    __shared__ M red[4];
    const int tid = threadIdx.x, g = tid / LPR, l = tid % LPR;
    const int64_t row = (int64_t)blockIdx.x * G + g;
    const bool row_ok = row < rows;
    const bool has_w = W != nullptr;
    float h[MAXV][8], w[MAXV][8];
    M ss = 0;
#pragma unroll
    for (int v = 0; v < MAXV; ++v) {
        const int col = (v * LPR + l) * 8;
        if (row_ok && col < ncols) {
            row_load8<TAIL>(X + row * ncols + col, ncols - col, h[v]);
            if (R != nullptr) {
                float r[8];
                row_load8<TAIL>(R + row * ncols + col, ncols - col, r);
#pragma unroll
                for (int j = 0; j < 8; ++j) h[v][j] = round_to<T>(h[v][j] + r[j]);
            }
            if (has_w) row_w8<TAIL>(W, w_dt, col, ncols - col, w[v]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) h[v][j] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += (M)h[v][j] * (M)h[v][j];
    }
    if constexpr (LPR <= 64) {
        ss = group_sum<LPR>(ss);
    } else {
        ss = group_sum<64>(ss);
        if ((tid & 63) == 0) red[tid >> 6] = ss;
        __syncthreads();
        ss = (red[0] + red[1]) + (red[2] + red[3]);
    }
    const M rstd = inverse_root(mean_of(ss, ncols, inv_n) + eps);
    const float hi = (float)rstd, lo = low_part(rstd, hi);
    if (row_ok && l == 0) RSTD[row] = hi;
#pragma unroll
    for (int v = 0; v < MAXV; ++v) {
        const int col = (v * LPR + l) * 8;
        const bool ok = row_ok && col < ncols;
        if (ok && H != nullptr) row_store8<TAIL>(H + row * ncols + col, ncols - col, h[v]);
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = ok && (!TAIL || col + j < ncols) ? normed<T, OUT>(h[v][j], hi, lo, w[v][j], has_w) : 0.f;
        if constexpr (OUT == OUT_SAME) {
            if (ok) row_store8<TAIL>(reinterpret_cast<T*>(Y) + row * ldy + col, ncols - col, y);
        } else {
            unsigned m = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, finite_mag(y[j]));
            const int b = scale_byte<OUT>(row16_umax(m));
            const float inv = inverse_scale(b);
            if (row_ok && col < ldy) {
                uint2 o;
                o.x = pack_fp8x4<OUT>(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
                o.y = pack_fp8x4<OUT>(y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv);
                *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(Y) + row * ldy + col) = o;
                if ((l & 15) == 0 && col < ncols) S[(col >> 7) * lds + row] = (uint8_t)b;
            }
        }
    }
}

// Rows longer than registers hold (16384): one workgroup per row.  h is formed twice (for the statistics and for the output)
// from x and residual, element by element by the lane that later overwrites it, so H may alias either.
template <typename T, int OUT>
__global__ __launch_bounds__(256) void add_rmsnorm_generic_kernel(const T* X, const T* R, const void* __restrict__ W, int w_dt,
                                                                  T* H, void* Y, int64_t ldy, uint8_t* __restrict__ S, int64_t lds,
                                                                  float* __restrict__ RSTD, int64_t rows, int ncols, double inv_n,
                                                                  typename NormMath<OUT>::type eps) {
    typedef typename NormMath<OUT>::type M;
    __shared__ M red[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x;
    const T* x = X + row * ncols;
    const T* r = R ? R + row * ncols : nullptr;
    // wave w takes blocks w, w + 4, ... of 128 columns; a lane the columns lane and lane + 64 of a block
    const int blocks = (ncols + 127) / 128;
    auto sum_at = [&](int c) { return r ? round_to<T>((float)x[c] + (float)r[c]) : (float)x[c]; };
    M ss = 0;
    for (int b = wave; b < blocks; b += 4)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int c = b * 128 + u * 64 + lane;
            if (c < ncols) {
                const M v = sum_at(c);
                ss += v * v;
            }
        }
    ss = group_sum<64>(ss);
    if (lane == 0) red[wave] = ss;
    __syncthreads();
    const M rstd = inverse_root(mean_of((red[0] + red[1]) + (red[2] + red[3]), ncols, inv_n) + eps);
    const float hi = (float)rstd, lo = low_part(rstd, hi);
    if (tid == 0) RSTD[row] = hi;
    for (int b = wave; b < blocks; b += 4) {
        float y[2];
        unsigned m = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int c = b * 128 + u * 64 + lane;
            y[u] = 0.f;
            if (c < ncols) {
                const float v = sum_at(c);
                y[u] = normed<T, OUT>(v, hi, lo, W ? norm_w1(W, w_dt, c) : 1.f, W != nullptr);
                if (H != nullptr) H[row * ncols + c] = (T)v;
                m = max(m, finite_mag(y[u]));
                if constexpr (OUT == OUT_SAME) reinterpret_cast<T*>(Y)[row * ldy + c] = (T)y[u];
            }
        }
        if constexpr (OUT != OUT_SAME) {
            const int sb = scale_byte<OUT>(group_umax<64>(m));
            const float inv = inverse_scale(sb);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int c = b * 128 + u * 64 + lane;
                if (c < ldy) reinterpret_cast<uint8_t*>(Y)[row * ldy + c] = (uint8_t)pack_fp8x4<OUT>(y[u] * inv, 0.f, 0.f, 0.f);
            }
            if (lane == 0) S[b * lds + row] = (uint8_t)sb;
        }
    }
}

template <typename T, int OUT>
static void launch_add_rmsnorm(const void* x, const void* r, const void* w, int w_dt, void* h, void* y, int64_t ldy, void* s,
                               int64_t lds, float* rstd, int64_t rows, int ncols, double eps, hipStream_t stream) {
    const T *X = (const T*)x, *R = (const T*)r;
    T* H = (T*)h;
#define GO_TAIL(L, V, TAIL_)                                                                                         \
    add_rmsnorm_kernel<T, L, V, OUT, TAIL_><<<dim3((unsigned)((rows + 256 / L - 1) / (256 / L))), 256, 0, stream>>>( \
        X, R, w, w_dt, H, y, ldy, (uint8_t*)s, lds, rstd, rows, ncols, 1.0 / ncols, (typename NormMath<OUT>::type)eps)
#define GO(L, V)                                                                                                     \
    do {                                                                                                             \
        if (ncols % 8) GO_TAIL(L, V, true);                                                                          \
        else GO_TAIL(L, V, false);                                                                                   \
    } while (0)
    if (ncols > 16384)
        add_rmsnorm_generic_kernel<T, OUT><<<dim3((unsigned)rows), 256, 0, stream>>>(X, R, w, w_dt, H, y, ldy, (uint8_t*)s, lds, rstd, rows, ncols, 1.0 / ncols, (typename NormMath<OUT>::type)eps);
    else if (ncols <= 128) GO(16, 1);
    else if (ncols <= 256) GO(32, 1);
    else if (ncols <= 512) GO(64, 1);
    else if (ncols <= 1024) GO(64, 2);
    else if (ncols <= 2048) GO(256, 1);
    else if (ncols <= 4096) GO(256, 2);
    else if (ncols <= 8192) GO(256, 4);
    else GO(256, 8);
#undef GO
#undef GO_TAIL
}

}  // namespace fx

using namespace fx;

extern "C" int fx_add_rmsnorm_fwd(const void* x, const void* residual, const void* w, void* h, void* y, int64_t ldy, void* s,
                                  int64_t lds, float* rstd, int64_t rows, int ncols, double eps, int x_dt, int w_dt, int y_dt,
                                  hipStream_t stream) {
    if (rows < 0 || ncols <= 0) FX_FAIL("fx_add_rmsnorm_fwd: bad shape rows=%lld ncols=%d", (long long)rows, ncols);
    if (x_dt != DT_F32 && x_dt != DT_F16 && x_dt != DT_BF16) FX_FAIL("fx_add_rmsnorm_fwd: unsupported dtype enum %d", x_dt);
    if (w && w_dt != DT_F32 && w_dt != DT_F16 && w_dt != DT_BF16) FX_FAIL("fx_add_rmsnorm_fwd: unsupported weight dtype enum %d", w_dt);
    if (y_dt != x_dt && !is_fp8_dt(y_dt)) FX_FAIL("fx_add_rmsnorm_fwd: the output has the input's dtype or an 8-bit one");
    if (rows > 0xffffff) FX_FAIL("fx_add_rmsnorm_fwd: too many rows");      // (a launch has 2^32 threads at most)
    if (rows == 0) return 0;
    if (!x || !y || !rstd || (is_fp8_dt(y_dt) && !s) || (residual && !h)) FX_FAIL("fx_add_rmsnorm_fwd: null pointer");
    if (is_fp8_dt(y_dt)) {
        if ((ldy & 15) || ldy < ncols || ldy - ncols >= 16 || !aligned16(y) || lds < rows)
            FX_FAIL("fx_add_rmsnorm_fwd: 8-bit rows start at 16-byte addresses, padded to the next multiple of 16, with a scale stride of at least the rows");
    } else if (ldy != ncols) {
        FX_FAIL("fx_add_rmsnorm_fwd: an output in the input's dtype is contiguous");
    }
    FX_DISPATCH_DTYPE(x_dt, T, {
        if (y_dt == DT_E4M3) launch_add_rmsnorm<T, DT_E4M3>(x, residual, w, w_dt, h, y, ldy, s, lds, rstd, rows, ncols, eps, stream);
        else if (y_dt == DT_E5M2) launch_add_rmsnorm<T, DT_E5M2>(x, residual, w, w_dt, h, y, ldy, s, lds, rstd, rows, ncols, eps, stream);
        else launch_add_rmsnorm<T, OUT_SAME>(x, residual, w, w_dt, h, y, ldy, s, lds, rstd, rows, ncols, eps, stream);
    });
    FX_CHECK_LAUNCH("fx_add_rmsnorm_fwd");
    return 0;
}
