// Host stand-in for <hip/hip_runtime.h>: the device code of this package's non-MFMA kernels compiled as
// ordinary C++ and run on the CPU, one workgroup at a time, every GPU lane a cooperative fiber.
//
// What it is for: running the real kernel source (and the real host-side launch code: grid sizes, kernel
// selection, workspace use) against buffers that end at inaccessible guard pages, so that an access one
// element outside any operand kills the test, and comparing results with the CPU oracle.  Test
// infrastructure only: nothing in the package includes it.
//
// Execution model: a launch runs its workgroups in order; a workgroup's lanes are fibers that
// run until they meet a workgroup barrier, a wave-level exchange or their end.  __syncthreads() releases
// when every lane still alive has arrived; wave operations exchange through one slot per lane.  Lanes
// that returned count as arrived (on the GPU their wave either left the barrier's count or carries them
// masked off).  __shared__ variables are statics: one workgroup exists at a time.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <vector>

#include <malloc.h>

#define __global__
#define __device__
#define __host__
#define __forceinline__ inline
#define __launch_bounds__(...)
#define __shared__ static
#define __align__(n) __attribute__((aligned(n)))
#define HIP_SYMBOL(x) (&(x))

using std::max;
using std::min;

struct dim3 {
    unsigned x, y, z;
    dim3(unsigned a = 1, unsigned b = 1, unsigned c = 1) : x(a), y(b), z(c) {}
};
struct alignas(16) float4 { float x, y, z, w; };
struct alignas(8) float2 { float x, y; };
struct alignas(16) int4 { int x, y, z, w; };
struct alignas(8) uint2 { unsigned x, y; };
struct alignas(16) uint4 { unsigned x, y, z, w; };
inline float4 make_float4(float x, float y, float z, float w) { return float4{x, y, z, w}; }
inline float2 make_float2(float x, float y) { return float2{x, y}; }
inline uint2 make_uint2(unsigned x, unsigned y) { return uint2{x, y}; }
typedef void* hipStream_t;
typedef int hipError_t;
enum { hipSuccess = 0, hipErrorInvalidValue = 1 };
enum { hipFuncAttributeMaxDynamicSharedMemorySize = 8, hipDeviceAttributeMultiprocessorCount = 63 };
inline hipError_t hipGetLastError() { return hipSuccess; }
inline const char* hipGetErrorString(hipError_t e) { return e == 2 ? "stream order violation (host simulation)" : "host simulation"; }
inline hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
inline hipError_t hipDeviceGetAttribute(int* v, int, int) { *v = 256; return hipSuccess; }
template <typename F> inline hipError_t hipFuncSetAttribute(F, int, int) { return hipSuccess; }
template <typename T> inline hipError_t hipGetSymbolAddress(void** out, T* sym) { *out = (void*)sym; return hipSuccess; }

// Copies, events and pinned memory for the streaming code: everything completes at the call (one of the
// orders the streams allow).  What events and waits still do is bookkeeping: every stream carries a vector
// clock (order.cpp), copies declare the bytes they read and write, and a copy that is not ordered after an
// earlier overlapping access on another stream fails like a failed HIP call.
extern "C" {
uint64_t hostsim_order_snapshot(uint64_t stream);
void hostsim_order_wait(uint64_t stream, uint64_t handle);
void hostsim_order_forget(uint64_t lo, uint64_t bytes);
int hostsim_order_enqueue(uint64_t stream, const char* what, int n, const uint64_t* lo, const uint64_t* bytes, const int* is_write);
}
enum { hipErrorStreamOrder = 2 };
struct hostsim_event { uint64_t snapshot; };
typedef struct hostsim_event* hipEvent_t;
enum hipMemcpyKind { hipMemcpyHostToDevice = 1, hipMemcpyDeviceToHost = 2, hipMemcpyDeviceToDevice = 3 };
enum { hipEventDisableTiming = 2, hipHostMallocDefault = 0 };
inline hipError_t hostsim_declare(hipStream_t stream, const char* what, const void* read, size_t read_bytes, void* write, size_t write_bytes) {
    const uint64_t lo[2] = {(uint64_t)(uintptr_t)read, (uint64_t)(uintptr_t)write}, bytes[2] = {read_bytes, write_bytes};
    const int is_write[2] = {0, 1};
    return hostsim_order_enqueue((uint64_t)(uintptr_t)stream, what, 2, lo, bytes, is_write) ? hipErrorStreamOrder : hipSuccess;
}
inline hipError_t hipMemcpyAsync(void* dst, const void* src, size_t n, hipMemcpyKind, hipStream_t stream) {
    const hipError_t e = hostsim_declare(stream, "copy", src, n, dst, n);
    memcpy(dst, src, n);
    return e;
}
inline hipError_t hipMemcpy2DAsync(void* dst, size_t dpitch, const void* src, size_t spitch, size_t width, size_t height, hipMemcpyKind,
                                   hipStream_t stream) {
    const hipError_t e = height ? hostsim_declare(stream, "2-D copy", src, (height - 1) * spitch + width, dst, (height - 1) * dpitch + width)
                                : hipSuccess;
    for (size_t r = 0; r < height; ++r) memcpy((char*)dst + r * dpitch, (const char*)src + r * spitch, width);
    return e;
}
inline hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) { *e = new hostsim_event{0}; return hipSuccess; }
inline hipError_t hipEventDestroy(hipEvent_t e) { delete e; return hipSuccess; }
inline hipError_t hipEventRecord(hipEvent_t e, hipStream_t s) { e->snapshot = hostsim_order_snapshot((uint64_t)(uintptr_t)s); return hipSuccess; }
inline hipError_t hipStreamWaitEvent(hipStream_t s, hipEvent_t e, unsigned) { hostsim_order_wait((uint64_t)(uintptr_t)s, e->snapshot); return hipSuccess; }
inline hipError_t hipHostMalloc(void** p, size_t n, unsigned) { *p = malloc(n); return *p ? hipSuccess : hipErrorInvalidValue; }
inline hipError_t hipHostFree(void* p) {
    if (p) hostsim_order_forget((uint64_t)(uintptr_t)p, malloc_usable_size(p));
    free(p);
    return hipSuccess;
}

namespace hostsim {

struct Idx { unsigned x, y, z; };
extern Idx g_thread, g_block;
extern dim3 g_block_dim, g_grid_dim;
extern unsigned char* g_dynamic_lds;

void launch(dim3 grid, dim3 block, size_t lds_bytes, const std::function<void()>& body);
void sync_threads();
void sync_wave();
unsigned lane_slot();                     // index of the running lane's exchange slot
extern uint64_t g_exchange[];             // one 8-byte slot per lane of the workgroup
extern unsigned char g_alive[];           // 1 while the lane has not returned
unsigned flat_thread();

template <typename T>
inline T exchange(T v, int src_lane_in_wave) {
    static_assert(sizeof(T) <= 8, "exchange slot");
    const unsigned me = flat_thread();
    const unsigned wave0 = me & ~63u;
    uint64_t raw = 0;
    memcpy(&raw, &v, sizeof(T));
    g_exchange[me] = raw;
    sync_wave();
    T out = v;
    const unsigned src = wave0 + (unsigned)src_lane_in_wave;
    if (src_lane_in_wave >= 0 && src_lane_in_wave < 64 && src < g_block_dim.x * g_block_dim.y * g_block_dim.z && g_alive[src])
        memcpy(&out, &g_exchange[src], sizeof(T));
    sync_wave();
    return out;
}

}  // namespace hostsim

#define threadIdx hostsim::g_thread
#define blockIdx hostsim::g_block
#define blockDim hostsim::g_block_dim
#define gridDim hostsim::g_grid_dim

inline void __syncthreads() { hostsim::sync_threads(); }
template <typename T> inline T __shfl_xor(T v, int mask, int width = 64) { (void)width; return hostsim::exchange(v, (int)((hostsim::flat_thread() & 63u) ^ (unsigned)mask)); }
template <typename T> inline T __shfl_up(T v, unsigned delta, int width = 64) {
    (void)width;
    const int lane = (int)(hostsim::flat_thread() & 63u);
    return hostsim::exchange(v, lane - (int)delta >= 0 ? lane - (int)delta : lane);
}
template <typename T> inline T __shfl_down(T v, unsigned delta, int width = 64) {
    (void)width;
    const int lane = (int)(hostsim::flat_thread() & 63u);
    return hostsim::exchange(v, lane + (int)delta < 64 ? lane + (int)delta : lane);
}
template <typename T> inline T __shfl(T v, int src, int width = 64) { (void)width; return hostsim::exchange(v, src); }
inline int __any(int pred) {
    const unsigned me = hostsim::flat_thread(), wave0 = me & ~63u;
    const unsigned lanes = hostsim::g_block_dim.x * hostsim::g_block_dim.y * hostsim::g_block_dim.z;
    hostsim::g_exchange[me] = pred != 0;
    hostsim::sync_wave();
    int any = 0;
    for (unsigned l = wave0; l < wave0 + 64 && l < lanes; ++l) any |= hostsim::g_alive[l] && hostsim::g_exchange[l] != 0;
    hostsim::sync_wave();
    return any;
}
inline unsigned long long __ballot(int pred) {
    const unsigned me = hostsim::flat_thread(), wave0 = me & ~63u;
    const unsigned lanes = hostsim::g_block_dim.x * hostsim::g_block_dim.y * hostsim::g_block_dim.z;
    hostsim::g_exchange[me] = pred != 0;
    hostsim::sync_wave();
    unsigned long long who = 0;
    for (unsigned l = wave0; l < wave0 + 64 && l < lanes; ++l)
        if (hostsim::g_alive[l] && hostsim::g_exchange[l] != 0) who |= 1ull << (l - wave0);
    hostsim::sync_wave();
    return who;
}
template <typename T> inline T atomicAdd(T* p, T v) { T old = *p; *p = old + v; return old; }      // fibers never preempt each other
template <typename T> inline T atomicOr(T* p, T v) { T old = *p; *p = old | v; return old; }
template <typename T> inline T atomicMax(T* p, T v) { T old = *p; *p = std::max(old, v); return old; }

namespace hostsim {
extern float (*g_wave_f32)[64][16];             // [wave][lane][8 of A, 8 of B]: operands published for a matrix instruction

// global_load_lds_dwordx4: lane l of the wave copies 16 bytes from its global address to lds_addr + 16 l.
// The copy is made as LATE as the hardware may make it: it is queued, and lands only when the lane's own
// `s_waitcnt vmcnt(n)` leaves at most n of its loads in flight (oldest first).  A kernel that reads a buffer
// before its counted wait has covered the loads that fill it, or re-uses a buffer that loads are still in
// flight to, computes from stale or overwritten data here and fails its comparison.  (Counting these loads
// alone is the weaker guarantee: other vector memory operations in the window only make the real wait cover
// more.)  Loads never waited for are dropped when the workgroup ends.
struct PendingDma { unsigned lds; const void* src; };
constexpr int kMaxPendingDma = 64;
extern PendingDma g_dma[][kMaxPendingDma];
extern int g_dma_first[], g_dma_count[];
extern int g_dma_eager;     // 1: the other extreme, every copy lands at its issue (a load into a buffer that
                            // lanes scheduled later still have to read then shows as wrong results)
inline void lds_dma16(unsigned lds_addr, const void* gptr) {
    const unsigned me = flat_thread();
    if (g_dma_eager) { memcpy(reinterpret_cast<void*>((uintptr_t)lds_addr + 16u * (me & 63u)), gptr, 16); return; }
    if (g_dma_count[me] == kMaxPendingDma) { fprintf(stderr, "hostsim: more than %d LDS loads in flight in one lane\n", kMaxPendingDma); abort(); }
    g_dma[me][(g_dma_first[me] + g_dma_count[me]++) % kMaxPendingDma] = PendingDma{lds_addr + 16u * (me & 63u), gptr};
}
inline void wait_vmcnt(int n) {
    const unsigned me = flat_thread();
    while (g_dma_count[me] > n) {
        const PendingDma& d = g_dma[me][g_dma_first[me]];
        memcpy(reinterpret_cast<void*>((uintptr_t)d.lds), d.src, 16);
        g_dma_first[me] = (g_dma_first[me] + 1) % kMaxPendingDma;
        --g_dma_count[me];
    }
}

// v_mfma_f32_32x32x16 (bf16 / f16): D = A (32 x 16) * B (16 x 32) + C.  Lane l supplies A[l % 32][8 (l / 32) .. + 7]
// and B[8 (l / 32) .. + 7][l % 32]; register v of lane l is D[8 (v / 4) + 4 (l / 32) + v % 4][l % 32].
template <typename Frag, typename Acc>
inline Acc mfma32x32x16(Frag a, Frag b, Acc c) {
    const unsigned me = flat_thread(), w = me >> 6, l = me & 63u;
    float* mine = g_wave_f32[w][l];
    for (int j = 0; j < 8; ++j) { mine[j] = (float)a[j]; mine[8 + j] = (float)b[j]; }
    sync_wave();
    const float* b_lo = g_wave_f32[w][l % 32] + 8;            // B[0 .. 7][col], B[8 .. 15][col]
    const float* b_hi = g_wave_f32[w][l % 32 + 32] + 8;
    for (int v = 0; v < 16; ++v) {
        const unsigned row = 8u * (v / 4) + 4u * (l / 32) + (unsigned)(v % 4);
        const float* a_lo = g_wave_f32[w][row];
        const float* a_hi = g_wave_f32[w][row + 32];
        float sum = c[v];
        for (int k = 0; k < 8; ++k) sum += a_lo[k] * b_lo[k];
        for (int k = 0; k < 8; ++k) sum += a_hi[k] * b_hi[k];
        c[v] = sum;
    }
    sync_wave();
    return c;
}

// 8-bit floating point: e4m3 (bias 7, no infinity, S.1111.111 is NaN) and e5m2 (bias 15, IEEE-like).
inline float fp8_value(unsigned char b, bool e5m2) {
    const int mbits = e5m2 ? 2 : 3, bias = e5m2 ? 15 : 7;
    const int mant = b & ((1 << mbits) - 1), ex = (b >> mbits) & (e5m2 ? 31 : 15);
    float v;
    if (e5m2 && ex == 31) v = mant ? NAN : INFINITY;
    else if (!e5m2 && ex == 15 && mant == 7) v = NAN;
    else v = ex ? ldexpf((float)(mant + (1 << mbits)), ex - bias - mbits) : ldexpf((float)mant, 1 - bias - mbits);
    return b & 0x80 ? -v : v;
}
struct Fp8Table {
    float value[2][256];
    Fp8Table() {
        for (int e = 0; e < 2; ++e)
            for (int b = 0; b < 256; ++b) value[e][b] = fp8_value((unsigned char)b, e == 1);
    }
};
inline const Fp8Table& fp8_table() { static const Fp8Table t; return t; }
// nearest even; finite values past the largest number become NaN (e4m3) or infinity (e5m2)
inline unsigned char fp8_code(float x, bool e5m2) {
    const int mbits = e5m2 ? 2 : 3, low = e5m2 ? -14 : -6;
    const unsigned char sign = std::signbit(x) ? 0x80 : 0, top = e5m2 ? 0x7b : 0x7e;
    if (std::isnan(x)) return sign | 0x7f;
    const float a = fabsf(x);
    if (std::isinf(a)) return sign | (e5m2 ? 0x7c : 0x7f);
    if (a == 0.f) return sign;
    int p;
    frexpf(a, &p);
    const int ex = std::max(p - 1, low);
    const double steps = nearbyint(ldexp((double)a, mbits - ex));       // of 2^(ex - mbits)
    const int code = (int)steps + ((ex - low) << mbits);                // the codes are consecutive across binades
    return sign | (unsigned char)(code > top ? (e5m2 ? 0x7c : 0x7f) : code);
}
inline int cvt_pk_8(float a, float b, int old, bool high, bool e5m2) {
    const unsigned two = fp8_code(a, e5m2) | ((unsigned)fp8_code(b, e5m2) << 8);
    return high ? (int)(((unsigned)old & 0xffffu) | (two << 16)) : (int)(((unsigned)old & 0xffff0000u) | two);
}

// v_cvt_scalef32_pk_{fp8,bf8}_{bf16,f16}: a pair divided by the power of two in the scale's exponent field, rounded once
template <typename S2, typename P2>
inline S2 cvt_scale_pk_8(S2 old, P2 src, float scale, bool high, bool e5m2) {
    unsigned bits;
    memcpy(&bits, &scale, 4);
    const int e = (int)((bits >> 23) & 255u) - 127;
    auto one = [&](float v) { return fp8_code((float)ldexp((double)v, -e), e5m2); };     // (2-byte values: exact in fp32 unless tiny)
    const unsigned two = one((float)src[0]) | ((unsigned)one((float)src[1]) << 8);
    old[high ? 1 : 0] = (short)two;
    return old;
}

// v_mfma_scale_f32_32x32x64_f8f6f4 with 8-bit operands: D = A (32 x 64) * B (64 x 32) + C, every 32 k of an
// operand row times 2^(byte - 127) (byte 255: NaN).  Lane l supplies A[l % 32][32 (l / 32) .. + 31], B likewise,
// and the scale bytes of those values; the accumulator layout is that of the 16-bit instruction.
// The 16x16x128 form: lane l supplies row l % 16, k 32 (l / 16) .. + 31; register v of lane l is
// D[4 (l / 16) + v][l % 16].
extern float (*g_wave_f8)[64][64];              // [wave][lane][32 of A, 32 of B], scaled
template <int N, typename Frag, typename Acc>
inline Acc mfma_scale(Frag a, Frag b, Acc c, int fmt_a, int fmt_b, int opsel_a, int scale_a, int opsel_b, int scale_b) {
    constexpr int K_LANES = 64 / N;             // lanes that share a row
    const unsigned me = flat_thread(), w = me >> 6, l = me & 63u;
    float* mine = g_wave_f8[w][l];
    const unsigned char *pa = reinterpret_cast<const unsigned char*>(&a), *pb = reinterpret_cast<const unsigned char*>(&b);
    const int ba = (scale_a >> (8 * opsel_a)) & 255, bb = (scale_b >> (8 * opsel_b)) & 255;
    const float sa = ba == 255 ? NAN : ldexpf(1.f, ba - 127), sb = bb == 255 ? NAN : ldexpf(1.f, bb - 127);
    const float *ta = fp8_table().value[fmt_a == 1], *tb = fp8_table().value[fmt_b == 1];
    for (int j = 0; j < 32; ++j) { mine[j] = ta[pa[j]] * sa; mine[32 + j] = tb[pb[j]] * sb; }
    sync_wave();
    for (int v = 0; v < N * N / 64; ++v) {
        const unsigned row = N == 32 ? 8u * (v / 4) + 4u * (l / 32) + (unsigned)(v % 4) : 4u * (l / 16) + (unsigned)v;
        float sum = c[v];
        for (int q = 0; q < K_LANES; ++q) {
            const float *x = g_wave_f8[w][row + N * q], *y = g_wave_f8[w][l % N + N * q] + 32;
            float part[8] = {0, 0, 0, 0, 0, 0, 0, 0};          // eight partial sums: the compiler's vectors
            for (int k = 0; k < 32; k += 8)
                for (int u = 0; u < 8; ++u) part[u] += x[k + u] * y[k + u];
            for (int u = 0; u < 8; ++u) sum += part[u];
        }
        c[v] = sum;
    }
    sync_wave();
    return c;
}

// Data-parallel operand of v_mov: row_shr:1..15 (0x111 ..), row_bcast:15 (0x142), row_bcast:31 (0x143).  A lane whose row is
// not in row_mask, or whose source does not exist, keeps `old`.
inline int update_dpp(int old, int v, int ctrl, int row_mask) {
    const unsigned l = flat_thread() & 63u, row = l >> 4;
    int src = -1;
    if (ctrl >= 0x111 && ctrl <= 0x11f) { const unsigned n = (unsigned)ctrl - 0x110; if ((l & 15u) >= n) src = (int)(l - n); }
    else if (ctrl >= 0x121 && ctrl <= 0x12f) src = (int)((l & ~15u) | ((l - ((unsigned)ctrl - 0x120)) & 15u));       // row_ror
    else if (ctrl == 0x142) { if (row >= 1) src = (int)(row * 16 - 1); }
    else if (ctrl == 0x143) { if (row >= 2) src = 31; }
    else { fprintf(stderr, "hostsim: data-parallel control 0x%x\n", ctrl); abort(); }
    const int got = exchange(v, src < 0 ? (int)l : src);
    return src >= 0 && ((row_mask >> row) & 1) ? got : old;
}
// v_permlane16_swap: the odd rows of 16 lanes of the first operand change places with the even rows of the second.
typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
inline u32x2_t permlane16_swap(unsigned a, unsigned b) {
    const unsigned l = flat_thread() & 63u;
    const unsigned b_even = exchange(b, (int)(l & ~16u)), a_odd = exchange(a, (int)(l | 16u));
    u32x2_t out = {l & 16u ? b_even : a, l & 16u ? b : a_odd};
    return out;
}
// v_permlane32_swap: the upper 32 lanes of the first operand change places with the lower 32 of the second.
inline u32x2_t permlane32_swap(unsigned a, unsigned b) {
    const unsigned l = flat_thread() & 63u;
    const unsigned b_lo = exchange(b, (int)(l & 31u)), a_hi = exchange(a, (int)((l & 31u) + 32u));
    u32x2_t out = {l < 32 ? a : b_lo, l < 32 ? a_hi : b};
    return out;
}

// ds_read_b64_tr_b16: inside each group of 16 lanes, lane s receives, for j = 0 .. 3, element s % 4 of the
// 8 bytes that lane 4 j + s / 4 of the group addressed.
template <typename V4>
inline V4 ds_read_tr16(const void* addr) {
    const unsigned me = flat_thread(), group0 = me & ~15u, s = me & 15u;
    g_exchange[me] = (uint64_t)(uintptr_t)addr;
    sync_wave();
    V4 out;
    for (unsigned j = 0; j < 4; ++j) {
        const short* src = reinterpret_cast<const short*>((uintptr_t)g_exchange[group0 + 4 * j + s / 4]);
        out[j] = src[s % 4];
    }
    sync_wave();
    return out;
}

// v_perm_b32: byte i of the result is byte sel[i] of the 8 bytes {hi : lo} (0-3 from lo, 4-7 from hi).
inline unsigned perm_b32(unsigned hi, unsigned lo, unsigned sel) {
    const uint64_t both = ((uint64_t)hi << 32) | lo;
    unsigned out = 0;
    for (int i = 0; i < 4; ++i) out |= (unsigned)((both >> (8 * ((sel >> (8 * i)) & 7))) & 0xff) << (8 * i);
    return out;
}
}  // namespace hostsim

#define __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, x, y, z) hostsim::mfma32x32x16(a, b, c)
#define __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, x, y, z) hostsim::mfma32x32x16(a, b, c)
#define __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, fa, fb, oa, sa, ob, sb) hostsim::mfma_scale<32>(a, b, c, fa, fb, oa, sa, ob, sb)
#define __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, fa, fb, oa, sa, ob, sb) hostsim::mfma_scale<16>(a, b, c, fa, fb, oa, sa, ob, sb)
#define __builtin_amdgcn_permlane16_swap(a, b, fi, bc) hostsim::permlane16_swap(a, b)
#define __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(old, src, scale, high) hostsim::cvt_scale_pk_8(old, src, scale, high, false)
#define __builtin_amdgcn_cvt_scalef32_pk_bf8_bf16(old, src, scale, high) hostsim::cvt_scale_pk_8(old, src, scale, high, true)
#define __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(old, src, scale, high) hostsim::cvt_scale_pk_8(old, src, scale, high, false)
#define __builtin_amdgcn_cvt_scalef32_pk_bf8_f16(old, src, scale, high) hostsim::cvt_scale_pk_8(old, src, scale, high, true)
#define __builtin_amdgcn_update_dpp(old, v, ctrl, rows, banks, bound) hostsim::update_dpp(old, v, ctrl, rows)
#define __builtin_amdgcn_readlane(v, lane) hostsim::exchange((int)(v), (int)(lane))
#define __builtin_amdgcn_permlane32_swap(a, b, fi, bc) hostsim::permlane32_swap(a, b)
#define __builtin_amdgcn_cvt_pk_fp8_f32(a, b, old, high) hostsim::cvt_pk_8(a, b, old, high, false)
#define __builtin_amdgcn_cvt_pk_bf8_f32(a, b, old, high) hostsim::cvt_pk_8(a, b, old, high, true)
#define __builtin_amdgcn_ds_read_tr16_b64_v4i16(p) hostsim::ds_read_tr16<short __attribute__((ext_vector_type(4)))>((const void*)(p))
#define __builtin_amdgcn_perm(hi, lo, sel) hostsim::perm_b32(hi, lo, sel)

// gfx950 builtins the kernels use, by their documented meaning
#define __builtin_amdgcn_rcpf(x) (1.0f / (x))
// (the instruction's estimate: the callers refine it)
#define __builtin_amdgcn_rsq(x) ((double)(float)(1.0 / sqrt(x)))
#define __builtin_amdgcn_exp2f(x) exp2f(x)
#define __builtin_amdgcn_readfirstlane(x) (x)          /* only ever applied to wave-uniform values */
#define __builtin_amdgcn_wave_barrier() hostsim::sync_wave()
#define __builtin_amdgcn_fence(...) ((void)0)
#define __builtin_amdgcn_sched_barrier(x) ((void)0)
#define __builtin_amdgcn_s_setprio(x) ((void)0)
inline float rsqrtf(float x) { return 1.0f / sqrtf(x); }
#define __expf(x) expf(x)
#define __logf(x) logf(x)
