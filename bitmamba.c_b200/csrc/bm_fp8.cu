// 8-bit floating point products with a scale for each block of 128: the
// quantisation of activations and the product on the fp8 tensor cores.
//
//   out[m, n] = sum_b sa[b][m] * sw[n / 128][b] * sum_{k in b} a[m, k] * w[n, k]
//
// The scales change every 128 columns of K, so a block's sum cannot stay in
// the tensor core's accumulator: each block is one fresh accumulation of four
// instructions into a tensor memory buffer, and the promotion warps read it
// back, scale it and add it to fp32 sums in registers while the tensor core
// works on the next buffer.
//
// Two shapes of tile:
//   few rows    128 rows of w (the accumulator's lanes) by NB = 16, 32, 64, 96
//               or 128 rows of a (its columns), so that a few rows cost a
//               narrow tile instead of a padded one.  Bound by the bytes of w: 1 x 50257 x
//               2048 takes 21 us, 4.9 TB/s.  In the middle, where a layer's
//               projection is a tile or two an SM, by latency: 72 x 8288 x 2048
//               takes 9.1 us, 16 x 2048 x 2048 already 5.5.
//   many rows   128 rows of a (lanes) by 128 rows of w: a thread's scale is
//               one value for its 128 columns.  (With w on the lanes every
//               column has its own scale, and fetching 128 of them a block
//               took twice as long as the tensor core's work.)
#include <cstdint>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "bm_ctx.cuh"
#include "bm_sampler.h"
#include "bm_tc.cuh"

namespace bml {
namespace {

// ------------------------------------------------------------- quantise --

constexpr int QV = 4;  // groups of 4 columns a thread holds: d <= 16 * threads per row

__device__ __forceinline__ float4 load4(const float *p) {
    return *reinterpret_cast<const float4 *>(p);
}
__device__ __forceinline__ float4 load4(const __nv_bfloat16 *p) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u),
                       __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
}

// x / s from r = 1 / s: the quotient's error is exact in one multiply-add, and
// corrects it (Markstein, IBM J. Res. Dev. 34, 1990).
__device__ __forceinline__ float divide(float x, float s, float r) {
    const float q = x * r;
    return fmaf(fmaf(-q, s, x), r, q);
}
__device__ __forceinline__ uint32_t to_e4m3(float4 v) { return __nv_fp8x4_e4m3(v).__x; }
__device__ __forceinline__ float4 times(float4 v, float k) {
    return make_float4(v.x * k, v.y * k, v.z * k, v.w * k);
}
// Of two neighbouring codes the one that 448 v / top rounds to: which side of
// the border (the mean of both, 5 bits) it is on, both multiplied by top, is
// exact in 64 bits; on it, the even one.
__device__ __forceinline__ uint32_t nearer(uint32_t lo, uint32_t hi, double v, double top) {
    auto value = [](uint32_t c) { return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3))); };
    const double border = 0.5f * fabsf(value(lo) + value(hi)), d = 448.0 * fabs(v) - border * top;
    return d > 0.0 ? hi : d < 0.0 ? lo : lo & 1u ? hi : lo;
}
__device__ __noinline__ uint32_t settle(uint32_t lo, uint32_t hi, double x, double y, double z, double w, double top) {
    const double f[4] = {x, y, z, w};
    uint32_t q = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) q |= nearer(lo >> (8 * i) & 255u, hi >> (8 * i) & 255u, f[i], top) << (8 * i);
    return q;
}
__device__ __noinline__ uint32_t settle(uint32_t lo, uint32_t hi, float4 v, float top) {
    const float f[4] = {v.x, v.y, v.z, v.w};
    uint32_t q = lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = lo >> (8 * i) & 255u, b = hi >> (8 * i) & 255u;
        if (a != b) q ^= (a ^ nearer(a, b, f[i], top)) << (8 * i);
    }
    return q;
}

// A block near the ends of the range of fp32, past them as products with the
// weight, or with values that are not finite: this thread's codes and the
// block's scale.  x is taken by a power of two kx and the weight by kw, whose
// product is back^-2; what is inexact then is far below the codes.
template <bool NORM>
__device__ __noinline__ uint2 at_the_ends(float4 x, float4 k, float rms, bool high) {
    const float kx = !NORM ? 0x1p-64f : high ? 0x1p-66f : 0x1p+64f, back = !NORM ? 0x1p+32f : high ? 0x1p+65f : 0x1p-32f;
    x = times(x, kx);
    if (NORM && high) k = times(k, 0x1p-64f);
    const float4 g = NORM ? make_float4(x.x * k.x, x.y * k.y, x.z * k.z, x.w * k.w) : x;
    const unsigned m = max(max(__float_as_uint(g.x) & 0x7fffffffu, __float_as_uint(g.y) & 0x7fffffffu),
                           max(__float_as_uint(g.z) & 0x7fffffffu, __float_as_uint(g.w) & 0x7fffffffu));
    const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, m)), most = NORM ? top * rms : top;
    const float sc = __fdiv_rn(most, 448.0f);
    if (!(top < __int_as_float(0x7f800000)) || most != most) {  // an infinity or NaN
        const float4 f = make_float4(__fdiv_rn(g.x * rms, sc), __fdiv_rn(g.y * rms, sc), __fdiv_rn(g.z * rms, sc),
                                     __fdiv_rn(g.w * rms, sc));
        return make_uint2(to_e4m3(f), __float_as_uint(sc));
    }
    if (!(most > 0.0f)) return make_uint2(0, __float_as_uint(1.0f));  // (rms is 0: the squares passed the range)
    const float r = __fdiv_rn(448.0f, top);
    const uint32_t lo = to_e4m3(times(g, r * (1.0f - 0x1p-20f))), hi = to_e4m3(times(g, r * (1.0f + 0x1p-20f)));
    uint32_t q;
    if (NORM) {
        const double e0 = (double)x.x * k.x, e1 = (double)x.y * k.y, e2 = (double)x.z * k.z, e3 = (double)x.w * k.w;
        double most_e = fmax(fmax(fabs(e0), fabs(e1)), fmax(fabs(e2), fabs(e3)));
        for (int o = 16; o > 0; o >>= 1) most_e = fmax(most_e, __shfl_xor_sync(0xffffffffu, most_e, o));
        q = settle(lo, hi, e0, e1, e2, e3, most_e);
    } else {
        q = settle(lo, hi, g, top);
    }
    return make_uint2(q, __float_as_uint(sc * back * back));
}

// TPR threads per row: a warp's 32 groups of 4 columns are one block of 128.
// Bound by memory: a row is read once and stays in registers.  8192 x 4096 fp32
// takes 27.9 us, 6.0 TB/s of reads and writes (the device copies at 6.5), bf16
// 24.7, with a norm 40.3 and 38.6.
template <typename T, int TPR, bool NORM>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR)
    quantize_kernel(const T *x, int rows, int d, int64_t ldx, const float *norm_w, uint8_t *q,
                    float *scale, int64_t ld_scale) {
    constexpr int NT = TPR < 256 ? 256 : TPR;
    __shared__ float part[NT / 32];
    const int t = threadIdx.x % TPR, lane = threadIdx.x & 31;
    const int row = blockIdx.x * (NT / TPR) + threadIdx.x / TPR;
    const bool live = row < rows;
    float4 v[QV];
#pragma unroll
    for (int i = 0; i < QV; ++i) {
        const int col = 4 * (t + i * TPR);
        v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (live && col < d) v[i] = load4(x + (int64_t)row * ldx + col);
    }
    // The norm's factor of the row is in the scale alone: it drops out of
    // x / scale, with its rounding.
    float rms = 1.0f;
    if (NORM) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < QV; ++i)
            s = fmaf(v[i].x, v[i].x, fmaf(v[i].y, v[i].y, fmaf(v[i].z, v[i].z, fmaf(v[i].w, v[i].w, s))));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (TPR > 32) {
            if (lane == 0) part[threadIdx.x >> 5] = s;
            __syncthreads();
            const int w0 = threadIdx.x / TPR * (TPR / 32);
            s = 0.f;
#pragma unroll
            for (int w = 0; w < TPR / 32; ++w) s += part[w0 + w];
        }
        rms = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(s, (float)d) + 1e-6f));
#pragma unroll
        for (int i = 0; i < QV; ++i) {
            const int col = 4 * (t + i * TPR);
            if (col < d) {
                const float4 w = load4(norm_w + col);
                v[i] = make_float4(v[i].x * w.x, v[i].y * w.y, v[i].z * w.z, v[i].w * w.w);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < QV; ++i) {
        const int col = 4 * (t + i * TPR);
        // the largest magnitude: as integers, whose order a NaN leads
        const unsigned m = max(max(__float_as_uint(v[i].x) & 0x7fffffffu, __float_as_uint(v[i].y) & 0x7fffffffu),
                               max(__float_as_uint(v[i].z) & 0x7fffffffu, __float_as_uint(v[i].w) & 0x7fffffffu));
        const unsigned bits = __reduce_max_sync(0xffffffffu, m);
        const float top = __uint_as_float(bits), most = NORM ? top * rms : top;
        float sc = 1.0f;
        uint32_t w = 0;
        // For bf16 alone one check of the bits, 2^-100 < top < 2^119 (448 times the
        // largest is in range); beyond, both sides of the quotient by 512.
        constexpr bool B16 = !NORM && sizeof(T) == 2;
        constexpr unsigned LEAST = (127 - 100) << 23, MOST = (127 + 119) << 23;
        if (B16 && bits - (LEAST + 1) >= MOST - (LEAST + 1)) {
            if (bits >= MOST) {
                const float4 f = times(v[i], 448.0f / 512.0f);
                const float s = top * 0x1p-9f;
                sc = __fdiv_rn(top, 448.0f);
                w = to_e4m3(make_float4(__fdiv_rn(f.x, s), __fdiv_rn(f.y, s), __fdiv_rn(f.z, s), __fdiv_rn(f.w, s)));
            }
        } else if (!B16 && (!(top < 0x1p+119f && most < 0x1p+119f) || (top <= 0x1p-100f && most > 0x1p-100f))) {
            float4 k = make_float4(1.f, 1.f, 1.f, 1.f);
            if (NORM && live && col < d) {
                v[i] = load4(x + (int64_t)row * ldx + col);
                k = load4(norm_w + col);
            }
            const uint2 c = at_the_ends<NORM>(v[i], k, rms, !(top <= 0x1p-100f));
            w = c.x;
            sc = __uint_as_float(c.y);
        } else if (B16 || most > 0x1p-100f) {
            sc = divide(most, 448.0f, 1.0f / 448.0f);
            // Rounded from both sides of the approximate quotients, by more than
            // these can be off (2 ulp of the reciprocal, 2 roundings: 2^-21.4;
            // with the norm's weight 2 more); where that differs, a border is
            // close and the exact ones decide.
            constexpr float margin = NORM ? 0x1p-20f : 0x1p-21f;
            float r;
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(top));
            uint32_t lo = 0;
            bool close = false;
            if (B16) {
                // 448 v is exact, its quotient by the 8 bits of top is on a border
                // or 2^-16 away: one corrected quotient is enough
                const float4 x448 = times(v[i], 448.0f);
                w = to_e4m3(make_float4(divide(x448.x, top, r), divide(x448.y, top, r), divide(x448.z, top, r),
                                        divide(x448.w, top, r)));
            } else {
                r *= 448.0f;
                w = to_e4m3(times(v[i], r * (1.0f + margin)));
                lo = to_e4m3(times(v[i], r * (1.0f - margin)));
                close = w != lo;
            }
            if (!NORM) {
                if (close) w = settle(lo, w, v[i], top);
            } else if (__any_sync(0xffffffffu, close)) {  // (top is the warp's)
                // the products with the weight unrounded, and their largest
                float4 f = make_float4(0.f, 0.f, 0.f, 0.f), k = f;
                if (live && col < d) {
                    f = load4(x + (int64_t)row * ldx + col);
                    k = load4(norm_w + col);
                }
                const double e0 = (double)f.x * k.x, e1 = (double)f.y * k.y, e2 = (double)f.z * k.z,
                             e3 = (double)f.w * k.w;
                double most_e = fmax(fmax(fabs(e0), fabs(e1)), fmax(fabs(e2), fabs(e3)));
                for (int o = 16; o > 0; o >>= 1) most_e = fmax(most_e, __shfl_xor_sync(0xffffffffu, most_e, o));
                if (close) w = settle(lo, w, e0, e1, e2, e3, most_e);
            }
        }
        if (live && col < d) {
            *reinterpret_cast<uint32_t *>(q + (int64_t)row * d + col) = w;
            if (lane == 0) scale[(int64_t)(col >> 7) * ld_scale + row] = sc;
        }
    }
}

template <typename T, bool NORM>
cudaError_t quantize(const T *x, int rows, int d, int64_t ldx, const float *norm_w, uint8_t *q,
                     float *scale, int64_t ld_scale, cudaStream_t s) {
#define BM_Q(TPR)                                                                               \
    if (d <= 4 * QV * TPR) {                                                                    \
        constexpr int per = TPR < 256 ? 256 / TPR : 1;                                          \
        return bmc::launch(quantize_kernel<T, TPR, NORM>, dim3((unsigned)((rows + per - 1) / per)), \
                           TPR < 256 ? 256 : TPR, 0, s, x, rows, d, ldx, norm_w, q, scale, ld_scale); \
    }
    BM_Q(32)
    BM_Q(128)
    BM_Q(256)
    BM_Q(1024)
#undef BM_Q
    return cudaErrorInvalidValue;
}

// -------------------------------------------------------------- product --

constexpr int BKB = 128;  // bytes (columns) of K per block

__device__ __forceinline__ void umma_f8(uint32_t tmem, uint64_t da, uint64_t db, uint32_t idesc,
                                        uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(tmem),
        "l"(da), "l"(db), "r"(idesc), "r"(accumulate));
}
// consecutive fp32 accumulator columns of this thread's lane; the registers
// hold them after tmem_wait
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
        "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
        "%28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
        "%11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
// (the registers pass through, so that no use moves before the wait)
template <int N>
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void arrive(uint64_t *b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(sa(b)) : "memory");
}
__device__ __forceinline__ void tmem_alloc(uint32_t *slot, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sa(slot)),
                 "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}
__device__ __forceinline__ void before_sync() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void after_sync() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// both operands e4m3 (formats 0) and K-major, D fp32, 128 lanes, n columns
__host__ __device__ constexpr uint32_t f8_desc(int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ float as_f(uint32_t v) { return __uint_as_float(v); }

struct ProductArgs {
    const float *sa, *sw;
    int64_t ld_scale, ldo;
    float *out;
    int M, K, N;
    int *err;
};

// ---- few rows
//
// Persistent CTAs with one tile after the other, or (split > 1) a cluster of
// `split` CTAs per tile, each with a part of K, whose sums they hand one
// another through shared memory and add in order.  The scales
// of a stay in shared memory, those of w in the lanes of a warp.  Two threads
// issue copies and two MMAs, each every other block: one alone spends some 800
// cycles a block on its waits, descriptors and commits (the blocks are
// accumulations of their own, so their order does not matter).
template <int NB>
struct Few {
    static constexpr int BV = 128;
    static constexpr int PW = NB >= 64 ? 8 : 4;  // promotion warps
    static constexpr int CW = NB / (PW / 4);     // columns per promotion warp
    static constexpr int TB = 4;                 // tensor memory buffers
    static constexpr int COLS = NB == 96 ? 512 : TB * NB;  // a power of two >= 32
    static constexpr int STAGE = BV * BKB + NB * BKB;
    static constexpr int THREADS = 32 * (4 + PW);
    static constexpr int MAX_STAGES = 12;
    static constexpr size_t BARS = (2 * MAX_STAGES + 2 * TB) * 8 + 16;
    static constexpr int SMEM = 220 * 1024;
    // As many stages as fit beside the scales of kb blocks, and an even number
    // of them: block j is in stage j % stages, so every use of a stage is of one
    // parity, by one of the copying threads and one of the MMA threads, and each
    // waits for the other's last use of it.  With an odd number a stage's uses
    // alternate between the threads, and the one parity bit of a wait tells a
    // use from the second to last before it only while the four accumulators
    // keep the threads closer than that: with five stages they do not, and a
    // block was overwritten before its MMAs read it.
    static constexpr int stages(int kb) {
        const int n = (int)((SMEM - 1024 - BARS - (size_t)kb * NB * 4) / STAGE);
        return (n < MAX_STAGES ? n : MAX_STAGES) & ~1;
    }
    static_assert(MAX_STAGES % 2 == 0, "stages");
};

template <int NB>
__global__ void __launch_bounds__(Few<NB>::THREADS, 1)
    few_rows_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmA,
                    const ProductArgs p, int stages, int split) {
    using S = Few<NB>;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    // (an offset, so that the compiler still knows it for shared memory)
    unsigned char *const smem = smem_raw + ((1024u - (sa(smem_raw) & 1023u)) & 1023u);
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + stages * S::STAGE);
    uint64_t *empty = full + S::MAX_STAGES;
    uint64_t *accf = empty + S::MAX_STAGES;  // [TB] a block's sums are complete
    uint64_t *acce = accf + S::TB;           // [TB] they are read
    uint32_t *tslot = reinterpret_cast<uint32_t *>(acce + S::TB);
    int *abort_ = reinterpret_cast<int *>(tslot + 1);
    float *scales = reinterpret_cast<float *>(tslot + 4);  // [blocks][NB]
    // (from lane 0, so that the compiler knows it for one value a warp)
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    // (several tiles of rows of a only where every CTA has one tile)
    const int MT = (p.M + NB - 1) / NB, tiles = (p.N + S::BV - 1) / S::BV * MT, KB = (p.K + BKB - 1) / BKB;
    const int rank = blockIdx.x % split, first = blockIdx.x / split, step = gridDim.x / split;
    const int m0 = first % MT * NB;
    const int kb0 = (int)((int64_t)KB * rank / split), nkb = (int)((int64_t)KB * (rank + 1) / split) - kb0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < S::TB; ++i) {
            mbar_init(&accf[i], 1);
            mbar_init(&acce[i], S::PW);
        }
        *abort_ = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) tmem_alloc(tslot, S::COLS);
    before_sync();
    __syncthreads();
    after_sync();
    const uint32_t tmem = *tslot;
    auto fail = [&]() { atomicOr(abort_, 1); };
    auto aborted = [&]() { return *reinterpret_cast<volatile int *>(abort_) != 0; };

    // blocks and stages in turn: this thread's next ones
    auto advance = [&](int &s, int &ph) {
        s += 2;
        if (s >= stages) {
            s -= stages;
            ph ^= 1;
        }
    };
    if (warp < 2) {
        if (lane == 0) {
            int s = warp, ph = 1, g = 0, issued = 0;
            for (int t = first; t < tiles && !aborted(); t += step) {
                for (int kb = (g ^ warp) & 1; kb < nkb; kb += 2) {
                    if (!mbar_wait(&empty[s], ph)) {  // (a fresh barrier is past phase 1)
                        fail();
                        break;
                    }
                    unsigned char *st = smem + (size_t)s * S::STAGE;
                    mbar_expect_tx(&full[s], S::STAGE);
                    tma_load_2d(st, &tmW, (kb0 + kb) * BKB, t / MT * S::BV, &full[s]);
                    tma_load_2d(st + S::BV * BKB, &tmA, (kb0 + kb) * BKB, m0, &full[s]);
                    advance(s, ph);
                    ++issued;
                }
                g += nkb;
            }
            if (aborted()) {  // no copy may outlive the CTA
                for (int i = min(issued, (stages + 1) / 2); i > 0; --i) {
                    s -= 2;
                    if (s < 0) {
                        s += stages;
                        ph ^= 1;
                    }
                    mbar_wait(&full[s], ph ^ 1);
                }
            }
        }
    } else if (warp < 4) {
        if (lane == 0) {
            int s = warp - 2, ph = 0, g = 0, last = -1;
            for (int t = first; t < tiles && !aborted(); t += step) {
                for (int kb = (g ^ warp) & 1; kb < nkb; kb += 2) {
                    const int b = (g + kb) % S::TB;
                    if (!mbar_wait(&acce[b], ((g + kb) / S::TB + 1) & 1) || !mbar_wait(&full[s], ph)) {
                        fail();
                        break;
                    }
                    after_sync();
                    const uint32_t w0 = sa(smem + (size_t)s * S::STAGE), a0 = w0 + S::BV * BKB;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        umma_f8(tmem + (uint32_t)(b * NB), sdesc(w0 + k * 32), sdesc(a0 + k * 32), f8_desc(NB),
                                k > 0 ? 1u : 0u);
                    umma_commit(&empty[s]);
                    umma_commit(&accf[b]);
                    advance(s, ph);
                    last = g + kb;
                }
                g += nkb;
            }
            if (aborted() && last >= 0) mbar_wait(&accf[last % S::TB], (last / S::TB) & 1);
        }
    } else {
        for (int i = threadIdx.x - 128; i < nkb * NB; i += 32 * S::PW) {
            const int m = m0 + i % NB;
            scales[i] = m < p.M ? p.sa[(kb0 + i / NB) * p.ld_scale + m] : 0.0f;
        }
        asm volatile("bar.sync 1, %0;" ::"r"(32 * S::PW) : "memory");
        const int q = warp & 3, c0 = ((warp - 4) >> 2) * S::CW;
        constexpr int LD = S::CW % 32 ? 16 : 32;
        int g = 0;
        // 32 blocks' scales of w in the lanes, the next ones on their way
        auto load_sw = [&](int t, int kb) {
            return t < tiles && kb + lane < nkb ? p.sw[(int64_t)(t / MT) * KB + kb0 + kb + lane] : 0.0f;
        };
        float sw_next = load_sw(first, 0);
        // (a cluster's barriers are reached whatever failed)
        for (int t = first; t < tiles && (split > 1 || !aborted()); t += step) {
            float2 acc[S::CW / 2];
#pragma unroll
            for (int j = 0; j < S::CW / 2; ++j) acc[j] = make_float2(0.0f, 0.0f);
            bool good = true;
            float sw = 0.0f;
            for (int kb = 0; kb < nkb; ++kb, ++g) {
                if (kb % 32 == 0) {
                    sw = sw_next;
                    sw_next = kb + 32 < nkb ? load_sw(t, kb + 32) : load_sw(t + step, 0);
                }
                const int b = g % S::TB;
                const bool ok = mbar_wait(&accf[b], (g / S::TB) & 1);
                if (__any_sync(0xffffffffu, !ok)) {
                    fail();
                    good = false;
                    break;
                }
                after_sync();
                const uint32_t tb = tmem + (uint32_t)(b * NB + c0) + ((uint32_t)(q * 32) << 16);
                const float k = __shfl_sync(0xffffffffu, sw, kb % 32);
                const float2 k2 = make_float2(k, k);
                const float4 *sc = reinterpret_cast<const float4 *>(scales + kb * NB + c0);
#pragma unroll
                for (int c = 0; c < S::CW; c += LD) {
                    uint32_t v[LD];
                    tmem_load(tb + c, v);
                    float4 f[LD / 4];
#pragma unroll
                    for (int j = 0; j < LD / 4; ++j) f[j] = sc[c / 4 + j];
                    tmem_wait(v);
                    if (c + LD == S::CW) {  // the sums are read: the buffer is free
                        before_sync();
                        __syncwarp();
                        if (lane == 0) arrive(&acce[b]);
                    }
#pragma unroll
                    for (int j = 0; j < LD; j += 4) {
                        const int at = (c + j) / 2;
                        acc[at] = __ffma2_rn(make_float2(as_f(v[j]), as_f(v[j + 1])),
                                             __fmul2_rn(make_float2(f[j / 4].x, f[j / 4].y), k2), acc[at]);
                        acc[at + 1] = __ffma2_rn(make_float2(as_f(v[j + 2]), as_f(v[j + 3])),
                                                 __fmul2_rn(make_float2(f[j / 4].z, f[j / 4].w), k2), acc[at + 1]);
                    }
                }
            }
            const int n = t / MT * S::BV + q * 32 + lane;
            float *o = p.out + (int64_t)(m0 + c0) * p.ldo + n;
            if (split == 1) {
                if (good && n < p.N) {
#pragma unroll
                    for (int j = 0; j < S::CW; ++j, o += p.ldo)
                        if (m0 + c0 + j < p.M) *o = j % 2 ? acc[j / 2].y : acc[j / 2].x;
                }
                continue;
            }
            // Each CTA of the cluster adds up a share of the columns: the sums of
            // this CTA's part of K go there, [part][column of the share][lane of
            // w], over the stages, which are idle by then (every tensor core has
            // read its own, else its CTA had not got to the barrier).  (100 x
            // 2048 x 4096: 9.9 us; all sums to the first CTA 12.2.)
            auto exchange = [&](auto parts) {
                constexpr int SPLIT = decltype(parts)::value, SHARE = S::CW / SPLIT, OF = S::PW / 4;
                const int of = (warp - 4) >> 2;
                const uint32_t mine = sa(smem) + (uint32_t)(((rank * OF + of) * SHARE * 128 + q * 32 + lane) * 4);
                asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
#pragma unroll
                for (int to = 0; to < SPLIT; ++to) {
                    uint32_t theirs;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(theirs) : "r"(mine), "r"(to));
#pragma unroll
                    for (int j = 0; j < SHARE; ++j) {
                        const int c = to * SHARE + j;
                        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(theirs + j * 512),
                                     "f"(c % 2 ? acc[c / 2].y : acc[c / 2].x)
                                     : "memory");
                    }
                }
                asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
                const float *from = reinterpret_cast<const float *>(smem) + of * SHARE * 128 + q * 32 + lane;
                const int own = m0 + c0 + rank * SHARE;
                o += (int64_t)rank * SHARE * p.ldo;
#pragma unroll
                for (int j = 0; j < SHARE; ++j, o += p.ldo) {
                    float sum = from[j * 128];
#pragma unroll
                    for (int r = 1; r < SPLIT; ++r) sum += from[(r * OF * SHARE + j) * 128];
                    if (good && n < p.N && own + j < p.M) *o = sum;
                }
            };
            if (split == 2) exchange(std::integral_constant<int, 2>());
            else exchange(std::integral_constant<int, 4>());
        }
    }
    if (split > 1 && warp < 4) {
        // the cluster's two barriers, for the warps without sums
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
        asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    __syncwarp();
    before_sync();
    __syncthreads();
    if (warp == 0) tmem_free(tmem, S::COLS);
    if (threadIdx.x == 0 && *abort_) atomicOr(p.err, 4);
}

template <int NB>
cudaError_t few_rows(const uint8_t *a, const uint8_t *w, const ProductArgs &p, int sms, cudaStream_t s) {
    using S = Few<NB>;
    CUtensorMap mw, ma;
    cudaError_t e = byte_map(&mw, w, p.N, p.K, S::BV);
    if (e == cudaSuccess) e = byte_map(&ma, a, p.M, p.K, NB);
    int device = 0;
    static bmc::SharedMemory shm;
    if (e == cudaSuccess) e = cudaGetDevice(&device);
    auto *k = few_rows_kernel<NB>;
    if (e == cudaSuccess) e = shm.allow(reinterpret_cast<const void *>(k), S::SMEM, device);
    if (e != cudaSuccess) return e;
    const int tiles = (p.N + S::BV - 1) / S::BV * ((p.M + NB - 1) / NB), KB = (p.K + BKB - 1) / BKB;
    // part of K each where tiles alone leave SMs idle: at least four blocks
    // (the sums, NB * 512 bytes, fit over any three stages).  Clusters of 8 are
    // slower: 16.2 us for 100 x 2048 x 4096 where those of 4 take 9.9.
    int split = 1;
    while (split < 4 && tiles * split * 2 <= sms && KB >= split * 2 * 4) split *= 2;
    const int stages = S::stages((KB + split - 1) / split);
    cudaLaunchConfig_t c{};
    cudaLaunchAttribute at[1];
    c.gridDim = dim3((unsigned)(split > 1 ? tiles * split : tiles < sms ? tiles : sms));
    c.blockDim = dim3(S::THREADS);
    c.dynamicSmemBytes = S::SMEM;
    c.stream = s;
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)split;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    c.attrs = at;
    c.numAttrs = split > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&c, k, mw, ma, p, stages, split);
}

// ---- many rows
//
// Persistent: CTA c takes tiles c, c + grid, ... of 128 x 128 (rows of a
// fastest, so CTAs running together share w tiles), in two pipelines of every
// other tile each: a thread that issues copies (warps 0, 1), one that issues
// MMAs (warps 2, 3), three stages, two tensor memory buffers and four warps
// that promote.  A promotion thread has a row of a and 128 columns, so one
// scale a block.  Promoting a block takes a warp longer than the tensor core
// needs for it, and a tile's sums take as long as several blocks to go out:
// with two pipelines, one works while the other waits.  2048 x 50257 x 2048
// takes 303 us alone and 350 among other work, under the power limit's clocks
// (1.39 and 1.21 PFLOP/s; 412 MB of stores), 300 when this was taken: 225 without the stores,
// 190 without the promotion's multiply-adds as well, 125 with one MMA of four;
// half the copies change nothing.  (One tile of 256 columns for all eight warps
// took 356 us, two groups behind one pipeline 327 when this took 322.)  128 sums and 64 values on
// their way from tensor memory take more registers than an equal share, so the
// first four warps give theirs up: 128 * 72 + 256 * 216 = 384 * 168, what the
// block was launched with.
constexpr int BM = 128, BN = 128, STAGES = 3, TBUF = 2;  // (of a pipeline)
constexpr int STAGE_BYTES = (BM + BN) * BKB;
constexpr int MANY_THREADS = 32 * (4 + 8);
constexpr int TURN = 36 * 16 * 4;  // a warp's 16 x 32 values on their way out, 16-byte words of 8 lanes in all banks
constexpr int KRING = 8;           // blocks whose scales a thread has at hand
constexpr size_t MANY_SMEM = 1024 + (size_t)2 * STAGES * STAGE_BYTES + 8 * TURN + KRING * 256 * 4 + 256;

__global__ void __launch_bounds__(MANY_THREADS, 1)
    many_rows_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                     const ProductArgs p) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    // (an offset, so that the compiler still knows it for shared memory)
    unsigned char *const smem = smem_raw + ((1024u - (sa(smem_raw) & 1023u)) & 1023u);
    unsigned char *const behind = smem + 2 * STAGES * STAGE_BYTES;
    // the pipeline of this thread, and its barriers
    // (from lane 0, so that the compiler knows it for one value a warp)
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int line = warp < 4 ? warp & 1 : (warp - 4) >> 2;
    uint64_t *const bars = reinterpret_cast<uint64_t *>(behind + 8 * TURN + KRING * 256 * 4);
    constexpr int BARS = 2 * STAGES + 2 * TBUF;
    uint64_t *const full = bars + line * BARS, *const empty = full + STAGES;
    uint64_t *const accf = empty + STAGES, *const acce = accf + TBUF;
    uint32_t *tslot = reinterpret_cast<uint32_t *>(bars + 2 * BARS);
    int *abort_ = reinterpret_cast<int *>(tslot + 1);
    unsigned char *const stages = smem + line * STAGES * STAGE_BYTES;
    const int MT = (p.M + BM - 1) / BM, NTL = (p.N + BN - 1) / BN, KB = (p.K + BKB - 1) / BKB;
    const int tiles = MT * NTL, step = gridDim.x;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2 * BARS; ++i) mbar_init(&bars[i], i % BARS < BARS - TBUF ? 1 : 4);
        *abort_ = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) tmem_alloc(tslot, 2 * TBUF * BN);
    before_sync();
    __syncthreads();
    after_sync();
    const uint32_t tmem = *tslot + (uint32_t)(line * TBUF * BN);
    auto fail = [&]() { atomicOr(abort_, 1); };
    auto aborted = [&]() { return *reinterpret_cast<volatile int *>(abort_) != 0; };

    const int first = blockIdx.x + line * step;
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp < 2 && lane == 0) {
            int s = 0, ph = 1, issued = 0;
            // Pipelines that all start at once all store at once.  Those with a
            // tile less than others start later, spread over half a tile's time
            // (2048 x 50257 x 2048: 324 us without, 304 so, 313 over three
            // quarters of it; never slower where tried).
            const int extra = tiles % (2 * step);
            if (extra > 0 && first >= extra && tiles > 2 * step) {
                const long long t0 = clock64(), late = (long long)(KB * 600 + 4400) * (first - extra) / (2 * step - extra);
                while (clock64() - t0 < late) {}
            }
            for (int t = first; t < tiles && !aborted(); t += 2 * step) {
                const int m0 = t % MT * BM, n0 = t / MT * BN;
                for (int kb = 0; kb < KB; ++kb) {
                    if (!mbar_wait(&empty[s], ph)) {  // (a fresh barrier is past phase 1)
                        fail();
                        break;
                    }
                    unsigned char *st = stages + s * STAGE_BYTES;
                    mbar_expect_tx(&full[s], STAGE_BYTES);
                    tma_load_2d(st, &tmA, kb * BKB, m0, &full[s]);
                    tma_load_2d(st + BM * BKB, &tmW, kb * BKB, n0, &full[s]);
                    ++issued;
                    if (++s == STAGES) {
                        s = 0;
                        ph ^= 1;
                    }
                }
            }
            if (aborted()) {  // no copy may outlive the CTA
                for (int i = min(issued, STAGES); i > 0; --i) {
                    if (--s < 0) {
                        s += STAGES;
                        ph ^= 1;
                    }
                    mbar_wait(&full[s], ph ^ 1);
                }
            }
        }
        if (warp >= 2 && lane == 0) {
            int g = 0, s = 0, ph = 0;
            for (int t = first; t < tiles && !aborted(); t += 2 * step) {
                for (int kb = 0; kb < KB; ++kb, ++g) {
                    const int b = g & 1;
                    if (!mbar_wait(&acce[b], (g / 2 + 1) & 1) || !mbar_wait(&full[s], ph)) {
                        fail();
                        break;
                    }
                    after_sync();
                    const uint32_t a0 = sa(stages + s * STAGE_BYTES), w0 = a0 + BM * BKB;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        umma_f8(tmem + (uint32_t)(b * BN), sdesc(a0 + k * 32), sdesc(w0 + k * 32), f8_desc(BN),
                                k > 0 ? 1u : 0u);
                    umma_commit(&empty[s]);
                    umma_commit(&accf[b]);
                    if (++s == STAGES) {
                        s = 0;
                        ph ^= 1;
                    }
                }
            }
            if (aborted() && g > 0) mbar_wait(&accf[(g - 1) & 1], ((g - 1) / 2) & 1);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int q = warp & 3;
        float *turn = reinterpret_cast<float *>(behind + (warp - 4) * TURN);
        // This thread's scale for each block, in a ring of its own: four blocks
        // are loaded while the four before are used, and multiplied only then
        // (a product right behind the loads would wait for them).  Rows and
        // tiles past the last take the last one's.
        float *kr = reinterpret_cast<float *>(behind + 8 * TURN) + threadIdx.x - 128;
        const float *pa = p.sa, *pw = p.sw;
        int ahead_t = first, ahead_kb = 0;
        float va[4], vw[4];
        auto load4 = [&]() {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (ahead_kb == 0) {
                    const int t = min(ahead_t, tiles - 1);
                    pa = p.sa + min(t % MT * BM + q * 32 + lane, p.M - 1);
                    pw = p.sw + (int64_t)(t / MT) * KB;
                }
                va[i] = *pa;
                vw[i] = *pw;
                pa += p.ld_scale;
                ++pw;
                if (++ahead_kb == KB) {
                    ahead_kb = 0;
                    ahead_t += 2 * step;
                }
            }
        };
        load4();
        int g = 0;
        for (int t = first; t < tiles && !aborted(); t += 2 * step) {
            const int m0 = t % MT * BM + q * 32, n0 = t / MT * BN;
            float acc[128];
#pragma unroll
            for (int j = 0; j < 128; ++j) acc[j] = 0.0f;
            bool good = true;
            for (int kb = 0; kb < KB; ++kb, ++g) {
                if (g % 4 == 0) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) kr[(g + i) % KRING * 256] = va[i] * vw[i];
                    load4();
                }
                const float k = kr[g % KRING * 256];
                const int b = g & 1;
                const bool ok = mbar_wait(&accf[b], (g / 2) & 1);
                if (__any_sync(0xffffffffu, !ok)) {
                    fail();
                    good = false;
                    break;
                }
                after_sync();
                const uint32_t tb = tmem + (uint32_t)(b * BN) + ((uint32_t)(q * 32) << 16);
#pragma unroll
                for (int c = 0; c < 128; c += 64) {
                    uint32_t v[2][32];
                    tmem_load(tb + c, v[0]);
                    tmem_load(tb + c + 32, v[1]);
                    tmem_wait(v[0]);
                    tmem_wait(v[1]);
                    if (c == 64) {  // the sums are read: the buffer is free
                        before_sync();
                        __syncwarp();
                        if (lane == 0) arrive(&acce[b]);
                    }
#pragma unroll
                    for (int j = 0; j < 64; ++j) acc[c + j] = fmaf(as_f(v[j / 32][j % 32]), k, acc[c + j]);
                }
            }
            // 32 columns of 16 rows at a time through shared memory: a store is
            // 32 consecutive values of a row, whatever the pitch (two rows of 16
            // took 6 % longer in all, whole 128-byte lines of rows staged in
            // full 60 %, as the warp's own work)
            const int rows = min(32, p.M - m0);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if (!good || rows <= 0 || n0 + c * 32 >= p.N) continue;
                const int n = n0 + c * 32 + lane;
#pragma unroll
                for (int r = 0; r < 32; r += 16) {
                    if ((lane & 16) == r) {
#pragma unroll
                        for (int j = 0; j < 32; j += 4)
                            *reinterpret_cast<float4 *>(turn + (lane & 15) * 36 + j) =
                                make_float4(acc[c * 32 + j], acc[c * 32 + j + 1], acc[c * 32 + j + 2], acc[c * 32 + j + 3]);
                    }
                    __syncwarp();
                    if (n < p.N) {
                        float *o = p.out + (int64_t)(m0 + r) * p.ldo + n;
                        if (rows == 32) {
#pragma unroll
                            for (int i = 0; i < 16; ++i, o += p.ldo) *o = turn[i * 36 + lane];
                        } else {
                            for (int i = 0; i < 16 && r + i < rows; ++i, o += p.ldo) *o = turn[i * 36 + lane];
                        }
                    }
                    __syncwarp();
                }
            }
        }
    }
    __syncwarp();
    before_sync();
    __syncthreads();
    if (warp == 0) tmem_free(*tslot, 2 * TBUF * BN);
    if (threadIdx.x == 0 && *abort_) atomicOr(p.err, 4);
}

cudaError_t many_rows(const uint8_t *a, const uint8_t *w, const ProductArgs &p, int sms, cudaStream_t s) {
    CUtensorMap mw, ma;
    cudaError_t e = byte_map(&mw, w, p.N, p.K, BN);
    if (e == cudaSuccess) e = byte_map(&ma, a, p.M, p.K, BM);
    int device = 0;
    static bmc::SharedMemory shm;
    if (e == cudaSuccess) e = cudaGetDevice(&device);
    if (e == cudaSuccess) e = shm.allow(reinterpret_cast<const void *>(many_rows_kernel), (int)MANY_SMEM, device);
    if (e != cudaSuccess) return e;
    const int64_t tiles = (int64_t)((p.M + BM - 1) / BM) * ((p.N + BN - 1) / BN);
    if (tiles > INT32_MAX / 2) return cudaErrorInvalidValue;
    return bmc::launch(many_rows_kernel, dim3((unsigned)(tiles < sms ? tiles : sms)), MANY_THREADS, MANY_SMEM, s, ma, mw, p);
}

cudaError_t product(const uint8_t *a, const uint8_t *w, const ProductArgs &p, int sms, cudaStream_t s) {
    if (p.M <= 16) return few_rows<16>(a, w, p, sms, s);
    if (p.M <= 32) return few_rows<32>(a, w, p, sms, s);
    if (p.M <= 64) return few_rows<64>(a, w, p, sms, s);
    if (p.M <= 96) return few_rows<96>(a, w, p, sms, s);
    if (p.M <= 128) return few_rows<128>(a, w, p, sms, s);
    // tiles that leave half the SMs idle: clusters with a part of K each (200 x
    // 2048 x 4096 in 11.3 us instead of 19.9)
    const int64_t tiles = (int64_t)((p.M + 127) / 128) * ((p.N + 127) / 128);
    if (tiles * 2 <= sms && p.K > 7 * BKB) return few_rows<128>(a, w, p, sms, s);
    return many_rows(a, w, p, sms, s);
}

bool misaligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

int check_d(int d) {
    if (d < 16 || d % 16 || d > 16384)
        return bm_detail_fail(BM_ERR_UNSUPPORTED, "d must be a multiple of 16, at most 16384");
    return BM_OK;
}

int check_rows(int rows, int n) {  // (so that rounding up to a tile stays in range)
    if (rows > INT32_MAX - 1024 || n > INT32_MAX - 1024)
        return bm_detail_fail(BM_ERR_UNSUPPORTED, "rows or n > 2^31 - 1025");
    return BM_OK;
}

int check_scale(const void *scale, int64_t ld_scale, int rows) {
    if (!scale || misaligned(scale, 16))
        return bm_detail_fail(BM_ERR_INVALID_ARG, "scales NULL or not 16-byte aligned");
    if (ld_scale < rows || ld_scale % 4)
        return bm_detail_fail(BM_ERR_INVALID_ARG, "ld_scale < rows or not a multiple of 4");
    return BM_OK;
}

int check_operands(const void *a, const void *w, const void *w_scale, const void *out) {
    if (!a || !w || !w_scale || !out)
        return bm_detail_fail(BM_ERR_INVALID_ARG, "a, w, w_scale and out must be non-NULL");
    if (misaligned(a, 16) || misaligned(w, 16) || misaligned(w_scale, 4) || misaligned(out, 4))
        return bm_detail_fail(BM_ERR_INVALID_ARG, "a or w not 16-byte, or w_scale or out not 4-byte aligned");
    return BM_OK;
}

}  // namespace
}  // namespace bml

extern "C" {

int bm_fp8_quantize(bm_ctx_t *ctx, const void *d_x, int type, int rows, int d, int64_t ldx,
                    const float *d_norm_w, uint8_t *d_q, float *d_scale, int64_t ld_scale,
                    void *stream) {
    if (!ctx) return bm_detail_fail(BM_ERR_INVALID_ARG, "ctx is NULL");
    if (type != BM_F32 && type != BM_BF16)
        return bm_detail_fail(BM_ERR_UNSUPPORTED, "type must be BM_F32 or BM_BF16");
    if (rows < 0) return bm_detail_fail(BM_ERR_INVALID_ARG, "rows < 0");
    int rc = bml::check_d(d);
    if (rc == BM_OK) rc = bml::check_rows(rows, 1);
    if (rc != BM_OK || rows == 0) return rc;
    if ((rc = bml::check_scale(d_scale, ld_scale, rows)) != BM_OK) return rc;
    if (!d_x || !d_q || ldx < d || ldx % 4)
        return bm_detail_fail(BM_ERR_INVALID_ARG, "x or q NULL, ldx < d or not a multiple of 4");
    if (bml::misaligned(d_x, type == BM_F32 ? 16 : 8) || bml::misaligned(d_q, 16) ||
        bml::misaligned(d_norm_w, 16))
        return bm_detail_fail(BM_ERR_INVALID_ARG, "x not aligned to 4 elements, or q or norm_w not 16-byte");
    int sms, *err;
    cudaStream_t s;
    bmc::DeviceGuard guard(bm_detail_ctx(ctx, &sms, &err, &s));
    BMC_CK(guard.error);
    if (stream) s = static_cast<cudaStream_t>(stream);
    const float *xf = static_cast<const float *>(d_x);
    const __nv_bfloat16 *xb = static_cast<const __nv_bfloat16 *>(d_x);
    cudaError_t e;
    if (type == BM_F32)
        e = d_norm_w ? bml::quantize<float, true>(xf, rows, d, ldx, d_norm_w, d_q, d_scale, ld_scale, s)
                     : bml::quantize<float, false>(xf, rows, d, ldx, nullptr, d_q, d_scale, ld_scale, s);
    else
        e = d_norm_w ? bml::quantize<__nv_bfloat16, true>(xb, rows, d, ldx, d_norm_w, d_q, d_scale, ld_scale, s)
                     : bml::quantize<__nv_bfloat16, false>(xb, rows, d, ldx, nullptr, d_q, d_scale, ld_scale, s);
    BMC_CK(e);
    return BM_OK;
}

int bm_fp8_product(bm_ctx_t *ctx, const uint8_t *d_a, const float *d_a_scale, int64_t ld_scale,
                   int rows, int d, const uint8_t *d_w, const float *d_w_scale, int n,
                   float *d_out, int64_t ldo, void *stream) {
    if (!ctx) return bm_detail_fail(BM_ERR_INVALID_ARG, "ctx is NULL");
    if (rows < 0 || n < 1 || ldo < n)
        return bm_detail_fail(BM_ERR_INVALID_ARG, "rows < 0, n < 1 or ldo < n");
    int rc = bml::check_d(d);
    if (rc == BM_OK) rc = bml::check_rows(rows, n);
    if (rc != BM_OK || rows == 0) return rc;
    if ((rc = bml::check_scale(d_a_scale, ld_scale, rows)) != BM_OK) return rc;
    if ((rc = bml::check_operands(d_a, d_w, d_w_scale, d_out)) != BM_OK) return rc;
    int sms, *err;
    cudaStream_t s;
    bmc::DeviceGuard guard(bm_detail_ctx(ctx, &sms, &err, &s));
    BMC_CK(guard.error);
    if (stream) s = static_cast<cudaStream_t>(stream);
    const bml::ProductArgs p{d_a_scale, d_w_scale, ld_scale, ldo, d_out, rows, d, n, err};
    BMC_CK(bml::product(d_a, d_w, p, sms, s));
    return BM_OK;
}

int bm_fp8_logits(bm_ctx_t *ctx, const float *d_hidden, int B, int d_model, const float *d_norm_w,
                  const uint8_t *d_w, const float *d_w_scale, int V, float *d_logits, int64_t ld,
                  void *stream) {
    if (!ctx) return bm_detail_fail(BM_ERR_INVALID_ARG, "ctx is NULL");
    if (B < 0 || V < 1 || ld < V) return bm_detail_fail(BM_ERR_INVALID_ARG, "B < 0, V < 1 or ld < V");
    int rc = bml::check_d(d_model);
    if (rc == BM_OK) rc = bml::check_rows(B, V);
    if (rc != BM_OK || B == 0) return rc;
    if (!d_hidden || bml::misaligned(d_hidden, 16) || bml::misaligned(d_norm_w, 16))
        return bm_detail_fail(BM_ERR_INVALID_ARG, "hidden NULL, or hidden or norm weight not 16-byte aligned");
    // (the product's too, before anything is launched)
    if ((rc = bml::check_operands(d_hidden, d_w, d_w_scale, d_logits)) != BM_OK) return rc;
    int sms, *err;
    cudaStream_t s;
    bmc::DeviceGuard guard(bm_detail_ctx(ctx, &sms, &err, &s));
    BMC_CK(guard.error);
    const int64_t lds = ((int64_t)B + 3) / 4 * 4;
    const size_t qb = ((size_t)B * d_model + 255) / 256 * 256;
    void *work;
    rc = bm_detail_work(ctx, BM_WORK_FP8, qb + (size_t)lds * ((d_model + 127) / 128) * 4, &work);
    if (rc != BM_OK) return rc;
    uint8_t *q = static_cast<uint8_t *>(work);
    float *sc = reinterpret_cast<float *>(q + qb);
    rc = bm_fp8_quantize(ctx, d_hidden, BM_F32, B, d_model, d_model, d_norm_w, q, sc, lds, stream);
    if (rc != BM_OK) return rc;
    return bm_fp8_product(ctx, q, sc, lds, B, d_model, d_w, d_w_scale, V, d_logits, ld, stream);
}

// The stages of a few-rows tile of nb rows with `blocks` blocks of K a CTA, 0
// for other nb.  Not part of the public ABI: for tests on the host.
int bm_detail_fp8_stages(int nb, int blocks) {
    switch (nb) {
        case 16: return bml::Few<16>::stages(blocks);
        case 32: return bml::Few<32>::stages(blocks);
        case 64: return bml::Few<64>::stages(blocks);
        case 96: return bml::Few<96>::stages(blocks);
        case 128: return bml::Few<128>::stages(blocks);
        default: return 0;
    }
}

}  // extern "C"
