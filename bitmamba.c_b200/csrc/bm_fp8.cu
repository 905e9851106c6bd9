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
// The tile is 128 rows of w (the accumulator's lanes) by NB rows of a (its
// columns).  With w on the lanes a warp's store covers 32 consecutive outputs
// of one row whatever the row pitch, the w scale is one value per tile and
// block, and few rows of a cost a narrow tile instead of a padded one.
#include <cstdint>

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

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// TPR threads per row: a warp's 32 groups of 4 columns are one block of 128.
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
        const float rms = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(s, (float)d) + 1e-6f));
#pragma unroll
        for (int i = 0; i < QV; ++i) {
            const int col = 4 * (t + i * TPR);
            if (col < d) {
                const float4 w = load4(norm_w + col);
                v[i] = make_float4(v[i].x * rms * w.x, v[i].y * rms * w.y, v[i].z * rms * w.z,
                                   v[i].w * rms * w.w);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < QV; ++i) {
        const int col = 4 * (t + i * TPR);
        float top = max_nan(max_nan(fabsf(v[i].x), fabsf(v[i].y)), max_nan(fabsf(v[i].z), fabsf(v[i].w)));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
        // !(top <= tiny): a NaN stays one
        const float sc = !(top <= 0x1p-100f) ? __fdiv_rn(top, 448.0f) : 1.0f;
        if (live && col < d) {
            const __nv_fp8x4_e4m3 r(make_float4(__fdiv_rn(v[i].x, sc), __fdiv_rn(v[i].y, sc),
                                                __fdiv_rn(v[i].z, sc), __fdiv_rn(v[i].w, sc)));
            *reinterpret_cast<uint32_t *>(q + (int64_t)row * d + col) = r.__x;
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
        quantize_kernel<T, TPR, NORM><<<(rows + per - 1) / per, TPR < 256 ? 256 : TPR, 0, s>>>( \
            x, rows, d, ldx, norm_w, q, scale, ld_scale);                                       \
        return cudaGetLastError();                                                              \
    }
    BM_Q(32)
    BM_Q(128)
    BM_Q(256)
    BM_Q(1024)
#undef BM_Q
    return cudaErrorInvalidValue;
}

// -------------------------------------------------------------- product --

constexpr int BV = 128, BKB = 128;  // rows of w per tile, bytes (columns) of K per block
constexpr int RING = 4;             // blocks of scales in shared memory

template <int NB>
struct Shape {
    static constexpr int PW = NB >= 64 ? 8 : 4;      // promotion warps
    static constexpr int CW = NB / (PW / 4);         // columns per promotion warp
    static constexpr int TB = NB == 256 ? 2 : 4;     // tensor memory buffers
    static constexpr int COLS = TB * NB;             // a power of two >= 32
    static constexpr int STAGE = BV * BKB + NB * BKB;
    static constexpr int STAGES = (192 * 1024) / STAGE;
    static constexpr int THREADS = 32 * (3 + PW);
    static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE + RING * NB * 4 + 512;
};

__device__ __forceinline__ void umma_f8(uint32_t tmem, uint64_t da, uint64_t db, uint32_t idesc,
                                        uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(tmem),
        "l"(da), "l"(db), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
        "%11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void arrive(uint64_t *b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(sa(b)) : "memory");
}

struct ProductArgs {
    const float *sa, *sw;
    int64_t ld_scale, ldo;
    float *out;
    int M, K, N;
    int *err;
};

// Persistent: CTA c takes tiles c, c + grid, ... (rows of a fastest, so CTAs
// running together share w tiles).  Warp 0 lane 0 is the TMA producer, warp 1
// lane 0 issues the MMAs, warp 2 multiplies and stages the scales, the
// promotion warps add.
template <int NB>
__global__ void __launch_bounds__(Shape<NB>::THREADS, 1)
    product_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmA,
                   const ProductArgs p) {
    using S = Shape<NB>;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    float *ring = reinterpret_cast<float *>(smem + S::STAGES * S::STAGE);
    uint64_t *full = reinterpret_cast<uint64_t *>(ring + RING * NB);
    uint64_t *empty = full + S::STAGES;
    uint64_t *accf = empty + S::STAGES;  // [TB] a block's sums are complete
    uint64_t *acce = accf + S::TB;       // [TB] they are read
    uint64_t *sf = acce + S::TB;         // [RING] scales staged
    uint64_t *se = sf + RING;            // [RING] scales read
    uint32_t *tslot = reinterpret_cast<uint32_t *>(se + RING);
    int *abort_ = reinterpret_cast<int *>(tslot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int MT = (p.M + NB - 1) / NB, NT = (p.N + BV - 1) / BV, KB = (p.K + BKB - 1) / BKB;
    const int tiles = MT * NT;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::STAGES; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < S::TB; ++i) {
            mbar_init(&accf[i], 1);
            mbar_init(&acce[i], S::PW);
        }
        for (int i = 0; i < RING; ++i) {
            mbar_init(&sf[i], 1);
            mbar_init(&se[i], S::PW);
        }
        *abort_ = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         sa(tslot)),
                     "r"((uint32_t)S::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tslot;
    auto fail = [&]() { atomicOr(abort_, 1); };
    auto aborted = [&]() { return *reinterpret_cast<volatile int *>(abort_) != 0; };

    if (threadIdx.x == 0) {
        int g = 0;
        for (int t = blockIdx.x; t < tiles && !aborted(); t += gridDim.x) {
            const int m0 = (t % MT) * NB, n0 = (t / MT) * BV;
            for (int kb = 0; kb < KB; ++kb, ++g) {
                const int s = g % S::STAGES;
                if (g >= S::STAGES && !mbar_wait(&empty[s], ((g / S::STAGES) - 1) & 1)) {
                    fail();
                    break;
                }
                unsigned char *st = smem + (size_t)s * S::STAGE;
                mbar_expect_tx(&full[s], S::STAGE);
                tma_load_2d(st, &tmW, kb * BKB, n0, &full[s]);
                tma_load_2d(st + BV * BKB, &tmA, kb * BKB, m0, &full[s]);
            }
        }
    } else if (threadIdx.x == 32) {
        // e4m3 x e4m3 -> fp32 (formats 0, D format 1), both K-major
        const uint32_t idesc = (1u << 4) | ((uint32_t)(NB >> 3) << 17) | ((uint32_t)(BV >> 4) << 24);
        int g = 0;
        for (int t = blockIdx.x; t < tiles && !aborted(); t += gridDim.x) {
            for (int kb = 0; kb < KB; ++kb, ++g) {
                const int s = g % S::STAGES, b = g % S::TB;
                if ((g >= S::TB && !mbar_wait(&acce[b], ((g / S::TB) - 1) & 1)) ||
                    !mbar_wait(&full[s], (g / S::STAGES) & 1)) {
                    fail();
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t w0 = sa(smem + (size_t)s * S::STAGE), a0 = w0 + BV * BKB;
                const uint32_t acc = tmem + (uint32_t)(b * NB);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    umma_f8(acc, sdesc(w0 + k * 32), sdesc(a0 + k * 32), idesc, k > 0 ? 1u : 0u);
                umma_commit(&empty[s]);
                umma_commit(&accf[b]);
            }
        }
    } else if (warp == 2) {
        int g = 0;
        for (int t = blockIdx.x; t < tiles && !aborted(); t += gridDim.x) {
            const int m0 = (t % MT) * NB, nt = t / MT;
            for (int kb = 0; kb < KB; ++kb, ++g) {
                const int r = g % RING;
                const bool ok = g < RING || mbar_wait(&se[r], ((g / RING) - 1) & 1);
                if (__any_sync(0xffffffffu, !ok)) {
                    fail();
                    break;
                }
                const float sw = p.sw[(int64_t)nt * KB + kb];
                for (int c = lane; c < NB; c += 32)
                    ring[r * NB + c] = m0 + c < p.M ? p.sa[kb * p.ld_scale + m0 + c] * sw : 0.0f;
                __syncwarp();
                if (lane == 0) arrive(&sf[r]);
            }
        }
    } else if (warp >= 3) {
        const int q = warp & 3, c0 = ((warp - 3) >> 2) * S::CW;
        int g = 0;
        for (int t = blockIdx.x; t < tiles && !aborted(); t += gridDim.x) {
            const int m0 = (t % MT) * NB, n0 = (t / MT) * BV;
            float acc[S::CW];
#pragma unroll
            for (int j = 0; j < S::CW; ++j) acc[j] = 0.0f;
            bool good = true;
            for (int kb = 0; kb < KB; ++kb, ++g) {
                const int b = g % S::TB, r = g % RING;
                const bool ok = mbar_wait(&sf[r], (g / RING) & 1) && mbar_wait(&accf[b], (g / S::TB) & 1);
                if (__any_sync(0xffffffffu, !ok)) {
                    fail();
                    good = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t tb = tmem + (uint32_t)(b * NB + c0) + ((uint32_t)(q * 32) << 16);
                const float *sc = ring + r * NB + c0;
#pragma unroll
                for (int c = 0; c < S::CW; c += 16) {
                    uint32_t v[16];
                    tmem_ld16(tb + c, v);
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        acc[c + j] = fmaf(__uint_as_float(v[j]), sc[c + j], acc[c + j]);
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    arrive(&acce[b]);
                    arrive(&se[r]);
                }
            }
            const int n = n0 + q * 32 + lane;
            if (good && n < p.N) {
                float *o = p.out + (int64_t)(m0 + c0) * p.ldo + n;
#pragma unroll
                for (int j = 0; j < S::CW; ++j, o += p.ldo)
                    if (m0 + c0 + j < p.M) *o = acc[j];
            }
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 0)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                     "r"((uint32_t)S::COLS)
                     : "memory");
    if (threadIdx.x == 0 && *abort_) atomicOr(p.err, 4);
}

template <int NB>
cudaError_t launch_product(const uint8_t *a, const uint8_t *w, const ProductArgs &p, int sms,
                           cudaStream_t s) {
    using S = Shape<NB>;
    CUtensorMap mw, ma;
    cudaError_t e = byte_map(&mw, w, p.N, p.K, BV);
    if (e == cudaSuccess) e = byte_map(&ma, a, p.M, p.K, NB);
    int device = 0;
    static bmc::SharedMemory shm;
    if (e == cudaSuccess) e = cudaGetDevice(&device);
    if (e == cudaSuccess)
        e = shm.allow(reinterpret_cast<const void *>(product_kernel<NB>), (int)S::SMEM, device);
    if (e != cudaSuccess) return e;
    const int64_t tiles = (int64_t)((p.M + NB - 1) / NB) * ((p.N + BV - 1) / BV);
    if (tiles > INT32_MAX / 2) return cudaErrorInvalidValue;
    product_kernel<NB><<<(int)(tiles < sms ? tiles : sms), S::THREADS, S::SMEM, s>>>(mw, ma, p);
    return cudaGetLastError();
}

cudaError_t product(const uint8_t *a, const uint8_t *w, const ProductArgs &p, int sms,
                    cudaStream_t s) {
    if (p.M <= 16) return launch_product<16>(a, w, p, sms, s);
    if (p.M <= 32) return launch_product<32>(a, w, p, sms, s);
    if (p.M <= 64) return launch_product<64>(a, w, p, sms, s);
    if (p.M <= 128) return launch_product<128>(a, w, p, sms, s);
    return launch_product<256>(a, w, p, sms, s);
}

bool misaligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

int check_d(int d) {
    if (d < 16 || d % 16 || d > 16384)
        return bm_detail_fail(BM_ERR_UNSUPPORTED, "d must be a multiple of 16, at most 16384");
    return BM_OK;
}

int check_scale(const void *scale, int64_t ld_scale, int rows) {
    if (!scale || misaligned(scale, 16))
        return bm_detail_fail(BM_ERR_INVALID_ARG, "scales NULL or not 16-byte aligned");
    if (ld_scale < rows || ld_scale % 4)
        return bm_detail_fail(BM_ERR_INVALID_ARG, "ld_scale < rows or not a multiple of 4");
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
    if (rc != BM_OK || rows == 0) return rc;
    if ((rc = bml::check_scale(d_a_scale, ld_scale, rows)) != BM_OK) return rc;
    if (!d_a || !d_w || !d_w_scale || !d_out)
        return bm_detail_fail(BM_ERR_INVALID_ARG, "a, w, w_scale and out must be non-NULL");
    if (bml::misaligned(d_a, 16) || bml::misaligned(d_w, 16) || bml::misaligned(d_w_scale, 4) ||
        bml::misaligned(d_out, 4))
        return bm_detail_fail(BM_ERR_INVALID_ARG, "a or w not 16-byte, or w_scale or out not 4-byte aligned");
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
    if (rc != BM_OK || B == 0) return rc;
    if (!d_hidden || bml::misaligned(d_hidden, 16) || bml::misaligned(d_norm_w, 16))
        return bm_detail_fail(BM_ERR_INVALID_ARG, "hidden NULL, or hidden or norm weight not 16-byte aligned");
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

}  // extern "C"
