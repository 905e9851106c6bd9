// The state space mixer between a layer's projections: short causal
// convolution, selective scan and gate, for prompts (bm_ssm_prefill) and
// single tokens (bm_ssm_step).  The formulas stand in include/bm_sampler.h;
// the layer loop they serve is jserv/bitmamba.c src/block.c:272-448.
//
// Everything is evaluated in fp32.  exp and log of the head scalars (a step's
// decay multiplies up over a whole sequence) are the full-precision functions;
// the two silu of each element use ex2.approx and rcp.approx, whose errors (2
// and 1 ulp) are not multiplied up.
#include <climits>
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "bm_ctx.cuh"
#include "bm_sampler.h"

namespace {

struct Layer {
    int H, P, C, n_slots;
    const float *conv_w, *conv_b, *dt_bias, *a_log, *d;
    void *conv;
    float *h;
};

struct Args {
    Layer l;
    const void *x, *z, *b, *c, *dt;
    int64_t ld;
    int rows;
    const int32_t *slots;
    void *y;
    int64_t ldy;
    // prompts
    const int64_t *off;
    int n_seq;
    const int32_t *fresh;
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

__device__ __forceinline__ float silu(float v) { return __fdividef(v, 1.0f + __expf(-v)); }
__device__ __forceinline__ float softplus(float v) {
    return fmaxf(v, 0.0f) + log1pf(expf(-fabsf(v)));
}

// A head's scalars for one token: the decay a, the input's factor g = d B and
// the output's C.
struct Head {
    float a, g, c;
};
template <typename T>
__device__ __forceinline__ Head head_of(const Args &p, int64_t row, int h) {
    const int64_t at = row * p.ld + h;
    const float d = softplus(to_f(static_cast<const T *>(p.dt)[at]) + p.l.dt_bias[h]);
    Head r;
    r.a = expf(-expf(p.l.a_log[h]) * d);
    r.g = d * to_f(static_cast<const T *>(p.b)[at]);
    r.c = to_f(static_cast<const T *>(p.c)[at]);
    return r;
}

// One thread per channel of a sequence, token after token.
template <typename T>
__global__ void __launch_bounds__(128) prefill_kernel(const Args p) {
    const int ch = blockIdx.x * 128 + threadIdx.x, s = blockIdx.y;
    if (ch >= p.l.C) return;
    const int slot = p.slots ? p.slots[s] : s;
    if (slot < 0 || slot >= p.l.n_slots) return;
    const int64_t r0 = max((int64_t)0, p.off[s]), r1 = min((int64_t)p.rows, p.off[s + 1]);
    const bool fresh = !p.fresh || p.fresh[s] != 0;
    T *cs = static_cast<T *>(p.l.conv) + ((int64_t)slot * 3) * p.l.C + ch;
    float *hs = p.l.h + (int64_t)slot * p.l.C + ch;
    const T zero = from_f<T>(0.0f);
    T x3 = fresh ? zero : cs[0], x2 = fresh ? zero : cs[p.l.C], x1 = fresh ? zero : cs[2 * p.l.C];
    float h = fresh ? 0.0f : *hs;
    const float4 w = reinterpret_cast<const float4 *>(p.l.conv_w)[ch];
    const float bias = p.l.conv_b[ch], d = p.l.d[ch];
    const int hd = ch / p.l.P;
    for (int64_t r = r0; r < r1; ++r) {
        const Head k = head_of<T>(p, r, hd);
        const T x0 = static_cast<const T *>(p.x)[r * p.ld + ch];
        const float u = silu(fmaf(
            w.w, to_f(x0), fmaf(w.z, to_f(x1), fmaf(w.y, to_f(x2), fmaf(w.x, to_f(x3), bias)))));
        h = fmaf(k.a, h, k.g * u);
        float y = fmaf(k.c, h, d * u);
        if (p.z) y *= silu(to_f(static_cast<const T *>(p.z)[r * p.ld + ch]));
        static_cast<T *>(p.y)[r * p.ldy + ch] = from_f<T>(y);
        x3 = x2;
        x2 = x1;
        x1 = x0;
    }
    cs[0] = x3;
    cs[p.l.C] = x2;
    cs[2 * p.l.C] = x1;
    *hs = h;
}

template <typename T>
__global__ void __launch_bounds__(128) step_kernel(const Args p) {
    const int ch = blockIdx.x * 128 + threadIdx.x;
    if (ch >= p.l.C) return;
    const float4 w = reinterpret_cast<const float4 *>(p.l.conv_w)[ch];
    const float bias = p.l.conv_b[ch], d = p.l.d[ch];
    const int hd = ch / p.l.P;
    for (int r = blockIdx.y; r < p.rows; r += gridDim.y) {
        const int slot = p.slots ? p.slots[r] : r;
        if (slot < 0 || slot >= p.l.n_slots) continue;
        T *cs = static_cast<T *>(p.l.conv) + ((int64_t)slot * 3) * p.l.C + ch;
        float *hs = p.l.h + (int64_t)slot * p.l.C + ch;
        const Head k = head_of<T>(p, r, hd);
        const T x3 = cs[0], x2 = cs[p.l.C], x1 = cs[2 * p.l.C];
        const T x0 = static_cast<const T *>(p.x)[r * p.ld + ch];
        const float u = silu(fmaf(
            w.w, to_f(x0), fmaf(w.z, to_f(x1), fmaf(w.y, to_f(x2), fmaf(w.x, to_f(x3), bias)))));
        const float h = fmaf(k.a, *hs, k.g * u);
        float y = fmaf(k.c, h, d * u);
        if (p.z) y *= silu(to_f(static_cast<const T *>(p.z)[r * p.ld + ch]));
        static_cast<T *>(p.y)[r * p.ldy + ch] = from_f<T>(y);
        cs[0] = x2;
        cs[p.l.C] = x1;
        cs[2 * p.l.C] = x0;
        *hs = h;
    }
}

bool misaligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

// The checks that both calls share; fills what they have in common.
int common(bm_ctx_t *ctx, const bm_ssm_layer_t *l, const void *x, const void *z, const void *b,
           const void *c, const void *dt, int64_t ld, int rows, const int32_t *slots, void *y,
           int64_t ldy, Args *out) {
    if (!ctx) return bm_detail_fail(BM_ERR_INVALID_ARG, "ctx is NULL");
    if (!l) return bm_detail_fail(BM_ERR_INVALID_ARG, "layer is NULL");
    if (l->type != BM_F32 && l->type != BM_BF16)
        return bm_detail_fail(BM_ERR_UNSUPPORTED, "layer type must be BM_F32 or BM_BF16");
    if (l->n_heads < 1 || l->head_dim < 1 || l->n_slots < 1)
        return bm_detail_fail(BM_ERR_INVALID_ARG, "n_heads, head_dim or n_slots < 1");
    if ((int64_t)l->n_heads * l->head_dim > (1 << 20))
        return bm_detail_fail(BM_ERR_UNSUPPORTED, "n_heads * head_dim > 2^20");
    if (!l->conv_w || !l->conv_b || !l->dt_bias || !l->a_log || !l->d || !l->conv_state ||
        !l->h_state)
        return bm_detail_fail(BM_ERR_INVALID_ARG, "layer weights and states must be non-NULL");
    const size_t e = l->type == BM_F32 ? 4 : 2;
    if (misaligned(l->conv_w, 16) || misaligned(l->conv_b, 4) || misaligned(l->dt_bias, 4) ||
        misaligned(l->a_log, 4) || misaligned(l->d, 4) || misaligned(l->conv_state, e) ||
        misaligned(l->h_state, 4))
        return bm_detail_fail(BM_ERR_INVALID_ARG,
                              "conv_w not 16-byte, or weights or states not element aligned");
    if (rows < 0) return bm_detail_fail(BM_ERR_INVALID_ARG, "rows < 0");
    const int C = l->n_heads * l->head_dim;
    if (rows > 0) {
        if (!x || !b || !c || !dt || !y)
            return bm_detail_fail(BM_ERR_INVALID_ARG, "x, b, c, dt and y must be non-NULL");
        if (misaligned(x, e) || misaligned(z, e) || misaligned(b, e) || misaligned(c, e) ||
            misaligned(dt, e) || misaligned(y, e))
            return bm_detail_fail(BM_ERR_INVALID_ARG, "x, z, b, c, dt or y not element aligned");
        if (ld < C || ldy < C)
            return bm_detail_fail(BM_ERR_INVALID_ARG, "ld or ldy < n_heads * head_dim");
    }
    out->l = Layer{l->n_heads, l->head_dim, C,       l->n_slots, l->conv_w, l->conv_b,
                   l->dt_bias, l->a_log,    l->d,    l->conv_state, l->h_state};
    out->x = x;
    out->z = z;
    out->b = b;
    out->c = c;
    out->dt = dt;
    out->ld = ld;
    out->rows = rows;
    out->slots = slots;
    out->y = y;
    out->ldy = ldy;
    return BM_OK;
}

}  // namespace

extern "C" {

int bm_ssm_prefill(bm_ctx_t *ctx, const bm_ssm_layer_t *layer, const void *d_x, const void *d_z,
                   const void *d_b, const void *d_c, const void *d_dt, int64_t ld, int rows,
                   const int64_t *d_seq_off, int n_seq, const int32_t *d_slots,
                   const int32_t *d_fresh, void *d_y, int64_t ldy, void *stream) {
    Args a{};
    const int rc =
        common(ctx, layer, d_x, d_z, d_b, d_c, d_dt, ld, rows, d_slots, d_y, ldy, &a);
    if (rc != BM_OK) return rc;
    if (n_seq < 0 || n_seq > layer->n_slots)
        return bm_detail_fail(BM_ERR_INVALID_ARG, "n_seq < 0 or more sequences than slots");
    if (n_seq == 0) return BM_OK;
    if (!d_seq_off || misaligned(d_seq_off, 8))
        return bm_detail_fail(BM_ERR_INVALID_ARG, "seq_off NULL or not 8-byte aligned");
    if (n_seq > 65535) return bm_detail_fail(BM_ERR_UNSUPPORTED, "n_seq > 65535");
    a.off = d_seq_off;
    a.n_seq = n_seq;
    a.fresh = d_fresh;
    int sms, *err;
    cudaStream_t s;
    bmc::DeviceGuard guard(bm_detail_ctx(ctx, &sms, &err, &s));
    BMC_CK(guard.error);
    if (stream) s = static_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)((a.l.C + 127) / 128), (unsigned)n_seq);
    if (layer->type == BM_F32)
        prefill_kernel<float><<<grid, 128, 0, s>>>(a);
    else
        prefill_kernel<__nv_bfloat16><<<grid, 128, 0, s>>>(a);
    BMC_CK(cudaGetLastError());
    return BM_OK;
}

int bm_ssm_step(bm_ctx_t *ctx, const bm_ssm_layer_t *layer, const void *d_x, const void *d_z,
                const void *d_b, const void *d_c, const void *d_dt, int64_t ld, int rows,
                const int32_t *d_slots, void *d_y, int64_t ldy, void *stream) {
    Args a{};
    const int rc =
        common(ctx, layer, d_x, d_z, d_b, d_c, d_dt, ld, rows, d_slots, d_y, ldy, &a);
    if (rc != BM_OK || rows == 0) return rc;
    if (rows > layer->n_slots)
        return bm_detail_fail(BM_ERR_INVALID_ARG, "more rows than slots");
    int sms, *err;
    cudaStream_t s;
    bmc::DeviceGuard guard(bm_detail_ctx(ctx, &sms, &err, &s));
    BMC_CK(guard.error);
    if (stream) s = static_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)((a.l.C + 127) / 128), (unsigned)(rows < 65535 ? rows : 65535));
    if (layer->type == BM_F32)
        step_kernel<float><<<grid, 128, 0, s>>>(a);
    else
        step_kernel<__nv_bfloat16><<<grid, 128, 0, s>>>(a);
    BMC_CK(cudaGetLastError());
    return BM_OK;
}

}  // extern "C"
