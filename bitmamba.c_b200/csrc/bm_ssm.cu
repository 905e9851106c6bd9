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

// One channel or two: two take the packed fp32 instructions, which do the
// arithmetic of a pair in one issue slot.
template <int VEC>
struct Vec;
template <>
struct Vec<1> {
    using type = float;
};
template <>
struct Vec<2> {
    using type = float2;
};
__device__ __forceinline__ float vfma(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float2 vfma(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float vmul(float a, float b) { return a * b; }
__device__ __forceinline__ float2 vmul(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float vadd(float a, float b) { return a + b; }
__device__ __forceinline__ float2 vadd(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ void vset(float &v, float a, float) { v = a; }
__device__ __forceinline__ void vset(float2 &v, float a, float b) { v = make_float2(a, b); }
__device__ __forceinline__ float lane0(float v) { return v; }
__device__ __forceinline__ float lane0(float2 v) { return v.x; }
__device__ __forceinline__ float lane1(float v) { return v; }
__device__ __forceinline__ float lane1(float2 v) { return v.y; }
__device__ __forceinline__ float ex2(float v) {
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(v));
    return v;
}
__device__ __forceinline__ float rcp(float v) {
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(v));
    return v;
}
// v / (1 + e^-v): where e^-v overflows the quotient's limit, -0
template <typename V>
__device__ __forceinline__ V silu(V v) {
    V k, one, e;
    vset(k, -1.44269504f, -1.44269504f);
    vset(one, 1.0f, 1.0f);
    const V t = vmul(v, k);
    vset(e, ex2(lane0(t)), ex2(lane1(t)));
    e = vadd(e, one);
    vset(e, rcp(lane0(e)), rcp(lane1(e)));
    return vmul(v, e);
}
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

// ---------------------------------------------------------------- prompts --
//
// The token axis of all sequences together is cut into tiles of ST * LC rows; a
// CTA takes one tile of CG * VEC channels, a thread VEC channels of one of the
// tile's ST parts from its first row to its last, with the convolution's
// window, the state and the outputs in registers.  The recurrence is linear,
// so a part first runs from a zero state:
//   s_t = local_t + (a_first ... a_t) * s_in,    s_out = S + A * s_in
// and the C s_t of its outputs is completed when s_in arrives: outputs wait
// in registers, x and z are read once and y is written once.  The parts of a
// tile are joined in shared memory, the tiles through published words.
//
// Narrow and long tiles (64 or 128 bytes of a row) keep few tiles of the same
// channels in flight and the chain over them short: with 128 threads side by
// side and tiles of 32 rows, 37 tiles of each channel were in flight and the
// look-back cost more than the scan (65536 x 4096 bf16: 1.98 ms).
//
// s_in comes from the tiles before (CTAs take tiles in order, by a ticket, so
// whoever is waited for is running or done).  Each tile publishes its
// channels' S and its heads' A, then looks back for the nearest tile whose
// s_out is final (it holds a sequence start, or has completed its own
// look-back) and applies the A and S of the tiles in between in order.  That
// is the chain s = A s + S that each of them applies too, so the result does
// not depend on how far back the final word was.
//
// A value is published as 8 bytes {tag, value} written at once, tag = 2 *
// epoch + (final or not): whoever reads the launch's tag has the value.  (16
// bytes in one relaxed b128 access were seen torn here: halves of two
// successive stores.)  The epoch is a counter in the workspace that the
// launch's last CTA advances, so nothing is cleared between launches or graph
// replays; a tag comes again after 2^31 launches.

constexpr unsigned long long WAIT_NS = 2000000000ull;  // bounded waits: 2 s

struct Control {
    unsigned ticket, done, epoch;
};
constexpr size_t CONTROL_BYTES = 256;

// The words of one or two channels: {tag, S} each.
using Word64 = unsigned long long;
template <typename V>
struct Words;
template <>
struct Words<float> {
    unsigned tag, tag1;
    float s;
};
template <>
struct Words<float2> {
    unsigned tag, tag1;
    float2 s;
};
__device__ __forceinline__ Word64 join(unsigned tag, float s) {
    return tag | ((Word64)__float_as_uint(s) << 32);
}
__device__ __forceinline__ void load_words(const Word64 *p, Words<float> &r) {
    Word64 w;
    asm volatile("ld.relaxed.gpu.global.b64 %0, [%1];" : "=l"(w) : "l"(p) : "memory");
    r.tag = r.tag1 = (unsigned)w;
    r.s = __uint_as_float((unsigned)(w >> 32));
}
__device__ __forceinline__ void load_words(const Word64 *p, Words<float2> &r) {
    Word64 w0, w1;
    asm volatile("ld.relaxed.gpu.global.v2.b64 {%0, %1}, [%2];" : "=l"(w0), "=l"(w1) : "l"(p) : "memory");
    r.tag = (unsigned)w0;
    r.tag1 = (unsigned)w1;
    r.s = make_float2(__uint_as_float((unsigned)(w0 >> 32)), __uint_as_float((unsigned)(w1 >> 32)));
}
__device__ __forceinline__ void store_words(Word64 *p, unsigned tag, float s) {
    asm volatile("st.relaxed.gpu.global.b64 [%0], %1;" ::"l"(p), "l"(join(tag, s)) : "memory");
}
__device__ __forceinline__ void store_words(Word64 *p, unsigned tag, float2 s) {
    asm volatile("st.relaxed.gpu.global.v2.b64 [%0], {%1, %2};" ::"l"(p), "l"(join(tag, s.x)),
                 "l"(join(tag, s.y))
                 : "memory");
}
__device__ __forceinline__ unsigned long long gtimer() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

// Copies to shared memory, each thread for itself: 4 bytes asynchronously, a
// 2-byte element through a register.
__device__ __forceinline__ void stage(void *dst, const void *src, float) {
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(d), "l"(src) : "memory");
}
__device__ __forceinline__ void stage(void *dst, const void *src, float2) {
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(d), "l"(src) : "memory");
}
__device__ __forceinline__ void stage(void *dst, const void *src, uint32_t) { stage(dst, src, 0.0f); }
__device__ __forceinline__ void stage(void *dst, const void *src, __nv_bfloat16) {
    *static_cast<__nv_bfloat16 *>(dst) = *static_cast<const __nv_bfloat16 *>(src);
}
template <int N>
__device__ __forceinline__ void stage_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void stage_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// VEC consecutive elements as they lie in memory, and as fp32.
template <typename T, int VEC>
struct Raw;
template <typename T>
struct Raw<T, 1> {
    using Word = T;
    T v;
    __device__ __forceinline__ void zero() { v = from_f<T>(0.0f); }
    __device__ __forceinline__ float get() const { return to_f(v); }
};
template <>
struct Raw<float, 2> {
    using Word = float2;
    float2 v;
    __device__ __forceinline__ void zero() { v = make_float2(0.0f, 0.0f); }
    __device__ __forceinline__ float2 get() const { return v; }
};
template <>
struct Raw<__nv_bfloat16, 2> {
    using Word = uint32_t;
    uint32_t v;
    __device__ __forceinline__ void zero() { v = 0; }
    __device__ __forceinline__ float2 get() const {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    }
};
__device__ __forceinline__ void put(float *p, float f) { *p = f; }
__device__ __forceinline__ void put(float *p, float2 f) { *reinterpret_cast<float2 *>(p) = f; }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float f) { *p = __float2bfloat16_rn(f); }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float2 f) {
    *reinterpret_cast<__nv_bfloat162 *>(p) = __floats2bfloat162_rn(f.x, f.y);
}

// The state that comes into a tile, from the words of the tiles before: `own`
// is this thread's word of this tile, `dec` its head's, with cw and H words a
// tile.  BACK tiles are read at a time; false when a word did not come in
// time.
template <typename V>
__device__ __forceinline__ bool look_back(const Word64 *own, int cw, const Word64 *dec, int H,
                                          int tile, unsigned tag, V &hin) {
    constexpr int BACK = 4;
    Words<V> w[BACK];
    Words<float> a[BACK];
    auto load = [&](int i, int j) {
        load_words(own - (int64_t)j * cw, w[i]);
        load_words(dec - (int64_t)j * H, a[i]);
    };
    // (a word that became final meanwhile holds what the chain gives)
    auto apply = [&](int i) {
        V aa;
        vset(aa, a[i].s, a[i].s);
        const V r = vfma(aa, hin, w[i].s);
        vset(hin, w[i].tag == tag + 1 ? lane0(w[i].s) : lane0(r), w[i].tag1 == tag + 1 ? lane1(w[i].s) : lane1(r));
    };
    unsigned long long t0 = 0;
    for (int j = 1;;) {
#pragma unroll
        for (int i = 0; i < BACK; ++i) load(i, min(j + i, tile));
        // the nearest final tile before any that is not ready, and how many
        // are ready
        int at = -1, ready = BACK;
#pragma unroll
        for (int i = BACK - 1; i >= 0; --i) {
            if (w[i].tag == tag + 1 && w[i].tag1 == tag + 1) {
                at = i;
            } else if ((w[i].tag | 1u) != tag + 1 || (w[i].tag1 | 1u) != tag + 1 || a[i].tag != tag) {
                at = -1;
                ready = i;
            }
        }
        if (at >= 0) {
#pragma unroll
            for (int i = BACK - 1; i >= 0; --i)
                if (i <= at) apply(i);
            for (--j; j > 0; j -= BACK) {
#pragma unroll
                for (int i = 0; i < BACK; ++i) load(i, max(j - i, 1));
#pragma unroll
                for (int i = 0; i < BACK; ++i)
                    if (j - i > 0) apply(i);
            }
            return true;
        }
        j += ready;  // (never beyond tile: tile 0 is final)
        if (ready == 0) {
            if (t0 == 0) t0 = gtimer();
            if (gtimer() - t0 > WAIT_NS) return false;
        }
    }
}

// How many offsets are <= r (a warp's lanes together, 32 probes a step).
__device__ __forceinline__ int count_offsets(const int64_t *off, int n_off, int64_t r, int lane) {
    const unsigned all = 0xffffffffu;
    int lo = 0, n = n_off;
    while (n > 32) {
        const int stride = (n + 31) / 32, at = lane * stride;
        const unsigned m = __ballot_sync(all, at < n && off[lo + at] <= r);
        if (m == 0) return lo;
        const int k = __popc(m) - 1;
        lo += k * stride;
        n = min(stride, n - k * stride);
    }
    return lo + __popc(__ballot_sync(all, lane < n && off[lo + lane] <= r));
}

// A tile's rows.  info: slot << 3 | fresh << 2 | place in the sequence (3 and
// above: 3), or -1 for a row of no sequence; the masks have a bit per row.
template <int ROWS>
struct Rows {
    int first, last;  // offsets <= the tile's first and last row
    int info[ROWS];
    unsigned valid[ROWS / 32], start[ROWS / 32], end[ROWS / 32];
};

// Shared memory of a CTA: x and z of the tile, then two buffers of the head
// scalars [heads][rows] (a, a, g, g | c, c, q, q: each twice for the packed
// instructions; q = C * the product of the part's decays up to the row) and of
// the parts' decays [heads][ST].  Odd parts are shifted by half a warp's words,
// so that the two parts of a warp do not meet in the banks.
template <typename T, int VEC, int CG, int ST, int LC>
struct Tile {
    static constexpr int NT = CG * ST, ROWS = ST * LC;
    static constexpr int PAD = CG == 16 ? 16 : 0;  // words per part
    static constexpr int WORDS = ROWS * CG + ST * PAD;
    static constexpr size_t STAGED = 2 * (size_t)WORDS * VEC * sizeof(T);
    static constexpr size_t PER_HEAD = 2 * (size_t)(ROWS * 32 + ST * 4);
};

// Persistent: while a CTA looks back and finishes a tile, the next one's
// inputs, weights, head scalars and row descriptions are on their way.
template <typename T, int VEC, int CG, int ST, int LC, int PER_SM>
__global__ void __launch_bounds__(CG *ST, PER_SM)
    prefill_kernel(const Args p, Control *ctl, Word64 *words, Word64 *decays, int n_cb, int n_items,
                   int max_heads, int wide, int *err) {
    using L = Tile<T, VEC, CG, ST, LC>;
    using Word = typename Raw<T, VEC>::Word;
    using V = typename Vec<VEC>::type;
    constexpr int NT = L::NT, ROWS = L::ROWS;
    static_assert(LC <= 32 && 32 % LC == 0 && ROWS % 32 == 0 && NT >= 96, "tile");
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int s_next;
    __shared__ unsigned s_epoch;
    __shared__ Rows<ROWS> rows_[2];
    __shared__ V part_s[ST][CG], came[CG];
    __shared__ float part_a[ST][CG];
    Word *const sx = reinterpret_cast<Word *>(smem), *const sz = sx + L::WORDS;
    float4 *const tabs = reinterpret_cast<float4 *>(smem + L::STAGED);
    float *const decs = reinterpret_cast<float *>(tabs + 2 * max_heads * ROWS * 2);
    const int C = p.l.C, P = p.l.P, tid = threadIdx.x, lane = tid & 31;
    const int cg = tid % CG, part = tid / CG, b0 = part * LC;
    constexpr unsigned mask = LC == 32 ? 0xffffffffu : (1u << LC % 32) - 1u;
    const float SET = -1.0f;  // in the place of A (a product of decays, >= 0)

    // ---- the steps that get an item ready
    auto stage_in = [&](int item, const void *from, Word *dst) {
        const int tile = item / n_cb, c0 = item % n_cb * (CG * VEC);
        const int64_t r0 = (int64_t)tile * ROWS;
        const int live = (int)min((int64_t)ROWS, p.rows - r0);
        const T *src = static_cast<const T *>(from) + r0 * p.ld + c0;
        if (wide) {  // 16 bytes at a time
            constexpr int E = 16 / (int)sizeof(T), CH = CG * VEC / E;  // elements, chunks of a row
            const int i = tid % CH;
            const T *q = src + i * E + tid / CH * p.ld;
            for (int r = tid / CH; r < live; r += NT / CH, q += NT / CH * p.ld) {
                const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst + r * CG + r / LC * L::PAD + i * (E / VEC));
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(q) : "memory");
            }
        } else if (c0 + cg * VEC < C) {
            for (int r = part; r < live; r += ST)
                stage(dst + r * CG + r / LC * L::PAD + cg, src + cg * VEC + r * p.ld, Word());
        }
    };
    V w0, w1, w2, w3, bias, dd;
    Raw<T, VEC> above[3];
    auto load_weights = [&](int item) {
        const int tile = item / n_cb, ch = item % n_cb * (CG * VEC) + cg * VEC;
        const int64_t r0 = (int64_t)tile * ROWS;
        const bool on = ch < C;
        float4 a = make_float4(0, 0, 0, 0), b = a;
        if (on) {
            a = reinterpret_cast<const float4 *>(p.l.conv_w)[ch];
            b = reinterpret_cast<const float4 *>(p.l.conv_w)[ch + VEC - 1];
        }
        vset(w0, a.x, b.x);
        vset(w1, a.y, b.y);
        vset(w2, a.z, b.z);
        vset(w3, a.w, b.w);
        vset(bias, on ? p.l.conv_b[ch] : 0.0f, on ? p.l.conv_b[ch + VEC - 1] : 0.0f);
        vset(dd, on ? p.l.d[ch] : 0.0f, on ? p.l.d[ch + VEC - 1] : 0.0f);
#pragma unroll
        for (int k = 0; k < 3; ++k) {  // the three rows above the tile
            above[k].zero();
            if (on && part == 0 && r0 > k && r0 - 1 - k < p.rows)
                above[k].v = *reinterpret_cast<const Word *>(static_cast<const T *>(p.x) + ch + (r0 - 1 - k) * p.ld);
        }
    };
    auto count = [&](int item, int buf, int warp) {  // warps 1 and 2
        const int64_t r0 = (int64_t)(item / n_cb) * ROWS;
        const int64_t r = warp == 1 ? r0 : min((int64_t)p.rows, r0 + ROWS) - 1;
        const int n = count_offsets(p.off, p.n_seq + 1, r, lane);
        if (lane == 0) (warp == 1 ? rows_[buf].first : rows_[buf].last) = n;
    };
    // entries i, i + step, ...: consecutive lanes are consecutive rows
    auto head_table = [&](int item, int buf, int i0, int step) {
        const int tile = item / n_cb, c0 = item % n_cb * (CG * VEC);
        const int64_t r0 = (int64_t)tile * ROWS;
        const int h0 = c0 / P, nh = (min(c0 + CG * VEC, C) - 1) / P - h0 + 1;
        float4 *tab = tabs + buf * max_heads * ROWS * 2;
        float *dec = decs + buf * max_heads * ST;
        for (int i = i0; i < nh * ROWS; i += step) {
            const int h = i / ROWS, t = i % ROWS;
            Head k{0.0f, 0.0f, 0.0f};
            if (r0 + t < p.rows) k = head_of<T>(p, r0 + t, h0 + h);
            float prod = k.a;
#pragma unroll
            for (int o = 1; o < LC; o <<= 1) {
                const float before = __shfl_up_sync(0xffffffffu, prod, o, LC);
                if (t % LC >= o) prod *= before;
            }
            tab[i * 2] = make_float4(k.a, k.a, k.g, k.g);
            tab[i * 2 + 1] = make_float4(k.c, k.c, k.c * prod, k.c * prod);
            if (t % LC == LC - 1) dec[h * ST + t / LC] = prod;
        }
    };
    auto describe_rows = [&](int item, int buf) {
        const int64_t r0 = (int64_t)(item / n_cb) * ROWS;
        Rows<ROWS> &rows = rows_[buf];
        for (int i = tid; i < (ROWS + NT - 1) / NT * NT; i += NT) {
            const int64_t r = r0 + i;
            // the offsets <= r, of which the tile has only a few
            int lo = rows.first, hi = max(rows.first, rows.last);
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (p.off[mid] <= r) lo = mid + 1;
                else hi = mid;
            }
            const int sid = lo - 1;
            int info = -1;
            bool first = false, last = false;
            if (i < ROWS && r < p.rows && sid >= 0 && sid < p.n_seq) {
                const int slot = p.slots ? p.slots[sid] : sid;
                if (slot >= 0 && slot < p.l.n_slots) {
                    const int64_t o0 = max((int64_t)0, p.off[sid]), o1 = min(p.off[sid + 1], (int64_t)p.rows);
                    const int fresh = p.fresh ? p.fresh[sid] != 0 : 1;
                    info = slot << 3 | fresh << 2 | (int)max((int64_t)0, min((int64_t)3, r - o0));
                    first = r == o0;
                    last = r == o1 - 1;
                }
            }
            const unsigned mv = __ballot_sync(0xffffffffu, info >= 0), ms = __ballot_sync(0xffffffffu, first),
                           me = __ballot_sync(0xffffffffu, last);
            if (i < ROWS) {
                rows.info[i] = info;
                if (lane == 0) {
                    rows.valid[i / 32] = mv;
                    rows.start[i / 32] = ms;
                    rows.end[i / 32] = me;
                }
            }
        }
    };

    if (tid == 0) {
        s_epoch = *reinterpret_cast<volatile unsigned *>(&ctl->epoch) + 1;
        s_next = (int)atomicAdd(&ctl->ticket, 1u);
    }
    __syncthreads();
    const unsigned epoch = s_epoch, tag = 2 * epoch;
    int item = s_next, buf = 0;
    if (item < n_items) {
        stage_in(item, p.x, sx);
        stage_commit();
        if (p.z) stage_in(item, p.z, sz);
        stage_commit();
        load_weights(item);
        if (tid >= 32 && tid < 96) count(item, 0, tid / 32);
        head_table(item, 0, tid, NT);
        __syncthreads();
        describe_rows(item, 0);
    }
    while (item < n_items) {
        stage_wait<1>();  // x; the gates may still be on their way
        __syncthreads();
        if (tid == 0) s_next = (int)atomicAdd(&ctl->ticket, 1u);
        const int tile = item / n_cb, cb = item % n_cb;
        const int64_t r0 = (int64_t)tile * ROWS;
        const int c0 = cb * CG * VEC, ch = c0 + cg * VEC;
        const bool on = ch < C;
        const Rows<ROWS> &rows = rows_[buf];
        const unsigned valid = rows.valid[b0 / 32] >> b0 % 32 & mask, start = rows.start[b0 / 32] >> b0 % 32 & mask,
                       end = rows.end[b0 / 32] >> b0 % 32 & mask;
        const int *info = rows.info + b0;
        const int head = (on ? ch : c0) / P, hh = head - c0 / P;
        const float4 *tb = tabs + ((buf * max_heads + hh) * ROWS + b0) * 2;
        const Word *xw = sx + b0 * CG + part * L::PAD + cg, *zw = sz + b0 * CG + part * L::PAD + cg;

        // x1, x2, x3: the inputs 1, 2, 3 tokens back; from the slot before the
        // sequence's first
        auto conv_at = [&](int slot, int j) {
            return static_cast<T *>(p.l.conv) + ((int64_t)slot * 3 + j) * C + ch;
        };
        auto back = [&](int k, int place, int t) {
            // the input k tokens before a token at `place` < k of its sequence
            Raw<T, VEC> r;
            r.zero();
            if (on && !(info[t] & 4)) r.v = *reinterpret_cast<const Word *>(conv_at(info[t] >> 3, 3 + place - k));
            return r.get();
        };
        auto keep = [&](int slot, V a, V b, V c, V s) {
            if (!on) return;
            put(conv_at(slot, 0), a);
            put(conv_at(slot, 1), b);
            put(conv_at(slot, 2), c);
            put(p.l.h + (int64_t)slot * C + ch, s);
        };
        if (part > 0) {
#pragma unroll
            for (int k = 0; k < 3; ++k) above[k].v = xw[-(k + 1) * CG - L::PAD];
        }
        V x1 = above[0].get(), x2 = above[1].get(), x3 = above[2].get();
        if ((valid & 1u) && !(start & 1u)) {
            const int place = info[0] & 3;
            if (place < 3) x3 = back(3, place, 0);
            if (place < 2) x2 = back(2, place, 0);
        }
        V h, y[LC];
        vset(h, 0.0f, 0.0f);
        // the end of the sequence that came in from the part before
        float Ae = 0.0f;
        V he = h, e1 = h, e2 = h, e3 = h;
        int end_slot = -1;
        auto token = [&](int t) {
            const float4 k0 = tb[t * 2], k1 = tb[t * 2 + 1];
            V a, g, c;
            vset(a, k0.x, k0.y);
            vset(g, k0.z, k0.w);
            vset(c, k1.x, k1.y);
            Raw<T, VEC> xr;
            xr.v = xw[t * CG];
            const V xt = xr.get();
            const V u = silu(vfma(w3, xt, vfma(w2, x1, vfma(w1, x2, vfma(w0, x3, bias)))));
            h = vfma(a, h, vmul(g, u));
            y[t] = vfma(c, h, vmul(dd, u));
            x3 = x2;
            x2 = x1;
            x1 = xt;
            return k0.x;
        };
        if (valid == mask && !start && !end) {
#pragma unroll
            for (int t = 0; t < LC; ++t) token(t);
        } else {
            float A = 1.0f;
#pragma unroll
            for (int t = 0; t < LC; ++t) {
                if (start >> t & 1u) {
                    x1 = back(1, 0, t);
                    x2 = back(2, 0, t);
                    x3 = back(3, 0, t);
                    const float *hs = p.l.h + (int64_t)(info[t] >> 3) * C + ch;
                    const bool from = on && !(info[t] & 4);
                    vset(h, from ? hs[0] : 0.0f, from ? hs[VEC - 1] : 0.0f);
                }
                A *= token(t);
                if (end >> t & 1u) {
                    if (start & ((2u << t) - 1u)) {
                        keep(info[t] >> 3, x3, x2, x1, h);
                    } else {
                        // completed and written below, when the state that came
                        // in is known: whoever starts from the slot has read it
                        // by then
                        end_slot = info[t] >> 3;
                        Ae = A;
                        he = h;
                        e1 = x1;
                        e2 = x2;
                        e3 = x3;
                    }
                }
            }
        }
        // the parts' S and A; with a start in a part its S is the state itself
        part_s[part][cg] = h;
        part_a[part][cg] = start ? SET : decs[(buf * max_heads + hh) * ST + part];
        auto pass = [&](int i, V s) {  // the state through part i
            const float a = part_a[i][cg];
            const V local = part_s[i][cg];
            V aa;
            vset(aa, a, a);
            const V r = vfma(aa, s, local);
            return a == SET ? local : r;
        };
        __syncthreads();

        // the next item on its way; part 0 joins the parts and looks back
        const int next = s_next;
        const bool more = next < n_items;
        if (more) {
            stage_in(next, p.x, sx);
            load_weights(next);
        }
        stage_commit();
        if (tid < 32) {
            if (part == 0) {
                // Every tile but the last publishes, whatever its rows are, so
                // that offsets that contradict each other make no tile wait
                // for a word that never comes.
                const bool need_in = tile > 0 && (valid & 1u) && !(start & 1u);
                const bool need_out = r0 + ROWS < p.rows;
                Word64 *own = words + (int64_t)tile * C + ch, *dec = decays + (int64_t)tile * p.l.H + head;
                float all = 1.0f;
                V S, hin;
                vset(S, 0.0f, 0.0f);
                vset(hin, 0.0f, 0.0f);
                bool is_final = !need_in;
                if (need_out) {
#pragma unroll 4
                    for (int i = 0; i < ST; ++i) {
                        S = pass(i, S);
                        is_final |= part_a[i][cg] == SET;
                        all *= part_a[i][cg];
                    }
                    if (on) {
                        store_words(own, is_final ? tag + 1 : tag, S);
                        // one thread a head (or more, with the same value)
                        if (!is_final && (tid == 0 || ch % P < VEC)) store_words(dec, tag, all);
                    }
                }
                if (need_in && on && !look_back(own, C, dec, p.l.H, tile, tag, hin)) atomicOr(err, 8);
                if (need_out && !is_final && on) {
                    V aa;
                    vset(aa, all, all);
                    store_words(own, tag + 1, vfma(aa, hin, S));
                }
                came[cg] = hin;
            }
            __syncwarp();
        } else if (more) {
            if (tid < 96) count(next, buf ^ 1, tid / 32);
            head_table(next, buf ^ 1, tid - 32, NT - 32);
        }
        stage_wait<1>();  // z
        __syncthreads();
        V hin = came[cg];
        for (int i = 0; i < part; ++i) hin = pass(i, hin);
        if (end_slot >= 0) {
            V aa;
            vset(aa, Ae, Ae);
            keep(end_slot, e3, e2, e1, vfma(aa, hin, he));
        }
        if (on) {
            const int first = start ? __ffs(start) - 1 : LC;
            T *py = static_cast<T *>(p.y) + ch + (r0 + b0) * p.ldy;
            auto finish = [&](int t, bool fix) {
                V o = y[t];
                if (fix) {
                    const float2 q2 = *reinterpret_cast<const float2 *>(&tb[t * 2 + 1].z);
                    V q;
                    vset(q, q2.x, q2.y);
                    o = vfma(q, hin, o);
                }
                if (p.z) {
                    Raw<T, VEC> zr;
                    zr.v = zw[t * CG];
                    o = vmul(o, silu(zr.get()));
                }
                put(py, o);
            };
            if (valid == mask && !start) {
#pragma unroll
                for (int t = 0; t < LC; ++t, py += p.ldy) finish(t, true);
            } else {
#pragma unroll
                for (int t = 0; t < LC; ++t, py += p.ldy)
                    if (valid >> t & 1u) finish(t, t < first);
            }
        }
        // sequences without tokens that start afresh: a zero state
        if (tile == 0) {
            __shared__ int empty[NT], n_empty;
            for (int s0 = 0; s0 < p.n_seq; s0 += NT) {
                const int s = s0 + tid;
                int slot = -1;
                if (s < p.n_seq && !(p.fresh && p.fresh[s] == 0) &&
                    max((int64_t)0, p.off[s]) >= min((int64_t)p.rows, p.off[s + 1])) {
                    slot = p.slots ? p.slots[s] : s;
                    if (slot >= p.l.n_slots) slot = -1;
                }
                if (!__syncthreads_or(slot >= 0)) continue;
                if (tid == 0) n_empty = 0;
                __syncthreads();
                if (slot >= 0) empty[atomicAdd(&n_empty, 1)] = slot;
                __syncthreads();
                V none;
                vset(none, 0.0f, 0.0f);
                for (int i = part; i < n_empty; i += ST) keep(empty[i], none, none, none, none);
                __syncthreads();
            }
        }
        if (more) describe_rows(next, buf ^ 1);
        __syncthreads();  // z and the parts are free
        if (more && p.z) stage_in(next, p.z, sz);
        stage_commit();
        item = next;
        buf ^= 1;
    }
    if (tid == 0) {
        __threadfence();
        if (atomicAdd(&ctl->done, 1u) == gridDim.x - 1) {
            ctl->ticket = 0;
            ctl->done = 0;
            __threadfence();
            ctl->epoch = epoch;
        }
    }
}

struct Launch {
    Args a;
    bm_ctx_t *ctx;
    int sms;
    int *err;
    cudaStream_t s;
};

template <typename T, int VEC, int CG, int ST, int LC, int PER_SM>
int launch_prefill(const Launch &l) {
    using L = Tile<T, VEC, CG, ST, LC>;
    const Args &a = l.a;
    const int C = a.l.C, P = a.l.P;
    const int n_cb = (C + CG * VEC - 1) / (CG * VEC);
    const int64_t tiles = a.rows > 0 ? ((int64_t)a.rows + L::ROWS - 1) / L::ROWS : 1;
    const int64_t items = tiles * n_cb;
    if (items > INT32_MAX / 2)
        return bm_detail_fail(BM_ERR_UNSUPPORTED, "rows * channels too large for one call");
    // a word per tile and channel, then one per tile and head
    const size_t n_words = ((size_t)tiles * C + 1) / 2 * 2;
    void *work;
    const int rc = bm_detail_work(l.ctx, BM_WORK_SCAN,
                                  CONTROL_BYTES + (n_words + (size_t)tiles * a.l.H) * sizeof(Word64), &work);
    if (rc != BM_OK) return rc;
    Word64 *words = reinterpret_cast<Word64 *>(static_cast<unsigned char *>(work) + CONTROL_BYTES);
    const int heads = min((CG * VEC + P - 2) / P + 1, a.l.H);
    auto *k = prefill_kernel<T, VEC, CG, ST, LC, PER_SM>;
    constexpr int most = 200 * 1024;
    const size_t bytes = L::STAGED + (size_t)heads * L::PER_HEAD;
    if (bytes > most) return bm_detail_fail(BM_ERR_UNSUPPORTED, "too many heads in a tile");
    BMC_CK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    auto even = [&](const void *q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
    const int wide = C % (CG * VEC) == 0 && even(a.x) && even(a.z) && a.ld * (int64_t)sizeof(T) % 16 == 0;
    const int64_t grid = items < (int64_t)PER_SM * l.sms ? items : (int64_t)PER_SM * l.sms;
    k<<<(int)grid, L::NT, bytes, l.s>>>(a, static_cast<Control *>(work), words, words + n_words, n_cb,
                                        (int)items, heads, wide, l.err);
    BMC_CK(cudaGetLastError());
    return BM_OK;
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
    a.off = d_seq_off;
    a.n_seq = n_seq;
    a.fresh = d_fresh;
    const size_t e = layer->type == BM_F32 ? 4 : 2;
    // two channels a thread: a pair is one head's, and every pair is aligned
    const bool pairs = a.l.P % 2 == 0 && a.l.P >= 16 && ld % 2 == 0 && ldy % 2 == 0 &&
                       !misaligned(d_x, 2 * e) && !misaligned(d_z, 2 * e) &&
                       !misaligned(d_y, 2 * e) && !misaligned(layer->conv_state, 2 * e) &&
                       !misaligned(layer->h_state, 8);
    Launch l{};
    l.ctx = ctx;
    bmc::DeviceGuard guard(bm_detail_ctx(ctx, &l.sms, &l.err, &l.s));
    BMC_CK(guard.error);
    if (stream) l.s = static_cast<cudaStream_t>(stream);
    l.a = a;
    // Tall tiles unless that leaves SMs without work.  One channel a thread,
    // in small tiles, for what cannot be paired and for heads so small that
    // their scalars would fill the shared memory.
    using bf16 = __nv_bfloat16;
    const bool few = ((int64_t)rows + 255) / 256 * ((a.l.C + 31) / 32) < 2 * l.sms;
    if (layer->type == BM_F32) {
        if (!pairs) return launch_prefill<float, 1, 32, 4, 8, 4>(l);
        return few ? launch_prefill<float, 2, 16, 8, 8, 4>(l) : launch_prefill<float, 2, 16, 8, 16, 4>(l);
    }
    if (!pairs) return launch_prefill<bf16, 1, 32, 4, 8, 4>(l);
    return few ? launch_prefill<bf16, 2, 16, 8, 8, 4>(l) : launch_prefill<bf16, 2, 16, 16, 16, 2>(l);
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
