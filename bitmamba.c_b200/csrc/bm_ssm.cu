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
#include <type_traits>

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
    // the head scalars of all rows, and the parts' decays (heads_kernel)
    const float4 *tab;
    const float *dec;
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
// a scalar with a pair: plain instructions, the packed ones would want it twice
__device__ __forceinline__ float sfma(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float2 sfma(float a, float2 b, float2 c) {
    return make_float2(fmaf(a, b.x, c.x), fmaf(a, b.y, c.y));
}
__device__ __forceinline__ float smul(float a, float b) { return a * b; }
__device__ __forceinline__ float2 smul(float a, float2 b) { return make_float2(a * b.x, a * b.y); }
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
// v / (1 + e^-v); where e^-v passes the range (v < -88.7) -0, as the quotient
// in fp32 gives, and NaN for -infinity.
__device__ __forceinline__ float silu(float v) { return v * rcp(ex2(v * -1.44269504f) + 1.0f); }
// Of a pair, with a reciprocal each.  (One of the product for both has to hold
// e^-v at 2^63, and then is v 2^-63 below -43, which grows with v; the same
// time in fp32, 3 % less for 65536 x 4096 bf16.)
__device__ __forceinline__ float2 silu(float2 v) { return make_float2(silu(v.x), silu(v.y)); }
__device__ __forceinline__ float softplus(float v) {
    return fmaxf(v, 0.0f) + log1pf(expf(-fabsf(v)));
}

// A head's scalars for one token: the decay a, the input's factor g = d B and
// the output's C.
struct Head {
    float a, g, c;
};
__device__ __forceinline__ Head head_of(float dt, float rate, float b, float c) {
    const float d = softplus(dt);
    Head r;
    r.a = expf(-rate * d);
    r.g = d * b;
    r.c = c;
    return r;
}
// ---------------------------------------------------------------- prompts --
//
// The token axis of all sequences together is cut into tiles of ST * LC rows.
// A CTA takes CG * VEC channels and goes down the tiles; a thread has VEC
// channels of one of a tile's ST parts, with the convolution's window, the
// state and the outputs in registers.  The recurrence is linear, so a part
// first runs from a zero state:
//   s_t = local_t + (a_first ... a_t) * s_in,    s_out = S + A * s_in
// the parts' (A, S) are joined by a scan over the lanes of a warp, and the
// outputs, which waited in registers, get their C a_first ... a_t s_in: x and
// z are read once, y is written once.  The next tile's x and z are copied to
// shared memory meanwhile.
//
// A CTA's channels are 64 to 128 bytes of a row, so a few dozen to hundreds of
// CTAs share a prompt with nothing between them.  Where that leaves SMs idle
// (few channels, many rows), a cluster takes as many tiles at once as it has
// CTAs: each leaves its tile's (A, S) in its shared memory, and after one
// cluster barrier reads the others' to know the state that comes in.  (In a
// launch for the sums of segments, one that starts from them and one that
// writes the states of sequences across them, 2000 x 2048 fp32 took 41 us.)
//
// Measured against it: tiles joined by published words and a look-back (one
// launch, any number of CTAs on an axis) took 0.91 ms for 65536 x 4096 bf16
// and 123 us for 4099 x 4096 fp32; the chain over the tiles was what it spent
// its time on.
//
// 65536 x 4096 bf16 takes 526 us (3.1 TB/s; 250 us at the device's 6.5): 73
// instructions a pair of channels and token keep the issue slots of the 128
// SMs that have channels 56 % busy, the 8 special functions among them half
// of their units' rate; the rest are waits for those and for shared memory, and
// two barriers a tile.  32768 x 4096 fp32 takes 351 us (4.7 TB/s), 4099 x 4096
// fp32 in 13 sequences 60 us, 53 as one sequence: a tile with a
// boundary has its rows looked up, and its warps wait for the one that has it.

// Copies to shared memory: 4 or 8 bytes asynchronously, a 2-byte element
// through a register.
__device__ __forceinline__ void stage(void *dst, const void *src, float) {
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(d), "l"(src) : "memory");
}
__device__ __forceinline__ void stage(void *dst, const void *src, uint32_t) { stage(dst, src, 0.0f); }
__device__ __forceinline__ void stage(void *dst, const void *src, __nv_bfloat16) {
    *static_cast<__nv_bfloat16 *>(dst) = *static_cast<const __nv_bfloat16 *>(src);
}
__device__ __forceinline__ void stage(void *dst, const void *src, float2) {
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(d), "l"(src) : "memory");
}

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

// In the place of A (a product of decays, >= 0): a sequence starts in there,
// S is the state itself.  Not A = 0, which a state that is not finite would
// survive.
constexpr float SET = -1.0f;
__device__ __forceinline__ float through(float a, float s, float S) { return a == SET ? S : fmaf(a, s, S); }
__device__ __forceinline__ float2 through(float a, float2 s, float2 S) {
    return a == SET ? S : __ffma2_rn(make_float2(a, a), s, S);
}
__device__ __forceinline__ float through(float a1, float a2) { return a2 == SET || a1 == SET ? SET : a1 * a2; }
__device__ __forceinline__ float shfl_up(float v, int o, int w) { return __shfl_up_sync(0xffffffffu, v, o, w); }
__device__ __forceinline__ float2 shfl_up(float2 v, int o, int w) {
    return make_float2(shfl_up(v.x, o, w), shfl_up(v.y, o, w));
}
__device__ __forceinline__ float shfl_at(float v, int l, int w) { return __shfl_sync(0xffffffffu, v, l, w); }
__device__ __forceinline__ float2 shfl_at(float2 v, int l, int w) {
    return make_float2(shfl_at(v.x, l, w), shfl_at(v.y, l, w));
}

constexpr int SEQ_CACHE = 1024;  // sequences whose offsets a CTA keeps in shared memory

template <typename T, int VEC, int CG, int ST, int LC, bool PRE>
struct Tile {
    static constexpr int NT = CG * ST, ROWS = ST * LC;
    // words: a part is shifted by CG words against the one before, so that the
    // parts of a warp (of half a warp, for 8-byte words) meet in no bank
    static constexpr int PAD = CG * VEC * sizeof(T) >= 128 ? 0 : CG;
    static constexpr int WORDS = ROWS * CG + ST * PAD;
    // x twice; z once, copied while the tile's scan runs, or twice, copied a
    // tile ahead.  Once, a long fp32 prompt's tiles waited for it (32768 x 4096
    // 383 us, twice 345); 16 tokens of bf16 take long enough (65536 x 4096 522
    // us, twice 528), and so do tiles that work out their head scalars (2048 x
    // 4096 fp32 36.8, twice 38.0).
    static constexpr int Z = PRE && sizeof(T) == 4 ? 2 : 1;
    static constexpr size_t STAGED = (2 + Z) * (size_t)WORDS * VEC * sizeof(T);
    // a head's scalars (a, g, c, C times the part's decays up to the row) and
    // its parts' decays, twice
    static constexpr size_t PER_HEAD = 2 * (size_t)(ROWS * 16 + ST * 4);
};

// The head scalars of all rows, [part of LC rows][head][LC], and the parts'
// decays, [part][head]: a thread a head and part.  Each head's are needed by
// every CTA that has channels of it; worked out by each of them they took a
// third of a long prompt's instructions.
template <typename T, int LC>
__global__ void __launch_bounds__(128) heads_kernel(const Args p, float4 *tab, float *dec) {
    const int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x;
    const int64_t part = i / p.l.H;
    const int h = (int)(i - part * p.l.H);
    if (part * LC >= p.rows) return;
    float4 *out = tab + i * LC;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const float bias = p.l.dt_bias[h], rate = expf(p.l.a_log[h]);
    T dt[LC], b[LC], c[LC];
#pragma unroll
    for (int t = 0; t < LC; ++t) {
        const int64_t at = min(part * LC + t, (int64_t)p.rows - 1) * p.ld + h;
        dt[t] = static_cast<const T *>(p.dt)[at];
        b[t] = static_cast<const T *>(p.b)[at];
        c[t] = static_cast<const T *>(p.c)[at];
    }
    float prod = 1.0f;
#pragma unroll
    for (int t = 0; t < LC; ++t) {
        const Head k = head_of(to_f(dt[t]) + bias, rate, to_f(b[t]), to_f(c[t]));
        prod *= k.a;
        out[t] = make_float4(k.a, k.g, k.c, k.c * prod);
    }
    dec[i] = prod;
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// a value in the shared memory of another CTA of the cluster
__device__ __forceinline__ uint32_t remote(const void *p, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ void load_remote(uint32_t at, float &v) {
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
}
__device__ __forceinline__ void load_remote(uint32_t at, float2 &v) {
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
}

// PRE: the head scalars come from p.tab.  gridDim.y: CTAs of a cluster.
template <typename T, int VEC, int CG, int ST, int LC, int PER_SM, bool PRE>
__global__ void __launch_bounds__(CG *ST, PER_SM) prefill_kernel(const Args p, int heads, int wide) {
    using L = Tile<T, VEC, CG, ST, LC, PRE>;
    using R = Raw<T, VEC>;
    using Word = typename R::Word;
    using V = typename Vec<VEC>::type;
    constexpr int NT = L::NT, ROWS = L::ROWS;
    static_assert(LC <= 32 && 32 % LC == 0 && ST <= 32 && ROWS % 32 == 0 && NT % 32 == 0 && LC >= 3, "tile");
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int s_off[SEQ_CACHE + 1], s_info[SEQ_CACHE];
    __shared__ int row_info[ROWS];
    __shared__ unsigned row_valid[ROWS / 32], row_start[ROWS / 32], row_end[ROWS / 32];
    __shared__ int last_begin, last_end, last_info, n_list, list[NT];
    // the state and inputs that the first sequence starting in a part of the
    // next tile takes from its slot
    __shared__ V init_h[ST][CG];
    __shared__ Word init_x[ST][3][CG];
    __shared__ V part_s[ST][CG + 1], came[ST][CG + 1];
    __shared__ float part_a[ST][CG + 1];
    __shared__ Word halo[2][3][CG];  // the three rows above the tile
    __shared__ float head_bias[CG * VEC], head_rate[CG * VEC];
    // the tile's (A, S), of this step and the one before
    __shared__ V tile_s[2][CG];
    __shared__ float tile_a[2][CG];
    Word *const sx = reinterpret_cast<Word *>(smem), *const sz = sx + 2 * L::WORDS;
    float4 *const tabs = reinterpret_cast<float4 *>(smem + L::STAGED);
    float *const decs = reinterpret_cast<float *>(tabs + 2 * heads * ROWS);
    const int C = p.l.C, P = p.l.P, tid = threadIdx.x, lane = tid & 31;
    const int cg = tid % CG, part = tid / CG, b0 = part * LC;
    const int rank = blockIdx.y, many = gridDim.y;  // (of a cluster)
    const int c0 = blockIdx.x * (CG * VEC), ch = c0 + cg * VEC;
    const int first = rank * ROWS, step = many * ROWS;  // this CTA's first row, and to its next tile
    const bool on = ch < C;
    const int h0 = c0 / P, nh = (min(c0 + CG * VEC, C) - 1) / P - h0 + 1, hh = (on ? ch : c0) / P - h0;
    constexpr unsigned mask = LC == 32 ? 0xffffffffu : (1u << LC % 32) - 1u;
    const bool gate = p.z != nullptr;

    // Copies of rows, 16 bytes a thread where that can be: COPIES for a tile,
    // the n-th of them by copy(n).
    constexpr int E = 16 / (int)sizeof(T), CH = CG * VEC / E;  // elements, chunks of a row
    constexpr int STEP = NT / CH, COPIES = ROWS / STEP;        // rows a copy
    static_assert(STEP % LC == 0 && COPIES * STEP == ROWS, "a copy is whole parts");
    const int copy_i = tid % CH, copy_r = tid / CH;
    const int copy_to = (copy_r * CG + copy_i * (E / VEC) + copy_r / LC * L::PAD) * (int)sizeof(Word);
    const int64_t copy_pitch = STEP * p.ld;
    // the next tile's first chunk of this thread; a tile's copies move them on
    const T *next_x = static_cast<const T *>(p.x) + (int64_t)(first + copy_r) * p.ld + c0 + copy_i * E;
    const T *next_z = static_cast<const T *>(p.z) + (next_x - static_cast<const T *>(p.x));
    // (a predicate, not a branch, which would keep the tokens from overlapping)
    auto copy = [&](const T *&from, uint32_t to, int n, bool yes) {
        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %2, 0;\n @p cp.async.cg.shared.global [%0], [%1], 16;\n}" ::"r"(
                         to + n * (STEP * CG + STEP / LC * L::PAD) * (int)sizeof(Word)),
                     "l"(from), "r"((int)yes)
                     : "memory");
        from += copy_pitch;
    };
    auto stage_rows = [&](int r0, const void *from, const T *next, Word *dst) {  // (at once)
        const int live = min(ROWS, p.rows - r0);
        if (wide) {
            const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst) + copy_to;
            for (int n = 0; copy_r + n * STEP < live; ++n) copy(next, to, n, true);
        } else if (on) {
            const T *src = static_cast<const T *>(from) + r0 * p.ld + c0;
            for (int r = part; r < live; r += ST)
                stage(dst + r * CG + r / LC * L::PAD + cg, src + cg * VEC + r * p.ld, Word());
        }
    };
    // what a tile needs besides: the rows above, the head scalars
    const bool halos = on && part < 3;
    const T *next_halo = static_cast<const T *>(p.x) + ch + (first - 1 - part) * p.ld;
    // (one head's entries are consecutive in a part, LC of them)
    const float4 *next_tab = p.tab + ((int64_t)(first / LC + tid / LC) * p.l.H + h0) * LC + tid % LC;
    const float *next_dec = p.dec + (int64_t)(first / LC + tid) * p.l.H + h0;
    auto stage_rest = [&](int r0, int buf) {
        if (halos && r0 > part) stage(&halo[buf][part][cg], next_halo, Word());
        next_halo += step * p.ld;
        if (PRE) {
            const int live = min(ROWS, p.rows - r0);
            for (int h = 0; h < nh; ++h) {
                if (tid < ROWS && tid / LC * LC < live) {
                    const uint32_t a = (uint32_t)__cvta_generic_to_shared(tabs + (buf * heads + h) * ROWS + tid);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(a), "l"(next_tab + h * LC) : "memory");
                }
                if (tid < ST && tid * LC < live) stage(decs + (buf * heads + h) * ST + tid, next_dec + h, 0.0f);
            }
            next_tab += (int64_t)step * p.l.H;
            next_dec += (int64_t)(step / LC) * p.l.H;
        }
    };
    static_assert(!PRE || ROWS <= NT, "an entry a thread");
    auto commit = []() { asm volatile("cp.async.commit_group;" ::: "memory"); };
    // The scalars of a tile's rows: entry i is row i % ROWS of head i / ROWS, so
    // consecutive lanes are consecutive rows.  A thread's first entry is loaded
    // early.
    T raw[3];
    auto load_head = [&](int r0, int i) {
        const int64_t at = (int64_t)min(r0 + i % ROWS, p.rows - 1) * p.ld + h0 + i / ROWS;
        raw[0] = static_cast<const T *>(p.dt)[at];
        raw[1] = static_cast<const T *>(p.b)[at];
        raw[2] = static_cast<const T *>(p.c)[at];
    };
    auto load_heads = [&](int r0) {
        if (tid < nh * ROWS) load_head(r0, tid);
    };
    auto head_table = [&](int r0, int buf) {
        for (int i = tid; i < nh * ROWS; i += NT) {
            const int h = i / ROWS, t = i % ROWS;
            if (i != tid) load_head(r0, i);
            Head k = head_of(to_f(raw[0]) + head_bias[h], head_rate[h], to_f(raw[1]), to_f(raw[2]));
            if (r0 + t >= p.rows) k = Head{0.0f, 0.0f, 0.0f};
            float prod = k.a;
#pragma unroll
            for (int o = 1; o < LC; o <<= 1) {
                const float before = shfl_up(prod, o, LC);
                if (t % LC >= o) prod *= before;
            }
            tabs[buf * heads * ROWS + i] = make_float4(k.a, k.g, k.c, k.c * prod);
            if (t % LC == LC - 1) decs[(buf * heads + h) * ST + t / LC] = prod;
        }
    };
    const bool cached = p.n_seq <= SEQ_CACHE;
    auto off_at = [&](int i) {
        return cached ? s_off[i] : (int)max((int64_t)0, min((int64_t)p.rows, p.off[i]));
    };
    // slot << 4 | fresh << 2, or -1
    auto load_info = [&](int s) {
        const int slot = p.slots ? p.slots[s] : s;
        const int fresh = p.fresh ? p.fresh[s] != 0 : 1;
        return slot >= 0 && slot < p.l.n_slots ? slot << 4 | fresh << 2 : -1;
    };
    // What the rows of a tile are, a thread a row.  row_info: slot << 4 | fresh
    // << 2 | place in the sequence (3 and above: 3), or -1 for a row of no
    // sequence; the masks have a bit per row.
    auto describe_rows = [&](int r0) {
        for (int i = tid; i < ROWS; i += NT) {  // (whole warps)
            const int r = r0 + i;
            int lo = 0, hi = p.n_seq + 1;  // the offsets <= r
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (off_at(mid) <= r) lo = mid + 1;
                else hi = mid;
            }
            const int sid = lo - 1;
            int info = -1, o0 = 0, o1 = 0;
            if (r < p.rows && sid >= 0 && sid < p.n_seq) {
                info = cached ? s_info[sid] : load_info(sid);
                o0 = off_at(sid);
                o1 = off_at(sid + 1);
                if (info >= 0) info |= max(0, min(3, r - o0));
            }
            const unsigned all = 0xffffffffu;
            const unsigned mv = __ballot_sync(all, info >= 0), ms = __ballot_sync(all, info >= 0 && r == o0),
                           me = __ballot_sync(all, info >= 0 && r == o1 - 1);
            row_info[i] = info;
            if (lane == 0) {
                row_valid[i / 32] = mv;
                row_start[i / 32] = ms;
                row_end[i / 32] = me;
            }
            if (i == ROWS - 1) {
                last_begin = o0;
                last_end = o1;
                last_info = info;
            }
        }
    };

    // ---- before the first tile
    if (first < p.rows) stage_rows(first, p.x, next_x, sx);
    next_x += step * p.ld;
    if (!PRE) {
        if (first < p.rows) load_heads(first);
        if (tid < nh) {
            head_bias[tid] = p.l.dt_bias[h0 + tid];
            head_rate[tid] = expf(p.l.a_log[h0 + tid]);
        }
    }
    V w0, w1, w2, w3, bias, dd;
    {
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
    }
    if (cached) {
        for (int i = tid; i <= p.n_seq; i += NT) {
            s_off[i] = (int)max((int64_t)0, min((int64_t)p.rows, p.off[i]));
            if (i < p.n_seq) s_info[i] = load_info(i);
        }
    }
    // the scan's view of the threads: each joins GP parts of a pair of channels
    // (a lane a part took 700 cycles a tile more, in shuffles)
    constexpr int GP = ST >= 16 ? 4 : 2, SG = ST / GP;
    const int sp = tid % SG, sc = tid / SG;
    const bool scans = tid < CG * SG;  // (whole warps)
    static_assert(CG * SG % 32 == 0, "scan");
    V carry;  // the state that comes into the cluster's tiles, of the scan's channels
    vset(carry, 0.0f, 0.0f);
    __syncthreads();
    if (!PRE && first < p.rows) head_table(first, 0);
    describe_rows(first);
    // until here the head scalars need not be there (launch_prefill)
    if (PRE) asm volatile("griddepcontrol.wait;" ::: "memory");
    if (first < p.rows) stage_rest(first, 0);
    commit();

    auto conv_at = [&](int slot, int j) {
        return static_cast<T *>(p.l.conv) + ((int64_t)slot * 3 + j) * C + ch;
    };
    auto back = [&](int k, int place, int info) {
        // the input k tokens before a token at `place` < k of its sequence
        R r;
        r.zero();
        if (on && !(info & 4)) r.v = *reinterpret_cast<const Word *>(conv_at(info >> 4, 3 + place - k));
        return r.get();
    };
    auto keep = [&](int slot, V a, V b, V c, V s) {
        if (!on) return;
        put(conv_at(slot, 0), a);
        put(conv_at(slot, 1), b);
        put(conv_at(slot, 2), c);
        put(p.l.h + (int64_t)slot * C + ch, s);
    };

    auto fetch_init = [&]() {
        const unsigned start = row_start[b0 / 32] >> b0 % 32 & mask;
        if (!start) return;
        const int info = row_info[b0 + __ffs(start) - 1];
        if (!on || (info & 4)) return;
        stage(&init_h[part][cg], p.l.h + (int64_t)(info >> 4) * C + ch, V());
#pragma unroll
        for (int k = 0; k < 3; ++k) stage(&init_x[part][k][cg], conv_at(info >> 4, k), Word());
        commit();
    };
    __syncthreads();
    fetch_init();

    constexpr bool Z2 = L::Z == 2;
    if (Z2 && gate && first < p.rows) stage_rows(first, p.z, next_z, sz);
    if (Z2) {
        next_z += step * p.ld;
        commit();
    }

    bool plain = false;
    int buf = 0;
    // (every CTA of a cluster takes as many turns, with no rows in the last
    // ones perhaps)
    for (int r0 = first; r0 - first < p.rows; r0 += step, buf ^= 1) {
        // (all but z, which is the last group)
        asm volatile("cp.async.wait_group %0;" ::"n"(Z2 ? 1 : 0) : "memory");
        __syncthreads();
        const int r1 = r0 + step;
        // z (this tile's, or the next one's between the outputs) and the next
        // tile's x are copied between the tokens: all at once, the copies' issue
        // held every thread for 1000 cycles (of 9800 a tile).
        const bool spread_x = wide && r1 + ROWS <= p.rows, spread_z = gate && wide && (Z2 ? r1 : r0) + ROWS <= p.rows;
        const uint32_t to_z = (uint32_t)__cvta_generic_to_shared(sz + (Z2 ? (buf ^ 1) * L::WORDS : 0)) + copy_to,
                       to_x = (uint32_t)__cvta_generic_to_shared(sx + (buf ^ 1) * L::WORDS) + copy_to;
        const T *from_z = next_z, *from_x = next_x;
        if (r1 < p.rows) stage_rest(r1, buf ^ 1);
        if (!PRE && r1 < p.rows) load_heads(r1);
        const bool rows_left = r0 < p.rows;
        unsigned valid = rows_left ? mask : 0, start = 0, end = 0;
        if (rows_left && !plain) {
            valid = row_valid[b0 / 32] >> b0 % 32 & mask;
            start = row_start[b0 / 32] >> b0 % 32 & mask;
            end = row_end[b0 / 32] >> b0 % 32 & mask;
        }
        const int *info = row_info + b0;
        const float4 *tb = tabs + (buf * heads + hh) * ROWS + b0;
        const uint32_t tb_at = (uint32_t)__cvta_generic_to_shared(tb);
        const Word *xw = sx + buf * L::WORDS + b0 * CG + part * L::PAD + cg, *zw = sz + (Z2 ? buf * L::WORDS : 0) + b0 * CG + part * L::PAD + cg;

        // x1, x2, x3: the inputs 1, 2, 3 tokens back; from the slot before the
        // sequence's first
        V x1, x2, x3;
        {
            R r;
            r.v = part ? xw[-CG - L::PAD] : halo[buf][0][cg];
            x1 = r.get();
            r.v = part ? xw[-2 * CG - L::PAD] : halo[buf][1][cg];
            x2 = r.get();
            r.v = part ? xw[-3 * CG - L::PAD] : halo[buf][2][cg];
            x3 = r.get();
        }
        V h, y[LC];
        vset(h, 0.0f, 0.0f);
        // the end of the sequence that came in from the part before
        float Ae = 0.0f;
        V he = h, e1 = h, e2 = h, e3 = h;
        int end_info = -1;
        auto token = [&](int t) {
            float4 k;
            // (all four at once: the compiler would take two loads for the three that are used)
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(k.x), "=f"(k.y), "=f"(k.z), "=f"(k.w)
                         : "r"(tb_at + t * 16));
            R xr;
            xr.v = xw[t * CG];
            const V xt = xr.get();
            const V u = silu(vfma(w3, xt, vfma(w2, x1, vfma(w1, x2, vfma(w0, x3, bias)))));
            h = sfma(k.x, h, smul(k.y, u));
            y[t] = sfma(k.z, h, vmul(dd, u));
            x3 = x2;
            x2 = x1;
            x1 = xt;
            // x during all of them, or z during the first half and x the second
            constexpr int X0 = Z2 ? 0 : LC / 2, SPAN = LC - X0, EVERY = SPAN / COPIES > 0 ? SPAN / COPIES : 1;
            constexpr int EACH = (COPIES + SPAN / EVERY - 1) / (SPAN / EVERY);
#pragma unroll
            for (int n = 0; n < EACH; ++n) {
                const int c = t % SPAN / EVERY * EACH + n;
                if ((t + 1) % EVERY == 0 && c < COPIES) {
                    if (t < X0) copy(from_z, to_z, c, spread_z);
                    else copy(from_x, to_x, c, spread_x);
                }
            }
            if (!Z2 && t == X0 - 1) commit();
            return k.x;
        };
        if (!Z2 && gate && rows_left && !spread_z) stage_rows(r0, p.z, next_z, sz);
        // (by warps: one with both kinds of part would run both loops)
        const bool even = rows_left && (plain || (valid == mask && !start && !end && (info[0] & 3) == 3));
        if (__all_sync(0xffffffffu, even)) {
#pragma unroll
            for (int t = 0; t < LC; ++t) token(t);
        } else {
            if (!even && (valid & 1u) && !(start & 1u)) {
                const int place = info[0] & 3;
                if (place < 3) x3 = back(3, place, info[0]);
                if (place < 2) x2 = back(2, place, info[0]);
            }
            float A = 1.0f;
            // One start at most and no end behind it: selects instead of
            // branches, which would keep the tokens from overlapping (one warp
            // took 250 cycles a token, and the others wait for it).
            if (__all_sync(0xffffffffu, !(start & (start - 1u)) && !(start && end >= start))) {
                const int first_t = __ffs(start) - 1, end_t = __ffs(end) - 1;
                R i1, i2, i3;
                i1.zero();
                i2.zero();
                i3.zero();
                V ih;
                vset(ih, 0.0f, 0.0f);
                if (start && on && !(info[first_t] & 4)) {
                    i1.v = init_x[part][2][cg];
                    i2.v = init_x[part][1][cg];
                    i3.v = init_x[part][0][cg];
                    ih = init_h[part][cg];
                }
                if (end) {
                    end_info = info[end_t];
                    R r;
                    r.v = xw[end_t * CG];
                    e1 = r.get();
                    e2 = x1;
                    e3 = end_t ? x1 : x2;
                    if (end_t >= 1) {
                        r.v = xw[(end_t - 1) * CG];
                        e2 = r.get();
                    }
                    if (end_t >= 2) {
                        r.v = xw[(end_t - 2) * CG];
                        e3 = r.get();
                    }
                }
#pragma unroll
                for (int t = 0; t < LC; ++t) {
                    const bool here = t == first_t;
                    x1 = here ? i1.get() : x1;
                    x2 = here ? i2.get() : x2;
                    x3 = here ? i3.get() : x3;
                    h = here ? ih : h;
                    A *= token(t);
                    he = t == end_t ? h : he;
                    Ae = t == end_t ? A : Ae;
                }
            } else {
#pragma unroll
            for (int t = 0; t < LC; ++t) {
                if (start >> t & 1u) {
                    const bool from = on && !(info[t] & 4);
                    if (from && (start & ((1u << t) - 1u)) == 0) {  // fetched
                        R r;
                        r.v = init_x[part][2][cg];
                        x1 = r.get();
                        r.v = init_x[part][1][cg];
                        x2 = r.get();
                        r.v = init_x[part][0][cg];
                        x3 = r.get();
                        h = init_h[part][cg];
                    } else {
                        x1 = back(1, 0, info[t]);
                        x2 = back(2, 0, info[t]);
                        x3 = back(3, 0, info[t]);
                        const float *hs = p.l.h + (int64_t)(info[t] >> 4) * C + ch;
                        vset(h, from ? hs[0] : 0.0f, from ? hs[VEC - 1] : 0.0f);
                    }
                }
                A *= token(t);
                if (end >> t & 1u) {
                    if (start & ((2u << t) - 1u)) {
                        keep(info[t] >> 4, x3, x2, x1, h);
                    } else {
                        // completed and written below, when the state that
                        // came in is known
                        end_info = info[t];
                        Ae = A;
                        he = h;
                        e1 = x1;
                        e2 = x2;
                        e3 = x3;
                    }
                }
            }
            }
        }
        part_s[part][cg] = h;
        part_a[part][cg] = start ? SET : decs[(buf * heads + hh) * ST + part];
        if (!PRE && r1 < p.rows) head_table(r1, buf ^ 1);
        if (r1 < p.rows && !spread_x) stage_rows(r1, p.x, next_x, sx + (buf ^ 1) * L::WORDS);
        next_x += step * p.ld;
        if (!Z2) next_z += step * p.ld;
        commit();
        __syncthreads();
        float a = 1.0f;
        V S;
        vset(S, 0.0f, 0.0f);
        float av[GP];
        V Sv[GP];
        if (scans) {
#pragma unroll
            for (int i = 0; i < GP; ++i) {
                av[i] = part_a[sp * GP + i][sc];
                Sv[i] = part_s[sp * GP + i][sc];
            }
#pragma unroll
            for (int i = 0; i < GP; ++i) {
                S = through(av[i], S, Sv[i]);
                a = through(a, av[i]);
            }
#pragma unroll
            for (int o = 1; o < SG; o <<= 1) {
                const float a1 = shfl_up(a, o, SG);
                const V S1 = shfl_up(S, o, SG);
                if (sp >= o) {
                    S = through(a, S1, S);
                    a = through(a1, a);
                }
            }
            if (many > 1 && sp == SG - 1) {
                tile_a[buf][sc] = a;
                tile_s[buf][sc] = S;
            }
        }
        if (many > 1) cluster_sync();
        if (scans) {
            const float a1 = shfl_up(a, 1, SG);
            const V S1 = shfl_up(S, 1, SG);
            float an = shfl_at(a, SG - 1, SG);
            V Sn = shfl_at(S, SG - 1, SG), in = carry;
            if (many > 1) {
                for (int j = 0; j < many; ++j) {
                    load_remote(remote(&tile_a[buf][sc], j), an);
                    load_remote(remote(&tile_s[buf][sc], j), Sn);
                    carry = through(an, carry, Sn);
                    if (j + 1 == rank) in = carry;
                }
            } else {
                carry = through(an, carry, Sn);
            }
            if (sp > 0) in = through(a1, in, S1);
#pragma unroll
            for (int i = 0; i < GP; ++i) {
                came[sp * GP + i][sc] = in;
                in = through(av[i], in, Sv[i]);
            }
        }
        // the next tile's rows: inside the sequence of this tile's last row,
        // nothing has to be looked up
        if (r1 < p.rows) {
            const bool same = (plain || (row_info[ROWS - 1] >= 0 && last_info >= 0)) && r1 >= last_begin + 3 &&
                              r1 + ROWS < last_end && r1 + ROWS <= p.rows;
            if (!same) {
                __syncthreads();  // every thread is done with this tile's rows
                describe_rows(r1);
            }
            plain = same;
        }
        asm volatile("cp.async.wait_group 1;" ::: "memory");  // z
        __syncthreads();
        if (Z2 && gate && r1 < p.rows && !spread_z) stage_rows(r1, p.z, next_z, sz + (buf ^ 1) * L::WORDS);
        if (r1 < p.rows && !plain) fetch_init();
        const V hin = came[part][cg];
        if (end_info >= 0) {
            V aa;
            vset(aa, Ae, Ae);
            keep(end_info >> 4, e3, e2, e1, vfma(aa, hin, he));
        }
        const bool whole = __all_sync(0xffffffffu, valid == mask && !start);
        if (on) {
            const int begin = start ? __ffs(start) - 1 : LC;
            T *py = static_cast<T *>(p.y) + ch + (r0 + b0) * p.ldy;
            auto ahead = [&](int t) {  // the next tile's z
                constexpr int EVERY = LC / COPIES > 0 ? LC / COPIES : 1, EACH = (COPIES + LC - 1) / LC;
                if (!Z2 || (t + 1) % EVERY) return;
#pragma unroll
                for (int n = 0; n < EACH; ++n)
                    if (t / EVERY * EACH + n < COPIES) copy(from_z, to_z, t / EVERY * EACH + n, spread_z);
            };
            auto finish = [&](int t, bool fix, auto gated) {
                V o = y[t];
                if (fix) o = sfma(tb[t].w, hin, o);
                if (decltype(gated)::value) {
                    R zr;
                    zr.v = zw[t * CG];
                    o = vmul(o, silu(zr.get()));
                }
                if (whole || (valid >> t & 1u)) put(py, o);
            };
            auto outputs = [&](auto gated) {
                if (whole) {
#pragma unroll
                    for (int t = 0; t < LC; ++t, py += p.ldy) {
                        ahead(t);
                        finish(t, true, gated);
                    }
                } else {
#pragma unroll
                    for (int t = 0; t < LC; ++t, py += p.ldy) {
                        ahead(t);
                        finish(t, t < begin, gated);  // (a branch for each would keep them from overlapping)
                    }
                }
            };
            if (gate) outputs(std::true_type());
            else outputs(std::false_type());
        }
        if (Z2) {
            next_z += step * p.ld;
            commit();
        }
    }
    if (many > 1) cluster_sync();  // (nobody reads here any more)
    // sequences without tokens that start afresh: a zero state
    if (rank == 0) {
        for (int s0 = 0; s0 < p.n_seq; s0 += NT) {
            const int s = s0 + tid;
            int slot = -1;
            if (s < p.n_seq && off_at(s) >= off_at(s + 1)) {
                const int i = cached ? s_info[s] : load_info(s);
                if (i >= 0 && (i & 4)) slot = i >> 4;
            }
            if (!__syncthreads_or(slot >= 0)) continue;
            if (tid == 0) n_list = 0;
            __syncthreads();
            if (slot >= 0) list[atomicAdd(&n_list, 1)] = slot;
            __syncthreads();
            V none;
            vset(none, 0.0f, 0.0f);
            for (int i = part; i < n_list; i += ST) keep(list[i], none, none, none, none);
            __syncthreads();
        }
    }
}

struct Launch {
    Args a;
    bm_ctx_t *ctx;
    int device, sms;
    cudaStream_t s;
};

// CTAs of a cluster, for SMs that would be idle.  Clusters of 8 only where they
// leave a third of the SMs: 16 of them do not fit the GPCs at once, and the
// second turn costs more than they save (1500 x 512 bf16 17 us, of 4 14).
int cluster_of(int n_cb, int64_t tiles, int at_once) {
    int many = 1;
    while (many < 8 && many < tiles && n_cb * many * 2 <= (many < 4 ? at_once : at_once * 2 / 3)) many *= 2;
    return many;
}

template <typename T, int VEC, int CG, int ST, int LC, int PER_SM, bool PRE>
int launch_prefill(Launch &l) {
    using L = Tile<T, VEC, CG, ST, LC, PRE>;
    Args &a = l.a;
    const int C = a.l.C, P = a.l.P, H = a.l.H;
    const int n_cb = (C + CG * VEC - 1) / (CG * VEC);
    const int tiles = a.rows > 0 ? (int)(((int64_t)a.rows + L::ROWS - 1) / L::ROWS) : 1;
    const int many = cluster_of(n_cb, tiles, l.sms * PER_SM);
    const int64_t parts = ((int64_t)a.rows + LC - 1) / LC;
    // (at most BM_WORK_SCAN_MOST: bm_ssm_prefill takes no table of more than 2^26
    // rows times heads, and a pair's heads have 16 channels or more)
    const size_t tab_bytes = PRE ? (size_t)parts * H * (LC * sizeof(float4) + sizeof(float)) : 0;
    if (PRE) {
        void *work;
        const int rc = bm_detail_work(l.ctx, BM_WORK_SCAN, tab_bytes, &work);
        if (rc != BM_OK) return rc;
        a.tab = static_cast<const float4 *>(work);
        a.dec = reinterpret_cast<const float *>(a.tab + parts * H * LC);
        const int64_t blocks = (parts * H + 127) / 128;
        if (blocks > INT32_MAX) return bm_detail_fail(BM_ERR_UNSUPPORTED, "rows * heads too large for one call");
        BMC_CK(bmc::launch(heads_kernel<T, LC>, dim3((unsigned)blocks), 128, 0, l.s, a, const_cast<float4 *>(a.tab),
                           const_cast<float *>(a.dec)));
    }
    int heads = (CG * VEC + P - 2) / P + 1;
    if (heads > H) heads = H;
    const size_t bytes = L::STAGED + (size_t)heads * L::PER_HEAD;
    // a pair's head has 16 channels or more (bm_ssm_prefill)
    constexpr int most = (int)(L::STAGED + (VEC == 2 ? (CG * VEC + 14) / 16 + 1 : CG) * L::PER_HEAD);
    if (bytes > most) return bm_detail_fail(BM_ERR_UNSUPPORTED, "too many heads in a tile");
    auto even = [&](const void *q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
    const int wide = C % (CG * VEC) == 0 && even(a.x) && even(a.z) && a.ld * (int64_t)sizeof(T) % 16 == 0;
    auto *k = prefill_kernel<T, VEC, CG, ST, LC, PER_SM, PRE>;
    static bmc::SharedMemory shm;
    BMC_CK(shm.allow(reinterpret_cast<const void *>(k), most, l.device));
    cudaLaunchConfig_t c{};
    cudaLaunchAttribute at[2];
    c.gridDim = dim3((unsigned)n_cb, (unsigned)many);
    c.blockDim = dim3(L::NT);
    c.dynamicSmemBytes = bytes;
    c.stream = l.s;
    c.attrs = at;
    if (many > 1) {
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = at[0].val.clusterDim.z = 1;
        at[0].val.clusterDim.y = (unsigned)many;
        c.numAttrs = 1;
    }
    if (PRE) {  // starts while heads_kernel runs, and waits for it before it uses the table
        at[c.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[c.numAttrs].val.programmaticStreamSerializationAllowed = 1;
        ++c.numAttrs;
    }
    BMC_CK(cudaLaunchKernelEx(&c, k, static_cast<const Args>(a), heads, wide));
    return BM_OK;
}

// ----------------------------------------------------------- single tokens --
//
// Bound by the bytes of the states: 4 of h and 3 inputs read and written per
// channel against one x, z and y.  A thread has VEC channels (16 bytes of
// fp32, 8 of bf16), loads everything of a row before it uses any of it, and
// keeps its weights for the next row that it takes.  1024 x 4096 fp32 takes 35
// us, 5.3 TB/s.
template <typename T, int VEC>
struct Pack;
template <>
struct Pack<float, 4> {
    float4 v;
    __device__ __forceinline__ float at(int i) const { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
    __device__ __forceinline__ void set(const float (&f)[4]) { v = make_float4(f[0], f[1], f[2], f[3]); }
};
template <>
struct Pack<__nv_bfloat16, 4> {
    uint2 v;
    __device__ __forceinline__ float at(int i) const {
        const uint32_t w = i < 2 ? v.x : v.y;
        return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
    }
    __device__ __forceinline__ void set(const float (&f)[4]) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
        v = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    }
};
template <typename T>
struct Pack<T, 1> {
    T v;
    __device__ __forceinline__ float at(int) const { return to_f(v); }
    __device__ __forceinline__ void set(const float (&f)[1]) { v = from_f<T>(f[0]); }
};

template <typename T, int VEC>
__global__ void __launch_bounds__(128) step_kernel(const Args p) {
    using W = Pack<T, VEC>;
    using F = Pack<float, VEC>;
    const int ch = (blockIdx.x * 128 + threadIdx.x) * VEC;
    if (ch >= p.l.C) return;
    const int hd = ch / p.l.P;  // (VEC > 1: one head's channels)
    float4 w[VEC];
    float bias[VEC], d[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        w[v] = reinterpret_cast<const float4 *>(p.l.conv_w)[ch + v];
        bias[v] = p.l.conv_b[ch + v];
        d[v] = p.l.d[ch + v];
    }
    const float dt_bias = p.l.dt_bias[hd], rate = expf(p.l.a_log[hd]);
    for (int r = blockIdx.y; r < p.rows; r += gridDim.y) {
        const int slot = p.slots ? p.slots[r] : r;
        if (slot < 0 || slot >= p.l.n_slots) continue;
        W *c0 = reinterpret_cast<W *>(static_cast<T *>(p.l.conv) + (int64_t)slot * 3 * p.l.C + ch);
        W *c1 = reinterpret_cast<W *>(reinterpret_cast<T *>(c0) + p.l.C), *c2 = reinterpret_cast<W *>(reinterpret_cast<T *>(c1) + p.l.C);
        F *hs = reinterpret_cast<F *>(p.l.h + (int64_t)slot * p.l.C + ch);
        const int64_t at = (int64_t)r * p.ld;
        const W x3 = *c0, x2 = *c1, x1 = *c2;
        F h = *hs;
        const W x0 = *reinterpret_cast<const W *>(static_cast<const T *>(p.x) + at + ch);
        W z = x0;
        if (p.z) z = *reinterpret_cast<const W *>(static_cast<const T *>(p.z) + at + ch);
        const T dt = static_cast<const T *>(p.dt)[at + hd], b = static_cast<const T *>(p.b)[at + hd],
                c = static_cast<const T *>(p.c)[at + hd];
        const Head k = head_of(to_f(dt) + dt_bias, rate, to_f(b), to_f(c));
        float hn[VEC], y[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const float u = silu(fmaf(
                w[v].w, x0.at(v), fmaf(w[v].z, x1.at(v), fmaf(w[v].y, x2.at(v), fmaf(w[v].x, x3.at(v), bias[v])))));
            hn[v] = fmaf(k.a, h.at(v), k.g * u);
            y[v] = fmaf(k.c, hn[v], d[v] * u);
            if (p.z) y[v] *= silu(z.at(v));
        }
        W o;
        o.set(y);
        *reinterpret_cast<W *>(static_cast<T *>(p.y) + (int64_t)r * p.ldy + ch) = o;
        *c0 = x2;
        *c1 = x1;
        *c2 = x0;
        h.set(hn);
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
    if (misaligned(slots, 4)) return bm_detail_fail(BM_ERR_INVALID_ARG, "slots not 4-byte aligned");
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
    if (misaligned(d_fresh, 4)) return bm_detail_fail(BM_ERR_INVALID_ARG, "fresh not 4-byte aligned");
    a.off = d_seq_off;
    a.n_seq = n_seq;
    a.fresh = d_fresh;
    const size_t e = layer->type == BM_F32 ? 4 : 2;
    // two channels a thread: a pair is one head's, and every pair is aligned
    const bool pairs = a.l.P % 2 == 0 && a.l.P >= 16 && ld % 2 == 0 && ldy % 2 == 0 &&
                       !misaligned(d_x, 2 * e) && !misaligned(d_z, 2 * e) &&
                       !misaligned(d_y, 2 * e) && !misaligned(layer->conv_state, 2 * e) &&
                       !misaligned(layer->h_state, 8);
    if (layer->n_slots > (1 << 27)) return bm_detail_fail(BM_ERR_UNSUPPORTED, "n_slots > 2^27");
    if (rows > INT32_MAX - 65536) return bm_detail_fail(BM_ERR_UNSUPPORTED, "rows > 2^31 - 65537");
    Launch l{};
    l.ctx = ctx;
    int *err;
    l.device = bm_detail_ctx(ctx, &l.sms, &err, &l.s);
    bmc::DeviceGuard guard(l.device);
    BMC_CK(guard.error);
    if (stream) l.s = static_cast<cudaStream_t>(stream);
    l.a = a;
    // Small tiles for few rows.  One channel a thread for what cannot be paired
    // and for heads so small that the scalars of a tall tile's rows would not
    // fit the shared memory.
    using bf16 = __nv_bfloat16;
    const bool f32 = layer->type == BM_F32;
    if (!pairs)
        return f32 ? launch_prefill<float, 1, 32, 16, 8, 1, false>(l) : launch_prefill<bf16, 1, 32, 16, 8, 1, false>(l);
    if (rows <= 64)
        return f32 ? launch_prefill<float, 2, 16, 8, 8, 4, false>(l) : launch_prefill<bf16, 2, 16, 8, 8, 4, false>(l);
    // The head scalars of few tiles cost less in the CTAs than a launch for them
    // (about 1 us), which in turn makes fp32's tiles of 256 rows 0.4 us shorter
    // (4 turns: 22.2 us instead of 23.0 for 4096 channels, 3 the same) and lets
    // bf16's have 512 rows (5.7 us a turn instead of 4.0 for 256).  A table
    // larger than the inputs is no use.
    const int n_cb = (a.l.C + 31) / 32;
    auto turns = [&](int tile) {
        const int64_t tiles = ((int64_t)rows + tile - 1) / tile;
        const int many = cluster_of(n_cb, tiles, l.sms);
        return (tiles + many - 1) / many;
    };
    const bool table = f32 ? turns(256) >= 4 : 57 * turns(512) + 10 < 40 * turns(256);
    if (!table || (int64_t)rows * a.l.H > ((int64_t)1 << 26))
        return f32 ? launch_prefill<float, 2, 16, 32, 8, 1, false>(l) : launch_prefill<bf16, 2, 16, 32, 8, 1, false>(l);
    return f32 ? launch_prefill<float, 2, 16, 32, 8, 1, true>(l) : launch_prefill<bf16, 2, 16, 32, 16, 1, true>(l);
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
    // (a CTA's next row, up to 65535 further, stays in 31 bits)
    if (rows > INT32_MAX - 65536) return bm_detail_fail(BM_ERR_UNSUPPORTED, "rows > 2^31 - 65537");
    int sms, *err;
    cudaStream_t s;
    bmc::DeviceGuard guard(bm_detail_ctx(ctx, &sms, &err, &s));
    BMC_CK(guard.error);
    if (stream) s = static_cast<cudaStream_t>(stream);
    const size_t e = layer->type == BM_F32 ? 4 : 2;
    const bool quads = a.l.P % 4 == 0 && ld % 4 == 0 && ldy % 4 == 0 && !misaligned(d_x, 4 * e) &&
                       !misaligned(d_z, 4 * e) && !misaligned(d_y, 4 * e) &&
                       !misaligned(layer->conv_state, 4 * e) && !misaligned(layer->h_state, 16);
    const int vec = quads ? 4 : 1;
    const unsigned across = (unsigned)((a.l.C + 128 * vec - 1) / (128 * vec));
    // about 16 CTAs per SM in all; beyond that, several rows each
    unsigned down = (unsigned)(16 * sms) / across + 1;
    if (down > 65535) down = 65535;
    if (down > (unsigned)rows) down = (unsigned)rows;
    const dim3 grid(across, down);
    using bf16 = __nv_bfloat16;
    auto *k = layer->type == BM_F32 ? (quads ? step_kernel<float, 4> : step_kernel<float, 1>)
                                    : (quads ? step_kernel<bf16, 4> : step_kernel<bf16, 1>);
    BMC_CK(bmc::launch(k, grid, 128, 0, s, a));
    return BM_OK;
}

}  // extern "C"
