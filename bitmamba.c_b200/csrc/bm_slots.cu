// Slots of a state cache moved within their arrays by a row map: copies, one
// slot forked to many, permutations and compaction, in place.
//
// Slot s takes what slot src[s] held before the call, for all s as if at
// once.  Columns of a row are independent, so a CTA owns one piece of columns
// of one plane for EVERY moved slot: it reads the pieces of all sources into
// shared memory, and only then writes the destinations.  No ordering between
// slots, no second copy of the cache and no wait between CTAs is needed, for
// any map.  Bound by memory: half of 1024 slots of 8 x 4096 fp32 states and
// convolution inputs (537 MB read and written) take 98 us, 5.5 TB/s.
#include <cstdint>
#include <cstdio>

#include <cuda_runtime.h>

#include "bm_ctx.cuh"
#include "bm_slots.cuh"

namespace {

constexpr int NT = 512;
constexpr int MAX_REGIONS = 2 * BM_SLOT_REGIONS;
constexpr int PIECE_MAX = 4096;

struct Region {
    unsigned char *base;
    int64_t row_bytes, row_pitch, outer_pitch;
    int n_outer, unit;  // unit: 16 or 4 bytes per access
};
struct Regions {
    Region r[MAX_REGIONS];
    int n;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Dynamic shared memory: the list of moves ((src << 16) | dst, n_slots words
// rounded up to 16 bytes), then `buffers` times `room` bytes of pieces: with
// two, the next piece's sources are read while this one's destinations are
// written (one after the other took 112 us where this takes 98: 537 MB).
__global__ void __launch_bounds__(NT)
    reorder_kernel(const __grid_constant__ Regions g, const int32_t *src, int n_slots, int room,
                   int buffers) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int n_moves, s_piece;
    __shared__ unsigned per[MAX_REGIONS], items[MAX_REGIONS];
    uint32_t *list = reinterpret_cast<uint32_t *>(smem);
    unsigned char *const bufs = smem + ((size_t)n_slots * 4 + 15) / 16 * 16;
    if (threadIdx.x == 0) n_moves = 0;
    __syncthreads();
    for (int s = threadIdx.x; s < n_slots; s += NT) {
        const int from = src[s];
        if (from != s && from >= 0 && from < n_slots)
            list[atomicAdd(&n_moves, 1)] = ((uint32_t)from << 16) | (uint32_t)s;
    }
    __syncthreads();
    const int n = n_moves;
    if (n == 0) return;
    // columns per piece: as many as fit the room n times, in lines of 128 bytes
    // (pieces of 96 bytes took 139 us where 128 take 98) or a power of two
    // below one; where that is less than a piece for every CTA, smaller ones
    if (threadIdx.x == 0) {
        int64_t columns = 0;
        for (int k = 0; k < g.n; ++k) columns += g.r[k].row_bytes * g.r[k].n_outer;
        int piece = min(PIECE_MAX, room / n);
        if (piece >= 128) {
            const int64_t share = (columns / gridDim.x + 127) & ~(int64_t)127;
            piece = (int)max((int64_t)128, min((int64_t)piece, share)) & ~127;
        } else {
            piece = 1 << (31 - __clz(piece));  // (16 at least: the room is 16 bytes a slot)
        }
        s_piece = piece;
        for (int k = 0; k < g.n; ++k) {
            per[k] = (unsigned)((g.r[k].row_bytes + piece - 1) / piece);
            items[k] = per[k] * (unsigned)g.r[k].n_outer;
        }
    }
    __syncthreads();
    const int piece = s_piece;
    // an item: a piece of columns of a plane of a region
    struct Item {
        int region;
        unsigned at;
    };
    auto settle = [&](Item &i) {  // to the region that it falls into; false: past the last
        for (; i.region < g.n; ++i.region) {
            if (i.at < items[i.region]) return true;
            i.at -= items[i.region];
        }
        return false;
    };
    auto each = [&](const Item &it, auto &&f) {
        const Region &r = g.r[it.region];
        const unsigned o = it.at / per[it.region];
        const int64_t col = (int64_t)(it.at - o * per[it.region]) * piece;
        unsigned char *plane = r.base + o * r.outer_pitch + col;
        const int words = (int)min((int64_t)piece, r.row_bytes - col) / r.unit, total = n * words;
        const unsigned inverse = 0xffffffffu / (unsigned)words + 1;  // (0 for one word)
        for (int i = threadIdx.x; i < total; i += NT) {
            // i / words, exact: i * words < 2^32
            const int m = words == 1 ? i : (int)__umulhi((unsigned)i, inverse), w = i - m * words;
            f(r.unit, plane + w * r.unit, r.row_pitch, list[m], m * piece + w * r.unit);
        }
    };
    auto read = [&](const Item &it, unsigned char *buf) {
        const uint32_t buf0 = (uint32_t)__cvta_generic_to_shared(buf);
        each(it, [&](int unit, unsigned char *p, int64_t pitch, uint32_t move, int at) {
            p += (int64_t)(move >> 16) * pitch;
            if (unit == 16) cp16(buf0 + at, p);
            else *reinterpret_cast<uint32_t *>(buf + at) = *reinterpret_cast<const uint32_t *>(p);
        });
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    Item now{0, blockIdx.x};
    bool more = settle(now);
    if (more) read(now, bufs);
    for (int k = 0; more; k ^= 1) {
        Item next{now.region, now.at + gridDim.x};
        more = settle(next);
        unsigned char *buf = bufs + (buffers == 2 ? k * room : 0);
        if (more && buffers == 2) {
            read(next, bufs + (k ^ 1) * room);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        __syncthreads();  // every source of this item is read
        each(now, [&](int unit, unsigned char *p, int64_t pitch, uint32_t move, int at) {
            p += (int64_t)(move & 0xffffu) * pitch;
            if (unit == 16) *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(buf + at);
            else *reinterpret_cast<uint32_t *>(p) = *reinterpret_cast<const uint32_t *>(buf + at);
        });
        __syncthreads();  // the buffer is free
        if (more && buffers == 1) read(next, bufs);
        now = next;
    }
}

bool all_multiple(const bm_slot_region_t &r, int64_t n) {
    return (int64_t)(reinterpret_cast<uintptr_t>(r.base) % (uintptr_t)n) == 0 &&
           r.row_bytes % n == 0 && r.row_pitch % n == 0 && r.outer_pitch % n == 0;
}

}  // namespace

namespace bms {

int check_regions(const bm_slot_region_t *regions, int n_regions) {
    if (n_regions < 0 || n_regions > BM_SLOT_REGIONS || (n_regions > 0 && !regions))
        return bm_detail_fail(BM_ERR_INVALID_ARG, "regions NULL, or their number outside [0, 8]");
    for (int i = 0; i < n_regions; ++i) {
        const bm_slot_region_t &r = regions[i];
        const char *why = nullptr;
        if (!r.base) why = "base is NULL";
        else if (r.row_bytes < 1 || r.n_outer < 1) why = "row_bytes or n_outer < 1";
        else if (!all_multiple(r, 4)) why = "base, row_bytes or a pitch not a multiple of 4";
        // (pieces of 16 bytes or more, counted in 32 bits with a grid to spare)
        else if (r.row_bytes > INT32_MAX || (r.row_bytes + 15) / 16 * r.n_outer > INT32_MAX)
            why = "more than 2^31 - 1 pieces of 16 bytes in the rows of a slot";
        else if (r.row_pitch < r.row_bytes || (r.n_outer > 1 && r.outer_pitch < r.row_bytes))
            why = "a pitch below row_bytes";
        if (why) {
            char buf[128];
            snprintf(buf, sizeof(buf), "region %d: %s", i, why);
            return bm_detail_fail(BM_ERR_INVALID_ARG, buf);
        }
    }
    return BM_OK;
}

cudaError_t reorder(const bm_slot_region_t *regions, int n_regions, const int32_t *d_src,
                    int n_slots, int sms, cudaStream_t s) {
    Regions g{};
    for (int i = 0; i < n_regions; ++i)
        g.r[i] = Region{static_cast<unsigned char *>(regions[i].base), regions[i].row_bytes,
                        regions[i].row_pitch, regions[i].outer_pitch, regions[i].n_outer,
                        all_multiple(regions[i], 16) ? 16 : 4};
    g.n = n_regions;
    // three CTAs per SM with a buffer of 64 KB each for few slots (64 of 8 x 4096
    // permuted: 12.4 us, 14.5 the other way), one CTA with two of 96 KB (300 of
    // 4 x 512: 6.3 us, 7.9 the other way), then one buffer
    const int list = (n_slots * 4 + 15) / 16 * 16, per_sm = n_slots <= 128 ? 3 : 1;
    const int buffers = n_slots > 128 && n_slots <= 4096 ? 2 : 1;
    const int room = n_slots <= 128 ? 64 * 1024 : n_slots <= 4096 ? 96 * 1024 : n_slots * 16;
    const size_t bytes = (size_t)list + (size_t)room * buffers;
    // the most that any call takes
    constexpr int most = 4096 * 4 + 2 * 96 * 1024;
    static_assert(most >= BM_SLOT_MAX * (4 + 16), "shared memory");
    int device;
    cudaError_t e = cudaGetDevice(&device);
    static bmc::SharedMemory shm;
    if (e == cudaSuccess) e = shm.allow(reinterpret_cast<const void *>(reorder_kernel), most, device);
    if (e != cudaSuccess) return e;
    return bmc::launch(reorder_kernel, dim3((unsigned)(sms * per_sm)), NT, bytes, s, g, d_src, n_slots, room, buffers);
}

}  // namespace bms

extern "C" int bm_slots_reorder(bm_ctx_t *ctx, const bm_slot_region_t *regions, int n_regions,
                                const int32_t *d_src, int n_slots, void *stream) {
    if (!ctx) return bm_detail_fail(BM_ERR_INVALID_ARG, "ctx is NULL");
    int rc = bms::check_regions(regions, n_regions);
    if (rc != BM_OK) return rc;
    if (n_slots < 0) return bm_detail_fail(BM_ERR_INVALID_ARG, "n_slots < 0");
    if (n_slots > BM_SLOT_MAX)
        return bm_detail_fail(BM_ERR_UNSUPPORTED, "n_slots > BM_SLOT_MAX (8192)");
    if (n_slots == 0 || n_regions == 0) return BM_OK;
    if (!d_src || reinterpret_cast<uintptr_t>(d_src) % 4)
        return bm_detail_fail(BM_ERR_INVALID_ARG, "src NULL or not 4-byte aligned");
    int sms, *err;
    cudaStream_t s;
    bmc::DeviceGuard guard(bm_detail_ctx(ctx, &sms, &err, &s));
    BMC_CK(guard.error);
    if (stream) s = static_cast<cudaStream_t>(stream);
    BMC_CK(bms::reorder(regions, n_regions, d_src, n_slots, sms, s));
    return BM_OK;
}
