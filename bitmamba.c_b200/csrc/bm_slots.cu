// Slots of a state cache moved within their arrays by a row map: copies, one
// slot forked to many, permutations and compaction, in place.
//
// Slot s takes what slot src[s] held before the call, for all s as if at
// once.  Columns of a row are independent, so a CTA owns one piece of columns
// of one plane for EVERY moved slot: it reads the pieces of all sources into
// shared memory, and only then writes the destinations.  No ordering between
// slots, no second copy of the cache and no wait between CTAs is needed, for
// any map.
#include <cstdint>
#include <cstdio>

#include <cuda_runtime.h>

#include "bm_ctx.cuh"
#include "bm_slots.cuh"

namespace {

constexpr int NT = 256;
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
// rounded up to 16 bytes), then `room` bytes of pieces.
__global__ void __launch_bounds__(NT)
    reorder_kernel(const __grid_constant__ Regions g, const int32_t *src, int n_slots, int room) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int n_moves;
    uint32_t *list = reinterpret_cast<uint32_t *>(smem);
    unsigned char *buf = smem + ((size_t)n_slots * 4 + 15) / 16 * 16;
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
    // columns per piece: a power of two of which n fit the room, and small
    // enough that every CTA has some
    int64_t columns = 0;
    for (int k = 0; k < g.n; ++k) columns += g.r[k].row_bytes * g.r[k].n_outer;
    int piece = PIECE_MAX;
    while (piece > 16 && ((int64_t)piece * n > room || (piece > 256 && columns < (int64_t)2 * piece * gridDim.x)))
        piece >>= 1;
    const uint32_t buf0 = (uint32_t)__cvta_generic_to_shared(buf);
    int64_t item = blockIdx.x;
    for (int k = 0; k < g.n; ++k) {
        const Region &r = g.r[k];
        const int64_t per = (r.row_bytes + piece - 1) / piece, items = per * r.n_outer;
        for (; item < items; item += gridDim.x) {
            const int64_t col = item % per * piece;
            unsigned char *plane = r.base + item / per * r.outer_pitch + col;
            const int bytes = (int)min((int64_t)piece, r.row_bytes - col);
            const int words = bytes / r.unit;
            const int total = n * words;
            for (int i = threadIdx.x; i < total; i += NT) {
                const int m = i / words, w = i - m * words;
                const unsigned char *p = plane + (int64_t)(list[m] >> 16) * r.row_pitch + w * r.unit;
                if (r.unit == 16)
                    cp16(buf0 + m * piece + w * 16, p);
                else
                    *reinterpret_cast<uint32_t *>(buf + m * piece + w * 4) =
                        *reinterpret_cast<const uint32_t *>(p);
            }
            asm volatile("cp.async.commit_group;\n cp.async.wait_all;" ::: "memory");
            __syncthreads();  // every source is read
            for (int i = threadIdx.x; i < total; i += NT) {
                const int m = i / words, w = i - m * words;
                unsigned char *p = plane + (int64_t)(list[m] & 0xffffu) * r.row_pitch + w * r.unit;
                if (r.unit == 16)
                    *reinterpret_cast<uint4 *>(p) =
                        *reinterpret_cast<const uint4 *>(buf + m * piece + w * 16);
                else
                    *reinterpret_cast<uint32_t *>(p) =
                        *reinterpret_cast<const uint32_t *>(buf + m * piece + w * 4);
            }
            __syncthreads();  // the buffer is free
        }
        item -= items;
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
    // 64 KB of pieces (three CTAs per SM), more where that is under 16 bytes a slot
    const int room = n_slots * 16 > 65536 ? n_slots * 16 : 65536;
    const size_t bytes = ((size_t)n_slots * 4 + 15) / 16 * 16 + (size_t)room;
    // the most that any call takes
    constexpr int most = BM_SLOT_MAX * 4 + BM_SLOT_MAX * 16;
    int device;
    cudaError_t e = cudaGetDevice(&device);
    static bmc::SharedMemory shm;
    if (e == cudaSuccess) e = shm.allow(reinterpret_cast<const void *>(reorder_kernel), most, device);
    if (e != cudaSuccess) return e;
    reorder_kernel<<<sms * 3, NT, bytes, s>>>(g, d_src, n_slots, room);
    return cudaGetLastError();
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
