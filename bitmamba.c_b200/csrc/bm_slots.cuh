// Moves of slots within arrays (bm_slots.cu), shared with the decode state.
// Not part of the public ABI.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

#include "bm_sampler.h"

namespace bms {

// As bm_slots_reorder, on checked arguments (1 <= n_regions <=
// 2 * BM_SLOT_REGIONS, 1 <= n_slots <= BM_SLOT_MAX) and the current device.
cudaError_t reorder(const bm_slot_region_t *regions, int n_regions, const int32_t *d_src,
                    int n_slots, int sms, cudaStream_t s);

// Checks a caller's regions; sets bm_last_error on failure.
int check_regions(const bm_slot_region_t *regions, int n_regions);

}  // namespace bms
