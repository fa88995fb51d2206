// Host-side helpers of the tensor-core kernels, shared by their launchers (defined in tc_kernels.cu).
#pragma once
#include "fb_params.h"

#include <cuda.h>

namespace fb {

// (head_dim, rows, heads) tensor map of a sequence tensor, box 64 x box_rows x 1, cached; an absent tensor gives zeros.
int tc_tensor_map(CUtensorMap* m, const SeqT& t, int dtype, int D, int64_t rows, int heads, int box_rows);
// Dynamic shared-memory limit of `kernel` on the current device (set once per device); its number of SMs.
int tc_prepare_launch(const void* kernel, int smem_bytes, int* sm_count);
// (head, batch) pairs per scheduling group.
int tc_choose_group(const Params& p, bool dkv, int ntiles, int sm_count);

}  // namespace fb
