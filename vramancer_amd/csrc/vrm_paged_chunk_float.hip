// Attention of a chunk over a paged cache: bf16 queries over a bf16 pool, fp16 over fp16.
#include <type_traits>

#include "vrm_chunk16.h"

namespace vrm {

void launch_chunk16_float(const ChunkArgs& a, dim3 grid, hipStream_t st) {
  if (a.q_type == VRM_SRC_BF16)
    launch_chunk16_t<Bf16, kSrcBf16>(a, grid, st);
  else
    launch_chunk16_t<F16, kSrcF16>(a, grid, st);
}

}  // namespace vrm
