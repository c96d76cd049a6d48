// Attention of a chunk over a paged cache: 16-bit queries over an fp8 pool.
#include <type_traits>

#include "vrm_chunk16.h"

namespace vrm {

void launch_chunk16_fp8(const ChunkArgs& a, dim3 grid, hipStream_t st) {
  if (a.q_type == VRM_SRC_BF16)
    launch_chunk16_t<Bf16, kSrcFp8>(a, grid, st);
  else
    launch_chunk16_t<F16, kSrcFp8>(a, grid, st);
}

}  // namespace vrm
