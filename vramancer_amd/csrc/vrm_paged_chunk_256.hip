// Attention of a chunk over a paged cache: head dims from 129 to 256.
#include <type_traits>

#include "vrm_chunk16.h"

namespace vrm {

namespace {
template <typename T, int KIND>
void launch(const ChunkArgs& a, dim3 grid, hipStream_t st) {
  hipLaunchKernelGGL((chunk_attn_kernel<T, KIND, 256>), grid, dim3(kChunkThreads), 0, st, a);
}
}  // namespace

void launch_chunk16_256(const ChunkArgs& a, int kind, dim3 grid, hipStream_t st) {
  const bool bf16 = a.q_type == VRM_SRC_BF16;
  if (kind == kSrcI8)
    bf16 ? launch<Bf16, kSrcI8>(a, grid, st) : launch<F16, kSrcI8>(a, grid, st);
  else if (kind == kSrcFp8)
    bf16 ? launch<Bf16, kSrcFp8>(a, grid, st) : launch<F16, kSrcFp8>(a, grid, st);
  else
    bf16 ? launch<Bf16, kSrcBf16>(a, grid, st) : launch<F16, kSrcF16>(a, grid, st);
}

}  // namespace vrm
