// Attention of a ragged batch's new tokens over a paged cache: the entry
// points, the choice of kernel and items, and the merge of items that share a
// tile.  The kernels are in vrm_chunk16.h and vrm_paged_chunk_f32.hip.
#include <math.h>

#include "vrm_chunk.h"

namespace vrm {
namespace {

// Joins the shares of a tile's rows, half a wavefront to a row: (max, sum,
// accumulator) of every share, 16 bytes of an accumulator to a lane, eight
// shares' loads under way (what another XCD wrote takes about 2 us to come).
// Bound: latency, 6 to 9 us; a wavefront to a row, share after share, took 12.
constexpr int kMergeRows = 16;  // rows of a workgroup
template <int DP>
__global__ void __launch_bounds__(256) chunk_merge_kernel(ChunkArgs a) {
  constexpr int VEC = DP <= 128 ? 1 : 2;  // 16-byte pieces of a lane
  const int vtile = blockIdx.x / a.KH, kvh = blockIdx.x % a.KH;
  const int2 r = a.rec[(long long)vtile * a.KH + kvh];
  int lo = 0, hi = a.B - 1;  // the last sequence whose tiles start at or before vtile
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (virtual_tile(a, clamp_int(a.cu[mid], 0, a.N), mid) <= vtile)
      lo = mid;
    else
      hi = mid - 1;
  }
  const Sequence s = load_sequence(a, lo);
  const int tile = vtile - virtual_tile(a, s.row0, lo);
  if (tile < 0 || tile >= tiles_of(a, s)) return;
  const int first = r.x, shares = r.y;
  if (shares <= 1 || first < 0 || shares > a.items || first > a.items - shares) return;
  const int rows = min(a.tile_rows, s.q_len * a.G - tile * a.tile_rows);
  const int l = threadIdx.x & 31;
#pragma unroll
  for (int turn = 0; turn < 2; ++turn) {
    const int row = blockIdx.y * kMergeRows + turn * 8 + (threadIdx.x >> 5);
    if (row >= rows) continue;
    const long long slot0 = ((long long)first * a.KH + kvh) * a.tile_rows + row;
    const long long next = (long long)a.KH * a.tile_rows;  // from a share's row to the next share's
    const float* const part = a.part + slot0 * DP + 4 * l;
    float top = -INFINITY, sum = 0.f;
    float4 acc[VEC] = {};
    for (int i0 = 0; i0 < shares; i0 += 8) {
      float2 ml[8];
      float4 x[8][VEC];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool on = i0 + j < shares;
        ml[j] = on ? a.ml[slot0 + (i0 + j) * next] : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int v = 0; v < VEC; ++v)
          x[j][v] = on && 4 * l + 128 * v < DP
                        ? *reinterpret_cast<const float4*>(part + (i0 + j) * next * DP + 128 * v)
                        : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float higher = top;
#pragma unroll
      for (int j = 0; j < 8; ++j) higher = fmaxf(higher, ml[j].x);
      const float f = top == -INFINITY ? 0.f : exp2f(top - higher);
      top = higher;
      sum *= f;
#pragma unroll
      for (int v = 0; v < VEC; ++v) acc[v].x *= f, acc[v].y *= f, acc[v].z *= f, acc[v].w *= f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // a share that saw nothing has no part (its maximum is -inf)
        const float w = ml[j].x == -INFINITY ? 0.f : exp2f(ml[j].x - top);
        sum += w * ml[j].y;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          acc[v].x += w * x[j][v].x, acc[v].y += w * x[j][v].y;
          acc[v].z += w * x[j][v].z, acc[v].w += w * x[j][v].w;
        }
      }
    }
    const int packed = tile * a.tile_rows + row;
    const int tok = packed / a.G;
    const long long at = (long long)(s.row0 + tok) * a.H + kvh * a.G + packed - tok * a.G;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const float y[4] = {acc[v].x * inv, acc[v].y * inv, acc[v].z * inv, acc[v].w * inv};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = 4 * l + 128 * v + e;
        if (d >= a.D) break;
        if (a.q_type == VRM_SRC_F32)
          static_cast<float*>(a.out)[at * a.D + d] = y[e];
        else if (a.q_type == VRM_SRC_F16)
          static_cast<uint16_t*>(a.out)[at * a.D + d] = __builtin_bit_cast(unsigned short, (_Float16)y[e]);
        else
          static_cast<uint16_t*>(a.out)[at * a.D + d] = __builtin_bit_cast(unsigned short, (__bf16)y[e]);
      }
    }
    if (a.lse && l == 0) a.lse[at] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
  }
}

// Items of a call, from its sizes and types alone (lengths are on the device).
struct ChunkPlan {
  bool wide;  // float32 products
  int kind;   // kSrc* of the pool
  int target, min_blocks, tile_rows, vtiles, items, dp;
  size_t rec_bytes, ml_bytes, bytes;
};

// Tiles that fill the GPU twice are left whole; fewer are cut into shares for
// about as many workgroups as are resident at once (for twice as many: a
// batch of 64 x 4 tokens over 4096 each 130 us for 118, two prompts within a
// window 123 for 87), at least kMinBlocks blocks each.  At 1, 2 and 4: 17
// tokens after 1531 21.5, 19.0 and 21.1 us, four such 27.6, 22.3 and 22.6; 5
// after 300 13.8, 14.6 and 15.9; 30 after 600 over int8 17.0, 18.1 and 23.0,
// four such 23.3, 20.4 and 24.2; 40 after 4000 30.1, 29.0 and 25.3.
constexpr int kMinBlocks = 2;

// Tiles of 256 rows from 128 rows a sequence, 1024 tokens in the table and
// this much rows x kv-heads x tokens; below, its longer start and its fewer
// workgroups cost more than its products gain.  Tiles of 128 and of 256 rows,
// 32 heads over 8 kv-heads of 128, bf16: one sequence after 2000 tokens 19.8
// and 22.5 us at 128 rows, 37.2 and 36.3 at 1024; 8 such 32.5 and 31.9 at 96,
// 85.0 and 60.9 at 384; 64 such 114 and 120 at 64, 140 and 135 at 128, 815 and
// 658 at 1024; 64 after 200 tokens 41 and 60 at 128, 226 and 242 at 1024.
// The tokens are those that a tile sees: the table's width, or what the caller
// expects, and not more than a window with the tile's own tokens and a block at
// its edge.  Within windows, after 4000 tokens: 8 sequences of 8192 rows 136
// and 188 us at a window of 64, 338 and 343 at 768, 417 and 402 at 1000, 730
// and 622 at 2000; one of 2048 rows 21 and 27, 34 and 36, 36 and 37, 48 and 44.
constexpr double kLargeWork = 1 << 24;
constexpr long long kLargeTokens = 1024;

int pool_kind(int kv_dtype) {
  switch (kv_dtype) {
    case VRM_KV_F32: return kSrcF32;
    case VRM_KV_F16: return kSrcF16;
    case VRM_KV_BF16: return kSrcBf16;
    case VRM_KV_I8:
    case VRM_KV_I8_INLINE: return kSrcI8;
    case VRM_KV_FP8E4M3:
    case VRM_KV_FP8E4M3_INLINE: return kSrcFp8;
    default: return -1;
  }
}

// expected: tokens that a sequence has, as far as the caller knows (0: the table's
// width).  With window it bears on the tiles' size only; items are counted for
// the table.
bool plan_chunk(int N, int B, int H, int KH, int D, int PS, int max_pp, int q_dtype, int kv_dtype, int expected,
                int window, ChunkPlan& p) {
  const long long G = H / KH;
  if ((long long)N * H > 0x7fff0000LL) return false;
  p.kind = pool_kind(kv_dtype);
  // 16-bit products where queries and keys have one 16-bit type (codes have any)
  p.wide = q_dtype == VRM_SRC_F32 || p.kind == kSrcF32 || (q_dtype == VRM_SRC_F16 && p.kind == kSrcBf16) ||
           (q_dtype == VRM_SRC_BF16 && p.kind == kSrcF16);
  p.dp = D <= 64 ? 64 : D <= 96 && !p.wide ? 96 : D <= 128 ? 128 : 256;
  const int block = p.wide ? 32 : 64;
  const long long tokens = (long long)max_pp * PS;           // of a sequence, at most
  const long long blocks = (tokens + block - 1) / block;
  long long seen = tokens;  // by a large tile
  if (expected > 0 && expected < seen) seen = expected;
  if (window > 0 && window + 256 / G + block < seen) seen = window + 256 / G + block;
  const bool large = !p.wide && D <= 128 && N * G >= 128LL * B && seen >= kLargeTokens &&
                     (double)(N * G) * KH * (double)seen >= kLargeWork;
  p.tile_rows = large ? 256 : 128;
  const int wanted = large ? 256 : 512;  // workgroups resident at once
  const long long vtiles = N * G / p.tile_rows + B;
  p.min_blocks = kMinBlocks;
  p.target = 0;
  long long items = vtiles;
  if (N * G / p.tile_rows * KH < 2 * wanted && blocks > kMinBlocks) {
    p.target = (wanted + KH - 1) / KH;
    const long long most = vtiles * ((blocks + kMinBlocks - 1) / kMinBlocks);
    // sum of tiles * ceil(blocks / share): target + one per tile, and the
    // rounding of the float sum that gives the share
    items = vtiles + p.target + p.target / 256 + 2;
    if (items > most) items = most;
  }
  // (a launch with 2^32 threads along x, the merge's 256 a tile too, would wrap)
  if (items * KH * (large ? kLargeThreads : kChunkThreads) > 0xffffffffLL) return false;
  p.vtiles = (int)vtiles;
  p.items = (int)items;
  p.rec_bytes = p.ml_bytes = p.bytes = 0;
  if (p.target) {
    p.rec_bytes = ((size_t)vtiles * KH * sizeof(int2) + 255) / 256 * 256;
    p.ml_bytes = (size_t)items * KH * p.tile_rows * sizeof(float2);
    p.bytes = p.rec_bytes + p.ml_bytes + (size_t)items * KH * p.tile_rows * p.dp * sizeof(float);
  }
  return true;
}

bool bad_sizes(int N, int B, int H, int KH, int D, int PS, int max_pp) {
  return N < 0 || B < 0 || H <= 0 || KH <= 0 || H % KH || D <= 0 || PS <= 0 || max_pp < 0;
}

}  // namespace
}  // namespace vrm

using namespace vrm;

extern "C" size_t vrm_paged_chunk_workspace_bytes(int N, int B, int H, int KH, int D, int PS, int max_pp, int q_dtype,
                                                  int kv_dtype) {
  ChunkPlan large, small;  // with the larger tiles, if these sizes can have them, and with the others
  if (bad_sizes(N, B, H, KH, D, PS, max_pp) || D > 256 || pool_kind(kv_dtype) < 0 ||
      !plan_chunk(N, B, H, KH, D, PS, max_pp, q_dtype, kv_dtype, 0, 0, large) ||
      !plan_chunk(N, B, H, KH, D, PS, max_pp, q_dtype, kv_dtype, 1, 0, small))
    return 0;
  return large.bytes > small.bytes ? large.bytes : small.bytes;
}

extern "C" int vrm_paged_chunk_attention(const void* query, int q_dtype, long long q_token_stride,
                                         long long q_head_stride, const void* kv_pool, const float* kv_scales,
                                         const int32_t* page_table, const int32_t* context_lens,
                                         const int32_t* cu_seqlens, void* out, float* lse, void* workspace,
                                         size_t workspace_bytes, int N, int B, int H, int KH, int D, int PS, int L,
                                         int P, int max_pp, int layer_idx, float scale, int causal, int window,
                                         int kv_dtype, vrm_stream_t stream) {
  return vrm_paged_chunk_attention_expecting(query, q_dtype, q_token_stride, q_head_stride, kv_pool, kv_scales,
                                             page_table, context_lens, cu_seqlens, out, lse, workspace,
                                             workspace_bytes, N, B, H, KH, D, PS, L, P, max_pp, layer_idx, scale,
                                             causal, window, 0, kv_dtype, stream);
}

extern "C" int vrm_paged_chunk_attention_expecting(
    const void* query, int q_dtype, long long q_token_stride, long long q_head_stride, const void* kv_pool,
    const float* kv_scales, const int32_t* page_table, const int32_t* context_lens, const int32_t* cu_seqlens,
    void* out, float* lse, void* workspace, size_t workspace_bytes, int N, int B, int H, int KH, int D, int PS, int L,
    int P, int max_pp, int layer_idx, float scale, int causal, int window, int expected_context, int kv_dtype,
    vrm_stream_t stream) {
  const char* who = "vrm_paged_chunk_attention";
  if (bad_sizes(N, B, H, KH, D, PS, max_pp) || L <= 0 || P <= 0 || window < 0 || expected_context < 0) {
    set_error("%s: bad sizes (N=%d B=%d H=%d KH=%d D=%d PS=%d L=%d P=%d max_pp=%d window=%d "
              "expected_context=%d; H a multiple of KH)",
              who, N, B, H, KH, D, PS, L, P, max_pp, window, expected_context);
    return VRM_ERR_ARG;
  }
  if (layer_idx < 0 || layer_idx >= L) {
    set_error("%s: layer_idx %d outside [0, %d)", who, layer_idx, L);
    return VRM_ERR_ARG;
  }
  const float sc = fabsf(scale) * 1.44269504088896341f;  // scores in base-2 logarithms
  if (!isfinite(sc)) {
    set_error("%s: scale is not finite, or its product with log2 e is not", who);
    return VRM_ERR_ARG;
  }
  if (q_dtype != VRM_SRC_F32 && q_dtype != VRM_SRC_F16 && q_dtype != VRM_SRC_BF16) {
    set_error("%s: unknown query dtype %d", who, q_dtype);
    return VRM_ERR_ARG;
  }
  const int kind = pool_kind(kv_dtype);
  if (kind < 0) {
    set_error("%s: unknown kv_dtype %d", who, kv_dtype);
    return VRM_ERR_ARG;
  }
  const long long row = kind == kSrcF32 ? 4LL * D : kind < kSrcI8 ? 2LL * D : D;  // bytes of a token
  if (D > 256) {
    set_error("%s: head_dim %d above 256", who, D);
    return VRM_ERR_UNSUPPORTED;
  }
  if (kind >= kSrcI8 && (D % 16 || PS % 4)) {
    set_error("%s: head_dim %d / page_size %d unsupported over a quantized pool (multiples of 16 / 4)", who, D, PS);
    return VRM_ERR_UNSUPPORTED;
  }
  ChunkPlan p;
  if (!plan_chunk(N, B, H, KH, D, PS, max_pp, q_dtype, kv_dtype, expected_context, window, p)) {
    set_error("%s: too many rows (N=%d H=%d B=%d)", who, N, H, B);
    return VRM_ERR_UNSUPPORTED;
  }
  if (N == 0 || B == 0) {
    clear_error();
    return VRM_OK;
  }
  if (!query || !kv_pool || !context_lens || !cu_seqlens || !out || (max_pp > 0 && !page_table)) {
    set_error("%s: null pointer argument", who);
    return VRM_ERR_ARG;
  }
  if ((kind >= kSrcI8) != (kv_scales != nullptr)) {
    set_error("%s: kv_scales is for int8 and fp8 pools, and they need it", who);
    return VRM_ERR_ARG;
  }
  if (kind >= kSrcI8) {
    const int rc = check_pool_scales(kv_dtype, kv_pool, kv_scales, KH, PS, D, L, P, who);
    if (rc) return rc;
  }
  const uintptr_t q_at = reinterpret_cast<uintptr_t>(query);
  if (p.bytes && (!workspace || workspace_bytes < p.bytes || reinterpret_cast<uintptr_t>(workspace) % 16)) {
    set_error("%s: workspace of %zu bytes, 16-byte aligned, needed (got %zu)", who, p.bytes, workspace_bytes);
    return VRM_ERR_WORKSPACE;
  }

  ChunkArgs a{};
  a.q = query;
  a.q_n = q_token_stride;
  a.q_h = q_head_stride;
  a.q_type = q_dtype;
  a.pool = static_cast<const uint8_t*>(kv_pool);
  a.scales = kv_scales;
  a.g = pool_geom(kv_dtype, KH, PS, D, row, P, L);
  a.layer_off = (long long)layer_idx * a.g.layer;
  a.s_layer_off = (long long)layer_idx * a.g.s_layer;
  a.table = page_table;
  a.lens = context_lens;
  a.cu = cu_seqlens;
  a.out = out;
  a.lse = lse;
  a.N = N, a.B = B, a.H = H, a.KH = KH, a.G = H / KH, a.D = D, a.PS = PS, a.P = P, a.max_pp = max_pp;
  a.ps_shift = (PS & (PS - 1)) ? -1 : __builtin_ctz(PS);
  a.causal = causal != 0;
  a.window = window < 1 << 30 ? window : 1 << 30;  // (positions less it stay in 32 bits)
  a.sc = scale == 0.f ? 1.f : sc;
  a.q_sign = scale == 0.f ? 0 : scale < 0.f ? -1 : 1;
  a.target = p.target;
  a.min_blocks = p.min_blocks;
  a.vtiles = p.vtiles;
  a.items = p.items;
  a.aligned = row % 16 == 0 && reinterpret_cast<uintptr_t>(kv_pool) % 16 == 0;
  a.q_aligned = q_at % 16 == 0 && q_token_stride % 8 == 0 && q_head_stride % 8 == 0;
  a.out_aligned = D % 4 == 0 && reinterpret_cast<uintptr_t>(out) % 8 == 0;
  a.dp = p.dp;
  a.tile_rows = p.tile_rows;
  a.tile_shift = p.tile_rows == 256 ? 8 : 7;
  char* ws = static_cast<char*>(workspace);
  if (p.target) {
    a.rec = reinterpret_cast<int2*>(ws);
    a.ml = reinterpret_cast<float2*>(ws + p.rec_bytes);
    a.part = reinterpret_cast<float*>(ws + p.rec_bytes + p.ml_bytes);
  }
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)p.items * (unsigned)KH);
  if (p.wide)
    launch_chunk_f32(a, kind, grid, st);
  else if (p.dp == 256)
    launch_chunk16_256(a, kind, grid, st);
  else if (kind == kSrcI8)
    launch_chunk16_i8(a, grid, st);
  else if (kind == kSrcFp8)
    launch_chunk16_fp8(a, grid, st);
  else
    launch_chunk16_float(a, grid, st);
  const int rc = launch_status(who);
  if (rc || !p.target) return rc;
  const dim3 merge((unsigned)p.vtiles * (unsigned)KH, a.tile_rows / kMergeRows);
  if (a.dp == 64)
    hipLaunchKernelGGL((chunk_merge_kernel<64>), merge, dim3(256), 0, st, a);
  else if (a.dp == 96)
    hipLaunchKernelGGL((chunk_merge_kernel<96>), merge, dim3(256), 0, st, a);
  else if (a.dp == 128)
    hipLaunchKernelGGL((chunk_merge_kernel<128>), merge, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((chunk_merge_kernel<256>), merge, dim3(256), 0, st, a);
  return launch_status(who);
}
