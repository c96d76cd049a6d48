// Device side of the paged cache manager: block-table build and raw slot
// writes.
//
// PagedKVCacheManager.compute_attention_decode (core/paged_attention.py:
// 1226-1248) fills a -1-padded [B, max_pp] int32 page table element by element
// from each request's page list, then the context lengths.  Here the host
// hands over the lists concatenated (flat_pages, offsets) and one kernel
// scatters them, so a batch costs one copy of sum(pages) ints instead of
// B * max_pp host writes and a B * max_pp upload.
//
// write_kv's raw index-put into a float pool (:611-612,
// pool[page, layer, 0|1, :, slot, :] = key|value) is vrm_kv_write: one
// wavefront per (token, K/V, kv-head) row converts the row to the pool's
// element type, rounding to nearest even as PyTorch's copy does.
//
// vrm_chunk_tables makes what a chunk of new tokens needs from lengths that are
// on the device already (tokens stored and new tokens of each request, a block
// table that stays there), so that a step whose lengths follow from the one
// before it, as accepted drafts do, starts without a copy to the host.
#include "vrm_common.h"

namespace vrm {
namespace {

constexpr int kTableThreads = 256;

__global__ void __launch_bounds__(kTableThreads)
    build_table_kernel(const int32_t* flat_pages, int n_flat, const int32_t* offsets, const int32_t* num_tokens,
                       int max_pp, int32_t* page_table, int32_t* context_lens) {
  const int b = blockIdx.y;
  const int p = blockIdx.x * kTableThreads + threadIdx.x;
  const int beg = offsets[b];
  const int end = offsets[b + 1];
  // A malformed list (offsets outside the flat array or decreasing) yields
  // absent pages rather than reads outside flat_pages.
  const bool ok = beg >= 0 && end >= beg && end <= n_flat;
  const int n = ok ? end - beg : 0;
  if (p < max_pp) page_table[(size_t)b * max_pp + p] = p < n ? flat_pages[beg + p] : -1;
  if (p == 0) context_lens[b] = num_tokens[b];
}

struct ChunkTableArgs {
  const int32_t* block_table;  // [R] rows of W, row_stride apart
  long long row_stride;
  int R, W;
  const int32_t* past;      // [R]
  const int32_t* counts;    // [B]
  const int32_t* requests;  // [B] or NULL
  int B, N, PS;
  int32_t* page_table;  // [B][max_pp]
  int max_pp;
  int32_t* context_lens;  // [B]
  int32_t* cu;            // [B + 1]
  int32_t* positions;     // [N]
  int32_t* page_ids;
  int32_t* slots;
  int32_t* sequences;

  // The request of sequence b, -1 where there is none of that number.
  __device__ __forceinline__ int request(int b) const {
    const int r = requests ? requests[b] : b;
    return r >= 0 && r < R ? r : -1;
  }
  __device__ __forceinline__ int stored(int r) const { return r >= 0 ? max(past[r], 0) : 0; }
  // New tokens that sequence b asks for; its positions stay below 2^31.
  __device__ __forceinline__ int asked(int b, int r) const {
    return r >= 0 ? min(max(counts[b], 0), 0x7fffffff - max(past[r], 0)) : 0;
  }
};

constexpr int kScanThreads = 1024;

// Offsets of the new tokens, cut at N, and the lengths that follow from them.
__global__ void __launch_bounds__(kScanThreads) chunk_offsets_kernel(ChunkTableArgs a) {
  __shared__ long long waves[kScanThreads / 64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  long long before = 0;
  if (threadIdx.x == 0) a.cu[0] = 0;
  for (int b0 = 0; b0 < a.B; b0 += kScanThreads) {
    const int b = b0 + threadIdx.x;
    const int r = b < a.B ? a.request(b) : -1;
    const long long n = b < a.B ? a.asked(b, r) : 0;
    long long run = n;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const long long o = __shfl_up(run, m);
      if (lane >= m) run += o;
    }
    __syncthreads();
    if (lane == 63) waves[wave] = run;
    __syncthreads();
    long long all = 0;
    for (int v = 0; v < kScanThreads / 64; ++v) {
      if (v == wave) run += before + all;
      all += waves[v];
    }
    before += all;
    if (b < a.B) {
      const long long end = min(run, (long long)a.N), beg = min(run - n, (long long)a.N);
      a.cu[b + 1] = (int)end;
      a.context_lens[b] = a.stored(r) + (int)(end - beg);
    }
  }
}

// Blocks 0 .. table_blocks: 1024 entries of a sequence's row of the page table
// each; the others 256 new tokens each.
__global__ void __launch_bounds__(kTableThreads) chunk_places_kernel(ChunkTableArgs a, int per_row, int table_blocks) {
  if ((int)blockIdx.x < table_blocks) {
    const int b = blockIdx.x / per_row, p0 = (blockIdx.x % per_row) * 4 * kTableThreads;
    const int r = a.request(b);
    const int held = (int)min(((long long)a.context_lens[b] + a.PS - 1) / a.PS, (long long)a.W);
    const int32_t* from = a.block_table + (r >= 0 ? r : 0) * a.row_stride;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = p0 + i * kTableThreads + threadIdx.x;
      if (p < a.max_pp) a.page_table[(size_t)b * a.max_pp + p] = r >= 0 && p < held ? from[p] : -1;
    }
    return;
  }
  const int n = ((int)blockIdx.x - table_blocks) * kTableThreads + threadIdx.x;
  if (n >= a.N) return;
  int pos = 0, page = -1, slot = -1, seq = -1;
  if (n < a.cu[a.B]) {
    int lo = 0, hi = a.B - 1;  // the last sequence that starts at or before n and is not empty
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (a.cu[mid + 1] > n) hi = mid;
      else lo = mid + 1;
    }
    seq = lo;
    const int r = a.request(seq);
    pos = a.stored(r) + n - a.cu[seq];
    slot = pos % a.PS;
    const int p = pos / a.PS;
    if (r >= 0 && p < a.W) page = a.block_table[r * a.row_stride + p];
  }
  a.positions[n] = pos;
  a.page_ids[n] = page;
  a.slots[n] = slot;
  a.sequences[n] = seq;
}

template <int SRC>
__device__ __forceinline__ float load_elem(const void* p, size_t i) {
  if constexpr (SRC == VRM_SRC_F32) {
    return static_cast<const float*>(p)[i];
  } else if constexpr (SRC == VRM_SRC_F16) {
    return f16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
  } else {
    return bf16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
  }
}

// float32 -> bfloat16 bits, round to nearest even; NaN stays a quiet NaN.
__device__ __forceinline__ uint16_t f32_to_bf16_bits(float x) {
  const uint32_t u = __float_as_uint(x);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
  return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

template <int DST>
__device__ __forceinline__ void store_elem(void* p, size_t i, float x) {
  if constexpr (DST == VRM_KV_F32) {
    static_cast<float*>(p)[i] = x;
  } else if constexpr (DST == VRM_KV_F16) {
    static_cast<uint16_t*>(p)[i] = __builtin_bit_cast(unsigned short, (_Float16)x);
  } else {
    static_cast<uint16_t*>(p)[i] = f32_to_bf16_bits(x);
  }
}

struct KvWriteArgs {
  const void* key;
  const void* value;
  const int32_t* page_ids;
  const int32_t* slots;
  void* pool;
  int KH, D, PS, L, P, layer;
};

// Row x = (n * 2 + kv) * KH + h; source rows are [N][KH][D].
template <int SRC, int DST>
__global__ void __launch_bounds__(64) kv_write_kernel(KvWriteArgs a) {
  const int x = blockIdx.x;
  const int h = x % a.KH;
  const int kv = (x / a.KH) & 1;
  const int n = x / (2 * a.KH);
  const int pid = a.page_ids[n];
  const int slot = a.slots[n];
  if (pid < 0 || pid >= a.P || slot < 0 || slot >= a.PS) return;  // rows aimed outside the pool are dropped
  const size_t src = ((size_t)n * a.KH + h) * a.D;
  const size_t dst = (((((size_t)pid * a.L + a.layer) * 2 + kv) * a.KH + h) * a.PS + slot) * a.D;
  const void* from = kv ? a.value : a.key;
  for (int d = threadIdx.x; d < a.D; d += 64) store_elem<DST>(a.pool, dst + d, load_elem<SRC>(from, src + d));
}

template <int SRC>
void launch_kv_write(const KvWriteArgs& a, int rows, int kv_dtype, hipStream_t st) {
  switch (kv_dtype) {
    case VRM_KV_F32: hipLaunchKernelGGL((kv_write_kernel<SRC, VRM_KV_F32>), dim3(rows), dim3(64), 0, st, a); break;
    case VRM_KV_F16: hipLaunchKernelGGL((kv_write_kernel<SRC, VRM_KV_F16>), dim3(rows), dim3(64), 0, st, a); break;
    default: hipLaunchKernelGGL((kv_write_kernel<SRC, VRM_KV_BF16>), dim3(rows), dim3(64), 0, st, a); break;
  }
}

}  // namespace
}  // namespace vrm

using namespace vrm;

extern "C" int vrm_build_block_table(const int32_t* flat_pages, int n_flat, const int32_t* offsets,
                                     const int32_t* num_tokens, int B, int max_pp, int32_t* page_table,
                                     int32_t* context_lens, vrm_stream_t stream) {
  const char* who = "vrm_build_block_table";
  if (B < 0 || max_pp < 0 || n_flat < 0) {
    set_error("%s: bad sizes (B=%d max_pp=%d n_flat=%d)", who, B, max_pp, n_flat);
    return VRM_ERR_ARG;
  }
  if (B > 65535) {
    set_error("%s: batch %d above 65535", who, B);
    return VRM_ERR_UNSUPPORTED;
  }
  if (B == 0) {
    clear_error();
    return VRM_OK;
  }
  if (!offsets || !num_tokens || !page_table || !context_lens || (n_flat > 0 && !flat_pages)) {
    set_error("%s: null pointer argument", who);
    return VRM_ERR_ARG;
  }
  const int bx = max_pp > 0 ? (max_pp + kTableThreads - 1) / kTableThreads : 1;
  hipLaunchKernelGGL(build_table_kernel, dim3(bx, B), dim3(kTableThreads), 0, reinterpret_cast<hipStream_t>(stream),
                     flat_pages, n_flat, offsets, num_tokens, max_pp, page_table, context_lens);
  return launch_status(who);
}

extern "C" int vrm_chunk_tables(const int32_t* block_table, long long row_stride, int R, int W, const int32_t* past_lens,
                                const int32_t* counts, const int32_t* requests, int B, int N, int PS,
                                int32_t* page_table, int max_pp, int32_t* context_lens, int32_t* cu_seqlens,
                                int32_t* positions, int32_t* page_ids, int32_t* slots, int32_t* sequences,
                                vrm_stream_t stream) {
  const char* who = "vrm_chunk_tables";
  if (R < 0 || W < 0 || B < 0 || N < 0 || PS <= 0 || max_pp < 0 || row_stride < 0) {
    set_error("%s: bad sizes (R=%d W=%d B=%d N=%d PS=%d max_pp=%d row stride %lld)", who, R, W, B, N, PS, max_pp,
              row_stride);
    return VRM_ERR_ARG;
  }
  if (!requests && B > R) {
    set_error("%s: %d sequences without requests for %d rows of the block table", who, B, R);
    return VRM_ERR_ARG;
  }
  if (!cu_seqlens || (B > 0 && (!counts || !context_lens || (R > 0 && !past_lens))) ||
      (B > 0 && max_pp > 0 && !page_table) || (R > 0 && W > 0 && !block_table) ||
      (N > 0 && (!positions || !page_ids || !slots || !sequences))) {
    set_error("%s: null pointer argument", who);
    return VRM_ERR_ARG;
  }
  const long long per_row = (max_pp + 4LL * kTableThreads - 1) / (4 * kTableThreads);
  const long long table_blocks = per_row * B, blocks = table_blocks + (N + kTableThreads - 1LL) / kTableThreads;
  if (blocks > (1LL << 32) / kTableThreads - 1) {  // a launch counts its threads in 32 bits
    set_error("%s: %d rows of %d pages and %d tokens are too many for one call", who, B, max_pp, N);
    return VRM_ERR_UNSUPPORTED;
  }
  const ChunkTableArgs a{block_table, row_stride, R, W, past_lens, counts, requests, B, N, PS, page_table, max_pp,
                         context_lens, cu_seqlens, positions, page_ids, slots, sequences};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(chunk_offsets_kernel, dim3(1), dim3(kScanThreads), 0, st, a);
  if (blocks > 0)
    hipLaunchKernelGGL(chunk_places_kernel, dim3((unsigned)blocks), dim3(kTableThreads), 0, st, a, (int)per_row,
                       (int)table_blocks);
  return launch_status(who);
}

extern "C" int vrm_kv_write(const void* key, const void* value, int src_dtype, const int32_t* page_ids,
                            const int32_t* slots, int N, void* kv_pool, int kv_dtype, int KH, int D, int PS, int L,
                            int P, int layer_idx, vrm_stream_t stream) {
  const char* who = "vrm_kv_write";
  if (N < 0 || KH <= 0 || D <= 0 || PS <= 0 || L <= 0 || P <= 0) {
    set_error("%s: bad sizes (N=%d KH=%d D=%d PS=%d L=%d P=%d)", who, N, KH, D, PS, L, P);
    return VRM_ERR_ARG;
  }
  if (layer_idx < 0 || layer_idx >= L) {
    set_error("%s: layer_idx %d outside [0, %d)", who, layer_idx, L);
    return VRM_ERR_ARG;
  }
  if (src_dtype != VRM_SRC_F32 && src_dtype != VRM_SRC_F16 && src_dtype != VRM_SRC_BF16) {
    set_error("%s: unknown source dtype %d", who, src_dtype);
    return VRM_ERR_ARG;
  }
  if (kv_dtype != VRM_KV_F32 && kv_dtype != VRM_KV_F16 && kv_dtype != VRM_KV_BF16) {
    set_error("%s: kv_dtype %d is not a float pool (quantized pools are written by vrm_kv_quant_append)", who,
              kv_dtype);
    return VRM_ERR_ARG;
  }
  if ((long long)N * 2 * KH > 0x7fffffffLL) {
    set_error("%s: too many rows (N=%d KH=%d)", who, N, KH);
    return VRM_ERR_UNSUPPORTED;
  }
  if (N == 0) {
    clear_error();
    return VRM_OK;
  }
  if (!key || !value || !page_ids || !slots || !kv_pool) {
    set_error("%s: null pointer argument", who);
    return VRM_ERR_ARG;
  }
  KvWriteArgs a{key, value, page_ids, slots, kv_pool, KH, D, PS, L, P, layer_idx};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int rows = N * 2 * KH;
  switch (src_dtype) {
    case VRM_SRC_F32: launch_kv_write<VRM_SRC_F32>(a, rows, kv_dtype, st); break;
    case VRM_SRC_F16: launch_kv_write<VRM_SRC_F16>(a, rows, kv_dtype, st); break;
    default: launch_kv_write<VRM_SRC_BF16>(a, rows, kv_dtype, st); break;
  }
  return launch_status(who);
}
