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
#include <algorithm>

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

constexpr int kScanThreads = 512;
constexpr int kScanPer = 4;
constexpr int kScanMost = kScanThreads * kScanPer;  // sequences whose offsets every workgroup can have
constexpr int kEntries = 4 * kScanThreads;          // page table entries of a workgroup

// Running sum over the workgroup's values, inclusive; `all` the whole.
__device__ __forceinline__ long long block_prefix(long long v, long long* waves, long long& all) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const long long o = __shfl_up(v, m);
    if (lane >= m) v += o;
  }
  __syncthreads();
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  all = 0;
  for (int w = 0; w < kScanThreads / 64; ++w) {
    if (w < wave) v += waves[w];
    all += waves[w];
  }
  return v;
}

// Every `parts`-th kEntries of one sequence's row of the page table.  (wide:
// rows of both tables start on 16 bytes and have whole vectors.)
__device__ __forceinline__ void fill_row(const ChunkTableArgs& a, int b, int part, int parts, int context, bool wide) {
  const int r = a.request(b);
  const int held = r >= 0 ? (int)min(((long long)context + a.PS - 1) / a.PS, (long long)a.W) : 0;
  const int32_t* from = a.block_table + (r >= 0 ? r : 0) * a.row_stride;
  int32_t* to = a.page_table + (size_t)b * a.max_pp;
  for (long long p0 = (long long)part * kEntries; p0 < a.max_pp; p0 += (long long)parts * kEntries) {
    if (wide) {
      const int p = (int)p0 + 4 * threadIdx.x;
      if (p >= a.max_pp) return;
      int4 v = make_int4(-1, -1, -1, -1);
      if (p < held) {
        v = *reinterpret_cast<const int4*>(from + p);
        if (p + 1 >= held) v.y = -1;
        if (p + 2 >= held) v.z = -1;
        if (p + 3 >= held) v.w = -1;
      }
      *reinterpret_cast<int4*>(to + p) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long p = p0 + i * kScanThreads + threadIdx.x;
        if (p < a.max_pp) to[p] = p < held ? from[p] : -1;
      }
    }
  }
}

// The place of new token n.
__device__ __forceinline__ void place_token(const ChunkTableArgs& a, const int* cu, int n) {
  int pos = 0, page = -1, slot = -1, seq = -1;
  if (n < cu[a.B]) {
    int lo = 0, hi = a.B - 1;  // the sequence that ends first after n
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (cu[mid + 1] > n) hi = mid;
      else lo = mid + 1;
    }
    seq = lo;
    const int r = a.request(seq);
    pos = a.stored(r) + n - cu[seq];
    slot = pos % a.PS;
    const int p = pos / a.PS;
    if (r >= 0 && p < a.W) page = a.block_table[r * a.row_stride + p];
  }
  a.positions[n] = pos;
  a.page_ids[n] = page;
  a.slots[n] = slot;
  a.sequences[n] = seq;
}

// Everything in one launch: up to kScanMost sequences each workgroup sums the
// counts by itself (12 bytes a sequence, from L2 but for the first), which costs
// less than a launch of its own for it.  Blocks 0 .. table_blocks fill the page
// table, the others place 512 new tokens each; the last one writes the offsets.
__global__ void __launch_bounds__(kScanThreads)
    chunk_tables_kernel(ChunkTableArgs a, int per_row, int table_blocks, bool wide) {
  __shared__ int cu[kScanMost + 1];
  __shared__ long long waves[kScanThreads / 64];
  int n[kScanPer], past[kScanPer];
  long long sum = 0, all;
#pragma unroll
  for (int i = 0; i < kScanPer; ++i) {
    const int b = kScanPer * threadIdx.x + i;
    const int r = b < a.B ? a.request(b) : -1;
    past[i] = a.stored(r);
    n[i] = r >= 0 ? a.asked(b, r) : 0;
    sum += n[i];
  }
  long long run = block_prefix(sum, waves, all) - sum;
  if (threadIdx.x == 0) cu[0] = 0;
  const bool writes = blockIdx.x == gridDim.x - 1;
  if (writes && threadIdx.x == 0) a.cu[0] = 0;
#pragma unroll
  for (int i = 0; i < kScanPer; ++i) {
    const int b = kScanPer * threadIdx.x + i;
    const int beg = (int)min(run, (long long)a.N);
    run += n[i];
    const int end = (int)min(run, (long long)a.N);
    if (b < a.B) {
      cu[b + 1] = end;
      if (writes) {
        a.cu[b + 1] = end;
        a.context_lens[b] = past[i] + (end - beg);
      }
    }
  }
  __syncthreads();
  if ((int)blockIdx.x < table_blocks) {
    const int b = blockIdx.x / per_row;
    fill_row(a, b, blockIdx.x % per_row, per_row, a.stored(a.request(b)) + cu[b + 1] - cu[b], wide);
    return;
  }
  const int token = ((int)blockIdx.x - table_blocks) * kScanThreads + threadIdx.x;
  if (token < a.N) place_token(a, cu, token);
}

// More sequences: the offsets first, by one workgroup.
__global__ void __launch_bounds__(kScanThreads) chunk_offsets_kernel(ChunkTableArgs a) {
  __shared__ long long waves[kScanThreads / 64];
  long long before = 0, all;
  if (threadIdx.x == 0) a.cu[0] = 0;
  for (int b0 = 0; b0 < a.B; b0 += kScanThreads) {
    const int b = b0 + threadIdx.x;
    const int r = b < a.B ? a.request(b) : -1;
    const long long n = r >= 0 ? a.asked(b, r) : 0;
    const long long run = before + block_prefix(n, waves, all);
    before += all;
    if (b < a.B) {
      const long long end = min(run, (long long)a.N), beg = min(run - n, (long long)a.N);
      a.cu[b + 1] = (int)end;
      a.context_lens[b] = a.stored(r) + (int)(end - beg);
    }
  }
}

__global__ void __launch_bounds__(kScanThreads)
    chunk_places_kernel(ChunkTableArgs a, int per_row, int table_blocks, bool wide) {
  if ((int)blockIdx.x < table_blocks) {
    const int b = blockIdx.x / per_row;
    fill_row(a, b, blockIdx.x % per_row, per_row, a.context_lens[b], wide);
    return;
  }
  const int token = ((int)blockIdx.x - table_blocks) * kScanThreads + threadIdx.x;
  if (token < a.N) place_token(a, a.cu, token);
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
  // Workgroups of a row: one, or more where rows are few (a thousand in all fill
  // the chip, and each sums the counts first).
  const long long per_row =
      max_pp == 0 ? 0 : B >= 1024 ? 1 : std::min((max_pp + kEntries - 1LL) / kEntries, 1024LL / std::max(B, 1));
  const long long table_blocks = per_row * B;
  const long long blocks = table_blocks + (N + kScanThreads - 1LL) / kScanThreads;
  if (blocks > (1LL << 32) / kScanThreads - 2) {  // a launch counts its threads in 32 bits
    set_error("%s: %d rows of %d pages and %d tokens are too many for one call", who, B, max_pp, N);
    return VRM_ERR_UNSUPPORTED;
  }
  const size_t seqs = B, rows = N;
  if (int rc = check_apart({{page_table, seqs * max_pp * 4},
                            {context_lens, seqs * 4},
                            {cu_seqlens, (seqs + 1) * 4},
                            {positions, rows * 4},
                            {page_ids, rows * 4},
                            {slots, rows * 4},
                            {sequences, rows * 4}},
                           {{block_table, R > 0 && W > 0 ? (size_t)((R - 1) * row_stride + W) * 4 : 0},
                            {past_lens, (size_t)R * 4},
                            {counts, seqs * 4},
                            {requests, seqs * 4}},
                           who))
    return rc;
  const ChunkTableArgs a{block_table, row_stride, R, W, past_lens, counts, requests, B, N, PS, page_table, max_pp,
                         context_lens, cu_seqlens, positions, page_ids, slots, sequences};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const bool wide = !(((uintptr_t)block_table | (uintptr_t)page_table) & 15) && !(row_stride & 3) && !(max_pp & 3) &&
                    !(W & 3);
  if (B <= kScanMost) {
    hipLaunchKernelGGL(chunk_tables_kernel, dim3((unsigned)(blocks > 0 ? blocks : 1)), dim3(kScanThreads), 0, st, a,
                       (int)per_row, (int)table_blocks, wide);
  } else {
    hipLaunchKernelGGL(chunk_offsets_kernel, dim3(1), dim3(kScanThreads), 0, st, a);
    if (blocks > 0)
      hipLaunchKernelGGL(chunk_places_kernel, dim3((unsigned)blocks), dim3(kScanThreads), 0, st, a, (int)per_row,
                         (int)table_blocks, wide);
  }
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
