// Attention of a ragged batch's new tokens over a paged cache: the call's
// arguments, its work items, and what both kernels (16-bit matrix products,
// float32 products) share.
//
// Rows.  The G = H / KH query heads of a kv-head read the same keys, so a
// sequence's q_b new tokens make q_b G rows of one matrix per kv-head: row r
// is head r % G of token r / G.  A tile is tile_rows of them.
// Items.  A workgroup takes one item: a tile of one kv-head over a share of
// the key blocks that its rows see.  A batch of few tiles is cut along the
// keys (find_item) so that the GPU is full; the shares' (max, sum,
// accumulator) go to the workspace and chunk_merge_kernel joins them.
#pragma once
#include <math.h>

#include "vrm_common.h"

namespace vrm {

constexpr int kChunkThreads = 256;  // four wavefronts: tiles of 128 rows
constexpr int kLargeThreads = 512;  // eight: tiles of 256

enum { kSrcF32 = 0, kSrcF16 = 1, kSrcBf16 = 2, kSrcI8 = 3, kSrcFp8 = 4 };  // element types of a pool

struct ChunkArgs {
  const void* q;
  long long q_n, q_h;  // elements from a token's row to the next token's, and from a head's to the next
  int q_type;          // VRM_SRC_*
  const uint8_t* pool;
  const float* scales;
  PoolGeom g;
  long long layer_off, s_layer_off;  // of the layer, in bytes and scale floats
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu;
  void* out;  // [N][H][D] of q_type
  float* lse;
  float* part;  // [items][tile_rows][dp]: accumulators of shares
  float2* ml;   // [items][tile_rows]: their max (log2 units) and sum
  int2* rec;    // [vtiles][KH]: first item and shares of a tile
  int N, B, H, KH, G, D, PS, P, max_pp;
  int dp;       // D as the kernel pads it
  int tile_rows, tile_shift;  // 128 or 256, and its logarithm
  int vtiles;   // tiles when every sequence has one more than its rows fill
  int items;    // items per kv-head that the grid (and the workspace) has room for
  int ps_shift;      // log2 PS, or -1
  int causal;
  int window;        // tokens a row sees up to its own; 0: all
  float sc;          // |scale| log2 e (1 for scale 0)
  int q_sign;        // -1: the queries enter negated; 0: as zeros
  int target;        // items wanted per kv-head; 0: one per tile
  int min_blocks;    // key blocks an item has at least
  int aligned;       // pool rows can be loaded 16 bytes at a time
  int q_aligned;     // query rows too
  int out_aligned;   // output rows can be stored 8 bytes at a time
};

struct Sequence {
  int row0, q_len;
  int ctx;   // tokens that the page table has room for
  int base;  // position of its first new token
};

__device__ __forceinline__ Sequence load_sequence(const ChunkArgs& a, int b) {
  Sequence s;
  s.row0 = clamp_int(a.cu[b], 0, a.N);
  s.q_len = max(clamp_int(a.cu[b + 1], 0, a.N) - s.row0, 0);
  const int len = max(a.lens[b], 0);
  s.ctx = (int)min((long long)len, (long long)a.max_pp * a.PS);
  s.base = len - s.q_len;
  return s;
}

// Tiles before those of sequence b when every sequence is given one more than
// its rows fill: known from cu[b] alone, and at least as many as it needs.
__device__ __forceinline__ int virtual_tile(const ChunkArgs& a, int row0, int b) {
  return (int)(((long long)row0 * a.G) >> a.tile_shift) + b;
}

__device__ __forceinline__ int tiles_of(const ChunkArgs& a, const Sequence& s) {
  return (s.q_len * a.G + a.tile_rows - 1) >> a.tile_shift;
}

// Key blocks of TN tokens that a tile of the sequence sees at most.
template <int TN>
__device__ __forceinline__ int blocks_of(const ChunkArgs& a, const Sequence& s) {
  int span = s.ctx;
  if (a.window) span = (int)min((long long)span, (long long)a.window + a.tile_rows / a.G + 1 + TN);
  return (span + TN - 1) / TN;
}

// What a block costs a tile of at most 32 rows, whose wavefronts wait for
// memory, against one of a larger tile.  A compromise: shares round up to whole
// items, more of them than are resident at once, and which cost leaves the last
// ones least to do differs from batch to batch.  At 1, 2 and 4, chunks beside
// single tokens: 509 beside 15, 28 heads over 4, 54, 48 and 62 us; 2000 beside
// 31 374, 354 and 311; four of 256 beside 12, 32 over 8, 97, 98 and 115; 512
// beside 15 at head_dim 256 278, 245 and 246; 512 beside 63 over int8, 40 over
// 8, 209, 206 and 215, but beside 31 103, 139 and 139; two of 300 beside 30 at
// head_dim 64 56, 71 and 74.
constexpr int kFewCost = 2;
__device__ __forceinline__ int block_cost(const ChunkArgs& a, const Sequence& s) {
  return s.q_len * a.G <= 32 ? kFewCost : 1;
}

// Inclusive prefix sum over the wavefront's lanes.
__device__ __forceinline__ int wave_scan(int v) {
  const int lane = __lane_id();
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int u = __shfl_up(v, d);
    if (lane >= d) v += u;
  }
  return v;
}

struct Item {
  int b, tile, share, shares;
  int first;  // item index of the tile's share 0 (per kv-head)
  Sequence s;
};

// What a wavefront's 32 rows from row0 of the tile are: lane's row (its column
// of the score tiles), its token and head, and the positions of the first and
// last row.
struct RowGroup {
  int row, tok, head, pos, first_pos, last_pos;
  bool real;
};
__device__ __forceinline__ RowGroup row_group(const ChunkArgs& a, const Item& it, int kvh, int rows, int row0) {
  RowGroup g;
  g.row = row0 + (__lane_id() & 31);
  const int packed = it.tile * a.tile_rows + g.row;
  g.tok = packed / a.G;
  g.head = kvh * a.G + packed - g.tok * a.G;
  g.real = g.row < rows;
  const int base = it.s.base;
  g.pos = base + g.tok;
  g.first_pos = base + (it.tile * a.tile_rows + row0) / a.G;
  g.last_pos = base + (it.tile * a.tile_rows + min(rows, row0 + 32) - 1) / a.G;
  return g;
}

// Item idx of a kv-head: the shares of the first sequence's tiles (later tiles
// first: under a causal mask they see more keys), then the next sequence's.
// Shares have about (work of the kv-head) / target, so that sequences of any
// lengths fill the GPU evenly, and two blocks at least; every wavefront finds
// its item itself, lane by lane over the sequences.
template <int TN>
__device__ __forceinline__ bool find_item(const ChunkArgs& a, int idx, Item& it) {
  const int lane = __lane_id();
  int share_work = 0x7fffffff;
  if (a.target > 0) {
    float work = 0.f;
    bool many = false;
    for (int b0 = 0; b0 < a.B; b0 += kWave) {
      const int b = b0 + lane;
      if (b < a.B) {
        const Sequence s = load_sequence(a, b);
        work += (float)tiles_of(a, s) * (float)block_cost(a, s) * (float)blocks_of<TN>(a, s);
        many |= block_cost(a, s) == 1 && tiles_of(a, s) > 0;
      }
    }
    work = group_sum<64>(work);
    const int unit = __any(many) ? 1 : kFewCost;
    share_work = unit * (int)fminf(fmaxf(ceilf(work / (float)(a.target * unit)), 1.f), 1e8f);
  }
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += kWave) {
    const int b = b0 + lane;
    Sequence s{0, 0, 0, 0};
    int tiles = 0, shares = 1;
    if (b < a.B) {
      s = load_sequence(a, b);
      tiles = tiles_of(a, s);
      const int blocks = blocks_of<TN>(a, s);
      const long long work = (long long)blocks * block_cost(a, s);
      shares = max(1, min((int)((work + share_work - 1) / share_work), (blocks + a.min_blocks - 1) / a.min_blocks));
    }
    const int upto = wave_scan(tiles * shares);
    const unsigned long long past = __ballot(before + upto > idx);
    if (past) {
      const int l = __ffsll(past) - 1;
      it.b = b0 + l;
      it.s.row0 = __builtin_amdgcn_readlane(s.row0, l);
      it.s.q_len = __builtin_amdgcn_readlane(s.q_len, l);
      it.s.ctx = __builtin_amdgcn_readlane(s.ctx, l);
      it.s.base = __builtin_amdgcn_readlane(s.base, l);
      it.shares = __builtin_amdgcn_readlane(shares, l);
      const int nt = __builtin_amdgcn_readlane(tiles, l);
      const int from = before + __builtin_amdgcn_readlane(upto, l) - nt * it.shares;
      const int rem = idx - from;
      it.tile = nt - 1 - rem / it.shares;
      it.share = rem % it.shares;
      it.first = idx - it.share;
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, kWave - 1);
  }
  return false;
}

// Key blocks [from, to) of an item: its share of those that the tile's rows see.
template <int TN>
__device__ __forceinline__ void item_blocks(const ChunkArgs& a, const Item& it, int& from, int& to) {
  const int rows = it.s.q_len * a.G;
  const int t0 = it.tile * a.tile_rows / a.G;                             // the tile's first token
  const int t1 = (min(rows, (it.tile + 1) * a.tile_rows) - 1) / a.G;      // and its last
  const int base = it.s.base;
  const int hi = a.causal ? clamp_int(base + t1 + 1, 0, it.s.ctx) : it.s.ctx;
  const int lo = a.window ? clamp_int(base + t0 - a.window + 1, 0, hi) : 0;
  const int b0 = lo / TN, n = (hi + TN - 1) / TN - b0;
  const int per = (n + it.shares - 1) / it.shares;
  from = b0 + min(n, it.share * per);
  to = b0 + min(n, (it.share + 1) * per);
}

// Share 0 leaves the merge the tile's first item and number of shares.
__device__ __forceinline__ void put_record(const ChunkArgs& a, const Item& it, int kvh) {
  const int vtile = virtual_tile(a, it.s.row0, it.b) + it.tile;
  if (a.target > 0 && it.share == 0 && threadIdx.x == 0 && vtile < a.vtiles)
    a.rec[(long long)vtile * a.KH + kvh] = make_int2(it.first, it.shares);
}

__device__ __forceinline__ int page_index(const ChunkArgs& a, int token) {
  return a.ps_shift >= 0 ? token >> a.ps_shift : token / a.PS;
}

__device__ __forceinline__ float load_q(const ChunkArgs& a, long long at) {
  if (a.q_type == VRM_SRC_F32) return static_cast<const float*>(a.q)[at];
  const uint32_t h = static_cast<const uint16_t*>(a.q)[at];
  return a.q_type == VRM_SRC_F16 ? f16_bits_to_f32(h) : bf16_bits_to_f32(h);
}

// 16 bytes of which the first `bytes` are there; the rest are zero.
__device__ __forceinline__ uint4 load16(const uint8_t* p, int bytes, bool vec) {
  if (vec && bytes >= 16) return *reinterpret_cast<const uint4*>(p);
  unsigned long long lo = 0, hi = 0;
#pragma unroll 1
  for (int i = min(bytes, 16) - 1; i >= 0; --i) {
    hi = hi << 8 | lo >> 56;
    lo = lo << 8 | p[i];
  }
  return make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
}

__device__ __forceinline__ float load_value(int kind, const uint8_t* p, int i) {
  switch (kind) {
    case kSrcF32: return reinterpret_cast<const float*>(p)[i];
    case kSrcF16: return f16_bits_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
    case kSrcBf16: return bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
    case kSrcI8: return (float)(int8_t)p[i];
    default: return e4m3fn_to_f32(p[i]);
  }
}

// Element of a page's V (of a kv-head) that is a slot's dim d.
__device__ __forceinline__ int value_at(const ChunkArgs& a, int kind, int slot, int d) {
  if (kind < kSrcI8) return slot * a.D + d;
  return (((slot >> 2) * 16 + (d & 15)) * (a.D >> 4) + (d >> 4)) * 4 + (slot & 3);
}

// Whether a row of the wavefront has a NaN in its accumulators (or infinities
// of both signs).
template <typename V, int NB>
__device__ __forceinline__ bool any_nan(const V (&o)[NB], bool real) {
  V x = o[0];
#pragma unroll
  for (int n = 1; n < NB; ++n) x += o[n];
  float y = x[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) y += x[i];
  return __any(real && y != y);
}

__device__ __forceinline__ bool not_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }

// Rows [row0, row1) of an item, of which some have a NaN in their accumulators
// (called by one wavefront, with the positions of the first and last row).
// In a matrix product the weight 0 of a token that a row does not see makes a
// NaN of an infinity or a NaN among its values, so if there is one within the
// item (a model that has overflowed), the rows are computed again, token by
// token over those that each sees.  Returns whether it did.
template <int TN>
__device__ __forceinline__ bool careful_rows(const ChunkArgs& a, const Item& it, int kvh, int kind, int row0, int row1,
                                             int first_pos, int last_pos, int from, int to) {
  const int lane = threadIdx.x & 63;
  const int32_t* const table = a.table + (long long)it.b * a.max_pp;
  const uint8_t* const k_base = a.pool + a.layer_off + (long long)kvh * a.g.head;
  const int end = min(to * TN, it.s.ctx);
  bool spoilt = false;
#pragma unroll 1
  for (int t = from * TN; t < end; ++t) {
    const bool unseen = (a.causal && t > first_pos) || (a.window && t <= last_pos - a.window);
    if (!unseen) {  // on to the tokens after the first row's position
      if (!a.causal) break;
      t = max(t, min(first_pos, end));
      continue;
    }
    const int pi = page_index(a, t), page = table[pi];
    if (page < 0 || page >= a.P) continue;
    const int slot = t - pi * a.PS;
    const uint8_t* const v = k_base + a.g.kv + (long long)page * a.g.page;
    for (int d = lane; d < a.D; d += kWave) spoilt |= not_finite(load_value(kind, v, value_at(a, kind, slot, d)));
    if (kind >= kSrcI8) {
      const float vs = a.scales[a.s_layer_off + (long long)page * a.g.s_page + (long long)kvh * a.g.s_head +
                                (kind == kSrcI8 ? slot : 0) + a.g.s_kv];
      spoilt |= not_finite(vs);
    }
  }
  if (!__any(spoilt)) return false;
#pragma unroll 1
  for (int row = row0; row < row1; ++row) {
    const int packed = it.tile * a.tile_rows + row, tok = packed / a.G, head = kvh * a.G + packed % a.G;
    const int pos = it.s.base + tok;
    const int t0 = max(from * TN, a.window ? pos - a.window + 1 : 0);
    const int t1 = min(min(to * TN, it.s.ctx), a.causal ? pos + 1 : it.s.ctx);
    float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
    const long long q_at = (long long)(it.s.row0 + tok) * a.q_n + (long long)head * a.q_h;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = lane + 64 * e;
      q[e] = d < a.D && a.q_sign ? load_q(a, q_at + d) * (float)a.q_sign : 0.f;
    }
#pragma unroll 1
    for (int t = t0; t < t1; ++t) {
      const int pi = page_index(a, t), page = table[pi];
      if (page < 0 || page >= a.P) continue;
      const int slot = t - pi * a.PS;
      const uint8_t* const k = k_base + (long long)page * a.g.page;
      const uint8_t* const v = k + a.g.kv;
      float ks = 1.f, vs = 1.f;
      if (kind >= kSrcI8) {
        const float* s = a.scales + a.s_layer_off + (long long)page * a.g.s_page + (long long)kvh * a.g.s_head +
                         (kind == kSrcI8 ? slot : 0);
        ks = s[0], vs = s[a.g.s_kv];
      }
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (lane + 64 * e < a.D) dot += q[e] * load_value(kind, k, slot * a.D + lane + 64 * e);
      const float s = group_sum<64>(dot) * ks * a.sc;
      const float next = fmaxf(m, s);
      const float f = m == -INFINITY ? 0.f : exp2f(m - next), p = s == -INFINITY ? 0.f : exp2f(s - next);
      m = next;
      l = l * f + p;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = lane + 64 * e;
        if (d < a.D) o[e] = o[e] * f + p * (load_value(kind, v, value_at(a, kind, slot, d)) * vs);
      }
    }
    const long long at = (long long)(it.s.row0 + tok) * a.H + head;
    const long long share = (long long)blockIdx.x * a.tile_rows + row;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = lane + 64 * e;
      if (d >= a.D) break;
      const float x = l == 0.f ? 0.f : o[e] / l;
      if (it.shares > 1)
        a.part[share * a.dp + d] = o[e];
      else if (a.q_type == VRM_SRC_F32)
        static_cast<float*>(a.out)[at * a.D + d] = x;
      else if (a.q_type == VRM_SRC_F16)
        static_cast<uint16_t*>(a.out)[at * a.D + d] = __builtin_bit_cast(unsigned short, (_Float16)x);
      else
        static_cast<uint16_t*>(a.out)[at * a.D + d] = __builtin_bit_cast(unsigned short, (__bf16)x);
    }
    if (lane == 0) {
      if (it.shares > 1)
        a.ml[share] = make_float2(m, l);
      else if (a.lse)
        a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
    }
  }
  return true;
}

// One launch of the attention kernel: float32 products (pool of kind kSrc*),
// 16-bit products over float, int8 and fp8 pools.
void launch_chunk_f32(const ChunkArgs& a, int kind, dim3 grid, hipStream_t st);
void launch_chunk16_float(const ChunkArgs& a, dim3 grid, hipStream_t st);
void launch_chunk16_i8(const ChunkArgs& a, dim3 grid, hipStream_t st);
void launch_chunk16_fp8(const ChunkArgs& a, dim3 grid, hipStream_t st);
void launch_chunk16_256(const ChunkArgs& a, int kind, dim3 grid, hipStream_t st);  // head dims above 128

}  // namespace vrm
