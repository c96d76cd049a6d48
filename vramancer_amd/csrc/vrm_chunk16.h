// chunk_attn_kernel: attention of a tile of rows over paged keys and values
// with 16-bit matrix products.
//
// One pass over the keys with a running maximum and sum (base-2 logarithms).
// A block of 64 tokens is gathered through the page table into registers
// while the block before it is computed, then laid into LDS.  The products
// are S^T = K Q^T and O^T += V^T P^T: with rows of the score matrix along the
// lanes of v_mfma_f32_32x32x16, lane l holds row l % 32's scores of 16 tokens,
// so the softmax needs one exchange (lanes l, l ^ 32) per block, and its
// weights are the next product's operand as they stand: the k-slots of
// 16 tokens are taken in the order the scores lie in (tokens 0-3, 8-11 in the
// lower lanes, 4-7, 12-15 in the upper), and V's operand follows, read
// transposed from row-major LDS (ds_read_b64_tr_b16), or from the transposed
// tile that the quantized pools store anyway.
//
// Precision.  Scores, maxima, sums and accumulators are float32.  Int8 and
// e4m3 codes are exact in bf16 and fp16, so K enters as codes and its scale
// multiplies the scores.  Weights are rounded to the 16-bit type once, because
// the second product takes 16-bit operands only: by at most half a step, 2^-8
// (bf16) or 2^-11 (fp16) of each, independent from token to token, where the
// output's own rounding is as large.  fp16 has a least step besides, 2^-24:
// fp16 weights are taken relative to a reference that keeps a row's largest
// between 2^7 and 2^15 (kMaxBias), so that it is at most 2^-31 of that one.
// Over quantized values weights are bf16 (fp16 would overflow under large
// scales), for fp16 queries as a high and a low part.
#pragma once
#include <type_traits>

#include "vrm_chunk.h"

namespace vrm {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

struct Bf16 {
  using v8 = bf16x8;
  using v2 = bf16x2;
  static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t from_fp8(uint32_t w, bool hi) {
    return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
  }
};
struct F16 {
  using v8 = f16x8;
  using v2 = f16x2;
  static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t from_fp8(uint32_t w, bool hi) {
    return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
  }
};

// Four codes of a dword as four 16-bit floats, exactly.
template <typename T, int KIND>
__device__ __forceinline__ uint2 codes4(uint32_t w) {
  if constexpr (KIND == kSrcFp8) {
    return make_uint2(T::from_fp8(w, false), T::from_fp8(w, true));
  } else {
    const f32x2 a = {(float)(int8_t)w, (float)(int8_t)(w >> 8)};
    const f32x2 b = {(float)(int8_t)(w >> 16), (float)(int8_t)(w >> 24)};
    return make_uint2(__builtin_bit_cast(uint32_t, __builtin_convertvector(a, typename T::v2)),
                      __builtin_bit_cast(uint32_t, __builtin_convertvector(b, typename T::v2)));
  }
}

// Bytes of a dword whose tokens (bits 0 .. 3) are there.
__device__ __forceinline__ uint32_t keep_bytes(uint32_t bits) {
  return ((bits & 1) * 0xffu) | ((bits >> 1 & 1) * 0xff00u) | ((bits >> 2 & 1) * 0xff0000u) |
         ((bits >> 3 & 1) * 0xff000000u);
}

constexpr int max3(int x, int y, int z) { return x > y ? (x > z ? x : z) : (y > z ? y : z); }

// Sizes of a block of 64 tokens in LDS.
template <int KIND, int DP>
struct ChunkTile {
  static constexpr bool kQuant = KIND >= kSrcI8;
  static constexpr int kTokens = 64;
  // K rows padded by 16 bytes: the 16-byte reads of 8 consecutive tokens fall
  // on different banks.  V rows (float pools) at 64 or 192 mod 256 bytes: so
  // do the transposed reads' four tokens of 64 bytes.
  static constexpr int kKStride = DP * 2 + 16;
  static constexpr int kVStride = DP * 2 + (DP * 2 % 128 == 0 ? 64 : 0);
  static constexpr int kKBytes = kTokens * kKStride;
  static constexpr int kVBytes = kQuant ? kTokens * DP * 2 : kTokens * kVStride;
  static constexpr int kBytes = kKBytes + kVBytes;
  static constexpr int kPerRow = kQuant ? DP / 16 : DP / 8;  // 16-byte pieces of a K row
  // 32 rows' accumulators, maxima and sums of a wavefront, for the merge of
  // wavefronts that shared rows (two at a time)
  static constexpr int kPartial = (DP / 32 * 16 + 2) * 64 * 4;
  // a wavefront's own 32 tokens of V (few_rows, float pools)
  static constexpr int kOwnV = kQuant ? 0 : 32 * kVStride;
};

// Rows of a group as the operand of the first product: lane (col, half) holds
// dims dim(kk) .. + 7 of its row for step kk.
template <typename T, int KK, typename Dim>
__device__ __forceinline__ void load_rows(const ChunkArgs& a, const Item& it, const RowGroup& g, Dim dim,
                                          typename T::v8 (&q)[KK]) {
  const uint16_t* src = static_cast<const uint16_t*>(a.q);
  if (g.real) src += (long long)(it.s.row0 + g.tok) * a.q_n + (long long)g.head * a.q_h;
  const uint32_t flip = a.q_sign < 0 ? 0x80008000u : 0u;
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    const int d = dim(kk);
    uint4 x = make_uint4(0, 0, 0, 0);
    if (g.real && a.q_sign) x = load16(reinterpret_cast<const uint8_t*>(src + d), (a.D - d) * 2, a.q_aligned);
    q[kk] = __builtin_bit_cast(typename T::v8, make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip));
  }
}

// Where 32 tokens of a score tile from t0 on lie for lane half `half`:
// register i is token t0 + 8 (i / 4) + 4 half + i % 4.
__device__ __forceinline__ bool needs_mask(const ChunkArgs& a, const RowGroup& g, int t0, uint32_t there) {
  return there != ~0u || (a.causal && t0 + 31 > g.first_pos) || (a.window && t0 <= g.last_pos - a.window);
}
__device__ __forceinline__ void mask_scores(const ChunkArgs& a, const Item& it, const RowGroup& g, int t0, uint32_t there,
                                            int half, f32x16& s) {
  const int hi = (a.causal ? min(g.pos, it.s.ctx - 1) : it.s.ctx - 1) - t0 - 4 * half;
  const int lo = a.window ? g.pos - a.window - t0 - 4 * half : -0x40000000;
  const uint32_t bits = there >> (4 * half);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int t = 8 * (i / 4) + i % 4;
    s[i] = t <= hi && t > lo && (bits >> t & 1) ? s[i] : -INFINITY;
  }
}

__device__ __forceinline__ float top_of(const f32x16& s) {
  float top = s[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
  return top;
}

// Weights are 2^(score - m).  The reference m is moved to kMaxBias below the
// running maximum, and only when that is kMaxLag above the maximum it was last
// moved for: the accumulators are rescaled a few times per row, not per block,
// and a row's largest weight stays between 2^kMaxBias and 2^(kMaxBias +
// kMaxLag).  P is the weights' type.
constexpr float kMaxLag = 8.f;
template <typename P>
constexpr float kMaxBias = std::is_same_v<P, F16> ? 7.f : 0.f;
template <typename P, int NB>
__device__ __forceinline__ void raise_max(float top, float& m, float& l, f32x16 (&o)[NB]) {
  if (__builtin_expect(__any(top > m + (kMaxBias<P> + kMaxLag)), 0)) {
    const float next = fmaxf(m, top - kMaxBias<P>);
    const float f = next == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - next);
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[n][i] *= f;
    l *= f;
    m = next;
  }
}

// A group's results: to the output, or to the workspace as a share's partial.
// Lane (col, half) holds dims dim(n, 2 i + 4 half) .. + 3 of its row in
// registers i .. i + 3 of block n.
template <typename T, int DP, typename Dim>
__device__ __forceinline__ void put_rows(const ChunkArgs& a, const Item& it, const RowGroup& g, float m, float l,
                                         const f32x16 (&o)[DP / 32], Dim dim) {
  constexpr int NB = DP / 32;
  const int half = __lane_id() >> 5;
  if (!g.real) return;
  if (it.shares > 1) {
    const long long slot = (long long)blockIdx.x * a.tile_rows + g.row;
    float* dst = a.part + slot * DP;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<float4*>(dst + dim(n, 2 * i + 4 * half)) =
            make_float4(o[n][i], o[n][i + 1], o[n][i + 2], o[n][i + 3]);
    if (half == 0) a.ml[slot] = make_float2(m, l);
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const long long at = (long long)(it.s.row0 + g.tok) * a.H + g.head;
  uint16_t* dst = static_cast<uint16_t*>(a.out) + at * a.D;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int d = dim(n, 2 * i + 4 * half);
      const f32x2 x = {o[n][i] * inv, o[n][i + 1] * inv}, y = {o[n][i + 2] * inv, o[n][i + 3] * inv};
      const uint2 w = make_uint2(__builtin_bit_cast(uint32_t, __builtin_convertvector(x, typename T::v2)),
                                 __builtin_bit_cast(uint32_t, __builtin_convertvector(y, typename T::v2)));
      if (a.out_aligned) {
        if (d < a.D) *reinterpret_cast<uint2*>(dst + d) = w;
      } else {
        if (d < a.D) dst[d] = (uint16_t)w.x;
        if (d + 1 < a.D) dst[d + 1] = (uint16_t)(w.x >> 16);
        if (d + 2 < a.D) dst[d + 2] = (uint16_t)w.y;
        if (d + 3 < a.D) dst[d + 3] = (uint16_t)(w.y >> 16);
      }
    }
  if (a.lse && half == 0) a.lse[at] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * 0.69314718055994531f;
}

// Joins the partials of wavefronts FROM .. into those before them through LDS
// (kPartial bytes each).  Every wavefront of the workgroup calls it.
template <int NB>
__device__ __forceinline__ void join(float* lds, bool give, bool take, int slot, float& m, float& l, f32x16 (&o)[NB]) {
  float* x = lds + slot * (NB * 16 + 2) * 64 + (threadIdx.x & 63);
  __syncthreads();
  if (give) {
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) x[(n * 16 + i) * 64] = o[n][i];
    x[NB * 16 * 64] = m;
    x[(NB * 16 + 1) * 64] = l;
  }
  __syncthreads();
  if (take) {
    const float m2 = x[NB * 16 * 64], l2 = x[(NB * 16 + 1) * 64];
    const float both = fmaxf(m, m2);
    const float f1 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - both);
    const float f2 = m2 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m2 - both);
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[n][i] = o[n][i] * f1 + x[(n * 16 + i) * 64] * f2;
    l = l * f1 + l2 * f2;
    m = both;
  }
}

// V's operand for 16 tokens (tokens 4 half .. + 3 and 8 + 4 half .. + 3 of
// them) and dims 32 n .. + 31, from row-major LDS.
template <typename V8>
__device__ __forceinline__ V8 read_v(const uint8_t* v_lds, int stride, int token0, int n) {
  typedef __attribute__((address_space(3))) s16x4* lds_t;
  const int lane = __lane_id();
  const uint8_t* x =
      v_lds + (token0 + 4 * (lane >> 5) + ((lane & 15) >> 2)) * stride + (n * 32 + (lane & 16) + (lane & 3) * 4) * 2;
  const s16x4 r0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)x);
  const s16x4 r1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(x + 8 * stride));
  return __builtin_bit_cast(V8, __builtin_shufflevector(r0, r1, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Gathers blocks of 64 tokens through the page table, a run of consecutive
// tokens to each of WAVES wavefronts, which finds its own pages (a block
// ahead): global memory to registers (load), registers to LDS (put).  A run
// within one page (page sizes that are multiples of its length) has one
// address; other page sizes, and runs with tokens that are not there, look up
// every row.
template <typename T, int KIND, int DP, int WAVES>
struct Stage {
  using Tile = ChunkTile<KIND, DP>;
  static constexpr bool QUANT = Tile::kQuant;
  static constexpr int TN = Tile::kTokens, RUN = TN / WAVES;
  static constexpr int kRun = RUN * Tile::kPerRow;  // 16-byte pieces of a run's K (and V)
  static constexpr int NP = (kRun + 63) / 64;       // per lane
  static constexpr bool kRagged = kRun % 64 != 0;
  static constexpr int kRing = 8;
  using Bits = std::conditional_t<RUN == 8, uint8_t, uint16_t>;
  struct Shared {
    unsigned long long there[kRing];  // tokens of a block that are there, a bit each
    alignas(16) float scale[kRing][2][QUANT ? TN : 4];
  };

  const ChunkArgs& a;
  Shared& sh;
  const uint8_t *k_base, *v_base;
  const float* s_base;
  const int32_t* table;
  int row_bytes, lane, wave;
  int limit;      // tokens from here on are not there
  bool one_page;  // a run lies in one page and is contiguous there
  uint4 kr[NP], vr[NP];
  int page;       // lane i: of token i % RUN of the run to be loaded next, -1: none
  uint32_t bits;  // tokens of the run in registers that are there
  float ks, vs;   // lane i < RUN: their scales

  __device__ __forceinline__ Stage(const ChunkArgs& args, const Item& it, int kvh, int blocks_end, Shared& shared)
      : a(args), sh(shared) {
    const int ctx = it.s.ctx, to = blocks_end;
    k_base = a.pool + a.layer_off + (long long)kvh * a.g.head;
    v_base = k_base + a.g.kv;
    s_base = QUANT ? a.scales + a.s_layer_off + (long long)kvh * a.g.s_head : nullptr;
    row_bytes = QUANT ? a.D : 2 * a.D;
    table = a.table + (long long)it.b * a.max_pp;
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    one_page = a.ps_shift >= 0 && a.PS >= RUN && a.aligned && a.D == DP;
    limit = min(ctx, to * TN);
  }

  // Page of the lane's token of a block (any entry of the table for a token
  // from `limit` on: load() drops those).
  __device__ __forceinline__ int page_of(int block) const {
    const int t = min(block * TN + RUN * wave + lane % RUN, limit - 1);
    return limit > 0 ? table[page_index(a, t)] : -1;
  }

  // `page` is the block's; on return it is the next block's.
  __device__ __forceinline__ void load(int block) {
    const int run0 = block * TN + RUN * wave, t = run0 + lane % RUN;
    const bool there = t < limit && page >= 0 && page < a.P;
    bits = (uint32_t)__ballot(there) & ((1u << RUN) - 1);
    reinterpret_cast<Bits*>(&sh.there[block % kRing])[wave] = (Bits)bits;  // (every lane the same)
    const bool fast = one_page && bits == (1u << RUN) - 1;
    const int slot = fast ? t & (a.PS - 1) : t - page_index(a, t) * a.PS;
    if constexpr (QUANT) {
      ks = vs = 0.f;
      if (there && lane < RUN) {
        const float* s = s_base + (long long)page * a.g.s_page + (KIND == kSrcI8 ? slot : 0);
        ks = s[0];
        vs = s[a.g.s_kv];
      }
    }
    if (__builtin_expect(fast, 1)) {
      const long long run = (long long)__builtin_amdgcn_readfirstlane(page) * a.g.page +
                            (long long)((run0 & (a.PS - 1)) * row_bytes);
      const uint8_t *k = k_base + run, *v = v_base + run;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const uint32_t off = (lane + 64 * i) * 16;
        if (kRagged && lane + 64 * i >= kRun) break;
        kr[i] = *reinterpret_cast<const uint4*>(k + off);
        vr[i] = *reinterpret_cast<const uint4*>(v + off);
      }
      page = page_of(block + 1);
      return;
    }
    const long long place = there ? (long long)page * a.g.page + (long long)slot * row_bytes : -1;
    page = page_of(block + 1);
    int first = lane;  // opaque: what follows from it stays here, in no register of the loop
    asm("" : "+v"(first));
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = first + 64 * i;
      kr[i] = vr[i] = make_uint4(0, 0, 0, 0);
      const int w = c % Tile::kPerRow;
      const long long at = __shfl(place, c / Tile::kPerRow % RUN);
      // V of the quantized pools: four tokens' codes of a dim in a dword
      const int w4 = c % (DP / 4);
      const long long at4 = QUANT ? __shfl(place, c / (DP / 4) * 4 % RUN) : 0;
      if (kRagged && c >= kRun) continue;
      if (at >= 0) kr[i] = load16(k_base + at + w * 16, row_bytes - w * 16, a.aligned);
      if constexpr (!QUANT) {
        if (at >= 0) vr[i] = load16(v_base + at + w * 16, row_bytes - w * 16, a.aligned);
      } else {
        if (at4 >= 0 && w4 * 4 < a.D) vr[i] = load16(v_base + at4 + w4 * 16, 16, a.aligned);
      }
    }
  }

  __device__ __forceinline__ void put(int block, uint8_t* k_lds, uint8_t* v_lds) {
    int first = lane;
    if constexpr (QUANT) asm("" : "+v"(first));  // (as in load: the places in LDS are not worth registers)
    if (QUANT && lane < RUN) {
      sh.scale[block % kRing][0][RUN * wave + lane] = ks;
      sh.scale[block % kRing][1][RUN * wave + lane] = vs;
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = first + 64 * i;
      if (kRagged && c >= kRun) break;
      const int t = RUN * wave + c / Tile::kPerRow, w = c % Tile::kPerRow;
      if constexpr (!QUANT) {
        *reinterpret_cast<uint4*>(k_lds + t * Tile::kKStride + w * 16) = kr[i];
        *reinterpret_cast<uint4*>(v_lds + t * Tile::kVStride + w * 16) = vr[i];
      } else {
        const uint2 k0 = codes4<T, KIND>(kr[i].x), k1 = codes4<T, KIND>(kr[i].y);
        const uint2 k2 = codes4<T, KIND>(kr[i].z), k3 = codes4<T, KIND>(kr[i].w);
        uint4* dst = reinterpret_cast<uint4*>(k_lds + t * Tile::kKStride + w * 32);
        dst[0] = make_uint4(k0.x, k0.y, k1.x, k1.y);
        dst[1] = make_uint4(k2.x, k2.y, k3.x, k3.y);
        // V^T: [16-token step][lane half][dim][8 tokens]
        const int quad = RUN / 4 * wave + c / (DP / 4), w4 = c % (DP / 4);
        uint8_t* vt = v_lds + ((quad >> 2) * 2 + (quad & 1)) * DP * 16 + (quad >> 1 & 1) * 8;
        uint32_t words[4] = {vr[i].x, vr[i].y, vr[i].z, vr[i].w};
        if (bits != (1u << RUN) - 1) {
          const uint32_t keep = keep_bytes(bits >> (c / (DP / 4) * 4));
#pragma unroll
          for (int j = 0; j < 4; ++j) words[j] &= keep;
        }
        if (DP % 64 == 0 && a.D == DP) {  // four dims 16 apart
          uint8_t* v0 = vt + (w4 * 4 / (DP / 16) + 16 * (w4 * 4 % (DP / 16))) * 16;
#pragma unroll
          for (int j = 0; j < 4; ++j) *reinterpret_cast<uint2*>(v0 + j * 256) = codes4<Bf16, KIND>(words[j]);
        } else if (w4 * 4 < a.D) {
          const int nd = a.D >> 4;
          int d0 = w4 * 4 / nd, d1 = w4 * 4 % nd;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            *reinterpret_cast<uint2*>(vt + (d0 + 16 * d1) * 16) = codes4<Bf16, KIND>(words[j]);
            if (++d1 == nd) d1 = 0, ++d0;
          }
        }
      }
    }
  }
};

// Dims D .. DP - 1 of a block's V^T, which no code is staged for: zeros, so that
// the accumulators of those dims are too (any_nan looks at all).  Once per
// buffer, by the whole workgroup.
template <int DP>
__device__ __forceinline__ void clear_padding(const ChunkArgs& a, uint8_t* v_lds) {
  const int pad = DP - a.D;
  for (int i = threadIdx.x; i < 8 * pad; i += blockDim.x)  // [4 steps of 16 tokens][2 halves] of DP x 16 bytes
    *reinterpret_cast<uint4*>(v_lds + (i / pad * DP + a.D + i % pad) * 16) = make_uint4(0, 0, 0, 0);
}

// Scores of 32 tokens times their K scales, and weights times their V scales.
__device__ __forceinline__ void scale_scores(const float* ks, int half, f32x16& s) {
#pragma unroll
  for (int i = 0; i < 16; i += 4) {
    const float4 x = *reinterpret_cast<const float4*>(ks + 2 * i + 4 * half);
    s[i] *= x.x, s[i + 1] *= x.y, s[i + 2] *= x.z, s[i + 3] *= x.w;
  }
}
__device__ __forceinline__ void scale_weights(const float* vs, int e, int half, f32x8& p) {
  const float4 x = *reinterpret_cast<const float4*>(vs + 16 * e + 4 * half);
  const float4 y = *reinterpret_cast<const float4*>(vs + 16 * e + 8 + 4 * half);
  p[0] *= x.x, p[1] *= x.y, p[2] *= x.z, p[3] *= x.w;
  p[4] *= y.x, p[5] *= y.y, p[6] *= y.z, p[7] *= y.w;
}

// A tile of at most 32 rows: every wavefront attends 32 tokens at a time of
// its own, with no barrier, and they join at the end.  K comes from
// memory in the layout of the matrix operand (a lane's 16-byte pieces of its
// token's row), refilled as soon as the scores are taken; V of the quantized
// pools too (its tiling puts a lane's four tokens of a dim in a dword), V of
// float pools through the wavefront's own LDS.
// Bound: memory.  64 sequences of 4 tokens after about 4050, 40 heads over 8,
// int8: 118 us with the merge, 4.7 TB/s (a copy reaches 5.0).
template <typename T, int KIND, int DP, int WAVES>
__device__ __forceinline__ void few_rows(const ChunkArgs& a, const Item& it, int kvh, int rows, int from, int to,
                                         uint8_t* lds, float (*own_scale)[2][32]) {
  using Tile = ChunkTile<KIND, DP>;
  using PT = std::conditional_t<KIND >= kSrcI8, Bf16, T>;
  constexpr bool QUANT = Tile::kQuant;
  constexpr bool SPLIT_P = QUANT && std::is_same_v<T, F16>;
  constexpr int NB = DP / 32, KK = DP / 16, KP = QUANT ? DP / 32 : DP / 16;
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const RowGroup g = row_group(a, it, kvh, rows, 0);

  typename T::v8 q[KK];
  load_rows<T, KK>(a, it, g, [&](int kk) { return QUANT ? (kk >> 1) * 32 + half * 16 + (kk & 1) * 8 : kk * 16 + half * 8; },
                   q);
  f32x16 o[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) o[n] = f32x16{};
  float m = -INFINITY, l = 0.f;

  const uint8_t* const k_base = a.pool + a.layer_off + (long long)kvh * a.g.head;
  const uint8_t* const v_base = k_base + a.g.kv;
  const float* const s_base = QUANT ? a.scales + a.s_layer_off + (long long)kvh * a.g.s_head : nullptr;
  const int32_t* const table = a.table + (long long)it.b * a.max_pp;
  const int row_bytes = QUANT ? a.D : 2 * a.D;
  const int nd = a.D >> 4;
  const bool whole = a.D == DP;  // a lane's dims of V are consecutive dwords
  uint8_t* const own_v = lds + wave * Tile::kOwnV;

  const auto page_of = [&](int sub) {
    const int t = sub * 32 + col;
    return sub < 2 * to && t < it.s.ctx ? table[page_index(a, t)] : -1;
  };
  const auto place_of = [&](int sub, int page) {
    const int t = sub * 32 + col;
    return page >= 0 && page < a.P ? (long long)page * a.g.page + (long long)(t - page_index(a, t) * a.PS) * row_bytes : -1;
  };
  // DEPTH x 32 tokens are under way per wavefront
  constexpr int DEPTH = QUANT ? 2 : 1;
  uint4 kr[DEPTH][KP], vr[DEPTH][QUANT ? 1 : KP];
  uint32_t vw[DEPTH][2][2][QUANT ? NB : 1];
  float ks[DEPTH], vs[DEPTH];
  long long at[DEPTH];
  int page[DEPTH];  // of the 32 tokens to be loaded next
  const auto load_k = [&](int b, int sub) {
#pragma unroll
    for (int p = 0; p < KP; ++p) {
      const int d = QUANT ? p * 32 + half * 16 : (p * 16 + half * 8) * 2;  // bytes into the row
      kr[b][p] = at[b] >= 0 ? load16(k_base + at[b] + d, row_bytes - d, a.aligned) : make_uint4(0, 0, 0, 0);
    }
    if constexpr (QUANT) {
      ks[b] = vs[b] = 0.f;
      if (at[b] >= 0) {
        const int t = sub * 32 + col;
        const float* s = s_base + (long long)page[b] * a.g.s_page + (KIND == kSrcI8 ? t - page_index(a, t) * a.PS : 0);
        ks[b] = s[0];
        vs[b] = s[a.g.s_kv];
      }
    }
  };
  const auto load_v = [&](int b) {
    if constexpr (QUANT) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const long long quad = __shfl(at[b], 16 * e + 8 * j + 4 * half);  // place of the four tokens' first
          uint32_t(&w)[NB] = vw[b][e][j];
          const uint8_t* p = v_base + quad + ((col & 15) * nd + (whole ? NB : 1) * (col >> 4)) * 4;
#pragma unroll
          for (int n = 0; n < NB; ++n) w[n] = 0;
          if (quad < 0) continue;
          if (whole && a.aligned) {
            __builtin_memcpy(w, __builtin_assume_aligned(p, NB % 4 == 0 ? 16 : NB % 2 == 0 ? 8 : 4), 4 * NB);
          } else {
#pragma unroll
            for (int n = 0; n < NB; ++n) {
              const uint8_t* x = p + (whole ? 4 * n : 8 * n);
              if (whole || 2 * n + (col >> 4) < nd)
                w[n] = x[0] | (uint32_t)x[1] << 8 | (uint32_t)x[2] << 16 | (uint32_t)x[3] << 24;
            }
          }
        }
    } else {
#pragma unroll
      for (int p = 0; p < KP; ++p) {
        const int d = (p * 16 + half * 8) * 2;
        vr[b][p] = at[b] >= 0 ? load16(v_base + at[b] + d, row_bytes - d, a.aligned) : make_uint4(0, 0, 0, 0);
      }
    }
  };

  int sub = 2 * from + wave;
#pragma unroll
  for (int b = 0; b < DEPTH; ++b) page[b] = page_of(sub + b * WAVES);
#pragma unroll
  for (int b = 0; b < DEPTH; ++b) {
    at[b] = place_of(sub + b * WAVES, page[b]);
    load_k(b, sub + b * WAVES);
    load_v(b);
  }
#pragma unroll
  for (int b = 0; b < DEPTH; ++b) page[b] = page_of(sub + (DEPTH + b) * WAVES);
  for (; sub < 2 * to; sub += DEPTH * WAVES) {
#pragma unroll
    for (int b = 0; b < DEPTH; ++b) {
      const int now = sub + b * WAVES, next = now + DEPTH * WAVES, t0 = now * 32;
      if (b > 0 && now >= 2 * to) break;
      const uint32_t there = (uint32_t)__ballot(at[b] >= 0);
      f32x16 s{};
#pragma unroll
      for (int p = 0; p < KP; ++p) {
        if constexpr (QUANT) {
          const uint2 x0 = codes4<T, KIND>(kr[b][p].x), x1 = codes4<T, KIND>(kr[b][p].y);
          const uint2 x2 = codes4<T, KIND>(kr[b][p].z), x3 = codes4<T, KIND>(kr[b][p].w);
          s = T::mfma(__builtin_bit_cast(typename T::v8, make_uint4(x0.x, x0.y, x1.x, x1.y)), q[2 * p], s);
          s = T::mfma(__builtin_bit_cast(typename T::v8, make_uint4(x2.x, x2.y, x3.x, x3.y)), q[2 * p + 1], s);
        } else {
          s = T::mfma(__builtin_bit_cast(typename T::v8, kr[b][p]), q[p], s);
        }
      }
      if constexpr (QUANT) {
        if (half == 0) {
          own_scale[wave][0][col] = ks[b];
          own_scale[wave][1][col] = vs[b];
        }
      }
      // this buffer's next K (its V still waits for the weights)
      const long long at1 = place_of(next, page[b]);
      at[b] = at1;
      load_k(b, next);
      __syncwarp();
      if constexpr (QUANT) scale_scores(own_scale[wave][0], half, s);
      if (needs_mask(a, g, t0, there)) mask_scores(a, it, g, t0, there, half, s);
      raise_max<PT, NB>(xor_max<32>(top_of(s)) * a.sc, m, l, o);
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.sc, -ref));
        l += s[i];
      }
      if constexpr (!QUANT) {
#pragma unroll
        for (int p = 0; p < KP; ++p)
          *reinterpret_cast<uint4*>(own_v + col * Tile::kVStride + (p * 16 + half * 8) * 2) = vr[b][p];
        load_v(b);
        __syncwarp();
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        f32x8 p;
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = s[8 * e + i];
        if constexpr (QUANT) scale_weights(own_scale[wave][1], e, half, p);
        const auto pb = __builtin_convertvector(p, typename PT::v8);
        typename PT::v8 low;
        if constexpr (SPLIT_P) low = __builtin_convertvector(p - __builtin_convertvector(pb, f32x8), typename PT::v8);
        const uint32_t k0 = keep_bytes(there >> (16 * e + 4 * half)), k1 = keep_bytes(there >> (16 * e + 8 + 4 * half));
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          typename PT::v8 v;
          if constexpr (QUANT) {
            const uint2 x0 = codes4<Bf16, KIND>(vw[b][e][0][n] & k0), x1 = codes4<Bf16, KIND>(vw[b][e][1][n] & k1);
            v = __builtin_bit_cast(typename PT::v8, make_uint4(x0.x, x0.y, x1.x, x1.y));
          } else {
            v = read_v<typename PT::v8>(own_v, Tile::kVStride, 16 * e, n);
          }
          o[n] = PT::mfma(v, pb, o[n]);
          if constexpr (SPLIT_P) o[n] = PT::mfma(v, low, o[n]);
        }
      }
      if constexpr (QUANT) load_v(b);
      page[b] = page_of(next + DEPTH * WAVES);
      __syncwarp();
    }
  }
  l = xor_add<32>(l);
#pragma unroll
  for (int n = WAVES / 2; n >= 1; n /= 2)
    join<NB>(reinterpret_cast<float*>(lds), wave >= n && wave < 2 * n, wave < n, wave & (n - 1), m, l, o);
  if (wave != 0) return;
  if (__builtin_expect(any_nan(o, g.real), 0) &&
      careful_rows<64>(a, it, kvh, KIND, 0, rows, g.first_pos, g.last_pos, from, to))
    return;
  put_rows<T, DP>(a, it, g, m, l, o, [&](int n, int r) {
    return QUANT && whole ? (r & 15) + 16 * (NB * (r >> 4) + n) : n * 32 + r;
  });
}

// Tiles of 128 rows, 32 to a wavefront, two workgroups to a CU: one's
// products run while the other's wavefronts are in their softmax.
// Bound: matrix cores in the products, LDS latency between them; a prompt
// that takes the kernel below 488 us takes this one 609.
template <typename T, int KIND, int DP>
__global__ void __launch_bounds__(kChunkThreads, DP <= 128 ? 2 : 1) chunk_attn_kernel(ChunkArgs a) {
  using Tile = ChunkTile<KIND, DP>;
  using Gather = Stage<T, KIND, DP, 4>;
  using PT = std::conditional_t<KIND >= kSrcI8, Bf16, T>;  // type of the second product
  constexpr bool QUANT = Tile::kQuant;
  constexpr bool SPLIT_P = QUANT && std::is_same_v<T, F16>;
  constexpr int TN = Tile::kTokens, NB = DP / 32, KK = DP / 16;
  constexpr int kLds = max3(Tile::kBytes, 2 * Tile::kPartial, 4 * Tile::kOwnV);
  __shared__ __align__(16) uint8_t lds[kLds];
  __shared__ __align__(16) typename Gather::Shared shared;
  __shared__ __align__(16) float own_scale[QUANT ? 4 : 1][2][32];
  uint8_t* const k_lds = lds;
  uint8_t* const v_lds = lds + Tile::kKBytes;

  const int kvh = blockIdx.x % a.KH;
  Item it;
  if (!find_item<TN>(a, blockIdx.x / a.KH, it)) return;
  int from, to;
  item_blocks<TN>(a, it, from, to);
  put_record(a, it, kvh);
  const int rows = min(a.tile_rows, it.s.q_len * a.G - it.tile * a.tile_rows);
  if constexpr (DP <= 128) {  // (at 256 its operands would not fit the registers)
    if (rows <= 32) {
      few_rows<T, KIND, DP, 4>(a, it, kvh, rows, from, to, lds, own_scale);
      return;
    }
  }

  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // up to 64 rows leave two wavefronts to a row group, one for each half of a
  // block's tokens
  const bool halves = rows <= 64;
  const int group = halves ? wave >> 1 : wave;
  const bool active = group * 32 < rows;
  const RowGroup g = row_group(a, it, kvh, rows, group * 32);
  typename T::v8 q[KK];
  load_rows<T, KK>(a, it, g, [&](int kk) { return kk * 16 + half * 8; }, q);
  f32x16 o[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) o[n] = f32x16{};
  float m = -INFINITY, l = 0.f;

  // NS x 32 tokens of a block from its 32-token part st0 on
  const auto compute = [&](int block, auto ns, int st0) {
    constexpr int NS = decltype(ns)::value;
    const int t0 = block * TN + st0 * 32;
    if (a.causal && t0 > g.last_pos) return;
    if (a.window && t0 + NS * 32 - 1 <= g.first_pos - a.window) return;
    const unsigned long long there = shared.there[block % Gather::kRing];
    const auto* scale = shared.scale[block % Gather::kRing];
    f32x16 s[NS];
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      s[u] = f32x16{};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const uint4 x = *reinterpret_cast<const uint4*>(k_lds + ((st0 + u) * 32 + col) * Tile::kKStride +
                                                        (kk * 16 + half * 8) * 2);
        s[u] = T::mfma(__builtin_bit_cast(typename T::v8, x), q[kk], s[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      if constexpr (QUANT) scale_scores(scale[0] + (st0 + u) * 32, half, s[u]);
      const uint32_t bits = (uint32_t)(there >> (32 * (st0 + u)));
      if (needs_mask(a, g, t0 + 32 * u, bits)) mask_scores(a, it, g, t0 + 32 * u, bits, half, s[u]);
      top = fmaxf(top, top_of(s[u]));
    }
    raise_max<PT, NB>(xor_max<32>(top) * a.sc, m, l, o);
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int u = 0; u < NS; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[u][i] = __builtin_amdgcn_exp2f(fmaf(s[u][i], a.sc, -ref));
        l += s[u][i];
      }
#pragma unroll
    for (int u = 0; u < NS; ++u)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        f32x8 p;
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = s[u][8 * e + i];
        if constexpr (QUANT) scale_weights(scale[1] + (st0 + u) * 32, e, half, p);
        const auto pb = __builtin_convertvector(p, typename PT::v8);
        typename PT::v8 low;
        if constexpr (SPLIT_P) low = __builtin_convertvector(p - __builtin_convertvector(pb, f32x8), typename PT::v8);
        const int step = (st0 + u) * 2 + e;  // of 16 tokens
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          typename PT::v8 v;
          if constexpr (QUANT)
            v = __builtin_bit_cast(typename PT::v8, *reinterpret_cast<const uint4*>(
                                                        v_lds + ((step * 2 + half) * DP + n * 32 + col) * 16));
          else
            v = read_v<typename PT::v8>(v_lds, Tile::kVStride, step * 16, n);
          o[n] = PT::mfma(v, pb, o[n]);
          if constexpr (SPLIT_P) o[n] = PT::mfma(v, low, o[n]);
        }
      }
  };

  Gather st(a, it, kvh, to, shared);
  st.page = st.page_of(from);
  if (from < to) st.load(from);
  if (QUANT && a.D < DP) clear_padding<DP>(a, v_lds);
  for (int block = from; block < to; ++block) {
    __syncthreads();  // the block before is computed
    st.put(block, k_lds, v_lds);
    __syncthreads();
    if (block + 1 < to) st.load(block + 1);
    if (active) {
      if (halves)
        compute(block, std::integral_constant<int, 1>{}, wave & 1);
      else
        compute(block, std::integral_constant<int, 2>{}, 0);
    }
  }
  l = xor_add<32>(l);
  if (halves) join<NB>(reinterpret_cast<float*>(lds), active && (wave & 1), active && !(wave & 1), group, m, l, o);
  if (!active || (halves && (wave & 1))) return;
  if (__builtin_expect(any_nan(o, g.real), 0) &&
      careful_rows<TN>(a, it, kvh, KIND, group * 32, min(rows, group * 32 + 32), g.first_pos, g.last_pos, from, to))
    return;
  put_rows<T, DP>(a, it, g, m, l, o, [](int n, int r) { return n * 32 + r; });
}

// Tiles of 256 rows, 32 to each of eight wavefronts, one workgroup to a CU.
// A wavefront forms the scores of the next block while the weights of this
// one are taken.  Its SIMD's other wavefront runs half a step behind: one
// meets the block's barrier at the end of a step, the other between the
// products of K and of V, so that one's masks, maxima and staging fall beside
// the other's products.  Four blocks are in LDS (the wavefronts ahead write
// block + 2 while those behind still read block - 1), a fifth in registers.
// Bound: matrix cores, 2048 cycles of a block at head_dim 128, and the vector
// work beside them.  A prompt of 8192 tokens, bf16: 490 us, 1.0 PFLOP/s (a
// library product of 8192^3 reaches 1.17), matrix cores busy 51 % of the
// cycles, vector ALUs 50 %; 256 tokens after 130,816 over fp8 1210 us, 0.91
// PFLOP/s, 40 and 58 % (codes to bf16).  At head_dim 128 all 256 registers are
// taken: 3 are spilled over float pools, 1 over int8 and fp8, 14 and 15 there
// with fp16 queries, whose weights are two operands.
template <typename T, int KIND, int DP>
__global__ void __launch_bounds__(kLargeThreads, 1) chunk_attn_large_kernel(ChunkArgs a) {
  using Tile = ChunkTile<KIND, DP>;
  using Gather = Stage<T, KIND, DP, 8>;
  using PT = std::conditional_t<KIND >= kSrcI8, Bf16, T>;
  constexpr bool QUANT = Tile::kQuant;
  constexpr bool SPLIT_P = QUANT && std::is_same_v<T, F16>;
  constexpr int TN = Tile::kTokens, NB = DP / 32, KK = DP / 16;
  constexpr int kLds = max3(4 * Tile::kBytes, 4 * Tile::kPartial, 8 * Tile::kOwnV);
  __shared__ __align__(16) uint8_t lds[kLds];
  __shared__ __align__(16) typename Gather::Shared shared;
  __shared__ __align__(16) float own_scale[QUANT ? 8 : 1][2][32];

  const int kvh = blockIdx.x % a.KH;
  Item it;
  if (!find_item<TN>(a, blockIdx.x / a.KH, it)) return;
  int from, to;
  item_blocks<TN>(a, it, from, to);
  put_record(a, it, kvh);
  const int rows = min(a.tile_rows, it.s.q_len * a.G - it.tile * a.tile_rows);
  if (rows <= 32) {
    few_rows<T, KIND, DP, 8>(a, it, kvh, rows, from, to, lds, own_scale);
    return;
  }

  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // up to 128 rows leave two wavefronts to a row group, one for each half of a
  // block's tokens
  const bool halves = rows <= 128;
  const int group = halves ? wave >> 1 : wave;
  const bool active = group * 32 < rows;
  const RowGroup g = row_group(a, it, kvh, rows, group * 32);
  typename T::v8 q[KK];
  load_rows<T, KK>(a, it, g, [&](int kk) { return kk * 16 + half * 8; }, q);
  f32x16 o[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) o[n] = f32x16{};
  float m = -INFINITY, l = 0.f;

  Gather st(a, it, kvh, to, shared);
  {
    Gather second = st;
    st.page = st.page_of(from);
    second.page = st.page_of(from + 1);
    st.load(from);
    second.load(from + 1);
    if (QUANT && a.D < DP)
      for (int i = 0; i < 4; ++i) clear_padding<DP>(a, lds + i * Tile::kBytes + Tile::kKBytes);
    __syncthreads();
    st.put(from, lds, lds + Tile::kKBytes);
    second.put(from + 1, lds + Tile::kBytes, lds + Tile::kBytes + Tile::kKBytes);
    st.page = second.page;
  }
  st.load(from + 2);
  __syncthreads();

  // NS x 32 tokens of each block from its 32-token part u0 on
  const auto blocks = [&](auto ns, auto behind, int u0) {
    constexpr int NS = decltype(ns)::value;
    constexpr bool BEHIND = decltype(behind)::value;
    constexpr int FIRST = NS * KK, SECOND = 2 * NS * NB, ALL = FIRST + SECOND;  // products of a step
    constexpr int AHEAD = 4;  // operands under way from LDS
    // operand of product i: K (16 dims of 32 tokens), then V (32 dims of 16 tokens)
    const auto read_k = [&](const uint8_t* k_lds, int i) {
      return *reinterpret_cast<const uint4*>(k_lds + ((u0 + i % NS) * 32 + col) * Tile::kKStride +
                                             (i / NS * 16 + half * 8) * 2);
    };
    const auto read_operand = [&](const uint8_t* k_lds, const uint8_t* v_lds, int i) {
      if (i < FIRST) return read_k(k_lds, i);
      const int part = 2 * u0 + (i - FIRST) / NB, n = (i - FIRST) % NB;
      if constexpr (QUANT)
        return *reinterpret_cast<const uint4*>(v_lds + ((part * 2 + half) * DP + n * 32 + col) * 16);
      else
        return read_v<uint4>(v_lds, Tile::kVStride, part * 16, n);
    };
    const auto k_scale = [&](int block, f32x16 (&s)[NS]) {
      if constexpr (QUANT) {
#pragma unroll
        for (int u = 0; u < NS; ++u)
          scale_scores(shared.scale[block % Gather::kRing][0] + (u0 + u) * 32, half, s[u]);
      }
    };

    float top = -INFINITY;  // of the scores `now` of the next step
    // of its block: tokens that are there; blocks [whole0, whole1) are seen
    // whole by every row of the group, as far as they are there
    uint32_t there[NS];
    const auto read_there = [&](int block) {
#pragma unroll
      for (int u = 0; u < NS; ++u)
        there[u] = __builtin_amdgcn_readfirstlane(
            reinterpret_cast<const uint32_t*>(&shared.there[block % Gather::kRing])[u0 + u]);
    };
    const int whole0 = a.window ? (max(g.last_pos - a.window + 1, 0) + TN - 1) / TN : 0;
    const int whole1 = a.causal ? (g.first_pos + 1) / TN : 0x7fffffff;
    // One block: the weights of its scores `now` and their product with V,
    // and the scores `next` of the block after it.  Written slot by slot, a
    // product each, with the operand four slots ahead and a share of the
    // vector work; nothing crosses a slot's end.  (Left to the compiler, each
    // product waited for the LDS read right before it.)
    const auto step = [&](int block, const uint8_t* v_lds, const uint8_t* next_k, f32x16 (&now)[NS],
                          f32x16 (&next)[NS]) {
      uint4 f[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) f[i] = read_operand(next_k, v_lds, i);
      bool mask = block < whole0 || block >= whole1;
#pragma unroll
      for (int u = 0; u < NS; ++u) mask |= there[u] != ~0u;
      if (__builtin_expect(mask, 0)) {
        top = -INFINITY;
#pragma unroll
        for (int u = 0; u < NS; ++u) {
          mask_scores(a, it, g, block * TN + 32 * (u0 + u), there[u], half, now[u]);
          top = fmaxf(top, top_of(now[u]));
        }
      }
      raise_max<PT, NB>(xor_max<32>(top) * a.sc, m, l, o);
      const float ref = m == -INFINITY ? 0.f : m;
      top = -INFINITY;
      typename PT::v8 pb[2 * NS], low[2 * NS];
#pragma unroll
      for (int u = 0; u < NS; ++u) next[u] = f32x16{};
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < ALL; ++i) {
        if (BEHIND && i == FIRST) __syncthreads();
        const uint4 x = f[i % AHEAD];
        if (i < FIRST) {
          next[i % NS] = T::mfma(__builtin_bit_cast(typename T::v8, x), q[i / NS], next[i % NS]);
        } else {
          const int e = (i - FIRST) / NB, n = (i - FIRST) % NB;
          o[n] = PT::mfma(__builtin_bit_cast(typename PT::v8, x), pb[e], o[n]);
          if constexpr (SPLIT_P) o[n] = PT::mfma(__builtin_bit_cast(typename PT::v8, x), low[e], o[n]);
        }
        if (i + AHEAD < ALL) f[i % AHEAD] = read_operand(next_k, v_lds, i + AHEAD);
        // weights, the last of them ready for the last 16 tokens' products
        constexpr int kUntil = FIRST + (2 * NS - 1) * NB;
        const int c0 = (16 * NS * i + kUntil - 1) / kUntil, c1 = (16 * NS * (i + 1) + kUntil - 1) / kUntil;
#pragma unroll
        for (int c = c0; c < (c1 < 16 * NS ? c1 : 16 * NS); ++c) {
          const float y = __builtin_amdgcn_exp2f(fmaf(now[c / 16][c % 16], a.sc, -ref));
          now[c / 16][c % 16] = y;
          l += y;
          if (c % 8 == 7) {
            const int e = c / 8;
            f32x8 p;
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = now[e / 2][8 * (e % 2) + j];
            if constexpr (QUANT)
              scale_weights(shared.scale[block % Gather::kRing][1] + (u0 + e / 2) * 32, e % 2, half, p);
            pb[e] = __builtin_convertvector(p, typename PT::v8);
            if constexpr (SPLIT_P)
              low[e] = __builtin_convertvector(p - __builtin_convertvector(pb[e], f32x8), typename PT::v8);
          }
        }
        if (i == ALL - 3) read_there(block + 1);
        // K scales and the maximum of the next scores, from two slots after they are whole
        if (i >= FIRST + 2) {
          constexpr int kSlots = SECOND - 2;
          const int t0 = 4 * NS * (i - FIRST - 2) / kSlots, t1 = 4 * NS * (i - FIRST - 1) / kSlots;
#pragma unroll
          for (int t = t0; t < t1; ++t) {
            f32x16& s = next[t / 4];
            const int j = t % 4 * 4;
            if constexpr (QUANT) {
              const float4 y = *reinterpret_cast<const float4*>(
                  shared.scale[(block + 1) % Gather::kRing][0] + (u0 + t / 4) * 32 + 2 * j + 4 * half);
              s[j] *= y.x, s[j + 1] *= y.y, s[j + 2] *= y.z, s[j + 3] *= y.w;
            }
            top = fmaxf(fmaxf(top, s[j]), s[j + 1]);
            top = fmaxf(fmaxf(top, s[j + 2]), s[j + 3]);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    const auto first_scores = [&](f32x16 (&s)[NS]) {
      read_there(from);
#pragma unroll
      for (int u = 0; u < NS; ++u) s[u] = f32x16{};
#pragma unroll
      for (int i = 0; i < FIRST; ++i)
        s[i % NS] = T::mfma(__builtin_bit_cast(typename T::v8, read_k(lds, i)), q[i / NS], s[i % NS]);
      k_scale(from, s);
#pragma unroll
      for (int u = 0; u < NS; ++u) top = fmaxf(top, top_of(s[u]));
    };

    f32x16 s0[NS], s1[NS];
    const auto turn = [&](int block, f32x16 (&now)[NS], f32x16 (&next)[NS]) {
      const auto slot = [&](int ahead) { return lds + ((block - from + ahead) & 3) * Tile::kBytes; };
      st.put(block + 2, slot(2), slot(2) + Tile::kKBytes);
      st.load(block + 3);
      if (active) step(block, slot(0) + Tile::kKBytes, slot(1), now, next);
      if (!BEHIND || !active) __syncthreads();
    };
    if (active) first_scores(s0);
    for (int block = from; block < to; block += 2) {
      turn(block, s0, s1);
      if (block + 1 < to) turn(block + 1, s1, s0);
    }
  };
  if (halves)
    blocks(std::integral_constant<int, 1>{}, std::false_type{}, wave & 1);
  else if (wave < 4)
    blocks(std::integral_constant<int, 2>{}, std::false_type{}, 0);
  else  // wavefronts w and w + 4 share a SIMD
    blocks(std::integral_constant<int, 2>{}, std::true_type{}, 0);
  l = xor_add<32>(l);
  if (halves) join<NB>(reinterpret_cast<float*>(lds), active && (wave & 1), active && !(wave & 1), group, m, l, o);
  if (!active || (halves && (wave & 1))) return;
  if (__builtin_expect(any_nan(o, g.real), 0) &&
      careful_rows<TN>(a, it, kvh, KIND, group * 32, min(rows, group * 32 + 32), g.first_pos, g.last_pos, from, to))
    return;
  put_rows<T, DP>(a, it, g, m, l, o, [](int n, int x) { return n * 32 + x; });
}

template <typename T, int KIND>
void launch_chunk16_t(const ChunkArgs& a, dim3 grid, hipStream_t st) {
  if (a.tile_rows == 256) {
    if (a.dp == 64)
      hipLaunchKernelGGL((chunk_attn_large_kernel<T, KIND, 64>), grid, dim3(kLargeThreads), 0, st, a);
    else if (a.dp == 96)
      hipLaunchKernelGGL((chunk_attn_large_kernel<T, KIND, 96>), grid, dim3(kLargeThreads), 0, st, a);
    else
      hipLaunchKernelGGL((chunk_attn_large_kernel<T, KIND, 128>), grid, dim3(kLargeThreads), 0, st, a);
    return;
  }
  if (a.dp == 64)
    hipLaunchKernelGGL((chunk_attn_kernel<T, KIND, 64>), grid, dim3(kChunkThreads), 0, st, a);
  else if (a.dp == 96)
    hipLaunchKernelGGL((chunk_attn_kernel<T, KIND, 96>), grid, dim3(kChunkThreads), 0, st, a);
  else
    hipLaunchKernelGGL((chunk_attn_kernel<T, KIND, 128>), grid, dim3(kChunkThreads), 0, st, a);
}

}  // namespace
}  // namespace vrm
