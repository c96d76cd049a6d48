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
// multiplies the scores.  Weights are rounded to the 16-bit type once (half a
// step, 2^-9 or 2^-12, independent from token to token: below the rounding of
// the output for two tokens or more); over quantized values they are bf16
// (fp16 would overflow under large scales), for fp16 queries as a high and a
// low part.
#pragma once
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

template <int KIND, int DP>
struct ChunkTile {
  static constexpr bool kQuant = KIND >= kSrcI8;
  static constexpr int kTokens = 64;
  // K rows padded by 16 bytes: the 16-byte reads of 8 consecutive tokens fall
  // on different banks.  V rows (float pools) at 64 or 192 mod 256 bytes: so
  // do the transposed reads' four tokens of 64 bytes.
  static constexpr int kKStride = DP * 2 + 16;
  static constexpr int kVStride = DP * 2 + (DP * 2 % 128 == 0 ? 64 : 0);
  static constexpr int kVBytes = kQuant ? kTokens * DP * 2 : kTokens * kVStride;
  static constexpr int kMerge = 2 * (DP / 32 * 16 + 2) * 64 * 4;  // two wavefronts' partials
  static constexpr int kTile = kTokens * kKStride + kVBytes;
  static constexpr int kBytes = kTile > kMerge ? kTile : kMerge;
  static constexpr int kPerRow = kQuant ? DP / 16 : DP / 8;          // 16-byte pieces of a K row
  static constexpr int kAll = kTokens * kPerRow;                     // of K (and of V)
  static constexpr int kPieces = (kAll + kChunkThreads - 1) / kChunkThreads;  // per thread
  static constexpr bool kRagged = kAll % kChunkThreads != 0;
};

template <typename T, int KIND, int DP>
__global__ void __launch_bounds__(kChunkThreads, DP <= 128 ? 2 : 1) chunk_attn_kernel(ChunkArgs a) {
  using Tile = ChunkTile<KIND, DP>;
  constexpr bool QUANT = Tile::kQuant;
  constexpr int TN = Tile::kTokens, NB = DP / 32, KK = DP / 16, NP = Tile::kPieces;
  using PT = std::conditional_t<QUANT, Bf16, T>;  // type of the second product
  constexpr bool SPLIT_P = QUANT && std::is_same_v<T, F16>;

  __shared__ __align__(16) uint8_t tile_lds[Tile::kBytes];
  __shared__ float scale_lds[2][TN];
  __shared__ long long place_lds[4][TN];  // a token's K row from the layer's start, -1: not there
  __shared__ unsigned long long there_lds[4];
  uint8_t* const k_lds = tile_lds;
  uint8_t* const v_lds = tile_lds + TN * Tile::kKStride;

  const int kvh = blockIdx.x % a.KH;
  Item it;
  if (!find_item<TN>(a, blockIdx.x / a.KH, it)) return;
  int from, to;
  item_blocks<TN>(a, it, from, to);
  put_record(a, it, kvh);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;

  // Rows of the tile over wavefronts: 32 each; few rows leave two wavefronts
  // to a row group, one for each half of a block's tokens.
  const int rows = min(kRows, it.s.q_len * a.G - it.tile * kRows);
  const bool halves = rows <= 64;
  const int group = halves ? wave >> 1 : wave;
  const bool active = group * 32 < rows;
  const int row = group * 32 + col;                    // of the tile
  const int tok = (it.tile * kRows + row) / a.G;       // the row's token
  const int head = kvh * a.G + (it.tile * kRows + row) % a.G;
  const int base = it.s.ctx - it.s.q_len;
  const bool real = row < rows;
  const int pos = base + tok;
  const int first_pos = base + (it.tile * kRows + group * 32) / a.G;
  const int last_pos = base + (it.tile * kRows + min(rows, group * 32 + 32) - 1) / a.G;

  typename T::v8 q[KK];
  {
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + (long long)(it.s.row0 + (real ? tok : 0)) * a.q_n +
                          (long long)(real ? head : 0) * a.q_h;
    const uint32_t flip = a.q_sign < 0 ? 0x80008000u : 0u;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const int d = kk * 16 + half * 8;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (real && active && a.q_sign)
        x = load16(reinterpret_cast<const uint8_t*>(src + d), (a.D - d) * 2, a.q_aligned);
      q[kk] = __builtin_bit_cast(typename T::v8, make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip));
    }
  }

  f32x16 o[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) o[n] = f32x16{};
  float m = -INFINITY, l = 0.f;

  // --- staging -------------------------------------------------------------
  const uint8_t* const k_base = a.pool + a.layer_off + (long long)kvh * a.g.head;
  const uint8_t* const v_base = k_base + a.g.kv;
  const int row_bytes = QUANT ? a.D : 2 * a.D;
  const int32_t* const table = a.table + (long long)it.b * a.max_pp;

  const auto page_of = [&](int block) {  // wavefront 0: the page of token `lane` of a block
    const int t = block * TN + lane;
    return block < to && t < it.s.ctx ? table[page_index(a, t)] : -1;
  };
  const auto put_places = [&](int block, int page) {
    const int t = block * TN + lane;
    const bool there = page >= 0 && page < a.P;
    const int slot = t - page_index(a, t) * a.PS;
    place_lds[block & 3][lane] = there ? (long long)page * a.g.page + (long long)slot * row_bytes : -1;
    const unsigned long long mask = __ballot(there);
    if (lane == 0) there_lds[block & 3] = mask;
  };
  uint4 kr[NP], vr[NP];
  float ksc = 0.f, vsc = 0.f;
  const auto load_tile = [&](int block) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = tid + i * kChunkThreads;
      kr[i] = vr[i] = make_uint4(0, 0, 0, 0);
      if (Tile::kRagged && c >= Tile::kAll) continue;
      const int t = c / Tile::kPerRow, w = c % Tile::kPerRow;
      const long long at = place_lds[block & 3][t];
      if (at >= 0) kr[i] = load16(k_base + at + w * 16, row_bytes - w * 16, a.aligned);
      if constexpr (!QUANT) {
        if (at >= 0) vr[i] = load16(v_base + at + w * 16, row_bytes - w * 16, a.aligned);
      } else {  // V: four tokens' codes of a dim in a dword, 4 D bytes for the four tokens
        const int t4 = c / (DP / 4) * 4, w4 = c % (DP / 4);
        const long long at4 = place_lds[block & 3][t4];
        if (at4 >= 0 && w4 * 4 < a.D) vr[i] = load16(v_base + at4 + w4 * 16, 16, a.aligned);
      }
    }
  };
  const auto load_scales = [&](int block, int page) {  // wavefront 0, quantized pools
    ksc = vsc = 0.f;
    if (page >= 0 && page < a.P) {
      const int t = block * TN + lane;
      const float* s = a.scales + a.s_layer_off + (long long)page * a.g.s_page + (long long)kvh * a.g.s_head +
                       (KIND == kSrcI8 ? t - page_index(a, t) * a.PS : 0);
      ksc = s[0];
      vsc = s[a.g.s_kv];
    }
  };
  const auto put_tile = [&](int block) {
    const unsigned long long there = there_lds[block & 3];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = tid + i * kChunkThreads;
      if (Tile::kRagged && c >= Tile::kAll) continue;
      const int t = c / Tile::kPerRow, w = c % Tile::kPerRow;
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
        const int quad = c / (DP / 4), w4 = c % (DP / 4);
        const uint32_t bits = (uint32_t)(there >> (4 * quad)) & 15u;
        const uint32_t keep = ((bits & 1) * 0xffu) | ((bits >> 1 & 1) * 0xff00u) | ((bits >> 2 & 1) * 0xff0000u) |
                              ((bits >> 3) * 0xff000000u);
        const int nd = a.D >> 4;
        int d0 = w4 * 4 / nd, d1 = w4 * 4 % nd;
        uint8_t* vt = v_lds + ((quad >> 2) * 2 + (quad & 1)) * DP * 16 + (quad >> 1 & 1) * 8;
        const uint32_t words[4] = {vr[i].x, vr[i].y, vr[i].z, vr[i].w};
        if (w4 * 4 < a.D) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            *reinterpret_cast<uint2*>(vt + (d0 + 16 * d1) * 16) = codes4<Bf16, KIND>(words[j] & keep);
            if (++d1 == nd) d1 = 0, ++d0;
          }
        }
      }
    }
    if (QUANT && wave == 0) {
      scale_lds[0][lane] = ksc;
      scale_lds[1][lane] = vsc;
    }
  };

  // --- one block's NS x 32 tokens from sub st0 -----------------------------
  const auto compute = [&](int block, auto ns, int st0) {
    constexpr int NS = decltype(ns)::value;
    const int t0 = block * TN + st0 * 32;
    if (a.causal && t0 > last_pos) return;
    if (a.window && t0 + NS * 32 - 1 <= first_pos - a.window) return;
    f32x16 s[NS];
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
    if constexpr (QUANT) {
#pragma unroll
      for (int u = 0; u < NS; ++u)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const float4 x = *reinterpret_cast<const float4*>(&scale_lds[0][(st0 + u) * 32 + 2 * i + 4 * half]);
          s[u][i] *= x.x, s[u][i + 1] *= x.y, s[u][i + 2] *= x.z, s[u][i + 3] *= x.w;
        }
    }
    const unsigned long long there = there_lds[block & 3];
    const bool mask = there != ~0ull || (a.causal && t0 + NS * 32 - 1 > first_pos) ||
                      (a.window && t0 <= last_pos - a.window);
    if (mask) {
      const int hi = (a.causal ? min(pos, it.s.ctx - 1) : it.s.ctx - 1) - t0 - 4 * half;
      const int lo = a.window ? pos - a.window - t0 - 4 * half : -0x40000000;
#pragma unroll
      for (int u = 0; u < NS; ++u) {
        const uint32_t bits = (uint32_t)(there >> (32 * (st0 + u))) >> (4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int t = 8 * (i / 4) + i % 4;
          const bool ok = 32 * u + t <= hi && 32 * u + t > lo && (bits >> t & 1);
          s[u][i] = ok ? s[u][i] : -INFINITY;
        }
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int u = 0; u < NS; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
    top = xor_max<32>(top) * a.sc;
    // The maximum moves only when it would leave weights above 2^8: the
    // accumulators are rescaled a few times per row, not per block.
    if (__any(top > m + 8.f)) {
      const float next = fmaxf(m, top);
      const float f = next == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - next);
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[n][i] *= f;
      l *= f;
      m = next;
    }
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
        if constexpr (QUANT) {
          const float* vs = &scale_lds[1][(st0 + u) * 32 + 16 * e + 4 * half];
          const float4 x = *reinterpret_cast<const float4*>(vs), y = *reinterpret_cast<const float4*>(vs + 8);
          p[0] *= x.x, p[1] *= x.y, p[2] *= x.z, p[3] *= x.w;
          p[4] *= y.x, p[5] *= y.y, p[6] *= y.z, p[7] *= y.w;
        }
        const auto pb = __builtin_convertvector(p, typename PT::v8);
        typename PT::v8 low;
        if constexpr (SPLIT_P) low = __builtin_convertvector(p - __builtin_convertvector(pb, f32x8), typename PT::v8);
        const int step = (st0 + u) * 2 + e;  // of 16 tokens
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          typename PT::v8 v;
          if constexpr (QUANT) {
            v = __builtin_bit_cast(typename PT::v8, *reinterpret_cast<const uint4*>(
                                                        v_lds + ((step * 2 + half) * DP + n * 32 + col) * 16));
          } else {
            typedef __attribute__((address_space(3))) s16x4* lds_t;
            const uint8_t* x = v_lds + (step * 16 + 4 * half + ((lane & 15) >> 2)) * Tile::kVStride +
                               (n * 32 + (lane & 16) + (lane & 3) * 4) * 2;
            const s16x4 r0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)x);
            const s16x4 r1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(x + 8 * Tile::kVStride));
            typedef short s16x8 __attribute__((ext_vector_type(8)));
            v = __builtin_bit_cast(typename PT::v8, __builtin_shufflevector(r0, r1, 0, 1, 2, 3, 4, 5, 6, 7));
          }
          o[n] = PT::mfma(v, pb, o[n]);
          if constexpr (SPLIT_P) o[n] = PT::mfma(v, low, o[n]);
        }
      }
  };

  // --- the item's blocks ---------------------------------------------------
  int page1 = -1, page2 = -1;  // wavefront 0: pages of the next block and the one after
  if (wave == 0) {
    const int page0 = page_of(from);
    page1 = page_of(from + 1);
    page2 = page_of(from + 2);
    put_places(from, page0);
    put_places(from + 1, page1);
    if (QUANT) load_scales(from, page0);
  }
  __syncthreads();
  if (from < to) load_tile(from);
  for (int block = from; block < to; ++block) {
    __syncthreads();  // the block before is computed
    put_tile(block);
    if (wave == 0) put_places(block + 2, page2);
    __syncthreads();
    if (block + 1 < to) load_tile(block + 1);
    if (wave == 0) {
      if (QUANT) load_scales(block + 1, page1);
      page1 = page2;
      page2 = page_of(block + 3);
    }
    if (active) {
      if (halves)
        compute(block, std::integral_constant<int, 1>{}, wave & 1);
      else
        compute(block, std::integral_constant<int, 2>{}, 0);
    }
  }

  // --- results -------------------------------------------------------------
  l = xor_add<32>(l);
  if (halves) {  // the two halves of a row group, joined in LDS
    __syncthreads();
    float* x = reinterpret_cast<float*>(tile_lds) + group * (NB * 16 + 2) * 64 + lane;
    if (active && (wave & 1)) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[(n * 16 + i) * 64] = o[n][i];
      x[NB * 16 * 64] = m;
      x[(NB * 16 + 1) * 64] = l;
    }
    __syncthreads();
    if (!active || (wave & 1)) return;
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
  if (!active || !real) return;
  if (it.shares > 1) {
    const long long slot = (long long)blockIdx.x * kRows + row;
    float* dst = a.part + slot * DP;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<float4*>(dst + n * 32 + 2 * i + 4 * half) =
            make_float4(o[n][i], o[n][i + 1], o[n][i + 2], o[n][i + 3]);
    if (half == 0) a.ml[slot] = make_float2(m, l);
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const long long at = (long long)(it.s.row0 + tok) * a.H + head;
  uint16_t* dst = static_cast<uint16_t*>(a.out) + at * a.D;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int d = n * 32 + 2 * i + 4 * half;
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

template <typename T, int KIND>
void launch_chunk16_t(const ChunkArgs& a, dim3 grid, hipStream_t st) {
  if (a.dp == 64)
    hipLaunchKernelGGL((chunk_attn_kernel<T, KIND, 64>), grid, dim3(kChunkThreads), 0, st, a);
  else if (a.dp == 96)
    hipLaunchKernelGGL((chunk_attn_kernel<T, KIND, 96>), grid, dim3(kChunkThreads), 0, st, a);
  else if (a.dp == 128)
    hipLaunchKernelGGL((chunk_attn_kernel<T, KIND, 128>), grid, dim3(kChunkThreads), 0, st, a);
  else
    hipLaunchKernelGGL((chunk_attn_kernel<T, KIND, 256>), grid, dim3(kChunkThreads), 0, st, a);
}

}  // namespace
}  // namespace vrm
