// Attention of a chunk over a paged cache with float32 products: float32
// queries or pools, and 16-bit queries over a pool of the other 16-bit type.
//
// The same pass as chunk_attn_kernel (vrm_chunk16.h), on
// v_mfma_f32_32x32x2_f32: nothing is rounded below float32 before the output.
// A block is 32 tokens, converted to float32 on its way into LDS (int8 and
// e4m3 codes exactly, their scales multiplying scores and weights).  The
// k-slots of a matrix product may come in any order that both operands
// share: lane half h takes dims 8 j + 4 h + e of K and Q (16-byte LDS reads),
// and tokens in the order the scores lie in.
// Bound: the float32 matrix rate, 1/16 of the 16-bit one, in long batches;
// four prompts' chunks of 100 to 160 tokens, 12 heads of 64, are a chain of
// dependent blocks: 35 us with the merge, 20 TFLOP/s.
#include <type_traits>

#include "vrm_chunk.h"

namespace vrm {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int KIND>
constexpr int kPieceElems = KIND == kSrcF32 ? 4 : KIND >= kSrcI8 ? 16 : 8;  // of 16 bytes

template <int KIND>
__device__ __forceinline__ void widen(const uint4& x, float (&f)[kPieceElems<KIND>]) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < kPieceElems<KIND>; ++i) {
    if constexpr (KIND == kSrcF32) f[i] = __uint_as_float(w[i]);
    if constexpr (KIND == kSrcF16) f[i] = f16_bits_to_f32(w[i / 2] >> (16 * (i & 1)) & 0xffffu);
    if constexpr (KIND == kSrcBf16) f[i] = bf16_bits_to_f32(w[i / 2] >> (16 * (i & 1)) & 0xffffu);
    if constexpr (KIND == kSrcI8) f[i] = (float)(int8_t)(w[i / 4] >> (8 * (i & 3)));
    if constexpr (KIND == kSrcFp8) f[i] = e4m3fn_to_f32(w[i / 4] >> (8 * (i & 3)) & 0xffu);
  }
}

__device__ __forceinline__ void store_out(const ChunkArgs& a, long long at, float x) {
  if (a.q_type == VRM_SRC_F32)
    static_cast<float*>(a.out)[at] = x;
  else if (a.q_type == VRM_SRC_F16)
    static_cast<uint16_t*>(a.out)[at] = __builtin_bit_cast(unsigned short, (_Float16)x);
  else
    static_cast<uint16_t*>(a.out)[at] = __builtin_bit_cast(unsigned short, (__bf16)x);
}

template <int KIND, int DP>
__global__ void __launch_bounds__(kChunkThreads, DP <= 128 ? 2 : 1) chunk_attn_f32_kernel(ChunkArgs a) {
  constexpr bool QUANT = KIND >= kSrcI8;
  constexpr int TN = 32, NB = DP / 32, E = kPieceElems<KIND>;
  // a half's 32 lanes read 32 dims of one token, the other half's of the
  // token four rows on: 4 (DP + 8) = 32 mod 64 banks apart
  constexpr int KS = DP + 4, VS = DP + 8;
  constexpr int kPieces = TN * DP / E, NP = (kPieces + kChunkThreads - 1) / kChunkThreads;
  __shared__ __align__(16) float k_lds[TN * KS];
  __shared__ __align__(16) float v_lds[TN * VS];
  __shared__ float scale_lds[2][TN];
  __shared__ long long place_lds[4][TN];
  __shared__ uint32_t there_lds[4];

  const int kvh = blockIdx.x % a.KH;
  Item it;
  if (!find_item<TN>(a, blockIdx.x / a.KH, it)) return;
  int from, to;
  item_blocks<TN>(a, it, from, to);
  put_record(a, it, kvh);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int rows = min(a.tile_rows, it.s.q_len * a.G - it.tile * a.tile_rows);
  const bool active = wave * 32 < rows;
  const RowGroup g = row_group(a, it, kvh, rows, wave * 32);
  const bool real = g.real;

  float q[DP / 2];
  {
    const long long at = (long long)(it.s.row0 + (real ? g.tok : 0)) * a.q_n + (long long)(real ? g.head : 0) * a.q_h;
#pragma unroll
    for (int j = 0; j < DP / 2; ++j) {
      const int d = j / 4 * 8 + half * 4 + j % 4;
      const float x = real && active && a.q_sign && d < a.D ? load_q(a, at + d) : 0.f;
      q[j] = a.q_sign < 0 ? -x : x;
    }
  }
  f32x16 o[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) o[n] = f32x16{};
  float m = -INFINITY, l = 0.f;

  const uint8_t* const k_base = a.pool + a.layer_off + (long long)kvh * a.g.head;
  const uint8_t* const v_base = k_base + a.g.kv;
  const int row_bytes = KIND == kSrcF32 ? 4 * a.D : QUANT ? a.D : 2 * a.D;
  const int32_t* const table = a.table + (long long)it.b * a.max_pp;

  // lanes 0 .. 31 of wavefront 0: token `lane` of a block
  const auto page_of = [&](int block) {
    const int t = block * TN + lane;
    return lane < TN && block < to && t < it.s.ctx ? table[page_index(a, t)] : -1;
  };
  const auto put_places = [&](int block, int page) {
    const int t = block * TN + lane;
    const bool there = page >= 0 && page < a.P;
    const int slot = t - page_index(a, t) * a.PS;
    if (lane < TN) place_lds[block & 3][lane] = there ? (long long)page * a.g.page + (long long)slot * row_bytes : -1;
    const uint32_t mask = (uint32_t)__ballot(there);
    if (lane == 0) there_lds[block & 3] = mask;
  };
  // dims D .. DP - 1 of V, which no code is staged for, are zeros (any_nan looks at all)
  if (QUANT && a.D < DP) {
    const int pad = DP - a.D;
    for (int i = tid; i < TN * pad; i += kChunkThreads) v_lds[i / pad * VS + a.D + i % pad] = 0.f;
  }
  uint4 kr[NP], vr[NP];
  float ksc = 0.f, vsc = 0.f;
  constexpr int kPerRow = DP / E;
  const auto load_tile = [&](int block) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = tid + i * kChunkThreads;
      kr[i] = vr[i] = make_uint4(0, 0, 0, 0);
      if (c >= kPieces) continue;
      const int t = c / kPerRow, w = c % kPerRow;
      const long long at = place_lds[block & 3][t];
      if (at >= 0) kr[i] = load16(k_base + at + w * 16, row_bytes - w * 16, a.aligned);
      if constexpr (!QUANT) {
        if (at >= 0) vr[i] = load16(v_base + at + w * 16, row_bytes - w * 16, a.aligned);
      } else {
        const int t4 = c / (DP / 4) * 4, w4 = c % (DP / 4);
        const long long at4 = place_lds[block & 3][t4];
        if (at4 >= 0 && w4 * 4 < a.D) vr[i] = load16(v_base + at4 + w4 * 16, 16, a.aligned);
      }
    }
  };
  const auto load_scales = [&](int block, int page) {
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
    const uint32_t there = there_lds[block & 3];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = tid + i * kChunkThreads;
      if (c >= kPieces) continue;
      const int t = c / kPerRow, w = c % kPerRow;
      float f[E];
      widen<KIND>(kr[i], f);
#pragma unroll
      for (int e = 0; e < E; e += 4)
        *reinterpret_cast<float4*>(&k_lds[t * KS + w * E + e]) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
      widen<KIND>(vr[i], f);
      if constexpr (!QUANT) {
#pragma unroll
        for (int e = 0; e < E; e += 4)
          *reinterpret_cast<float4*>(&v_lds[t * VS + w * E + e]) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
      } else {
        const int quad = c / (DP / 4), w4 = c % (DP / 4);
        const int nd = a.D >> 4;
        int d0 = w4 * 4 / nd, d1 = w4 * 4 % nd;
        if (w4 * 4 < a.D) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              v_lds[(quad * 4 + e) * VS + d0 + 16 * d1] = there >> (quad * 4 + e) & 1 ? f[4 * j + e] : 0.f;
            if (++d1 == nd) d1 = 0, ++d0;
          }
        }
      }
    }
    if (QUANT && wave == 0 && lane < TN) {
      scale_lds[0][lane] = ksc;
      scale_lds[1][lane] = vsc;
    }
  };

  const auto compute = [&](int block) {
    const int t0 = block * TN;
    if (a.causal && t0 > g.last_pos) return;
    if (a.window && t0 + TN - 1 <= g.first_pos - a.window) return;
    f32x16 s{};
#pragma unroll
    for (int j = 0; j < DP / 8; ++j) {
      const float4 x = *reinterpret_cast<const float4*>(&k_lds[col * KS + j * 8 + half * 4]);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.x, q[4 * j], s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.y, q[4 * j + 1], s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.z, q[4 * j + 2], s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.w, q[4 * j + 3], s, 0, 0, 0);
    }
    if constexpr (QUANT) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] *= scale_lds[0][i / 4 * 8 + 4 * half + i % 4];
    }
    const uint32_t there = there_lds[block & 3];
    if (there != ~0u || (a.causal && t0 + TN - 1 > g.first_pos) || (a.window && t0 <= g.last_pos - a.window)) {
      const int hi = (a.causal ? min(g.pos, it.s.ctx - 1) : it.s.ctx - 1) - t0 - 4 * half;
      const int lo = a.window ? g.pos - a.window - t0 - 4 * half : -0x40000000;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int t = 8 * (i / 4) + i % 4;
        const bool ok = t <= hi && t > lo && (there >> (4 * half) >> t & 1);
        s[i] = ok ? s[i] : -INFINITY;
      }
    }
    float top = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
    top = xor_max<32>(top) * a.sc;
    if (__any(top > m + 8.f)) {
      const float next = fmaxf(m, top);
      const float f = next == -INFINITY ? 1.f : exp2f(m - next);
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[n][i] *= f;
      l *= f;
      m = next;
    }
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.sc, -ref));
      l += s[i];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int t = i / 4 * 8 + 4 * half + i % 4;
      const float p = QUANT ? s[i] * scale_lds[1][t] : s[i];
#pragma unroll
      for (int n = 0; n < NB; ++n)
        o[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(v_lds[t * VS + n * 32 + col], p, o[n], 0, 0, 0);
    }
  };

  int page1 = -1, page2 = -1;
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
    __syncthreads();
    put_tile(block);
    if (wave == 0) put_places(block + 2, page2);
    __syncthreads();
    if (block + 1 < to) load_tile(block + 1);
    if (wave == 0) {
      if (QUANT) load_scales(block + 1, page1);
      page1 = page2;
      page2 = page_of(block + 3);
    }
    if (active) compute(block);
  }

  l = xor_add<32>(l);
  if (!active) return;
  if (__builtin_expect(any_nan(o, real), 0) &&
      careful_rows<TN>(a, it, kvh, KIND, wave * 32, min(rows, wave * 32 + 32), g.first_pos, g.last_pos, from, to))
    return;
  if (!real) return;
  if (it.shares > 1) {
    const long long slot = (long long)blockIdx.x * a.tile_rows + g.row;
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
  const long long at = (long long)(it.s.row0 + g.tok) * a.H + g.head;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int d = n * 32 + 8 * (i / 4) + 4 * half + i % 4;
      if (d < a.D) store_out(a, at * a.D + d, l == 0.f ? 0.f : o[n][i] / l);
    }
  if (a.lse && half == 0) a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

template <int KIND>
void launch_f32(const ChunkArgs& a, dim3 grid, hipStream_t st) {
  if (a.dp == 64)
    hipLaunchKernelGGL((chunk_attn_f32_kernel<KIND, 64>), grid, dim3(kChunkThreads), 0, st, a);
  else if (a.dp == 128)
    hipLaunchKernelGGL((chunk_attn_f32_kernel<KIND, 128>), grid, dim3(kChunkThreads), 0, st, a);
  else
    hipLaunchKernelGGL((chunk_attn_f32_kernel<KIND, 256>), grid, dim3(kChunkThreads), 0, st, a);
}

}  // namespace

void launch_chunk_f32(const ChunkArgs& a, int kind, dim3 grid, hipStream_t st) {
  switch (kind) {
    case kSrcF32: launch_f32<kSrcF32>(a, grid, st); break;
    case kSrcF16: launch_f32<kSrcF16>(a, grid, st); break;
    case kSrcBf16: launch_f32<kSrcBf16>(a, grid, st); break;
    case kSrcI8: launch_f32<kSrcI8>(a, grid, st); break;
    default: launch_f32<kSrcFp8>(a, grid, st); break;
  }
}

}  // namespace vrm
