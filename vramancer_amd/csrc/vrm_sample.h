// Weights of the tokens of a row of logits, in 64 bits, as the kernels that
// draw and verify tokens share them (vrm_sample.hip, vrm_sample_cut.hip).
//
// A row's token i has weight w_i = 2^((l_i - m) c), c = log2(e) / T, m the
// row's maximum; the probability is w_i over their sum.  A token is an answer
// in whole numbers that follows running sums over up to 10^5 weights next to
// borders, so that an error of 1e-7 in each weight would change one in some
// thousand draws from flat rows.  Weights are therefore float64: a conversion,
// a subtraction, a product and a polynomial of 10 steps, on a vector unit whose
// float64 rate is its float32 rate.  Logits that are -inf or NaN weigh nothing.
#pragma once
#include "vrm_common.h"

namespace vrm {

constexpr int kSampleThreads = 256;
constexpr int kSamplePer = 32;                               // logits of a thread in a chunk
constexpr int kSampleChunk = kSampleThreads * kSamplePer;    // logits of a chunk

// Rows of logits and the parameters of the sequence they belong to.  Sequence
// b has rows cu[b] .. cu[b + 1] (K + 1 each without cu), of which the first
// K + 1 count; slot b (K + 1) + i stands for its row i.
struct SampleRows {
  const void* logits;
  long long stride;  // elements from a row to the next
  const int32_t* cu;
  int N, B, K, V;
  const float* temperature;
  float temperature_all;
  const int32_t* top_k;
  int top_k_all;
  const float* top_p;
  float top_p_all;

  __device__ __forceinline__ int first(int b) const { return cu ? clamp_int(cu[b], 0, N) : b * (K + 1); }
  __device__ __forceinline__ int count(int b) const {
    return cu ? min(max(clamp_int(cu[b + 1], 0, N) - first(b), 0), K + 1) : K + 1;
  }
  __device__ __forceinline__ float temp(int b) const { return temperature ? temperature[b] : temperature_all; }
  __device__ __forceinline__ int limit(int b) const { return top_k ? top_k[b] : top_k_all; }
  __device__ __forceinline__ float nucleus(int b) const { return top_p ? top_p[b] : top_p_all; }
};

// What a chunk of a row says about it: its maximum, that one's first place,
// and the sum of its weights relative to it.
struct ChunkRec {
  double sum;
  float top;
  int arg;
};

// Which tokens of a row stay (those whose order value is at least `cut`) and
// the sum of their weights.
struct RowCut {
  unsigned long long cut;
  double sum;
};

// A sequence's draw: the row it draws from, with the row's scale, and the
// drafted token that is refused (-1: none), whose place in the drafts is `at`.
struct DrawRec {
  double c;                // 0 with greedy
  double sum;              // of the row's weights that stay
  unsigned long long cut;
  float top;
  int row;                 // -1: the sequence has none
  int arg;                 // greedy: the answer; otherwise -2
  int refused;
  int at;
  int pad;
};

__device__ __forceinline__ double sample_scale(float t) { return 1.4426950408889634074 / (double)t; }

// 2^y for y <= 0, to 6e-16 of the value: y = n + r, 2^r = 1 + r q(r) with q
// interpolated at Chebyshev nodes of [-1/2, 1/2]; exactly 1 at 0.
__device__ __forceinline__ double exp2_neg(double y) {
  const double big = y + 6755399441055744.0;  // 1.5 2^52: the sum's last digits are the nearest integer
  const double r = y - (big - 6755399441055744.0);
  double q = 0x1.e5e9f548e5725p-28;
  q = fma(q, r, 0x1.b6571de2f2351p-24);
  q = fma(q, r, 0x1.62bfe46117445p-20);
  q = fma(q, r, 0x1.ffcb76789860fp-17);
  q = fma(q, r, 0x1.4309130378460p-13);
  q = fma(q, r, 0x1.5d87fe908f88ap-10);
  q = fma(q, r, 0x1.3b2ab6fba385fp-7);
  q = fma(q, r, 0x1.c6b08d7044119p-5);
  q = fma(q, r, 0x1.ebfbdff82c590p-3);
  q = fma(q, r, 0x1.62e42fefa39f7p-1);
  return __builtin_ldexp(fma(q, r, 1.0), (int)__double_as_longlong(big));
}

// Weight of a logit against the row's maximum.  A NaN (of the logit, of
// inf - inf) is taken as the lower bound by the maximum and weighs nothing;
// rows whose maximum is +inf weigh their +inf alone.
__device__ __forceinline__ double sample_weight(float l, float top, double c) {
  if (top == INFINITY) return l == INFINITY ? 1.0 : 0.0;
  return exp2_neg(fmax(((double)l - (double)top) * c, -1100.0));
}

// Order value of token i: larger for what comes first (larger logit, then
// lower index), never 0.  -0 and +0 are equal.
__device__ __forceinline__ uint32_t logit_key(float l) {
  const uint32_t u = __float_as_uint(l + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long order_value(float l, int i) {
  return ((unsigned long long)logit_key(l) << 32) | (uint32_t)~i;
}

template <int SRC>
struct Logit;  // element type of a row
template <>
struct Logit<VRM_SRC_F32> {
  using Raw = uint32_t;
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float value(uint32_t u) { return __uint_as_float(u); }
};
template <>
struct Logit<VRM_SRC_F16> {
  using Raw = uint16_t;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float value(uint16_t u) { return f16_bits_to_f32(u); }
};
template <>
struct Logit<VRM_SRC_BF16> {
  using Raw = uint16_t;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float value(uint16_t u) { return bf16_bits_to_f32(u); }
};

// 16 bytes from an address that is aligned to its elements only: rows of odd
// vocabularies start anywhere.
template <typename Raw>
struct __attribute__((packed, aligned(sizeof(Raw)))) Unaligned16 {
  Raw v[16 / sizeof(Raw)];
};

// Elements e0 .. e0 + kVec of a row of V, -inf past its end.
template <int SRC>
__device__ __forceinline__ void load_vec(const typename Logit<SRC>::Raw* row, int e0, int V, float* x) {
  using L = Logit<SRC>;
  if (e0 + L::kVec <= V) {
    const auto raw = *reinterpret_cast<const Unaligned16<typename L::Raw>*>(row + e0);
#pragma unroll
    for (int e = 0; e < L::kVec; ++e) x[e] = L::value(raw.v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < L::kVec; ++e) x[e] = e0 + e < V ? L::value(row[e0 + e]) : -INFINITY;
  }
}

template <int SRC>
__device__ __forceinline__ const typename Logit<SRC>::Raw* row_at(const SampleRows& r, int row) {
  return static_cast<const typename Logit<SRC>::Raw*>(r.logits) + (long long)row * r.stride;
}

// A chunk's elements of this thread: vector i is elements (i 256 + tid) kVec ..
template <int SRC>
__device__ __forceinline__ void load_chunk(const typename Logit<SRC>::Raw* row, int chunk, int V, float* x) {
  constexpr int kVec = Logit<SRC>::kVec;
#pragma unroll
  for (int i = 0; i < kSamplePer / kVec; ++i)
    load_vec<SRC>(row, chunk * kSampleChunk + (i * kSampleThreads + (int)threadIdx.x) * kVec, V, x + i * kVec);
}

// Sums, largest and smallest values over a wavefront, every lane has them; the
// sums' order is fixed.
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) v += __shfl_xor(v, m);
  return v;
}
__device__ __forceinline__ double wave_prefix(double v) {  // inclusive
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) {
    const double o = __shfl_up(v, m);
    if ((int)(threadIdx.x & 63) >= m) v += o;
  }
  return v;
}
__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) v = min(v, __shfl_xor(v, m));
  return v;
}

// A row's maximum, the sum of its weights relative to it (scale c, 0 for
// greedy rows, whose sum is not asked for) and the maximum's first place, from
// its chunks; by one wavefront.
__device__ __forceinline__ void combine_chunks(const ChunkRec* rec, int nc, double c, float& top, double& sum, int& arg) {
  const int lane = threadIdx.x & 63;
  float m = -INFINITY;
  for (int j = lane; j < nc; j += kWave) m = fmaxf(m, rec[j].top);
  m = group_max<64>(m);
  double s = 0.0;
  int first = 0x7fffffff;
  for (int j = lane; j < nc; j += kWave) {
    const ChunkRec r = rec[j];
    if (r.top == m) first = min(first, r.arg);
    if (r.top > -INFINITY) s += r.sum * sample_weight(r.top, m, c);
  }
  top = m;
  sum = wave_sum(s);
  arg = wave_min(first);
}

int launch_sample_cut(const SampleRows& r, int dtype, int nc, const ChunkRec* rec, RowCut* cuts, hipStream_t st);

}  // namespace vrm
