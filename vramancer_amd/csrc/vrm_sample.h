// Weights of the tokens of a row of logits, in 64 bits, as the kernels that
// draw and verify tokens share them (vrm_sample.hip, vrm_sample_cut.hip).
//
// Token i of a row weighs w_i = 2^((l_i - max l) c), c = log2(e) / T; its
// probability is w_i over their sum.  A token is an answer in whole numbers
// that follows running sums over up to 10^5 weights next to borders, so that an
// error of 1e-7 in each weight would change one in some thousand draws from
// flat rows.  Weights are therefore float64, at 15 instructions each on a vector
// unit whose float64 rate is its float32 rate (4.7 to 5.6 cycles a wavefront's
// instruction, float32 4.0 to 4.4).  The largest weight is exactly 1, so that
// draws from tokens that are all equal to it are exact where their number times
// the random number is whole.  Logits that are -inf or NaN weigh nothing.
#pragma once
#include "vrm_common.h"

namespace vrm {

constexpr int kSampleThreads = 256;
constexpr int kSamplePer = 32;                     // logits of a lane in a segment
constexpr int kSegment = kWave * kSamplePer;       // logits of a wavefront
constexpr int kSampleBlock = 4 * kSegment;         // of a workgroup

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
  __host__ __device__ __forceinline__ int segments() const { return (V + kSegment - 1) / kSegment; }
};

// What a segment of a row says about it: a maximum (of the segment or of some
// more of the row around it), that one's first place, and the sum of the
// segment's weights by the scale of that maximum.
struct SegRec {
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

// A sequence's draw: the row it draws from, and the drafted token that is
// refused (-1: none), whose place in the drafts is `at`.
struct DrawRec {
  double sum;              // of the row's weights that stay
  unsigned long long cut;
  float top;
  int row;                 // -1: the sequence has none
  int arg;                 // the answer where it is known (greedy, no token); otherwise -2
  int refused;
  int at;
  int pad;
};

// The scale of a row, or of a part of one.
struct Scale {
  double top, c, low;  // low: a difference from top at which the weight is 0
  bool infinite;       // the maximum is +inf: those tokens alone
};

__device__ __forceinline__ Scale make_scale(float top, float t) {
  Scale s;
  s.infinite = top == INFINITY;
  s.top = top;
  s.c = fmax(1.4426950408889634074 / (double)t, 1e-290);  // (an infinite temperature: every weight is 1)
  s.low = -1100.0 / s.c;
  return s;
}

// Weights of N logits.  (l - top) c = n + r; 2^r = 1 + r q(r) with q
// interpolated at 8 Chebyshev nodes of [-1/2, 1/2], to 2.2e-12 of the value
// (the same for equal logits).  n comes out of an addition at 2^52, r of the
// same product again.  A NaN (of the logit, of -inf against -inf) is taken as
// the lower bound by fmax.
// The polynomial's steps, four values side by side, are written out with their
// coefficients in scalar registers: the compiler takes the form of the
// instruction that adds onto its result, and copies each coefficient into
// vector registers first, two instructions more for each step (the sums of 960
// rows of 131072 took 123 us with them).
template <int N>
__device__ __forceinline__ void sample_weights(const float* l, const Scale& s, double* w) {
  static_assert(N % 4 == 0, "four values side by side");
  if (s.infinite) {
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = l[e] == INFINITY ? 1.0 : 0.0;
    return;
  }
  constexpr double kBig = 6755399441055744.0;  // 1.5 2^52: a sum's last digits are the nearest integer
#pragma unroll
  for (int e = 0; e < N; e += 4) {
    double r[4], q[4];
    int n[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const double x = fmax((double)l[e + i] - s.top, s.low);
      const double big = fma(x, s.c, kBig);
      n[i] = (int)__double_as_longlong(big);
      r[i] = fma(x, s.c, -(big - kBig));
    }
#define VRM_STEP(c)                          \
  "v_fma_f64 %0, %0, %4, " c "\n\t"          \
  "v_fma_f64 %1, %1, %5, " c "\n\t"          \
  "v_fma_f64 %2, %2, %6, " c "\n\t"          \
  "v_fma_f64 %3, %3, %7, " c "\n\t"
    asm("v_fma_f64 %0, %15, %4, %8\n\t"
        "v_fma_f64 %1, %15, %5, %8\n\t"
        "v_fma_f64 %2, %15, %6, %8\n\t"
        "v_fma_f64 %3, %15, %7, %8\n\t" VRM_STEP("%9") VRM_STEP("%10") VRM_STEP("%11") VRM_STEP("%12")
            VRM_STEP("%13") VRM_STEP("%14") VRM_STEP("1.0")
        : "=&v"(q[0]), "=&v"(q[1]), "=&v"(q[2]), "=&v"(q[3])
        : "v"(r[0]), "v"(r[1]), "v"(r[2]), "v"(r[3]), "s"(0x1.00c0e4e15189cp-16), "s"(0x1.4308c7183d6a2p-13),
          "s"(0x1.5d877598350dep-10), "s"(0x1.3b2ab70ad2565p-7), "s"(0x1.c6b08da70cce3p-5),
          "s"(0x1.ebfbdff82a734p-3), "s"(0x1.62e42fef9cc69p-1), "v"(0x1.63b2d7971923fp-20));
#undef VRM_STEP
#pragma unroll
    for (int i = 0; i < 4; ++i) w[e + i] = __builtin_ldexp(q[i], n[i]);
  }
}
// The same for one logit, to the same bits (the steps are the same).
__device__ __forceinline__ double sample_weight(float l, const Scale& s) {
  if (s.infinite) return l == INFINITY ? 1.0 : 0.0;
  constexpr double kBig = 6755399441055744.0;
  const double x = fmax((double)l - s.top, s.low);
  const double big = fma(x, s.c, kBig);
  const double r = fma(x, s.c, -(big - kBig));
  double q = fma(0x1.63b2d7971923fp-20, r, 0x1.00c0e4e15189cp-16);
  q = fma(q, r, 0x1.4308c7183d6a2p-13);
  q = fma(q, r, 0x1.5d877598350dep-10);
  q = fma(q, r, 0x1.3b2ab70ad2565p-7);
  q = fma(q, r, 0x1.c6b08da70cce3p-5);
  q = fma(q, r, 0x1.ebfbdff82a734p-3);
  q = fma(q, r, 0x1.62e42fef9cc69p-1);
  return __builtin_ldexp(fma(q, r, 1.0), (int)__double_as_longlong(big));
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

__device__ __forceinline__ float order_logit(unsigned long long order) {
  const uint32_t key = (uint32_t)(order >> 32);
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

template <int SRC>
struct Logit;  // element type of a row
template <>
struct Logit<VRM_SRC_F32> {
  using Raw = uint32_t;
  static constexpr int kVec = 4, kZeros = 0;  // (last bits that are 0 in every value as float32)
  static constexpr Raw kMinus = 0xff800000u;  // -inf
  static __device__ __forceinline__ float value(uint32_t u) { return __uint_as_float(u); }
};
template <>
struct Logit<VRM_SRC_F16> {
  using Raw = uint16_t;
  static constexpr int kVec = 8, kZeros = 13;
  static constexpr Raw kMinus = 0xfc00;  // -inf
  static __device__ __forceinline__ float value(uint16_t u) { return f16_bits_to_f32(u); }
};
template <>
struct Logit<VRM_SRC_BF16> {
  using Raw = uint16_t;
  static constexpr int kVec = 8, kZeros = 16;
  static constexpr Raw kMinus = 0xff80;  // -inf
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

// The first element of a lane's vector i of a segment; a wavefront's load is
// 1 KB without a gap.
template <int SRC>
__device__ __forceinline__ int segment_element(int seg, int i) {
  return seg * kSegment + (i * kWave + (int)(threadIdx.x & 63)) * Logit<SRC>::kVec;
}

// A lane's elements of a segment.  All loads of a whole segment are under way
// before the first is waited for.
template <int SRC>
__device__ __forceinline__ void load_segment(const typename Logit<SRC>::Raw* row, int seg, int V, float* x) {
  using L = Logit<SRC>;
  constexpr int kVec = L::kVec, kGroups = kSamplePer / kVec;
  const int e0 = segment_element<SRC>(seg, 0);
  if ((seg + 1) * kSegment <= V) {
    Unaligned16<typename L::Raw> raw[kGroups];
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
      raw[i] = *reinterpret_cast<const Unaligned16<typename L::Raw>*>(row + e0 + i * kWave * kVec);
#pragma unroll
    for (int i = 0; i < kSamplePer; ++i) x[i] = L::value(raw[i / kVec].v[i % kVec]);
  } else {
#pragma unroll
    for (int i = 0; i < kSamplePer; ++i) {
      const int e = e0 + (i / kVec) * kWave * kVec + i % kVec;
      x[i] = e < V ? L::value(row[e]) : -INFINITY;
    }
  }
}

// Prefixes over a wavefront on the vector ALU, and from them sums, largest and
// smallest values as scalars: within a row of 16 lanes, then from row to row.
// (Exchanges through the LDS unit answer after some 100 cycles, and 16
// wavefronts that all reduce wait for each other there: a bin of the cut took
// 12,000 cycles to find with them.)  The order of a sum is fixed.
template <typename T>
__device__ __forceinline__ T lane_value(T v, int lane) {  // lane: the same in all
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
  } else {
    const auto u = __builtin_bit_cast(unsigned long long, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
    return __builtin_bit_cast(T, ((unsigned long long)hi << 32) | lo);
  }
}

template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T lane_move(T v, T identity) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, identity),
                                                             __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
  } else {
    const auto u = __builtin_bit_cast(unsigned long long, v), i = __builtin_bit_cast(unsigned long long, identity);
    const uint32_t lo = __builtin_amdgcn_update_dpp((int)(uint32_t)i, (int)(uint32_t)u, CTRL, ROWS, 0xf, false);
    const uint32_t hi =
        __builtin_amdgcn_update_dpp((int)(uint32_t)(i >> 32), (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(T, ((unsigned long long)hi << 32) | lo);
  }
}

template <typename T, typename Op>
__device__ __forceinline__ T wave_scan(T v, T identity, Op op) {  // inclusive
  v = op(v, lane_move<0x111, 0xf>(v, identity));  // row_shr 1, 2, 4, 8
  v = op(v, lane_move<0x112, 0xf>(v, identity));
  v = op(v, lane_move<0x114, 0xf>(v, identity));
  v = op(v, lane_move<0x118, 0xf>(v, identity));
  v = op(v, lane_move<0x142, 0xa>(v, identity));  // row_bcast 15 into rows 1 and 3
  v = op(v, lane_move<0x143, 0xc>(v, identity));  // row_bcast 31 into rows 2 and 3
  return v;
}
template <typename T>
__device__ __forceinline__ T wave_prefix(T v) {
  return wave_scan(v, T(0), [](T a, T b) { return a + b; });
}
template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
  return lane_value(wave_prefix(v), 63);
}
template <typename T>
__device__ __forceinline__ T wave_min(T v, T most) {
  return lane_value(wave_scan(v, most, [](T a, T b) { return a < b ? a : b; }), 63);
}
template <typename T>
__device__ __forceinline__ T wave_max(T v, T least) {
  return lane_value(wave_scan(v, least, [](T a, T b) { return a < b ? b : a; }), 63);
}

// A segment's sum by its row's scale.
__device__ __forceinline__ double segment_sum(const SegRec& r, const Scale& s) {
  return r.top > -INFINITY ? r.sum * sample_weight(r.top, s) : 0.0;
}

// A row from its segments, by one wavefront: its maximum, that one's first
// place (greedy rows), its scale and the sum of its weights (the others).
__device__ __forceinline__ void combine_segments(const SegRec* rec, int ns, float t, float& top, int& arg, Scale& scale,
                                                 double& sum) {
  const int lane = threadIdx.x & 63;
  float m = -INFINITY;
  for (int j = lane; j < ns; j += kWave) m = fmaxf(m, rec[j].top);
  top = wave_max(m, -INFINITY);
  arg = -1;
  sum = 0.0;
  if (top == -INFINITY) return;
  if (!(t > 0.0f)) {
    int first = 0x7fffffff;
    for (int j = lane; j < ns; j += kWave)
      if (rec[j].top == top) first = min(first, rec[j].arg);
    arg = wave_min(first, 0x7fffffff);
    sum = 1.0;
    return;
  }
  arg = -2;
  scale = make_scale(top, t);
  double s = 0.0;
  for (int j = lane; j < ns; j += kWave) s += segment_sum(rec[j], scale);
  sum = wave_sum(s);
}

// Probabilities e0 .. e0 + N of a row of V, 0 past its end.
template <int N>
__device__ __forceinline__ void load_probs(const float* q, int e0, int V, float* x) {
  if (e0 + N <= V) {
#pragma unroll
    for (int h = 0; h < N; h += 4) {
      const auto raw = *reinterpret_cast<const Unaligned16<uint32_t>*>(q + e0 + h);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[h + e] = __uint_as_float(raw.v[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = e0 + e < V ? q[e0 + e] : 0.0f;
  }
}

// What the tokens e0 .. e0 + N weigh in the draw: p, or where a draft was
// refused max(p - q, 0), in units of 1 / sum.
template <int N>
__device__ __forceinline__ void draw_weights(const DrawRec& w, const Scale& scale, const float* q, bool rest, int e0,
                                             int V, const float* x, double* out) {
  float qx[N];
  if (rest && q) load_probs<N>(q, e0, V, qx);
  bool in[N], any = true;
  if (w.cut) {
    any = false;
    const float border = order_logit(w.cut);
    const int last = (int)(uint32_t)~w.cut - e0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      in[e] = x[e] > border || (x[e] == border && e <= last);
      any |= in[e];
    }
  }
  if (!__any(any)) {  // (what is cut weighs nothing, and most wavefronts of a short list have nothing else)
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = 0.0;
    return;
  }
  sample_weights<N>(x, scale, out);
  if (w.cut) {
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = in[e] ? out[e] : 0.0;
  }
  if (rest) {
    if (q) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const double d = fma(-(double)(qx[e] < 0.0f ? 0.0f : qx[e]), w.sum, out[e]);
        out[e] = d > 0.0 ? d : 0.0;  // (nothing where q is NaN)
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (e0 + e == w.refused) out[e] = 0.0;
    }
  }
}

// *out: the token at which the running sum passes u of the whole, -1 without
// mass.  mass(j): the sum of segment j's weights.  By a workgroup of WAVES
// wavefronts: the first finds the segment, then each takes vectors of it, so
// that one load and one vector's code are waited for (16 rows of 32000: 7.7 us
// with one wavefront for all of it, 6.0 with four).
template <int SRC>
struct PickShared {
  double left, totals[kSamplePer / Logit<SRC>::kVec];
  int seg, rest;
};

template <int SRC, typename Mass>
__device__ __forceinline__ void pick_segment(PickShared<SRC>& shared, const typename Logit<SRC>::Raw* row, int V, int ns,
                                             const DrawRec& w, const Scale& scale, bool rest, double u, Mass mass) {
  constexpr int kVec = Logit<SRC>::kVec, kGroups = kSamplePer / kVec;
  const int lane = threadIdx.x & 63;
  const auto segment_mass = [&](int j) -> double { return j < ns ? mass(j) : 0.0; };
  // The segment: the first whose running sum passes u of the whole, or the last
  // that weighs anything (rounding of the sums, a random number of 1).
  double total = 0.0;
  for (int j0 = 0; j0 < ns; j0 += kWave) total += wave_sum(segment_mass(j0 + lane));
  double target = u * total, before = 0.0, left = 0.0;
  int seg = -1;
  bool passed = false;
  for (int j0 = 0; j0 < ns && !passed; j0 += kWave) {
    const double v = segment_mass(j0 + lane);
    const double run = before + wave_prefix(v);
    const unsigned long long some = __ballot(v > 0.0), hit = __ballot(v > 0.0 && run > target);
    if (some) {
      passed = hit != 0;
      const int at = passed ? __ffsll(hit) - 1 : 63 - __clzll(some);
      seg = j0 + at;
      left = target - (lane_value(run, at) - lane_value(v, at));
    }
    before = lane_value(run, 63);
  }
  if (seg < 0) {
    // Nothing is left of p - q: the row's p itself, whose segments have not
    // been summed (its cut tokens out), so that this walks the row twice.
    for (int turn = 0; turn < 2 && rest; ++turn) {
      if (turn == 1) rest = false;
      target = u * before;  // (turn 1: of the whole, summed in the same order)
      before = 0.0;
      for (int j = 0; j < ns; ++j) {
        double s = 0.0;
#pragma unroll 1
        for (int i = 0; i < kGroups; ++i) {
          const int e0 = segment_element<SRC>(j, i);
          float x[kVec];
          double p[kVec];
          load_vec<SRC>(row, e0, V, x);
          draw_weights<kVec>(w, scale, nullptr, false, e0, V, x, p);
#pragma unroll
          for (int e = 0; e < kVec; ++e) s += p[e];
        }
        s = wave_sum(s);
        if (turn == 1 && s > 0.0) {
          seg = j;
          left = target - before;
          if (before + s > target) break;
        }
        before += s;
      }
    }
  }
  if (lane == 0) {
    shared.seg = seg;
    shared.left = left;
    shared.rest = rest;
  }
}

template <int SRC, int WAVES, typename Mass>
__device__ __forceinline__ void pick_token(PickShared<SRC>& shared, const typename Logit<SRC>::Raw* row, int V, int ns,
                                           const DrawRec& w, const Scale& scale, const float* q, bool rest, double u,
                                           Mass mass, long long* out) {
  constexpr int kVec = Logit<SRC>::kVec, kGroups = kSamplePer / kVec, kMine = (kGroups + WAVES - 1) / WAVES;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (wave == 0) pick_segment<SRC>(shared, row, V, ns, w, scale, rest, u, mass);
  __syncthreads();
  const int seg = shared.seg;
  if (seg < 0) {
    if (threadIdx.x == 0) *out = -1;
    return;
  }
  // Running sums over the segment in the order of its indices: a group is a
  // wavefront's load.
  double p[kMine][kVec], run[kMine], sum[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int g = wave + i * WAVES;
    if (g >= kGroups) continue;
    const int e0 = segment_element<SRC>(seg, g);
    float x[kVec];
    load_vec<SRC>(row, e0, V, x);
    draw_weights<kVec>(w, scale, q, shared.rest, e0, V, x, p[i]);
    sum[i] = 0.0;
#pragma unroll
    for (int e = 0; e < kVec; ++e) sum[i] += p[i][e];
    run[i] = wave_prefix(sum[i]);
    if (lane == 63) shared.totals[g] = run[i];
  }
  __syncthreads();
  const double target = shared.left;
  int at = -1;
  bool passed = false;
  double before = 0.0, left = 0.0;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const double s = shared.totals[g];
    if (!passed && s > 0.0) {
      at = g;
      left = target - before;
      passed = before + s > target;
    }
    before += s;
  }
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    if (at < 0 || wave + i * WAVES != at) continue;
    const unsigned long long some = __ballot(sum[i] > 0.0), hit = __ballot(sum[i] > 0.0 && run[i] > left);
    const int which = hit ? __ffsll(hit) - 1 : 63 - __clzll(some);  // (rounding: the last that weighs anything)
    if (lane != which) continue;
    double up_to = run[i] - sum[i];
    int last = 0, first = -1;
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      up_to += p[i][e];
      if (p[i][e] > 0.0) {
        last = e;
        if (first < 0 && up_to > left) first = e;
      }
    }
    *out = segment_element<SRC>(seg, at) + (hit && first >= 0 ? first : last);
  }
  if (at < 0 && threadIdx.x == 0) *out = -1;
}

// Histograms of the workgroups' parts of a row, for top_k and top_p: bins are
// steps of a tenth of a factor of 2 in the weight, counted from the bin of the
// part's maximum on.  The steps are absolute (floor of l times 10 c, within 24
// bits), so that the parts of a row differ by a shift only; the bin of a logit
// is monotone in it, and what is past the last bin weighs less than 2^-51 of
// the part's maximum, which is 0 as an integer.  Where the maximum is +inf, that is the top bin and the
// finite logits are past the last one.  Sums are integers, weights times 2^49
// rounded: they do not depend on the order of the atomics.
constexpr int kBins = 512;
constexpr int kBinBits = 49;
constexpr float kBinMost = 8000000.0f;

struct Histogram {
  unsigned long long sum[kBins];
  uint32_t count[kBins];  // (where a top_k is given)
};

__device__ __forceinline__ float bin_scale(const Scale& s) { return s.infinite ? 1e-30f : (float)fmin(10.0 * s.c, 3e38); }
__device__ __forceinline__ int bin_of(float l, float c, float most = kBinMost) {
  int bin;  // floor and conversion in one instruction
  asm("v_cvt_flr_i32_f32 %0, %1" : "=v"(bin) : "v"(__builtin_amdgcn_fmed3f(l * c, -most, most)));
  return bin;
}

// Weight as an integer, in units of 2^-bits (the rounding of a sum at 2^52).
__device__ __forceinline__ unsigned long long fixed_weight(double w, double unit) {
  double sum;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(sum) : "v"(w), "v"(unit), "s"(4503599627370496.0));
  return (unsigned long long)__double_as_longlong(sum) & 0xfffffffffffffULL;
}

// Whether a row's parameters may drop tokens.
__device__ __forceinline__ bool row_filters(const SampleRows& r, int b, float t, bool& by_k, bool& by_p) {
  const int k = r.limit(b);
  by_k = k > 0 && k < r.V;
  by_p = r.nucleus(b) < 1.0f;
  return t > 0.0f && (by_k || by_p);
}

// The first place of a segment's maximum.
template <int SRC>
__device__ __forceinline__ int first_place(const float* x, float m, int seg) {
  constexpr int kVec = Logit<SRC>::kVec;
  int arg = 0x7fffffff;
#pragma unroll
  for (int e = kSamplePer - 1; e >= 0; --e)
    if (x[e] == m) arg = segment_element<SRC>(seg, e / kVec) + e % kVec;
  return wave_min(arg, 0x7fffffff);
}

// A segment's record by the maximum of its workgroup's part of a row, and in h,
// which is clear, the histogram of the part where tokens may be dropped.
template <int SRC>
__device__ __forceinline__ SegRec part_sums(const float* x, int seg, float t, bool filters, bool by_k, float* tops,
                                            Histogram& h) {
  float m = -INFINITY;
#pragma unroll
  for (int e = 0; e < kSamplePer; ++e) m = fmaxf(m, x[e]);
  m = wave_max(m, -INFINITY);
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  SegRec g{0.0, m, -1};
  if (m > -INFINITY) {
    if (t > 0.0f) {
      const Scale s = make_scale(m, t);
      const float bins = bin_scale(s);
      const int top_bin = bin_of(m, bins);
      constexpr double kUnit = (double)(1ULL << kBinBits);
      float most = kBinMost;
      asm("" : "+v"(most));  // (kept in a register: one move less for each logit)
#pragma unroll
      for (int e = 0; e < kSamplePer; e += 8) {
        double w[8];
        sample_weights<8>(x + e, s, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) g.sum += w[j];
        if (filters) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int bin = top_bin - bin_of(x[e + j], bins, most);
            const unsigned long long fixed = fixed_weight(w[j], kUnit);
            if (fixed != 0) {  // (bin is below kBins then)
              if (by_k) atomicAdd(&h.count[bin], 1u);
              atomicAdd(&h.sum[bin], fixed);
            }
          }
        }
      }
      g.sum = wave_sum(g.sum);
    } else {
      g.arg = first_place<SRC>(x, m, seg);
    }
  }
  return g;
}

// What a row's cut looks for (vrm_sample_cut.hip).  Bins are absolute; first is
// the one of the larger logits.
constexpr int kListed = 4096;  // tokens that a row's list holds
constexpr int kBelow = 1;      // the bins to list have k tokens or more
constexpr int kWhole = 2;      // they have all tokens that weigh anything

struct CutPlan {
  double kept;                // the sum of the row's weights, all of them
  double total;               // the same by the histograms
  double k_before, p_before;  // sums before the bins of the borders
  float top;
  int arg;                    // as DrawRec's
  int filters;                // whether anything is cut
  int k;                      // top_k's, 0 where it cuts nothing
  uint32_t k_count;           // tokens before its bin
  int by_p;
  int k_first, k_last, p_first, p_last;
  int list_first, list_last, also, also_first, also_last;  // bins to list
  int all_listed;             // every token that can stay is in them
  int deep;                   // top_k's border lies past the bins: kBelow or kWhole
  int listed;                 // how many tokens they have
};

// Finds every row's cut from the histograms of its parts (cuts; with draws,
// sequences of one row, its draw too), or with tokens draws from it: mass then
// takes the sums of a row's segments, at most kDrawSegments.  lists: kListed
// order values a row.  Rows of one part are summed here (rec, which is input
// otherwise) and need no histograms, plans and lists.
constexpr int kDrawSegments = 1024;
int launch_sample_cut(const SampleRows& r, int dtype, SegRec* rec, const Histogram* hist, CutPlan* plans,
                      unsigned long long* lists, RowCut* cuts, DrawRec* draws, double* mass, const float* uniforms,
                      long long* tokens, hipStream_t st);

}  // namespace vrm
