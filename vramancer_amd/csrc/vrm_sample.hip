// From logits to tokens: a token per row (vrm_sample_tokens), and drafted
// tokens verified against the target's probabilities (vrm_verify_drafts).  No
// counterpart in the reference, whose batcher samples on the host.
//
// Both are passes over rows of V logits, cut into segments of 2048, one for a
// wavefront, so that few rows fill the chip too:
//   1. sample_segment_kernel    every row's segments: maximum, sum of weights;
//      sample_histogram_kernel  the same and histograms, where top_k or top_p
//                               may drop tokens
//   2. launch_sample_cut        which tokens stay (vrm_sample_cut.hip); for rows
//                               of up to 8192 logits also 1, in one launch
//   3. sample_choose_kernel     a sequence's drafts: accepted ones, the row its
//                               next token is drawn from (for small batches in
//                               the launch that follows)
//   4. sample_mass_kernel       that row's segments: the mass to draw from
//   5. sample_pick_kernel       the segment and the token where the running sum
//                               passes the random number
// Large batches of drafts run 1, 4 and 5 in forms of their own, in float32 where
// that decides (sample_rough_*).
// A draw without top_k and top_p is 1 and 5, one with them 1 and 2 (which picks
// too), and 1, 2, 4 and 5 where its distribution is asked for.
#include <algorithm>

#include "vrm_sample.h"

namespace vrm {
namespace {

// ---------------------------------------------------------------------------
// 1. Segments of rows
// ---------------------------------------------------------------------------

template <int SRC>
__global__ void __launch_bounds__(kSampleThreads) sample_segment_kernel(SampleRows r, int ns, int blocks, SegRec* rec) {
  const int slot = blockIdx.x / blocks, seg = (blockIdx.x % blocks) * 4 + (threadIdx.x >> 6);
  const int b = slot / (r.K + 1), i = slot % (r.K + 1);
  if (seg >= ns || i >= r.count(b)) return;
  float x[kSamplePer];
  load_segment<SRC>(row_at<SRC>(r, r.first(b) + i), seg, r.V, x);
  const float t = r.temp(b);
  float m = -INFINITY;
#pragma unroll
  for (int e = 0; e < kSamplePer; ++e) m = fmaxf(m, x[e]);
  m = wave_max(m, -INFINITY);
  SegRec g{0.0, m, -1};
  if (m > -INFINITY) {
    if (t > 0.0f) {
      const Scale s = make_scale(m, t);
#pragma unroll
      for (int e = 0; e < kSamplePer; e += 8) {
        double w[8];
        sample_weights<8>(x + e, s, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) g.sum += w[j];
      }
      g.sum = wave_sum(g.sum);
    } else {
      g.arg = first_place<SRC>(x, m, seg);
    }
  }
  if ((threadIdx.x & 63) == 0) rec[(long long)slot * ns + seg] = g;
}

// The same with the histogram of the workgroup's four segments, whose common
// maximum gives the scale.  (Five wavefronts a SIMD here and in
// sample_collect_kernel, at the price of three registers that spill: more loads
// are under way where there are wavefronts for it.  Calls with five and with four:
// 52.9 and 56.1 us for 64 rows of 152000, 59.8 and 60.8 for 96 of 131072, 124 and
// 134 for 300 of 128256; 40.5 and 40.3 for 20 of 100003, 43.4 and 43.1 for 128 of
// 50000.)
template <int SRC>
__global__ void __launch_bounds__(kSampleThreads, 5)
    sample_histogram_kernel(SampleRows r, int ns, int blocks, SegRec* rec, Histogram* hist) {
  __shared__ Histogram h;
  __shared__ float tops[4];
  const int slot = blockIdx.x / blocks, wave = threadIdx.x >> 6, seg = (blockIdx.x % blocks) * 4 + wave;
  const int b = slot / (r.K + 1), i = slot % (r.K + 1);
  if (i >= r.count(b)) return;
  for (int j = threadIdx.x; j < kBins; j += kSampleThreads) {
    h.sum[j] = 0;
    h.count[j] = 0;
  }
  float x[kSamplePer];
  load_segment<SRC>(row_at<SRC>(r, r.first(b) + i), seg, r.V, x);
  const float t = r.temp(b);
  bool by_k, by_p;
  const bool filters = row_filters(r, b, t, by_k, by_p);
  const SegRec g = part_sums<SRC>(x, seg, t, filters, by_k, tops, h);
  if ((threadIdx.x & 63) == 0 && seg < ns) rec[(long long)slot * ns + seg] = g;
  if (!filters) return;
  __syncthreads();
  Histogram& to = hist[blockIdx.x];
  for (int j = threadIdx.x; j < kBins; j += kSampleThreads) {
    to.sum[j] = h.sum[j];
    if (by_k) to.count[j] = h.count[j];
  }
}

// The same as sample_segment_kernel in float32, for large batches of drafts: all
// that most rows are for is the test of one draft.  Sums are within kRough of the
// exact ones: a term errs by 3 2^-24 |y| ln 2 + 2^-23 of itself (the difference,
// the scale and their product, and the exponential's last place), which is
// 4.1e-6 for |y| <= 32; what lies below weighs V 2^-32 of the largest at most;
// 32 terms of a lane, added in pairs, add 5 2^-24: 4.4e-6 in all.  Differences
// are taken in halves where whole ones could overflow, and times 2^64 where the
// scale could (temperatures below 1e-38 tell subnormal logits apart; logits
// above 1e18 then differ by nothing or by everything).  A subnormal scale errs by
// more, and is of |y| < 3.
constexpr double kRough = 5e-6;

template <int SRC>
__global__ void __launch_bounds__(kSampleThreads) sample_rough_kernel(SampleRows r, int ns, int blocks, SegRec* rec) {
  const int slot = blockIdx.x / blocks, seg = (blockIdx.x % blocks) * 4 + (threadIdx.x >> 6);
  const int b = slot / (r.K + 1), i = slot % (r.K + 1);
  if (seg >= ns || i >= r.count(b)) return;
  float x[kSamplePer];
  load_segment<SRC>(row_at<SRC>(r, r.first(b) + i), seg, r.V, x);
  const float t = r.temp(b);
  float m = -INFINITY;
#pragma unroll
  for (int e = 0; e < kSamplePer; ++e) m = fmaxf(m, x[e]);
  m = wave_max(m, -INFINITY);
  SegRec g{0.0, m, -1};
  if (m > -INFINITY) {
    if (t > 0.0f) {
      const float unit = m > 1e30f ? 0.5f : t < 1e-38f && fabsf(m) < 1e18f ? 0x1p64f : 1.0f;
      const float c = fminf((float)(1.4426950408889634074 / ((double)t * unit)), 3e38f), top = -m * unit;
#pragma unroll
      for (int e = 0; e < kSamplePer; ++e) {
        const float y = fmaxf(fmaf(x[e], unit, top) * c, -200.0f);  // (a NaN is the lower bound, which underflows)
        x[e] = m == INFINITY ? (x[e] == m ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(y);
      }
#pragma unroll
      for (int n = kSamplePer / 2; n > 0; n /= 2)
#pragma unroll
        for (int e = 0; e < n; ++e) x[e] += x[e + n];
      g.sum = wave_sum((double)x[0]);
    } else {
      g.arg = first_place<SRC>(x, m, seg);
    }
  }
  if ((threadIdx.x & 63) == 0) rec[(long long)slot * ns + seg] = g;
}

// The exact sum of a row's weights, by one wavefront.
template <int SRC>
__device__ __forceinline__ double exact_sum(const typename Logit<SRC>::Raw* row, int V, int ns, const Scale& scale) {
  constexpr int kVec = Logit<SRC>::kVec;
  double sum = 0.0;
#pragma unroll 1
  for (int g = 0; g < ns * (kSamplePer / kVec); ++g) {
    float x[kVec];
    double w[kVec];
    load_vec<SRC>(row, segment_element<SRC>(g / (kSamplePer / kVec), g % (kSamplePer / kVec)), V, x);
    sample_weights<kVec>(x, scale, w);
#pragma unroll
    for (int e = 0; e < kVec; ++e) sum += w[e];
  }
  return wave_sum(sum);
}

// ---------------------------------------------------------------------------
// 3. Accepted drafts and the row to draw from: one workgroup per sequence, a
// wavefront per row in turn.  The drafts are tested at once and not one after
// the other, since each test waits for memory and few are refused.
// ---------------------------------------------------------------------------

struct Drafts {
  const void* ids;  // [B][K] of id_bytes
  int id_bytes;
  const float* probs;  // [B][K][V] with strides, or NULL: certain drafts
  long long seq_stride, draft_stride;
  const float* accept;  // [B][K]

  __device__ __forceinline__ long long id(long long at) const {
    return id_bytes == 8 ? static_cast<const long long*>(ids)[at] : (long long)static_cast<const int32_t*>(ids)[at];
  }
};

// What a row's segments and cut say about it.
struct RowSum {
  double sum;
  unsigned long long cut;
  float top;
  int arg;
  int id;  // its draft, -1: none, or outside the vocabulary
};
constexpr int kHeldRows = 16;  // rows of a sequence whose sums are held for the draw

// A row's, by one wavefront.
__device__ __forceinline__ RowSum row_sum(const SegRec* rec, const RowCut* cuts, long long slot, int ns, float t,
                                          Scale& scale) {
  RowSum g;
  combine_segments(rec + slot * ns, ns, t, g.top, g.arg, scale, g.sum);
  g.cut = 0;
  g.id = -1;
  if (cuts && g.arg == -2) {
    g.cut = cuts[slot].cut;
    g.sum = cuts[slot].sum;
  }
  return g;
}

// The drafts that sequence b accepts and its draw, for every thread of the
// workgroup.  Answers (tokens, accepted, draws) are written by the workgroup
// that has `writes`.  Every row is summed with the drafts' tests, also the one
// behind the last draft, so that the draw waits for nothing more.  With ROUGH
// sums are within kRough: a test that lies within that of its border is made
// again with the exact sum (one in 10^5), and the draw's sum is a rough one.
template <int SRC, bool ROUGH, int THREADS>
__device__ __forceinline__ DrawRec choose(const SampleRows& r, const Drafts& d, int ns, const SegRec* rec,
                                          const RowCut* cuts, int b, bool writes, DrawRec* draws, long long* tokens,
                                          int32_t* accepted, Scale& scale) {
  __shared__ int stop;  // the first row whose draft is refused, or the last row
  __shared__ RowSum held[kHeldRows];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int n = r.count(b), first = r.first(b);
  if (threadIdx.x == 0) stop = n - 1;
  __syncthreads();
  const float t = r.temp(b);
  for (int i = wave; i < n; i += THREADS / kWave) {
    if (i == n - 1 && i >= kHeldRows) break;
    const long long slot = (long long)b * (r.K + 1) + i, at = (long long)b * r.K + i;
    const bool draft = i < n - 1;
    const long long x = draft ? d.id(at) : -1;
    const bool known = x >= 0 && x < r.V;
    const float u = draft ? fminf(fmaxf(d.accept[at], 0.0f), 1.0f) : 0.0f;
    const float l = known ? Logit<SRC>::value(row_at<SRC>(r, first + i)[x]) : 0.0f;
    const float qx = known && d.probs ? d.probs[b * d.seq_stride + i * d.draft_stride + x] : 1.0f;
    Scale at_row;
    RowSum g = row_sum(rec, cuts, slot, ns, t, at_row);
    if (known) g.id = (int)x;
    if (i < kHeldRows && lane == 0) held[i] = g;
    if (!draft) break;
    bool ok = false;
    if (known && g.arg != -1) {
      double w = x == g.arg ? 1.0 : 0.0;
      if (g.arg == -2) {
        w = sample_weight(l, at_row);
        if (cuts && order_value(l, (int)x) < g.cut) w = 0.0;
      }
      const double uq = (double)u * (double)(qx < 0.0f ? 0.0f : qx);
      if (ROUGH && g.arg == -2 && uq * g.sum * (1.0 - kRough) < w && !(uq * g.sum * (1.0 + kRough) < w))
        g.sum = exact_sum<SRC>(row_at<SRC>(r, first + i), r.V, ns, at_row);
      ok = uq * g.sum < w;
    }
    if (!ok && lane == 0) atomicMin(&stop, i);
  }
  __syncthreads();
  const int a = max(stop, 0);
  if (writes) {
    for (int i = threadIdx.x; i <= r.K; i += THREADS)
      tokens[(long long)b * (r.K + 1) + i] = i < a && n > 0 ? d.id((long long)b * r.K + i) : -1;
    if (threadIdx.x == 0) accepted[b] = n > 0 ? a : 0;
  }
  if (a >= kHeldRows && n > 0) {  // (the same for every thread)
    if (wave == 0) {
      Scale at_row;
      RowSum g = row_sum(rec, cuts, (long long)b * (r.K + 1) + a, ns, t, at_row);
      if (a < n - 1) {
        const long long x = d.id((long long)b * r.K + a);
        if (x >= 0 && x < r.V) g.id = (int)x;
      }
      if (lane == 0) held[0] = g;
    }
    __syncthreads();
  }
  DrawRec w{};
  w.row = -1;
  if (n > 0) {
    const RowSum g = held[a < kHeldRows ? a : 0];
    w.sum = g.sum;
    w.cut = g.cut;
    w.top = g.top;
    w.row = first + a;
    w.arg = g.arg;
    w.refused = g.id;
    w.at = a;
    if (g.arg == -2) scale = make_scale(g.top, t);
  }
  if (writes && threadIdx.x == 0) draws[b] = w;
  return w;
}

constexpr int kChooseThreads = 512;  // (256 waited for a second row of a wavefront: 6.5 us, 5.1 now)

template <int SRC, bool ROUGH>
__global__ void __launch_bounds__(kChooseThreads)
    sample_choose_kernel(SampleRows r, Drafts d, int ns, const SegRec* rec, const RowCut* cuts, DrawRec* draws,
                         long long* tokens, int32_t* accepted) {
  Scale scale;
  choose<SRC, ROUGH, kChooseThreads>(r, d, ns, rec, cuts, blockIdx.x, true, draws, tokens, accepted, scale);
}

// ---------------------------------------------------------------------------
// 4. and 5. The mass of a row's tokens and the token
// ---------------------------------------------------------------------------

// A sequence's draw; without one made before, the whole of row b (by one
// wavefront).
__device__ __forceinline__ DrawRec draw_of(const SampleRows& r, const DrawRec* draws, const SegRec* rec, int ns, int b,
                                           Scale& scale) {
  DrawRec w{};
  const float t = r.temp(b);
  if (draws) {
    w = draws[b];
    if (w.row >= 0 && w.arg == -2) scale = make_scale(w.top, t);
  } else {
    combine_segments(rec + (long long)b * ns, ns, t, w.top, w.arg, scale, w.sum);
    w.row = b;
    w.refused = -1;
  }
  return w;
}

__device__ __forceinline__ const float* draft_row(const Drafts& d, const DrawRec& w, int b) {
  return d.probs ? d.probs + b * d.seq_stride + w.at * d.draft_stride : nullptr;
}

// With CHOOSE each workgroup finds its sequence's draw by itself first (the first
// one of a sequence writes tokens and accepted): a few KB of segment records
// each, and no launch between.
template <int SRC, bool CHOOSE>
__global__ void __launch_bounds__(kSampleThreads)
    sample_mass_kernel(SampleRows r, Drafts d, int ns, int blocks, const SegRec* rec, const RowCut* cuts, DrawRec* draws,
                       double* mass, float* probs, long long* tokens, int32_t* accepted) {
  const int b = blockIdx.x / blocks, part = blockIdx.x % blocks, seg = part * 4 + (threadIdx.x >> 6);
  constexpr int kVec = Logit<SRC>::kVec, kGroups = kSamplePer / kVec;
  Scale scale;
  const DrawRec w = CHOOSE ? choose<SRC, false, kSampleThreads>(r, d, ns, rec, cuts, b, part == 0, draws, tokens,
                                                                accepted, scale)
                           : draw_of(r, draws, rec, ns, b, scale);
  if (seg >= ns) return;
  if (w.row < 0 || (w.arg != -2 && !probs)) return;
  const bool known = w.arg != -2;  // greedy, or no token
  const bool rest = w.refused >= 0;
  const auto* row = row_at<SRC>(r, w.row);
  const float* q = draft_row(d, w, b);
  const double inv = 1.0 / w.sum;
  float x[kSamplePer];
  if (!known) load_segment<SRC>(row, seg, r.V, x);
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const int e0 = segment_element<SRC>(seg, i);
    double p[kVec];
    if (known) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) p[e] = e0 + e == w.arg ? w.sum : 0.0;
    } else {
      draw_weights<kVec>(w, scale, q, rest, e0, r.V, x + i * kVec, p);
#pragma unroll
      for (int e = 0; e < kVec; ++e) s += p[e];
    }
    if (probs) {
      float* to = probs + (long long)b * r.V + e0;
      const double by = known ? 1.0 : inv;
      if (e0 + kVec <= r.V) {
#pragma unroll
        for (int h = 0; h < kVec; h += 4) {
          Unaligned16<uint32_t> raw;
#pragma unroll
          for (int e = 0; e < 4; ++e) raw.v[e] = __float_as_uint((float)(p[h + e] * by));
          *reinterpret_cast<Unaligned16<uint32_t>*>(to + h) = raw;
        }
      } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e)
          if (e0 + e < r.V) to[e] = (float)(p[e] * by);
      }
    }
  }
  if (known) return;
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) mass[(long long)b * ns + seg] = s;
}

// The masses of a draw whose row's sum is known roughly: what max(p - q, 0) adds
// up to is the weight of the tokens that are above q by more than the sum can
// be off, less their q times the exact sum, which is the sum of `all`.  A token
// nearer to its border than that (a few in a row) is kept beside them; segments
// with more than one (near > 1) are summed again (with all of them summed again
// the pick took 10.2 us for 160 rows of 131072, 5.6 now).
struct RoughMass {
  double all, above, q, near_weight, near_q;
  long long near;
};

template <int SRC>
__global__ void __launch_bounds__(kSampleThreads)
    sample_rough_mass_kernel(SampleRows r, Drafts d, int ns, int blocks, const DrawRec* draws, RoughMass* mass) {
  const int b = blockIdx.x / blocks, seg = (blockIdx.x % blocks) * 4 + (threadIdx.x >> 6);
  if (seg >= ns) return;
  constexpr int kVec = Logit<SRC>::kVec, kGroups = kSamplePer / kVec;
  const DrawRec w = draws[b];
  if (w.row < 0 || w.arg != -2) return;
  const Scale scale = make_scale(w.top, r.temp(b));
  const float* q = w.refused >= 0 ? draft_row(d, w, b) : nullptr;
  const double low = w.sum * (1.0 - 1.01 * kRough), high = w.sum * (1.0 + 1.01 * kRough);
  float x[kSamplePer];
  load_segment<SRC>(row_at<SRC>(r, w.row), seg, r.V, x);
  RoughMass g{};
  uint32_t near = 0;
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const int e0 = segment_element<SRC>(seg, i);
    float qx[kVec];
    double p[kVec];
    if (q) load_probs<kVec>(q, e0, r.V, qx);
    sample_weights<kVec>(x + i * kVec, scale, p);
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      g.all += p[e];
      if (q) {
        const double qe = qx[e] < 0.0f ? 0.0f : qx[e];
        const bool above = p[e] > qe * high;
        g.above += above ? p[e] : 0.0;
        g.q += above ? qe : 0.0;
        if (!above && p[e] > qe * low) near |= 1u << (i * kVec + e);
      } else {
        g.above += e0 + e == w.refused ? 0.0 : p[e];
      }
    }
  }
  g.all = wave_sum(g.all);
  g.above = wave_sum(g.above);
  g.q = wave_sum(g.q);
  const unsigned long long some = __ballot(near != 0);
  if (some) {
    const int lane = __ffsll(some) - 1;
    const uint32_t bits = lane_value(near, lane);
    g.near = (some & (some - 1)) || (bits & (bits - 1)) ? 2 : 1;
    if (near) {  // (read again: registers have no index)
      const int bit = __ffs(near) - 1, at = segment_element<SRC>(seg, bit / kVec) + bit % kVec;
      g.near_weight = sample_weight(Logit<SRC>::value(row_at<SRC>(r, w.row)[at]), scale);
      g.near_q = q[at];
    }
    g.near_weight = lane_value(g.near_weight, lane);
    g.near_q = lane_value(g.near_q, lane);
  }
  if ((threadIdx.x & 63) == 0) mass[(long long)b * ns + seg] = g;
}

// The exact masses from these, and the token; one workgroup per sequence.
template <int SRC>
__global__ void __launch_bounds__(kSampleThreads)
    sample_rough_pick_kernel(SampleRows r, Drafts d, int ns, const DrawRec* draws, const RoughMass* rough, double* mass,
                             const float* uniforms, long long* tokens) {
  __shared__ PickShared<SRC> shared;
  const int b = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const float u = uniforms[b];
  DrawRec w = draws[b];
  if (w.row < 0) return;
  long long* out = tokens + (long long)b * (r.K + 1) + w.at;
  if (w.arg != -2) {
    if (threadIdx.x == 0) *out = w.arg;
    return;
  }
  constexpr int kVec = Logit<SRC>::kVec, kGroups = kSamplePer / kVec;
  const auto* row = row_at<SRC>(r, w.row);
  const float* q = draft_row(d, w, b);
  const bool rest = w.refused >= 0;
  const Scale scale = make_scale(w.top, r.temp(b));
  const RoughMass* from = rough + (long long)b * ns;
  double* to = mass + (long long)b * ns;
  double sum = 0.0;
  for (int j = lane; j < ns; j += kWave) sum += from[j].all;
  w.sum = wave_sum(sum);
  int turn = 0;  // the marked segments, to the wavefronts in turn
  for (int j0 = 0; j0 < ns; j0 += kWave) {
    const int j = j0 + lane;
    const RoughMass g = j < ns ? from[j] : RoughMass{};
    if (wave == 0 && j < ns && g.near <= 1) {
      const double near = g.near ? fmax(fma(-g.near_q, w.sum, g.near_weight), 0.0) : 0.0;
      to[j] = rest ? fmax(fma(-g.q, w.sum, g.above), 0.0) + near : g.all;
    }
    unsigned long long near = __ballot(g.near > 1);
    for (; near; near &= near - 1, ++turn) {
      if (turn % (kSampleThreads / kWave) != wave) continue;
      const int at = __ffsll(near) - 1;
      float x[kSamplePer];
      load_segment<SRC>(row, j0 + at, r.V, x);
      double s = 0.0;
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        double p[kVec];
        draw_weights<kVec>(w, scale, q, rest, segment_element<SRC>(j0 + at, i), r.V, x + i * kVec, p);
#pragma unroll
        for (int e = 0; e < kVec; ++e) s += p[e];
      }
      s = wave_sum(s);
      if (lane == at) to[j] = s;
    }
  }
  __syncthreads();
  pick_token<SRC, kSampleThreads / kWave>(shared, row, r.V, ns, w, scale, q, rest, fmin(fmax((double)u, 0.0), 1.0),
                                          [&](int j) { return to[j]; }, out);
}

// One workgroup per sequence.  mass == NULL: a draw from row b by its segments'
// sums.
template <int SRC>
__global__ void __launch_bounds__(kSampleThreads)
    sample_pick_kernel(SampleRows r, Drafts d, int ns, const SegRec* rec, const DrawRec* draws, const double* mass,
                       const float* uniforms, long long* tokens) {
  __shared__ PickShared<SRC> shared;
  __shared__ DrawRec draw;
  const int b = blockIdx.x;
  const float u = uniforms[b];
  Scale scale;
  DrawRec w;
  if (draws) {
    w = draw_of(r, draws, rec, ns, b, scale);
  } else {
    if (threadIdx.x < kWave) {
      w = draw_of(r, draws, rec, ns, b, scale);
      if (threadIdx.x == 0) draw = w;
    }
    __syncthreads();
    w = draw;
    if (w.arg == -2) scale = make_scale(w.top, r.temp(b));
  }
  if (w.row < 0) return;
  long long* out = tokens + (long long)b * (r.K + 1) + w.at;
  if (w.arg != -2) {
    if (threadIdx.x == 0) *out = w.arg;
    return;
  }
  pick_token<SRC, kSampleThreads / kWave>(shared, row_at<SRC>(r, w.row), r.V, ns, w, scale, draft_row(d, w, b),
                                          w.refused >= 0, fmin(fmax((double)u, 0.0), 1.0),
                                          [&](int j) {
                                            return mass ? mass[(long long)b * ns + j]
                                                        : segment_sum(rec[(long long)b * ns + j], scale);
                                          },
                                          out);
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

size_t up(size_t n) { return (n + 255) & ~(size_t)255; }

// What a call runs and where its workspace holds what.
struct Plan {
  long long slots;
  int ns, blocks;  // segments and workgroups of a row
  bool filtered, drafts, masses;
  bool fused;  // the cut draws by itself
  bool rough;  // rows summed in float32 first
  size_t rough_mass, hist, plans, lists, cuts, draws, mass, bytes;
};

// From how many logits of all rows on they are summed in float32 first: 45.0 us a
// call against 46.5 for 48 sequences of 4 drafts and 152000 (36 million), 46.9
// against 48.1 for 200 and 32000 (32 million); 38.0 against 35.6 for 32 and
// 152000 (24 million), 25.1 against 22.1 for 256 and 8192 (10 million).
constexpr long long kRoughLogits = 1 << 25;

Plan plan_of(long long B, int K, int V, bool filtered, bool drafts, bool probs) {
  Plan p{};
  p.slots = B * (K + 1);
  p.ns = (V + kSegment - 1) / kSegment;
  p.blocks = (V + kSampleBlock - 1) / kSampleBlock;
  p.filtered = filtered;
  p.drafts = drafts;
  p.masses = filtered || drafts || probs;
  p.fused = filtered && !drafts && !probs && p.ns <= kDrawSegments;
  p.rough = drafts && !filtered && p.slots * V >= kRoughLogits;
  size_t at = up((size_t)p.slots * p.ns * sizeof(SegRec));
  if (p.rough) {
    p.rough_mass = at;
    at += up((size_t)B * p.ns * sizeof(RoughMass));
  }
  if (filtered) {
    if (p.blocks > 1) {
      p.hist = at;
      at += up((size_t)p.slots * p.blocks * sizeof(Histogram));
      p.plans = at;
      at += up((size_t)p.slots * sizeof(CutPlan));
      p.lists = at;
      at += up((size_t)p.slots * kListed * sizeof(unsigned long long));
    }
    p.cuts = at;
    at += up((size_t)p.slots * sizeof(RowCut));
  }
  if (filtered || drafts) {
    p.draws = at;
    at += up((size_t)B * sizeof(DrawRec));
  }
  if (p.masses) {
    p.mass = at;
    at += up((size_t)B * p.ns * sizeof(double));
  }
  p.bytes = at;
  return p;
}

// Up to this many workgroups, which the chip has at once, every one of a
// sequence's masses tests its drafts (for a few drafts): 9.7 us against 5.2 + 7.0
// in two launches for 8 sequences of 3 drafts and 32000 logits (32 workgroups),
// 15.6 against 7.0 + 10.7 for 37 of 7 and 100003 (481); 23.5 against 6.0 + 15.8
// for 64 of 4 and 152000 (1216).  Of many drafts each workgroup repeats as many
// tests: 23.7 us a call against 25.3 for 8 sequences of 9 and 32000, 24.6 and 25.0
// for 12, 26.4 and 25.8 for 16, 30.6 and 28.4 for 24.
constexpr int kChooseBlocks = 768, kChooseDrafts = 12;

// A launch counts its threads in 32 bits.
constexpr long long kMostBlocks = (1LL << 32) / 1024 - 1;

template <int SRC>
int run(const SampleRows& r, const Drafts& d, const Plan& p, char* ws, const float* uniforms, float* probs,
        long long* tokens, int32_t* accepted, hipStream_t st, const char* who) {
  auto* rec = reinterpret_cast<SegRec*>(ws);
  auto* draws = p.draws ? reinterpret_cast<DrawRec*>(ws + p.draws) : nullptr;
  auto* mass = p.masses ? reinterpret_cast<double*>(ws + p.mass) : nullptr;
  const dim3 row_blocks((unsigned)(p.slots * p.blocks)), threads(kSampleThreads);
  RowCut* cuts = nullptr;
  if (p.filtered) {
    auto* hist = reinterpret_cast<Histogram*>(ws + p.hist);
    cuts = reinterpret_cast<RowCut*>(ws + p.cuts);
    if (p.blocks > 1)
      hipLaunchKernelGGL((sample_histogram_kernel<SRC>), row_blocks, threads, 0, st, r, p.ns, p.blocks, rec, hist);
    if (int rc = launch_sample_cut(r, SRC, rec, hist, reinterpret_cast<CutPlan*>(ws + p.plans),
                                   reinterpret_cast<unsigned long long*>(ws + p.lists), cuts,
                                   p.drafts ? nullptr : draws, mass, uniforms, p.fused ? tokens : nullptr, st))
      return rc;
    if (p.fused) return launch_status(who);
  } else if (p.rough) {
    hipLaunchKernelGGL((sample_rough_kernel<SRC>), row_blocks, threads, 0, st, r, p.ns, p.blocks, rec);
  } else {
    hipLaunchKernelGGL((sample_segment_kernel<SRC>), row_blocks, threads, 0, st, r, p.ns, p.blocks, rec);
  }
  const dim3 mass_blocks((unsigned)((long long)r.B * p.blocks));
  if (p.rough) {
    auto* rough = reinterpret_cast<RoughMass*>(ws + p.rough_mass);
    hipLaunchKernelGGL((sample_choose_kernel<SRC, true>), dim3(r.B), dim3(kChooseThreads), 0, st, r, d, p.ns, rec,
                       nullptr, draws, tokens, accepted);
    hipLaunchKernelGGL((sample_rough_mass_kernel<SRC>), mass_blocks, threads, 0, st, r, d, p.ns, p.blocks, draws, rough);
    hipLaunchKernelGGL((sample_rough_pick_kernel<SRC>), dim3(r.B), threads, 0, st, r, d, p.ns, draws, rough, mass,
                       uniforms, tokens);
    return launch_status(who);
  }
  if (p.drafts && r.K <= kChooseDrafts && mass_blocks.x <= (unsigned)kChooseBlocks) {
    hipLaunchKernelGGL((sample_mass_kernel<SRC, true>), mass_blocks, threads, 0, st, r, d, p.ns, p.blocks, rec, cuts,
                       draws, mass, nullptr, tokens, accepted);
  } else {
    if (p.drafts)
      hipLaunchKernelGGL((sample_choose_kernel<SRC, false>), dim3(r.B), dim3(kChooseThreads), 0, st, r, d, p.ns, rec,
                         cuts, draws, tokens, accepted);
    if (p.masses)
      hipLaunchKernelGGL((sample_mass_kernel<SRC, false>), mass_blocks, threads, 0, st, r, d, p.ns, p.blocks, rec, cuts,
                         draws, mass, probs, nullptr, nullptr);
  }
  hipLaunchKernelGGL((sample_pick_kernel<SRC>), dim3(r.B), threads, 0, st, r, d, p.ns, rec, draws, mass, uniforms,
                     tokens);
  return launch_status(who);
}

int run_typed(const SampleRows& r, int dtype, const Drafts& d, const Plan& p, char* ws, const float* uniforms,
              float* probs, long long* tokens, int32_t* accepted, hipStream_t st, const char* who) {
  switch (dtype) {
    case VRM_SRC_F32: return run<VRM_SRC_F32>(r, d, p, ws, uniforms, probs, tokens, accepted, st, who);
    case VRM_SRC_F16: return run<VRM_SRC_F16>(r, d, p, ws, uniforms, probs, tokens, accepted, st, who);
    default: return run<VRM_SRC_BF16>(r, d, p, ws, uniforms, probs, tokens, accepted, st, who);
  }
}

int check_sizes(long long B, int K, int V, int dtype, long long stride, const char* who) {
  if (B < 0 || K < 0 || V <= 0 || stride < 0) {
    set_error("%s: bad sizes (sequences %lld, drafts %d, V=%d, row stride %lld)", who, B, K, V, stride);
    return VRM_ERR_ARG;
  }
  if (dtype != VRM_SRC_F32 && dtype != VRM_SRC_F16 && dtype != VRM_SRC_BF16) {
    set_error("%s: unknown logits dtype %d", who, dtype);
    return VRM_ERR_ARG;
  }
  if (V > VRM_SAMPLE_MAX_V) {
    set_error("%s: V=%d above %d", who, V, VRM_SAMPLE_MAX_V);
    return VRM_ERR_UNSUPPORTED;
  }
  const long long blocks = (V + kSampleBlock - 1) / kSampleBlock;
  if (B > 0 && ((long long)K + 1 > kMostBlocks / blocks / B)) {
    set_error("%s: %lld sequences of %d rows of %d logits are too many for one call", who, B, K + 1, V);
    return VRM_ERR_UNSUPPORTED;
  }
  return VRM_OK;
}

int check_workspace(const void* ws, size_t bytes, size_t need, const char* who) {
  if (!ws || bytes < need) {
    set_error("%s: workspace of %zu bytes, %zu needed", who, ws ? bytes : (size_t)0, need);
    return VRM_ERR_WORKSPACE;
  }
  if (reinterpret_cast<uintptr_t>(ws) & 15) {
    set_error("%s: workspace must be 16-byte aligned", who);
    return VRM_ERR_ARG;
  }
  return VRM_OK;
}

// Bytes of n rows of V elements, stride elements apart.
size_t row_bytes(long long n, int V, long long stride, int dtype) {
  return n > 0 ? (size_t)((n - 1) * stride + V) * (dtype == VRM_SRC_F32 ? 4 : 2) : 0;
}

// Whether any row may lose tokens to top_k or top_p.
bool filters(const int32_t* top_k, int top_k_all, const float* top_p, float top_p_all, int V) {
  return top_k || (top_k_all > 0 && top_k_all < V) || top_p || top_p_all < 1.0f;
}

}  // namespace
}  // namespace vrm

using namespace vrm;

extern "C" size_t vrm_sample_workspace_bytes(int N, int V, int filtered, int with_probs) {
  if (check_sizes(N, 0, V, VRM_SRC_F32, 0, "vrm_sample_workspace_bytes")) return 0;
  return plan_of(N, 0, V, filtered != 0, false, with_probs != 0).bytes;
}

extern "C" int vrm_sample_tokens(const void* logits, int dtype, long long row_stride, const float* uniforms,
                                 const float* temperature, float temperature_all, const int32_t* top_k, int top_k_all,
                                 const float* top_p, float top_p_all, float* probs, int64_t* tokens, void* workspace,
                                 size_t workspace_bytes, int N, int V, vrm_stream_t stream) {
  const char* who = "vrm_sample_tokens";
  if (int rc = check_sizes(N, 0, V, dtype, row_stride, who)) return rc;
  if (N == 0) {
    clear_error();
    return VRM_OK;
  }
  if (!logits || !uniforms || !tokens) {
    set_error("%s: null pointer argument", who);
    return VRM_ERR_ARG;
  }
  const Plan p = plan_of(N, 0, V, filters(top_k, top_k_all, top_p, top_p_all, V), false, probs != nullptr);
  if (int rc = check_workspace(workspace, workspace_bytes, p.bytes, who)) return rc;
  const size_t n = N;
  if (int rc = check_apart({{tokens, n * 8}, {probs, n * V * 4}, {workspace, p.bytes}},
                           {{logits, row_bytes(N, V, row_stride, dtype)},
                            {uniforms, n * 4},
                            {temperature, n * 4},
                            {top_k, n * 4},
                            {top_p, n * 4}},
                           who))
    return rc;
  const SampleRows r{logits, row_stride, nullptr, N, N, 0, V, temperature, temperature_all, top_k, top_k_all, top_p,
                     top_p_all};
  return run_typed(r, dtype, Drafts{}, p, static_cast<char*>(workspace), uniforms, probs,
                   reinterpret_cast<long long*>(tokens), nullptr, reinterpret_cast<hipStream_t>(stream), who);
}

extern "C" size_t vrm_verify_workspace_bytes(int B, int K, int V, int filtered) {
  if (check_sizes(B, K, V, VRM_SRC_F32, 0, "vrm_verify_workspace_bytes")) return 0;
  // (of a large batch of short rows the calls without top_k and top_p need more)
  const size_t plain = plan_of(B, K, V, false, true, false).bytes;
  return filtered ? std::max(plan_of(B, K, V, true, true, false).bytes, plain) : plain;
}

extern "C" int vrm_verify_drafts(const void* logits, int dtype, long long row_stride, const int32_t* cu_seqlens,
                                 const void* drafts, int draft_bytes, const float* draft_probs,
                                 long long probs_seq_stride, long long probs_draft_stride,
                                 const float* accept_uniforms, const float* draw_uniforms, const float* temperature,
                                 float temperature_all, const int32_t* top_k, int top_k_all, const float* top_p,
                                 float top_p_all, int64_t* tokens, int32_t* accepted, void* workspace,
                                 size_t workspace_bytes, int N, int B, int K, int V, vrm_stream_t stream) {
  const char* who = "vrm_verify_drafts";
  if (int rc = check_sizes(B, K, V, dtype, row_stride, who)) return rc;
  if (N < 0 || (!cu_seqlens && (long long)B * (K + 1) != N)) {
    set_error("%s: %d rows of logits for %d sequences of %d drafts", who, N, B, K);
    return VRM_ERR_ARG;
  }
  if (draft_bytes != 4 && draft_bytes != 8) {
    set_error("%s: drafts are integers of 4 or 8 bytes, got %d", who, draft_bytes);
    return VRM_ERR_ARG;
  }
  if (probs_seq_stride < 0 || probs_draft_stride < 0) {
    set_error("%s: negative stride of draft_probs", who);
    return VRM_ERR_ARG;
  }
  if (B == 0) {
    clear_error();
    return VRM_OK;
  }
  if ((N > 0 && !logits) || (K > 0 && (!drafts || !accept_uniforms)) || !draw_uniforms || !tokens || !accepted) {
    set_error("%s: null pointer argument", who);
    return VRM_ERR_ARG;
  }
  const Plan p = plan_of(B, K, V, filters(top_k, top_k_all, top_p, top_p_all, V), true, false);
  if (int rc = check_workspace(workspace, workspace_bytes, p.bytes, who)) return rc;
  const size_t n = B, k = K;
  const size_t last_draft = K > 0 ? (n - 1) * probs_seq_stride + (k - 1) * probs_draft_stride + V : 0;
  if (int rc = check_apart({{tokens, n * (k + 1) * 8}, {accepted, n * 4}, {workspace, p.bytes}},
                           {{logits, row_bytes(N, V, row_stride, dtype)},
                            {cu_seqlens, (n + 1) * 4},
                            {drafts, n * k * draft_bytes},
                            {draft_probs, last_draft * 4},
                            {accept_uniforms, n * k * 4},
                            {draw_uniforms, n * 4},
                            {temperature, n * 4},
                            {top_k, n * 4},
                            {top_p, n * 4}},
                           who))
    return rc;
  const SampleRows r{logits, row_stride, cu_seqlens, N, B, K, V, temperature, temperature_all, top_k, top_k_all, top_p,
                     top_p_all};
  const Drafts d{drafts, draft_bytes, draft_probs, probs_seq_stride, probs_draft_stride, accept_uniforms};
  return run_typed(r, dtype, d, p, static_cast<char*>(workspace), draw_uniforms, nullptr,
                   reinterpret_cast<long long*>(tokens), accepted, reinterpret_cast<hipStream_t>(stream), who);
}
