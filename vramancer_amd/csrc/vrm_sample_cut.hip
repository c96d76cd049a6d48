// Which tokens of a row stay under top_k and top_p.
//
// Tokens are in the order (logit descending, index ascending).  top_k keeps the
// first k; top_p the shortest prefix of those whose weights reach top_p times
// the sum of theirs.  Either is a border in that order, and nothing is sorted to
// find it.  The histograms of the row's parts, made with its sums, are added
// up; the border's bin is found by a prefix sum over the bins; a pass over the
// row collects that bin's tokens, and bins of their order values narrow them
// down until 64 are left, which are compared with each other.
//
// Counts and sums do not depend on the order in which tokens are collected: the
// parts' sums are integers, added in 64-bit floats part by part; within a bin
// weights are integers in units of 2^-S, S such that V of them stay below 2^63
// (S = 45 for V up to 2^17).  Tokens below 2^-51 of the row's largest may weigh
// nothing here; where such a token would be the border nothing is cut.
#include "vrm_sample.h"

namespace vrm {
namespace {

constexpr int kCutThreads = 1024;
constexpr int kCutWaves = kCutThreads / kWave;
constexpr int kSub = 2048;   // bins of order values
constexpr int kList = 4096;  // tokens of a bin that fit in LDS
constexpr int kFew = 64;     // tokens that are compared with each other

using u64 = unsigned long long;

struct CutShared {
  double bin_sum[kBins];
  uint32_t bin_count[kBins];
  double half_sum[kBins];
  uint32_t half_count[kBins];
  double part_factor[kCutThreads];
  int part_shift[kCutThreads];
  u64 sub_sum[kSub];
  uint32_t sub_count[kSub];
  u64 list[kList];  // order values
  u64 few_order[kFew];
  u64 few_sum[kFew];
  double wave_sum[kCutWaves];
  u64 wave_fixed[kCutWaves];
  u64 wave_low[kCutWaves], wave_high[kCutWaves];
  uint32_t wave_count[kCutWaves];
  double before_sum;     // of the tokens before the border's bin
  u64 before_fixed;      // and, within the bin, before the interval
  u64 border;            // the answer: the border's order value
  double kept;           // and the sum up to it
  uint32_t before_count, count;
  int bin, fill;
  float top;
  int arg;
  double row_sum;
};

__device__ __forceinline__ float order_logit(u64 order) {
  const uint32_t key = (uint32_t)(order >> 32);
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// A row as the passes see it.
template <int SRC>
struct Row {
  const typename Logit<SRC>::Raw* at;
  int V;
  Scale scale;
  float bins;   // bin_scale
  int top_bin;
  double unit;  // 2^S

  // f(order value) of the tokens in the absolute bins first .. last.  Four
  // loads of a lane are under way at once: a workgroup has a row to itself, and
  // waits for memory otherwise.
  template <typename F>
  __device__ __forceinline__ void of_bins(int first, int last, F f) const {
    using L = Logit<SRC>;
    constexpr int kVec = L::kVec, kAhead = 4, kStep = kCutThreads * kVec;
    // floor of the clamped product in first .. last, as two comparisons
    const float low = first <= -(int)kBinMost ? -INFINITY : (float)first;
    const float high = last >= (int)kBinMost ? INFINITY : (float)(last + 1);
    const bool open = high == INFINITY;
    const auto test = [&](const float* x, int e0) {
      bool any = false, in[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const float y = x[e] * bins;
        in[e] = y >= low && (open || y < high);
        any |= in[e];
      }
      if (any) {
#pragma unroll
        for (int e = 0; e < kVec; ++e)
          if (in[e] && x[e] > -INFINITY) f(order_value(x[e], e0 + e));
      }
    };
#pragma unroll 1
    for (int base = 0; base < V; base += kAhead * kStep) {
      const int e0 = base + (int)threadIdx.x * kVec;
      float x[kVec];
      if (base + kAhead * kStep <= V) {
        Unaligned16<typename L::Raw> raw[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
          raw[i] = *reinterpret_cast<const Unaligned16<typename L::Raw>*>(at + e0 + i * kStep);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
#pragma unroll
          for (int e = 0; e < kVec; ++e) x[e] = L::value(raw[i].v[e]);
          test(x, e0 + i * kStep);
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < kAhead; ++i) {
          load_vec<SRC>(at, e0 + i * kStep, V, x);
          test(x, e0 + i * kStep);
        }
      }
    }
  }
  // A token's weight as an integer.
  __device__ __forceinline__ u64 weight(u64 order) const {
    return fixed_weight(sample_weight(order_logit(order), scale), unit);
  }
};

template <typename T>
__device__ __forceinline__ T prefix(T v) {  // inclusive, over a wavefront
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) {
    const T o = __shfl_up(v, m);
    if ((int)(threadIdx.x & 63) >= m) v += o;
  }
  return v;
}

// The bin of the row in which the running count reaches k (by_count) or the
// running sum goal: in s.bin (kBins: none), and what is before it in
// s.before_count and s.before_sum.
__device__ __forceinline__ void find_bin(CutShared& s, bool by_count, uint32_t k, double goal) {
  const int t = threadIdx.x, wave = t >> 6;
  const bool mine = t < kBins;
  const uint32_t c = mine ? s.bin_count[t] : 0;
  const double w = mine ? s.bin_sum[t] : 0.0;
  uint32_t rc = prefix(c);
  double rw = prefix(w);
  if ((t & 63) == 63) {
    s.wave_count[wave] = rc;
    s.wave_sum[wave] = rw;
  }
  if (t == 0) s.bin = kBins;
  __syncthreads();
  uint32_t c0 = 0;
  double w0 = 0.0;
  for (int v = 0; v < wave; ++v) {
    c0 += s.wave_count[v];
    w0 += s.wave_sum[v];
  }
  rc += c0;
  rw += w0;
  // (The least bin: running sums in floating point may step back by a rounding.)
  if (mine && (by_count ? rc >= k : rw >= goal)) atomicMin(&s.bin, t);
  const double lower = __shfl_up(rw, 1);
  __syncthreads();
  if (t == s.bin) {
    s.before_count = rc - c;
    s.before_sum = (t & 63) ? lower : w0;
  }
  __syncthreads();
}

// The step of order values in which the border is, likewise, within a bin:
// counts and integer sums after what s.before_count and s.before_fixed hold.
__device__ __forceinline__ void find_step(CutShared& s, bool by_count, uint32_t k, u64 goal) {
  const int t = threadIdx.x, wave = t >> 6;
  const uint32_t c0 = s.sub_count[2 * t], c1 = s.sub_count[2 * t + 1];
  const u64 w0 = s.sub_sum[2 * t], w1 = s.sub_sum[2 * t + 1];
  const uint32_t rc = prefix(c0 + c1);
  const u64 rw = prefix(w0 + w1);
  if ((t & 63) == 63) {
    s.wave_count[wave] = rc;
    s.wave_fixed[wave] = rw;
  }
  uint32_t c = s.before_count + rc - (c0 + c1);
  u64 w = s.before_fixed + rw - (w0 + w1);
  __syncthreads();
  for (int v = 0; v < wave; ++v) {
    c += s.wave_count[v];
    w += s.wave_fixed[v];
  }
  const auto hit = [&](uint32_t cb, u64 wb, uint32_t cn, u64 wn) {
    return by_count ? cb < k && cb + cn >= k : wb < goal && wb + wn >= goal;
  };
  int at = -1;
  if (hit(c, w, c0, w0)) {
    at = 2 * t;
  } else if (hit(c + c0, w + w0, c1, w1)) {
    at = 2 * t + 1;
    c += c0;
    w += w0;
  }
  if (at >= 0) {  // (one thread)
    s.bin = at;
    s.count = s.sub_count[at];
    s.before_count = c;
    s.before_fixed = w;
  }
  __syncthreads();
}

// The sum of a value over the workgroup, for every thread.
__device__ __forceinline__ u64 block_sum(CutShared& s, u64 v) {
  v = prefix(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) s.wave_fixed[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
  for (int w = 0; w < kCutWaves; ++w) v += s.wave_fixed[w];
  return v;
}

// Puts the tokens of bins first .. last into the list; how many there are (at
// most kList of them are in it).
template <int SRC>
__device__ __forceinline__ int collect(CutShared& s, const Row<SRC>& row, int first, int last) {
  __syncthreads();
  if (threadIdx.x == 0) s.fill = 0;
  __syncthreads();
  row.of_bins(first, last, [&](u64 o) {
    const int j = atomicAdd(&s.fill, 1);
    if (j < kList) s.list[j] = o;
  });
  __syncthreads();
  return s.fill;
}

// The border by count (the k-th token) or by sum (the first token with which
// the sum reaches goal): its order value in s.border, the sum up to it in
// s.kept.  False where the border would be among tokens that weigh nothing.
// `listed` tokens of the bins down to `list_bin` are in the list already.
template <int SRC>
__device__ bool find_border(CutShared& s, const Row<SRC>& row, bool by_count, uint32_t k, double goal, int& listed,
                            int& list_bin) {
  const int t = threadIdx.x;
  __syncthreads();
  find_bin(s, by_count, k, goal);
  if (s.bin == kBins) return false;
  const int bin = row.top_bin - s.bin;
  const double before = s.before_sum;
  if (bin < list_bin) {
    // All tokens down to this bin, if they fit (a count is known with top_k
    // alone): the border by sum, which comes before, is among them then.
    const bool all = by_count && s.before_count + s.bin_count[s.bin] <= (uint32_t)kList;
    const int n = collect(s, row, bin, all ? row.top_bin : bin);
    listed = n <= kList ? n : -1;
    list_bin = all ? bin : 0x7fffffff;
  }
  u64 low = 0, high = ~0ULL, fixed_goal = 0;
  // f(order value) of the bin's tokens within the interval: from the list, or
  // where they do not fit it by another pass over the row
  const auto each = [&](auto f) {
    if (listed >= 0) {
      for (int j = t; j < listed; j += kCutThreads) {
        const u64 o = s.list[j];
        if (o >= low && o <= high && bin_of(order_logit(o), row.bins) == bin) f(o);
      }
    } else {
      row.of_bins(bin, bin, [&](u64 o) {
        if (o >= low && o <= high) f(o);
      });
    }
  };
  // How many there are, and what they weigh.
  u64 sum = 0;
  uint32_t mine = 0;
  each([&](u64 o) {
    ++mine;
    if (!by_count) sum += row.weight(o);
  });
  uint32_t n = (uint32_t)block_sum(s, mine);
  if (!by_count) {
    // The part of the goal that is within the bin, at most what the bin's
    // integers add up to (they are rounded apart from the histograms').
    sum = block_sum(s, sum);
    if (sum == 0) return false;
    const double want = ceil((goal - before) * row.unit);
    fixed_goal = want < 1.0 ? 1 : min((u64)want, sum);
  }
  if (t == 0) {
    s.before_fixed = 0;
    s.fill = 0;
  }
  __syncthreads();
  while (n > (uint32_t)kFew) {
    // The interval that the tokens really take, and 2048 steps of it.
    u64 a = ~0ULL, z = 0;
    each([&](u64 o) {
      a = min(a, o);
      z = max(z, o);
    });
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) {
      a = min(a, (u64)__shfl_xor(a, m));
      z = max(z, (u64)__shfl_xor(z, m));
    }
    if ((t & 63) == 0) {
      s.wave_low[t >> 6] = a;
      s.wave_high[t >> 6] = z;
    }
    for (int j = t; j < kSub; j += kCutThreads) {
      s.sub_count[j] = 0;
      s.sub_sum[j] = 0;
    }
    __syncthreads();
    for (int v = 0; v < kCutWaves; ++v) {
      a = min(a, s.wave_low[v]);
      z = max(z, s.wave_high[v]);
    }
    low = a;
    high = z;
    const int shift = max(0, 64 - __clzll(high - low) - 11);  // (high - low) >> shift < 2048
    each([&](u64 o) {
      const int j = (int)((high - o) >> shift);
      atomicAdd(&s.sub_count[j], 1u);
      if (!by_count) atomicAdd(&s.sub_sum[j], row.weight(o));
    });
    __syncthreads();
    find_step(s, by_count, k, fixed_goal);
    n = s.count;
    const u64 j = s.bin;  // (there is one: the interval has the border)
    const u64 top = high - (j << shift);
    const u64 span = (1ULL << shift) - 1;
    low = top - low > span ? top - span : low;
    high = top;
    __syncthreads();
  }
  each([&](u64 o) {
    const int j = atomicAdd(&s.fill, 1);
    s.few_order[j] = o;
    s.few_sum[j] = row.weight(o);
  });
  __syncthreads();
  if (t < (int)n) {
    const u64 o = s.few_order[t], w = s.few_sum[t];
    uint32_t c = s.before_count;
    u64 up_to = s.before_fixed;
    for (uint32_t j = 0; j < n; ++j) {
      if (s.few_order[j] > o) {
        ++c;
        up_to += s.few_sum[j];
      }
    }
    if (by_count ? c + 1 == k : up_to < fixed_goal && up_to + w >= fixed_goal) s.border = o;  // (one of them)
  }
  __syncthreads();
  // The sum of the bin's tokens up to the border.
  low = s.border;
  high = ~0ULL;
  sum = 0;
  each([&](u64 o) { sum += row.weight(o); });
  sum = block_sum(s, sum);
  if (t == 0) s.kept = before + (double)sum / row.unit;
  __syncthreads();
  return true;
}

// One workgroup per row.
template <int SRC>
__global__ void __launch_bounds__(kCutThreads)
    sample_cut_kernel(SampleRows r, int ns, int parts, int bits, const SegRec* rec, const Histogram* hist, RowCut* cuts,
                      DrawRec* draws) {
  __shared__ CutShared s;
  const int slot = blockIdx.x, b = slot / (r.K + 1), i = slot % (r.K + 1), t = threadIdx.x;
  if (i >= r.count(b)) return;
  const float temp = r.temp(b);
  if (t < kWave) {
    float top;
    int arg;
    Scale scale;
    double sum;
    combine_segments(rec + (long long)slot * ns, ns, temp, top, arg, scale, sum);
    if (t == 0) {
      s.top = top;
      s.arg = arg;
      s.row_sum = sum;
    }
  }
  __syncthreads();
  bool by_k, by_p;
  const bool filters = row_filters(r, b, temp, by_k, by_p) && s.arg == -2;
  u64 cut = 0;
  double kept = s.row_sum;
  if (filters) {
    Row<SRC> row;
    row.at = row_at<SRC>(r, r.first(b) + i);
    row.V = r.V;
    row.scale = make_scale(s.top, temp);
    row.bins = bin_scale(row.scale);
    row.unit = (double)(1ULL << bits);
    row.top_bin = bin_of(s.top, row.bins);
    // The parts' histograms, shifted to the row's bins and scaled; the even
    // parts by the first 512 threads, the odd ones by the others.
    const int mine = t & (kBins - 1), half = t / kBins;
    double sum = 0.0;
    uint32_t count = 0;
    for (int p0 = 0; p0 < parts; p0 += kCutThreads) {
      __syncthreads();
      const int p = p0 + t;
      if (p < parts) {
        const float top = rec[(long long)slot * ns + p * 4].top;  // (of the whole part)
        const SegRec one{1.0 / (double)(1ULL << kBinBits), top, 0};
        const double factor = segment_sum(one, row.scale);
        s.part_factor[t] = factor;
        // (a part that weighs nothing has no bins in the row)
        s.part_shift[t] = factor > 0.0 ? row.top_bin - bin_of(top, row.bins) : kBins;
      }
      __syncthreads();
      const int n = min(parts - p0, kCutThreads);
#pragma unroll 8
      for (int j = half; j < n; j += kCutThreads / kBins) {
        const int at = mine - s.part_shift[j];
        if (at >= 0) {
          const Histogram& h = hist[(long long)slot * parts + p0 + j];
          sum += (double)h.sum[at] * s.part_factor[j];
          if (by_k) count += h.count[at];
        }
      }
    }
    if (half) {
      s.half_sum[mine] = sum;
      s.half_count[mine] = count;
    }
    __syncthreads();
    if (!half) {
      sum += s.half_sum[mine];
      s.bin_sum[mine] = sum;
      s.bin_count[mine] = count + s.half_count[mine];
    }
    sum = prefix(half ? 0.0 : sum);
    if ((t & 63) == 63) s.wave_sum[t >> 6] = sum;
    __syncthreads();
    sum = 0.0;
    for (int v = 0; v < kCutWaves; ++v) sum += s.wave_sum[v];
    int listed = -1, list_bin = 0x7fffffff;
    if (by_k && find_border(s, row, true, (uint32_t)r.limit(b), 0.0, listed, list_bin)) {
      cut = s.border;
      sum = kept = s.kept;
    }
    if (by_p) {
      const double goal = fmin(fmax((double)r.nucleus(b) * sum, 0x1p-200), sum);
      if (find_border(s, row, false, 0, goal, listed, list_bin)) {
        cut = s.border;
        kept = s.kept;
      }
    }
  }
  if (t != 0) return;
  cuts[slot] = RowCut{cut, kept};
  if (draws) {
    DrawRec w{};
    w.sum = kept;
    w.cut = cut;
    w.top = s.top;
    w.row = r.first(b);
    w.arg = s.arg;
    w.refused = -1;
    draws[b] = w;
  }
}

template <int SRC>
void launch(const SampleRows& r, int bits, const SegRec* rec, const Histogram* hist, RowCut* cuts, DrawRec* draws,
            hipStream_t st) {
  const int parts = (r.V + kSampleBlock - 1) / kSampleBlock;
  hipLaunchKernelGGL((sample_cut_kernel<SRC>), dim3((unsigned)((long long)r.B * (r.K + 1))), dim3(kCutThreads), 0, st, r,
                     r.segments(), parts, bits, rec, hist, cuts, draws);
}

}  // namespace

int launch_sample_cut(const SampleRows& r, int dtype, const SegRec* rec, const Histogram* hist, RowCut* cuts,
                      DrawRec* draws, hipStream_t st) {
  int bits = 45;
  while ((1LL << (62 - bits)) < (long long)r.V) --bits;
  switch (dtype) {
    case VRM_SRC_F32: launch<VRM_SRC_F32>(r, bits, rec, hist, cuts, draws, st); break;
    case VRM_SRC_F16: launch<VRM_SRC_F16>(r, bits, rec, hist, cuts, draws, st); break;
    default: launch<VRM_SRC_BF16>(r, bits, rec, hist, cuts, draws, st); break;
  }
  return launch_status("sample_cut");
}

}  // namespace vrm
