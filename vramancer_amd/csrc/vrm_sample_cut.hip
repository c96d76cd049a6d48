// Which tokens of a row stay under top_k and top_p.
//
// Tokens are in the order (logit descending, index ascending).  top_k keeps the
// first k; top_p the shortest prefix of those whose weights reach top_p times
// the sum of theirs.  Either is a border in that order, and nothing is sorted to
// find it: a pass over the row counts tokens and adds weights into 2048 bins,
// equal steps of the logarithm of the weight, the border's bin is found by a
// prefix sum over them, and only that bin's tokens are looked at further, by
// bins of their order values, until 64 are left, which are compared with each
// other.
//
// Weights are added as integers, w 2^S rounded, S such that V of them stay
// below 2^63 (S = 45 for V up to 2^18): sums do not depend on the order of the
// atomics, and are within V 2^-(S + 1) of the exact ones at the very worst.
// Tokens below 2^-(S + 1) of the row's largest weigh nothing here; where such a
// token would be the border nothing is cut.
#include "vrm_sample.h"

namespace vrm {
namespace {

constexpr int kCutThreads = 1024;
constexpr int kCutWaves = kCutThreads / kWave;
constexpr int kBins = 2048;
constexpr int kList = 2048;  // tokens of a bin that fit in LDS
constexpr int kFew = 64;     // tokens that are compared with each other

using u64 = unsigned long long;

struct CutShared {
  u64 bin_sum[kBins];   // by weight
  u64 sub_sum[kBins];   // by order value, within a bin
  u64 list_order[kList];
  u64 list_sum[kList];
  uint32_t bin_count[kBins];
  uint32_t sub_count[kBins];
  u64 few_order[kFew];
  u64 few_sum[kFew];
  u64 wave_sum[kCutWaves];
  uint32_t wave_count[kCutWaves];
  u64 low, high;        // order values of the border's interval
  u64 before_sum;       // of the tokens before the border's bin
  u64 border, kept;     // the answer
  uint32_t before_count, count;
  int bin, fill;
  ChunkRec row;
  double row_sum;
};

// A row as the passes see it.
template <int SRC>
struct Row {
  const typename Logit<SRC>::Raw* at;
  int V;
  float top;
  double c;
  float step;   // bins per unit of logit
  double unit;  // 2^S

  __device__ __forceinline__ int bin(float l) const {  // monotone in l; kBins - 1: weighs nothing
    if (l == top) return 0;
    return (int)fminf((top - l) * step, (float)(kBins - 1));  // (a NaN is the last bin too)
  }
  __device__ __forceinline__ u64 weight(float l) const {
    const double w = fma(sample_weight(l, top, c), unit, 4503599627370496.0);  // 2^52: rounds to an integer
    return (u64)__double_as_longlong(w) & 0xfffffffffffffULL;
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    constexpr int kVec = Logit<SRC>::kVec;
    for (int e0 = threadIdx.x * kVec; e0 < V; e0 += kCutThreads * kVec) {
      float x[kVec];
      load_vec<SRC>(at, e0, V, x);
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (x[e] > -INFINITY) f(x[e], e0 + e);
    }
  }
};

__device__ __forceinline__ u64 prefix64(u64 v) {
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) {
    const u64 o = __shfl_up(v, m);
    if ((int)(threadIdx.x & 63) >= m) v += o;
  }
  return v;
}
__device__ __forceinline__ uint32_t prefix32(uint32_t v) {
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) {
    const uint32_t o = __shfl_up(v, m);
    if ((int)(threadIdx.x & 63) >= m) v += o;
  }
  return v;
}

// The bin in which the running count reaches `k` (by_count) or the running sum
// reaches `goal`, both after what s.before_* holds; -1 if none.  Leaves the bin
// in s.bin, its count in s.count and what is before it added to s.before_*.
__device__ __forceinline__ void find_bin(CutShared& s, const uint32_t* count, const u64* sum, bool by_count, uint32_t k,
                                         u64 goal) {
  const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
  const uint32_t c0 = count[2 * t], c1 = count[2 * t + 1];
  const u64 w0 = sum[2 * t], w1 = sum[2 * t + 1];
  const uint32_t rc = prefix32(c0 + c1);
  const u64 rw = prefix64(w0 + w1);
  if (lane == 63) {
    s.wave_count[wave] = rc;
    s.wave_sum[wave] = rw;
  }
  const uint32_t c_before = s.before_count;
  const u64 w_before = s.before_sum;
  if (t == 0) s.bin = -1;
  __syncthreads();
  uint32_t c = c_before + rc - (c0 + c1);
  u64 w = w_before + rw - (w0 + w1);
  for (int v = 0; v < wave; ++v) {
    c += s.wave_count[v];
    w += s.wave_sum[v];
  }
  const auto hit = [&](uint32_t cb, u64 wb, uint32_t cn, u64 wn) {
    return by_count ? cb < k && cb + cn >= k : wb < goal && wb + wn >= goal;
  };
  __syncthreads();
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
    s.count = count[at];
    s.before_count = c;
    s.before_sum = w;
  }
  __syncthreads();
}

// The border by count (the k-th token) or by sum (the first token with which
// the sum reaches goal): s.border its order value, s.kept the sum up to it.
// False where the border would be among tokens that weigh nothing.
template <int SRC>
__device__ bool find_border(CutShared& s, const Row<SRC>& row, bool by_count, uint32_t k, u64 goal) {
  const int t = threadIdx.x;
  __syncthreads();
  if (t == 0) {
    s.before_count = 0;
    s.before_sum = 0;
  }
  __syncthreads();
  find_bin(s, s.bin_count, s.bin_sum, by_count, k, goal);
  const int bin = s.bin;
  if (bin < 0) return false;
  u64 low = 0, high = ~0ULL;
  bool listed = false;
  int in_list = 0;
  // f(order value, weight) of the tokens of the bin that are within the interval
  const auto each = [&](auto f) {
    if (listed) {
      for (int j = t; j < in_list; j += kCutThreads) {
        const u64 o = s.list_order[j];
        if (o >= low && o <= high) f(o, [&] { return s.list_sum[j]; });
      }
    } else {
      row.each([&](float l, int i) {
        if (row.bin(l) != bin) return;
        const u64 o = order_value(l, i);
        if (o >= low && o <= high) f(o, [&] { return row.weight(l); });
      });
    }
  };
  while (true) {
    const uint32_t n = s.count;
    __syncthreads();
    if (t == 0) {
      s.fill = 0;
      s.low = ~0ULL;
      s.high = 0;
    }
    __syncthreads();
    if (n <= (uint32_t)kFew) break;
    if (!listed && n <= (uint32_t)kList) {
      each([&](u64 o, auto w) {
        const int j = atomicAdd(&s.fill, 1);
        s.list_order[j] = o;
        s.list_sum[j] = w();
      });
      __syncthreads();
      listed = true;
      in_list = n;
    }
    // The interval that the tokens really take, and 2048 steps of it.
    u64 a = ~0ULL, z = 0;
    each([&](u64 o, auto) {
      a = min(a, o);
      z = max(z, o);
    });
    if (z) {
      atomicMin(&s.low, a);
      atomicMax(&s.high, z);
    }
    for (int j = t; j < kBins; j += kCutThreads) {
      s.sub_count[j] = 0;
      s.sub_sum[j] = 0;
    }
    __syncthreads();
    low = s.low;
    high = s.high;
    int shift = 0;
    while (((high - low) >> shift) >= (u64)kBins) ++shift;
    each([&](u64 o, auto w) {
      const int j = (int)((high - o) >> shift);
      atomicAdd(&s.sub_count[j], 1u);
      atomicAdd(&s.sub_sum[j], w());
    });
    __syncthreads();
    find_bin(s, s.sub_count, s.sub_sum, by_count, k, goal);
    const u64 j = s.bin;  // (there is one: the bin as a whole has the border)
    const u64 top = high - (j << shift);
    const u64 span = (1ULL << shift) - 1;
    low = top - low > span ? top - span : low;
    high = top;
  }
  each([&](u64 o, auto w) {
    const int j = atomicAdd(&s.fill, 1);
    s.few_order[j] = o;
    s.few_sum[j] = w();
  });
  __syncthreads();
  const int n = s.fill;
  if (t < n) {
    const u64 mine = s.few_order[t], w = s.few_sum[t];
    uint32_t c = s.before_count;
    u64 before = s.before_sum;
    for (int j = 0; j < n; ++j) {
      if (s.few_order[j] > mine) {
        ++c;
        before += s.few_sum[j];
      }
    }
    if (by_count ? c + 1 == k : before < goal && before + w >= goal) {  // (one of them)
      s.border = mine;
      s.kept = before + w;
    }
  }
  __syncthreads();
  return true;
}

template <int SRC>
__global__ void __launch_bounds__(kCutThreads)
    sample_cut_kernel(SampleRows r, int nc, int bits, const ChunkRec* rec, RowCut* cuts) {
  __shared__ CutShared s;
  const int slot = blockIdx.x, b = slot / (r.K + 1), i = slot % (r.K + 1), t = threadIdx.x;
  if (i >= r.count(b)) return;
  const float temp = r.temp(b);
  const bool greedy = !(temp > 0.0f);
  const double c = greedy ? 0.0 : sample_scale(temp);
  if (t < kWave) {
    float top;
    double sum;
    int arg;
    combine_chunks(rec + (long long)slot * nc, nc, c, top, sum, arg);
    if (t == 0) {
      s.row.top = top;
      s.row_sum = greedy ? 1.0 : sum;
    }
  }
  __syncthreads();
  const int k = r.limit(b);
  const float p = r.nucleus(b);
  const bool by_k = k > 0 && k < r.V, by_p = p < 1.0f;
  const float top = s.row.top;
  if (greedy || top == -INFINITY || (!by_k && !by_p)) {
    if (t == 0) cuts[slot] = RowCut{0, s.row_sum};
    return;
  }
  Row<SRC> row;
  row.at = row_at<SRC>(r, r.first(b) + i);
  row.V = r.V;
  row.top = top;
  row.c = c;
  row.step = (float)fmin(c * (kBins - 1) / (bits + 1), 3.0e38);
  row.unit = (double)(1ULL << bits);
  for (int j = t; j < kBins; j += kCutThreads) {
    s.bin_count[j] = 0;
    s.bin_sum[j] = 0;
  }
  __syncthreads();
  row.each([&](float l, int) {
    const int j = row.bin(l);
    if (j == kBins - 1) return;
    atomicAdd(&s.bin_count[j], 1u);
    atomicAdd(&s.bin_sum[j], row.weight(l));
  });
  __syncthreads();
  // The sum of all: by the bins.
  u64 total;
  {
    const u64 w = prefix64(s.bin_sum[2 * t] + s.bin_sum[2 * t + 1]);
    if ((t & 63) == 63) s.wave_sum[t >> 6] = w;
    __syncthreads();
    total = 0;
    for (int v = 0; v < kCutWaves; ++v) total += s.wave_sum[v];
  }
  u64 cut = 0, kept = total;
  if (by_k && find_border(s, row, true, (uint32_t)k, 0)) {
    cut = s.border;
    kept = s.kept;
  }
  if (by_p) {
    const double want = ceil((double)fmaxf(p, 0.0f) * (double)kept);
    const u64 goal = want < 1.0 ? 1 : min((u64)want, kept);
    if (find_border(s, row, false, 0, goal)) {
      cut = s.border;
      kept = s.kept;
    }
  }
  if (t == 0) cuts[slot] = RowCut{cut, cut ? (double)kept / row.unit : s.row_sum};
}

template <int SRC>
void launch(const SampleRows& r, int nc, int bits, const ChunkRec* rec, RowCut* cuts, hipStream_t st) {
  hipLaunchKernelGGL((sample_cut_kernel<SRC>), dim3((unsigned)((long long)r.B * (r.K + 1))), dim3(kCutThreads), 0, st, r,
                     nc, bits, rec, cuts);
}

}  // namespace

int launch_sample_cut(const SampleRows& r, int dtype, int nc, const ChunkRec* rec, RowCut* cuts, hipStream_t st) {
  int bits = 63;
  while (bits > 45 || ((1LL << (63 - bits)) < (long long)r.V)) --bits;
  switch (dtype) {
    case VRM_SRC_F32: launch<VRM_SRC_F32>(r, nc, bits, rec, cuts, st); break;
    case VRM_SRC_F16: launch<VRM_SRC_F16>(r, nc, bits, rec, cuts, st); break;
    default: launch<VRM_SRC_BF16>(r, nc, bits, rec, cuts, st); break;
  }
  return launch_status("sample_cut");
}

}  // namespace vrm
