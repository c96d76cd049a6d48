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
// weights are integers in units of 2^-S, S such that V of them stay below 2^62
// (S = 45 for V up to 2^17).  Tokens below 2^-51 of the row's largest may weigh
// nothing here; where such a token would be the border nothing is cut.
//
// One workgroup has a row.  It runs each part of its code a few times at most,
// so that fetching the code is what short code saves: the pass over the row, the
// narrowing and the comparison stand here once, in loops over what they are for.
// (With a copy for each use, in 170 KB, a row of 131072 took 42 us.)
#include "vrm_sample.h"

namespace vrm {
namespace {

constexpr int kCutThreads = 1024;
constexpr int kCutWaves = kCutThreads / kWave;
constexpr int kSub = 2048;   // steps of order values
constexpr int kList = 4096;  // tokens that fit the list
constexpr int kFew = 64;     // tokens that are compared with each other

using u64 = unsigned long long;

__device__ __forceinline__ float order_logit(u64 order) {
  const uint32_t key = (uint32_t)(order >> 32);
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

template <int SRC>
__global__ void __launch_bounds__(kCutThreads)
    sample_cut_kernel(SampleRows r, int ns, int parts, int bits, const SegRec* rec, const Histogram* hist, RowCut* cuts,
                      DrawRec* draws) {
  __shared__ u64 list[kList], list_weight[kList];  // order values, weights as integers
  __shared__ u64 sub_sum[kSub];
  __shared__ uint32_t sub_count[kSub];
  __shared__ double bin_sum[kBins];
  __shared__ uint32_t bin_count[kBins];
  __shared__ u64 few[kFew], few_weight[kFew];
  __shared__ u64 wave_fixed[kCutWaves], wave_low[kCutWaves], wave_high[kCutWaves];
  __shared__ uint32_t wave_count[kCutWaves];
  __shared__ double s_before_sum, s_goal, s_row_sum;
  __shared__ u64 s_before_fixed, s_border;
  __shared__ uint32_t s_before_count, s_count;
  __shared__ int s_bin, s_fill, s_arg;
  __shared__ float s_top;

  const int slot = blockIdx.x, b = slot / (r.K + 1), i = slot % (r.K + 1);
  const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
  if (i >= r.count(b)) return;
  const float temp = r.temp(b);
  if (wave == 0) {
    float top;
    int arg;
    Scale scale;
    double sum;
    combine_segments(rec + (long long)slot * ns, ns, temp, top, arg, scale, sum);
    if (lane == 0) {
      s_top = top;
      s_arg = arg;
      s_row_sum = sum;
    }
  }
  __syncthreads();
  bool by_k, by_p;
  const bool filters = row_filters(r, b, temp, by_k, by_p) && s_arg == -2;
  u64 cut = 0;
  double kept = s_row_sum;
  if (filters) {
    using L = Logit<SRC>;
    const auto* row = row_at<SRC>(r, r.first(b) + i);
    const int V = r.V;
    const Scale scale = make_scale(s_top, temp);
    const float bins = bin_scale(scale);
    const int top_bin = bin_of(s_top, bins);
    const double unit = (double)(1ULL << bits);

    // The parts' histograms, shifted to the row's bins and scaled; the even
    // parts by the first 512 threads, the odd ones by the others.
    {
      double* part_factor = reinterpret_cast<double*>(list);
      int* part_shift = reinterpret_cast<int*>(list_weight);
      const int mine = t & (kBins - 1), half = t / kBins;
      double sum = 0.0;
      uint32_t count = 0;
      for (int p0 = 0; p0 < parts; p0 += kCutThreads) {
        __syncthreads();
        if (p0 + t < parts) {
          const float top = rec[(long long)slot * ns + (p0 + t) * 4].top;  // (of the whole part)
          const SegRec one{1.0 / (double)(1ULL << kBinBits), top, 0};
          const double factor = segment_sum(one, scale);
          part_factor[t] = factor;
          part_shift[t] = factor > 0.0 ? top_bin - bin_of(top, bins) : kBins;  // (weighs nothing: no bins)
        }
        __syncthreads();
        const int n = min(parts - p0, kCutThreads);
#pragma unroll 8
        for (int j = half; j < n; j += kCutThreads / kBins) {
          const int at = mine - part_shift[j];
          const Histogram& h = hist[(long long)slot * parts + p0 + j];
          const u64 w = h.sum[max(at, 0)];
          const uint32_t c = by_k ? h.count[max(at, 0)] : 0;
          sum += at >= 0 ? (double)w * part_factor[j] : 0.0;
          count += at >= 0 ? c : 0;
        }
      }
      double* half_sum = reinterpret_cast<double*>(sub_sum);
      if (half) {
        half_sum[mine] = sum;
        sub_count[mine] = count;
      }
      __syncthreads();
      if (!half) {
        bin_sum[mine] = sum + half_sum[mine];
        bin_count[mine] = count + sub_count[mine];
      }
      __syncthreads();
    }

    int listed = -1, list_bin = 0x7fffffff;  // the list holds `listed` tokens, all down to list_bin
#pragma unroll 1
    for (int turn = 0; turn < 2; ++turn) {
      const bool by_count = turn == 0;
      if (!(by_count ? by_k : by_p)) continue;
      __syncthreads();  // (a turn may end at any of its tests of shared values)
      const uint32_t k = (uint32_t)r.limit(b);

      // The border's bin: the first at which the running count reaches k, or the
      // running sum top_p of the whole (after a top_k: of what that keeps).
      // By one wavefront, 8 bins a lane.
      if (wave == 0) {
        constexpr int kPer = kBins / kWave;
        uint32_t c[kPer], lane_count = 0;
        double w[kPer], lane_sum = 0.0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          c[j] = bin_count[lane * kPer + j];
          w[j] = bin_sum[lane * kPer + j];
          lane_count += c[j];
          lane_sum += w[j];
        }
        uint32_t count = wave_prefix(lane_count) - lane_count;
        const double up_to = wave_prefix(lane_sum);
        double sum = lane_move<0x138, 0xf>(up_to, 0.0);  // wave_shr 1: what is before the lane
        const double total = cut ? kept : lane_value(up_to, 63);
        const double goal = fmin(fmax((double)r.nucleus(b) * total, 0x1p-200), total);
        // (The first bin of the first lane: running sums in floating point may
        // step back by a rounding.)
        const u64 here = __ballot(by_count ? count + lane_count >= k : up_to >= goal);
        const int which = here ? __ffsll(here) - 1 : -1;
        if (which < 0) {
          if (lane == 0) s_bin = kBins;
        } else if (lane == which) {
          int j = 0;
          while (j < kPer - 1 && !(by_count ? count + c[j] >= k : sum + w[j] >= goal)) {
            count += c[j];
            sum += w[j];
            ++j;
          }
          s_bin = lane * kPer + j;
          s_before_count = count;
          s_before_sum = sum;
          s_goal = goal;
        }
      }
      __syncthreads();
      uint32_t before_count = s_before_count;
      const double before = s_before_sum, goal = s_goal;
      if (s_bin == kBins) continue;
      const int bin = top_bin - s_bin;

      // Its tokens, by a pass over the row: into the list; with a top_k, whose
      // bins have counts, all tokens down to the bin where they fit, among which
      // the border of a top_p is too.  Where a bin's tokens do not fit, passes
      // narrow its order values by 11 bits each before.
      u64 low = 0, high = ~0ULL, fixed_goal = 0, before_fixed = 0;
      bool have_goal = by_count;
      if (bin < list_bin) {
        const bool all = by_count && before_count + bin_count[s_bin] <= (uint32_t)kList;
        const int last = bin, first = all ? top_bin : bin;
        const float f_low = last <= -(int)kBinMost ? -INFINITY : (float)last;
        const float f_high = first >= (int)kBinMost ? INFINITY : (float)(first + 1);
        const bool open = f_high == INFINITY;
        int shift = -1;  // -1: into the list
#pragma unroll 1
        while (true) {
          __syncthreads();
          if (t == 0) s_fill = 0;
          if (shift >= 0) {
            for (int j = t; j < kSub; j += kCutThreads) {
              sub_count[j] = 0;
              sub_sum[j] = 0;
            }
          }
          __syncthreads();
          // The pass.  Eight loads of a lane are under way at once: the
          // workgroup has its compute unit to itself and would wait for each.
          // Hits go to the list by their index alone; only a pass over an
          // interval looks at them here.
          constexpr int kVec = L::kVec, kAhead = 8, kStep = kCutThreads * kVec;
          const bool by_index = shift < 0 && low == 0;
#pragma unroll 1
          for (int base = 0; base < V; base += kAhead * kStep) {
            const int e0 = base + t * kVec;
            Unaligned16<typename L::Raw> raw[kAhead];
            if (base + kAhead * kStep <= V) {
#pragma unroll
              for (int a = 0; a < kAhead; ++a)
                raw[a] = *reinterpret_cast<const Unaligned16<typename L::Raw>*>(row + e0 + a * kStep);
            } else {
#pragma unroll
              for (int a = 0; a < kAhead; ++a) {
                const int e = e0 + a * kStep;
                if (e + kVec <= V) {
                  raw[a] = *reinterpret_cast<const Unaligned16<typename L::Raw>*>(row + e);
                } else {
#pragma unroll
                  for (int j = 0; j < kVec; ++j) raw[a].v[j] = e + j < V ? row[e + j] : (typename L::Raw)0;
                }
              }
            }
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
              uint32_t hits = 0;
#pragma unroll
              for (int e = 0; e < kVec; ++e) {
                const float y = L::value(raw[a].v[e]) * bins;
                if (y >= f_low && (open || y < f_high)) hits |= 1u << e;
              }
              while (hits) {
                const int e = e0 + a * kStep + __ffs(hits) - 1;
                hits &= hits - 1;
                if (e >= V) break;
                if (by_index) {
                  const int j = atomicAdd(&s_fill, 1);
                  if (j < kList) list[j] = (u64)e;
                  continue;
                }
                const float l = L::value(row[e]);
                const u64 o = order_value(l, e);
                if (!(l > -INFINITY) || o < low || o > high) continue;
                if (shift < 0) {
                  list[atomicAdd(&s_fill, 1)] = o;  // (there are as many as the last pass counted)
                } else {
                  const int j = (int)((high - o) >> shift);
                  atomicAdd(&sub_count[j], 1u);
                  atomicAdd(&sub_sum[j], fixed_weight(sample_weight(l, scale), unit));
                }
              }
            }
          }
          __syncthreads();
          if (shift < 0) {
            listed = s_fill;
            if (listed <= kList) {
              if (by_index) {
                // (-inf is in the last bin where that is unbounded)
                for (int j = t; j < listed; j += kCutThreads) {
                  const int e = (int)list[j];
                  const float l = L::value(row[e]);
                  list[j] = l > -INFINITY ? order_value(l, e) : 0;
                }
                __syncthreads();
              }
              break;
            }
            shift = 64 - 11;  // (by 11 bits of the order value: more than the list holds cannot be one token)
            listed = -1;
            continue;
          }
          {
            const uint32_t c0 = sub_count[2 * t], c1 = sub_count[2 * t + 1];
            const u64 w0 = sub_sum[2 * t], w1 = sub_sum[2 * t + 1];
            const uint32_t pc = wave_prefix(c0 + c1);
            const u64 pw = wave_prefix(w0 + w1);
            if (lane == 63) {
              wave_count[wave] = pc;
              wave_fixed[wave] = pw;
            }
            __syncthreads();
            uint32_t c = before_count + pc - (c0 + c1);
            u64 w = before_fixed + pw - (w0 + w1), all_weight = 0;
            for (int v = 0; v < kCutWaves; ++v) {
              if (v < wave) {
                c += wave_count[v];
                w += wave_fixed[v];
              }
              all_weight += wave_fixed[v];
            }
            if (!have_goal) {
              const double want = ceil((goal - before) * unit);
              fixed_goal = want < 1.0 ? 1 : min((u64)want, all_weight);
              have_goal = true;
            }
            const bool in0 = by_count ? c < k && c + c0 >= k : w < fixed_goal && w + w0 >= fixed_goal;
            const bool in1 =
                by_count ? c + c0 < k && c + c0 + c1 >= k : w + w0 < fixed_goal && w + w0 + w1 >= fixed_goal;
            if (t == 0) s_bin = -1;
            __syncthreads();
            if (in0 || in1) {  // (one thread)
              s_bin = 2 * t + (in0 ? 0 : 1);
              s_count = in0 ? c0 : c1;
              s_before_count = in0 ? c : c + c0;
              s_before_fixed = in0 ? w : w + w0;
            }
            __syncthreads();
          }
          if (s_bin < 0) break;  // (nothing in the bin weighs anything)
          before_count = s_before_count;
          before_fixed = s_before_fixed;
          const u64 top = high - ((u64)s_bin << shift), span = (1ULL << shift) - 1;
          low = top - low > span ? top - span : low;
          high = top;
          shift = s_count <= (uint32_t)kList ? -1 : max(0, 64 - __clzll(high - low) - 11);
        }
        list_bin = all ? bin : 0x7fffffff;
        if (listed < 0) continue;
        for (int j = t; j < listed; j += kCutThreads)
          list_weight[j] = fixed_weight(sample_weight(order_logit(list[j]), scale), unit);
        __syncthreads();
      }

      // Narrow the listed tokens of the bin that are within low .. high.
      uint32_t n = 0;
#pragma unroll 1
      while (true) {
        // How many there are, what they weigh, and the interval that they take.
        u64 a = ~0ULL, z = 0, sum = 0;
        uint32_t count = 0;
        for (int j = t; j < listed; j += kCutThreads) {
          const u64 o = list[j];
          if (o >= low && o <= high && bin_of(order_logit(o), bins) == bin) {
            ++count;
            sum += list_weight[j];
            a = min(a, o);
            z = max(z, o);
          }
        }
        count = wave_sum(count);
        sum = wave_sum(sum);
        a = wave_min(a, ~0ULL);
        z = wave_max(z, 0ULL);
        if (lane == 0) {
          wave_count[wave] = count;
          wave_fixed[wave] = sum;
          wave_low[wave] = a;
          wave_high[wave] = z;
        }
        for (int j = t; j < kSub; j += kCutThreads) {
          sub_count[j] = 0;
          sub_sum[j] = 0;
        }
        if (t == 0) s_fill = 0;
        __syncthreads();
        n = 0;
        sum = 0;
        for (int v = 0; v < kCutWaves; ++v) {
          n += wave_count[v];
          sum += wave_fixed[v];
          a = min(a, wave_low[v]);
          z = max(z, wave_high[v]);
        }
        if (!have_goal) {
          // The part of the goal that is within the bin, at most what the bin's
          // integers add up to (they are rounded apart from the histograms').
          const double want = ceil((goal - before) * unit);
          fixed_goal = want < 1.0 ? 1 : min((u64)want, sum);
          have_goal = true;
          if (sum == 0) n = 0;
        }
        if (n <= (uint32_t)kFew) break;
        low = a;
        high = z;
        const int shift = max(0, 64 - __clzll(high - low) - 11);  // (high - low) >> shift is below 2048
        for (int j = t; j < listed; j += kCutThreads) {
          const u64 o = list[j];
          if (o >= low && o <= high && bin_of(order_logit(o), bins) == bin) {
            atomicAdd(&sub_count[(high - o) >> shift], 1u);
            atomicAdd(&sub_sum[(high - o) >> shift], list_weight[j]);
          }
        }
        __syncthreads();
        const uint32_t c0 = sub_count[2 * t], c1 = sub_count[2 * t + 1];
        const u64 w0 = sub_sum[2 * t], w1 = sub_sum[2 * t + 1];
        const uint32_t pc = wave_prefix(c0 + c1);
        const u64 pw = wave_prefix(w0 + w1);
        if (lane == 63) {
          wave_count[wave] = pc;
          wave_fixed[wave] = pw;
        }
        __syncthreads();
        uint32_t c = before_count + pc - (c0 + c1);
        u64 w = before_fixed + pw - (w0 + w1);
        for (int v = 0; v < wave; ++v) {
          c += wave_count[v];
          w += wave_fixed[v];
        }
        const bool in0 = by_count ? c < k && c + c0 >= k : w < fixed_goal && w + w0 >= fixed_goal;
        const bool in1 = by_count ? c + c0 < k && c + c0 + c1 >= k : w + w0 < fixed_goal && w + w0 + w1 >= fixed_goal;
        if (in0 || in1) {  // (one thread: the interval has the border)
          s_bin = 2 * t + (in0 ? 0 : 1);
          s_before_count = in0 ? c : c + c0;
          s_before_fixed = in0 ? w : w + w0;
        }
        __syncthreads();
        before_count = s_before_count;
        before_fixed = s_before_fixed;
        const u64 top = high - ((u64)s_bin << shift), span = (1ULL << shift) - 1;
        low = top - low > span ? top - span : low;
        high = top;
      }
      if (n == 0) continue;  // (the same for every thread)
      // The few that are left, each against the others.
      for (int j = t; j < listed; j += kCutThreads) {
        const u64 o = list[j];
        if (o >= low && o <= high && bin_of(order_logit(o), bins) == bin) {
          const int f = atomicAdd(&s_fill, 1);
          few[f] = o;
          few_weight[f] = list_weight[j];
        }
      }
      __syncthreads();
      if (t < (int)n) {
        const u64 o = few[t], w = few_weight[t];
        uint32_t c = before_count;
        u64 up_to = before_fixed;
        for (uint32_t j = 0; j < n; ++j) {
          if (few[j] > o) {
            ++c;
            up_to += few_weight[j];
          }
        }
        if (by_count ? c + 1 == k : up_to < fixed_goal && up_to + w >= fixed_goal) {  // (one of them)
          s_border = o;
          s_before_fixed = up_to + w;
        }
      }
      __syncthreads();
      cut = s_border;
      kept = before + (double)s_before_fixed / unit;
      __syncthreads();
    }
  }
  if (t != 0) return;
  cuts[slot] = RowCut{cut, kept};
  if (draws) {
    DrawRec w{};
    w.sum = kept;
    w.cut = cut;
    w.top = s_top;
    w.row = r.first(b);
    w.arg = s_arg;
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
