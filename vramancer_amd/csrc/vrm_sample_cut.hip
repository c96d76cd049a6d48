// Which tokens of a row stay under top_k and top_p.
//
// Tokens are in the order (logit descending, index ascending).  top_k keeps the
// first k; top_p the shortest prefix of those whose weights reach top_p times
// the sum of theirs.  Either is a border in that order, and nothing is sorted to
// find it:
//   sample_bins_kernel     adds up the histograms of the row's parts, made with
//                          its sums, and finds the bins that hold the borders
//   sample_collect_kernel  lists those bins' tokens (a wavefront per segment)
//   sample_border_kernel   narrows the list down by bins of order values until
//                          64 tokens are left, which it compares with each other
// Rows of up to 8192 logits (one part) go through all of it, their histogram
// included, in one launch: sample_short_kernel.
// A draw that needs nothing else comes out of the same launches: the second one
// adds up what the segments hold above the border's bins, the third adds the
// listed tokens that stay and picks.
// Three launches where one workgroup per row could do all of it: to look through
// its row alone took that workgroup 7 us (131072 float32) to 12 (152000 bf16) at
// 16 to 24 bytes a cycle, and 512 rows 28; a launch of the whole chip takes as
// long for 64 rows as for one.
//
// Counts and sums do not depend on the order in which tokens are listed: the
// parts' sums are integers, added in 64-bit floats part by part; among listed
// tokens weights are integers in units of 2^-S, S such that V of them stay below
// 2^62 (S = 45 for V up to 2^17).  Tokens below 2^-49 of the row's largest may
// count and weigh nothing in the histograms: top_p's sums leave them out, and a
// top_k that reaches them has its border found among all tokens by their order.
//
// A workgroup of the first and the last kernel runs each part of its code a few
// times at most, so that fetching it is what short code saves (170 KB, with a
// copy of the narrowing for each use, took 42 us for a row of 131072).
#include "vrm_sample.h"

namespace vrm {
namespace {

constexpr int kCutThreads = 512;  // = kBins
constexpr int kFew = 64;           // tokens that are compared with each other
constexpr int kPartsAhead = 24;
constexpr int kShortListed = 2048;  // tokens of a short row's list
static_assert(2 * kCutThreads >= kDrawSegments, "a sum for each segment");
// Down to here every token is counted in its bin, since it is at least one as an
// integer of its part's histogram: 488 tenths and one for the roundings of two
// products are 2^-49 of the row's largest, kBinBits being 49.
constexpr int kSureBins = 488;
constexpr int kNoBins = 1 << 30;  // the shift of a part that weighs nothing
constexpr int kLeastBits = 1100;  // a factor of 2^-1100 of the row's largest is 0

using u64 = unsigned long long;

// Whether a logit's bin, floor of the clamped product with `bins`, is within
// last .. first, as two comparisons.
struct BinRange {
  float low, high;
  __device__ __forceinline__ BinRange(int last, int first) {
    low = last <= -(int)kBinMost ? -INFINITY : (float)last;
    high = first >= (int)kBinMost ? NAN : (float)(first + 1);
  }
  __device__ __forceinline__ bool holds(float y) const { return y >= low && !(y >= high); }
};

// The first bin at which the running count reaches k (by_count) or the running
// sum goal, and what is before it: by one wavefront, 8 bins a lane.  kBins if
// there is none.  (The first of the first lane: running sums in floating point
// may step back by a rounding.)
struct BinScan {
  static constexpr int kPer = kBins / kWave;
  uint32_t c[kPer], count, lane_count;
  double w[kPer], sum, up_to, total;

  __device__ __forceinline__ BinScan(const uint32_t* counts, const double* sums) {
    const int lane = threadIdx.x & 63;
    lane_count = 0;
    double lane_sum = 0.0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      c[j] = counts[lane * kPer + j];
      w[j] = sums[lane * kPer + j];
      lane_count += c[j];
      lane_sum += w[j];
    }
    count = wave_prefix(lane_count) - lane_count;
    up_to = wave_prefix(lane_sum);
    sum = lane_move<0x138, 0xf>(up_to, 0.0);  // wave_shr 1: what is before the lane
    total = lane_value(up_to, 63);
  }
  __device__ __forceinline__ uint32_t all() const { return lane_value(count + lane_count, kWave - 1); }
  __device__ __forceinline__ int find(bool by_count, uint32_t k, double goal, uint32_t& before_count,
                                      double& before_sum, uint32_t& bin_count, double& bin_sum) const {
    const u64 here = __ballot(by_count ? count + lane_count >= k : up_to >= goal);
    if (!here) return kBins;
    const int which = __ffsll(here) - 1;
    uint32_t n = count, nb = c[0];
    double s = sum, sb = w[0];
    int at = 0;
#pragma unroll
    for (int j = 0; j < kPer - 1; ++j) {
      const bool next = at == j && !(by_count ? n + c[j] >= k : s + w[j] >= goal);
      n = next ? n + c[j] : n;
      s = next ? s + w[j] : s;
      nb = next ? c[j + 1] : nb;
      sb = next ? w[j + 1] : sb;
      at = next ? j + 1 : at;
    }
    before_count = lane_value(n, which);
    before_sum = lane_value(s, which);
    bin_count = lane_value(nb, which);
    bin_sum = lane_value(sb, which);
    return which * kPer + lane_value(at, which);
  }
};

// The bins of a row's borders, by one wavefront.
__device__ __forceinline__ void plan_cut(CutPlan& plan, const BinScan& scan, const SampleRows& r, int b, int top_bin,
                                         bool by_k, bool by_p) {
  const double p = fmax((double)r.nucleus(b), 0.0);
  plan.k = by_k ? r.limit(b) : 0;
  double least = scan.total, most = scan.total;  // what top_p takes its part of
  int last = kBins - 1;                          // the last bin that it can end in
  if (by_k) {
    uint32_t n_before, n_bin;
    double s_before, s_bin;
    const int at = scan.find(true, (uint32_t)plan.k, 0.0, n_before, s_before, n_bin, s_bin);
    if (at >= kSureBins) {
      // The k-th token weighs so little that some before it may not be counted.
      // A top_p ends before it; without one all tokens down to a bin that has the
      // border at the latest are listed (those that weigh anything, unless the
      // caller finds one), and the border found by order alone.
      if (by_p) {
        plan.k = 0;
      } else {
        plan.deep = at < kBins ? kBelow : kWhole;
        plan.all_listed = 1;
        plan.k_first = plan.list_first = top_bin;
        plan.k_last = plan.list_last = top_bin - (at < kBins ? at : 10 * kLeastBits + 2);
      }
    } else {
      plan.k_first = plan.k_last = top_bin - at;
      plan.k_count = n_before;
      plan.k_before = s_before;
      if (n_before + n_bin <= (uint32_t)kListed) {
        // All tokens down to this bin are listed: the border of a top_p is
        // among them.
        plan.list_first = top_bin;
        plan.list_last = top_bin - at;
        plan.p_first = top_bin;
        plan.p_last = top_bin - at;
        plan.p_before = 0.0;
        plan.by_p = by_p;
        plan.all_listed = 1;
        by_p = false;
      } else {
        plan.list_first = plan.list_last = top_bin - at;
      }
      least = s_before;
      most = s_before + s_bin;
      last = at;
    }
  }
  plan.filters = plan.k > 0;
  plan.total = scan.total;
  if (by_p) {
    // One bin; after a top_k, whose sum lies between two values still, what the
    // border of the smaller and of the larger one enclose.
    uint32_t n;
    double s, before, unused;
    const int from = scan.find(false, 0, fmin(fmax(p * least, 0x1p-200), least), n, before, n, s);
    const int to = scan.find(false, 0, fmin(fmax(p * most, 0x1p-200), most), n, unused, n, s);
    if (from < kBins) {
      plan.by_p = 1;
      plan.filters = 1;
      plan.p_first = top_bin - from;
      plan.p_last = top_bin - min(to, last);
      plan.p_before = before;
      if (plan.k > 0) {
        plan.also_first = plan.p_first;
        plan.also_last = plan.p_last;
        plan.also = 1;
      } else {
        plan.list_first = plan.p_first;
        plan.list_last = plan.p_last;
      }
    }
  }
}

// One workgroup per row.
__global__ void __launch_bounds__(kCutThreads)
    sample_bins_kernel(SampleRows r, int ns, int parts, const SegRec* rec, const Histogram* hist, CutPlan* plans) {
  __shared__ double part_factor[kCutThreads], bin_sum[kBins];
  __shared__ int part_shift[kCutThreads];
  __shared__ uint32_t bin_count[kBins];
  __shared__ double s_row_sum;
  __shared__ int s_arg;
  __shared__ float s_top;
  const int slot = blockIdx.x, b = slot / (r.K + 1), i = slot % (r.K + 1);
  const int t = threadIdx.x, lane = t & 63;
  if (i >= r.count(b)) return;
  const float temp = r.temp(b);
  if (t < kWave) {
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
  CutPlan plan{};
  plan.top = s_top;
  plan.arg = s_arg;
  plan.kept = s_row_sum;
  if (!filters) {
    if (t == 0) plans[slot] = plan;
    return;
  }
  // The parts' histograms, shifted to the row's bins and scaled; a bin a thread.
  const Scale scale = make_scale(s_top, temp);
  const float bins = bin_scale(scale);
  const int top_bin = bin_of(s_top, bins);
  double sum = 0.0;
  uint32_t count = 0;
  for (int p0 = 0; p0 < parts; p0 += kCutThreads) {
    __syncthreads();
    if (p0 + t < parts) {
      const float top = rec[(long long)slot * ns + (p0 + t) * 4].top;  // (of the whole part)
      const SegRec one{1.0 / (double)(1ULL << kBinBits), top, 0};
      const double factor = segment_sum(one, scale);
      part_factor[t] = factor;
      part_shift[t] = factor > 0.0 ? top_bin - bin_of(top, bins) : kNoBins;
    }
    __syncthreads();
    const int n = min(parts - p0, kCutThreads);
    // (24 loads under way at once)
#pragma unroll 1
    for (int j0 = 0; j0 < n; j0 += kPartsAhead) {
      u64 w[kPartsAhead];
      uint32_t c[kPartsAhead];
#pragma unroll
      for (int j = 0; j < kPartsAhead; ++j) {
        const int p = min(j0 + j, n - 1);
        const Histogram& h = hist[(long long)slot * parts + p0 + p];
        const int at = max(t - part_shift[p], 0);
        w[j] = h.sum[at];
        c[j] = by_k ? h.count[at] : 0;
      }
#pragma unroll
      for (int j = 0; j < kPartsAhead; ++j) {
        const int p = j0 + j;
        if (p >= n || t < part_shift[p]) continue;
        sum += (double)w[j] * part_factor[p];
        count += c[j];
      }
    }
  }
  bin_sum[t] = sum;
  bin_count[t] = count;
  __syncthreads();
  if (t >= kWave) return;
  const BinScan scan(bin_count, bin_sum);
  plan_cut(plan, scan, r, b, top_bin, by_k, by_p);
  if (lane == 0) plans[slot] = plan;
  if (plan.deep != kWhole || parts > kCutThreads) return;
  // The border of top_k lies past these bins (a few tokens far above the others,
  // a low temperature).  A part's histogram counts from its own maximum on, so
  // that the parts without those tokens still tell a bin down to which there are
  // k tokens at least: what is listed down to it has the border.  Counts of
  // further bins, 512 at a time, from where there are any.  (The draw of a row of
  // 152000 with top_k 50 and a token 50 bits above the others: 49 us; 104 with
  // everything listed, which overflows the list.)
  uint32_t counted = scan.all();
#pragma unroll 1
  for (int from = kBins;; from += kBins) {
    int next = kNoBins;
    for (int p = lane; p < parts; p += kWave)
      if (part_shift[p] + kBins > from) next = min(next, max(part_shift[p], from));
    from = wave_min(next, kNoBins);
    if (from >= 10 * kLeastBits) return;
    uint32_t c[BinScan::kPer] = {};
#pragma unroll 2
    for (int p = 0; p < parts; ++p) {
      const int at = from + lane * BinScan::kPer - part_shift[p];
      const uint32_t* counts = hist[(long long)slot * parts + p].count;
#pragma unroll
      for (int j = 0; j < BinScan::kPer; ++j)
        if (at + j >= 0 && at + j < kBins) c[j] += counts[at + j];
    }
#pragma unroll
    for (int j = 0; j < BinScan::kPer; ++j) bin_count[lane * BinScan::kPer + j] = c[j];
    const BinScan more(bin_count, bin_sum);
    uint32_t before, in_bin;
    double unused;
    const int at = more.find(true, (uint32_t)plan.k - counted, 0.0, before, unused, in_bin, unused);
    if (at < kBins) {
      plan.deep = kBelow;
      plan.k_last = plan.list_last = top_bin - from - at;
      if (lane == 0) plans[slot] = plan;
      return;
    }
    counted += more.all();
  }
}

// Which of a lane's logits are in the bins to list.
__device__ __forceinline__ uint32_t plan_hits(const CutPlan& plan, const float* x, float bins) {
  const BinRange main(plan.list_last, plan.list_first), second(plan.also_last, plan.also_first);
  const bool two = plan.also != 0;
  uint32_t hits = 0;
#pragma unroll
  for (int e = 0; e < kSamplePer; ++e) {
    const float y = x[e] * bins;
    if ((main.holds(y) || (two && second.holds(y))) && x[e] > -INFINITY) hits |= 1u << e;
  }
  return hits;
}

// A wavefront per segment: the tokens of the bins of the plan go to the row's
// list, by their order values; plan.listed counts them, and only kListed fit.
// With MASS, mass takes the weights of the segment's tokens above the first of
// those bins, which stay whatever the border.  (The segment is under way before
// the plan that says whether it is needed.  Five wavefronts a SIMD, as the
// histograms.)
template <int SRC, bool MASS>
__global__ void __launch_bounds__(kSampleThreads, 5)
    sample_collect_kernel(SampleRows r, int ns, int blocks, CutPlan* plans, u64* lists, double* mass) {
  __shared__ int wave_hits[kSampleThreads / kWave], base;
  const int wave = threadIdx.x >> 6, slot = blockIdx.x / blocks, seg = (blockIdx.x % blocks) * 4 + wave;
  const int b = slot / (r.K + 1), i = slot % (r.K + 1);
  if (i >= r.count(b)) return;
  CutPlan& plan = plans[slot];
  constexpr int kVec = Logit<SRC>::kVec;
  const auto* row = row_at<SRC>(r, r.first(b) + i);
  float x[kSamplePer];
  load_segment<SRC>(row, seg, r.V, x);
  if (!plan.filters) return;
  const Scale scale = make_scale(plan.top, r.temp(b));
  const float bins = bin_scale(scale);
  uint32_t hits = plan_hits(plan, x, bins);
  const int mine = __popc(hits);
  const int up_to = wave_prefix(mine), all = lane_value(up_to, 63);
  // (One addition to the row's counter for a workgroup: with one for each
  // wavefront 76 of a row waited for each other.)
  if ((threadIdx.x & 63) == 0) wave_hits[wave] = all;
  __syncthreads();
  int at = up_to - mine, block = 0;
  for (int v = 0; v < kSampleThreads / kWave; ++v) {
    if (v < wave) at += wave_hits[v];
    block += wave_hits[v];
  }
  if (block != 0) {  // (the same for every thread)
    if (threadIdx.x == 0) base = atomicAdd(&plan.listed, block);
    __syncthreads();
  }
  if (all != 0) {
    at += base;
    u64* list = lists + (long long)slot * kListed;
    // (A lane has three at most, mostly: their logits are read again, since
    // registers have no index.)
#pragma unroll 1
    for (; hits && at < kListed; hits &= hits - 1, ++at) {
      const int bit = __ffs(hits) - 1, e = segment_element<SRC>(seg, bit / kVec) + bit % kVec;
      list[at] = order_value(Logit<SRC>::value(row[e]), e);
    }
  }
  if constexpr (!MASS) return;
  if (plan.all_listed) return;
  const float above = plan.by_p ? BinRange(0, plan.p_first).high : BinRange(0, plan.k_first).high;
  double s = 0.0;
#pragma unroll
  for (int e = 0; e < kSamplePer; e += 8) {
    bool in[8], any = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      in[j] = x[e + j] * bins >= above;
      any |= in[j];
    }
    if (!__any(any)) continue;
    double w[8];
    sample_weights<8>(x + e, scale, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) s += in[j] ? w[j] : 0.0;
  }
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0 && seg < ns) mass[(long long)slot * ns + seg] = s;
}

// Order values without the bits that are the same for all of a row: the zeros
// that end 16-bit logits as float32 and the ones above an index of V.  Ten bits
// of the distance between two of them then tell equal logits apart by index:
// 775 bf16 logits of a bin are down to 64 in one step of the narrowing, where
// plain order values took two (the kernel 18.2 us for 64 rows of 152000, 15.4 with
// this and the weights worked out once).
template <int SRC>
struct Packed {
  static constexpr int kZeros = Logit<SRC>::kZeros;
  int index_bits;
  uint32_t mask;

  __device__ __forceinline__ explicit Packed(int V) : index_bits(32 - __clz(V)), mask((1u << index_bits) - 1) {}
  __device__ __forceinline__ int bits() const { return 32 - kZeros + index_bits; }
  __device__ __forceinline__ u64 pack(u64 order) const {
    return (order >> (32 + kZeros)) << index_bits | ((uint32_t)order & mask);
  }
  __device__ __forceinline__ u64 order(u64 p) const {
    uint32_t key = (uint32_t)(p >> index_bits) << kZeros;
    if (!(key & 0x80000000u)) key |= (1u << kZeros) - 1;  // (of negative logits the bits are inverted)
    return (u64)key << 32 | ((uint32_t)p & mask) | (uint32_t)~mask;
  }
  __device__ __forceinline__ float logit(u64 p) const { return order_logit(order(p)); }
  __device__ __forceinline__ int index(u64 p) const { return (int)(~(uint32_t)p & mask); }
};

// What a workgroup of THREADS needs to find the borders of a row whose list has
// up to LISTED tokens.
template <int SRC, int THREADS, int LISTED>
struct CutShared {
  static constexpr int kThreads = THREADS, kWaves = THREADS / kWave;
  static constexpr int kSub = 2 * THREADS, kSubBits = 31 - __builtin_clz(kSub);  // steps of order values
  u64 sub_sum[kSub];
  uint32_t sub_count[kSub];
  ulonglong2 few[kFew];  // (order, weight)
  u64 wave_fixed[kWaves], wave_low[kWaves], wave_high[kWaves];
  u64 before_fixed_, border_;
  uint32_t wave_count[kWaves];
  uint32_t before_count_, count_;
  int bin_, fill_;
  PickShared<SRC> pick;
  // Packed order values, weights as integers; last, so that the others are within
  // the 16 bits of an LDS instruction's offset.
  u64 list[LISTED], weight[LISTED];

  __device__ __forceinline__ void put(int at, u64 order, const Packed<SRC>& packed, const Scale& scale, double unit) {
    list[at] = packed.pack(order);
    weight[at] = fixed_weight(sample_weight(order_logit(order), scale), unit);
  }
};

// The borders of a row, and where tokens are asked for the draw, by a workgroup.
// `listing` tokens are those of the plan's bins: with LISTS in `lists` (thread t
// has one of them, ahead), otherwise in sh.list already; more than LISTED are in
// neither.  With LISTS mass has the sums of sample_collect_kernel.
template <bool LISTS, int SRC, int THREADS, int LISTED>
__device__ __forceinline__ void find_border(CutShared<SRC, THREADS, LISTED>& sh, const SampleRows& r, int ns, int bits,
                                            const SegRec* rec, const CutPlan& plan, int listing, const u64* lists,
                                            u64 ahead, RowCut* cuts, DrawRec* draws, double* mass, float u,
                                            long long* tokens) {
  constexpr int kThreads = THREADS, kWaves = THREADS / kWave;
  const int slot = blockIdx.x, b = slot / (r.K + 1), i = slot % (r.K + 1);
  const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
  const Packed<SRC> packed(r.V);
  u64 border = 0;  // packed; 0: no cut
  double kept = plan.kept;
  bool fits = true, of_p = false;  // whether the cut is top_p's
  int listed = 0;
  if (plan.filters) {
    using L = Logit<SRC>;
    const auto* row = row_at<SRC>(r, r.first(b) + i);
    const int V = r.V;
    const Scale scale = make_scale(plan.top, r.temp(b));
    const float bins = bin_scale(scale);
    const double unit = (double)(1ULL << bits);
    const auto put = [&](int at, u64 order) { sh.put(at, order, packed, scale, unit); };
    fits = listing <= LISTED;
    listed = fits ? listing : 0;
    if constexpr (LISTS) {
      if (t < listed) put(t, ahead);
      for (int j = t + kThreads; j < listed; j += kThreads) put(j, lists[j]);
    }
    kept = plan.total;
#pragma unroll 1
    for (int turn = 0; turn < 2; ++turn) {
      const bool by_count = turn == 0;
      if (!(by_count ? plan.k > 0 : plan.by_p != 0)) continue;
      if (plan.deep == kWhole && listing <= plan.k) continue;  // (all that weighs anything stays)
      const uint32_t k = (uint32_t)plan.k;
      const int first = by_count ? plan.k_first : plan.p_first, last = by_count ? plan.k_last : plan.p_last;
      BinRange range(last, first);
      float steps = bins;  // what range's bins are of
      const double before = by_count ? plan.k_before : plan.p_before;
      const double goal = fmin(fmax((double)r.nucleus(b) * kept, 0x1p-200), kept);
      uint32_t before_count = by_count ? plan.k_count : 0;
      u64 low = 0, high = (1ULL << packed.bits()) - 1, fixed_goal = 0, before_fixed = 0;
      bool have_goal = by_count, lost = false;

      // The part of the goal that is among these tokens, at most what their
      // integers add up to (they are rounded apart from the histograms').
      const auto set_goal = [&](u64 all) {
        const double want = ceil((goal - before) * unit);
        fixed_goal = want < 1.0 ? 1 : min((u64)want, all);
        have_goal = true;
        lost = all == 0;
      };
      // The step with the border, by the counts and sums of all of them.
      // orders: steps are of order values, of which low .. high are left then.
      const auto narrow = [&](int shift, bool orders) {
        const uint32_t c0 = sh.sub_count[2 * t], c1 = sh.sub_count[2 * t + 1];
        const u64 w0 = sh.sub_sum[2 * t], w1 = sh.sub_sum[2 * t + 1];
        const uint32_t pc = wave_prefix(c0 + c1);
        const u64 pw = wave_prefix(w0 + w1);
        if (lane == 63) {
          sh.wave_count[wave] = pc;
          sh.wave_fixed[wave] = pw;
        }
        __syncthreads();
        uint32_t c = before_count + pc - (c0 + c1);
        u64 w = before_fixed + pw - (w0 + w1), all = 0;
        for (int v = 0; v < kWaves; ++v) {
          if (v < wave) {
            c += sh.wave_count[v];
            w += sh.wave_fixed[v];
          }
          all += sh.wave_fixed[v];
        }
        if (!have_goal) set_goal(all);
        const bool in0 = by_count ? c < k && c + c0 >= k : w < fixed_goal && w + w0 >= fixed_goal;
        const bool in1 = by_count ? c + c0 < k && c + c0 + c1 >= k : w + w0 < fixed_goal && w + w0 + w1 >= fixed_goal;
        if (in0 || in1) {  // (one thread: the interval has the border)
          sh.bin_ = 2 * t + (in0 ? 0 : 1);
          sh.count_ = in0 ? c0 : c1;
          sh.before_count_ = in0 ? c : c + c0;
          sh.before_fixed_ = in0 ? w : w + w0;
        }
        __syncthreads();
        before_count = sh.before_count_;
        before_fixed = sh.before_fixed_;
        if (!orders) return;
        const u64 top = high - ((u64)sh.bin_ << shift), span = (1ULL << shift) - 1;
        low = top - low > span ? top - span : low;
        high = top;
      };

      if (!fits) {
        // The list does not hold these bins' tokens (logits that lie closer
        // together than a bin is wide): passes over the row narrow their order
        // values by 10 bits each until what is left fits it.  Where the border
        // lies past the bins (and the row is long) the first pass counts by wider
        // ones, which reach down to weights of 0: a border behind those cuts
        // nothing.
        int shift = max(0, packed.bits() - sh.kSubBits);
        const float wide = bins * ((sh.kSub - 4) / (10.0f * kLeastBits));
        const int wide_top = bin_of(plan.top, wide);
        bool by_steps = LISTS && by_count && plan.deep != 0;
        const auto take = [&](int e, float l) {
          const u64 order = order_value(l, e), o = packed.pack(order);
          if (o < low || o > high) return;
          if (shift < 0) {  // (there are as many as the last pass counted, which fit)
            const int at = atomicAdd(&sh.fill_, 1);
            if (at < LISTED) put(at, order);
          } else {
            atomicAdd(&sh.sub_count[(high - o) >> shift], 1u);
            atomicAdd(&sh.sub_sum[(high - o) >> shift], fixed_weight(sample_weight(l, scale), unit));
          }
        };
#pragma unroll 1
        while (true) {
          __syncthreads();
          for (int j = t; j < sh.kSub; j += kThreads) {
            sh.sub_count[j] = 0;
            sh.sub_sum[j] = 0;
          }
          if (t == 0) sh.fill_ = 0;
          __syncthreads();
          if constexpr (LISTS) {
            // (Two vectors of a lane at once, and the few logits that are in the
            // bins read again, as sample_collect_kernel does.)
            constexpr int kAhead = 2, kChunk = kAhead * kWave * L::kVec;
#pragma unroll 1
            for (int c0 = wave * kChunk; c0 < V; c0 += kWaves * kChunk) {
              const int e0 = c0 + lane * L::kVec;
              Unaligned16<typename L::Raw> raw[kAhead];
#pragma unroll
              for (int i = 0; i < kAhead; ++i) {
                const int at = e0 + i * kWave * L::kVec;
                if (at + L::kVec <= V) {
                  raw[i] = *reinterpret_cast<const Unaligned16<typename L::Raw>*>(row + at);
                } else {
#pragma unroll
                  for (int j = 0; j < L::kVec; ++j) raw[i].v[j] = at + j < V ? row[at + j] : L::kMinus;
                }
              }
              uint32_t hits = 0;
#pragma unroll
              for (int i = 0; i < kAhead; ++i) {
#pragma unroll
                for (int j = 0; j < L::kVec; ++j) {
                  const float l = L::value(raw[i].v[j]);
                  if (!(l > -INFINITY)) continue;
                  if (by_steps) {
                    atomicAdd(&sh.sub_count[min(wide_top - bin_of(l, wide), sh.kSub - 1)], 1u);
                  } else if (range.holds(l * steps)) {
                    hits |= 1u << (i * L::kVec + j);
                  }
                }
              }
#pragma unroll 1
              for (; hits; hits &= hits - 1) {
                const int bit = __ffs(hits) - 1, e = e0 + bit / L::kVec * kWave * L::kVec + bit % L::kVec;
                take(e, L::value(row[e]));
              }
            }
          } else {  // (a short row: one logit a lane, no registers for more)
#pragma unroll 1
            for (int e = t; e < V; e += kThreads) {
              const float l = L::value(row[e]);
              if (range.holds(l * steps) && l > -INFINITY) take(e, l);
            }
          }
          __syncthreads();
          if (shift < 0) break;
          narrow(shift, !by_steps);
          if (by_steps) {
            by_steps = false;
            lost = sh.bin_ == sh.kSub - 1;
            steps = wide;
            range = BinRange(wide_top - sh.bin_, wide_top - sh.bin_);
            if (sh.count_ <= (uint32_t)LISTED) shift = -1;
          } else {
            shift = sh.count_ <= (uint32_t)LISTED ? -1 : max(0, 64 - __clzll(high - low) - sh.kSubBits);
          }
          if (lost) break;
        }
        listed = lost ? 0 : min(sh.fill_, LISTED);
      }

      // Narrow the listed tokens of the bins that are within low .. high.  (A
      // bin's tokens are an interval of order values: the first look finds it.)
      uint32_t n;
#pragma unroll 1
      for (bool first_look = true;; first_look = false) {
        __syncthreads();
        // How many there are, what they weigh, and the interval that they take.
        u64 a = ~0ULL, z = 0, sum = 0;
        uint32_t count = 0;
        for (int j = t; j < listed; j += kThreads) {
          const u64 o = sh.list[j];
          if (o >= low && o <= high && (!first_look || range.holds(packed.logit(o) * steps))) {
            ++count;
            if (!have_goal) sum += sh.weight[j];
            a = min(a, o);
            z = max(z, o);
          }
        }
        count = wave_sum(count);
        sum = wave_sum(sum);
        a = wave_min(a, ~0ULL);
        z = wave_max(z, 0ULL);
        if (lane == 0) {
          sh.wave_count[wave] = count;
          sh.wave_fixed[wave] = sum;
          sh.wave_low[wave] = a;
          sh.wave_high[wave] = z;
        }
        for (int j = t; j < sh.kSub; j += kThreads) {
          sh.sub_count[j] = 0;
          sh.sub_sum[j] = 0;
        }
        if (t < kFew) sh.few[t] = make_ulonglong2(0, 0);
        if (t == 0) sh.fill_ = 0;
        __syncthreads();
        n = 0;
        sum = 0;
        for (int v = 0; v < kWaves; ++v) {
          n += sh.wave_count[v];
          sum += sh.wave_fixed[v];
          a = min(a, sh.wave_low[v]);
          z = max(z, sh.wave_high[v]);
        }
        if (!have_goal) set_goal(sum);
        low = a;
        high = z;
        if (n <= (uint32_t)kFew || lost) break;
        const int shift = max(0, 64 - __clzll(high - low) - sh.kSubBits);  // (high - low) >> shift is below kSub
        for (int j = t; j < listed; j += kThreads) {
          const u64 o = sh.list[j];
          if (o >= low && o <= high) {
            atomicAdd(&sh.sub_count[(high - o) >> shift], 1u);
            atomicAdd(&sh.sub_sum[(high - o) >> shift], sh.weight[j]);
          }
        }
        __syncthreads();
        narrow(shift, true);
      }
      if (lost || n == 0) continue;  // (the same for every thread)
      // The few that are left, each against the others: a thread has one and a
      // part of the others.  (One wavefront with all of them took 3.8 us for 50;
      // 128 instead of 64 take 1 us longer where they are not needed and save as
      // much where they are.)
      for (int j = t; j < listed; j += kThreads) {
        const u64 o = sh.list[j];
        if (o >= low && o <= high) {
          const int f = atomicAdd(&sh.fill_, 1);
          sh.few[f] = make_ulonglong2(o, sh.weight[j]);
        }
      }
      __syncthreads();
      constexpr int kEach = kFew * kFew / kThreads;
      const int mine = t % kFew, others = t / kFew * kEach;
      if (others < (int)n) {
        const u64 o = sh.few[mine].x;
        uint32_t c = 0;
        u64 w = 0;
#pragma unroll 1
        for (int j = 0; j < kEach; j += 8) {
          ulonglong2 other[8];  // (0 behind the last one)
#pragma unroll
          for (int e = 0; e < 8; ++e) other[e] = sh.few[others + j + e];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            c += other[e].x > o ? 1 : 0;
            w += other[e].x > o ? other[e].y : 0;
          }
        }
        if (c != 0) {
          atomicAdd(&sh.sub_count[mine], c);
          atomicAdd(&sh.sub_sum[mine], w);
        }
      }
      __syncthreads();
      if (t < (int)n) {
        const uint32_t c = before_count + sh.sub_count[t];
        const u64 up_to = before_fixed + sh.sub_sum[t], w = sh.few[t].y;
        if (by_count ? c + 1 == k : up_to < fixed_goal && up_to + w >= fixed_goal) {  // (one of them)
          sh.border_ = sh.few[t].x;
          sh.before_fixed_ = up_to + w;
        }
      }
      __syncthreads();
      border = sh.border_;
      of_p = !by_count;
      kept = plan.deep ? plan.total : before + (double)sh.before_fixed_ / unit;
      __syncthreads();
    }
    if (border == 0) kept = plan.kept;
  }
  const u64 cut = border ? packed.order(border) : 0;
  DrawRec w{};
  w.sum = kept;
  w.cut = cut;
  w.top = plan.top;
  w.row = r.first(b) + i;
  w.arg = plan.arg;
  w.refused = -1;
  if (!tokens) {
    if (t == 0) {
      cuts[slot] = RowCut{cut, kept};
      if (draws) draws[b] = w;
    }
    return;
  }
  // The draw (rows and sequences are the same here, ns is at most kSub).
  if (w.arg != -2) {
    if (t == 0) tokens[b] = w.arg;
    return;
  }
  const auto* row = row_at<SRC>(r, w.row);
  const Scale scale = make_scale(w.top, r.temp(b));
  double* masses = mass + (long long)slot * ns;
  const double unit = (double)(1ULL << bits);
  // What the second launch summed is right where the cut is in the bins that it
  // listed; the segments are summed here otherwise, and for random numbers next
  // to 0 and of 1 (one draw in 65536), for which tokens count that are little or
  // nothing as integers.
  const bool summed = LISTS && plan.filters && cut != 0 && fits && u > 0x1p-16f && u < 1.0f &&
                      (plan.all_listed || of_p == (plan.by_p != 0));
  if (summed) {
    for (int j = t; j < ns; j += kThreads) sh.sub_sum[j] = 0;
    __syncthreads();
    const BinRange range(plan.by_p ? plan.p_last : plan.k_last, plan.by_p ? plan.p_first : plan.k_first);
    const float bins = bin_scale(scale);
    for (int j = t; j < listed; j += kThreads) {
      const u64 o = sh.list[j];
      if (o >= border && (plan.all_listed || range.holds(packed.logit(o) * bins)))
        atomicAdd(&sh.sub_sum[packed.index(o) / kSegment], sh.weight[j]);
    }
  } else if (cut != 0) {
    for (int seg = wave; seg < ns; seg += kWaves) {
      float x[kSamplePer];
      load_segment<SRC>(row, seg, r.V, x);
      constexpr int kVec = Logit<SRC>::kVec;
      double s = 0.0;
#pragma unroll
      for (int g = 0; g < kSamplePer / kVec; ++g) {
        double p[kVec];
        draw_weights<kVec>(w, scale, nullptr, false, segment_element<SRC>(seg, g), r.V, x + g * kVec, p);
#pragma unroll
        for (int e = 0; e < kVec; ++e) s += p[e];
      }
      s = wave_sum(s);
      if (lane == 0) masses[seg] = s;
    }
  }
  __syncthreads();
  const SegRec* recs = rec + (long long)slot * ns;
  pick_token<SRC, kWaves>(sh.pick, row, r.V, ns, w, scale, nullptr, false, fmin(fmax((double)u, 0.0), 1.0),
                             [&](int j) {
                               if (cut == 0) return segment_sum(recs[j], scale);
                               if (!summed) return masses[j];
                               return (plan.all_listed ? 0.0 : masses[j]) + (double)sh.sub_sum[j] / unit;
                             },
                             tokens + b);
}

// One workgroup per row.  (128 registers, so that a compute unit has two rows.)
template <int SRC>
__global__ void __launch_bounds__(kCutThreads, 4)
    sample_border_kernel(SampleRows r, int ns, int bits, const SegRec* rec, const CutPlan* plans, const u64* lists,
                         RowCut* cuts, DrawRec* draws, double* mass, const float* uniforms, long long* tokens) {
  __shared__ CutShared<SRC, kCutThreads, kListed> sh;
  const int slot = blockIdx.x, b = slot / (r.K + 1), t = threadIdx.x;
  if (slot % (r.K + 1) >= r.count(b)) return;
  const CutPlan plan = plans[slot];
  const float u = tokens ? uniforms[b] : 0.0f;
  const u64* list = lists + (long long)slot * kListed;
  // (under way with the plan; what is not listed is not used)
  const u64 ahead = list[t];
  find_border<true>(sh, r, ns, bits, rec, plan, plan.listed, list, ahead, cuts, draws, mass, u, tokens);
}

// All of it for rows of one part, whose logits stay in registers until they are
// listed: one launch instead of four.  (Drafts of 952 rows of 1325, top_k 1000,
// 73.6 us in four, 46.3 so; of 1773 rows of 2722 with top_p 88.7 and 51.9; draws
// from 300 rows of 8192 39.3 and 24.9, from one 27.3 and 21.5.)
template <int SRC>
__global__ void __launch_bounds__(kSampleThreads, 4)
    sample_short_kernel(SampleRows r, int ns, int bits, SegRec* rec, RowCut* cuts, DrawRec* draws, double* mass,
                        const float* uniforms, long long* tokens) {
  __shared__ union {
    struct {
      Histogram hist;
      double bin_sum[kBins];
    } bins;
    CutShared<SRC, kSampleThreads, kShortListed> cut;
  } both;  // (40 KB, so that a compute unit has four rows)
  auto& sh = both.cut;
  Histogram& h = both.bins.hist;
  double* const bin_sum = both.bins.bin_sum;
  __shared__ float tops[4];
  __shared__ SegRec part[4];
  __shared__ CutPlan s_plan;
  __shared__ int listing;
  const int slot = blockIdx.x, b = slot / (r.K + 1), i = slot % (r.K + 1);
  const int t = threadIdx.x, seg = t >> 6, lane = t & 63;
  if (i >= r.count(b)) return;
  for (int j = t; j < kBins; j += kSampleThreads) {
    h.sum[j] = 0;
    h.count[j] = 0;
  }
  if (t == 0) listing = 0;
  constexpr int kVec = Logit<SRC>::kVec;
  const auto* row = row_at<SRC>(r, r.first(b) + i);
  const float u = tokens ? uniforms[b] : 0.0f;
  float x[kSamplePer];
  load_segment<SRC>(row, seg, r.V, x);
  const float temp = r.temp(b);
  bool by_k, by_p;
  const bool filters = row_filters(r, b, temp, by_k, by_p);
  const SegRec g = part_sums<SRC>(x, seg, temp, filters, by_k, tops, h);
  if (lane == 0) {
    part[seg] = g;
    if (seg < ns) rec[(long long)slot * ns + seg] = g;
  }
  __syncthreads();
  for (int j = t; j < kBins; j += kSampleThreads) bin_sum[j] = (double)h.sum[j] * (1.0 / (double)(1ULL << kBinBits));
  __syncthreads();
  if (t < kWave) {
    CutPlan plan{};
    Scale scale;
    combine_segments(part, ns, temp, plan.top, plan.arg, scale, plan.kept);
    if (filters && plan.arg == -2)
      plan_cut(plan, BinScan(h.count, bin_sum), r, b, bin_of(plan.top, bin_scale(scale)), by_k, by_p);
    if (lane == 0) s_plan = plan;
  }
  __syncthreads();
  const CutPlan plan = s_plan;
  if (plan.filters) {
    const Scale scale = make_scale(plan.top, temp);
    const float bins = bin_scale(scale);
    const double unit = (double)(1ULL << bits);
    const Packed<SRC> packed(r.V);
    uint32_t hits = plan_hits(plan, x, bins);
    int at = hits ? atomicAdd(&listing, __popc(hits)) : 0;
#pragma unroll 1
    for (; hits && at < kShortListed; hits &= hits - 1, ++at) {  // (read again: registers have no index)
      const int bit = __ffs(hits) - 1, e = segment_element<SRC>(seg, bit / kVec) + bit % kVec;
      sh.put(at, order_value(Logit<SRC>::value(row[e]), e), packed, scale, unit);
    }
  }
  __syncthreads();
  find_border<false>(sh, r, ns, bits, rec, plan, listing, nullptr, 0, cuts, draws, mass, u, tokens);
}

template <int SRC>
void launch(const SampleRows& r, int bits, SegRec* rec, const Histogram* hist, CutPlan* plans, u64* lists,
            RowCut* cuts, DrawRec* draws, double* mass, const float* uniforms, long long* tokens, hipStream_t st) {
  const int blocks = (r.V + kSampleBlock - 1) / kSampleBlock;
  const long long slots = (long long)r.B * (r.K + 1);
  if (blocks == 1) {
    hipLaunchKernelGGL((sample_short_kernel<SRC>), dim3((unsigned)slots), dim3(kSampleThreads), 0, st, r, r.segments(),
                       bits, rec, cuts, draws, mass, uniforms, tokens);
    return;
  }
  hipLaunchKernelGGL(sample_bins_kernel, dim3((unsigned)slots), dim3(kCutThreads), 0, st, r, r.segments(), blocks, rec,
                     hist, plans);
  if (tokens)
    hipLaunchKernelGGL((sample_collect_kernel<SRC, true>), dim3((unsigned)(slots * blocks)), dim3(kSampleThreads), 0, st,
                       r, r.segments(), blocks, plans, lists, mass);
  else
    hipLaunchKernelGGL((sample_collect_kernel<SRC, false>), dim3((unsigned)(slots * blocks)), dim3(kSampleThreads), 0,
                       st, r, r.segments(), blocks, plans, lists, nullptr);
  hipLaunchKernelGGL((sample_border_kernel<SRC>), dim3((unsigned)slots), dim3(kCutThreads), 0, st, r, r.segments(), bits,
                     rec, plans, lists, cuts, draws, mass, uniforms, tokens);
}

}  // namespace

int launch_sample_cut(const SampleRows& r, int dtype, SegRec* rec, const Histogram* hist, CutPlan* plans,
                      u64* lists, RowCut* cuts, DrawRec* draws, double* mass, const float* uniforms, long long* tokens,
                      hipStream_t st) {
  int bits = 45;
  while ((1LL << (62 - bits)) < (long long)r.V) --bits;
  switch (dtype) {
    case VRM_SRC_F32: launch<VRM_SRC_F32>(r, bits, rec, hist, plans, lists, cuts, draws, mass, uniforms, tokens, st); break;
    case VRM_SRC_F16: launch<VRM_SRC_F16>(r, bits, rec, hist, plans, lists, cuts, draws, mass, uniforms, tokens, st); break;
    default: launch<VRM_SRC_BF16>(r, bits, rec, hist, plans, lists, cuts, draws, mass, uniforms, tokens, st); break;
  }
  return launch_status("sample_cut");
}

}  // namespace vrm
