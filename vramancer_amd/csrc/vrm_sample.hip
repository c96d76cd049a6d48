// From logits to tokens: a token per row (vrm_sample_tokens), and drafted
// tokens verified against the target's probabilities (vrm_verify_drafts).  No
// counterpart in the reference, whose batcher samples on the host.
//
// Both are passes over rows of V logits, cut into chunks of 8192 so that few
// rows fill the chip too:
//   1. sample_chunk_kernel  every row's chunks: maximum, sum of weights
//   2. sample_cut_kernel    (top_k, top_p) which tokens stay (vrm_sample_cut.hip)
//   3. sample_choose_kernel a sequence's drafts: accepted ones, the row its next
//                           token is drawn from
//   4. sample_mass_kernel   that row's chunks: the mass to draw from
//   5. sample_pick_kernel   the chunk and the token where the running sum
//                           passes the random number
// A plain draw without top_k, top_p and probabilities is 1 and 5.
#include "vrm_sample.h"

namespace vrm {
namespace {

// ---------------------------------------------------------------------------
// 1. Chunks of rows
// ---------------------------------------------------------------------------

template <int SRC>
__global__ void __launch_bounds__(kSampleThreads) sample_chunk_kernel(SampleRows r, int nc, ChunkRec* rec) {
  __shared__ float tops[4];
  __shared__ double sums[4];
  __shared__ int args[4];
  const int slot = blockIdx.x / nc, chunk = blockIdx.x % nc;
  const int b = slot / (r.K + 1), i = slot % (r.K + 1);
  if (i >= r.count(b)) return;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  float x[kSamplePer];
  load_chunk<SRC>(row_at<SRC>(r, r.first(b) + i), chunk, r.V, x);
  float m = -INFINITY;
#pragma unroll
  for (int e = 0; e < kSamplePer; ++e) m = fmaxf(m, x[e]);
  m = group_max<64>(m);
  if (lane == 0) tops[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const float t = r.temp(b);
  double s = 0.0;
  int arg = 0x7fffffff;
  if (t > 0.0f) {
    const double c = sample_scale(t);
    if (m > -INFINITY) {
#pragma unroll
      for (int e = 0; e < kSamplePer; ++e) s += sample_weight(x[e], m, c);
    }
  } else if (m > -INFINITY) {
    constexpr int kVec = Logit<SRC>::kVec;
#pragma unroll
    for (int e = kSamplePer - 1; e >= 0; --e)
      if (x[e] == m)
        arg = chunk * kSampleChunk + ((e / kVec) * kSampleThreads + (int)threadIdx.x) * kVec + e % kVec;
  }
  s = wave_sum(s);
  arg = wave_min(arg);
  if (lane == 0) {
    sums[wave] = s;
    args[wave] = arg;
  }
  __syncthreads();
  if (threadIdx.x == 0)
    rec[(long long)slot * nc + chunk] = ChunkRec{(sums[0] + sums[1]) + (sums[2] + sums[3]), m,
                                                 min(min(args[0], args[1]), min(args[2], args[3]))};
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

template <int SRC>
__global__ void __launch_bounds__(kSampleThreads)
    sample_choose_kernel(SampleRows r, Drafts d, int nc, const ChunkRec* rec, const RowCut* cuts, DrawRec* draws,
                         long long* tokens, int32_t* accepted) {
  __shared__ int stop;  // the first row whose draft is refused, or the last row
  const int b = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int n = r.count(b), first = r.first(b);
  if (threadIdx.x == 0) stop = n - 1;
  __syncthreads();
  const float t = r.temp(b);
  const bool greedy = !(t > 0.0f);
  const double c = greedy ? 0.0 : sample_scale(t);
  for (int i = wave; i < n - 1; i += kSampleThreads / kWave) {
    const long long slot = (long long)b * (r.K + 1) + i, at = (long long)b * r.K + i;
    float top;
    double sum;
    int arg;
    combine_chunks(rec + slot * nc, nc, c, top, sum, arg);
    const long long x = d.id(at);
    bool ok = false;
    if (x >= 0 && x < r.V && top > -INFINITY) {
      double w;
      if (greedy) {
        w = x == arg ? 1.0 : 0.0;
        sum = 1.0;
      } else {
        const float l = Logit<SRC>::value(row_at<SRC>(r, first + i)[x]);
        w = sample_weight(l, top, c);
        if (cuts) {
          const RowCut cut = cuts[slot];
          sum = cut.sum;
          if (order_value(l, (int)x) < cut.cut) w = 0.0;
        }
      }
      const double q = d.probs ? (double)d.probs[b * d.seq_stride + i * d.draft_stride + x] : 1.0;
      const double u = (double)fmaxf(d.accept[at], 0.0f);
      ok = u * (q < 0.0 ? 0.0 : q) * sum < w;
    }
    if (!ok && lane == 0) atomicMin(&stop, i);
  }
  __syncthreads();
  const int a = max(stop, 0);
  if (tokens) {
    for (int i = threadIdx.x; i <= r.K; i += kSampleThreads)
      tokens[(long long)b * (r.K + 1) + i] = i < a && n > 0 ? d.id((long long)b * r.K + i) : -1;
    if (threadIdx.x == 0) accepted[b] = n > 0 ? a : 0;
  }
  if (wave != 0) return;
  DrawRec w{};
  w.row = -1;
  if (n > 0) {
    const long long slot = (long long)b * (r.K + 1) + a;
    int arg;
    combine_chunks(rec + slot * nc, nc, c, w.top, w.sum, arg);
    w.c = c;
    w.row = first + a;
    w.arg = w.top == -INFINITY ? -1 : greedy ? arg : -2;
    w.at = a;
    w.refused = -1;
    if (a < n - 1) {
      const long long x = d.id((long long)b * r.K + a);
      if (x >= 0 && x < r.V) w.refused = (int)x;
    }
    if (cuts && !greedy) {
      w.cut = cuts[slot].cut;
      w.sum = cuts[slot].sum;
    }
  }
  if (lane == 0) draws[b] = w;
}

// ---------------------------------------------------------------------------
// 4. and 5. The mass of a row's tokens and the token
// ---------------------------------------------------------------------------

// What the tokens of the vector at e0 weigh in the draw: p, or where a draft
// was refused max(p - q, 0), in units of 1 / sum.
template <int SRC>
__device__ __forceinline__ void draw_weights(const DrawRec& w, const float* q, bool rest, int e0, int V, const float* x,
                                             double* out) {
  constexpr int kVec = Logit<SRC>::kVec;
  float qx[kVec];
  if (rest && q) {
    if (e0 + kVec <= V) {
#pragma unroll
      for (int h = 0; h < kVec; h += 4) {
        const auto raw = *reinterpret_cast<const Unaligned16<uint32_t>*>(q + e0 + h);
#pragma unroll
        for (int e = 0; e < 4; ++e) qx[h + e] = __uint_as_float(raw.v[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) qx[e] = e0 + e < V ? q[e0 + e] : 0.0f;
    }
  }
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    double p = sample_weight(x[e], w.top, w.c);
    if (w.cut && order_value(x[e], e0 + e) < w.cut) p = 0.0;
    if (rest) {
      if (q) {
        const double d = fma(-(double)(qx[e] < 0.0f ? 0.0f : qx[e]), w.sum, p);
        p = d > 0.0 ? d : 0.0;  // (nothing where q is NaN)
      } else if (e0 + e == w.refused) {
        p = 0.0;
      }
    }
    out[e] = p;
  }
}

__device__ __forceinline__ const float* draft_row(const Drafts& d, const DrawRec& w, int b) {
  return d.probs ? d.probs + b * d.seq_stride + w.at * d.draft_stride : nullptr;
}

template <int SRC>
__global__ void __launch_bounds__(kSampleThreads)
    sample_mass_kernel(SampleRows r, Drafts d, int nc, const DrawRec* draws, double* mass, float* probs) {
  __shared__ double sums[4];
  const int b = blockIdx.x / nc, chunk = blockIdx.x % nc;
  const DrawRec w = draws[b];
  if (w.row < 0) return;
  constexpr int kVec = Logit<SRC>::kVec;
  if (w.arg >= -1) {  // greedy, or nothing to draw from
    if (probs) {
      for (int i = threadIdx.x; i < kSampleChunk; i += kSampleThreads) {
        const long long e = (long long)chunk * kSampleChunk + i;
        if (e < r.V) probs[(long long)b * r.V + e] = e == w.arg ? 1.0f : 0.0f;
      }
    }
    return;
  }
  const auto* row = row_at<SRC>(r, w.row);
  const float* q = draft_row(d, w, b);
  const double inv = 1.0 / w.sum;
  double s = 0.0;
#pragma unroll 2
  for (int i = 0; i < kSamplePer / kVec; ++i) {
    const int e0 = chunk * kSampleChunk + (i * kSampleThreads + (int)threadIdx.x) * kVec;
    float x[kVec];
    double p[kVec];
    load_vec<SRC>(row, e0, r.V, x);
    draw_weights<SRC>(w, q, w.refused >= 0, e0, r.V, x, p);
#pragma unroll
    for (int e = 0; e < kVec; ++e) s += p[e];
    if (probs) {
      float* to = probs + (long long)b * r.V + e0;
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (e0 + e < r.V) to[e] = (float)(p[e] * inv);
    }
  }
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) mass[(long long)b * nc + chunk] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// One workgroup per sequence.  mass == NULL: a draw from a row by its chunk
// records alone (slot b); draws == NULL then.
template <int SRC>
__global__ void __launch_bounds__(kSampleThreads)
    sample_pick_kernel(SampleRows r, Drafts d, int nc, const ChunkRec* rec, const DrawRec* draws, const double* mass,
                       const float* uniforms, long long* tokens) {
  __shared__ double totals[kSamplePer / 4][4];
  __shared__ double base;
  __shared__ int where, found, last;
  constexpr int kVec = Logit<SRC>::kVec, kGroups = kSamplePer / kVec;
  const int b = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  DrawRec w{};
  if (draws) {
    w = draws[b];
  } else {
    const float t = r.temp(b);
    const bool greedy = !(t > 0.0f);
    w.c = greedy ? 0.0 : sample_scale(t);
    int arg;
    combine_chunks(rec + (long long)b * nc, nc, w.c, w.top, w.sum, arg);
    w.row = b;
    w.arg = w.top == -INFINITY ? -1 : greedy ? arg : -2;
    w.refused = -1;
  }
  if (w.row < 0) return;
  long long* out = tokens + (draws ? (long long)b * (r.K + 1) + w.at : b);
  if (w.arg >= -1) {
    if (threadIdx.x == 0) *out = w.arg;
    return;
  }
  const auto* row = row_at<SRC>(r, w.row);
  const float* q = draft_row(d, w, b);
  const double u = fmin(fmax((double)uniforms[b], 0.0), 1.0);
  bool rest = w.refused >= 0;
  // The chunk: by one wavefront, 64 at a time.
  const auto chunk_mass = [&](int j) -> double {
    if (mass) return mass[(long long)b * nc + j];
    const ChunkRec g = rec[(long long)b * nc + j];
    return g.top > -INFINITY ? g.sum * sample_weight(g.top, w.top, w.c) : 0.0;
  };
  if (wave == 0) {
    double total = 0.0;
    for (int j0 = 0; j0 < nc; j0 += kWave) total += wave_sum(j0 + lane < nc ? chunk_mass(j0 + lane) : 0.0);
    const double target = u * total;
    double before = 0.0;
    int at = -1, some = -1;
    double left = 0.0, some_left = 0.0;
    for (int j0 = 0; j0 < nc && at < 0; j0 += kWave) {
      const double v = j0 + lane < nc ? chunk_mass(j0 + lane) : 0.0;
      const double run = before + wave_prefix(v);
      const unsigned long long hit = __ballot(v > 0.0 && run > target), any = __ballot(v > 0.0);
      if (hit) {
        const int l = __ffsll(hit) - 1;
        at = j0 + l;
        left = target - (__shfl(run, l) - __shfl(v, l));
      } else if (any) {
        const int l = 63 - __clzll(any);
        some = j0 + l;
        some_left = target - (__shfl(run, l) - __shfl(v, l));
      }
      before = __shfl(run, 63);
    }
    if (at < 0) {  // rounding of the sums, or a random number of 1: the last token that weighs anything
      at = some;
      left = some_left;
    }
    if (lane == 0) {
      where = at;
      base = left;
      found = 0x7fffffff;
      last = -1;
    }
  }
  __syncthreads();
  int chunk = where;
  double target = base;
  if (chunk < 0) {
    // Nothing is left of p - q: the row's p itself.  Its chunks have not been
    // summed, so this (a q that is p but for rounding, or no distribution) walks
    // the row twice.
    if (!rest) {
      if (threadIdx.x == 0) *out = -1;
      return;
    }
    rest = false;
    double total = 0.0, goal = 0.0, before = 0.0;
    int lastc = -1;
    double lastg = 0.0;
    for (int turn = 0; turn < 2; ++turn) {
      before = 0.0;
      for (int j = 0; j < nc; ++j) {
        double s = 0.0;
        for (int i = 0; i < kGroups; ++i) {
          const int e0 = j * kSampleChunk + (i * kSampleThreads + (int)threadIdx.x) * kVec;
          float x[kVec];
          double p[kVec];
          load_vec<SRC>(row, e0, r.V, x);
          draw_weights<SRC>(w, nullptr, false, e0, r.V, x, p);
#pragma unroll
          for (int e = 0; e < kVec; ++e) s += p[e];
        }
        s = wave_sum(s);
        __syncthreads();
        if (lane == 0) totals[0][wave] = s;
        __syncthreads();
        s = (totals[0][0] + totals[0][1]) + (totals[0][2] + totals[0][3]);
        if (turn == 1 && s > 0.0) {
          lastc = j;
          lastg = goal - before;
          if (before + s > goal) break;
        }
        before += s;
      }
      if (turn == 0) {
        total = before;
        goal = u * total;
      }
    }
    __syncthreads();
    chunk = lastc;
    target = lastg;
    if (chunk < 0) {
      if (threadIdx.x == 0) *out = -1;
      return;
    }
  }
  // The token: running sums over the chunk in the order of its indices.
  double p[kSamplePer], run[kGroups];
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const int e0 = chunk * kSampleChunk + (i * kSampleThreads + (int)threadIdx.x) * kVec;
    float x[kVec];
    load_vec<SRC>(row, e0, r.V, x);
    draw_weights<SRC>(w, rest ? q : nullptr, rest, e0, r.V, x, p + i * kVec);
    double s = 0.0;
#pragma unroll
    for (int e = 0; e < kVec; ++e) s += p[i * kVec + e];
    run[i] = wave_prefix(s) - s;
    if (lane == 63) totals[i][wave] = run[i] + s;
  }
  __syncthreads();
  double before = 0.0;
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      if (v == wave) {
        double sum = before + run[i];
        int hit = -1, some = -1;
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          sum += p[i * kVec + e];
          if (p[i * kVec + e] > 0.0) {
            some = e;
            if (hit < 0 && sum > target) hit = e;
          }
        }
        const int e0 = chunk * kSampleChunk + (i * kSampleThreads + (int)threadIdx.x) * kVec;
        if (hit >= 0) atomicMin(&found, e0 + hit);
        if (some >= 0) atomicMax(&last, e0 + some);
      }
      before += totals[i][v];
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) *out = found != 0x7fffffff ? found : last;
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

size_t up(size_t n) { return (n + 255) & ~(size_t)255; }

struct Plan {
  long long slots;
  int nc;
  bool filtered, direct;  // direct: chunks and pick alone
  size_t rec, cuts, draws, mass, bytes;
};

Plan plan_of(long long B, int K, int V, bool filtered, bool direct) {
  Plan p{};
  p.slots = B * (K + 1);
  p.nc = (V + kSampleChunk - 1) / kSampleChunk;
  p.filtered = filtered;
  p.direct = direct && !filtered;
  size_t at = up((size_t)p.slots * p.nc * sizeof(ChunkRec));
  if (filtered) {
    p.cuts = at;
    at += up((size_t)p.slots * sizeof(RowCut));
  }
  if (!p.direct) {
    p.draws = at;
    at += up((size_t)B * sizeof(DrawRec));
    p.mass = at;
    at += up((size_t)B * p.nc * sizeof(double));
  }
  p.bytes = at;
  return p;
}

// A launch counts its threads in 32 bits.
constexpr long long kMostBlocks = (1LL << 32) / 1024 - 1;

template <int SRC>
int run(const SampleRows& r, const Drafts& d, const Plan& p, char* ws, const float* uniforms, float* probs,
        long long* tokens, int32_t* accepted, hipStream_t st, const char* who) {
  auto* rec = reinterpret_cast<ChunkRec*>(ws);
  auto* cuts = p.filtered ? reinterpret_cast<RowCut*>(ws + p.cuts) : nullptr;
  hipLaunchKernelGGL((sample_chunk_kernel<SRC>), dim3((unsigned)(p.slots * p.nc)), dim3(kSampleThreads), 0, st, r, p.nc,
                     rec);
  DrawRec* draws = nullptr;
  double* mass = nullptr;
  if (!p.direct) {
    draws = reinterpret_cast<DrawRec*>(ws + p.draws);
    mass = reinterpret_cast<double*>(ws + p.mass);
    if (cuts) {
      const int rc = launch_sample_cut(r, SRC, p.nc, rec, cuts, st);
      if (rc) return rc;
    }
    hipLaunchKernelGGL((sample_choose_kernel<SRC>), dim3(r.B), dim3(kSampleThreads), 0, st, r, d, p.nc, rec, cuts,
                       draws, accepted ? tokens : nullptr, accepted);
    hipLaunchKernelGGL((sample_mass_kernel<SRC>), dim3((unsigned)((long long)r.B * p.nc)), dim3(kSampleThreads), 0, st,
                       r, d, p.nc, draws, mass, probs);
  }
  hipLaunchKernelGGL((sample_pick_kernel<SRC>), dim3(r.B), dim3(kSampleThreads), 0, st, r, d, p.nc, rec, draws, mass,
                     uniforms, tokens);
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
  const long long nc = (V + kSampleChunk - 1) / kSampleChunk;
  if (B > 0 && ((long long)K + 1 > kMostBlocks / nc / B)) {
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

// Whether any row may lose tokens to top_k or top_p.
bool filters(const int32_t* top_k, int top_k_all, const float* top_p, float top_p_all, int V) {
  return top_k || (top_k_all > 0 && top_k_all < V) || top_p || top_p_all < 1.0f;
}

}  // namespace
}  // namespace vrm

using namespace vrm;

extern "C" size_t vrm_sample_workspace_bytes(int N, int V, int filtered, int with_probs) {
  if (check_sizes(N, 0, V, VRM_SRC_F32, 0, "vrm_sample_workspace_bytes")) return 0;
  return plan_of(N, 0, V, filtered != 0, !with_probs).bytes;
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
  const Plan p = plan_of(N, 0, V, filters(top_k, top_k_all, top_p, top_p_all, V), !probs);
  if (int rc = check_workspace(workspace, workspace_bytes, p.bytes, who)) return rc;
  const SampleRows r{logits, row_stride, nullptr, N, N, 0, V, temperature, temperature_all, top_k, top_k_all, top_p,
                     top_p_all};
  return run_typed(r, dtype, Drafts{}, p, static_cast<char*>(workspace), uniforms, probs,
                   reinterpret_cast<long long*>(tokens), nullptr, reinterpret_cast<hipStream_t>(stream), who);
}

extern "C" size_t vrm_verify_workspace_bytes(int B, int K, int V, int filtered) {
  if (check_sizes(B, K, V, VRM_SRC_F32, 0, "vrm_verify_workspace_bytes")) return 0;
  return plan_of(B, K, V, filtered != 0, false).bytes;
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
  const Plan p = plan_of(B, K, V, filters(top_k, top_k_all, top_p, top_p_all, V), false);
  if (int rc = check_workspace(workspace, workspace_bytes, p.bytes, who)) return rc;
  const SampleRows r{logits, row_stride, cu_seqlens, N, B, K, V, temperature, temperature_all, top_k, top_k_all, top_p,
                     top_p_all};
  const Drafts d{drafts, draft_bytes, draft_probs, probs_seq_stride, probs_draft_stride, accept_uniforms};
  return run_typed(r, dtype, d, p, static_cast<char*>(workspace), draw_uniforms, nullptr,
                   reinterpret_cast<long long*>(tokens), accepted, reinterpret_cast<hipStream_t>(stream), who);
}
