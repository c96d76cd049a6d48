// RMS norm of every query and key head, the rotation by position, and the
// append of rotated keys and of values to a paged cache, in one pass.
//
//   x' = w x / sqrt(mean(x^2) + eps)
//   (a, b) -> (a cos - b sin, b cos + a sin)   pairs (d, d + rot / 2), or
//                                              (2 d, 2 d + 1) interleaved
// in float32, rounded once: to the output's type, or to the pool's (float
// types, int8 codes per token and head, e4m3 codes per page and head).
// cos and sin come from a float32 table that the caller computes once: angles
// of far positions need 64 bits (131072 radians are 0.008 off in float32).
//
// Bound: memory; each row is read and written once.  Rows (a token's query,
// key or value head) go to groups of lanes: a lane holds two 8-element pieces
// chosen so that both members of a pair are in it, a head of 128 takes 8
// lanes, and the sum of squares three DPP steps.  A group takes up to
// kRopeHeads heads of a token, whose cosines, sines and weights it loads once.
// Rows whose sizes or alignment do not allow 16-byte accesses take a wavefront
// each.
// Quantized pools: a workgroup takes the new tokens of one page, K or V, and
// two kv-heads: their rows are laid into LDS (16 tokens at a time) and leave
// as whole dwords of codes, K token-major, V four tokens of a dim to a dword;
// an fp8 page's scale needs its tokens' maximum first.
// Measured, kernels alone: norm and rotation of 2.0e8 bytes of queries and
// keys 43.6 us (4.6 TB/s; a copy reaches 5.0); prompts of about 8000 tokens,
// 40 heads over 8, into int8 pages 70 us, vector ALUs busy 65 % of it (codes,
// and divisions by D in the store loop); one token of a batch 5.9 to 6.9 us.
// The wavefront-a-row path: the same norm and rotation with 40 dims rotated
// 122 us for 38 (in a replayed graph).
// Int8 keys as rows straight from registers were slower (81 us: 130 registers,
// three wavefronts a SIMD).
#include <math.h>

#include <type_traits>

#include "vrm_kv_codes.h"

namespace vrm {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeTokens = 16;  // of a page in LDS at a time
constexpr int kRopeHeads = 4;    // of a token to a group of lanes
constexpr int kPageHeads = 2;    // of a page to a workgroup
constexpr uint32_t kGridX = 1u << 23;  // a launch has less than 2^32 threads along x: further workgroups along y

struct RopeArgs {
  const void *q, *k, *v;
  long long q_n, q_h, k_n, k_h, v_n, v_h;  // element strides of a token and of a head
  void *q_out, *k_out;                     // dense [N][H][D], [N][KH][D] of the source type; k_out NULL: no copy
  const float* cos_sin;                    // [top][rot]: rot / 2 cosines, then sines; NULL: no rotation
  int rot, top, interleaved;
  const void* positions;  // NULL: from the batch's geometry
  int pos_bytes;          // 4 or 8
  const void *qw, *kw;    // [D] or NULL: no norm
  int w_type;
  float eps;
  int N, H, KH, D;
  // the cache (pool NULL: none)
  uint8_t* pool;
  float* scales;
  PoolGeom g;
  long long layer_off, s_layer_off;
  int kv_dtype, fp8;
  const int32_t *table, *lens, *cu;
  int B, PS, P, max_pp;
  int q_units, kv_units;  // groups' shares of a token's queries, and of its keys (and of its values)
  int units;              // of a token: q_units, kv_units, kv_units as far as they take part
  uint32_t units_mul;     // n / units = (t + ((n - t) >> 1)) >> units_shift, t = high half of n units_mul
  int units_shift;
  int row_blocks;         // workgroups of rows; page workgroups follow
};

template <int T>
__device__ __forceinline__ void load8(const void* p, long long at, float (&x)[8]) {
  if constexpr (T == VRM_SRC_F32) {
    const float4* f = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    const float4 a = f[0], b = f[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t h = (w[i / 2] >> (16 * (i & 1))) & 0xffffu;
      x[i] = T == VRM_SRC_F16 ? f16_bits_to_f32(h) : bf16_bits_to_f32(h);
    }
  }
}

// The types of vrm_src_dtype and of the float vrm_kv_dtype have the same codes.
static_assert((int)VRM_SRC_F32 == (int)VRM_KV_F32 && (int)VRM_SRC_F16 == (int)VRM_KV_F16 &&
              (int)VRM_SRC_BF16 == (int)VRM_KV_BF16);

__device__ __forceinline__ uint32_t to_bits16(float x, int type) {
  return type == VRM_SRC_F16 ? (uint32_t)__builtin_bit_cast(unsigned short, (_Float16)x)
                             : (uint32_t)__builtin_bit_cast(unsigned short, (__bf16)x);
}

__device__ __forceinline__ void store8(void* p, long long at, int type, const float (&x)[8]) {
  if (type == VRM_SRC_F32) {
    float4* f = reinterpret_cast<float4*>(static_cast<float*>(p) + at);
    f[0] = make_float4(x[0], x[1], x[2], x[3]);
    f[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = to_bits16(x[2 * i], type) | to_bits16(x[2 * i + 1], type) << 16;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + at) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

__device__ __forceinline__ float load1(const void* p, long long at, int type) {
  if (type == VRM_SRC_F32) return static_cast<const float*>(p)[at];
  const uint32_t h = static_cast<const uint16_t*>(p)[at];
  return type == VRM_SRC_F16 ? f16_bits_to_f32(h) : bf16_bits_to_f32(h);
}

__device__ __forceinline__ void store1(void* p, long long at, int type, float x) {
  if (type == VRM_SRC_F32)
    static_cast<float*>(p)[at] = x;
  else
    static_cast<uint16_t*>(p)[at] = (uint16_t)to_bits16(x, type);
}

// Where token n belongs: its position in its sequence, and the row of the
// rotation table.  False for rows of no sequence.
struct Token {
  int b, pos;
  long long angle;
};

__device__ __forceinline__ bool locate(const RopeArgs& a, int n, Token& t) {
  t.b = 0;
  t.pos = 0;
  if (a.cu) {
    int lo = 0, hi = a.B - 1;
    // one token per sequence: row n starts sequence n, which is not empty (of
    // an empty one the row is a later sequence's)
    if (a.N == a.B && a.cu[n] == n && a.cu[n + 1] > n) lo = hi = n;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.cu[mid] <= n)
        lo = mid;
      else
        hi = mid - 1;
    }
    const int c0 = a.cu[lo], c1 = min(a.cu[lo + 1], a.N);
    if (n < c0 || n >= c1) return false;
    t.b = lo;
    t.pos = a.lens[lo] - c1 + n;
  }
  t.angle = t.pos;
  if (a.positions)
    t.angle = a.pos_bytes == 8 ? static_cast<const long long*>(a.positions)[n] : static_cast<const int32_t*>(a.positions)[n];
  return true;
}

__device__ __forceinline__ bool in_table(const RopeArgs& a, const Token& t) {
  return !a.cos_sin || (t.angle >= 0 && t.angle < a.top);
}

// Page of a position, -1 where there is none.
__device__ __forceinline__ int page_at(const RopeArgs& a, int b, int pos) {
  if (pos < 0 || pos / a.PS >= a.max_pp) return -1;
  const int p = a.table[(long long)b * a.max_pp + pos / a.PS];
  return p >= 0 && p < a.P ? p : -1;
}

// n / units for n < 2^31 (Granlund and Montgomery 1994).
__device__ __forceinline__ uint32_t div_units(const RopeArgs& a, uint32_t n) {
  if (a.units == 1) return n;
  const uint32_t t = __umulhi(n, a.units_mul);
  return (t + ((n - t) >> 1)) >> a.units_shift;
}

// First dims of the two pieces of lane l (of D / 16) of a row, and whether
// they are rotated: both members of every pair are in the lane.
struct Pieces {
  int a, b;
  bool turn;
};
__device__ __forceinline__ Pieces pieces(const RopeArgs& a, int l) {
  if (a.interleaved) return {16 * l, 16 * l + 8, 16 * l < a.rot};
  const int r = a.rot >> 4;
  if (l < r) return {8 * l, (a.rot >> 1) + 8 * l, true};
  const int d = a.rot + 16 * (l - r);
  return {d, d + 8, false};
}

// What a lane needs of the weights and of a position's angles.
struct Lane {
  Pieces p;
  bool on;  // lanes l >= D / 16 hold zeros
  float wx[8], wy[8], c[8], s[8];
};
__device__ __forceinline__ void load_weights(const RopeArgs& a, const void* w, Lane& n) {
  if (!w || !n.on) return;
  const auto both = [&](auto type) {
    load8<decltype(type)::value>(w, n.p.a, n.wx);
    load8<decltype(type)::value>(w, n.p.b, n.wy);
  };
  if (a.w_type == VRM_SRC_F32)
    both(std::integral_constant<int, VRM_SRC_F32>{});
  else if (a.w_type == VRM_SRC_F16)
    both(std::integral_constant<int, VRM_SRC_F16>{});
  else
    both(std::integral_constant<int, VRM_SRC_BF16>{});
}
__device__ __forceinline__ void load_angles(const RopeArgs& a, long long angle, int l, Lane& n) {
  if (!n.p.turn || !n.on) return;
  load8<VRM_SRC_F32>(a.cos_sin, angle * a.rot + 8 * l, n.c);
  load8<VRM_SRC_F32>(a.cos_sin, angle * a.rot + (a.rot >> 1) + 8 * l, n.s);
}

// Norm (w != NULL) and rotation of one row held by LG lanes, a lane with the
// pieces x, y.
template <int LG>
__device__ __forceinline__ void norm_turn(const RopeArgs& a, bool norm, bool turn, const Lane& n, float (&x)[8],
                                          float (&y)[8]) {
  if (norm) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += x[i] * x[i] + y[i] * y[i];
    s = group_sum<LG>(s);
    const float inv = 1.f / sqrtf(s / (float)a.D + a.eps);
    if (n.on) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] *= inv * n.wx[i];
        y[i] *= inv * n.wy[i];
      }
    }
  }
  if (!turn || !n.p.turn || !n.on) return;
  const float *c = n.c, *s = n.s;
  if (a.interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x0 = x[2 * i], x1 = x[2 * i + 1], y0 = y[2 * i], y1 = y[2 * i + 1];
      x[2 * i] = x0 * c[i] - x1 * s[i];
      x[2 * i + 1] = x1 * c[i] + x0 * s[i];
      y[2 * i] = y0 * c[4 + i] - y1 * s[4 + i];
      y[2 * i + 1] = y1 * c[4 + i] + y0 * s[4 + i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x0 = x[i], y0 = y[i];
      x[i] = x0 * c[i] - y0 * s[i];
      y[i] = y0 * c[i] + x0 * s[i];
    }
  }
}

// The same for a row held by a wavefront in LDS (any D, rot, alignment):
// row[d] is normed in place, and the rotated value of dim d returned.
__device__ __forceinline__ void norm_row(const RopeArgs& a, const void* w, float* row) {
  const int lane = threadIdx.x & 63;
  if (w) {
    float s = 0.f;
    for (int d = lane; d < a.D; d += kWave) s += row[d] * row[d];
    s = group_sum<64>(s);
    const float inv = 1.f / sqrtf(s / (float)a.D + a.eps);
    for (int d = lane; d < a.D; d += kWave) row[d] *= inv * load1(w, d, a.w_type);
  }
  __syncwarp();
}
__device__ __forceinline__ float turned(const RopeArgs& a, bool turn, long long angle, const float* row, int d) {
  if (!turn || d >= a.rot) return row[d];
  const int half = a.rot >> 1;
  const int pair = a.interleaved ? d >> 1 : d % half;
  const bool second = a.interleaved ? d & 1 : d >= half;
  const float x = row[a.interleaved ? d & ~1 : pair], y = row[a.interleaved ? d | 1 : pair + half];
  const float c = a.cos_sin[angle * a.rot + pair], s = a.cos_sin[angle * a.rot + half + pair];
  return second ? y * c + x * s : x * c - y * s;
}

// One unit of the row workgroups: up to kRopeHeads heads of a token, by LG
// lanes (64: the general path, a row at a time).
template <int T, int LG, bool GENERAL>
__device__ __forceinline__ void do_unit(const RopeArgs& a, uint32_t unit, float* lds) {
  const int n = (int)div_units(a, unit);
  int u = (int)(unit - (uint32_t)n * a.units);
  Token t;
  if (!locate(a, n, t)) return;
  const int what = u < a.q_units ? 0 : u < a.q_units + a.kv_units ? 1 : 2;  // query, key, value
  u -= what == 0 ? 0 : what == 1 ? a.q_units : a.q_units + a.kv_units;
  const int head0 = u * kRopeHeads, heads = min(kRopeHeads, (what == 0 ? a.H : a.KH) - head0);
  const bool ok = in_table(a, t);
  // (three branches: selects between the argument struct's fields would copy
  // it to scratch memory)
  const void *src, *w = nullptr;
  long long step, row;
  if (what == 0) {
    src = a.q, w = a.qw, step = a.q_h, row = a.q_n;
  } else if (what == 1) {
    src = a.k, w = a.kw, step = a.k_h, row = a.k_n;
  } else {
    src = a.v, step = a.v_h, row = a.v_n;
  }
  const long long from = n * row + head0 * step;
  // destination of head0, in elements of `type`, and from a head to the next
  void* dst;
  long long at, next = a.D;
  int type = T;
  if (what == 0) {
    dst = a.q_out, at = ((long long)n * a.H + head0) * a.D;
  } else if (!a.pool) {
    dst = a.k_out, at = ((long long)n * a.KH + head0) * a.D;
  } else {
    const int page = page_at(a, t.b, t.pos);
    if (page < 0 || !ok) return;
    type = a.kv_dtype;
    dst = a.pool + a.layer_off + (long long)page * a.g.page + (what == 2 ? a.g.kv : 0);
    next = (long long)a.PS * a.D;
    at = head0 * next + (long long)(t.pos % a.PS) * a.D;
  }
  const bool turn = a.cos_sin && what < 2 && ok;
  // a position outside the table has no rotation: such rows are made NaN
  const float spoil = ok ? 0.f : __uint_as_float(0x7fc00000u);
  if constexpr (GENERAL) {
    const int lane = threadIdx.x & 63;
    for (int h = 0; h < heads; ++h) {
      for (int d = lane; d < a.D; d += kWave) lds[d] = load1(src, from + h * step + d, T);
      __syncwarp();
      norm_row(a, w, lds);
      for (int d = lane; d < a.D; d += kWave)
        store1(dst, at + h * next + d, type, turned(a, turn, t.angle, lds, d) + spoil);
      __syncwarp();
    }
  } else {
    const int l = threadIdx.x & (LG - 1);
    Lane ln;
    ln.p = pieces(a, l);
    ln.on = 16 * l < a.D;
    float x[kRopeHeads][8], y[kRopeHeads][8];
#pragma unroll
    for (int h = 0; h < kRopeHeads; ++h) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[h][i] = y[h][i] = 0.f;
      if (ln.on && h < heads) {
        load8<T>(src, from + h * step + ln.p.a, x[h]);
        load8<T>(src, from + h * step + ln.p.b, y[h]);
      }
    }
    load_weights(a, w, ln);
    if (turn) load_angles(a, t.angle, l, ln);
#pragma unroll
    for (int h = 0; h < kRopeHeads; ++h) {
      norm_turn<LG>(a, w, turn, ln, x[h], y[h]);
      if (!ok)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[h][i] = y[h][i] = spoil;
      if (ln.on && h < heads) {
        store8(dst, at + h * next + ln.p.a, type, x[h]);
        store8(dst, at + h * next + ln.p.b, type, y[h]);
      }
    }
  }
}

// The new tokens of one page of a quantized pool, K or V, kPageHeads kv-heads.
// Sequence b owns virtual pages cu[b] / PS + 2 b .. of the launch: at least as
// many as its tokens can touch, known without the lengths before it.
constexpr int kPageRows = kRopeTokens * kPageHeads;
struct PageShared {
  float rows[kPageRows][256 + 4];
  float max[kPageRows];               // of a row's magnitudes
  float scale[kPageRows], inv[kPageRows];
  int ok[kPageRows];                  // whether it is a new token
};

template <int T, int LG, bool GENERAL>
__device__ __forceinline__ void do_page(const RopeArgs& a, int block, PageShared& sh) {
  const int pairs = (a.KH + kPageHeads - 1) / kPageHeads;
  const int vpage = block / (2 * pairs), kv = block / pairs % 2, head0 = block % pairs * kPageHeads;
  const auto vfirst = [&](int b) { return clamp_int(a.cu[b], 0, a.N) / a.PS + 2 * b; };
  int lo = 0, hi = a.B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (vfirst(mid) <= vpage)
      lo = mid;
    else
      hi = mid - 1;
  }
  const int c0 = clamp_int(a.cu[lo], 0, a.N), c1 = clamp_int(a.cu[lo + 1], 0, a.N), j = vpage - vfirst(lo);
  if (c1 <= c0 || j < 0) return;
  const int len = a.lens[lo], start = len - (c1 - c0), from = max(start, 0);
  const int pi = from / a.PS + j;
  if (pi >= a.max_pp) return;
  const int page_pos = pi * a.PS;
  if (page_pos >= len) return;
  const int pid = page_at(a, lo, page_pos);
  if (pid < 0) return;
  const int s0 = max(from, page_pos) - page_pos, s1 = min(len - page_pos, a.PS);  // its new slots
  if (s0 >= s1) return;
  const int heads = min(kPageHeads, a.KH - head0);
  uint8_t* const dst0 = a.pool + a.layer_off + (long long)pid * a.g.page + (long long)head0 * a.g.head + (kv ? a.g.kv : 0);
  float* const sc0 =
      a.scales + a.s_layer_off + (long long)pid * a.g.s_page + (long long)head0 * a.g.s_head + (kv ? a.g.s_kv : 0);
  const int tid = threadIdx.x, lane = tid & 63;
  const int D = a.D;
  const void *src, *w = nullptr;
  long long src_n, src_h;
  if (kv) {
    src = a.v, src_n = a.v_n, src_h = a.v_h;
  } else {
    src = a.k, w = a.kw, src_n = a.k_n, src_h = a.k_h;
  }
  const bool turn = a.cos_sin && kv == 0;

  // rows of slots c .. c + 15 (row i: slot c + i % 16 of head i / 16) into LDS
  const auto fill = [&](int c) {
    constexpr int kLanes = GENERAL ? 64 : LG;
    Lane ln;
    if constexpr (!GENERAL) {
      ln.p = pieces(a, tid & (LG - 1));
      ln.on = 16 * (tid & (LG - 1)) < D;
      load_weights(a, w, ln);
    }
    for (int i = tid / kLanes; i < kPageRows; i += kRopeThreads / kLanes) {
      const int slot = c + i % kRopeTokens, h = i / kRopeTokens;
      const int n = c0 + page_pos + slot - start;
      bool ok = slot >= s0 && slot < s1 && h < heads;
      Token t;
      t.b = lo, t.pos = page_pos + slot, t.angle = t.pos;
      if (ok && a.positions)
        t.angle =
            a.pos_bytes == 8 ? static_cast<const long long*>(a.positions)[n] : static_cast<const int32_t*>(a.positions)[n];
      ok = ok && in_table(a, t);
      const long long at = n * src_n + (head0 + h) * src_h;
      float big = 0.f;
      if constexpr (GENERAL) {
        float* const row = sh.rows[i];
        for (int d = lane; d < D; d += kWave) row[d] = ok ? load1(src, at + d, T) : 0.f;
        __syncwarp();
        if (ok) norm_row(a, w, row);
        float z[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = lane + 64 * e;
          z[e] = d < D ? turned(a, turn && ok, t.angle, row, d) : 0.f;
          big = fmaxf(big, fabsf(z[e]));
        }
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (lane + 64 * e < D) row[lane + 64 * e] = z[e];
        big = group_max<64>(big);
      } else {
        float x[8] = {}, y[8] = {};
        if (ok && ln.on) {
          load8<T>(src, at + ln.p.a, x);
          load8<T>(src, at + ln.p.b, y);
        }
        if (turn && ok) load_angles(a, t.angle, tid & (LG - 1), ln);
        norm_turn<LG>(a, w, turn && ok, ln, x, y);
        if (ln.on) {
#pragma unroll
          for (int e = 0; e < 8; ++e) big = fmaxf(big, fmaxf(fabsf(x[e]), fabsf(y[e])));
          float4* const fx = reinterpret_cast<float4*>(&sh.rows[i][ln.p.a]);
          float4* const fy = reinterpret_cast<float4*>(&sh.rows[i][ln.p.b]);
          fx[0] = make_float4(x[0], x[1], x[2], x[3]), fx[1] = make_float4(x[4], x[5], x[6], x[7]);
          fy[0] = make_float4(y[0], y[1], y[2], y[3]), fy[1] = make_float4(y[4], y[5], y[6], y[7]);
        }
        big = group_max<LG>(big);
      }
      if (tid % kLanes == 0) {
        sh.max[i] = big;
        sh.ok[i] = ok;
        if (!a.fp8) {
          const float s = __fdiv_rn(big, 127.f);
          sh.scale[i] = s;
          sh.inv[i] = __fdiv_rn(1.f, s);
        }
      }
    }
  };

  const int c_first = s0 / kRopeTokens * kRopeTokens;
  const bool once = c_first + kRopeTokens >= s1;
  float scale[kPageHeads] = {}, inv[kPageHeads] = {};
  if (a.fp8) {
    float old[kPageHeads], big[kPageHeads] = {};
#pragma unroll
    for (int h = 0; h < kPageHeads; ++h) old[h] = h < heads && s0 > 0 ? sc0[h * a.g.s_head] : 0.f;
    for (int c = c_first; c < s1; c += kRopeTokens) {
      __syncthreads();
      fill(c);
      __syncthreads();
#pragma unroll
      for (int h = 0; h < kPageHeads; ++h) big[h] = fmaxf(big[h], group_max<16>(sh.max[h * kRopeTokens + (lane & 15)]));
    }
    __syncthreads();  // every thread has the old scales
#pragma unroll
    for (int h = 0; h < kPageHeads; ++h) {
      scale[h] = fmaxf(old[h], __fdiv_rn(big[h], 448.f));
      inv[h] = __fdiv_rn(1.f, scale[h]);
      if (h >= heads) break;
      if (tid == 0) sc0[h * a.g.s_head] = scale[h];
      if (s0 > 0 && scale[h] > old[h]) {  // the page's earlier codes against the new scale
        uint8_t* const dst = dst0 + h * a.g.head;
        for (int i = tid; i < s0 * D; i += kRopeThreads) {
          const int t = i / D, d = i % D;
          uint8_t* p = dst + (kv ? (((t >> 2) * 16 + (d & 15)) * (D >> 4) + (d >> 4)) * 4 + (t & 3) : t * D + d);
          *p = fp8_code(e4m3fn_to_f32(*p) * old[h], scale[h]);
        }
      }
    }
  }
  for (int c = c_first; c < s1; c += kRopeTokens) {
    if (!a.fp8 || !once) {
      __syncthreads();
      fill(c);
      __syncthreads();
    }
#pragma unroll
    for (int h = 0; h < kPageHeads; ++h) {
      if (h >= heads) break;
      const int r0 = h * kRopeTokens;
      uint8_t* const dst = dst0 + h * a.g.head + (long long)c * D;
      float* const sc = sc0 + h * a.g.s_head;
      if (!a.fp8 && tid < kRopeTokens && sh.ok[r0 + tid]) sc[c + tid] = sh.scale[r0 + tid];
      // four codes of (row, dim) .. with their scales
      const auto codes = [&](const float (&x)[4], const float (&s)[4], const float (&y)[4]) -> uint32_t {
        const bool quick = fast_scale(s[0]) && fast_scale(s[1]) && fast_scale(s[2]) && fast_scale(s[3]);
        if (quick) {
          float q[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) q[e] = div_by(x[e], s[e], y[e]);
          if (a.fp8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) q[e] = copysignf(q[e], x[e]);  // -0 stays -0
            int k = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
            k = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], k, true);
            // a NaN's code (seven low bits set): the general path
            if (((~(uint32_t)k & 0x7f7f7f7fu) - 0x01010101u & 0x80808080u) == 0) return (uint32_t)k;
          } else {
            uint32_t k[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              k[e] = __float_as_uint(__fadd_rn(fminf(fmaxf(q[e], -127.f), 127.f), 12582912.f)) & 0xffu;
            return pack4(k[0], k[1], k[2], k[3]);
          }
        }
        uint32_t k[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) k[e] = a.fp8 ? fp8_code(x[e], s[e]) : (uint8_t)int8_code(x[e], s[e]);
        return pack4(k[0], k[1], k[2], k[3]);
      };
      for (int i = tid; i < kRopeTokens * D / 4; i += kRopeThreads) {
        if (kv == 0) {
          const int t = i / (D / 4), d = i % (D / 4) * 4, r = r0 + t;
          if (!sh.ok[r]) continue;
          const float4 f = *reinterpret_cast<const float4*>(&sh.rows[r][d]);
          const float s = a.fp8 ? scale[h] : sh.scale[r], y = a.fp8 ? inv[h] : sh.inv[r];
          *reinterpret_cast<uint32_t*>(dst + (long long)t * D + d) = codes({f.x, f.y, f.z, f.w}, {s, s, s, s}, {y, y, y, y});
        } else {
          const int t = i / D * 4, x = i % D, r = r0 + t;
          const int d = x / (D >> 4) + 16 * (x % (D >> 4));
          const int have = sh.ok[r] | sh.ok[r + 1] << 1 | sh.ok[r + 2] << 2 | sh.ok[r + 3] << 3;
          if (!have) continue;
          float s[4], y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) s[e] = a.fp8 ? scale[h] : sh.scale[r + e], y[e] = a.fp8 ? inv[h] : sh.inv[r + e];
          const uint32_t word = codes({sh.rows[r][d], sh.rows[r + 1][d], sh.rows[r + 2][d], sh.rows[r + 3][d]}, s, y);
          uint8_t* const p = dst + (long long)t * D + x * 4;
          if (have == 15) {
            *reinterpret_cast<uint32_t*>(p) = word;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (have >> e & 1) p[e] = (uint8_t)(word >> (8 * e));
          }
        }
      }
    }
  }
}

template <int T, int LG, bool GENERAL, bool QUANT>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(RopeArgs a) {
  const uint32_t block = blockIdx.y * kGridX + blockIdx.x;
  if constexpr (QUANT) {
    if ((int)block >= a.row_blocks) {
      __shared__ __align__(16) PageShared sh;
      do_page<T, LG, GENERAL>(a, block - a.row_blocks, sh);
      return;
    }
  }
  constexpr int kLanes = GENERAL ? 64 : LG;
  __shared__ float row[GENERAL ? 4 : 1][GENERAL ? 256 : 1];
  const uint32_t unit = block * (kRopeThreads / kLanes) + threadIdx.x / kLanes;
  if (unit < (uint32_t)a.N * a.units) do_unit<T, LG, GENERAL>(a, unit, row[GENERAL ? threadIdx.x / 64 : 0]);
}

template <int T, bool QUANT>
void launch_rope(RopeArgs& a, bool fast, hipStream_t st) {
  const int lg = !fast ? 64 : a.D <= 64 ? 4 : a.D <= 128 ? 8 : 16;
  const long long per = kRopeThreads / lg;
  a.q_units = (a.H + kRopeHeads - 1) / kRopeHeads;
  a.kv_units = (a.KH + kRopeHeads - 1) / kRopeHeads;
  a.units = QUANT ? a.q_units : a.q_units + a.kv_units * (a.pool ? 2 : 1);
  a.units_shift = 0;
  while ((1LL << a.units_shift) < a.units) ++a.units_shift;
  if (a.units > 1) {
    a.units_mul = (uint32_t)(((1ULL << 32) * ((1ULL << a.units_shift) - a.units)) / a.units + 1);
    --a.units_shift;
  }
  a.row_blocks = (int)(((long long)a.N * a.units + per - 1) / per);
  const long long pages =
      QUANT ? ((long long)a.N / a.PS + 2LL * a.B) * 2 * ((a.KH + kPageHeads - 1) / kPageHeads) : 0;
  const uint32_t blocks = (uint32_t)(a.row_blocks + pages);
  if (blocks == 0) return;
  const dim3 grid(blocks < kGridX ? blocks : kGridX, (blocks + kGridX - 1) / kGridX), block(kRopeThreads);
  if (lg == 64)
    hipLaunchKernelGGL((rope_kernel<T, 64, true, QUANT>), grid, block, 0, st, a);
  else if (lg == 4)
    hipLaunchKernelGGL((rope_kernel<T, 4, false, QUANT>), grid, block, 0, st, a);
  else if (lg == 8)
    hipLaunchKernelGGL((rope_kernel<T, 8, false, QUANT>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((rope_kernel<T, 16, false, QUANT>), grid, block, 0, st, a);
}

bool on16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Argument checks that both entries share.
int check_rope(int src_dtype, const float* cos_sin, int rot, int top, const void* qw, const void* kw, int w_dtype, int N,
               int H, int KH, int D, float eps, const char* who) {
  if (N < 0 || H < 0 || KH < 0 || D <= 0 || !(eps >= 0.f)) {
    set_error("%s: bad sizes (N=%d H=%d KH=%d D=%d)", who, N, H, KH, D);
    return VRM_ERR_ARG;
  }
  if (D > 256) {
    set_error("%s: head_dim %d above 256", who, D);
    return VRM_ERR_UNSUPPORTED;
  }
  if (src_dtype != VRM_SRC_F32 && src_dtype != VRM_SRC_F16 && src_dtype != VRM_SRC_BF16) {
    set_error("%s: unknown source dtype %d", who, src_dtype);
    return VRM_ERR_ARG;
  }
  if ((qw || kw) && w_dtype != VRM_SRC_F32 && w_dtype != VRM_SRC_F16 && w_dtype != VRM_SRC_BF16) {
    set_error("%s: unknown weight dtype %d", who, w_dtype);
    return VRM_ERR_ARG;
  }
  if (cos_sin && (rot <= 0 || rot % 2 || rot > D || top <= 0)) {
    set_error("%s: rotary_dim %d must be even and in [2, head_dim %d], over %d > 0 positions", who, rot, D, top);
    return VRM_ERR_ARG;
  }
  if ((long long)N * (H + 2LL * KH) > 0x3fffffffLL) {
    set_error("%s: too many rows (N=%d H=%d KH=%d)", who, N, H, KH);
    return VRM_ERR_UNSUPPORTED;
  }
  return VRM_OK;
}

// Whether every 8-element piece of every row starts on 16 bytes.
bool rope_fast(const RopeArgs& a, int src_dtype) {
  const int per16 = src_dtype == VRM_SRC_F32 ? 4 : 8;
  const auto rows = [&](const void* p, long long n, long long h) { return on16(p) && n % per16 == 0 && h % per16 == 0; };
  if (a.D % 16 || a.rot % 16 || !on16(a.cos_sin) || !on16(a.qw) || !on16(a.kw)) return false;
  if (a.H && (!rows(a.q, a.q_n, a.q_h) || !on16(a.q_out))) return false;
  if (a.KH && (!rows(a.k, a.k_n, a.k_h) || !on16(a.k_out))) return false;
  if (a.pool && (!rows(a.v, a.v_n, a.v_h) || !on16(a.pool))) return false;
  return true;
}

template <bool QUANT>
int run_rope(RopeArgs& a, int src_dtype, hipStream_t st, const char* who) {
  const bool fast = rope_fast(a, src_dtype);
  switch (src_dtype) {
    case VRM_SRC_F32: launch_rope<VRM_SRC_F32, QUANT>(a, fast, st); break;
    case VRM_SRC_F16: launch_rope<VRM_SRC_F16, QUANT>(a, fast, st); break;
    default: launch_rope<VRM_SRC_BF16, QUANT>(a, fast, st); break;
  }
  return launch_status(who);
}

}  // namespace
}  // namespace vrm

using namespace vrm;

extern "C" int vrm_qk_norm_rope(const void* query, long long q_token_stride, long long q_head_stride, const void* key,
                                long long k_token_stride, long long k_head_stride, int src_dtype, const float* cos_sin,
                                int rotary_dim, int max_positions, const void* positions, int position_bytes,
                                const void* q_weight, const void* k_weight, int weight_dtype, float eps,
                                int interleaved, void* query_out, void* key_out, int N, int H, int KH, int D,
                                vrm_stream_t stream) {
  const char* who = "vrm_qk_norm_rope";
  int rc = check_rope(src_dtype, cos_sin, rotary_dim, max_positions, q_weight, k_weight, weight_dtype, N, H, KH, D, eps, who);
  if (rc) return rc;
  if (cos_sin && position_bytes != 4 && position_bytes != 8) {
    set_error("%s: positions must be 4 or 8 byte integers", who);
    return VRM_ERR_ARG;
  }
  if (N == 0 || H + KH == 0) {
    clear_error();
    return VRM_OK;
  }
  if ((H && (!query || !query_out)) || (KH && (!key || !key_out)) || (cos_sin && !positions)) {
    set_error("%s: null pointer argument", who);
    return VRM_ERR_ARG;
  }
  RopeArgs a{};
  a.q = query, a.q_n = q_token_stride, a.q_h = q_head_stride;
  a.k = key, a.k_n = k_token_stride, a.k_h = k_head_stride;
  a.q_out = query_out, a.k_out = key_out;
  a.cos_sin = cos_sin, a.rot = cos_sin ? rotary_dim : 0, a.top = max_positions, a.interleaved = interleaved != 0;
  a.positions = cos_sin ? positions : nullptr, a.pos_bytes = position_bytes;
  a.qw = q_weight, a.kw = k_weight, a.w_type = weight_dtype, a.eps = eps;
  a.N = N, a.H = H, a.KH = KH, a.D = D;
  return run_rope<false>(a, src_dtype, reinterpret_cast<hipStream_t>(stream), who);
}

extern "C" int vrm_rope_append(const void* query, long long q_token_stride, long long q_head_stride, const void* key,
                               long long k_token_stride, long long k_head_stride, const void* value,
                               long long v_token_stride, long long v_head_stride, int src_dtype, const float* cos_sin,
                               int rotary_dim, int max_positions, const void* positions, int position_bytes,
                               const void* q_weight, const void* k_weight, int weight_dtype, float eps, int interleaved,
                               void* query_out, void* kv_pool, float* kv_scales, int kv_dtype,
                               const int32_t* page_table, const int32_t* context_lens, const int32_t* cu_seqlens, int N,
                               int B, int H, int KH, int D, int PS, int L, int P, int max_pp, int layer_idx,
                               vrm_stream_t stream) {
  const char* who = "vrm_rope_append";
  int rc = check_rope(src_dtype, cos_sin, rotary_dim, max_positions, q_weight, k_weight, weight_dtype, N, H, KH, D, eps, who);
  if (rc) return rc;
  if (B < 0 || KH <= 0 || PS <= 0 || L <= 0 || P <= 0 || max_pp < 0) {
    set_error("%s: bad sizes (B=%d KH=%d PS=%d L=%d P=%d max_pp=%d)", who, B, KH, PS, L, P, max_pp);
    return VRM_ERR_ARG;
  }
  if (layer_idx < 0 || layer_idx >= L) {
    set_error("%s: layer_idx %d outside [0, %d)", who, layer_idx, L);
    return VRM_ERR_ARG;
  }
  if (positions && position_bytes != 4 && position_bytes != 8) {
    set_error("%s: positions must be 4 or 8 byte integers", who);
    return VRM_ERR_ARG;
  }
  long long row;
  bool quant = true;
  switch (kv_dtype) {
    case VRM_KV_F32: row = 4LL * D, quant = false; break;
    case VRM_KV_F16:
    case VRM_KV_BF16: row = 2LL * D, quant = false; break;
    case VRM_KV_I8:
    case VRM_KV_I8_INLINE:
    case VRM_KV_FP8E4M3:
    case VRM_KV_FP8E4M3_INLINE: row = D; break;
    default: set_error("%s: unknown kv_dtype %d", who, kv_dtype); return VRM_ERR_ARG;
  }
  if (quant && (D % 16 || PS % 4)) {
    set_error("%s: head_dim %d / page_size %d unsupported over a quantized pool (multiples of 16 / 4)", who, D, PS);
    return VRM_ERR_UNSUPPORTED;
  }
  if (((long long)N / PS + 2LL * B) * 2 * KH > 0x3fffffffLL) {
    set_error("%s: too many pages (N=%d B=%d KH=%d)", who, N, B, KH);
    return VRM_ERR_UNSUPPORTED;
  }
  if (N == 0 || B == 0) {
    clear_error();
    return VRM_OK;
  }
  if ((H && (!query || !query_out)) || !key || !value || !kv_pool || !context_lens || !cu_seqlens ||
      (max_pp > 0 && !page_table)) {
    set_error("%s: null pointer argument", who);
    return VRM_ERR_ARG;
  }
  if (quant != (kv_scales != nullptr)) {
    set_error("%s: kv_scales is for int8 and fp8 pools, and they need it", who);
    return VRM_ERR_ARG;
  }
  if (quant) {
    if (!on16(kv_pool)) {
      set_error("%s: a quantized pool must be 16-byte aligned", who);
      return VRM_ERR_ARG;
    }
    rc = check_pool_scales(kv_dtype, kv_pool, kv_scales, KH, PS, D, L, P, who);
    if (rc) return rc;
  }
  RopeArgs a{};
  a.q = query, a.q_n = q_token_stride, a.q_h = q_head_stride;
  a.k = key, a.k_n = k_token_stride, a.k_h = k_head_stride;
  a.v = value, a.v_n = v_token_stride, a.v_h = v_head_stride;
  a.q_out = query_out;
  a.cos_sin = cos_sin, a.rot = cos_sin ? rotary_dim : 0, a.top = max_positions, a.interleaved = interleaved != 0;
  a.positions = cos_sin ? positions : nullptr, a.pos_bytes = position_bytes;
  a.qw = q_weight, a.kw = k_weight, a.w_type = weight_dtype, a.eps = eps;
  a.N = N, a.H = H, a.KH = KH, a.D = D;
  a.pool = static_cast<uint8_t*>(kv_pool);
  a.scales = kv_scales;
  a.g = pool_geom(kv_dtype, KH, PS, D, row, P, L);
  a.layer_off = (long long)layer_idx * a.g.layer;
  a.s_layer_off = (long long)layer_idx * a.g.s_layer;
  a.kv_dtype = kv_dtype;
  a.fp8 = kv_dtype == VRM_KV_FP8E4M3 || kv_dtype == VRM_KV_FP8E4M3_INLINE;
  a.table = page_table, a.lens = context_lens, a.cu = cu_seqlens;
  a.B = B, a.PS = PS, a.P = P, a.max_pp = max_pp;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return quant ? run_rope<true>(a, src_dtype, st, who) : run_rope<false>(a, src_dtype, st, who);
}
