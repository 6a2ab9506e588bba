// The step of a serving loop between the projections and paged attention: RMS norm (optional) and rotation of every query
// and key head, queries into a tensor of their own, keys beside their values into the paged caches, of 16 bits or of 8
// (e4m3 codes with an fp32 scale for each block and kv head).  One launch; a decode step is bound by its chain of
// dependent loads (length, table, scale), a prompt by HBM: 4 bytes an element of q, 4 or 3 of k and of v.
//
// A token's sequence, place and block come from query_starts, context_lens and block_tables, so all new tokens that fall
// into one block are known to one warp: its scale, codes that move because the scale grew, and its new codes have one
// writer and no atomic.  (Addressing by slots would leave the tokens of a block to whoever finds them.)
//
// Scales are powers of two, the least that holds the block.  That costs a floating code nothing (e4m3 has the same
// relative step at every exponent), and when a later token needs a larger one the old codes only move in exponent: exact
// but below 2^-6 of the new scale, where e4m3 loses bits.  A block filled token by token is the block filled at once.
// An e4m3 code jumps at its borders, and so does a scale: a key is worked out in 64 bits and taken to fp32 by rounding to odd
// (truncated, the last bit set if anything was lost), which keeps comparisons and the second rounding right under a scale that is
// a power of two (another one, in a cache that was not filled here: divide_units()).  (fp32 with a
// known error and 64 bits only where that leaves two codes: slower, 7.3 us for 4.5 at 64 single tokens, 53 for 44 at 5800
// rows of prompts.  Some warp always has such an element, and the second way costs the first one its registers.)

#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "flagattn_b200.h"
#include "rotary_common.cuh"

namespace fa {

constexpr int kCacheThreads = 128;
constexpr int kTile = 32;     // rows whose units a CTA of the 8-bit part finds at once, one a lane
constexpr int kAhead = 4;     // heads of a row whose loads are in flight
// passes over a unit whose values wait for its scale in shared memory, 8 KB each (blocks of 64 tokens, head 128, 5800 rows of
// prompts: 64 us, worked out twice 81)
constexpr int kKept = 3;

struct RotaryCache {
  fa_rotary_cache_args p;
  int unit_ctas;    // CTAs of the unit part, in front
  int per_cta;      // heads one of them walks
  int chunks;       // CTAs that share a group of tokens, and how many of them have heads of q, of k and of v
  int chunks_of[3];
  int unit_ctas_y;  // CTAs that share a tile of rows
  int unit_heads;   // heads of a block that a CTA takes in turn, and how many CTAs that is for k or v
  int unit_chunks;
};

__device__ __forceinline__ uint4 read16(const void *p) { return *reinterpret_cast<const uint4 *>(p); }

// ---- where a token goes ------------------------------------------------------------------------------------------------
struct Token {
  int seq, place, left;   // left: new tokens of its sequence from this one on
  bool first, valid;      // first: of its sequence's new tokens
};
// Called by whole warps; every lane has a row of its own (row >= num_tokens: none).
__device__ __forceinline__ Token find_token(const fa_rotary_cache_args &p, int row) {
  Token t{row, 0, 1, true, false};
  int to_end = 1;   // `left`, and those tokens of its sequence that the call has no rows for
  if (p.query_starts) {
    // the last start that is not behind the row, 32 starts at a time: their loads do not depend on one another
    int before = 0;
    for (int base = 0; base <= p.num_seqs; base += 32) {
      const int i = base + (int)(threadIdx.x & 31);
      const int start = i <= p.num_seqs ? p.query_starts[i] : INT_MAX;
      int at = 0;
#pragma unroll
      for (int step = 16; step; step /= 2)
        if (__shfl_sync(0xffffffffu, start, at + step - 1) <= row) at += step;
      if (__shfl_sync(0xffffffffu, start, at) <= row) ++at;
      before += at;
    }
    t.seq = before - 1;
    if (t.seq < 0 || t.seq >= p.num_seqs || row >= p.num_tokens) return t;
    const int end = p.query_starts[t.seq + 1];
    to_end = end - row, t.left = min(end, p.num_tokens) - row;
    t.first = row == p.query_starts[t.seq];
  } else if (row >= p.num_tokens) {
    return t;
  }
  const int len = p.context_lens[t.seq];
  if (to_end > len) return t;   // in front of its sequence
  t.place = len - to_end;
  t.valid = t.left > 0 && t.place / p.block_size < p.table_cols;
  return t;
}
// The block that holds logical block `i` of a sequence, or -1 for an id outside the cache.
__device__ __forceinline__ int64_t block_of(const fa_rotary_cache_args &p, int seq, int i) {
  const int64_t at = (int64_t)seq * p.bt_stride_s + i;
  const int64_t id = p.block_table_is_i64 ? static_cast<const int64_t *>(p.block_tables)[at]
                                          : (int64_t) static_cast<const int32_t *>(p.block_tables)[at];
  return id >= 0 && id < p.num_blocks ? id : -1;
}
__device__ __forceinline__ int64_t table_row(const fa_rotary_cache_args &p, int row, int place) {
  const int64_t pos = p.positions ? p.positions[row] : place;
  return pos < 0 ? 0 : (pos >= p.table_rows ? p.table_rows - 1 : pos);
}

// ---- a thread's sixteen elements of a row --------------------------------------------------------------------------------
template <int LPR, bool IL>
struct Lane {
  int j, off_a, off_b;
  bool turns;
  __device__ __forceinline__ explicit Lane(int rotary_dim) {
    j = threadIdx.x % LPR;
    turns = j < rotary_dim / 16;
    off_a = IL || !turns ? 16 * j : 8 * j;
    off_b = IL || !turns ? 16 * j + 8 : rotary_dim / 2 + 8 * j;
  }
  __device__ __forceinline__ void angles(const fa_rotary_cache_args &p, int64_t row, bool here, float (&c)[8],
                                         float (&s)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = 1.f, s[i] = 0.f;
    if (turns && here) {
      const int64_t at = row * (p.rotary_dim / 2) + 8 * j;
      load8(c, p.cos + at);
      load8(s, p.sin + at);
    }
  }
  template <typename T>
  __device__ __forceinline__ void weights(const fa_rotary_cache_args &p, const void *w, float (&lo)[8],
                                          float (&hi)[8]) const {
    float a[8], b[8];
    if (p.weight_is_f32) {
      load8(a, static_cast<const float *>(w) + off_a);
      load8(b, static_cast<const float *>(w) + off_b);
    } else {
      unpack8<T>(a, read16(static_cast<const T *>(w) + off_a));
      unpack8<T>(b, read16(static_cast<const T *>(w) + off_b));
    }
    to_pairs<IL>(lo, hi, a, b);
  }
};
template <int LPR, typename F>
__device__ __forceinline__ F lanes_sum(F v) {
#pragma unroll
  for (int m = 1; m < LPR; m *= 2) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

// ---- rows: queries, and with a 16-bit cache keys and values --------------------------------------------------------------
template <typename T, int LPR, bool IL>
__device__ __forceinline__ void row_part(const RotaryCache &a) {
  const fa_rotary_cache_args &p = a.p;
  constexpr int kRows = kCacheThreads / LPR;
  const Lane<LPR, IL> lane(p.rotary_dim);
  const unsigned cta = blockIdx.x - a.unit_ctas;
  int z = cta % a.chunks;
  const int row = (int)(cta / a.chunks) * kRows + (int)threadIdx.x / LPR;
  const bool here = row < p.num_tokens;
  // a CTA has heads of q, of k or of v
  int kind = 0;
  if (z >= a.chunks_of[0]) z -= a.chunks_of[0], kind = 1;
  if (kind && z >= a.chunks_of[1]) z -= a.chunks_of[1], kind = 2;
  const int heads = kind ? p.num_kv_heads : p.num_q_heads;
  const int h_lo = z * a.per_cta, count = min(heads - h_lo, a.per_cta);
  const int64_t src_h = kind == 0 ? p.q_stride_h : kind == 1 ? p.k_stride_h : p.v_stride_h;
  const T *src = static_cast<const T *>(kind == 0 ? p.query : kind == 1 ? p.key : p.value) +
                 row * (kind == 0 ? p.q_stride_t : kind == 1 ? p.k_stride_t : p.v_stride_t) + h_lo * src_h;
  uint4 ua[kAhead], ub[kAhead];
  auto load = [&](int left) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      ua[u] = ub[u] = make_uint4(0, 0, 0, 0);
      if (here && u < left) {
        ua[u] = read16(src + lane.off_a);
        ub[u] = read16(src + lane.off_b);
      }
      src += src_h;
    }
  };
  load(count);   // in flight while the rows' places are found
  const Token t = find_token(p, row);
  T *dst;
  int64_t dst_h = kind ? p.kv_stride_h : p.o_stride_h;
  bool writes = here;
  if (kind) {
    const int64_t blk = t.valid ? block_of(p, t.seq, t.place / p.block_size) : -1;
    writes = blk >= 0;
    dst = static_cast<T *>(kind == 1 ? p.key_cache : p.value_cache) + max(blk, (int64_t)0) * p.kv_stride_b +
          (int64_t)(t.place % p.block_size) * p.kv_stride_t;
  } else {
    dst = static_cast<T *>(p.out) + row * p.o_stride_t;
  }
  dst += h_lo * dst_h;
  auto store = [&](int u) {
    if (writes) {
      *reinterpret_cast<uint4 *>(dst + lane.off_a) = ua[u];
      *reinterpret_cast<uint4 *>(dst + lane.off_b) = ub[u];
    }
    dst += dst_h;
  };
  if (kind == 2) {
    for (int left = count;;) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (u < left) store(u);
      if ((left -= kAhead) <= 0) return;
      load(left);
    }
  }
  // the rotation and the weights in one: y_lo = r (x_lo ll - x_hi lh), y_hi = r (x_hi hh + x_lo hl)
  float ll[8], lh[8], hh[8], hl[8];
  lane.angles(p, t.valid ? table_row(p, row, t.place) : 0, t.valid, ll, lh);
  const bool norm = p.q_weight != nullptr;
  {
    float wlo[8], whi[8];
    if (norm) lane.template weights<T>(p, kind ? p.k_weight : p.q_weight, wlo, whi);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c = ll[i], s = lh[i], l = norm ? wlo[i] : 1.f, h = norm ? whi[i] : 1.f;
      ll[i] = c * l, hh[i] = c * h, lh[i] = lane.turns ? s * h : 0.f, hl[i] = lane.turns ? s * l : 0.f;
    }
  }
  const float inv_d = 1.f / p.head_size;
  for (int left = count;;) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (u >= left) break;   // the same for the whole CTA
      float va[8], vb[8], lo[8], hi[8], ylo[8], yhi[8];
      unpack8<T>(va, ua[u]);
      unpack8<T>(vb, ub[u]);
      float r = 1.f;
      if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(va[i], va[i], fmaf(vb[i], vb[i], ss));
        r = rsqrtf(fmaf(lanes_sum<LPR>(ss), inv_d, p.eps));
      }
      to_pairs<IL>(lo, hi, va, vb);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // (elements that only pass have no partner: 0 times an infinity would be NaN)
        ylo[i] = (lo[i] * ll[i] - (lane.turns ? hi[i] : 0.f) * lh[i]) * r;
        yhi[i] = (hi[i] * hh[i] + (lane.turns ? lo[i] : 0.f) * hl[i]) * r;
      }
      from_pairs<IL>(va, vb, ylo, yhi);
      ua[u] = pack8<T>(va), ub[u] = pack8<T>(vb);
      if (!t.valid) ua[u] = ub[u] = make_uint4(0, 0, 0, 0);   // (whatever the row holds)
      store(u);
    }
    if ((left -= kAhead) <= 0) return;
    load(left);
  }
}

// ---- units of an 8-bit cache: the new tokens of one block and kv head, of k or of v --------------------------------------
// Taken by a CTA, a row of a pass to each group of lanes; or by a warp where every unit is one token.
// fp32 by rounding to odd: between the 64-bit value and any number of fewer bits it compares as the value does, and
// rounds to where the value would
__device__ __forceinline__ float to_odd(double v) {
  const float f = __double2float_rz(v);
  return (double)f == v || f != f ? f : __uint_as_float(__float_as_uint(f) | 1u);
}
__device__ __forceinline__ uint32_t pack_e4m3(float x, float y, float z, float w) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(lo) : "f"(y), "f"(x));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(hi) : "f"(w), "f"(z));
  return (uint32_t)lo | (uint32_t)hi << 16;
}
__device__ __forceinline__ float2 unpack_e4m3(uint16_t two) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(h2) : "h"(two));
  return Elem<__half>::unpack(h2);
}
// the least power of two s with bits <= 448 s = 1.75 2^8 s, of a finite non-negative number's bits
__device__ __forceinline__ float scale_for(uint32_t bits) {
  const int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);   // biased
  return __uint_as_float((uint32_t)max(e, 1) << 23);
}

// A key's pairs (lo, hi) normed and rotated in 64 bits: f(k, lo[k], hi[k]).  Whole warps.
template <typename T, int LPR, bool IL, typename F>
__device__ __forceinline__ void key_pairs(const fa_rotary_cache_args &p, const Lane<LPR, IL> &lane, const float (&c)[8],
                                          const float (&s)[8], const float (&lo)[8], const float (&hi)[8], F f) {
  float wlo[8], whi[8];
  double r = 1.0;
  if (p.k_weight) {
    double ss = 0.0;
#pragma unroll
    for (int k = 0; k < 8; ++k) ss += (double)lo[k] * lo[k] + (double)hi[k] * hi[k];
    r = 1.0 / sqrt(lanes_sum<LPR>(ss) / p.head_size + ((double)p.eps + p.eps_low));
    lane.template weights<T>(p, p.k_weight, wlo, whi);
  }
  if (lane.turns) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      double l = lo[k], h = hi[k];
      if (p.k_weight) l *= r * wlo[k], h *= r * whi[k];
      f(k, l * c[k] - h * s[k], h * c[k] + l * s[k]);
    }
  } else if (p.k_weight) {   // elements that only pass have no partner: 0 times an infinity would be NaN
#pragma unroll
    for (int k = 0; k < 8; ++k) f(k, lo[k] * (r * wlo[k]), hi[k] * (r * whi[k]));
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) f(k, (double)lo[k], (double)hi[k]);
  }
}

// The threads that work on a unit, TEAM of them, and the row of a pass that each has a part of.
template <typename T, int LPR, bool IL, int TEAM>
struct Unit {
  static constexpr int kRowsPass = TEAM / LPR;
  const fa_rotary_cache_args &p;
  const Lane<LPR, IL> &lane;
  int row0, place0, n;   // first token: its row and place; tokens of the unit
  bool key;

  static __device__ __forceinline__ int thread() { return threadIdx.x % TEAM; }
  static __device__ __forceinline__ int row_of(int pass) { return pass * kRowsPass + thread() / LPR; }

  __device__ __forceinline__ const T *source(int i, int head) const {
    return key ? static_cast<const T *>(p.key) + (row0 + i) * p.k_stride_t + head * p.k_stride_h
               : static_cast<const T *>(p.value) + (row0 + i) * p.v_stride_t + head * p.v_stride_h;
  }
  __device__ __forceinline__ void load(int pass, int head, uint4 (&u)[2]) const {
    const int i = row_of(pass);
    u[0] = u[1] = make_uint4(0, 0, 0, 0);
    if (i < n) {
      const T *src = source(i, head);
      u[0] = read16(src + lane.off_a);
      u[1] = read16(src + lane.off_b);
    }
  }
  __device__ __forceinline__ void angles(int pass, float (&c)[8], float (&s)[8]) const {
    const int i = row_of(pass);
    if (key) lane.angles(p, i < n ? table_row(p, row0 + i, place0 + i) : 0, i < n, c, s);
  }
  // fp32 values of what load() brought, of a key from 64 bits
  __device__ __forceinline__ void values(const uint4 (&u)[2], const float (&c)[8], const float (&s)[8], float (&lo)[8],
                                         float (&hi)[8]) const {
    float va[8], vb[8];
    unpack8<T>(va, u[0]);
    unpack8<T>(vb, u[1]);
    to_pairs<IL>(lo, hi, va, vb);
    if (key)
      key_pairs<T>(p, lane, c, s, lo, hi, [&](int k, double l, double h) { lo[k] = to_odd(l), hi[k] = to_odd(h); });
  }
  __device__ __forceinline__ uint32_t largest(int pass, const float (&lo)[8], const float (&hi)[8]) const {
    float most = 0.f;   // an infinity saturates, a NaN stays one (a maximum passes over it): no scale holds them
#pragma unroll
    for (int k = 0; k < 8; ++k) most = fmaxf(most, fmaxf(fabsf(lo[k]), fabsf(hi[k])));
    if (most == INFINITY) {
      most = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (fabsf(lo[k]) < INFINITY) most = fmaxf(most, fabsf(lo[k]));
        if (fabsf(hi[k]) < INFINITY) most = fmaxf(most, fabsf(hi[k]));
      }
    }
    return row_of(pass) < n ? __float_as_uint(most) : 0u;
  }
  __device__ __forceinline__ void store(int pass, const float (&lo)[8], const float (&hi)[8], float scale,
                                        uint8_t *dst) const {
    const int i = row_of(pass);
    if (i >= n) return;
    const float inv = 1.f / scale;   // (products with it are exact)
    float x[8], y[8], a[8], b[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = lo[k] * inv, y[k] = hi[k] * inv;
    from_pairs<IL>(a, b, x, y);
    uint8_t *at = dst + i * p.kv_stride_t;
    *reinterpret_cast<uint2 *>(at + lane.off_a) =
        make_uint2(pack_e4m3(a[0], a[1], a[2], a[3]), pack_e4m3(a[4], a[5], a[6], a[7]));
    *reinterpret_cast<uint2 *>(at + lane.off_b) =
        make_uint2(pack_e4m3(b[0], b[1], b[2], b[3]), pack_e4m3(b[4], b[5], b[6], b[7]));
  }
};

// codes of `rows` rows by `ratio` < 1, `threads` threads of which this is the `thread`-th
__device__ __forceinline__ void move_codes(uint8_t *dst, int64_t stride, int rows, int head_size, double ratio, int thread,
                                           int threads) {
  const int per_row = head_size / 16;
#pragma unroll 1
  for (int i = thread; i < rows * per_row; i += threads) {
    uint4 *at = reinterpret_cast<uint4 *>(dst + (i / per_row) * stride + i % per_row * 16);
    const uint4 u = *at;
    uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 a = unpack_e4m3((uint16_t)w[k]), b = unpack_e4m3((uint16_t)(w[k] >> 16));
      w[k] = pack_e4m3(to_odd(a.x * ratio), to_odd(a.y * ratio), to_odd(b.x * ratio), to_odd(b.y * ratio));
    }
    *at = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// The units of a block's heads [h_lo, h_hi), one after another: the next head's loads are in flight, and the rows' angles
// stay in registers.  `kept` has room for the values of kKept passes.  Returns the mantissas of their scales, 0 where those are
// powers of two.
template <typename T, int LPR, bool IL, int TEAM>
__device__ __forceinline__ uint32_t units_of(const fa_rotary_cache_args &p, const Lane<LPR, IL> &lane, int row, int seq, int place,
                                         int left, int h_lo, int h_hi, bool key, uint32_t *shared_most, float4 *kept) {
  constexpr int kWarps = TEAM / 32;
  const int off = place % p.block_size;
  const Unit<T, LPR, IL, TEAM> u{p, lane, row, place, min(left, p.block_size - off), key};
  const int passes = (u.n + u.kRowsPass - 1) / u.kRowsPass;
  uint4 x[2];
  float c[8], s[8], lo[8], hi[8];
  u.load(0, h_lo, x);
  u.angles(0, c, s);
  const int64_t blk = block_of(p, seq, place / p.block_size);
  if (blk < 0) return 0;   // (the same for the whole team)
  float *scales = (key ? p.key_scales : p.value_scales) + blk * p.num_kv_heads;
  uint8_t *caches = static_cast<uint8_t *>(key ? p.key_cache : p.value_cache) + blk * p.kv_stride_b;
  uint32_t mantissas = 0;
#pragma unroll 1
  for (int h = h_lo; h < h_hi; ++h) {
    const float old = off ? scales[h] : 0.f;   // a block's first token: what the block held before is over
    uint8_t *cache = caches + h * p.kv_stride_h, *dst = cache + off * p.kv_stride_t;
    // The values' maximum, in one step for each pass; then their codes: of the last pass from registers, of the first
    // ones as they were kept (by the thread that needs them again), of those between by the same steps once more.
    const int steps = passes + max(passes - 1 - kKept, 0);
    const auto pass_of = [&](int step) { return step < passes ? step : step - passes + kKept; };
    uint32_t most = 0;
    float now = 0.f;
#pragma unroll 1
    for (int step = 0; step < steps; ++step) {
      const int pass = pass_of(step), next = step + 1 < steps ? pass_of(step + 1) : 0;
      u.values(x, c, s, lo, hi);
      // what the next step works on, under the rest of this one
      if (step + 1 < steps || h + 1 < h_hi) {
        u.load(next, step + 1 < steps ? h : h + 1, x);
        if (passes > 1) u.angles(next, c, s);
      }
      if (step < passes) most = max(most, u.largest(pass, lo, hi));
      if (step < kKept && step + 1 < passes) {
        float4 *at = kept + step * 4 * TEAM + u.thread();
        at[0] = make_float4(lo[0], lo[1], lo[2], lo[3]), at[TEAM] = make_float4(lo[4], lo[5], lo[6], lo[7]);
        at[2 * TEAM] = make_float4(hi[0], hi[1], hi[2], hi[3]), at[3 * TEAM] = make_float4(hi[4], hi[5], hi[6], hi[7]);
      }
      if (step == passes - 1) {
        most = __reduce_max_sync(0xffffffffu, most);
        if (kWarps > 1) {   // the team's
          uint32_t *shared = shared_most + (h & 1) * kWarps;   // (no warp is a whole head ahead of another)
          if ((threadIdx.x & 31) == 0) shared[threadIdx.x / 32] = most;
          __syncthreads();   // (and every thread has its old scale)
#pragma unroll
          for (int w = 0; w < kWarps; ++w) most = max(most, shared[w]);
        }
        now = scale_for(most);
        now = fmaxf(old, now);
        mantissas |= __float_as_uint(now) & 0x7fffffu;
        if (off && now > old)
          move_codes(cache, p.kv_stride_t, off, p.head_size, (double)old / (double)now, u.thread(), TEAM);
      }
      if (step >= passes - 1) u.store(pass, lo, hi, now, dst);
    }
    if (kWarps > 1) {
#pragma unroll 1
      for (int pass = 0; pass < min(kKept, passes - 1); ++pass) {
        const float4 *at = kept + pass * 4 * TEAM + u.thread();
        const float4 v[4] = {at[0], at[TEAM], at[2 * TEAM], at[3 * TEAM]};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          lo[4 * k] = v[k].x, lo[4 * k + 1] = v[k].y, lo[4 * k + 2] = v[k].z, lo[4 * k + 3] = v[k].w;
          hi[4 * k] = v[2 + k].x, hi[4 * k + 1] = v[2 + k].y, hi[4 * k + 2] = v[2 + k].z, hi[4 * k + 3] = v[2 + k].w;
        }
        u.store(pass, lo, hi, now, dst);
      }
    }
    if (u.thread() == 0) scales[h] = now;
  }
  return mantissas;
}

// The codes of those heads whose scale is no power of two, which only a cache that someone else filled has, once more from
// the operands.  A border between two codes times such a scale has up to 29 bits, so neither the 24 bits of a key tell on
// which side of it the key is, nor does a product with the scale's reciprocal.
template <typename T, int LPR, bool IL, int TEAM>
__device__ __forceinline__ void divide_units(const fa_rotary_cache_args &p, const Lane<LPR, IL> &lane, int row, int seq,
                                             int place, int left, int h_lo, int h_hi, bool key) {
  const int off = place % p.block_size;
  const Unit<T, LPR, IL, TEAM> u{p, lane, row, place, min(left, p.block_size - off), key};
  const int64_t blk = block_of(p, seq, place / p.block_size);
  if (blk < 0) return;
  const float *scales = (key ? p.key_scales : p.value_scales) + blk * p.num_kv_heads;
  uint8_t *caches = static_cast<uint8_t *>(key ? p.key_cache : p.value_cache) + blk * p.kv_stride_b;
#pragma unroll 1
  for (int h = h_lo; h < h_hi; ++h) {
    const float scale = scales[h];
    if ((__float_as_uint(scale) & 0x7fffffu) == 0) continue;
#pragma unroll 1
    for (int pass = 0; pass * u.kRowsPass < u.n; ++pass) {
      uint4 x[2];
      float c[8], s[8], va[8], vb[8], lo[8], hi[8];
      u.load(pass, h, x);
      u.angles(pass, c, s);
      unpack8<T>(va, x[0]);
      unpack8<T>(vb, x[1]);
      to_pairs<IL>(lo, hi, va, vb);
      const auto code = [&](int k, double l, double h) { lo[k] = to_odd(l / scale), hi[k] = to_odd(h / scale); };
      if (key) {
        key_pairs<T>(p, lane, c, s, lo, hi, code);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) code(k, lo[k], hi[k]);
      }
      u.store(pass, lo, hi, 1.f, caches + h * p.kv_stride_h + off * p.kv_stride_t);
    }
  }
}

// A CTA's units, f(team, row, seq, place, left, first head, last + 1, key) each: by the CTA's threads or by a warp's.
template <int N>
using Team = std::integral_constant<int, N>;
template <bool ONE, typename F>
__device__ __forceinline__ void each_units(const RotaryCache &a, F f) {
  const fa_rotary_cache_args &p = a.p;
  const int per_row = 2 * p.num_kv_heads, warp = threadIdx.x / 32, lane_id = threadIdx.x & 31;
  if (ONE) {
    const int64_t i = (int64_t)blockIdx.x * (kCacheThreads / 32) + warp;
    const int row = (int)(i / per_row), rest = (int)(i % per_row);
    if (row >= p.num_tokens) return;
    const Token t = find_token(p, row);
    if (t.valid) f(Team<32>(), row, t.seq, t.place, 1, rest / 2, rest / 2 + 1, rest % 2 == 0);
    return;
  }
  const int tile = blockIdx.x / a.unit_ctas_y, y = blockIdx.x % a.unit_ctas_y;
  const Token t = find_token(p, tile * kTile + lane_id);
  const bool leads = t.valid && (t.first || t.place == 0 || t.place % p.block_size == 0);
  const unsigned several = __ballot_sync(0xffffffffu, leads && t.left > 1), single = __ballot_sync(0xffffffffu, leads && t.left == 1);
  auto from_lane = [&](int x, int from) { return __shfl_sync(0xffffffffu, x, from); };
  // blocks that take several tokens: a CTA for each and some of its heads, of k or of v
  const int per_block = 2 * a.unit_chunks, items = __popc(several) * per_block;
  for (int i = y; i < items; i += a.unit_ctas_y) {
    const int from = __fns(several, 0, i / per_block + 1), rest = i % per_block, h = rest / 2 * a.unit_heads;
    f(Team<kCacheThreads>(), tile * kTile + from, from_lane(t.seq, from), from_lane(t.place, from), from_lane(t.left, from), h,
      min(h + a.unit_heads, p.num_kv_heads), rest % 2 == 0);
    __syncthreads();   // the shared memory is the next one's
  }
  // single tokens: a warp for each and head
  const int ones = __popc(single) * per_row;
  for (int i = y * (kCacheThreads / 32) + warp; i < ones; i += a.unit_ctas_y * (kCacheThreads / 32)) {
    const int from = __fns(single, 0, i / per_row + 1), rest = i % per_row;
    f(Team<32>(), tile * kTile + from, from_lane(t.seq, from), from_lane(t.place, from), 1, rest / 2, rest / 2 + 1,
      rest % 2 == 0);
  }
}

// (a function of its own, at the end, where it takes no registers from the units)
template <typename T, int LPR, bool IL, bool ONE>
__device__ __noinline__ void divide_part(const RotaryCache &a) {
  const Lane<LPR, IL> lane(a.p.rotary_dim);
  each_units<ONE>(a, [&](auto team, int row, int seq, int place, int left, int h_lo, int h_hi, bool key) {
    divide_units<T, LPR, IL, decltype(team)::value>(a.p, lane, row, seq, place, left, h_lo, h_hi, key);
  });
}
template <typename T, int LPR, bool IL, bool ONE>
__device__ __forceinline__ void unit_part(const RotaryCache &a) {
  __shared__ uint32_t shared_most[ONE ? 1 : 2 * kCacheThreads / 32];
  __shared__ float4 kept[ONE ? 1 : kKept * 4 * kCacheThreads];
  const Lane<LPR, IL> lane(a.p.rotary_dim);
  uint32_t mantissas = 0;
  each_units<ONE>(a, [&](auto team, int row, int seq, int place, int left, int h_lo, int h_hi, bool key) {
    mantissas |= units_of<T, LPR, IL, decltype(team)::value>(a.p, lane, row, seq, place, left, h_lo, h_hi, key, shared_most, kept);
  });
  // (with barriers: a team's threads see the scales that one of them wrote)
  if (ONE) __syncwarp();
  if (ONE ? mantissas != 0 : __syncthreads_or(mantissas != 0)) divide_part<T, LPR, IL, ONE>(a);
}

// UNITS: 0 none (a cache of 16 bits), 1 of one token each, 2 of up to a block's (which spill 32 to 68 bytes at 96 registers)
template <typename T, int LPR, bool IL, int UNITS>
__global__ void __launch_bounds__(kCacheThreads, UNITS == 1 ? 4 : 5) rotary_cache_kernel(const __grid_constant__ RotaryCache a) {
  if (UNITS && (int)blockIdx.x < a.unit_ctas) unit_part<T, LPR, IL, UNITS == 1>(a);
  else row_part<T, LPR, IL>(a);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
namespace {

int check_cache(const fa_rotary_cache_args *a) {
  if (!a || (a->dtype != FA_F16 && a->dtype != FA_BF16)) return FA_ERR_BAD_ARG;
  if (a->num_tokens < 0 || a->num_seqs < 0 || a->num_q_heads <= 0 || a->num_kv_heads <= 0 || a->block_size <= 0 ||
      a->num_blocks < 0 || a->table_cols < 0 || a->table_rows <= 0 || a->rotary_dim < 0)
    return FA_ERR_BAD_ARG;
  const int D = a->head_size;
  if (!(D == 16 || D == 32 || D == 64 || D == 128 || D == 256)) return FA_ERR_UNSUPPORTED;
  if (a->rotary_dim % 16 || a->rotary_dim > D) return FA_ERR_UNSUPPORTED;
  if (a->num_tokens == 0) return FA_OK;
  if (!a->query || !a->key || !a->value || !a->out || !a->key_cache || !a->value_cache || !a->context_lens ||
      !a->block_tables || !a->cos || !a->sin)
    return FA_ERR_BAD_ARG;
  if (!a->query_starts && a->num_tokens != a->num_seqs) return FA_ERR_BAD_ARG;
  if (!a->key_scales != !a->value_scales || !a->q_weight != !a->k_weight) return FA_ERR_BAD_ARG;
  for (const void *p : {a->query, a->key, a->value, (const void *)a->out, (const void *)a->key_cache,
                        (const void *)a->value_cache, (const void *)a->cos, (const void *)a->sin, a->q_weight, a->k_weight})
    if (!aligned16(p)) return FA_ERR_ALIGNMENT;
  for (int64_t s : {a->q_stride_t, a->q_stride_h, a->k_stride_t, a->k_stride_h, a->v_stride_t, a->v_stride_h, a->o_stride_t,
                    a->o_stride_h})
    if (s % 8) return FA_ERR_ALIGNMENT;
  for (int64_t s : {a->kv_stride_b, a->kv_stride_h, a->kv_stride_t})
    if (s % (a->key_scales ? 16 : 8)) return FA_ERR_ALIGNMENT;
  return FA_OK;
}

template <typename T, int LPR, bool IL>
int launch_cache(RotaryCache &a, cudaStream_t s) {
  const fa_rotary_cache_args &p = a.p;
  const int rows = kCacheThreads / LPR;
  const int64_t groups = (p.num_tokens + rows - 1) / rows;
  const int heads = p.num_q_heads + (p.key_scales ? 0 : 2 * p.num_kv_heads);
  // heads a thread walks with a token's angles in its registers: up to 8, fewer where the grid would be shallow
  int per = 1;
  while (per < 8 && groups * ((heads + 2 * per - 1) / (2 * per)) >= 148 * 16) per *= 2;
  a.per_cta = per;
  a.chunks_of[0] = (p.num_q_heads + per - 1) / per;
  a.chunks_of[1] = a.chunks_of[2] = p.key_scales ? 0 : (p.num_kv_heads + per - 1) / per;
  a.chunks = a.chunks_of[0] + a.chunks_of[1] + a.chunks_of[2];
  int64_t unit_ctas = 0;
  if (p.key_scales) {
    const int per_row = 2 * p.num_kv_heads;
    if (!p.query_starts) {
      unit_ctas = ((int64_t)p.num_tokens * per_row + kCacheThreads / 32 - 1) / (kCacheThreads / 32);
    } else {
      // A tile of a prompt's rows has a unit for each block it meets, and CTAs for those.  Heads share their rows' angles
      // where a block is one pass of them and units are many (5800 rows of prompts, 8 heads, us: 70 with a head each, 44
      // with 4, 46 with 8); longer blocks are work enough.
      const int64_t tiles = (p.num_tokens + kTile - 1) / kTile, blocks = kTile / p.block_size + 1, ctas = 148 * 5;
      a.unit_heads = p.block_size <= rows && tiles * blocks * per_row > 2 * ctas ? 4 : 1;
      a.unit_chunks = (p.num_kv_heads + a.unit_heads - 1) / a.unit_heads;
      // A tile of short sequences has up to a unit of one warp for each row and head: as many CTAs as the GPU has at once.
      const int64_t most = kTile / (kCacheThreads / 32) * per_row, fill = ctas / tiles;
      a.unit_ctas_y = (int)std::max(2 * a.unit_chunks * blocks, std::min(most, fill));
      unit_ctas = tiles * a.unit_ctas_y;
    }
  }
  const int64_t grid = unit_ctas + groups * a.chunks;
  if (grid >= (1ll << 31)) return FA_ERR_TOO_LARGE;
  a.unit_ctas = (int)unit_ctas;
  auto kern = !p.key_scales ? rotary_cache_kernel<T, LPR, IL, 0>
              : !p.query_starts ? rotary_cache_kernel<T, LPR, IL, 1> : rotary_cache_kernel<T, LPR, IL, 2>;
  kern<<<(unsigned)grid, kCacheThreads, 0, s>>>(a);
  FA_CHECK_LAUNCH();
  return FA_OK;
}
template <typename T, bool IL>
int dispatch_cache(RotaryCache &a, cudaStream_t s) {
  switch (a.p.head_size) {
    case 16: return launch_cache<T, 1, IL>(a, s);
    case 32: return launch_cache<T, 2, IL>(a, s);
    case 64: return launch_cache<T, 4, IL>(a, s);
    case 128: return launch_cache<T, 8, IL>(a, s);
    default: return launch_cache<T, 16, IL>(a, s);
  }
}

}  // namespace
}  // namespace fa

using namespace fa;

extern "C" int fa_rotary_cache(const fa_rotary_cache_args *p, void *stream) {
  if (int st = check_cache(p)) return st;
  if (p->num_tokens == 0) return FA_OK;
  RotaryCache a{};
  a.p = *p;
  auto s = static_cast<cudaStream_t>(stream);
  if (p->dtype == FA_F16) return p->interleaved ? dispatch_cache<__half, true>(a, s) : dispatch_cache<__half, false>(a, s);
  return p->interleaved ? dispatch_cache<__nv_bfloat16, true>(a, s) : dispatch_cache<__nv_bfloat16, false>(a, s);
}
