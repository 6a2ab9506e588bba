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
// An e4m3 code jumps at its borders, so a key is worked out in 64 bits and taken to fp32 by rounding to odd (truncate, and
// set the last bit if anything was lost): that keeps every comparison and the second rounding right.  The 64-bit
// units do it beside the stream: three operations an element of k, a tenth of the elements of a grouped-query layer.
#include <cuda_runtime.h>

#include <climits>
#include <cstdint>

#include "common.cuh"
#include "flagattn_b200.h"
#include "rotary_common.cuh"

namespace fa {

constexpr int kCacheThreads = 128;
constexpr int kTile = 32;     // rows whose units a CTA of the 8-bit part finds at once, one a lane
constexpr int kPasses = 4;    // 16-byte pieces of a thread that stay in registers between the maximum and the codes

struct RotaryCache {
  fa_rotary_cache_args p;
  int unit_ctas;    // CTAs of the unit part, in front: a unit takes longer than a row
  int per_cta;      // heads one of them walks
  int chunks;       // CTAs that share a group of tokens
  int unit_ctas_y;  // 8 bits: CTAs that share a tile of rows
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
    t.left = min(p.query_starts[t.seq + 1], p.num_tokens) - row;
    t.first = row == p.query_starts[t.seq];
  } else if (row >= p.num_tokens) {
    return t;
  }
  const int len = p.context_lens[t.seq];
  if (t.left > len) return t;   // in front of its sequence
  t.place = len - t.left;
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
  const int z = cta % a.chunks, row = (int)(cta / a.chunks) * kRows + (int)threadIdx.x / LPR;
  const Token t = find_token(p, row);
  const bool here = row < p.num_tokens;
  const int heads = p.num_q_heads + (p.key_scales ? 0 : 2 * p.num_kv_heads);
  const int h_lo = z * a.per_cta, h_hi = min(heads, h_lo + a.per_cta);
  const int v_lo = p.num_q_heads + p.num_kv_heads;   // heads from here on are values
  int64_t blk = -1;
  if (h_hi > p.num_q_heads && t.valid) blk = block_of(p, t.seq, t.place / p.block_size);
  const int64_t slot = blk * p.kv_stride_b + (int64_t)(t.place % p.block_size) * p.kv_stride_t;
  float c[8], s[8], wlo[8], whi[8];
  if (h_lo < v_lo) lane.angles(p, t.valid ? table_row(p, row, t.place) : 0, t.valid, c, s);
  const bool norm = p.q_weight != nullptr;
  const float inv_d = 1.f / p.head_size;
  int have = -1;   // whose weights are in the registers: 0 q, 1 k

  for (int h0 = h_lo; h0 < h_hi; h0 += kPasses) {
    uint4 ua[kPasses], ub[kPasses];
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
      const int h = h0 + u;
      ua[u] = ub[u] = make_uint4(0, 0, 0, 0);
      if (!here || h >= h_hi || !t.valid) continue;
      const T *src = h < p.num_q_heads ? static_cast<const T *>(p.query) + row * p.q_stride_t + h * p.q_stride_h
                     : h < v_lo ? static_cast<const T *>(p.key) + row * p.k_stride_t + (h - p.num_q_heads) * p.k_stride_h
                                : static_cast<const T *>(p.value) + row * p.v_stride_t + (h - v_lo) * p.v_stride_h;
      ua[u] = read16(src + lane.off_a);
      ub[u] = read16(src + lane.off_b);
    }
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
      const int h = h0 + u;
      if (h >= h_hi) break;   // (as in all comparisons of h: the same for the whole CTA)
      if (h < v_lo) {
        float va[8], vb[8], lo[8], hi[8], ylo[8], yhi[8];
        unpack8<T>(va, ua[u]);
        unpack8<T>(vb, ub[u]);
        to_pairs<IL>(lo, hi, va, vb);
        if (norm) {
          const int e = h >= p.num_q_heads;
          if (have != e) lane.template weights<T>(p, e ? p.k_weight : p.q_weight, wlo, whi);
          have = e;
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) ss = fmaf(va[i], va[i], fmaf(vb[i], vb[i], ss));
          const float r = rsqrtf(fmaf(lanes_sum<LPR>(ss), inv_d, p.eps));
#pragma unroll
          for (int i = 0; i < 8; ++i) lo[i] *= r * wlo[i], hi[i] *= r * whi[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ylo[i] = lo[i] * c[i] - hi[i] * s[i];
          yhi[i] = hi[i] * c[i] + lo[i] * s[i];
        }
        from_pairs<IL>(va, vb, ylo, yhi);
        if (t.valid) ua[u] = pack8<T>(va), ub[u] = pack8<T>(vb);   // (a row without a place stays 0)
      }
      T *dst;
      if (h < p.num_q_heads) {
        if (!here) continue;
        dst = static_cast<T *>(p.out) + row * p.o_stride_t + h * p.o_stride_h;
      } else {
        if (blk < 0) continue;
        dst = h < v_lo ? static_cast<T *>(p.key_cache) + slot + (h - p.num_q_heads) * p.kv_stride_h
                       : static_cast<T *>(p.value_cache) + slot + (h - v_lo) * p.kv_stride_h;
      }
      *reinterpret_cast<uint4 *>(dst + lane.off_a) = ua[u];
      *reinterpret_cast<uint4 *>(dst + lane.off_b) = ub[u];
    }
  }
}

// ---- units of an 8-bit cache: the new tokens of one block and kv head, of k or of v, one warp ------------------------------
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

template <typename T, int LPR, bool IL>
struct Unit {
  static constexpr int kRowsPass = 32 / LPR;
  static constexpr int kRowsChunk = kRowsPass * kPasses;
  const fa_rotary_cache_args &p;
  const Lane<LPR, IL> &lane;
  const T *src;        // the head's row of the first token
  int64_t src_stride;
  int row0, place0, n;   // first token: its row and place; tokens of the unit
  bool key;

  // fp32 values of this thread's elements of the rows chunk * kRowsChunk + pass * kRowsPass + lane / LPR
  __device__ __forceinline__ void values(int chunk, float (&v)[kPasses][16]) const {
    uint4 ua[kPasses], ub[kPasses];
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
      const int i = chunk * kRowsChunk + u * kRowsPass + (int)(threadIdx.x & 31) / LPR;
      ua[u] = ub[u] = make_uint4(0, 0, 0, 0);
      if (i < n) {
        ua[u] = read16(src + i * src_stride + lane.off_a);
        ub[u] = read16(src + i * src_stride + lane.off_b);
      }
    }
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
      if (chunk * kRowsChunk + u * kRowsPass >= n) break;   // the same for the whole warp
      const int i = chunk * kRowsChunk + u * kRowsPass + (int)(threadIdx.x & 31) / LPR;
      float va[8], vb[8];
      unpack8<T>(va, ua[u]);
      unpack8<T>(vb, ub[u]);
      if (key) {
        float c[8], s[8], lo[8], hi[8], wlo[8], whi[8];
        lane.angles(p, i < n ? table_row(p, row0 + i, place0 + i) : 0, i < n, c, s);
        double r = 1.0;
        if (p.k_weight) {
          double ss = 0.0;
#pragma unroll
          for (int k = 0; k < 8; ++k) ss += (double)va[k] * va[k] + (double)vb[k] * vb[k];
          r = 1.0 / sqrt(lanes_sum<LPR>(ss) / p.head_size + (double)p.eps);
          lane.template weights<T>(p, p.k_weight, wlo, whi);
        }
        to_pairs<IL>(lo, hi, va, vb);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          double l = lo[k], h = hi[k];
          if (p.k_weight) l *= r * wlo[k], h *= r * whi[k];
          lo[k] = to_odd(l * c[k] - h * s[k]);
          hi[k] = to_odd(h * c[k] + l * s[k]);
        }
        from_pairs<IL>(va, vb, lo, hi);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) v[u][k] = va[k], v[u][8 + k] = vb[k];
    }
  }
  __device__ __forceinline__ uint32_t largest(int chunk, const float (&v)[kPasses][16]) const {
    uint32_t most = 0;
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
      if (chunk * kRowsChunk + u * kRowsPass >= n) break;
      if (chunk * kRowsChunk + u * kRowsPass + (int)(threadIdx.x & 31) / LPR < n) {
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const uint32_t bits = __float_as_uint(v[u][k]) & 0x7fffffffu;
          most = max(most, bits < 0x7f800000u ? bits : 0u);   // an infinity saturates, a NaN stays one: no scale holds them
        }
      }
    }
    return most;
  }
  __device__ __forceinline__ void store(int chunk, const float (&v)[kPasses][16], float scale, uint8_t *dst) const {
    const double inv = 1.0 / (double)scale;
    const float inv_f = (float)inv;
    const bool power = (__float_as_uint(scale) & 0x7fffffu) == 0;   // as this kernel leaves them: the product is exact
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
      if (chunk * kRowsChunk + u * kRowsPass >= n) break;
      const int i = chunk * kRowsChunk + u * kRowsPass + (int)(threadIdx.x & 31) / LPR;
      if (i >= n) continue;
      float q[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) q[k] = power ? v[u][k] * inv_f : to_odd((double)v[u][k] * inv);
      uint8_t *at = dst + i * p.kv_stride_t;
      *reinterpret_cast<uint2 *>(at + lane.off_a) =
          make_uint2(pack_e4m3(q[0], q[1], q[2], q[3]), pack_e4m3(q[4], q[5], q[6], q[7]));
      *reinterpret_cast<uint2 *>(at + lane.off_b) =
          make_uint2(pack_e4m3(q[8], q[9], q[10], q[11]), pack_e4m3(q[12], q[13], q[14], q[15]));
    }
  }
};

// codes of `rows` rows by `ratio` < 1
__device__ __forceinline__ void move_codes(uint8_t *dst, int64_t stride, int rows, int head_size, double ratio) {
  const int per_row = head_size / 16;
  for (int i = threadIdx.x & 31; i < rows * per_row; i += 32) {
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

template <typename T, int LPR, bool IL>
__device__ __forceinline__ void unit(const fa_rotary_cache_args &p, const Lane<LPR, IL> &lane, int row, int seq, int place,
                                     int left, int head, bool key) {
  const int64_t blk = block_of(p, seq, place / p.block_size);
  if (blk < 0) return;
  const int off = place % p.block_size;
  const T *src = key ? static_cast<const T *>(p.key) + row * p.k_stride_t + head * p.k_stride_h
                     : static_cast<const T *>(p.value) + row * p.v_stride_t + head * p.v_stride_h;
  const Unit<T, LPR, IL> u{p, lane, src, key ? p.k_stride_t : p.v_stride_t, row, place, min(left, p.block_size - off), key};
  float *scale = (key ? p.key_scales : p.value_scales) + blk * p.num_kv_heads + head;
  uint8_t *cache = static_cast<uint8_t *>(key ? p.key_cache : p.value_cache) + blk * p.kv_stride_b + head * p.kv_stride_h;
  const float old = off ? *scale : 0.f;   // a block's first token: what the block held before is over
  const int chunks = (u.n + u.kRowsChunk - 1) / u.kRowsChunk;
  float v[kPasses][16];
  uint32_t most = 0;
  for (int i = 0; i < chunks; ++i) {
    u.values(i, v);
    most = max(most, u.largest(i, v));
  }
  most = __reduce_max_sync(0xffffffffu, most);
  const float now = fmaxf(old, scale_for(most));
  if (off && now > old) move_codes(cache, p.kv_stride_t, off, p.head_size, (double)old / (double)now);
  uint8_t *dst = cache + off * p.kv_stride_t;
  for (int i = 0; i < chunks; ++i) {
    if (chunks > 1) u.values(i, v);   // what one chunk holds stays in the registers
    u.store(i, v, now, dst);
  }
  if ((threadIdx.x & 31) == 0) *scale = now;
}

template <typename T, int LPR, bool IL>
__device__ __forceinline__ void unit_part(const RotaryCache &a) {
  const fa_rotary_cache_args &p = a.p;
  const Lane<LPR, IL> lane(p.rotary_dim);
  const int cta = blockIdx.x, warp = threadIdx.x / 32;
  const int tile = cta / a.unit_ctas_y, stride = a.unit_ctas_y * (kCacheThreads / 32);
  const int lane_id = threadIdx.x & 31;
  // (one token a sequence: every row is a unit, and a tile has as many as it has rows)
  const Token t = find_token(p, tile * kTile + lane_id);
  const bool leads = t.valid && (t.first || t.place == 0 || t.place % p.block_size == 0);
  const unsigned leaders = __ballot_sync(0xffffffffu, leads);
  const int units = __popc(leaders) * p.num_kv_heads * 2;
  for (int i = cta % a.unit_ctas_y * (kCacheThreads / 32) + warp; i < units; i += stride) {
    const int from = __fns(leaders, 0, i / (2 * p.num_kv_heads) + 1), rest = i % (2 * p.num_kv_heads);
    unit<T, LPR, IL>(p, lane, tile * kTile + from, __shfl_sync(0xffffffffu, t.seq, from),
                     __shfl_sync(0xffffffffu, t.place, from), __shfl_sync(0xffffffffu, t.left, from), rest / 2,
                     rest % 2 == 0);
  }
}

template <typename T, int LPR, bool IL>
__global__ void __launch_bounds__(kCacheThreads) rotary_cache_kernel(const __grid_constant__ RotaryCache a) {
  if ((int)blockIdx.x < a.unit_ctas) unit_part<T, LPR, IL>(a);
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
  while (per < 8 && groups * ((heads + 2 * per - 1) / (2 * per)) >= 148 * 8 * 4) per *= 2;
  a.per_cta = per, a.chunks = (heads + per - 1) / per;
  int64_t unit_ctas = 0;
  if (p.key_scales) {
    const int warps = kCacheThreads / 32, per_row = 2 * p.num_kv_heads;
    // a tile of rows of prompts has a unit for each block it meets, a tile of single tokens one for each row
    const int64_t units = (int64_t)per_row * (p.query_starts ? kTile / p.block_size + 2 : kTile);
    a.unit_ctas_y = (int)((units + warps - 1) / warps);
    unit_ctas = (int64_t)((p.num_tokens + kTile - 1) / kTile) * a.unit_ctas_y;
  }
  const int64_t grid = unit_ctas + groups * a.chunks;
  if (grid >= (1ll << 31)) return FA_ERR_TOO_LARGE;
  a.unit_ctas = (int)unit_ctas;
  rotary_cache_kernel<T, LPR, IL><<<(unsigned)grid, kCacheThreads, 0, s>>>(a);
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
  RotaryCache a{*p, 0, 0, 0, 0};
  auto s = static_cast<cudaStream_t>(stream);
  if (p->dtype == FA_F16) return p->interleaved ? dispatch_cache<__half, true>(a, s) : dispatch_cache<__half, false>(a, s);
  return p->interleaved ? dispatch_cache<__nv_bfloat16, true>(a, s) : dispatch_cache<__nv_bfloat16, false>(a, s);
}
