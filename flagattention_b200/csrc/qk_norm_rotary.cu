// RMS norm of every head of q and k and their rotation by position, in one pass:
//   n = x r w,  r = 1 / sqrt(mean(x^2) + eps);   y = R(p) n on the first `rotary_dim` elements, y = n on the others,
// and its backward:
//   h = R(p)^T g;  dw = sum over rows of h x r;  a = h w;  dx = r (a - x r mean(a x r)).
// All of it is fp32 from 16-bit operands, each result rounded once.  HBM-bound: 4 bytes of traffic an element forward, 6
// backward, some ten operations.
//
// A row's 16 D / 16 elements go to the LPR = 2^k >= D / 16 lanes of a group (rotary_pair's layout: 8 rotation pairs a
// thread in either pair layout, or 16 elements that only pass), so the row's sum is a few shuffles.  A group keeps the
// cos / sin values of its position and the weights in registers and walks heads of that position, the loads of
// `kAhead` heads in flight; q and k share the launch (a small call is bound by launches), a CTA has heads of one of them.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "attn_params.cuh"
#include "common.cuh"
#include "flagattn_b200.h"
#include "rotary_common.cuh"

namespace fa {

constexpr int kNormThreads = 128;
constexpr int kAhead = 4;      // heads whose loads are in flight, forward
constexpr int kForwardCtas = 5, kBackwardCtas = 4;   // resident on an SM
constexpr int kRing = 3;     // backward: heads in flight and in work, 8 KB each

struct NormSide {   // q or k
  const void *x, *g;
  void *y;          // forward: the result; backward: dx
  Strides sx, sg, sy;
  const void *weight;
  int heads;
};
struct NormArgs {
  NormSide side[2];
  const float *cos, *sin;
  const int64_t *positions;
  int64_t pos_stride_b;
  float eps;
  int B, L, D, R, table_rows, weight_is_f32;
  int per_cta[2];   // heads a CTA walks
  int chunks[2];    // and the CTAs that share a position's heads
  int64_t items[2]; // backward: strips of positions x chunks, of q and of k
};

__device__ __forceinline__ uint4 load16(const void *p) { return *reinterpret_cast<const uint4 *>(p); }

template <typename T>
__device__ __forceinline__ void load_weight8(float (&w)[8], const void *weight, int at, bool f32) {
  if (f32) load8(w, static_cast<const float *>(weight) + at);
  else unpack8<T>(w, load16(static_cast<const T *>(weight) + at));
}

// What a thread of a group holds for all its heads.
template <typename T, int LPR, bool IL>
struct NormLane {
  int off_a, off_b, b, l, h_lo, h_hi, e;   // e: 0 q, 1 k
  bool live, turns;
  float c[8], s[8], wlo[8], whi[8];

  __device__ __forceinline__ void columns(const NormArgs &a) {
    const int j = threadIdx.x % LPR;
    turns = j < a.R / 16;
    off_a = IL || !turns ? 16 * j : 8 * j;
    off_b = IL || !turns ? 16 * j + 8 : a.R / 2 + 8 * j;
    live = j < a.D / 16;
  }
  __device__ __forceinline__ void place(const NormArgs &a) {
    columns(a);
    const int Z = a.chunks[0] + a.chunks[1];
    int z = blockIdx.x % Z;
    e = z >= a.chunks[0];
    if (e) z -= a.chunks[0];
    h_lo = z * a.per_cta[e];
    h_hi = min(a.side[e].heads, h_lo + a.per_cta[e]);
    b = (blockIdx.x / Z) % a.B;
  }
  __device__ __forceinline__ void weights(const NormArgs &a) {
    float wa[8], wb[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) wa[i] = wb[i] = 1.f;
    const void *w = a.side[e].weight;
    if (live && w) {
      load_weight8<T>(wa, w, off_a, a.weight_is_f32);
      load_weight8<T>(wb, w, off_b, a.weight_is_f32);
    }
    to_pairs<IL>(wlo, whi, wa, wb);
  }
  // the position of row `row` of the batch element, and its angles
  __device__ __forceinline__ void turn_to(const NormArgs &a, int row) {
    l = row;
    const bool here = live && l < a.L;
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = 1.f, s[i] = 0.f;
    if (here && turns) {
      int64_t pos = a.positions ? a.positions[b * a.pos_stride_b + l] : l;
      // a position outside the tables reads the nearest row instead of foreign memory
      pos = pos < 0 ? 0 : (pos >= a.table_rows ? a.table_rows - 1 : pos);
      const int64_t at = pos * (a.R / 2) + 8 * (threadIdx.x % LPR);
      load8(c, a.cos + at);
      load8(s, a.sin + at);
    }
  }
};

template <int LPR>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int m = 1; m < LPR; m *= 2) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

template <typename T, int LPR, bool IL>
__global__ void __launch_bounds__(kNormThreads, kForwardCtas) qk_norm_rotary_fwd_kernel(const NormArgs a) {
  NormLane<T, LPR, IL> t;
  t.place(a);
  const int rows = kNormThreads / LPR;
  const int Z = a.chunks[0] + a.chunks[1];
  t.turn_to(a, (int)(blockIdx.x / ((unsigned)Z * a.B)) * rows + threadIdx.x / LPR);
  t.weights(a);
  const bool here = t.live && t.l < a.L;
  const NormSide &side = a.side[t.e];
  const T *x = static_cast<const T *>(side.x) + t.b * side.sx.b + (here ? t.l * side.sx.l : 0);
  T *y = static_cast<T *>(side.y) + t.b * side.sy.b + (here ? t.l * side.sy.l : 0);
  const float inv_d = 1.f / a.D;
  // the rotation and the weights in one: y_lo = r (x_lo ll - x_hi lh), y_hi = r (x_hi hh + x_lo hl)
  float ll[8], lh[8], hh[8], hl[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    ll[i] = t.c[i] * t.wlo[i], hh[i] = t.c[i] * t.whi[i];
    lh[i] = t.turns ? t.s[i] * t.whi[i] : 0.f, hl[i] = t.turns ? t.s[i] * t.wlo[i] : 0.f;
  }
  x += t.h_lo * side.sx.h;
  y += t.h_lo * side.sy.h;
  for (int left = t.h_hi - t.h_lo; left > 0; left -= kAhead) {
    uint4 ua[kAhead], ub[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      ua[u] = ub[u] = make_uint4(0, 0, 0, 0);
      if (here && u < left) {
        ua[u] = load16(x + t.off_a);
        ub[u] = load16(x + t.off_b);
      }
      x += side.sx.h;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (u >= left) break;   // the same for the whole CTA
      float va[8], vb[8], lo[8], hi[8], ylo[8], yhi[8];
      unpack8<T>(va, ua[u]);
      unpack8<T>(vb, ub[u]);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(va[i], va[i], fmaf(vb[i], vb[i], ss));
      const float r = rsqrtf(fmaf(group_sum<LPR>(ss), inv_d, a.eps));
      to_pairs<IL>(lo, hi, va, vb);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // (elements that only pass have no partner: 0 times an infinity would be NaN)
        ylo[i] = (lo[i] * ll[i] - (t.turns ? hi[i] : 0.f) * lh[i]) * r;
        yhi[i] = (hi[i] * hh[i] + (t.turns ? lo[i] : 0.f) * hl[i]) * r;
      }
      from_pairs<IL>(va, vb, ylo, yhi);
      if (here) {
        *reinterpret_cast<uint4 *>(y + t.off_a) = pack8<T>(va);
        *reinterpret_cast<uint4 *>(y + t.off_b) = pack8<T>(vb);
      }
      y += side.sy.h;
    }
  }
}

// Backward.  `ctas` CTAs take equal shares of the work items (a strip of positions, some heads of q or of k), those of q
// first, and leave a row of dw's sums for q and one for k each: partial[0 .. ctas) and [ctas .. 2 ctas) of D floats.  Shares
// and sums depend on the shape and the number of SMs alone: dw is the same bits every time.
// x and g of a head go through a ring of asynchronous copies, kRing heads deep and across items, in which every thread
// reads back what it asked for itself: no barrier, and loads in flight all the time, which registers had no room for.
// B=2, H=32+8, L=4096, D=128 in bf16, forward and backward: 107 us with two heads' loads in registers and a row of sums
// for each of 5120 CTAs (7 of them to add those up), 81 so (5200 GB/s); 4 CTAs an SM: a fifth spills, 96.
template <typename T, int LPR, bool IL>
__global__ void __launch_bounds__(kNormThreads, kBackwardCtas) qk_norm_rotary_bwd_kernel(const NormArgs a, float *partial) {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");   // the sum of the partial rows waits for all of this grid
  constexpr int kRows = kNormThreads / LPR, kWarps = kNormThreads / 32;
  __shared__ __align__(16) uint8_t ring[kRing * 4 * kNormThreads * 16];
  float(*sums)[16 * LPR] = reinterpret_cast<float(*)[16 * LPR]>(ring);   // at the end of a side
  static_assert(kWarps * 16 * LPR * 4 <= (int)sizeof(ring), "the sums go over the ring");
  const uint32_t slot = smem_u32(ring) + threadIdx.x * 16;
  const float inv_d = 1.f / a.D;
  const int group = threadIdx.x / LPR;

  for (int e = 0; e < 2; ++e) {
    const NormSide &side = a.side[e];
    // this CTA's share [lo, hi) of the side's items; item = (strip * B + b) * chunks + chunk
    const int64_t all_q = a.items[0], all = all_q + a.items[1];
    const int64_t from = all * blockIdx.x / gridDim.x, to = all * (blockIdx.x + 1) / gridDim.x;
    const int64_t lo = e ? max(from, all_q) - all_q : min(from, all_q), hi = e ? max(to, all_q) - all_q : min(to, all_q);
    NormLane<T, LPR, IL> t;
    t.columns(a);
    float dlo[8], dhi[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) dlo[i] = dhi[i] = 0.f;
    if (lo < hi) {
      t.e = e;
      t.weights(a);
      // where the copies are: an item and a head in it
      int64_t item = lo;
      int head = 0, left = 0, row = 0, batch = 0;
      const T *x = nullptr, *g = nullptr;
      auto open = [&]() {   // of `item`
        const int chunk = (int)(item % a.chunks[e]);
        const int64_t rest = item / a.chunks[e];
        batch = (int)(rest % a.B), row = (int)(rest / a.B) * kRows + group;
        head = chunk * a.per_cta[e], left = min(side.heads - head, a.per_cta[e]);
        const int64_t l = row < a.L ? row : 0;
        x = static_cast<const T *>(side.x) + batch * side.sx.b + l * side.sx.l + head * side.sx.h;
        g = static_cast<const T *>(side.g) + batch * side.sg.b + l * side.sg.l + head * side.sg.h;
      };
      int stage = 0;
      auto fetch = [&]() {   // the next head, or nothing behind the last item
        if (item < hi) {
          const bool here = t.live && row < a.L;
          const uint32_t at = slot + stage * (4 * kNormThreads * 16);
          const T *sx = here ? x : static_cast<const T *>(side.x), *sg = here ? g : static_cast<const T *>(side.g);
          cp_async16(at, sx + (here ? t.off_a : 0), here);
          cp_async16(at + kNormThreads * 16, sx + (here ? t.off_b : 0), here);
          cp_async16(at + 2 * kNormThreads * 16, sg + (here ? t.off_a : 0), here);
          cp_async16(at + 3 * kNormThreads * 16, sg + (here ? t.off_b : 0), here);
          x += side.sx.h, g += side.sg.h;
          if (--left == 0 && ++item < hi) open();
        }
        cp_async_commit();
        stage = stage + 1 == kRing ? 0 : stage + 1;
      };
      open();
      // where the arithmetic is
      int64_t item_c = lo;
      int stage_c = 0;
#pragma unroll 1
      for (int i = 0; i < kRing - 1; ++i) fetch();
#pragma unroll 1
      for (; item_c < hi; ++item_c) {
        const int chunk = (int)(item_c % a.chunks[e]);
        const int64_t rest = item_c / a.chunks[e];
        t.b = (int)(rest % a.B);
        t.turn_to(a, (int)(rest / a.B) * kRows + group);
        const int h0 = chunk * a.per_cta[e], count = min(side.heads - h0, a.per_cta[e]);
        // (places behind the last position are rows of zeros, which would have no r with eps = 0)
        const float eps = t.l < a.L ? a.eps : 1.f;
        const bool here = t.live && t.l < a.L;
        T *y = static_cast<T *>(side.y) + t.b * side.sy.b + (here ? t.l * side.sy.l : 0) + h0 * side.sy.h;
#pragma unroll 1
        for (int h = 0; h < count; ++h) {
          fetch();
          cp_async_wait<kRing - 1>();
          const uint32_t at = slot + stage_c * (4 * kNormThreads * 16);
          stage_c = stage_c + 1 == kRing ? 0 : stage_c + 1;
          float va[8], vb[8], xlo[8], xhi[8], glo[8], ghi[8];
          unpack8<T>(va, lds16(at));
          unpack8<T>(vb, lds16(at + kNormThreads * 16));
          to_pairs<IL>(xlo, xhi, va, vb);
          unpack8<T>(va, lds16(at + 2 * kNormThreads * 16));
          unpack8<T>(vb, lds16(at + 3 * kNormThreads * 16));
          to_pairs<IL>(glo, ghi, va, vb);
          float ss = 0.f, ax = 0.f;
          float tlo[8], thi[8];   // h x
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            ss = fmaf(xlo[i], xlo[i], fmaf(xhi[i], xhi[i], ss));
            // (elements that only pass have no partner: 0 times an infinity would be NaN)
            const float hl = t.turns ? glo[i] * t.c[i] + ghi[i] * t.s[i] : glo[i];
            const float hh = t.turns ? ghi[i] * t.c[i] - glo[i] * t.s[i] : ghi[i];
            tlo[i] = hl * xlo[i], thi[i] = hh * xhi[i];
            ax = fmaf(tlo[i], t.wlo[i], fmaf(thi[i], t.whi[i], ax));
            glo[i] = hl * t.wlo[i], ghi[i] = hh * t.whi[i];
          }
          const float r = rsqrtf(fmaf(group_sum<LPR>(ss), inv_d, eps));
          const float k = group_sum<LPR>(ax) * inv_d * r * r * r;   // dx = r a - k x (in this order: r^3 may be below fp32's range)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            dlo[i] = fmaf(tlo[i], r, dlo[i]);
            dhi[i] = fmaf(thi[i], r, dhi[i]);
            glo[i] = fmaf(r, glo[i], -k * xlo[i]);
            ghi[i] = fmaf(r, ghi[i], -k * xhi[i]);
          }
          from_pairs<IL>(va, vb, glo, ghi);
          if (here) {
            *reinterpret_cast<uint4 *>(y + t.off_a) = pack8<T>(va);
            *reinterpret_cast<uint4 *>(y + t.off_b) = pack8<T>(vb);
          }
          y += side.sy.h;
        }
      }
      cp_async_wait<0>();
    }
    if (!partial) continue;
    // groups of a warp, then warps, then one row
    float va[8], vb[8];
    from_pairs<IL>(va, vb, dlo, dhi);
#pragma unroll
    for (int m = LPR; m < 32; m *= 2)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        va[i] += __shfl_xor_sync(0xffffffffu, va[i], m);
        vb[i] += __shfl_xor_sync(0xffffffffu, vb[i], m);
      }
    __syncthreads();   // every thread is through with the ring
    if ((threadIdx.x & 31) < LPR && t.live) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sums[threadIdx.x / 32][t.off_a + i] = va[i];
        sums[threadIdx.x / 32][t.off_b + i] = vb[i];
      }
    }
    __syncthreads();
    float *out = partial + ((int64_t)e * gridDim.x + blockIdx.x) * a.D;
    for (int d = threadIdx.x; d < a.D; d += kNormThreads) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v += sums[w][d];
      out[d] = v;
    }
    __syncthreads();   // before the next side's copies
  }
}

// dw from the partial rows: a CTA has 8 columns of one side, 128 threads a column, and adds them in a fixed order.
struct WeightGrad {
  void *out[2];
  int rows;
};
template <typename T>
__global__ void __launch_bounds__(1024) weight_grad_kernel(const float *partial, WeightGrad w, int D, int f32) {
  __shared__ float sums[128][9];
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const int e = blockIdx.y, col = blockIdx.x * 8 + threadIdx.x % 8, lane = threadIdx.x / 8;
  const float *p = partial + (int64_t)e * w.rows * D + col;
  float v = 0.f;
#pragma unroll 8
  for (int i = lane; i < w.rows; i += 128) v += p[(int64_t)i * D];
  sums[lane][threadIdx.x % 8] = v;
  __syncthreads();
  for (int n = 64; n >= 1; n /= 2) {
    if (lane < n) sums[lane][threadIdx.x % 8] += sums[lane + n][threadIdx.x % 8];
    __syncthreads();
  }
  if (lane == 0 && w.out[e]) {
    if (f32) static_cast<float *>(w.out[e])[col] = sums[0][threadIdx.x];
    else static_cast<T *>(w.out[e])[col] = T(sums[0][threadIdx.x]);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
namespace {

int lanes_per_row(int D) {
  int n = 1;
  while (n < D / 16) n *= 2;
  return n;
}

int check_norm(const fa_norm_rotary_args *a) {
  if (!a || (a->dtype != FA_F16 && a->dtype != FA_BF16)) return FA_ERR_BAD_ARG;
  if (a->B < 0 || a->L < 0 || a->H <= 0 || a->Hk <= 0 || a->D <= 0 || a->table_rows <= 0 || a->rotary_dim < 0)
    return FA_ERR_BAD_ARG;
  if (!a->cos || !a->sin) return FA_ERR_BAD_ARG;
  if (a->D % 16 || a->D > 512 || a->rotary_dim % 16 || a->rotary_dim > a->D) return FA_ERR_UNSUPPORTED;
  if (!aligned16(a->cos) || !aligned16(a->sin) || !aligned16(a->q_weight) || !aligned16(a->k_weight))
    return FA_ERR_ALIGNMENT;
  return FA_OK;
}

int sms() {
  const int n = sm_count_of_device();
  return n ? n : 148;   // (sizes asked for without a GPU)
}

// Heads that a thread walks with a position's angles and the weights in its registers: as many as leave the grid `waves` of
// `resident` CTAs an SM deep, `most` at most.  Forward, B=2 H=48+8 L=16384 D=128: 163 us with up to 16 heads, 170 with up
// to 8; B=3 H=20+4 L=1999 D=64: 12 us by this rule, 15 with grids 8 waves deep, whose threads load angles and weights for
// each head.  Returns the number of (strip of positions, chunk of heads).
int64_t plan_norm(const fa_norm_rotary_args *s, NormArgs *a, int resident, int waves, int most) {
  const int rows = kNormThreads / lanes_per_row(s->D);
  const int64_t positions = (int64_t)((s->L + rows - 1) / rows) * s->B, want = (int64_t)sms() * resident * waves;
  const int all = s->H + s->Hk;
  int per = 1;
  while (per < most && positions * ((all + 2 * per - 1) / (2 * per)) >= want) per *= 2;
  for (int e = 0; e < 2; ++e) {
    const int heads = e ? s->Hk : s->H;
    a->per_cta[e] = std::min(per, heads);
    a->chunks[e] = (heads + a->per_cta[e] - 1) / a->per_cta[e];
    a->items[e] = positions * a->chunks[e];
  }
  return a->items[0] + a->items[1];
}
// CTAs of the backward: all that are resident at once, each with a share of the items
int64_t backward_ctas(int64_t items) { return std::min(items, (int64_t)sms() * kBackwardCtas); }

void fill_norm(const fa_norm_rotary_args *s, NormArgs *a) {
  a->cos = s->cos, a->sin = s->sin, a->positions = s->positions, a->pos_stride_b = s->pos_stride_b, a->eps = s->eps;
  a->B = s->B, a->L = s->L, a->D = s->D, a->R = s->rotary_dim, a->table_rows = s->table_rows;
  a->weight_is_f32 = s->weight_is_f32;
  a->side[0].weight = s->q_weight, a->side[1].weight = s->k_weight;
  a->side[0].heads = s->H, a->side[1].heads = s->Hk;
}

template <typename T, int LPR, bool IL>
int launch_norm(const NormArgs &a, int64_t grid, bool backward, float *partial, cudaStream_t s) {
  if (backward) qk_norm_rotary_bwd_kernel<T, LPR, IL><<<(unsigned)grid, kNormThreads, 0, s>>>(a, partial);
  else qk_norm_rotary_fwd_kernel<T, LPR, IL><<<(unsigned)grid, kNormThreads, 0, s>>>(a);
  FA_CHECK_LAUNCH();
  return FA_OK;
}
template <typename T, bool IL>
int dispatch_lanes(int D, const NormArgs &a, int64_t grid, bool backward, float *partial, cudaStream_t s) {
  switch (lanes_per_row(D)) {
    case 1: return launch_norm<T, 1, IL>(a, grid, backward, partial, s);
    case 2: return launch_norm<T, 2, IL>(a, grid, backward, partial, s);
    case 4: return launch_norm<T, 4, IL>(a, grid, backward, partial, s);
    case 8: return launch_norm<T, 8, IL>(a, grid, backward, partial, s);
    case 16: return launch_norm<T, 16, IL>(a, grid, backward, partial, s);
    default: return launch_norm<T, 32, IL>(a, grid, backward, partial, s);
  }
}
int dispatch_norm(const fa_norm_rotary_args *p, const NormArgs &a, int64_t grid, bool backward, float *partial,
                  cudaStream_t s) {
  if (grid >= (1ll << 31)) return FA_ERR_TOO_LARGE;
  if (p->dtype == FA_F16)
    return p->interleaved ? dispatch_lanes<__half, true>(p->D, a, grid, backward, partial, s)
                          : dispatch_lanes<__half, false>(p->D, a, grid, backward, partial, s);
  return p->interleaved ? dispatch_lanes<__nv_bfloat16, true>(p->D, a, grid, backward, partial, s)
                        : dispatch_lanes<__nv_bfloat16, false>(p->D, a, grid, backward, partial, s);
}

}  // namespace
}  // namespace fa

using namespace fa;

extern "C" int fa_qk_norm_rotary_fwd(const fa_norm_rotary_args *p, const fa_tensor4 *q, const fa_tensor4 *k,
                                     const fa_tensor4 *q_out, const fa_tensor4 *k_out, void *stream) {
  if (int st = check_norm(p)) return st;
  if (p->B == 0 || p->L == 0) return FA_OK;
  for (const fa_tensor4 *t : {q, k, q_out, k_out}) {
    if (!tensor_ok(t)) return FA_ERR_BAD_ARG;
    if (!tensor_aligned(t)) return FA_ERR_ALIGNMENT;
  }
  NormArgs a{};
  fill_norm(p, &a);
  a.side[0].x = q->ptr, a.side[0].sx = strides_of(q), a.side[0].y = q_out->ptr, a.side[0].sy = strides_of(q_out);
  a.side[1].x = k->ptr, a.side[1].sx = strides_of(k), a.side[1].y = k_out->ptr, a.side[1].sy = strides_of(k_out);
  return dispatch_norm(p, a, plan_norm(p, &a, kForwardCtas, 1, 16), false, nullptr, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t fa_qk_norm_rotary_bwd_workspace_bytes(const fa_norm_rotary_args *p) {
  if (check_norm(p) || p->B == 0 || p->L == 0) return 0;
  NormArgs a{};
  return 2 * backward_ctas(plan_norm(p, &a, kBackwardCtas, 4, 8)) * p->D * 4;
}

extern "C" int fa_qk_norm_rotary_bwd(const fa_norm_rotary_args *p, const fa_tensor4 *q, const fa_tensor4 *k,
                                     const fa_tensor4 *gq, const fa_tensor4 *gk, const fa_tensor4 *dq,
                                     const fa_tensor4 *dk, void *dq_weight, void *dk_weight, void *workspace,
                                     int64_t workspace_bytes, void *stream) {
  if (int st = check_norm(p)) return st;
  auto s = static_cast<cudaStream_t>(stream);
  const bool weights = dq_weight || dk_weight;
  if (p->B == 0 || p->L == 0) {
    const size_t bytes = (size_t)p->D * (p->weight_is_f32 ? 4 : 2);
    for (void *w : {dq_weight, dk_weight})
      if (w && cudaMemsetAsync(w, 0, bytes, s) != cudaSuccess) return FA_ERR_LAUNCH;
    return FA_OK;
  }
  for (const fa_tensor4 *t : {q, k, gq, gk, dq, dk}) {
    if (!tensor_ok(t)) return FA_ERR_BAD_ARG;
    if (!tensor_aligned(t)) return FA_ERR_ALIGNMENT;
  }
  NormArgs a{};
  fill_norm(p, &a);
  const fa_tensor4 *xs[2] = {q, k}, *gs[2] = {gq, gk}, *ds[2] = {dq, dk};
  for (int e = 0; e < 2; ++e) {
    a.side[e].x = xs[e]->ptr, a.side[e].sx = strides_of(xs[e]);
    a.side[e].g = gs[e]->ptr, a.side[e].sg = strides_of(gs[e]);
    a.side[e].y = ds[e]->ptr, a.side[e].sy = strides_of(ds[e]);
  }
  const int64_t grid = backward_ctas(plan_norm(p, &a, kBackwardCtas, 4, 8));
  if (weights && (!workspace || !aligned16(workspace) || workspace_bytes < 2 * grid * p->D * 4)) return FA_ERR_WORKSPACE;
  float *partial = weights ? static_cast<float *>(workspace) : nullptr;
  if (int st = dispatch_norm(p, a, grid, true, partial, s)) return st;
  if (!weights) return FA_OK;
  const WeightGrad w{{dq_weight, dk_weight}, (int)grid};
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p->D / 8, 2), cfg.blockDim = dim3(1024), cfg.stream = s, cfg.attrs = &attr, cfg.numAttrs = 1;
  const cudaError_t st =
      p->dtype == FA_F16
          ? cudaLaunchKernelEx(&cfg, weight_grad_kernel<__half>, (const float *)partial, w, (int)p->D, (int)p->weight_is_f32)
          : cudaLaunchKernelEx(&cfg, weight_grad_kernel<__nv_bfloat16>, (const float *)partial, w, (int)p->D,
                               (int)p->weight_is_f32);
  if (st != cudaSuccess) return FA_ERR_LAUNCH;
  FA_CHECK_LAUNCH();
  return FA_OK;
}
