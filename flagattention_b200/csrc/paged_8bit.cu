// paged_attention_8bit decode: paged.cu's gather over a cache of e4m3 codes with an fp32 scale for each block and kv head.
//
// Bytes are half of that and products are not, so instructions count: every warp streams groups of codes through a
// cp.async ring of its own, and codes, turned to fp16 exactly on their way from shared memory, are the left operands of both
// products, S^T = K Q^T and O^T = V^T P^T.  Queries are the 8 columns of a fragment, so that a group of 8 heads or fewer
// wastes nothing (as 16 rows of the left operand they fill half of it and need twice the accumulators: 12 warps an SM
// instead of 16, 64 sequences of 1K-32K tokens 381 us instead of 355).
//  * S^T contracts over the head, in whatever order both operands agree on: a lane takes 16 codes that lie side by side as
//    four steps of its K fragment, so K needs neither ldmatrix nor a transposition, and Q's fragments are read in that
//    order.
//  * O^T contracts over tokens, whose codes lie apart: a lane reads the same 16 head elements of four tokens and
//    interleaves them two by two (one byte permutation for two conversions).  Rows of the accumulator are head elements in
//    that order, so a lane ends with consecutive ones.  P^T comes from S^T by transposing 8 x 8 tiles in registers.
// Which 8 tokens a fragment's rows mean (token_of) and where a row's 16-byte pieces lie (code_offset) are chosen so that
// both reads hit every bank once.
//
// The scale of K goes into the score.  The scale of V cannot go into the accumulator, which many blocks share, nor into
// P alone, whose 16 bits would not hold its range: a token's weight in O is exp2(score) 2^E f for a scale 2^E f, 1 <= f < 2,
// and O has a running reference of its own over score + E, beside the maximum that the sum of the softmax goes by.  So
// weights stay in range whatever the scales are.
// bf16 queries are brought to fp16 by a power of two for each row, its maximum to [2^14, 2^15): an element keeps
// its bits or loses 2^-39 of the maximum at most (half of fp16's least step).
#include <cfloat>
#include <climits>

#include "common.cuh"
#include "paged_parts.cuh"

namespace fa {
// Weights of O run up to 2^(kLift + 8 + 1) and so stay in fp16; the lift keeps 2^kLift more of the small ones above its
// least number.
constexpr float kLift = 6.f;
constexpr float kNone = -FLT_MAX;   // a reference of no scores: -inf - kNone and kNone - kNone are numbers or -inf

template <int D, int NQ>
struct Paged8Cfg {
  static constexpr int kD = D < 64 ? 64 : D;   // shorter heads are padded with zeros in shared memory
  static constexpr int kWarps = 4, kRows = 8 * NQ;
  // Warps as the registers allow (two columns at head 64 and below spill 20 to 32 bytes), groups as short as the bookkeeping between
  // them allows.  us for 64
  // sequences, tokens of a group x CTAs: head 128, 8 kv heads of 4, 1K-32K tokens 16 x 4 355, 32 x 3 355 (one sequence of
  // 131071: 51, 52), 32 x 2 362, 2 kv heads of 16, 1K-16K 16 x 4 94, 16 x 3 with queries in registers 102, 32 x 3 106; head
  // 64, 8 kv heads of 4, 1K-16K 32 x 4 115, 16 x 4 124, 16 x 5 118, 64 x 3 121; head 256, 32 sequences of 4 kv heads 16 x 2
  // 113, x 3 with a stage less 121.
  static constexpr int kStages = D <= 64 ? 2 : 3;
  static constexpr int kTokens = D <= 64 ? 32 : 16;     // tokens of a group
  static constexpr int kCtas = D <= 128 ? 4 : 2;        // on an SM
  static constexpr int kGroupBytes = kTokens * kD;            // of K or of V
  static constexpr int kStageBytes = 2 * kGroupBytes;
  static constexpr int kWarpBytes = kStages * kStageBytes;
  static constexpr int kQBytes = kRows * kD * 2;
  static constexpr int kScales = kQBytes;                     // per warp: of 64 pieces, K and V
  static constexpr int kRowScale = kScales + kWarps * 64 * 8;
  static constexpr int kStats = kRowScale + kRows * 4;           // per warp and row: maximum, sum, reference of O
  static constexpr int kRing = (kStats + 3 * kWarps * kRows * 4 + 127) / 128 * 128;
  static constexpr int kRingBytes = kWarps * kWarpBytes;
  static constexpr int kMergeBytes = kWarps * kRows * kD * 4;    // fp32 partial outputs, over the ring
  static constexpr int kTotal = kRing + (kRingBytes > kMergeBytes ? kRingBytes : kMergeBytes);
};

// the token, of 8, that row n of a score fragment stands for
template <int KD>
__device__ __forceinline__ constexpr int token_of(int n) {
  const int n0 = n & 1, n1 = n >> 1 & 1, n2 = n >> 2;
  return KD == 64 ? n2 << 2 | n1 << 1 | (n0 ^ n2) : (n0 ^ n2) << 2 | n1 << 1 | n0;
}
// byte offset of 16-byte piece `piece` of row `row` in a group
template <int KD>
__device__ __forceinline__ constexpr uint32_t code_offset(int row, int piece) {
  return (uint32_t)(row * KD + 16 * (KD == 64 ? piece ^ (row & 2) : piece ^ (row & 7)));
}

// two e4m3 codes of a word, as two fp16 numbers
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) {
  uint32_t h;
  asm("{.reg .b16 lo, hi; mov.b32 {lo, hi}, %1; cvt.rn.f16x2.e4m3x2 %0, lo;}\n" : "=r"(h) : "r"(w));
  return h;
}
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) {
  uint32_t h;
  asm("{.reg .b16 lo, hi; mov.b32 {lo, hi}, %1; cvt.rn.f16x2.e4m3x2 %0, hi;}\n" : "=r"(h) : "r"(w));
  return h;
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(dst), "l"(src));
}
// scale = 2^exponent x fraction, 1 <= fraction < 2; below the normal numbers, 0 among them, exponent -126 and a fraction below
// 1, whose weights keep fewer bits (off by 2^-31 of 2^-126 at most); an infinity or NaN is its own fraction
__device__ __forceinline__ void split_scale(float scale, float &exponent, float &fraction) {
  const uint32_t bits = __float_as_uint(scale), e = bits >> 23 & 255u;
  exponent = e == 255u ? 0.f : (float)(max((int)e, 1) - 127);
  fraction = e == 255u ? scale : e ? __uint_as_float((bits & 0x7fffffu) | 0x3f800000u) : scale * 0x1p126f;
}

// an 8 x 8 matrix of 16-bit numbers, two of row lane / 4 a lane, into its transpose in the same layout
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float over_tokens_max(float v) {
#pragma unroll
  for (int m = 4; m < 32; m *= 2) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, m));
  return v;
}
__device__ __forceinline__ float over_tokens_sum(float v) {
#pragma unroll
  for (int m = 4; m < 32; m *= 2) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

// NQ: columns of 8 query rows
template <typename T, int D, typename IdxT, int NQ>
__global__ void __launch_bounds__(Paged8Cfg<D, NQ>::kWarps * 32, Paged8Cfg<D, NQ>::kCtas)
    paged_8bit_kernel(const __grid_constant__ fa_paged_8bit_args p, const Sizing z) {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");   // the reduction waits for all of this grid by itself
  using C = Paged8Cfg<D, NQ>;
  constexpr int KD = C::kD, NW = C::kWarps, NS = C::kStages, GT = C::kTokens;
  constexpr int R = 2 * NQ;         // query rows of a thread: 2 t4, 2 t4 + 1 of each column
  constexpr int KJ = KD / 64;       // 16-byte pieces of a row that a lane of a quad takes for S
  constexpr int VW = KD / 32;       // 4-byte words of a row that a lane takes for O
  constexpr int NH = GT / 16;       // 16-token pieces of a group
  extern __shared__ __align__(128) uint8_t smem_raw[];
  const uint32_t smem = smem_u32(smem_raw);
  const fa_paged_args &a = p.paged;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  // the heads of a sequence side by side: their pieces of a block are neighbours in memory
  const int G = a.num_q_heads / a.num_kv_heads;
  const int q_tiles = (G + 15) / 16, heads = a.num_kv_heads * q_tiles;
  const int seq = blockIdx.x / heads, head = blockIdx.x % heads;
  const int hk = head / q_tiles, qt = head % q_tiles;
  const int part = blockIdx.y;
  const int rows = min(16, G - qt * 16);          // valid query rows of this CTA
  const int qh0 = hk * G + qt * 16;               // first query head

  const int ctx = context_len(a, seq);
  int t_begin = 0, t_end = ctx;
  if (a.partition_size > 0) {
    const LaneLens lens = lane_lens(a, z);   // in flight together with ctx
    if ((long long)part * (z.finest ? z.finest : a.partition_size) >= ctx) return;
    const int size = partition_tokens(a, z, lens, ctx, gridDim.y);
    if ((long long)part * size >= ctx) return;
    t_begin = part * size;
    t_end = (int)min((long long)ctx, (long long)t_begin + size);
  }
  const int BS = a.block_size;
  t_end = (int)min((long long)t_end, (long long)p.table_cols * BS);   // (a table narrower than the length)

  // ---- this warp's token groups ---------------------------------------------
  const int n_groups = t_end > t_begin ? (t_end - t_begin + GT - 1) / GT : 0;
  const int my_groups = n_groups > warp ? (n_groups - warp + NW - 1) / NW : 0;
  const uint32_t ring = smem + C::kRing + warp * C::kWarpBytes;
  const uint32_t scales = smem + C::kScales + warp * 64 * 8;
  const uint8_t *kc = static_cast<const uint8_t *>(a.key_cache) + (int64_t)hk * a.kv_stride_h;
  const uint8_t *vc = static_cast<const uint8_t *>(a.value_cache) + (int64_t)hk * a.kv_stride_h;
  const int64_t v_minus_k = vc - kc;
  const int bs_shift = (BS & (BS - 1)) == 0 ? 31 - __clz(BS) : -1;

  // A lane copies 16-byte piece `ch` of rows c * RPC + lane_r of a group, of K and of V.
  constexpr int CPR = D / 16, RPC = 32 / CPR, NC = (GT + RPC - 1) / RPC;
  const int lane_r = lane / CPR, ch = lane % CPR;
  uint32_t dst_off[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) dst_off[c] = code_offset<KD>(c * RPC + lane_r, ch);
  const int64_t lane_src = (int64_t)lane_r * a.kv_stride_t + ch * 16;

  // Where the warp's 16-token pieces lie is worked out for 32 of them at a time, one a lane, and handed on by shuffles: the
  // table, its bounds and the 64-bit products would otherwise be a sixth of a group's instructions (422 us for 381).
  const auto piece_tok = [&](int q) { return t_begin + (warp + q / NH * NW) * GT + 16 * (q % NH); };
  int64_t id_ahead = 0;   // of the 32 pieces behind those of `place`
  int64_t place = -1;  // byte offset of this lane's piece; -1: without a token, -2: its id is outside the cache
  const auto look_up = [&](int q0) {
    const int q = q0 + lane, tok = piece_tok(q);
    if (q < my_groups * NH && tok < t_end)
      id_ahead = phys_block<IdxT>(a.block_tables, a.bt_stride_s, seq, bs_shift >= 0 ? tok >> bs_shift : tok / BS);
  };
  const auto settle = [&](int q0) {   // the next 32 pieces: their places, their scales into shared memory
    const int q = q0 + lane, tok = piece_tok(q);
    const bool here = q < my_groups * NH && tok < t_end, ok = here && id_ahead >= 0 && id_ahead < p.num_blocks;
    const int in_blk = bs_shift >= 0 ? tok & (BS - 1) : tok % BS;
    place = ok ? id_ahead * a.kv_stride_b + (int64_t)in_blk * a.kv_stride_t : here ? -2 : -1;
    const uint32_t at = scales + (q & 63) * 8;
    if (ok) {
      const int64_t from = id_ahead * a.num_kv_heads + hk;
      cp_async4(at, p.key_scales + from);
      cp_async4(at + 4, p.value_scales + from);
    } else {   // a block outside the cache makes its sequence's output NaN; a piece without tokens counts as nothing
      const float none = here ? NAN : 0.f;
      asm volatile("st.shared.v2.f32 [%0], {%1, %1};\n" ::"r"(at), "f"(none) : "memory");
    }
    look_up(q0 + 32);
  };
  const uint8_t *k_lane = kc + lane_src;
  const int64_t c_step = (int64_t)RPC * a.kv_stride_t;
  const bool packed = a.kv_stride_t == D;   // steps that are known when this is compiled
  const auto issue = [&](int i) {   // i-th group of this warp -> stage i % NS
    if (i * NH % 32 == 0) settle(i * NH);
    const int tok0 = t_begin + (warp + i * NW) * GT;
    const uint32_t st = ring + (i % NS) * C::kStageBytes;
    int64_t at[NH];
    bool whole = tok0 + GT <= t_end;
#pragma unroll
    for (int s = 0; s < NH; ++s) {
      at[s] = __shfl_sync(0xffffffffu, place, (i * NH + s) % 32);
      whole = whole && at[s] >= 0;
    }
    if (RPC <= 16 && whole && packed) {
#pragma unroll
      for (int s = 0; s < NH; ++s) {
        const uint8_t *sk = k_lane + at[s], *sv = sk + v_minus_k;
#pragma unroll
        for (int c = s * (NC / NH); c < (s + 1) * (NC / NH); ++c) {
          cp_async16(st + dst_off[c], sk + c * RPC % 16 * D, true);
          cp_async16(st + C::kGroupBytes + dst_off[c], sv + c * RPC % 16 * D, true);
        }
      }
    } else if (RPC <= 16 && whole) {
#pragma unroll
      for (int s = 0; s < NH; ++s) {
        const uint8_t *sk = k_lane + at[s];
#pragma unroll
        for (int c = s * (NC / NH); c < (s + 1) * (NC / NH); ++c) {
          cp_async16(st + dst_off[c], sk, true);
          cp_async16(st + C::kGroupBytes + dst_off[c], sk + v_minus_k, true);
          sk += c_step;
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int row = c * RPC + lane_r, s = row / 16;   // (a row of 16 bytes: a step covers both pieces)
        const uint8_t *sk = kc;
        bool ok = tok0 + row < t_end;
#pragma unroll
        for (int k = 0; k < NH; ++k)
          if (s == k) {
            ok = ok && at[k] >= 0;
            sk = k_lane + at[k] + (int64_t)(RPC <= 16 ? c * RPC % 16 : -16 * k) * a.kv_stride_t;
          }
        if (s >= NH) ok = false;
        if (!ok) sk = kc;
        if (row < GT) {
          cp_async16(st + dst_off[c], sk, ok);
          cp_async16(st + C::kGroupBytes + dst_off[c], sk + v_minus_k, ok);
        }
      }
    }
  };

  look_up(0);
  if (D < KD) {   // the padding of shorter heads
    for (int i = tid; i < C::kRingBytes / 16; i += NW * 32)
      reinterpret_cast<uint4 *>(smem_raw + C::kRing)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) {
    if (i < my_groups) issue(i);
    cp_async_commit();
  }

  // ---- query group -> shared as fp16 (rows >= `rows` are zero) -----------------
  float *row_scale = reinterpret_cast<float *>(smem_raw + C::kRowScale);
  // threads of a row, and their 8-element pieces; whole warps
  constexpr int TPR = NW * 32 / C::kRows < KD / 8 ? NW * 32 / C::kRows : KD / 8, PIECES = KD / 8 / TPR;
  if (tid < C::kRows * TPR) {
    const int r = tid / TPR, t = tid % TPR;
    const T *q = static_cast<const T *>(a.query) + (int64_t)seq * a.q_stride_s + (int64_t)(qh0 + r) * a.q_stride_h;
    uint4 u[PIECES];
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int piece = t + i * TPR;
      u[i] = make_uint4(0, 0, 0, 0);
      if (r < rows && piece * 8 < D) u[i] = *reinterpret_cast<const uint4 *>(q + piece * 8);
      if (!std::is_same<T, __half>::value) {
        const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = Elem<T>::unpack(w[k]);
          most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
    }
    float up = 1.f, down = 1.f;
    if (!std::is_same<T, __half>::value) {
#pragma unroll
      for (int m = 1; m < TPR; m *= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, m));
      if (most > 0.f && most < INFINITY) {
        // 2^(14 - exponent of the maximum), inside the normal numbers, and its inverse
        const int e = min(max(14 - ((int)(__float_as_uint(most) >> 23) - 127), -126), 126);
        up = __uint_as_float((uint32_t)(127 + e) << 23), down = __uint_as_float((uint32_t)(127 - e) << 23);
      }
    }
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      if (!std::is_same<T, __half>::value) {
        uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = Elem<T>::unpack(w[k]);
          w[k] = Elem<__half>::pack(f.x * up, f.y * up);
        }
        u[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
      *reinterpret_cast<uint4 *>(smem_raw + (r * KD + (t + i * TPR) * 8) * 2) = u[i];
    }
    if (t == 0) row_scale[r] = a.attn_scale * kLog2e * down;
  }
  __syncthreads();

  float q_scale[R];
#pragma unroll
  for (int r = 0; r < R; ++r) q_scale[r] = row_scale[8 * (r >> 1) + 2 * t4 + (r & 1)];
  // step (j, w) of the contraction is elements 64 j + 16 t4 + 4 w .. + 3 of a row
  constexpr bool kQInRegs = D * NQ <= 128;   // beyond it they would cost a fourth of the warps
  const auto q_step = [&](int j, int w, int n) {
    return lds8(smem + (uint32_t)((8 * n + g) * KD + 64 * j + 16 * t4 + 4 * w) * 2);
  };
  uint2 qf[kQInRegs ? 4 * KJ : 1][NQ];
  if (kQInRegs) {
#pragma unroll
    for (int i = 0; i < 4 * KJ; ++i)
#pragma unroll
      for (int n = 0; n < NQ; ++n) qf[i][n] = q_step(i / 4, i % 4, n);
  }

  // acc[m][n]: head elements (lane / 4)'s 2 m and 2 m + 1 of query rows 2 t4, 2 t4 + 1 of column n
  constexpr int W = VW < 4 ? VW : 4, JV = (VW + 3) / 4;
  float acc[2 * W * JV][NQ][4];
#pragma unroll
  for (int m = 0; m < 2 * W * JV; ++m)
#pragma unroll
    for (int n = 0; n < NQ; ++n) acc[m][n][0] = acc[m][n][1] = acc[m][n][2] = acc[m][n][3] = 0.f;
  // references: of the sum, close to the maximum of the scores, and of acc, close to that of score + exponent of V's scale
  float m_i[R], w_i[R], l_i[R];
#pragma unroll
  for (int r = 0; r < R; ++r) m_i[r] = w_i[r] = kNone, l_i[r] = 0.f;

#pragma unroll 1
  for (int i = 0; i < my_groups; ++i) {
    if (i + NS - 1 < my_groups) issue(i + NS - 1);
    cp_async_commit();
    cp_async_wait<NS - 1>();
    __syncwarp();

    const int tok0 = t_begin + (warp + i * NW) * GT;
    const uint32_t st = ring + (i % NS) * C::kStageBytes, sv = st + C::kGroupBytes;
    const int my_token = token_of<KD>(g);            // of each eight, as a row of S^T
    const int col[2] = {token_of<KD>(2 * t4), token_of<KD>(2 * t4 + 1)};   // and as a step of O^T

    float s[NH][NQ][4];   // [.][.][2 u + e]: token my_token + 8 u, query row 2 t4 + e
    float ve[NH], vf[NH];
#pragma unroll
    for (int h = 0; h < NH; ++h) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) s[h][n][0] = s[h][n][1] = s[h][n][2] = s[h][n][3] = 0.f;
#pragma unroll
      for (int j = 0; j < KJ; ++j) {
        const uint4 k0 = lds16(st + code_offset<KD>(16 * h + my_token, 4 * j + t4));
        const uint4 k1 = lds16(st + code_offset<KD>(16 * h + 8 + my_token, 4 * j + t4));
        const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t ka[4] = {codes_lo(w0[w]), codes_lo(w1[w]), codes_hi(w0[w]), codes_hi(w1[w])};
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            const uint2 qb = kQInRegs ? qf[4 * j + w][n] : q_step(j, w, n);
            Elem<__half>::mma(s[h][n], ka, qb.x, qb.y);
          }
        }
      }
      const uint2 sc = lds8(scales + (i * NH + h) % 64 * 8);
      split_scale(__uint_as_float(sc.y), ve[h], vf[h]);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float by = q_scale[r] * __uint_as_float(sc.x);
        s[h][r >> 1][r & 1] *= by, s[h][r >> 1][2 + (r & 1)] *= by;
      }
    }
    if (tok0 + GT > t_end) {
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (tok0 + 16 * h + 8 * u + my_token >= t_end)
#pragma unroll
            for (int n = 0; n < NQ; ++n) s[h][n][2 * u] = s[h][n][2 * u + 1] = -INFINITY;
    }
    // lazy, as in paged.cu: references move when one is 2^8 behind, and only then are lanes' maxima put together
    float mx[NH][R];
    bool need = false;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        mx[h][r] = fmaxf(s[h][r >> 1][r & 1], s[h][r >> 1][2 + (r & 1)]);
        need = need || mx[h][r] - m_i[r] > 8.f || mx[h][r] + (ve[h] - w_i[r]) > 8.f;
      }
    if (__any_sync(0xffffffffu, need)) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float m_new = m_i[r], w_new = w_i[r];
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          const float most = over_tokens_max(mx[h][r]);
          m_new = fmaxf(m_new, most), w_new = fmaxf(w_new, most + ve[h]);
        }
        l_i[r] *= fast_exp2(m_i[r] - m_new);
        const float alpha = fast_exp2(w_i[r] - w_new);
        m_i[r] = m_new, w_i[r] = w_new;
#pragma unroll
        for (int m = 0; m < 2 * W * JV; ++m) acc[m][r >> 1][r & 1] *= alpha, acc[m][r >> 1][2 + (r & 1)] *= alpha;
      }
    }
#pragma unroll
    for (int h = 0; h < NH; ++h) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float by = ve[h] - w_i[r] + kLift;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float &x = s[h][r >> 1][2 * u + (r & 1)];
          l_i[r] += fast_exp2(x - m_i[r]);
          x = fast_exp2(x + by) * vf[h];
        }
      }
      // P goes in as a 16-bit value and a 16-bit remainder, as in paged.cu
      uint32_t pv[NQ][2], pr[NQ][2];
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          split_weights<__half>(s[h][n][2 * u], s[h][n][2 * u + 1], pv[n][u], pr[n][u]);
          pv[n][u] = transposed(pv[n][u]), pr[n][u] = transposed(pr[n][u]);
        }
#pragma unroll
      for (int j = 0; j < JV; ++j) {
        uint32_t v[4][W];   // tokens 2 t4, 2 t4 + 1 of the first eight and of the second
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int row = 16 * h + 8 * (k >> 1) + col[k & 1];
          if constexpr (W == 4) {
            const uint4 x = lds16(sv + code_offset<KD>(row, g + 8 * j));
            v[k][0] = x.x, v[k][1] = x.y, v[k][2] = x.z, v[k][3] = x.w;
          } else {
            const uint2 x = lds8(sv + code_offset<KD>(row, g >> 1) + 8 * (g & 1));
            v[k][0] = x.x, v[k][1] = x.y;
          }
        }
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int pick = e ? 0x7362 : 0x5140;
            const uint32_t x = __byte_perm(v[0][w], v[1][w], pick), y = __byte_perm(v[2][w], v[3][w], pick);
            const uint32_t va[4] = {codes_lo(x), codes_hi(x), codes_lo(y), codes_hi(y)};
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
              Elem<__half>::mma(acc[2 * (W * j + w) + e][n], va, pv[n][0], pv[n][1]);
              Elem<__half>::mma(acc[2 * (W * j + w) + e][n], va, pr[n][0], pr[n][1]);
            }
          }
      }
    }
    __syncwarp();  // stage may be refilled by the next iteration's issue
  }
  cp_async_wait<0>();

  // ---- merge the warps' partial states --------------------------------------
  float *stat_m = reinterpret_cast<float *>(smem_raw + C::kStats);
  float *stat_l = stat_m + NW * C::kRows, *stat_w = stat_l + NW * C::kRows;
  float *merge = reinterpret_cast<float *>(smem_raw + C::kRing);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = 8 * (r >> 1) + 2 * t4 + (r & 1);
    const float l = over_tokens_sum(l_i[r]);
    if (g == 0) {
      stat_m[warp * C::kRows + row] = m_i[r] == kNone ? -INFINITY : m_i[r];
      stat_l[warp * C::kRows + row] = l;
      stat_w[warp * C::kRows + row] = w_i[r] == kNone ? -INFINITY : w_i[r];
    }
  }
  __syncthreads();  // stats visible; every warp has drained its ring
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = 8 * (r >> 1) + 2 * t4 + (r & 1), n = r >> 1, e = r & 1;
    if (row >= rows) continue;
    float ww = -INFINITY;
#pragma unroll
    for (int w2 = 0; w2 < NW; ++w2) ww = fmaxf(ww, stat_w[w2 * C::kRows + row]);
    const float scale_w = w_i[r] == kNone ? 0.f : fast_exp2(w_i[r] - ww);
#pragma unroll
    for (int j = 0; j < JV; ++j)
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float(&x)[4] = acc[2 * (W * j + w)][n], (&y)[4] = acc[2 * (W * j + w) + 1][n];
        *reinterpret_cast<float4 *>(merge + (warp * C::kRows + row) * KD + 128 * j + 4 * W * g + 4 * w) =
            make_float4(x[e] * scale_w, x[2 + e] * scale_w, y[e] * scale_w, y[2 + e] * scale_w);
      }
  }
  __syncthreads();

  for (int idx = tid; idx < rows * (D / 4); idx += NW * 32) {
    const int row = idx / (D / 4), c4 = idx % (D / 4);
    float mm = -INFINITY, ww = -INFINITY;
#pragma unroll
    for (int w2 = 0; w2 < NW; ++w2) {
      mm = fmaxf(mm, stat_m[w2 * C::kRows + row]);
      ww = fmaxf(ww, stat_w[w2 * C::kRows + row]);
    }
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w2 = 0; w2 < NW; ++w2) {
      const float mw = stat_m[w2 * C::kRows + row];
      if (mw != -INFINITY) l += stat_l[w2 * C::kRows + row] * fast_exp2(mw - mm);
      else l += stat_l[w2 * C::kRows + row];   // 0, or NaN where every score was
      const float4 v = *reinterpret_cast<const float4 *>(merge + (w2 * C::kRows + row) * KD + c4 * 4);
      o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
    }
    // from the reference of O to that of the sum, in two steps where one would be below the normal numbers; a sequence without
    // tokens has 0, a NaN stays one
    const float by = ww - kLift - mm, rest = by < -100.f ? 0x1p-64f : 1.f;
    const float inv = l == 0.f ? 0.f : (ww == -INFINITY ? 1.f : fast_exp2(by < -100.f ? by + 64.f : by)) / l;
    o.x = o.x * inv * rest, o.y = o.y * inv * rest, o.z = o.z * inv * rest, o.w = o.w * inv * rest;
    const int qh = qh0 + row;
    if (a.partition_size > 0) {
      const int P = partitions_of(a);
      const int64_t pi = ((int64_t)seq * a.num_q_heads + qh) * P + part;
      *reinterpret_cast<float4 *>(a.part_out + pi * D + c4 * 4) = o;
      if (c4 == 0) {
        a.part_max[pi] = mm;
        a.part_sum[pi] = l;
      }
    } else {
      T *dst = reinterpret_cast<T *>(a.out) + (int64_t)seq * a.o_stride_s +
               (int64_t)qh * a.o_stride_h + c4 * 4;
      uint2 pk;
      pk.x = Elem<T>::pack(o.x, o.y);
      pk.y = Elem<T>::pack(o.z, o.w);
      *reinterpret_cast<uint2 *>(dst) = pk;
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
static int validate_8bit(const fa_paged_8bit_args *p) {
  if (!p) return FA_ERR_BAD_ARG;
  const fa_paged_args *a = &p->paged;
  if (!a->query || !a->key_cache || !a->value_cache || !a->out || !a->context_lens || !a->block_tables ||
      !p->key_scales || !p->value_scales)
    return FA_ERR_BAD_ARG;
  if (a->dtype != FA_F16 && a->dtype != FA_BF16) return FA_ERR_BAD_ARG;
  if (a->num_seqs <= 0 || a->num_q_heads <= 0 || a->num_kv_heads <= 0 || a->block_size <= 0 ||
      a->max_context_len <= 0 || a->partition_size < 0 || p->num_blocks < 0 || p->table_cols <= 0)
    return FA_ERR_BAD_ARG;
  if (a->num_q_heads % a->num_kv_heads != 0 || a->block_size % 16 != 0 || a->partition_size % 16 != 0 ||
      a->causal_rows != 0 || (a->block_table_is_i64 != 0 && a->block_table_is_i64 != 1))
    return FA_ERR_BAD_ARG;
  const int D = a->head_size;
  if (!(D == 16 || D == 32 || D == 64 || D == 128 || D == 256)) return FA_ERR_UNSUPPORTED;
  if (!aligned16(a->query) || !aligned16(a->key_cache) || !aligned16(a->value_cache) || !aligned16(a->out))
    return FA_ERR_ALIGNMENT;
  if (a->q_stride_s % 8 || a->q_stride_h % 8 || a->kv_stride_b % 16 || a->kv_stride_h % 16 ||
      a->kv_stride_t % 16 || a->o_stride_s % 4 || a->o_stride_h % 4)
    return FA_ERR_ALIGNMENT;
  if (a->partition_size > 0 && (!a->part_out || !a->part_max || !a->part_sum)) return FA_ERR_WORKSPACE;
  const int64_t q_tiles = (a->num_q_heads / a->num_kv_heads + 15) / 16;   // (what a grid holds)
  if (a->num_q_heads > 65535 || (int64_t)a->num_seqs * a->num_kv_heads * q_tiles > INT_MAX ||
      (a->partition_size > 0 && (a->max_context_len - 1) / a->partition_size >= 65535))
    return FA_ERR_TOO_LARGE;
  return FA_OK;
}

template <typename T, int D, typename IdxT, int NQ>
static int launch_8bit(const fa_paged_8bit_args *p, const Sizing &z, cudaStream_t stream) {
  using C = Paged8Cfg<D, NQ>;
  const fa_paged_args *a = &p->paged;
  auto kern = paged_8bit_kernel<T, D, IdxT, NQ>;
  static unsigned long long attr_done = 0;  // per instantiation, one bit per device
  if (int st = ensure_dyn_smem(kern, C::kTotal, &attr_done)) return st;
  const int q_tiles = (a->num_q_heads / a->num_kv_heads + 15) / 16;
  const int P = a->partition_size > 0 ? partitions_of(*a) : 1;
  kern<<<dim3(a->num_seqs * a->num_kv_heads * q_tiles, P), C::kWarps * 32, C::kTotal, stream>>>(*p, z);
  FA_CHECK_LAUNCH();
  return FA_OK;
}

template <typename T, typename IdxT>
static int dispatch_8bit(const fa_paged_8bit_args *p, const Sizing &z, cudaStream_t s) {
  const bool one = p->paged.num_q_heads / p->paged.num_kv_heads <= 8;
  switch (p->paged.head_size) {
    case 16: return one ? launch_8bit<T, 16, IdxT, 1>(p, z, s) : launch_8bit<T, 16, IdxT, 2>(p, z, s);
    case 32: return one ? launch_8bit<T, 32, IdxT, 1>(p, z, s) : launch_8bit<T, 32, IdxT, 2>(p, z, s);
    case 64: return one ? launch_8bit<T, 64, IdxT, 1>(p, z, s) : launch_8bit<T, 64, IdxT, 2>(p, z, s);
    case 128: return one ? launch_8bit<T, 128, IdxT, 1>(p, z, s) : launch_8bit<T, 128, IdxT, 2>(p, z, s);
    default: return one ? launch_8bit<T, 256, IdxT, 1>(p, z, s) : launch_8bit<T, 256, IdxT, 2>(p, z, s);
  }
}

}  // namespace fa

using namespace fa;

extern "C" int fa_paged_attention_8bit(const fa_paged_8bit_args *p, int32_t finest, int32_t coarsest, int32_t ctas,
                                       int32_t parts, void *stream) {
  if (int st = validate_8bit(p)) return st;
  const fa_paged_args *a = &p->paged;
  const Sizing z{finest, coarsest, ctas, parts};
  if (finest && !sizing_ok(*a, z)) return FA_ERR_BAD_ARG;
  auto s = static_cast<cudaStream_t>(stream);
  int st;
  if (a->dtype == FA_F16)
    st = a->block_table_is_i64 ? dispatch_8bit<__half, int64_t>(p, z, s) : dispatch_8bit<__half, int32_t>(p, z, s);
  else
    st = a->block_table_is_i64 ? dispatch_8bit<__nv_bfloat16, int64_t>(p, z, s)
                               : dispatch_8bit<__nv_bfloat16, int32_t>(p, z, s);
  if (st != FA_OK || a->partition_size == 0) return st;
  return reduce(a, z, s);
}
