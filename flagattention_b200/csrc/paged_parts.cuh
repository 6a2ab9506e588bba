// What the decode kernels over a paged cache share, of 16 bits and of 8: the block table, the lengths, the partitions and
// the reduction of their results.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "flagattn_b200.h"

namespace fa {

// IdxT: the table's entry type, or InPlace where there is no table (FA_BLOCK_TABLE_IN_PLACE)
struct InPlace {};
template <typename IdxT>
__device__ __forceinline__ int64_t phys_block(const void *block_tables, int64_t bt_stride_s,
                                              int seq, int logical_block) {
  const int64_t i = (int64_t)seq * bt_stride_s + logical_block;
  if constexpr (std::is_same<IdxT, InPlace>::value) return i;
  else return (int64_t) reinterpret_cast<const IdxT *>(block_tables)[i];
}
__device__ __forceinline__ int context_len(const fa_paged_args &a, int seq) {
  return a.context_lens ? a.context_lens[seq] : a.max_context_len;
}

// the partitions of a row in the workspace (the bound and a partition may come to more than 32 bits)
__host__ __device__ inline int partitions_of(const fa_paged_args &a) { return (a.max_context_len - 1) / a.partition_size + 1; }

// How the kernels size the partitions of fa_paged_attention from the lengths themselves; finest == 0: every sequence
// takes a.partition_size.  Sizes are finest * 2^k.
struct Sizing {
  int finest, coarsest;
  int ctas;    // > 0: the largest size, up to `coarsest`, that leaves the whole call this many CTAs
  int parts;   // ctas == 0: the smallest size that cuts a sequence into this many at most
};
// The lengths of the first 64 sequences, two a lane, requested ahead of their use.
struct LaneLens {
  int first, second;
};
__device__ __forceinline__ LaneLens lane_lens(const fa_paged_args &a, const Sizing &z) {
  const int lane = threadIdx.x & 31;
  return LaneLens{z.ctas > 0 && lane < a.num_seqs ? context_len(a, lane) : 0,
                  z.ctas > 0 && lane + 32 < a.num_seqs ? context_len(a, lane + 32) : 0};
}
// Tokens per partition of a sequence of `ctx` tokens, called by whole warps; never more partitions than the P of the
// workspace.
__device__ __forceinline__ int partition_tokens(const fa_paged_args &a, const Sizing &z, LaneLens lens, int ctx, int P) {
  if (z.finest == 0) return a.partition_size;
  int k = 0;
  if (z.ctas > 0) {
    auto count = [&](int len) { return min(((unsigned)max(len, 0) + z.finest - 1) / z.finest, 1u << 20); };
    unsigned lane_n = count(lens.first) + count(lens.second);
    for (int i = (threadIdx.x & 31) + 64; i < a.num_seqs; i += 32) lane_n += count(context_len(a, i));
    // (a sum below 2^32: at most 2048 sequences)
    const unsigned long long n = (unsigned long long)__reduce_add_sync(0xffffffffu, lane_n) *
                                 (a.num_kv_heads * ((a.num_q_heads / a.num_kv_heads + 15) / 16));
    while ((z.finest << k) < z.coarsest && (n >> (k + 1)) >= (unsigned)z.ctas) ++k;
  }
  const int parts = z.ctas > 0 ? P : min(P, z.parts);
  while ((z.finest << k) < a.partition_size && (long long)parts * (z.finest << k) < ctx) ++k;
  return z.finest << k;
}
// size / finest is a power of two
inline bool nests(int size, int finest) {
  return size % finest == 0 && ((size / finest) & (size / finest - 1)) == 0;
}
inline bool sizing_ok(const fa_paged_args &a, const Sizing &z) {
  if (a.partition_size <= 0 || a.partition_size > (1 << 24) || z.finest <= 0 || z.finest % 16 || z.finest > a.partition_size ||
      z.coarsest < z.finest || z.coarsest > (1 << 24) || !nests(a.partition_size, z.finest) || !nests(z.coarsest, z.finest))
    return false;
  return z.ctas >= 0 && (z.ctas > 0 || z.parts > 0) && (z.ctas == 0 || a.num_seqs <= 2048);
}

// a.out from the partial results of a.partition_size > 0 (paged.cu)
int reduce(const fa_paged_args *a, const Sizing &z, cudaStream_t s);

}  // namespace fa
