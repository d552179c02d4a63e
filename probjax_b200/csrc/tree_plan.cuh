// What the kernels of the tree attention share: the drafts' tree, and how the tiles of a ragged batch are dealt to CTAs.
#pragma once

#include "pjx_common.cuh"

namespace pjx {

// Parents of the drafts into `par` [N]: -1 hangs on the context, 0 <= parent < own index on a draft; everything else is absent
// (-2).  All threads of the CTA take part; one barrier.
__device__ __forceinline__ void load_tree(const TreeParams& p, int b, int16_t* par, int tid, int n_threads) {
  const int32_t* src = p.parents + b * p.parents_bs;
  for (int i = tid; i < p.N; i += n_threads) {
    const int v = src[i];
    par[i] = (int16_t)(v >= -1 && v < i ? v : -2);
  }
  __syncthreads();
}
// Whether draft i hangs on the context: what hangs on an absent draft is absent too.  Parents come before their children, so the
// walk ends.
__device__ __forceinline__ bool tree_present(const int16_t* par, int i) {
  while (i >= 0) i = par[i];
  return i == -1;
}

__device__ __forceinline__ int tree_prefix(const TreeParams& p, int b) { return max(0, min(p.capacity, p.kv_lengths[b])); }
__device__ __forceinline__ int tree_tiles(const TreeParams& p, int prefix) {
  return (prefix + kTreeTile - 1) / kTreeTile + (p.N + kTreeTile - 1) / kTreeTile;
}

// Splits of the batch: every split is a run of at most `unit` tiles of one sequence, numbered through the batch.  With per_seq > 0 every
// sequence has that many; otherwise `unit` is the smallest (up to a sixteenth) with which the batch has no more than p.splits.
// Computed by whole warps.
constexpr int kTreePlanSeqs = 128;  // sequences that are dealt out on the device: four per lane
struct TreeSplit {
  int b;          // sequence, -1: none
  int prefix;     // its cached keys
  int first, end; // tiles
};
struct TreePlan {
  int unit;
  int n[kTreePlanSeqs / 32], first[kTreePlanSeqs / 32];
};
__device__ __forceinline__ TreePlan tree_plan(const TreeParams& p) {
  constexpr int PER = kTreePlanSeqs / 32;
  const int lane = threadIdx.x & 31;
  TreePlan r;
  int tiles[PER], total = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = lane + 32 * i;
    tiles[i] = b < p.B ? tree_tiles(p, tree_prefix(p, b)) : 0;
    total += tiles[i];
  }
  total = __reduce_add_sync(0xffffffffu, total);
  r.unit = max(1, (total + p.splits - 1) / p.splits);
  while (true) {  // ends: p.splits >= B, and the longest sequence's tiles as the unit give one split each
    int cnt = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      r.n[i] = (tiles[i] + r.unit - 1) / r.unit;
      cnt += r.n[i];
    }
    if (static_cast<int>(__reduce_add_sync(0xffffffffu, cnt)) <= p.splits) break;
    r.unit += max(1, r.unit / 16);
  }
  int before = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    int incl = r.n[i];
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    r.first[i] = before + incl - r.n[i];
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return r;
}
// What split x of the batch is.
__device__ __forceinline__ TreeSplit tree_split(const TreeParams& p, int x) {
  TreeSplit s = {-1, 0, 0, 0};
  int unit;
  int index = 0;
  if (p.per_seq > 0) {
    s.b = x / p.per_seq;
    index = x - s.b * p.per_seq;
  } else {
    const TreePlan plan = tree_plan(p);
    unit = plan.unit;
#pragma unroll
    for (int i = 0; i < kTreePlanSeqs / 32; ++i) {
      const unsigned mine = __ballot_sync(0xffffffffu, x >= plan.first[i] && x < plan.first[i] + plan.n[i]);
      if (mine) {
        s.b = __ffs(mine) - 1 + 32 * i;
        index = x - __shfl_sync(0xffffffffu, plan.first[i], __ffs(mine) - 1);
      }
    }
    if (s.b < 0) return s;
  }
  s.prefix = tree_prefix(p, s.b);
  const int tiles = tree_tiles(p, s.prefix);
  if (p.per_seq > 0) unit = (tiles + p.per_seq - 1) / p.per_seq;
  s.first = index * unit;
  s.end = min(tiles, s.first + unit);
  if (s.first >= s.end) s.b = -1;
  return s;
}
// The splits of sequence b: their number and the first one's.
__device__ __forceinline__ void tree_splits_of(const TreeParams& p, int b, int& first, int& n) {
  if (p.per_seq > 0) {
    const int tiles = tree_tiles(p, tree_prefix(p, b));
    const int unit = (tiles + p.per_seq - 1) / p.per_seq;
    first = b * p.per_seq;
    n = (tiles + unit - 1) / unit;
    return;
  }
  const TreePlan plan = tree_plan(p);
  first = n = 0;
#pragma unroll
  for (int i = 0; i < kTreePlanSeqs / 32; ++i)
    if (b / 32 == i) {
      first = __shfl_sync(0xffffffffu, plan.first[i], b & 31);
      n = __shfl_sync(0xffffffffu, plan.n[i], b & 31);
    }
}

bool tree_sm100_supported(const TreeParams& p, int dtype, const char** why);
int launch_tree_sm100(const TreeParams& p, int dtype, cudaStream_t stream);

}  // namespace pjx
