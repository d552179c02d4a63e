// What the kernels of the tree attention share: the drafts' tree, and how the work of a ragged batch is dealt to the CTAs.
#pragma once

#include "pjx_common.cuh"

namespace pjx {

// Parent of draft i: -1 hangs on the context, 0 <= parent < i on that draft, everything else is absent (-2).
__device__ __forceinline__ int tree_parent(const int32_t* parents, int i) {
  const int v = __ldg(parents + i);
  return v >= -1 && v < i ? v : -2;
}
// Whether draft i hangs on the context: what hangs on an absent draft is absent too.  Parents come before their children, so the
// walk ends.
__device__ __forceinline__ bool tree_present(const int32_t* parents, int i) {
  while (i >= 0) i = tree_parent(parents, i);
  return i == -1;
}

__device__ __forceinline__ int tree_prefix(const TreeParams& p, int b) { return max(0, min(p.capacity, p.kv_lengths[b])); }
__device__ __forceinline__ int tree_tiles(const TreeParams& p, int prefix) {
  return (prefix + kTreeTile - 1) / kTreeTile + (p.N + kTreeTile - 1) / kTreeTile;
}

// The work is a line: for every column (a tile of query rows of one KV head) all key tiles of all sequences.  It is cut into
// equal runs, one per CTA, so that a ragged batch balances without knowing the lengths on the host, and a CTA's run falls into segments
// of one column and sequence.  Every segment leaves a partial result in a slot of its own: from one segment to the next on the line
// either the CTA or the (column, sequence) pair moves on by one, so their sum numbers the slots.
// All functions are computed by whole warps.
struct TreeLine {
  int tiles;       // key tiles of the batch
  int64_t length;  // tiles of all columns
  int ctas;        // CTAs that have work
};
__device__ __forceinline__ TreeLine tree_line(const TreeParams& p) {
  const int lane = threadIdx.x & 31;
  int sum = 0;
  for (int b = lane; b < p.B; b += 32) sum += tree_tiles(p, tree_prefix(p, b));
  TreeLine l;
  l.tiles = __reduce_add_sync(0xffffffffu, sum);
  l.length = (int64_t)l.tiles * p.columns;
  l.ctas = (int)min((int64_t)p.ctas, l.length);
  return l;
}
struct TreeSegment {
  int b, prefix;   // sequence, its cached keys
  int column;
  int first, end;  // tiles of the sequence
  bool last;       // its last tile is among them
  int64_t slot;
  int64_t pair;    // number of the (column, sequence)
};
// The segment at `pos` of CTA `cta`, whose run ends at `stop`.
__device__ __forceinline__ TreeSegment tree_segment(const TreeParams& p, const TreeLine& l, int cta, int64_t pos, int64_t stop) {
  const int lane = threadIdx.x & 31;
  TreeSegment s;
  s.column = (int)(pos / l.tiles);
  int at = (int)(pos - (int64_t)s.column * l.tiles);
  s.b = s.prefix = s.first = s.end = 0;
  for (int base = 0; base < p.B; base += 32) {
    const int prefix = base + lane < p.B ? tree_prefix(p, base + lane) : 0;
    const int tiles = base + lane < p.B ? tree_tiles(p, prefix) : 0;
    int incl = tiles;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    const unsigned past = __ballot_sync(0xffffffffu, at < incl);
    if (past) {
      const int src = __ffs(past) - 1;
      s.b = base + src;
      s.prefix = __shfl_sync(0xffffffffu, prefix, src);
      s.end = __shfl_sync(0xffffffffu, tiles, src);
      s.first = at - (__shfl_sync(0xffffffffu, incl, src) - s.end);
      break;
    }
    at -= __shfl_sync(0xffffffffu, incl, 31);
  }
  s.last = s.end <= s.first + (stop - pos);
  s.end = (int)min((int64_t)s.end, s.first + (stop - pos));
  s.pair = (int64_t)s.column * p.B + s.b;
  s.slot = cta + s.pair;
  return s;
}
__device__ __forceinline__ int64_t tree_run(const TreeLine& l, int cta) { return l.length * cta / l.ctas; }

bool tree_sm100_supported(const TreeParams& p, int dtype, const char** why);
// Geometry of the tensor-core kernel: rows of a column, columns, CTAs.
void tree_sm100_geometry(TreeParams& p);
int launch_tree_sm100(const TreeParams& p, int dtype, cudaStream_t stream);

}  // namespace pjx
