// Attention of a tree of drafted tokens over a KV cache: draft i of sequence b sees the kv_lengths[b] cached keys and, among the
// drafts, itself and its ancestors.  o_i = sum_j softmax_j(sm_scale q_i . k_j) v_j; a draft that does not hang on the context
// (padding of a ragged batch) gives o = 0 and lse = +inf.
//
// This file holds the exact fp32 kernel on CUDA cores (fp32 inputs, head widths and alignments that the tensor-core kernel of
// attn_tree_sm100.cu does not take; P stays in 32 bits, the one rounding is the result's), the exact combine of the splits, and the entry point.
//
// The work is cut into equal runs of (row tile, key tile) pairs, one per CTA (tree_plan.cuh); every segment of a run leaves O,
// normalised by its own sum, and a base-2 log-sum-exp in fp32.
#include "tile_f32.cuh"
#include "tree_plan.cuh"

namespace pjx {
namespace {

constexpr int NT = 256;
constexpr int BN = 64;
constexpr int PP = BN + 4;
constexpr int kWords = kTreeMaxNodes / 32;

// Row of the cache that holds key `key` of sequence b, -1 for a page outside the pool.
__device__ __forceinline__ int64_t cache_row(const TreeParams& p, int b, int key) {
  if (!p.block_table) return (int64_t)b * p.capacity + key;
  const int page = p.block_table[(int64_t)b * p.max_pages + key / p.page_size];
  if (page < 0 || page >= p.num_pages) return -1;
  return (int64_t)page * p.page_size + key % p.page_size;
}

// 64 keys (or values) of `width` elements as fp32; what is not there, and the padding to a multiple of four, as zeros.
template <typename T>
__device__ __forceinline__ void load_keys(const TreeParams& p, float* dst, int width, const void* cache, const void* fresh, int64_t bs, int64_t ts,
                                          int b, int hk, int prefix, int key0, int node0, const int32_t* parents) {
  const int pitch = pitch4(width), u = threadIdx.x & 7;
  for (int r = threadIdx.x >> 3; r < BN; r += NT / 8) {
    const T* row = nullptr;
    if (node0 >= 0) {  // a tile of drafts: absent ones are nobody's keys, whatever they hold
      if (node0 + r < p.N && tree_present(parents, node0 + r)) row = static_cast<const T*>(fresh) + b * bs + (node0 + r) * ts + (int64_t)hk * width;
    } else if (key0 + r < prefix) {
      const int64_t at = cache_row(p, b, key0 + r);
      if (at >= 0) row = static_cast<const T*>(cache) + (at * p.Hkv + hk) * width;
    }
    for (int d = u; d < (width + 3) / 4 * 4; d += 8) dst[r * pitch + d] = row && d < width ? Elem<T>::to_f(row[d]) : 0.f;
  }
}

// NCOL: groups of 64 output columns.  RT: rows per thread; 16 RT rows a tile (with few rows the 64-row tile would work on padding).
template <typename T, int NCOL, int RT>
__global__ void __launch_bounds__(NT) attn_tree_kernel(const TreeParams p) {
  constexpr int BM = 16 * RT;
  extern __shared__ float smem[];
  __shared__ uint32_t sees[BM][kWords];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int D = p.D, Dv = p.Dv, Dp = pitch4(D), Dvp = pitch4(Dv);
  float* Qs = smem;           // [BM][Dp]
  float* Ks = Qs + BM * Dp;   // [BN][Dp]
  float* Vs = Ks + BN * Dp;   // [BN][Dvp]
  float* Ps = Vs + BN * Dvp;  // [BM][PP]
  const int G = p.Hq / p.Hkv, rows = p.N * G, row_tiles = p.columns / p.Hkv;
  const float c1 = p.sm_scale * kLog2e;
  const TreeLine line = tree_line(p);
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  if ((int)blockIdx.x >= line.ctas) return;
  const int64_t stop = tree_run(line, blockIdx.x + 1);
  for (int64_t pos = tree_run(line, blockIdx.x); pos < stop;) {
    const TreeSegment sg = tree_segment(p, line, blockIdx.x, pos, stop);
    pos += sg.end - sg.first;
    const int b = sg.b, hk = sg.column / row_tiles, r0 = (sg.column - hk * row_tiles) * BM;
    const int prefix_tiles = (sg.prefix + kTreeTile - 1) / kTreeTile;
    const int32_t* parents = p.parents + b * p.parents_bs;
    if (tid == 0) {  // the combine's list
      if (sg.first == 0) p.slots[2 * sg.pair] = (int)sg.slot;
      if (sg.last) p.slots[2 * sg.pair + 1] = (int)sg.slot;
    }
    if (sg.first == 0 && sg.column == 0)
      for (int i = tid; i < p.N; i += NT) p.present[(int64_t)b * p.N + i] = tree_present(parents, i);
    __syncthreads();  // the segment before is done with shared memory
    if (tid < BM) {
#pragma unroll
      for (int w = 0; w < kWords; ++w) sees[tid][w] = 0;
      const int node = (r0 + tid) / G;
      if (r0 + tid < rows && tree_present(parents, node))
        for (int i = node; i >= 0; i = tree_parent(parents, i)) sees[tid][i >> 5] |= 1u << (i & 31);
    }
    for (int i = tid; i < BM * Dp; i += NT) {
      const int r = i / Dp, d = i - r * Dp, row = r0 + r, t = row / G;
      Qs[i] = row < rows && d < D ? Elem<T>::to_f(static_cast<const T*>(p.q)[b * p.q_bs + t * p.q_ts + (int64_t)(hk * G + row - t * G) * D + d]) : 0.f;
    }
    float m[RT], l[RT];
    float4 acc[RT][NCOL];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int c = 0; c < NCOL; ++c) acc[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int half = 2 * sg.first; half < 2 * sg.end; ++half) {  // 64 keys: half a tile
      const bool drafts = half >= 2 * prefix_tiles;
      const int key0 = half * BN, node0 = drafts ? (half - 2 * prefix_tiles) * BN : -1;
      if (drafts ? node0 >= p.N : key0 >= sg.prefix) continue;
      __syncthreads();  // the tile before is consumed (and Qs, sees are written)
      load_keys<T>(p, Ks, D, p.k, p.k_new, p.kn_bs, p.kn_ts, b, hk, sg.prefix, key0, node0, parents);
      load_keys<T>(p, Vs, Dv, p.v, p.v_new, p.vn_bs, p.vn_ts, b, hk, sg.prefix, key0, node0, parents);
      __syncthreads();
      float s[RT][4] = {};
#pragma unroll 4
      for (int d = 0; d < D; d += 4) {
        float4 qv[RT], kv[4];
#pragma unroll
        for (int i = 0; i < RT; ++i) qv[i] = ld4(Qs + (ty * RT + i) * Dp + d);
#pragma unroll
        for (int c = 0; c < 4; ++c) kv[c] = ld4(Ks + (tx + 16 * c) * Dp + d);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[i][c] = dot4(qv[i], kv[c], s[i][c]);
      }
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const int r = ty * RT + i;
        float tmax = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int j = tx + 16 * c;
          bool keep;
          if (drafts)
            keep = node0 + j < p.N && (sees[r][(node0 + j) >> 5] >> ((node0 + j) & 31) & 1);
          else
            keep = key0 + j < sg.prefix;
          s[i][c] = keep ? s[i][c] * c1 : -INFINITY;
          tmax = fmaxf(tmax, s[i][c]);
        }
#pragma unroll
        for (int off = 8; off >= 1; off >>= 1) tmax = fmaxf(tmax, __shfl_xor_sync(0xffffffffu, tmax, off));
        const float m_new = fmaxf(m[i], tmax);
        const float m_safe = m_new == -INFINITY ? 0.f : m_new;
        const float corr = exp2f(m[i] - m_safe);
        float rsum = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float pv = exp2f(s[i][c] - m_safe);
          rsum += pv;
          Ps[r * PP + tx + 16 * c] = pv;
        }
#pragma unroll
        for (int off = 8; off >= 1; off >>= 1) rsum += __shfl_xor_sync(0xffffffffu, rsum, off);
        l[i] = l[i] * corr + rsum;
        m[i] = m_new;
#pragma unroll
        for (int c = 0; c < NCOL; ++c) {
          acc[i][c].x *= corr;
          acc[i][c].y *= corr;
          acc[i][c].z *= corr;
          acc[i][c].w *= corr;
        }
      }
      __syncthreads();
      for (int kk = 0; kk < BN; kk += 4) {
        float4 pv[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) pv[i] = ld4(Ps + (ty * RT + i) * PP + kk);
#pragma unroll
        for (int c = 0; c < NCOL; ++c) {
          const int d = tx * 4 + 64 * c;
          if (d >= Dv) break;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float4 x = ld4(Vs + (kk + e) * Dvp + d);
#pragma unroll
            for (int i = 0; i < RT; ++i) {
              const float w = e == 0 ? pv[i].x : e == 1 ? pv[i].y : e == 2 ? pv[i].z : pv[i].w;
              acc[i][c].x = fmaf(w, x.x, acc[i][c].x);
              acc[i][c].y = fmaf(w, x.y, acc[i][c].y);
              acc[i][c].z = fmaf(w, x.z, acc[i][c].z);
              acc[i][c].w = fmaf(w, x.w, acc[i][c].w);
            }
          }
        }
      }
    }
    const int64_t part = sg.slot * p.column_rows;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int r = ty * RT + i;
      if (r0 + r >= rows) continue;
      const bool there = l[i] != 0.f;  // (a sum that is not a number stays one, in the output and in the log-sum-exp)
      const float inv = there ? 1.f / l[i] : 0.f;
#pragma unroll
      for (int c = 0; c < NCOL; ++c) {
        const float x[4] = {acc[i][c].x, acc[i][c].y, acc[i][c].z, acc[i][c].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = tx * 4 + 64 * c + e;
          if (d < Dv) p.o_part[(part + r) * Dv + d] = there ? x[e] * inv : 0.f;
        }
      }
      if (tx == 0) p.lse_part[part + r] = there ? m[i] + log2f(l[i]) : -INFINITY;
    }
  }
}

template <typename TO>
__device__ __forceinline__ void store_row4(TO* out, int d, int width, float4 x) {
  const float y[4] = {x.x, x.y, x.z, x.w};
  if (width % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & (4 * sizeof(TO) - 1)) == 0) {
    if (d < width) {
      struct alignas(4 * sizeof(TO)) Four { TO v[4]; } four;
#pragma unroll
      for (int e = 0; e < 4; ++e) four.v[e] = Elem<TO>::from_f(y[e]);
      *reinterpret_cast<Four*>(out + d) = four;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (d + e < width) out[d + e] = Elem<TO>::from_f(y[e]);
  }
}
__device__ __forceinline__ float4 load_part4(const float* x, int d, int width) {
  if (width % 4 == 0) return d < width ? *reinterpret_cast<const float4*>(x + d) : make_float4(0.f, 0.f, 0.f, 0.f);
  return make_float4(d < width ? x[d] : 0.f, d + 1 < width ? x[d + 1] : 0.f, d + 2 < width ? x[d + 2] : 0.f, d + 3 < width ? x[d + 3] : 0.f);
}
__device__ __forceinline__ void add4(float4& acc, float w, float4 x) {
  acc.x = fmaf(w, x.x, acc.x);
  acc.y = fmaf(w, x.y, acc.y);
  acc.z = fmaf(w, x.z, acc.z);
  acc.w = fmaf(w, x.w, acc.w);
}

// Exact combine of the rows' segments, EACH rows a warp.  The chain of a row is slot range -> log-sum-exps and partial rows -> result; the
// rows of a warp take it side by side, with the first two partial rows loaded before their weights are known (B16 N64 32/8
// heads of 128, by itself under a profiler: 28-29 us before, 26-29 now).  Rows of absent drafts come out empty whatever the segments hold.
template <typename TO, int EACH>
__global__ void __launch_bounds__(256) tree_combine_kernel(const TreeParams p) {
  const int b = blockIdx.y, lane = threadIdx.x & 31, G = p.Hq / p.Hkv, total = p.N * p.Hq;
  const int row0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * EACH;
  if (row0 >= total) return;
  // lane e: row row0 + e
  const int my_t = min(row0 + lane, total - 1) / p.Hq, my_h = min(row0 + lane, total - 1) - my_t * p.Hq, my_hk = my_h / G;
  const int my_r = my_t * G + my_h - my_hk * G, my_column = my_hk * (p.columns / p.Hkv) + my_r / p.column_rows;
  const bool mine = lane < EACH && row0 + lane < total;
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  int my_ns = 0;
  int64_t my_base = 0;
  if (mine) {
    const bool there = p.present[(int64_t)b * p.N + my_t] != 0;
    const int2 range = *reinterpret_cast<const int2*>(p.slots + 2 * ((int64_t)my_column * p.B + b));
    // (a kernel that gave up may have left no slots)
    if (there && range.x >= 0 && range.y >= range.x && range.y < p.ctas + (int64_t)p.columns * p.B) my_ns = range.y - range.x + 1;
    my_base = (int64_t)range.x * p.column_rows + my_r % p.column_rows;
  }
  int ns[EACH];
  int64_t base[EACH];
  float l[EACH];  // lane s: log-sum-exp of segment s
  float4 x[EACH][2];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    ns[e] = __shfl_sync(0xffffffffu, my_ns, e);
    base[e] = __shfl_sync(0xffffffffu, my_base, e);
    l[e] = lane < ns[e] ? p.lse_part[base[e] + (int64_t)lane * p.column_rows] : -INFINITY;
#pragma unroll
    for (int s = 0; s < 2; ++s)
      x[e][s] = s < ns[e] ? load_part4(p.o_part + (base[e] + (int64_t)s * p.column_rows) * p.Dv, lane * 4, p.Dv) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    if (row0 + e >= total) break;
    const float* lses = p.lse_part + base[e];
    float m = l[e];
    for (int s = 32 + lane; s < ns[e]; s += 32) m = fmaxf(m, lses[(int64_t)s * p.column_rows]);
#pragma unroll
    for (int o = 16; o > 0; o /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float msafe = m == -INFINITY ? 0.f : m;
    const float w0 = exp2f(l[e] - msafe);
    float denom = w0;
    for (int s = 32 + lane; s < ns[e]; s += 32) denom += exp2f(lses[(int64_t)s * p.column_rows] - msafe);
#pragma unroll
    for (int o = 16; o > 0; o /= 2) denom += __shfl_xor_sync(0xffffffffu, denom, o);
    const float inv = denom != 0.f ? 1.f / denom : 0.f;
    const int t = (row0 + e) / p.Hq, h = row0 + e - t * p.Hq;
    TO* out = static_cast<TO*>(p.o) + (((int64_t)b * p.N + t) * p.Hq + h) * p.Dv;
    for (int d = lane * 4; d - lane * 4 < p.Dv; d += 128) {
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int s0 = 0; s0 < ns[e]; s0 += 32) {
        const float w_mine = s0 == 0 ? w0 : s0 + lane < ns[e] ? exp2f(lses[(int64_t)(s0 + lane) * p.column_rows] - msafe) : 0.f;
        const int many = min(32, ns[e] - s0);
        int s = 0;
        if (s0 == 0 && d < 128) {
          add4(acc, __shfl_sync(0xffffffffu, w_mine, 0), x[e][0]);
          add4(acc, __shfl_sync(0xffffffffu, w_mine, 1), x[e][1]);  // (zero with a weight of zero where there is one segment)
          s = 2;
        }
#pragma unroll 4
        for (; s < many; ++s)
          add4(acc, __shfl_sync(0xffffffffu, w_mine, s), load_part4(p.o_part + (base[e] + (int64_t)(s0 + s) * p.column_rows) * p.Dv, d, p.Dv));
      }
      store_row4(out, d, p.Dv, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
    }
    if (p.lse && lane == 0) p.lse[((int64_t)b * p.Hq + h) * p.N + t] = denom != 0.f ? (msafe + log2f(denom)) * kLn2 : INFINITY;
  }
}

constexpr int generic_rows(int rows) { return rows <= 16 ? 16 : 64; }

template <typename T, int RT>
int launch_generic_t(const TreeParams& p, cudaStream_t stream) {
  constexpr int BM = 16 * RT;
  const int ncol = (p.Dv + 63) / 64;
  auto kern = ncol == 1   ? attn_tree_kernel<T, 1, RT>
              : ncol == 2 ? attn_tree_kernel<T, 2, RT>
              : ncol == 3 ? attn_tree_kernel<T, 3, RT>
                          : attn_tree_kernel<T, 4, RT>;
  auto smem_bytes = [](int D, int Dv) { return ((BM + BN) * pitch4(D) + BN * pitch4(Dv) + BM * PP) * (int)sizeof(float); };
  const int smem = smem_bytes(p.D, p.Dv);
  static std::atomic<uint64_t> allowed[4] = {};  // (for the widest call: another thread's must not lower it before this launch)
  int rc = allow_smem(reinterpret_cast<const void*>(kern), smem_bytes(256, 64 * ncol), allowed[ncol - 1]);
  if (rc) return rc;
  kern<<<p.ctas, NT, smem, stream>>>(p);
  count_launch();
  return check_cuda(cudaGetLastError(), "tree attention launch");
}

template <typename T>
int launch_generic(const TreeParams& p, cudaStream_t stream) {
  return generic_rows(p.N * (p.Hq / p.Hkv)) == 16 ? launch_generic_t<T, 1>(p, stream) : launch_generic_t<T, 4>(p, stream);
}

int launch_combine(const TreeParams& p, int dtype, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  const int each = (int64_t)p.N * p.Hq * p.B >= 148 * 64 ? 4 : 1;  // (few rows: all of them at once)
  cfg.gridDim = dim3((p.N * p.Hq + 8 * each - 1) / (8 * each), p.B);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto kern = dtype == PJX_F32    ? (each == 1 ? tree_combine_kernel<float, 1> : tree_combine_kernel<float, 4>)
              : dtype == PJX_BF16 ? (each == 1 ? tree_combine_kernel<__nv_bfloat16, 1> : tree_combine_kernel<__nv_bfloat16, 4>)
                                  : (each == 1 ? tree_combine_kernel<__half, 1> : tree_combine_kernel<__half, 4>);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  count_launch();
  return check_cuda(e, "tree combine launch");
}

inline size_t align256(size_t x) { return (x + 255) / 256 * 256; }

// Columns of 16 or 64 rows.  Two runs per SM: shared memory holds two CTAs where a call's tiles take up to 113 KB (64 rows of width 96, 16
// of width 128), otherwise (64 rows of width 128: 119 KB) one, and the runs follow one another.
void generic_geometry(TreeParams& p) {
  const int rows = p.N * (p.Hq / p.Hkv), tile = generic_rows(rows);
  p.column_rows = rows < tile ? rows : tile;
  p.columns = p.Hkv * ((rows + tile - 1) / tile);
  p.ctas = 2 * 148;
}

size_t partial_rows(const TreeParams& p) { return ((size_t)p.ctas + (size_t)p.columns * p.B) * p.column_rows; }
size_t partial_bytes(const TreeParams& p) {
  return align256(partial_rows(p) * p.Dv * sizeof(float)) + align256(partial_rows(p) * sizeof(float)) +
         align256((size_t)p.columns * p.B * 2 * sizeof(int32_t)) + align256((size_t)p.B * p.N);
}

}  // namespace

}  // namespace pjx

extern "C" {

size_t pjx_attn_decode_tree_workspace_bytes(int B, int N, int Hq, int Hkv, int Dv, int capacity) {
  using namespace pjx;
  if (B < 1 || N < 1 || N > kTreeMaxNodes || Hq < 1 || Hkv < 1 || Dv < 1 || capacity < 0 || Hq % Hkv) return 0;
  TreeParams p = {};
  p.B = B; p.N = N; p.Hq = Hq; p.Hkv = Hkv; p.Dv = Dv; p.capacity = capacity;
  generic_geometry(p);
  size_t need = partial_bytes(p);
  if (Hq / Hkv <= 128) {  // (enough for either kernel)
    tree_sm100_geometry(p);
    const size_t other = partial_bytes(p);
    if (other > need) need = other;
  }
  return need;
}

int pjx_attn_decode_tree(const void* q, int64_t q_batch_stride, int64_t q_token_stride, const void* k_new, int64_t k_new_batch_stride,
                         int64_t k_new_token_stride, const void* v_new, int64_t v_new_batch_stride, int64_t v_new_token_stride,
                         const void* k_cache, const void* v_cache, const int32_t* parents, int64_t parents_batch_stride,
                         const int32_t* kv_lengths, const int32_t* block_table, void* o, float* lse, int B, int N, int Hq, int Hkv, int D,
                         int Dv, int capacity, int page_size, int max_pages, int num_pages, int dtype, float sm_scale, int impl,
                         void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  using namespace pjx;
  if (dtype != PJX_F32 && dtype != PJX_BF16 && dtype != PJX_F16)
    return fail(PJX_ERR_BAD_ARG, "dtype must be float32, bfloat16 or float16 (got code %d)", dtype);
  if (B < 0 || N < 0 || Hq < 1 || Hkv < 1 || D < 1 || Dv < 1 || capacity < 0)
    return fail(PJX_ERR_BAD_ARG, "negative or zero dimension (B=%d N=%d Hq=%d Hkv=%d D=%d Dv=%d capacity=%d)", B, N, Hq, Hkv, D, Dv, capacity);
  if (Hq % Hkv != 0) return fail(PJX_ERR_BAD_ARG, "query heads %d must be a multiple of kv heads %d", Hq, Hkv);
  if (impl != PJX_IMPL_AUTO && impl != PJX_IMPL_GENERIC && impl != PJX_IMPL_SM100)
    return fail(PJX_ERR_BAD_ARG, "impl must be 0 (auto), 1 (generic) or 2 (tcgen05), got %d", impl);
  if (q_batch_stride < 0 || q_token_stride < 0 || k_new_batch_stride < 0 || k_new_token_stride < 0 || v_new_batch_stride < 0 ||
      v_new_token_stride < 0 || parents_batch_stride < 0)
    return fail(PJX_ERR_BAD_ARG, "tree: strides must be non-negative");
  if (block_table) {
    if (page_size < 16 || page_size % 16) return fail(PJX_ERR_BAD_ARG, "page_size must be a positive multiple of 16 (got %d)", page_size);
    if (max_pages < 0 || num_pages < 0 || (int64_t)max_pages * page_size >= PJX_BAND_NO_UPPER)
      return fail(PJX_ERR_BAD_ARG, "max_pages * page_size must be below 2^30");
    capacity = max_pages * page_size;
  }
  if (B == 0 || N == 0) return PJX_OK;
  if (!q || !k_new || !v_new || !o || !parents || !kv_lengths || (capacity > 0 && !(block_table && num_pages == 0) && (!k_cache || !v_cache)))
    return fail(PJX_ERR_BAD_ARG, "tree: null buffer");
  if (N > kTreeMaxNodes) return fail(PJX_ERR_UNSUPPORTED, "tree: at most %d drafts a sequence (got %d)", kTreeMaxNodes, N);
  if (capacity >= PJX_BAND_NO_UPPER) return fail(PJX_ERR_UNSUPPORTED, "tree: cache capacity must be below 2^30 (got %d)", capacity);
  if (B > 65535 || Hq > 16384 || (int64_t)B * Hkv * N > (1 << 30))
    return fail(PJX_ERR_UNSUPPORTED, "tree: at most 65535 sequences, 16384 heads and 2^30 rows per call (got B=%d, N=%d, Hq=%d)", B, N, Hq);
  if ((int64_t)B * ((capacity + kTreeTile - 1) / kTreeTile + 2) > 0x7fffffffLL)
    return fail(PJX_ERR_UNSUPPORTED, "tree: at most 2^31 key tiles of %d per call (B=%d, capacity=%d)", kTreeTile, B, capacity);
  TreeParams p = {};
  p.q = q; p.k_new = k_new; p.v_new = v_new; p.k = k_cache; p.v = v_cache;
  p.q_bs = q_batch_stride; p.q_ts = q_token_stride;
  p.kn_bs = k_new_batch_stride; p.kn_ts = k_new_token_stride;
  p.vn_bs = v_new_batch_stride; p.vn_ts = v_new_token_stride;
  p.parents = parents; p.parents_bs = parents_batch_stride;
  p.kv_lengths = kv_lengths; p.block_table = block_table;
  p.page_size = page_size; p.max_pages = max_pages; p.num_pages = num_pages;
  p.o = o; p.lse = lse;
  p.B = B; p.N = N; p.Hq = Hq; p.Hkv = Hkv; p.D = D; p.Dv = Dv; p.capacity = capacity;
  p.sm_scale = sm_scale;
  p.status = status;
  const char* why = nullptr;
  const bool tc = impl != PJX_IMPL_GENERIC && tree_sm100_supported(p, dtype, &why);
  if (!tc && impl == PJX_IMPL_SM100) return fail(PJX_ERR_UNSUPPORTED, "tcgen05 tree attention: %s", why);
  if (!tc && (D > 256 || Dv > 256)) return fail(PJX_ERR_UNSUPPORTED, "tree: head widths up to 256 (got %d, %d)", D, Dv);
  const size_t need = pjx_attn_decode_tree_workspace_bytes(B, N, Hq, Hkv, Dv, capacity);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))
    return fail(PJX_ERR_WORKSPACE, "tree workspace: need %zu bytes, 16-byte aligned, got %zu", need, workspace ? workspace_bytes : (size_t)0);
  if (tc)
    tree_sm100_geometry(p);
  else
    generic_geometry(p);
  p.o_part = static_cast<float*>(workspace);
  p.lse_part = reinterpret_cast<float*>(static_cast<char*>(workspace) + align256(partial_rows(p) * Dv * sizeof(float)));
  p.slots = reinterpret_cast<int32_t*>(reinterpret_cast<char*>(p.lse_part) + align256(partial_rows(p) * sizeof(float)));
  p.present = reinterpret_cast<uint8_t*>(p.slots) + align256((size_t)p.columns * B * 2 * sizeof(int32_t));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int rc = tc ? launch_tree_sm100(p, dtype, st)
              : dtype == PJX_F32 ? launch_generic<float>(p, st) : dtype == PJX_BF16 ? launch_generic<__nv_bfloat16>(p, st) : launch_generic<__half>(p, st);
  if (rc) return rc;
  return launch_combine(p, dtype, st);
}

}  // extern "C"
