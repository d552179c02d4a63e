// Attention of a tree of drafted tokens over a KV cache: draft i of sequence b sees the kv_lengths[b] cached keys and, among the
// drafts, itself and its ancestors.  o_i = sum_j softmax_j(sm_scale q_i . k_j) v_j; a draft that does not hang on the context
// (padding of a ragged batch) gives o = 0 and lse = +inf.
//
// This file holds the exact fp32 kernel on CUDA cores (fp32 inputs, head widths and alignments that the tensor-core kernel of
// attn_tree_sm100.cu does not take), the exact combine of the splits, and the entry point.
//
// The keys of the batch are cut into splits, the query rows (t, g) of a KV head's group into tiles; a CTA takes one of each and
// leaves O, normalised by its own sum, and a base-2 log-sum-exp in fp32.
#include "tree_plan.cuh"

namespace pjx {
namespace {

constexpr int NT = 256;
constexpr int BM = 64, BN = 64;
constexpr int PP = BN + 4;
constexpr int kWords = kTreeMaxNodes / 32;

__host__ __device__ inline int pitch4(int d) { return (d + 3) / 4 * 4 + 4; }
__device__ __forceinline__ float4 ld4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float dot4(float4 a, float4 b, float s) {
  return fmaf(a.w, b.w, fmaf(a.z, b.z, fmaf(a.y, b.y, fmaf(a.x, b.x, s))));
}

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
                                          int b, int hk, int prefix, int key0, int node0, const int16_t* par) {
  const int pitch = pitch4(width), u = threadIdx.x & 7;
  for (int r = threadIdx.x >> 3; r < BN; r += NT / 8) {
    const T* row = nullptr;
    if (node0 >= 0) {  // a tile of drafts: absent ones are nobody's keys, whatever they hold
      if (node0 + r < p.N && tree_present(par, node0 + r)) row = static_cast<const T*>(fresh) + b * bs + (node0 + r) * ts + (int64_t)hk * width;
    } else if (key0 + r < prefix) {
      const int64_t at = cache_row(p, b, key0 + r);
      if (at >= 0) row = static_cast<const T*>(cache) + (at * p.Hkv + hk) * width;
    }
    for (int d = u; d < (width + 3) / 4 * 4; d += 8) dst[r * pitch + d] = row && d < width ? Elem<T>::to_f(row[d]) : 0.f;
  }
}

template <typename T, int NCOL>  // NCOL: groups of 64 output columns
__global__ void __launch_bounds__(NT) attn_tree_kernel(const TreeParams p) {
  extern __shared__ float smem[];
  __shared__ int16_t par[kTreeMaxNodes];
  __shared__ uint32_t sees[BM][kWords];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int D = p.D, Dv = p.Dv, Dp = pitch4(D), Dvp = pitch4(Dv);
  float* Qs = smem;           // [BM][Dp]
  float* Ks = Qs + BM * Dp;   // [BN][Dp]
  float* Vs = Ks + BN * Dp;   // [BN][Dvp]
  float* Ps = Vs + BN * Dvp;  // [BM][PP]
  const TreeSplit sp = tree_split(p, blockIdx.x);
  if (sp.b < 0) return;  // (the combine never reads this split)
  const int G = p.Hq / p.Hkv, rows = p.N * G, row_tiles = (rows + BM - 1) / BM;
  const int hk = blockIdx.y / row_tiles, r0 = (blockIdx.y - hk * row_tiles) * BM;
  const int b = sp.b, prefix_tiles = (sp.prefix + kTreeTile - 1) / kTreeTile;
  load_tree(p, b, par, tid, NT);
  if (tid < BM) {
#pragma unroll
    for (int w = 0; w < kWords; ++w) sees[tid][w] = 0;
    const int node = (r0 + tid) / G;
    if (r0 + tid < rows && tree_present(par, node))
      for (int i = node; i >= 0; i = par[i]) sees[tid][i >> 5] |= 1u << (i & 31);
  }
  for (int i = tid; i < BM * Dp; i += NT) {
    const int r = i / Dp, d = i - r * Dp, row = r0 + r, t = row / G;
    Qs[i] = row < rows && d < D ? Elem<T>::to_f(static_cast<const T*>(p.q)[b * p.q_bs + t * p.q_ts + (int64_t)(hk * G + row - t * G) * D + d]) : 0.f;
  }
  float m[4], l[4];
  float4 acc[4][NCOL];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < NCOL; ++c) acc[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const float c1 = p.sm_scale * kLog2e;
  for (int half = 2 * sp.first; half < 2 * sp.end; ++half) {  // 64 keys: half a tile
    const bool drafts = half >= 2 * prefix_tiles;
    const int key0 = half * BN, node0 = drafts ? (half - 2 * prefix_tiles) * BN : -1;
    if (drafts ? node0 >= p.N : key0 >= sp.prefix) continue;
    __syncthreads();  // the tile before is consumed (and Qs, sees are written)
    load_keys<T>(p, Ks, D, p.k, p.k_new, p.kn_bs, p.kn_ts, b, hk, sp.prefix, key0, node0, par);
    load_keys<T>(p, Vs, Dv, p.v, p.v_new, p.vn_bs, p.vn_ts, b, hk, sp.prefix, key0, node0, par);
    __syncthreads();
    float s[4][4] = {};
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
      float4 qv[4], kv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) qv[i] = ld4(Qs + (ty * 4 + i) * Dp + d);
#pragma unroll
      for (int c = 0; c < 4; ++c) kv[c] = ld4(Ks + (tx + 16 * c) * Dp + d);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[i][c] = dot4(qv[i], kv[c], s[i][c]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = ty * 4 + i;
      float tmax = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int j = tx + 16 * c;
        bool keep;
        if (drafts)
          keep = node0 + j < p.N && (sees[r][(node0 + j) >> 5] >> ((node0 + j) & 31) & 1);
        else
          keep = key0 + j < sp.prefix;
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
        Ps[r * PP + tx + 16 * c] = Elem<T>::round(pv);  // as the other attention kernels round P before the product with V
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
      float4 pv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) pv[i] = ld4(Ps + (ty * 4 + i) * PP + kk);
#pragma unroll
      for (int c = 0; c < NCOL; ++c) {
        const int d = tx * 4 + 64 * c;
        if (d >= Dv) break;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4 x = ld4(Vs + (kk + e) * Dvp + d);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
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
  const int64_t part = ((int64_t)hk * p.splits + blockIdx.x) * rows;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + ty * 4 + i;
    if (r >= rows) continue;
    const bool there = l[i] > 0.f && tree_present(par, r / G);
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

// Exact combine of a row's splits, a warp per row.
template <typename TO>
__global__ void __launch_bounds__(256) tree_combine_kernel(const TreeParams p) {
  const int b = blockIdx.y, lane = threadIdx.x & 31;
  int first, ns;
  tree_splits_of(p, b, first, ns);  // (reads the lengths only: before the wait for the split kernel)
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= p.N * p.Hq) return;
  const int t = row / p.Hq, h = row - t * p.Hq, G = p.Hq / p.Hkv, hk = h / G;
  const int64_t rows = (int64_t)p.N * G;
  const int64_t base = ((int64_t)hk * p.splits + first) * rows + (int64_t)t * G + (h - hk * G);
  float m = -INFINITY;
  for (int s = lane; s < ns; s += 32) m = fmaxf(m, p.lse_part[base + s * rows]);
#pragma unroll
  for (int o = 16; o > 0; o /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float msafe = m == -INFINITY ? 0.f : m;
  float denom = 0.f;
  for (int s = lane; s < ns; s += 32) denom += exp2f(p.lse_part[base + s * rows] - msafe);
#pragma unroll
  for (int o = 16; o > 0; o /= 2) denom += __shfl_xor_sync(0xffffffffu, denom, o);
  const float inv = denom > 0.f ? 1.f / denom : 0.f;
  TO* out = static_cast<TO*>(p.o) + (((int64_t)b * p.N + t) * p.Hq + h) * p.Dv;
  if (p.Dv % 4 == 0) {
    for (int d = lane * 4; d < p.Dv; d += 128) {
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int s = 0; s < ns; ++s) {
        const float w = exp2f(p.lse_part[base + s * rows] - msafe);
        const float4 x = *reinterpret_cast<const float4*>(p.o_part + (base + s * rows) * p.Dv + d);
        acc.x = fmaf(w, x.x, acc.x);
        acc.y = fmaf(w, x.y, acc.y);
        acc.z = fmaf(w, x.z, acc.z);
        acc.w = fmaf(w, x.w, acc.w);
      }
      out[d] = Elem<TO>::from_f(acc.x * inv);
      out[d + 1] = Elem<TO>::from_f(acc.y * inv);
      out[d + 2] = Elem<TO>::from_f(acc.z * inv);
      out[d + 3] = Elem<TO>::from_f(acc.w * inv);
    }
  } else {
    for (int d = lane; d < p.Dv; d += 32) {
      float acc = 0.f;
      for (int s = 0; s < ns; ++s) acc = fmaf(exp2f(p.lse_part[base + s * rows] - msafe), p.o_part[(base + s * rows) * p.Dv + d], acc);
      out[d] = Elem<TO>::from_f(acc * inv);
    }
  }
  if (p.lse && lane == 0) p.lse[((int64_t)b * p.Hq + h) * p.N + t] = denom > 0.f ? (msafe + log2f(denom)) * kLn2 : INFINITY;
}

template <typename T>
int launch_generic(const TreeParams& p, cudaStream_t stream) {
  const int ncol = (p.Dv + 63) / 64;
  auto kern = ncol == 1 ? attn_tree_kernel<T, 1> : ncol == 2 ? attn_tree_kernel<T, 2> : ncol == 3 ? attn_tree_kernel<T, 3> : attn_tree_kernel<T, 4>;
  const int smem = (2 * BM * pitch4(p.D) + BN * pitch4(p.Dv) + BM * PP) * (int)sizeof(float);
  int rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "cudaFuncSetAttribute(tree)");
  if (rc) return rc;
  const int row_tiles = (p.N * (p.Hq / p.Hkv) + BM - 1) / BM;
  kern<<<dim3(p.splits, p.Hkv * row_tiles), NT, smem, stream>>>(p);
  count_launch();
  return check_cuda(cudaGetLastError(), "tree attention launch");
}

int launch_combine(const TreeParams& p, int dtype, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.N * p.Hq + 7) / 8, p.B);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = dtype == PJX_F32    ? cudaLaunchKernelEx(&cfg, tree_combine_kernel<float>, p)
                        : dtype == PJX_BF16 ? cudaLaunchKernelEx(&cfg, tree_combine_kernel<__nv_bfloat16>, p)
                                            : cudaLaunchKernelEx(&cfg, tree_combine_kernel<__half>, p);
  count_launch();
  return check_cuda(e, "tree combine launch");
}

inline size_t align256(size_t x) { return (x + 255) / 256 * 256; }

// Splits of the batch and where their number comes from.  A CTA per SM and (KV head, row tile) in `waves` waves, so that a
// ragged batch balances; the smallest split is one tile of keys.
void plan_splits(TreeParams& p) {
  const int G = p.Hq / p.Hkv;
  const int64_t units = (int64_t)p.Hkv * ((p.N * G + 127) / 128);  // CTAs that share a split of the keys
  const int64_t most = (p.capacity + kTreeTile - 1) / kTreeTile + (p.N + kTreeTile - 1) / kTreeTile;  // tiles of a sequence
  const int waves = 4;
  int64_t s = 148 * waves / units;
  if (s < p.B) s = p.B;
  if (s > most * p.B) s = most * p.B;
  if (p.B <= kTreePlanSeqs) {
    p.splits = (int)s;
    p.per_seq = 0;
  } else {
    p.per_seq = (int)(s / p.B);
    p.splits = p.per_seq * p.B;
  }
}

}  // namespace

}  // namespace pjx

extern "C" {

size_t pjx_attn_decode_tree_workspace_bytes(int B, int N, int Hq, int Hkv, int Dv, int capacity) {
  using namespace pjx;
  if (B < 1 || N < 1 || N > kTreeMaxNodes || Hq < 1 || Hkv < 1 || Dv < 1 || capacity < 0 || Hq % Hkv) return 0;
  TreeParams p = {};
  p.B = B; p.N = N; p.Hq = Hq; p.Hkv = Hkv; p.capacity = capacity;
  plan_splits(p);
  const size_t parts = (size_t)Hkv * p.splits * N * (Hq / Hkv);
  return align256(parts * Dv * sizeof(float)) + align256(parts * sizeof(float));
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
  if (!q || !k_new || !v_new || !o || !parents || !kv_lengths || (capacity > 0 && (!k_cache || !v_cache)))
    return fail(PJX_ERR_BAD_ARG, "tree: null buffer");
  if (N > kTreeMaxNodes) return fail(PJX_ERR_UNSUPPORTED, "tree: at most %d drafts a sequence (got %d)", kTreeMaxNodes, N);
  if (capacity >= PJX_BAND_NO_UPPER) return fail(PJX_ERR_UNSUPPORTED, "tree: cache capacity must be below 2^30 (got %d)", capacity);
  if (B > 65535 || Hq > 16384)
    return fail(PJX_ERR_UNSUPPORTED, "tree: at most 65535 sequences and 16384 heads per call (got B=%d, Hq=%d)", B, Hq);
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
  plan_splits(p);
  if ((int64_t)p.Hkv * ((p.N * (Hq / Hkv) + BM - 1) / BM) > 65535)
    return fail(PJX_ERR_UNSUPPORTED, "tree: too many rows for one launch (N=%d, Hq=%d)", N, Hq);
  const size_t parts = (size_t)Hkv * p.splits * N * (Hq / Hkv);
  const size_t o_bytes = align256(parts * Dv * sizeof(float)), need = o_bytes + align256(parts * sizeof(float));
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))
    return fail(PJX_ERR_WORKSPACE, "tree workspace: need %zu bytes, 16-byte aligned, got %zu", need, workspace ? workspace_bytes : (size_t)0);
  p.o_part = static_cast<float*>(workspace);
  p.lse_part = reinterpret_cast<float*>(static_cast<char*>(workspace) + o_bytes);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const char* why = nullptr;
  int rc;
  if (impl != PJX_IMPL_GENERIC && tree_sm100_supported(p, dtype, &why)) {
    rc = launch_tree_sm100(p, dtype, st);
  } else if (impl == PJX_IMPL_SM100) {
    return fail(PJX_ERR_UNSUPPORTED, "tcgen05 tree attention: %s", why);
  } else {
    if (D > 256 || Dv > 256) return fail(PJX_ERR_UNSUPPORTED, "tree: head widths up to 256 (got %d, %d)", D, Dv);
    rc = dtype == PJX_F32 ? launch_generic<float>(p, st) : dtype == PJX_BF16 ? launch_generic<__nv_bfloat16>(p, st) : launch_generic<__half>(p, st);
  }
  if (rc) return rc;
  return launch_combine(p, dtype, st);
}

}  // extern "C"
