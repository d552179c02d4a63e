// Two updates of a KV cache that are more than an append at the end:
//
//  * accept: the accepted path of a tree of drafted tokens enters the cache.  Row path[b, i] of the drafts' keys and values
//    goes to cache row lengths[b] + i, i < counts[b], and the lengths advance on the device.
//  * evict: every (sequence, KV head) keeps the `recent` last keys and, of the others, those with the most accumulated
//    attention (the lowest index first where weights tie); the kept rows move to the front in their order.
//
// Measured on a cache of 16 ragged sequences of 4k-32k keys, 8 heads of 128, bf16, cut to 8192 keys: the call 213 us; in
// a trace selection 36 (259 with the weights read again in every pass, 11-bit digits and clusters), movement 177 = 5.8 TB/s of rows
// read and written.  One sequence of 4001 keys cut to 1024: 11 and 6 us on the device, the call 20.  In place 190 and 26-28 us: rows that stay
// are not moved, but a head of one sequence has a CTA per 128 bytes of its rows only.
//
// No counterpart in the reference, whose cache only grows (probjax/nn/layers/attention.py:631-643).
#include <cooperative_groups.h>

#include "pjx_common.cuh"

namespace cg = cooperative_groups;

namespace pjx {
namespace {

// ------------------------------------------------------------------------------------------------ accept

constexpr int kAcceptCluster = 8;

struct AcceptParams {
  void *k_cache, *v_cache;
  const char *k_new, *v_new;             // row (b, n) at b * bs + n * ts bytes
  int64_t kn_bs, kn_ts, vn_bs, vn_ts;
  const int32_t *lengths, *path, *counts, *block_table;
  int32_t *lengths_out, *overflow;
  int capacity, N, P, page_size, max_pages, num_pages;
  int k_units, v_units;                  // 16-byte units of a token's keys and values
};

// One cluster per sequence: its CTAs share the rows, and all of them have read the length before one writes the new one, so
// that lengths_out may be lengths.  A few rows of a few KB each: bound by the latency of one launch and one dependent load.
__global__ void __cluster_dims__(kAcceptCluster, 1, 1) __launch_bounds__(256) kv_accept_kernel(const AcceptParams p) {
  const int b = blockIdx.y;
  const int len = max(0, p.lengths[b]);
  const int count = max(0, min(p.P, p.counts[b]));
  cg::this_cluster().sync();
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    p.lengths_out[b] = (int)min((int64_t)p.capacity, (int64_t)len + count);
    if (p.overflow && (int64_t)len + count > p.capacity) atomicExch(p.overflow, 1);
  }
  const int per_row = p.k_units + p.v_units;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < (int64_t)count * per_row; i += kAcceptCluster * blockDim.x) {
    const int t = (int)(i / per_row);
    int u = (int)(i - (int64_t)t * per_row);
    const int node = p.path[(int64_t)b * p.P + t];
    const int64_t row = (int64_t)len + t;
    if (node < 0 || node >= p.N || row >= p.capacity) continue;
    int64_t at = (int64_t)b * p.capacity + row;
    if (p.block_table) {
      const int page = p.block_table[(int64_t)b * p.max_pages + row / p.page_size];
      if (page < 0 || page >= p.num_pages) continue;
      at = (int64_t)page * p.page_size + row % p.page_size;
    }
    if (u < p.k_units) {
      static_cast<uint4*>(p.k_cache)[at * p.k_units + u] = reinterpret_cast<const uint4*>(p.k_new + b * p.kn_bs + node * p.kn_ts)[u];
    } else {
      u -= p.k_units;
      static_cast<uint4*>(p.v_cache)[at * p.v_units + u] = reinterpret_cast<const uint4*>(p.v_new + b * p.vn_bs + node * p.vn_ts)[u];
    }
  }
}

// ------------------------------------------------------------------------------------------------ evict: selection

constexpr int kSelThreads = 1024;
constexpr int kBins = 8192;
constexpr int kBinsPerThread = kBins / kSelThreads;
constexpr int kHeldKeys = 32768;  // keys of a CTA that stay in shared memory (128 KB beside 32 KB of bins)

struct EvictParams {
  const float* weights;      // [B, Hkv, capacity]
  const int32_t* lengths;    // [B]
  int32_t* kept;             // [B, Hkv, keep]
  int2* info;                // [B, Hkv] (new length, old length)
  int B, Hkv, capacity, keep, recent;
  // movement
  const char *k, *v;
  char *k_out, *v_out;
  float* w_out;
  int32_t* lengths_out;
  int cap_out, in_place;
  int row_k, row_v;          // bytes of a row of one head
  int slices_k, slices_v, slice_units, row_splits;
  int held_keys;             // keys of a slice that stay in shared memory
};

// Order of the weights as unsigned integers: larger is better, NaN is worst, -0 equals 0.
__device__ __forceinline__ uint32_t weight_order(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

// Inclusive sum over the CTA's threads in thread order; `total` is the sum of all.  `scratch` holds a word per warp.
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t* scratch, uint32_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // (the scratch of an earlier call has been read)
  if (lane == 31) scratch[warp] = x;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelThreads / 32; ++w) {
    const uint32_t s = scratch[w];
    before += w < warp ? s : 0u;
    all += s;
  }
  total = all;
  return x + before;
}

// A CTA per (sequence, head), or a cluster with a slice of the keys per CTA.  The weights are read once and stay in shared memory as
// integers of the same order (what lies past 32768 keys a CTA is read again).  The threshold -- the weight of rank keep - recent --
// is found digit by digit with a histogram per CTA that the cluster adds up through distributed shared memory; exact, so ties can
// be cut by index.  13 bits of the first digit hold four mantissa bits: with two, weights that span a few octaves meet
// in so few bins that the additions queue.  A last pass numbers the kept keys in order.
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictParams p) {
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
  const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  extern __shared__ uint32_t select_smem[];
  uint32_t* hist = select_smem;           // [kBins]
  uint32_t* held_keys = hist + kBins;     // the slice's first p.held_keys keys
  __shared__ uint32_t scratch[kSelThreads / 32];
  __shared__ uint32_t found[3];     // digit, the count still wanted inside it, and its keys
  __shared__ uint32_t counts[2];    // keys of this slice above the threshold, and equal to it
  const int64_t unit = (int64_t)b * p.Hkv + h;
  const float* w = p.weights + unit * p.capacity;
  int32_t* kept = p.kept + unit * p.keep;
  const int n = max(0, min(p.capacity, p.lengths[b]));
  const int held = min(n, p.keep);
  if (rank == 0 && tid == 0) p.info[unit] = make_int2(held, n);
  if (n <= p.keep) {
    for (int i = rank * kSelThreads + tid; i < p.keep; i += ranks * kSelThreads) kept[i] = i < n ? i : -1;
    return;  // (the whole cluster)
  }
  const int old = n - p.recent, want = p.keep - p.recent;
  for (int i = rank * kSelThreads + tid; i < p.recent; i += ranks * kSelThreads) kept[want + i] = old + i;
  if (want == 0) return;
  const int per = ((old + ranks - 1) / ranks + 3) / 4 * 4;
  const int begin = min(old, rank * per), end = min(old, begin + per);
  {  // eight loads in flight per thread
    const int stop = min(end, begin + p.held_keys);
    int j = begin + tid;
    for (; j + 7 * kSelThreads < stop; j += 8 * kSelThreads) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = w[j + e * kSelThreads];
#pragma unroll
      for (int e = 0; e < 8; ++e) held_keys[j + e * kSelThreads - begin] = weight_order(x[e]);
    }
    for (; j < stop; j += kSelThreads) held_keys[j - begin] = weight_order(w[j]);
  }
  auto sync = [&] {
    if (ranks == 1)
      __syncthreads();
    else
      cluster.sync();
  };
  auto key_at = [&](int j) { return j - begin < p.held_keys ? held_keys[j - begin] : weight_order(w[j]); };
  uint32_t prefix = 0, rest = (uint32_t)want;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    constexpr int kShift[3] = {19, 6, 0}, kBits[3] = {13, 13, 6};
    const int shift = kShift[pass], bits = kBits[pass];
    const uint32_t high = pass == 0 ? 0u : ~0u << (shift + bits);
    for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int j = begin + tid; j < end; j += kSelThreads) {
      const uint32_t key = key_at(j);
      if ((key & high) == prefix) atomicAdd(&hist[(key >> shift) & ((1u << bits) - 1)], 1u);
    }
    sync();
    // bins from the top: thread i takes the next kBinsPerThread below kBins - kBinsPerThread i
    uint32_t bin[kBinsPerThread] = {}, sum = 0;
    for (int r = 0; r < ranks; ++r) {
      const uint4* theirs = reinterpret_cast<const uint4*>(ranks == 1 ? hist : cluster.map_shared_rank(hist, r)) + (kSelThreads - 1 - tid) * (kBinsPerThread / 4);
#pragma unroll
      for (int v = 0; v < kBinsPerThread / 4; ++v) {
        const uint4 x = theirs[v];
        bin[kBinsPerThread - 1 - 4 * v] += x.x;
        bin[kBinsPerThread - 2 - 4 * v] += x.y;
        bin[kBinsPerThread - 3 - 4 * v] += x.z;
        bin[kBinsPerThread - 4 - 4 * v] += x.w;
      }
    }
#pragma unroll
    for (int e = 0; e < kBinsPerThread; ++e) sum += bin[e];
    uint32_t total;
    uint32_t before = block_scan(sum, scratch, total) - sum;
#pragma unroll
    for (int e = 0; e < kBinsPerThread; ++e) {
      if (before < rest && before + bin[e] >= rest) {
        found[0] = (uint32_t)(kBins - 1 - (kBinsPerThread * tid + e));
        found[1] = rest - before;
        found[2] = bin[e];
      }
      before += bin[e];
    }
    sync();  // (the histograms have been read; `found` is written)
    prefix |= found[0] << shift;
    rest = found[1];
    if (rest == found[2]) {  // the whole bin is kept: everything above its lowest value less one
      --prefix;
      rest = 0;
      break;
    }
  }
  uint32_t run_above = 0, run_equal = 0;  // keys above the threshold, and equal to it, in the slices before this one
  if (ranks > 1) {
    uint32_t above = 0, equal = 0;
    for (int j = begin + tid; j < end; j += kSelThreads) {
      const uint32_t key = key_at(j);
      above += key > prefix;
      equal += key == prefix;
    }
    uint32_t t_above, t_equal;
    block_scan(above, scratch, t_above);
    block_scan(equal, scratch, t_equal);
    if (tid == 0) {
      counts[0] = t_above;
      counts[1] = t_equal;
    }
    cluster.sync();
    for (int r = 0; r < rank; ++r) {
      run_above += cluster.map_shared_rank(counts, r)[0];
      run_equal += cluster.map_shared_rank(counts, r)[1];
    }
  }
  for (int j0 = begin; j0 < end; j0 += kSelThreads * 4) {
    uint32_t key[4], packed = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = j0 + tid * 4 + e;
      key[e] = j < end ? key_at(j) : 0u;
      if (j < end) packed += key[e] > prefix ? 0x10000u : key[e] == prefix ? 1u : 0u;
    }
    uint32_t total;
    const uint32_t upto = block_scan(packed, scratch, total) - packed;
    uint32_t a = run_above + (upto >> 16), q = run_equal + (upto & 0xffffu);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = j0 + tid * 4 + e;
      if (j >= end) break;
      if (key[e] > prefix) {
        kept[a + min(q, rest)] = j;
        ++a;
      } else if (key[e] == prefix) {
        if (q < rest) kept[a + q] = j;
        ++q;
      }
    }
    run_above += total >> 16;
    run_equal += total & 0xffffu;
  }
  sync();  // (no CTA leaves while another may read its shared memory)
}

// ------------------------------------------------------------------------------------------------ evict: movement

// One CTA moves a column slice of the rows of one (sequence, head), in order.  In place that is safe without a copy: row i comes from
// row kept[i] >= i, a chunk of rows is read before any of it is written, and what later chunks read lies behind what this one
// writes.  Slices of one row share nothing.  The last slice index moves the weights and clears those behind the kept keys.
template <typename U>
__global__ void __launch_bounds__(256) evict_move_kernel(const EvictParams p) {
  constexpr int UN = 8;
  const int h = blockIdx.y, b = blockIdx.z / p.row_splits, split = blockIdx.z % p.row_splits;
  const int64_t unit = (int64_t)b * p.Hkv + h;
  const int2 info = p.info[unit];
  const int held = info.x;
  const int32_t* kept = p.kept + unit * p.keep;
  int slice = blockIdx.x;
  const int tid = threadIdx.x;
  if (slice == p.slices_k + p.slices_v) {
    if (split) return;
    if (h == 0 && tid == 0) p.lengths_out[b] = held;
    const float* w = p.weights + unit * p.capacity;
    float* wo = p.w_out + unit * p.cap_out;
    for (int i0 = 0; i0 < held; i0 += 256 * UN) {
      float x[UN];
#pragma unroll
      for (int k = 0; k < UN; ++k) {
        const int i = i0 + k * 256 + tid;
        if (i < held) x[k] = w[kept[i]];
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < UN; ++k) {
        const int i = i0 + k * 256 + tid;
        if (i < held) wo[i] = x[k];
      }
    }
    const int clear = p.in_place ? info.y : p.cap_out;
    for (int i = held + tid; i < clear; i += 256) wo[i] = 0.f;
    return;
  }
  const bool keys = slice < p.slices_k;
  if (!keys) slice -= p.slices_k;
  const int row_units = (keys ? p.row_k : p.row_v) / (int)sizeof(U);
  const U* src = reinterpret_cast<const U*>(keys ? p.k : p.v) + ((int64_t)b * p.capacity * p.Hkv + h) * row_units;
  U* dst = reinterpret_cast<U*>(keys ? p.k_out : p.v_out) + ((int64_t)b * p.cap_out * p.Hkv + h) * row_units;
  const int64_t step = (int64_t)p.Hkv * row_units;
  const int rows = 256 / p.slice_units;
  const int u = slice * p.slice_units + tid % p.slice_units, r = tid / p.slice_units;
  const bool mine = r < rows && u < row_units;
  const int chunk = rows * UN;
  for (int i0 = split * chunk; i0 < held; i0 += p.row_splits * chunk) {
    U x[UN];
    int from[UN];
#pragma unroll
    for (int k = 0; k < UN; ++k) {
      const int i = i0 + k * rows + r;
      from[k] = mine && i < held ? kept[i] : -1;
      if (p.in_place && from[k] == i) from[k] = -1;  // a row that stays
    }
#pragma unroll
    for (int k = 0; k < UN; ++k)
      if (from[k] >= 0) x[k] = src[from[k] * step + u];
    if (p.in_place) __syncthreads();
#pragma unroll
    for (int k = 0; k < UN; ++k)
      if (from[k] >= 0) dst[(int64_t)(i0 + k * rows + r) * step + u] = x[k];
  }
}

// Whether [a, a + na) and [b, b + nb) share a byte.
bool overlap(const void* a, size_t na, const void* b, size_t nb) {
  const char *x = static_cast<const char*>(a), *y = static_cast<const char*>(b);
  return x < y + nb && y < x + na;
}

}  // namespace
}  // namespace pjx

extern "C" {

int pjx_kv_cache_accept(void* k_cache, void* v_cache, const void* k_new, int64_t k_new_batch_stride, int64_t k_new_token_stride,
                        const void* v_new, int64_t v_new_batch_stride, int64_t v_new_token_stride, const int32_t* lengths,
                        const int32_t* path, const int32_t* counts, const int32_t* block_table, int B, int N, int P, int Hkv, int D,
                        int Dv, int capacity, int page_size, int max_pages, int num_pages, int dtype, int32_t* lengths_out,
                        int32_t* overflow, void* stream) {
  using namespace pjx;
  if (dtype != PJX_F32 && dtype != PJX_BF16 && dtype != PJX_F16)
    return fail(PJX_ERR_BAD_ARG, "dtype must be float32, bfloat16 or float16 (got code %d)", dtype);
  if (B < 0 || N < 0 || P < 0 || Hkv < 1 || D < 1 || Dv < 1 || capacity < 0) return fail(PJX_ERR_BAD_ARG, "negative or zero dimension");
  if (k_new_batch_stride < 0 || k_new_token_stride < 0 || v_new_batch_stride < 0 || v_new_token_stride < 0)
    return fail(PJX_ERR_BAD_ARG, "accept: strides must be non-negative");
  if (block_table) {
    if (page_size < 1 || max_pages < 0 || num_pages < 0 || (int64_t)max_pages * page_size >= PJX_BAND_NO_UPPER)
      return fail(PJX_ERR_BAD_ARG, "accept: page_size must be positive and max_pages * page_size below 2^30");
    capacity = max_pages * page_size;
  }
  if (B == 0) return PJX_OK;
  if (!lengths || !counts || !lengths_out) return fail(PJX_ERR_BAD_ARG, "accept: null buffer");
  const bool rows_there = capacity > 0 && !(block_table && num_pages == 0);  // (an empty pool has no address)
  if (P > 0 && N > 0 && rows_there && (!k_cache || !v_cache || !k_new || !v_new || !path)) return fail(PJX_ERR_BAD_ARG, "accept: null buffer");
  if (P > 0 && !path) return fail(PJX_ERR_BAD_ARG, "accept: null buffer");
  if (B > 65535) return fail(PJX_ERR_UNSUPPORTED, "accept: batch above 65535");
  const size_t es = dtype_size(dtype);
  if ((Hkv * (size_t)D * es) % 16 || (Hkv * (size_t)Dv * es) % 16 || (k_new_batch_stride * es) % 16 || (k_new_token_stride * es) % 16 ||
      (v_new_batch_stride * es) % 16 || (v_new_token_stride * es) % 16)
    return fail(PJX_ERR_UNSUPPORTED, "accept: a token's keys and values, and the drafts' strides, must be multiples of 16 bytes");
  if ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) | reinterpret_cast<uintptr_t>(k_new) |
       reinterpret_cast<uintptr_t>(v_new)) & 15)
    return fail(PJX_ERR_UNSUPPORTED, "accept: buffers must be 16-byte aligned");
  // a cache whose values are its keys, and drafts to match: their rows are written once
  const bool one = k_cache == v_cache && k_new == v_new && D == Dv && k_new_batch_stride == v_new_batch_stride && k_new_token_stride == v_new_token_stride;
  if (P > 0 && N > 0 && rows_there) {  // (the drafts are read while the cache is written)
    const size_t rows = block_table ? (size_t)num_pages * page_size : (size_t)B * capacity;
    const size_t k_span = ((size_t)(B - 1) * k_new_batch_stride + (size_t)(N - 1) * k_new_token_stride + (size_t)Hkv * D) * es;
    const size_t v_span = ((size_t)(B - 1) * v_new_batch_stride + (size_t)(N - 1) * v_new_token_stride + (size_t)Hkv * Dv) * es;
    const size_t k_bytes = rows * Hkv * D * es, v_bytes = rows * Hkv * Dv * es;
    if (overlap(k_new, k_span, k_cache, k_bytes) || overlap(k_new, k_span, v_cache, v_bytes) || overlap(v_new, v_span, k_cache, k_bytes) ||
        overlap(v_new, v_span, v_cache, v_bytes))
      return fail(PJX_ERR_BAD_ARG, "accept: the drafts lie inside the cache that is written");
    if (!one && overlap(k_cache, k_bytes, v_cache, v_bytes))
      return fail(PJX_ERR_BAD_ARG, "accept: the caches of keys and values share memory");
  }
  AcceptParams p = {};
  p.k_cache = k_cache; p.v_cache = v_cache;
  p.k_new = static_cast<const char*>(k_new); p.v_new = static_cast<const char*>(v_new);
  p.kn_bs = k_new_batch_stride * (int64_t)es; p.kn_ts = k_new_token_stride * (int64_t)es;
  p.vn_bs = v_new_batch_stride * (int64_t)es; p.vn_ts = v_new_token_stride * (int64_t)es;
  p.lengths = lengths; p.path = path; p.counts = counts; p.block_table = block_table;
  p.lengths_out = lengths_out; p.overflow = overflow;
  p.capacity = capacity; p.N = N; p.P = P; p.page_size = page_size; p.max_pages = max_pages; p.num_pages = num_pages;
  p.k_units = (int)(Hkv * (size_t)D * es / 16); p.v_units = one ? 0 : (int)(Hkv * (size_t)Dv * es / 16);
  kv_accept_kernel<<<dim3(kAcceptCluster, B), 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
  count_launch();
  return check_cuda(cudaGetLastError(), "kv cache accept launch");
}

size_t pjx_kv_cache_evict_workspace_bytes(int B, int Hkv) { return B < 1 || Hkv < 1 ? 0 : (size_t)B * Hkv * sizeof(int2); }

int pjx_kv_cache_evict(const void* k_cache, const void* v_cache, const float* weights, const int32_t* lengths, void* k_out, void* v_out,
                       float* weights_out, int32_t* lengths_out, int32_t* kept, int B, int Hkv, int D, int Dv, int capacity,
                       int capacity_out, int keep, int recent, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace pjx;
  if (dtype != PJX_F32 && dtype != PJX_BF16 && dtype != PJX_F16)
    return fail(PJX_ERR_BAD_ARG, "dtype must be float32, bfloat16 or float16 (got code %d)", dtype);
  if (B < 0 || Hkv < 1 || D < 1 || Dv < 1 || capacity < 0 || capacity_out < 0) return fail(PJX_ERR_BAD_ARG, "negative or zero dimension");
  if (keep < 1 || recent < 0 || recent > keep) return fail(PJX_ERR_BAD_ARG, "evict: keep must be positive and recent in [0, keep] (got %d, %d)", keep, recent);
  if (capacity_out < (keep < capacity ? keep : capacity))
    return fail(PJX_ERR_BAD_ARG, "evict: the kept keys (%d) do not fit into a capacity of %d", keep < capacity ? keep : capacity, capacity_out);
  if (B == 0) return PJX_OK;
  if (!lengths || !lengths_out || !kept) return fail(PJX_ERR_BAD_ARG, "evict: null buffer");
  if ((capacity > 0 && (!k_cache || !v_cache || !weights)) || (capacity_out > 0 && (!k_out || !v_out || !weights_out)))
    return fail(PJX_ERR_BAD_ARG, "evict: null buffer");
  if (capacity >= PJX_BAND_NO_UPPER || capacity_out >= PJX_BAND_NO_UPPER || keep >= PJX_BAND_NO_UPPER)
    return fail(PJX_ERR_UNSUPPORTED, "evict: cache capacity must be below 2^30");
  if (B > 8191 || Hkv > 65535) return fail(PJX_ERR_UNSUPPORTED, "evict: at most 8191 sequences and 65535 kv heads per call (got B=%d, Hkv=%d)", B, Hkv);
  const size_t es = dtype_size(dtype);
  const size_t rows = (size_t)B * Hkv;
  const bool in_place = k_out == k_cache;
  if ((v_out == v_cache) != in_place || (weights_out == weights) != in_place || (in_place && capacity_out != capacity))
    return fail(PJX_ERR_BAD_ARG, "evict: keys, values and weights move in place together, or all into other buffers");
  const bool one = k_cache == v_cache && k_out == v_out && D == Dv;  // the values are the keys: their rows move once
  const void *from[3] = {k_cache, v_cache, weights}, *to[3] = {k_out, v_out, weights_out};
  const size_t row_bytes[3] = {D * es, Dv * es, 4};
  for (int i = 0; i < 3; ++i)
    for (int j = 0; j < 3; ++j) {
      if (!in_place && overlap(from[i], rows * capacity * row_bytes[i], to[j], rows * capacity_out * row_bytes[j]))
        return fail(PJX_ERR_BAD_ARG, "evict: source and result overlap in part");
      if (i < j && !(one && j == 1) && overlap(to[i], rows * capacity_out * row_bytes[i], to[j], rows * capacity_out * row_bytes[j]))
        return fail(PJX_ERR_BAD_ARG, "evict: keys, values and weights share memory that is written");
    }
  const size_t need = pjx_kv_cache_evict_workspace_bytes(B, Hkv);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 7))
    return fail(PJX_ERR_WORKSPACE, "evict workspace: need %zu bytes, 8-byte aligned, got %zu", need, workspace ? workspace_bytes : (size_t)0);
  EvictParams p = {};
  p.weights = weights; p.lengths = lengths; p.kept = kept;
  p.info = static_cast<int2*>(workspace);
  p.B = B; p.Hkv = Hkv; p.capacity = capacity; p.keep = keep; p.recent = recent;
  p.k = static_cast<const char*>(k_cache); p.v = static_cast<const char*>(v_cache);
  p.k_out = static_cast<char*>(k_out); p.v_out = static_cast<char*>(v_out);
  p.w_out = weights_out; p.lengths_out = lengths_out;
  p.cap_out = capacity_out; p.in_place = in_place;
  p.row_k = (int)(D * es); p.row_v = (int)(Dv * es);
  cudaStream_t st = static_cast<cudaStream_t>(stream);

  // a CTA per (sequence, head) up to 32768 keys, a cluster beyond
  int ranks = 1;
  while (ranks < 8 && capacity > ranks * kHeldKeys) ranks *= 2;
  p.held_keys = ((capacity + ranks - 1) / ranks + 3) / 4 * 4;
  if (p.held_keys > kHeldKeys) p.held_keys = kHeldKeys;
  const size_t select_smem = (size_t)(kBins + p.held_keys) * sizeof(uint32_t);
  static std::atomic<uint64_t> allowed{0};
  int rc = allow_smem(reinterpret_cast<const void*>(evict_select_kernel), (kBins + kHeldKeys) * (int)sizeof(uint32_t), allowed);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ranks, Hkv, B);
  cfg.blockDim = dim3(kSelThreads);
  cfg.dynamicSmemBytes = select_smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  rc = check_cuda(cudaLaunchKernelEx(&cfg, evict_select_kernel, p), "evict selection launch");
  count_launch();
  if (rc) return rc;

  const bool vec = p.row_k % 16 == 0 && p.row_v % 16 == 0 &&
                   ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) | reinterpret_cast<uintptr_t>(k_out) |
                     reinterpret_cast<uintptr_t>(v_out)) & 15) == 0;
  const int unit = vec ? 16 : (int)es;
  p.slice_units = 128 / unit;  // 128 bytes of a row
  p.slices_k = (p.row_k / unit + p.slice_units - 1) / p.slice_units;
  p.slices_v = one ? 0 : (p.row_v / unit + p.slice_units - 1) / p.slice_units;
  p.row_splits = 1;
  if (!in_place)  // rows move independently: enough CTAs for eight per SM, at least two chunks each
    while (p.row_splits < 8 && (int64_t)B * Hkv * (p.slices_k + p.slices_v) * p.row_splits < 148 * 8 &&
           keep > p.row_splits * 2 * (256 / p.slice_units) * 8)
      p.row_splits *= 2;
  const dim3 grid(p.slices_k + p.slices_v + 1, Hkv, B * p.row_splits);
  if (vec)
    evict_move_kernel<uint4><<<grid, 256, 0, st>>>(p);
  else if (es == 4)
    evict_move_kernel<uint32_t><<<grid, 256, 0, st>>>(p);
  else
    evict_move_kernel<uint16_t><<<grid, 256, 0, st>>>(p);
  count_launch();
  return check_cuda(cudaGetLastError(), "evict movement launch");
}

}  // extern "C"
