// Attention received by every key on the tensor cores: transposed scores S^T = K.Q^T with the keys on the lanes of tensor memory, so
// that a key's sum over all query rows is one thread's: w_j += sum_r exp2(c q_r.k_j - lse2_r), no exchange between threads.
//
// With few rows the call is bound by HBM (K once), from some 160 rows per KV head on by the exponentials (16 per clock and SM).
// 256 keys a step, as two 128-key tiles with a group of 128 threads each; rows (t, g) in chunks of up to 128; every chunk of
// scores is double-buffered in tensor memory (2 tiles x 2 x 128 columns), so the MMAs run ahead of the exponentials.
//
//   warp 0       TMA producer: pairs of key tiles (two stages), chunks of Q and their log-sum-exps (QST stages)
//   warp 1       MMA issuer
//   warps 2-5, 6-9   the two groups: one thread per key
//
// RESIDENT: all rows fit into the stages, stay there while the CTA walks the keys of one (sequence, head), and the key steps are dealt
// in contiguous runs; otherwise the rows stream past every key step out of L2 and the steps are dealt in turn, which balances a
// causal mask.  Every wait is bounded as in the other tcgen05 kernels.
#include "sm100_softmax.cuh"

namespace pjx {

int make_tmap_blhd(CUtensorMap* m, const void* base, int dtype, int B, int L, int H, int Dim, int rows);
int make_tmap_16bit(CUtensorMap* m, const void* base, int dtype, int rank, const uint64_t* dims, const uint64_t* strides, const uint32_t* box);

namespace {

using namespace sm100;

constexpr int BT = 128;          // keys of a tile, rows of a chunk
constexpr int STEP = 2 * BT;     // keys of a step
constexpr int NTHREADS = 320;

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1, int c2, int c3, int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5, %6, %7}], [%2];\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}

template <int HD>
struct Cfg {
  static constexpr int SUB = HD / 64;
  static constexpr int TILE_BYTES = SUB * BT * 128;
  static constexpr int QST = HD == 128 ? 3 : 6;
  static constexpr int OFF_K = 0;                              // [2 stages][2 tiles]
  static constexpr int OFF_Q = OFF_K + 4 * TILE_BYTES;         // [QST]
  static constexpr int OFF_LSE = OFF_Q + QST * TILE_BYTES;     // [QST][BT] minus the base-2 log-sum-exp
  static constexpr int OFF_BAR = OFF_LSE + QST * BT * 4;
  static constexpr int N_BAR = 4 + 2 * QST + 8;
  static constexpr int SMEM_BYTES = OFF_BAR + N_BAR * 8 + 16 + 1024;
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory budget");
};

struct KeyGeometry {
  int tokens;  // query tokens of a chunk
  int chunks;  // chunks of all rows
};

// Key steps of the batch as a line: for every KV head those of all sequences, ceil(valid keys / STEP) each.
__device__ __forceinline__ int key_len(const KeyWeightsParams& p, int b) {
  return p.kv_lengths ? max(0, min(p.Lkv, p.kv_lengths[b])) : p.Lkv;
}
__device__ __forceinline__ int key_line(const KeyWeightsParams& p) {
  int sum = 0;
  for (int b = threadIdx.x & 31; b < p.B; b += 32) sum += (key_len(p, b) + STEP - 1) / STEP;
  return __reduce_add_sync(0xffffffffu, sum);
}
struct KeyStep {
  int b, hk, len, k0;
};
__device__ __forceinline__ KeyStep key_step(const KeyWeightsParams& p, int per_head, int64_t pos) {
  const int lane = threadIdx.x & 31;
  KeyStep s;
  s.hk = (int)(pos / per_head);
  int at = (int)(pos - (int64_t)s.hk * per_head);
  s.b = s.len = s.k0 = 0;
  for (int base = 0; base < p.B; base += 32) {
    const int len = base + lane < p.B ? key_len(p, base + lane) : 0;
    const int steps = (len + STEP - 1) / STEP;
    int incl = steps;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    const unsigned past = __ballot_sync(0xffffffffu, at < incl);
    if (past) {
      const int src = __ffs(past) - 1;
      s.b = base + src;
      s.len = __shfl_sync(0xffffffffu, len, src);
      s.k0 = (at - (__shfl_sync(0xffffffffu, incl, src) - __shfl_sync(0xffffffffu, steps, src))) * STEP;
      break;
    }
    at -= __shfl_sync(0xffffffffu, incl, 31);
  }
  return s;
}

template <int HD, bool BF16, bool RESIDENT>
__global__ void __launch_bounds__(NTHREADS, 1)
key_weights_sm100_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_q, const KeyWeightsParams p,
                         const KeyGeometry geo) {
  using C = Cfg<HD>;
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_unaligned) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = uniform(smem_u32(smem));
  auto BAR = [&](int i) { return sbase + C::OFF_BAR + 8u * i; };
  constexpr int K_FULL = 0, K_EMPTY = 2, Q_FULL = 4, Q_EMPTY = Q_FULL + C::QST, S_FULL = Q_EMPTY + C::QST, S_FREE = S_FULL + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_BAR + C::N_BAR * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* lse_s = reinterpret_cast<float*>(smem + C::OFF_LSE);
  const int warp = uniform(static_cast<int>(threadIdx.x >> 5)), lane = threadIdx.x & 31;
  const int G = p.Hq / p.Hkv;
  const int per_head = key_line(p);
  const int64_t total = (int64_t)per_head * p.Hkv;
  // this CTA's steps: pos = start, start + stride, .. below stop
  const int64_t start = RESIDENT ? total * blockIdx.x / gridDim.x : blockIdx.x;
  const int64_t stop = RESIDENT ? total * (blockIdx.x + 1) / gridDim.x : total;
  const int64_t stride = RESIDENT ? 1 : gridDim.x;
  // chunks whose tokens see a key of the step
  auto chunk_range = [&](const KeyStep& s, int& c0, int& c1) {
    const int t_first = (int)max((int64_t)0, (int64_t)s.k0 - p.band_hi);
    const int t_last = (int)min((int64_t)p.Lq, (int64_t)min(s.k0 + STEP, s.len) - p.band_lo);  // (one past)
    c0 = min(t_first, p.Lq) / geo.tokens;
    c1 = t_last > t_first ? (t_last + geo.tokens - 1) / geo.tokens : c0;
    if constexpr (RESIDENT) {  // all chunks, so that the stages stay what they are
      c0 = 0;
      c1 = geo.chunks;
    }
  };

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::N_BAR; ++i)
      mbar_init(BAR(i), i >= Q_FULL && i < Q_EMPTY ? 33u : i >= Q_EMPTY && i < S_FULL ? 257u : i >= S_FREE ? 128u : 1u);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);

  if (warp == 0) {
    const uint32_t leader = elect_leader();
    if (leader) {
      prefetch_tmap(&tm_k);
      prefetch_tmap(&tm_q);
    }
    bool ok = true;
    int step = 0, fill = 0, held_b = -1, held_hk = -1;  // steps, Q stages filled so far, whose rows they hold
    auto load_chunk = [&](const KeyStep& s, int c) {
      const int st = fill % C::QST;
      ok = ok && mbar_wait_all(BAR(Q_EMPTY + st), ((fill / C::QST) & 1) ^ 1, abort_flag);
      if (!ok) return;
      ++fill;
      for (int i = lane; i < BT; i += 32) {
        const int t = c * geo.tokens + i / G, h = s.hk * G + i % G;
        float l = INFINITY;  // rows that are not there, and rows without keys, add nothing
        if (i < geo.tokens * G && t < p.Lq) l = p.lse[((int64_t)s.b * p.Hq + h) * p.Lq + t] * kLog2e;
        lse_s[st * BT + i] = -l;
      }
      mbar_arrive(BAR(Q_FULL + st));
      if (leader) {
        mbar_arrive_expect_tx(BAR(Q_FULL + st), C::SUB * (uint32_t)(geo.tokens * G) * 128u);
#pragma unroll
        for (int u = 0; u < C::SUB; ++u)
          tma_load_5d(sbase + C::OFF_Q + st * C::TILE_BYTES + u * BT * 128, &tm_q, BAR(Q_FULL + st), u * 64, 0, s.hk, c * geo.tokens, s.b);
      }
    };
    for (int64_t pos = start; ok && pos < stop; pos += stride, ++step) {
      const KeyStep s = key_step(p, per_head, pos);
      const int ks = step & 1;
      ok = mbar_wait_all(BAR(K_EMPTY + ks), ((step >> 1) & 1) ^ 1, abort_flag);
      if (!ok) break;
      if (leader) {
        mbar_arrive_expect_tx(BAR(K_FULL + ks), 2 * C::TILE_BYTES);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int u = 0; u < C::SUB; ++u)
            tma_load_4d(sbase + C::OFF_K + (ks * 2 + t) * C::TILE_BYTES + u * BT * 128, &tm_k, BAR(K_FULL + ks), u * 64, s.hk, s.k0 + t * BT, s.b);
      }
      int c0, c1;
      chunk_range(s, c0, c1);
      if (RESIDENT && s.b == held_b && s.hk == held_hk) continue;
      for (int c = c0; ok && c < c1; ++c) load_chunk(s, c);
      held_b = s.b;
      held_hk = s.hk;
    }
  } else if (warp == 1) {
    const uint32_t leader = elect_leader();
    constexpr uint32_t idesc = make_idesc(BT, BT, BF16, false, false);
    bool ok = true;
    int step = 0, used = 0, base = 0, n_s = 0, held_b = -1, held_hk = -1;  // Q stages used, the first of the resident ones, score tiles
    for (int64_t pos = start; ok && pos < stop; pos += stride, ++step) {
      const KeyStep s = key_step(p, per_head, pos);
      int c0, c1;
      chunk_range(s, c0, c1);
      const bool fresh = !RESIDENT || s.b != held_b || s.hk != held_hk;
      const KeyStep after = RESIDENT && pos + 1 < stop ? key_step(p, per_head, pos + 1) : s;
      const bool last = RESIDENT && pos + 1 < stop && (after.b != s.b || after.hk != s.hk);  // the rows are done with this step
      held_b = s.b;
      held_hk = s.hk;
      if (RESIDENT && fresh) {
        base = used;
        used += geo.chunks;
      }
      ok = mbar_wait_all(BAR(K_FULL + (step & 1)), (step >> 1) & 1, abort_flag);
      for (int c = c0; ok && c < c1; ++c, ++n_s) {
        const int f = RESIDENT ? base + c : used++;
        const int st = f % C::QST;
        if (fresh) ok = mbar_wait_all(BAR(Q_FULL + st), (f / C::QST) & 1, abort_flag);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int buf = t * 2 + (n_s & 1);
          ok = ok && mbar_wait_all(BAR(S_FREE + buf), ((n_s >> 1) & 1) ^ 1, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint32_t ka = sbase + C::OFF_K + ((step & 1) * 2 + t) * C::TILE_BYTES, qa = sbase + C::OFF_Q + st * C::TILE_BYTES;
#pragma unroll
          for (int u = 0; u < C::SUB; ++u)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_ss(tmem + buf * BT, make_smem_desc(ka + u * BT * 128 + kk * 32, 16, 1024),
                     make_smem_desc(qa + u * BT * 128 + kk * 32, 16, 1024), idesc, (u | kk) != 0, leader);
          mma_commit(BAR(S_FULL + buf), leader);
        }
        if (ok && (!RESIDENT || last)) mma_commit(BAR(Q_EMPTY + st), leader);
      }
      if (ok) mma_commit(BAR(K_EMPTY + (step & 1)), leader);
    }
  } else {
    const int t = (warp - 2) >> 2;
    const int key_in = (warp & 3) * 32 + lane;  // tensor-memory lane
    const uint32_t lane_sel = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const float c1 = p.sm_scale * kLog2e;
    const float2 cc = make_float2(c1, c1);
    if (p.weights_in != p.weights_out) {  // behind the valid keys: what was there
      const int tid = threadIdx.x - 64;
      for (int64_t row = blockIdx.x; row < (int64_t)p.B * p.Hkv; row += gridDim.x) {
        const int len = key_len(p, (int)(row / p.Hkv));
        for (int j = len + tid; j < p.Lkv; j += 256) p.weights_out[row * p.Lkv + j] = p.weights_in ? p.weights_in[row * p.Lkv + j] : 0.f;
      }
    }
    bool ok = true;
    int step = 0, used = 0, base = 0, n_s = 0, held_b = -1, held_hk = -1;
    for (int64_t pos = start; ok && pos < stop; pos += stride, ++step) {
      const KeyStep s = key_step(p, per_head, pos);
      int c_first, c_last;
      chunk_range(s, c_first, c_last);
      const bool fresh = !RESIDENT || s.b != held_b || s.hk != held_hk;
      const KeyStep after = RESIDENT && pos + 1 < stop ? key_step(p, per_head, pos + 1) : s;
      const bool last = RESIDENT && pos + 1 < stop && (after.b != s.b || after.hk != s.hk);
      held_b = s.b;
      held_hk = s.hk;
      if (RESIDENT && fresh) {
        base = used;
        used += geo.chunks;
      }
      const int first_key = s.k0 + t * BT, key = first_key + key_in;
      float2 sum0 = make_float2(0.f, 0.f), sum1 = make_float2(0.f, 0.f);
      for (int c = c_first; ok && c < c_last; ++c, ++n_s) {
        const int f = RESIDENT ? base + c : used++;
        const int st = f % C::QST, buf = t * 2 + (n_s & 1);
        if (fresh) ok = mbar_wait(BAR(Q_FULL + st), (f / C::QST) & 1, abort_flag);
        ok = ok && mbar_wait(BAR(S_FULL + buf), (n_s >> 1) & 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const int t0 = c * geo.tokens, toks = min(geo.tokens, p.Lq - t0);
        const int cols = toks * G;
        // rows of the chunk that see this key: [lo, hi)
        int lo = 0, hi = cols;
        const bool whole = first_key + BT <= s.len && first_key >= (int64_t)t0 + toks - 1 + p.band_lo && first_key + BT - 1 <= (int64_t)t0 + p.band_hi;
        if (!whole) {
          const int64_t a = ((int64_t)key - p.band_hi - t0) * G, e = ((int64_t)key - p.band_lo - t0 + 1) * G;
          lo = (int)max((int64_t)0, min((int64_t)cols, a));
          hi = key < s.len ? (int)max((int64_t)0, min((int64_t)cols, e)) : 0;
        }
        const float4* nl = reinterpret_cast<const float4*>(lse_s + st * BT);
        for (int c32 = 0; c32 * 32 < cols; ++c32) {
          float x[32];
          tmem_ld32f(tmem + lane_sel + buf * BT + c32 * 32, x);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float4 l4 = nl[c32 * 8 + i];
            const float2 a = __ffma2_rn(make_float2(x[4 * i], x[4 * i + 1]), cc, make_float2(l4.x, l4.y));
            const float2 e = __ffma2_rn(make_float2(x[4 * i + 2], x[4 * i + 3]), cc, make_float2(l4.z, l4.w));
            x[4 * i] = a.x; x[4 * i + 1] = a.y; x[4 * i + 2] = e.x; x[4 * i + 3] = e.y;
          }
          if (!whole || c32 * 32 + 32 > cols) {  // (columns past the rows hold anything)
#pragma unroll
            for (int i = 0; i < 32; ++i) x[i] = c32 * 32 + i >= lo && c32 * 32 + i < hi ? x[i] : -INFINITY;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            sum0 = __fadd2_rn(sum0, make_float2(ex2_approx(x[4 * i]), ex2_approx(x[4 * i + 1])));
            sum1 = __fadd2_rn(sum1, make_float2(ex2_approx(x[4 * i + 2]), ex2_approx(x[4 * i + 3])));
          }
        }
        tc_fence_before();
        mbar_arrive(BAR(S_FREE + buf));
        if (!RESIDENT || last) mbar_arrive(BAR(Q_EMPTY + st));
      }
      if (ok && key < s.len) {
        const int64_t at = ((int64_t)s.b * p.Hkv + s.hk) * p.Lkv + key;
        p.weights_out[at] = (p.weights_in ? p.weights_in[at] : 0.f) + ((sum0.x + sum0.y) + (sum1.x + sum1.y));
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tmem_dealloc(tmem, 512);
    if (lane == 0 && *abort_flag && p.status) atomicExch(p.status, (int)PJX_ERR_DEVICE_TIMEOUT);
  }
}

template <int HD, bool BF16>
int launch_t(const KeyWeightsParams& p, int dtype, cudaStream_t stream) {
  using C = Cfg<HD>;
  const int G = p.Hq / p.Hkv;
  KeyGeometry geo;
  geo.tokens = BT / G < p.Lq ? BT / G : p.Lq;
  geo.chunks = (p.Lq + geo.tokens - 1) / geo.tokens;
  CUtensorMap tk, tq;
  int rc;
  if ((rc = make_tmap_blhd(&tk, p.k, dtype, p.B, p.Lkv, p.Hkv, HD, BT))) return rc;
  const uint64_t dims[5] = {(uint64_t)HD, (uint64_t)G, (uint64_t)p.Hkv, (uint64_t)p.Lq, (uint64_t)p.B};
  const uint64_t strides[4] = {(uint64_t)HD * 2, (uint64_t)G * HD * 2, (uint64_t)p.Hq * HD * 2, (uint64_t)p.Lq * p.Hq * HD * 2};
  const uint32_t box[5] = {64, (uint32_t)G, 1, (uint32_t)geo.tokens, 1};
  if ((rc = make_tmap_16bit(&tq, p.q, dtype, 5, dims, strides, box))) return rc;
  const bool resident = geo.chunks <= C::QST;
  auto kern = resident ? key_weights_sm100_kernel<HD, BF16, true> : key_weights_sm100_kernel<HD, BF16, false>;
  if ((rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES), "cudaFuncSetAttribute(key weights)")))
    return rc;
  kern<<<148, NTHREADS, C::SMEM_BYTES, stream>>>(tk, tq, p, geo);
  count_launch();
  return check_cuda(cudaGetLastError(), "key weights launch");
}

}  // namespace

bool key_weights_sm100_supported(const KeyWeightsParams& p, int dtype) {
  if (dtype != PJX_BF16 && dtype != PJX_F16) return false;
  if (p.D != 64 && p.D != 128) return false;
  if (p.Hq / p.Hkv > BT || p.Lq < 1) return false;
  return ((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k)) & 15) == 0;
}

int launch_key_weights_sm100(const KeyWeightsParams& p, int dtype, cudaStream_t stream) {
  if (dtype == PJX_BF16) return p.D == 128 ? launch_t<128, true>(p, dtype, stream) : launch_t<64, true>(p, dtype, stream);
  return p.D == 128 ? launch_t<128, false>(p, dtype, stream) : launch_t<64, false>(p, dtype, stream);
}

}  // namespace pjx
