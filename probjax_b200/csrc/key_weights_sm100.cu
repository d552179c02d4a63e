// Attention received by every key on the tensor cores: transposed scores S^T = K.Q^T with the keys on the lanes of tensor memory, so
// that a key's sum over all query rows is one thread's: w_j += sum_r exp2(c q_r.k_j - lse2_r), no exchange between threads.
//
// With few rows the call is bound by HBM (K once); at 256 rows per KV head the exponentials (16 per clock and SM) take longer than K.
// 128 keys a step, the even and the odd steps with groups of threads and two score buffers (128 columns each) of their own, so that the
// MMAs run ahead of the exponentials; rows (t, g) in chunks of up to 128.  The log-sum-exp of a row is subtracted by the MMAs too: one
// more step of 16 columns multiplies -lse2 / c, split into three 16-bit numbers (24 bits and more), with a constant; read per column and
// thread out of shared memory, the loads took a third of the peak rate of shared-memory wavefronts.
//
//   warp 0       producer: key tiles (KST stages) and chunks of Q (QST stages) by TMA, the chunks' log-sum-exp columns
//   warp 1       MMA issuer
//   warps 2-17   four groups of 128 threads, two per parity: a key has a thread for the first 64 rows of a chunk and one for the
//                others (with one thread per key, 2.5 warps per scheduler, the kernel waits for latencies)
//
// 8 prompts of 32k keys, 8 KV heads of 128 (537 MB of keys), whole calls by CUDA events, us: 4 rows per KV head 103 (5.2 TB/s),
// 64 rows 101, 128 rows 107, 256 rows (a prompt's window under its causal mask) 197-210, 173 inside a graph, where the exponentials alone
// take 131 at 1.73 GHz.  Steps at 256 rows (the kernel in a trace, causal): a thread per key 259, two threads 224, log-sum-exps inside the
// MMAs 198, sums of the second half added a step later and short loops around the MMAs 183.  A part of the exponentials as a polynomial on
// the FMA pipe (a quarter, a third, a half) is no faster (187, 185, 209), so they are not the bound; no unit is full, and the compute warps
// wait for each load of scores before they start on it.
//
// Rows apart: a row without keys (lse = +inf) may hold anything in its query, and NaN plus -inf is NaN; a log-sum-exp whose three parts pass
// the type (fp16: |lse / scale| from 2.6 * 10^8 on) would come out as infinite.  Where a chunk has such a row, the producer leaves what to
// add to each of its rows in 32 bits (-inf: the row adds nothing, whatever its score) instead of in the MMA's columns, the issuer hands it
// to the score buffer, and the compute warps take it from there: a load from shared memory per row and key (4, 64, 128 rows with such
// rows among them: 113, 111, 146 us).  A chunk without them pays for a flag (2 us of the 103).
//
// RESIDENT: all rows fit into the stages, stay there while the CTA walks the keys of one (sequence, head), and the key steps of all heads
// are dealt in contiguous runs, one per CTA (a run may go on into the next sequence or head, whose rows it then loads; with a CTA bound to
// a head, 100 heads took 180 us instead of 134); otherwise the rows stream past every key step out of L2 and the steps are dealt in turn,
// which balances a causal mask.  Every wait is bounded as in the other tcgen05 kernels.
#include <type_traits>

#include "sm100_softmax.cuh"

namespace pjx {

int make_tmap_blhd(CUtensorMap* m, const void* base, int dtype, int B, int L, int H, int Dim, int rows);
int make_tmap_16bit(CUtensorMap* m, const void* base, int dtype, int rank, const uint64_t* dims, const uint64_t* strides, const uint32_t* box);

namespace {

using namespace sm100;

constexpr int BT = 128;          // keys of a tile, rows of a chunk
constexpr int STEP = BT;         // keys of a step
constexpr int NTHREADS = 576;


__device__ __forceinline__ void st_shared1(uint32_t addr, float x) { asm volatile("st.shared.f32 [%0], %1;\n" ::"r"(addr), "f"(x) : "memory"); }
__device__ __forceinline__ float ld_shared1(uint32_t addr) {
  float x;
  asm volatile("ld.shared.f32 %0, [%1];\n" : "=f"(x) : "r"(addr) : "memory");
  return x;
}

template <int HD>
struct Cfg {
  static constexpr int SUB = HD / 64;
  static constexpr int TILE_BYTES = SUB * BT * 128;
  static constexpr int QST = HD == 128 ? 2 : 3;
  static constexpr int KST = HD == 128 ? 4 : 6;
  static constexpr int OFF_K = 0;                              // [KST]
  static constexpr int OFF_Q = OFF_K + KST * TILE_BYTES;       // [QST]
  static constexpr int OFF_EXT = OFF_Q + QST * TILE_BYTES;     // 128 rows of 4 x 16 columns: the QST stages' log-sum-exps, then the constant
  static constexpr int OFF_SUM = OFF_EXT + BT * 128;           // [4 steps][2 parities][BT] sums of the second halves
  static constexpr int OFF_APART = OFF_SUM + 8 * BT * 4;       // [QST stages, then 4 score buffers][BT] what is added to rows apart (below)
  static constexpr int OFF_FLAG = OFF_APART + (QST + 4) * BT * 4;  // [QST + 4] whether a stage, a score buffer holds such rows
  static constexpr int OFF_BAR = OFF_FLAG + 32;
  static constexpr int N_BAR = 2 * KST + 2 * QST + 8 + 32;
  static constexpr int SMEM_BYTES = OFF_BAR + N_BAR * 8 + 16 + 1024;
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory budget");
  static_assert(QST <= 3, "the constant takes the last of the four column groups");
  static_assert((QST + 4) * 4 <= 32, "flags");
};
// -lse2 / c = 4096 a + 64 b + c': in fp16 that reaches to 2.6 * 10^8 (rows beyond are added apart) and down to 6 * 10^-8.
constexpr float kExt0 = 4096.f, kExt1 = 64.f;

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
  int n;  // steps of a run that follow on, with the same rows
};
__device__ __forceinline__ KeyStep key_step(const KeyWeightsParams& p, int per_head, int64_t pos) {
  const int lane = threadIdx.x & 31;
  KeyStep s;
  s.hk = (int)(pos / per_head);
  int at = (int)(pos - (int64_t)s.hk * per_head);
  s.b = s.len = s.k0 = 0;
  s.n = 1;
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
  constexpr int K_FULL = 0, K_EMPTY = C::KST, Q_FULL = 2 * C::KST, Q_EMPTY = Q_FULL + C::QST, S_FULL = Q_EMPTY + C::QST, S_FREE = S_FULL + 4,
                SUM = S_FREE + 4;  // [4 steps][2 parities][4 warps] the second half's sums are there
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_BAR + C::N_BAR * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const uint32_t apart = sbase + C::OFF_APART, apart_flag = sbase + C::OFF_FLAG;
  const int warp = uniform(static_cast<int>(threadIdx.x >> 5)), lane = threadIdx.x & 31;
  const int G = p.Hq / p.Hkv;
  const int per_head = key_line(p);
  const int64_t total = (int64_t)per_head * p.Hkv;
  // this CTA's steps: pos = start, start + stride, .. below stop
  const int64_t start = RESIDENT ? total * blockIdx.x / gridDim.x : blockIdx.x;
  const int64_t stop = RESIDENT ? total * (blockIdx.x + 1) / gridDim.x : total;
  // The run of steps at `pos` (one step where the rows stream).
  auto run_at = [&](int64_t pos) {
    KeyStep s = key_step(p, per_head, pos);
    if constexpr (RESIDENT) s.n = (int)min((int64_t)(s.len - s.k0 + STEP - 1) / STEP, stop - pos);
    s.b = uniform(s.b);
    s.hk = uniform(s.hk);
    s.len = uniform(s.len);
    s.k0 = uniform(s.k0);
    s.n = uniform(s.n);
    return s;
  };
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
      mbar_init(BAR(i), (i >= Q_FULL && i < Q_EMPTY) || (i >= S_FULL && i < S_FREE) ? 2u : i >= S_FREE && i < SUM ? 8u : 1u);
    for (int i = 0; i < C::QST + 4; ++i) st_shared1(apart_flag + 4 * i, 0.f);
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
    using T = std::conditional_t<BF16, __nv_bfloat16, __half>;
    auto write_ext = [&](int row, int group, uint32_t first, uint32_t second) {  // 16 columns of a 128-byte-swizzled row: three numbers
      const uint32_t at = sbase + C::OFF_EXT + row * 128;
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %3};\n" ::"r"(at + (((2 * group) ^ (row & 7)) << 4)), "r"(first), "r"(second), "r"(0) : "memory");
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n" ::"r"(at + (((2 * group + 1) ^ (row & 7)) << 4)), "r"(0) : "memory");
    };
    for (int i = lane; i < BT; i += 32) write_ext(i, 3, pack16<BF16>(kExt0, kExt1), pack16<BF16>(1.f, 0.f));  // (fenced with the first chunk)
    bool ok = true;
    int fill = 0, ks = 0, kp = 1;  // Q stages filled so far; K stage and the parity its freedom is waited with
    auto load_chunk = [&](const KeyStep& s, int c) {
      const int st = fill % C::QST;
      ok = ok && mbar_wait_all(BAR(Q_EMPTY + st), ((fill / C::QST) & 1) ^ 1, abort_flag);
      if (!ok) return;
      ++fill;
      float l[BT / 32], x[BT / 32];
      bool any = false;
#pragma unroll
      for (int k = 0; k < BT / 32; ++k) {
        const int i = lane + 32 * k, t = c * geo.tokens + i / G, h = s.hk * G + i % G;
        const bool row = i < geo.tokens * G && t < p.Lq;  // (columns past the rows are masked)
        l[k] = row ? p.lse[((int64_t)s.b * p.Hq + h) * p.Lq + t] * kLog2e : 0.f;
      }
#pragma unroll
      for (int k = 0; k < BT / 32; ++k) {
        x[k] = -l[k] / (p.sm_scale * kLog2e);
        any |= !(fabsf(Elem<T>::round(x[k] / kExt0)) < INFINITY);
      }
      any = __any_sync(0xffffffffu, any);
#pragma unroll
      for (int k = 0; k < BT / 32; ++k) {
        const int i = lane + 32 * k;
        if (any) {
          st_shared1(apart + (st * BT + i) * 4, -l[k]);
          x[k] = 0.f;
        }
        const float hi = Elem<T>::round(x[k] / kExt0), rest = fmaf(-kExt0, hi, x[k]);
        const float mid = Elem<T>::round(rest / kExt1), lo = fmaf(-kExt1, mid, rest);
        write_ext(i, st, pack16<BF16>(hi, mid), pack16<BF16>(lo, 0.f));
      }
      if (lane == 0) st_shared1(apart_flag + 4 * st, any ? 1.f : 0.f);
      fence_proxy_async();
      __syncwarp();
      if (leader) {
        mbar_arrive(BAR(Q_FULL + st));
        mbar_arrive_expect_tx(BAR(Q_FULL + st), C::SUB * (uint32_t)(geo.tokens * G) * 128u);
#pragma unroll
        for (int u = 0; u < C::SUB; ++u)
          tma_load_5d(sbase + C::OFF_Q + st * C::TILE_BYTES + u * BT * 128, &tm_q, BAR(Q_FULL + st), u * 64, 0, s.hk, c * geo.tokens, s.b);
      }
    };
    for (int64_t pos = start; ok && pos < stop;) {
      const KeyStep s = run_at(pos);
      int c0, c1;
      chunk_range(s, c0, c1);
      for (int j = 0; ok && j < s.n; ++j) {
        if (!(ok = mbar_wait_all(BAR(K_EMPTY + ks), kp, abort_flag))) break;
        if (leader) {
          mbar_arrive_expect_tx(BAR(K_FULL + ks), C::TILE_BYTES);
#pragma unroll
          for (int u = 0; u < C::SUB; ++u)
            tma_load_4d(sbase + C::OFF_K + ks * C::TILE_BYTES + u * BT * 128, &tm_k, BAR(K_FULL + ks), u * 64, s.hk, s.k0 + j * STEP, s.b);
        }
        if (++ks == C::KST) {
          ks = 0;
          kp ^= 1;
        }
        if (j == 0)
          for (int c = c0; ok && c < c1; ++c) load_chunk(s, c);
      }
      pos += RESIDENT ? s.n : stride;
    }
  } else if (warp == 1) {
    const uint32_t leader = elect_leader();
    constexpr uint32_t idesc = make_idesc(BT, BT, BF16, false, false);
    // (descriptors differ in the address field, in units of 16 bytes)
    const uint64_t k_desc = make_smem_desc(sbase + C::OFF_K, 16, 1024), q_desc = make_smem_desc(sbase + C::OFF_Q, 16, 1024);
    const uint64_t ext_desc = make_smem_desc(sbase + C::OFF_EXT, 16, 1024);
    // (Few instructions between the MMAs: this warp shares its scheduler with compute warps, and a slow step here is one for all.)
    bool ok = true;
    int used = 0, ks = 0, kp = 0, step = 0;  // Q stages used; K stage and parity; steps
    uint32_t n_s = 0x0000;                   // score tiles of either parity, mod 4: bits 0-1 and 2-3
    uint32_t odd = 0;                        // stages and (bits 4-7) score buffers with rows apart
    for (int64_t pos = start; ok && pos < stop;) {
      const KeyStep s = run_at(pos);
      int c0, c1;
      chunk_range(s, c0, c1);
      for (int j = 0; ok && j < s.n; ++j, ++step) {
        const int t = step & 1;
        if (!(ok = mbar_wait_all(BAR(K_FULL + ks), kp, abort_flag))) break;
        const uint64_t ka = k_desc + ks * (C::TILE_BYTES / 16);
        const bool last = !RESIDENT || j == s.n - 1;
        for (int c = c0; c < c1; ++c) {
          const int f = used + c - c0, st = f % C::QST;
          if (j == 0) {
            if (!(ok = mbar_wait_all(BAR(Q_FULL + st), (f / C::QST) & 1, abort_flag))) break;
            odd = (odd & ~(1u << st)) | (uniform(ld_shared1(apart_flag + 4 * st)) != 0.f ? 1u << st : 0u);
          }
          const uint32_t n = (n_s >> (2 * t)) & 3u, buf = t * 2 + (n & 1);
          if (!(ok = mbar_wait_all(BAR(S_FREE + buf), (n >> 1) ^ 1, abort_flag))) break;
          n_s = (n_s & ~(3u << (2 * t))) | (((n + 1) & 3u) << (2 * t));
          tc_fence_after();
          if (((odd >> st) | (odd >> (4 + buf))) & 1u) {  // (the buffer's readers are done with it, as with its scores)
            const bool now = (odd >> st) & 1u;
            if (now)
              for (int i = lane; i < BT; i += 32) st_shared1(apart + ((C::QST + buf) * BT + i) * 4, ld_shared1(apart + (st * BT + i) * 4));
            if (lane == 0) st_shared1(apart_flag + 4 * (C::QST + buf), now ? 1.f : 0.f);
            odd = (odd & ~(16u << buf)) | (now ? 16u << buf : 0u);
            __syncwarp();
          }
          const uint64_t qa = q_desc + st * (C::TILE_BYTES / 16);
#pragma unroll
          for (int u = 0; u < C::SUB; ++u)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_ss(tmem + buf * BT, ka + (u * BT * 128 + kk * 32) / 16, qa + (u * BT * 128 + kk * 32) / 16, idesc, (u | kk) != 0, leader);
          // (last: one more rounding at the size of the result)
          mma_ss(tmem + buf * BT, ext_desc + 3 * 2, ext_desc + st * 2, idesc, true, leader);
          mma_commit(BAR(S_FULL + buf), leader);
          if (leader) mbar_arrive(BAR(S_FULL + buf));  // (for what was written above: the commit speaks for the MMAs)
          if (last) mma_commit(BAR(Q_EMPTY + st), leader);
        }
        if (ok) mma_commit(BAR(K_EMPTY + ks), leader);
        if (++ks == C::KST) {
          ks = 0;
          kp ^= 1;
        }
      }
      used += c1 - c0;
      pos += RESIDENT ? s.n : stride;
    }
  } else {
    const int t = ((warp - 2) >> 2) & 1, half = (warp - 2) >> 3;
    const int key_in = (warp & 3) * 32 + lane;  // tensor-memory lane
    const uint32_t lane_sel = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const float c1 = p.sm_scale * kLog2e;
    const float2 cc = make_float2(c1, c1);
    if (p.weights_in != p.weights_out) {  // behind the valid keys: what was there
      const int tid = threadIdx.x - 64;
      for (int64_t row = blockIdx.x; row < (int64_t)p.B * p.Hkv; row += gridDim.x) {
        const int len = key_len(p, (int)(row / p.Hkv));
        for (int j = len + tid; j < p.Lkv; j += NTHREADS - 64) p.weights_out[row * p.Lkv + j] = p.weights_in ? p.weights_in[row * p.Lkv + j] : 0.f;
      }
    }
    // The first half's thread adds the second's sum one step later, when it has long been there.
    float* sums = reinterpret_cast<float*>(smem + C::OFF_SUM) + t * BT + key_in;
    auto sum_bar = [&](int m) { return BAR(SUM + ((m & 3) * 2 + t) * 4 + (warp & 3)); };
    float held_part = 0.f;
    float* held_out = nullptr;  // where the sum of the step before goes
    const float* held_in = nullptr;
    bool ok = true, holds = false;
    auto finish = [&](int m) {
      ok = ok && mbar_wait(sum_bar(m), (m >> 2) & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (ok && held_out) *held_out = (held_in ? *held_in : 0.f) + (held_part + sums[(m & 3) * 2 * BT]);
    };
    int step = 0, n_s = 0, mine = 0;  // steps, score tiles and steps of this parity
    for (int64_t pos = start; ok && pos < stop;) {
      const KeyStep s = run_at(pos);
      int c_first, c_last;
      chunk_range(s, c_first, c_last);
      const int64_t row = ((int64_t)s.b * p.Hkv + s.hk) * p.Lkv;
      float* out = p.weights_out + row;
      const float* in = p.weights_in ? p.weights_in + row : nullptr;
      const int open_from = p.Lq - 1 + p.band_lo, open_to = p.band_hi;  // keys that every row sees
      const int first = (step & 1) == t ? 0 : 1;                        // this parity's steps of the run
      step += s.n;
      pos += RESIDENT ? s.n : stride;
      for (int j = first; ok && j < s.n; j += 2) {
        const int k0 = s.k0 + j * STEP, key = k0 + key_in;
        const bool all = k0 + BT <= s.len && k0 >= open_from && k0 + BT - 1 <= open_to;  // every row sees every key of the step
        float2 sum[4] = {};
        for (int c = c_first; ok && c < c_last; ++c, ++n_s) {
          const int buf = t * 2 + (n_s & 1);
          ok = mbar_wait(BAR(S_FULL + buf), (n_s >> 1) & 1, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          const int t0 = c * geo.tokens, cols = min(geo.tokens, p.Lq - t0) * G;
          int lo = 0, hi = cols;  // rows of the chunk that see this key
          if (!all) {
            const int64_t a = ((int64_t)key - p.band_hi - t0) * G, e = ((int64_t)key - p.band_lo - t0 + 1) * G;
            lo = (int)max((int64_t)0, min((int64_t)cols, a));
            hi = key < s.len ? (int)max((int64_t)0, min((int64_t)cols, e)) : 0;
          }
          const uint32_t s_addr = tmem + lane_sel + buf * BT;
          const int end = min((cols + 31) / 32, 2 * half + 2);
          for (int c32 = 2 * half; c32 < end; ++c32) {
            float x[32];
            tmem_ld32f(s_addr + c32 * 32, x);
            const bool has_apart = ld_shared1(apart_flag + 4 * (C::QST + buf)) != 0.f;
            tmem_wait_ld();
            if (has_apart) {
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const float add = ld_shared1(apart + ((C::QST + buf) * BT + c32 * 32 + i) * 4);
                x[i] = add == -INFINITY ? -INFINITY : fmaf(x[i], c1, add);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float2 a = __fmul2_rn(make_float2(x[2 * i], x[2 * i + 1]), cc);
                x[2 * i] = a.x; x[2 * i + 1] = a.y;
              }
            }
            if (!all || c32 * 32 + 32 > cols) {  // (columns past the rows hold anything)
#pragma unroll
              for (int i = 0; i < 32; ++i) x[i] = c32 * 32 + i >= lo && c32 * 32 + i < hi ? x[i] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 v = make_float2(x[2 * i], x[2 * i + 1]);
              sum[i & 3] = __fadd2_rn(sum[i & 3], make_float2(ex2_approx(x[2 * i]), ex2_approx(x[2 * i + 1])));
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(BAR(S_FREE + buf));  // (an arrival per warp: 256 on one word took as long as the MMAs)
        }
        const float2 s01 = __fadd2_rn(sum[0], sum[1]), s23 = __fadd2_rn(sum[2], sum[3]);
        const float part = (s01.x + s01.y) + (s23.x + s23.y);
        if (c_first == c_last) {  // no row sees a key of the step
          if (half == 0 && key < s.len) out[key] = in ? in[key] : 0.f;
          continue;
        }
        if (half == 1) {
          sums[(mine & 3) * 2 * BT] = part;
          __syncwarp();
          if (lane == 0) mbar_arrive(sum_bar(mine));
        } else {
          if (holds) finish(mine - 1);
          held_part = part;
          held_out = key < s.len ? out + key : nullptr;
          held_in = in ? in + key : nullptr;
          holds = true;
        }
        ++mine;
      }
    }
    if (half == 0 && holds && ok) finish(mine - 1);
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
  static std::atomic<uint64_t> allowed[2] = {};
  if ((rc = allow_smem(reinterpret_cast<const void*>(kern), C::SMEM_BYTES, allowed[resident]))) return rc;
  kern<<<148, NTHREADS, C::SMEM_BYTES, stream>>>(tk, tq, p, geo);
  count_launch();
  return check_cuda(cudaGetLastError(), "key weights launch");
}

}  // namespace

bool key_weights_sm100_supported(const KeyWeightsParams& p, int dtype) {
  if (dtype != PJX_BF16 && dtype != PJX_F16) return false;
  if (p.D != 64 && p.D != 128) return false;
  if (p.Hq / p.Hkv > BT || p.Lq < 1) return false;
  if (!(fabsf(p.sm_scale) >= 1e-4f && fabsf(p.sm_scale) <= 1e4f)) return false;  // (-lse2 / c stays in range)
  return ((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k)) & 15) == 0;
}

int launch_key_weights_sm100(const KeyWeightsParams& p, int dtype, cudaStream_t stream) {
  if (dtype == PJX_BF16) return p.D == 128 ? launch_t<128, true>(p, dtype, stream) : launch_t<64, true>(p, dtype, stream);
  return p.D == 128 ? launch_t<128, false>(p, dtype, stream) : launch_t<64, false>(p, dtype, stream);
}

}  // namespace pjx
