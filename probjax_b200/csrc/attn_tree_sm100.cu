// Tree attention on the tensor cores: up to 128 query rows (t, g) of a KV head's group per tile, the keys of a split streamed
// through shared memory by TMA, both products as tcgen05 MMAs with accumulators in tensor memory.
//
//   o_i = sum_j softmax_j(sm_scale q_i . k_j) v_j over the cached prefix and i's ancestors among the drafts
//
// With few rows the call is bound by HBM (every K and V byte once); 256 rows per KV head do as much arithmetic per byte as the
// tensor cores can take.  One CTA per SM:
//
//   warp 0       TMA producer: the Q tile(s), then a K ring and a V ring of 128-key tiles; pages are fetched in boxes that never
//                straddle one
//   warp 1       MMA issuer: S = Q.K^T, O += P.V with P read from tensor memory
//   warps 2-5, 6-9   two softmax groups, one thread per row
//   warp 10      clears the values of keys that nobody sees (behind the prefix, absent drafts): 0 x NaN is not 0
//
// One row tile (ROWS = 1): the groups take the even and the odd key tiles, each with a running (max, sum, O) of its own, so that
// one group's softmax runs beside the other's MMAs; they are merged at the end.  Two row tiles (ROWS = 2): a group per row tile, and
// both use every key tile.  A draft's ancestors are found by walking the parents, only in the (at most two) tiles that hold
// drafts: 128 keep bits per row and tile.
//
// A CTA's run of the work (tree_plan.cuh) is a few segments, each a stretch of one sequence's keys; barriers and rings run on
// through all of them, and since the output leaves through the Q tile's shared memory, the next segment's keys are
// fetched meanwhile.
//
// Every barrier wait is bounded: on expiry the role raises the CTA's abort flag, all roles drain, tensor memory is freed and the
// status word gets PJX_ERR_DEVICE_TIMEOUT.
//
// Measured over the whole call with CUDA events (bf16, 16 sequences of 16384 keys, 8 KV heads of 128, 1.07 GB of K and V, us): 4 rows
// per KV head 192 (5.6 TB/s), 32 rows 197, 64 rows 201 (5.3), 128 rows 241 (4.5), 256 rows 345 (3.1).  In a profiler's trace the kernel
// without the combine takes 190, 191, 193, 199 and 262; the rest is the combine, and at 256 rows, where calls follow one another
// without a pause, clocks under the power cap (1.46 GHz seen).  At 256 rows the chain softmax -> P.V -> next scores of the two row tiles
// bounds the kernel.  Pages: at 4 rows 128 and 64 cost nothing, 16 costs 19 % (a tile is eight loads); at 64 rows 3, 8 and 32 %.  Head
// width 64, half the bytes: 177 (3.0 TB/s), 166, 291 at 4, 64, 256 rows: a key tile takes half the time to load but the same chain.
// Equal runs of the work on 148 CTAs against 592 splits (16 ragged sequences of 1k-32k keys in pages of 128, 256 rows, whole call): 371
// against 426; masked tiles in a copy of the code of their own and one barrier arrival per warp instead of one per thread: 322 -> 280
// in the trace.
#include <type_traits>

#include "sm100_softmax.cuh"
#include "tree_plan.cuh"

namespace pjx {

int make_tmap_blhd(CUtensorMap* m, const void* base, int dtype, int B, int L, int H, int Dim, int rows);
int make_tmap_16bit(CUtensorMap* m, const void* base, int dtype, int rank, const uint64_t* dims, const uint64_t* strides, const uint32_t* box);

namespace {

using namespace sm100;

constexpr int BN = kTreeTile;
constexpr int NTHREADS = 352;

__device__ __forceinline__ void st_shared4(uint32_t addr, float a, float b, float c, float d) {
  asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};\n" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}
__device__ __forceinline__ float4 ld_shared4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

template <int HD, int ROWS>
struct Cfg {
  static constexpr int SUB = HD / 64;
  static constexpr int TILE_BYTES = SUB * 128 * 128;  // 128 rows of Q, K or V
  static constexpr int KST = HD == 128 ? (ROWS == 1 ? 3 : 2) : 6;
  static constexpr int VST = HD == 128 ? 3 : 6;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + ROWS * TILE_BYTES;
  static constexpr int OFF_V = OFF_K + KST * TILE_BYTES;
  static constexpr int OFF_ML = OFF_V + VST * TILE_BYTES;  // (max, sum) of the second group's rows
  static constexpr int OFF_WORK = OFF_ML + 128 * 8;        // the softmax warps' segments
  static constexpr int OFF_LINE = OFF_WORK + 8 * 64;       // this CTA's run
  static constexpr int OFF_BAR = OFF_LINE + 64;
  static constexpr int N_BAR = 2 + 2 * KST + 2 * VST + 2 + 2 + 2 + 1 + 2;
  static constexpr int SMEM_BYTES = OFF_BAR + N_BAR * 8 + 16 + 1024;  // + alignment slack
  static constexpr int TMEM_COLS = 512;
  static_assert(2 * BN + 2 * HD <= TMEM_COLS, "tensor memory has 512 columns");
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory budget");
};

struct TreeGeometry {
  int tokens;    // query tokens of a row tile
  int box_rows;  // keys per TMA box of the cache
};

template <int HD, bool BF16, int ROWS>
__global__ void __launch_bounds__(NTHREADS, 1)
attn_tree_sm100_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_kn,
                       const __grid_constant__ CUtensorMap tm_vn, const TreeParams p, const TreeGeometry geo) {
  using C = Cfg<HD, ROWS>;
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_unaligned) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = uniform(smem_u32(smem));
  auto BAR = [&](int i) { return sbase + C::OFF_BAR + 8u * i; };
  constexpr int Q_FULL = 0, Q_FREE = 1;  // Q_FREE: the output staged over Q has left
  constexpr int K_FULL = 2, K_EMPTY = K_FULL + C::KST;
  constexpr int V_FULL = K_EMPTY + C::KST, V_EMPTY = V_FULL + C::VST;
  constexpr int S_FULL = V_EMPTY + C::VST;  // [2]
  constexpr int P_FULL = S_FULL + 2;        // [2]
  constexpr int V_LANDED = P_FULL + 2;      // a tile that may hold keys nobody sees is there
  constexpr int V_CLEAN = V_LANDED + 1;     // their values are cleared
  constexpr int O_DONE = V_CLEAN + 1;
  constexpr int MEET = O_DONE + 1;          // [2] the softmax threads that stage a tile meet here (bounded, unlike a named barrier)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_BAR + C::N_BAR * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = uniform(static_cast<int>(threadIdx.x >> 5)), lane = threadIdx.x & 31;
  const TreeLine line = tree_line(p);
  // The combine may be resident early; it waits for this grid.
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  if ((int)blockIdx.x >= line.ctas) return;
  const int64_t start = tree_run(line, blockIdx.x);
  // (in shared memory, not in registers: it is looked at once a segment)
  struct Run {
    int64_t stop, length;
    int tiles, ctas;
  };
  volatile Run* run = reinterpret_cast<volatile Run*>(smem + C::OFF_LINE);
  if (threadIdx.x == 0) {
    run->stop = tree_run(line, blockIdx.x + 1);
    run->length = line.length;
    run->tiles = line.tiles;
    run->ctas = line.ctas;
  }
  // What the roles need of a segment; every warp walks the same segments.
  struct Work {
    int b, hk, t0, first, n, prefix, prefix_tiles, clean0;
    int64_t slot, pair;
    bool last;
  };
  auto next = [&](int64_t& pos, Work& w) {
    const int64_t stop = run->stop;
    if (pos >= stop) return false;
    TreeLine l;
    l.tiles = run->tiles;
    l.length = run->length;
    l.ctas = run->ctas;
    const TreeSegment sg = tree_segment(p, l, blockIdx.x, pos, stop);
    const int row_tiles = p.columns / p.Hkv;
    w.b = uniform(sg.b);
    w.prefix = uniform(sg.prefix);
    w.first = uniform(sg.first);
    w.n = uniform(sg.end - sg.first);
    w.slot = sg.slot;
    w.pair = sg.pair;
    w.last = sg.last;
    w.hk = uniform(sg.column / row_tiles);
    w.t0 = uniform((sg.column - w.hk * row_tiles) * ROWS * geo.tokens);
    w.prefix_tiles = (w.prefix + BN - 1) / BN;
    w.clean0 = max(0, w.prefix / BN - w.first);  // first tile of the segment that may hold a key nobody sees
    pos += w.n;
    return true;
  };

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::N_BAR; ++i)
      mbar_init(BAR(i), i == Q_FREE ? 8u : i >= P_FULL && i < P_FULL + 2 ? 4u : i >= MEET ? (ROWS == 1 ? 8u : 4u) : 1u);  // (an arrival per warp)
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(tmem_slot), C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    // (converged: every lane runs the loop, one issues)
    const uint32_t leader = elect_leader();
    if (leader) {
      prefetch_tmap(&tm_q);
      prefetch_tmap(&tm_k);
      prefetch_tmap(&tm_v);
    }
    const int boxes = BN / geo.box_rows;  // per tile: 1, 2, 4 or 8
    int g = 0, seg = 0;                   // tiles loaded so far, segments
    bool ok = true;
    Work w = {};
    auto load_q = [&] {
      ok = mbar_wait_all(BAR(Q_FREE), (seg & 1) ^ 1, abort_flag);
      if (!ok || !leader) return;
      mbar_arrive_expect_tx(BAR(Q_FULL), ROWS * C::SUB * (uint32_t)(geo.tokens * (p.Hq / p.Hkv)) * 128u);
#pragma unroll
      for (int t = 0; t < ROWS; ++t)
#pragma unroll
        for (int s = 0; s < C::SUB; ++s)
          tma_load_5d(sbase + C::OFF_Q + t * C::TILE_BYTES + s * 128 * 128, &tm_q, BAR(Q_FULL), s * 64, 0, w.hk, w.t0 + t * geo.tokens, w.b);
    };
    for (int64_t pos = start; ok && next(pos, w); ++seg) {
      // The first key tiles of a later segment are fetched before its queries, whose place is still in use.
      const int ahead = seg == 0 ? 0 : min(w.n, min(C::KST, C::VST));
      for (int j = 0; ok && j < w.n; ++j, ++g) {
        if (j == ahead) load_q();
        const int tile = w.first + j;
        const bool drafts = tile >= w.prefix_tiles;
        const int key0 = tile * BN;
        int page_row = p.num_pages * p.page_size;  // lane i: pool row of box i of the tile; past the pool: zeros
        if (p.block_table && !drafts) {
          const int key = key0 + lane * geo.box_rows;
          if (lane < boxes && key < w.prefix) {
            const int page = p.block_table[(int64_t)w.b * p.max_pages + key / p.page_size];
            if (page >= 0 && page < p.num_pages) page_row = page * p.page_size + key % p.page_size;
          }
        }
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          constexpr int ST[2] = {C::KST, C::VST}, OFF[2] = {C::OFF_K, C::OFF_V}, FULL[2] = {K_FULL, V_FULL}, EMPTY[2] = {K_EMPTY, V_EMPTY};
          const int st = g % ST[kv];
          ok = ok && mbar_wait_all(BAR(EMPTY[kv] + st), ((g / ST[kv]) & 1) ^ 1, abort_flag);
          if (!ok) break;
          const uint32_t bar = BAR(FULL[kv] + st), dst = sbase + OFF[kv] + st * C::TILE_BYTES;
          if (leader) mbar_arrive_expect_tx(bar, C::TILE_BYTES);
          if (drafts) {
            if (leader) {
#pragma unroll
              for (int s = 0; s < C::SUB; ++s)
                tma_load_4d(dst + s * 128 * 128, kv ? &tm_vn : &tm_kn, bar, s * 64, w.hk, (tile - w.prefix_tiles) * BN, w.b);
            }
          } else if (!p.block_table) {
            if (leader) {
#pragma unroll
              for (int s = 0; s < C::SUB; ++s) tma_load_4d(dst + s * 128 * 128, kv ? &tm_v : &tm_k, bar, s * 64, w.hk, key0, w.b);
            }
          } else {
            for (int i = 0; i < boxes; ++i) {
              const int row = __shfl_sync(0xffffffffu, page_row, i);
              if (leader) {
#pragma unroll
                for (int s = 0; s < C::SUB; ++s)
                  tma_load_4d(dst + s * 128 * 128 + i * geo.box_rows * 128, kv ? &tm_v : &tm_k, bar, s * 64, w.hk, row, 0);
              }
            }
          }
        }
      }
      if (ok && ahead == w.n) load_q();  // (a short segment: its keys went first)
    }
  } else if (warp == 1) {
    // -------------------------------------------------------------- MMA issuer
    const uint32_t leader = elect_leader();
    constexpr uint32_t idesc_s = make_idesc(128, BN, BF16, false, false);
    constexpr uint32_t idesc_o = make_idesc(128, HD, BF16, false, true);
    // (descriptors differ in the address field, in units of 16 bytes)
    const uint64_t q_desc = make_smem_desc(sbase + C::OFF_Q, 16, 1024), k_desc = make_smem_desc(sbase + C::OFF_K, 16, 1024);
    const uint64_t v_desc = make_smem_desc(sbase + C::OFF_V, 128 * 128, 1024);
    int ks = 0, kp = 0, vs = 0, vp = 0;  // the next K and V tiles' stages, and the parities their arrival is waited with
    int seg = 0, cleaned = 0;            // segments, tiles handed to the clearing warp
    int p_done[2] = {0, 0};              // P tiles of each group so far
    bool ok = true;
    Work w = {};
    auto issue_s = [&](int t) {  // scores of the next K tile into buffer t
      const uint64_t qa = q_desc + (ROWS == 2 ? t : 0) * (C::TILE_BYTES / 16), ka = k_desc + ks * (C::TILE_BYTES / 16);
#pragma unroll
      for (int s = 0; s < C::SUB; ++s)
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_ss(tmem + t * BN, qa + (s * 128 * 128 + kk * 32) / 16, ka + (s * 128 * 128 + kk * 32) / 16, idesc_s, (s | kk) != 0, leader);
      mma_commit(BAR(S_FULL + t), leader);
    };
    auto issue_pv = [&](int t, bool fresh) {
      const uint64_t va = v_desc + vs * (C::TILE_BYTES / 16);
#pragma unroll
      for (int kk = 0; kk < BN / 16; ++kk)
        mma_ts(tmem + 2 * BN + t * HD, tmem + t * BN + kk * 8, va + kk * 2048 / 16, idesc_o, !fresh || kk != 0, leader);
    };
    auto wait_k = [&] {
      const bool there = mbar_wait_all(BAR(K_FULL + ks), kp, abort_flag);
      tc_fence_after();
      return there;
    };
    auto free_k = [&] {
      mma_commit(BAR(K_EMPTY + ks), leader);
      if (++ks == C::KST) {
        ks = 0;
        kp ^= 1;
      }
    };
    auto wait_v = [&](int j) {
      bool there = mbar_wait_all(BAR(V_FULL + vs), vp, abort_flag);
      if (there && j >= w.clean0) {
        if (leader) mbar_arrive(BAR(V_LANDED));
        there = mbar_wait_all(BAR(V_CLEAN), cleaned++ & 1, abort_flag);
      }
      return there;
    };
    auto free_v = [&] {
      mma_commit(BAR(V_EMPTY + vs), leader);
      if (++vs == C::VST) {
        vs = 0;
        vp ^= 1;
      }
    };
    auto wait_p = [&](int t) {
      const bool there = mbar_wait_all(BAR(P_FULL + t), (t ? p_done[1]++ : p_done[0]++) & 1, abort_flag);
      tc_fence_after();
      return there;
    };
    for (int64_t pos = start; ok && next(pos, w); ++seg) {
      const int n = w.n;
      ok = mbar_wait_all(BAR(Q_FULL), seg & 1, abort_flag);
      if constexpr (ROWS == 1) {
        for (int j = 0; ok && j < min(2, n); ++j) {
          if (!(ok = wait_k())) break;
          issue_s(j);
          free_k();
        }
        for (int j = 0; ok && j < n; ++j) {
          const int t = j & 1;
          if (!(ok = wait_v(j) && wait_p(t))) break;
          issue_pv(t, j < 2);
          free_v();
          if (j + 2 < n) {
            if (!(ok = wait_k())) break;
            issue_s(t);
            free_k();
          }
        }
      } else {
        if (ok && (ok = wait_k())) {
          issue_s(0);
          issue_s(1);
          free_k();
        }
        for (int j = 0; ok && j < n; ++j) {
          const bool more = j + 1 < n;
          if (!(ok = wait_v(j) && (!more || wait_k()))) break;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!(ok = ok && wait_p(t))) break;
            issue_pv(t, j == 0);
            if (more) issue_s(t);
          }
          if (!ok) break;
          free_v();
          if (more) free_k();
        }
      }
      if (ok) mma_commit(BAR(O_DONE), leader);
    }
  } else if (warp == 10) {
    // ------------------------------------------- values of keys that nobody sees
    // (told by the issuer, which follows the V ring; the two take turns)
    int g = 0, cleaned = 0;
    bool ok = true;
    Work w = {};
    for (int64_t pos = start; ok && next(pos, w); g += w.n) {
      const int32_t* parents = p.parents + w.b * p.parents_bs;
      if (w.first == 0 && w.pair < p.B)  // (once for every sequence, for the combine)
        for (int i = lane; i < p.N; i += 32) p.present[(int64_t)w.b * p.N + i] = tree_present(parents, i);
      for (int j = w.clean0; ok && j < w.n; ++j, ++cleaned) {
        const int tile = w.first + j, st = (g + j) % C::VST;
        ok = mbar_wait_all(BAR(V_LANDED), cleaned & 1, abort_flag);
        if (!ok) break;
        bool wrote = false;
        for (int r = lane; r < BN; r += 32) {
          const int node = (tile - w.prefix_tiles) * BN + r;  // (drafts past the last one arrive as zeros)
          const bool seen = tile < w.prefix_tiles ? tile * BN + r < w.prefix : node >= p.N || tree_present(parents, node);
          if (seen) continue;
          wrote = true;
          const uint32_t row = sbase + C::OFF_V + st * C::TILE_BYTES + r * 128;
#pragma unroll
          for (int s = 0; s < C::SUB; ++s)
#pragma unroll
            for (int u = 0; u < 8; ++u)
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n" ::"r"(row + s * 128 * 128 + u * 16), "r"(0) : "memory");
        }
        if (wrote) fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(BAR(V_CLEAN));
      }
    }
  } else {
    // ------------------------------------------------------------ softmax warps
    const int t = (warp - 2) >> 2;
    const int quarter = warp & 3;  // tensor-memory lane quarter this warp may access
    const int r_in = quarter * 32 + lane;
    const uint32_t lane_sel = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem + lane_sel + t * BN;
    const uint32_t o_addr = tmem + lane_sel + 2 * BN + t * HD;
    const float c1 = p.sm_scale * kLog2e;
    constexpr int STEP = ROWS == 1 ? 2 : 1;
    // The segment lives in shared memory: the registers hold the scores of a row and little else.
    struct Held {
      int b, t0, first, prefix, prefix_tiles, last;
      int64_t slot, pos, pair;
    };
    static_assert(sizeof(Held) <= 64, "a warp's slot");
    volatile Held* held = reinterpret_cast<volatile Held*>(smem + C::OFF_WORK + (warp - 2) * 64);
    int it = 0, seg = 0, met = 0;  // score tiles of this group so far, segments, meetings
    bool ok = true;
    auto meet = [&] {
      const uint32_t bar = BAR(MEET + (ROWS == 1 ? 0 : t));
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
      const bool there = mbar_wait(bar, met++ & 1, abort_flag);
      ok = __all_sync(0xffffffffu, there) && ok;
    };
    auto next_held = [&](int& n, int& clean0) {
      Work w;
      int64_t pos = seg == 0 ? start : held->pos;
      if (!next(pos, w)) return false;
      __syncwarp();
      if (lane == 0) {
        held->b = w.b;
        held->t0 = w.t0;
        held->first = w.first;
        held->prefix = w.prefix;
        held->prefix_tiles = w.prefix_tiles;
        held->slot = w.slot;
        held->pair = w.pair;
        held->last = w.last;
        held->pos = pos;
      }
      __syncwarp();
      n = w.n;
      clean0 = w.clean0;
      return true;
    };
    int n, clean0;
    for (; ok && next_held(n, clean0); ++seg) {
      float m_ref = -INFINITY, l = 0.f;
      // One score tile; the few tiles that hold keys not everybody sees have a copy of the code of their own.
      auto score_tile = [&](int j, auto masked) {
        ok = mbar_wait(BAR(S_FULL + t), it & 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        tc_fence_after();
        float s[BN];
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) tmem_ld32f(s_addr + c * 32, &s[c * 32]);
        tmem_wait_ld();
        if constexpr (decltype(masked)::value) {  // keep bits of the tile's 128 keys
          const int tile = held->first + j;
          uint32_t bits[4];
          if (tile < held->prefix_tiles) {
            const int valid = held->prefix - tile * BN;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int k = valid - 32 * c;
              bits[c] = k >= 32 ? 0xffffffffu : k <= 0 ? 0u : (1u << k) - 1u;
            }
          } else {
            const int node0 = (tile - held->prefix_tiles) * BN;
            const int32_t* parents = p.parents + held->b * p.parents_bs;
            uint32_t b0 = 0, b1 = 0, b2 = 0, b3 = 0;
            const int G = p.Hq / p.Hkv;
            const int node = held->t0 + (ROWS == 2 ? t * geo.tokens : 0) + r_in / G;
            int i = r_in < geo.tokens * G && node < p.N ? node : -1;
            while (i >= 0) {
              const int k = i - node0;
              const uint32_t bit = 1u << (k & 31);
              b0 |= k >= 0 && k < 32 ? bit : 0u;
              b1 |= k >= 32 && k < 64 ? bit : 0u;
              b2 |= k >= 64 && k < 96 ? bit : 0u;
              b3 |= k >= 96 && k < 128 ? bit : 0u;
              i = tree_parent(parents, i);
            }
            if (i != -1) b0 = b1 = b2 = b3 = 0;  // absent: sees nothing (and the combine drops its row)
            bits[0] = b0; bits[1] = b1; bits[2] = b2; bits[3] = b3;
          }
#pragma unroll
          for (int i = 0; i < BN; ++i) s[i] = (bits[i / 32] >> (i % 32)) & 1u ? s[i] : -INFINITY;
        }
        float mx;
        {
          float m[8];  // independent chains
#pragma unroll
          for (int i = 0; i < 8; ++i) m[i] = fmaxf(s[2 * i], s[2 * i + 1]);
#pragma unroll
          for (int i = 1; i < BN / 16; ++i)
#pragma unroll
            for (int u = 0; u < 8; ++u) m[u] = fmax3(m[u], s[16 * i + 2 * u], s[16 * i + 2 * u + 1]);
          mx = fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), fmaxf(fmaxf(m[4], m[5]), fmaxf(m[6], m[7])));
        }
        mx *= c1;  // c1 > 0
        // lazy running maximum: advance only when it grew by more than 8 (base 2)
        const bool need = (mx > m_ref + 8.f) || (m_ref == -INFINITY && mx > -INFINITY);
        const bool rescale = __any_sync(0xffffffffu, need);
        float corr = 1.f;
        if (rescale) {
          const float m_new = fmaxf(m_ref, mx);
          corr = (m_new == -INFINITY) ? 1.f : exp2f(m_ref - m_new);
          m_ref = m_new;
          l *= corr;
        }
        const float neg_m = (m_ref == -INFINITY) ? 0.f : -m_ref;
        float2 sum0 = make_float2(0.f, 0.f), sum1 = make_float2(0.f, 0.f);
        exp_pack_store<BN, BF16>(s, make_float2(c1, c1), make_float2(neg_m, neg_m), sum0, sum1, s_addr);
        const float lsum = (sum0.x + sum0.y) + (sum1.x + sum1.y);
        // the group's previous P.V completed before these scores became visible
        if (rescale && j >= STEP) {
#pragma unroll
          for (int c = 0; c < HD / 32; ++c) {
            float o[32];
            tmem_ld32f(o_addr + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= corr;
            tmem_st32f(o_addr + c * 32, o);
          }
        }
        l += lsum;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(BAR(P_FULL + t));
      };
      int j = ROWS == 1 ? t : 0;
      for (; ok && j < min(n, clean0); j += STEP, ++it) score_tile(j, std::false_type{});
      for (; ok && j < n; j += STEP, ++it) score_tile(j, std::true_type{});
      const bool any = ROWS == 2 || n > t;  // this group has accumulated a tile of the segment
      ok = ok && mbar_wait(BAR(O_DONE), seg & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      if (warp == 2 && lane == 0) {  // the combine's list: first and last slot of the (sequence, column)
        if (held->first == 0) p.slots[2 * held->pair] = (int)held->slot;
        if (held->last) p.slots[2 * held->pair + 1] = (int)held->slot;
      }
      // All products of the segment are done and Q is dead.  The rows leave through Q's shared memory, half a row (HD / 2 floats) at a
      // time, 16-byte units swizzled by row, so that whole lines are written; the rings go on loading.
      constexpr int HALF = HD / 2, UNITS = HALF / 4;
      const int G = p.Hq / p.Hkv, tile_rows = geo.tokens * G;
      const int token0 = held->t0 + (ROWS == 2 ? t * geo.tokens : 0);
      const int n_rows = min(geo.tokens, p.N - token0) * G;  // rows of the tile that exist (may be none)
      const int64_t part = held->slot * p.column_rows + (ROWS == 2 ? t * tile_rows : 0);
      const uint32_t stage = sbase + C::OFF_Q + (ROWS == 2 ? t : 0) * C::TILE_BYTES;
      const uint32_t my_row = stage + r_in * (HALF * 4);
      const bool writer = ROWS == 2 || t == 0;
      float* ml = reinterpret_cast<float*>(smem + C::OFF_ML);
      if (ROWS == 1 && t == 1) {  // the odd tiles' state
        ml[2 * r_in] = m_ref;
        ml[2 * r_in + 1] = l;
      }
      float wa = 1.f, wb = 0.f, inv = 0.f;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if constexpr (ROWS == 1) {
          if (t == 1 && any && ok) {
#pragma unroll
            for (int c = 0; c < HALF / 32; ++c) {
              float o[32];
              tmem_ld32f(o_addr + half * HALF + c * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 8; ++i)
                st_shared4(my_row + (((c * 8 + i) ^ (r_in & 7)) << 4), o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            }
          }
          meet();
        }
        if (writer && ok) {
          if (half == 0) {
            float m = m_ref, lsum = l;
            if constexpr (ROWS == 1) {
              const float m1 = ml[2 * r_in], l1 = ml[2 * r_in + 1];
              m = fmaxf(m_ref, m1);
              wa = m_ref == -INFINITY ? 0.f : exp2f(m_ref - m);
              wb = m1 == -INFINITY ? 0.f : exp2f(m1 - m);
              lsum = l * wa + l1 * wb;
            }
            inv = lsum != 0.f ? 1.f / lsum : 0.f;  // (NaN stays NaN)
            if (r_in < n_rows) p.lse_part[part + r_in] = lsum != 0.f ? m + log2f(lsum) : -INFINITY;
          }
#pragma unroll
          for (int c = 0; c < HALF / 32; ++c) {
            float o[32];
            tmem_ld32f(o_addr + half * HALF + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint32_t at = my_row + (((c * 8 + i) ^ (r_in & 7)) << 4);
              float4 v = make_float4(o[4 * i] * wa, o[4 * i + 1] * wa, o[4 * i + 2] * wa, o[4 * i + 3] * wa);
              if (ROWS == 1 && wb != 0.f) {
                const float4 u = ld_shared4(at);
                v = make_float4(fmaf(u.x, wb, v.x), fmaf(u.y, wb, v.y), fmaf(u.z, wb, v.z), fmaf(u.w, wb, v.w));
              }
              st_shared4(at, v.x * inv, v.y * inv, v.z * inv, v.w * inv);
            }
          }
        }
        meet();
        if (ok) {
          constexpr int THREADS = ROWS == 1 ? 256 : 128;
          const int tid = (ROWS == 1 ? t * 128 : 0) + r_in;
          float* out = p.o_part + part * HD + half * HALF;
          for (int i = tid; i < n_rows * UNITS; i += THREADS) {
            const int r = i / UNITS, u = i % UNITS;
            *reinterpret_cast<float4*>(out + (int64_t)r * HD + u * 4) = ld_shared4(stage + r * (HALF * 4) + ((u ^ (r & 7)) << 4));
          }
        }
        if (half == 0) meet();  // (the second half goes where the first one lay)
      }
      fence_proxy_async();  // the queries of the next segment are written here by TMA
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(BAR(Q_FREE));
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tmem_dealloc(tmem, C::TMEM_COLS);
    if (lane == 0 && *abort_flag && p.status) atomicExch(p.status, (int)PJX_ERR_DEVICE_TIMEOUT);
  }
}

// Query tokens of a row tile.
int tree_tokens(const TreeParams& p) {
  const int most = 128 / (p.Hq / p.Hkv);
  return most < p.N ? most : p.N;
}

template <int HD, bool BF16, int ROWS>
int launch_t(const TreeParams& p, int dtype, cudaStream_t stream) {
  using C = Cfg<HD, ROWS>;
  const int G = p.Hq / p.Hkv;
  TreeGeometry geo;
  geo.tokens = tree_tokens(p);
  geo.box_rows = BN;
  while (p.block_table && p.page_size % geo.box_rows) geo.box_rows /= 2;
  int rc = bind_context();
  if (rc) return rc;
  CUtensorMap tq, tk, tv, tkn, tvn;
  // (the stride of a dimension of one entry means nothing, but has to be one)
  auto token = [&](int64_t s, int heads) { return (uint64_t)(p.N > 1 ? s : (int64_t)heads * HD) * 2; };
  auto sequence = [&](int64_t s, int heads) { return (uint64_t)(p.B > 1 ? s : (int64_t)p.N * heads * HD) * 2; };
  {
    const uint64_t dims[5] = {(uint64_t)HD, (uint64_t)G, (uint64_t)p.Hkv, (uint64_t)p.N, (uint64_t)p.B};
    const uint64_t strides[4] = {(uint64_t)HD * 2, (uint64_t)G * HD * 2, token(p.q_ts, p.Hq), sequence(p.q_bs, p.Hq)};
    const uint32_t box[5] = {64, (uint32_t)G, 1, (uint32_t)geo.tokens, 1};
    if ((rc = make_tmap_16bit(&tq, p.q, dtype, 5, dims, strides, box))) return rc;
  }
  for (int kv = 0; kv < 2; ++kv) {
    const uint64_t dims[4] = {(uint64_t)HD, (uint64_t)p.Hkv, (uint64_t)p.N, (uint64_t)p.B};
    const uint64_t strides[3] = {(uint64_t)HD * 2, token(kv ? p.vn_ts : p.kn_ts, p.Hkv), sequence(kv ? p.vn_bs : p.kn_bs, p.Hkv)};
    const uint32_t box[4] = {64, 1, BN, 1};
    if ((rc = make_tmap_16bit(kv ? &tvn : &tkn, kv ? p.v_new : p.k_new, dtype, 4, dims, strides, box))) return rc;
    const void* base = kv ? p.v : p.k;
    CUtensorMap* m = kv ? &tv : &tk;
    const int rows = p.block_table ? p.num_pages * p.page_size : p.capacity;
    if (rows == 0)
      *m = kv ? tvn : tkn;  // no cache: never used
    else if ((rc = make_tmap_blhd(m, base, dtype, p.block_table ? 1 : p.B, rows, p.Hkv, HD, geo.box_rows)))
      return rc;
  }
  auto kern = attn_tree_sm100_kernel<HD, BF16, ROWS>;
  static std::atomic<uint64_t> allowed{0};
  if ((rc = allow_smem(reinterpret_cast<const void*>(kern), C::SMEM_BYTES, allowed))) return rc;
  kern<<<p.ctas, NTHREADS, C::SMEM_BYTES, stream>>>(tq, tk, tv, tkn, tvn, p, geo);
  count_launch();
  return check_cuda(cudaGetLastError(), "tree attention launch");
}

template <int HD, bool BF16>
int launch_rows(const TreeParams& p, int dtype, cudaStream_t stream) {
  return p.N > tree_tokens(p) ? launch_t<HD, BF16, 2>(p, dtype, stream) : launch_t<HD, BF16, 1>(p, dtype, stream);
}

}  // namespace

bool tree_sm100_supported(const TreeParams& p, int dtype, const char** why) {
  const char* w = nullptr;
  const int64_t units = p.q_bs | p.q_ts | p.kn_bs | p.kn_ts | p.vn_bs | p.vn_ts;
  if (dtype != PJX_BF16 && dtype != PJX_F16) w = "dtype must be bf16 or fp16";
  else if (p.D != p.Dv || (p.D != 64 && p.D != 128)) w = "head widths must be (64, 64) or (128, 128)";
  else if (p.Hq / p.Hkv > 128) w = "at most 128 query heads a KV head";
  else if (!(p.sm_scale > 0.f)) w = "sm_scale must be positive";
  else if (units % 8) w = "strides must be whole 16 bytes";
  else if ((p.B > 1 && (p.q_bs == 0 || p.kn_bs == 0 || p.vn_bs == 0)) || (p.N > 1 && (p.q_ts == 0 || p.kn_ts == 0 || p.vn_ts == 0)))
    w = "rows must not share memory";
  else if ((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) |
            reinterpret_cast<uintptr_t>(p.k_new) | reinterpret_cast<uintptr_t>(p.v_new)) & 15)
    w = "addresses must be 16-byte aligned";
  else if (p.block_table && (p.num_pages == 0 || (int64_t)p.num_pages * p.page_size >= 0x7fffffff)) w = "a pool of 1 to 2^31 - 2 rows";
  if (why) *why = w;
  return w == nullptr;
}

void tree_sm100_geometry(TreeParams& p) {
  const int tokens = tree_tokens(p), rows = p.N > tokens ? 2 : 1;
  p.column_rows = rows * tokens * (p.Hq / p.Hkv);
  p.columns = p.Hkv * ((p.N + rows * tokens - 1) / (rows * tokens));
  p.ctas = 148;  // one CTA per SM
}

int launch_tree_sm100(const TreeParams& p, int dtype, cudaStream_t stream) {
  if (dtype == PJX_BF16) return p.D == 128 ? launch_rows<128, true>(p, dtype, stream) : launch_rows<64, true>(p, dtype, stream);
  return p.D == 128 ? launch_rows<128, false>(p, dtype, stream) : launch_rows<64, false>(p, dtype, stream);
}

}  // namespace pjx
