// Rotary position embedding with several axes (time, height, width of video or image tokens) and a position of its own for
// every token of every sequence: pair (a, b) of a head vector becomes (a cos - b sin, b cos + a sin) of the angle
// positions[b, t, axis(pair)] * frequency(pair).  The gradient is the rotation by the negative angle, the same kernel.
//
// The floor is HBM's: the tensor is read once and written once, 16 bytes per access.  A CTA takes a few tokens.  Its threads issue
// their first loads, compute the tokens' cosines and sines meanwhile, one angle each, into shared memory, and the H heads of
// the tokens share them.  The angle is taken in turns in 64 bits (a position of 10^6 times a frequency near 1 would lose five digits in 32)
// and reduced to half a turn before it is rounded: two 64-bit operations per (token, pair), nothing next to the traffic.
//
// It is not reached (4.6 of 6.55 TB/s): a CTA loads once, forms its angles, synchronises and stores, with nothing of further tokens in flight.
//
// Measured: 4 x 4096 tokens of 32 heads of 128 in bf16, three axes, queries out of a fused projection: 58 us = 4.6 TB/s (65 with the
// loads behind the angles and a 64-bit division per access; 64 and 61 with 128 and 512 angles a CTA), the kernel in a trace; forward and
// gradient by events 118-120.  Four loads in flight instead of eight and six CTAs an SM: 55 here, but 14 against 11 in fp32 with halves.
#include <math.h>
#include <string.h>

#include "pjx_common.cuh"

namespace pjx {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 256;
constexpr int kTableAngles = 256;  // angles of one CTA (more only if one token has more pairs)
constexpr int kMaxAxes = 8;

struct RopeAxesTable {
  double turns[kMaxPairs];  // frequency of a pair over 2 pi
  uint8_t axis[kMaxPairs];
};

struct RopeAxesParams {
  const void* x;
  void* y;
  const void* positions;
  int64_t x_bs, x_ts;  // strides of a sequence and of a token of x in elements; heads are dense, y is dense
  int64_t pos_bs;      // entries between sequences of positions (0: shared)
  int64_t tokens;      // B * T
  int T, H, D, axes, pairs, pos_type, inverse, tokens_per_cta;
  uint32_t inv_heads;  // ceil(2^32 / H): the token of a head vector by a multiplication (H > 1; at most 2^16 vectors a CTA)
};

__device__ __forceinline__ double load_position(const RopeAxesParams& p, int64_t at) {
  if (p.pos_type == PJX_POS_F32) return (double)static_cast<const float*>(p.positions)[at];
  if (p.pos_type == PJX_POS_I32) return (double)static_cast<const int32_t*>(p.positions)[at];
  return (double)static_cast<const int64_t*>(p.positions)[at];
}

template <typename T>
__device__ __forceinline__ void rotate(T& a, T& b, float2 cs) {
  const float fa = Elem<T>::to_f(a), fb = Elem<T>::to_f(b);
  a = Elem<T>::from_f(fa * cs.x - fb * cs.y);
  b = Elem<T>::from_f(fb * cs.x + fa * cs.y);
}

// HALVES: pair i is (x[i], x[pairs + i]); otherwise (x[2i], x[2i + 1]).  VEC: 16-byte accesses.  x and y may be one buffer
// (a thread reads both elements of its pairs before it writes them).
template <typename T, bool HALVES, bool VEC>
__global__ void __launch_bounds__(kThreads) rope_axes_kernel(const RopeAxesParams p, const __grid_constant__ RopeAxesTable table) {
  extern __shared__ float2 cs[];  // [tokens of the CTA][pairs]
  __shared__ int64_t from[kTableAngles];  // where the tokens lie in x
  const int64_t n0 = (int64_t)blockIdx.x * p.tokens_per_cta;
  const int n_tok = (int)min((int64_t)p.tokens_per_cta, p.tokens - n0);
  const T* x = static_cast<const T*>(p.x);
  T* y = static_cast<T*>(p.y);
  const int vectors = n_tok * p.H;  // head vectors of the CTA
  for (int i = threadIdx.x; i < n_tok; i += kThreads) {
    const int64_t b = (n0 + i) / p.T;
    from[i] = b * p.x_bs + (n0 + i - b * p.T) * p.x_ts;
  }
  __syncthreads();
  auto token_of = [&](int v) { return (int)__umulhi((unsigned)v, p.inv_heads) + (p.H == 1 ? v : 0); };
  auto angles = [&] {
    for (int i = threadIdx.x; i < n_tok * p.pairs; i += kThreads) {
      const int tok = i / p.pairs, pair = i - tok * p.pairs;
      const int64_t n = n0 + tok, b = n / p.T, t = n - b * p.T;
      const double turns = load_position(p, b * p.pos_bs + t * p.axes + table.axis[pair]) * table.turns[pair];
      float s, c;
      sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
      cs[i] = make_float2(c, p.inverse ? -s : s);
    }
    __syncthreads();
  };
  if constexpr (VEC) {
    constexpr int V = 16 / sizeof(T);
    // units of a head vector: HALVES V pairs each (two accesses) and then the columns that do not rotate
    const int pair_units = HALVES ? p.pairs / V : 0;
    const int units = HALVES ? pair_units + (p.D - 2 * p.pairs) / V : p.D / V;
    const int rows = kThreads / units;
    const int u = threadIdx.x % units, row = threadIdx.x / units;
    const bool active = row < rows;
    const bool two = HALVES && u < pair_units;
    const int d0 = HALVES ? (two ? u * V : 2 * p.pairs + (u - pair_units) * V) : u * V;
    constexpr int UN = HALVES ? 4 : 8;
    uint4 lo[UN], hi[HALVES ? UN : 1];
    auto load = [&](int v0) {
#pragma unroll
      for (int k = 0; k < UN; ++k) {
        const int v = v0 + k * rows;
        if (!active || v >= vectors) break;
        const int tok = token_of(v);
        const T* src = x + from[tok] + (int64_t)(v - tok * p.H) * p.D + d0;
        lo[k] = *reinterpret_cast<const uint4*>(src);
        if (two) hi[k] = *reinterpret_cast<const uint4*>(src + p.pairs);
      }
    };
    load(row);
    angles();
    for (int v0 = row; active && v0 < vectors; v0 += UN * rows) {
      if (v0 != row) load(v0);
#pragma unroll
      for (int k = 0; k < UN; ++k) {
        const int v = v0 + k * rows;
        if (v >= vectors) break;
        T* dst = y + (n0 * p.H + v) * (int64_t)p.D + d0;
        const float2* c = cs + token_of(v) * p.pairs;
        T* a = reinterpret_cast<T*>(&lo[k]);
        if (two) {
          T* b = reinterpret_cast<T*>(&hi[k]);
#pragma unroll
          for (int e = 0; e < V; ++e) rotate(a[e], b[e], c[d0 + e]);
          *reinterpret_cast<uint4*>(dst + p.pairs) = hi[k];
        } else if (!HALVES) {
#pragma unroll
          for (int e = 0; e < V / 2; ++e)
            if (d0 / 2 + e < p.pairs) rotate(a[2 * e], a[2 * e + 1], c[d0 / 2 + e]);
        }
        *reinterpret_cast<uint4*>(dst) = lo[k];
      }
    }
  } else {
    angles();
    const int items = p.pairs + (p.D - 2 * p.pairs);  // pairs, then single columns
    for (int64_t i = threadIdx.x; i < (int64_t)vectors * items; i += kThreads) {
      const int v = (int)(i / items), it = (int)(i - (int64_t)v * items);
      const int tok = v / p.H, h = v - tok * p.H;
      const T* src = x + from[tok] + (int64_t)h * p.D;
      T* dst = y + (n0 * p.H + v) * (int64_t)p.D;
      if (it < p.pairs) {
        const int ia = HALVES ? it : 2 * it, ib = HALVES ? p.pairs + it : 2 * it + 1;
        T a = src[ia], bb = src[ib];
        rotate(a, bb, cs[tok * p.pairs + it]);
        dst[ia] = a;
        dst[ib] = bb;
      } else {
        dst[p.pairs + it] = src[p.pairs + it];
      }
    }
  }
}

template <typename T>
int launch_rope_axes(const RopeAxesParams& p, const RopeAxesTable& table, bool halves, bool vec, cudaStream_t stream) {
  const int64_t ctas = (p.tokens + p.tokens_per_cta - 1) / p.tokens_per_cta;
  if (ctas > 0x7fffffffLL) return fail(PJX_ERR_UNSUPPORTED, "rope: tensor too large for one launch");
  const size_t smem = (size_t)p.tokens_per_cta * p.pairs * sizeof(float2);
  auto kern = halves ? (vec ? rope_axes_kernel<T, true, true> : rope_axes_kernel<T, true, false>)
                     : (vec ? rope_axes_kernel<T, false, true> : rope_axes_kernel<T, false, false>);
  kern<<<(unsigned)ctas, kThreads, smem, stream>>>(p, table);
  count_launch();
  return check_cuda(cudaGetLastError(), "rope launch");
}

}  // namespace
}  // namespace pjx

extern "C" int pjx_rope_axes(const void* x, int64_t x_batch_stride, int64_t x_token_stride, void* y, const void* positions,
                             int position_type, int64_t position_batch_stride, int axes, const int32_t* sections, int B, int T,
                             int H, int D, int shared, int interleaved, int inverse, float base, int dtype, void* stream) {
  using namespace pjx;
  if (dtype != PJX_F32 && dtype != PJX_BF16 && dtype != PJX_F16)
    return fail(PJX_ERR_BAD_ARG, "dtype must be float32, bfloat16 or float16 (got code %d)", dtype);
  if (position_type != PJX_POS_F32 && position_type != PJX_POS_I32 && position_type != PJX_POS_I64)
    return fail(PJX_ERR_BAD_ARG, "positions must be float32, int32 or int64 (got code %d)", position_type);
  if (B < 0 || T < 0 || H < 1 || D < 1) return fail(PJX_ERR_BAD_ARG, "negative or zero dimension");
  if (axes < 1 || axes > kMaxAxes || !sections) return fail(PJX_ERR_BAD_ARG, "rope: 1 to %d axes with a section each", kMaxAxes);
  if (!(base > 0.f) || isinf(base)) return fail(PJX_ERR_BAD_ARG, "base must be positive and finite");
  int total = 0;
  for (int a = 0; a < axes; ++a) {
    if (sections[a] < 0 || sections[a] % 2 || sections[a] > D)
      return fail(PJX_ERR_BAD_ARG, "rope: a section must be even and at most the head width (got %d for D=%d)", sections[a], D);
    total += sections[a];
  }
  if (total > D) return fail(PJX_ERR_BAD_ARG, "rope: the sections take %d elements of a head width of %d", total, D);
  if (x_batch_stride < 0 || x_token_stride < 0 || position_batch_stride < 0) return fail(PJX_ERR_BAD_ARG, "rope: strides must be non-negative");
  if (B == 0 || T == 0) return PJX_OK;
  if (!x || !y || !positions) return fail(PJX_ERR_BAD_ARG, "rope: null buffer");
  if (total / 2 > kMaxPairs) return fail(PJX_ERR_UNSUPPORTED, "rope: at most %d rotated elements", 2 * kMaxPairs);
  RopeAxesTable table;
  memset(&table, 0, sizeof(table));
  int pair = 0;
  const double log2_base = log2((double)base);
  for (int a = 0; a < axes; ++a)
    for (int i = 0; i < sections[a] / 2; ++i, ++pair) {
      const double e = shared ? 2.0 * pair / total : 2.0 * i / sections[a];
      table.turns[pair] = exp2(-e * log2_base) / (2.0 * M_PI);
      table.axis[pair] = (uint8_t)a;
    }
  RopeAxesParams p = {};
  p.x = x; p.y = y; p.positions = positions;
  p.x_bs = x_batch_stride; p.x_ts = x_token_stride; p.pos_bs = position_batch_stride;
  p.tokens = (int64_t)B * T;
  p.T = T; p.H = H; p.D = D; p.axes = axes; p.pairs = pair; p.pos_type = position_type; p.inverse = inverse != 0;
  // as many tokens as give every thread an angle, but a few CTAs per SM first
  const int64_t most = pair > 0 ? (kTableAngles / pair < 1 ? 1 : kTableAngles / pair) : 8;
  int64_t tok = p.tokens / (148 * 8);
  tok = tok < 1 ? 1 : tok > most ? most : tok;
  while (tok > 1 && tok * H > 65536) --tok;
  p.tokens_per_cta = (int)tok;
  p.inv_heads = H > 1 ? (uint32_t)(((1ull << 32) + H - 1) / H) : 0u;
  const size_t es = dtype_size(dtype);
  const int V = (int)(16 / es);
  const bool vec = D % V == 0 && D / V <= kThreads && H <= 65536 && (interleaved || pair % V == 0) && x_batch_stride % V == 0 && x_token_stride % V == 0 &&
                   ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15) == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case PJX_F32: return launch_rope_axes<float>(p, table, !interleaved, vec, st);
    case PJX_BF16: return launch_rope_axes<__nv_bfloat16>(p, table, !interleaved, vec, st);
    default: return launch_rope_axes<__half>(p, table, !interleaved, vec, st);
  }
}
