// Attention that every cached key receives from a window of queries, summed over the query heads of its group: the quantity
// that decides which keys a bounded cache keeps.  With the log-sum-exp of the attention call known, one pass over the keys:
//   out[b, hk, j] = in[b, hk, j] + sum over visible rows (t, h) of exp(sm_scale q[b, t, h] . k[b, j, hk] - lse[b, h, t]).
//
// This file holds the exact fp32 kernel on CUDA cores, for fp32 inputs and head widths that the tensor-core kernel
// (key_weights_sm100.cu) does not take.  One CTA owns 64 keys of one (sequence, KV head) and walks the packed rows
// (t, g) in tiles of 64; 16 x 16 threads with 4 x 4 scores each.  Bound by shared-memory loads.
#include "pjx_common.cuh"
#include "tile_f32.cuh"

namespace pjx {
namespace {

constexpr int NT = 256;
constexpr int BT = 64;  // keys and rows per tile

// One row of `width` elements, zeros where there is none and up to a multiple of four; u: one of 8 threads.
template <typename T>
__device__ __forceinline__ void load_row(float* dst, const T* row, int width, bool there, int u) {
  if (sizeof(T) == 4 && width % 4 == 0 && (reinterpret_cast<uintptr_t>(row) & 15) == 0) {
    for (int d = u * 4; d < width; d += 32)
      *reinterpret_cast<float4*>(dst + d) = there ? __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(row) + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
  } else {
    for (int d = u; d < (width + 3) / 4 * 4; d += 8) dst[d] = there && d < width ? Elem<T>::to_f(row[d]) : 0.f;
  }
}

template <typename T>
__global__ void __launch_bounds__(NT) key_weights_kernel(const KeyWeightsParams p) {
  extern __shared__ float smem[];
  const int D = p.D, Dp = pitch4(D);
  float* Ks = smem;                // [BT][Dp]
  float* Qs = Ks + BT * Dp;        // [BT][Dp]
  float* lse2 = Qs + BT * Dp;      // [BT]
  float* sums = lse2 + BT;         // [16][BT]
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int k0 = blockIdx.x * BT, hk = blockIdx.y, b = blockIdx.z;
  const int G = p.Hq / p.Hkv, rows = p.Lq * G;
  const T* q = static_cast<const T*>(p.q);
  const T* k = static_cast<const T*>(p.k);
  const int len = p.kv_lengths ? max(0, min(p.Lkv, p.kv_lengths[b])) : p.Lkv;
  float w[4] = {0.f, 0.f, 0.f, 0.f};
  // query tokens that see a key of this tile
  const int t_first = (int)max((int64_t)0, (int64_t)k0 - p.band_hi);
  const int t_last = (int)min((int64_t)p.Lq, (int64_t)k0 + BT - p.band_lo);
  if (k0 < len && t_first < t_last) {
    for (int r = tid >> 3; r < BT; r += NT / 8)
      load_row<T>(Ks + r * Dp, k + (((int64_t)b * p.Lkv + k0 + r) * p.Hkv + hk) * D, D, k0 + r < len, tid & 7);
    const float c1 = p.sm_scale * kLog2e;
    for (int r0 = t_first * G; r0 < t_last * G; r0 += BT) {
      __syncthreads();
      for (int r = tid >> 3; r < BT; r += NT / 8) {
        const int row = r0 + r, t = row / G, g = row - t * G;
        load_row<T>(Qs + r * Dp, q + (((int64_t)b * p.Lq + t) * p.Hq + hk * G + g) * D, D, row < rows, tid & 7);
      }
      if (tid < BT) {
        const int row = r0 + tid, t = row / G, g = row - t * G;
        lse2[tid] = row < rows ? p.lse[((int64_t)b * p.Hq + hk * G + g) * p.Lq + t] * kLog2e : INFINITY;
      }
      __syncthreads();
      float s[4][4] = {};
#pragma unroll 4
      for (int d = 0; d < D; d += 4) {
        float4 a[4], c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a[i] = ld4(Qs + (ty * 4 + i) * Dp + d);
          c[i] = ld4(Ks + (tx + 16 * i) * Dp + d);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][e] = dot4(a[i], c[e], s[i][e]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float l = lse2[ty * 4 + i];
        const int t = (r0 + ty * 4 + i) / G;
        if (l == INFINITY) continue;  // a row without keys
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = k0 + tx + 16 * e;
          const bool keep = key < len && key <= (int64_t)t + p.band_hi && key >= (int64_t)t + p.band_lo;
          w[e] += keep ? exp2f(fmaf(s[i][e], c1, -l)) : 0.f;
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) sums[ty * BT + tx + 16 * e] = w[e];
  __syncthreads();
  const int key = k0 + tid;
  if (tid < BT && key < p.Lkv) {
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) total += sums[i * BT + tid];
    const int64_t at = ((int64_t)b * p.Hkv + hk) * p.Lkv + key;
    p.weights_out[at] = (p.weights_in ? p.weights_in[at] : 0.f) + (key < len ? total : 0.f);
  }
}

template <typename T>
int launch_t(const KeyWeightsParams& p, cudaStream_t stream) {
  auto smem_bytes = [](int D) { return (2 * BT * pitch4(D) + BT + 16 * BT) * (int)sizeof(float); };
  const int smem = smem_bytes(p.D);
  static std::atomic<uint64_t> allowed{0};  // (for the widest call: another thread's must not lower it before this launch)
  int rc = allow_smem(reinterpret_cast<const void*>(key_weights_kernel<T>), smem_bytes(256), allowed);
  if (rc) return rc;
  key_weights_kernel<T><<<dim3((p.Lkv + BT - 1) / BT, p.Hkv, p.B), NT, smem, stream>>>(p);
  count_launch();
  return check_cuda(cudaGetLastError(), "key weights launch");
}

}  // namespace

int launch_key_weights(const KeyWeightsParams& p, int dtype, int impl, cudaStream_t stream) {
  if (impl != PJX_IMPL_GENERIC && key_weights_sm100_supported(p, dtype)) return launch_key_weights_sm100(p, dtype, stream);
  if (impl == PJX_IMPL_SM100)
    return fail(PJX_ERR_UNSUPPORTED, "the tcgen05 key weights take bf16/fp16, D in {64, 128}, at most 128 query heads a KV head and 16-byte aligned q / k");
  if (p.D > 256) return fail(PJX_ERR_UNSUPPORTED, "key weights: head width up to 256 (got %d)", p.D);
  switch (dtype) {
    case PJX_F32: return launch_t<float>(p, stream);
    case PJX_BF16: return launch_t<__nv_bfloat16>(p, stream);
    default: return launch_t<__half>(p, stream);
  }
}

}  // namespace pjx

extern "C" int pjx_attn_key_weights(const void* q, const void* k, const float* lse, const float* weights_in, float* weights_out,
                                    const int32_t* kv_lengths, int B, int Lq, int Lkv, int Hq, int Hkv, int D, int dtype, int band_lo,
                                    int band_hi, float sm_scale, int impl, int32_t* status, void* stream) {
  using namespace pjx;
  if (dtype != PJX_F32 && dtype != PJX_BF16 && dtype != PJX_F16)
    return fail(PJX_ERR_BAD_ARG, "dtype must be float32, bfloat16 or float16 (got code %d)", dtype);
  if (B < 0 || Lq < 0 || Lkv < 0 || Hq < 1 || Hkv < 1 || D < 1) return fail(PJX_ERR_BAD_ARG, "negative or zero dimension");
  if (Hq % Hkv != 0) return fail(PJX_ERR_BAD_ARG, "query heads %d must be a multiple of kv heads %d", Hq, Hkv);
  if (impl != PJX_IMPL_AUTO && impl != PJX_IMPL_GENERIC && impl != PJX_IMPL_SM100)
    return fail(PJX_ERR_BAD_ARG, "impl must be 0 (auto), 1 (generic) or 2 (tcgen05), got %d", impl);
  if (B == 0 || Lkv == 0) return PJX_OK;
  if (!k || !weights_out || (Lq > 0 && (!q || !lse))) return fail(PJX_ERR_BAD_ARG, "key weights: null buffer");
  if (Lq >= PJX_BAND_NO_UPPER || Lkv >= PJX_BAND_NO_UPPER) return fail(PJX_ERR_BAD_ARG, "sequence lengths must be below 2^30");
  if (B > 65535 || Hkv > 65535 || (int64_t)Lq * (Hq / Hkv) > 0x7fffff00)
    return fail(PJX_ERR_UNSUPPORTED, "key weights: at most 65535 sequences and kv heads and 2^31 query rows a kv head per call");
  KeyWeightsParams p = {};
  p.q = q; p.k = k; p.lse = lse; p.weights_in = weights_in; p.weights_out = weights_out; p.kv_lengths = kv_lengths;
  p.B = B; p.Lq = Lq; p.Lkv = Lkv; p.Hq = Hq; p.Hkv = Hkv; p.D = D;
  p.band_lo = band_lo < PJX_BAND_NO_LOWER ? PJX_BAND_NO_LOWER : band_lo > PJX_BAND_NO_UPPER ? PJX_BAND_NO_UPPER : band_lo;
  p.band_hi = band_hi > PJX_BAND_NO_UPPER ? PJX_BAND_NO_UPPER : band_hi < PJX_BAND_NO_LOWER ? PJX_BAND_NO_LOWER : band_hi;
  p.sm_scale = sm_scale;
  p.status = status;
  return launch_key_weights(p, dtype, impl, static_cast<cudaStream_t>(stream));
}
