// merge_states.cu — merge of attention states over disjoint parts of the keys
// (the LSE rule of cute_attention/cluster_decode/cluster_decode_reduce.py:
// 67-91): M = max_i lse_i, w_i = e^(lse_i - M), out = sum w_i out_i / sum w_i,
// lse = M + ln sum w_i.
//
// HBM-bound: every state is read once, the result written once.  A thread
// owns 8 consecutive elements of a row (16-byte loads; two for fp32) and takes
// the states U at a time: their values and lse are loaded together, one round
// trip to memory, and folded in with a running maximum.  It computes the
// row's weights itself, from broadcast loads: cheaper than a barrier.  A state
// with lse = -inf is left out, not multiplied by 0, so it may hold anything.
// 8 bf16 states of [256, 32, 128], 19 MB: 6.6 us, 2.9 TB/s, of which about 3 us
// are launch and one round trip.
#include <type_traits>

#include "b2d_decode.h"
#include "common.cuh"
#include "gqa_kernel.cuh"

namespace b2d {

struct MergeParams {
  const void* outs;
  int64_t sn, st, sh;
  const float* lses;
  int64_t ln, lt, lh;
  void* out;
  int64_t ot, oh;
  float* lse;
  int64_t let, leh;
  int N, H, D8;
  int64_t work;  // rows * D / 8
};

// 8 elements as they lie in memory.
template <typename T>
struct Raw8 {
  uint4 w;
  __device__ __forceinline__ void get(float* v) const {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 f;
      if constexpr (std::is_same<T, __nv_bfloat16>::value) f = bf16x2_to_f2(x[i]);
      else f = f16x2_to_f2(x[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
};
template <>
struct __align__(16) Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void get(float* v) const {
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
};

template <typename T>
__device__ __forceinline__ void store8(T* dst, const float* v) {
  if constexpr (std::is_same<T, float>::value) {
    reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    store_out8<T>(dst, v);
  }
}

template <typename IT, typename OT>
__global__ void __launch_bounds__(256) merge_states_kernel(const MergeParams p) {
  constexpr float kLog2e = 1.4426950408889634f;
  constexpr int U = std::is_same<IT, float>::value ? 4 : 8;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= p.work) return;
  const int64_t row = i / p.D8;
  const int c = (int)(i - row * p.D8) * 8;
  const int64_t t = row / p.H;
  const int h = (int)(row - t * p.H);
  const float* ls = p.lses + t * p.lt + (int64_t)h * p.lh;
  const IT* src = reinterpret_cast<const IT*>(p.outs) + t * p.st + (int64_t)h * p.sh + c;
  float mx = -INFINITY;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, sum = 0.f;
  for (int n0 = 0; n0 < p.N; n0 += U) {
    Raw8<IT> raw[U];
    float l[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int n = n0 + u < p.N ? n0 + u : p.N - 1;
      raw[u] = *reinterpret_cast<const Raw8<IT>*>(src + n * p.sn);
      l[u] = n0 + u < p.N ? ls[n * p.ln] : -INFINITY;
    }
    float nm = mx;
#pragma unroll
    for (int u = 0; u < U; ++u) nm = fmaxf(nm, l[u]);
    const float mz = nm == -INFINITY ? 0.f : nm, old = fast_exp2((mx - mz) * kLog2e);
    sum *= old;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= old;
    mx = nm;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (l[u] == -INFINITY) continue;
      const float w = fast_exp2((l[u] - mz) * kLog2e);
      float v[8];
      raw[u].get(v);
      sum += w;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += w * v[e];
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] *= inv;
  store8<OT>(reinterpret_cast<OT*>(p.out) + t * p.ot + (int64_t)h * p.oh + c, acc);
  if (p.lse != nullptr && c == 0) p.lse[t * p.let + (int64_t)h * p.leh] = mx == -INFINITY ? mx + sum : mx + logf(sum);
}

}  // namespace b2d

using namespace b2d;

extern "C" int b2d_merge_states(const b2d_merge_args* a, void* stream) {
  if (!a) return B2D_ERR_INVALID_ARG;
  if (a->num_states <= 0 || a->num_tokens < 0 || a->num_heads <= 0 || a->head_dim <= 0)
    return B2D_ERR_INVALID_ARG;
  if (a->head_dim % 8 != 0 || a->head_dim > 1024) return B2D_ERR_UNSUPPORTED;
  const bool in32 = a->in_dtype == B2D_FP32, out32 = a->out_dtype == B2D_FP32;
  if (!in32 && a->in_dtype != B2D_BF16 && a->in_dtype != B2D_FP16) return B2D_ERR_UNSUPPORTED;
  if (a->out_dtype != a->in_dtype && !(in32 && (a->out_dtype == B2D_BF16 || a->out_dtype == B2D_FP16)))
    return B2D_ERR_UNSUPPORTED;
  if (a->num_tokens == 0) return B2D_OK;
  if (!a->outs || !a->lses || !a->out) return B2D_ERR_INVALID_ARG;
  const int is = in32 ? 4 : 2, os = out32 ? 4 : 2;
  if (((uintptr_t)a->outs & 15) || ((uintptr_t)a->out & 15) || (a->outs_stride_n * is) % 16 ||
      (a->outs_stride_t * is) % 16 || (a->outs_stride_h * is) % 16 || (a->out_stride_t * os) % 16 ||
      (a->out_stride_h * os) % 16)
    return B2D_ERR_ALIGNMENT;
  MergeParams p{};
  p.outs = a->outs;
  p.sn = a->outs_stride_n;
  p.st = a->outs_stride_t;
  p.sh = a->outs_stride_h;
  p.lses = a->lses;
  p.ln = a->lses_stride_n;
  p.lt = a->lses_stride_t;
  p.lh = a->lses_stride_h;
  p.out = a->out;
  p.ot = a->out_stride_t;
  p.oh = a->out_stride_h;
  p.lse = a->lse;
  p.let = a->lse_stride_t;
  p.leh = a->lse_stride_h;
  p.N = a->num_states;
  p.H = a->num_heads;
  p.D8 = a->head_dim / 8;
  p.work = (int64_t)a->num_tokens * a->num_heads * p.D8;
  if (p.work > (int64_t)INT32_MAX * 256) return B2D_ERR_TOO_LARGE;
  const int blocks = (int)((p.work + 255) / 256);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!in32) {
    if (a->in_dtype == B2D_BF16) merge_states_kernel<__nv_bfloat16, __nv_bfloat16><<<blocks, 256, 0, s>>>(p);
    else merge_states_kernel<__half, __half><<<blocks, 256, 0, s>>>(p);
  } else if (out32) {
    merge_states_kernel<float, float><<<blocks, 256, 0, s>>>(p);
  } else if (a->out_dtype == B2D_BF16) {
    merge_states_kernel<float, __nv_bfloat16><<<blocks, 256, 0, s>>>(p);
  } else {
    merge_states_kernel<float, __half><<<blocks, 256, 0, s>>>(p);
  }
  return cudaGetLastError() == cudaSuccess ? B2D_OK : B2D_ERR_CUDA;
}
