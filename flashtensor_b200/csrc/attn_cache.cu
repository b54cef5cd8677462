// Attention of new tokens over a KV cache of ragged sequences, 16 or 8 bits, and over a prefix that they share.
//
// One softmax over the prefix's rows and the sequence's own: a warp takes a query row and walks both with a
// running maximum and sum.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "kernels.h"
#include "sm100_ptx.cuh"

namespace asuka {
using namespace sm100;

namespace {

constexpr int kThreads = 128;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool kBF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (kBF16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool kBF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (kBF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// four values of row `off` (elements) from column 4 lane on
template <bool kBF16>
__device__ __forceinline__ float4 load4(const void* base, int64_t off, int lane, int format) {
  if (format == CACHE_16) {
    const uint2 w = reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + off)[lane];
    const float2 a = unpack2<kBF16>(w.x), b = unpack2<kBF16>(w.y);
    return make_float4(a.x, a.y, b.x, b.y);
  }
  const uint32_t w = reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(base) + off)[lane];
  if (format == CACHE_I8)
    return make_float4(static_cast<int8_t>(w), static_cast<int8_t>(w >> 8), static_cast<int8_t>(w >> 16), static_cast<int8_t>(w >> 24));
  const __half2 lo(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xffffu), __NV_E4M3));
  const __half2 hi(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3));
  const float2 a = __half22float2(lo), b = __half22float2(hi);
  return make_float4(a.x, a.y, b.x, b.y);
}

template <bool kBF16>
__global__ void __launch_bounds__(kThreads) attn_cache_kernel(const CacheAttnArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  griddep_wait();
  griddep_launch_dependents();
  if (row >= static_cast<int64_t>(a.B) * a.Sq * a.H) return;
  const int h = static_cast<int>(row % a.H), i = static_cast<int>(row / a.H % a.Sq), b = static_cast<int>(row / a.H / a.Sq);
  const int hk = h / a.group;
  const float4 q = load4<kBF16>(a.q, b * a.q_sb + i * a.q_ss + h * a.q_sh, lane, CACHE_16);
  const float mul = a.softmax_scale * 1.4426950408889634f;
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int which = 0; which < 2; ++which) {
    const CacheRows& c = which == 0 ? a.prefix : a.own;
    if (c.N == 0) continue;
    const int n = b / (a.B / c.N);
    int seen = c.len != nullptr ? min(max(c.len[n], 0), c.S) : c.S;
    if (which == 1 && a.causal) seen = min(seen, seen - a.Sq + 1 + i);
    for (int64_t j = 0; j < seen; ++j) {
      const float4 k = load4<kBF16>(c.k, n * c.k_sb + j * c.k_ss + hk * c.k_sh, lane, c.format);
      float s = q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      s *= mul;
      if (c.format != CACHE_16) s *= c.k_scale[n * c.ks_sb + hk * c.ks_sh + j];
      const float top = fmaxf(m, s), ref = top > -INFINITY ? top : 0.f;
      const float w = ex2(m - ref), p = ex2(s - ref);
      m = top;
      l = l * w + p;
      const float pv = c.format != CACHE_16 ? p * c.v_scale[n * c.vs_sb + hk * c.vs_sh + j] : p;
      const float4 v = load4<kBF16>(c.v, n * c.v_sb + j * c.v_ss + hk * c.v_sh, lane, c.format);
      o = make_float4(fmaf(pv, v.x, o.x * w), fmaf(pv, v.y, o.y * w), fmaf(pv, v.z, o.z * w), fmaf(pv, v.w, o.w * w));
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  reinterpret_cast<uint2*>(a.out + b * a.o_sb + i * a.o_ss + h * a.o_sh)[lane] =
      make_uint2(pack2<kBF16>(o.x * inv, o.y * inv), pack2<kBF16>(o.z * inv, o.w * inv));
  if (a.lse2 != nullptr && lane == 0) a.lse2[(static_cast<int64_t>(b) * a.H + h) * a.Sq + i] = m + log2f(l);
}

}  // namespace

size_t attn_cache_ws_bytes(const CacheAttnArgs&, int) { return 0; }

cudaError_t launch_attn_cache(const CacheAttnArgs& a, void*, int, cudaStream_t stream) {
  const int64_t rows = static_cast<int64_t>(a.B) * a.Sq * a.H;
  const auto kern = a.bf16 ? attn_cache_kernel<true> : attn_cache_kernel<false>;
  const cudaError_t e = launch_dependent(kern, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(kThreads), 0, stream, a);
  count_launch();
  return e;
}

}  // namespace asuka
