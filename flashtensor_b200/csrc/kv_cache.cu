// An 8-bit KV cache: rows written (and, with indices, compacted) into it, and read back.
//
// A row x of 128 values becomes codes and one f32 scale: a = max(max |x|, M 2^-100), scale = a / M,
// code = round_to_even(x M / a), M = 127 (int8) or 448 (e4m3, whose rounding is the type's).  x M is exact in f32 (11 + 9
// bits) and the quotient correctly rounded, so a code is the one exact arithmetic gives, ties included.  The lower bound on a
// keeps scale and quotient normal numbers whatever the row holds; a row with an infinity or a NaN has no such code and
// gets the scale NaN, which is what attention over the unquantised row would give.
//
// Both kernels are streams: 256 bytes of a row on one side, 132 on the other, nothing twice.  Eight lanes take a row (16
// values each, two 16-byte accesses on the 16-bit side and one on the other), 32 rows of one head a CTA, so that the rows' scales
// and, in a cache whose heads are each side by side, the codes too are one run of memory.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "kernels.h"
#include "sm100_ptx.cuh"

namespace asuka {
using namespace sm100;

namespace {

constexpr int kRowsPerCta = 32;
constexpr int kLanes = 8;  // per row
constexpr int kThreads = kRowsPerCta * kLanes;

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

// Codes of this lane's 16 values (every lane of the row calls it) and the row's scale.
template <bool kBF16, bool kE4M3>
__device__ __forceinline__ uint4 quantise(const uint32_t (&x)[8], float* scale) {
  constexpr float kMost = kE4M3 ? 448.f : 127.f;
  constexpr uint32_t kInf = kBF16 ? 0x7f80u : 0x7c00u;
  // magnitudes compare as integers, infinities and NaN behind all others
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = __vmaxu2(top, x[i] & 0x7fff7fffu);
#pragma unroll
  for (int d = kLanes / 2; d > 0; d >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, d));
  const uint32_t bits = max(top & 0xffffu, top >> 16);
  const bool fine = bits < kInf;
  const float amax = fmaxf(unpack2<kBF16>(bits).x, kMost * 0x1p-100f);
  *scale = fine ? __fdiv_rn(amax, kMost) : __int_as_float(0x7fffffff);
  // (bf16 values may be so large that x M is not; both sides of the quotient times a power of two then)
  const float small = kBF16 && amax > 0x1p100f ? 0x1p-32f : 1.f, most = kMost * small, div = amax * small;
  uint32_t code[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = unpack2<kBF16>(x[2 * i]), b = unpack2<kBF16>(x[2 * i + 1]);
    const float y[4] = {__fdiv_rn(a.x * most, div), __fdiv_rn(a.y * most, div), __fdiv_rn(b.x * most, div),
                        __fdiv_rn(b.y * most, div)};
    if constexpr (kE4M3) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
      code[i] = lo | hi << 16;
    } else {
      const uint32_t lo = __byte_perm(__float2int_rn(y[0]), __float2int_rn(y[1]), 0x0040);
      const uint32_t hi = __byte_perm(__float2int_rn(y[2]), __float2int_rn(y[3]), 0x0040);
      code[i] = __byte_perm(lo, hi, 0x5410);
    }
    if (!fine) code[i] = 0;
  }
  return make_uint4(code[0], code[1], code[2], code[3]);
}

template <bool kBF16, bool kE4M3>
__global__ void __launch_bounds__(kThreads) quant_kv_kernel(const QuantKvArgs a) {
  const int h = blockIdx.y, b = blockIdx.z;
  const int lane = threadIdx.x % kLanes;
  griddep_wait();
  griddep_launch_dependents();
  const int count = a.count != nullptr ? min(a.count[b], a.n) : a.n;
  const int64_t start = a.start != nullptr ? a.start[b] : 0;
  for (int i0 = blockIdx.x * kRowsPerCta; i0 < count; i0 += gridDim.x * kRowsPerCta) {  // (the same for the CTA)
    const int i = i0 + threadIdx.x / kLanes;
    const int64_t to = start + i;
    const bool live = i < count && to >= 0 && to < a.cache.S;
    uint32_t k[8] = {}, v[8] = {};
    if (live) {
      int from = i;
      if (a.idx != nullptr) from = min(max(a.idx[(static_cast<int64_t>(b) * a.H + h) * a.n + i], 0), a.T - 1);
      const uint4* ks = reinterpret_cast<const uint4*>(a.k + b * a.k_sb + from * a.k_ss + h * a.k_sh) + 2 * lane;
      const uint4* vs = reinterpret_cast<const uint4*>(a.v + b * a.v_sb + from * a.v_ss + h * a.v_sh) + 2 * lane;
      *reinterpret_cast<uint4*>(&k[0]) = ks[0];
      *reinterpret_cast<uint4*>(&k[4]) = ks[1];
      *reinterpret_cast<uint4*>(&v[0]) = vs[0];
      *reinterpret_cast<uint4*>(&v[4]) = vs[1];
    }
    float k_scale, v_scale;
    const uint4 kc = quantise<kBF16, kE4M3>(k, &k_scale), vc = quantise<kBF16, kE4M3>(v, &v_scale);
    if (live) {
      uint8_t* kd = static_cast<uint8_t*>(a.cache.k) + b * a.cache.k_sb + to * a.cache.k_ss + h * a.cache.k_sh;
      uint8_t* vd = static_cast<uint8_t*>(a.cache.v) + b * a.cache.v_sb + to * a.cache.v_ss + h * a.cache.v_sh;
      reinterpret_cast<uint4*>(kd)[lane] = kc;
      reinterpret_cast<uint4*>(vd)[lane] = vc;
      if (lane == 0) {
        a.cache.k_scale[b * a.cache.ks_sb + h * a.cache.ks_sh + to] = k_scale;
        a.cache.v_scale[b * a.cache.vs_sb + h * a.cache.vs_sh + to] = v_scale;
      }
    }
  }
}

// 16 codes times their row's scale, rounded once.
template <bool kBF16, bool kE4M3>
__device__ __forceinline__ void restore(const uint4& c, float scale, uint32_t (&y)[8]) {
  const uint32_t code[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x[4];
    if constexpr (kE4M3) {
      const __half2 lo(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(code[i] & 0xffffu), __NV_E4M3));
      const __half2 hi(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(code[i] >> 16), __NV_E4M3));
      const float2 a = __half22float2(lo), b = __half22float2(hi);
      x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
    } else {
      // (code + 128 as the low byte of 2^23's significand, less 2^23 + 128)
      const uint32_t u = code[i] ^ 0x80808080u;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7650 + e)) - 8388736.f;
    }
    y[2 * i] = pack2<kBF16>(x[0] * scale, x[1] * scale);
    y[2 * i + 1] = pack2<kBF16>(x[2] * scale, x[3] * scale);
  }
}

template <bool kBF16, bool kE4M3>
__global__ void __launch_bounds__(kThreads) dequant_kv_kernel(const DequantKvArgs a) {
  const int h = blockIdx.y, b = blockIdx.z;
  const int lane = threadIdx.x % kLanes;
  griddep_wait();
  griddep_launch_dependents();
  const int len = a.cache.len != nullptr ? min(a.cache.len[b], a.cache.S) : a.cache.S;
  for (int i = blockIdx.x * kRowsPerCta + threadIdx.x / kLanes; i < a.n; i += gridDim.x * kRowsPerCta) {
    int64_t from = i;
    if (a.idx != nullptr)
      from = min(max(a.idx[(static_cast<int64_t>(b) * a.H + h) * a.n + i], 0), a.cache.S - 1);
    uint32_t k[8] = {}, v[8] = {};
    if (from < len) {
      const uint8_t* ks = static_cast<const uint8_t*>(a.cache.k) + b * a.cache.k_sb + from * a.cache.k_ss + h * a.cache.k_sh;
      const uint8_t* vs = static_cast<const uint8_t*>(a.cache.v) + b * a.cache.v_sb + from * a.cache.v_ss + h * a.cache.v_sh;
      const uint4 kc = reinterpret_cast<const uint4*>(ks)[lane], vc = reinterpret_cast<const uint4*>(vs)[lane];
      restore<kBF16, kE4M3>(kc, a.cache.k_scale[b * a.cache.ks_sb + h * a.cache.ks_sh + from], k);
      restore<kBF16, kE4M3>(vc, a.cache.v_scale[b * a.cache.vs_sb + h * a.cache.vs_sh + from], v);
    }
    uint4* kd = reinterpret_cast<uint4*>(a.k_out + b * a.k_sb + i * a.k_ss + h * a.k_sh) + 2 * lane;
    uint4* vd = reinterpret_cast<uint4*>(a.v_out + b * a.v_sb + i * a.v_ss + h * a.v_sh) + 2 * lane;
    kd[0] = *reinterpret_cast<const uint4*>(&k[0]);
    kd[1] = *reinterpret_cast<const uint4*>(&k[4]);
    vd[0] = *reinterpret_cast<const uint4*>(&v[0]);
    vd[1] = *reinterpret_cast<const uint4*>(&v[4]);
  }
}

unsigned row_blocks(int rows) { return static_cast<unsigned>((static_cast<int64_t>(rows) + kRowsPerCta - 1) / kRowsPerCta); }

}  // namespace

cudaError_t launch_quant_kv(const QuantKvArgs& a, cudaStream_t stream) {
  const bool e4m3 = a.cache.format == CACHE_E4M3;
  const auto kern = a.bf16 ? (e4m3 ? quant_kv_kernel<true, true> : quant_kv_kernel<true, false>)
                           : (e4m3 ? quant_kv_kernel<false, true> : quant_kv_kernel<false, false>);
  const cudaError_t e = launch_dependent(kern, dim3(row_blocks(a.n), a.H, a.B), dim3(kThreads), 0, stream, a);
  count_launch();
  return e;
}

cudaError_t launch_dequant_kv(const DequantKvArgs& a, cudaStream_t stream) {
  const bool e4m3 = a.cache.format == CACHE_E4M3;
  const auto kern = a.bf16 ? (e4m3 ? dequant_kv_kernel<true, true> : dequant_kv_kernel<true, false>)
                           : (e4m3 ? dequant_kv_kernel<false, true> : dequant_kv_kernel<false, false>);
  const cudaError_t e = launch_dependent(kern, dim3(row_blocks(a.n), a.H, a.cache.N), dim3(kThreads), 0, stream, a);
  count_launch();
  return e;
}

}  // namespace asuka
