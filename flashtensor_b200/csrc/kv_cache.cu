// An 8-bit KV cache: rows written (and, with indices, compacted) into it, and read back.
//
// A row x of 128 values becomes codes and one f32 scale: a = max(max |x|, M 2^-100), scale = a / M,
// code = round_to_even(x M / a), M = 127 (int8) or 448 (e4m3, whose rounding is the type's).  x M is exact in f32 (11 + 9
// bits) and the quotient correctly rounded, so a code is the one exact arithmetic gives, ties included.  The lower bound on a
// keeps scale and quotient normal numbers whatever the row holds; a row with an infinity or a NaN has no such code and
// gets the scale NaN, which is what attention over the unquantised row would give.
//
// The quotient is a product with the reciprocal of a, corrected by its remainder, which one fused multiply-add gives exactly
// but for its last bit (Markstein, IBM J. Res. Dev. 34, 1990): 2 instructions for a value, where a division takes ten and more.
//
// Both kernels are streams: 256 bytes of a row on one side, 132 on the other, nothing twice.  Eight lanes take a row of the keys or of
// the values (16 values each, two 16-byte accesses on the 16-bit side and two of 8 on the other), 32 rows of one head a CTA, so that the
// rows' scales and, in a cache whose heads are each side by side, the codes too are one run of memory; with fewer rows to a
// head, as in a decode step, the heads follow each other.  What is read does not wait for what says whether it counts.
// On the device: 32 sequences of up to 2001 tokens, 8 heads, to e4m3 (301 MB moved) 66 us = 4.6 TB/s, one token of 16 sequences 1.6 us;
// 2 sequences of 5003 rows, 8 heads, back to bf16 (60 MB moved) 11.4 us = 5.2 TB/s.
#include <cuda_fp8.h>

#include "attn_cache.cuh"

namespace asuka {

namespace {

constexpr int kRowsPerCta = 32;
constexpr int kLanes = 8;  // per row
constexpr int kThreads = kRowsPerCta * kLanes;

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
  const float amax = fmaxf(unpack2<kBF16>(fine ? bits : 0u).x, kMost * 0x1p-100f);
  *scale = fine ? __fdiv_rn(amax, kMost) : __int_as_float(0x7fffffff);
  // (bf16 values may be so large that x M is not; both sides of the quotient times a power of two then)
  const float small = kBF16 && amax > 0x1p100f ? 0x1p-32f : 1.f, most = fine ? kMost * small : 0.f, div = amax * small;
  const float inv = __frcp_rn(div);
  const float2 most2 = make_float2(most, most), inv2 = make_float2(inv, inv), minus2 = make_float2(-div, -div);
  uint32_t code[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 y[2];
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      float2 v = unpack2<kBF16>(x[2 * i + z]);
      if (!fine) v = make_float2(0.f, 0.f);
      const float2 n = __fmul2_rn(v, most2), q = __fmul2_rn(n, inv2);
      y[z] = __ffma2_rn(__ffma2_rn(q, minus2, n), inv2, q);
    }
    if constexpr (kE4M3) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(y[0], __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(y[1], __NV_SATFINITE, __NV_E4M3);
      code[i] = lo | hi << 16;
    } else {
      // (the integer nearest, ties to even, as the low bits of 1.5 * 2^23 + y)
      const float2 even = make_float2(12582912.f, 12582912.f);
      const float2 a = __fadd2_rn(y[0], even), b = __fadd2_rn(y[1], even);
      const uint32_t lo = __byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040);
      const uint32_t hi = __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040);
      code[i] = __byte_perm(lo, hi, 0x5410);
    }
  }
  return make_uint4(code[0], code[1], code[2], code[3]);
}

// Which rows a group of lanes takes: kEach of the keys or of the values, 32 rows apart, row `i` of `n` of a head, or with few rows to a
// head (gridDim.y = 1) of all heads in turn.  (Heads as the fast index of the grid, whose rows of a token lie side by side on the
// 16-bit side: 10.8 -> 11.3 us for four prompts of 2001 tokens.)
struct At {
  int h, i;
  bool live;
};
template <int kEach>
__device__ __forceinline__ At row_at(int z, int n, int H) {
  const int r = (static_cast<int>(blockIdx.x >> 1) * kEach + z) * kRowsPerCta + static_cast<int>(threadIdx.x) / kLanes;
  At x;
  if (n < kRowsPerCta) {
    x.h = r / n;
    x.i = r - x.h * n;
    x.live = x.h < H;
  } else {
    x.h = blockIdx.y;
    x.i = r;
    x.live = r < n;
  }
  return x;
}

template <bool kBF16, bool kE4M3, int kEach>
__global__ void __launch_bounds__(kThreads) quant_kv_kernel(const QuantKvArgs a) {
  const int b = blockIdx.z, lane = threadIdx.x % kLanes;
  const bool values = blockIdx.x & 1;
  const CacheRows& c = a.cache;
  const uint16_t* src = values ? a.v + b * a.v_sb : a.k + b * a.k_sb;
  const int64_t src_s = values ? a.v_ss : a.k_ss, src_h = values ? a.v_sh : a.k_sh;
  uint8_t* dst = values ? static_cast<uint8_t*>(c.v) + b * c.v_sb : static_cast<uint8_t*>(c.k) + b * c.k_sb;
  const int64_t dst_s = values ? c.v_ss : c.k_ss, dst_h = values ? c.v_sh : c.k_sh;
  float* scales = values ? c.v_scale + b * c.vs_sb : c.k_scale + b * c.ks_sb;
  const int64_t scales_h = values ? c.vs_sh : c.ks_sh;
  griddep_wait();
  griddep_launch_dependents();
  At at[kEach];
#pragma unroll
  for (int z = 0; z < kEach; ++z) at[z] = row_at<kEach>(z, a.n, a.H);
  uint32_t x[kEach][8] = {};
#pragma unroll
  for (int z = 0; z < kEach; ++z) {
    if (!at[z].live) continue;
    int from = at[z].i;
    if (a.idx != nullptr) from = min(max(a.idx[(static_cast<int64_t>(b) * a.H + at[z].h) * a.n + from], 0), a.T - 1);
    const uint4* row = reinterpret_cast<const uint4*>(src + from * src_s + at[z].h * src_h);
    *reinterpret_cast<uint4*>(&x[z][0]) = row[lane];
    *reinterpret_cast<uint4*>(&x[z][4]) = row[lane + kLanes];
  }
  const int64_t start = a.start != nullptr ? a.start[b] : 0;
  const int count = a.count != nullptr ? a.count[b] : a.n;
#pragma unroll
  for (int z = 0; z < kEach; ++z) {
    float scale;
    const uint4 code = quantise<kBF16, kE4M3>(x[z], &scale);
    const int64_t to = start + at[z].i;
    if (!at[z].live || at[z].i >= count || to < 0 || to >= c.S) continue;
    uint2* row = reinterpret_cast<uint2*>(dst + to * dst_s + at[z].h * dst_h);
    row[lane] = make_uint2(code.x, code.y);
    row[lane + kLanes] = make_uint2(code.z, code.w);
    if (lane == 0) scales[at[z].h * scales_h + to] = scale;
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

template <bool kBF16, bool kE4M3, int kEach>
__global__ void __launch_bounds__(kThreads) dequant_kv_kernel(const DequantKvArgs a) {
  const int b = blockIdx.z, lane = threadIdx.x % kLanes;
  const bool values = blockIdx.x & 1;
  const CacheRows& c = a.cache;
  const uint8_t* src = values ? static_cast<const uint8_t*>(c.v) + b * c.v_sb : static_cast<const uint8_t*>(c.k) + b * c.k_sb;
  const int64_t src_s = values ? c.v_ss : c.k_ss, src_h = values ? c.v_sh : c.k_sh;
  const float* scales = values ? c.v_scale + b * c.vs_sb : c.k_scale + b * c.ks_sb;
  const int64_t scales_h = values ? c.vs_sh : c.ks_sh;
  uint16_t* dst = values ? a.v_out + b * a.v_sb : a.k_out + b * a.k_sb;
  const int64_t dst_s = values ? a.v_ss : a.k_ss, dst_h = values ? a.v_sh : a.k_sh;
  griddep_wait();
  griddep_launch_dependents();
  At at[kEach];
#pragma unroll
  for (int z = 0; z < kEach; ++z) at[z] = row_at<kEach>(z, a.n, a.H);
  uint2 lo[kEach], hi[kEach];
  float scale[kEach];
  int64_t from[kEach];
#pragma unroll
  for (int z = 0; z < kEach; ++z) {
    if (!at[z].live) continue;
    from[z] = at[z].i;
    if (a.idx != nullptr) from[z] = min(max(a.idx[(static_cast<int64_t>(b) * a.H + at[z].h) * a.n + at[z].i], 0), c.S - 1);
    const uint2* row = reinterpret_cast<const uint2*>(src + from[z] * src_s + at[z].h * src_h);
    lo[z] = row[lane];
    hi[z] = row[lane + kLanes];
    scale[z] = scales[at[z].h * scales_h + from[z]];
  }
  const int len = c.len != nullptr ? c.len[b] : c.S;
#pragma unroll
  for (int z = 0; z < kEach; ++z) {
    if (!at[z].live) continue;
    uint32_t x[8];
    restore<kBF16, kE4M3>(make_uint4(lo[z].x, lo[z].y, hi[z].x, hi[z].y), scale[z], x);
    if (from[z] >= len) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0u;
    }
    uint4* row = reinterpret_cast<uint4*>(dst + at[z].i * dst_s + at[z].h * dst_h);
    row[lane] = *reinterpret_cast<const uint4*>(&x[0]);
    row[lane + kLanes] = *reinterpret_cast<const uint4*>(&x[4]);
  }
}

// Rows to a group of lanes where there are enough.  us, one / two / four: four prompts of 2001 tokens 11.8 / 10.8 / 11.8, 32 of
// them 75.8 / 66.1 / 64.6; 768 of 4096 rows compacted 6.7 / 6.7 / 8.6; two times 5003 rows read back 11.6 / 11.4 / 11.5, 512 rows of four times 32
// heads 12.2 / 11.4 / 13.6.
constexpr int kMany = 2;

// (twice the CTAs of the rows: keys and values)
dim3 grid_of(int n, int H, int B, int each) {
  const int rows = n < kRowsPerCta ? n * H : n, per = kRowsPerCta * each;
  return dim3(2u * ((rows + per - 1) / per), n < kRowsPerCta ? 1 : H, B);
}
template <bool kBF16, bool kE4M3>
cudaError_t launch_quant(const QuantKvArgs& a, cudaStream_t stream) {
  const int each = a.n >= kRowsPerCta * kMany ? kMany : 1;
  return launch_dependent(each > 1 ? quant_kv_kernel<kBF16, kE4M3, kMany> : quant_kv_kernel<kBF16, kE4M3, 1>,
                          grid_of(a.n, a.H, a.B, each), dim3(kThreads), 0, stream, a);
}
template <bool kBF16, bool kE4M3>
cudaError_t launch_dequant(const DequantKvArgs& a, cudaStream_t stream) {
  const int each = a.n >= kRowsPerCta * kMany ? kMany : 1;
  return launch_dependent(each > 1 ? dequant_kv_kernel<kBF16, kE4M3, kMany> : dequant_kv_kernel<kBF16, kE4M3, 1>,
                          grid_of(a.n, a.H, a.cache.N, each), dim3(kThreads), 0, stream, a);
}

}  // namespace

cudaError_t launch_quant_kv(const QuantKvArgs& a, cudaStream_t stream) {
  const bool e4m3 = a.cache.format == CACHE_E4M3;
  const cudaError_t e = a.bf16 ? (e4m3 ? launch_quant<true, true>(a, stream) : launch_quant<true, false>(a, stream))
                               : (e4m3 ? launch_quant<false, true>(a, stream) : launch_quant<false, false>(a, stream));
  count_launch();
  return e;
}

cudaError_t launch_dequant_kv(const DequantKvArgs& a, cudaStream_t stream) {
  const bool e4m3 = a.cache.format == CACHE_E4M3;
  const cudaError_t e = a.bf16 ? (e4m3 ? launch_dequant<true, true>(a, stream) : launch_dequant<true, false>(a, stream))
                               : (e4m3 ? launch_dequant<false, true>(a, stream) : launch_dequant<false, false>(a, stream));
  count_launch();
  return e;
}

}  // namespace asuka
