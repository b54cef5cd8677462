// What the kernels of a cache share: pairs of 16-bit values, a segment's rows, partial results, codes, tensor maps.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.h"
#include "sm100_ptx.cuh"
#include "tma_host.h"

namespace asuka {
using namespace sm100;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Over 8 bits the reference of a row's exponentials contains the values' scales (2^-76 to 2^121, smaller ones count as 2^-76), so that
// the largest term of their sum may be anything from 2^-121 to 2^76, and one that counts a little less.  While they are summed
// they are kept times 2^kLift: neither end leaves f32's normal numbers, and what a term may lose is below 2^-28 of the largest.
// What takes a sum from one reference to the next may be smaller than any of those; it comes as the square of `half_step`.
constexpr int kLeast = -76;
constexpr float kLeastScale = 0x1p-76f;
constexpr int kLift = 24;
constexpr float kLiftUp = 0x1p24f, kLiftDown = 0x1p-24f;
__device__ __forceinline__ float half_step(float from, float to) { return ex2(0.5f * (from - to)); }
// (Without scales above kLarge a sum is 2^-20 at least, and no reference that counts is 2^126 below another's.)
constexpr float kLarge = 0x1p20f;
// Such a sum and its reference as others are: the sum in [0.5, 1), the reference with what that takes.  Returns what takes the
// weighted values along.  (Nothing seen, or nothing but NaN, stays what it is.)
__device__ __forceinline__ float unlift(float& ref, float& sum) {
  const int e = min(max(static_cast<int>(__float_as_uint(sum) >> 23 & 0xffu), 25), 252) - 126;  // (both factors normal numbers)
  sum *= __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  ref += static_cast<float>(e - kLift);
  return __uint_as_float(static_cast<uint32_t>(127 + kLift - e) << 23);
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
__device__ __forceinline__ void lds4(uint32_t addr, uint32_t* r) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// ---- a segment's rows ----------------------------------------------------------------------------
struct Segment {
  int N, S, n;     // sequences, rows of each at most, sequences of q to each
  int rows;        // query rows of a unit: n * Sq * group
  int causal;
  const int32_t* len;
};
struct RowShape {
  int Sq, H, Hkv, group;
};
// Row r of a unit: (sequence of q, position, head in the group), heads fastest.
struct Row {
  int b, pos, h;
};
__device__ __forceinline__ Row decode_row(int r, int seq, int hk, const Segment& s, const RowShape& q) {
  const int g = r % q.group, x = r / q.group;
  return {seq * s.n + x / q.Sq, x % q.Sq, hk * q.group + g};
}
__device__ __forceinline__ int seen_of(const Segment& s, int seq) {
  return s.len != nullptr ? min(max(__ldcg(s.len + seq), 0), s.S) : s.S;
}
// Partial results of a query row, numbered in the output's own order: `parts` of each, in part order.
// (A row that saw nothing but NaN has a NaN sum under the reference 0.)
struct Partials {
  float* o;   // [B * Sq * H][parts][128], unnormalised
  float* ml;  // [B * Sq * H][parts][2]: reference of the exponentials (-inf: nothing seen) and their sum
  int parts;
};

// ... or those of a launch that deals the keys out (attn_cache.cu): units are `keys`-key tiles, those of all units numbered
// through, and every worker has an equal range of them.  A unit in one worker's range has its results under `whole`, by row (or
// has been finished); of one that begins in a range and goes on behind it the worker's slot 1 has a part, of one that
// began before it slot 0.
struct Dealt {
  int keys;
  int slot_rows;
  int2* workers;     // [N * Hkv] first and last worker of a unit (not written for one without keys)
  float* slot_o;     // [workers][2][slot_rows][128]
  float* slot_ml;    // [workers][2][slot_rows][2]
  float* whole_o;    // [B * Sq * H][128]
  float* whole_ml;
};
// A segment's partial results, whichever they are.
struct Source {
  Segment segment;
  bool dealt;
  Partials fixed;  // parts = 0 and not dealt: nothing
  Dealt deal;
};

// Codes of four consecutive bytes as f16 pairs: (0, 1) and (2, 3).
template <int kFmt>
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (kFmt == CACHE_E4M3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
  } else {
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __floats2half2_rn(1152.f, 1152.f);
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), off), y = __hsub2(*reinterpret_cast<__half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
}

// ---- host side -------------------------------------------------------------------------------------
inline Segment segment_of(const CacheRows& c, const CacheAttnArgs& a, bool causal) {
  Segment s;
  s.N = c.N;
  s.S = c.S;
  s.n = a.B / c.N;
  s.rows = s.n * a.Sq * a.group;
  s.causal = causal ? 1 : 0;
  s.len = c.len;
  return s;
}

inline int make_rows_map(CUtensorMap* m, const CacheRows& c, bool values, int H, bool bf16, uint32_t box_rows) {
  const void* base = values ? c.v : c.k;
  const int64_t sb = values ? c.v_sb : c.k_sb, ss = values ? c.v_ss : c.k_ss, sh = values ? c.v_sh : c.k_sh;
  return c.format == CACHE_16 ? tma_host::make_bshd_map(m, base, bf16, c.N, c.S, H, 128, sb, ss, sh, box_rows)
                              : tma_host::make_bshd_bytes_map(m, base, c.N, c.S, H, sb, ss, sh, box_rows);
}
inline int make_scale_map(CUtensorMap* m, const CacheRows& c, bool values, int H, uint32_t box) {
  const uint64_t dims[4] = {static_cast<uint64_t>(c.S), static_cast<uint64_t>(H), static_cast<uint64_t>(c.N), 1};
  const uint64_t sb = static_cast<uint64_t>(values ? c.vs_sb : c.ks_sb) * 4, sh = static_cast<uint64_t>(values ? c.vs_sh : c.ks_sh) * 4;
  const uint64_t strides[3] = {sh, sb, sb};
  const uint32_t boxes[4] = {box, 1, 1, 1};
  return tma_host::make_f32_map(m, values ? c.v_scale : c.k_scale, dims, strides, boxes, false);
}

// attn_rows.cu: a segment leaves its partial results at `mine` (mine.parts of each row), or with `finish`, one part that is all there
// is, the output
int attn_rows_parts(const Segment& s, const RowShape& q, int num_sms);
cudaError_t launch_attn_rows(const CacheRows& c, const Segment& s, const CacheAttnArgs& a, const Partials& mine, bool finish,
                             bool chained, cudaStream_t stream);
// ... and the output is what the partial results of up to two segments add up to.  `finished`: units that lay in one range are the
// output already.
cudaError_t launch_attn_merge(const CacheAttnArgs& a, const Source& first, const Source& second, bool finished, int workers,
                              cudaStream_t stream);

}  // namespace asuka
