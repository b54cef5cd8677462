// Attention of new tokens over a KV cache of ragged sequences, 16 or 8 bits, and over a prefix that they share.
//
// Everything here is softmax(q K^T scale) V over the rows of a prefix and of the sequence's own cache, one softmax over
// both.  Each is a segment: N sequences, and to each (sequence, key/value head) -- a unit -- the query rows that read it: all
// heads of the group at all new positions, and for a prefix those of all sequences that share it.  A segment leaves, for every
// query row, an unnormalised output, the reference of its exponentials and their sum; the last one merges and divides.
//
// attn_stream_kernel, for up to 16 rows to a unit: the keys and values are used by so few rows that the work is one read of the
// cache, and the floor its bytes over the HBM bandwidth.  As in attn_decode.cu a unit's keys are cut into up to eight parts, the
// CTAs of a cluster, each streaming stages of 32 KB by TMA through a ring to four warps, which take their keys of a
// stage with 16x8x16 matrix instructions and a running maximum and sum of their own; the warps' and CTAs' results are merged at the
// end.  What differs: lengths are read on the device, so a part is a share of what the sequence has, and rows behind it (which may
// hold anything) count for nothing; and codes of 8 bits go from shared memory straight into matrix fragments:
//   - codes become f16, exactly (int8 as the low bits of 1024 + 128 + code, less 1152; e4m3 by conversion), and q is brought
//     to f16 too, a bf16 row times the power of two that puts its largest value in [1, 2): what is lost is below 2^-24 of it;
//   - the order of a contraction's terms is free: lane l & 3 = t takes columns 32 t .. 32 t + 31 of its keys' rows, 16 bytes at a
//     time, and the query fragments are loaded in that order; for the second product lane l >> 2 = c takes columns 16 c .. 16 c + 15
//     of four keys, whose bytes are interleaved to pairs of keys.  With the 128-byte swizzle neither read has a bank conflict;
//   - a key's scale multiplies its logits; a value's scale s multiplies the weights, w s = exp2(x) s, rounded to f16.  The reference of
//     the exponentials is the largest x + log2(s), so w s <= 1 and the rounding is 2^-11 of it (2^-25 of the largest where it is
//     subnormal).
#include "attn_cache.cuh"

namespace asuka {
namespace {

// ---- up to 16 rows to a unit -----------------------------------------------------------------------
constexpr int kRows = 16;
constexpr int kWarps = 4;
constexpr int kStreamThreads = (kWarps + 1) * 32;
constexpr int kMaxStages = 6;
constexpr int kMaxCluster = 8;
constexpr uint32_t kMergeBytes = (kWarps + 1) * kRows * 128 * 4;  // O partials of the warps and of the CTA (over the stages)
template <int kFmt> struct Stage {
  static constexpr int kWarpKeys = kFmt == CACHE_16 ? 16 : 32;
  static constexpr int kKeys = kWarps * kWarpKeys;
  static constexpr uint32_t kK = kKeys * (kFmt == CACHE_16 ? 256 : 128);  // bytes of the keys, and of the values
  static constexpr uint32_t kBytes = 2 * kK + (kFmt == CACHE_16 ? 0 : 2 * kKeys * 4);
  static constexpr uint32_t kHalf = kK / 2;  // (16 bits) one 64-column half
  static_assert(kBytes % 1024 == 0, "stages start on a swizzle atom");
};

struct StreamParams {
  Segment s;
  RowShape q;
  int stages;
  float scale_log2;
  const uint16_t* qp;
  int64_t q_sb, q_ss, q_sh;
  uint16_t* out;
  int64_t o_sb, o_ss, o_sh;
  float* lse2;
  Partials prior;  // (last segment) what the one before left; parts = 0: none
  Partials mine;   // (not the last) where to leave this one's, one part
  uint32_t* status;
};
struct StreamMaps {
  CUtensorMap k, v, ks, vs;
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void lds4(uint32_t addr, uint32_t* r) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ float2 lds2f(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
template <bool kBF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kBF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(uint32_t smem_addr, uint32_t rank) {
  uint32_t remote;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}

// Grid: units x parts, the parts of a unit a cluster.  kLast: this segment's results, with what the one before left, are the output.
template <bool kBF16, int kFmt, bool kLast>
__global__ void __launch_bounds__(kStreamThreads, 2)
attn_stream_kernel(const __grid_constant__ StreamMaps maps, const StreamParams p) {
  using St = Stage<kFmt>;
  constexpr bool k8 = kFmt != CACHE_16;
  constexpr int kSub = St::kWarpKeys / 16;  // a warp's blocks of 16 keys in a stage
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages];
  __shared__ uint32_t abort_s;
  __shared__ float warp_ml[kWarps][2][kRows];  // running reference (log2 units) and sum of every warp's rows
  __shared__ float cta_ml[2][kRows];           // the CTA's, read by the whole cluster

  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  float* merge = reinterpret_cast<float*>(smem_raw + (smem_base - smem_u32(smem_raw)));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile uint32_t* abortp = &abort_s;
  const int parts = static_cast<int>(cluster_size()), part = static_cast<int>(cluster_rank());
  const int unit = static_cast<int>(blockIdx.x) / parts;
  const int seq = unit / p.q.Hkv, hk = unit % p.q.Hkv;

  if (tid == 0) {
    abort_s = 0;
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(smem_u32(&full[i]), 1);
      mbar_init(smem_u32(&empty[i]), kWarps);
    }
    mbar_fence_init();
    tma_prefetch_desc(&maps.k);
    tma_prefetch_desc(&maps.v);
    if (k8) {
      tma_prefetch_desc(&maps.ks);
      tma_prefetch_desc(&maps.vs);
    }
  }
  __syncthreads();
  griddep_wait();
  griddep_launch_dependents();

  // this CTA's stages of what the sequence has
  const int len = seen_of(p.s, seq);
  const int n_tiles = (len + St::kKeys - 1) / St::kKeys;
  const int t_lo = static_cast<int>(static_cast<int64_t>(n_tiles) * part / parts);
  const int t_hi = static_cast<int>(static_cast<int64_t>(n_tiles) * (part + 1) / parts);

  if (warp == kWarps) {
    if (lane == 0) {
      int c = 0;
      bool ok = true;
      for (int t = t_lo; t < t_hi; ++t, ++c) {
        const int st = c % p.stages, use = c / p.stages;
        if (use > 0 && !mbar_wait(smem_u32(&empty[st]), (use - 1) & 1, abortp)) {
          atomicAdd(&p.status[0], 1u);
          p.status[1] = 81;
          ok = false;
          break;
        }
        if (use > 0) fence_proxy_async_smem();  // (the consumers' reads, behind the wait above, before the copy)
        const uint32_t bar = smem_u32(&full[st]), dst = smem_base + st * St::kBytes;
        mbar_expect_tx(bar, St::kBytes);
        tma_load_4d(dst, &maps.k, bar, 0, hk, t * St::kKeys, seq);
        if constexpr (k8) {
          tma_load_4d(dst + St::kK, &maps.v, bar, 0, hk, t * St::kKeys, seq);
          tma_load_4d(dst + 2 * St::kK, &maps.ks, bar, t * St::kKeys, hk, seq, 0);
          tma_load_4d(dst + 2 * St::kK + St::kKeys * 4, &maps.vs, bar, t * St::kKeys, hk, seq, 0);
        } else {
          tma_load_4d(dst + St::kHalf, &maps.k, bar, 64, hk, t * St::kKeys, seq);
          tma_load_4d(dst + St::kK, &maps.v, bar, 0, hk, t * St::kKeys, seq);
          tma_load_4d(dst + St::kK + St::kHalf, &maps.v, bar, 64, hk, t * St::kKeys, seq);
        }
      }
      if (!ok) {
        // give copies already in flight a bounded chance to land before the CTA retires
        volatile uint32_t none = 0;
        for (int x = c > p.stages ? c - p.stages : 0; x < c; ++x)
          mbar_wait(smem_u32(&full[x % p.stages]), (x / p.stages) & 1, &none);
      }
    }
    __syncwarp();
  } else {
    // Query rows of this thread: r0 and r0 + 8 of the tile, as matrix fragments (in the order of terms that the keys' have).
    const int r0 = lane >> 2, t4 = lane & 3;
    uint32_t qf[8][4];
    int lim[2];      // last visible key of either row
    float mul[2];    // of a dot product, to a logit in log2 units
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = r0 + 8 * x;
      const Row row = decode_row(min(r, p.s.rows - 1), seq, hk, p.s, p.q);
      lim[x] = p.s.causal ? min(len - 1, row.pos + len - p.q.Sq) : len - 1;
      mul[x] = p.scale_log2;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(p.qp + row.b * p.q_sb + row.pos * p.q_ss + row.h * p.q_sh);
      const bool live = r < p.s.rows;
      if constexpr (!k8) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          qf[kk][x] = live ? __ldg(src + t4 + kk * 8) : 0u;
          qf[kk][2 + x] = live ? __ldg(src + t4 + kk * 8 + 4) : 0u;
        }
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint4 w = live ? __ldg(reinterpret_cast<const uint4*>(src) + t4 * 4 + c) : make_uint4(0, 0, 0, 0);
          qf[2 * c][x] = w.x;
          qf[2 * c][2 + x] = w.y;
          qf[2 * c + 1][x] = w.z;
          qf[2 * c + 1][2 + x] = w.w;
        }
        if constexpr (kBF16) {
          float top = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 v = unpack2<true>(qf[i >> 1][(i & 1) * 2 + x]);
            top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          // (rows of zeros, and of nothing but values under 2^-100, stay as they are or vanish)
          const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23), 27), 253);
          const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
          mul[x] *= __uint_as_float(static_cast<uint32_t>(e) << 23);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            uint32_t& w = qf[i >> 1][(i & 1) * 2 + x];
            const float2 v = unpack2<true>(w);
            w = pack2<false>(v.x * down, v.y * down);
          }
        }
      }
    }
    // (no row's limit is below the first's)
    const int min_lim = p.s.causal ? min(len - 1, len - p.q.Sq) : len - 1;

    float o[16][4];
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // l: this thread's columns only
    bool ok = true;

    int c = 0;
    for (int t = t_lo; t < t_hi; ++t, ++c) {
      const int st = c % p.stages;
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&full[st]), (c / p.stages) & 1, abortp));
      if (!ok) {
        if (lane == 0) {
          atomicAdd(&p.status[0], 1u);
          p.status[1] = 82;
        }
        break;
      }
      const uint32_t sK = smem_base + st * St::kBytes, sV = sK + St::kK, sKs = sV + St::kK, sVs = sKs + St::kKeys * 4;
      const int wkey = warp * St::kWarpKeys;   // this warp's first key in the stage
      const int key0 = t * St::kKeys + wkey;   // ... and in the sequence
      const bool ragged = key0 + St::kWarpKeys > len;
      // s[j][e]: row r0 (e < 2) or r0 + 8, key 8 j + 2 t4 + (e & 1)
      float s[2 * kSub][4];
#pragma unroll
      for (int j = 0; j < 2 * kSub; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
      float2 vs[2 * kSub];
      if constexpr (k8) {
#pragma unroll
        for (int j = 0; j < 2 * kSub; ++j) {
          uint32_t w[8];
          lds4(sK + sw128_offset(wkey + 8 * j + r0, 2 * t4), w);
          lds4(sK + sw128_offset(wkey + 8 * j + r0, 2 * t4 + 1), w + 4);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            uint32_t b0, b1;
            codes_to_f16<kFmt>(w[kk], b0, b1);
            mma16816<false>(s[j], qf[kk], b0, b1);
          }
        }
#pragma unroll
        for (int j = 0; j < 2 * kSub; ++j) {
          const float2 ks = lds2f(sKs + (wkey + 8 * j + 2 * t4) * 4);
          vs[j] = lds2f(sVs + (wkey + 8 * j + 2 * t4) * 4);
          s[j][0] *= ks.x * mul[0];
          s[j][1] *= ks.y * mul[0];
          s[j][2] *= ks.x * mul[1];
          s[j][3] *= ks.y * mul[1];
        }
      } else {
        // addresses of this lane's rows for the 8x8 blocks: keys of the warp's 16, 16-byte chunk of a row
        const int k_row = wkey + ((lane >> 4) << 3) + (lane & 7), k_chunk = (lane >> 3) & 1;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          uint32_t kf[4];  // keys 0-7: k 0-7, 8-15; keys 8-15: k 0-7, 8-15
          ldsm4(sK + (kk >> 2) * St::kHalf + sw128_offset(k_row, (kk & 3) * 2 + k_chunk), kf);
          mma16816<kBF16>(s[0], qf[kk], kf[0], kf[1]);
          mma16816<kBF16>(s[1], qf[kk], kf[2], kf[3]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[j][e] *= mul[0];
      }
      if (key0 + St::kWarpKeys - 1 > min_lim) {
#pragma unroll
        for (int j = 0; j < 2 * kSub; ++j) {
          const int key = key0 + 8 * j + 2 * t4;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key + (e & 1) > lim[e >> 1]) s[j][e] = -INFINITY;
          if constexpr (k8) {
            if (key >= len) vs[j].x = 0.f;
            if (key + 1 >= len) vs[j].y = 0.f;
          }
        }
      }
      float w[2];
      {
        float2 lv[2 * kSub];  // log2 of the values' scales
        if constexpr (k8) {
#pragma unroll
          for (int j = 0; j < 2 * kSub; ++j)
            lv[j] = make_float2(lg2(fmaxf(fabsf(vs[j].x), 0x1p-100f)), lg2(fmaxf(fabsf(vs[j].y), 0x1p-100f)));
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float mx = m[x];
#pragma unroll
          for (int j = 0; j < 2 * kSub; ++j) {
            if constexpr (k8) mx = fmaxf(mx, fmaxf(s[j][2 * x] + lv[j].x, s[j][2 * x + 1] + lv[j].y));
            else mx = fmaxf(mx, fmaxf(s[j][2 * x], s[j][2 * x + 1]));
          }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float ref = mx > -INFINITY ? mx : 0.f;
          w[x] = ex2(m[x] - ref);
          m[x] = mx;
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < 2 * kSub; ++j) {
            s[j][2 * x] = ex2(s[j][2 * x] - ref);
            s[j][2 * x + 1] = ex2(s[j][2 * x + 1] - ref);
            sum += s[j][2 * x] + s[j][2 * x + 1];
          }
          l[x] = l[x] * w[x] + sum;
        }
      }
      if (__any_sync(0xffffffffu, w[0] != 1.f || w[1] != 1.f)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          o[i][0] *= w[0];
          o[i][1] *= w[0];
          o[i][2] *= w[1];
          o[i][3] *= w[1];
        }
      }
#pragma unroll
      for (int u = 0; u < kSub; ++u) {
        const int kb = wkey + 16 * u;  // block of 16 keys
        uint32_t pf[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = 2 * u + (e >> 1), x = 2 * (e & 1);
          if constexpr (k8) pf[e] = pack2<false>(s[j][x] * vs[j].x, s[j][x + 1] * vs[j].y);
          else pf[e] = pack2<kBF16>(s[j][x], s[j][x + 1]);
        }
        if constexpr (k8) {
          uint32_t v[4][4];  // keys 2 t4, 2 t4 + 1, 8 + 2 t4, 9 + 2 t4 of the block, 16 columns each
#pragma unroll
          for (int i = 0; i < 4; ++i) lds4(sV + sw128_offset(kb + (i >> 1) * 8 + 2 * t4 + (i & 1), r0), v[i]);
          if (ragged) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (t * St::kKeys + kb + (i >> 1) * 8 + 2 * t4 + (i & 1) >= len) v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0u;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t b0[4], b1[4];  // columns 4 i .. 4 i + 3
            codes_to_f16<kFmt>(__byte_perm(v[0][i], v[1][i], 0x5140), b0[0], b0[1]);
            codes_to_f16<kFmt>(__byte_perm(v[0][i], v[1][i], 0x7362), b0[2], b0[3]);
            codes_to_f16<kFmt>(__byte_perm(v[2][i], v[3][i], 0x5140), b1[0], b1[1]);
            codes_to_f16<kFmt>(__byte_perm(v[2][i], v[3][i], 0x7362), b1[2], b1[3]);
#pragma unroll
            for (int x = 0; x < 4; ++x) mma16816<false>(o[4 * i + x], pf, b0[x], b1[x]);
          }
        } else {
          const int v_row = kb + (((lane >> 3) & 1) << 3) + (lane & 7), v_chunk = lane >> 4;
          uint32_t keep[2] = {0xffffffffu, 0xffffffffu};  // (what lies behind the sequence may be infinite or NaN)
          if (ragged) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int key = key0 + 8 * x + 2 * t4;
              keep[x] = (key < len ? 0xffffu : 0u) | (key + 1 < len ? 0xffff0000u : 0u);
            }
          }
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            uint32_t vf[4];  // columns 16d + 0-7: keys 0-7, 8-15; columns 16d + 8-15: keys 0-7, 8-15
            ldsm4_t(sV + (d >> 2) * St::kHalf + sw128_offset(v_row, (d & 3) * 2 + v_chunk), vf);
            mma16816<kBF16>(o[2 * d], pf, vf[0] & keep[0], vf[1] & keep[1]);
            mma16816<kBF16>(o[2 * d + 1], pf, vf[2] & keep[0], vf[3] & keep[1]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&empty[st]));
    }
    if (!ok) *abortp = 1u;
    // row sums over the four threads of a row
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
      if (t4 == 0) {
        warp_ml[warp][0][r0 + 8 * x] = m[x];
        warp_ml[warp][1][r0 + 8 * x] = l[x];
      }
    }
    // every warp has consumed every stage (and so every copy has landed): the ring becomes the
    // merge buffer
    named_bar_sync(1, kWarps * 32);
    float* mine = merge + warp * (kRows * 128);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float* row = mine + (r0 + 8 * x) * 128;
      if constexpr (k8) {
        // o[i]: columns 32 t4 + i and 32 t4 + 16 + i
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          *reinterpret_cast<float4*>(row + 32 * t4 + i) = make_float4(o[i][2 * x], o[i + 1][2 * x], o[i + 2][2 * x], o[i + 3][2 * x]);
          *reinterpret_cast<float4*>(row + 32 * t4 + 16 + i) =
              make_float4(o[i][2 * x + 1], o[i + 1][2 * x + 1], o[i + 2][2 * x + 1], o[i + 3][2 * x + 1]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          *reinterpret_cast<float2*>(row + i * 8 + 2 * t4) = make_float2(o[i][2 * x], o[i][2 * x + 1]);
      }
    }
    named_bar_sync(1, kWarps * 32);
    // the four warps' partial results to one per CTA, in warp order; thread = output column
    float* cta = merge + kWarps * (kRows * 128);
    for (int r = 0; r < p.s.rows; ++r) {
      float mm = -INFINITY;
#pragma unroll
      for (int x = 0; x < kWarps; ++x) mm = fmaxf(mm, warp_ml[x][0][r]);
      float acc = 0.f, ll = 0.f;
#pragma unroll
      for (int x = 0; x < kWarps; ++x) {
        const float wt = warp_ml[x][0][r] > -INFINITY ? ex2(warp_ml[x][0][r] - mm) : 0.f;
        acc = fmaf(wt, merge[x * (kRows * 128) + r * 128 + tid], acc);
        ll = fmaf(wt, warp_ml[x][1][r], ll);
      }
      cta[r * 128 + tid] = acc;
      if (tid == 0) {
        cta_ml[0][r] = mm;
        cta_ml[1][r] = ll;
      }
    }
  }

  // ---- merge over the cluster, in rank order; row r is finished by the CTA of rank r mod parts
  cluster_sync();
  if (warp < kWarps) {
    const uint32_t cta_addr = smem_base + kWarps * (kRows * 128) * 4;
    for (int r = part; r < p.s.rows; r += parts) {
      float pm[kMaxCluster], pl[kMaxCluster], po[kMaxCluster];
#pragma unroll
      for (int x = 0; x < kMaxCluster; ++x) {
        if (x < parts) {
          pm[x] = ld_cluster(smem_u32(&cta_ml[0][r]), x);
          pl[x] = ld_cluster(smem_u32(&cta_ml[1][r]), x);
          po[x] = ld_cluster(cta_addr + (r * 128 + tid) * 4, x);
        }
      }
      float mm = -INFINITY, ll = 0.f, acc = 0.f;
#pragma unroll
      for (int x = 0; x < kMaxCluster; ++x)
        if (x < parts) mm = fmaxf(mm, pm[x]);
#pragma unroll
      for (int x = 0; x < kMaxCluster; ++x) {
        if (x < parts) {
          const float wt = pm[x] > -INFINITY ? ex2(pm[x] - mm) : 0.f;
          ll = fmaf(wt, pl[x], ll);
          acc = fmaf(wt, po[x], acc);
        }
      }
      const Row row = decode_row(r, seq, hk, p.s, p.q);
      const int64_t number = (static_cast<int64_t>(row.b) * p.q.Sq + row.pos) * p.q.H + row.h;
      if constexpr (!kLast) {
        if (!(mm > -INFINITY) && ll != 0.f) mm = 0.f;  // (nothing but NaN: the sum)
        p.mine.o[number * 128 + tid] = acc;
        if (tid == 0) *reinterpret_cast<float2*>(p.mine.ml + number * 2) = make_float2(mm, ll);
      } else {
        for (int x = 0; x < p.prior.parts; ++x) {
          const float2 ml = *reinterpret_cast<const float2*>(p.prior.ml + (number * p.prior.parts + x) * 2);
          const float other = p.prior.o[(number * p.prior.parts + x) * 128 + tid];
          if (ml.x > -INFINITY) {
            const float top = fmaxf(mm, ml.x), w0 = ex2(mm - top), w1 = ex2(ml.x - top);
            ll = fmaf(w1, ml.y, ll * w0);
            acc = fmaf(w1, other, acc * w0);
            mm = top;
          }
        }
        const float y = ll == 0.f ? 0.f : acc / ll;
        const float hi = __shfl_down_sync(0xffffffffu, y, 1);
        if ((tid & 1) == 0)
          *reinterpret_cast<uint32_t*>(p.out + row.b * p.o_sb + row.pos * p.o_ss + row.h * p.o_sh + tid) = pack2<kBF16>(y, hi);
        if (p.lse2 != nullptr && tid == 0)
          p.lse2[(static_cast<int64_t>(row.b) * p.q.H + row.h) * p.q.Sq + row.pos] = mm + log2f(ll);
      }
    }
  }
  cluster_sync();  // no CTA leaves while another still reads its shared memory
}

template <int kFmt, bool kLast>
cudaError_t launch_stream_fmt(const CacheRows& c, StreamParams& p, bool bf16, int num_sms, cudaStream_t stream) {
  using St = Stage<kFmt>;
  StreamMaps maps;
  if (make_rows_map(&maps.k, c, false, p.q.Hkv, bf16, St::kKeys) || make_rows_map(&maps.v, c, true, p.q.Hkv, bf16, St::kKeys))
    return cudaErrorInvalidValue;
  if (kFmt != CACHE_16) {
    if (make_scale_map(&maps.ks, c, false, p.q.Hkv, St::kKeys) || make_scale_map(&maps.vs, c, true, p.q.Hkv, St::kKeys))
      return cudaErrorInvalidValue;
  } else {
    maps.ks = maps.vs = maps.k;
  }
  // Parts: as many as bring the launch to two CTAs per SM (what fits side by side), at least two stages each.
  const long long units = static_cast<long long>(p.s.N) * p.q.Hkv;
  const int n_tiles = (p.s.S + St::kKeys - 1) / St::kKeys;
  int parts = 1;
  while (parts < kMaxCluster && units * parts * 2 <= 2LL * num_sms && n_tiles >= parts * 4) parts *= 2;
  // Two CTAs per SM share its memory; a launch that gives every SM one at most takes the whole of it.
  p.stages = units * parts > num_sms ? 3 : kMaxStages;
  const uint32_t smem = (p.stages * St::kBytes > kMergeBytes ? p.stages * St::kBytes : kMergeBytes) + 1024;
  const auto kern = bf16 ? attn_stream_kernel<true, kFmt, kLast> : attn_stream_kernel<false, kFmt, kLast>;
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), kMaxStages * St::kBytes + 1024);
  if (e != cudaSuccess) return e;
  e = launch_dependent_cluster(kern, dim3(static_cast<unsigned>(units * parts)), dim3(kStreamThreads), smem,
                               static_cast<unsigned>(parts), stream, maps, p);
  count_launch();
  return e;
}

template <bool kLast>
cudaError_t launch_stream(const CacheRows& c, StreamParams& p, bool bf16, int num_sms, cudaStream_t stream) {
  switch (c.format) {
    case CACHE_I8: return launch_stream_fmt<CACHE_I8, kLast>(c, p, bf16, num_sms, stream);
    case CACHE_E4M3: return launch_stream_fmt<CACHE_E4M3, kLast>(c, p, bf16, num_sms, stream);
    default: return launch_stream_fmt<CACHE_16, kLast>(c, p, bf16, num_sms, stream);
  }
}

// Query rows are few enough for the stream's one 16-row tile.
bool streams(const Segment& s) { return s.rows <= kRows; }

// How the work of a call is cut: the prefix's partial results first in the workspace, then the own rows', where those do not
// finish it themselves.
struct Plan {
  Segment prefix, own;
  int prefix_parts, own_parts;  // 0: none kept
};
Plan plan_of(const CacheAttnArgs& a, int num_sms) {
  const RowShape q{a.Sq, a.H, a.H / a.group, a.group};
  Plan x;
  x.own = segment_of(a.own, a, a.causal != 0);
  x.own_parts = streams(x.own) ? 0 : attn_rows_parts(x.own, q, num_sms);
  x.prefix_parts = 0;
  if (a.prefix.N > 0) {
    x.prefix = segment_of(a.prefix, a, false);
    x.prefix_parts = streams(x.prefix) ? 1 : attn_rows_parts(x.prefix, q, num_sms);
  }
  return x;
}
size_t row_count(const CacheAttnArgs& a) { return static_cast<size_t>(a.B) * a.Sq * a.H; }
size_t partial_bytes(const CacheAttnArgs& a, int parts) {
  return (row_count(a) * parts * (128 + 2) * sizeof(float) + 255) / 256 * 256;
}
Partials partials_at(void* ws, const CacheAttnArgs& a, int parts) {
  Partials x;
  x.parts = parts;
  x.o = static_cast<float*>(ws);
  x.ml = x.o + row_count(a) * parts * 128;
  return x;
}

}  // namespace

size_t attn_cache_ws_bytes(const CacheAttnArgs& a, int num_sms) {
  const Plan x = plan_of(a, num_sms);
  return partial_bytes(a, x.prefix_parts) + partial_bytes(a, x.own_parts);
}

cudaError_t launch_attn_cache(const CacheAttnArgs& a, void* ws, int num_sms, cudaStream_t stream) {
  const Plan x = plan_of(a, num_sms);
  const Partials first = partials_at(ws, a, x.prefix_parts);
  StreamParams p;
  p.q = RowShape{a.Sq, a.H, a.H / a.group, a.group};
  p.scale_log2 = a.softmax_scale * 1.4426950408889634f;
  p.qp = a.q;
  p.q_sb = a.q_sb; p.q_ss = a.q_ss; p.q_sh = a.q_sh;
  p.out = a.out;
  p.o_sb = a.o_sb; p.o_ss = a.o_ss; p.o_sh = a.o_sh;
  p.lse2 = a.lse2;
  p.status = device_status_words();
  p.prior = p.mine = first;
  cudaError_t e = cudaSuccess;
  if (x.prefix_parts > 0) {
    p.s = x.prefix;
    e = streams(x.prefix) ? launch_stream<false>(a.prefix, p, a.bf16, num_sms, stream)
                          : launch_attn_rows(a.prefix, x.prefix, a, first, num_sms, stream);
    if (e != cudaSuccess) return e;
  }
  if (x.own_parts == 0) {
    p.s = x.own;
    return launch_stream<true>(a.own, p, a.bf16, num_sms, stream);
  }
  const Partials second = partials_at(static_cast<uint8_t*>(ws) + partial_bytes(a, x.prefix_parts), a, x.own_parts);
  e = launch_attn_rows(a.own, x.own, a, second, num_sms, stream);
  return e != cudaSuccess ? e : launch_attn_merge(a, first, second, stream);
}

}  // namespace asuka
