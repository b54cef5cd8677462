// Attention of new tokens over a KV cache of ragged sequences, 16 or 8 bits, and over a prefix that they share.
//
// Everything here is softmax(q K^T scale) V over the rows of a prefix and of the sequence's own cache, one softmax over
// both.  Each is a segment: N sequences, and to each (sequence, key/value head) -- a unit -- the query rows that read it: all
// heads of the group at all new positions, and for a prefix those of all sequences that share it.  A segment leaves, for every
// query row, an unnormalised output, the reference of its exponentials and their sum; the last one merges and divides.
//
// attn_stream_kernel, for up to 16 rows to a unit: the keys and values are used by so few rows that the work is one read of the
// cache, and the floor its bytes over the HBM bandwidth.  Sequences are of any lengths, known on the device only, and units may be
// many and short or few and long; so the work is dealt out there:
//   - a unit's keys are tiles of 32 (8 bits) or 16 (16 bits), 8 KB of keys and values, and the tiles of all units of all segments are
//     numbered through.  Every warp of the launch is a worker with an equal, contiguous range of them, which may begin and end
//     inside a unit: no SM waits for the longest sequence, and a warp waits for no other;
//   - a warp fetches its own tiles by TMA into a ring of its own, across the ends of units, and works on them with 16x8x16 matrix
//     instructions and a running maximum and sum;
//   - a unit that lies in one range is finished there; what a range has of a unit that others share goes to the workspace
//     and is merged by attn_merge_kernel in the order of the keys, so results do not depend on which warp was first.
// Codes of 8 bits go from shared memory straight into matrix fragments:
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
constexpr int kWarps = 12;   // workers of a CTA, one CTA to an SM
constexpr int kStages = 2;   // of each worker's ring
constexpr int kThreads = kWarps * 32;
constexpr int kMinTiles = 2;  // a worker's share is no less
template <int kFmt> struct Tile {
  static constexpr int kKeys = kFmt == CACHE_16 ? 16 : 32;
  static constexpr uint32_t kHalf = 2048;                  // (16 bits) one 64-column half of the keys or values
  static constexpr uint32_t kK = 4096;                     // the keys, and the values
  static constexpr uint32_t kScales = kFmt == CACHE_16 ? 0 : 2 * kKeys * 4;
};
constexpr uint32_t kTileBytes = 8192;

struct StreamParams {
  Segment s[2];    // numbered through in this order
  int segments;
  RowShape q;
  float scale_log2;
  const uint16_t* qp;
  int64_t q_sb, q_ss, q_sh;
  uint16_t* out;
  int64_t o_sb, o_ss, o_sh;
  float* lse2;
  int finish;      // whole units are the output (no other segment)
  Dealt deal[2];
  uint32_t* status;
};
struct StreamMaps {
  struct {
    CUtensorMap k, v, ks, vs;
  } s[2];
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
// Where a worker is: a tile of a unit.
struct Cursor {
  int seg, seq, hk, tile;
  int len, tiles;  // of the sequence
};

// One CTA to an SM; a warp is a worker.
template <bool kBF16, int kFmt>
__global__ void __launch_bounds__(kThreads, 1)
attn_stream_kernel(const __grid_constant__ StreamMaps maps, const StreamParams p) {
  using T = Tile<kFmt>;
  constexpr bool k8 = kFmt != CACHE_16;
  constexpr int kSub = T::kKeys / 16;  // blocks of 16 keys in a tile
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[kWarps][kStages];
  __shared__ uint32_t abort_s;
  __shared__ int64_t ahead_s[kThreads];  // tiles ahead of a thread's sequences
  __shared__ int64_t warp_sum_s[kWarps];

  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile uint32_t* abortp = &abort_s;

  if (tid == 0) abort_s = 0;
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(smem_u32(&full[warp][i]), 1);
    mbar_fence_init();
    for (int x = 0; x < p.segments; ++x) {
      tma_prefetch_desc(&maps.s[x].k);
      tma_prefetch_desc(&maps.s[x].v);
    }
  }
  griddep_wait();
  griddep_launch_dependents();

  // ---- the deal: every CTA adds up the tiles of all sequences (a thread has `per` consecutive ones)
  const int n_seqs = p.s[0].N + (p.segments > 1 ? p.s[1].N : 0);
  auto at = [&](int i, Cursor& c) {  // sequence i of all segments
    c.seg = i >= p.s[0].N ? 1 : 0;
    c.seq = i - (c.seg ? p.s[0].N : 0);
    c.len = seen_of(p.s[c.seg], c.seq);
    c.tiles = (c.len + T::kKeys - 1) / T::kKeys;
  };
  const int per = (n_seqs + kThreads - 1) / kThreads;
  int64_t mine = 0;
  for (int i = tid * per; i < min(n_seqs, (tid + 1) * per); ++i) {
    Cursor c;
    at(i, c);
    mine += static_cast<int64_t>(c.tiles) * p.q.Hkv;
  }
  int64_t upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += x;
  }
  if (lane == 31) warp_sum_s[warp] = upto;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int x = 0; x < kWarps; ++x) {
    if (x < warp) before += warp_sum_s[x];
    total += warp_sum_s[x];
  }
  ahead_s[tid] = before + upto - mine;
  const int64_t workers = static_cast<int64_t>(gridDim.x) * kWarps;
  const int64_t share = max((total + workers - 1) / workers, static_cast<int64_t>(kMinTiles));
  __syncthreads();

  // (neighbours in the numbering on different SMs, so that a small launch uses all of them)
  const int64_t worker = static_cast<int64_t>(warp) * gridDim.x + blockIdx.x;
  const int64_t lo = worker * share;
  const int count = static_cast<int>(min(share, total - lo));  // (a worker's tiles are 8 KB each: far below 2^31)
  if (count <= 0) return;

  Cursor c;
  {
    int x = 0;  // the last thread whose sequences begin at or before the range
    for (int step = 256; step > 0; step >>= 1)
      if (x + step < kThreads && ahead_s[x + step] <= lo) x += step;
    int i = x * per;
    int64_t rest = lo - ahead_s[x];
    for (;; ++i) {  // (bounded, should another stream change the lengths in between)
      at(i, c);
      const int64_t in_seq = static_cast<int64_t>(c.tiles) * p.q.Hkv;
      if (rest < in_seq || i + 1 == n_seqs) break;
      rest -= in_seq;
    }
    c.tiles = max(c.tiles, 1);
    c.hk = static_cast<int>(min(rest / c.tiles, static_cast<int64_t>(p.q.Hkv - 1)));
    c.tile = static_cast<int>(rest % c.tiles);
  }
  auto advance = [&](Cursor& x) {  // (only where a tile follows)
    if (++x.tile < x.tiles) return;
    x.tile = 0;
    if (++x.hk < p.q.Hkv) return;
    x.hk = 0;
    int i = x.seq + (x.seg ? p.s[0].N : 0);
    while (i + 1 < n_seqs) {
      at(++i, x);
      if (x.tiles > 0) break;
    }
  };

  const uint32_t ring = smem_base + warp * kStages * kTileBytes;
  const uint32_t scales = smem_base + kWarps * kStages * kTileBytes + warp * kStages * T::kScales;
  auto fetch = [&](const Cursor& x, int st) {
    const uint32_t bar = smem_u32(&full[warp][st]), dst = ring + st * kTileBytes;
    const auto& m = maps.s[x.seg];
    const int key = x.tile * T::kKeys;
    mbar_expect_tx(bar, kTileBytes + T::kScales);
    tma_load_4d(dst, &m.k, bar, 0, x.hk, key, x.seq);
    if constexpr (k8) {
      tma_load_4d(dst + T::kK, &m.v, bar, 0, x.hk, key, x.seq);
      tma_load_4d(scales + st * T::kScales, &m.ks, bar, key, x.hk, x.seq, 0);
      tma_load_4d(scales + st * T::kScales + T::kKeys * 4, &m.vs, bar, key, x.hk, x.seq, 0);
    } else {
      tma_load_4d(dst + T::kHalf, &m.k, bar, 64, x.hk, key, x.seq);
      tma_load_4d(dst + T::kK, &m.v, bar, 0, x.hk, key, x.seq);
      tma_load_4d(dst + T::kK + T::kHalf, &m.v, bar, 64, x.hk, key, x.seq);
    }
  };

  Cursor ahead = c;  // the next tile to fetch
  int fetched = 0;
  for (; fetched < kStages && fetched < count; ++fetched) {
    if (lane == 0) fetch(ahead, fetched);
    if (fetched + 1 < count) advance(ahead);
  }

  const int r0 = lane >> 2, t4 = lane & 3;  // query rows of this thread: r0 and r0 + 8 of the unit's 16
  uint32_t qf[8][4];                        // as matrix fragments (in the order of terms that the keys' have)
  int lim[2];                               // last visible key of either row
  int min_lim = 0;                          // no row's is below this
  float mul[2];                             // of a dot product, to a logit in log2 units
  float o[16][4], m[2], l[2];               // (l: this thread's columns only)
  int first = 0;                            // the unit's first tile in this range
  bool ok = true, begin = true;

  for (int n = 0; n < count; ++n) {
    if (begin) {  // a unit begins, or this range of it
      begin = false;
      first = c.tile;
      const Segment& s = p.s[c.seg];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = r0 + 8 * x;
        const Row row = decode_row(min(r, s.rows - 1), c.seq, c.hk, s, p.q);
        lim[x] = s.causal ? min(c.len - 1, row.pos + c.len - p.q.Sq) : c.len - 1;
        mul[x] = p.scale_log2;
        m[x] = -INFINITY;
        l[x] = 0.f;
        const uint32_t* src = reinterpret_cast<const uint32_t*>(p.qp + row.b * p.q_sb + row.pos * p.q_ss + row.h * p.q_sh);
        const bool live = r < s.rows;
        if constexpr (!k8) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            qf[kk][x] = live ? __ldg(src + t4 + kk * 8) : 0u;
            qf[kk][2 + x] = live ? __ldg(src + t4 + kk * 8 + 4) : 0u;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4 w = live ? __ldg(reinterpret_cast<const uint4*>(src) + t4 * 4 + i) : make_uint4(0, 0, 0, 0);
            qf[2 * i][x] = w.x;
            qf[2 * i][2 + x] = w.y;
            qf[2 * i + 1][x] = w.z;
            qf[2 * i + 1][2 + x] = w.w;
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
      min_lim = s.causal ? min(c.len - 1, c.len - p.q.Sq) : c.len - 1;
      if (first == 0 && lane == 0) {
        const int rest = c.tiles - (count - n);  // behind this worker's range
        p.deal[c.seg].workers[static_cast<int64_t>(c.seq) * p.q.Hkv + c.hk] =
            make_int2(static_cast<int>(worker), static_cast<int>(worker + (rest > 0 ? (rest + share - 1) / share : 0)));
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    }

    const int st = n % kStages;
    ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&full[warp][st]), (n / kStages) & 1, abortp));
    if (!ok) {
      if (lane == 0) {
        atomicAdd(&p.status[0], 1u);
        p.status[1] = 82;
      }
      break;
    }
    const uint32_t sK = ring + st * kTileBytes, sV = sK + T::kK, sKs = scales + st * T::kScales, sVs = sKs + T::kKeys * 4;
    const int key0 = c.tile * T::kKeys;
    const bool ragged = key0 + T::kKeys > c.len;
    // s[j][e]: row r0 (e < 2) or r0 + 8, key 8 j + 2 t4 + (e & 1)
    float s[2 * kSub][4];
#pragma unroll
    for (int j = 0; j < 2 * kSub; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
    float2 vs[2 * kSub];
    if constexpr (k8) {
#pragma unroll
      for (int j = 0; j < 2 * kSub; ++j) {
        uint32_t w[8];
        lds4(sK + sw128_offset(8 * j + r0, 2 * t4), w);
        lds4(sK + sw128_offset(8 * j + r0, 2 * t4 + 1), w + 4);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          uint32_t b0, b1;
          codes_to_f16<kFmt>(w[kk], b0, b1);
          mma16816<false>(s[j], qf[kk], b0, b1);
        }
      }
#pragma unroll
      for (int j = 0; j < 2 * kSub; ++j) {
        const float2 ks = lds2f(sKs + (8 * j + 2 * t4) * 4);
        vs[j] = lds2f(sVs + (8 * j + 2 * t4) * 4);
        s[j][0] *= ks.x * mul[0];
        s[j][1] *= ks.y * mul[0];
        s[j][2] *= ks.x * mul[1];
        s[j][3] *= ks.y * mul[1];
      }
    } else {
      // addresses of this lane's rows for the 8x8 blocks: keys of the tile's 16, 16-byte chunk of a row
      const int k_row = ((lane >> 4) << 3) + (lane & 7), k_chunk = (lane >> 3) & 1;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        uint32_t kf[4];  // keys 0-7: k 0-7, 8-15; keys 8-15: k 0-7, 8-15
        ldsm4(sK + (kk >> 2) * T::kHalf + sw128_offset(k_row, (kk & 3) * 2 + k_chunk), kf);
        mma16816<kBF16>(s[0], qf[kk], kf[0], kf[1]);
        mma16816<kBF16>(s[1], qf[kk], kf[2], kf[3]);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] *= mul[0];
    }
    if (key0 + T::kKeys - 1 > min_lim) {
#pragma unroll
      for (int j = 0; j < 2 * kSub; ++j) {
        const int key = key0 + 8 * j + 2 * t4;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (key + (e & 1) > lim[e >> 1]) s[j][e] = -INFINITY;
        if constexpr (k8) {
          if (key >= c.len) vs[j].x = 0.f;
          if (key + 1 >= c.len) vs[j].y = 0.f;
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
      const int kb = 16 * u;  // block of 16 keys
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
            if (key0 + kb + (i >> 1) * 8 + 2 * t4 + (i & 1) >= c.len) v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0u;
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
            keep[x] = (key < c.len ? 0xffffu : 0u) | (key + 1 < c.len ? 0xffff0000u : 0u);
          }
        }
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          uint32_t vf[4];  // columns 16d + 0-7: keys 0-7, 8-15; columns 16d + 8-15: keys 0-7, 8-15
          ldsm4_t(sV + (d >> 2) * T::kHalf + sw128_offset(v_row, (d & 3) * 2 + v_chunk), vf);
          mma16816<kBF16>(o[2 * d], pf, vf[0] & keep[0], vf[1] & keep[1]);
          mma16816<kBF16>(o[2 * d + 1], pf, vf[2] & keep[0], vf[3] & keep[1]);
        }
      }
    }
    __syncwarp();
    if (fetched < count) {
      if (lane == 0) {
        fence_proxy_async_smem();  // (the warp's reads of the stage before the copy)
        fetch(ahead, st);
      }
      ++fetched;
      if (fetched < count) advance(ahead);
    }

    if (c.tile + 1 == c.tiles || n + 1 == count) {
      // ---- the unit ends, or this range of it
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
      }
      const Segment& sg = p.s[c.seg];
      const bool whole = first == 0 && c.tile + 1 == c.tiles;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = r0 + 8 * x;
        if (r >= sg.rows) continue;
        const Row row = decode_row(r, c.seq, c.hk, sg, p.q);
        if (whole && p.finish) {
          const float inv = l[x] == 0.f ? 0.f : 1.f / l[x];
          uint16_t* dst = p.out + row.b * p.o_sb + row.pos * p.o_ss + row.h * p.o_sh;
          if constexpr (k8) {  // o[i]: columns 32 t4 + i and 32 t4 + 16 + i
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
              for (int i = 0; i < 16; i += 8) {
                uint32_t v[4];
#pragma unroll
                for (int z = 0; z < 4; ++z)
                  v[z] = pack2<kBF16>(o[i + 2 * z][2 * x + y] * inv, o[i + 2 * z + 1][2 * x + y] * inv);
                *reinterpret_cast<uint4*>(dst + 32 * t4 + 16 * y + i) = make_uint4(v[0], v[1], v[2], v[3]);
              }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              *reinterpret_cast<uint32_t*>(dst + i * 8 + 2 * t4) = pack2<kBF16>(o[i][2 * x] * inv, o[i][2 * x + 1] * inv);
          }
          if (p.lse2 != nullptr && t4 == 0)
            p.lse2[(static_cast<int64_t>(row.b) * p.q.H + row.h) * p.q.Sq + row.pos] = m[x] + log2f(l[x]);
          continue;
        }
        const Dealt& d = p.deal[c.seg];
        const int64_t number = (static_cast<int64_t>(row.b) * p.q.Sq + row.pos) * p.q.H + row.h;
        const int64_t slot = (worker * 2 + (first > 0 ? 0 : 1)) * d.slot_rows + r;
        float* dst = whole ? d.whole_o + number * 128 : d.slot_o + slot * 128;
        float* ml = whole ? d.whole_ml + number * 2 : d.slot_ml + slot * 2;
        if constexpr (k8) {
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              *reinterpret_cast<float4*>(dst + 32 * t4 + 16 * y + i) =
                  make_float4(o[i][2 * x + y], o[i + 1][2 * x + y], o[i + 2][2 * x + y], o[i + 3][2 * x + y]);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) *reinterpret_cast<float2*>(dst + i * 8 + 2 * t4) = make_float2(o[i][2 * x], o[i][2 * x + 1]);
        }
        if (t4 == 0) {
          const float ref = m[x] > -INFINITY || l[x] == 0.f ? m[x] : 0.f;  // (nothing but NaN: the sum)
          *reinterpret_cast<float2*>(ml) = make_float2(ref, l[x]);
        }
      }
      begin = true;
    }
    if (n + 1 < count) advance(c);
  }
  if (!ok) {
    // give copies already in flight a bounded chance to land before the CTA retires
    volatile uint32_t none = 0;
    for (int n = fetched > kStages ? fetched - kStages : 0; n < fetched; ++n)
      mbar_wait(smem_u32(&full[warp][n % kStages]), (n / kStages) & 1, &none);
  }
}

template <int kFmt>
cudaError_t launch_stream_fmt(const CacheRows* const* c, StreamParams& p, bool bf16, int num_sms, cudaStream_t stream) {
  using T = Tile<kFmt>;
  StreamMaps maps;
  for (int x = 0; x < 2; ++x) {
    auto& m = maps.s[x];
    const CacheRows& r = *c[x < p.segments ? x : 0];
    if (make_rows_map(&m.k, r, false, p.q.Hkv, bf16, T::kKeys) || make_rows_map(&m.v, r, true, p.q.Hkv, bf16, T::kKeys))
      return cudaErrorInvalidValue;
    if (kFmt != CACHE_16) {
      if (make_scale_map(&m.ks, r, false, p.q.Hkv, T::kKeys) || make_scale_map(&m.vs, r, true, p.q.Hkv, T::kKeys))
        return cudaErrorInvalidValue;
    } else {
      m.ks = m.vs = m.k;
    }
  }
  const uint32_t smem = kWarps * kStages * (kTileBytes + T::kScales) + 1024;
  const auto kern = bf16 ? attn_stream_kernel<true, kFmt> : attn_stream_kernel<false, kFmt>;
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem);
  if (e != cudaSuccess) return e;
  e = launch_dependent(kern, dim3(static_cast<unsigned>(num_sms)), dim3(kThreads), smem, stream, maps, p);
  count_launch();
  return e;
}

cudaError_t launch_stream(const CacheRows* const* c, StreamParams& p, bool bf16, int num_sms, cudaStream_t stream) {
  switch (c[0]->format) {
    case CACHE_I8: return launch_stream_fmt<CACHE_I8>(c, p, bf16, num_sms, stream);
    case CACHE_E4M3: return launch_stream_fmt<CACHE_E4M3>(c, p, bf16, num_sms, stream);
    default: return launch_stream_fmt<CACHE_16>(c, p, bf16, num_sms, stream);
  }
}

// Query rows are few enough for the stream's one 16-row tile.
bool streams(const Segment& s) { return s.rows <= kRows; }

size_t row_count(const CacheAttnArgs& a) { return static_cast<size_t>(a.B) * a.Sq * a.H; }

// Hands out pieces of the workspace, or only adds them up (base null).
struct Carver {
  uint8_t* base;
  size_t used;
  template <typename X>
  X* take(size_t count) {
    X* at = reinterpret_cast<X*>(base + used);
    used += (count * sizeof(X) + 255) / 256 * 256;
    return at;
  }
};

// How a call is cut: the prefix and the own rows, each streamed (in one launch where their formats agree) or in tiles of many
// rows, and a merge.
struct Plan {
  Segment s[2];        // prefix, own
  const CacheRows* c[2];
  bool have[2], stream[2], together;
  Source from[2];      // partial results
  size_t bytes;
};
Plan plan_of(const CacheAttnArgs& a, void* ws, int num_sms) {
  const RowShape q{a.Sq, a.H, a.H / a.group, a.group};
  Plan x;
  x.c[0] = &a.prefix;
  x.c[1] = &a.own;
  x.have[0] = a.prefix.N > 0;
  x.have[1] = true;
  x.stream[0] = false;
  for (int i = 0; i < 2; ++i) {
    x.from[i] = Source{};
    if (!x.have[i]) continue;
    x.s[i] = segment_of(*x.c[i], a, i == 1 && a.causal);
    x.stream[i] = streams(x.s[i]);
  }
  x.together = x.stream[0] && x.stream[1] && a.prefix.format == a.own.format;
  Carver w{static_cast<uint8_t*>(ws), 0};
  const size_t rows = row_count(a), workers = static_cast<size_t>(num_sms) * kWarps;
  for (int i = 0; i < 2; ++i) {
    if (!x.have[i]) continue;
    Source& f = x.from[i];
    f.segment = x.s[i];
    f.dealt = x.stream[i];
    if (!f.dealt) {
      f.fixed.parts = attn_rows_parts(x.s[i], q, num_sms);
      f.fixed.o = w.take<float>(rows * f.fixed.parts * 128);
      f.fixed.ml = w.take<float>(rows * f.fixed.parts * 2);
      continue;
    }
    Dealt& d = f.deal;
    d.keys = x.c[i]->format == CACHE_16 ? Tile<CACHE_16>::kKeys : Tile<CACHE_I8>::kKeys;
    d.workers = w.take<int2>(static_cast<size_t>(x.s[i].N) * q.Hkv);
    if (i == 1 && x.together) {
      d.slot_rows = x.from[0].deal.slot_rows;
      d.slot_o = x.from[0].deal.slot_o;
      d.slot_ml = x.from[0].deal.slot_ml;
    } else {
      d.slot_rows = x.s[i].rows > x.s[1].rows ? x.s[i].rows : x.s[1].rows;
      if (!x.together) d.slot_rows = x.s[i].rows;
      d.slot_o = w.take<float>(workers * 2 * d.slot_rows * 128);
      d.slot_ml = w.take<float>(workers * 2 * d.slot_rows * 2);
    }
    if (x.have[0]) {
      d.whole_o = w.take<float>(rows * 128);
      d.whole_ml = w.take<float>(rows * 2);
    }
  }
  x.bytes = w.used;
  return x;
}

}  // namespace

size_t attn_cache_ws_bytes(const CacheAttnArgs& a, int num_sms) { return plan_of(a, nullptr, num_sms).bytes; }

cudaError_t launch_attn_cache(const CacheAttnArgs& a, void* ws, int num_sms, cudaStream_t stream) {
  const Plan x = plan_of(a, ws, num_sms);
  StreamParams p;
  p.q = RowShape{a.Sq, a.H, a.H / a.group, a.group};
  p.scale_log2 = a.softmax_scale * 1.4426950408889634f;
  p.qp = a.q;
  p.q_sb = a.q_sb; p.q_ss = a.q_ss; p.q_sh = a.q_sh;
  p.out = a.out;
  p.o_sb = a.o_sb; p.o_ss = a.o_ss; p.o_sh = a.o_sh;
  p.lse2 = a.lse2;
  p.finish = x.have[0] ? 0 : 1;
  p.status = device_status_words();
  for (int i = 0; i < 2; ++i) {
    if (!x.have[i] || (i == 1 && x.together)) continue;
    cudaError_t e;
    if (x.stream[i]) {
      p.segments = x.together ? 2 : 1;
      for (int y = 0; y < p.segments; ++y) {
        p.s[y] = x.s[i + y];
        p.deal[y] = x.from[i + y].deal;
      }
      e = launch_stream(x.c + i, p, a.bf16, num_sms, stream);
    } else {
      e = launch_attn_rows(*x.c[i], x.s[i], a, x.from[i].fixed, stream);
    }
    if (e != cudaSuccess) return e;
  }
  return launch_attn_merge(a, x.from[0], x.from[1], p.finish != 0 && x.stream[1], num_sms * kWarps, stream);
}

}  // namespace asuka
