// Attention of new tokens over a KV cache of ragged sequences, 16 or 8 bits, and over a prefix that they share.
//
// Everything here is softmax(q K^T scale) V over the rows of a prefix and of the sequence's own cache, one softmax over
// both.  Each is a segment: N sequences, and to each (sequence, key/value head) -- a unit -- the query rows that read it: all
// heads of the group at all new positions, and for a prefix those of all sequences that share it.  A segment leaves, for every
// query row, an unnormalised output, the reference of its exponentials and their sum; the last one merges and divides.
//
// attn_stream_kernel, for up to 16 rows to a unit (see `streams`): the keys and values are used by so few rows that the work is one read of the
// cache, and the floor its bytes over the HBM bandwidth.  Sequences are of any lengths, known on the device only, and units may be
// many and short or few and long; so the work is dealt out there:
//   - a unit's keys are tiles of 32 (8 bits) or 16 (16 bits), 8 KB of keys and values, and the tiles of all units of all segments are
//     numbered through.  Every warp of the launch is a worker with an equal, contiguous range of them, which may begin and end
//     inside a unit: no SM waits for the longest sequence, and a warp waits for no other;
//   - a warp fetches its own tiles by TMA into a ring of its own, across the ends of units, and works on them with 16x8x16 matrix
//     instructions and a running maximum and sum.  The keys are the 16 rows of the first product, S^T = K Q^T, and the columns
//     of the values those of the second, O^T = V^T P^T, so that eight query rows, the usual case, cost half of what sixteen do;
//     the weights get from one to the other by transposing 8x8 blocks between registers;
//   - a unit that lies in one range is finished there; what a range has of a unit that others share goes to the workspace
//     and is merged by attn_merge_kernel in the order of the keys, so results do not depend on which warp was first.
// Small calls are bound by the launches and by one unit's latency, not by bytes: there a cluster of up to eight CTAs takes a unit, its warps
// an equal range each, and merges through its distributed shared memory (see `cluster_of`); there is no deal, workspace or second launch.
// Over 16 bits the weights are rounded to the values' type, as the operands of one product have the same (bf16: 2^-9 on average).
// Codes of 8 bits go from shared memory straight into matrix fragments:
//   - codes become f16, exactly (int8 as the low bits of 1024 + 128 + code, less 1152; e4m3 by conversion), and q is brought
//     to f16 too, a bf16 row times the power of two that puts its largest value in [1, 2): what is lost is below 2^-24 of it;
//   - the order of a contraction's terms is free, and so is that of a product's rows: lane l & 3 = t takes columns 32 t .. 32 t + 31 of
//     its keys' rows, 16 bytes at a time, and of its query row; for the second product lane l >> 2 = c takes columns
//     16 c .. 16 c + 15 of four keys, whose bytes are interleaved to pairs of keys.  With the 128-byte swizzle neither read has a
//     bank conflict;
//   - a key's scale multiplies its logits; a value's scale s multiplies the weights, w s = exp2(x) s, rounded to f16.  The reference of
//     the exponentials is the largest x + log2(s), so w s <= 1 and the rounding is 2^-11 of it (2^-25 of the largest where it is
//     subnormal, as all are whose scale is far below 2^-76, the least that counts there).
#include "attn_cache.cuh"

namespace asuka {
namespace {

// ---- up to 16 rows to a unit -----------------------------------------------------------------------
constexpr int kRows = 16;
constexpr int kWarps = 12;   // workers of a CTA, one CTA to an SM
constexpr int kStages = 2;   // of each worker's ring
constexpr int kThreads = kWarps * 32;
constexpr int kMinTiles = 2;  // a worker's share is no less
constexpr int kMaxCluster = 8;  // CTAs to a unit
constexpr int kFewTiles = 10;  // of a warp of the cluster form, at most
template <int kFmt> struct Tile {
  static constexpr int kKeys = kFmt == CACHE_16 ? 16 : 32;
  static constexpr uint32_t kHalf = 2048;                  // (16 bits) one 64-column half of the keys or values
  static constexpr uint32_t kK = 4096;                     // the keys, and the values
};
constexpr uint32_t kTileBytes = 8192;

struct StreamParams {
  Segment s[2];    // numbered through in this order
  const float* k_scale[2];
  const float* v_scale[2];
  int64_t ks_sb[2], ks_sh[2], vs_sb[2], vs_sh[2];
  int segments;
  RowShape q;
  float scale_log2;
  const uint16_t* qp;
  int64_t q_sb, q_ss, q_sh;
  uint16_t* out;
  int64_t o_sb, o_ss, o_sh;
  float* lse2;
  int finish;      // whole units are the output (no other segment)
  int chained;     // the kernel ahead is this call's, of the other segment: only the merge needs its results
  Dealt deal[2];
  uint32_t* status;
};
struct StreamMaps {
  struct {
    CUtensorMap k, v;
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
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
// x / y, y > 0, in 32 bits where they fit (a 64-bit division takes 0.2 us)
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {
  if (static_cast<uint64_t>(x | y) >> 32 == 0) return static_cast<uint32_t>(x) / static_cast<uint32_t>(y);
  return x / y;
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
// an 8x8 block of 16-bit values, rows and columns exchanged
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
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

// One CTA to an SM; a warp is a worker.  kOct: eights of query rows to a unit.
// kCluster: few units and few keys.  A unit is a cluster of CTAs, whose warps share its tiles and whose results are merged through
// distributed shared memory, in the order of the keys' owners: no second launch, and no deal.
template <bool kBF16, int kFmt, int kOct, bool kCluster>
__global__ void __launch_bounds__(kThreads, 1)
attn_stream_kernel(const __grid_constant__ StreamMaps maps, const StreamParams p) {
  using T = Tile<kFmt>;
  constexpr bool k8 = kFmt != CACHE_16;
  constexpr int kSub = T::kKeys / 16;  // blocks of 16 keys in a tile
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[kWarps][kStages];
  __shared__ uint32_t abort_s;
  __shared__ float2 ml_s[kCluster ? kWarps : 1][8 * kOct];    // (kCluster) every warp's reference and sum of every row
  __shared__ float cta_o[kCluster ? 8 * kOct : 1][128];       // the CTA's results, read by the whole cluster
  __shared__ float2 cta_ml[8 * kOct];

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
  // Behind this call's own kernel for the prefix the work begins as SMs become free: what this kernel reads was complete
  // before that one let it start, and what it writes is its own.  (Reads are from L2, and the wait is at the end: the merge follows on
  // both.)  128 sequences behind 32768 bf16 rows 106.7 -> 101.7 us.
  if (!p.chained) griddep_wait();
  griddep_launch_dependents();

  __syncthreads();

  // ---- the deal: every warp adds up the tiles of all sequences by itself (a lane has `per` consecutive ones)
  const int n_seqs = p.s[0].N + (p.segments > 1 ? p.s[1].N : 0);
  auto at = [&](int i, Cursor& c) {  // sequence i of all segments
    c.seg = i >= p.s[0].N ? 1 : 0;
    c.seq = i - (c.seg ? p.s[0].N : 0);
    c.len = seen_of(p.s[c.seg], c.seq);
    c.tiles = (c.len + T::kKeys - 1) / T::kKeys;
  };
  int64_t worker = 0, share = 0;
  int count;
  Cursor c;
  if constexpr (kCluster) {
    const int unit = static_cast<int>(blockIdx.x / cluster_size());
    at(unit / p.q.Hkv, c);
    c.hk = unit % p.q.Hkv;
    const int each = max((c.tiles + static_cast<int>(cluster_size()) * kWarps - 1) / (static_cast<int>(cluster_size()) * kWarps), 1);
    c.tile = (warp * static_cast<int>(cluster_size()) + static_cast<int>(cluster_rank())) * each;
    count = max(min(each, c.tiles - c.tile), 0);
  } else {
    const int per = (n_seqs + 31) / 32;
    int64_t upto = 0;
#pragma unroll 4
    for (int i = lane * per; i < min(n_seqs, (lane + 1) * per); ++i) {
      Cursor c;
      at(i, c);
      upto += c.tiles;
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += x;
    }
    upto *= p.q.Hkv;  // tiles of this lane's sequences and those before
    const int64_t total = __shfl_sync(0xffffffffu, upto, 31);
    const int64_t workers = static_cast<int64_t>(gridDim.x) * kWarps;
    share = max(static_cast<int64_t>(quotient(total + workers - 1, workers)), static_cast<int64_t>(kMinTiles));

    // (neighbours in the numbering on different SMs, so that a small launch uses all of them)
    worker = static_cast<int64_t>(warp) * gridDim.x + blockIdx.x;
    const int64_t lo = worker * share;
    count = static_cast<int>(min(share, total - lo));  // (a worker's tiles are 8 KB each: far below 2^31)
    if (count <= 0) {
      if (p.chained) griddep_wait();
      return;
    }

    {
      const int x = __ffs(__ballot_sync(0xffffffffu, upto > lo)) - 1;  // the lane whose sequences the range begins in
      int64_t rest = lo - (x > 0 ? __shfl_sync(0xffffffffu, upto, max(x - 1, 0)) : 0);
      for (int i = x * per;; ++i) {  // (bounded, should another stream change the lengths in between)
        at(i, c);
        const int64_t in_seq = static_cast<int64_t>(c.tiles) * p.q.Hkv;
        if (rest < in_seq || i + 1 == n_seqs) break;
        rest -= in_seq;
      }
      c.tiles = max(c.tiles, 1);
      const int64_t hk = quotient(rest, c.tiles);
      c.hk = static_cast<int>(min(hk, static_cast<int64_t>(p.q.Hkv - 1)));
      c.tile = static_cast<int>(min(rest - hk * c.tiles, static_cast<int64_t>(c.tiles - 1)));
    }
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

  // The query rows of a unit whose keys are next, to L2: behind the first tiles, of which all warps ask for at once, they would
  // wait for 4 us.
  auto prefetch_rows = [&](const Cursor& x) {
    const Segment& s = p.s[x.seg];
#pragma unroll
    for (int y = 0; y < kOct; ++y) {
      const Row row = decode_row(min(8 * y + (lane >> 2), s.rows - 1), x.seq, x.hk, s, p.q);
      prefetch_l2(p.qp + row.b * p.q_sb + row.pos * p.q_ss + row.h * p.q_sh + (lane & 3) * 32);
    }
  };
  const uint32_t ring = smem_base + warp * kStages * kTileBytes;
  auto fetch = [&](const Cursor& x, int st) {
    const uint32_t bar = smem_u32(&full[warp][st]), dst = ring + st * kTileBytes;
    const auto& m = maps.s[x.seg];
    const int key = x.tile * T::kKeys;
    mbar_expect_tx(bar, kTileBytes);
    tma_load_4d(dst, &m.k, bar, 0, x.hk, key, x.seq);
    if constexpr (k8) {
      tma_load_4d(dst + T::kK, &m.v, bar, 0, x.hk, key, x.seq);
    } else {
      tma_load_4d(dst + T::kHalf, &m.k, bar, 64, x.hk, key, x.seq);
      tma_load_4d(dst + T::kK, &m.v, bar, 0, x.hk, key, x.seq);
      tma_load_4d(dst + T::kK + T::kHalf, &m.v, bar, 64, x.hk, key, x.seq);
    }
  };

  // Key lane's scales of the fetched tiles (8 bits), in the order of the tiles.
  float ks_of[kStages], vs_of[kStages];
  auto fetch_scales = [&](const Cursor& x, float& ks, float& vs) {
    if constexpr (k8) {
      const int key = x.tile * T::kKeys + lane;
      const bool live = key < x.len;  // (what lies behind the sequence may be anything)
      ks = live ? __ldcg(p.k_scale[x.seg] + x.seq * p.ks_sb[x.seg] + x.hk * p.ks_sh[x.seg] + key) : 0.f;
      vs = live ? __ldcg(p.v_scale[x.seg] + x.seq * p.vs_sb[x.seg] + x.hk * p.vs_sh[x.seg] + key) : 0.f;
    }
  };

  Cursor ahead = c;  // the next tile to fetch
  int fetched = 0;
  if (count > 0) prefetch_rows(c);
#pragma unroll
  for (int i = 0; i < kStages; ++i) {
    if (i >= count) continue;
    if (lane == 0) fetch(ahead, i);
    fetch_scales(ahead, ks_of[i], vs_of[i]);
    ++fetched;
    if (fetched < count) advance(ahead);
  }

  const int r0 = lane >> 2, t4 = lane & 3;
  uint32_t qf[kOct][16];      // query row 8 y + r0 as matrix fragments (in the order of terms that the keys' have)
  int lim[kOct][2];           // last visible key of rows 8 y + 2 t4 and 8 y + 2 t4 + 1, whose logits this thread has
  int min_lim = 0;            // no row's is below this
  float mul[kOct][2];         // of a dot product, to a logit in log2 units
  float o[kOct][8][4], m[kOct][2], l[kOct][2];  // (l: this thread's keys only)
  [[maybe_unused]] float v_most = 0.f;          // (8 bits) largest value scale of this lane's keys
  int first = 0;              // the unit's first tile in this range
  bool ok = true, begin = true, far = false;
  // (8 bits) Ends row 8 y + 2 t4 + x.  Where no value is large its sum is not small, and parts meet as they are; `unlift` waits
  // for the sum before the stores: one token, 1000 keys of 8 heads 6.0 -> 6.15 us where it is always done.  (With 16 rows there is no
  // register for the question: 16 sequences of 4001 keys 42.7 us with it, 42.0 without.)
  auto settle = [&](int y, int x, float& ref, float& sum) {
    if (!far) {
      sum *= kLiftDown;
      return;
    }
    const float take = unlift(ref, sum);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o[y][i][x] *= take;
      o[y][i][2 + x] *= take;
    }
  };

  for (int n = 0; n < count; ++n) {
    if (begin) {  // a unit begins, or this range of it
      begin = false;
      first = c.tile;
      v_most = 0.f;
      const Segment& s = p.s[c.seg];
#pragma unroll
      for (int y = 0; y < kOct; ++y) {
        const int r = 8 * y + r0;
        const Row row = decode_row(min(r, s.rows - 1), c.seq, c.hk, s, p.q);
        const uint32_t* src = reinterpret_cast<const uint32_t*>(p.qp + row.b * p.q_sb + row.pos * p.q_ss + row.h * p.q_sh);
        const bool live = r < s.rows;
        float unit = p.scale_log2;  // of this thread's own row
        if constexpr (!k8) {
#pragma unroll
          for (int kk = 0; kk < 16; ++kk) qf[y][kk] = live ? __ldcg(src + t4 + kk * 4) : 0u;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4 w = live ? __ldcg(reinterpret_cast<const uint4*>(src) + t4 * 4 + i) : make_uint4(0, 0, 0, 0);
            qf[y][4 * i] = w.x;
            qf[y][4 * i + 1] = w.y;
            qf[y][4 * i + 2] = w.z;
            qf[y][4 * i + 3] = w.w;
          }
          if constexpr (kBF16) {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 v = unpack2<true>(qf[y][i]);
              top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // (rows of zeros, and of nothing but values under 2^-100, stay as they are or vanish)
            const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23), 27), 253);
            const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
            unit *= __uint_as_float(static_cast<uint32_t>(e) << 23);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 v = unpack2<true>(qf[y][i]);
              qf[y][i] = pack2<false>(v.x * down, v.y * down);
            }
          }
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          mul[y][x] = __shfl_sync(0xffffffffu, unit, (2 * t4 + x) * 4);
          const int pos = min(8 * y + 2 * t4 + x, s.rows - 1) / p.q.group % p.q.Sq;
          lim[y][x] = s.causal ? min(c.len - 1, pos + c.len - p.q.Sq) : c.len - 1;
          m[y][x] = -INFINITY;
          l[y][x] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) o[y][i][0] = o[y][i][1] = o[y][i][2] = o[y][i][3] = 0.f;
      }
      min_lim = s.causal ? min(c.len - 1, c.len - p.q.Sq) : c.len - 1;
      if (!kCluster && first == 0 && lane == 0) {
        const int rest = c.tiles - (count - n);  // behind this worker's range
        p.deal[c.seg].workers[static_cast<int64_t>(c.seq) * p.q.Hkv + c.hk] =
            make_int2(static_cast<int>(worker), static_cast<int>(worker + (rest > 0 ? quotient(rest + share - 1, share) : 0)));
      }
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
    const uint32_t sK = ring + st * kTileBytes, sV = sK + T::kK;
    const int key0 = c.tile * T::kKeys;
    // s[u][y][e]: key 16 u + r0 (e < 2) or 16 u + 8 + r0, query row 8 y + 2 t4 + (e & 1)
    float s[kSub][kOct][4];
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int y = 0; y < kOct; ++y) s[u][y][0] = s[u][y][1] = s[u][y][2] = s[u][y][3] = 0.f;
    float ks[2 * kSub], vs[2 * kSub];  // scales of keys 8 j + r0
    if constexpr (k8) {
#pragma unroll
      for (int u = 0; u < kSub; ++u) {
        uint32_t a[8], b[8];
        lds4(sK + sw128_offset(16 * u + r0, 2 * t4), a);
        lds4(sK + sw128_offset(16 * u + r0, 2 * t4 + 1), a + 4);
        lds4(sK + sw128_offset(16 * u + 8 + r0, 2 * t4), b);
        lds4(sK + sw128_offset(16 * u + 8 + r0, 2 * t4 + 1), b + 4);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          uint32_t kf[4];
          codes_to_f16<kFmt>(a[kk], kf[0], kf[2]);
          codes_to_f16<kFmt>(b[kk], kf[1], kf[3]);
#pragma unroll
          for (int y = 0; y < kOct; ++y) mma16816<false>(s[u][y], kf, qf[y][2 * kk], qf[y][2 * kk + 1]);
        }
      }
#pragma unroll
      for (int j = 0; j < 2 * kSub; ++j) {
        ks[j] = __shfl_sync(0xffffffffu, ks_of[0], 8 * j + r0);
        vs[j] = __shfl_sync(0xffffffffu, vs_of[0], 8 * j + r0);
      }
      v_most = fmaxf(v_most, fabsf(vs_of[0]));
    } else {
      // this lane's row of the 8x8 blocks: keys 0-7 and 8-15, columns 0-7 and 8-15
      const int k_row = (((lane >> 3) & 1) << 3) + (lane & 7), k_chunk = lane >> 4;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        uint32_t kf[4];
        ldsm4(sK + (kk >> 2) * T::kHalf + sw128_offset(k_row, (kk & 3) * 2 + k_chunk), kf);
#pragma unroll
        for (int y = 0; y < kOct; ++y) mma16816<kBF16>(s[0][y], kf, qf[y][2 * kk], qf[y][2 * kk + 1]);
      }
    }
    if constexpr (k8) {
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int y = 0; y < kOct; ++y)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[u][y][e] *= ks[2 * u + (e >> 1)] * mul[y][e & 1];
    } else {
#pragma unroll
      for (int y = 0; y < kOct; ++y)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[0][y][e] *= p.scale_log2;
    }
    const bool ragged = key0 + T::kKeys - 1 > min_lim;
    if (ragged) {
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const int key = key0 + 16 * u + 8 * z + r0;
#pragma unroll
          for (int y = 0; y < kOct; ++y)
#pragma unroll
            for (int x = 0; x < 2; ++x)
              if (key > lim[y][x]) s[u][y][2 * z + x] = -INFINITY;
        }
    }
    float w[kOct][2];
    bool moved = false;
    {
      float lv[2 * kSub];  // log2 of the values' scales
      if constexpr (k8) {
#pragma unroll
        for (int j = 0; j < 2 * kSub; ++j) lv[j] = lg2(fmaxf(fabsf(vs[j]), kLeastScale));
      }
#pragma unroll
      for (int y = 0; y < kOct; ++y) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float mx = m[y][x];
#pragma unroll
          for (int j = 0; j < 2 * kSub; ++j) mx = fmaxf(mx, k8 ? s[j >> 1][y][2 * (j & 1) + x] + lv[j] : s[j >> 1][y][2 * (j & 1) + x]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float ref = mx > -INFINITY ? mx : 0.f;
          const float step = k8 ? half_step(m[y][x], ref) : ex2(m[y][x] - ref);
          w[y][x] = k8 ? step * step : step;
          moved = moved || step != 1.f;
          m[y][x] = mx;
          const float low = k8 ? ref - static_cast<float>(kLift) : ref;
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < 2 * kSub; ++j) {
            float& e = s[j >> 1][y][2 * (j & 1) + x];
            e = ex2(e - low);
            sum += e;
          }
          l[y][x] = (k8 ? l[y][x] * step : l[y][x]) * step + sum;
        }
      }
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int y = 0; y < kOct; ++y)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          o[y][i][0] *= w[y][0];
          o[y][i][1] *= w[y][1];
          o[y][i][2] *= w[y][0];
          o[y][i][3] *= w[y][1];
        }
    }
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      uint32_t pf[kOct][2];  // the weights, rows and keys exchanged: keys 2 t4, 2 t4 + 1 (and 8 further) of row r0
#pragma unroll
      for (int y = 0; y < kOct; ++y)
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const float f = k8 ? vs[2 * u + z] * kLiftDown : 1.f;
          pf[y][z] = transpose8(k8 ? pack2<false>(s[u][y][2 * z] * f, s[u][y][2 * z + 1] * f)
                                   : pack2<kBF16>(s[u][y][2 * z], s[u][y][2 * z + 1]));
        }
      if constexpr (k8) {
        uint32_t v[4][4];  // keys 2 t4, 2 t4 + 1, 8 + 2 t4, 9 + 2 t4 of the block, columns 16 r0 .. 16 r0 + 15
#pragma unroll
        for (int i = 0; i < 4; ++i) lds4(sV + sw128_offset(16 * u + (i >> 1) * 8 + 2 * t4 + (i & 1), r0), v[i]);
        if (ragged) {  // (what lies behind the sequence may be NaN)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (key0 + 16 * u + (i >> 1) * 8 + 2 * t4 + (i & 1) >= c.len) v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0u;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t vf[2][4];  // columns 4 i, 4 i + 1 and 4 i + 2, 4 i + 3
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            codes_to_f16<kFmt>(__byte_perm(v[2 * z][i], v[2 * z + 1][i], 0x5140), vf[0][2 * z], vf[0][2 * z + 1]);
            codes_to_f16<kFmt>(__byte_perm(v[2 * z][i], v[2 * z + 1][i], 0x7362), vf[1][2 * z], vf[1][2 * z + 1]);
          }
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int y = 0; y < kOct; ++y) mma16816<false>(o[y][2 * i + x], vf[x], pf[y][0], pf[y][1]);
        }
      } else {
        // 8x8 blocks with rows and columns exchanged: columns 0-7 and 8-15 of keys 0-7, then of keys 8-15
        const int v_row = ((lane >> 4) << 3) + (lane & 7), v_chunk = (lane >> 3) & 1;
        uint32_t keep[2] = {0xffffffffu, 0xffffffffu};  // (what lies behind the sequence may be infinite or NaN)
        if (ragged) {
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const int key = key0 + 8 * z + 2 * t4;
            keep[z] = (key < c.len ? 0xffffu : 0u) | (key + 1 < c.len ? 0xffff0000u : 0u);
          }
        }
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          uint32_t vf[4];
          ldsm4_t(sV + (d >> 2) * T::kHalf + sw128_offset(v_row, (d & 3) * 2 + v_chunk), vf);
#pragma unroll
          for (int z = 0; z < 4; ++z) vf[z] &= keep[z >> 1];
#pragma unroll
          for (int y = 0; y < kOct; ++y) mma16816<kBF16>(o[y][d], vf, pf[y][0], pf[y][1]);
        }
      }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i + 1 < kStages; ++i) {
      ks_of[i] = ks_of[i + 1];
      vs_of[i] = vs_of[i + 1];
    }
    if (fetched < count) {
      if (lane == 0) {
        fence_proxy_async_smem();  // (the warp's reads of the stage before the copy)
        fetch(ahead, st);
      }
      fetch_scales(ahead, ks_of[kStages - 1], vs_of[kStages - 1]);
      if (ahead.tile == 0) prefetch_rows(ahead);
      ++fetched;
      if (fetched < count) advance(ahead);
    }

    if (!kCluster && (c.tile + 1 == c.tiles || n + 1 == count)) {
      // ---- the unit ends, or this range of it
      const Segment& sg = p.s[c.seg];
      if constexpr (k8) far = kOct > 1 || __any_sync(0xffffffffu, v_most > kLarge);
      const bool whole = first == 0 && c.tile + 1 == c.tiles;
#pragma unroll
      for (int y = 0; y < kOct; ++y) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float sum = l[y][x];
          sum += __shfl_xor_sync(0xffffffffu, sum, 4);
          sum += __shfl_xor_sync(0xffffffffu, sum, 8);
          sum += __shfl_xor_sync(0xffffffffu, sum, 16);
          const int r = 8 * y + 2 * t4 + x;
          if (r >= sg.rows) continue;
          if constexpr (k8) settle(y, x, m[y][x], sum);
          const Row row = decode_row(r, c.seq, c.hk, sg, p.q);
          // this thread's columns of the row: 8 bits: 16 r0 + 2 i and + 1 in o[i][x] and o[i][2 + x]; 16 bits: 16 i + r0 and + 8
          if (whole && p.finish) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            uint16_t* dst = p.out + row.b * p.o_sb + row.pos * p.o_ss + row.h * p.o_sh;
            if constexpr (k8) {
              uint32_t v[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] = pack2<kBF16>(o[y][i][x] * inv, o[y][i][2 + x] * inv);
              *reinterpret_cast<uint4*>(dst + 16 * r0) = make_uint4(v[0], v[1], v[2], v[3]);
              *reinterpret_cast<uint4*>(dst + 16 * r0 + 8) = make_uint4(v[4], v[5], v[6], v[7]);
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const uint32_t v = pack2<kBF16>(o[y][i][x] * inv, o[y][i][2 + x] * inv);
                dst[16 * i + r0] = static_cast<uint16_t>(v);
                dst[16 * i + 8 + r0] = static_cast<uint16_t>(v >> 16);
              }
            }
            if (p.lse2 != nullptr && r0 == 0)
              p.lse2[(static_cast<int64_t>(row.b) * p.q.H + row.h) * p.q.Sq + row.pos] = m[y][x] + log2f(sum);
            continue;
          }
          const Dealt& d = p.deal[c.seg];
          const int64_t number = (static_cast<int64_t>(row.b) * p.q.Sq + row.pos) * p.q.H + row.h;
          const int64_t slot = (worker * 2 + (first > 0 ? 0 : 1)) * d.slot_rows + r;
          float* dst = whole ? d.whole_o + number * 128 : d.slot_o + slot * 128;
          float* ml = whole ? d.whole_ml + number * 2 : d.slot_ml + slot * 2;
          if constexpr (k8) {
#pragma unroll
            for (int i = 0; i < 8; i += 2)
              *reinterpret_cast<float4*>(dst + 16 * r0 + 2 * i) = make_float4(o[y][i][x], o[y][i][2 + x], o[y][i + 1][x], o[y][i + 1][2 + x]);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              dst[16 * i + r0] = o[y][i][x];
              dst[16 * i + 8 + r0] = o[y][i][2 + x];
            }
          }
          if (r0 == 0) {
            const float ref = m[y][x] > -INFINITY || sum == 0.f ? m[y][x] : 0.f;  // (nothing but NaN: the sum)
            *reinterpret_cast<float2*>(ml) = make_float2(ref, sum);
          }
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
  if (p.chained) griddep_wait();
  if constexpr (kCluster) {
    // ---- the warps' results, one CTA's, the cluster's; a ring whose tiles are all used holds its warp's
    const Segment& sg = p.s[0];
    if constexpr (k8) far = kOct > 1 || __any_sync(0xffffffffu, v_most > kLarge);
    float* results = reinterpret_cast<float*>(smem_raw + (smem_base - smem_u32(smem_raw)));
    float* mine = results + warp * (kStages * kTileBytes / 4);
#pragma unroll
    for (int y = 0; y < kOct; ++y) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = 8 * y + 2 * t4 + x;
        float sum = count > 0 ? l[y][x] : 0.f;
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        float ref = count > 0 ? m[y][x] : -INFINITY;
        if constexpr (k8) settle(y, x, ref, sum);
        if (r0 == 0) ml_s[warp][r] = make_float2(ref, sum);
        if (count <= 0 || r >= sg.rows) continue;
        if constexpr (k8) {
#pragma unroll
          for (int i = 0; i < 8; i += 2)
            *reinterpret_cast<float4*>(mine + r * 128 + 16 * r0 + 2 * i) = make_float4(o[y][i][x], o[y][i][2 + x], o[y][i + 1][x], o[y][i + 1][2 + x]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            mine[r * 128 + 16 * i + r0] = o[y][i][x];
            mine[r * 128 + 16 * i + 8 + r0] = o[y][i][2 + x];
          }
        }
      }
    }
    __syncthreads();
    const int cols = tid & 127;  // three rows at a time, a thread to a column
    for (int r = tid >> 7; r < sg.rows; r += kThreads / 128) {
      float top = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml_s[w][r].x);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 ml = ml_s[w][r];
        if (ml.x > -INFINITY || ml.y != 0.f) {  // (else nothing seen; nothing but NaN: the sum)
          const float f = ml.x > -INFINITY ? ex2(ml.x - top) : 1.f;
          sum = fmaf(f, ml.y, sum);
          acc = fmaf(f, results[w * (kStages * kTileBytes / 4) + r * 128 + cols], acc);
        }
      }
      cta_o[r][cols] = acc;
      if (cols == 0) cta_ml[r] = make_float2(top, sum);
    }
    cluster_sync();
    const int parts = static_cast<int>(cluster_size());
    for (int r = static_cast<int>(cluster_rank()) + parts * (tid >> 7); r < sg.rows; r += parts * (kThreads / 128)) {
      float2 ml[kMaxCluster];
      float po[kMaxCluster];
      float top = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
      for (int x = 0; x < kMaxCluster; ++x) {
        if (x >= parts) continue;
        ml[x].x = ld_cluster(smem_u32(&cta_ml[r].x), x);
        ml[x].y = ld_cluster(smem_u32(&cta_ml[r].y), x);
        po[x] = ld_cluster(smem_u32(&cta_o[r][cols]), x);
      }
#pragma unroll
      for (int x = 0; x < kMaxCluster; ++x)
        if (x < parts) top = fmaxf(top, ml[x].x);
#pragma unroll
      for (int x = 0; x < kMaxCluster; ++x) {
        if (x < parts && (ml[x].x > -INFINITY || ml[x].y != 0.f)) {
          const float f = ml[x].x > -INFINITY ? ex2(ml[x].x - top) : 1.f;
          sum = fmaf(f, ml[x].y, sum);
          acc = fmaf(f, po[x], acc);
        }
      }
      const Row row = decode_row(r, c.seq, c.hk, sg, p.q);
      const float y = sum == 0.f ? 0.f : acc / sum;
      const float next = __shfl_down_sync(0xffffffffu, y, 1);
      if ((cols & 1) == 0)
        *reinterpret_cast<uint32_t*>(p.out + row.b * p.o_sb + row.pos * p.o_ss + row.h * p.o_sh + cols) = pack2<kBF16>(y, next);
      if (p.lse2 != nullptr && cols == 0)
        p.lse2[(static_cast<int64_t>(row.b) * p.q.H + row.h) * p.q.Sq + row.pos] = top + log2f(sum);
    }
    cluster_sync();  // no CTA leaves while another still reads its shared memory
  }
}

template <int kFmt>
cudaError_t launch_stream_fmt(const CacheRows* const* c, StreamParams& p, bool bf16, int cluster, int num_sms, cudaStream_t stream) {
  using T = Tile<kFmt>;
  StreamMaps maps;
  for (int x = 0; x < 2; ++x) {
    auto& m = maps.s[x];
    const CacheRows& r = *c[x < p.segments ? x : 0];
    if (make_rows_map(&m.k, r, false, p.q.Hkv, bf16, T::kKeys) || make_rows_map(&m.v, r, true, p.q.Hkv, bf16, T::kKeys))
      return cudaErrorInvalidValue;
    p.k_scale[x] = r.k_scale;
    p.v_scale[x] = r.v_scale;
    p.ks_sb[x] = r.ks_sb;
    p.ks_sh[x] = r.ks_sh;
    p.vs_sb[x] = r.vs_sb;
    p.vs_sh[x] = r.vs_sh;
  }
  const uint32_t smem = kWarps * kStages * kTileBytes + 1024;
  bool wide = false;
  for (int x = 0; x < p.segments; ++x) wide = wide || p.s[x].rows > 8;
  if (cluster > 0) {
    constexpr int kWide = kFmt == CACHE_16 ? 1 : 2;  // (16 bits: up to eight rows, see cluster_of)
    const auto kern = bf16 ? (wide ? attn_stream_kernel<true, kFmt, kWide, true> : attn_stream_kernel<true, kFmt, 1, true>)
                           : (wide ? attn_stream_kernel<false, kFmt, kWide, true> : attn_stream_kernel<false, kFmt, 1, true>);
    cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem);
    if (e != cudaSuccess) return e;
    e = launch_dependent_cluster(kern, dim3(static_cast<unsigned>(p.s[0].N * p.q.Hkv * cluster)), dim3(kThreads), smem,
                                 static_cast<unsigned>(cluster), stream, maps, p);
    count_launch();
    return e;
  }
  const auto kern = bf16 ? (wide ? attn_stream_kernel<true, kFmt, 2, false> : attn_stream_kernel<true, kFmt, 1, false>)
                         : (wide ? attn_stream_kernel<false, kFmt, 2, false> : attn_stream_kernel<false, kFmt, 1, false>);
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem);
  if (e != cudaSuccess) return e;
  e = launch_dependent(kern, dim3(static_cast<unsigned>(num_sms)), dim3(kThreads), smem, stream, maps, p);
  count_launch();
  return e;
}

cudaError_t launch_stream(const CacheRows* const* c, StreamParams& p, bool bf16, int cluster, int num_sms, cudaStream_t stream) {
  switch (c[0]->format) {
    case CACHE_I8: return launch_stream_fmt<CACHE_I8>(c, p, bf16, cluster, num_sms, stream);
    case CACHE_E4M3: return launch_stream_fmt<CACHE_E4M3>(c, p, bf16, cluster, num_sms, stream);
    default: return launch_stream_fmt<CACHE_16>(c, p, bf16, cluster, num_sms, stream);
  }
}

// Which kernel takes a segment of up to 16 rows to a unit; the other one's tiles (attn_rows.cu) are mostly empty then, but
// 16-bit keys come in copies four times as large and need no instruction of a warp.  It has a CTA for a unit, or several,
// and nothing to follow a short one; the stream is even whatever the units are.  Dealt out / tiles, us:
//   16 bits, 4 rows   8 units 8000 keys 17.7/14.6; 32 units 4001 keys 18.1/16.6, 128 units 43.8/41.4;
//                     128 units 16384 keys 140/135; 256 units 1000 keys 26.6/28.4, 512 units 500 keys 26.7/39.4
//   16 bits, 16 rows  16 units 8003 keys 25.3/17.2, 128 units 4001 keys 52/43
//   8 bits, 4 rows    8 units 8000 keys 13.7/15.0; 128 units 4001 keys 30.6/57.8
//   8 bits, 16 rows   16 units 8003 keys 26/20; 8 units 32000 keys 34/37 (few units of many keys:
//                     given up for a rule on their number); 128 units 4001 keys 44/58
bool streams(const Segment& s, const RowShape& q, int format, int num_sms) {
  if (s.rows > kRows) return false;
  const int64_t units = static_cast<int64_t>(s.N) * q.Hkv;
  return format == CACHE_16 ? units > num_sms : s.rows <= 8 || 4 * units > num_sms;
}

// CTAs of a cluster for each unit of a lone segment, or 0 for none.  The cluster form is one launch and has no deal, 2.5 us less, and costs
// what a unit's warps have more tiles to do (2 us each) than an even share.  Clusters / the form that `streams` chooses, us, 4 rows,
// 8 heads, sequences of half to all of the longest:
//   8 bits   B1 1000 keys 5.9/8.6, 4000 7.9/11.1, 16000 16.7/18.5; B4 1000 6.4/9.2, 4000 12.2/15.1, 16000 28.4/28.1;
//            B16 1000 12.7/16.1, 4000 28.7/29.1; B2 16000 with four CTAs 25.6/20.6
//   16 bits  B1 1000 keys 6.5/7.8, 4000 10.2/12.7, 16000 23.8/17.3; B4 1000 8.5/10.3, 4000 15.2/16.9; B16 1000 15.2/15.1, 4000 43/39
// Of clusters of eight only some fit at once: 8 bits, B2 4000 keys, 16 units, 14.8 with eight CTAs to each, 10.9 with four.
int cluster_of(const Segment& s, const RowShape& q, int format, int num_sms) {
  if (s.rows > (format == CACHE_16 ? 8 : kRows)) return 0;
  const int64_t units = static_cast<int64_t>(s.N) * q.Hkv;
  const int keys = format == CACHE_16 ? Tile<CACHE_16>::kKeys : Tile<CACHE_I8>::kKeys, tiles = (s.S + keys - 1) / keys;
  int parts = 1;
  while (parts < kMaxCluster && units * parts * 2 <= (parts == kMaxCluster / 2 ? 2 * num_sms / 3 : num_sms) && tiles > parts * kWarps)
    parts *= 2;
  const int64_t each = (tiles + parts * kWarps - 1) / (parts * kWarps), workers = static_cast<int64_t>(num_sms) * kWarps;
  const int64_t share = (units * tiles + workers - 1) / workers;
  return units * parts <= num_sms && each <= kFewTiles && each <= (share > kMinTiles ? share : kMinTiles) + 3 ? parts : 0;
}

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
  bool finished;       // the own rows' kernel leaves nothing to merge
  int cluster;         // CTAs to a unit of the stream's cluster form, 0: dealt out
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
    x.stream[i] = streams(x.s[i], q, x.c[i]->format, num_sms);
  }
  x.finished = false;
  x.cluster = x.have[0] ? 0 : cluster_of(x.s[1], q, a.own.format, num_sms);
  if (x.cluster > 0) x.stream[1] = true;
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
      x.finished = !x.have[0] && f.fixed.parts == 1;
      if (x.finished) continue;
      f.fixed.o = w.take<float>(rows * f.fixed.parts * 128);
      f.fixed.ml = w.take<float>(rows * f.fixed.parts * 2);
      continue;
    }
    if (x.cluster > 0) {
      x.finished = true;
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
    const bool chained = i == 1 && x.have[0];
    cudaError_t e;
    if (x.stream[i]) {
      p.segments = x.together ? 2 : 1;
      p.chained = chained ? 1 : 0;
      for (int y = 0; y < p.segments; ++y) {
        p.s[y] = x.s[i + y];
        p.deal[y] = x.from[i + y].deal;
      }
      e = launch_stream(x.c + i, p, a.bf16, x.cluster, num_sms, stream);
    } else {
      e = launch_attn_rows(*x.c[i], x.s[i], a, x.from[i].fixed, x.finished, chained, stream);
    }
    if (e != cudaSuccess) return e;
  }
  if (x.finished) return cudaSuccess;
  return launch_attn_merge(a, x.from[0], x.from[1], p.finish != 0 && x.stream[1], num_sms * kWarps, stream);
}

}  // namespace asuka
