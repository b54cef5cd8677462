// Attention of many query rows to a unit over a cache or a shared prefix (attn_cache.cu has the segments, units and partial
// results, and the kernel for up to 16 rows).
//
// The rows of all sequences that share a prefix -- times their new positions, times the heads of a group -- are rows of one
// matrix product with its keys: tiles of 128 (a tensor map whose box is group x positions x sequences gathers them), so that a
// key is read and multiplied once for all of them.  A CTA takes one or two tiles and a part of the keys:
//   warp 0        TMA: Q once, K (8-bit caches: the codes of K and V in turn, and their scales)
//   warp 2        TMA: V
//   warp 1        issues S = Q_t K^T (tcgen05.mma, SMEM x SMEM)
//   warp 3        issues O_t += P_t V (TMEM x SMEM)
//   warps 4-11    softmax, a thread to a row of S
//   warps 12-15   (8-bit caches) codes to 16-bit tiles
// The two softmax slots ping-pong as in attn_fwd.cu, one S in tensor memory serving both: with two tiles each has one of them and a K/V
// tile serves both; with one tile a slot has the even key tiles and the other the odd ones, merged at the end.  What is left of a
// part goes to the workspace unnormalised.
//
// 8-bit codes become f16 tiles in warps of their own: a thread takes one row's 128 codes from the swizzled stage, all at once so that
// the stage is free again, and writes them times their scale in the two swizzled halves that the tensor pipe reads, neither with a
// bank conflict; where the next tile has landed, its codes are loaded between the stores (G4 B32 H40/8 P6001 e4m3 37.9 -> 36.9 us, two query
// tiles unchanged).  A code times its scale is rounded once, to f16 (2^-12 on average): the scale, under the power of two of the largest of
// the warp's 32 keys or of the tile's 128 values, is two f16 terms, so that a pair of codes takes two instructions.  The softmax takes the keys'
// powers of two with the logits' factor; the values' go into the exponent, exp2(x + e - reference), and out of the row sum again.  bf16
// queries become f16 too, a row times the power of two that puts its largest value in [1, 2).
// With f16 output, finer than those roundings together (f16 keys, values and weights: 4.0e-4 to 4.8e-4 of it, the output's own 2.1e-4), and one
// query tile the f16 tiles are the codes, exactly, and the softmax multiplies logits and weights by the scales in f32 (kExact):
// 2.8e-4, G4 B32 H40/8 P6001 e4m3 36.9 -> 39.1 us.  bf16 output does not show them (1.7e-3 by itself), and for two query tiles, for which
// shared memory has no room for the scales as they are, it stays at 3.6e-4 to 5.4e-4.
//
// Over 16 bits the weights have the values' type, since the operands of one product have: with bf16 they are rounded to 2^-9 on average
// (the error of bf16 output 1.7e-3 -> 2.3e-3), as the prefill's are.
//
// Where the time goes, by the clock inside (int8, B2 Sq100 H32/8, 8003 keys: two tiles, 16 key tiles to a CTA; 41 us): set-up 0.7 us, 5.6 until the
// first S (4.4 of them until the queries are converted and the first codes have come), 30.5 the key tiles, 2.9 the end.  A key tile takes
// 3750 clk, of which the tensor pipe works for 2050 and the converting warps for 3500: they bound it.  Over 16 bits it takes 2530.  With
// one query tile of 40 rows it takes 2500 clk over e4m3, of which the converting warps work for 2290.
#include "attn_cache.cuh"

namespace asuka {

namespace {

constexpr int kTile = 128;
constexpr uint32_t kTileBytes = 128 * 128 * 2;  // [128 x 128] 16-bit: two swizzled halves
constexpr uint32_t kHalfBytes = kTileBytes / 2;
constexpr uint32_t kRawBytes = 128 * 128;       // [128 x 128] codes
constexpr float kRescaleLimit = 6.0f;           // log2 of the largest exponential tolerated under a stale reference

// kPair: two query tiles; else one.  Shared memory: Q, rings of 16-bit K and V tiles; with 8 bits one ring of both in turn, one of codes,
// and the scales that come with them.
template <bool kBF16, int kFmt, bool kPair> struct Cfg {
  static constexpr bool k8 = kFmt != CACHE_16;
  // Scales of keys and values as f32 in the softmax, and the f16 tiles exact
  static constexpr bool kExact = k8 && !kBF16 && !kPair;
  static constexpr int kQ = kPair ? 2 : 1;
  static constexpr int kK = k8 ? 4 : 3;                      // (8 bits: K and V in turn)
  static constexpr int kV = k8 ? 0 : (kPair ? 2 : 3);
  static constexpr int kRaw = k8 ? (kPair ? 2 : 3) : 0;
  static constexpr int kRawScales = kRaw == 2 ? 1 : kRaw;    // (they come with K, which with two stages is always in the first)
  // Powers of two of the scales: a K tile takes the place in the ring of the one two steps ago when its QK^T is complete; a softmax
  // slot may then be a step behind that one, or with one query tile, whose slots have every other tile, two.
  static constexpr int kPowers = kPair ? 4 : 8;
  static constexpr uint32_t kSmem = (kQ + kK + kV) * kTileBytes + kRaw * kRawBytes + kRawScales * 1024 + 1024;
  static constexpr int kThreads = k8 ? 512 : 384;
  // setmaxnreg: what the roles ask for is what the block gets at launch
  static constexpr int kLaunchRegs = k8 ? 128 : 168;
  static constexpr int kUtil = k8 ? 48 : 88;
  static constexpr int kConvert = 80;
  static constexpr int kSoftmax = k8 ? 192 : 208;
  static constexpr int kBlockRegs = 128 * kUtil + 256 * kSoftmax + (k8 ? 128 * kConvert : 0);
  static_assert(kBlockRegs <= kThreads * kLaunchRegs, "setmaxnreg would wait for ever");
  static_assert(kSmem <= 226 * 1024, "shared memory of an SM");
};

struct RowsParams {
  Segment s;
  RowShape q;
  int tile_b, tile_pos;   // sequences and positions of a query tile: its rows are tile_b x tile_pos x group
  int pos_tiles;          // tiles along the positions (1 where a tile holds whole sequences)
  int tiles, blocks;      // query tiles of a unit, and the CTAs' one or two of them
  int parts;
  float scale_log2;
  Partials mine;
  uint16_t* out;          // (kFinish)
  int64_t o_sb, o_ss, o_sh;
  float* lse2;
  int chained;            // as the stream's (attn_cache.cu)
  uint32_t* status;
};

struct RowsMaps {
  CUtensorMap q, k, v, ks, vs;
};

struct Bars {
  uint64_t q_full[2], q_ready[2];
  uint64_t k_full[4], k_empty[4];
  uint64_t v_full[3], v_empty[3];
  uint64_t raw_full[3], raw_empty[3], powers_full[8];
  uint64_t s_full[2], s_free, p_ready[2], pv_done[2];
};

__device__ __forceinline__ void st_global_v8(void* ptr, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(ptr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ void sts4(uint32_t addr, const uint32_t* r) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
__device__ __forceinline__ float ldsf(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void record_timeout(uint32_t* status, uint32_t site) {
  atomicAdd(&status[0], 1u);
  status[1] = site;
}

// Grid: parts of the keys x blocks of query tiles x units, the blocks of a part side by side (they read the same keys).
// kFinish: one part that is all there is, and the output instead of partial results (an instantiation of its own: what a CTA does
// once it also fetches its instructions for, and both ways in one kernel took 1.2 us longer).
template <bool kBF16, int kFmt, bool kPair, bool kFinish>
__global__ void __launch_bounds__(Cfg<kBF16, kFmt, kPair>::kThreads, 1)
attn_rows_kernel(const __grid_constant__ RowsMaps maps, const RowsParams p) {
  using C = Cfg<kBF16, kFmt, kPair>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) Bars bars;
  // What the softmax needs of the scales of a tile: 2^e of the keys' for each quarter, e of the values' and 2^(kLift - e).
  __shared__ float4 k_power_s[C::k8 && !C::kExact ? C::kPowers : 1];
  __shared__ float2 v_power_s[C::k8 ? C::kPowers : 1];
  __shared__ float4 scales_s[C::kExact ? C::kPowers : 1][2][kTile / 4];  // (kExact) the keys', and the values' times 2^-e
  __shared__ uint8_t unit_s[C::k8 && kBF16 ? C::kQ : 1][kTile];  // exponent of a query row's power of two, as f32 has it
  __shared__ float2 row_s[kPair ? 1 : kTile];  // (one tile) second slot's reference and sum; then both slots' factors
  __shared__ float take_s[C::k8 && !kPair ? kTile : 1];  // (one tile) second slot's `take`
  __shared__ uint32_t tmem_base_s;
  __shared__ uint32_t abort_s;

  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t sQ = smem_base, sK = sQ + C::kQ * kTileBytes, sV = sK + C::kK * kTileBytes;
  const uint32_t sRaw = sV + C::kV * kTileBytes, sRawScale = sRaw + C::kRaw * kRawBytes;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile uint32_t* abortp = &abort_s;

  int x = static_cast<int>(blockIdx.x);
  const int block = x % p.blocks;
  x /= p.blocks;
  const int part = x % p.parts, unit = x / p.parts;
  const int seq = unit / p.q.Hkv, hk = unit % p.q.Hkv;
  const int tile0 = kPair ? 2 * block : block;
  const bool two = kPair && tile0 + 1 < p.tiles;

  if (tid == 0) {
    abort_s = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bars.q_full[i]), 1);
      mbar_init(smem_u32(&bars.q_ready[i]), 128);
      mbar_init(smem_u32(&bars.s_full[i]), 1);
      mbar_init(smem_u32(&bars.p_ready[i]), 128);
      mbar_init(smem_u32(&bars.pv_done[i]), 1);
    }
    mbar_init(smem_u32(&bars.s_free), 128);
    for (int i = 0; i < 4; ++i) {
      mbar_init(smem_u32(&bars.k_full[i]), C::k8 ? 4 : 1);
      mbar_init(smem_u32(&bars.k_empty[i]), 1);
    }
    for (int i = 0; i < C::kPowers; ++i) mbar_init(smem_u32(&bars.powers_full[i]), 4);
    for (int i = 0; i < 3; ++i) {
      mbar_init(smem_u32(&bars.v_full[i]), 1);
      mbar_init(smem_u32(&bars.v_empty[i]), 1);
      mbar_init(smem_u32(&bars.raw_full[i]), 1);
      mbar_init(smem_u32(&bars.raw_empty[i]), 4);
    }
    mbar_fence_init();
    tma_prefetch_desc(&maps.q);
    tma_prefetch_desc(&maps.k);
    tma_prefetch_desc(&maps.v);
  }
  if (warp == 1) {
    __syncwarp();
    tmem_alloc(smem_u32(&tmem_base_s), 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tbase = tmem_base_s;
  if (!p.chained) griddep_wait();
  griddep_launch_dependents();

  // This CTA's key tiles: its part of what the sequence has, and of what the block's last rows see.  (A causal segment is of the
  // sequences' own rows: a block's tiles are of one sequence, next to each other.  A prompt of 1000, 2000, 4000 tokens, 32 heads over 8,
  // 16 bits: 20.6, 53.8, 245 us, to the end of the sequence for every block of two tiles 22.8, 68.7, 333.)
  const int len = seen_of(p.s, seq);
  int limit = len;
  if (p.s.causal) {
    const int last = min(tile0 + (two ? 1 : 0), p.tiles - 1) % p.pos_tiles;
    const int last_pos = p.pos_tiles == 1 ? p.q.Sq - 1 : min((last + 1) * p.tile_pos, p.q.Sq) - 1;
    limit = max(0, min(len, last_pos + len - p.q.Sq + 1));
  }
  const int all = (limit + kTile - 1) / kTile;
  const int j0 = static_cast<int>(static_cast<int64_t>(all) * part / p.parts);
  const int n = static_cast<int>(static_cast<int64_t>(all) * (part + 1) / p.parts) - j0;
  const int n0 = kPair ? n : (n + 1) / 2;            // steps of either slot
  const int n1 = kPair ? (two ? n : 0) : n / 2;

  // The stage of K or V tile c, its barriers and the use of it that this is.
  struct Stage {
    uint32_t at;
    uint64_t *full, *empty;
    int use;
  };
  auto k_stage = [&](int c) -> Stage {
    const int u = C::k8 ? 2 * c : c, st = u % C::kK;
    return {sK + st * kTileBytes, &bars.k_full[st], &bars.k_empty[st], u / C::kK};
  };
  auto v_stage = [&](int c) -> Stage {
    if constexpr (C::k8) {
      const int u = 2 * c + 1, st = u % C::kK;
      return {sK + st * kTileBytes, &bars.k_full[st], &bars.k_empty[st], u / C::kK};
    } else {
      const int st = c % C::kV;
      return {sV + st * kTileBytes, &bars.v_full[st], &bars.v_empty[st], c / C::kV};
    }
  };
  auto wait_all = [&](uint64_t* bar, uint32_t parity, uint32_t site) -> bool {
    const bool good = __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, abortp));
    if (!good && lane == 0) record_timeout(p.status, site);
    return good;
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA: Q, then K or codes
    reg_dealloc<C::kUtil>();
    if (lane == 0 && n > 0) {
      const uint32_t q_bytes = static_cast<uint32_t>(p.tile_b * p.tile_pos * p.q.group) * 128u;  // of a half
      for (int t = 0; t < (two ? 2 : 1); ++t) {
        const int tile = tile0 + t;
        const int b = seq * p.s.n + (p.pos_tiles == 1 ? tile * p.tile_b : tile / p.pos_tiles);
        const int pos = p.pos_tiles == 1 ? 0 : tile % p.pos_tiles * p.tile_pos;
        const uint32_t bar = smem_u32(&bars.q_full[t]);
        mbar_expect_tx(bar, 2 * q_bytes);
        tma_load_4d(sQ + t * kTileBytes, &maps.q, bar, 0, hk * p.q.group, pos, b);
        tma_load_4d(sQ + t * kTileBytes + kHalfBytes, &maps.q, bar, 64, hk * p.q.group, pos, b);
      }
      if constexpr (C::k8) {
        bool ok = true;
        int c = 0;
        for (; c < 2 * n; ++c) {  // K and V in turn
          const int st = c % C::kRaw, use = c / C::kRaw, key = (j0 + c / 2) * kTile;
          if (use > 0 && !mbar_wait(smem_u32(&bars.raw_empty[st]), (use - 1) & 1, abortp)) {
            record_timeout(p.status, 91);
            ok = false;
            break;
          }
          if (use > 0) fence_proxy_async_smem();  // (the consumers' reads, behind the wait above, before the copy)
          const uint32_t bar = smem_u32(&bars.raw_full[st]);
          mbar_expect_tx(bar, kRawBytes + (c & 1 ? 0u : 1024u));
          tma_load_4d(sRaw + st * kRawBytes, (c & 1) ? &maps.v : &maps.k, bar, 0, hk, key, seq);
          if ((c & 1) == 0) {  // (both scales with the keys: the softmax needs them first)
            const uint32_t at = sRawScale + st % C::kRawScales * 1024;
            tma_load_4d(at, &maps.ks, bar, key, hk, seq, 0);
            tma_load_4d(at + 512, &maps.vs, bar, key, hk, seq, 0);
          }
        }
        if (!ok) {
          // give copies already in flight a bounded chance to land before the CTA retires
          volatile uint32_t none = 0;
          for (int i = c > C::kRaw ? c - C::kRaw : 0; i < c; ++i)
            mbar_wait(smem_u32(&bars.raw_full[i % C::kRaw]), (i / C::kRaw) & 1, &none);
        }
      } else {
        bool ok = true;
        int c = 0;
        for (; c < n; ++c) {
          const int st = c % C::kK, use = c / C::kK;
          if (use > 0 && !mbar_wait(smem_u32(&bars.k_empty[st]), (use - 1) & 1, abortp)) {
            record_timeout(p.status, 92);
            ok = false;
            break;
          }
          const uint32_t bar = smem_u32(&bars.k_full[st]);
          mbar_expect_tx(bar, kTileBytes);
          tma_load_4d(sK + st * kTileBytes, &maps.k, bar, 0, hk, (j0 + c) * kTile, seq);
          tma_load_4d(sK + st * kTileBytes + kHalfBytes, &maps.k, bar, 64, hk, (j0 + c) * kTile, seq);
        }
        if (!ok) {
          volatile uint32_t none = 0;
          for (int i = c > C::kK ? c - C::kK : 0; i < c; ++i)
            mbar_wait(smem_u32(&bars.k_full[i % C::kK]), (i / C::kK) & 1, &none);
        }
      }
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ TMA: V
    reg_dealloc<C::kUtil>();
    if (!C::k8 && lane == 0) {
      bool ok = true;
      int c = 0;
      for (; c < n; ++c) {
        const int st = c % C::kV, use = c / C::kV;
        if (use > 0 && !mbar_wait(smem_u32(&bars.v_empty[st]), (use - 1) & 1, abortp)) {
          record_timeout(p.status, 93);
          ok = false;
          break;
        }
        const uint32_t bar = smem_u32(&bars.v_full[st]);
        mbar_expect_tx(bar, kTileBytes);
        tma_load_4d(sV + st * kTileBytes, &maps.v, bar, 0, hk, (j0 + c) * kTile, seq);
        tma_load_4d(sV + st * kTileBytes + kHalfBytes, &maps.v, bar, 64, hk, (j0 + c) * kTile, seq);
      }
      if (!ok) {
        volatile uint32_t none = 0;
        for (int i = c > C::kV ? c - C::kV : 0; i < c; ++i)
          mbar_wait(smem_u32(&bars.v_full[i % C::kV]), (i / C::kV) & 1, &none);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ QK^T issuer
    // Step j of slot 0, step j of slot 1, step j + 1 of slot 0, ...: each when the softmax warps have the one before
    // it in registers.
    reg_dealloc<C::kUtil>();
    constexpr uint32_t kFmtBits = kBF16 && !C::k8 ? UMMA_BF16 : UMMA_F16;
    constexpr uint32_t idesc = umma_idesc_f16(kFmtBits, UMMA_K_MAJOR, UMMA_K_MAJOR, 128, 128);
    bool ok = true;
    uint32_t uses = 0;  // of S so far
    for (int j = 0; j < n0 && ok; ++j) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (j >= (t ? n1 : n0)) continue;
        const Stage k = k_stage(kPair ? j : 2 * j + t);
        const bool k_hit = mbar_try_wait(smem_u32(k.full), k.use & 1);
        const bool s_hit = uses == 0 || mbar_try_wait(smem_u32(&bars.s_free), (uses - 1) & 1);
        if (j == 0 && (kPair || t == 0)) ok = wait_all(C::k8 && kBF16 ? &bars.q_ready[t] : &bars.q_full[t], 0, 94);
        if (ok && !__all_sync(0xffffffffu, k_hit)) ok = wait_all(k.full, k.use & 1, 95);
        if (ok && !__all_sync(0xffffffffu, s_hit)) ok = wait_all(&bars.s_free, (uses - 1) & 1, 96);
        if (!ok) break;
        ++uses;
        tc_fence_after_sync();
        if (elect_one()) {
          const uint64_t kdesc = umma_smem_desc_sw128(k.at, 16, 1024);
          const uint64_t qdesc = umma_smem_desc_sw128(sQ + (kPair ? t : 0) * kTileBytes, 16, 1024);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            const uint64_t off = static_cast<uint64_t>((kk & 3) * 2 + (kk >> 2) * (kHalfBytes >> 4));
            umma_ss(tbase, qdesc + off, kdesc + off, idesc, kk > 0 ? 1u : 0u);
          }
          umma_commit(smem_u32(&bars.s_full[t]));
          // the K stage is free after the last QK^T that reads it
          if (!kPair || t == 1 || !two) umma_commit(smem_u32(k.empty));
        }
        __syncwarp();
      }
    }
  } else if (warp == 3) {
    // ------------------------------------------------------------------ P.V issuer
    reg_dealloc<C::kUtil>();
    constexpr uint32_t kFmtBits = kBF16 && !C::k8 ? UMMA_BF16 : UMMA_F16;
    constexpr uint32_t idesc = umma_idesc_f16(kFmtBits, UMMA_K_MAJOR, UMMA_MN_MAJOR, 128, 128);
    bool ok = true;
    int cleared = -1;
    for (int j = 0; j < n0 && ok; ++j) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (j >= (t ? n1 : n0)) continue;
        const int c = kPair ? j : 2 * j + t;
        const Stage v = v_stage(c);
        ok = wait_all(v.full, v.use & 1, 97);
        if (!ok) break;
        if (!C::k8 && (j0 + c + 1) * kTile > len && cleared != c) {
          // what lies behind the sequence may be infinite or NaN, and its weights of 0 would not stop that
          cleared = c;
          const int live = len - (j0 + c) * kTile;
          const uint32_t zero[4] = {0, 0, 0, 0};
          for (int i = live * 16 + lane; i < kTile * 16; i += 32)
            sts4(v.at + (i & 8) * (kHalfBytes / 8) + (i >> 4) * 128 + (i & 7) * 16, zero);
          fence_proxy_async_smem();
          __syncwarp();
        }
        ok = wait_all(&bars.p_ready[t], j & 1, 98);
        if (!ok) break;
        tc_fence_after_sync();
        if (elect_one()) {
          const uint64_t vdesc = umma_smem_desc_sw128(v.at, kHalfBytes, 1024);
          const uint32_t tP = tbase + 128 + t * 64, tO = tbase + 256 + t * 128;
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            umma_ts(tO, tP + kk * 8, vdesc + static_cast<uint64_t>(kk * (2048 >> 4)), idesc, (j > 0 || kk > 0) ? 1u : 0u);
          umma_commit(smem_u32(&bars.pv_done[t]));
          // the V stage is free after the last P.V that reads it
          if (!kPair || t == 1 || !two) umma_commit(smem_u32(v.empty));
        }
        __syncwarp();
      }
    }
  } else if (warp >= 12) {
    // ------------------------------------------------------------------ codes to f16 tiles, a row to a thread
    if constexpr (C::k8) {
      reg_dealloc<C::kConvert>();
      bool ok = true;
      if constexpr (kBF16) {
        const int row = tid - 384;
        for (int t = 0; t < (two ? 2 : 1) && n > 0 && ok; ++t) {
          ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars.q_full[t]), 0, abortp));
          if (!ok) break;
          float top = 0.f;
#pragma unroll
          for (int ch = 0; ch < 16; ++ch) {
            uint32_t w[4];
            lds4(sQ + t * kTileBytes + (ch >> 3) * kHalfBytes + sw128_offset(row, ch & 7), w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 v = unpack2<true>(w[i]);
              top = max3(top, fabsf(v.x), fabsf(v.y));
            }
          }
          // (rows of zeros, and of nothing but values under 2^-100, stay as they are or vanish: logits of 0)
          const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23), 27), 253);
          const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
          unit_s[t][row] = static_cast<uint8_t>(e);
#pragma unroll 4
          for (int ch = 0; ch < 16; ++ch) {
            const uint32_t at = sQ + t * kTileBytes + (ch >> 3) * kHalfBytes + sw128_offset(row, ch & 7);
            uint32_t w[4];
            lds4(at, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 v = unpack2<true>(w[i]);
              w[i] = pack2<false>(v.x * down, v.y * down);
            }
            sts4(at, w);
          }
          fence_proxy_async_smem();
          mbar_arrive(smem_u32(&bars.q_ready[t]));
        }
      }
      const int row = tid - 384;
      float vs = 0.f;               // the row's value scale, from the keys' turn to the values'
      float v_up = 0.f;             // 2^-e of the tile
      int v_least = kLeast;         // (e does not fall by more than 40 from its largest: what is smaller still is lost in an output)
      uint32_t w[32];               // the row's codes
      bool loaded = false;          // (under the conversion of the tile before)
      for (int c = 0; c < 2 * n && ok; ++c) {
        const int st = c % C::kRaw, j = c >> 1;
        const bool is_v = c & 1;
        const Stage to = is_v ? v_stage(j) : k_stage(j);
        const bool live = (j0 + j) * kTile + row < len;  // (what lies behind the sequence may be anything)
        if (!loaded) {
          ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars.raw_full[st]), (c / C::kRaw) & 1, abortp));
          if (!ok) break;
          const uint32_t src = sRaw + st * kRawBytes;
#pragma unroll
          for (int ch = 0; ch < 8; ++ch) lds4(src + sw128_offset(row, ch), w + 4 * ch);
        }
        float scale;
        if (!is_v) {
          const uint32_t at = sRawScale + st % C::kRawScales * 1024;
          scale = live ? ldsf(at + row * 4) : 0.f;
          vs = live ? ldsf(at + 512 + row * 4) : 0.f;
          // exponents of the largest of the warp's 32 key scales, and of all 128 value scales: the four warps' are the same, so that
          // none falls far below the others' in the softmax (of what is finite: the others are what they are)
          auto bits = [](float x) {
            const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
            return b < 0x7f800000u ? b : 0u;
          };
          auto exponent = [](uint32_t b) { return static_cast<int>(__reduce_max_sync(0xffffffffu, b) >> 23) - 127; };
          [[maybe_unused]] int ke;
          if constexpr (!C::kExact) {
            ke = min(max(exponent(bits(scale)), -100), 126);
          }
          float four[4];
          lds4(at + 512 + lane * 16, reinterpret_cast<uint32_t*>(four));
          const int there = len - (j0 + j) * kTile;  // (what lies behind the sequence may be anything)
          if (there < kTile) {
#pragma unroll
            for (int i = 0; i < 4; ++i) four[i] = lane * 4 + i < there ? four[i] : 0.f;
          }
          int v_top = exponent(__float_as_uint(fmaxf(fmaxf(fabsf(four[0]), fabsf(four[1])), fmaxf(fabsf(four[2]), fabsf(four[3])))));
          if (v_top == 128) v_top = exponent(max(max(bits(four[0]), bits(four[1])), max(bits(four[2]), bits(four[3]))));
          v_least = max(v_least, v_top - 40);
          const int ve = min(max(v_top, v_least), 126);
          v_up = __uint_as_float(static_cast<uint32_t>(127 - ve) << 23);
          if constexpr (C::kExact) {
            float* s = reinterpret_cast<float*>(scales_s[j % C::kPowers]);
            s[row] = scale;
            s[kTile + row] = vs * v_up;
            __syncwarp();
          } else {
            scale *= __uint_as_float(static_cast<uint32_t>(127 - ke) << 23);
          }
          if (lane == 0) {
            if constexpr (!C::kExact)
              reinterpret_cast<float*>(&k_power_s[j % C::kPowers])[warp - 12] = __uint_as_float(static_cast<uint32_t>(127 + ke) << 23);
            if (warp == 12) v_power_s[j % C::kPowers] = make_float2(static_cast<float>(ve), v_up * kLiftUp);
            mbar_arrive(smem_u32(&bars.powers_full[j % C::kPowers]));
          }
        } else {
          scale = vs * v_up;
        }
        if (!live) {  // (codes may be NaN)
#pragma unroll
          for (int i = 0; i < 32; ++i) w[i] = 0u;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bars.raw_empty[st]));
        if (to.use > 0) {
          ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(to.empty), (to.use - 1) & 1, abortp));
          if (!ok) break;
        }
        const int next = (c + 1) % C::kRaw;
        loaded = c + 1 < 2 * n && __all_sync(0xffffffffu, mbar_test_wait(smem_u32(&bars.raw_full[next]), ((c + 1) / C::kRaw) & 1));
        const __half hi = __float2half_rn(scale), lo = __float2half_rn(scale - __half2float(hi));
        const __half2 hi2 = __half2half2(hi), lo2 = __half2half2(lo);
#pragma unroll
        for (int ch = 0; ch < 8; ++ch) {
          uint32_t y[8];
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            codes_to_f16<kFmt>(w[4 * ch + z], y[2 * z], y[2 * z + 1]);
#pragma unroll
            for (int x = 0; x < (C::kExact ? 0 : 2); ++x) {
              __half2& v = *reinterpret_cast<__half2*>(&y[2 * z + x]);
              v = __hfma2(v, hi2, __hmul2(v, lo2));
            }
          }
          const uint32_t half = to.at + (ch >> 2) * kHalfBytes;
          sts4(half + sw128_offset(row, (ch & 3) * 2), y);
          sts4(half + sw128_offset(row, (ch & 3) * 2 + 1), y + 4);
          if (loaded) lds4(sRaw + next * kRawBytes + sw128_offset(row, ch), w + 4 * ch);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(to.full));
      }
      if (!ok && lane == 0) record_timeout(p.status, 99);
    }
  } else {
    // ------------------------------------------------------------------ softmax + epilogue
    reg_alloc<C::kSoftmax>();
    const int t = (warp - 4) >> 2;
    const int wq = warp & 3;                     // TMEM lane quarter this warp may touch
    const int r_in_tile = wq * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>(wq * 32) << 16;
    const uint32_t tS = tbase + lane_base;
    const uint32_t tP = tbase + lane_base + 128 + t * 64;
    const uint32_t tO = tbase + lane_base + 256 + t * 128;
    float mul = p.scale_log2;
    const int n_t = t ? n1 : n0;
    // this thread's query row
    const int tile = tile0 + (kPair ? t : 0);
    bool live = (!kPair || t == 0 || two) && r_in_tile < p.tile_b * p.tile_pos * p.q.group;
    int64_t number = 0, out_at = 0, lse_at = 0;
    int lim = len - 1, min_lim = len - 1;        // last visible key of the row, and the least of the tile's
    {
      const int per = p.tile_pos * p.q.group;    // rows of a sequence in the tile
      const int i = p.pos_tiles == 1 ? tile * p.tile_b + r_in_tile / per : tile / p.pos_tiles;
      const int first_pos = p.pos_tiles == 1 ? 0 : tile % p.pos_tiles * p.tile_pos;
      const int pos = first_pos + r_in_tile % per / p.q.group;
      live = live && i < p.s.n && pos < p.q.Sq;
      const int64_t b = seq * p.s.n + i, h = hk * p.q.group + r_in_tile % p.q.group;
      number = (b * p.q.Sq + pos) * p.q.H + h;
      out_at = b * p.o_sb + pos * p.o_ss + h * p.o_sh;
      lse_at = (b * p.q.H + h) * p.q.Sq + pos;
      if (p.s.causal) {
        lim = min(lim, pos + len - p.q.Sq);
        min_lim = min(min_lim, first_pos + len - p.q.Sq);
      }
    }
    bool ok = true;
    float m_ref = -INFINITY;             // exponent reference of this row, in log2 units of the scaled logit
    float l = 0.f;                       // row sum under the current reference; 8 bits: times 2^kLift
    for (int j = 0; j < n_t && ok; ++j) {
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars.s_full[t]), j & 1, abortp));
      if (!ok) { if (lane == 0) record_timeout(p.status, 100); break; }
      tc_fence_after_sync();
      const int jk = (j0 + (kPair ? j : 2 * j + t)) * kTile;  // first key of this tile
      const int thr = lim - jk;  // columns > thr of this tile are masked for this row
      // The whole 128-wide row goes to registers at once, and S to the next QK^T.
      float e[128];
      float4 k_power;   // (8 bits) of the tile's quarters
      float2 v_power;
      {
        uint32_t(&u)[128] = *reinterpret_cast<uint32_t(*)[128]>(e);
        tmem_ld32(tS + 0, *reinterpret_cast<uint32_t(*)[32]>(&u[0]));
        tmem_ld32(tS + 32, *reinterpret_cast<uint32_t(*)[32]>(&u[32]));
        tmem_ld32(tS + 64, *reinterpret_cast<uint32_t(*)[32]>(&u[64]));
        tmem_ld32(tS + 96, *reinterpret_cast<uint32_t(*)[32]>(&u[96]));
        if constexpr (C::k8) {
          const int c = kPair ? j : 2 * j + t;  // the tile, of the CTA's
          ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars.powers_full[c % C::kPowers]), (c / C::kPowers) & 1, abortp));
          if constexpr (!C::kExact) k_power = k_power_s[c % C::kPowers];
          v_power = v_power_s[c % C::kPowers];
        }
        tmem_wait_ld();
      }
      if (C::k8 && !ok) { if (lane == 0) record_timeout(p.status, 103); break; }
      tc_fence_before_sync();
      mbar_arrive(smem_u32(&bars.s_free));
      const float4* scale = scales_s[C::kExact ? (2 * j + t) % C::kPowers : 0][0];
      if constexpr (C::kExact) {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float4 f = scale[i];
          const float2 a = __fmul2_rn(make_float2(e[4 * i], e[4 * i + 1]), make_float2(f.x, f.y));
          const float2 b = __fmul2_rn(make_float2(e[4 * i + 2], e[4 * i + 3]), make_float2(f.z, f.w));
          e[4 * i] = a.x;
          e[4 * i + 1] = a.y;
          e[4 * i + 2] = b.x;
          e[4 * i + 3] = b.y;
        }
      }
      if (C::k8 && kBF16 && j == 0) mul = p.scale_log2 * __uint_as_float(static_cast<uint32_t>(unit_s[kPair ? t : 0][r_in_tile]) << 23);
      if (jk + kTile - 1 > min_lim) {
#pragma unroll
        for (int i = 0; i < 128; ++i) e[i] = (i > thr) ? -INFINITY : e[i];
      }
      // The tile's row maximum is the reference of a first tile; a later one only moves the reference up
      // (and rescales what was accumulated under the old one) when it exceeds it by too much.
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // of the quarters
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
#pragma unroll
        for (int g = 0; g < 4; ++g) mx4[g] = max3(mx4[g], e[32 * g + i], e[32 * g + i + 1]);
      }
      float mx;
      [[maybe_unused]] float factor[4];  // (8 bits) of the quarters' logits; not 0, which masked ones, -inf, would make NaN
      if constexpr (C::k8) {
        if constexpr (C::kExact) {
          mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * mul + v_power.x;
        } else {
          const float of[4] = {k_power.x, k_power.y, k_power.z, k_power.w};
          mx = -INFINITY;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            factor[g] = fmaxf(mul * of[g], 0x1p-126f);
            mx = fmaxf(mx, mx4[g] * factor[g]);
          }
          mx += v_power.x;
        }
      } else {
        mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * mul;
      }
      if (j == 0) {
        m_ref = mx;
      } else {
        const bool need = live && mx > m_ref + kRescaleLimit;
        if (__any_sync(0xffffffffu, need)) {
          float alpha = 1.f;
          if (need) {
            const float step = C::k8 ? half_step(m_ref, mx) : ex2(m_ref - mx);
            alpha = C::k8 ? step * step : step;
            m_ref = mx;
            l = (C::k8 ? l * step : l) * step;
          }
          // O_t is the sum over this slot's earlier tiles, complete with their last P.V
          ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars.pv_done[t]), (j - 1) & 1, abortp));
          if (!ok) { if (lane == 0) record_timeout(p.status, 101); break; }
          tc_fence_after_sync();
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint32_t o[16];
            tmem_ld16(tO + c * 16, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st16(tO + c * 16, o);
          }
          tmem_wait_st();
        }
      }
      // two logits per FMA instruction (packed f32x2); P is packed to 16 bits right away
      const float ref = m_ref > -INFINITY ? m_ref : 0.f;
      float2 ts4[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      uint32_t pk[64];
      if constexpr (C::k8) {
        const float up = v_power.x - ref;
        const float2 up2 = make_float2(up, up);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float f = C::kExact ? mul : factor[g];
          const float2 mul2 = make_float2(f, f);
#pragma unroll
          for (int i = 16 * g; i < 16 * g + 16; ++i) {
            float2 v = __ffma2_rn(make_float2(e[2 * i], e[2 * i + 1]), mul2, up2);
            v.x = ex2(v.x);
            v.y = ex2(v.y);
            ts4[g] = __fadd2_rn(ts4[g], v);
            if constexpr (C::kExact) v = __fmul2_rn(v, reinterpret_cast<const float2*>(scale + kTile / 4)[i]);
            pk[i] = pack2<false>(v.x, v.y);
          }
          l = fmaf(ts4[g].x + ts4[g].y, v_power.y, l);
        }
      } else {
        const float2 mul2 = make_float2(mul, mul), neg_m2 = make_float2(-ref, -ref);
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          float2 v = __ffma2_rn(make_float2(e[2 * i], e[2 * i + 1]), mul2, neg_m2);
          v.x = ex2(v.x);
          v.y = ex2(v.y);
          ts4[i & 3] = __fadd2_rn(ts4[i & 3], v);
          pk[i] = pack2<kBF16>(v.x, v.y);
        }
        const float2 ts2 = __fadd2_rn(__fadd2_rn(ts4[0], ts4[1]), __fadd2_rn(ts4[2], ts4[3]));
        l += ts2.x + ts2.y;
      }
      if (j > 0) {  // P_t is free when the last P.V has read it
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars.pv_done[t]), (j - 1) & 1, abortp));
        if (!ok) { if (lane == 0) record_timeout(p.status, 101); break; }
        tc_fence_after_sync();
      }
      tmem_st32(tP, *reinterpret_cast<uint32_t(*)[32]>(&pk[0]));
      tmem_st32(tP + 32, *reinterpret_cast<uint32_t(*)[32]>(&pk[32]));
      tmem_wait_st();
      tc_fence_before_sync();
      mbar_arrive(smem_u32(&bars.p_ready[t]));
    }
    if (n_t > 0 && ok) {
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars.pv_done[t]), (n_t - 1) & 1, abortp));
      if (!ok && lane == 0) record_timeout(p.status, 102);
      tc_fence_after_sync();
    }
    // ---- the part's results: unnormalised O, reference, sum
    const float take = C::k8 ? unlift(m_ref, l) : 1.f;  // (of this slot's O)
    if (l == 0.f) m_ref = -INFINITY;                // (nothing seen)
    else if (!(m_ref > -INFINITY)) m_ref = 0.f;     // (nothing but NaN: the sum)
    if constexpr (!kFinish) {
      float* orow = p.mine.o + (number * p.mine.parts + part) * 128;
      float2* ml = reinterpret_cast<float2*>(p.mine.ml) + number * p.mine.parts + part;
      if constexpr (kPair) {
        if (live) *ml = make_float2(m_ref, l);
        if (n_t > 0) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t o[32];
            tmem_ld32(tO + c * 32, o);
            tmem_wait_ld();
            if constexpr (C::k8) {
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * take);
            }
            if (live) {
#pragma unroll
              for (int g = 0; g < 4; ++g) st_global_v8(orow + c * 32 + g * 8, &o[g * 8]);
            }
          }
        }
      } else {
        // the slots' factors to a common reference; each writes half of the columns
        // (every softmax warp gets to the barriers, expired waits or not)
        if (t == 1) {
          row_s[r_in_tile] = make_float2(m_ref, l);
          if constexpr (C::k8) take_s[r_in_tile] = take;
        }
        tc_fence_before_sync();
        named_bar_sync(1, 256);
        float f0, f1;
        if (t == 0) {
          const float2 o = row_s[r_in_tile];
          const float mm = fmaxf(m_ref, o.x);
          f0 = m_ref > -INFINITY ? ex2(m_ref - mm) : 0.f;
          f1 = o.x > -INFINITY ? ex2(o.x - mm) : 0.f;
          if (live) *ml = make_float2(mm, fmaf(f1, o.y, f0 * l));
          if constexpr (C::k8) {
            f0 *= take;
            f1 *= take_s[r_in_tile];
          }
          row_s[r_in_tile] = make_float2(f0, f1);
        }
        named_bar_sync(1, 256);
        tc_fence_after_sync();
        if (t == 1) {
          f0 = row_s[r_in_tile].x;
          f1 = row_s[r_in_tile].y;
        }
        const uint32_t tA = tbase + lane_base + 256 + t * 64;
        if (n > 0) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t o0[32], o1[32];
            tmem_ld32(tA + c * 32, o0);
            if (n1 > 0) tmem_ld32(tA + 128 + c * 32, o1);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              float y = __uint_as_float(o0[i]) * f0;
              if (n1 > 0) y = fmaf(__uint_as_float(o1[i]), f1, y);
              o0[i] = __float_as_uint(y);
            }
            if (live) {
#pragma unroll
              for (int g = 0; g < 4; ++g) st_global_v8(orow + t * 64 + c * 32 + g * 8, &o0[g * 8]);
            }
          }
        }
      }
    } else {
      // 32 columns from `col` on, zeros where nothing was seen
      auto put = [&](const float (&o)[32], int col) {
        if (!live) return;
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = pack2<kBF16>(o[2 * i], o[2 * i + 1]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<uint4*>(p.out + out_at + col + 8 * i) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      };
      float f0 = l == 0.f ? 0.f : take / l, f1 = 0.f, ref = m_ref, sum = l;
      if constexpr (!kPair) {
        if (t == 1) {
          row_s[r_in_tile] = make_float2(m_ref, l);
          if constexpr (C::k8) take_s[r_in_tile] = take;
        }
        tc_fence_before_sync();
        named_bar_sync(1, 256);
        if (t == 0) {
          const float2 o = row_s[r_in_tile];
          ref = fmaxf(m_ref, o.x);
          f0 = m_ref > -INFINITY ? ex2(m_ref - ref) : 0.f;
          f1 = o.x > -INFINITY ? ex2(o.x - ref) : 0.f;
          sum = fmaf(f1, o.y, f0 * l);
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          f0 *= inv * take;
          f1 *= C::k8 ? inv * take_s[r_in_tile] : inv;
          row_s[r_in_tile] = make_float2(f0, f1);
        }
        named_bar_sync(1, 256);
        tc_fence_after_sync();
        if (t == 1) {
          f0 = row_s[r_in_tile].x;
          f1 = row_s[r_in_tile].y;
        }
      }
      if (live && p.lse2 != nullptr && (kPair || t == 0)) p.lse2[lse_at] = ref + log2f(sum);
      // (two tiles: a slot's own 128 columns; one: half of both accumulators')
      const uint32_t tA = kPair ? tO : tbase + lane_base + 256 + t * 64;
#pragma unroll
      for (int c = 0; c < (kPair ? 4 : 2); ++c) {
        uint32_t o0[32], o1[32];
        float y[32];
        if (n > 0) {
          tmem_ld32(tA + c * 32, o0);
          if (!kPair && n1 > 0) tmem_ld32(tA + 128 + c * 32, o1);
          tmem_wait_ld();
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          y[i] = n > 0 ? __uint_as_float(o0[i]) * f0 : 0.f;
          if (!kPair && n1 > 0) y[i] = fmaf(__uint_as_float(o1[i]), f1, y[i]);
        }
        put(y, kPair ? c * 32 : t * 64 + c * 32);
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tbase, 512);
  }
  if (p.chained) griddep_wait();
}

// ---- merge: parts in the order of the keys -------------------------------------------------------------
// Bound by latency: first what says where the parts lie, for both segments at once, then the parts, up to kBatch of a warp in flight.
struct MergeParams {
  Source in[2];
  bool finished;
  int workers;
  RowShape q;
  uint16_t* out;
  int64_t o_sb, o_ss, o_sh;
  float* lse2;
  int B;
};
// One segment's parts of a row: the first, and the others `step` rows from one to the next.
struct Parts {
  int count;
  const float* first_o;
  const float* first_ml;
  const float* o;
  const float* ml;
  int64_t step;
};
__device__ __forceinline__ Parts parts_of(const Source& f, const RowShape& q, int workers, int row, int b, int pos, int h) {
  Parts x;
  if (!f.dealt) {
    x.count = f.fixed.parts;
    x.first_o = f.fixed.o + static_cast<int64_t>(row) * x.count * 128;
    x.first_ml = f.fixed.ml + static_cast<int64_t>(row) * x.count * 2;
    x.o = x.first_o;
    x.ml = x.first_ml;
    x.step = 1;
    return x;
  }
  const Dealt& d = f.deal;
  const int seq = b / f.segment.n;
  const int2 w = d.workers[static_cast<int64_t>(seq) * q.Hkv + h / q.group];
  const bool some = seen_of(f.segment, seq) > 0;
  x.count = some ? min(max(w.y - w.x, 0) + 1, workers) : 0;  // (bounded, should another stream have changed the length)
  const int r = ((b - seq * f.segment.n) * q.Sq + pos) * q.group + h % q.group;
  const int64_t at = static_cast<int64_t>(min(max(w.x, 0), workers - x.count)) * 2 * d.slot_rows + r;
  x.o = d.slot_o + at * 128;    // slot 0, of all workers but the first
  x.ml = d.slot_ml + at * 2;
  x.step = 2 * d.slot_rows;
  x.first_o = x.count == 1 ? d.whole_o + static_cast<int64_t>(row) * 128 : x.o + static_cast<int64_t>(d.slot_rows) * 128;
  x.first_ml = x.count == 1 ? d.whole_ml + static_cast<int64_t>(row) * 2 : x.ml + static_cast<int64_t>(d.slot_rows) * 2;
  return x;
}

// kWarps warps to a query row, each with every kWarps-th part, four columns to a lane.
constexpr int kMergeThreads = 256;
template <bool kBF16, int kWarps>
__global__ void __launch_bounds__(kMergeThreads) attn_merge_kernel(const MergeParams p) {
  __shared__ float4 acc_s[kWarps > 1 ? kWarps : 1][32];
  __shared__ float2 ml_s[kWarps > 1 ? kWarps : 1];
  const int lane = threadIdx.x & 31, w = (threadIdx.x >> 5) % kWarps;
  const int row = static_cast<int>(blockIdx.x) * (kMergeThreads / 32 / kWarps) + static_cast<int>(threadIdx.x >> 5) / kWarps;
  const int h = row % p.q.H, pos = row / p.q.H % p.q.Sq, b = row / p.q.H / p.q.Sq;
  griddep_wait();
  griddep_launch_dependents();
  if (b >= p.B) return;  // (with more warps than one a row is a CTA)
  const Parts x0 = parts_of(p.in[0], p.q, p.workers, row, b, pos, h), x1 = parts_of(p.in[1], p.q, p.workers, row, b, pos, h);
  if (p.finished && x1.count == 1) return;
  const int count = x0.count + x1.count;
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int kBatch = 10;
  for (int i0 = w; i0 < count; i0 += kBatch * kWarps) {
    float2 ml[kBatch];
    float4 o[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int part = i0 + i * kWarps;
      ml[i] = make_float2(-INFINITY, 0.f);
      if (part < count) {
        const bool second = part >= x0.count;
        const int y = second ? part - x0.count : part;
        const int64_t off = y * (second ? x1.step : x0.step);
        const float* at_o = second ? (y == 0 ? x1.first_o : x1.o + off * 128) : (y == 0 ? x0.first_o : x0.o + off * 128);
        const float* at_ml = second ? (y == 0 ? x1.first_ml : x1.ml + off * 2) : (y == 0 ? x0.first_ml : x0.ml + off * 2);
        ml[i] = *reinterpret_cast<const float2*>(at_ml);
        o[i] = reinterpret_cast<const float4*>(at_o)[lane];
      }
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) top = fmaxf(top, ml[i].x);
    const float down = m > -INFINITY ? ex2(m - top) : 0.f;
    m = top;
    l *= down;
    acc = make_float4(acc.x * down, acc.y * down, acc.z * down, acc.w * down);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (ml[i].x > -INFINITY) {  // (a part that saw nothing has left nothing)
        const float f = ex2(ml[i].x - m);
        l = fmaf(f, ml[i].y, l);
        acc.x = fmaf(f, o[i].x, acc.x);
        acc.y = fmaf(f, o[i].y, acc.y);
        acc.z = fmaf(f, o[i].z, acc.z);
        acc.w = fmaf(f, o[i].w, acc.w);
      }
    }
  }
  if constexpr (kWarps > 1) {
    acc_s[w][lane] = acc;
    if (lane == 0) ml_s[w] = make_float2(m, l);
    __syncthreads();
    if (w != 0) return;
    for (int x = 0; x < kWarps; ++x) m = fmaxf(m, ml_s[x].x);
    l = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int x = 0; x < kWarps; ++x) {
      const float2 ml = ml_s[x];
      if (ml.x > -INFINITY) {
        const float4 o = acc_s[x][lane];
        const float f = ex2(ml.x - m);
        l = fmaf(f, ml.y, l);
        acc = make_float4(fmaf(f, o.x, acc.x), fmaf(f, o.y, acc.y), fmaf(f, o.z, acc.z), fmaf(f, o.w, acc.w));
      }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  reinterpret_cast<uint2*>(p.out + b * p.o_sb + pos * p.o_ss + h * p.o_sh)[lane] =
      make_uint2(pack2<kBF16>(acc.x * inv, acc.y * inv), pack2<kBF16>(acc.z * inv, acc.w * inv));
  if (p.lse2 != nullptr && lane == 0) p.lse2[(static_cast<int64_t>(b) * p.q.H + h) * p.q.Sq + pos] = m + log2f(l);
}

// How the rows of a unit make query tiles: whole sequences where one fits, else stretches of one sequence's positions.
struct Tiles {
  int b, pos, pos_tiles, count;
};
Tiles tiles_of(const Segment& s, const RowShape& q) {
  Tiles t;
  const int64_t per = static_cast<int64_t>(q.Sq) * q.group;
  if (per <= kTile) {
    t.b = static_cast<int>(kTile / per);
    if (t.b > s.n) t.b = s.n;
    t.pos = q.Sq;
    t.pos_tiles = 1;
    t.count = (s.n + t.b - 1) / t.b;
  } else {
    t.b = 1;
    t.pos = kTile / q.group;
    t.pos_tiles = (q.Sq + t.pos - 1) / t.pos;
    t.count = s.n * t.pos_tiles;
  }
  return t;
}

template <bool kBF16, int kFmt, bool kPair, bool kFinish>
cudaError_t launch_rows_of(const CacheRows& c, const CacheAttnArgs& a, RowsParams& p, const Tiles& tiles, cudaStream_t stream) {
  using C = Cfg<kBF16, kFmt, kPair>;
  RowsMaps maps;
  const uint32_t box[4] = {64, static_cast<uint32_t>(p.q.group), static_cast<uint32_t>(tiles.pos), static_cast<uint32_t>(tiles.b)};
  if (tma_host::make_boxed_map(&maps.q, a.q, kBF16, a.B, a.Sq, a.H, 128, a.q_sb, a.q_ss, a.q_sh, box) ||
      make_rows_map(&maps.k, c, false, p.q.Hkv, kBF16, kTile) ||
      make_rows_map(&maps.v, c, true, p.q.Hkv, kBF16, kTile))
    return cudaErrorInvalidValue;
  if (C::k8) {
    if (make_scale_map(&maps.ks, c, false, p.q.Hkv, kTile) || make_scale_map(&maps.vs, c, true, p.q.Hkv, kTile))
      return cudaErrorInvalidValue;
  } else {
    maps.ks = maps.vs = maps.k;
  }
  const auto kern = attn_rows_kernel<kBF16, kFmt, kPair, kFinish>;
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), C::kSmem);
  if (e != cudaSuccess) return e;
  e = check_register_budget(reinterpret_cast<const void*>(kern), C::kThreads, C::kBlockRegs);
  if (e != cudaSuccess) return e;
  const unsigned grid = static_cast<unsigned>(static_cast<int64_t>(p.s.N) * p.q.Hkv * p.parts * p.blocks);
  e = launch_dependent(kern, dim3(grid), dim3(C::kThreads), C::kSmem, stream, maps, p);
  count_launch();
  return e;
}

template <bool kBF16, int kFmt>
cudaError_t launch_rows_fmt(const CacheRows& c, const CacheAttnArgs& a, RowsParams& p, const Tiles& tiles, cudaStream_t stream) {
  if (p.out != nullptr)
    return tiles.count > 1 ? launch_rows_of<kBF16, kFmt, true, true>(c, a, p, tiles, stream)
                           : launch_rows_of<kBF16, kFmt, false, true>(c, a, p, tiles, stream);
  return tiles.count > 1 ? launch_rows_of<kBF16, kFmt, true, false>(c, a, p, tiles, stream)
                         : launch_rows_of<kBF16, kFmt, false, false>(c, a, p, tiles, stream);
}

}  // namespace

// Parts of the keys: what makes the CTAs' rounds times the length of one least.  A CTA's set-up, first loads and
// epilogue count as four steps of a tile of keys, with one query tile, whose steps are half as long, as eight.
int attn_rows_parts(const Segment& s, const RowShape& q, int num_sms) {
  const Tiles tiles = tiles_of(s, q);
  const int64_t items = static_cast<int64_t>(s.N) * q.Hkv * ((tiles.count + 1) / 2);
  const int key_tiles = (s.S + kTile - 1) / kTile, fixed = tiles.count > 1 ? 4 : 8;
  int best = 1;
  int64_t least = INT64_MAX;
  for (int parts = 1; parts <= key_tiles && parts <= 64; ++parts) {
    const int64_t cost = (items * parts + num_sms - 1) / num_sms * ((key_tiles + parts - 1) / parts + fixed);
    if (cost < least) {
      least = cost;
      best = parts;
    }
  }
  return best;
}

cudaError_t launch_attn_rows(const CacheRows& c, const Segment& s, const CacheAttnArgs& a, const Partials& mine,
                             bool finish, bool chained, cudaStream_t stream) {
  RowsParams p;
  p.s = s;
  p.q = RowShape{a.Sq, a.H, a.H / a.group, a.group};
  const Tiles tiles = tiles_of(s, p.q);
  p.tile_b = tiles.b;
  p.tile_pos = tiles.pos;
  p.pos_tiles = tiles.pos_tiles;
  p.tiles = tiles.count;
  p.blocks = (tiles.count + 1) / 2;
  p.parts = mine.parts;
  p.scale_log2 = a.softmax_scale * 1.4426950408889634f;
  p.mine = mine;
  p.out = finish ? a.out : nullptr;
  p.o_sb = a.o_sb; p.o_ss = a.o_ss; p.o_sh = a.o_sh;
  p.lse2 = a.lse2;
  p.chained = chained ? 1 : 0;
  p.status = device_status_words();
  if (a.bf16) {
    if (c.format == CACHE_I8) return launch_rows_fmt<true, CACHE_I8>(c, a, p, tiles, stream);
    if (c.format == CACHE_E4M3) return launch_rows_fmt<true, CACHE_E4M3>(c, a, p, tiles, stream);
    return launch_rows_fmt<true, CACHE_16>(c, a, p, tiles, stream);
  }
  if (c.format == CACHE_I8) return launch_rows_fmt<false, CACHE_I8>(c, a, p, tiles, stream);
  if (c.format == CACHE_E4M3) return launch_rows_fmt<false, CACHE_E4M3>(c, a, p, tiles, stream);
  return launch_rows_fmt<false, CACHE_16>(c, a, p, tiles, stream);
}

cudaError_t launch_attn_merge(const CacheAttnArgs& a, const Source& first, const Source& second, bool finished, int workers,
                              cudaStream_t stream) {
  MergeParams p;
  p.in[0] = first;
  p.in[1] = second;
  p.finished = finished;
  p.workers = workers;
  p.q = RowShape{a.Sq, a.H, a.H / a.group, a.group};
  p.out = a.out;
  p.o_sb = a.o_sb; p.o_ss = a.o_ss; p.o_sh = a.o_sh;
  p.lse2 = a.lse2;
  p.B = a.B;
  // Parts of a row: as many as it is given, or as workers share a unit.  A warp has kBatch in flight; eight warps to a row from 17 on
  // (from 11 on, 128 sequences behind 32768 bf16 rows took 23 us longer).
  int64_t parts = 0;
  for (const Source* f : {&first, &second}) {
    if (f->dealt) {
      const int64_t tiles = (f->segment.S + f->deal.keys - 1) / f->deal.keys, units = static_cast<int64_t>(f->segment.N) * p.q.Hkv;
      const int64_t shared = workers / units + 2;
      parts += shared < tiles ? shared : tiles;
    } else {
      parts += f->fixed.parts;
    }
  }
  const bool wide = parts > 16;
  const int64_t rows = static_cast<int64_t>(a.B) * a.Sq * a.H, per_cta = wide ? 1 : kMergeThreads / 32;
  const auto kern = a.bf16 ? (wide ? attn_merge_kernel<true, 8> : attn_merge_kernel<true, 1>)
                           : (wide ? attn_merge_kernel<false, 8> : attn_merge_kernel<false, 1>);
  const cudaError_t e = launch_dependent(kern, dim3(static_cast<unsigned>((rows + per_cta - 1) / per_cta)), dim3(kMergeThreads),
                                         0, stream, p);
  count_launch();
  return e;
}

}  // namespace asuka
