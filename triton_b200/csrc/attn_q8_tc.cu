// Attention over the 8-bit key/value cache for many query rows per kv head (prompts, chunks, many heads on one kv head): the
// mathematics of attn_q8.cu on tcgen05 tensor cores.
//
// The M * Hq / Hkv rows of a (b, kv head) are taken in tiles of 128 (row r = query r / G, head r % G, so a tile of a causal
// call spans few queries); a CTA works on two neighbouring tiles against the same keys, so that one tile's softmax runs
// while the other's products do.
//   warps 0-2    convert: TMA brings the next 128 positions' codes to a raw tile; when a stage is free they are written as
//                fp16 (exact) into the 128-byte-swizzled tiles the tensor core reads, with the scales of their 16-position
//                groups.  (Codes fetched to registers instead made the proxy fence that publishes a tile wait for the
//                fetches under way.)
//   warps 4-7,   softmax of tile 0 / 1, one thread per row: q -> shared memory as fp16 times a power of two; then per block of
//   warps 8-11   128 positions  t = s * (c ks),  E = 2^(t - m'),  l += E,  P' = E vs, packed to fp16 over s in tensor memory
//                (m' as in attn_q8.cu);  o is rescaled only when a row's maximum grew by more than 2^8 since the last time
//   warp 3       issues S_t = q_t k^T and O_t += P'_t v (P' from tensor memory)
// ks enters the multiply-add that the softmax makes anyway, vs costs half a (packed) multiplication a score; both change every
// 16 columns at most.  P' enters as hi + lo, with single_p as one fp16 part (see attn_q8.cu).
// Few CTAs (less than one for each SM): the key blocks are divided among several, merged by the kernel in attn_q8.cu.
//
// Algorithmic flops: 4 * D per visible (row, position).
//
// Measured: 2 x 2048 queries on 8192 positions, 32 / 8 heads of 128, causal, bf16: 685 to 728 us (at the power cap) = 700 to 660
// TFLOP/s, 42 to 40 % of the measured product rate; fp16 698; single_p 609 (790 TFLOP/s) and 597.  Bound by the softmax warps' chain
// (tensor memory -> maximum -> exponential -> tensor memory; ncu: tensor pipe 47 %, ALU 36 %, XU 33 %); with p in one part, without
// conversion 4 % less, without exponentials 12 % less; per CTA 9 us of set-up, q and output.  The 16-bit attention core of this
// library takes 605 us for the shape (single_p 524).
#include <type_traits>

#include "attn_q8.cuh"

namespace trn {
namespace {

constexpr int kTcRows = 128, kTcKeys = 128;
constexpr int kTcThreads = 12 * 32;
constexpr int kTcConvert = 96;                // threads that convert: warps 0-2
constexpr int kTcMmaWarp = 3;
static_assert(kTcConvert == 32 * kTcMmaWarp && kTcThreads == 32 * (kTcMmaWarp + 1 + 8), "warps: convert, MMA, softmax from warp 4");
constexpr int kTcTmemCols = 512;              // S0 [0,128) S1 [128,256) O0 [256,256+D) O1 [384,384+D)
constexpr float kTcRescale = 8.0f;            // log2 units a row's maximum may pass the offset in use
constexpr float kTcPBias = 6.0f;              // P' <= 2^14 with it
// Pieces of a pair at most.  One round and 4 pairs without a mask, 6144 positions: 153 us with 16, 160 with 8; and 12 pairs 156, 159;
// more pairs than that leave room for 8 or less
constexpr int kTcMaxCut = 16;
// 512 pairs without a mask: 16 key blocks 218 us whole, 234 with the last round in pieces; 32: 393, 394; 40: 481, 472; 64: 744, 711
constexpr int kTcMinCutBlocks = 40;
// Key blocks of a pair from which on few pairs are divided, down to one a CTA.  40 queries of 8 heads of 128 on 8: 3 blocks 17.2 us
// whole, 18.7 divided; 4 blocks 19.7 and 18.9 (21.9 with two a CTA at least); 8 blocks 26.8 and 18.8 (22.6); 71 heads of 64 x 16
// queries on one: 3 blocks 15.8, 18.7; 9 blocks 24.9, 19.5 (23.0); from 24 blocks on one and two are alike
constexpr int kTcMinDivide = 4;

struct TcParams {
  Q8Params c;
  int pairs;
  int ctas;          // CTAs the key blocks of all pairs of tiles are divided among; 0: a CTA per pair
  int whole, cut;    // ctas == 0: the first `whole` pairs are not divided, the rest into `cut` pieces each
};

template <int D>
struct TcSmem {
  static constexpr int kStages = D == 128 ? 2 : 4;
  static constexpr int kChunks = D / 64;
  static constexpr int kChunkBytes = 128 * 128;            // 128 rows x 64 fp16
  static constexpr int kTile = kChunks * kChunkBytes;
  static constexpr int kQ = 0;                             // two q tiles
  static constexpr int kKV = 2 * kTile;
  static constexpr int kRaw = kKV + kStages * 2 * kTile;             // codes of k, codes of v
  static constexpr int kRawTile = 128 * D;
  static constexpr int kScales = kRaw + 2 * kRawTile;         // [stage][8 groups] (ks, log2 vs rounded up, vs 2^-18, -)
  static constexpr int kNan = kScales + kStages * 8 * 16;            // [D] first position with a NaN code in v
  static constexpr int kBars = kNan + D * 4;
  static constexpr int kTotal = kBars + 256 + 1024;
};

// 16 codes -> 16 fp16: units `first` and `first ^ 1` of the row, in an order in which 8 lanes' stores meet all banks
__device__ __forceinline__ void expand16(uint32_t tile, uint32_t row, uint32_t unit, bool swap, const uint4& c) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  uint32_t r[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[2 * i] = e4m3x2_to_f16x2(w[i]);
    r[2 * i + 1] = e4m3x2_to_f16x2(w[i] >> 16);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bool hi = (i != 0) != swap;
    const uint32_t a = tile + swz128(row, unit + (hi ? 1u : 0u));
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};"
                 ::"r"(a), "r"(hi ? r[4] : r[0]), "r"(hi ? r[5] : r[1]), "r"(hi ? r[6] : r[2]), "r"(hi ? r[7] : r[3])
                 : "memory");
  }
}

// 32 lanes x 16 consecutive 32-bit columns of tensor memory
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// GRP: positions that share a scale within the kernel, 16 or (blocks of 32 and more) 32
// SPLIT: P' enters the product as two fp16 parts
template <typename T, int D, int GRP, bool SPLIT>
__global__ void __launch_bounds__(kTcThreads, 1)
attn_q8_tc_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                  const __grid_constant__ TcParams tp) {
  using SM = TcSmem<D>;
  constexpr int KS = SM::kStages;
  const Q8Params& p = tp.c;
  extern __shared__ uint8_t tc_smem_raw[];
  const uint32_t base = (smem_u32(tc_smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = tc_smem_raw + (base - smem_u32(tc_smem_raw));
  const uint32_t bars = base + SM::kBars;
  auto k_full = [&](int s) { return bars + 8u * s; };
  auto v_full = [&](int s) { return bars + 8u * (KS + s); };
  auto kv_empty = [&](int s) { return bars + 8u * (2 * KS + s); };
  auto s_full = [&](int t) { return bars + 8u * (3 * KS + t); };
  auto pv_done = [&](int t) { return bars + 8u * (3 * KS + 2 + t); };
  auto q_full = [&](int t) { return bars + 8u * (3 * KS + 4 + t); };
  // P' becomes ready in two halves (positions 0..63, 64..127), so that P' v starts on the first
  auto p_ready = [&](int t, int half) { return bars + 8u * (3 * KS + 6 + 2 * t + half); };
  auto raw_full = [&](int kv) { return bars + 8u * (3 * KS + 10 + kv); };
  auto raw_empty = [&](int kv) { return bars + 8u * (3 * KS + 12 + kv); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gen + SM::kBars + 8 * (3 * KS + 14));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* nan_any = reinterpret_cast<int*>(tmem_slot + 2);
  int* nan_from = reinterpret_cast<int*>(gen + SM::kNan);
  float4* scales = reinterpret_cast<float4*>(gen + SM::kScales);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Ctl ctl{p.status, abort_flag};
  if (threadIdx.x == 0) {
    for (int s = 0; s < KS; ++s) {
      mbar_init(k_full(s), kTcConvert);
      mbar_init(v_full(s), kTcConvert);
      mbar_init(kv_empty(s), 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(s_full(t), 1);
      mbar_init(pv_done(t), 1);
      mbar_init(q_full(t), 128);
      mbar_init(raw_full(t), 1);
      mbar_init(raw_empty(t), kTcConvert);
      mbar_init(p_ready(t, 0), 128);
      mbar_init(p_ready(t, 1), 128);
    }
    *abort_flag = 0;
    *nan_any = 0;
    fence_mbar_init();
  }
  if (threadIdx.x == 32) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  for (int i = threadIdx.x; i < D; i += kTcThreads) nan_from[i] = 0x7fffffff;
  if (warp == kTcMmaWarp) {
    tmem_alloc(smem_u32(tmem_slot), kTcTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  griddep_wait();                              // q, the codes and the lengths may come from the launch before
  griddep_launch();
  bool dead = *reinterpret_cast<volatile int*>(p.status) != 0;

  // ---- which rows and blocks
  const int cta = static_cast<int>(blockIdx.x);
  int b, h, pair, split = 0, pieces = 1;
  if (tp.ctas == 0) {
    int u = cta;                                                   // late (heavy) pairs of tiles first
    if (u >= tp.whole) {                                           // those of the last, incomplete round of CTAs: in pieces
      pieces = tp.cut;
      split = (cta - tp.whole) % tp.cut;
      u = tp.whole + (cta - tp.whole) / tp.cut;
    }
    pair = tp.pairs - 1 - u / (p.B * p.Hkv);
    h = u % p.Hkv;
    b = u / p.Hkv % p.B;
  } else {
    // A pair's key blocks are cut into pieces of at most `share`: the least share with which all pairs' pieces find a CTA
    const int per = p.Hkv * tp.pairs;
    auto blocks_of = [&](int i) { return max((p.len(i) + kTcKeys - 1) / kTcKeys, 1); };
    unsigned sum = 0u;
    for (int i = lane; i < p.B; i += 32) sum += blocks_of(i);
    const int total = static_cast<int>(__reduce_add_sync(0xffffffffu, sum)) * per;
    int share = max((total + tp.ctas - 1) / tp.ctas, 1);
    for (;;) {
      unsigned c = 0u;
      for (int i = lane; i < p.B; i += 32) c += (blocks_of(i) + share - 1) / share;
      if (static_cast<int>(__reduce_add_sync(0xffffffffu, c)) * per <= tp.ctas || share >= total) break;
      share += max(share >> 3, 1);
    }
    int at = cta;
    b = -1;
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      const int c = b0 + lane < p.B ? (blocks_of(b0 + lane) + share - 1) / share * per : 0;
      int incl = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, incl > at);
      if (past != 0u) {
        const int l = __ffs(past) - 1;
        b = b0 + l;
        at -= __shfl_sync(0xffffffffu, incl - c, l);
        break;
      }
      at -= __shfl_sync(0xffffffffu, incl, 31);
    }
    const bool idle = b < 0;                   // more CTAs than pieces: no blocks, and nothing written
    if (idle) b = 0;
    pieces = (blocks_of(b) + share - 1) / share;
    split = idle ? 0 : at % pieces;
    const int u = idle ? 0 : min(at / pieces, per - 1);
    h = u / tp.pairs;
    pair = u % tp.pairs;
    dead = dead || idle;
  }
  const int bh = b * p.Hkv + h;
  const int n = p.len(b);
  int n_blocks[2], lim_max[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int r0 = (2 * pair + t) * kTcRows;
    lim_max[t] = r0 < p.R ? last_seen(p, n, min(r0 + kTcRows, p.R) - 1) : -1;
    n_blocks[t] = (lim_max[t] + kTcKeys) / kTcKeys;
  }
  int j0 = 0;
  if (pieces > 1) {
    const int full = max(n_blocks[0], n_blocks[1]);
    j0 = full * split / pieces;
    const int j1 = full * (split + 1) / pieces;
    n_blocks[0] = max(0, min(j1, n_blocks[0]) - j0);
    n_blocks[1] = max(0, min(j1, n_blocks[1]) - j0);
  }
  if (dead) n_blocks[0] = n_blocks[1] = 0;
  const int n_max = max(n_blocks[0], n_blocks[1]);
  const int first_lim = last_seen(p, n, 2 * pair * kTcRows);       // of the CTA's first row: the least any row sees
  auto q_s = [&](int t) { return base + SM::kQ + t * SM::kTile; };
  auto k_s = [&](int s) { return base + SM::kKV + s * 2 * SM::kTile; };
  auto v_s = [&](int s) { return k_s(s) + SM::kTile; };

  if (warp < kTcConvert / 32) {
    // ------------------------------- convert -------------------------------
    constexpr int SEG = D / 16, UNITS = kTcKeys * SEG;             // 16-byte units of a row, of a raw tile
    constexpr int PER = 4;                                         // units a thread has in hand
    float ks = 1.f, vs = 1.f;
    auto bring = [&](int kv, int j) {                              // thread 0
      mbar_expect_tx(raw_full(kv), SM::kRawTile);
      tma_load_head_tile(base + SM::kRaw + kv * SM::kRawTile, kv == 0 ? &tm_k : &tm_v, raw_full(kv), kv == 0 ? p.ki : p.vi, 0,
                         (j0 + j) * kTcKeys, h, b);
    };
    auto fetch_scales = [&](int j) {
      const int key = (j0 + j) * kTcKeys + 16 * static_cast<int>(threadIdx.x);
      if (threadIdx.x < 8) {
        ks = key < n ? *p.ks.at(b, key >> p.shift, h) : 1.f;
        vs = key < n ? *p.vs.at(b, key >> p.shift, h) : 1.f;
      }
    };
    // raw tile kv of block j -> fp16 tile at dst; edge: some row does not see some position of the block
    auto convert = [&](int kv, uint32_t dst, int kv0, bool edge) {
      const uint32_t raw = base + SM::kRaw + kv * SM::kRawTile;
#pragma unroll 1
      for (int u0 = static_cast<int>(threadIdx.x); u0 < UNITS; u0 += PER * kTcConvert) {
        uint4 c[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const uint32_t u = min(u0 + i * kTcConvert, UNITS - 1);
          c[i] = lds128(raw + q8_off<D>(u / SEG, u % SEG));
        }
        if (edge && kv == 1) {
          // v behind the sequence counts as 0 whatever lies there, and so do NaN codes, whose first positions are kept
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            const int u = min(u0 + i * kTcConvert, UNITS - 1), key = kv0 + u / SEG;
            uint32_t w[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (key >= n) w[e] = 0u;
              const uint32_t bad = nan_bytes(w[e]);
              if (bad != 0u) {
                w[e] &= ~bad;
                *nan_any = 1;
                for (int x = 0; x < 4; ++x)
                  if ((bad >> (8 * x)) & 1u) atomicMin(&nan_from[u % SEG * 16 + 4 * e + x], key);
              }
            }
            c[i] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const uint32_t u = u0 + i * kTcConvert, seg = u % SEG;
          if (u < UNITS) expand16(dst + (seg >> 2) * SM::kChunkBytes, u / SEG, (seg & 3) * 2, seg >= 4, c[i]);
        }
      }
      fence_proxy_async_smem();
    };
    if (n_max > 0) {
      if (threadIdx.x == 0) {
        bring(0, 0);
        bring(1, 0);
      }
      fetch_scales(0);
    }
    for (int j = 0; j < n_max; ++j) {
      const int st = j % KS, kv0 = (j0 + j) * kTcKeys;
      const bool edge = kv0 + kTcKeys - 1 > first_lim;
      bool ok = mbar_wait(raw_full(0), j & 1, ctl, KST_TIMEOUT_PRODUCER);
      if (ok) ok = mbar_wait(kv_empty(st), ((j / KS) & 1) ^ 1u, ctl, KST_TIMEOUT_PRODUCER);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (threadIdx.x < 8) {
        float lg, f;
        v_scale_terms(vs, lg, f);
        scales[st * 8 + threadIdx.x] = make_float4(ks, lg, f, 0.f);
      }
      convert(0, k_s(st), kv0, edge);
      mbar_arrive(k_full(st));
      if (j + 1 < n_max) fetch_scales(j + 1);
      // every converting thread is done with the raw tile: the next block's codes may take its place.  (After a wait that ran
      // out a warp leaves the loop; named barriers count threads, so the others must not wait for it: they meet in
      // mbarriers only.)
      mbar_arrive(raw_empty(0));
      if (threadIdx.x == 0 && j + 1 < n_max && mbar_wait(raw_empty(0), j & 1, ctl, KST_TIMEOUT_PRODUCER)) bring(0, j + 1);
      ok = mbar_wait(raw_full(1), j & 1, ctl, KST_TIMEOUT_PRODUCER);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      convert(1, v_s(st), kv0, edge);
      mbar_arrive(v_full(st));
      mbar_arrive(raw_empty(1));
      if (threadIdx.x == 0 && j + 1 < n_max && mbar_wait(raw_empty(1), j & 1, ctl, KST_TIMEOUT_PRODUCER)) bring(1, j + 1);
      __syncwarp();
    }
  } else if (warp == kTcMmaWarp) {
    // ------------------------------- MMA issuer -------------------------------
    constexpr uint32_t idesc_qk = make_idesc_f16(0, 0, 0, kTcRows, kTcKeys);
    constexpr uint32_t idesc_pv = make_idesc_f16(0, 0, 1, kTcRows, D);
    bool ok = true;
    auto wait = [&](uint32_t bar, uint32_t parity) {
      ok = mbar_wait(bar, parity, ctl, KST_TIMEOUT_MMA);
      ok = __all_sync(0xffffffffu, ok);
      return ok;
    };
    auto issue_qk = [&](int t, int j) {
      tc_fence_after();
      if (lane == 0) {
        const int st = j % KS;
        const uint64_t qd = make_smem_desc(q_s(t), 0, 1024), kd = make_smem_desc(k_s(st), 0, 1024);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint64_t off = static_cast<uint64_t>(((kk >> 2) * SM::kChunkBytes + (kk & 3) * 32) >> 4);
          umma_ss(tmem + t * kTcKeys, qd + off, kd + off, idesc_qk, kk != 0 ? 1u : 0u);
        }
        umma_commit(s_full(t));
      }
      __syncwarp();
    };
    if (n_max > 0 && wait(k_full(0), 0)) {
      for (int t = 0; t < 2 && ok; ++t)
        if (n_blocks[t] > 0 && wait(q_full(t), 0)) issue_qk(t, 0);
    }
    for (int j = 0; j < n_max && ok; ++j) {
      const int st = j % KS;
      bool next = false;
      for (int t = 0; t < 2 && ok; ++t) {
        if (j >= n_blocks[t]) continue;
        if (!wait(v_full(st), (j / KS) & 1)) break;
        const uint64_t vd = make_smem_desc(v_s(st), SM::kChunkBytes, 1024);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (!wait(p_ready(t, half), j & 1)) break;
          tc_fence_after();
          if (lane == 0) {
            // P'_t lies over S_t, per 32 columns [hi of 32 positions | lo of the same], 16 columns each; one MMA takes 16
            // positions = 8 columns
#pragma unroll
            for (int k4 = 0; k4 < kTcKeys / 32; ++k4) {
              const int kk = half * (kTcKeys / 32) + k4;
              const uint32_t a = tmem + t * kTcKeys + (kk >> 1) * 32 + (kk & 1) * 8;
              const uint32_t o = tmem + 2 * kTcKeys + t * 128;
              const uint64_t bd = vd + static_cast<uint64_t>((kk * 2048) >> 4);
              umma_ts(o, a, bd, idesc_pv, (j | kk) != 0 ? 1u : 0u);
              if constexpr (SPLIT) umma_ts(o, a + 16, bd, idesc_pv, 1u);
            }
            if (half == 1) umma_commit(pv_done(t));
          }
          __syncwarp();
        }
        if (!ok) break;
        if (j + 1 < n_blocks[t]) {
          if (!next && !wait(k_full((j + 1) % KS), ((j + 1) / KS) & 1)) break;
          next = true;
          issue_qk(t, j + 1);
        }
      }
      if (!ok) break;
      if (lane == 0) umma_commit(kv_empty(st));
      __syncwarp();
    }
  } else {
    // ------------------------------- softmax / epilogue -------------------------------
    const int t = (warp - 4) >> 2, quad = warp & 3;
    const int lrow = quad * 32 + lane;
    const int r = (2 * pair + t) * kTcRows + lrow;
    const bool there = r < p.R;
    const int nb = n_blocks[t];
    const int limit = there ? last_seen(p, n, r) : -1;
    const int limit_min = last_seen(p, n, min((2 * pair + t) * kTcRows, p.R - 1));
    const bool warp_active = (2 * pair + t) * kTcRows + quad * 32 < p.R;       // else it only keeps the barriers going
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t s_tmem = tmem + t * kTcKeys + lanes, o_tmem = tmem + 2 * kTcKeys + t * 128 + lanes;
    bool ok = true;
    float c_row = 0.f;
    // ---- q rows -> fp16 times 2^(14 - exponent of a row's largest element), swizzled.  D / 8 lanes take a row, so that a
    // warp reads whole lines (a row per thread: 8 us more for each CTA); lane L ends up with row L's factor.
    {                                          // whether or not a block follows: that takes the sequence's length to know
      constexpr int LPR = D / 8, RPI = 32 / LPR;                   // lanes per row, rows per iteration
      const int sub = lane / LPR, u = lane % LPR;
      constexpr int IT = 32 / RPI, AHEAD = 8;                      // rows of 8 iterations are under way together
#pragma unroll 1
      for (int it0 = 0; it0 < IT; it0 += AHEAD) {
        uint4 rows[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          const int rr = (2 * pair + t) * kTcRows + quad * 32 + (it0 + i) * RPI + sub;
          rows[i] = make_uint4(0u, 0u, 0u, 0u);
          if (rr < p.R)
            rows[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q.ptr) + b * p.q.stride_b + static_cast<long long>(rr / p.G) * p.q.stride_s +
                                                      static_cast<long long>(h * p.G + rr % p.G) * p.q.stride_h + u * 8);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          const int it = it0 + i, lr = quad * 32 + it * RPI + sub;
          const uint4 x = rows[i];
          // largest magnitude by its bits: 0x7f80 (bf16) / 0x7c00 (fp16) and up is not finite
          uint32_t top = __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
          top = max(top & 0xffffu, top >> 16);
#pragma unroll
          for (int o = LPR / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
          float up = 1.f, down = 1.f;
          if constexpr (Io<T>::kFmt == 1) {
            const int e = min(max(static_cast<int>(top >> 7) - 127, -100), 127);
            up = exp2_int(14 - e);
            down = exp2_int(e - 14);
          }
          // a row with an infinite or NaN element: every score is infinite or NaN, and so is its softmax NaN
          const float c = top >= (Io<T>::kFmt == 1 ? 0x7f80u : 0x7c00u) ? __uint_as_float(0x7fffffffu) : p.scale_log2 * down;
          const float mine = __shfl_sync(0xffffffffu, c, (lane % RPI) * LPR);
          if (lane / RPI == it) c_row = mine;
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
          uint32_t f[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 g = Io<T>::unpack2(w[e]);
            f[e] = Io<__half>::pack2(g.x * up, g.y * up);
          }
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};"
                       ::"r"(q_s(t) + (u >> 3) * SM::kChunkBytes + swz128(lr, u & 7)), "r"(f[0]), "r"(f[1]), "r"(f[2]), "r"(f[3])
                       : "memory");
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(q_full(t));
    }
    float m_run = -INFINITY, l_run = 0.f;
    uint32_t x[32];
    for (int j = 0; j < nb; ++j) {
      const int st = j % KS, kv0 = (j0 + j) * kTcKeys;
      ok = mbar_wait(k_full(st), (j / KS) & 1, ctl, KST_TIMEOUT_CONSUMER);       // the block's scales
      if (ok) ok = mbar_wait(s_full(t), j & 1, ctl, KST_TIMEOUT_CONSUMER);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      if (!warp_active) {
        mbar_arrive(p_ready(t, 0));
        mbar_arrive(p_ready(t, 1));
        continue;
      }
      const float4* sc = scales + st * 8;
      const bool masked = kv0 + kTcKeys - 1 > limit_min;
      // ---- pass 1: the block's maximum of t + log2 vs
      float mb = -INFINITY;
#pragma unroll
      for (int c = 0; c < kTcKeys / 32; ++c) {
        tmem_ld32(s_tmem + c * 32, x);
        tmem_wait_ld();
#pragma unroll
        for (int g0 = 0; g0 < 32; g0 += GRP) {
          float m0 = -INFINITY;
          if (masked) {
#pragma unroll
            for (int i = 0; i < GRP; ++i)
              if (kv0 + c * 32 + g0 + i <= limit) m0 = fmaxf(m0, __uint_as_float(x[g0 + i]));
          } else {
            float m1 = fmaxf(__uint_as_float(x[g0]), __uint_as_float(x[g0 + 1]));
            m0 = fmaxf(__uint_as_float(x[g0 + 2]), __uint_as_float(x[g0 + 3]));
#pragma unroll
            for (int i = 4; i < GRP; i += 4) {
              m0 = fmax3(m0, __uint_as_float(x[g0 + i]), __uint_as_float(x[g0 + i + 1]));
              m1 = fmax3(m1, __uint_as_float(x[g0 + i + 2]), __uint_as_float(x[g0 + i + 3]));
            }
            m0 = fmaxf(m0, m1);
          }
          const float4 f = sc[c * 2 + g0 / 16];
          if (!masked || m0 != -INFINITY) mb = fmaxf(mb, fmaf(m0, c_row * f.x, f.y));
        }
      }
      const float m_new = mb - kTcPBias;
      const bool grow = m_new - m_run > kTcRescale;                // first block: m_run = -inf
      float alpha = 1.0f;
      if (grow) {
        alpha = ex2_approx(m_run - m_new);                         // 0 on the first block
        l_run = sum_moved(l_run, m_run - m_new);
        m_run = m_new;
      }
      // S_t(j) was produced after P'_t(j-1) v (MMAs run in issue order), so O_t is quiescent here
      if (j > 0 && __any_sync(0xffffffffu, grow)) {
#pragma unroll 1
        for (int c = 0; c < D / 16; ++c) {
          uint32_t y[16];
          tmem_ld16(o_tmem + c * 16, y);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * alpha);
          tmem_st16(o_tmem + c * 16, y);
        }
      }
      // ---- pass 2: P' = 2^(t - m') vs, written over S (hi | lo per 32 columns); compiled twice, without and with masks
      auto pass2 = [&](auto masked_tag) {
        constexpr bool kMasked = decltype(masked_tag)::value;
        auto chunk_p = [&](const uint32_t (&src)[32], int c, uint32_t (&pk)[SPLIT ? 32 : 16]) {
          float2 sum;
          float4 f;
#pragma unroll
          for (int i0 = 0; i0 < 16; i0 += 8) {                     // pairs of columns, eight at a time
            if (GRP == 16 || i0 == 0) f = sc[c * 2 + i0 / 8];
            const float a = c_row * f.x, d = kQ8LBias - m_run;
            const float2 a2 = make_float2(a, a), d2 = make_float2(d, d), f2 = make_float2(f.z, f.z);
            float2 pp[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
              pp[i] = __ffma2_rn(make_float2(__uint_as_float(src[2 * (i0 + i)]), __uint_as_float(src[2 * (i0 + i) + 1])), a2, d2);
#pragma unroll
            for (int i = 0; i < 8; ++i) pp[i] = make_float2(ex2_approx(pp[i].x), ex2_approx(pp[i].y));
            if constexpr (kMasked) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int key = kv0 + c * 32 + 2 * (i0 + i);
                if (key > limit) pp[i].x = 0.f;
                if (key + 1 > limit) pp[i].y = 0.f;
              }
            }
            sum = GRP == 16 || i0 == 0 ? pp[0] : __fadd2_rn(sum, pp[0]);
#pragma unroll
            for (int i = 1; i < 8; ++i) sum = __fadd2_rn(sum, pp[i]);
            if (GRP == 16 || i0 == 8) l_run += sum.x + sum.y;
#pragma unroll
            for (int i = 0; i < 8; ++i) pp[i] = __fmul2_rn(pp[i], f2);
#pragma unroll
            for (int i = 0; i < 8; ++i) pk[i0 + i] = Io<__half>::pack2(pp[i].x, pp[i].y);
            if constexpr (SPLIT) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float2 lo = __ffma2_rn(Io<__half>::unpack2(pk[i0 + i]), make_float2(-1.f, -1.f), pp[i]);
                pk[16 + i0 + i] = Io<__half>::pack2(lo.x, lo.y);
              }
            }
          }
        };
        auto store_p = [&](int c, uint32_t (&pk)[SPLIT ? 32 : 16]) {
          if constexpr (SPLIT) tmem_st32(s_tmem + c * 32, *reinterpret_cast<uint32_t(*)[32]>(pk));
          else tmem_st16(s_tmem + c * 32, *reinterpret_cast<uint32_t(*)[16]>(pk));
        };
        // two register buffers: the next columns are on their way while these are worked on
        uint32_t y[32];
        tmem_ld32(s_tmem, x);
        tmem_wait_ld();
#pragma unroll 1
        for (int c = 0; c < kTcKeys / 32; c += 2) {
          uint32_t pk[SPLIT ? 32 : 16];
          tmem_ld32(s_tmem + (c + 1) * 32, y);
          chunk_p(x, c, pk);
          store_p(c, pk);
          tmem_wait_ld();
          if (c + 2 < kTcKeys / 32) tmem_ld32(s_tmem + (c + 2) * 32, x);
          chunk_p(y, c + 1, pk);
          store_p(c + 1, pk);
          if (c == 0) {                                            // the first half of P' is written
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(p_ready(t, 0));
          }
          tmem_wait_ld();
        }
      };
      if (masked) pass2(std::true_type{});
      else pass2(std::false_type{});
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(p_ready(t, 1));
    }
    // ---- epilogue.  A row without a block (or without a visible position) has l = 0: o = 0, lse = -inf
    if (ok && nb > 0 && warp_active) {
      ok = mbar_wait(pv_done(t), (nb - 1) & 1, ctl, KST_TIMEOUT_CONSUMER);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
    }
    if (ok && !dead && warp_active) {
      const int tile = 2 * pair + t;
      // Dealt out: a piece begins a new pair, a new CTA or both, so pair + CTA numbers the pieces.  Tile 1's behind tile 0's.
      const int all_pairs = p.B * p.Hkv * tp.pairs;
      const long long slot = tp.ctas > 0 ? static_cast<long long>(t) * (all_pairs + tp.ctas) + bh * tp.pairs + pair + cta
                                         : static_cast<long long>(t) * (all_pairs - tp.whole) * tp.cut + cta - tp.whole;
      const bool parts = pieces > 1, any_nan = *reinterpret_cast<volatile int*>(nan_any) != 0;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        if (nb > 0) {
          tmem_ld32(o_tmem + c * 32, x);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = 0u;
        }
        if (any_nan) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (nan_from[c * 32 + i] <= limit) x[i] = 0x7fffffffu;
        }
        if (parts) {
          if (!there) continue;
          float* dst = p.part_o + (slot * kTcRows + lrow) * D + c * 32;
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(dst + i) = make_float4(__uint_as_float(x[i]), __uint_as_float(x[i + 1]),
                                                              __uint_as_float(x[i + 2]), __uint_as_float(x[i + 3]));
        } else {
          // rows meet in the q tile's place (its products are done), so that the warp can write whole lines
          const float inv = l_run == 0.f ? 0.f : 262144.f / l_run;         // 2^kQ8LBias
#pragma unroll
          for (int i = 0; i < 32; i += 8)
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};"
                         ::"r"(q_s(t) + (c >> 1) * SM::kChunkBytes + swz128(lrow, (c & 1) * 4 + (i >> 3))),
                           "r"(Io<T>::pack2(__uint_as_float(x[i]) * inv, __uint_as_float(x[i + 1]) * inv)),
                           "r"(Io<T>::pack2(__uint_as_float(x[i + 2]) * inv, __uint_as_float(x[i + 3]) * inv)),
                           "r"(Io<T>::pack2(__uint_as_float(x[i + 4]) * inv, __uint_as_float(x[i + 5]) * inv)),
                           "r"(Io<T>::pack2(__uint_as_float(x[i + 6]) * inv, __uint_as_float(x[i + 7]) * inv))
                         : "memory");
        }
      }
      if (!parts) {
        __syncwarp();
        constexpr int LPR = D / 8, RPI = 32 / LPR;
        const int sub = lane / LPR, u = lane % LPR;
#pragma unroll 4
        for (int it = 0; it < 32 / RPI; ++it) {
          const int lr = quad * 32 + it * RPI + sub, rr = (2 * pair + t) * kTcRows + lr;
          const uint4 v = lds128(q_s(t) + (u >> 3) * SM::kChunkBytes + swz128(lr, u & 7));
          if (rr < p.R)
            *reinterpret_cast<uint4*>(static_cast<T*>(p.o.ptr) + b * p.o.stride_b + static_cast<long long>(rr / p.G) * p.o.stride_s +
                                      static_cast<long long>(h * p.G + rr % p.G) * p.o.stride_h + u * 8) = v;
        }
      }
      if (there) {
        if (parts) p.part_ml[slot * kTcRows + lrow] = make_float2(m_run + kQ8PBias, l_run);    // in the merge's convention
        else if (p.lse != nullptr)
          p.lse[(static_cast<long long>(b) * p.Hq + h * p.G + r % p.G) * p.M + r / p.G] = m_run - kQ8LBias + log2f(l_run);
      }
      if (p.pieces != nullptr && (tp.ctas > 0 || parts) && split == 0 && lrow == 0) {      // where the merge finds them: slot = unit + entry
        const int u = bh * p.tiles + tile, first = static_cast<int>(slot) - u;
        p.pieces[u] = make_int2(first, first + pieces - 1);
      }
      tc_fence_before();
    }
  }

  // ------------------------------- teardown -------------------------------
  __syncthreads();
  if (*abort_flag) {                           // a wait ran out: time for the products under way to end
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == kTcMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTcTmemCols);
  }
}

struct TcPlan {
  int tiles, pairs, ctas, whole, cut;
  size_t ml_off, o_off, piece_off, total;
};

// key blocks divided among one CTA for each SM where that is at least two CTAs a pair
TcPlan tc_plan(const TrnAttnQ8Args& a) {
  TcPlan w{};
  const int R = a.M * (a.Hq / a.Hkv);
  w.tiles = (R + kTcRows - 1) / kTcRows;
  w.pairs = (w.tiles + 1) / 2;
  const long long pairs = static_cast<long long>(a.B) * a.Hkv * w.pairs;
  const int longest = a.kv_len != nullptr ? a.cache.S : min(max(a.kv_len_all, 1), a.cache.S);
  const int blocks = (longest - 1) / kTcKeys + 1;
  size_t rows;
  if (2 * pairs <= kAttnNominalSMs && blocks >= kTcMinDivide) {
    w.ctas = static_cast<int>(min(static_cast<long long>(kAttnNominalSMs), pairs * blocks));
    rows = 2 * static_cast<size_t>(pairs + w.ctas) * kTcRows;
  } else {
    // Whole rounds of CTAs, and a last one that would leave most SMs idle: its pairs are cut into pieces that fill it (512
    // pairs: 3 rounds and 68 pairs in two pieces each, instead of 4 rounds).  256 queries a pair, 6144 positions, whole / pieces: 1 round
    // and 20 pairs 246 / 167 us, 8 and 20 1088 / 1029, 12 and 8 1566 / 1499, 12 and 72 1577 / 1578 (causal 1602 / 1614)
    w.whole = static_cast<int>(min(pairs, 0x7fffffffLL));
    w.cut = 1;
    const long long rest = pairs % kAttnNominalSMs, rounds = pairs / kAttnNominalSMs;
    if (rest == 0 || rounds == 0 || blocks < kTcMinCutBlocks) return w;
    const int cut = static_cast<int>(min(kAttnNominalSMs / rest, static_cast<long long>(kTcMaxCut)));
    if (cut < 2) return w;
    w.cut = cut;
    w.whole = static_cast<int>(pairs - rest);
    rows = 2 * static_cast<size_t>(rest * cut) * kTcRows;
  }
  w.ml_off = 0;
  w.o_off = up256(rows * sizeof(float2));
  w.piece_off = w.o_off + up256(rows * a.D * sizeof(float));
  w.total = w.piece_off + up256(static_cast<size_t>(a.B) * a.Hkv * w.tiles * sizeof(int2));
  return w;
}

template <typename T, int D, int GRP, bool SPLIT>
int launch_grp(const TrnAttnQ8Args& a, cudaStream_t st, const DeviceState& ds) {
  using SM = TcSmem<D>;
  TcPlan w = tc_plan(a);
  const long long pairs = static_cast<long long>(a.B) * a.Hkv * w.pairs;
  if (pairs > 0x7fffffffLL || static_cast<long long>(a.B) * a.Hkv * w.tiles > 0x7fffffffLL) return TRN_E_SHAPE;
  if (a.workspace == nullptr) {                          // nothing is divided
    w.ctas = 0;
    w.cut = 1;
    w.whole = static_cast<int>(pairs);
  }
  TcParams tp{};
  tp.c = q8_params(a, ds);
  tp.pairs = w.pairs;
  tp.ctas = w.ctas;
  tp.whole = w.whole;
  tp.cut = w.cut;
  tp.c.tiles = w.tiles;
  tp.c.tile_rows = kTcRows;
  const bool parts = w.ctas > 0 || w.cut > 1;
  if (parts) {
    uint8_t* ws = static_cast<uint8_t*>(a.workspace);
    tp.c.part_ml = reinterpret_cast<float2*>(ws + w.ml_off);
    tp.c.part_o = reinterpret_cast<float*>(ws + w.o_off);
    tp.c.pieces = reinterpret_cast<int2*>(ws + w.piece_off);
  }
  const long long grid = w.ctas > 0 ? w.ctas : w.whole + (pairs - w.whole) * w.cut;
  if (w.ctas == 0 && parts) {                            // the merge visits the pairs in pieces alone
    tp.c.join_pairs = w.pairs;
    tp.c.join_first = w.whole;
  }
  CUtensorMap tm_k, tm_v;
  int rc = make_code_tmap(&tm_k, &tp.c.ki, a.cache.k, a.cache.S, a.Hkv, a.B, D, kTcKeys);
  if (rc == TRN_OK) rc = make_code_tmap(&tm_v, &tp.c.vi, a.cache.v, a.cache.S, a.Hkv, a.B, D, kTcKeys);
  if (rc != TRN_OK) return rc;
  auto kern = attn_q8_tc_kernel<T, D, GRP, SPLIT>;
  rc = ensure_dyn_smem(reinterpret_cast<const void*>(kern), SM::kTotal, ds.device);
  if (rc != TRN_OK) return rc;
  TRN_CUDA_TRY(launch_pdl(kern, dim3(static_cast<unsigned>(grid)), dim3(kTcThreads), SM::kTotal, st, tm_k, tm_v, tp));
  return parts ? launch_q8_join(tp.c, a, true, st) : TRN_OK;
}

template <typename T, int D>
int launch_typed(const TrnAttnQ8Args& a, cudaStream_t st, const DeviceState& ds) {
  if (a.single_p != 0) return a.cache.block == 16 ? launch_grp<T, D, 16, false>(a, st, ds) : launch_grp<T, D, 32, false>(a, st, ds);
  return a.cache.block == 16 ? launch_grp<T, D, 16, true>(a, st, ds) : launch_grp<T, D, 32, true>(a, st, ds);
}

}  // namespace

// More than 32 rows per kv head (bf16, us here and in attn_q8.cu: 24 rows of 8 x 8 heads, 4096 positions 65.0, 50.9; 32 rows 65.8, 51.7; 36
// rows 65.5, 66.2; 36 rows of 16 x 8 heads, 2048 positions 52.9, 74.6; 60 rows of 32 x 1 head, 4674 positions 48.1, 56.3; 71 rows of
// 32 x 1 head of 64, 4096 positions 32.9, 42.9.  Few units of few positions would still be faster there: 36 rows of 8 heads, 1000
// positions 18.6, 11.9; 71 rows of one head, 4096 positions 19.5, 15.1), and
// no weights (those are summed from scores that attn_q8.cu keeps; kept here, by threads with a row each, p in one part: 36 rows of
// 8 x 8 heads, 4096 positions 95.8 us, there 78.1; 568 rows of one head of 64, 8192 positions 67.6, 55.8)
bool attn_q8_tc_applies(const TrnAttnQ8Args& a) {
  return a.weight == nullptr && static_cast<long long>(a.M) * (a.Hq / a.Hkv) > 32;
}

size_t attn_q8_tc_workspace(const TrnAttnQ8Args& a) { return tc_plan(a).total; }

int launch_attn_q8_tc(const TrnAttnQ8Args& a, cudaStream_t st, const DeviceState& ds) {
  if (a.dtype == TRN_BF16)
    return a.D == 128 ? launch_typed<__nv_bfloat16, 128>(a, st, ds) : launch_typed<__nv_bfloat16, 64>(a, st, ds);
  return a.D == 128 ? launch_typed<__half, 128>(a, st, ds) : launch_typed<__half, 64>(a, st, ds);
}

}  // namespace trn
