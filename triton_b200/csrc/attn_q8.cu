// Attention over the 8-bit key/value cache: o = softmax(scale * q k^T) v with k = kc * ks, v = vc * vs (e4m3 codes, one
// fp32 scale per `block` positions and kv head), sequences of their own lengths, causal or not, any Hq / Hkv.
//
// Mathematics.  e4m3 codes are fp16 values exactly (one conversion instruction for two of them), so both products run in
// fp16 with fp32 accumulation and no scale ever enters them:
//   * q enters as fp16 times a power of two per row (2^(14 - e), e the exponent of the row's largest element): exact for
//     fp16 q, and for bf16 q but for elements 2^-28 below the row's largest, whose error is at most 2^-39 of that one;
//   * ks multiplies the score:  t = acc * (scale * log2 e * row factor * ks);
//   * vs is folded into the exponent:  t' = t + log2 vs,  running maximum m' of t',  P' = 2^(t' - m') <= 1,
//     O = sum P' vc,  l = sum P' / vs,  o = O / l,  lse = m' + log2 l  (P' / vs = 2^(t - m')).
//     P' is what its key adds to O whatever its block's scale, so its rounding to 16 bits is relative to the output.
// P' carries a factor 2^12 into the product (it cancels in O / l), which keeps weights down to 2^-26 of the row's largest out of
// fp16's subnormals.  bf16 outputs take P' as one fp16 (error 2^-12 against the output's 2^-9); fp16 outputs take it as
// hi + lo, since one part alone would err as much as the output's own rounding.
//
// This kernel is for few query rows per kv head: a CTA of four warps owns 16 of the M * Hq / Hkv rows of a (b, kv head) and
// 1 / n_splits of its positions; each warp walks its quarter in chunks of 32 positions through its own ring of TMA
// tiles.  It is bound by memory (2 * D bytes per position and kv head): the ring keeps 3 x 8 KB per warp in flight, and
// codes go from shared memory to registers as the 16 bytes a lane needs (the order of the d axis inside a product and of the
// columns inside the output is free, so the m16n8k16 fragments are picked such that 128-bit reads have no bank conflicts
// under the TMA swizzle: K lane (g, t) reads 16-byte units 2t and 2t + 1 of key g, V lane (g, t) unit g of keys 2t, 2t + 1).
// Partial results of the splits are merged by a second small kernel, which also sums the per-position weights from the
// scores kept in the workspace.  Rows, splits and sums are taken in a fixed order: bitwise reproducible.
//
// What must not be seen cannot hurt: scores behind a row's last position are replaced, not weighted, and in the
// chunks where that happens NaN codes of v are taken as 0 in the product (0 * NaN would poison rows that do not see them) and
// put back as NaN into the outputs of the rows that do.
#include <math.h>

#include "attn_common.cuh"
#include "q8.cuh"
#include "small_mma.cuh"

namespace trn {
namespace {

constexpr int kQ8Warps = 4;
constexpr int kQ8Threads = 32 * kQ8Warps;
constexpr int kQ8Keys = 32;                    // positions per chunk
constexpr int kQ8Stages = 3;
constexpr int kQ8Rows = 16;
constexpr float kQ8PBias = 12.f;               // log2 of the factor P' carries into the product
constexpr float kMinVScale = 7.888609052210118e-31f;   // 2^-100: smaller scales (a block of zeros) count as this
constexpr int kQ8TargetCtas = 2;               // resident CTAs per SM (registers and shared memory)

template <int D>
struct Q8Smem {
  static constexpr int kTile = kQ8Keys * D;                        // bytes of k or v of a chunk
  static constexpr int kWarpRing = kQ8Stages * 2 * kTile;
  static constexpr int kRing = kQ8Warps * kWarpRing;
  static constexpr int kRow = D + 4;                               // o | max, sum  of a warp's partial result
  static constexpr int kPart = kQ8Warps * kQ8Rows * kRow * 4;      // overlays the ring after the key loop
  static constexpr int kBody = kRing > kPart ? kRing : kPart;
  static constexpr int kBars = kBody;
  static constexpr int kTotal = kBars + 128 + 1024;                // + slack to align the base to 1024 bytes
};

struct Q8Params {
  TrnHeadTensor q, o;
  HeadMapInfo ki, vi;
  ScaleTable ks, vs;
  KvLen len;
  float* lse;
  int B, M, Hq, Hkv, G, R;                     // R = M * G rows per (b, kv head): row r = query r / G, head r % G
  int tiles;                                   // 16-row tiles per (b, kv head)
  int causal;
  float scale_log2;
  int shift;                                   // log2(block)
  int n_splits;
  float* part_o;                               // [n_splits][units][16][D], units = B * Hkv * tiles
  float2* part_ml;                             // [n_splits][units][16]
  float* scores;                               // [B * Hkv][R][pitch], log2 domain, or NULL
  long long pitch;
  float* weight;
  long long w_sb, w_sh;
  int weight_add;
  int* status;
};

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
// 0xff in every byte of w that holds a NaN code (0x7f or 0xff)
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  return ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu;
}
// byte offset of 16-byte unit u of row r in a tile as TMA wrote it: 128-byte rows with the 128-byte swizzle, 64-byte rows
// with the 64-byte swizzle
template <int D>
__device__ __forceinline__ uint32_t q8_off(uint32_t r, uint32_t u) {
  if constexpr (D == 128) return r * 128u + ((u ^ (r & 7u)) << 4);
  else return r * 64u + ((u ^ ((r >> 1) & 3u)) << 4);
}
// which row of an 8-row block column c of a score block is.  64-byte rows: a quad's even columns 0, 2, 4, 6 and the lane
// groups' neighbours have to meet different halves of a 128-byte line, hence 0 3 1 2 4 7 5 6
template <int D>
__device__ __forceinline__ int q8_key(int c) {
  if constexpr (D == 128) return c;
  else return (c & 4) + ((0x2130 >> ((c & 3) * 4)) & 3) ;
}

// HILO: P' enters the product as two fp16 parts.
template <typename T, int D, bool HILO>
__global__ void __launch_bounds__(kQ8Threads)
attn_q8_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
               const __grid_constant__ Q8Params p) {
  using SM = Q8Smem<D>;
  constexpr int KS = D / 16;                   // k steps of q k^T
  constexpr int NB = D / 8;                    // 8-column blocks of o
  constexpr int KU = D / 64;                   // 16-byte units a lane reads per key row
  extern __shared__ uint8_t q8_smem_raw[];
  __shared__ int nan_from[D];                  // first position whose v code of this column is NaN, in edge chunks
  __shared__ int s_abort;
  const uint32_t base = (smem_u32(q8_smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = q8_smem_raw + (base - smem_u32(q8_smem_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t bars = base + SM::kBars + warp * kQ8Stages * 8;
  Ctl ctl{p.status, &s_abort};
  if (lane == 0) {
    for (int s = 0; s < kQ8Stages; ++s) mbar_init(bars + 8 * s, 1);
    fence_mbar_init();
  }
  if (threadIdx.x == 0) s_abort = 0;
  for (int i = threadIdx.x; i < D; i += kQ8Threads) nan_from[i] = 0x7fffffff;
  __syncthreads();
  griddep_wait();                              // q, the codes and the lengths may come from the launch before
  griddep_launch();
  if (*reinterpret_cast<volatile int*>(p.status) != 0) return;

  const int split = static_cast<int>(blockIdx.x) % p.n_splits;
  const int unit = static_cast<int>(blockIdx.x) / p.n_splits;
  const int tile = unit % p.tiles, bh = unit / p.tiles;
  const int b = bh / p.Hkv, h = bh % p.Hkv;
  const int n = p.len(b);
  const int r0 = tile * kQ8Rows, rows = min(kQ8Rows, p.R - r0);
  // rows g and g + 8: their last visible position (-1: none)
  auto last_of = [&](int r) { return r >= rows ? -1 : p.causal ? max(n - p.M + (r0 + r) / p.G, -1) : n - 1; };
  const int lim_lo = last_of(g), lim_hi = last_of(g + 8);
  const int lim_min = last_of(0), lim_max = last_of(rows - 1);

  // ---- q fragments as fp16 times 2^(14 - exponent of the row's largest element); k step ks = 4 h + j of lane t holds
  // d = (KU t + h) 16 + 4 j + {0, 1} in registers 0 / 1 and + {2, 3} in 2 / 3
  uint32_t qa[KS][4];
  float c_lo = 0.f, c_hi = 0.f;                // scale * log2 e / row factor
  {
    auto row_ptr = [&](int r) {
      const int rr = r0 + min(r, rows - 1);
      return static_cast<const T*>(p.q.ptr) + b * p.q.stride_b + static_cast<long long>(rr / p.G) * p.q.stride_s +
             static_cast<long long>(h * p.G + rr % p.G) * p.q.stride_h + t * KU * 16;
    };
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const T* src = row_ptr(g + 8 * half);
      uint4 x[2 * KU];
#pragma unroll
      for (int i = 0; i < 2 * KU; ++i) x[i] = *reinterpret_cast<const uint4*>(src + i * 8);
      float f[KU * 16], amax = 0.f;
      bool bad = false;
#pragma unroll
      for (int i = 0; i < 2 * KU; ++i) {
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 v = Io<T>::unpack2(w[e]);
          f[i * 8 + 2 * e] = v.x;
          f[i * 8 + 2 * e + 1] = v.y;
          bad = bad || !(fabsf(v.x) <= FLT_MAX) || !(fabsf(v.y) <= FLT_MAX);
          amax = fmaxf(amax, fmaxf(fabsf(v.x), fabsf(v.y)));
        }
      }
      float up = 1.f, down = 1.f;
      if constexpr (Io<T>::kFmt == 1) {
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const int e = max(static_cast<int>(__float_as_uint(amax) >> 23) - 127, -100);
        up = exp2_int(14 - min(e, 127));
        down = exp2_int(min(e, 127) - 14);
      }
      bad = (__ballot_sync(0xffffffffu, bad) >> (g * 4)) & 0xfu;
      // a row with an infinite or NaN element: every score is infinite or NaN, and so is its softmax NaN
      const float c = bad ? __uint_as_float(0x7fffffffu) : p.scale_log2 * down;
      if (half == 0) c_lo = c; else c_hi = c;
      const bool there = g + 8 * half < rows;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const int d = (i >> 2) * 16 + (i & 3) * 4;
        const __half2 a = __floats2half2_rn(f[d] * up, f[d + 1] * up), c2 = __floats2half2_rn(f[d + 2] * up, f[d + 3] * up);
        qa[i][half] = there ? *reinterpret_cast<const uint32_t*>(&a) : 0u;
        qa[i][2 + half] = there ? *reinterpret_cast<const uint32_t*>(&c2) : 0u;
      }
    }
  }

  // ---- this warp's chunks: dealt out evenly to the warps of all splits
  const int total = (lim_max + kQ8Keys) / kQ8Keys;                 // lim_max = -1: none
  const int n_warps = kQ8Warps * p.n_splits, wi = split * kQ8Warps + warp;
  const int chunk0 = static_cast<int>(static_cast<long long>(total) * wi / n_warps);
  const int n_chunks = static_cast<int>(static_cast<long long>(total) * (wi + 1) / n_warps) - chunk0;
  const uint32_t ring = base + warp * SM::kWarpRing;
  auto k_tile = [&](int s) { return ring + s * 2 * SM::kTile; };
  auto load = [&](int c) {                                         // lane 0
    const int s = c % kQ8Stages, key0 = (chunk0 + c) * kQ8Keys;
    mbar_expect_tx(bars + 8 * s, 2 * SM::kTile);
    tma_load_head_tile(k_tile(s), &tm_k, bars + 8 * s, p.ki, 0, key0, h, b);
    tma_load_head_tile(k_tile(s) + SM::kTile, &tm_v, bars + 8 * s, p.vi, 0, key0, h, b);
  };
  if (lane == 0)
    for (int c = 0; c < min(kQ8Stages, n_chunks); ++c) load(c);
  // scales of a chunk: two halves of 16 positions (the same block unless block is 16)
  auto scales_of = [&](int c, float (&ks)[2], float (&vs)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int key = (chunk0 + c) * kQ8Keys + 16 * i;
      const bool in = c < n_chunks && key <= lim_max;
      ks[i] = in ? *p.ks.at(b, key >> p.shift, h) : 1.f;
      const float v = in ? *p.vs.at(b, key >> p.shift, h) : 1.f;
      vs[i] = v < kMinVScale ? kMinVScale : v;
    }
  };

  float oacc[NB][4];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) oacc[i][j] = 0.f;
  float m_lo = -INFINITY, m_hi = -INFINITY, l_lo = 0.f, l_hi = 0.f;
  float* sc_lo = nullptr;
  float* sc_hi = nullptr;
  if (p.scores != nullptr) {
    if (g < rows) sc_lo = p.scores + (static_cast<long long>(bh) * p.R + r0 + g) * p.pitch;
    if (g + 8 < rows) sc_hi = p.scores + (static_cast<long long>(bh) * p.R + r0 + g + 8) * p.pitch;
  }
  float ks_next[2], vs_next[2];
  scales_of(0, ks_next, vs_next);
  bool ok = true;

  for (int c = 0; c < n_chunks; ++c) {
    const int s = c % kQ8Stages, key0 = (chunk0 + c) * kQ8Keys;
    const float ks[2] = {ks_next[0], ks_next[1]}, vs[2] = {vs_next[0], vs_next[1]};
    scales_of(c + 1, ks_next, vs_next);
    const bool edge = key0 + kQ8Keys - 1 > lim_min;                // some row does not see some position of the chunk
    ok = mbar_wait(bars + 8 * s, (c / kQ8Stages) & 1, ctl, KST_TIMEOUT_CONSUMER);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) break;
    // ---- scores of four 8-position blocks
    float sacc[4][4];
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) {
#pragma unroll
      for (int j = 0; j < 4; ++j) sacc[nb][j] = 0.f;
      const uint32_t row = nb * 8 + q8_key<D>(g);
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        const uint4 w = lds128(k_tile(s) + q8_off<D>(row, KU * t + u));
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          mma16816<__half>(sacc[nb], qa[4 * u + j], e4m3x2_to_f16x2(ww[j]), e4m3x2_to_f16x2(ww[j] >> 16));
      }
    }
    // ---- t = acc * c * ks, t' = t + log2 vs
    float lv[2], inv[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) { lv[i] = log2f(vs[i]); inv[i] = 1.0f / vs[i]; }
    float mb_lo = -INFINITY, mb_hi = -INFINITY;
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) {
      const float a_lo = c_lo * ks[nb >> 1], a_hi = c_hi * ks[nb >> 1], l = lv[nb >> 1];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = sacc[nb][e] * a_lo, y = sacc[nb][2 + e] * a_hi;
        const int key = key0 + nb * 8 + q8_key<D>(2 * t + e);
        // whoever reads the kept scores knows which of them a row sees
        if (sc_lo != nullptr) sc_lo[key] = x;
        if (sc_hi != nullptr) sc_hi[key] = y;
        x += l;
        y += l;
        if (edge) {
          if (key > lim_lo) x = -INFINITY;
          if (key > lim_hi) y = -INFINITY;
        }
        sacc[nb][e] = x;
        sacc[nb][2 + e] = y;
        mb_lo = fmaxf(mb_lo, x);
        mb_hi = fmaxf(mb_hi, y);
      }
    }
    mb_lo = fmaxf(mb_lo, __shfl_xor_sync(0xffffffffu, mb_lo, 1)); mb_lo = fmaxf(mb_lo, __shfl_xor_sync(0xffffffffu, mb_lo, 2));
    mb_hi = fmaxf(mb_hi, __shfl_xor_sync(0xffffffffu, mb_hi, 1)); mb_hi = fmaxf(mb_hi, __shfl_xor_sync(0xffffffffu, mb_hi, 2));
    const float mn_lo = fmaxf(m_lo, mb_lo), mn_hi = fmaxf(m_hi, mb_hi);
    if (__any_sync(0xffffffffu, mn_lo > m_lo || mn_hi > m_hi)) {
      const float al_lo = mn_lo == -INFINITY ? 1.f : ex2_approx(m_lo - mn_lo);
      const float al_hi = mn_hi == -INFINITY ? 1.f : ex2_approx(m_hi - mn_hi);
      m_lo = mn_lo; m_hi = mn_hi;
      l_lo *= al_lo; l_hi *= al_hi;
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        oacc[i][0] *= al_lo; oacc[i][1] *= al_lo;
        oacc[i][2] *= al_hi; oacc[i][3] *= al_hi;
      }
    }
    const float use_lo = (m_lo == -INFINITY ? 0.f : m_lo) - kQ8PBias, use_hi = (m_hi == -INFINITY ? 0.f : m_hi) - kQ8PBias;
    uint32_t ph[4][2], pl[4][2];
    float sum_lo = 0.f, sum_hi = 0.f;
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) {
      const float a0 = ex2_approx(sacc[nb][0] - use_lo), a1 = ex2_approx(sacc[nb][1] - use_lo);
      const float b0 = ex2_approx(sacc[nb][2] - use_hi), b1 = ex2_approx(sacc[nb][3] - use_hi);
      sum_lo = fmaf(a0 + a1, inv[nb >> 1], sum_lo);
      sum_hi = fmaf(b0 + b1, inv[nb >> 1], sum_hi);
      ph[nb][0] = Io<__half>::pack2(a0, a1);
      ph[nb][1] = Io<__half>::pack2(b0, b1);
      if constexpr (HILO) {
        const float2 ra = Io<__half>::unpack2(ph[nb][0]), rb = Io<__half>::unpack2(ph[nb][1]);
        pl[nb][0] = Io<__half>::pack2(a0 - ra.x, a1 - ra.y);
        pl[nb][1] = Io<__half>::pack2(b0 - rb.x, b1 - rb.y);
      }
    }
    l_lo += sum_lo;
    l_hi += sum_hi;
    // ---- o += P' v: two steps of 16 positions.  Column block j of lane g's output holds d = g * (D / 8) + j.
    const uint32_t vt = k_tile(s) + SM::kTile;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const uint32_t ah[4] = {ph[2 * kk][0], ph[2 * kk][1], ph[2 * kk + 1][0], ph[2 * kk + 1][1]};
      uint32_t al[4] = {0u, 0u, 0u, 0u};
      if constexpr (HILO) {
        al[0] = pl[2 * kk][0]; al[1] = pl[2 * kk][1]; al[2] = pl[2 * kk + 1][0]; al[3] = pl[2 * kk + 1][1];
      }
      constexpr int W = D / 32;                // 32-bit words a lane takes of a row: 4 or 2
      uint32_t v[4][W];                        // rows: positions 2t, 2t + 1 of the step's two blocks
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int rr = (2 * kk + (i >> 1)) * 8 + q8_key<D>(2 * t + (i & 1));
        if constexpr (D == 128) {
          const uint4 w = lds128(vt + q8_off<D>(rr, g));
          v[i][0] = w.x; v[i][1] = w.y; v[i][2] = w.z; v[i][3] = w.w;
        } else {
          const uint2 w = lds64(vt + q8_off<D>(rr, g >> 1) + (g & 1) * 8);
          v[i][0] = w.x; v[i][1] = w.y;
        }
        if (edge) {
          const int key = key0 + rr;
#pragma unroll
          for (int w = 0; w < W; ++w) {
            const uint32_t bad = nan_bytes(v[i][w]);
            if (bad != 0u) {
              v[i][w] &= ~bad;
              if (key <= lim_max)
                for (int e = 0; e < 4; ++e)
                  if ((bad >> (8 * e)) & 1u) atomicMin(&nan_from[g * (D / 8) + 4 * w + e], key);
            }
          }
        }
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
        // bytes of two positions side by side: (k, k + 1) pairs of column 4 w + e
        const uint32_t x0 = __byte_perm(v[0][w], v[1][w], 0x5140), x1 = __byte_perm(v[0][w], v[1][w], 0x7362);
        const uint32_t y0 = __byte_perm(v[2][w], v[3][w], 0x5140), y1 = __byte_perm(v[2][w], v[3][w], 0x7362);
        const uint32_t b0[4] = {e4m3x2_to_f16x2(x0), e4m3x2_to_f16x2(x0 >> 16), e4m3x2_to_f16x2(x1), e4m3x2_to_f16x2(x1 >> 16)};
        const uint32_t b1[4] = {e4m3x2_to_f16x2(y0), e4m3x2_to_f16x2(y0 >> 16), e4m3x2_to_f16x2(y1), e4m3x2_to_f16x2(y1 >> 16)};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          mma16816<__half>(oacc[4 * w + e], ah, b0[e], b1[e]);
          if constexpr (HILO) mma16816<__half>(oacc[4 * w + e], al, b0[e], b1[e]);
        }
      }
    }
    __syncwarp();                              // every lane has read stage s
    if (lane == 0 && c + kQ8Stages < n_chunks) load(c + kQ8Stages);
  }
  l_lo += __shfl_xor_sync(0xffffffffu, l_lo, 1); l_lo += __shfl_xor_sync(0xffffffffu, l_lo, 2);
  l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 1); l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 2);
  __syncthreads();                             // the partial results take the rings' place
  if (s_abort) {
    // a wait ran out: give copies in flight time to land before shared memory is given up
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    return;
  }
  // ---- the warps' partial results -> shared memory [warp][row][D | max, sum], merged in fixed order.  Block j, column
  // pair (2t, 2t + 1) of this lane's accumulators: d = 2t * (D / 8) + j and (2t + 1) * (D / 8) + j
  float* part = reinterpret_cast<float*>(gen);
  {
    float* lo = part + (warp * kQ8Rows + g) * SM::kRow;
    float* hi = lo + 8 * SM::kRow;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int j = 0; j < NB; j += 4) {
        const int d = (2 * t + i) * (D / 8) + j;
        *reinterpret_cast<float4*>(lo + d) = make_float4(oacc[j][i], oacc[j + 1][i], oacc[j + 2][i], oacc[j + 3][i]);
        *reinterpret_cast<float4*>(hi + d) =
            make_float4(oacc[j][2 + i], oacc[j + 1][2 + i], oacc[j + 2][2 + i], oacc[j + 3][2 + i]);
      }
    }
    if (t == 0) {
      *reinterpret_cast<float2*>(lo + D) = make_float2(m_lo, l_lo);
      *reinterpret_cast<float2*>(hi + D) = make_float2(m_hi, l_hi);
    }
  }
  __syncthreads();
  constexpr int TPR = kQ8Threads / kQ8Rows, CW = D / TPR;          // threads per row, columns per thread
  const int row = threadIdx.x / TPR, c0 = (threadIdx.x % TPR) * CW;
  float mx = -INFINITY, tot = 0.f, acc[CW];
#pragma unroll
  for (int c = 0; c < CW; ++c) acc[c] = 0.f;
#pragma unroll
  for (int w = 0; w < kQ8Warps; ++w) mx = fmaxf(mx, part[(w * kQ8Rows + row) * SM::kRow + D]);
#pragma unroll
  for (int w = 0; w < kQ8Warps; ++w) {
    const float* src = part + (w * kQ8Rows + row) * SM::kRow;
    if (src[D + 1] == 0.f) continue;                               // saw no position of this row
    const float f = ex2_approx(src[D] - mx);
    tot = fmaf(f, src[D + 1], tot);
#pragma unroll
    for (int c = 0; c < CW; ++c) acc[c] = fmaf(f, src[c0 + c], acc[c]);
  }
  if (row >= rows) return;
  const int lim = last_of(row);
#pragma unroll
  for (int c = 0; c < CW; ++c)
    if (nan_from[c0 + c] <= lim) acc[c] = __uint_as_float(0x7fffffffu);
  if (p.n_splits > 1) {
    const long long at = (static_cast<long long>(split) * p.B * p.Hkv * p.tiles + unit) * kQ8Rows + row;
#pragma unroll
    for (int c = 0; c < CW; c += 4)
      *reinterpret_cast<float4*>(p.part_o + at * D + c0 + c) = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
    if (c0 == 0) p.part_ml[at] = make_float2(mx, tot);
    return;
  }
  const int rr = r0 + row, i = rr / p.G, hq = h * p.G + rr % p.G;
  const float inv = tot == 0.f ? 0.f : 1.0f / tot;
  T* dst = static_cast<T*>(p.o.ptr) + b * p.o.stride_b + static_cast<long long>(i) * p.o.stride_s +
           static_cast<long long>(hq) * p.o.stride_h + c0;
#pragma unroll
  for (int c = 0; c < CW; c += 8) {
    uint4 v;
    v.x = Io<T>::pack2(acc[c] * inv, acc[c + 1] * inv); v.y = Io<T>::pack2(acc[c + 2] * inv, acc[c + 3] * inv);
    v.z = Io<T>::pack2(acc[c + 4] * inv, acc[c + 5] * inv); v.w = Io<T>::pack2(acc[c + 6] * inv, acc[c + 7] * inv);
    *reinterpret_cast<uint4*>(dst + c) = v;
  }
  if (c0 == 0) {
    const float lse = mx - kQ8PBias + log2f(tot);
    if (p.lse != nullptr) p.lse[(static_cast<long long>(b) * p.Hq + hq) * p.M + i] = lse;
    if (p.part_ml != nullptr) p.part_ml[static_cast<long long>(unit) * kQ8Rows + row] = make_float2(mx, tot);
  }
}

// Merge of the splits and weights of the positions.  CTAs [0, merge_ctas): one warp per row; the rest: one thread per
// position of a (b, kv head), rows in ascending order.
constexpr int kQ8JoinThreads = 256;
template <typename T, int D>
__global__ void __launch_bounds__(kQ8JoinThreads)
attn_q8_join_kernel(const __grid_constant__ Q8Params p, int merge_ctas, int key_tiles) {
  extern __shared__ float q8_lse[];            // [R] (weight CTAs)
  griddep_wait();
  griddep_launch();
  if (*reinterpret_cast<volatile int*>(p.status) != 0) return;
  const long long units = static_cast<long long>(p.B) * p.Hkv * p.tiles;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (static_cast<int>(blockIdx.x) < merge_ctas) {
    const long long id = static_cast<long long>(blockIdx.x) * (kQ8JoinThreads / 32) + warp;     // (bh, r)
    if (id >= static_cast<long long>(p.B) * p.Hkv * p.R) return;
    const int r = static_cast<int>(id % p.R), bh = static_cast<int>(id / p.R);
    const long long at = (static_cast<long long>(bh) * p.tiles + r / kQ8Rows) * kQ8Rows + r % kQ8Rows;
    const long long step = units * kQ8Rows;
    constexpr int VPL = D / 32;
    float m = -INFINITY, tot = 0.f, acc[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) acc[i] = 0.f;
    for (int s = 0; s < p.n_splits; ++s) m = fmaxf(m, p.part_ml[s * step + at].x);
    for (int s = 0; s < p.n_splits; ++s) {
      const float2 ml = p.part_ml[s * step + at];
      if (ml.y == 0.f) continue;
      const float w = ex2_approx(ml.x - m);
      tot = fmaf(w, ml.y, tot);
      const float* src = p.part_o + (s * step + at) * D + lane * VPL;
#pragma unroll
      for (int i = 0; i < VPL; i += 2) {
        const float2 v = *reinterpret_cast<const float2*>(src + i);
        acc[i] = fmaf(w, v.x, acc[i]);
        acc[i + 1] = fmaf(w, v.y, acc[i + 1]);
      }
    }
    const int b = bh / p.Hkv, hq = (bh % p.Hkv) * p.G + r % p.G, i = r / p.G;
    const float inv = tot == 0.f ? 0.f : 1.0f / tot;
    T* dst = static_cast<T*>(p.o.ptr) + b * p.o.stride_b + static_cast<long long>(i) * p.o.stride_s +
             static_cast<long long>(hq) * p.o.stride_h + lane * VPL;
#pragma unroll
    for (int e = 0; e < VPL; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = Io<T>::pack2(acc[e] * inv, acc[e + 1] * inv);
    if (lane == 0 && p.lse != nullptr) p.lse[(static_cast<long long>(b) * p.Hq + hq) * p.M + i] = m - kQ8PBias + log2f(tot);
    return;
  }
  const int id = static_cast<int>(blockIdx.x) - merge_ctas;
  const int bh = id / key_tiles, b = bh / p.Hkv, h = bh % p.Hkv;
  const int n = p.len(b);
  const int key = (id % key_tiles) * kQ8JoinThreads + static_cast<int>(threadIdx.x);
  if ((id % key_tiles) * kQ8JoinThreads >= n) return;
  const long long step = units * kQ8Rows;
  for (int r = threadIdx.x; r < p.R; r += kQ8JoinThreads) {
    const long long at = (static_cast<long long>(bh) * p.tiles + r / kQ8Rows) * kQ8Rows + r % kQ8Rows;
    float m = -INFINITY, tot = 0.f;
    for (int s = 0; s < p.n_splits; ++s) m = fmaxf(m, p.part_ml[s * step + at].x);
    for (int s = 0; s < p.n_splits; ++s) {
      const float2 ml = p.part_ml[s * step + at];
      if (ml.y != 0.f) tot = fmaf(ex2_approx(ml.x - m), ml.y, tot);
    }
    q8_lse[r] = m - kQ8PBias + log2f(tot);
  }
  __syncthreads();
  if (key >= n) return;
  // causal: position j is seen by the queries i >= j - (n - M)
  const int first = p.causal ? max(key - (n - p.M), 0) * p.G : 0;
  const float* src = p.scores + static_cast<long long>(bh) * p.R * p.pitch + key;
  float acc = 0.f;
#pragma unroll 4
  for (int r = first; r < p.R; ++r) acc += ex2_approx(src[r * p.pitch] - q8_lse[r]);
  float* w = p.weight + b * p.w_sb + h * p.w_sh + key;
  *w = p.weight_add ? *w + acc : acc;
}

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

struct Q8Plan {
  int tiles, n_splits;
  size_t ml_off, o_off, score_off, total;
  long long pitch;
};

// How many CTAs share a (b, kv head, row tile)'s positions: enough to fill the SMs, at least two chunks a warp
Q8Plan plan_of(const TrnAttnQ8Args& a, int sm_count, bool splits_allowed) {
  Q8Plan w{};
  const int R = a.M * (a.Hq / a.Hkv);
  w.tiles = (R + kQ8Rows - 1) / kQ8Rows;
  const long long units = static_cast<long long>(a.B) * a.Hkv * w.tiles;
  const long long chunks = (static_cast<long long>(a.cache.S) + kQ8Keys - 1) / kQ8Keys;
  long long ns = static_cast<long long>(sm_count) * kQ8TargetCtas / units;
  if (ns > chunks / (2 * kQ8Warps)) ns = chunks / (2 * kQ8Warps);
  w.n_splits = ns < 1 || !splits_allowed ? 1 : static_cast<int>(ns);
  w.pitch = (a.cache.S + 31LL) / 32 * 32;
  size_t off = 0;
  w.ml_off = off;
  off += up256(static_cast<size_t>(w.n_splits) * units * kQ8Rows * sizeof(float2));
  w.o_off = off;
  if (w.n_splits > 1) off += up256(static_cast<size_t>(w.n_splits) * units * kQ8Rows * a.D * sizeof(float));
  w.score_off = off;
  if (a.weight != nullptr) off += up256(static_cast<size_t>(a.B) * a.Hkv * R * w.pitch * sizeof(float));
  w.total = off;
  if (w.n_splits == 1 && a.weight == nullptr) w.total = 0;
  return w;
}

template <typename T, int D>
int launch_typed(const TrnAttnQ8Args& a, cudaStream_t st, const DeviceState& ds) {
  using SM = Q8Smem<D>;
  constexpr bool HILO = Io<T>::kFmt == 0;
  const Q8Plan w = plan_of(a, kAttnNominalSMs, a.workspace != nullptr);
  Q8Params p{};
  p.q = a.q; p.o = a.o;
  CUtensorMap tm_k, tm_v;
  int rc = make_code_tmap(&tm_k, &p.ki, a.cache.k, a.cache.S, a.Hkv, a.B, D, kQ8Keys);
  if (rc == TRN_OK) rc = make_code_tmap(&tm_v, &p.vi, a.cache.v, a.cache.S, a.Hkv, a.B, D, kQ8Keys);
  if (rc != TRN_OK) return rc;
  p.ks = scale_table(a.cache.k_scale); p.vs = scale_table(a.cache.v_scale);
  p.len = KvLen{a.kv_len, a.kv_len_all, a.cache.S};
  p.lse = a.lse;
  p.B = a.B; p.M = a.M; p.Hq = a.Hq; p.Hkv = a.Hkv; p.G = a.Hq / a.Hkv; p.R = a.M * p.G;
  p.tiles = w.tiles; p.n_splits = w.n_splits;
  p.causal = a.causal;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.shift = block_shift(a.cache.block);
  p.status = ds.status;
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  if (w.total > 0) {
    p.part_ml = reinterpret_cast<float2*>(ws + w.ml_off);
    if (w.n_splits > 1) p.part_o = reinterpret_cast<float*>(ws + w.o_off);
    if (a.weight != nullptr) p.scores = reinterpret_cast<float*>(ws + w.score_off);
  }
  p.pitch = w.pitch;
  p.weight = a.weight; p.w_sb = a.weight_stride_b; p.w_sh = a.weight_stride_h; p.weight_add = a.weight_add;
  const long long units = static_cast<long long>(a.B) * a.Hkv * w.tiles;
  if (units * w.n_splits > 0x7fffffffLL) return TRN_E_SHAPE;
  auto kern = attn_q8_kernel<T, D, HILO>;
  rc = ensure_dyn_smem(reinterpret_cast<const void*>(kern), SM::kTotal, ds.device);
  if (rc != TRN_OK) return rc;
  const long long merge = w.n_splits > 1 ? (static_cast<long long>(a.B) * a.Hkv * p.R + 7) / 8 : 0;
  const int longest = a.kv_len != nullptr ? a.cache.S : min(max(a.kv_len_all, 0), a.cache.S);
  const int key_tiles = a.weight != nullptr ? (longest + kQ8JoinThreads - 1) / kQ8JoinThreads : 0;
  const long long join = merge + static_cast<long long>(a.B) * a.Hkv * key_tiles;
  if (join > 0x7fffffffLL) return TRN_E_SHAPE;
  TRN_CUDA_TRY(launch_pdl(kern, dim3(static_cast<unsigned>(units * w.n_splits)), dim3(kQ8Threads), SM::kTotal, st, tm_k, tm_v, p));
  if (join > 0)
    TRN_CUDA_TRY(launch_pdl(attn_q8_join_kernel<T, D>, dim3(static_cast<unsigned>(join)), dim3(kQ8JoinThreads),
                            a.weight != nullptr ? p.R * sizeof(float) : 0, st, p, static_cast<int>(merge), max(key_tiles, 1)));
  return TRN_OK;
}

constexpr int kQ8MaxWeightQueries = 16;
constexpr int kQ8MaxWeightRows = 8192;         // their log-sum-exps lie in 32 KB of shared memory

}  // namespace

int check_attention_q8(const TrnAttnQ8Args& a) {
  if (a.dtype != TRN_BF16 && a.dtype != TRN_FP16) return TRN_E_DTYPE;
  if (a.M <= 0 || a.Hq <= 0 || a.Hkv <= 0 || a.Hq % a.Hkv != 0) return TRN_E_SHAPE;
  if (static_cast<long long>(a.M) * a.Hq > 0x3fffffffLL) return TRN_E_SHAPE;
  if (!(a.scale > 0.f) || !(a.scale <= FLT_MAX)) return TRN_E_SHAPE;
  int rc = check_cache_q8(a.cache, a.B, a.Hkv, a.D);
  if (rc == TRN_OK) rc = check_rows(a.q, a.B, a.M, a.Hq, 8);
  if (rc == TRN_OK) rc = check_rows_distinct(a.o, a.B, a.M, a.Hq, 8, a.D);
  if (rc != TRN_OK) return rc;
  if (a.weight != nullptr) {
    if (a.M > kQ8MaxWeightQueries || a.M * (a.Hq / a.Hkv) > kQ8MaxWeightRows) return TRN_E_SHAPE;
    if ((a.B > 1 && a.weight_stride_b < 1) || (a.Hkv > 1 && a.weight_stride_h < 1)) return TRN_E_SHAPE;
  }
  const Q8Plan w = plan_of(a, kAttnNominalSMs, a.workspace != nullptr);
  if (w.total > 0 && (a.workspace == nullptr || (reinterpret_cast<uintptr_t>(a.workspace) & 255u) != 0 || a.workspace_bytes < w.total))
    return TRN_E_WORKSPACE;
  return TRN_OK;
}

int launch_attention_q8(const TrnAttnQ8Args& a, cudaStream_t st, const DeviceState& ds) {
  if (a.dtype == TRN_BF16)
    return a.D == 128 ? launch_typed<__nv_bfloat16, 128>(a, st, ds) : launch_typed<__nv_bfloat16, 64>(a, st, ds);
  return a.D == 128 ? launch_typed<__half, 128>(a, st, ds) : launch_typed<__half, 64>(a, st, ds);
}

size_t attention_q8_workspace(const TrnAttnQ8Args& a) {
  if (a.B <= 0 || a.M <= 0 || a.Hq <= 0 || a.Hkv <= 0 || a.Hq % a.Hkv != 0 || a.cache.S <= 0 || (a.D != 64 && a.D != 128)) return 0;
  return plan_of(a, kAttnNominalSMs, true).total;
}

}  // namespace trn
