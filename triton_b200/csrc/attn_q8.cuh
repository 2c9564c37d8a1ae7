// Pieces shared by the two kernels of the attention over the 8-bit cache (attn_q8.cu: few query rows per kv head, bound by
// memory; attn_q8_tc.cu: many, on the tensor cores of the 5th generation) and the merge of their partial results.
#pragma once

#include <math.h>

#include "attn_common.cuh"
#include "q8.cuh"

namespace trn {

// v's scale stands at its whole power of two in the running maximum, m' = max (t + ceil log2 vs), and as itself in the factor of
// the product:  E = 2^(t - m'),  l = sum E,  P' = E vs.  With vs within [2^-64, 2^120] the terms E of a row reach from
// 2^-120 (the maximum's own, at the largest scale) to 2^64, so the sum of up to 2^29 of them stays inside 32 bits with a
// factor of 2^30 (kQ8PBias + kQ8LBias), and what lies under 2^-126, which is flushed, is 2^-36 of the row's sum or less (2^-30 in
// attn_q8_tc.cu, whose P' carries at least 2^6 in the place of 2^12).  (l as sum of
// P' / vs loses the terms whose P' is flushed, although 1 / vs may make them the largest: scales 2^138 apart.)
constexpr float kQ8PBias = 12.f;               // log2 of the factor P' carries into the product
constexpr float kQ8LBias = 18.f;               // log2 of the factor E carries beside that
constexpr float kMinVScale = 5.421010862427522e-20f;   // 2^-64: in the maximum, smaller scales (0: a block of zeros) count as this

struct Q8Params {
  TrnHeadTensor q, o;
  HeadMapInfo ki, vi;
  ScaleTable ks, vs;
  KvLen len;
  float* lse;
  int B, M, Hq, Hkv, G, R;                     // R = M * G rows per (b, kv head): row r = query r / G, head r % G
  int tiles, tile_rows;                        // row tiles per (b, kv head), rows of one
  int causal;
  float scale_log2;
  int shift;                                   // log2(block)
  int ctas;                                    // CTAs the chunks are dealt out to; 0: a CTA per unit, nothing divided
  float* part_o;                               // [units + ctas][tile_rows][D], units = B * Hkv * tiles
  float2* part_ml;                             // [units + ctas][tile_rows]; without division [units][tile_rows] or NULL
  int2* pieces;                                // [units] CTAs of a unit's first and last piece
  // join_pairs > 0: the merge visits only the pairs of row tiles from join_first on, in the order late pairs first
  int join_pairs, join_first;
  int join_rows;                               // rows a CTA of the merge takes: 1, or as many as its threads are for
  int join_keys;                               // positions a CTA that sums weights takes
  float* scores;                               // [B * Hkv][R][pitch], log2 domain, or NULL
  long long pitch;
  float* weight;
  long long w_sb, w_sh;
  int weight_add;
  int* status;
};

// merge of the pieces (merge: whether there are any) and weights of the positions, by the kernel in attn_q8.cu
int launch_q8_join(const Q8Params& p, const TrnAttnQ8Args& a, bool merge, cudaStream_t st);
// many query rows per kv head (attn_q8_tc.cu): whether that kernel takes the call, its scratch, its launch
bool attn_q8_tc_applies(const TrnAttnQ8Args& a);
size_t attn_q8_tc_workspace(const TrnAttnQ8Args& a);
int launch_attn_q8_tc(const TrnAttnQ8Args& a, cudaStream_t st, const DeviceState& ds);

namespace {

__device__ __forceinline__ int last_seen(const Q8Params& p, int n, int r) {      // by row r of a (b, kv head); -1: nothing
  return p.causal ? max(n - p.M + r / p.G, -1) : n - 1;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
// byte offset of 16-byte unit u of row r in a tile as TMA wrote it: 128-byte rows with the 128-byte swizzle, 64-byte rows
// with the 64-byte swizzle
template <int D>
__device__ __forceinline__ uint32_t q8_off(uint32_t r, uint32_t u) {
  if constexpr (D == 128) return r * 128u + ((u ^ (r & 7u)) << 4);
  else return r * 64u + ((u ^ ((r >> 1) & 3u)) << 4);
}
// a scale of v: exponent of the next power of two in the running maximum, and the factor from E to P'
__device__ __forceinline__ void v_scale_terms(float s, float& lg, float& f) {
  lg = static_cast<float>(static_cast<int>((__float_as_uint(fmaxf(s, kMinVScale)) + 0x7fffffu) >> 23) - 127);
  f = s * 3.814697265625e-06f;                 // 2^-kQ8LBias
}
// a sum l moved to a maximum that is larger by -d: 2^d by halves, since d reaches -184 between a small and a large scale of v
// while what is left of l may still be most of the row's sum
__device__ __forceinline__ float sum_moved(float l, float d) {
  const float h = ex2_approx(0.5f * d);
  return l * h * h;
}
// 0xff in every byte of w that holds a NaN code (0x7f or 0xff)
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  return ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu;
}
// CW columns of a finished row, and its log-sum-exp
template <typename T, int CW>
__device__ __forceinline__ void q8_store_row(const Q8Params& p, int b, int h, int r, int c0, const float* acc, float mx, float tot) {
  const int i = r / p.G, hq = h * p.G + r % p.G;
  const float inv = tot == 0.f ? 0.f : 262144.f / tot;                // 2^kQ8LBias
  T* dst = static_cast<T*>(p.o.ptr) + b * p.o.stride_b + static_cast<long long>(i) * p.o.stride_s +
           static_cast<long long>(hq) * p.o.stride_h + c0;
#pragma unroll
  for (int c = 0; c < CW; c += 2) *reinterpret_cast<uint32_t*>(dst + c) = Io<T>::pack2(acc[c] * inv, acc[c + 1] * inv);
  if (c0 == 0 && p.lse != nullptr) p.lse[(static_cast<long long>(b) * p.Hq + hq) * p.M + i] = mx - (kQ8PBias + kQ8LBias) + log2f(tot);
}

inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }
// the parts of a call's parameters that do not depend on the kernel
inline Q8Params q8_params(const TrnAttnQ8Args& a, const DeviceState& ds) {
  Q8Params p{};
  p.q = a.q; p.o = a.o;
  p.ks = scale_table(a.cache.k_scale); p.vs = scale_table(a.cache.v_scale);
  p.len = KvLen{a.kv_len, a.kv_len_all, a.cache.S};
  p.lse = a.lse;
  p.B = a.B; p.M = a.M; p.Hq = a.Hq; p.Hkv = a.Hkv; p.G = a.Hq / a.Hkv; p.R = a.M * p.G;
  p.causal = a.causal;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.shift = block_shift(a.cache.block);
  p.status = ds.status;
  p.weight = a.weight; p.w_sb = a.weight_stride_b; p.w_sh = a.weight_stride_h; p.weight_add = a.weight_add;
  return p;
}

}  // namespace
}  // namespace trn
