// Pieces shared by the kernels of the 8-bit key/value cache (cache_q8.cu, cache_evict.cu, attn_q8.cu, attn_q8_tc.cu):
// argument checks, how many positions a sequence holds, e4m3 conversions and power-of-two scales.
#pragma once

#include <float.h>

#include "common.cuh"
#include "host.h"

namespace trn {
namespace {

constexpr float kE4m3Max = 448.f;
constexpr int kScaleExpMin = -64, kScaleExpMax = 120;

// positions sequence b holds, within [0, S]
struct KvLen {
  const int32_t* ptr;
  int all, S;
  __device__ __forceinline__ int operator()(int b) const {
    const int n = ptr != nullptr ? ptr[b] : all;
    return min(max(n, 0), S);
  }
};

// fp32 scale table (b, block, h)
struct ScaleTable {
  float* ptr;
  long long sb, sj, sh;
  __device__ __forceinline__ float* at(int b, int j, int h) const { return ptr + b * sb + j * sj + h * sh; }
};
inline ScaleTable scale_table(const TrnHeadTensor& t) {
  return ScaleTable{static_cast<float*>(t.ptr), t.stride_b, t.stride_s, t.stride_h};
}

// ---- conversions ---------------------------------------------------------------------------------
// two e4m3 codes (low byte first) -> two fp16 values: exact, NaN stays NaN
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t codes) {
  uint32_t r;
  const uint16_t c = static_cast<uint16_t>(codes);
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
  return r;
}
__device__ __forceinline__ float2 e4m3x2_to_f32(uint32_t codes) {
  const uint32_t h = e4m3x2_to_f16x2(codes);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// two fp32 values -> two e4m3 codes (lo in the low byte), nearest even, saturating; NaN -> NaN
__device__ __forceinline__ uint32_t f32_to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// smallest e with amax <= 448 * 2^e = 1.75 * 2^(e + 8), clamped; amax finite, >= 0
__device__ __forceinline__ int scale_exp(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kScaleExpMin), kScaleExpMax);
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// ---- host-side checks ------------------------------------------------------------------------------
// base and strides of a (b, s, h, d) tensor whose rows are moved 16 bytes at a time: `mult` elements are 16 bytes.
// Dims of extent 1 may carry any stride.
inline int check_rows(const TrnHeadTensor& t, int B, int S, int H, int mult) {
  if (t.ptr == nullptr) return TRN_E_NULL;
  if (!aligned16(t.ptr)) return TRN_E_ALIGN;
  const int64_t st[3] = {t.stride_b, t.stride_s, t.stride_h};
  const int ext[3] = {B, S, H};
  for (int i = 0; i < 3; ++i) {
    if (ext[i] <= 1) continue;
    if (st[i] < 0) return TRN_E_SHAPE;
    if (st[i] % mult != 0) return TRN_E_ALIGN;
  }
  return TRN_OK;
}
// the same for a tensor that is written (or read by TMA): no two rows may share an address through a zero stride
inline int check_rows_distinct(const TrnHeadTensor& t, int B, int S, int H, int mult, int D) {
  const int rc = check_rows(t, B, S, H, mult);
  if (rc != TRN_OK) return rc;
  const int64_t st[3] = {t.stride_b, t.stride_s, t.stride_h};
  const int ext[3] = {B, S, H};
  for (int i = 0; i < 3; ++i)
    if (ext[i] > 1 && st[i] < D) return TRN_E_SHAPE;
  return TRN_OK;
}
inline int check_scales(const TrnHeadTensor& t, int B, int blocks, int H) {
  if (t.ptr == nullptr) return TRN_E_NULL;
  if ((reinterpret_cast<uintptr_t>(t.ptr) & 3u) != 0) return TRN_E_ALIGN;
  if ((B > 1 && t.stride_b < 1) || (blocks > 1 && t.stride_s < 1) || (H > 1 && t.stride_h < 1)) return TRN_E_SHAPE;
  return TRN_OK;
}
constexpr int kMaxPositions = 1 << 29;      // positions and block starts stay in 32 bits
inline bool q8_block_ok(int block) { return block == 16 || block == 32 || block == 64 || block == 128; }
// a whole 8-bit cache
inline int check_cache_q8(const TrnCacheQ8& c, int B, int Hkv, int D) {
  if (B <= 0 || Hkv <= 0 || c.S <= 0 || c.S > kMaxPositions) return TRN_E_SHAPE;
  if (D != 64 && D != 128) return TRN_E_SHAPE;
  if (!q8_block_ok(c.block)) return TRN_E_SHAPE;
  int rc = check_rows_distinct(c.k, B, c.S, Hkv, 16, D);
  if (rc == TRN_OK) rc = check_rows_distinct(c.v, B, c.S, Hkv, 16, D);
  const int blocks = (c.S - 1) / c.block + 1;
  if (rc == TRN_OK) rc = check_scales(c.k_scale, B, blocks, Hkv);
  if (rc == TRN_OK) rc = check_scales(c.v_scale, B, blocks, Hkv);
  return rc;
}
inline int block_shift(int block) { return block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : 7; }

}  // namespace
}  // namespace trn
