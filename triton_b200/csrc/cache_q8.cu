// Append to and read from the 8-bit key/value cache: e4m3 codes with one power-of-two scale per `block` positions and kv
// head.  The 16-bit caches of the reference (convert_eval_rms.py:62-108) have no counterpart.
//
// Append:  e = min { e : amax <= 448 * 2^e } over the finite new elements of a block, s = 2^e (a block that already holds
// positions keeps max(s_old, s)), code = rne_e4m3(x / s); older codes c become rne_e4m3(c * s_old / s) where s grew.
// A power of two costs e4m3 nothing (its relative error is the same anywhere in its range) and makes x / s and the
// rewriting exact, so growing a scale token by token loses nothing but what falls under the smallest code.
//
// Both kernels are bound by memory: append reads 2 and writes 1 byte per new element, read the other way round.  8 x 2048 rows of
// 8 heads of 128 (100 MB each): 17.7 us a call (5.7 TB/s, 88 % of the copy rate) and 17.7; a single row 3.1 to 4.2 us by itself, 1.4 and
// 1.7 behind other launches of a graph.
#include "q8.cuh"

namespace trn {
namespace {

constexpr int kAppendThreads = 128;

struct AppendParams {
  TrnHeadTensor code[2], src[2];      // keys, values
  ScaleTable scale[2];
  KvLen len;
  int Hkv, M, block, shift;
  int blocks_per_seq;                 // blocks M new rows can touch
};

// One CTA per (b, h, touched block, keys or values): every thread holds VPT 8-element pieces of the block's T * D elements
// in registers between the block maximum and the conversion, so the new rows are read once.
template <typename T, int D, int VPT>
__global__ void __launch_bounds__(kAppendThreads)
cache_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int SEG = D / 8;
  griddep_wait();
  griddep_launch();
  int u = static_cast<int>(blockIdx.x);
  const int kv = u & 1;
  u >>= 1;
  const int jb = u % p.blocks_per_seq;
  u /= p.blocks_per_seq;
  const int h = u % p.Hkv, b = u / p.Hkv;
  const int held = p.len(b);
  const int first = ((held >> p.shift) + jb) << p.shift;                 // first position of this CTA's block
  const int end = static_cast<int>(min(static_cast<long long>(p.len.S), static_cast<long long>(held) + p.M));
  if (first >= end) return;
  const int older = max(0, held - first);                                // rows of the block that already hold positions
  const TrnHeadTensor src = p.src[kv], code = p.code[kv];
  const T* x0 = static_cast<const T*>(src.ptr) + b * src.stride_b + h * src.stride_h;
  uint8_t* c0 = static_cast<uint8_t*>(code.ptr) + b * code.stride_b + h * code.stride_h + first * code.stride_s;
  float* const slot = p.scale[kv].at(b, first >> p.shift, h);
  const float s_old = older > 0 ? *slot : 0.f;

  uint4 x[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = i * kAppendThreads + static_cast<int>(threadIdx.x);
    const int row = v / SEG, seg = v % SEG;
    x[i] = make_uint4(0u, 0u, 0u, 0u);
    if (row >= older && first + row < end)
      x[i] = *reinterpret_cast<const uint4*>(x0 + (first + row - held) * src.stride_s + seg * 8);
  }
  // largest magnitude: the bits without the sign order as the values do, two at a time; what is not finite has all
  // exponent bits set and sends the block through the loop that leaves such elements out
  __shared__ uint32_t part[kAppendThreads / 32];
  auto block_max = [&](uint32_t m) {
    m = max(m & 0xffffu, m >> 16);
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();                                                     // also: every thread has read the old scale
#pragma unroll
    for (int i = 0; i < kAppendThreads / 32; ++i) m = max(m, part[i]);
    return m;
  };
  constexpr uint32_t kInf = Io<T>::kFmt == 1 ? 0x7f80u : 0x7c00u;
  uint32_t top = 0u;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    top = __vmaxu2(top, __vmaxu2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu));
    top = __vmaxu2(top, __vmaxu2(x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu));
  }
  top = block_max(top);
  const bool all_finite = top < kInf;
  // the paths below that few blocks take are rolled loops that read the rows again: unrolled over the pieces in registers,
  // they were most of the kernel's code, and every CTA waited for it to be fetched (8 x 2048 rows of 8 heads of 128: 32.4 us against 17.5)
  auto again = [&](int i, uint32_t (&w)[4], int& row, int& seg) {
    const int v = i * kAppendThreads + static_cast<int>(threadIdx.x);
    row = v / SEG;
    seg = v % SEG;
    if (row < older || first + row >= end) return false;
    const uint4 y = *reinterpret_cast<const uint4*>(x0 + (first + row - held) * src.stride_s + seg * 8);
    w[0] = y.x; w[1] = y.y; w[2] = y.z; w[3] = y.w;
    return true;
  };
  if (!all_finite) {
    top = 0u;
#pragma unroll 1
    for (int i = 0; i < VPT; ++i) {
      uint32_t w[4];
      int row, seg;
      if (!again(i, w, row, seg)) continue;
      for (int e = 0; e < 4; ++e) {
        const uint32_t a = w[e] & 0x7fffu, c = (w[e] >> 16) & 0x7fffu;
        if (a < kInf) top = max(top, a);
        if (c < kInf) top = max(top, c);
      }
    }
    __syncthreads();                                                     // part is free again
    top = block_max(top);
  }
  const float amax = Io<T>::unpack2(top).x;
  const float need = exp2_int(scale_exp(amax));
  const bool grew = !(s_old >= need);
  const float s = grew ? need : s_old;
  if (threadIdx.x == 0 && (grew || older == 0)) *slot = s;
  auto put = [&](int row, int seg, const float (&f)[8]) {
    uint2 r;
    r.x = f32_to_e4m3x2(f[0], f[1]) | (f32_to_e4m3x2(f[2], f[3]) << 16);
    r.y = f32_to_e4m3x2(f[4], f[5]) | (f32_to_e4m3x2(f[6], f[7]) << 16);
    *reinterpret_cast<uint2*>(c0 + row * code.stride_s + seg * 8) = r;
  };
  if (older > 0 && grew) {                                               // older codes move to the larger scale
    const float ratio = s_old / s;
#pragma unroll 1
    for (int v = static_cast<int>(threadIdx.x); v < older * SEG; v += kAppendThreads) {
      const int row = v / SEG, seg = v % SEG;
      const uint2 c = *reinterpret_cast<const uint2*>(c0 + row * code.stride_s + seg * 8);
      const float2 a0 = e4m3x2_to_f32(c.x & 0xffffu), a1 = e4m3x2_to_f32(c.x >> 16);
      const float2 a2 = e4m3x2_to_f32(c.y & 0xffffu), a3 = e4m3x2_to_f32(c.y >> 16);
      put(row, seg, {a0.x * ratio, a0.y * ratio, a1.x * ratio, a1.y * ratio, a2.x * ratio, a2.y * ratio, a3.x * ratio, a3.y * ratio});
    }
  }
  // a power of two has an exact reciprocal; a foreign scale (a cache the caller filled) divides
  if (all_finite && (__float_as_uint(s) & 0x7fffffu) == 0u) {
    const float inv = 1.0f / s;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = i * kAppendThreads + static_cast<int>(threadIdx.x);
      const int row = v / SEG, seg = v % SEG;
      if (row < older || first + row >= end) continue;
      const float2 a0 = Io<T>::unpack2(x[i].x), a1 = Io<T>::unpack2(x[i].y), a2 = Io<T>::unpack2(x[i].z), a3 = Io<T>::unpack2(x[i].w);
      put(row, seg, {a0.x * inv, a0.y * inv, a1.x * inv, a1.y * inv, a2.x * inv, a2.y * inv, a3.x * inv, a3.y * inv});
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < VPT; ++i) {
      uint32_t w[4];
      int row, seg;
      if (!again(i, w, row, seg)) continue;
      float f[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 g = Io<T>::unpack2(w[e]);
        f[2 * e] = g.x;
        f[2 * e + 1] = g.y;
      }
      for (int e = 0; e < 8; ++e) f[e] = fabsf(f[e]) <= FLT_MAX ? __fdiv_rn(f[e], s) : __uint_as_float(0x7fffffffu);
      put(row, seg, f);
    }
  }
}

constexpr int kReadThreads = 256;

struct ReadParams {
  TrnHeadTensor code[2], dst[2];
  ScaleTable scale[2];
  KvLen len;
  int Hkv, shift, tiles;
};

// One CTA per (b, h, tile of positions, keys or values); a thread turns 8 codes into 16 bytes, kReadAhead rows at a time: every
// load and store of a warp covers whole lines
constexpr int kReadAhead = 4;
template <typename T, int D>
__global__ void __launch_bounds__(kReadThreads)
cache_read_kernel(const __grid_constant__ ReadParams p) {
  constexpr int SEG = D / 8, ROWS = kReadThreads / SEG;
  griddep_wait();
  griddep_launch();
  int u = static_cast<int>(blockIdx.x);
  const int kv = u & 1;
  u >>= 1;
  const int tile = u % p.tiles;
  u /= p.tiles;
  const int h = u % p.Hkv, b = u / p.Hkv;
  const int n = p.len(b);
  const TrnHeadTensor dst = p.dst[kv], code = p.code[kv];
  const int seg = static_cast<int>(threadIdx.x) % SEG, row0 = tile * kReadAhead * ROWS + static_cast<int>(threadIdx.x) / SEG;
  const uint8_t* c0 = static_cast<const uint8_t*>(code.ptr) + b * code.stride_b + h * code.stride_h + seg * 8;
  T* y0 = static_cast<T*>(dst.ptr) + b * dst.stride_b + h * dst.stride_h + seg * 8;
  uint2 c[kReadAhead];
  float s[kReadAhead];
#pragma unroll
  for (int i = 0; i < kReadAhead; ++i) {
    const int row = row0 + i * ROWS;
    if (row < n) {
      c[i] = *reinterpret_cast<const uint2*>(c0 + row * code.stride_s);
      s[i] = *p.scale[kv].at(b, row >> p.shift, h);
    }
  }
#pragma unroll
  for (int i = 0; i < kReadAhead; ++i) {
    const int row = row0 + i * ROWS;
    if (row >= n) continue;
    const float2 a0 = e4m3x2_to_f32(c[i].x & 0xffffu), a1 = e4m3x2_to_f32(c[i].x >> 16);
    const float2 a2 = e4m3x2_to_f32(c[i].y & 0xffffu), a3 = e4m3x2_to_f32(c[i].y >> 16);
    *reinterpret_cast<uint4*>(y0 + row * dst.stride_s) =
        make_uint4(Io<T>::pack2(a0.x * s[i], a0.y * s[i]), Io<T>::pack2(a1.x * s[i], a1.y * s[i]),
                   Io<T>::pack2(a2.x * s[i], a2.y * s[i]), Io<T>::pack2(a3.x * s[i], a3.y * s[i]));
  }
}

template <typename T, int D>
int append_typed(const TrnCacheAppendArgs& a, const AppendParams& p, unsigned grid, cudaStream_t st) {
  const int vpt = a.cache.block * D / 8 / kAppendThreads;
  const dim3 g(grid), t(kAppendThreads);
  switch (vpt) {
    case 1: TRN_CUDA_TRY(launch_pdl(cache_append_kernel<T, D, 1>, g, t, 0, st, p)); break;
    case 2: TRN_CUDA_TRY(launch_pdl(cache_append_kernel<T, D, 2>, g, t, 0, st, p)); break;
    case 4: TRN_CUDA_TRY(launch_pdl(cache_append_kernel<T, D, 4>, g, t, 0, st, p)); break;
    case 8: TRN_CUDA_TRY(launch_pdl(cache_append_kernel<T, D, 8>, g, t, 0, st, p)); break;
    default: TRN_CUDA_TRY(launch_pdl(cache_append_kernel<T, D, 16>, g, t, 0, st, p)); break;
  }
  return TRN_OK;
}

template <typename T, int D>
int read_typed(const TrnCacheReadArgs& a, ReadParams& p, cudaStream_t st) {
  constexpr int kRows = kReadAhead * kReadThreads / (D / 8);
  const int room = p.len.S, longest = a.kv_len != nullptr ? room : min(max(a.kv_len_all, 0), room);
  p.tiles = (longest + kRows - 1) / kRows;
  const long long grid = 2LL * a.B * a.Hkv * p.tiles;
  if (grid > 0x7fffffffLL) return TRN_E_SHAPE;
  if (grid == 0) return TRN_OK;
  TRN_CUDA_TRY(launch_pdl(cache_read_kernel<T, D>, dim3(static_cast<unsigned>(grid)), dim3(kReadThreads), 0, st, p));
  return TRN_OK;
}

}  // namespace

int check_cache_append(const TrnCacheAppendArgs& a) {
  if (a.dtype != TRN_BF16 && a.dtype != TRN_FP16) return TRN_E_DTYPE;
  if (a.M <= 0) return TRN_E_SHAPE;
  int rc = check_cache_q8(a.cache, a.B, a.Hkv, a.D);
  if (rc == TRN_OK) rc = check_rows(a.k_new, a.B, a.M, a.Hkv, 8);
  if (rc == TRN_OK) rc = check_rows(a.v_new, a.B, a.M, a.Hkv, 8);
  return rc;
}

int launch_cache_append(const TrnCacheAppendArgs& a, cudaStream_t st) {
  AppendParams p{};
  p.code[0] = a.cache.k; p.code[1] = a.cache.v;
  p.src[0] = a.k_new; p.src[1] = a.v_new;
  p.scale[0] = scale_table(a.cache.k_scale); p.scale[1] = scale_table(a.cache.v_scale);
  p.len = KvLen{a.kv_len, a.kv_len_all, a.cache.S};
  p.Hkv = a.Hkv; p.M = a.M; p.block = a.cache.block; p.shift = block_shift(a.cache.block);
  const int rows = min(a.M, a.cache.S);
  p.blocks_per_seq = (rows - 1 + p.block - 1) / p.block + 1;            // the first block may be entered at its last row
  const long long grid = 2LL * a.B * a.Hkv * p.blocks_per_seq;
  if (grid > 0x7fffffffLL) return TRN_E_SHAPE;
  const unsigned g = static_cast<unsigned>(grid);
  if (a.dtype == TRN_BF16)
    return a.D == 128 ? append_typed<__nv_bfloat16, 128>(a, p, g, st) : append_typed<__nv_bfloat16, 64>(a, p, g, st);
  return a.D == 128 ? append_typed<__half, 128>(a, p, g, st) : append_typed<__half, 64>(a, p, g, st);
}

int check_cache_read(const TrnCacheReadArgs& a) {
  if (a.dtype != TRN_BF16 && a.dtype != TRN_FP16) return TRN_E_DTYPE;
  int rc = check_cache_q8(a.cache, a.B, a.Hkv, a.D);
  if (rc == TRN_OK && a.S_out <= 0) rc = TRN_E_SHAPE;
  if (rc == TRN_OK) rc = check_rows_distinct(a.k_out, a.B, a.S_out, a.Hkv, 8, a.D);
  if (rc == TRN_OK) rc = check_rows_distinct(a.v_out, a.B, a.S_out, a.Hkv, 8, a.D);
  return rc;
}

int launch_cache_read(const TrnCacheReadArgs& a, cudaStream_t st) {
  ReadParams p{};
  p.code[0] = a.cache.k; p.code[1] = a.cache.v;
  p.dst[0] = a.k_out; p.dst[1] = a.v_out;
  p.scale[0] = scale_table(a.cache.k_scale); p.scale[1] = scale_table(a.cache.v_scale);
  p.len = KvLen{a.kv_len, a.kv_len_all, min(a.cache.S, a.S_out)};
  p.Hkv = a.Hkv; p.shift = block_shift(a.cache.block);
  if (a.dtype == TRN_BF16)
    return a.D == 128 ? read_typed<__nv_bfloat16, 128>(a, p, st) : read_typed<__nv_bfloat16, 64>(a, p, st);
  return a.D == 128 ? read_typed<__half, 128>(a, p, st) : read_typed<__half, 64>(a, p, st);
}

}  // namespace trn
