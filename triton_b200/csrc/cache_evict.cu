// Eviction from a key/value cache by accumulated attention weight: what KeyFormer and RoCo keep their per-key statistics
// for (the reference reports the statistics and stops there, keyformer_llama_benchmark.py:74-79).
//
// Per (batch item, kv head) row of n positions: w[j] = sum over the row's score heads (64 bits, rounded to fp32); kept are
// j < first, j >= n - recent and of the others the largest w (equal ones by the lower j), min(n, keep) in all, in order.
//
// Launch 1 selects: one thread-block cluster per row, a CTA per slice of the positions, the slice's order-preserving 32-bit
// keys in shared memory.  A radix select finds the key of the last position kept, eight bits a pass: histogram of the
// slice, sum of the cluster's histograms, descent.  Then counts of kept positions per warp, CTA and cluster give every
// position its place, so the output is in order without a sort (a sort of 4096 scores by topk.cu: 27 us).
// Launch 2 moves: one CTA per (row, keys or values, group of destination positions) copies the kept rows; for 8-bit caches
// the group is a scale block, whose scale becomes the largest its rows had.
//
// Calls one behind another, and the launches by themselves (cold): 4 x 8 rows of 4096 positions (4 heads each), 1024 kept in 8 bits:
// 14.6 us; select 12.4, on as many CTAs as there are rows, and move 7.5 (two empty launches: 3.8).  2 rows of 32768 positions (71 heads
// each), 2048 kept in 16 bits: 20.5 us; sums 14.8 (17.8 MB: bound by the widening to 64 bits), select 12.4, move 4.2.  32 rows of
// 1040, 520 kept: 10.6 us; 8.8 and 5.5.  One row of 262144, 70001 kept: 38 us.
#include "q8.cuh"
#include "small_mma.cuh"

namespace trn {
namespace {

constexpr int kEvMaxCluster = 8;
constexpr int kEvMaxN = 262144;
constexpr int kEvThreads = 1024;
constexpr int kEvAhead = 4;             // positions a thread sums side by side
constexpr int kEvWarps = kEvThreads / 32;
static_assert(kEvWarps == 32, "one lane for each warp's counts");
constexpr int kEvMoveThreads = 256;
constexpr int kEvGroup16 = 64;          // destination positions per CTA of a 16-bit move

struct EvictParams {
  const float* scores;
  long long sc_sb, sc_sh;
  int group;                            // score heads per kv head
  int32_t* idx;
  float* scores_out;
  int32_t* len_out;
  KvLen len;
  int Hkv, keep, recent, first;
  int slice;                            // positions per CTA of a cluster
};

// ascending unsigned order == ascending float order; NaN of either sign above +inf, -0 as +0
__device__ __forceinline__ uint32_t order_key(float s) {
  if (s != s) return 0xfffffffeu;
  const uint32_t u = __float_as_uint(s + 0.0f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_score(uint32_t k) {
  if (k == 0xfffffffeu) return __uint_as_float(0x7fffffffu);
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// Long rows with many score heads: the heads' sums by the whole GPU first.  (Widening to 64 bits runs at a few lanes per
// clock: two clusters of 8 CTAs took 30 us for 71 heads of 32768 positions.)  A CTA takes kEvSumKeys positions, each by
// kEvSumParts threads that share its heads, so that a position's loads are under way together.
constexpr int kEvSumKeys = 64, kEvSumParts = 4;
// First head of part q: a position's sum is that of its kEvSumParts parts in order, whichever kernel takes it, so that the result
// does not depend on whether there is scratch.
__device__ __forceinline__ int part_begin(int group, int q) { return static_cast<int>(static_cast<long long>(group) * q / kEvSumParts); }
__global__ void __launch_bounds__(kEvSumKeys * kEvSumParts)
evict_sum_kernel(const float* __restrict__ scores, long long sc_sb, long long sc_sh, int group, KvLen len, int Hkv, int S, float* __restrict__ out) {
  __shared__ double part[kEvSumParts][kEvSumKeys];
  griddep_wait();
  griddep_launch();
  const int tiles = (S + kEvSumKeys - 1) / kEvSumKeys;
  const int row = static_cast<int>(blockIdx.x) / tiles, k = static_cast<int>(threadIdx.x) % kEvSumKeys, q = static_cast<int>(threadIdx.x) / kEvSumKeys;
  const int j = static_cast<int>(blockIdx.x) % tiles * kEvSumKeys + k;
  const int b = row / Hkv, h = row % Hkv;
  const bool there = j < len(b);
  double acc = 0.0;
  if (there) {
    const int g0 = part_begin(group, q), g1 = part_begin(group, q + 1);
    const float* src = scores + b * sc_sb + static_cast<long long>(h) * group * sc_sh + j;
#pragma unroll 10
    for (int g = g0; g < g1; ++g) acc += static_cast<double>(src[g * sc_sh]);
  }
  part[q][k] = acc;
  __syncthreads();
  if (q == 0 && there) {
#pragma unroll
    for (int i = 1; i < kEvSumParts; ++i) acc += part[i][k];
    out[static_cast<long long>(row) * S + j] = static_cast<float>(acc);
  }
}

__global__ void __launch_bounds__(kEvThreads)
evict_select_kernel(const __grid_constant__ EvictParams p, int cluster) {
  extern __shared__ __align__(16) uint32_t ev_keys[];          // [slice]
  // Three histograms in turn, so that one cluster barrier a pass is enough: pass i clears the one of pass i + 1, which the
  // other CTAs last read in pass i - 2, before the barrier of pass i - 1.
  __shared__ uint32_t hist[3][256];
  __shared__ uint32_t sum_of[256];
  __shared__ uint32_t found[3];                                // bin of the last kept key, keys above that bin, keys in it
  __shared__ uint32_t warp_gt[kEvWarps], warp_eq[kEvWarps];
  __shared__ uint32_t cta_cnt[2];
  const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31;
  griddep_wait();
  griddep_launch();
  const int rank = static_cast<int>(cluster_ctarank());
  const int row = static_cast<int>(blockIdx.x) / cluster;
  const int b = row / p.Hkv, h = row % p.Hkv;
  const int n = p.len(b);
  const int m = min(n, p.keep);
  const int lo = min(rank * p.slice, n), hi = min(lo + p.slice, n), cnt = hi - lo;
  const int tail0 = max(n - p.recent, 0);
  if (rank == 0 && h == 0 && tid == 0 && p.len_out != nullptr) p.len_out[b] = m;
  int32_t* idx = p.idx + static_cast<long long>(row) * p.keep;
  float* sout = p.scores_out != nullptr ? p.scores_out + static_cast<long long>(row) * p.keep : nullptr;
  for (int i = m + rank * kEvThreads + tid; i < p.keep; i += cluster * kEvThreads) {
    idx[i] = -1;
    if (sout != nullptr) sout[i] = 0.f;
  }
  // ---- keys of this CTA's slice
  const float* sc = p.scores + b * p.sc_sb + static_cast<long long>(h) * p.group * p.sc_sh + lo;
  if (p.group == 1) {
    for (int j = tid; j < cnt; j += kEvThreads) ev_keys[j] = order_key(sc[j]);
  } else {
    // kEvAhead positions at a time, so that enough loads are under way: a row's sum is one chain of Hs / Hkv adds.  (With less
    // heads than parts no part holds two, and the chain alone has the parts' order.)
    static_assert(kEvSumParts == 4, "three inner borders");
    const int e1 = part_begin(p.group, 1), e2 = part_begin(p.group, 2), e3 = part_begin(p.group, 3);
    for (int j0 = tid; j0 < cnt; j0 += kEvAhead * kEvThreads) {
      double acc[kEvAhead] = {}, done[kEvAhead] = {};
#pragma unroll 6
      for (int g = 0; g < p.group; ++g) {
        const float* src = sc + g * p.sc_sh + j0;
        if (g == e1 || g == e2 || g == e3) {                     // the part before is complete
#pragma unroll
          for (int i = 0; i < kEvAhead; ++i) {
            done[i] += acc[i];
            acc[i] = 0.0;
          }
        }
#pragma unroll
        for (int i = 0; i < kEvAhead; ++i)
          if (j0 + i * kEvThreads < cnt) acc[i] += static_cast<double>(src[i * kEvThreads]);
      }
#pragma unroll
      for (int i = 0; i < kEvAhead; ++i)
        if (j0 + i * kEvThreads < cnt) ev_keys[j0 + i * kEvThreads] = order_key(static_cast<float>(done[i] + acc[i]));
    }
  }
  if (tid < 256) hist[0][tid] = 0u;
  __syncthreads();
  auto eff = [&](int j) {                                      // protected positions rank above everything
    const int at = lo + j;
    return (at < p.first || at >= tail0) ? 0xffffffffu : ev_keys[j];
  };
  // ---- radix select: prefix = leading bits of the last kept key, need = how many of the keys with that prefix are kept
  uint32_t prefix = 0u, need = static_cast<uint32_t>(m), have = static_cast<uint32_t>(n);
  int shift = 32;                                              // keys >> shift == prefix is the undecided class
  int buf = 0;
  while (shift > 0 && need < have) {                           // uniform over the cluster
    const int ns = shift - 8;
    for (int j = tid; j < cnt; j += kEvThreads) {
      const uint32_t k = eff(j);
      if (shift == 32 || (k >> shift) == prefix) atomicAdd(&hist[buf][(k >> ns) & 255u], 1u);
    }
    if (tid < 256) hist[buf == 2 ? 0 : buf + 1][tid] = 0u;
    const uint32_t* bins = hist[buf];
    if (cluster > 1) {
      cluster_sync_all();
      if (tid < 256) {
        const uint32_t a = smem_u32(&hist[buf][tid]);
        uint32_t c = 0u;
#pragma unroll
        for (int r = 0; r < kEvMaxCluster; ++r)
          if (r < cluster) c += ld_cluster_u32(map_to_rank(a, static_cast<uint32_t>(r)));
        sum_of[tid] = c;
      }
      bins = sum_of;
    }
    __syncthreads();
    if (warp == 0) {
      // lane L owns bins 255 - 8 L ... 248 - 8 L, from the largest
      uint32_t c[8], mine = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        c[i] = bins[255 - 8 * lane - i];
        mine += c[i];
      }
      uint32_t incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      uint32_t above = incl - mine;
      if (above < need && incl >= need) {                      // the last kept key is in one of this lane's bins
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (above < need && above + c[i] >= need) {
            found[0] = static_cast<uint32_t>(255 - 8 * lane - i);
            found[1] = above;
            found[2] = c[i];
          }
          above += c[i];
        }
      }
    }
    __syncthreads();
    prefix = (shift == 32 ? 0u : prefix << 8) | found[0];
    need -= found[1];
    have = found[2];
    shift = ns;
    buf = buf == 2 ? 0 : buf + 1;
  }
  // kept: key >> shift above prefix, or equal to it and among the first `need` of those.  need == have: all of them.
  // ---- counts per warp (each owns a contiguous piece of the slice), then per CTA and cluster
  const int per = (cnt + kEvWarps - 1) / kEvWarps;
  const int w0 = min(warp * per, cnt), w1 = min(w0 + per, cnt);
  auto classify = [&](int j, bool& gt, bool& eq) {
    const uint32_t k = shift == 32 ? 0u : eff(j) >> shift;     // shift == 32: every position is kept
    gt = k > prefix;
    eq = k == prefix;
  };
  uint32_t ngt = 0u, neq = 0u;
  for (int j0 = w0; j0 < w1; j0 += 32) {
    bool gt = false, eq = false;
    if (j0 + lane < w1) classify(j0 + lane, gt, eq);
    ngt += __popc(__ballot_sync(0xffffffffu, gt));
    neq += __popc(__ballot_sync(0xffffffffu, eq));
  }
  if (lane == 0) { warp_gt[warp] = ngt; warp_eq[warp] = neq; }
  __syncthreads();
  if (warp == 0) {                                             // kEvWarps == 32: one warp's counts a lane
    const uint32_t x = warp_gt[lane], y = warp_eq[lane];
    uint32_t a = x, e = y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, a, o), v = __shfl_up_sync(0xffffffffu, e, o);
      if (lane >= o) { a += u; e += v; }
    }
    warp_gt[lane] = a - x;
    warp_eq[lane] = e - y;
    if (lane == 31) { cta_cnt[0] = a; cta_cnt[1] = e; }
  }
  if (cluster > 1) cluster_sync_all(); else __syncthreads();
  uint32_t gt0 = warp_gt[warp], eq0 = warp_eq[warp];
  for (int r = 0; r < rank; ++r) {
    gt0 += ld_cluster_u32(map_to_rank(smem_u32(&cta_cnt[0]), static_cast<uint32_t>(r)));
    eq0 += ld_cluster_u32(map_to_rank(smem_u32(&cta_cnt[1]), static_cast<uint32_t>(r)));
  }
  const uint32_t below = (1u << lane) - 1u;
  for (int j0 = w0; j0 < w1; j0 += 32) {
    bool gt = false, eq = false;
    if (j0 + lane < w1) classify(j0 + lane, gt, eq);
    const uint32_t bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq);
    const uint32_t g = gt0 + __popc(bg & below), e = eq0 + __popc(be & below);
    if (gt || (eq && e < need)) {
      const uint32_t at = g + min(e, need);
      idx[at] = lo + j0 + lane;
      if (sout != nullptr) sout[at] = key_score(ev_keys[j0 + lane]);
    }
    gt0 += __popc(bg);
    eq0 += __popc(be);
  }
  if (cluster > 1) cluster_sync_all();                         // no CTA leaves while its counts may be read
}

struct MoveParams {
  TrnHeadTensor src[2], dst[2];
  ScaleTable s_src[2], s_dst[2];
  const int32_t* idx;
  KvLen len;
  int Hkv, keep, shift, groups;
};

// rows of RB bytes.  Q8: a group is the 2^shift positions of a destination scale block; else kEvGroup16 positions.
template <int RB, bool Q8>
__global__ void __launch_bounds__(kEvMoveThreads)
evict_move_kernel(const __grid_constant__ MoveParams p) {
  constexpr int SEG = RB / 16, ROWS = kEvMoveThreads / SEG;
  constexpr int ELEM = Q8 ? 1 : 2;
  __shared__ int32_t from[128];
  __shared__ float had[128];
  __shared__ float part[kEvMoveThreads / 32];
  griddep_wait();
  griddep_launch();
  int u = static_cast<int>(blockIdx.x);
  const int kv = u & 1;
  u >>= 1;
  const int grp = u % p.groups, row = u / p.groups;
  const int b = row / p.Hkv, h = row % p.Hkv;
  const int m = min(p.len(b), p.keep);
  const int size = Q8 ? 1 << p.shift : kEvGroup16;
  const int g0 = grp * size, g1 = min(g0 + size, m);
  if (g0 >= g1) return;
  const int tid = static_cast<int>(threadIdx.x);
  float mine = 0.f;
  if (tid < g1 - g0) {
    const int j = p.idx[static_cast<long long>(row) * p.keep + g0 + tid];
    from[tid] = j;
    if constexpr (Q8) mine = *p.s_src[kv].at(b, j >> p.shift, h);
  }
  __syncthreads();
  // the rows are asked for before the scales are looked at: one memory latency for both
  constexpr int ITER = ((Q8 ? 128 : kEvGroup16) + ROWS - 1) / ROWS;
  const TrnHeadTensor src = p.src[kv], dst = p.dst[kv];
  const int seg = tid % SEG, r0 = tid / SEG;
  const uint8_t* s0 = static_cast<const uint8_t*>(src.ptr) + (b * src.stride_b + h * src.stride_h) * ELEM + seg * 16;
  uint8_t* d0 = static_cast<uint8_t*>(dst.ptr) + (b * dst.stride_b + h * dst.stride_h) * ELEM + seg * 16;
  uint4 c[ITER];
#pragma unroll
  for (int i = 0; i < ITER; ++i)
    if (r0 + i * ROWS < g1 - g0) c[i] = *reinterpret_cast<const uint4*>(s0 + from[r0 + i * ROWS] * (src.stride_s * ELEM));
  float top = 0.f;
  if constexpr (Q8) {
    if (tid < g1 - g0) had[tid] = mine;
    top = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((tid & 31) == 0) part[tid >> 5] = top;
    __syncthreads();
    top = part[0];
#pragma unroll
    for (int i = 1; i < kEvMoveThreads / 32; ++i) top = fmaxf(top, part[i]);
    if (tid == 0) *p.s_dst[kv].at(b, grp, h) = top;
  }
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int r = r0 + i * ROWS;
    if (r >= g1 - g0) continue;
    if constexpr (Q8) {
      const float s = had[r];
      if (s != top) {                                          // s < top (or NaN): the codes move to the larger scale
        const float ratio = s / top;
        uint32_t w[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 a = e4m3x2_to_f32(w[e] & 0xffffu), g = e4m3x2_to_f32(w[e] >> 16);
          w[e] = f32_to_e4m3x2(a.x * ratio, a.y * ratio) | (f32_to_e4m3x2(g.x * ratio, g.y * ratio) << 16);
        }
        c[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    *reinterpret_cast<uint4*>(d0 + (g0 + r) * (dst.stride_s * ELEM)) = c[i];
  }
}

// [lowest, highest) byte a (b, s, h, d) tensor touches, for the overlap check
void byte_range(const TrnHeadTensor& t, int B, int S, int H, int D, int elem, uintptr_t* lo, uintptr_t* hi) {
  *lo = reinterpret_cast<uintptr_t>(t.ptr);
  *hi = *lo + static_cast<uintptr_t>(((B - 1) * t.stride_b + (S - 1) * t.stride_s + (H - 1) * t.stride_h + D) * elem);
}

// whether the score heads are summed by a launch of their own: many scores a row, and scratch for the sums
bool evict_sums_first(const TrnCacheEvictArgs& a) { return a.workspace != nullptr && cache_evict_workspace(a) > 0; }

template <int RB, bool Q8>
int launch_move(const MoveParams& p, unsigned grid, cudaStream_t st) {
  TRN_CUDA_TRY(launch_pdl(evict_move_kernel<RB, Q8>, dim3(grid), dim3(kEvMoveThreads), 0, st, p));
  return TRN_OK;
}

}  // namespace

// below about 32 K scores a row the launch costs more than the sums
size_t cache_evict_workspace(const TrnCacheEvictArgs& a) {
  if (a.B <= 0 || a.Hkv <= 0 || a.Hs <= a.Hkv || a.Hs % a.Hkv != 0 || a.src.S <= 0) return 0;
  if (static_cast<long long>(a.src.S) * (a.Hs / a.Hkv) <= 32768) return 0;
  return static_cast<size_t>(a.B) * a.Hkv * a.src.S * sizeof(float);
}

int check_cache_evict(const TrnCacheEvictArgs& a) {
  if (a.workspace != nullptr && ((reinterpret_cast<uintptr_t>(a.workspace) & 3u) != 0 || a.workspace_bytes < cache_evict_workspace(a)))
    return TRN_E_WORKSPACE;
  if (a.scores == nullptr || a.idx == nullptr) return TRN_E_NULL;
  if (a.src.block != a.dst.block) return TRN_E_VARIANT;
  if (a.B <= 0 || a.Hkv <= 0 || a.Hs <= 0 || a.Hs % a.Hkv != 0) return TRN_E_SHAPE;
  if (a.D != 64 && a.D != 128) return TRN_E_SHAPE;
  if (a.keep <= 0 || a.recent < 0 || a.first < 0 || a.recent > a.keep || a.first > a.keep - a.recent) return TRN_E_SHAPE;
  if (a.src.S <= 0 || a.src.S > kEvMaxN || a.dst.S < a.keep || a.keep > kMaxPositions) return TRN_E_SHAPE;
  if (a.score_stride_b < 0 || a.score_stride_h < 0) return TRN_E_SHAPE;
  const bool q8 = a.src.block != 0;
  const TrnHeadTensor* t[4] = {&a.src.k, &a.src.v, &a.dst.k, &a.dst.v};
  for (int i = 0; i < 4; ++i) {
    const int S = i < 2 ? a.src.S : a.keep;
    const int rc = i < 2 ? check_rows(*t[i], a.B, S, a.Hkv, q8 ? 16 : 8)
                         : check_rows_distinct(*t[i], a.B, S, a.Hkv, q8 ? 16 : 8, a.D);
    if (rc != TRN_OK) return rc;
  }
  if (q8) {
    if (!q8_block_ok(a.src.block)) return TRN_E_SHAPE;
    int rc = check_scales(a.src.k_scale, a.B, (a.src.S - 1) / a.src.block + 1, a.Hkv);
    if (rc == TRN_OK) rc = check_scales(a.src.v_scale, a.B, (a.src.S - 1) / a.src.block + 1, a.Hkv);
    if (rc == TRN_OK) rc = check_scales(a.dst.k_scale, a.B, (a.keep - 1) / a.src.block + 1, a.Hkv);
    if (rc == TRN_OK) rc = check_scales(a.dst.v_scale, a.B, (a.keep - 1) / a.src.block + 1, a.Hkv);
    if (rc != TRN_OK) return rc;
  }
  // rows move in parallel: a destination inside the source's range could be overwritten before it is read.
  // Positions, scores and lengths of the result, and the scratch, are written while other rows' scores and lengths are read.
  const int64_t kept = static_cast<int64_t>(a.B) * a.Hkv * a.keep;
  const struct { const void* ptr; int64_t bytes; } area[6] = {
      {a.scores, ((a.B - 1) * a.score_stride_b + (a.Hs - 1) * a.score_stride_h + a.src.S) * 4}, {a.kv_len, a.B * 4LL}, {a.idx, kept * 4},
      {a.scores_out, kept * 4}, {a.kv_len_out, a.B * 4LL}, {a.workspace, static_cast<int64_t>(cache_evict_workspace(a))}};
  for (int i = 0; i < 6; ++i)
    for (int j = max(i + 1, 2); j < 6; ++j) {
      const uintptr_t l0 = reinterpret_cast<uintptr_t>(area[i].ptr), l1 = reinterpret_cast<uintptr_t>(area[j].ptr);
      if (l0 != 0 && l1 != 0 && area[j].bytes > 0 && l0 < l1 + area[j].bytes && l1 < l0 + area[i].bytes) return TRN_E_VARIANT;
    }
  for (int i = 0; i < 2; ++i)
    for (int j = 2; j < 4; ++j) {
      uintptr_t l0, h0, l1, h1;
      byte_range(*t[i], a.B, a.src.S, a.Hkv, a.D, q8 ? 1 : 2, &l0, &h0);
      byte_range(*t[j], a.B, a.keep, a.Hkv, a.D, q8 ? 1 : 2, &l1, &h1);
      if (l0 < h1 && l1 < h0) return TRN_E_VARIANT;
    }
  if (q8) {
    const TrnHeadTensor* ts[4] = {&a.src.k_scale, &a.src.v_scale, &a.dst.k_scale, &a.dst.v_scale};
    const int src_blocks = (a.src.S - 1) / a.src.block + 1, dst_blocks = (a.keep - 1) / a.src.block + 1;
    for (int i = 0; i < 2; ++i)
      for (int j = 2; j < 4; ++j) {
        uintptr_t l0, h0, l1, h1;
        byte_range(*ts[i], a.B, src_blocks, a.Hkv, 1, 4, &l0, &h0);
        byte_range(*ts[j], a.B, dst_blocks, a.Hkv, 1, 4, &l1, &h1);
        if (l0 < h1 && l1 < h0) return TRN_E_VARIANT;
      }
  }
  return TRN_OK;
}

int launch_cache_evict(const TrnCacheEvictArgs& a, cudaStream_t st, const DeviceState& ds) {
  const bool q8 = a.src.block != 0;
  const long long rows = static_cast<long long>(a.B) * a.Hkv;
  const int longest = a.kv_len != nullptr ? a.src.S : min(max(a.kv_len_all, 0), a.src.S);

  const int group = a.Hs / a.Hkv;
  const bool sum_first = evict_sums_first(a);
  // a cluster pays a barrier among its CTAs for each digit: it splits a row only where its scores are many (and SMs idle)
  int cluster = 1;
  const long long row_scores = static_cast<long long>(longest) * (sum_first ? 1 : group);
  while (cluster < kEvMaxCluster && (longest > 4096LL * cluster || row_scores > 32768LL * cluster) && rows * cluster * 2 <= ds.sm_count) cluster *= 2;
  while (cluster < kEvMaxCluster && longest > 32768 * cluster) cluster *= 2;      // 128 KB of keys at most
  EvictParams p{};
  p.scores = a.scores;
  p.sc_sb = a.score_stride_b; p.sc_sh = a.score_stride_h;
  p.group = group;
  if (sum_first) {
    p.scores = static_cast<const float*>(a.workspace);
    p.sc_sb = static_cast<long long>(a.Hkv) * a.src.S; p.sc_sh = a.src.S;
    p.group = 1;
  }
  p.idx = a.idx; p.scores_out = a.scores_out; p.len_out = a.kv_len_out;
  p.len = KvLen{a.kv_len, a.kv_len_all, a.src.S};
  p.Hkv = a.Hkv; p.keep = a.keep; p.recent = a.recent; p.first = a.first;
  p.slice = (max(longest, 1) + cluster - 1) / cluster;
  if (rows * cluster > 0x7fffffffLL) return TRN_E_SHAPE;

  MoveParams mv{};
  mv.src[0] = a.src.k; mv.src[1] = a.src.v;
  mv.dst[0] = a.dst.k; mv.dst[1] = a.dst.v;
  if (q8) {
    mv.s_src[0] = scale_table(a.src.k_scale); mv.s_src[1] = scale_table(a.src.v_scale);
    mv.s_dst[0] = scale_table(a.dst.k_scale); mv.s_dst[1] = scale_table(a.dst.v_scale);
    mv.shift = block_shift(a.src.block);
  }
  mv.idx = a.idx;
  mv.len = p.len;
  mv.Hkv = a.Hkv; mv.keep = a.keep;
  const int size = q8 ? a.src.block : kEvGroup16;
  mv.groups = (a.keep + size - 1) / size;
  const long long grid = 2LL * rows * mv.groups;
  if (grid > 0x7fffffffLL) return TRN_E_SHAPE;

  const size_t smem = static_cast<size_t>(p.slice) * sizeof(uint32_t);
  const int rc = ensure_dyn_smem(reinterpret_cast<const void*>(evict_select_kernel), 32768 * 4, ds.device);
  if (rc != TRN_OK) return rc;
  if (sum_first) {
    const long long sum_grid = rows * ((a.src.S + kEvSumKeys - 1) / kEvSumKeys);
    if (sum_grid > 0x7fffffffLL) return TRN_E_SHAPE;
    TRN_CUDA_TRY(launch_pdl(evict_sum_kernel, dim3(static_cast<unsigned>(sum_grid)), dim3(kEvSumKeys * kEvSumParts), 0, st, a.scores,
                            static_cast<long long>(a.score_stride_b), static_cast<long long>(a.score_stride_h), group, p.len, a.Hkv,
                            a.src.S, static_cast<float*>(a.workspace)));
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * cluster), 1, 1);
  cfg.blockDim = dim3(kEvThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  TRN_CUDA_TRY(cudaLaunchKernelEx(&cfg, evict_select_kernel, p, cluster));

  const unsigned g = static_cast<unsigned>(grid);
  if (q8) return a.D == 128 ? launch_move<128, true>(mv, g, st) : launch_move<64, true>(mv, g, st);
  return a.D == 128 ? launch_move<256, false>(mv, g, st) : launch_move<128, false>(mv, g, st);
}

}  // namespace trn
