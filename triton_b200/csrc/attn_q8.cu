// Attention over the 8-bit key/value cache: o = softmax(scale * q k^T) v with k = kc * ks, v = vc * vs (e4m3 codes, one
// fp32 scale per `block` positions and kv head), sequences of their own lengths, causal or not, any Hq / Hkv.
//
// Mathematics.  e4m3 codes are fp16 values exactly (one conversion instruction for two of them), so both products run in
// fp16 with fp32 accumulation and no scale ever enters them:
//   * q enters as fp16 times a power of two per row (2^(14 - e), e the exponent of the row's largest element): exact for
//     fp16 q, and for bf16 q but for elements 2^-28 below the row's largest, whose error is at most 2^-39 of that one;
//   * ks multiplies the score:  t = acc * (scale * log2 e * row factor * ks);
//   * vs enters the running maximum and one multiplication:  m' = max (t + log2 vs),  E = 2^(t - m'),  l = sum E,
//     P' = E vs <= 1,  O = sum P' vc,  o = O / l,  lse = m' + log2 l.
//     P' is what its key adds to O whatever its block's scale, so its rounding to 16 bits is relative to the largest of
//     these, taken over the row.  (A column in which the blocks of large scale hold nothing but zeros gets its values from P' that
//     are smaller by the scales' ratio: with scales 2^26 (attn_q8_tc.cu: 2^20) and more apart these are subnormal in fp16, and such
//     a column is off by up to 448 * 2^-37 (2^-31) of the row's largest p vs for each position.)
// P' carries a factor 2^12 into the product (it cancels in O / l), which keeps weights down to 2^-26 of the row's largest out of
// fp16's subnormals.  P' goes into the product as two fp16 parts, hi + lo, off by 2^-22 of itself; with single_p as one, off by
// 2^-11 (the outputs' own rounding: bf16 2^-8, fp16 2^-11).
//
// This kernel is for few query rows per kv head: a CTA of four warps owns up to 8 NT of the M * Hq / Hkv rows of a (b, kv head)
// and a share of its positions; each warp walks its quarter in chunks of 32 positions through its own ring of TMA
// tiles.  Both products are taken transposed, s^T = k q^T and o^T = v^T p^T, so that positions and head_dim fill the
// 16-row side of m16n8k16 and eight query rows the 8-column side: a decode step of 4 to 8 heads per kv head wastes
// little.  p^T becomes an operand with one 8x8 transposition (movmatrix) per 8 positions.  Codes go from shared memory to
// registers as the 16 bytes a lane needs: the order of the d axis inside a product and of the rows inside the output is
// free, so the fragments are picked such that the reads have no bank conflicts under the TMA swizzle (k: lane (g, t)
// reads units 2t and 2t + 1 of positions g, g + 8; v: unit g of positions 2t, 2t + 1).  The running maximum is shared by a
// row's lanes and only raised when some score passes it by 2^3, so most chunks need no reduction across lanes.
// Long caches: the chunks of all units are dealt out in equal shares to one round of CTAs, and a second small kernel merges
// the pieces and sums the per-position weights from scores kept in the workspace.  Short ones: a cluster per unit meets in
// shared memory, one launch.  Pieces, rows and sums are taken in a fixed order: bitwise reproducible.
//
// Measured (calls one behind another on inputs that change; 5 to 10 % more on other machines): 2 sequences of 100001 and 131071
// positions, 32 / 8 heads of 128, fp16 (473 MB): 88 us = 5.4 TB/s, 83 % of the copy rate, of which the merge 5 us; 32 of 1000..8192
// with weights, bf16 (307 MB): 79 us, 66 without (4.7 TB/s: a CTA ends one unit and begins the next with an empty ring); one of
// 1040: 9.1 us, launch and the chain length -> tile -> scores -> product -> cluster.
//
// What must not be seen cannot hurt: scores behind a row's last position are replaced, not weighted, and in the
// chunks where that happens NaN codes of v are taken as 0 in the product (0 * NaN would poison rows that do not see them) and
// put back as NaN into the outputs of the rows that do.
#include "attn_q8.cuh"
#include "small_mma.cuh"

namespace trn {
namespace {

constexpr int kQ8Warps = 4;
constexpr int kQ8Threads = 32 * kQ8Warps;
constexpr int kQ8Keys = 32;                    // positions per chunk
constexpr float kQ8Slack = 3.f;                // log2 of how far a score may pass the running maximum (2^15 fits fp16)
constexpr int kQ8MaxCluster = 8;
constexpr int kQ8Keep = 4;                     // chunks a warp of a cluster takes at most
// Stages of a warp's ring, and how many CTAs an SM then has room for.  Three CTAs of two stages where units are many (a CTA
// ends one and begins others, while the rest of the SM keeps loading); two CTAs of three stages where a unit lies on
// two CTAs and more.  Measured at head_dim 128 (us, bf16), two stages and three: 256 units of 1000..8192 positions 66.4, 71.4; 16 units
// of 100001..131071 92.0, 86.6; 128 units of 16384 100.0, 97.0; 152 of these 117, 114, and 256 of them 184, 179: it is units of
// unequal lengths that gain from the first form.  Head_dim 64 keeps that (26.9 against 31.9, p in one part).
// Two CTAs also where a lane's 200 and more registers leave no room for a third: 16 rows of head_dim 128, 32 of 64.
int q8_stages(int D, int tile_rows, long long units, int sm_count) {
  return D == 128 && (tile_rows == 16 || units <= sm_count) ? 3 : 2;
}
int q8_ctas(int D, int tile_rows, int stages) { return stages == 3 || (D == 64 && tile_rows == 32) ? 2 : 3; }

// rows a CTA takes: 8, 16 or (head_dim 64, where the output leaves registers for it) 32
__host__ __device__ constexpr int q8_max_tiles(int D) { return D == 64 ? 4 : 2; }

template <int D, int NT, int ST>
struct Q8Smem {
  static constexpr int kRows = 8 * NT;
  static constexpr int kTile = kQ8Keys * D;                        // bytes of k or v of a chunk
  static constexpr int kWarpRing = ST * 2 * kTile;
  static constexpr int kRing = kQ8Warps * kWarpRing;
  static constexpr int kRow = D + 4;                               // o | max, sum  of a warp's partial result
  static constexpr int kPart = kQ8Warps * kRows * kRow * 4;        // overlays the ring after the key loop
  static constexpr int kTPR = kQ8Threads / kRows;                  // threads and columns a thread of the merge
  static constexpr int kCW = D / kTPR;
  static constexpr int kMine = kPart;                              // a CTA's merged result, read by its cluster
  static constexpr int kEnd = kMine + kRows * kRow * 4;
  static constexpr int kBody = kRing > kEnd ? kRing : kEnd;
  static constexpr int kBars = kBody;
  static constexpr int kTotal = kBars + 128 + 1024;                // + slack to align the base to 1024 bytes
  // launches of clusters that also sum weights: [warp][row][kKeptPitch] scores.  The pitch spreads a warp's stores (eight
  // positions of four rows two apart) over all banks.
  static constexpr int kKept = kBars + 128;
  static constexpr int kKeptPitch = kQ8Keep * kQ8Keys + 4;
  static constexpr int kTotalKept = kTotal + kQ8Warps * kRows * kKeptPitch * 4;
};

__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
// which row of an 8-row block column c of a score block is.  64-byte rows: a quad's even columns 0, 2, 4, 6 and the lane
// groups' neighbours have to meet different halves of a 128-byte line, hence 0 3 1 2 4 7 5 6
template <int D>
__device__ __forceinline__ int q8_key(int c) {
  if constexpr (D == 128) return c;
  else return (c & 4) + ((0x2130 >> ((c & 3) * 4)) & 3) ;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
// transposes an 8x8 matrix of 16-bit values held two to a lane
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// ---- who does what.  A unit is a (b, kv head, row tile) with the chunks its sequence holds (one where it holds none, to write
// the empty rows; a tile whose rows do not see the last ones skips them).  All units' chunks, in order, are dealt out in equal
// contiguous shares, so a CTA's share may end one unit and begin others, and a unit lies on CTAs [first, last]: pieces.
// Each new piece begins a new unit, a new CTA or both, so slot = unit + CTA numbers the pieces' partial results, a
// unit's side by side.
__device__ __forceinline__ int chunks_of(int n) { return max((n + kQ8Keys - 1) / kQ8Keys, 1); }
// chunks of the sequences before b and of all, for one (kv head, row tile) (a whole warp, same arguments)
__device__ __forceinline__ int2 chunks_before(const Q8Params& p, int b) {
  int x = 0, y = 0;
  for (int i = threadIdx.x & 31; i < p.B; i += 32) {
    const int c = chunks_of(p.len(i));
    y += c;
    if (i < b) x += c;
  }
  return make_int2(static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(x))),
                   static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(y))));
}
__device__ __forceinline__ unsigned share_of(const Q8Params& p, int all) {       // chunks of one CTA, at least one a warp
  return max((static_cast<unsigned>(all) * p.Hkv * p.tiles + p.ctas - 1) / p.ctas, static_cast<unsigned>(kQ8Warps));
}
// What a warp of a CTA has to do for one piece of a unit.
struct Q8Piece {
  int b, h, n, r0, rows;                       // sequence, kv head, its length; first row and rows of the tile
  int lim_min, lim_max;                        // last position that the tile's first / last row sees
  int chunk0, n_chunks;                        // of this warp
  int loaded;                                  // chunks this warp's ring has taken before: stage and parity go on
  float* kept;                                 // where row 0 keeps its scores (log2 domain), or NULL
  long long kept_pitch;
  int kept_from;                               // the position that lies at kept[0]
  __device__ __forceinline__ int last_of(const Q8Params& p, int r) const { return r >= rows ? -1 : last_seen(p, n, r0 + r); }
};
// the tile's rows and this warp's quarter of chunks [skip, skip + many) of unit (b, h, tile): those that some row sees
__device__ __forceinline__ Q8Piece piece_of(const Q8Params& p, int b, int h, int tile, int skip, int many, int warp) {
  Q8Piece w{};
  w.b = b; w.h = h; w.n = p.len(b);
  w.r0 = tile * p.tile_rows;
  w.rows = min(p.tile_rows, p.R - w.r0);
  w.lim_min = w.last_of(p, 0);
  w.lim_max = w.last_of(p, w.rows - 1);
  const int seen = max(min(skip + many, (w.lim_max + kQ8Keys) / kQ8Keys) - skip, 0);
  w.chunk0 = skip + seen * warp / kQ8Warps;
  w.n_chunks = skip + seen * (warp + 1) / kQ8Warps - w.chunk0;
  return w;
}

// One piece: every warp walks its chunks, then the warps' results are merged.  Thread (row, column group) of the CTA is left
// with its row's running maximum, sum and CW columns of the unnormalised output.  HILO: P' enters the product as two
// fp16 parts.  All threads of the CTA; the rings are empty and shared memory is free for the next piece's tiles after a
// proxy fence and a barrier.
template <typename T, int D, int NT, bool HILO, int ST>
__device__ __forceinline__ void q8_piece(const Q8Params& p, const CUtensorMap& tm_k, const CUtensorMap& tm_v, const Q8Piece& w,
                                         uint8_t* gen, uint32_t base, int* nan_from, const Ctl& ctl,
                                         float (&acc)[Q8Smem<D, NT, ST>::kCW], float& mx, float& tot) {
  using SM = Q8Smem<D, NT, ST>;
  constexpr int ROWS = SM::kRows, CW = SM::kCW;
  constexpr int KS = D / 16;                   // k steps of k q^T
  constexpr int DT = D / 16;                   // 16-row blocks of o^T
  constexpr int KU = D / 64;                   // 16-byte units a lane reads per key row
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t bars = base + SM::kBars + warp * ST * 8;
  int lim[NT][2];                              // last position seen of this lane's columns: rows 8 nt + 2t, + 1
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) lim[nt][e] = w.last_of(p, 8 * nt + 2 * t + e);
  const uint32_t ring = base + warp * SM::kWarpRing;
  auto k_tile = [&](int s) { return ring + s * 2 * SM::kTile; };
  auto load = [&](int c) {                                         // lane 0
    const int s = (w.loaded + c) % ST, key0 = (w.chunk0 + c) * kQ8Keys;
    mbar_expect_tx(bars + 8 * s, 2 * SM::kTile);
    tma_load_head_tile(k_tile(s), &tm_k, bars + 8 * s, p.ki, 0, key0, w.h, w.b);
    tma_load_head_tile(k_tile(s) + SM::kTile, &tm_v, bars + 8 * s, p.vi, 0, key0, w.h, w.b);
  };
  if (lane == 0)
    for (int c = 0; c < min(ST, w.n_chunks); ++c) load(c);
  // scales of a chunk: two halves of 16 positions (the same block unless block is 16)
  auto scales_of = [&](int c, float (&ks)[2], float (&vs)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int key = (w.chunk0 + c) * kQ8Keys + 16 * i;
      const bool in = c < w.n_chunks && key <= w.lim_max;
      ks[i] = in ? *p.ks.at(w.b, key >> p.shift, w.h) : 1.f;
      vs[i] = in ? *p.vs.at(w.b, key >> p.shift, w.h) : 1.f;
    }
  };
  float ks_next[2], vs_next[2];
  scales_of(0, ks_next, vs_next);

  // ---- q as the B operand: fp16 times 2^(14 - exponent of the row's largest element).  Column g of k step 4 u + j holds
  // d = (KU t + u) 16 + 4 j + {0, 1} in register 0 and + {2, 3} in register 1
  uint32_t qb[NT][KS][2];
  float cq[NT][2];                             // scale * log2 e / row factor of this lane's columns
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = 8 * nt + g, rr = w.r0 + min(r, w.rows - 1);
    const T* src = static_cast<const T*>(p.q.ptr) + w.b * p.q.stride_b + static_cast<long long>(rr / p.G) * p.q.stride_s +
                   static_cast<long long>(w.h * p.G + rr % p.G) * p.q.stride_h + t * KU * 16;
    uint4 x[2 * KU];
#pragma unroll
    for (int i = 0; i < 2 * KU; ++i) x[i] = *reinterpret_cast<const uint4*>(src + i * 8);
    float f[KU * 16], amax = 0.f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 2 * KU; ++i) {
      const uint32_t xx[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 v = Io<T>::unpack2(xx[e]);
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
      const int e = min(max(static_cast<int>(__float_as_uint(amax) >> 23) - 127, -100), 127);
      up = exp2_int(14 - e);
      down = exp2_int(e - 14);
    }
    bad = ((__ballot_sync(0xffffffffu, bad) >> (g * 4)) & 0xfu) != 0u;
    // a row with an infinite or NaN element: every score is infinite or NaN, and so is its softmax NaN
    const float c = bad ? __uint_as_float(0x7fffffffu) : p.scale_log2 * down;
#pragma unroll
    for (int e = 0; e < 2; ++e) cq[nt][e] = __shfl_sync(0xffffffffu, c, (2 * t + e) * 4);
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const int d = (i >> 2) * 16 + (i & 3) * 4;
      qb[nt][i][0] = r < w.rows ? Io<__half>::pack2(f[d] * up, f[d + 1] * up) : 0u;
      qb[nt][i][1] = r < w.rows ? Io<__half>::pack2(f[d + 2] * up, f[d + 3] * up) : 0u;
    }
  }

  float oacc[NT][DT][4];
  float m_ref[NT][2], l_run[NT][2];
  float* sc[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) oacc[nt][i][j] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      m_ref[nt][e] = -INFINITY;
      l_run[nt][e] = 0.f;
      const int r = 8 * nt + 2 * t + e;
      sc[nt][e] = w.kept != nullptr && r < w.rows ? w.kept + r * w.kept_pitch - w.kept_from : nullptr;
    }
  }
  bool ok = true;

  for (int c = 0; c < w.n_chunks; ++c) {
    const int s = (w.loaded + c) % ST, key0 = (w.chunk0 + c) * kQ8Keys;
    float lv[2], vf[2];
    const float ks[2] = {ks_next[0], ks_next[1]};
#pragma unroll
    for (int i = 0; i < 2; ++i) v_scale_terms(vs_next[i], lv[i], vf[i]);
    scales_of(c + 1, ks_next, vs_next);
    const bool edge = key0 + kQ8Keys - 1 > w.lim_min;                // some row does not see some position of the chunk
    ok = mbar_wait(bars + 8 * s, ((w.loaded + c) / ST) & 1, ctl, KST_TIMEOUT_CONSUMER);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) break;
    // ---- s^T of two blocks of 16 positions; rows g, g + 8 of a block are its positions q8_key(g), 8 + q8_key(g)
    float st[2][NT][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 4; ++j) st[i][nt][j] = 0.f;
    }
#pragma unroll
    for (int u = 0; u < KU; ++u) {
      uint4 kk[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) kk[i] = lds128(k_tile(s) + q8_off<D>(8 * i + q8_key<D>(g), KU * t + u));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t lo = j == 0 ? kk[2 * i].x : j == 1 ? kk[2 * i].y : j == 2 ? kk[2 * i].z : kk[2 * i].w;
          const uint32_t hi = j == 0 ? kk[2 * i + 1].x : j == 1 ? kk[2 * i + 1].y : j == 2 ? kk[2 * i + 1].z : kk[2 * i + 1].w;
          const uint32_t a0 = e4m3x2_to_f16x2(lo), a1 = e4m3x2_to_f16x2(hi);
          const uint32_t a2 = e4m3x2_to_f16x2(lo >> 16), a3 = e4m3x2_to_f16x2(hi >> 16);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_f16(st[i][nt], a0, a1, a2, a3, qb[nt][4 * u + j][0], qb[nt][4 * u + j][1]);
        }
      }
    }
    // ---- t = acc * c * ks.  Accumulator (2 k + e): position 8 k + q8_key(g) of the block, column 2t + e
    bool raise = false;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float a = cq[nt][e] * ks[i], over = m_ref[nt][e] + kQ8Slack - lv[i];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int key = key0 + 16 * i + 8 * k + q8_key<D>(g);
            float x = st[i][nt][2 * k + e] * a;
            // whoever reads the kept scores knows which of them a row sees
            if (sc[nt][e] != nullptr) sc[nt][e][key] = x;
            if (edge && key > lim[nt][e]) x = -INFINITY;
            st[i][nt][2 * k + e] = x;
            raise = raise || x > over;
          }
        }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float al[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(fmaxf(st[0][nt][e], st[0][nt][2 + e]) + lv[0], fmaxf(st[1][nt][e], st[1][nt][2 + e]) + lv[1]);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          const float mn = fmaxf(m_ref[nt][e], mx);
          const float d = mn == -INFINITY ? 0.f : m_ref[nt][e] - mn;
          al[e] = ex2_approx(d);
          m_ref[nt][e] = mn;
          l_run[nt][e] = sum_moved(l_run[nt][e], d);
        }
#pragma unroll
        for (int i = 0; i < DT; ++i) {
          oacc[nt][i][0] *= al[0]; oacc[nt][i][1] *= al[1];
          oacc[nt][i][2] *= al[0]; oacc[nt][i][3] *= al[1];
        }
      }
    }
    // ---- E = 2^(t - m'), P' = E vs, transposed into the B operand of o^T += v^T P'^T
    uint32_t ph[2][NT][2], pl[2][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float use[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) use[e] = kQ8PBias + kQ8LBias - (m_ref[nt][e] == -INFINITY ? 0.f : m_ref[nt][e]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float a = ex2_approx(st[i][nt][2 * k] + use[0]), c2 = ex2_approx(st[i][nt][2 * k + 1] + use[1]);
          l_run[nt][0] += a;
          l_run[nt][1] += c2;
          a *= vf[i];
          c2 *= vf[i];
          const uint32_t hi = Io<__half>::pack2(a, c2);
          ph[i][nt][k] = transpose8(hi);
          if constexpr (HILO) {
            const float2 r = Io<__half>::unpack2(hi);
            pl[i][nt][k] = transpose8(Io<__half>::pack2(a - r.x, c2 - r.y));
          }
        }
      }
    }
    // ---- rows g, g + 8 of block j of o^T hold d = g * (D / 8) + 2 j, + 1
    const uint32_t vt = k_tile(s) + SM::kTile;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      constexpr int W = D / 32;                // 32-bit words a lane takes of a row: 4 or 2
      uint32_t v[4][W];                        // positions 2t, 2t + 1, 2t + 8, 2t + 9 of the block
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int rr = (2 * kk + (i >> 1)) * 8 + q8_key<D>(2 * t + (i & 1));
        if constexpr (D == 128) {
          const uint4 x = lds128(vt + q8_off<D>(rr, g));
          v[i][0] = x.x; v[i][1] = x.y; v[i][2] = x.z; v[i][3] = x.w;
        } else {
          const uint2 x = lds64(vt + q8_off<D>(rr, g >> 1) + (g & 1) * 8);
          v[i][0] = x.x; v[i][1] = x.y;
        }
        if (edge) {
          const int key = key0 + rr;
#pragma unroll
          for (int j = 0; j < W; ++j) {
            const uint32_t bad = nan_bytes(v[i][j]);
            if (bad != 0u) {
              v[i][j] &= ~bad;
              if (key <= w.lim_max)
                for (int e = 0; e < 4; ++e)
                  if ((bad >> (8 * e)) & 1u) atomicMin(&nan_from[g * (D / 8) + 4 * j + e], key);
            }
          }
        }
      }
#pragma unroll
      for (int j = 0; j < W; ++j) {
        // bytes of two positions side by side: (k, k + 1) pairs of d = 4 j + {0, 1}, {2, 3}
        const uint32_t x0 = __byte_perm(v[0][j], v[1][j], 0x5140), x1 = __byte_perm(v[0][j], v[1][j], 0x7362);
        const uint32_t y0 = __byte_perm(v[2][j], v[3][j], 0x5140), y1 = __byte_perm(v[2][j], v[3][j], 0x7362);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t x = e == 0 ? x0 : x1, y = e == 0 ? y0 : y1;
          const uint32_t a0 = e4m3x2_to_f16x2(x), a1 = e4m3x2_to_f16x2(x >> 16);
          const uint32_t a2 = e4m3x2_to_f16x2(y), a3 = e4m3x2_to_f16x2(y >> 16);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_f16(oacc[nt][2 * j + e], a0, a1, a2, a3, ph[kk][nt][0], ph[kk][nt][1]);
            if constexpr (HILO) mma_f16(oacc[nt][2 * j + e], a0, a1, a2, a3, pl[kk][nt][0], pl[kk][nt][1]);
          }
        }
      }
    }
    __syncwarp();                              // every lane has read stage s
    if (lane == 0 && c + ST < w.n_chunks) load(c + ST);
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l_run[nt][e] += __shfl_xor_sync(0xffffffffu, l_run[nt][e], o);
  __syncthreads();                             // the partial results take the rings' place
  if (*ctl.abort) {
    // a wait ran out: give copies in flight time to land before shared memory is put to another use
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  // ---- the warps' partial results -> shared memory [warp][row][D | max, sum], merged in fixed order
  float* part = reinterpret_cast<float*>(gen);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float* dst = part + (warp * ROWS + 8 * nt + 2 * t + e) * SM::kRow;
#pragma unroll
      for (int j = 0; j < DT; j += 2)
        *reinterpret_cast<float4*>(dst + g * (D / 8) + 2 * j) =
            make_float4(oacc[nt][j][e], oacc[nt][j][2 + e], oacc[nt][j + 1][e], oacc[nt][j + 1][2 + e]);
      if (g == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(m_ref[nt][e], l_run[nt][e]);
    }
  __syncthreads();
  const int row = threadIdx.x / SM::kTPR, c0 = (threadIdx.x % SM::kTPR) * CW;
  mx = -INFINITY;
  tot = 0.f;
#pragma unroll
  for (int c = 0; c < CW; ++c) acc[c] = 0.f;
#pragma unroll
  for (int i = 0; i < kQ8Warps; ++i) mx = fmaxf(mx, part[(i * ROWS + row) * SM::kRow + D]);
#pragma unroll
  for (int i = 0; i < kQ8Warps; ++i) {
    const float* src = part + (i * ROWS + row) * SM::kRow;
    if (src[D + 1] == 0.f) continue;                               // saw no position of this row
    const float f = ex2_approx(src[D] - mx);
    tot += sum_moved(src[D + 1], src[D] - mx);
#pragma unroll
    for (int c = 0; c < CW; ++c) acc[c] = fmaf(f, src[c0 + c], acc[c]);
  }
  const int last = w.last_of(p, row);
#pragma unroll
  for (int c = 0; c < CW; ++c)
    if (nan_from[c0 + c] <= last) acc[c] = __uint_as_float(0x7fffffffu);
}

// barriers and the table of NaN columns; then the wait for the launch before this one.  Returns whether an earlier kernel gave up.
template <int D, int NT, int ST>
__device__ __forceinline__ bool q8_begin(const Q8Params& p, const CUtensorMap& tm_k, const CUtensorMap& tm_v, uint32_t base,
                                         int* nan_from, int* s_abort) {
  if ((threadIdx.x & 31) == 0) {
    for (int s = 0; s < ST; ++s) mbar_init(base + Q8Smem<D, NT, ST>::kBars + ((threadIdx.x >> 5) * ST + s) * 8, 1);
    fence_mbar_init();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (threadIdx.x == 0) *s_abort = 0;
  for (int i = threadIdx.x; i < D; i += kQ8Threads) nan_from[i] = 0x7fffffff;
  __syncthreads();
  griddep_wait();                              // q, the codes and the lengths may come from the launch before
  griddep_launch();
  return *reinterpret_cast<volatile int*>(p.status) != 0;
}

// Long caches: each CTA takes its share of all chunks, a piece of a unit after the other.
template <typename T, int D, int NT, bool HILO, int ST>
__global__ void __launch_bounds__(kQ8Threads)
attn_q8_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
               const __grid_constant__ Q8Params p) {
  using SM = Q8Smem<D, NT, ST>;
  constexpr int ROWS = SM::kRows, CW = SM::kCW;
  extern __shared__ uint8_t q8_smem_raw[];
  __shared__ int nan_from[D];                  // first position whose v code of this column is NaN, in edge chunks
  __shared__ int s_abort;
  const uint32_t base = (smem_u32(q8_smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = q8_smem_raw + (base - smem_u32(q8_smem_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Ctl ctl{p.status, &s_abort};
  if (q8_begin<D, NT, ST>(p, tm_k, tm_v, base, nan_from, &s_abort)) return;

  // ---- this CTA's share: chunks [at, end) of all, beginning `skip` chunks into unit (b, h, tile)
  const int cta = static_cast<int>(blockIdx.x);
  int b, h, tile, skip = 0, left;              // left: chunks still to do
  unsigned share = 1u;
  if (p.ctas == 0) {
    tile = cta % p.tiles;
    h = cta / p.tiles % p.Hkv;
    b = cta / p.tiles / p.Hkv;
    left = chunks_of(p.len(b));
  } else {
    const int all = chunks_before(p, 0).y;
    share = share_of(p, all);
    const unsigned per = p.Hkv * p.tiles, end = static_cast<unsigned>(all) * per;
    unsigned at = cta * share;
    if (at >= end) return;
    left = static_cast<int>(min(end - at, share));
    // the sequence the share begins in: running sums over 32 sequences at a time
    b = p.B;
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      const unsigned c = b0 + lane < p.B ? chunks_of(p.len(b0 + lane)) * per : 0u;
      unsigned incl = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned v = __shfl_up_sync(0xffffffffu, incl, o);
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
    if (b == p.B) return;                      // lengths that change under the kernel: nothing sensible to do, nothing unsafe done
    const unsigned mine = chunks_of(p.len(b)), u = min(at / mine, per - 1);
    skip = static_cast<int>(at - u * mine);
    h = static_cast<int>(u / p.tiles);
    tile = static_cast<int>(u % p.tiles);
  }
  for (int loaded = 0;;) {
    const int bh = b * p.Hkv + h, unit = bh * p.tiles + tile;
    const int total = chunks_of(p.len(b)), many = max(min(total - skip, left), 1);
    Q8Piece w = piece_of(p, b, h, tile, skip, many, warp);
    w.loaded = loaded;
    if (p.scores != nullptr) {
      w.kept = p.scores + (static_cast<long long>(bh) * p.R + w.r0) * p.pitch;
      w.kept_pitch = p.pitch;
    }
    float acc[CW], mx, tot;
    q8_piece<T, D, NT, HILO, ST>(p, tm_k, tm_v, w, gen, base, nan_from, ctl, acc, mx, tot);
    if (s_abort) return;
    const int row = threadIdx.x / SM::kTPR, c0 = (threadIdx.x % SM::kTPR) * CW;
    if (row < w.rows) {
      const long long at = static_cast<long long>(unit + (p.ctas > 0 ? cta : 0)) * ROWS + row;
      if (many < total) {
#pragma unroll
        for (int c = 0; c < CW; c += 4)
          *reinterpret_cast<float4*>(p.part_o + at * D + c0 + c) = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
      } else {
        q8_store_row<T, CW>(p, b, h, w.r0 + row, c0, acc, mx, tot);
      }
      if (c0 == 0 && p.part_ml != nullptr) p.part_ml[at] = make_float2(mx, tot);
    }
    if (skip == 0 && threadIdx.x == 0 && p.pieces != nullptr) {    // the unit begins in this share, with `left` chunks of it to go
      const int rest = total - left;                               // chunks that fall to the CTAs behind
      p.pieces[unit] = make_int2(p.ctas > 0 ? cta : 0, (p.ctas > 0 ? cta : 0) + (rest > 0 ? (rest + static_cast<int>(share) - 1) / static_cast<int>(share) : 0));
    }
    // ---- the next piece of the share begins with the next unit
    left -= many;
    if (left <= 0) return;
    loaded += w.n_chunks;
    skip = 0;
    if (++tile == p.tiles) {
      tile = 0;
      if (++h == p.Hkv) {
        h = 0;
        if (++b == p.B) return;
      }
    }
    fence_proxy_async_smem();                  // the partial results gave way to the next piece's tiles
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += kQ8Threads) nan_from[i] = 0x7fffffff;
    __syncthreads();
  }
}

// Short caches (at most kQ8Keep chunks a warp): a cluster of CTAs per unit, which meet in shared memory, so that one launch
// does everything, the weights too: each warp keeps its scores on chip until the rows' log-sum-exps are known.
template <typename T, int D, int NT, bool HILO, int ST>
__global__ void __launch_bounds__(kQ8Threads)
attn_q8_cluster_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                       const __grid_constant__ Q8Params p, int cluster) {
  using SM = Q8Smem<D, NT, ST>;
  constexpr int ROWS = SM::kRows, CW = SM::kCW;
  extern __shared__ uint8_t q8_smem_raw[];
  __shared__ int nan_from[D];
  __shared__ int s_abort;
  __shared__ float lse_of[ROWS];
  const uint32_t base = (smem_u32(q8_smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = q8_smem_raw + (base - smem_u32(q8_smem_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Ctl ctl{p.status, &s_abort};
  // no CTA leaves before the cluster's last barrier; one that must not work writes nothing
  const bool dead = q8_begin<D, NT, ST>(p, tm_k, tm_v, base, nan_from, &s_abort);
  const int rank = static_cast<int>(cluster_ctarank()), unit = static_cast<int>(blockIdx.x) / cluster;
  const int tile = unit % p.tiles, h = unit / p.tiles % p.Hkv, b = unit / p.tiles / p.Hkv;
  const int total = chunks_of(p.len(b)), skip = total * rank / cluster;
  Q8Piece w = piece_of(p, b, h, tile, skip, total * (rank + 1) / cluster - skip, warp);
  if (dead) w.n_chunks = 0;
  if (p.weight != nullptr) {
    w.kept = reinterpret_cast<float*>(gen + SM::kKept) + warp * ROWS * SM::kKeptPitch;
    w.kept_pitch = SM::kKeptPitch;
    w.kept_from = w.chunk0 * kQ8Keys;
  }
  float acc[CW], mx, tot;
  q8_piece<T, D, NT, HILO, ST>(p, tm_k, tm_v, w, gen, base, nan_from, ctl, acc, mx, tot);
  const bool write = !dead && s_abort == 0;
  float* mine = reinterpret_cast<float*>(gen + SM::kMine);         // [ROWS][kRow], behind the warps' results
  {
    const int row = threadIdx.x / SM::kTPR, c0 = (threadIdx.x % SM::kTPR) * CW;
#pragma unroll
    for (int c = 0; c < CW; c += 4)
      *reinterpret_cast<float4*>(mine + row * SM::kRow + c0 + c) = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
    if (c0 == 0) *reinterpret_cast<float2*>(mine + row * SM::kRow + D) = make_float2(mx, tot);
  }
  if (cluster > 1) cluster_sync_all(); else __syncthreads();
  const uint32_t mine_s = base + SM::kMine;
  // ---- rows rank, rank + cluster, ... : two columns a thread, the ranks' results in ascending order
  auto ml_of = [&](int r, int i) { return ld_cluster_f2(map_to_rank(mine_s + (r * SM::kRow + D) * 4, static_cast<uint32_t>(i))); };
  for (int r = rank + cluster * (static_cast<int>(threadIdx.x) / (D / 2)); r < w.rows; r += cluster * (kQ8Threads / (D / 2))) {
    const int d = (threadIdx.x % (D / 2)) * 2;
    float2 ml[kQ8MaxCluster], v[kQ8MaxCluster];
#pragma unroll
    for (int i = 0; i < kQ8MaxCluster; ++i)
      if (i < cluster) {
        ml[i] = ml_of(r, i);
        v[i] = ld_cluster_f2(map_to_rank(mine_s + (r * SM::kRow + d) * 4, static_cast<uint32_t>(i)));
      }
    float m = -INFINITY, sum = 0.f, o[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kQ8MaxCluster; ++i)
      if (i < cluster) m = fmaxf(m, ml[i].x);
#pragma unroll
    for (int i = 0; i < kQ8MaxCluster; ++i)
      if (i < cluster && ml[i].y != 0.f) {
        const float f = ex2_approx(ml[i].x - m);
        sum += sum_moved(ml[i].y, ml[i].x - m);
        o[0] = fmaf(f, v[i].x, o[0]);
        o[1] = fmaf(f, v[i].y, o[1]);
      }
    if (write) q8_store_row<T, 2>(p, b, h, w.r0 + r, d, o, m, sum);
  }
  if (p.weight != nullptr) {
    for (int r = threadIdx.x; r < w.rows; r += kQ8Threads) {
      float m = -INFINITY, sum = 0.f;
      for (int i = 0; i < cluster; ++i) m = fmaxf(m, ml_of(r, i).x);
      for (int i = 0; i < cluster; ++i) {
        const float2 ml = ml_of(r, i);
        if (ml.y != 0.f) sum += sum_moved(ml.y, ml.x - m);
      }
      lse_of[r] = m - (kQ8PBias + kQ8LBias) + log2f(sum);
    }
    __syncthreads();
    // only launched with one row tile per (b, kv head): the rows of the tile are all that see a position
    float* out = p.weight + b * p.w_sb + h * p.w_sh;
    for (int i = lane; i < w.n_chunks * kQ8Keys; i += 32) {
      const int key = w.kept_from + i;
      if (key >= w.n) break;
      const int first = p.causal ? max(key - (w.n - p.M), 0) * p.G : 0;
      float sum = 0.f;
      for (int r = first; r < w.rows; ++r) sum += ex2_approx(w.kept[r * SM::kKeptPitch + i] - lse_of[r]);
      if (write) out[key] = p.weight_add ? out[key] + sum : sum;
    }
  }
  if (cluster > 1) cluster_sync_all();                             // no CTA leaves while its results may be read
}

// Merge of the pieces, and weights of the positions.  CTAs [0, merge_ctas): join_rows rows of a unit each; the rest: positions
// of a (b, kv head), four at a time a thread, rows in ascending order.
constexpr int kQ8JoinThreads = 256;
constexpr int kQ8JoinWarps = kQ8JoinThreads / 32;
// Positions of a weight CTA: with few rows per kv head its threads are for positions, with more they share the rows.  From 256
// rows on 32 positions, so that the rows are shared 32 ways: 568 rows of one head of 64 and 8192 positions 36 us the call (p in
// one part here; two: 37), 55 with 128 positions, 223 with all rows in a thread; 1136 rows, 8192 positions 54, 94.  Below, every CTA's own pass over the
// rows' sums weighs more (64 rows of 8 x 8 heads, 4096 positions: 133, 103), so there 128, unless those CTAs are fewer than the
// SMs (142 rows of one head, 2000 positions: 21.2, 26.1); 32 rows and fewer gain nothing there either (20 rows of 8 heads,
// 2000 positions: 24.1, 21.5).
// The border between the two forms: 16 rows of 8 heads, 8192 positions 35.5 us with the threads for positions, 31.5 shared; eight such
// sequences 75.3, 82.2; 12 rows of 2 heads, 40000 positions 28.9, 55.1; 20 and 32 rows of 8 heads, 8192 positions 41.7, 33.4 and 51.2, 35.3.
constexpr int kQ8FewRows = 16, kQ8JoinKeys = 8 * kQ8JoinThreads, kQ8JoinKeysRows = 128, kQ8JoinKeysShort = 32, kQ8RowsShort = 256;
// maximum and sum of a row over its pieces by one warp; at: the row in the first piece's slot
__device__ __forceinline__ float2 join_ml(const Q8Params& p, long long at, int here, int lane) {
  float2 mine = make_float2(-INFINITY, 0.f);   // a lane's pieces lane, lane + 32, ...
  for (int s = lane; s < here; s += 32) {
    const float2 ml = p.part_ml[at + static_cast<long long>(s) * p.tile_rows];
    if (ml.y == 0.f) continue;
    const float m = fmaxf(mine.x, ml.x);
    mine.y = (mine.y == 0.f ? 0.f : sum_moved(mine.y, mine.x - m)) + sum_moved(ml.y, ml.x - m);
    mine.x = m;
  }
  float m = mine.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float tot = mine.y == 0.f ? 0.f : sum_moved(mine.y, mine.x - m);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) tot += __shfl_xor_sync(0xffffffffu, tot, o);
  return make_float2(m, tot);
}

template <typename T, int D>
__global__ void __launch_bounds__(kQ8JoinThreads)
attn_q8_join_kernel(const __grid_constant__ Q8Params p, int merge_ctas, int key_tiles) {
  extern __shared__ float q8_join[];           // weight CTAs: [R] log-sum-exps
  constexpr int GROUPS = kQ8JoinThreads / (D / 2);
  __shared__ float2 all[GROUPS], part[GROUPS][D / 2];
  griddep_wait();
  griddep_launch();
  if (*reinterpret_cast<volatile int*>(p.status) != 0) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (static_cast<int>(blockIdx.x) < merge_ctas) {
    const int per_unit = p.tile_rows / p.join_rows;
    int unit = static_cast<int>(blockIdx.x) / per_unit;
    const int r_first = static_cast<int>(blockIdx.x) % per_unit * p.join_rows;
    if (p.join_pairs > 0) {
      const int u = p.join_first + unit / 2, t = 2 * (p.join_pairs - 1 - u / (p.B * p.Hkv)) + unit % 2;
      if (t >= p.tiles) return;
      unit = u % (p.B * p.Hkv) * p.tiles + t;
    }
    const int tile = unit % p.tiles, bh = unit / p.tiles, rows = min(p.tile_rows, p.R - tile * p.tile_rows);
    if (r_first >= rows) return;
    const int2 on = p.pieces[unit];
    const int here = on.y - on.x + 1;
    if (here == 1) return;                     // written by the one piece itself
    const long long at = static_cast<long long>(unit + on.x) * p.tile_rows + r_first;
    if (warp < p.join_rows && r_first + warp < rows) {
      const float2 ml = join_ml(p, at + warp, here, lane);
      if (lane == 0) all[warp] = ml;
    }
    __syncthreads();
    // a group of D / 2 threads, two columns each, has a row of its own, or all groups share one row's pieces
    const bool share = p.join_rows == 1;
    const int g = tid / (D / 2), d = (tid % (D / 2)) * 2, r = share ? 0 : g, step = share ? GROUPS : 1;
    const bool there = r_first + r < rows;
    const float2 ml = all[r];
    float acc[2] = {0.f, 0.f};
    if (there) {
#pragma unroll 8
      for (int s = share ? g : 0; s < here; s += step) {
        const long long row = at + r + static_cast<long long>(s) * p.tile_rows;
        const float2 x = p.part_ml[row];
        const float2 v = *reinterpret_cast<const float2*>(p.part_o + row * D + d);
        const float w = x.y == 0.f ? 0.f : ex2_approx(x.x - ml.x);
        if (x.y != 0.f) {                      // a piece that saw nothing has nothing to weigh
          acc[0] = fmaf(w, v.x, acc[0]);
          acc[1] = fmaf(w, v.y, acc[1]);
        }
      }
    }
    if (share) {
      part[g][tid % (D / 2)] = make_float2(acc[0], acc[1]);
      __syncthreads();
      if (g != 0) return;
#pragma unroll
      for (int i = 1; i < GROUPS; ++i) {
        acc[0] += part[i][tid].x;
        acc[1] += part[i][tid].y;
      }
    }
    if (there) q8_store_row<T, 2>(p, bh / p.Hkv, bh % p.Hkv, tile * p.tile_rows + r_first + r, d, acc, ml.x, ml.y);
    return;
  }
  const int id = static_cast<int>(blockIdx.x) - merge_ctas;
  const int bh = id / key_tiles, b = bh / p.Hkv, h = bh % p.Hkv;
  const int n = p.len(b);
  const int keys = p.join_keys, key0 = (id % key_tiles) * keys;
  if (key0 >= n) return;
  auto ml_at = [&](int r, int& here) {
    const int unit = bh * p.tiles + r / p.tile_rows;
    const int2 on = p.pieces[unit];
    here = on.y - on.x + 1;
    return static_cast<long long>(unit + on.x) * p.tile_rows + r % p.tile_rows;
  };
  if (p.R <= kQ8FewRows) {                     // a warp for each row: its pieces side by side
    for (int r = warp; r < p.R; r += kQ8JoinWarps) {
      int here;
      const long long at = ml_at(r, here);
      const float2 ml = join_ml(p, at, here, lane);
      if (lane == 0) q8_join[r] = ml.x - (kQ8PBias + kQ8LBias) + log2f(ml.y);
    }
  } else {                                     // a thread for each row: rows side by side
    for (int r = tid; r < p.R; r += kQ8JoinThreads) {
      int here;
      const long long at = ml_at(r, here);
      float m = -INFINITY, l = 0.f;
#pragma unroll 4
      for (int s = 0; s < here; ++s) {
        const float2 ml = p.part_ml[at + static_cast<long long>(s) * p.tile_rows];
        const float mn = fmaxf(m, ml.x);
        if (ml.y != 0.f) {
          l = (l == 0.f ? 0.f : sum_moved(l, m - mn)) + sum_moved(ml.y, ml.x - mn);
          m = mn;
        }
      }
      q8_join[r] = m - (kQ8PBias + kQ8LBias) + log2f(l);
    }
  }
  __syncthreads();
  // causal: position j is seen by the queries i >= j - (n - M).  What a row kept of positions that it does not see is not
  // taken, whatever it is.
  auto sum_rows = [&](int key, int r0, int step, float (&acc)[4]) {
    const int first = p.causal ? max(key - (n - p.M), 0) * p.G : 0;
    const float* src = p.scores + static_cast<long long>(bh) * p.R * p.pitch + key;
    const bool edge = key + 3 > last_seen(p, n, first);
#pragma unroll 8
    for (int r = first + r0; r < p.R; r += step) {
      const float4 x = *reinterpret_cast<const float4*>(src + r * p.pitch);
      const float l = q8_join[r];
      const int seen = edge ? last_seen(p, n, r) - key : 3;
      acc[0] += ex2_approx(x.x - l);
      if (seen >= 1) acc[1] += ex2_approx(x.y - l);
      if (seen >= 2) acc[2] += ex2_approx(x.z - l);
      if (seen >= 3) acc[3] += ex2_approx(x.w - l);
    }
  };
  auto put = [&](int key, const float (&acc)[4]) {
    float* w = p.weight + b * p.w_sb + h * p.w_sh + key;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (key + e < n) w[e] = p.weight_add ? w[e] + acc[e] : acc[e];
  };
  if (p.R <= kQ8FewRows) {
    for (int key = key0 + 4 * tid; key < n && key < key0 + keys; key += 4 * kQ8JoinThreads) {
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      sum_rows(key, 0, 1, acc);
      put(key, acc);
    }
    return;
  }
  // many rows: LANES x 4 positions, the rows dealt out to the groups of as many lanes, which meet in fixed order
  __shared__ float4 sums[kQ8JoinThreads];
  auto weigh = [&](auto lanes) {
    constexpr int LANES = decltype(lanes)::value, N = kQ8JoinThreads / LANES;
    const int key = key0 + 4 * (tid % LANES);
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    if (key < n) sum_rows(key, tid / LANES, N, acc);
    sums[tid] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    __syncthreads();
    if (tid >= LANES || key >= n) return;
#pragma unroll
    for (int i = 1; i < N; ++i) {
      const float4 x = sums[i * LANES + tid];
      acc[0] += x.x; acc[1] += x.y; acc[2] += x.z; acc[3] += x.w;
    }
    put(key, acc);
  };
  if (keys == kQ8JoinKeysShort) weigh(std::integral_constant<int, kQ8JoinKeysShort / 4>{});
  else weigh(std::integral_constant<int, kQ8JoinKeysRows / 4>{});
}

struct Q8Plan {
  int tiles, tile_rows, stages, ctas, cluster;         // cluster > 0: one launch of clusters, no scratch
  long long units;
  size_t ml_off, o_off, piece_off, score_off, total;
  long long pitch;
};

// Short caches: clusters of CTAs, when kQ8Keep chunks a warp suffice with as many CTAs per unit (a power of two) as fill one
// round of resident CTAs (with weights: if one row tile holds all rows).  Else the chunks are dealt out to one round
// of resident CTAs, fewer where that would leave a warp without a chunk.
Q8Plan plan_of(const TrnAttnQ8Args& a, int sm_count, bool divide) {
  Q8Plan w{};
  const int R = a.M * (a.Hq / a.Hkv);
  w.tile_rows = 8;
  while (w.tile_rows < R && w.tile_rows < 8 * q8_max_tiles(a.D)) w.tile_rows *= 2;
  w.tiles = (R + w.tile_rows - 1) / w.tile_rows;
  w.units = static_cast<long long>(a.B) * a.Hkv * w.tiles;
  const int longest = a.kv_len != nullptr ? a.cache.S : min(max(a.kv_len_all, 1), a.cache.S);
  const int unit_chunks = (longest - 1) / kQ8Keys + 1;
  w.stages = q8_stages(a.D, w.tile_rows, w.units, sm_count);
  const long long round = static_cast<long long>(sm_count) * q8_ctas(a.D, w.tile_rows, w.stages);
  int cluster = 1;
  while (cluster < kQ8MaxCluster && 2 * cluster * w.units <= 3LL * sm_count && 2 * cluster * kQ8Warps <= unit_chunks + kQ8Warps - 1) cluster *= 2;
  if (unit_chunks <= kQ8Keep * kQ8Warps * cluster && (a.weight == nullptr || w.tiles == 1)) {
    w.cluster = cluster;
    return w;
  }
  const long long chunks = w.units * unit_chunks;
  if (chunks > 0x3fffffffLL) divide = false;             // chunk numbers stay in 32 bits
  w.ctas = divide ? static_cast<int>(min((chunks + kQ8Warps - 1) / kQ8Warps, round)) : 0;
  w.pitch = (a.cache.S + 31LL) / 32 * 32;
  const size_t slots = static_cast<size_t>(w.units + w.ctas) * w.tile_rows;
  size_t off = 0;
  w.ml_off = off;
  off += up256(slots * sizeof(float2));
  w.o_off = off;
  if (divide) off += up256(slots * a.D * sizeof(float));
  w.piece_off = off;
  off += up256(static_cast<size_t>(w.units) * sizeof(int2));
  w.score_off = off;
  if (a.weight != nullptr) off += up256(static_cast<size_t>(a.B) * a.Hkv * R * w.pitch * sizeof(float));
  w.total = divide || a.weight != nullptr ? off : 0;
  return w;
}

template <typename T, int D, int NT, bool HILO>
int launch_cluster(const TrnAttnQ8Args& a, const Q8Plan& w, const CUtensorMap& tm_k, const CUtensorMap& tm_v, const Q8Params& p,
                   cudaStream_t st, const DeviceState& ds) {
  using SM = Q8Smem<D, NT, 2>;
  auto kern = attn_q8_cluster_kernel<T, D, NT, HILO, 2>;
  const int rc = ensure_dyn_smem(reinterpret_cast<const void*>(kern), SM::kTotalKept, ds.device);
  if (rc != TRN_OK) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(w.units * w.cluster), 1, 1);
  cfg.blockDim = dim3(kQ8Threads, 1, 1);
  cfg.dynamicSmemBytes = a.weight != nullptr ? SM::kTotalKept : SM::kTotal;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(w.cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  TRN_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, tm_k, tm_v, p, w.cluster));
  return TRN_OK;
}

template <typename T, int D, int NT, int ST, bool HILO>
int launch_parts(const TrnAttnQ8Args& a, const Q8Plan& w, cudaStream_t st, const DeviceState& ds) {
  using SM = Q8Smem<D, NT, ST>;
  Q8Params p = q8_params(a, ds);
  CUtensorMap tm_k, tm_v;
  int rc = make_code_tmap(&tm_k, &p.ki, a.cache.k, a.cache.S, a.Hkv, a.B, D, kQ8Keys);
  if (rc == TRN_OK) rc = make_code_tmap(&tm_v, &p.vi, a.cache.v, a.cache.S, a.Hkv, a.B, D, kQ8Keys);
  if (rc != TRN_OK) return rc;
  p.tiles = w.tiles; p.tile_rows = w.tile_rows; p.ctas = w.ctas;
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  if (w.total > 0) {
    p.part_ml = reinterpret_cast<float2*>(ws + w.ml_off);
    p.pieces = reinterpret_cast<int2*>(ws + w.piece_off);
    if (w.ctas > 0) p.part_o = reinterpret_cast<float*>(ws + w.o_off);
    if (a.weight != nullptr) p.scores = reinterpret_cast<float*>(ws + w.score_off);
  }
  p.pitch = w.pitch;
  if (w.units * max(w.cluster, 1) + w.ctas > 0x7fffffffLL) return TRN_E_SHAPE;
  if (w.cluster > 0) return launch_cluster<T, D, NT, HILO>(a, w, tm_k, tm_v, p, st, ds);
  auto kern = attn_q8_kernel<T, D, NT, HILO, ST>;
  rc = ensure_dyn_smem(reinterpret_cast<const void*>(kern), SM::kTotal, ds.device);
  if (rc != TRN_OK) return rc;
  const unsigned grid = static_cast<unsigned>(w.ctas > 0 ? w.ctas : w.units);
  TRN_CUDA_TRY(launch_pdl(kern, dim3(grid), dim3(kQ8Threads), SM::kTotal, st, tm_k, tm_v, p));
  if (w.ctas > 0 || a.weight != nullptr) return launch_q8_join(p, a, w.ctas > 0, st);
  return TRN_OK;
}

template <typename T, int D, int NT, int ST>
int launch_tiles(const TrnAttnQ8Args& a, const Q8Plan& w, cudaStream_t st, const DeviceState& ds) {
  return a.single_p != 0 ? launch_parts<T, D, NT, ST, false>(a, w, st, ds) : launch_parts<T, D, NT, ST, true>(a, w, st, ds);
}

template <typename T, int D>
int launch_typed(const TrnAttnQ8Args& a, cudaStream_t st, const DeviceState& ds) {
  const Q8Plan w = plan_of(a, kAttnNominalSMs, a.workspace != nullptr);
  if constexpr (D == 128) {
    if (w.tile_rows == 16) return launch_tiles<T, D, 2, 3>(a, w, st, ds);
    return w.stages == 3 ? launch_tiles<T, D, 1, 3>(a, w, st, ds) : launch_tiles<T, D, 1, 2>(a, w, st, ds);
  } else {
    if (w.tile_rows == 8) return launch_tiles<T, D, 1, 2>(a, w, st, ds);
    if (w.tile_rows == 16) return launch_tiles<T, D, 2, 2>(a, w, st, ds);
    return launch_tiles<T, D, 4, 2>(a, w, st, ds);
  }
}

template <typename T, int D>
int launch_join(const Q8Params& p, const TrnAttnQ8Args& a, bool merge, cudaStream_t st) {
  const long long bh = static_cast<long long>(a.B) * a.Hkv;
  const long long units = p.join_pairs > 0 ? 2 * (bh * p.join_pairs - p.join_first) : bh * p.tiles;
  // Few units lie on many CTAs each: then a CTA merges one row, its threads sharing the pieces
  Q8Params jp = p;
  jp.join_rows = p.ctas >= 4 * bh * p.tiles ? 1 : kQ8JoinThreads / (D / 2);
  const long long merge_ctas = merge ? units * (p.tile_rows / jp.join_rows) : 0;
  const int longest = a.kv_len != nullptr ? a.cache.S : min(max(a.kv_len_all, 0), a.cache.S);
  jp.join_keys = p.R <= kQ8FewRows ? kQ8JoinKeys : kQ8JoinKeysRows;
  if (p.R >= kQ8RowsShort || (p.R > 32 && bh * ((longest + kQ8JoinKeysRows - 1) / kQ8JoinKeysRows) <= kAttnNominalSMs))
    jp.join_keys = kQ8JoinKeysShort;
  const int keys = jp.join_keys;
  const int key_tiles = a.weight != nullptr ? (longest + keys - 1) / keys : 0;
  const long long grid = merge_ctas + static_cast<long long>(a.B) * a.Hkv * key_tiles;
  if (grid > 0x7fffffffLL) return TRN_E_SHAPE;
  if (grid > 0)
    TRN_CUDA_TRY(launch_pdl(attn_q8_join_kernel<T, D>, dim3(static_cast<unsigned>(grid)), dim3(kQ8JoinThreads),
                            a.weight != nullptr ? p.R * sizeof(float) : 0, st, jp, static_cast<int>(merge_ctas), max(key_tiles, 1)));
  return TRN_OK;
}

constexpr int kQ8MaxWeightQueries = 16;
constexpr int kQ8MaxWeightRows = 8192;         // their log-sum-exps lie in 32 KB of shared memory

}  // namespace

int launch_q8_join(const Q8Params& p, const TrnAttnQ8Args& a, bool merge, cudaStream_t st) {
  if (a.dtype == TRN_BF16)
    return a.D == 128 ? launch_join<__nv_bfloat16, 128>(p, a, merge, st) : launch_join<__nv_bfloat16, 64>(p, a, merge, st);
  return a.D == 128 ? launch_join<__half, 128>(p, a, merge, st) : launch_join<__half, 64>(p, a, merge, st);
}

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
  // scratch: needed where weights are summed from kept scores, else optional; what is given has to be right
  const bool tc = attn_q8_tc_applies(a);
  const size_t need = tc ? attn_q8_tc_workspace(a) : plan_of(a, kAttnNominalSMs, a.workspace != nullptr).total;
  if (a.workspace != nullptr && ((reinterpret_cast<uintptr_t>(a.workspace) & 255u) != 0 || a.workspace_bytes < need)) return TRN_E_WORKSPACE;
  if (a.workspace == nullptr && !tc && need > 0) return TRN_E_WORKSPACE;
  return TRN_OK;
}

int launch_attention_q8(const TrnAttnQ8Args& a, cudaStream_t st, const DeviceState& ds) {
  if (attn_q8_tc_applies(a)) return launch_attn_q8_tc(a, st, ds);
  if (a.dtype == TRN_BF16)
    return a.D == 128 ? launch_typed<__nv_bfloat16, 128>(a, st, ds) : launch_typed<__nv_bfloat16, 64>(a, st, ds);
  return a.D == 128 ? launch_typed<__half, 128>(a, st, ds) : launch_typed<__half, 64>(a, st, ds);
}

size_t attention_q8_workspace(const TrnAttnQ8Args& a) {
  if (a.B <= 0 || a.M <= 0 || a.Hq <= 0 || a.Hkv <= 0 || a.Hq % a.Hkv != 0 || a.cache.S <= 0 || (a.D != 64 && a.D != 128)) return 0;
  TrnAttnQ8Args full = a;                      // whatever the sequences hold when the call comes
  full.kv_len = nullptr;
  full.kv_len_all = a.cache.S;
  return attn_q8_tc_applies(full) ? attn_q8_tc_workspace(full) : plan_of(full, kAttnNominalSMs, true).total;
}

}  // namespace trn
