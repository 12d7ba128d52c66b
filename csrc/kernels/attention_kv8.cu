// Paged attention over the 8-bit KV arena (kv8.cuh) with few query rows per sequence: one token
// per sequence (decode), or tiles of a few rows (verify chunks, short chunks).
//
// The rows of a tile times the G query heads of a KV head are the columns of one product:
//   S^T (16 tokens x 8 columns)  = K_page (16 x 128)   . Q^T      mma.m16n8k16, fp16, fp32 sums
//   O^T (16 dims   x 8 columns) += V_page^T (16 x 16)  . P^T
// With the tokens on the 16-row side a page costs 16 MMAs for 8 columns; with the columns on that
// side it would cost 32 and, at G = 4, leave three quarters of their rows empty.
// e4m3 -> fp16 is exact (one conversion for two codes), q is brought into fp16 by a power of two
// per column (bf16 has 8 significant bits, fp16 has 11; what falls below 2^-38 of the column's
// largest element is lost), so S carries only the rounding of fp32 sums. The scales stay outside
// the products: a token's K scale multiplies its scores, its V scale enters the exponent of P.
//
// Softmax without a maximum per page: z = scores in log2 units, w = z + log2(V scale). A column
// keeps a base m for z and a base bo for w that move only when a page has a z or w more than 8
// above them, so a page costs one vote instead of six shuffles and 32 multiplications. The two
// bases keep p = 2^(z-m) (summed in fp32) and P = 2^(w-bo+7) <= 2^15 (fp16, what the product
// needs) in range whatever the tokens' scales are.
//
// Work is cut by pages, not by sequences: the pages of every (sequence, KV head, column group) are
// laid end to end, a segment counting kSegCost pages more for its start and join, and each CTA takes
// an equal run of them, whatever the lengths are (all CTAs resident). A segment that lies within one
// CTA's run goes straight to the output; a CTA has at most two pieces of segments (its first and its
// last) that go to the workspace, and a second kernel joins them in the order of the CTAs, so results
// do not depend on timing. A few segments of few pages, of 256 items at most, are not cut (four sequences of
// 200 tokens: 7.1 us instead of 12.5), and when no block table is wider than kKv8WholePages, none is and there is no second
// kernel (5.7 us).
//
// In a CTA one warp copies pages into a ring (bulk copies of 4128 bytes, page ids fetched 32 at a
// time, queries of the next segment ahead) and the others take pages in turn: with 8 columns two at
// once, since a page alone is a chain of dependent products, exponentials and products of ~1400
// cycles and two cost little more; with more columns the groups fill the chain's gaps.
//
// Measured, 32 query and 8 KV heads: 256 sequences of 2304 tokens 200 us for the kernel alone, 6.25 TB/s of
// DRAM reads (0.95 of the copy rate): memory; 220 us a call with cold caches. One of 8192 tokens 17 us: start (4.5 us to the first page) and join (2 us of
// waiting, 4 of loads). 16 of 5 rows behind 300 to 2000 tokens 28.5 us: MMAs at 16 cycles, 48 a page for
// three groups, in 11 us of steps, the rest start, sums of the warps and join.
#include <algorithm>

#include <math_constants.h>

#include "common.cuh"
#include "kv8.cuh"
#include "lakeb_kernels.h"
#include "mma_sync.cuh"
#include "tma_host.h"

namespace lakeb {
namespace {

constexpr int kApartPages = 48;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.f;  // a base trails the true maximum by at most this
constexpr float kPBias = 7.f;  // P = 2^(w - bo + 7): fp16 subnormals begin at 2^-21 of the base

constexpr int kSegCost = 6;    // pages that the start and the join of a segment cost as much as

// Bytes of a column of Q and floats of a column of a warp's sums in shared memory: a quarter-warp's
// accesses to several columns fall on different banks (16 sequences of 5 rows: 31.5 -> 28.7 us).
constexpr int kQPitch = 256 + 32;
constexpr int kOPitch = kKv8Dim + 4;

// Shared memory of a CTA with NT groups of 8 columns: ring of pages, two query buffers, the
// consumers' sums for the join at a segment's end. One group: two CTAs per SM. More groups need more
// registers: one CTA per SM (with two of 16 columns the sums spill at 168 registers).
template <int NT>
struct Smem {
  static constexpr int kCols = 8 * NT;
  static constexpr int kWarps = NT == 1 ? 5 : 7;  // consumers; one more warp loads
  static constexpr int kThreads = kWarps * 32 + 32;
  static constexpr int kPerSm = NT == 1 ? 2 : 1;
  static constexpr int kPages = NT == 1 ? 2 : 1;  // of a step
  static constexpr int kSlots = NT == 1 ? 10 : 28;
  static constexpr int kQ = kSlots * kPages * kKv8Head;
  static constexpr int kO = kQ + 2 * kCols * kQPitch;
  static constexpr int kStat = kO + kWarps * kCols * kOPitch * 4;  // [warp][col][m, bo, l]
  static constexpr int kBar = kStat + kWarps * kCols * 3 * 4;
  static constexpr int kBytes = kBar + (2 * kSlots + 4) * 8;
  // A slot belongs to one warp: pages land out of order, and a warp that had not itself waited for
  // the slot's last phase could take it for the one it waits for.
  static_assert(kSlots % kWarps == 0, "");
  static_assert(kQ % 16 == 0 && kO % 16 == 0 && kBar % 8 == 0 && kBytes <= (NT == 1 ? 113 : 227) * 1024, "");
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma_f16_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t movmatrix_t(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// One warp's running state for 8 columns; this lane holds columns 2t and 2t+1 (t = lane & 3).
struct ColState {
  float o[8][4];            // [16-dim chunk][dim 2g: col 2t, 2t+1; dim 2g+1: col 2t, 2t+1]
  float m[2], bo[2], l[2];  // bases and this lane's part of the sum of p
};

// Adds NP pages (16 tokens each, from tok0) to the states. lim[n][e]: keys of column 8n+2t+e end
// before it; len: tokens from len on are not the sequence's (their bytes may be anything).
template <int NT, int NP>
__device__ __forceinline__ void pages_step(const uint8_t* pages, int tok0, int len, const int (&lim)[NT][2],
                                          const uint32_t (&qf)[NT][8][2], const float (&cq)[NT][2], int lane,
                                          ColState (&st)[NT]) {
  const int g = lane >> 2, j = lane >> 3, r8 = lane & 7;
  const int tok = (j & 1) * 8 + r8;
  const uint32_t kb = smem_u32(pages), vb = kb + kKv8Side;
  float s[NP][NT][4];
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[p][n][e] = 0.f;
#pragma unroll
  for (int c2 = 0; c2 < 4; ++c2)
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      uint32_t m0, m1, m2, m3;
      ldsm_x4(kb + p * kKv8Head + kv8_chunk(tok, 2 * c2 + (j >> 1)), m0, m1, m2, m3);
      const uint32_t a0 = f16x2_lo(m0), a1 = f16x2_lo(m1), a2 = f16x2_hi(m0), a3 = f16x2_hi(m1);
      const uint32_t b0 = f16x2_lo(m2), b1 = f16x2_lo(m3), b2 = f16x2_hi(m2), b3 = f16x2_hi(m3);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma_f16_16816(s[p][n], a0, a1, a2, a3, qf[n][2 * c2][0], qf[n][2 * c2][1]);
        mma_f16_16816(s[p][n], b0, b1, b2, b3, qf[n][2 * c2 + 1][0], qf[n][2 * c2 + 1][1]);
      }
    }
  float ev[NP][2];
  bool grow = false;
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) {
      const int tk = g + 8 * hi;
      const uint8_t* sk = pages + p * kKv8Head + kKv8Page * kKv8Dim + tk;
      const float ks = kv8_scale(*sk);
      const int b = sk[kKv8Side];
      ev[p][hi] = b == 255 ? CUDART_NAN_F : static_cast<float>(b - 127);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& z = s[p][n][2 * hi + e];
          z = tok0 + 16 * p + tk < lim[n][e] ? z * (ks * cq[n][e]) : -CUDART_INF_F;
          grow |= z > st[n].m[e] + kSlack || z + ev[p][hi] > st[n].bo[e] + kSlack;
        }
    }
  // w = z + ev: -inf where the key is not seen, whatever its scale byte is
  auto w = [&](int p, int n, int x) {
    const float z = s[p][n][x];
    return z == -CUDART_INF_F ? z : z + ev[p][x >> 1];
  };
  if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float zm = -CUDART_INF_F, wm = -CUDART_INF_F;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          zm = fmaxf(zm, fmaxf(s[p][n][e], s[p][n][2 + e]));
          wm = fmaxf(wm, fmaxf(w(p, n, e), w(p, n, 2 + e)));
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          zm = fmaxf(zm, __shfl_xor_sync(0xffffffffu, zm, o));
          wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, o));
        }
        ColState& c = st[n];
        const float mn = fmaxf(c.m[e], zm), bn = fmaxf(c.bo[e], wm);
        const float al = mn == -CUDART_INF_F ? 1.f : ex2(c.m[e] - mn);
        const float be = bn == -CUDART_INF_F ? 1.f : ex2(c.bo[e] - bn);
        c.m[e] = mn;
        c.bo[e] = bn;
        c.l[e] *= al;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          c.o[k][e] *= be;
          c.o[k][2 + e] *= be;
        }
      }
  }
  uint32_t p0[NP][NT], p1[NP][NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float mb[2], bb[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      mb[e] = st[n].m[e] == -CUDART_INF_F ? 0.f : st[n].m[e];
      bb[e] = st[n].bo[e] == -CUDART_INF_F ? 0.f : st[n].bo[e] - kPBias;
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      float P[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        st[n].l[x & 1] += ex2(s[p][n][x] - mb[x & 1]);
        P[x] = ex2(w(p, n, x) - bb[x & 1]);
      }
      p0[p][n] = movmatrix_t(pack_f16x2(P[0], P[1]));
      p1[p][n] = movmatrix_t(pack_f16x2(P[2], P[3]));
    }
  }
  const int t2 = (lane & 3) * 2;
  const bool tail = tok0 + NP * kKv8Page > len;
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
    if (tail) {  // codes past the sequence's end may be NaNs: P is 0 there, but 0 * NaN is not
      const int left = len - (tok0 + 16 * p + t2);
      keep0 = (left > 0 ? 0x00ff00ffu : 0u) | (left > 1 ? 0xff00ff00u : 0u);
      keep1 = (left > 8 ? 0x00ff00ffu : 0u) | (left > 9 ? 0xff00ff00u : 0u);
    }
#pragma unroll
    for (int c2 = 0; c2 < 4; ++c2) {
      uint32_t m0, m1, m2, m3;
      ldsm_x4_t(vb + p * kKv8Head + kv8_chunk(tok, 2 * c2 + (j >> 1)), m0, m1, m2, m3);
      // a transposed register holds (token 2t: dims 2g, 2g+1), (token 2t+1: the same): pair the tokens
      m0 = __byte_perm(m0, 0, 0x3120) & keep0;
      m1 = __byte_perm(m1, 0, 0x3120) & keep1;
      m2 = __byte_perm(m2, 0, 0x3120) & keep0;
      m3 = __byte_perm(m3, 0, 0x3120) & keep1;
      const uint32_t a0 = f16x2_lo(m0), a1 = f16x2_hi(m0), a2 = f16x2_lo(m1), a3 = f16x2_hi(m1);
      const uint32_t b0 = f16x2_lo(m2), b1 = f16x2_hi(m2), b2 = f16x2_lo(m3), b3 = f16x2_hi(m3);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma_f16_16816(st[n].o[2 * c2], a0, a1, a2, a3, p0[p][n], p1[p][n]);
        mma_f16_16816(st[n].o[2 * c2 + 1], b0, b1, b2, b3, p0[p][n], p1[p][n]);
      }
    }
  }
}

// Column g of `q` (bf16 rows of 128 in shared memory, `real` of them) as this lane's B fragment,
// times a power of two that brings the column's largest element to [2^14, 2^15).
__device__ __forceinline__ void load_columns(const uint8_t* q, int real, float scale, int lane, uint32_t (&qf)[8][2],
                                             float (&cq)[2]) {
  const int g = lane >> 2, t = lane & 3;
  float x[32];
  float top = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint2 u = g < real ? *reinterpret_cast<const uint2*>(q + g * kQPitch + k * 32 + t * 8) : make_uint2(0, 0);
    x[4 * k] = __uint_as_float(u.x << 16);
    x[4 * k + 1] = __uint_as_float(u.x & 0xffff0000u);
    x[4 * k + 2] = __uint_as_float(u.y << 16);
    x[4 * k + 3] = __uint_as_float(u.y & 0xffff0000u);
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(x[4 * k + i]));
  }
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const int E = static_cast<int>(__float_as_uint(top) >> 23);
  const int up = E == 255 ? 0 : min(141 - E, 126);
  const float f = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    qf[k][0] = pack_f16x2(x[4 * k] * f, x[4 * k + 1] * f);
    qf[k][1] = pack_f16x2(x[4 * k + 2] * f, x[4 * k + 3] * f);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int u = __shfl_sync(0xffffffffu, up, (2 * t + e) * 4);
    cq[e] = scale * kLog2e * __uint_as_float(static_cast<uint32_t>(127 - u) << 23);
  }
}

// The tiles' work where both kernels run (every lane calls it).
template <bool kMixed>
__device__ __forceinline__ int64_t warp_work(const Kv8AttnArgs& a, int lane) {
  if (!kMixed) return 0;
  const Kv8Packing pk = kv8_packing(a.n_q_heads / a.n_kv_heads, a.products);
  int sum = 0;
  for (int s = lane; s < min(a.num_tiles, kKv8Ranked); s += 32) {
    const int4 t = a.tiles[s];
    if (t.z > 0 && kv8_tile_ok(a, t)) sum += kv8_tile_work(a, pk, t, kv8_tile_keys(a, t));
  }
  return static_cast<int64_t>(__reduce_add_sync(0xffffffffu, sum)) * a.n_kv_heads;
}

// One item of work: a sequence (decode) or a tile. Its segments are `units` = KV heads x groups of
// `cols` columns, of `pages` pages each.
struct Item {
  int seq, row0, nq, pos0, len, pages, groups, units;
};
template <int NT, bool kMixed>
__device__ __forceinline__ Item get_item(const Kv8AttnArgs& a, int s, int64_t work) {
  Item it = {};
  if (a.tiles) {
    const int4 t = a.tiles[s];
    // A tile without rows names nothing (its sequence may be any number), a refused one no sequence of this
    // call, and a call may have no sequences at all: no length is read for them.
    if (t.z <= 0 || !kv8_tile_ok(a, t)) return it;
    if (kMixed && !kv8_tile_is_few(a, t, kv8_tile_keys(a, t), work)) return it;
    it.seq = t.x, it.row0 = t.y, it.nq = t.z, it.pos0 = t.w;
  } else {
    it.seq = it.row0 = s, it.nq = 1;
  }
  it.len = kv8_seq_len(a, it.seq);
  if (!a.tiles) it.pos0 = it.len - 1;
  const int G = a.n_q_heads / a.n_kv_heads;
  it.groups = (it.nq * G + 8 * NT - 1) / (8 * NT);
  it.units = a.n_kv_heads * it.groups;
  it.pages = (max(0, min(it.len, it.pos0 + it.nq)) + kKv8Page - 1) / kKv8Page;
  return it;
}

// A place in the laid-out work, in pages: the item and the offset in it (each of its units is
// kSegCost + pages long, the start's cost first).
struct Place {
  int item;
  int in_item;
};
template <int NT, bool kMixed>
__device__ __forceinline__ int item_cost(const Kv8AttnArgs& a, int s, int64_t work) {
  const Item it = get_item<NT, kMixed>(a, s, work);
  return it.pages > 0 ? (it.pages + kSegCost) * it.units : 0;
}
// The whole length, the number of segments and the pages of the longest one (for every lane; more than 256
// items: as if it were too long for `apart`). The first 256 items' lengths and segments stay in `keep` and
// `units`, for find_place.
struct Total {
  int64_t cost;
  int segments, longest;
};
template <int NT, bool kMixed>
__device__ __forceinline__ Total total_cost(const Kv8AttnArgs& a, int items, int64_t work, int lane, int (&keep)[8],
                                            int (&units)[8]) {
  int64_t sum = 0;
  int segments = 0, longest = items > 256 ? INT32_MAX : 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    keep[k] = units[k] = 0;
    if (32 * k < items) {  // (a branch for the whole warp: code that is not run is not fetched either)
      if (32 * k + lane < items) {
        const Item it = get_item<NT, kMixed>(a, 32 * k + lane, work);
        if (it.pages > 0) {
          units[k] = it.units;
          keep[k] = (it.pages + kSegCost) * it.units;
          longest = max(longest, it.pages);
        }
      }
      sum += keep[k];
      segments += units[k];
    }
  }
  for (int s = 256 + lane; s < items; s += 32) sum += item_cost<NT, kMixed>(a, s, work);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return {sum, static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(segments))),
          __reduce_max_sync(0xffffffffu, longest)};
}
// A few short segments are not cut: each has a CTA, and there is nothing to join. (Four or sixteen of 63
// pages a head take 1 us less when they are.)
__device__ __forceinline__ bool apart(const Total& t, int ctas) { return t.longest <= kApartPages && t.segments <= ctas; }
// Place `at` (every lane of the warp calls it); past the end: item == items.
template <int NT, bool kMixed>
__device__ __forceinline__ Place find_place(const Kv8AttnArgs& a, int items, int64_t work, int64_t at, int lane,
                                            const int (&keep)[8]) {
  // the 32 items that hold it, by their sums; then the item, by a scan of them
  int s0 = 0, mine = 0;
  bool hit = false;
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (!hit) {
      const unsigned sum = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(keep[k]));
      hit = at < sum;
      if (hit) s0 = 32 * k, mine = keep[k];
      else at -= sum;
    }
  for (int s = 256; s < items && !hit; s += 32) {
    const int n = s + lane < items ? item_cost<NT, kMixed>(a, s + lane, work) : 0;
    const unsigned sum = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(n));
    hit = at < sum;
    if (hit) s0 = s, mine = n;
    else at -= sum;
  }
  if (!hit) return {items, 0};
  int sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += up;
  }
  const int l = __ffs(__ballot_sync(0xffffffffu, sum > static_cast<int>(at))) - 1;
  return {s0 + l, static_cast<int>(at) - __shfl_sync(0xffffffffu, sum - mine, l)};
}
// Length of a CTA's run; below 32 pages a run is not worth its joining.
__device__ __forceinline__ int64_t run_length(int64_t total, int ctas) {
  const int64_t per = total < (int64_t(1) << 31) ? static_cast<uint32_t>(total + ctas - 1) / static_cast<uint32_t>(ctas)
                                                 : (total + ctas - 1) / ctas;
  return per < 32 ? 32 : per;
}

__device__ __forceinline__ float base_or_zero(float x) { return x == -CUDART_INF_F ? 0.f : x; }
__device__ __forceinline__ float factor(float x, float to) { return x == -CUDART_INF_F ? 1.f : ex2(x - to); }
// Sums of a column as the output: acc * 2^(B - M - kPBias) / L. The power goes in as two halves, since it
// alone may be below fp32's smallest (values near bf16's own: V scales of 2^-119 and less).
__device__ __forceinline__ uint2 column_out(const float4& acc, float M, float B, float L) {
  const float h = ex2(0.5f * (base_or_zero(B) - base_or_zero(M) - kPBias)), f = L == 0.f ? 0.f : h / L;
  return make_uint2(pack_bf16x2(acc.x * f * h, acc.y * f * h), pack_bf16x2(acc.z * f * h, acc.w * f * h));
}

// The pieces that a CTA's run cuts out of the segments, in order. Loader and consumers walk the same.
template <int NT, bool kMixed>
struct Walk {
  int s;            // item
  Item it;
  int64_t left;     // of the run, from offset x of segment `unit` on
  int unit, x;
  int64_t work;
  __device__ void start(const Kv8AttnArgs& a, int item, int in_item, int64_t n) {
    s = item;
    left = n;
    if (n <= 0) return;
    it = get_item<NT, kMixed>(a, s, work);
    unit = in_item / (it.pages + kSegCost);
    x = in_item - unit * (it.pages + kSegCost);
    if (count() == 0) left = 0;
  }
  __device__ int end() const {  // offset in the segment at which the run leaves it
    return static_cast<int>(min(static_cast<int64_t>(it.pages + kSegCost), x + left));
  }
  __device__ int page() const { return max(0, x - kSegCost); }
  __device__ int count() const { return max(0, end() - kSegCost) - page(); }  // pages of the piece
  __device__ void next(const Kv8AttnArgs& a) {
    left -= end() - x;
    if (left <= 0) return;
    x = 0;
    if (++unit == it.units) {
      unit = 0;
      do it = get_item<NT, kMixed>(a, ++s, work);
      while (it.pages == 0);
    }
    if (count() == 0) left = 0;  // the run ends in the segment's start cost: all its pages are the next one's
  }
};

__device__ __forceinline__ int whole_ctas(const Kv8AttnArgs& a, int whole) { return a.n_kv_heads * max(whole, 1); }

template <int NT, bool kMixed>
__global__ void __launch_bounds__(Smem<NT>::kThreads, Smem<NT>::kPerSm) kv8_attn_kernel(const Kv8AttnArgs a, const int whole) {
  using S = Smem<NT>;
  constexpr int kWarps = S::kWarps;
  extern __shared__ __align__(128) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBar);
  uint64_t* empty = full + S::kSlots;
  uint64_t* q_full = empty + S::kSlots;
  uint64_t* q_empty = q_full + 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.n_q_heads / a.n_kv_heads;
  const int items = a.tiles ? a.num_tiles : a.num_seqs;

  if (threadIdx.x < 2 * S::kSlots + 4) {
    mbar_init(full + threadIdx.x, threadIdx.x < 2 * S::kSlots + 2 ? 1 : kWarps);
    fence_mbar_init();
  }
  __syncthreads();
  after_previous();

  Walk<NT, kMixed> w;
  const int64_t work = warp_work<kMixed>(a, lane);
  w.work = work;
  // whole: CTA = (item, KV head, part of its column groups); `whole` parts
  const int own = static_cast<int>(blockIdx.x) / whole_ctas(a, whole), own_part = static_cast<int>(blockIdx.x) % max(whole, 1);
  const int own_head = static_cast<int>(blockIdx.x) % whole_ctas(a, whole) / max(whole, 1);
  if (whole) {
    const Item it = get_item<NT, kMixed>(a, own, work);
    const int each = (it.groups + whole - 1) / whole, g0 = min(own_part * each, it.groups), g1 = min(g0 + each, it.groups);
    const int cost = it.pages > 0 ? it.pages + kSegCost : 0;
    w.start(a, own, (own_head * it.groups + g0) * cost, (g1 - g0) * cost);
  } else {
    int keep[8], units[8];
    const Total total = total_cost<NT, kMixed>(a, items, work, lane, keep, units);
    if (apart(total, gridDim.x)) {
      const Place p = find_place<NT, kMixed>(a, items, work, blockIdx.x, lane, units);
      const int n = p.item < items ? get_item<NT, kMixed>(a, p.item, work).pages + kSegCost : 0;
      w.start(a, p.item, p.in_item * n, n);
    } else {
      const int64_t per = run_length(total.cost, gridDim.x), run0 = blockIdx.x * per;
      const Place p = find_place<NT, kMixed>(a, items, work, run0, lane, keep);
      w.start(a, p.item, p.in_item, max(int64_t(0), min(per, total.cost - run0)));
    }
  }

  if (warp == kWarps) {
    // -------------------------------------------------------------- loader
    bool ok = true;
    int n = 0;  // steps so far
    for (int piece = 0; w.left > 0 && ok; ++piece, w.next(a)) {
      const int kvh = w.unit / w.it.groups, cg = w.unit % w.it.groups;
      const int cnt = w.count();
      const int* bt = a.block_tables + static_cast<int64_t>(w.it.seq) * a.bt_stride + w.page();
      int ids = lane < cnt ? bt[lane] : 0;
      // queries: the group's columns c = row * G + head, bf16 rows of 256 bytes
      const int qb = piece & 1, c0 = cg * S::kCols, c1 = min(w.it.nq * G, c0 + S::kCols);
      ok = __all_sync(0xffffffffu, mbar_wait(&q_empty[qb], ((piece >> 1) & 1) ^ 1, nullptr, a.status));
      if (!ok) break;
      if (lane == 0) mbar_expect_tx(&q_full[qb], (c1 - c0) * 256);
      __syncwarp();
      if (c0 + lane < c1)
        bulk_load(smem + S::kQ + (qb * S::kCols + lane) * kQPitch,
                  a.q + static_cast<int64_t>(w.it.row0 + (c0 + lane) / G) * a.q_stride +
                      (static_cast<int64_t>(kvh) * G + (c0 + lane) % G) * kKv8Dim,
                  256, &q_full[qb]);
      const uint8_t* base = a.arena + a.layer_offset + static_cast<int64_t>(kvh) * kKv8Head;
      for (int i0 = 0; i0 < cnt && ok; i0 += 32) {
        int now = ids;
        if (i0 + 32 + lane < cnt) ids = bt[i0 + 32 + lane];
        if (i0 + lane < cnt && (now < 0 || now >= a.num_blocks)) {
          record_error(a.status, kErrBounds);
          now = 0;
        }
        const int m = min(32, cnt - i0);
        for (int i = 0; i < m; i += S::kPages, ++n) {
          const int slot = n % S::kSlots, here = min(S::kPages, m - i);
          const int id = __shfl_sync(0xffffffffu, now, i + lane % S::kPages);
          ok = __all_sync(0xffffffffu, mbar_wait(&empty[slot], ((n / S::kSlots) & 1) ^ 1, nullptr, a.status));
          if (!ok) break;
          if (lane == 0) mbar_expect_tx(&full[slot], here * kKv8Head);
          __syncwarp();
          if (lane < here)
            bulk_load(smem + (S::kPages * slot + lane) * kKv8Head, base + id * a.block_bytes, kKv8Head, &full[slot]);
        }
      }
    }
    return;
  }

  // ---------------------------------------------------------------- consumers
  float* mo = reinterpret_cast<float*>(smem + S::kO);
  float* ms = reinterpret_cast<float*>(smem + S::kStat);
  const int g = lane >> 2, t2 = (lane & 3) * 2;
  // rows of sequences without keys
  for (int s = whole ? (own_part ? items : own) : blockIdx.x; s < items; s += whole ? items : gridDim.x) {
    const Item it = get_item<NT, kMixed>(a, s, work);
    if (it.pages > 0) continue;
    const int h0 = whole ? own_head * G : 0, nh = whole ? G : a.n_q_heads;
    for (int i = threadIdx.x; i < it.nq * nh * kKv8Dim; i += kWarps * 32)
      a.out[static_cast<int64_t>(it.row0 + i / (nh * kKv8Dim)) * a.out_stride + h0 * kKv8Dim + i % (nh * kKv8Dim)] =
          __float2bfloat16(0.f);
  }
  bool ok = true;
  int n = 0;
  for (int piece = 0; w.left > 0; ++piece, w.next(a)) {
    const Item& it = w.it;
    const int kvh = w.unit / it.groups, cb = w.unit % it.groups * S::kCols;
    const int ncols = min(S::kCols, it.nq * G - cb);
    const int cnt = w.count();
    uint32_t qf[NT][8][2];
    float cq[NT][2];
    int lim[NT][2];
    ColState st[NT];
    const int qb = piece & 1;
    ok = __all_sync(0xffffffffu, ok && mbar_wait(&q_full[qb], (piece >> 1) & 1, nullptr, a.status));
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      load_columns(smem + S::kQ + (qb * S::kCols + 8 * k) * kQPitch, ncols - 8 * k, a.scale, lane, qf[k], cq[k]);
#pragma unroll
      for (int c = 0; c < 8; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) st[k].o[c][e] = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        st[k].m[e] = st[k].bo[e] = -CUDART_INF_F;
        st[k].l[e] = 0.f;
        const int col = 8 * k + t2 + e;
        lim[k][e] = col < ncols ? min(it.len, it.pos0 + (cb + col) / G + 1) : 0;
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&q_empty[qb]);
    const int steps = (cnt + S::kPages - 1) / S::kPages;
    for (int i = (warp + kWarps - n % kWarps) % kWarps; i < steps; i += kWarps) {
      const int slot = (n + i) % S::kSlots;
      ok = __all_sync(0xffffffffu, ok && mbar_wait(&full[slot], ((n + i) / S::kSlots) & 1, nullptr, a.status));
      if (!ok) break;
      // a piece's last step may have fewer pages: the rest of its slot is not the piece's
      const int end = (w.page() + cnt) * kKv8Page;
      int lm[NT][2];
#pragma unroll
      for (int k = 0; k < NT; ++k) lm[k][0] = min(lim[k][0], end), lm[k][1] = min(lim[k][1], end);
      pages_step<NT, S::kPages>(smem + S::kPages * slot * kKv8Head, (w.page() + S::kPages * i) * kKv8Page,
                                min(it.len, end), lm, qf, cq, lane, st);
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[slot]);
    }
    n += steps;
    // join the warps' sums
#pragma unroll
    for (int k = 0; k < NT; ++k) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) st[k].l[e] += __shfl_xor_sync(0xffffffffu, st[k].l[e], o);
      float* d = mo + (warp * S::kCols + 8 * k + t2) * kOPitch + 2 * g;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        *reinterpret_cast<float2*>(d + 16 * c) = make_float2(st[k].o[c][0], st[k].o[c][2]);
        *reinterpret_cast<float2*>(d + kOPitch + 16 * c) = make_float2(st[k].o[c][1], st[k].o[c][3]);
      }
      if (g == 0)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float* x = ms + (warp * S::kCols + 8 * k + t2 + e) * 3;
          x[0] = st[k].m[e], x[1] = st[k].bo[e], x[2] = st[k].l[e];
        }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");
    const bool entire = cnt == it.pages;
    const int64_t part = (2 * static_cast<int64_t>(blockIdx.x) + (piece > 0)) * S::kCols;
    for (int col = warp; col < ncols; col += kWarps) {
      float M = -CUDART_INF_F, B = -CUDART_INF_F;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        M = fmaxf(M, ms[(k * S::kCols + col) * 3]);
        B = fmaxf(B, ms[(k * S::kCols + col) * 3 + 1]);
      }
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float L = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        const float* x = ms + (k * S::kCols + col) * 3;
        L += x[2] * factor(x[0], M);
        const float f = factor(x[1], B);
        const float4 v = *reinterpret_cast<const float4*>(mo + (k * S::kCols + col) * kOPitch + 4 * lane);
        acc.x += v.x * f;
        acc.y += v.y * f;
        acc.z += v.z * f;
        acc.w += v.w * f;
      }
      if (entire) {
        const int c = cb + col;
        *reinterpret_cast<uint2*>(a.out + static_cast<int64_t>(it.row0 + c / G) * a.out_stride +
                                  (kvh * G + c % G) * kKv8Dim + 4 * lane) = column_out(acc, M, B, L);
      } else {
        *reinterpret_cast<float4*>(a.ws_o + (part + col) * kKv8Dim + 4 * lane) = acc;
        if (lane == 0) *reinterpret_cast<float4*>(a.ws_ml + (part + col) * 4) = make_float4(M, B, L, 0.f);
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");
  }
}

// Joins the segment whose pages begin in CTA run c and end in a later one (CTA c of this kernel). Its
// first piece is c's last one, the others are the first pieces of the runs c + 1, c + 2, ...
template <int NT, bool kMixed>
__global__ void __launch_bounds__(256) kv8_join_kernel(const Kv8AttnArgs a) {
  constexpr int kCols = 8 * NT;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.n_q_heads / a.n_kv_heads;
  const int items = a.tiles ? a.num_tiles : a.num_seqs;
  asm volatile("griddepcontrol.launch_dependents;");
  // lengths and tiles are not the first kernel's to write: the search needs no wait
  int keep[8], units[8];
  const int64_t work = warp_work<kMixed>(a, lane);
  const Total t = total_cost<NT, kMixed>(a, items, work, lane, keep, units);
  const int64_t total = t.cost, per = run_length(total, gridDim.x);
  const int64_t run0 = blockIdx.x * per, run1 = run0 + per;
  // (every CTA waits for the first kernel, those with nothing to do as well: what is launched next
  // follows this kernel's end alone)
  if (run1 >= total || apart(t, gridDim.x)) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const Place p = find_place<NT, kMixed>(a, items, work, run1 - 1, lane, keep);
  const Item it = get_item<NT, kMixed>(a, p.item, work);
  const int unit = p.in_item / (it.pages + kSegCost);
  const int64_t seg0 = run1 - 1 - p.in_item % (it.pages + kSegCost);
  const int64_t seg1 = seg0 + kSegCost + it.pages;
  const int64_t first = seg0 + kSegCost;  // its first page
  if (first < run0 || first >= run1 || seg1 <= run1) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const int pieces = static_cast<int>((seg1 - 1) / per - blockIdx.x) + 1;
  const int slot0 = 2 * static_cast<int>(blockIdx.x) + (seg0 > run0);
  const int kvh = unit / it.groups, cb = unit % it.groups * kCols;
  const int ncols = min(kCols, it.nq * G - cb);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // A warp has the columns warp, warp + 8, ... all at once: one after the other, each would wait twice
  // for memory.
  float M[NT], B[NT], L[NT];
  float4 acc[NT];
  auto slot = [&](int i, int k) {
    return static_cast<int64_t>(i == 0 ? slot0 : 2 * (static_cast<int>(blockIdx.x) + i)) * kCols + warp + 8 * k;
  };
#pragma unroll
  for (int k = 0; k < NT; ++k) {
    M[k] = B[k] = -CUDART_INF_F;
    L[k] = 0.f;
    acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int i = 0; i < pieces; i += 2) {
    float4 x[2][NT], v[2][NT];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int k = 0; k < NT; ++k) {
        const bool real = i + j < pieces && warp + 8 * k < ncols;
        x[j][k] = real ? *reinterpret_cast<const float4*>(a.ws_ml + slot(i + j, k) * 4)
                       : make_float4(-CUDART_INF_F, -CUDART_INF_F, 0.f, 0.f);
        v[j][k] = real ? *reinterpret_cast<const float4*>(a.ws_o + slot(i + j, k) * kKv8Dim + 4 * lane)
                       : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int k = 0; k < NT; ++k) {
        const float m = fmaxf(M[k], x[j][k].x), b = fmaxf(B[k], x[j][k].y);
        const float fl = factor(M[k], m), gl = factor(x[j][k].x, m), fo = factor(B[k], b), go = factor(x[j][k].y, b);
        L[k] = L[k] * fl + x[j][k].z * gl;
        acc[k].x = acc[k].x * fo + v[j][k].x * go;
        acc[k].y = acc[k].y * fo + v[j][k].y * go;
        acc[k].z = acc[k].z * fo + v[j][k].z * go;
        acc[k].w = acc[k].w * fo + v[j][k].w * go;
        M[k] = m;
        B[k] = b;
      }
  }
#pragma unroll
  for (int k = 0; k < NT; ++k)
    if (warp + 8 * k < ncols) {
      const int c = cb + warp + 8 * k;
      *reinterpret_cast<uint2*>(a.out + static_cast<int64_t>(it.row0 + c / G) * a.out_stride +
                                (kvh * G + c % G) * kKv8Dim + 4 * lane) = column_out(acc[k], M[k], B[k], L[k]);
    }
}

// Whether a CTA takes whole segments: few pages.
bool takes_whole(const Kv8AttnArgs& a) { return a.max_blocks <= kKv8WholePages; }

template <int NT, bool kMixed>
int launch(const Kv8AttnArgs& a, cudaStream_t stream) {
  const int items = a.tiles ? a.num_tiles : a.num_seqs;
  if (int e = ensure_smem_attr(reinterpret_cast<const void*>(kv8_attn_kernel<NT, kMixed>), Smem<NT>::kBytes)) return e;
  if (takes_whole(a)) {
    // each column group of an average tile has a CTA
    const int64_t cols = (a.tiles ? (a.num_rows + a.num_tiles - 1) / a.num_tiles : 1) * int64_t(a.n_q_heads / a.n_kv_heads);
    const int64_t parts = std::max<int64_t>(1, (cols + 8 * NT - 1) / (8 * NT)), ctas = parts * items * a.n_kv_heads;
    if (ctas > INT32_MAX) return -1;
    return launch_ahead(kv8_attn_kernel<NT, kMixed>, static_cast<unsigned>(ctas), Smem<NT>::kThreads, Smem<NT>::kBytes,
                        stream, a, static_cast<int>(parts));
  }
  const int ctas = Smem<NT>::kPerSm * num_sms();
  if (int e = launch_ahead(kv8_attn_kernel<NT, kMixed>, ctas, Smem<NT>::kThreads, Smem<NT>::kBytes, stream, a, 0)) return e;
  return launch_ahead(kv8_join_kernel<NT, kMixed>, ctas, 256, 0, stream, a);  // its search runs while the first ends
}

}  // namespace

int64_t kv8_attention_ws_floats(const Kv8AttnArgs& a) {
  const int nt = kv8_attention_groups(a);
  return takes_whole(a) ? 0 : int64_t(2) * (nt == 1 ? 2 : 1) * num_sms() * 8 * nt * (kKv8Dim + 4);
}

int kv8_attention_launches(const Kv8AttnArgs& a) {
  return (a.tiles ? a.num_tiles : a.num_seqs) <= 0 ? 0 : takes_whole(a) ? 1 : 2;
}

// Groups of 8 columns that a CTA holds at once, by the columns of a tile on average: a pass over the
// pages costs 16 MMAs of 16 cycles per page and group, so a group that stays empty costs as much as
// a full one, and columns beyond the groups cost another pass.
int kv8_attention_groups(const Kv8AttnArgs& a) {
  const int64_t rows = !a.tiles ? 1 : a.few_rows > 0 ? a.few_rows : (a.num_rows + a.num_tiles - 1) / a.num_tiles;
  const int64_t groups = (rows * (a.n_q_heads / a.n_kv_heads) + 7) / 8;
  return groups < 1 ? 1 : groups < 3 ? static_cast<int>(groups) : 3;  // (no rows: empty tiles alone)
}

int kv8_attention(const Kv8AttnArgs& a, cudaStream_t stream) {
  if ((a.tiles ? a.num_tiles : a.num_seqs) <= 0) return 0;
  const int64_t rows = !a.tiles ? 1 : a.few_rows > 0 ? a.few_rows : kKv8TileRows;
  const int64_t cols = 8 * kv8_attention_groups(a);
  const int64_t units = a.n_kv_heads * ((rows * (a.n_q_heads / a.n_kv_heads) + cols - 1) / cols);
  if (units > INT32_MAX / 32 || (int64_t(a.max_blocks) + kSegCost) * units > INT32_MAX / 32) return -1;
  // Launches that share the tiles with kv8_prefill (their tiles fill three groups) have kernels of their
  // own: the others are short, and slower by the code that they would have to fetch (one sequence of
  // 8192 tokens 20 us instead of 18).
  switch (kv8_attention_groups(a)) {
    case 1: return launch<1, false>(a, stream);
    case 2: return launch<2, false>(a, stream);
    default: return a.few_rows > 0 ? launch<3, true>(a, stream) : launch<3, false>(a, stream);
  }
}

}  // namespace lakeb
