// Causal prefill attention over the 8-bit KV arena on tcgen05 tensor cores (sm_100a).
//
// A CTA owns up to 128 query rows of two query heads A and B of one KV head (the last head of an
// odd group runs alone), so each K/V tile that it brings in and converts serves both. Per tile of
// 128 keys:
//   S_h   = Q_h K_j^T           tcgen05.mma fp16 (M=128, N=128, K=128), fp32 in tensor memory
//   P_h   = 2^(S_h c + e_j - b) softmax warpgroup h: thread = query row; fp16 over S_h's columns
//   O_h  += P_h V_j             tcgen05.mma, A = P_h from tensor memory, V_j MN-major in shared memory
// The MMA warp issues PV_A(j), S_A(j+1), PV_B(j), S_B(j+1): one head's products run while the
// other head's softmax does.
//
// 8-bit operands become fp16 ones in shared memory: bulk copies bring the tile's eight pages
// (4128 bytes each, K, V and scales) into a staging buffer, a warpgroup of converters turns codes
// into fp16 rows of the 128-byte swizzle (thread = key; e4m3 -> fp16 is exact). The tensor cores'
// own fp8 products would need Q and P in 8 bits as well, or twice the products. A tile is scaled
// against its own largest K scale and V scale: a row keeps code * 2^(e_row - e_tile), exact while
// e_tile - e_row <= 15 (a code's last bit is 2^-9, fp16's 2^-24), and e_tile itself is one
// multiplier of the tile's scores, or one addend of its exponents, not work per element. Where
// rows of one tile differ by more than 2^15, the small rows' last bits are lost: an error of
// 2^-24 of the largest element of the tile.
//
// Softmax statistics: w = score in log2 units + e_j, b = a base that follows the largest w of the
// row lazily (it moves when w grows by more than 2^8), P = 2^(w - b + 7) <= 2^15. The row sum is
// kept in fp32 over sum_j 2^(e_0 - e_j) rowsum(P_j), so O / sum needs 2^(e_0) at the end.
//
// Warps: 0 = loads, 1 = tensor memory and MMA issue, 2-3 idle, 4-7 = converters, 8-11 and 12-15 =
// softmax of head A and B. Registers are moved from the first two warpgroups to the softmax ones,
// which hold a row of 128 scores. Every wait is bounded; a role whose wait ran out goes on through
// its loop without work, so that the converters' named barrier is always reached by all of them.
#include <math_constants.h>

#include "common.cuh"
#include "kv8.cuh"
#include "lakeb_kernels.h"
#include "softmax_tc.cuh"
#include "tma_host.h"

namespace lakeb {
namespace {

constexpr int kTile = 128;
constexpr int kHalf = 128 * 128;      // 128 rows x 64 dims x 2 B
constexpr int kOperand = 2 * kHalf;   // 32 KB: both 64-dim halves
constexpr int kQ = 0;                 // Q of head A, B
constexpr int kK = 2 * kOperand;      // fp16 K, 2 stages
constexpr int kV = kK + 2 * kOperand; // fp16 V, 2 stages
constexpr int kRaw = kV + 2 * kOperand;              // staging: 8 pages as they lie in the arena
constexpr int kBars = kRaw + 8 * kKv8Head;           // 229,632
constexpr int kParams = kBars + 192;                 // [4] TileParams
constexpr int kRed = kParams + 4 * 32;               // [2][4] converter warps' maxima and flags
constexpr int kSmem = kRed + 2 * 4 * 16 + 1024;      // + the 1024-byte alignment
constexpr int kThreads = 512;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.0f;
constexpr float kPBias = 7.0f;
constexpr int kConvBar = 1;

// e_tile of K and V, and the keys whose V row is NaN (their codes are 0: the softmax makes the
// scores of rows that see them NaN, so that rows that do not stay clean).
struct TileParams {
  int ek, ev;
  uint32_t nan[4];
  int any_nan, pad;
};
static_assert(sizeof(TileParams) == 32, "");

// fp16 x fp16 -> fp32, both K-major; with bmn B is MN-major.
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, bool bmn) {
  return (1u << 4) | (bmn ? 1u << 16 : 0u) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// 2^d as fp16 pair for d <= 0 (0 below fp16's range).
__device__ __forceinline__ uint32_t f16x2_exp2(int d) {
  const __half h = __float2half_rn(d < -40 ? 0.f : __uint_as_float(static_cast<uint32_t>(127 + d) << 23));
  const __half2 r = __halves2half2(h, h);
  return *reinterpret_cast<const uint32_t*>(&r);
}

// One row of 128 codes (chunk c at kv8_chunk) -> fp16 row `row` of a swizzled two-half tile.
__device__ __forceinline__ void convert_row(const uint8_t* side, int t, uint8_t* dst, int row, uint32_t f) {
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const uint4 q = *reinterpret_cast<const uint4*>(side + kv8_chunk(t, c));
    uint8_t* d = dst + (c >> 2) * kHalf + row * 128;
    const int k = (c & 3) * 2, sw = row & 7;
    *reinterpret_cast<uint4*>(d + ((k ^ sw) << 4)) = make_uint4(hmul2(f16x2_lo(q.x), f), hmul2(f16x2_hi(q.x), f),
                                                                hmul2(f16x2_lo(q.y), f), hmul2(f16x2_hi(q.y), f));
    *reinterpret_cast<uint4*>(d + (((k + 1) ^ sw) << 4)) = make_uint4(
        hmul2(f16x2_lo(q.z), f), hmul2(f16x2_hi(q.z), f), hmul2(f16x2_lo(q.w), f), hmul2(f16x2_hi(q.w), f));
  }
}
__device__ __forceinline__ void zero_row(uint8_t* dst, int row) {
#pragma unroll
  for (int c = 0; c < 16; ++c)
    *reinterpret_cast<uint4*>(dst + (c >> 3) * kHalf + row * 128 + (((c ^ row) & 7) << 4)) = make_uint4(0, 0, 0, 0);
}

__global__ void __launch_bounds__(kThreads, 1)
    kv8_prefill_kernel(const __grid_constant__ CUtensorMap qmap, const Kv8AttnArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kBars);
  uint64_t* q_full = bars + 0;    // Q in shared memory as bf16
  uint64_t* q_ready = bars + 1;   // Q converted to fp16
  uint64_t* raw_full = bars + 2;
  uint64_t* raw_empty = bars + 3;
  uint64_t* k_full = bars + 4;    // [2 stages]
  uint64_t* k_empty = bars + 6;   // [2]
  uint64_t* v_full = bars + 8;    // [2]
  uint64_t* v_empty = bars + 10;  // [2]
  uint64_t* s_full = bars + 12;   // [2 heads]
  uint64_t* p_full = bars + 14;   // [2 heads]
  uint64_t* o_done = bars + 16;   // [2 heads]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 18);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 19);
  TileParams* params = reinterpret_cast<TileParams*>(smem + kParams);

  // heavy (late) query tiles first: the grid runs in reverse tile order
  const int4 tile = a.tiles[a.num_tiles - 1 - static_cast<int>(blockIdx.x)];
  const int seq = tile.x, qrow0 = tile.y, nq = tile.z, pos0 = tile.w;
  if (nq <= 0) return;
  const int G = a.n_q_heads / a.n_kv_heads, pairs = (G + 1) / 2;
  const int kvh = static_cast<int>(blockIdx.y) / pairs, pair = static_cast<int>(blockIdx.y) % pairs;
  const int qh0 = kvh * G + 2 * pair;
  const int heads = min(2, G - 2 * pair);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = min(a.seq_lens[seq], a.max_blocks * kKv8Page);
  const int max_pos = min(pos0 + nq - 1, len - 1);
  const int n_tiles = max_pos < 0 ? 0 : max_pos / kTile + 1;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_ready, 128 * heads);
    mbar_init(raw_full, 1);
    mbar_init(raw_empty, 128);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 128);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 128);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&o_done[i], 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t t_s[2] = {tmem, tmem + 128};        // S of head A, B (P overwrites its first 64 columns)
  const uint32_t t_o[2] = {tmem + 256, tmem + 384};  // O of head A, B

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0 && n_tiles > 0) {
      // ------------------------------------------------------------ loads
      if (lane == 0) {
        mbar_expect_tx(q_full, heads * kOperand);
        for (int h = 0; h < heads; ++h)
          for (int half = 0; half < 2; ++half)
            tma_load_2d(smem + kQ + h * kOperand + half * kHalf, &qmap, q_full, (qh0 + h) * 128 + half * 64, qrow0);
      }
      const int* bt = a.block_tables + static_cast<int64_t>(seq) * a.bt_stride;
      const int nblk = (len + kKv8Page - 1) / kKv8Page;
      const uint8_t* base = a.arena + a.layer_offset + static_cast<int64_t>(kvh) * kKv8Head;
      bool ok = true;
      int next = lane < min(8, nblk) ? bt[lane] : 0;
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int n = min(8, nblk - 8 * j);
        int page = next;
        next = lane < min(8, nblk - 8 * (j + 1)) ? bt[8 * (j + 1) + lane] : 0;
        if (page < 0 || page >= a.num_blocks) {
          record_error(a.status, kErrBounds);
          page = 0;
        }
        ok = __all_sync(0xffffffffu, mbar_wait(raw_empty, (j & 1) ^ 1, abort_flag, a.status));
        if (ok && lane == 0) mbar_expect_tx(raw_full, n * kKv8Head);
        __syncwarp();
        if (ok && lane < n) bulk_load(smem + kRaw + lane * kKv8Head, base + page * a.block_bytes, kKv8Head, raw_full);
      }
      // the release arrivals of the last two tiles must land before the CTA exits
      for (int j = max(0, n_tiles - 2); j < n_tiles && ok; ++j)
        ok = mbar_wait(&k_empty[j & 1], (j >> 1) & 1, abort_flag, a.status) &&
             mbar_wait(&v_empty[j & 1], (j >> 1) & 1, abort_flag, a.status);
    } else if (warp == 1 && lane == 0 && n_tiles > 0) {
      // ------------------------------------------------------------ MMA issue
      constexpr uint32_t idesc_s = idesc_f16(128, 128, false);
      constexpr uint32_t idesc_o = idesc_f16(128, 128, true);
      auto issue_s = [&](int h, int j) {
        const uint32_t q_base = smem_u32(smem + kQ + h * kOperand);
        const uint32_t k_base = smem_u32(smem + kK + (j & 1) * kOperand);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t off = (k >> 2) * kHalf + (k & 3) * 32;
          umma_f16(t_s[h], umma_desc_sw128(q_base + off), umma_desc_sw128(k_base + off), idesc_s, k > 0);
        }
        umma_commit(&s_full[h]);
      };
      auto issue_pv = [&](int h, int j) {
        const uint32_t v_base = smem_u32(smem + kV + (j & 1) * kOperand);
#pragma unroll
        for (int k = 0; k < 8; ++k)  // 16 keys per step: P columns 8k..8k+7, V rows 16k..16k+15
          umma_f16_ts(t_o[h], t_s[h] + 8 * k, desc_sw128_mn(v_base + k * 2048, kHalf), idesc_o, (j > 0) || (k > 0));
        umma_commit(&o_done[h]);
      };
      bool ok = mbar_wait(q_ready, 0, abort_flag, a.status) && mbar_wait(&k_full[0], 0, abort_flag, a.status);
      if (ok) {
        tc_fence_after();
        for (int h = 0; h < heads; ++h) issue_s(h, 0);
        umma_commit(&k_empty[0]);
      }
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int s = j & 1, sn = (j + 1) & 1;
        const bool more = j + 1 < n_tiles;
        ok = mbar_wait(&v_full[s], (j >> 1) & 1, abort_flag, a.status);
        for (int h = 0; h < heads && ok; ++h) {
          if (!mbar_wait(&p_full[h], j & 1, abort_flag, a.status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          issue_pv(h, j);
          if (h == heads - 1) umma_commit(&v_empty[s]);
          if (more) {
            if (h == 0) {
              if (!mbar_wait(&k_full[sn], ((j + 1) >> 1) & 1, abort_flag, a.status)) {
                ok = false;
                break;
              }
              tc_fence_after();
            }
            issue_s(h, j + 1);  // after PV(h, j) in issue order: P's columns are read before S overwrites them
          }
        }
        if (ok && more) umma_commit(&k_empty[sn]);
      }
    }
  } else if (warp < 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    // -------------------------------------------------------------- converters: thread = key of the tile
    const int row = threadIdx.x - 128, t = row & 15;
    const uint8_t* page = smem + kRaw + (row >> 4) * kKv8Head;
    int* red = reinterpret_cast<int*>(smem + kRed);  // [2 tiles][4 warps][K max, V max, NaN keys]
    constexpr int kNone = -1000;
    int ev_last = kNone, ev_top = kNone;
    bool ok = true;
    for (int j = 0; j < n_tiles; ++j) {
      const int s = j & 1;
      const uint32_t ph = ((j >> 1) & 1) ^ 1;
      ok = ok && mbar_wait(raw_full, j & 1, abort_flag, a.status);
      const bool real = ok && j * kTile + row < len;
      const int kb = real ? page[kKv8Page * kKv8Dim + t] : 0, vb = real ? page[kKv8Side + kKv8Page * kKv8Dim + t] : 0;
      // rows of zeros (b <= 1) and NaN rows (255) say nothing about the tile's scale
      const int km = __reduce_max_sync(0xffffffffu, kb > 1 && kb < 255 ? kb - 127 : kNone);
      const int vm = __reduce_max_sync(0xffffffffu, vb > 1 && vb < 255 ? vb - 127 : kNone);
      const uint32_t nan = __ballot_sync(0xffffffffu, vb == 255);
      if (lane == 0) {
        int* r = red + (s * 4 + (warp - 4)) * 4;
        r[0] = km, r[1] = vm, r[2] = static_cast<int>(nan);
      }
      asm volatile("bar.sync %0, 128;" ::"n"(kConvBar) : "memory");
      int ek = kNone, et = kNone;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        ek = max(ek, red[(s * 4 + w) * 4]);
        et = max(et, red[(s * 4 + w) * 4 + 1]);
      }
      if (ek == kNone) ek = 0;
      // V's reference may fall by 15 per tile (what fp16 holds exactly) and to 2^-80 of the largest so
      // far, so that the sum's factor 2^(e_0 - e_j) stays within fp32
      int ev = et == kNone ? (ev_last == kNone ? -30 : ev_last) : max(et, -90);
      if (ev_last != kNone) ev = max(ev, max(ev_last - 15, ev_top - 80));
      ev_last = ev;
      ev_top = max(ev_top, ev);
      if (row == 0) {
        TileParams& p = params[j & 3];  // tile j - 4's was read before PV(j - 4), which v_empty below waited for
        p.ek = ek;
        p.ev = ev;
        int any = 0;
        for (int w = 0; w < 4; ++w) {
          p.nan[w] = static_cast<uint32_t>(red[(s * 4 + w) * 4 + 2]);
          any |= red[(s * 4 + w) * 4 + 2];
        }
        p.any_nan = any;
      }
      ok = ok && mbar_wait(&k_empty[s], ph, abort_flag, a.status);
      if (ok) {
        uint8_t* kd = smem + kK + s * kOperand;
        if (real) convert_row(page, t, kd, row, kb == 255 ? 0x7fff7fffu : f16x2_exp2(min(kb - 127 - ek, 0)));
        else zero_row(kd, row);
        fence_proxy_async_smem();
        mbar_arrive(&k_full[s]);
      }
      ok = ok && mbar_wait(&v_empty[s], ph, abort_flag, a.status);
      if (ok) {
        uint8_t* vd = smem + kV + s * kOperand;
        if (real && vb != 255) convert_row(page + kKv8Side, t, vd, row, f16x2_exp2(min(vb - 127 - ev, 0)));
        else zero_row(vd, row);
        fence_proxy_async_smem();
        mbar_arrive(&v_full[s]);
        mbar_arrive(raw_empty);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
    // -------------------------------------------------------------- softmax + epilogue: thread = query row
    const int h = (warp - 8) >> 2;
    const int r = (warp & 3) * 32 + lane;  // query row in the tile = TMEM lane
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    if (h < heads && n_tiles > 0) {
      const int kmax = min(pos0 + r, len - 1);  // last key this row may see
      bool ok = __all_sync(0xffffffffu, mbar_wait(q_full, 0, abort_flag, a.status));
      // Q: bf16 -> fp16 in place, times a power of two that brings the row's largest element to [2^14, 2^15)
      float cr;
      {
        uint8_t* qrow = smem + kQ + h * kOperand + r * 128;
        auto at = [&](int c) { return reinterpret_cast<uint4*>(qrow + (c >> 3) * kHalf + (((c ^ r) & 7) << 4)); };
        uint4 x[16];
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          x[c] = *at(c);
          const uint32_t w[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
        }
        const int E = static_cast<int>(top >> 7);
        const int up = E == 255 ? 0 : min(141 - E, 126);
        const float f = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
        cr = a.scale * kLog2e * __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
        auto two = [&](uint32_t u) {
          return pack_f16x2(__uint_as_float(u << 16) * f, __uint_as_float(u & 0xffff0000u) * f);
        };
#pragma unroll
        for (int c = 0; c < 16; ++c)
          *at(c) = make_uint4(two(x[c].x), two(x[c].y), two(x[c].z), two(x[c].w));
      }
      fence_proxy_async_smem();
      if (ok) mbar_arrive(q_ready);
      float bo = -CUDART_INF_F;  // base of w, at most kSlack below the largest w so far
      float l = 0.f;
      int e0 = 0;
      for (int j = 0; j < n_tiles; ++j) {
        if (!__all_sync(0xffffffffu, ok && mbar_wait(&s_full[h], j & 1, abort_flag, a.status))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int k0 = j * kTile;
        const TileParams& tp = params[j & 3];
        uint32_t sv[128];
#pragma unroll
        for (int c = 0; c < 4; ++c)
          tmem_ld32(t_s[h] + lane_off + c * 32, *reinterpret_cast<uint32_t(*)[32]>(sv + 32 * c));
        const float ev = static_cast<float>(tp.ev);
        const float c = cr * __uint_as_float(static_cast<uint32_t>(127 + tp.ek) << 23);
        if (j == 0) e0 = tp.ev;
        const float unscale = exp2f(static_cast<float>(e0 - tp.ev));
        const bool nan = tp.any_nan != 0;
        tmem_ld_wait();
        if (k0 + kTile - 1 > kmax) {  // the diagonal or the sequence end: keys past this row's last
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (k0 + i > kmax) sv[i] = __float_as_uint(-CUDART_INF_F);
        }
        if (nan) {
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (((tp.nan[i >> 5] >> (i & 31)) & 1u) && k0 + i <= kmax) sv[i] = 0x7fffffffu;
        }
        // row max: eight independent three-input chains, then a short tree
        float mv[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) mv[q] = max3f(__uint_as_float(sv[q]), __uint_as_float(sv[8 + q]), -CUDART_INF_F);
#pragma unroll
        for (int i = 16; i < 128; i += 16)
#pragma unroll
          for (int q = 0; q < 8; ++q) mv[q] = max3f(mv[q], __uint_as_float(sv[i + q]), __uint_as_float(sv[i + 8 + q]));
        const float mx =
            fmaf(max3f(max3f(mv[0], mv[1], mv[2]), max3f(mv[3], mv[4], mv[5]), fmaxf(mv[6], mv[7])), c, ev);
        const bool grow = mx > bo + kSlack;
        const float old = bo;
        if (grow) bo = mx;
        const float add = bo == -CUDART_INF_F ? 0.f : ev - bo + kPBias;
        float2 rs[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        const float2 cv = make_float2(c, c), av = make_float2(add, add);
#pragma unroll
        for (int k = 0; k < 64; ++k) {  // key pair k -> packed column k (written over consumed scores)
          const float2 z = fma2(make_float2(__uint_as_float(sv[2 * k]), __uint_as_float(sv[2 * k + 1])), cv, av);
          const float2 p = make_float2(ex2(z.x), ex2(z.y));
          rs[k & 3] = add2(rs[k & 3], p);
          sv[k] = pack_f16x2(p.x, p.y);
          if (k == 31) tmem_st32(t_s[h] + lane_off, *reinterpret_cast<uint32_t(*)[32]>(sv));
        }
        tmem_st32(t_s[h] + lane_off + 32, *reinterpret_cast<uint32_t(*)[32]>(sv + 32));
        rs[0] = add2(add2(rs[0], rs[1]), add2(rs[2], rs[3]));
        // O and l still hold sums against the old base. tcgen05.ld/st are warp-collective: the whole
        // warp rescales when any of its rows needs it (rows that do not keep alpha = 1).
        float alpha = 1.f;
        if (__any_sync(0xffffffffu, grow && j > 0)) {
          if (!__all_sync(0xffffffffu, mbar_wait(&o_done[h], (j - 1) & 1, abort_flag, a.status))) {
            ok = false;
            break;
          }
          tc_fence_after();
          alpha = (grow && old != -CUDART_INF_F) ? ex2(old - bo) : 1.f;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t ov[32];
            tmem_ld32(t_o[h] + lane_off + q * 32, ov);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
            tmem_st32(t_o[h] + lane_off + q * 32, ov);
          }
        }
        l = fmaf(l, alpha, (rs[0].x + rs[0].y) * unscale);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_full[h]);
      }
      if (ok && __all_sync(0xffffffffu, mbar_wait(&o_done[h], (n_tiles - 1) & 1, abort_flag, a.status))) {
        tc_fence_after();
        const float inv = l == 0.f ? 0.f : exp2f(static_cast<float>(e0)) / l;
        __nv_bfloat16* orow = a.out + static_cast<int64_t>(qrow0 + r) * a.out_stride + (qh0 + h) * 128;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t ov[32];
          tmem_ld32(t_o[h] + lane_off + c * 32, ov);
          tmem_ld_wait();
          if (r < nq) {
            uint4* dst = reinterpret_cast<uint4*>(orow + c * 32);
            auto two = [&](int i) {
              return pack_bf16x2(__uint_as_float(ov[i]) * inv, __uint_as_float(ov[i + 1]) * inv);
            };
#pragma unroll
            for (int v = 0; v < 4; ++v) dst[v] = make_uint4(two(8 * v), two(8 * v + 2), two(8 * v + 4), two(8 * v + 6));
          }
        }
      }
      tc_fence_before();
    } else if (h < heads && r < nq) {  // an empty context
      uint4* dst = reinterpret_cast<uint4*>(a.out + static_cast<int64_t>(qrow0 + r) * a.out_stride + (qh0 + h) * 128);
#pragma unroll
      for (int v = 0; v < 16; ++v) dst[v] = make_uint4(0, 0, 0, 0);
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace

int kv8_prefill_tc(const Kv8AttnArgs& a, cudaStream_t stream) {
  if (a.num_tiles <= 0) return 0;
  CUtensorMap qmap;
  const int64_t cols = static_cast<int64_t>(a.n_q_heads) * 128;
  if (!encode_bf16_map(&qmap, a.q, a.num_rows, cols, a.num_rows > 1 ? a.q_stride : cols, 128, 64)) return -5;
  if (int e = ensure_smem_attr(reinterpret_cast<const void*>(kv8_prefill_kernel), kSmem)) return e;
  const int G = a.n_q_heads / a.n_kv_heads;
  kv8_prefill_kernel<<<dim3(a.num_tiles, a.n_kv_heads * ((G + 1) / 2)), kThreads, kSmem, stream>>>(qmap, a);
  return cudaGetLastError();
}

}  // namespace lakeb
