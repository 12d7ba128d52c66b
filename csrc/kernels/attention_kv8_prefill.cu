// Causal prefill attention over the 8-bit KV arena on tcgen05 tensor cores (sm_100a).
//
// A CTA owns two products A and B of 128 rows, which are query rows and heads of one KV head
// (kv8_packing), so each K/V tile of 128 keys that it brings in and converts serves both; where a tile's
// rows or an odd group's heads end in A, it runs alone. Per step of 64 keys and h = A, B:
//   S_h   = Q_h K_i^T           tcgen05.mma fp16 (M=128, N=64, K=128), fp32 in tensor memory
//   P_h   = 2^(S_h c + e - b)   softmax warpgroup h: thread = row; fp16 over S_h's columns
//   O_h  += P_h V_i             tcgen05.mma, A = P_h from tensor memory, V_i MN-major in shared memory
// A product has two S buffers of 64 columns: S(i+1) is there when the softmax of step i ends, and PV(i)
// and S(i+2) run behind it. With one buffer of 128 columns (tensor memory holds no more beside the
// two O) softmax and tensor cores take turns, and 128 keys of both took 5.1k cycles; so they take
// 4.4k, of which the products run 2.6k and the exponentials 2.0k. What binds is shared
// memory (products' operands, conversion and copies move ~390 KB per tile, 3.0k cycles) and the
// hand-offs that wait behind it. Measured, single calls: one 8192-token prompt of 32 query and 8 KV heads
// 0.57 to 0.64 ms by its data, 860 to 960 TFLOP/s; four of 2048 tokens 0.21 ms, 660 TFLOP/s. A CTA spends ~7 us around its main loop
// (1.9 us until its queries arrive, 1.6 to convert them, about as long for the output, the rest start
// and end), so eight prompts of 500 tokens, four tiles of keys a CTA at most, run at 255 TFLOP/s. CTAs
// that stay and take tile after tile overlapped little of that and issued products more slowly (1152
// rows behind 7040 tokens: 181 us against 165), so a CTA has one tile. The grid goes tile by tile,
// heaviest first, all heads of a tile side by side: head by head, the last heads' heavy tiles started
// late (0.63 ms).
//
// 8-bit operands become fp16 ones in shared memory: bulk copies bring the K and the V sides of the
// tile's eight pages (2064 bytes each, scales included) into a staging buffer each, a warpgroup for
// each side turns codes into fp16 rows of the 128-byte swizzle (thread = key; e4m3 -> fp16 is
// exact). The tensor cores' own fp8 products would need Q and P in 8 bits as well, or twice the
// products. Where the K scales of a tile's keys lie within 2^15 of each other, its rows are kept against
// the largest: code * 2^(e_row - e_K), exact (a code's last bit is 2^-9, fp16's 2^-24), and e_K is one
// multiplier of the tile's scores. Where the V scales lie within 2^8, the same: e_V is one addend of the
// tile's exponents. (The largest scale may be that of a key that a row does not see, or sees with no weight:
// its P are up to 2^8 smaller for it, of the 2^21 between P's base and fp16's subnormals.) A tile of a wider
// range keeps its codes as they are, and each key's scale enters its own scores and exponents, as in
// kv8_attention: then what a row does not see has no part in it whatever it holds. Tokens' scales lie within a
// few octaves of each other as a rule; a prompt of 8192 tokens whose every tile is wider takes 2.7 ms, 4.7 times as
// long (its steps are a function of their own: within the loop they cost the others registers, 2 % of the time).
//
// Softmax statistics, for each row: z = score in log2 units, w = z + e (e of V, the key's or the tile's). bo
// follows the largest w and m the largest z, lazily: O is kept against 2^(bo - 7), with P = 2^(w - bo + 7)
// <= 2^15, and the sum l of 2^z against 2^m. Of a tile with one e, l gets the sum of P times 2^(bo - 7 - e - m);
// where that factor is past 2^82, P may be below fp32's range and 2^(z - m) not: such a tile's steps take the
// exponentials of both.
//
// Warps: 0 = loads, 1 = tensor memory and MMA issue, 2-3 idle, 4-7 = converters of K, 8-11 = of V,
// 12-15 and 16-19 = softmax of A and B. Registers move from the first three warpgroups to the
// softmax ones (80, 80, 80, 120 and 120 of 96 each: the split with the fewest spills). Every wait is
// bounded; a role whose wait ran out goes on through its loop without work, so that the converters'
// named barriers are always reached by all of their warps.
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
constexpr int kRaw = kV + 2 * kOperand;              // staging: the K and the V sides of 8 pages
constexpr int kBars = kRaw + 8 * kKv8Head;           // 229,632
constexpr int kParams = kBars + 256;                 // [4] TileParams
constexpr int kScales = kParams + 4 * 32;            // [4][K, V][128] scale bytes of the keys as they were converted
constexpr int kRed = kScales + 4 * 2 * kTile;        // [2 tiles][K, V][4] converter warps' extremes and flags
constexpr int kSmem = kRed + 2 * 2 * 4 * 8;
static_assert(kSmem <= 227 * 1024, "");
constexpr int kThreads = 640;
constexpr int kStep = 64;                            // keys per softmax step
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.0f;
constexpr float kPBias = 7.0f;
constexpr float kSumSlack = 40.0f;                   // m trails the largest z by at most this (l <= 2^60 for 2^20 keys)
constexpr float kSumFactor = 82.0f;
constexpr int kSpanK = 15, kSpanV = 8;               // octaves between a tile's scales that one factor serves

// e of K and V (of a tile within kSpanK, kSpanV), and the keys whose V row is NaN (their codes are 0: the softmax
// makes the scores of rows that see them NaN, so that rows that do not stay clean).
struct TileParams {
  int ek, ev;
  uint32_t nan[4];
  int wide_k, wide_v;  // wide_v: bit 0; bit 1: there are NaN keys
};
static_assert(sizeof(TileParams) == 32, "");

// Product A's first row in q and head, the rows from there to the tile's end, its first row's position,
// and how far B's are from A's.
struct Rows {
  int row, head, left, pos, row_b, head_b;
};

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

// A value that every lane holds, as the result of a vote: the compiler then knows it to be the same
// in the whole warp (uniform registers and branches; the 8192-token prompt 640 -> 626 us).
__device__ __forceinline__ int uniform(int v) {
  return static_cast<int>(__ballot_sync(0xffffffffu, (v >> (threadIdx.x & 31)) & 1));
}

// One lane of the warp, the same each time. The MMA warp runs its loop as a whole and this lane's
// products take effect: descriptors stay in uniform registers, and products issue as fast as they
// run (48 cycles for 128 x 64 x 16, 64 for 128 x 128 x 16; from a branch of one lane ~120).
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(r));
  return r;
}
// Products and commits that take effect in the lane with lead != 0.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t lead) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t lead) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead));
}
__device__ __forceinline__ void commit(uint64_t* bar, uint32_t lead) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(smem_u32(bar)),
      "r"(lead)
      : "memory");
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
// Whether a row of codes has any that is not 0.
__device__ __forceinline__ bool any_code(const uint8_t* side, int t) {
  uint32_t any = 0;
#pragma unroll 1
  for (int c = 0; c < 8; ++c) {
    const uint4 q = *reinterpret_cast<const uint4*>(side + t * kKv8Dim + c * 16);
    any |= (q.x | q.y | q.z | q.w) & 0x7f7f7f7fu;
  }
  return any != 0;
}
__device__ __forceinline__ void zero_row(uint8_t* dst, int row) {
#pragma unroll
  for (int c = 0; c < 16; ++c)
    *reinterpret_cast<uint4*>(dst + (c >> 3) * kHalf + row * 128 + (((c ^ row) & 7) << 4)) = make_uint4(0, 0, 0, 0);
}

__device__ __forceinline__ void tma_load_3d(void* dst, const void* tmap, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

// A softmax step of 64 keys where each has scales of its own (kb: the keys' K scales, their V scales one kTile
// behind; keys past `last` are not seen): P over S in tensor memory, the row's bases and l brought up to date,
// the step's part of l added to `sum`.
__device__ __noinline__ void slow_step(uint32_t t_s, const uint8_t* kb, const uint32_t* nan, float cr, int last, float& bo, float& m,
                               float& l, float& sum) {
  const uint8_t* vb = kb + kTile;
  uint32_t x[32], p[32];
  auto scores = [&](int q) {
    tmem_ld32(t_s + 32 * q, x);
    tmem_ld_wait();
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      float z = __uint_as_float(x[k]) * (cr * kv8_scale(kb[32 * q + k]));
      if ((nan[q] >> k) & 1u) z = CUDART_NAN_F;
      x[k] = __float_as_uint(32 * q + k > last ? -CUDART_INF_F : z);
      if ((k & 3) == 3) asm volatile("" ::: "memory");  // (few scales at a time: they are registers)
    }
  };
  float zt = -CUDART_INF_F, wt = -CUDART_INF_F;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    scores(q);
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      zt = fmaxf(zt, __uint_as_float(x[k]));
      wt = fmaxf(wt, __uint_as_float(x[k]) + static_cast<float>(vb[32 * q + k] - 127));
      if ((k & 3) == 3) asm volatile("" ::: "memory");
    }
  }
  if (wt > bo + kSlack) bo = wt;
  if (zt > m + kSumSlack) l *= ex2(m - zt), m = zt;
  const float zb = m == -CUDART_INF_F ? 0.f : m, wb = (bo == -CUDART_INF_F ? 0.f : bo - kPBias) + 127.f;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    scores(q);
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float z0 = __uint_as_float(x[2 * k]), z1 = __uint_as_float(x[2 * k + 1]);
      const float e0 = static_cast<float>(vb[32 * q + 2 * k]), e1 = static_cast<float>(vb[32 * q + 2 * k + 1]);
      sum += ex2(z0 - zb) + ex2(z1 - zb);
      p[16 * q + k] = pack_f16x2(ex2(z0 + (e0 - wb)), ex2(z1 + (e1 - wb)));
      if ((k & 3) == 3) asm volatile("" ::: "memory");
    }
  }
  tmem_st32(t_s, p);
}

__global__ void __launch_bounds__(kThreads, 1)
    kv8_prefill_kernel(const __grid_constant__ CUtensorMap qmap, const Kv8AttnArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kBars);
  uint64_t* q_full = bars + 0;      // Q in shared memory as bf16
  uint64_t* q_ready = bars + 1;     // Q converted to fp16
  uint64_t* raw_full = bars + 2;    // [K, V]
  uint64_t* raw_empty = bars + 4;   // [K, V]
  uint64_t* k_full = bars + 6;      // [2 stages]
  uint64_t* k_empty = bars + 8;     // [2]
  uint64_t* v_full = bars + 10;     // [2]
  uint64_t* v_empty = bars + 12;    // [2]
  uint64_t* s_full = bars + 14;     // [2 heads][2 buffers]
  uint64_t* p_full = bars + 18;     // [2 heads][2 buffers]
  uint64_t* o_done = bars + 22;     // [2 heads], a phase per step
  uint64_t* o_last = bars + 24;     // [2 heads], the last step's PV
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 26);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 27);
  // This CTA's rows for the softmax warps, which read them again at the end rather than hold them.
  volatile Rows* rows = reinterpret_cast<volatile Rows*>(bars + 28);
  TileParams* params = reinterpret_cast<TileParams*>(smem + kParams);

  // (behind kv8_attention it waits at its end: what that read was there before it began)
  if (a.few_rows == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
  // Heavy query tiles first, or one of them would run on alone at the end. Of one sequence they are the
  // late ones; of several, each CTA finds the tile of its rank by the keys that it sees.
  if (smem_u32(smem) & 1023) {  // the swizzled tiles need it; the launch gives it
    if (threadIdx.x == 0) record_error(a.status, kErrBadArg);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const int G = a.n_q_heads / a.n_kv_heads;
  const Kv8Packing pk = kv8_packing(G, a.products);
  const int place = static_cast<int>(blockIdx.x) / (a.n_kv_heads * pk.units);  // all heads of a tile side by side
  const int at = static_cast<int>(blockIdx.x) % (a.n_kv_heads * pk.units);
  int rank = a.num_tiles - 1 - place;
  int64_t work = 0;
  if (a.num_seqs > 1) {
    int* keys = reinterpret_cast<int*>(smem + kK);
    int* sums = keys + kKv8Ranked;  // of each warp's tiles; then the rank's tile
    const int t = threadIdx.x;
    int4 x = make_int4(0, 0, 0, 0);
    int n = 0;
    if (t < kKv8Ranked) {
      if (t < a.num_tiles) x = a.tiles[t];
      const bool ok = x.z > 0 && kv8_tile_ok(a, x);
      if (ok) n = kv8_tile_keys(a, x);
      const int sum = __reduce_add_sync(0xffffffffu, ok ? kv8_tile_work(a, pk, x, n) : 0);
      if ((t & 31) == 0) sums[t >> 5] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kKv8Ranked / 32; ++w) work += sums[w];
    work *= a.n_kv_heads;
    if (a.num_tiles <= kKv8Ranked) {
      if (n > 0 && kv8_tile_is_few(a, x, n, work)) n = 0;
      if (t < kKv8Ranked) keys[t] = t < a.num_tiles ? n : -1;
      __syncthreads();
      if (t < a.num_tiles) {
        int before = 0;
        for (int u = 0; u < a.num_tiles; u += 4) {
          const int4 k = *reinterpret_cast<const int4*>(keys + u);
          before += (k.x > n || (k.x == n && u < t)) + (k.y > n || (k.y == n && u + 1 < t)) +
                    (k.z > n || (k.z == n && u + 2 < t)) + (k.w > n || (k.w == n && u + 3 < t));
        }
        if (before == place) sums[kKv8Ranked / 32] = t;
      }
      __syncthreads();
      rank = sums[kKv8Ranked / 32];
    }
  }
  const int4 tile = a.tiles[rank];
  const int seq = tile.x, pos0 = tile.w;
  // this CTA's rows of the tile: the last rows, with the most keys, first
  const int sub = pk.pack > 1 ? pk.subs - 1 - at % pk.subs : 0, row_a = sub * a.products * pk.rows;
  const int nq = pk.pack > 1 ? min(tile.z, row_a + a.products * pk.rows) : tile.z;  // rows of the tile up to this CTA's last
  if (nq <= row_a || !kv8_tile_ok(a, tile) || (a.few_rows > 0 && kv8_tile_is_few(a, tile, kv8_tile_keys(a, tile), work))) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const int unit = at % pk.units;
  const int head_a = at / pk.units * G + (pk.pack > 1 ? unit / pk.subs * pk.pack : a.products * unit);
  const int row_b = pk.pack > 1 ? pk.rows : 0, head_b = pk.pack > 1 ? 0 : 1;  // product B begins so much later
  const int heads = uniform(pk.pack > 1 ? (nq > row_a + pk.rows ? 2 : 1) : min(a.products, G - a.products * unit));
  const int kvh = at / pk.units;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = kv8_seq_len(a, seq);
  const int max_pos = min(pos0 + nq - 1, len - 1);
  const int n_steps = uniform(max_pos < 0 ? 0 : max_pos / kStep + 1);
  const int n_tiles = (n_steps + 1) / 2;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_ready, 128 * heads);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], 128);
      mbar_init(&k_full[i], 128);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 128);
      mbar_init(&v_empty[i], 1);
      mbar_init(&o_done[i], 1);
      mbar_init(&o_last[i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
    }
    *abort_flag = 0;
    rows->row = tile.y + row_a;
    rows->head = head_a;
    rows->left = nq - row_a;
    rows->pos = pos0 + row_a;
    rows->row_b = row_b;
    rows->head_b = head_b;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  const uint32_t t_s[2] = {tmem, tmem + 128};        // S of head A, B: two buffers of 64 columns (P over the first 32)
  const uint32_t t_o[2] = {tmem + 256, tmem + 384};  // O of head A, B

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == 0 && n_tiles > 0) {
      // ------------------------------------------------------------ loads
      if (lane == 0) {
        mbar_expect_tx(q_full, heads * kOperand);
        for (int h = 0; h < heads; ++h)
          for (int half = 0; half < 2; ++half)
            tma_load_3d(smem + kQ + h * kOperand + half * kHalf, &qmap, q_full, half * 64, head_a + h * head_b,
                        tile.y + row_a + h * row_b);
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
        for (int kv = 0; kv < 2; ++kv) {
          ok = __all_sync(0xffffffffu, ok && mbar_wait(&raw_empty[kv], (j & 1) ^ 1, abort_flag, a.status));
          if (ok && lane == 0) mbar_expect_tx(&raw_full[kv], n * kKv8Side);
          __syncwarp();
          if (ok && lane < n)
            bulk_load(smem + kRaw + (kv * 8 + lane) * kKv8Side, base + page * a.block_bytes + kv * kKv8Side, kKv8Side,
                      &raw_full[kv]);
        }
      }
      // the release arrivals of the last two tiles must land before the CTA exits
      for (int j = max(0, n_tiles - 2); j < n_tiles && ok; ++j)
        ok = mbar_wait(&k_empty[j & 1], (j >> 1) & 1, abort_flag, a.status) &&
             mbar_wait(&v_empty[j & 1], (j >> 1) & 1, abort_flag, a.status);
    } else if (warp == 1 && n_tiles > 0) {
      // ------------------------------------------------------------ MMA issue
      // The whole warp runs this loop and one elected lane's instructions take effect: descriptors stay
      // in uniform registers (from a branch of one lane each product cost ~120 cycles of issue, twice
      // its run time).
      constexpr uint32_t idesc_s = idesc_f16(128, kStep, false);
      constexpr uint32_t idesc_o = idesc_f16(128, 128, true);
      const uint32_t lead = elect_one();
      const uint64_t q_desc = umma_desc_sw128(smem_u32(smem + kQ)), k_desc = umma_desc_sw128(smem_u32(smem + kK));
      const uint64_t v_desc = desc_sw128_mn(smem_u32(smem + kV), kHalf);
      auto issue_s = [&](int h, int i) {
        const uint64_t qd = q_desc + h * (kOperand >> 4);
        const uint64_t kd = k_desc + ((i >> 1) & 1) * (kOperand >> 4) + (i & 1) * (kStep * 128 >> 4);
        const uint32_t d = tmem + h * 128 + (i & 1) * kStep;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          constexpr int kNext = kHalf >> 4;
          const int off = (k >> 2) * kNext + (k & 3) * 2;
          mma_ss(d, qd + off, kd + off, idesc_s, k > 0, lead);
        }
        commit(&s_full[2 * h + (i & 1)], lead);
      };
      auto issue_pv = [&](int h, int i) {  // 16 keys per product: 8 columns of P, 16 rows of V
        const uint64_t vd = v_desc + ((i >> 1) & 1) * (kOperand >> 4) + (i & 1) * (kStep * 128 >> 4);
        const uint32_t d = tmem + 256 + h * 128, p = tmem + h * 128 + (i & 1) * kStep;
#pragma unroll
        for (int k = 0; k < 4; ++k) mma_ts(d, p + 8 * k, vd + k * 128, idesc_o, i > 0 || k > 0, lead);
        commit(&o_done[h], lead);
        if (i == n_steps - 1) commit(&o_last[h], lead);
      };
      bool ok = mbar_wait(q_ready, 0, abort_flag, a.status) && mbar_wait(&k_full[0], 0, abort_flag, a.status);
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        tc_fence_after();
        for (int i = 0; i < min(2, n_steps); ++i)
          for (int h = 0; h < heads; ++h) issue_s(h, i);
        commit(&k_empty[0], lead);
      }
      auto wait = [&](uint64_t* bar, int parity) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, a.status));
      };
      // S(h, i) goes over P(h, i - 2): PV(h, i - 2) has to be done with it, not just issued (products of
      // different shapes may overlap). It is issued behind the other head's next PV, so that the wait
      // for o_done finds it done.
      auto next_s = [&](int h, int i) {
        if (i < 2 || i >= n_steps) return true;
        if (h == 0 && (i & 1) == 0 && !wait(&k_full[(i >> 1) & 1], (i >> 2) & 1)) return false;
        if (!wait(&o_done[h], i & 1)) return false;
        tc_fence_after();
        issue_s(h, i);
        if (h == heads - 1 && ((i & 1) || i + 1 == n_steps)) commit(&k_empty[(i >> 1) & 1], lead);
        return true;
      };
      for (int i = 0; i < n_steps && ok; ++i) {
        const int j = i >> 1;
        if ((i & 1) == 0) ok = wait(&v_full[j & 1], (j >> 1) & 1);
        for (int h = 0; h < heads && ok; ++h) {
          ok = wait(&p_full[2 * h + (i & 1)], j & 1);
          if (!ok) break;
          tc_fence_after();
          issue_pv(h, i);
          if (h == heads - 1 && ((i & 1) || i + 1 == n_steps)) commit(&v_empty[j & 1], lead);
          ok = heads == 1 ? next_s(0, i + 2) : h == 0 ? next_s(1, i + 1) : next_s(0, i + 2);
        }
      }
    }
  } else if (warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    // ------------------------------- converters of K (kv = 0) and of V (kv = 1): thread = key of the tile
    const int kv = (warp - 4) >> 2, row = (threadIdx.x - 128) & 127, t = row & 15;
    const uint8_t* side = smem + kRaw + (kv * 8 + (row >> 4)) * kKv8Side;
    int e = kv ? -126 : 0;
    bool ok = true;
    for (int j = 0; j < n_tiles; ++j) {
      const int s = j & 1;
      uint4* red = reinterpret_cast<uint4*>(smem + kRed) + (s * 2 + kv) * 2;  // each warp's extremes and NaN keys
      // tile j - 4's was read before PV(j - 4) and S(j - 3), which the waits of tile j - 1 waited for
      TileParams& p = params[j & 3];
      ok = ok && mbar_wait(&raw_full[kv], j & 1, abort_flag, a.status);
      const bool real = ok && j * kTile + row < len;
      const int b = real ? side[kKv8Page * kKv8Dim + t] : 0;
      // rows of NaNs (255) and of zeros (the smallest scale, as rows that are not zeros may have) say nothing
      bool counts = true;
      uint32_t nan = 0;
      if (__any_sync(0xffffffffu, b <= 1 || b == 255)) {
        nan = __ballot_sync(0xffffffffu, b == 255);
        counts = b > 0 && b < 255 && (b > 1 || any_code(side, t));
      }
      const uint32_t top = __reduce_max_sync(0xffffffffu, counts ? b : 0u), low = __reduce_max_sync(0xffffffffu, counts ? 255u - b : 0u);
      if (lane == 0) reinterpret_cast<uint2*>(red)[warp & 3] = make_uint2(top << 16 | low, nan);
      asm volatile("bar.sync %0, 128;" ::"r"(1 + kv) : "memory");
      const uint4 r0 = red[0], r1 = red[1];
      const uint32_t both = __vmaxu2(__vmaxu2(r0.x, r0.z), __vmaxu2(r1.x, r1.z));
      const int hi = both >> 16, lo = 255 - static_cast<int>(both & 0xffffu);
      const bool wide = hi - lo > (kv ? kSpanV : kSpanK);
      if (hi > 0) e = hi - 127;  // (a tile without any keeps the last one's)
      smem[kScales + ((j & 3) * 2 + kv) * kTile + row] = static_cast<uint8_t>(wide ? b : e + 127);
      if (row == 0) {
        if (kv == 0) {
          p.ek = e;
          p.wide_k = wide;
        } else {
          p.ev = e;
          p.nan[0] = r0.y, p.nan[1] = r0.w, p.nan[2] = r1.y, p.nan[3] = r1.w;
          const uint32_t any = r0.y | r0.w | r1.y | r1.w;
          p.wide_v = (wide ? 1 : 0) | (any ? 2 : 0);
        }
      }
      ok = ok && mbar_wait(kv ? &v_empty[s] : &k_empty[s], ((j >> 1) & 1) ^ 1, abort_flag, a.status);
      if (ok) {
        uint8_t* dst = smem + (kv ? kV : kK) + s * kOperand;
        // a NaN row of K gives NaN scores; one of V becomes zeros, its NaNs come through P. (b = 0: never written)
        if (b > 0 && !(kv && b == 255))
          convert_row(side, t, dst, row, b == 255 ? 0x7fff7fffu : f16x2_exp2(wide ? 0 : min(b - 127 - e, 0)));
        else
          zero_row(dst, row);
        fence_proxy_async_smem();
        mbar_arrive(kv ? &v_full[s] : &k_full[s]);
        mbar_arrive(&raw_empty[kv]);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 120;");
    // -------------------------------------------------------------- softmax + epilogue: thread = query row
    const int h = (warp - 12) >> 2;
    const int r = (warp & 3) * 32 + lane;  // row of the product = TMEM lane: a query row and head
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    if (h < heads && n_steps > 0) {
      const int kmax = min(rows->pos + h * rows->row_b + (r >> pk.shift), len - 1);  // last key this row may see
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
          for (int i = 0; i < 4; ++i) top = __vmaxu2(top, w[i] & 0x7fff7fffu);
        }
        const int E = static_cast<int>(max(top >> 16, top & 0xffffu) >> 7);
        const int up = E == 255 ? 0 : min(141 - E, 126);
        const float f = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
        cr = a.scale * kLog2e * __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
        auto two = [&](uint32_t u) {
          return pack_f16x2(__uint_as_float(u << 16) * f, __uint_as_float(u & 0xffff0000u) * f);
        };
#pragma unroll
        for (int c = 0; c < 16; ++c) *at(c) = make_uint4(two(x[c].x), two(x[c].y), two(x[c].z), two(x[c].w));
      }
      fence_proxy_async_smem();
      if (ok) mbar_arrive(q_ready);
      float bo = -CUDART_INF_F;  // base of w, at most kSlack below the largest w so far
      float m = -CUDART_INF_F;   // base of l
      float l = 0.f, c = 0.f, ev = 0.f;
      int flags = 0;     // of the tile: bit 0: a wide range of scales; bit 1: NaN keys
      bool far = false;  // its steps are slow ones
      for (int i = 0; i < n_steps; ++i) {
        const int j = i >> 1, buf = i & 1;
        const TileParams& tp = params[j & 3];
        ok = ok && mbar_wait(&s_full[2 * h + buf], j & 1, abort_flag, a.status);
        if (buf == 0) ok = ok && mbar_wait(&v_full[j & 1], (j >> 1) & 1, abort_flag, a.status);  // e_j of V
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t t_mine = t_s[h] + lane_off + kStep * buf;
        if (buf == 0) {
          ev = static_cast<float>(tp.ev);
          flags = tp.wide_k | tp.wide_v;
          // (a step leaves bo - ev - m as it is, or less, or at most kSumSlack: this holds for both of the tile)
          far = __any_sync(0xffffffffu, (flags & 1) || bo - kPBias - ev - m > kSumFactor);
          // (not 0, where a row of zeros or small keys would make it that: masked scores are -infinity)
          c = fmaxf(cr * __uint_as_float(static_cast<uint32_t>(127 + tp.ek) << 23), 0x1p-126f);
        }
        const int k0 = i * kStep;
        const float old = bo;
        float sum = 0.f, power = 0.f;  // l gets 2^power sum
        if (far) {
          slow_step(t_mine, smem + kScales + (j & 3) * 2 * kTile + buf * kStep, tp.nan + buf * 2, cr, kmax - k0, bo, m, l, sum);
        } else {
          uint32_t sv[64];
          tmem_ld32(t_mine, *reinterpret_cast<uint32_t(*)[32]>(sv));
          tmem_ld32(t_mine + 32, *reinterpret_cast<uint32_t(*)[32]>(sv + 32));
          const bool nan = (flags & 2) != 0;
          tmem_ld_wait();
          if (k0 + kStep - 1 > kmax) {  // the diagonal or the sequence end: keys past this row's last
#pragma unroll
            for (int k = 0; k < 64; ++k)
              if (k0 + k > kmax) sv[k] = __float_as_uint(-CUDART_INF_F);
          }
          if (nan) {
#pragma unroll
            for (int k = 0; k < 64; ++k)
              if (((tp.nan[buf * 2 + (k >> 5)] >> (k & 31)) & 1u) && k0 + k <= kmax) sv[k] = 0x7fffffffu;
          }
          // row max: four independent three-input chains, then a short tree
          float mv[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) mv[q] = max3f(__uint_as_float(sv[q]), __uint_as_float(sv[4 + q]), -CUDART_INF_F);
#pragma unroll
          for (int k = 8; k < 64; k += 8)
#pragma unroll
            for (int q = 0; q < 4; ++q) mv[q] = max3f(mv[q], __uint_as_float(sv[k + q]), __uint_as_float(sv[k + 4 + q]));
          const float sx = fmaxf(max3f(mv[0], mv[1], mv[2]), mv[3]), mx = fmaf(sx, c, ev);
          if (mx > bo + kSlack) bo = mx;
          const float add = bo == -CUDART_INF_F ? 0.f : ev - bo + kPBias;
          float2 rs[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          const float2 cv = make_float2(c, c), av = make_float2(add, add);
#pragma unroll
          for (int k = 0; k < 32; ++k) {  // key pair k -> packed column k (written over consumed scores)
            const float2 z = fma2(make_float2(__uint_as_float(sv[2 * k]), __uint_as_float(sv[2 * k + 1])), cv, av);
            const float2 p = make_float2(ex2(z.x), ex2(z.y));
            rs[k & 1] = add2(rs[k & 1], p);
            sv[k] = pack_f16x2(p.x, p.y);
          }
          tmem_st32(t_mine, *reinterpret_cast<uint32_t(*)[32]>(sv));
          rs[0] = add2(rs[0], rs[1]);
          sum = rs[0].x + rs[0].y;
          const float zx = sx * c;
          if (zx > m + kSumSlack) l *= ex2(m - zx), m = zx;
          power = bo == -CUDART_INF_F ? 0.f : -add - m;
        }
        const bool grow = bo > old;
        // O still holds sums against the old base. tcgen05.ld/st are warp-collective: the whole
        // warp rescales when any of its rows needs it (rows that do not keep alpha = 1).
        if (__any_sync(0xffffffffu, grow && i > 0)) {
          if (!__all_sync(0xffffffffu, mbar_wait(&o_done[h], (i - 1) & 1, abort_flag, a.status))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const float alpha = (grow && old != -CUDART_INF_F) ? ex2(old - bo) : 1.f;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t ov[32];
            tmem_ld32(t_o[h] + lane_off + q * 32, ov);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 32; ++k) ov[k] = __float_as_uint(__uint_as_float(ov[k]) * alpha);
            tmem_st32(t_o[h] + lane_off + q * 32, ov);
          }
        }
        l = fmaf(sum, ex2(power), l);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_full[2 * h + buf]);
      }
      // (o_done's last phases may pass before this warp looks, or be two behind: parity alone cannot tell)
      ok = ok && mbar_wait(&o_last[h], 0, abort_flag, a.status);
      if (__all_sync(0xffffffffu, ok)) {
        tc_fence_after();
        // O * 2^(bo - 7 - m) / l, the power in two halves: alone it may be past what fp32 holds
        const float half = bo == -CUDART_INF_F ? 1.f : ex2(0.5f * (bo - kPBias - m));
        const float inv = l == 0.f ? 0.f : half / l;
        // Rows go through this head's Q, which no product reads any more, so that the warp stores whole
        // rows two at a time (a row per lane, 16 bytes at a time: eight prompts of 500 tokens 62.5 us
        // instead of 59). Chunk c of row r lies at chunk c ^ (r & 7): both ways are free of bank conflicts.
        uint8_t* stage = smem + kQ + h * kOperand + (warp & 3) * 32 * 256;
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {
          uint32_t ov[32];
          tmem_ld32(t_o[h] + lane_off + q * 32, ov);
          tmem_ld_wait();
          auto two = [&](int k) {
            return pack_bf16x2(__uint_as_float(ov[k]) * inv * half, __uint_as_float(ov[k + 1]) * inv * half);
          };
#pragma unroll
          for (int v = 0; v < 4; ++v)
            *reinterpret_cast<uint4*>(stage + lane * 256 + (((4 * q + v) ^ (lane & 7)) << 4)) =
                make_uint4(two(8 * v), two(8 * v + 2), two(8 * v + 4), two(8 * v + 6));
        }
        __syncwarp();
        const int l = lane & 15, row0 = (warp & 3) * 32;
        const int first = h * rows->row_b, left = rows->left, shift = kv8_packing(a.n_q_heads / a.n_kv_heads, 2).shift;
        __nv_bfloat16* o0 = a.out + rows->row * a.out_stride + (rows->head + h * rows->head_b) * 128 + l * 8;
#pragma unroll 2
        for (int i = 0; i < 16; ++i) {
          const int x = 2 * i + (lane >> 4), row = first + ((row0 + x) >> shift);
          if (row < left)
            *reinterpret_cast<uint4*>(o0 + row * a.out_stride + ((row0 + x) & ((1 << shift) - 1)) * 128) =
                *reinterpret_cast<const uint4*>(stage + x * 256 + ((l ^ (x & 7)) << 4));
        }
      }
      tc_fence_before();
    } else if (h < heads && h * rows->row_b + (r >> pk.shift) < rows->left) {  // an empty context
      uint4* dst = reinterpret_cast<uint4*>(a.out + (rows->row + h * rows->row_b + (r >> pk.shift)) * a.out_stride +
                                            (rows->head + h * rows->head_b + (r & (pk.pack - 1))) * 128);
#pragma unroll
      for (int v = 0; v < 16; ++v) dst[v] = make_uint4(0, 0, 0, 0);
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  // after kv8_attention's kernels for the small tiles, which this one does not read from: the call is
  // done when all are
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

}  // namespace

int kv8_prefill_tc(const Kv8AttnArgs& a, cudaStream_t stream) {
  if (a.num_tiles <= 0) return 0;
  CUtensorMap qmap;
  const Kv8Packing pk = kv8_packing(a.n_q_heads / a.n_kv_heads, a.products);
  const int64_t stride = a.num_rows > 1 ? a.q_stride : int64_t(a.n_q_heads) * 128;
  if (!encode_heads_map(&qmap, a.q, a.num_rows, a.n_q_heads, stride, pk.rows, pk.pack)) return -5;
  if (int e = ensure_smem_attr(reinterpret_cast<const void*>(kv8_prefill_kernel), kSmem)) return e;
  const int64_t items = static_cast<int64_t>(a.num_tiles) * a.n_kv_heads * pk.units;
  if (items > INT32_MAX) return -1;
  return launch_ahead(kv8_prefill_kernel, static_cast<unsigned>(items), kThreads, kSmem, stream, qmap, a);
}

}  // namespace lakeb
