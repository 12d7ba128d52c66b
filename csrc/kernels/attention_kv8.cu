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
#include <math_constants.h>

#include "common.cuh"
#include "kv8.cuh"
#include "lakeb_kernels.h"
#include "mma_sync.cuh"
#include "tma_host.h"

namespace lakeb {
namespace {

constexpr int kWarps = 4;
constexpr int kSlots = 20;  // pages in flight per CTA: 82,560 bytes, two CTAs per SM
constexpr int kCols = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.f;  // a base trails the true maximum by at most this
constexpr float kPBias = 7.f;  // P = 2^(w - bo + 7): fp16 subnormals begin at 2^-21 of the base

constexpr int kMergeFloats = kWarps * kCols * kKv8Dim;
constexpr int kRingBytes = kSlots * kKv8Head;
constexpr int kMergeOff = (kRingBytes + 15) / 16 * 16;
constexpr int kStatOff = kMergeOff + kMergeFloats * 4;
constexpr int kBarOff = kStatOff + kWarps * kCols * 3 * 4;
constexpr int kSmem = kBarOff + kSlots * 8;

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

// Adds one page (16 tokens from tok0) to the state. lim[e]: keys of column 2t+e end before lim[e];
// len: tokens from len on are not the sequence's (their bytes may be anything).
__device__ __forceinline__ void page_step(const uint8_t* page, int tok0, int len, const int (&lim)[2],
                                          const uint32_t (&qf)[8][2], const float (&cq)[2], int lane, ColState& st) {
  const int g = lane >> 2, j = lane >> 3, r8 = lane & 7;
  const int tok = (j & 1) * 8 + r8;
  const uint32_t kb = smem_u32(page), vb = kb + kKv8Side;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c2 = 0; c2 < 4; ++c2) {
    uint32_t m0, m1, m2, m3;
    ldsm_x4(kb + kv8_chunk(tok, 2 * c2 + (j >> 1)), m0, m1, m2, m3);
    mma_f16_16816(s, f16x2_lo(m0), f16x2_lo(m1), f16x2_hi(m0), f16x2_hi(m1), qf[2 * c2][0], qf[2 * c2][1]);
    mma_f16_16816(s, f16x2_lo(m2), f16x2_lo(m3), f16x2_hi(m2), f16x2_hi(m3), qf[2 * c2 + 1][0], qf[2 * c2 + 1][1]);
  }
  const uint8_t* sk = page + kKv8Page * kKv8Dim;
  const uint8_t* sv = sk + kKv8Side;
  float z[4], w[4];
  bool grow = false;
#pragma unroll
  for (int hi = 0; hi < 2; ++hi) {
    const int tk = g + 8 * hi;
    const float ks = kv8_scale(sk[tk]);
    const int b = sv[tk];
    const float ev = b == 255 ? CUDART_NAN_F : static_cast<float>(b - 127);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const bool see = tok0 + tk < lim[e];
      z[2 * hi + e] = see ? s[2 * hi + e] * (ks * cq[e]) : -CUDART_INF_F;
      w[2 * hi + e] = see ? z[2 * hi + e] + ev : -CUDART_INF_F;
      grow |= z[2 * hi + e] > st.m[e] + kSlack || w[2 * hi + e] > st.bo[e] + kSlack;
    }
  }
  if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float zm = fmaxf(z[e], z[2 + e]), wm = fmaxf(w[e], w[2 + e]);
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        zm = fmaxf(zm, __shfl_xor_sync(0xffffffffu, zm, o));
        wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, o));
      }
      const float mn = fmaxf(st.m[e], zm), bn = fmaxf(st.bo[e], wm);
      const float al = mn == -CUDART_INF_F ? 1.f : ex2(st.m[e] - mn);
      const float be = bn == -CUDART_INF_F ? 1.f : ex2(st.bo[e] - bn);
      st.m[e] = mn;
      st.bo[e] = bn;
      st.l[e] *= al;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        st.o[c][e] *= be;
        st.o[c][2 + e] *= be;
      }
    }
  }
  float P[4];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const float mb = st.m[e] == -CUDART_INF_F ? 0.f : st.m[e];
    const float bb = st.bo[e] == -CUDART_INF_F ? 0.f : st.bo[e] - kPBias;
    st.l[e] += ex2(z[e] - mb) + ex2(z[2 + e] - mb);
    P[e] = ex2(w[e] - bb);
    P[2 + e] = ex2(w[2 + e] - bb);
  }
  const uint32_t b0 = movmatrix_t(pack_f16x2(P[0], P[1])), b1 = movmatrix_t(pack_f16x2(P[2], P[3]));
  const bool tail = tok0 + kKv8Page > len;
  const int t2 = (lane & 3) * 2;
  uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
  if (tail) {  // codes past the sequence's end may be NaNs: P is 0 there, but 0 * NaN is not
    keep0 = (tok0 + t2 < len ? 0x00ff00ffu : 0u) | (tok0 + t2 + 1 < len ? 0xff00ff00u : 0u);
    keep1 = (tok0 + t2 + 8 < len ? 0x00ff00ffu : 0u) | (tok0 + t2 + 9 < len ? 0xff00ff00u : 0u);
  }
#pragma unroll
  for (int c2 = 0; c2 < 4; ++c2) {
    uint32_t m0, m1, m2, m3;
    ldsm_x4_t(vb + kv8_chunk(tok, 2 * c2 + (j >> 1)), m0, m1, m2, m3);
    // a transposed register holds (token 2t: dims 2g, 2g+1), (token 2t+1: the same): pair the tokens
    m0 = __byte_perm(m0, 0, 0x3120) & keep0;
    m1 = __byte_perm(m1, 0, 0x3120) & keep1;
    m2 = __byte_perm(m2, 0, 0x3120) & keep0;
    m3 = __byte_perm(m3, 0, 0x3120) & keep1;
    mma_f16_16816(st.o[2 * c2], f16x2_lo(m0), f16x2_hi(m0), f16x2_lo(m1), f16x2_hi(m1), b0, b1);
    mma_f16_16816(st.o[2 * c2 + 1], f16x2_lo(m2), f16x2_hi(m2), f16x2_lo(m3), f16x2_hi(m3), b0, b1);
  }
}

// Columns c = row * G + head-in-group of one tile: column base + g as this lane's B fragment.
// q is scaled by a power of two so that the column's largest element is in [2^14, 2^15).
__device__ __forceinline__ void load_columns(const Kv8AttnArgs& a, int row0, int kvh, int G, int ncols, int base,
                                             int lane, uint32_t (&qf)[8][2], float (&cq)[2]) {
  const int g = lane >> 2, t = lane & 3;
  const int col = base + g;
  float x[32];
  float top = 0.f;
  const bool real = col < ncols;
  const int c = real ? col : 0;
  const __nv_bfloat16* q =
      a.q + static_cast<int64_t>(row0 + c / G) * a.q_stride + (static_cast<int64_t>(kvh) * G + c % G) * kKv8Dim + 4 * t;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint2 u = real ? *reinterpret_cast<const uint2*>(q + 16 * k) : make_uint2(0, 0);
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
    cq[e] = a.scale * kLog2e * __uint_as_float(static_cast<uint32_t>(127 - u) << 23);
  }
}

// grid: (splits, kv heads * column groups, tiles). Four warps take a page each in turn.
__global__ void __launch_bounds__(kWarps * 32) kv8_attn_kernel(const Kv8AttnArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kBarOff);
  float* mo = reinterpret_cast<float*>(smem + kMergeOff);
  float* ms = reinterpret_cast<float*>(smem + kStatOff);  // [warp][col][m, bo, l]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.n_q_heads / a.n_kv_heads;
  int seq, row0, nq, pos0;
  if (a.tiles) {
    const int4 t = a.tiles[blockIdx.z];
    seq = t.x, row0 = t.y, nq = t.z, pos0 = t.w;
  } else {
    seq = row0 = blockIdx.z, nq = 1, pos0 = 0;
  }
  const int kvh = blockIdx.y;
  const int len = min(a.seq_lens[seq], a.max_blocks * kKv8Page);
  if (!a.tiles) pos0 = len - 1;
  const int ncols = nq * G;
  const int nblk = (max(len, 0) + kKv8Page - 1) / kKv8Page;
  const int per = (nblk + a.splits - 1) / a.splits;
  const int b0 = blockIdx.x * per, b1 = min(nblk, b0 + per);
  const int n = max(0, b1 - b0);
  const int* bt = a.block_tables + static_cast<int64_t>(seq) * a.bt_stride;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
  }
  __syncthreads();
  const uint8_t* base = a.arena + a.layer_offset + static_cast<int64_t>(kvh) * kKv8Head;
  int issued = 0;  // pages of this warp issued since the kernel's start (warp w owns slots w, w + 4, ...)
  int used = 0;
  bool ok = true;
  constexpr int kOwn = kSlots / kWarps;
  for (int cb = 0; cb < ncols; cb += kCols) {
    uint32_t qf[8][2];
    float cq[2];
    load_columns(a, row0, kvh, G, ncols, cb, lane, qf, cq);
    ColState st;
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) st.o[c][e] = 0.f;
    int lim[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      st.m[e] = st.bo[e] = -CUDART_INF_F;
      st.l[e] = 0.f;
      const int col = cb + (lane & 3) * 2 + e;
      lim[e] = col < ncols ? min(len, pos0 + col / G + 1) : 0;
    }
    auto issue = [&](int i) {  // lane 0: page b0 + warp + i * kWarps into the warp's next slot
      const int slot = (issued % kOwn) * kWarps + warp;
      int page = bt[b0 + warp + i * kWarps];
      if (page < 0 || page >= a.num_blocks) {
        record_error(a.status, kErrBounds);
        page = 0;
      }
      mbar_expect_tx(&full[slot], kKv8Head);
      bulk_load(smem + slot * kKv8Head, base + page * a.block_bytes, kKv8Head, &full[slot]);
      ++issued;
    };
    const int mine = n > warp ? (n - warp + kWarps - 1) / kWarps : 0;
    if (lane == 0)
      for (int i = 0; i < min(mine, kOwn); ++i) issue(i);
    for (int i = 0; i < mine; ++i) {
      const int slot = (used % kOwn) * kWarps + warp;
      ok = __all_sync(0xffffffffu, ok && mbar_wait(&full[slot], (used / kOwn) & 1, nullptr, a.status));
      if (!ok) break;
      page_step(smem + slot * kKv8Head, (b0 + warp + i * kWarps) * kKv8Page, len, lim, qf, cq, lane, st);
      __syncwarp();
      ++used;
      if (lane == 0 && i + kOwn < mine) issue(i + kOwn);  // every lane has read the slot
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) st.l[e] += __shfl_xor_sync(0xffffffffu, st.l[e], o);
    const int g = lane >> 2, t2 = (lane & 3) * 2;
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        mo[(warp * kCols + t2 + (e & 1)) * kKv8Dim + 16 * c + 2 * g + (e >> 1)] = st.o[c][e];
    if (g == 0)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float* d = ms + (warp * kCols + t2 + e) * 3;
        d[0] = st.m[e], d[1] = st.bo[e], d[2] = st.l[e];
      }
    __syncthreads();
    for (int idx = threadIdx.x; idx < min(kCols, ncols - cb) * kKv8Dim; idx += kWarps * 32) {
      const int col = idx / kKv8Dim, d = idx % kKv8Dim;
      float M = -CUDART_INF_F, B = -CUDART_INF_F;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        M = fmaxf(M, ms[(w * kCols + col) * 3]);
        B = fmaxf(B, ms[(w * kCols + col) * 3 + 1]);
      }
      float acc = 0.f, L = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float* x = ms + (w * kCols + col) * 3;
        const float fm = x[0] == -CUDART_INF_F ? 1.f : ex2(x[0] - M), fb = x[1] == -CUDART_INF_F ? 1.f : ex2(x[1] - B);
        L += x[2] * fm;
        acc += mo[(w * kCols + col) * kKv8Dim + d] * fb;
      }
      const int gc = cb + col;
      const int row = row0 + gc / G, head = kvh * G + gc % G;
      if (a.splits == 1) {
        const float o = L == 0.f ? 0.f : acc / L * ex2((B == -CUDART_INF_F ? 0.f : B) - (M == -CUDART_INF_F ? 0.f : M) - kPBias);
        a.out[static_cast<int64_t>(row) * a.out_stride + head * kKv8Dim + d] = __float2bfloat16(o);
      } else {
        const int64_t part = (static_cast<int64_t>(row) * a.n_q_heads + head) * a.splits + blockIdx.x;
        a.ws_o[part * kKv8Dim + d] = acc;
        if (d == 0) {
          float* x = a.ws_ml + part * 4;
          x[0] = M, x[1] = B, x[2] = L;
        }
      }
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kKv8Dim) kv8_combine_kernel(const Kv8AttnArgs a) {
  const int head = blockIdx.x, row = blockIdx.y, d = threadIdx.x;
  const int64_t base = (static_cast<int64_t>(row) * a.n_q_heads + head) * a.splits;
  float M = -CUDART_INF_F, B = -CUDART_INF_F;
  for (int s = 0; s < a.splits; ++s) {
    M = fmaxf(M, a.ws_ml[(base + s) * 4]);
    B = fmaxf(B, a.ws_ml[(base + s) * 4 + 1]);
  }
  float acc = 0.f, L = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float* x = a.ws_ml + (base + s) * 4;
    L += x[2] * (x[0] == -CUDART_INF_F ? 1.f : ex2(x[0] - M));
    acc += a.ws_o[(base + s) * kKv8Dim + d] * (x[1] == -CUDART_INF_F ? 1.f : ex2(x[1] - B));
  }
  const float o = L == 0.f ? 0.f : acc / L * ex2((B == -CUDART_INF_F ? 0.f : B) - (M == -CUDART_INF_F ? 0.f : M) - kPBias);
  a.out[static_cast<int64_t>(row) * a.out_stride + head * kKv8Dim + d] = __float2bfloat16(o);
}

}  // namespace

int kv8_attention(const Kv8AttnArgs& a, cudaStream_t stream) {
  const int items = a.tiles ? a.num_tiles : a.num_seqs;
  if (items <= 0) return 0;
  if (int e = ensure_smem_attr(reinterpret_cast<const void*>(kv8_attn_kernel), kSmem)) return e;
  kv8_attn_kernel<<<dim3(a.splits, a.n_kv_heads, items), kWarps * 32, kSmem, stream>>>(a);
  if (a.splits > 1) kv8_combine_kernel<<<dim3(a.n_q_heads, a.num_rows), kKv8Dim, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace lakeb
