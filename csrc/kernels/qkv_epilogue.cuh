// QKV projection epilogue shared by the single-SM and the two-SM tcgen05 GEMMs: for one
// 128-wide head of one accumulator row, optional per-head RMSNorm (Qwen3), RoPE, and the
// stores (q rows to C; k / v rows into the paged KV arena and, for PD-split, into the decode
// instance's arena through its peer mapping).
#pragma once

#include "common.cuh"
#include "kv8.cuh"
#include "lakeb_kernels.h"

namespace lakeb {
namespace {

__device__ __forceinline__ void store_bf16x32(__nv_bfloat16* dst, const float* v) {
  uint4* d = reinterpret_cast<uint4*>(dst);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint4 u;
    u.x = pack_bf16x2(v[8 * i + 0], v[8 * i + 1]);
    u.y = pack_bf16x2(v[8 * i + 2], v[8 * i + 3]);
    u.z = pack_bf16x2(v[8 * i + 4], v[8 * i + 5]);
    u.w = pack_bf16x2(v[8 * i + 6], v[8 * i + 7]);
    d[i] = u;
  }
}

// Warp-collective store of one 64-byte piece per lane (32 fp32 -> bf16) to `dst` (this lane's
// row; nullptr: no store). The pieces pass through `stage` (2 KB of this warp's shared memory)
// so that each store instruction writes 8 rows x 64 contiguous bytes instead of 32 rows x 16
// bytes: over NVLink (peer arenas) that is 8 runs of 64 bytes rather than 32 scattered 16-byte
// writes. Chunk c of row r sits at r*4 + ((c + r/2) & 3) so both the row-wise writes and the
// chunk-wise reads are free of bank conflicts. Every lane of the warp must call it.
__device__ __forceinline__ void warp_store_rows64(uint4* stage, __nv_bfloat16* dst, const float* v, int lane) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint4 u;
    u.x = pack_bf16x2(v[8 * c + 0], v[8 * c + 1]);
    u.y = pack_bf16x2(v[8 * c + 2], v[8 * c + 3]);
    u.z = pack_bf16x2(v[8 * c + 4], v[8 * c + 5]);
    u.w = pack_bf16x2(v[8 * c + 6], v[8 * c + 7]);
    stage[lane * 4 + ((c + (lane >> 1)) & 3)] = u;
  }
  __syncwarp();
  const unsigned long long mine = reinterpret_cast<unsigned long long>(dst);
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int r = it * 8 + (lane >> 2), c = lane & 3;
    const unsigned long long d = __shfl_sync(0xffffffffu, mine, r);
    const uint4 u = stage[r * 4 + ((c + (r >> 1)) & 3)];
    if (d) reinterpret_cast<uint4*>(d)[c] = u;
  }
  __syncwarp();
}

__device__ __forceinline__ __nv_bfloat16* kv_ptr(const KVArenaView& kv, int64_t slot, int head, int which) {
  const int64_t blk = slot / kv.block_size;
  const int64_t off = slot - blk * kv.block_size;
  return kv.base + blk * kv.block_stride + kv.layer_offset + which * kv.kv_stride + head * kv.head_stride +
         off * 128;
}

// K (roped, optionally normed before) or V of one head and row into an 8-bit arena: the row's scale
// needs its largest element first, so K goes back into the accumulators as it is found and both are read
// a second time (a TMEM load costs less than holding 128 results, and far less than each lane's 512
// bytes of rotations again). The row is quantised from fp32; the codes go to token t of the page side
// `row` of this arena and to the peer's (nullptr: neither). Measured, 4096 -> 6144 with 32 query and 8 KV
// heads, 80 / 512 / 8192 rows: 32.8 / 45.1 / 295 us, as with a bf16 arena (45 / 74 / 355 with the
// rotations read twice).
// Not inlined: the bf16 epilogue keeps its registers.
__device__ __noinline__ void qkv_head_kv8(uint32_t tbase, bool is_k, uint8_t* row, uint8_t* peer_row, int t, int peer_t,
                                          const float4* cs, const __nv_bfloat16* nw, float inv) {
  uint32_t top = 0;
#pragma unroll 1
  for (int half = 0; half < 2; ++half) {  // elements 32 * half.., 64 + 32 * half..
    uint32_t r1[32], r2[32];
    tmem_ld32(tbase + half * 32, r1);
    tmem_ld32(tbase + 64 + half * 32, r2);
    tmem_ld_wait();
    if (is_k) {
#pragma unroll
      for (int j = 0; j < 32; j += 2) {
        const float4 c = cs[half * 16 + j / 2];  // two rotations
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x1 = __uint_as_float(r1[j + e]), x2 = __uint_as_float(r2[j + e]);
          if (nw) {
            x1 *= inv * __bfloat162float(nw[half * 32 + j + e]);
            x2 *= inv * __bfloat162float(nw[64 + half * 32 + j + e]);
          }
          const float co = e ? c.z : c.x, si = e ? c.w : c.y;
          r1[j + e] = __float_as_uint(x1 * co - x2 * si);
          r2[j + e] = __float_as_uint(x2 * co + x1 * si);
        }
      }
      tmem_st32(tbase + half * 32, r1);
      tmem_st32(tbase + 64 + half * 32, r2);
    }
#pragma unroll
    for (int j = 0; j < 32; ++j) top = max(top, max(r1[j] & 0x7fffffffu, r2[j] & 0x7fffffffu));
  }
  tmem_st_wait();
  const int b = kv8_scale_byte(top);
  const float f = kv8_inv_scale(b);
#pragma unroll 1
  for (int half = 0; half < 2; ++half) {
    uint32_t r1[32], r2[32];
    __syncwarp();  // the stores before are each lane's own
    tmem_ld32(tbase + half * 32, r1);
    tmem_ld32(tbase + 64 + half * 32, r2);
    tmem_ld_wait();
    auto two = [&](const uint32_t (&r)[32], int j) {
      return e4m3x2(__uint_as_float(r[j]) * f, __uint_as_float(r[j + 1]) * f);
    };
    uint32_t q[2][8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      q[0][j] = two(r1, 4 * j) | two(r1, 4 * j + 2) << 16;
      q[1][j] = two(r2, 4 * j) | two(r2, 4 * j + 2) << 16;
      if (b == 255) q[0][j] = q[1][j] = 0;
    }
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      uint8_t* side = d ? peer_row : row;
      const int tok = d ? peer_t : t;
      if (!side) continue;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        *reinterpret_cast<uint4*>(side + kv8_chunk(tok, (c >> 1) * 4 + half * 2 + (c & 1))) =
            make_uint4(q[c >> 1][4 * (c & 1)], q[c >> 1][4 * (c & 1) + 1], q[c >> 1][4 * (c & 1) + 2],
                       q[c >> 1][4 * (c & 1) + 3]);
      if (half == 0) side[kKv8Page * kKv8Dim + tok] = static_cast<uint8_t>(b);
    }
  }
}

// Head `head` of accumulator row `row` (this thread's TMEM lane; `tbase` addresses the head's
// 128 fp32 columns). Every lane of the warp calls it (the TMEM loads are warp-aligned). With
// `stage` (2 KB of this warp's shared memory) the peer-arena K/V stores are coalesced per warp.
__device__ __forceinline__ void qkv_head_epilogue(const GemmArgs& p, uint32_t tbase, int head, int row, bool row_ok,
                                                  uint4* stage = nullptr) {
  const int lane = threadIdx.x & 31;
  const bool is_q = head < p.n_q_heads;
  const bool is_k = !is_q && head < p.n_q_heads + p.n_kv_heads;
  int pos = 0;
  int64_t slot = -1, pslot = -1;
  if (row_ok) {
    pos = p.positions[row];
    if (!is_q) {
      slot = p.slots ? p.slots[row] : -1;
      if ((p.peer_kv.base || p.peer_kv.base8) && p.peer_slots) pslot = p.peer_slots[row];
      // debug build: a slot past the arena is reported and its store skipped
      if (slot >= 0 && !in_bounds(p.kv.num_slots <= 0 || slot < p.kv.num_slots, p.status)) slot = -1;
      if (pslot >= 0 && !in_bounds(p.peer_kv.num_slots <= 0 || pslot < p.peer_kv.num_slots, p.status))
        pslot = -1;
    }
  }
  if (p.kv.base8 && !is_q) {
    // 8-bit arena: a slot past it is reported and skipped
    if (slot >= p.kv.num_slots) record_error(p.status, kErrBounds), slot = -1;
    if (p.peer_kv.base8 && pslot >= p.peer_kv.num_slots) record_error(p.status, kErrBounds), pslot = -1;
    float inv = 1.f;
    if (is_k && p.k_norm_w) {
      float ss = 0.f;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t r[32];
        tmem_ld32(tbase + c * 32, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) ss += __uint_as_float(r[j]) * __uint_as_float(r[j]);
      }
      inv = rsqrtf(ss * (1.f / 128.f) + p.qk_eps);
    }
    const int64_t in_page = (head - p.n_q_heads - (is_k ? 0 : p.n_kv_heads)) * kKv8Head + (is_k ? 0 : kKv8Side);
    uint8_t* mine = slot < 0 ? nullptr
                             : p.kv.base8 + (slot / kKv8Page) * p.kv.block_stride + p.kv.layer_offset + in_page;
    uint8_t* theirs = pslot < 0 || !p.peer_kv.base8 ? nullptr
                                                    : p.peer_kv.base8 + (pslot / kKv8Page) * p.peer_kv.block_stride +
                                                          p.peer_kv.layer_offset + in_page;
    // (a row outside the matrix has slot -1 and position 0: it stores nothing)
    qkv_head_kv8(tbase, is_k, mine, theirs, static_cast<int>(slot & (kKv8Page - 1)),
                 static_cast<int>(pslot & (kKv8Page - 1)),
                 reinterpret_cast<const float4*>(p.rope_cs + static_cast<int64_t>(pos) * 64),
                 is_k ? p.k_norm_w : nullptr, inv);
    return;
  }
  if (is_q || is_k) {
    const int kvh = head - p.n_q_heads;
    // per-head RMSNorm before RoPE (Qwen3): one pass over the head's 128 accumulators first
    const __nv_bfloat16* nw = is_q ? p.q_norm_w : p.k_norm_w;
    float inv = 1.f;
    if (nw) {
      float ss = 0.f;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t r[32];
        tmem_ld32(tbase + c * 32, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) ss += __uint_as_float(r[j]) * __uint_as_float(r[j]);
      }
      inv = rsqrtf(ss * (1.f / 128.f) + p.qk_eps);
    }
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
      uint32_t r1[32], r2[32];
      tmem_ld32(tbase + half * 32, r1);
      tmem_ld32(tbase + 64 + half * 32, r2);
      tmem_ld_wait();
      float o1[32], o2[32];
      if (row_ok) {
        const float2* cs = p.rope_cs + static_cast<int64_t>(pos) * 64 + half * 32;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const float2 c = cs[j];
          float x1 = __uint_as_float(r1[j]);
          float x2 = __uint_as_float(r2[j]);
          if (nw) {
            x1 *= inv * __bfloat162float(nw[half * 32 + j]);
            x2 *= inv * __bfloat162float(nw[64 + half * 32 + j]);
          }
          o1[j] = x1 * c.x - x2 * c.y;
          o2[j] = x2 * c.x + x1 * c.y;
        }
        if (is_q) {
          __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(p.C) + row * p.ldc + head * 128;
          store_bf16x32(dst + half * 32, o1);
          store_bf16x32(dst + 64 + half * 32, o2);
        } else {
          if (slot >= 0) {
            __nv_bfloat16* dst = kv_ptr(p.kv, slot, kvh, 0);
            store_bf16x32(dst + half * 32, o1);
            store_bf16x32(dst + 64 + half * 32, o2);
          }
          if (pslot >= 0 && !stage) {
            __nv_bfloat16* dst = kv_ptr(p.peer_kv, pslot, kvh, 0);
            store_bf16x32(dst + half * 32, o1);
            store_bf16x32(dst + 64 + half * 32, o2);
          }
        }
      }
      if (is_k && stage && p.peer_kv.base) {  // warp-uniform: the head is the same for every lane
        __nv_bfloat16* dst = pslot >= 0 ? kv_ptr(p.peer_kv, pslot, kvh, 0) : nullptr;
        warp_store_rows64(stage, dst ? dst + half * 32 : nullptr, o1, lane);
        warp_store_rows64(stage, dst ? dst + 64 + half * 32 : nullptr, o2, lane);
      }
    }
  } else {
    const int kvh = head - p.n_q_heads - p.n_kv_heads;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
      uint32_t r[32];
      tmem_ld32(tbase + c * 32, r);
      tmem_ld_wait();
      float v[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
      if (row_ok) {
        if (slot >= 0) store_bf16x32(kv_ptr(p.kv, slot, kvh, 1) + c * 32, v);
        if (pslot >= 0 && !stage) store_bf16x32(kv_ptr(p.peer_kv, pslot, kvh, 1) + c * 32, v);
      }
      if (stage && p.peer_kv.base)
        warp_store_rows64(stage, pslot >= 0 ? kv_ptr(p.peer_kv, pslot, kvh, 1) + c * 32 : nullptr, v, lane);
    }
  }
}

}  // namespace
}  // namespace lakeb
