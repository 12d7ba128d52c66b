// The 8-bit KV arena: uint8 [num_blocks, layers, kv_heads, 2 (K, V), 16 * 128 + 16].
//
// For one page, layer, head and side: 16 rows of 128 e4m3 codes, then the page's scale line, one
// power-of-two byte b per token (E8M0): value = code * 2^(b - 127); b = 255 marks a row that held
// an infinity or a NaN (its codes are 0, it reads back as NaN).
//
//  * A row's bytes are a function of the row alone (no scale shared between tokens that could
//    grow as a page fills): pages are content-addressed by their tokens and shared by prefix, so a
//    page filled token by token, in one chunk, or after a rejected draft has the same bytes.
//  * Powers of two: dequantising is exact in fp16 and bf16 products, nothing is rounded twice.
//  * Row t keeps its 16-byte chunk c at chunk c ^ (t & 7), so the bytes as they lie in memory are
//    free of bank conflicts for ldmatrix, and K, V and both scale lines of a page and head arrive
//    in shared memory with one bulk copy of 4128 contiguous bytes (129 sectors of 32 bytes).
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"
#include "lakeb_kernels.h"

namespace lakeb {

constexpr int kKv8Page = 16;
constexpr int kKv8Dim = 128;
constexpr int kKv8Side = kKv8Page * kKv8Dim + kKv8Page;  // 2064 bytes: codes, scale line
constexpr int kKv8Head = 2 * kKv8Side;                   // K and V of one page and head

// Byte offset of 16-byte chunk `c` of token `t` inside one side.
__host__ __device__ __forceinline__ int kv8_chunk(int t, int c) { return t * kKv8Dim + ((c ^ (t & 7)) << 4); }

// Scale byte of a row from the largest |x| bit pattern of its elements (as integers, so that NaN
// and infinity sort above every finite value): the smallest e >= -126 with amax <= 448 * 2^e.
__device__ __forceinline__ int kv8_scale_byte(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return 255;
  const int e = static_cast<int>(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, -126) + 127;
}
// 2^(127 - b): the factor that brings a row into e4m3's range (0 for a NaN row: codes 0).
__device__ __forceinline__ float kv8_inv_scale(int b) {
  return b == 255 ? 0.f : __uint_as_float(static_cast<uint32_t>(254 - b) << 23);
}
// 2^(b - 127); NaN for b = 255 (b = 0 counts as 0: an arena that was never written reads as zeros).
__device__ __forceinline__ float kv8_scale(int b) {
  return __uint_as_float(b == 255 ? 0x7fffffffu : static_cast<uint32_t>(b) << 23);
}

// A query tile names a sequence and up to kKv8TileRows rows of the call (otherwise it is reported and
// skipped).
__device__ __forceinline__ bool kv8_tile_ok(const Kv8AttnArgs& a, const int4& t) {
  const bool ok = t.z <= 0 || (t.x >= 0 && t.x < a.num_seqs && t.y >= 0 && t.y < a.num_rows && t.z <= kKv8TileRows &&
                               t.z <= a.num_rows - t.y && t.w >= 0 && t.w < (1 << 30));
  if (!ok) record_error(a.status, kErrBounds);
  return ok;
}

// A sequence's length in the pages that its block table holds; one past them, or negative, is reported and cut off.
__device__ __forceinline__ int kv8_seq_len(const Kv8AttnArgs& a, int seq) {
  const int len = a.seq_lens[seq], most = a.max_blocks * kKv8Page;
  if (len < 0 || len > most) record_error(a.status, kErrBounds);
  return max(0, min(len, most));
}

// kv8_prefill: how the 128 rows of a CTA's two products are filled from a tile's query rows and the G query heads
// of a KV head: with `pack` heads of a row side by side, pack the largest power of two in G, so that a
// tile of few rows fills them too and a CTA's keys end close behind its rows. The two products then
// take consecutive blocks of rows; with an odd G they take all the tile's rows of two heads. A launch
// that leaves more than half of the SMs idle has one product in a CTA, and twice the CTAs.
struct Kv8Packing {
  int pack, shift, rows;  // heads of a row, log2; rows of a product
  int subs;               // CTAs that share a tile's rows
  int units;              // CTAs of a tile and KV head
};
__host__ __device__ __forceinline__ Kv8Packing kv8_packing(int G, int products) {
  Kv8Packing p;
  p.shift = 0;
  while (p.shift < 7 && !(G >> p.shift & 1)) ++p.shift;
  p.pack = 1 << p.shift;
  p.rows = kKv8TileRows >> p.shift;
  p.subs = p.pack > 1 ? p.pack / products : 1;
  p.units = p.pack > 1 ? G / products : (G + products - 1) / products;
  return p;
}
// Which kernel a tile belongs to when both run (few_rows > 0; both find the same). In units of 128 keys of
// a kv8_prefill CTA (2.3 us; its start and end cost three), a tile of few rows takes `own` of time in
// kv8_prefill, beside the others, whose CTAs take their work / sms. In kv8_attention it takes the whole GPU
// for own * groups / sms, groups of 24 columns, and four for start and join. So tiles of few rows go there
// that are longer than all of that together.
// Measured, 64 query and 8 KV heads: chunks of 42 to 1500 rows take 106 us, with one of 17 rows behind 6001
// keys 131 us in kv8_prefill, 144 in both; two of 32 rows behind 3000 keys 56 us in kv8_prefill, 72 in
// kv8_attention.
constexpr int kKv8Ranked = 256;  // tiles that are looked at: in a call of more the rest count no work, and tiles run in their order
constexpr int kKv8CtaCost = 3;
__device__ __forceinline__ int kv8_tile_keys(const Kv8AttnArgs& a, const int4& t) {
  return max(0, min(min(t.w + t.z, a.seq_lens[t.x]), a.max_blocks * kKv8Page));
}
// A tile's work per KV head (cut off where a sum of kKv8Ranked could pass 32 bits).
__device__ __forceinline__ int kv8_tile_work(const Kv8AttnArgs& a, const Kv8Packing& pk, const int4& t, int keys) {
  int n = pk.units;
  if (t.z <= a.few_rows) n = (t.z * (a.n_q_heads / a.n_kv_heads) + 23) / 24;
  else if (pk.pack > 1) n = pk.units / pk.subs * ((t.z + a.products * pk.rows - 1) / (a.products * pk.rows));
  return min(((keys + 127) >> 7) + kKv8CtaCost, (1 << 22) / n) * n;
}
__device__ __forceinline__ bool kv8_tile_is_few(const Kv8AttnArgs& a, const int4& t, int keys, int64_t work) {
  const int own = ((keys + 127) >> 7) + kKv8CtaCost;
  return t.z <= a.few_rows && static_cast<int64_t>(own - 4) * a.sms > work;
}

// The kernels of this cache are launched ahead of the end of the one before (launch_ahead), so that their
// start does not add to a chain of short ones. Each calls after_previous before it reads anything but its
// arguments: then all that ran before is done, and the kernel after this one may come ahead too.
__device__ __forceinline__ void after_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
}
template <class Kernel, class... Args>
int launch_ahead(Kernel kernel, unsigned grid, int threads, int smem, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Two fp32 -> two e4m3 codes (round to nearest even), lo in the low byte.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two e4m3 codes (low half of x) -> f16x2, exact.
__device__ __forceinline__ uint32_t f16x2_of_e4m3(uint16_t x) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(x));
  return r;
}
__device__ __forceinline__ uint32_t f16x2_lo(uint32_t x) { return f16x2_of_e4m3(static_cast<uint16_t>(x)); }
__device__ __forceinline__ uint32_t f16x2_hi(uint32_t x) { return f16x2_of_e4m3(static_cast<uint16_t>(x >> 16)); }

}  // namespace lakeb
