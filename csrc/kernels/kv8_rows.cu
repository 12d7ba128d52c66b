// Rows in and out of the 8-bit KV arena (kv8.cuh), and the tables of an engine step.
//
//  * kv8_write: bf16 K and V rows -> e4m3 codes and scale bytes at the rows' slots.
//  * kv8_read: the cached rows of a list of slots -> dense bf16 rows.
//  * step_tables: positions, slots, query starts, block tables and query tiles from request lengths.
//
// The first two move bytes: 258 + 512 per (row, head), against which 256 conversions are nothing. A
// warp takes one row and up to four heads at a time, half of it K and half V, 16 bytes of bf16 and 8
// bytes of codes per lane and head: both sides of a head move as whole 128- and 256-byte rows, and
// four independent loads per lane are in flight behind the one load of the slot. Measured: 16384 rows of
// 8 heads in 22.8 us (4.4 TB/s read and written, 0.68 of the copy rate; codes are written in 128-byte
// rows), 24 prefixes of 33 to 4097 tokens read in 23.7 us (0.86); a few rows are a launch of 3.3 us.
// step_tables is one launch and three dependent loads: 3.9 us for 256 decode rows, 5.3 us for a step of
// 8448 rows.
#include "common.cuh"
#include "kv8.cuh"
#include "lakeb_kernels.h"
#include "tma_host.h"

namespace lakeb {
namespace {

constexpr int kRowWarps = 8;
constexpr int kHeads = 4;  // of one warp's turn

// Warp `u` of the launch: row and first head.
__device__ __forceinline__ bool row_unit(const Kv8RowArgs& a, uint32_t u, int& row, int& head, int64_t& slot) {
  const uint32_t groups = (a.heads + kHeads - 1) / kHeads;
  row = static_cast<int>(u / groups);
  head = static_cast<int>(u % groups) * kHeads;
  if (row >= a.rows) return false;
  slot = a.slots[row];
  if (slot >= a.num_blocks * kKv8Page) {
    if ((threadIdx.x & 31) == 0) record_error(a.status, kErrBounds);
    slot = -1;
  }
  return true;
}

__global__ void __launch_bounds__(kRowWarps * 32) kv8_write_kernel(const Kv8RowArgs a) {
  after_previous();
  const int lane = threadIdx.x & 31, side = lane >> 4, l = lane & 15;
  int row, head;
  int64_t slot;
  if (!row_unit(a, blockIdx.x * kRowWarps + (threadIdx.x >> 5), row, head, slot) || slot < 0) return;
  const __nv_bfloat16* src = (side ? a.v + row * a.v_stride : a.k + row * a.k_stride) + head * kKv8Dim + l * 8;
  const int t = static_cast<int>(slot & (kKv8Page - 1));
  uint8_t* dst = a.arena + (slot / kKv8Page) * a.block_bytes + a.layer_offset + head * kKv8Head + side * kKv8Side;
  const int n = min(kHeads, a.heads - head);
  uint4 x[kHeads];
#pragma unroll
  for (int h = 0; h < kHeads; ++h)
    x[h] = h < n ? __ldcs(reinterpret_cast<const uint4*>(src + h * kKv8Dim)) : make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    const uint32_t w[4] = {x[h].x, x[h].y, x[h].z, x[h].w};
    uint32_t top = 0;  // |bf16| as integers, both halves of each word
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
    top = __reduce_max_sync(side ? 0xffff0000u : 0x0000ffffu, top);
    const int b = kv8_scale_byte(top << 16);
    const float f = kv8_inv_scale(b);
    uint32_t q[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float x0 = __uint_as_float(w[2 * i] << 16) * f, x1 = __uint_as_float(w[2 * i] & 0xffff0000u) * f;
      const float x2 = __uint_as_float(w[2 * i + 1] << 16) * f, x3 = __uint_as_float(w[2 * i + 1] & 0xffff0000u) * f;
      q[i] = e4m3x2(x0, x1) | e4m3x2(x2, x3) << 16;
    }
    if (b == 255) q[0] = q[1] = 0;
    if (h < n) {
      *reinterpret_cast<uint2*>(dst + h * kKv8Head + kv8_chunk(t, l >> 1) + (l & 1) * 8) = make_uint2(q[0], q[1]);
      if (l == 0) dst[h * kKv8Head + kKv8Page * kKv8Dim + t] = static_cast<uint8_t>(b);
    }
  }
}

__global__ void __launch_bounds__(kRowWarps * 32) kv8_read_kernel(const Kv8RowArgs a) {
  after_previous();
  const int lane = threadIdx.x & 31, side = lane >> 4, l = lane & 15;
  int row, head;
  int64_t slot;
  if (!row_unit(a, blockIdx.x * kRowWarps + (threadIdx.x >> 5), row, head, slot)) return;
  const int n = min(kHeads, a.heads - head);
  const int t = static_cast<int>(slot & (kKv8Page - 1));
  const uint8_t* src =
      a.arena + (max(slot, int64_t(0)) / kKv8Page) * a.block_bytes + a.layer_offset + head * kKv8Head + side * kKv8Side;
  uint2 q[kHeads];
  int b[kHeads];
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    const bool real = slot >= 0 && h < n;
    q[h] = real ? *reinterpret_cast<const uint2*>(src + h * kKv8Head + kv8_chunk(t, l >> 1) + (l & 1) * 8)
                : make_uint2(0, 0);
    b[h] = real ? src[h * kKv8Head + kKv8Page * kKv8Dim + t] : 0;
  }
  __nv_bfloat16* dst = (side ? a.v_out + row * a.v_stride : a.k_out + row * a.k_stride) + head * kKv8Dim + l * 8;
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    const float f = kv8_scale(b[h]);
    auto two = [&](uint32_t c) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&c));
      return pack_bf16x2(v.x * f, v.y * f);
    };
    if (h < n)
      *reinterpret_cast<uint4*>(dst + h * kKv8Dim) =
          make_uint4(two(f16x2_lo(q[h].x)), two(f16x2_hi(q[h].x)), two(f16x2_lo(q[h].y)), two(f16x2_hi(q[h].y)));
  }
}

int64_t row_grid(const Kv8RowArgs& a) {
  return (static_cast<int64_t>(a.rows) * ((a.heads + kHeads - 1) / kHeads) + kRowWarps - 1) / kRowWarps;
}

// ------------------------------------------------------------------ step tables
constexpr int kTabThreads = 256;

// Exclusive prefix sums of the new tokens and of the query tiles of every sequence, in shared
// memory of every CTA: a step has at most a few hundred sequences, so scanning them again costs
// less than a second launch. Rows of all parts are then found by binary search.
__global__ void __launch_bounds__(kTabThreads) step_tables_kernel(const StepTableArgs a) {
  extern __shared__ int sm[];
  int* start = sm;                    // [seqs + 1]
  int* first = sm + a.num_seqs + 1;   // [seqs + 1]
  __shared__ int part[2][kTabThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool lead = blockIdx.x == 0;
  int base_n = 0, base_t = 0;
  after_previous();
  for (int s0 = 0; s0 < a.num_seqs; s0 += kTabThreads) {
    const int s = s0 + tid;
    const int raw = s < a.num_seqs ? a.new_lens[s] : 0;
    // a length that no table has room for is reported with the totals: cut off here, sums stay in 32 bits
    const int n = min(max(raw, 0), a.max_tokens + 1), t = s >= a.num_decode ? (n + a.tile - 1) / a.tile : 0;
    if (raw < 0 && lead) record_error(a.status, kErrBadArg);
    int cn = n, ct = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int pn = __shfl_up_sync(0xffffffffu, cn, o), pt = __shfl_up_sync(0xffffffffu, ct, o);
      if (lane >= o) cn += pn, ct += pt;
    }
    if (lane == 31) part[0][warp] = cn, part[1][warp] = ct;
    __syncthreads();
    int bn = base_n, bt = base_t;
    for (int w = 0; w < kTabThreads / 32; ++w) {
      if (w < warp) bn += part[0][w], bt += part[1][w];
      base_n += part[0][w];
      base_t += part[1][w];
    }
    if (s < a.num_seqs) start[s] = bn + cn - n, first[s] = bt + ct - t;
    __syncthreads();
  }
  if (tid == 0) start[a.num_seqs] = base_n, first[a.num_seqs] = base_t;
  __syncthreads();

  const int total = base_n, tiles = base_t;
  const int stride = gridDim.x * kTabThreads, gid = blockIdx.x * kTabThreads + tid;
  if (lead && tid == 0) {
    a.counts[0] = total;
    a.counts[1] = tiles;
    if (total > a.max_tokens || tiles > a.max_tiles) record_error(a.status, kErrBadArg);
  }
  // the last sequence whose prefix is <= i (empty ones share a prefix: the search ends past them)
  auto find = [&](const int* pre, int i) {
    int lo = 0, hi = a.num_seqs;  // pre[lo] <= i < pre[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= i) lo = mid; else hi = mid;
    }
    return lo;
  };
  auto row_of = [&](int s) {
    const int r = a.rows[s];
    if (r >= 0 && r < a.num_rows) return r;
    record_error(a.status, kErrBounds);
    return -1;
  };
  // (a context past 2^30 tokens is reported with its pages: cut off, so that lengths stay in 32 bits)
  auto context = [&](int s) { return min(a.context_lens[s], 1 << 30); };
  for (int s = gid; s <= a.num_seqs; s += stride) {
    a.query_start[s] = start[s];
    if (s < a.num_seqs) a.seq_lens[s] = context(s) + (start[s + 1] - start[s]);
  }
  for (int i = gid; i < a.max_tokens; i += stride) {
    int pos = 0;
    int64_t slot = -1;
    if (i < total) {
      const int s = find(start, i), r = row_of(s);
      pos = context(s) + (i - start[s]);
      const int p = pos / a.block_size;
      if (r >= 0 && pos >= 0 && p < a.max_blocks) {
        const int page = a.pages[static_cast<int64_t>(r) * a.pages_stride + p];
        if (page >= 0) slot = static_cast<int64_t>(page) * a.block_size + (pos - p * a.block_size);
      }
      if (slot < 0) record_error(a.status, kErrBounds);
    }
    a.positions[i] = pos;
    a.slots[i] = slot;
  }
  for (int i = gid; i < a.max_tiles; i += stride) {
    int4 t = make_int4(0, 0, 0, 0);
    if (i < tiles) {
      const int s = find(first, i), at = (i - first[s]) * a.tile;
      t = make_int4(s, start[s] + at, min(a.tile, start[s + 1] - start[s] - at), context(s) + at);
    }
    a.tiles[i] = t;
  }
  // block tables: a CTA per sequence, entries past the sequence's pages 0
  for (int s = blockIdx.x; s < a.num_seqs; s += gridDim.x) {
    const int ctx = context(s), len = ctx + (start[s + 1] - start[s]);
    const int need = len > 0 ? (len - 1) / a.block_size + 1 : 0, nb = min(need, a.max_blocks);
    const int r = row_of(s);
    if (tid == 0 && (ctx < 0 || need > a.max_blocks)) record_error(a.status, kErrBounds);
    const int* src = a.pages + static_cast<int64_t>(max(r, 0)) * a.pages_stride;
    int* dst = a.block_tables + static_cast<int64_t>(s) * a.max_blocks;
    for (int p = tid; p < a.max_blocks; p += kTabThreads) {
      int page = 0;
      if (r >= 0 && p < nb) {
        page = src[p];
        if (page < 0) {
          record_error(a.status, kErrBounds);
          page = 0;
        }
      }
      dst[p] = page;
    }
  }
}

}  // namespace

int kv8_write(const Kv8RowArgs& a, cudaStream_t stream) {
  if (a.rows <= 0) return 0;
  if (row_grid(a) * kRowWarps >= (int64_t(1) << 32) || row_grid(a) >= (int64_t(1) << 31)) return -1;
  return launch_ahead(kv8_write_kernel, static_cast<unsigned>(row_grid(a)), kRowWarps * 32, 0, stream, a);
}

int kv8_read(const Kv8RowArgs& a, cudaStream_t stream) {
  if (a.rows <= 0) return 0;
  if (row_grid(a) * kRowWarps >= (int64_t(1) << 32) || row_grid(a) >= (int64_t(1) << 31)) return -1;
  return launch_ahead(kv8_read_kernel, static_cast<unsigned>(row_grid(a)), kRowWarps * 32, 0, stream, a);
}

int step_tables(const StepTableArgs& a, cudaStream_t stream) {
  const int smem = 2 * (a.num_seqs + 1) * static_cast<int>(sizeof(int));
  if (int e = ensure_smem_attr(reinterpret_cast<const void*>(step_tables_kernel), kStepTableMaxSeqs * 8 + 8)) return e;
  int grid = (a.max_tokens + kTabThreads - 1) / kTabThreads;
  if (a.num_seqs > grid) grid = a.num_seqs;
  if (grid > 2 * num_sms()) grid = 2 * num_sms();
  if (grid < 1) grid = 1;
  return launch_ahead(step_tables_kernel, grid, kTabThreads, smem, stream, a);
}

}  // namespace lakeb
