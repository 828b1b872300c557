// Page moves of a paged cache: whole pages copied inside a pool (or into another of the same page shape), and
// a fragmented pool compacted.
//
// A page is a run of `page_bytes` at a fixed stride in each of `planes` arrays (K and V of every layer), so
// the copies know nothing of the element type; an 8-bit cache's scales are a second, small set of runs.
#include "kv8.cuh"

namespace ssd {
namespace {

constexpr int kCopyThreads = 128;

struct PageRuns {
  const char* src;
  char* dst;
  int64_t bytes;                 // of one page in one plane; multiple of `vec`
  int64_t src_plane, dst_plane;  // bytes between planes
};

struct CopyArgs {
  PageRuns data, scales;         // scales.bytes = 0: none
  const int32_t* src_ids;
  const int32_t* dst_ids;
  int64_t src_step, dst_step;    // elements between ids (0: the same id for every pair)
  const int32_t* count;          // pairs on the device, or NULL (= n)
  int n, planes;
  int src_blocks, dst_blocks;
};

// One CTA per (part, pair): a part is kCopyItems vectors a thread out of the pair's pages in all planes, their loads
// in flight together.  Neighbouring CTAs take the same part of neighbouring pairs, so that what is in flight lies close
// together in one plane (742 moves of 36 planes of 8 KB: 85 us where the parts of a pair were neighbours 91, and 80
// with 128 threads for 256; one plane a CTA reached half of that).  Pairs with an id out of range on either side (-1)
// are skipped.  Bound: HBM (1100 pages of 36 planes of 32 KB: 2.6 GB in 387 us, 6.7 TB/s).
constexpr int kCopyItems = 8;

template <typename V>
__global__ void __launch_bounds__(kCopyThreads) page_copy_kernel(const CopyArgs a) {
  pdl_wait();
  pdl_trigger();
  const int i = (int)(blockIdx.x % a.n), part = (int)(blockIdx.x / a.n);
  // ids past the count are read too (they are there) so that the two loads do not wait for each other
  const int s = ld_act(a.src_ids + i * a.src_step), d = ld_act(a.dst_ids + i * a.dst_step);
  if (a.count && i >= ld_act(a.count)) return;
  if ((unsigned)s >= (unsigned)a.src_blocks || (unsigned)d >= (unsigned)a.dst_blocks) return;
  const int64_t items = a.data.bytes / (int64_t)sizeof(V), total = items * a.planes;
  const char* from = a.data.src + s * a.data.bytes;
  char* to = a.data.dst + d * a.data.bytes;
  if (from == to && a.data.src == a.data.dst) return;
  const int64_t k0 = (int64_t)part * (kCopyItems * kCopyThreads) + threadIdx.x;
  V x[kCopyItems];
  int64_t at[kCopyItems];
#pragma unroll
  for (int q = 0; q < kCopyItems; ++q) {
    const int64_t k = k0 + q * kCopyThreads;
    at[q] = -1;
    if (k < total) {
      const int plane = total <= 0xffffffffll ? (int)((uint32_t)k / (uint32_t)items) : (int)(k / items);
      const int64_t off = (k - plane * items) * (int64_t)sizeof(V);
      x[q] = __ldcg(reinterpret_cast<const V*>(from + plane * a.data.src_plane + off));
      at[q] = plane * a.data.dst_plane + off;
    }
  }
#pragma unroll
  for (int q = 0; q < kCopyItems; ++q)
    if (at[q] >= 0) *reinterpret_cast<V*>(to + at[q]) = x[q];
  if (part == 0 && a.scales.bytes) {
    const int per = (int)(a.scales.bytes / 4);
    for (int k = threadIdx.x; k < per * a.planes; k += kCopyThreads) {
      const int plane = k / per, h = k - plane * per;
      reinterpret_cast<float*>(a.scales.dst + plane * a.scales.dst_plane + d * a.scales.bytes)[h] =
          __ldcg(reinterpret_cast<const float*>(a.scales.src + plane * a.scales.src_plane + s * a.scales.bytes) + h);
    }
  }
}

// ---------------------------------------------------------------------------------------- compaction
// U = blocks not on the free list.  The k-th of them at U or above (ascending) moves to the k-th free block
// below U: the fewest moves there can be, and no block is both read and written.  One CTA: the pool's state
// is a few integers per block; each thread owns a run of blocks, ranks come from block-wide scans, and what is
// free or used is kept in shared memory (a byte a block; pools past kFlagCap in the remap array itself).  The
// same CTA then rewrites the tables.  Bound by latency: 7 us with the copies of a pool of 256 blocks, some 10 us of
// the 80 that 3000 blocks of 18 layers take (438 MB moved).
constexpr int kPlanThreads = 1024;
constexpr int kFlagCap = 160 * 1024;

struct TableArgs {
  const int32_t* in;
  int32_t* out;
  const int32_t* lens;
  int rows, max_blocks;
};

struct CompactArgs {
  const int32_t *free_list, *free_top, *ref_counts;
  int32_t *free_list_out, *free_top_out, *ref_counts_out;
  int32_t *remap, *src, *dst, *moves;  // [num_blocks], [num_blocks / 2], [num_blocks / 2], [1]
  int num_blocks;
  TableArgs tables[2];                 // tables that this kernel rewrites (rows = 0: none)
};

__device__ __forceinline__ int2 block_scan2(int2 v, int2* tmp, int2* total) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  int2 x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, x.x, o), b = __shfl_up_sync(0xffffffffu, x.y, o);
    if (lane >= o) { x.x += a; x.y += b; }
  }
  if (lane == 31) tmp[wid] = x;
  __syncthreads();
  if (wid == 0) {
    int2 y = tmp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, y.x, o), b = __shfl_up_sync(0xffffffffu, y.y, o);
      if (lane >= o) { y.x += a; y.y += b; }
    }
    tmp[lane] = y;
  }
  __syncthreads();
  const int2 base = wid ? tmp[wid - 1] : make_int2(0, 0);
  *total = tmp[31];
  __syncthreads();
  return make_int2(base.x + x.x - v.x, base.y + x.y - v.y);  // exclusive
}

// out[b][i] = remap[in[b][i]] for i < lens[b], -1 behind (ids out of range become -1).
__device__ __forceinline__ void remap_entry(const TableArgs& t, int64_t e, const int32_t* remap, int num_blocks) {
  const int b = (int)(e / t.max_blocks), i = (int)(e % t.max_blocks);
  const int blk = i < ld_act(t.lens + b) ? ld_act(t.in + e) : -1;
  t.out[e] = (unsigned)blk < (unsigned)num_blocks ? ld_act(remap + blk) : -1;
}

template <bool SMEM>
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const CompactArgs a) {
  extern __shared__ uint8_t used_s[];
  __shared__ int2 tmp[32];
  pdl_wait();
  const int nb = a.num_blocks, tid = threadIdx.x;
  auto is_used = [&](int i) { return SMEM ? used_s[i] != 0 : a.remap[i] >= 0; };
  for (int i = tid; i < nb; i += kPlanThreads) {
    if (SMEM) used_s[i] = 1;
    else a.remap[i] = i;
  }
  const int top = min(max(ld_act(a.free_top), 0), nb);
  __syncthreads();
  for (int i = tid; i < nb; i += kPlanThreads) {
    const int f = ld_act(a.free_list + i);  // entries past the top are read and dropped
    if (i < top && (unsigned)f < (unsigned)nb) {
      if (SMEM) used_s[f] = 0;
      else a.remap[f] = -1;
    }
  }
  __syncthreads();
  const int per = (nb + kPlanThreads - 1) / kPlanThreads;
  const int i0 = min(nb, tid * per), i1 = min(nb, i0 + per);
  int used = 0;
  for (int i = i0; i < i1; ++i) used += is_used(i);
  int2 total;
  block_scan2(make_int2(used, 0), tmp, &total);
  const int U = total.x;
  // free blocks below U, used blocks at or above it
  int2 mine = make_int2(0, 0);
  for (int i = i0; i < i1; ++i) {
    const bool u = is_used(i);
    mine.x += !u && i < U;
    mine.y += u && i >= U;
  }
  int2 at = block_scan2(mine, tmp, &total);
  for (int i = i0; i < i1; ++i) {
    const bool u = is_used(i);
    if (!u && i < U) a.dst[at.x++] = i;
    if (u && i >= U) a.src[at.y++] = i;
  }
  for (int i = tid; i < nb; i += kPlanThreads) {
    if (SMEM) a.remap[i] = is_used(i) ? i : -1;
    a.free_list_out[i] = i < nb - U ? nb - 1 - i : -1;  // pops hand out U, U + 1, ...
    if (a.ref_counts_out != a.ref_counts) a.ref_counts_out[i] = ld_act(a.ref_counts + i);
  }
  const int n = total.y;  // == total.x: both count U minus the used blocks below U
  if (tid == 0) {
    *a.moves = n;
    *a.free_top_out = nb - U;
  }
  __syncthreads();
  for (int k = tid; k < n; k += kPlanThreads) {
    const int s = a.src[k], d = a.dst[k];
    a.remap[s] = d;
    a.ref_counts_out[d] = ld_act(a.ref_counts + s);
    a.ref_counts_out[s] = 0;
  }
  pdl_trigger();
  __syncthreads();
  for (int x = 0; x < 2; ++x) {
    const int64_t entries = (int64_t)a.tables[x].rows * a.tables[x].max_blocks;
    for (int64_t e = tid; e < entries; e += kPlanThreads) remap_entry(a.tables[x], e, a.remap, nb);
  }
}

__global__ void table_remap_kernel(const TableArgs t, const int32_t* remap, int num_blocks) {
  pdl_wait();
  pdl_trigger();
  const int64_t entries = (int64_t)t.rows * t.max_blocks;
  for (int64_t e = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; e < entries; e += (int64_t)gridDim.x * blockDim.x)
    remap_entry(t, e, remap, num_blocks);
}

template <typename V>
int launch_copy(cudaStream_t st, const CopyArgs& a) {
  const int64_t items = a.data.bytes / (int64_t)sizeof(V) * a.planes;
  const int64_t parts = (items + kCopyThreads * kCopyItems - 1) / (kCopyThreads * kCopyItems);
  if (parts * a.n > 0x7fffffff) return SSD_ERR_UNSUPPORTED;
  SSD_PDL(page_copy_kernel<V>, (unsigned)(parts * a.n), kCopyThreads, 0, st, a);
  return SSD_OK;
}

inline bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int copy_common(cudaStream_t st, const CopyArgs& a) {
  auto fits = [&](size_t v) {
    return a.data.bytes % v == 0 && a.data.src_plane % v == 0 && a.data.dst_plane % v == 0 &&
           aligned_to(a.data.src, v) && aligned_to(a.data.dst, v);
  };
  if (fits(16)) return launch_copy<uint4>(st, a);
  if (fits(4)) return launch_copy<uint32_t>(st, a);
  return launch_copy<uint8_t>(st, a);
}

}  // namespace
}  // namespace ssd

using namespace ssd;

extern "C" int ssd_page_copy(ssd_stream_t stream, const void* src_pages, const float* src_scales, int src_blocks,
                             void* dst_pages, float* dst_scales, int dst_blocks, int planes, size_t page_bytes,
                             int scales_per_page, const int32_t* src_ids, int64_t src_step, const int32_t* dst_ids,
                             int64_t dst_step, int n, const int32_t* count) {
  if (n < 0 || planes <= 0 || page_bytes == 0 || src_blocks <= 0 || dst_blocks <= 0 || scales_per_page < 0 ||
      src_step < 0 || dst_step < 0 || !src_pages || !dst_pages)
    return SSD_ERR_INVALID;
  if (scales_per_page > 0 && (!src_scales || !dst_scales)) return SSD_ERR_INVALID;
  if (n == 0) return SSD_OK;
  if (!src_ids || !dst_ids) return SSD_ERR_INVALID;
  if (page_bytes > (size_t)1 << 31) return SSD_ERR_UNSUPPORTED;
  CopyArgs a{};
  a.data = {reinterpret_cast<const char*>(src_pages), reinterpret_cast<char*>(dst_pages), (int64_t)page_bytes,
            (int64_t)page_bytes * src_blocks, (int64_t)page_bytes * dst_blocks};
  const int64_t sb = (int64_t)scales_per_page * (int64_t)sizeof(float);
  a.scales = {reinterpret_cast<const char*>(src_scales), reinterpret_cast<char*>(dst_scales), sb, sb * src_blocks,
              sb * dst_blocks};
  a.src_ids = src_ids;
  a.dst_ids = dst_ids;
  a.src_step = src_step;
  a.dst_step = dst_step;
  a.count = count;
  a.n = n;
  a.planes = planes;
  a.src_blocks = src_blocks;
  a.dst_blocks = dst_blocks;
  return copy_common((cudaStream_t)stream, a);
}

extern "C" int ssd_page_compact(ssd_stream_t stream, const int32_t* free_list, const int32_t* free_top,
                                const int32_t* ref_counts, int num_blocks, int32_t* free_list_out,
                                int32_t* free_top_out, int32_t* ref_counts_out, int32_t* remap, int32_t* move_src,
                                int32_t* move_dst, int32_t* num_moves, const int32_t* tables, int32_t* tables_out,
                                const int32_t* lens, int max_blocks, int B, const int32_t* draft_tables,
                                int32_t* draft_tables_out, const int32_t* draft_lens, int draft_max_blocks,
                                int draft_B) {
  if (num_blocks <= 0 || !free_list || !free_top || !ref_counts || !free_list_out || !free_top_out ||
      !ref_counts_out || !remap || !move_src || !move_dst || !num_moves || B < 0 || draft_B < 0)
    return SSD_ERR_INVALID;
  if (B > 0 && (!tables || !tables_out || !lens || max_blocks <= 0)) return SSD_ERR_INVALID;
  if (draft_B > 0 && (!draft_tables || !draft_tables_out || !draft_lens || draft_max_blocks <= 0))
    return SSD_ERR_INVALID;
  cudaStream_t st = (cudaStream_t)stream;
  CompactArgs a{free_list, free_top, ref_counts, free_list_out, free_top_out, ref_counts_out,
                remap, move_src, move_dst, num_moves, num_blocks, {}};
  const TableArgs t[2] = {{tables, tables_out, lens, B, max_blocks},
                          {draft_tables, draft_tables_out, draft_lens, draft_B, draft_max_blocks}};
  // up to 16 entries a thread in the plan's own CTA; larger tables get a launch of their own
  bool own[2];
  for (int x = 0; x < 2; ++x) {
    own[x] = (int64_t)t[x].rows * t[x].max_blocks > 16 * kPlanThreads;
    if (!own[x]) a.tables[x] = t[x];
  }
  if (num_blocks <= kFlagCap) {
    static std::atomic<uint64_t> ready{0};
    if (num_blocks > 40 * 1024 && !allow_smem(ready, compact_plan_kernel<true>, kFlagCap)) return SSD_ERR_LAUNCH;
    SSD_PDL(compact_plan_kernel<true>, 1, kPlanThreads, num_blocks, st, a);
  } else {
    SSD_PDL(compact_plan_kernel<false>, 1, kPlanThreads, 0, st, a);
  }
  for (int x = 0; x < 2; ++x) {
    if (!own[x]) continue;
    const int64_t ctas = ((int64_t)t[x].rows * t[x].max_blocks + 255) / 256;
    SSD_PDL(table_remap_kernel, (unsigned)(ctas < 1184 ? ctas : 1184), 256, 0, st, t[x], remap, num_blocks);
  }
  return SSD_OK;
}
