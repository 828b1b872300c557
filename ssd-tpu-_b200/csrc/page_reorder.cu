// Paged rows re-ordered by their parents (beam search): row i of a request becomes what row parents[i] was.
//
// A parent's whole pages are shared by its children, its partial last page stays with the first of them and is copied
// for the others, and pages that no row refers to any more go back on the free list.  Nothing of a whole page moves, so
// what a step cannot do without is the tables' entries, once read and once written, and the copied rows.
//
//   reorder kernel  one cluster of CTAs (hardware barriers between its phases, no second launch): reference counts
//                   change by (children - 1) for each entry; entries whose count has come to nothing are marked; the
//                   tables are permuted in place, a stripe of columns at a time through shared memory; the marked
//                   blocks are pushed in ascending order and the fresh ones popped in row order, so that the free
//                   list does not depend on which thread came first.
//   row copy kernel the first rows of a page in all planes, a CTA a piece of one plane of one pair.
#include "kv8.cuh"

namespace ssd {
namespace {

constexpr int kMaxReorder = 1024;   // rows
constexpr int kReorderThreads = 512;
constexpr int kCluster = 8;
constexpr int kStripe = 4096;       // table entries of a stripe
constexpr int kGone = 1 << 30;      // in a reference count's place: nobody refers to the block any more

struct Reorder {
  int32_t *tables, *lens;
  int max_blocks;
  int32_t *free_list, *free_top, *refs;
  int num_blocks;
  const int32_t *parents, *held;
  int B, W, block_size;
  uint8_t* ok;
  int32_t *src, *dst, *rows;        // the copies: pages and how many rows of them; -1: none
};

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return (int)r;
}
// Reads an int of CTA `rank`'s shared memory.
__device__ __forceinline__ int ld_cluster(const int* p, int rank) {
  uint32_t a = (uint32_t)__cvta_generic_to_shared(p), b;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(a), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(b) : "memory");
  return v;
}

// Exclusive sum over the CTA; `tmp` holds a number a warp.
__device__ __forceinline__ int block_scan(int v, int* tmp, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) tmp[warp] = x;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < (int)blockDim.x / 32; ++w) {
    if (w < warp) before += tmp[w];
    all += tmp[w];
  }
  *total = all;
  return before + x - v;
}

__global__ void __launch_bounds__(kReorderThreads) page_reorder_kernel(const Reorder a) {
  __shared__ int stripe[kStripe];
  __shared__ int16_t parent_s[kMaxReorder];            // -1: the row is emptied
  __shared__ int children[kMaxReorder], first[kMaxReorder];
  __shared__ int need_s[kMaxReorder], len_s[kMaxReorder];  // blocks that a row's tokens take, and that it has
  __shared__ int part_s[kMaxReorder];                  // index of the partial page (-1: none)
  __shared__ int tmp[kReorderThreads / 32], mine_s, top_s;
  const int tid = threadIdx.x, rank = cluster_rank();
  pdl_wait();
  for (int i = tid; i < a.B; i += kReorderThreads) {
    children[i] = 0;
    first[i] = a.B;
    const int len = min(max(ld_act(a.lens + i), 0), a.max_blocks), n = max(ld_act(a.held + i), 0);
    const int full = min(n / a.block_size, len);
    const bool part = full < len && n % a.block_size != 0;
    need_s[i] = full + part;
    len_s[i] = len;
    part_s[i] = part ? full : -1;
  }
  if (tid == 0) top_s = ld_act(a.free_top);
  __syncthreads();
  for (int i = tid; i < a.B; i += kReorderThreads) {
    const int p = ld_act(a.parents + i);
    const int at = (unsigned)p < (unsigned)a.W ? i / a.W * a.W + p : -1;
    parent_s[i] = (int16_t)at;
    if (at >= 0) {
      atomicAdd(&children[at], 1);
      atomicMin(&first[at], i);
    }
  }
  __syncthreads();
  int used = 0;
  for (int i = 0; i < a.B; ++i) used = max(used, len_s[i]);
  // change of a block's count for entry j of row b
  auto change = [&](int b, int j) {
    if (j >= len_s[b]) return 0;
    if (j >= need_s[b]) return -1;
    const int c = children[b];
    return j == part_s[b] ? (c > 0 ? 0 : -1) : c - 1;
  };
  const int cols = max(1, kStripe / a.B);  // columns of a stripe
  const int stripes = (used + cols - 1) / cols;
  for (int s = rank; s < stripes; s += kCluster) {
    for (int e = tid; e < a.B * cols; e += kReorderThreads) {
      const int b = e / cols, j = s * cols + e % cols, d = change(b, j);
      if (d == 0) continue;
      const int blk = ld_act(a.tables + (int64_t)b * a.max_blocks + j);
      if ((unsigned)blk < (unsigned)a.num_blocks) atomicAdd(a.refs + blk, d);
    }
  }
  cluster_barrier();
  for (int s = rank; s < stripes; s += kCluster) {
    __syncthreads();
    for (int e = tid; e < a.B * cols; e += kReorderThreads) {
      const int b = e / cols, j = s * cols + e % cols;
      int blk = -1;
      if (j < len_s[b]) blk = ld_act(a.tables + (int64_t)b * a.max_blocks + j);
      stripe[e] = blk;
      if ((unsigned)blk < (unsigned)a.num_blocks && change(b, j) < 0 && ld_act(a.refs + blk) <= 0)
        __stcg(a.refs + blk, kGone);
    }
    __syncthreads();
    for (int e = tid; e < a.B * cols; e += kReorderThreads) {
      const int b = e / cols, j = s * cols + e % cols, p = parent_s[b];
      if (p == b && need_s[b] == len_s[b] && (part_s[b] < 0 || first[b] == b)) continue;
      const int had = len_s[b], has = p >= 0 ? need_s[p] : 0;
      if (j >= max(had, has) || j >= a.max_blocks) continue;
      int blk = -1;
      if (j < has && (j != part_s[p] || first[p] == b)) blk = stripe[p * cols + (e % cols)];
      else if (j < has) blk = -2 - stripe[p * cols + (e % cols)];  // a copy is wanted; the page it is of
      a.tables[(int64_t)b * a.max_blocks + j] = blk;
    }
  }
  cluster_barrier();
  // the blocks that are gone: each CTA a run of blocks, in ascending order
  const int run = (a.num_blocks + kCluster - 1) / kCluster, lo = min(rank * run, a.num_blocks),
            hi = min(lo + run, a.num_blocks);
  const int per = (hi - lo + kReorderThreads - 1) / kReorderThreads;
  const int my0 = min(lo + tid * per, hi), my1 = min(my0 + per, hi);
  int n = 0;
  for (int i = my0; i < my1; ++i) n += ld_act(a.refs + i) == kGone;
  int total;
  int at = block_scan(n, tmp, &total);
  if (tid == 0) mine_s = total;
  cluster_barrier();
  int freed = 0;
  for (int r = 0; r < kCluster; ++r) {
    const int x = ld_cluster(&mine_s, r);
    if (r < rank) at += x;
    freed += x;
  }
  const int top = min(max(top_s, 0), a.num_blocks);
  at += top;
  for (int i = my0; i < my1; ++i) {
    if (ld_act(a.refs + i) != kGone) continue;
    __stcg(a.refs + i, 0);
    if (at < a.num_blocks) __stcg(a.free_list + at, i);
    ++at;
  }
  cluster_barrier();  // (also: no CTA leaves while another may read its shared memory)
  if (rank != 0) return;
  // fresh pages, popped in row order
  int avail = min(top + freed, a.num_blocks);
  for (int b0 = 0; b0 < a.B; b0 += kReorderThreads) {
    const int b = b0 + tid, p = b < a.B ? parent_s[b] : -1;
    const bool take = p >= 0 && part_s[p] >= 0 && first[p] != b;
    int all;
    const int nth = block_scan(take, tmp, &all), slot = avail - 1 - nth;
    if (b < a.B) {
      int src = -1, dst = -1, rows = 0;
      bool ok = true;
      int len = p >= 0 ? need_s[p] : 0;
      if (take) {
        int32_t* row = a.tables + (int64_t)b * a.max_blocks;
        const int full = part_s[p];
        src = -2 - __ldcg(row + full);
        dst = slot >= 0 ? __ldcg(a.free_list + slot) : -1;
        if ((unsigned)dst < (unsigned)a.num_blocks) {
          __stcg(a.free_list + slot, -1);
          a.refs[dst] = 1;
          row[full] = dst;
          rows = ld_act(a.held + p) % a.block_size;
        } else {  // no page left: the row is left empty (its siblings keep the shared pages alive)
          ok = false;
          for (int j = 0; j < len; ++j) {
            const int blk = __ldcg(row + j);
            if (j < full && (unsigned)blk < (unsigned)a.num_blocks) atomicSub(a.refs + blk, 1);
            row[j] = -1;
          }
          src = dst = -1;
          len = 0;
        }
      }
      a.lens[b] = len;
      if (a.ok) a.ok[b] = ok;
      a.src[b] = src;
      a.dst[b] = dst;
      a.rows[b] = rows;
    }
    avail = max(avail - all, 0);
  }
  if (tid == 0) *a.free_top = avail;
  pdl_trigger();
}

constexpr int kRowsThreads = 256, kRowsItems = 4;

struct RowCopy {
  char* pages;
  int64_t plane, page, row;   // bytes between planes, of a page in one plane, of one of its rows
  float* scales;
  int64_t scale_plane;
  int per_page;               // scales of a page (0: none)
  const int32_t *src, *dst, *rows;
  int num_blocks, block_size;
};

template <typename V>
__global__ void __launch_bounds__(kRowsThreads) page_copy_rows_kernel(const RowCopy a) {
  const int pair = blockIdx.x, plane = blockIdx.y, part = blockIdx.z;
  pdl_wait();
  const int s = ld_act(a.src + pair), d = ld_act(a.dst + pair), n = min(ld_act(a.rows + pair), a.block_size);
  if ((unsigned)s >= (unsigned)a.num_blocks || (unsigned)d >= (unsigned)a.num_blocks || s == d || n <= 0) return;
  const int64_t items = a.row * n / (int64_t)sizeof(V);
  const V* from = reinterpret_cast<const V*>(a.pages + plane * a.plane + s * a.page);
  V* to = reinterpret_cast<V*>(a.pages + plane * a.plane + d * a.page);
  V x[kRowsItems];
  const int64_t k0 = (int64_t)part * (kRowsItems * kRowsThreads) + threadIdx.x;
#pragma unroll
  for (int q = 0; q < kRowsItems; ++q)
    if (k0 + q * kRowsThreads < items) x[q] = __ldcg(from + k0 + q * kRowsThreads);
#pragma unroll
  for (int q = 0; q < kRowsItems; ++q)
    if (k0 + q * kRowsThreads < items) __stcg(to + k0 + q * kRowsThreads, x[q]);
  if (part == 0)
    for (int i = threadIdx.x; i < a.per_page; i += kRowsThreads) {
      float* sc = a.scales + plane * a.scale_plane;
      sc[(int64_t)d * a.per_page + i] = ld_act(sc + (int64_t)s * a.per_page + i);
    }
}

}  // namespace
}  // namespace ssd

using namespace ssd;

extern "C" int ssd_page_reorder(ssd_stream_t stream, int32_t* block_tables, int32_t* table_lens, int max_blocks,
                                int32_t* free_list, int32_t* free_top, int32_t* ref_counts, int num_blocks,
                                const int32_t* parents, const int32_t* num_tokens, int block_size, uint8_t* ok,
                                int32_t* copy_src, int32_t* copy_dst, int32_t* copy_rows, int G, int W) {
  if (G < 0 || W <= 0 || max_blocks <= 0 || num_blocks <= 0 || block_size <= 0) return SSD_ERR_INVALID;
  if (G == 0) return SSD_OK;
  if (!block_tables || !table_lens || !free_list || !free_top || !ref_counts || !parents || !num_tokens || !copy_src ||
      !copy_dst || !copy_rows)
    return SSD_ERR_INVALID;
  if ((int64_t)G * W > kMaxReorder || num_blocks >= kGone) return SSD_ERR_UNSUPPORTED;
  const Reorder a{block_tables, table_lens, max_blocks, free_list, free_top, ref_counts, num_blocks, parents, num_tokens,
                  G * W, W, block_size, ok, copy_src, copy_dst, copy_rows};
  if (launch_pdl_cluster(page_reorder_kernel, dim3(kCluster), dim3(kReorderThreads), 0, (cudaStream_t)stream, kCluster,
                         a) != cudaSuccess) {
    (void)cudaGetLastError();
    return SSD_ERR_LAUNCH;
  }
  return SSD_OK;
}

extern "C" int ssd_page_copy_rows(ssd_stream_t stream, void* pages, float* scales, int num_blocks, int block_size,
                                  int planes, size_t row_bytes, int scales_per_page, const int32_t* src_ids,
                                  const int32_t* dst_ids, const int32_t* rows, int n) {
  if (num_blocks <= 0 || block_size <= 0 || planes <= 0 || row_bytes == 0 || scales_per_page < 0 || n < 0)
    return SSD_ERR_INVALID;
  if (n == 0) return SSD_OK;
  if (!pages || (scales_per_page > 0 && !scales) || !src_ids || !dst_ids || !rows) return SSD_ERR_INVALID;
  const uint64_t page = (uint64_t)row_bytes * block_size;
  if (row_bytes > (1u << 31) || page > (1ull << 31) || planes > 65535) return SSD_ERR_UNSUPPORTED;
  const RowCopy a{reinterpret_cast<char*>(pages), (int64_t)page * num_blocks, (int64_t)page, (int64_t)row_bytes, scales,
                  (int64_t)scales_per_page * num_blocks, scales_per_page, src_ids, dst_ids, rows, num_blocks, block_size};
  const bool v16 = row_bytes % 16 == 0 && !(reinterpret_cast<uintptr_t>(pages) & 15);
  const uint64_t items = page / (v16 ? 16 : 1), parts = (items + kRowsItems * kRowsThreads - 1) / (kRowsItems * kRowsThreads);
  if (parts > 65535) return SSD_ERR_UNSUPPORTED;
  const dim3 grid(n, planes, (unsigned)parts);
  if (v16) SSD_PDL(page_copy_rows_kernel<uint4>, grid, kRowsThreads, 0, stream, a);
  else SSD_PDL(page_copy_rows_kernel<uint8_t>, grid, kRowsThreads, 0, stream, a);
  return SSD_OK;
}
