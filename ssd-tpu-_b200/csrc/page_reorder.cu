// Paged rows re-ordered by their parents (beam search): row i of a request becomes what row parents[i] was.
//
// A parent's whole pages are shared by its children, its partial last page stays with the first of them and is copied
// for the others, and pages that no row refers to any more go back on the free list.  Nothing of a whole page moves, so
// what a step cannot do without is the tables' entries, once read and once written, and the copied rows.
//
//   reorder kernel  one cluster of CTAs (hardware barriers between its phases, no second launch), or one CTA for small
//                   tables.  A thread takes one column of one request at a time, its W entries in registers: reference
//                   counts change by (children - 1) for each, summed up first where all rows hold one page (a shared
//                   prompt: no atomics).  Then entries whose count has come to nothing are marked and the columns
//                   written in their new order.  The marked blocks are pushed in ascending order and the fresh ones
//                   popped in row order, so that the free list does not depend on which thread came first.
//   row copy kernel the first rows of a page in all planes, a CTA a piece of one plane of one pair.
// Bound by latency: for four beams a chain of eight or so trips to L2 with barriers between them (4.5 us), then the copies
// (28 layers, 16 heads of 256: 22 MB in 9 us); 256 rows with 200 to 4000 tokens 22 us, 13 of them the tables, scattered counts
// and one CTA's walk over all of them, 9 the copies (13 MB each way).
#include <algorithm>

#include "kv8.cuh"

namespace ssd {
namespace {

constexpr int kMaxReorder = 1024;   // rows
constexpr int kMaxBeams = 32;       // of a request
constexpr int kReorderThreads = 1024;
// 16 CTAs: 32 requests of 8 beams with 200 to 4000 tokens 21.9 us, 8 CTAs 27.1, the copies included: most of it is
// scattered reads and atomics of the counts, which each SM takes one after another.
constexpr int kCluster = 16;
// Columns of all requests that one CTA takes alone (a cluster for the toy pair's 4 rows 9.5 us instead of 8.7, for four beams of
// 530 tokens 15.8 instead of 14.8; one CTA for 256 rows 49 instead of 22).
constexpr int kOneCta = 4096;
constexpr int kMaxColumns = 1 << 30;  // of all requests: counted in 32 bits, a step of all threads behind the last included
constexpr int kGone = 1 << 30;      // in a reference count's place: nobody refers to the block any more

struct Reorder {
  int32_t *tables, *lens;
  int max_blocks;
  int32_t *free_list, *free_top, *refs;
  int num_blocks;
  const int32_t *parents, *held;
  int G, W, block_size;
  uint8_t* ok;
  int32_t *src, *dst, *rows;        // the copies: pages and how many rows of them; -1: none
};

__device__ __forceinline__ void cluster_barrier() {
  if (gridDim.x == 1) {
    __syncthreads();
    return;
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
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
  const int mine = tmp[lane];  // 32 warps
  int y = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int z = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) y += z;
  }
  *total = __shfl_sync(0xffffffffu, y, 31);
  return __shfl_sync(0xffffffffu, y - mine, warp) + x - v;
}

// WM: at least W.
template <int WM>
__global__ void __launch_bounds__(kReorderThreads) page_reorder_kernel(const Reorder a) {
  __shared__ int16_t parent_s[kMaxReorder];            // -1: the row is emptied
  __shared__ int children[kMaxReorder], first[kMaxReorder];
  __shared__ int need_s[kMaxReorder], len_s[kMaxReorder];  // blocks that a row's tokens take, and that it has
  __shared__ int part_s[kMaxReorder];                  // index of the partial page (-1: none)
  __shared__ int whole_s[kMaxReorder];                 // of a request: columns that are whole pages of all its rows
  __shared__ int used_s, tmp[32];
  const int tid = threadIdx.x, B = a.G * a.W;
  pdl_wait();
  pdl_trigger();
  int parent = 0, len = 0, held = 0;
  if (tid < B) {
    parent = ld_act(a.parents + tid);
    len = ld_act(a.lens + tid);
    held = ld_act(a.held + tid);
  }
  const int top = min(max(ld_act(a.free_top), 0), a.num_blocks);
  if (tid == 0) used_s = 0;
  children[tid] = 0;
  first[tid] = B;
  whole_s[tid] = a.max_blocks;
  __syncthreads();
  len = min(max(len, 0), a.max_blocks);
  held = max(held, 0);
  parent = tid < B && (unsigned)parent < (unsigned)a.W ? tid / a.W * a.W + parent : -1;
  const int full = min(held / a.block_size, len);
  const bool part = full < len && held % a.block_size != 0;
  if (tid < B) {
    need_s[tid] = full + part;
    len_s[tid] = len;
    part_s[tid] = part ? full : -1;
    parent_s[tid] = (int16_t)parent;
    atomicMin(&whole_s[tid / a.W], parent >= 0 ? full : 0);
    if (parent >= 0) {
      atomicAdd(&children[parent], 1);
      atomicMin(&first[parent], tid);
    }
  }
  const int longest = __reduce_max_sync(0xffffffffu, tid < B ? len : 0);
  if ((tid & 31) == 0 && longest > 0) atomicMax(&used_s, longest);
  __syncthreads();
  const int used = used_s, items = a.G * used;
  // change of a block's count for entry j of row b
  auto change = [&](int b, int j) {
    if (j >= len_s[b]) return 0;
    if (j >= need_s[b]) return -1;
    const int c = children[b];
    return j == part_s[b] ? (c > 0 ? 0 : -1) : c - 1;
  };
  auto entries = [&](int g, int j, int* e) {
#pragma unroll
    for (int w = 0; w < WM; ++w) {
      e[w] = -1;
      if (w < a.W && j < len_s[g * a.W + w]) e[w] = ld_act(a.tables + (int64_t)(g * a.W + w) * a.max_blocks + j);
    }
  };
  const int step = gridDim.x * kReorderThreads, i0 = blockIdx.x * kReorderThreads + tid;
  int kept[WM <= 8 ? WM : 1];  // the thread's first column (registers that the larger kernel has not got)
  uint32_t same = 0;           // bit k: the k-th column stays as it is
  for (int i = i0, k = 0; i < items; i += step, ++k) {
    const int g = i / used, j = i - g * used;
    int e[WM], net = 0;
    entries(g, j, e);
    if constexpr (WM <= 8) {
      if (k == 0) {
#pragma unroll
        for (int w = 0; w < WM; ++w) kept[w] = e[w];
      }
    }
    bool one = true;
#pragma unroll
    for (int w = 0; w < WM; ++w)
      if (w < a.W) one &= e[w] == e[0];
    if (one && j < whole_s[g]) {  // the prompt's pages: shared by the parents, shared by the children
      if (k < 32) same |= 1u << k;
      continue;
    }
#pragma unroll
    for (int w = 0; w < WM; ++w)
      if (w < a.W) net += change(g * a.W + w, j);
    if (one) {
      if (net != 0 && (unsigned)e[0] < (unsigned)a.num_blocks) atomicAdd(a.refs + e[0], net);
      continue;
    }
#pragma unroll
    for (int w = 0; w < WM; ++w)
      if (w < a.W && (unsigned)e[w] < (unsigned)a.num_blocks) {
        const int d = change(g * a.W + w, j);
        if (d != 0) atomicAdd(a.refs + e[w], d);
      }
  }
  cluster_barrier();
  for (int i = i0, k = 0; i < items; i += step, ++k) {
    if (k < 32 && (same >> k & 1)) continue;
    const int g = i / used, j = i - g * used;
    int e[WM], refs[WM];
    if (WM <= 8 && k == 0) {
#pragma unroll
      for (int w = 0; w < WM; ++w) e[w] = kept[WM <= 8 ? w : 0];
    } else {
      entries(g, j, e);
    }
#pragma unroll
    for (int w = 0; w < WM; ++w)
      refs[w] = w < a.W && (unsigned)e[w] < (unsigned)a.num_blocks && change(g * a.W + w, j) < 0 ? ld_act(a.refs + e[w]) : 1;
#pragma unroll
    for (int w = 0; w < WM; ++w)
      if (refs[w] <= 0) __stcg(a.refs + e[w], kGone);
#pragma unroll
    for (int w = 0; w < WM; ++w) {
      if (w >= a.W) continue;
      const int b = g * a.W + w, p = parent_s[b], has = p >= 0 ? need_s[p] : 0;
      if (j >= max(len_s[b], has)) continue;
      int blk = -1;
      if (j < has) {
        const int from = p - g * a.W;
#pragma unroll
        for (int x = 0; x < WM; ++x)
          if (x == from) blk = e[x];
        if (j == part_s[p] && first[p] != b) blk = -2 - blk;  // a copy is wanted; the page it is of
      }
      if (blk != e[w]) __stcg(a.tables + (int64_t)b * a.max_blocks + j, blk);
    }
  }
  cluster_barrier();
  if (blockIdx.x != 0) return;
  // the blocks that are gone, pushed in ascending order: a run of them a thread
  const int run = (a.num_blocks + kReorderThreads - 1) / kReorderThreads, lo = min(tid * run, a.num_blocks),
            hi = min(lo + run, a.num_blocks);
  int n = 0;
  uint32_t which = 0;  // of the first 32 (runs are seldom longer)
  constexpr int AT_ONCE = 8;
  for (int i = lo; i < hi; i += AT_ONCE) {
    int refs[AT_ONCE];
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) refs[k] = i + k < hi ? ld_act(a.refs + i + k) : 0;
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k)
      if (refs[k] == kGone) {
        ++n;
        if (i + k - lo < 32) which |= 1u << (i + k - lo);
      }
  }
  int freed;
  int at = top + block_scan(n, tmp, &freed);
  auto push = [&](int i) {
    __stcg(a.refs + i, 0);
    if (at < a.num_blocks) __stcg(a.free_list + at, i);
    ++at;
  };
  for (; which; which &= which - 1) push(lo + __ffs(which) - 1);
  for (int i = lo + 32; i < hi; ++i)
    if (ld_act(a.refs + i) == kGone) push(i);
  // fresh pages, popped in row order
  const int avail = min(top + freed, a.num_blocks);
  const int b = tid, p = parent;
  const bool take = p >= 0 && part_s[p] >= 0 && first[p] != b;
  int all;
  const int nth = block_scan(take, tmp, &all), slot = avail - 1 - nth;  // (its barriers: the pushes are there)
  if (b < B) {
    int src = -1, dst = -1, rows = 0;
    bool ok = true;
    int now = p >= 0 ? need_s[p] : 0;
    if (take) {
      int32_t* row = a.tables + (int64_t)b * a.max_blocks;
      const int at_part = part_s[p];
      src = -2 - __ldcg(row + at_part);
      dst = slot >= 0 ? __ldcg(a.free_list + slot) : -1;
      if ((unsigned)dst < (unsigned)a.num_blocks) {
        __stcg(a.free_list + slot, -1);
        a.refs[dst] = 1;
        row[at_part] = dst;
        rows = ld_act(a.held + p) % a.block_size;
      } else {  // no page left: the row is left empty (its siblings keep the shared pages alive)
        ok = false;
        for (int j = 0; j < now; ++j) {
          const int blk = __ldcg(row + j);
          if (j < at_part && (unsigned)blk < (unsigned)a.num_blocks) atomicSub(a.refs + blk, 1);
          row[j] = -1;
        }
        src = dst = -1;
        now = 0;
      }
    }
    a.lens[b] = now;
    if (a.ok) a.ok[b] = ok;
    a.src[b] = src;
    a.dst[b] = dst;
    a.rows[b] = rows;
  }
  if (tid == 0) *a.free_top = max(avail - all, 0);
}

bool allow_cluster(std::atomic<uint64_t>& ready, void (*kern)(Reorder)) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  if (ready.load(std::memory_order_acquire) >> dev & 1) return true;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
    (void)cudaGetLastError();
    return false;
  }
  ready.fetch_or(1ull << dev, std::memory_order_release);
  return true;
}

template <int WM>
int launch_reorder(cudaStream_t st, const Reorder& a) {
  static std::atomic<uint64_t> ready{0};  // devices whose limit is raised
  if ((int64_t)a.G * a.max_blocks <= kOneCta) {
    SSD_PDL(page_reorder_kernel<WM>, 1, kReorderThreads, 0, st, a);
    return SSD_OK;
  }
  if (!allow_cluster(ready, page_reorder_kernel<WM>)) return SSD_ERR_LAUNCH;
  if (launch_pdl_cluster(page_reorder_kernel<WM>, dim3(kCluster), dim3(kReorderThreads), 0, st, kCluster, a) != cudaSuccess) {
    (void)cudaGetLastError();
    return SSD_ERR_LAUNCH;
  }
  return SSD_OK;
}

constexpr int kRowsThreads = 128, kRowsItems = 8;

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
  if (W > kMaxBeams || (int64_t)G * W > kMaxReorder || num_blocks >= kGone || (int64_t)G * max_blocks > kMaxColumns)
    return SSD_ERR_UNSUPPORTED;
  const Reorder a{block_tables, table_lens, max_blocks, free_list, free_top, ref_counts, num_blocks, parents, num_tokens,
                  G, W, block_size, ok, copy_src, copy_dst, copy_rows};
  cudaStream_t st = (cudaStream_t)stream;
  return W <= 8 ? launch_reorder<8>(st, a) : launch_reorder<kMaxBeams>(st, a);
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
