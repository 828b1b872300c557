// Attention of a batch whose rows share long prefixes (beams, branches, samples of one prompt; a common system prompt).
//
// Rows starts[g] .. starts[g+1]-1 of the batch form group g and agree on their first prefix_lens[g] = P positions.
// For query row (b, t, head) at position p = seq_lens[b] - q_lens[b] + t:
//   out = sum_j e^(s_j - M) v_j / sum_j e^(s_j - M),  s_j = scale q . k_j,  j <= p,
// where positions j < P are read through the group's first row's table and the others through the row's own.
//
// The query rows of several sequences of a group (G query heads of a KV head times the new tokens of each) stand in one
// row tile.  What a tile sees is a list of positions: the prefix once, then each of its sequences' tails, which only
// that sequence's rows see.  Every K and V byte is so read once for all rows of the tile, where attention by rows
// reads a prefix once for each row.  A tile's list is cut into parts, whose unnormalised sums a second kernel joins
// in order.
#include <float.h>

#include <algorithm>

#include "kv8.cuh"
#include "linear.cuh"
#include "tcgen05.cuh"

namespace ssd {
namespace {

constexpr int kMaxRowsB = 1024;        // sequences, and groups, of one call
constexpr int kMaxPos = 1 << 30;       // positions of a sequence

struct PrefixAttn {
  const void* q;
  const void* pages;
  void* out;
  int64_t plane;         // elements of one K (or V) plane
  int64_t layer;         // element offset of the layer inside a plane
  const int32_t *tables, *seq_lens, *q_lens, *starts, *prefixes;
  float scale;
  int B, T, hq, hkv, G, groups, num_blocks, block_size, max_blocks;
  int cap;               // positions of a sequence that may be read
  int R;                 // query rows of a sequence and KV head: G * T
  int tile_rows;         // query rows of a row tile
  int spt_inv;           // 65536 / spt + 1
  int spt, tps;          // sequences of a row tile (R <= its rows), else tiles of a sequence
  int tiles;             // bound on the row tiles of all groups
  int num_layers, layer_no;
  uint32_t polls;        // of each device-side wait
  int q_box;             // query rows that a fetch of Q brings in
  int nsplit;            // parts of a tile's list (CUDA-core kernel)
  float* ws_o;           // [part][row][D] unnormalised sums
  float2* ws_ml;         // [part][row] what they are relative to, sum of weights
  // [sequence, or slice of one where it takes several tiles][head]: first part, parts (1: the kernel has
  // written the rows itself), step from part to part, the sequence's first row
  int4* parts;
  bool whole;            // lists are not cut
};

struct RowTile {
  int group;             // -1: none
  int first;             // first row of the group: the prefix is read through its table
  int seq0, nseq;        // the tile's sequences
  int part;              // which slice of the sequence's rows (tps > 1)
};

__device__ __forceinline__ int group_tiles(const PrefixAttn& a, int rows) {
  return rows <= 0 ? 0 : a.tps > 1 ? rows * a.tps : (rows + a.spt - 1) / a.spt;
}
__device__ __forceinline__ int clamped(int x, int hi) { return min(max(x, 0), hi); }

// Tile `tile` of the batch: groups in order, their tiles in order.  A start below one before it counts as that one, so that
// no row is in two groups.  For whole warps.
__device__ __forceinline__ RowTile find_tile(const PrefixAttn& a, int tile) {
  const int lane = threadIdx.x & 31;
  int before = 0, high = 0;  // high: the largest start so far
  for (int g0 = 0; g0 < a.groups; g0 += 32) {
    const int g = g0 + lane;
    int s = high, e = high;
    if (g < a.groups) {
      s = clamped(ld_act(a.starts + g), a.B);
      e = clamped(ld_act(a.starts + g + 1), a.B);
    }
    if (__any_sync(0xffffffffu, e < s || s < high)) {
      s = max(s, high);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) s = max(s, __shfl_up_sync(0xffffffffu, s, o));  // (lane 0 .. o-1: its own)
      e = max(s, e);
    }
    high = __shfl_sync(0xffffffffu, e, 31);
    const int n = group_tiles(a, e - s);
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    const int at = before + incl - n;
    const uint32_t hit = __ballot_sync(0xffffffffu, tile >= at && tile < at + n);
    if (hit) {
      const int from = __ffs(hit) - 1;
      const int k = tile - __shfl_sync(0xffffffffu, at, from);
      s = __shfl_sync(0xffffffffu, s, from);
      e = __shfl_sync(0xffffffffu, e, from);
      RowTile t;
      t.group = g0 + from;
      t.first = s;
      t.seq0 = a.tps > 1 ? s + k / a.tps : s + k * a.spt;
      t.nseq = a.tps > 1 ? 1 : min(a.spt, e - t.seq0);
      t.part = a.tps > 1 ? k % a.tps : 0;
      return t;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return RowTile{-1, 0, 0, 0, 0};
}

__device__ __forceinline__ int new_tokens(const PrefixAttn& a, int b) {
  return a.q_lens ? clamped(ld_act(a.q_lens + b), a.T) : a.T;
}
// Positions of the group's prefix that may be read.
__device__ __forceinline__ int prefix_of(const PrefixAttn& a, int group) {
  return clamped(ld_act(a.prefixes + group), a.cap);
}
// Where query row r of a tile stands in q and out, and its position (-1: no such row).
struct RowAt {
  int b, t, pos, seq;    // seq: the sequence's number in the tile
  int64_t at;            // element offset of the row
};
template <int D>
__device__ __forceinline__ RowAt row_at(const PrefixAttn& a, const RowTile& tl, int head, int r, int rows,
                                        const int* seq_s = nullptr, const uint16_t* ql_s = nullptr) {
  RowAt w;
  const int gr = tl.part * rows + r;
  w.seq = a.tps > 1 ? 0 : gr / a.R;
  const int in = gr - w.seq * a.R;
  w.t = in / a.G;
  w.b = tl.seq0 + w.seq;
  w.pos = -1;
  w.at = -1;
  if (tl.group >= 0 && r < rows && w.seq < tl.nseq && in < a.R) {
    w.at = (((int64_t)w.b * a.T + w.t) * a.hq + head * a.G + (in - w.t * a.G)) * D;
    const int seq = seq_s ? seq_s[w.b] : ld_act(a.seq_lens + w.b), ql = ql_s ? ql_s[w.b] : new_tokens(a, w.b);
    if (w.t < ql) w.pos = max(seq - ql + w.t, -1);
  }
  return w;
}

// ------------------------------------------------------------------ CUDA-core kernel
// fp32 caches, and bf16 ones whose pages are no whole runs of 16 rows.  A CTA takes 8 query rows of one KV head and a
// part of their list, 256 positions at a time: a thread scores one position against all rows (q broadcast from shared
// memory), the rows' maxima and sums are taken over the CTA, and for P V a thread holds 4 dims of all rows over
// every PG-th position.  Bound on long contexts by waiting for its loads: 8 sequences of 8000 fp32 positions and 8 query heads
// over 4 KV heads of 256 take 53.5 us (66 MB, which two row tiles read: L2 sends 219 MB, since a thread's 16 bytes of its own K
// row leave half a sector for later; FMAs 18 % busy), in bf16 over pages of 4 rows 49.2 us.  Bound by the chain of reads
// (lengths, table, page) and barriers of one chunk on short ones: two groups of 3 and 4 fp32 rows with at most 120 positions
// take 9.1 us.
constexpr int kRowsC = 8, kChunkC = 256, kWarpsC = kChunkC / 32;
constexpr int kMaxSplitC = 32;
// Positions of a tile's list: counted in 32 bits, the chunks that the last part may have behind the list's end included.  The
// tails of so long contexts stand in tiles with fewer sequences.  (Counted in 64 bits the toy pair's call took 9.4 us instead of 9.1.)
constexpr int64_t kMaxList = 0x7fffffff - (kMaxSplitC + 1) * kChunkC;

template <typename KV>
__device__ __forceinline__ void load4(const KV* p, float* f) {
  if constexpr (sizeof(KV) == 4) {
    const uint4 u = ld_act_v4(p);
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  } else {
    const uint2 u = __ldcg(reinterpret_cast<const uint2*>(p));
    f[0] = __uint_as_float(u.x << 16); f[1] = __uint_as_float(u.x & 0xffff0000u);
    f[2] = __uint_as_float(u.y << 16); f[3] = __uint_as_float(u.y & 0xffff0000u);
  }
}

// The sequences before the first group and behind the last: zeros in a head's rows, and nothing to join.  For a whole warp.
template <typename KV, int D>
__device__ __forceinline__ void rows_of_no_group(const PrefixAttn& a, int head) {
  const int lane = threadIdx.x & 31;
  int end = 0;
  for (int g = lane; g <= a.groups; g += 32) end = max(end, clamped(ld_act(a.starts + g), a.B));
  end = __reduce_max_sync(0xffffffffu, end);
  const int first = clamped(ld_act(a.starts), a.B), n = first + a.B - end;
  for (int k = 0; k < n; ++k) {
    const int b = k < first ? k : end + k - first;
    for (int t = 0; t < a.T; ++t) {
      KV* to = reinterpret_cast<KV*>(a.out) + (((int64_t)b * a.T + t) * a.hq + head * a.G) * D;
      for (int i = lane; i < a.G * D; i += 32) to[i] = from_f<KV>(0.f);
    }
    if (a.nsplit > 1)
      for (int p = lane; p < a.tps; p += 32) a.parts[((int64_t)b * a.tps + p) * a.hkv + head] = make_int4(0, 1, 0, 0);
  }
}

template <typename KV, int D>
__global__ void __launch_bounds__(kChunkC) prefix_attention_cc_kernel(const PrefixAttn a) {
  constexpr int DG = D / 4, PG = kChunkC / DG;
  __shared__ uint32_t see_s[kChunkC];           // rows that see the position
  __shared__ int64_t v_s[kChunkC];              // element offset of the position's V row (-1: none)
  // q and the weights of a chunk's positions until the last chunk is added, then the threads' sums
  __shared__ __align__(16) float o_s[PG][kRowsC][D / 4][4];
  float(*q_s)[kRowsC] = reinterpret_cast<float(*)[kRowsC]>(&o_s[0][0][0][0]);
  float4(*p_s)[2] = reinterpret_cast<float4(*)[2]>(&o_s[0][0][0][0] + D * kRowsC);
  static_assert(sizeof(o_s) >= sizeof(float) * kRowsC * (D + kChunkC));
  __shared__ float red[2][kWarpsC][kRowsC];
  __shared__ float run[kRowsC], fac[kRowsC], sum[kRowsC];
  __shared__ RowAt row_s[kRowsC];
  __shared__ int cum[kRowsC + 2];               // ends of the prefix and of the sequences' tails in the list
  const int split = blockIdx.x, head = blockIdx.y, tile = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_trigger();
  const RowTile tl = find_tile(a, tile);
  if (tile == 0 && split == 0 && warp == kWarpsC - 1) rows_of_no_group<KV, D>(a, head);
  if (tl.group < 0) return;
  const int P = prefix_of(a, tl.group);
  if (warp == 1 && lane < kRowsC) {
    row_s[lane] = row_at<D>(a, tl, head, lane, kRowsC);
    run[lane] = -INFINITY;
    sum[lane] = 0.f;
  }
  if (warp == 0) {
    int tail = 0;
    if (lane < tl.nseq) {
      const int seq = ld_act(a.seq_lens + tl.seq0 + lane), ql = new_tokens(a, tl.seq0 + lane);
      if (ql > 0) tail = max(min(seq, a.cap) - P, 0);
    }
    int incl = tail;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 0) cum[0] = P;
    if (lane < kRowsC) cum[1 + lane] = P + incl;
  }
  __syncthreads();
  for (int i = tid; i < kRowsC * D; i += kChunkC) {
    const int r = i / D, d = i % D;
    const RowAt& w = row_s[r];
    q_s[d][r] = w.pos >= 0 ? to_f(ld_act(reinterpret_cast<const KV*>(a.q) + w.at + d)) : 0.f;
  }
  const int len = cum[kRowsC];
  const int chunks = (len + kChunkC - 1) / kChunkC;
  const int per = max(1, (chunks + a.nsplit - 1) / a.nsplit);
  const int parts = max(1, (chunks + per - 1) / per);
  if (a.nsplit > 1 && split == 0 && tid < tl.nseq)
    a.parts[(int64_t)(a.tps > 1 ? tl.seq0 * a.tps + tl.part : tl.seq0 + tid) * a.hkv + head] =
        make_int4((tile * a.hkv + head) * a.nsplit, parts, 1, a.tps > 1 ? 0 : tid * a.R);
  if (split >= parts) return;
  const int lo = split * per * kChunkC, hi = min(len, lo + per * kChunkC);
  const KV* pages = reinterpret_cast<const KV*>(a.pages) + a.layer;
  const int dg = tid % DG, pg = tid / DG;
  float o[kRowsC][4];
#pragma unroll
  for (int r = 0; r < kRowsC; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[r][i] = 0.f;
  for (int c0 = lo; c0 < hi; c0 += kChunkC) {
    const int i = c0 + tid;
    uint32_t see = 0;
    int64_t off = -1;
    if (i < hi) {
      int owner = -1, pos = i, from = tl.first;
      if (i >= P) {
        owner = 0;
        while (i >= cum[owner + 1]) ++owner;
        pos = P + i - cum[owner];
        from = tl.seq0 + owner;
      }
      const int blk = ld_act(a.tables + (int64_t)from * a.max_blocks + pos / a.block_size);
      if ((unsigned)blk < (unsigned)a.num_blocks) {
        off = (((int64_t)blk * a.block_size + pos % a.block_size) * a.hkv + head) * D;
#pragma unroll
        for (int r = 0; r < kRowsC; ++r)
          if (pos <= row_s[r].pos && (owner < 0 || owner == row_s[r].seq)) see |= 1u << r;
      }
    }
    __syncthreads();  // q is there; the chunk before has been added
    float s[kRowsC];
#pragma unroll
    for (int r = 0; r < kRowsC; ++r) s[r] = 0.f;
    if (see) {
#pragma unroll 8
      for (int d = 0; d < D; d += 4) {
        float k[4];
        load4(pages + off + d, k);
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int r = 0; r < kRowsC; ++r) s[r] = fmaf(q_s[d + x][r], k[x], s[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < kRowsC; ++r) {
      const bool in = see >> r & 1;
      s[r] *= a.scale;
      // finite once a position is seen, a NaN score included: it spoils the sums below
      const float x = warp_max(in ? fmaxf(s[r], -FLT_MAX) : -INFINITY);
      if (lane == 0) red[0][warp][r] = x;
    }
    see_s[tid] = see;
    v_s[tid] = see ? off + a.plane : -1;
    __syncthreads();
    if (tid < kRowsC) {
      float m = run[tid];
#pragma unroll
      for (int w = 0; w < kWarpsC; ++w) m = fmaxf(m, red[0][w][tid]);
      fac[tid] = m == -INFINITY ? 1.f : expf(run[tid] - m);
      run[tid] = m;
    }
    __syncthreads();
    float p[kRowsC];
#pragma unroll
    for (int r = 0; r < kRowsC; ++r) {
      p[r] = see >> r & 1 ? expf(s[r] - run[r]) : 0.f;
      const float x = warp_sum(p[r]);
      if (lane == 0) red[1][warp][r] = x;
    }
    p_s[tid][0] = make_float4(p[0], p[1], p[2], p[3]);
    p_s[tid][1] = make_float4(p[4], p[5], p[6], p[7]);
    __syncthreads();
    if (tid < kRowsC) {
      float l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarpsC; ++w) l += red[1][w][tid];
      sum[tid] = sum[tid] * fac[tid] + l;
    }
#pragma unroll
    for (int r = 0; r < kRowsC; ++r)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[r][x] *= fac[r];
    const int n = min(kChunkC, hi - c0);
    constexpr int AT_ONCE = 4;  // V rows on their way
#pragma unroll 1
    for (int j0 = pg; j0 < n; j0 += AT_ONCE * PG) {
      float v[AT_ONCE][4];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const int64_t vo = j0 + k * PG < n ? v_s[j0 + k * PG] : -1;
        v[k][0] = v[k][1] = v[k][2] = v[k][3] = 0.f;
        if (vo >= 0) load4(pages + vo + 4 * dg, v[k]);
      }
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const int j = min(j0 + k * PG, kChunkC - 1);  // (past n: zeros)
        const float4 pa = p_s[j][0], pb = p_s[j][1];
        const float pr[8] = {pa.x, pa.y, pa.z, pa.w, pb.x, pb.y, pb.z, pb.w};
        if (fabsf(v[k][0]) + fabsf(v[k][1]) + fabsf(v[k][2]) + fabsf(v[k][3]) <= FLT_MAX) {
#pragma unroll
          for (int r = 0; r < kRowsC; ++r)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[r][x] = fmaf(pr[r], v[k][x], o[r][x]);
        } else {  // an infinity or NaN (or a sum past fp32) reaches the rows that see the position, no others
          const uint32_t in = see_s[j];
#pragma unroll
          for (int r = 0; r < kRowsC; ++r)
            if (in >> r & 1) {
#pragma unroll
              for (int x = 0; x < 4; ++x) o[r][x] = fmaf(pr[r], v[k][x], o[r][x]);
            }
        }
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRowsC; ++r)
    *reinterpret_cast<float4*>(o_s[pg][r][dg]) = make_float4(o[r][0], o[r][1], o[r][2], o[r][3]);
  __syncthreads();
  for (int i = tid; i < kRowsC * D; i += kChunkC) {
    const int r = i / D, d = i % D;
    if (row_s[r].at < 0) continue;
    float O = 0.f;
#pragma unroll
    for (int x = 0; x < PG; ++x) O += o_s[x][r][d / 4][d % 4];
    if (parts == 1) {
      reinterpret_cast<KV*>(a.out)[row_s[r].at + d] = from_f<KV>(sum[r] != 0.f ? O / sum[r] : 0.f);
    } else {
      const int64_t at = ((int64_t)(tile * a.hkv + head) * a.nsplit + split) * kRowsC + r;
      a.ws_o[at * D + d] = O;
      if (d == 0) a.ws_ml[at] = make_float2(run[r], sum[r]);
    }
  }
}

// ------------------------------------------------------------------ tensor-core kernel (bf16, pages of 16 k rows)
// Persistent CTAs, one an SM, share out the positions of all row tiles and KV heads in equal runs of 16 (units), so
// a CTA works through one or more segments: a run of units of one tile and head.  128 query rows (TMEM lanes) a tile:
//   S = Q K^T   for 64 positions (M = 128, N = 64), Q from TMEM, K as it lies in the pages (K-major)
//   O += P V    (N = D), P in bf16 from TMEM, V as it lies in the pages (MN-major)
// A unit is 16 rows of one page, so a tile of positions mixes pages of any kind, the prefix's and tails of different
// sequences; which rows see which of its positions is said by 16 bytes a unit.  Rows that see nothing of a unit put
// zero weights on it: that wastes products, of which there are enough, and saves bytes, of which there are not.
//   warps 0-15  two sets of eight that take tiles of positions in turn, in each two threads a query row with half a
//               tile's positions each: scores out of TMEM, maxima (exchanged between the two), weights, rescaling of
//               O (only when a row's reference has to move).  Set 0 also writes results, set 1 brings Q into TMEM.
//   warp 16     walks the tables and fetches Q and the units of K by TMA into a ring of stages: a line of 64 dims of
//               a unit's 16 rows at a time, which is what lays all of a tile's lines out as one operand
//   warp 18     does the same for V, whole units at a time (each is an operand of its own); a warp alone would be
//               held up by the issue of the copies, some 45 cycles each
//   warp 17     issues the products in the order S(j + 2), O(j): S has one place in TMEM, free again as soon as the
//               scores have been read (O(j) runs meanwhile), and the weights two
// The sets share a row's reference M through shared memory: tile j decides on it once tile j - 1 has (`decided`), which
// is early in a tile's work; the weights themselves overlap.
// A product with weight zero still spreads infinities and NaN of V over rows that do not see them.  Then a row's O is
// not finite although its sum of weights is, and the row is worked out again by itself, from the pages.
// Bound by DRAM on long contexts: 32 rows of 7 tokens under a prompt of 8000, 16 KV heads of 256, take 79 us for 334 MB (4.2 TB/s
// over the call; 5.9 TB/s in the loop, before it 3 us of plan, behind it 4 of partial sums and 8 of joining them).  Eight prompts
// of 1000 to 8190 positions with 4 to 8 rows of one KV head take 24 to 29 us for 41 MB: 8 tiles a CTA, fewer than its start, end and
// join are worth.
// All waits are bounded, and a warp's lanes give up together.  A CTA that gives up raises `gave_up`, lets its copies and
// products end, frees its TMEM and leaves NaN in the rows that it has not finished.  (A wait for a phase of a barrier is
// only begun when the phase before is known to be over: parities tell no more apart.)
namespace tile {

constexpr int ROWS = 128;              // query rows of a CTA: TMEM lanes
constexpr int TILE = 64;               // positions of a tile
constexpr int UNITS = TILE / 16;
constexpr int HALF = TILE / 2;         // positions of a thread
constexpr int SET = 256;               // threads of a set of row warps
constexpr int SETW = SET / 32;
constexpr int THREADS = 2 * SET + 96;
constexpr int META = 16;               // tiles whose units are described: more than there are between fetch and use
constexpr int kMaxTiles = 256;         // also sequences and groups: their numbers are kept in shared memory
constexpr int kMinUnits = 8;           // of a run, so that short batches are not cut to crumbs (4 and 16 measure alike)
// Units that the start of a list is worth: what a CTA spends on results and Q where it goes on to another list.  0, 24 and
// 48: 28.2, 21.1 and 21.2 us for 15 rows under a prompt of 2000, 87.8, 83.6 and 79.2 for 32 of 7 tokens under one of 8000.
constexpr int kStart = 48;
// Lists of at most so many units are not cut: the results go straight out and nothing is joined (four beams of 530
// positions 11.8 us, cut and joined 13.4, both before the groups' order was looked at, which costs 0.1).
constexpr int kWhole = 64;
// CTAs that walk a group's lists side by side, so that a prefix comes from DRAM once however many tiles read it (two
// tiles under the prompt of 8000: 79.2 us, each by itself 93.1).
constexpr int kMaxTeam = 8;
constexpr float kSpan = 8.f;           // weights are at most 2^8
constexpr float kNothing = -1e38f;     // M of a row that has seen nothing
constexpr uint32_t kPolls = 1u << 24;
__device__ uint32_t gave_up;           // 1 once a CTA's wait ran out

template <int D>
struct Cfg {
  static constexpr int STAGES = D == 256 ? 3 : 6;  // of K (and Q), and of V
  static constexpr uint32_t KV = TILE * D * 2;     // bytes of one tile's K or V
  static constexpr uint32_t KS = KV < 16384 ? 16384 : KV;  // of a stage of K
  static constexpr int QST = ROWS * D * 2 / KS;    // stages that Q takes: lines of 64 dims, ROWS of them to a chunk
  static constexpr int CPS = KS / 16384;           // chunks of a stage
  static constexpr uint32_t v = STAGES * KS, ring = v + STAGES * KV;
  static constexpr uint32_t pref = ring;                              // int [kMaxTiles + 1], see Walk
  static constexpr uint32_t units = pref + 4 * (kMaxTiles + 4);       // int [kMaxTiles]: units of each tile
  static constexpr uint32_t info = units + 4 * kMaxTiles;             // int2 [kMaxTiles]
  static constexpr uint32_t seq = info + 8 * kMaxTiles;               // int [kMaxTiles]: lengths,
  static constexpr uint32_t ql = seq + 4 * kMaxTiles;                 // uint16: new tokens of the sequences,
  static constexpr uint32_t pre = ql + 2 * kMaxTiles;                 // prefixes of the groups
  static constexpr uint32_t first = pre + 4 * kMaxTiles;              // int [kMaxTiles + 1]: first sequences
  static constexpr uint32_t spt = first + 4 * (kMaxTiles + 4);        // int [kMaxTiles]: sequences of a group's tiles
  static constexpr uint32_t cum = spt + 4 * kMaxTiles;                       // int [2][ROWS + 4]: units before a sequence's tail, for either fetching warp
  static constexpr uint32_t meta = cum + 8 * (ROWS + 4);              // int4 [META][UNITS]
  static constexpr uint32_t pairs = meta + 16 * META * UNITS;         // float [set][turn][half][ROWS]: maxima
  static constexpr uint32_t refs = pairs + 4 * 8 * ROWS;              // float [tile parity][ROWS]: M
  static constexpr uint32_t sums = refs + 4 * 2 * ROWS;               // float [segment parity][set, half][ROWS]
  static constexpr uint32_t bars = sums + 4 * 8 * ROWS;
  static constexpr uint32_t misc = bars + 8 * (4 * STAGES + 32);
  static constexpr size_t smem = 1024 + misc + 32;
  // TMEM columns: scores, two tiles' weights (two bf16 to a column), Q (likewise), O
  static constexpr uint32_t p_col = TILE, q_col = 2 * TILE, o_col = q_col + D / 2, tmem_cols = D == 64 ? 256 : 512;
  static_assert(o_col + D <= tmem_cols);
  static_assert(smem <= 227 * 1024);
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 16 TMEM lanes by N fp32 columns (16, 32 or 64): lane L holds, of every 8 columns, 2 (L % 4) and the one behind it of row
// L / 4 (r[0], r[1]) and of row L / 4 + 8 (r[2], r[3]).
template <int N>
__device__ __forceinline__ void tmem_fragments(uint32_t addr, uint32_t* r) {
  if constexpr (N == 16) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr)
                 : "memory");
  } else if constexpr (N == 32) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
  } else {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
  }
}
__device__ __forceinline__ uint4 lds128(uint32_t p) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two or three waits at once, as a rule over: the polls stand in one block so that their latencies overlap.
__device__ __forceinline__ bool try2(uint32_t b0, uint32_t p0, uint32_t b1, uint32_t p1) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n\t"
      "and.pred p, p, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(b0), "r"(p0), "r"(b1), "r"(p1)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool try3(uint32_t b0, uint32_t p0, uint32_t b1, uint32_t p1, uint32_t b2, uint32_t p2) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q, r;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 r, [%5], %6;\n\t"
      "and.pred p, p, q;\n\t"
      "and.pred p, p, r;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(b0), "r"(p0), "r"(b1), "r"(p1), "r"(b2), "r"(p2)
      : "memory");
  return ok != 0;
}
// For whole warps: true in every lane, or false in every lane (the branches are uniform: a wait that is over costs
// little more than its poll).
template <typename Poll>
__device__ __forceinline__ bool wait_for(Poll poll, volatile int* stop, uint32_t polls) {
  for (uint32_t i = 0;; ++i) {
    if (__all_sync(0xffffffffu, poll())) return true;
    if (i >= polls || ((i & 255u) == 255u && __any_sync(0xffffffffu, *stop))) break;
  }
  *stop = 1;
  return false;
}
// bf16 operands, fp32 accumulator, M = 128; B's long side contiguous (MN-major) or not.
template <int N, bool B_MN>
__host__ __device__ constexpr uint32_t idesc() {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((B_MN ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(ROWS >> 4) << 24);
}
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap* map, uint32_t bar, int chunk, int head,
                                         int row) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::
          "r"(dst), "l"(map), "r"(bar), "r"(0), "r"(chunk), "r"(head), "r"(row)
      : "memory");
}

__device__ __forceinline__ void tma_unit(uint32_t dst, const CUtensorMap* map, uint32_t bar, int row, int head) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::
          "r"(dst), "l"(map), "r"(bar), "r"(0), "r"(row), "r"(0), "r"(head)
      : "memory");
}

// A run of units of one tile and head.
struct Segment {
  int tile, head, lo, hi;   // units [lo, hi) of the tile's list
  int slot;                 // of partials; -1: the whole list, straight to the output
  int parts;                // with lo = 0: of the list
  RowTile rows;
};
// How the units are shared out.  They stand in a row: tile after tile, in each the KV heads, in each the tile's list;
// every CTA takes a run of them.  A list counts kStart units more than it has, about what a CTA loses where it goes on to
// another list (results out, Q in).  Where all groups have the same few (nm) tiles, nm CTAs work as a team: the lists
// of a group's tiles are walked side by side, one CTA a tile, so that the prefix that they all read is fetched from
// DRAM once and found in L2 after that.  Where a list is short whatever the lengths (`whole`), runs end with lists:
// nothing is joined.
struct Shares {
  int nm;           // CTAs of a team (1: no teams)
  int runs;         // runs that the units are cut into
  int all;          // units, over all heads (of the longest list of each group, where there are teams)
  bool whole;
  __device__ int start(int run) const {  // all * run / runs, without an overflow
    const int q = all / runs;
    return run * q + run * (all - q * runs) / runs;
  }
};
// Tile m of the group that starts with sequence `first` and has `spt` of them to a tile.
__device__ __forceinline__ int team_tile(const PrefixAttn& a, int first, int spt, int m) {
  return a.tps > 1 ? first * a.tps + m : first + m * spt;
}
// x / spt (x < 512).
__device__ __forceinline__ int by_spt(const PrefixAttn& a, int x) { return (x * a.spt_inv) >> 16; }
struct Walk {
  int pos, end;
  int at;           // tile (group, where there are teams) that pos is in
  __device__ Walk(const PrefixAttn& a, const Shares& sh, const int* pref, int n) : at(0) {
    const int run = (int)blockIdx.x / sh.nm;
    pos = end = 0;
    if (run >= sh.runs) return;
    if (sh.whole) {
      const int lists = n * a.hkv, l0 = lists * run / sh.runs, l1 = lists * (run + 1) / sh.runs;
      auto start = [&](int l) {
        const int t = l / a.hkv;
        return t >= n ? sh.all : pref[t] * a.hkv + (l - t * a.hkv) * (pref[t + 1] - pref[t]);
      };
      pos = start(l0);
      end = start(l1);
    } else {
      pos = sh.start(run);
      end = sh.start(run + 1);
    }
    while (n > 1) {  // the last one that starts at or before pos
      const int half = n / 2;
      if (pref[at + half] * a.hkv <= pos) at += half, n -= half;
      else n = half;
    }
  }
  __device__ bool next(const PrefixAttn& a, const Shares& sh, const int* pref, const int* units_s, const int2* info,
                       const int* first_s, const int* spt_s, Segment& s) {
    while (pos < end) {
      while (pref[at + 1] * a.hkv <= pos) ++at;
      const int list = pref[at + 1] - pref[at], first = pref[at] * a.hkv;
      s.head = (pos - first) / list;
      const int base = first + s.head * list + kStart;  // of the list's first unit
      s.tile = sh.nm > 1 ? team_tile(a, first_s[at], spt_s[at], (int)blockIdx.x % sh.nm) : at;
      const int units = units_s[s.tile];
      s.lo = max(pos - base, 0);
      s.hi = min(min(base - kStart + list, end) - base, units);
      pos = min(base - kStart + list, end);
      if (s.lo >= s.hi) continue;
      const bool all = s.lo == 0 && s.hi == units;
      s.slot = all ? -1 : s.lo > 0 ? 2 * (int)blockIdx.x : 2 * (int)blockIdx.x + 1;
      s.parts = 1;
      if (s.lo == 0 && !all) {
        int run = (int)blockIdx.x / sh.nm;
        while (sh.start(run + 1) < base + units) ++run;  // the run that the last unit is in
        s.parts = run - (int)blockIdx.x / sh.nm + 1;
      }
      const int2 t = info[s.tile];
      s.rows.seq0 = t.x & 0xffff;
      s.rows.nseq = a.tps > 1 ? 1 : t.x >> 16;
      s.rows.part = a.tps > 1 ? t.x >> 16 : 0;
      s.rows.group = t.y & 0xffff;
      s.rows.first = t.y >> 16;
      return true;
    }
    return false;
  }
};

// Units of the prefix and of a sequence's tail (which begins with the unit that holds position P, if that is a part).
__device__ __forceinline__ int prefix_units(int P) { return (P + 15) / 16; }
__device__ __forceinline__ int tail_units(const PrefixAttn& a, int seq, int ql, int P) {
  const int n = min(seq, a.cap);
  return ql > 0 && n > P ? (n + 15) / 16 - P / 16 : 0;
}

// Row r of the segment once more, alone: dims [d0, d0 + D / 4) of sum_j w_j v_j over the positions that it sees, weights
// as the tensor cores had them.  For whole warps.
template <int D>
__device__ __noinline__ void row_again(const PrefixAttn& a, const Segment& sg, int seq, int pos, int64_t at, float c,
                                       float M, int d0, float k, float* to_f32, bf16* to_bf16) {
  constexpr int PL = D / 32, HL = D >= 128 ? D / 128 : 1;  // (of 64 dims every second lane's sums are not used)
  const int lane = threadIdx.x & 31;
  const bf16* pages = reinterpret_cast<const bf16*>(a.pages) + a.layer;
  const int P = prefix_of(a, sg.rows.group);
  float q[PL], o[HL];
#pragma unroll
  for (int i = 0; i < PL; ++i) {
    q[i] = to_f(ld_act(reinterpret_cast<const bf16*>(a.q) + at + lane + 32 * i));
    if (a.scale < 0.f) q[i] = -q[i];
  }
#pragma unroll
  for (int i = 0; i < HL; ++i) o[i] = 0.f;
  int before = prefix_units(P);  // units before the sequence's tail
  auto units = [&](int b) { return tail_units(a, ld_act(a.seq_lens + b), new_tokens(a, b), P); };
  for (int i = 0; i < seq; ++i) before += units(sg.rows.seq0 + i);
  const int own = units(sg.rows.seq0 + seq);
  const int end = min(min(ld_act(a.seq_lens + sg.rows.seq0 + seq), a.cap), pos + 1);
  for (int pass = 0; pass < 2; ++pass) {
    const int first = pass ? before : 0, n = pass ? own : prefix_units(P);
    const int row = pass ? sg.rows.seq0 + seq : sg.rows.first;
    for (int u = max(sg.lo, first); u < min(sg.hi, first + n); ++u) {
      const int p0 = 16 * (u - first + (pass ? P / 16 : 0));
      for (int j = max(p0, pass ? P : 0); j < min(p0 + 16, pass ? end : min(P, pos + 1)); ++j) {
        const int blk = ld_act(a.tables + (int64_t)row * a.max_blocks + j / a.block_size);
        if ((unsigned)blk >= (unsigned)a.num_blocks) continue;
        const bf16* kr = pages + (((int64_t)blk * a.block_size + j % a.block_size) * a.hkv + sg.head) * D;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < PL; ++i) s = fmaf(q[i], to_f(ld_act(kr + lane + 32 * i)), s);
        const float w = round_bf16(ex2(fmaf(warp_sum(s), c, -M)));
#pragma unroll
        for (int i = 0; i < HL; ++i) o[i] = fmaf(w, to_f(ld_act(kr + a.plane + d0 + lane % (D / 4) + 32 * i)), o[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < HL; ++i) {
    if (lane >= D / 4) continue;
    if (to_f32) to_f32[d0 + lane + 32 * i] = o[i];
    else to_bf16[d0 + lane + 32 * i] = __float2bfloat16_rn(o[i] * k);
  }
}

// Where the join finds the parts of a tile's list: for each of its sequences (from `i`, every `by`-th) the first part,
// their number, the step from part to part, and the sequence's first row.
__device__ __forceinline__ void put_parts(const PrefixAttn& a, int2 info, int tile, int head, int first, int parts,
                                          int step, int i, int by) {
  const int seq0 = info.x & 0xffff, n = a.tps > 1 ? 1 : info.x >> 16;
  for (; i < n; i += by)
    a.parts[(int64_t)(a.tps > 1 ? tile : seq0 + i) * a.hkv + head] = make_int4(first, parts, step, a.tps > 1 ? 0 : i * a.R);
}

template <int D>
__global__ void __launch_bounds__(THREADS, 1)
prefix_attention_tc_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ CUtensorMap vmap,
                           const __grid_constant__ CUtensorMap qmap,
                           const __grid_constant__ PrefixAttn a) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = tc::smem_u32(smem_raw), sm = (raw + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (sm - raw);
  int* pref = reinterpret_cast<int*>(gen + C::pref);
  int* units_s = reinterpret_cast<int*>(gen + C::units);
  int2* info = reinterpret_cast<int2*>(gen + C::info);
  int* seq_s = reinterpret_cast<int*>(gen + C::seq);
  uint16_t* ql_s = reinterpret_cast<uint16_t*>(gen + C::ql);
  int* pre_s = reinterpret_cast<int*>(gen + C::pre);
  int* first_s = reinterpret_cast<int*>(gen + C::first);
  int* spt_s = reinterpret_cast<int*>(gen + C::spt);
  int4* meta = reinterpret_cast<int4*>(gen + C::meta);
  float* pair_s = reinterpret_cast<float*>(gen + C::pairs);
  float* ref_s = reinterpret_cast<float*>(gen + C::refs);
  float* sum_s = reinterpret_cast<float*>(gen + C::sums);
  auto bar = [&](int i) { return sm + C::bars + 8 * i; };
  auto full = [&](int s) { return bar(s); };
  auto freed = [&](int s) { return bar(C::STAGES + s); };
  auto v_full = [&](int s) { return bar(2 * C::STAGES + s); };
  auto v_freed = [&](int s) { return bar(3 * C::STAGES + s); };
  constexpr int B0 = 4 * C::STAGES;
  auto s_full = [&](int s) { return bar(B0 + s); };      // scores of a set's tile
  auto p_full = [&](int s) { return bar(B0 + 2 + s); };  // weights of a set's tile
  auto added = [&](int s) { return bar(B0 + 4 + s); };   // a set's tile is in O
  const uint32_t s_free = bar(B0 + 6), q_tmem = bar(B0 + 7), q_free = bar(B0 + 8), o_free = bar(B0 + 9),
                 drained = bar(B0 + 10);
  auto pair = [&](int set, int q) { return bar(B0 + 12 + 4 * set + q); };
  auto decided = [&](int set, int q) { return bar(B0 + 20 + 4 * set + q); };
  auto summed = [&](int q) { return bar(B0 + 28 + q); };
  uint32_t* slot = reinterpret_cast<uint32_t*>(gen + C::misc);
  volatile int* stop = reinterpret_cast<volatile int*>(slot + 1);
  auto held = [&](uint32_t b, uint32_t parity) {
    return wait_for([&] { return tc::mbar_try_wait(b, parity); }, stop, a.polls);
  };

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      tc::mbar_init(full(s), 1);
      tc::mbar_init(freed(s), 1);
      tc::mbar_init(v_full(s), 1);
      tc::mbar_init(v_freed(s), 1);
    }
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(s_full(s), 1);
      tc::mbar_init(p_full(s), SETW);
      tc::mbar_init(added(s), 1);
      for (int q = 0; q < 4; ++q) {
        tc::mbar_init(pair(s, q), 2);
        tc::mbar_init(decided(s, q), 2);
      }
    }
    for (int q = 0; q < 4; ++q) tc::mbar_init(summed(q), 4);
    tc::mbar_init(s_free, SETW);
    tc::mbar_init(q_tmem, SETW);
    tc::mbar_init(q_free, 1);
    tc::mbar_init(o_free, 2 * SETW);
    tc::mbar_init(drained, 1);
    *stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&vmap) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&qmap) : "memory");
  }
  if (warp == THREADS / 32 - 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(slot)),
                 "r"(C::tmem_cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // parameters come into the constant cache where they are first used: what comes next, all at once
  asm volatile("" ::"r"(a.B), "r"(a.T), "r"(a.groups), "r"(a.tiles), "r"(a.spt), "r"(a.hkv), "r"(a.block_size), "l"(a.tables),
               "l"(a.parts), "l"(a.starts));
  pdl_wait();
  pdl_trigger();

  // ---------------------------------------------------------------- the tiles and their units
  // A tile goes by the number of its first sequence (times tps, plus its slice, where a sequence has several): numbers in
  // between stand for nothing.
  {
    static_assert(THREADS > kMaxTiles);  // a thread a sequence, group and tile
    int seq = 0, ql = 0, start = 0, end = 0, P = 0;
    if (tid < a.B) {
      seq = ld_act(a.seq_lens + tid);
      ql = a.q_lens ? ld_act(a.q_lens + tid) : a.T;
    }
    if (tid < a.groups) {
      start = ld_act(a.starts + tid);
      end = ld_act(a.starts + tid + 1);
      P = ld_act(a.prefixes + tid);
    }
    if (tid < a.tiles) {
      info[tid] = make_int2(-1, 0);
      units_s[tid] = 0;
    }
    ql = clamped(ql, a.T);
    start = clamped(start, a.B);
    end = clamped(end, a.B);
    if (tid < a.B) {
      seq_s[tid] = seq;
      ql_s[tid] = (uint16_t)ql;  // (as many as fit the tiles that there may be)
    }
    if (tid < a.groups) {
      first_s[tid] = start;
      pre_s[tid] = clamped(P, a.cap);
      if (tid == a.groups - 1) first_s[a.groups] = end;
    }
    // tiles of the group, and sequences of each: as even as they come
    int of_group;
    auto even = [&] {
      of_group = a.tps > 1 ? (end - start) * a.tps : by_spt(a, end - start + a.spt - 1);
      if (tid < a.groups) {
        spt_s[tid] = a.tps > 1 || of_group < 1 ? 1 : (end - start + of_group - 1) / of_group;
        if (tid == 0) slot[3] = of_group;
      }
    };
    const bool ascends = start <= end;
    end = max(start, end);
    even();
    if (!__syncthreads_and(ascends)) {  // a start below one before it counts as that one: no row is in two groups
      if (tid == 0)
        for (int g = 1; g <= a.groups; ++g) first_s[g] = max(first_s[g], first_s[g - 1]);
      __syncthreads();
      if (tid < a.groups) {
        start = first_s[tid];
        end = first_s[tid + 1];
      }
      even();
      __syncthreads();
    }
    const int nm = slot[3];  // tiles of the first group: of all, if there are to be teams
    const bool same = tid >= a.groups || nm == of_group;
    int g = 0, s = 0, e = 0;
    if (tid < a.B) {
      int n = a.groups;
      while (n > 1) {  // the last group that starts at or before the sequence
        const int half = n / 2;
        if (first_s[g + half] <= tid) g += half, n -= half;
        else n = half;
      }
      s = first_s[g];
      e = first_s[g + 1];
    }
    if (tid >= s && tid < e) {
      const int own = pre_s[g], tail = tail_units(a, seq, ql, own), k = tid - s;
      const int spt = spt_s[g], seq0 = s + k / spt * spt;
      const bool lead = seq0 == tid;
      for (int p = 0; p < a.tps; ++p) {
        const int t = seq0 * a.tps + p;
        atomicAdd(&units_s[t], tail + (lead ? prefix_units(own) : 0));
        if (lead) info[t] = make_int2(tid | (a.tps > 1 ? p : min(spt, e - tid)) << 16, g | s << 16);
      }
    } else if (tid < a.B) {  // before the first group or behind the last: a tile of its own that sees nothing
      for (int p = 0; p < a.tps; ++p) info[tid * a.tps + p] = make_int2(tid | (a.tps > 1 ? p : 1) << 16, 0);
    }
    const bool team = __syncthreads_and(same) && nm > 1 && nm <= kMaxTeam && nm * 4 <= (int)gridDim.x && !a.whole;
    if (warp == 0) {
      const int lists = team ? a.groups : a.tiles, per = (lists + 31) / 32;
      int sum = 0, starts = 0;
      for (int i = 0; i < per; ++i) {
        const int t = lane * per + i;
        int n = 0;
        if (t < lists) {
          if (team) {
            for (int m = 0; m < nm; ++m) n = max(n, units_s[team_tile(a, first_s[t], spt_s[t], m)]);
          } else {
            n = units_s[t];
          }
          if (n > 0) n += kStart, ++starts;
          pref[1 + t] = n;
        }
        sum += n;
      }
      int incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      int before = incl - sum;
      for (int i = 0; i < per; ++i) {
        const int t = lane * per + i;
        if (t < lists) pref[1 + t] = before += pref[1 + t];
      }
      starts = __reduce_add_sync(0xffffffffu, starts);
      if (lane == 0) {
        pref[0] = 0;
        slot[2] = starts;
        slot[3] = team ? nm : 1;
      }
    }
    for (int t = blockIdx.x; t < a.tiles; t += gridDim.x) {  // rows that see nothing
      const int2 in = info[t];
      if (in.x < 0 || units_s[t] != 0) continue;
      const int seq0 = in.x & 0xffff, n = a.tps > 1 ? (in.x >> 16 ? 0 : 1) : in.x >> 16;
      const int64_t row = (int64_t)a.T * a.hq * D / 8;
      for (int64_t i = tid; i < n * row; i += THREADS)
        reinterpret_cast<uint4*>(a.out)[seq0 * row + i] = make_uint4(0, 0, 0, 0);
      for (int h = tid; h < a.hkv; h += THREADS) put_parts(a, in, t, h, 0, 1, 0, 0, 1);
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *slot;
  Shares sh;
  sh.nm = slot[3];
  const int lists = sh.nm > 1 ? a.groups : a.tiles;
  sh.all = pref[lists] * a.hkv;
  sh.whole = a.whole;
  sh.runs = max(1, min((int)gridDim.x / sh.nm, sh.whole ? lists * a.hkv : (sh.all - kStart * (int)slot[2] * a.hkv) / kMinUnits));
  Walk walk(a, sh, pref, lists);
  Segment sg;
  const float c = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-38f);  // not 0: keeps the mask's infinity an infinity
  int jg = 0;  // tiles before this segment

  if (warp < 2 * SETW) {
    // -------------------------------------------------------------- rows
    const int quad = warp & 3, half = warp >> 2 & 1, set = warp / SETW;
    const int r = quad * 32 + lane;               // TMEM lanes 32 quad .., positions HALF half .. of a tile
    const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
    int swaps = 0, n = 0;  // n: stages of K filled before
    bool ok = a.polls > 0;  // (0: gives up before the first wait)
    for (int seg = 0; walk.next(a, sh, pref, units_s, info, first_s, spt_s, sg); ++seg) {
      const int tiles = (sg.hi - sg.lo + UNITS - 1) / UNITS, last = jg + tiles - 1;
      const RowAt w = row_at<D>(a, sg.rows, sg.head, r, a.tile_rows, seq_s, ql_s);
      if (sg.lo == 0 && warp == SETW)
        put_parts(a, info[sg.tile], sg.tile, sg.head, 2 * (int)blockIdx.x + 1, sg.parts, 2 * sh.nm, lane, 32);
      const bool real = w.pos >= 0;
      const bool busy = __any_sync(0xffffffffu, real);
      if (set == 1) {
        // this thread's half of its row of Q out of the ring into TMEM (rows that are not there may hold anything)
        ok = ok && (seg == 0 || held(q_free, (seg - 1) & 1)) && held(full(n % C::STAGES), (n / C::STAGES) & 1) &&
             (C::QST == 1 || held(full((n + 1) % C::STAGES), ((n + 1) / C::STAGES) & 1));
        if (ok) {
          tc::tc_fence_after();
          const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
          for (int i = 0; i < D / 64; ++i) {  // 32 dims at a time: 4 pieces of 16 bytes
            const int dim = half * (D / 2) + 32 * i;
            const int ch = dim / 64;
            const uint32_t line = sm + (n + ch / C::CPS) % C::STAGES * C::KS + ch % C::CPS * (ROWS * 128) + r * 128;
            uint32_t y[16];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint4 v = lds128(line + ((((dim % 64) / 8 + k) ^ (r & 7)) << 4));
              y[4 * k] = v.x ^ flip;
              y[4 * k + 1] = v.y ^ flip;
              y[4 * k + 2] = v.z ^ flip;
              y[4 * k + 3] = v.w ^ flip;
            }
            tc::tmem_store16(lanes + C::q_col + dim / 2, y);
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(q_tmem);
        }
      }
      n += C::QST + tiles;
      // M: what the weights are relative to
      float M = kNothing, l = 0.f;
#pragma unroll 1
      for (int jt = jg + ((jg ^ set) & 1); ok && jt <= last; jt += 2) {
        const bool first = jt == jg;
        ok = held(s_full(set), (jt >> 1) & 1);  // (and the tile's units are described: that was before K came in)
        if (!ok) break;
        tc::tc_fence_after();
        uint32_t x[HALF];
        uint32_t see = 0;
        bool none = true;
        float m = kNothing;
        if (busy) {
          tc::tmem_load32(lanes + half * HALF, x);
          // which of this thread's positions its row sees
          const int4* mt = meta + (jt % META) * UNITS + half * (UNITS / 2);
#pragma unroll
          for (int u = 0; u < UNITS / 2; ++u) {
            const int4 d = mt[u];  // first position, positions from, to, whose (-1: every row's)
            const int to = min(min(d.z, w.pos + 1) - d.x, 16), from = max(d.y - d.x, 0);
            uint32_t bits = to > from ? (0xffffu >> (16 - to)) & (0xffffu << from) : 0u;
            if (d.w >= 0 && d.w != w.seq) bits = 0;
            see |= bits << (16 * u);
          }
          if (!real) see = 0xffffffffu;  // nobody asks for the row: no reason to mask
          const bool all_seen = __all_sync(0xffffffffu, see == 0xffffffffu);
          none = !all_seen && __all_sync(0xffffffffu, see == 0 || !real);
          tc::tmem_ready(x);
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(s_free);
          if (!none) {
            if (!all_seen) {
#pragma unroll
              for (int i = 0; i < HALF; ++i)
                if (!(see >> i & 1)) x[i] = 0xff800000u;
            }
            float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
            for (int i = 0; i < HALF; i += 8) {
              m0 = fmaxf(m0, fmaxf(__uint_as_float(x[i]), __uint_as_float(x[i + 1])));
              m1 = fmaxf(m1, fmaxf(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])));
              m2 = fmaxf(m2, fmaxf(__uint_as_float(x[i + 4]), __uint_as_float(x[i + 5])));
              m3 = fmaxf(m3, fmaxf(__uint_as_float(x[i + 6]), __uint_as_float(x[i + 7])));
            }
            m = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
            m = fmaxf(m * c, kNothing);  // a NaN score counts as the lowest value here and spoils the sums
          }
        }
        if (!busy && lane == 0) tc::mbar_arrive(s_free);
        float* at = pair_s + (set * 2 + (swaps & 1)) * 2 * ROWS;
        at[half * ROWS + r] = m;
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(pair(set, quad));
        // the other half's maxima; the tile before's M; and the weights of two tiles before have been used (`decided`
        // says that too).  A barrier in its first phase has no phase before that: waits for parity 1 are over.
        const uint32_t b0 = pair(set, quad), b1 = first ? b0 : decided(set ^ 1, quad), p0 = swaps & 1,
                       p1 = first ? p0 : ((jt - 1) >> 1) & 1;
        ok = wait_for([&] { return try3(b0, p0, b1, p1, added(set), ((jt >> 1) - 1) & 1); }, stop, a.polls);
        if (!ok) break;
        ++swaps;
        const float before = first ? kNothing : ref_s[((jt - 1) & 1) * ROWS + r];
        m = fmaxf(m, at[(half ^ 1) * ROWS + r]);
        const bool moved = real && m > before + kSpan;
        const float now = moved ? m : before;
        if (half == 0) ref_s[(jt & 1) * ROWS + r] = now;
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(decided(set, quad));
        if (busy) {
          if (now != M) {
            l *= ex2(M - now);
            M = now;
          }
          uint32_t p[HALF / 2];
          if (none) {
#pragma unroll
            for (int i = 0; i < HALF / 2; ++i) p[i] = 0;
          } else {
            float2 s0 = make_float2(0.f, 0.f), s1 = s0;
            const float2 c2 = make_float2(c, c), o2 = make_float2(-M, -M);
#pragma unroll
            for (int i = 0; i < HALF; i += 4) {
              float2 e = tc::fma2(make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), c2, o2);
              float2 d = tc::fma2(make_float2(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])), c2, o2);
              e = make_float2(ex2(e.x), ex2(e.y));
              d = make_float2(ex2(d.x), ex2(d.y));
              s0 = tc::add2(s0, e);
              s1 = tc::add2(s1, d);
              p[i / 2] = pack_bf16(e.x, e.y);
              p[i / 2 + 1] = pack_bf16(d.x, d.y);
            }
            l += (s0.x + s0.y) + (s1.x + s1.y);
          }
          tc::tc_fence_after();
          tc::tmem_store16(lanes + C::p_col + set * (TILE / 2) + half * (HALF / 2), p);
          // (a row that has seen nothing has zeros in O, or what it is worked out again for: nothing to rescale)
          const bool shift = moved && before > kNothing;
          if (__any_sync(0xffffffffu, shift)) {  // half of O each, once the tile before has been added
            ok = held(added(set ^ 1), ((jt - 1) >> 1) & 1);
            if (!ok) break;
            tc::tc_fence_after();
            const float f = shift ? ex2(before - now) : 1.f;
#pragma unroll 1
            for (int i = half * (D / 2); i < (half + 1) * (D / 2); i += 32) {
              uint32_t y[32];
              tc::tmem_load32(lanes + C::o_col + i, y);
              tc::tmem_ready(y);
#pragma unroll
              for (int k = 0; k < 32; ++k) y[k] = __float_as_uint(__uint_as_float(y[k]) * f);
              tc::tmem_store32(lanes + C::o_col + i, y);
            }
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(p_full(set));
      }
      if (ok) {
        // the row's four threads add up what they have, relative to the last tile's M
        // (of its own last tile a thread has M; the other half may not have written it down yet)
        const bool other = (last & 1) != set;
        if (other) ok = held(decided(set ^ 1, quad), (last >> 1) & 1);
        const float now = ok && other ? ref_s[(last & 1) * ROWS + r] : M;
        float* to = sum_s + (seg & 1) * 4 * ROWS + r;
        to[(2 * set + half) * ROWS] = l == 0.f ? 0.f : l * ex2(M - now);
        M = now;
        __syncwarp();
        if (ok && lane == 0) tc::mbar_arrive(summed(quad));
        ok = ok && held(summed(quad), seg & 1);
        l = (to[0] + to[ROWS]) + (to[2 * ROWS] + to[3 * ROWS]);
      }
      jg += tiles;
      ok = ok && held(added(last & 1), (last >> 1) & 1);
      tc::tc_fence_after();
      const float nan = __int_as_float(0x7fc00000);
      const bool direct = sg.slot < 0;
      const int po = max(sg.slot, 0) * ROWS + quad * 32;
      if (!direct && half == 0 && set == 0) a.ws_ml[po + lane] = make_float2(M, !real ? 0.f : ok ? l : nan);
      const bool any = real && l != 0.f;  // l is NaN, not 0, where a seen score is
      // a row's scale; -1: nothing to write
      float k = any ? 1.f / l : 0.f;
      if (!ok) {
        if (lane == 0) atomicExch(&gave_up, 1u);
        k = real ? nan : 0.f;
      }
      // A warp takes D / 4 dims of its 32 rows, fragments of 8 rows by 8 dims: a row's 8 dims lie in 4 lanes.
      const int exist = w.at >= 0 ? (int)(w.at / D) : -1, q4 = 2 * (lane & 3), d0 = (2 * half + set) * (D / 4);
      uint32_t bad = 0;  // rows that hold an infinity or NaN
#pragma unroll 1
      for (int h = 0; h < 32; h += 16) {
        const int r0 = h + (lane >> 2), r1 = r0 + 8;
        const float k0 = __shfl_sync(0xffffffffu, k, r0), k1 = __shfl_sync(0xffffffffu, k, r1);
        const int e0 = __shfl_sync(0xffffffffu, exist, r0), e1 = __shfl_sync(0xffffffffu, exist, r1);
        float odd0 = 0.f, odd1 = 0.f;  // NaN once an element is not finite
        constexpr int NF = D / 32;  // fragments of 8 dims
        uint32_t y[4 * NF];
        if (ok && busy) {
          tmem_fragments<D / 4>(lanes + ((uint32_t)h << 16) + C::o_col + d0, y);
#pragma unroll
          for (int i = 0; i < NF; ++i) {
            odd0 = fmaf(__uint_as_float(y[4 * i]), 0.f, fmaf(__uint_as_float(y[4 * i + 1]), 0.f, odd0));
            odd1 = fmaf(__uint_as_float(y[4 * i + 2]), 0.f, fmaf(__uint_as_float(y[4 * i + 3]), 0.f, odd1));
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4 * NF; ++i) y[i] = 0x7fc00000u;  // (not `busy`: nobody reads it)
        }
        if (direct) {
          // (O may be anything where a row sees nothing)
          bf16* to = reinterpret_cast<bf16*>(a.out) + d0 + q4;
          if (e0 >= 0) {
#pragma unroll
            for (int i = 0; i < NF; ++i)
              *reinterpret_cast<uint32_t*>(to + (int64_t)e0 * D + 8 * i) =
                  k0 == 0.f ? 0u : pack_bf16(__uint_as_float(y[4 * i]) * k0, __uint_as_float(y[4 * i + 1]) * k0);
          }
          if (e1 >= 0) {
#pragma unroll
            for (int i = 0; i < NF; ++i)
              *reinterpret_cast<uint32_t*>(to + (int64_t)e1 * D + 8 * i) =
                  k1 == 0.f ? 0u : pack_bf16(__uint_as_float(y[4 * i + 2]) * k1, __uint_as_float(y[4 * i + 3]) * k1);
          }
        } else {
          float* to = a.ws_o + (int64_t)po * D + d0 + q4;
          if (k0 != 0.f) {
#pragma unroll
            for (int i = 0; i < NF; ++i)
              *reinterpret_cast<uint2*>(to + r0 * D + 8 * i) = make_uint2(y[4 * i], y[4 * i + 1]);
          }
          if (k1 != 0.f) {
#pragma unroll
            for (int i = 0; i < NF; ++i)
              *reinterpret_cast<uint2*>(to + r1 * D + 8 * i) = make_uint2(y[4 * i + 2], y[4 * i + 3]);
          }
        }
        // the lanes of a row are four in a row
        const uint32_t b0 = __ballot_sync(0xffffffffu, odd0 != 0.f), b1 = __ballot_sync(0xffffffffu, odd1 != 0.f);
        if (b0 | b1)
          for (int i = 0; i < 8; ++i) {
            if (b0 >> (4 * i) & 15u) bad |= 1u << (h + i);
            if (b1 >> (4 * i) & 15u) bad |= 1u << (h + 8 + i);
          }
      }
      // rows that V's infinities or NaN have reached: seen ones come out as they are, others are taken out
      for (uint32_t left = __ballot_sync(0xffffffffu, any && l == l && (bad >> lane & 1)); left; left &= left - 1) {
        const int from = __ffs(left) - 1;
        const int64_t at = __shfl_sync(0xffffffffu, w.at, from);
        row_again<D>(a, sg, __shfl_sync(0xffffffffu, w.seq, from), __shfl_sync(0xffffffffu, w.pos, from), at, c,
                     __shfl_sync(0xffffffffu, M, from), d0, __shfl_sync(0xffffffffu, k, from),
                     direct ? nullptr : a.ws_o + (int64_t)(po + from) * D,
                     direct ? reinterpret_cast<bf16*>(a.out) + at : nullptr);
      }
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(o_free);
    }
  } else if (warp != 2 * SETW + 1) {
    // -------------------------------------------------------------- pages
    uint32_t lead;    // one lane issues: operands of the copies then stay in uniform registers
    asm volatile("{.reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p;}" : "=r"(lead));
    const bool is_v = warp != 2 * SETW;
    const uint32_t ring = sm + (is_v ? C::v : 0u);
    int* cum = reinterpret_cast<int*>(gen + C::cum) + (is_v ? ROWS + 4 : 0);
    auto filled = [&](int s) { return is_v ? v_full(s) : full(s); };
    auto emptied = [&](int s) { return is_v ? v_freed(s) : freed(s); };
    const int plane_row = ((is_v ? a.num_layers : 0) + a.layer_no) * a.num_blocks * a.block_size;
    int n = 0;        // stages filled
    bool ok = a.polls > 0;
    for (int seg = 0; ok && walk.next(a, sh, pref, units_s, info, first_s, spt_s, sg); ++seg) {
      const int tiles = (sg.hi - sg.lo + UNITS - 1) / UNITS;
      const int P = pre_s[sg.rows.group], pu = prefix_units(P);
      int before = pu;
      for (int i0 = 0; i0 < sg.rows.nseq; i0 += 32) {
        const int i = i0 + lane, b = sg.rows.seq0 + i;
        const int t = i < sg.rows.nseq ? tail_units(a, seq_s[b], ql_s[b], P) : 0;
        int incl = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += y;
        }
        if (i < sg.rows.nseq) cum[i] = before + incl - t;
        before += __shfl_sync(0xffffffffu, incl, 31);
      }
      __syncwarp();
      // units of a batch of tiles, a lane each: where their rows are, and who sees them.  The table is read a batch ahead.
      constexpr int BATCH = 32 / UNITS;
      int4 next_m;
      int next_blk;
      auto look = [&](int j0) {
        const int u = sg.lo + j0 * UNITS + lane;
        next_m = make_int4(0, 0, 0, -1);
        next_blk = -1;
        if (u < sg.hi) {
          int from = sg.rows.first;
          next_m = make_int4(16 * u, 0, P, -1);
          if (u >= pu) {
            int owner = 0;
            for (int step = sg.rows.nseq; step > 1;) {  // the last sequence whose tail starts at or before u
              const int hf = step / 2;
              if (cum[owner + hf] <= u) owner += hf, step -= hf;
              else step = hf;
            }
            from = sg.rows.seq0 + owner;
            next_m = make_int4(16 * (P / 16 + u - cum[owner]), P, min(seq_s[from], a.cap), owner);
          }
          next_blk = ld_act(a.tables + (int64_t)from * a.max_blocks + next_m.x / a.block_size);
        }
      };
      int4 m;
      int vrow = 0;  // rows of this lane's unit
      auto advance = [&] {
        const bool there = (unsigned)next_blk < (unsigned)a.num_blocks;
        m = there ? next_m : make_int4(0, 0, 0, -1);
        int row = there ? next_blk * a.block_size + next_m.x % a.block_size : 0;
        // units that are not there fetch the batch's first rows: finite values as a rule, and no bytes of DRAM
        const int first = __shfl_sync(0xffffffffu, row, 0);
        if (!there) row = first;
        vrow = row;
      };
      look(0);
      // Q: rows of all of the tile's tokens and heads, 64 dims at a time
      for (int h = 0; ok && !is_v && h < C::QST; ++h, ++n) {
        const int st = n % C::STAGES;
        ok = n < C::STAGES || held(freed(st), (n / C::STAGES - 1) & 1);
        if (!ok) break;
        if (lead) {
          tc::mbar_expect_tx(full(st), C::CPS * a.q_box * 128);
#pragma unroll
          for (int ch = 0; ch < C::CPS; ++ch)
            tma_rows(sm + st * C::KS + ch * (ROWS * 128), &qmap, full(st), h * C::CPS + ch, sg.head * a.G,
                     sg.rows.seq0 * a.T + sg.rows.part * (a.tile_rows / a.G));
        }
        __syncwarp();
      }
      for (int j = 0; ok && j < tiles; ++j, ++n) {
        if (j % BATCH == 0) {
          advance();
          look(j + BATCH);
        }
        const int jt = jg + j, st = n % C::STAGES;
        if (!is_v && lane / UNITS == j % BATCH) meta[(jt % META) * UNITS + lane % UNITS] = m;
        ok = n < C::STAGES || held(emptied(st), (n / C::STAGES - 1) & 1);
        if (!ok) break;
        int rows[UNITS];
#pragma unroll
        for (int u = 0; u < UNITS; ++u) rows[u] = plane_row + __shfl_sync(0xffffffffu, vrow, (j % BATCH) * UNITS + u);
        __syncwarp();
        if (lead) {
          const uint32_t to = ring + st * (is_v ? C::KV : C::KS);
          tc::mbar_expect_tx(filled(st), C::KV);
          if (is_v) {
#pragma unroll
            for (int u = 0; u < UNITS; ++u) tma_unit(to + u * (16 * D * 2), &vmap, filled(st), rows[u], sg.head);
          } else {
#pragma unroll
            for (int u = 0; u < UNITS; ++u)
#pragma unroll
              for (int ch = 0; ch < D / 64; ++ch)
                tma_rows(to + ch * (TILE * 128) + u * 2048, &map, filled(st), ch, sg.head, rows[u]);
          }
        }
        __syncwarp();
      }
      jg += tiles;
    }
    {  // copies in flight land before shared memory goes, whoever has given up
      for (int i = max(0, n - C::STAGES); i < n; ++i)
        for (uint32_t p = 0; p < kPolls && !tc::mbar_try_wait(filled(i % C::STAGES), (i / C::STAGES) & 1); ++p) {}
    }
    __syncwarp();
  } else {
    // -------------------------------------------------------------- products
    // The whole warp walks the loop and one elected lane issues, so that addresses and descriptors stay in uniform
    // registers.
    uint32_t lead;
    asm volatile("{.reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p;}" : "=r"(lead));
    int n = 0, nv = 0;  // stages of K, of V used
    bool ok = a.polls > 0;
    auto ready = [&](uint32_t b0, uint32_t p0, uint32_t b1, uint32_t p1) {
      const bool yes = wait_for([&] { return try2(b0, p0, b1, p1); }, stop, a.polls);
      tc::tc_fence_after();
      return yes;
    };
    auto scores = [&](int jt, bool is_last) {
      const int s = n % C::STAGES;
      // (no scores before the first ones: a wait for parity 1 of a barrier in its first phase is over)
      if (!ready(full(s), (n / C::STAGES) & 1, s_free, (jt - 1) & 1)) return false;
      const uint64_t kd = tc::sw128_desc(sm + s * C::KS);
      if (lead) {
#pragma unroll
        for (int d = 0; d < D / 64; ++d)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            tc::umma_ts(tmem, tmem + C::q_col + d * 32 + 8 * k, kd + d * ((TILE * 128) >> 4) + 2 * k,
                        idesc<TILE, false>(), d || k);
        tc::umma_commit(s_full(jt & 1));
        tc::umma_commit(freed(s));
        if (is_last) tc::umma_commit(q_free);
      }
      ++n;
      return true;
    };
    for (int seg = 0; ok && walk.next(a, sh, pref, units_s, info, first_s, spt_s, sg); ++seg) {
      const int tiles = (sg.hi - sg.lo + UNITS - 1) / UNITS;
      ok = ready(q_tmem, seg & 1, q_tmem, seg & 1);
      if (!ok) break;
      for (int h = 0; h < C::QST; ++h, ++n)
        if (lead) tc::mbar_arrive(freed(n % C::STAGES));  // Q has left the ring
      ok = scores(jg, tiles == 1) && (tiles < 2 || scores(jg + 1, tiles == 2)) && ready(o_free, (seg - 1) & 1, o_free, (seg - 1) & 1);
#pragma unroll 1
      for (int j = 0; ok && j < tiles; ++j) {
        const int jt = jg + j;
        if (j + 2 < tiles) ok = scores(jt + 2, j + 3 == tiles);
        const int s = nv % C::STAGES;
        ok = ok && ready(v_full(s), (nv / C::STAGES) & 1, p_full(jt & 1), (jt >> 1) & 1);
        if (!ok) break;
        const uint64_t vd = tc::mn128_desc<16>(sm + C::v + s * C::KV);
        if (lead) {
#pragma unroll
          for (int k = 0; k < UNITS; ++k)  // 16 positions: 8 columns of P, a unit of V
            tc::umma_ts(tmem + C::o_col, tmem + C::p_col + (jt & 1) * (TILE / 2) + 8 * k, vd + ((16 * D * 2) >> 4) * k,
                        idesc<D, true>(), j || k);
          tc::umma_commit(added(jt & 1));
          tc::umma_commit(v_freed(s));
        }
        ++nv;
      }
      jg += tiles;
    }
    if (!ok) {  // let the products issued so far end before TMEM goes back
      if (lead) tc::umma_commit(drained);
      for (uint32_t i = 0; i < kPolls && !tc::mbar_try_wait(drained, 0); ++i) {}
    }
    __syncwarp();
  }
  __syncthreads();
  if (warp == THREADS / 32 - 1) {
    tc::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::tmem_cols) : "memory");
  }
}

}  // namespace tile

// ------------------------------------------------------------------ join
// out = sum_i w_i o_i / sum_i w_i l_i over a row's parts, w_i = e^(m_i - M).  NW warps a query row, each every NW-th part,
// a lane D / 32 dims.  Bound by latency: where the parts are, then their statistics and sums at once, then (NW = 4)
// the exchange between the warps.
constexpr int kJoinParts = 160;
// Rows up to which four warps take a row: so many CTAs are there at once (480 rows of some 9 parts: 21.2 against 22.9 us for
// the whole call; 3584 rows of 4 or 5: 80.5 against 78.2).
constexpr int64_t kJoinFew = 148 * 16;

template <typename T, int D, int ROWS, bool LOG2, int NW>
__global__ void __launch_bounds__(128) prefix_join_kernel(const PrefixAttn a) {
  constexpr int PL = D / 32, VL = PL < 4 ? PL : 4, NV = PL / VL, AHEAD = NW == 1 ? 6 : 4;
  __shared__ float2 ml_s[4 / NW][kJoinParts];
  __shared__ __align__(16) float o_s[NW == 1 ? 1 : NW - 1][D];
  __shared__ float sum_s[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % NW, mine = warp / NW;
  const int64_t row = (int64_t)blockIdx.x * (4 / NW) + mine;
  if (row >= (int64_t)a.B * a.T * a.hq) return;  // (NW = 1: whole warps, which do not wait for one another)
  const int h = (int)(row % a.hq), t = (int)(row / a.hq % a.T), b = (int)(row / a.hq / a.T);
  const int head = h / a.G;
  const int in = t * a.G + h % a.G;  // among the sequence's rows of this KV head
  pdl_wait();
  const int4 at = __ldcg(a.parts + (int64_t)(a.tps > 1 ? b * a.tps + in / a.tile_rows : b) * a.hkv + head);
  const int r = a.tps > 1 ? in % a.tile_rows : at.w + in;
  if (at.y == 1 || (unsigned)at.y > (unsigned)kJoinParts || (unsigned)r >= (unsigned)ROWS) return;
  auto part = [&](int i) { return (int64_t)(i == 0 ? at.x : (LOG2 ? at.x & ~1 : at.x) + i * at.z) * ROWS + r; };
  auto sums = [&](int i, float* v) {
    const float* from = a.ws_o + part(i) * D + lane * VL;
#pragma unroll
    for (int x = 0; x < NV; ++x) {
      if constexpr (VL == 4) {
        const float4 y = __ldcg(reinterpret_cast<const float4*>(from + x * 128));
        v[4 * x] = y.x; v[4 * x + 1] = y.y; v[4 * x + 2] = y.z; v[4 * x + 3] = y.w;
      } else {
        const float2 y = __ldcg(reinterpret_cast<const float2*>(from));
        v[0] = y.x; v[1] = y.y;
      }
    }
  };
  float v[AHEAD][PL];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k)  // the first parts' sums before anything is known of their weights
    if (sub + k * NW < at.y) sums(sub + k * NW, v[k]);
  for (int i = lane + 32 * sub; i < at.y; i += 32 * NW) ml_s[mine][i] = __ldcg(a.ws_ml + part(i));
  if constexpr (NW == 1) __syncwarp();
  else __syncthreads();
  float M = -INFINITY;
  for (int i = lane; i < at.y; i += 32) M = fmaxf(M, ml_s[mine][i].x);
  M = warp_max(M);
  float o[PL], L = 0.f;
#pragma unroll
  for (int x = 0; x < PL; ++x) o[x] = 0.f;
  for (int i0 = sub; i0 < at.y; i0 += AHEAD * NW) {
    if (i0 != sub) {
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        if (i0 + k * NW < at.y) sums(i0 + k * NW, v[k]);
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int i = i0 + k * NW;
      if (i >= at.y) break;
      const float2 ml = ml_s[mine][i];
      if (ml.y == 0.f) continue;  // a part that the row sees nothing of is passed over, whatever it left
      const float w = LOG2 ? exp2f(ml.x - M) : expf(ml.x - M);
      L = fmaf(w, ml.y, L);
#pragma unroll
      for (int x = 0; x < PL; ++x) o[x] = fmaf(w, v[k][x], o[x]);
    }
  }
  if constexpr (NW > 1) {
    if (sub > 0) {
#pragma unroll
      for (int x = 0; x < PL; ++x) o_s[sub - 1][lane * VL + x % VL + x / VL * 128] = o[x];
      if (lane == 0) sum_s[sub] = L;
    }
    __syncthreads();
    if (sub > 0) return;
#pragma unroll
    for (int k = 1; k < NW; ++k) {
      L += sum_s[k];
#pragma unroll
      for (int x = 0; x < PL; ++x) o[x] += o_s[k - 1][lane * VL + x % VL + x / VL * 128];
    }
  }
  const float k = L != 0.f ? 1.f / L : 0.f;
  T* out = reinterpret_cast<T*>(a.out) + row * D + lane * VL;
#pragma unroll
  for (int x = 0; x < PL; x += 2) {
    const float y0 = L != 0.f ? o[x] * k : 0.f, y1 = L != 0.f ? o[x + 1] * k : 0.f;
    T* to = out + x % VL + x / VL * 128;
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<__nv_bfloat162*>(to) = __floats2bfloat162_rn(y0, y1);
    else
      *reinterpret_cast<float2*>(to) = make_float2(y0, y1);
  }
}

// ------------------------------------------------------------------ host
inline size_t up256(size_t x) { return (x + 255) & ~size_t(255); }

std::atomic<uint32_t> wait_polls{tile::kPolls};
constexpr int kSms = 148;

struct PrefixLayout {
  bool tc;               // tensor-core kernel
  int rows;              // of a row tile's partials
  int tile_rows;
  int ctas;
  int R, spt, tps, tiles, nsplit;
  size_t parts;          // rows of partials
  bool whole;            // no list is long enough to be cut
  size_t off_ml, off_parts, total;
};

PrefixLayout prefix_layout(int dtype, int B, int T, int hq, int hkv, int D, int block_size, int groups,
                           int max_seq_len) {
  PrefixLayout L{};
  L.R = hq / hkv * T;
  auto tiles_of = [&](int rows, int64_t most) {
    L.rows = rows;
    L.spt = (int)std::max<int64_t>(1, std::min<int64_t>(rows / L.R, most));
    L.tps = L.R > rows ? (L.R + rows - 1) / rows : 1;
    // every group starts a tile of its own
    L.tile_rows = rows;
    const int64_t n = L.tps > 1 ? (int64_t)B * L.tps : std::min<int64_t>(B, (int64_t)B / L.spt + groups);
    L.tiles = (int)std::min<int64_t>(n, 0x7fffffff);
  };
  const int G = hq / hkv;
  if (dtype == SSD_DTYPE_BF16 && block_size % 16 == 0 && G <= tile::ROWS) {
    tiles_of(tile::ROWS / G * G, tile::ROWS);  // whole tokens
    L.tiles = (int)std::min<int64_t>((int64_t)B * L.tps, 0x7fffffff);  // (numbers of tiles, see the kernel)
    // (the units are counted in 32 bits)
    L.tc = L.tiles <= tile::kMaxTiles && groups <= tile::kMaxTiles &&
           (((int64_t)max_seq_len + 15) / 16 + tile::kStart) * (L.tiles + B) * hkv < (1 << 30);
  }
  const int64_t units = ((int64_t)max_seq_len + 15) / 16;  // of a sequence
  if (L.tc) {
    L.rows = tile::ROWS;
    // a list is longest where nothing is shared
    L.whole = units * std::min(L.spt, B) <= tile::kWhole;
    const int64_t most = L.whole ? (int64_t)L.tiles * hkv
                                 : (units * (L.tiles + B) * hkv + tile::kMinUnits - 1) / tile::kMinUnits;
    L.ctas = (int)std::min<int64_t>(kSms, most);
    L.nsplit = 0;
    L.parts = L.whole ? 0 : (size_t)2 * L.ctas * L.rows;
  } else {
    tiles_of(kRowsC, kMaxList / max_seq_len);
    const int64_t ctas = (int64_t)L.tiles * hkv;
    const int64_t chunks = ((int64_t)max_seq_len + kChunkC - 1) / kChunkC;
    L.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>({kMaxSplitC, chunks, 592 / ctas}));
    L.parts = L.nsplit == 1 ? 0 : (size_t)ctas * L.nsplit * L.rows;
  }
  L.off_ml = up256(sizeof(float) * L.parts * D);
  L.off_parts = L.off_ml + up256(sizeof(float2) * L.parts);
  L.total = L.off_parts + up256(sizeof(int4) * (size_t)(L.tps > 1 ? L.tiles : B) * hkv);
  return L;
}

template <int D>
int launch_tc(cudaStream_t st, const PrefixAttn& a, int ctas) {
  CUtensorMap map, vmap, qmap;
  if (!make_kv_row_map(&map, a.pages, (int64_t)2 * a.num_layers * a.num_blocks * a.block_size, a.hkv, D, 1, 16) ||
      !make_kv_unit_map(&vmap, a.pages, (int64_t)2 * a.num_layers * a.num_blocks * a.block_size, a.hkv, D) ||
      !make_kv_row_map(&qmap, a.q, (int64_t)a.B * a.T, a.hq, D, a.G, tile::ROWS / a.G))
    return SSD_ERR_LAUNCH;
  auto kern = tile::prefix_attention_tc_kernel<D>;
  constexpr size_t smem = tile::Cfg<D>::smem;
  static std::atomic<uint64_t> ready{0};
  if (!allow_smem(ready, kern, (int)smem)) return SSD_ERR_LAUNCH;
  SSD_PDL(kern, ctas, tile::THREADS, smem, st, map, vmap, qmap, a);
  const int64_t rows = (int64_t)a.B * a.T * a.hq;
  if (a.whole) return SSD_OK;
  if (rows > kJoinFew)
    SSD_PDL((prefix_join_kernel<bf16, D, tile::ROWS, true, 1>), (unsigned)((rows + 3) / 4), 128, 0, st, a);
  else
    SSD_PDL((prefix_join_kernel<bf16, D, tile::ROWS, true, 4>), (unsigned)rows, 128, 0, st, a);
  return SSD_OK;
}

template <typename T, int D>
int launch_cc(cudaStream_t st, const PrefixAttn& a) {
  SSD_PDL((prefix_attention_cc_kernel<T, D>), dim3(a.nsplit, a.hkv, a.tiles), kChunkC, 0, st, a);
  if (a.nsplit == 1) return SSD_OK;
  const int64_t rows = (int64_t)a.B * a.T * a.hq;
  SSD_PDL((prefix_join_kernel<T, D, kRowsC, false, 4>), (unsigned)rows, 128, 0, st, a);
  return SSD_OK;
}

template <typename T>
int launch_cc(cudaStream_t st, const PrefixAttn& a, int D) {
  return D == 256 ? launch_cc<T, 256>(st, a) : D == 128 ? launch_cc<T, 128>(st, a) : launch_cc<T, 64>(st, a);
}

bool sizes_ok(int B, int T, int hq, int hkv, int D, int groups, int max_seq_len) {
  return B > 0 && T > 0 && hq > 0 && hkv > 0 && hq % hkv == 0 && D > 0 && groups > 0 && max_seq_len > 0 &&
         max_seq_len <= kMaxPos && (int64_t)hq / hkv * T <= (1 << 20);
}

}  // namespace
}  // namespace ssd

using namespace ssd;

extern "C" size_t ssd_shared_prefix_attention_workspace_size(int dtype, int B, int T, int num_heads, int num_kv_heads,
                                                             int head_dim, int block_size, int num_groups,
                                                             int max_seq_len) {
  if (!sizes_ok(B, T, num_heads, num_kv_heads, head_dim, num_groups, max_seq_len) || block_size <= 0 ||
      (dtype != SSD_DTYPE_BF16 && dtype != SSD_DTYPE_F32))
    return 0;
  return prefix_layout(dtype, B, T, num_heads, num_kv_heads, head_dim, block_size, num_groups, max_seq_len).total;
}

extern "C" int ssd_shared_prefix_attention(ssd_stream_t stream, const void* q, const void* pages, int dtype,
                                           int num_layers, int num_blocks, int block_size, int num_kv_heads,
                                           int head_dim, int layer, const int32_t* block_tables, int max_blocks,
                                           const int32_t* seq_lens, const int32_t* q_lens,
                                           const int32_t* group_starts, const int32_t* prefix_lens, int num_groups,
                                           void* out, float scale, int B, int T, int num_heads, int max_seq_len,
                                           void* workspace, size_t workspace_bytes) {
  if (num_layers <= 0 || num_blocks <= 0 || block_size <= 0 || num_kv_heads <= 0 || layer < 0 || layer >= num_layers ||
      B < 0 || T < 0 || num_groups < 0 || num_heads <= 0 || num_heads % num_kv_heads || max_blocks <= 0 ||
      max_seq_len <= 0 || !pages || (dtype != SSD_DTYPE_BF16 && dtype != SSD_DTYPE_F32))
    return SSD_ERR_INVALID;
  if (B == 0 || T == 0) return SSD_OK;  // arrays of nothing may have no address
  if (num_groups == 0 || !q || !out || !block_tables || !seq_lens || !group_starts || !prefix_lens ||
      (int64_t)max_blocks * block_size < max_seq_len)
    return SSD_ERR_INVALID;
  if ((head_dim != 64 && head_dim != 128 && head_dim != 256) || B > kMaxRowsB || num_groups > kMaxRowsB ||
      !sizes_ok(B, T, num_heads, num_kv_heads, head_dim, num_groups, max_seq_len) || !kv8_aligned(q) ||
      !kv8_aligned(out) || !kv8_aligned(pages) || (int64_t)2 * num_layers * num_blocks * block_size > 0x7fffffff ||
      num_kv_heads > 65535)
    return SSD_ERR_UNSUPPORTED;
  const PrefixLayout L =
      prefix_layout(dtype, B, T, num_heads, num_kv_heads, head_dim, block_size, num_groups, max_seq_len);
  if (L.tiles > 65535) return SSD_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < L.total) return SSD_ERR_WORKSPACE;
  if (!kv8_aligned(workspace)) return SSD_ERR_UNSUPPORTED;
  if (out == q) return SSD_ERR_INVALID;
  char* w = reinterpret_cast<char*>(workspace);
  PrefixAttn a{};
  a.q = q;
  a.pages = pages;
  a.out = out;
  const int64_t per_layer = (int64_t)num_blocks * block_size * num_kv_heads * head_dim;
  a.plane = per_layer * num_layers;
  a.layer = per_layer * layer;
  a.tables = block_tables;
  a.seq_lens = seq_lens;
  a.q_lens = q_lens;
  a.starts = group_starts;
  a.prefixes = prefix_lens;
  a.scale = scale;
  a.B = B;
  a.T = T;
  a.hq = num_heads;
  a.hkv = num_kv_heads;
  a.G = num_heads / num_kv_heads;
  a.groups = num_groups;
  a.num_blocks = num_blocks;
  a.block_size = block_size;
  a.max_blocks = max_blocks;
  a.cap = max_seq_len;
  a.R = L.R;
  a.tile_rows = L.tile_rows;
  a.q_box = tile::ROWS / a.G * a.G;
  a.spt = L.spt;
  a.spt_inv = 65536 / L.spt + 1;
  a.tps = L.tps;
  a.tiles = L.tiles;
  a.nsplit = L.nsplit;
  a.num_layers = num_layers;
  a.layer_no = layer;
  a.polls = wait_polls.load(std::memory_order_relaxed);
  a.ws_o = reinterpret_cast<float*>(w);
  a.ws_ml = reinterpret_cast<float2*>(w + L.off_ml);
  a.parts = reinterpret_cast<int4*>(w + L.off_parts);
  a.whole = L.whole;
  cudaStream_t st = (cudaStream_t)stream;
  if (L.tc)
    return head_dim == 256   ? launch_tc<256>(st, a, L.ctas)
           : head_dim == 128 ? launch_tc<128>(st, a, L.ctas)
                             : launch_tc<64>(st, a, L.ctas);
  return dtype == SSD_DTYPE_BF16 ? launch_cc<bf16>(st, a, head_dim) : launch_cc<float>(st, a, head_dim);
}

extern "C" int ssd_shared_prefix_attention_status(ssd_stream_t stream) {
  cudaStream_t st = (cudaStream_t)stream;
  uint32_t gave_up = 0;
  bool ok = cudaMemcpyFromSymbolAsync(&gave_up, tile::gave_up, sizeof(gave_up), 0, cudaMemcpyDeviceToHost, st) ==
                cudaSuccess &&
            cudaStreamSynchronize(st) == cudaSuccess;
  if (ok && gave_up) {
    const uint32_t none = 0;
    ok = cudaMemcpyToSymbolAsync(tile::gave_up, &none, sizeof(none), 0, cudaMemcpyHostToDevice, st) == cudaSuccess &&
         cudaStreamSynchronize(st) == cudaSuccess;
  }
  if (!ok) {
    (void)cudaGetLastError();
    return SSD_ERR_LAUNCH;
  }
  return gave_up ? SSD_ERR_TIMEOUT : SSD_OK;
}

extern "C" int ssd_shared_prefix_attention_set_polls(int polls) {
  if (polls < -1) return SSD_ERR_INVALID;
  wait_polls.store(polls < 0 ? tile::kPolls : (uint32_t)polls, std::memory_order_relaxed);
  return SSD_OK;
}
