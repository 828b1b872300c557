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
  int spt, tps;          // sequences of a row tile (R <= its rows), else tiles of a sequence
  int tiles;             // bound on the row tiles of all groups
  int nsplit;            // parts of a tile's list (CUDA-core kernel)
  float* ws_o;           // [part][row][D] unnormalised sums
  float2* ws_ml;         // [part][row] what they are relative to, sum of weights
  int2* plan;            // [tile][head]: first part, parts (0: the tile sees nothing; 1: written by the kernel itself)
  int2* place;           // [sequence]: its (first) tile, its number in that tile
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

// Tile `tile` of the batch: groups in order, their tiles in order.  For whole warps.
__device__ __forceinline__ RowTile find_tile(const PrefixAttn& a, int tile) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int g0 = 0; g0 < a.groups; g0 += 32) {
    const int g = g0 + lane;
    int s = 0, e = 0;
    if (g < a.groups) {
      s = clamped(ld_act(a.starts + g), a.B);
      e = clamped(ld_act(a.starts + g + 1), a.B);
    }
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
__device__ __forceinline__ RowAt row_at(const PrefixAttn& a, const RowTile& tl, int head, int r, int rows) {
  RowAt w;
  const int gr = tl.part * rows + r;
  w.seq = a.tps > 1 ? 0 : gr / a.R;
  const int in = gr - w.seq * a.R;
  w.t = in / a.G;
  w.b = tl.seq0 + w.seq;
  w.pos = -1;
  w.at = -1;
  if (tl.group >= 0 && w.seq < tl.nseq && in < a.R) {
    w.at = (((int64_t)w.b * a.T + w.t) * a.hq + head * a.G + (in - w.t * a.G)) * D;
    const int ql = new_tokens(a, w.b);
    if (w.t < ql) w.pos = max(ld_act(a.seq_lens + w.b) - ql + w.t, -1);
  }
  return w;
}

// ------------------------------------------------------------------ CUDA-core kernel
// fp32 caches, and bf16 ones whose pages are no whole runs of 16 rows.  A CTA takes 8 query rows of one KV head and a
// part of their list, 256 positions at a time: a thread scores one position against all rows (q broadcast from shared
// memory), the rows' maxima and sums are taken over the CTA, and for P V a thread holds 4 dims of all rows over
// every PG-th position.
constexpr int kRowsC = 8, kChunkC = 256, kWarpsC = kChunkC / 32;
constexpr int kMaxSplitC = 32;

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
  if (tl.group < 0) return;
  const int P = prefix_of(a, tl.group);
  if (tid < kRowsC) {
    row_s[tid] = row_at<D>(a, tl, head, tid, kRowsC);
    run[tid] = -INFINITY;
    sum[tid] = 0.f;
  }
  if (warp == 0) {
    int tail = 0;
    if (lane < tl.nseq && new_tokens(a, tl.seq0 + lane) > 0)
      tail = max(min(ld_act(a.seq_lens + tl.seq0 + lane), a.cap) - P, 0);
    int incl = tail;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 0) cum[0] = P;
    if (lane < kRowsC) cum[1 + lane] = P + incl;
  }
  if (split == 0 && tid < tl.nseq && head == 0) a.place[tl.seq0 + tid] = make_int2(tile - tl.part, tid);
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
  if (a.plan && split == 0 && tid == 0) a.plan[tile * a.hkv + head] = make_int2(0, parts);
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
#pragma unroll 4
    for (int j = pg; j < n; j += PG) {
      const int64_t vo = v_s[j];
      if (vo < 0) continue;
      float v[4];
      load4(pages + vo + 4 * dg, v);
      const float4 pa = p_s[j][0], pb = p_s[j][1];
      const float pr[8] = {pa.x, pa.y, pa.z, pa.w, pb.x, pb.y, pb.z, pb.w};
      if (fabsf(v[0]) + fabsf(v[1]) + fabsf(v[2]) + fabsf(v[3]) <= FLT_MAX) {
#pragma unroll
        for (int r = 0; r < kRowsC; ++r)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[r][x] = fmaf(pr[r], v[x], o[r][x]);
      } else {  // an infinity or NaN (or a sum past fp32) reaches the rows that see the position, no others
        const uint32_t in = see_s[j];
#pragma unroll
        for (int r = 0; r < kRowsC; ++r)
          if (in >> r & 1) {
#pragma unroll
            for (int x = 0; x < 4; ++x) o[r][x] = fmaf(pr[r], v[x], o[r][x]);
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

// ------------------------------------------------------------------ join
// out = sum_i w_i o_i / sum_i w_i l_i over a row's parts, w_i = e^(m_i - M).  A warp a query row; bound by latency.
template <typename T, int D, int ROWS, bool TC>
__global__ void __launch_bounds__(128) prefix_join_kernel(const PrefixAttn a) {
  constexpr int PL = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= (int64_t)a.B * a.T * a.hq) return;
  const int h = (int)(row % a.hq), t = (int)(row / a.hq % a.T), b = (int)(row / a.hq / a.T);
  const int head = h / a.G;
  const int in = t * a.G + h % a.G;  // among the sequence's rows of this KV head
  pdl_wait();
  const int2 pl = __ldcg(a.place + b);
  const int tile = pl.x + (a.tps > 1 ? in / ROWS : 0);
  const int r = a.tps > 1 ? in % ROWS : pl.y * a.R + in;
  if ((unsigned)tile >= (unsigned)a.tiles || (unsigned)r >= (unsigned)ROWS) return;
  const int2 plan = __ldcg(a.plan + (int64_t)tile * a.hkv + head);
  if (plan.y == 1) return;
  auto part = [&](int i) -> int64_t {
    if constexpr (TC) return i == 0 ? plan.x : (plan.x & ~1) + 2 * i;
    else return (int64_t)(tile * a.hkv + head) * a.nsplit + i;
  };
  float M = -INFINITY, L = 0.f;
  for (int i = lane; i < plan.y; i += 32) M = fmaxf(M, __ldcg(a.ws_ml + part(i) * ROWS + r).x);
  M = warp_max(M);
  float o[PL];
#pragma unroll
  for (int x = 0; x < PL; ++x) o[x] = 0.f;
  for (int i0 = 0; i0 < plan.y; i0 += 32) {
    float w = 0.f;
    if (i0 + lane < plan.y) {
      const float2 ml = __ldcg(a.ws_ml + part(i0 + lane) * ROWS + r);
      // a part that the row sees nothing of has no weight and is passed over, whatever it left
      w = ml.y == 0.f ? -1.f : TC ? exp2f(ml.x - M) : expf(ml.x - M);
      if (ml.y != 0.f) L = fmaf(w, ml.y, L);
    }
    const int n = min(32, plan.y - i0);
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float wi = __shfl_sync(0xffffffffu, w, i);
      if (wi < 0.f) continue;
      const float* p = a.ws_o + (part(i0 + i) * ROWS + r) * D + lane * 2;
#pragma unroll
      for (int x = 0; x < PL; x += 2) {
        const float2 v = __ldcg(reinterpret_cast<const float2*>(p + x * 32));
        o[x] = fmaf(wi, v.x, o[x]);
        o[x + 1] = fmaf(wi, v.y, o[x + 1]);
      }
    }
  }
  L = warp_sum(L);
  const float k = L != 0.f ? 1.f / L : 0.f;
  T* out = reinterpret_cast<T*>(a.out) + row * D + lane * 2;
#pragma unroll
  for (int x = 0; x < PL; x += 2) {
    const float y0 = L != 0.f ? o[x] * k : 0.f, y1 = L != 0.f ? o[x + 1] * k : 0.f;
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<__nv_bfloat162*>(out + x * 32) = __floats2bfloat162_rn(y0, y1);
    else
      *reinterpret_cast<float2*>(out + x * 32) = make_float2(y0, y1);
  }
}

// ------------------------------------------------------------------ host
inline size_t up256(size_t x) { return (x + 255) & ~size_t(255); }

struct PrefixLayout {
  int rows;              // of a row tile
  int R, spt, tps, tiles, nsplit;
  size_t parts;          // rows of partials
  size_t off_ml, off_plan, off_place, total;
};

PrefixLayout prefix_layout(int B, int T, int hq, int hkv, int D, int groups, int max_seq_len) {
  PrefixLayout L{};
  L.rows = kRowsC;
  L.R = hq / hkv * T;
  L.spt = std::max(1, L.rows / L.R);
  L.tps = L.R > L.rows ? (L.R + L.rows - 1) / L.rows : 1;
  // every group starts a tile of its own
  L.tiles = L.tps > 1 ? B * L.tps : (int)std::min<int64_t>(B, (int64_t)B / L.spt + groups);
  const int64_t ctas = (int64_t)L.tiles * hkv;
  const int64_t chunks = ((int64_t)max_seq_len + kChunkC - 1) / kChunkC;
  L.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>({kMaxSplitC, chunks, 592 / ctas}));
  L.parts = L.nsplit == 1 ? 0 : (size_t)ctas * L.nsplit * L.rows;
  L.off_ml = up256(sizeof(float) * L.parts * D);
  L.off_plan = L.off_ml + up256(sizeof(float2) * L.parts);
  L.off_place = L.off_plan + up256(sizeof(int2) * (size_t)ctas);
  L.total = L.off_place + up256(sizeof(int2) * B);
  return L;
}

template <typename T, int D>
int launch_cc(cudaStream_t st, const PrefixAttn& a) {
  SSD_PDL((prefix_attention_cc_kernel<T, D>), dim3(a.nsplit, a.hkv, a.tiles), kChunkC, 0, st, a);
  if (a.nsplit == 1) return SSD_OK;
  const int64_t rows = (int64_t)a.B * a.T * a.hq;
  SSD_PDL((prefix_join_kernel<T, D, kRowsC, false>), (unsigned)((rows + 3) / 4), 128, 0, st, a);
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
  return prefix_layout(B, T, num_heads, num_kv_heads, head_dim, num_groups, max_seq_len).total;
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
      !kv8_aligned(out) || !kv8_aligned(pages) || (int64_t)num_blocks * block_size > 0x7fffffff ||
      num_kv_heads > 65535)
    return SSD_ERR_UNSUPPORTED;
  const PrefixLayout L = prefix_layout(B, T, num_heads, num_kv_heads, head_dim, num_groups, max_seq_len);
  if (L.tiles > 65535) return SSD_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < L.total) return SSD_ERR_WORKSPACE;
  if (!kv8_aligned(workspace)) return SSD_ERR_UNSUPPORTED;
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
  a.spt = L.spt;
  a.tps = L.tps;
  a.tiles = L.tiles;
  a.nsplit = L.nsplit;
  a.ws_o = reinterpret_cast<float*>(w);
  a.ws_ml = reinterpret_cast<float2*>(w + L.off_ml);
  a.plan = reinterpret_cast<int2*>(w + L.off_plan);
  a.place = reinterpret_cast<int2*>(w + L.off_place);
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == SSD_DTYPE_BF16 ? launch_cc<bf16>(st, a, head_dim) : launch_cc<float>(st, a, head_dim);
}
