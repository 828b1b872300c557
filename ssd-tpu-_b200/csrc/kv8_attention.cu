// Attention over the 8-bit paged KV cache.
//
// For query row r at position P_r (token t of sequence b sits at seq_lens[b] - q_lens[b] + t) and the
// positions j <= P_r of its sequence, with K_j = k_j 2^a(j), V_j = v_j 2^c(j) (a, c: scale exponents of j's
// page and head):
//   s_j = scale * 2^a(j) * (q_r . k_j),   out_r = sum_j e^(s_j - M) 2^c(j) v_j / sum_j e^(s_j - M).
// Rows past q_lens[b] and rows that see no position are zeros.
//
// A CTA owns one KV head of one sequence, a slice of its positions (a split) and a group of query rows (G query heads
// times the new tokens).  Up to kFewTokens new tokens the slices are fixed, so a query's result does not depend on how
// many tokens stand beside it.
// Splits leave unnormalised partials, which a second kernel joins in split order.  It needs no counters, so a
// workspace holds nothing between calls and may come uninitialised from any allocator.  Times below are of both
// kernels, from replayed graphs, on a GPU that copies 6.5 TB/s.
#include <float.h>

#include <algorithm>

#include "kv8.cuh"
#include "tcgen05.cuh"

namespace ssd {
namespace {

struct Kv8Attn {
  Kv8Cache c;
  const void* q;        // [B, T, hq, D]
  void* out;            // [B, T, hq, D]
  const int32_t* tables;
  int max_blocks;
  const int32_t* seq_lens;
  const int32_t* q_lens;
  float scale;
  int B, T, hq, G, row_groups, nsplit, split;  // split: positions of one
  float* ws_o;          // [group][split][rows][D]
  float4* ws_ml;        // [group][split][rows]: maximum that o is relative to, that l is relative to, l
  // With a plan (many rows), the splits go by the sequences' own lengths: nsplit of them for all sequences together,
  // partials [head][row group][split][rows], and plan[b] says which are sequence b's: the first, and how many.
  int2* plan;
  uint32_t polls;       // of a device-side wait before the CTA gives up
};

constexpr int kMaxSeqLen = 1 << 30;  // so that a position behind the last split's end is still an int

// Splits of a sequence that hold positions (at least one, which writes its zero rows).
__device__ __forceinline__ int splits_of(int seq, int split) { return max(1, (seq + split - 1) / split); }

// A row group's partials: how many, and the index of the first.
__device__ __forceinline__ int partials_of(const Kv8Attn& a, int b, int head, int rg, int64_t grp, int64_t& first) {
  if (a.plan) {
    const int2 p = __ldcg(a.plan + b);
    first = (int64_t)(head * a.row_groups + rg) * a.nsplit + p.x;
    return p.y;
  }
  first = grp * a.nsplit;
  return splits_of(min(min(ld_act(a.seq_lens + b), a.max_blocks * a.c.block_size), a.nsplit * a.split), a.split);
}

// out = sum_s e^(m_s - M) o_s / sum_s e^(n_s - N) l_s * e^(M - N), M and N the largest m_s and n_s.  The last factor is
// applied as its square root, twice: M - N, about V's exponent less 7 to 15, may lie below fp32's.  One CTA per
// query row: its threads hold 4 dims of every SG-th split each and add the groups up in order, so that the
// loads of many splits are in flight at once.  LOG2: the maxima are in powers of two.  Bound by latency: two dependent
// reads, 2 to 3 us of a call.
// The weight of a split in the join; -1 where the row saw none of it, so that what it left (zeros, or NaN of other
// rows' positions) is passed over.  A seen split counts however small its weight: its NaN has to come through.
template <bool LOG2>
__device__ __forceinline__ float split_weight(float m, float M) {
  if (m <= (LOG2 ? -1e38f : -INFINITY)) return -1.f;
  return LOG2 ? exp2f(m - M) : expf(m - M);
}

constexpr int kJoinThreads = 256;
constexpr int kJoinChunk = 256;  // splits whose weights are held at a time

template <typename T, int D, int R, bool LOG2>
__global__ void __launch_bounds__(kJoinThreads) kv8_join_kernel(const Kv8Attn a) {
  constexpr int DQ = D / 4, SG = kJoinThreads / DQ;
  __shared__ float w_s[kJoinChunk];
  __shared__ float red[32];
  __shared__ float4 part[SG][DQ];
  const int tid = threadIdx.x;
  const int r = blockIdx.x % R;
  const int64_t grp = blockIdx.x / R;
  const int rg = (int)(grp % a.row_groups), head = (int)(grp / a.row_groups % a.c.hkv);
  const int b = (int)(grp / a.row_groups / a.c.hkv);
  const int gr = rg * R + r, t = gr / a.G, g = gr % a.G;
  pdl_wait();
  pdl_trigger();
  if (t >= a.T) return;
  const int ql = a.q_lens ? min(max(ld_act(a.q_lens + b), 0), a.T) : a.T;
  int64_t s0;
  const int ns = partials_of(a, b, head, rg, grp, s0);
  auto ex = [](float v) { return LOG2 ? exp2f(v) : expf(v); };
  const float4* ml = a.ws_ml + s0 * R + r;
  float M = -INFINITY, N = -INFINITY;
  for (int s = tid; s < ns; s += kJoinThreads) {
    const float4 v = __ldcg(ml + (int64_t)s * R);
    M = fmaxf(M, v.x);
    N = fmaxf(N, v.y);
  }
  M = block_reduce(M, red, OpMax());
  N = block_reduce(N, red, OpMax());
  const int d4 = tid % DQ, sg = tid / DQ;
  const float* po = a.ws_o + (s0 * R + r) * D + d4 * 4;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float L = 0.f;
  for (int c0 = 0; c0 < ns; c0 += kJoinChunk) {
    const int n = min(kJoinChunk, ns - c0);
    if (tid < n) {
      const float4 v = __ldcg(ml + (int64_t)(c0 + tid) * R);
      if (v.y != -INFINITY) L += v.z * ex(v.y - N);
      w_s[tid] = split_weight<LOG2>(v.x, M);
    }
    __syncthreads();
#pragma unroll 4
    for (int s = sg; s < n; s += SG) {
      const float f = w_s[s];
      const float4 x = __ldcg(reinterpret_cast<const float4*>(po + (int64_t)(c0 + s) * R * D));
      if (f >= 0.f) {
        o.x = fmaf(f, x.x, o.x);
        o.y = fmaf(f, x.y, o.y);
        o.z = fmaf(f, x.z, o.z);
        o.w = fmaf(f, x.w, o.w);
      }
    }
    __syncthreads();
  }
  part[sg][d4] = o;
  L = block_reduce(L, red, OpSum());
  const bool real = t < ql && L != 0.f;  // L is NaN, not 0, where a seen score is
  if (tid < DQ) {
    o = part[0][tid];
#pragma unroll
    for (int x = 1; x < SG; ++x) {
      const float4 p = part[x][tid];
      o.x += p.x; o.y += p.y; o.z += p.z; o.w += p.w;
    }
    const float f = ex(0.5f * (M - N));
    T* out = reinterpret_cast<T*>(a.out) + (((int64_t)b * a.T + t) * a.hq + head * a.G + g) * D + tid * 4;
    out[0] = from_f<T>(real ? o.x / L * f * f : 0.f);
    out[1] = from_f<T>(real ? o.y / L * f * f : 0.f);
    out[2] = from_f<T>(real ? o.z / L * f * f : 0.f);
    out[3] = from_f<T>(real ? o.w / L * f * f : 0.f);
  }
}

// The same for few splits (up to 16 a sequence): one warp a row, 4 dims of a lane at a time, the weights of 32 splits
// in its lanes; no barrier, and four rows a CTA where the kernel above takes one (2048 rows of 9 splits: 34.4 against
// 41.6 us for the whole call).
template <typename T, int D, int R, bool LOG2>
__global__ void __launch_bounds__(128) kv8_join_few_kernel(const Kv8Attn a, int64_t rows) {
  constexpr int DQ = D / 4, PL = DQ < 32 ? 1 : DQ / 32;  // float4 of a row, of a lane
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int r = (int)(row % R);
  const int64_t grp = row / R;
  const int rg = (int)(grp % a.row_groups), head = (int)(grp / a.row_groups % a.c.hkv);
  const int b = (int)(grp / a.row_groups / a.c.hkv);
  const int gr = rg * R + r, t = gr / a.G, g = gr % a.G;
  pdl_wait();
  pdl_trigger();
  if (row >= rows || t >= a.T) return;
  const int ql = a.q_lens ? min(max(ld_act(a.q_lens + b), 0), a.T) : a.T;
  int64_t s0;
  const int ns = partials_of(a, b, head, rg, grp, s0);
  auto ex = [](float v) { return LOG2 ? exp2f(v) : expf(v); };
  const float4* ml = a.ws_ml + s0 * R + r;
  float M = -INFINITY, N = -INFINITY;
  float4 v;
  for (int c0 = 0; c0 < ns; c0 += 32) {
    v = make_float4(-INFINITY, -INFINITY, 0.f, 0.f);
    if (c0 + lane < ns) v = __ldcg(ml + (int64_t)(c0 + lane) * R);
    M = fmaxf(M, v.x);
    N = fmaxf(N, v.y);
  }
  M = warp_max(M);
  N = warp_max(N);
  float L = 0.f;
  const float4* po = reinterpret_cast<const float4*>(a.ws_o) + (s0 * R + r) * DQ;
  float4 o[PL];
#pragma unroll
  for (int i = 0; i < PL; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int c0 = 0; c0 < ns; c0 += 32) {
    if (ns > 32) {  // else they are still there
      v = make_float4(-INFINITY, -INFINITY, 0.f, 0.f);
      if (c0 + lane < ns) v = __ldcg(ml + (int64_t)(c0 + lane) * R);
    }
    L += v.y == -INFINITY ? 0.f : v.z * ex(v.y - N);
    const float w = split_weight<LOG2>(v.x, M);
    const int n = min(32, ns - c0);
#pragma unroll 4
    for (int s = 0; s < n; ++s) {
      const float f = __shfl_sync(0xffffffffu, w, s);
#pragma unroll
      for (int i = 0; i < PL; ++i) {
        if (DQ < 32 && lane >= DQ) continue;
        const float4 x = __ldcg(po + (int64_t)(c0 + s) * R * DQ + i * 32 + lane);
        if (f >= 0.f) {
          o[i].x = fmaf(f, x.x, o[i].x);
          o[i].y = fmaf(f, x.y, o[i].y);
          o[i].z = fmaf(f, x.z, o[i].z);
          o[i].w = fmaf(f, x.w, o[i].w);
        }
      }
    }
  }
  L = warp_sum(L);
  const bool real = t < ql && L != 0.f;
  const float k = ex(0.5f * (M - N));
  T* out = reinterpret_cast<T*>(a.out) + (((int64_t)b * a.T + t) * a.hq + head * a.G + g) * D;
#pragma unroll
  for (int i = 0; i < PL; ++i) {
    if (DQ < 32 && lane >= DQ) continue;
    T y[4] = {from_f<T>(real ? o[i].x / L * k * k : 0.f), from_f<T>(real ? o[i].y / L * k * k : 0.f),
              from_f<T>(real ? o[i].z / L * k * k : 0.f), from_f<T>(real ? o[i].w / L * k * k : 0.f)};
    T* to = out + (i * 32 + lane) * 4;
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<uint2*>(to) = *reinterpret_cast<uint2*>(y);
    else
      *reinterpret_cast<uint4*>(to) = *reinterpret_cast<uint4*>(y);
  }
}

template <typename T, int D, int R, bool LOG2>
int launch_join(cudaStream_t st, const Kv8Attn& a, int B) {
  const int64_t rows = (int64_t)B * a.c.hkv * a.row_groups * R;
  if (rows > 0x7fffffff) return SSD_ERR_UNSUPPORTED;
  if ((a.plan ? a.nsplit / B : a.nsplit) <= 16)
    SSD_PDL((kv8_join_few_kernel<T, D, R, LOG2>), (unsigned)((rows + 3) / 4), 128, 0, st, a, rows);
  else
    SSD_PDL((kv8_join_kernel<T, D, R, LOG2>), (unsigned)rows, kJoinThreads, 0, st, a);
  return SSD_OK;
}

// ------------------------------------------------------------------ CUDA-core kernel (fp32 models)
// fp32 queries keep fp32 products.  A CTA takes 8 query rows and 256 positions: a thread scores one position
// against all rows (Q broadcast from shared memory, no reduction across lanes), the rows' maxima and sums are
// taken over the CTA, and for P V a thread holds 4 dims of all rows over every PG-th position.  Used by the fp32
// (toy) models, whose forward takes at most 16 rows: bound by latency, not by bytes (two sequences of 77 and 200
// positions, 20 rows of 64 dims: 10.3 us; with 128 positions a CTA, hence a join, 13.9).
constexpr int kCcRows = 8;
constexpr int kCcSplit = 256;
constexpr int kCcWarps = kCcSplit / 32;

template <int D>
__global__ void __launch_bounds__(kCcSplit) kv8_attention_cc_kernel(const Kv8Attn a) {
  constexpr int DG = D / 4, PG = kCcSplit / DG;
  __shared__ float4 p_s[kCcSplit][2];          // weights of position j
  __shared__ __align__(16) float o_s[PG][kCcRows][D];
  __shared__ float red[2][kCcWarps][kCcRows];
  static_assert(sizeof(o_s) >= sizeof(float4) * 2 * D);
  float4(*q_s)[2] = reinterpret_cast<float4(*)[2]>(o_s);  // dim d of rows 0-3 and 4-7, until the scores are done
  __shared__ int pos_s[kCcRows];
  __shared__ int64_t v_s[kCcSplit];            // byte offset of a position's V row (-1: none)
  __shared__ float vs_s[kCcSplit];
  const int split = blockIdx.x, b = blockIdx.z;
  const int head = blockIdx.y / a.row_groups, rg = blockIdx.y % a.row_groups;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_trigger();
  const int j = split * kCcSplit + tid;        // this thread's position
  const int page = j / a.c.block_size;
  int blk = -1;                                // read whatever the length says, so as not to wait for it
  if (page < a.max_blocks) blk = ld_act(a.tables + (int64_t)b * a.max_blocks + page);
  const int seq_full = ld_act(a.seq_lens + b);
  const int ql = a.q_lens ? min(max(ld_act(a.q_lens + b), 0), a.T) : a.T;
  // positions beyond the table or the split count are never read (a seq_len larger than the caller's bound)
  const int seq = min(min(seq_full, a.max_blocks * a.c.block_size), a.nsplit * kCcSplit);
  const int row0 = rg * kCcRows;
  const int nrows = min(kCcRows, a.G * a.T - row0);
  if (split >= splits_of(seq, kCcSplit)) return;
  for (int i = tid; i < kCcRows * D; i += kCcSplit) {
    const int r = i / D, d = i % D;
    const int gr = row0 + r, t = gr / a.G, g = gr % a.G;
    float x = 0.f;
    if (r < nrows) x = ld_act(reinterpret_cast<const float*>(a.q) + (((int64_t)b * a.T + t) * a.hq + head * a.G + g) * D + d);
    if (fabsf(x) == INFINITY) x = __int_as_float(0x7fc00000);  // the row's scores hold NaN or an infinity less itself
    reinterpret_cast<float*>(q_s[d])[r] = x;
  }
  if (tid < kCcRows) {
    const int t = (row0 + tid) / a.G;
    pos_s[tid] = (tid < nrows && t < ql) ? seq_full - ql + t : -1;
  }
  const bool there = j < seq && (unsigned)blk < (unsigned)a.c.num_blocks;
  float s[kCcRows];
#pragma unroll
  for (int r = 0; r < kCcRows; ++r) s[r] = 0.f;
  uint4 w[D / 16];
  float ks = 0.f, vs = 0.f;
  int64_t off = -1;
  if (there) {
    off = a.c.layer + (((int64_t)blk * a.c.block_size + j % a.c.block_size) * a.c.hkv + head) * D;
    const float* sc = a.c.scales + a.c.scale_layer + (int64_t)blk * a.c.hkv + head;
    ks = stored_scale(ld_act(sc));
    vs = stored_scale(ld_act(sc + a.c.scale_plane));
#pragma unroll
    for (int i = 0; i < D / 16; ++i) w[i] = ld_act_v4(a.c.pages + off + 16 * i);
  }
  v_s[tid] = there ? off + a.c.plane : -1;
  vs_s[tid] = vs;
  __syncthreads();
  if (there) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const uint32_t in[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const float2 k = e4m3_pair(in[x >> 1] >> (x & 1 ? 16 : 0));
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float kd = y ? k.y : k.x;
          const float4 qa = q_s[16 * i + 2 * x + y][0], qb = q_s[16 * i + 2 * x + y][1];
          s[0] = fmaf(qa.x, kd, s[0]); s[1] = fmaf(qa.y, kd, s[1]); s[2] = fmaf(qa.z, kd, s[2]); s[3] = fmaf(qa.w, kd, s[3]);
          s[4] = fmaf(qb.x, kd, s[4]); s[5] = fmaf(qb.y, kd, s[5]); s[6] = fmaf(qb.z, kd, s[6]); s[7] = fmaf(qb.w, kd, s[7]);
        }
      }
    }
  }
  float m[kCcRows];
#pragma unroll
  for (int r = 0; r < kCcRows; ++r) {
    s[r] = there && j <= pos_s[r] ? s[r] * ks * a.scale : -INFINITY;
    // finite once a position is seen, a NaN score included: it spoils the sums below
    const float x = warp_max(there && j <= pos_s[r] ? fmaxf(s[r], -FLT_MAX) : -INFINITY);
    if (lane == 0) red[0][warp][r] = x;
  }
  __syncthreads();
  float p[kCcRows];
#pragma unroll
  for (int r = 0; r < kCcRows; ++r) {
    m[r] = red[0][0][r];
#pragma unroll
    for (int w = 1; w < kCcWarps; ++w) m[r] = fmaxf(m[r], red[0][w][r]);
    p[r] = there && j <= pos_s[r] ? expf(s[r] - m[r]) : 0.f;
    const float x = warp_sum(p[r]);
    if (lane == 0) red[1][warp][r] = x;
  }
  p_s[tid][0] = make_float4(p[0], p[1], p[2], p[3]);
  p_s[tid][1] = make_float4(p[4], p[5], p[6], p[7]);
  __syncthreads();
  {
    const int dg = tid % DG, pg = tid / DG;
    float o[kCcRows][4];
#pragma unroll
    for (int r = 0; r < kCcRows; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[r][i] = 0.f;
    const int n = min(kCcSplit, seq - split * kCcSplit);
#pragma unroll 8
    for (int i = pg; i < n; i += PG) {
      const int64_t vo = v_s[i];
      if (vo < 0) continue;
      uint32_t v4 = __ldcg(reinterpret_cast<const uint32_t*>(a.c.pages + vo + 4 * dg));
      if (nan_marks(v4)) {  // rare: NaN reaches the rows that see the position, no others
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if ((v4 >> (8 * x) & 0x7fu) == 0x7fu)
#pragma unroll
            for (int r = 0; r < kCcRows; ++r)
              if (split * kCcSplit + i <= pos_s[r]) o[r][x] = __int_as_float(0x7fc00000);
        v4 = clear_nan(v4);
      }
      const float2 lo = e4m3_pair(v4), hi = e4m3_pair(v4 >> 16);
      const float f = vs_s[i];
      const float v[4] = {lo.x * f, lo.y * f, hi.x * f, hi.y * f};
      const float4 pa = p_s[i][0], pb = p_s[i][1];
      const float pr[8] = {pa.x, pa.y, pa.z, pa.w, pb.x, pb.y, pb.z, pb.w};
#pragma unroll
      for (int r = 0; r < kCcRows; ++r)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[r][x] = fmaf(pr[r], v[x], o[r][x]);
    }
#pragma unroll
    for (int r = 0; r < kCcRows; ++r)
      *reinterpret_cast<float4*>(&o_s[pg][r][4 * dg]) = make_float4(o[r][0], o[r][1], o[r][2], o[r][3]);
  }
  __syncthreads();
  const int64_t grp = ((int64_t)b * a.c.hkv + head) * a.row_groups + rg;
  for (int i = tid; i < nrows * D; i += kCcSplit) {
    const int r = i / D, d = i % D;
    float O = 0.f;
#pragma unroll
    for (int x = 0; x < PG; ++x) O += o_s[x][r][d];
    float L = 0.f, M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kCcWarps; ++w) {
      L += red[1][w][r];
      M = fmaxf(M, red[0][w][r]);
    }
    const int64_t at = (grp * a.nsplit + split) * kCcRows + r;
    if (a.nsplit == 1) {
      const int gr = row0 + r, t = gr / a.G, g = gr % a.G;
      reinterpret_cast<float*>(a.out)[(((int64_t)b * a.T + t) * a.hq + head * a.G + g) * D + d] =
          pos_s[r] >= 0 && L != 0.f ? O / L : 0.f;
    } else {
      a.ws_o[at * D + d] = O;
      if (d == 0) a.ws_ml[at] = make_float4(M, M, L, 0.f);
    }
  }
}

// ------------------------------------------------------------------ few query rows (bf16): decode and verify
// Bound by HBM: every K and V byte of the context is read once for up to 8 NT rows (32 sequences of 2000 to 8192
// positions, 16 heads of 256, 5 or 7 new tokens: 1.34 GB in 222 us, 6.0 TB/s; 8 sequences of 512 to 4096, 4 or 5:
// 152 MB in 34.7 us, 4.4 TB/s, where the CTAs of the longest sequences end last).  The transposed products
//   S^T = K Q^T   and   O^T = V^T P^T   (m16n8k16, f16 operands, fp32 sums)
// put the 16 positions of a tile and 16 head dims on the instruction's long side and the query rows on its
// short one, so few rows waste little.  Each warp owns every fourth tile of 16 positions and a ring of tiles
// in shared memory that only it fills (cp.async, zeros for rows that are not there) and reads, so the loop has
// no barrier.  The order of the summed-over index is free, so a lane's operands are whole 16-byte pieces:
//   K: lane (g, t) = (lane / 4, lane % 4) takes positions g and g + 8, dims 64 c + 16 t .. + 15; word j of a
//      piece is the A operand of step 4 c + j.  Q's registers follow the same order.
//   V: positions 2t, 2t+1, 2t+8, 2t+9, dims 128 h + 16 g .. + 15 (D = 64: 8 g .. + 7); byte pairs of two
//      positions become the A operand, m-tile i carrying dims 2i and 2i + 1 of each lane.
//   P: the S^T accumulators, rounded to f16 pairs and transposed by movmatrix, are the B operand.
// e4m3 converts to f16 exactly.  q is scaled per row by a power of two, its largest into [2^14, 2^15), which keeps
// bf16's eight bits (elements below 2^-28 of the row's largest lose the last ones).  V's page scales join the
// weights' exponents: the reference M is put kBelow = 7 (log2) below the largest s_j + c_j seen, and moves when one
// passes it by kSpan = 15, so a weight 2^(s_j + c_j - M) is at most 2^15 (f16 holds nearly 2^16) and the largest is at
// least 2^7: weights keep f16's 11 bits down to 2^-21 of the largest and are off by 2^-32 of it below, whatever the
// pages' scales.
constexpr int kFewWarps = 4;
constexpr float kBelow = 7.f, kSpan = 15.f;

__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {  // 2^x to 2^-22, zero below 2^-126
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds128(uint32_t p) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(p));
  return r;
}

template <int D, int NT, bool UNI>
struct FewSmem {
  static constexpr int STAGES = D == 256 ? 2 : 4;
  static constexpr int TILE = 16 * D;          // bytes of a tile's K (or V) rows
  static constexpr int PITCH = D + D / 8 + 4;  // floats of a row of the join: 16 dims then 2 of padding
  static constexpr size_t ring = (size_t)kFewWarps * STAGES * 2 * TILE;
  static_assert(sizeof(float) * kFewWarps * 8 * PITCH <= ring, "the join reuses the rings");
  static constexpr size_t qs = sizeof(uint2) * NT * (D / 16) * 32;  // Q operands, in lane order
  static size_t total(int split) { return ring + qs + (UNI ? 0 : (size_t)split * 12); }
};

// UNI: block_size is a multiple of 16, so a tile lies in one page and has one pair of scales.
template <int D, int NT, bool UNI>
__global__ void __launch_bounds__(kFewWarps * 32, NT == 1 ? 3 : 2) kv8_attention_few_kernel(const Kv8Attn a) {
  constexpr int CK = D / 64;
  constexpr int HV = D >= 128 ? D / 128 : 1;
  constexpr int VW = D >= 128 ? 4 : 2;  // 32-bit words of V a lane takes per position
  constexpr int MT = 2 * VW;            // m-tiles of one V half
  constexpr int R = 8 * NT;
  constexpr int PCS = D / 16;           // 16-byte pieces of a row
  using S = FewSmem<D, NT, UNI>;
  extern __shared__ __align__(128) unsigned char smem[];
  float* os = reinterpret_cast<float*>(smem);
  uint2* qsm = reinterpret_cast<uint2*>(smem + S::ring);
  // !UNI, per position: row number in the layer (-1: none), K scale, exponent of V's scale
  int* row_s = reinterpret_cast<int*>(smem + S::ring + S::qs);
  float* ks_s = reinterpret_cast<float*>(row_s + a.split);
  float* ve_s = ks_s + a.split;
  __shared__ float4 ml_s[kFewWarps][R], fin_s[R];
  __shared__ float qscale_s[R];
  __shared__ int nan_seen;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  const int split = blockIdx.x, b = blockIdx.z;
  const int head = blockIdx.y / a.row_groups, rg = blockIdx.y % a.row_groups;
  const int row0 = rg * R;
  pdl_wait();
  // Block ids do not wait for the lengths: entries of this split that the table has.  UNI: lane k of a warp keeps
  // row number (-1: none) and scales of the warp's k-th tile; otherwise shared memory holds them per position.
  const int base = split * a.split;
  const int32_t* table = a.tables + (int64_t)b * a.max_blocks;
  const float* sc = a.c.scales + a.c.scale_layer + head;
  int row_l = -1;
  float ks_l = 1.f, ve_l = 0.f;
  if constexpr (UNI) {
    const int j = base + (warp + lane * kFewWarps) * 16, page = j / a.c.block_size;
    if (lane * kFewWarps * 16 < a.split && page < a.max_blocks) {
      const int blk = ld_act(table + page);
      if ((unsigned)blk < (unsigned)a.c.num_blocks) {
        row_l = blk * a.c.block_size + (j - page * a.c.block_size);
        ks_l = ld_act(sc + (int64_t)blk * a.c.hkv);
        ve_l = ld_act(sc + a.c.scale_plane + (int64_t)blk * a.c.hkv);
      }
    }
  }
  const int seq_full = ld_act(a.seq_lens + b);
  const int ql = a.q_lens ? min(max(ld_act(a.q_lens + b), 0), a.T) : a.T;
  const int seq = min(min(seq_full, a.max_blocks * a.c.block_size), a.nsplit * a.split);
  if (split > 0 && base >= seq) return;
  const int kn = min(max(seq - base, 0), a.split);  // positions of this split that exist
  const int total_rows = a.G * a.T;
  if constexpr (!UNI) {
    for (int i = tid; i < ((kn + 15) & ~15); i += kFewWarps * 32) {
      int row = -1;
      float ks = 1.f, ve = 0.f;
      if (i < kn) {
        const int j = base + i, page = j / a.c.block_size;
        const int blk = ld_act(table + page);
        if ((unsigned)blk < (unsigned)a.c.num_blocks) {
          row = blk * a.c.block_size + (j - page * a.c.block_size);
          ks = stored_scale(ld_act(sc + (int64_t)blk * a.c.hkv));
          ve = (float)scale_exponent(ld_act(sc + a.c.scale_plane + (int64_t)blk * a.c.hkv));
        }
      }
      row_s[i] = row;
      ks_s[i] = ks;
      ve_s[i] = ve;
    }
    __syncthreads();
  }
  if (tid == 0) nan_seen = 0;

  const int64_t rs = (int64_t)a.c.hkv * D;
  // the ring: piece p of row r lies at p ^ 4 (r & 1) of K's rows and p ^ (r & 6) of V's, so that a quarter warp's
  // 16-byte reads meet no bank twice (D = 64: a line holds two rows, V's 8-byte reads meet each bank twice)
  auto k_piece = [](int r, int p) { return r * PCS + (D >= 128 ? p ^ ((r & 1) << 2) : p); };
  auto v_piece = [](int r, int p) { return r * PCS + (D >= 128 ? p ^ (r & 6) : p ^ (r >> 1 & 3)); };
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * (S::STAGES * 2 * S::TILE);
  const uint8_t* kp = a.c.pages + a.c.layer + (int64_t)head * D + (lane % PCS) * 16;
  const int tiles = (kn + 15) / 16;
  const int mine = warp < tiles ? (tiles - warp + kFewWarps - 1) / kFewWarps : 0;
  auto issue = [&](int k) {  // this warp's k-th tile, into stage k % STAGES
    const int first_l = UNI ? __shfl_sync(0xffffffffu, row_l, k & 31) : 0;
    if (k < mine) {
      const int i0 = (warp + k * kFewWarps) * 16;
      const uint32_t st = ring + (k % S::STAGES) * (2 * S::TILE);
      constexpr int RPI = 32 / PCS;  // rows an instruction covers
      if constexpr (UNI) {
        // one product a tile: its rows lie rs apart, and past the sequence's end they are in the page all the same
        const uint8_t* src = kp + (int64_t)(max(first_l, 0) + lane / PCS) * rs;
        const int left = first_l < 0 ? 0 : kn - i0 - lane / PCS;  // row x RPI of the lane is there where it is below
#pragma unroll
        for (int x = 0; x < 16 / RPI; ++x) {
          const int r = x * RPI + lane / PCS;
          cp_async16(st + k_piece(r, lane % PCS) * 16, src, x * RPI < left);
          cp_async16(st + S::TILE + v_piece(r, lane % PCS) * 16, src + a.c.plane, x * RPI < left);
          src += RPI * rs;
        }
      } else {
#pragma unroll
        for (int x = 0; x < 16 / RPI; ++x) {
          const int r = x * RPI + lane / PCS;
          const int first = row_s[i0 + r];
          const uint8_t* src = kp + max(first, 0) * rs;
          cp_async16(st + k_piece(r, lane % PCS) * 16, src, first >= 0);
          cp_async16(st + S::TILE + v_piece(r, lane % PCS) * 16, src + a.c.plane, first >= 0);
        }
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int k = 0; k < S::STAGES - 1; ++k) issue(k);
  // ---- Q, scaled into f16, in the order of the lanes' operands: a warp takes two rows of 8 (16 lanes a row)
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = 2 * warp + (lane >> 4), gr = row0 + 8 * nt + r, t = gr / a.G;
    const bool real = gr < total_rows && t < ql;
    const bf16* src = reinterpret_cast<const bf16*>(a.q) +
                      (((int64_t)b * a.T + t) * a.hq + head * a.G + (gr - t * a.G)) * D + (lane & 15) * (D / 16);
    float f[D / 16], amax = 0.f;
#pragma unroll
    for (int k = 0; k < D / 16; k += 4) {
      uint2 w = make_uint2(0, 0);
      if (real) w = __ldcg(reinterpret_cast<const uint2*>(src + k));
      const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w.x));
      const float2 y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w.y));
      f[k] = x.x; f[k + 1] = x.y; f[k + 2] = y.x; f[k + 3] = y.y;
#pragma unroll
      for (int j = 0; j < 4; ++j) amax = fmaxf(amax, fabsf(f[k + j]));  // NaN reaches the scores by itself
    }
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, x));
    const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127 - 14, -118), 120);
    const float inv = exp2i(-e);
    // an infinity in q leaves no finite score, or one less itself: NaN
    if ((lane & 15) == 0)
      qscale_s[8 * nt + r] = amax == INFINITY ? __int_as_float(0x7fc00000) : exp2i(e) * a.scale * 1.4426950408889634f;
#pragma unroll
    for (int k = 0; k < D / 16; k += 4) {
      const int d = (lane & 15) * (D / 16) + k, c = d >> 6, tt = (d >> 4) & 3, j = (d >> 2) & 3;
      qsm[(nt * CK * 4 + 4 * c + j) * 32 + r * 4 + tt] =
          make_uint2(pack_f16(f[k] * inv, f[k + 1] * inv), pack_f16(f[k + 2] * inv, f[k + 3] * inv));
    }
  }
  __syncthreads();
  // this lane's columns: rows 8 nt + 2 t4 + {0, 1}
  float qs[NT][2];
  int pos[NT][2];
  int kmin = 0x7fffffff;  // the last position that every real row of the group sees
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      qs[nt][e] = qscale_s[8 * nt + 2 * t4 + e];
      const int gr = row0 + 8 * nt + 2 * t4 + e, t = gr / a.G;
      pos[nt][e] = (gr < total_rows && t < ql) ? seq_full - ql + t : -1;
      if (pos[nt][e] >= 0) kmin = min(kmin, pos[nt][e]);
    }
  kmin = min(kmin, __shfl_xor_sync(0xffffffffu, kmin, 1));
  kmin = min(kmin, __shfl_xor_sync(0xffffffffu, kmin, 2));
  uint2 qf[NT == 1 ? CK * 4 : 1];
  if constexpr (NT == 1) {
#pragma unroll
    for (int i = 0; i < CK * 4; ++i) qf[i] = qsm[i * 32 + lane];
  }

  float M[NT][2], N[NT][2], l[NT][2], o[NT][HV * MT][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      M[nt][e] = N[nt][e] = -INFINITY;
      l[nt][e] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < HV * MT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.f;
  }
  if constexpr (UNI) {
    ks_l = stored_scale(ks_l);
    ve_l = (float)scale_exponent(ve_l);
  }
  for (int k = 0; k < mine; ++k) {
    cp_async_wait<S::STAGES - 2>();
    __syncwarp();  // every lane's copies of tile k are there, and every lane is done with tile k - 1
    issue(k + S::STAGES - 1);
    const int i0 = (warp + k * kFewWarps) * 16;
    const uint32_t st = ring + (k % S::STAGES) * (2 * S::TILE);
    // ---- S^T = K Q^T
    float s[NT][4], s2[NT][4];  // two chains: an instruction does not wait for the one before it
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][e] = s2[nt][e] = 0.f;
#pragma unroll
    for (int c = 0; c < CK; ++c) {
      const uint4 p0 = lds128(st + k_piece(g, 4 * c + t4) * 16), p1 = lds128(st + k_piece(g + 8, 4 * c + t4) * 16);
      const uint32_t w0[4] = {p0.x, p0.y, p0.z, p0.w};
      const uint32_t w1[4] = {p1.x, p1.y, p1.z, p1.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t a0, a1, a2, a3;
        f16x4_of(w0[j], a0, a2);
        f16x4_of(w1[j], a1, a3);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          uint2 q;
          if constexpr (NT == 1) q = qf[4 * c + j];
          else q = qsm[(nt * CK * 4 + 4 * c + j) * 32 + lane];
          mma_f16(j & 1 ? s2[nt] : s[nt], a0, a1, a2, a3, q.x, q.y);
        }
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][e] += s2[nt][e];
    // ---- running maxima and weights
    // a position without a row lies behind every query
    int at0 = base + i0 + g, at1 = at0 + 8;
    float k0, k1, e0, e1;
    if constexpr (UNI) {
      const bool has = __shfl_sync(0xffffffffu, row_l, k) >= 0;
      if (!has || i0 + g >= kn) at0 = 0x7fffffff;
      if (!has || i0 + g + 8 >= kn) at1 = 0x7fffffff;
      k0 = k1 = __shfl_sync(0xffffffffu, ks_l, k);
      e0 = e1 = __shfl_sync(0xffffffffu, ve_l, k);
    } else {
      if (row_s[i0 + g] < 0) at0 = 0x7fffffff;
      if (row_s[i0 + g + 8] < 0) at1 = 0x7fffffff;
      k0 = ks_s[i0 + g], k1 = ks_s[i0 + g + 8];
      e0 = ve_s[i0 + g], e1 = ve_s[i0 + g + 8];
    }
    uint32_t pb[NT][2];
    bool moved = false;
    float f[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const bool see0 = at0 <= pos[nt][e], see1 = at1 <= pos[nt][e];
        const float s0 = s[nt][e] * (qs[nt][e] * k0), s1 = s[nt][2 + e] * (qs[nt][e] * k1);
        // a NaN score counts as the lowest value here and spoils the sums below
        float n = see0 ? fmaxf(s0, -1e38f) : -INFINITY, m = n + e0;
        const float n1 = see1 ? fmaxf(s1, -1e38f) : -INFINITY;
        if constexpr (!UNI) m = fmaxf(m, n1 + e1);
        n = fmaxf(n, n1);
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          if constexpr (!UNI) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
          n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, x));
        }
        if constexpr (UNI) m = n + e0;
        // most tiles move no reference and rescale nothing
        f[nt][e] = 1.f;
        if (m > M[nt][e] + kSpan) {
          m -= kBelow;
          f[nt][e] = ex2(M[nt][e] - m);
          M[nt][e] = m;
          moved = true;
        }
        if (n > N[nt][e] + 8.f) {
          l[nt][e] *= ex2(N[nt][e] - n);
          N[nt][e] = n;
        }
        w[e] = see0 ? ex2(s0 + e0 - M[nt][e]) : 0.f;
        w[2 + e] = see1 ? ex2(s1 + e1 - M[nt][e]) : 0.f;
        if (see0) l[nt][e] += ex2(s0 - N[nt][e]);
        if (see1) l[nt][e] += ex2(s1 - N[nt][e]);
      }
      pb[nt][0] = transpose8x8(pack_f16(w[0], w[1]));
      pb[nt][1] = transpose8x8(pack_f16(w[2], w[3]));
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < HV * MT; ++i) {
          o[nt][i][0] *= f[nt][0];
          o[nt][i][1] *= f[nt][1];
          o[nt][i][2] *= f[nt][0];
          o[nt][i][3] *= f[nt][1];
        }
    }
    // ---- V; NaN of positions that some row does not see are taken out here and put back by row below
    uint32_t vr[HV][4][VW];
#pragma unroll
    for (int h = 0; h < HV; ++h)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int r = 2 * t4 + (x & 1) + 8 * (x >> 1);
        if constexpr (VW == 4) {
          const uint4 w = lds128(st + S::TILE + v_piece(r, 8 * h + g) * 16);
          vr[h][x][0] = w.x; vr[h][x][1] = w.y; vr[h][x][2] = w.z; vr[h][x][3] = w.w;
        } else {
          asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];"
                       : "=r"(vr[h][x][0]), "=r"(vr[h][x][1])
                       : "r"(st + S::TILE + v_piece(r, g >> 1) * 16 + (g & 1) * 8));
        }
      }
    if (base + i0 + 15 > kmin) {
      uint32_t marks = 0;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (base + i0 + 2 * t4 + (x & 1) + 8 * (x >> 1) <= kmin) continue;
#pragma unroll
        for (int h = 0; h < HV; ++h)
#pragma unroll
          for (int y = 0; y < VW; ++y) {
            marks |= nan_marks(vr[h][x][y]);
            vr[h][x][y] = clear_nan(vr[h][x][y]);
          }
      }
      if (marks) nan_seen = 1;
    }
    // ---- O^T += V^T P^T
#pragma unroll
    for (int h = 0; h < HV; ++h)
#pragma unroll
      for (int x = 0; x < VW; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint32_t sel = y ? 0x7362u : 0x5140u;
          uint32_t a0, a1, a2, a3;
          f16x4_of(__byte_perm(vr[h][0][x], vr[h][1][x], sel), a0, a1);
          f16x4_of(__byte_perm(vr[h][2][x], vr[h][3][x], sel), a2, a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][h * MT + 2 * x + y], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
        }
  }
  pdl_trigger();

  // ---- join the warps, in warp order
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = l[nt][e];
#pragma unroll
      for (int m = 4; m < 32; m <<= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
      if (g == 0) ml_s[warp][8 * nt + 2 * t4 + e] = make_float4(M[nt][e], N[nt][e], x, 0.f);
    }
  __syncthreads();
  if (tid < R) {
    float m = -INFINITY, n = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
      m = fmaxf(m, ml_s[w][tid].x);
      n = fmaxf(n, ml_s[w][tid].y);
    }
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w)
      if (ml_s[w][tid].y != -INFINITY) L += ml_s[w][tid].z * ex2(ml_s[w][tid].y - n);
    fin_s[tid] = make_float4(m, n, L, 0.f);
  }
  const int64_t grp = ((int64_t)b * a.c.hkv + head) * a.row_groups + rg;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float f[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 8 * nt + 2 * t4 + e;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) m = fmaxf(m, ml_s[w][r].x);
      f[e] = M[nt][e] == -INFINITY ? 0.f : ex2(M[nt][e] - m);
    }
    float* ow = os + (warp * 8 + 2 * t4) * S::PITCH;
#pragma unroll
    for (int h = 0; h < HV; ++h)
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const float* c = o[nt][h * MT + i];
        const int d = (D >= 128 ? 128 * h + 16 * g : 8 * g) + 2 * i;
        const int at = d + (d >> 4) * 2;
        *reinterpret_cast<float2*>(ow + at) = make_float2(c[0] * f[0], c[2] * f[0]);
        *reinterpret_cast<float2*>(ow + S::PITCH + at) = make_float2(c[1] * f[1], c[3] * f[1]);
      }
    __syncthreads();
    for (int i = tid; i < 4 * D; i += kFewWarps * 32) {
      const int r = i / (D / 2), d = i % (D / 2) * 2, at = d + (d >> 4) * 2;
      const int gr = row0 + 8 * nt + r;
      if (gr >= total_rows) continue;
      float2 O = make_float2(0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) {
        const float2 x = *reinterpret_cast<const float2*>(os + (w * 8 + r) * S::PITCH + at);
        O.x += x.x;
        O.y += x.y;
      }
      const int t = gr / a.G;
      const int p = t < ql ? seq_full - ql + t : -1;
      if (nan_seen) {  // rare: a position past kmin holds NaN in V
        for (int j = max(kmin + 1, base); j <= min(p, base + kn - 1); ++j) {
          const int blk = ld_act(table + j / a.c.block_size);
          if ((unsigned)blk >= (unsigned)a.c.num_blocks) continue;
          const int64_t row = (int64_t)blk * a.c.block_size + j % a.c.block_size;
          const uint32_t v = __ldcg(reinterpret_cast<const uint16_t*>(a.c.pages + a.c.plane + a.c.layer + row * rs +
                                                                      (int64_t)head * D + d));
          if ((v & 0x7fu) == 0x7fu) O.x = __int_as_float(0x7fc00000);
          if ((v & 0x7f00u) == 0x7f00u) O.y = __int_as_float(0x7fc00000);
        }
      }
      if (a.nsplit == 1) {
        const float4 z = fin_s[8 * nt + r];
        const float k = ex2(0.5f * (z.x - z.y));  // twice, as in the join
        const bool ok = p >= 0 && z.z != 0.f;
        *reinterpret_cast<__nv_bfloat162*>(reinterpret_cast<bf16*>(a.out) +
                                           (((int64_t)b * a.T + t) * a.hq + head * a.G + (gr - t * a.G)) * D + d) =
            __floats2bfloat162_rn(ok ? O.x / z.z * k * k : 0.f, ok ? O.y / z.z * k * k : 0.f);
      } else {
        *reinterpret_cast<float2*>(a.ws_o + ((grp * a.nsplit + split) * R + 8 * nt + r) * D + d) = O;
      }
    }
    __syncthreads();
  }
  if (a.nsplit > 1 && tid < R) a.ws_ml[(grp * a.nsplit + split) * R + tid] = fin_s[tid];
}


// ------------------------------------------------------------------ many query rows (bf16): prompt chunks
// A CTA takes 128 query rows of one KV head and a split of the positions, on the tensor cores (tcgen05, f16
// operands, fp32 accumulators in TMEM): S = Q K^T for a tile of 64 positions (M = 128, N = 64), weights in f16
// to shared memory, O += P V (N = D).  K and V become f16 on the way into shared memory, in one layout: rows
// are positions, 64 dims to a 128-byte swizzled line.  That is K-major for K and, with V's dims as the long
// side of its operand, MN-major for V, so nothing is transposed.
//   warps 0-7   two threads a query row, half a tile's positions each: scores out of TMEM, maxima (exchanged between
//               the two), weights, rescaling of O (only when a row's reference has to move, see the few-row
//               kernel), the result
//   warps 8-15  pages to f16 tiles, four warps a tile in turn, the bytes of the next two tiles in flight
//   warp 16     issues the products: S of tile j + 1 goes before O of tile j, so the weights of one tile are
//               made while the tensor cores work on the next
// A tile takes 2300 cycles, its products alone 1080: bound by the latency of the chain scores - maxima - weights of
// its 8 row warps, which 17 warps and two stages do not hide (issue slots 40 % busy, tensor cores 23 %).  Four
// sequences of 1000 to 8192 positions, 512 rows each (one 344): 27 us, 307 TFLOP/s.  Two groups of row warps that take
// tiles in turn came out no faster (their two P tiles cost as much shared memory as a third stage would).
// All waits are bounded, and a warp's lanes give up together.  A CTA that gives up raises `gave_up`, lets its copies and
// products end, frees its TMEM and writes NaN to the rows that it has not finished, straight to global memory: warps
// that have not noticed may still be writing tiles where results are staged.  (A row that is finished has waited for
// the last product, hence for every tile.)
namespace many {

constexpr int ROWS = 128;    // query rows of a CTA: TMEM lanes
constexpr int TILE = 64;     // positions of a tile
constexpr int SOFT = 256;    // threads of the row warps: two a query row, 32 positions of a tile each
constexpr int CONV = 256;    // threads of the converting warps
constexpr int THREADS = SOFT + CONV + 32;
constexpr int kMinTiles = 2; // of a split
constexpr int META = 4;      // tiles whose scales are kept: a tile's are read until its weights are done
constexpr uint32_t kPolls = 1u << 24;
// Stands in a scale's place for a position without a row: a NaN of no computation.  No flag of its own and no change of
// sign, since the scales are not touched before their tile is converted (touching them where they are fetched costs the
// loads' latency: 41 -> 46 us for 4 sequences of 500 to 4000 positions, 16 heads of 256, 64 rows each).
constexpr uint32_t kNoRow = 0xffc0a5e1u;
__device__ uint32_t gave_up;  // 1 once a CTA's wait ran out (ssd_kv8_attention_status)

template <int D>
struct Cfg {
  static constexpr uint32_t KV = TILE * D * 2, P = ROWS * TILE * 2;
  static constexpr uint32_t PITCH = D * 4 + 16;  // bytes of a row of the result, which leaves through K, V and P
  static_assert(ROWS * PITCH <= 4 * KV + P);
  // Q comes in through V and P, rows QPITCH bytes apart
  static constexpr uint32_t QPITCH = D * 2 + 16;
  static_assert(ROWS * QPITCH <= 2 * KV + P);
  static constexpr uint32_t k = 0, v = 2 * KV, p = v + 2 * KV, pairs = p + P;
  static constexpr uint32_t meta = pairs + 2 * 2 * ROWS * 8, bars = meta + META * TILE * 4;
  static constexpr size_t smem = 1024 + bars + 192;  // 22 barriers, TMEM address, two flags
  // TMEM columns: two tiles' scores, Q (two f16 to a column), O
  static constexpr uint32_t q_col = 2 * TILE, o_col = q_col + D / 2, tmem_cols = D == 64 ? 256 : 512;
  static_assert(o_col + D <= tmem_cols);
};
// A position's scale exponents in one word: K's + 256 in the upper half (0: the position has no row), V's + 256 below.
__device__ __forceinline__ uint32_t pack_meta(int ke, int ve) { return (uint32_t)(ke + 256) << 16 | (uint32_t)(ve + 256); }
__device__ __forceinline__ int meta_k(uint32_t m) { return (int)(m >> 16) - 256; }
__device__ __forceinline__ float meta_v(uint32_t m) { return (float)((int)(m & 0xffffu) - 256); }

// For whole warps: true in every lane, or false in every lane (some lanes' waits may have ended: nothing goes by that).
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int* stop, uint32_t polls) {
  bool ok = false;
  for (uint32_t i = 0; i < polls; ++i) {
    ok = tc::mbar_try_wait(bar, parity);
    if (ok || ((i & 255u) == 255u && *stop)) break;
  }
  if (!ok) *stop = 1;
  return __all_sync(0xffffffffu, ok);
}

using tc::add2;
using tc::fma2;
using tc::tmem_load32;
using tc::tmem_ready;
using tc::tmem_store16;
using tc::tmem_store32;
using tc::umma_ts;

// 16-byte piece `c` (of 64-dim lines) of row r of an operand whose lines of `rows` rows lie line after line.
__device__ __forceinline__ uint32_t piece(uint32_t base, int rows, int r, int c) {
  return base + (c >> 3) * (rows * 128) + (r >> 3) * 1024 + (r & 7) * 128 + (((c & 7) ^ (r & 7)) << 4);
}
__device__ __forceinline__ void sts128(uint32_t p, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// f16 operands, fp32 accumulator, M = 128; B's long side contiguous (MN-major) or not.
template <int N, bool B_MN>
__host__ __device__ constexpr uint32_t idesc() {
  return (1u << 4) | ((B_MN ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);
}
__device__ __forceinline__ uint64_t mn_desc(uint32_t saddr) { return tc::mn128_desc<TILE>(saddr); }

// Which part of which sequence split `slot` is, where the splits go by the sequences' lengths: the shortest split of
// whole tiles with which all sequences together make no more than nsplit, found by bisection.  Every warp works it out
// for itself; lane x holds sequences x, x + 32, ..
struct Part {
  int b, split, span;  // sequence (-1: none), number in it, positions of a split
  int seq, ql;         // its lengths
};
constexpr int kPlanRegs = 3;          // 148 splits at most, two of them at least for each sequence

__device__ __forceinline__ Part find_part(const Kv8Attn& a, int slot, bool publish) {
  const int lane = threadIdx.x & 31;
  int seq[kPlanRegs], ql[kPlanRegs];
#pragma unroll
  for (int k = 0; k < kPlanRegs; ++k) {
    seq[k] = lane + 32 * k < a.B ? ld_act(a.seq_lens + lane + 32 * k) : 0;
    ql[k] = lane + 32 * k < a.B && a.q_lens ? ld_act(a.q_lens + lane + 32 * k) : a.T;
  }
  uint32_t t[kPlanRegs], total = 0;
#pragma unroll
  for (int k = 0; k < kPlanRegs; ++k) {
    const int n = max(min(seq[k], min(a.max_blocks * a.c.block_size, kMaxSeqLen)), 0);
    t[k] = (uint32_t)(n / TILE + (n % TILE != 0));
    total += t[k];
  }
  total = __reduce_add_sync(0xffffffffu, total);
  auto parts = [&](int k, uint32_t span) {
    return lane + 32 * k < a.B ? max(1u, (t[k] + span - 1) / span) : 0u;
  };
  const uint32_t N = (uint32_t)a.nsplit, extra = N - (uint32_t)a.B;
  uint32_t lo = max((uint32_t)kMinTiles, (total + N - 1) / N), hi = max(lo, (total + extra - 1) / extra);
  while (lo < hi) {
    const uint32_t mid = (lo + hi) / 2;
    uint32_t n = 0;
#pragma unroll
    for (int k = 0; k < kPlanRegs; ++k) n += parts(k, mid);
    if (__reduce_add_sync(0xffffffffu, n) <= N) hi = mid;
    else lo = mid + 1;
  }
  Part p{-1, 0, (int)(lo * TILE), 0, 0};
  uint32_t before = 0;
#pragma unroll
  for (int k = 0; k < kPlanRegs; ++k) {
    if (32 * k >= a.B) break;
    const uint32_t mine = parts(k, lo);
    uint32_t x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    const int first = (int)(before + x - mine);
    if (publish && mine) a.plan[lane + 32 * k] = make_int2(first, (int)mine);
    const uint32_t hit = __ballot_sync(0xffffffffu, slot >= first && slot < first + (int)mine);
    if (hit) {
      const int from = __ffs(hit) - 1;
      p.b = from + 32 * k;
      p.split = slot - __shfl_sync(0xffffffffu, first, from);
      p.seq = __shfl_sync(0xffffffffu, seq[k], from);
      p.ql = __shfl_sync(0xffffffffu, ql[k], from);
    }
    before += __shfl_sync(0xffffffffu, x, 31);
  }
  return p;
}

// UNI: block_size is a multiple of 16.
template <int D, bool UNI>
__global__ void __launch_bounds__(THREADS, 1) kv8_attention_many_kernel(const Kv8Attn a) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = tc::smem_u32(smem_raw), sm = (raw + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (sm - raw);
  uint32_t* meta = reinterpret_cast<uint32_t*>(gen + C::meta);  // [META][TILE], see pack_meta
  auto bar = [&](int i) { return sm + C::bars + 8 * i; };
  const uint32_t q_in = bar(0), o_done = bar(1), drained = bar(2), p_full = bar(3), q_tmem = bar(4);
  auto k_full = [&](int s) { return bar(7 + s); };
  auto k_free = [&](int s) { return bar(9 + s); };
  auto v_full = [&](int s) { return bar(11 + s); };
  auto v_free = [&](int s) { return bar(13 + s); };
  auto s_full = [&](int s) { return bar(15 + s); };
  auto pair = [&](int q) { return bar(18 + q); };
  float2* pair_s = reinterpret_cast<float2*>(gen + C::pairs);  // [tile parity][half][row]: the threads' maxima
  uint32_t* slot = reinterpret_cast<uint32_t*>(gen + C::bars + 176);
  volatile int* stop = reinterpret_cast<volatile int*>(slot + 1);
  volatile int* nan_seen = reinterpret_cast<volatile int*>(slot + 2);
  auto held = [&](uint32_t b, uint32_t parity) { return wait(b, parity, stop, a.polls); };

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int head = blockIdx.y / a.row_groups, rg = blockIdx.y % a.row_groups;
  if (tid == 0) {
    tc::mbar_init(q_in, ROWS);
    tc::mbar_init(q_tmem, SOFT);
    tc::mbar_init(p_full, SOFT);
    tc::mbar_init(o_done, 1);
    tc::mbar_init(drained, 1);
    for (int q = 0; q < 4; ++q) tc::mbar_init(pair(q), 64);
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(k_full(s), CONV / 2);
      tc::mbar_init(k_free(s), 1);
      tc::mbar_init(v_full(s), CONV / 2);
      tc::mbar_init(v_free(s), 1);
      tc::mbar_init(s_full(s), 1);
    }
    *stop = 0;
    *nan_seen = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == THREADS / 32 - 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(slot)),
                 "r"(C::tmem_cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *slot;
  pdl_wait();

  Part part;
  if (a.plan) {
    part = find_part(a, blockIdx.x, blockIdx.x == 0 && blockIdx.y == 0 && warp == 0);
  } else {
    const int z = blockIdx.z;
    part = Part{z, 0, a.split, ld_act(a.seq_lens + z), a.q_lens ? ld_act(a.q_lens + z) : a.T};
  }
  const bool idle = part.b < 0;  // fewer splits than there may be
  const int b = idle ? 0 : part.b, span = part.span, seq_full = part.seq, ql = min(max(part.ql, 0), a.T);
  const int seq = min(min(seq_full, a.max_blocks * a.c.block_size), a.plan ? kMaxSeqLen : span);
  const int base = part.split * span;
  const int row0 = rg * ROWS, rows = min(ROWS, a.G * a.T - row0);
  const int n0 = seq_full - ql;
  const int t0 = row0 / a.G, t1 = min((row0 + rows - 1) / a.G, ql - 1);  // the group's first and last real token
  const int kmin = max(n0 + t0, 0);                                       // every row that sees anything sees 0..kmin
  const int kn = idle || t0 > t1 ? 0 : min(min(seq, base + span), n0 + t1 + 1) - base;
  const int tiles = kn > 0 ? (kn + TILE - 1) / TILE : 0;
  const int32_t* table = a.tables + (int64_t)b * a.max_blocks;

  if (warp < SOFT / 32) {
    // -------------------------------------------------------------- rows
    const int quad = warp & 3, half = warp >> 2;  // TMEM lanes 32 quad .., positions 32 half .. of a tile
    const int r = quad * 32 + lane, gr = row0 + r, t = gr / a.G, g = gr - t * a.G;
    const bool real = r < rows && t < ql && n0 + t >= 0;
    const int pos = real ? n0 + t : -1;
    const int64_t at = (((int64_t)b * a.T + t) * a.hq + head * a.G + g) * D;
    const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
    // The row's two threads swap a pair of numbers; false when the CTA gives up.  `k`: how many swaps went before.
    auto swap = [&](float2* at2, int k, float& x, float& y) {
      at2[((k & 1) * 2 + half) * ROWS + r] = make_float2(x, y);
      tc::mbar_arrive(pair(quad));
      if (!held(pair(quad), k & 1)) return false;
      const float2 z = at2[((k & 1) * 2 + (half ^ 1)) * ROWS + r];
      x = z.x;
      y = z.y;
      return true;
    };
    float qs = 1.f;
    bool ok = true;
    if (tiles > 0) {
      // Q: rows to shared memory by bulk copies, then this thread's half of its row, in f16 under a power of two of
      // the row, into TMEM as the first operand (from shared memory it would cost S more of that memory's bandwidth
      // than K does)
      constexpr int NQ = D / 16;
      const uint32_t row = sm + C::v + r * C::QPITCH;
      if (half == 0) {
        if (real) {
          tc::mbar_expect_tx(q_in, D * 2);
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(row),
                       "l"(reinterpret_cast<const bf16*>(a.q) + at), "r"(D * 2), "r"(q_in)
                       : "memory");
        } else {
          tc::mbar_arrive(q_in);
        }
      }
      ok = held(q_in, 0);
      uint4 w[NQ];
#pragma unroll
      for (int i = 0; i < NQ; ++i) w[i] = real && ok ? lds128(row + half * D + 16 * i) : make_uint4(0, 0, 0, 0);
      __nv_bfloat162 t2 = __float2bfloat162_rn(0.f);
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) t2 = __hmax2(t2, __habs2(h[j]));
      }
      // largest magnitude, NaN aside (it reaches the scores by itself)
      float top = fmaxf(__low2float(t2), __high2float(t2)), other = top, unused = 0.f;
      ok = ok && swap(pair_s, 0, other, unused);
      top = fmaxf(top, other);
      const int e = min(max((int)(__float_as_uint(top) >> 23) - 127 - 14, -118), 120);
      // The row's factor is never negative.  A row with an infinity has no finite score, or one less itself: NaN, put
      // into Q so that only positions that it sees bring it in.
      const float inv = top == INFINITY ? __int_as_float(0x7fc00000) : copysignf(exp2i(-e), a.scale);
      qs = exp2i(e) * fabsf(a.scale) * 1.4426950408889634f;
#pragma unroll
      for (int c = 0; c < NQ; c += 4) {
        uint32_t y[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t v[4] = {w[c + i].x, w[c + i].y, w[c + i].z, w[c + i].w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            y[4 * i + j] = pack_f16(__uint_as_float(v[j] << 16) * inv, __uint_as_float(v[j] & 0xffff0000u) * inv);
        }
        tmem_store16(lanes + C::q_col + half * (D / 4) + 4 * c, y);
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      tc::tc_fence_before();
      if (ok) tc::mbar_arrive(q_tmem);
    }
    // M: what the weights are relative to, N: what l is; -1e38 where nothing has been seen
    float M = -1e38f, N = -1e38f, l = 0.f;
#pragma unroll 1
    for (int j = 0; ok && j < tiles; ++j) {
      ok = held(s_full(j & 1), (j >> 1) & 1);
      if (!ok) break;
      tc::tc_fence_after();
      const int p0 = base + j * TILE + 32 * half;  // this thread's 32 positions
      const uint32_t* mt = meta + (j % META) * TILE + half * (UNI ? 2 : 32);
      uint32_t x[32];
      tmem_load32(lanes + (j & 1) * TILE + 32 * half, x);
      float m = -1e38f, n = -1e38f, f = 1.f;
      // a NaN score counts as the lowest value in the maxima and spoils the sums
      float ca = 0.f, cb = 0.f, va = 0.f, vb2 = 0.f;
      if constexpr (UNI) {
        // two groups of 16 positions, one pair of scales each
        uint32_t wa = mt[0], wb = mt[1];
        const bool ina = wa >= 65536u, inb = wb >= 65536u;
        if (!ina) wa = pack_meta(0, 0);
        if (!inb) wb = pack_meta(0, 0);
        ca = qs * exp2i(meta_k(wa));
        cb = qs * exp2i(meta_k(wb));
        // keeps the mask's infinity out of 0 * infinity (the scores stay below 2^-90): all-zero pages, zero rows
        if (ca == 0.f) ca = 1e-38f;
        if (cb == 0.f) cb = 1e-38f;
        va = meta_v(wa);
        vb2 = meta_v(wb);
        tmem_ready(x);
        if (p0 + 31 > kmin || p0 + 32 > base + kn || !ina || !inb) {  // hide what the row does not see
          const int k = min(pos, base + kn - 1) - p0;
          uint32_t keep = k >= 31 ? 0xffffffffu : k < 0 ? 0u : (2u << k) - 1;
          if (!ina) keep &= 0xffff0000u;
          if (!inb) keep &= 0x0000ffffu;
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(keep >> i & 1)) x[i] = 0xff800000u;
        }
        float ya = -INFINITY, yb = -INFINITY;  // of the raw products: their factors are positive
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          ya = fmaxf(ya, fmaxf(__uint_as_float(x[i]), __uint_as_float(x[i + 1])));
          yb = fmaxf(yb, fmaxf(__uint_as_float(x[16 + i]), __uint_as_float(x[17 + i])));
        }
        ya = fmaxf(ya * ca, -1e38f);
        yb = fmaxf(yb * cb, -1e38f);
        n = fmaxf(ya, yb);
        m = fmaxf(ya + va, yb + vb2);
      } else {
        tmem_ready(x);
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const uint32_t w = mt[i];
          const bool see = w >= 65536u && p0 + i <= pos;
          const float s = see ? __uint_as_float(x[i]) * (qs * exp2i(meta_k(w))) : -INFINITY;
          x[i] = __float_as_uint(s);
          if (see) {
            const float y = fmaxf(s, -1e38f);
            n = fmaxf(n, y);
            m = fmaxf(m, y + meta_v(w));
          }
        }
      }
      float mo = m, no = n;
      ok = swap(pair_s, j + 1, mo, no);
      if (!ok) break;
      m = fmaxf(m, mo);
      n = fmaxf(n, no);
      if (m > M + kSpan) {
        m -= kBelow;
        f = ex2(M - m);
        M = m;
      }
      if (n > N + 8.f) {
        l *= ex2(N - n);
        N = n;
      }
      uint32_t w[16];
      if constexpr (UNI) {
        // Weights are 2^(s + v - M), l's terms 2^(s - N): a group's sum of weights is carried over by 2^(M - v - N).
        // Not where v lies more than 40 below M - N (a page of small V beside one of large V, whichever of the row's two
        // threads has it): there weights vanish below 2^-126 that count in l, 2^-86 of its largest and up, and the
        // factor may overflow.  Then l takes its own exponentials.
        const bool wide = fminf(va, vb2) < M - N - 40.f;
        if (wide) {
#pragma unroll
          for (int i = 0; i < 32; ++i) l += ex2(fmaf(__uint_as_float(x[i]), i < 16 ? ca : cb, -N));
        }
        const float oa = va - M, ob = vb2 - M;
        float2 sa = make_float2(0.f, 0.f), sb = sa;
        const float2 ca2 = make_float2(ca, ca), cb2 = make_float2(cb, cb);
        const float2 oa2 = make_float2(oa, oa), ob2 = make_float2(ob, ob);
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          float2 e = fma2(make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), ca2, oa2);
          float2 d = fma2(make_float2(__uint_as_float(x[16 + i]), __uint_as_float(x[17 + i])), cb2, ob2);
          e = make_float2(ex2(e.x), ex2(e.y));
          d = make_float2(ex2(d.x), ex2(d.y));
          sa = add2(sa, e);
          sb = add2(sb, d);
          w[i / 2] = pack_f16(e.x, e.y);
          w[8 + i / 2] = pack_f16(d.x, d.y);
        }
        if (!wide) {
          l = fmaf(sa.x + sa.y, ex2(-oa - N), l);
          l = fmaf(sb.x + sb.y, ex2(-ob - N), l);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const float s0 = __uint_as_float(x[i]), s1 = __uint_as_float(x[i + 1]);
          w[i / 2] = pack_f16(ex2(s0 + (meta_v(mt[i]) - M)), ex2(s1 + (meta_v(mt[i + 1]) - M)));
          l += ex2(s0 - N) + ex2(s1 - N);
        }
      }
      if (j > 0) {  // the tile before has been added: its weights may go, and O may be rescaled
        ok = held(o_done, (j - 1) & 1);
        if (!ok) break;
        tc::tc_fence_after();
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sts128(piece(sm + C::p, ROWS, r, 4 * half + i),
               make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
      if (j > 0 && __any_sync(0xffffffffu, f != 1.f)) {  // half of O each
#pragma unroll 1
        for (int c = half * (D / 2); c < (half + 1) * (D / 2); c += 32) {
          uint32_t y[32];
          tmem_load32(lanes + C::o_col + c, y);
          tmem_ready(y);
#pragma unroll
          for (int i = 0; i < 32; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * f);
          tmem_store32(lanes + C::o_col + c, y);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc::tc_fence_before();
      tc::mbar_arrive(p_full);
    }
    if (ok && tiles > 0) {
      float lo = l, unused = 0.f;
      ok = swap(pair_s, tiles + 1, lo, unused);
      l += lo;
      ok = ok && held(o_done, (tiles - 1) & 1);
    }
    tc::tc_fence_after();
    const bool partial = a.plan != nullptr;
    const int64_t po = ((int64_t)blockIdx.y * a.nsplit + blockIdx.x) * ROWS + r;
    const bool any = real && l != 0.f;  // l is NaN, not 0, where a seen score is
    const float nan = __int_as_float(0x7fc00000);
    if (partial && !idle && half == 0) a.ws_ml[po] = make_float4(M, N, ok ? l : nan, 0.f);
    if (!ok) {
      if (lane == 0) atomicExch(&gave_up, 1u);
      // Q's copies land before shared memory goes
      for (uint32_t i = 0; i < kPolls && !tc::mbar_try_wait(q_in, 0); ++i) {}
#pragma unroll 1
      for (int d = half * (D / 2); d < (half + 1) * (D / 2); ++d) {
        if (partial) a.ws_o[po * D + d] = nan;
        else if (r < rows) reinterpret_cast<bf16*>(a.out)[at + d] = __float2bfloat16_rn(real ? nan : 0.f);
      }
    } else if (!partial || tiles > 0) {
      // O through the shared memory of K, V and P (every product is done): a thread puts its half row there and
      // sends it off with one bulk copy
      const float kk = partial ? 1.f : any ? ex2(0.5f * (M - N)) : 0.f, k = partial ? 1.f : any ? kk / l : 0.f;
      const bool zero = !partial && !any;  // O may be anything where a row sees nothing
      constexpr int HD = D / 2;
      const uint32_t mine = sm + r * C::PITCH + half * (HD * 4);
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t y[32];
        if (tiles > 0) {
          tmem_load32(lanes + C::o_col + half * HD + c, y);
          tmem_ready(y);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) y[i] = 0;
        }
        if (partial) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            sts128(mine + c * 4 + 16 * i, make_uint4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]));
        } else {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint32_t z[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              const __nv_bfloat162 v2 = __floats2bfloat162_rn(__uint_as_float(y[i + 2 * h]) * k * kk,
                                                              __uint_as_float(y[i + 2 * h + 1]) * k * kk);
              z[h] = zero ? 0u : *reinterpret_cast<const uint32_t*>(&v2);
            }
            sts128(mine + c * 2 + i * 2, make_uint4(z[0], z[1], z[2], z[3]));
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      if (partial || r < rows) {
        const void* to = partial ? (const void*)(a.ws_o + po * D + half * HD)
                                      : (const void*)(reinterpret_cast<bf16*>(a.out) + at + half * HD);
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to), "r"(mine),
                     "r"(partial ? HD * 4 : HD * 2)
                     : "memory");
      }
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // before shared memory goes, and before the NaN below
      if (*nan_seen && real) {  // rare: a position past kmin holds NaN in V
#pragma unroll 1
        for (int j = max(kmin + 1, base); j <= min(pos, base + kn - 1); ++j) {
          const int blk2 = ld_act(table + j / a.c.block_size);
          if ((unsigned)blk2 >= (unsigned)a.c.num_blocks) continue;
          const uint8_t* v = a.c.pages + a.c.plane + a.c.layer +
                             (((int64_t)blk2 * a.c.block_size + j % a.c.block_size) * a.c.hkv + head) * D;
#pragma unroll 1
          for (int d = half * HD; d < (half + 1) * HD; ++d) {
            if ((__ldcg(v + d) & 0x7f) != 0x7f) continue;
            if (partial) a.ws_o[po * D + d] = __int_as_float(0x7fc00000);
            else reinterpret_cast<bf16*>(a.out)[at + d] = __ushort_as_bfloat16(0x7fc0);
          }
        }
      }
    }
    tc::tc_fence_before();
  } else if (warp < (SOFT + CONV) / 32) {
    // -------------------------------------------------------------- pages to f16 tiles
    // Four warps take the even tiles, four the odd ones (a warp's waits and addresses cost as much as its rows), a
    // warp 16 positions of a tile: RPI of them at a time, 16 dims a lane, eight lanes on four pieces of an even and
    // an odd row (their 16-byte stores then meet no bank twice).  The bytes come through registers: shared memory's
    // bandwidth is what a tile takes most of.
    constexpr int PCS = D / 16, RPI = 32 / PCS, NI = 16 / RPI, NB = UNI ? 1 : NI;
    const int set = (warp - SOFT / 32) >> 2, cw = warp & 3;
    const int rr = ((lane >> 2) & 1) | ((lane >> 3) / (PCS / 4)) << 1, pc = (lane & 3) | ((lane >> 3) % (PCS / 4)) << 2;
    const uint8_t* kp = a.c.pages + a.c.layer + (int64_t)head * D + pc * 16;
    const float* sc = a.c.scales + a.c.scale_layer + head;
    const int64_t rs = (int64_t)a.c.hkv * D;
    int blk[NB], off[NB];        // of the tile to be fetched next
    uint4 kb[NI], vb[NI];        // this tile's bytes, then the next one's as soon as they are converted: they have two
    uint32_t ks[NB], vs[NB];     // tiles' time to arrive; and the bits of the scales (kNoRow: no row)
    int ids = -1;          // UNI: lane x has the block id of the warp's positions in its tile 32 k + x
    auto look = [&](int j) {
      if constexpr (UNI) {
        const int mine = j >> 1;
        if ((mine & 31) == 0) {
          // whatever the length says: a tile's rows are bounded where they are fetched
          const int p = (j + 2 * lane) * TILE + 16 * cw, page = (base + p) / a.c.block_size;
          ids = page < a.max_blocks && p < span ? ld_act(table + page) : -1;
        }
        blk[0] = __shfl_sync(0xffffffffu, ids, mine & 31);
        if (mine == 0) {
          off[0] = (base + j * TILE + 16 * cw) % a.c.block_size;
        } else {
          off[0] += 2 * TILE % a.c.block_size;
          if (off[0] >= a.c.block_size) off[0] -= a.c.block_size;
        }
      } else {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const int p = j * TILE + 16 * cw + rr + i * RPI;
          blk[i] = -1;
          off[i] = 0;
          if (p < kn) {
            const int page = (base + p) / a.c.block_size;
            blk[i] = ld_act(table + page);
            off[i] = base + p - page * a.c.block_size;
          }
        }
      }
    };
    // load tile j's K (plane 0) or V rows and scales (zeros where there is no row)
    auto fetch = [&](int j, int plane, uint4* x, uint32_t* xs) {
      const uint32_t* from = reinterpret_cast<const uint32_t*>(sc + plane * a.c.scale_plane);
#pragma unroll
      for (int i = 0; i < NB; ++i)
        xs[i] = (unsigned)blk[i] < (unsigned)a.c.num_blocks ? ld_act(from + (int64_t)blk[i] * a.c.hkv) : kNoRow;
      if constexpr (UNI) {
        const bool in = (unsigned)blk[0] < (unsigned)a.c.num_blocks;
        const uint8_t* s = kp + plane * a.c.plane + (in ? ((int64_t)blk[0] * a.c.block_size + off[0] + rr) * rs : 0);
        const int left = in ? kn - j * TILE - 16 * cw - rr : 0;  // row i of the lane is there where i RPI < left
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          x[i] = make_uint4(0, 0, 0, 0);
          if (i * RPI < left) x[i] = ld_act_v4(s);
          s += RPI * rs;
        }
      } else {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int n = i % NB;
          x[i] = make_uint4(0, 0, 0, 0);
          if ((unsigned)blk[n] < (unsigned)a.c.num_blocks)
            x[i] = ld_act_v4(kp + plane * a.c.plane + ((int64_t)blk[n] * a.c.block_size + off[n]) * rs);
        }
      }
    };
    if (set < tiles) {
      look(set);
      fetch(set, 0, kb, ks);
      fetch(set, 1, vb, vs);
      look(set + 2);
    }
    // row rr + i RPI of the warp's 16: 128 bytes a row, pieces swizzled by it
    const uint32_t to = (pc >> 2) * (TILE * 128) + cw * 2048 + rr * 128 + ((((2 * pc) & 7) ^ rr) << 4);
    auto put = [&](uint32_t tile, int i, uint4 w) {
      uint4 lo, hi;
      f16x4_of(w.x, lo.x, lo.y);
      f16x4_of(w.y, lo.z, lo.w);
      f16x4_of(w.z, hi.x, hi.y);
      f16x4_of(w.w, hi.z, hi.w);
      const uint32_t at = ((tile + to) ^ ((i * RPI & 7) * 16)) + i * RPI * 128;
      sts128(at, lo);
      sts128(at ^ 16, hi);
    };
    const uint32_t kt = sm + C::k + set * C::KV, vt = sm + C::v + set * C::KV;
#pragma unroll 1
    for (int j = set; j < tiles; j += 2) {
      if (j >= 2 && !held(k_free(set), ((j >> 1) - 1) & 1)) break;
      uint32_t* mt = meta + (j % META) * TILE;
      if (UNI ? lane == 0 : pc == 0) {
#pragma unroll
        for (int i = 0; i < NB; ++i)
          mt[UNI ? cw : 16 * cw + rr + i * RPI] =
              ks[i] == kNoRow ? 0u
                              : pack_meta(scale_exponent(__uint_as_float(ks[i])), scale_exponent(__uint_as_float(vs[i])));
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) put(kt, i, kb[i]);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc::mbar_arrive(k_full(set));
      fetch(j + 2, 0, kb, ks);
      if (j < 2 && !held(q_tmem, 0)) break;  // V's tiles hold Q until then
      if (j >= 2 && !held(v_free(set), ((j >> 1) - 1) & 1)) break;
      if (base + j * TILE + 16 * cw + 15 > kmin) {  // NaN of positions that some row does not see: put back by row above
        uint32_t marks = 0;
#pragma unroll
        for (int i = 0; i < NI; ++i)
          if (base + j * TILE + 16 * cw + rr + i * RPI > kmin)
            marks |= nan_marks(vb[i].x) | nan_marks(vb[i].y) | nan_marks(vb[i].z) | nan_marks(vb[i].w);
        if (marks) {
          *nan_seen = 1;
#pragma unroll
          for (int i = 0; i < NI; ++i)
            if (base + j * TILE + 16 * cw + rr + i * RPI > kmin)
              vb[i] = make_uint4(clear_nan(vb[i].x), clear_nan(vb[i].y), clear_nan(vb[i].z), clear_nan(vb[i].w));
        }
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) put(vt, i, vb[i]);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc::mbar_arrive(v_full(set));
      fetch(j + 2, 1, vb, vs);
      look(j + 4);
    }
    __syncwarp();
  } else {
    // -------------------------------------------------------------- products
    // The whole warp walks the loop and one elected lane issues, so that addresses and descriptors stay in uniform
    // registers: with the loop inside one lane's branch every product waited for them to be moved there.
    if (tiles > 0) {
      uint32_t lead;
      asm volatile("{.reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p;}" : "=r"(lead));
      auto ready = [&](uint32_t b, uint32_t parity) {
        const bool ok = held(b, parity);
        tc::tc_fence_after();
        return ok;
      };
      auto scores = [&](int j) {
        const int s = j & 1;
        if (!ready(k_full(s), (j >> 1) & 1)) return false;
        const uint64_t kd = tc::sw128_desc(sm + C::k + s * C::KV);
        if (lead) {
#pragma unroll
          for (int d = 0; d < D / 64; ++d)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_ts(tmem + s * TILE, tmem + C::q_col + d * 32 + 8 * k, kd + d * ((TILE * 128) >> 4) + 2 * k,
                      idesc<TILE, false>(), d || k);
          tc::umma_commit(k_free(s));
          tc::umma_commit(s_full(s));
        }
        return true;
      };
      bool ok = ready(q_tmem, 0) && scores(0);
#pragma unroll 1
      for (int j = 0; ok && j < tiles; ++j) {
        const int s = j & 1;
        if (j + 1 < tiles) ok = scores(j + 1);
        ok = ok && ready(p_full, j & 1) && ready(v_full(s), (j >> 1) & 1);
        if (!ok) break;
        const uint64_t pd = tc::sw128_desc(sm + C::p);
        const uint64_t vd = mn_desc(sm + C::v + s * C::KV);
        if (lead) {
#pragma unroll
          for (int k = 0; k < TILE / 16; ++k)  // 16 positions: 32 bytes of P's line, two groups of 8 rows of V
            tc::umma_bf16(tmem + C::o_col, pd + 2 * k, vd + (2048 >> 4) * k, idesc<D, true>(), j || k);
          tc::umma_commit(v_free(s));
          tc::umma_commit(o_done);
        }
      }
      if (!ok) {  // let the products issued so far end before TMEM goes back
        if (lead) tc::umma_commit(drained);
        for (uint32_t i = 0; i < kPolls && !tc::mbar_try_wait(drained, 0); ++i) {}
      }
    }
    __syncwarp();
  }
  pdl_trigger();
  __syncthreads();
  if (warp == THREADS / 32 - 1) {
    tc::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::tmem_cols) : "memory");
  }
}

}  // namespace many

std::atomic<uint32_t> wait_polls{many::kPolls};

struct Kv8Layout {
  bool cc;              // CUDA-core kernel (fp32)
  int rows;             // query rows of a group
  int split;            // positions of a split
  int64_t row_groups;
  int nsplit;
  bool planned;         // the splits go by the sequences' lengths
  size_t partials;      // rows of them
  size_t off_ml, off_plan, total;
};

inline size_t up256(size_t x) { return (x + 255) & ~size_t(255); }

// Which kernel: above 32 query rows of a KV head, and more than 8 new tokens, the many-row one (16 heads, one query
// head a KV head, 8 sequences of 500 to 4000 positions: 85 us at any T, where the few-row kernel takes 81 at T = 32
// and 107 at 40; one sequence of 2000: 19.0 against 17.9 and 28.6).  Up to 8 tokens always the few-row one, so that a
// verify step gives a query the bits that decoding it alone does (40 rows, 32 sequences of 500 to 4000, one KV head:
// 48 us, where the other kernel takes 27).
constexpr int kManyRows = 32, kFewTokens = 8;
constexpr int kMaxFewSplit = 1024;  // positions of a split of the few-row kernel, at most

Kv8Layout kv8_layout(bool cc, int B, int T, int hq, int hkv, int D, int max_seq_len) {
  Kv8Layout L{};
  const int64_t total = (int64_t)(hq / hkv) * T;
  L.cc = cc;
  L.rows = cc ? kCcRows : total > kManyRows && T > kFewTokens ? many::ROWS : total > 8 ? 16 : 8;
  // Few rows: 256 positions keep a short context's CTAs many (one sequence of 8192 positions, one KV head: 11.9 us
  // against 18.7 us at 1024); where there is work for every SM either way, longer splits cost fewer prologues and
  // partials (8 sequences, 16 heads, 512 to 4096 positions: 34.5 us at 832, 38.1 at 1024, 43.2 at 256), up to 1024,
  // which leaves many sequences enough CTAs to balance.  Three CTAs an SM, half as many again since not every
  // sequence is as long as the bound.  A bound of 512 stays in one split, which needs no join (one sequence of 500
  // positions, 8 heads of 64: 5.9 against 7.2 us; four of 16 heads of 256: 10.5 against 13.8), but where 8 or more
  // query heads share a KV head and a verify step has several row groups (16.1 against 13.3).  The rule goes by the
  // sequences and the model, never by the new tokens, so a query's bits do not depend on how many stand beside it.
  const int64_t groups = (int64_t)B * hkv, n = groups >= 666 ? 1 : 666 / groups;
  const int64_t even = ((max_seq_len + n - 1) / n + 63) / 64 * 64;
  const int least = max_seq_len <= 512 && hq / hkv < 8 ? 512 : 256;
  L.split = cc ? kCcSplit : (int)(even < least ? least : even > kMaxFewSplit ? kMaxFewSplit : even);
  L.row_groups = (total + L.rows - 1) / L.rows;
  if (L.rows == many::ROWS) {
    // One CTA an SM: as many splits, over all sequences, as one wave of them takes (four sequences of 8192 positions,
    // 256 rows each: 42 us in 128 CTAs, 58 us in 160), where that is two a sequence or more; a context of up to 512
    // positions stays whole (12.9 against 20.6 us at 300).  The sequences' lengths decide on the device (equal shares
    // of the bound instead: 53 against 42 us for 4 sequences of 500 to 4000 positions, 16 heads).
    const int64_t most = B * (((int64_t)max_seq_len - 1) / (many::kMinTiles * many::TILE) + 1);
    const int64_t n = std::min(148 / (hkv * L.row_groups), most);
    L.planned = n >= (int64_t)2 * B && max_seq_len > 512;
    L.nsplit = L.planned ? (int)n : 1;
    L.split = (max_seq_len + many::TILE - 1) / many::TILE * many::TILE;
    L.partials = L.planned ? (size_t)(hkv * L.row_groups * n * L.rows) : 0;
  } else {
    L.nsplit = (max_seq_len + L.split - 1) / L.split;
    L.partials = L.nsplit == 1 ? 0 : (size_t)(groups * L.row_groups) * L.nsplit * L.rows;
  }
  L.off_ml = up256(sizeof(float) * L.partials * D);
  L.off_plan = L.off_ml + up256(sizeof(float4) * L.partials);
  L.total = L.partials ? L.off_plan + up256(sizeof(int2) * B) : 0;
  return L;
}

template <int D>
int launch_cc(cudaStream_t st, const Kv8Attn& a, int B) {
  const dim3 grid(a.nsplit, a.c.hkv * a.row_groups, B);
  SSD_PDL(kv8_attention_cc_kernel<D>, grid, kCcSplit, 0, st, a);
  return a.nsplit == 1 ? SSD_OK : launch_join<float, D, kCcRows, false>(st, a, B);
}

template <int D, int NT, bool UNI>
int launch_few(cudaStream_t st, const Kv8Attn& a, int B) {
  const size_t smem = FewSmem<D, NT, UNI>::total(a.split);
  const dim3 grid(a.nsplit, a.c.hkv * a.row_groups, B);
  auto kern = kv8_attention_few_kernel<D, NT, UNI>;
  static std::atomic<uint64_t> ready{0};
  if (!allow_smem(ready, kern, (int)FewSmem<D, NT, UNI>::total(kMaxFewSplit))) return SSD_ERR_LAUNCH;
  SSD_PDL(kern, grid, kFewWarps * 32, smem, st, a);
  return a.nsplit == 1 ? SSD_OK : launch_join<bf16, D, 8 * NT, true>(st, a, B);
}

template <int D, bool UNI>
int launch_many(cudaStream_t st, const Kv8Attn& a, int B) {
  auto kern = many::kv8_attention_many_kernel<D, UNI>;
  constexpr size_t smem = many::Cfg<D>::smem;
  static_assert(smem <= 227 * 1024);
  static std::atomic<uint64_t> ready{0};
  if (!allow_smem(ready, kern, (int)smem)) return SSD_ERR_LAUNCH;
  SSD_PDL(kern, dim3(a.nsplit, a.c.hkv * a.row_groups, a.plan ? 1 : B), many::THREADS, smem, st, a);
  return !a.plan ? SSD_OK : launch_join<bf16, D, many::ROWS, true>(st, a, B);
}

template <int D>
int launch_bf16(cudaStream_t st, const Kv8Attn& a, const Kv8Layout& L, int B) {
  if (L.rows == many::ROWS) return a.c.block_size % 16 == 0 ? launch_many<D, true>(st, a, B) : launch_many<D, false>(st, a, B);
  if (a.c.block_size % 16 == 0) return L.rows == 8 ? launch_few<D, 1, true>(st, a, B) : launch_few<D, 2, true>(st, a, B);
  return L.rows == 8 ? launch_few<D, 1, false>(st, a, B) : launch_few<D, 2, false>(st, a, B);
}

}  // namespace
}  // namespace ssd

using namespace ssd;

extern "C" size_t ssd_kv8_attention_workspace_size_for(int dtype, int B, int T, int num_heads, int num_kv_heads,
                                                       int head_dim, int max_seq_len) {
  if (B <= 0 || T <= 0 || num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads || head_dim <= 0 ||
      max_seq_len <= 0 || max_seq_len > kMaxSeqLen || (dtype != SSD_DTYPE_BF16 && dtype != SSD_DTYPE_F32))
    return 0;
  return kv8_layout(dtype == SSD_DTYPE_F32, B, T, num_heads, num_kv_heads, head_dim, max_seq_len).total;
}

extern "C" size_t ssd_kv8_attention_workspace_size(int B, int T, int num_heads, int num_kv_heads, int head_dim,
                                                   int max_seq_len) {
  return std::max(
      ssd_kv8_attention_workspace_size_for(SSD_DTYPE_F32, B, T, num_heads, num_kv_heads, head_dim, max_seq_len),
      ssd_kv8_attention_workspace_size_for(SSD_DTYPE_BF16, B, T, num_heads, num_kv_heads, head_dim, max_seq_len));
}

extern "C" int ssd_kv8_attention(ssd_stream_t stream, const void* q, const void* pages, const float* scales,
                                 int dtype, int num_layers, int num_blocks, int block_size, int num_kv_heads,
                                 int head_dim, int layer, const int32_t* block_tables, int max_blocks,
                                 const int32_t* seq_lens, const int32_t* q_lens, void* out, float scale, int B, int T,
                                 int num_heads, int max_seq_len, void* workspace, size_t workspace_bytes) {
  if (int rc = kv8_check(pages, scales, num_layers, num_blocks, block_size, num_kv_heads, head_dim, layer)) return rc;
  if (B < 0 || T < 0 || num_heads <= 0 || num_heads % num_kv_heads || max_blocks <= 0 || max_seq_len <= 0 ||
      (dtype != SSD_DTYPE_BF16 && dtype != SSD_DTYPE_F32))
    return SSD_ERR_INVALID;
  if (B == 0 || (T == 0 && block_tables && seq_lens)) return SSD_OK;  // arrays of nothing may have no address
  if (!block_tables || !seq_lens || !q || !out || (int64_t)max_blocks * block_size < max_seq_len) return SSD_ERR_INVALID;
  if (!kv8_aligned(q) || !kv8_aligned(out) ||
      (int64_t)max_blocks * block_size > 0x7fffffff || max_seq_len > kMaxSeqLen)
    return SSD_ERR_UNSUPPORTED;
  const Kv8Layout L = kv8_layout(dtype == SSD_DTYPE_F32, B, T, num_heads, num_kv_heads, head_dim, max_seq_len);
  if (B > 65535 || L.row_groups > 65535 || num_kv_heads * L.row_groups > 65535)
    return SSD_ERR_UNSUPPORTED;
  if (L.total && (!workspace || workspace_bytes < L.total)) return SSD_ERR_WORKSPACE;
  if (L.total && !kv8_aligned(workspace)) return SSD_ERR_UNSUPPORTED;
  char* w = reinterpret_cast<char*>(workspace);
  Kv8Attn a{};
  a.c = kv8_cache(const_cast<void*>(pages), const_cast<float*>(scales), num_layers, num_blocks, block_size,
                  num_kv_heads, head_dim, layer);
  a.q = q;
  a.out = out;
  a.tables = block_tables;
  a.max_blocks = max_blocks;
  a.seq_lens = seq_lens;
  a.q_lens = q_lens;
  a.scale = scale;
  a.B = B;
  a.T = T;
  a.hq = num_heads;
  a.G = num_heads / num_kv_heads;
  a.row_groups = (int)L.row_groups;
  a.nsplit = L.nsplit;
  a.split = L.split;
  a.polls = wait_polls.load(std::memory_order_relaxed);
  a.ws_o = reinterpret_cast<float*>(w);
  a.ws_ml = reinterpret_cast<float4*>(w + L.off_ml);
  a.plan = L.planned ? reinterpret_cast<int2*>(w + L.off_plan) : nullptr;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == SSD_DTYPE_BF16) {
    if (head_dim == 256) return launch_bf16<256>(st, a, L, B);
    if (head_dim == 128) return launch_bf16<128>(st, a, L, B);
    return launch_bf16<64>(st, a, L, B);
  }
  if (head_dim == 256) return launch_cc<256>(st, a, B);
  if (head_dim == 128) return launch_cc<128>(st, a, B);
  return launch_cc<64>(st, a, B);
}

extern "C" int ssd_kv8_attention_status(ssd_stream_t stream) {
  cudaStream_t st = (cudaStream_t)stream;
  uint32_t gave_up = 0;
  bool ok = cudaMemcpyFromSymbolAsync(&gave_up, many::gave_up, sizeof(gave_up), 0, cudaMemcpyDeviceToHost, st) ==
                cudaSuccess &&
            cudaStreamSynchronize(st) == cudaSuccess;
  if (ok && gave_up) {
    const uint32_t none = 0;
    ok = cudaMemcpyToSymbolAsync(many::gave_up, &none, sizeof(none), 0, cudaMemcpyHostToDevice, st) == cudaSuccess &&
         cudaStreamSynchronize(st) == cudaSuccess;
  }
  if (!ok) {
    (void)cudaGetLastError();
    return SSD_ERR_LAUNCH;
  }
  return gave_up ? SSD_ERR_TIMEOUT : SSD_OK;
}

extern "C" int ssd_kv8_attention_set_polls(int polls) {
  if (polls < -1) return SSD_ERR_INVALID;
  wait_polls.store(polls < 0 ? many::kPolls : (uint32_t)polls, std::memory_order_relaxed);
  return SSD_OK;
}
