// Attention over the 8-bit paged KV cache.
//
// For query row r at position P_r (token t of sequence b sits at seq_lens[b] - q_lens[b] + t) and the
// positions j <= P_r of its sequence, with K_j = k_j 2^a(j), V_j = v_j 2^c(j) (a, c: scale exponents of j's
// page and head):
//   s_j = scale * 2^a(j) * (q_r . k_j),   out_r = sum_j e^(s_j - M) 2^c(j) v_j / sum_j e^(s_j - M).
// Rows past q_lens[b] and rows that see no position are zeros.
//
// A CTA owns one KV head of one sequence, a fixed slice of its positions (a split) and a group of query rows
// (G query heads times the new tokens), so a query's result does not depend on how many rows stand beside it.
// Splits leave unnormalised partials, which a second kernel joins in split order.  It needs no counters, so a
// workspace holds nothing between calls and may come uninitialised from any allocator.
#include <float.h>

#include "kv8.cuh"

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
  int T, hq, G, row_groups, nsplit;
  float* ws_o;          // [group][split][rows][D]
  float4* ws_ml;        // [group][split][rows]: maximum that o is relative to, that l is relative to, l
};

// Splits of a sequence that hold positions (at least one, which writes its zero rows).
__device__ __forceinline__ int splits_of(int seq, int split) { return max(1, (seq + split - 1) / split); }

// out = sum_s e^(m_s - M) o_s / sum_s e^(n_s - N) l_s * e^(M - N), M and N the largest m_s and n_s; one warp per
// query row, lanes over the head dims.  LOG2: the maxima are in powers of two.
template <typename T, int D, int R, int SPLIT, bool LOG2>
__global__ void __launch_bounds__(128) kv8_join_kernel(const Kv8Attn a, int64_t rows) {
  constexpr int DPL = D / 32;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int64_t x = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (x >= rows) return;
  const int r = (int)(x % R);
  const int64_t grp = x / R;
  const int rg = (int)(grp % a.row_groups), head = (int)(grp / a.row_groups % a.c.hkv);
  const int b = (int)(grp / a.row_groups / a.c.hkv);
  const int gr = rg * R + r, t = gr / a.G, g = gr % a.G;
  if (t >= a.T) return;
  const int seq_full = a.seq_lens[b];
  const int seq = min(min(seq_full, a.max_blocks * a.c.block_size), a.nsplit * SPLIT);
  const int ql = a.q_lens ? min(max(a.q_lens[b], 0), a.T) : a.T;
  const int ns = splits_of(seq, SPLIT);
  auto ex = [](float v) { return LOG2 ? exp2f(v) : expf(v); };
  const float4* ml = a.ws_ml + grp * a.nsplit * R + r;
  float M = -INFINITY, N = -INFINITY;
  for (int s = lane; s < ns; s += 32) {
    const float4 v = __ldcg(ml + (int64_t)s * R);
    M = fmaxf(M, v.x);
    N = fmaxf(N, v.y);
  }
  M = warp_max(M);
  N = warp_max(N);
  float L = 0.f;
  for (int s = lane; s < ns; s += 32) {
    const float4 v = __ldcg(ml + (int64_t)s * R);
    if (v.y != -INFINITY) L += v.z * ex(v.y - N);
  }
  L = warp_sum(L);
  float o[DPL];
#pragma unroll
  for (int i = 0; i < DPL; ++i) o[i] = 0.f;
  const float* po = a.ws_o + (grp * a.nsplit * R + r) * D + lane;
  if (t < ql && L != 0.f) {  // L is NaN, not 0, where a seen score is
#pragma unroll 4
    for (int s = 0; s < ns; ++s) {
      const float m = __ldcg(ml + (int64_t)s * R).x;
      if (m == -INFINITY) continue;
      const float f = ex(m - M);
#pragma unroll
      for (int i = 0; i < DPL; ++i) o[i] = fmaf(f, __ldcg(po + (int64_t)s * R * D + i * 32), o[i]);
    }
    const float f = ex(M - N);
#pragma unroll
    for (int i = 0; i < DPL; ++i) o[i] = o[i] / L * f;
  }
  T* out = reinterpret_cast<T*>(a.out) + (((int64_t)b * a.T + t) * a.hq + head * a.G + g) * D + lane;
#pragma unroll
  for (int i = 0; i < DPL; ++i) out[i * 32] = from_f<T>(o[i]);
}

template <typename T, int D, int R, int SPLIT, bool LOG2>
int launch_join(cudaStream_t st, const Kv8Attn& a, int B) {
  const int64_t rows = (int64_t)B * a.c.hkv * a.row_groups * R;
  SSD_PDL((kv8_join_kernel<T, D, R, SPLIT, LOG2>), (unsigned)((rows + 3) / 4), 128, 0, st, a, rows);
  return SSD_OK;
}

// ------------------------------------------------------------------ CUDA-core kernel (fp32 models)
// fp32 queries keep fp32 products: a warp walks its positions one by one with the running maximum and sum
// of each row, lanes over the head dims.  Used for the fp32 (toy) models, whose forward takes at most 16 rows.
constexpr int kCcRows = 8;
constexpr int kCcSplit = 128;
constexpr int kCcWarps = 4;

template <int N>
__device__ __forceinline__ void load_e4m3(const uint8_t* p, float* f) {
  if constexpr (N == 8) {
    const uint2 w = __ldcg(reinterpret_cast<const uint2*>(p));
    const float2 a = e4m3_pair(w.x), b = e4m3_pair(w.x >> 16), c = e4m3_pair(w.y), d = e4m3_pair(w.y >> 16);
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y; f[4] = c.x; f[5] = c.y; f[6] = d.x; f[7] = d.y;
  } else if constexpr (N == 4) {
    const uint32_t w = __ldcg(reinterpret_cast<const uint32_t*>(p));
    const float2 a = e4m3_pair(w), b = e4m3_pair(w >> 16);
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
  } else {
    const float2 a = e4m3_pair(__ldcg(reinterpret_cast<const uint16_t*>(p)));
    f[0] = a.x; f[1] = a.y;
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kCcWarps * 32) kv8_attention_cc_kernel(const Kv8Attn a) {
  constexpr int DPL = D / 32;
  __shared__ float qs[kCcRows][D];
  __shared__ float os[kCcWarps][kCcRows][D];
  __shared__ float2 mls[kCcWarps][kCcRows];
  __shared__ int pos_s[kCcRows];
  pdl_wait();
  pdl_trigger();
  const int split = blockIdx.x, b = blockIdx.z;
  const int head = blockIdx.y / a.row_groups, rg = blockIdx.y % a.row_groups;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int seq_full = a.seq_lens[b];
  // positions beyond the table or the split count are never read (a seq_len larger than the caller's bound)
  const int seq = min(min(seq_full, a.max_blocks * a.c.block_size), a.nsplit * kCcSplit);
  const int ql = a.q_lens ? min(max(a.q_lens[b], 0), a.T) : a.T;
  const int row0 = rg * kCcRows;
  const int nrows = min(kCcRows, a.G * a.T - row0);
  const int ns = splits_of(seq, kCcSplit);
  if (split >= ns) return;
  if (tid < kCcRows) {
    const int t = (row0 + tid) / a.G;
    pos_s[tid] = (tid < nrows && t < ql) ? seq_full - ql + t : -1;
  }
  for (int i = tid; i < kCcRows * D; i += blockDim.x) {
    const int r = i / D, d = i % D;
    const int gr = row0 + r, t = gr / a.G, g = gr % a.G;
    qs[r][d] = r < nrows ? to_f(ld_act(reinterpret_cast<const T*>(a.q) +
                                       (((int64_t)b * a.T + t) * a.hq + head * a.G + g) * D + d)) : 0.f;
  }
  __syncthreads();
  float m[kCcRows], l[kCcRows], o[kCcRows][DPL];
#pragma unroll
  for (int r = 0; r < kCcRows; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < DPL; ++i) o[r][i] = 0.f;
  }
  const int k1 = min(seq, (split + 1) * kCcSplit);
  const int32_t* table = a.tables + (int64_t)b * a.max_blocks;
  for (int j = split * kCcSplit + warp; j < k1; j += kCcWarps) {
    const int blk = ld_act(table + j / a.c.block_size);
    if ((unsigned)blk >= (unsigned)a.c.num_blocks) continue;
    const int64_t off = a.c.layer + (((int64_t)blk * a.c.block_size + j % a.c.block_size) * a.c.hkv + head) * D;
    const int64_t so = a.c.scale_layer + (int64_t)blk * a.c.hkv + head;
    const float ks = ld_act(a.c.scales + so), vs = ld_act(a.c.scales + a.c.scale_plane + so);
    float k[DPL], v[DPL];
    load_e4m3<DPL>(a.c.pages + off + lane * DPL, k);
    load_e4m3<DPL>(a.c.pages + a.c.plane + off + lane * DPL, v);
#pragma unroll
    for (int i = 0; i < DPL; ++i) v[i] *= vs;
#pragma unroll
    for (int r = 0; r < kCcRows; ++r) {
      if (pos_s[r] < j) continue;  // the same for every lane
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < DPL; ++i) s = fmaf(qs[r][lane * DPL + i], k[i], s);
      s = warp_sum(s) * ks * a.scale;
      const float mn = fmaxf(m[r], fmaxf(s, -FLT_MAX));  // finite once a position is seen, a NaN score included
      const float f = m[r] == -INFINITY ? 0.f : expf(m[r] - mn), p = expf(s - mn);
      l[r] = l[r] * f + p;
#pragma unroll
      for (int i = 0; i < DPL; ++i) o[r][i] = fmaf(p, v[i], o[r][i] * f);
      m[r] = mn;
    }
  }
#pragma unroll
  for (int r = 0; r < kCcRows; ++r) {
    if (lane == 0) mls[warp][r] = make_float2(m[r], l[r]);
#pragma unroll
    for (int i = 0; i < DPL; ++i) os[warp][r][lane * DPL + i] = o[r][i];
  }
  __syncthreads();
  // join the warps in warp order
  const int64_t grp = ((int64_t)b * a.c.hkv + head) * a.row_groups + rg;
  T* out = reinterpret_cast<T*>(a.out);
  auto out_at = [&](int r, int d) -> T& {
    const int gr = row0 + r, t = gr / a.G, g = gr % a.G;
    return out[(((int64_t)b * a.T + t) * a.hq + head * a.G + g) * D + d];
  };
  for (int i = tid; i < nrows * D; i += blockDim.x) {
    const int r = i / D, d = i % D;
    float M = -INFINITY;
    for (int w = 0; w < kCcWarps; ++w) M = fmaxf(M, mls[w][r].x);
    float O = 0.f, L = 0.f;
    for (int w = 0; w < kCcWarps; ++w) {
      const float f = mls[w][r].x == -INFINITY ? 0.f : expf(mls[w][r].x - M);
      L += mls[w][r].y * f;
      if (f != 0.f) O += os[w][r][d] * f;
    }
    if (a.nsplit == 1) {
      out_at(r, d) = from_f<T>(pos_s[r] >= 0 && L != 0.f ? O / L : 0.f);
    } else {
      a.ws_o[((grp * a.nsplit + split) * kCcRows + r) * D + d] = O;
      if (d == 0) a.ws_ml[(grp * a.nsplit + split) * kCcRows + r] = make_float4(M, M, L, 0.f);
    }
  }
}

struct Kv8Layout {
  int row_groups, nsplit;
  size_t groups, off_o, off_ml, total;
};

inline size_t up256(size_t x) { return (x + 255) & ~size_t(255); }

Kv8Layout kv8_layout(int B, int T, int hq, int hkv, int D, int max_seq_len) {
  Kv8Layout L;
  L.row_groups = (int)(((int64_t)(hq / hkv) * T + kCcRows - 1) / kCcRows);
  L.nsplit = (max_seq_len + kCcSplit - 1) / kCcSplit;
  L.groups = (size_t)B * hkv * L.row_groups;
  const size_t rows = L.groups * L.nsplit * kCcRows;
  L.off_o = 0;
  L.off_ml = L.off_o + up256(sizeof(float) * rows * D);
  L.total = L.off_ml + up256(sizeof(float4) * rows);
  return L;
}

template <typename T, int D>
int launch_cc(cudaStream_t st, const Kv8Attn& a, int B) {
  const dim3 grid(a.nsplit, a.c.hkv * a.row_groups, B);
  SSD_PDL((kv8_attention_cc_kernel<T, D>), grid, kCcWarps * 32, 0, st, a);
  return a.nsplit == 1 ? SSD_OK : launch_join<T, D, kCcRows, kCcSplit, false>(st, a, B);
}

}  // namespace
}  // namespace ssd

using namespace ssd;

extern "C" size_t ssd_kv8_attention_workspace_size(int B, int T, int num_heads, int num_kv_heads, int head_dim,
                                                   int max_seq_len) {
  if (B <= 0 || T <= 0 || num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads || head_dim <= 0 ||
      max_seq_len <= 0)
    return 0;
  return kv8_layout(B, T, num_heads, num_kv_heads, head_dim, max_seq_len).total;
}

extern "C" int ssd_kv8_attention(ssd_stream_t stream, const void* q, const void* pages, const float* scales,
                                 int dtype, int num_layers, int num_blocks, int block_size, int num_kv_heads,
                                 int head_dim, int layer, const int32_t* block_tables, int max_blocks,
                                 const int32_t* seq_lens, const int32_t* q_lens, void* out, float scale, int B, int T,
                                 int num_heads, int max_seq_len, void* workspace, size_t workspace_bytes) {
  if (int rc = kv8_check(pages, scales, num_layers, num_blocks, block_size, num_kv_heads, head_dim, layer)) return rc;
  if (B < 0 || T < 0 || num_heads <= 0 || num_heads % num_kv_heads || max_blocks <= 0 || max_seq_len <= 0 ||
      !block_tables || !seq_lens || (dtype != SSD_DTYPE_BF16 && dtype != SSD_DTYPE_F32))
    return SSD_ERR_INVALID;
  if (B == 0 || T == 0) return SSD_OK;
  if (!q || !out || (int64_t)max_blocks * block_size < max_seq_len) return SSD_ERR_INVALID;
  if (!kv8_aligned(q) || !kv8_aligned(out) || (int64_t)max_blocks * block_size > 0x7fffffff)
    return SSD_ERR_UNSUPPORTED;
  const Kv8Layout L = kv8_layout(B, T, num_heads, num_kv_heads, head_dim, max_seq_len);
  if (B > 65535 || (int64_t)num_kv_heads * L.row_groups > 65535)
    return SSD_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < L.total) return SSD_ERR_WORKSPACE;
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
  a.T = T;
  a.hq = num_heads;
  a.G = num_heads / num_kv_heads;
  a.row_groups = L.row_groups;
  a.nsplit = L.nsplit;
  a.ws_o = reinterpret_cast<float*>(w + L.off_o);
  a.ws_ml = reinterpret_cast<float4*>(w + L.off_ml);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == SSD_DTYPE_BF16) {
    if (head_dim == 256) return launch_cc<bf16, 256>(st, a, B);
    if (head_dim == 128) return launch_cc<bf16, 128>(st, a, B);
    return launch_cc<bf16, 64>(st, a, B);
  }
  if (head_dim == 256) return launch_cc<float, 256>(st, a, B);
  if (head_dim == 128) return launch_cc<float, 128>(st, a, B);
  return launch_cc<float, 64>(st, a, B);
}
