// Beam search's selection: of W beams of each request and a vocabulary of V, the W best continuations.
//
// With lse_w = log sum_v e^x[w][v] a live beam w offers every token v at score s = scores[w] + x[w][v] - lse_w, ranked
// by s / (lengths[w] + 1)^alpha; a finished beam offers itself, at its score and lengths[w]^alpha.  Within a beam
// candidates are in the order of x (one length, one lse), so no score is computed but of the few that can win.
//
//   rows kernel   a CTA holds a slice of one beam's logits in registers: its maximum and sum of exponentials, and its W
//                 largest logits.  One pass over the data; beams that offer one candidate or none are not read.
//   merge kernel  a CTA a request: the slices' statistics become lse_w, the slices' candidates are ranked in 64
//                 bits, the W best are written in order.
// The W largest of a CTA: the maxima of 32 groups of threads, the W-th largest of these as a bound that at least W values
// reach (and seldom more than a few times W), those values to shared memory, and each one's rank by counting the
// larger ones.  Where more values reach the bound than fit (long runs of equal logits, sorted rows), W rounds of a
// maximum over the CTA.  Order never depends on which thread comes first: equal values rank by their index.
#include "tcgen05.cuh"

namespace ssd {
namespace {

constexpr int kMaxBeams = 32;
constexpr int kRowThreads = 256, kMergeThreads = 512;
constexpr int kList = 256;             // candidates that reach the bound
constexpr unsigned kAll = 0xffffffffu;

// Lane's rank among the warp's 32 values (largest first, lower lanes before equal ones).
template <typename T>
__device__ __forceinline__ int lane_rank(T v) {
  const int lane = threadIdx.x & 31;
  int rank = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const T o = __shfl_sync(kAll, v, i);
    rank += o > v || (o == v && i < lane);
  }
  return rank;
}

// The W-th largest of the maxima of 32 groups of THREADS / 32 threads, for every thread; `maxima` and `bound` are shared
// memory.
template <int THREADS, typename T>
__device__ __forceinline__ T select_bound(T mine, int W, T* maxima, T* bound) {
  constexpr int N = THREADS / 32;
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) {
    const T y = __shfl_xor_sync(kAll, mine, o);
    mine = y > mine ? y : mine;
  }
  if (threadIdx.x % N == 0) maxima[threadIdx.x / N] = mine;
  __syncthreads();
  if (threadIdx.x < 32) {
    const T v = maxima[threadIdx.x];
    if (lane_rank(v) == W - 1) *bound = v;
  }
  __syncthreads();
  return *bound;
}

// Zeros of either sign are one value.
__device__ __forceinline__ unsigned long long logit_key(float x, uint32_t i) { return argmax_key(x + 0.f, i); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;

struct BeamRows {
  const float* logits;
  int64_t ld;
  const float* scores;
  const uint8_t* finished;
  int W, V, slices;
  float2* stats;                 // [row][slice] maximum, sum of e^(x - maximum)
  unsigned long long* keys;      // [row][slice][W] argmax_key, largest first; 0: none
};

__device__ __forceinline__ bool reads_logits(const float* scores, const uint8_t* finished, int row) {
  return ld_act(scores + row) > -INFINITY && !(finished && ld_act(finished + row));
}

template <int ITEMS, bool VEC>
__global__ void __launch_bounds__(kRowThreads, 4) beam_rows_kernel(const BeamRows a) {
  __shared__ unsigned long long list[kList];
  __shared__ float maxima[32];
  __shared__ float2 ms[kRowThreads / 32];
  __shared__ float bound_s;
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slice = blockIdx.x, row = blockIdx.y;
  pdl_wait();
  pdl_trigger();
  if (!reads_logits(a.scores, a.finished, row)) return;
  const int v0 = slice * (ITEMS * kRowThreads), n = min(ITEMS * kRowThreads, a.V - v0);
  const float* x = a.logits + row * a.ld + v0;
  float v[ITEMS];
  auto index = [&](int i) { return VEC ? ((i >> 2) * kRowThreads + tid) * 4 + (i & 3) : i * kRowThreads + tid; };
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < ITEMS; i += 4) {
      uint4 u = make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u);
      if (index(i) < n) u = ld_act_v4(x + index(i));  // n is a multiple of 4
      v[i] = __uint_as_float(u.x);
      v[i + 1] = __uint_as_float(u.y);
      v[i + 2] = __uint_as_float(u.z);
      v[i + 3] = __uint_as_float(u.w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) v[i] = index(i) < n ? ld_act(x + index(i)) : -INFINITY;
  }
  if (tid == 0) count = 0;
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) m = fmaxf(m, v[i]);
  const float t = select_bound<kRowThreads>(m, a.W, maxima, &bound_s);
  // statistics: the thread's own maximum as reference, 0 where nothing is left of its part.  e^(x - m) as 2^((x - m) log2 e):
  // the difference first, which is exact where it counts.
  const float ref = m == -INFINITY ? 0.f : m;
  {
    float2 s2 = make_float2(0.f, 0.f);
    const float2 l2 = make_float2(kLog2e, kLog2e), r2 = make_float2(-ref, -ref), none = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < ITEMS; i += 2) {
      const float2 e = tc::fma2(tc::add2(make_float2(v[i], v[i + 1]), r2), l2, none);
      s2 = tc::add2(s2, make_float2(ex2(e.x), ex2(e.y)));
    }
    const float s = s2.x + s2.y;
    const float M = warp_max(m), R = M == -INFINITY ? 0.f : M;
    const float S = warp_sum(m == -INFINITY ? s : s * ex2((m - R) * kLog2e));
    if (lane == 0) ms[warp] = make_float2(M, S);
  }
  const float least = fmaxf(t, -3.402823466e38f);  // -inf is never taken
  if (m >= least) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (v[i] >= least) {
        const int at = atomicAdd(&count, 1);
        if (at < kList) list[at] = logit_key(v[i], (uint32_t)(v0 + index(i)));
      }
    }
  }
  __syncthreads();
  const int64_t out = (int64_t)row * a.slices + slice;
  if (warp == 0) {
    const float2 w = lane < kRowThreads / 32 ? ms[lane] : make_float2(-INFINITY, 0.f);
    const float M = warp_max(w.x), R = M == -INFINITY ? 0.f : M;
    const float S = warp_sum(w.x == -INFINITY ? w.y : w.y * ex2((w.x - R) * kLog2e));
    if (lane == 0) a.stats[out] = make_float2(M, S);
  }
  unsigned long long* keys = a.keys + out * a.W;
  const int found = count;
  if (found <= kList) {
    if (tid < found) {
      const unsigned long long mine = list[tid];
      int rank = 0;
      for (int i = 0; i < found; ++i) rank += list[i] > mine;
      if (rank < a.W) keys[rank] = mine;
    }
    if (tid >= found && tid < a.W) keys[tid] = 0;
    return;
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < a.W; ++k) {
    unsigned long long best = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (!(v[i] > -INFINITY)) continue;
      const unsigned long long key = logit_key(v[i], (uint32_t)(v0 + index(i)));
      if (key < last && key > best) best = key;
    }
    best = block_reduce(best, list, OpMax());
    if (tid == 0) keys[k] = best;
    if (best == 0) {
      for (int i = k + 1 + tid; i < a.W; i += kRowThreads) keys[i] = 0;
      return;
    }
    last = best;
  }
}

struct BeamMerge {
  BeamRows r;
  const int32_t* lengths;
  int eos;
  double alpha;
  float* out_scores;
  int32_t *out_parents, *out_tokens, *out_lengths;
  uint8_t* out_finished;
};

// A candidate by its rank (as ordered bits, larger is better) and flat index w V + v (smaller is better).
struct Cand {
  unsigned long long key;
  uint32_t flat;
};
__device__ __forceinline__ unsigned long long double_key(double x) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(x);
  return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ bool better(unsigned long long ka, uint32_t fa, unsigned long long kb, uint32_t fb) {
  return ka > kb || (ka == kb && fa < fb);
}

__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const BeamMerge a) {
  __shared__ unsigned long long maxima[32], bound_s;
  __shared__ unsigned long long list_k[kList];
  __shared__ uint32_t list_f[kList];
  __shared__ double lse[kMaxBeams], base[kMaxBeams], inv[kMaxBeams];
  __shared__ int kind[kMaxBeams];  // 0: offers nothing, 1: its tokens, 2: itself
  __shared__ int count;
  __shared__ unsigned long long red_k[kMergeThreads / 32];
  __shared__ uint32_t red_f[kMergeThreads / 32];
  const BeamRows& r = a.r;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = blockIdx.x, W = r.W;
  pdl_wait();
  for (int w = warp; w < W; w += kMergeThreads / 32) {
    const int row = g * W + w;
    const float sc = ld_act(r.scores + row);
    const bool done = r.finished && ld_act(r.finished + row);
    const int len = a.lengths ? ld_act(a.lengths + row) : 0;
    const int k = sc > -INFINITY ? (done ? 2 : 1) : 0;
    double l = 0.0;
    if (k == 1) {
      const float2* st = r.stats + (int64_t)row * r.slices;
      float M = -INFINITY;
      for (int i = lane; i < r.slices; i += 32) M = fmaxf(M, __ldcg(st + i).x);
      M = warp_max(M);
      const float R = M == -INFINITY ? 0.f : M;
      double S = 0.0;
      for (int i = lane; i < r.slices; i += 32) {
        const float2 y = __ldcg(st + i);
        S += y.x == -INFINITY ? (double)y.y : (double)y.y * exp((double)y.x - (double)R);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) S += __shfl_xor_sync(kAll, S, o);
      l = (double)R + log(S);
    }
    if (lane == 0) {
      lse[w] = l;
      base[w] = sc;
      kind[w] = k;
      inv[w] = a.alpha == 0.0 ? 1.0 : pow((double)(k == 2 ? max(len, 1) : len + 1), -a.alpha);
    }
  }
  if (tid == 0) count = 0;
  __syncthreads();
  // A beam's candidates go to T threads of the CTA, the first of them also standing for a finished beam.
  const int per = r.slices * W;
  int shift = 9;  // log2 of T
  while (kMergeThreads >> shift < W) --shift;
  const int w = tid >> shift, i0 = tid & ((1 << shift) - 1), step = 1 << shift;
  const int mine = w < W ? kind[w] : 0;
  auto cand = [&](unsigned long long key) {
    Cand c{0, 0xffffffffu};
    if (key == 0) return c;
    const uint32_t token = argmax_key_index(key);
    const double rank = (base[w] + ((double)argmax_key_value(key) - lse[w])) * inv[w];
    if (!(rank > -INFINITY)) return c;  // NaN too
    c.key = double_key(rank + 0.0);
    c.flat = (uint32_t)w * (uint32_t)r.V + token;
    return c;
  };
  const unsigned long long* keys = r.keys + ((int64_t)g * W + w) * per;
  Cand self{0, 0xffffffffu};
  if (mine == 2 && i0 == 0) {
    const double rank = base[w] * inv[w];
    if (rank > -INFINITY) self = Cand{double_key(rank + 0.0), (uint32_t)w * (uint32_t)r.V + (uint32_t)a.eos};
  }
  // the thread's first candidates stay in registers
  constexpr int HELD = 4;
  Cand held[HELD];
  unsigned long long best = self.key, raw[HELD];
#pragma unroll
  for (int k = 0; k < HELD; ++k) {
    const int i = i0 + k * step;
    raw[k] = mine == 1 && i < per ? __ldcg(keys + i) : 0;
  }
#pragma unroll
  for (int k = 0; k < HELD; ++k) {
    held[k] = cand(raw[k]);
    best = max(best, held[k].key);
  }
  const int more = mine == 1 ? per : 0;
  for (int i = i0 + HELD * step; i < more; i += step) best = max(best, cand(__ldcg(keys + i)).key);
  const unsigned long long t = select_bound<kMergeThreads>(best, W, maxima, &bound_s);
  auto take = [&](const Cand& c) {
    if (c.key == 0 || c.key < t) return;
    const int at = atomicAdd(&count, 1);
    if (at < kList) {
      list_k[at] = c.key;
      list_f[at] = c.flat;
    }
  };
  if (best >= t) {
    take(self);
#pragma unroll
    for (int k = 0; k < HELD; ++k) take(held[k]);
    for (int i = i0 + HELD * step; i < more; i += step) take(cand(__ldcg(keys + i)));
  }
  __syncthreads();
  auto put = [&](int k, unsigned long long key, uint32_t flat) {
    const int at = g * W + k;
    float score = -INFINITY;
    int parent = -1, token = -1, len = 0, fin = 1;
    if (key != 0) {
      parent = (int)(flat / (uint32_t)r.V);
      token = (int)(flat - (uint32_t)parent * (uint32_t)r.V);
      const int before = a.lengths ? ld_act(a.lengths + g * W + parent) : 0;
      if (kind[parent] == 2) {
        score = (float)base[parent];
        len = before;
      } else {
        const float x = ld_act(r.logits + (int64_t)(g * W + parent) * r.ld + token);
        score = (float)(base[parent] + ((double)x - lse[parent]));
        len = before + 1;
        fin = token == a.eos;
      }
    }
    a.out_scores[at] = score;
    a.out_parents[at] = parent;
    a.out_tokens[at] = token;
    if (a.out_lengths) a.out_lengths[at] = len;
    if (a.out_finished) a.out_finished[at] = (uint8_t)fin;
  };
  const int found = count;
  if (found <= kList) {
    if (tid < found) {
      const unsigned long long key = list_k[tid];
      const uint32_t flat = list_f[tid];
      int rank = 0;
      for (int i = 0; i < found; ++i) rank += better(list_k[i], list_f[i], key, flat);
      if (rank < W) put(rank, key, flat);
    }
    if (tid >= found && tid < W) put(tid, 0, 0);
  } else {
    unsigned long long last_k = ~0ull;
    uint32_t last_f = 0;
    for (int k = 0; k < W; ++k) {
      unsigned long long bk = 0;
      uint32_t bf = 0xffffffffu;
      auto next = [&](const Cand& c) {
        if (c.key != 0 && better(last_k, last_f, c.key, c.flat) && better(c.key, c.flat, bk, bf)) {
          bk = c.key;
          bf = c.flat;
        }
      };
      next(self);
      for (int i = i0; i < more; i += step) next(cand(__ldcg(keys + i)));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long ok = __shfl_xor_sync(kAll, bk, o);
        const uint32_t of = __shfl_xor_sync(kAll, bf, o);
        if (better(ok, of, bk, bf)) { bk = ok; bf = of; }
      }
      __syncthreads();
      if (lane == 0) { red_k[warp] = bk; red_f[warp] = bf; }
      __syncthreads();
      for (int i = 0; i < kMergeThreads / 32; ++i)
        if (better(red_k[i], red_f[i], bk, bf)) { bk = red_k[i]; bf = red_f[i]; }
      if (tid == 0) put(k, bk, bf);
      last_k = bk;
      last_f = bf;
    }
  }
  pdl_trigger();
}

constexpr int kFewItems = 16, kManyItems = 32;

struct BeamLayout {
  int items, slices;
  size_t off_keys, total;
};

BeamLayout beam_layout(int G, int W, int V) {
  BeamLayout L;
  const int64_t rows = (int64_t)G * W;
  L.items = rows * ((V + kManyItems * kRowThreads - 1) / (kManyItems * kRowThreads)) >= 2 * 148 ? kManyItems : kFewItems;
  L.slices = (V + L.items * kRowThreads - 1) / (L.items * kRowThreads);
  L.off_keys = (sizeof(float2) * (size_t)rows * L.slices + 255) & ~size_t(255);
  L.total = L.off_keys + sizeof(unsigned long long) * (size_t)rows * L.slices * W;
  return L;
}

bool beam_sizes_ok(int G, int W, int V) {
  return G >= 0 && W >= 1 && V >= 1;
}

}  // namespace
}  // namespace ssd

using namespace ssd;

extern "C" size_t ssd_beam_select_workspace_size(int G, int W, int V) {
  if (!beam_sizes_ok(G, W, V) || G == 0 || W > kMaxBeams) return 0;
  return beam_layout(G, W, V).total;
}

extern "C" int ssd_beam_select(ssd_stream_t stream, const float* logits, int64_t ld, const float* scores,
                               const int32_t* lengths, const uint8_t* finished, int eos, float length_penalty,
                               float* out_scores, int32_t* out_parents, int32_t* out_tokens, int32_t* out_lengths,
                               uint8_t* out_finished, void* workspace, size_t workspace_bytes, int G, int W, int V) {
  if (!beam_sizes_ok(G, W, V) || ld < V || eos < -1 || eos >= V || (finished && eos < 0) ||
      !(length_penalty == length_penalty) || (length_penalty != 0.f && !lengths))
    return SSD_ERR_INVALID;
  if (G == 0) return SSD_OK;
  if (!logits || !scores || !out_scores || !out_parents || !out_tokens) return SSD_ERR_INVALID;
  if (W > kMaxBeams || (int64_t)G * W > 65535 || V > (1 << 27) - 1) return SSD_ERR_UNSUPPORTED;
  const BeamLayout L = beam_layout(G, W, V);
  if (!workspace || workspace_bytes < L.total) return SSD_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return SSD_ERR_UNSUPPORTED;
  char* w = reinterpret_cast<char*>(workspace);
  BeamRows r{logits, ld, scores, finished, W, V, L.slices, reinterpret_cast<float2*>(w),
             reinterpret_cast<unsigned long long*>(w + L.off_keys)};
  const dim3 grid(L.slices, G * W);
  const bool vec = !(reinterpret_cast<uintptr_t>(logits) & 15) && ld % 4 == 0 && V % 4 == 0;
  if (L.items == kManyItems) {
    if (vec) SSD_PDL((beam_rows_kernel<kManyItems, true>), grid, kRowThreads, 0, stream, r);
    else SSD_PDL((beam_rows_kernel<kManyItems, false>), grid, kRowThreads, 0, stream, r);
  } else {
    if (vec) SSD_PDL((beam_rows_kernel<kFewItems, true>), grid, kRowThreads, 0, stream, r);
    else SSD_PDL((beam_rows_kernel<kFewItems, false>), grid, kRowThreads, 0, stream, r);
  }
  const BeamMerge m{r, lengths, eos, (double)length_penalty, out_scores, out_parents, out_tokens, out_lengths,
                    out_finished};
  SSD_PDL(beam_merge_kernel, G, kMergeThreads, 0, stream, m);
  return SSD_OK;
}
