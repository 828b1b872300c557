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
// reach (and of a slice's logits seldom more than a few times W), those values to shared memory, and each one's rank by
// counting the larger ones.  Where more values reach the bound than fit, W rounds of a maximum over the CTA.  Order never
// depends on which thread comes first: equal values rank by their index.
// More than fit are long runs of equal logits in the rows kernel.  In the merge a beam has 512 / W of the threads (W rounded up
// to a power of two), so the bound is as low as the worst beam's best candidate, and there is none where fewer than W
// groups hold a candidate, as at a first step, where one beam is live: all its slices * W candidates are taken then.  From 9
// beams over 256000 tokens on these do not fit, and the rounds, in which 16 or 32 threads read and rank every candidate
// again, make up most of the call: one request's first step takes 12.6 us with 8 beams, 110 with 16, 705 with 32, a
// step in mid-flight (scores within 5 of each other) 9.2, 21 and 950 us.
// Bound by DRAM for many rows: 256 rows of 256000 logits take 51 us, the rows kernel 46 of them (262 MB, 5.7 TB/s), 32
// rows 11.7 us; few rows by the two kernels' chains of reads and barriers: one row of 256000 logits 7 us.
#include <algorithm>

#include "tcgen05.cuh"

namespace ssd {
namespace {

constexpr int kMaxBeams = 32;
constexpr int kRowThreads = 256, kMergeThreads = 512;
constexpr int kList = 256;             // candidates that there is room for
// Logits of a thread.  16: 71 us instead of 51 for 256 rows of 256000, 7.0 instead of 6.6 for one: what a CTA does once, some
// 2 us of it, is worth more than the second wave that small slices save.  Slices fetched ahead into shared memory by CTAs
// that stay (one pass, a running bound) came out at 60 us: the slices' barriers leave less in flight than CTAs that come and go.
constexpr int kItems = 32;
constexpr int kSlice = kItems * kRowThreads;
constexpr unsigned kAll = 0xffffffffu;

// The largest value that at least W of the maxima of 32 groups of THREADS / 32 threads reach; `maxima` is shared memory.
// Every warp finds it for itself, which takes one barrier.
template <int THREADS, typename T>
__device__ __forceinline__ T select_bound(T mine, int W, T* maxima) {
  constexpr int N = THREADS / 32;
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) {
    const T y = __shfl_xor_sync(kAll, mine, o);
    mine = y > mine ? y : mine;
  }
  if (threadIdx.x % N == 0) maxima[threadIdx.x / N] = mine;
  __syncthreads();
  const T v = maxima[threadIdx.x & 31];
  int reach = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) reach += maxima[i] >= v;
  const int least = __reduce_min_sync(kAll, reach >= W ? reach : 33);
  return __shfl_sync(kAll, v, __ffs(__ballot_sync(kAll, reach == least)) - 1);
}

// Zeros of either sign are one value.
__device__ __forceinline__ unsigned long long logit_key(float x, uint32_t i) { return argmax_key(x + 0.f, i); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;

// What a sum of e^(x - m) is worth relative to M >= m (not both -inf).  e^(x - m) as 2^((x - m) log2 e): the difference first,
// which is exact where it counts.
__device__ __forceinline__ float to_larger(float m, float M) { return ex2((m - M) * kLog2e); }

struct BeamRows {
  const float* logits;
  int64_t ld;
  const float* scores;
  const uint8_t* finished;
  int W, V, slices;              // slices of a row
  float2* stats;                 // [row][slice] maximum, sum of e^(x - maximum)
  unsigned long long* keys;      // [row][slice][W] argmax_key, largest first; 0: none
};

__device__ __forceinline__ bool reads_logits(const float* scores, const uint8_t* finished, int row) {
  const float score = ld_act(scores + row);
  const uint8_t done = finished ? ld_act(finished + row) : 0;  // (both loads at once)
  return score > -INFINITY && !done;
}

struct RowShared {
  unsigned long long list[kList];  // candidates of the part so far
  unsigned long long red[32];
  float maxima[32];
  float sums[kRowThreads / 32];
  int count;
};

// More of a slice reaches its bound than there is room for (runs of equal logits): the W best, one after another.  The logits
// are read again.  Returns how many there are.
__device__ __noinline__ int crowded(RowShared& sh, const float* x, int n, int v0, int W) {
  unsigned long long last = ~0ull;
  int found = 0;
#pragma unroll 1
  for (; found < W; ++found) {
    unsigned long long best = 0;
#pragma unroll 1
    for (int i = threadIdx.x; i < n; i += kRowThreads) {
      const float y = ld_act(x + i);
      const unsigned long long key = logit_key(y, (uint32_t)(v0 + i));
      if (y > -INFINITY && key < last && key > best) best = key;
    }
    best = block_reduce(best, sh.red, OpMax());
    if (best == 0) break;
    if (threadIdx.x == 0) sh.list[found] = best;
    last = best;
  }
  __syncthreads();
  return found;
}

// VEC: 16 bytes a load, where the rows' alignment allows it (256 rows of 256000 logits 53 us, of 255999 58).  Five CTAs an
// SM (48 registers): 51 us, four 56, six 52.
template <bool VEC>
__global__ void __launch_bounds__(kRowThreads, 5) beam_rows_kernel(const BeamRows a) {
  __shared__ RowShared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slice = blockIdx.x, row = blockIdx.y;
  pdl_wait();
  pdl_trigger();
  if (!reads_logits(a.scores, a.finished, row)) return;
  const int v0 = slice * kSlice, n = min(kSlice, a.V - v0);
  const float* x = a.logits + row * a.ld + v0;
  auto at = [&](int i) { return VEC ? ((i >> 2) * kRowThreads + tid) * 4 + (i & 3) : i * kRowThreads + tid; };
  float v[kItems];
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < kItems; i += 4) {
      uint4 u = make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u);
      if (at(i) < n) u = ld_act_v4(x + at(i));  // n is a multiple of 4
      v[i] = __uint_as_float(u.x);
      v[i + 1] = __uint_as_float(u.y);
      v[i + 2] = __uint_as_float(u.z);
      v[i + 3] = __uint_as_float(u.w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kItems; ++i) v[i] = at(i) < n ? ld_act(x + at(i)) : -INFINITY;
  }
  if (tid == 0) sh.count = 0;
  float m = -INFINITY, most[kItems / 8];
#pragma unroll
  for (int k = 0; k < kItems / 8; ++k) {
    most[k] = v[8 * k];
#pragma unroll
    for (int i = 1; i < 8; ++i) most[k] = fmaxf(most[k], v[8 * k + i]);
    m = fmaxf(m, most[k]);  // (NaN counts as -inf)
  }
  const float bound = fmaxf(select_bound<kRowThreads>(m, a.W, sh.maxima), -3.402823466e38f);  // -inf is never taken
  if (m >= bound) {
#pragma unroll
    for (int k = 0; k < kItems / 8; ++k) {
      if (!(most[k] >= bound)) continue;
#pragma unroll
      for (int i = 8 * k; i < 8 * k + 8; ++i) {
        if (v[i] >= bound) {
          const int place = atomicAdd(&sh.count, 1);
          if (place < kList) sh.list[place] = logit_key(v[i], (uint32_t)(v0 + at(i)));
        }
      }
    }
  }
  // the thread's sum, relative to its maximum (0 where nothing is left of its part)
  const float ref = m == -INFINITY ? 0.f : m;
  float2 s2 = make_float2(0.f, 0.f);
  {
    const float2 l2 = make_float2(kLog2e, kLog2e), r2 = make_float2(-ref, -ref), none = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kItems; i += 2) {
      const float2 e = tc::fma2(tc::add2(make_float2(v[i], v[i + 1]), r2), l2, none);
      s2 = tc::add2(s2, make_float2(ex2(e.x), ex2(e.y)));
    }
  }
  __syncthreads();
  // the candidates in order, and the sums relative to the largest of them
  int found = sh.count;
  if (found > kList) found = crowded(sh, x, n, v0, a.W);
  unsigned long long* keys = a.keys + ((int64_t)row * a.slices + slice) * a.W;
  if (tid < found) {
    const unsigned long long mine = sh.list[tid];
    int rank = 0;
#pragma unroll 4
    for (int i = 0; i < found; ++i) rank += sh.list[i] > mine;
    if (rank < a.W) keys[rank] = mine;
  }
  if (tid >= found && tid < a.W) keys[tid] = 0;
  const float M = key_float(__reduce_max_sync(kAll, float_key(sh.maxima[lane])));
  const float S = warp_sum(m == -INFINITY ? s2.x + s2.y : (s2.x + s2.y) * to_larger(m, M));
  if (lane == 0) sh.sums[warp] = S;
  __syncthreads();
  if (tid == 0) {
    float total = sh.sums[0];
#pragma unroll
    for (int i = 1; i < kRowThreads / 32; ++i) total += sh.sums[i];
    a.stats[(int64_t)row * a.slices + slice] = make_float2(M, total);
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

// A CTA a request: bound by latency, of the fp64 logarithms and powers and a handful of barriers (some 4 us; 32 requests of 8
// beams, 2048 candidates each, 5 us).
__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const BeamMerge a) {
  __shared__ unsigned long long maxima[32];
  __shared__ unsigned long long list_k[kList];
  __shared__ uint32_t list_f[kList];
  __shared__ float list_x[kList];
  __shared__ double lse[kMaxBeams], base[kMaxBeams], inv[kMaxBeams];
  __shared__ int kind[kMaxBeams], len_s[kMaxBeams];  // 0: offers nothing, 1: its tokens, 2: itself
  __shared__ int count;
  __shared__ unsigned long long red_k[kMergeThreads / 32];
  __shared__ uint32_t red_f[kMergeThreads / 32];
  const BeamRows& r = a.r;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = blockIdx.x, W = r.W;
  pdl_wait();
  pdl_trigger();
  // two tasks a beam, a warp each: log sum e^x, and length^-alpha
  for (int task = warp; task < 2 * W; task += kMergeThreads / 32) {
    const int w = task < W ? task : task - W, row = g * W + w;
    const float sc = ld_act(r.scores + row);
    const bool done = r.finished && ld_act(r.finished + row);
    const int k = sc > -INFINITY ? (done ? 2 : 1) : 0;
    if (task >= W) {
      const int len = a.lengths ? ld_act(a.lengths + row) : 0;
      const double y = a.alpha == 0.0 ? 1.0 : pow((double)(k == 2 ? max(len, 1) : len + 1), -a.alpha);
      if (lane == 0) {
        inv[w] = y;
        len_s[w] = len;
      }
      continue;
    }
    double l = 0.0;
    if (k == 1) {
      const float2* st = r.stats + (int64_t)row * r.slices;
      const int n = r.slices;
      float M = -INFINITY;
      for (int i = lane; i < n; i += 32) M = fmaxf(M, __ldcg(st + i).x);
      M = warp_max(M);
      double S = 0.0;
      for (int i = lane; i < n; i += 32) {
        const float2 y = __ldcg(st + i);
        S += (double)(y.x == -INFINITY ? y.y : y.y * to_larger(y.x, M));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) S += __shfl_xor_sync(kAll, S, o);
      l = (M == -INFINITY ? 0.0 : (double)M) + log(S);
    }
    if (lane == 0) {
      lse[w] = l;
      base[w] = sc;
      kind[w] = k;
    }
  }
  if (tid == 0) count = 0;
  __syncthreads();
  // A beam's candidates go to T threads of the CTA, the first of them also standing for a finished beam.
  int shift = 9;  // log2 of T
  while (kMergeThreads >> shift < W) --shift;
  const int w = tid >> shift, i0 = tid & ((1 << shift) - 1), step = 1 << shift;
  const int mine = w < W ? kind[w] : 0, per = mine == 1 ? r.slices * W : 0;
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
  const unsigned long long* keys = r.keys + ((int64_t)g * W + w) * r.slices * W;
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
    raw[k] = i < per ? __ldcg(keys + i) : 0;
  }
#pragma unroll
  for (int k = 0; k < HELD; ++k) {
    held[k] = cand(raw[k]);
    best = max(best, held[k].key);
  }
  for (int i = i0 + HELD * step; i < per; i += step) best = max(best, cand(__ldcg(keys + i)).key);
  const unsigned long long t = select_bound<kMergeThreads>(best, W, maxima);
  auto take = [&](const Cand& c, float x) {
    if (c.key == 0 || c.key < t) return;
    const int at = atomicAdd(&count, 1);
    if (at < kList) {
      list_k[at] = c.key;
      list_f[at] = c.flat;
      list_x[at] = x;
    }
  };
  if (best >= t) {
    take(self, 0.f);
#pragma unroll
    for (int k = 0; k < HELD; ++k) take(held[k], argmax_key_value(raw[k]));
    for (int i = i0 + HELD * step; i < per; i += step) {
      const unsigned long long key = __ldcg(keys + i);
      take(cand(key), argmax_key_value(key));
    }
  }
  __syncthreads();
  auto put = [&](int k, unsigned long long key, uint32_t flat, float x) {
    const int at = g * W + k;
    float score = -INFINITY;
    int parent = -1, token = -1, len = 0, fin = 1;
    if (key != 0) {
      parent = (int)(flat / (uint32_t)r.V);
      token = (int)(flat - (uint32_t)parent * (uint32_t)r.V);
      const int before = len_s[parent];
      if (kind[parent] == 2) {
        score = (float)base[parent];
        len = before;
      } else {
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
      if (rank < W) put(rank, key, flat, list_x[tid]);
    }
    if (tid >= found && tid < W) put(tid, 0, 0, 0.f);
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
      for (int i = i0; i < per; i += step) next(cand(__ldcg(keys + i)));
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
      if (tid == 0) {
        const uint32_t parent = bf / (uint32_t)r.V;
        put(k, bk, bf, bk ? ld_act(r.logits + (int64_t)(g * W + parent) * r.ld + (bf - parent * (uint32_t)r.V)) : 0.f);
      }
      last_k = bk;
      last_f = bf;
    }
  }
}

struct BeamLayout {
  int slices;
  size_t off_keys, total;
};

BeamLayout beam_layout(int G, int W, int V) {
  BeamLayout L;
  const size_t rows = (size_t)G * W;
  L.slices = (int)(((int64_t)V + kSlice - 1) / kSlice);
  L.off_keys = (sizeof(float2) * rows * L.slices + 255) & ~size_t(255);
  L.total = L.off_keys + sizeof(unsigned long long) * rows * L.slices * W;
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
  const BeamRows r{logits, ld, scores, finished, W, V, L.slices, reinterpret_cast<float2*>(w),
                   reinterpret_cast<unsigned long long*>(w + L.off_keys)};
  const dim3 grid(L.slices, G * W);
  const bool vec = !(reinterpret_cast<uintptr_t>(logits) & 15) && ld % 4 == 0 && V % 4 == 0;
  if (vec) SSD_PDL(beam_rows_kernel<true>, grid, kRowThreads, 0, stream, r);
  else SSD_PDL(beam_rows_kernel<false>, grid, kRowThreads, 0, stream, r);
  const BeamMerge m{r, lengths, eos, (double)length_penalty, out_scores, out_parents, out_tokens, out_lengths,
                    out_finished};
  SSD_PDL(beam_merge_kernel, G, kMergeThreads, 0, stream, m);
  return SSD_OK;
}
