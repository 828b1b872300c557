// 8-bit paged KV cache: quantised append (plain, and fused with the rotary embedding) and read-back.
//
// Append.  New rows enter at the end of each sequence, at the positions the attention calls use: token t
// of row b at n0 + t, n0 = seq_lens[b] - q_lens[b].  For one page, KV head and plane let R be the new rows:
//   e = smallest exponent with max |R| <= 448 2^e;   if rows before R are in the page: e = max(e, e_page)
//   stored = e4m3(R 2^-e),   earlier rows = e4m3(old 2^(e_page - e))  where e grew, else untouched.
// A page whose first row is among the new ones starts over: what it held counts for nothing.  Rows behind
// the last new one keep their bytes.
//
// One warp per (sequence, touched page, KV head, plane): the page's scale has one owner, no atomics, no barrier, and
// the result does not depend on scheduling.  The rows stay in registers, as they came, between the maximum and the
// rounding, all their loads in flight at once (8 KB a warp for a page of 16 rows of 256 in bf16); old rows are read
// only when the scale grows.  Bound: HBM for prompts (4 sequences, 5500 rows of 16 heads of 256 in bf16: 135 MB in
// 25.0 us, 5.4 TB/s; with the rows converted to fp32 before the maximum, 57 us), launch latency for single tokens
// (2 to 4 us).
#include <type_traits>

#include "kv8.cuh"

namespace ssd {
namespace {

// 8 values as they came, and as fp32.
template <typename T> struct Raw8;
template <> struct Raw8<bf16> {
  uint4 a;
  __device__ __forceinline__ void load(const bf16* p) { a = ld_act_v4(p); }
  __device__ __forceinline__ void get(float* f) const { unpack8(a, f); }
  __device__ __forceinline__ float largest() const {  // magnitude, NaN not counted
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&a);
    const __nv_bfloat162 m = __hmax2(__hmax2(__habs2(h[0]), __habs2(h[1])), __hmax2(__habs2(h[2]), __habs2(h[3])));
    return fmaxf(__low2float(m), __high2float(m));
  }
};
template <> struct Raw8<float> {
  uint4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = ld_act_v4(p);
    b = ld_act_v4(p + 4);
  }
  __device__ __forceinline__ void get(float* f) const {
    f[0] = __uint_as_float(a.x); f[1] = __uint_as_float(a.y); f[2] = __uint_as_float(a.z); f[3] = __uint_as_float(a.w);
    f[4] = __uint_as_float(b.x); f[5] = __uint_as_float(b.y); f[6] = __uint_as_float(b.z); f[7] = __uint_as_float(b.w);
  }
  __device__ __forceinline__ float largest() const {
    float f[8], m = 0.f;
    get(f);
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(f[i]));
    return m;
  }
};
__device__ __forceinline__ void store8(bf16* p, const float* f) {
  uint4 u;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = u;
}
__device__ __forceinline__ void store8(float* p, const float* f) {
  *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
}

struct AppendArgs {
  Kv8Cache c;
  const int32_t* tables;
  int max_blocks;
  const int32_t* seq_lens;
  const int32_t* q_lens;
  const void* k;        // row m, head h at k + m * row + h * D
  const void* v;
  int64_t row;          // elements between token rows
  int T, pages_per_seq, units, kv_ctas;
  // rotary embedding (nullptr cos: none)
  const void* q;
  void* q_out;          // [B*T, hq, D]
  const float* cos_t;   // [rope_max_pos, D/2]
  const float* sin_t;
  int hq, rope_max_pos, total_rows;
};

// y1 = x1 c - x2 s, y2 = x2 c + x1 s, the products rounded one by one (as ssd_rope_kv_write does)
__device__ __forceinline__ void rotate8(float* x1, float* x2, const float* c, const float* s) {
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    const float4 cv = *reinterpret_cast<const float4*>(c + i), sv = *reinterpret_cast<const float4*>(s + i);
    const float cc[4] = {cv.x, cv.y, cv.z, cv.w}, ss[4] = {sv.x, sv.y, sv.z, sv.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a = x1[i + j], b = x2[i + j];
      x1[i + j] = __fsub_rn(__fmul_rn(a, cc[j]), __fmul_rn(b, ss[j]));
      x2[i + j] = __fadd_rn(__fmul_rn(b, cc[j]), __fmul_rn(a, ss[j]));
    }
  }
}

// An item: dims d .. d + 7 and D/2 + d .. D/2 + d + 7 of a row, so a rotation pair where K is rotated.
template <typename T, int D>
struct Rows {
  const AppendArgs& a;
  const T* base;  // head's values in the token row of position `first`
  int first;      // first new position in the page
  bool rotated;
  struct Item { Raw8<T> lo, hi; };
  __device__ __forceinline__ void load(int i, Item& x) const {
    const T* p = base + (i / (D / 16)) * a.row + (i % (D / 16)) * 8;
    x.lo.load(p);
    x.hi.load(p + D / 2);
  }
  __device__ __forceinline__ void get(int i, const Item& x, float* f) const {  // 16 values
    x.lo.get(f);
    x.hi.get(f + 8);
    if (rotated) {
      const int p = min(first + i / (D / 16), a.rope_max_pos - 1);
      const int64_t at = (int64_t)p * (D / 2) + (i % (D / 16)) * 8;
      rotate8(f, f + 8, a.cos_t + at, a.sin_t + at);
    }
  }
};

template <typename T, int D>
__device__ __forceinline__ void rope_q_cta(const AppendArgs& a, int cta) {
  // one CTA a token row, its threads over the heads: items of 16 dims
  constexpr int PER = D / 16;
  const int items = a.hq * PER;
  const int64_t m = cta;
  const int b = (int)(m / a.T), t = (int)(m % a.T);
  const int seq = ld_act(a.seq_lens + b);
  const int ql = a.q_lens ? min(max(ld_act(a.q_lens + b), 0), a.T) : a.T;
  const int pos = seq - ql + t;
  const bool real = t < ql && pos >= 0;
  const int p = real ? min(pos, a.rope_max_pos - 1) : 0;
  const T* src = reinterpret_cast<const T*>(a.q) + m * a.row;
  T* dst = reinterpret_cast<T*>(a.q_out) + m * a.hq * D;
  for (int i = threadIdx.x; i < items; i += blockDim.x) {
    const int h = i / PER, d = (i % PER) * 8;
    float x0[8], x1[8];
    if (real) {
      Raw8<T> lo, hi;
      lo.load(src + h * D + d);
      hi.load(src + h * D + d + D / 2);
      lo.get(x0);
      hi.get(x1);
      rotate8(x0, x1, a.cos_t + (int64_t)p * (D / 2) + d, a.sin_t + (int64_t)p * (D / 2) + d);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x0[j] = x1[j] = 0.f;
    }
    store8(dst + h * D + d, x0);
    store8(dst + h * D + d + D / 2, x1);
  }
}

// KEEP: items a lane holds between the two passes; a page's items beyond KEEP * 32 are read a second time (L2).
constexpr int kAppendWarps = 4;

template <typename T, int D, int KEEP>
__global__ void __launch_bounds__(kAppendWarps * 32, 4) kv8_append_kernel(const AppendArgs a) {
  pdl_wait();
  pdl_trigger();
  if ((int)blockIdx.x >= a.kv_ctas) {
    rope_q_cta<T, D>(a, blockIdx.x - a.kv_ctas);
    return;
  }
  const int lane = threadIdx.x & 31;
  int u = blockIdx.x * kAppendWarps + (threadIdx.x >> 5);
  if (u >= a.units) return;
  const int plane = u & 1;
  u >>= 1;
  const int head = u % a.c.hkv;
  u /= a.c.hkv;
  const int i = u % a.pages_per_seq, b = u / a.pages_per_seq;
  const int bs = a.c.block_size;
  const int seq = ld_act(a.seq_lens + b);
  const int ql = a.q_lens ? min(max(ld_act(a.q_lens + b), 0), a.T) : a.T;
  const int n0 = seq - ql;
  const int start = max(n0, 0);
  const int page = start / bs + i;
  const int64_t p0 = (int64_t)page * bs;
  if (p0 >= seq || page >= a.max_blocks) return;
  const int first = max(start, (int)p0);
  const int rows = (int)min((int64_t)seq, p0 + bs) - first;
  if (rows <= 0) return;
  const int blk = ld_act(a.tables + (int64_t)b * a.max_blocks + page);

  constexpr int PER = D / 16;
  const Rows<T, D> src{a, reinterpret_cast<const T*>(plane ? a.v : a.k) + ((int64_t)b * a.T + (first - n0)) * a.row +
                              (int64_t)head * D, first, a.cos_t != nullptr && plane == 0};
  const int items = rows * PER;
  typename Rows<T, D>::Item x[KEEP];
#pragma unroll
  for (int k = 0; k < KEEP; ++k)
    if (lane + 32 * k < items) src.load(lane + 32 * k, x[k]);
  if ((unsigned)blk >= (unsigned)a.c.num_blocks) return;
  float* scale = a.c.scales + plane * a.c.scale_plane + a.c.scale_layer + (int64_t)blk * a.c.hkv + head;
  uint8_t* base = a.c.pages + plane * a.c.plane + a.c.layer + ((int64_t)blk * bs * a.c.hkv + head) * D;
  const int64_t rstride = (int64_t)a.c.hkv * D;
  const int r0 = first - (int)p0;  // first new row of the page
  const int eo = r0 > 0 ? scale_exponent(ld_act(scale)) : kKv8MinExp;

  auto each = [&](auto&& use) {
#pragma unroll
    for (int k = 0; k < KEEP; ++k)
      if (lane + 32 * k < items) use(lane + 32 * k, x[k]);
    for (int it = lane + 32 * KEEP; it < items; it += 32) {
      typename Rows<T, D>::Item y;
      src.load(it, y);
      use(it, y);
    }
  };
  float amax = 0.f;
  if (src.rotated) {
    each([&](int it, const typename Rows<T, D>::Item& y) {
      float f[16];
      src.get(it, y, f);
#pragma unroll
      for (int j = 0; j < 16; ++j) amax = fmaxf(amax, fabsf(f[j]));
    });
  } else {
    each([&](int, const typename Rows<T, D>::Item& y) { amax = fmaxf(amax, fmaxf(y.lo.largest(), y.hi.largest())); });
  }
  amax = warp_max(amax);
  const bool inf = amax > 3.402823466e38f;
  if (inf) {  // rare: the scale goes by the finite values
    amax = 0.f;
    each([&](int it, const typename Rows<T, D>::Item& y) {
      float f[16];
      src.get(it, y, f);
#pragma unroll
      for (int j = 0; j < 16; ++j) amax = fmaxf(amax, finite_abs(f[j]));
    });
    amax = warp_max(amax);
  }
  int e = kv8_exponent(amax);
  if (r0 > 0 && e > eo) {
    // the earlier rows move to the larger scale; exp2i's range holds the difference down to 2^-126, below
    // which every value rounds to zero anyway
    const float f = exp2i(max(eo - e, -126));
    for (int it = lane; it < r0 * PER; it += 32) {
      uint4* p = reinterpret_cast<uint4*>(base + (it / PER) * rstride + (it % PER) * 16);
      const uint4 w = ld_act_v4(p);
      const uint32_t in[4] = {w.x, w.y, w.z, w.w};
      uint32_t out[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 lo = e4m3_pair(in[j]), hi = e4m3_pair(in[j] >> 16);
        const float v[4] = {lo.x, lo.y, hi.x, hi.y};
        out[j] = e4m3x4(v, f);
      }
      *p = make_uint4(out[0], out[1], out[2], out[3]);
    }
  }
  e = max(e, eo);
  __syncwarp();  // every lane has read the old scale
  if (lane == 0) *scale = exp2i(e);
  const float inv = exp2i(-e);
  auto put = [&](int it, const typename Rows<T, D>::Item& y, auto may_inf) {
    constexpr bool INF = decltype(may_inf)::value;
    float f[16];
    src.get(it, y, f);
    uint8_t* p = base + (r0 + it / PER) * rstride + (it % PER) * 8;
    *reinterpret_cast<uint2*>(p) = make_uint2(e4m3x4<INF>(f, inv), e4m3x4<INF>(f + 4, inv));
    *reinterpret_cast<uint2*>(p + D / 2) = make_uint2(e4m3x4<INF>(f + 8, inv), e4m3x4<INF>(f + 12, inv));
  };
  if (!inf)
    each([&](int it, const typename Rows<T, D>::Item& y) { put(it, y, std::false_type()); });
  else
    each([&](int it, const typename Rows<T, D>::Item& y) { put(it, y, std::true_type()); });
}

template <typename T, int D>
int launch_append_d(cudaStream_t st, const AppendArgs& a) {
  constexpr int KEEP = sizeof(T) == 2 ? 8 : 4;
  const int64_t q_ctas = a.cos_t ? (int64_t)a.total_rows : 0;
  if (a.kv_ctas + q_ctas > 0x7fffffff) return SSD_ERR_UNSUPPORTED;
  SSD_PDL((kv8_append_kernel<T, D, KEEP>), (unsigned)(a.kv_ctas + q_ctas), kAppendWarps * 32, 0, st, a);
  return SSD_OK;
}

template <typename T>
int launch_append(cudaStream_t st, const AppendArgs& a, int D) {
  if (D == 256) return launch_append_d<T, 256>(st, a);
  if (D == 128) return launch_append_d<T, 128>(st, a);
  return launch_append_d<T, 64>(st, a);
}

int append_common(ssd_stream_t stream, AppendArgs a, int dtype, int B, int T, int D) {
  const int bs = a.c.block_size;
  const int64_t pages = ((int64_t)T + bs - 2) / bs + 1;  // pages that T consecutive rows can touch
  const int64_t units = (int64_t)B * pages * a.c.hkv * 2;
  if (units > 0x7fffffff - kAppendWarps || (int64_t)B * T > 0x7fffffff) return SSD_ERR_UNSUPPORTED;
  a.T = T;
  a.total_rows = B * T;
  a.pages_per_seq = (int)pages;
  a.units = (int)units;
  a.kv_ctas = (int)((units + kAppendWarps - 1) / kAppendWarps);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == SSD_DTYPE_BF16) return launch_append<bf16>(st, a, D);
  return launch_append<float>(st, a, D);
}

// K and V rows of positions [B][N] (-1: zeros).  A row of one position is 2 Hkv D values; a warp takes up to
// kGatherItems * 32 groups of 8 of them (8 bytes in, 16 or 32 out, neighbouring lanes on neighbouring groups), all
// loads in flight at once (4 or 16 groups a lane: 10 to 14 % slower).  Bound: HBM (the rows above with their pages' earlier
// ones, 5533 of 6128 positions: 146 MB in 27.2 us, 5.4 TB/s).
constexpr int kGatherItems = 8;

template <typename T, int D>
__global__ void __launch_bounds__(256) kv8_gather_kernel(const Kv8Cache c, const int32_t* tables, int max_blocks,
                                                         const int32_t* positions, int64_t rows, int N, int chunks,
                                                         T* k, T* v) {
  pdl_wait();
  pdl_trigger();
  constexpr int PER = D / 8;
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (w >= rows * chunks) return;
  const int64_t m = w / chunks;
  const int first = (int)(w - m * chunks) * (kGatherItems * 32) + lane;
  const int b = (int)(m / N);
  const int pos = ld_act(positions + m);
  int blk = -1;
  if (pos >= 0 && pos / c.block_size < max_blocks)
    blk = ld_act(tables + (int64_t)b * max_blocks + pos / c.block_size);
  const bool ok = (unsigned)blk < (unsigned)c.num_blocks;
  const int items = c.hkv * PER;
  const uint8_t* row = c.pages + c.layer + (ok ? (int64_t)blk * c.block_size + pos % c.block_size : 0) * c.hkv * D;
  const float* sc = c.scales + c.scale_layer + (ok ? (int64_t)blk * c.hkv : 0);
  uint2 x[kGatherItems];
  float s[kGatherItems];
#pragma unroll
  for (int i = 0; i < kGatherItems; ++i) {
    const int it = first + 32 * i;
    const int plane = it >= items, j = plane ? it - items : it;
    x[i] = make_uint2(0, 0);
    s[i] = 0.f;
    if (ok && it < 2 * items) {
      x[i] = __ldcg(reinterpret_cast<const uint2*>(row + plane * c.plane + (int64_t)j * 8));
      s[i] = ld_act(sc + plane * c.scale_plane + j / PER);
    }
  }
#pragma unroll
  for (int i = 0; i < kGatherItems; ++i) {
    const int it = first + 32 * i;
    const int plane = it >= items, j = plane ? it - items : it;
    if (it >= 2 * items) break;
    const uint32_t in[2] = {x[i].x, x[i].y};
    asm volatile("" : "+f"(s[i]));  // keeps the next line behind all loads: among them it costs 3.5 us more than 27
    const float by = stored_scale(s[i]);
    float f[8];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float2 lo = e4m3_pair(in[q]), hi = e4m3_pair(in[q] >> 16);
      f[4 * q] = lo.x * by; f[4 * q + 1] = lo.y * by; f[4 * q + 2] = hi.x * by; f[4 * q + 3] = hi.y * by;
    }
    store8((plane ? v : k) + m * c.hkv * D + (int64_t)j * 8, f);
  }
}

template <typename T>
int launch_gather(cudaStream_t st, const Kv8Cache& c, const int32_t* tables, int max_blocks, const int32_t* positions,
                  int64_t rows, int N, void* k, void* v, int D) {
  const int chunks = (2 * c.hkv * (D / 8) + kGatherItems * 32 - 1) / (kGatherItems * 32);
  const int64_t ctas = (rows * chunks + 7) / 8;
  if (ctas > 0x7fffffff) return SSD_ERR_UNSUPPORTED;
  const unsigned grid = (unsigned)ctas;
  T* ko = reinterpret_cast<T*>(k);
  T* vo = reinterpret_cast<T*>(v);
  if (D == 256)
    SSD_PDL((kv8_gather_kernel<T, 256>), grid, 256, 0, st, c, tables, max_blocks, positions, rows, N, chunks, ko, vo);
  else if (D == 128)
    SSD_PDL((kv8_gather_kernel<T, 128>), grid, 256, 0, st, c, tables, max_blocks, positions, rows, N, chunks, ko, vo);
  else
    SSD_PDL((kv8_gather_kernel<T, 64>), grid, 256, 0, st, c, tables, max_blocks, positions, rows, N, chunks, ko, vo);
  return SSD_OK;
}

}  // namespace
}  // namespace ssd

using namespace ssd;

extern "C" int ssd_kv8_append(ssd_stream_t stream, void* pages, float* scales, int num_layers, int num_blocks,
                              int block_size, int num_kv_heads, int head_dim, int layer, const int32_t* block_tables,
                              int max_blocks, const int32_t* seq_lens, const int32_t* q_lens, const void* k,
                              const void* v, int dtype, int B, int T) {
  if (int rc = kv8_check(pages, scales, num_layers, num_blocks, block_size, num_kv_heads, head_dim, layer)) return rc;
  if (B < 0 || T < 0 || max_blocks <= 0 || (dtype != SSD_DTYPE_BF16 && dtype != SSD_DTYPE_F32)) return SSD_ERR_INVALID;
  if (B == 0 || (T == 0 && block_tables && seq_lens)) return SSD_OK;  // arrays of nothing may have no address
  if (!block_tables || !seq_lens || !k || !v) return SSD_ERR_INVALID;
  if (!kv8_aligned(k) || !kv8_aligned(v)) return SSD_ERR_UNSUPPORTED;
  AppendArgs a{};
  a.c = kv8_cache(pages, scales, num_layers, num_blocks, block_size, num_kv_heads, head_dim, layer);
  a.tables = block_tables;
  a.max_blocks = max_blocks;
  a.seq_lens = seq_lens;
  a.q_lens = q_lens;
  a.k = k;
  a.v = v;
  a.row = (int64_t)num_kv_heads * head_dim;
  return append_common(stream, a, dtype, B, T, head_dim);
}

extern "C" int ssd_kv8_rope_append(ssd_stream_t stream, const void* qkv, void* q_out, void* pages, float* scales,
                                   int dtype, int num_layers, int num_blocks, int block_size, int num_heads,
                                   int num_kv_heads, int head_dim, int layer, const int32_t* block_tables,
                                   int max_blocks, const int32_t* seq_lens, const int32_t* q_lens,
                                   const float* rope_cos, const float* rope_sin, int rope_max_pos, int B, int T) {
  if (int rc = kv8_check(pages, scales, num_layers, num_blocks, block_size, num_kv_heads, head_dim, layer)) return rc;
  if (B < 0 || T < 0 || max_blocks <= 0 || num_heads <= 0 || rope_max_pos <= 0 || !rope_cos || !rope_sin ||
      (dtype != SSD_DTYPE_BF16 && dtype != SSD_DTYPE_F32))
    return SSD_ERR_INVALID;
  if (B == 0 || (T == 0 && block_tables && seq_lens)) return SSD_OK;
  if (!block_tables || !seq_lens || !qkv || !q_out) return SSD_ERR_INVALID;
  if (!kv8_aligned(qkv) || !kv8_aligned(q_out) || !kv8_aligned(rope_cos) || !kv8_aligned(rope_sin))
    return SSD_ERR_UNSUPPORTED;
  const size_t es = dtype == SSD_DTYPE_BF16 ? 2 : 4;
  AppendArgs a{};
  a.c = kv8_cache(pages, scales, num_layers, num_blocks, block_size, num_kv_heads, head_dim, layer);
  a.tables = block_tables;
  a.max_blocks = max_blocks;
  a.seq_lens = seq_lens;
  a.q_lens = q_lens;
  a.q = qkv;
  a.k = reinterpret_cast<const char*>(qkv) + es * (size_t)num_heads * head_dim;
  a.v = reinterpret_cast<const char*>(qkv) + es * (size_t)(num_heads + num_kv_heads) * head_dim;
  a.row = (int64_t)(num_heads + 2 * num_kv_heads) * head_dim;
  a.q_out = q_out;
  a.cos_t = rope_cos;
  a.sin_t = rope_sin;
  a.hq = num_heads;
  a.rope_max_pos = rope_max_pos;
  return append_common(stream, a, dtype, B, T, head_dim);
}

extern "C" int ssd_kv8_gather(ssd_stream_t stream, const void* pages, const float* scales, int num_layers,
                              int num_blocks, int block_size, int num_kv_heads, int head_dim, int layer,
                              const int32_t* block_tables, int max_blocks, const int32_t* positions, void* k, void* v,
                              int dtype, int B, int N) {
  if (int rc = kv8_check(pages, scales, num_layers, num_blocks, block_size, num_kv_heads, head_dim, layer)) return rc;
  if (B < 0 || N < 0 || max_blocks <= 0 || (dtype != SSD_DTYPE_BF16 && dtype != SSD_DTYPE_F32)) return SSD_ERR_INVALID;
  if (B == 0 || (N == 0 && block_tables)) return SSD_OK;
  if (!block_tables || !positions || !k || !v) return SSD_ERR_INVALID;
  if (!kv8_aligned(k) || !kv8_aligned(v)) return SSD_ERR_UNSUPPORTED;
  const int64_t rows = (int64_t)B * N;
  const Kv8Cache c = kv8_cache(const_cast<void*>(pages), const_cast<float*>(scales), num_layers, num_blocks,
                               block_size, num_kv_heads, head_dim, layer);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == SSD_DTYPE_BF16)
    return launch_gather<bf16>(st, c, block_tables, max_blocks, positions, rows, N, k, v, head_dim);
  return launch_gather<float>(st, c, block_tables, max_blocks, positions, rows, N, k, v, head_dim);
}
