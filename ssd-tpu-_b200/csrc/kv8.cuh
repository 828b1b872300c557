// Shared pieces of the 8-bit paged KV cache (not part of the C ABI).
//
// pages  [2][L][NB][BS][Hkv][D] e4m3, scales [2][L][NB][Hkv] fp32: element = byte value * scale of its
// (plane, layer, page, head).  Every scale is a power of two, so dividing by it is exact, an e4m3 value
// keeps its four significant bits whatever the scale, and a page whose scale has to grow is rewritten
// without rounding again, but for values that fall among e4m3's subnormals: below 2^-6 of the scale, hence at most
// 2^-13.8 of the largest value that the page has held.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <atomic>

#include "common.cuh"

namespace ssd {

constexpr int kKv8MinExp = -118;  // scale exponents: 2^-118 .. 2^120, so 2^e and 2^-e are normal fp32 values

// Smallest e >= kKv8MinExp with amax <= 448 * 2^e (448 = 1.75 * 2^8, e4m3's largest value).
__device__ __forceinline__ int kv8_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, kKv8MinExp);
}
__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
// Exponent of a stored scale.  A page that nothing was appended to may hold anything there: clamped, and every kernel
// takes a scale by this exponent, so that a page reads the same whichever is chosen.
__device__ __forceinline__ int scale_exponent(float s) {
  return min(max((int)((__float_as_uint(s) >> 23) & 0xffu) - 127, kKv8MinExp), 120);
}
__device__ __forceinline__ float stored_scale(float s) {  // exp2i(scale_exponent(s)) in three instructions
  return fminf(fmaxf(__uint_as_float(__float_as_uint(s) & 0x7f800000u), 3.009265538e-36f), 1.329227996e36f);
}

// |x| where x is finite, else 0 (the scale goes by the finite values; the others are stored as NaN).
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}

// Two fp32 values (already divided by the scale, hence within 448 unless infinite) to e4m3, nearest even.  NaN stays
// NaN; so do infinities where INF says that there may be some (the conversion alone would make them 448).
template <bool INF = false>
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint32_t r = __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
  if (INF) {
    if (!(fabsf(lo) <= 3.402823466e38f)) r = (r & 0xff00u) | 0x7fu;
    if (!(fabsf(hi) <= 3.402823466e38f)) r = (r & 0x00ffu) | 0x7f00u;
  }
  return r;
}
template <bool INF = false>
__device__ __forceinline__ uint32_t e4m3x4(const float* f, float inv) {
  return e4m3x2<INF>(f[0] * inv, f[1] * inv) | (e4m3x2<INF>(f[2] * inv, f[3] * inv) << 16);
}
// e4m3 pair (low 16 bits) -> f16 pair, exact.
__device__ __forceinline__ uint32_t f16x2_of(uint32_t pair) {
  uint32_t r;
  asm("{.reg .b16 p; cvt.u16.u32 p, %1; cvt.rn.f16x2.e4m3x2 %0, p;}" : "=r"(r) : "r"(pair));
  return r;
}
// The four e4m3 values of a word -> two f16 pairs (bytes 0, 1 and bytes 2, 3).
__device__ __forceinline__ void f16x4_of(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{.reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b;}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
__device__ __forceinline__ float2 e4m3_pair(uint32_t pair) {
  const uint32_t h = f16x2_of(pair & 0xffffu);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Bytes of w that are e4m3 NaN (0x7f, 0xff), as 0x80 marks.
__device__ __forceinline__ uint32_t nan_marks(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ uint32_t clear_nan(uint32_t w) { return w & ~((nan_marks(w) >> 7) * 0xffu); }

struct Kv8Cache {
  uint8_t* pages;
  float* scales;
  int64_t plane;        // bytes of one K (or V) plane
  int64_t layer;        // byte offset of the layer inside a plane
  int64_t scale_plane;  // scales of one plane
  int64_t scale_layer;  // first scale of the layer inside a plane
  int num_blocks, block_size, hkv;
};

inline Kv8Cache kv8_cache(void* pages, float* scales, int num_layers, int num_blocks, int block_size, int hkv, int D,
                          int layer) {
  Kv8Cache c;
  c.pages = reinterpret_cast<uint8_t*>(pages);
  c.scales = scales;
  const int64_t per_layer = (int64_t)num_blocks * block_size * hkv * D;
  c.plane = per_layer * num_layers;
  c.layer = per_layer * layer;
  c.scale_plane = (int64_t)num_layers * num_blocks * hkv;
  c.scale_layer = (int64_t)layer * num_blocks * hkv;
  c.num_blocks = num_blocks;
  c.block_size = block_size;
  c.hkv = hkv;
  return c;
}

inline bool kv8_aligned(const void* p) { return !(reinterpret_cast<uintptr_t>(p) & 15); }

// Host checks shared by every entry point over an 8-bit cache.
inline int kv8_check(const void* pages, const float* scales, int num_layers, int num_blocks, int block_size, int hkv,
                     int D, int layer) {
  if (!pages || !scales || num_layers <= 0 || num_blocks <= 0 || block_size <= 0 || hkv <= 0 || layer < 0 ||
      layer >= num_layers)
    return SSD_ERR_INVALID;
  if (D != 64 && D != 128 && D != 256) return SSD_ERR_UNSUPPORTED;
  // row numbers, and the pieces of a page's rows, are 32-bit
  if ((int64_t)num_blocks * block_size > 0x7fffffff || block_size > 1 << 20) return SSD_ERR_UNSUPPORTED;
  if (!kv8_aligned(pages)) return SSD_ERR_UNSUPPORTED;
  return SSD_OK;
}

// A kernel's dynamic shared memory limit belongs to each device's context: raised once per device (`ready`: one
// bit a device), always to the same size.
template <typename K>
bool allow_smem(std::atomic<uint64_t>& ready, K kern, int bytes) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  if (ready.load(std::memory_order_acquire) >> dev & 1) return true;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
    (void)cudaGetLastError();
    return false;
  }
  ready.fetch_or(1ull << dev, std::memory_order_release);
  return true;
}

}  // namespace ssd
