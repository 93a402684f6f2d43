// The paged cache of keys and values in 8 bits: geometry, scales and payload conversions shared by its kernels.
//
// Payload [num_pages, Hkv, page_size, width], one byte per value; scale [num_pages, Hkv] fp32, a power of two 2^e.
// A page of one kv head is contiguous, so a kernel that reads a head's tokens reads page_size * width bytes in a row.
// Why a power of two: x 2^-e and payload * 2^e are exact, so the only rounding is that to the payload's grid, reading
// back is exact, and a page whose scale grows when a token is appended rounds what it held on the new grid without the
// error of a quotient.  For e4m3, whose precision is relative, a finer scale would buy nothing; for int8 it costs at
// most one of seven bits.
#pragma once

#include <cuda_fp8.h>

#include "fm_common.cuh"

namespace fm {

struct KvGeom {
  int num_pages, page_log2, Hkv, max_pages;
  int cap;                       // positions of a row of the page table
  int64_t table_stride;
};

// Page of position `pos` of the sequence whose page table row is `row`, or -1: the position is outside of the table, or
// the table names no page of the cache.  The only place where a page number is turned into something to address with;
// fm_kv_locate runs it on the host.  In two steps for who has other work while the table is read.
__host__ __device__ __forceinline__ int kv_page_number(const KvGeom& g, const int32_t* row, int pos) {
  const int j = pos >> g.page_log2;
  return pos < 0 || j >= g.max_pages ? -1 : row[j];
}
__host__ __device__ __forceinline__ int kv_page_in(const KvGeom& g, int page) { return page >= 0 && page < g.num_pages ? page : -1; }
__host__ __device__ __forceinline__ int kv_page(const KvGeom& g, const int32_t* row, int pos) { return kv_page_in(g, kv_page_number(g, row, pos)); }

// Length of a sequence as the kernels use it: never beyond its page table.
__host__ __device__ __forceinline__ int kv_len(const KvGeom& g, int len) { return len < 0 ? 0 : (len > g.cap ? g.cap : len); }

constexpr int kCacheMinExp = -64;
template <bool INT8> constexpr int kCacheMaxExp = INT8 ? 121 : 119;     // largest e with a finite 127 * 2^e | 448 * 2^e

// Least e with amax <= M 2^e (M = 448 = 1.75 * 2^8 or 127 = 1.984375 * 2^6), in range; amax >= 0 and finite.
template <bool INT8>
__device__ __forceinline__ int cache_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int x = (int)(u >> 23) - 127;                                   // (zero and subnormals: below the range)
  const int e = x - (INT8 ? 6 : 8) + ((u & 0x7fffffu) > (INT8 ? 0x7e0000u : 0x600000u) ? 1 : 0);
  return min(max(e, kCacheMinExp), kCacheMaxExp<INT8>);
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 <= e <= 127

// Two values to two payload bytes (the first in the low byte).  Nearest even, saturating; NaN stays NaN in e4m3 (int8
// has none: the caller takes it out).
template <bool INT8>
__device__ __forceinline__ uint32_t to_payload2(float lo, float hi) {
  if constexpr (INT8) {
    const int a = __float2int_rn(fminf(fmaxf(lo, -127.f), 127.f)), b = __float2int_rn(fminf(fmaxf(hi, -127.f), 127.f));
    return (uint32_t)(a & 0xff) | (uint32_t)(b & 0xff) << 8;
  } else {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
  }
}

// 0x80 in every byte of w that is an e4m3 NaN (0x7f, 0xff).
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// Payload bytes 0, 1 (`lo`) and 2, 3 (`hi`) of a word as pairs of fp16: every payload value is an fp16 value.
template <bool INT8>
__device__ __forceinline__ void from_payload4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (INT8) {
    // 1024 + (x + 128) is the fp16 with the byte x ^ 0x80 below the exponent of 1024
    w ^= 0x80808080u;
    const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));     // 1152
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), off), y = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(w));
  }
}

// The same as fp32.
template <bool INT8>
__device__ __forceinline__ void payload_f32(uint32_t w, float (&x)[4]) {
  uint32_t lo, hi;
  from_payload4<INT8>(w, lo, hi);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
}

// A pair of 16-bit inputs as fp32.
template <bool IS_BF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (IS_BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

}  // namespace fm
