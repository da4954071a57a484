// Device view of a paged key / value cache, element types, and the place of a row in it.
//
// Position p of sequence b lies in page page_table[b][p / page_size], slot p % page_size. Row i of a call belongs to the
// sequence b with cu_rows[b] <= i < cu_rows[b + 1] and stands for position lens[b] + i - cu_rows[b]. A position at or behind
// the end of the sequence's page list, or whose page number is outside [0, n_pages), does not exist: it is neither read nor
// written. Element offsets are 64-bit everywhere.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/spfa_b200.h"

namespace spfa {

struct e4m3 {
  uint8_t bits;
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// One 32-bit value of an element, and back (rounding to nearest even; e4m3 saturates at 448).
__device__ __forceinline__ float up1(float x) { return x; }
__device__ __forceinline__ float up1(__half x) { return __half2float(x); }
__device__ __forceinline__ float up1(__nv_bfloat16 x) { return __bfloat162float(x); }
// 8388608 + (code + 128) has the code's bits as its last
__device__ __forceinline__ float up1(int8_t x) { return __uint_as_float(0x4b000000u | ((uint8_t)x ^ 0x80u)) - 8388736.f; }
__device__ __forceinline__ float up1(e4m3 x) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)x.bits, __NV_E4M3)));
}
__device__ __forceinline__ void down1(float& y, float x) { y = x; }
__device__ __forceinline__ void down1(__half& y, float x) { y = __float2half_rn(x); }
__device__ __forceinline__ void down1(__nv_bfloat16& y, float x) { y = __float2bfloat16_rn(x); }
// |x| <= 127 (1 + 2^-23) here: row_scale's inverse times an element of its row
// (the sum is rounded to a whole number, to even where it is half way: its last byte is the code; x itself was
// rounded before)
__device__ __forceinline__ void down1(int8_t& y, float x) { y = (int8_t)__float_as_uint(__fadd_rn(x, 12582912.f)); }
__device__ __forceinline__ void down1(e4m3& y, float x) { y.bits = __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3); }

template <class T> struct IsByte { static constexpr bool value = sizeof(T) == 1; };

// N elements that lie together and aligned to their common size (at most 16 bytes), as 32-bit values.
template <int Bytes> struct RawOf;
template <> struct RawOf<1> { using type = uint8_t; };
template <> struct RawOf<2> { using type = uint16_t; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<16> { using type = uint4; };

template <class T, int N>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[N]) {
  using Raw = typename RawOf<N * (int)sizeof(T)>::type;
  union {
    Raw raw;
    T e[N];
  } u;
  u.raw = *reinterpret_cast<const Raw*>(p);
  if constexpr (std::is_same<T, e4m3>::value && N % 2 == 0) {  // the conversion instruction takes pairs
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(u.e[i].bits | (u.e[i + 1].bits << 8)), __NV_E4M3);
      const float2 f = __half22float2(__half2(h));
      x[i] = f.x;
      x[i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = up1(u.e[i]);
  }
}
// (all zeros where `none`)
template <class T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[N], bool none = false) {
  using Raw = typename RawOf<N * (int)sizeof(T)>::type;
  union {
    Raw raw;
    T e[N];
  } u;
  if constexpr (std::is_same<T, e4m3>::value && N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const __nv_fp8x2_storage_t h = __nv_cvt_float2_to_fp8x2(make_float2(x[i], x[i + 1]), __NV_SATFINITE, __NV_E4M3);
      u.e[i].bits = (uint8_t)h;
      u.e[i + 1].bits = (uint8_t)(h >> 8);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) down1(u.e[i], x[i]);
  }
  if (none) u.raw = Raw{};
  *reinterpret_cast<Raw*>(p) = u.raw;
}

struct Pages {  // one of K and V
  char* data;
  float* scale;         // null where the cache holds its values as they are
  int64_t stride[3];    // elements from page to page, slot to slot, head to head
  int64_t s_stride[3];  // the same of the scales
  __device__ __forceinline__ int64_t at(int64_t page, int64_t slot, int64_t head) const {
    return page * stride[0] + slot * stride[1] + head * stride[2];
  }
  __device__ __forceinline__ int64_t scale_at(int64_t page, int64_t slot, int64_t head) const {
    return page * s_stride[0] + slot * s_stride[1] + head * s_stride[2];
  }
};

struct CacheView {
  Pages K, V;
  const int32_t* table;
  const int32_t* lens;
  int64_t n_pages;
  int32_t page_size, n_heads, d, n_seq;
  int64_t table_width, capacity;  // pages and positions of a sequence (capacity is below 2^31: positions are 32-bit)

  // Page of position p of sequence b, or -1 where the position does not exist.
  __device__ __forceinline__ int32_t page_of(int32_t b, int64_t p) const {
    if (p < 0 || p >= capacity) return -1;
    const int32_t page = __ldg(table + (int64_t)b * table_width + (uint32_t)p / (uint32_t)page_size);
    return (page >= 0 && page < n_pages) ? page : -1;
  }
  __device__ __forceinline__ int32_t slot_of(int64_t p) const { return (int32_t)((uint32_t)p % (uint32_t)page_size); }
  // Committed length of sequence b, within what its page list can hold.
  __device__ __forceinline__ int64_t len_of(int32_t b) const {
    const int64_t n = __ldg(lens + b);
    return n < 0 ? 0 : (n < capacity ? n : capacity);
  }
};

// Rows [begin, end) of sequence b among the n rows of a call.
__device__ __forceinline__ void rows_of(const int32_t* cu, int32_t b, int64_t n, int64_t& begin, int64_t& end) {
  const int64_t x = __ldg(cu + b), y = __ldg(cu + b + 1);
  begin = x < 0 ? 0 : (x < n ? x : n);
  end = y < begin ? begin : (y < n ? y : n);
}

// The sequence that row i belongs to, or -1 (rows before the first sequence or behind the last).
__device__ __forceinline__ int32_t sequence_of(const int32_t* cu, int32_t n_seq, int64_t i) {
  int32_t lo = 0, hi = n_seq;  // the first b of [0, n_seq] whose cu[b + 1] is above i
  while (lo < hi) {
    const int32_t mid = (lo + hi) >> 1;
    if ((int64_t)__ldg(cu + mid + 1) > i) hi = mid;
    else lo = mid + 1;
  }
  return (lo < n_seq && (int64_t)__ldg(cu + lo) <= i) ? lo : -1;
}

// The scale of a quantised row, from the largest magnitude of its elements (`top`; NaN and infinity included).
//   e4m3  2^e with the smallest e >= -126 for which top <= 448 2^e: a division by it and the product with it are exact
//   int8  top / 127; rows below 2^-100 count as zeros (127 / top has to stay finite)
// `inverse` is what an element is multiplied by before it is rounded. A row with a value that is not finite gets scale NaN:
// it reads back as NaN, and attention over it gives NaN.
template <class T>
__device__ __forceinline__ float row_scale(float top, float& inverse);
template <>
__device__ __forceinline__ float row_scale<e4m3>(float top, float& inverse) {
  if (!(top <= 3.402823466e38f)) {
    inverse = 0.f;
    return __int_as_float(0x7fc00000);
  }
  // top = 1.f 2^(x - 127): 448 = 1.75 2^8
  const uint32_t bits = __float_as_uint(top);
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = e < -126 ? -126 : e;
  inverse = __uint_as_float((uint32_t)(127 - e) << 23);
  return __uint_as_float((uint32_t)(127 + e) << 23);
}
template <>
__device__ __forceinline__ float row_scale<int8_t>(float top, float& inverse) {
  if (!(top <= 3.402823466e38f)) {
    inverse = 0.f;
    return __int_as_float(0x7fc00000);
  }
  const bool some = top >= 7.8886090522101181e-31f;  // 2^-100
  inverse = some ? __fdiv_rn(127.f, top) : 0.f;
  return some ? __fdiv_rn(top, 127.f) : 0.f;
}

}  // namespace spfa
