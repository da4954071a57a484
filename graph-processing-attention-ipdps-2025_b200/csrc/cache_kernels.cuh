// Writing rows into a paged key / value cache, reading them back, and moving kept rows to the front.
//
// All three move bytes: a row (one head of one token) is taken once, its largest magnitude found by shuffles in the lanes that
// hold it, and it leaves in the cache's type; nothing is staged. The work of a call is known to the host up to which sequence a
// row belongs to, which every group of lanes finds by a binary search in cu_rows.
#pragma once
#include "cache_common.cuh"

namespace spfa {
namespace cache {

struct RowsView {  // rows of a call: [n_rows, heads, d], d contiguous
  char *K, *V;
  int64_t k_stride[2], v_stride[2];  // elements from row to row, head to head
  const int32_t* cu_rows;
  int64_t n_rows;
  int64_t first;  // of the launch: its group numbers are 32-bit
};

// Where row i of a call lies in the cache; page -1: nowhere.
struct Place {
  int32_t page, slot;
};
__device__ __forceinline__ Place place_of(const CacheView& c, const int32_t* cu, int64_t i) {
  Place at = {-1, 0};
  const int32_t b = sequence_of(cu, c.n_seq, i);
  if (b < 0) return at;
  const int64_t p = (int64_t)__ldg(c.lens + b) + (i - __ldg(cu + b));
  at.page = c.page_of(b, p);
  if (at.page >= 0) at.slot = c.slot_of(p);
  return at;
}

constexpr int kThreads = 256;

// Which row and heads a group of lanes works on: rows first, then pieces of `HC` heads.
template <int LPR, int HC>
struct Task {
  uint32_t i;
  int32_t h0;
  __device__ __forceinline__ Task(const CacheView& c) {
    const uint32_t group = (blockIdx.x * (uint32_t)kThreads + threadIdx.x) / LPR, parts = (uint32_t)(c.n_heads + HC - 1) / HC;
    i = group / parts;
    h0 = (int32_t)(group - i * parts) * HC;
  }
};

// One group of LPR lanes per row and HC heads, VE elements of K and of V of every head in each lane: all loads are in flight
// together, and the row's place in the cache is found once. d <= VE * LPR, d % VE == 0, every row VE elements aligned (to 16 bytes in
// the wider of the two types). Bound by the bytes that it reads and writes.
template <class TIn, class TC, int VE, int LPR, int HC>
__global__ void __launch_bounds__(kThreads) append_kernel(const RowsView rows, const CacheView c) {
  using Raw = typename RawOf<VE * (int)sizeof(TIn)>::type;
  const Task<LPR, HC> task(c);
  const int e0 = (threadIdx.x % LPR) * VE;
  const int64_t i = rows.first + task.i;
  const bool row = i < rows.n_rows, some = row && e0 < c.d;  // lanes without elements take part in the shuffles
  Raw raw[HC][2];
#pragma unroll
  for (int x = 0; x < HC; ++x) {
    raw[x][0] = raw[x][1] = Raw{};
    if (some && task.h0 + x < c.n_heads) {
      const int64_t h = task.h0 + x;
      raw[x][0] = __ldcs(reinterpret_cast<const Raw*>(reinterpret_cast<const TIn*>(rows.K) + i * rows.k_stride[0] + h * rows.k_stride[1] + e0));
      raw[x][1] = __ldcs(reinterpret_cast<const Raw*>(reinterpret_cast<const TIn*>(rows.V) + i * rows.v_stride[0] + h * rows.v_stride[1] + e0));
    }
  }
  Place at = {-1, 0};
  if (row) at = place_of(c, rows.cu_rows, i);
#pragma unroll
  for (int x = 0; x < HC; ++x) {
    const int64_t h = task.h0 + x;
    const bool here = some && at.page >= 0 && h < c.n_heads;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const Pages& pages = kv ? c.V : c.K;
      float y[VE];
      load_vec<TIn, VE>(reinterpret_cast<const TIn*>(&raw[x][kv]), y);
      bool none = false;
      if constexpr (IsByte<TC>::value) {
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < VE; ++e) top = max_nan(top, fabsf(y[e]));
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
        float inverse;
        const float scale = row_scale<TC>(top, inverse);
        none = scale != scale;
#pragma unroll
        for (int e = 0; e < VE; ++e) y[e] *= inverse;
        if (here && e0 == 0) pages.scale[pages.scale_at(at.page, at.slot, h)] = scale;
      }
      if (here) store_vec<TC, VE>(reinterpret_cast<TC*>(pages.data) + pages.at(at.page, at.slot, h) + e0, y, none);
    }
  }
}

// Any d, any alignment: one warp per row and head, element by element; the row is read twice where it is quantised.
template <class TIn, class TC>
__global__ void __launch_bounds__(kThreads) append_any_kernel(const RowsView rows, const CacheView c) {
  const uint32_t group = (blockIdx.x * (uint32_t)kThreads + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  const int64_t i = rows.first + group / c.n_heads;
  const int32_t h = (int32_t)(group % c.n_heads);
  if (i >= rows.n_rows) return;
  const Place at = place_of(c, rows.cu_rows, i);
  if (at.page < 0) return;
  auto one = [&](const TIn* src, const Pages& pages) {
    float inverse = 1.f;
    bool none = false;
    if constexpr (IsByte<TC>::value) {
      float top = 0.f;
      for (int e = lane; e < c.d; e += 32) top = max_nan(top, fabsf(up1(src[e])));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float scale = row_scale<TC>(top, inverse);
      none = scale != scale;
      if (lane == 0) pages.scale[pages.scale_at(at.page, at.slot, h)] = scale;
    }
    TC* dst = reinterpret_cast<TC*>(pages.data) + pages.at(at.page, at.slot, h);
    for (int e = lane; e < c.d; e += 32) down1(dst[e], none ? 0.f : up1(src[e]) * inverse);
  };
  one(reinterpret_cast<const TIn*>(rows.K) + i * rows.k_stride[0] + h * rows.k_stride[1], c.K);
  one(reinterpret_cast<const TIn*>(rows.V) + i * rows.v_stride[0] + h * rows.v_stride[1], c.V);
}

// The way back: x = q * scale in 32 bits, rounded once to the output's type. Same groups of lanes as append_kernel.
template <class TOut, class TC, int VE, int LPR, int HC>
__global__ void __launch_bounds__(kThreads) read_kernel(const RowsView rows, const CacheView c) {
  using Raw = typename RawOf<VE * (int)sizeof(TC)>::type;
  const Task<LPR, HC> task(c);
  const int e0 = (threadIdx.x % LPR) * VE;
  const int64_t i = rows.first + task.i;
  if (i >= rows.n_rows || e0 >= c.d) return;
  const Place at = place_of(c, rows.cu_rows, i);
  if (at.page < 0) return;
  Raw raw[HC][2];
  float scale[HC][2];
#pragma unroll
  for (int x = 0; x < HC; ++x) {
    const int64_t h = task.h0 + x;
    if (h >= c.n_heads) continue;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const Pages& pages = kv ? c.V : c.K;
      raw[x][kv] = *reinterpret_cast<const Raw*>(reinterpret_cast<const TC*>(pages.data) + pages.at(at.page, at.slot, h) + e0);
      if constexpr (IsByte<TC>::value) scale[x][kv] = pages.scale[pages.scale_at(at.page, at.slot, h)];
    }
  }
#pragma unroll
  for (int x = 0; x < HC; ++x) {
    const int64_t h = task.h0 + x;
    if (h >= c.n_heads) continue;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      float y[VE];
      load_vec<TC, VE>(reinterpret_cast<const TC*>(&raw[x][kv]), y);
      if constexpr (IsByte<TC>::value) {
#pragma unroll
        for (int e = 0; e < VE; ++e) y[e] *= scale[x][kv];
      }
      TOut* dst = kv ? reinterpret_cast<TOut*>(rows.V) + i * rows.v_stride[0] + h * rows.v_stride[1]
                     : reinterpret_cast<TOut*>(rows.K) + i * rows.k_stride[0] + h * rows.k_stride[1];
      store_vec<TOut, VE>(dst + e0, y);
    }
  }
}

template <class TOut, class TC>
__global__ void __launch_bounds__(kThreads) read_any_kernel(const RowsView rows, const CacheView c) {
  const uint32_t group = (blockIdx.x * (uint32_t)kThreads + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  const int64_t i = rows.first + group / c.n_heads;
  const int32_t h = (int32_t)(group % c.n_heads);
  if (i >= rows.n_rows) return;
  const Place at = place_of(c, rows.cu_rows, i);
  if (at.page < 0) return;
  auto one = [&](const Pages& pages, TOut* dst) {
    float scale = 1.f;
    if constexpr (IsByte<TC>::value) scale = pages.scale[pages.scale_at(at.page, at.slot, h)];
    const TC* src = reinterpret_cast<const TC*>(pages.data) + pages.at(at.page, at.slot, h);
    for (int e = lane; e < c.d; e += 32) down1(dst[e], up1(src[e]) * scale);
  };
  one(c.K, reinterpret_cast<TOut*>(rows.K) + i * rows.k_stride[0] + h * rows.k_stride[1]);
  one(c.V, reinterpret_cast<TOut*>(rows.V) + i * rows.v_stride[0] + h * rows.v_stride[1]);
}

// Position lens[b] + i := position lens[b] + kept[b][i] for i < n_kept[b], `kept` ascending. One block per sequence and head
// walks the rows in order, a chunk at a time: everything of a chunk is in registers before any of it is stored, and what an
// earlier chunk stored (positions below the chunk's first i) is no source of a later one, because kept[i] >= i. Rows are moved
// as units of type U (a divisor of the row's bytes and of every address).
template <class U>
__global__ void __launch_bounds__(128) keep_kernel(const CacheView c, const int32_t* __restrict__ kept, int64_t width,
                                                   const int32_t* __restrict__ n_kept, int32_t elem_bytes) {
  constexpr int kUnits = 4;  // of K and of V in a thread
  const int32_t b = (int32_t)(blockIdx.x / (uint32_t)c.n_heads), h = (int32_t)(blockIdx.x % (uint32_t)c.n_heads);
  const int64_t first = __ldg(c.lens + b);
  int64_t n = __ldg(n_kept + b);
  n = n < 0 ? 0 : (n < width ? n : width);
  const int32_t per_row = c.d * elem_bytes / (int32_t)sizeof(U);
  const int64_t total = n * per_row;
  for (int64_t base = 0; base < total; base += 128 * kUnits) {
    U k[kUnits], v[kUnits];
    float sk[kUnits], sv[kUnits];
    int64_t to_k[kUnits], to_v[kUnits], to_sk[kUnits], to_sv[kUnits];
#pragma unroll
    for (int x = 0; x < kUnits; ++x) {
      const int64_t t = base + x * 128 + threadIdx.x;
      to_k[x] = -1;
      to_sk[x] = -1;
      if (t >= total) continue;
      const int64_t i = t / per_row;
      const int32_t u = (int32_t)(t - i * per_row);
      const int32_t j = __ldg(kept + (int64_t)b * width + i);
      const int64_t src = first + j, dst = first + i;
      const int32_t sp = (j < 0 || j == i) ? -1 : c.page_of(b, src), dp = c.page_of(b, dst);
      if (sp < 0 || dp < 0) continue;
      const int32_t ss = c.slot_of(src), ds = c.slot_of(dst);
      k[x] = reinterpret_cast<const U*>(c.K.data + c.K.at(sp, ss, h) * elem_bytes)[u];
      v[x] = reinterpret_cast<const U*>(c.V.data + c.V.at(sp, ss, h) * elem_bytes)[u];
      to_k[x] = c.K.at(dp, ds, h) * elem_bytes + u * (int64_t)sizeof(U);
      to_v[x] = c.V.at(dp, ds, h) * elem_bytes + u * (int64_t)sizeof(U);
      if (u == 0 && c.K.scale) {
        sk[x] = c.K.scale[c.K.scale_at(sp, ss, h)];
        sv[x] = c.V.scale[c.V.scale_at(sp, ss, h)];
        to_sk[x] = c.K.scale_at(dp, ds, h);
        to_sv[x] = c.V.scale_at(dp, ds, h);
      }
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < kUnits; ++x) {
      if (to_k[x] >= 0) {
        *reinterpret_cast<U*>(c.K.data + to_k[x]) = k[x];
        *reinterpret_cast<U*>(c.V.data + to_v[x]) = v[x];
      }
      if (to_sk[x] >= 0) {
        c.K.scale[to_sk[x]] = sk[x];
        c.V.scale[to_sv[x]] = sv[x];
      }
    }
    __syncthreads();
  }
}

}  // namespace cache
}  // namespace spfa
