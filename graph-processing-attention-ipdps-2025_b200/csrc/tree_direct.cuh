// Tree attention of small calls in one launch: every drafted token walks all keys of its sequence itself, committed and drafted ones
// alike, without pieces and without a second kernel. What counts here is the chain of dependent latencies.
//
// One CTA per token and key head, up to eight query heads of it at a time (the rows). A warp takes 32 keys at a time: their K and V
// rows are all requested at once (cp.async into the warp's own shared memory), then a lane owns a key for the scores (broadcast reads
// of Q, no shuffles), and P V goes key by key with the columns spread over the lanes. The warps' states meet in shared memory at the
// end. All arithmetic is in 32 bits. One token of 8 heads over 500 keys of 64: 10.2 us, where the two kernels took 14.3.
#pragma once
#include "tree_kernels.cuh"

namespace spfa {
namespace tree {

constexpr int kDirectRows = 8;

// Shared memory of a call: Q, then K and V of 32 keys for each warp (rows 16 bytes further round the banks), then the warps' states.
struct DirectPlan {
  int units, pitch, warps;  // 16-byte units of a cache row, bytes from row to row, warps of a CTA
  int kv_bytes, bytes;      // of a warp's K and V, of everything
  __host__ __device__ explicit DirectPlan(int row_bytes) {
    units = row_bytes / 16;
    pitch = (units | 1) * 16;
    warps = row_bytes <= 128 ? 16 : row_bytes <= 256 ? 8 : 4;
    kv_bytes = 2 * 32 * pitch;
    bytes = kDirectRows * 128 * 4 + warps * kv_bytes + warps * kDirectRows * (8 + 128 * 4);
  }
};

// d <= 128; rows of the cache are whole 16-byte units, rows of Q and O whole 4-element pieces. R: rows of a CTA (query heads of its
// key head), the last ones idle where the group does not fill them.
template <class TQ, class TC, int R>
__global__ void __launch_bounds__(512) direct_kernel(const Call a, const MergeArgs g) {
  constexpr int DP = 128, VE = 16 / (int)sizeof(TC);
  extern __shared__ __align__(16) uint8_t smem[];
  const DirectPlan plan(a.c.d * (int)sizeof(TC));
  const int W = plan.warps;
  float* q_s = reinterpret_cast<float*>(smem);  // [R][DP]
  uint8_t* kv = smem + kDirectRows * DP * 4;
  float2* ml_s = reinterpret_cast<float2*>(kv + W * plan.kv_bytes);  // [W][R]
  float* o_s = reinterpret_cast<float*>(ml_s + W * R);               // [W][R][DP]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = a.c.d;
  const uint32_t parts = (uint32_t)(a.group + R - 1) / R, rest = blockIdx.x / parts;
  const int32_t h = (int32_t)(rest % (uint32_t)a.c.n_heads);
  const int64_t n = rest / (uint32_t)a.c.n_heads;
  const int32_t row0 = (int32_t)(blockIdx.x - rest * parts) * R, rows = min(R, a.group - row0), hq0 = h * a.group + row0;
  // requested first, needed last
  constexpr int QN = R * DP / 4 / 128 > 0 ? R * DP / 4 / 128 : 1;  // four columns each; at least 128 threads
  float q[QN][4];
#pragma unroll
  for (int i = 0; i < QN; ++i) {
    const int x = i * W * 32 + threadIdx.x, r = x / (DP / 4), e = x % (DP / 4) * 4;
#pragma unroll
    for (int k = 0; k < 4; ++k) q[i][k] = 0.f;
    if (r < rows && e < d) load_vec<TQ, 4>(reinterpret_cast<const TQ*>(a.Q) + n * a.q_stride[0] + (int64_t)(hq0 + r) * a.q_stride[1] + e, q[i]);
  }
  const int32_t b = sequence_of(a.cu_rows, a.c.n_seq, n);
  if (b < 0) return;
  int64_t begin, end;
  rows_of(a.cu_rows, b, a.n_rows, begin, end);
  const int64_t len = a.c.len_of(b), tokens = end - begin, total = len + (tokens < g.mask_width ? tokens : g.mask_width);

  float m[R], l[R], o[R][4];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = neg_inf();
    l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[r][e] = 0.f;
  }
  uint8_t* k_s = kv + warp * plan.kv_bytes;
  uint8_t* v_s = k_s + 32 * plan.pitch;
  int lpr = 1;  // lanes that copy a row
  while (lpr < plan.units) lpr *= 2;
  const int u = lane & (lpr - 1), first = lane / lpr, step = 32 / lpr;
  bool q_stored = false;
  for (int64_t p0 = (int64_t)warp * 32;; p0 += W * 32) {
    const bool here = p0 < total;
    const int64_t p = p0 + lane;
    bool on = false;
    float fk = 1.f, fv = 1.f;
    if (here) {
      const int32_t page = p < total ? a.c.page_of(b, p) : -1;
      on = page >= 0 && (p < len || __ldg(g.mask + n * g.mask_width + (p - len)) != 0);
      const int32_t slot = on ? a.c.slot_of(p) : 0;
      const unsigned some = __ballot_sync(kFullMask, on);
      const int64_t k_at = on ? a.c.K.at(page, slot, h) : 0, v_at = on ? a.c.V.at(page, slot, h) : 0;
#pragma unroll 2
      for (int r = first; r < 32; r += step) {
        const int64_t ka = __shfl_sync(kFullMask, k_at, r), va = __shfl_sync(kFullMask, v_at, r);
        if (u < plan.units) {
          const uint32_t to = (uint32_t)__cvta_generic_to_shared(k_s + r * plan.pitch + u * 16), bytes = (some >> r) & 1u ? 16 : 0;
          // keys that nobody sees become zeros, whatever lies there
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(reinterpret_cast<const TC*>(a.c.K.data) + ka + u * VE),
                       "r"(bytes) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + 32 * plan.pitch),
                       "l"(reinterpret_cast<const TC*>(a.c.V.data) + va + u * VE), "r"(bytes) : "memory");
        }
      }
      if constexpr (IsByte<TC>::value) {
        fk = fv = 0.f;
        if (on) {
          fk = a.c.K.scale[a.c.K.scale_at(page, slot, h)];
          fv = a.c.V.scale[a.c.V.scale_at(page, slot, h)];
        }
      }
    }
    if (!q_stored) {
#pragma unroll
      for (int i = 0; i < QN; ++i) {
        const int x = i * W * 32 + threadIdx.x;
        if (x < R * DP / 4) reinterpret_cast<float4*>(q_s)[x] = make_float4(q[i][0], q[i][1], q[i][2], q[i][3]);
      }
      __syncthreads();
      q_stored = true;
    }
    if (!here) break;
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    float s[R];
#pragma unroll
    for (int r = 0; r < R; ++r) s[r] = 0.f;
#pragma unroll 2
    for (int x = 0; x < plan.units; ++x) {
      float k[VE];
      load_vec<TC, VE>(reinterpret_cast<const TC*>(k_s + lane * plan.pitch + x * 16), k);
      if constexpr (IsByte<TC>::value) {
#pragma unroll
        for (int i = 0; i < VE; ++i) k[i] *= fk;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int i = 0; i < VE; i += 4) {
          const float4 y = *reinterpret_cast<const float4*>(q_s + r * DP + x * VE + i);
          s[r] = fmaf(y.x, k[i], fmaf(y.y, k[i + 1], fmaf(y.z, k[i + 2], fmaf(y.w, k[i + 3], s[r]))));
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[r] = on ? s[r] * a.scale_log2e : neg_inf();
      float top = s[r];
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) top = max_nan(top, __shfl_xor_sync(kFullMask, top, x));
      top = max_nan(top, m[r]);
      const float ref = top == neg_inf() ? 0.f : top, f = fast_exp2(m[r] - ref);
      s[r] = fast_exp2(s[r] - ref);  // now the probability; the lanes' sums are added up last
      l[r] = l[r] * f + s[r];
      m[r] = top;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[r][e] *= f;
    }
#pragma unroll 8
    for (int key = 0; key < 32; ++key) {
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      if (lane * 4 < d) load_vec<TC, 4>(reinterpret_cast<const TC*>(v_s + key * plan.pitch) + lane * 4, v);
      if constexpr (IsByte<TC>::value) {
        const float f = __shfl_sync(kFullMask, fv, key);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= f;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float pr = __shfl_sync(kFullMask, s[r], key);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[r][e] = fmaf(pr, v[e], o[r][e]);
      }
    }
    __syncwarp();  // the next keys are copied over these
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float sum = l[r];
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(kFullMask, sum, x);
    if (lane == 0) ml_s[warp * R + r] = make_float2(m[r], sum);
    *reinterpret_cast<float4*>(o_s + (warp * R + r) * DP + lane * 4) = make_float4(o[r][0], o[r][1], o[r][2], o[r][3]);
  }
  __syncthreads();
  for (int r = warp; r < rows; r += W) {  // a warp finishes a row
    const float2 ml = lane < W ? ml_s[lane * R + r] : make_float2(neg_inf(), 0.f);
    float M = ml.x, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) M = max_nan(M, __shfl_xor_sync(kFullMask, M, x));
    M = __shfl_sync(kFullMask, M, 0);  // W is at most 16
    const float f = fast_exp2(ml.x - (M == neg_inf() ? 0.f : M));
    float L = ml.y * f;
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) L += __shfl_xor_sync(kFullMask, L, x);
    L = __shfl_sync(kFullMask, L, 0);
#pragma unroll 4
    for (int x = 0; x < W; ++x) {
      const float fx = __shfl_sync(kFullMask, f, x);
      const float4 y = *reinterpret_cast<const float4*>(o_s + (x * R + r) * DP + lane * 4);
      acc[0] = fmaf(fx, y.x, acc[0]);
      acc[1] = fmaf(fx, y.y, acc[1]);
      acc[2] = fmaf(fx, y.z, acc[2]);
      acc[3] = fmaf(fx, y.w, acc[3]);
    }
    finish_row<TQ, 4, 1>(a, g, n, hq0 + r, lane, M, L, acc);
  }
}

}  // namespace tree
}  // namespace spfa
