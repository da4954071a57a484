// Attention of drafted token trees over a paged cache.
//
// Row i of sequence b (one query head of one drafted token) sees every committed key [0, len_b) and, of the drafted rows, the
// keys len_b + j that tree_mask names. That is a dense part and a few entries, and they are computed apart:
//
//   context kernel  softmax partials over the committed keys. All rows see all of them, so there is no mask; the g query heads
//                   of a key head and the tokens of a sequence are the rows of one product. (b, key head, row tile) is a unit;
//                   the units' key tiles, one after the other, are one long list that is cut evenly over the CTAs of one
//                   wave, whatever the lengths are: lens and cu_rows are read on the device. A piece (unit x CTA) leaves an
//                   un-normalised O row with its maximum and sum in the workspace.
//   merge kernel    one warp per row: the drafted keys that its mask names, its pieces, the incoming (m, l, O), and the store.
//
// Scores are kept in units of log2: s2 = (q . k) log2(e) / sqrt(d).
#pragma once
#include "cache_common.cuh"
#include "spfa_common.cuh"

namespace spfa {
namespace tree {

struct Call {
  CacheView c;
  const char* Q;
  int64_t q_stride[2];  // elements from row to row, head to head
  const int32_t* cu_rows;
  int64_t n_rows;
  int32_t n_q_heads, group;  // group = query heads of a key head
  float scale_log2e;
  // cutting the list of key tiles
  int32_t row_tile, tile_keys;  // rows that a CTA has room for, keys of a tile
  int32_t unit_rows;            // rows of a unit: whole tokens where row_tile holds one
  int32_t page_tiles;           // tiles of a page (pages of tile_keys positions and more), 0: a tile spans whole pages
  int32_t n_cta;                // grid of the context kernel
  int32_t direct;               // the call runs as one launch of direct_kernel
  // workspace
  int64_t* cut;   // [0]: tiles per CTA, [1 + b]: first tile of sequence b in the list
  float2* ml;     // maximum and sum of a piece's row
  float* O;       // [rows][d_pad]
  int32_t d_pad;

  __host__ __device__ __forceinline__ int64_t tiles_of(int64_t len) const {
    if (page_tiles == 0) return (len + tile_keys - 1) / tile_keys;
    const int64_t full = len / c.page_size, rest = len - full * c.page_size;
    return full * page_tiles + (rest + tile_keys - 1) / tile_keys;
  }
  __device__ __forceinline__ int64_t row_tiles(int64_t tokens) const { return (tokens * group + unit_rows - 1) / unit_rows; }
  // Key tiles of all units of sequence b.
  __device__ __forceinline__ int64_t weight(int32_t b) const {
    int64_t begin, end;
    rows_of(cu_rows, b, n_rows, begin, end);
    return end == begin ? 0 : tiles_of(c.len_of(b)) * row_tiles(end - begin) * c.n_heads;
  }
  // First partial row of local row x of key head h in CTA `cta`: rows of a sequence lie together, the CTAs of a row row_tile
  // apart. Pieces follow each other with growing unit or growing CTA, so no two of them meet.
  __device__ __forceinline__ int64_t partial_row(int64_t begin, int64_t tokens, int32_t h, int64_t x, int64_t cta) const {
    return begin * n_q_heads + (int64_t)h * tokens * group + x + cta * row_tile;
  }
};

struct Cut {  // what block_cut leaves in shared memory
  int64_t first, last;  // this CTA's key tiles in the list
  int64_t start;        // first tile of sequence b
  int32_t b;
  int64_t warp_sum[32];
};

// Finds this CTA's share of the list (all NT threads). CTA 0 leaves the starts of the sequences for the merge kernel.
template <int NT>
__device__ __forceinline__ void block_cut(const Call& a, Cut* s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int32_t n_seq = a.c.n_seq;
  int64_t own = 0;  // of sequence threadIdx.x; kept, as most calls have no more sequences than threads
  int64_t sum = 0;
  for (int32_t b = threadIdx.x; b < n_seq; b += NT) {
    const int64_t w = a.weight(b);
    if (b == (int32_t)threadIdx.x) own = w;
    sum += w;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
  if (lane == 0) s->warp_sum[warp] = sum;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) total += s->warp_sum[w];
  int64_t chunk = (total + a.n_cta - 1) / a.n_cta;
  const int64_t first = (int64_t)blockIdx.x * chunk;
  if (threadIdx.x == 0) {
    s->first = first < total ? first : total;
    s->last = first + chunk < total ? first + chunk : total;
    s->b = n_seq;
    if (blockIdx.x == 0) a.cut[0] = chunk;
  }
  __syncthreads();
  int64_t base = 0;
  for (int32_t b0 = 0; b0 < n_seq; b0 += NT) {
    const int32_t b = b0 + (int32_t)threadIdx.x;
    const int64_t w = b0 == 0 ? own : (b < n_seq ? a.weight(b) : 0);
    int64_t x = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(kFullMask, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s->warp_sum[warp] = x;
    __syncthreads();
    int64_t before = base;
    for (int w2 = 0; w2 < NT / 32; ++w2) {
      if (w2 < warp) before += s->warp_sum[w2];
      base += s->warp_sum[w2];
    }
    const int64_t start = before + x - w;
    if (blockIdx.x == 0 && b < n_seq) a.cut[1 + b] = start;
    if (w > 0 && s->first >= start && s->first < start + w) {  // one thread at most
      s->b = b;
      s->start = start;
    }
    __syncthreads();
  }
}

// Walks the pieces of a CTA: piece = consecutive key tiles [t0, t0 + n) of one unit. Every role of a CTA walks on its own. Rows, key
// tiles of a sequence and positions fit in 32 bits, the list does not have to.
struct Walk {
  int64_t at, last, start, weight;
  int32_t b, h, begin, tokens, len, tiles;
  int32_t row0;  // first row of the unit's row tile among the tokens * group rows of the key head
  int32_t t0, n;

  __device__ __forceinline__ void open(const Call& a) {
    int64_t x, y;
    rows_of(a.cu_rows, b, a.n_rows, x, y);
    begin = (int32_t)x;
    tokens = (int32_t)(y - x);
    len = (int32_t)a.c.len_of(b);
    tiles = (int32_t)a.tiles_of(len);
    weight = tokens ? tiles * a.row_tiles(tokens) * a.c.n_heads : 0;
  }
  __device__ __forceinline__ void init(const Call& a, const Cut* s) {
    at = s->first;
    last = s->last;
    b = s->b;
    start = s->start;
    n = 0;
    if (at < last) open(a);
  }
  // The next piece; false behind the last one.
  __device__ __forceinline__ bool next(const Call& a) {
    at += n;
    if (at >= last) return false;
    while (at >= start + weight) {  // ends: `at` is below the list's total
      start += weight;
      ++b;
      open(a);
    }
    const uint64_t in = (uint64_t)(at - start);
    const uint32_t u = (uint32_t)(in / (uint32_t)tiles);
    t0 = (int32_t)(in - (uint64_t)u * (uint32_t)tiles);
    n = tiles - t0 < last - at ? tiles - t0 : (int32_t)(last - at);
    const uint32_t rt = (uint32_t)a.row_tiles(tokens);
    h = (int32_t)(u / rt);
    row0 = (int32_t)(u - (uint32_t)h * rt) * a.unit_rows;
    return true;
  }
  __device__ __forceinline__ int rows(const Call& a) const {  // of the unit
    const int32_t left = tokens * a.group - row0;
    return left < a.unit_rows ? left : a.unit_rows;
  }
};

// ---- context kernel without tensor cores: 32-bit products, any types and any d ---------------------------------------------
//
// 256 threads, 16 or 32 rows, TK keys at a time in shared memory as 32-bit values. Shared memory feeds the products, so a thread takes
// many rows: for the scores 8 rows x 2 keys of a slice of d (d <= 128; a warp reads 64 keys, and Q by broadcast), for P V 8 rows x 4
// columns of O in registers and a share of the keys. Larger d leaves room for fewer keys: 4 rows x 2 keys, 4 rows x 4 columns. Pairs of
// products share an instruction. A tile is a chain of short phases between barriers; other CTAs of the SM fill its gaps.
// float32, 4 sequences of 16 drafted tokens, 2 heads a key head, up to 4096 keys, d = 64: 30 us with the merge, 0.8 TB/s: 2.5 tiles for a CTA,
// so that the chain of a tile's phases counts. 64 sequences of one token over 2000 keys of 8 heads of 128: 520 us,
// 2.0 TB/s.
__host__ __device__ constexpr int any_tile_keys(int dp) { return dp <= 128 ? 64 : (dp == 256 ? 32 : 16); }
template <int DP, int R>
struct PlanAny {
  static constexpr int kThreads = 256, kRows = R;
  static constexpr int kCtasPerSm = DP <= 256 ? 2 : 1;
  static constexpr int TK = any_tile_keys(DP);
  // scores: KB blocks of keys x RB blocks of rows x DS slices of d = 8 warps; TR rows of a thread, here and in P V
  static constexpr bool kTall = TK == 64;
  static constexpr int TR = kTall ? 8 : 4, KB = kTall ? 1 : TK / 16, RB = kTall ? R / 8 : R / 16, DS = 8 / (KB * RB);
  static constexpr int RG = R / TR, CGT = DP / 4 < 64 ? DP / 4 : 64, NCG = DP / 4 / CGT, KS = 256 / (RG * CGT);
  static constexpr int kPitch = DP + 4;  // floats: rows start 16 bytes further round the banks
  static constexpr int kPitchP = R + 4;
  static constexpr int kOffQ = 0, kOffK = kOffQ + kRows * kPitch * 4, kOffV = kOffK + TK * kPitch * 4;
  static constexpr int kOffS = kOffV + TK * kPitch * 4, kOffP = kOffS + DS * kRows * TK * 4, kOffRow = kOffP + TK * kPitchP * 4;
  static constexpr int kOffKey = kOffRow + 3 * kRows * 4, kOffCut = kOffKey + TK * 24, kBytes = kOffCut + (int)sizeof(Cut);
  static_assert(DS >= 1 && KS >= 1, "every warp has work");
  static_assert(KS * kRows * DP <= (TK * kPitch) * 2, "the shares of O are added up where K and V were");
};

// Two products and sums in one instruction.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ uint64_t pair_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float2 halves(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}

template <int DP, int R, class TQ, class TC>
__global__ void __launch_bounds__(256, PlanAny<DP, R>::kCtasPerSm) context_any_kernel(const Call a, const int vec) {
  using P = PlanAny<DP, R>;
  constexpr int TK = P::TK, PITCH = P::kPitch, PP = P::kPitchP;
  extern __shared__ __align__(16) uint8_t smem[];
  float* Qs = reinterpret_cast<float*>(smem + P::kOffQ);
  float* Ks = reinterpret_cast<float*>(smem + P::kOffK);
  float* Vs = reinterpret_cast<float*>(smem + P::kOffV);
  float* Ss = reinterpret_cast<float*>(smem + P::kOffS);
  float* Ps = reinterpret_cast<float*>(smem + P::kOffP);  // [key][PP]
  float* row_m = reinterpret_cast<float*>(smem + P::kOffRow);
  float* row_l = row_m + R;
  float* row_f = row_l + R;
  int64_t* k_at = reinterpret_cast<int64_t*>(smem + P::kOffKey);
  int64_t* v_at = k_at + TK;
  float* k_sc = reinterpret_cast<float*>(v_at + TK);
  float* v_sc = k_sc + TK;
  Cut* cut = reinterpret_cast<Cut*>(smem + P::kOffCut);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int d = a.c.d;

  block_cut<256>(a, cut);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Walk w;
  w.init(a, cut);
  while (w.next(a)) {
    const int rows = w.rows(a);
    __syncthreads();
    for (int x = tid; x < R * (DP / 4); x += 256) {
      const int r = x / (DP / 4), e = (x % (DP / 4)) * 4;
      float q[4] = {0.f, 0.f, 0.f, 0.f};
      if (r < rows) {
        const int32_t xr = w.row0 + r, t = xr / a.group;
        const TQ* src = reinterpret_cast<const TQ*>(a.Q) + (int64_t)(w.begin + t) * a.q_stride[0] +
                        (w.h * (int64_t)a.group + (xr - t * a.group)) * a.q_stride[1];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (e + i < d) q[i] = up1(src[e + i]);
      }
      *reinterpret_cast<float4*>(Qs + r * PITCH + e) = make_float4(q[0], q[1], q[2], q[3]);
    }
    if (tid < R) {
      row_m[tid] = neg_inf();
      row_l[tid] = 0.f;
    }
    constexpr int TR = P::TR;
    uint64_t o[TR][P::NCG][2];  // pairs of columns
#pragma unroll
    for (int r = 0; r < TR; ++r)
#pragma unroll
      for (int g = 0; g < P::NCG; ++g) o[r][g][0] = o[r][g][1] = 0ull;
    const int cg = tid % P::CGT, rg = tid / P::CGT % P::RG, ks = tid / (P::RG * P::CGT);

    auto page_at = [&](int32_t t) -> int32_t {  // of this thread's key of tile t: looked up a tile ahead
      const int64_t p = (int64_t)t * TK + tid;
      return tid < TK && t < w.t0 + w.n && p < w.len ? a.c.page_of(w.b, p) : -1;
    };
    int32_t next_page = page_at(w.t0);
    for (int32_t t = w.t0; t < w.t0 + w.n; ++t) {
      __syncthreads();  // the last tile's K, V and P are done with
      const int32_t page = next_page;
      next_page = page_at(t + 1);
      if (tid < TK) {
        const int64_t p = (int64_t)t * TK + tid;
        k_at[tid] = -1;
        if (page >= 0) {
          const int32_t slot = a.c.slot_of(p);
          k_at[tid] = a.c.K.at(page, slot, w.h);
          v_at[tid] = a.c.V.at(page, slot, w.h);
          if constexpr (IsByte<TC>::value) {
            k_sc[tid] = a.c.K.scale[a.c.K.scale_at(page, slot, w.h)];
            v_sc[tid] = a.c.V.scale[a.c.V.scale_at(page, slot, w.h)];
          }
        }
      }
      __syncthreads();
#pragma unroll 4
      for (int x = tid; x < TK * (DP / 4); x += 256) {
        const int key = x / (DP / 4), e = (x % (DP / 4)) * 4;
        float k[4] = {0.f, 0.f, 0.f, 0.f}, v[4] = {0.f, 0.f, 0.f, 0.f};
        const int64_t ka = k_at[key];
        if (ka >= 0) {
          const TC* kp = reinterpret_cast<const TC*>(a.c.K.data) + ka + e;
          const TC* vp = reinterpret_cast<const TC*>(a.c.V.data) + v_at[key] + e;
          if (vec) {  // d and every stride divide by 4
            if (e < d) {
              load_vec<TC, 4>(kp, k);
              load_vec<TC, 4>(vp, v);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (e + i < d) {
                k[i] = up1(kp[i]);
                v[i] = up1(vp[i]);
              }
          }
          if constexpr (IsByte<TC>::value) {
            const float fk = k_sc[key], fv = v_sc[key];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              k[i] *= fk;
              v[i] *= fv;
            }
          }
        }
        *reinterpret_cast<float4*>(Ks + key * PITCH + e) = make_float4(k[0], k[1], k[2], k[3]);
        *reinterpret_cast<float4*>(Vs + key * PITCH + e) = make_float4(v[0], v[1], v[2], v[3]);
      }
      __syncthreads();
      if constexpr (P::kTall) {  // scores
        const int rb = warp % P::RB, ds = warp / P::RB;
        const float* qp = Qs + rb * 8 * PITCH + ds * (DP / P::DS);
        const float* kp = Ks + lane * PITCH + ds * (DP / P::DS);
        uint64_t s[8][2] = {};
#pragma unroll 2
        for (int e = 0; e < DP / P::DS; e += 4) {
          const ulonglong2 k0 = *reinterpret_cast<const ulonglong2*>(kp + e);
          const ulonglong2 k1 = *reinterpret_cast<const ulonglong2*>(kp + 32 * PITCH + e);
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(qp + r * PITCH + e);
            s[r][0] = pair_fma(q.y, k0.y, pair_fma(q.x, k0.x, s[r][0]));
            s[r][1] = pair_fma(q.y, k1.y, pair_fma(q.x, k1.x, s[r][1]));
          }
        }
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const float2 x = halves(s[r][0]), y = halves(s[r][1]);
          Ss[(ds * R + rb * 8 + r) * TK + lane] = x.x + x.y;
          Ss[(ds * R + rb * 8 + r) * TK + lane + 32] = y.x + y.y;
        }
      } else {
        const int kb = warp % P::KB, rb = warp / P::KB % P::RB, ds = warp / (P::KB * P::RB), r0 = rb * 16 + (lane >> 3) * 4, kg = lane & 7;
        const float* qp = Qs + r0 * PITCH + ds * (DP / P::DS);
        const float* kp = Ks + (kb * 16 + kg) * PITCH + ds * (DP / P::DS);
        uint64_t s[4][2] = {};
#pragma unroll 4
        for (int e = 0; e < DP / P::DS; e += 4) {
          const ulonglong2 k0 = *reinterpret_cast<const ulonglong2*>(kp + e);
          const ulonglong2 k1 = *reinterpret_cast<const ulonglong2*>(kp + 8 * PITCH + e);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(qp + r * PITCH + e);
            s[r][0] = pair_fma(q.y, k0.y, pair_fma(q.x, k0.x, s[r][0]));
            s[r][1] = pair_fma(q.y, k1.y, pair_fma(q.x, k1.x, s[r][1]));
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float2 x = halves(s[r][0]), y = halves(s[r][1]);
          Ss[(ds * R + r0 + r) * TK + kb * 16 + kg] = x.x + x.y;
          Ss[(ds * R + r0 + r) * TK + kb * 16 + kg + 8] = y.x + y.y;
        }
      }
      __syncthreads();
      {  // softmax: a warp takes two rows or four, side by side
        constexpr int KL = (TK + 31) / 32, N = R / 8;
        float x[N][KL], top[N], m_old[N], sum[N];
#pragma unroll
        for (int rr = 0; rr < N; ++rr) {
          const int r = warp * N + rr;
          top[rr] = m_old[rr] = row_m[r];
#pragma unroll
          for (int i = 0; i < KL; ++i) {
            const int key = lane + 32 * i;
            x[rr][i] = neg_inf();
            if (key < TK && k_at[key] >= 0) {
              float y = 0.f;
#pragma unroll
              for (int ds = 0; ds < P::DS; ++ds) y += Ss[(ds * R + r) * TK + key];
              x[rr][i] = y * a.scale_log2e;
            }
            top[rr] = max_nan(top[rr], x[rr][i]);
          }
        }
#pragma unroll
        for (int o2 = 16; o2 > 0; o2 >>= 1)
#pragma unroll
          for (int rr = 0; rr < N; ++rr) top[rr] = max_nan(top[rr], __shfl_xor_sync(kFullMask, top[rr], o2));
#pragma unroll
        for (int rr = 0; rr < N; ++rr) {
          const float ref = top[rr] == neg_inf() ? 0.f : top[rr];  // nothing seen yet: every exponent stays -inf
          sum[rr] = 0.f;
#pragma unroll
          for (int i = 0; i < KL; ++i) {
            const int key = lane + 32 * i;
            const float p = fast_exp2(x[rr][i] - ref);
            sum[rr] += p;
            if (key < TK) Ps[key * PP + warp * N + rr] = p;
          }
        }
#pragma unroll
        for (int o2 = 16; o2 > 0; o2 >>= 1)
#pragma unroll
          for (int rr = 0; rr < N; ++rr) sum[rr] += __shfl_xor_sync(kFullMask, sum[rr], o2);
        if (lane == 0) {
#pragma unroll
          for (int rr = 0; rr < N; ++rr) {
            const int r = warp * N + rr;
            const float f = fast_exp2(m_old[rr] - (top[rr] == neg_inf() ? 0.f : top[rr]));
            row_f[r] = f;
            row_l[r] = row_l[r] * f + sum[rr];
            row_m[r] = top[rr];
          }
        }
      }
      __syncthreads();
      {  // O = O f + P V
#pragma unroll
        for (int r = 0; r < TR; ++r) {
          const float f = row_f[rg * TR + r];
          const uint64_t f2 = pair(f, f);
#pragma unroll
          for (int g = 0; g < P::NCG; ++g)
#pragma unroll
            for (int i = 0; i < 2; ++i) o[r][g][i] = pair_fma(o[r][g][i], f2, 0ull);
        }
        constexpr int KPS = TK / P::KS;
#pragma unroll 2
        for (int key = ks * KPS; key < ks * KPS + KPS; ++key) {
          uint64_t p2[TR];
#pragma unroll
          for (int r = 0; r < TR; r += 4) {
            const float4 p = *reinterpret_cast<const float4*>(Ps + key * PP + rg * TR + r);
            p2[r] = pair(p.x, p.x);
            p2[r + 1] = pair(p.y, p.y);
            p2[r + 2] = pair(p.z, p.z);
            p2[r + 3] = pair(p.w, p.w);
          }
#pragma unroll
          for (int g = 0; g < P::NCG; ++g) {
            const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(Vs + key * PITCH + (g * P::CGT + cg) * 4);
#pragma unroll
            for (int r = 0; r < TR; ++r) {
              o[r][g][0] = pair_fma(p2[r], v.x, o[r][g][0]);
              o[r][g][1] = pair_fma(p2[r], v.y, o[r][g][1]);
            }
          }
        }
      }
    }
    // the shares of the keys are added up where K and V were, then the rows leave
    __syncthreads();
    float* Os = Ks;
#pragma unroll
    for (int r = 0; r < TR; ++r)
#pragma unroll
      for (int g = 0; g < P::NCG; ++g)
        *reinterpret_cast<ulonglong2*>(Os + (ks * R + rg * TR + r) * DP + (g * P::CGT + cg) * 4) = make_ulonglong2(o[r][g][0], o[r][g][1]);
    __syncthreads();
    const int64_t out = a.partial_row(w.begin, w.tokens, w.h, w.row0, blockIdx.x);
    for (int x = tid; x < rows * (DP / 4); x += 256) {
      const int r = x / (DP / 4), e = (x % (DP / 4)) * 4;
      if (e >= a.d_pad) continue;
      float4 y = *reinterpret_cast<const float4*>(Os + r * DP + e);
#pragma unroll
      for (int s2 = 1; s2 < P::KS; ++s2) {
        const float4 z = *reinterpret_cast<const float4*>(Os + (s2 * R + r) * DP + e);
        y = make_float4(y.x + z.x, y.y + z.y, y.z + z.z, y.w + z.w);
      }
      *reinterpret_cast<float4*>(a.O + (out + r) * a.d_pad + e) = y;
    }
    if (tid < rows) a.ml[out + tid] = make_float2(row_m[tid], row_l[tid]);
  }
}

// ---- merge kernel -----------------------------------------------------------------------------------------------------------
//
// One warp per token and GR query heads of a key head (the rows); a lane holds columns (i * 32 + lane) * VE. The drafted keys come
// first: they need nothing of the context kernel, so their loads run while it drains. A warp is a chain of dependent loads, so many
// are in flight together: four keys of K and of V, and the pieces' O rows eight at a time. Four rows share the loads of K and V and the
// lookups; calls that leave the machine empty take one row a warp instead (kMergeRows).
struct MergeArgs {
  const uint8_t* mask;
  int64_t mask_width;
  float *m, *l;
  char* O;
  int64_t o_stride[2];
  int first;
};

// The last of a row (one warp): its keys' maximum M, sum L and un-normalised O meet the incoming state, and the row is stored.
template <class TQ, int VE, int NC>
__device__ __forceinline__ void finish_row(const Call& a, const MergeArgs& g, int64_t n, int32_t hq, int lane, float M, float L,
                                           float (&acc)[NC * VE]) {
  const int d = a.c.d;
  auto col = [&](int i) { return (i * 32 + lane) * VE; };
  float* m = g.m + n * a.n_q_heads + hq;
  float* l = g.l + n * a.n_q_heads + hq;
  const bool none = M == neg_inf();  // no key, or none with a score above -inf
  if (none && !g.first) return;
  TQ* O = reinterpret_cast<TQ*>(g.O) + n * g.o_stride[0] + hq * g.o_stride[1];
  float m_out = M * 0.6931471805599453f, keep = 0.f, mine = 1.f;
  if (!g.first) {
    const float m_in = *m, l_in = *l;
    if (l_in != 0.f) {  // a row with l = 0 is empty: what its O holds does not count
      const float m2 = m_in * kLog2e, top = max_nan(m2, M);
      if (!(M > m2)) m_out = top != top ? top : m_in;
      mine = fast_exp2(M - top);
      keep = l_in * fast_exp2(m2 - top);
      L = fmaf(L, mine, keep);
    }
  }
  const float inv = none ? 0.f : 1.f / L;
#pragma unroll
  for (int i = 0; i < NC; ++i)
    if (col(i) < d) {
      float y[VE];
      if (keep != 0.f) load_vec<TQ, VE>(O + col(i), y);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float x = acc[i * VE + e] * mine;
        y[e] = (keep != 0.f ? fmaf(keep, y[e], x) : x) * inv;
      }
      store_vec<TQ, VE>(O + col(i), y);
    }
  __syncwarp();
  if (lane == 0) {
    *m = m_out;
    *l = none ? 0.f : L;
  }
}

template <class TQ, class TC, int VE, int NC, int GR>
__global__ void __launch_bounds__(128) merge_kernel(const Call a, const MergeArgs g) {
  constexpr int NE = NC * VE;
  const int lane = threadIdx.x & 31;
  const uint32_t warp = blockIdx.x * 4 + (threadIdx.x >> 5), parts = (uint32_t)(a.group + GR - 1) / GR, per_row = parts * (uint32_t)a.c.n_heads;
  const int64_t n = warp / per_row;
  const int32_t in = (int32_t)(warp - (uint32_t)n * per_row), h = in / (int32_t)parts, g0 = (in - h * (int32_t)parts) * GR;
  const int rows = GR == 1 ? 1 : min(GR, a.group - g0);
  const int32_t hq = h * a.group + g0;
  const int32_t b = n < a.n_rows ? sequence_of(a.cu_rows, a.c.n_seq, n) : -1;
  if (b < 0) {  // the grid ends behind the context kernel's end, whatever its rows are
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  int64_t begin, end;
  rows_of(a.cu_rows, b, a.n_rows, begin, end);
  const int64_t tokens = end - begin, len = a.c.len_of(b);
  const int d = a.c.d;

  float q[GR][NE], acc[GR][NE], M[GR], L[GR];
  auto col = [&](int i) { return (i * 32 + lane) * VE; };
#pragma unroll
  for (int r = 0; r < GR; ++r) {
    M[r] = neg_inf();
    L[r] = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      float x[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) x[e] = acc[r][i * VE + e] = 0.f;
      if (r < rows && col(i) < d)
        load_vec<TQ, VE>(reinterpret_cast<const TQ*>(a.Q) + n * a.q_stride[0] + (hq + r) * a.q_stride[1] + col(i), x);
#pragma unroll
      for (int e = 0; e < VE; ++e) q[r][i * VE + e] = x[e];
    }
  }

  constexpr int KB = NE <= 8 ? 4 : 1;  // keys at a time: as registers allow
  const int64_t cols = tokens < g.mask_width ? tokens : g.mask_width;
  for (int64_t j0 = 0; j0 < cols; j0 += 32) {
    const bool on = j0 + lane < cols && __ldg(g.mask + n * g.mask_width + j0 + lane) != 0;
    // each lane finds the page of its own key, before the keys are taken one after the other
    const int64_t p = len + j0 + lane;
    const int32_t my_page = on ? a.c.page_of(b, p) : -1;
    const int32_t my_slot = my_page >= 0 ? a.c.slot_of(p) : 0;
    const int64_t my_k = my_page >= 0 ? a.c.K.at(my_page, my_slot, h) : 0, my_v = my_page >= 0 ? a.c.V.at(my_page, my_slot, h) : 0;
    float my_fk = 1.f, my_fv = 1.f;
    if constexpr (IsByte<TC>::value) {
      if (my_page >= 0) {
        my_fk = a.c.K.scale[a.c.K.scale_at(my_page, my_slot, h)];
        my_fv = a.c.V.scale[a.c.V.scale_at(my_page, my_slot, h)];
      }
    }
    unsigned bits = __ballot_sync(kFullMask, my_page >= 0);
    while (bits) {
      float k[KB][NE], v[KB][NE], s[KB][GR], fk[KB], fv[KB];
      int taken = 0;
#pragma unroll
      for (int x = 0; x < KB; ++x) {
        fk[x] = fv[x] = 1.f;
#pragma unroll
        for (int e = 0; e < NE; ++e) k[x][e] = v[x][e] = 0.f;
        if (bits == 0) continue;
        const int j = __ffs(bits) - 1;
        bits &= bits - 1;
        ++taken;
        const TC* kp = reinterpret_cast<const TC*>(a.c.K.data) + __shfl_sync(kFullMask, my_k, j);
        const TC* vp = reinterpret_cast<const TC*>(a.c.V.data) + __shfl_sync(kFullMask, my_v, j);
#pragma unroll
        for (int i = 0; i < NC; ++i)
          if (col(i) < d) {
            float y[VE];
            load_vec<TC, VE>(kp + col(i), y);
#pragma unroll
            for (int e = 0; e < VE; ++e) k[x][i * VE + e] = y[e];
            load_vec<TC, VE>(vp + col(i), y);
#pragma unroll
            for (int e = 0; e < VE; ++e) v[x][i * VE + e] = y[e];
          }
        if constexpr (IsByte<TC>::value) {
          fk[x] = __shfl_sync(kFullMask, my_fk, j);
          fv[x] = __shfl_sync(kFullMask, my_fv, j);
        }
      }
#pragma unroll
      for (int x = 0; x < KB; ++x)
#pragma unroll
        for (int r = 0; r < GR; ++r) {
          s[x][r] = 0.f;
#pragma unroll
          for (int e = 0; e < NE; ++e) s[x][r] = fmaf(q[r][e], IsByte<TC>::value ? k[x][e] * fk[x] : k[x][e], s[x][r]);
        }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int x = 0; x < KB; ++x)
#pragma unroll
          for (int r = 0; r < GR; ++r) s[x][r] += __shfl_xor_sync(kFullMask, s[x][r], o);
#pragma unroll
      for (int r = 0; r < GR; ++r) {
        float top = M[r];
#pragma unroll
        for (int x = 0; x < KB; ++x) {
          s[x][r] = x < taken ? s[x][r] * a.scale_log2e : neg_inf();
          top = max_nan(top, s[x][r]);
        }
        const float ref = top == neg_inf() ? 0.f : top, f = fast_exp2(M[r] - ref);
        L[r] *= f;
#pragma unroll
        for (int e = 0; e < NE; ++e) acc[r][e] *= f;
#pragma unroll
        for (int x = 0; x < KB; ++x) {
          if (x >= taken) continue;
          const float pr = fast_exp2(s[x][r] - ref);
          L[r] += pr;
#pragma unroll
          for (int e = 0; e < NE; ++e) acc[r][e] = fmaf(pr, IsByte<TC>::value ? v[x][e] * fv[x] : v[x][e], acc[r][e]);
        }
        M[r] = top;
      }
    }
  }

  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t tiles = a.tiles_of(len);
  if (tiles > 0) {
    const int64_t x = (n - begin) * a.group + g0;  // the rows lie in one unit (GR > 1: units hold whole tokens)
    const int64_t u = (int64_t)h * a.row_tiles(tokens) + x / a.unit_rows;
    const int64_t chunk = a.cut[0], t = a.cut[1 + b] + u * tiles;
    const int64_t c0 = t / chunk, c1 = (t + tiles - 1) / chunk;
    for (int64_t c = c0; c <= c1; c += 32) {
      const int np = (int)(c1 - c + 1 < 32 ? c1 - c + 1 : 32);
      const int64_t row = a.partial_row(begin, tokens, h, x, c);
      float2 ml[GR];
      float wgt[GR];
#pragma unroll
      for (int r = 0; r < GR; ++r) {
        ml[r] = make_float2(neg_inf(), 0.f);
        if (lane < np && r < rows) ml[r] = a.ml[row + (int64_t)lane * a.row_tile + r];
      }
#pragma unroll
      for (int r = 0; r < GR; ++r) {
        float top = ml[r].x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(kFullMask, top, o));
        top = max_nan(top, M[r]);
        const float ref = top == neg_inf() ? 0.f : top, f = fast_exp2(M[r] - ref);
        wgt[r] = fast_exp2(ml[r].x - ref);
        float sum = wgt[r] * ml[r].y;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
        L[r] = L[r] * f + sum;
#pragma unroll
        for (int e = 0; e < NE; ++e) acc[r][e] *= f;
        M[r] = top;
      }
      constexpr int PB = NE * GR <= 8 ? 8 : 2;  // pieces whose rows are in flight together
      for (int k0 = 0; k0 < np; k0 += PB) {
        float y[PB][GR][NE];
#pragma unroll
        for (int k = 0; k < PB; ++k)
#pragma unroll
          for (int r = 0; r < GR; ++r) {
            const float* src = a.O + (row + (int64_t)(k0 + k) * a.row_tile + r) * a.d_pad;
#pragma unroll
            for (int i = 0; i < NC; ++i) {
              float z[VE];
#pragma unroll
              for (int e = 0; e < VE; ++e) z[e] = 0.f;
              if (k0 + k < np && r < rows && col(i) < d) load_vec<float, VE>(src + col(i), z);
#pragma unroll
              for (int e = 0; e < VE; ++e) y[k][r][i * VE + e] = z[e];
            }
          }
#pragma unroll
        for (int k = 0; k < PB; ++k)
#pragma unroll
          for (int r = 0; r < GR; ++r) {
            const float wk = __shfl_sync(kFullMask, wgt[r], (k0 + k) & 31);
#pragma unroll
            for (int e = 0; e < NE; ++e) acc[r][e] = fmaf(k0 + k < np ? wk : 0.f, y[k][r][e], acc[r][e]);
          }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < GR; ++r)
    if (r < rows) finish_row<TQ, VE, NC>(a, g, n, hq + r, lane, M[r], L[r], acc[r]);
}

}  // namespace tree
}  // namespace spfa
