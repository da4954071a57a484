// Tree attention over the committed positions on the tensor cores: float16 / bfloat16 Q, a cache of the same type or of 8 bits,
// d <= 128. Part of the scheme of tree_kernels.cuh (units, pieces, partial rows).
//
// One CTA, two on an SM, takes its share of the list of key tiles piece by piece. A unit is 128 query rows (tokens x the query
// heads of one key head) and a tile 64 keys:
//   S  = Q K_j^T           128 x 64 fp32 in TMEM, two buffers, issued two tiles ahead
//   P  = exp2(S c - shift) in registers, one thread a row, rounded to 16 bits and written over S
//   O += P V_j             128 x DP fp32 in TMEM
// Rows beyond a unit's are not computed: their warps only keep step. Roles (256 threads):
//   warps 0-3  Q, softmax and the pieces' epilogue: thread t <-> row t <-> TMEM lane t
//   warp 4     TMA producer of K, masks and scales: page numbers 32 at a time in the lanes, one box for each page of a tile and 128
//              bytes of d. Pages that do not exist are fetched from behind the last one, where the copy engine fills with zeros.
//   warp 5     MMA issuer
//   warp 6     TMA producer of V
//   warps 8-11 (8-bit caches) the conversion of V, and of int8 K, to 16 bits
//   With two row tiles: warps 0-7 softmax, 8-11 the roles of 4-7 (11 the second tile's MMA issuer), 12-19 the conversion.
// A unit of at most 64 (32) rows has them two (four) times in Q: each copy takes half (a quarter) of every tile's columns, so that all
// four softmax warps work, and the copies are added up at the end of the piece.
// An 8-bit tile meets the tensor cores as float16 numbers that equal its codes (11 bits hold e4m3 and int8), except K of e4m3 under
// bfloat16 Q: that meets them as it lies, in the products of 8-bit numbers, and Q as two terms, each the rounding of what is left, the
// first e4m3, the second e5m2. A row is first multiplied by a power of two that brings its largest element to [2^7, 2^8): the terms are
// an element exactly then, down to 2^-13 of the largest (2^-6, where e4m3's subnormal numbers begin), and smaller ones are held to 2^-21
// of it. (e4m3 alone, which ends at 2^-9, showed in l: 9e-7 of it, float32 sums 4e-7.) Without K's conversion, which passes the tile
// through shared memory twice: 437 -> 366 us, e4m3 call below. float16 elements take three terms, and their products cost more than the
// conversion: 491 us against 458. bfloat16 Q over int8 becomes float16 times such a power: none of its 8 bits is lost above 2^-29 of the
// row's largest element.
// The rows' scales stay in fp32: K's multiplies the score, V's the probability before that is rounded, and the row's reference is the
// largest such product.
// P is rounded to 16 bits. Where that alone would be as large as the rounding of the result (all but 8-bit caches under bfloat16 Q),
// sequences of at most 128 rows for a key head carry a second 16-bit term, the rounding's remainder: they wait for memory, and the second
// product is hidden. Those of more rows are bound by arithmetic, and have one: float16 over int8 is off by 3.0e-4 of the result then, with
// two terms by 2.1e-4, the result's own rounding.
//
// What bounds it, on 32 sequences of up to 32768 keys, 8 tokens, 4 heads a key head (32 rows a unit), d = 128: a bfloat16 cache memory,
// 460 us, 5.9 TB/s; e4m3 366 us, 3.9 TB/s, and int8 488 us, 2.9 TB/s, shared memory: V's (int8: K's too) way through the converting warps,
// Q and the converted tiles on theirs to the tensor cores add up to its 128 bytes a cycle. Units of 256 rows are bound by the softmax
// warps, each of which owns a row of 64 scores a tile: 302 us, 910 TFLOP/s for 8 sequences of 64 tokens, 64 heads on 8, over 16384
// bfloat16 keys; 168 us, 454 TFLOP/s for 8 of up to 64 tokens, 32 heads on 4, over up to 16384 int8 keys under float16 Q.
#pragma once
#include "tile_kernels_16.cuh"
#include "tree_kernels.cuh"

namespace spfa {
namespace tree {

using namespace tile;

// NSUB: 128-row tiles that a CTA works on together, against the same K and V. One, and two CTAs share an SM; or two, and a CTA has it
// alone: K and V are fetched and converted once for both.
template <int DP, class T, class TC, int NSUB>
struct PlanTree {
  static constexpr bool kQuant = sizeof(TC) == 1, kRawK = std::is_same<TC, e4m3>::value && std::is_same<T, __nv_bfloat16>::value, kConvertK = kQuant && !kRawK;
  static constexpr int kTerms = 2;  // 8-bit numbers of an element of Q (kRawK)
  static constexpr int kSoftmaxWarps = 4 * NSUB, kAux = 4 * NSUB /* first of four warps */, kConvertFrom = kAux + 4;
  static constexpr int kConvert = kQuant ? 128 * NSUB : 0, kThreads = 128 * NSUB + 128 + kConvert, kCtasPerSm = 3 - NSUB;
  static constexpr int kRegsLaunch = NSUB == 1 ? (kQuant ? 80 : 128) : (kQuant ? 96 : 168);
  static constexpr int kRegsSoftmax = NSUB == 1 ? (kQuant ? 128 : 168) : (kQuant ? 152 : 184);
  static constexpr int kRegsAux = NSUB == 1 ? (kQuant ? 56 : 88) : (kQuant ? 56 : 136);
  static constexpr int kRegsNeeded = kRegsSoftmax * 128 * NSUB + kRegsAux * (kThreads - 128 * NSUB);
  static_assert(kRegsNeeded <= kRegsLaunch * kThreads, "setmaxnreg budgets exceed the launch pool");
  static constexpr int TK = 64, kRows = 128 * NSUB, kChunks = DP / 64;
  // (two row tiles and kRawK: a term's room is left free, 160 us against 170 with the stages right behind the terms)
  static constexpr int kQChunk = 128 * 128, kKVChunk = TK * 128;
  static constexpr int kQSub = (!kRawK ? kChunks : NSUB == 2 ? kTerms + 1 : kTerms) * kQChunk, kQBytes = NSUB * kQSub;
  static constexpr int kTile = kChunks * kKVChunk;               // a 16-bit tile of K or V
  static constexpr int kStage = kQuant ? TK * DP : kTile;        // a tile as it is fetched
  static constexpr int kStageK = kRawK ? TK * 128 : kStage;      // K's, where it meets the tensor cores so: in their swizzle
  static constexpr int NS = (DP == 64 || NSUB == 2) ? 4 : kRawK ? 3 : 2;  // stages of K and of V: what memory allows
  static constexpr int NC = kQuant ? NSUB : 1;                   // converted tiles of K and of V
  static constexpr int kRing = 8;                                // tiles whose masks and scales are kept
  static constexpr int kOffQ = 0, kOffK = kQBytes, kOffV = kOffK + NS * kStageK, kOffCK = kOffV + NS * kStage;
  static constexpr int kOffCV = kOffCK + (kConvertK ? NC * kTile : 0), kOffScale = kOffCV + (kQuant ? NC * kTile : 0);
  static constexpr int kOffRow = kOffScale + (kQuant ? kRing * 2 * TK * 4 : 0), kOffMask = kOffRow + 128 * 8;
  static constexpr int kOffBar = kOffMask + kRing * 8, kNumBars = 4 * NS + 4 * NC + 7 * NSUB + 1;
  static constexpr int kOffCut = kOffBar + kNumBars * 8, kOffMisc = kOffCut + (int)sizeof(Cut);
  static constexpr int kDynSmem = kOffMisc + 16 + 1024;
  static_assert(kCtasPerSm * (kDynSmem + 1024) <= 228 * 1024, "shared memory of an SM");
  // The producer writes the ring's entry of a tile once the tile NS before has left its stage, which is behind the softmax of the
  // tile two (K converted: two and NC) before that one.
  static_assert(NS + 2 + NC <= kRing, "ring entries are written again only after they were read");
  static constexpr int kColS = 0, kColO = NSUB * 2 * TK, kTmemCols = 256 * NSUB;
  static_assert(kColO + NSUB * DP <= kTmemCols, "S buffers and the O accumulators exceed the TMEM allocation");
  static __device__ __forceinline__ uint32_t unit(int row, int u) { return (uint32_t)(row * 128 + ((u ^ (row & 7)) << 4)); }
};

// mbar_wait of tile_kernels_sm100.cuh with a time hint: a warp of this kernel often waits for several tiles' worth of other roles, and a
// waiting warp that polls takes issue slots from them.
__device__ __forceinline__ bool mbar_try_for(uint32_t bar, uint32_t parity, uint32_t ns) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(ns)
      : "memory");
  return ok != 0;
}
// All lanes of a converged warp.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* err, int code) {
  bool done = mbar_try_for(bar, parity, 10000u);
  if (!__all_sync(kFullMask, done)) {
    const uint64_t t0 = globaltimer();
    while (!__all_sync(kFullMask, done = done || mbar_try_for(bar, parity, 10000u))) {
      const bool late = globaltimer() - t0 > kWaitNs;
      if (__any_sync(kFullMask, *abort_flag || late)) {
        if (late) {
          *abort_flag = 1;
          atomicCAS(err, 0, code);
        }
        return false;
      }
    }
  }
  return true;
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* tm, int32_t x, int32_t y, int32_t z, int32_t w, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(tm), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld4(uint32_t taddr, uint32_t (&r)[4]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void mma8_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(acc)
      : "memory");
}
// Two 8-bit numbers of a term in the low half of a word, x's in its lower byte, and what their rounding leaves of x (exact).
// The first term is e4m3, the others e5m2: its 3 bits hold what 4 bits leave of 8, and its range goes on down to 2^-16.
template <bool kFirst>
__device__ __forceinline__ uint32_t take_term(float2& x) {
  uint16_t y;
  uint32_t back;
  if constexpr (kFirst) {
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(y) : "f"(x.y), "f"(x.x));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(y));
  } else {
    asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(y) : "f"(x.y), "f"(x.x));
    asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(back) : "h"(y));
  }
  const float2 held = Half16<__half>::up(back);
  x = make_float2(x.x - held.x, x.y - held.y);
  return y;
}

__device__ __forceinline__ void cp_async4(uint32_t dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// Four codes to float16. The bytes of an int8 word leave in the order 0 2 1 3, where masks alone widen them: the order of d does not
// matter to Q K^T as long as Q has it too, and O's columns are put right when they are stored.
template <class TC> struct Widen {  // a cache that holds its values as they are is not converted
  static constexpr bool kSwap = false;
};
template <> struct Widen<e4m3> {
  static constexpr bool kSwap = false;
  static __device__ __forceinline__ void four(uint32_t w, uint32_t& a, uint32_t& b) {
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
        : "=r"(a), "=r"(b)
        : "r"(w));
  }
};
template <> struct Widen<int8_t> {
  static constexpr bool kSwap = true;
  // 1024 + (code + 128) has the code's bits as its last, and 1152 less is exact
  static __device__ __forceinline__ uint32_t off(uint32_t x) {
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2(__half2_raw{0x6480, 0x6480}));
    return *reinterpret_cast<const uint32_t*>(&y);
  }
  static __device__ __forceinline__ void four(uint32_t w, uint32_t& a, uint32_t& b) {
    a = off((w & 0x00ff00ffu) ^ 0x64806480u);
    b = off(((w >> 8) & 0x00ff00ffu) ^ 0x64806480u);
  }
};

// p V_j for an infinite V_j is that infinity, but its products with what stands for p here need not add up to it: a term that is zero or
// negative makes NaN, and so do the zeros of a copied unit and a p that 16 bits round to zero. Where a piece's accumulator is not finite,
// V itself tells what it has to hold: +inf, -inf, or NaN where both or a NaN are among the keys [p, p_end) that all rows of the piece
// see. One warp goes through the piece once for all columns: 16 bytes a lane, the rows of 32 keys in flight together, their pages
// looked up 32 keys ahead: 3 ms for 170000 keys of 64 elements, a hundredth of what the CTA's other roles wait (kWaitNs). Bit i of
// word w is column 32 w + i.
template <int DP>
struct Infinities {
  uint32_t up[DP / 32], down[DP / 32], nan[DP / 32];
};
template <int DP, class T>
__device__ __noinline__ void find_infinities(const Call& a, int32_t b, int32_t h, int64_t p, int64_t p_end, Infinities<DP>& found) {
  constexpr int kLanes = DP / 8, kRows = 32 / kLanes;  // lanes of a row, rows of a load
  constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u, kInf2 = kInf << 16 | kInf;
  const int lane = threadIdx.x & 31, col = lane % kLanes * 8, sub = lane / kLanes;
  const T* V = reinterpret_cast<const T*>(a.c.V.data) + (int64_t)h * a.c.V.stride[2] + col;
  auto page_at = [&](int64_t q) -> int32_t { return q < p_end ? a.c.page_of(b, q) : -1; };
  uint32_t bits = 0;  // of this lane's columns: +inf, -inf, NaN in eight each
  int32_t next = page_at(p + lane);
  for (; p < p_end; p += 32) {
    const int32_t page = next, slot = a.c.slot_of(p + lane);
    next = page_at(p + 32 + lane);
    uint4 x[kLanes];
#pragma unroll
    for (int i = 0; i < kLanes; ++i) {
      const int32_t pg = __shfl_sync(kFullMask, page, i * kRows + sub), sl = __shfl_sync(kFullMask, slot, i * kRows + sub);
      x[i] = make_uint4(0, 0, 0, 0);
      if (pg >= 0 && col < a.c.d) x[i] = __ldg(reinterpret_cast<const uint4*>(V + pg * a.c.V.stride[0] + sl * a.c.V.stride[1]));
    }
#pragma unroll
    for (int i = 0; i < kLanes; ++i) {
      const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
      uint32_t any = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) any |= __vcmpgeu2(w[k] & 0x7fff7fffu, kInf2);
      if (any == 0) continue;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t v = (w[k / 2] >> (k % 2 * 16)) & 0xffffu, top = v & 0x7fffu;
        if (top >= kInf) bits |= (top > kInf ? 0x10000u : v >> 15 ? 0x100u : 1u) << k;
      }
    }
  }
#pragma unroll
  for (int o = kLanes; o < 32; o <<= 1) bits |= __shfl_xor_sync(kFullMask, bits, o);
  bits |= (bits & bits >> 8 & 0xffu) << 16;  // both signs
#pragma unroll
  for (int w = 0; w < DP / 32; ++w) {
    found.up[w] = found.down[w] = found.nan[w] = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t y = __shfl_sync(kFullMask, bits, w * 4 + k);
      found.up[w] |= (y & 0xffu) << (8 * k);
      found.down[w] |= (y >> 8 & 0xffu) << (8 * k);
      found.nan[w] |= (y >> 16 & 0xffu) << (8 * k);
    }
  }
}

template <int DP, class T, class TC, int NSUB>
__global__ void __launch_bounds__(PlanTree<DP, T, TC, NSUB>::kThreads, PlanTree<DP, T, TC, NSUB>::kCtasPerSm)
context_tiled_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Call a,
                     int* __restrict__ err) {
  using P = PlanTree<DP, T, TC, NSUB>;
  constexpr int TK = P::TK, NS = P::NS, NC = P::NC;
  constexpr bool kQuant = P::kQuant, kRawK = P::kRawK, kConvertK = P::kConvertK;
  constexpr int kTerms = P::kTerms;
  using TP = typename std::conditional<kQuant, __half, T>::type;  // operands of both products
  constexpr bool kMaySplit = !(kQuant && std::is_same<T, __nv_bfloat16>::value);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);  // an offset: through an integer, every access below would be a generic one
  const uint32_t sbase = smem_u32(smem);
  auto bar = [&](int i) { return sbase + P::kOffBar + 8u * i; };
  constexpr int B_KFULL = 0, B_KEMPTY = NS, B_VFULL = 2 * NS, B_VEMPTY = 3 * NS, B_CK = 4 * NS /* full [NC], empty [NC] */, B_CV = B_CK + 2 * NC, B_SREADY = B_CK + 4 * NC,
                B_PREADY = B_SREADY + 2 * NSUB, B_OREADY = B_SREADY + 4 * NSUB /* [sub][buffer] */, B_QFULL = B_SREADY + 6 * NSUB, B_GROUP = B_QFULL + NSUB;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + P::kOffMisc + 4);
  Cut* cut = reinterpret_cast<Cut*>(smem + P::kOffCut);
  uint64_t* ring_mask = reinterpret_cast<uint64_t*>(smem + P::kOffMask);
  float* ring_scale = reinterpret_cast<float*>(smem + P::kOffScale);  // [ring][K, V][TK]
  float2* row_ml = reinterpret_cast<float2*>(smem + P::kOffRow);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int32_t ps = a.c.page_size;
  const int n_pages_tile = a.page_tiles ? 1 : a.tile_keys / ps;  // pages of a tile

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(bar(B_KFULL + s), kQuant ? 33 : 1);
      mbar_init(bar(B_KEMPTY + s), kConvertK ? P::kConvert / 32 : NSUB);
      mbar_init(bar(B_VFULL + s), 1);
      mbar_init(bar(B_VEMPTY + s), kQuant ? P::kConvert / 32 : NSUB);
    }
    for (int x = 0; x < NC; ++x) {
      mbar_init(bar(B_CK + x), kQuant ? P::kConvert / 32 : 1);
      mbar_init(bar(B_CK + NC + x), NSUB);
      mbar_init(bar(B_CV + x), kQuant ? P::kConvert / 32 : 1);
      mbar_init(bar(B_CV + NC + x), NSUB);
    }
    for (int x = 0; x < 2 * NSUB; ++x) {
      mbar_init(bar(B_SREADY + x), 1);
      mbar_init(bar(B_PREADY + x), 4);
      mbar_init(bar(B_OREADY + x), 1);
    }
    for (int x = 0; x < NSUB; ++x) mbar_init(bar(B_QFULL + x), 4);
    mbar_init(bar(B_GROUP), 4);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == P::kAux) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sbase + P::kOffMisc), "r"(P::kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x == P::kAux * 32 + 32) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmK)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmV)) : "memory");
  }
  if (!kQuant && a.tile_keys < TK) {  // rows that no box reaches: zero V, finite K
    for (int x = threadIdx.x; x < NS * (P::kStageK + P::kStage) / 16; x += P::kThreads) reinterpret_cast<uint4*>(smem + P::kOffK)[x] = make_uint4(0, 0, 0, 0);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  block_cut<P::kThreads>(a, cut);  // ends with a barrier
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + P::kOffMisc);

  Walk w;
  w.init(a, cut);
  // Keys of tile t (the rest of its rows are masked): whole pages of a sequence, or a part of one page.
  auto keys_of = [&](int32_t t, int32_t& first_page, int32_t& slot) -> int {
    int32_t left;
    if (a.page_tiles) {
      first_page = t / a.page_tiles;
      slot = (t - first_page * a.page_tiles) * TK;
      left = min(w.len - first_page * ps, ps) - slot;
    } else {
      first_page = t * n_pages_tile;
      slot = 0;
      left = w.len - t * a.tile_keys;
    }
    return min(left, a.tile_keys);
  };

  if (warp >= P::kAux) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(P::kRegsAux));
    if (warp == P::kAux || warp == P::kAux + 2) {
      // =============================== TMA producers: one warp K, masks and scales, one V ===============================
      const bool is_k = warp == P::kAux;
      const CUtensorMap* tm = is_k ? &tmK : &tmV;
      const int full = is_k ? B_KFULL : B_VFULL, empty = is_k ? B_KEMPTY : B_VEMPTY, off = is_k ? P::kOffK : P::kOffV;
      const bool el = elect_one();
      // page (within a tile) and slot of this lane's two keys
      int key_page[2], key_slot[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int key = lane + 32 * x;
        key_page[x] = a.page_tiles ? 0 : min(key / ps, n_pages_tile - 1);
        key_slot[x] = key - key_page[x] * ps;
      }
      const uint32_t stage = is_k ? P::kStageK : P::kStage, key_bytes = stage / TK;
      const uint32_t tile_bytes = (uint32_t)(a.page_tiles ? TK : ps) * key_bytes * n_pages_tile;
      const uint32_t every = 0xffffffffu >> (32 - n_pages_tile);
      uint32_t jj = 0;
      bool ok = true;
      while (ok && w.next(a)) {
        const int32_t* table = a.c.table + (int64_t)w.b * a.c.table_width;
        auto pages_at = [&](int32_t i) -> int32_t { return i + lane < a.c.table_width ? __ldg(table + i + lane) : -1; };
        int32_t first, slot;  // of the tile
        keys_of(w.t0, first, slot);
        int32_t base = first, nxt = pages_at(base), cur = 0;
        uint32_t valid = 0;
        auto turn = [&](int32_t more) {  // the next 32 pages; pages that do not exist become the one behind the last: zeros
          const bool in = nxt >= 0 && nxt < a.c.n_pages;
          valid = __ballot_sync(kFullMask, in);
          cur = in ? nxt : (int32_t)a.c.n_pages;
          nxt = pages_at(more);
        };
        turn(base + 32);
        [[maybe_unused]] const float *ks[2], *vs[2];  // scales of this lane's two keys, on page 0
        if (kQuant && is_k) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            ks[x] = a.c.K.scale + a.c.K.scale_at(0, key_slot[x], w.h);
            vs[x] = a.c.V.scale + a.c.V.scale_at(0, key_slot[x], w.h);
          }
        }
        for (int32_t t = 0; t < w.n; ++t, ++jj) {
          const int st = jj % NS;
          ok = warp_wait(bar(empty + st), ((jj / NS) & 1) ^ 1u, abort_flag, err, is_k ? 111 : 112);
          if (!ok) break;
          const int at = first - base;
          if (is_k) {
            const int n = min(a.page_tiles ? min(w.len - first * ps, ps) - slot : w.len - (w.t0 + t) * a.tile_keys, a.tile_keys);
            uint64_t mask = n >= 64 ? ~0ull : (1ull << n) - 1;
            if (((valid >> at) & every) != every) {
              for (int i = 0; i < n_pages_tile; ++i)
                if (!((valid >> (at + i)) & 1u)) mask &= a.page_tiles ? 0ull : ~(((1ull << ps) - 1) << (i * ps));
            }
            if (el) ring_mask[jj % P::kRing] = mask;
            if constexpr (kQuant) {
              const uint32_t dst = sbase + P::kOffScale + ((jj % P::kRing) * 2 * TK + lane) * 4;
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const int32_t page = __shfl_sync(kFullMask, cur, at + key_page[x]);
                if (lane + 32 * x < n && page < a.c.n_pages) {
                  cp_async4(dst + 128 * x, ks[x] + page * a.c.K.s_stride[0] + slot * a.c.K.s_stride[1]);
                  cp_async4(dst + 128 * x + TK * 4, vs[x] + page * a.c.V.s_stride[0] + slot * a.c.V.s_stride[1]);
                } else {
                  asm volatile("st.shared.f32 [%0], %1;" ::"r"(dst + 128 * x), "f"(1.f) : "memory");  // its score is -inf, and stays that
                  asm volatile("st.shared.f32 [%0], %1;" ::"r"(dst + 128 * x + TK * 4), "f"(0.f) : "memory");
                }
              }
              cp_async_arrive(bar(B_KFULL + st));
              __syncwarp();
            }
          }
          if (el) mbar_expect_tx(bar(full + st), tile_bytes);
          uint32_t to = sbase + off + st * stage;
          for (int i = 0; i < n_pages_tile; ++i) {
            const int32_t page = __shfl_sync(kFullMask, cur, at + i);
            if (el) {
              if constexpr (kQuant) {
                tma_load_4d(to, tm, 0, slot, w.h, page, bar(full + st));
              } else {
#pragma unroll
                for (int c = 0; c < P::kChunks; ++c) tma_load_4d(to + c * P::kKVChunk, tm, c * 64, slot, w.h, page, bar(full + st));
              }
            }
            to += ps * (kQuant ? key_bytes : 128);
          }
          __syncwarp();
          if (a.page_tiles) {
            slot += TK;
            if (slot >= ps) {
              slot = 0;
              ++first;
            }
          } else {
            first += n_pages_tile;
          }
          if (first >= base + 32) {
            base += 32;
            turn(base + 32);
          }
        }
      }
      if constexpr (kQuant) asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == P::kAux + 1 || (NSUB == 2 && warp == P::kAux + 3)) {
      // =============================== MMA issuers: one for each row tile ===============================
      const int sub = NSUB == 2 && warp == P::kAux + 3 ? 1 : 0;
      const bool el = elect_one();
      // (kind::f8f6f4: e4m3 has the code of float16 in the descriptor, e5m2 that of bfloat16)
      constexpr uint32_t kIdescS = idesc_16<TP>(128, TK, 0), kIdescO = idesc_16<TP>(128, DP, 1);
      const uint64_t qd = smem_desc(sbase + P::kOffQ + sub * P::kQSub, 16, 1024, kLayoutSw128);
      const uint32_t s_at = tmem + P::kColS + 2 * TK * sub, o_at = tmem + P::kColO + sub * DP;
      const int b_sready = B_SREADY + 2 * sub, b_pready = B_PREADY + 2 * sub, b_oready = B_OREADY + 2 * sub;
      uint32_t jj = 0, done = 0, unit = 0;  // tiles of the CTA, tiles and units of this row tile
      bool ok = true;
      while (ok && w.next(a)) {
        const int32_t n = w.n;
        const bool split = w.tokens * a.group <= 128;
        const bool idle = NSUB == 2 && sub == 1 && w.rows(a) <= 128;  // the unit has no second tile: only the stages are handed on
        auto k_ready = [&](uint32_t j) -> bool {
          return warp_wait(bar(kConvertK ? B_CK + j % NC : B_KFULL + j % NS), kConvertK ? (j / NC) & 1 : (j / NS) & 1, abort_flag, err, 212);
        };
        auto v_ready = [&](uint32_t j) -> bool {
          return warp_wait(bar(kQuant ? B_CV + j % NC : B_VFULL + j % NS), kQuant ? (j / NC) & 1 : (j / NS) & 1, abort_flag, err, 214);
        };
        if (idle) {
          for (int32_t t = 0; t < n && ok; ++t, ++jj) {
            ok = k_ready(jj);
            if (ok && el) mbar_arrive(bar(kConvertK ? B_CK + NC + jj % NC : B_KEMPTY + jj % NS));
            ok = ok && v_ready(jj);
            if (ok && el) mbar_arrive(bar(kQuant ? B_CV + NC + jj % NC : B_VEMPTY + jj % NS));
          }
          continue;
        }
        ok = warp_wait(bar(B_QFULL + sub), unit & 1, abort_flag, err, 211);
        ++unit;
        if (!ok) break;
        auto issue_S = [&](int32_t t) -> bool {
          if (t >= n) return true;
          const uint32_t j = jj + (uint32_t)t, buf = (done + (uint32_t)t) & 1;
          const int st = kConvertK ? j % NC : j % NS;
          if (!k_ready(j)) return false;
          tc_fence_after();
          const uint64_t kd = smem_desc(sbase + (kConvertK ? P::kOffCK + st * P::kTile : P::kOffK + st * P::kStageK), 16, 1024, kLayoutSw128);
          if (el) {
            if constexpr (kRawK) {  // 32 elements (32 bytes) of the contraction per MMA, Q's terms one after the other
#pragma unroll
              for (int kk = 0; kk < kTerms * DP / 32; ++kk) {
                const int term = kk / (DP / 32), in = kk % (DP / 32) * 32;
                mma8_ss(s_at + TK * buf, qd + (uint64_t)((term * P::kQChunk + in) >> 4), kd + (uint64_t)(in >> 4),
                        kIdescS | (term ? 1u << 7 : 0u), kk ? 1u : 0u);
              }
            } else {
#pragma unroll
              for (int kk = 0; kk < DP / 16; ++kk) {  // 16 elements (32 bytes) of the contraction per MMA
                const int c = kk / 4, in = kk % 4 * 32;
                mma16_ss(s_at + TK * buf, qd + (uint64_t)((c * P::kQChunk + in) >> 4), kd + (uint64_t)((c * P::kKVChunk + in) >> 4), kIdescS,
                         kk ? 1u : 0u);
              }
            }
            tc_commit(bar(b_sready + buf));
            tc_commit(bar(kConvertK ? B_CK + NC + st : B_KEMPTY + st));
          }
          __syncwarp();
          return true;
        };
        ok = issue_S(0) && issue_S(1);
        for (int32_t t = 0; t < n && ok; ++t) {
          const uint32_t j = jj + (uint32_t)t, own = done + (uint32_t)t;
          const int st = kQuant ? j % NC : j % NS;
          ok = v_ready(j);
          if (!ok) break;
          const uint32_t v_at = sbase + (kQuant ? P::kOffCV + st * P::kTile : P::kOffV + st * P::kStage);
          if constexpr (!kQuant) {  // rows behind the sequence's end hold anything, and 0 times anything may be NaN
            if (w.t0 + t == w.tiles - 1) {
              int32_t first, slot;
              const int keys = keys_of(w.t0 + t, first, slot);
              for (int x = keys * 8 + lane; x < TK * 8; x += 32)
#pragma unroll
                for (int c = 0; c < P::kChunks; ++c)
                  *reinterpret_cast<uint4*>(smem + P::kOffV + st * P::kStage + c * P::kKVChunk + x * 16) = make_uint4(0, 0, 0, 0);
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              __syncwarp();
            }
          }
          // 16 keys per MMA = two 8-row swizzle groups; 64 columns of d lie kKVChunk apart
          const uint64_t vd = smem_desc(v_at, P::kKVChunk, 1024, kLayoutSw128);
          ok = warp_wait(bar(b_pready + (own & 1)), (own >> 1) & 1, abort_flag, err, 213);
          if (!ok) break;
          tc_fence_after();
          const uint32_t p_at = s_at + TK * (own & 1);
          if (el) {
#pragma unroll
            for (int kk = 0; kk < TK / 16; ++kk)
              mma16_ts(o_at, p_at + kk * 8, vd + (uint64_t)((kk * 16 * 128) >> 4), kIdescO, kk ? 1u : (t > 0 ? 1u : 0u));
            if (kMaySplit && split) {
#pragma unroll
              for (int kk = 0; kk < TK / 16; ++kk)
                mma16_ts(o_at, p_at + TK / 2 + kk * 8, vd + (uint64_t)((kk * 16 * 128) >> 4), kIdescO, 1u);
            }
            tc_commit(bar(b_oready + (own & 1)));
            tc_commit(bar(kQuant ? B_CV + NC + st : B_VEMPTY + st));
          }
          __syncwarp();
          ok = issue_S(t + 2);  // its S buffer is free once the product above is queued (the pipe runs them in order)
        }
        jj += (uint32_t)n;
        done += (uint32_t)n;
      }
    } else if (kQuant && warp >= P::kConvertFrom) {
      // =============================== the tiles of an 8-bit cache ===============================
      if constexpr (kQuant) {
        // K one tile ahead of V, as S runs ahead of P V: K0, K1 V0, K2 V1, ... V(n-1); or V alone
        constexpr int UPT = DP / 16, R = P::kConvert / UPT;  // 16-byte units of a row of codes, rows of one step
        const int tid = threadIdx.x - P::kConvertFrom * 32, r0 = tid / UPT, u = tid % UPT, ch = u / 4, s = ch & 1;
        // the two halves of d would meet in the same banks: the second one turns its pieces round
        const uint32_t to0 = ch * P::kKVChunk + P::unit(r0, (u % 4) * 2 + s), to1 = ch * P::kKVChunk + P::unit(r0, (u % 4) * 2 + (s ^ 1));
        uint32_t jj = 0;
        bool ok = true;
        while (ok && w.next(a)) {
          const int32_t steps = kConvertK ? 2 * w.n : w.n;
          for (int32_t step = 0; step < steps && ok; ++step) {
            const bool is_v = !kConvertK || (step > 0 && ((step & 1) == 0 || step == steps - 1));
            const int32_t t = !kConvertK ? step : step == steps - 1 ? w.n - 1 : (step + 1) / 2 - (is_v ? 1 : 0);
            const uint32_t j = jj + (uint32_t)t;
            const int st = j % NS, done = (is_v ? B_CV : B_CK) + j % NC;
            ok = warp_wait(bar((is_v ? B_VFULL : B_KFULL) + st), (j / NS) & 1, abort_flag, err, 412) &&
                 warp_wait(bar(done + NC), ((j / NC) & 1) ^ 1u, abort_flag, err, 413);
            if (!ok) break;
            int keys = is_v ? a.tile_keys : TK;  // behind them lies what no box reaches
            if (is_v && w.t0 + t == w.tiles - 1) {  // rows behind the sequence's end hold anything
              int32_t first, slot;
              keys = keys_of(w.t0 + t, first, slot);
            }
            const uint8_t* src = smem + (is_v ? P::kOffV : P::kOffK) + st * P::kStage + tid * 16;
            uint8_t* dst = smem + (is_v ? P::kOffCV : P::kOffCK) + j % NC * P::kTile;
#pragma unroll
            for (int i = 0; i < TK / R; ++i) {
              uint4 c = *reinterpret_cast<const uint4*>(src + i * R * DP);
              if (s) c = make_uint4(c.z, c.w, c.x, c.y);
              if (keys < TK && r0 + i * R >= keys) c = make_uint4(0, 0, 0, 0);
              uint4 y0, y1;
              Widen<TC>::four(c.x, y0.x, y0.y);
              Widen<TC>::four(c.y, y0.z, y0.w);
              Widen<TC>::four(c.z, y1.x, y1.y);
              Widen<TC>::four(c.w, y1.z, y1.w);
              *reinterpret_cast<uint4*>(dst + to0 + i * R * 128) = y0;
              *reinterpret_cast<uint4*>(dst + to1 + i * R * 128) = y1;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {  // one arrival a warp: those of 32 lanes would take as many turns at the barrier
              mbar_arrive(bar(done));
              mbar_arrive(bar((is_v ? B_VEMPTY : B_KEMPTY) + st));
            }
          }
          jj += (uint32_t)w.n;
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(P::kRegsSoftmax));
    // =============================== softmax: one thread owns one query row ===============================
    // P = 2^(s - shift). A row's shift is the maximum it was last set at, less kLift: of s, or over an 8-bit cache of s plus the exponent
    // of V's scale (from 2^-80 on), as what is rounded to 16 bits is their product. It is set anew only when that maximum outgrows it
    // by kSlack. A maximum of s and the tile's largest exponent bounds it; where that would set it anew and the tile's scales lie more
    // than 2^kNear apart, the maximum is taken key by key: a large V that a row gives no weight does not count. (64 tokens of 8 heads
    // over 16384 int8 keys 170 us, 265 where scales from 2^-4 to 2^4 are mixed in every tile; 32 sequences of up to 65536 e4m3 keys 712
    // and 744.) A float16 probability times its scale is below 2^(kLift + kSlack + 1) = 2^15 then, the row's largest is at 2^4 at least
    // (native caches 2^8), and the others keep 11 bits down to 2^-18 of it and steps of 2^-28 below. Each new shift holds a warp up for
    // some 2000 cycles, and the product with it: a slack of 4 set one every fourth tile of a sequence of normal numbers.
    // A bfloat16 probability stays below 1: V may be as large as in the kernels that compute in 32 bits.
    // What few tiles need (keys that do not exist, scales far apart) is written small, in a loop over columns that are read from tensor
    // memory again: the code of the other tiles, with that of the other roles, just fits the instruction cache. All of it in registers,
    // calls of 128 rows a unit over 8-bit caches took up to 20 % longer, with four times the cache's misses.
    constexpr bool kHalfP = std::is_same<TP, __half>::value;
    constexpr float kSlack = kHalfP ? 6.f : 8.f, kLift = kHalfP ? 8.f : -8.f;
    constexpr int kNear = 4;
    const uint64_t minus1 = pack2(-1.f, -1.f);
    constexpr uint64_t kMinusZero2 = 0x8000000080000000ull;  // x y + -0 is the product, signs of zeros included
    const int sub = warp / 4, tid = threadIdx.x % 128;
    const uint32_t lane_base = (uint32_t)(warp % 4 * 32) << 16;
    const uint32_t tO = tmem + lane_base + P::kColO + sub * DP, tS0 = tmem + lane_base + P::kColS + 2 * TK * sub;
    const int b_sready = B_SREADY + 2 * sub, b_pready = B_PREADY + 2 * sub, b_oready = B_OREADY + 2 * sub;
    // The four warps of a unit with copies (one row tile). A barrier that is waited for with a limit, like all others: a warp that gave
    // up does not come.
    uint32_t meetings = 0;
    auto group_sync = [&]() -> bool {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_GROUP));
      return warp_wait(bar(B_GROUP), meetings++ & 1, abort_flag, err, 313);
    };
    uint32_t jj = 0, ring = 0;  // tiles of this row tile, and of the CTA
    bool ok = true;

    // One piece. kCols: the columns of a tile that a thread works on, 64 over the number of copies of the unit's rows.
    auto piece = [&](auto cols_tag) -> bool {
      constexpr int kCols = decltype(cols_tag)::value, kCopies = 64 / kCols, kBlock = 128 / kCopies;
      const int rows = w.rows(a) - sub * 128;
      const int row = tid % kBlock, copy = tid / kBlock, col0 = copy * kCols;  // the copy is the warp's
      const bool mine = row < rows;
      if (NSUB > 1 && rows <= 0) {  // the unit has no second tile
        ring += (uint32_t)w.n;
        return true;
      }
      // ---- Q: every product with the last unit's has completed ----
      float sc = a.scale_log2e;
      if (mine) {
        const int32_t xr = w.row0 + sub * 128 + row, t = xr / a.group;
        const T* src = reinterpret_cast<const T*>(a.Q) + (int64_t)(w.begin + t) * a.q_stride[0] +
                       ((int64_t)w.h * a.group + (xr - t * a.group)) * a.q_stride[1];
        uint4 q[DP / 8];  // all in flight together
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
          q[i] = make_uint4(0, 0, 0, 0);
          if (i * 8 < a.c.d) q[i] = __ldg(reinterpret_cast<const uint4*>(src) + i);
        }
        [[maybe_unused]] float f = 1.f;
        if constexpr (kRawK || (kQuant && std::is_same<T, __nv_bfloat16>::value)) {  // times 2^(kTop - exponent of the row's largest element)
          constexpr int kTop = kRawK ? 7 : 14;
          uint32_t top = 0;
#pragma unroll
          for (int i = 0; i < DP / 8; ++i) {
            const uint32_t x = __vmaxu2(__vmaxu2(q[i].x & 0x7fff7fffu, q[i].y & 0x7fff7fffu),
                                        __vmaxu2(q[i].z & 0x7fff7fffu, q[i].w & 0x7fff7fffu));
            top = max(top, max(x & 0xffffu, x >> 16));
          }
          int e = (int)(__float_as_uint(Half16<T>::up(top).x) >> 23) - 127;
          const bool finite = e <= 127;
          e = !finite ? kTop : (e < -100 ? -100 : e);
          f = __uint_as_float((uint32_t)(127 + kTop - e) << 23);
          sc *= __uint_as_float((uint32_t)(127 - kTop + e) << 23);
          if (kRawK && !finite) f = __int_as_float(0x7fc00000);  // e4m3 has no infinities: the row is NaN
        }
        uint8_t* dst = smem + P::kOffQ + sub * P::kQSub;
        if constexpr (kRawK) {
#pragma unroll
          for (int i = 0; i < DP / 8; i += 2) {
            uint32_t codes[kTerms][4];
            const uint32_t v[8] = {q[i].x, q[i].y, q[i].z, q[i].w, q[i + 1].x, q[i + 1].y, q[i + 1].z, q[i + 1].w};
#pragma unroll
            for (int k = 0; k < 8; k += 2) {
              float2 x = Half16<T>::up(v[k]), y = Half16<T>::up(v[k + 1]);
              x = make_float2(x.x * f, x.y * f);
              y = make_float2(y.x * f, y.y * f);
#pragma unroll
              for (int term = 0; term < kTerms; ++term) {
                const uint32_t lo = term == 0 ? take_term<true>(x) : take_term<false>(x);
                const uint32_t hi = term == 0 ? take_term<true>(y) : take_term<false>(y);
                codes[term][k / 2] = lo | (hi << 16);
              }
            }
#pragma unroll
            for (int term = 0; term < kTerms; ++term)
              *reinterpret_cast<uint4*>(dst + term * P::kQChunk + P::unit(tid, i / 2)) =
                  make_uint4(codes[term][0], codes[term][1], codes[term][2], codes[term][3]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < DP / 8; ++i) {
            uint32_t v[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
            if constexpr (kQuant && std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float2 y = Half16<__nv_bfloat16>::up(v[k]);
                v[k] = Half16<__half>::down(y.x * f, y.y * f);
              }
            }
            if constexpr (Widen<TC>::kSwap) {
#pragma unroll
              for (int k = 0; k < 4; k += 2) {
                const uint32_t x = v[k], y = v[k + 1];
                v[k] = (x & 0xffffu) | (y << 16);
                v[k + 1] = (x >> 16) | (y & 0xffff0000u);
              }
            }
            *reinterpret_cast<uint4*>(dst + i / 8 * P::kQChunk + P::unit(tid, i % 8)) = make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
      }  // rows beyond the unit's keep what was there: no row's result depends on another's
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_QFULL + sub));
      if (kCopies == 1 && warp % 4 * 32 >= rows) {  // nothing here: keep step with the barriers
        ring += (uint32_t)w.n;
        for (int32_t t = 0; t < w.n; ++t, ++jj) {
          if (!warp_wait(bar(b_sready + (jj & 1)), (jj >> 1) & 1, abort_flag, err, 315)) return false;
          if (lane == 0) mbar_arrive(bar(b_pready + (jj & 1)));
        }
        return true;
      }
      const bool split = kMaySplit && w.tokens * a.group <= 128;
      float m_true = neg_inf(), shift = neg_inf();
      uint64_t l2[2] = {0ull, 0ull};
      for (int32_t t = 0; t < w.n; ++t, ++jj, ++ring) {
        const uint32_t tS = tS0 + TK * (jj & 1);
        if (!warp_wait(bar(b_sready + (jj & 1)), (jj >> 1) & 1, abort_flag, err, 311)) return false;
        tc_fence_after();
        const uint64_t mask = *reinterpret_cast<volatile uint64_t*>(ring_mask + ring % P::kRing);
        if (mask != ~0ull) {  // keys that do not exist
#pragma unroll 1
          for (int c = 0; c < kCols; c += 16) {
            uint32_t s16[16];
            tmem_ld16(tS + col0 + c, s16);
            tc_wait_ld();
            const uint32_t here = (uint32_t)(mask >> (col0 + c));
#pragma unroll
            for (int e = 0; e < 16; ++e) s16[e] = (here >> e) & 1u ? s16[e] : 0xff800000u;
            tmem_st8(tS + col0 + c, *reinterpret_cast<const uint32_t(*)[8]>(s16));
            tmem_st8(tS + col0 + c + 8, *reinterpret_cast<const uint32_t(*)[8]>(s16 + 8));
          }
          tc_wait_st();
        }
        uint32_t sr[kCols];
        if constexpr (kCols == 16) tmem_ld16(tS + col0, sr);
        if constexpr (kCols == 32) tmem_ld32(tS + col0, sr);
        if constexpr (kCols == 64) {
          tmem_ld32(tS, *reinterpret_cast<uint32_t(*)[32]>(sr));
          tmem_ld32(tS + 32, *reinterpret_cast<uint32_t(*)[32]>(sr + 32));
        }
        [[maybe_unused]] const float* scales = ring_scale + (ring % P::kRing) * 2 * TK + col0;
        [[maybe_unused]] const ulonglong2 *ks = reinterpret_cast<const ulonglong2*>(scales), *vs = reinterpret_cast<const ulonglong2*>(scales + TK);
        [[maybe_unused]] int v_top = 0;  // exponent of the largest of V's scales here, with its bias
        if constexpr (kQuant) {
          const volatile uint32_t* all = reinterpret_cast<const volatile uint32_t*>(scales + TK - col0);
          // NaN is the largest, but then every row of the unit becomes NaN
          v_top = (int)(__reduce_max_sync(kFullMask, max(all[lane] & 0x7fffffffu, all[lane + 32] & 0x7fffffffu)) >> 23);
        }
        tc_wait_ld();
        if constexpr (kQuant) {
#pragma unroll
          for (int e = 0; e < kCols; e += 4) {
            const ulonglong2 f = ks[e / 4];
            float x0, x1, x2, x3;
            unpack2(fma2(pack2(__uint_as_float(sr[e]), __uint_as_float(sr[e + 1])), f.x, kMinusZero2), x0, x1);
            unpack2(fma2(pack2(__uint_as_float(sr[e + 2]), __uint_as_float(sr[e + 3])), f.y, kMinusZero2), x2, x3);
            sr[e] = __float_as_uint(x0);
            sr[e + 1] = __float_as_uint(x1);
            sr[e + 2] = __float_as_uint(x2);
            sr[e + 3] = __float_as_uint(x3);
          }
        }
        float mx[4] = {neg_inf(), neg_inf(), neg_inf(), neg_inf()};
#pragma unroll
        for (int e = 0; e < kCols; e += 2)
          mx[(e >> 1) & 3] = fmaxf(fmaxf(mx[(e >> 1) & 3], __uint_as_float(sr[e])), __uint_as_float(sr[e + 1]));
        const float t_max = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc;  // sc > 0
        m_true = fmaxf(m_true, t_max);
        float want = kQuant ? t_max + ((float)(min(max(v_top, 47), 227) - 127) - kLift) : t_max - kLift;
        bool move = want > shift + kSlack;
        if (__any_sync(kFullMask, move)) {
          if constexpr (kQuant) {  // a closer look, before it is believed
            const volatile uint32_t* all = reinterpret_cast<const volatile uint32_t*>(scales + TK - col0);
            const uint32_t x = all[lane] & 0x7fffffffu, y = all[lane + 32] & 0x7fffffffu;
            const int low = (int)(__reduce_min_sync(kFullMask, min(x ? x : ~0u, y ? y : ~0u)) >> 23);  // zeros (also: no key) do not count
            if (v_top - low > kNear) {
              float best = neg_inf();
#pragma unroll 1
              for (int c = 0; c < kCols; c += 4) {
                uint32_t s4[4];
                tmem_ld4(tS + col0 + c, s4);
                const float4 fk = *reinterpret_cast<const float4*>(scales + c);
                const uint4 fv = *reinterpret_cast<const uint4*>(scales + TK + c);
                tc_wait_ld();
                auto one = [&](uint32_t raw, float k, uint32_t v) {
                  const float y = fmaf(__uint_as_float(raw) * k, sc, (float)(int)(v >> 23));
                  if (v) best = fmaxf(best, y);
                };
                one(s4[0], fk.x, fv.x);
                one(s4[1], fk.y, fv.y);
                one(s4[2], fk.z, fv.z);
                one(s4[3], fk.w, fv.w);
              }
              want = fminf(fmaxf(best - 127.f, t_max - 80.f), t_max + 100.f) - kLift;
              move = want > shift + kSlack;
            }
          }
          const float new_shift = move ? want : shift;
          // Scales lie up to 2^180 apart, and so do shifts, whatever the scores are: what a factor of 2^-180 leaves of l may still be most
          // of it. So the factor's root, twice.
          const float f = move ? ((shift == neg_inf()) ? 0.f : fast_exp2(kQuant ? 0.5f * (shift - new_shift) : shift - new_shift)) : 1.0f;
          const uint64_t f2 = pack2(f, f);
#pragma unroll
          for (int i = 0; i < (kQuant ? 2 : 1); ++i) {
            l2[0] = fma2(l2[0], f2, 0ull);
            l2[1] = fma2(l2[1], f2, 0ull);
          }
          const float f_O = kQuant ? f * f : f;
          if (t > 0) {  // O of this row up to the previous tile is final once that tile's barrier has completed
            if (!warp_wait(bar(b_oready + ((jj - 1) & 1)), ((jj - 1) >> 1) & 1, abort_flag, err, 312)) return false;
            tc_fence_after();
            uint32_t ob[32];
#pragma unroll 1
            for (int c = 0; c < DP / 32; ++c) {
              tmem_ld32(tO + c * 32, ob);
              tc_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) ob[e] = __float_as_uint(__uint_as_float(ob[e]) * f_O);
              tmem_st32(tO + c * 32, ob);
            }
          }
          shift = new_shift;
        }
        const float neg_shift = (shift == neg_inf()) ? 0.f : -shift;
        const uint64_t ns2 = pack2(neg_shift, neg_shift), sc2 = pack2(sc, sc);
        // the first term, and with kLo the second: what the rounding left. The columns of other copies are zeros here.
        auto probabilities = [&](auto lo_tag) {
          constexpr bool kLo = decltype(lo_tag)::value;
          uint32_t hi[kCols / 2], lo[kLo ? kCols / 2 : 1];
#pragma unroll
          for (int e = 0; e < kCols / 2; ++e) {
            float x0, x1;
            unpack2(fma2(pack2(__uint_as_float(sr[2 * e]), __uint_as_float(sr[2 * e + 1])), sc2, ns2), x0, x1);
            uint64_t p = pack2(fast_exp2(x0), fast_exp2(x1));
            l2[e & 1] = add2(l2[e & 1], p);
            if constexpr (kQuant) {
              const ulonglong2 f = vs[e / 2];
              p = fma2(p, e & 1 ? f.y : f.x, kMinusZero2);
            }
            float p0, p1;
            unpack2(p, p0, p1);
            hi[e] = Half16<TP>::down(p0, p1);
            if constexpr (kLo) {
              const float2 h = Half16<TP>::up(hi[e]);
              unpack2(fma2(pack2(h.x, h.y), minus1, p), p0, p1);  // exact
              lo[e] = Half16<TP>::down(p0, p1);
            }
          }
          auto store = [&](uint32_t to, const uint32_t* x) {
            if constexpr (kCopies == 1) {
              tmem_st32(to, *reinterpret_cast<const uint32_t(*)[32]>(x));
            } else {
              const uint32_t zero[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if (i / (kCols / 16) == copy) tmem_st8(to + i * 8, *reinterpret_cast<const uint32_t(*)[8]>(x + i % (kCols / 16) * 8));
                else tmem_st8(to + i * 8, zero);
              }
            }
          };
          store(tS, hi);
          if constexpr (kLo) store(tS + 32, lo);
        };
        if (kMaySplit && split) probabilities(std::integral_constant<bool, kMaySplit>());
        else probabilities(std::integral_constant<bool, false>());
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(b_pready + (jj & 1)));
      }
      // ---- the piece's rows leave ----
      if (!warp_wait(bar(b_oready + ((jj - 1) & 1)), ((jj - 1) >> 1) & 1, abort_flag, err, 314)) return false;
      tc_fence_after();
      float la, lb, lc, ld;
      unpack2(l2[0], la, lb);
      unpack2(l2[1], lc, ld);
      const float l_run = (la + lb) + (lc + ld);
      float rel = (m_true == neg_inf()) ? 0.f : fast_exp2(shift - m_true);
      // a NaN score passes the maximum by and shows in the sum
      float m = (l_run != l_run && m_true < __int_as_float(0x7f800000)) ? l_run : m_true, l = l_run * rel;
      if constexpr (kCopies > 1) {
        row_ml[tid] = make_float2(m, l);
        if (!group_sync()) return false;
        float top = neg_inf();
#pragma unroll
        for (int c = 0; c < kCopies; ++c) top = max_nan(top, row_ml[c * kBlock + row].x);
        const float ref = top == neg_inf() ? 0.f : top;
        rel *= fast_exp2(m - ref);
        l = 0.f;
#pragma unroll
        for (int c = 0; c < kCopies; ++c) {
          const float2 x = row_ml[c * kBlock + row];
          l += x.y * fast_exp2(x.x - ref);
        }
        m = top;
      }
      const int64_t out = a.partial_row(w.begin, w.tokens, w.h, w.row0 + sub * 128, blockIdx.x);
      if (mine && copy == 0) a.ml[out + row] = make_float2(m, l);
      [[maybe_unused]] Infinities<DP> found;
      [[maybe_unused]] bool searched = false;
      constexpr int kAtOnce = P::kQSub / (128 * 128) >= 2 && DP >= 64 ? 2 : 1;  // pieces of 32 columns that find room where Q was
#pragma unroll 1
      for (int c = 0; c < DP / 32; ++c) {
        uint32_t ob[32];
        tmem_ld32(tO + c * 32, ob);
        tc_wait_ld();
        [[maybe_unused]] uint64_t zero[2] = {0ull, 0ull};  // stay 0 while every value is finite
        if constexpr (!kQuant) {
#pragma unroll
          for (int e = 0; e < 32; e += 2)
            zero[(e >> 1) & 1] = fma2(pack2(__uint_as_float(ob[e]), __uint_as_float(ob[e + 1])), 0ull, zero[(e >> 1) & 1]);
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) ob[e] = __float_as_uint(__uint_as_float(ob[e]) * rel);
        if constexpr (!kQuant) {  // (a row whose sum is NaN is that throughout)
          if (__any_sync(kFullMask, mine && l == l && ((zero[0] | zero[1]) & 0x7fffffff7fffffffull) != 0ull)) {
            if (!searched) {
              int32_t first, last, slot, end_slot;
              keys_of(w.t0, first, slot);
              const int left = keys_of(w.t0 + w.n - 1, last, end_slot);
              find_infinities<DP, T>(a, w.b, w.h, (int64_t)first * ps + slot, (int64_t)last * ps + end_slot + left, found);
              searched = true;
            }
            uint32_t up = 0, down = 0, nan = 0;
#pragma unroll
            for (int k = 0; k < DP / 32; ++k)
              if (k == c) {
                up = found.up[k];
                down = found.down[k];
                nan = found.nan[k];
              }
            if (l == l) {
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (((up | down | nan) >> e) & 1u) ob[e] = (nan >> e) & 1u ? 0x7fc00000u : (up >> e) & 1u ? 0x7f800000u : 0xff800000u;
            }
          }
        }
        constexpr int kA = Widen<TC>::kSwap ? 2 : 1, kB = 3 - kA;  // the columns of 1 and 2
        auto four = [&](int e) { return make_uint4(ob[e], ob[e + kA], ob[e + kB], ob[e + 3]); };
        if constexpr (kCopies == 1) {
          if (mine) {
            float* dst = a.O + (out + row) * a.d_pad + c * 32;
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              if (c * 32 + e < a.d_pad) *reinterpret_cast<uint4*>(dst + e) = four(e);
          }
          __syncwarp();
        } else {  // the copies are added up where Q was
          const int part = c % kAtOnce;
#pragma unroll
          for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4*>(smem + P::kOffQ + part * P::kQChunk + P::unit(tid, e / 4)) = four(e);
          if (part < kAtOnce - 1) continue;
          if (!group_sync()) return false;
          for (int x = tid; x < rows * 8 * kAtOnce; x += 128) {
            const int r = x / (8 * kAtOnce), u = x % (8 * kAtOnce), col = (c - part) * 32 + u * 4;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < kCopies; ++k) {
              const float4 z = *reinterpret_cast<const float4*>(smem + P::kOffQ + u / 8 * P::kQChunk + P::unit(k * kBlock + r, u % 8));
              y = make_float4(y.x + z.x, y.y + z.y, y.z + z.z, y.w + z.w);
            }
            if (col < a.d_pad) *reinterpret_cast<float4*>(a.O + (out + r) * a.d_pad + col) = y;
          }
          if (!group_sync()) return false;
        }
      }
      tc_fence_before();
      return true;
    };
    while (ok && w.next(a)) {
      const int rows = w.rows(a);
      if constexpr (NSUB > 1) {
        ok = piece(std::integral_constant<int, 64>());
        continue;
      }
      if (rows <= 32) ok = piece(std::integral_constant<int, 16>());
      else if (rows <= 64) ok = piece(std::integral_constant<int, 32>());
      else ok = piece(std::integral_constant<int, 64>());
    }
  }

  // ---- common exit: everyone is done with TMEM before it is released ----
  tc_fence_before();
  __syncthreads();
  if (warp == P::kAux) {
    tc_fence_after();
    if (*abort_flag && lane == 0) {  // copies that may still be in flight land before the CTA's shared memory is reused
      const uint64_t t0 = globaltimer();
      while (globaltimer() - t0 < 2000000ull) {
      }
    }
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(P::kTmemCols) : "memory");
  }
}

}  // namespace tree
}  // namespace spfa
