// The copy-ring tile product shared by the grouped output projection, the decode-row projections and the
// adapter projections: sums of one weight-row x query-row tile over one contraction range, both operands
// copied global -> LDS (global_load_lds_dwordx4) in 32- or 64-channel steps.
#pragma once

#include "mfma.h"

namespace dsv41 {

struct WoaArgs {
  const bf16_t* o;     // [rows, groups * d]
  const bf16_t* w;     // [groups * r, d]; split: [r, groups * d]
  void* out;           // [rows, groups * r], bf16 or fp32
  int rows, groups, d, r;
  int split;           // 1: one dense weight whose contraction is cut into `groups` ranges of d
  const bf16_t* w1;    // split only: weight rows [r0, r) come from w1 [r - r0, groups * d]
  int r0;              // (two weights applied to the same rows; r0 a multiple of the tile's rows)
};

// Two 16 x 16 tiles of results side by side (lane (g, l16): columns 4 g .. 4 g + 3 of row l16 of each) as bf16: after two
// row swaps a lane holds columns 8 (g / 2) .. + 7 of tile g % 2, so that a row's 32 columns are one 64-byte store of its
// four lanes. Swaps use every lane.
__device__ __forceinline__ uint4 pair_of(f32x4 v0, f32x4 v1) {
  const auto lo = __builtin_amdgcn_permlane16_swap(pack2_bf16(v0[0], v0[1]), pack2_bf16(v1[0], v1[1]), false, false);
  const auto hi = __builtin_amdgcn_permlane16_swap(pack2_bf16(v0[2], v0[3]), pack2_bf16(v1[2], v1[3]), false, false);
  return make_uint4(lo[0], hi[0], lo[1], hi[1]);
}

// Four consecutive outputs of one query row.
template <typename TO>
__device__ __forceinline__ void store4(TO* p, f32x4 v);
template <>
__device__ __forceinline__ void store4<bf16_t>(bf16_t* p, f32x4 v) {
  uint2 s;
  s.x = pack2_bf16(v[0], v[1]);
  s.y = pack2_bf16(v[2], v[3]);
  *reinterpret_cast<uint2*>(p) = s;
}
template <>
__device__ __forceinline__ void store4<float>(float* p, f32x4 v) {
  *reinterpret_cast<f32x4*>(p) = v;
}

constexpr int kTileR = 128;   // weight rows of the smallest output tile (r is a multiple of it)
constexpr int kWideR = 256;   // weight rows of the large tile

// 16-byte chunk c of tile row `row` (rows of BK bf16: BK / 8 chunks) sits at slot c ^ swz(row).
// A fragment read takes one chunk of 16 consecutive rows; with these slots no two of those lanes
// share a bank, whether the banks serve 8 lanes of 16 bytes (128 bytes) per cycle or 16 lanes
// (256 bytes).
template <int BK>
__device__ __forceinline__ int tile_swz(int row) {
  if constexpr (BK == 64) return (row & 7) ^ ((row >> 3) & 1);
  else return ((row >> 1) & 3) ^ ((row >> 3) & 1);
}

// Output tile of 16 WR GR weight rows x 16 WM GM query rows: a GR x GM grid of waves, each
// 16 WR x 16 WM (WR x WM MFMA tiles). BK channels per step; NS steps of both operand tiles in LDS
// at once (NS - 1 in flight while one is multiplied).
template <int WR, int WM, int GR, int GM, int BK, int NS>
struct TileCfg {
  static constexpr int NWV = GR * GM, NT = 64 * NWV;
  static constexpr int TR = 16 * WR * GR, TM = 16 * WM * GM;
  static constexpr int RB = BK * 2;                 // bytes per tile row
  static constexpr int CPR = BK / 8;                // 16-byte chunks per row
  static constexpr int RPI = 1024 / RB;             // rows per copy instruction
  static constexpr int NW = TR * RB / (1024 * NWV), NO = TM * RB / (1024 * NWV);   // copies per wave per step
  static constexpr int STAGE = (TR + TM) * RB;
  static constexpr int LDS = NS * STAGE;
  static_assert(BK == 32 || BK == 64, "32- or 64-channel steps");
};

// The same for deep rings: at most `pending` (clamped to P) later steps of N copies each may
// stay in flight; N * P stays within the 6-bit vmcnt field.
template <int N, int P>
__device__ __forceinline__ void wait_copies_deep(int pending) {
  static_assert(N * P <= 63, "vmcnt holds 6 bits");
  if constexpr (P > 0) {
    if (pending >= P) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N * P) : "memory");
      return;
    }
    wait_copies_deep<N, P - 1>(pending);
  } else {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
}

template <int N>
__device__ __forceinline__ void wait_copies(int pending) {
  // at most `pending` later steps of per_step copies each may stay in flight
  if constexpr (N >= 3) {
    if (pending >= 3) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(3 * N) : "memory");
      return;
    }
  }
  if constexpr (N >= 2) {
    if (pending == 2) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * N) : "memory");
      return;
    }
  }
  if (pending >= 1) {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
    return;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// Sums of output tile (rt, mt) over contraction range or group grp, left in acc: lane (g, l16) of a wave holds
// weight rows 16 i + 4 g .. + 3 and query row 16 j + l16 of the wave's block. lds: C::LDS bytes, 16-byte aligned.
// beside() runs once the ring's first copies are on their way, on sums of zero, which it may add to; what it leaves
// outstanding it waits for itself.
struct NothingBeside {
  __device__ __forceinline__ void operator()() const {}
};
template <int WR, int WM, int GR, int GM, int BK, int NS, typename Beside = NothingBeside>
__device__ __forceinline__ void tile_sums(const WoaArgs& a, uint8_t* lds, int rt, int mt, int grp,
                                          f32x4 (&acc)[WR][WM], Beside beside = Beside()) {
  using C = TileCfg<WR, WM, GR, GM, BK, NS>;
  static_assert(C::NW * 1024 * C::NWV == C::TR * C::RB && C::NO * 1024 * C::NWV == C::TM * C::RB,
                "whole copy instructions per wave");
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wr = (wave % GR) * 16 * WR, wm = (wave / GR) * 16 * WM;   // this wave's block

  // copy sources: wave w fills rows [w TR/NWV, (w+1) TR/NWV) of the weight tile and [w TM/NWV, ..)
  // of the query tile, RPI rows per instruction; lane l writes slot l % CPR of row l / CPR of its
  // instruction's rows, i.e. chunk slot ^ swz(row) of that row
  uint64_t wsrc[C::NW], osrc[C::NO];
#pragma unroll
  for (int j = 0; j < C::NW; ++j) {
    const int row = wave * (C::TR / C::NWV) + j * C::RPI + lane / C::CPR;
    const int chunk = (lane % C::CPR) ^ tile_swz<BK>(row);
    // grouped: group grp's weight rows; split: range grp of every weight row (row stride groups * d),
    // rows from r0 on in w1 when it is given
    const int wr_all = rt * C::TR + row;
    const bool second = a.w1 != nullptr && wr_all >= a.r0;
    const bf16_t* wbase = second ? a.w1 : a.w;
    const int64_t wrow = a.split ? (int64_t)(second ? wr_all - a.r0 : wr_all) * ((int64_t)a.groups * a.d) + (int64_t)grp * a.d
                                 : ((int64_t)grp * a.r + wr_all) * a.d;
    wsrc[j] = reinterpret_cast<uint64_t>(wbase + wrow + 8 * chunk);
  }
#pragma unroll
  for (int j = 0; j < C::NO; ++j) {
    const int row = wave * (C::TM / C::NWV) + j * C::RPI + lane / C::CPR;
    const int chunk = (lane % C::CPR) ^ tile_swz<BK>(row);
    const int64_t orow = min(mt * C::TM + row, a.rows - 1);   // rows past the end: not stored
    osrc[j] = reinterpret_cast<uint64_t>(a.o + orow * a.groups * a.d + (int64_t)grp * a.d + 8 * chunk);
  }
  const uint32_t lds0 = lds_offset(lds);
  auto issue = [&](int buf, int k) {
    const uint32_t wdst = (uint32_t)__builtin_amdgcn_readfirstlane(
        (int)(lds0 + (uint32_t)(buf * C::STAGE) + (uint32_t)(wave * (C::TR / C::NWV) * C::RB)));   // wave-uniform: M0
    const uint32_t odst = (uint32_t)__builtin_amdgcn_readfirstlane(
        (int)(lds0 + (uint32_t)(buf * C::STAGE + C::TR * C::RB) + (uint32_t)(wave * (C::TM / C::NWV) * C::RB)));
    const uint64_t kb = (uint64_t)k * 2;
#pragma unroll
    for (int j = 0; j < C::NW; ++j) dma16_vaddr(wsrc[j] + kb, wdst + j * 1024);
#pragma unroll
    for (int j = 0; j < C::NO; ++j) dma16_vaddr(osrc[j] + kb, odst + j * 1024);
  };
  auto frag = [&](const uint8_t* t, int row, int chunk) {
    return as_bf16x8(*reinterpret_cast<const uint4*>(t + row * C::RB + ((chunk ^ tile_swz<BK>(row)) << 4)));
  };

#pragma unroll
  for (int i = 0; i < WR; ++i)
#pragma unroll
    for (int j = 0; j < WM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // One barrier per step: after it, step kt is in LDS for every wave and every wave is done with
  // step kt - 1, whose buffer then takes step kt + NS - 1.
  const int nk = a.d / BK;
#pragma unroll
  for (int p = 0; p < NS - 1; ++p)
    if (p < nk) issue(p, p * BK);
  beside();
  for (int kt = 0; kt < nk; ++kt) {
    if constexpr (NS <= 4) wait_copies<C::NW + C::NO>(min(NS - 2, nk - 1 - kt));   // this wave's copies of step kt landed
    else wait_copies_deep<C::NW + C::NO, NS - 2>(min(NS - 2, nk - 1 - kt));
    __syncthreads();
    if (kt + NS - 1 < nk) issue((kt + NS - 1) % NS, (kt + NS - 1) * BK);
    const uint8_t* wt = lds + (kt % NS) * C::STAGE;
    const uint8_t* qt = wt + C::TR * C::RB;
#pragma unroll
    for (int ks = 0; ks < BK / 32; ++ks) {
      bf16x8 af[WR], bf[WM];
#pragma unroll
      for (int i = 0; i < WR; ++i) af[i] = frag(wt, wr + 16 * i + l16, 4 * ks + g);
#pragma unroll
      for (int j = 0; j < WM; ++j) bf[j] = frag(qt, wm + 16 * j + l16, 4 * ks + g);
#pragma unroll
      for (int i = 0; i < WR; ++i)
#pragma unroll
        for (int j = 0; j < WM; ++j) acc[i][j] = mfma16x16x32(af[i], bf[j], acc[i][j]);
    }
  }
}

// tile_sums for large tiles (the split form, r0 a multiple of the tile's weight rows; two ring stages of 64 channels):
// the fragments of each 32-channel half step are read while the half before is multiplied, across the step's barrier
// too. Half way through a step every wave has its second half in registers, so the barrier there frees the step's stage
// for the copies of the step after next, which then have a whole step to land. Same order of additions as tile_sums.
template <int WR, int WM, int GR, int GM, typename Beside = NothingBeside>
__device__ __forceinline__ void tile_sums_ahead(const WoaArgs& a, uint8_t* lds, int rt, int mt, int grp,
                                                f32x4 (&acc)[WR][WM], Beside beside = Beside()) {
  using C = TileCfg<WR, WM, GR, GM, 64, 2>;
  static_assert(C::TR % (8 * C::NWV) == 0 && C::TM % (8 * C::NWV) == 0 && C::NWV % 2 == 0,
                "copies of 8 tile rows, in turn over the waves");
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wr = (wave % GR) * 16 * WR, wm = (wave / GR) * 16 * WM;
  const uint32_t row_bytes = (uint32_t)a.groups * (uint32_t)a.d * 2;
  // Copies of 8 tile rows in turn over the waves: copy j of a wave takes rows 8 (wave + NWV j) .. + 7. Sources: a
  // wave-uniform base, the lane's row and swizzled chunk (tile_swz: the row's low bits and the parity of wave + NWV j,
  // the wave's) as a 32-bit offset.
  constexpr int kW = C::TR / 8 / C::NWV, kO = C::TM / 8 / C::NWV, kCopies = kW + kO, kFrags = WM + WR;
  const uint32_t chunk = 16u * (uint32_t)((lane & 7) ^ (lane >> 3) ^ (wave & 1));
  const uint32_t woff = (uint32_t)(lane >> 3) * row_bytes + chunk;
  uint32_t ooff[kO];
#pragma unroll
  for (int j = 0; j < kO; ++j)
    ooff[j] = (uint32_t)min(8 * (wave + C::NWV * j) + (lane >> 3), a.rows - 1 - mt * C::TM) * row_bytes + chunk;
  const int uwave = __builtin_amdgcn_readfirstlane(wave);
  const uint64_t range = (uint64_t)grp * a.d * 2;
  const bool second = a.w1 != nullptr && rt * C::TR >= a.r0;
  const uint64_t wbase = reinterpret_cast<uint64_t>(second ? a.w1 : a.w) + range +
                         ((uint64_t)(rt * C::TR - (second ? a.r0 : 0)) + (uint64_t)(8 * uwave)) * row_bytes;
  const uint64_t obase = reinterpret_cast<uint64_t>(a.o) + range + (uint64_t)mt * C::TM * row_bytes;
  const uint32_t lds0 = lds_offset(lds);
  // copies [first, last) of a step, the weight's first
  auto issue = [&](int stage, int kt, int first, int last) {
    const uint32_t at = (uint32_t)__builtin_amdgcn_readfirstlane((int)(lds0 + (uint32_t)(stage * C::STAGE + 8 * uwave * C::RB)));
    const uint64_t kb = (uint64_t)kt * C::RB;
#pragma unroll
    for (int c = 0; c < kCopies; ++c) {
      if (c < first || c >= last) continue;
      if (c < kW)
        dma16_sgpr(wbase + kb + (uint64_t)(8 * C::NWV * c) * row_bytes, woff, at + (uint32_t)(8 * C::NWV * c * C::RB));
      else
        dma16_sgpr(obase + kb, ooff[c - kW], at + (uint32_t)((C::TR + 8 * C::NWV * (c - kW)) * C::RB));
    }
  };
  const int swz = (l16 & 7) ^ (l16 >> 3);
  const uint8_t* wl = lds + (wr + l16) * C::RB;
  const uint8_t* ol = lds + C::TR * C::RB + (wm + l16) * C::RB;
  // fragments [first, last) of a half step: the query's, then the weight's in the order of their use
  auto read = [&](int stage, int half, int first, int last, bf16x8 (&af)[WR], bf16x8 (&bf)[WM]) {
    const int at = stage * C::STAGE + (((4 * half + g) ^ swz) << 4);
#pragma unroll
    for (int f = 0; f < kFrags; ++f) {
      if (f < first || f >= last) continue;
      if (f < WM) bf[f] = as_bf16x8(*reinterpret_cast<const uint4*>(ol + at + 16 * f * C::RB));
      else af[f - WM] = as_bf16x8(*reinterpret_cast<const uint4*>(wl + at + 16 * (f - WM) * C::RB));
    }
  };
  auto multiply = [&](int i, const bf16x8 (&af)[WR], const bf16x8 (&bf)[WM]) {
#pragma unroll
    for (int j = 0; j < WM; ++j) acc[i][j] = mfma16x16x32(af[i], bf[j], acc[i][j]);
    __builtin_amdgcn_sched_barrier(0);
  };
#pragma unroll
  for (int i = 0; i < WR; ++i)
#pragma unroll
    for (int j = 0; j < WM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int nk = a.d / 64;
  bf16x8 a0[WR], b0[WM], a1[WR], b1[WM];
  // Eight waves, alone on their CU: reads and copies between the products, a few at a time. In a burst behind the barrier
  // both waves of a SIMD issue them at once and its matrix core waits (8,192 rows 8192 -> 5120: 699 us, 620 between).
  // Four waves with a second workgroup beside them fare better with the burst (4,096 rows: 340 us, 375 between).
  constexpr bool kBetween = C::NWV == 8;
  issue(0, 0, 0, kCopies);
  if (nk > 1) issue(1, 1, 0, kCopies);
  beside();
  if (nk > 1) wait_vmcnt<kCopies>();
  else wait_vmcnt<0>();
  __syncthreads();
  read(0, 0, 0, kFrags, a0, b0);
  for (int kt = 0; kt < nk; ++kt) {
    const int stage = kt & 1;
    const bool copy = kt + 2 < nk, more = kt + 1 < nk;
    if constexpr (kBetween) {
#pragma unroll
      for (int i = 0; i < WR; ++i) {
        read(stage, 1, i * kFrags / WR, (i + 1) * kFrags / WR, a1, b1);
        multiply(i, a0, b0);
      }
    } else {
      read(stage, 1, 0, kFrags, a1, b1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < WR; ++i) multiply(i, a0, b0);
    }
    // step kt + 1, issued a step ago, has landed, and this wave has read stage `stage`; then every wave's
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();
    if constexpr (kBetween) {
#pragma unroll
      for (int i = 0; i < WR; ++i) {
        if (copy) issue(stage, kt + 2, i * kCopies / WR, (i + 1) * kCopies / WR);
        if (more) read(stage ^ 1, 0, i * kFrags / WR, (i + 1) * kFrags / WR, a0, b0);
        multiply(i, a1, b1);
      }
    } else {
      if (copy) issue(stage, kt + 2, 0, kCopies);
      if (more) read(stage ^ 1, 0, 0, kFrags, a0, b0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < WR; ++i) multiply(i, a1, b1);
    }
  }
}

// Split contraction at 33-64 query rows: 128- or 160-row weight tiles where each range is long
// (>= 1024 channels) and the tiles fill the chip once (128-256 workgroups; of the two, the one with
// more workgroups). A 32-row tile reads the 64 query rows from L2 for every 32 weight rows it
// streams, twice the weight's bytes; a 128-row one half of them (measured at 64 rows: wq_b
// 1280 -> 32768 19.1 us against 21.5 for hipBLASLt; wo_b 8192 -> 5120 in 4 ranges on 128-row tiles
// 26.5 us, 160 workgroups, and in 8 ranges on 160-row tiles 23.4-23.8 us, 256 workgroups, against
// 29.6-30.1 for hipBLASLt; 32-row tiles 32.8 us). Returns the tile's weight rows, 0 for none.
__host__ __device__ inline int wide_split_tile(int rows, int d, int n, int ranges) {
  if (rows <= 32 || rows > 64 || d < 1024) return 0;
  int best = 0;
  int64_t best_t = 0;
  for (int tr = 128; tr <= 160; tr += 32) {
    const int64_t t = (int64_t)(n / tr) * ranges;
    if (n % tr == 0 && t >= 128 && t <= 256 && t > best_t) {
      best = tr;
      best_t = t;
    }
  }
  return best;
}

}  // namespace dsv41
