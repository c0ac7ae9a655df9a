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
  static_assert(NW * 1024 * NWV == TR * RB && NO * 1024 * NWV == TM * RB, "whole copy instructions per wave");
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
// beside() runs once the ring's first copies are on their way; what it leaves outstanding it waits for itself.
struct NothingBeside {
  __device__ __forceinline__ void operator()() const {}
};
template <int WR, int WM, int GR, int GM, int BK, int NS, typename Beside = NothingBeside>
__device__ __forceinline__ void tile_sums(const WoaArgs& a, uint8_t* lds, int rt, int mt, int grp,
                                          f32x4 (&acc)[WR][WM], Beside beside = Beside()) {
  using C = TileCfg<WR, WM, GR, GM, BK, NS>;
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
