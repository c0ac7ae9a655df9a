// Products of 8-bit rows and 8-bit weights (mx8.h has the format) on the block-scaled matrix instructions:
//
//   y[m, j] = bf16(act(sum_k x[m, k] w[j, k] + bias[j]) + residual[m, j])
//
// The block-scaled instructions multiply e4m3 codes, apply both operands' scale bytes per 32 channels and add the sum of 64 or
// 128 products to a float32 accumulator. Products are exact. They are summed eight neighbouring channels at a time, lined
// up at the largest of the eight, and of each what lies under 2^-13 of that one's power of two is cut off; the eights'
// sums keep float32's bits. So a result is within 7 * 2^-13 of sum |x w| of the exact one at worst (1.4e-5 of it, in the
// 2-norm, on normal values), which is little beside its one rounding to bf16 (2^-8): results are bf16 only. Dequantizing to
// bf16 instead would keep every bit and cost half the matrix rate or more.
#include <type_traits>
#include <utility>

#include "mx8.h"
#include "tiles.h"

namespace dsv41 {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) int i32x4;

enum Act { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

struct Mx8Args {
  const uint8_t* x;      // [rows, k] codes
  const uint8_t* xs;     // [rows, k / 32] scales
  const uint8_t* w[2];   // [n[i], k] codes
  const uint8_t* ws[2];  // [ceil(n[i] / 2^shift), k / 32] scales
  bf16_t* y[2];          // [rows, n[i]]
  const float* bias;     // [n[0]], or null
  const bf16_t* residual;  // [rows, n[0]], or null
  int n[2];              // a second product of the same rows, or 0
  int tiles0, tiles;     // weight tiles of the first product and of both
  int mtiles, panel;     // tiles of x's rows, and how many of them one weight tile meets before the next
  int whole;             // tiles that are multiplied whole, where others are in parts
  int rows, k, shift, act;
};

// This workgroup's weight tile and tile of x's rows. Workgroups go round the eight XCDs; each XCD takes a run of the tiles,
// in panels of a few tiles of x under all weight tiles, so that what its CUs multiply at a time is a block of both and its
// L2 brings every line once for several of them.
struct TileAt {
  int w, m;
};
__device__ __forceinline__ TileAt tile_of(const Mx8Args& a, int unit) {
  const int panel = unit / (a.panel * a.tiles), at = unit - panel * a.panel * a.tiles;
  const int high = min(a.panel, a.mtiles - panel * a.panel);
  return TileAt{at / high, panel * a.panel + at % high};
}

__device__ __forceinline__ TileAt tile_at(const Mx8Args& a, int total) {
  const int b = (int)blockIdx.x, xcd = b % 8;
  return tile_of(a, xcd * (total / 8) + min(xcd, total % 8) + b / 8);
}

// The part of a call that one workgroup's weight tile belongs to.
struct Mx8Side {
  const uint8_t* w;
  const uint8_t* ws;
  bf16_t* y;
  int n, tile;
};
__device__ __forceinline__ Mx8Side side_of(const Mx8Args& a, int tile, int split = 1) {      // split: parts of the call's tiles
  const int i = tile >= split * a.tiles0;
  return Mx8Side{a.w[i], a.ws[i], a.y[i], a.n[i], tile - (i ? split * a.tiles0 : 0)};
}

__device__ __forceinline__ i32x8 join(i32x4 lo, i32x4 hi) {
  return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// v (1 + erf(v / sqrt 2)) / 2. With a = |v|, erfc(a / sqrt 2) / 2 = q(a) exp(-a^2 / 2), and q is t (c1 + c2 t + .. + c6 t^5) with
// t = 1 / (1 + 0.3085 a): the coefficients of least largest relative error over 0 <= a <= 14.5, 4.1e-6 (a linear program over
// 1,200 points; the factor in t is the best one to four digits). The left tail is v q exp(-a^2 / 2), without 1 + erf's cancellation, and
// keeps its relative error: some (93 + 1.25 v^2) 2^-24 with the roundings, far under bf16's half step down to the type's smallest
// normal value (a formula whose error is absolute, 1.5e-7, is off by 0.16 % at -5, 1 % at -8). 8,192 rows 2304 -> 1112: 36.9 us, 31.5
// without.
__device__ __forceinline__ float gelu(float v) {
  const float t = __builtin_amdgcn_rcpf(1.0f + 0.3085f * fabsf(v)), e = __expf(-0.5f * v * v);
  const float q = t * (0.123305418f + t * (0.119289074f + t * (0.135692362f +
                  t * (0.009501506f + t * (0.187247440f + t * -0.075037509f)))));
  return v >= 0.0f ? v * (1.0f - q * e) : v * q * e;
}

// v / (1 + exp(-v)) by the hardware's exponential and reciprocal, numerator and denominator 2^8 times too small: the denominator then
// has a normal reciprocal until the result is under the smallest normal value (unscaled it ends at v = -87.3, where results are
// -1e-36). Some (16 + 1.5 |v|) 2^-24 of the result, far under its rounding to bf16. 8,192 rows 2304 -> 1112 32.6 -> 32.9 us (none: 32.1).
__device__ __forceinline__ float silu(float v) {
  const float u = __builtin_amdgcn_exp2f(__builtin_fmaf(v, -1.44269504f, -8.0f));
  return v * 0x1p-8f * __builtin_amdgcn_rcpf(u + 0x1p-8f);
}

// v[e] = act(v[e]), the choice outside of the values.
template <int N, typename V>
__device__ __forceinline__ void activate(V& v, int act) {
  if (act == ACT_RELU) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = v[e] > 0.0f || v[e] != v[e] ? v[e] : 0.0f;
  } else if (act == ACT_SILU) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = silu(v[e]);
  } else if (act == ACT_GELU) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = gelu(v[e]);
  }
}

// The epilogue of N outputs at row[e], j[e], in float32 and rounded once, for rows of a width that does not align them: all
// are read (they lie in the tensor), and those with mine[e] are written. The loads stand together, in front of what waits for
// them, and a wave's lanes take outputs side by side: 8,192 rows 2304 -> 1111 with bias, SiLU and a residual 109 -> 53 us.
template <int N>
__device__ __forceinline__ void finish_each(const Mx8Args& a, const Mx8Side& s, const int (&row)[N], const int (&j)[N],
                                            const bool (&mine)[N], float (&v)[N]) {
  if (a.bias) {
    float b[N];
#pragma unroll
    for (int e = 0; e < N; ++e) b[e] = a.bias[j[e]];
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] += b[e];
  }
  activate<N>(v, a.act);
  if (a.residual) {
    bf16_t r[N];
#pragma unroll
    for (int e = 0; e < N; ++e) r[e] = a.residual[(int64_t)row[e] * s.n + j[e]];
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] += bf2f(r[e]);
  }
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (mine[e]) s.y[(int64_t)row[e] * s.n + j[e]] = f2bf(v[e]);
}

// Four consecutive outputs j .. j + 3, j a multiple of 4, some of them perhaps past the row's end.
__device__ __forceinline__ void finish4(const Mx8Args& a, const Mx8Side& s, int m, int j, f32x4 v) {
  if ((s.n & 3) != 0) {
    const int rows[4] = {m, m, m, m}, at[4] = {j, min(j + 1, s.n - 1), min(j + 2, s.n - 1), min(j + 3, s.n - 1)};
    const bool mine[4] = {true, j + 1 < s.n, j + 2 < s.n, j + 3 < s.n};
    float f[4] = {v[0], v[1], v[2], v[3]};
    finish_each(a, s, rows, at, mine, f);
    return;
  }
  const int64_t at = (int64_t)m * s.n + j;
  if (a.bias) v += *reinterpret_cast<const f32x4*>(a.bias + j);
  activate<4>(v, a.act);
  if (a.residual) {
    const uint2 u = *reinterpret_cast<const uint2*>(a.residual + at);
    v[0] += bf2f((bf16_t)(u.x & 0xFFFFu)), v[1] += bf2f((bf16_t)(u.x >> 16));
    v[2] += bf2f((bf16_t)(u.y & 0xFFFFu)), v[3] += bf2f((bf16_t)(u.y >> 16));
  }
  *reinterpret_cast<uint2*>(s.y + at) = make_uint2(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]));
}

// The same for eight outputs from `at` on, aligned, with their bias b and residual r.
__device__ __forceinline__ void finish8(const Mx8Args& a, const Mx8Side& s, int64_t at, const float (&b)[8], const Eight<bf16_t>& r,
                                        float (&v)[8]) {
  if (a.bias) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += b[e];
  }
  activate<8>(v, a.act);
  if (a.residual) {
    float f[8];
    r.get(f);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += f[e];
  }
  // past the L2, which keeps the operands that the other tiles read (999 rows 1280 -> 32768: 59 -> 52 us, 8,192 rows 1280 ->
  // 8192: 110 -> 93)
  Eight<bf16_t> out;
  out.round(v);
  out.store_past(s.y + at);
}

// ------------------------------------------------------------------ few rows

// A workgroup owns 16 RT weight rows and 16 WM rows of x; its NW waves share the channels out, 128 at a time and each a run of
// its own. Every wave copies both operands into a ring of its own in LDS, D steps deep, and waits for nothing but its copies
// until the sums meet in LDS, in the waves' order. Copies take whole 128-byte lines, 8 rows per instruction: fragments
// loaded straight into the instruction's registers touch a row per lane and cost 64 cycles a load (64 rows 5120 -> 1792:
// 18.3 us).
template <int RT, int WM, int NW, int D>
struct Mx8Rows {
  static constexpr int ROWS = 16 * (RT + WM), COPIES = 2 * (RT + WM);        // of a step, and copies of 8 rows each
  static constexpr int SEG = 8;                                              // steps whose scales are in LDS at once
  static constexpr int RING = D * ROWS * 128, WAVE = RING + ROWS * 4 * SEG;
  static constexpr int SUMS = RT * WM * 1024;                                // a wave's sums
  static constexpr int LDS = NW * (WAVE > SUMS ? WAVE : SUMS);
  static_assert(COPIES * D <= 63, "vmcnt holds 6 bits");
};
typedef __attribute__((aligned(1))) uint32_t u32_any;

template <int RT, int WM, int NW, int D>
__global__ __launch_bounds__(64 * NW) void mx8_rows_kernel(Mx8Args a) {
  using C = Mx8Rows<RT, WM, NW, D>;
  __shared__ __align__(16) uint8_t lds[C::LDS];
  const TileAt at = tile_at(a, (int)gridDim.x);
  const Mx8Side s = side_of(a, at.w);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int j0 = s.tile * 16 * RT, m0 = at.m * 16 * WM;
  const int kb = a.k / 32, steps = a.k / 128, share = (steps + NW - 1) / NW;
  const int first = min(wave * share, steps), last = min(first + share, steps);
  const uint8_t* const wt = s.w + (int64_t)j0 * a.k;
  const uint8_t* const xt = a.x + (int64_t)m0 * a.k;
  // rows of the tile, the weight's then x's, as rows of their tensors from the tile's first on; rows past the end repeat
  // the last one and are not stored
  auto tile_row = [&](int r) { return r < 16 * RT ? min(r, s.n - 1 - j0) : min(r - 16 * RT, a.rows - 1 - m0); };
  auto scales_of = [&](int r) {
    return r < 16 * RT ? s.ws + (int64_t)((j0 + tile_row(r)) >> a.shift) * kb : a.xs + (int64_t)(m0 + tile_row(r)) * kb;
  };
  f32x4 acc[RT][WM];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < WM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](const i32x8 (&wf)[RT], const i32x8 (&xf)[WM], const uint32_t (&wsc)[RT], const uint32_t (&xsc)[WM]) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < WM; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[i], xf[j], acc[i][j], 0, 0, 0, (int)wsc[i], 0, (int)xsc[j]);
  };

  // copies: lane l of copy c brings chunk (l % 8) ^ swizzle of row 8 c + l / 8 (tile_swz<64>: fragment reads without conflicts)
  uint32_t off[C::COPIES];
#pragma unroll
  for (int c = 0; c < C::COPIES; ++c)
    off[c] = (uint32_t)tile_row(8 * c + (lane >> 3)) * (uint32_t)a.k + 16u * (uint32_t)((lane & 7) ^ (lane >> 3) ^ (c & 1));
  uint8_t* const mine = lds + wave * C::WAVE;
  const uint32_t ring = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_offset(mine));
  auto issue = [&](int stage, int t) {
    const uint32_t at = ring + (uint32_t)(stage * C::ROWS * 128);
#pragma unroll
    for (int c = 0; c < C::COPIES; ++c)
      dma16_sgpr(reinterpret_cast<uint64_t>(c < 2 * RT ? wt : xt) + (uint64_t)t * 128, off[c], at + 1024u * c);
  };
  const int swz = (l16 & 7) ^ (l16 >> 3);
  auto frag = [&](int stage, int row) {
    const uint8_t* p = mine + (stage * C::ROWS + row + l16) * 128;
    return join(*reinterpret_cast<const i32x4*>(p + ((g ^ swz) << 4)), *reinterpret_cast<const i32x4*>(p + (((4 + g) ^ swz) << 4)));
  };
  uint8_t* const sc = mine + C::RING;
  const int ufirst = __builtin_amdgcn_readfirstlane(first), ulast = __builtin_amdgcn_readfirstlane(last);
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (ufirst + d < ulast) issue(d, ufirst + d);
  int stage = 0;
  for (int seg = ufirst; seg < ulast; seg += C::SEG) {
    // the segment's scales, four of a row and step in a word, the row's words side by side
#pragma unroll
    for (int e = 0; e < C::ROWS * C::SEG / 64; ++e) {
      const int r = (64 * e + lane) / C::SEG, t = min(seg + lane % C::SEG, ulast - 1);
      reinterpret_cast<uint32_t*>(sc)[64 * e + lane] = *reinterpret_cast<const u32_any*>(scales_of(r) + 4 * t);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    const int end = min(seg + C::SEG, ulast);
    for (int t = seg; t < end; ++t) {
      wait_copies_deep<C::COPIES, D - 1>(ulast - 1 - t);
      i32x8 wf[RT], xf[WM];
      uint32_t wsc[RT], xsc[WM];
#pragma unroll
      for (int i = 0; i < RT; ++i) wf[i] = frag(stage, 16 * i), wsc[i] = sc[((16 * i + l16) * C::SEG + t - seg) * 4 + g];
#pragma unroll
      for (int j = 0; j < WM; ++j)
        xf[j] = frag(stage, 16 * (RT + j)), xsc[j] = sc[((16 * (RT + j) + l16) * C::SEG + t - seg) * 4 + g];
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // the stage is in registers
      if (t + D < ulast) issue(stage, t + D);
      multiply(wf, xf, wsc, xsc);
      stage = stage + 1 < D ? stage + 1 : 0;
    }
  }
  const int left = a.k - 128 * steps;      // the last 32, 64 or 96 channels, straight from memory
  if (left && wave == NW - 1) {
    const i32x4 zero = {0, 0, 0, 0};
    const bool lo = 16 * g < left, hi = 64 + 16 * g < left, in = 32 * g < left;
    i32x8 wf[RT], xf[WM];
    uint32_t wsc[RT], xsc[WM];
    auto part = [&](const uint8_t* tensor, int r, i32x8& f, uint32_t& fs) {
      const uint8_t* p = tensor + (int64_t)tile_row(r) * a.k + 128 * (int64_t)steps + 16 * g;
      f = join(lo ? *reinterpret_cast<const i32x4*>(p) : zero, hi ? *reinterpret_cast<const i32x4*>(p + 64) : zero);
      fs = in ? scales_of(r)[4 * steps + g] : 127u;
    };
#pragma unroll
    for (int i = 0; i < RT; ++i) part(wt, 16 * i + l16, wf[i], wsc[i]);
#pragma unroll
    for (int j = 0; j < WM; ++j) part(xt, 16 * (RT + j) + l16, xf[j], xsc[j]);
    multiply(wf, xf, wsc, xsc);
  }
#pragma unroll
  for (int i = 0; i < RT; ++i) settle(acc[i]);
  __syncthreads();                         // every wave's ring is done with
  f32x4* const sums = reinterpret_cast<f32x4*>(lds);
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < WM; ++j) sums[(wave * RT * WM + i * WM + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int q = threadIdx.x; q < RT * WM * 64; q += 64 * NW) {
    const int tile = q >> 6, l = q & 63;
    f32x4 v = sums[q];
#pragma unroll
    for (int z = 1; z < NW; ++z) v += sums[z * RT * WM * 64 + q];
    const int m = m0 + 16 * (tile % WM) + (l & 15);
    const int j = j0 + 16 * (tile / WM) + 4 * (l >> 4);
    if (m < a.rows && j < s.n) finish4(a, s, m, j, v);
  }
}

// Launches `threads` threads for each of the tiles of tr weight rows x tm rows of x, the weight tile fastest; false when a
// launch does not hold so many.
template <typename K>
static bool launch_tiles(K kernel, Mx8Args a, int tr, int tm, int threads, hipStream_t stream) {
  a.tiles0 = (a.n[0] + tr - 1) / tr;
  a.tiles = a.tiles0 + (a.n[1] + tr - 1) / tr;
  a.mtiles = (a.rows + tm - 1) / tm;
  a.panel = a.mtiles < 8 ? a.mtiles : 8;
  const int64_t groups = (int64_t)a.tiles * a.mtiles;
  if (groups * threads >= (1ll << 32)) return false;
  hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3((unsigned)threads), 0, stream, a);
  return true;
}

template <int RT, int WM, int NW, int D>
static bool launch_rows(const Mx8Args& a, hipStream_t stream) {
  return launch_tiles(mx8_rows_kernel<RT, WM, NW, D>, a, 16 * RT, 16 * WM, 64 * NW, stream);
}

// ------------------------------------------------------------------ many rows


// A tile of 32 WR GR weight rows x 32 WM GM rows of x on GR x GM waves, 128 channels a step, two steps in LDS.
template <int WR, int WM, int GR, int GM>
struct Mx8Tile {
  static constexpr int NWV = GR * GM, NT = 64 * NWV;
  static constexpr int TR = 32 * WR * GR, TM = 32 * WM * GM, ROWS = TR + TM;
  static constexpr int STAGE = ROWS * 128;              // both operands' codes of a step
  static constexpr int SCALES = ROWS * 16;              // their scales of four steps
  static constexpr int PITCH = 32 * WR * 4 + 16;        // bytes of a row of results on their way out, padded for the banks
  static constexpr int RING = 2 * (STAGE + SCALES), OUT = NWV * 32 * PITCH;
  static constexpr int LDS = RING + 256 * NWV > OUT ? RING + 256 * NWV : OUT;      // behind the ring, where prefetches end
  static constexpr int WIDE = LDS <= 80 * 1024 ? 8 : 4;  // weight tiles that an XCD multiplies at a time with a panel of 8
  static constexpr int kW = TR / 8 / NWV, kX = TM / 8 / NWV, kCopies = kW + kX;   // copies of 8 rows per wave and step
  static_assert(TR % (8 * NWV) == 0 && TM % (8 * NWV) == 0 && NWV % 2 == 0, "whole copies, in turn over the waves");
};

// A value that is the same in every lane, in scalar registers.
__device__ __forceinline__ uint64_t uniform(uint64_t v) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v) |
         (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32)) << 32;
}

// dma16_sgpr with a constant added to the LDS offset on the way into M0: one scalar register for all copies of a step.
template <int OFF>
__device__ __forceinline__ void dma16_at(uint64_t base, uint32_t voff, uint32_t lds) {
  asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(base), "s"(lds), "n"(OFF)
               : "memory", "m0", "scc");
}

// A word per lane from a lane's own address.
__device__ __forceinline__ void dma4_vaddr(uint64_t addr, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(addr), "s"(lds) : "memory", "m0");
}

// f(0), f(1) .. f(N - 1) with compile-time indexes.
template <typename F, int... I>
__device__ __forceinline__ void each(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}

// Eight bytes at any address: the scales of a pair of steps.
typedef __attribute__((ext_vector_type(2), aligned(1))) uint32_t u32x2_any;

// acc += wf xf^T over 64 channels, scale byte OP of both words.
template <int OP>
__device__ __forceinline__ f32x16 mfma_mx8(i32x8 wf, i32x8 xf, f32x16 acc, uint32_t ws, uint32_t xs) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf, xf, acc, 0, 0, OP, (int)ws, OP, (int)xs);
}

// A wave's sums to y. Lane (g, l32) holds outputs 8 q + 4 g .. + 3 of row l32, q = 0 .. 3. Through LDS (the wave's own part,
// 32 rows of x at a time; rows padded by 16 bytes for the banks) a row's outputs come to lie side by side in the wave's
// lanes: stores of whole lines, and an epilogue that is written once. n0, m0: the wave's first output and row; outputs
// before own_r and rows before own_m are another tile's.
template <typename C, int WR, int WM>
__device__ __forceinline__ void store_tile(const Mx8Args& a, const Mx8Side& s, uint8_t* lds, const f32x16 (&acc)[WR][WM], int own_r,
                                           int n0, int own_m, int m0) {
  constexpr int COLS = 32 * WR, LPR = 4 * WR, RPT = 64 / LPR;     // outputs of a wave's row, lanes per row, rows at a time
  constexpr int kTurns = (32 + RPT - 1) / RPT;
  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
  uint8_t* const mine = lds + (threadIdx.x >> 6) * 32 * C::PITCH;
  const bool aligned = (s.n & 7) == 0;
  const int n = n0 + 8 * (lane % LPR);
  float b[8];
  if (a.bias && aligned) load8(a.bias + n, b);
  __syncthreads();                         // the ring is done with; from here on each wave keeps to its own part
#pragma unroll
  for (int j = 0; j < WM; ++j) {
    // the residual's rows are on their way while the sums cross LDS (with each wave on its own here: 8,192 rows 8192 -> 5120
    // 301 -> 287 us, 999 rows 1280 -> 32768 74 -> 61)
    Eight<bf16_t> held[kTurns];
    if (a.residual && aligned) {
#pragma unroll
      for (int t = 0; t < kTurns; ++t)
        held[t].load_past(a.residual + (int64_t)(m0 + 32 * j + min(lane / LPR + RPT * t, 31)) * s.n + n);
    }
#pragma unroll
    for (int i = 0; i < WR; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(mine + l32 * C::PITCH + (32 * i + 8 * q + 4 * g) * 4) =
            f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (aligned) {
#pragma unroll
      for (int t = 0; t < kTurns; ++t) {
        const int r = lane / LPR + RPT * t, m = m0 + 32 * j + r;
        if (r < 32 && lane < LPR * RPT && m >= own_m && n >= own_r) {      // own_r is a multiple of 8 here, or n0 on
          float v[8];
          load8(reinterpret_cast<const float*>(mine + r * C::PITCH) + 8 * (lane % LPR), v);
          finish8(a, s, (int64_t)m * s.n + n, b, held[t], v);
        }
      }
    } else {                               // a value per lane, in the row's order
#pragma unroll 1
      for (int q = lane; q < 32 * COLS; q += 64 * 8) {
        int row[8], col[8];
        bool own[8];
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int r = (q + 64 * e) / COLS, c = (q + 64 * e) % COLS;
          row[e] = m0 + 32 * j + r, col[e] = n0 + c, own[e] = row[e] >= own_m && col[e] >= own_r;
          v[e] = reinterpret_cast<const float*>(mine + r * C::PITCH)[c];
        }
        finish_each(a, s, row, col, own, v);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // read, before the next rows are written
  }
}

template <int WR, int WM, int GR, int GM>
__device__ __forceinline__ void multiply_tile(const Mx8Args& a, TileAt tile, uint8_t* lds) {
  using C = Mx8Tile<WR, WM, GR, GM>;
  const Mx8Side s = side_of(a, tile.w);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
  const int wr = (wave % GR) * 32 * WR, wm = (wave / GR) * 32 * WM;
  const int kb = a.k / 32, pairs = a.k / 256;           // pairs of steps; the rest of a row is multiplied after them

  // The last tile of a side lies back from its end, whole: rows that the tile before owns are multiplied and not stored.
  const int own_r = s.tile * C::TR, r0 = min(own_r, s.n - C::TR);
  const int own_m = tile.m * C::TM, m0 = min(own_m, a.rows - C::TM);

  // copies of 8 tile rows, in turn over the waves: lane l brings chunk (l % 8) ^ swizzle of row l / 8
  const uint32_t off = (uint32_t)(lane >> 3) * (uint32_t)a.k + 16u * (uint32_t)((lane & 7) ^ (lane >> 3) ^ (wave & 1));
  const int uwave = __builtin_amdgcn_readfirstlane(wave);
  uint64_t wnext = reinterpret_cast<uint64_t>(s.w) + (uint64_t)(r0 + 8 * uwave) * (uint64_t)a.k;   // the next step's channels
  uint64_t xnext = reinterpret_cast<uint64_t>(a.x) + (uint64_t)(m0 + 8 * uwave) * (uint64_t)a.k;
  const uint32_t pitch = (uint32_t)(8 * C::NWV) * (uint32_t)a.k;
  const uint32_t lds0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)(lds_offset(lds) + (uint32_t)(8 * uwave * 128)));
  int ahead = 2 * pairs - 1;                            // steps left after the next copied one
  // copies [first, last) of a step into a stage (both stages of the weight's, then both of x's). Past the last step they
  // bring it once more, which nobody reads: no branch stands between the products.
  auto issue = [&](auto stage, int first, int last) {
    constexpr int S = decltype(stage)::value;
    each([&](auto copy) {
      constexpr int c = decltype(copy)::value;
      constexpr int at = c < C::kW ? S * C::TR + 8 * C::NWV * c : 2 * C::TR + S * C::TM + 8 * C::NWV * (c - C::kW);
      if (c >= first && c < last)
        dma16_at<at * 128>((c < C::kW ? wnext : xnext) + (uint64_t)(c < C::kW ? c : c - C::kW) * pitch, off, lds0);
    }, std::make_integer_sequence<int, C::kCopies>{});
    if (last == C::kCopies) {
      const uint64_t by = ahead > 0 ? 128 : 0;
      wnext += by, xnext += by, --ahead;
    }
  };
  // The step after those that are copied goes from memory into the XCD's L2, one line per lane and nothing kept of it: each
  // tile brings its share of the rows that the tiles beside it multiply too (TM / WIDE of x's, TR / panel of the weight's).
  // Copies then find it there; without, each step waited for the slowest miss (8192 rows 8192 -> 5120: 313 -> 301 us, 2048
  // rows 97 -> 90).
  const int xshare = C::TM / C::WIDE, wshare = C::TR / a.panel, each_wave = (xshare + wshare + C::NWV - 1) / C::NWV;
  const int mine = min(wave * each_wave + lane, xshare + wshare - 1);
  uint64_t ahead_of = mine < xshare ? reinterpret_cast<uint64_t>(a.x) + (uint64_t)(m0 + tile.w % C::WIDE * xshare + mine) * (uint64_t)a.k
                                    : reinterpret_cast<uint64_t>(s.w) + (uint64_t)(r0 + tile.m % a.panel * wshare + mine - xshare) * (uint64_t)a.k;
  ahead_of += 128 * (uint64_t)min(3, max(2 * pairs - 1, 0));
  int unseen = 2 * pairs - 4;                           // steps left after the next prefetched one
  const uint32_t nowhere = (uint32_t)__builtin_amdgcn_readfirstlane((int)(lds_offset(lds) + (uint32_t)(C::RING + 256 * uwave)));
  auto prefetch = [&]() {
    if (lane < each_wave) dma4_vaddr(ahead_of, nowhere);
    ahead_of += unseen > 0 ? 128 : 0, --unseen;
  };
  // scales: thread t brings rows t, t + NT .. of the tile, four steps at a time
  constexpr int kS = (C::ROWS + C::NT - 1) / C::NT;
  const uint8_t* srow[kS];
#pragma unroll
  for (int i = 0; i < kS; ++i) {
    const int r = (int)threadIdx.x + C::NT * i;
    srow[i] = r < C::TR ? s.ws + (int64_t)((r0 + r) >> a.shift) * kb : a.xs + (int64_t)(m0 + min(r, C::ROWS - 1) - C::TR) * kb;
  }
  uint8_t* const sc = lds + 2 * C::STAGE;
  u32x2_any held[kS][2];
  // the scales of four steps from step 4 f on; past the last pair they repeat its
  auto load_scales = [&](int f) {
#pragma unroll
    for (int i = 0; i < kS; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) held[i][e] = *reinterpret_cast<const u32x2_any*>(srow[i] + 8 * min(2 * f + e, pairs - 1));
  };
  // into LDS as lanes take them: of lane group g and a pair, blocks g, 2 + g, 4 + g, 6 + g (its four half steps) in a word
  auto store_scales = [&](int f) {
#pragma unroll
    for (int i = 0; i < kS; ++i) {
      const int r = (int)threadIdx.x + C::NT * i;
      if (C::ROWS % C::NT == 0 || r < C::ROWS)
        *reinterpret_cast<uint4*>(sc + (f & 1) * C::SCALES + 16 * r) =
            make_uint4(__builtin_amdgcn_perm(held[i][0][1], held[i][0][0], 0x06040200u),
                       __builtin_amdgcn_perm(held[i][1][1], held[i][1][0], 0x06040200u),
                       __builtin_amdgcn_perm(held[i][0][1], held[i][0][0], 0x07050301u),
                       __builtin_amdgcn_perm(held[i][1][1], held[i][1][0], 0x07050301u));
    }
  };

  // LDS addresses of this lane's row in both operands, for each half step and each half of a fragment's 32 bytes, and of its
  // scale words; everything else is a constant offset. (The empty asm keeps the compiler from making one register per read.)
  const int swz = (l32 & 7) ^ ((l32 >> 3) & 1);
  uint32_t wadr[2][2], xadr[2][2];
  uint32_t wsadr = lds_offset(sc) + (uint32_t)(16 * (wr + l32) + 8 * g), xsadr = lds_offset(sc) + (uint32_t)(16 * (C::TR + wm + l32) + 8 * g);
  asm volatile("" : "+v"(wsadr), "+v"(xsadr));
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      wadr[h][e] = lds_offset(lds) + (uint32_t)((wr + l32) * 128 + (((4 * h + 2 * e + g) ^ swz) << 4));
      xadr[h][e] = lds_offset(lds) + (uint32_t)((2 * C::TR + wm + l32) * 128 + (((4 * h + 2 * e + g) ^ swz) << 4));
      asm volatile("" : "+v"(wadr[h][e]), "+v"(xadr[h][e]));
    }
  constexpr int kFrags = WR + WM;
  auto frag = [&](const uint32_t (&adr)[2], int at) {
    typedef const __attribute__((address_space(3))) i32x4* lds_i32x4;
    return join(*(lds_i32x4)(uintptr_t)(adr[0] + (uint32_t)at), *(lds_i32x4)(uintptr_t)(adr[1] + (uint32_t)at));
  };
  // fragments [first, last) of a half step: x's, then the weight's in the order of their use
  auto read = [&](int stage, int half, int first, int last, i32x8 (&wf)[WR], i32x8 (&xf)[WM]) {
#pragma unroll
    for (int f = 0; f < kFrags; ++f) {
      if (f < first || f >= last) continue;
      if (f < WM) xf[f] = frag(xadr[half], (stage * C::TM + 32 * f) * 128);
      else wf[f - WM] = frag(wadr[half], (stage * C::TR + 32 * (f - WM)) * 128);
    }
  };
  // the scale words of a pair of steps (bytes: half steps)
  auto read_scales = [&](int q, uint32_t (&wsc)[WR], uint32_t (&xsc)[WM]) {
    typedef const __attribute__((address_space(3))) uint32_t* lds_u32;
    const uint32_t at = (uint32_t)(((q >> 1) & 1) * C::SCALES + 4 * (q & 1));
#pragma unroll
    for (int j = 0; j < WM; ++j) xsc[j] = *(lds_u32)(uintptr_t)(xsadr + at + (uint32_t)(16 * 32 * j));
#pragma unroll
    for (int i = 0; i < WR; ++i) wsc[i] = *(lds_u32)(uintptr_t)(wsadr + at + (uint32_t)(16 * 32 * i));
  };

  f32x16 acc[WR][WM];
#pragma unroll
  for (int i = 0; i < WR; ++i)
#pragma unroll
    for (int j = 0; j < WM; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

  i32x8 w0[WR], x0[WM], w1[WR], x1[WM];
  uint32_t wsc[WR], xsc[WM], wsn[WR], xsn[WM];
  // One step at stage P and scale bytes 2 P, 2 P + 1: the second half's fragments are read while the first is multiplied;
  // at the barrier every wave has read the stage and the next step has landed; then the step after next is copied into
  // the stage and the next step's first half read while the second half is multiplied.
  auto step = [&](int q, auto parity) {
    constexpr int P = decltype(parity)::value;
#pragma unroll
    for (int i = 0; i < WR; ++i) {
      read(P, 1, i * kFrags / WR, (i + 1) * kFrags / WR, w1, x1);
#pragma unroll
      for (int j = 0; j < WM; ++j) {
        acc[i][j] = mfma_mx8<2 * P>(w0[i], x0[j], acc[i][j], wsc[i], xsc[j]);
        asm volatile("" : "+v"(acc[i][j]));        // in this order: the compiler gathers products of one sum otherwise
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    asm volatile("s_waitcnt vmcnt(1) lgkmcnt(0)" ::: "memory");      // the prefetch may be on its way
    if (P == 1 && (q & 1) == 0) store_scales((q >> 1) + 1);      // that buffer was last read in an earlier step
    __syncthreads();
    if (P == 1 && (q & 1) == 0) load_scales((q >> 1) + 2);
#pragma unroll
    for (int i = 0; i < WR; ++i) {
      issue(parity, i * C::kCopies / WR, (i + 1) * C::kCopies / WR);
      if (i == WR - 1) prefetch();
      read(P ^ 1, 0, i * kFrags / WR, (i + 1) * kFrags / WR, w0, x0);
      if (P == 1 && i == 0) read_scales(q + 1, wsn, xsn);
#pragma unroll
      for (int j = 0; j < WM; ++j) {
        acc[i][j] = mfma_mx8<2 * P + 1>(w1[i], x1[j], acc[i][j], wsc[i], xsc[j]);
        asm volatile("" : "+v"(acc[i][j]));
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (P == 1) {
#pragma unroll
      for (int i = 0; i < WR; ++i) wsc[i] = wsn[i];
#pragma unroll
      for (int j = 0; j < WM; ++j) xsc[j] = xsn[j];
    }
  };
  if (pairs > 0) {
    load_scales(0);
    issue(std::integral_constant<int, 0>{}, 0, C::kCopies);
    issue(std::integral_constant<int, 1>{}, 0, C::kCopies);
    store_scales(0);
    load_scales(1);
    wait_vmcnt<0>();
    prefetch();
    __syncthreads();
    read(0, 0, 0, kFrags, w0, x0);
    read_scales(0, wsc, xsc);
    for (int q = 0; q < pairs; ++q) {
      step(q, std::integral_constant<int, 0>{});
      step(q, std::integral_constant<int, 1>{});
    }
    wait_vmcnt<0>();                       // no copy may land in LDS any more
  }

  // the last channels (fewer than 256), straight from memory
  for (int at = pairs * 256; at < a.k; at += 64) {
    const i32x4 zero = {0, 0, 0, 0};
    const bool lo = at + 16 * g < a.k, hi = at + 32 + 16 * g < a.k, in = at + 32 * g < a.k;
    i32x8 wf[WR];
#pragma unroll
    for (int i = 0; i < WR; ++i) {
      const int64_t row = r0 + wr + 32 * i + l32;
      const uint8_t* p = s.w + row * a.k + at + 16 * g;
      wf[i] = join(lo ? *reinterpret_cast<const i32x4*>(p) : zero, hi ? *reinterpret_cast<const i32x4*>(p + 32) : zero);
      wsc[i] = in ? s.ws[(row >> a.shift) * kb + at / 32 + g] : 127u;
    }
#pragma unroll
    for (int j = 0; j < WM; ++j) {
      const int64_t row = m0 + wm + 32 * j + l32;
      const uint8_t* p = a.x + row * a.k + at + 16 * g;
      const i32x8 xf = join(lo ? *reinterpret_cast<const i32x4*>(p) : zero,
                            hi ? *reinterpret_cast<const i32x4*>(p + 32) : zero);
      const uint32_t xc = in ? a.xs[row * kb + at / 32 + g] : 127u;
#pragma unroll
      for (int i = 0; i < WR; ++i) acc[i][j] = mfma_mx8<0>(wf[i], xf, acc[i][j], wsc[i], xc);
    }
  }
#pragma unroll
  for (int i = 0; i < WR; ++i) settle(acc[i]);

  store_tile<C, WR, WM>(a, s, lds, acc, own_r, r0 + wr, own_m, m0 + wm);
}

template <int WR, int WM, int GR, int GM>
__global__ __launch_bounds__(64 * GR * GM, (Mx8Tile<WR, WM, GR, GM>::LDS <= 80 * 1024) ? 2 : 1) void mx8_tiles_kernel(
    Mx8Args a) {
  __shared__ __align__(16) uint8_t lds[Mx8Tile<WR, WM, GR, GM>::LDS];
  multiply_tile<WR, WM, GR, GM>(a, tile_at(a, (int)gridDim.x), lds);
}

// ------------------------------------------------------------------ tiles on few workgroups

// Rows of whole steps: where the scale word of step kt lies behind a row's first byte in the two buffers of `rows` rows x 16 bytes,
// four steps each, the last four steps side by side where fewer are left. Steps past the last have its word again.
constexpr __host__ __device__ __forceinline__ int ring_scales_at(int kt, int steps, int rows) {
  const int now = kt < steps ? kt : steps - 1, group = now & ~3;
  return ((now >> 2) & 1) * rows * 16 + 4 * (now - (group < steps - 4 ? group : steps - 4));
}
constexpr bool ring_scales_inside(int rows) {
  for (int steps = 4; steps < 24; ++steps)             // every remainder of eight, with the second buffer and without
    for (int kt = 0; kt <= steps; ++kt) {
      const int at = ring_scales_at(kt, steps, rows) % (rows * 16);
      if (at < 0 || at + 4 > 16) return false;          // in its own row's 16 bytes
    }
  return true;
}

// The same tile over a ring of NS steps: a workgroup that has its CU to itself waits for the memory's answer every step
// (about 1 us whatever the tile) unless several steps are on their way. For rows of four steps and more: scales come by copies
// too, four steps of a row at a time; three where they lie off words or the last step is a part of one (ANY).
template <int WR, int WM, int GR, int GM, int NS, bool ANY = false>
struct Mx8Ring {
  static constexpr int NWV = GR * GM, NT = 64 * NWV;
  static constexpr int TR = 32 * WR * GR, TM = 32 * WM * GM, ROWS = TR + TM;
  static constexpr int kW = TR / 8 / NWV, kX = TM / 8 / NWV, kCopies = kW + kX;   // copies of 8 rows per wave and step
  static constexpr int CODES = NS * ROWS * 128;
  static constexpr int PITCH = 32 * WR * 4 + 16;        // bytes of a row of results on their way out, padded for the banks
  static constexpr int RING = CODES + 2 * ROWS * 16 + (ANY ? 16 : 0), OUT = NWV * 32 * PITCH;      // ANY: a word more is read
  static constexpr int LDS = RING > OUT ? RING : OUT;
  static_assert(TR % (8 * NWV) == 0 && TM % (8 * NWV) == 0 && NWV % 2 == 0, "whole copies, in turn over the waves");
  static_assert(TR % 64 == 0 && TM % 64 == 0 && ROWS <= 64 * NWV, "one copy of 64 rows' scales per wave");
  static_assert(ring_scales_inside(ROWS), "the reads ahead stay in the buffers");
  static_assert(kCopies * (NS - 1) <= 63 && NS >= 3 && NS <= 4, "vmcnt holds 6 bits; scales land in time");
};

template <int WR, int WM, int GR, int GM, int NS, bool ANY = false>
__device__ __forceinline__ void multiply_ring_tile(const Mx8Args& a, TileAt tile, uint8_t* lds, int split = 1) {
  using C = Mx8Ring<WR, WM, GR, GM, NS, ANY>;
  const Mx8Side s = side_of(a, tile.w, split);
  if (split > 1 && (s.tile * C::TR >= s.n || tile.m * C::TM >= a.rows)) return;       // a part behind the end
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
  const int wr = (wave % GR) * 32 * WR, wm = (wave / GR) * 32 * WM;
  // ANY: the last step lies back from the row's end, whole, and its first `again` blocks, which the step before has, are
  // multiplied as zeros
  const int kb = a.k / 32, steps = ANY ? (a.k + 127) / 128 : a.k / 128, again = 4 * steps - kb;
  // The last tile of a side lies back from its end, whole: rows that the tile before owns are multiplied and not stored.
  const int own_r = s.tile * C::TR, r0 = min(own_r, s.n - C::TR);
  const int own_m = tile.m * C::TM, m0 = min(own_m, a.rows - C::TM);

  // copies of 8 tile rows, in turn over the waves: lane l brings chunk (l % 8) ^ swizzle of row l / 8
  const uint32_t off = (uint32_t)(lane >> 3) * (uint32_t)a.k + 16u * (uint32_t)((lane & 7) ^ (lane >> 3) ^ (wave & 1));
  const int uwave = __builtin_amdgcn_readfirstlane(wave);
  uint64_t wnext = reinterpret_cast<uint64_t>(s.w) + (uint64_t)(r0 + 8 * uwave) * (uint64_t)a.k;   // the next step's channels
  uint64_t xnext = reinterpret_cast<uint64_t>(a.x) + (uint64_t)(m0 + 8 * uwave) * (uint64_t)a.k;
  const uint32_t pitch = (uint32_t)(8 * C::NWV) * (uint32_t)a.k;
  const uint32_t lds0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_offset(lds));
  const uint32_t mine0 = lds0 + (uint32_t)(8 * uwave * 128);
  int ahead = steps - 1;                                // steps left after the next copied one
  int into = 0;                                         // the stage that it goes to
  // copies [first, last) of a step (all stages of the weight's, then of x's). Past the last step they bring it once more,
  // which nobody reads: no branch stands between the products, and waits count the same everywhere.
  auto issue = [&](int first, int last) {
    const uint32_t wdst = mine0 + (uint32_t)(into * C::TR * 128), xdst = mine0 + (uint32_t)(into * C::TM * 128);
    each([&](auto copy) {
      constexpr int c = decltype(copy)::value;
      if (c < first || c >= last) return;
      if constexpr (c < C::kW) dma16_at<8 * C::NWV * c * 128>(wnext + (uint64_t)c * pitch, off, wdst);
      else dma16_at<(NS * C::TR + 8 * C::NWV * (c - C::kW)) * 128>(xnext + (uint64_t)(c - C::kW) * pitch, off, xdst);
    }, std::make_integer_sequence<int, C::kCopies>{});
    if (last == C::kCopies) {
      const uint64_t by = ahead > 0 ? (ANY && ahead == 1 ? 128 - 32 * again : 128) : 0;
      wnext += by, xnext += by, --ahead;
      into = into + 1 < NS ? into + 1 : 0;
    }
  };
  // scales: 64 rows per wave (one without any of its own repeats the last), the words of kGroup steps of a row side by side; the
  // last kGroup steps where fewer are left. ANY: 16 bytes from the word on that a row's first scale byte lies in hold three
  // steps' whatever its place; the last 16 end with the word that the row's last byte lies in. So no copy touches a word
  // without a byte of its row.
  constexpr int kGroup = ANY ? 3 : 4;
  const int srow = 64 * min(uwave, C::ROWS / 64 - 1), lastg = (steps - 1) / kGroup;
  const bool of_w = srow < C::TR;
  const int from = of_w ? r0 + srow : m0 + srow - C::TR, shift = of_w ? a.shift : 0;
  const uint64_t sfrom = uniform(reinterpret_cast<uint64_t>(of_w ? s.ws : a.xs) + (uint64_t)(from >> shift) * (uint64_t)kb);
  const uint64_t sbase = ANY ? sfrom & ~3ull : sfrom;
  const uint32_t sat = (uint32_t)(((from + lane) >> shift) - (from >> shift)) * (uint32_t)kb + (uint32_t)(sfrom - sbase);
  const uint32_t soff = ANY ? sat & ~3u : sat, slast = ((sat + (uint32_t)kb + 3u) & ~3u) - 16u;
  auto copy_scales = [&](int f) {
    const uint32_t to = lds0 + (uint32_t)(C::CODES + (f & 1) * C::ROWS * 16 + srow * 16);
    if constexpr (ANY) dma16_sgpr(sbase + (uint64_t)(f < lastg ? 12 * f : 0), f < lastg ? soff : slast, to);
    else dma16_sgpr(sbase + (uint64_t)(4 * min(4 * f, steps - 4)), soff, to);
  };

  // LDS addresses of this lane's row in both operands, for each half step and each half of a fragment's 32 bytes, in the
  // stage that is read next, and of its scale words; everything else is a constant offset. (The empty asm keeps the compiler
  // from making one register per read.)
  const int swz = (l32 & 7) ^ ((l32 >> 3) & 1);
  uint32_t wadr[2][2], xadr[2][2];
  uint32_t wsadr = lds0 + (uint32_t)(C::CODES + 16 * (wr + l32)), xsadr = lds0 + (uint32_t)(C::CODES + 16 * (C::TR + wm + l32));
  asm volatile("" : "+v"(wsadr), "+v"(xsadr));
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      wadr[h][e] = lds0 + (uint32_t)((wr + l32) * 128 + (((4 * h + 2 * e + g) ^ swz) << 4));
      xadr[h][e] = lds0 + (uint32_t)((NS * C::TR + wm + l32) * 128 + (((4 * h + 2 * e + g) ^ swz) << 4));
    }
  int at = 0;                                           // the stage that the addresses point into
  auto advance = [&]() {
    const int by = at + 1 < NS ? 1 : 1 - NS;
    at += by;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        wadr[h][e] += (uint32_t)(by * C::TR * 128);
        xadr[h][e] += (uint32_t)(by * C::TM * 128);
        asm volatile("" : "+v"(wadr[h][e]), "+v"(xadr[h][e]));
      }
  };
  constexpr int kFrags = WR + WM;
  typedef const __attribute__((address_space(3))) i32x4* lds_i32x4;
  typedef const __attribute__((address_space(3))) uint32_t* lds_u32;
  auto frag = [&](const uint32_t (&adr)[2], int by) {
    return join(*(lds_i32x4)(uintptr_t)(adr[0] + (uint32_t)by), *(lds_i32x4)(uintptr_t)(adr[1] + (uint32_t)by));
  };
  // fragments [first, last) of half a step: x's, then the weight's in the order of their use
  auto read = [&](int h, int first, int last, i32x8 (&wf)[WR], i32x8 (&xf)[WM]) {
#pragma unroll
    for (int f = 0; f < kFrags; ++f) {
      if (f < first || f >= last) continue;
      if (f < WM) xf[f] = frag(xadr[h], 32 * f * 128);
      else wf[f - WM] = frag(wadr[h], 32 * (f - WM) * 128);
    }
  };
  // step kt's scale words (blocks 0 .. 3). ANY: from two words, at the place of this lane's row
  int wlow[WR], xlow[WM];                               // where a row's first scale byte lies in its word
  if constexpr (ANY) {
#pragma unroll
    for (int i = 0; i < WR; ++i)
      wlow[i] = (int)((reinterpret_cast<uintptr_t>(s.ws) + (uintptr_t)((r0 + wr + 32 * i + l32) >> a.shift) * (uintptr_t)kb) & 3u);
#pragma unroll
    for (int j = 0; j < WM; ++j)
      xlow[j] = (int)((reinterpret_cast<uintptr_t>(a.xs) + (uintptr_t)(m0 + wm + 32 * j + l32) * (uintptr_t)kb) & 3u);
  }
  auto read_scales = [&](int kt, uint32_t (&wsc)[WR], uint32_t (&xsc)[WM]) {
    if constexpr (ANY) {
      const int now = min(kt, steps - 1), f = now / 3, byte = now == steps - 1 ? kb - 4 : 4 * now;      // in the row
      auto word = [&](uint32_t adr, int low) {
        const uint32_t at = (uint32_t)(byte + low - (f < lastg ? 12 * f : ((low + kb + 3) & ~3) - 16));
        const uint32_t p = adr + (uint32_t)((f & 1) * C::ROWS * 16) + (at & ~3u);
        return __builtin_amdgcn_alignbyte(*(lds_u32)(uintptr_t)(p + 4u), *(lds_u32)(uintptr_t)p, at);
      };
#pragma unroll
      for (int j = 0; j < WM; ++j) xsc[j] = word(xsadr + (uint32_t)(16 * 32 * j), xlow[j]);
#pragma unroll
      for (int i = 0; i < WR; ++i) wsc[i] = word(wsadr + (uint32_t)(16 * 32 * i), wlow[i]);
    } else {
      const uint32_t by = (uint32_t)ring_scales_at(kt, steps, C::ROWS);
#pragma unroll
      for (int j = 0; j < WM; ++j) xsc[j] = *(lds_u32)(uintptr_t)(xsadr + by + (uint32_t)(16 * 32 * j));
#pragma unroll
      for (int i = 0; i < WR; ++i) wsc[i] = *(lds_u32)(uintptr_t)(wsadr + by + (uint32_t)(16 * 32 * i));
    }
  };
  // the weight's codes of the blocks that the last step has again as zeros: a fragment's halves are blocks 0 and 1, 2 and 3
  auto once = [&](int kt, int half, int i, i32x8 (&wf)[WR]) {
    if constexpr (ANY) {
      const int n = kt == steps - 1 ? again - 2 * half : 0, lo = n > 0 ? 0 : -1, hi = n > 1 ? 0 : -1;
#pragma unroll
      for (int e = 0; e < 4; ++e) wf[i][e] &= lo, wf[i][4 + e] &= hi;
    }
  };

  f32x16 acc[WR][WM];
#pragma unroll
  for (int i = 0; i < WR; ++i)
#pragma unroll
    for (int j = 0; j < WM; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
  i32x8 w0[WR], x0[WM], w1[WR], x1[WM];
  uint32_t wsc[WR], xsc[WM], wsn[WR], xsn[WM];
  copy_scales(0);
#pragma unroll
  for (int d = 0; d < NS; ++d) issue(0, C::kCopies);
  wait_vmcnt<(NS - 1) * C::kCopies>();
  __syncthreads();
  read(0, 0, kFrags, w0, x0);
  read_scales(0, wsn, xsn);
  for (int kt = 0; kt < steps; ++kt) {
    // bytes 0 and 2: this lane group's blocks of the first and the second half
#pragma unroll
    for (int i = 0; i < WR; ++i) wsc[i] = wsn[i] >> (8 * g);
#pragma unroll
    for (int j = 0; j < WM; ++j) xsc[j] = xsn[j] >> (8 * g);
    // the second half's fragments are read while the first is multiplied
#pragma unroll
    for (int i = 0; i < WR; ++i) {
      read(1, i * kFrags / WR, (i + 1) * kFrags / WR, w1, x1);
      once(kt, 0, i, w0);
#pragma unroll
      for (int j = 0; j < WM; ++j) {
        acc[i][j] = mfma_mx8<0>(w0[i], x0[j], acc[i][j], wsc[i], xsc[j]);
        asm volatile("" : "+v"(acc[i][j]));        // in this order: the compiler gathers products of one sum otherwise
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    advance();
    // this wave has read the stage and its copies of the next step have landed; then every wave's
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NS - 2) * C::kCopies) : "memory");
    __syncthreads();
    // the scales of the steps after the next kGroup: that buffer was last read two steps ago, and they land two steps before
    // they are read, at the latest with the wait then
    if (kt % kGroup == 0) copy_scales(kt / kGroup + 1);
    // the stage takes step kt + NS, and the next step's first half is read, while the second half is multiplied
#pragma unroll
    for (int i = 0; i < WR; ++i) {
      issue(i * C::kCopies / WR, (i + 1) * C::kCopies / WR);
      read(0, i * kFrags / WR, (i + 1) * kFrags / WR, w0, x0);
      if (i == 0) read_scales(kt + 1, wsn, xsn);
      once(kt, 1, i, w1);
#pragma unroll
      for (int j = 0; j < WM; ++j) {
        acc[i][j] = mfma_mx8<2>(w1[i], x1[j], acc[i][j], wsc[i], xsc[j]);
        asm volatile("" : "+v"(acc[i][j]));
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  wait_vmcnt<0>();                         // no copy may land in LDS any more
#pragma unroll
  for (int i = 0; i < WR; ++i) settle(acc[i]);
  store_tile<C, WR, WM>(a, s, lds, acc, own_r, r0 + wr, own_m, m0 + wm);
}

template <int WR, int WM, int GR, int GM, int NS, bool ANY>
__global__ __launch_bounds__(64 * GR * GM, 1) void mx8_ring_kernel(Mx8Args a) {
  __shared__ __align__(16) uint8_t lds[Mx8Ring<WR, WM, GR, GM, NS, ANY>::LDS];
  multiply_ring_tile<WR, WM, GR, GM, NS, ANY>(a, tile_at(a, (int)gridDim.x), lds);
}

// Tiles of 256 x 256 in whole rounds of the 256 CUs, and what is left in parts over a ring: half a round or less as two tiles of
// 256 x 128 each, a quarter or less as four of 128 x 128, so that the last round takes half or a third of a whole one's time.
// 8,192 rows 8192 -> 5120 (2 1/2 rounds): 297 -> 283 us; 4,096 rows (1 1/4) 189 -> 157 in halves, 154 in quarters, by tiles
// of 192 x 256 170.
template <int PARTS>
__global__ __launch_bounds__(512, 1) void mx8_parts_kernel(Mx8Args a) {
  using Whole = Mx8Tile<4, 2, 2, 4>;
  using Half = Mx8Ring<2, 2, 4, 2, 3>;
  using Quarter = Mx8Ring<2, 1, 2, 4, 4>;
  static_assert(Whole::NT == Half::NT && Whole::TR == Half::TR && Whole::TM == 2 * Half::TM, "two halves make a tile");
  static_assert(Whole::NT == Quarter::NT && Whole::TR == 2 * Quarter::TR && Whole::TM == 2 * Quarter::TM, "four quarters do");
  constexpr int RING = PARTS == 2 ? Half::LDS : Quarter::LDS;
  __shared__ __align__(16) uint8_t lds[Whole::LDS > RING ? Whole::LDS : RING];
  if ((int)blockIdx.x < a.whole) {
    multiply_tile<4, 2, 2, 4>(a, tile_at(a, a.whole), lds);
    return;
  }
  const int b = (int)blockIdx.x - a.whole, part = b / 8 % PARTS, unit = a.whole + b / (8 * PARTS) * 8 + b % 8;   // parts on one XCD
  if (unit >= a.tiles * a.mtiles) return;
  TileAt tile = tile_of(a, unit);
  tile.m = 2 * tile.m + part % 2;
  if constexpr (PARTS == 2) {
    if (tile.m * Half::TM < a.rows) multiply_ring_tile<2, 2, 4, 2, 3>(a, tile, lds);
  } else {
    tile.w = 2 * tile.w + part / 2;
    multiply_ring_tile<2, 1, 2, 4, 4>(a, tile, lds, 2);
  }
}

// Whole tiles of this shape are in the call.
template <int WR, int WM, int GR, int GM>
static bool holds(const Mx8Args& a) {
  using C = Mx8Tile<WR, WM, GR, GM>;
  return a.rows >= C::TM && a.n[0] >= C::TR && (a.n[1] == 0 || a.n[1] >= C::TR);
}

// The same, and rows that the ring's kernel takes. Rows of whole steps whose scales lie on words have a kernel of their own: the
// other one's shifts and masks cost 777 rows 2304 -> 1111 8.6 -> 10.9 us, 300 rows 2048 -> 8192 15.0 -> 16.7. Where rows are no
// whole lines, copies straddle two besides: 300 rows 2272 -> 8192 take 21.4 us (29.4 in tiles of two steps), 777 rows 2336 -> 1111
// 11.2 (13.5 as few rows).
template <int WR, int WM, int GR, int GM>
static bool holds_ring(const Mx8Args& a) {
  return holds<WR, WM, GR, GM>(a) && a.k >= 512;
}
static bool on_steps(const Mx8Args& a) {
  auto on_words = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; };
  return a.k % 128 == 0 && on_words(a.xs) && on_words(a.ws[0]) && on_words(a.ws[1]);
}
template <int WR, int WM, int GR, int GM, int NS>
static bool launch_ring(const Mx8Args& a, hipStream_t stream) {
  using C = Mx8Ring<WR, WM, GR, GM, NS>;
  if (on_steps(a)) return launch_tiles(mx8_ring_kernel<WR, WM, GR, GM, NS, false>, a, C::TR, C::TM, C::NT, stream);
  return launch_tiles(mx8_ring_kernel<WR, WM, GR, GM, NS, true>, a, C::TR, C::TM, C::NT, stream);
}

template <int WR, int WM, int GR, int GM>
static bool launch_many(const Mx8Args& a, hipStream_t stream) {
  using C = Mx8Tile<WR, WM, GR, GM>;
  return launch_tiles(mx8_tiles_kernel<WR, WM, GR, GM>, a, C::TR, C::TM, C::NT, stream);
}

static int64_t tiles_of(const Mx8Args& a, int tr, int tm) {
  return (int64_t)((a.n[0] + tr - 1) / tr + (a.n[1] + tr - 1) / tr) * ((a.rows + tm - 1) / tm);
}

// Whole rounds of 256 x 256 tiles, and a part of a round that takes PARTS workgroups a tile.
template <int PARTS>
static bool holds_parts(const Mx8Args& a) {
  const int64_t tiles = tiles_of(a, 256, 256);
  return holds_ring<4, 2, 2, 4>(a) && on_steps(a) && tiles > 256 && tiles % 256 > 0 && tiles % 256 * PARTS <= 256;
}
template <int PARTS>
static bool launch_parts(const Mx8Args& args, hipStream_t stream) {
  Mx8Args a = args;
  a.tiles0 = (a.n[0] + 255) / 256;
  a.tiles = a.tiles0 + (a.n[1] + 255) / 256;
  a.mtiles = (a.rows + 255) / 256;
  a.panel = a.mtiles < 8 ? a.mtiles : 8;
  const int64_t tiles = (int64_t)a.tiles * a.mtiles, rest = tiles % 256;
  if (tiles * 512 >= (1ll << 32) - (1 << 20)) return false;
  a.whole = (int)(tiles - rest);
  hipLaunchKernelGGL(mx8_parts_kernel<PARTS>, dim3((unsigned)(a.whole + (rest + 7) / 8 * 8 * PARTS)), dim3(512), 0, stream, a);
  return true;
}

// ------------------------------------------------------------------ which tile

static bool any(const Mx8Args&) { return true; }

// A tile shape, the ranges of k that one workgroup's waves share out (parts of the last tiles for kind 3), workgroups that a CU
// holds, and what a call's time was measured to consist of, in us: 1 + per round of all CUs + per round and step + per tile of a CU
// + per tile and step + per GB that tiles read + per 10 MB of results. Fitted to 290 to 420 sizes for each (1 to 8,192 rows, k 256
// to 8,192, n 512 to 32,768, no bias or residual): 9 of 10 estimates of those are within 10 to 15 % of the time (rows of odd
// widths, stored by the value, take up to a third longer than estimated, whatever the shape).
struct Mx8Shape {
  int kind, tr, tm, ranges, held;      // kind 0: few rows, 1: tiles, 2: tiles over a ring, 3: tiles, the last in parts
  float us[7];
  bool (*launch)(const Mx8Args&, hipStream_t);
  bool (*takes)(const Mx8Args&);
};
// what the last tiles' parts are, and tiles of their own
static const Mx8Shape kQuarter = {2, 128, 128, 1, 1, {2.33f, 2.59f, 0.426f, 0.f, 0.f, 10.9f, 0.786f}, launch_ring<2, 1, 2, 4, 4>, holds_ring<2, 1, 2, 4>};
static const Mx8Shape kHalf = {2, 256, 128, 1, 1, {1.43f, 0.f, 0.646f, 5.26f, 0.f, 12.9f, 0.237f}, launch_ring<2, 2, 4, 2, 3>, holds_ring<2, 2, 4, 2>};
static const Mx8Shape kShapes[] = {
    {0, 16, 16, 8, 2, {2.52f, 0.f, 0.203f, 0.644f, 0.0547f, 19.9f, 0.f}, launch_rows<1, 1, 8, 2>, any},
    {0, 32, 16, 8, 1, {1.78f, 1.45f, 0.f, 0.f, 0.405f, 17.2f, 0.f}, launch_rows<2, 1, 8, 2>, any},
    {0, 32, 16, 2, 5, {2.64f, 0.f, 0.229f, 0.244f, 0.0015f, 24.2f, 0.f}, launch_rows<2, 1, 2, 2>, any},
    {0, 32, 32, 4, 1, {1.81f, 1.43f, 0.f, 0.f, 0.35f, 9.63f, 6.44f}, launch_rows<2, 2, 4, 3>, any},
    {0, 32, 48, 8, 1, {2.f, 1.32f, 0.f, 0.f, 0.759f, 12.2f, 5.09f}, launch_rows<2, 3, 8, 1>, any},
    {0, 64, 32, 8, 1, {2.06f, 1.38f, 0.981f, 0.f, 0.f, 11.f, 4.42f}, launch_rows<4, 2, 8, 1>, any},
    {0, 64, 64, 8, 1, {2.19f, 2.1f, 0.f, 0.f, 1.4f, 8.71f, 2.88f}, launch_rows<4, 4, 8, 1>, any},
    {0, 64, 96, 4, 1, {2.96f, 2.97f, 0.f, 0.f, 0.957f, 3.52f, 4.05f}, launch_rows<4, 6, 4, 1>, any},
    {1, 64, 64, 1, 4, {2.61f, 0.f, 0.344f, 0.774f, 0.0668f, 14.3f, 0.f}, launch_many<1, 1, 2, 2>, holds<1, 1, 2, 2>},
    {1, 128, 128, 1, 2, {2.79f, 0.979f, 0.429f, 1.35f, 0.236f, 1.67f, 0.906f}, launch_many<2, 2, 2, 2>, holds<2, 2, 2, 2>},
    {1, 192, 256, 1, 1, {0.895f, 0.f, 1.06f, 7.03f, 0.f, 3.36f, 0.757f}, launch_many<3, 2, 2, 4>, holds<3, 2, 2, 4>},
    {1, 256, 256, 1, 1, {0.f, 0.f, 0.f, 9.14f, 1.19f, 9.09f, 0.658f}, launch_many<4, 2, 2, 4>, holds<4, 2, 2, 4>},
    {2, 64, 64, 1, 2, {2.97f, 0.f, 0.0924f, 0.815f, 0.125f, 8.08f, 0.f}, launch_ring<1, 1, 2, 2, 4>, holds_ring<1, 1, 2, 2>},
    {2, 128, 64, 1, 1, {2.53f, 1.46f, 0.32f, 0.f, 0.f, 6.83f, 1.64f}, launch_ring<1, 1, 4, 2, 4>, holds_ring<1, 1, 4, 2>},
    kQuarter,
    kHalf,
    {3, 256, 256, 2, 1, {0.f, 0.f, 0.f, 9.14f, 1.19f, 9.09f, 0.658f}, launch_parts<2>, holds_parts<2>},
    {3, 256, 256, 4, 1, {0.f, 0.f, 0.f, 9.14f, 1.19f, 9.09f, 0.658f}, launch_parts<4>, holds_parts<4>},
};

// The shape whose estimate is the least. On 1,000 other sizes of those ranges, 3 of 10 with a residual, 1 in 4 of a width that is
// no multiple of 8 and 1 in 5 with a part of a step: 1.0 % slower than the best shape in the mean, 6 % at most for 19 of 20, 39 % at worst
// (459 rows 384 -> 1392 5.9 us in place of 4.2: widths of three steps, which the ring does not take, are the worst ones).
static const Mx8Shape& shape_of(const Mx8Args& a) {
  const float out = 2.0f * (float)a.rows * (float)(a.n[0] + a.n[1]) * 1e-7f;
  auto rounds_of = [&](const Mx8Shape& s, int64_t tiles) {
    const int64_t cu = (tiles + 255) / 256, rounds = (cu + s.held - 1) / s.held;
    const int ranges = s.kind == 0 ? s.ranges : 1;
    const float steps = (float)(((s.kind == 2 ? a.k + 127 : a.k) / 128 + ranges - 1) / ranges);
    const float gb = (float)tiles * (float)(s.tr + s.tm) * (float)a.k * 1e-9f;
    return (float)rounds * (s.us[1] + steps * s.us[2]) + (float)cu * (s.us[3] + steps * s.us[4]) + gb * s.us[5];
  };
  const Mx8Shape* best = kShapes;
  float least = 0.0f;
  for (const Mx8Shape& s : kShapes) {
    if (!s.takes(a)) continue;
    const int64_t tiles = tiles_of(a, s.tr, s.tm), rest = s.kind == 3 ? tiles % 256 : 0;
    const float us = s.us[0] + out * s.us[6] + rounds_of(s, tiles - rest) + (rest ? rounds_of(s.ranges == 2 ? kHalf : kQuarter, s.ranges * rest) : 0.0f);
    if (&s == kShapes || us < least) best = &s, least = us;
  }
  return *best;
}

}  // namespace dsv41

using namespace dsv41;

static int run_linear_mx8(const char* what, const Mx8Args& a, hipStream_t stream) {
  DSV41_REQUIRE(a.x && a.xs && a.w[0] && a.ws[0] && a.y[0], DSV41_E_ARG, "%s: null tensor", what);
  DSV41_REQUIRE(a.n[1] == 0 || (a.w[1] && a.ws[1] && a.y[1]), DSV41_E_ARG, "%s: null tensor of the second product", what);
  DSV41_REQUIRE(a.rows >= 0 && a.k > 0 && a.k % 32 == 0 && a.n[0] > 0 && a.n[1] >= 0, DSV41_E_SHAPE,
                "%s: rows %d, k %d (whole blocks of 32), n %d + %d", what, a.rows, a.k, a.n[0], a.n[1]);
  DSV41_REQUIRE(a.k <= (1 << 20) && a.n[0] <= (1 << 24) && a.n[1] <= (1 << 24) && a.rows <= (1 << 20), DSV41_E_SHAPE,
                "%s: rows %d and k %d up to 2^20, n %d + %d up to 2^24", what, a.rows, a.k, a.n[0], a.n[1]);
  DSV41_REQUIRE(a.shift == 0 || a.shift == 5, DSV41_E_SHAPE, "%s: a weight's scale covers 1 or 32 rows", what);
  DSV41_REQUIRE(a.act >= ACT_NONE && a.act <= ACT_GELU, DSV41_E_ARG, "%s: activation %d", what, a.act);
  DSV41_REQUIRE(aligned16(a.x) && aligned16(a.w[0]) && aligned16(a.y[0]) && (!a.n[1] || (aligned16(a.w[1]) && aligned16(a.y[1])))
                    && (!a.bias || aligned16(a.bias)) && (!a.residual || aligned16(a.residual)),
                DSV41_E_ARG, "%s: tensors must be 16-byte aligned", what);
  if (a.rows == 0) return 0;
  const bool ok = shape_of(a).launch(a, stream);
  DSV41_REQUIRE(ok, DSV41_E_SHAPE, "%s: rows %d, n %d + %d make too many tiles for one launch", what, a.rows, a.n[0], a.n[1]);
  return check_launch(what);
}

extern "C" int dsv41_linear_mx8(const uint8_t* x, const uint8_t* x_scales, const uint8_t* w, const uint8_t* w_scales,
                                const float* bias, const void* residual, void* y, int32_t rows, int32_t k, int32_t n,
                                int32_t scale_rows, int32_t act, hipStream_t stream) {
  Mx8Args a{};
  a.x = x, a.xs = x_scales, a.w[0] = w, a.ws[0] = w_scales, a.y[0] = static_cast<bf16_t*>(y);
  a.bias = bias, a.residual = static_cast<const bf16_t*>(residual);
  a.n[0] = n, a.rows = rows, a.k = k, a.act = act, a.shift = scale_rows == 32 ? 5 : scale_rows == 1 ? 0 : -1;
  return run_linear_mx8("dsv41_linear_mx8", a, stream);
}

extern "C" int dsv41_linear_mx8_pair(const uint8_t* x, const uint8_t* x_scales, const uint8_t* w0,
                                     const uint8_t* w0_scales, const uint8_t* w1, const uint8_t* w1_scales, void* y0,
                                     void* y1, int32_t rows, int32_t k, int32_t n0, int32_t n1, int32_t scale_rows,
                                     hipStream_t stream) {
  const char* what = "dsv41_linear_mx8_pair";
  DSV41_REQUIRE(n1 > 0, DSV41_E_SHAPE, "%s: the second product is missing", what);
  Mx8Args a{};
  a.x = x, a.xs = x_scales, a.w[0] = w0, a.ws[0] = w0_scales, a.w[1] = w1, a.ws[1] = w1_scales;
  a.y[0] = static_cast<bf16_t*>(y0), a.y[1] = static_cast<bf16_t*>(y1);
  a.n[0] = n0, a.n[1] = n1, a.rows = rows, a.k = k, a.shift = scale_rows == 32 ? 5 : scale_rows == 1 ? 0 : -1;
  return run_linear_mx8(what, a, stream);
}

extern "C" int dsv41_linear_mx8_plan(int32_t rows, int32_t k, int32_t n0, int32_t n1, int32_t plan[4]) {
  const char* what = "dsv41_linear_mx8_plan";
  DSV41_REQUIRE(plan, DSV41_E_ARG, "%s: null plan", what);
  DSV41_REQUIRE(rows > 0 && k > 0 && k % 32 == 0 && n0 > 0 && n1 >= 0, DSV41_E_SHAPE, "%s: rows %d, k %d, n %d + %d", what, rows,
                k, n0, n1);
  DSV41_REQUIRE(k <= (1 << 20) && n0 <= (1 << 24) && n1 <= (1 << 24) && rows <= (1 << 20), DSV41_E_SHAPE,
                "%s: rows %d and k %d up to 2^20, n %d + %d up to 2^24", what, rows, k, n0, n1);
  Mx8Args a{};
  a.rows = rows, a.k = k, a.n[0] = n0, a.n[1] = n1;
  const Mx8Shape& s = shape_of(a);
  plan[0] = s.kind, plan[1] = s.tr, plan[2] = s.tm, plan[3] = s.ranges;
  return 0;
}
