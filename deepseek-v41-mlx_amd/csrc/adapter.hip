// Low-rank adapters of many sequences beside one shared projection. Row m belongs to sequence m / tokens, whose
// adapter is t = ids[m / tokens]; for t in [0, slots)
//
//   h[m, :] = x[m, :] A_t^T                       A_t [rank, k]
//   y[m, :] = x[m, :] w^T + scale_t (h[m, :] B_t^T)      B_t [n, rank]
//
// and y[m, :] = x[m, :] w^T for any other t, whatever the adapters hold. h and all sums are float32, y is rounded
// once.
//
// bf16 launch shapes (the plan below picks by sizes; us of kernels on one MI355X):
//   few rows   the projection's weight is streamed once in split sums; h is computed beside it, and a second launch sums
//              the ranges and adds the adapters' part. Bound by the weight and, where every row names another adapter,
//              by B: 64 rows 1280 -> 32768 under 64 adapters of rank 16 (158 MB) 41 us, 3.9 TB/s.
//   prompts    h first, then the projection's tiles with the adapters' part in their sums when the products begin:
//              8,192 rows 8192 -> 5120 at rank 64 594 us, 1.18 PFLOP/s; few tiles split the contraction and end
//              in the same second launch.
#include <type_traits>

#include "tiles.h"

namespace dsv41 {

// ------------------------------------------------------------------ any shape

// Most workgroups of a launch that takes its items in turn: a grid holds fewer than 2^32 threads.
constexpr int64_t kMostBlocks = 1 << 23;

// h[m, r] in float32 for any width, rank and type: a workgroup per row, a wave per rank, the channels over its lanes.
template <typename T>
__global__ __launch_bounds__(256) void adapter_shrink_plain_kernel(const T* __restrict__ x, const T* __restrict__ a,
                                                                   const int32_t* __restrict__ ids,
                                                                   float* __restrict__ h, int64_t rows, int tokens,
                                                                   int k, int rank, int slots) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int64_t m = blockIdx.x; m < rows; m += gridDim.x) {
    const int t = ids[m / tokens];
    if (t < 0 || t >= slots) continue;
    const T* xp = x + m * k;
    for (int r = wave; r < rank; r += 4) {
      const T* ap = a + ((int64_t)t * rank + r) * k;
      float s = 0.0f;
      for (int c = lane; c < k; c += 64) s = fmaf(io<T>::ld(xp + c), io<T>::ld(ap + c), s);
      s = group_sum(s, 64);
      if (lane == 0) h[m * rank + r] = s;
    }
  }
}

// out[m, j] = y[m, j] + scale_t sum_r h[m, r] B_t[j, r]: one thread per output, the ranks in order.
template <typename T>
__global__ __launch_bounds__(256) void adapter_expand_plain_kernel(const T* y, const T* __restrict__ b,
                                                                   const float* __restrict__ scale,
                                                                   const int32_t* __restrict__ ids,
                                                                   const float* __restrict__ h, T* out, int64_t rows,
                                                                   int tokens, int n, int rank, int slots) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * n; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / n;
    const int j = (int)(i - m * n), t = ids[m / tokens];
    if (t < 0 || t >= slots) {
      out[i] = y[i];
      continue;
    }
    const T* bp = b + ((int64_t)t * n + j) * rank;
    const float* hp = h + m * rank;
    float s = 0.0f;
    for (int r = 0; r < rank; ++r) s = fmaf(hp[r], io<T>::ld(bp + r), s);
    io<T>::st(out + i, fmaf(scale[t], s, io<T>::ld(y + i)));
  }
}

// The projection and its adapters for any width and type on the float32 matrix cores (v_mfma_f32_16x16x4_f32: exact
// float32 arithmetic in the order of the channels): a wave per 16 rows and 16 WR output columns. Rows are the MFMA's
// columns; a lane supplies 4 channels of its row and of its weight row per load, the same 4 channels of both. The first
// product's result - ranks 4 g .. 4 g + 3 of row l16 in lane (g, l16) - is the operand of the second as it lies. Every
// adapter of the 16 rows multiplies all of them, a lane keeps its own row's. VEC: widths in whole steps of 16 channels
// and ranks of 4, loaded 4 at a time; else one by one, with zeros past the ends.
template <typename T, bool VEC>
__device__ __forceinline__ f32x4 load4(const T* p, int at, int end) {
  f32x4 v;
  if constexpr (VEC && sizeof(T) == 4) {
    v = *reinterpret_cast<const f32x4*>(p + at);
  } else if constexpr (VEC) {
    const uint2 u = *reinterpret_cast<const uint2*>(p + at);
    v = f32x4{__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16),
              __uint_as_float(u.y & 0xFFFF0000u)};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = at + e < end ? io<T>::ld(p + at + e) : 0.0f;
  }
  return v;
}

template <typename T, int WR, bool VEC>
__global__ __launch_bounds__(256) void adapter_plain_kernel(const T* __restrict__ x, const T* __restrict__ w,
                                                            const T* __restrict__ a, const T* __restrict__ b,
                                                            const float* __restrict__ scale,
                                                            const int32_t* __restrict__ ids, T* __restrict__ y, int rows,
                                                            int tokens, int k, int n, int rank, int slots) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int ctiles = (n + 16 * WR - 1) / (16 * WR);
  const int64_t tile = (int64_t)blockIdx.x * 4 + wave;
  if (tile >= (int64_t)ctiles * ((rows + 15) / 16)) return;
  const int col = (int)(tile % ctiles) * 16 * WR, m = (int)(tile / ctiles) * 16 + l16;
  const T* xp = x + (int64_t)min(m, rows - 1) * k;
  const T* wp[WR];
  f32x4 acc[WR];
#pragma unroll
  for (int i = 0; i < WR; ++i) {
    wp[i] = w + (int64_t)min(col + 16 * i + l16, n - 1) * k;
    acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll 4
  for (int c = 0; c < k; c += 16) {
    const f32x4 xf = load4<T, VEC>(xp, c + 4 * g, k);
#pragma unroll
    for (int i = 0; i < WR; ++i) {
      const f32x4 wf = load4<T, VEC>(wp[i], c + 4 * g, k);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(wf[e], xf[e], acc[i], 0, 0, 0);
    }
  }
  settle(acc);
  const int t0 = m < rows ? ids[m / tokens] : -1, id = (uint32_t)t0 < (uint32_t)slots ? t0 : -1;
  const float s = id < 0 ? 0.0f : scale[id];
  uint32_t todo = (uint32_t)__ballot(id >= 0) & 0xFFFFu;
  while (todo) {
    const int t = __builtin_amdgcn_readlane(id, __builtin_ctz(todo));
    todo &= ~(uint32_t)__ballot(id == t);
    f32x4 sum[WR];
#pragma unroll
    for (int i = 0; i < WR; ++i) sum[i] = acc[i];
    for (int q = 0; q < rank; q += 16) {
      f32x4 h[1] = {{0.f, 0.f, 0.f, 0.f}};
      const T* ap = a + ((int64_t)t * rank + min(q + l16, rank - 1)) * k;
#pragma unroll 4
      for (int c = 0; c < k; c += 16) {
        const f32x4 xf = load4<T, VEC>(xp, c + 4 * g, k), af = load4<T, VEC>(ap, c + 4 * g, k);
#pragma unroll
        for (int e = 0; e < 4; ++e) h[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(af[e], xf[e], h[0], 0, 0, 0);
      }
      settle(h);
#pragma unroll
      for (int e = 0; e < 4; ++e) h[0][e] = q + 4 * g + e < rank ? h[0][e] * s : 0.0f;
#pragma unroll
      for (int i = 0; i < WR; ++i) {
        const T* bp = b + ((int64_t)t * n + min(col + 16 * i + l16, n - 1)) * rank;
        // a rank tile's last chunks may lie past the ranks, where B is not read
        const f32x4 bf = VEC && q + 4 * g >= rank ? f32x4{0.f, 0.f, 0.f, 0.f} : load4<T, VEC>(bp, q + 4 * g, rank);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(bf[e], h[0][e], sum[i], 0, 0, 0);
      }
    }
    settle(sum);
#pragma unroll
    for (int i = 0; i < WR; ++i) acc[i] = id == t ? sum[i] : acc[i];
  }
  if (m >= rows) return;
#pragma unroll
  for (int i = 0; i < WR; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = col + 16 * i + 4 * g + e;
      if (c < n) io<T>::st(y + (int64_t)m * n + c, acc[i][e]);
    }
}

// The same for few tiles: a workgroup per 16 rows and 16 columns, its four waves a quarter of the channels each (16 at a
// time in turn), which meet in LDS; up to four adapters' first products at once, and each wave the second product of
// every fourth adapter. A short chain of loads where the other form has a long one: 256 rows 256 -> 128 in float32
// 6.2 against 9.6 us, 128 sequences 64 -> 256 under 64 adapters 8.8 against 23.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void adapter_plain_split_kernel(const T* __restrict__ x, const T* __restrict__ w,
                                                                  const T* __restrict__ a, const T* __restrict__ b,
                                                                  const float* __restrict__ scale,
                                                                  const int32_t* __restrict__ ids, T* __restrict__ y,
                                                                  int rows, int tokens, int k, int n, int rank,
                                                                  int slots) {
  extern __shared__ __align__(16) float lds[];              // [4][16][stride] partial h, then [4][16][16] results
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int stride = (rank + 15) / 16 * 16 + 4;
  float* out = lds + 4 * 16 * stride;
  const int ctiles = (n + 15) / 16, col = (int)(blockIdx.x % ctiles) * 16, m = (int)(blockIdx.x / ctiles) * 16 + l16;
  const T* xp = x + (int64_t)min(m, rows - 1) * k;
  const T* wp = w + (int64_t)min(col + l16, n - 1) * k;
  const int t0 = m < rows ? ids[m / tokens] : -1, id = (uint32_t)t0 < (uint32_t)slots ? t0 : -1;
  const uint32_t named = (uint32_t)__ballot(id >= 0) & 0xFFFFu;
  auto next = [&](uint32_t& todo) {
    const int t = __builtin_amdgcn_readlane(id, __builtin_ctz(todo));
    todo &= ~(uint32_t)__ballot(id == t);
    return t;
  };
  f32x4 acc[1] = {{0.f, 0.f, 0.f, 0.f}};
#pragma unroll 4
  for (int c = 16 * wave; c < k; c += 64) {
    const f32x4 xf = load4<T, VEC>(xp, c + 4 * g, k), wf = load4<T, VEC>(wp, c + 4 * g, k);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(wf[e], xf[e], acc[0], 0, 0, 0);
  }
  settle(acc);
  if (named) {
    for (int q = 0; q < rank; q += 16) {
      f32x4 res = {0.f, 0.f, 0.f, 0.f};
      uint32_t todo = named;
      while (todo) {
        int t[4];
        t[0] = next(todo);
#pragma unroll
        for (int u = 1; u < 4; ++u) t[u] = todo ? next(todo) : t[0];
        f32x4 h[4];
        const T* ap[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          h[u] = f32x4{0.f, 0.f, 0.f, 0.f};
          ap[u] = a + ((int64_t)t[u] * rank + min(q + l16, rank - 1)) * k;
        }
#pragma unroll 4
        for (int c = 16 * wave; c < k; c += 64) {
          const f32x4 xf = load4<T, VEC>(xp, c + 4 * g, k);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const f32x4 af = load4<T, VEC>(ap[u], c + 4 * g, k);
#pragma unroll
            for (int e = 0; e < 4; ++e) h[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(af[e], xf[e], h[u], 0, 0, 0);
          }
        }
        settle(h);
#pragma unroll
        for (int u = 0; u < 4; ++u) res = id == t[u] ? h[u] : res;
      }
      *reinterpret_cast<f32x4*>(lds + (wave * 16 + l16) * stride + q + 4 * g) = res;
    }
    __syncthreads();
    // each wave sums what it needs itself: its lanes' own rows
    const float s = id < 0 ? 0.0f : scale[id];
    uint32_t todo = named;
    for (int at = 0; todo; ++at) {
      const int t = next(todo);
      if ((at & 3) != wave) continue;
      f32x4 sum[1] = {acc[0]};
      const T* bp = b + ((int64_t)t * n + min(col + l16, n - 1)) * rank;
#pragma unroll 4
      for (int q = 0; q < rank; q += 16) {
        const float* hp = lds + l16 * stride + q + 4 * g;
        f32x4 h = *reinterpret_cast<const f32x4*>(hp);
#pragma unroll
        for (int v = 1; v < 4; ++v) {
          const f32x4 more = *reinterpret_cast<const f32x4*>(hp + v * 16 * stride);
#pragma unroll
          for (int e = 0; e < 4; ++e) h[e] += more[e];
        }
        const f32x4 bf = VEC && q + 4 * g >= rank ? f32x4{0.f, 0.f, 0.f, 0.f} : load4<T, VEC>(bp, q + 4 * g, rank);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = q + 4 * g + e < rank ? h[e] * s : 0.0f;
          sum[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(bf[e], v, sum[0], 0, 0, 0);
        }
      }
      settle(sum);
      acc[0] = id == t ? sum[0] : acc[0];
    }
  }
  // lane (g, l16) holds columns 4 g .. 4 g + 3 of row l16
  *reinterpret_cast<f32x4*>(out + (wave * 16 + l16) * 16 + 4 * g) = acc[0];
  __syncthreads();
  const int row = threadIdx.x >> 4, c = col + (threadIdx.x & 15), mo = (int)(blockIdx.x / ctiles) * 16 + row;
  if (mo < rows && c < n) {
    float v = out[threadIdx.x];
#pragma unroll
    for (int u = 1; u < 4; ++u) v += out[u * 256 + threadIdx.x];
    io<T>::st(y + (int64_t)mo * n + c, v);
  }
}

// ------------------------------------------------------------------ matrix cores (bf16)

// One projection's adapters as the kernels see them.
struct Bank {
  const bf16_t* a;       // [slots, rank, k]
  const bf16_t* b;       // [slots, n, rank]
  const float* scale;    // [slots]
  float* h;              // x A^T per contraction chunk: [chunks, rows, rank]
  int rank, slots;       // rank a multiple of 8, at most kMaxRank; slots 0: no bank
};

constexpr int kMaxRank = 128;

struct AdapterArgs {
  WoaArgs t;             // the projection itself: split form, t.groups contraction ranges of t.d channels, weight rows
                         // [t.r0, t.r) in t.w1 when there are two; t.out: float32 parts or the result
  Bank bank[2];          // of weight rows [0, t.r0) and [t.r0, t.r)
  const int32_t* ids;    // [rows / tokens]
  int tokens, k;
  int chunk, chunks;     // channels of one partial h, and how many
  int sub;               // rows of a share of it: 4 or 16
  int done;              // h is finished before the tiles' launch
  int apart;             // leading workgroups that compute shares of h and no tile (0: the tiles' workgroups do)
  bf16_t* y;             // [rows, t.r0]
  bf16_t* y1;            // [rows, t.r - t.r0]
};

// The adapter of row m: -1 for none.
__device__ __forceinline__ int row_adapter(const AdapterArgs& a, const Bank& bk, int m) {
  const int t = m < a.t.rows ? a.ids[m / a.tokens] : -1;
  return (uint32_t)t < (uint32_t)bk.slots ? t : -1;
}

// The next adapter that occurs in a tile of 16 rows (lane l holds row l % 16's): takes its rows out of `todo`.
__device__ __forceinline__ int next_adapter(uint32_t& todo, int id) {
  const int t = __builtin_amdgcn_readlane(id, __builtin_ctz(todo));
  todo &= ~(uint32_t)__ballot(id == t);
  return t;
}

__device__ __forceinline__ bf16x8 or_zero(uint4 v, bool live) {
  return as_bf16x8(live ? v : make_uint4(0, 0, 0, 0));
}

// Partial x A^T of `sub` rows (4 or 16), one chunk of channels, 16 ranks: the chunk's 32-channel steps in turn over the
// workgroup's four waves. Rows are the MFMA's columns, so every adapter of the tile multiplies all of them and each lane
// keeps the product with its own row's: nothing another row's adapter holds can reach it. U adapters and four steps at
// once keep that many loads in flight; a step past the end multiplies nothing.
template <int U>
__device__ __forceinline__ void shrink_steps(const bf16_t* xp, const bf16_t* const (&ap)[U], int first, int steps,
                                             f32x4 (&acc)[U]) {
#pragma unroll
  for (int u = 0; u < U; ++u) acc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s = first; s < steps; s += 16) {
    uint4 xf[4], af[4][U];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int at = 32 * min(s + 4 * e, steps - 1);
      xf[e] = *reinterpret_cast<const uint4*>(xp + at);
#pragma unroll
      for (int u = 0; u < U; ++u) af[e][u] = *reinterpret_cast<const uint4*>(ap[u] + at);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool live = s + 4 * e < steps;
#pragma unroll
      for (int u = 0; u < U; ++u) acc[u] = mfma16x16x32(or_zero(af[e][u], live), or_zero(xf[e], live), acc[u]);
    }
  }
  settle(acc);
}

__device__ __forceinline__ int shrink_items(const AdapterArgs& a, const Bank& bk) {
  return bk.slots ? (a.t.rows + a.sub - 1) / a.sub * a.chunks * ((bk.rank + 15) / 16) : 0;
}

__device__ __forceinline__ void shrink_item(const AdapterArgs& a, const Bank& bk, int item, float* red) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int ranks = (bk.rank + 15) / 16;
  const int rq = item % ranks, chunk = item / ranks % a.chunks, tile = item / ranks / a.chunks;
  const int m0 = tile * a.sub + (l16 & (a.sub - 1));       // 4 rows: each four times
  const int id = row_adapter(a, bk, m0);
  const int k0 = chunk * a.chunk, steps = min(a.chunk, a.k - k0) / 32;
  const bf16_t* xp = a.t.o + (int64_t)min(m0, a.t.rows - 1) * a.k + k0 + 8 * g;
  const int64_t arow = (int64_t)min(rq * 16 + l16, bk.rank - 1) * a.k + k0 + 8 * g;   // ranks past the end: not stored
  const int64_t slot = (int64_t)bk.rank * a.k;
  f32x4 res = {0.f, 0.f, 0.f, 0.f};
  uint32_t todo = (uint32_t)__ballot(id >= 0) & ((1u << a.sub) - 1u);
  while (todo) {
    int t[4];
    t[0] = next_adapter(todo, id);
    if (todo == 0) {
      f32x4 acc[1];
      const bf16_t* const ap[1] = {bk.a + t[0] * slot + arow};
      shrink_steps<1>(xp, ap, wave, steps, acc);
      res = id == t[0] ? acc[0] : res;
      break;
    }
#pragma unroll
    for (int u = 1; u < 4; ++u) t[u] = todo ? next_adapter(todo, id) : t[0];
    f32x4 acc[4];
    const bf16_t* const ap[4] = {bk.a + t[0] * slot + arow, bk.a + t[1] * slot + arow, bk.a + t[2] * slot + arow,
                                 bk.a + t[3] * slot + arow};
    shrink_steps<4>(xp, ap, wave, steps, acc);
#pragma unroll
    for (int u = 0; u < 4; ++u) res = id == t[u] ? acc[u] : res;
  }
  // the four waves' sums, in order; lane (g, l16) holds ranks 4 g .. 4 g + 3 of row l16
  *reinterpret_cast<f32x4*>(red + (wave * 16 + l16) * 16 + 4 * g) = res;
  __syncthreads();
  const int row = threadIdx.x >> 4, r = rq * 16 + (threadIdx.x & 15), m = tile * a.sub + row;
  if (row < a.sub && m < a.t.rows && r < bk.rank) {
    float s = red[threadIdx.x];
#pragma unroll
    for (int w = 1; w < 4; ++w) s += red[w * 256 + threadIdx.x];
    bk.h[((int64_t)chunk * a.t.rows + m) * bk.rank + r] = s;
  }
  __syncthreads();
}

// Ranks 8 c .. 8 c + 7 of scale h as an operand of the second product: it takes the sum of three bf16 values - the upper
// 8 bits, cut off, the next 8, cut off, and what is left, 8 bits again - so that all 24 bits count; each is multiplied
// with the same bf16 B, exactly. An infinite value has no lower parts.
__device__ __forceinline__ uint4 part_of(const float* v, int part) {
  uint32_t w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t upper = __float_as_uint(v[e]) & 0xFFFF0000u;
    const float rest = upper << 1 == 0xFF000000u ? 0.0f : v[e] - __uint_as_float(upper);
    const uint32_t next = __float_as_uint(rest) & 0xFFFF0000u;
    const uint32_t last = __float_as_uint(rest - __uint_as_float(next));
    w[e] = part == 0 ? upper : part == 1 ? next : last;
  }
  auto pair = [&](int e) { return (w[e] >> 16) | (w[e + 1] & 0xFFFF0000u); };
  return make_uint4(pair(0), pair(2), pair(4), pair(6));
}

// The operands that lane group g supplies to step q of the second product: parts of one rank chunk of 8. Up to 16 ranks
// are one step of one MFMA for the chunks' upper, next and last parts in turn, and a second one for the last parts that
// it has no room for (two chunks' six parts). More take 4 chunks a step and an MFMA per part, on one load of B (16
// sequences' own B of rank 64 for 32768 outputs: 24.6 us, 43 when it was loaded for each of two parts).
struct RankSlot {
  int c, part;                                             // the chunk, and its part in the first MFMA
  bool live, last;                                         // in the first MFMA (and the next part's), in the last part's
  __device__ __forceinline__ RankSlot(int q, int r8) {
    const int g = (threadIdx.x >> 4) & 3;
    const bool few = r8 <= 2;
    part = few ? min(g / r8, 2) : 0;
    c = few ? g % r8 : 4 * q + g;
    live = few ? g < 3 * r8 : c < r8;
    last = few ? g < 3 * r8 - 4 : live;
    if (!live) c = 0;
  }
  __device__ __forceinline__ static int steps(int r8) { return r8 <= 2 ? 1 : (r8 + 3) / 4; }
};

// The whole first product of up to 16 MT rows of one sequence - so of one adapter - and 16 RT ranks. x and A come to LDS
// 256 channels at a time (a copy instruction takes 512 bytes of each of two rows: fragments loaded from memory directly
// touch 16 rows per instruction: 8,192 rows of 8192 channels at rank 64 took 63 us, 41 this way), NS - 1 steps ahead;
// MT RT waves take a 16 x 16 tile each, times KS that share a step's channels. Writes the second product's operand: per
// row the upper parts of scale h's ranks, then the next ones, then the last ([rows, 3 rank] bf16). Rows without an
// adapter are left as they are.
//
// A step's tile row is 32 chunks of 16 bytes; chunk c of row r lies at c ^ (r & 15) (and within the 32), so that the 16
// rows of a fragment read start in different banks.
template <int MT, int RT, int KS>
struct ShrinkCfg {
  static constexpr int NW = MT * RT * KS, ROWS = 16 * (MT + RT), STAGE = ROWS * 512;
  static constexpr int COPIES = ROWS / 2 / NW;                                     // per wave and step
  static constexpr int NS = 156 * 1024 / STAGE > 6 ? 6 : 156 * 1024 / STAGE;
  static_assert(COPIES * NW * 2 == ROWS, "whole copies per wave");
  static_assert(KS * MT * RT * 1024 <= NS * STAGE, "the waves' sums fit the ring");
};

template <int MT, int RT, int KS>
__global__ __launch_bounds__(64 * MT * RT * KS) void adapter_shrink_kernel(AdapterArgs a) {
  using C = ShrinkCfg<MT, RT, KS>;
  __shared__ __align__(16) uint8_t ring[C::NS * C::STAGE];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  // rank tiles of the first bank, then the second's
  const int rtiles0 = (a.bank[0].rank + 16 * RT - 1) / (16 * RT), rtiles = rtiles0 + (a.bank[1].rank + 16 * RT - 1) / (16 * RT);
  const int mtiles = (a.tokens + 16 * MT - 1) / (16 * MT);
  const int rt = (int)(blockIdx.x % rtiles), mt = (int)(blockIdx.x / rtiles % mtiles), seq = (int)(blockIdx.x / rtiles / mtiles);
  const Bank& bk = a.bank[rt >= rtiles0];
  const int t = a.ids[seq];
  if ((uint32_t)t >= (uint32_t)bk.slots) return;
  const int r0 = (rt >= rtiles0 ? rt - rtiles0 : rt) * 16 * RT, rows = min(16 * MT, a.tokens - mt * 16 * MT);
  const int64_t m0 = (int64_t)seq * a.tokens + mt * 16 * MT;
  // copy j of a wave: tile rows 2 (wave COPIES + j) and + 1, x's first; lane l takes position l % 32 of its row. Rows past
  // the sequence or the ranks repeat the last one: not stored
  uint64_t src[C::COPIES];
  int chunk[C::COPIES];
#pragma unroll
  for (int j = 0; j < C::COPIES; ++j) {
    const int r = 2 * (wave * C::COPIES + j) + (lane >> 5);
    chunk[j] = (lane & 31) ^ (r & 15);
    src[j] = r < 16 * MT ? reinterpret_cast<uint64_t>(a.t.o + (m0 + min(r, rows - 1)) * a.k)
                         : reinterpret_cast<uint64_t>(bk.a + ((int64_t)t * bk.rank + min(r0 + r - 16 * MT, bk.rank - 1)) * a.k);
  }
  const uint32_t lds0 = lds_offset(ring);
  const int chunks = a.k / 8, steps = (a.k + 255) / 256;
  auto issue = [&](int buf, int step) {
    const uint32_t at = (uint32_t)__builtin_amdgcn_readfirstlane((int)(lds0 + (uint32_t)(buf * C::STAGE + wave * C::COPIES * 1024)));
#pragma unroll
    for (int j = 0; j < C::COPIES; ++j)      // chunks past the last channel repeat the last: not multiplied
      dma16_vaddr(src[j] + 16 * (uint64_t)min(32 * step + chunk[j], chunks - 1), at + j * 1024);
  };
  const int part = wave % KS, j0 = wave / KS % MT, i0 = wave / KS / MT;     // this wave's channels and tile
  f32x4 acc[1] = {{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
  for (int p = 0; p < C::NS - 1; ++p)
    if (p < steps) issue(p, p);
  for (int st = 0; st < steps; ++st) {
    wait_copies_deep<C::COPIES, C::NS - 2>(min(C::NS - 2, steps - 1 - st));
    __syncthreads();
    if (st + C::NS - 1 < steps) issue((st + C::NS - 1) % C::NS, st + C::NS - 1);
    const uint8_t* xt = ring + (st % C::NS) * C::STAGE + (16 * j0 + l16) * 512;
    const uint8_t* at = ring + (st % C::NS) * C::STAGE + (16 * (MT + i0) + l16) * 512;
    const int live = min(8, (a.k - 256 * st) / 32);
#pragma unroll
    for (int s = 0; s < 8; s += KS) {
      if (s + part >= live) continue;
      const int c = ((4 * (s + part) + g) ^ l16) << 4;
      acc[0] = mfma16x16x32(ld_bf16x8(at + c), ld_bf16x8(xt + c), acc[0]);
    }
  }
  settle(acc);
  // lane (g, l16) holds ranks 4 g .. 4 g + 3 of row l16 of its tile
  __syncthreads();
  float* red = reinterpret_cast<float*>(ring);               // [KS][16 MT][16 RT]
  *reinterpret_cast<f32x4*>(red + ((part * 16 * MT + 16 * j0 + l16) * RT + i0) * 16 + 4 * g) = acc[0];
  __syncthreads();
  uint16_t* hl = reinterpret_cast<uint16_t*>(bk.h);
  const float scale = bk.scale[t];
  for (int q = threadIdx.x; q < MT * RT * 32; q += 64 * C::NW) {           // 8 ranks of one row each
    const int row = q / (2 * RT), r = r0 + 8 * (q % (2 * RT));
    if (row >= rows || r >= bk.rank) continue;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float sum = red[q * 8 + e];
#pragma unroll
      for (int w = 1; w < KS; ++w) sum += red[w * MT * RT * 256 + q * 8 + e];
      v[e] = sum * scale;
    }
    uint16_t* to = hl + (m0 + row) * 3 * bk.rank + r;
#pragma unroll
    for (int part = 0; part < 3; ++part) *reinterpret_cast<uint4*>(to + part * bk.rank) = part_of(v, part);
  }
}

// The second product for 16 rows (lane l16's, adapter id) and WR tiles of 16 output columns, in steps of one rank group
// (32 of the rank operands) and up to U adapters, each step's B loaded a step ahead; the first one's before the
// caller has h at all. Rows are the MFMA's columns: each adapter multiplies all of them, a lane keeps its own row's.
// FEW: up to 16 ranks.
template <int WR, int U, bool FEW>
struct Expand {
  const bf16_t* b;       // slot 0, the lane's first output column
  int64_t slot;
  int rank, id;
  uint32_t named, todo;  // rows with an adapter; those whose adapter is still to come in this rank group
  int q;                 // the rank step
  int t[U];
  uint4 next[U][WR];

  __device__ __forceinline__ void load() {
    t[0] = next_adapter(todo, id);
#pragma unroll
    for (int u = 1; u < U; ++u) t[u] = todo ? next_adapter(todo, id) : t[0];
    const bf16_t* p = b + 8 * RankSlot(q, rank >> 3).c;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < WR; ++i) next[u][i] = *reinterpret_cast<const uint4*>(p + t[u] * slot + (int64_t)16 * i * rank);
  }
  __device__ __forceinline__ Expand(const Bank& bk, int n, int col, int id_, uint32_t named_)
      : b(bk.b + (int64_t)(col + (threadIdx.x & 15)) * bk.rank), slot((int64_t)n * bk.rank), rank(bk.rank), id(id_),
        named(named_), todo(named_), q(0) {
    load();
  }
  // operand(c, part) gives a part of scale h's ranks 8 c .. 8 c + 7 of the lane's row
  template <typename H>
  __device__ __forceinline__ void add(f32x4 (&acc)[WR], H operand) {
    const int r8 = rank >> 3, end = RankSlot::steps(r8);
    bf16x8 upper, next_part, last;
    bool fresh = true;
    for (;;) {
      const RankSlot at(q, r8);
      if (fresh) {
        upper = or_zero(operand(at.c, at.part), at.live);
        if constexpr (!FEW) next_part = or_zero(operand(at.c, 1), at.live);
        last = or_zero(operand(at.c, 2), at.last);
      }
      int now[U];
      uint4 cur[U][WR];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        now[u] = t[u];
#pragma unroll
        for (int i = 0; i < WR; ++i) cur[u][i] = next[u][i];
      }
      fresh = todo == 0;
      if (fresh) {
        ++q;
        todo = named;
      }
      const bool more = q < end;
      if (more) load();
      // no branch between an MFMA and the choice of its result
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < WR; ++i) {
          // an operand that is not there multiplies no B either: 0 times infinity would stay
          f32x4 sum = mfma16x16x32(or_zero(cur[u][i], at.live), upper, acc[i]);
          if constexpr (!FEW) sum = mfma16x16x32(or_zero(cur[u][i], at.live), next_part, sum);
          sum = mfma16x16x32(or_zero(cur[u][i], at.last), last, sum);
          acc[i] = id == now[u] && (u == 0 || now[u] != now[0]) ? sum : acc[i];
        }
      if (!more) return;
    }
  }
};

// acc[i][j] += scale (h B^T) for a wave's block of 16 WM rows from m0 on and 16 WR columns from col on, h from the
// finished first product. One adapter for all rows that are stored: its products go straight into the sums. Several:
// each multiplies the groups of 16 rows that name it and every lane keeps its own row's, one result beside the sums at a
// time where they fill the registers (110 rows of 32768 outputs under 64 adapters of rank 64: 169 us, 299 when each
// adapter met all rows, whose operands come through the L2 for every adapter).
template <int WR, int WM>
__device__ __forceinline__ void expand_block(f32x4 (&acc)[WR][WM], const AdapterArgs& a, const Bank& bk, int n, int m0,
                                             int col) {
  const int l16 = threadIdx.x & 15, r8 = bk.rank >> 3;
  int id[WM];
  uint32_t todo[WM];
  const uint16_t* hp[WM];
  int t = -1;
#pragma unroll
  for (int j = 0; j < WM; ++j) {
    const int m = m0 + 16 * j + l16;
    id[j] = row_adapter(a, bk, m);
    todo[j] = (uint32_t)__ballot(id[j] >= 0) & 0xFFFFu;
    if (t < 0 && todo[j]) t = __builtin_amdgcn_readlane(id[j], __builtin_ctz(todo[j]));
    hp[j] = reinterpret_cast<const uint16_t*>(bk.h) + (int64_t)min(m, a.t.rows - 1) * 3 * bk.rank;
  }
  if (t < 0) return;
  // A load behind a branch, which the compiler takes to be on its way still, would have it wait in the tile's loop, for
  // the copies there too (4,096 rows 5120 -> 1280: 98 us against 82). The copies issued so far have come before the loads.
  auto drained = [&]() { __builtin_amdgcn_s_waitcnt(0x0F70); };        // vmcnt(0)
  bool one = true;
#pragma unroll
  for (int j = 0; j < WM; ++j) one = one && __ballot(id[j] != t && m0 + 16 * j + l16 < a.t.rows) == 0;
  const bf16_t* b0 = bk.b + (int64_t)(col + l16) * bk.rank;
  const int64_t slot = (int64_t)n * bk.rank;
  // an operand that is not there multiplies no B either: 0 times infinity would stay
  if (one) {
    for (int q = 0; q < RankSlot::steps(r8); ++q) {
      const RankSlot at(q, r8);
      const bf16_t* bp = b0 + t * slot + 8 * at.c;
      bf16x8 bf[WR];
#pragma unroll
      for (int i = 0; i < WR; ++i) bf[i] = or_zero(*reinterpret_cast<const uint4*>(bp + (int64_t)16 * i * bk.rank), at.live);
      auto load = [&](bf16x8 (&h)[WM], int part, bool live) {
#pragma unroll
        for (int j = 0; j < WM; ++j) h[j] = or_zero(*reinterpret_cast<const uint4*>(hp[j] + 8 * at.c + part * bk.rank), live);
      };
      auto multiply = [&](const bf16x8 (&h)[WM]) {
#pragma unroll
        for (int j = 0; j < WM; ++j)
#pragma unroll
          for (int i = 0; i < WR; ++i) acc[i][j] = mfma16x16x32(bf[i], h[j], acc[i][j]);
      };
      auto mask = [&]() {
#pragma unroll
        for (int i = 0; i < WR; ++i) bf[i] = or_zero(__builtin_bit_cast(uint4, bf[i]), at.last);
      };
      if constexpr (WR * WM <= 20) {
        bf16x8 h0[WM], h1[WM], h2[WM];
        load(h0, at.part, at.live);
        if (r8 > 2) load(h1, 1, at.live);
        if (r8 > 1) load(h2, 2, at.last);
        multiply(h0);
        if (r8 > 2) multiply(h1);
        if (r8 > 1) {
          mask();
          multiply(h2);
        }
      } else {
        bf16x8 h[WM];                                      // one part at a time: all of them spill 127 registers
#pragma unroll 1
        for (int p = 0; p < (r8 < 3 ? r8 : 3); ++p) {
          load(h, p == 0 ? at.part : r8 > 2 ? p : 2, p == 0 || r8 > 2 ? at.live : at.last);
          if (p > 0) mask();                               // the same lanes again beyond 16 ranks
          multiply(h);
        }
      }
    }
    drained();
#pragma unroll
    for (int i = 0; i < WR; ++i) settle(acc[i]);
    return;
  }
  while (t >= 0) {
    uint32_t hit[WM];
#pragma unroll
    for (int j = 0; j < WM; ++j) {
      hit[j] = (uint32_t)__ballot(id[j] == t) & 0xFFFFu;
      todo[j] &= ~hit[j];
    }
    // B is loaded once for its parts; 16 rows without this adapter are passed over
    for (int q = 0; q < RankSlot::steps(r8); ++q) {
      const RankSlot at(q, r8);
      const bf16_t* bp = b0 + t * slot + 8 * at.c;
      bf16x8 bf[WR];
#pragma unroll
      for (int i = 0; i < WR; ++i) bf[i] = ld_bf16x8(bp + (int64_t)16 * i * bk.rank);
      auto load = [&](uint4 (&h)[WM], int part) {
#pragma unroll
        for (int j = 0; j < WM; ++j)
          if (hit[j]) h[j] = *reinterpret_cast<const uint4*>(hp[j] + 8 * at.c + part * bk.rank);
      };
      auto multiply = [&](const uint4 (&h)[WM], bool live) {
#pragma unroll
        for (int i = 0; i < WR; ++i) bf[i] = or_zero(__builtin_bit_cast(uint4, bf[i]), live);
#pragma unroll
        for (int j = 0; j < WM; ++j) {
          if (hit[j] == 0) continue;
          const bf16x8 hf = or_zero(h[j], live);
#pragma unroll
          for (int i = 0; i < WR; ++i) {
            const f32x4 sum = mfma16x16x32(bf[i], hf, acc[i][j]);
            acc[i][j] = id[j] == t ? sum : acc[i][j];
            if constexpr (WR * WM > 8) __builtin_amdgcn_sched_barrier(0);
          }
        }
      };
      if constexpr (WR * WM <= 8) {
        uint4 h0[WM], h1[WM], h2[WM];
        load(h0, at.part);
        if (r8 > 2) load(h1, 1);
        if (r8 > 1) load(h2, 2);
        multiply(h0, at.live);
        if (r8 > 2) multiply(h1, at.live);
        if (r8 > 1) multiply(h2, at.last);
      } else {
        uint4 now[WM], next[WM];                           // one part ahead: more leave no registers
        load(next, at.part);
#pragma unroll 1
        for (int p = 0, parts = r8 < 3 ? r8 : 3; p < parts; ++p) {
#pragma unroll
          for (int j = 0; j < WM; ++j) now[j] = next[j];
          if (p + 1 < parts) load(next, r8 > 2 ? p + 1 : 2);
          __builtin_amdgcn_sched_barrier(0);
          multiply(now, p == 0 || r8 > 2 ? at.live : at.last);
        }
      }
    }
    t = -1;
#pragma unroll
    for (int j = 0; j < WM; ++j)
      if (t < 0 && todo[j]) t = __builtin_amdgcn_readlane(id[j], __builtin_ctz(todo[j]));
  }
  drained();
}

// The projection's tiles. DIRECT: the adapters' part is added to the float32 sums in registers and the result stored,
// rounded once (h complete before the launch). Else the sums of one contraction range go to t.out in float32, and h is
// computed beside them: by workgroups of their own where the launch leaves room for them, else by the tiles' own, each
// its share while its first copies are on their way.
template <int WR, int WM, int GR, int GM, int BK, int NS, bool DIRECT>
__global__ __launch_bounds__(64 * GR * GM, (TileCfg<WR, WM, GR, GM, BK, NS>::LDS <= 72 * 1024) ? 2 : 1) void
adapter_tiles_kernel(AdapterArgs a) {
  using C = TileCfg<WR, WM, GR, GM, BK, NS>;
  __shared__ __align__(16) uint8_t lds[C::LDS];
  const int mtiles = (a.t.rows + C::TM - 1) / C::TM, rtiles = a.t.r / C::TR;
  const int apart = DIRECT ? 0 : a.apart, total = (int)gridDim.x - apart, block = (int)blockIdx.x - apart;
  int rt, mt, grp = 0;
  if constexpr (!DIRECT) {
    // consecutive tiles on one XCD, the weight tile fastest, as the output projection's
    const int tile = total % 8 ? block : (block % 8) * (total / 8) + block / 8;
    rt = tile % rtiles;
    mt = (tile / rtiles) % mtiles;
    grp = tile / (rtiles * mtiles);
  } else {
    // consecutive tiles on one XCD, in bands of 4 query tiles: 32 CUs work on 4 x 8 tiles and share their 12 operand
    // panels in the XCD's L2, where 1 x 32 tiles read 33 (no faster by itself; bands of 2, 8 and 16 measure alike)
    constexpr int kBand = 4;
    const int xcd = block % 8, per = total / 8, more = total % 8;
    const int tile = xcd * per + min(xcd, more) + block / 8;
    const int band = tile / (kBand * rtiles), in = tile - band * kBand * rtiles, width = min(kBand, mtiles - band * kBand);
    rt = in / width;
    mt = band * kBand + in - rt * width;
  }
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wr = (wave % GR) * 16 * WR, wm = (wave / GR) * 16 * WM;   // this wave's block
  f32x4 acc[WR][WM];
  if constexpr (DIRECT) {
    // a tile lies within one of the two projections
    const int sel = rt * C::TR >= a.t.r0, n = sel ? a.t.r - a.t.r0 : a.t.r0, col = rt * C::TR + wr - (sel ? a.t.r0 : 0);
    const Bank& bk = a.bank[sel];
    bf16_t* y = sel ? a.y1 : a.y;
    // the adapters' part first, while the ring's first copies are on their way
    auto beside = [&]() { expand_block<WR, WM>(acc, a, bk, n, mt * C::TM + wm, col); };
    if constexpr (BK == 64 && NS == 2) tile_sums_ahead<WR, WM, GR, GM>(a.t, lds, rt, mt, grp, acc, beside);
    else tile_sums<WR, WM, GR, GM, BK, NS>(a.t, lds, rt, mt, grp, acc, beside);
#pragma unroll
    for (int i = 0; i < WR; ++i) settle(acc[i]);
#pragma unroll
    for (int j = 0; j < WM; ++j) {
      const int m = mt * C::TM + wm + 16 * j + l16;
      bf16_t* to = y + (int64_t)m * n + col;
      // the swaps of a pair need every lane: a row past the end gives the store up after them
#pragma unroll
      for (int i = 0; i + 1 < WR; i += 2) {
        uint4 v = pair_of(acc[i][j], acc[i + 1][j]);
        if (m < a.t.rows) *reinterpret_cast<uint4*>(to + 16 * i + 16 * (g & 1) + 8 * (g >> 1)) = v;
      }
      if constexpr (WR % 2 != 0)
        if (m < a.t.rows) store4<bf16_t>(to + 16 * (WR - 1) + 4 * g, acc[WR - 1][j]);
    }
  } else {
    static_assert(GR * GM == 4, "a partial h is the work of four waves");
    __shared__ __align__(16) float red[4 * 256];
    auto shares = [&](int first, int step) {
      const int items0 = shrink_items(a, a.bank[0]), items = items0 + shrink_items(a, a.bank[1]);
      for (int it = first; it < items; it += step)
        if (it < items0) shrink_item(a, a.bank[0], it, red);
        else shrink_item(a, a.bank[1], it - items0, red);
      return first < items;
    };
    if (block < 0) {
      shares(blockIdx.x, apart);
      return;
    }
    auto beside = [&]() {
      // the ring's waits count its own copies only
      if (!a.done && apart == 0 && shares(block, total)) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    };
    if constexpr (BK == 64 && NS == 2) tile_sums_ahead<WR, WM, GR, GM>(a.t, lds, rt, mt, grp, acc, beside);
    else tile_sums<WR, WM, GR, GM, BK, NS>(a.t, lds, rt, mt, grp, acc, beside);
#pragma unroll
    for (int i = 0; i < WR; ++i) settle(acc[i]);
    const int64_t ostride = (int64_t)a.t.groups * a.t.r;
    float* out = reinterpret_cast<float*>(a.t.out);
#pragma unroll
    for (int j = 0; j < WM; ++j) {
      const int m = mt * C::TM + wm + 16 * j + l16;
      if (m >= a.t.rows) continue;
#pragma unroll
      for (int i = 0; i < WR; ++i)
        store4<float>(out + m * ostride + (int64_t)grp * a.t.r + rt * C::TR + wr + 16 * i + 4 * g, acc[i][j]);
    }
  }
}

// The contraction ranges' parts summed in order, plus the adapters' part, rounded once: a workgroup per SUB rows (4, each
// four times in the MFMA, where they may all name different adapters: one load of B behind another for each; else 16) and
// 64 WR columns, a wave per 16 WR of them (whole blocks of one projection: n0 and n are multiples of 16 WR). The first
// adapters' B and the first range's parts are on their way while h is summed over its chunks into LDS; the other ranges'
// parts come one behind another. DONE: h is the finished first
// product, as it lies.
template <int WR, bool DONE, int SUB>
__global__ __launch_bounds__(256) void adapter_reduce_kernel(AdapterArgs a) {
  constexpr int kStride = kMaxRank + 4;
  __shared__ __align__(16) float hs[DONE ? 1 : 2][DONE ? 4 : SUB * kStride];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int ctiles = (a.t.r + 64 * WR - 1) / (64 * WR);
  const int col0 = (int)(blockIdx.x % ctiles) * 64 * WR, m0 = (int)(blockIdx.x / ctiles) * SUB;
  const int m = m0 + (l16 & (SUB - 1)), col = min(col0 + wave * 16 * WR, a.t.r - 16 * WR);   // a wave past the end repeats the last
  const int sel = col >= a.t.r0, n = sel ? a.t.r - a.t.r0 : a.t.r0, at = sel ? col - a.t.r0 : col;
  const Bank& bk = a.bank[sel];
  const int id = row_adapter(a, bk, m);
  const uint32_t named = (uint32_t)__ballot(id >= 0) & ((1u << SUB) - 1u);
  const float* part = reinterpret_cast<const float*>(a.t.out) + (int64_t)min(m, a.t.rows - 1) * a.t.groups * a.t.r + col + 4 * g;
  f32x4 acc[WR];

  auto sum_parts = [&]() {
#pragma unroll
    for (int i = 0; i < WR; ++i) acc[i] = *reinterpret_cast<const f32x4*>(part + 16 * i);
    for (int p = 1; p < a.t.groups; ++p)
#pragma unroll
      for (int i = 0; i < WR; ++i) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(part + (int64_t)p * a.t.r + 16 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] = acc[i][e] + v[e];
      }
  };
  auto sum_h = [&]() {
    if constexpr (DONE) return;
#pragma unroll
    for (int s = 0; s < 2 && !DONE; ++s) {
      const Bank& bs = a.bank[s];
      if (bs.slots == 0 || (s == 0 ? col0 >= a.t.r0 : col0 + 64 * WR <= a.t.r0)) continue;
      const int quads = bs.rank >> 2;
      for (int i = threadIdx.x; i < SUB * quads; i += 256) {
        const int row = i / quads, r = (i - row * quads) * 4, t = row_adapter(a, bs, m0 + row);
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (t >= 0) {
          const float* hp = bs.h + (int64_t)(m0 + row) * bs.rank + r;
          const int64_t step = (int64_t)a.t.rows * bs.rank;
          const float scale = bs.scale[t];
#pragma unroll 8
          for (int p = 0; p < a.chunks; ++p) {
            const f32x4 h = *reinterpret_cast<const f32x4*>(hp + p * step);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += h[e];
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] *= scale;
        }
        *reinterpret_cast<f32x4*>(hs[s] + row * kStride + r) = v;
      }
    }
    __syncthreads();
  };
  auto operand = [&](int c, int which) {
    if constexpr (DONE) {
      const uint16_t* from = reinterpret_cast<const uint16_t*>(bk.h) + (int64_t)min(m, a.t.rows - 1) * 3 * bk.rank;
      return *reinterpret_cast<const uint4*>(from + 8 * c + which * bk.rank);
    } else {
      float v[8];
      const float* from = hs[sel] + (l16 & (SUB - 1)) * kStride + 8 * c;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = from[e];
      return part_of(v, which);
    }
  };
  // Where the workgroup's columns are of both projections its waves may go different ways below: h is summed, and the
  // waves meet, before they part. Elsewhere all of them see the same bank and rows and meet inside one branch.
  const bool border = col0 < a.t.r0 && col0 + 64 * WR > a.t.r0;
  if (border) sum_h();
  const bool one = named == 0 || __ballot(id >= 0 && id != __builtin_amdgcn_readlane(id, __builtin_ctz(named | 0x10000u))) == 0;
  auto both = [&](auto adapters, auto few) {
    Expand<WR, decltype(adapters)::value, decltype(few)::value> ex(bk, n, at, id, named);
    sum_parts();
    if (!border) sum_h();
    ex.add(acc, operand);
  };
  const std::integral_constant<int, 1> single;
  const std::integral_constant<int, 4> several;
  if (named == 0) {
    sum_parts();
    if (!border) sum_h();
  } else if (bk.rank <= 16) {
    if (one) both(single, std::true_type());
    else both(several, std::true_type());
  } else {
    if (one) both(single, std::false_type());
    else both(several, std::false_type());
  }
  if (m < a.t.rows && l16 < SUB)
#pragma unroll
    for (int i = 0; i < WR; ++i) store4<bf16_t>((sel ? a.y1 : a.y) + (int64_t)m * n + at + 16 * i + 4 * g, acc[i]);
}

// ------------------------------------------------------------------ plan

enum AdapterTile { kRows32, kRows64, kRows64Deep, kRows96, kRows128, kWide128, kWide160, kTile256, kTile160, kTile128,
                   kTile64, kTile32 };

struct AdapterPlan {
  AdapterTile tile;
  int tr, tm;            // the tile's weight rows and query rows
  int splits;            // contraction ranges; 1 with direct
  bool direct;
  bool done;             // h finished by a launch of its own; else in shares beside the split sums
  int chunk, chunks, sub;
  bool two;              // two of the tile's workgroups fit a CU
  int rcols, rrows;      // columns and rows per workgroup of the second launch (0 with direct)
};

// Ranges for decode row counts, near the rule of the decode-row projections: at 33-64 rows the ranges whose wide tiles
// make the most workgroups when some do, otherwise the most that keep n / 32 x ranges workgroups within 256.
static int decode_splits(int rows, int k, int n) {
  int best = 0;
  int64_t most = 0;
  for (int s = 1; s <= 64; ++s) {
    if (k % (64 * s)) continue;
    const int tr = wide_split_tile(rows, k / s, n, s);
    if (tr && (int64_t)(n / tr) * s >= most) {
      most = (int64_t)(n / tr) * s;
      best = s;
    }
  }
  if (best) return best;
  best = 1;
  for (int s = 1; s <= 64; ++s)
    if (k % (64 * s) == 0 && (int64_t)(n / 32) * s <= 256) best = s;
  // up to 32 rows two workgroups share a CU: a few more ranges where a quarter of the CUs would have none (8192 -> 5120,
  // 160 tiles, 2 rows: two ranges 28.8 us, one 38.4; but 5120 -> 1280 at 8 rows: five ranges 17.9, ten 20.2)
  for (int s = best + 1; rows <= 32 && s <= 64 && (int64_t)(n / 32) * best < 192 && (int64_t)(n / 32) * s <= 512; ++s)
    if (k % (64 * s) == 0) best = s;
  return best;
}

// n0: weight rows of the first of two projections (n of one).
static AdapterPlan adapter_plan(int rows, int k, int n, int n0, int rank) {
  AdapterPlan p;
  p.splits = 1;
  p.direct = p.done = false;
  // up to 64 rows, and up to 128 of narrow projections, tiles of few weight rows that stream the weight; wide ones at 65
  // to 128 rows take the prompts' tiles (90 rows 1280 -> 32768: 29 against 51 us, 8192 -> 5120: 47 against 56)
  if (rows <= 64 || (rows <= 128 && n <= 4096)) {
    p.splits = decode_splits(rows, k, n);
    const int wide = wide_split_tile(rows, k / p.splits, n, p.splits);
    if (wide && n0 % wide == 0) {
      p.tile = wide == 160 ? kWide160 : kWide128;
      p.tr = wide;
      p.tm = 64;
    } else {
      const int q = (rows + 31) / 32;
      p.tile = q == 1 ? kRows32 : q == 2 ? ((int64_t)(n / 32) * p.splits > 256 ? kRows64 : kRows64Deep) : q == 3 ? kRows96 : kRows128;
      p.tr = 32;
      p.tm = 32 * q;
    }
    p.two = p.tile == kRows32 || p.tile == kRows64;      // 68 and 76 KB of LDS
    // partial h: one share per CU, of 512 to 1024 channels (4 to 8 steps of each wave)
    p.sub = 4;
    const int64_t tiles = (int64_t)((rows + 3) / 4) * ((rank + 15) / 16);
    const int64_t chunk = ((int64_t)k * tiles / 256 + 127) / 128 * 128;
    p.chunk = (int)(chunk < 512 ? 512 : chunk > 1024 ? 1024 : chunk);
  } else {
    p.sub = 16;
    // The shape and ranges whose estimate is the least. A tile's time is fixed us (prologue, first loads, epilogue) and
    // us per 64-channel step, alone on its CU or as one of two; measured on 4096 rows of 1280 -> 32768 (20 steps), 8192
    // of 8192 -> 5120 (128) and single tiles of 5120 channels (80).
    struct Shape {
      AdapterTile tile;
      int tr, tm;
      double fixed, alone, paired;     // paired 0: one per CU
      bool split;
    };
    static const Shape shapes[] = {{kTile256, 256, 256, 20.0, 1.30, 0.0, false},
                                   {kTile160, 160, 128, 8.0, 0.80, 1.29, true},
                                   {kTile128, 128, 128, 7.6, 0.71, 1.04, true},
                                   {kTile64, 64, 128, 4.3, 0.51, 0.67, true},
                                   {kTile32, 32, 128, 4.0, 0.45, 0.55, true}};
    double best = 1e30;
    for (const Shape& s : shapes) {
      if (n0 % s.tr || n % s.tr) continue;
      const int64_t tiles = (int64_t)(n / s.tr) * ((rows + s.tm - 1) / s.tm);
      for (int splits = 1; splits <= (s.split ? 16 : 1); ++splits) {
        if (k % (64 * splits) || (splits > 1 && tiles * splits > 512)) continue;
        const int64_t t = tiles * splits;
        const double steps = k / 64 / splits;
        const int64_t full = s.paired > 0 ? t / 512 : t / 256, left = t - full * (s.paired > 0 ? 512 : 256);
        double us = full * (s.fixed + steps * (s.paired > 0 ? s.paired : s.alone));
        if (left) us += s.fixed + steps * (left > 256 ? s.paired : s.alone);
        // apart: the finished first product before the tiles, or the parts' way through memory after them
        us += splits == 1 ? 8.0 : 6.0 + (double)rows * n * splits * 8e-6 / 4.5;
        if (us < best) {
          best = us;
          p.tile = s.tile;
          p.tr = s.tr;
          p.tm = s.tm;
          p.splits = splits;
        }
      }
    }
    p.direct = p.splits == 1;
    // h in shares beside split sums while it is few tiles of 16 rows and 16 ranks, in a launch of its own beyond (200 rows
    // 5120 -> 512 at rank 64, 52 tiles: 30 against 39 us; 4,144 rows, 1,036 tiles: 122 against 92)
    const int64_t items = (int64_t)((rows + 15) / 16) * ((rank + 15) / 16);   // rank: both banks'
    p.done = p.direct || items > 128;
    // 32 x 128 on three ring stages: four leave room for one workgroup, whose shares of h delay its tile (200 rows
    // 5120 -> 1280: 30.5 against 26.3 us)
    p.two = p.tile != kTile256;
    // enough shares to fill the chip, at most 8 for the next kernel to sum
    const int parts = (int)((768 + items - 1) / items > 8 ? 8 : (768 + items - 1) / items);
    p.chunk = p.done ? k : ((k + parts - 1) / parts + 127) / 128 * 128;
  }
  p.chunks = (k + p.chunk - 1) / p.chunk;
  // 256 columns per workgroup where that still gives every CU two of them, 64 otherwise; 4 rows where 16 leave CUs
  // without two (28 rows of 512 outputs at rank 64: 12.6 against 21.5 us; 64 rows of 32768 at rank 16: 26.8 against 18.5)
  const int64_t mtiles = (rows + 15) / 16, wide = mtiles * ((n + 255) / 256), narrow = mtiles * ((n + 63) / 64);
  p.rcols = p.direct ? 0 : n0 % 64 == 0 && n % 64 == 0 && wide >= 512 ? 256 : 64;
  p.rrows = p.direct ? 0 : p.rcols == 256 || p.done || p.sub == 16 || narrow >= 512 ? 16 : 4;
  return p;
}

static size_t pad256(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

// h of one bank: three bf16 parts of the finished product, else float32 per chunk of channels
static size_t h_bytes(const AdapterPlan& p, int rows, int rank) {
  return pad256((size_t)rows * rank * (p.done ? 3 * sizeof(bf16_t) : p.chunks * sizeof(float)));
}

static size_t plan_bytes(const AdapterPlan& p, int rows, int n, int rank0, int rank1) {
  const size_t parts = p.direct ? 0 : (size_t)rows * p.splits * n * sizeof(float);
  return pad256(parts) + h_bytes(p, rows, rank0) + h_bytes(p, rows, rank1);
}

template <int WR, int WM, int GR, int GM, int BK, int NS, bool DIRECT>
static void launch_adapter_tiles(const AdapterArgs& a, int64_t tiles, hipStream_t stream) {
  hipLaunchKernelGGL((adapter_tiles_kernel<WR, WM, GR, GM, BK, NS, DIRECT>), dim3((unsigned)tiles), dim3(64 * GR * GM), 0,
                     stream, a);
}

// Rows and ranks per workgroup of the finished first product (one per CU): 32 rows where the fewer rounds are the less,
// each about 1.35 of one of 16 rows (5120 channels at rank 64: 20.1 against 14.7 us, at rank 16 12.5 against 9.6).
static int64_t shrink_blocks(int64_t rows, int tokens, int rank0, int rank1, int mt, int rt) {
  return rows / tokens * ((tokens + 16 * mt - 1) / (16 * mt)) *
         ((rank0 + 16 * rt - 1) / (16 * rt) + (rank1 + 16 * rt - 1) / (16 * rt));
}

static void launch_shrink(const AdapterArgs& a, hipStream_t stream) {
  const int rank0 = a.bank[0].rank, rank1 = a.bank[1].rank, rank = rank0 > rank1 ? rank0 : rank1;
  const int rt = rank <= 16 ? 1 : rank <= 32 ? 2 : 4;
  auto rounds = [&](int mt) { return (double)((shrink_blocks(a.t.rows, a.tokens, rank0, rank1, mt, rt) + 255) / 256); };
  const bool two = 1.35 * rounds(2) < rounds(1);
  auto go = [&](auto kernel, int mt, int waves) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)shrink_blocks(a.t.rows, a.tokens, rank0, rank1, mt, rt)), dim3(64 * waves), 0, stream,
                       a);
  };
  if (rt == 1) two ? go(adapter_shrink_kernel<2, 1, 2>, 2, 4) : go(adapter_shrink_kernel<1, 1, 4>, 1, 4);
  else if (rt == 2) two ? go(adapter_shrink_kernel<2, 2, 1>, 2, 4) : go(adapter_shrink_kernel<1, 2, 2>, 1, 4);
  else two ? go(adapter_shrink_kernel<2, 4, 1>, 2, 8) : go(adapter_shrink_kernel<1, 4, 2>, 1, 8);
}

static void launch_projection(const AdapterArgs& a, const AdapterPlan& p, hipStream_t stream) {
  const int64_t tiles = (int64_t)(a.t.r / p.tr) * ((a.t.rows + p.tm - 1) / p.tm) * p.splits + a.apart;
  switch (p.tile) {
    case kRows32: launch_adapter_tiles<1, 1, 2, 2, 64, 8, false>(a, tiles, stream); break;
    case kRows64: launch_adapter_tiles<1, 2, 2, 2, 64, 6, false>(a, tiles, stream); break;
    case kRows64Deep: launch_adapter_tiles<1, 2, 2, 2, 64, 8, false>(a, tiles, stream); break;
    case kRows96: launch_adapter_tiles<1, 3, 2, 2, 64, 8, false>(a, tiles, stream); break;
    case kRows128: launch_adapter_tiles<1, 4, 2, 2, 64, 4, false>(a, tiles, stream); break;
    case kWide128: launch_adapter_tiles<4, 2, 2, 2, 64, 4, false>(a, tiles, stream); break;
    case kWide160: launch_adapter_tiles<5, 2, 2, 2, 64, 4, false>(a, tiles, stream); break;
    case kTile256: launch_adapter_tiles<8, 4, 2, 4, 64, 2, true>(a, tiles, stream); break;
    case kTile160:
      if (p.direct) launch_adapter_tiles<5, 4, 2, 2, 64, 2, true>(a, tiles, stream);
      else launch_adapter_tiles<5, 4, 2, 2, 64, 2, false>(a, tiles, stream);
      break;
    case kTile128:
      if (p.direct) launch_adapter_tiles<4, 4, 2, 2, 64, 2, true>(a, tiles, stream);
      else launch_adapter_tiles<4, 4, 2, 2, 64, 2, false>(a, tiles, stream);
      break;
    case kTile64:
      if (p.direct) launch_adapter_tiles<2, 4, 2, 2, 64, 3, true>(a, tiles, stream);
      else launch_adapter_tiles<2, 4, 2, 2, 64, 3, false>(a, tiles, stream);
      break;
    case kTile32:
      if (p.direct) launch_adapter_tiles<1, 4, 2, 2, 64, 3, true>(a, tiles, stream);
      else launch_adapter_tiles<1, 4, 2, 2, 64, 3, false>(a, tiles, stream);
      break;
  }
}

}  // namespace dsv41

using namespace dsv41;

extern "C" size_t dsv41_adapter_add_workspace_bytes(int64_t rows, int32_t rank) {
  return rows > 0 && rank > 0 ? (size_t)rows * (size_t)rank * sizeof(float) : 0;
}

template <typename T>
static void launch_add(const void* x, const void* a, const void* b, const float* scale, const int32_t* ids,
                       const void* y, void* out, float* h, int64_t rows, int tokens, int k, int n, int rank, int slots,
                       hipStream_t stream) {
  auto grid = [](int64_t blocks) { return dim3((unsigned)(blocks < kMostBlocks ? blocks : kMostBlocks)); };
  hipLaunchKernelGGL((adapter_shrink_plain_kernel<T>), grid(rows), dim3(256), 0, stream, static_cast<const T*>(x),
                     static_cast<const T*>(a), ids, h, rows, tokens, k, rank, slots);
  hipLaunchKernelGGL((adapter_expand_plain_kernel<T>), grid((rows * n + 255) / 256), dim3(256), 0, stream,
                     static_cast<const T*>(y), static_cast<const T*>(b), scale, ids, h, static_cast<T*>(out), rows,
                     tokens, n, rank, slots);
}

extern "C" int dsv41_adapter_add(const void* x, const void* a, const void* b, const float* scale, const int32_t* ids,
                                 const void* y, void* out, void* workspace, size_t workspace_bytes, int64_t rows,
                                 int32_t tokens, int32_t k, int32_t n, int32_t rank, int32_t slots, int32_t dtype,
                                 hipStream_t stream) {
  const char* what = "dsv41_adapter_add";
  DSV41_REQUIRE(rows >= 0 && tokens > 0 && k > 0 && n > 0 && rank > 0 && slots > 0 && rows % tokens == 0, DSV41_E_ARG,
                "%s: rows %lld, tokens %d, k %d, n %d, rank %d, slots %d", what, (long long)rows, tokens, k, n, rank,
                slots);
  DSV41_REQUIRE(dtype == DSV41_BF16 || dtype == DSV41_F32, DSV41_E_DTYPE, "%s: dtype %d not supported (BF16 or F32)",
                what, dtype);
  DSV41_REQUIRE(rows < (1ll << 31) && rows * n < (1ll << 39), DSV41_E_ARG, "%s: too many outputs", what);
  if (rows == 0) return 0;
  DSV41_REQUIRE(x && a && b && scale && ids && y && out, DSV41_E_ARG, "%s: null tensor", what);
  const size_t need = dsv41_adapter_add_workspace_bytes(rows, rank);
  DSV41_REQUIRE(workspace && workspace_bytes >= need && aligned16(workspace), DSV41_E_WORKSPACE,
                "%s: workspace of %zu bytes needed, %zu given", what, need, workspace_bytes);
  float* h = static_cast<float*>(workspace);
  if (dtype == DSV41_BF16) launch_add<bf16_t>(x, a, b, scale, ids, y, out, h, rows, tokens, k, n, rank, slots, stream);
  else launch_add<float>(x, a, b, scale, ids, y, out, h, rows, tokens, k, n, rank, slots, stream);
  return check_launch(what);
}

// ------------------------------------------------------------------ the projection and its adapters

static bool projection_sizes(int64_t rows, int32_t k, int32_t n0, int32_t n1, int32_t rank0, int32_t rank1) {
  return rows > 0 && rows < (1ll << 30) && k > 0 && k < (1 << 22) && k % 64 == 0 && n0 > 0 && n1 >= 0 && n0 % 32 == 0 && n1 % 32 == 0 &&
         (int64_t)n0 + n1 < (1ll << 30) && rank0 >= 0 && rank1 >= 0 && rank0 <= kMaxRank && rank1 <= kMaxRank &&
         rank0 % 8 == 0 && rank1 % 8 == 0;
}

extern "C" size_t dsv41_adapter_linear_workspace_bytes(int64_t rows, int32_t k, int32_t n0, int32_t n1, int32_t rank0,
                                                       int32_t rank1) {
  if (!projection_sizes(rows, k, n0, n1, rank0, rank1)) return 0;
  return plan_bytes(adapter_plan((int)rows, k, n0 + n1, n0, rank0 + rank1), (int)rows, n0 + n1, rank0, rank1);
}

extern "C" int dsv41_adapter_linear_plan(int64_t rows, int32_t k, int32_t n0, int32_t n1, int32_t rank0, int32_t rank1,
                                         int32_t* plan) {
  const char* what = "dsv41_adapter_linear_plan";
  DSV41_REQUIRE(projection_sizes(rows, k, n0, n1, rank0, rank1) && plan, DSV41_E_ARG,
                "%s: rows %lld, k %d, n %d + %d, rank %d and %d", what, (long long)rows, k, n0, n1, rank0, rank1);
  const AdapterPlan p = adapter_plan((int)rows, k, n0 + n1, n0, rank0 + rank1);
  const int32_t v[] = {p.tr, p.tm, p.splits, p.done, p.two ? 2 : 1, p.rcols, p.rrows};
  for (size_t i = 0; i < sizeof(v) / sizeof(v[0]); ++i) plan[i] = v[i];
  return 0;
}

static int run_adapter_linear(const char* what, const void* x, const void* w0, const void* w1, const Bank* banks,
                              const int32_t* ids, void* y0, void* y1, void* workspace, size_t workspace_bytes,
                              int64_t rows, int32_t tokens, int32_t k, int32_t n0, int32_t n1, int32_t dtype,
                              hipStream_t stream) {
  DSV41_REQUIRE(dtype == DSV41_BF16, DSV41_E_DTYPE, "%s: bf16 only (dtype %d)", what, dtype);
  DSV41_REQUIRE(rows >= 0 && rows < (1ll << 30) && tokens > 0 && rows % tokens == 0 && k > 0 && k < (1 << 22) && n0 > 0 &&
                    n1 >= 0 && (int64_t)n0 + n1 < (1ll << 30),
                DSV41_E_ARG, "%s: rows %lld of %d tokens, k %d, n %d + %d", what, (long long)rows, tokens, k, n0, n1);
  for (int s = 0; s < 2; ++s) {
    const Bank& b = banks[s];
    DSV41_REQUIRE(b.slots >= 0 && (b.slots == 0 || (b.rank > 0 && b.a && b.b && b.scale)), DSV41_E_ARG,
                  "%s: bank %d of %d slots, rank %d", what, s, b.slots, b.rank);
    DSV41_REQUIRE(b.slots == 0 || (b.rank % 8 == 0 && b.rank <= kMaxRank), DSV41_E_SHAPE,
                  "%s: rank %d must be a multiple of 8, at most %d", what, b.rank, kMaxRank);
    DSV41_REQUIRE(b.slots == 0 || (aligned16(b.a) && aligned16(b.b)), DSV41_E_ARG,
                  "%s: adapters must be 16-byte aligned", what);
  }
  DSV41_REQUIRE(k % 64 == 0 && n0 % 32 == 0 && n1 % 32 == 0, DSV41_E_SHAPE,
                "%s: k = %d must be a multiple of 64, n = %d (+ %d) of 32", what, k, n0, n1);
  if (rows == 0) return 0;
  DSV41_REQUIRE(x && w0 && y0 && ids && (n1 == 0 || (w1 && y1)), DSV41_E_ARG, "%s: null tensor", what);
  DSV41_REQUIRE(aligned16(x) && aligned16(w0) && aligned16(y0) && (n1 == 0 || (aligned16(w1) && aligned16(y1))),
                DSV41_E_ARG, "%s: tensors must be 16-byte aligned", what);
  const int rank0 = banks[0].slots ? banks[0].rank : 0, rank1 = banks[1].slots ? banks[1].rank : 0, n = n0 + n1;
  const AdapterPlan p = adapter_plan((int)rows, k, n, n0, rank0 + rank1);
  const int64_t tiles = (int64_t)(n / p.tr) * ((rows + p.tm - 1) / p.tm) * p.splits;
  const int64_t shrinks = p.done ? shrink_blocks(rows, tokens, rank0, rank1, 1, 1)
                                 : (rows + p.sub - 1) / p.sub * p.chunks * ((rank0 + 15) / 16 + (rank1 + 15) / 16);
  const int64_t reduces = (rows + 3) / 4 * ((n + 63) / 64);
  DSV41_REQUIRE(tiles < kMostBlocks && (p.done ? shrinks < kMostBlocks : shrinks < (1ll << 31)) &&
                    (p.direct || reduces < kMostBlocks),
                DSV41_E_ARG, "%s: too many tiles", what);
  const size_t need = plan_bytes(p, (int)rows, n, rank0, rank1);
  DSV41_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned16(workspace))), DSV41_E_WORKSPACE,
                "%s: workspace of %zu bytes needed, %zu given", what, need, workspace_bytes);
  AdapterArgs a;
  a.t = WoaArgs{static_cast<const bf16_t*>(x), static_cast<const bf16_t*>(w0), workspace, (int)rows, p.splits,
                k / p.splits, n, 1, static_cast<const bf16_t*>(n1 ? w1 : nullptr), n0};
  a.bank[0] = banks[0];
  a.bank[1] = banks[1];
  a.bank[0].rank = rank0;
  a.bank[1].rank = rank1;
  uint8_t* at = static_cast<uint8_t*>(workspace) + (p.direct ? 0 : pad256((size_t)rows * p.splits * n * sizeof(float)));
  a.bank[0].h = reinterpret_cast<float*>(at);
  a.bank[1].h = reinterpret_cast<float*>(at + h_bytes(p, (int)rows, rank0));
  a.ids = ids;
  a.tokens = tokens;
  a.k = k;
  a.chunk = p.chunk;
  a.chunks = p.chunks;
  a.sub = p.sub;
  // shares of h on workgroups of their own while all of them and all tiles run at once (a multiple of 8, so that the
  // tiles keep their XCDs): one row 5120 -> 1280 + 512 at rank 16 7.2 against 9.8 us
  const int64_t room = p.two ? 512 : 256, spare = (shrinks + 7) / 8 * 8;
  a.apart = !p.done && tiles + spare <= room ? (int)spare : 0;
  a.done = p.done;
  a.y = static_cast<bf16_t*>(y0);
  a.y1 = static_cast<bf16_t*>(y1);
  if (p.done && shrinks) launch_shrink(a, stream);
  launch_projection(a, p, stream);
  if (!p.direct) {
    auto reduce = [&](auto kernel) {
      const int64_t blocks = (rows + p.rrows - 1) / p.rrows * ((n + p.rcols - 1) / p.rcols);
      hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a);
    };
    if (p.rcols == 256) p.done ? reduce(adapter_reduce_kernel<4, true, 16>) : reduce(adapter_reduce_kernel<4, false, 16>);
    else if (p.done) reduce(adapter_reduce_kernel<1, true, 16>);
    else if (p.rrows == 16) reduce(adapter_reduce_kernel<1, false, 16>);
    else reduce(adapter_reduce_kernel<1, false, 4>);
  }
  return check_launch(what);
}

template <typename T, bool VEC>
static void launch_plain(const void* x, const void* w, const void* a, const void* b, const float* scale,
                         const int32_t* ids, void* y, int rows, int tokens, int k, int n, int rank, int slots,
                         hipStream_t stream) {
  // 64 columns per wave where that still gives every SIMD a wave; a workgroup per tile up to one per CU
  // (1024 rows 64 -> 256, 1,024 tiles: 7.0 against 5.3 us)
  const int64_t mtiles = (rows + 15) / 16, wide = mtiles * ((n + 63) / 64), narrow = mtiles * ((n + 15) / 16);
  auto go = [&](auto kernel, int64_t blocks, size_t lds) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), lds, stream, static_cast<const T*>(x),
                       static_cast<const T*>(w), static_cast<const T*>(a), static_cast<const T*>(b), scale, ids,
                       static_cast<T*>(y), rows, tokens, k, n, rank, slots);
  };
  if (wide >= 1024) go(adapter_plain_kernel<T, 4, VEC>, (wide + 3) / 4, 0);
  else if (narrow <= 256 && rank <= kMaxRank)
    go(adapter_plain_split_kernel<T, VEC>, narrow, (4 * 16 * ((size_t)(rank + 15) / 16 * 16 + 4) + 4 * 256) * sizeof(float));
  else go(adapter_plain_kernel<T, 1, VEC>, (narrow + 3) / 4, 0);
}

extern "C" int dsv41_adapter_plain(const void* x, const void* w, const void* a, const void* b, const float* scale,
                                   const int32_t* ids, void* y, int64_t rows, int32_t tokens, int32_t k, int32_t n,
                                   int32_t rank, int32_t slots, int32_t dtype, hipStream_t stream) {
  const char* what = "dsv41_adapter_plain";
  DSV41_REQUIRE(rows >= 0 && tokens > 0 && k > 0 && n > 0 && rank > 0 && slots > 0 && rows % tokens == 0, DSV41_E_ARG,
                "%s: rows %lld, tokens %d, k %d, n %d, rank %d, slots %d", what, (long long)rows, tokens, k, n, rank,
                slots);
  DSV41_REQUIRE(dtype == DSV41_BF16 || dtype == DSV41_F32, DSV41_E_DTYPE, "%s: dtype %d not supported (BF16 or F32)",
                what, dtype);
  DSV41_REQUIRE(rows < (1ll << 30) && k < (1 << 30) && n < (1 << 30) && rank < (1 << 30) &&
                    (rows + 15) / 16 * ((n + 63) / 64) < 4 * kMostBlocks,
                DSV41_E_ARG, "%s: too many outputs", what);
  if (rows == 0) return 0;
  DSV41_REQUIRE(x && w && a && b && scale && ids && y, DSV41_E_ARG, "%s: null tensor", what);
  const int m = (int)rows;
  const bool vec = k % 16 == 0 && rank % 4 == 0 && aligned16(x) && aligned16(w) && aligned16(a) && aligned16(b);
  if (dtype == DSV41_BF16) {
    if (vec) launch_plain<bf16_t, true>(x, w, a, b, scale, ids, y, m, tokens, k, n, rank, slots, stream);
    else launch_plain<bf16_t, false>(x, w, a, b, scale, ids, y, m, tokens, k, n, rank, slots, stream);
  } else {
    if (vec) launch_plain<float, true>(x, w, a, b, scale, ids, y, m, tokens, k, n, rank, slots, stream);
    else launch_plain<float, false>(x, w, a, b, scale, ids, y, m, tokens, k, n, rank, slots, stream);
  }
  return check_launch(what);
}

extern "C" int dsv41_adapter_linear(const void* x, const void* w, const void* a, const void* b, const float* scale,
                                    const int32_t* ids, void* y, void* workspace, size_t workspace_bytes, int64_t rows,
                                    int32_t tokens, int32_t k, int32_t n, int32_t rank, int32_t slots, int32_t dtype,
                                    hipStream_t stream) {
  const char* what = "dsv41_adapter_linear";
  DSV41_REQUIRE(slots > 0, DSV41_E_ARG, "%s: %d slots", what, slots);
  const Bank banks[2] = {{static_cast<const bf16_t*>(a), static_cast<const bf16_t*>(b), scale, nullptr, rank, slots}, {}};
  return run_adapter_linear(what, x, w, nullptr, banks, ids, y, nullptr, workspace, workspace_bytes, rows, tokens, k, n, 0,
                            dtype, stream);
}

extern "C" int dsv41_adapter_linear_pair(const void* x, const void* w0, const void* w1, const void* a0, const void* b0,
                                         const float* scale0, const void* a1, const void* b1, const float* scale1,
                                         const int32_t* ids, void* y0, void* y1, void* workspace, size_t workspace_bytes,
                                         int64_t rows, int32_t tokens, int32_t k, int32_t n0, int32_t n1, int32_t rank0,
                                         int32_t rank1, int32_t slots0, int32_t slots1, int32_t dtype,
                                         hipStream_t stream) {
  const char* what = "dsv41_adapter_linear_pair";
  DSV41_REQUIRE(n1 > 0, DSV41_E_ARG, "%s: the second weight is missing", what);
  DSV41_REQUIRE(slots0 > 0 || slots1 > 0, DSV41_E_ARG, "%s: %d and %d slots", what, slots0, slots1);
  const Bank banks[2] = {{static_cast<const bf16_t*>(a0), static_cast<const bf16_t*>(b0), scale0, nullptr, rank0, slots0},
                         {static_cast<const bf16_t*>(a1), static_cast<const bf16_t*>(b1), scale1, nullptr, rank1, slots1}};
  return run_adapter_linear(what, x, w0, w1, banks, ids, y0, y1, workspace, workspace_bytes, rows, tokens, k, n0, n1, dtype,
                            stream);
}
