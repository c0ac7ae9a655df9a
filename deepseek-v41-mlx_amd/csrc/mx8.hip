// Quantization to 8 bits with block scales and back, and the RMS norm that ends in it (mx8.h has the format).
#include "mx8.h"

namespace dsv41 {

// ------------------------------------------------------------------ rows

// Rows of whole 32-channel blocks are one run of blocks: a thread takes 8 values, four neighbouring lanes a block. Bound by
// memory: (size + 33/32) bytes a value.
template <typename T>
__global__ __launch_bounds__(256) void quant_rows_kernel(const T* x, uint8_t* codes, uint8_t* scales, int64_t blocks) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;      // over the eights of all blocks
  if (i >= blocks * 4) return;                                    // whole groups of four leave together
  Eight<T> e;
  e.load(x + 8 * i);
  float v[8], inv;
  e.get(v);
  const uint32_t byte = mx8_scale(group_max_u(e.top(), 4), inv);
  put_codes8(codes + 8 * i, v, inv, byte);
  if ((threadIdx.x & 3) == 0) scales[i >> 2] = (uint8_t)byte;
}

// ------------------------------------------------------------------ weights

// A wave takes 32 rows x 256 channels, two rows per load (512 bytes of each); a block's maximum is over the 16 loads of four
// lanes of each half. Everything stays in registers, so the weight is read once.
template <typename T>
__global__ __launch_bounds__(256) void quant_blocks_kernel(const T* w, uint8_t* codes, uint8_t* scales, int64_t n, int k) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int strips = (k + 255) / 256;
  const int64_t unit = (int64_t)blockIdx.x * 4 + wave;
  const int64_t r0 = unit / strips * 32 + (lane >> 5);
  const int c = (int)(unit % strips) * 256 + (lane & 31) * 8;
  if (unit / strips * 32 >= n) return;                            // whole waves
  const bool in = c < k;                                          // whole blocks: k is a multiple of 32
  // rows past the end (and lanes past the row) read the last of theirs again: no load waits behind a branch
  const int64_t last = n - 1;
  const T* const from = w + (in ? c : k - 8);
  Eight<T> v[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j].load(from + min(r0 + 2 * j, last) * k);
  uint32_t m = 0u;
#pragma unroll
  for (int j = 0; j < 16; ++j) m = max(m, v[j].top());
  m = group_max_u(m, 4);
  m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
  float inv;
  const uint32_t byte = mx8_scale(m, inv);
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    float f[8];
    v[j].get(f);
    if (in && r0 + 2 * j < n) put_codes8(codes + (r0 + 2 * j) * k + c, f, inv, byte);
  }
  if (in && (lane & 35) == 0) scales[r0 / 32 * (k / 32) + c / 32] = (uint8_t)byte;
}

// ------------------------------------------------------------------ back

// codes times their scale, exact in float32 and (but for magnitudes under 2^-126) in bf16. A scale covers 32 channels of
// 1 << shift rows. Eight values per thread.
template <typename T>
__global__ __launch_bounds__(256) void dequant_kernel(const uint8_t* codes, const uint8_t* scales, T* x, int64_t eights,
                                                      int k, int shift) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= eights) return;
  const uint2 c = *reinterpret_cast<const uint2*>(codes + 8 * i);
  int64_t at = i >> 2;                                            // one scale per block of a row
  if (shift) {
    const int64_t row = i / (k / 8);
    at = (row >> shift) * (k / 32) + ((i - row * (k / 8)) >> 2);
  }
  const float s = e8m0_to_float(scales[at]);
  typedef __attribute__((ext_vector_type(2))) float f2;
  const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8(c.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(c.x, true);
  const f2 d = __builtin_amdgcn_cvt_pk_f32_fp8(c.y, false), e = __builtin_amdgcn_cvt_pk_f32_fp8(c.y, true);
  const float v[8] = {a[0] * s, a[1] * s, b[0] * s, b[1] * s, d[0] * s, d[1] * s, e[0] * s, e[1] * s};
  Eight<T> out;
  out.round(v);
  out.store_past(x + 8 * i);
}

// ------------------------------------------------------------------ norm

// The sum over a wave's lanes.
__device__ __forceinline__ double wave_total(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// 1 / sqrt(m): the hardware's estimate and one Newton step, which leaves some 2^-50. m = 0 and infinity keep the estimate.
__device__ __forceinline__ double inverse_root(double m) {
  const double r = __builtin_amdgcn_rsq(m);
  return r > 0.0 && r < (double)INFINITY ? r * (1.5 - 0.5 * m * r * r) : r;
}

// v[i] = g[i] v[i] inv to within 1/2 + 2^-20 of float32's step, where inv = hi + lo: the products with their rounding errors, whose
// own roundings come to some 2^-44. Errors that are no numbers, or zero, are not added: infinities and a zero's sign stay.
__device__ __forceinline__ void scale_exactly(float* v, const float* g, float hi, float lo) {
#pragma clang fp contract(off)
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float p = v[i] * hi, pe = __builtin_fmaf(v[i], hi, -p) + v[i] * lo;
    const float q = g[i] * p, qe = __builtin_fmaf(g[i], p, -q) + g[i] * pe;
    v[i] = __builtin_amdgcn_classf(qe, 0x198) ? q + qe : q;        // normal or subnormal
  }
}

// The same as far as T tells: for bf16 the plain products, unless one of the eight lies within 4 float32 steps of the middle
// between two bf16 values (they are 3 off at most). About one wave in ten takes the long way.
template <typename T>
__device__ __forceinline__ void scale_rows(float* v, const float* g, float hi, float lo) {
  if constexpr (sizeof(T) == 2) {
    float q[8];
    uint32_t near = 0xFFFFu;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      q[i] = g[i] * (v[i] * hi);
      near = min(near, (__float_as_uint(q[i]) - 0x7FFCu) & 0xFFFFu);
    }
    if (near > 8u) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = q[i];
      return;
    }
  }
  scale_exactly(v, g, hi, lo);
}

// The residual addition first (x <- cast(x + delta), stored back), the norm of the rounded sum, the normed row rounded to its
// type -- what every other reader of the row gets -- and that row's blocks in 8 bits. Everything between stays in registers, so
// every tensor crosses the bus once. A value in 8 bits has steps of an eighth: a normed value that is rounded to the other side
// of a border is a whole step off. So the squares are summed in float64 and the products carried past float32 where it
// matters: bf16 rows are the formula's values rounded (through float32), whatever the order of the sum. In float32 one value
// in a few million came out a step of 8 bits off. It costs 32,768 rows of 1,280 alone 26.6 -> 30.0 us, 8,192 rows of 8,192 with the
// addition and the row kept 115.6 -> 116.9, one row of 5,120 3.4 -> 3.6.
// Thread t holds eights t, t + 256 .. of a row, C of them. WAVE: one wave takes the row (dim at most 2,048), its lanes four
// times 64 eights, without a barrier.
template <typename T, int C, bool ADD, bool KEEP, bool WAVE>
__global__ __launch_bounds__(256) void rmsnorm_mx8_kernel(T* x, const T* delta, const float* w, T* y, uint8_t* codes,
                                                          uint8_t* scales, int64_t rows, int dim, float eps) {
  constexpr int SPAN = WAVE ? 64 : 256;
  __shared__ double red[4];
  const int64_t row = WAVE ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (WAVE && row >= rows) return;         // whole waves, which wait for nobody
  const int t = WAVE ? threadIdx.x & 63 : threadIdx.x, eights = dim / 8;
  Eight<T> e[C];
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (t + SPAN * c < eights) e[c].load(x + row * dim + 8 * (t + SPAN * c));
  double ss = 0.0;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (t + SPAN * c < eights) {
      float v[8];
      e[c].get(v);
      if constexpr (ADD) {
        float d[8];
        load8(delta + row * dim + 8 * (t + SPAN * c), d);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] + d[i];
        e[c].round(v);
        e[c].get(v);
        e[c].store_past(x + row * dim + 8 * (t + SPAN * c));
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = __builtin_fma((double)v[i], (double)v[i], ss);
    }
  }
  ss = wave_total(ss);
  if constexpr (!WAVE) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = ss;
    __syncthreads();
    ss = (red[0] + red[1]) + (red[2] + red[3]);
  }
  const double inv = inverse_root(ss / dim + (double)eps);
  const float hi = (float)inv, lo = (float)(inv - (double)hi);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int ch = t + SPAN * c;
    if (ch < eights) {                     // dim is a multiple of 32: a block's four lanes are here or not
      float g[8], v[8], s;
      load8(w + 8 * ch, g);
      e[c].get(v);
      scale_rows<T>(v, g, hi, lo);
      e[c].round(v);
      e[c].get(v);
      if constexpr (KEEP) e[c].store_past(y + row * dim + 8 * ch);
      const uint32_t byte = mx8_scale(group_max_u(e[c].top(), 4), s);
      put_codes8(codes + row * dim + 8 * ch, v, s, byte);
      if ((ch & 3) == 0) scales[row * (dim / 32) + (ch >> 2)] = (uint8_t)byte;
    }
  }
}

constexpr int kNormDim = 16384;            // the widest row: eight eights per thread

// A wave per row where the row fits and rows are many; for a few the row's eights side by side in four waves are quicker.
constexpr int64_t kWaveRows = 1024;

template <typename T, bool ADD, bool KEEP>
static void launch_norm(void* x, const void* delta, const float* w, void* y, uint8_t* codes, uint8_t* scales,
                        int64_t rows, int dim, float eps, hipStream_t stream) {
  T* xt = static_cast<T*>(x);
  const T* dt = static_cast<const T*>(delta);
  T* yt = static_cast<T*>(y);
#define DSV41_NORM(C, WAVE)                                                                                             \
  hipLaunchKernelGGL((rmsnorm_mx8_kernel<T, C, ADD, KEEP, WAVE>), dim3((unsigned)(WAVE ? (rows + 3) / 4 : rows)), dim3(256), 0, \
                     stream, xt, dt, w, yt, codes, scales, rows, dim, eps)
  const int eights = dim / 8, per = (eights + 255) / 256;
  if (per == 1 && rows >= kWaveRows) {
    if (eights <= 64) DSV41_NORM(1, true);
    else if (eights <= 128) DSV41_NORM(2, true);
    else if (eights <= 192) DSV41_NORM(3, true);
    else DSV41_NORM(4, true);
  } else if (per == 1) DSV41_NORM(1, false);
  else if (per == 2) DSV41_NORM(2, false);
  else if (per == 3) DSV41_NORM(3, false);
  else if (per == 4) DSV41_NORM(4, false);
  else DSV41_NORM(8, false);
#undef DSV41_NORM
}

template <typename T>
static void launch_norm_any(void* x, const void* delta, const float* w, void* y, uint8_t* codes, uint8_t* scales,
                            int64_t rows, int dim, float eps, hipStream_t stream) {
  if (delta && y) launch_norm<T, true, true>(x, delta, w, y, codes, scales, rows, dim, eps, stream);
  else if (delta) launch_norm<T, true, false>(x, delta, w, y, codes, scales, rows, dim, eps, stream);
  else if (y) launch_norm<T, false, true>(x, delta, w, y, codes, scales, rows, dim, eps, stream);
  else launch_norm<T, false, false>(x, delta, w, y, codes, scales, rows, dim, eps, stream);
}

static int check_mx8(const char* what, const void* x, const void* codes, const void* scales, int64_t rows, int k,
                     int dtype) {
  DSV41_REQUIRE(x && codes && scales, DSV41_E_ARG, "%s: null tensor", what);
  DSV41_REQUIRE(dtype == DSV41_F32 || dtype == DSV41_BF16, DSV41_E_DTYPE, "%s: dtype %d not supported", what, dtype);
  DSV41_REQUIRE(rows >= 0 && k > 0 && k % 32 == 0, DSV41_E_SHAPE, "%s: rows %lld, k %d: whole blocks of 32 channels needed",
                what, (long long)rows, k);
  DSV41_REQUIRE(rows <= (1ll << 34) / k, DSV41_E_SHAPE, "%s: %lld rows of %d are over 2^34 values", what, (long long)rows, k);
  DSV41_REQUIRE(aligned16(x) && aligned16(codes), DSV41_E_ARG, "%s: tensors must be 16-byte aligned", what);
  return 0;
}

}  // namespace dsv41

using namespace dsv41;

extern "C" int dsv41_quant_mx8(const void* x, uint8_t* codes, uint8_t* scales, int64_t rows, int32_t k, int32_t dtype,
                               hipStream_t stream) {
  const char* what = "dsv41_quant_mx8";
  const int rc = check_mx8(what, x, codes, scales, rows, k, dtype);
  if (rc || rows == 0) return rc;
  const int64_t blocks = rows * (k / 32);
  const dim3 grid((unsigned)((blocks * 4 + 255) / 256));
  if (dtype == DSV41_F32)
    hipLaunchKernelGGL(quant_rows_kernel<float>, grid, dim3(256), 0, stream, (const float*)x, codes, scales, blocks);
  else
    hipLaunchKernelGGL(quant_rows_kernel<bf16_t>, grid, dim3(256), 0, stream, (const bf16_t*)x, codes, scales, blocks);
  return check_launch(what);
}

extern "C" int dsv41_quant_mx8_blocks(const void* w, uint8_t* codes, uint8_t* scales, int64_t n, int32_t k,
                                      int32_t dtype, hipStream_t stream) {
  const char* what = "dsv41_quant_mx8_blocks";
  const int rc = check_mx8(what, w, codes, scales, n, k, dtype);
  if (rc || n == 0) return rc;
  const int64_t waves = (n + 31) / 32 * ((k + 255) / 256);
  const dim3 grid((unsigned)((waves + 3) / 4));
  if (dtype == DSV41_F32)
    hipLaunchKernelGGL(quant_blocks_kernel<float>, grid, dim3(256), 0, stream, (const float*)w, codes, scales, n, k);
  else
    hipLaunchKernelGGL(quant_blocks_kernel<bf16_t>, grid, dim3(256), 0, stream, (const bf16_t*)w, codes, scales, n, k);
  return check_launch(what);
}

extern "C" int dsv41_dequant_mx8(const uint8_t* codes, const uint8_t* scales, void* x, int64_t rows, int32_t k,
                                 int32_t scale_rows, int32_t dtype, hipStream_t stream) {
  const char* what = "dsv41_dequant_mx8";
  const int rc = check_mx8(what, x, codes, scales, rows, k, dtype);
  if (rc) return rc;
  DSV41_REQUIRE(scale_rows == 1 || scale_rows == 32, DSV41_E_SHAPE, "%s: a scale covers 1 or 32 rows, not %d", what,
                scale_rows);
  if (rows == 0) return 0;
  const int64_t eights = rows * (k / 8);
  const dim3 grid((unsigned)((eights + 255) / 256));
  const int shift = scale_rows == 32 ? 5 : 0;
  if (dtype == DSV41_F32)
    hipLaunchKernelGGL(dequant_kernel<float>, grid, dim3(256), 0, stream, codes, scales, (float*)x, eights, k, shift);
  else
    hipLaunchKernelGGL(dequant_kernel<bf16_t>, grid, dim3(256), 0, stream, codes, scales, (bf16_t*)x, eights, k, shift);
  return check_launch(what);
}

extern "C" int dsv41_rmsnorm_mx8(void* x, const void* delta, const float* weight, void* y, uint8_t* codes,
                                 uint8_t* scales, int64_t rows, int32_t dim, float eps, int32_t dtype,
                                 hipStream_t stream) {
  const char* what = "dsv41_rmsnorm_mx8";
  const int rc = check_mx8(what, x, codes, scales, rows, dim, dtype);
  if (rc) return rc;
  DSV41_REQUIRE(weight, DSV41_E_ARG, "%s: null weight", what);
  DSV41_REQUIRE(dim <= kNormDim && rows < (1ll << 24), DSV41_E_SHAPE, "%s: %lld rows (under 2^24) of %d (at most %d)",
                what, (long long)rows, dim, kNormDim);
  DSV41_REQUIRE(aligned16(weight) && (!delta || aligned16(delta)) && (!y || aligned16(y)), DSV41_E_ARG,
                "%s: tensors must be 16-byte aligned", what);
  if (rows == 0) return 0;
  if (dtype == DSV41_F32) launch_norm_any<float>(x, delta, weight, y, codes, scales, rows, dim, eps, stream);
  else launch_norm_any<bf16_t>(x, delta, weight, y, codes, scales, rows, dim, eps, stream);
  return check_launch(what);
}
