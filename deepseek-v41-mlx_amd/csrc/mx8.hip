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
  float v[8];
  load8(x + 8 * i, v);
  uint32_t m = 0u;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, abs_bits(v[e]));
  float inv;
  const uint32_t byte = mx8_scale(group_max_u(m, 4), inv);
  *reinterpret_cast<uint2*>(codes + 8 * i) = make_uint2(mx8_codes(v, inv, byte), mx8_codes(v + 4, inv, byte));
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
  float v[16][8];
  uint32_t m = 0u;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    if (in && r0 + 2 * j < n) {
      load8(w + (r0 + 2 * j) * k + c, v[j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) m = max(m, abs_bits(v[j][e]));
    }
  }
  m = max(group_max_u(m, 4), (uint32_t)__shfl_xor((int)group_max_u(m, 4), 32, 64));
  float inv;
  const uint32_t byte = mx8_scale(m, inv);
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (in && r0 + 2 * j < n)
      *reinterpret_cast<uint2*>(codes + (r0 + 2 * j) * k + c) =
          make_uint2(mx8_codes(v[j], inv, byte), mx8_codes(v[j] + 4, inv, byte));
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
  store8(x + 8 * i, v);
}

// ------------------------------------------------------------------ norm

// One workgroup per row, C eights of it in each thread's registers: the residual addition first (x <- cast(x + delta),
// stored back), the norm of the rounded sum with float32 statistics, the normed row rounded to its type -- what the
// separate operators store between them and what every other reader of the row gets -- and that row's blocks in 8 bits.
// Bound by memory: every tensor crosses the bus once.
template <typename T, int C, bool ADD, bool KEEP>
__global__ __launch_bounds__(256) void rmsnorm_mx8_kernel(T* x, const T* delta, const float* w, T* y, uint8_t* codes,
                                                          uint8_t* scales, int dim, float eps) {
  __shared__ float red[4];
  const int64_t row = blockIdx.x;
  const int eights = dim / 8;
  float v[C][8];
  float ss = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int ch = threadIdx.x + 256 * c;
    if (ch < eights) {
      load8(x + row * dim + 8 * ch, v[c]);
      if constexpr (ADD) {
        float d[8];
        load8(delta + row * dim + 8 * ch, d);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[c][i] = io<T>::rnd(v[c][i] + d[i]);
        store8(x + row * dim + 8 * ch, v[c]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += v[c][i] * v[c][i];
    }
  }
  ss = group_sum(ss, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = ss;
  __syncthreads();
  const float tot = (red[0] + red[1]) + (red[2] + red[3]);
  const float inv = 1.0f / sqrtf(tot / (float)dim + eps);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int ch = threadIdx.x + 256 * c;
    if (ch < eights) {                     // dim is a multiple of 32: a block's four lanes are here or not
      float g[8];
      load8(w + 8 * ch, g);
      uint32_t m = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[c][i] = io<T>::rnd(g[i] * (v[c][i] * inv));
        m = max(m, abs_bits(v[c][i]));
      }
      if constexpr (KEEP) store8(y + row * dim + 8 * ch, v[c]);
      float s;
      const uint32_t byte = mx8_scale(group_max_u(m, 4), s);
      *reinterpret_cast<uint2*>(codes + row * dim + 8 * ch) =
          make_uint2(mx8_codes(v[c], s, byte), mx8_codes(v[c] + 4, s, byte));
      if ((ch & 3) == 0) scales[row * (dim / 32) + (ch >> 2)] = (uint8_t)byte;
    }
  }
}

constexpr int kNormDim = 16384;            // the widest row: eight eights per thread

template <typename T, bool ADD, bool KEEP>
static void launch_norm(void* x, const void* delta, const float* w, void* y, uint8_t* codes, uint8_t* scales,
                        int64_t rows, int dim, float eps, hipStream_t stream) {
  const dim3 grid((unsigned)rows), block(256);
  T* xt = static_cast<T*>(x);
  const T* dt = static_cast<const T*>(delta);
  T* yt = static_cast<T*>(y);
#define DSV41_NORM(C) \
  hipLaunchKernelGGL((rmsnorm_mx8_kernel<T, C, ADD, KEEP>), grid, block, 0, stream, xt, dt, w, yt, codes, scales, dim, eps)
  const int per = (dim / 8 + 255) / 256;
  if (per == 1) DSV41_NORM(1);
  else if (per == 2) DSV41_NORM(2);
  else if (per == 3) DSV41_NORM(3);
  else if (per == 4) DSV41_NORM(4);
  else DSV41_NORM(8);
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
