// Rows and weights in 8 bits: e4m3fn codes with one power-of-two scale byte (ue8m0, 2^(byte - 127)) per block of 32 channels
// of a row, or per 32 x 32 block of a weight -- the form the release stores its projections in and quantizes their inputs
// to (docs/reference/kernel.py:40-124 with round_scale; deepseek_v41_mlx/fakequant.py:83-93).
#pragma once

#include "mfma.h"

namespace dsv41 {

// |v| as bits: ordered as the magnitudes are, infinity above every number and NaN above infinity, so that a block's
// maximum also says whether all of it is finite.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

constexpr uint32_t kNotFinite = 0x7F800000u;

// The scale of a block whose largest magnitude has these bits: the smallest power of two s with max(amax, 1e-4) <= 448 s
// (act_quant's formula; its product with 1/448, rounded to float32, is above a power of two exactly where the quotient
// is). The byte, and 1 / s. A block that holds an infinity or NaN has the byte 255 (NaN).
__device__ __forceinline__ uint32_t mx8_scale(uint32_t amax_bits, float& inv) {
  const float s = pow2_ceil_log2(fmaxf(__uint_as_float(amax_bits), 1e-4f) * (float)(1.0 / 448.0));
  inv = pow2_inverse(s);
  return amax_bits >= kNotFinite ? 255u : __float_as_uint(s) >> 23;
}

// Four values of a block as codes, ties to even (v_cvt_pk_fp8_f32: nothing exceeds 448, so nothing is cut off). v / s is
// exact as v * (1 / s). Codes under the byte 255 are NaN too.
__device__ __forceinline__ uint32_t mx8_codes(const float* v, float inv, uint32_t byte) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, w, true);
  return byte == 255u ? 0x7F7F7F7Fu : (uint32_t)w;
}

// Largest of a value over an aligned group of `width` lanes.
__device__ __forceinline__ uint32_t group_max_u(uint32_t v, int width) {
  for (int o = width >> 1; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
  return v;
}

// Loads and stores of data that this launch does not meet again, which the L2 need not keep. What large calls write then leaves
// the L2 to what they read: 8,192 rows of 5,120 quantized 24.0 -> 20.7 us, read back 24.8 -> 19.8.
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2_once;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_once;
template <typename V>
__device__ __forceinline__ V past_l2(const void* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
}
template <typename V>
__device__ __forceinline__ void past_l2(void* p, V v) {
  __builtin_nontemporal_store(v, reinterpret_cast<V*>(p));
}

// Eight consecutive values of a row as they lie in memory. Rounding, maxima and widening work on pairs of bf16 as they are
// (one instruction for two values instead of six for each: norm over 8,192 rows of 5,120 34.5 -> 29.9 us).
template <typename T> struct Eight;
template <> struct Eight<bf16_t> {
  uint4 u;
  __device__ __forceinline__ void load(const bf16_t* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void load_past(const bf16_t* p) { u = __builtin_bit_cast(uint4, past_l2<u32x4_once>(p)); }
  __device__ __forceinline__ void store_past(bf16_t* p) const { past_l2(p, __builtin_bit_cast(u32x4_once, u)); }
  __device__ __forceinline__ void get(float* v) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  __device__ __forceinline__ void round(const float* v) {
    u = make_uint4(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]), pack2_bf16(v[4], v[5]), pack2_bf16(v[6], v[7]));
  }
  // the largest magnitude, as abs_bits of the float
  __device__ __forceinline__ uint32_t top() const {
    typedef __attribute__((ext_vector_type(2))) uint16_t u16x2;
    auto mag = [](uint32_t w) { return __builtin_bit_cast(u16x2, w & 0x7FFF7FFFu); };
    const u16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(mag(u.x), mag(u.y)),
                                              __builtin_elementwise_max(mag(u.z), mag(u.w)));
    return (uint32_t)max(m[0], m[1]) << 16;
  }
};
template <> struct Eight<float> {
  f32x4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
  }
  __device__ __forceinline__ void store_past(float* p) const { past_l2(p, a), past_l2(p + 4, b); }
  __device__ __forceinline__ void get(float* v) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
  }
  __device__ __forceinline__ void round(const float* v) { a = f32x4{v[0], v[1], v[2], v[3]}, b = f32x4{v[4], v[5], v[6], v[7]}; }
  __device__ __forceinline__ uint32_t top() const {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, max(abs_bits(a[i]), abs_bits(b[i])));
    return m;
  }
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* v) {
  Eight<T> e;
  e.load(p);
  e.get(v);
}
// Eight values of a block as codes, to p.
__device__ __forceinline__ void put_codes8(uint8_t* p, const float* v, float inv, uint32_t byte) {
  past_l2(p, u32x2_once{mx8_codes(v, inv, byte), mx8_codes(v + 4, inv, byte)});
}

}  // namespace dsv41
