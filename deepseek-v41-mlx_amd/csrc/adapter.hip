// Low-rank adapters of many sequences beside one shared projection. Row m belongs to sequence m / tokens, whose
// adapter is t = ids[m / tokens]; for t in [0, slots)
//
//   h[m, :] = x[m, :] A_t^T                       A_t [rank, k]
//   y[m, :] = x[m, :] w^T + scale_t (h[m, :] B_t^T)      B_t [n, rank]
//
// and y[m, :] = x[m, :] w^T for any other t, whatever the adapters hold. h and all sums are float32, y is rounded
// once.
#include "tiles.h"

namespace dsv41 {

// ------------------------------------------------------------------ any shape

// h[m, r] in float32 for any width, rank and type: a workgroup per row, a wave per rank, the channels over its lanes.
template <typename T>
__global__ __launch_bounds__(256) void adapter_shrink_plain_kernel(const T* __restrict__ x, const T* __restrict__ a,
                                                                   const int32_t* __restrict__ ids,
                                                                   float* __restrict__ h, int tokens, int k, int rank,
                                                                   int slots) {
  const int64_t m = blockIdx.x;
  const int t = ids[m / tokens];
  if (t < 0 || t >= slots) return;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const T* xp = x + m * k;
  for (int r = wave; r < rank; r += 4) {
    const T* ap = a + ((int64_t)t * rank + r) * k;
    float s = 0.0f;
    for (int c = lane; c < k; c += 64) s = fmaf(io<T>::ld(xp + c), io<T>::ld(ap + c), s);
    s = group_sum(s, 64);
    if (lane == 0) h[m * rank + r] = s;
  }
}

// out[m, j] = y[m, j] + scale_t sum_r h[m, r] B_t[j, r]: one thread per output, the ranks in order.
template <typename T>
__global__ __launch_bounds__(256) void adapter_expand_plain_kernel(const T* y, const T* __restrict__ b,
                                                                   const float* __restrict__ scale,
                                                                   const int32_t* __restrict__ ids,
                                                                   const float* __restrict__ h, T* out, int64_t rows,
                                                                   int tokens, int n, int rank, int slots) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * n) return;
  const int64_t m = i / n;
  const int j = (int)(i - m * n), t = ids[m / tokens];
  if (t < 0 || t >= slots) {
    out[i] = y[i];
    return;
  }
  const T* bp = b + ((int64_t)t * n + j) * rank;
  const float* hp = h + m * rank;
  float s = 0.0f;
  for (int r = 0; r < rank; ++r) s = fmaf(hp[r], io<T>::ld(bp + r), s);
  io<T>::st(out + i, fmaf(scale[t], s, io<T>::ld(y + i)));
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
  hipLaunchKernelGGL((adapter_shrink_plain_kernel<T>), dim3((unsigned)rows), dim3(256), 0, stream,
                     static_cast<const T*>(x), static_cast<const T*>(a), ids, h, tokens, k, rank, slots);
  hipLaunchKernelGGL((adapter_expand_plain_kernel<T>), dim3((unsigned)((rows * n + 255) / 256)), dim3(256), 0, stream,
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
  DSV41_REQUIRE(rows < (1ll << 31) && (rows * n + 255) / 256 < (1ll << 31), DSV41_E_ARG, "%s: too many outputs", what);
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
