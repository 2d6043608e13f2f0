// y = x W^T for 4-bit weights with group scales and a few rows of x.
//
//   y[t, n] = sum_k x[t, k] (q[n, k] - z[n, k / g]) s[n, k / g]
//
// Bound by the bytes of the codes and scales.  A CTA owns 16 rows of W and all
// rows of x (up to 8 NB; more run as further grid columns): its eight warps
// split the reduction in whole groups, and their 32-bit sums meet in shared
// memory in warp order, so results do not depend on timing.
#include "hca_stream.cuh"

namespace hca {
namespace {

constexpr int kWarps = 8;

template <int F, typename T, int NB>
__global__ void __launch_bounds__(kWarps * 32) w4_linear_kernel(
    T* __restrict__ out, int64_t out_stride, const T* x, int64_t x_stride, const uint8_t* q, const T* scales,
    const uint8_t* zeros, int tokens, int n, int k) {
  using W = WTraits<F>;
  __shared__ float red[kWarps][NB * 8][16];
  pdl_wait_and_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n0 = blockIdx.x * 16, t0 = blockIdx.y * 8 * NB;
  const int units = k / W::kUnitK;

  WRows<T> rows;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t row = min(n0 + (lane >> 2) + 8 * r, n - 1);  // rows past the end are read again, not stored
    rows.data[r] = q + row * W::row_bytes(k);
    rows.scale[r] = scales + row * units;
    rows.zero[r] = zeros == nullptr ? nullptr : zeros + row * units;
  }
  int64_t x_off[NB];
  const int live = min(NB, (tokens - t0 + 7) / 8);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int t = t0 + 8 * b + (lane >> 2);
    x_off[b] = t < tokens ? t * x_stride : -1;
  }
  float acc[NB][4] = {};
  stream_rows<F, T, NB>(acc, rows, x, x_off, live, k, units * warp / kWarps, units * (warp + 1) / kWarps);

#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) red[warp][8 * b + 2 * (lane & 3) + (i & 1)][(lane >> 2) + 8 * (i >> 1)] = acc[b][i];
  __syncthreads();
  for (int i = threadIdx.x; i < 8 * NB * 16; i += kWarps * 32) {
    const int row = n0 + (i & 15), t = t0 + (i >> 4);
    if (row >= n || t >= tokens) continue;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += red[w][i >> 4][i & 15];
    out[t * out_stride + row] = MmaType<T>::from_float(v);
  }
}

template <int F, typename T, int NB>
int launch(void* out, int64_t out_stride, const void* x, int64_t x_stride, const uint8_t* q, const void* scales,
           const uint8_t* zeros, int tokens, int n, int k, cudaStream_t s) {
  return launch_pdl(w4_linear_kernel<F, T, NB>, dim3(cdiv(n, 16), cdiv(tokens, 8 * NB)), dim3(kWarps * 32), 0, s,
                    static_cast<T*>(out), out_stride, static_cast<const T*>(x), x_stride, q,
                    static_cast<const T*>(scales), zeros, tokens, n, k);
}

template <int F, typename T>
int by_rows(void* out, int64_t out_stride, const void* x, int64_t x_stride, const uint8_t* q, const void* scales,
            const uint8_t* zeros, int tokens, int n, int k, cudaStream_t s) {
  if (tokens <= 8) return launch<F, T, 1>(out, out_stride, x, x_stride, q, scales, zeros, tokens, n, k, s);
  if (tokens <= 16) return launch<F, T, 2>(out, out_stride, x, x_stride, q, scales, zeros, tokens, n, k, s);
  return launch<F, T, 4>(out, out_stride, x, x_stride, q, scales, zeros, tokens, n, k, s);
}

template <typename T>
int by_group(int group, void* out, int64_t out_stride, const void* x, int64_t x_stride, const uint8_t* q,
             const void* scales, const uint8_t* zeros, int tokens, int n, int k, cudaStream_t s) {
  switch (group) {
    case 32: return by_rows<kW4G32, T>(out, out_stride, x, x_stride, q, scales, zeros, tokens, n, k, s);
    case 64: return by_rows<kW4G64, T>(out, out_stride, x, x_stride, q, scales, zeros, tokens, n, k, s);
    case 128: return by_rows<kW4G128, T>(out, out_stride, x, x_stride, q, scales, zeros, tokens, n, k, s);
    default: return HCA_E_UNSUPPORTED;
  }
}

}  // namespace
}  // namespace hca

extern "C" int hca_w4_linear(void* out, int64_t out_stride, const void* x, int64_t x_stride, const uint8_t* q,
                             const void* scales, const uint8_t* zeros, int32_t num_tokens, int32_t n, int32_t k,
                             int32_t group_size, int32_t is_fp16, void* stream) {
  using namespace hca;
  if (group_size != 32 && group_size != 64 && group_size != 128) return HCA_E_UNSUPPORTED;
  HCA_CHECK_ARG(num_tokens >= 0 && n > 0 && k > 0 && k % group_size == 0);
  if (num_tokens == 0) return HCA_OK;
  HCA_CHECK_ARG(out && x && q && scales);
  HCA_CHECK_ARG(x_stride % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0);
  HCA_CHECK_ARG(reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(scales) % 2 == 0 &&
                reinterpret_cast<uintptr_t>(out) % 2 == 0);
  // grid columns hold 32 rows of x
  HCA_CHECK_ARG(cdiv(num_tokens, 32) <= 65535);
  cudaStream_t s = as_stream(stream);
  return is_fp16 ? by_group<__half>(group_size, out, out_stride, x, x_stride, q, scales, zeros, num_tokens, n, k, s)
                 : by_group<__nv_bfloat16>(group_size, out, out_stride, x, x_stride, q, scales, zeros, num_tokens, n,
                                           k, s);
}
