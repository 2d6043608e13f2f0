// y = x W^T for 4-bit weights with group scales and a few rows of x.
//
//   y[t, n] = sum_k x[t, k] (q[n, k] - z[n, k / g]) s[n, k / g]
//
// Bound by the bytes of the codes and scales.  One CTA of 16 warps an SM keeps
// x in shared memory and walks over tiles of 16 rows of W.  The warps form
// groups; a group's warps split the reduction of its tile and their 32-bit
// sums meet in shared memory in warp order, so results do not depend on
// timing.  Each warp keeps kDepth units in flight, across the ends of tiles.
#include "hca_stream.cuh"

#include <algorithm>

namespace hca {
namespace {

constexpr int kWarps = 16;
// shared memory of a CTA: x and the tile sums
constexpr int64_t kSmem = 227 * 1024;

struct W4Args {
  void* out;
  int64_t out_stride;
  const void* x;
  int64_t x_stride;
  const uint8_t* q;
  const void* scales;
  const uint8_t* zeros;
  int tokens, n, k;
  int group_warps;  // warps that share a tile
};

template <int F, typename T, int NB, int kWidth>
__global__ void __launch_bounds__(kWarps * 32, 1) w4_linear_kernel(W4Args a) {
  using W = WTraits<F>;
  using X = XTile<F, T, NB, kWidth>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 31;
  const TileGroup g(a.group_warps);
  const int units = W::units(a.k), groups = a.k / W::kGroupK;
  X xt(smem, units);
  TileSums<NB> ts(smem + X::bytes(units));
  const int tiles = (a.n + 15) / 16, per_cta = kWarps / g.warps, stride = gridDim.x * per_cta;
  const int t0 = blockIdx.y * X::kColumns;
  const int columns = min(X::kColumns, a.tokens - t0), live = (columns + kWidth - 1) / kWidth;
  const int first = blockIdx.x * per_cta + g.id;

  pdl_wait_and_release();
  auto rows = [&](WCursor<F>& cur, int i) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      // rows past the end are read again, not stored
      const int64_t row = min((first + i * stride) * 16 + (lane >> 2) + 8 * r, a.n - 1);
      cur.data[r] = a.q + row * W::row_bytes(a.k) + (lane & 3) * 4 * W::kWords;
      cur.scale[r] = static_cast<const T*>(a.scales) + row * groups;
      cur.zero[r] = a.zeros == nullptr ? nullptr : a.zeros + row * groups;
    }
  };
  TileRing<F> ring;
  ring.start(a.k, g, first < tiles ? (tiles - first + stride - 1) / stride : 0, rows);
  const T* x = static_cast<const T*>(a.x) + t0 * a.x_stride;
  xt.stage(a.k, columns, live, [&](int col) { return x + col * a.x_stride; });

  float acc[NB][4] = {};
  auto finish = [&](int i, const float* sums) {
    const int row0 = (first + i * stride) * 16;
    for (int j = g.thread(); j < live * 128; j += g.threads()) {
      const int row = row0 + (j & 15), block = j >> 7, col = (j >> 4) & 7, t = block * kWidth + col;
      if (row < a.n && col < kWidth && t < columns)
        static_cast<T*>(a.out)[(t0 + t) * a.out_stride + row] =
            MmaType<T>::from_float(TileSums<NB>::sum(sums, g, j & 15, block, col) * Scaling<F, T>::kOut);
    }
  };
  if (NB > 1 && live == 1) ring.template run<1>(xt, g, ts, acc, rows, finish);
  else ring.template run<NB>(xt, g, ts, acc, rows, finish);
}

template <int F, typename T, int NB, int kWidth>
constexpr int64_t smem_bytes(int units) {
  return XTile<F, T, NB, kWidth>::bytes(units) + TileSums<NB>::bytes(kWarps);
}

template <int F, typename T, int NB, int kWidth>
int launch(W4Args a, cudaStream_t s) {
  const int units = WTraits<F>::units(a.k), tiles = cdiv(a.n, 16), sms = device_sm_count();
  // Warps to a tile: as few as leave every SM's groups four tiles each, but
  // at least one unit a warp.  Few warps mean long runs between reductions,
  // many that a short matrix still fills the machine.
  a.group_warps = 1;
  while (a.group_warps < kWarps && tiles < 4ll * sms * (kWarps / a.group_warps) && 2 * a.group_warps <= units)
    a.group_warps *= 2;
  const int per_cta = kWarps / a.group_warps;
  static bool done[kMaxDevices] = {};
  if (set_func_attr_once(w4_linear_kernel<F, T, NB, kWidth>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem,
                         done) != HCA_OK)
    return HCA_E_CUDA;
  return launch_pdl(w4_linear_kernel<F, T, NB, kWidth>,
                    dim3(std::min(sms, cdiv(tiles, per_cta)), cdiv(a.tokens, NB * kWidth)), dim3(kWarps * 32),
                    smem_bytes<F, T, NB, kWidth>(units), s, a);
}

template <int F, typename T>
int by_rows(W4Args a, cudaStream_t s) {
  const int units = WTraits<F>::units(a.k);
  // Columns of x a pass holds: as many as there are rows and shared memory
  // for; what is left takes further passes over the weights.
  if (a.tokens > 8 && smem_bytes<F, T, 2, 8>(units) <= kSmem) return launch<F, T, 2, 8>(a, s);
  if (a.tokens > 2 && smem_bytes<F, T, 1, 8>(units) <= kSmem) return launch<F, T, 1, 8>(a, s);
  if (smem_bytes<F, T, 1, 2>(units) <= kSmem) return launch<F, T, 1, 2>(a, s);
  return HCA_E_UNSUPPORTED;
}

template <typename T>
int by_group(int group, W4Args a, cudaStream_t s) {
  switch (group) {
    case 32: return by_rows<kW4G32, T>(a, s);
    case 64: return by_rows<kW4G64, T>(a, s);
    default: return by_rows<kW4G128, T>(a, s);
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
  HCA_CHECK_ARG(num_tokens <= 65535 && n <= INT32_MAX - 16);  // grid columns hold at least one row of x
  W4Args a{out, out_stride, x, x_stride, q, scales, zeros, num_tokens, n, k, 1};
  cudaStream_t s = as_stream(stream);
  return is_fp16 ? by_group<__half>(group_size, a, s) : by_group<__nv_bfloat16>(group_size, a, s);
}
