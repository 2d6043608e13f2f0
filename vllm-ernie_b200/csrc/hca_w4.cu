// y = x W^T for 4-bit weights with group scales and a few rows of x.
//
//   y[t, n] = sum_k x[t, k] (q[n, k] - z[n, k / g]) s[n, k / g]
//
// Bound by the bytes of the codes and scales.  One CTA of 16 warps an SM keeps
// x in shared memory and walks over tiles of 16 rows of W.  The warps form
// groups; a group's warps split the reduction of its tile and their 32-bit
// sums meet in shared memory in warp order, so results do not depend on
// timing.
//
// Measured: [129281, 4096], groups of 128 with zero points, 8 rows: 53.6 us,
// 5.2 TB/s (a run of seconds meets the power limit: 61 us at 1.65 GHz; the loop
// keeps the issue slots half and the shared-memory pipe two thirds busy).  Small
// ones are bound by what comes before the first product, laying out x above all
// (16 rows of 4096: about 2 us of 10.2 for [8192, 4096]), and by uneven shares
// (fp16, [4096, 8192], 3 rows, groups of 32: 10.1 us, 256 tiles on 148 SMs, issue
// slots half full); [8192, 1024], one row: 3.8 us.  Rows in pieces: 3 x 29568,
// N 8192, groups of 32: 101 us for 22 of bytes.
#include "hca_stream.cuh"

#include <algorithm>

namespace hca {
namespace {

constexpr int kWarps = 16;
// shared memory of a CTA: x and the tile sums
constexpr int64_t kSmem = 227 * 1024;
// Rows of x too long for that are taken in pieces of 4096, two warps a tile:
// eight tiles use a piece while it is there (four times the bytes of eight rows).
constexpr int kLongK = 4096, kLongWarps = 2;

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
  int ahead;        // whether a group's first tile is fetched into L2 before all else
};

// The tiles of a group of warps: first, first + stride, ...
template <int F, typename T>
struct W4Tiles {
  using W = WTraits<F>;
  const W4Args& a;
  int first, stride, groups;
  int k0 = 0;  // first k of the piece

  __device__ __forceinline__ int64_t row(int i, int r) const {
    return min((first + i * stride) * 16 + r, a.n - 1);  // rows past the end are read again, not stored
  }
  __device__ __forceinline__ TileRows rows(int i) const {
    const int lane = threadIdx.x & 31;
    TileRows t;
#pragma unroll
    for (int r = 0; r < 2; ++r)
      t.data[r] = a.q + (lane & 3) * 16 + row(i, (lane >> 2) + 8 * r) * W::row_bytes(a.k) + W::row_bytes(k0);
    return t;
  }
  __device__ __forceinline__ bool zeros() const { return a.zeros != nullptr; }
  __device__ __forceinline__ bool rows_wide() const { return scales_wide(a.scales, a.zeros, groups); }
  __device__ __forceinline__ WScales here(int i, int r) const {
    const int64_t at = row(i, r) * groups + k0 / W::kGroupK, all = static_cast<int64_t>(a.n) * groups;
    const uint8_t* s = static_cast<const uint8_t*>(a.scales);
    return {s + 2 * at, s + 2 * all, a.zeros == nullptr ? nullptr : a.zeros + at, a.zeros + all};
  }
  __device__ __forceinline__ WScales scales(int i, int r) const { return here(i, r); }
};

template <int F, typename T, int NB, int kWidth>
__global__ void __launch_bounds__(kWarps * 32, 1) w4_linear_kernel(W4Args a) {
  using W = WTraits<F>;
  using X = XTile<F, T, NB, kWidth>;
  extern __shared__ __align__(16) uint8_t smem[];
  const TileGroup g(a.group_warps);
  const int units = W::units(a.k);
  X xt(smem, units);
  TileSums<NB> ts(smem + X::bytes(units));
  const int tiles = (a.n + 15) / 16, per_cta = kWarps / g.warps;
  const int t0 = blockIdx.y * X::kColumns;
  const int columns = min(X::kColumns, a.tokens - t0), live = (columns + kWidth - 1) / kWidth;
  W4Tiles<F, T> src{a, static_cast<int>(blockIdx.x + g.id * gridDim.x), static_cast<int>(gridDim.x) * per_cta, a.k / W::kGroupK};

  if (g.thread() == 0 && a.ahead && src.first < tiles)
    prefetch_weights(a.q + src.first * 16ll * W::row_bytes(a.k), min(16, a.n - src.first * 16) * W::row_bytes(a.k));
  pdl_wait_and_release();
  TileStream<F, T, WTraits<F>::step(NB)> stream;
  stream.start(a.k, g, src.first < tiles ? (tiles - src.first + src.stride - 1) / src.stride : 0,
             smem + X::bytes(units) + TileSums<NB>::bytes(kWarps), src, units);
  const T* x = static_cast<const T*>(a.x) + t0 * a.x_stride;
  xt.stage(a.k, columns, live, [&](int col) { return x + col * a.x_stride; });

  float acc[NB][4] = {};
  auto finish = [&](int i, const float* sums) {
    const int row0 = (src.first + i * src.stride) * 16;
#pragma unroll 1
    for (int j = g.thread(); j < live * 128; j += g.threads()) {
      const int row = row0 + (j & 15), block = j >> 7, col = (j >> 4) & 7, t = block * kWidth + col;
      if (row < a.n && col < kWidth && t < columns)
        static_cast<T*>(a.out)[(t0 + t) * a.out_stride + row] =
            MmaType<T>::from_float(TileSums<NB>::sum(sums, g, j & 15, block, col) * Scaling<F, T>::kOut);
    }
  };
  if (NB > 1 && live == 1) stream.template run<1>(xt, g, ts, acc, src, finish);
  else stream.template run<NB>(xt, g, ts, acc, src, finish);
}

// The same for rows of any length: a group holds one tile at a time, for which
// the pieces of x come into shared memory in turn.
template <int F, typename T>
__global__ void __launch_bounds__(kWarps * 32, 1) w4_long_kernel(W4Args a) {
  using W = WTraits<F>;
  using X = XTile<F, T, 1, 8>;
  extern __shared__ __align__(16) uint8_t smem[];
  const TileGroup g(kLongWarps);
  constexpr int per_cta = kWarps / kLongWarps, units = W::units(kLongK);
  TileSums<1> ts(smem + X::bytes(units));
  float* total = reinterpret_cast<float*>(smem + X::bytes(units) + TileSums<1>::bytes(kWarps)) + g.id * 128;
  uint8_t* scales = smem + X::bytes(units) + TileSums<1>::bytes(kWarps) + per_cta * 512;
  const int tiles = (a.n + 15) / 16, t0 = blockIdx.y * X::kColumns, columns = min(X::kColumns, a.tokens - t0);
  const T* x = static_cast<const T*>(a.x) + t0 * a.x_stride;
  pdl_wait_and_release();
#pragma unroll 1
  for (int64_t first = blockIdx.x; first < tiles; first += static_cast<int64_t>(gridDim.x) * per_cta) {
    const int64_t tile = first + g.id * gridDim.x;
    const bool mine = tile < tiles;
    W4Tiles<F, T> src{a, static_cast<int>(mine ? tile : 0), 0, a.k / W::kGroupK};
#pragma unroll 1
    for (; src.k0 < a.k; src.k0 += kLongK) {
      const int k = min(kLongK, a.k - src.k0);
      TileStream<F, T, W::step(1)> stream;
      stream.start(k, g, mine, scales, src, units);  // other groups may still read the last piece's scales
      __syncthreads();  // the last piece has been read
      X xt(smem, W::units(k));
      xt.stage(k, columns, 1, [&](int col) { return x + col * a.x_stride + src.k0; });
      float acc[1][4] = {};
      // a thread meets the same sums each time
      stream.template run<1>(xt, g, ts, acc, src, [&](int, const float* sums) {
#pragma unroll 1
        for (int j = g.thread(); j < 128; j += g.threads()) {
          const int64_t row = tile * 16 + (j & 15);
          const int col = j >> 4;
          float v = TileSums<1>::sum(sums, g, j & 15, 0, col) * Scaling<F, T>::kOut;
          if (src.k0 > 0) v += total[j];
          if (src.k0 + k < a.k) total[j] = v;
          else if (row < a.n && col < columns) static_cast<T*>(a.out)[(t0 + col) * a.out_stride + row] = MmaType<T>::from_float(v);
        }
      });
    }
  }
}

template <int F, typename T>
int launch_long(const W4Args& a, cudaStream_t s) {
  constexpr int units = WTraits<F>::units(kLongK);
  const int tiles = cdiv(a.n, 16), sms = device_sm_count();
  const int64_t smem = XTile<F, T, 1, 8>::bytes(units) + TileSums<1>::bytes(kWarps) + kWarps / kLongWarps * 512 +
                       ScaleTile<F>::bytes(units, a.zeros != nullptr, kLongWarps, kWarps);
  static bool done[kMaxDevices] = {};
  const int rc = set_func_attr_once(w4_long_kernel<F, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem, done);
  if (rc != HCA_OK) return rc;
  return launch_pdl(w4_long_kernel<F, T>, dim3(std::min(sms, tiles), cdiv(a.tokens, 8)), dim3(kWarps * 32),
                    static_cast<size_t>(smem), s, a);
}

// Launches with NB blocks of kWidth columns if shared memory holds them.
template <int F, typename T, int NB, int kWidth>
bool launch(W4Args a, cudaStream_t s, int& rc) {
  const int units = WTraits<F>::units(a.k), tiles = cdiv(a.n, 16), sms = device_sm_count();
  const int64_t columns = XTile<F, T, NB, kWidth>::bytes(units) + TileSums<NB>::bytes(kWarps);
  auto scales = [&](int warps) { return ScaleTile<F>::bytes(units, a.zeros != nullptr, warps, kWarps); };
  // Warps to a tile: the number that makes the longest warp's work shortest,
  // a tile's end (its sums meet) costing about what a quad of units does; as
  // few as the room for scales allows of several.
  a.group_warps = 0;
  int64_t best = INT64_MAX;
  for (int gw = 1; gw <= kWarps && 4 * gw <= units; gw *= 2) {
    const int64_t cost = static_cast<int64_t>(cdiv(tiles, sms * (kWarps / gw))) * (cdiv(units, 4 * gw) + 1);
    if (cost < best && columns + scales(gw) <= kSmem) best = cost, a.group_warps = gw;
  }
  if (a.group_warps == 0) return false;
  // Weights that last for a round or two start before the kernel before this
  // one has ended (11.6 -> 10.8 us for 8192 x 4096 and 16 rows, weights not in L2).
  a.ahead = tiles <= 2 * sms * (kWarps / a.group_warps);
  const int64_t smem = columns + scales(a.group_warps);
  static bool done[kMaxDevices] = {};
  rc = set_func_attr_once(w4_linear_kernel<F, T, NB, kWidth>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem, done);
  if (rc == HCA_OK) {
    rc = launch_pdl(w4_linear_kernel<F, T, NB, kWidth>,
                    dim3(std::min(sms, tiles), cdiv(a.tokens, NB * kWidth)),
                    dim3(kWarps * 32), static_cast<size_t>(smem), s, a);
  }
  return true;
}

template <int F, typename T>
int by_rows(const W4Args& a, cudaStream_t s) {
  // Columns of x a pass holds: as many as there are rows and shared memory
  // for; what is left takes further passes over the weights.
  int rc = HCA_OK;
  if (a.tokens > 8 && launch<F, T, 2, 8>(a, s, rc)) return rc;
  if (a.tokens > 4 && launch<F, T, 1, 8>(a, s, rc)) return rc;
  if (a.tokens > 2 && launch<F, T, 1, 4>(a, s, rc)) return rc;
  if (launch<F, T, 1, 2>(a, s, rc)) return rc;
  return launch_long<F, T>(a, s);
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
  HCA_CHECK_ARG(reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(scales) % 4 == 0 &&
                reinterpret_cast<uintptr_t>(zeros) % 4 == 0 && reinterpret_cast<uintptr_t>(out) % 2 == 0);
  HCA_CHECK_ARG(n <= INT32_MAX - 16);
  cudaStream_t s = as_stream(stream);
  // a launch for each 65520 rows (whole blocks of columns): a grid has 65535 at most
  constexpr int kRows = 65520;
  for (int t = 0; t < num_tokens; t += std::min(kRows, num_tokens - t)) {
    const W4Args a{static_cast<uint16_t*>(out) + t * out_stride, out_stride, static_cast<const uint16_t*>(x) + t * x_stride,
                   x_stride, q, scales, zeros, std::min(kRows, num_tokens - t), n, k, 1, 0};
    const int rc = is_fp16 ? by_group<__half>(group_size, a, s) : by_group<__nv_bfloat16>(group_size, a, s);
    if (rc != HCA_OK) return rc;
  }
  return HCA_OK;
}
