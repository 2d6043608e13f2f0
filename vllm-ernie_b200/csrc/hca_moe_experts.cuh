// The second launch of the few-token mixture-of-experts layer.
//
//   h[t, j] = w[t, j] silu(W1_e x_t) * (W3_e x_t),  e = ids[t, j]
//   y[t]    = sum_j W2_e h[t, j]  (+ the shared expert's with weight 1)
//
// Both products are bound by the bytes of the chosen experts' weights, each
// read once for all tokens that chose the expert (hca_stream.cuh).  A CTA of
// 16 warps takes a contiguous run of (expert, 16 rows) tiles, so that it meets
// few experts and lays out their columns in shared memory once.  The second
// product leaves each (token, slot) pair's share of y in 32 bits, and the last
// step adds a token's shares in the order of its slots: no atomics, and a
// token's result does not depend on what else is in the batch.  h is rounded
// to bf16 once, its weight included.
//
// One launch with two grid barriers, since each of the steps is short at one
// token: the weights of the second product start on their way before the
// barrier that its activations wait for.
#pragma once

#include <algorithm>

#include "hca_moe.cuh"
#include "hca_stream.cuh"

namespace hca {
namespace moe {

constexpr int kWarps = 16;
constexpr int kThreads = kWarps * 32;
// shared memory of a CTA for columns and tile sums, beside the plan
constexpr int64_t kSmem = 208 * 1024;

// Who computes what, made by every CTA from the ids (at most 1024 of them) in
// shared memory.  A pair is t * top_k + j; the shared expert's are tokens *
// top_k + t.  An entry is up to `columns` pairs of one expert, so that every
// entry's weights cost one pass; entries are in the experts' order, the
// shared expert (number `experts`) last, and pairs in theirs.
template <int kColumns>
struct Plan {
  static constexpr int kEntries = kMoeExperts + 1 + kMoePairs / kColumns;
  int entries, routed;        // with and without the shared expert's
  int16_t expert[kEntries];   // entry -> expert
  int16_t start[kEntries + 1];  // entry -> first pair
  int16_t pair[kMoePairs];
  int16_t id[kMoePairs];        // pair -> expert, or -1
  float weight[kMoePairs];
  int16_t rank[kMoePairs];      // pair -> place in its expert's list
  int16_t list[kMoeExperts + 1];  // expert -> number of pairs, then first pair
};

template <int kColumns>
__device__ __forceinline__ void build_plan(Plan<kColumns>& pl, const MoePass& p) {
  const int lane = threadIdx.x & 31, top_k = p.routing.top_k, experts = p.routing.experts;
  const int routed = p.tokens * top_k, n = routed + p.tokens;
  if (p.logits != nullptr) {
    for (int t = threadIdx.x >> 5; t < p.tokens; t += kWarps) {
      int id;
      float weight;
      choose_experts(p.logits + static_cast<int64_t>(t) * experts, p.routing, t, id, weight);
      if (lane < top_k) pl.id[t * top_k + lane] = static_cast<int16_t>(id), pl.weight[t * top_k + lane] = weight;
    }
  } else {
    for (int i = threadIdx.x; i < routed; i += kThreads) {
      const int e = p.routing.mask == nullptr || p.routing.mask[i / top_k] ? p.ids[i] : -1;
      pl.id[i] = static_cast<int16_t>(e >= 0 && e < experts ? e : -1);
      pl.weight[i] = p.weights[i];
    }
  }
  for (int t = threadIdx.x; t < p.tokens; t += kThreads) {
    const bool in = p.shared_inner > 0 && (p.routing.mask == nullptr || p.routing.mask[t]);
    pl.id[routed + t] = static_cast<int16_t>(in ? experts : -1);
    pl.weight[routed + t] = 1.0f;
  }
  for (int e = threadIdx.x; e <= experts; e += kThreads) pl.list[e] = 0;
  __syncthreads();
  if (threadIdx.x < 32) {
    // 32 pairs at a time, so that the lists come out in order
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int i = i0 + lane;
      const int e = i < n ? pl.id[i] : -1;
      const unsigned same = __match_any_sync(0xffffffffu, e);
      const int before = __popc(same & ((1u << lane) - 1));
      int base = 0;
      if (e >= 0) base = pl.list[e];
      __syncwarp();
      if (e >= 0 && before == 0) pl.list[e] = static_cast<int16_t>(base + __popc(same));
      __syncwarp();
      if (e >= 0) pl.rank[i] = static_cast<int16_t>(base + before);
    }
    int entries = 0, pairs = 0;
    for (int e0 = 0; e0 <= experts; e0 += 32) {
      const int e = e0 + lane;
      const int c = e <= experts ? pl.list[e] : 0, pieces = (c + kColumns - 1) / kColumns;
      int before = c | pieces << 16;  // inclusive sums of both
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
      }
      const int first = pairs + (before & 0xffff) - c, at = entries + (before >> 16) - pieces;
      if (c > 0) pl.list[e] = static_cast<int16_t>(first);
      for (int i = 0; i < pieces; ++i) {
        pl.expert[at + i] = static_cast<int16_t>(e);
        pl.start[at + i] = static_cast<int16_t>(first + i * kColumns);
      }
      if (e == experts) pl.routed = at;
      const int all = __shfl_sync(0xffffffffu, before, 31);
      pairs += all & 0xffff, entries += all >> 16;
    }
    if (lane == 0) pl.entries = entries, pl.start[entries] = static_cast<int16_t>(pairs);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads)
    if (pl.id[i] >= 0) pl.pair[pl.list[pl.id[i]] + pl.rank[i]] = static_cast<int16_t>(i);
  __syncthreads();
}

// Every CTA of the grid has arrived `phase` times.  False if one does not in
// two seconds (none can be missing in a cooperative launch).
__device__ __forceinline__ void grid_arrive(uint32_t* barrier) {
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    atomicAdd(barrier, 1u);
  }
}
__device__ __forceinline__ bool grid_wait(uint32_t* barrier, uint32_t phase, int32_t* error) {
  int ok = 1;
  if (threadIdx.x == 0) {
    const uint32_t target = phase * gridDim.x;
    uint64_t t0 = 0, now;
    for (;;) {
      uint32_t v;
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];\n" : "=r"(v) : "l"(barrier) : "memory");
      if (v >= target) break;
      asm volatile("mov.u64 %0, %globaltimer;\n" : "=l"(now));
      if (t0 == 0) t0 = now;
      if (now - t0 > 2000000000ull) {
        atomicOr(error, kErrMoe);
        ok = 0;
        break;
      }
    }
    __threadfence();
  }
  return __syncthreads_and(ok || threadIdx.x != 0);
}

// Row `row` of matrix e of a stack of matrices with n rows of k.
template <int F>
__device__ __forceinline__ void set_row(WCursor<F>& cur, int r, const MoeMatrix& m, int64_t e, int n, int row, int k) {
  using W = WTraits<F>;
  const int64_t at = e * n + row;
  cur.data[r] = m.data + at * W::row_bytes(k) + (threadIdx.x & 3) * 4 * W::kWords;
  if constexpr (W::kIs4) {
    const int groups = k / W::kGroupK;
    cur.scale[r] = static_cast<const __nv_bfloat16*>(m.scale) + at * groups;
    cur.zero[r] = m.zero == nullptr ? nullptr : m.zero + at * groups;
  } else if constexpr (F == kWFp8) {
    const int64_t kb = (k + 127) / 128, nb = (n + 127) / 128;
    cur.scale[r] = static_cast<const float*>(m.scale) + (e * nb + row / 128) * kb;
  }
}

struct Shape {
  int up_warps, down_warps;  // warps that share a tile of either product
  int dense;                 // the first product's columns are the tokens, the same for every expert
};

// One of the products over this CTA's run of (entry, tile) items.  kUp: h from
// x (fragment rows 0..7 of a tile are gate rows, 8..15 the up rows of the same
// inner columns, so a lane holds both factors); else part from h.
template <int F, int NB, int kWidth, bool kUp>
struct Product {
  using W = WTraits<F>;
  using X = XTile<F, __nv_bfloat16, NB, kWidth>;
  using P = Plan<NB * kWidth>;
  const MoePass& p;
  const MoeWeights& w;
  const P& pl;
  uint8_t* smem;
  TileGroup g;
  bool dense;
  int per_cta, tiles, pairs, from, to, end;  // [from, to) is the segment
  int first_entry, first_tile;               // of the group in the segment
  TileRing<F> ring;

  __device__ __forceinline__ Product(const MoePass& p_, const MoeWeights& w_, const P& pl_, uint8_t* smem_, int warps, bool dense_)
      : p(p_), w(w_), pl(pl_), smem(smem_), g(warps), dense(dense_) {
    per_cta = kWarps / g.warps;
    tiles = kUp ? p.inner / 8 : p.hidden / 16;  // of a routed entry
    pairs = p.tokens * p.routing.top_k;
    const int shared_tiles = kUp ? p.shared_inner / 8 : tiles;
    const int64_t items = static_cast<int64_t>(pl.routed) * tiles + static_cast<int64_t>(pl.entries - pl.routed) * shared_tiles;
    from = to = static_cast<int>(items * blockIdx.x / gridDim.x);
    end = static_cast<int>(items * (blockIdx.x + 1) / gridDim.x);
  }
  __device__ __forceinline__ int tiles_of(int entry) const { return kUp && entry >= pl.routed ? p.shared_inner / 8 : tiles; }
  __device__ __forceinline__ int k_of(int entry) const {
    return kUp ? p.hidden : entry >= pl.routed ? p.shared_inner : p.inner;
  }
  // The item `by` after (entry, tile).
  __device__ __forceinline__ void move(int& entry, int& tile, int by) const {
    tile += by;
    for (int n = tiles_of(entry); tile >= n && entry + 1 < pl.entries; n = tiles_of(entry)) tile -= n, ++entry;
  }
  __device__ __forceinline__ void rows(WCursor<F>& cur, int entry, int tile) const {
    const bool shared = entry >= pl.routed;
    const int e = shared ? 0 : pl.expert[entry], row = (threadIdx.x & 31) >> 2;
    if (kUp) {
      const int inner = shared ? p.shared_inner : p.inner;
      const MoeMatrix& m = shared ? w.shared13 : w.w13;
      set_row<F>(cur, 0, m, e, 2 * inner, tile * 8 + row, p.hidden);
      set_row<F>(cur, 1, m, e, 2 * inner, inner + tile * 8 + row, p.hidden);
    } else {
      const MoeMatrix& m = shared ? w.shared2 : w.w2;
      set_row<F>(cur, 0, m, e, p.hidden, tile * 16 + row, k_of(entry));
      set_row<F>(cur, 1, m, e, p.hidden, tile * 16 + 8 + row, k_of(entry));
    }
  }
  __device__ __forceinline__ __nv_bfloat16* h_row(int pair) const {
    return pair < pairs ? p.h + static_cast<int64_t>(pair) * p.inner
                        : p.h + static_cast<int64_t>(pairs) * p.inner + static_cast<int64_t>(pair - pairs) * p.shared_inner;
  }
  __device__ __forceinline__ int token(int pair) const { return pair < pairs ? pair / p.routing.top_k : pair - pairs; }

  // Starts the loads of the next segment, the run of tiles that one layout of
  // columns serves: all with dense columns, else those of one entry.
  __device__ __forceinline__ bool start() {
    from = to;
    if (from >= end) return false;
    const int routed_items = pl.routed * tiles;
    if (from < routed_items) first_entry = from / tiles, first_tile = from - first_entry * tiles;
    else {
      const int n = tiles_of(pl.routed);
      first_entry = (from - routed_items) / n, first_tile = from - routed_items - first_entry * n;
      first_entry += pl.routed;
    }
    to = dense ? end : min(end, from - first_tile + tiles_of(first_entry));
    int e = first_entry, t = first_tile, at = 0;
    move(e, t, g.id);
    const int count = to - from > g.id ? (to - from - g.id + per_cta - 1) / per_cta : 0;
    load_entry = e, load_tile = t;
    (void)at;
    ring.start(k_of(first_entry), g, count, [this](WCursor<F>& cur, int i) { next_rows(cur, i); });
    return true;
  }
  int load_entry, load_tile;
  __device__ __forceinline__ void next_rows(WCursor<F>& cur, int i) {
    if (i > 0) move(load_entry, load_tile, per_cta);
    rows(cur, load_entry, load_tile);
  }

  // Lays out the segment's columns and consumes its tiles.  Both ends are
  // block barriers for the columns.
  __device__ __forceinline__ void run(TileSums<NB>& ts) {
    const int k = k_of(first_entry), l0 = pl.start[first_entry];
    const int columns = dense ? p.tokens : pl.start[first_entry + 1] - l0;
    const int live = (columns + kWidth - 1) / kWidth;
    X xt(smem, W::units(k));
    xt.stage(k, columns, live, [&](int col) -> const __nv_bfloat16* {
      if (kUp && dense)
        return p.routing.mask == nullptr || p.routing.mask[col] ? p.x + col * p.x_stride : nullptr;
      const int pair = pl.pair[l0 + col];
      return kUp ? p.x + token(pair) * p.x_stride : h_row(pair);
    });
    int entry = first_entry, tile = first_tile;
    move(entry, tile, g.id);
    float acc[NB][4] = {};
    auto finish = [&](int, const float* sums) {
      constexpr int kCols = kUp ? 8 : 16;
      const int s0 = pl.start[entry], n = (pl.start[entry + 1] - s0) * kCols;
      for (int i = g.thread(); i < n; i += g.threads()) {
        const int pair = pl.pair[s0 + i / kCols], c = i % kCols;
        const int col = dense ? token(pair) : i / kCols;
        const float v = TileSums<NB>::sum(sums, g, c, col / kWidth, col % kWidth) * Scaling<F, __nv_bfloat16>::kOut;
        if (kUp) {
          const float up = TileSums<NB>::sum(sums, g, c + 8, col / kWidth, col % kWidth) * Scaling<F, __nv_bfloat16>::kOut;
          h_row(pair)[tile * 8 + c] = __float2bfloat16_rn(v / (1.0f + expf(-v)) * up * pl.weight[pair]);
        } else {
          p.part[static_cast<int64_t>(pair) * p.hidden + tile * 16 + c] = v;
        }
      }
      move(entry, tile, per_cta);
    };
    auto next = [this](WCursor<F>& cur, int i) { next_rows(cur, i); };
    if (NB > 1 && live == 1) ring.template run<1>(xt, g, ts, acc, next, finish);
    else ring.template run<NB>(xt, g, ts, acc, next, finish);
    __syncthreads();
  }
};

template <int F, int NB, int kWidth>
__global__ void __launch_bounds__(kThreads, 1) moe_layer_kernel(MoePass p, MoeWeights w, Shape shape) {
  using X = XTile<F, __nv_bfloat16, NB, kWidth>;
  __shared__ Plan<NB * kWidth> pl;
  extern __shared__ __align__(16) uint8_t smem[];
  build_plan(pl, p);
  const int k_max = max(p.hidden, max(p.inner, p.shared_inner));
  TileSums<NB> ts(smem + X::bytes(WTraits<F>::units(k_max)));
  {
    Product<F, NB, kWidth, true> up(p, w, pl, smem, shape.up_warps, shape.dense);
    while (up.start()) up.run(ts);
  }
  grid_arrive(p.barrier);
  {
    Product<F, NB, kWidth, false> down(p, w, pl, smem, shape.down_warps, false);
    bool more = down.start();
    if (!grid_wait(p.barrier, 1, p.error)) return;
    while (more) {
      down.run(ts);
      more = down.start();
    }
  }
  grid_arrive(p.barrier);
  if (!grid_wait(p.barrier, 2, p.error)) return;
  // y: a token's shares, in the order of its slots, four columns a thread
  const int quads = p.hidden / 4, top_k = p.routing.top_k;
  for (int i = blockIdx.x * kThreads + threadIdx.x; i < p.tokens * quads; i += gridDim.x * kThreads) {
    const int t = i / quads, n = (i - t * quads) * 4;
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int j = 0; j <= top_k; ++j) {
      const int pair = j < top_k ? t * top_k + j : p.tokens * top_k + t;
      if (pl.id[pair] < 0) continue;
      const float4 v = *reinterpret_cast<const float4*>(p.part + static_cast<int64_t>(pair) * p.hidden + n);
      y.x += v.x, y.y += v.y, y.z += v.z, y.w += v.w;
    }
    __nv_bfloat16* out = p.out + t * p.out_stride + n;
    out[0] = __float2bfloat16_rn(y.x);
    out[1] = __float2bfloat16_rn(y.y);
    out[2] = __float2bfloat16_rn(y.z);
    out[3] = __float2bfloat16_rn(y.w);
  }
}

template <int F, int NB, int kWidth>
constexpr int64_t smem_bytes(int units) {
  return XTile<F, __nv_bfloat16, NB, kWidth>::bytes(units) + TileSums<NB>::bytes(kWarps);
}

template <int F, int NB, int kWidth>
int launch(const MoePass& p, const MoeWeights& w, int units, cudaStream_t s) {
  using W = WTraits<F>;
  const int sms = device_sm_count();
  // Warps to a tile: as few as leave every group of every SM two tiles (if
  // every pair chose another expert), but at least one unit a warp.
  auto warps = [&](int64_t tiles, int64_t shared_tiles, int least_units) {
    const int64_t n = std::min(p.routing.experts, p.tokens * p.routing.top_k) * tiles + shared_tiles;
    int gw = 1;
    while (gw < kWarps && n < 2ll * sms * (kWarps / gw) && 2 * gw <= least_units) gw *= 2;
    return gw;
  };
  Shape shape;
  shape.up_warps = warps(p.inner / 8, p.shared_inner / 8, W::units(p.hidden));
  shape.down_warps = warps(p.hidden / 16, p.shared_inner > 0 ? p.hidden / 16 : 0,
                           W::units(p.shared_inner > 0 ? std::min(p.inner, p.shared_inner) : p.inner));
  // columns that hold every token serve every expert as they are
  shape.dense = p.tokens <= NB * kWidth;
  static bool done[kMaxDevices] = {};
  if (set_func_attr_once(moe_layer_kernel<F, NB, kWidth>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem, done) !=
      HCA_OK)
    return HCA_E_CUDA;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sms);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem_bytes<F, NB, kWidth>(units));
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, moe_layer_kernel<F, NB, kWidth>, p, w, shape));
}

}  // namespace moe

template <int F>
int moe_experts_pass(const MoePass& p, const MoeWeights& w, cudaStream_t s) {
  // Columns of an entry: as many as an expert may get and shared memory holds.
  const int units = WTraits<F>::units(std::max(p.hidden, std::max(p.inner, p.shared_inner)));
  if (p.tokens > 8 && moe::smem_bytes<F, 2, 8>(units) <= moe::kSmem) return moe::launch<F, 2, 8>(p, w, units, s);
  if (p.tokens > 2 && moe::smem_bytes<F, 1, 8>(units) <= moe::kSmem) return moe::launch<F, 1, 8>(p, w, units, s);
  if (moe::smem_bytes<F, 1, 2>(units) <= moe::kSmem) return moe::launch<F, 1, 2>(p, w, units, s);
  return HCA_E_UNSUPPORTED;
}

}  // namespace hca
