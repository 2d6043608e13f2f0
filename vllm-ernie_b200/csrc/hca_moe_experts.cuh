// The second launch of the few-token mixture-of-experts layer.
//
//   h[t, j] = w[t, j] silu(W1_e x_t) * (W3_e x_t),  e = ids[t, j]
//   y[t]    = sum_j W2_e h[t, j]  (+ the shared expert's with weight 1)
//
// Both products go through the chosen experts' weights, each read once for a
// block of columns of the tokens that chose the expert (hca_stream.cuh).  A CTA of
// 16 warps takes a contiguous run of (expert, 16 rows) tiles, so that it meets
// few experts and lays out their columns in shared memory once.  The second
// product leaves each (token, slot) pair's share of y in 32 bits, and the last
// step adds a token's shares in the order of its slots: no atomics, and a
// token's result depends on how many others are in the batch, not on which.  h,
// its weight included, is kept as two bf16 numbers, rounded and rest: with one,
// results were 1.4 to 1.6 times as far from the definition as with 32 bits
// between the products (0.0024 for 0.0017, the rounding of the result itself),
// for 5 to 7 % less time with more than four tokens and none with fewer.
//
// One launch with two grid barriers, since each of the steps is short at one
// token: the weights of the second product start on their way before the
// barrier that its activations wait for.
//
// Measured, router and all, and the rate by the bytes of the chosen experts: e4m3,
// 8 tokens, 8 of 128 experts (41 different ones), 4096 x 1024 and a shared one: 122
// us, 4.4 TB/s; bf16, one token, 6 of 64: 37.6 us, 4.0 TB/s; 4-bit, 59 tokens, 8 of
// 128 (83): 192 us, 2.8 TB/s, since experts with more than eight tokens are read
// for each eight (649 MB instead of 547).  Bound by latency at 16 warps an SM:
// waiting for loads and at the groups' barriers, no pipe above two thirds.
// Of a small layer's 18 us (4-bit, 2 tokens, 4 of 32, 1024 x 512), 3 are the
// router, 3 the plan, 3 1/2 the starts of the products, 6 the products and 2 1/2
// the barriers.
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
constexpr int kParts = 2;  // bf16 numbers that an h is kept as
constexpr int64_t kPrefetch = 256 * 1024;  // weights of a CTA on their way into L2 at the grid barrier
static_assert(kWarps * 64 > kMoeExperts, "the plan's lanes hold two experts each");

// Who computes what, made by every CTA from the ids (at most 1024 of them) in
// shared memory.  A pair is t * top_k + j; the shared expert's are tokens *
// top_k + t.  An id that repeats in a token counts once, with the weights'
// sum.  An entry is up to `columns` pairs of one expert, so that every entry's
// weights cost one pass; entries are in the experts' order, the shared expert
// (number `experts`) last, and pairs in the tokens'.
template <int kColumns>
struct Plan {
  static constexpr int kEntries = kColumns == 1 ? kMoePairs : kMoeExperts + 1 + kMoePairs / kColumns;
  int entries, routed;          // with and without the shared expert's
  int16_t expert[kEntries];     // entry -> expert
  int16_t start[kEntries + 1];  // entry -> first pair
  int16_t pair[kMoePairs];
  int16_t id[kMoePairs];  // pair -> expert, or -1
  float weight[kMoePairs];
  uint64_t who[kMoeExperts + 1];  // expert -> its tokens
  int16_t list[kMoeExperts + 1];  // expert -> first pair
  int sums[kWarps];               // of 64 experts: pairs, and entries from bit 16 on
  int nan;                        // e4m3: a tile of the segment has one
};

template <int kColumns>
__device__ __forceinline__ void build_plan(Plan<kColumns>& pl, const MoePass& p) {
  const int lane = threadIdx.x & 31, top_k = p.routing.top_k, experts = p.routing.experts;
  const int routed = p.tokens * top_k, n = routed + p.tokens;
  const uint8_t* mask = p.routing.mask;
#pragma unroll 1
  for (int e = threadIdx.x; e < experts; e += kThreads) pl.who[e] = 0;
  if (p.logits != nullptr) {
    choose_all(p.logits, p.routing, threadIdx.x >> 5, kWarps, p.tokens, [&](int t, int id, float weight) {
      pl.id[t * top_k + lane] = static_cast<int16_t>(id);
      pl.weight[t * top_k + lane] = weight;
    });
  } else {
#pragma unroll 1
    for (int i = threadIdx.x; i < routed; i += kThreads) {
      const int t = i / top_k;
      const int32_t* ids = p.ids + static_cast<int64_t>(t) * top_k;
      const float* weights = p.weights + static_cast<int64_t>(t) * top_k;
      const int j = i - t * top_k, e = ids[j];
      bool in = e >= 0 && e < experts && (mask == nullptr || mask[t]);
      float weight = 0.0f;
#pragma unroll 1
      for (int o = 0; o < top_k; ++o) {
        if (ids[o] != e) continue;
        if (o < j) in = false;
        weight += weights[o];
      }
      pl.id[i] = static_cast<int16_t>(in ? e : -1);
      pl.weight[i] = weight;
    }
  }
  if (threadIdx.x == 0) pl.nan = 0;
  if (threadIdx.x < kMoeTokens) {
    const int t = threadIdx.x;
    const bool in = t < p.tokens && p.shared_inner > 0 && (mask == nullptr || mask[t]);
    const uint32_t half = __ballot_sync(0xffffffffu, in);
    if (lane == 0) reinterpret_cast<uint32_t*>(&pl.who[experts])[t / 32] = half;
    if (t < p.tokens) {
      pl.id[routed + t] = static_cast<int16_t>(in ? experts : -1);
      pl.weight[routed + t] = 1.0f;
    }
  }
  __syncthreads();
  auto token = [&](int i) { return i < routed ? i / top_k : i - routed; };
#pragma unroll 1
  for (int i = threadIdx.x; i < routed; i += kThreads)
    if (pl.id[i] >= 0) atomicOr(reinterpret_cast<unsigned long long*>(&pl.who[pl.id[i]]), 1ull << token(i));
  __syncthreads();
  {
    // pairs and entries before each expert, two experts a lane
    const int warp = threadIdx.x >> 5, e0 = warp * 64 + 2 * lane;
    auto pieces = [](int c) { return (c + kColumns - 1) / kColumns; };
    int c[2], own = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      c[i] = e0 + i <= experts ? __popcll(pl.who[e0 + i]) : 0;
      own += c[i] | pieces(c[i]) << 16;
    }
    int at = own;  // inclusive sums of both
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += v;
    }
    if (lane == 31) pl.sums[warp] = at;
    __syncthreads();
    const int other = lane < kWarps ? pl.sums[lane] : 0;
    at += static_cast<int>(__reduce_add_sync(0xffffffffu, lane < warp ? other : 0)) - own;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int e = e0 + i, first = at & 0xffff, entry = at >> 16;
      if (c[i] > 0) pl.list[e] = static_cast<int16_t>(first);
#pragma unroll 1
      for (int j = 0; j < pieces(c[i]); ++j) {
        pl.expert[entry + j] = static_cast<int16_t>(e);
        pl.start[entry + j] = static_cast<int16_t>(first + j * kColumns);
      }
      if (e == experts) pl.routed = entry;
      at += c[i] | pieces(c[i]) << 16;
    }
    const int all = static_cast<int>(__reduce_add_sync(0xffffffffu, other));
    if (threadIdx.x == 0) pl.entries = all >> 16, pl.start[all >> 16] = static_cast<int16_t>(all & 0xffff);
  }
  __syncthreads();
#pragma unroll 1
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int e = pl.id[i];
    if (e >= 0) pl.pair[pl.list[e] + __popcll(pl.who[e] & ((1ull << token(i)) - 1))] = static_cast<int16_t>(i);
  }
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

struct Shape {
  int up_warps, down_warps;  // warps that share a tile of either product
  int dense;                 // the first product's columns are the tokens, the same for every expert
  int room;                  // bytes for columns
};

// Columns of the products.  h comes in two parts: where a block has room for
// them the second parts are columns of their own, kWidth after the first, and
// cost no product; else each weight's fragment meets both.
template <int F, int NB, int kWidth, bool kUp>
struct Columns {
  static constexpr bool kBeside = !kUp && kWidth < 8;
  using X = XTile<F, __nv_bfloat16, NB, kBeside ? 2 * kWidth : kWidth, kUp || kBeside ? 1 : kParts>;
};

// One of the products over this CTA's run of (entry, tile) items.  kUp: h from
// x (fragment rows 0..7 of a tile are gate rows, 8..15 the up rows of the same
// inner columns, so a lane holds both factors); else part from h.
template <int F, int NB, int kWidth, bool kUp>
struct Product {
  using W = WTraits<F>;
  static constexpr bool kBeside = Columns<F, NB, kWidth, kUp>::kBeside;
  using X = typename Columns<F, NB, kWidth, kUp>::X;
  using P = Plan<NB * kWidth>;
  const MoePass& p;
  const MoeWeights& w;
  P& pl;
  uint8_t *smem, *scale_smem;
  int room;  // bytes for columns
  TileGroup g;
  bool dense;
  int per_cta, tiles, pairs, from, to, end;  // [from, to) is the segment
  int first_entry;
  // a tile of the segment: this group's first, next to load, next to fetch
  // scales of, and now consumed
  struct Place {
    int entry, tile;
  } first, loading, fetching, now;

  __device__ __forceinline__ Product(const MoePass& p_, const MoeWeights& w_, P& pl_, uint8_t* smem_, int room_,
                                     uint8_t* scale_smem_, int warps, bool dense_)
      : p(p_), w(w_), pl(pl_), smem(smem_), scale_smem(scale_smem_), room(room_), g(warps), dense(dense_) {
    per_cta = kWarps / g.warps;
    tiles = kUp ? p.inner / 8 : p.hidden / 16;  // of a routed entry
    pairs = p.tokens * p.routing.top_k;
    const int shared_tiles = kUp ? p.shared_inner / 8 : tiles;
    // Even shares of the units to read: a tile costs its reduction length.  (At
    // most 1100 entries of a few thousand tiles of a few hundred units.)
    const uint32_t cost = W::units(kUp ? p.hidden : p.inner), shared_cost = kUp || p.shared_inner == 0 ? cost : W::units(p.shared_inner);
    const uint32_t routed_items = pl.routed * tiles, routed_cost = routed_items * cost;
    const uint32_t all = routed_cost + (pl.entries - pl.routed) * shared_tiles * shared_cost;
    auto boundary = [&](uint32_t block) -> int {
      const uint32_t at = all / gridDim.x * block + all % gridDim.x * block / gridDim.x;
      return at < routed_cost ? at / cost : routed_items + (at - routed_cost) / shared_cost;
    };
    from = to = boundary(blockIdx.x);
    end = boundary(blockIdx.x + 1);
  }
  __device__ __forceinline__ int tiles_of(int entry) const { return kUp && entry >= pl.routed ? p.shared_inner / 8 : tiles; }
  __device__ __forceinline__ int k_of(int entry) const {
    return kUp ? p.hidden : entry >= pl.routed ? p.shared_inner : p.inner;
  }
  __device__ __forceinline__ void move(Place& at, int by) const {
    at.tile += by;
#pragma unroll 1
    for (int n = tiles_of(at.entry); at.tile >= n && at.entry + 1 < pl.entries; n = tiles_of(at.entry)) at.tile -= n, ++at.entry;
  }
  // The matrix of a tile's rows, and the number of its fragment row r.
  __device__ __forceinline__ const MoeMatrix& matrix(const Place& at, int64_t& e) const {
    const bool shared = at.entry >= pl.routed;
    e = shared ? 0 : pl.expert[at.entry];
    return kUp ? (shared ? w.shared13 : w.w13) : (shared ? w.shared2 : w.w2);
  }
  __device__ __forceinline__ int rows_of(int entry) const {
    return kUp ? 2 * (entry >= pl.routed ? p.shared_inner : p.inner) : p.hidden;
  }
  __device__ __forceinline__ int row(const Place& at, int r) const {
    if (!kUp) return at.tile * 16 + r;
    return at.tile * 8 + (r < 8 ? r : r - 8 + rows_of(at.entry) / 2);
  }
  // What the stream asks of its source.
  __device__ __forceinline__ TileRows rows(int i) {
    if (i > 0) move(loading, per_cta);
    int64_t e;
    const MoeMatrix& m = matrix(loading, e);
    const int n = rows_of(loading.entry), k = k_of(loading.entry), lane = threadIdx.x & 31;
    TileRows t;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int at = row(loading, (lane >> 2) + 8 * r);
      t.data[r] = m.data + (e * n + at) * W::row_bytes(k) + (lane & 3) * 16;
      if constexpr (F == kWFp8)
        t.scale[r] = static_cast<const float*>(m.scale) + (e * ((n + 127) / 128) + at / 128) * ((k + 127) / 128);
    }
    return t;
  }
  __device__ __forceinline__ bool zeros() const { return (kUp ? w.w13.zero : w.w2.zero) != nullptr; }
  __device__ __forceinline__ bool rows_wide() const {
    const MoeMatrix &m = kUp ? w.w13 : w.w2, &one = kUp ? w.shared13 : w.shared2;
    const int groups = k_of(first_entry) / W::kGroupK;
    // of one segment all entries are the experts' or the shared one's
    return dense || first_entry < pl.routed ? scales_wide(m.scale, m.zero, groups) &&
                                                  (!dense || p.shared_inner == 0 || scales_wide(one.scale, one.zero, groups))
                                            : scales_wide(one.scale, one.zero, groups);
  }
  __device__ __forceinline__ WScales scales_of(const Place& at, int r) const {
    int64_t e;
    const MoeMatrix& m = matrix(at, e);
    const int n = rows_of(at.entry), k = k_of(at.entry);
    const uint8_t* s = static_cast<const uint8_t*>(m.scale);
    const int groups = k / W::kGroupK;
    const int64_t first_group = (e * n + row(at, r)) * groups;
    const int64_t all = static_cast<int64_t>(at.entry >= pl.routed ? 1 : p.routing.experts) * n * groups;
    return {s + 2 * first_group, s + 2 * all, m.zero == nullptr ? nullptr : m.zero + first_group, m.zero + all};
  }
  __device__ __forceinline__ WScales scales(int i, int r) {
    if (i > 0) move(fetching, per_cta);
    return scales_of(fetching, r);
  }
  __device__ __forceinline__ WScales here(int, int r) const { return scales_of(now, r); }
  __device__ __forceinline__ void met_nan() { pl.nan = 1; }

  __device__ __forceinline__ __nv_bfloat16* h_row(int pair) const {
    return p.h + kParts * (pair < pairs ? static_cast<int64_t>(pair) * p.inner
                                        : static_cast<int64_t>(pairs) * p.inner + static_cast<int64_t>(pair - pairs) * p.shared_inner);
  }
  __device__ __forceinline__ int token(int pair) const { return pair < pairs ? pair / p.routing.top_k : pair - pairs; }

  // Starts the loads of the next segment, the run of tiles that one layout of
  // columns serves: with dense columns all, else those of as many entries as
  // shared memory holds the columns of (of one reduction length).
  template <typename Stream>
  __device__ __forceinline__ bool start(Stream& stream) {
    from = to;
    if (from >= end) return false;
    const int routed_items = pl.routed * tiles;
    int tile;
    if (from < routed_items) first_entry = from / tiles, tile = from - first_entry * tiles;
    else {
      const int n = tiles_of(pl.routed);
      first_entry = (from - routed_items) / n, tile = from - routed_items - first_entry * n;
      first_entry += pl.routed;
    }
    to = end;
    if (!dense) {
      const int hold = max(1, room / static_cast<int>(X::bytes(W::units(k_of(first_entry)))));
      to = min(end, from - tile + hold * tiles_of(first_entry));
      if (first_entry < pl.routed) to = min(to, routed_items);
    }
    first = {first_entry, tile};
    move(first, g.id);
    loading = fetching = now = first;
    const int k = k_of(first_entry);
    stream.start(k, g, to - from > g.id ? (to - from - g.id + per_cta - 1) / per_cta : 0, scale_smem, *this, W::units(k));
    return true;
  }

  // The segment's first weights into L2, by one thread.
  __device__ __forceinline__ void prefetch() const {
    const int tile = first.tile - g.id;  // thread 0's group
    int64_t e;
    const MoeMatrix& m = matrix(first, e);
    const int64_t row = W::row_bytes(k_of(first_entry));
    const int n = min(to - from, tiles - tile);
    if (n > 0) prefetch_weights(m.data + (e * p.hidden + tile * 16) * row, min(n * 16 * row, kPrefetch));
  }

  // Lays out the segment's columns and consumes its tiles.  Both ends are
  // block barriers for the columns.
  template <typename Stream>
  __device__ __forceinline__ void run(Stream& stream, TileSums<NB>& ts) {
    ts.half = 0;  // groups of other warps may have taken another number of tiles
    const int k = k_of(first_entry);
    const int64_t tile_bytes = X::bytes(W::units(k));
    Place end_at = {first_entry, 0};
    if (!dense) {
      // the segment's last entry
      end_at.tile = to - 1 - (first_entry < pl.routed ? first_entry * tiles : pl.routed * tiles + (first_entry - pl.routed) * tiles_of(pl.routed));
      move(end_at, 0);
    }
    int most = 0;  // blocks of columns of an entry
#pragma unroll 1
    for (int entry = first_entry; entry <= end_at.entry; ++entry) {
      const int l0 = pl.start[entry];
      const int columns = dense ? p.tokens : pl.start[entry + 1] - l0;
      most = max(most, (columns + kWidth - 1) / kWidth);
    }
#pragma unroll 1
    for (int entry = first_entry; entry <= end_at.entry; ++entry) {
      const int l0 = pl.start[entry];
      X xt(smem + (entry - first_entry) * tile_bytes, W::units(k));
      const int n = dense ? p.tokens : pl.start[entry + 1] - l0;
      xt.stage(k, kBeside ? kWidth + n : n, most, [&](int col) -> const __nv_bfloat16* {
        if (kUp && dense)
          return p.routing.mask == nullptr || p.routing.mask[col] ? p.x + col * p.x_stride : nullptr;
        if (kBeside && col % kWidth >= n) return nullptr;
        const int pair = pl.pair[l0 + (kBeside ? col % kWidth : col)];
        return kUp ? p.x + token(pair) * p.x_stride : h_row(pair) + (kBeside && col >= kWidth ? k : 0);
      });
    }
    X xt(smem, W::units(k));
    auto select = [&]() {
      if (!dense) xt = X(smem + (now.entry - first_entry) * tile_bytes, W::units(k));
    };
    select();
    float acc[NB][4] = {};
    auto finish = [&](int, const float* sums) {
      constexpr int kCols = kUp ? 8 : 16;
      const int s0 = pl.start[now.entry], n = (pl.start[now.entry + 1] - s0) * kCols;
#pragma unroll 1
      for (int i = g.thread(); i < n; i += g.threads()) {
        const int pair = pl.pair[s0 + i / kCols], c = i % kCols;
        const int col = dense ? token(pair) : i / kCols;
        float v = TileSums<NB>::sum(sums, g, c, col / kWidth, col % kWidth) * Scaling<F, __nv_bfloat16>::kOut;
        if (kBeside) v += TileSums<NB>::sum(sums, g, c, 0, kWidth + col) * Scaling<F, __nv_bfloat16>::kOut;
        if (kUp) {
          const float up = TileSums<NB>::sum(sums, g, c + 8, col / kWidth, col % kWidth) * Scaling<F, __nv_bfloat16>::kOut;
          const float h = __fdividef(v, 1.0f + __expf(-v)) * up * pl.weight[pair];
          __nv_bfloat16* to = h_row(pair) + now.tile * 8 + c;
          const __nv_bfloat16 first = __float2bfloat16_rn(h);
          *to = first;
          const float rest = h - __bfloat162float(first);
          to[now.entry >= pl.routed ? p.shared_inner : p.inner] = __float2bfloat16_rn(isfinite(rest) ? rest : 0.0f);
        } else {
          p.part[static_cast<int64_t>(pair) * p.hidden + now.tile * 16 + c] = v;
        }
      }
      move(now, per_cta);
      select();
    };
    if (NB > 1 && most == 1) stream.template run<1>(xt, g, ts, acc, *this, finish);
    else stream.template run<NB>(xt, g, ts, acc, *this, finish);
    __syncthreads();
    if (F == kWFp8 && pl.nan) spread_nans(stream.count);
  }

  // Looks for the NaN among the segment's e4m3 weights, a warp to a row, and
  // makes what came of their rows NaN.  Ends with a block barrier.
  __device__ __forceinline__ void spread_nans(int count) {
    const int lane = threadIdx.x & 31, k = k_of(first_entry);
    Place at = first;
#pragma unroll 1
    for (int i = 0; i < count; ++i, move(at, per_cta)) {
      int64_t e;
      const MoeMatrix& m = matrix(at, e);
#pragma unroll 1
      for (int r = g.index; r < 16; r += g.warps) {
        const uint8_t* from = m.data + (e * rows_of(at.entry) + row(at, r)) * k;
        uint32_t nans = 0;
#pragma unroll 1
        for (int b = lane * 4; b < k; b += 128) {
          const uint32_t v = *reinterpret_cast<const uint32_t*>(from + b);
          nans |= (v ^ (v + 0x01010101u)) & 0x80808080u;
        }
        if (!__any_sync(0xffffffffu, nans)) continue;
#pragma unroll 1
        for (int j = pl.start[at.entry] + lane; j < pl.start[at.entry + 1]; j += 32) {
          const int pair = pl.pair[j];
          if (kUp) h_row(pair)[at.tile * 8 + r % 8] = __float2bfloat16_rn(NAN);
          else p.part[static_cast<int64_t>(pair) * p.hidden + at.tile * 16 + r] = NAN;
        }
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) pl.nan = 0;
    __syncthreads();
  }
};

template <int F, int NB, int kWidth>
__global__ void __launch_bounds__(kThreads, 1)
    moe_layer_kernel(MoePass p, MoeWeights w, Shape shape) {
  __shared__ Plan<NB * kWidth> pl;
  static_assert(sizeof(pl) + kSmem <= 227 * 1024, "shared memory of a block");
  extern __shared__ __align__(16) uint8_t smem[];
  build_plan(pl, p);
  TileStream<F, __nv_bfloat16, WTraits<F>::step(NB)> stream;
  const int room = shape.room;
  uint8_t* sums = smem + room;
  TileSums<NB> ts(sums);
  uint8_t* scales = sums + TileSums<NB>::bytes(kWarps);
  {
    Product<F, NB, kWidth, true> up(p, w, pl, smem, room, scales, shape.up_warps, shape.dense);
    while (up.start(stream)) up.run(stream, ts);
  }
  grid_arrive(p.barrier);
  {
    Product<F, NB, kWidth, false> down(p, w, pl, smem, room, scales, shape.down_warps, false);
    bool more = down.start(stream);
    // bf16 weights come slower than they are used, so they go on coming while
    // the CTAs meet (38.8 -> 37.9 us at one token; 4-bit and e4m3 lost 0.5 %)
    if (F == kWBf16 && more && threadIdx.x == 0) down.prefetch();
    if (!grid_wait(p.barrier, 1, p.error)) {
      asm volatile("cp.async.wait_all;\n" ::: "memory");
      return;
    }
    while (more) {
      down.run(stream, ts);
      more = down.start(stream);
    }
  }
  grid_arrive(p.barrier);
  if (!grid_wait(p.barrier, 2, p.error)) return;
  // y: a token's shares, in the order of its slots, four columns a thread
  const int quads = p.hidden / 4, top_k = p.routing.top_k;
#pragma unroll 1
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

// Launches with entries of NB blocks of kWidth columns if shared memory holds them.
template <int F, int NB, int kWidth>
bool launch(const MoePass& p, const MoeWeights& w, cudaStream_t s, int& rc) {
  using W = WTraits<F>;
  const int sms = device_sm_count();
  const int inner = std::max(p.inner, p.shared_inner);
  // the shares of the work are counted in 32 bits: every pair an entry at most
  const int64_t units = std::max(static_cast<int64_t>(inner / 8) * W::units(p.hidden),
                                 static_cast<int64_t>(p.hidden / 16) * W::units(inner));
  if (units * p.tokens * (p.routing.top_k + 1) > UINT32_MAX) return false;
  Shape shape;
  shape.room = static_cast<int>(std::max(Columns<F, NB, kWidth, true>::X::bytes(W::units(p.hidden)),
                                         Columns<F, NB, kWidth, false>::X::bytes(W::units(inner))));
  // Columns of h of the experts that a CTA's run meets, as long as they are
  // small: a second layout costs a small layer 3 us of 18, but loads on their
  // way need what shared memory leaves of L1.
  const int64_t meets = cdiv(std::min(p.routing.experts, p.tokens * p.routing.top_k), sms) + 1;
  const int64_t met = meets * Columns<F, NB, kWidth, false>::X::bytes(W::units(p.inner));
  shape.room = static_cast<int>(std::max<int64_t>(shape.room, std::min<int64_t>(met, 64 * 1024)));
  const int64_t columns = shape.room + TileSums<NB>::bytes(kWarps);
  const bool zeros = w.w13.zero != nullptr || w.w2.zero != nullptr;
  auto scales = [&](int k, int warps) { return ScaleTile<F>::bytes(W::units(k), zeros, warps, kWarps); };
  // Warps to a tile: the number that makes the longest warp's work shortest (if
  // every pair chose another expert).  Runs begin and end inside an expert, so a
  // round more than the average has to be counted; a tile's end costs half of
  // what a quad of units does, and more the more warps meet there.  (e4m3, rows
  // of 4096, 56 tiles a CTA: 122 us with one warp, 114 with two, 113 with four,
  // 115 with eight; 4-bit, 112 tiles: 192, 188, 198, 240.)
  auto warps = [&](int64_t tiles, int64_t shared_tiles, int k, int least_k) {
    const int64_t n = std::min(p.routing.experts, p.tokens * p.routing.top_k) * tiles + shared_tiles;
    int best = 0;
    double least = INFINITY;
    // (no more than the shorter rows have quads, unless scales need the room)
    for (int gw = 1; gw <= kWarps && (4 * gw <= W::units(least_k) || best == 0); gw *= 2) {
      const double rounds = static_cast<double>(n) * gw / (kWarps * sms) + 1, quads = W::units(k) / (4.0 * gw);
      const double cost = rounds * (quads + 0.5 + gw / 64.0);
      if (cost < least && columns + scales(k, gw) <= kSmem) least = cost, best = gw;
    }
    return best;
  };
  shape.up_warps = warps(p.inner / 8, p.shared_inner / 8, p.hidden, p.hidden);
  shape.down_warps = warps(p.hidden / 16, p.shared_inner > 0 ? p.hidden / 16 : 0, inner,
                           p.shared_inner > 0 ? std::min(p.inner, p.shared_inner) : p.inner);
  // columns that hold every token serve every expert as they are
  shape.dense = p.tokens <= NB * kWidth;
  if (shape.up_warps == 0 || shape.down_warps == 0) return false;
  const int64_t smem = columns + std::max(scales(p.hidden, shape.up_warps), scales(inner, shape.down_warps));
  static bool done[kMaxDevices] = {};
  rc = set_func_attr_once(moe_layer_kernel<F, NB, kWidth>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem, done);
  if (rc != HCA_OK) return true;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sms);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  rc = cuda_status(cudaLaunchKernelEx(&cfg, moe_layer_kernel<F, NB, kWidth>, p, w, shape));
  return true;
}

}  // namespace moe

template <int F>
int moe_experts_pass(const MoePass& p, const MoeWeights& w, cudaStream_t s) {
  // Columns of an entry, where shared memory holds them: two blocks of eight if
  // an expert gets more than eight tokens on average, or all tokens fit and it
  // gets more than two; else one, which an expert with more tokens passes
  // several times (with h in one part, at 64 tokens, four an expert, 188 us for 226
  // with 4-bit weights, 96 for 106 with e4m3; at 12 tokens, three an expert, 40 for 34 and
  // 47 for 41).  bf16 weights, with nothing to unpack, gain from two blocks
  // whenever there are more than eight tokens (58 us for 47 at 12 tokens).
  int rc = HCA_OK;
  const int64_t pairs = static_cast<int64_t>(p.tokens) * p.routing.top_k;
  const bool many = F == kWBf16 || pairs > static_cast<int64_t>(p.routing.experts) * (p.tokens <= 16 ? 2 : 8);
  if (p.tokens > 8 && many && moe::launch<F, 2, 8>(p, w, s, rc)) return rc;
  if (p.tokens > 4 && moe::launch<F, 1, 8>(p, w, s, rc)) return rc;
  if (p.tokens > 2 && moe::launch<F, 1, 4>(p, w, s, rc)) return rc;
  if (moe::launch<F, 1, 2>(p, w, s, rc)) return rc;
  // rows so long that shared memory has no room for the parts of two: a pass
  // over an expert's weights for each of its tokens
  if (moe::launch<F, 1, 1>(p, w, s, rc)) return rc;
  return HCA_E_UNSUPPORTED;
}

}  // namespace hca
