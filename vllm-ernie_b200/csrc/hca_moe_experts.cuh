// The expert kernels of the few-token mixture-of-experts layer.
//
//   h[t, j] = w[t, j] silu(W1_e x_t) * (W3_e x_t),  e = ids[t, j]
//   y[t]    = sum_j W2_e h[t, j]  (+ the shared expert's with weight 1)
//
// Both are bound by the bytes of the chosen experts' weights, each read once
// for all tokens that chose the expert (hca_stream.cuh).
//
// The routing weight goes into h, so that the second product can sum over
// (expert, inner) as over one long axis and needs no weights, no atomics and
// no second pass: h is rounded to bf16 once, after the weight, and the sums
// over experts stay in 32 bits.
#pragma once

#include <algorithm>

#include "hca_moe.cuh"
#include "hca_stream.cuh"

namespace hca {
namespace moe {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;

// Who computes what, built by every CTA from ids (at most 1024 of them) in
// shared memory: the experts that some token chose, in ascending order, and
// the (token, slot) pairs of each.  A pair is t * top_k + j; the shared
// expert is a last entry with pairs tokens * top_k + t.
struct Plan {
  int count;                                  // entries
  int16_t expert[kMoeExperts + 1];            // entry -> expert; `experts` = shared
  int16_t start[kMoeExperts + 2];             // entry -> first pair
  int16_t pair[kMoeTokens * (kMoeTopK + 1)];
  int cursor[kMoeExperts + 1];                // by expert, while building
};

__device__ __forceinline__ void build_plan(Plan& pl, const MoePass& p) {
  const int n = p.tokens * p.top_k;
  for (int e = threadIdx.x; e <= p.experts; e += kThreads) pl.cursor[e] = 0;
  __syncthreads();
  auto expert_of = [&](int i) -> int {  // of pair i, or -1
    if (i >= n) return p.shared_inner > 0 && (p.mask == nullptr || p.mask[i - n]) ? p.experts : -1;
    if (p.mask != nullptr && !p.mask[i / p.top_k]) return -1;
    const int e = p.ids[i];
    return e >= 0 && e < p.experts ? e : -1;
  };
  for (int i = threadIdx.x; i < n + p.tokens; i += kThreads) {
    const int e = expert_of(i);
    if (e >= 0) atomicAdd(&pl.cursor[e], 1);
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int entries = 0, pairs = 0;
    for (int e0 = 0; e0 <= p.experts; e0 += 32) {
      const int e = e0 + lane;
      const int c = e <= p.experts ? pl.cursor[e] : 0;
      const unsigned active = __ballot_sync(0xffffffffu, c > 0);
      int before = c;  // inclusive sum of counts
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
      }
      if (c > 0) {
        const int at = entries + __popc(active & ((1u << lane) - 1));
        pl.expert[at] = static_cast<int16_t>(e);
        pl.start[at] = static_cast<int16_t>(pairs + before - c);
        pl.cursor[e] = pairs + before - c;
      }
      entries += __popc(active);
      pairs += __shfl_sync(0xffffffffu, before, 31);
    }
    if (lane == 0) {
      pl.count = entries;
      pl.start[entries] = static_cast<int16_t>(pairs);
    }
  }
  __syncthreads();
  // The order of an expert's pairs may differ from run to run; it only says
  // which column of a product a pair takes, which its values do not depend on.
  for (int i = threadIdx.x; i < n + p.tokens; i += kThreads) {
    const int e = expert_of(i);
    if (e >= 0) pl.pair[atomicAdd(&pl.cursor[e], 1)] = static_cast<int16_t>(i);
  }
  __syncthreads();
}

// Row pointers of rows `row` of matrix `e` (rows_e rows of k) of a stack.
template <int F>
__device__ __forceinline__ void set_row(WRows<__nv_bfloat16>& rows, int r, const MoeMatrix& m, int64_t e, int rows_e,
                                        int row, int k) {
  using W = WTraits<F>;
  const int64_t at = e * rows_e + row;
  rows.data[r] = m.data + at * W::row_bytes(k);
  if constexpr (W::kIs4) {
    const int groups = k / W::kUnitK;
    rows.scale[r] = static_cast<const __nv_bfloat16*>(m.scale) + at * groups;
    rows.zero[r] = m.zero == nullptr ? nullptr : m.zero + at * groups;
  } else if constexpr (F == kWFp8) {
    const int64_t kb = (k + 127) / 128, rb = (rows_e + 127) / 128;
    rows.scale[r] = static_cast<const float*>(m.scale) + (e * rb + row / 128) * kb;
    rows.zero[r] = nullptr;
  } else {
    rows.scale[r] = nullptr;
    rows.zero[r] = nullptr;
  }
}

// h.  A work item is 8 inner columns of one entry: fragment rows 0..7 are
// their gate rows and 8..15 their up rows, so a lane holds both factors.  The
// warps split hidden; items go round the resident CTAs.
template <int F, int NB>
__global__ void __launch_bounds__(kThreads) gate_up_kernel(MoePass p, MoeWeights w) {
  using W = WTraits<F>;
  __shared__ Plan pl;
  __shared__ float red[kWarps][NB * 8][16];
  pdl_wait_and_release();
  build_plan(pl, p);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tiles = p.inner / 8, shared_tiles = p.shared_inner / 8;
  const bool has_shared = pl.count > 0 && pl.expert[pl.count - 1] == p.experts;
  const int routed = pl.count - (has_shared ? 1 : 0);
  const int items = routed * tiles + (has_shared ? shared_tiles : 0);
  const int units = (p.hidden + W::kUnitK - 1) / W::kUnitK;
  const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(p.x);
  const int pairs = p.tokens * p.top_k;

  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int entry = min(item / tiles, routed), tile = item - entry * tiles;
    const bool shared = entry == routed;
    const int inner = shared ? p.shared_inner : p.inner;
    const int e = shared ? 0 : pl.expert[entry];
    const MoeMatrix& m = shared ? w.shared13 : w.w13;
    WRows<__nv_bfloat16> rows;
    const int col = tile * 8 + (lane >> 2);
    set_row<F>(rows, 0, m, e, 2 * inner, col, p.hidden);
    set_row<F>(rows, 1, m, e, 2 * inner, inner + col, p.hidden);
    const int end = pl.start[entry + 1];
    for (int first = pl.start[entry]; first < end; first += 8 * NB) {
      int64_t x_off[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int at = first + 8 * b + (lane >> 2);
        const int i = at < end ? pl.pair[at] : -1;
        x_off[b] = i < 0 ? -1 : (i < pairs ? i / p.top_k : i - pairs) * p.x_stride;
      }
      float acc[NB][4] = {};
      stream_rows<F, __nv_bfloat16, NB>(acc, rows, x, x_off, min(NB, (end - first + 7) / 8), p.hidden,
                                        units * warp / kWarps, units * (warp + 1) / kWarps);
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          red[warp][8 * b + 2 * (lane & 3) + (i & 1)][(lane >> 2) + 8 * (i >> 1)] = acc[b][i];
      __syncthreads();
      for (int i = threadIdx.x; i < 8 * NB * 8; i += kThreads) {
        const int at = first + (i >> 3), c = i & 7;
        if (at >= end) continue;
        float gate = 0.0f, up = 0.0f;
#pragma unroll
        for (int v = 0; v < kWarps; ++v) {
          gate += red[v][i >> 3][c];
          up += red[v][i >> 3][c + 8];
        }
        const int pair = pl.pair[at];
        const float weight = pair < pairs ? p.weights[pair] : 1.0f;
        const float v = gate / (1.0f + expf(-gate)) * up * weight;
        __nv_bfloat16* h = pair < pairs ? p.h + static_cast<int64_t>(pair) * p.inner
                                        : p.h + static_cast<int64_t>(pairs) * p.inner +
                                              static_cast<int64_t>(pair - pairs) * p.shared_inner;
        h[tile * 8 + c] = __float2bfloat16_rn(v);
      }
      __syncthreads();
    }
  }
}

// y.  A CTA owns 16 columns of y for all tokens; its warps split the joined
// (entry, inner) axis evenly.  At the end of an entry a warp adds its columns
// to its own 32-bit [tokens, 16] sums in shared memory, one column after
// another since two may belong to one token; the warps' sums are added in
// warp order.
template <int F, int NB>
__global__ void __launch_bounds__(kThreads) down_kernel(MoePass p, MoeWeights w) {
  using W = WTraits<F>;
  __shared__ Plan pl;
  extern __shared__ float sums[];  // [kWarps][tokens][16]
  // The plan needs what the router wrote: complete, because gate_up released
  // this launch only after its own wait for the router.
  for (int i = threadIdx.x; i < kWarps * p.tokens * 16; i += kThreads) sums[i] = 0.0f;
  build_plan(pl, p);
  pdl_wait_and_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n0 = blockIdx.x * 16;
  const bool has_shared = pl.count > 0 && pl.expert[pl.count - 1] == p.experts;
  const int routed = pl.count - (has_shared ? 1 : 0);
  const int units = (p.inner + W::kUnitK - 1) / W::kUnitK;
  const int shared_units = (p.shared_inner + W::kUnitK - 1) / W::kUnitK;
  const int total = routed * units + (has_shared ? shared_units : 0);
  const int begin = static_cast<int>(static_cast<int64_t>(total) * warp / kWarps);
  const int end = static_cast<int>(static_cast<int64_t>(total) * (warp + 1) / kWarps);
  const int pairs = p.tokens * p.top_k;
  float* mine = sums + warp * p.tokens * 16;

  for (int at = begin; at < end;) {
    const int entry = min(at / units, routed);
    const bool shared = entry == routed;
    const int inner = shared ? p.shared_inner : p.inner;
    const int u0 = at - entry * units;
    const int u1 = min(shared ? shared_units : units, u0 + end - at);
    at += u1 - u0;
    const MoeMatrix& m = shared ? w.shared2 : w.w2;
    const __nv_bfloat16* h = shared ? p.h + static_cast<int64_t>(pairs) * p.inner : p.h;
    WRows<__nv_bfloat16> rows;
#pragma unroll
    for (int r = 0; r < 2; ++r)
      set_row<F>(rows, r, m, shared ? 0 : pl.expert[entry], p.hidden, n0 + 8 * r + (lane >> 2), inner);
    const int last = pl.start[entry + 1];
    for (int first = pl.start[entry]; first < last; first += 8 * NB) {
      int64_t h_off[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int j = first + 8 * b + (lane >> 2);
        const int i = j < last ? pl.pair[j] : -1;
        h_off[b] = i < 0 ? -1 : static_cast<int64_t>(shared ? i - pairs : i) * inner;
      }
      float acc[NB][4] = {};
      const int live = min(NB, (last - first + 7) / 8);
      stream_rows<F, __nv_bfloat16, NB>(acc, rows, h, h_off, live, inner, u0, u1);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        if (b >= live) break;
        for (int col = 0; col < 8 && first + 8 * b + col < last; ++col) {
          if ((lane & 3) == col >> 1) {
            const int i = pl.pair[first + 8 * b + col];
            float* y = mine + (i < pairs ? i / p.top_k : i - pairs) * 16;
            y[lane >> 2] += (col & 1) ? acc[b][1] : acc[b][0];
            y[(lane >> 2) + 8] += (col & 1) ? acc[b][3] : acc[b][2];
          }
          __syncwarp();
        }
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.tokens * 16; i += kThreads) {
    float v = 0.0f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) v += sums[k * p.tokens * 16 + i];
    p.out[(i >> 4) * p.out_stride + n0 + (i & 15)] = __float2bfloat16_rn(v);
  }
}

template <int F, int NB>
int launch(const MoePass& p, const MoeWeights& w, cudaStream_t s) {
  // Work items of gate_up if every pair chose another expert; two CTAs fit an SM.
  const int64_t most = static_cast<int64_t>(std::min(p.experts, p.tokens * p.top_k)) * (p.inner / 8) + p.shared_inner / 8;
  const int grid = static_cast<int>(std::min<int64_t>(std::max<int64_t>(most, 1), 2 * device_sm_count()));
  const int rc = launch_pdl(gate_up_kernel<F, NB>, dim3(grid), dim3(kThreads), 0, s, p, w);
  if (rc != HCA_OK) return rc;
  return launch_pdl(down_kernel<F, NB>, dim3(p.hidden / 16), dim3(kThreads), kWarps * p.tokens * 16 * sizeof(float), s,
                    p, w);
}

}  // namespace moe

template <int F>
int moe_experts_pass(const MoePass& p, const MoeWeights& w, cudaStream_t s) {
  // An expert's pairs are columns, 8 to a block.  With up to 8 tokens one
  // block holds them (unless an id repeats); with more, two blocks hold what
  // most experts get, and an expert that got more is passed over again.
  return p.tokens <= 8 ? moe::launch<F, 1>(p, w, s) : moe::launch<F, 2>(p, w, s);
}

}  // namespace hca
