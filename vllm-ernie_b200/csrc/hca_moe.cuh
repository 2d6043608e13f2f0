// Shared by the kernels of the few-token mixture-of-experts layer.
//
// A call is two launches (above 16 tokens a third between them chooses the
// experts).  The first computes the router's logits over the whole GPU and
// clears the second's barrier; the second, one CTA an SM,
// resident together, chooses the experts, runs both of their products and adds
// up the result, with a grid barrier between the steps.
#pragma once

#include "hca_common.cuh"

namespace hca {

constexpr int kMoeTokens = 64;    // tokens of one pass; more run as further passes
constexpr int kMoeTopK = 16;      // most experts a token may choose
constexpr int kMoeExperts = 512;  // most experts of a layer
constexpr int kMoePairs = kMoeTokens * (kMoeTopK + 1);  // with the shared expert's

// hca_device_error bit of the layer's grid barrier
constexpr int kErrMoe = 1 << 6;

// How a token's experts follow from its logits.
struct MoeRouting {
  const float* bias;    // [experts] or null
  const uint8_t* mask;  // [tokens] or null: tokens with 0 take no part
  int experts, top_k, sigmoid, renormalize;
  float scale;
};

// What the layer needs for one pass of up to kMoeTokens tokens.
struct MoePass {
  const __nv_bfloat16* x;  // [tokens, hidden]
  int64_t x_stride;
  const float* logits;   // [tokens, experts], or null: ids and weights are given
  const int32_t* ids;    // [tokens, top_k], negative or >= experts: skipped
  const float* weights;  // [tokens, top_k]
  __nv_bfloat16* h;      // [tokens * top_k, 2, inner], then [tokens, 2, shared_inner]: rounded, and what that left
  float* part;           // [tokens * (top_k + 1), hidden]: a pair's share of y
  uint32_t* barrier;     // 0 before the launch
  int32_t* error;        // device error word
  __nv_bfloat16* out;    // [tokens, hidden]
  int64_t out_stride;
  MoeRouting routing;
  int tokens, hidden, inner, shared_inner;
};

// One weight matrix per expert, row major.
struct MoeMatrix {
  const uint8_t* data;
  const void* scale;
  const uint8_t* zero;
};

struct MoeWeights {
  MoeMatrix w13, w2, shared13, shared2;
};

// Runs a pass with weights of format F (an hca_stream.cuh WFormat).  One
// instantiation per source file.
template <int F>
int moe_experts_pass(const MoePass& p, const MoeWeights& w, cudaStream_t s);

// Order-preserving key of a float; NaN below everything, -0 as +0.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// One warp: the experts of tokens t0, t0 + step, .. (NT of them, side by side,
// since each choice waits for the one before; tokens from `tokens` on are left
// out).  Lane j < top_k calls store(t, id, weight) for the j-th choice (-1 and 0
// for a token that takes no part).  kPer: experts a lane holds.  The exponential
// is expf: __expf is off by 30 units in the last place for logits 60 apart, and
// near-ties with a bias would fall differently.  __fdividef is within 2 units
// (0 for scores below 2^-126) and takes 0.5 us less than a rounded division.
template <int kPer, int NT, typename Store>
__device__ __forceinline__ void choose_experts(const float* logits, const MoeRouting& r, int t0, int step, int tokens, Store store) {
  const int lane = threadIdx.x & 31;
  float score[NT][kPer], bias[kPer];
  uint32_t key[NT][kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = lane + 32 * j;
    bias[j] = r.bias != nullptr && e < r.experts ? r.bias[e] : 0.0f;
#pragma unroll
    for (int n = 0; n < NT; ++n)
      score[n][j] = e < r.experts ? logits[static_cast<int64_t>(min(t0 + n * step, tokens - 1)) * r.experts + e] : -INFINITY;
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (r.sigmoid) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) score[n][j] = __fdividef(1.0f, 1.0f + expf(-score[n][j]));
    } else {
      float m = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int j = 0; j < kPer; ++j) m = fmaxf(m, score[n][j]);
      m = warp_max(m);
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        score[n][j] = expf(score[n][j] - m);
        if (lane + 32 * j < r.experts) sum += score[n][j];
      }
      sum = 1.0f / warp_sum(sum);
#pragma unroll
      for (int j = 0; j < kPer; ++j) score[n][j] *= sum;
    }
    // experts' keys are at least 1 (NaN's), absent and taken ones 0
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      key[n][j] = lane + 32 * j < r.experts ? order_key(r.bias == nullptr ? score[n][j] : score[n][j] + bias[j]) + 1 : 0;
  }
  float weight[NT];
  int id[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) weight[n] = 0.0f, id[n] = -1;
#pragma unroll 1
  for (int c = 0; c < r.top_k; ++c) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      uint32_t best = 0;
      int at = 0;
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (key[n][j] > best) best = key[n][j], at = j, s = score[n][j];
      const uint32_t top = __reduce_max_sync(0xffffffffu, best);
      const uint32_t e = __reduce_min_sync(0xffffffffu, best == top ? static_cast<uint32_t>(at * 32 + lane) : ~0u);
      const float v = __shfl_sync(0xffffffffu, s, e & 31);
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (static_cast<uint32_t>(lane + 32 * j) == e) key[n][j] = 0;
      if (lane == c) weight[n] = v, id[n] = static_cast<int>(e);
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int t = t0 + n * step;
    float w = weight[n];
    if (r.renormalize) {
      const float sum = warp_sum(w);
      w = sum == 0.0f ? 0.0f : w / sum;  // every chosen score underflowed: no expert has weight
    }
    const bool in = t < tokens && (r.mask == nullptr || r.mask[t]);
    if (lane < r.top_k && t < tokens) store(t, in ? id[n] : -1, in ? w * r.scale : 0.0f);
  }
}

// The experts of tokens t0, t0 + step, .. below `tokens`.
template <typename Store>
__device__ __forceinline__ void choose_all(const float* logits, const MoeRouting& r, int t0, int step, int tokens, Store store) {
  if (r.experts > 128) {
#pragma unroll 1
    for (int t = t0; t < tokens; t += step) choose_experts<kMoeExperts / 32, 1>(logits, r, t, step, tokens, store);
  } else {
#pragma unroll 1
    for (int t = t0; t < tokens; t += step) choose_experts<4, 1>(logits, r, t, step, tokens, store);
  }
}

}  // namespace hca
