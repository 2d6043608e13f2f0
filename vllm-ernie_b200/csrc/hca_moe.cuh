// Shared by the kernels of the few-token mixture-of-experts layer.
//
// A call is two launches.  The first computes the router's logits over the
// whole GPU and clears the second's barrier; the second, one CTA an SM,
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
  __nv_bfloat16* h;      // [tokens * top_k, inner], then [tokens, shared_inner]
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

// One warp: the experts of token t.  Lane j < top_k returns with the j-th
// choice and its weight (-1 and 0 for a token that takes no part).
__device__ __forceinline__ void choose_experts(const float* logits, const MoeRouting& r, int t, int& id, float& weight) {
  const int lane = threadIdx.x & 31;
  constexpr int kPer = kMoeExperts / 32;
  const int per = (r.experts + 31) / 32;
  float score[kPer];
  uint32_t key[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (j >= per) break;
    const int e = lane + 32 * j;
    score[j] = e < r.experts ? logits[e] : -INFINITY;
  }
  if (r.sigmoid) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (j >= per) break;
      score[j] = 1.0f / (1.0f + expf(-score[j]));
    }
  } else {
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (j >= per) break;
      m = fmaxf(m, score[j]);
    }
    m = warp_max(m);
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (j >= per) break;
      score[j] = expf(score[j] - m);
      if (lane + 32 * j < r.experts) sum += score[j];
    }
    sum = warp_sum(sum);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (j >= per) break;
      score[j] /= sum;
    }
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (j >= per) break;
    const int e = lane + 32 * j;
    // experts' keys are at least 1 (NaN's), absent and taken ones 0
    key[j] = e < r.experts ? order_key(r.bias == nullptr ? score[j] : score[j] + r.bias[e]) + 1 : 0;
  }
  weight = 0.0f, id = -1;
  for (int c = 0; c < r.top_k; ++c) {
    uint32_t best = 0;
    int at = 0;
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (j >= per) break;
      if (key[j] > best) best = key[j], at = j, s = score[j];
    }
    const uint32_t top = __reduce_max_sync(0xffffffffu, best);
    const uint32_t e = __reduce_min_sync(0xffffffffu, best == top ? static_cast<uint32_t>(at * 32 + lane) : ~0u);
    const float v = __shfl_sync(0xffffffffu, s, e & 31);
    if (lane == static_cast<int>(e & 31)) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (j >= per) break;
        if (j == static_cast<int>(e >> 5)) key[j] = 0;
      }
    }
    if (lane == c) weight = v, id = static_cast<int>(e);
  }
  if (r.renormalize) {
    const float sum = warp_sum(weight);
    weight = sum == 0.0f ? 0.0f : weight / sum;  // every chosen score underflowed: no expert has weight
  }
  weight *= r.scale;
  if (r.mask != nullptr && !r.mask[t]) id = -1, weight = 0.0f;
}

}  // namespace hca
