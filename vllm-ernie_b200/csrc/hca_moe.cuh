// Shared by the router and the expert kernels of the few-token
// mixture-of-experts layer.
#pragma once

#include "hca_common.cuh"

namespace hca {

constexpr int kMoeTokens = 64;    // tokens of one pass; more run as further passes
constexpr int kMoeTopK = 16;      // most experts a token may choose
constexpr int kMoeExperts = 512;  // most experts of a layer

// What the expert kernels need for one pass of up to kMoeTokens tokens.
struct MoePass {
  const void* x;  // bf16 [tokens, hidden]
  int64_t x_stride;
  const int32_t* ids;     // [tokens, top_k], negative or >= experts: skipped
  const float* weights;   // [tokens, top_k]
  const uint8_t* mask;    // [tokens] or null: tokens with 0 take no part
  __nv_bfloat16* h;       // [tokens * top_k, inner], then [tokens, shared_inner]
  __nv_bfloat16* out;     // [tokens, hidden]
  int64_t out_stride;
  int tokens, top_k, experts, hidden, inner, shared_inner;
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

// Runs the two expert kernels of a pass with weights of format F (an
// hca_stream.cuh WFormat).  One instantiation per source file.
template <int F>
int moe_experts_pass(const MoePass& p, const MoeWeights& w, cudaStream_t s);

}  // namespace hca
