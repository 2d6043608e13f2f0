// The router of the few-token mixture-of-experts layer, and its C entries.
//
//   l[t, e] = x_t . Wr_e;  p = softmax(l) or 1 / (1 + exp(-l))
//   ids[t] = the top_k largest of p + bias, ties to the lower expert
//   weights[t, j] = p[t, ids[t, j]] (/ their sum) * scale
//
// Latency-bound (E * hidden weights, a few MB at most): a cluster of eight
// CTAs handles up to eight tokens.  Each CTA computes an eighth of the experts
// for all of them, in 32-bit multiply-adds (a bf16 tensor product would make
// near-ties of a 32-bit router fall differently), sends each token's logits to
// the CTA of that token over distributed shared memory, and one warp there
// picks the experts.  Nothing is counted in global memory, so nothing has to
// be cleared between calls and calls on several streams do not meet.
#include "hca_moe.cuh"
#include "hca_stream.cuh"

#include <algorithm>
#include <cooperative_groups.h>

namespace hca {
namespace {

namespace cg = cooperative_groups;

constexpr int kCluster = 8;
constexpr int kWarps = 8;
constexpr int kGroup = 4;  // experts of a warp at a time

template <typename WT>
__device__ __forceinline__ void load8(float (&v)[8], const WT* p) {
  if constexpr (sizeof(WT) == 2) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
}

// Order-preserving key of a float; NaN below everything.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0;
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 orders as +0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <typename WT, int TB>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kWarps * 32)
    moe_route_kernel(int32_t* ids, float* weights, const __nv_bfloat16* x, int64_t x_stride, const WT* router,
                     const float* bias, const uint8_t* mask, int tokens, int experts, int hidden, int top_k,
                     int sigmoid, int renormalize, float scale) {
  __shared__ float part[kWarps][kMoeExperts / kCluster * TB];  // [warp][expert of the CTA * TB + token]
  __shared__ float logits[kMoeExperts];                        // of this CTA's token
  pdl_wait_and_release();
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t0 = blockIdx.x / kCluster * TB;
  const int per = (experts + kCluster - 1) / kCluster;
  const int e0 = rank * per, mine = max(0, min(per, experts - e0));

  // warps split hidden in steps of 256 (8 values a lane)
  const int steps = (hidden + 255) / 256;
  const int s0 = steps * warp / kWarps, s1 = steps * (warp + 1) / kWarps;
  for (int g = 0; g < mine; g += kGroup) {
    float acc[kGroup][TB] = {};
    for (int s = s0; s < s1; ++s) {
      const int k = s * 256 + lane * 8;
      if (k >= hidden) break;  // hidden is a multiple of 8
      float wv[kGroup][8];
#pragma unroll
      for (int i = 0; i < kGroup; ++i)
        load8(wv[i], router + static_cast<int64_t>(e0 + min(g + i, mine - 1)) * hidden + k);
#pragma unroll
      for (int t = 0; t < TB; ++t) {
        float xv[8];
        load8(xv, x + min(t0 + t, tokens - 1) * x_stride + k);
#pragma unroll
        for (int i = 0; i < kGroup; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[i][t] = fmaf(xv[j], wv[i][j], acc[i][t]);
      }
    }
#pragma unroll
    for (int i = 0; i < kGroup; ++i)
#pragma unroll
      for (int t = 0; t < TB; ++t) {
        const float v = warp_sum(acc[i][t]);
        if (lane == 0 && g + i < mine) part[warp][(g + i) * TB + t] = v;
      }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < mine * TB; i += kWarps * 32) {
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += part[w][i];
    *cluster.map_shared_rank(&logits[e0 + i / TB], i % TB) = v;
  }
  cluster.sync();  // every logit has arrived; no CTA touches another's memory after this

  const int t = t0 + rank;
  if (warp != 0 || rank >= TB || t >= tokens) return;
  constexpr int kPer = kMoeExperts / 32;
  float score[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = lane + 32 * j;
    score[j] = e < experts ? logits[e] : -INFINITY;
  }
  if (sigmoid) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) score[j] = 1.0f / (1.0f + expf(-score[j]));
  } else {
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kPer; ++j) m = fmaxf(m, score[j]);
    m = warp_max(m);
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (lane + 32 * j < experts) {
        score[j] = expf(score[j] - m);
        sum += score[j];
      }
    }
    sum = warp_sum(sum);
#pragma unroll
    for (int j = 0; j < kPer; ++j) score[j] /= sum;
  }
  uint32_t key[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = lane + 32 * j;
    // 0 is NaN's key, so real experts take key + 1 (no key is 2^32 - 1: that would be a NaN's) and taken or absent ones 0
    key[j] = e < experts ? order_key(bias == nullptr ? score[j] : score[j] + bias[e]) + 1 : 0;
  }
  float chosen = 0.0f;  // lane j: the j-th choice's score
  int chosen_id = -1;
  for (int c = 0; c < top_k; ++c) {
    uint32_t best = 0;
    int at = 0;
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (key[j] > best) best = key[j], at = j, s = score[j];
    const uint32_t top = __reduce_max_sync(0xffffffffu, best);
    const uint32_t e = __reduce_min_sync(0xffffffffu, best == top ? static_cast<uint32_t>(at * 32 + lane) : ~0u);
    const float v = __shfl_sync(0xffffffffu, s, e & 31);
    if (lane == static_cast<int>(e & 31)) {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (j == static_cast<int>(e >> 5)) key[j] = 0;
    }
    if (lane == c) chosen = v, chosen_id = static_cast<int>(e);
  }
  float w = chosen;
  if (renormalize) {
    const float sum = warp_sum(lane < top_k ? chosen : 0.0f);
    w = sum == 0.0f ? 0.0f : chosen / sum;  // every chosen score underflowed: no expert has weight
  }
  if (lane < top_k) {
    const bool in = mask == nullptr || mask[t] != 0;
    ids[t * top_k + lane] = in ? chosen_id : -1;
    weights[t * top_k + lane] = in ? w * scale : 0.0f;
  }
}

template <typename WT, int TB>
int launch_route(int32_t* ids, float* weights, const void* x, int64_t x_stride, const void* router, const float* bias,
                 const uint8_t* mask, int tokens, int experts, int hidden, int top_k, int sigmoid, int renormalize,
                 float scale, cudaStream_t s) {
  return launch_pdl(moe_route_kernel<WT, TB>, dim3(cdiv(tokens, TB) * kCluster), dim3(kWarps * 32), 0, s, ids, weights,
                    static_cast<const __nv_bfloat16*>(x), x_stride, static_cast<const WT*>(router), bias, mask, tokens,
                    experts, hidden, top_k, sigmoid, renormalize, scale);
}

template <typename WT, typename... A>
int route_by_tokens(int tokens, A... a) {
  if (tokens <= 1) return launch_route<WT, 1>(a...);
  if (tokens <= 2) return launch_route<WT, 2>(a...);
  if (tokens <= 4) return launch_route<WT, 4>(a...);
  return launch_route<WT, 8>(a...);
}

bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int check_sizes(int tokens, int experts, int hidden, int top_k) {
  HCA_CHECK_ARG(tokens >= 0 && experts > 0 && hidden > 0 && top_k > 0 && top_k <= experts);
  if (experts > kMoeExperts || top_k > kMoeTopK || hidden % 32 != 0) return HCA_E_UNSUPPORTED;
  return HCA_OK;
}

int route(int32_t* ids, float* weights, const void* x, int64_t x_stride, const void* router, int router_fp32,
          const float* bias, const uint8_t* mask, int tokens, int experts, int hidden, int top_k, int sigmoid,
          int renormalize, float scale, cudaStream_t s) {
  HCA_CHECK_ARG(ids && weights && x && router);
  HCA_CHECK_ARG(aligned(x, 16) && x_stride % 8 == 0 && aligned(router, 16));
  HCA_CHECK_ARG(cdiv(tokens, 8) <= 1 << 20);
  return router_fp32 ? route_by_tokens<float>(tokens, ids, weights, x, x_stride, router, bias, mask, tokens, experts,
                                              hidden, top_k, sigmoid, renormalize, scale, s)
                     : route_by_tokens<__nv_bfloat16>(tokens, ids, weights, x, x_stride, router, bias, mask, tokens,
                                                      experts, hidden, top_k, sigmoid, renormalize, scale, s);
}

int64_t align_up(int64_t v) { return (v + 255) / 256 * 256; }

int64_t h_bytes(int tokens, int top_k, int inner, int shared_inner) {
  const int64_t t = std::min(tokens, kMoeTokens);
  return align_up(t * (static_cast<int64_t>(top_k) * inner + shared_inner) * 2);
}

int experts_passes(void* out, int64_t out_stride, const void* x, int64_t x_stride, const int32_t* ids,
                   const float* weights, const uint8_t* mask, int format, int group, const MoeWeights& w, int tokens,
                   int experts, int hidden, int inner, int shared_inner, int top_k, __nv_bfloat16* h, cudaStream_t s) {
  HCA_CHECK_ARG(out && x && ids && weights);
  HCA_CHECK_ARG(aligned(x, 16) && x_stride % 8 == 0 && aligned(out, 2));
  for (int t = 0; t < tokens; t += kMoeTokens) {
    MoePass p;
    p.x = static_cast<const __nv_bfloat16*>(x) + t * x_stride;
    p.x_stride = x_stride;
    p.ids = ids + static_cast<int64_t>(t) * top_k;
    p.weights = weights + static_cast<int64_t>(t) * top_k;
    p.mask = mask == nullptr ? nullptr : mask + t;
    p.h = h;
    p.out = static_cast<__nv_bfloat16*>(out) + t * out_stride;
    p.out_stride = out_stride;
    p.tokens = std::min(tokens - t, kMoeTokens);
    p.top_k = top_k, p.experts = experts, p.hidden = hidden, p.inner = inner, p.shared_inner = shared_inner;
    int rc = HCA_E_UNSUPPORTED;
    if (format == HCA_WEIGHT_BF16) rc = moe_experts_pass<kWBf16>(p, w, s);
    else if (format == HCA_WEIGHT_FP8) rc = moe_experts_pass<kWFp8>(p, w, s);
    else if (group == 32) rc = moe_experts_pass<kW4G32>(p, w, s);
    else if (group == 64) rc = moe_experts_pass<kW4G64>(p, w, s);
    else if (group == 128) rc = moe_experts_pass<kW4G128>(p, w, s);
    if (rc != HCA_OK) return rc;
  }
  return HCA_OK;
}

int check_matrix(const MoeMatrix& m, int format) {
  HCA_CHECK_ARG(m.data && aligned(m.data, 16));
  HCA_CHECK_ARG(format == HCA_WEIGHT_BF16 || (m.scale && aligned(m.scale, format == HCA_WEIGHT_FP8 ? 4 : 2)));
  return HCA_OK;
}

int check_weights(const MoeWeights& w, int format, int group, int hidden, int inner, int shared_inner) {
  if (format != HCA_WEIGHT_BF16 && format != HCA_WEIGHT_FP8 && format != HCA_WEIGHT_W4) return HCA_E_UNSUPPORTED;
  if (format == HCA_WEIGHT_W4) {
    if (group != 32 && group != 64 && group != 128) return HCA_E_UNSUPPORTED;
    HCA_CHECK_ARG(hidden % group == 0 && inner % group == 0 && shared_inner % group == 0);
  }
  HCA_CHECK_ARG(inner > 0 && shared_inner >= 0);
  if (inner % 32 != 0 || shared_inner % 32 != 0) return HCA_E_UNSUPPORTED;
  int rc = check_matrix(w.w13, format);
  if (rc == HCA_OK) rc = check_matrix(w.w2, format);
  if (rc == HCA_OK && shared_inner > 0) rc = check_matrix(w.shared13, format);
  if (rc == HCA_OK && shared_inner > 0) rc = check_matrix(w.shared2, format);
  return rc;
}

MoeMatrix matrix(const void* data, const void* scale, const uint8_t* zero) {
  return {static_cast<const uint8_t*>(data), scale, zero};
}

}  // namespace
}  // namespace hca

extern "C" int hca_moe_route(int32_t* ids, float* weights, const void* x, int64_t x_stride, const void* router,
                             int32_t router_fp32, const float* router_bias, const uint8_t* token_mask,
                             int32_t num_tokens, int32_t num_experts, int32_t hidden, int32_t top_k, int32_t sigmoid,
                             int32_t renormalize, float routed_scale, void* stream) {
  using namespace hca;
  const int rc = check_sizes(num_tokens, num_experts, hidden, top_k);
  if (rc != HCA_OK || num_tokens == 0) return rc;
  return route(ids, weights, x, x_stride, router, router_fp32, router_bias, token_mask, num_tokens, num_experts,
               hidden, top_k, sigmoid, renormalize, routed_scale, as_stream(stream));
}

extern "C" int64_t hca_moe_workspace_bytes(int32_t num_tokens, int32_t top_k, int32_t inner, int32_t shared_inner) {
  if (num_tokens <= 0 || top_k <= 0 || inner <= 0 || shared_inner < 0) return 0;
  return hca::h_bytes(num_tokens, top_k, inner, shared_inner) +
         2 * hca::align_up(static_cast<int64_t>(num_tokens) * top_k * 4);
}

extern "C" int hca_moe_experts(void* out, int64_t out_stride, const void* x, int64_t x_stride, const int32_t* ids,
                               const float* weights, const uint8_t* token_mask, int32_t format, int32_t group_size,
                               const void* w13, const void* w13_scale, const uint8_t* w13_zero, const void* w2,
                               const void* w2_scale, const uint8_t* w2_zero, const void* shared13,
                               const void* shared13_scale, const uint8_t* shared13_zero, const void* shared2,
                               const void* shared2_scale, const uint8_t* shared2_zero, int32_t num_tokens,
                               int32_t num_experts, int32_t hidden, int32_t inner, int32_t shared_inner,
                               int32_t top_k, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace hca;
  const MoeWeights w{matrix(w13, w13_scale, w13_zero), matrix(w2, w2_scale, w2_zero),
                     matrix(shared13, shared13_scale, shared13_zero), matrix(shared2, shared2_scale, shared2_zero)};
  // ids may come from elsewhere and repeat, so top_k may exceed the experts of this rank
  HCA_CHECK_ARG(num_tokens >= 0 && num_experts > 0 && hidden > 0 && top_k > 0);
  if (num_experts > kMoeExperts || top_k > kMoeTopK || hidden % 32 != 0) return HCA_E_UNSUPPORTED;
  const int rc = check_weights(w, format, group_size, hidden, inner, shared_inner);
  if (rc != HCA_OK || num_tokens == 0) return rc;
  if (workspace_bytes < h_bytes(num_tokens, top_k, inner, shared_inner)) return HCA_E_WORKSPACE;
  HCA_CHECK_ARG(workspace && aligned(workspace, 16));
  return experts_passes(out, out_stride, x, x_stride, ids, weights, token_mask, format, group_size, w, num_tokens,
                        num_experts, hidden, inner, shared_inner, top_k, static_cast<__nv_bfloat16*>(workspace),
                        as_stream(stream));
}

extern "C" int hca_moe_decode(void* out, int64_t out_stride, const void* x, int64_t x_stride, const void* router,
                              int32_t router_fp32, const float* router_bias, int32_t sigmoid, int32_t renormalize,
                              float routed_scale, const uint8_t* token_mask, int32_t format, int32_t group_size,
                              const void* w13, const void* w13_scale, const uint8_t* w13_zero, const void* w2,
                              const void* w2_scale, const uint8_t* w2_zero, const void* shared13,
                              const void* shared13_scale, const uint8_t* shared13_zero, const void* shared2,
                              const void* shared2_scale, const uint8_t* shared2_zero, int32_t num_tokens,
                              int32_t num_experts, int32_t hidden, int32_t inner, int32_t shared_inner, int32_t top_k,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace hca;
  const MoeWeights w{matrix(w13, w13_scale, w13_zero), matrix(w2, w2_scale, w2_zero),
                     matrix(shared13, shared13_scale, shared13_zero), matrix(shared2, shared2_scale, shared2_zero)};
  int rc = check_sizes(num_tokens, num_experts, hidden, top_k);
  if (rc == HCA_OK) rc = check_weights(w, format, group_size, hidden, inner, shared_inner);
  if (rc != HCA_OK || num_tokens == 0) return rc;
  if (workspace_bytes < hca_moe_workspace_bytes(num_tokens, top_k, inner, shared_inner)) return HCA_E_WORKSPACE;
  HCA_CHECK_ARG(workspace && aligned(workspace, 16));
  HCA_CHECK_ARG(out && aligned(out, 2));
  uint8_t* at = static_cast<uint8_t*>(workspace);
  __nv_bfloat16* h = reinterpret_cast<__nv_bfloat16*>(at);
  at += h_bytes(num_tokens, top_k, inner, shared_inner);
  int32_t* ids = reinterpret_cast<int32_t*>(at);
  at += align_up(static_cast<int64_t>(num_tokens) * top_k * 4);
  float* weights = reinterpret_cast<float*>(at);
  rc = route(ids, weights, x, x_stride, router, router_fp32, router_bias, token_mask, num_tokens, num_experts, hidden,
             top_k, sigmoid, renormalize, routed_scale, as_stream(stream));
  if (rc != HCA_OK) return rc;
  return experts_passes(out, out_stride, x, x_stride, ids, weights, token_mask, format, group_size, w, num_tokens,
                        num_experts, hidden, inner, shared_inner, top_k, h, as_stream(stream));
}
