// The router of the few-token mixture-of-experts layer, and the C entries.
//
//   l[t, e] = x_t . Wr_e;  p = softmax(l) or 1 / (1 + exp(-l))
//   ids[t] = the top_k largest of p + bias, ties to the lower expert
//   weights[t, j] = p[t, ids[t, j]] (/ their sum) * scale
//
// The logits are latency-bound (experts * hidden weights, a few MB at most),
// so they are spread over the whole GPU: a CTA computes two experts for up to
// eight tokens, its warps splitting hidden.  Products and sums are
// 32-bit multiply-adds: a bf16 tensor product would make near-ties of a 32-bit
// router fall differently.  The choice itself is one warp's work a token, and up
// to 16 tokens every CTA of the expert kernel makes it for itself.  About 3 us
// for 64 experts of 4096 and one token, most of it launch and one round of loads.
#include "hca_moe.cuh"
#include "hca_stream.cuh"

#include <algorithm>

namespace hca {

namespace {

constexpr int kWarps = 8;
constexpr int kExperts = 2;  // of a CTA of the logits kernel

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

// Sums of N values (a power of two up to 32) over the warp: each exchange adds
// halves, so lane l ends with value `index` and N + 4 shuffles do for 5 N.
template <int N>
__device__ __forceinline__ float warp_sums(float (&v)[N], int& index) {
  const int lane = threadIdx.x & 31;
  index = 0;
  int n = N;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (n > 1) {
      n >>= 1;
      const bool upper = lane & o;
#pragma unroll
      for (int i = 0; i < N / 2; ++i)
        if (i < n) {
          const float keep = upper ? v[i + n] : v[i], give = upper ? v[i] : v[i + n];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
      if (upper) index += n;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    }
  }
  return v[0];
}

// logits[t, e] for kExperts experts and TB tokens; block (0, 0) also clears
// the words of `barriers`.
template <typename WT, int TB>
__global__ void __launch_bounds__(kWarps * 32)
    moe_logits_kernel(float* logits, const __nv_bfloat16* x, int64_t x_stride, const WT* router, int tokens,
                      int experts, int hidden, uint32_t* barriers, int num_barriers) {
  __shared__ float part[kWarps][kExperts * TB];
  pdl_wait_and_release();
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int i = threadIdx.x; i < num_barriers; i += kWarps * 32) barriers[i] = 0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int e0 = blockIdx.x * kExperts, t0 = blockIdx.y * TB;
  float acc[kExperts * TB] = {};
#pragma unroll 2
  for (int k = (warp * 32 + lane) * 8; k < hidden; k += kWarps * 256) {  // hidden is a multiple of 8
    float wv[kExperts][8];
#pragma unroll
    for (int i = 0; i < kExperts; ++i) load8(wv[i], router + static_cast<int64_t>(min(e0 + i, experts - 1)) * hidden + k);
#pragma unroll
    for (int t = 0; t < TB; ++t) {
      float xv[8];
      load8(xv, x + min(t0 + t, tokens - 1) * x_stride + k);
#pragma unroll
      for (int i = 0; i < kExperts; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i * TB + t] = fmaf(xv[j], wv[i][j], acc[i * TB + t]);
    }
  }
  int index;
  const float v = warp_sums(acc, index);
  part[warp][index] = v;
  __syncthreads();
  for (int i = threadIdx.x; i < kExperts * TB; i += kWarps * 32) {
    const int e = e0 + i / TB, t = t0 + i % TB;
    if (e >= experts || t >= tokens) continue;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += part[w][i];
    logits[static_cast<int64_t>(t) * experts + e] = sum;
  }
}

template <typename WT, int TB>
int launch_logits(float* logits, const void* x, int64_t x_stride, const void* router, int tokens, int experts,
                  int hidden, uint32_t* barriers, int num_barriers, cudaStream_t s) {
  return launch_pdl(moe_logits_kernel<WT, TB>, dim3(cdiv(experts, kExperts), cdiv(tokens, TB)),
                    dim3(kWarps * 32), 0, s, logits, static_cast<const __nv_bfloat16*>(x), x_stride,
                    static_cast<const WT*>(router), tokens, experts, hidden, barriers, num_barriers);
}

template <typename WT, typename... A>
int logits_by_tokens(int tokens, A... a) {
  // Few tokens: more CTAs than reuse of the weights.  (Router with its choice,
  // 128 experts of 4096, fp32: one token 3.6 us by ones, 5.0 by eights; eight
  // 4.5 by fours, 5.5 by eights; 32 7.1 by fours, 6.1 by eights.)
  if (tokens <= 1) return launch_logits<WT, 1>(a...);
  if (tokens <= 2) return launch_logits<WT, 2>(a...);
  if (tokens <= 8) return launch_logits<WT, 4>(a...);
  return launch_logits<WT, 8>(a...);
}

__global__ void __launch_bounds__(kWarps * 32)
    moe_choose_kernel(int32_t* ids, float* weights, const float* logits, int tokens, MoeRouting r) {
  pdl_wait_and_release();
  const int t = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  choose_all(logits, r, t, tokens, tokens, [&](int t, int id, float weight) {
    ids[static_cast<int64_t>(t) * r.top_k + lane] = id;
    weights[static_cast<int64_t>(t) * r.top_k + lane] = weight;
  });
}

int choose(int32_t* ids, float* weights, const float* logits, int tokens, const MoeRouting& r, cudaStream_t s) {
  return launch_pdl(moe_choose_kernel, dim3(cdiv(tokens, kWarps)), dim3(kWarps * 32), 0, s, ids, weights, logits, tokens,
                    r);
}

bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int check_sizes(int tokens, int experts, int hidden, int top_k) {
  HCA_CHECK_ARG(tokens >= 0 && experts > 0 && hidden > 0 && top_k > 0 && top_k <= experts);
  if (experts > kMoeExperts || top_k > kMoeTopK || hidden % 32 != 0) return HCA_E_UNSUPPORTED;
  return HCA_OK;
}

int check_rows(const void* x, int64_t x_stride) {
  HCA_CHECK_ARG(x && aligned(x, 16) && x_stride % 8 == 0);
  return HCA_OK;
}

int compute_logits(float* logits, const void* x, int64_t x_stride, const void* router, int router_fp32, int tokens,
                   int experts, int hidden, uint32_t* barriers, int num_barriers, cudaStream_t s) {
  // a launch for each 524280 tokens, a grid's 65535 eights; the first clears the barriers
  constexpr int kTokens = 8 * 65535;
  for (int t = 0; t < tokens; t += std::min(kTokens, tokens - t)) {
    const int n = std::min(kTokens, tokens - t), clear = t == 0 ? num_barriers : 0;
    float* to = logits + static_cast<int64_t>(t) * experts;
    const void* from = static_cast<const uint16_t*>(x) + t * x_stride;
    const int rc = router_fp32
                       ? logits_by_tokens<float>(n, to, from, x_stride, router, n, experts, hidden, barriers, clear, s)
                       : logits_by_tokens<__nv_bfloat16>(n, to, from, x_stride, router, n, experts, hidden, barriers, clear, s);
    if (rc != HCA_OK) return rc;
  }
  return HCA_OK;
}

int64_t align_up(int64_t v) { return (v + 255) / 256 * 256; }
int64_t logit_bytes(int tokens, int experts) { return align_up(static_cast<int64_t>(tokens) * experts * 4); }

// Scratch of a call: gated products and the pairs' shares of y of one pass,
// a barrier word a pass, and the logits.
struct Scratch {
  int64_t h, part, barriers, logits, ids, weights, total;
  int passes;
  Scratch(int tokens, int experts, int top_k, int hidden, int inner, int shared_inner) {
    const int64_t t = std::min(tokens, kMoeTokens);
    passes = cdiv(tokens, kMoeTokens);
    h = 0;
    part = align_up(t * (static_cast<int64_t>(top_k) * inner + shared_inner) * 4);  // h in two bf16 parts
    barriers = part + align_up(t * (top_k + 1) * hidden * 4);
    logits = barriers + align_up(4ll * passes);
    ids = logits + logit_bytes(tokens, experts);
    weights = ids + align_up(4ll * tokens * top_k);
    total = weights + align_up(4ll * tokens * top_k);
  }
};

int check_matrix(const MoeMatrix& m, int format) {
  HCA_CHECK_ARG(m.data && aligned(m.data, 16));
  HCA_CHECK_ARG(format == HCA_WEIGHT_BF16 || (m.scale && aligned(m.scale, 4) && aligned(m.zero, 4)));
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
  // zero points are a part of the format that both share
  HCA_CHECK_ARG(shared_inner == 0 || ((w.w13.zero == nullptr) == (w.shared13.zero == nullptr) &&
                                      (w.w2.zero == nullptr) == (w.shared2.zero == nullptr)));
  return rc;
}

// One layer's passes over 64 tokens each; either logits or ids and weights.
int experts_passes(void* out, int64_t out_stride, const void* x, int64_t x_stride, const float* logits,
                   const int32_t* ids, const float* weights, const MoeRouting& routing, int format, int group,
                   const MoeWeights& w, int tokens, int hidden, int inner, int shared_inner, uint8_t* workspace,
                   const Scratch& at, cudaStream_t s) {
  int32_t* error = device_error_word();
  if (error == nullptr) return HCA_E_CUDA;
  for (int i = 0; i < at.passes; ++i) {
    const int t = i * kMoeTokens;
    MoePass p;
    p.x = static_cast<const __nv_bfloat16*>(x) + t * x_stride;
    p.x_stride = x_stride;
    p.logits = logits == nullptr ? nullptr : logits + static_cast<int64_t>(t) * routing.experts;
    p.ids = ids == nullptr ? nullptr : ids + static_cast<int64_t>(t) * routing.top_k;
    p.weights = weights == nullptr ? nullptr : weights + static_cast<int64_t>(t) * routing.top_k;
    p.h = reinterpret_cast<__nv_bfloat16*>(workspace + at.h);
    p.part = reinterpret_cast<float*>(workspace + at.part);
    p.barrier = reinterpret_cast<uint32_t*>(workspace + at.barriers) + i;
    p.error = error;
    p.out = static_cast<__nv_bfloat16*>(out) + t * out_stride;
    p.out_stride = out_stride;
    p.routing = routing;
    if (p.routing.mask != nullptr) p.routing.mask += t;
    p.tokens = std::min(tokens - t, kMoeTokens);
    p.hidden = hidden, p.inner = inner, p.shared_inner = shared_inner;
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

MoeMatrix matrix(const void* data, const void* scale, const uint8_t* zero) {
  return {static_cast<const uint8_t*>(data), scale, zero};
}

}  // namespace
}  // namespace hca

extern "C" int64_t hca_moe_route_workspace_bytes(int32_t num_tokens, int32_t num_experts) {
  return num_tokens <= 0 || num_experts <= 0 ? 0 : hca::logit_bytes(num_tokens, num_experts);
}

extern "C" int hca_moe_route(int32_t* ids, float* weights, const void* x, int64_t x_stride, const void* router,
                             int32_t router_fp32, const float* router_bias, const uint8_t* token_mask,
                             int32_t num_tokens, int32_t num_experts, int32_t hidden, int32_t top_k, int32_t sigmoid,
                             int32_t renormalize, float routed_scale, void* workspace, int64_t workspace_bytes,
                             void* stream) {
  using namespace hca;
  int rc = check_sizes(num_tokens, num_experts, hidden, top_k);
  if (rc != HCA_OK || num_tokens == 0) return rc;
  rc = check_rows(x, x_stride);
  if (rc != HCA_OK) return rc;
  HCA_CHECK_ARG(ids && weights && router && aligned(router, 16));
  if (workspace_bytes < logit_bytes(num_tokens, num_experts)) return HCA_E_WORKSPACE;
  HCA_CHECK_ARG(workspace && aligned(workspace, 16));
  cudaStream_t s = as_stream(stream);
  float* logits = static_cast<float*>(workspace);
  rc = compute_logits(logits, x, x_stride, router, router_fp32, num_tokens, num_experts, hidden, nullptr, 0, s);
  if (rc != HCA_OK) return rc;
  const MoeRouting r{router_bias, token_mask, num_experts, top_k, sigmoid, renormalize, routed_scale};
  return choose(ids, weights, logits, num_tokens, r, s);
}

extern "C" int64_t hca_moe_workspace_bytes(int32_t num_tokens, int32_t num_experts, int32_t top_k, int32_t hidden,
                                           int32_t inner, int32_t shared_inner) {
  if (num_tokens <= 0 || num_experts <= 0 || top_k <= 0 || hidden <= 0 || inner <= 0 || shared_inner < 0) return 0;
  return hca::Scratch(num_tokens, num_experts, top_k, hidden, inner, shared_inner).total;
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
  int rc = check_weights(w, format, group_size, hidden, inner, shared_inner);
  if (rc != HCA_OK || num_tokens == 0) return rc;
  const Scratch at(num_tokens, num_experts, top_k, hidden, inner, shared_inner);
  if (workspace_bytes < at.total) return HCA_E_WORKSPACE;
  HCA_CHECK_ARG(workspace && aligned(workspace, 16));
  HCA_CHECK_ARG(out && aligned(out, 2) && ids && weights);
  rc = check_rows(x, x_stride);
  if (rc != HCA_OK) return rc;
  cudaStream_t s = as_stream(stream);
  uint8_t* scratch = static_cast<uint8_t*>(workspace);
  rc = cuda_status(cudaMemsetAsync(scratch + at.barriers, 0, 4ll * at.passes, s));
  if (rc != HCA_OK) return rc;
  const MoeRouting r{nullptr, token_mask, num_experts, top_k, 0, 0, 1.0f};
  return experts_passes(out, out_stride, x, x_stride, nullptr, ids, weights, r, format, group_size, w, num_tokens,
                        hidden, inner, shared_inner, scratch, at, s);
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
  const Scratch at(num_tokens, num_experts, top_k, hidden, inner, shared_inner);
  if (workspace_bytes < at.total) return HCA_E_WORKSPACE;
  HCA_CHECK_ARG(workspace && aligned(workspace, 16));
  HCA_CHECK_ARG(out && aligned(out, 2) && router && aligned(router, 16));
  rc = check_rows(x, x_stride);
  if (rc != HCA_OK) return rc;
  cudaStream_t s = as_stream(stream);
  uint8_t* scratch = static_cast<uint8_t*>(workspace);
  float* logits = reinterpret_cast<float*>(scratch + at.logits);
  rc = compute_logits(logits, x, x_stride, router, router_fp32, num_tokens, num_experts, hidden,
                      reinterpret_cast<uint32_t*>(scratch + at.barriers), at.passes, s);
  if (rc != HCA_OK) return rc;
  const MoeRouting r{router_bias, token_mask, num_experts, top_k, sigmoid, renormalize, routed_scale};
  // Choosing is a warp's work a token: every CTA of the expert kernel does it
  // while its warps do not have to take turns (2 us), else a launch does (with
  // 64 tokens 3 us for 9).
  if (num_tokens > 16) {
    int32_t* ids = reinterpret_cast<int32_t*>(scratch + at.ids);
    float* weights = reinterpret_cast<float*>(scratch + at.weights);
    rc = choose(ids, weights, logits, num_tokens, r, s);
    return rc != HCA_OK ? rc
                        : experts_passes(out, out_stride, x, x_stride, nullptr, ids, weights, r, format, group_size, w,
                                         num_tokens, hidden, inner, shared_inner, scratch, at, s);
  }
  return experts_passes(out, out_stride, x, x_stride, logits, nullptr, nullptr, r, format, group_size, w, num_tokens,
                        hidden, inner, shared_inner, scratch, at, s);
}
