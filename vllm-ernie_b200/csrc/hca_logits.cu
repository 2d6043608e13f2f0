// Penalties for repeated tokens, biases and grammar masks on logits, in place.
//
//   x += bias[v];  if v was seen in prompt or answer: x > 0 ? x / r : x * r
//   x -= frequency * (times v occurs in the answer) + presence * (v occurs there)
//   x = -inf where the bit mask does not allow v
//
// Only the logits that change are read or written: those of distinct history
// tokens and biased ones, and (written only) the masked ones.  A row's
// vocabulary is dealt in chunks of 32 to a few CTAs, so that the low ids that
// texts crowd into spread over all of them.  Each CTA reads the row's whole
// history (from L2 but for the first) and counts its own tokens in shared
// memory; counts are whole numbers, so their order does not matter, and no
// table lives in global memory.  Then a warp goes over a chunk at a time, a
// lane a token, several chunks' loads under way.
#include <algorithm>

#include <cuda_fp16.h>

#include "hca_common.cuh"

namespace hca {
namespace {

constexpr int kThreads = 512;
constexpr int kAhead = 8;  // chunks of a warp under way
constexpr int kMostSlices = 1024;

__device__ __forceinline__ float load_logit(const float* p) { return *p; }
__device__ __forceinline__ float load_logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_logit(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void store_logit(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_logit(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_logit(__half* p, float v) { *p = __float2half_rn(v); }

struct LogitArgs {
  void* logits;
  int64_t stride;
  const int32_t* req_index;  // row -> row of the per-request tables, or null: the same
  const int32_t* token_ids;  // [requests, >= seq_len], or null
  int64_t token_stride;
  const int32_t* prompt_lens;  // by row
  const int32_t* seq_lens;     // by row
  const float* repetition;     // by request; null: 1
  const float* frequency;      // null: 0
  const float* presence;       // null: 0
  const int32_t* bias_ids;     // [requests, bias_width]
  const float* bias_values;
  int64_t bias_stride;
  const int32_t* allowed;  // [rows, ceil(vocab / 32)], or null
  int64_t allowed_stride;
  int vocab, bias_width, token_width, num_reqs, slices_log2;
};

// A CTA's share of a row: chunks rank, rank + slices, ... of 32 tokens.  Tables
// by local chunk: counts (16 bits where the history cannot hold more than
// 65535 tokens, else 32), a word of prompt bits, a word of biased tokens' bits.
template <typename T, typename Count>
__global__ void __launch_bounds__(kThreads, 2) logit_penalty_kernel(LogitArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int slices = 1 << a.slices_log2;
  const int64_t row = blockIdx.x >> a.slices_log2;
  const int rank = blockIdx.x & (slices - 1);
  const int all_chunks = (a.vocab + 31) / 32;
  const int most = (all_chunks + slices - 1) / slices;  // the same for every CTA
  const int chunks = (all_chunks - rank + slices - 1) / slices;
  uint32_t* prompt = reinterpret_cast<uint32_t*>(smem);
  uint32_t* biased = prompt + most;
  Count* count = reinterpret_cast<Count*>(smem + (8 * most + 15) / 16 * 16);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  {
    const int words = ((8 * most + 15) / 16 * 16 + 32 * most * static_cast<int>(sizeof(Count))) / 16;
    for (int i = threadIdx.x; i < words; i += kThreads) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  }
  pdl_wait_and_release();
  const int64_t req = a.req_index == nullptr ? row : a.req_index[row];
  if (req < 0 || req >= a.num_reqs) return;  // the whole CTA
  T* logits = static_cast<T*>(a.logits) + row * a.stride;
  __syncthreads();

  // v's local chunk and bit, if it is this CTA's
  auto mine = [&](int32_t v, int& chunk, int& bit) -> bool {
    const uint32_t c = static_cast<uint32_t>(v) >> 5;
    chunk = static_cast<int>(c >> a.slices_log2), bit = v & 31;
    return static_cast<uint32_t>(v) < static_cast<uint32_t>(a.vocab) && static_cast<int>(c & (slices - 1)) == rank;
  };
  if (a.token_ids != nullptr) {
    const int32_t* tokens = a.token_ids + req * a.token_stride;
    const int seq_len = min(a.seq_lens[row], a.token_width), prompt_len = min(a.prompt_lens[row], seq_len);
    auto see = [&](int32_t v, bool answer) {
      int c, bit;
      if (!mine(v, c, bit)) return;
      if (!answer) atomicOr(prompt + c, 1u << bit);
      else if constexpr (sizeof(Count) == 4) atomicAdd(reinterpret_cast<uint32_t*>(count) + 32 * c + bit, 1u);
      // two counts to a word: neither passes 65535, so none carries
      else atomicAdd(reinterpret_cast<uint32_t*>(count) + 16 * c + (bit >> 1), bit & 1 ? 0x10000u : 1u);
    };
    // four tokens at a time from the first 16-byte boundary on
    const int lead = static_cast<int>(-(reinterpret_cast<intptr_t>(tokens) >> 2) & 3);
    const int head = min(lead, max(seq_len, 0));
    if (static_cast<int>(threadIdx.x) < head) see(tokens[threadIdx.x], static_cast<int>(threadIdx.x) >= prompt_len);
    const int quads = max(seq_len - head, 0) / 4;
    const int4* body = reinterpret_cast<const int4*>(tokens + head);
#pragma unroll 4
    for (int i = threadIdx.x; i < quads; i += kThreads) {
      const int4 v = body[i];
      const int at = head + 4 * i;
      see(v.x, at >= prompt_len);
      see(v.y, at + 1 >= prompt_len);
      see(v.z, at + 2 >= prompt_len);
      see(v.w, at + 3 >= prompt_len);
    }
    const int done = head + 4 * quads;
    if (static_cast<int>(threadIdx.x) < seq_len - done)
      see(tokens[done + threadIdx.x], done + static_cast<int>(threadIdx.x) >= prompt_len);
  }
  const int32_t* bias_ids = a.bias_ids + req * a.bias_stride;
  for (int i = threadIdx.x; i < a.bias_width; i += kThreads) {
    int c, bit;
    if (mine(bias_ids[i], c, bit)) atomicOr(biased + c, 1u << bit);
  }
  __syncthreads();

  const float rep = a.repetition == nullptr ? 1.0f : a.repetition[req];
  const float freq = a.frequency == nullptr ? 0.0f : a.frequency[req];
  const float pres = a.presence == nullptr ? 0.0f : a.presence[req];
  const int32_t* allowed = a.allowed == nullptr ? nullptr : a.allowed + row * a.allowed_stride;
  auto penalise = [&](float x, uint32_t n, bool seen) {
    if (seen) x = x > 0.0f ? x / rep : x * rep;
    if (n != 0) x = x - freq * static_cast<float>(n) - pres;
    return x;
  };
  for (int c0 = warp; c0 < chunks; c0 += kAhead * (kThreads / 32)) {
    // what is to be done with the lane's token of each chunk: 0 nothing, 1 penalties, 2 -inf
    int what[kAhead];
    uint32_t n[kAhead];
    bool seen[kAhead];
    float x[kAhead];
    uint32_t word[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int c = c0 + j * (kThreads / 32);
      word[j] = ~0u;
      if (allowed != nullptr && c < chunks) word[j] = static_cast<uint32_t>(allowed[c * slices + rank]);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int c = c0 + j * (kThreads / 32);
      what[j] = 0, n[j] = 0, x[j] = 0.0f, seen[j] = false;
      const int v = (c * slices + rank) * 32 + lane;
      if (c >= chunks || v >= a.vocab) continue;
      n[j] = count[32 * c + lane];
      seen[j] = n[j] != 0 || (prompt[c] >> lane & 1);
      if (!(word[j] >> lane & 1)) what[j] = 2;
      else if (seen[j] && !(biased[c] >> lane & 1)) what[j] = 1;
      if (what[j] == 1) x[j] = load_logit(logits + v);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int v = ((c0 + j * (kThreads / 32)) * slices + rank) * 32 + lane;
      if (what[j] != 0) store_logit(logits + v, what[j] == 2 ? -INFINITY : penalise(x[j], n[j], seen[j]));
    }
  }
  for (int i = threadIdx.x; i < a.bias_width; i += kThreads) {
    const int v = bias_ids[i];
    int c, bit;
    if (!mine(v, c, bit)) continue;
    bool last = true;  // an id listed twice: the later entry counts
    for (int j = i + 1; j < a.bias_width; ++j) last = last && bias_ids[j] != v;
    if (!last || (allowed != nullptr && !(static_cast<uint32_t>(allowed[v >> 5]) >> bit & 1))) continue;
    const uint32_t k = count[32 * c + bit];
    const float x = load_logit(logits + v) + a.bias_values[req * a.bias_stride + i];
    store_logit(logits + v, penalise(x, k, k != 0 || (prompt[c] >> bit & 1)));
  }
}

template <typename T, typename Count>
int launch(LogitArgs a, int rows, cudaStream_t s) {
  const int chunks = (a.vocab + 31) / 32, sms = device_sm_count();
  auto bytes = [&](int log2) {
    const int64_t most = (chunks + (1 << log2) - 1) >> log2;
    return (8 * most + 15) / 16 * 16 + 32 * most * static_cast<int64_t>(sizeof(Count));
  };
  // Slices of a row: so many that two CTAs fit an SM, and while SMs would be
  // left without one, more, down to 64 chunks each.
  a.slices_log2 = 0;
  while (bytes(a.slices_log2) > 108 * 1024 ||
         ((static_cast<int64_t>(rows) << a.slices_log2) < 2 * sms && (chunks >> a.slices_log2) >= 128))
    ++a.slices_log2;
  if (1 << a.slices_log2 > kMostSlices) return HCA_E_UNSUPPORTED;
  static bool done[kMaxDevices] = {};
  if (set_func_attr_once(logit_penalty_kernel<T, Count>, cudaFuncAttributeMaxDynamicSharedMemorySize, 108 * 1024,
                         done) != HCA_OK)
    return HCA_E_CUDA;
  return launch_pdl(logit_penalty_kernel<T, Count>, dim3(static_cast<unsigned>(rows) << a.slices_log2), dim3(kThreads),
                    static_cast<size_t>(bytes(a.slices_log2)), s, a);
}

template <typename T>
int by_count(const LogitArgs& a, int rows, cudaStream_t s) {
  return a.token_width <= 65535 ? launch<T, uint16_t>(a, rows, s) : launch<T, uint32_t>(a, rows, s);
}

}  // namespace
}  // namespace hca

extern "C" int hca_logit_penalties(void* logits, int64_t logits_stride, int32_t type, const int32_t* req_index,
                                   int32_t num_reqs, const int32_t* token_ids, int64_t token_stride,
                                   int32_t token_width, const int32_t* prompt_lens, const int32_t* seq_lens,
                                   const float* repetition, const float* frequency, const float* presence,
                                   const int32_t* bias_ids, const float* bias_values, int64_t bias_stride,
                                   int32_t bias_width, const int32_t* allowed_bitmask, int64_t allowed_stride,
                                   int32_t num_rows, int32_t vocab, void* stream) {
  using namespace hca;
  HCA_CHECK_ARG(num_rows >= 0 && vocab > 0 && bias_width >= 0 && token_width >= 0);
  if (type != HCA_LOGITS_FP32 && type != HCA_LOGITS_BF16 && type != HCA_LOGITS_FP16) return HCA_E_UNSUPPORTED;
  if (num_rows == 0) return HCA_OK;
  HCA_CHECK_ARG(logits && reinterpret_cast<uintptr_t>(logits) % (type == HCA_LOGITS_FP32 ? 4 : 2) == 0);
  HCA_CHECK_ARG(req_index || num_reqs >= num_rows);
  HCA_CHECK_ARG(token_ids == nullptr || (prompt_lens && seq_lens));
  HCA_CHECK_ARG(bias_width == 0 || (bias_ids && bias_values));
  HCA_CHECK_ARG(num_rows <= INT32_MAX / kMostSlices);
  LogitArgs a;
  a.logits = logits, a.stride = logits_stride, a.req_index = req_index, a.num_reqs = num_reqs;
  a.token_ids = token_ids, a.token_stride = token_stride, a.token_width = token_width;
  a.prompt_lens = prompt_lens, a.seq_lens = seq_lens;
  a.repetition = repetition, a.frequency = frequency, a.presence = presence;
  a.bias_ids = bias_ids, a.bias_values = bias_values, a.bias_stride = bias_stride, a.bias_width = bias_width;
  a.allowed = allowed_bitmask, a.allowed_stride = allowed_stride, a.vocab = vocab, a.slices_log2 = 0;
  cudaStream_t s = as_stream(stream);
  if (type == HCA_LOGITS_FP32) return by_count<float>(a, num_rows, s);
  if (type == HCA_LOGITS_BF16) return by_count<__nv_bfloat16>(a, num_rows, s);
  return by_count<__half>(a, num_rows, s);
}
