// Penalties for repeated tokens, biases and grammar masks on logits, in place.
//
//   x += bias[v];  if v was seen in prompt or answer: x > 0 ? x / r : x * r
//   x -= frequency * (times v occurs in the answer) + presence * (v occurs there)
//   x = -inf where the bit mask does not allow v
//
// Only the logits that change are read or written: those of distinct history
// tokens and biased ones, and (written only) the masked ones.  A cluster of
// eight CTAs owns a row.  It splits the vocabulary into eight slices, each
// CTA keeping a slice's counts in its shared memory; each reads an eighth of
// the history and counts into the slice's owner over distributed shared
// memory (whole numbers, so the order does not matter), and then walks its
// own slice.  The history is read once, and no table lives in global memory.
// Vocabularies beyond what eight CTAs hold take further rounds over slices.
#include <algorithm>

#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "hca_common.cuh"

namespace hca {
namespace {

namespace cg = cooperative_groups;

constexpr int kCluster = 8;
constexpr int kThreads = 512;
constexpr uint32_t kPrompt = 0x80000000u;
// entries of a slice: a count, and with biases a position, of 4 bytes each
constexpr int kSliceBytes = 208 * 1024;

template <typename T>
__device__ __forceinline__ float load_logit(const T* p);
template <>
__device__ __forceinline__ float load_logit<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float load_logit<__nv_bfloat16>(const __nv_bfloat16* p) { return __bfloat162float(*p); }
template <>
__device__ __forceinline__ float load_logit<__half>(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void store_logit(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_logit(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_logit(__half* p, float v) { *p = __float2half_rn(v); }

struct LogitArgs {
  void* logits;
  int64_t stride;
  const int32_t* req_index;  // row -> row of the per-request tables, or null: the same
  const int32_t* token_ids;  // [requests, >= seq_len]
  int64_t token_stride;
  const int32_t* prompt_lens;  // by row
  const int32_t* seq_lens;     // by row
  const float* repetition;     // by request; null: 1
  const float* frequency;      // null: 0
  const float* presence;       // null: 0
  const int32_t* bias_ids;     // [requests, bias_width]
  const float* bias_values;
  int64_t bias_stride;
  const int32_t* allowed;  // [rows, ceil(vocab / 32)]
  int64_t allowed_stride;
  int vocab, bias_width, token_width, num_reqs, slice;
};

template <typename T>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads) logit_penalty_kernel(LogitArgs a) {
  extern __shared__ __align__(16) uint32_t table[];  // counts [slice], bias positions + 1 [slice]
  pdl_wait_and_release();
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  const int64_t row = blockIdx.x / kCluster;
  const int64_t req = a.req_index == nullptr ? row : a.req_index[row];
  if (req < 0 || req >= a.num_reqs) return;  // the same for the whole cluster
  T* logits = static_cast<T*>(a.logits) + row * a.stride;
  const bool biased = a.bias_width > 0;
  const uint32_t slice = static_cast<uint32_t>(a.slice);
  const int words = biased ? 2 * a.slice : a.slice;
  const int prompt_len = a.token_ids == nullptr ? 0 : a.prompt_lens[row];
  const int seq_len = a.token_ids == nullptr ? 0 : min(a.seq_lens[row], a.token_width);
  const int32_t* tokens = a.token_ids + req * a.token_stride;
  const float rep = a.repetition == nullptr ? 1.0f : a.repetition[req];
  const float freq = a.frequency == nullptr ? 0.0f : a.frequency[req];
  const float pres = a.presence == nullptr ? 0.0f : a.presence[req];

  for (int64_t base = 0; base < a.vocab; base += static_cast<int64_t>(slice) * kCluster) {
    for (int i = threadIdx.x; i < words / 4; i += kThreads) reinterpret_cast<uint4*>(table)[i] = make_uint4(0, 0, 0, 0);
    cluster.sync();
    const int64_t left = a.vocab - base;
    const uint32_t span = static_cast<uint32_t>(left < static_cast<int64_t>(slice) * kCluster ? left : slice * kCluster);
    for (int64_t i = static_cast<int64_t>(rank) * kThreads + threadIdx.x; i < seq_len; i += kCluster * kThreads) {
      // ids outside the vocabulary (-1 padding among them) wrap to large values here
      const uint32_t id = static_cast<uint32_t>(tokens[i]) - static_cast<uint32_t>(base);
      if (tokens[i] < 0 || id >= span) continue;
      uint32_t* at = cluster.map_shared_rank(&table[id % slice], id / slice);
      if (i < prompt_len) atomicOr(at, kPrompt);
      else atomicAdd(at, 1u);
    }
    if (biased) {
      for (int i = rank * kThreads + threadIdx.x; i < a.bias_width; i += kCluster * kThreads) {
        const int v = a.bias_ids[req * a.bias_stride + i];
        const uint32_t id = static_cast<uint32_t>(v) - static_cast<uint32_t>(base);
        if (v < 0 || id >= span) continue;
        // an id listed twice: the later entry counts
        atomicMax(cluster.map_shared_rank(&table[slice + id % slice], id / slice), static_cast<uint32_t>(i + 1));
      }
    }
    cluster.sync();
    const int64_t first = base + static_cast<int64_t>(rank) * slice;
    const int n = static_cast<int>(min(static_cast<int64_t>(slice), a.vocab - first));  // may be negative
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const int64_t v = first + i;
      if (a.allowed != nullptr) {
        const uint32_t word = static_cast<uint32_t>(a.allowed[row * a.allowed_stride + v / 32]);
        if (!(word >> (v & 31) & 1)) {
          store_logit(logits + v, -INFINITY);
          continue;
        }
      }
      const uint32_t c = table[i];
      const uint32_t b = biased ? table[slice + i] : 0;
      if (c == 0 && b == 0) continue;
      float x = load_logit(logits + v);
      if (b != 0) x += a.bias_values[req * a.bias_stride + b - 1];
      if (c != 0) x = x > 0.0f ? x / rep : x * rep;
      const uint32_t count = c & ~kPrompt;
      if (count != 0) x = x - freq * static_cast<float>(count) - pres;
      store_logit(logits + v, x);
    }
    cluster.sync();  // before the table is cleared, or a CTA leaves, while others may still write into it
  }
}

template <typename T>
int launch(LogitArgs a, int rows, cudaStream_t s) {
  const int entry = a.bias_width > 0 ? 8 : 4;
  const int most = kSliceBytes / entry / 32 * 32;
  a.slice = std::min(most, (cdiv(a.vocab, kCluster) + 31) / 32 * 32);  // whole mask words
  static bool done[kMaxDevices] = {};
  if (set_func_attr_once(logit_penalty_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSliceBytes, done) !=
      HCA_OK)
    return HCA_E_CUDA;
  return launch_pdl(logit_penalty_kernel<T>, dim3(rows * kCluster), dim3(kThreads),
                    static_cast<size_t>(a.slice) * entry, s, a);
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
  HCA_CHECK_ARG(num_rows <= INT32_MAX / kCluster);
  LogitArgs a;
  a.logits = logits, a.stride = logits_stride, a.req_index = req_index, a.num_reqs = num_reqs;
  a.token_ids = token_ids, a.token_stride = token_stride, a.token_width = token_width;
  a.prompt_lens = prompt_lens, a.seq_lens = seq_lens;
  a.repetition = repetition, a.frequency = frequency, a.presence = presence;
  a.bias_ids = bias_ids, a.bias_values = bias_values, a.bias_stride = bias_stride, a.bias_width = bias_width;
  a.allowed = allowed_bitmask, a.allowed_stride = allowed_stride, a.vocab = vocab, a.slice = 0;
  cudaStream_t s = as_stream(stream);
  if (type == HCA_LOGITS_FP32) return launch<float>(a, num_rows, s);
  if (type == HCA_LOGITS_BF16) return launch<__nv_bfloat16>(a, num_rows, s);
  return launch<__half>(a, num_rows, s);
}
