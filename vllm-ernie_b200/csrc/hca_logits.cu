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
// table lives in global memory.  Then each warp lists the tokens seen among a
// few hundred and its lanes share them out, so that their loads run together.
//
// Bound by scattered accesses of a sector for two or four bytes.  Measured: 192
// rows of 151937 bf16 logits with histories up to 32768: 55 us (47 MB of sectors
// read and written, 25 MB of histories; two fifths of a CTA's time go into
// clearing its tables and counting, which nothing overlaps, one CTA filling an
// SM's shared memory); 64 rows of 129280 fp32 logits with masks: 16.4 us; one
// row with a short history: 3.4 us.
#include <algorithm>

#include <cuda_fp16.h>

#include "hca_common.cuh"

namespace hca {
namespace {

constexpr int kAhead = 2;  // logits of a lane under way
constexpr int kSmem = 224 * 1024;  // of an SM, for one CTA of 1024 threads or two of 512

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
// by local chunk: a word of prompt bits, a word of biased tokens' bits, counts
// (16 bits where the history cannot hold more than 65535 tokens, else 32).
template <typename Count>
struct Tables {
  static constexpr int kEntry = static_cast<int>(sizeof(Count));
  static constexpr int kSpan = 16;  // tokens of a lane at a time
  static constexpr int kListBytes = kSpan * 2;  // of a thread
  // chunks, rounded up so that every lane's span exists
  static __host__ __device__ int64_t padded(int64_t chunks) { return (chunks + 15) / 16 * 16; }
  static __host__ __device__ int64_t bytes(int64_t chunks) { return padded(chunks) * (8 + 32 * kEntry); }
};

template <typename T, typename Count, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) logit_penalty_kernel(LogitArgs a) {
  using Tab = Tables<Count>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int next_span;
  const int slices = 1 << a.slices_log2;
  const int64_t row = blockIdx.x >> a.slices_log2;
  const int rank = blockIdx.x & (slices - 1);
  const int all_chunks = (a.vocab + 31) / 32;
  const int chunks = (all_chunks - rank + slices - 1) >> a.slices_log2;
  const int padded = static_cast<int>(Tab::padded((all_chunks + slices - 1) >> a.slices_log2));
  uint32_t* prompt = reinterpret_cast<uint32_t*>(smem);
  uint32_t* biased = prompt + padded;
  Count* count = reinterpret_cast<Count*>(biased + padded);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint16_t* list = reinterpret_cast<uint16_t*>(count + 32 * padded) + warp * 32 * Tab::kSpan;
  for (int i = threadIdx.x; i < Tab::bytes(padded) / 16; i += kThreads)
    reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  if (threadIdx.x == 0) next_span = 0;
  pdl_wait_and_release();
  // what the row needs, in two rounds of loads
  const int64_t req = a.req_index == nullptr ? row : a.req_index[row];
  const bool history = a.token_ids != nullptr;
  const int seq_len = history ? max(min(a.seq_lens[row], a.token_width), 0) : 0;
  const int prompt_len = history ? max(min(a.prompt_lens[row], seq_len), 0) : 0;
  if (req < 0 || req >= a.num_reqs) return;  // the whole CTA
  const float rep = a.repetition == nullptr ? 1.0f : a.repetition[req];
  const float freq = a.frequency == nullptr ? 0.0f : a.frequency[req];
  const float pres = a.presence == nullptr ? 0.0f : a.presence[req];
  T* logits = static_cast<T*>(a.logits) + row * a.stride;
  __syncthreads();

  // Whether v is this CTA's, and its place in the tables.
  const uint32_t owner = static_cast<uint32_t>(rank) << 5, owner_mask = static_cast<uint32_t>(slices - 1) << 5;
  const int shift = 5 + a.slices_log2;
  auto mine = [&](int32_t v) {
    return ((static_cast<uint32_t>(v) ^ owner) & owner_mask) == 0 && static_cast<uint32_t>(v) < static_cast<uint32_t>(a.vocab);
  };
  auto place = [&](int32_t v) { return (v >> shift) * 32 + (v & 31); };
  if (history) {
    const int32_t* tokens = a.token_ids + req * a.token_stride;
    auto see = [&](int32_t v, bool answer) {
      if (!mine(v)) return;
      const int at = place(v);
      if (!answer) atomicOr(prompt + (at >> 5), 1u << (at & 31));
      else if constexpr (Tab::kEntry == 4) atomicAdd(reinterpret_cast<uint32_t*>(count) + at, 1u);
      // two counts to a word: neither passes 65535, so none carries
      else atomicAdd(reinterpret_cast<uint32_t*>(count) + (at >> 1), at & 1 ? 0x10000u : 1u);
    };
    // four tokens at a time from the first 16-byte boundary on
    const int head = min(static_cast<int>(-(reinterpret_cast<intptr_t>(tokens) >> 2) & 3), seq_len);
    if (static_cast<int>(threadIdx.x) < head) see(tokens[threadIdx.x], static_cast<int>(threadIdx.x) >= prompt_len);
    const int quads = (seq_len - head) / 4, done = head + 4 * quads;
    const int4* body = reinterpret_cast<const int4*>(tokens + head);
#pragma unroll 4
    for (int i = threadIdx.x; i < quads; i += kThreads) {
      const int4 v = body[i];
      const int at = head + 4 * i;
      if (at >= prompt_len) {  // the same for almost every warp
        see(v.x, true), see(v.y, true), see(v.z, true), see(v.w, true);
      } else {
        see(v.x, false), see(v.y, at + 1 >= prompt_len), see(v.z, at + 2 >= prompt_len), see(v.w, at + 3 >= prompt_len);
      }
    }
    if (static_cast<int>(threadIdx.x) < seq_len - done)
      see(tokens[done + threadIdx.x], done + static_cast<int>(threadIdx.x) >= prompt_len);
  }
  const int32_t* bias_ids = a.bias_ids + req * a.bias_stride;
  for (int i = threadIdx.x; i < a.bias_width; i += kThreads) {
    const int v = bias_ids[i];
    if (mine(v)) atomicOr(biased + (place(v) >> 5), 1u << (v & 31));
  }
  __syncthreads();

  const int32_t* allowed = a.allowed == nullptr ? nullptr : a.allowed + row * a.allowed_stride;
  // x / rep as the 64-bit product with 1 / rep, off by 2^-52 at most, where the
  // quotient of two 24-bit numbers is at least 2^-49 off the middle of two others:
  // it rounds as a normal quotient does.  (A 32-bit division branches where x is
  // tiny, as it becomes when a buffer is penalised over and over: 65 us for 55.)
  const double inverse = 1.0 / static_cast<double>(rep);
  auto penalise = [&](float x, uint32_t n, bool seen) {
    if (seen) x = x > 0.0f ? static_cast<float>(static_cast<double>(x) * inverse) : x * rep;
    if (n != 0) x = x - freq * static_cast<float>(n) - pres;
    return x;
  };
  // the token of a place, and back to its logit
  auto token = [&](int at) { return ((at >> 5 << a.slices_log2) + rank) * 32 + (at & 31); };

  // Masked places, a warp to 32 chunks: a lane loads a chunk's word, then is a bit of each.
  auto close = [&]() {
    for (int c0 = warp * 32; c0 < chunks; c0 += kThreads) {
      const int own = c0 + lane;
      uint32_t words = own < chunks ? static_cast<uint32_t>(allowed[(own << a.slices_log2) + rank]) : ~0u;
      const int over = token(own * 32) + 32 - a.vocab;  // places past the vocabulary's end
      if (over > 0 && over < 32) words |= ~0u << (32 - over);
      T* at = logits + token(c0 * 32) + lane;
      const uint32_t bit = 1u << lane;
      const int step = 1 << shift;
#pragma unroll 16
      for (int j = 0; j < 32; ++j, at += step)
        if (!(__shfl_sync(0xffffffffu, words, j) & bit)) store_logit(at, -INFINITY);
    }
  };
  // Seen, allowed and not biased ones: a lane finds those of kSpan places, the
  // warp lists them and shares them out.
  if (allowed != nullptr && (warp & 1)) close();  // half the warps first, half last: stores beside latency
  // whoever is free takes the next span: the low ids' are the longest
  for (;;) {
    int c0 = lane == 0 ? atomicAdd(&next_span, Tab::kSpan) : 0;
    c0 = __shfl_sync(0xffffffffu, c0, 0);
    if (c0 >= chunks) break;
    const int base = c0 * 32 + lane * Tab::kSpan, c = base >> 5, bit = base & 31;
    uint32_t may = ~0u;
    if (allowed != nullptr && c < chunks) may = static_cast<uint32_t>(allowed[(c << a.slices_log2) + rank]);
    uint32_t bits = prompt[c] >> bit, pairs = 0;
#pragma unroll
    for (int i = 0; i < Tab::kSpan * Tab::kEntry / 16; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(count + base)[i];
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (Tab::kEntry == 4) bits |= min(w[j], 1u) << (4 * i + j);
        else pairs |= __vminu2(w[j], 0x00010001u) << (8 * i + 2 * j);  // even places from bit 0 on, odd ones from bit 16
      }
    }
    bits |= (pairs & 0x5555u) | (pairs >> 15 & 0xaaaau);
    bits &= (may & ~biased[c]) >> bit & ((1u << Tab::kSpan) - 1);
    const int mine_n = __popc(bits);
    int before = mine_n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += v;
    }
    const int total = __shfl_sync(0xffffffffu, before, 31);
    before -= mine_n;
    for (; bits != 0; bits &= bits - 1) list[before++] = static_cast<uint16_t>(base - c0 * 32 + __ffs(bits) - 1);
    __syncwarp();
    for (int i0 = 0; i0 < total; i0 += 32 * kAhead) {
      int at[kAhead];
      float x[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int i = i0 + 32 * j + lane;
        at[j] = i < total ? c0 * 32 + list[i] : -1;
        if (at[j] >= 0) x[j] = load_logit(logits + token(at[j]));
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (at[j] >= 0) store_logit(logits + token(at[j]), penalise(x[j], count[at[j]], true));
    }
    __syncwarp();
  }
  if (allowed != nullptr && !(warp & 1)) close();
  for (int i = threadIdx.x; i < a.bias_width; i += kThreads) {
    const int v = bias_ids[i];
    if (!mine(v)) continue;
    bool last = true;  // an id listed twice: the later entry counts
#pragma unroll 8
    for (int j = i + 1; j < a.bias_width; ++j) last &= bias_ids[j] != v;
    if (!last || (allowed != nullptr && !(static_cast<uint32_t>(allowed[v >> 5]) >> (v & 31) & 1))) continue;
    const int at = place(v);
    const uint32_t n = count[at];
    const float y = load_logit(logits + v) + a.bias_values[req * a.bias_stride + i];
    store_logit(logits + v, penalise(y, n, n != 0 || (prompt[at >> 5] >> (at & 31) & 1)));
  }
}

template <typename T, typename Count, int kThreads>
int launch(LogitArgs a, int rows, cudaStream_t s) {
  using Tab = Tables<Count>;
  constexpr int kMost = kSmem / (1024 / kThreads);
  const int64_t chunks = (static_cast<int64_t>(a.vocab) + 31) / 32, sms = device_sm_count();
  auto bytes = [&](int log2) { return Tab::bytes((chunks + (1 << log2) - 1) >> log2) + Tab::kListBytes * kThreads; };
  // Slices of a row: as few as shared memory allows, since each reads the
  // history; while they leave half the SMs without work twice as many, down to
  // 64 chunks each.
  a.slices_log2 = 0;
  while (bytes(a.slices_log2) > kMost ||
         ((static_cast<int64_t>(rows) << (a.slices_log2 + 1)) <= sms && (chunks >> a.slices_log2) >= 128))
    ++a.slices_log2;
  if ((static_cast<int64_t>(rows) << a.slices_log2) > INT32_MAX) return HCA_E_INVALID;
  // Two CTAs an SM where there are more rows than SMs and a row's tables take
  // half of an SM's memory at most (256 rows of 32000: 9.3 us for 12.6); longer
  // rows would need twice the slices (192 of 151937: 68 us for 57).
  if constexpr (kThreads == 1024)
    if (a.slices_log2 == 0 && rows > sms && Tab::bytes(chunks) + Tab::kListBytes * 512 <= kSmem / 2)
      return launch<T, Count, 512>(a, rows, s);
  static bool done[kMaxDevices] = {};
  if (set_func_attr_once(logit_penalty_kernel<T, Count, kThreads>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost,
                         done) != HCA_OK)
    return HCA_E_CUDA;
  return launch_pdl(logit_penalty_kernel<T, Count, kThreads>, dim3(static_cast<unsigned>(rows) << a.slices_log2),
                    dim3(kThreads), static_cast<size_t>(bytes(a.slices_log2)), s, a);
}

template <typename T>
int by_count(const LogitArgs& a, int rows, cudaStream_t s) {
  return a.token_width <= 65535 ? launch<T, uint16_t, 1024>(a, rows, s) : launch<T, uint32_t, 1024>(a, rows, s);
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
