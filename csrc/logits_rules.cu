// Rules on the logits of a step: penalties for repeated tokens, biases and
// grammar masks, and the greedy token of each resulting row.
//
//   x = logit
//   seen(v):  x = x > 0 ? x / repetition : x * repetition
//   x = x - frequency * count(v);   count(v) > 0:  x = x - presence
//   x = x + bias(v);   grammar bit of v clear:  x = -inf
// seen / count run over the request's committed tokens (count only from the
// end of its prompt) and over the drafted tokens on the row's own tree path.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"
#include "tree_ops.h"

namespace kvs {
namespace {

constexpr int kRuleThreads = 256;
constexpr int kChunk = 4096;
constexpr uint32_t kSeen = 0x80000000u;

struct RuleArgs {
  const void* logits;
  void* out;
  int64_t in_stride, out_stride;
  int R, V, vocab_begin;
  const int32_t* request;
  int B;
  const int32_t* tokens;
  int64_t tokens_stride;
  int tokens_len;
  const int32_t *lens, *prompt;
  const float *repetition, *frequency, *presence;
  const int32_t* bias_ids;
  const float* bias_values;
  int64_t bias_stride, bias_value_stride;
  int num_bias;
  const int32_t* allowed;
  int64_t allowed_stride;
  int allowed_rows;
  const int32_t* allowed_index;
  const int32_t *drafts, *indptr, *mask, *positions;
  int mask_words;
  unsigned long long* best;
};

template <typename T>
__device__ __forceinline__ float load(const T* p);
template <>
__device__ __forceinline__ float load<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float load<bf16>(const bf16* p) { return __bfloat162float(*p); }
template <>
__device__ __forceinline__ float load<__half>(const __half* p) { return __half2float(*p); }
template <typename T>
__device__ __forceinline__ T round_to(float x);
template <>
__device__ __forceinline__ float round_to<float>(float x) { return x; }
template <>
__device__ __forceinline__ bf16 round_to<bf16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half round_to<__half>(float x) { return __float2half_rn(x); }

// Order of the greedy choice as one 64-bit maximum: larger value first, then
// the lower index.  +0 and -0 compare equal; a NaN comes before any number.
__device__ __forceinline__ unsigned long long greedy_key(float x, int v) {
  const uint32_t o = isnan(x) ? 0xffffffffu : float_to_ordered(x + 0.0f);
  return (uint64_t(o) << 32) | uint32_t(~v);
}

template <typename T>
__global__ void __launch_bounds__(kRuleThreads) logits_rules_kernel(RuleArgs a) {
  __shared__ uint32_t s_count[kChunk];
  __shared__ float s_bias[kChunk];
  __shared__ unsigned long long s_best[kRuleThreads / 32];
  const int r = blockIdx.y, v0 = blockIdx.x * kChunk, nv = min(kChunk, a.V - v0);
  const int id0 = a.vocab_begin + v0;
  const int b = a.request ? a.request[r] : r;
  const bool has = b >= 0 && b < a.B;
  for (int i = threadIdx.x; i < kChunk; i += kRuleThreads) {
    s_count[i] = 0;
    s_bias[i] = 0.f;
  }
  __syncthreads();
  const int prompt = has && a.prompt ? a.prompt[b] : 0;
  if (has && a.tokens) {
    const int len = min(a.lens[b], a.tokens_len);
    for (int i = threadIdx.x; i < len; i += kRuleThreads) {
      const int v = a.tokens[b * a.tokens_stride + i] - id0;
      if (v >= 0 && v < nv) {
        atomicOr(&s_count[v], kSeen);
        if (i >= prompt) atomicAdd(&s_count[v], 1u);
      }
    }
  }
  if (has && a.drafts) {
    const int lo = min(max(a.indptr[b], 0), a.R), n = min(a.indptr[b + 1], a.R) - lo;
    for (int j = threadIdx.x; j < n; j += kRuleThreads) {
      const bool on = a.mask ? j < 32 * a.mask_words && (a.mask[int64_t(r) * a.mask_words + (j >> 5)] >> (j & 31)) & 1
                             : lo + j <= r;
      const int v = a.drafts[lo + j] - id0;
      if (on && v >= 0 && v < nv) {
        atomicOr(&s_count[v], kSeen);
        if (a.positions[lo + j] >= prompt) atomicAdd(&s_count[v], 1u);
      }
    }
  }
  if (has && a.num_bias && threadIdx.x == 0) {
    for (int i = 0; i < a.num_bias; ++i) {
      const int id = a.bias_ids[b * a.bias_stride + i], v = id - id0;
      if (id >= 0 && v >= 0 && v < nv) s_bias[v] += a.bias_values[b * a.bias_value_stride + i];
    }
  }
  __syncthreads();
  const float rep = has && a.repetition ? a.repetition[b] : 1.f;
  const float freq = has && a.frequency ? a.frequency[b] : 0.f;
  const float pres = has && a.presence ? a.presence[b] : 0.f;
  int g = -1;
  if (a.allowed) g = a.allowed_index ? a.allowed_index[r] : r;
  const int32_t* bits = g >= 0 && g < a.allowed_rows ? a.allowed + g * a.allowed_stride : nullptr;
  const T* in = reinterpret_cast<const T*>(a.logits) + r * a.in_stride + v0;
  T* out = reinterpret_cast<T*>(a.out) + r * a.out_stride + v0;
  unsigned long long best = 0;
  for (int i = threadIdx.x; i < nv; i += kRuleThreads) {
    float x = load(in + i);
    const uint32_t c = s_count[i];
    if (c & kSeen) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
    const uint32_t count = c & ~kSeen;
    if (count) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, float(count))), pres);
    x = __fadd_rn(x, s_bias[i]);
    if (bits && !((bits[(v0 + i) >> 5] >> ((v0 + i) & 31)) & 1)) x = -INFINITY;
    const T y = round_to<T>(x);
    out[i] = y;
    const unsigned long long key = greedy_key(load(&y), v0 + i);
    best = key > best ? key : best;
  }
  if (a.best) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) {
      const unsigned long long o = __shfl_xor_sync(0xffffffffu, best, m);
      best = o > best ? o : best;
    }
    if ((threadIdx.x & 31) == 0) s_best[threadIdx.x >> 5] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < kRuleThreads / 32; ++w) best = s_best[w] > best ? s_best[w] : best;
      atomicMax(a.best + r, best);
    }
  }
}

__global__ void greedy_finish_kernel(const unsigned long long* best, int R, int vocab_begin, int32_t* greedy,
                                     float* value) {
  const int r = blockIdx.x * blockDim.x + threadIdx.x;
  if (r >= R) return;
  const unsigned long long k = best[r];
  greedy[r] = vocab_begin + int(~uint32_t(k));
  if (value) {
    const uint32_t o = uint32_t(k >> 32);
    value[r] = o == 0xffffffffu ? NAN : ordered_to_float(o);
  }
}

}  // namespace

void process_logits(torch::Tensor logits, torch::Tensor out, c10::optional<torch::Tensor> row_request,
                    c10::optional<torch::Tensor> tokens, c10::optional<torch::Tensor> token_lens,
                    c10::optional<torch::Tensor> prompt_lens, c10::optional<torch::Tensor> repetition,
                    c10::optional<torch::Tensor> frequency, c10::optional<torch::Tensor> presence,
                    c10::optional<torch::Tensor> bias_ids, c10::optional<torch::Tensor> bias_values,
                    c10::optional<torch::Tensor> allowed, c10::optional<torch::Tensor> allowed_index,
                    c10::optional<torch::Tensor> draft_ids, c10::optional<torch::Tensor> indptr,
                    c10::optional<torch::Tensor> tree_mask, c10::optional<torch::Tensor> positions,
                    int64_t vocab_begin, c10::optional<torch::Tensor> greedy, c10::optional<torch::Tensor> greedy_val) {
  const auto dt = logits.scalar_type();
  KVS_CHECK_ARG(logits.is_cuda() && logits.dim() == 2 && logits.stride(1) == 1 &&
                    (dt == at::kBFloat16 || dt == at::kHalf || dt == at::kFloat),
                "process_logits: logits [R, V] bf16, fp16 or fp32 with contiguous rows");
  KVS_CHECK_ARG(out.is_cuda() && out.sizes() == logits.sizes() && out.scalar_type() == dt && out.stride(1) == 1 &&
                    out.device() == logits.device(),
                "process_logits: out has the shape and type of logits");
  const int64_t R = logits.size(0), V = logits.size(1);
  KVS_CHECK_ARG(V >= 1 && vocab_begin >= 0 && vocab_begin + V <= INT32_MAX && R <= 65535,
                "process_logits: vocabulary range or number of rows");
  RuleArgs a{};
  auto on = [&](const torch::Tensor& t, at::ScalarType want, const char* msg) {
    KVS_CHECK_ARG(t.is_cuda() && t.device() == logits.device() && t.scalar_type() == want, msg);
  };
  auto vec = [&](const c10::optional<torch::Tensor>& t, at::ScalarType want, int64_t n, const char* msg) {
    if (!t.has_value()) return;
    on(*t, want, msg);
    KVS_CHECK_ARG(t->dim() == 1 && t->is_contiguous() && t->numel() == n, msg);
  };
  // the number of requests comes from whichever per-request tensor is there
  int64_t B = -1;
  for (const auto* t : {&token_lens, &prompt_lens, &repetition, &frequency, &presence})
    if (t->has_value() && B < 0) B = (*t)->numel();
  if (B < 0 && indptr.has_value()) B = indptr->numel() - 1;
  if (B < 0 && bias_ids.has_value()) B = bias_ids->size(0);
  if (B < 0) B = R;
  KVS_CHECK_ARG(row_request.has_value() || B == R, "process_logits: row_request is needed unless row r is request r");
  vec(row_request, at::kInt, R, "process_logits: row_request int32 [R]");
  vec(token_lens, at::kInt, B, "process_logits: token_lens int32 [B]");
  vec(prompt_lens, at::kInt, B, "process_logits: prompt_lens int32 [B]");
  vec(repetition, at::kFloat, B, "process_logits: repetition fp32 [B]");
  vec(frequency, at::kFloat, B, "process_logits: frequency fp32 [B]");
  vec(presence, at::kFloat, B, "process_logits: presence fp32 [B]");
  vec(indptr, at::kInt, B + 1, "process_logits: indptr int32 [B + 1]");
  vec(draft_ids, at::kInt, R, "process_logits: draft_ids int32 [R]");
  vec(positions, at::kInt, R, "process_logits: positions int32 [R]");
  vec(allowed_index, at::kInt, R, "process_logits: allowed_index int32 [R]");
  vec(greedy, at::kInt, R, "process_logits: greedy int32 [R]");
  vec(greedy_val, at::kFloat, R, "process_logits: greedy_val fp32 [R]");
  KVS_CHECK_ARG(tokens.has_value() == token_lens.has_value(), "process_logits: tokens and token_lens go together");
  KVS_CHECK_ARG(bias_ids.has_value() == bias_values.has_value(), "process_logits: bias_ids and bias_values go together");
  KVS_CHECK_ARG(draft_ids.has_value() == indptr.has_value() && draft_ids.has_value() == positions.has_value(),
                "process_logits: draft_ids, indptr and positions go together");
  KVS_CHECK_ARG(draft_ids.has_value() || !tree_mask.has_value(), "process_logits: tree_mask needs draft_ids");
  KVS_CHECK_ARG(allowed.has_value() || !allowed_index.has_value(), "process_logits: allowed_index needs allowed");
  KVS_CHECK_ARG(greedy.has_value() || !greedy_val.has_value(), "process_logits: greedy_val needs greedy");
  if (tokens.has_value()) {
    on(*tokens, at::kInt, "process_logits: tokens int32 [B, M]");
    KVS_CHECK_ARG(tokens->dim() == 2 && tokens->size(0) == B && tokens->stride(1) == 1 &&
                      tokens->size(1) <= INT32_MAX,
                  "process_logits: tokens int32 [B, M] with contiguous rows");
    a.tokens = tokens->data_ptr<int32_t>();
    a.tokens_stride = tokens->stride(0);
    a.tokens_len = int(tokens->size(1));
    a.lens = token_lens->data_ptr<int32_t>();
  }
  if (bias_ids.has_value()) {
    on(*bias_ids, at::kInt, "process_logits: bias_ids int32 [B, K]");
    on(*bias_values, at::kFloat, "process_logits: bias_values fp32 [B, K]");
    KVS_CHECK_ARG(bias_ids->dim() == 2 && bias_ids->size(0) == B && bias_values->sizes() == bias_ids->sizes() &&
                      bias_ids->stride(1) == 1 && bias_values->stride(1) == 1,
                  "process_logits: bias_ids and bias_values [B, K] with contiguous rows");
    KVS_CHECK_ARG(bias_ids->size(1) <= INT32_MAX, "process_logits: too many biases");
    a.bias_ids = bias_ids->data_ptr<int32_t>();
    a.bias_values = bias_values->data_ptr<float>();
    a.bias_stride = bias_ids->stride(0);
    a.bias_value_stride = bias_values->stride(0);
    a.num_bias = int(bias_ids->size(1));
  }
  if (allowed.has_value()) {
    on(*allowed, at::kInt, "process_logits: allowed int32 [A, ceil(V / 32)]");
    KVS_CHECK_ARG(allowed->dim() == 2 && allowed->stride(1) == 1 && allowed->size(1) >= (V + 31) / 32 &&
                      (allowed_index.has_value() || allowed->size(0) == R) && allowed->size(0) <= INT32_MAX,
                  "process_logits: allowed int32 [A, ceil(V / 32)], A = R without allowed_index");
    a.allowed = allowed->data_ptr<int32_t>();
    a.allowed_stride = allowed->stride(0);
    a.allowed_rows = int(allowed->size(0));
    a.allowed_index = allowed_index.has_value() ? allowed_index->data_ptr<int32_t>() : nullptr;
  }
  if (tree_mask.has_value()) {
    on(*tree_mask, at::kInt, "process_logits: tree_mask int32 [R, W]");
    KVS_CHECK_ARG(tree_mask->dim() == 2 && tree_mask->size(0) == R && tree_mask->is_contiguous() &&
                      tree_mask->size(1) >= 1,
                  "process_logits: tree_mask int32 [R, W]");
    a.mask = tree_mask->data_ptr<int32_t>();
    a.mask_words = int(tree_mask->size(1));
  }
  if (R == 0) return;
  const c10::cuda::CUDAGuard guard(logits.device());
  auto ip = [](const c10::optional<torch::Tensor>& t) { return t.has_value() ? t->data_ptr<int32_t>() : nullptr; };
  auto fp = [](const c10::optional<torch::Tensor>& t) { return t.has_value() ? t->data_ptr<float>() : nullptr; };
  a.logits = logits.data_ptr();
  a.out = out.data_ptr();
  a.in_stride = logits.stride(0);
  a.out_stride = out.stride(0);
  a.R = int(R);
  a.V = int(V);
  a.vocab_begin = int(vocab_begin);
  a.B = int(B);
  a.request = ip(row_request);
  a.prompt = ip(prompt_lens);
  a.repetition = fp(repetition);
  a.frequency = fp(frequency);
  a.presence = fp(presence);
  a.drafts = ip(draft_ids);
  a.indptr = ip(indptr);
  a.positions = ip(positions);
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  torch::Tensor best;
  if (greedy.has_value()) {
    best = torch::zeros({R}, logits.options().dtype(at::kLong));
    a.best = reinterpret_cast<unsigned long long*>(best.data_ptr<int64_t>());
  }
  const dim3 grid(unsigned((V + kChunk - 1) / kChunk), unsigned(R));
  if (dt == at::kBFloat16)
    logits_rules_kernel<bf16><<<grid, kRuleThreads, 0, st>>>(a);
  else if (dt == at::kHalf)
    logits_rules_kernel<__half><<<grid, kRuleThreads, 0, st>>>(a);
  else
    logits_rules_kernel<float><<<grid, kRuleThreads, 0, st>>>(a);
  if (greedy.has_value())
    greedy_finish_kernel<<<unsigned((R + 255) / 256), 256, 0, st>>>(a.best, int(R), int(vocab_begin),
                                                                    greedy->data_ptr<int32_t>(), fp(greedy_val));
  KVS_CUDA_CHECK(cudaGetLastError());
}

}  // namespace kvs
