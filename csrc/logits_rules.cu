// Rules on the logits of a step: penalties for repeated tokens, biases and
// grammar masks, and the greedy token of each resulting row.
//
//   x = logit
//   seen(v):  x = x > 0 ? x / repetition : x * repetition
//   x = x - frequency * count(v);   count(v) > 0:  x = x - presence
//   x = x + bias(v);   grammar bit of v clear:  x = -inf
// seen / count run over the request's committed tokens (count only from the
// end of its prompt) and over the drafted tokens on the row's own tree path.
//
// Every logit is read and written once: bound by HBM for many rows, by
// latency for one.  A CTA takes a slice of the vocabulary for a few rows: it
// counts the request's tokens that fall into the slice in shared memory (a
// word an entry, integer atomics, so the order does not matter), once for all
// rows of a request, and marks the entries that any rule touches in a bit
// map.  The rows then stream through 16-byte loads and stores; eight entries
// whose bits are clear cost two bit tests, the others take the slow path.
// A row's path tokens are added before it and taken back after it.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"
#include "tree_ops.h"

namespace kvs {
namespace {

constexpr int kRuleThreads = 512;
constexpr int kMaxSlice = 16384;  // entries: 64 KB of counts, two CTAs on an SM
constexpr int kMinSlice = 1024;
constexpr int kMaxBias = 2047;
// a count word: bit 31 seen in the prompt, bits 20..30 bias number + 1, then
// the count of generated occurrences
constexpr uint32_t kSeen = 0x80000000u;
constexpr int kBiasShift = 20;
constexpr uint32_t kCountMask = (1u << kBiasShift) - 1u;

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
  int slice, slices, rows_per_cta;
  unsigned long long* best;  // [R, slices]
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

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

template <typename T>
__global__ void __launch_bounds__(kRuleThreads, 2) logits_rules_kernel(const RuleArgs a) {
  pdl_trigger();
  constexpr int VEC = 16 / sizeof(T);
  extern __shared__ uint32_t sm[];
  __shared__ unsigned long long s_best[kRuleThreads / 32];
  uint32_t* s_count = sm;                     // [slice]
  uint32_t* s_bits = s_count + a.slice;       // [slice / 32 + 1] entries that a rule may change
  float* s_bias = reinterpret_cast<float*>(s_bits + a.slice / 32 + 1);  // [num_bias]
  const int tid = threadIdx.x, lane = tid & 31;
  const int v0 = blockIdx.x * a.slice, nv = min(a.slice, a.V - v0), id0 = a.vocab_begin + v0;
  const int row0 = blockIdx.y * a.rows_per_cta, row1 = min(row0 + a.rows_per_cta, a.R);
  int counted = -1;  // request whose tokens the table holds
  for (int r = row0; r < row1; ++r) {
    const int b = a.request ? a.request[r] : r;
    const bool has = b >= 0 && b < a.B;
    const int prompt = has && a.prompt ? a.prompt[b] : 0;
    if (has && b != counted) {
      for (int i = tid; i < a.slice / 4; i += kRuleThreads) reinterpret_cast<uint4*>(s_count)[i] = make_uint4(0, 0, 0, 0);
      for (int i = tid; i <= a.slice / 32; i += kRuleThreads) s_bits[i] = 0;
      __syncthreads();
      if (a.tokens) {
        const int len = min(a.lens[b], a.tokens_len);
        const int32_t* tok = a.tokens + b * a.tokens_stride;
#pragma unroll 8
        for (int i = tid; i < len; i += kRuleThreads) {
          const uint32_t v = uint32_t(tok[i]) - uint32_t(id0);
          if (v < uint32_t(nv)) {
            if (i >= prompt) atomicAdd(&s_count[v], 1u);
            else atomicOr(&s_count[v], kSeen);
            atomicOr(&s_bits[v >> 5], 1u << (v & 31));
          }
        }
      }
      if (a.num_bias && tid < 32) {
        // in the order of the list, so that an id listed several times gets
        // the same sum every time; the first of equal ids owns the sum
        for (int i0 = 0; i0 < a.num_bias; i0 += 32) {
          const int i = i0 + lane;
          const int id = i < a.num_bias ? a.bias_ids[b * a.bias_stride + i] : -1;
          const uint32_t v = uint32_t(id) - uint32_t(id0);
          const bool in = id >= 0 && v < uint32_t(nv);
          const float value = in ? a.bias_values[b * a.bias_value_stride + i] : 0.f;
          const uint32_t same = __match_any_sync(0xffffffffu, in ? int(v) : -1 - lane);
          float sum = 0.f;
          int number = -1;
          if (in) {
            number = int((s_count[v] & ~kSeen) >> kBiasShift) - 1;
            if (number >= 0) sum = s_bias[number];
          }
          for (uint32_t rest = 0xffffffffu; rest; rest &= rest - 1) {
            const int from = __ffs(rest) - 1;
            const float x = __shfl_sync(0xffffffffu, value, from);
            if ((same >> from) & 1u) sum = __fadd_rn(sum, x);
          }
          if (in && __ffs(same) - 1 == lane) {
            if (number < 0) {
              number = i;
              atomicOr(&s_count[v], uint32_t(i + 1) << kBiasShift);
              atomicOr(&s_bits[v >> 5], 1u << (v & 31));
            }
            s_bias[number] = sum;
          }
          __syncwarp();
        }
      }
      counted = b;
    }
    // the row's own path
    int lo = 0, n = 0;
    if (has && a.drafts) {
      lo = min(max(a.indptr[b], 0), a.R);
      n = min(a.indptr[b + 1], a.R) - lo;
    }
    auto path = [&](auto&& use) {
      for (int j = tid; j < n; j += kRuleThreads) {
        const bool on = a.mask ? j < 32 * a.mask_words && (a.mask[int64_t(r) * a.mask_words + (j >> 5)] >> (j & 31)) & 1
                               : lo + j <= r;
        const uint32_t v = on ? uint32_t(a.drafts[lo + j]) - uint32_t(id0) : 0xffffffffu;
        if (v < uint32_t(nv)) use(v, a.positions[lo + j] >= prompt);
      }
    };
    bool lasting = false;
    path([&](uint32_t v, bool made) {
      if (made) atomicAdd(&s_count[v], 1u);
      else lasting = true, atomicOr(&s_count[v], kSeen);
      atomicOr(&s_bits[v >> 5], 1u << (v & 31));
    });
    if (__syncthreads_or(lasting)) counted = -1;  // a prompt token of the path stays in the table

    const float rep = has && a.repetition ? a.repetition[b] : 1.f;
    const float freq = has && a.frequency ? a.frequency[b] : 0.f;
    const float pres = has && a.presence ? a.presence[b] : 0.f;
    int g = -1;
    if (a.allowed) g = a.allowed_index ? a.allowed_index[r] : r;
    // grammar words of the slice (slices begin at whole words)
    const uint32_t* bits =
        g >= 0 && g < a.allowed_rows ? reinterpret_cast<const uint32_t*>(a.allowed + g * a.allowed_stride) + (v0 >> 5) : nullptr;
    const T* in = reinterpret_cast<const T*>(a.logits) + r * a.in_stride + v0;
    T* out = reinterpret_cast<T*>(a.out) + r * a.out_stride + v0;
    auto rules = [&](float x, int i) {  // entry i of the slice, not masked
      const uint32_t c = s_count[i], count = c & kCountMask, number = (c & ~kSeen) >> kBiasShift;
      if ((c & kSeen) || count) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
      if (count) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, float(count))), pres);
      if (number) x = __fadd_rn(x, s_bias[number - 1]);
      return x;
    };
    float top = NAN;              // largest value of the 16-byte pieces so far (NaN: none yet, or it is one)
    unsigned long long best = 0;  // largest key so far
    auto one = [&](int i) {
      float x = load(in + i);
      if (has && (s_bits[i >> 5] >> (i & 31)) & 1u) x = rules(x, i);
      if (bits && !((bits[i >> 5] >> (i & 31)) & 1u)) x = -INFINITY;
      const T y = round_to<T>(x);
      out[i] = y;
      const unsigned long long key = greedy_key(load(&y), v0 + i);
      best = key > best ? key : best;
    };
    // 16-byte pieces where input and output have one misalignment
    const int skew = int((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T));
    const bool wide = (reinterpret_cast<uintptr_t>(in) & 15) == (reinterpret_cast<uintptr_t>(out) & 15);
    const int head = wide ? min(nv, (VEC - skew) % VEC) : nv, pieces = (nv - head) / VEC;
    for (int i = tid; i < head; i += kRuleThreads) one(i);
    for (int i = head + pieces * VEC + tid; i < nv; i += kRuleThreads) one(i);
#pragma unroll 2
    for (int p = tid; p < pieces; p += kRuleThreads) {
      const int i = head + p * VEC, w = i >> 5;
      uint4 raw = *reinterpret_cast<const uint4*>(in + i);
      uint32_t touched = 0, free = ~0u;
      if (has) touched = __funnelshift_r(s_bits[w], s_bits[w + 1], i & 31);
      if (bits) free = __funnelshift_r(bits[w], (i & 31) + VEC > 32 ? bits[w + 1] : 0u, i & 31);
      constexpr uint32_t kAll = (1u << VEC) - 1u;
      T* e = reinterpret_cast<T*>(&raw);
      if ((touched | ~free) & kAll) {
#pragma unroll
        for (int x = 0; x < VEC; ++x) {
          if (!((free >> x) & 1u)) e[x] = round_to<T>(-INFINITY);
          else if ((touched >> x) & 1u) e[x] = round_to<T>(rules(load(e + x), i + x));
        }
      }
      *reinterpret_cast<uint4*>(out + i) = raw;
      if (a.best) {
        float mx = load(e);
#pragma unroll
        for (int x = 1; x < VEC; ++x) mx = max_nan(mx, load(e + x));
        if (!(mx <= top)) {  // larger than all before, or NaN, or the first
          top = mx;
#pragma unroll
          for (int x = 0; x < VEC; ++x) {
            const unsigned long long key = greedy_key(load(e + x), v0 + i + x);
            best = key > best ? key : best;
          }
        }
      }
    }
    if (a.best) {
#pragma unroll
      for (int m = 16; m > 0; m >>= 1) {
        const unsigned long long o = __shfl_xor_sync(0xffffffffu, best, m);
        best = o > best ? o : best;
      }
      if (lane == 0) s_best[tid >> 5] = best;
    }
    __syncthreads();
    if (a.best && tid == 0) {
      for (int w = 1; w < kRuleThreads / 32; ++w) best = s_best[w] > best ? s_best[w] : best;
      a.best[int64_t(r) * a.slices + blockIdx.x] = best;
    }
    if (counted >= 0 && r + 1 < row1)
      path([&](uint32_t v, bool) { atomicSub(&s_count[v], 1u); });
    __syncthreads();
  }
}

// Largest key of a row's slices, a warp a row.
__global__ void __launch_bounds__(128) greedy_finish_kernel(const unsigned long long* best, int R, int slices,
                                                            int vocab_begin, int32_t* greedy, float* value) {
  pdl_wait();
  const int r = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (r >= R) return;
  unsigned long long k = 0;
  for (int i = lane; i < slices; i += 32) {
    const unsigned long long o = best[int64_t(r) * slices + i];
    k = o > k ? o : k;
  }
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) {
    const unsigned long long o = __shfl_xor_sync(0xffffffffu, k, m);
    k = o > k ? o : k;
  }
  if (lane != 0) return;
  greedy[r] = vocab_begin + int(~uint32_t(k));
  if (value) {
    const uint32_t o = uint32_t(k >> 32);
    value[r] = o == 0xffffffffu ? NAN : ordered_to_float(o);
  }
}

template <typename T>
void launch_rules(const RuleArgs& a, dim3 grid, size_t smem, cudaStream_t st) {
  KVS_CUDA_CHECK(cudaFuncSetAttribute(logits_rules_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
  logits_rules_kernel<T><<<grid, kRuleThreads, smem, st>>>(a);
  KVS_CUDA_CHECK(cudaGetLastError());
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
                      tokens->size(1) + R < int64_t(kCountMask),
                  "process_logits: tokens int32 [B, M] with contiguous rows, M below 2^20");
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
    KVS_CHECK_ARG(bias_ids->size(1) <= kMaxBias, "process_logits: at most 2047 biases a request");
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
  // Rows of a CTA share one count of their request's tokens, and a wide slice
  // reads the tokens less often (16384 entries: 8 to 10 times a row); but
  // first the GPU's 2 x 148 places have to be filled.
  int64_t slice = kMaxSlice, rows = 8;
  auto ctas = [&] { return ((V + slice - 1) / slice) * ((R + rows - 1) / rows); };
  while (rows > 1 && ctas() < 2 * 2 * kNumSMs) rows /= 2;
  while (slice > kMinSlice && ctas() < 2 * kNumSMs) slice /= 2;
  a.slice = int(slice);
  a.slices = int((V + slice - 1) / slice);
  a.rows_per_cta = int(rows);
  const dim3 grid{unsigned(a.slices), unsigned((R + rows - 1) / rows)};
  const size_t smem = size_t(slice + slice / 32 + 1 + a.num_bias) * 4;
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  torch::Tensor best;
  if (greedy.has_value()) {
    best = torch::empty({R * a.slices}, logits.options().dtype(at::kLong));
    a.best = reinterpret_cast<unsigned long long*>(best.data_ptr<int64_t>());
  }
  if (dt == at::kBFloat16) launch_rules<bf16>(a, grid, smem, st);
  else if (dt == at::kHalf) launch_rules<__half>(a, grid, smem, st);
  else launch_rules<float>(a, grid, smem, st);
  if (greedy.has_value())
    launch_pdl(greedy_finish_kernel, dim3(unsigned((R + 3) / 4)), dim3(128), 0, st, a.best, int(R), a.slices,
               int(vocab_begin), greedy->data_ptr<int32_t>(), fp(greedy_val));
}

}  // namespace kvs
