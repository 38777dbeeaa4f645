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
// latency for one.  A CTA takes a slice of the vocabulary for a few rows.  For
// each run of rows of one request it counts the request's tokens that fall
// into the slice in shared memory (a word an entry, integer atomics, so the
// order does not matter) and lists the entries that any rule touches, the
// request's drafted tokens among them.  Then its warps go their own ways, a
// row or a part of one each: a stream of 16-byte loads and stores that knows
// only the grammar bits, then the listed entries, where a drafted token's
// count adds those on the row's own path.  With the rules inside the stream a
// warp took their branches for nearly every piece, and with the block on one
// row at a time it waited at barriers (8 trees of 32, V = 152064: 82 us; now
// 68 us; 512 rows of 128256 fp32 with 8000 tokens each 200 us = 2.7 TB/s, 218
// in place; one row 7.4 us; in a CUDA graph).  What bounds it now is the count
// before the stream: every slice of a row clears its table, reads the whole
// history and waits for the block, and shared memory admits two CTAs an SM.
// Half of the issue slots are used (48 and 52 %), DRAM to 13 and 30 %; an issued
// instruction stands for 4.3 and 2.5 warps at a barrier, 3.9 and 3.5 at loads.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"
#include "tree_ops.h"

namespace kvs {
namespace {

constexpr int kRuleThreads = 512;
constexpr int kRuleWarps = kRuleThreads / 32;
constexpr int kMaxSlice = 16384;  // entries: 64 KB of counts and 32 KB of list, two CTAs on an SM
constexpr int kMinSlice = 1024;
constexpr int kMaxBias = 2047;
// a count word: bit 31 seen in the prompt, bits 20..30 bias number + 1, bit 19
// drafted, then the count of generated occurrences
constexpr uint32_t kSeen = 0x80000000u;
constexpr int kBiasShift = 20;
constexpr uint32_t kDrafted = 1u << 19;
constexpr uint32_t kCountMask = kDrafted - 1u;

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
__device__ __forceinline__ uint32_t order_of(float x) { return isnan(x) ? 0xffffffffu : float_to_ordered(x + 0.0f); }

// 16 bytes of logits: entries whose bit in `keep` is clear become -inf; the
// largest entry (NaN if there is one).  16-bit types go by pairs.
template <typename T>
struct Pack;
template <>
struct Pack<float> {
  static __device__ __forceinline__ uint4 keep(uint4 w, uint32_t k) {
    w.x = k & 1u ? w.x : 0xff800000u;
    w.y = k & 2u ? w.y : 0xff800000u;
    w.z = k & 4u ? w.z : 0xff800000u;
    w.w = k & 8u ? w.w : 0xff800000u;
    return w;
  }
  static __device__ __forceinline__ float largest(const uint4& w) {
    return max_nan(max_nan(__uint_as_float(w.x), __uint_as_float(w.y)),
                   max_nan(__uint_as_float(w.z), __uint_as_float(w.w)));
  }
};
template <uint32_t kNegInf2>
__device__ __forceinline__ uint4 keep_halves(uint4 w, uint32_t k) {
  auto pair = [](uint32_t x, uint32_t b) {  // b: two bits
    const uint32_t m = (b & 1u) * 0xffffu + (b >> 1 & 1u) * 0xffff0000u;
    return (x & m) | (kNegInf2 & ~m);
  };
  return make_uint4(pair(w.x, k), pair(w.y, k >> 2), pair(w.z, k >> 4), pair(w.w, k >> 6));
}
template <>
struct Pack<bf16> {
  static __device__ __forceinline__ uint4 keep(const uint4& w, uint32_t k) { return keep_halves<0xff80ff80u>(w, k); }
  static __device__ __forceinline__ float largest(const uint4& w) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w);
    const float2 m = __bfloat1622float2(__hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3])));
    return max_nan(m.x, m.y);
  }
};
template <>
struct Pack<__half> {
  static __device__ __forceinline__ uint4 keep(const uint4& w, uint32_t k) { return keep_halves<0xfc00fc00u>(w, k); }
  static __device__ __forceinline__ float largest(const uint4& w) {
    const __half2* h = reinterpret_cast<const __half2*>(&w);
    const float2 m = __half22float2(__hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3])));
    return max_nan(m.x, m.y);
  }
};

// Largest of the warp's 64-bit keys.
__device__ __forceinline__ unsigned long long warp_max(unsigned long long k) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, uint32_t(k >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, uint32_t(k >> 32) == hi ? uint32_t(k) : 0u);
  return (uint64_t(hi) << 32) | lo;
}

constexpr int kMaxRows = 8;   // rows of a CTA
constexpr int kBatch = 4;     // 16-byte pieces of a lane in flight
constexpr int kAhead = 8;     // tokens of a thread read while the table is cleared
constexpr int kPartPieces = 64;  // pieces of a warp's part of a row, at least

template <typename T>
__global__ void __launch_bounds__(kRuleThreads, 2) logits_rules_kernel(const RuleArgs a) {
  pdl_trigger();
  constexpr int VEC = 16 / sizeof(T);
  extern __shared__ uint32_t sm[];
  uint32_t* s_count = sm;                     // [slice]
  uint32_t* s_bits = s_count + a.slice;       // [slice / 32 + 4] entries that a rule may change ...
  uint16_t* s_list = reinterpret_cast<uint16_t*>(s_bits + a.slice / 32 + 4);  // [slice] ... and their list
  float* s_bias = reinterpret_cast<float*>(s_list + a.slice);                 // [num_bias]
  __shared__ int s_listed;
  __shared__ unsigned long long s_best[kMaxRows];
  __shared__ int s_request[kMaxRows];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int v0 = blockIdx.x * a.slice, nv = min(a.slice, a.V - v0), id0 = a.vocab_begin + v0;
  const int row0 = blockIdx.y * a.rows_per_cta, row1 = min(row0 + a.rows_per_cta, a.R);
  if (tid < row1 - row0) {
    const int b = a.request ? a.request[row0 + tid] : row0 + tid;
    s_request[tid] = b >= 0 && b < a.B ? b : -1;
  }
  __syncthreads();
  auto touch = [&](uint32_t v) {
    const uint32_t bit = 1u << (v & 31);
    if (!(atomicOr(&s_bits[v >> 5], bit) & bit)) s_list[atomicAdd(&s_listed, 1)] = uint16_t(v);
  };

  for (int r0 = row0; r0 < row1;) {
    const int b = s_request[r0 - row0];
    int run = 1;
    while (r0 + run < row1 && s_request[r0 + run - row0] == b) ++run;
    const bool has = b >= 0;
    const int prompt = has && a.prompt ? a.prompt[b] : 0;
    int lo = 0, n = 0;
    if (tid < kMaxRows) s_best[tid] = 0;
    if (tid == 0) s_listed = 0;
    if (has) {
      const int len = a.tokens ? min(a.lens[b], a.tokens_len) : 0;
      const int32_t* tok = a.tokens + b * a.tokens_stride;
      int32_t ahead[kAhead];
#pragma unroll
      for (int x = 0; x < kAhead; ++x) ahead[x] = tid + x * kRuleThreads < len ? tok[tid + x * kRuleThreads] : -1;
      if (a.drafts) {
        lo = min(max(a.indptr[b], 0), a.R);
        n = min(a.indptr[b + 1], a.R) - lo;
      }
      for (int i = tid; i < a.slice / 4; i += kRuleThreads) reinterpret_cast<uint4*>(s_count)[i] = make_uint4(0, 0, 0, 0);
      for (int i = tid; i <= a.slice / 32; i += kRuleThreads) s_bits[i] = 0;
      __syncthreads();
      auto count = [&](int32_t id, int i) {
        const uint32_t v = uint32_t(id) - uint32_t(id0);
        if (id >= 0 && v < uint32_t(nv)) {
          if (i >= prompt) atomicAdd(&s_count[v], 1u);
          else atomicOr(&s_count[v], kSeen);
          touch(v);
        }
      };
#pragma unroll
      for (int x = 0; x < kAhead; ++x) count(ahead[x], tid + x * kRuleThreads);
      for (int i0 = kAhead * kRuleThreads; i0 < len; i0 += kAhead * kRuleThreads) {
#pragma unroll
        for (int x = 0; x < kAhead; ++x) {
          const int i = i0 + tid + x * kRuleThreads;
          ahead[x] = i < len ? tok[i] : -1;
        }
#pragma unroll
        for (int x = 0; x < kAhead; ++x) count(ahead[x], i0 + tid + x * kRuleThreads);
      }
      for (int j = tid; j < n; j += kRuleThreads) {
        const int32_t id = a.drafts[lo + j];
        const uint32_t v = uint32_t(id) - uint32_t(id0);
        if (id >= 0 && v < uint32_t(nv)) {
          atomicOr(&s_count[v], kDrafted);
          touch(v);
        }
      }
      if (a.num_bias && warp == kRuleWarps - 1) {
        // in the order of the list, so that an id listed several times gets
        // the same sum every time; the first of equal ids owns the sum
        for (int i0 = 0; i0 < a.num_bias; i0 += 32) {
          const int i = i0 + lane;
          const int id = i < a.num_bias ? a.bias_ids[b * a.bias_stride + i] : -1;
          const uint32_t v = uint32_t(id) - uint32_t(id0);
          const bool in = id >= 0 && v < uint32_t(nv);
          const uint32_t any = __ballot_sync(0xffffffffu, in);
          if (!any) continue;
          const float value = in ? a.bias_values[b * a.bias_value_stride + i] : 0.f;
          const uint32_t same = __match_any_sync(0xffffffffu, in ? int(v) : -1 - lane);
          float sum = 0.f;
          int number = -1;
          if (in) {
            number = int((s_count[v] & ~kSeen) >> kBiasShift) - 1;
            if (number >= 0) sum = s_bias[number];
          }
          for (uint32_t rest = any; rest; rest &= rest - 1) {
            const int from = __ffs(rest) - 1;
            const float x = __shfl_sync(0xffffffffu, value, from);
            if ((same >> from) & 1u) sum = __fadd_rn(sum, x);
          }
          if (in && __ffs(same) - 1 == lane) {
            if (number < 0) {
              number = i;
              atomicOr(&s_count[v], uint32_t(i + 1) << kBiasShift);
              touch(v);
            }
            s_bias[number] = sum;
          }
          __syncwarp();
        }
      }
    }
    __syncthreads();

    // one row, or a part of one, to each warp
    const int row_parts = kRuleWarps / run, x = warp / row_parts, part = warp % row_parts, r = r0 + x;
    const T* in = reinterpret_cast<const T*>(a.logits) + r * a.in_stride + v0;
    T* out = reinterpret_cast<T*>(a.out) + r * a.out_stride + v0;
    // 16-byte pieces where input and output have one misalignment
    const uint32_t skew = reinterpret_cast<uintptr_t>(in) & 15;
    const bool wide = skew == (reinterpret_cast<uintptr_t>(out) & 15);
    const int head = wide ? min(nv, int((16 - skew) & 15) / int(sizeof(T))) : nv, pieces = (nv - head) / VEC;
    const int parts = wide ? max(1, min(row_parts, (pieces + kPartPieces - 1) / kPartPieces)) : row_parts;
    if (x < run && part < parts) {
      int g = -1;
      if (a.allowed) g = a.allowed_index ? a.allowed_index[r] : r;
      // grammar words of the slice (slices begin at whole words)
      const uint32_t* bits = g >= 0 && g < a.allowed_rows
                                 ? reinterpret_cast<const uint32_t*>(a.allowed + g * a.allowed_stride) + (v0 >> 5)
                                 : nullptr;
      // largest entry of the lane's 16-byte pieces (as an ordered integer) and
      // the first piece that has it; largest key of the other entries
      uint32_t top = 0;
      int top_piece = -1;
      unsigned long long best = 0;
      auto touched_at = [&](int i) { return has && (s_bits[i >> 5] >> (i & 31)) & 1u; };
      auto free_at = [&](int i) { return !bits || (bits[i >> 5] >> (i & 31)) & 1u; };
      auto consider = [&](float y, int i) {
        const unsigned long long key = greedy_key(y, v0 + i);
        best = key > best ? key : best;
      };
      const int per = (pieces + parts - 1) / parts, p_end = min(pieces, (part + 1) * per);
      for (int p0 = part * per; p0 < p_end; p0 += 32 * kBatch) {
        uint4 raw[kBatch];
        uint32_t free[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int p = p0 + u * 32 + lane, i = head + p * VEC, at = i >> 5;
          free[u] = ~0u;
          if (p < p_end) {
            raw[u] = *reinterpret_cast<const uint4*>(in + i);
            if (bits) free[u] = __funnelshift_r(bits[at], (i & 31) + VEC > 32 ? bits[at + 1] : 0u, i & 31);
          }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int p = p0 + u * 32 + lane, i = head + p * VEC, at = i >> 5;
          if (p >= p_end) continue;
          if (bits) raw[u] = Pack<T>::keep(raw[u], free[u]);
          *reinterpret_cast<uint4*>(out + i) = raw[u];
          if (a.best) {
            // Listed entries count as -inf here; their own value comes in the
            // second pass and is no smaller.
            if (has) {
              const uint32_t listed = __funnelshift_r(s_bits[at], s_bits[at + 1], i & 31);
              if (listed & ((1u << VEC) - 1u)) raw[u] = Pack<T>::keep(raw[u], ~listed);
            }
            const uint32_t o = order_of(Pack<T>::largest(raw[u]));
            if (o > top) {
              top = o;
              top_piece = p;
            }
          }
        }
      }
      auto one = [&](int i) {
        const T y = free_at(i) ? in[i] : round_to<T>(-INFINITY);
        out[i] = y;
        if (!touched_at(i)) consider(load(&y), i);
      };
      const int at = part * 32 + lane, step = parts * 32;
      for (int i = at; i < head; i += step) one(i);
      for (int i = head + pieces * VEC + at; i < nv; i += step) one(i);
      if (has) {
        // The stream left listed entries as they were (or -inf), so they can
        // be read back also where the output is the input.
        __syncwarp();
        asm volatile("bar.sync %0, %1;" ::"r"(1 + x), "r"(parts * 32) : "memory");
        const float rep = a.repetition ? a.repetition[b] : 1.f;
        const float freq = a.frequency ? a.frequency[b] : 0.f;
        const float pres = a.presence ? a.presence[b] : 0.f;
        const int listed = s_listed;
        for (int j = at; j < listed; j += step) {
          const int i = s_list[j];
          T y = round_to<T>(-INFINITY);
          if (free_at(i)) {
            float v = load(in + i);
            const uint32_t c = s_count[i], number = (c & ~kSeen) >> kBiasShift;
            uint32_t times = c & kCountMask;
            bool seen = c & kSeen;
            if (c & kDrafted) {  // on the row's own path
              for (int k = 0; k < n; ++k) {
                const bool on = a.mask ? k < 32 * a.mask_words &&
                                             (a.mask[int64_t(r) * a.mask_words + (k >> 5)] >> (k & 31)) & 1
                                       : lo + k <= r;
                if (!on || a.drafts[lo + k] != id0 + i) continue;
                if (a.positions[lo + k] >= prompt) ++times;
                else seen = true;
              }
            }
            if (seen || times) v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
            if (times) v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, float(times))), pres);
            if (number) v = __fadd_rn(v, s_bias[number - 1]);
            y = round_to<T>(v);
            out[i] = y;
          }
          consider(load(&y), i);
        }
      }
      if (a.best) {
        // where in the piece: only the lanes that hold the warp's largest entry
        __syncwarp();
        const uint32_t highest = __reduce_max_sync(0xffffffffu, top);
        if (top_piece >= 0 && top == highest) {
          const int i = head + top_piece * VEC;
          for (int e = 0; e < VEC; ++e) {
            const T y = out[i + e];
            consider(touched_at(i + e) ? -INFINITY : load(&y), i + e);
          }
        }
        __syncwarp();
        best = warp_max(best);
        if (lane == 0) atomicMax(&s_best[x], best);
      }
    }
    __syncthreads();
    if (a.best && tid < run) a.best[int64_t(r0 + tid) * a.slices + blockIdx.x] = s_best[tid];
    r0 += run;
    if (r0 < row1) __syncthreads();
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
                  "process_logits: tokens int32 [B, M] with contiguous rows, M + R below 2^19");
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
  int64_t slice = kMaxSlice, rows = kMaxRows;
  auto ctas = [&] { return ((V + slice - 1) / slice) * ((R + rows - 1) / rows); };
  while (rows > 1 && (rows > (R + B - 1) / B || ctas() < 2 * 2 * kNumSMs)) rows /= 2;
  while (slice > kMinSlice && ctas() < 2 * kNumSMs) slice /= 2;
  a.slice = int(slice);
  a.slices = int((V + slice - 1) / slice);
  a.rows_per_cta = int(rows);
  const dim3 grid{unsigned(a.slices), unsigned((R + rows - 1) / rows)};
  const size_t smem = size_t(slice + slice / 32 + 4 + slice / 2 + a.num_bias) * 4;
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
