// Attention of drafted trees over the paged KV cache.
//
// Row r of request b (node i of its tree) attends to the request's ctx_b
// committed tokens in the cache and to the tree rows j of the step with bit j
// of mask(r) set (without a mask: j <= i):
//   o = sum_t p_t v_t,  p = softmax_t(scale q . k_t);  nothing visible: o = 0.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"
#include "ops.h"

namespace kvs {
namespace {

struct TreeArgs {
  const void *q, *kt, *vt, *kc, *vc;
  void* out;
  int64_t q_r, q_h, kt_r, kt_h, vt_r, vt_h, out_r, out_h;
  int64_t kc_b, kc_t, kc_h, vc_b, vc_t, vc_h;
  const int32_t *tables, *ctx, *indptr, *mask;
  int64_t table_stride;
  int width, words, R, B, group, bs;
  float scale_log2;
};

template <typename T>
__device__ __forceinline__ float as_float(T v);
template <>
__device__ __forceinline__ float as_float<bf16>(bf16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float as_float<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ bf16 from_float<bf16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

template <typename T, int D>
__global__ void __launch_bounds__(128) tree_attention_kernel(TreeArgs a) {
  constexpr int E = D / 32;
  __shared__ float s_m[4], s_l[4], s_o[4][D];
  const int h = blockIdx.x, r = blockIdx.y, kvh = h / a.group;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int b = 0;
  for (int lo = 0, hi = a.B; hi - lo > 0;) {
    const int mid = (lo + hi) >> 1;
    if (a.indptr[mid + 1] > r) { hi = mid; b = mid; } else { lo = mid + 1; b = lo; }
  }
  T* out = reinterpret_cast<T*>(a.out) + r * a.out_r + h * a.out_h;
  if (b >= a.B) {
    for (int d = threadIdx.x; d < D; d += 128) out[d] = from_float<T>(0.f);
    return;
  }
  const int lo = max(a.indptr[b], 0), n = min(a.indptr[b + 1], a.R) - lo;
  const int ctx = int(max(min(int64_t(a.ctx[b]), int64_t(a.width) * a.bs), int64_t(0)));
  float q[E], o[E], m = -INFINITY, l = 0.f;
  for (int e = 0; e < E; ++e) {
    q[e] = as_float(reinterpret_cast<const T*>(a.q)[r * a.q_r + h * a.q_h + lane + 32 * e]) * a.scale_log2;
    o[e] = 0.f;
  }
  for (int t = warp; t < ctx + n; t += 4) {
    const T *k, *v;
    if (t < ctx) {
      const int64_t blk = a.tables[b * a.table_stride + t / a.bs];
      k = reinterpret_cast<const T*>(a.kc) + blk * a.kc_b + (t % a.bs) * a.kc_t + kvh * a.kc_h;
      v = reinterpret_cast<const T*>(a.vc) + blk * a.vc_b + (t % a.bs) * a.vc_t + kvh * a.vc_h;
    } else {
      const int j = t - ctx;
      const bool on = a.mask ? j < 32 * a.words && (a.mask[int64_t(r) * a.words + (j >> 5)] >> (j & 31)) & 1
                             : lo + j <= r;
      if (!on) continue;
      k = reinterpret_cast<const T*>(a.kt) + (lo + j) * a.kt_r + kvh * a.kt_h;
      v = reinterpret_cast<const T*>(a.vt) + (lo + j) * a.vt_r + kvh * a.vt_h;
    }
    float s = 0.f;
    for (int e = 0; e < E; ++e) s = fmaf(q[e], as_float(k[lane + 32 * e]), s);
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    const float mx = fmaxf(m, s);
    const float f = m == -INFINITY ? 0.f : exp2f(m - mx), p = mx == -INFINITY ? 0.f : exp2f(s - mx);
    l = l * f + p;
    for (int e = 0; e < E; ++e) o[e] = fmaf(p, as_float(v[lane + 32 * e]), o[e] * f);
    m = mx;
  }
  if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
  for (int e = 0; e < E; ++e) s_o[warp][lane + 32 * e] = o[e];
  __syncthreads();
  float mx = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  for (int d = threadIdx.x; d < D; d += 128) {
    float lsum = 0.f, acc = 0.f;
    for (int w = 0; w < 4 && mx != -INFINITY; ++w) {
      const float f = exp2f(s_m[w] - mx);
      lsum += s_l[w] * f;
      acc += s_o[w][d] * f;
    }
    out[d] = from_float<T>(mx == -INFINITY ? 0.f : acc / lsum);
  }
}

}  // namespace

void paged_tree_attention(torch::Tensor q, torch::Tensor k_tree, torch::Tensor v_tree, torch::Tensor k_cache,
                          torch::Tensor v_cache, torch::Tensor block_tables, torch::Tensor ctx_lens,
                          torch::Tensor indptr, c10::optional<torch::Tensor> tree_mask, double scale,
                          torch::Tensor out) {
  const auto dt = q.scalar_type();
  KVS_CHECK_ARG(q.is_cuda() && (dt == at::kBFloat16 || dt == at::kHalf), "tree attention: bf16 or fp16 CUDA tensors");
  for (const torch::Tensor* t : {&k_tree, &v_tree, &k_cache, &v_cache, &out})
    KVS_CHECK_ARG(t->is_cuda() && t->scalar_type() == dt && t->device() == q.device(),
                  "tree attention: q, K, V and out have one type and device");
  KVS_CHECK_ARG(q.dim() == 3 && out.dim() == 3 && out.sizes() == q.sizes() && k_tree.dim() == 3 &&
                    v_tree.sizes() == k_tree.sizes() && k_cache.dim() == 4 && v_cache.sizes() == k_cache.sizes(),
                "tree attention: q/out [R, Hq, D], k_tree/v_tree [R, Hkv, D], caches [blocks, block_size, Hkv, D]");
  const int64_t R = q.size(0), Hq = q.size(1), D = q.size(2), Hkv = k_cache.size(2);
  KVS_CHECK_ARG(D == 64 || D == 128, "tree attention: head_dim must be 64 or 128");
  KVS_CHECK_ARG(Hkv >= 1 && Hq % Hkv == 0 && k_tree.size(0) == R && k_tree.size(1) == Hkv && k_tree.size(2) == D &&
                    k_cache.size(3) == D,
                "tree attention: head layout");
  for (const torch::Tensor* t : {&q, &k_tree, &v_tree, &k_cache, &v_cache, &out}) {
    bool ok = t->stride(-1) == 1 && (reinterpret_cast<uintptr_t>(t->data_ptr()) & 15) == 0;
    for (int64_t d = 0; d + 1 < t->dim(); ++d) ok = ok && t->stride(d) % 8 == 0;
    KVS_CHECK_ARG(ok, "tree attention: head rows must be contiguous and start at 16-byte boundaries");
  }
  const int64_t B = ctx_lens.numel();
  for (const torch::Tensor* t : {&ctx_lens, &indptr})
    KVS_CHECK_ARG(t->is_cuda() && t->device() == q.device() && t->scalar_type() == at::kInt && t->dim() == 1 &&
                      t->is_contiguous(),
                  "tree attention: ctx_lens, indptr are int32 vectors");
  KVS_CHECK_ARG(B >= 1 && indptr.numel() == B + 1, "tree attention: ctx_lens [B], indptr [B + 1]");
  KVS_CHECK_ARG(block_tables.is_cuda() && block_tables.device() == q.device() && block_tables.dim() == 2 &&
                    block_tables.scalar_type() == at::kInt && block_tables.size(0) == B &&
                    block_tables.stride(1) == 1,
                "tree attention: block_tables [B, W] int32 with contiguous rows");
  TreeArgs a{};
  if (tree_mask.has_value()) {
    KVS_CHECK_ARG(tree_mask->is_cuda() && tree_mask->device() == q.device() && tree_mask->dim() == 2 &&
                      tree_mask->scalar_type() == at::kInt && tree_mask->is_contiguous() && tree_mask->size(0) == R &&
                      tree_mask->size(1) >= 1,
                  "tree attention: tree_mask [R, W] int32");
    a.mask = tree_mask->data_ptr<int32_t>();
    a.words = int(tree_mask->size(1));
  }
  if (R == 0) return;
  KVS_CHECK_ARG(R <= 65535, "tree attention: at most 65535 rows");
  const c10::cuda::CUDAGuard guard(q.device());
  a.q = q.data_ptr();
  a.kt = k_tree.data_ptr();
  a.vt = v_tree.data_ptr();
  a.kc = k_cache.data_ptr();
  a.vc = v_cache.data_ptr();
  a.out = out.data_ptr();
  a.q_r = q.stride(0);
  a.q_h = q.stride(1);
  a.kt_r = k_tree.stride(0);
  a.kt_h = k_tree.stride(1);
  a.vt_r = v_tree.stride(0);
  a.vt_h = v_tree.stride(1);
  a.out_r = out.stride(0);
  a.out_h = out.stride(1);
  a.kc_b = k_cache.stride(0);
  a.kc_t = k_cache.stride(1);
  a.kc_h = k_cache.stride(2);
  a.vc_b = v_cache.stride(0);
  a.vc_t = v_cache.stride(1);
  a.vc_h = v_cache.stride(2);
  a.tables = block_tables.data_ptr<int32_t>();
  a.table_stride = block_tables.stride(0);
  a.width = int(block_tables.size(1));
  a.ctx = ctx_lens.data_ptr<int32_t>();
  a.indptr = indptr.data_ptr<int32_t>();
  a.R = int(R);
  a.B = int(B);
  a.group = int(Hq / Hkv);
  a.bs = int(k_cache.size(1));
  a.scale_log2 = float(scale * 1.4426950408889634);
  const dim3 grid{unsigned(Hq), unsigned(R)};
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  if (dt == at::kBFloat16) {
    if (D == 128) tree_attention_kernel<bf16, 128><<<grid, 128, 0, st>>>(a);
    else tree_attention_kernel<bf16, 64><<<grid, 128, 0, st>>>(a);
  } else {
    if (D == 128) tree_attention_kernel<__half, 128><<<grid, 128, 0, st>>>(a);
    else tree_attention_kernel<__half, 64><<<grid, 128, 0, st>>>(a);
  }
  KVS_CUDA_CHECK(cudaGetLastError());
}

}  // namespace kvs
