// Greedy verification of a drafted tree and commit of the accepted path.
//
// Node 0 of a request's tree is its last chosen token, which is certain.
// From cur = 0: while a child c of cur (the lowest one) carries the token that
// the model chose after cur (draft[c] == target[cur]), cur = c.  The nodes
// passed are the path; the model's choice after the last one is the next
// token.  The K/V rows of the path go from the step's staging rows to the
// cache slots of positions ctx, ctx + 1, ..., for every layer in one launch.
//
// Each row of K or V is read and written once; a single request is bound by
// latency.  A full batch is not bound by HBM (11 % of it) but by the walk, at
// whose barriers most stalled warps wait, and the index arithmetic of every
// 16-byte word (55 % of the issue slots).  A CTA takes some (layer, part) planes
// of one request and repeats the walk over its few hundred bytes in shared
// memory, instead of waiting for another launch to write the path down; it
// takes more planes as requests fill the GPU, so that the walk's latency is
// paid once (128 trees, 56 planes of 1 KB rows: 20 us, 22.8 with a CTA a
// plane; one tree of 32 layers 3.7 us; in a CUDA graph).
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"
#include "tree_ops.h"

namespace kvs {
namespace {

constexpr int kCommitThreads = 256;
constexpr int kMaxTree = 1024;
constexpr int kCommitCtas = 8 * kNumSMs;  // CTAs of a full GPU's batch; 40 registers a thread let six on an SM at a time

struct CommitArgs {
  const int32_t *drafts, *targets, *parents, *indptr, *ctx, *slots;
  int R;
  const uint4* src;  // staging rows [L, 2, R, Hkv, D], strides in 16-byte words
  int64_t src_l, src_p, src_r, src_h;
  uint4* dst;  // cache [L, 2, blocks, bs, Hkv, D]
  int64_t dst_l, dst_p, dst_b, dst_t, dst_h;
  int planes, planes_per_cta, heads, words, bs;  // words: 16-byte words of one head's row
  int64_t num_slots;
  int32_t* tokens;
  int64_t tokens_stride;
  int tokens_len;
  int32_t *accepted, *path, *next, *ctx_out;
  uint32_t* status;
};

__global__ void __launch_bounds__(kCommitThreads) tree_commit_kernel(const CommitArgs a) {
  pdl_trigger();
  __shared__ int s_draft[kMaxTree], s_target[kMaxTree], s_parent[kMaxTree], s_slot[kMaxTree];
  __shared__ uint16_t s_path[kMaxTree];
  __shared__ int s_len, s_ctx;
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int lo = min(max(a.indptr[b], 0), a.R), hi = min(max(a.indptr[b + 1], lo), a.R);
  const int n = min(hi - lo, kMaxTree);
  // read before the barriers: `ctx_out` may be `ctx`, and its store comes after them
  if (tid == 0) s_ctx = a.ctx[b];
  for (int i = tid; i < n; i += kCommitThreads) {
    s_draft[i] = a.drafts[lo + i];
    s_target[i] = a.targets[lo + i];
    s_parent[i] = a.parents ? a.parents[lo + i] : i - 1;
    s_slot[i] = a.slots[lo + i];
  }
  __syncthreads();
  if (warp == 0) {
    int len = 0, cur = n > 0 ? 0 : -1;
    while (cur >= 0) {
      if (lane == 0) s_path[len] = uint16_t(cur);
      ++len;
      const int want = s_target[cur];
      int child = -1;
      for (int base = (cur + 1) & ~31; base < n && child < 0; base += 32) {
        const int i = base + lane;
        const bool is = i > cur && i < n && s_parent[i] == cur && s_draft[i] == want;
        const unsigned hit = __ballot_sync(0xffffffffu, is);
        if (hit) child = base + __ffs(hit) - 1;
      }
      cur = child;  // indices only grow, so the walk ends
    }
    if (lane == 0) s_len = len;
  }
  __syncthreads();
  const int len = s_len;
  if (blockIdx.x == 0) {
    const int ctx = s_ctx;
    for (int k = tid; k < hi - lo; k += kCommitThreads) {
      a.path[lo + k] = k < len ? int(s_path[k]) : -1;
      if (k < len && a.tokens != nullptr) {
        const int64_t at = int64_t(ctx) + k;
        if (at >= 0 && at < a.tokens_len)
          a.tokens[b * a.tokens_stride + at] = s_draft[s_path[k]];
        else
          atomicCAS(a.status, 0u, uint32_t(kStatusBadSize));
      }
    }
    if (tid == 0) {
      a.accepted[b] = len;
      a.next[b] = len > 0 ? s_target[s_path[len - 1]] : -1;
      a.ctx_out[b] = ctx + len;
      if (hi - lo > kMaxTree) atomicCAS(a.status, 0u, uint32_t(kStatusBadSize));
    }
    if (b == 0)  // rows past the last request
      for (int r = min(max(a.indptr[gridDim.y], 0), a.R) + tid; r < a.R; r += kCommitThreads) a.path[r] = -1;
  }
  if (a.src == nullptr) return;
  // 16-byte words of all rows and planes, four in flight a thread
  const int first = blockIdx.x * a.planes_per_cta, count = min(a.planes_per_cta, a.planes - first);
  const int row = a.heads * a.words, total = count * len * row;
  for (int e0 = tid; e0 < total; e0 += 4 * kCommitThreads) {
    uint4 v[4];
    uint4* to[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int e = e0 + u * kCommitThreads;
      to[u] = nullptr;
      if (e < total) {
        const int x = e / row, c = e - x * row, plane = first + x / len, k = x % len, h = c / a.words, w = c - h * a.words;
        const int slot = s_slot[k];
        if (slot >= 0 && slot < a.num_slots) {
          v[u] = a.src[(plane >> 1) * a.src_l + (plane & 1) * a.src_p + (lo + s_path[k]) * a.src_r + h * a.src_h + w];
          to[u] = a.dst + (plane >> 1) * a.dst_l + (plane & 1) * a.dst_p + (slot / a.bs) * a.dst_b +
                  (slot % a.bs) * a.dst_t + h * a.dst_h + w;
        } else if (c == 0) {
          atomicCAS(a.status, 0u, uint32_t(kStatusBadSize));
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (to[u]) *to[u] = v[u];
  }
}

}  // namespace

std::vector<torch::Tensor> commit_tree(torch::Tensor draft_ids, torch::Tensor target_ids,
                                       c10::optional<torch::Tensor> parents, torch::Tensor indptr,
                                       torch::Tensor ctx_lens, torch::Tensor slot_mapping,
                                       c10::optional<torch::Tensor> tree_kv, c10::optional<torch::Tensor> kv_cache,
                                       c10::optional<torch::Tensor> tokens, std::vector<torch::Tensor> out,
                                       torch::Tensor status) {
  const int64_t R = draft_ids.numel(), B = ctx_lens.numel();
  KVS_CHECK_ARG(draft_ids.is_cuda() && draft_ids.scalar_type() == at::kInt, "commit_tree: int32 CUDA tensors");
  if (out.empty()) {
    // one piece of memory for all outputs
    const torch::Tensor all = torch::empty({3 * B + R}, draft_ids.options());
    out = {all.narrow(0, 0, B), all.narrow(0, B, R), all.narrow(0, B + R, B), all.narrow(0, 2 * B + R, B)};
  }
  KVS_CHECK_ARG(out.size() == 4, "commit_tree: four outputs");
  const torch::Tensor &accepted = out[0], &path = out[1], &next_ids = out[2], &ctx_out = out[3];
  auto vec = [&](const torch::Tensor& t, int64_t n, const char* msg) {
    KVS_CHECK_ARG(t.is_cuda() && t.dim() == 1 && t.is_contiguous() && t.scalar_type() == at::kInt &&
                      t.numel() == n && t.device() == draft_ids.device(),
                  msg);
  };
  const char* rows = "commit_tree: draft_ids, target_ids, parents, slot_mapping, path are int32 [R] on one CUDA device";
  const char* reqs = "commit_tree: ctx_lens, accepted, next_ids are int32 [B], indptr [B + 1]";
  vec(draft_ids, R, rows);
  vec(target_ids, R, rows);
  vec(slot_mapping, R, rows);
  vec(path, R, rows);
  if (parents.has_value()) vec(*parents, R, rows);
  vec(indptr, B + 1, reqs);
  vec(ctx_lens, B, reqs);
  vec(accepted, B, reqs);
  vec(next_ids, B, reqs);
  vec(ctx_out, B, reqs);
  KVS_CHECK_ARG(B >= 1 && B <= 65535, "commit_tree: 1 to 65535 requests");
  KVS_CHECK_ARG(R < (int64_t(1) << 30), "commit_tree: too many rows");
  KVS_CHECK_ARG(tree_kv.has_value() == kv_cache.has_value(), "commit_tree: tree_kv and kv_cache go together");
  CommitArgs a{};
  if (tokens.has_value()) {
    KVS_CHECK_ARG(tokens->is_cuda() && tokens->dim() == 2 && tokens->size(0) == B && tokens->stride(1) == 1 &&
                      tokens->scalar_type() == at::kInt && tokens->device() == draft_ids.device(),
                  "commit_tree: tokens [B, M] int32 with contiguous rows");
    a.tokens = tokens->data_ptr<int32_t>();
    a.tokens_stride = tokens->stride(0);
    a.tokens_len = int(std::min<int64_t>(tokens->size(1), INT32_MAX));
  }
  a.planes = a.planes_per_cta = 1;
  if (tree_kv.has_value() && R > 0) {
    const torch::Tensor &s = *tree_kv, &c = *kv_cache;
    KVS_CHECK_ARG(s.is_cuda() && c.is_cuda() && s.dim() == 5 && c.dim() == 6 && s.scalar_type() == c.scalar_type() &&
                      s.device() == draft_ids.device() && c.device() == draft_ids.device(),
                  "commit_tree: tree_kv [L, 2, R, Hkv, D] and kv_cache [L, 2, blocks, block_size, Hkv, D] of one type");
    KVS_CHECK_ARG(s.size(0) == c.size(0) && s.size(1) == 2 && c.size(1) == 2 && s.size(2) >= R &&
                      s.size(3) == c.size(4) && s.size(4) == c.size(5) && s.size(0) >= 1,
                  "commit_tree: tree_kv and kv_cache shapes differ");
    const int64_t item = s.element_size();
    bool wide = s.stride(4) == 1 && c.stride(5) == 1 && (s.size(4) * item) % 16 == 0 &&
                (reinterpret_cast<uintptr_t>(s.data_ptr()) & 15) == 0 &&
                (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15) == 0;
    for (int d = 0; d < 4; ++d) wide = wide && (s.stride(d) * item) % 16 == 0;
    for (int d = 0; d < 5; ++d) wide = wide && (c.stride(d) * item) % 16 == 0;
    KVS_CHECK_ARG(wide, "commit_tree: head rows must be contiguous multiples of 16 bytes at 16-byte boundaries");
    a.src = reinterpret_cast<const uint4*>(s.data_ptr());
    a.dst = reinterpret_cast<uint4*>(c.data_ptr());
    auto words = [&](int64_t stride) { return stride * item / 16; };
    a.src_l = words(s.stride(0));
    a.src_p = words(s.stride(1));
    a.src_r = words(s.stride(2));
    a.src_h = words(s.stride(3));
    a.dst_l = words(c.stride(0));
    a.dst_p = words(c.stride(1));
    a.dst_b = words(c.stride(2));
    a.dst_t = words(c.stride(3));
    a.dst_h = words(c.stride(4));
    a.heads = int(s.size(3));
    a.words = int(s.size(4) * item / 16);
    a.bs = int(c.size(3));
    a.num_slots = c.size(2) * c.size(3);
    KVS_CHECK_ARG(int64_t(a.heads) * a.words * kMaxTree * s.size(0) * 2 <= INT32_MAX,
                  "commit_tree: K/V rows too long");
    a.planes = int(s.size(0) * 2);
    a.planes_per_cta = int(std::max<int64_t>(1, std::min<int64_t>(a.planes, a.planes * B / kCommitCtas)));
  }
  const c10::cuda::CUDAGuard guard(draft_ids.device());
  a.drafts = draft_ids.data_ptr<int32_t>();
  a.targets = target_ids.data_ptr<int32_t>();
  a.parents = parents.has_value() ? parents->data_ptr<int32_t>() : nullptr;
  a.indptr = indptr.data_ptr<int32_t>();
  a.ctx = ctx_lens.data_ptr<int32_t>();
  a.slots = slot_mapping.data_ptr<int32_t>();
  a.R = int(R);
  a.accepted = accepted.data_ptr<int32_t>();
  a.path = path.data_ptr<int32_t>();
  a.next = next_ids.data_ptr<int32_t>();
  a.ctx_out = ctx_out.data_ptr<int32_t>();
  a.status = reinterpret_cast<uint32_t*>(status.data_ptr<int32_t>());
  const int groups = (a.planes + a.planes_per_cta - 1) / a.planes_per_cta;
  tree_commit_kernel<<<dim3(unsigned(groups), unsigned(B)), kCommitThreads, 0, at::cuda::getCurrentCUDAStream()>>>(a);
  KVS_CUDA_CHECK(cudaGetLastError());
  return out;
}

}  // namespace kvs
