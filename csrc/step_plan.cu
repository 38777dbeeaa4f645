// Plan of one multi-token step, from request lengths that live on the GPU.
//
// Request b holds ctx_b committed tokens in held_b blocks and adds n_b rows.
//   indptr    = exclusive sum of n                     (rows of b: indptr_b ..)
//   need_b    = max(0, ceil((ctx_b + n_b) / bs) - held_b), taken from the ring
//               of free blocks in request order (first in, first out)
//   slot(r)   = table[b, p / bs] * bs + p % bs with p = ctx_b + (r - indptr_b)
//   mask(r)   = mask(parent) | own bit, position(r) = ctx_b + depth(r)
// A request with n_b < 0 has ended: its blocks go back to the end of the ring.
//
// The work is a few words a row, so the call is bound by latency.  Every CTA
// repeats the (cheap) sums over the requests in its own shared memory, four
// requests a thread, and takes a share of the rows, so no sum crosses CTAs.
// The state may be updated in place, so its update comes after the last read
// of the old one: a step of up to 1024 rows and requests is one CTA and one
// launch, a larger one spreads its rows over the GPU and a second small kernel
// follows (2048 requests, 60000 rows: 10 us; 31 us as one cluster of 8 CTAs;
// 8 trees of 16: 7.6 us; in a CUDA graph).
// Whole numbers and fixed order: the result does not depend on timing.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"
#include "tree_ops.h"

namespace kvs {
namespace {

constexpr int kPlanThreads = 512;
constexpr int kMaxRequests = 16384;
constexpr int kItems = 4;         // requests a thread sums
constexpr int kOneCta = 1024;     // rows and requests of a step that one CTA plans

struct PlanArgs {
  const int32_t *ctx, *fresh, *held;
  int32_t* table;
  int64_t table_stride;
  int width;
  int32_t* queue;
  int cap;
  const int64_t* cursor;
  const int32_t* parents;
  int B, bs, R, words;
  int32_t *indptr, *request, *positions, *slots, *mask, *held_out;
  int64_t* cursor_out;
  int32_t* totals;  // blocks taken and returned, and whether the ring was too short (null: one CTA does all)
  uint32_t* status;
};

// Exclusive sum over the block of one 64-bit value a thread (two 32-bit sums
// packed); `total` is the block's sum.
__device__ __forceinline__ uint64_t block_exclusive(uint64_t v, uint64_t* warp_sum, uint64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint64_t y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) warp_sum[warp] = x;
  __syncthreads();
  uint64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    const uint64_t s = warp_sum[w];
    before += w < warp ? s : 0;
    all += s;
  }
  __syncthreads();
  total = all;
  return before + x - v;
}

// Largest b with sums[b] <= at (sums ascending, sums[0] = 0, at < sums[B]).
__device__ __forceinline__ int owner(const int* sums, int B, int at) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= at) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int64_t blocks_for(const PlanArgs& a, int ctx, int n) {
  return (int64_t(max(ctx, 0)) + n + a.bs - 1) / a.bs;
}

__device__ __forceinline__ int ring(int at, int cap) { return at >= cap ? at - cap : at; }

__global__ void __launch_bounds__(kPlanThreads) step_plan_kernel(PlanArgs a) {
  pdl_trigger();
  extern __shared__ int sm[];
  __shared__ uint64_t warp_sum[kPlanThreads / 32];
  __shared__ int s_bad;
  int* s_rows = sm;                    // [B + 1] indptr
  int* s_need = s_rows + a.B + 1;      // [B + 1] exclusive sum of taken blocks
  int* s_free = s_need + a.B + 1;      // [B + 1] exclusive sum of returned blocks
  const int rank = blockIdx.x;
  const int first = rank * kPlanThreads + threadIdx.x, step = gridDim.x * kPlanThreads;
  if (threadIdx.x == 0) s_bad = 0;
  const int64_t head = a.cursor[0], tail = a.cursor[1];
  const int h0 = int(uint64_t(head) % uint64_t(a.cap)), t0 = int(uint64_t(tail) % uint64_t(a.cap));
  const int rounds = (a.B + kItems * kPlanThreads - 1) / (kItems * kPlanThreads);

  uint64_t carry = 0, total = 0;
  for (int it = 0; it < rounds; ++it) {
    const int b0 = (it * kPlanThreads + threadIdx.x) * kItems;
    uint32_t n[kItems];
    uint64_t sum = 0;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      n[i] = b0 + i < a.B ? uint32_t(max(a.fresh[b0 + i], 0)) : 0u;
      sum += n[i];
    }
    uint64_t at = carry + block_exclusive(sum, warp_sum, total);
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (b0 + i < a.B) s_rows[b0 + i] = int(min(at, uint64_t(a.R)));  // rows past the last one that fits are dropped
      at += n[i];
    }
    carry += total;
  }
  if (threadIdx.x == 0) {
    s_rows[a.B] = int(min(carry, uint64_t(a.R)));
    if (carry > uint64_t(a.R)) s_bad = kStatusBadSize;
  }
  __syncthreads();
  carry = 0;
  for (int it = 0; it < rounds; ++it) {
    const int b0 = (it * kPlanThreads + threadIdx.x) * kItems;
    uint64_t v[kItems], sum = 0;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int b = b0 + i;
      v[i] = 0;
      if (b < a.B) {
        const int held = min(max(a.held[b], 0), a.width);
        if (a.fresh[b] < 0) {
          v[i] = uint64_t(held) << 32;
        } else {
          const int n = s_rows[b + 1] - s_rows[b];
          const int64_t blocks = blocks_for(a, a.ctx[b], n);
          if (blocks > a.width) s_bad = kStatusBadSize;
          v[i] = uint64_t(max(min(blocks, int64_t(a.width)) - held, int64_t(0)));
          if (a.parents != nullptr && n > 32 * a.words) s_bad = kStatusBadSize;
        }
      }
      sum += v[i];
    }
    uint64_t at = carry + block_exclusive(sum, warp_sum, total);
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (b0 + i < a.B) {
        s_need[b0 + i] = int(uint32_t(at));
        s_free[b0 + i] = int(at >> 32);
      }
      at += v[i];
    }
    carry += total;
  }
  if (threadIdx.x == 0) {
    s_need[a.B] = int(uint32_t(carry));
    s_free[a.B] = int(carry >> 32);
  }
  __syncthreads();
  const int rows = s_rows[a.B], freed = s_free[a.B];
  int need = s_need[a.B];
  const bool dry = int64_t(need) > tail - head;  // not enough free blocks: nobody gets one
  if (dry) need = 0;

  // new table entries and returned blocks
  for (int e = first; e < need; e += step) {
    const int b = owner(s_need, a.B, e);
    const int held = min(max(a.held[b], 0), a.width);
    a.table[b * a.table_stride + held + (e - s_need[b])] = a.queue[ring(h0 + e, a.cap)];
  }
  for (int e = first; e < freed; e += step) {
    const int b = owner(s_free, a.B, e);
    // at most `cap` blocks exist, so e < cap for any consistent state
    a.queue[(t0 + e) % a.cap] = a.table[b * a.table_stride + (e - s_free[b])];
  }
  // rows
  bool bad_parent = false;
  for (int r = first; r < a.R; r += step) {
    int b = -1, pos = 0, slot = -1;
    if (r < rows) {
      b = owner(s_rows, a.B, r);
      const int i = r - s_rows[b], c = max(a.ctx[b], 0), held = min(max(a.held[b], 0), a.width);
      const int64_t p = int64_t(c) + i;
      const int64_t blk = p / a.bs;
      if (blk < held) {
        slot = a.table[b * a.table_stride + blk] * a.bs + int(p % a.bs);
      } else if (!dry && blk < held + (s_need[b + 1] - s_need[b])) {
        slot = a.queue[ring(h0 + s_need[b] + int(blk - held), a.cap)] * a.bs + int(p % a.bs);
      }
      pos = int(p);
      if (a.parents != nullptr) {
        // Parents have lower indices, so the walk to the root meets the bits
        // of the mask in descending order: each word is written once.
        int32_t* out = a.mask + int64_t(r) * a.words;
        const int32_t* par = a.parents + s_rows[b];
        int w = a.words - 1, depth = 0, j = i;
        uint32_t bits = 0;
        while (true) {
          for (; w > (j >> 5); --w) {
            out[w] = int32_t(bits);
            bits = 0;
          }
          if (w == (j >> 5)) bits |= 1u << (j & 31);
          const int up = par[j];
          if (up < -1 || up >= j) bad_parent = true;
          if (up < 0 || up >= j) break;
          j = up;
          ++depth;
        }
        for (; w >= 0; --w) {
          out[w] = int32_t(bits);
          bits = 0;
        }
        pos = c + depth;
      }
    } else if (a.parents != nullptr) {
      for (int w = 0; w < a.words; ++w) a.mask[int64_t(r) * a.words + w] = 0;
    }
    a.request[r] = b;
    a.positions[r] = pos;
    a.slots[r] = slot;
  }
  for (int b = first; b <= a.B; b += step) a.indptr[b] = s_rows[b];
  if (bad_parent) s_bad = kStatusBadSymbol;
  __syncthreads();
  if (threadIdx.x == 0) {
    if (rank == 0 && dry) atomicCAS(a.status, 0u, uint32_t(kStatusNoBlocks));
    if (s_bad) atomicCAS(a.status, 0u, uint32_t(s_bad));
    if (rank == 0 && a.totals != nullptr) {
      a.totals[0] = need;
      a.totals[1] = freed;
      a.totals[2] = dry;
    }
  }
  if (a.totals == nullptr) {  // the only CTA: all of the old state has been read
    for (int b = threadIdx.x; b < a.B; b += kPlanThreads) {
      const int held = min(max(a.held[b], 0), a.width);
      a.held_out[b] = a.fresh[b] < 0 ? 0 : held + (dry ? 0 : s_need[b + 1] - s_need[b]);
    }
    if (threadIdx.x == 0) {
      a.cursor_out[0] = head + need;
      a.cursor_out[1] = tail + freed;
    }
  }
}

// The new state of a step that several CTAs planned.
__global__ void __launch_bounds__(256) step_state_kernel(PlanArgs a) {
  pdl_wait();
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b < a.B) {
    const int held = min(max(a.held[b], 0), a.width);
    const int64_t blocks = min(blocks_for(a, a.ctx[b], a.indptr[b + 1] - a.indptr[b]), int64_t(a.width));
    a.held_out[b] = a.fresh[b] < 0 ? 0 : a.totals[2] ? held : max(held, int(blocks));
  }
  if (b == 0) {
    a.cursor_out[0] = a.cursor[0] + a.totals[0];
    a.cursor_out[1] = a.cursor[1] + a.totals[1];
  }
}

const int32_t* ints(const torch::Tensor& t) { return t.data_ptr<int32_t>(); }

}  // namespace

std::vector<torch::Tensor> plan_step(torch::Tensor ctx_lens, torch::Tensor new_lens, torch::Tensor block_tables,
                                     torch::Tensor held, torch::Tensor free_queue, torch::Tensor cursor,
                                     int64_t block_size, int64_t num_rows, c10::optional<torch::Tensor> parents,
                                     int64_t max_tree, std::vector<torch::Tensor> out, torch::Tensor status) {
  const int64_t B = ctx_lens.numel(), R = num_rows;
  KVS_CHECK_ARG(ctx_lens.is_cuda() && ctx_lens.scalar_type() == at::kInt, "plan_step: ctx_lens int32 on a CUDA device");
  KVS_CHECK_ARG(R >= 0 && R < (int64_t(1) << 30), "plan_step: too many rows");
  KVS_CHECK_ARG(max_tree >= 1 && max_tree <= 32768, "plan_step: max_tree must be 1 to 32768");
  const int64_t words = parents.has_value() ? (max_tree + 31) / 32 : 0;
  if (out.empty()) {
    // one piece of memory for all outputs
    const torch::Tensor all = torch::empty({2 * B + 1 + R * (3 + words)}, ctx_lens.options());
    int64_t at = 0;
    auto take = [&](int64_t n) {
      at += n;
      return all.narrow(0, at - n, n);
    };
    out = {take(B + 1), take(R), take(R), take(R)};
    if (words) out.push_back(take(R * words).view({R, words}));
    out.push_back(take(B));
    out.push_back(torch::empty({2}, cursor.options()));
  }
  KVS_CHECK_ARG(out.size() == (words ? 7u : 6u), "plan_step: out was made for a step with other parents");
  const torch::Tensor &indptr = out[0], &row_request = out[1], &positions = out[2], &slot_mapping = out[3],
                      &held_out = out[out.size() - 2], &cursor_out = out[out.size() - 1];
  c10::optional<torch::Tensor> tree_mask;
  if (words) tree_mask = out[4];
  KVS_CHECK_ARG(row_request.numel() == R, "plan_step: out was made for another number of rows");
  for (const torch::Tensor* t : std::initializer_list<const torch::Tensor*>{
           &ctx_lens, &new_lens, &held, &free_queue, &indptr, &row_request, &positions, &slot_mapping, &held_out})
    KVS_CHECK_ARG(t->is_cuda() && t->dim() == 1 && t->is_contiguous() && t->scalar_type() == at::kInt &&
                      t->device() == ctx_lens.device(),
                  "plan_step: lengths, queue and row tensors are contiguous int32 vectors on one CUDA device");
  for (const torch::Tensor* t : std::initializer_list<const torch::Tensor*>{&cursor, &cursor_out})
    KVS_CHECK_ARG(t->is_cuda() && t->is_contiguous() && t->scalar_type() == at::kLong && t->numel() == 2 &&
                      t->device() == ctx_lens.device(),
                  "plan_step: cursor is int64 [2] on the same device");
  KVS_CHECK_ARG(new_lens.numel() == B && held.numel() == B && held_out.numel() == B && indptr.numel() == B + 1,
                "plan_step: ctx_lens, new_lens, held [B], indptr [B + 1]");
  KVS_CHECK_ARG(B >= 1 && B <= kMaxRequests, "plan_step: 1 to 16384 requests");
  KVS_CHECK_ARG(block_tables.is_cuda() && block_tables.dim() == 2 && block_tables.size(0) == B &&
                    block_tables.scalar_type() == at::kInt && block_tables.stride(1) == 1 &&
                    block_tables.size(1) >= 1 && block_tables.device() == ctx_lens.device(),
                "plan_step: block_tables [B, W] int32 with contiguous rows");
  KVS_CHECK_ARG(block_tables.size(1) <= INT32_MAX / B, "plan_step: block_tables has too many entries");
  KVS_CHECK_ARG(positions.numel() == R && slot_mapping.numel() == R, "plan_step: row tensors have one length");
  KVS_CHECK_ARG(free_queue.numel() >= 1 && free_queue.numel() < (int64_t(1) << 30), "plan_step: free_queue size");
  KVS_CHECK_ARG(block_size >= 1 && block_size * free_queue.numel() <= INT32_MAX,
                "plan_step: slots (blocks x block_size) must fit in 32 bits");
  PlanArgs a{};
  if (parents.has_value()) {
    KVS_CHECK_ARG(parents->is_cuda() && parents->scalar_type() == at::kInt && parents->dim() == 1 &&
                      parents->is_contiguous() && parents->numel() == R && parents->device() == ctx_lens.device(),
                  "plan_step: parents is an int32 vector with one entry a row");
    KVS_CHECK_ARG(tree_mask->is_cuda() && tree_mask->scalar_type() == at::kInt && tree_mask->dim() == 2 &&
                      tree_mask->is_contiguous() && tree_mask->size(0) == R && tree_mask->size(1) >= 1,
                  "plan_step: tree_mask [R, W] int32");
    a.parents = ints(*parents);
    a.mask = tree_mask->data_ptr<int32_t>();
    a.words = int(tree_mask->size(1));
  }
  const c10::cuda::CUDAGuard guard(ctx_lens.device());
  a.ctx = ints(ctx_lens);
  a.fresh = ints(new_lens);
  a.held = ints(held);
  a.table = block_tables.data_ptr<int32_t>();
  a.table_stride = block_tables.stride(0);
  a.width = int(block_tables.size(1));
  a.queue = free_queue.data_ptr<int32_t>();
  a.cap = int(free_queue.numel());
  a.cursor = cursor.data_ptr<int64_t>();
  a.B = int(B);
  a.bs = int(block_size);
  a.R = int(R);
  a.indptr = indptr.data_ptr<int32_t>();
  a.request = row_request.data_ptr<int32_t>();
  a.positions = positions.data_ptr<int32_t>();
  a.slots = slot_mapping.data_ptr<int32_t>();
  a.held_out = held_out.data_ptr<int32_t>();
  a.cursor_out = cursor_out.data_ptr<int64_t>();
  a.status = reinterpret_cast<uint32_t*>(status.data_ptr<int32_t>());
  const int64_t work = std::max(R, B);
  const int ctas = work <= kOneCta ? 1 : int(std::min<int64_t>(kNumSMs, (work + kPlanThreads - 1) / kPlanThreads));
  torch::Tensor totals;
  if (ctas > 1) {
    totals = torch::empty({4}, ctx_lens.options());
    a.totals = totals.data_ptr<int32_t>();
  }
  const size_t smem = size_t(3) * (B + 1) * sizeof(int);
  if (smem > 40 * 1024)
    KVS_CUDA_CHECK(cudaFuncSetAttribute(step_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  step_plan_kernel<<<ctas, kPlanThreads, smem, st>>>(a);
  KVS_CUDA_CHECK(cudaGetLastError());
  if (ctas > 1) launch_pdl(step_state_kernel, dim3(unsigned((B + 255) / 256)), dim3(256), 0, st, a);
  return out;
}

}  // namespace kvs
