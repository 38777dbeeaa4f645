// Attention of drafted trees over the paged KV cache.
//
// Row r of request b (node i of its tree) attends to the request's ctx_b
// committed tokens in the cache and to the tree rows j of the step with bit j
// of mask(r) set (without a mask: j <= i):
//   o = sum_t p_t v_t,  p = softmax_t(scale q . k_t);  nothing visible: o = 0.
//
// All n_b * G query rows of a KV head (G = Hq / Hkv) share its K and V, so
// they are packed into 128-row tiles for tcgen05: S = Q K^T and O += P V, both
// accumulated in TMEM.  A K/V byte serves n_b * G rows: up to about 256 rows
// the kernel is bound by HBM, above by the tensor pipe and the exponentials.
//
// Work is cut by K/V tiles of 64 tokens, not by requests: the tiles of all
// (request, KV head, row tile) items form one sequence and every CTA takes an
// equal, contiguous share of it, whatever the lengths are.  They live on the
// GPU only, so each CTA sums them itself.  A CTA that gets only a part of an
// item leaves an fp32 record (row maximum, row sum, O) that a second small
// kernel joins in a fixed order.
//
// Measured (B200, device time in a CUDA graph; called one after another in
// brackets; 128-wide heads): 64 requests of 16 nodes over up to 2900 tokens,
// 32/8 heads, 131 to 134 us = 4.2 to 4.3 TB/s (142; HBM floor 87); 128 single
// tokens over 2047, 28/4 heads, fp16, 87 us = 4.4 TB/s (90; floor 59); one
// tree of 64 over 131000 tokens, 64/8 heads, 324 us = 848 TFLOP/s (331; tensor
// floor 163); one tree of 8 over 700 tokens 16.2 us (18.2), all latency.  The
// 64 requests with 64-wide heads 113 us (floor 44), with blocks of 8 tokens,
// whose TMA boxes are half as large, 156 us.  Blocks that are no multiple of 8
// tokens go through one copying warp each for K and V: 2404 us.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <type_traits>

#include "common.cuh"
#include "sm100.cuh"
#include "tree_ops.h"

namespace kvs {
namespace {

constexpr int BM = 128;      // query rows of a tile (the MMA's M)
constexpr int BN = 64;       // tokens of a K/V tile
constexpr int kThreads = 448;  // warps 0..3 and 4..7 softmax of the two streams, 8 and 9 loaders, 10..13 MMA issuers
constexpr float kRescaleThreshold = 8.0f;  // log2: P stays below 2^8 between rescalings
// log2 of a factor on P, its row sums and O that cancels in the end.  fp16 has
// normal numbers down to 2^-14 only: with 2^7, probabilities keep all their
// bits down to 2^-21 of the largest one and end at 2^-32 (without it 2^-14 and
// 2^-25: many tokens under one of large weight lost their share); 2^(8 + 7) is
// below fp16's largest number.  bf16 has the exponents of fp32.
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 7.0f : 0.0f;

struct TreeArgs {
  const void *q, *kt, *vt, *kc, *vc;
  void* out;
  int64_t q_r, q_h, kt_r, kt_h, vt_r, vt_h, out_r, out_h;
  int64_t kc_b, kc_t, kc_h, vc_b, vc_t, vc_h;
  const int32_t *tables, *ctx, *indptr, *mask;
  int64_t table_stride, num_blocks;
  int width, words, R, B, hkv, group, bs;
  int box;         // tokens of one TMA box of the cache (0: rows are copied by the loader warp)
  bool tree_tma;   // tree rows by TMA
  bool q_tma;      // query rows by TMA
  int q_box;       // tree nodes of one TMA box of q
  int nodes;       // tree nodes of a row tile (nodes * group <= BM)
  bool k_head_first, v_head_first, kt_head_first, vt_head_first;  // order of the middle tensor-map dimensions
  int ctas;
  int part_rows;   // rows kept per partial record
  float scale_log2;
  float4* part_o;   // [4 * CTAs, D / 4, part_rows]: neighbouring lanes write neighbouring rows
  float2* part_ml;  // [4 * CTAs, part_rows]
  int4* meta;       // [CTAs] request of the CTA's first tile, that request's first tile, share, total
  uint32_t* err;
};

// ------------------------------------------------------------------ schedule
struct Shape {  // of one request
  int lo, n, ctx, nt_ctx, nt, mt, pairs;
};
__device__ __forceinline__ Shape request_shape(const TreeArgs& a, int b) {
  Shape s;
  s.lo = min(max(a.indptr[b], 0), a.R);
  s.n = max(min(a.indptr[b + 1], a.R) - s.lo, 0);
  s.ctx = int(max(min(int64_t(a.ctx[b]), int64_t(a.width) * a.bs), int64_t(0)));
  s.nt_ctx = (s.ctx + BN - 1) / BN;
  s.mt = (s.n + a.nodes - 1) / a.nodes;
  s.pairs = (s.mt + 1) / 2;
  s.nt = s.n > 0 ? s.nt_ctx + (s.n + BN - 1) / BN : 0;
  return s;
}
__device__ __forceinline__ int64_t tile_count(const TreeArgs& a, const Shape& s) {
  return int64_t(a.hkv) * s.pairs * s.nt;
}
// The pairs of row tiles of one KV head read the same K/V.  Items with
// several pairs are cut into segments of at least one CTA share and ordered
// (segment, pair), so the CTAs that read one segment run side by side and all
// but the first find it in L2.
struct Segments {
  int count, len, longer;  // `longer` segments of len + 1 tiles, then segments of len
  __device__ __forceinline__ Segments(const Shape& s, int share) {
    count = 1;
    len = s.nt;
    longer = 0;
    if (s.pairs > 1 && s.nt > share) {
      count = s.nt / share;
      len = s.nt / count;
      longer = s.nt - len * count;
    }
  }
  __device__ __forceinline__ int length(int i) const { return len + (i < longer ? 1 : 0); }
  __device__ __forceinline__ int start(int i) const { return i * len + min(i, longer); }
};

struct Piece {  // consecutive tiles of one item (request, KV head, pair of row tiles)
  Shape s;
  int b, h, pair;
  int segment, offset;  // of its first tile
  int t0, t1;           // tiles [t0, t1) of the item
  __device__ __forceinline__ bool starts() const { return offset == 0; }  // begins its segment
  __device__ __forceinline__ bool whole() const { return t1 - t0 == s.nt; }
  // the pair has two row tiles: each stream takes one; else the streams take turns in tiles
  __device__ __forceinline__ bool two() const { return 2 * pair + 1 < s.mt; }
  __device__ __forceinline__ int rows(const TreeArgs& a, int k) const {
    return min(s.n - (2 * pair + k) * a.nodes, a.nodes) * a.group;
  }
};

// The item, segment and tile that the tile with number x of a request is.
__device__ __forceinline__ void locate(const Shape& s, const Segments& seg, int x, Piece& p) {
  const int per_head = s.pairs * s.nt;
  p.h = x / per_head;
  int y = x - p.h * per_head;
  p.segment = p.pair = 0;
  if (s.pairs > 1) {
    const int big = (seg.len + 1) * s.pairs;
    if (y < big * seg.longer) {
      p.segment = y / big;
    } else if (seg.count > 1) {
      p.segment = seg.longer + (y - big * seg.longer) / (seg.len * s.pairs);
    }
    y -= seg.start(p.segment) * s.pairs;
    p.pair = y / seg.length(p.segment);
    y -= p.pair * seg.length(p.segment);
  }
  p.offset = y;
  p.t0 = seg.start(p.segment) + y;
}

struct Walker {  // the pieces of one CTA's share, in order
  int at, end, base, share, b;
  Shape s;
  __device__ __forceinline__ bool next(const TreeArgs& a, Piece& p) {
    if (at >= end) return false;
    while (at >= base + int(tile_count(a, s))) {
      base += int(tile_count(a, s));
      s = request_shape(a, ++b);
    }
    const Segments seg(s, share);
    p.s = s;
    p.b = b;
    locate(s, seg, at - base, p);
    const int take = min(seg.length(p.segment) - p.offset, end - at);
    p.t1 = p.t0 + take;
    at += take;
    return true;
  }
};

// ------------------------------------------------------------- small helpers
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<bf16>(float a, float b) {
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ float as_float(T v);
template <>
__device__ __forceinline__ float as_float<bf16>(bf16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float as_float<__half>(__half v) { return __half2float(v); }
// any of the two 16-bit floats of a word infinite or NaN (all exponent bits set)
template <typename T>
__device__ __forceinline__ bool odd2(uint32_t w) {
  constexpr uint32_t e = std::is_same<T, bf16>::value ? 0x7f80u : 0x7c00u;
  return (w & e) == e || (w >> 16 & e) == e;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float m;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}
__device__ __forceinline__ void fma2s(float& d0, float& d1, float a0, float a1, float b, float c) {
  asm("{.reg .b64 ra, rb, rc, rd;\n"
      "mov.b64 ra, {%2,%3};\n"
      "mov.b64 rb, {%4,%4};\n"
      "mov.b64 rc, {%5,%5};\n"
      "fma.rn.f32x2 rd, ra, rb, rc;\n"
      "mov.b64 {%0,%1}, rd;}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b), "f"(c));
}
__device__ __forceinline__ void add2(float& s0, float& s1, float a0, float a1) {
  asm("{.reg .b64 ra, rb, rd;\n"
      "mov.b64 ra, {%0,%1};\n"
      "mov.b64 rb, {%2,%3};\n"
      "add.rn.f32x2 rd, ra, rb;\n"
      "mov.b64 {%0,%1}, rd;}"
      : "+f"(s0), "+f"(s1)
      : "f"(a0), "f"(a1));
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{.reg .pred q;\n.reg .b32 r;\nelect.sync r|q, 0xffffffff;\nselp.u32 %0, 1, 0, q;}" : "=r"(p));
  return p != 0;
}
// Named barriers: 1 and 2 the warpgroup of stream 0 and 1 (128 threads), 3
// both on a shared V tile, 4 both at the end of a piece (256).
__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

__device__ __forceinline__ void tma_load_3d(void* dst, const void* map, int c0, int c1, int c2, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          sm100::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(sm100::smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* dst, const void* map, int c0, int c1, int c2, int c3, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(sm100::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(sm100::smem_u32(bar))
      : "memory");
}

// Byte offset of 16-byte chunk c of row r in a tile of `rows` rows: panels of
// 64 elements, 128-byte swizzle (chunk index xor row mod 8), the layout that
// both TMA and the MMA descriptors use.
__device__ __forceinline__ uint32_t tile_offset(int rows, int r, int c) {
  return uint32_t(c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

struct Shared {
  float2 ml[2][BM];       // row maximum and sum of the two streams
  int64_t sum[kThreads / 32];
  int base, b;
  uint32_t tmem;
  uint32_t odd[4];        // 1 + the last unit whose tree V held values that are not finite
  uint32_t piece_odd[2];  // ... in the streams' tiles of the piece
};

template <int D>
struct Layout {
  static constexpr int STAGES = D == 128 ? 5 : 10;
  static constexpr int PANELS = D / 64;
  static constexpr int Q_BYTES = BM * D * 2;
  static constexpr int TILE = BN * D * 2;
  static constexpr int OFF_K = 2 * Q_BYTES, OFF_V = OFF_K + STAGES * TILE, OFF_BAR = OFF_V + STAGES * TILE;
  // barriers: k_full, k_empty, v_full, v_empty [STAGES] each, s_full[4],
  // p_full[4], pv_done[4], q_full[2], q_empty[2], o_full, o_empty, drain[4]
  static constexpr int NUM_BARS = 4 * STAGES + 22;
  static constexpr int OFF_SHARED = OFF_BAR + NUM_BARS * 8;
  static constexpr int SMEM = OFF_SHARED + int(sizeof(Shared)) + (D == 128 ? 0 : 1024);
  static constexpr uint32_t TMEM_COLS = 512;  // S/P of 4 units (64 each), O of 2 streams (128 each)
};
static_assert(Layout<128>::SMEM <= 232448 && Layout<64>::SMEM <= 232448, "shared memory of one SM");

// Copies the rows of one K or V tile with plain loads (one warp): caches
// whose blocks TMA boxes do not tile (64 requests over 2900 tokens 2404 us
// instead of 134).  Rows at or past `valid` become zero.
template <int D>
__device__ __forceinline__ void copy_tile(uint8_t* dst, const uint16_t* src, int64_t row_stride, int valid, int lane) {
  constexpr int C = D / 8;
  for (int e = lane; e < BN * C; e += 32) {
    const int r = e / C, c = e % C;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < valid) v = *reinterpret_cast<const uint4*>(src + r * row_stride + c * 8);
    *reinterpret_cast<uint4*>(dst + tile_offset(BN, r, c)) = v;
  }
}
template <int D>
__device__ __forceinline__ void copy_paged_tile(uint8_t* dst, const uint16_t* cache, int64_t s_b, int64_t s_t,
                                                int64_t head_off, const int32_t* table, const TreeArgs& a, int t0,
                                                int valid, int lane) {
  constexpr int C = D / 8;
  for (int e = lane; e < BN * C; e += 32) {
    const int r = e / C, c = e % C;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < valid) {
      const int t = t0 + r, blk = table[t / a.bs];
      if (blk >= 0 && blk < a.num_blocks)
        v = *reinterpret_cast<const uint4*>(cache + blk * s_b + (t % a.bs) * s_t + head_off + c * 8);
    }
    *reinterpret_cast<uint4*>(dst + tile_offset(BN, r, c)) = v;
  }
}

// One CTA per SM.  A unit is one row tile against one K/V tile:
//   S(u) = Q K^T -> softmax -> P(u) over S(u) in TMEM -> O += P(u) V.
// Units alternate between two streams (u mod 2), each with its own softmax
// warpgroup and O accumulator, so one stream's softmax runs under the other's
// products; S has four buffers, so a stream's softmax does not wait for its
// own products either.  An item with two row
// tiles gives each stream one of them (a K/V tile feeds both); with one row
// tile the streams take turns in its K/V tiles and are joined at the end.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    tree_attention_kernel(const __grid_constant__ CUtensorMap m_kc, const __grid_constant__ CUtensorMap m_vc,
                          const __grid_constant__ CUtensorMap m_kt, const __grid_constant__ CUtensorMap m_vt,
                          const __grid_constant__ CUtensorMap m_q, const TreeArgs a) {
  using Lay = Layout<D>;
  using namespace sm100;
  constexpr int ST = Lay::STAGES;
  // the tiles fill the SM, so the 1024-byte alignment that their swizzle needs
  // is asked for instead of padded for, and checked
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023) {
    if (threadIdx.x == 0) {
      a.meta[blockIdx.x] = make_int4(0, 0, 1, 0);  // no tiles: the joining kernel reads it all the same
      atomicCAS(a.err, 0u, uint32_t(kStatusBadSize));
    }
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Lay::OFF_BAR);
  uint64_t *k_full = bars, *k_empty = bars + ST, *v_full = bars + 2 * ST, *v_empty = bars + 3 * ST;
  uint64_t *s_full = bars + 4 * ST, *p_full = s_full + 4, *pv_done = s_full + 8, *q_full = s_full + 12,
           *q_empty = s_full + 14, *o_full = s_full + 16, *o_empty = s_full + 17,
           *drain = s_full + 18;
  Shared& sh = *reinterpret_cast<Shared*>(smem + Lay::OFF_SHARED);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_trigger();

  if (threadIdx.x < Lay::NUM_BARS) {
    const int i = threadIdx.x, sb = i - 4 * ST;  // position after the ring's barriers
    uint32_t arrivals = 1;
    if ((i >= ST && i < 2 * ST) || (i >= 3 * ST && i < 4 * ST)) arrivals = 2;  // k_empty, v_empty: both streams
    if (sb >= 4 && sb < 8) arrivals = 4;       // p_full: the warps of a stream
    if (sb >= 14 && sb < 17) arrivals = 2;     // q_empty, o_full: both streams
    if (sb == 17) arrivals = 8;                // o_empty: all softmax warps
    mbar_init(&bars[i], arrivals);
    fence_barrier_init();
  } else if (threadIdx.x < 64 + 5) {
    if (threadIdx.x >= 64) {
      const int i = threadIdx.x - 64;
      tma_prefetch_desc(i == 0 ? &m_kc : i == 1 ? &m_vc : i == 2 ? &m_kt : i == 3 ? &m_vt : &m_q);
    }
  } else if (threadIdx.x >= 96 && threadIdx.x < 100) {
    sh.odd[threadIdx.x - 96] = 0;
  }
  if (warp == 9) tmem_alloc<Lay::TMEM_COLS>(&sh.tmem);

  // Sum the tiles of all requests for the total (and with it the share), and
  // find the request that this CTA's share begins in; a second pass is needed
  // only where the requests outnumber the threads.
  Walker walk;
  walk.share = 1;
  walk.at = walk.end = 0;
  for (int pass = 0; pass < 2; ++pass) {
    int64_t carry = 0;
    int from = 0, mine = 0;
    auto settle = [&](int b) {
      if (b < a.B && walk.at >= from && walk.at - from < mine) {
        sh.b = b;
        sh.base = from;
      }
    };
    for (int b0 = 0; b0 < a.B; b0 += kThreads) {
      const int b = b0 + threadIdx.x;
      const int64_t count = b < a.B ? tile_count(a, request_shape(a, b)) : 0;
      int64_t x = count;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
      }
      __syncthreads();
      if (lane == 31) sh.sum[warp] = x;
      __syncthreads();
      int64_t before = carry + x - count;
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) {
        before += w < warp ? sh.sum[w] : 0;
        carry += sh.sum[w];
      }
      from = int(before);
      mine = int(count);
      if (pass == 1) settle(b);
    }
    if (pass == 0) {
      if (carry > INT32_MAX - 4096) {  // numbers of tiles are 32 bits; nothing is computed
        if (threadIdx.x == 0) atomicCAS(a.err, 0u, uint32_t(kStatusBadSize));
        carry = 0;
        mine = 0;
      }
      const int total = int(carry);
      walk.share = max((total + int(gridDim.x) - 1) / int(gridDim.x), 1);
      walk.at = int(min(int64_t(blockIdx.x) * walk.share, int64_t(total)));
      walk.end = min(walk.at + walk.share, total);
      if (a.B <= kThreads) {
        settle(threadIdx.x);
        break;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  const uint32_t tO = tmem + 4 * BN;  // O of stream s at tO + s * 128
  const bool busy = walk.at < walk.end;
  if (busy) {
    walk.b = sh.b;
    walk.base = sh.base;
    walk.s = request_shape(a, walk.b);
  }
  if (threadIdx.x == 0)
    a.meta[blockIdx.x] = busy ? make_int4(walk.b, walk.base, walk.share, 1) : make_int4(0, 0, 1, 0);
  Piece p;

  if (busy && (warp == 8 || warp == 9)) {
    // ------------------------------------------------------------ loaders
    // Warp 8 loads Q and K, warp 9 loads V: one warp for both could not issue
    // the 2 KB boxes of 16-token blocks as fast as HBM delivers them.
    const bool is_v = warp == 9;
    uint64_t *full = is_v ? v_full : k_full, *empty = is_v ? v_empty : k_empty;
    uint8_t* ring = smem + (is_v ? Lay::OFF_V : Lay::OFF_K);
    const CUtensorMap *m_c = is_v ? &m_vc : &m_kc, *m_t = is_v ? &m_vt : &m_kt;
    const bool c_head_first = is_v ? a.v_head_first : a.k_head_first;
    const bool t_head_first = is_v ? a.vt_head_first : a.kt_head_first;
    bool ok = true;
    int g = 0, qc = 0;  // K/V tiles and Q tiles so far
    // waits of the whole warp
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      ok = ok && mbar_wait(bar, parity, a.err);
      ok = __all_sync(0xffffffffu, ok);
      return ok;
    };
    auto publish = [&](uint64_t* bar) {  // after plain stores of the warp
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    const int lane_box = lane / Lay::PANELS, lane_c = lane % Lay::PANELS;  // lane = (box, panel of 64 columns)
    while (ok && walk.next(a, p)) {
      const int32_t* table = a.tables + p.b * a.table_stride;
      // block and offset of this lane's box in tile j
      auto block_of = [&](int j, int& blk, int& off) {
        const int t = j * BN + lane_box * a.box;
        if (j < p.s.nt_ctx && j < p.t1 && lane_box * a.box < BN && t < p.s.ctx) {
          blk = table[t / a.bs];
          off = t % a.bs;
        }
      };
      int next_blk = 0, next_off = 0;
      if (a.box > 0) block_of(p.t0, next_blk, next_off);
      for (int k = 0; !is_v && k <= int(p.two()); ++k, ++qc) {
        const int node0 = (2 * p.pair + k) * a.nodes, nodes = min(p.s.n - node0, a.nodes);
        uint8_t* dq = smem + (qc & 1) * Lay::Q_BYTES;
        if (!wait(&q_empty[qc & 1], ((qc >> 1) & 1) ^ 1)) break;
        if (a.q_tma) {
          const int boxes = (nodes + a.q_box - 1) / a.q_box, box_rows = a.q_box * a.group;
          if (lane == 0) mbar_arrive_expect_tx(&q_full[qc & 1], uint32_t(boxes) * box_rows * D * 2);
          __syncwarp();
          if (lane < boxes)
            for (int c = 0; c < Lay::PANELS; ++c)
              tma_load_3d(dq + c * BM * 128 + lane * box_rows * 128, &m_q, c * 64, p.h * a.group,
                          p.s.lo + node0 + lane * a.q_box, &q_full[qc & 1]);
        } else {
          const uint16_t* q = reinterpret_cast<const uint16_t*>(a.q);
          constexpr int C = D / 8;
          for (int e = lane; e < nodes * a.group * C; e += 32) {
            const int r = e / C, c = e % C, node = node0 + r / a.group, hg = r % a.group;
            *reinterpret_cast<uint4*>(dq + tile_offset(BM, r, c)) = *reinterpret_cast<const uint4*>(
                q + int64_t(p.s.lo + node) * a.q_r + int64_t(p.h * a.group + hg) * a.q_h + c * 8);
          }
          publish(&q_full[qc & 1]);
        }
      }
      for (int j = p.t0; j < p.t1 && ok; ++j) {
        const int st = g % ST;
        uint8_t* dst = ring + st * Lay::TILE;
        const int blk = next_blk, off = next_off;
        if (a.box > 0) block_of(j + 1, next_blk, next_off);
        if (!wait(&empty[st], ((g / ST) & 1) ^ 1)) break;
        if (j < p.s.nt_ctx) {
          const int t0 = j * BN, valid = min(BN, p.s.ctx - t0);
          if (a.box > 0) {
            const int boxes = (valid + a.box - 1) / a.box;
            if (lane == 0) mbar_arrive_expect_tx(&full[st], uint32_t(boxes) * a.box * D * 2);
            __syncwarp();
            if (lane_box < boxes)
              tma_load_4d(dst + lane_c * BN * 128 + lane_box * a.box * 128, m_c, lane_c * 64,
                          c_head_first ? p.h : off, c_head_first ? off : p.h, blk, &full[st]);
          } else {
            copy_paged_tile<D>(dst, reinterpret_cast<const uint16_t*>(is_v ? a.vc : a.kc), is_v ? a.vc_b : a.kc_b,
                               is_v ? a.vc_t : a.kc_t, p.h * (is_v ? a.vc_h : a.kc_h), table, a, t0, valid, lane);
            publish(&full[st]);
          }
        } else {
          const int r0 = (j - p.s.nt_ctx) * BN, row = p.s.lo + r0;
          if (a.tree_tma) {
            if (lane == 0) mbar_arrive_expect_tx(&full[st], Lay::TILE);
            __syncwarp();
            if (lane < Lay::PANELS)
              tma_load_3d(dst + lane * BN * 128, m_t, lane * 64, t_head_first ? p.h : row, t_head_first ? row : p.h,
                          &full[st]);
          } else {
            const int64_t s_r = is_v ? a.vt_r : a.kt_r;
            copy_tile<D>(dst, reinterpret_cast<const uint16_t*>(is_v ? a.vt : a.kt) + row * s_r +
                                  p.h * (is_v ? a.vt_h : a.kt_h),
                         s_r, min(BN, p.s.n - r0), lane);
            publish(&full[st]);
          }
        }
        ++g;
      }
    }
    // every issued copy lands before the CTA may exit
    for (int i = max(0, g - ST); i < g; ++i) mbar_wait(&full[i % ST], (i / ST) & 1, nullptr);
    for (int i = max(0, qc - 2); i < qc; ++i) mbar_wait(&q_full[i & 1], (i >> 1) & 1, nullptr);
  } else if (busy && warp >= 10) {
    // -------------------------------------------------------- MMA issuers
    // Warps 10 and 11 issue S = Q K^T of streams 0 and 1, warps 12 and 13
    // issue O += P V.  Issue is the narrow place: the products of a unit take
    // 640 cycles, but a wait that need not wait costs 100 and a commit 50 to
    // 100; one warp for all needed 1430 cycles a unit, two needed 1100.
    // The warps run their loops whole, on values that the compiler can see to
    // be uniform (counts broadcast by shuffles, no early exits), so that the
    // descriptors live in uniform registers: 29 cycles to issue an MMA; from a
    // lane-0 branch it took 95 to 115.  After a wait that ran out, later
    // waits are skipped and the loop ends.
    constexpr uint32_t fmt = std::is_same<T, bf16>::value ? ~0u : ~((1u << 7) | (1u << 10));  // f16: type 0
    constexpr uint32_t idesc_qk = idesc_bf16(BM, BN, false) & fmt;
    constexpr uint32_t idesc_pv = idesc_bf16(BM, D, true) & fmt;
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const int role = __shfl_sync(0xffffffffu, warp, 0) - 10;
    const int stream = role & 1;
    bool alive = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (alive) alive = mbar_wait(bar, parity, a.err);
      __syncwarp();
    };
    // A parity wait is right only for the phase after the last one that is
    // known to be complete, and loads may complete out of order.  So both
    // streams' issuers wait for every phase of every full barrier in order,
    // also of tiles that only the other stream uses, and both arrive on the
    // empty barriers (two arrivals): by commit after their products, plainly
    // where they have none.
    int g0 = 0, u0 = 0, qc = 0, item = 0;  // tiles, units, Q tiles, pieces before this one
    const uint64_t dq0 = smem_desc_sw128(smem_u32(smem), 16, 1024);
    const uint64_t dk0 = smem_desc_sw128(smem_u32(smem + Lay::OFF_K), 16, 1024);
    const uint64_t dv0 = smem_desc_sw128(smem_u32(smem + Lay::OFF_V), BN * 128, 1024);
    while (__shfl_sync(0xffffffffu, int(walk.next(a, p)), 0)) {
      const int tiles = __shfl_sync(0xffffffffu, p.t1 - p.t0, 0);
      const int two = __shfl_sync(0xffffffffu, int(p.two()), 0);
      // tokens from the piece's first tile to the end of the context, the
      // tiles that hold them, and tree rows from the first tree tile on
      const int ctx_left = __shfl_sync(0xffffffffu, p.s.ctx - p.t0 * BN, 0);
      const int nt_ctx = __shfl_sync(0xffffffffu, max(p.s.nt_ctx - p.t0, 0), 0);
      const int n_left = __shfl_sync(0xffffffffu, p.s.n - max(p.t0 - p.s.nt_ctx, 0) * BN, 0);
      const int k = two ? stream ^ (u0 & 1) : 0;
      const int i0 = two ? 0 : (u0 & 1) ^ stream, di = 2 - two;
      const bool idle = i0 >= tiles;  // a single tile, and the other stream has it
      if (role < 2) {
        const int qb = (qc + k) & 1;
        for (int x = 0; x <= two; ++x) {
          const int buf = (qc + x) & 1;
          wait(&q_full[buf], ((qc + x) >> 1) & 1);
          if ((idle || x != k) && elect_one()) mbar_arrive(&q_empty[buf]);
          __syncwarp();
        }
        const uint64_t dq = dq0 + uint64_t(uint32_t(qb * Lay::Q_BYTES) >> 4);
        for (int i = 0; i < tiles; ++i) {
          const int g = g0 + i, st = g % ST;
          wait(&k_full[st], (g / ST) & 1);
          if (two || (i & 1) == i0) {
            const int u = two ? u0 + 2 * i + k : u0 + i;
            wait(&pv_done[u & 3], ((u >> 2) & 1) ^ 1);  // P(u - 4) has been read
            tc_fence_after();
            if (elect_one()) {
              const uint64_t dk = dk0 + uint64_t(uint32_t(st * Lay::TILE) >> 4);
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk)
                umma_f16(tm + (u & 3) * BN, dq + (((kk >> 2) * BM * 128 + (kk & 3) * 32) >> 4),
                         dk + (((kk >> 2) * BN * 128 + (kk & 3) * 32) >> 4), idesc_qk, kk > 0 ? 1u : 0u);
              umma_commit(&s_full[u & 3]);
              umma_commit(&k_empty[st]);
              if (i + di >= tiles) umma_commit(&q_empty[qb]);
            }
          } else if (elect_one()) {
            mbar_arrive(&k_empty[st]);
          }
          __syncwarp();
        }
        qc += 1 + two;
      } else {
        // the first product of a piece overwrites O, which the rows of the
        // piece before must have left
        wait(o_empty, (item & 1) ^ 1);
        for (int i = 0; i < tiles; ++i) {
          const int g = g0 + i, st = g % ST;
          wait(&v_full[st], (g / ST) & 1);
          if (two || (i & 1) == i0) {
            const int u = two ? u0 + 2 * i + k : u0 + i;
            // rows past the end take no part, but for the rest of the last 16
            const int steps = (min(BN, i < nt_ctx ? ctx_left - i * BN : n_left - (i - nt_ctx) * BN) + 15) / 16;
            wait(&p_full[u & 3], (u >> 2) & 1);
            tc_fence_after();
            if (elect_one()) {
              const uint64_t dv = dv0 + uint64_t(uint32_t(st * Lay::TILE) >> 4);
              const uint32_t to = tm + 4 * BN + stream * 128, tp = tm + (u & 3) * BN;
#pragma unroll
              for (int kk = 0; kk < BN / 16; ++kk)
                if (kk < steps)
                  umma_f16_ta(to, tp + kk * 8, dv + kk * (2048 >> 4), idesc_pv, (i != i0 || kk > 0) ? 1u : 0u);
              umma_commit(&pv_done[u & 3]);
              umma_commit(&v_empty[st]);
              if (i + di >= tiles) umma_commit(o_full);
            }
          } else if (elect_one()) {
            mbar_arrive(&v_empty[st]);
          }
          __syncwarp();
        }
        if (idle && elect_one()) mbar_arrive(o_full);
        __syncwarp();
        ++item;
      }
      g0 += tiles;
      u0 += tiles * (1 + two);
    }
    // every product and every arrival of this warp is done before the CTA
    // gives its memory back
    if (elect_one()) umma_commit(&drain[role]);
    __syncwarp();
    mbar_wait(&drain[role], 0, nullptr);
  } else if (busy) {
    // ------------------------------------------------------------ softmax
    const int stream = warp >> 2;
    const int row = threadIdx.x & 127;
    const uint32_t lane_off = uint32_t((warp & 3) * 32) << 16;
    const uint32_t tOs = tO + stream * 128 + lane_off;
    const float sl2 = a.scale_log2;
    int g = 0, u0 = 0, item = 0;  // tiles and units before the piece, pieces
    // after a wait that ran out (recorded), later ones are skipped
    bool alive = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (alive) alive = mbar_wait(bar, parity, a.err);
      __syncwarp();
    };
    bool more = walk.next(a, p);
    while (more) {
      const int tiles = p.t1 - p.t0;
      const int k = p.two() ? stream ^ (u0 & 1) : 0;  // this stream's row tile
      const int rows = p.rows(a, k);
      const bool live = (warp & 3) * 32 < rows;  // warps without a valid row only keep the barriers going
      const int node = (2 * p.pair + k) * a.nodes + row / a.group;
      const bool mine = row < rows;
      float m_ref = -INFINITY, l0 = 0.f, l1 = 0.f;
      // mask words of the piece's first tree tile, read ahead
      const int tree0 = max(p.t0, p.s.nt_ctx);
      uint32_t ahead[2] = {0u, 0u};
      if (tree0 < p.t1 && mine && a.mask != nullptr) {
        const int word = (tree0 - p.s.nt_ctx) * (BN / 32);
        const int32_t* mp = a.mask + int64_t(p.s.lo + node) * a.words;
        if (word < a.words) ahead[0] = uint32_t(mp[word]);
        if (word + 1 < a.words) ahead[1] = uint32_t(mp[word + 1]);
      }
      bool odd = false;   // the piece's tree V holds values that are not finite
      bool fresh = true;  // no unit of this stream yet
      const int i0 = p.two() ? 0 : (u0 & 1) ^ stream, di = p.two() ? 1 : 2;
      for (int i = i0; i < tiles; i += di) {
        const int j = p.t0 + i, u = p.two() ? u0 + 2 * i + k : u0 + i;
        const int buf = u & 3;
        const uint32_t tS = tmem + buf * BN + lane_off;
        const bool tree = j >= p.s.nt_ctx;
        const int col0 = tree ? (j - p.s.nt_ctx) * BN : j * BN;
        const int valid = min(BN, (tree ? p.s.n : p.s.ctx) - col0);
        wait(&s_full[buf], (u >> 2) & 1);
        tc_fence_after();
        if (tree || valid < BN) {
          // P is zero in masked places, but zero times an infinity or NaN is
          // not: rows past the end are cleared, and values of tree rows that
          // are not finite are cleared here and added back to the rows that
          // see them after the last product.  (The stage's phase before this
          // one is complete: S(u) came after P V of unit u - 4, at most four
          // tiles back, whose issuer had waited for every tile before it.)
          const int st = (g + i) % ST;
          wait(&v_full[st], ((g + i) / ST) & 1);
          const int tag = p.two() ? u0 + 2 * i : u;
          const int part = p.two() ? threadIdx.x : row, parts = p.two() ? 256 : 128;
          {
            // the products read whole steps of 16 rows: clear the rest of the
            // last one; look through the rows of a tree tile
            uint8_t* v = smem + Lay::OFF_V + st * Lay::TILE;
            const int from = tree ? 0 : valid * (D / 8), upto = (valid + 15) / 16 * 16 * (D / 8);
#pragma unroll 2
            for (int e = from + part; e < upto; e += parts) {
              uint4* w = reinterpret_cast<uint4*>(v + tile_offset(BN, e / (D / 8), e % (D / 8)));
              if (e >= valid * (D / 8)) {
                *w = make_uint4(0, 0, 0, 0);
              } else {
                const uint4 x = *w;
                if (odd2<T>(x.x) || odd2<T>(x.y) || odd2<T>(x.z) || odd2<T>(x.w)) {
                  uint16_t* h = reinterpret_cast<uint16_t*>(w);
                  for (int c = 0; c < 8; ++c)
                    if (odd2<T>(h[c])) h[c] = 0;
                  sh.odd[tag & 3] = uint32_t(tag) + 1;
                }
              }
            }
            fence_proxy_async_smem();
          }
          __syncwarp();  // bar.sync and the tcgen05 loads and stores want whole warps
          bar_sync(p.two() ? 3 : 1 + stream, parts);
          if (tree) odd = odd || sh.odd[tag & 3] == uint32_t(tag) + 1;
        }
        if (live) {
          uint32_t r[2][32];
          tmem_ld32(tS, r[0]);
          tmem_ld32(tS + 32, r[1]);
          tmem_wait_ld();
          if (tree || valid < BN) {
            uint32_t vis[2] = {0, 0};
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              const int left = valid - 32 * w;
              uint32_t in = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
              if (tree) {
                if (a.mask != nullptr) {
                  const int word = (col0 >> 5) + w;
                  if (j == tree0) in &= ahead[w];
                  else in &= mine && word < a.words ? uint32_t(a.mask[int64_t(p.s.lo + node) * a.words + word]) : 0u;
                } else {
                  const int upto = node - col0 - 32 * w + 1;  // rows up to itself
                  in &= upto >= 32 ? 0xffffffffu : upto <= 0 ? 0u : (1u << upto) - 1u;
                }
              }
              vis[w] = in;
            }
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((vis[c] >> e) & 1u)) r[c][e] = __float_as_uint(-INFINITY);
          }
          float mxa[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) mxa[x] = -INFINITY;
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 32; e += 2)
              mxa[c * 2 + (e >> 4)] =
                  max3(mxa[c * 2 + (e >> 4)], __uint_as_float(r[c][e]), __uint_as_float(r[c][e + 1]));
          const float mxs = max3(fmaxf(mxa[0], mxa[1]), mxa[2], mxa[3]) * sl2;
          // rescale lazily: only when the maximum grew by more than the threshold
          const bool rescale = mxs > m_ref + kRescaleThreshold;
          const float m_use = rescale ? mxs : m_ref;
          const float neg_m = m_use == -INFINITY ? 0.f : kLift<T> - m_use;  // nothing visible yet: all P are 0
          float sa[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float x0, x1;
              fma2s(x0, x1, __uint_as_float(r[c][2 * e]), __uint_as_float(r[c][2 * e + 1]), sl2, neg_m);
              const float p0 = ex2(x0), p1 = ex2(x1);
              add2(sa[c][0], sa[c][1], p0, p1);
              // P in the type of V for the second product (its row sum stays fp32)
              pk[e] = pack2<T>(p0, p1);
            }
            tmem_st16(tS + c * 16, pk);
          }
          if (!fresh && __any_sync(0xffffffffu, rescale)) {
            wait(&pv_done[(u - 2) & 3], ((u - 2) >> 2) & 1);
            tc_fence_after();
            const float f = rescale ? ex2(m_ref - m_use) : 1.0f;
            __syncwarp();
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(tOs + c * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st32(tOs + c * 32, o);
            }
            l0 *= f;
            l1 *= f;
          }
          tmem_wait_st();
          if (rescale) m_ref = m_use;
          l0 += sa[0][0] + sa[1][0];
          l1 += sa[0][1] + sa[1][1];
        }
        fresh = false;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[buf]);
      }
      // find the next piece while the last products run
      const Piece e = p;
      more = walk.next(a, p);
      const bool two = e.two(), whole = e.whole();
      float l = l0 + l1, f0 = 1.f, f1 = 0.f, m = m_ref;
      const bool join = !two && tiles > 1;  // both streams hold a part of every row
      if (!two) {
        // every warp has read the piece before's (it gave O back after that)
        wait(o_empty, (item & 1) ^ 1);
        sh.ml[stream][row] = make_float2(m_ref, l);
        if (row == 0) sh.piece_odd[stream] = odd;
        __syncwarp();
        bar_sync(4, 256);
        const float2 x = sh.ml[0][row], y = sh.ml[1][row];
        m = fmaxf(x.x, y.x);
        // weights of the two streams; the one without a unit is not read
        const int only = u0 & 1;
        f0 = join || only == 0 ? (x.x == -INFINITY ? 0.f : ex2(x.x - m)) : 0.f;
        f1 = join || only == 1 ? (y.x == -INFINITY ? 0.f : ex2(y.x - m)) : 0.f;
        l = x.y * f0 + y.y * f1;
        odd = sh.piece_odd[0] || sh.piece_odd[1];
      }
      wait(o_full, item & 1);  // the piece's O is complete
      tc_fence_after();
      if (live) {
        const int slot = (2 * int(blockIdx.x) + (e.starts() ? 1 : 0)) * 2 + k;
        const float inv = whole ? (l > 0.f || l != l ? 1.0f / l : 0.f) : 1.0f;
        const int qh = e.h * a.group + row % a.group;
        uint16_t* orow = reinterpret_cast<uint16_t*>(a.out) + int64_t(e.s.lo + node) * a.out_r + int64_t(qh) * a.out_h;
        float4* prow = a.part_o + int64_t(slot) * (D / 4) * a.part_rows + row;
        // two row tiles: all columns of the own one; else half of the columns of both streams' O
        constexpr int NC = D / 32;
        const int c_lo = two ? 0 : stream * (NC / 2), c_hi = two ? NC : c_lo + NC / 2;
#pragma unroll 1
        for (int c = c_lo; c < c_hi; ++c) {
          uint32_t o[32];
          __syncwarp();
          if (two) {
            tmem_ld32(tOs + c * 32, o);
            tmem_wait_ld();
          } else {
            tmem_ld32(tO + ((u0 & 1) ? 128 : 0) + lane_off + c * 32, o);
            if (join) {
              uint32_t o2[32];
              tmem_ld32(tO + ((u0 & 1) ? 0 : 128) + lane_off + c * 32, o2);
              tmem_wait_ld();
              const float fa = (u0 & 1) ? f1 : f0, fb = (u0 & 1) ? f0 : f1;
#pragma unroll
              for (int x = 0; x < 32; ++x)
                o[x] = __float_as_uint(fmaf(__uint_as_float(o[x]), fa, __uint_as_float(o2[x]) * fb));
            } else {
              tmem_wait_ld();
            }
          }
          if (c + 1 == c_hi) {  // O is read: the next piece's products may begin
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(o_empty);
          }
          if (mine && odd) {
            const int from = max(e.t0 - e.s.nt_ctx, 0) * BN, upto = min((e.t1 - e.s.nt_ctx) * BN, e.s.n);
            for (int t = from; t < upto; ++t) {
              const bool sees =
                  a.mask == nullptr
                      ? t <= node
                      : (t >> 5) < a.words &&
                            (uint32_t(a.mask[int64_t(e.s.lo + node) * a.words + (t >> 5)]) >> (t & 31)) & 1u;
              if (!sees) continue;
              const T* v = reinterpret_cast<const T*>(a.vt) + int64_t(e.s.lo + t) * a.vt_r + e.h * a.vt_h + c * 32;
#pragma unroll
              for (int x = 0; x < 32; ++x) {
                const float y = as_float<T>(v[x]);
                if (!(fabsf(y) < INFINITY)) o[x] = __float_as_uint(__uint_as_float(o[x]) + y);
              }
            }
          }
          if (mine && whole) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              uint4 w;
              w.x = pack2<T>(__uint_as_float(o[8 * v + 0]) * inv, __uint_as_float(o[8 * v + 1]) * inv);
              w.y = pack2<T>(__uint_as_float(o[8 * v + 2]) * inv, __uint_as_float(o[8 * v + 3]) * inv);
              w.z = pack2<T>(__uint_as_float(o[8 * v + 4]) * inv, __uint_as_float(o[8 * v + 5]) * inv);
              w.w = pack2<T>(__uint_as_float(o[8 * v + 6]) * inv, __uint_as_float(o[8 * v + 7]) * inv);
              *reinterpret_cast<uint4*>(orow + c * 32 + v * 8) = w;
            }
          } else if (mine) {
#pragma unroll
            for (int v = 0; v < 8; ++v)
              prow[(c * 8 + v) * a.part_rows] =
                  make_float4(__uint_as_float(o[4 * v]), __uint_as_float(o[4 * v + 1]), __uint_as_float(o[4 * v + 2]),
                              __uint_as_float(o[4 * v + 3]));
          }
        }
        if (mine && !whole && (two || stream == 0)) a.part_ml[int64_t(slot) * a.part_rows + row] = make_float2(m, l);
      }
      if (!live && lane == 0) mbar_arrive(o_empty);
      __syncwarp();
      ++item;
      g += tiles;
      u0 += tiles * (two ? 2 : 1);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    __syncwarp();
    tmem_dealloc<Lay::TMEM_COLS>(tmem);
  }
}

// Joins the records of items that several CTAs shared.  An item has a worker
// for each CTA whose share begins inside it (an item that no share begins
// inside of, or only at its first tile and that ends before the next, was
// whole), so the work is spread like the main kernel's.  A warp joins two
// neighbouring rows at a time, records in the order of their tiles, sixteen in
// a round: their maxima and sums first (one lane a record and row), then O,
// with the loads of four records in flight.  Rows of no request become zero.
// All of it is a few dependent reads from L2: bound by latency (64 requests:
// the call took 130 us in a CUDA graph; 142 with a block on a batch of rows at
// a time).
constexpr int kMergeThreads = 256;
constexpr int kMergeSplit = 4;  // CTAs a worker

template <typename T, int D>
__global__ void __launch_bounds__(kMergeThreads) tree_merge_kernel(const TreeArgs a) {
  constexpr int NC = D / 64;  // float4 of a row that a lane takes
  const int lane = threadIdx.x & 31, rr = lane & 1, c0 = lane >> 1;
  {  // inputs only, so before the wait
    const int lo = min(max(a.indptr[0], 0), a.R), hi = min(max(a.indptr[a.B], lo), a.R);
    const int hq = a.hkv * a.group, free_rows = lo + a.R - hi;
    const int64_t step = int64_t(gridDim.x) * kMergeThreads;
    for (int64_t e = int64_t(blockIdx.x) * kMergeThreads + threadIdx.x; e < int64_t(free_rows) * hq * (D / 8); e += step) {
      const int64_t rh = e / (D / 8);
      int r = int(rh / hq);
      r = r < lo ? r : hi + r - lo;
      *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + r * a.out_r + (rh % hq) * a.out_h +
                                (e % (D / 8)) * 8) = make_uint4(0, 0, 0, 0);
    }
  }
  pdl_wait();
  const int cta = blockIdx.x / kMergeSplit, part = blockIdx.x % kMergeSplit;
  const int4 meta = a.meta[cta];
  if (!meta.w) return;
  const int share = meta.z, at = cta * share;
  Piece p;
  p.s = request_shape(a, meta.x);
  const Segments seg(p.s, share);
  locate(p.s, seg, at - meta.y, p);
  const int head = meta.y + p.h * p.s.pairs * p.s.nt;
  auto first_tile = [&](int i) { return head + seg.start(i) * p.s.pairs + p.pair * seg.length(i); };
  int workers = 0, rank = 0, records = 0;
#pragma unroll 1
  for (int i = 0; i < seg.count; ++i) {
    const int x = first_tile(i), y = x + seg.length(i) - 1;
    const int first = x / share, last = y / share, begins = first + (first * share < x ? 1 : 0);
    if (i == p.segment) rank = workers + cta - begins;
    workers += last - begins + 1;
    records += last - first + 1;
  }
  if (records == 1) return;  // one CTA had the whole item
  const int rows0 = p.rows(a, 0), rows = rows0 + (p.two() ? p.rows(a, 1) : 0);
  const int stride = workers * kMergeSplit * (kMergeThreads / 32);
#pragma unroll 1
  for (int pr = (rank * kMergeSplit + part) * (kMergeThreads / 32) + (threadIdx.x >> 5); 2 * pr < rows; pr += stride) {
    const int abs = min(2 * pr + rr, rows - 1), tile = abs >= rows0, row = abs - (tile ? rows0 : 0);
    float m = -INFINITY, l = 0.f;
    float4 acc[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int k0 = 0; k0 < records; k0 += 16) {
      int k = k0 + c0, slot = -1;
      float2 ml = make_float2(-INFINITY, 0.f);
      if (k < records) {
        // records are numbered along the segments
        int first = first_tile(0) / share;
        if (seg.count > 1) {
#pragma unroll 1
          for (int i = 0;; ++i) {
            const int x = first_tile(i);
            first = x / share;
            const int n = (x + seg.length(i) - 1) / share - first + 1;
            if (k < n || i + 1 == seg.count) break;
            k -= n;
          }
        }
        slot = (2 * (first + k) + (k == 0 ? 1 : 0)) * 2 + tile;
        ml = a.part_ml[int64_t(slot) * a.part_rows + row];
      }
      float mx = fmaxf(m, ml.x);
#pragma unroll
      for (int d = 16; d > 1; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
      const float f = m == -INFINITY ? 0.f : ex2(m - mx), w = ml.x == -INFINITY ? 0.f : ex2(ml.x - mx);
      float sum = ml.y * w;
#pragma unroll
      for (int d = 16; d > 1; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      l = l * f + sum;
      m = mx;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        acc[i].x *= f;
        acc[i].y *= f;
        acc[i].z *= f;
        acc[i].w *= f;
      }
      const int n = min(16, records - k0);
#pragma unroll 1
      for (int x = 0; x < n; x += 4) {
        float4 o[4][NC];
        float wx[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          wx[y] = __shfl_sync(0xffffffffu, w, (2 * (x + y) + rr) & 31);
          const int s = __shfl_sync(0xffffffffu, slot, (2 * (x + y) + rr) & 31);
#pragma unroll
          for (int i = 0; i < NC; ++i)
            o[y][i] = x + y < n ? a.part_o[(int64_t(s) * (D / 4) + c0 + 16 * i) * a.part_rows + row]
                                : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int i = 0; i < NC; ++i) {
            acc[i].x = fmaf(o[y][i].x, wx[y], acc[i].x);
            acc[i].y = fmaf(o[y][i].y, wx[y], acc[i].y);
            acc[i].z = fmaf(o[y][i].z, wx[y], acc[i].z);
            acc[i].w = fmaf(o[y][i].w, wx[y], acc[i].w);
          }
      }
    }
    if (2 * pr + rr < rows) {
      const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
      const int node = (2 * p.pair + tile) * a.nodes + row / a.group, qh = p.h * a.group + row % a.group;
      uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + int64_t(p.s.lo + node) * a.out_r + int64_t(qh) * a.out_h;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        uint2 v;
        v.x = pack2<T>(acc[i].x * inv, acc[i].y * inv);
        v.y = pack2<T>(acc[i].z * inv, acc[i].w * inv);
        *reinterpret_cast<uint2*>(out + (c0 + 16 * i) * 4) = v;
      }
    }
    __syncwarp();
  }
}

// Tensor map of rows of D elements with up to three outer dimensions, outer
// dimensions in the order of their strides as the encoder wants them.
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    KVS_CUDA_CHECK(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q));
    KVS_CHECK_ARG(p != nullptr && q == cudaDriverEntryPointSuccess, "cuTensorMapEncodeTiled not available");
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

// `t` [..., rows, heads, D] (3-D) or [blocks, rows, heads, D] (4-D); false if
// the layout does not fit a tensor map.
bool encode_rows(CUtensorMap& m, const torch::Tensor& t, int box_rows, bool& head_first, int box_heads = 1) {
  const int rank = int(t.dim());
  const int64_t rows = t.size(rank - 3), heads = t.size(rank - 2);
  const int64_t s_row = t.stride(rank - 3) * 2, s_head = t.stride(rank - 2) * 2;
  head_first = heads == 1 || (rows > 1 && s_head <= s_row);
  const cuuint64_t row_bytes = cuuint64_t(t.size(rank - 1)) * 2;
  cuuint64_t dims[4] = {cuuint64_t(t.size(rank - 1)), 0, 0, rank == 4 ? cuuint64_t(t.size(0)) : 1};
  cuuint64_t strides[3] = {0, 0, 0};
  cuuint32_t box[4] = {64, 1, 1, 1}, unit[4] = {1, 1, 1, 1};
  const int dr = head_first ? 2 : 1, dh = head_first ? 1 : 2;
  dims[dr] = cuuint64_t(rows);
  dims[dh] = cuuint64_t(heads);
  // a dimension of size one may have any stride: give it one that fits
  strides[dr - 1] = rows == 1 ? (head_first ? cuuint64_t(std::max<int64_t>(s_head, row_bytes)) * heads : row_bytes)
                              : cuuint64_t(s_row);
  strides[dh - 1] = heads == 1 ? (head_first ? row_bytes : cuuint64_t(std::max<int64_t>(s_row, row_bytes)) * rows)
                               : cuuint64_t(s_head);
  if (rank == 4)
    strides[2] = t.size(0) == 1 ? std::max(strides[0] * dims[1], strides[1] * dims[2]) : cuuint64_t(t.stride(0) * 2);
  for (int d = 0; d + 1 < rank; ++d)
    if (strides[d] < row_bytes || strides[d] % 16 != 0 || strides[d] >= (cuuint64_t(1) << 40)) return false;
  box[dr] = cuuint32_t(box_rows);
  box[dh] = cuuint32_t(box_heads);
  return encode_fn()(&m,
                     t.scalar_type() == at::kHalf ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                     cuuint32_t(rank), t.data_ptr(), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
void launch(const CUtensorMap* m, const TreeArgs& a, int grid, cudaStream_t st) {
  // per device, so set at every launch (a few hundred nanoseconds)
  KVS_CUDA_CHECK(cudaFuncSetAttribute(tree_attention_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      Layout<D>::SMEM));
  tree_attention_kernel<T, D><<<grid, kThreads, Layout<D>::SMEM, st>>>(m[0], m[1], m[2], m[3], m[4], a);
  KVS_CUDA_CHECK(cudaGetLastError());
  launch_pdl(tree_merge_kernel<T, D>, dim3(unsigned(grid * kMergeSplit)), dim3(kMergeThreads), 0, st, a);
}

}  // namespace

void paged_tree_attention(torch::Tensor q, torch::Tensor k_tree, torch::Tensor v_tree, torch::Tensor k_cache,
                          torch::Tensor v_cache, torch::Tensor block_tables, torch::Tensor ctx_lens,
                          torch::Tensor indptr, c10::optional<torch::Tensor> tree_mask, double scale,
                          torch::Tensor out, torch::Tensor status) {
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
  KVS_CHECK_ARG(Hq / Hkv <= BM, "tree attention: at most 128 query heads per KV head");
  KVS_CHECK_ARG(scale > 0, "tree attention: scale must be positive");
  KVS_CHECK_ARG(R * Hq < (int64_t(1) << 30) && k_cache.size(1) >= 1 && k_cache.size(0) >= 1 &&
                    k_cache.size(0) <= INT32_MAX && k_cache.size(1) <= INT32_MAX,
                "tree attention: too many rows, or an empty cache");
  if (R == 0) return;
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
  a.hkv = int(Hkv);
  a.num_blocks = k_cache.size(0);
  a.err = reinterpret_cast<uint32_t*>(status.data_ptr<int32_t>());
  // TMA boxes of the cache: the largest power of two of at least 8 tokens that
  // tiles both a block and a K/V tile; other block sizes are copied
  CUtensorMap m[5] = {};
  const int box = std::min(BN, a.bs & -a.bs);
  a.box = box >= 8 && encode_rows(m[0], k_cache, box, a.k_head_first) && encode_rows(m[1], v_cache, box, a.v_head_first)
              ? box
              : 0;
  a.tree_tma = encode_rows(m[2], k_tree, BN, a.kt_head_first) && encode_rows(m[3], v_tree, BN, a.vt_head_first);
  // Row tiles end at a tree node, and q boxes of 8 nodes (one box for large
  // groups) keep every box at the start of a swizzle pattern.
  a.q_box = a.group <= 16 ? 8 : BM / a.group;
  a.nodes = BM / a.group / a.q_box * a.q_box;
  bool q_head_first = false;
  a.q_tma = encode_rows(m[4], q, a.q_box, q_head_first, a.group) && q_head_first;
  const int grid = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  a.part_rows = int(std::min<int64_t>(BM, R * a.group));
  a.ctas = grid;
  const int64_t recs = int64_t(4) * grid * a.part_rows;
  // records (O, then maxima and sums) and the CTAs' places in the schedule, 16-byte words
  const int64_t words = recs * (D / 4) + (recs + 1) / 2 + grid;
  torch::Tensor scratch = torch::empty({words * 4}, q.options().dtype(at::kFloat));
  a.part_o = reinterpret_cast<float4*>(scratch.data_ptr<float>());
  a.part_ml = reinterpret_cast<float2*>(a.part_o + recs * (D / 4));
  a.meta = reinterpret_cast<int4*>(a.part_o + recs * (D / 4) + (recs + 1) / 2);
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  if (dt == at::kBFloat16) {
    if (D == 128) launch<bf16, 128>(m, a, grid, st);
    else launch<bf16, 64>(m, a, grid, st);
  } else {
    if (D == 128) launch<__half, 128>(m, a, grid, st);
    else launch<__half, 64>(m, a, grid, st);
  }
}

}  // namespace kvs
