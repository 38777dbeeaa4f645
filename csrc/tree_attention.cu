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
constexpr int kThreads = 192;  // warps 0..3 softmax, 4 loader, 5 MMA issuer
constexpr float kRescaleThreshold = 8.0f;  // log2: P stays below 2^8 between rescalings

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
  bool k_head_first, v_head_first, kt_head_first, vt_head_first;  // order of the middle tensor-map dimensions
  int min_share;
  int part_rows;   // rows kept per partial record
  float scale_log2;
  float* part_o;    // [2 * CTAs, part_rows, D]
  float2* part_ml;  // [2 * CTAs, part_rows]
  int64_t* base;    // [B + 1] first tile of each request, then the share
  uint32_t* err;
};

// ------------------------------------------------------------------ schedule
struct Shape {  // of one request
  int lo, n, ctx, nt_ctx, nt, mt;
};
__device__ __forceinline__ Shape request_shape(const TreeArgs& a, int b) {
  Shape s;
  s.lo = min(max(a.indptr[b], 0), a.R);
  s.n = max(min(a.indptr[b + 1], a.R) - s.lo, 0);
  s.ctx = int(max(min(int64_t(a.ctx[b]), int64_t(a.width) * a.bs), int64_t(0)));
  s.nt_ctx = (s.ctx + BN - 1) / BN;
  s.mt = int((int64_t(s.n) * a.group + BM - 1) / BM);
  s.nt = s.n > 0 ? s.nt_ctx + (s.n + BN - 1) / BN : 0;
  return s;
}
// Row tiles of one KV head read the same K/V.  Items with several row tiles
// are cut into segments of at least one CTA share and ordered (segment, row
// tile), so the CTAs that read one segment run side by side and all but the
// first find it in L2.
struct Segments {
  int count, len, longer;  // `longer` segments of len + 1 tiles, then segments of len
  __device__ __forceinline__ Segments(const Shape& s, int64_t share) {
    count = s.mt > 1 ? int(max(int64_t(1), int64_t(s.nt) / share)) : 1;
    len = s.nt / count;
    longer = s.nt % count;
  }
  __device__ __forceinline__ int length(int i) const { return len + (i < longer ? 1 : 0); }
  __device__ __forceinline__ int start(int i) const { return i * len + min(i, longer); }
};

struct Piece {  // consecutive tiles of one item
  Shape s;
  int b, h, mi;
  int t0, t1;    // tiles [t0, t1) of the item
  bool starts;   // begins its segment
  bool whole;    // the complete item
};

struct Walker {  // the pieces of one CTA's share, in order
  int64_t at, end, base, share;
  int b;
  Shape s;
  __device__ __forceinline__ bool next(const TreeArgs& a, Piece& p) {
    if (at >= end) return false;
    while (at >= base + int64_t(a.hkv) * s.mt * s.nt) {
      base += int64_t(a.hkv) * s.mt * s.nt;
      s = request_shape(a, ++b);
    }
    const Segments seg(s, share);
    const int64_t x = at - base;
    const int64_t per_head = int64_t(s.mt) * s.nt;
    p.s = s;
    p.b = b;
    p.h = int(x / per_head);
    const int64_t y = x - p.h * per_head;
    const int64_t big = int64_t(seg.len + 1) * s.mt;
    int i;
    if (y < big * seg.longer) i = int(y / big);
    else i = seg.longer + int((y - big * seg.longer) / (int64_t(seg.len) * s.mt));
    const int64_t z = y - int64_t(seg.start(i)) * s.mt;
    const int len = seg.length(i);
    p.mi = int(z / len);
    const int off = int(z - int64_t(p.mi) * len);
    const int take = int(min(int64_t(len - off), end - at));
    p.t0 = seg.start(i) + off;
    p.t1 = p.t0 + take;
    p.starts = off == 0;
    p.whole = take == s.nt;
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
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

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

template <int D>
struct Layout {
  static constexpr int STAGES = D == 128 ? 2 : 4;
  static constexpr int PANELS = D / 64;
  static constexpr int Q_BYTES = BM * D * 2;
  static constexpr int TILE = BN * D * 2;
  static constexpr int OFF_K = Q_BYTES, OFF_V = OFF_K + STAGES * TILE, OFF_BAR = OFF_V + STAGES * TILE;
  // barriers: k_full, k_empty, v_full, v_empty [STAGES] each, s_full[2],
  // p_full[2], pv_done[2], q_full, o_full
  static constexpr int NUM_BARS = 4 * STAGES + 8;
  static constexpr int SMEM = OFF_BAR + NUM_BARS * 8 + 1024;
  static constexpr uint32_t TMEM_COLS = 256;  // S/P double buffered (2 x 64), O (D)
};

// Copies the rows of one K or V tile with plain loads (one warp): caches
// whose blocks TMA boxes do not tile.  Rows at or past `valid` become zero.
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

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2)
    tree_attention_kernel(const __grid_constant__ CUtensorMap m_kc, const __grid_constant__ CUtensorMap m_vc,
                          const __grid_constant__ CUtensorMap m_kt, const __grid_constant__ CUtensorMap m_vt,
                          const TreeArgs a) {
  using Lay = Layout<D>;
  using namespace sm100;
  constexpr int ST = Lay::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Lay::OFF_BAR);
  uint64_t *k_full = bars, *k_empty = bars + ST, *v_full = bars + 2 * ST, *v_empty = bars + 3 * ST;
  uint64_t *s_full = bars + 4 * ST, *p_full = s_full + 2, *pv_done = s_full + 4, *q_full = s_full + 6,
           *o_full = s_full + 7;
  __shared__ uint32_t s_tmem;
  __shared__ int64_t s_sum[kThreads / 32];
  __shared__ int64_t s_base;
  __shared__ int s_b;
  __shared__ uint32_t s_odd[2];  // 1 + number of the last tile whose tree V held values that are not finite
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_trigger();

  if (threadIdx.x == 0) {
    for (int i = 0; i < Lay::NUM_BARS; ++i) mbar_init(&bars[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&p_full[i], 4);  // one arrival per softmax warp
    mbar_init(q_full, 128);
    fence_barrier_init();
    s_odd[0] = s_odd[1] = 0;
  }
  if (warp == 5) tmem_alloc<Lay::TMEM_COLS>(&s_tmem);

  // sum the tiles of all requests, twice: once for the total (and with it the
  // share), once to find the request that this CTA's share begins in
  Walker walk;
  walk.share = 0;
  int64_t total = 0;
  for (int pass = 0; pass < 2; ++pass) {
    int64_t carry = 0;
    for (int b0 = 0; b0 < a.B; b0 += kThreads) {
      const int b = b0 + threadIdx.x;
      int64_t mine = 0;
      if (b < a.B) {
        const Shape s = request_shape(a, b);
        mine = int64_t(a.hkv) * s.mt * s.nt;
      }
      int64_t x = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
      }
      __syncthreads();
      if (lane == 31) s_sum[warp] = x;
      __syncthreads();
      int64_t before = carry;
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) {
        before += w < warp ? s_sum[w] : 0;
        carry += s_sum[w];
      }
      if (pass == 1 && b < a.B) {
        const int64_t from = before + x - mine;
        if (blockIdx.x == 0) a.base[b] = from;
        if (walk.at >= from && walk.at < from + mine) {
          s_b = b;
          s_base = from;
        }
      }
    }
    if (pass == 0) {
      total = carry;
      walk.share = max((total + gridDim.x - 1) / int64_t(gridDim.x), int64_t(a.min_share));
      walk.at = blockIdx.x * walk.share;
      walk.end = min(walk.at + walk.share, total);
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.base[a.B] = walk.share;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const uint32_t tO = tmem + 2 * BN;
  const bool busy = walk.at < walk.end;
  if (busy) {
    walk.b = s_b;
    walk.base = s_base;
    walk.s = request_shape(a, walk.b);
  }
  Piece p;

  if (busy && warp == 4) {
    // ------------------------------------------------------------- loader
    bool ok = true;
    int g = 0;  // tiles so far, over all pieces
    while (ok && walk.next(a, p)) {
      const int32_t* table = a.tables + p.b * a.table_stride;
      for (int j = p.t0; j < p.t1 && ok; ++j, ++g) {
        const int st = g % ST;
        const uint32_t free_parity = ((g / ST) & 1) ^ 1;
        uint8_t *dk = smem + Lay::OFF_K + st * Lay::TILE, *dv = smem + Lay::OFF_V + st * Lay::TILE;
        if (j < p.s.nt_ctx) {
          const int t0 = j * BN, valid = min(BN, p.s.ctx - t0);
          if (a.box > 0) {
            const int boxes = (valid + a.box - 1) / a.box;
            int blk = 0, off = 0;
            if (lane < boxes) {
              const int t = t0 + lane * a.box;
              blk = table[t / a.bs];
              off = t % a.bs;
            }
            const uint32_t bytes = uint32_t(boxes) * a.box * D * 2;
            ok = mbar_wait(&k_empty[st], free_parity, a.err);
            if (lane == 0 && ok) mbar_arrive_expect_tx(&k_full[st], bytes);
            ok = __all_sync(0xffffffffu, ok);
            if (lane < boxes && ok)
              for (int c = 0; c < Lay::PANELS; ++c)
                tma_load_4d(dk + c * BN * 128 + lane * a.box * 128, &m_kc, c * 64, a.k_head_first ? p.h : off,
                            a.k_head_first ? off : p.h, blk, &k_full[st]);
            if (ok) ok = mbar_wait(&v_empty[st], free_parity, a.err);
            if (lane == 0 && ok) mbar_arrive_expect_tx(&v_full[st], bytes);
            ok = __all_sync(0xffffffffu, ok);
            if (lane < boxes && ok)
              for (int c = 0; c < Lay::PANELS; ++c)
                tma_load_4d(dv + c * BN * 128 + lane * a.box * 128, &m_vc, c * 64, a.v_head_first ? p.h : off,
                            a.v_head_first ? off : p.h, blk, &v_full[st]);
          } else {
            ok = __all_sync(0xffffffffu, mbar_wait(&k_empty[st], free_parity, a.err));
            if (ok) {
              copy_paged_tile<D>(dk, reinterpret_cast<const uint16_t*>(a.kc), a.kc_b, a.kc_t, p.h * a.kc_h, table, a,
                                 t0, valid, lane);
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) mbar_arrive(&k_full[st]);
              ok = __all_sync(0xffffffffu, mbar_wait(&v_empty[st], free_parity, a.err));
            }
            if (ok) {
              copy_paged_tile<D>(dv, reinterpret_cast<const uint16_t*>(a.vc), a.vc_b, a.vc_t, p.h * a.vc_h, table, a,
                                 t0, valid, lane);
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) mbar_arrive(&v_full[st]);
            }
          }
        } else {
          const int r0 = (j - p.s.nt_ctx) * BN, valid = min(BN, p.s.n - r0), row = p.s.lo + r0;
          ok = __all_sync(0xffffffffu, mbar_wait(&k_empty[st], free_parity, a.err));
          if (a.tree_tma) {
            if (ok && lane == 0) {
              mbar_arrive_expect_tx(&k_full[st], Lay::TILE);
              for (int c = 0; c < Lay::PANELS; ++c)
                tma_load_3d(dk + c * BN * 128, &m_kt, c * 64, a.kt_head_first ? p.h : row,
                            a.kt_head_first ? row : p.h, &k_full[st]);
            }
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&v_empty[st], free_parity, a.err));
            if (ok && lane == 0) {
              mbar_arrive_expect_tx(&v_full[st], Lay::TILE);
              for (int c = 0; c < Lay::PANELS; ++c)
                tma_load_3d(dv + c * BN * 128, &m_vt, c * 64, a.vt_head_first ? p.h : row,
                            a.vt_head_first ? row : p.h, &v_full[st]);
            }
          } else {
            if (ok) {
              copy_tile<D>(dk, reinterpret_cast<const uint16_t*>(a.kt) + row * a.kt_r + p.h * a.kt_h, a.kt_r, valid,
                           lane);
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) mbar_arrive(&k_full[st]);
              ok = __all_sync(0xffffffffu, mbar_wait(&v_empty[st], free_parity, a.err));
            }
            if (ok) {
              copy_tile<D>(dv, reinterpret_cast<const uint16_t*>(a.vt) + row * a.vt_r + p.h * a.vt_h, a.vt_r, valid,
                           lane);
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) mbar_arrive(&v_full[st]);
            }
          }
        }
      }
    }
    // every issued copy lands before the CTA may exit
    for (int i = max(0, g - ST); i < g; ++i) {
      mbar_wait(&k_full[i % ST], (i / ST) & 1, nullptr);
      mbar_wait(&v_full[i % ST], (i / ST) & 1, nullptr);
    }
  } else if (busy && warp == 5) {
    // --------------------------------------------------------- MMA issuer
    if (lane == 0) {
      constexpr uint32_t fmt = std::is_same<T, bf16>::value ? ~0u : ~((1u << 7) | (1u << 10));  // f16: type 0
      constexpr uint32_t idesc_qk = idesc_bf16(BM, BN, false) & fmt;
      constexpr uint32_t idesc_pv = idesc_bf16(BM, D, true) & fmt;
      const uint32_t q0 = smem_u32(smem), k0 = smem_u32(smem + Lay::OFF_K), v0 = smem_u32(smem + Lay::OFF_V);
      bool ok = true;
      int g = 0, item = 0;
      auto pv = [&](int gg, bool first) {
        const int st = gg % ST;
        ok = mbar_wait(&p_full[gg & 1], (gg >> 1) & 1, a.err) && mbar_wait(&v_full[st], (gg / ST) & 1, a.err);
        if (!ok) return;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < BN / 16; ++kk)
          umma_f16_ta(tO, tmem + (gg & 1) * BN + kk * 8, smem_desc_sw128(v0 + st * Lay::TILE + kk * 2048, BN * 128, 1024),
                      idesc_pv, (!first || kk > 0) ? 1u : 0u);
        umma_commit(&v_empty[st]);
        umma_commit(&pv_done[gg & 1]);
      };
      while (ok && walk.next(a, p)) {
        ok = mbar_wait(q_full, item & 1, a.err);
        for (int j = p.t0; j < p.t1 && ok; ++j, ++g) {
          const int st = g % ST;
          ok = mbar_wait(&k_full[st], (g / ST) & 1, a.err);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma_f16(tmem + (g & 1) * BN, smem_desc_sw128(q0 + (kk >> 2) * BM * 128 + (kk & 3) * 32, 16, 1024),
                     smem_desc_sw128(k0 + st * Lay::TILE + (kk >> 2) * BN * 128 + (kk & 3) * 32, 16, 1024), idesc_qk,
                     kk > 0 ? 1u : 0u);
          umma_commit(&s_full[g & 1]);
          umma_commit(&k_empty[st]);
          if (j > p.t0) pv(g - 1, j - 1 == p.t0);
        }
        if (ok) pv(g - 1, p.t1 - 1 == p.t0);
        if (ok) umma_commit(o_full);
        ++item;
      }
    }
  } else if (busy) {
    // ------------------------------------------------------------ softmax
    const int row = threadIdx.x;
    const uint32_t lane_off = uint32_t(warp * 32) << 16;
    const float sl2 = a.scale_log2;
    bool ok = true;
    int g = 0, item = 0;
    while (walk.next(a, p)) {
      const int rows = p.s.n * a.group - p.mi * BM;  // valid rows of the tile (may exceed it)
      // Q rows: the previous piece's last S tile has been seen, so its Q is free
      {
        const uint16_t* q = reinterpret_cast<const uint16_t*>(a.q);
        constexpr int C = D / 8;
        const int most = min(rows, BM);
        for (int e = threadIdx.x; e < most * C; e += 128) {
          const int r = e / C, c = e % C, flat = p.mi * BM + r, node = flat / a.group, hg = flat % a.group;
          const uint4 v = *reinterpret_cast<const uint4*>(q + int64_t(p.s.lo + node) * a.q_r +
                                                          int64_t(p.h * a.group + hg) * a.q_h + c * 8);
          *reinterpret_cast<uint4*>(smem + tile_offset(BM, r, c)) = v;
        }
        fence_proxy_async_smem();
        mbar_arrive(q_full);
      }
      const bool live = warp * 32 < rows;  // warps without a valid row only keep the barriers going
      const int flat = p.mi * BM + row, node = flat / a.group;
      const bool mine = row < rows;
      float m_ref = -INFINITY, l0 = 0.f, l1 = 0.f;
      bool odd = false;  // the piece's tree V holds values that are not finite
      for (int j = p.t0; j < p.t1; ++j, ++g) {
        const int buf = g & 1, st = g % ST;
        const uint32_t tS = tmem + buf * BN + lane_off;
        const bool tree = j >= p.s.nt_ctx;
        const int col0 = tree ? (j - p.s.nt_ctx) * BN : j * BN;
        const int valid = min(BN, (tree ? p.s.n : p.s.ctx) - col0);
        ok = ok && mbar_wait(&s_full[buf], (g >> 1) & 1, a.err);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
        if (tree || valid < BN) {
          // P is zero in masked places, but zero times an infinity or NaN is
          // not: rows past the end are cleared, and values of tree rows that
          // are not finite are cleared here and added back to the rows that
          // see them after the last product.
          ok = ok && mbar_wait(&v_full[st], (g / ST) & 1, a.err);
          ok = __all_sync(0xffffffffu, ok);
          if (ok) {
            const int r = row >> 1, part = row & 1;
            constexpr int HC = D / 16;  // 16-byte chunks of half a row
            uint8_t* v = smem + Lay::OFF_V + st * Lay::TILE;
            if (r >= valid) {
              for (int c = 0; c < HC; ++c)
                *reinterpret_cast<uint4*>(v + tile_offset(BN, r, part * HC + c)) = make_uint4(0, 0, 0, 0);
            } else if (tree) {
              for (int c = 0; c < HC; ++c) {
                uint32_t* w = reinterpret_cast<uint32_t*>(v + tile_offset(BN, r, part * HC + c));
                for (int e = 0; e < 4; ++e)
                  if (odd2<T>(w[e])) {
                    uint16_t* h = reinterpret_cast<uint16_t*>(w + e);
                    if (odd2<T>(h[0])) h[0] = 0;
                    if (odd2<T>(h[1])) h[1] = 0;
                    s_odd[buf] = uint32_t(g) + 1;
                  }
              }
            }
            fence_proxy_async_smem();
          }
          softmax_sync();
          if (tree) odd = odd || s_odd[buf] == uint32_t(g) + 1;
        }
        if (live && ok) {
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
                  in &= mine && word < a.words ? uint32_t(a.mask[int64_t(p.s.lo + node) * a.words + word]) : 0u;
                } else {
                  const int upto = node - col0 - 32 * w + 1;  // rows up to itself
                  in &= upto >= 32 ? 0xffffffffu : upto <= 0 ? 0u : (1u << upto) - 1u;
                }
              }
              vis[w] = in;
            }
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((vis[c] >> e) & 1u)) r[c][e] = __float_as_uint(-INFINITY);
          }
          float mxa[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) mxa[i] = -INFINITY;
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
          const float neg_m = m_use == -INFINITY ? 0.f : -m_use;  // nothing visible yet: all P are 0
          float sa[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
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
          if (__any_sync(0xffffffffu, rescale && j > p.t0)) {
            ok = mbar_wait(&pv_done[buf ^ 1], ((g - 1) >> 1) & 1, a.err);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            const float f = rescale ? ex2(m_ref - m_use) : 1.0f;
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(tO + lane_off + c * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st32(tO + lane_off + c * 32, o);
            }
            l0 *= f;
            l1 *= f;
          }
          tmem_wait_st();
          if (rescale) m_ref = m_use;
          l0 += sa[0][0] + sa[1][0];
          l1 += sa[0][1] + sa[1][1];
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0 && ok) mbar_arrive(&p_full[buf]);
      }
      // the piece's O is complete
      ok = ok && mbar_wait(o_full, item & 1, a.err);
      ok = __all_sync(0xffffffffu, ok);
      ++item;
      if (!ok || !live) continue;
      tc_fence_after();
      const float l = l0 + l1;
      const int64_t slot = 2 * int64_t(blockIdx.x) + (p.starts ? 1 : 0);
      const float inv = p.whole ? (l > 0.f || l != l ? 1.0f / l : 0.f) : 1.0f;
      const int qh = p.h * a.group + flat % a.group;
      uint16_t* orow = reinterpret_cast<uint16_t*>(a.out) + int64_t(p.s.lo + node) * a.out_r + int64_t(qh) * a.out_h;
      float* prow = a.part_o + (slot * a.part_rows + row) * D;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(tO + lane_off + c * 32, o);
        tmem_wait_ld();
        if (mine && odd) {
          const int from = max(p.t0 - p.s.nt_ctx, 0) * BN, upto = min((p.t1 - p.s.nt_ctx) * BN, p.s.n);
          for (int t = from; t < upto; ++t) {
            const bool sees = a.mask == nullptr
                                  ? t <= node
                                  : (t >> 5) < a.words &&
                                        (uint32_t(a.mask[int64_t(p.s.lo + node) * a.words + (t >> 5)]) >> (t & 31)) & 1u;
            if (!sees) continue;
            const T* v = reinterpret_cast<const T*>(a.vt) + int64_t(p.s.lo + t) * a.vt_r + p.h * a.vt_h + c * 32;
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float x = as_float<T>(v[e]);
              if (!(fabsf(x) < INFINITY)) o[e] = __float_as_uint(__uint_as_float(o[e]) + x);
            }
          }
        }
        if (mine && p.whole) {
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
            *reinterpret_cast<uint4*>(prow + c * 32 + v * 4) =
                make_uint4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
        }
      }
      if (mine && !p.whole) a.part_ml[slot * a.part_rows + row] = make_float2(m_ref, l);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc<Lay::TMEM_COLS>(tmem);
  }
}

// Joins the records of items that several CTAs shared: one warp per (row,
// head), records in the order of their tiles.  Padding rows become zero.
template <typename T, int D>
__global__ void __launch_bounds__(128) tree_merge_kernel(const TreeArgs a) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t w = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int hq = a.hkv * a.group;
  const int r = int(w / hq), qh = int(w % hq);
  if (r >= a.R) return;
  constexpr int E = D / 32;
  T* out = reinterpret_cast<T*>(a.out) + r * a.out_r + qh * a.out_h + lane * E;
  auto store = [&](const float (&v)[E]) {
#pragma unroll
    for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(out + e) = pack2<T>(v[e], v[e + 1]);
  };
  // the last request with indptr[b] <= r
  int b = 0;
  for (int hi = a.B; hi - b > 1;) {
    const int mid = (b + hi) >> 1;
    if (a.indptr[mid] <= r) b = mid; else hi = mid;
  }
  const Shape s = request_shape(a, b);
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  if (r >= s.lo + s.n || r < s.lo) {
    store(acc);
    return;
  }
  const int64_t share = a.base[a.B];
  const int h = qh / a.group, flat = (r - s.lo) * a.group + qh % a.group, mi = flat / BM, row = flat % BM;
  const Segments seg(s, share);
  const int64_t first = a.base[b] + int64_t(h) * s.mt * s.nt;
  float m = -INFINITY, l = 0.f;
  for (int i = 0; i < seg.count; ++i) {
    const int64_t g0 = first + int64_t(seg.start(i)) * s.mt + int64_t(mi) * seg.length(i);
    const int64_t c0 = g0 / share, c1 = (g0 + seg.length(i) - 1) / share;
    if (seg.count == 1 && c0 == c1) return;  // one CTA had the whole item
    for (int64_t c = c0; c <= c1; ++c) {
      const int64_t rec = (2 * c + (c == c0 ? 1 : 0)) * a.part_rows + row;
      const float2 ml = a.part_ml[rec];
      float o[E];
      const float* po = a.part_o + rec * D + lane * E;
      if constexpr (E == 4) *reinterpret_cast<float4*>(o) = *reinterpret_cast<const float4*>(po);
      else *reinterpret_cast<float2*>(o) = *reinterpret_cast<const float2*>(po);
      const float mx = fmaxf(m, ml.x);
      if (mx == -INFINITY) {  // nothing visible so far; a NaN sum still counts
        l += ml.y;
        continue;
      }
      const float f = ex2(m - mx), k = ex2(ml.x - mx);
      l = l * f + ml.y * k;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = acc[e] * f + (ml.x == -INFINITY ? 0.f : o[e] * k);
      m = mx;
    }
  }
  const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] *= inv;
  store(acc);
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
bool encode_rows(CUtensorMap& m, const torch::Tensor& t, int box_rows, bool& head_first) {
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
  tree_attention_kernel<T, D><<<grid, kThreads, Layout<D>::SMEM, st>>>(m[0], m[1], m[2], m[3], a);
  KVS_CUDA_CHECK(cudaGetLastError());
  const int64_t warps = int64_t(a.R) * a.hkv * a.group;
  launch_pdl(tree_merge_kernel<T, D>, dim3(unsigned((warps + 3) / 4)), dim3(128), 0, st, a);
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
  a.min_share = 1;
  a.err = reinterpret_cast<uint32_t*>(status.data_ptr<int32_t>());
  // TMA boxes of the cache: the largest power of two of at least 8 tokens that
  // tiles both a block and a K/V tile; other block sizes are copied
  CUtensorMap m[4] = {};
  const int box = std::min(BN, a.bs & -a.bs);
  a.box = box >= 8 && encode_rows(m[0], k_cache, box, a.k_head_first) && encode_rows(m[1], v_cache, box, a.v_head_first)
              ? box
              : 0;
  a.tree_tma = encode_rows(m[2], k_tree, BN, a.kt_head_first) && encode_rows(m[3], v_tree, BN, a.vt_head_first);
  const int grid = 2 * at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  a.part_rows = int(std::min<int64_t>(BM, R * a.group));
  const int64_t recs = int64_t(2) * grid * a.part_rows;
  torch::Tensor scratch = torch::empty({recs * (D + 2) + 2 * (B + 1)}, q.options().dtype(at::kFloat));
  a.part_o = scratch.data_ptr<float>();
  a.part_ml = reinterpret_cast<float2*>(a.part_o + recs * D);
  a.base = reinterpret_cast<int64_t*>(a.part_o + recs * (D + 2));
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
