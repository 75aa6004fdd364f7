// Head norms of queries and keys with the position rotation in one pass, and
// the backward pass, sm_100a.  (The reference has no head norm and rotates
// inside its forward-only attention kernel, src/smooth_attn/kernels.py:
// 2147-2159; the map of one row is stated in qk_rope.cuh.)
//
// Backward of one row, with n, r of the forward and dn the rotation's
// transpose applied to dy:
//   dn[i]       = dy[i] c_i + dy[i + R/2] s_i
//   dn[i + R/2] = dy[i + R/2] c_i - dy[i] s_i
//   g  = dn * w
//   dx = r (g - x r^2 mean(g x))
//   dw = sum over rows of dn x r
// r is formed again from x, which the backward reads anyhow, so the forward
// saves nothing.
//
// Bound: HBM.  Forward reads x and writes y (2 x 168 MB at [4, 32 + 8, 4096, 128]
// bf16: 57 us, 0.92 of the measured copy rate), backward reads x and dy and writes
// dx (85 us, 0.92).  The rows go through the walk of qk_rope.cuh, q's and k's warps
// side by side in one launch, shared out by the work of each.  dw: every lane keeps
// fp32 sums of its own 16 channels over the rows it meets, a block adds its warps'
// sums in a fixed order and writes one row of partial sums for each of q and k,
// and a second small kernel (4 us) adds those in a fixed order: no atomics,
// bitwise the same from run to run.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "qk_rope.cuh"
#include "smooth_attn_b200.h"

int sa_record_cuda_error(cudaError_t e);

namespace sa {
namespace qkr {

static __device__ unsigned g_bad_positions;

struct Side {
  const void* x;
  void* y;          // forward: y; backward: dx
  const void* dy;   // backward
  const void* w;    // nullable
  int64_t xb, xh, xt, yb, yh, yt, gb, gh, gt;  // element strides
  int64_t units;    // groups * per
  int H, C, per;    // heads, heads of a unit, units of a token group
};

struct Shape {
  int64_t N, T;     // B * T tokens
  int64_t q_warps;  // warps that walk over q; the others walk over k
  int w_dtype;
  FastDiv by_T;     // where N < 2^31
};

struct Token {
  int64_t b, t;
  bool valid;
};

template <int L>
__device__ __forceinline__ Token token_of(const Shape& sh, int64_t group) {
  const int64_t n = group * (32 / L) + (threadIdx.x & 31) / L;
  Token k;
  k.valid = n < sh.N;
  k.b = !k.valid ? 0 : sh.N <= INT32_MAX ? (int64_t)sh.by_T.div((uint32_t)n) : n / sh.T;
  k.t = k.valid ? n - k.b * sh.T : 0;
  return k;
}

// A token's position: its index along T, or what `positions` says.
template <int L> struct Where {
  const Tables& tb;
  const Shape& sh;
  using Pos = RawInt;
  __device__ __forceinline__ bool fetch(int64_t group, RawInt& p) const {
    const Token k = token_of<L>(sh, group);
    if (!k.valid || tb.R == 0) return false;
    if (tb.pos_bytes) p.load(tb.pos, tb.pos_bytes, k.b * tb.pos_sb + k.t);
    else p.v.x = (uint32_t)k.t;
    return true;
  }
  __device__ __forceinline__ int64_t get(const RawInt& p) const { return p.get(tb.pos_bytes); }
};

// A warp's units of q or of k.
struct Part {
  bool is_q;
  Units un;
};
__device__ __forceinline__ Part part_of_warp(const Side& q, const Side& k, const Shape& sh) {
  const int64_t warp = (int64_t)blockIdx.x * (kWalkThreads / 32) + (threadIdx.x >> 5);
  const int64_t all = (int64_t)gridDim.x * (kWalkThreads / 32);
  Part p;
  p.is_q = warp < sh.q_warps;
  const Side& sd = p.is_q ? q : k;
  p.un = make_units(p.is_q ? warp : warp - sh.q_warps, p.is_q ? sh.q_warps : all - sh.q_warps, sd.units, sd.H, sd.C,
                    sd.per);
  return p;
}

// Depth of the ring and resident blocks an SM: four forward blocks of 41 KB (16-bit)
// and 128 registers a thread (three of 49 KB for fp32), three backward blocks of at most 65 KB and 168
// registers (at 128 the backward spills), or two with a deeper ring: see bwd_blocks().
template <typename E> constexpr int kFwdRing = sizeof(E) == 4 ? 6 : 10;
template <typename E, int Blocks> constexpr int kBwdRing = sizeof(E) == 4 ? 4 : Blocks == 2 ? 9 : 6;
template <typename E> constexpr int kFwdBlocks = sizeof(E) == 4 ? 3 : 4;
constexpr int kBwdBlocks = 3;  // at most

// ---- forward ----------------------------------------------------------------

template <typename E, int L, bool Partial>
__global__ void __launch_bounds__(kWalkThreads, kFwdBlocks<E>)
    qk_norm_rope_fwd(Side q, Side k, Tables tb, Shape sh) {
  extern __shared__ __align__(16) uint4 ring[];
  const Part part = part_of_warp(q, k, sh);
  if (part.un.count == 0) return;
  const Side& sd = part.is_q ? q : k;
  const Lane ln = lane_of<E, L>(tb);
  const Where<L> where{tb, sh};
  Angles<E, Where<L>> ang(tb, ln, &g_bad_positions, part.un, where);
  Map map;
  E* y = nullptr;  // the row that comes next
  bool on = false;
  walk_rows<E, 1, kFwdRing<E>>(
      part.un, ln, ring,
      [&](int64_t g) {
        const Token tk = token_of<L>(sh, g);
        return Source<E, 1>{{static_cast<const E*>(sd.x) + tk.b * sd.xb + tk.t * sd.xt}, {sd.xh},
                            ln.active && tk.valid};
      },
      [&]() { ang.begin(); },
      [&](int64_t g, int h) {
        float2 c[4], s[4], w1[4], w2[4];
        load_weights<E>(sd.w, sh.w_dtype, ln, w1, w2);
        ang.enter(c, s);
        map.make(c, s, w1, w2);
        const Token tk = token_of<L>(sh, g);
        on = ln.active && tk.valid;
        y = static_cast<E*>(sd.y) + tk.b * sd.yb + tk.t * sd.yt + h * sd.yh + ln.o1;
      },
      [&](Raw8<E> (&rows)[2]) {
        norm_rope<E, L, Partial>(tb, ln, map, rows[0], rows[1]);
        if (on && SA_DCHECK(ln.o2 + ln.ps + 4 <= tb.D)) {
          rows[0].store(y, ln.ps);
          rows[1].store(y + (ln.o2 - ln.o1), ln.ps);
        }
        y += sd.yh;
      });
}

// ---- backward ---------------------------------------------------------------

// part_sums: [2][gridDim.x][D] fp32 (q's rows, then k's), or null without dw.
template <typename E, int L, int Blocks, bool Partial>
__global__ void __launch_bounds__(kWalkThreads, Blocks)
    qk_norm_rope_bwd(Side q, Side k, Tables tb, Shape sh, float* part_sums) {
  extern __shared__ __align__(16) uint4 ring[];
  const Part part = part_of_warp(q, k, sh);
  const Side& sd = part.is_q ? q : k;
  const Lane ln = lane_of<E, L>(tb);
  const Where<L> where{tb, sh};
  Angles<E, Where<L>> ang(tb, ln, &g_bad_positions, part.un, where);
  float2 c[4], s[4], w1[4], w2[4], dw1[4], dw2[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) dw1[i] = dw2[i] = splat(0.f);
  load_weights<E>(sd.w, sh.w_dtype, ln, w1, w2);
  E* dx = nullptr;  // the row that comes next
  bool on = false;
  // A row that does not exist is zeros: without eps its root would be infinite and 0 * inf reach dw.
  // (Set once a unit: a select at each row's root cost [4, 32 + 8, 4096, 128] 0.5 of 87.5 us.)
  float eps = 1.f;
  walk_rows<E, 2, kBwdRing<E, Blocks>>(
      part.un, ln, ring,
      [&](int64_t g) {
        const Token tk = token_of<L>(sh, g);
        return Source<E, 2>{{static_cast<const E*>(sd.x) + tk.b * sd.xb + tk.t * sd.xt,
                             static_cast<const E*>(sd.dy) + tk.b * sd.gb + tk.t * sd.gt},
                            {sd.xh, sd.gh},
                            ln.active && tk.valid};
      },
      [&]() { ang.begin(); },
      [&](int64_t g, int h) {
        ang.enter(c, s);
        const Token tk = token_of<L>(sh, g);
        on = ln.active && tk.valid;
        eps = on ? tb.eps : 1.f;
        dx = static_cast<E*>(sd.y) + tk.b * sd.yb + tk.t * sd.yt + h * sd.yh + ln.o1;
      },
      [&](Raw8<E> (&rows)[4]) {
        float2 x1[4], x2[4], g1[4], g2[4];  // g becomes dn
        rows[0].get(x1);
        rows[1].get(x2);
        rows[2].get(g1);
        rows[3].get(g2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float2 t1 = fmul2(g2[i], s[i]), t2 = fmul2(g1[i], s[i]);
          if constexpr (Partial) t1 = pair_only(ln, t1, -0.f), t2 = pair_only(ln, t2, 0.f);
          const float2 n1 = ffma2(g1[i], c[i], t1);
          g2[i] = fsub2(fmul2(g2[i], c[i]), t2);
          g1[i] = n1;
        }
        if (tb.normalize) {
          float2 ss = fmul2(x1[0], x1[0]), gx = splat(0.f), v1[4], v2[4];  // v: dn w
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (i) ss = ffma2(x1[i], x1[i], ss);
            ss = ffma2(x2[i], x2[i], ss);
            v1[i] = fmul2(g1[i], w1[i]);
            v2[i] = fmul2(g2[i], w2[i]);
            gx = ffma2(v1[i], x1[i], gx);
            gx = ffma2(v2[i], x2[i], gx);
          }
          const float sum = row_sum<L>(ss.x + ss.y), dot = row_sum<L>(gx.x + gx.y);
          const float r = rsqrtf(fmaf(sum, tb.inv_d, eps));
          const float2 r2 = splat(r), m2 = splat(-(dot * tb.inv_d) * r * r * r);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            dw1[i] = ffma2(g1[i], fmul2(x1[i], r2), dw1[i]);
            dw2[i] = ffma2(g2[i], fmul2(x2[i], r2), dw2[i]);
            g1[i] = ffma2(x1[i], m2, fmul2(v1[i], r2));
            g2[i] = ffma2(x2[i], m2, fmul2(v2[i], r2));
          }
        }
        if (on && SA_DCHECK(ln.o2 + ln.ps + 4 <= tb.D)) {
          rows[2].set(g1);
          rows[3].set(g2);
          rows[2].store(dx, ln.ps);
          rows[3].store(dx + (ln.o2 - ln.o1), ln.ps);
        }
        dx += sd.yh;
      });
  if (part_sums == nullptr) return;
  // lanes that hold the same channels (one per token of the group), then the block's warps of one side
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int m = L; m < 32; m <<= 1) {
      dw1[i].x += __shfl_xor_sync(0xffffffffu, dw1[i].x, m);
      dw1[i].y += __shfl_xor_sync(0xffffffffu, dw1[i].y, m);
      dw2[i].x += __shfl_xor_sync(0xffffffffu, dw2[i].x, m);
      dw2[i].y += __shfl_xor_sync(0xffffffffu, dw2[i].y, m);
    }
  }
  constexpr int W = kWalkThreads / 32;
  float* red = reinterpret_cast<float*>(ring);  // [W][D]; every warp's copies have landed and been read
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();
  if (lane < L && ln.active) {
    float* to = red + warp * tb.D;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = i / 2 * ln.ps + i % 2 * 2;
      *reinterpret_cast<float2*>(to + ln.o1 + d) = dw1[i];
      *reinterpret_cast<float2*>(to + ln.o2 + d) = dw2[i];
    }
  }
  __syncthreads();
  const int64_t w0 = (int64_t)blockIdx.x * W;
  for (int d = threadIdx.x; d < tb.D; d += kWalkThreads) {
    float vq = 0.f, vk = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w0 + w < sh.q_warps) vq += red[w * tb.D + d];
      else vk += red[w * tb.D + d];
    }
    part_sums[(int64_t)blockIdx.x * tb.D + d] = vq;
    part_sums[((int64_t)gridDim.x + blockIdx.x) * tb.D + d] = vk;
  }
}

__device__ __forceinline__ void store_any(void* p, int at, int dtype, float v) {
  if (dtype == SA_F32)
    static_cast<float*>(p)[at] = v;
  else if (dtype == SA_BF16)
    static_cast<__nv_bfloat16*>(p)[at] = from_f<__nv_bfloat16>(v);
  else
    static_cast<__half*>(p)[at] = from_f<__half>(v);
}

// Adds the blocks' partial rows: one block per 32 channels of one side, 32
// threads along the rows, joined in a fixed order.
__global__ void __launch_bounds__(1024) qk_dw_sum(const float* part_sums, void* dwq, void* dwk, int w_dtype, int D,
                                                  int blocks) {
  __shared__ float red[32][33];
  void* out = blockIdx.y == 0 ? dwq : dwk;
  if (out == nullptr) return;
  const float* part = part_sums + (int64_t)blockIdx.y * blocks * D;
  const int col = threadIdx.x & 31, row = threadIdx.x >> 5, d = blockIdx.x * 32 + col;
  float v = 0.f;
  if (d < D) {
#pragma unroll 8
    for (int r = row; r < blocks; r += 32) v += __ldg(part + (int64_t)r * D + d);
  }
  red[row][col] = v;
  __syncthreads();
  // transposed: warp `row` now sums column `row` over its 32 lanes
  v = red[col][row];
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  const int dd = blockIdx.x * 32 + row;
  if (col == 0 && dd < D) store_any(out, dd, w_dtype, v);
}

// ---- host side ----------------------------------------------------------------

static int check_rows(const void* p, const int64_t* s, int esize) {
  if (!p || !s) return SA_ERR_ARG;
  if (!al16(p) || s[3] != 1) return SA_ERR_ALIGN;
  for (int i = 0; i < 3; ++i)
    if ((s[i] * esize) % 16 != 0) return SA_ERR_ALIGN;
  return SA_OK;
}

static int check_shape(int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t D, int dtype) {
  if (B < 0 || Hq < 0 || Hkv < 0 || T < 0 || D <= 0) return SA_ERR_ARG;
  if (dtype != SA_F32 && dtype != SA_F16 && dtype != SA_BF16) return SA_ERR_UNSUPPORTED;
  if (Hq > (1 << 20) || Hkv > (1 << 20) || B > INT32_MAX || T > INT32_MAX || (T > 0 && B > ((int64_t)1 << 33) / T))
    return SA_ERR_UNSUPPORTED;
  return SA_OK;
}

static Side side_of(const void* x, void* y, const void* dy, const void* w, int64_t H, const int64_t* xs,
                    const int64_t* ys, const int64_t* gs, int64_t groups, int C) {
  Side s{};
  s.x = x, s.y = y, s.dy = dy, s.w = w;
  s.H = (int)H, s.C = C, s.per = (int)((H + C - 1) / C);
  s.units = groups * s.per;
  if (H == 0) return s;
  s.xb = xs[0], s.xh = xs[1], s.xt = xs[2];
  s.yb = ys[0], s.yh = ys[1], s.yt = ys[2];
  if (gs) s.gb = gs[0], s.gh = gs[1], s.gt = gs[2];
  return s;
}

static int64_t groups_of(int64_t N, int64_t D) {
  const int64_t per = 32 / lanes_for(D);
  return (N + per - 1) / per;
}

// Blocks, and the warps of q by its share of the work: at least one for each side that has any.
static int64_t plan(const Side& q, const Side& k, Shape* sh, int per_sm) {
  const int64_t blocks = walk_blocks(q.units + k.units, per_sm), warps = blocks * (kWalkThreads / 32);
  if (blocks == 0) return 0;
  const double cq = walk_cost(q.per ? q.units / q.per * q.H : 0, q.units);
  const double ck = walk_cost(k.per ? k.units / k.per * k.H : 0, k.units);
  sh->q_warps = (int64_t)((double)warps * cq / (cq + ck) + 0.5);
  if (q.units) sh->q_warps = std::max<int64_t>(1, sh->q_warps);
  if (k.units) sh->q_warps = std::min(sh->q_warps, warps - 1);  // (four warps a block: one is left)
  return blocks;
}

template <typename E, int L, bool Partial>
static int launch_fwd_lp(const Side& q, const Side& k, const Tables& tb, const Shape& sh, int64_t blocks,
                        cudaStream_t st) {
  constexpr int smem = Ring<E, 1, kFwdRing<E>>::kBytesPerThread * kWalkThreads;
  static_assert(smem <= 56 * 1024, "four blocks an SM");
  const int rc = sa_record_cuda_error(opt_in_once<&qk_norm_rope_fwd<E, L, Partial>, smem>());
  if (rc != SA_OK) return rc;
  qk_norm_rope_fwd<E, L, Partial><<<(unsigned)blocks, kWalkThreads, smem, st>>>(q, k, tb, sh);
  return sa_record_cuda_error(cudaGetLastError());
}

template <typename E, int L>
static int launch_fwd_l(const Side& q, const Side& k, const Tables& tb, const Shape& sh, int64_t blocks,
                        cudaStream_t st) {
  return tb.R < tb.D ? launch_fwd_lp<E, L, true>(q, k, tb, sh, blocks, st)
                     : launch_fwd_lp<E, L, false>(q, k, tb, sh, blocks, st);
}

template <typename E>
static int launch_fwd(const Side& q, const Side& k, const Tables& tb, const Shape& sh, int64_t blocks,
                      cudaStream_t st) {
  switch (lanes_for(tb.D)) {
    case 1: return launch_fwd_l<E, 1>(q, k, tb, sh, blocks, st);
    case 2: return launch_fwd_l<E, 2>(q, k, tb, sh, blocks, st);
    case 4: return launch_fwd_l<E, 4>(q, k, tb, sh, blocks, st);
    case 8: return launch_fwd_l<E, 8>(q, k, tb, sh, blocks, st);
    default: return launch_fwd_l<E, 16>(q, k, tb, sh, blocks, st);
  }
}

// Blocks an SM of the backward pass.  Many whole 16-bit rows in full units are bound by
// DRAM, and fewer warps that ask further ahead serve it better: [4, 32 + 8, 4096, 128] in
// bf16 takes 84 us with two blocks of nine stages, 88-91 with three of six;
// [4, 64 + 16, 4096, 64] 83-86 and 88-94; 16 + 16 heads of 128 70 and 72; 32 + 4 81 and 82.
// Where instructions or the last round bind it, the third block's warps count: D = 80
// (five lanes of eight) 79 with two and 72 with three; units of 6 heads (6 + 6 heads) 58 and
// 53; 7 + 1 heads 49 and 46; 4 units a warp ([4, 32 + 8, 1024, 128]) 26 and 24 (8 units:
// equal); D = 256 90 and 87.  D = 32 and fp32 rows: equal.
static int bwd_blocks(const Side& q, const Side& k, int64_t D, int dtype) {
  const int64_t warps = 2 * (int64_t)sm_count() * (kWalkThreads / 32);
  const bool full = q.H + k.H >= 7 * (q.per + k.per), many = q.units + k.units >= 8 * warps;
  return dtype != SA_F32 && (D == 64 || D == 128) && full && many ? 2 : kBwdBlocks;
}

template <typename E, int L, int Blocks, bool Partial>
static int launch_bwd_lbp(const Side& q, const Side& k, const Tables& tb, const Shape& sh, float* part, int64_t blocks,
                         cudaStream_t st) {
  constexpr int smem = Ring<E, 2, kBwdRing<E, Blocks>>::kBytesPerThread * kWalkThreads;
  static_assert(smem >= kWalkThreads / 32 * 256 * 4, "the block's dw sums");
  static_assert(Blocks * (smem + 1024) <= 227 * 1024, "the blocks of an SM");
  const int rc = sa_record_cuda_error(opt_in_once<&qk_norm_rope_bwd<E, L, Blocks, Partial>, smem>());
  if (rc != SA_OK) return rc;
  qk_norm_rope_bwd<E, L, Blocks, Partial><<<(unsigned)blocks, kWalkThreads, smem, st>>>(q, k, tb, sh, part);
  return sa_record_cuda_error(cudaGetLastError());
}

template <typename E, int L, int Blocks>
static int launch_bwd_lb(const Side& q, const Side& k, const Tables& tb, const Shape& sh, float* part, int64_t blocks,
                         cudaStream_t st) {
  return tb.R < tb.D ? launch_bwd_lbp<E, L, Blocks, true>(q, k, tb, sh, part, blocks, st)
                     : launch_bwd_lbp<E, L, Blocks, false>(q, k, tb, sh, part, blocks, st);
}

template <typename E, int L>
static int launch_bwd_l(const Side& q, const Side& k, const Tables& tb, const Shape& sh, float* part, int64_t blocks,
                        int per_sm, cudaStream_t st) {
  if constexpr (sizeof(E) == 2 && (L == 4 || L == 8)) {
    if (per_sm == 2) return launch_bwd_lb<E, L, 2>(q, k, tb, sh, part, blocks, st);
  }
  return launch_bwd_lb<E, L, kBwdBlocks>(q, k, tb, sh, part, blocks, st);
}

template <typename E>
static int launch_bwd(const Side& q, const Side& k, const Tables& tb, const Shape& sh, float* part, int64_t blocks,
                      int per_sm, cudaStream_t st) {
  switch (lanes_for(tb.D)) {
    case 1: return launch_bwd_l<E, 1>(q, k, tb, sh, part, blocks, per_sm, st);
    case 2: return launch_bwd_l<E, 2>(q, k, tb, sh, part, blocks, per_sm, st);
    case 4: return launch_bwd_l<E, 4>(q, k, tb, sh, part, blocks, per_sm, st);
    case 8: return launch_bwd_l<E, 8>(q, k, tb, sh, part, blocks, per_sm, st);
    default: return launch_bwd_l<E, 16>(q, k, tb, sh, part, blocks, per_sm, st);
  }
}

}  // namespace qkr

int qk_bad_positions(int reset, cudaStream_t st) {
  unsigned v = 0;
  cudaMemcpyFromSymbolAsync(&v, qkr::g_bad_positions, sizeof(v), 0, cudaMemcpyDeviceToHost, st);
  cudaStreamSynchronize(st);
  if (reset) {
    const unsigned z = 0;
    cudaMemcpyToSymbolAsync(qkr::g_bad_positions, &z, sizeof(z), 0, cudaMemcpyHostToDevice, st);
    cudaStreamSynchronize(st);
  }
  return (int)v;
}

}  // namespace sa

extern "C" int sa_qk_norm_rope(const void* q, const void* k, void* q_out, void* k_out, const void* q_weight,
                               const void* k_weight, int w_dtype, const void* cos_table, const void* sin_table,
                               int cs_dtype, const void* positions, int pos_bytes, int64_t pos_batch_stride,
                               int64_t num_pos, int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t D,
                               int64_t rotary_dim, const int64_t* q_strides, const int64_t* k_strides,
                               const int64_t* qo_strides, const int64_t* ko_strides, float eps, int normalize,
                               int dtype, void* stream) {
  using namespace sa::qkr;
  int rc = check_shape(B, Hq, Hkv, T, D, dtype);
  if (rc != SA_OK) return rc;
  Tables tb;
  rc = make_tables(&tb, cos_table, sin_table, cs_dtype, positions, pos_bytes, pos_batch_stride, num_pos, T, D,
                   rotary_dim, eps, normalize, q_weight, k_weight, w_dtype);
  if (rc != SA_OK) return rc;
  if (B == 0 || T == 0 || Hq + Hkv == 0) return SA_OK;
  const int es = dtype == SA_F32 ? 4 : 2;
  if (Hq > 0 && ((rc = check_rows(q, q_strides, es)) != SA_OK || (rc = check_rows(q_out, qo_strides, es)) != SA_OK))
    return rc;
  if (Hkv > 0 && ((rc = check_rows(k, k_strides, es)) != SA_OK || (rc = check_rows(k_out, ko_strides, es)) != SA_OK))
    return rc;
  if (!normalize) q_weight = k_weight = nullptr;  // n = x
  const int64_t groups = groups_of(B * T, D);
  const int per_sm = dtype == SA_F32 ? kFwdBlocks<float> : kFwdBlocks<__half>;
  const int C = unit_heads(groups * (Hq + Hkv), (int64_t)per_sm * sm_count() * (kWalkThreads / 32));
  const Side a = side_of(q, q_out, nullptr, q_weight, Hq, q_strides, qo_strides, nullptr, groups, C);
  const Side b = side_of(k, k_out, nullptr, k_weight, Hkv, k_strides, ko_strides, nullptr, groups, C);
  Shape sh{B * T, T, 0, w_dtype, FastDiv((uint32_t)T)};
  const int64_t blocks = plan(a, b, &sh, per_sm);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == SA_F32) return launch_fwd<float>(a, b, tb, sh, blocks, st);
  if (dtype == SA_BF16) return launch_fwd<__nv_bfloat16>(a, b, tb, sh, blocks, st);
  return launch_fwd<__half>(a, b, tb, sh, blocks, st);
}

extern "C" int64_t sa_qk_norm_rope_bwd_workspace_size(int64_t D) {
  if (D <= 0 || D > 256) return SA_ERR_UNSUPPORTED;
  return 2ll * sa::qkr::kBwdBlocks * sa::qkr::sm_count() * D * 4;
}

extern "C" int sa_qk_norm_rope_bwd(const void* q, const void* k, const void* dq_out, const void* dk_out, void* dq,
                                   void* dk, const void* q_weight, const void* k_weight, int w_dtype,
                                   void* dq_weight, void* dk_weight, const void* cos_table, const void* sin_table,
                                   int cs_dtype, const void* positions, int pos_bytes, int64_t pos_batch_stride,
                                   int64_t num_pos, void* workspace, int64_t workspace_bytes, int64_t B, int64_t Hq,
                                   int64_t Hkv, int64_t T, int64_t D, int64_t rotary_dim, const int64_t* q_strides,
                                   const int64_t* k_strides, const int64_t* dqo_strides, const int64_t* dko_strides,
                                   const int64_t* dq_strides, const int64_t* dk_strides, float eps, int normalize,
                                   int dtype, void* stream) {
  using namespace sa::qkr;
  int rc = check_shape(B, Hq, Hkv, T, D, dtype);
  if (rc != SA_OK) return rc;
  Tables tb;
  rc = make_tables(&tb, cos_table, sin_table, cs_dtype, positions, pos_bytes, pos_batch_stride, num_pos, T, D,
                   rotary_dim, eps, normalize, q_weight, k_weight, w_dtype);
  if (rc != SA_OK) return rc;
  const bool dw = dq_weight != nullptr || dk_weight != nullptr;
  if (dw) {
    if (!normalize || (dq_weight && !q_weight) || (dk_weight && !k_weight)) return SA_ERR_ARG;
    if (!workspace || workspace_bytes < sa_qk_norm_rope_bwd_workspace_size(D)) return SA_ERR_ARG;
    if (!al16(workspace)) return SA_ERR_ALIGN;
  }
  const int es = dtype == SA_F32 ? 4 : 2;
  const bool work = B > 0 && T > 0;
  const int64_t hq = work ? Hq : 0, hk = work ? Hkv : 0;
  if (hq > 0 && ((rc = check_rows(q, q_strides, es)) != SA_OK || (rc = check_rows(dq_out, dqo_strides, es)) != SA_OK ||
                 (rc = check_rows(dq, dq_strides, es)) != SA_OK))
    return rc;
  if (hk > 0 && ((rc = check_rows(k, k_strides, es)) != SA_OK || (rc = check_rows(dk_out, dko_strides, es)) != SA_OK ||
                 (rc = check_rows(dk, dk_strides, es)) != SA_OK))
    return rc;
  if (!normalize) q_weight = k_weight = nullptr;  // n = x
  const int64_t groups = work ? groups_of(B * T, D) : 0;
  const int C = unit_heads(groups * (hq + hk), (int64_t)kBwdBlocks * sm_count() * (kWalkThreads / 32));
  const Side a = side_of(q, dq, dq_out, q_weight, hq, q_strides, dq_strides, dqo_strides, groups, C);
  const Side b = side_of(k, dk, dk_out, k_weight, hk, k_strides, dk_strides, dko_strides, groups, C);
  Shape sh{B * T, work ? T : 1, 0, w_dtype, FastDiv(work ? (uint32_t)T : 1u)};
  const int per_sm = bwd_blocks(a, b, D, dtype);
  const int64_t blocks = plan(a, b, &sh, per_sm);
  float* part = dw ? static_cast<float*>(workspace) : nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (blocks > 0) {
    rc = dtype == SA_F32    ? launch_bwd<float>(a, b, tb, sh, part, blocks, per_sm, st)
         : dtype == SA_BF16 ? launch_bwd<__nv_bfloat16>(a, b, tb, sh, part, blocks, per_sm, st)
                            : launch_bwd<__half>(a, b, tb, sh, part, blocks, per_sm, st);
    if (rc != SA_OK) return rc;
  }
  if (dw) {  // also without rows: zeros
    qk_dw_sum<<<dim3((unsigned)((D + 31) / 32), 2), 1024, 0, st>>>(part, dq_weight, dk_weight, w_dtype, (int)D,
                                                                   (int)blocks);
    rc = sa_record_cuda_error(cudaGetLastError());
  }
  return rc;
}
SA_BOUNDS_ACCESSOR(qk_norm_rope_bounds)
