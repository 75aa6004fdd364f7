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
// Bound: HBM.  Forward reads x and writes y; backward reads x and dy and
// writes dx.  A warp owns 32 / L neighbouring tokens (L lanes a row) and walks
// over some of their heads, so a token's cos / sin stay in registers for all
// of them.  dw: every lane keeps fp32 sums of its own 16 channels over the
// rows it meets, a block adds its warps' sums in a fixed order and writes one
// row of partial sums, and a second small kernel adds those in a fixed order:
// no atomics, bitwise the same from run to run.
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

constexpr int kWarps = 8;

struct Side {
  const void* x;
  void* y;          // forward: y; backward: dx
  const void* dy;   // backward
  const void* w;    // nullable
  int64_t xb, xh, xt, yb, yh, yt, gb, gh, gt;  // element strides
  int H, hc, chunks;  // heads, heads a warp takes, ceil(H / hc)
};

struct Shape {
  int64_t N, T;     // B * T tokens
  int64_t groups;   // of 32 / L tokens
  int w_dtype;
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
  k.b = k.valid ? n / sh.T : 0;
  k.t = k.valid ? n - k.b * sh.T : 0;
  return k;
}

__device__ __forceinline__ int64_t pos_of(const Tables& tb, const Token& k) {
  return tb.pos_bytes ? read_pos(tb.pos, tb.pos_bytes, k.b * tb.pos_sb + k.t) : k.t;
}

// ---- forward ----------------------------------------------------------------

template <typename E, int L>
__global__ void __launch_bounds__(kWarps * 32) qk_norm_rope_fwd(Side q, Side k, Tables tb, Shape sh) {
  const int per = q.chunks + k.chunks;
  const int64_t task = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (task >= sh.groups * per) return;  // the whole warp
  const int64_t group = task / per;
  int chunk = (int)(task - group * per);
  const bool is_q = chunk < q.chunks;
  const Side& sd = is_q ? q : k;
  if (!is_q) chunk -= q.chunks;

  const Lane ln = lane_of<L>(tb);
  const Token tk = token_of<L>(sh, group);
  const bool on = ln.active && tk.valid;
  float c[8], s[8], w1[8], w2[8];
  Lane la = ln;
  la.active = on;
  load_angles(tb, la, pos_of(tb, tk), &g_bad_positions, c, s);
  load_weights(sd.w, sh.w_dtype, la, w1, w2);
  const E* x = static_cast<const E*>(sd.x) + tk.b * sd.xb + tk.t * sd.xt;
  E* y = static_cast<E*>(sd.y) + tk.b * sd.yb + tk.t * sd.yt;
  const int h0 = chunk * sd.hc, h1 = min(sd.H, h0 + sd.hc);
  constexpr int U = 4;  // heads in flight
  for (int h = h0; h < h1; h += U) {
    Raw8<E> a[U], b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (on && h + u < h1) {
        a[u].load(x + (h + u) * sd.xh + ln.o1);
        b[u].load(x + (h + u) * sd.xh + ln.o2);
      } else {
        a[u].zero();
        b[u].zero();
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (h + u >= h1) break;  // uniform over the warp
      norm_rope<E, L>(tb, a[u], b[u], w1, w2, c, s);
      if (on && SA_DCHECK(tk.t < sh.T && h + u < sd.H && ln.o2 + 8 <= tb.D)) {
        a[u].store(y + (h + u) * sd.yh + ln.o1);
        b[u].store(y + (h + u) * sd.yh + ln.o2);
      }
    }
  }
}

// ---- backward ---------------------------------------------------------------

// Blocks [0, q_blocks) walk over q's tasks, the others over k's, so a lane
// keeps one set of dw sums.  part: [gridDim.x][D] fp32, or null without dw.
template <typename E, int L>
__global__ void __launch_bounds__(kWarps * 32, 2)
    qk_norm_rope_bwd(Side q, Side k, Tables tb, Shape sh, float* part, int q_blocks) {
  extern __shared__ float red[];  // [kWarps][D]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool is_q = (int)blockIdx.x < q_blocks;
  const Side& sd = is_q ? q : k;
  const int64_t first = (int64_t)(is_q ? blockIdx.x : blockIdx.x - q_blocks) * kWarps + warp;
  const int64_t step = (int64_t)(is_q ? q_blocks : gridDim.x - q_blocks) * kWarps;
  const Lane ln = lane_of<L>(tb);
  float w1[8], w2[8], dw1[8], dw2[8];
  load_weights(sd.w, sh.w_dtype, ln, w1, w2);
#pragma unroll
  for (int i = 0; i < 8; ++i) dw1[i] = dw2[i] = 0.f;

  const int64_t tasks = sh.groups * sd.chunks;
  for (int64_t task = first; task < tasks; task += step) {
    const int64_t group = task / sd.chunks;
    const int chunk = (int)(task - group * sd.chunks);
    const Token tk = token_of<L>(sh, group);
    const bool on = ln.active && tk.valid;
    float c[8], s[8];
    Lane la = ln;
    la.active = on;
    load_angles(tb, la, pos_of(tb, tk), &g_bad_positions, c, s);
    const E* x = static_cast<const E*>(sd.x) + tk.b * sd.xb + tk.t * sd.xt;
    const E* dy = static_cast<const E*>(sd.dy) + tk.b * sd.gb + tk.t * sd.gt;
    E* dx = static_cast<E*>(sd.y) + tk.b * sd.yb + tk.t * sd.yt;
    const int h0 = chunk * sd.hc, h1 = min(sd.H, h0 + sd.hc);
    constexpr int U = sizeof(E) == 4 ? 1 : 2;
    for (int h = h0; h < h1; h += U) {
      Raw8<E> xa[U], xb[U], ga[U], gb[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (on && h + u < h1) {
          xa[u].load(x + (h + u) * sd.xh + ln.o1);
          xb[u].load(x + (h + u) * sd.xh + ln.o2);
          ga[u].load(dy + (h + u) * sd.gh + ln.o1);
          gb[u].load(dy + (h + u) * sd.gh + ln.o2);
        } else {
          xa[u].zero(), xb[u].zero(), ga[u].zero(), gb[u].zero();
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (h + u >= h1) break;  // uniform over the warp
        float x1[8], x2[8], g1[8], g2[8];
        xa[u].get(x1);
        xb[u].get(x2);
        ga[u].get(g1);
        gb[u].get(g2);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float n1 = g1[i] * c[i] + g2[i] * s[i], n2 = g2[i] * c[i] - g1[i] * s[i];
          g1[i] = n1, g2[i] = n2;
        }
        if (tb.normalize) {
          float ss = 0.f, gx = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            ss = fmaf(x1[i], x1[i], ss);
            ss = fmaf(x2[i], x2[i], ss);
            gx = fmaf(g1[i] * w1[i], x1[i], gx);
            gx = fmaf(g2[i] * w2[i], x2[i], gx);
          }
          ss = row_sum<L>(ss);
          gx = row_sum<L>(gx);
          const float r = rsqrtf(fmaf(ss, tb.inv_d, tb.eps));
          const float m = gx * tb.inv_d * r * r;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            dw1[i] = fmaf(g1[i], x1[i] * r, dw1[i]);
            dw2[i] = fmaf(g2[i], x2[i] * r, dw2[i]);
            g1[i] = r * (g1[i] * w1[i] - x1[i] * m);
            g2[i] = r * (g2[i] * w2[i] - x2[i] * m);
          }
        }
        if (on && SA_DCHECK(tk.t < sh.T && h + u < sd.H && ln.o2 + 8 <= tb.D)) {
          ga[u].set(g1);
          gb[u].set(g2);
          ga[u].store(dx + (h + u) * sd.yh + ln.o1);
          gb[u].store(dx + (h + u) * sd.yh + ln.o2);
        }
      }
    }
  }
  if (part == nullptr) return;
  // lanes that hold the same channels (one per token of the warp), then warps
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int m = L; m < 32; m <<= 1) {
      dw1[i] += __shfl_xor_sync(0xffffffffu, dw1[i], m);
      dw2[i] += __shfl_xor_sync(0xffffffffu, dw2[i], m);
    }
  }
  if (lane < L && ln.active) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      red[warp * tb.D + ln.o1 + i] = dw1[i];
      red[warp * tb.D + ln.o2 + i] = dw2[i];
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < tb.D; d += kWarps * 32) {
    float v = 0.f;
#pragma unroll
    for (int wi = 0; wi < kWarps; ++wi) v += red[wi * tb.D + d];
    part[(int64_t)blockIdx.x * tb.D + d] = v;
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
__global__ void __launch_bounds__(1024) qk_dw_sum(const float* part, void* dwq, void* dwk, int w_dtype, int D,
                                                  int q_blocks, int blocks) {
  __shared__ float red[32][33];
  const bool is_q = blockIdx.y == 0;
  void* out = is_q ? dwq : dwk;
  if (out == nullptr) return;
  const int col = threadIdx.x & 31, row = threadIdx.x >> 5, d = blockIdx.x * 32 + col;
  const int lo = is_q ? 0 : q_blocks, hi = is_q ? q_blocks : blocks;
  float v = 0.f;
  if (d < D)
    for (int r = lo + row; r < hi; r += 32) v += part[(int64_t)r * D + d];
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

static int sm_count() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
    cudaGetLastError();
    n = 148;
  }
  return n;
}

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
                    const int64_t* ys, const int64_t* gs, int hc) {
  Side s;
  s.x = x, s.y = y, s.dy = dy, s.w = w;
  s.xb = xs[0], s.xh = xs[1], s.xt = xs[2];
  s.yb = ys[0], s.yh = ys[1], s.yt = ys[2];
  s.gb = gs ? gs[0] : 0, s.gh = gs ? gs[1] : 0, s.gt = gs ? gs[2] : 0;
  s.H = (int)H, s.hc = hc, s.chunks = (int)((H + hc - 1) / hc);
  return s;
}

static Shape shape_of(int64_t B, int64_t T, int64_t D, int w_dtype) {
  Shape sh;
  sh.N = B * T, sh.T = T, sh.w_dtype = w_dtype;
  const int per = 32 / lanes_for(D);
  sh.groups = (sh.N + per - 1) / per;
  return sh;
}

template <typename E>
static int launch_fwd(const Side& q, const Side& k, const Tables& tb, const Shape& sh, cudaStream_t st) {
  const int64_t tasks = sh.groups * (q.chunks + k.chunks), blocks = (tasks + kWarps - 1) / kWarps;
  if (blocks > INT32_MAX) return SA_ERR_UNSUPPORTED;
  switch (lanes_for(tb.D)) {
    case 1: qk_norm_rope_fwd<E, 1><<<(unsigned)blocks, kWarps * 32, 0, st>>>(q, k, tb, sh); break;
    case 2: qk_norm_rope_fwd<E, 2><<<(unsigned)blocks, kWarps * 32, 0, st>>>(q, k, tb, sh); break;
    case 4: qk_norm_rope_fwd<E, 4><<<(unsigned)blocks, kWarps * 32, 0, st>>>(q, k, tb, sh); break;
    case 8: qk_norm_rope_fwd<E, 8><<<(unsigned)blocks, kWarps * 32, 0, st>>>(q, k, tb, sh); break;
    default: qk_norm_rope_fwd<E, 16><<<(unsigned)blocks, kWarps * 32, 0, st>>>(q, k, tb, sh); break;
  }
  return sa_record_cuda_error(cudaGetLastError());
}

struct BwdPlan {
  int64_t blocks, q_blocks;
};

// Two resident blocks an SM, split between q and k by their heads.
static BwdPlan plan_bwd(int64_t tasks_q, int64_t tasks_k, int64_t Hq, int64_t Hkv) {
  const int64_t most = 2ll * sm_count();
  const int64_t need_q = (tasks_q + kWarps - 1) / kWarps, need_k = (tasks_k + kWarps - 1) / kWarps;
  BwdPlan p;
  const int64_t share = std::max<int64_t>(1, std::min<int64_t>(most - 1, (most * Hq + (Hq + Hkv) / 2) / std::max<int64_t>(1, Hq + Hkv)));
  p.q_blocks = std::min(need_q, share);
  p.blocks = p.q_blocks + std::min(need_k, most - share);
  return p;
}

template <typename E>
static int launch_bwd(const Side& q, const Side& k, const Tables& tb, const Shape& sh, float* part, const BwdPlan& p,
                      cudaStream_t st) {
  const size_t smem = part ? (size_t)kWarps * tb.D * 4 : 0;  // at most 8 KB
  const unsigned g = (unsigned)p.blocks;
  const int qb = (int)p.q_blocks;
  switch (lanes_for(tb.D)) {
    case 1: qk_norm_rope_bwd<E, 1><<<g, kWarps * 32, smem, st>>>(q, k, tb, sh, part, qb); break;
    case 2: qk_norm_rope_bwd<E, 2><<<g, kWarps * 32, smem, st>>>(q, k, tb, sh, part, qb); break;
    case 4: qk_norm_rope_bwd<E, 4><<<g, kWarps * 32, smem, st>>>(q, k, tb, sh, part, qb); break;
    case 8: qk_norm_rope_bwd<E, 8><<<g, kWarps * 32, smem, st>>>(q, k, tb, sh, part, qb); break;
    default: qk_norm_rope_bwd<E, 16><<<g, kWarps * 32, smem, st>>>(q, k, tb, sh, part, qb); break;
  }
  return sa_record_cuda_error(cudaGetLastError());
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
  const int64_t none[4] = {0, 0, 0, 1};
  if (Hq > 0 && ((rc = check_rows(q, q_strides, es)) != SA_OK || (rc = check_rows(q_out, qo_strides, es)) != SA_OK))
    return rc;
  if (Hkv > 0 && ((rc = check_rows(k, k_strides, es)) != SA_OK || (rc = check_rows(k_out, ko_strides, es)) != SA_OK))
    return rc;
  const Shape sh = shape_of(B, T, D, w_dtype);
  const int hc = heads_per_warp(sh.groups, Hq + Hkv, 16ll * sm_count());
  const Side a = side_of(q, q_out, nullptr, q_weight, Hq, Hq ? q_strides : none, Hq ? qo_strides : none, nullptr, hc);
  const Side b = side_of(k, k_out, nullptr, k_weight, Hkv, Hkv ? k_strides : none, Hkv ? ko_strides : none, nullptr, hc);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == SA_F32) return launch_fwd<float>(a, b, tb, sh, st);
  if (dtype == SA_BF16) return launch_fwd<__nv_bfloat16>(a, b, tb, sh, st);
  return launch_fwd<__half>(a, b, tb, sh, st);
}

extern "C" int64_t sa_qk_norm_rope_bwd_workspace_size(int64_t D) {
  if (D <= 0 || D > 256) return SA_ERR_UNSUPPORTED;
  return 2ll * sa::qkr::sm_count() * D * 4;
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
  const int64_t none[4] = {0, 0, 0, 1};
  const int64_t hq = work ? Hq : 0, hk = work ? Hkv : 0;
  if (hq > 0 && ((rc = check_rows(q, q_strides, es)) != SA_OK || (rc = check_rows(dq_out, dqo_strides, es)) != SA_OK ||
                 (rc = check_rows(dq, dq_strides, es)) != SA_OK))
    return rc;
  if (hk > 0 && ((rc = check_rows(k, k_strides, es)) != SA_OK || (rc = check_rows(dk_out, dko_strides, es)) != SA_OK ||
                 (rc = check_rows(dk, dk_strides, es)) != SA_OK))
    return rc;
  const Shape sh = shape_of(work ? B : 0, work ? T : 1, D, w_dtype);
  const int hc = heads_per_warp(sh.groups, Hq + Hkv, 16ll * sm_count());
  const Side a = side_of(q, dq, dq_out, q_weight, hq, hq ? q_strides : none, hq ? dq_strides : none,
                         hq ? dqo_strides : none, hc);
  const Side b = side_of(k, dk, dk_out, k_weight, hk, hk ? k_strides : none, hk ? dk_strides : none,
                         hk ? dko_strides : none, hc);
  const BwdPlan p = plan_bwd(sh.groups * a.chunks, sh.groups * b.chunks, hq, hk);
  float* part = dw ? static_cast<float*>(workspace) : nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p.blocks > 0) {
    rc = dtype == SA_F32    ? launch_bwd<float>(a, b, tb, sh, part, p, st)
         : dtype == SA_BF16 ? launch_bwd<__nv_bfloat16>(a, b, tb, sh, part, p, st)
                            : launch_bwd<__half>(a, b, tb, sh, part, p, st);
    if (rc != SA_OK) return rc;
  }
  if (dw) {  // also without rows: zeros
    qk_dw_sum<<<dim3((unsigned)((D + 31) / 32), 2), 1024, 0, st>>>(part, dq_weight, dk_weight, w_dtype, (int)D,
                                                                   (int)p.q_blocks, (int)p.blocks);
    rc = sa_record_cuda_error(cudaGetLastError());
  }
  return rc;
}
SA_BOUNDS_ACCESSOR(qk_norm_rope_bounds)
