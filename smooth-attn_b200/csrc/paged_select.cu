// Decode over chosen pages of a paged key-value cache, sm_100a: mean keys of
// full pages, the choice of each sequence's and key head's pages by a cheap
// score, and the attention over these alone.  (No reference counterpart: the
// reference's decode, src/smooth_attn/kernels.py:2681-2829, reads every page.)
//
// Score.  The normaliser of squareplus attention is a plain sum, so a page's
// share of it is the sum of its tokens' weights; the score estimates that at
// the page's mean key, summed over the group's query heads:
//   score(page) = sum_g y(2 scale q_g . mean_key(page) - 1),
//   y(a) = squareplus(a)^2
// A sequence of n pages keeps its last page (the newest tokens; it may be part
// filled and needs no mean) and the num_pages - 1 others of the highest score,
// ties to the lowest page; NaN counts as the highest.  The
// choice hangs on the order of close values, so scores are summed in 64 bits:
// they then do not depend on how the work is cut.
//
// The attention itself is the decode kernel's (paged.cu, paged_tc.cu): seen as
// B * Hkv sequences of one key head over a cache of num_blocks * Hkv pages,
// every key head has a block table of its own.  The chosen pages are written
// in ascending order, so the part-filled page is the last one, and the chosen
// pages' table, the lengths and the decode's tickets are all made on the
// device, without the host.
//
// Bound: the mean keys (1 / block_size of K) and the chosen pages, at HBM's
// rate, for large batches; the chain of three launches for small ones.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "qk_rope.cuh"
#include "smooth_attn_b200.h"

int sa_record_cuda_error(cudaError_t e);

namespace sa {
namespace pgs {

using qkr::Raw8;
using qkr::al16;

static __device__ unsigned g_bad_pages;

// ---- mean keys ------------------------------------------------------------------

struct MeansArgs {
  const void* kc;
  void* means;
  const int32_t* bt;
  const int32_t* cl;
  const int32_t* start;  // nullable: 0
  int64_t num_blocks;
  int Hkv, bs, max_blocks;
};

// One warp: one page of one key head; LPR lanes a row, 32 / LPR rows at once.
template <typename E, int D>
__global__ void __launch_bounds__(256) paged_key_means_kernel(MeansArgs a) {
  constexpr int LPR = D / 8, RPW = 32 / LPR, U = 8;
  const int b = blockIdx.y, lane = threadIdx.x & 31;
  const int64_t cap = (int64_t)a.max_blocks * a.bs;
  const int ctx = (int)max((int64_t)0, min(cap, (int64_t)a.cl[b]));
  const int from = a.start ? max(0, a.start[b]) / a.bs : 0;
  const int64_t n = (int64_t)max(0, ctx / a.bs - from) * a.Hkv;
  for (int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < n; w += (int64_t)gridDim.x * 8) {
    const int j = (int)(w / a.Hkv), h = (int)(w - (int64_t)j * a.Hkv);
    const int64_t page = a.bt[(int64_t)b * a.max_blocks + from + j];
    if (page < 0 || page >= a.num_blocks) {
      if (lane == 0 && h == 0) atomicAdd(&g_bad_pages, 1u);
      continue;
    }
    const E* base = static_cast<const E*>(a.kc) + (page * a.Hkv + h) * a.bs * D + (lane % LPR) * 8;
    float sum[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] = 0.f;
    for (int r0 = lane / LPR; r0 < a.bs; r0 += RPW * U) {
      Raw8<E> x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (r0 + u * RPW < a.bs) x[u].load(base + (int64_t)(r0 + u * RPW) * D);
        else x[u].zero();
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[8];
        x[u].get(f);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += f[i];
      }
    }
    const float inv = 1.0f / (float)a.bs;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int m = LPR; m < 32; m <<= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], m);
      sum[i] *= inv;
    }
    if (lane < LPR) {
      Raw8<E> o;
      o.set(sum);
      o.store(static_cast<E*>(a.means) + (page * a.Hkv + h) * D + lane * 8);
    }
  }
}

// ---- scores ---------------------------------------------------------------------

struct SelectArgs {
  const void* q;       // [B, Hq, D]
  const void* means;   // [num_blocks, Hkv, D]
  const int32_t* bt;
  const int32_t* cl;
  unsigned long long* keys;  // [B * Hkv][max_blocks] scores, in an order that integers keep
  int32_t* pages;            // nullable [B, Hkv, K]: chosen pages of the sequence, ascending, then -1
  int32_t* table;            // nullable [B * Hkv, K]: the same as pages of single heads, physical
  int32_t* lens;             // [B * Hkv] tokens in them
  int32_t* tickets;          // nullable: words to clear for the decode that follows
  int64_t num_blocks, num_tickets;
  double scale2;             // 2 * scale
  int Hkv, G, bs, max_blocks, K;
};

struct Seq {
  int ctx, n;  // tokens, pages
};

__device__ __forceinline__ Seq seq_of(const SelectArgs& a, int b) {
  Seq s;
  s.ctx = (int)max((int64_t)0, min((int64_t)a.max_blocks * a.bs, (int64_t)a.cl[b]));
  s.n = (s.ctx + a.bs - 1) / a.bs;
  return s;
}

// squareplus(a)^2 without the cancellation of negative a, in 64 bits.
__device__ __forceinline__ double weight64(double a) {
  const double root = sqrt(a * a + 4.0);
  const double sp = a < 0 ? 2.0 / (root - a) : 0.5 * (a + root);
  return sp * sp;
}

__device__ __forceinline__ unsigned long long key_of(double score) {
  // scores are not negative, so their bits order as they do; NaN above all
  return isnan(score) ? 0x7ff8000000000000ull : (unsigned long long)__double_as_longlong(score);
}

// One thread: one page; PAGES pages of one key head a block, their mean keys
// staged through shared memory (16 bytes of padding a row: conflict-free),
// the group's queries as doubles beside them, GT heads at a time.
template <typename E, int D, int GT, int PAGES>
__global__ void __launch_bounds__(PAGES) paged_score_kernel(SelectArgs a) {
  constexpr int ROW = D * 2 + 16;
  extern __shared__ __align__(16) uint8_t smem[];
  double* qs = reinterpret_cast<double*>(smem);  // [D][GT]
  uint8_t* rows = smem + (size_t)D * GT * 8;
  const int u = blockIdx.y, b = u / a.Hkv, h = u - b * a.Hkv;
  const Seq s = seq_of(a, b);
  const int m = s.n - 1, p0 = blockIdx.x * PAGES;  // candidates: all but the last
  if (m <= a.K - 1 || p0 >= m) return;             // all of them are taken: nothing to score
  constexpr int LPR = D / 8;
  for (int i = threadIdx.x; i < PAGES * LPR; i += PAGES) {
    const int r = i / LPR, c = i - r * LPR;
    if (p0 + r >= m) break;
    int64_t page = a.bt[(int64_t)b * a.max_blocks + p0 + r];
    if (page < 0 || page >= a.num_blocks) {
      if (c == 0 && h == 0) atomicAdd(&g_bad_pages, 1u);
      page = 0;
    }
    *reinterpret_cast<uint4*>(rows + r * ROW + c * 16) =
        __ldg(reinterpret_cast<const uint4*>(static_cast<const E*>(a.means) + (page * a.Hkv + h) * D) + c);
  }
  double score = 0.0;
  for (int g0 = 0; g0 < a.G; g0 += GT) {
    if (g0) __syncthreads();  // the last group's queries have been read
    const E* q = static_cast<const E*>(a.q) + ((int64_t)u * a.G + g0) * D;
    for (int i = threadIdx.x; i < D * GT; i += PAGES) qs[(i % D) * GT + i / D] = (double)to_f<E>(q[i]);
    __syncthreads();
    double dot[GT];
#pragma unroll
    for (int g = 0; g < GT; ++g) dot[g] = 0.0;
    for (int c = 0; c < LPR; ++c) {
      float f[8];
      unpack<E, 8>(rows + threadIdx.x * ROW + c * 16, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double x = (double)f[e];
#pragma unroll
        for (int g = 0; g < GT; ++g) dot[g] = fma(x, qs[(c * 8 + e) * GT + g], dot[g]);
      }
    }
#pragma unroll
    for (int g = 0; g < GT; ++g) score += weight64(fma(a.scale2, dot[g], -1.0));
  }
  const int p = p0 + threadIdx.x;
  if (p < m && SA_DCHECK(p < a.max_blocks)) a.keys[(int64_t)u * a.max_blocks + p] = key_of(score);
}

// ---- choice ---------------------------------------------------------------------

constexpr int kSelThreads = 512;
constexpr int kBins = 2048;

// One block: one sequence and key head.  The threshold is found by counting
// keys in kBins equal ranges of [lo, hi], which is narrowed to the range that
// holds the last chosen key until all of that range is chosen or it is one
// value; then one ordered pass writes what is chosen.
__global__ void __launch_bounds__(kSelThreads) paged_choose_kernel(SelectArgs a) {
  __shared__ int bins[kBins];
  __shared__ unsigned long long ends[2][kSelThreads / 32];
  __shared__ int warp_sums[kSelThreads / 32];
  __shared__ int found_bin, found_above, found_count;
  const int u = blockIdx.x, b = u / a.Hkv, h = u - b * a.Hkv, tid = threadIdx.x;
  const int lane = tid & 31, warp = tid >> 5, NW = kSelThreads / 32;
  for (int64_t i = (int64_t)u * kSelThreads + tid; i < a.num_tickets; i += (int64_t)gridDim.x * kSelThreads)
    a.tickets[i] = 0;
  const Seq s = seq_of(a, b);
  const int m = s.n - 1, need = min(a.K, s.n) - 1;  // of the m candidates
  const int32_t* bt = a.bt + (int64_t)b * a.max_blocks;
  const unsigned long long* keys = a.keys + (int64_t)u * a.max_blocks;
  unsigned long long lo = 0, hi = 0;  // keys above hi are chosen; `rest` of those in [lo, hi], lowest pages first
  int rest = need;
  if (m > need && need > 0) {
    unsigned long long mn = ~0ull, mx = 0;
    for (int i = tid; i < m; i += kSelThreads) {
      const unsigned long long k = keys[i];
      mn = min(mn, k);
      mx = max(mx, k);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      mn = min(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
    if (lane == 0) ends[0][warp] = mn, ends[1][warp] = mx;
    __syncthreads();
    lo = ~0ull, hi = 0;
    for (int w = 0; w < NW; ++w) {
      lo = min(lo, ends[0][w]);
      hi = max(hi, ends[1][w]);
    }
    while (lo < hi) {  // each round cuts hi - lo by kBins / 2 or more: at most 7
      const unsigned long long span = hi - lo;
      int sh = 0;
      while ((span >> sh) >= kBins) ++sh;
      for (int i = tid; i < kBins; i += kSelThreads) bins[i] = 0;
      __syncthreads();
      for (int i = tid; i < m; i += kSelThreads) {
        const unsigned long long k = keys[i];
        if (k >= lo && k <= hi) atomicAdd(&bins[(int)((k - lo) >> sh)], 1);
      }
      __syncthreads();
      // from the top: the bin where the count reaches rest
      constexpr int PER = kBins / kSelThreads;
      int mine = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) mine += bins[kBins - 1 - (tid * PER + j)];
      int inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      if (lane == 31) warp_sums[warp] = inc;
      __syncthreads();
      int before = inc - mine;
      for (int w = 0; w < warp; ++w) before += warp_sums[w];
      if (before < rest && before + mine >= rest) {
        int acc = before;
        for (int j = 0; j < PER; ++j) {
          const int bin = kBins - 1 - (tid * PER + j), c = bins[bin];
          if (acc + c >= rest) {
            found_bin = bin;
            found_above = acc;
            found_count = c;
            break;
          }
          acc += c;
        }
      }
      __syncthreads();
      rest -= found_above;
      const unsigned long long top = hi;
      lo += (unsigned long long)found_bin << sh;
      hi = min(top, lo + ((1ull << sh) - 1));
      const bool whole = found_count == rest;
      __syncthreads();  // found_* and bins are free again
      if (whole) break;
    }
  }
  // ordered write: pages in ascending order, the last one behind them
  int* const pg = a.pages ? a.pages + (int64_t)u * a.K : nullptr;
  int* const tb = a.table ? a.table + (int64_t)u * a.K : nullptr;
  auto put = [&](int at, int page) {
    if (!SA_DCHECK(at < a.K && page < a.max_blocks)) return;
    if (pg) pg[at] = page;
    if (tb) {
      int64_t phys = bt[page];
      if (phys < 0 || phys >= a.num_blocks) {
        if (h == 0) atomicAdd(&g_bad_pages, 1u);
        phys = 0;
      }
      tb[at] = (int32_t)(phys * a.Hkv + h);
    }
  };
  const bool all = m <= need;
  int base = 0, base_in = 0;  // chosen and in-range keys of earlier pages
  for (int i0 = 0; i0 < m && need > 0; i0 += kSelThreads) {
    const int i = i0 + tid;
    bool above = false, in = false;
    if (i < m) {
      const unsigned long long k = all ? 0 : keys[i];
      above = all || k > hi;
      in = !all && k >= lo && k <= hi;
    }
    const unsigned in_w = __ballot_sync(0xffffffffu, in), ab_w = __ballot_sync(0xffffffffu, above);
    const unsigned below = (1u << lane) - 1;
    if (lane == 0) warp_sums[warp] = __popc(in_w) | (__popc(ab_w) << 16);
    __syncthreads();
    int in_before = base_in + __popc(in_w & below), ab_before = __popc(ab_w & below), in_all = 0, ab_all = 0;
    for (int w = 0; w < NW; ++w) {
      const int c = warp_sums[w];
      if (w < warp) in_before += c & 0xffff, ab_before += c >> 16;
      in_all += c & 0xffff;
      ab_all += c >> 16;
    }
    // chosen before this page: the above ones, and of the in-range ones the first `rest`
    const int at = base + ab_before + min(in_before, rest) - min(base_in, rest);
    if (above || (in && in_before < rest)) put(at, i);
    base += ab_all + min(base_in + in_all, rest) - min(base_in, rest);
    base_in += in_all;
    __syncthreads();
  }
  const int chosen = s.n > 0 ? need + 1 : 0;
  if (tid == 0) {
    if (s.n > 0) put(need, m);
    a.lens[u] = s.n > 0 ? need * a.bs + s.ctx - m * a.bs : 0;
  }
  for (int i = chosen + tid; i < a.K; i += kSelThreads) {
    if (pg) pg[i] = -1;
    if (tb) tb[i] = 0;
  }
}

// ---- host side --------------------------------------------------------------------

template <typename E, int D>
static int launch_means(const MeansArgs& a, int64_t B, cudaStream_t st) {
  // enough blocks for 8 an SM, each a contiguous stride of warps; a sequence without new pages leaves at once
  const int64_t most = ((int64_t)a.max_blocks * a.Hkv + 7) / 8;
  const int64_t x = std::max<int64_t>(1, std::min<int64_t>(most, (16ll * qkr::sm_count() + B - 1) / B));
  paged_key_means_kernel<E, D><<<dim3((unsigned)x, (unsigned)B), 256, 0, st>>>(a);
  return sa_record_cuda_error(cudaGetLastError());
}

template <typename E>
static int launch_means_d(const MeansArgs& a, int64_t B, int64_t D, cudaStream_t st) {
  switch (D) {
    case 32: return launch_means<E, 32>(a, B, st);
    case 64: return launch_means<E, 64>(a, B, st);
    case 128: return launch_means<E, 128>(a, B, st);
    default: return launch_means<E, 256>(a, B, st);
  }
}

template <typename E, int D, int GT>
static int launch_score(const SelectArgs& a, int64_t units, cudaStream_t st) {
  constexpr int PAGES = D == 256 ? 64 : 128;
  constexpr size_t smem = (size_t)D * GT * 8 + (size_t)PAGES * (D * 2 + 16);
  static_assert(smem <= 64 * 1024, "score kernel's shared memory");
  auto kfn = paged_score_kernel<E, D, GT, PAGES>;
  if (smem > 48 * 1024) {
    const int rc = sa_record_cuda_error(cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    if (rc != SA_OK) return rc;
  }
  kfn<<<dim3((unsigned)((a.max_blocks + PAGES - 1) / PAGES), (unsigned)units), PAGES, smem, st>>>(a);
  return sa_record_cuda_error(cudaGetLastError());
}

template <typename E, int D>
static int launch_score_g(const SelectArgs& a, int64_t units, cudaStream_t st) {
  if (a.G % 8 == 0) return launch_score<E, D, 8>(a, units, st);
  if (a.G % 4 == 0) return launch_score<E, D, 4>(a, units, st);
  if (a.G % 2 == 0) return launch_score<E, D, 2>(a, units, st);
  return launch_score<E, D, 1>(a, units, st);
}

template <typename E>
static int launch_score_d(const SelectArgs& a, int64_t units, int64_t D, cudaStream_t st) {
  switch (D) {
    case 32: return launch_score_g<E, 32>(a, units, st);
    case 64: return launch_score_g<E, 64>(a, units, st);
    case 128: return launch_score_g<E, 128>(a, units, st);
    default: return launch_score_g<E, 256>(a, units, st);
  }
}

static int check_cache(int64_t B, int64_t Hkv, int64_t num_blocks, int64_t bs, int64_t max_blocks, int64_t D,
                       int dtype) {
  if (B < 0 || Hkv <= 0 || num_blocks <= 0 || bs <= 0 || max_blocks <= 0) return SA_ERR_ARG;
  if (dtype != SA_BF16 && dtype != SA_F16) return SA_ERR_UNSUPPORTED;
  if (D != 32 && D != 64 && D != 128 && D != 256) return SA_ERR_UNSUPPORTED;
  if (B > 65535 || Hkv > (1 << 16) || B * Hkv > 65535 || bs > (1 << 16) || max_blocks * bs > ((int64_t)1 << 30) ||
      num_blocks > INT32_MAX / Hkv)
    return SA_ERR_UNSUPPORTED;
  return SA_OK;
}

static int64_t pad256(int64_t n) { return (n + 255) / 256 * 256; }

struct Layout {  // workspace of the choice, then of the decode that follows it
  int64_t keys, table, lens, decode, total;
};

static int layout_of(int64_t B, int64_t Hq, int64_t Hkv, int64_t max_blocks, int64_t K, int64_t bs, int64_t D,
                     int dtype, bool decode, Layout* l) {
  const int64_t units = B * Hkv;
  l->keys = 0;
  int64_t at = pad256(units * max_blocks * 8);
  l->table = at;
  if (decode) at += pad256(units * K * 4);
  l->lens = at;
  at += pad256(units * 4);
  l->decode = at;
  if (decode) {
    const int64_t n = sa_paged_decode_workspace_size(units, Hq / Hkv, 1, K, bs, D, dtype);
    if (n < 0) return (int)n;
    at += std::max(pad256(n), pad256(B * Hq * 4));
  }
  l->total = at;
  return SA_OK;
}

static int run_choice(SelectArgs& a, const void* q, const void* means, const int32_t* bt, const int32_t* cl,
                      int64_t B, int64_t Hq, int64_t Hkv, int64_t num_blocks, int64_t bs, int64_t max_blocks, int64_t K,
                      int64_t D, double scale, int dtype, cudaStream_t st) {
  a.q = q, a.means = means, a.bt = bt, a.cl = cl;
  a.num_blocks = num_blocks;
  a.scale2 = 2.0 * scale;
  a.Hkv = (int)Hkv, a.G = (int)(Hq / Hkv), a.bs = (int)bs, a.max_blocks = (int)max_blocks, a.K = (int)K;
  const int64_t units = B * Hkv;
  if (max_blocks > K) {  // else every page is taken
    const int rc = dtype == SA_BF16 ? launch_score_d<__nv_bfloat16>(a, units, D, st)
                                    : launch_score_d<__half>(a, units, D, st);
    if (rc != SA_OK) return rc;
  }
  paged_choose_kernel<<<(unsigned)units, kSelThreads, 0, st>>>(a);
  return sa_record_cuda_error(cudaGetLastError());
}

}  // namespace pgs

int paged_select_bad_pages(int reset, cudaStream_t st) {
  unsigned v = 0;
  cudaMemcpyFromSymbolAsync(&v, pgs::g_bad_pages, sizeof(v), 0, cudaMemcpyDeviceToHost, st);
  cudaStreamSynchronize(st);
  if (reset) {
    const unsigned z = 0;
    cudaMemcpyToSymbolAsync(pgs::g_bad_pages, &z, sizeof(z), 0, cudaMemcpyHostToDevice, st);
    cudaStreamSynchronize(st);
  }
  return (int)v;
}

}  // namespace sa

extern "C" int sa_paged_key_means(const void* k_cache, void* key_means, const int32_t* block_table,
                                  const int32_t* context_lens, const int32_t* start_lens, int64_t B, int64_t Hkv,
                                  int64_t num_blocks, int64_t block_size, int64_t max_blocks, int64_t D, int dtype,
                                  void* stream) {
  using namespace sa::pgs;
  const int rc = check_cache(B, Hkv, num_blocks, block_size, max_blocks, D, dtype);
  if (rc != SA_OK) return rc;
  if (B == 0) return SA_OK;
  if (!k_cache || !key_means || !block_table || !context_lens) return SA_ERR_ARG;
  if (!al16(k_cache) || !al16(key_means)) return SA_ERR_ALIGN;
  const MeansArgs a{k_cache, key_means, block_table, context_lens, start_lens, num_blocks, (int)Hkv, (int)block_size,
                    (int)max_blocks};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == SA_BF16 ? launch_means_d<__nv_bfloat16>(a, B, D, st) : launch_means_d<__half>(a, B, D, st);
}

static int check_choice(int64_t B, int64_t Hq, int64_t Hkv, int64_t num_blocks, int64_t bs, int64_t max_blocks,
                        int64_t K, int64_t D, double scale, int dtype) {
  const int rc = sa::pgs::check_cache(B, Hkv, num_blocks, bs, max_blocks, D, dtype);
  if (rc != SA_OK) return rc;
  if (Hq <= 0 || Hq % Hkv != 0 || K <= 0 || K > max_blocks || !(scale == scale)) return SA_ERR_ARG;
  return Hq > (1 << 20) ? SA_ERR_UNSUPPORTED : SA_OK;
}

extern "C" int64_t sa_paged_select_workspace_size(int64_t B, int64_t Hkv, int64_t max_blocks) {
  if (B < 0 || Hkv <= 0 || max_blocks <= 0) return SA_ERR_ARG;
  if (B > 65535 || Hkv > 65535 || B * Hkv > 65535 || max_blocks > ((int64_t)1 << 30)) return SA_ERR_UNSUPPORTED;
  return sa::pgs::pad256(B * Hkv * max_blocks * 8);
}

extern "C" int sa_paged_select(const void* q, const void* key_means, const int32_t* block_table,
                               const int32_t* context_lens, int32_t* pages, int32_t* lens, void* workspace,
                               int64_t workspace_bytes, int64_t B, int64_t Hq, int64_t Hkv, int64_t num_blocks,
                               int64_t block_size, int64_t max_blocks, int64_t num_pages, int64_t D, double scale,
                               int dtype, void* stream) {
  using namespace sa::pgs;
  const int rc = check_choice(B, Hq, Hkv, num_blocks, block_size, max_blocks, num_pages, D, scale, dtype);
  if (rc != SA_OK) return rc;
  if (B == 0) return SA_OK;
  if (!q || !key_means || !block_table || !context_lens || !pages || !lens || !workspace) return SA_ERR_ARG;
  if (workspace_bytes < sa_paged_select_workspace_size(B, Hkv, max_blocks)) return SA_ERR_ARG;
  if (!al16(q) || !al16(key_means) || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return SA_ERR_ALIGN;
  SelectArgs a{};
  a.keys = static_cast<unsigned long long*>(workspace);
  a.pages = pages;
  a.lens = lens;
  return run_choice(a, q, key_means, block_table, context_lens, B, Hq, Hkv, num_blocks, block_size, max_blocks,
                    num_pages, D, scale, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t sa_sparse_paged_decode_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t max_blocks,
                                                         int64_t num_pages, int64_t block_size, int64_t D,
                                                         int dtype) {
  const int rc = check_choice(B, Hq, Hkv, 1, block_size, max_blocks, num_pages, D, 1.0, dtype);
  if (rc != SA_OK) return rc;
  if (B == 0) return 0;
  sa::pgs::Layout l;
  const int lrc = sa::pgs::layout_of(B, Hq, Hkv, max_blocks, num_pages, block_size, D, dtype, true, &l);
  return lrc != SA_OK ? lrc : l.total;
}

extern "C" int sa_sparse_paged_decode(const void* q, const void* k_cache, const void* v_cache, const void* key_means,
                                      void* out, const int32_t* block_table, const int32_t* context_lens,
                                      int32_t* pages, void* workspace, int64_t workspace_bytes, int64_t B, int64_t Hq,
                                      int64_t Hkv, int64_t num_blocks, int64_t block_size, int64_t max_blocks,
                                      int64_t num_pages, int64_t D, double scale, int dtype, void* stream) {
  using namespace sa::pgs;
  int rc = check_choice(B, Hq, Hkv, num_blocks, block_size, max_blocks, num_pages, D, scale, dtype);
  if (rc != SA_OK) return rc;
  if (B == 0) return SA_OK;
  if (!q || !k_cache || !v_cache || !key_means || !out || !block_table || !context_lens || !workspace)
    return SA_ERR_ARG;
  if (!al16(q) || !al16(k_cache) || !al16(v_cache) || !al16(key_means) || !al16(out) ||
      (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0)
    return SA_ERR_ALIGN;
  Layout l;
  rc = layout_of(B, Hq, Hkv, max_blocks, num_pages, block_size, D, dtype, true, &l);
  if (rc != SA_OK) return rc;
  if (workspace_bytes < l.total) return SA_ERR_ARG;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  SelectArgs a{};
  a.keys = reinterpret_cast<unsigned long long*>(ws + l.keys);
  a.pages = pages;
  a.table = reinterpret_cast<int32_t*>(ws + l.table);
  a.lens = reinterpret_cast<int32_t*>(ws + l.lens);
  a.tickets = reinterpret_cast<int32_t*>(ws + l.decode);  // at most one word per query head
  a.num_tickets = B * Hq;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  rc = run_choice(a, q, key_means, block_table, context_lens, B, Hq, Hkv, num_blocks, block_size, max_blocks, num_pages,
                  D, scale, dtype, st);
  if (rc != SA_OK) return rc;
  return sa_paged_decode(q, k_cache, v_cache, out, a.table, a.lens, ws + l.decode, l.total - l.decode, B * Hkv, Hq / Hkv,
                         1, num_blocks * Hkv, block_size, num_pages, D, (float)scale, dtype, stream);
}
SA_BOUNDS_ACCESSOR(paged_select_bounds)
