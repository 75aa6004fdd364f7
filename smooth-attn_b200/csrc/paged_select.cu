// Decode over chosen pages of a paged key-value cache, sm_100a: mean keys of
// full pages, the choice of each sequence's and key head's pages by a cheap
// score, and the attention over these alone.  (No reference counterpart: the
// reference's decode, src/smooth_attn/kernels.py:2681-2829, reads every page.)
//
// Score.  The normaliser of squareplus attention is a plain sum, so a page's
// share of one head's is the sum of its tokens' weights; the score estimates that
// at the page's mean key and adds it up over the group's query heads:
//   score(page) = sum_g y(2 scale q_g . mean_key(page) - 1),
//   y(a) = squareplus(a)^2
// The heads' weights are added as they are, not divided by each head's normaliser
// (which would take every page's score of every head first), so a head with
// large queries has more say in what the group reads.
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
// Bound.  32 sequences of 5000 to 8192 tokens, 64 pages of each and 8 key heads
// (27 MB of mean keys, 134 MB of chosen pages: 25 us at the measured copy rate):
// scores and choice 24 us (21 with the means in L2), the decode 35 us.  Of the 21 the choice
// is 4; the products are 9 to 11 on the 64-bit matrix pipe, 17 cycles each, half of
// their eight columns empty for groups of four heads; the rest is the launch and the
// chain from lengths to page ids to rows.  Built too: fp32 scores with proven bounds and 64
// bits where those overlap (164 instructions for two rows, a second order
// statistic, and the rare 64-bit path in some block of every launch: 34 us against
// 26), and plain 64-bit multiply-adds of the four heads alone with the rows through a ring in
// shared memory (20 us against 21, and groups of one head 15.5 against 14.4).  One sequence
// of 32768 tokens, 128 pages: 11 us + 10 us, launches and the chain of dependent reads.
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

// One warp: one page of one key head; LPR lanes a row, 32 / LPR rows at once.  A
// warp takes several pages and asks for the next one's first rows (and the table
// entry behind it) before it adds this one's up.
template <typename E, int D>
__global__ void __launch_bounds__(256) paged_key_means_kernel(MeansArgs a) {
  constexpr int LPR = D / 8, RPW = 32 / LPR, U = 8;
  const int b = blockIdx.y, lane = threadIdx.x & 31;
  const int64_t cap = (int64_t)a.max_blocks * a.bs;
  const int ctx = (int)max((int64_t)0, min(cap, (int64_t)a.cl[b]));
  const int from = a.start ? max(0, a.start[b]) / a.bs : 0;
  const int64_t n = (int64_t)max(0, ctx / a.bs - from) * a.Hkv;
  const int32_t* bt = a.bt + (int64_t)b * a.max_blocks + from;
  const int64_t step = (int64_t)gridDim.x * 8;
  int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (w >= n) return;
  const float inv = 1.0f / (float)a.bs;
  const int r0 = lane / LPR;
  auto page_at = [&](int64_t i) { return i < n ? __ldg(bt + i / a.Hkv) : 0; };
  auto rows_of = [&](int64_t i, int page) {
    const bool ok = page >= 0 && page < a.num_blocks;
    return static_cast<const E*>(a.kc) + ((ok ? (int64_t)page : 0) * a.Hkv + i % a.Hkv) * a.bs * D + (lane % LPR) * 8;
  };
  auto load = [&](Raw8<E> (&x)[U], const E* base, int r) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r + u * RPW < a.bs) x[u].load(base + (int64_t)(r + u * RPW) * D);
      else x[u].zero();
    }
  };
  Raw8<E> x[U];
  int page = page_at(w), next = page_at(w + step);
  load(x, rows_of(w, page), r0);
  for (; w < n; w += step) {
    float2 sum[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
    auto add = [&](const Raw8<E> (&y)[U]) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float2 f[4];
        y[u].get(f);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = fadd2(sum[i], f[i]);
      }
    };
    const E* base = rows_of(w, page);
    const int mine = page;
    add(x);
    page = next;
    if (w + step < n) load(x, rows_of(w + step, page), r0);
    next = page_at(w + 2 * step);
    for (int r = r0 + RPW * U; r - r0 < a.bs; r += RPW * U) {  // pages of more rows than one batch
      Raw8<E> y[U];
      load(y, base, r);
      add(y);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int m = LPR; m < 32; m <<= 1) {
        sum[i].x += __shfl_xor_sync(0xffffffffu, sum[i].x, m);
        sum[i].y += __shfl_xor_sync(0xffffffffu, sum[i].y, m);
      }
      sum[i] = fmul2(sum[i], make_float2(inv, inv));
    }
    if (mine < 0 || mine >= a.num_blocks) {
      if (lane == 0 && w % a.Hkv == 0) atomicAdd(&g_bad_pages, 1u);
    } else if (lane < LPR) {
      Raw8<E> o;
      o.set(sum);
      o.store(static_cast<E*>(a.means) + ((int64_t)mine * a.Hkv + w % a.Hkv) * D + lane * 8);
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

// squareplus(a)^2 in 64 bits.  a + sqrt(a^2 + 4) loses about a^2 roundings for
// negative a: the quotient that is equal to it takes over where that passes 64.
__device__ __forceinline__ double weight64(double a) {
  const double root = sqrt(fma(a, a, 4.0));
  double sp = 0.5 * (a + root);
  if (a < -8.0) sp = 2.0 / (root - a);
  return sp * sp;
}

// Zeros in the decode's tickets: its next launch finds a workspace of undefined contents.
__device__ __forceinline__ void clear_tickets(const SelectArgs& a, int64_t first, int64_t step) {
  for (int64_t i = first; i < a.num_tickets; i += step) a.tickets[i] = 0;
}

__device__ __forceinline__ unsigned long long key_of(double score) {
  // scores are not negative, so their bits order as they do; NaN above all
  return isnan(score) ? 0x7ff8000000000000ull : (unsigned long long)__double_as_longlong(score);
}

// D += A B with A [8 pages x 4 channels], B [4 channels x 8 heads] in 64 bits: lane
// l holds A[l / 4][l % 4], B[l % 4][l / 4] and D[l / 4][2 (l % 4) + {0, 1}].
__device__ __forceinline__ void mma64(double (&d)[2], double a, double b) {
  asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};"
               : "+d"(d[0]), "+d"(d[1])
               : "d"(a), "d"(b));
}

// ---- choice ---------------------------------------------------------------------

constexpr int kScoreThreads = 256;
constexpr int kBins = 2048;
constexpr int kKeep = 8;    // keys a thread keeps in registers
constexpr int kShort = 64;  // keys that are ranked by comparing each with each

// One block chooses for one sequence and key head.  The threshold is found by
// counting keys in kBins equal ranges of [lo, hi], which is narrowed to the range
// that holds the last chosen key until all of that range is chosen, it is one
// value, or so few keys that they are ranked directly; then an ordered pass writes
// what is chosen.
template <int kSelThreads> struct ChooseShared {
  int bins[kBins];
  unsigned long long ends[2][kSelThreads / 32], few[kShort];
  int warp_sums[kSelThreads / 32], counts[kKeep * (kSelThreads / 32)];
  int found_bin, found_above, found_count, nfew;
};

template <int kSelThreads>
__device__ __forceinline__ void choose_pages(const SelectArgs& a, int u, ChooseShared<kSelThreads>& sh) {
  constexpr int kSelWarps = kSelThreads / 32;
  auto& bins = sh.bins;
  auto& ends = sh.ends;
  auto& few = sh.few;
  auto& warp_sums = sh.warp_sums;
  auto& counts = sh.counts;
  int &found_bin = sh.found_bin, &found_above = sh.found_above, &found_count = sh.found_count, &nfew = sh.nfew;
  const int b = u / a.Hkv, h = u - b * a.Hkv, tid = threadIdx.x;
  const int lane = tid & 31, warp = tid >> 5;
  const int32_t* bt = a.bt + (int64_t)b * a.max_blocks;
  const unsigned long long* keys = a.keys + (int64_t)u * a.max_blocks;
  // read beside the length, not after it: what lies behind the candidates is not looked at
  // (so are the pages' places in the cache, which only what is chosen needs)
  unsigned long long mine[kKeep];
  int place[kKeep];
#pragma unroll
  for (int j = 0; j < kKeep; ++j) {
    const int i = j * kSelThreads + tid;
    place[j] = i < a.max_blocks && a.table ? __ldg(bt + i) : 0;
    mine[j] = i < a.max_blocks && a.max_blocks > a.K ? __ldcg(keys + i) : 0;  // (other SMs' writes)
  }
  const Seq s = seq_of(a, b);
  const int m = s.n - 1, need = min(a.K, s.n) - 1;  // of the m candidates
  const int last_place = tid == 0 && m >= 0 && a.table ? __ldg(bt + m) : 0;
  // keys above hi are chosen, and `rest` of those in [lo, hi], lowest pages first
  unsigned long long lo = 0, hi = ~0ull;
  int rest = need;
  const bool kept = m <= kKeep * kSelThreads;
  auto each_key = [&](auto&& f) {
    if (kept) {
#pragma unroll
      for (int j = 0; j < kKeep; ++j)
        if (j * kSelThreads + tid < m) f(mine[j]);
    } else {
      for (int i = tid; i < m; i += kSelThreads) f(__ldcg(keys + i));
    }
  };
  if (m > need && need > 0) {
    unsigned long long mn = ~0ull, mx = 0;
    each_key([&](unsigned long long k) {
      mn = min(mn, k);
      mx = max(mx, k);
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      mn = min(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
    if (lane == 0) ends[0][warp] = mn, ends[1][warp] = mx;
    for (int i = tid; i < kBins; i += kSelThreads) bins[i] = 0;
    __syncthreads();
    mn = ends[0][lane % kSelWarps];
    mx = ends[1][lane % kSelWarps];
#pragma unroll
    for (int o = kSelWarps / 2; o > 0; o >>= 1) {
      mn = min(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
    lo = mn, hi = mx;
    while (lo < hi) {  // each round cuts hi - lo by kBins / 2 or more: at most 7
      const int sh = max(0, 64 - 11 - __clzll((long long)(hi - lo)));  // (hi - lo) >> sh < kBins = 2^11
      each_key([&](unsigned long long k) {
        if (k >= lo && k <= hi) atomicAdd(&bins[(int)((k - lo) >> sh)], 1);
      });
      __syncthreads();
      // from the top: the bin where the count reaches rest
      constexpr int PER = kBins / kSelThreads;
      int cnt[PER], sum = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) sum += cnt[j] = bins[kBins - 1 - (tid * PER + j)];
      int inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      if (lane == 31) warp_sums[warp] = inc;
      if (tid == 0) nfew = 0;
      __syncthreads();
      int before = inc - sum;
#pragma unroll
      for (int w = 0; w < kSelWarps; ++w) before += w < warp ? warp_sums[w] : 0;
      if (before < rest && before + sum >= rest) {
        int acc = before;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          if (acc < rest && acc + cnt[j] >= rest) {
            found_bin = kBins - 1 - (tid * PER + j);
            found_above = acc;
            found_count = cnt[j];
          }
          acc += cnt[j];
        }
      }
#pragma unroll
      for (int j = 0; j < PER; ++j) bins[kBins - 1 - (tid * PER + j)] = 0;  // for the next round
      __syncthreads();
      rest -= found_above;
      lo += (unsigned long long)found_bin << sh;
      hi = min(hi, lo + ((1ull << sh) - 1));
      const int count = found_count;
      if (count == rest) break;  // the whole range is chosen
      if (count <= kShort) {
        each_key([&](unsigned long long k) {
          if (k >= lo && k <= hi) few[atomicAdd(&nfew, 1)] = k;
        });
        __syncthreads();
        if (tid < count) {
          int above = 0, same = 0;
          const unsigned long long k = few[tid];
#pragma unroll 8
          for (int j = 0; j < count; ++j) {
            above += few[j] > k;
            same += few[j] == k;
          }
          if (above < rest && above + same >= rest) {  // the last chosen value; equal keys write the same
            ends[0][0] = k;
            found_above = above;
          }
        }
        __syncthreads();
        lo = hi = ends[0][0];
        rest -= found_above;
        break;
      }
    }
  }
  // ordered write: pages in ascending order, the last one behind them
  int* const pg = a.pages ? a.pages + (int64_t)u * a.K : nullptr;
  int* const tb = a.table ? a.table + (int64_t)u * a.K : nullptr;
  auto put = [&](int at, int page, int64_t phys) {
    if (!SA_DCHECK(at < a.K && page < a.max_blocks)) return;
    if (pg) pg[at] = page;
    if (tb) {
      if (phys < 0 || phys >= a.num_blocks) {
        if (h == 0) atomicAdd(&g_bad_pages, 1u);
        phys = 0;
      }
      tb[at] = (int32_t)(phys * a.Hkv + h);
    }
  };
  if (m <= need) {
#pragma unroll
    for (int j = 0; j < kKeep; ++j)
      if (j * kSelThreads + tid < m) put(j * kSelThreads + tid, j * kSelThreads + tid, place[j]);
    for (int i = kKeep * kSelThreads + tid; i < m; i += kSelThreads) put(i, i, __ldg(bt + i));
  } else if (need > 0) {
    // a batch of kKeep * kSelThreads pages at a time; a count is in-range keys, and above ones << 16
    int base = 0, base_in = 0;  // chosen and in-range keys of earlier batches
    for (int i0 = 0; i0 < m; i0 += kKeep * kSelThreads) {
      unsigned in_w[kKeep], ab_w[kKeep];
#pragma unroll
      for (int j = 0; j < kKeep; ++j) {
        const int i = i0 + j * kSelThreads + tid;
        const unsigned long long k = i >= m ? 0 : kept ? mine[j] : __ldcg(keys + i);
        in_w[j] = __ballot_sync(0xffffffffu, i < m && k >= lo && k <= hi);
        ab_w[j] = __ballot_sync(0xffffffffu, i < m && k > hi);
        if (lane == 0) counts[j * kSelWarps + warp] = __popc(in_w[j]) | (__popc(ab_w[j]) << 16);
      }
      __syncthreads();
      if (warp == 0) {  // exclusive scan of the kKeep * kSelWarps counts, in page order
        constexpr int PER = kKeep * kSelWarps / 32;
        int c[PER], sum = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) sum += c[j] = counts[lane * PER + j];
        int inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += v;
        }
        int at = inc - sum;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          counts[lane * PER + j] = at;
          at += c[j];
        }
        if (lane == 31) found_count = inc;  // of the whole batch
      }
      __syncthreads();
      const unsigned below = (1u << lane) - 1;
#pragma unroll
      for (int j = 0; j < kKeep; ++j) {
        const int c = counts[j * kSelWarps + warp], i = i0 + j * kSelThreads + tid;
        const int in_before = base_in + (c & 0xffff) + __popc(in_w[j] & below);
        const int ab_before = (c >> 16) + __popc(ab_w[j] & below);
        const bool in = (in_w[j] >> lane) & 1, above = (ab_w[j] >> lane) & 1;
        // chosen before this page: the above ones, and of the in-range ones the first `rest`
        if (above || (in && in_before < rest))
          put(base + ab_before + min(in_before, rest) - min(base_in, rest), i,
              i0 == 0 ? place[j] : a.table ? __ldg(bt + i) : 0);
      }
      const int c = found_count;
      base += (c >> 16) + min(base_in + (c & 0xffff), rest) - min(base_in, rest);
      base_in += c & 0xffff;
      __syncthreads();  // counts are free again
    }
  }
  const int chosen = s.n > 0 ? need + 1 : 0;
  if (tid == 0) {
    if (s.n > 0) put(need, m, last_place);
    a.lens[u] = s.n > 0 ? need * a.bs + s.ctx - m * a.bs : 0;
  }
  for (int i = chosen + tid; i < a.K; i += kSelThreads) {
    if (pg) pg[i] = -1;
    if (tb) tb[i] = 0;
  }
}

// ---- scores, and the choice behind them ---------------------------------------------

// One block: 128 pages of one key head at a time, 16 a warp (two row blocks of the
// product above).  Lane l reads every fourth 16-byte piece of rows l / 4 and 8 + l / 4, so
// four lanes read 64 neighbouring bytes, and the channels of a product step are
// the same element of four neighbouring pieces; the queries lie in shared memory
// as each lane's B of every step.  Heads go eight at a time.  (One page a thread
// with plain fused multiply-adds, the queries broadcast from shared memory, took
// 12.5 us for 2048 pages of 8 key heads, this 4.1 us.)
template <typename E, int D>
__global__ void __launch_bounds__(kScoreThreads, 2) paged_score_kernel(SelectArgs a, int choose) {
  constexpr int P = D / 32;  // 16-byte pieces a lane holds of a row
  constexpr bool kAhead = P <= 4;  // the next tile's rows are asked for before this one's product (at D = 256 no room)
  constexpr int TILE = kScoreThreads / 2;  // pages of a block: 16 a warp
  constexpr int NQ = (D + kScoreThreads - 1) / kScoreThreads;
  __shared__ double qs[D / 4][32];
  __shared__ ChooseShared<kScoreThreads> sh;
  const int u = blockIdx.y, b = u / a.Hkv, h = u - b * a.Hkv;
  clear_tickets(a, ((int64_t)u * gridDim.x + blockIdx.x) * kScoreThreads + threadIdx.x,
                (int64_t)gridDim.x * gridDim.y * kScoreThreads);
  const int lane = threadIdx.x & 31, c = lane & 3, step = gridDim.x * TILE;
  int p0 = blockIdx.x * TILE + (threadIdx.x >> 5) * 16 + (lane >> 2);
  const int32_t* bt = a.bt + (int64_t)b * a.max_blocks;
  // the first tile's ids and the queries are asked for beside the length, not after it
  int page[2];
  auto ids = [&](int at, int end) {
#pragma unroll
    for (int r = 0; r < 2; ++r) page[r] = at + 8 * r < end ? __ldg(bt + at + 8 * r) : 0;
  };
  auto load_q = [&](int g0, uint4 (&v)[NQ]) {
    const uint4* q = reinterpret_cast<const uint4*>(static_cast<const E*>(a.q) + ((int64_t)u * a.G + g0) * D);
#pragma unroll
    for (int j = 0; j < NQ; ++j) {  // 8 heads of D / 8 pieces
      const int i = threadIdx.x + j * kScoreThreads;
      v[j] = i < D && i / (D / 8) < a.G - g0 ? __ldg(q + i) : make_uint4(0, 0, 0, 0);
    }
  };
  uint4 qv[NQ];
  ids(p0, a.max_blocks);
  load_q(0, qv);
  const Seq s = seq_of(a, b);
  const int m = s.n - 1;                            // candidates: all but the last page
  const bool score_any = m > a.K - 1 && (int)blockIdx.x * TILE < m;  // else all are taken, or none is this block's
  auto load = [&](uint4 (&x)[2][P], int at) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if (at + 8 * r >= m) page[r] = 0;  // (an entry behind the context says nothing)
      if (page[r] < 0 || page[r] >= a.num_blocks) {
        if (c == 0 && h == 0) atomicAdd(&g_bad_pages, 1u);
        page[r] = 0;
      }
      const uint4* row =
          reinterpret_cast<const uint4*>(static_cast<const E*>(a.means) + ((int64_t)page[r] * a.Hkv + h) * D);
#pragma unroll
      for (int i = 0; i < P; ++i) x[r][i] = __ldg(row + 4 * i + c);
    }
  };
  uint4 x[2][P];
  if (score_any) {
    load(x, p0);
    ids(p0 + step, m);
  }
  for (int t0 = blockIdx.x * TILE; score_any && t0 < m; t0 += step, p0 += step) {
    uint4 y[2][kAhead ? P : 1];
    if constexpr (kAhead) {
      if (t0 + step < m) {
        load(y, p0 + step);
        ids(p0 + 2 * step, m);
      }
    }
    double score[2] = {0.0, 0.0};
    for (int g0 = 0; g0 < a.G; g0 += 8) {
      const int heads = min(8, a.G - g0);
      if (a.G > 8 || t0 < step) {  // one group of heads stays in place
        if (g0 || t0 >= step) __syncthreads();  // the last heads' queries have been read
        if (g0 || t0 >= step) load_q(g0, qv);
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          const int i = threadIdx.x + j * kScoreThreads, g = i / (D / 8), piece = i % (D / 8);
          if (i >= D) break;
          float f[8];
          unpack<E, 8>(&qv[j], f);
#pragma unroll
          for (int e = 0; e < 8; ++e) qs[(piece / 4) * 8 + e][g * 4 + piece % 4] = (double)f[e];
        }
        __syncthreads();
      }
      double d0[2] = {0.0, 0.0}, d1[2] = {0.0, 0.0}, o0[2] = {0.0, 0.0}, o1[2] = {0.0, 0.0};  // even and odd steps
#pragma unroll
      for (int i = 0; i < P; ++i) {
        float f0[8], f1[8];
        unpack<E, 8>(&x[0][i], f0);
        unpack<E, 8>(&x[1][i], f1);
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const double qa = qs[i * 8 + e][lane], qb = qs[i * 8 + e + 1][lane];
          mma64(d0, (double)f0[e], qa);
          mma64(d1, (double)f1[e], qa);
          mma64(o0, (double)f0[e + 1], qb);
          mma64(o1, (double)f1[e + 1], qb);
        }
      }
      if (heads <= 4) {  // half the lanes have no head: they take the second row block's
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const double other = __shfl_xor_sync(0xffffffffu, d1[e] + o1[e], 2);
          const double w = (c < 2 ? 2 * c + e : 2 * c - 4 + e) < heads
                               ? weight64(fma(a.scale2, c < 2 ? d0[e] + o0[e] : other, -1.0)) : 0.0;
          score[0] += c < 2 ? w : 0.0;
          score[1] += c < 2 ? 0.0 : w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (2 * c + e < heads) {
            score[0] += weight64(fma(a.scale2, d0[e] + o0[e], -1.0));
            score[1] += weight64(fma(a.scale2, d1[e] + o1[e], -1.0));
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      score[r] += __shfl_xor_sync(0xffffffffu, score[r], 1);
      score[r] += __shfl_xor_sync(0xffffffffu, score[r], 2);
      if (c == r && p0 + 8 * r < m && SA_DCHECK(p0 + 8 * r < a.max_blocks))
        a.keys[(int64_t)u * a.max_blocks + p0 + 8 * r] = key_of(score[r]);
    }
    if constexpr (kAhead) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < P; ++i) x[r][i] = y[r][i];
    } else {
      if (t0 + step < m) {
        load(x, p0 + step);
        ids(p0 + 2 * step, m);
      }
    }
  }
  if (!choose) return;
  // the cluster's blocks have scored the sequence's pages; its first one chooses
  if (gridDim.x > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    if (blockIdx.x != 0) return;
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else {
    __syncthreads();
  }
  choose_pages<kScoreThreads>(a, u, sh);
}

// The choice by itself: long tables, after their scores, and tables whose every page is taken.
template <int NT> __global__ void __launch_bounds__(NT) paged_choose_kernel(SelectArgs a) {
  __shared__ ChooseShared<NT> sh;
  clear_tickets(a, (int64_t)blockIdx.x * NT + threadIdx.x, (int64_t)gridDim.x * NT);
  choose_pages<NT>(a, blockIdx.x, sh);
}

// ---- host side --------------------------------------------------------------------

// Blocks an SM of the mean keys: 8 prompts of 8191 tokens 26.7 us (4 an SM: 30, 6: 26), and one new token for
// 64 sequences, of which few have a page to do, 2.9 us (4: 3.3, 6: 3.6).
constexpr int kMeansBlocks = 2;

template <typename E, int D>
static int launch_means(const MeansArgs& a, int64_t B, cudaStream_t st) {
  // one resident wave (kMeansBlocks an SM) over all sequences; one without new pages leaves at once
  const int64_t most = ((int64_t)a.max_blocks * a.Hkv + 7) / 8;
  const int64_t x = std::max<int64_t>(1, std::min<int64_t>(most, ((int64_t)kMeansBlocks * qkr::sm_count() + B - 1) / B));
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

// Scores, and with `choose` the choice, in one launch: the blocks of one sequence
// and key head are a cluster, as many as one resident wave (two an SM) has for it,
// at most 8 (16 measured the same), tiles of 128 pages dealt to them.
template <typename E, int D>
static int launch_score_d(const SelectArgs& a, int64_t units, int choose, cudaStream_t st) {
  auto kfn = paged_score_kernel<E, D>;
  const int64_t tiles = (a.max_blocks + kScoreThreads / 2 - 1) / (kScoreThreads / 2), wave = 2ll * qkr::sm_count();
  int64_t x = std::max<int64_t>(1, std::min(tiles, wave / units));
  if (choose) x = std::min<int64_t>(x, 8);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)x, (unsigned)units);
  cfg.blockDim = dim3(kScoreThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  if (choose && x > 1) {
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)x;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
  }
  return sa_record_cuda_error(cudaLaunchKernelEx(&cfg, kfn, a, choose));
}

template <typename E>
static int launch_score(const SelectArgs& a, int64_t units, int64_t D, int choose, cudaStream_t st) {
  switch (D) {
    case 32: return launch_score_d<E, 32>(a, units, choose, st);
    case 64: return launch_score_d<E, 64>(a, units, choose, st);
    case 128: return launch_score_d<E, 128>(a, units, choose, st);
    default: return launch_score_d<E, 256>(a, units, choose, st);
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
  // a block of 256 threads holds the keys of up to 2048 pages in registers and chooses right behind the scores;
  // longer tables take a launch of 1024 threads for it
  const bool at_once = max_blocks <= kKeep * kScoreThreads;
  if (max_blocks > K) {
    const int rc = dtype == SA_BF16 ? launch_score<__nv_bfloat16>(a, units, D, at_once, st)
                                    : launch_score<__half>(a, units, D, at_once, st);
    if (rc != SA_OK || at_once) return rc;
  }
  if (at_once) paged_choose_kernel<256><<<(unsigned)units, 256, 0, st>>>(a);
  else paged_choose_kernel<1024><<<(unsigned)units, 1024, 0, st>>>(a);
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
