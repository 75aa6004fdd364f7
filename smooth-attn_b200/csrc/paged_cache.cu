// A paged key-value cache's bookkeeping and its writer, sm_100a: slots and
// block tables from request lengths, pages given back, and the append of new
// tokens (head norm and rotation on the way).  (No reference counterpart: the
// reference's paged decode, src/smooth_attn/kernels.py:2681-2829, is handed a
// filled cache and a block table built on the host.)
//
// Slots.  Request b holds context_lens[b] tokens in pages block_table[b, ..]
// and gets new_lens[b] more, taken from a flat buffer of N tokens in request
// order (cu = exclusive scan of new_lens).  With held = ceil(ctx / bs) pages
// and need = ceil((ctx + new) / bs) - held further ones, an exclusive scan of
// `need` says where in the pool's list its new pages begin: first come, first
// served.  What does not fit (the table's row, the pool, the buffer) is left
// out: those tokens get slot -1 and are not counted in the new length.
// Both scans are over B <= 16384 requests, a few microseconds' work of one
// block, so every block does them again for itself instead of waiting for
// another: one launch, no workspace, nothing to reset.  A token finds its
// request by a binary search of cu in shared memory, and the first token of a
// new page writes the table's entry.  Bound: the launch and the chain of loads
// and scans (64 requests, one token each: 3.7 us, an empty launch 2.2); for a
// million tokens (12 MB written: 1.9 us at the measured copy rate) the scans that
// every block repeats and the searches: 10 us.
//
// Append.  The walk of qk_rope.cuh over the q, k and v rows, each warp a part of
// one of the three: q rows go to a dense buffer, k and v rows to their slot's
// page.  Bound: HBM (8191 tokens of 32 + 8 + 8 heads of 128, 205 MB: 39 us, 0.81 of
// the measured copy rate; the shares of 1776 warps are 7 units of 8 heads each).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "qk_rope.cuh"
#include "smooth_attn_b200.h"

int sa_record_cuda_error(cudaError_t e);

namespace sa {
namespace pgc {

static __device__ unsigned g_bad_entries;  // slots past the cache, positions past the tables, negative pages, a pool given too much back

constexpr int kThreads = 512;
constexpr int kMaxRequests = 16384;  // 12 bytes each of shared memory

// Exclusive scan of one int64 per thread over the block; returns the sum before
// this thread, the total in *all.  warp_sums: used by no other scan of the block.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* all, int64_t* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int NW = kThreads / 32;
  int64_t inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  int64_t s = lane < NW ? warp_sums[lane] : 0;  // every warp scans the warps' sums for itself
#pragma unroll
  for (int o = 1; o < NW; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  const int64_t before = __shfl_sync(0xffffffffu, s, warp ? warp - 1 : 0);
  *all = __shfl_sync(0xffffffffu, s, NW - 1);
  return (warp ? before : 0) + inc - v;
}

struct AssignArgs {
  int32_t* table;
  int64_t ld;
  const int32_t* ctx;
  const int32_t* fresh;  // new_lens
  const int32_t* pool;
  const int32_t* head;
  long long* slots;
  int32_t* positions;
  int32_t* cu;
  int32_t* ctx_out;
  int32_t* head_out;
  int64_t num_free;
  int B, N, max_blocks, bs;
  qkr::FastDiv by_bs;
};

// V neighbouring tokens a thread: 4 share one search and are stored 16 bytes at a
// time; 1 where there are so few tokens that each should have a thread of its own
// (64 tokens of 64 requests: 3.7 us, 5.9 us with 4; a million tokens of 512 requests:
// 10 us with 4, 14 us with 1).
template <int V>
__global__ void __launch_bounds__(kThreads, 2) paged_assign_kernel(AssignArgs a) {
  extern __shared__ int32_t sm[];  // cu[B + 1], at[B], fits[B]
  __shared__ int64_t warp_sums[2][kThreads / 32];
  int32_t* cu = sm;
  int32_t* at = cu + a.B + 1;
  int32_t* fits = at + a.B;
  const int64_t cap = (int64_t)a.max_blocks * a.bs;  // at most 2^30
  const int per = (a.B + kThreads - 1) / kThreads;
  const int b0 = min(a.B, (int)threadIdx.x * per), b1 = min(a.B, b0 + per);
  auto ctx_of = [&](int b) { return (int)max((int64_t)0, min(cap, (int64_t)__ldg(a.ctx + b))); };
  auto pages = [&](int64_t tokens) { return (int64_t)a.by_bs.div((uint32_t)(tokens + a.bs - 1)); };

  const int64_t head = max((int64_t)0, min(a.num_free, (int64_t)__ldg(a.head)));
  int64_t sum = 0, all;
  for (int b = b0; b < b1; ++b) {
    const int n = max(0, __ldg(a.fresh + b));
    at[b] = n;
    sum += n;
  }
  int64_t run = block_scan(sum, &all, warp_sums[0]);
  sum = 0;
  for (int b = b0; b < b1; ++b) {
    const int64_t lo = min((int64_t)a.N, run), ctx = ctx_of(b);
    run += at[b];
    const int64_t want = min(min((int64_t)a.N, run) - lo, cap - ctx);
    cu[b] = (int32_t)lo;
    fits[b] = (int32_t)want;
    sum += pages(ctx + want) - pages(ctx);
  }
  if (threadIdx.x == 0) cu[a.B] = (int32_t)min((int64_t)a.N, all);
  run = head + block_scan(sum, &all, warp_sums[1]);
  for (int b = b0; b < b1; ++b) {
    const int64_t ctx = ctx_of(b), held = pages(ctx), need = pages(ctx + fits[b]) - held;
    const int64_t have = max((int64_t)0, min(need, a.num_free - run));
    fits[b] = (int32_t)min((int64_t)fits[b], (held + have) * a.bs - ctx);
    at[b] = (int32_t)(min(run, a.num_free) - held);  // the list's entry for page 0, were it in it
    run += need;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int b = threadIdx.x; b <= a.B; b += kThreads) {
      a.cu[b] = cu[b];
      if (b < a.B) a.ctx_out[b] = ctx_of(b) + fits[b];
    }
    if (threadIdx.x == 0) *a.head_out = (int32_t)min(head + all, a.num_free);
  }

  const int total = cu[a.B];
  for (int64_t i0 = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * V; i0 < a.N;
       i0 += (int64_t)gridDim.x * kThreads * V) {
    long long slot[V];
    int pos[V];
    int b = 0, end = 0, ctx = 0, seen = -1, page = 0;  // the request, where it ends, the last page looked up
    bool found = false;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i = (int)i0 + j;
      slot[j] = -1;
      pos[j] = 0;
      if (i >= total) continue;
      if (!found || i >= end) {  // the last b with cu[b] <= i: the one that holds token i (empty ones lie before it)
        int lo = found ? b : 0, hi = a.B;
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (cu[mid] <= i) lo = mid;
          else hi = mid;
        }
        b = lo;
        end = cu[b + 1];
        ctx = ctx_of(b);
        found = true;
        seen = -1;
      }
      const int off = i - cu[b];
      if (off >= fits[b]) continue;
      const int p = ctx + off, pi = (int)a.by_bs.div((uint32_t)p);
      if (!SA_DCHECK(pi < a.max_blocks)) continue;
      if (pi != seen) {
        int32_t* entry = a.table + b * a.ld + pi;
        if (pi * a.bs < ctx) {  // a page that the request held already
          page = *entry;
        } else {
          page = __ldg(a.pool + at[b] + pi);
          if (p == pi * a.bs) *entry = page;
        }
        if (page < 0) atomicAdd(&g_bad_entries, 1u);  // its tokens have no slot
        seen = pi;
      }
      pos[j] = p;
      if (page >= 0) slot[j] = (long long)page * a.bs + (p - pi * a.bs);
    }
    if constexpr (V == 4) {
      if (i0 + 4 <= a.N) {  // (both buffers start on 16 bytes)
        *reinterpret_cast<int4*>(a.positions + i0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
        *reinterpret_cast<longlong2*>(a.slots + i0) = make_longlong2(slot[0], slot[1]);
        *reinterpret_cast<longlong2*>(a.slots + i0 + 2) = make_longlong2(slot[2], slot[3]);
        continue;
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (i0 + j < a.N) {
        a.positions[i0 + j] = pos[j];
        a.slots[i0 + j] = slot[j];
      }
    }
  }
}

struct ReleaseArgs {
  const int32_t* table;
  int64_t ld;
  const int32_t* ctx;
  const uint8_t* done;
  int32_t* pool;
  const int32_t* head;
  int32_t* ctx_out;
  int32_t* head_out;
  int64_t num_free;
  int B, max_blocks, bs;
};

// Every block scans the ended requests' page counts; a warp copies one
// request's pages to the list's entries in front of its head.
__global__ void __launch_bounds__(kThreads) paged_release_kernel(ReleaseArgs a) {
  extern __shared__ int64_t off[];  // [B]
  __shared__ int64_t warp_sums[kThreads / 32];
  const int64_t cap = (int64_t)a.max_blocks * a.bs;
  const int per = (a.B + kThreads - 1) / kThreads;
  const int b0 = min(a.B, (int)threadIdx.x * per), b1 = min(a.B, b0 + per);
  auto pages_of = [&](int b) {
    return a.done[b] ? (int)((max((int64_t)0, min(cap, (int64_t)a.ctx[b])) + a.bs - 1) / a.bs) : 0;
  };
  int64_t sum = 0, all;
  for (int b = b0; b < b1; ++b) sum += pages_of(b);
  int64_t run = block_scan(sum, &all, warp_sums);
  for (int b = b0; b < b1; ++b) {
    off[b] = run;
    run += pages_of(b);
  }
  __syncthreads();
  const int64_t head = max((int64_t)0, min(a.num_free, (int64_t)*a.head));
  const int64_t first = head - all;
  if (blockIdx.x == 0) {
    for (int b = threadIdx.x; b < a.B; b += kThreads) a.ctx_out[b] = a.done[b] ? 0 : a.ctx[b];
    if (threadIdx.x == 0) {
      *a.head_out = (int32_t)max((int64_t)0, first);
      if (first < 0) atomicAdd(&g_bad_entries, 1u);  // more pages than the pool had given out
    }
  }
  const int lane = threadIdx.x & 31;
  for (int64_t b = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); b < a.B;
       b += (int64_t)gridDim.x * (kThreads / 32)) {
    const int n = pages_of((int)b);
    bool none = false;
    for (int j = lane; j < n; j += 32) {
      const int64_t to = first + off[b] + j;
      if (to >= 0 && SA_DCHECK(to < a.num_free && j < a.max_blocks)) {
        const int32_t page = a.table[b * a.ld + j];
        none |= page < 0;
        a.pool[to] = page;
      }
    }
    if (none) atomicAdd(&g_bad_entries, 1u);  // the list is short of a page
  }
}

// 64-bit lengths and pages as 32-bit ones; what does not fit stays out of range.  (One launch,
// as torch's conversion: with a clamp of torch's in front a call of two such tensors took 72 us
// for 55.)
__global__ void __launch_bounds__(256) narrow_kernel(const long long* src, int32_t* dst, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    dst[i] = (int32_t)max(-1ll, min((long long)INT32_MAX, src[i]));
}

// ---- append -------------------------------------------------------------------

using namespace qkr;

struct AppendSide {
  const void* x;
  const void* w;
  int64_t xt, xh;   // token and head strides
  int64_t units;    // groups * per
  int64_t warp0;    // first warp of this side
  int H, C, per;    // heads, heads of a unit, units of a token group
};

struct AppendArgs {
  AppendSide s[3];  // q, k, v
  void* q_out;      // [N, Hq, D]
  void* cache[2];   // k, v: [num_blocks, Hkv, bs, D]
  const long long* slots;
  int64_t N, num_slots, warps;
  int w_dtype, bs;
  FastDiv by_bs;
};

constexpr int kAppendRing = 8, kAppendBlocks = 3;  // 33 KB and 168 registers a thread (at 128 it spills: 46 us for 39)

// A token's position; a padding token's (its slot is negative) says nothing and counts as 0.
template <int L> struct Where {
  const Tables& tb;
  const AppendArgs& a;
  struct Pos {
    RawInt pos, slot;
  };
  __device__ __forceinline__ bool fetch(int64_t group, Pos& p) const {
    const int64_t n = group * (32 / L) + (threadIdx.x & 31) / L;
    if (n >= a.N || tb.R == 0) return false;
    p.slot.load(a.slots, 8, n);
    if (tb.pos_bytes) p.pos.load(tb.pos, tb.pos_bytes, n);
    else p.pos.v = make_uint2((uint32_t)n, 0);
    return true;
  }
  __device__ __forceinline__ int64_t get(const Pos& p) const {
    return p.slot.get(8) < 0 ? 0 : p.pos.get(tb.pos_bytes);
  }
};

template <typename E, int L, bool Partial>
__global__ void __launch_bounds__(kWalkThreads, kAppendBlocks) qk_norm_rope_append(AppendArgs a, Tables tb) {
  extern __shared__ __align__(16) uint4 ring[];
  const int64_t warp = (int64_t)blockIdx.x * (kWalkThreads / 32) + (threadIdx.x >> 5);
  const int side = warp >= a.s[2].warp0 ? 2 : warp >= a.s[1].warp0 ? 1 : 0;
  const AppendSide& sd = a.s[side];
  const int64_t warps = (side == 2 ? a.warps : a.s[side + 1].warp0) - sd.warp0;
  const Units un = make_units(warp - sd.warp0, warps, sd.units, sd.H, sd.C, sd.per);
  if (un.count == 0) return;
  const Lane ln = lane_of<E, L>(tb);
  auto token = [&](int64_t g) { return g * (32 / L) + (threadIdx.x & 31) / L; };
  const Where<L> where{tb, a};
  Angles<E, Where<L>> ang(tb, ln, &g_bad_entries, un, where);
  Map map;
  E* y = nullptr;  // the row that comes next
  int64_t yh = 0;
  RawInt next_slot;
  Cursor slot_ahead(un);  // of next_slot
  int64_t more_slots = un.count - 1;
  auto ask_slot = [&]() {
    const int64_t n = token(slot_ahead.group);
    if (n < a.N) next_slot.load(a.slots, 8, n);
  };
  bool write = false, padding = false;
  walk_rows<E, 1, kAppendRing>(
      un, ln, ring,
      [&](int64_t g) {
        const int64_t n = token(g);
        return Source<E, 1>{{static_cast<const E*>(sd.x) + (n < a.N ? n : 0) * sd.xt}, {sd.xh}, ln.active && n < a.N};
      },
      [&]() {
        ask_slot();
        if (side < 2) ang.begin();
      },
      [&](int64_t g, int h) {
        if (side < 2) {
          float2 c[4], s[4], w1[4], w2[4];
          load_weights<E>(sd.w, a.w_dtype, ln, w1, w2);
          ang.enter(c, s);
          map.make(c, s, w1, w2);
        }
        const int64_t n = token(g);
        int64_t slot = n < a.N ? next_slot.get(8) : -1;
        if (more_slots-- > 0) {
          slot_ahead.next(un);
          ask_slot();
        }
        if (slot >= a.num_slots) {
          if (side == 1 && ln.o1 == 0) atomicAdd(&g_bad_entries, 1u);  // (by k's warps: there may be no query heads)
          slot = -1;
        }
        padding = slot < 0;
        if (side == 0) {  // a padding token's q row is zeros
          write = ln.active && n < a.N;
          y = static_cast<E*>(a.q_out) + n * sd.H * tb.D;
          yh = tb.D;
        } else {
          write = ln.active && !padding;
          const int64_t page = padding ? 0 : slot <= INT32_MAX ? (int64_t)a.by_bs.div((uint32_t)slot) : slot / a.bs;
          y = static_cast<E*>(a.cache[side - 1]) + (page * sd.H * a.bs + (padding ? 0 : slot - page * a.bs)) * tb.D;
          yh = (int64_t)a.bs * tb.D;
        }
        y += h * yh + ln.o1;
      },
      [&](Raw8<E> (&rows)[2]) {
        if (side < 2) norm_rope<E, L, Partial>(tb, ln, map, rows[0], rows[1]);
        if (padding) rows[0].zero(), rows[1].zero();
        if (write && SA_DCHECK(ln.o2 + ln.ps + 4 <= tb.D)) {
          rows[0].store(y, ln.ps);
          rows[1].store(y + (ln.o2 - ln.o1), ln.ps);
        }
        y += yh;
      });
}

// Dynamic shared memory of the requests' scans.  The kernels are opted in to the largest
// batch's once: the limit is the kernel's, and set to each call's own size another thread's
// larger launch between that and its own was refused.
constexpr int assign_smem(int64_t B) { return (int)((3 * B + 1) * 4); }
constexpr int release_smem(int64_t B) { return (int)std::max<int64_t>(B, 1) * 8; }

template <typename E, int L, bool Partial>
static int launch_append_lp(const AppendArgs& a, const Tables& tb, cudaStream_t st) {
  constexpr int smem = Ring<E, 1, kAppendRing>::kBytesPerThread * kWalkThreads;
  static_assert(smem <= 56 * 1024, "three blocks an SM");
  const int rc = sa_record_cuda_error(opt_in_once<&qk_norm_rope_append<E, L, Partial>, smem>());
  if (rc != SA_OK) return rc;
  const unsigned blocks = (unsigned)(a.warps / (kWalkThreads / 32));
  qk_norm_rope_append<E, L, Partial><<<blocks, kWalkThreads, smem, st>>>(a, tb);
  return sa_record_cuda_error(cudaGetLastError());
}

template <typename E, int L>
static int launch_append_l(const AppendArgs& a, const Tables& tb, cudaStream_t st) {
  return tb.R < tb.D ? launch_append_lp<E, L, true>(a, tb, st) : launch_append_lp<E, L, false>(a, tb, st);
}

template <typename E>
static int launch_append(const AppendArgs& a, const Tables& tb, cudaStream_t st) {
  switch (lanes_for(tb.D)) {
    case 1: return launch_append_l<E, 1>(a, tb, st);
    case 2: return launch_append_l<E, 2>(a, tb, st);
    case 4: return launch_append_l<E, 4>(a, tb, st);
    case 8: return launch_append_l<E, 8>(a, tb, st);
    default: return launch_append_l<E, 16>(a, tb, st);
  }
}

static int check_requests(int64_t B, int64_t max_blocks, int64_t bs, int64_t ld, int64_t num_free) {
  if (B < 0 || max_blocks <= 0 || bs <= 0 || ld < max_blocks || num_free < 0) return SA_ERR_ARG;
  if (B > kMaxRequests || max_blocks > INT32_MAX || bs > (1 << 16) || max_blocks * bs > ((int64_t)1 << 30) ||
      num_free > INT32_MAX)
    return SA_ERR_UNSUPPORTED;
  return SA_OK;
}

}  // namespace pgc

int paged_cache_bad_entries(int reset, cudaStream_t st) {
  unsigned v = 0;
  cudaMemcpyFromSymbolAsync(&v, pgc::g_bad_entries, sizeof(v), 0, cudaMemcpyDeviceToHost, st);
  cudaStreamSynchronize(st);
  if (reset) {
    const unsigned z = 0;
    cudaMemcpyToSymbolAsync(pgc::g_bad_entries, &z, sizeof(z), 0, cudaMemcpyHostToDevice, st);
    cudaStreamSynchronize(st);
  }
  return (int)v;
}

}  // namespace sa

extern "C" int sa_paged_assign_slots(int32_t* block_table, int64_t table_stride, const int32_t* context_lens,
                                     const int32_t* new_lens, const int32_t* free_pages, int64_t num_free,
                                     const int32_t* free_head, int64_t* slots, int32_t* positions,
                                     int32_t* cu_seqlens, int32_t* context_lens_out, int32_t* free_head_out,
                                     int64_t B, int64_t num_tokens, int64_t max_blocks, int64_t block_size,
                                     void* stream) {
  using namespace sa::pgc;
  const int rc = check_requests(B, max_blocks, block_size, table_stride, num_free);
  if (rc != SA_OK) return rc;
  if (num_tokens < 0) return SA_ERR_ARG;
  if (num_tokens > INT32_MAX - kThreads) return SA_ERR_UNSUPPORTED;
  if (!free_head || !cu_seqlens || !free_head_out) return SA_ERR_ARG;
  if (B > 0 && (!block_table || !context_lens || !new_lens || !context_lens_out)) return SA_ERR_ARG;
  if (num_free > 0 && !free_pages) return SA_ERR_ARG;
  if (num_tokens > 0 && (!slots || !positions)) return SA_ERR_ARG;
  if (!sa::qkr::al16(slots) || !sa::qkr::al16(positions)) return SA_ERR_ALIGN;
  AssignArgs a{block_table, table_stride, context_lens, new_lens, free_pages, free_head,
               reinterpret_cast<long long*>(slots), positions, cu_seqlens, context_lens_out, free_head_out, num_free,
               (int)B, (int)num_tokens, (int)max_blocks, (int)block_size,
               sa::qkr::FastDiv((uint32_t)block_size)};
  // one token a thread where half a wave (two blocks an SM) holds them, else four in equal rounds
  const int64_t wave = 2ll * sm_count();
  const bool few = num_tokens <= wave * kThreads / 2;
  const int64_t each = few ? kThreads : 4 * kThreads;
  const int64_t tiles = std::max<int64_t>(1, (num_tokens + each - 1) / each), rounds = (tiles + wave - 1) / wave;
  const unsigned blocks = (unsigned)((tiles + rounds - 1) / rounds);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int orc = sa_record_cuda_error(few ? opt_in_once<&paged_assign_kernel<1>, assign_smem(kMaxRequests)>()
                                           : opt_in_once<&paged_assign_kernel<4>, assign_smem(kMaxRequests)>());
  if (orc != SA_OK) return orc;
  if (few) paged_assign_kernel<1><<<blocks, kThreads, assign_smem(B), st>>>(a);
  else paged_assign_kernel<4><<<blocks, kThreads, assign_smem(B), st>>>(a);
  return sa_record_cuda_error(cudaGetLastError());
}

extern "C" int sa_paged_release_pages(const int32_t* block_table, int64_t table_stride, const int32_t* context_lens,
                                      const uint8_t* done, int32_t* free_pages, int64_t num_free,
                                      const int32_t* free_head, int32_t* context_lens_out, int32_t* free_head_out,
                                      int64_t B, int64_t max_blocks, int64_t block_size, void* stream) {
  using namespace sa::pgc;
  const int rc = check_requests(B, max_blocks, block_size, table_stride, num_free);
  if (rc != SA_OK) return rc;
  if (!free_head || !free_head_out) return SA_ERR_ARG;
  if (B > 0 && (!block_table || !context_lens || !done || !context_lens_out)) return SA_ERR_ARG;
  if (num_free > 0 && !free_pages) return SA_ERR_ARG;
  ReleaseArgs a{block_table, table_stride, context_lens, done, free_pages, free_head, context_lens_out, free_head_out,
                num_free, (int)B, (int)max_blocks, (int)block_size};
  const int orc = sa_record_cuda_error(opt_in_once<&paged_release_kernel, release_smem(kMaxRequests)>());
  if (orc != SA_OK) return orc;
  const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>((B + 15) / 16, sm_count()));
  paged_release_kernel<<<(unsigned)blocks, kThreads, release_smem(B), static_cast<cudaStream_t>(stream)>>>(a);
  return sa_record_cuda_error(cudaGetLastError());
}

extern "C" int sa_narrow_i64(const int64_t* src, int32_t* dst, int64_t n, void* stream) {
  using namespace sa::pgc;
  if (n < 0) return SA_ERR_ARG;
  if (n == 0) return SA_OK;
  if (!src || !dst) return SA_ERR_ARG;
  const int64_t blocks = std::min<int64_t>((n + 255) / 256, 8ll * sm_count());
  narrow_kernel<<<(unsigned)blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      reinterpret_cast<const long long*>(src), dst, n);
  return sa_record_cuda_error(cudaGetLastError());
}

extern "C" int sa_qk_norm_rope_paged_append(const void* q, const void* k, const void* v, void* q_out, void* k_cache,
                                            void* v_cache, const int64_t* slots, const void* q_weight,
                                            const void* k_weight, int w_dtype, const void* cos_table,
                                            const void* sin_table, int cs_dtype, const void* positions,
                                            int pos_bytes, int64_t num_pos, int64_t N, int64_t Hq, int64_t Hkv,
                                            int64_t D, int64_t rotary_dim, int64_t num_blocks, int64_t block_size,
                                            const int64_t* q_strides, const int64_t* k_strides,
                                            const int64_t* v_strides, float eps, int normalize, int dtype,
                                            void* stream) {
  using namespace sa::pgc;
  if (N < 0 || Hq < 0 || Hkv <= 0 || num_blocks < 0 || block_size <= 0) return SA_ERR_ARG;
  if (dtype != SA_BF16 && dtype != SA_F16) return SA_ERR_UNSUPPORTED;
  if (Hq > (1 << 20) || Hkv > (1 << 20) || N > ((int64_t)1 << 33) || block_size > (1 << 16) ||
      num_blocks > ((int64_t)1 << 40))
    return SA_ERR_UNSUPPORTED;
  sa::qkr::Tables tb;
  const int rc = sa::qkr::make_tables(&tb, cos_table, sin_table, cs_dtype, positions, pos_bytes, 0, num_pos, N, D,
                                      rotary_dim, eps, normalize, q_weight, k_weight, w_dtype);
  if (rc != SA_OK) return rc;
  if (N == 0) return SA_OK;
  if (!slots || !q_strides || !k_strides || !v_strides || !k || !v || (Hq > 0 && (!q || !q_out)) ||
      (num_blocks > 0 && (!k_cache || !v_cache)))
    return SA_ERR_ARG;
  using sa::qkr::al16;
  if (!al16(q) || !al16(k) || !al16(v) || !al16(q_out) || !al16(k_cache) || !al16(v_cache)) return SA_ERR_ALIGN;
  const int64_t* st3[3] = {q_strides, k_strides, v_strides};
  for (const int64_t* s : st3)
    if (s[2] != 1 || s[0] % 8 != 0 || s[1] % 8 != 0) return SA_ERR_ALIGN;
  AppendArgs a;
  const int per = 32 / sa::qkr::lanes_for(D);
  const int64_t groups = (N + per - 1) / per;
  a.N = N;
  a.num_slots = num_blocks * block_size;
  a.w_dtype = w_dtype;
  a.bs = (int)block_size;
  a.by_bs = sa::qkr::FastDiv((uint32_t)block_size);
  a.q_out = q_out;
  a.cache[0] = k_cache;
  a.cache[1] = v_cache;
  a.slots = reinterpret_cast<const long long*>(slots);
  const void* xs[3] = {q, k, v};
  const void* ws[3] = {normalize ? q_weight : nullptr, normalize ? k_weight : nullptr, nullptr};  // else n = x
  const int C = sa::qkr::unit_heads(groups * (Hq + 2 * Hkv), (int64_t)kAppendBlocks * sa::qkr::sm_count() * (sa::qkr::kWalkThreads / 32));
  int64_t units = 0;
  for (int i = 0; i < 3; ++i) {
    a.s[i].x = xs[i];
    a.s[i].w = ws[i];
    a.s[i].xt = st3[i][0];
    a.s[i].xh = st3[i][1];
    a.s[i].H = (int)(i == 0 ? Hq : Hkv);
    a.s[i].C = C;
    a.s[i].per = (a.s[i].H + C - 1) / C;
    a.s[i].units = groups * a.s[i].per;
    units += a.s[i].units;
  }
  // warps by each side's share of the work, at least one where it has any (four warps a block: always enough)
  a.warps = sa::qkr::walk_blocks(units, kAppendBlocks) * (sa::qkr::kWalkThreads / 32);
  const double cq = sa::qkr::walk_cost(groups * Hq, a.s[0].units), ck = sa::qkr::walk_cost(groups * Hkv, a.s[1].units);
  const int64_t q_warps = (int64_t)((double)a.warps * cq / (cq + 2 * ck) + 0.5);
  const int64_t qk_warps = (int64_t)((double)a.warps * (cq + ck) / (cq + 2 * ck) + 0.5);
  a.s[0].warp0 = 0;
  a.s[1].warp0 = std::min<int64_t>(a.warps - 2, std::max<int64_t>(Hq > 0, q_warps));
  a.s[2].warp0 = std::min<int64_t>(a.warps - 1, std::max<int64_t>(a.s[1].warp0 + 1, qk_warps));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == SA_BF16 ? launch_append<__nv_bfloat16>(a, tb, st) : launch_append<__half>(a, tb, st);
}
SA_BOUNDS_ACCESSOR(paged_cache_bounds)
