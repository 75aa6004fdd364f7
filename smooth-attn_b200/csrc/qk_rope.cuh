// One head row of queries or keys: its root-mean-square norm and the rotation
// of its position, shared by the training operator (qk_norm_rope.cu) and the
// append into a paged cache (paged_cache.cu).
//
//   n = x * rsqrt(mean(x^2) + eps) * w            (over the row's D channels)
//   y[i]       = n[i] c_i - n[i + R/2] s_i        i < R/2, c, s of the row's position
//   y[i + R/2] = n[i + R/2] c_i + n[i] s_i
//   y[j]       = n[j]                             R <= j < D
//
// A row belongs to L = 1, 2, 4, 8 or 16 neighbouring lanes of a warp, each
// with two 8-element chunks that the rotation pairs (16-bit: x[8g..], x[R/2 + 8g..]),
// so the rotation needs no exchange and the norm's sum log2(L) shuffles.
// Everything between the loads and the one rounding of y is fp32.
#pragma once

#include <stdint.h>

#include <atomic>

#include "sa_common.cuh"

namespace sa {
namespace qkr {

// 8 elements of E as they lie in memory, and as fp32 pairs (the arithmetic runs
// in packed two-element instructions: with scalar ones the forward was bound by
// issue slots at 0.75 of HBM's rate).
template <typename E> struct Raw8 {
  uint4 u[sizeof(E) / 2];
  __device__ __forceinline__ void load(const E* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(E) / 2; ++i) u[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (int)sizeof(E) / 2; ++i) u[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void get(float2 (&f)[4]) const {
    float g[8];
    unpack<E, 8>(u, g);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = make_float2(g[2 * i], g[2 * i + 1]);
  }
  __device__ __forceinline__ void set(const float2 (&f)[4]) {
    if constexpr (sizeof(E) == 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        u[i] = make_uint4(__float_as_uint(f[2 * i].x), __float_as_uint(f[2 * i].y), __float_as_uint(f[2 * i + 1].x),
                          __float_as_uint(f[2 * i + 1].y));
    } else if constexpr (std::is_same<E, __nv_bfloat16>::value) {
      __nv_bfloat162 h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = __float22bfloat162_rn(f[i]);
      u[0] = *reinterpret_cast<const uint4*>(h);
    } else {
      __half2 h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = __float22half2_rn(f[i]);
      u[0] = *reinterpret_cast<const uint4*>(h);
    }
  }
  __device__ __forceinline__ void store(E* p) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(E) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = u[i];
  }
  // fp32: the second 4 elements ps behind the first (16-bit: all 8 together, ps is 4)
  __device__ __forceinline__ void store(E* p, int ps) const {
    *reinterpret_cast<uint4*>(p) = u[0];
    if constexpr (sizeof(E) == 4) *reinterpret_cast<uint4*>(p + ps) = u[1];
  }
};

// The 8 elements of a table or weight that go with a lane's chunk, of a type known
// at run time (one uniform branch): 4 at `at` and 4 at `at + ps`, neighbours but for
// fp32 rows (see Lane).
template <typename E>
__device__ __forceinline__ void raw8_any(const void* p, int64_t at, int ps, int dtype, uint4& lo, uint4& hi) {
  if (dtype == SA_F32) {
    lo = __ldg(reinterpret_cast<const uint4*>(static_cast<const float*>(p) + at));
    hi = __ldg(reinterpret_cast<const uint4*>(static_cast<const float*>(p) + at + ps));
  } else if constexpr (sizeof(E) == 4) {
    const uint2 a = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + at));
    const uint2 b = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + at + ps));
    lo = make_uint4(a.x, a.y, b.x, b.y);
  } else {
    lo = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at));
  }
}
__device__ __forceinline__ void open8_any(const uint4& lo, const uint4& hi, int dtype, float2 (&f)[4]) {
  if (dtype == SA_F32) {
    Raw8<float> r;
    r.u[0] = lo, r.u[1] = hi;
    r.get(f);
  } else if (dtype == SA_BF16) {
    Raw8<__nv_bfloat16> r;
    r.u[0] = lo;
    r.get(f);
  } else {
    Raw8<__half> r;
    r.u[0] = lo;
    r.get(f);
  }
}

// What a lane owns of every row, and the tables it reads.
struct Tables {
  const void* cosv;
  const void* sinv;
  const void* pos;    // nullable: the token's index along T
  int64_t num_pos;    // rows of the tables
  int64_t pos_sb;     // stride of pos between batches (0: one row for all)
  int cs_dtype;
  int pos_bytes;      // 0, 4 or 8
  int D, R;
  int normalize;
  float eps, inv_d;
};

// A chunk is two groups of 4 elements: neighbours in 16-bit rows (16 bytes in
// all); in fp32 rows, 16 bytes each, a group's lanes apart, so that one
// instruction's lanes read whole 32-byte sectors.
struct Lane {
  int o1, o2;     // offsets of the lane's two chunks in the row
  int ps;         // from a chunk's first group to its second
  bool active;    // the lane has a chunk at all (D / 16 need not be a power of two)
  bool rotated;   // its chunks are a rotated pair
};

template <typename E, int L>
__device__ __forceinline__ Lane lane_of(const Tables& t) {
  constexpr int kStep = sizeof(E) == 4 ? 4 : 8;
  const int g = (threadIdx.x & 31) % L, nr = t.R / 16;
  Lane l;
  l.active = g < t.D / 16;
  l.rotated = g < nr;
  l.o1 = l.rotated ? kStep * g : t.R + kStep * (g - nr);
  l.o2 = l.o1 + (l.rotated ? t.R : t.D - t.R) / 2;
  l.ps = sizeof(E) == 4 ? (l.rotated ? t.R : t.D - t.R) / 4 : 4;
  return l;
}

// A 4- or 8-byte integer as loaded, so that a load can be issued long before its
// value is looked at (a conversion beside the load would wait for it).
struct RawInt {
  uint2 v;
  __device__ __forceinline__ void load(const void* p, int bytes, int64_t at) {
    if (bytes == 8) v = __ldg(static_cast<const uint2*>(p) + at);
    else v.x = __ldg(static_cast<const unsigned*>(p) + at);
  }
  __device__ __forceinline__ int64_t get(int bytes) const {
    return bytes == 8 ? (int64_t)(((uint64_t)v.y << 32) | v.x) : (int64_t)(int)v.x;
  }
};

// Sum over the L lanes of a row; every lane of the warp takes part.
template <int L> __device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int m = L / 2; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

__device__ __forceinline__ float2 splat(float v) { return make_float2(v, v); }

// The forward map of a token's rows for one lane's channels, the weights folded
// into the rotation: y1 = r (x1 a1 - x2 b1), y2 = r (x2 a2 + x1 b2).
struct Map {
  float2 a1[4], b1[4], a2[4], b2[4];  // w1 c, -w2 s, w2 c, w1 s
  __device__ __forceinline__ void make(const float2 (&c)[4], const float2 (&s)[4], const float2 (&w1)[4],
                                       const float2 (&w2)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a1[i] = fmul2(w1[i], c[i]);
      b1[i] = fmul2(w2[i], make_float2(-s[i].x, -s[i].y));
      a2[i] = fmul2(w2[i], c[i]);
      b2[i] = fmul2(w1[i], s[i]);
    }
  }
};

// v where the lane's chunks are a rotated pair, else `none`: -0 in a sum, 0 behind a minus, which leave even the
// sign of a zero alone.
__device__ __forceinline__ float2 pair_only(const Lane& l, float2 v, float none) {
  return make_float2(l.rotated ? v.x : none, l.rotated ? v.y : none);
}

// y of one row from its two raw chunks (zeros in lanes without one).  Partial:
// some channels are not rotated, and there the other one of the pair is left out:
// times a sine of 0 an infinity in it would arrive as NaN.  (The selects cost rows of
// 80 channels of which 16 are rotated 3 to 4 %, a branch 5 to 8 %; rows
// that are rotated throughout need none, hence the parameter: with a branch for all the
// backward of [4, 32 + 8, 4096, 128] took 90 us for 87.5.)
template <typename E, int L, bool Partial>
__device__ __forceinline__ void norm_rope(const Tables& t, const Lane& l, const Map& m, Raw8<E>& a, Raw8<E>& b) {
  float2 x1[4], x2[4], y1[4], y2[4];
  a.get(x1);
  b.get(x2);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 t1 = fmul2(x2[i], m.b1[i]), t2 = fmul2(x1[i], m.b2[i]);
    if constexpr (Partial) t1 = pair_only(l, t1, -0.f), t2 = pair_only(l, t2, -0.f);
    y1[i] = ffma2(x1[i], m.a1[i], t1);
    y2[i] = ffma2(x2[i], m.a2[i], t2);
  }
  if (t.normalize) {
    float2 ss = fmul2(x1[0], x1[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) ss = ffma2(x1[i], x1[i], ss);
#pragma unroll
    for (int i = 0; i < 4; ++i) ss = ffma2(x2[i], x2[i], ss);
    const float2 r = splat(rsqrtf(fmaf(row_sum<L>(ss.x + ss.y), t.inv_d, t.eps)));
#pragma unroll
    for (int i = 0; i < 4; ++i) y1[i] = fmul2(y1[i], r), y2[i] = fmul2(y2[i], r);
  }
  a.set(y1);
  b.set(y2);
}

template <typename E>
__device__ __forceinline__ void load_weights(const void* w, int w_dtype, const Lane& l, float2 (&w1)[4],
                                             float2 (&w2)[4]) {
  if (w != nullptr && l.active) {
    uint4 a, b, c, d;
    raw8_any<E>(w, l.o1, l.ps, w_dtype, a, b);
    raw8_any<E>(w, l.o2, l.ps, w_dtype, c, d);
    open8_any(a, b, w_dtype, w1);
    open8_any(c, d, w_dtype, w2);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) w1[i] = w2[i] = splat(1.f);
  }
}

// ---- the walk over rows ----------------------------------------------------------

// The rows are cut into units: a token group (32 / L neighbouring tokens, one
// row per L lanes) and C neighbouring heads.  Warp w of W takes units w, w + W,
// ..., so what all warps read and write at a time lies close together.  Inside a
// unit an item is one head.  Every lane streams its own 16-byte chunks of the rows
// through a private ring in shared memory with cp.async, RING - 1 items ahead:
// the bytes in flight then cost no registers (with plain loads 128 registers a
// thread held only one item's), and since a lane reads only what it copied
// itself there is no barrier, only its own wait.
// (A plain contiguous range per warp ran the backward at 0.77 of HBM's rate, these
// interleaved units at 0.92: the pages of memory in use at a time are few.)
struct Units {
  int64_t step_group;  // step = step_group * per + step_part
  int64_t group0;      // this warp's first unit
  int64_t count;       // and how many it has
  int part0, step_part;
  int H, C, per;       // heads, heads of a unit, units of a group
};

__device__ __forceinline__ Units make_units(int64_t first, int64_t step, int64_t all, int H, int C, int per) {
  Units u;
  u.count = first < all ? (all - first - 1) / step + 1 : 0;
  u.group0 = first / per;
  u.part0 = (int)(first - u.group0 * per);
  u.step_group = step / per;
  u.step_part = (int)(step - u.step_group * per);
  u.H = H, u.C = C, u.per = per;
  return u;
}

// A place in a warp's units (no division on the way).
struct Cursor {
  int64_t group;
  int part;
  __device__ __forceinline__ explicit Cursor(const Units& u) : group(u.group0), part(u.part0) {}
  __device__ __forceinline__ void next(const Units& u) {
    group += u.step_group;
    part += u.step_part;
    if (part >= u.per) part -= u.per, ++group;
  }
};

constexpr int kWalkThreads = 128;

template <typename E, int NSRC> struct Source {
  const E* base[NSRC];  // the lane's token, head 0
  int64_t hs[NSRC];     // head strides
  bool on;              // the lane has a chunk of an existing token
};

template <typename E, int NSRC, int RING> struct Ring {
  static constexpr int kChunk = sizeof(E) / 2;                 // 16-byte pieces of 8 elements
  static constexpr int kPieces = NSRC * 2 * kChunk;       // pieces a lane copies per item
  static constexpr int kBytesPerThread = RING * kPieces * 16;
};

// 16 bytes to shared memory, or zeros (nothing is read) where !valid.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}

// ring: the block's shared memory, blockDim.x * kBytesPerThread bytes.
// source(group) gives a group's Source; begin() is called after the first rows
// were asked for, enter(group, head) when the walk comes to a unit, use(rows) for
// each of the unit's heads in order, with the 2 * NSRC raw chunks (zeros where
// Source.on is false).  All are called by the whole warp.
template <typename E, int NSRC, int RING, class FSource, class FBegin, class FEnter, class FUse>
__device__ __forceinline__ void walk_rows(const Units& un, const Lane& ln, uint4* ring, FSource&& source,
                                          FBegin&& begin, FEnter&& enter, FUse&& use) {
  using R = Ring<E, NSRC, RING>;
  if (un.count <= 0) return;
  constexpr uint32_t kSlot = kWalkThreads * 16, kStage = R::kPieces * kSlot;
  const uint32_t mine = smem_u32(ring) + threadIdx.x * 16;
  Cursor ahead(un);           // unit of the next item to ask for
  int64_t more = un.count;    // units not yet wholly asked for
  int pn = 0;                 // heads of `ahead` not yet asked for
  const E* at[NSRC];
  int64_t hs[NSRC];
  bool on = false;
  const int d12 = ln.o2 - ln.o1;
  auto open = [&]() {
    const int h = ahead.part * un.C;
    const Source<E, NSRC> src = source(ahead.group);
    on = src.on;
    pn = min(un.C, un.H - h);
#pragma unroll
    for (int k = 0; k < NSRC; ++k) {
      hs[k] = src.hs[k];
      at[k] = src.base[k] + h * hs[k] + ln.o1;
    }
  };
  open();
  uint32_t ask_slot = mine, use_slot = mine;
  auto ask = [&]() {
    if (more > 0) {
#pragma unroll
      for (int k = 0; k < NSRC; ++k) {
        const uint32_t to = ask_slot + k * 2 * R::kChunk * kSlot;
#pragma unroll
        for (int c = 0; c < R::kChunk; ++c) {
          cp_async16(to + c * kSlot, at[k] + c * ln.ps, on);
          cp_async16(to + (R::kChunk + c) * kSlot, at[k] + d12 + c * ln.ps, on);
        }
        at[k] += hs[k];
      }
      if (--pn == 0 && --more > 0) {
        ahead.next(un);
        open();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    ask_slot = ask_slot == mine + (RING - 1) * kStage ? mine : ask_slot + kStage;
  };
#pragma unroll
  for (int s = 0; s < RING - 1; ++s) ask();
  begin();
  Cursor cur(un);
  for (int64_t j = un.count; j > 0; --j, cur.next(un)) {
    const int h = cur.part * un.C;
    enter(cur.group, h);
    for (int n = min(un.C, un.H - h); n > 0; --n) {
      asm volatile("cp.async.wait_group %0;" ::"n"(RING - 2) : "memory");
      Raw8<E> rows[2 * NSRC];
#pragma unroll
      for (int k = 0; k < 2 * NSRC; ++k)
#pragma unroll
        for (int c = 0; c < R::kChunk; ++c) {
          uint4& v = rows[k].u[c];
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                       : "r"(use_slot + (k * R::kChunk + c) * kSlot)
                       : "memory");
        }
      use_slot = use_slot == mine + (RING - 1) * kStage ? mine : use_slot + kStage;
      ask();  // into the slot of the item before this one: its rows were used
      use(rows);
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");  // nothing of this walk is left in flight
}

// cos and sin of a walk's units, asked for one unit ahead (the position two
// ahead), so that entering a unit waits for neither.  Where.fetch(group, pos)
// loads what the lane's position there is made of (false: it has no token);
// Where.get(pos) is called a unit later.
template <typename E, class Where> struct Angles {
  const Tables& t;
  const Lane& l;
  unsigned* bad;
  const Units& un;
  const Where& where;
  Cursor ahead;     // of next
  int64_t more;     // units behind it
  typename Where::Pos next;
  bool next_on;
  uint4 raw[4];
  bool have;

  __device__ __forceinline__ Angles(const Tables& tb, const Lane& ln, unsigned* b, const Units& u, const Where& w)
      : t(tb), l(ln), bad(b), un(u), where(w), ahead(u), more(u.count - 1), next_on(false), have(false) {}
  // The first unit's, once the walk has asked for its first rows.
  __device__ __forceinline__ void begin() {
    next_on = where.fetch(ahead.group, next);
    step();
  }
  // Asks for the angles of `next`, and for the position behind it.
  __device__ __forceinline__ void step() {
    have = next_on && l.active && l.rotated;
    const int64_t pos = have ? where.get(next) : 0;
    next_on = false;
    if (more > 0) {
      ahead.next(un);
      --more;
      next_on = where.fetch(ahead.group, next);
    }
    if (!have) return;
    int64_t p = pos;
    if (p < 0 || p >= t.num_pos) {
      if (l.o1 == 0) atomicAdd(bad, 1u);
      p = 0;
    }
    const int64_t at = p * (t.R / 2) + l.o1;
    raw8_any<E>(t.cosv, at, l.ps, t.cs_dtype, raw[0], raw[1]);
    raw8_any<E>(t.sinv, at, l.ps, t.cs_dtype, raw[2], raw[3]);
  }
  // cos and sin of the unit that the walk enters.
  __device__ __forceinline__ void enter(float2 (&c)[4], float2 (&s)[4]) {
    if (!have) {
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = splat(1.f), s[i] = splat(0.f);
    } else {
      open8_any(raw[0], raw[1], t.cs_dtype, c);
      open8_any(raw[2], raw[3], t.cs_dtype, s);
    }
    step();
  }
};

// n / d for 0 <= n < 2^31 by a multiplication.
struct FastDiv {
  uint32_t d, mul, shift;
  __host__ FastDiv() : d(1), mul(0), shift(0) {}
  __host__ explicit FastDiv(uint32_t divisor) : d(divisor), mul(0), shift(0) {
    if (d <= 1) return;
    uint32_t bits = 0;
    while ((1ull << bits) < d) ++bits;  // 2^bits >= d
    // n mul / 2^(31 + bits) passes n / d by less than n / 2^(31 + bits) < 1 / d: the floors are the same
    mul = (uint32_t)(((1ull << (31 + bits)) + d - 1) / d);
    shift = bits - 1;
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return mul ? __umulhi(n, mul) >> shift : n; }
};

// ---- host side ----------------------------------------------------------------

inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// SMs of the current device (asked once per device: the query costs as much as a launch).
inline int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64) {
    n = known[dev].load(std::memory_order_relaxed);
    if (n > 0) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && n > 0) {
      known[dev].store(n, std::memory_order_relaxed);
      return n;
    }
  }
  cudaGetLastError();
  return 148;
}

// Opt-in of a kernel to a fixed `kBytes` of dynamic shared memory on the current
// device, once per kernel and device (the call costs as much as a third of a launch).
template <auto kKernel, int kBytes> inline cudaError_t opt_in_once() {
  if constexpr (kBytes > 48 * 1024) {
    static std::atomic<uint64_t> done{0};  // bit d: on device d
    int dev = 0;
    const cudaError_t g = cudaGetDevice(&dev);
    if (g != cudaSuccess) return g;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (e != cudaSuccess) return e;
    done.fetch_or(bit, std::memory_order_release);
  }
  return cudaSuccess;
}

// Lanes of a row: the power of two that holds its D / 16 chunk pairs.
inline int lanes_for(int64_t D) {
  int l = 1;
  while (l < D / 16) l *= 2;
  return l;
}

// Checks what both operators share and fills Tables.
inline int make_tables(Tables* t, const void* cosv, const void* sinv, int cs_dtype, const void* positions,
                       int pos_bytes, int64_t pos_sb, int64_t num_pos, int64_t T, int64_t D, int64_t R, float eps,
                       int normalize, const void* wq, const void* wk, int w_dtype) {
  if (D <= 0 || D % 16 != 0 || D > 256 || R < 0 || R % 16 != 0 || R > D) return SA_ERR_UNSUPPORTED;
  if (R > 0) {
    if (!cosv || !sinv || num_pos <= 0) return SA_ERR_ARG;
    if (cs_dtype != SA_F32 && cs_dtype != SA_F16 && cs_dtype != SA_BF16) return SA_ERR_UNSUPPORTED;
    if (!al16(cosv) || !al16(sinv)) return SA_ERR_ALIGN;
    if (pos_bytes != 0 && pos_bytes != 4 && pos_bytes != 8) return SA_ERR_UNSUPPORTED;
    if (pos_bytes != 0 && !positions) return SA_ERR_ARG;
    if (pos_bytes == 0 && num_pos < T) return SA_ERR_ARG;  // token t reads row t
  }
  if (normalize && !(eps >= 0.f)) return SA_ERR_ARG;
  if (wq || wk) {
    if (w_dtype != SA_F32 && w_dtype != SA_F16 && w_dtype != SA_BF16) return SA_ERR_UNSUPPORTED;
    if (!al16(wq) || !al16(wk)) return SA_ERR_ALIGN;
  }
  t->cosv = cosv;
  t->sinv = sinv;
  t->pos = positions;
  t->pos_bytes = R > 0 ? pos_bytes : 0;
  t->pos_sb = pos_sb;
  t->num_pos = num_pos;
  t->cs_dtype = cs_dtype;
  t->D = (int)D;
  t->R = (int)R;
  t->normalize = normalize != 0;
  t->eps = eps;
  t->inv_d = 1.0f / (float)D;
  return SA_OK;
}

// What `units` units of in all `rows` heads' groups cost a warp, in rows.
constexpr double kUnitCost = 1.5;
inline double walk_cost(int64_t rows, int64_t units) { return (double)rows + kUnitCost * (double)units; }

// Heads of a unit, for `rows` (token group, head) pairs on `warps` warps: the
// choice among 1, 2, 4 and 8 with the shortest busiest warp, a unit costing its heads
// and about one and a half more for its angles and addresses.  Many rows take 8:
// a block's four warps then cover 32 neighbouring heads of their tokens (backward
// of [4, 32 + 8, 4096, 128]: 84 us; 96 us with 4, 98 us with 16).
inline int unit_heads(int64_t rows, int64_t warps) {
  int best = 1;
  double cost = 0;
  for (int c = 1; c <= 8; c *= 2) {
    const int64_t units = (rows + c - 1) / c, rounds = (units + warps - 1) / warps;
    const double t = (double)rounds * (c + kUnitCost);
    if (c == 1 || t < cost) best = c, cost = t;
  }
  return best;
}

// Blocks of kWalkThreads for `units`: one resident wave of `per_sm` blocks an
// SM, fewer when there are not that many units for the warps.
inline int64_t walk_blocks(int64_t units, int per_sm) {
  const int64_t need = (units + kWalkThreads / 32 - 1) / (kWalkThreads / 32);
  const int64_t wave = (int64_t)per_sm * sm_count();
  return need < wave ? need : wave;
}

}  // namespace qkr
}  // namespace sa
