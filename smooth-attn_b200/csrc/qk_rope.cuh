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
// with two 8-element chunks that the rotation pairs (x[8g..], x[R/2 + 8g..]),
// so the rotation needs no exchange and the norm's sum log2(L) shuffles.
// Everything between the loads and the one rounding of y is fp32.
#pragma once

#include <stdint.h>

#include "sa_common.cuh"

namespace sa {
namespace qkr {

// 8 elements of E as they lie in memory.
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
  __device__ __forceinline__ void get(float (&f)[8]) const { unpack<E, 8>(u, f); }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    if constexpr (sizeof(E) == 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        u[i] = make_uint4(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]), __float_as_uint(f[4 * i + 2]),
                          __float_as_uint(f[4 * i + 3]));
    } else {
      Pack<E, 8> p;
#pragma unroll
      for (int i = 0; i < 8; ++i) p.set(i, f[i]);
      u[0] = p.u;
    }
  }
  __device__ __forceinline__ void store(E* p) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(E) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = u[i];
  }
};

// 8 elements of a table or weight of a type known at run time (one uniform branch).
__device__ __forceinline__ void load8_any(const void* p, int64_t at, int dtype, float (&f)[8]) {
  if (dtype == SA_F32) {
    Raw8<float> r;
    r.load(static_cast<const float*>(p) + at);
    r.get(f);
  } else if (dtype == SA_BF16) {
    Raw8<__nv_bfloat16> r;
    r.load(static_cast<const __nv_bfloat16*>(p) + at);
    r.get(f);
  } else {
    Raw8<__half> r;
    r.load(static_cast<const __half*>(p) + at);
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

struct Lane {
  int o1, o2;     // offsets of the lane's two chunks in the row
  bool active;    // the lane has a chunk at all (D / 16 need not be a power of two)
  bool rotated;   // its chunks are a rotated pair
};

template <int L>
__device__ __forceinline__ Lane lane_of(const Tables& t) {
  const int g = (threadIdx.x & 31) % L, nr = t.R / 16;
  Lane l;
  l.active = g < t.D / 16;
  l.rotated = g < nr;
  l.o1 = l.rotated ? 8 * g : t.R + 8 * (g - nr);
  l.o2 = l.rotated ? t.R / 2 + 8 * g : t.R + (t.D - t.R) / 2 + 8 * (g - nr);
  return l;
}

// cos and sin of one token for this lane; a position outside the tables is
// read as 0 and counted (the caller's counter).
__device__ __forceinline__ void load_angles(const Tables& t, const Lane& l, int64_t p, unsigned* bad, float (&c)[8],
                                            float (&s)[8]) {
  if (l.active && l.rotated) {
    if (p < 0 || p >= t.num_pos) {
      if (l.o1 == 0) atomicAdd(bad, 1u);
      p = 0;
    }
    load8_any(t.cosv, p * (t.R / 2) + l.o1, t.cs_dtype, c);
    load8_any(t.sinv, p * (t.R / 2) + l.o1, t.cs_dtype, s);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = 1.f, s[i] = 0.f;
  }
}

__device__ __forceinline__ int64_t read_pos(const void* pos, int bytes, int64_t at) {
  return bytes == 8 ? __ldg(static_cast<const long long*>(pos) + at) : (int64_t)__ldg(static_cast<const int*>(pos) + at);
}

// Sum over the L lanes of a row; every lane of the warp takes part.
template <int L> __device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int m = L / 2; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

template <int L>
__device__ __forceinline__ float row_rscale(const Tables& t, const float (&x1)[8], const float (&x2)[8]) {
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = fmaf(x1[i], x1[i], ss);
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = fmaf(x2[i], x2[i], ss);
  return rsqrtf(fmaf(row_sum<L>(ss), t.inv_d, t.eps));
}

// y of one row from its two raw chunks (zeros in lanes without one).
template <typename E, int L>
__device__ __forceinline__ void norm_rope(const Tables& t, Raw8<E>& a, Raw8<E>& b, const float (&w1)[8],
                                          const float (&w2)[8], const float (&c)[8], const float (&s)[8]) {
  float x1[8], x2[8];
  a.get(x1);
  b.get(x2);
  if (t.normalize) {
    const float r = row_rscale<L>(t, x1, x2);
#pragma unroll
    for (int i = 0; i < 8; ++i) x1[i] = x1[i] * r * w1[i], x2[i] = x2[i] * r * w2[i];
  }
  float y1[8], y2[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y1[i] = x1[i] * c[i] - x2[i] * s[i];
    y2[i] = x2[i] * c[i] + x1[i] * s[i];
  }
  a.set(y1);
  b.set(y2);
}

__device__ __forceinline__ void load_weights(const void* w, int w_dtype, const Lane& l, float (&w1)[8],
                                             float (&w2)[8]) {
  if (w != nullptr && l.active) {
    load8_any(w, l.o1, w_dtype, w1);
    load8_any(w, l.o2, w_dtype, w2);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) w1[i] = w2[i] = 1.f;
  }
}

// ---- host side ----------------------------------------------------------------

inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

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

// Heads a warp takes per token: 8 (the angles are loaded once for all of them)
// unless that leaves fewer than `want` warps, then fewer.
inline int heads_per_warp(int64_t groups, int64_t heads, int64_t want) {
  int hc = 8;
  while (hc > 1 && groups * ((heads + hc - 1) / hc) < want) hc /= 2;
  return hc;
}

}  // namespace qkr
}  // namespace sa
