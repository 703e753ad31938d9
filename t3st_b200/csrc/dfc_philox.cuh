// Counter-based dropout masks (no reference counterpart): the random words of
// element i are a function of (seed, offset, i) alone, so a mask is never
// stored -- the backward pass computes it again.
//
// Generator: Philox4x32 with 10 rounds (Salmon et al., "Parallel random
// numbers: as easy as 1, 2, 3", SC 2011).  Key: the 64-bit seed.  Counter:
// (g low, g high | half << 31, offset low, offset high) for the group g = i / 8
// of eight elements.  half 0 gives eight 16-bit numbers, the high halves of
// the elements' 32-bit words u (element 2k in the low half of word k, element
// 2k + 1 in the high half); half 1 gives their low halves.  Element i is kept
// when u >= T, T = floor(p * 2^32 + 1/2).
//
// The high half decides unless it equals T >> 16, so the second Philox call is
// made only by a thread that sees such a tie (8 in 65,536), and never when the
// low half of T is zero: one call serves eight elements at the full 32-bit
// resolution of p.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "dfc_common.cuh"

namespace dfc {

struct DropArgs {
  uint64_t seed;
  uint64_t offset;
  const uint64_t* state;  // NULL, or {seed, offset base} in device memory
  uint32_t t_hi;          // T >> 16
  uint32_t t_lo;          // T & 0xFFFF
  uint32_t cmp;           // threshold of the 16-bit comparison, shifted left by 16
  uint32_t all;           // non-zero: T = 2^32, nothing is kept
  float scale;            // 1 / (1 - p)
};

// Arguments of a call, or an error code; *active = some element can be dropped.
inline int make_drop_args(const DfcDropout* d, DropArgs* a, bool* active) {
  *a = DropArgs{};
  *active = false;
  if (!d) return DFC_OK;
  if (!(d->p >= 0.0 && d->p <= 1.0)) return DFC_ERR_VALUE;
  if (!aligned(d->state, 8)) return DFC_ERR_ALIGN;
  a->seed = d->seed;
  a->offset = d->offset;
  a->state = d->state;
  const uint64_t t = static_cast<uint64_t>(floor(d->p * 4294967296.0 + 0.5));
  *active = t != 0;
  a->all = t >> 32 ? 1u : 0u;
  a->t_hi = static_cast<uint32_t>(t >> 16) & 0xFFFFu;
  a->t_lo = static_cast<uint32_t>(t & 0xFFFFu);
  // ties are settled before the comparison, as 0xFFFF or 0; a threshold of 0
  // would keep a dropped tie
  a->cmp = (a->t_hi == 0 ? 1u : a->t_hi) << 16;
  a->scale = d->p < 1.0 ? static_cast<float>(1.0 / (1.0 - d->p)) : 0.0f;
  return DFC_OK;
}

struct DropKey {
  uint32_t k0, k1, o0, o1;
};

__device__ __forceinline__ DropKey drop_key(const DropArgs& a) {
  uint64_t seed = a.seed, off = a.offset;
  if (a.state) {
    seed = a.state[0];
    off += a.state[1];
  }
  return {static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32),
          static_cast<uint32_t>(off), static_cast<uint32_t>(off >> 32)};
}

__device__ __forceinline__ void philox_round(uint32_t& c0, uint32_t& c1, uint32_t& c2, uint32_t& c3,
                                             uint32_t k0, uint32_t k1) {
  const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u;
  const uint64_t b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
  c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
  c1 = static_cast<uint32_t>(b);
  c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
  c3 = static_cast<uint32_t>(a);
}

__device__ __forceinline__ uint4 philox10(uint32_t c0, uint32_t c1, const DropKey& k) {
  uint32_t c2 = k.o0, c3 = k.o1;
#pragma unroll
  for (int r = 0; r < 10; ++r)
    philox_round(c0, c1, c2, c3, k.k0 + r * 0x9E3779B9u, k.k1 + r * 0xBB67AE85u);
  return make_uint4(c0, c1, c2, c3);
}

// Bit 15 or 31 is set when a 16-bit half of w is zero (and maybe when the
// half below it is; never when neither is).
__device__ __forceinline__ uint32_t zero_half(uint32_t w) { return (w - 0x00010001u) & ~w; }

// A word of two high halves with its ties settled by the low halves.
__device__ __forceinline__ uint32_t settle(uint32_t w, uint32_t low, const DropArgs& a) {
  uint32_t h0 = w & 0xFFFFu, h1 = w >> 16;
  if (h0 == a.t_hi) h0 = (low & 0xFFFFu) >= a.t_lo ? 0xFFFFu : 0u;
  if (h1 == a.t_hi) h1 = (low >> 16) >= a.t_lo ? 0xFFFFu : 0u;
  return h0 | (h1 << 16);
}

// The comparison words of N groups: kept(w, j) tells element j's fate.  The
// groups go through the rounds together: they share the round keys, and the
// rare ties are looked for once.
template <int N>
__device__ __forceinline__ void drop_words(const uint64_t (&g)[N], const DropArgs& a, const DropKey& k,
                                           uint4 (&w)[N]) {
  uint32_t c0[N], c1[N], c2[N], c3[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    c0[i] = static_cast<uint32_t>(g[i]);
    c1[i] = static_cast<uint32_t>(g[i] >> 32);
    c2[i] = k.o0;
    c3[i] = k.o1;
  }
  uint32_t k0 = k.k0, k1 = k.k1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
#pragma unroll
    for (int i = 0; i < N; ++i) philox_round(c0[i], c1[i], c2[i], c3[i], k0, k1);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = make_uint4(c0[i], c1[i], c2[i], c3[i]);
  if (a.t_lo) {
    const uint32_t t2 = a.t_hi * 0x00010001u;
    uint32_t tie = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
      tie |= zero_half(w[i].x ^ t2) | zero_half(w[i].y ^ t2) | zero_half(w[i].z ^ t2) | zero_half(w[i].w ^ t2);
    if (tie & 0x80008000u) {
#pragma unroll 1
      for (int i = 0; i < N; ++i) {
        const uint4 l = philox10(static_cast<uint32_t>(g[i]), static_cast<uint32_t>(g[i] >> 32) | 0x80000000u, k);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          if (i == j) {
            w[j].x = settle(w[j].x, l.x, a);
            w[j].y = settle(w[j].y, l.y, a);
            w[j].z = settle(w[j].z, l.z, a);
            w[j].w = settle(w[j].w, l.w, a);
          }
        }
      }
    }
  }
  if (a.all) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = make_uint4(0u, 0u, 0u, 0u);
  }
}

__device__ __forceinline__ bool kept(const uint4& w, int j, uint32_t cmp) {
  const uint32_t x = j < 4 ? (j < 2 ? w.x : w.y) : (j < 6 ? w.z : w.w);
  return ((j & 1) ? x : x << 16) >= cmp;
}

// Eight elements: v[j] = kept ? v[j] * scale : 0.
__device__ __forceinline__ void drop8(float (&v)[8], const uint4& w, const DropArgs& a) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = kept(w, j, a.cmp) ? __fmul_rn(v[j], a.scale) : 0.0f;
}

// ---- element types --------------------------------------------------------
using bf16 = __nv_bfloat16;
using f16 = __half;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(f16 x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ f16 from_f32<f16>(float x) { return __float2half_rn(x); }

// Eight elements as they lie in memory, in registers (16-byte pieces).
template <typename T>
struct Raw8 {
  uint4 q[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    v[0] = u2f(r.q[0].x), v[1] = u2f(r.q[0].y), v[2] = u2f(r.q[0].z), v[3] = u2f(r.q[0].w);
    v[4] = u2f(r.q[1].x), v[5] = u2f(r.q[1].y), v[6] = u2f(r.q[1].z), v[7] = u2f(r.q[1].w);
  } else {
    const uint32_t u[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (sizeof(T) == 2 && __is_same(T, bf16)) {
        v[2 * k] = u2f(u[k] << 16);
        v[2 * k + 1] = u2f(u[k] & 0xFFFF0000u);
      } else {
        __half2 h;
        memcpy(&h, &u[k], 4);
        const float2 f = __half22float2(h);
        v[2 * k] = f.x;
        v[2 * k + 1] = f.y;
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ Raw8<T> pack8(const float (&v)[8]) {
  Raw8<T> r;
  if constexpr (sizeof(T) == 4) {
    r.q[0] = make_uint4(f2u(v[0]), f2u(v[1]), f2u(v[2]), f2u(v[3]));
    r.q[1] = make_uint4(f2u(v[4]), f2u(v[5]), f2u(v[6]), f2u(v[7]));
  } else {
    uint32_t u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (__is_same(T, bf16)) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
        memcpy(&u[k], &h, 4);
      } else {
        const __half2 h = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
        memcpy(&u[k], &h, 4);
      }
    }
    r.q[0] = make_uint4(u[0], u[1], u[2], u[3]);
  }
  return r;
}

// p is 16-byte aligned; FP32 with wide != 0: 32-byte aligned, and the eight
// elements move in one access, so that a warp writes whole 32-byte sectors
// (two 16-byte accesses 32 bytes apart write half sectors).
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p, int wide) {
  Raw8<T> r;
  const uint4* q = reinterpret_cast<const uint4*>(p);
  if constexpr (sizeof(T) == 4) {
    if (wide) {
      asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(r.q[0].x), "=r"(r.q[0].y), "=r"(r.q[0].z), "=r"(r.q[0].w), "=r"(r.q[1].x),
                     "=r"(r.q[1].y), "=r"(r.q[1].z), "=r"(r.q[1].w)
                   : "l"(p));
      return r;
    }
    r.q[1] = q[1];
  }
  r.q[0] = q[0];
  return r;
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const Raw8<T>& r, int wide) {
  uint4* q = reinterpret_cast<uint4*>(p);
  if constexpr (sizeof(T) == 4) {
    if (wide) {
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r.q[0].x),
                   "r"(r.q[0].y), "r"(r.q[0].z), "r"(r.q[0].w), "r"(r.q[1].x), "r"(r.q[1].y),
                   "r"(r.q[1].z), "r"(r.q[1].w)
                   : "memory");
      return;
    }
    q[1] = r.q[1];
  }
  q[0] = r.q[0];
}

// Eight elements from any address p (aligned to T) of an array that occupies
// [lo, hi): the 16-byte blocks around them, to be shifted into place.
template <typename T>
struct Blocks {
  static constexpr int N = sizeof(T) / 2 + 1;
  uint4 q[N];

  // The blocks lie within the array.
  __device__ __forceinline__ static bool within(const T* p, const void* lo, const void* hi) {
    const uintptr_t first = reinterpret_cast<uintptr_t>(p) & ~uintptr_t{15};
    return first >= reinterpret_cast<uintptr_t>(lo) && first + 16 * N <= reinterpret_cast<uintptr_t>(hi);
  }

  __device__ __forceinline__ void load(const T* p) {
    const uint4* first = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t{15});
#pragma unroll
    for (int b = 0; b < N; ++b) q[b] = first[b];
  }

  // The elements: down by p's offset in its block, in steps of two words, one
  // word and half a word.
  __device__ __forceinline__ Raw8<T> at(const T* p) const {
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 15);
    uint32_t w[4 * N];
#pragma unroll
    for (int b = 0; b < N; ++b) w[4 * b] = q[b].x, w[4 * b + 1] = q[b].y, w[4 * b + 2] = q[b].z, w[4 * b + 3] = q[b].w;
#pragma unroll
    for (int i = 0; i < 4 * N - 2; ++i) w[i] = off & 8 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 4 * N - 3; ++i) w[i] = off & 4 ? w[i + 1] : w[i];
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], off & 2 ? 16 : 0);
    }
    Raw8<T> r;
#pragma unroll
    for (int b = 0; b < N - 1; ++b) r.q[b] = make_uint4(w[4 * b], w[4 * b + 1], w[4 * b + 2], w[4 * b + 3]);
    return r;
  }
};

// The first `count` of eight elements, one by one; the others are zero.
template <typename T>
__device__ __forceinline__ Raw8<T> load8_single(const T* p, int count) {
  T v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = j < count ? p[j] : T(0.0f);
  Raw8<T> r;
  memcpy(&r, v, sizeof(r));
  return r;
}

// Eight elements from any address of [lo, hi).
template <typename T>
__device__ __forceinline__ Raw8<T> load8_any(const T* p, const void* lo, const void* hi) {
  if (!Blocks<T>::within(p, lo, hi)) return load8_single(p, 8);
  Blocks<T> b;
  b.load(p);
  return b.at(p);
}

inline bool known_dtype(int32_t d) {
  return d == DFC_DTYPE_F32 || d == DFC_DTYPE_BF16 || d == DFC_DTYPE_F16;
}
inline uintptr_t dtype_size(int32_t d) { return d == DFC_DTYPE_F32 ? 4 : 2; }

}  // namespace dfc
