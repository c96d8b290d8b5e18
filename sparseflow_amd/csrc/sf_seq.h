// Device helpers shared by the state space operators (convolution, scan, norm).
// gfx950 only.
#pragma once

#include "sf_internal.h"

namespace sf {
namespace {

// V elements of T, loaded and stored at once.
template <typename T, int V>
struct alignas(V * sizeof(T) < 16 ? V * sizeof(T) : 16) Vec {
  T e[V];
};

// 16 and 8 bytes at the address of any 16-bit element.
typedef uint32_t AnyX4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t AnyX2 __attribute__((ext_vector_type(2), aligned(2)));

// V elements at p, aligned to one element only: global memory takes 8 and 16 bytes at
// any address.  ONCE: read once, and more than the caches hold (read_once): they do not
// keep it.
template <typename T, int V, bool ONCE = false>
__device__ __forceinline__ Vec<T, V> load_any(const T* __restrict__ p) {
  Vec<T, V> q;
  if constexpr (ONCE && sizeof(q) % 16 == 0) {
    AnyX4 u[sizeof(q) / 16];
#pragma unroll
    for (int i = 0; i < (int)sizeof(q) / 16; ++i) u[i] = __builtin_nontemporal_load(reinterpret_cast<const AnyX4*>(p) + i);
    __builtin_memcpy(&q, u, sizeof(q));
  } else if constexpr (ONCE && sizeof(q) == 8) {
    const AnyX2 u = __builtin_nontemporal_load(reinterpret_cast<const AnyX2*>(p));
    __builtin_memcpy(&q, &u, sizeof(q));
  } else {
    __builtin_memcpy(&q, p, sizeof(q));
  }
  return q;
}
template <typename T, int V, bool ONCE = false>
__device__ __forceinline__ void load_any_f32(const T* __restrict__ p, float (&v)[V]) {
  const Vec<T, V> q = load_any<T, V, ONCE>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = to_f32<T>(q.e[i]);
}
template <typename T, int V, bool ONCE = false>
__device__ __forceinline__ void store_any_f32(T* __restrict__ p, const float (&v)[V]) {
  Vec<T, V> q;
#pragma unroll
  for (int i = 0; i < V; ++i) q.e[i] = from_f32<T>(v[i]);
  if constexpr (ONCE) {
    static_assert(sizeof(q) == 16, "one access");
    AnyX4 u;
    __builtin_memcpy(&u, &q, sizeof(q));
    __builtin_nontemporal_store(u, reinterpret_cast<AnyX4*>(p));
  } else {
    __builtin_memcpy(p, &q, sizeof(q));
  }
}

// Aligned to all of them, or to 16 bytes.
template <typename T, int V>
__device__ __forceinline__ void load_f32(const T* __restrict__ p, float (&v)[V]) {
  const Vec<T, V> q = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = to_f32<T>(q.e[i]);
}

template <typename T, int V>
__device__ __forceinline__ void store_f32(T* __restrict__ p, const float (&v)[V]) {
  Vec<T, V> q;
#pragma unroll
  for (int i = 0; i < V; ++i) q.e[i] = from_f32<T>(v[i]);
  *reinterpret_cast<Vec<T, V>*>(p) = q;
}

// Rows [first, first + n) of the token axis that are sequence b's (b the same in
// all lanes).
__device__ __forceinline__ void seq_rows(const SeqAxis& s, int64_t b, int64_t& first, int64_t& n) {
  if (s.offsets == nullptr) {
    first = 0;
    n = s.tokens;
    return;
  }
  const int64_t lo = __builtin_amdgcn_readfirstlane(s.offsets[b]), hi = __builtin_amdgcn_readfirstlane(s.offsets[b + 1]);
  first = lo < 0 ? 0 : (lo > s.tokens ? s.tokens : lo);
  const int64_t end = hi > s.tokens ? s.tokens : hi;
  n = end > first ? end - first : 0;
}

// Sequence b's row of the pool, or -1.
__device__ __forceinline__ int64_t seq_slot(const SeqAxis& s, int64_t b) {
  const int64_t r = s.slots == nullptr ? b : (int64_t)s.slots[b];
  return r >= 0 && r < s.states ? r : -1;
}

// 2^v by the hardware's exponential (relative error 2^-23; results below the
// normal range are 0).
__device__ __forceinline__ float exp2_hw(float v) { return __builtin_amdgcn_exp2f(v); }

// log(1 + exp(v)) = max(v, 0) + log1p(e), e = exp(-|v|), so that neither end
// overflows and the far negative one keeps its relative accuracy.  e is
// 2^(hi + lo) with hi + lo = -|v| log2(e) to more than 24 bits, and log1p(e) =
// 2 atanh(s), s = e / (2 + e) <= 1/3: the odd series up to s^15 (the next term is
// below 2^-29 of the sum).
__device__ __forceinline__ float softplus(float v) {
  const float a = -fabsf(v);
  const float hi = a * 1.44269502f, lo = fmaf(a, 1.44269502f, -hi) + a * 1.92596303e-8f;
  const float p = exp2_hw(hi);
  const float e = a < -120.f ? p : fmaf(p * 0.693147182f, lo, p);  // (-inf: lo is NaN)
  const float den = 2.f + e;
  float r = __builtin_amdgcn_rcpf(den);
  r = fmaf(fmaf(-den, r, 1.f), r, r);
  const float s = e * r, q = s * s;
  float t = 1.f / 15.f;
  t = fmaf(t, q, 1.f / 13.f);
  t = fmaf(t, q, 1.f / 11.f);
  t = fmaf(t, q, 1.f / 9.f);
  t = fmaf(t, q, 1.f / 7.f);
  t = fmaf(t, q, 1.f / 5.f);
  t = fmaf(t, q, 1.f / 3.f);
  t = fmaf(t * q, s, s);
  return fmaxf(v, 0.f) + (t + t);
}

// sigmoid(v) and v sigmoid(v) by the hardware's exponential and reciprocal: each is
// good to a unit in the last place.  (With expf and a division the convolution of bf16
// rows was bound by arithmetic: 183 us for 2 x 16384 x 4352, against 130.)  The
// exponent's rounding costs up to |v| units in 1 + exp(-v) where v < 0: with F32, for
// results that are float32, what it loses is made good (e = 2^(hi + lo), as above); 16-bit
// ones have none of those bits.
template <bool F32>
__device__ __forceinline__ float sigmoid(float v) {
  const float hi = v * -1.44269502f;
  float e = exp2_hw(hi);
  if constexpr (F32) {
    const float lo = fmaf(v, -1.44269502f, -hi) + v * -1.92596303e-8f;
    e = fabsf(hi) < 127.f ? fmaf(e * 0.693147182f, lo, e) : e;  // (past it e is 0, huge or no number)
  }
  return __builtin_amdgcn_rcpf(1.f + e);
}
template <bool F32>
__device__ __forceinline__ float silu(float v) { return v * sigmoid<F32>(v); }

}  // namespace

// Whether a kernel that reads `bytes` once leaves them out of the caches: half of what
// the memory side's holds, so that less than that still lies there from the kernel that
// wrote it, or for the next.  Kept and left out: norm of 32768 x 1024 float32 (134 MB) 75
// and 64 us, of 32768 x 384 25 and 29, of 32768 x 2048 f16 with gate and float32 residual
// 215 and 207; states of 1 GB and 100 MB a step's 210 and 192, 38 and 40.  (The
// convolution reads a run's last tokens again: 2 x 16384 x 4352 bf16 130 and 136.)
inline bool read_once(int64_t bytes) { return bytes >= (int64_t)128 << 20; }

// A launch holds fewer than 2^32 threads: `blocks` workgroups in as many
// launches as that takes, block0 being the first of each.
template <typename Args, typename Launch>
int launch_blocks(Args a, int64_t Args::*first, int64_t blocks, Launch&& launch) {
  constexpr int64_t kMost = (int64_t)1 << 21;
  for (int64_t at = 0; at < blocks; at += kMost) {
    a.*first = at;
    launch(a, (unsigned)(blocks - at < kMost ? blocks - at : kMost));
    const int rc = (int)hipGetLastError();
    if (rc != (int)hipSuccess) return rc;
  }
  return (int)hipSuccess;
}

}  // namespace sf
