// Device helpers shared by the state space operators (convolution, scan, norm).
// gfx950 only.
#pragma once

#include "sf_internal.h"

namespace sf {
namespace {

// V elements of T, loaded and stored at once (p aligned to all of them).
template <typename T, int V>
struct alignas(V * sizeof(T)) Vec {
  T e[V];
};

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

// Rows [first, first + n) of the token axis that are sequence b's.
__device__ __forceinline__ void seq_rows(const SeqAxis& s, int64_t b, int64_t& first, int64_t& n) {
  if (s.offsets == nullptr) {
    first = 0;
    n = s.tokens;
    return;
  }
  const int64_t lo = s.offsets[b], hi = s.offsets[b + 1];
  first = lo < 0 ? 0 : (lo > s.tokens ? s.tokens : lo);
  const int64_t end = hi > s.tokens ? s.tokens : hi;
  n = end > first ? end - first : 0;
}

// Sequence b's row of the pool, or -1.
__device__ __forceinline__ int64_t seq_slot(const SeqAxis& s, int64_t b) {
  const int64_t r = s.slots == nullptr ? b : (int64_t)s.slots[b];
  return r >= 0 && r < s.states ? r : -1;
}

// log(1 + exp(v)), from the larger of 0 and v so that neither end overflows.
__device__ __forceinline__ float softplus(float v) { return fmaxf(v, 0.f) + log1pf(expf(-fabsf(v))); }

// v * sigmoid(v): 0 at the far negative end (v / inf), NaN where v is.
__device__ __forceinline__ float sigmoid(float v) { return 1.f / (1.f + expf(-v)); }
__device__ __forceinline__ float silu(float v) { return v / (1.f + expf(-v)); }

}  // namespace

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

inline bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace sf
