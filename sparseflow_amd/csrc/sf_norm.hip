// The norms around a block with its gate and residual scale, in one pass over
// each row:
//   t = act(gate) x (gate first), t *= w / rms(t) over each group, t *= act(gate),
//   r = residual + scale t, h = r w' / rms(r)
// A row is held in registers by LT threads, vectors of V elements: x, gate and residual
// are all loaded before the first sum, and h is written after the second.  Bound by
// HBM: 32768 x 4096 bf16, gated, groups of 512 (805 MB) 157 us, 5.1 TB/s; 32768 x 2048
// f16 with gate, float32 residual and h (940 MB) 183 us, 5.1 TB/s.  Short rows (up to 3
// vectors a lane) are a wavefront's, whose sums need no barrier: 32768 x 384 float32 25
// us, as a workgroup's 37; of 768 53 and 57; of four vectors, 2048 bf16, 86 and 77.
//
// Groups are rows of their own where no norm of the whole row follows; otherwise
// a workgroup holds the row and the groups' sums meet in LDS.
#include "sf_seq.h"

#include <type_traits>

namespace sf {

namespace {

constexpr int kBlock = 256;
// Rows of whole vectors; those whose inputs the caches are not to keep; rows that end
// inside a vector (32768 x 2047 bf16: 142 us, by single elements 238; the checks for it
// would cost whole rows, 2048, 92 against 70).
constexpr int kPlain = 0, kOnce = 1, kRagged = 2;

template <bool F32>
__device__ __forceinline__ float act_of(int act, float v) {
  return act == SF_ACT_SILU ? silu<F32>(v) : act == SF_ACT_SIGMOID ? sigmoid<F32>(v) : v;
}

// The sum of v over the LT threads of a row (in an order of its own for every
// thread of a wavefront, the same bits in all: xor butterflies).
template <int LT>
__device__ __forceinline__ float row_sum(float v, float* s_part) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  if constexpr (LT > kWave) {
    __syncthreads();  // an earlier sum's readers
    if (lane_id() == 0) s_part[threadIdx.x / kWave] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < LT / kWave; ++w) v += s_part[w];
  }
  return v;
}

// sub: groups that are rows of their own (1: the whole row).  GROUPED: groups
// inside the row (LT = the workgroup, group % V == 0).  (Workgroups that go row after
// row with their weights in registers were no faster: 226 against 214 us at
// 32768 x 2048, f16 with a float32 residual.)
template <typename T, typename TR, int LT, int V, int NV, bool GROUPED, int MODE>
__global__ __launch_bounds__(LT > kBlock ? LT : kBlock) void k_block_norm(NormArgs a, int sub) {
  constexpr bool ONCE = MODE == kOnce, RAGGED = MODE == kRagged;
  constexpr int kRowsPerBlock = (LT > kBlock ? LT : kBlock) / LT;
  __shared__ float s_part[LT / kWave];
  const int lt = threadIdx.x % LT;
  const int width = a.dim / sub;
  const int64_t item = (a.item0 + blockIdx.x) * kRowsPerBlock + threadIdx.x / LT;
  if (item >= a.outer * a.inner * sub) return;  // (LT > 64 has one row to a workgroup)
  const int64_t row = sub == 1 ? item : item / sub;
  const int c0 = sub == 1 ? 0 : (int)(item - row * sub) * width;
  const int64_t o = a.outer == 1 ? 0 : row / a.inner, i = row - o * a.inner;
  const T* __restrict__ x = static_cast<const T*>(a.x) + o * a.x_o + i * a.x_i + c0;
  const T* __restrict__ g = static_cast<const T*>(a.gate) + o * a.g_o + i * a.g_i + c0;
  const TR* __restrict__ res = static_cast<const TR*>(a.res) + o * a.res_o + i * a.res_i + c0;
  Vec<T, V> gv[NV];
  Vec<TR, V> rv[NV];
  float t[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * LT + lt) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) t[k][e] = 0.f;
    if (c >= width) continue;
    if (RAGGED && c + V > width) {
      // The end of a row that is not whole vectors: zeros behind it.
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int at = min(c + e, width - 1);
        if (c + e < width) t[k][e] = to_f32<T>(x[at]);
        if (a.gate != nullptr) gv[k].e[e] = g[at];
        if (a.res != nullptr) rv[k].e[e] = res[at];
      }
      continue;
    }
    load_any_f32<T, V, ONCE>(x + c, t[k]);
    if (a.gate != nullptr) gv[k] = load_any<T, V, ONCE>(g + c);
    if (a.res != nullptr) rv[k] = load_any<TR, V, ONCE>(res + c);
  }
  auto gate = [&]() {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if ((k * LT + lt) * V >= width) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) t[k][e] *= act_of<sizeof(TR) == 4>(a.act, to_f32<T>(gv[k].e[e]));
    }
  };
  // The weights of a vector's columns (behind the row's end the last one).
  auto weights = [&](const float* __restrict__ w, int c, float (&v)[V]) {
    if (!RAGGED || c + V <= width) {
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = w[c0 + c + e];
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = w[c0 + min(c + e, width - 1)];
    }
  };
  auto store = [&](auto* __restrict__ p, int c, const float (&v)[V]) {
    typedef std::remove_reference_t<decltype(*p)> E;
    if (!RAGGED || c + V <= width) {
      store_any_f32<E, V>(p + c, v);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (c + e < width) p[c + e] = from_f32<E>(v[e]);
    }
  };
  auto squares = [&]() {
    float s = 0.f;
    if constexpr (RAGGED) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * LT + lt) * V;
        if (c < width && c + V > width) {
          // (What a gate or weight that is not finite made of the zeros.)
#pragma unroll
          for (int e = 0; e < V; ++e) t[k][e] = c + e < width ? t[k][e] : 0.f;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) s = fmaf(t[k][e], t[k][e], s);
    return s;
  };
  if (a.gate != nullptr && a.gate_first) gate();
  if (a.post_w != nullptr) {
    if constexpr (GROUPED) {
      extern __shared__ float s_group[];  // a sum of squares per vector, then 1 / rms per group
      const int vecs = a.dim / V, per = a.group / V, groups = a.dim / a.group;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) s = fmaf(t[k][e], t[k][e], s);
        if (k * LT + lt < vecs) s_group[k * LT + lt] = s;
      }
      __syncthreads();
      for (int q = threadIdx.x / kWave; q < groups; q += LT / kWave) {
        float s = 0.f;
        for (int v = lane_id(); v < per; v += kWave) s += s_group[q * per + v];
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, kWave);
        if (lane_id() == 0) s_group[vecs + q] = 1.f / sqrtf(s / (float)a.group + a.eps);
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * LT + lt) * V;
        if (c >= width) continue;
        const float f = s_group[vecs + c / a.group];
#pragma unroll
        for (int e = 0; e < V; ++e) t[k][e] *= f;
      }
    } else {
      const float f = 1.f / sqrtf(row_sum<LT>(squares(), s_part) / (float)width + a.eps);
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) t[k][e] *= f;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * LT + lt) * V;
      if (c >= width) continue;
      float w[V];
      weights(a.post_w, c, w);
#pragma unroll
      for (int e = 0; e < V; ++e) t[k][e] *= w[e];
    }
  }
  if (a.gate != nullptr && !a.gate_first) gate();
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * LT + lt) * V;
    if (c >= width) continue;
    float w[V] = {};
    if (a.scale_w != nullptr) weights(a.scale_w, c, w);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float f = a.scale_w != nullptr ? a.scale * w[e] : a.scale;
      t[k][e] = a.res != nullptr ? fmaf(f, t[k][e], to_f32<TR>(rv[k].e[e])) : f * t[k][e];
    }
    if (a.r != nullptr) store(static_cast<TR*>(a.r) + o * a.r_o + i * a.r_i + c0, c, t[k]);
  }
  if (a.pre_w != nullptr) {
    const float f = 1.f / sqrtf(row_sum<LT>(squares(), s_part) / (float)width + a.eps);
    T* __restrict__ h = static_cast<T*>(a.h) + o * a.h_o + i * a.h_i;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * LT + lt) * V;
      if (c >= width) continue;
      float w[V];
      weights(a.pre_w, c, w);
#pragma unroll
      for (int e = 0; e < V; ++e) t[k][e] *= f * w[e];
      store(h + c0, c, t[k]);
    }
  }
}

template <typename T, typename TR, int LT, int V, int NV, bool GROUPED, int MODE>
int launch_norm_k(const NormArgs& a, int sub, hipStream_t stream) {
  constexpr int threads = LT > kBlock ? LT : kBlock, rows = threads / LT;
  const int64_t items = a.outer * a.inner * sub;
  const size_t lds = GROUPED ? (size_t)(a.dim / V + a.dim / a.group) * sizeof(float) : 0;
  if (lds > 48 * 1024) {
    const int rc = set_lds_limit_once<k_block_norm<T, TR, LT, V, NV, GROUPED, MODE>>(kMaxLdsBytes - 1024);
    if (rc != (int)hipSuccess) return rc;
  }
  return launch_blocks(a, &NormArgs::item0, (items + rows - 1) / rows, [&](const NormArgs& la, unsigned n) {
    hipLaunchKernelGGL((k_block_norm<T, TR, LT, V, NV, GROUPED, MODE>), dim3(n), dim3(threads), lds, stream, la, sub);
  });
}

// M vectors a thread hold the widest row that 1024 threads take.
// Groups inside a row that has a norm of its own, too.
template <typename T, typename TR, int V, int M, int MODE>
int launch_norm_grouped(const NormArgs& a, hipStream_t stream) {
  if (a.dim <= 256 * V * M) return launch_norm_k<T, TR, 256, V, M, true, MODE>(a, 1, stream);
  return launch_norm_k<T, TR, 1024, V, M, true, MODE>(a, 1, stream);
}

// Rows, or groups as rows of their own.
template <typename T, typename TR, int V, int M, int MODE>
int launch_norm_rows(const NormArgs& a, hipStream_t stream) {
  const int sub = a.post_w != nullptr ? a.dim / a.group : 1, width = a.dim / sub;
  if (width <= 64 * V) return launch_norm_k<T, TR, 64, V, 1, false, MODE>(a, sub, stream);
  if (width <= 64 * V * 2) return launch_norm_k<T, TR, 64, V, 2, false, MODE>(a, sub, stream);
  if (width <= 64 * V * 3) return launch_norm_k<T, TR, 64, V, 3, false, MODE>(a, sub, stream);
  if (width <= 256 * V) return launch_norm_k<T, TR, 256, V, 1, false, MODE>(a, sub, stream);
  if (width <= 256 * V * 2) return launch_norm_k<T, TR, 256, V, 2, false, MODE>(a, sub, stream);
  if (width <= 256 * V * 4) return launch_norm_k<T, TR, 256, V, 4, false, MODE>(a, sub, stream);
  return launch_norm_k<T, TR, 1024, V, M, false, MODE>(a, sub, stream);
}

template <typename T, typename TR>
int launch_norm_t(const NormArgs& a, hipStream_t stream) {
  // 16 bytes of the widest type.
  constexpr int V = 16 / (sizeof(T) > sizeof(TR) ? sizeof(T) : sizeof(TR));
  const bool grouped = a.post_w != nullptr && a.pre_w != nullptr && a.group != a.dim;
  const bool whole = (a.post_w != nullptr ? a.group : a.dim) % V == 0;
  const int64_t bytes = (a.gate != nullptr ? 2 : 1) * (int64_t)sizeof(T) + (a.res != nullptr ? (int64_t)sizeof(TR) : 0);
  const bool once = read_once(a.outer * a.inner * a.dim * bytes);
  if (grouped) {
    // Groups that are not whole vectors: single elements.
    if (!whole) return launch_norm_grouped<T, TR, 1, 16, kPlain>(a, stream);
    return once ? launch_norm_grouped<T, TR, V, 16 / V, kOnce>(a, stream)
                : launch_norm_grouped<T, TR, V, 16 / V, kPlain>(a, stream);
  }
  if (!whole) return launch_norm_rows<T, TR, V, 16 / V, kRagged>(a, stream);
  return once ? launch_norm_rows<T, TR, V, 16 / V, kOnce>(a, stream) : launch_norm_rows<T, TR, V, 16 / V, kPlain>(a, stream);
}

template <typename T>
int launch_norm_r(const NormArgs& a, int res_dtype, hipStream_t stream) {
  if (res_dtype == SF_F32) return launch_norm_t<T, float>(a, stream);
  return launch_norm_t<T, T>(a, stream);
}

}  // namespace

int launch_block_norm(const NormArgs& a, int dtype, int res_dtype, hipStream_t stream) {
  timing_begin(K_NORM, stream);
  const int rc = dtype == SF_F16    ? launch_norm_r<__half>(a, res_dtype, stream)
                 : dtype == SF_BF16 ? launch_norm_r<__hip_bfloat16>(a, res_dtype, stream)
                                    : launch_norm_r<float>(a, res_dtype, stream);
  timing_end(K_NORM, stream);
  return rc;
}

}  // namespace sf
