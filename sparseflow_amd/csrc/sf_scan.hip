// Selective state space scan, token by token: per sequence and head
//   h = exp(A d) h + (d x) (outer) B,  y = h C + D x
// with d = dt + dt_bias or its softplus.
//
// A workgroup owns rows of one head's state [head_dim, state_dim]; a row lies
// over TN lanes, four columns in each, R rows to a thread.  The state stays in
// registers from the first token to the last, and y is a sum over the TN lanes.
// For one token (the step) this is bound by HBM: the state in and out, 16 bytes
// a load, R loads in flight per thread.  256 sequences, 64 heads x 64, N 128, bf16
// (1.08 GB): 193 us, 5.6 TB/s.
#include "sf_seq.h"

namespace sf {

namespace {

constexpr int kThreads = 256;

template <typename T, int TN, int R, bool VEC, bool ONCE>
__global__ __launch_bounds__(kThreads) void k_scan_seq(ScanArgs a, int slices) {
  constexpr int kRows = kThreads / TN;  // rows a pass
  const int64_t block = a.block0 + blockIdx.x;
  const int64_t bh = block / slices;
  const int slice = (int)(block - bh * slices);
  const int64_t b = bh / a.heads;
  const int hd = (int)(bh - b * a.heads);
  const int g = hd / (a.heads / a.groups);
  const int nl = threadIdx.x % TN, n0 = nl * 4;
  const int p0 = slice * kRows * R + threadIdx.x / TN;
  const int P = a.head_dim, N = a.state_dim;
  int64_t first, n;
  seq_rows(a.seq, b, first, n);
  const T* __restrict__ x = static_cast<const T*>(a.x) + b * a.x_b + first * a.x_t + hd * a.x_h;
  const T* __restrict__ dt = static_cast<const T*>(a.dt) + b * a.dt_b + first * a.dt_t + hd * a.dt_h;
  const T* __restrict__ B = static_cast<const T*>(a.b) + b * a.b_b + first * a.b_t + g * a.b_g;
  const T* __restrict__ C = static_cast<const T*>(a.c) + b * a.c_b + first * a.c_t + g * a.c_g;
  T* __restrict__ y = static_cast<T*>(a.y) + b * a.y_b + first * a.y_t + hd * a.y_h;
  const int64_t slot = seq_slot(a.seq, b);
  const float A = a.A[hd], D = a.D != nullptr ? a.D[hd] : 0.f, bias = a.dt_bias != nullptr ? a.dt_bias[hd] : 0.f;
  const int64_t head_row = (slot * a.heads + hd) * (int64_t)P * N;

  if (a.step && slot < 0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int p = p0 + r * kRows;
      if (nl == 0 && p < P) y[p] = from_f32<T>(0.f);
    }
    return;
  }
  float h[R][4];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int p = p0 + r * kRows;
#pragma unroll
    for (int i = 0; i < 4; ++i) h[r][i] = 0.f;
    if (a.h0 != nullptr && slot >= 0 && p < P) {
      const float* row = a.h0 + head_row + (int64_t)p * N;
      if constexpr (VEC) {
        if (n0 < N) load_any_f32<float, 4, ONCE>(row + n0, h[r]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n0 + i < N) h[r][i] = row[n0 + i];
      }
    }
  }
  for (int64_t t = 0; t < n; ++t) {
    // (All of a token's loads before the first use: rows and columns past the end read
    // the last ones, and go nowhere.)
    T xr[R], br[4], cr[4];
    Vec<T, 4> bq, cq;
    const T dr = dt[t * a.dt_t];
    if constexpr (VEC) {
      bq = load_any<T, 4>(B + t * a.b_t + min(n0, N - 4));
      cq = load_any<T, 4>(C + t * a.c_t + min(n0, N - 4));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        br[i] = B[t * a.b_t + min(n0 + i, N - 1)];
        cr[i] = C[t * a.c_t + min(n0 + i, N - 1)];
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) xr[r] = x[t * a.x_t + min(p0 + r * kRows, P - 1)];
    float bv[4], cv[4], xv[R], s[R];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bv[i] = to_f32<T>(VEC ? bq.e[i] : br[i]);
      cv[i] = to_f32<T>(VEC ? cq.e[i] : cr[i]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) xv[r] = to_f32<T>(xr[r]);
    float d = to_f32<T>(dr) + bias;
    if (a.softplus) d = softplus(d);
    const float decay = expf(A * d);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float u = d * xv[r];
      s[r] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        h[r][i] = fmaf(decay, h[r][i], u * bv[i]);
        // (Columns past the end stay out of the sum: a state that is not finite
        // times their zero C would not be zero.)
        s[r] = VEC || n0 + i < N ? fmaf(h[r][i], cv[i], s[r]) : s[r];
      }
      if (VEC && n0 >= N) s[r] = 0.f;
    }
#pragma unroll
    for (int off = TN / 2; off > 0; off >>= 1)
#pragma unroll
      for (int r = 0; r < R; ++r) s[r] += __shfl_xor(s[r], off, kWave);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int p = p0 + r * kRows;
      if (nl == 0 && p < P) y[t * a.y_t + p] = from_f32<T>(a.D != nullptr ? fmaf(D, xv[r], s[r]) : s[r]);
    }
  }
  if (a.h1 != nullptr && slot >= 0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int p = p0 + r * kRows;
      if (p >= P) continue;
      float* row = a.h1 + head_row + (int64_t)p * N;
      if constexpr (VEC) {
        if (n0 < N) store_any_f32<float, 4, ONCE>(row + n0, h[r]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n0 + i < N) row[n0 + i] = h[r][i];
      }
    }
  }
}

template <typename T, int TN, int R, bool VEC, bool ONCE = false>
int launch_seq_r(const ScanArgs& a, hipStream_t stream) {
  constexpr int rows = kThreads / TN * R;
  const int slices = (a.head_dim + rows - 1) / rows;
  return launch_blocks(a, &ScanArgs::block0, a.seq.batch * a.heads * slices, [&](const ScanArgs& la, unsigned n) {
    hipLaunchKernelGGL((k_scan_seq<T, TN, R, VEC, ONCE>), dim3(n), dim3(kThreads), 0, stream, la, slices);
  });
}

template <typename T, int TN>
int launch_seq_n(const ScanArgs& a, hipStream_t stream) {
  const bool vec = a.state_dim % 4 == 0;
  // As many rows to a thread as the head has, up to 8 (a step of 256 sequences, 64 heads x
  // 64, N 128: 212 us, with two rows 218, with one 316).
  constexpr int kRows = kThreads / TN;
  const int r = (a.head_dim + kRows - 1) / kRows;
  if (!vec) return r <= 2 ? launch_seq_r<T, TN, 2, false>(a, stream) : launch_seq_r<T, TN, 8, false>(a, stream);
  if (r > 4 && read_once(a.seq.batch * a.heads * (int64_t)a.head_dim * a.state_dim * (int64_t)sizeof(float)))
    return launch_seq_r<T, TN, 8, true, true>(a, stream);
  if (r <= 1) return launch_seq_r<T, TN, 1, true>(a, stream);
  if (r <= 2) return launch_seq_r<T, TN, 2, true>(a, stream);
  if (r <= 4) return launch_seq_r<T, TN, 4, true>(a, stream);
  return launch_seq_r<T, TN, 8, true>(a, stream);
}

template <typename T>
int launch_seq_t(const ScanArgs& a, hipStream_t stream) {
  if (a.state_dim <= 32) return launch_seq_n<T, 8>(a, stream);
  if (a.state_dim <= 64) return launch_seq_n<T, 16>(a, stream);
  if (a.state_dim <= 128) return launch_seq_n<T, 32>(a, stream);
  return launch_seq_n<T, 64>(a, stream);
}

}  // namespace

int launch_scan_seq(const ScanArgs& a, int dtype, hipStream_t stream) {
  timing_begin(K_SCAN_SEQ, stream);
  const int rc = dtype == SF_F16    ? launch_seq_t<__half>(a, stream)
                 : dtype == SF_BF16 ? launch_seq_t<__hip_bfloat16>(a, stream)
                                    : launch_seq_t<float>(a, stream);
  timing_end(K_SCAN_SEQ, stream);
  return rc;
}

}  // namespace sf
