// Causal depthwise convolution over the token axis:
//   y[t, c] = act(bias[c] + sum_k w[c, k] u[t - K + 1 + k, c])
// (u before the sequence's start: the state, or zeros).
//
// A thread owns V neighbouring channels and a run of tokens: the last K - 1 inputs
// stay in registers as the run is walked, every input of the run is one load of 16
// bytes, kBatch of them under way at a time, and the K - 1 before the run are read
// again (from the cache: a neighbouring thread's run).  Bound by HBM: x in, y out;
// 2 x 16384 x 4352 bf16, K = 4: 130 us, 4.4 TB/s; ragged sequences of 16,064 x 1037
// float32, whose rows begin anywhere: 39 us, 3.4 TB/s; one token of 256 x 2304: 10 us, a
// call's own time.
#include "sf_seq.h"
#include "sf_tile.h"

namespace sf {

namespace {

constexpr int kBatch = 8;  // tokens loaded at a time
constexpr int kThreads = 256;

template <typename T, int K, int V>
__global__ __launch_bounds__(kThreads) void k_causal_conv1d(Conv1dArgs a, int cv, int blocks_per_seq, int runs,
                                                            int length, int keep) {
  const int64_t block = a.block0 + blockIdx.x;
  const int64_t b = block / blocks_per_seq;
  const int64_t item = (block - b * blocks_per_seq) * kThreads + threadIdx.x;
  const int run = (int)(item / cv);
  if (run >= runs) return;
  // (A row's last thread takes its last V channels, some of them another's too.)
  const int ch = min((int)(item - (int64_t)run * cv) * V, a.channels - V);
  int64_t first, n;
  seq_rows(a.seq, b, first, n);
  const int64_t t0 = (int64_t)run * length;
  if (t0 >= n && run > 0) return;
  // (max_len sizes the launch: where a sequence is longer, its last run goes on.)
  const int64_t t1 = run == runs - 1 ? n : (t0 + length < n ? t0 + length : n);
  const bool last = t1 == n;
  const T* __restrict__ x = static_cast<const T*>(a.x) + b * a.x_b + first * a.x_t;
  T* __restrict__ y = static_cast<T*>(a.y) + b * a.y_b + first * a.y_t;
  const int64_t slot = seq_slot(a.seq, b);
  const T* before = a.before != nullptr && slot >= 0
                        ? static_cast<const T*>(a.before) + slot * (K - 1) * (int64_t)a.channels
                        : nullptr;
  if (a.step && slot < 0) {
    float z[V];
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = 0.f;
    store_any_f32<T, V>(y + ch, z);
    return;
  }
  float w[K][V], bias[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = a.bias != nullptr ? a.bias[ch + i] : 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) w[k][i] = a.weight[(int64_t)(ch + i) * K + k];
  }
  // u[k]: the input of token t - (K - 1) + k.
  float u[K][V];
#pragma unroll
  for (int k = 0; k < K - 1; ++k) {
    const int64_t t = t0 - (K - 1) + k;
    if (t >= 0) {
      load_any_f32<T, V>(x + t * a.x_t + ch, u[k]);
    } else if (before != nullptr) {
      load_any_f32<T, V>(before + (t + K - 1) * (int64_t)a.channels + ch, u[k]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) u[k][i] = 0.f;
    }
  }
  const T* __restrict__ xt = x + t0 * a.x_t + ch;
  T* __restrict__ yt = y + t0 * a.y_t + ch;
  // One token: u's last input has come in.
  auto token = [&]() {
    float s[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      s[i] = bias[i];
#pragma unroll
      for (int k = 0; k < K; ++k) s[i] = fmaf(w[k][i], u[k][i], s[i]);
      if (a.act == SF_ACT_SILU) s[i] = silu<sizeof(T) == 4>(s[i]);
    }
    store_any_f32<T, V>(yt, s);
    yt += a.y_t;
#pragma unroll
    for (int k = 0; k + 1 < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) u[k][i] = u[k + 1][i];
  };
  int64_t left = t1 - t0;
  for (; left >= kBatch; left -= kBatch) {
    Vec<T, V> in[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      in[j] = load_any<T, V>(xt);
      xt += a.x_t;
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
#pragma unroll
      for (int i = 0; i < V; ++i) u[K - 1][i] = to_f32<T>(in[j].e[i]);
      token();
    }
  }
  for (; left > 0; --left) {
    load_any_f32<T, V>(xt, u[K - 1]);
    xt += a.x_t;
    token();
  }
  if (last && keep && slot >= 0) {
    T* after = static_cast<T*>(a.after) + slot * (K - 1) * (int64_t)a.channels;
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      store_any_f32<T, V>(after + (int64_t)k * a.channels + ch, u[k]);
    }
  }
}

// The final states alone, where they overwrite the initial ones that other
// threads of the convolution read: a thread reads all of its rows first.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_conv1d_state(Conv1dArgs a, int blocks_per_seq) {
  const int64_t block = a.block0 + blockIdx.x;
  const int64_t b = block / blocks_per_seq;
  const int ch = (int)(block - b * blocks_per_seq) * kThreads + threadIdx.x;
  const int64_t slot = seq_slot(a.seq, b);
  if (ch >= a.channels || slot < 0) return;
  int64_t first, n;
  seq_rows(a.seq, b, first, n);
  const T* __restrict__ x = static_cast<const T*>(a.x) + b * a.x_b + first * a.x_t;
  const int m = a.kernel - 1;
  const int64_t row = slot * m * (int64_t)a.channels;
  const T* before = static_cast<const T*>(a.before) + row;
  T* after = static_cast<T*>(a.after) + row;
  T v[8];
  for (int k = 0; k < m; ++k) {
    const int64_t t = n - m + k;
    v[k] = t >= 0 ? x[t * a.x_t + ch] : before[(t + m) * (int64_t)a.channels + ch];
  }
  for (int k = 0; k < m; ++k) after[(int64_t)k * a.channels + ch] = v[k];
}

template <typename T, int K, int V>
int launch_conv1d_v(const Conv1dArgs& a, hipStream_t stream) {
  const int cv = (a.channels + V - 1) / V;
  // Runs as long as leave a few wavefronts for every SIMD (8 tokens read 3 / 8 of their
  // inputs twice, 64 less than a twentieth): 2 x 16384 x 4352 bf16 takes 132 us in runs of
  // 64 and 170 in runs of 8, 2048 x 1024 24 us in runs of 64 and 9 in runs of 8.
  int length = 64;
  while (length > 8 && a.seq.batch * cv * ((a.max_len + length - 1) / length) < (int64_t)num_cus() * 4 * 4 * kWave) length /= 2;
  const int64_t runs = a.max_len > length ? (a.max_len + length - 1) / length : 1;
  const int64_t per_seq = (runs * cv + kThreads - 1) / kThreads;
  // In place: a step's thread holds all that it overwrites; in a prompt the
  // thread that writes a state is not the one that read it, unless there is one
  // run and no channel has two threads.
  const size_t pool = (size_t)a.seq.states * (K - 1) * a.channels * sizeof(T);
  const char *p0 = static_cast<const char*>(a.before), *p1 = static_cast<const char*>(a.after);
  const bool keep = a.after != nullptr && K > 1;
  const bool apart = keep && (runs > 1 || a.channels % V != 0) && a.before != nullptr && p0 < p1 + pool && p1 < p0 + pool;
  int rc = launch_blocks(a, &Conv1dArgs::block0, a.seq.batch * per_seq, [&](const Conv1dArgs& la, unsigned n) {
    hipLaunchKernelGGL((k_causal_conv1d<T, K, V>), dim3(n), dim3(kThreads), 0, stream, la, cv, (int)per_seq,
                       (int)runs, length, keep && !apart ? 1 : 0);
  });
  if (rc != (int)hipSuccess || !apart) return rc;
  const int64_t blocks = (a.channels + kThreads - 1) / kThreads;
  return launch_blocks(a, &Conv1dArgs::block0, a.seq.batch * blocks, [&](const Conv1dArgs& la, unsigned n) {
    hipLaunchKernelGGL((k_conv1d_state<T>), dim3(n), dim3(kThreads), 0, stream, la, (int)blocks);
  });
}

template <typename T, int K>
int launch_conv1d_k(const Conv1dArgs& a, hipStream_t stream) {
  // 16 bytes an access, at any address.  A step in place has one thread to a channel.
  constexpr int V = 16 / sizeof(T);
  return a.channels % V == 0 || (a.channels > V && !a.step) ? launch_conv1d_v<T, K, V>(a, stream)
                                                            : launch_conv1d_v<T, K, 1>(a, stream);
}

template <typename T>
int launch_conv1d_t(const Conv1dArgs& a, hipStream_t stream) {
  switch (a.kernel) {
    case 1: return launch_conv1d_k<T, 1>(a, stream);
    case 2: return launch_conv1d_k<T, 2>(a, stream);
    case 3: return launch_conv1d_k<T, 3>(a, stream);
    case 4: return launch_conv1d_k<T, 4>(a, stream);
    case 5: return launch_conv1d_k<T, 5>(a, stream);
    case 6: return launch_conv1d_k<T, 6>(a, stream);
    case 7: return launch_conv1d_k<T, 7>(a, stream);
    default: return launch_conv1d_k<T, 8>(a, stream);
  }
}

}  // namespace

int launch_conv1d(const Conv1dArgs& a, int dtype, hipStream_t stream) {
  timing_begin(K_CONV1D, stream);
  const int rc = dtype == SF_F16    ? launch_conv1d_t<__half>(a, stream)
                 : dtype == SF_BF16 ? launch_conv1d_t<__hip_bfloat16>(a, stream)
                                    : launch_conv1d_t<float>(a, stream);
  timing_end(K_CONV1D, stream);
  return rc;
}

}  // namespace sf
