// The Linear over microscaled 4-bit weights:
//   y[m, n] = bias[n] + sum_k x[m, k] w[n, k]
// A weight of the format is a bf16 number, so that bf16 x goes to the matrix cores as it
// is, f16 in two and float32 in three bf16 parts: every product is exact and the sums are
// float32.  4-bit x goes to the scaled 4-bit instructions.
#include "sf_mx4.h"

namespace sf {
namespace {

// ---- few rows: the weights are read once, straight into the matrix operands -----
//
// A wavefront takes 16 weight rows and 16 MT rows of x.  In a step of 128 columns lane
// (r, g) = (lane % 16, lane / 16) holds the whole block g of weight row r, 16 bytes and one
// scale, and block g of x row r: instruction j takes columns 32 g + 8 j .. + 7 of both (the
// order of a sum's terms is free).  The wavefronts of a workgroup take steps in turn; their
// sums meet in LDS.
constexpr int kRowsWaves = 4;

struct Four {};  // x in the format

template <typename T, int MT>
__global__ __launch_bounds__(kRowsWaves* kWave) void k_mx4_linear_rows(Mx4LinearArgs a) {
  constexpr bool FOUR = sizeof(T) == sizeof(Four);
  __shared__ float sums[kRowsWaves][MT][kWave][4];
  const int lane = lane_id(), wave = threadIdx.x / kWave, r = lane & 15, g = lane >> 4;
  const int64_t tile = a.block0 + blockIdx.x, n0 = (tile % a.n_tiles) * 16, m0 = tile / a.n_tiles * (16 * MT);
  const int64_t n = n0 + r < a.n ? n0 + r : a.n - 1;
  const uint8_t* w = a.w + n * a.blocks * 16;
  const uint8_t* ws = a.w_scales + n * a.blocks;
  f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  int64_t m[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) m[t] = m0 + 16 * t + r < a.m ? m0 + 16 * t + r : a.m - 1;
  const int steps = (a.blocks + 3) / 4;
  for (int s = wave; s < steps; s += kRowsWaves) {
    const int b = 4 * s + g;
    const bool live = b < a.blocks;
    const u32x4 codes = live ? *reinterpret_cast<const u32x4*>(w + (int64_t)b * 16) : u32x4{0, 0, 0, 0};
    const uint32_t byte = live ? ws[b] : 0;
    if constexpr (FOUR) {
      const i32x8 wa = {(int)codes.x, (int)codes.y, (int)codes.z, (int)codes.w, 0, 0, 0, 0};
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const int64_t at = m[t] * a.blocks + b;
        const u32x4 xc = live ? reinterpret_cast<const u32x4*>(a.x)[at] : u32x4{0, 0, 0, 0};
        const int xs = live ? a.x_scales[at] : 0;
        const i32x8 xb = {(int)xc.x, (int)xc.y, (int)xc.z, (int)xc.w, 0, 0, 0, 0};
        acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, xb, acc[t], 4, 4, 0, (int)byte, 0, xs);
      }
    } else {
      constexpr int NP = Parts<T>::n;
      const float scale = mx4_scale(byte);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bf16x8 wa = mx4_bf16(codes[j], scale);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          float v[8];
          load8<T>(reinterpret_cast<const T*>(a.x) + m[t] * a.x_stride, (int64_t)b * kMx4Block + 8 * j, a.k, v);
          bf16x8 p[NP];
          split8<NP>(v, p);
#pragma unroll
          for (int q = 0; q < NP; ++q) acc[t] = mfma16(wa, p[q], acc[t]);
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[wave][t][lane][i] = acc[t][i];
  __syncthreads();
  // Element i of lane (r, g): output n0 + 4 g + i of row m0 + 16 t + r.
  for (int t = wave; t < MT; t += kRowsWaves) {
    const int64_t row = m0 + 16 * t + r;
    if (row >= a.m) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t c = n0 + 4 * g + i;
      if (c >= a.n) continue;
      float v = a.bias == nullptr ? 0.f : a.bias[c];
#pragma unroll
      for (int k = 0; k < kRowsWaves; ++k) v += sums[k][t][lane][i];
      const int64_t at = row * a.y_stride + c;
      if (a.y_dtype == SF_F16) reinterpret_cast<__half*>(a.y)[at] = from_f32<__half>(v);
      else if (a.y_dtype == SF_BF16) reinterpret_cast<__hip_bfloat16*>(a.y)[at] = from_f32<__hip_bfloat16>(v);
      else reinterpret_cast<float*>(a.y)[at] = v;
    }
  }
}

template <typename T, int MT>
int launch_rows(Mx4LinearArgs a, hipStream_t stream) {
  a.n_tiles = (a.n + 15) / 16;
  const int64_t blocks = a.n_tiles * ((a.m + 16 * MT - 1) / (16 * MT));
  return launch_blocks(a, &Mx4LinearArgs::block0, blocks, [&](const Mx4LinearArgs& part, unsigned grid) {
    k_mx4_linear_rows<T, MT><<<grid, kRowsWaves * kWave, 0, stream>>>(part);
  });
}

template <typename T>
int launch_linear(const Mx4LinearArgs& a, hipStream_t stream) {
  return a.m <= 16 ? launch_rows<T, 1>(a, stream) : a.m <= 32 ? launch_rows<T, 2>(a, stream) : launch_rows<T, 4>(a, stream);
}

}  // namespace

int launch_mx4_linear(const Mx4LinearArgs& a, int x_dtype, hipStream_t stream) {
  timing_begin(K_MX4_LINEAR, stream);
  const int rc = x_dtype == SF_MX4    ? launch_linear<Four>(a, stream)
                 : x_dtype == SF_F16  ? launch_linear<__half>(a, stream)
                 : x_dtype == SF_BF16 ? launch_linear<__hip_bfloat16>(a, stream)
                                      : launch_linear<float>(a, stream);
  timing_end(K_MX4_LINEAR, stream);
  return rc;
}

}  // namespace sf
