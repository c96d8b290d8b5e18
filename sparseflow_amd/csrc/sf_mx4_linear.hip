// The Linear over microscaled 4-bit weights:
//   y[m, n] = bias[n] + sum_k x[m, k] w[n, k]
// A weight of the format is a bf16 number, so that bf16 x goes to the matrix cores as it
// is, f16 in two and float32 in three bf16 parts: every product is exact and the sums are
// float32.  4-bit x goes to the scaled 4-bit instructions.
#include <type_traits>

#include "sf_mx4.h"

namespace sf {
namespace {

// ---- few rows: the weights are read once, straight into the matrix operands -----
//
// A wavefront takes 16 NT weight rows and 16 MT rows of x.  In a step of 128 columns lane
// (r, g) = (lane % 16, lane / 16) holds the whole block g of a weight row r, 16 bytes and one
// scale, and block g of x row r: instruction j takes columns 32 g + 8 j .. + 7 of both (the
// order of a sum's terms is free).  The wavefronts of a workgroup take steps in turn, or U steps
// of which a lane has U blocks next to each other, loaded before the first is worked on; their
// sums meet in LDS.
//
// Bound by the reading of W: 1 x 4096 x 12288 of bf16 10.4 us with W from memory (27 MB, 2.6
// TB/s: launch, first loads and the sums' meeting are a third of it), 1 x 16384 x 16384 46 us
// (3.1 TB/s), 37 x 1000 x 1037 of float32 6.1.
struct Four {};  // x in the format

template <typename T>
struct XBlock {  // a lane's 32 values, as they lie in memory
  Vec<T, 8> v[4];
  // ALL: every block of the step is a whole one.
  template <bool ALL>
  __device__ __forceinline__ void load(const Mx4LinearArgs& a, int64_t m, int b) {
    const T* row = reinterpret_cast<const T*>(a.x) + m * a.x_stride;
    const int64_t k = (int64_t)b * kMx4Block;
    if (ALL || k + kMx4Block <= a.k) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = load_any<T, 8>(row + k + 8 * j);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j].e[i] = k + 8 * j + i < a.k ? row[k + 8 * j + i] : from_f32<T>(0.f);
    }
  }
};
template <>
struct XBlock<Four> {
  u32x4 codes;
  int byte;
  template <bool ALL>
  __device__ __forceinline__ void load(const Mx4LinearArgs& a, int64_t m, int b) {
    const int64_t at = m * a.blocks + b;
    const bool live = ALL || b < a.blocks;
    codes = live ? reinterpret_cast<const u32x4*>(a.x)[at] : u32x4{0, 0, 0, 0};
    byte = live ? a.x_scales[at] : 0;
  }
};

template <typename T, int MT, int NT>
struct RowsStep {
  u32x4 codes[NT];
  uint32_t byte[NT];
  XBlock<T> x[MT];

  template <bool ALL>
  __device__ __forceinline__ void load(const Mx4LinearArgs& a, const int64_t (&wrow)[NT], const int64_t (&m)[MT], int b) {
    const bool live = ALL || b < a.blocks;
#pragma unroll
    for (int q = 0; q < NT; ++q) {
      codes[q] = live ? reinterpret_cast<const u32x4*>(a.w)[wrow[q] + b] : u32x4{0, 0, 0, 0};
      byte[q] = live ? a.w_scales[wrow[q] + b] : 0;
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) x[t].template load<ALL>(a, m[t], b);
  }

  __device__ __forceinline__ void add(f32x4 (&acc)[MT][NT]) const {
    if constexpr (std::is_same<T, Four>::value) {
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const u32x4 xc = x[t].codes;
        const i32x8 xb = {(int)xc.x, (int)xc.y, (int)xc.z, (int)xc.w, 0, 0, 0, 0};
#pragma unroll
        for (int q = 0; q < NT; ++q) {
          const i32x8 wa = {(int)codes[q].x, (int)codes[q].y, (int)codes[q].z, (int)codes[q].w, 0, 0, 0, 0};
          acc[t][q] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, xb, acc[t][q], 4, 4, 0, (int)byte[q], 0, x[t].byte);
        }
      }
    } else {
      constexpr int NP = Parts<T>::n;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bf16x8 wa[NT];
#pragma unroll
        for (int q = 0; q < NT; ++q) wa[q] = mx4_bf16(codes[q][j], mx4_scale(byte[q]));
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          bf16x8 p[NP];
          if constexpr (NP == 1) {
            __builtin_memcpy(&p[0], &x[t].v[j], 16);
          } else {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(x[t].v[j].e[i]);
            split8<NP>(v, p);
          }
#pragma unroll
          for (int k = 0; k < NP; ++k)
#pragma unroll
            for (int q = 0; q < NT; ++q) acc[t][q] = mfma16(wa[q], p[k], acc[t][q]);
        }
      }
    }
  }
};

template <typename T, int MT, int NT, int W, int U>
__global__ __launch_bounds__(W* kWave) void k_mx4_linear_rows(Mx4LinearArgs a) {
  __shared__ f32x4 sums[W][MT * NT][kWave];
  const int lane = lane_id(), wave = threadIdx.x / kWave, r = lane & 15, g = lane >> 4;
  const int64_t tile = a.block0 + blockIdx.x, n0 = tile % a.n_tiles * (16 * NT), m0 = tile / a.n_tiles * (16 * MT);
  int64_t wrow[NT], m[MT];
  f32x4 acc[MT][NT];
#pragma unroll
  for (int q = 0; q < NT; ++q) wrow[q] = (n0 + 16 * q + r < a.n ? n0 + 16 * q + r : a.n - 1) * a.blocks;
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    m[t] = m0 + 16 * t + r < a.m ? m0 + 16 * t + r : a.m - 1;
#pragma unroll
    for (int q = 0; q < NT; ++q) acc[t][q] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int steps = (a.blocks + 3) / 4, whole = (int)(a.k / (4 * U * kMx4Block));
  const int first = __builtin_amdgcn_readfirstlane(wave);
  for (int s = first; s < whole; s += W) {
    RowsStep<T, MT, NT> e[U];
#pragma unroll
    for (int u = 0; u < U; ++u) e[u].template load<true>(a, wrow, m, U * (4 * s + g) + u);
#pragma unroll
    for (int u = 0; u < U; ++u) e[u].add(acc);
  }
  // (The rest begins with the wavefront whose turn it is.)
  for (int s = U * whole + ((first - whole) & (W - 1)); s < steps; s += W) {
    RowsStep<T, MT, NT> e;
    e.template load<false>(a, wrow, m, 4 * s + g);
    e.add(acc);
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int q = 0; q < NT; ++q) sums[wave][t * NT + q][lane] = acc[t][q];
  __syncthreads();
  // Element i of lane (r, g): output n0 + 16 q + 4 g + i of row m0 + 16 t + r.
  for (int tq = wave; tq < MT * NT; tq += W) {
    const int64_t row = m0 + 16 * (tq / NT) + r, c = n0 + 16 * (tq % NT) + 4 * g;
    if (row >= a.m) continue;
    f32x4 v = sums[0][tq][lane];
#pragma unroll
    for (int k = 1; k < W; ++k) v += sums[k][tq][lane];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (c + i >= a.n) continue;
      const float s = v[i] + (a.bias == nullptr ? 0.f : a.bias[c + i]);
      const int64_t at = row * a.y_stride + c + i;
      if (a.y_dtype == SF_F16) reinterpret_cast<__half*>(a.y)[at] = from_f32<__half>(s);
      else if (a.y_dtype == SF_BF16) reinterpret_cast<__hip_bfloat16*>(a.y)[at] = from_f32<__hip_bfloat16>(s);
      else reinterpret_cast<float*>(a.y)[at] = s;
    }
  }
}

template <typename T, int MT, int NT, int W, int U>
int launch_rows(Mx4LinearArgs a, hipStream_t stream) {
  a.n_tiles = (a.n + 16 * NT - 1) / (16 * NT);
  const int64_t blocks = a.n_tiles * ((a.m + 16 * MT - 1) / (16 * MT));
  return launch_blocks(a, &Mx4LinearArgs::block0, blocks, [&](const Mx4LinearArgs& part, unsigned grid) {
    k_mx4_linear_rows<T, MT, NT, W, U><<<grid, W * kWave, 0, stream>>>(part);
  });
}

template <typename T>
constexpr bool four_bits = std::is_same<T, Four>::value;

// Weight rows by how many workgroups they make.
template <typename T, int MT>
int launch_rows_n(const Mx4LinearArgs& a, hipStream_t stream) {
  if constexpr (MT == 1) {
    // As long as x is little beside W, few weight rows a workgroup and four blocks of each at a
    // time (128 bytes of a weight row in one place; x K x N in us: 1 x 4096 x 12288 bf16 12.5 ->
    // 10.4, four 11.7 -> 8.5, 1 x 12288 x 4096 bf16 13.4 -> 11.4, 16 x 12288 x 4096 f32 41 -> 34;
    // but 16 x 12288 x 4096 bf16 20 -> 22, 4 x 8192 x 8192 bf16 15 -> 17 and f32 24 -> 27, f32 of
    // 1000 columns, which are the first wavefronts' alone, 4.7 -> 6.0, 1 x 12288 x 4096 f16 16 -> 19).
    const bool narrow = a.n <= 32 * 160;
    if constexpr (four_bits<T>) return launch_rows<T, 1, 1, 8, 4>(a, stream);
    else if constexpr (Parts<T>::n == 1) {
      if (a.m <= 2 || (narrow && a.m <= 8)) return launch_rows<T, 1, 1, 8, 4>(a, stream);
    } else if constexpr (Parts<T>::n == 3) {
      if (narrow && a.k >= 4096) return launch_rows<T, 1, 1, 8, 4>(a, stream);
    }
  }
  if constexpr (MT > 1 || !four_bits<T>) {
    if (a.n > 64 * 160) return launch_rows<T, MT, MT == 4 ? 2 : 4, 8, 1>(a, stream);
    if (a.n > 32 * 160) return launch_rows<T, MT, 2, 8, 1>(a, stream);
    return launch_rows<T, MT, 1, MT == 4 ? 8 : 16, 1>(a, stream);
  }
}

template <typename T>
int launch_linear(const Mx4LinearArgs& a, bool few, hipStream_t stream) {
  return few || a.m <= 16 ? launch_rows_n<T, 1>(a, stream) : a.m <= 32 ? launch_rows_n<T, 2>(a, stream) : launch_rows_n<T, 4>(a, stream);
}

}  // namespace

int launch_mx4_linear(const Mx4LinearArgs& a, int x_dtype, hipStream_t stream) {
  timing_begin(K_MX4_LINEAR, stream);
  // Where y is so few pieces of 16 x 16 that the CUs hold a workgroup for each, the wavefronts
  // that share its K are worth more than what they read twice (x K x N in us, as wider pieces or
  // tiles / so; 37 x 1000 x 1037: f32 10.3 / 6.1, bf16 8.0 / 4.9; 64 x 8192 x 1024: bf16 35 / 14,
  // f32 77 / 21, four 21 / 8; 128 x 8192 x 1024: bf16 36 / 24; but 200 x 4096 x 1024 bf16 21 / 23,
  // 20 x 4096 x 4096 bf16 10.6 / 12.2).
  const int64_t pieces = (a.m + 15) / 16 * ((a.n + 15) / 16);
  const bool few = pieces <= (a.m <= 32 ? 320 : 512) || (x_dtype == SF_MX4 && a.k >= 4096 && pieces <= 1024);
  // Where tiles of 64 rows fill the CUs by themselves they are better from 33 rows on; with less
  // of them, a wavefront to few columns reads W sooner (this kernel / tiles; 64 x 4096 x 12288:
  // bf16 41 / 22, f32 102 / 45, four 25 / 16; 33 x 4096 x 4096: bf16 13 / 20, f32 45 / 39, four
  // 9 / 14; 17 to 32 rows: never worse by more than a us).
  // (4-bit x whose blocks are no multiple of four, or whose scales or W's are not 4-byte aligned, has
  // no tiles and stays here at any number of rows, where floats would be sooner; four / bf16: 8192 x
  // 4100 x 16380 1860 / 1050, 8192 x 1056 x 4096 201 / 91, 4096 x 192 x 904 13.5 / 8.6.)
  const int64_t filling = x_dtype == SF_F32 ? 2048 : 10240;
  const bool tiles = !few && a.m > (a.n > filling ? 32 : 64) && (x_dtype != SF_MX4 || mx4_gemm_takes_four(a));
  const int rc = tiles                ? launch_mx4_gemm(a, x_dtype, stream)
                 : x_dtype == SF_MX4  ? launch_linear<Four>(a, few, stream)
                 : x_dtype == SF_F16  ? launch_linear<__half>(a, few, stream)
                 : x_dtype == SF_BF16 ? launch_linear<__hip_bfloat16>(a, few, stream)
                                      : launch_linear<float>(a, few, stream);
  timing_end(K_MX4_LINEAR, stream);
  return rc;
}

}  // namespace sf
