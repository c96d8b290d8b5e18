// Floats to microscaled 4-bit blocks and back (see sparseflow.h for the format).
//
// Four lanes to a block, eight values each: a lane's load is 16 bytes of 16-bit rows,
// the block's largest magnitude is two exchanges away, and a lane writes its four bytes
// of codes.  Both directions are bound by memory: 32768 x 8192 of bf16 take 136 us there (4.9
// TB/s) and 116 back (5.8), where a large copy moves 5.15 TB/s.
#include "sf_mx4.h"

namespace sf {
namespace {

constexpr int kThreads = 256;

// Block and first element of this thread's eight, and their row; false behind the last.
__device__ __forceinline__ bool mx4_place(const Mx4Args& a, int64_t item, int64_t& row, int& blk) {
  if (item >= a.rows * a.blocks) return false;
  if (a.rows * a.blocks <= 0x7fffffff) {
    row = (uint32_t)item / (uint32_t)a.blocks;
  } else {
    row = item / a.blocks;
  }
  blk = (int)(item - row * a.blocks);
  return true;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void k_mx4_quantize(Mx4Args a) {
  const int64_t at = (a.block0 + blockIdx.x) * kThreads + threadIdx.x;
  const int part = threadIdx.x & 3;
  int64_t row;
  int blk;
  const bool live = mx4_place(a, at >> 2, row, blk);
  float v[8];
  if (live) {
    const int64_t outer = a.inner == 1 ? row : row / a.inner;
    const T* x = reinterpret_cast<const T*>(a.x) + outer * a.x_o + (row - outer * a.inner) * a.x_i;
    load8<T>(x, (int64_t)blk * kMx4Block + part * 8, a.dim, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
  }
  uint32_t byte;
  const uint32_t codes = mx4_encode(v, byte);
  if (!live) return;
  reinterpret_cast<uint32_t*>(a.codes)[at] = codes;
  if (part == 0) a.scales[at >> 2] = (uint8_t)byte;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void k_mx4_dequantize(Mx4Args a) {
  const int64_t at = (a.block0 + blockIdx.x) * kThreads + threadIdx.x;
  const int part = threadIdx.x & 3;
  int64_t row;
  int blk;
  if (!mx4_place(a, at >> 2, row, blk)) return;
  float v[8];
  mx4_f32(reinterpret_cast<const uint32_t*>(a.codes)[at], mx4_scale(a.scales[at >> 2]), v);
  const int64_t k = (int64_t)blk * kMx4Block + part * 8;
  T* y = reinterpret_cast<T*>(const_cast<void*>(a.x)) + row * a.dim + k;
  if (k + 8 <= a.dim) {
    store_any_f32<T, 8>(y, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < a.dim) y[i] = from_f32<T>(v[i]);
  }
}

template <typename T>
int launch_mx4_of(const Mx4Args& a, bool back, hipStream_t stream) {
  const int64_t blocks = (a.rows * a.blocks * 4 + kThreads - 1) / kThreads;
  return launch_blocks(a, &Mx4Args::block0, blocks, [&](const Mx4Args& part, unsigned grid) {
    if (back) k_mx4_dequantize<T><<<grid, kThreads, 0, stream>>>(part);
    else k_mx4_quantize<T><<<grid, kThreads, 0, stream>>>(part);
  });
}

}  // namespace

int launch_mx4(const Mx4Args& a, int dtype, bool back, hipStream_t stream) {
  const int id = back ? K_MX4_DEQUANTIZE : K_MX4_QUANTIZE;
  timing_begin(id, stream);
  const int rc = dtype == SF_F16    ? launch_mx4_of<__half>(a, back, stream)
                 : dtype == SF_BF16 ? launch_mx4_of<__hip_bfloat16>(a, back, stream)
                                    : launch_mx4_of<float>(a, back, stream);
  timing_end(id, stream);
  return rc;
}

}  // namespace sf
