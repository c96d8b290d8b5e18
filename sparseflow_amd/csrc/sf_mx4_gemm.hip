// The Linear over microscaled 4-bit weights for many rows: tiles of y in the matrix
// cores' accumulators (see sf_mx4_linear.hip for the mathematics and for few rows).
//
// A workgroup makes BM rows x BN columns of y, a wavefront MT x NT tiles of 32 x 32.  A stage
// is 64 columns of x (4-bit x: 128): x and the weights' codes and scales lie in LDS, the
// weights as they are, a quarter of what bf16 would take; each wavefront turns them into bf16
// operands itself.  Lane (row, h) of an instruction has the whole block h of its row, so that
// its codes are one 16-byte read, its scale one byte, and instruction j takes columns
// 32 h + 8 j .. + 7 (of x too: the order of a sum's terms is free).  Rows of x lie in LDS as
// 16-byte units, unit u of row r at u ^ (r >> 1 & 7): 16 rows' reads of one unit meet all banks.
//
// Bound by the matrix cores: 8192 x 4096 x 16384 in 989 us (bf16, 1.11 PFLOP/s where a library
// product of 8192^3 reaches 1.24), 436 with x in 4 bits, its quantising included (2.5 PFLOP/s),
// f16 1960 and float32 2630 (two and three parts).
#include "sf_mx4.h"
#include "sf_tile.h"

namespace sf {
namespace {

// The fewest tiles of a size that it is taken for: what is left of a round of the CUs.
constexpr int64_t kGemmTiles = 192;
constexpr int64_t kCus = 256;

// What a load of columns that are not there reads.
__device__ const u32x4 kNothing = {0, 0, 0, 0};

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 in the clobber list
// 16 and 4 bytes a lane from `base` + the lane's offset into LDS from `to` (a place that all
// lanes name), lane after lane; waited for by gemm_wait.
__device__ __forceinline__ void dma16(const void* base, uint32_t off, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(to) : "m0", "memory");
}
__device__ __forceinline__ void dma4(const void* base, uint32_t off, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(to) : "m0", "memory");
}
// The same from a pointer of the lane's own.
__device__ __forceinline__ void dma16_from(const void* src, uint32_t to) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(to) : "m0", "memory");
}
#pragma clang diagnostic pop
// A place in LDS as those take it, the same in all lanes.
__device__ __forceinline__ uint32_t lds_place(const void* p) {
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_ptr_t)const_cast<void*>(p));
}
// All but the newest N of this wavefront's loads have landed, its LDS reads are done, and
// so are the other wavefronts'.
template <int N>
__device__ __forceinline__ void gemm_wait() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// Tile of the workgroup: those of an XCD (every eighth workgroup) lie side by side, eight
// row tiles to a column tile, so that its L2 holds what they share.
__device__ __forceinline__ void gemm_tile(int64_t id, int64_t mt, int64_t nt, int64_t& m, int64_t& n) {
  const int64_t total = mt * nt, per = total / 8, rest = total % 8, x = id & 7;
  const int64_t t = x * per + (x < rest ? x : rest) + (id >> 3);
  const int64_t group = 8 * nt, g = t / group, first = g * 8;
  const int64_t rows = mt - first < 8 ? mt - first : 8, in = t - g * group;
  m = first + in % rows;
  n = in / rows;
}

// y of a wavefront's tiles.  Column (lane % 32) of the accumulators is a row of y and element
// i its column 8 (i / 4) + 4 h + i % 4: stored from there, a row's lines would be written in
// 16-byte pieces, 32 rows at a time (63 us for a tile of 256 x 256, of the 93 that 4-bit x and
// 4096 columns took).  By way of LDS, 32 rows of 256 bytes or less, the wavefront's own, they
// go out as whole lines.
constexpr int kEpilogueRow = 272;  // bytes; 16 on, other banks

template <typename Y, int MT, int NT>
__device__ __forceinline__ void gemm_store(const Mx4LinearArgs& a, const f32x16 (&acc)[MT][NT], int64_t m0, int64_t n0, int lane,
                                           char* lds) {
  constexpr int PT = NT * 32 * (int)sizeof(Y) <= 256 ? NT : 256 / (32 * (int)sizeof(Y));  // column tiles at a time
  constexpr int V = 16 / (int)sizeof(Y), U = PT * 32 / V;                                 // 16-byte units of a row
  const int h = lane >> 5;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int n1 = 0; n1 < NT; n1 += PT) {
      wave_lds_sync();
#pragma unroll
      for (int nt = 0; nt < PT; ++nt)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = 32 * nt + 8 * q + 4 * h;
          float v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = acc[mt][n1 + nt][4 * q + i];
          store_f32<Y, 4>(reinterpret_cast<Y*>(lds + (lane & 31) * kEpilogueRow) + c, v);
        }
      wave_lds_sync();
#pragma unroll
      for (int k = 0; k < U / 2; ++k) {
        const int row = (k * kWave + lane) / U, u = (k * kWave + lane) % U;
        const Vec<Y, V> q = *reinterpret_cast<const Vec<Y, V>*>(lds + row * kEpilogueRow + 16 * u);
        const int64_t m = m0 + 32 * mt + row, c = n0 + 32 * n1 + V * u;
        if (m >= a.m || c >= a.n) continue;
        Y* y = reinterpret_cast<Y*>(a.y) + m * a.y_stride + c;
        if (c + V <= a.n) {
          __builtin_memcpy(y, &q, 16);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (c + i < a.n) y[i] = q.e[i];
        }
      }
    }
}
template <int MT, int NT>
__device__ __forceinline__ void gemm_store(const Mx4LinearArgs& a, const f32x16 (&acc)[MT][NT], int64_t m0, int64_t n0, int lane,
                                           int wave, char* smem) {
  char* lds = smem + wave * 32 * kEpilogueRow;
  if (a.y_dtype == SF_BF16) gemm_store<__hip_bfloat16>(a, acc, m0, n0, lane, lds);
  else if (a.y_dtype == SF_F16) gemm_store<__half>(a, acc, m0, n0, lane, lds);
  else gemm_store<float>(a, acc, m0, n0, lane, lds);
}

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Tiles of a workgroup: WM x WN wavefronts of MT x NT tiles of 32 x 32 each; S stages.
template <int WM_, int WN_, int MT_, int NT_, int S_>
struct Shape {
  static constexpr int WM = WM_, WN = WN_, MT = MT_, NT = NT_, S = S_;
  static constexpr int waves = WM * WN, threads = waves * kWave, BM = WM * MT * 32, BN = WN * NT * 32;
};

// The sums begin with the bias of their columns from n0.
template <int MT, int NT>
__device__ __forceinline__ void gemm_begin(const Mx4LinearArgs& a, int64_t n0, int h, f32x16 (&acc)[MT][NT], bool bias = true) {
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int64_t c = n0 + 32 * j + 8 * (e >> 2) + 4 * h + (e & 3);
      const float b = a.bias == nullptr || !bias ? 0.f : a.bias[c < a.n ? c : a.n - 1];
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i][j][e] = b;
    }
}

// ---- bf16 x, straight from memory into LDS -------------------------------------------
//
// S stages: while one is worked on, the next has landed or is about to, and others are under
// way.  One barrier a stage.  Every wavefront issues as many loads a stage, so that the waits
// can count them; where there is less to load than wavefronts, several load the same.
template <typename P>
struct alignas(16) Bf16Stage {
  uint16_t x[P::BM][64];
  uint32_t w[P::BN][8];  // 16-byte units, unit u of row r at u ^ (r >> 3 & 1)
  uint32_t ws[P::BN];    // the scales of four blocks, of which the stage has two
};

template <typename P>
__global__ __launch_bounds__(P::threads, 2) void k_mx4_gemm_bf16(Mx4LinearArgs a) {
  constexpr int XL = P::BM / (8 * P::waves), loads = XL + 2;
  extern __shared__ __align__(16) char smem[];
  auto* stage = reinterpret_cast<Bf16Stage<P>*>(smem);
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), r = lane & 31, h = lane >> 5;
  int64_t mi, ni;
  gemm_tile(a.block0 + blockIdx.x, (a.m + P::BM - 1) / P::BM, a.n_tiles, mi, ni);
  const int64_t m0 = mi * P::BM, n0 = ni * P::BN;
  const int steps = a.blocks / 2;

  // This lane's places: rows of x (8 to a load), of codes (32 to a load) and of scales, as
  // offsets into the tile's.
  const uint32_t mlast = (uint32_t)(a.m - m0 < P::BM ? a.m - m0 : P::BM) - 1, nlast = (uint32_t)(a.n - n0 < P::BN ? a.n - n0 : P::BN) - 1;
  uint32_t xo[XL], xu[XL];
#pragma unroll
  for (int i = 0; i < XL; ++i) {
    const uint32_t row = 8 * (XL * wave + i) + (lane >> 3);
    xu[i] = (lane & 7) ^ (row >> 1 & 7);  // its unit of a stage's eight
    xo[i] = (row < mlast ? row : mlast) * (2 * (uint32_t)a.x_stride) + 16 * xu[i];
  }
  static_assert(P::BN / 32 <= P::waves && P::BM % (8 * P::waves) == 0, "a load of codes to a wavefront");
  const int wl = wave % (P::BN / 32), sl = wave % (P::BN / 64);
  const uint32_t wr = 32 * wl + (lane >> 1), wu = (lane & 1) ^ (wr >> 3 & 1);
  const uint32_t wo = (wr < nlast ? wr : nlast) * (16 * (uint32_t)a.blocks) + 16 * wu;
  const uint32_t sr = 64 * sl + lane, so = (sr < nlast ? sr : nlast) * (uint32_t)a.blocks;
  const char* xb = reinterpret_cast<const char*>(a.x) + m0 * a.x_stride * 2;
  const uint8_t* wb = a.w + n0 * a.blocks * 16;
  const uint8_t* sb = a.w_scales + n0 * a.blocks;
  const int units = (int)(a.k / 8);

  // Load i of a stage's: x's, then the codes', then the scales'.
  auto load = [&](int s, int i, Bf16Stage<P>& to) {
    if (i < XL) {
      const uint32_t at = lds_place(&to.x[8 * (XL * wave + i)][0]);
      if (8 * s + 8 <= units) dma16(xb + 128 * (int64_t)s, xo[i], at);
      else dma16_from(8 * s + (int)xu[i] < units ? xb + 128 * (int64_t)s + xo[i] : (const char*)&kNothing, at);
    } else if (i == XL) {
      dma16(wb + 32 * (int64_t)s, wo, lds_place(&to.w[32 * wl][0]));
    } else {
      dma4(sb + 4 * (s >> 1), so, lds_place(&to.ws[64 * sl]));
    }
  };

  const int wm = wave % P::WM * (32 * P::MT), wc = wave / P::WM * (32 * P::NT);
  f32x16 acc[P::MT][P::NT];
  gemm_begin(a, n0 + wc, h, acc);
#pragma unroll
  for (int s = 0; s < P::S - 1; ++s)
    if (s < steps)
#pragma unroll
      for (int i = 0; i < loads; ++i) load(s, i, stage[s]);
  for (int s = 0, at = 0; s < steps; ++s) {
    if (s + P::S - 2 < steps) gemm_wait<(P::S - 2) * loads>();
    else gemm_wait<0>();
    const Bf16Stage<P>& t = stage[at];
    Bf16Stage<P>& next = stage[at == 0 ? P::S - 1 : at - 1];
    at = at == P::S - 1 ? 0 : at + 1;
    const bool more = s + P::S - 1 < steps;
    // Everything that the stage's instructions take is asked for at once; the next loads go out
    // between them.
    u32x4 codes[P::NT];
    uint32_t ws[P::NT];
    bf16x8 xf[4][P::MT];
#pragma unroll
    for (int j = 0; j < P::NT; ++j) {
      const int row = wc + 32 * j + r;
      ws[j] = t.ws[row];
      codes[j] = *reinterpret_cast<const u32x4*>(&t.w[row][4 * (h ^ (row >> 3 & 1))]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < P::MT; ++i) {
        const int row = wm + 32 * i + r;
        xf[k][i] = *reinterpret_cast<const bf16x8*>(&t.x[row][8 * ((4 * h + k) ^ (row >> 1 & 7))]);
      }
    float scale[P::NT];
#pragma unroll
    for (int j = 0; j < P::NT; ++j) scale[j] = mx4_scale(ws[j] >> (16 * (s & 1) + 8 * h) & 255);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int j = 0; j < P::NT; ++j) {
        const bf16x8 wf = mx4_bf16(codes[j][k], scale[j]);
#pragma unroll
        for (int i = 0; i < P::MT; ++i) acc[i][j] = mfma32(wf, xf[k][i], acc[i][j]);
      }
      if (more) {
#pragma unroll
        for (int i = k * loads / 4; i < (k + 1) * loads / 4; ++i) load(s + P::S - 1, i, next);
      }
    }
  }
  __syncthreads();  // (the stages are done with)
  gemm_store(a, acc, m0 + wm, n0 + wc, lane, wave, smem);
}

// ---- x in the format -----------------------------------------------------------------
template <typename P>
struct alignas(16) FourStage {
  uint32_t x[P::BM][16];  // 16-byte units, unit u of row r at u ^ (r >> 2 & 3)
  uint32_t w[P::BN][16];
  uint32_t xs[P::BM], ws[P::BN];
};

template <typename P>
__global__ __launch_bounds__(P::threads, 2) void k_mx4_gemm_four(Mx4LinearArgs a) {
  constexpr int XL = P::BM / (16 * P::waves), WL = P::BN / (16 * P::waves), loads = XL + WL + 1;
  static_assert(P::BM % (16 * P::waves) == 0 && P::BN % (16 * P::waves) == 0, "whole loads to a wavefront");
  extern __shared__ __align__(16) char smem[];
  auto* stage = reinterpret_cast<FourStage<P>*>(smem);
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), r = lane & 31, h = lane >> 5;
  int64_t mi, ni;
  gemm_tile(a.block0 + blockIdx.x, (a.m + P::BM - 1) / P::BM, a.n_tiles, mi, ni);
  const int64_t m0 = mi * P::BM, n0 = ni * P::BN;
  const int steps = a.blocks / 4;

  const uint32_t mlast = (uint32_t)(a.m - m0 < P::BM ? a.m - m0 : P::BM) - 1, nlast = (uint32_t)(a.n - n0 < P::BN ? a.n - n0 : P::BN) - 1;
  const uint32_t row_bytes = 16 * (uint32_t)a.blocks;
  uint32_t xo[XL], wo[WL];
  const int u = (lane & 3) ^ (lane >> 4 & 3);
#pragma unroll
  for (int i = 0; i < XL; ++i) {
    const uint32_t row = 16 * (XL * wave + i) + (lane >> 2);
    xo[i] = (row < mlast ? row : mlast) * row_bytes + 16 * u;
  }
#pragma unroll
  for (int i = 0; i < WL; ++i) {
    const uint32_t row = 16 * (WL * wave + i) + (lane >> 2);
    wo[i] = (row < nlast ? row : nlast) * row_bytes + 16 * u;
  }
  // Scales: the first loads' are x's, the others' the weights'.
  constexpr int SX = P::BM / 64;
  const int sl = wave % (SX + P::BN / 64);
  const uint32_t sr = 64 * (sl < SX ? sl : sl - SX) + lane, slast = sl < SX ? mlast : nlast;
  const uint32_t so = (sr < slast ? sr : slast) * (uint32_t)a.blocks;
  const uint8_t* xb = reinterpret_cast<const uint8_t*>(a.x) + m0 * row_bytes;
  const uint8_t* wb = a.w + n0 * row_bytes;
  const uint8_t* sb = sl < SX ? a.x_scales + m0 * a.blocks : a.w_scales + n0 * a.blocks;

  auto load = [&](int s, int i, FourStage<P>& to) {
    if (i < XL) dma16(xb + 64 * (int64_t)s, xo[i], lds_place(&to.x[16 * (XL * wave + i)][0]));
    else if (i < XL + WL) dma16(wb + 64 * (int64_t)s, wo[i - XL], lds_place(&to.w[16 * (WL * wave + i - XL)][0]));
    else dma4(sb + 4 * s, so, lds_place(sl < SX ? &to.xs[64 * sl] : &to.ws[64 * (sl - SX)]));
  };

  const int wm = wave % P::WM * (32 * P::MT), wc = wave / P::WM * (32 * P::NT);
  f32x16 acc[P::MT][P::NT];
  gemm_begin(a, n0 + wc, h, acc);
#pragma unroll
  for (int s = 0; s < P::S - 1; ++s)
    if (s < steps)
#pragma unroll
      for (int i = 0; i < loads; ++i) load(s, i, stage[s]);
  for (int s = 0, at = 0; s < steps; ++s) {
    if (s + P::S - 2 < steps) gemm_wait<(P::S - 2) * loads>();
    else gemm_wait<0>();
    const FourStage<P>& t = stage[at];
    FourStage<P>& next = stage[at == 0 ? P::S - 1 : at - 1];
    at = at == P::S - 1 ? 0 : at + 1;
    const bool more = s + P::S - 1 < steps;
    // (Lane h has blocks h and 2 + h of its row: the scales' bytes 0 and 2 after the shift.)
    int xs[P::MT], ws[P::NT];
    u32x4 xf[2][P::MT], wf[2][P::NT];
#pragma unroll
    for (int i = 0; i < P::MT; ++i) xs[i] = (int)t.xs[wm + 32 * i + r];
#pragma unroll
    for (int j = 0; j < P::NT; ++j) ws[j] = (int)t.ws[wc + 32 * j + r];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int i = 0; i < P::MT; ++i) {
        const int row = wm + 32 * i + r;
        xf[k][i] = *reinterpret_cast<const u32x4*>(&t.x[row][4 * ((2 * k + h) ^ (row >> 2 & 3))]);
      }
#pragma unroll
      for (int j = 0; j < P::NT; ++j) {
        const int row = wc + 32 * j + r;
        wf[k][j] = *reinterpret_cast<const u32x4*>(&t.w[row][4 * ((2 * k + h) ^ (row >> 2 & 3))]);
      }
    }
#pragma unroll
    for (int i = 0; i < P::MT; ++i) xs[i] = (int)((uint32_t)xs[i] >> (8 * h));
#pragma unroll
    for (int j = 0; j < P::NT; ++j) ws[j] = (int)((uint32_t)ws[j] >> (8 * h));
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int j = 0; j < P::NT; ++j) {
        const i32x8 wv = {(int)wf[k][j].x, (int)wf[k][j].y, (int)wf[k][j].z, (int)wf[k][j].w, 0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < P::MT; ++i) {
          const i32x8 xv = {(int)xf[k][i].x, (int)xf[k][i].y, (int)xf[k][i].z, (int)xf[k][i].w, 0, 0, 0, 0};
          acc[i][j] = k == 0 ? __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv, xv, acc[i][j], 4, 4, 0, ws[j], 0, xs[i])
                             : __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv, xv, acc[i][j], 4, 4, 2, ws[j], 2, xs[i]);
        }
      }
      if (more) {
#pragma unroll
        for (int i = k * loads / 2; i < (k + 1) * loads / 2; ++i) load(s + P::S - 1, i, next);
      }
    }
  }
  __syncthreads();  // (the stages are done with)
  gemm_store(a, acc, m0 + wm, n0 + wc, lane, wave, smem);
}

// ---- any x: through registers, in NP bf16 parts ----------------------------------------
//
// Two stages in LDS, and the two after them on their way in registers: loaded as they lie,
// taken apart and written to LDS while the stage before is worked on.  A barrier does not wait
// for loads.  (With x loaded one stage ahead only, bf16 of 8192 x 4100 x 16380: 1990 us.)
//
// KG groups of wavefronts take stages in turn, each with LDS of its own, and add up what they
// have at the end: where y has no more tiles than there are CUs, the time is a tile's stages one
// after another, half a us each (128 x 4096 x 4096: bf16 32.6 -> 21.4 us, f32 63.6 -> 43;
// 256 x 8192 x 1024: 70 -> 36, 123 -> 78).
template <typename P, int NP>
struct alignas(16) AnyStage {
  uint16_t x[NP][P::BM][64];
  uint32_t w[P::BN][8];
  uint16_t ws[P::BN];  // two blocks' scales
};

__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <typename T, typename P, int KG>
__global__ __launch_bounds__(P::threads* KG, KG == 4 ? 4 : 2) void k_mx4_gemm_any(Mx4LinearArgs a) {
  constexpr int NP = Parts<T>::n, XL = P::BM * 8 / P::threads, RL = P::threads / 8, WL = P::BN * 2 < P::threads ? 1 : P::BN * 2 / P::threads;
  static_assert(P::BM * 8 % P::threads == 0 && (P::BN * 2 % P::threads == 0 || P::threads % (P::BN * 2) == 0), "whole loads to a thread");
  extern __shared__ __align__(16) char smem[];
  const int lane = lane_id(), wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), r = lane & 31, h = lane >> 5;
  const int group = wave_all / P::waves, wave = wave_all % P::waves, tid = threadIdx.x % P::threads;
  auto* stage = reinterpret_cast<AnyStage<P, NP>*>(smem) + 2 * group;
  int64_t mi, ni;
  gemm_tile(a.block0 + blockIdx.x, (a.m + P::BM - 1) / P::BM, a.n_tiles, mi, ni);
  const int64_t m0 = mi * P::BM, n0 = ni * P::BN;
  const int whole = (int)(a.k / 64);  // stages without an end of a row

  // Unit tid % 8 of x's rows tid / 8 + RL i; block tid % 2 of the weights' rows tid / 2 + threads / 2 i
  // (more threads than blocks: some load the same).
  const int xr = tid >> 3, xu = tid & 7, wt = tid % (2 * P::BN), wr = wt >> 1, wu = wt & 1;
  const T* xp[XL];
  const uint8_t *wp[WL], *sp[WL];
#pragma unroll
  for (int i = 0; i < XL; ++i) {
    const int64_t row = m0 + xr + RL * i;
    xp[i] = reinterpret_cast<const T*>(a.x) + (row < a.m ? row : a.m - 1) * a.x_stride + 8 * xu;
  }
#pragma unroll
  for (int i = 0; i < WL; ++i) {
    const int64_t row = n0 + wr + P::threads / 2 * i, at = (row < a.n ? row : a.n - 1) * a.blocks + wu;
    wp[i] = a.w + at * 16;
    sp[i] = a.w_scales + at;
  }

  struct Raw {
    Vec<T, 8> x[XL];
    u32x4 w[WL];
    uint32_t s[WL];
  };
  auto load = [&](int s, Raw& q) {
#pragma unroll
    for (int i = 0; i < XL; ++i) q.x[i] = load_any<T, 8>(xp[i] + 64 * (int64_t)s);
#pragma unroll
    for (int i = 0; i < WL; ++i) {
      q.w[i] = *reinterpret_cast<const u32x4*>(wp[i] + 32 * (int64_t)s);
      q.s[i] = sp[i][2 * (int64_t)s];
    }
  };
  auto put = [&](const Raw& q, AnyStage<P, NP>& to) {
#pragma unroll
    for (int i = 0; i < XL; ++i) {
      const int row = xr + RL * i;
      bf16x8 p[NP];
      if constexpr (NP == 1) {
        __builtin_memcpy(&p[0], &q.x[i], 16);
      } else {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = to_f32<T>(q.x[i].e[e]);
        split8<NP>(v, p);
      }
#pragma unroll
      for (int k = 0; k < NP; ++k) *reinterpret_cast<bf16x8*>(&to.x[k][row][8 * (xu ^ (row >> 1 & 7))]) = p[k];
    }
#pragma unroll
    for (int i = 0; i < WL; ++i) {
      const int row = wr + P::threads / 2 * i;
      *reinterpret_cast<u32x4*>(&to.w[row][4 * (wu ^ (row >> 3 & 1))]) = q.w[i];
      reinterpret_cast<uint8_t*>(to.ws)[2 * row + wu] = (uint8_t)q.s[i];
    }
  };

  const int wm = wave % P::WM * (32 * P::MT), wc = wave / P::WM * (32 * P::NT);
  f32x16 acc[P::MT][P::NT];
  gemm_begin(a, n0 + wc, h, acc, group == 0);
  auto work = [&](const AnyStage<P, NP>& t) {
    u32x4 codes[P::NT];
    float scale[P::NT];
#pragma unroll
    for (int j = 0; j < P::NT; ++j) {
      const int row = wc + 32 * j + r;
      codes[j] = *reinterpret_cast<const u32x4*>(&t.w[row][4 * (h ^ (row >> 3 & 1))]);
      scale[j] = mx4_scale((uint32_t)t.ws[row] >> (8 * h) & 255);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      bf16x8 wf[P::NT];
#pragma unroll
      for (int j = 0; j < P::NT; ++j) wf[j] = mx4_bf16(codes[j][k], scale[j]);
#pragma unroll
      for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int i = 0; i < P::MT; ++i) {
          const int row = wm + 32 * i + r;
          const bf16x8 xf = *reinterpret_cast<const bf16x8*>(&t.x[q][row][8 * ((4 * h + k) ^ (row >> 1 & 7))]);
#pragma unroll
          for (int j = 0; j < P::NT; ++j) acc[i][j] = mfma32(wf[j], xf, acc[i][j]);
        }
    }
  };

  if (whole > 0) {
    // (Behind the last whole stage it is loaded again: loads that only some iterations make would
    // be waited for at once.)
    auto stage_of = [&](int i) { return group + KG * i < whole ? group + KG * i : whole - 1; };
    const int turns = (whole + KG - 1) / KG;
    Raw raw[2];
    load(stage_of(0), raw[0]);
    load(stage_of(1), raw[1]);
    put(raw[0], stage[0]);
    load(stage_of(2), raw[0]);
    lds_barrier();
    for (int i = 0; i < turns; i += 2) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (i + u >= turns) break;
        if (KG == 1 || group + KG * (i + u) < whole) work(stage[u]);
        put(raw[1 - u], stage[1 - u]);
        load(stage_of(i + u + 3), raw[1 - u]);
        lds_barrier();
      }
    }
  }
  if (a.k % 64 != 0 && group == 0) {
    Raw end;
#pragma unroll
    for (int i = 0; i < XL; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int64_t k = 64 * (int64_t)whole + 8 * xu + e;
        end.x[i].e[e] = k < a.k ? xp[i][64 * (int64_t)whole + e] : from_f32<T>(0.f);
      }
#pragma unroll
    for (int i = 0; i < WL; ++i) {
      const bool there = 2 * whole + wu < a.blocks;
      end.w[i] = there ? *reinterpret_cast<const u32x4*>(wp[i] + 32 * (int64_t)whole) : u32x4{0, 0, 0, 0};
      end.s[i] = there ? sp[i][2 * (int64_t)whole] : 0;
    }
    put(end, stage[0]);
  }
  if (a.k % 64 != 0) {
    lds_barrier();
    if (group == 0) work(stage[0]);
  }
  if constexpr (KG > 1) {
    // A wavefront's sums of the groups behind the first, [tile, element, lane].
    __syncthreads();
    float* sums = reinterpret_cast<float*>(smem);
    constexpr int per = P::MT * P::NT * 16 * kWave;
    if (group > 0) {
#pragma unroll
      for (int i = 0; i < P::MT; ++i)
#pragma unroll
        for (int j = 0; j < P::NT; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            sums[((group - 1) * P::waves + wave) * per + ((i * P::NT + j) * 16 + e) * kWave + lane] = acc[i][j][e];
    }
    __syncthreads();
    if (group == 0) {
#pragma unroll
      for (int g = 0; g < KG - 1; ++g)
#pragma unroll
        for (int i = 0; i < P::MT; ++i)
#pragma unroll
          for (int j = 0; j < P::NT; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] += sums[(g * P::waves + wave) * per + ((i * P::NT + j) * 16 + e) * kWave + lane];
    }
    __syncthreads();  // (a wavefront's rows on their way out lie over sums that others read)
    if (group > 0) return;
  } else {
    __syncthreads();  // (the stages are done with)
  }
  gemm_store(a, acc, m0 + wm, n0 + wc, lane, wave, smem);
}

template <auto K, typename P, typename Stage, int KG = 1>
int launch_gemm(Mx4LinearArgs a, hipStream_t stream) {
  constexpr int stages = KG * P::S * (int)sizeof(Stage), rows = P::waves * 32 * kEpilogueRow;
  constexpr int sums = (KG - 1) * P::waves * P::MT * P::NT * 16 * kWave * 4;
  constexpr int most = rows > sums ? rows : sums, lds = stages > most ? stages : most;
  static_assert(lds <= kMaxLdsBytes, "LDS");
  const int rc = set_lds_limit_once<K>(lds);
  if (rc != (int)hipSuccess) return rc;
  a.n_tiles = (a.n + P::BN - 1) / P::BN;
  return launch_blocks(a, &Mx4LinearArgs::block0, a.n_tiles * ((a.m + P::BM - 1) / P::BM),
                       [&](const Mx4LinearArgs& part, unsigned grid) { K<<<grid, P::threads * KG, lds, stream>>>(part); });
}

template <typename P>
int launch_bf16(const Mx4LinearArgs& a, hipStream_t stream) {
  return launch_gemm<k_mx4_gemm_bf16<P>, P, Bf16Stage<P>>(a, stream);
}
template <typename P>
int launch_four(const Mx4LinearArgs& a, hipStream_t stream) {
  return launch_gemm<k_mx4_gemm_four<P>, P, FourStage<P>>(a, stream);
}
template <typename T, typename P, int KG>
int launch_any(const Mx4LinearArgs& a, hipStream_t stream) {
  return launch_gemm<k_mx4_gemm_any<T, P, KG>, P, AnyStage<P, Parts<T>::n>, KG>(a, stream);
}

// How many tiles of bm x bn y has.
int64_t tiles_of(const Mx4LinearArgs& a, int bm, int bn) { return (a.m + bm - 1) / bm * ((a.n + bn - 1) / bn); }

template <typename T>
int launch_any(const Mx4LinearArgs& a, hipStream_t stream) {
  if constexpr (Parts<T>::n == 1) {
    if (tiles_of(a, 256, 256) >= kGemmTiles) return launch_any<T, Shape<4, 2, 2, 4, 2>, 1>(a, stream);
  }
  if (tiles_of(a, 128, 256) >= kGemmTiles) return launch_any<T, Shape<2, 4, 2, 2, 2>, 1>(a, stream);
  // (2050 x 6000, bf16 / f32 in us: 65 rows of 188 tiles take 13.3 / 24.9 in groups and 15.2 / 37.6
  // without, 256 rows of 376 tiles 26.7 / 50.4 and 19.5 / 45.7.)
  if (tiles_of(a, 64, 64) <= kCus) return launch_any<T, Shape<2, 2, 1, 1, 2>, Parts<T>::n == 1 ? 4 : 2>(a, stream);
  return launch_any<T, Shape<2, 2, 1, 1, 2>, 1>(a, stream);
}

}  // namespace

bool mx4_gemm_takes_four(const Mx4LinearArgs& a) {
  return a.blocks % 4 == 0 && a.blocks < 1 << 19 && aligned_to(a.x_scales, 4) && aligned_to(a.w_scales, 4);
}

int launch_mx4_gemm(const Mx4LinearArgs& a, int x_dtype, hipStream_t stream) {
  const bool large = tiles_of(a, 256, 256) >= kGemmTiles, middle = tiles_of(a, 128, 128) >= kGemmTiles;
  if (x_dtype == SF_MX4)
    return large    ? launch_four<Shape<4, 2, 2, 4, 3>>(a, stream)
           : middle ? launch_four<Shape<2, 2, 2, 2, 3>>(a, stream)
                    : launch_four<Shape<2, 2, 1, 1, 6>>(a, stream);
  if (x_dtype == SF_F32) return launch_any<float>(a, stream);
  if (x_dtype == SF_F16) return launch_any<__half>(a, stream);
  // (Offsets within a tile are 32-bit.)
  const bool direct = aligned_to(a.x, 16) && a.x_stride % 8 == 0 && a.k % 8 == 0 && a.blocks % 4 == 0 &&
                      aligned_to(a.w_scales, 4) && a.x_stride >= 0 && a.x_stride < 1 << 22 && a.blocks < 1 << 19;
  if (!direct) return launch_any<__hip_bfloat16>(a, stream);
  // (The smallest tiles, one to a CU: 100 x 4096 x 4096 20.8 us in groups of stages, 32.5 here.)
  const bool few = tiles_of(a, 64, 64) <= kCus;
  return large    ? launch_bf16<Shape<4, 2, 2, 4, 3>>(a, stream)
         : middle ? launch_bf16<Shape<2, 2, 2, 2, 3>>(a, stream)
         : few    ? launch_any<__hip_bfloat16>(a, stream)
                  : launch_bf16<Shape<2, 2, 1, 1, 6>>(a, stream);
}

}  // namespace sf
