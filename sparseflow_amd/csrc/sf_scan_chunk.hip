// Selective state space scan of prompts, chunk by chunk on the matrix cores.
//
// With L_t the sum of log2(exp(A d)) over a chunk's tokens up to t, and h the
// state before it,
//   y_i = 2^L_i C_i h^T + sum_{j <= i} (C_i . B_j) 2^(L_i - L_j) d_j x_j + D x_i
//   h  <- 2^L_end h + sum_j (2^(L_end - L_j) d_j x_j) (outer) B_j
// so a chunk of Q tokens is four products: G = B C^T (shared by the heads of a
// group), h C^T, x^T S with S the decayed and masked G, and B^T v with v the
// decayed x.
//
// A wavefront owns 32 columns of one head's x and the state's rows for them, and
// walks the chunks with that state in its accumulators; the wavefronts of a
// workgroup share B, C and G in LDS.  Every product is laid out so that what one
// leaves in the accumulators (lane = column, registers = rows 8 q + 4 half + e) is
// an operand of the next as it stands: G's are the S of the third product, the
// state's the h of the second.  B and x are also needed with tokens along the
// registers: they are read from LDS transposed.
//
// Rounding.  bf16: C, B and x are exact; S and h are rounded to bf16 as operands
// of y, which is rounded to bf16 itself.  v is split into three bf16 parts (its 24
// bits), so that the state, which is summed up over all tokens, stays a float32
// one.  float32 and f16 inputs use the float32 matrix instructions.  L is summed in
// 64 bits: differences of it are exponents.
//
// Few heads and long sequences: the token axis is cut into segments.  A first
// pass walks each segment from a zero state for its own part of the state
// (the last product alone), a second one chains the parts, and the main pass
// starts each segment from its true state.
#include "sf_seq.h"
#include "sf_tile.h"

namespace sf {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

constexpr int kSlice = 32;   // columns of x of a wavefront
constexpr int kMaxWaves = 4;

// ---- the two kinds of products ------------------------------------------------
// A fragment is a lane's 8 values of a 16-deep slice of an operand: depths
// 4 half + {0, 1, 2, 3} and 8 + 4 half + {0, 1, 2, 3}, half = lane / 32.

struct MathBf16 {
  typedef uint16_t E;      // as in LDS
  typedef bf16x8 Frag;
  static constexpr int Q = 64;
  static constexpr int kUnit = 8;  // elements of 16 bytes
  static constexpr int kXStride = 40;
  static constexpr int kPlanes = 3;
  static constexpr bool kPair = false;  // L as one float in the chunk

  // Row of the 16-byte unit u of token j's row: spread so that neither a read
  // of one unit of 16 rows nor a transposed one of two units of 4 rows meets a
  // bank twice.
  template <int NP>
  static __device__ __forceinline__ int unit(int j, int u) {
    if constexpr (NP >= 128) return u ^ ((2 * (j & 7)) | ((j >> 3) & 1));
    else if constexpr (NP == 64) return u ^ ((2 * ((j >> 1) & 3)) | ((j >> 3) & 1));
    else return u ^ ((2 * ((j >> 2) & 1)) | ((j >> 3) & 1));
  }
  // Tokens as lanes: row j of tile m [.][NP], depths from n0 = 16 k.
  template <int NP>
  static __device__ __forceinline__ Frag row(const E* m, int j, int k, int half) {
    const bf16x4 lo = *reinterpret_cast<const bf16x4*>(m + j * NP + unit<NP>(j, 2 * k) * 8 + 4 * half);
    const bf16x4 hi = *reinterpret_cast<const bf16x4*>(m + j * NP + unit<NP>(j, 2 * k + 1) * 8 + 4 * half);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  // Tokens as depth: columns n0 + lane % 32 of tile m, tokens from 16 k.  Four
  // lanes point at a token's 16 columns, and lane l of each 16 gets column l of
  // the four tokens.
  static __device__ __forceinline__ bf16x4 transposed(const E* p) {
    typedef __attribute__((address_space(3))) bf16x4 Lds;
    return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((Lds*)(const_cast<E*>(p)));
  }
  template <int NP>
  static __device__ __forceinline__ Frag col(const E* m, int n0, int k, int lane) {
    const int half = lane >> 5, s = lane & 15, n = n0 + (lane & 16) + 4 * (s & 3);
    const int j = 16 * k + 4 * half + (s >> 2);
    const bf16x4 lo = transposed(m + j * NP + unit<NP>(j, n >> 3) * 8 + (n & 7));
    const bf16x4 hi = transposed(m + (j + 8) * NP + unit<NP>(j + 8, n >> 3) * 8 + (n & 7));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  static __device__ __forceinline__ Frag xcol(const E* x, int k, int lane) {
    const int half = lane >> 5, s = lane & 15, n = (lane & 16) + 4 * (s & 3);
    const int j = 16 * k + 4 * half + (s >> 2);
    const bf16x4 lo = transposed(x + j * kXStride + n);
    const bf16x4 hi = transposed(x + (j + 8) * kXStride + n);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  static __device__ __forceinline__ Frag of(const float (&v)[8]) {
    Frag f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (__bf16)v[e];
    return f;
  }
  static __device__ __forceinline__ float get(const Frag& f, int e) { return (float)f[e]; }
  static __device__ __forceinline__ bool finite(const Frag (&x)[Q / 16]) {
    typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
    u16x8 most = {};
#pragma unroll
    for (int k = 0; k < Q / 16; ++k)
      most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x8, x[k]) & (uint16_t)0x7fff);
    bool ok = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) ok = ok && most[e] < 0x7f80;
    return ok;
  }
  static __device__ __forceinline__ void four(const E* p, float (&v)[4]) {
    const bf16x4 q = *reinterpret_cast<const bf16x4*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)q[e];
  }
  // v as a sum of kPlanes fragments.
  static __device__ __forceinline__ void split(const float (&v)[8], Frag (&f)[kPlanes]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float r = v[e];
#pragma unroll
      for (int p = 0; p < kPlanes; ++p) {
        f[p][e] = (__bf16)r;
        r -= (float)f[p][e];
      }
    }
  }
  static __device__ __forceinline__ f32x16 mma(const Frag& a, const Frag& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ E pack(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
};

struct MathF32 {
  typedef float E;
  struct Frag {
    float e[8];
  };
  static constexpr int Q = 32;
  static constexpr int kUnit = 4;
  static constexpr int kXStride = 36;
  static constexpr int kPlanes = 1;
  static constexpr bool kPair = true;

  template <int NP>
  static __device__ __forceinline__ int unit(int j, int u) {
    return u ^ (j & 7);
  }
  template <int NP>
  static __device__ __forceinline__ Frag row(const E* m, int j, int k, int half) {
    Frag f;
    const float4 lo = *reinterpret_cast<const float4*>(m + j * NP + unit<NP>(j, 4 * k + half) * 4);
    const float4 hi = *reinterpret_cast<const float4*>(m + j * NP + unit<NP>(j, 4 * k + 2 + half) * 4);
    f.e[0] = lo.x, f.e[1] = lo.y, f.e[2] = lo.z, f.e[3] = lo.w;
    f.e[4] = hi.x, f.e[5] = hi.y, f.e[6] = hi.z, f.e[7] = hi.w;
    return f;
  }
  template <int NP>
  static __device__ __forceinline__ Frag col(const E* m, int n0, int k, int lane) {
    const int half = lane >> 5, n = n0 + (lane & 31);
    Frag f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int j = 16 * k + 8 * (e >> 2) + 4 * half + (e & 3);
      f.e[e] = m[j * NP + unit<NP>(j, n >> 2) * 4 + (n & 3)];
    }
    return f;
  }
  static __device__ __forceinline__ Frag xcol(const E* x, int k, int lane) {
    const int half = lane >> 5;
    Frag f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f.e[e] = x[(16 * k + 8 * (e >> 2) + 4 * half + (e & 3)) * kXStride + (lane & 31)];
    return f;
  }
  static __device__ __forceinline__ Frag of(const float (&v)[8]) {
    Frag f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f.e[e] = v[e];
    return f;
  }
  static __device__ __forceinline__ float get(const Frag& f, int e) { return f.e[e]; }
  static __device__ __forceinline__ bool finite(const Frag (&x)[Q / 16]) {
    bool ok = true;
#pragma unroll
    for (int k = 0; k < Q / 16; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) ok = ok && fabsf(x[k].e[e]) < __builtin_huge_valf();
    return ok;
  }
  static __device__ __forceinline__ void four(const E* p, float (&v)[4]) { load_f32<float, 4>(p, v); }
  static __device__ __forceinline__ void split(const float (&v)[8], Frag (&f)[kPlanes]) { f[0] = of(v); }
  static __device__ __forceinline__ f32x16 mma(const Frag& a, const Frag& b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.e[e], b.e[e], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ E pack(float v) { return v; }
};

// Per token of a chunk, for one head.
template <int Q>
struct alignas(16) ChunkScalars {
  float l[Q];   // L
  float ll[Q];  // what L loses as one float
  float d[Q];
  float w[Q];   // 2^(L_end - L) d
  float ab[Q];  // tokens before 32: 2^(L_31 - L) d, from 32 on: 2^(L - L_31)
};

template <typename M, int NP>
struct ChunkLds {
  static constexpr int tile = M::Q * NP * (int)sizeof(typename M::E);
  static constexpr int tiles = M::Q == 64 ? 3 : 1;  // 32 x 32 tiles of G on and below the diagonal
  static constexpr int x = M::Q * M::kXStride * (int)sizeof(typename M::E);
  static constexpr int wave = x + (int)sizeof(ChunkScalars<M::Q>);
  static constexpr int bytes(int waves, bool states) {
    return (states ? tile : 2 * tile + tiles * 4096) + waves * wave;
  }
};

// kUnit elements of a row into LDS; what lies outside becomes 0.
template <typename T, typename M>
__device__ __forceinline__ void stage_unit(typename M::E* to, const T* __restrict__ from, int left, bool vec) {
  float v[M::kUnit];
  if (vec && left >= M::kUnit) {
    if constexpr (sizeof(T) == 2 && sizeof(typename M::E) == 2) {
      *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
      return;
    } else {
      load_f32<T, M::kUnit>(from, v);
    }
  } else {
#pragma unroll
    for (int e = 0; e < M::kUnit; ++e) v[e] = e < left ? to_f32<T>(from[e]) : 0.f;
  }
#pragma unroll
  for (int e = 0; e < M::kUnit; ++e) to[e] = M::pack(v[e]);
}

// STATES: a segment's own part of the state, from a zero state, to `parts`, with
// the sum of its exponents to `sums`.  Otherwise y, from the segment's true state.
template <typename T, typename M, int NP, bool STATES>
__global__ __launch_bounds__(64 * kMaxWaves, NP == 256 ? 1 : 2) void k_scan_chunk(ScanArgs a, ScanSplit sp, bool vec) {
  typedef typename M::E E;
  typedef typename M::Frag Frag;
  constexpr int Q = M::Q, KB = Q / 16, IT = Q / 32, NT = NP / 32;
  constexpr int U = M::kUnit;
  typedef ChunkLds<M, NP> Lds;
  extern __shared__ __align__(16) char lds[];
  const int lane = lane_id(), half = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int threads = blockDim.x;
  E* s_b = reinterpret_cast<E*>(lds);
  E* s_c = reinterpret_cast<E*>(lds + Lds::tile);
  float* s_g = reinterpret_cast<float*>(lds + 2 * Lds::tile);
  char* s_wave = lds + (STATES ? Lds::tile : 2 * Lds::tile + Lds::tiles * 4096) + wave * Lds::wave;
  E* s_x = reinterpret_cast<E*>(s_wave);
  ChunkScalars<Q>& sc = *reinterpret_cast<ChunkScalars<Q>*>(s_wave + Lds::x);

  // This workgroup's sequence, segment and group; this wavefront's head and columns.
  int64_t item = a.block0 + blockIdx.x;
  const int ub = (int)(item % sp.blocks);
  item /= sp.blocks;
  const int g = (int)(item % a.groups);
  item /= a.groups;
  const int seg = (int)(item % (STATES ? sp.segments - 1 : sp.segments));
  const int64_t b = item / (STATES ? sp.segments - 1 : sp.segments);
  const int per_group = a.heads / a.groups, slices = (a.head_dim + kSlice - 1) / kSlice;
  const int unit = ub * (threads / 64) + wave;
  const bool on = unit < per_group * slices;
  const int hd = g * per_group + (on ? unit / slices : 0);
  const int p0 = on ? unit % slices * kSlice : 0;
  const int P = a.head_dim, N = a.state_dim;
  int64_t first, n;
  seq_rows(a.seq, b, first, n);
  const int64_t per_seg = (int64_t)sp.chunks * Q;
  int64_t t0 = seg * per_seg, t1 = t0 + per_seg;
  if (t1 > n || (!STATES && seg == sp.segments - 1)) t1 = n;
  const T* __restrict__ x = static_cast<const T*>(a.x) + b * a.x_b + first * a.x_t + hd * a.x_h + p0;
  const T* __restrict__ dt = static_cast<const T*>(a.dt) + b * a.dt_b + first * a.dt_t + hd * a.dt_h;
  const T* __restrict__ B = static_cast<const T*>(a.b) + b * a.b_b + first * a.b_t + g * a.b_g;
  const T* __restrict__ C = static_cast<const T*>(a.c) + b * a.c_b + first * a.c_t + g * a.c_g;
  T* __restrict__ y = static_cast<T*>(a.y) + b * a.y_b + first * a.y_t + hd * a.y_h + p0;
  const int64_t slot = seq_slot(a.seq, b);
  const float D = a.D != nullptr ? a.D[hd] : 0.f, bias = a.dt_bias != nullptr ? a.dt_bias[hd] : 0.f;
  const double A2 = (double)a.A[hd] * 1.4426950408889634;  // exponents of 2

  // The state: register r of tile nt is row p0 + col, column
  // 32 nt + 8 (r / 4) + 4 half + r % 4.
  f32x16 h[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int r = 0; r < 16; ++r) h[nt][r] = 0.f;
  const int p = p0 + col;
  const bool mine = on && p < P;
  const bool vec_n = N % 4 == 0;
  const int64_t plane = (int64_t)P * N;
  const float* from = nullptr;
  float* to = nullptr;
  if constexpr (STATES) {
    to = sp.parts + ((b * sp.segments + seg) * a.heads + hd) * plane;
  } else {
    from = sp.segments > 1 ? sp.parts + ((b * sp.segments + seg) * a.heads + hd) * plane
           : a.h0 != nullptr && slot >= 0 ? a.h0 + (slot * a.heads + hd) * plane
                                          : nullptr;
    if (seg == sp.segments - 1 && a.h1 != nullptr && slot >= 0) to = a.h1 + (slot * a.heads + hd) * plane;
  }
  if (from != nullptr && mine) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n0 = 32 * nt + 8 * q + 4 * half;
        const float* src = from + (int64_t)p * N + n0;
        if (vec_n && n0 < N) {
          const float4 v = *reinterpret_cast<const float4*>(src);
          h[nt][4 * q] = v.x, h[nt][4 * q + 1] = v.y, h[nt][4 * q + 2] = v.z, h[nt][4 * q + 3] = v.w;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n0 + e < N) h[nt][4 * q + e] = src[e];
        }
      }
  }
  double l_seg = 0.0;

  for (int64_t t = t0; t < t1; t += Q) {
    const int len = (int)(t1 - t < Q ? t1 - t : Q);
    // ---- B, C (all wavefronts) and x, L (this one) into LDS ----
    for (int i = threadIdx.x; i < Q * (NP / U); i += threads) {
      const int j = i / (NP / U), u = i % (NP / U);
      const int left = j < len ? N - u * U : 0;
      stage_unit<T, M>(s_b + j * NP + M::template unit<NP>(j, u) * U, B + (t + j) * a.b_t + u * U, left, vec);
      if constexpr (!STATES)
        stage_unit<T, M>(s_c + j * NP + M::template unit<NP>(j, u) * U, C + (t + j) * a.c_t + u * U, left, vec);
    }
    for (int i = lane; i < Q * (kSlice / U); i += kWave) {
      const int j = i / (kSlice / U), u = i % (kSlice / U);
      stage_unit<T, M>(s_x + j * M::kXStride + u * U, x + (t + j) * a.x_t + u * U, j < len && on ? P - p0 - u * U : 0, vec);
    }
    float decay;  // 2^L_end
    float my_l[IT], my_ll[IT], my_e[IT], my_alpha = 0.f;  // of the tokens col, 32 + col
    {
      float d = 0.f;
      if (lane < len) {
        d = to_f32<T>(dt[(t + lane) * a.dt_t]) + bias;
        if (a.softplus) d = softplus(d);
      }
      double l = lane < len ? A2 * (double)d : 0.0;
#pragma unroll
      for (int off = 1; off < Q; off <<= 1) {
        const double v = __shfl_up(l, off, kWave);
        if (lane >= off) l += v;
      }
      const double end = __shfl(l, Q - 1, kWave);
      decay = exp2f((float)end);
      l_seg += end;
      const float lf = (float)l, lr = (float)(l - (double)lf);
      if (lane < Q) {
        sc.l[lane] = lf;
        if constexpr (M::kPair) sc.ll[lane] = lr;
        sc.d[lane] = d;
        sc.w[lane] = exp2f((float)(end - l)) * d;
      }
      if constexpr (IT == 2 && !STATES) {
        const double mid = __shfl(l, 31, kWave);
        sc.ab[lane] = lane < 32 ? exp2f((float)(mid - l)) * d : exp2f((float)(l - mid));
      }
      if constexpr (!STATES) {
#pragma unroll
        for (int it = 0; it < IT; ++it) {
          my_l[it] = __shfl(lf, 32 * it + col, kWave);
          my_ll[it] = __shfl(lr, 32 * it + col, kWave);
          my_e[it] = exp2f(my_l[it]);
        }
      }
    }
    __syncthreads();
    if constexpr (IT == 2 && !STATES) my_alpha = sc.ab[32 + col];
    Frag xf[KB];
#pragma unroll
    for (int k = 0; k < KB; ++k) xf[k] = M::xcol(s_x, k, lane);

    if constexpr (!STATES) {
      // ---- G = B C^T: lane = token i of C, registers = tokens j of B ----
      for (int tile = wave; tile < Lds::tiles; tile += threads / 64) {
        const int it = tile == 0 ? 0 : 1, jt = tile == 2 ? 1 : 0;  // (0, 0), (1, 0), (1, 1)
        f32x16 acc;
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[r] = 0.f;
#pragma unroll
        for (int k = 0; k < NP / 16; ++k)
          acc = M::mma(M::template row<NP>(s_b, 32 * jt + col, k, half), M::template row<NP>(s_c, 32 * it + col, k, half), acc);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<float4*>(s_g + ((tile * 4 + q) * 64 + lane) * 4) =
              make_float4(acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]);
      }
      // ---- 2^L_i h C_i^T + D x: lane = token i, registers = columns p ----
      f32x16 acc[IT];
#pragma unroll
      for (int it = 0; it < IT; ++it)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[it][r] = 0.f;
#pragma unroll
      for (int k = 0; k < NP / 16; ++k) {
        float hv[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) hv[e] = h[k / 2][8 * (k % 2) + e];
        const Frag hf = M::of(hv);
#pragma unroll
        for (int it = 0; it < IT; ++it) acc[it] = M::mma(hf, M::template row<NP>(s_c, 32 * it + col, k, half), acc[it]);
      }
#pragma unroll
      for (int it = 0; it < IT; ++it)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float xv[4];
          M::four(s_x + (32 * it + col) * M::kXStride + 8 * q + 4 * half, xv);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[it][4 * q + e] = fmaf(acc[it][4 * q + e], my_e[it], D * xv[e]);
        }
      __syncthreads();

      // ---- x^T S: S[i][j] = G[i][j] 2^(L_i - L_j) d_j for j <= i ----
      if (__ballot(!M::finite(xf)) == 0ull) {
#pragma unroll
        for (int it = 0; it < IT; ++it) {
#pragma unroll
          for (int k = 0; k < 2 * (it + 1); ++k) {
            float s[8];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int j0 = 16 * k + 8 * q + 4 * half;
              float gv[4];
              load_f32<float, 4>(s_g + (((it + k / 2) * 4 + 2 * (k % 2) + q) * 64 + lane) * 4, gv);
              if (k / 2 < it) {
                float bv[4];
                load_f32<float, 4>(sc.ab + j0, bv);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[4 * q + e] = gv[e] * (my_alpha * bv[e]);
              } else {
                float lv[4], dv[4], rv[4] = {0.f, 0.f, 0.f, 0.f};
                load_f32<float, 4>(sc.l + j0, lv);
                load_f32<float, 4>(sc.d + j0, dv);
                if constexpr (M::kPair) load_f32<float, 4>(sc.ll + j0, rv);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  float delta = my_l[it] - lv[e];
                  if constexpr (M::kPair) delta += my_ll[it] - rv[e];
                  const float v = gv[e] * (exp2f(delta) * dv[e]);
                  s[4 * q + e] = j0 + e <= 32 * it + col ? v : 0.f;
                }
              }
            }
            acc[it] = M::mma(xf[k], M::of(s), acc[it]);
          }
        }
      } else {
        // An x that is not finite must not meet the zeros of S: its terms one by one.
#pragma unroll
        for (int it = 0; it < IT; ++it) {
          for (int j = 0; j < 32 * (it + 1); ++j) {
            const int tile = it + j / 32, jj = j % 32;
            const float gv = s_g[((tile * 4 + jj / 8) * 64 + col + 32 * ((jj / 4) % 2)) * 4 + jj % 4];
            float delta = my_l[it] - sc.l[j];
            if constexpr (M::kPair) delta += my_ll[it] - sc.ll[j];
            const float s = gv * (exp2f(delta) * sc.d[j]);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              float xv[4];
              M::four(s_x + j * M::kXStride + 8 * q + 4 * half, xv);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                acc[it][4 * q + e] = j <= 32 * it + col ? fmaf(s, xv[e], acc[it][4 * q + e]) : acc[it][4 * q + e];
            }
          }
        }
      }
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        if (!on || 32 * it + col >= len) continue;
        T* row = y + (t + 32 * it + col) * a.y_t;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = 8 * q + 4 * half;
          const float v[4] = {acc[it][4 * q], acc[it][4 * q + 1], acc[it][4 * q + 2], acc[it][4 * q + 3]};
          if (vec && p0 + c + 4 <= P) {
            store_f32<T, 4>(row + c, v);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (p0 + c + e < P) row[c + e] = from_f32<T>(v[e]);
          }
        }
      }
    }

    // ---- h <- 2^L_end h + B^T v ----
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 16; ++r) h[nt][r] *= decay;
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      float v[8];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const float4 wq = *reinterpret_cast<const float4*>(sc.w + 16 * k + 8 * q + 4 * half);
        const float wv[4] = {wq.x, wq.y, wq.z, wq.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * q + e] = M::get(xf[k], 4 * q + e) * wv[e];
      }
      Frag vf[M::kPlanes];
      M::split(v, vf);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const Frag bt = M::template col<NP>(s_b, 32 * nt, k, lane);
#pragma unroll
        for (int pl = 0; pl < M::kPlanes; ++pl) h[nt] = M::mma(bt, vf[pl], h[nt]);
      }
    }
    __syncthreads();
  }

  if (to != nullptr && mine) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n0 = 32 * nt + 8 * q + 4 * half;
        float* dst = to + (int64_t)p * N + n0;
        if (vec_n && n0 < N) {
          *reinterpret_cast<float4*>(dst) =
              make_float4(h[nt][4 * q], h[nt][4 * q + 1], h[nt][4 * q + 2], h[nt][4 * q + 3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n0 + e < N) dst[e] = h[nt][4 * q + e];
        }
      }
  }
  if (STATES && on && p0 == 0 && lane == 0) sp.sums[(b * sp.segments + seg) * a.heads + hd] = (float)l_seg;
}

// Segment by segment, the state that each starts from in place of the part that
// the first pass left there.
constexpr int kChainThreads = 256;
__global__ __launch_bounds__(kChainThreads) void k_scan_chain(ScanArgs a, ScanSplit sp, int blocks) {
  int64_t item = a.block0 + blockIdx.x;
  const int part = (int)(item % blocks);
  item /= blocks;
  const int hd = (int)(item % a.heads);
  const int64_t b = item / a.heads;
  const int64_t plane = (int64_t)a.head_dim * a.state_dim;
  const int64_t e = (int64_t)part * kChainThreads + threadIdx.x;
  if (e >= plane) return;
  const int64_t slot = seq_slot(a.seq, b);
  float h = a.h0 != nullptr && slot >= 0 ? a.h0[(slot * a.heads + hd) * plane + e] : 0.f;
  for (int s = 0; s < sp.segments; ++s) {
    float* at = sp.parts + ((b * sp.segments + s) * a.heads + hd) * plane + e;
    const float own = s + 1 < sp.segments ? *at : 0.f;
    *at = h;
    if (s + 1 < sp.segments) h = fmaf(h, exp2f(sp.sums[(b * sp.segments + s) * a.heads + hd]), own);
  }
}

template <typename T, typename M, int NP, bool STATES>
int launch_chunk_k(const ScanArgs& a, const ScanSplit& sp, int waves, hipStream_t stream) {
  typedef ChunkLds<M, NP> Lds;
  const int rc = set_lds_limit_once<k_scan_chunk<T, M, NP, STATES>>(kMaxLdsBytes);
  if (rc != (int)hipSuccess) return rc;
  constexpr int U = M::kUnit;
  // kUnit elements of a row at a time (y: four).
  const int64_t strides = a.x_b | a.x_t | a.x_h | a.b_b | a.b_t | a.b_g | a.c_b | a.c_t | a.c_g | a.y_b | a.y_t | a.y_h;
  const bool vec = strides % U == 0 && aligned_to(a.x, U * sizeof(T)) && aligned_to(a.b, U * sizeof(T)) &&
                   aligned_to(a.c, U * sizeof(T)) && aligned_to(a.y, 4 * sizeof(T));
  const int64_t blocks = a.seq.batch * (STATES ? sp.segments - 1 : sp.segments) * a.groups * sp.blocks;
  return launch_blocks(a, &ScanArgs::block0, blocks, [&](const ScanArgs& la, unsigned n) {
    hipLaunchKernelGGL((k_scan_chunk<T, M, NP, STATES>), dim3(n), dim3(64 * waves), Lds::bytes(waves, STATES), stream, la,
                       sp, vec);
  });
}

template <typename T, typename M, int NP>
int launch_chunk_n(const ScanArgs& a, const ScanSplit& sp, int waves, hipStream_t stream) {
  if (sp.segments > 1) {
    timing_begin(K_SCAN_PARTS, stream);
    int rc = launch_chunk_k<T, M, NP, true>(a, sp, waves, stream);
    if (rc == (int)hipSuccess) {
      const int64_t plane = (int64_t)a.head_dim * a.state_dim;
      const int64_t blocks = (plane + kChainThreads - 1) / kChainThreads;
      rc = launch_blocks(a, &ScanArgs::block0, a.seq.batch * a.heads * blocks, [&](const ScanArgs& la, unsigned n) {
        hipLaunchKernelGGL(k_scan_chain, dim3(n), dim3(kChainThreads), 0, stream, la, sp, (int)blocks);
      });
    }
    timing_end(K_SCAN_PARTS, stream);
    if (rc != (int)hipSuccess) return rc;
  }
  timing_begin(K_SCAN_CHUNK, stream);
  const int rc = launch_chunk_k<T, M, NP, false>(a, sp, waves, stream);
  timing_end(K_SCAN_CHUNK, stream);
  return rc;
}

template <typename T, typename M>
int launch_chunk_m(const ScanArgs& a, const ScanSplit& sp, int waves, hipStream_t stream) {
  if (a.state_dim <= 32) return launch_chunk_n<T, M, 32>(a, sp, waves, stream);
  if (a.state_dim <= 64) return launch_chunk_n<T, M, 64>(a, sp, waves, stream);
  if (a.state_dim <= 128) return launch_chunk_n<T, M, 128>(a, sp, waves, stream);
  return launch_chunk_n<T, M, 256>(a, sp, waves, stream);
}

size_t align16(size_t v) { return (v + 15) / 16 * 16; }

}  // namespace

ScanPlan scan_plan(int64_t batch, int64_t max_len, int heads, int head_dim, int groups, int state_dim, int dtype) {
  ScanPlan p{};
  // Fewer tokens than half a chunk: the walk token by token.
  p.chunked = max_len >= kScanChunkFrom;
  if (!p.chunked || batch < 1) return p;
  const int q = dtype == SF_BF16 ? MathBf16::Q : MathF32::Q;
  const int units = heads / groups * ((head_dim + kSlice - 1) / kSlice);
  p.waves = units >= 3 ? 4 : units;
  p.split.blocks = (units + p.waves - 1) / p.waves;
  // Segments: enough workgroups for two on a CU, with at least four chunks each.
  const int64_t chunks = (max_len + q - 1) / q;
  const int64_t base = batch * groups * p.split.blocks;
  int64_t segs = (2 * (int64_t)num_cus() + base - 1) / base;
  if (segs > chunks / 4) segs = chunks / 4;
  if (segs < 1) segs = 1;
  const int64_t per = (chunks + segs - 1) / segs;
  p.split.chunks = (int)per;
  p.split.segments = (int)((chunks + per - 1) / per);
  if (p.split.segments > 1) {
    const size_t rows = (size_t)batch * p.split.segments * heads;
    p.sums_at = align16(rows * head_dim * state_dim * sizeof(float));
    p.bytes = p.sums_at + align16(rows * sizeof(float));
  }
  return p;
}

int launch_scan_chunk(const ScanArgs& a, const ScanPlan& p, void* workspace, int dtype, hipStream_t stream) {
  ScanSplit sp = p.split;
  sp.parts = static_cast<float*>(workspace);
  sp.sums = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.sums_at);
  if (dtype == SF_BF16) return launch_chunk_m<__hip_bfloat16, MathBf16>(a, sp, p.waves, stream);
  if (dtype == SF_F16) return launch_chunk_m<__half, MathF32>(a, sp, p.waves, stream);
  return launch_chunk_m<float, MathF32>(a, sp, p.waves, stream);
}

}  // namespace sf
