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
// All of it runs on the bf16 instructions, whatever the inputs: x, B and C are taken
// apart into bf16 parts (bf16 one, f16 two, float32 three: all of their bits), S and h
// into two, two and three, and a product of two sums of parts leaves out the terms below
// the last part (two products for bf16, three for f16 and six for float32, a sixth of
// the time that the float32 instructions take).  So S and h are rounded to 16 bits for
// bf16 and f16 outputs, which have 8 and 11 themselves: what y loses is its own rounding
// (as one part for bf16, y was off by more than that where its terms cancel; 2 x 16384
// tokens took 390 us with one and take 445).  v is split into three parts, its 24 bits,
// always: the state is summed up over all tokens and stays a float32 one.  L is summed
// in 64 bits: differences of it are exponents.
//
// Bound by the chain of products and the waits between them, not by memory: 2 x 16384
// tokens, 64 heads x 64, N 128, bf16 (562 MB, 290 GFLOP of products) take 445 us, 650
// TFLOP/s and 1.3 TB/s; alone, the main pass 365 us, the segments' own parts 162, the
// chain 16; rows at any address, by way of registers, as long; 23 ragged sequences of up
// to 1500 of f16, 24 heads, 199 us.
//
// Where products are not finite, a wavefront does its segment again, token by token:
// infinities, NaN and results near the ends of a float's range are those of the
// recurrence.
//
// Few heads and long sequences: the token axis is cut into segments.  A first
// pass walks each segment from a zero state for its own part of the state
// (the last product alone), a second one chains the parts, and the main pass
// starts each segment from its true state.  Of such a sequence the main pass does not
// read the states that the call began with: it writes the final ones, maybe to the same
// rows, and its workgroups are in no order.
#include "sf_seq.h"
#include "sf_tile.h"

#include <type_traits>

namespace sf {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kChunk = 32;  // tokens
constexpr int kSlice = 32;  // columns of x of a wavefront
constexpr int kWaves = 4;   // of a workgroup
constexpr int kThreads = kWaves * kWave;

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const f32x2 v = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}
__device__ __forceinline__ float low_bf16(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float high_bf16(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// ---- fragments ------------------------------------------------------------------
// A fragment is a lane's 8 values of a 16-deep slice of an operand, as bf16: depths
// 8 half to 8 half + 7, half = lane / 32.  A product leaves rows 8 q + 4 half + e in
// register 4 q + e; with its rows of 4 in the order 0, 2, 1, 3 of each 16 (order4),
// registers 8 k to 8 k + 7 are a fragment.
typedef u32x4 Frag;  // pairs of bf16
__device__ __forceinline__ int order4(int b) { return (b >> 1) | ((b & 1) << 1); }

// Place of 16-byte unit u (8 elements) in token j's row of a tile [32][NP]: spread over
// the banks, for a read of one unit of 16 rows and a transposed one of two units of 4
// rows.  (A third of the LDS's cycles are bank conflicts all the same, counted over the
// main pass of 2 x 16384 tokens: G's reads, 16 bytes every 32, meet theirs twice.)
template <int NP>
constexpr __device__ __forceinline__ int unit_place(int j, int u) {
  if constexpr (NP >= 128) return u ^ ((2 * (j & 7)) | ((j >> 3) & 1));
  else if constexpr (NP == 64) return u ^ ((2 * ((j >> 1) & 3)) | ((j >> 3) & 1));
  else return u ^ ((2 * ((j >> 2) & 1)) | ((j >> 3) & 1));
}

// Tokens as lanes: token j's row, depths from 16 k (place: where its first ones are;
// the others differ in single bits of it).
template <int NP>
__device__ __forceinline__ int row_place(int j, int half) {
  return j * NP + unit_place<NP>(j, half) * 8;
}
__device__ __forceinline__ Frag row_frag(const uint16_t* m, int place, int k) {
  return *reinterpret_cast<const Frag*>(m + (place ^ (16 * k)));
}

// Tokens as depth: columns in the order of order4, tokens from 16 k.  Four lanes
// point at a token's 16 columns, and lane l of each 16 gets column l of the four
// tokens.
__device__ __forceinline__ Frag join(bf16x4 lo, bf16x4 hi) {
  return __builtin_bit_cast(Frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}
__device__ __forceinline__ bf16x4 transposed(const uint16_t* p) {
  typedef __attribute__((address_space(3))) bf16x4 Lds;
  return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((Lds*)(const_cast<uint16_t*>(p)));
}
template <int NP>
__device__ __forceinline__ int col_place(int lane) {
  const int half = lane >> 5, s = lane & 15, n = (lane & 16) + 4 * order4(s & 3), j = 8 * half + (s >> 2);
  return j * NP + unit_place<NP>(j, n >> 3) * 8 + (n & 7);
}
// (Four tokens on: only the bits of j & 4 differ.)
template <int NP>
__device__ __forceinline__ Frag col_frag(const uint16_t* m, int place, int nt, int k) {
  constexpr int next = unit_place<NP>(4, 0) * 8;
  return join(transposed(m + (place ^ (32 * nt)) + 16 * k * NP),
              transposed(m + (place ^ (32 * nt) ^ next) + (16 * k + 4) * NP));
}
// The same of a slice of x, rows of 64 bytes, its columns in their own order: 4 rows
// are read at once transposed, 16 as rows.
__device__ __forceinline__ int x_place(int j, int c) {
  return j * kSlice + ((c >> 3) ^ ((j >> 2) & 3)) * 8 + (c & 7);
}
__device__ __forceinline__ Frag x_frag(const uint16_t* x, int k, int lane) {
  const int half = lane >> 5, s = lane & 15, n = (lane & 16) + 4 * (s & 3);
  const int j = 16 * k + 8 * half + (s >> 2);
  return join(transposed(x + x_place(j, n)), transposed(x + x_place(j + 4, n)));
}

__device__ __forceinline__ float get(const Frag& f, int e) {
  return e % 2 == 0 ? low_bf16(f[e / 2]) : high_bf16(f[e / 2]);
}

// v as a sum of PL bf16 values: PL = 3 are all of its 24 bits.
template <int PL>
__device__ __forceinline__ void split(const float (&v)[8], Frag (&f)[PL]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
    for (int p = 0; p < PL; ++p) {
      const uint32_t w = pack_bf16(a, b);
      f[p][i] = w;
      a -= low_bf16(w);
      b -= high_bf16(w);
    }
  }
}

// z (0 or NaN), or NaN if any of v is not finite.
__device__ __forceinline__ float not_finite(const f32x16& v, float z) {
#pragma unroll
  for (int r = 0; r < 16; ++r) z = fmaf(v[r], 0.f, z);
  return z;
}

__device__ __forceinline__ f32x16 mma(const Frag& a, const Frag& b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(const Frag& a, const Frag& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// The product of two sums of parts, without the terms below the last part's (P
// parts of a value have its last bits at 2^-8 P of it).
template <int PA, int PB>
__device__ __forceinline__ f32x16 mma_parts(const Frag (&a)[PA], const Frag (&b)[PB], f32x16 c) {
#pragma unroll
  for (int i = 0; i < PA; ++i)
#pragma unroll
    for (int j = 0; j < PB; ++j)
      if (i + j < (PA > PB ? PA : PB)) c = mma(a[i], b[j], c);
  return c;
}

// Per token of a chunk, for one head.  The state in the accumulators is 2^-K h, K
// between 0 and kScaleMost (the range that it costs is at the small end), so that a
// chunk's decay need not be multiplied in each time; K' is its value after the chunk.
// (K is taken back by whole numbers, so that the state is multiplied by powers of two.)
//            factors apart      a factor per element (wide)
//   w        2^(L_end - L - K') d, both
//   p        2^(L + K)          L + K
//   q        2^(-L - K) d       d
//   r                           what L + K loses as one float
struct alignas(16) ChunkScalars {
  float w[kChunk], p[kChunk], q[kChunk], r[kChunk];
};
constexpr double kScaleMost = 20.0, kScaleFrom = 16.0;  // (a chunk that decays nothing leaves K alone)
constexpr float kApartMost = 100.f;  // exponents of factors apart

// 2^v of an exponent of more than a float's bits: as one float it would be rounded to
// 2^-20 of itself from 16 on.
__device__ __forceinline__ float exp2_of(double v) {
  const double whole = floor(v);
  return v < -200.0 ? 0.f : __builtin_amdgcn_ldexpf(exp2_hw((float)(v - whole)), (int)fmin(whole, 200.0));
}

// The sum of v over this half wavefront's lanes up to this one.
__device__ __forceinline__ double half_sum_up_to(double v) {
  auto step = [&](auto ctrl, auto rows) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    v += __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
  };
  typedef std::integral_constant<int, 0xf> All;
  step(std::integral_constant<int, 0x111>(), All());  // within rows of 16: from 1, 2, 4 and 8 lanes below
  step(std::integral_constant<int, 0x112>(), All());
  step(std::integral_constant<int, 0x114>(), All());
  step(std::integral_constant<int, 0x118>(), All());
  step(std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xa>());  // lane 15 to row 1, 47 to row 3
  return v;
}

// A value that is the same in all lanes, held once for them.
__device__ __forceinline__ float uniform(float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); }
__device__ __forceinline__ double uniform(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)u), hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(u >> 32));
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

__device__ __forceinline__ double lane_of(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

template <int PL, int NP>
struct ChunkLds {
  static constexpr int tile = PL * kChunk * NP * 2;
  static constexpr int x_bytes = PL * kChunk * kSlice * 2;
  // B, and a slice of x for each wavefront, for this chunk and `depth - 1` after it
  // that are on their way; the scalars of two chunks for each wavefront; C, G.
  static constexpr int x(int depth) { return depth * tile; }
  static constexpr int scalars(int depth) { return x(depth) + depth * kWaves * x_bytes; }
  static constexpr int c(int depth) { return scalars(depth) + 2 * kWaves * (int)sizeof(ChunkScalars); }
  static constexpr int g(int depth) { return c(depth) + tile; }
  static constexpr int bytes(int depth, bool states) { return states ? c(depth) : g(depth) + kChunk * kChunk * 4; }
};

// Chunks in LDS at a time: by way of registers one; straight into LDS two, or three
// where as many workgroups fit a CU with them.
template <int NP, bool DIRECT, bool STATES>
constexpr int chunk_depth() {
  return !DIRECT ? 1 : STATES && NP <= 128 ? 3 : 2;
}

// 64 lanes' 16 bytes from base + off (bytes) to LDS at dst and on, lane by lane
// (lanes that are off leave theirs as it was).  In asm because the compiler would
// wait for the builtin's loads before the next LDS read of any kind: the caller
// waits (lds_dma_wait) before the barrier that hands the data over.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 in the clobber list
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t off, const void* dst) {
  const uint32_t l = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_ptr_t)dst);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(l) : "m0", "memory");
}
#pragma clang diagnostic pop

// Waits until at most KEEP of this wavefront's latest memory operations are not
// done (they are done in their order).
template <int KEEP>
__device__ __forceinline__ void wait_memory() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(KEEP) : "memory");
}

// 8 elements of a row on their way to LDS; what lies outside becomes 0.
template <typename T>
__device__ __forceinline__ void load_unit(const T* __restrict__ from, int left, uint32_t (&v)[2 * sizeof(T)]) {
#pragma unroll
  for (int i = 0; i < (int)(2 * sizeof(T)); ++i) v[i] = 0u;
  if (left >= 8) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      const AnyX4 q = reinterpret_cast<const AnyX4*>(from)[i];
      v[4 * i] = q[0], v[4 * i + 1] = q[1], v[4 * i + 2] = q[2], v[4 * i + 3] = q[3];
    }
  } else if constexpr (sizeof(T) == 2) {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(from);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) v[e / 2] |= (uint32_t)p[e] << (16 * (e % 2));
  } else {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(from);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) v[e] = p[e];
  }
}

// ... and into LDS as PL parts, `apart` elements from one to the next.
template <typename T, int PL>
__device__ __forceinline__ void store_unit(uint16_t* to, int apart, const uint32_t (&v)[2 * sizeof(T)]) {
  if constexpr (std::is_same<T, __hip_bfloat16>::value) {
    *reinterpret_cast<uint4*>(to) = make_uint4(v[0], v[1], v[2], v[3]);
  } else {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (sizeof(T) == 4) f[e] = __uint_as_float(v[e]);
      else f[e] = __half2float(__ushort_as_half((unsigned short)(v[e / 2] >> (16 * (e % 2)))));
    }
    Frag p[PL];
    split(f, p);
#pragma unroll
    for (int i = 0; i < PL; ++i) *reinterpret_cast<Frag*>(to + i * apart) = p[i];
  }
}

// The last segment of a sequence of n tokens: it takes the tokens beyond the longest
// sequence that the call was cut for, too.
__device__ __forceinline__ int last_segment(const ScanSplit& sp, int64_t n) {
  const int64_t s = (n + (int64_t)sp.chunks * kChunk - 1) / ((int64_t)sp.chunks * kChunk) - 1;
  return (int)(s < 0 ? 0 : s >= sp.segments ? sp.segments - 1 : s);
}

// The workspace's row of the first segment of a cut sequence whose tokens begin at
// `first`.  By tokens: it has more than a segment's tokens, n > s, so that the next cut
// one begins floor(n / s) >= 1 segments on or later, and 2 floor(n / s) >= ceil(n / s)
// rows are its own.  (A packed call of one long sequence and many short ones has many
// segments times many sequences, hardly any of which are cut: of 16384 tokens and 255
// times 16, 64 heads x 64, N 128, 6.4 GB by their numbers, 63 MB by tokens.)
__device__ __forceinline__ int64_t first_row(const ScanSplit& sp, int64_t b, int64_t first) {
  return sp.by_tokens ? first / ((int64_t)sp.chunks * kChunk) * 2 : b * sp.segments;
}

// A workgroup's sequence, segment (tokens t0 to t1 of the sequence) and group; a
// wavefront's head and columns.
struct ChunkWork {
  int64_t b, first, t0, t1, slot, row0;  // (row0: first_row)
  int g, seg, last, hd, p0;
  bool on, idle;  // whether the wavefront has columns; whether there is no such segment
};
template <bool STATES>
__device__ __forceinline__ ChunkWork chunk_work(const ScanArgs& a, const ScanSplit& sp, int64_t item, int wave) {
  ChunkWork w;
  const int segs = STATES ? sp.segments - 1 : sp.segments;
  const int ub = (int)(item % sp.blocks);
  item /= sp.blocks;
  w.g = (int)(item % a.groups);
  item /= a.groups;
  w.seg = (int)(item % segs);
  w.b = item / segs;
  int64_t n;
  seq_rows(a.seq, w.b, w.first, n);
  w.last = last_segment(sp, n);
  w.idle = STATES ? w.seg >= w.last : w.seg > w.last;
  const int per_group = a.heads / a.groups, slices = (a.head_dim + kSlice - 1) / kSlice;
  const int unit = ub * kWaves + wave;
  w.on = unit < per_group * slices;
  w.hd = w.g * per_group + (w.on ? unit / slices : 0);
  w.p0 = w.on ? unit % slices * kSlice : 0;
  const int64_t per_seg = (int64_t)sp.chunks * kChunk;
  w.t0 = w.seg * per_seg;
  w.t1 = w.seg == w.last ? n : w.t0 + per_seg;
  w.slot = seq_slot(a.seq, w.b);
  w.row0 = first_row(sp, w.b, w.first);
  return w;
}

// STATES: a segment's own part of the state, from a zero state, to `parts`, with
// the sum of its exponents to `sums`.  Otherwise y, from the segment's true state.
// PL: bf16 parts of an element of x, B and C.  DIRECT: rows of whole aligned units,
// which go straight into LDS.
template <typename T, int PL, int NP, bool DIRECT, bool STATES>
__global__ __launch_bounds__(kThreads, NP == 256 ? 1 : PL > 1 || (NP == 128 && !STATES) ? 2 : 3) void k_scan_chunk(ScanArgs a, ScanSplit sp) {
  constexpr int Q = kChunk, KB = Q / 16, NT = NP / 32, U = 8;
  constexpr int kRowUnits = NP / U, kRows = kThreads / kRowUnits;  // of B and C at a time
  constexpr int kRounds = Q > kRows ? Q / kRows : 1;
  constexpr int kXUnits = kSlice / U, kXRows = kWave / kXUnits, kXRounds = Q / kXRows;
  constexpr int kDepth = chunk_depth<NP, DIRECT, STATES>();
  constexpr int kTile = Q * NP, kX = Q * kSlice;  // elements of a part
  constexpr bool kPair = PL == 3;                 // exponents to more than a float's bits
  constexpr int SP = PL > 2 ? PL : 2;             // parts of S and h
  constexpr bool kTight = PL == 1 && NP == 128 && !STATES;  // registers for three workgroups a CU, and none to spare
  typedef ChunkLds<PL, NP> Lds;
  extern __shared__ __align__(16) char lds[];
  const int lane = lane_id(), half = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint16_t* const s_b0 = reinterpret_cast<uint16_t*>(lds);
  uint16_t* const s_x0 = reinterpret_cast<uint16_t*>(lds + Lds::x(kDepth) + wave * kDepth * Lds::x_bytes);
  ChunkScalars* s_sc = reinterpret_cast<ChunkScalars*>(lds + Lds::scalars(kDepth)) + 2 * wave;
  uint16_t* s_c = reinterpret_cast<uint16_t*>(lds + Lds::c(kDepth));
  float* const s_g = reinterpret_cast<float*>(lds + Lds::g(kDepth));

  // (In the order of the launch: given to the XCDs so that those of one sequence and
  // group share an L2 for B and C, ragged calls take up to a third longer.)
  const ChunkWork work = chunk_work<STATES>(a, sp, a.block0 + blockIdx.x, wave);
  if (work.idle) return;
  const int64_t b = work.b, first = work.first, t0 = work.t0, t1 = work.t1;
  const int g = work.g, hd = work.hd, p0 = work.p0, P = a.head_dim, N = a.state_dim;
  const bool on = work.on;
  // (The launcher takes token strides below 2^24 only.)
  const int x_t = (int)a.x_t, dt_t = (int)a.dt_t, b_t = (int)a.b_t, c_t = (int)a.c_t, y_t = (int)a.y_t;
  const T* __restrict__ x = static_cast<const T*>(a.x) + b * a.x_b + (first + t0) * a.x_t + hd * a.x_h + p0;
  const T* __restrict__ B = static_cast<const T*>(a.b) + b * a.b_b + (first + t0) * a.b_t + g * a.b_g;
  const T* __restrict__ C = static_cast<const T*>(a.c) + b * a.c_b + (first + t0) * a.c_t + g * a.c_g;
  T* __restrict__ y = static_cast<T*>(a.y) + b * a.y_b + (first + t0) * a.y_t + hd * a.y_h + p0;
  const float D = uniform(a.D != nullptr ? a.D[hd] : 0.f);

  // The scalars of two chunks at once, one to each half wavefront.
  const T* __restrict__ dt = static_cast<const T*>(a.dt) + b * a.dt_b + (first + t0) * a.dt_t + hd * a.dt_h;
  const float bias = uniform(a.dt_bias != nullptr ? a.dt_bias[hd] : 0.f);
  const double A2 = uniform((double)a.A[hd] * 1.4426950408889634);  // exponents of 2
  double k_state = 0.0, l_seg = 0.0;  // (l_seg: the sum of the exponents)
  // Of each of the two: what the state is multiplied by before the chunk's part comes in;
  // whether the factors are an element's.
  float rescale_of[2];
  bool wide_of[2];
  T next_dt = from_f32<T>(0.f);
  // rest: tokens from the first of the two chunks on.
  auto load_dt = [&](const T* from, int64_t rest) {
    if (lane < rest) next_dt = from[lane * dt_t];
  };
  auto write_scalars = [&](int64_t rest) {
    float d = 0.f;
    if (lane < rest) {
      d = to_f32<T>(next_dt) + bias;
      if (a.softplus) d = softplus(d);
    }
    const double l = half_sum_up_to(lane < rest ? A2 * (double)d : 0.0);
    const double end[2] = {lane_of(l, 31), lane_of(l, 63)};
    double k[3] = {k_state, 0.0, 0.0};
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      rescale_of[c] = 1.f;
      k[c + 1] = k[c] + end[c];
      if constexpr (STATES) l_seg = uniform(l_seg + end[c]);
      if (!(k[c + 1] >= 0.0 && k[c + 1] < kScaleMost)) {
        const double to = end[c] < 0.0 ? kScaleFrom : 0.0, by = floor(k[c + 1] - to);
        rescale_of[c] = uniform(exp2_of(by));
        k[c + 1] = fabs(by) < 1e6 ? k[c + 1] - by : to;
      }
    }
    k_state = uniform(k[2]);
    ChunkScalars& sc = s_sc[half];
    sc.w[col] = exp2_of((half == 0 ? end[0] - k[1] : end[1] - k[2]) - l) * d;
    if constexpr (!STATES) {
      const double lk = l + (half == 0 ? k[0] : k[1]);
      float p = (float)lk, q = d;
      sc.r[col] = (float)(lk - (double)p);
      if constexpr (kPair) {
        wide_of[0] = wide_of[1] = true;
      } else {
        const float off = p, fall = exp2_hw(-off) * d;
        // (Also where a factor of a later token is no number: it meets zeros of G.)
        const uint64_t no = __ballot(!(fabsf(off) < kApartMost && fabsf(fall) < __builtin_huge_valf()));
        wide_of[0] = (uint32_t)no != 0u;
        wide_of[1] = (uint32_t)(no >> 32) != 0u;
        if (half == 0 ? !wide_of[0] : !wide_of[1]) {
          p = exp2_hw(off);
          q = fall;
        }
      }
      sc.p[col] = p;
      sc.q[col] = q;
    }
  };

  // The state: register r of tile nt is row p0 + col, column
  // 32 nt + 16 (r / 8) + 8 half + r % 8.
  f32x16 h[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int r = 0; r < 16; ++r) h[nt][r] = 0.f;
  const int p = p0 + col;
  const bool mine = on && p < P;
  const bool vec_n = N % 4 == 0;
  const int64_t plane = (int64_t)P * N;
  // The state that a segment starts from.  (Of a sequence that is cut, segment 0's is the
  // chain's copy too: the last segment may write the pool's row before segment 0 would
  // have read it.)
  auto start_of = [&](const ChunkWork& w, const ScanArgs& args, const ScanSplit& split) -> const float* {
    const bool kept = args.h0 != nullptr && w.slot >= 0;
    return w.seg > 0 || (kept && w.last > 0) ? split.parts + ((w.row0 + w.seg) * args.heads + w.hd) * plane
           : kept                            ? args.h0 + (w.slot * args.heads + w.hd) * plane
                                             : nullptr;
  };
  const float* const from = STATES ? nullptr : start_of(work, a, sp);
  if (from != nullptr && mine) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n0 = 32 * nt + 16 * (q / 2) + 8 * half + 4 * (q % 2);
        const float* src = from + (int64_t)p * N + n0;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (vec_n) {
          if (n0 < N) load_any_f32<float, 4>(src, v);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n0 + e < N) v[e] = src[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) h[nt][4 * q + e] = v[e];
      }
  }

  // (Opaque where registers are tight, so that what the last chunk, by way of registers,
  // makes of it is not kept in them.)
  auto thread = []() {
    int t = threadIdx.x;
    if constexpr (kTight) asm volatile("" : "+v"(t));
    return t;
  };
  const bool whole_n = N == NP, whole_p = p0 + kSlice <= P;
  // DIRECT: a whole chunk goes from memory to LDS while chunks before it are worked on:
  // B and x to a buffer of their own, C once its readers are done.  (The last chunk, if
  // it is not whole, is staged by way of registers when its turn comes.)
  auto ahead = [&](int64_t rest) { return DIRECT && rest >= Q; };
  auto load_rows = [&](const T* base, int stride, uint16_t* to) {
    const char* from = reinterpret_cast<const char*>(base);
    const int bj = threadIdx.x / kRowUnits, bv = threadIdx.x % kRowUnits;
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int u = unit_place<NP>(r * kRows + bj, bv);
      const uint32_t off = (uint32_t)(bj * stride + u * U) * (uint32_t)sizeof(T);
      uint16_t* dst = to + (r * kThreads + wave * kWave) * U;
      if (kRows <= Q && whole_n) load_to_lds(from, off, dst);
      else if (u * U < N && bj < Q) load_to_lds(from, off, dst);
      from += (uint32_t)(kRows * stride) * (uint32_t)sizeof(T);
    }
  };
  auto load_x = [&](uint16_t* to) {
    if (!on) return;
    const char* from = reinterpret_cast<const char*>(x);
    const int xj = threadIdx.x % kWave / kXUnits, xv = threadIdx.x % kXUnits;
#pragma unroll
    for (int r = 0; r < kXRounds; ++r) {
      const int u = x_place(r * kXRows + xj, xv * U) % kSlice / U;
      const uint32_t off = (uint32_t)(xj * x_t + u * U) * (uint32_t)sizeof(T);
      if (whole_p) load_to_lds(from, off, to + r * kWave * U);
      else if (p0 + u * U < P) load_to_lds(from, off, to + r * kWave * U);
      from += (uint32_t)(kXRows * x_t) * (uint32_t)sizeof(T);
    }
  };
  // By way of registers: the next chunk's B, C and x wait in them.
  constexpr int kWords = 2 * (int)sizeof(T);
  uint32_t nb[kRounds][kWords], nc[STATES ? 1 : kRounds][kWords], nx[kXRounds][kWords];
  auto fetch = [&](const T* b_from, const T* c_from, const T* x_from, int len) {
    const int bj = thread() / kRowUnits, bv = thread() % kRowUnits, xj = thread() % kWave / kXUnits, xv = thread() % kXUnits;
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int j = r * kRows + bj;
      load_unit<T>(b_from + ((int64_t)(r * kRows) * b_t + (bj * b_t + bv * U)), j < len ? N - bv * U : 0, nb[r]);
      if constexpr (!STATES)
        load_unit<T>(c_from + ((int64_t)(r * kRows) * c_t + (bj * c_t + bv * U)), j < len ? N - bv * U : 0, nc[r]);
    }
#pragma unroll
    for (int r = 0; r < kXRounds; ++r)
      load_unit<T>(x_from + ((int64_t)(r * kXRows) * x_t + (xj * x_t + xv * U)),
                   on && r * kXRows + xj < len ? P - p0 - xv * U : 0, nx[r]);
  };
  auto unload = [&](uint16_t* to_b, uint16_t* to_x) {
    const int bj = thread() / kRowUnits, bv = thread() % kRowUnits, xj = thread() % kWave / kXUnits, xv = thread() % kXUnits;
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int j = r * kRows + bj;
      if (kRows > Q && j >= Q) break;
      const int at = j * NP + unit_place<NP>(j, bv) * U;
      store_unit<T, PL>(to_b + at, kTile, nb[r]);
      if constexpr (!STATES) store_unit<T, PL>(s_c + at, kTile, nc[r]);
    }
#pragma unroll
    for (int r = 0; r < kXRounds; ++r) store_unit<T, PL>(to_x + x_place(r * kXRows + xj, xv * U), kX, nx[r]);
  };
  int64_t left = t1 - t0;  // tokens from this chunk on
  for (int i = threadIdx.x * 4; i < Lds::bytes(kDepth, STATES) / 4; i += kThreads * 4)
    store_f32<float, 4>(reinterpret_cast<float*>(lds) + i, {0.f, 0.f, 0.f, 0.f});
  __syncthreads();
  if constexpr (DIRECT) {
#pragma unroll
    for (int c = 0; c < kDepth - 1; ++c) {
      if (ahead(left - c * Q)) {
        load_rows(B, b_t, s_b0 + c * kTile);
        if (c == 0 && !STATES) load_rows(C, c_t, s_c);
        load_x(s_x0 + c * kX);
      }
      B += (int64_t)Q * b_t;
      x += (int64_t)Q * x_t;
    }
  } else if (left > 0) {
    fetch(B, C, x, (int)(left < Q ? left : Q));
  }
  load_dt(dt, left);
  write_scalars(left);
  // Every wavefront issues as many memory operations to a chunk as any: the latest
  // may be left under way at the next.
  const bool counted = DIRECT && on && whole_n && whole_p && kRows <= Q;

  float bad = 0.f;  // not 0 (NaN) where products have not been finite
  for (int i = 0; left > 0; left -= Q, ++i) {
    const int len = (int)(left < Q ? left : Q);
    const int at = i % kDepth, at_last = (i + kDepth - 1) % kDepth;
    const uint16_t* s_b = s_b0 + at * PL * kTile;
    const uint16_t* s_x = s_x0 + at * PL * kX;
    if constexpr (DIRECT) {
      if (!ahead(left)) {
        fetch(B - (int64_t)(kDepth - 1) * Q * b_t, C, x - (int64_t)(kDepth - 1) * Q * x_t, len);
        unload(s_b0 + at * kTile, s_x0 + at * kX);
      }
      // This chunk has arrived.  Issued after it: the chunk before's y (four stores), or
      // the next chunk's B and x.
      if (counted && (STATES ? kDepth == 3 && ahead(left - Q) : i > 0)) wait_memory<STATES ? kRounds + kXRounds : 4>();
      else wait_memory<0>();
      __syncthreads();
      if (ahead(left - (kDepth - 1) * Q)) {
        load_rows(B, b_t, s_b0 + at_last * kTile);
        load_x(s_x0 + at_last * kX);
      }
    } else {
      if (i > 0) __syncthreads();  // the chunk before's readers
      unload(s_b0, s_x0);
      __syncthreads();
    }
    // The steps to the next chunk.
    B += (int64_t)Q * b_t;
    C += (int64_t)Q * c_t;
    x += (int64_t)Q * x_t;
    if constexpr (!DIRECT) {
      if (left > Q) fetch(B, C, x, (int)(left - Q < Q ? left - Q : Q));
    }
    if (i % 2 == 0) {
      dt += (int64_t)(2 * Q) * dt_t;
      load_dt(dt, left - 2 * Q);
    }
    const ChunkScalars& sc = s_sc[i & 1];
    const float rescale = i % 2 == 0 ? rescale_of[0] : rescale_of[1];
    // (Opaque: places of single reads and comparisons are made from these when they
    // are wanted.  Kept in registers from chunk to chunk they would spill, and a
    // reload waits for all of the loads ahead: a quarter more time.)
    int row_at = row_place<NP>(col, half), col_at = col_place<NP>(lane), ln = lane;
    asm volatile("" : "+v"(row_at), "+v"(col_at), "+v"(ln));
    Frag xf[KB][PL];
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
      for (int pl = 0; pl < PL; ++pl) xf[k][pl] = x_frag(s_x + pl * kX, k, ln);

    if constexpr (!STATES) {
      // Element (i, j) of G: the 8 tokens j of a fragment lie together.
      auto g_at = [&](int i, int j) { return s_g + ((j / 8) * 32 + i) * 8 + j % 8; };
      // ---- G = B C^T, lane = token i of C, registers = tokens j of B: the three 16 x 16
      // quadrants on and below the diagonal ----
      if (wave < 3) {
        const int iq = wave > 0 ? 1 : 0, jq = wave > 1 ? 1 : 0, ci = ln & 15, j0 = 4 * (ln >> 4);
        const int place = ci * NP + unit_place<NP>(ci, ln >> 4) * 8;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NP / 32; ++k) {
          Frag bf[PL], cf[PL];
#pragma unroll
          for (int pl = 0; pl < PL; ++pl) {
            bf[pl] = *reinterpret_cast<const Frag*>(s_b + pl * kTile + 16 * jq * NP + (place ^ (32 * k)));
            cf[pl] = *reinterpret_cast<const Frag*>(s_c + pl * kTile + 16 * iq * NP + (place ^ (32 * k)));
          }
#pragma unroll
          for (int u = 0; u < PL; ++u)
#pragma unroll
            for (int v = 0; u + v < PL; ++v) acc = mma16(bf[u], cf[v], acc);
        }
        float gv[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) gv[e] = iq > jq || j0 + e <= ci ? acc[e] : 0.f;
        store_f32<float, 4>(g_at(16 * iq + ci, 16 * jq + j0), gv);
      }
      // ---- h C_i^T: lane = token i, registers = columns p ----
      f32x16 acc;
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[r] = 0.f;
#pragma unroll
      for (int k = 0; k < NP / 16; ++k) {
        float hv[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) hv[e] = h[k / 2][8 * (k % 2) + e];
        Frag hf[SP], cf[PL];
        split(hv, hf);
#pragma unroll
        for (int pl = 0; pl < PL; ++pl) cf[pl] = row_frag(s_c + pl * kTile, row_at, k);
        acc = mma_parts(hf, cf, acc);
      }
      // This token's x, for D.
      auto own_x = [&](int q, float (&v)[4]) {
        v[0] = v[1] = v[2] = v[3] = 0.f;
#pragma unroll
        for (int pl = PL - 1; pl >= 0; --pl) {
          const uint2 u = *reinterpret_cast<const uint2*>(s_x + pl * kX + x_place(ln & 31, 8 * q + 4 * (ln >> 5)));
          v[0] += low_bf16(u.x), v[1] += high_bf16(u.x), v[2] += low_bf16(u.y), v[3] += high_bf16(u.y);
        }
      };
      constexpr bool kEarly = PL == 1 && !kTight;
      uint2 xr[kEarly ? 4 : 1];  // (one part: read before the barrier)
      if constexpr (kEarly) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          xr[q] = *reinterpret_cast<const uint2*>(s_x + x_place(ln & 31, 8 * q + 4 * (ln >> 5)));
      }
      const float my_p = sc.p[ln & 31];
      const bool wide = kPair || (i % 2 == 0 ? wide_of[0] : wide_of[1]);
      __syncthreads();
      if (ahead(left - Q)) load_rows(C, c_t, s_c);

      // ---- x^T S: S[i][j] = G[i][j] 2^(L_i - L_j) d_j for j <= i ----
      // Factors apart: 2^(L_i + K) is multiplied in at the end; G is 0 above the diagonal.
      const float my_r = kPair || wide ? sc.r[ln & 31] : 0.f;
      auto factor = [&](float pj, float qj, float rj) { return exp2_hw((my_p - pj) + (my_r - rj)) * qj; };
      if (wide) {
        const float whole = exp2_hw(my_p), f = fmaf(whole * 0.693147182f, my_r, whole);
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[r] *= f;
      }
      if (kPair || !wide) {
#pragma unroll
        for (int k = 0; k < KB; ++k) {
          float s[8];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int j0 = 16 * k + 8 * (ln >> 5) + 4 * q;
            float gv[4], pv[4], qv[4], rv[4];
            load_f32<float, 4>(g_at(ln & 31, j0), gv);
            load_f32<float, 4>(sc.q + j0, qv);
            if constexpr (kPair) {
              load_f32<float, 4>(sc.p + j0, pv);
              load_f32<float, 4>(sc.r + j0, rv);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if constexpr (kPair) {
                const float v = gv[e] * factor(pv[e], qv[e], rv[e]);
                s[4 * q + e] = j0 + e <= (ln & 31) ? v : 0.f;
              } else {
                s[4 * q + e] = gv[e] * qv[e];
              }
            }
          }
          Frag sf[SP];
          split(s, sf);
          acc = mma_parts(xf[k], sf, acc);
        }
      } else {
        // Term by term: a decay that leaves a float's range in the chunk has no factors
        // apart.
        for (int j = 0; j < Q; ++j) {
          const float gv = *g_at(ln & 31, j);
          const float s = gv * factor(sc.p[j], sc.q[j], sc.r[j]);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float xq[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int pl = PL - 1; pl >= 0; --pl) {
              const uint2 u = *reinterpret_cast<const uint2*>(s_x + pl * kX + x_place(j, 8 * q + 4 * (ln >> 5)));
              xq[0] += low_bf16(u.x), xq[1] += high_bf16(u.x), xq[2] += low_bf16(u.y), xq[3] += high_bf16(u.y);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[4 * q + e] = j <= (ln & 31) ? fmaf(s, xq[e], acc[4 * q + e]) : acc[4 * q + e];
          }
        }
      }
      bad = not_finite(acc, bad);
      const float f = wide ? 1.f : my_p;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float xq[4];
        if constexpr (kEarly) xq[0] = low_bf16(xr[q].x), xq[1] = high_bf16(xr[q].x), xq[2] = low_bf16(xr[q].y), xq[3] = high_bf16(xr[q].y);
        else own_x(q, xq);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[4 * q + e] = fmaf(acc[4 * q + e], f, D * xq[e]);
      }
      if (on && (ln & 31) < len) {
        T* row = y + ((ln & 31) * y_t + 4 * (ln >> 5));
        if (whole_p) {
#pragma unroll
          for (int q = 0; q < 4; ++q) store_any_f32<T, 4>(row + 8 * q, {acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]});
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (p0 + 8 * (r / 4) + 4 * (ln >> 5) + r % 4 < P) row[8 * (r / 4) + r % 4] = from_f32<T>(acc[r]);
        }
      }
      y += (int64_t)Q * y_t;
    }

    // ---- h <- 2^L_end h + B^T v ----
    if (rescale != 1.f) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 16; ++r) h[nt][r] *= rescale;
    }
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      float v[8];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float wv[4];
        load_f32<float, 4>(sc.w + 16 * k + 8 * (ln >> 5) + 4 * q, wv);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float xv = get(xf[k][PL - 1], 4 * q + e);
#pragma unroll
          for (int pl = PL - 2; pl >= 0; --pl) xv += get(xf[k][pl], 4 * q + e);
          v[4 * q + e] = xv * wv[e];
        }
      }
      Frag vf[3];
      split(v, vf);
      // (All 24 bits of v against the parts of B, largest terms first.)
#pragma unroll
      for (int pl = 0; pl < PL; ++pl) {
        Frag bt[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) bt[nt] = col_frag<NP>(s_b + pl * kTile, col_at, nt, k);
#pragma unroll
        for (int u = 0; u + pl < 3; ++u)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) h[nt] = mma(bt[nt], vf[u], h[nt]);
      }
    }
    if (i % 2 == 1 && left > Q) write_scalars(left - Q);
  }

  if constexpr (STATES) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) bad = not_finite(h[nt], bad);
  }
  // (Found again, and from the arguments themselves: kept over the chunks, all of this
  // takes registers from them.)
  struct Args {
    ScanArgs a;
    ScanSplit sp;
  };
  static_assert(alignof(ScanArgs) == alignof(ScanSplit), "the kernel's arguments, one after the other");
  typedef const __attribute__((address_space(4))) Args* ArgsAt;
  ArgsAt args = (ArgsAt)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(args));
  const ScanArgs& ea = ((const Args*)args)->a;
  const ScanSplit& esp = ((const Args*)args)->sp;
  const ChunkWork end = chunk_work<STATES>(ea, esp, ea.block0 + blockIdx.x, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
  if (end.on && __ballot(bad != 0.f) != 0ull) {
    // The recurrence itself, token by token, from the segment's start.  The products meet
    // zeros that it does not have (of S, of an exact number's lower parts, of padding), and
    // leave a float's range where factors apart or a part's rounding do: where they are not
    // finite they do not say what the result is.  2 x 16384 tokens, 64 heads x 64, N 128,
    // with an infinity in one head take 8 ms.  (The y stored so far are in place before they
    // are written again.)
    wait_memory<0>();
    int64_t t = end.t0;
    const int64_t row = end.first + t;
    const T* b_from = static_cast<const T*>(ea.b) + end.b * ea.b_b + row * ea.b_t + end.g * ea.b_g;
    const T* c_from = static_cast<const T*>(ea.c) + end.b * ea.c_b + row * ea.c_t + end.g * ea.c_g;
    const T* x_from = static_cast<const T*>(ea.x) + end.b * ea.x_b + row * ea.x_t + end.hd * ea.x_h + min(end.p0 + col, P - 1);
    const T* dt_from = static_cast<const T*>(ea.dt) + end.b * ea.dt_b + row * ea.dt_t + end.hd * ea.dt_h;
    T* y_to = static_cast<T*>(ea.y) + end.b * ea.y_b + row * ea.y_t + end.hd * ea.y_h + end.p0 + col;
    const float rate = ea.A[end.hd], skip = ea.D != nullptr ? ea.D[end.hd] : 0.f;
    const float shift = ea.dt_bias != nullptr ? ea.dt_bias[end.hd] : 0.f;
    const float* start = STATES ? nullptr : start_of(end, ea, esp);
    float hv[NT * 16];
#pragma unroll
    for (int r = 0; r < NT * 16; ++r) {
      const int n = 32 * (r / 16) + 16 * (r / 8 % 2) + 8 * half + r % 8;
      hv[r] = start != nullptr ? start[(int64_t)min(end.p0 + col, P - 1) * N + min(n, N - 1)] : 0.f;
    }
    for (; t < end.t1; ++t) {
      float d = to_f32<T>(*dt_from) + shift;
      if (ea.softplus) d = softplus(d);
      const float decay = expf(rate * d), xv = to_f32<T>(*x_from), u = d * xv;
      float s = 0.f;
      int at = 8 * half;  // (opaque: what is made of it is not kept over the tokens)
      asm volatile("" : "+v"(at));
#pragma unroll
      for (int q = 0; q < 4 * NT; ++q) {
        const int n = 32 * (q / 4) + 16 * (q / 2 % 2) + 4 * (q % 2) + at;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int from = min(n + e, N - 1);
          float& now = hv[4 * q + e];
          now = fmaf(decay, now, u * to_f32<T>(b_from[from]));
          // (Columns past the end go nowhere.)
          if constexpr (!STATES)
            s += __uint_as_float(__float_as_uint(now * to_f32<T>(c_from[from])) & (uint32_t)((n + e - N) >> 31));
        }
        if (q % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (!STATES) {
        s += __shfl_xor(s, 32, kWave);
        if (half == 0 && end.p0 + col < P) *y_to = from_f32<T>(ea.D != nullptr ? fmaf(skip, xv, s) : s);
        c_from += ea.c_t;
        y_to += ea.y_t;
      }
      b_from += ea.b_t;
      x_from += ea.x_t;
      dt_from += ea.dt_t;
    }
#pragma unroll
    for (int r = 0; r < NT * 16; ++r) h[r / 16][r % 16] = hv[r];
    k_state = 0.0;
  }
  float* to = nullptr;
  if (STATES) to = esp.parts + ((end.row0 + end.seg) * ea.heads + end.hd) * plane;
  else if (end.seg == end.last && ea.h1 != nullptr && end.slot >= 0) to = ea.h1 + (end.slot * ea.heads + end.hd) * plane;
  const int p_end = end.p0 + col;
  if (to != nullptr && end.on && p_end < P) {
    const float f = exp2_of(k_state);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n0 = 32 * nt + 16 * (q / 2) + 8 * half + 4 * (q % 2);
        float* dst = to + (int64_t)p_end * N + n0;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = h[nt][4 * q + e] * f;
        if (vec_n) {
          if (n0 < N) store_any_f32<float, 4>(dst, v);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n0 + e < N) dst[e] = v[e];
        }
      }
  }
  if (STATES && end.on && end.p0 == 0 && lane == 0) esp.sums[(end.row0 + end.seg) * ea.heads + end.hd] = (float)l_seg;
}

// Segment by segment, the state that the next one starts from, in the place of that
// one's own part; the first one's, from the pool, in the place of its own.
constexpr int kChainThreads = 256;
template <int V>
__global__ __launch_bounds__(kChainThreads) void k_scan_chain(ScanArgs a, ScanSplit sp, int blocks) {
  int64_t item = a.block0 + blockIdx.x;
  const int part = (int)(item % blocks);
  item /= blocks;
  const int hd = (int)(item % a.heads);
  const int64_t b = item / a.heads;
  int64_t first, n;
  seq_rows(a.seq, b, first, n);
  const int last = last_segment(sp, n);
  const int64_t plane = (int64_t)a.head_dim * a.state_dim;
  const int64_t e = ((int64_t)part * kChainThreads + threadIdx.x) * V;
  if (last == 0 || e >= plane) return;
  const int64_t slot = seq_slot(a.seq, b);
  float h[V] = {};
  const int64_t row0 = first_row(sp, b, first);
  float* at = sp.parts + (row0 * a.heads + hd) * plane + e;
  const float* sum = sp.sums + row0 * a.heads + hd;
  float own[V];
  load_any_f32<float, V>(at, own);
  if (a.h0 != nullptr && slot >= 0) {
    load_any_f32<float, V>(a.h0 + (slot * a.heads + hd) * plane + e, h);
    store_any_f32<float, V>(at, h);
  }
  for (int s = 0; s < last; ++s) {
    float* const next = at + a.heads * plane;
    float next_own[V] = {};
    if (s + 1 < last) load_any_f32<float, V>(next, next_own);
    const float decay = exp2f(*sum);
    // (Infinity times each of a segment's decays stays so, though their product is 0.)
    const bool stays = decay == 0.f && *sum > -__builtin_huge_valf();
#pragma unroll
    for (int i = 0; i < V; ++i) {
      h[i] = stays && fabsf(h[i]) == __builtin_huge_valf() ? h[i] + own[i] : fmaf(h[i], decay, own[i]);
      own[i] = next_own[i];
    }
    store_any_f32<float, V>(next, h);
    at = next;
    sum += a.heads;
  }
}

template <typename T, int PL, int NP, bool DIRECT, bool STATES>
int launch_chunk_k(const ScanArgs& a, const ScanSplit& sp, hipStream_t stream) {
  const int rc = set_lds_limit_once<k_scan_chunk<T, PL, NP, DIRECT, STATES>>(kMaxLdsBytes);
  if (rc != (int)hipSuccess) return rc;
  constexpr int lds = ChunkLds<PL, NP>::bytes(chunk_depth<NP, DIRECT, STATES>(), STATES);
  static_assert(lds <= kMaxLdsBytes, "a workgroup's LDS");
  const int64_t blocks = a.seq.batch * (STATES ? sp.segments - 1 : sp.segments) * a.groups * sp.blocks;
  return launch_blocks(a, &ScanArgs::block0, blocks, [&](const ScanArgs& la, unsigned n) {
    hipLaunchKernelGGL((k_scan_chunk<T, PL, NP, DIRECT, STATES>), dim3(n), dim3(kThreads), lds, stream, la, sp);
  });
}

template <int V>
int launch_chain(const ScanArgs& a, const ScanSplit& sp, hipStream_t stream) {
  constexpr int each = kChainThreads * V;
  const int64_t blocks = ((int64_t)a.head_dim * a.state_dim + each - 1) / each;
  return launch_blocks(a, &ScanArgs::block0, a.seq.batch * a.heads * blocks, [&](const ScanArgs& la, unsigned n) {
    hipLaunchKernelGGL(k_scan_chain<V>, dim3(n), dim3(kChainThreads), 0, stream, la, sp, (int)blocks);
  });
}

template <typename T, int PL, int NP, bool DIRECT>
int launch_chunk_n(const ScanArgs& a, const ScanSplit& sp, hipStream_t stream) {
  if (sp.segments > 1) {
    timing_begin(K_SCAN_PARTS, stream);
    int rc = launch_chunk_k<T, PL, NP, DIRECT, true>(a, sp, stream);
    if (rc == (int)hipSuccess) {
      rc = a.state_dim % 4 == 0 ? launch_chain<4>(a, sp, stream) : launch_chain<1>(a, sp, stream);
    }
    timing_end(K_SCAN_PARTS, stream);
    if (rc != (int)hipSuccess) return rc;
  }
  timing_begin(K_SCAN_CHUNK, stream);
  const int rc = launch_chunk_k<T, PL, NP, DIRECT, false>(a, sp, stream);
  timing_end(K_SCAN_CHUNK, stream);
  return rc;
}

template <typename T, int PL, bool DIRECT>
int launch_chunk_m(const ScanArgs& a, const ScanSplit& sp, hipStream_t stream) {
  if (a.state_dim <= 32) return launch_chunk_n<T, PL, 32, DIRECT>(a, sp, stream);
  if (a.state_dim <= 64) return launch_chunk_n<T, PL, 64, DIRECT>(a, sp, stream);
  if (a.state_dim <= 128) return launch_chunk_n<T, PL, 128, DIRECT>(a, sp, stream);
  return launch_chunk_n<T, PL, 256, DIRECT>(a, sp, stream);
}

size_t align16(size_t v) { return (v + 15) / 16 * 16; }

}  // namespace

ScanPlan scan_plan(int64_t batch, int64_t tokens, int64_t max_len, int heads, int head_dim, int groups, int state_dim, int dtype) {
  ScanPlan p{};
  p.chunked = max_len >= kScanChunkFrom;
  if (!p.chunked || batch < 1) return p;
  const int units = heads / groups * ((head_dim + kSlice - 1) / kSlice);
  p.split.blocks = (units + kWaves - 1) / kWaves;
  // Segments: as many as the CUs hold workgroups for at once (fit: of a CU), since one
  // more makes all wait for a second turn (32 x 1024 tokens of f16, 24 heads x 64, N 128:
  // 334 us as 768 workgroups, 245 as 384), and of two chunks or more (1 x 512 of bf16, 16
  // heads: 43 us in segments of four, 39 of two).  In a packed call the sequences are
  // taken to fill their tokens with their longest.
  // Whole, a call of up to a workgroup to a CU takes a time per chunk; cut, one per chunk
  // and workgroup that comes to the same near a workgroup for each of 7/8 of the CUs, and
  // for the passes and their launches the time of 14 chunks (bf16), 8 (f16) or 6
  // (float32).  Whole and cut, us, 24 heads x 64, N 128 (other shapes of a head were not
  // measured): bf16 2 x 512 57 and 46, 5 x 512 59 and 61, 8 x 1024 104 and 94, 16 x 1024
  // 108 and 126, 16 x 4096 390 and 366, 21 x 4096 400 and 426; f16 5 x 512 76 and 66, 11 x
  // 512 79 and 93, 11 x 1024 145 and 133, 16 x 1024 146 and 166; float32 8 x 256 58 and 67,
  // 8 x 512 105 and 90, 16 x 512 108 and 128.
  const int64_t fit = state_dim > 128 ? 1 : dtype == SF_BF16 ? 3 : 2;
  const int64_t passes = dtype == SF_BF16 ? 14 : dtype == SF_F16 ? 8 : 6;
  const int64_t chunks = (max_len + kChunk - 1) / kChunk, cus = num_cus();
  int64_t full = batch;
  if (max_len < tokens && (tokens + max_len - 1) / max_len < full) full = (tokens + max_len - 1) / max_len;
  const int64_t base = full * groups * p.split.blocks;
  int64_t segs = chunks * (7 * cus - 8 * base) > passes * 7 * cus ? fit * cus / base : 1;
  if (segs > chunks / 2) segs = chunks / 2;
  if (segs < 1) segs = 1;
  const int64_t per = (chunks + segs - 1) / segs;
  p.split.chunks = (int)per;
  p.split.segments = (int)((chunks + per - 1) / per);
  if (p.split.segments > 1) {
    // (max_len < tokens: a packed call, batch sequences of `tokens` tokens in all.)
    const int64_t by_number = batch * p.split.segments, by_tokens = tokens / (per * kChunk) * 2 + 2;
    p.split.by_tokens = max_len < tokens && by_tokens < by_number ? 1 : 0;
    const size_t rows = (size_t)(p.split.by_tokens ? by_tokens : by_number) * heads;
    p.sums_at = align16(rows * head_dim * state_dim * sizeof(float));
    p.bytes = p.sums_at + align16(rows * sizeof(float));
  }
  return p;
}

bool scan_chunk_takes(const ScanArgs& a) {
  const int64_t most = 1 << 24;
  for (const int64_t s : {a.x_t, a.dt_t, a.b_t, a.c_t, a.y_t})
    if (s < 0 || s > most) return false;
  return true;
}

int launch_scan_chunk(const ScanArgs& a, const ScanPlan& p, void* workspace, int dtype, hipStream_t stream) {
  ScanSplit sp = p.split;
  // (A descriptor of dense sequences whose max_len is not their tokens: not cut.)
  if (a.seq.offsets == nullptr && sp.by_tokens) sp.segments = 1;
  sp.parts = static_cast<float*>(workspace);
  sp.sums = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.sums_at);
  if (dtype == SF_F32) return launch_chunk_m<float, 3, false>(a, sp, stream);
  if (dtype == SF_F16) return launch_chunk_m<__half, 2, false>(a, sp, stream);
  // Rows of whole aligned units: straight into LDS (us of a call's kernels, and by way of
  // registers: 2 x 16384, 64 heads x 64, N 128, 535 and 590, 64 x 1024, 24 heads, 245 and
  // 290; of N up to 64 and of 256 the same within 4%).
  const int64_t strides = a.x_b | a.x_t | a.x_h | a.b_b | a.b_t | a.b_g | a.c_b | a.c_t | a.c_g;
  const bool units = strides % 8 == 0 && a.head_dim % 8 == 0 && a.state_dim % 8 == 0 && aligned_to(a.x, 16) &&
                     aligned_to(a.b, 16) && aligned_to(a.c, 16);
  if (units) return launch_chunk_m<__hip_bfloat16, 1, true>(a, sp, stream);
  return launch_chunk_m<__hip_bfloat16, 1, false>(a, sp, stream);
}

}  // namespace sf
