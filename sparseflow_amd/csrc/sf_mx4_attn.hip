// Attention over a paged cache in the microscaled 4-bit format, and the writing of it:
//   y_i = sum_t softmax_t(scale q_i . k_t) v_t   over the tokens t <= the query's own
//
// A query row is a (token, head) pair; the heads that share keys and values lie side by
// side, so that a tile of 16 rows is a token's heads, or several tokens'.
#include <type_traits>

#include "sf_mx4_cache.h"

namespace sf {
namespace {

// ---- writing -----------------------------------------------------------------
//
// Four lanes to a block as in sf_mx4.hip; a workgroup's threads walk the blocks of one
// sequence's new rows, keys and values in turn.
constexpr int kAppendThreads = 256;

template <typename T>
__global__ __launch_bounds__(kAppendThreads) void k_mx4_append(Mx4AppendArgs a) {
  const CacheView& c = a.cache;
  const int64_t id = a.block0 + blockIdx.x;
  const int64_t b = id / a.chunks;
  int64_t first, n;
  seq_rows(a.seq, b, first, n);
  const int64_t slot = seq_slot(a.seq, b);
  const int64_t per = (int64_t)c.heads * c.blocks * 2;  // blocks of a token
  const int64_t item = (id - b * a.chunks) * (kAppendThreads / 4) + (threadIdx.x >> 2);
  const int part = threadIdx.x & 3;
  bool live = slot >= 0 && item < n * per;
  float v[8];
  int64_t row = -1;
  int blk = 0, value = 0;
  if (live) {
    const int64_t i = item / per;
    const int rest = (int)(item - i * per), hb = rest >> 1;
    value = rest & 1;
    const int h = hb / c.blocks;
    blk = hb - h * c.blocks;
    const int64_t t = (int64_t)c.lengths[slot] - n + i;
    live = t >= 0 && t < cache_room(c);
    if (live) {
      const int32_t p = cache_page(c, c.tables + slot * c.width, t);
      row = cache_place(c, p, h, t);
      live = p >= 0;
    }
    if (live) {
      const int64_t* st = value ? a.v_strides : a.k_strides;
      const T* x = reinterpret_cast<const T*>(value ? a.v : a.k) + b * st[0] + (first + i) * st[1] + (int64_t)h * st[2];
      load8<T>(x, blk * kMx4Block + part * 8, a.head_dim, v);
    }
  }
  if (!live) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
  }
  uint32_t byte;
  const uint32_t codes = mx4_encode(v, byte);
  if (!live) return;
  const int64_t at = row * c.blocks + blk;
  reinterpret_cast<uint32_t*>(value ? c.v : c.k)[at * 4 + part] = codes;
  if (part == 0) (value ? c.v_scales : c.k_scales)[at] = (uint8_t)byte;
}

// ---- reading: 16 query rows to a workgroup ---------------------------------------
//
// One pass with the running maximum and sum of the softmax.  A wavefront takes 32 tokens
// at a time.  S = K Q^T comes from the matrix cores with a lane's column the query row and
// its four elements four tokens, which is what the second product wants of its depth when
// tokens are counted 4 g + i, 16 + 4 g + i; it takes V^T from LDS, where V lies as bf16, by
// transposing loads.  K's codes go straight from memory into the operand: lane (token, g)
// holds 8 NB columns of its token from 8 NB g, and Q's fragments are laid out the same.  The
// next tokens' codes are loaded before these are worked on, and the pages after those.
constexpr int kAttnWaves = 4;
constexpr int kAttnTokens = 32;

template <int NB>
struct AttnLds {
  static constexpr int stride = value_stride(NB);
  union {
    uint16_t v[kAttnWaves][kAttnTokens * stride];
    float o[kAttnWaves][16][32 * NB];
  };
  float m[kAttnWaves][16], l[kAttnWaves][16];
};

// 4 NB bytes of codes.
template <int NB>
__device__ __forceinline__ void load_codes(const uint8_t* __restrict__ from, uint32_t (&c)[NB]) {
  const uint32_t* p = reinterpret_cast<const uint32_t*>(from);
  if constexpr (NB % 4 == 0) {
#pragma unroll
    for (int i = 0; i < NB / 4; ++i) {
      const u32x4 u = reinterpret_cast<const u32x4*>(p)[i];
      c[4 * i] = u.x, c[4 * i + 1] = u.y, c[4 * i + 2] = u.z, c[4 * i + 3] = u.w;
    }
  } else if constexpr (NB % 2 == 0) {
#pragma unroll
    for (int i = 0; i < NB / 2; ++i) {
      const u32x2 u = reinterpret_cast<const u32x2*>(p)[i];
      c[2 * i] = u.x, c[2 * i + 1] = u.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NB; ++i) c[i] = p[i];
  }
}

// A row's NB scales, at any address.
template <int NB>
__device__ __forceinline__ uint64_t load_scales(const uint8_t* __restrict__ p) {
  if constexpr (NB == 1) {
    return *p;
  } else {
    uint64_t s = 0;
    __builtin_memcpy(&s, p, NB);
    return s;
  }
}

// 32 tokens as they lie in memory: keys of tokens r and 16 + r, values as 16-byte blocks
// lane + 64 u, block `% NB` of token `/ NB`.
template <int NB>
struct RawTokens {
  static constexpr int VU = (NB + 1) / 2;
  uint32_t k[2][NB];
  uint64_t ks[2];
  u32x4 v[VU];
  uint32_t vs[VU];
  uint32_t have;  // which tokens have a page
  bool far;       // some value's scale is kFarScale or more

  // pages: lane t's is token t0 + t's, or -1 (t < 32).
  __device__ __forceinline__ void load(const CacheView& c, int64_t t0, int kvh, int32_t pages, int lane) {
    const int r = lane & 15, g = lane >> 4;
    have = (uint32_t)__ballot(pages >= 0);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int t = 16 * u + r;
      const int32_t p = __shfl(pages, t, kWave);
      const int64_t at = cache_place(c, p, kvh, t0 + t);
      load_codes<NB>(token_or_none(p >= 0, c.k + at * (16 * NB) + 4 * NB * g), k[u]);
      ks[u] = load_scales<NB>(token_or_none(p >= 0, c.k_scales + at * NB));
    }
#pragma unroll
    for (int u = 0; u < VU; ++u) {
      const int at = lane + kWave * u, tok = at / NB, blk = at - tok * NB;
      const int32_t p = __shfl(pages, tok & 31, kWave);
      const bool there = p >= 0 && (NB % 2 == 0 || at < kAttnTokens * NB);
      const int64_t row = cache_place(c, p, kvh, t0 + tok) * NB + blk;
      v[u] = *token_or_none(there, reinterpret_cast<const u32x4*>(c.v) + row);
      vs[u] = *token_or_none(there, c.v_scales + row);
    }
  }

  // The values as bf16 into LDS.
  __device__ __forceinline__ void put(uint16_t* vt, int lane) {
    far = false;
#pragma unroll
    for (int u = 0; u < VU; ++u) {
      const int at = lane + kWave * u, tok = at / NB, blk = at - tok * NB;
      const bool off = vs[u] >= kFarScale;
      far |= off;
      const float scale = mx4_scale(off ? 0 : vs[u]);
      if (off) v[u] = u32x4{0, 0, 0, 0};
      if (NB % 2 == 0 || at < kAttnTokens * NB) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<bf16x8*>(vt + tok * value_stride(NB) + blk * 32 + 8 * value_unit(j, tok)) = mx4_bf16(v[u][j], scale);
      }
    }
  }
};

template <typename T, int NB>
__global__ __launch_bounds__(kAttnWaves* kWave, NB * Parts<T>::n <= 8 ? 2 : 1) void k_mx4_attn_rows(Mx4AttnArgs a) {
  constexpr int NP = Parts<T>::n;
  constexpr int stride = AttnLds<NB>::stride;
  __shared__ AttnLds<NB> lds;
  const CacheView& c = a.cache;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), r = lane & 15, g = lane >> 4;

  // Which sequence, shared head, rows and part of the tokens.
  int64_t id = a.block0 + blockIdx.x;
  const int split = (int)(id % a.splits);
  id /= a.splits;
  const int64_t tile = id % a.tiles;
  id /= a.tiles;
  const int kvh = (int)(id % c.heads);
  const int64_t b = id / c.heads;
  int64_t first, n;
  seq_rows(a.seq, b, first, n);
  const int64_t slot = seq_slot(a.seq, b);
  const int group = a.group;
  const int64_t row0 = tile * 16, rows = n * group;
  if (row0 >= rows) return;
  const int64_t length = slot < 0 ? 0 : c.lengths[slot];
  const int64_t room = cache_room(c);

  // This lane's query row.
  const int64_t row = row0 + r < rows ? row0 + r : rows - 1;
  const int64_t i = row / group;
  const int head = kvh * group + (int)(row - i * group);
  const int64_t place = slot < 0 ? -1 : length - n + i;
  bf16x8 qf[NB][NP];
  {
    const T* q = reinterpret_cast<const T*>(a.q) + b * a.q_strides[0] + (first + i) * a.q_strides[1] + (int64_t)head * a.q_strides[2];
#pragma unroll
    for (int j = 0; j < NB; ++j) load_query<T, NP>(q, 8 * (NB * g + j), a.head_dim, a.scale, qf[j]);
  }

  // The keys that any of the tile's rows sees, and this part's share of them.
  const int64_t last_row = row0 + 15 < rows - 1 ? row0 + 15 : rows - 1;
  int64_t keys = slot < 0 ? 0 : length - n + last_row / group + 1;
  keys = keys < 0 ? 0 : keys > room ? room : keys;
  const int64_t place0 = length - n + row0 / group;  // the tile's first row's
  const int64_t chunks = (keys + kAttnTokens - 1) / kAttnTokens;
  const int64_t begin = chunks * split / a.splits, end = chunks * (split + 1) / a.splits;
  const int32_t* table = slot < 0 ? nullptr : c.tables + slot * c.width;
  auto pages_at = [&](int64_t ch) {
    const int64_t t = ch * kAttnTokens + (lane & 31);
    const int32_t p = cache_page(c, table, t < keys ? t : keys - 1);
    return ch < end && t < keys ? p : -1;
  };

  float ref = -INFINITY, l = 0.f;  // the running maximum, times scale and log2(e)
  f32x4 o[2 * NB];
#pragma unroll
  for (int d = 0; d < 2 * NB; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  const float c2 = score_factor(a.scale);
  uint16_t* vt = lds.v[wave];

  auto work = [&](int64_t t0, RawTokens<NB>& raw) {
    f32x4 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const bf16x8 kf = mx4_bf16(raw.k[u][j], mx4_scale((uint32_t)(raw.ks[u] >> (8 * ((NB * g + j) >> 2))) & 255));
#pragma unroll
        for (int p = 0; p < NP; ++p) s[u] = mfma16(kf, qf[j][p], s[u]);
      }
    }
    wave_lds_sync();
    raw.put(vt, lane);
    wave_lds_sync();

    // Which of this lane's tokens (t0 + 16 u + 4 g + k) its row sees.
    uint32_t seen = 255;
    if (t0 + kAttnTokens - 1 > place0 || raw.have != 0xffffffffu) {
      const int64_t d = place - t0;
      const uint32_t to = d < 0 ? 0 : d >= 31 ? 0xffffffffu : (2u << d) - 1, see = (raw.have & to) >> (4 * g);
      seen = (see & 15) | (see >> 12 & 0xf0);
#pragma unroll
      for (int k = 0; k < 8; ++k) s[k >> 2][k & 3] = seen >> k & 1 ? s[k >> 2][k & 3] : -INFINITY;
    }
    float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    top = fmaxf(top, __shfl_xor(top, 16, kWave));
    top = fmaxf(top, __shfl_xor(top, 32, kWave)) * c2;
    if (__any(top > ref + kRefSlack)) {
      const float was = ref;
      ref = fmaxf(ref, top);
      const float back = exp2_hw(was - (ref == -INFINITY ? 0.f : ref));  // (was = -inf: 0)
      l *= back;
#pragma unroll
      for (int d = 0; d < 2 * NB; ++d) o[d] *= back;
    }
    const float from = ref == -INFINITY ? 0.f : ref;  // (a row that has seen nothing yet)
    float pr[8], sum = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      pr[k] = exp2_hw(fmaf(s[k >> 2][k & 3], c2, -from));
      sum += pr[k];
    }
    l += sum;
    bf16x8 pf[NP];
    weight_parts<NP>(pr, pf);
#pragma unroll
    for (int d = 0; d < 2 * NB; ++d) {
      const int tok = 4 * g + (r >> 2);
      const uint16_t* at = vt + tok * stride + 32 * (d >> 1) + 8 * value_unit(2 * (d & 1) + (r >> 1 & 1), tok) + 4 * (r & 1);
      const bf16x8 vf = __builtin_shufflevector(lds_transposed(at), lds_transposed(at + 16 * stride), 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
      for (int p = 0; p < NP; ++p) o[d] = mfma16(vf, pf[p], o[d]);
    }
    if (__any(raw.far)) {
      for (int t = 0; t < kAttnTokens; ++t) {
        if (!(raw.have >> t & 1)) continue;
        const int64_t at = cache_place(c, cache_page(c, table, t0 + t), kvh, t0 + t) * NB;
        const int lane_of = 16 * ((t & 15) >> 2) + r, k = 4 * (t >> 4) + (t & 3);
        float p = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e == k) p = __shfl(pr[e], lane_of, kWave);
        if (t0 + t > place) continue;
#pragma unroll
        for (int d = 0; d < 2 * NB; ++d) {
          const uint32_t byte = c.v_scales[at + (d >> 1)];
          if (byte < kFarScale) continue;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            o[d][e] += p * far_value(reinterpret_cast<const uint32_t*>(c.v) + (at + (d >> 1)) * 4, byte, 16 * (d & 1) + 4 * g + e);
        }
      }
    }
  };

  // (The pages first: loads come back in order, and those of the tokens need not be waited for
  // when the pages are needed.)
  RawTokens<NB> raw[2];
  int64_t ch = begin + wave;
  if (ch < end) {
    int32_t pages = pages_at(ch), after = pages_at(ch + kAttnWaves);
    raw[0].load(c, ch * kAttnTokens, kvh, pages, lane);
    for (; ch < end; ch += 2 * kAttnWaves) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int64_t at = ch + u * kAttnWaves;
        if (at >= end) break;
        pages = after;
        after = pages_at(at + 2 * kAttnWaves);
        raw[1 - u].load(c, (at + kAttnWaves) * kAttnTokens, kvh, pages, lane);
        work(at * kAttnTokens, raw[u]);
      }
    }
  }
  l += __shfl_xor(l, 16, kWave);
  l += __shfl_xor(l, 32, kWave);

  // The wavefronts' parts together.
  __syncthreads();
  if (g == 0) lds.m[wave][r] = ref, lds.l[wave][r] = l;
#pragma unroll
  for (int d = 0; d < 2 * NB; ++d) *reinterpret_cast<f32x4*>(&lds.o[wave][r][16 * d + 4 * g]) = o[d];
  __syncthreads();
  // (Thread: row threadIdx.x / 16, columns threadIdx.x % 16 + 16 k.)
  const int wr = threadIdx.x >> 4, wc = threadIdx.x & 15;
  const int64_t orow = row0 + wr;
  if (orow >= rows) return;
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < kAttnWaves; ++w) top = fmaxf(top, lds.m[w][wr]);
  const float from = top == -INFINITY ? 0.f : top;
  float f[kAttnWaves], total = 0.f;
#pragma unroll
  for (int w = 0; w < kAttnWaves; ++w) {
    f[w] = exp2_hw(lds.m[w][wr] - from);
    total += f[w] * lds.l[w][wr];
  }
  if (a.splits > 1) {
    const int64_t base = (((b * c.heads + kvh) * a.tiles + tile) * a.splits + split) * 16 + wr;
    if (wc == 0) a.parts_ml[2 * base] = top, a.parts_ml[2 * base + 1] = total;
#pragma unroll
    for (int k = 0; k < 2 * NB; ++k) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kAttnWaves; ++w) v += f[w] * lds.o[w][wr][16 * k + wc];
      a.parts_o[base * (32 * NB) + 16 * k + wc] = v;
    }
    return;
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const int64_t oi = orow / group;
  T* y = reinterpret_cast<T*>(a.y) + b * a.y_strides[0] + (first + oi) * a.y_strides[1] +
         (int64_t)(kvh * group + (int)(orow - oi * group)) * a.y_strides[2];
#pragma unroll
  for (int k = 0; k < 2 * NB; ++k) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kAttnWaves; ++w) v += f[w] * lds.o[w][wr][16 * k + wc];
    if (16 * k + wc < a.head_dim) y[16 * k + wc] = from_f32<T>(total == 0.f ? 0.f : v * inv);
  }
}

// The parts of a row's tokens together: a workgroup to a row, a wavefront to every fourth
// part, a lane to its columns; four parts under way at a time.
template <typename T, int NB>
__global__ __launch_bounds__(256) void k_mx4_attn_join(Mx4AttnArgs a) {
  constexpr int C = (32 * NB + kWave - 1) / kWave;
  __shared__ float sums[4][kWave * C + 1];
  const CacheView& c = a.cache;
  const int lane = lane_id(), wave = threadIdx.x / kWave;
  const int64_t id = a.block0 + blockIdx.x;  // (b, kvh, tile, row of it)
  const int64_t tile_id = id / a.tile_rows;
  const int wr = (int)(id - tile_id * a.tile_rows);
  const int64_t tile = tile_id % a.tiles, bh = tile_id / a.tiles;
  const int kvh = (int)(bh % c.heads);
  const int64_t b = bh / c.heads;
  int64_t first, n;
  seq_rows(a.seq, b, first, n);
  const int64_t row = tile * a.tile_rows + wr;
  if (row >= n * a.group) return;
  const int64_t base = tile_id * a.splits * a.tile_rows + wr;
  float top = -INFINITY;
  for (int s = lane; s < a.splits; s += kWave) top = fmaxf(top, a.parts_ml[2 * (base + (int64_t)a.tile_rows * s)]);
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) top = fmaxf(top, __shfl_xor(top, d, kWave));
  const float from = top == -INFINITY ? 0.f : top;
  float total = 0.f, v[C] = {};
  for (int s0 = wave; s0 < a.splits; s0 += 16) {
    float f[4], q[4], p[4][C];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool in = s0 + 4 * k < a.splits;
      const int64_t at = base + (int64_t)a.tile_rows * (in ? s0 + 4 * k : s0);
      f[k] = in ? a.parts_ml[2 * at] : -INFINITY;
      q[k] = a.parts_ml[2 * at + 1];
#pragma unroll
      for (int e = 0; e < C; ++e) p[k][e] = kWave * e + lane < 32 * NB ? a.parts_o[at * (32 * NB) + kWave * e + lane] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (f[k] == -INFINITY) continue;  // (nothing seen there)
      const float g = exp2_hw(f[k] - from);
      total += g * q[k];
#pragma unroll
      for (int e = 0; e < C; ++e) v[e] += g * p[k][e];
    }
  }
#pragma unroll
  for (int e = 0; e < C; ++e) sums[wave][kWave * e + lane] = v[e];
  if (lane == 0) sums[wave][kWave * C] = total;
  __syncthreads();
  const int64_t i = row / a.group;
  T* y = reinterpret_cast<T*>(a.y) + b * a.y_strides[0] + (first + i) * a.y_strides[1] +
         (int64_t)(kvh * a.group + (int)(row - i * a.group)) * a.y_strides[2];
  total = (sums[0][kWave * C] + sums[1][kWave * C]) + (sums[2][kWave * C] + sums[3][kWave * C]);
  for (int k = threadIdx.x; k < a.head_dim; k += 256) {
    const float w = (sums[0][k] + sums[1][k]) + (sums[2][k] + sums[3][k]);
    y[k] = from_f32<T>(total == 0.f ? 0.f : w / total);
  }
}

template <typename T>
struct DType {
  static constexpr int code = sizeof(T) == 4 ? SF_F32 : std::is_same<T, __half>::value ? SF_F16 : SF_BF16;
};

template <typename T, int NB>
int launch_attn_nb(const Mx4AttnArgs& a, hipStream_t stream) {
  const int64_t tiles = a.seq.batch * a.cache.heads * a.tiles;
  int rc = a.tile_rows > 16 ? launch_mx4_attn_tiles(a, DType<T>::code, stream)
                            : launch_blocks(a, &Mx4AttnArgs::block0, tiles * a.splits, [&](const Mx4AttnArgs& part, unsigned grid) {
                                k_mx4_attn_rows<T, NB><<<grid, kAttnWaves * kWave, 0, stream>>>(part);
                              });
  if (rc != (int)hipSuccess || a.splits == 1) return rc;
  return launch_blocks(a, &Mx4AttnArgs::block0, tiles * a.tile_rows, [&](const Mx4AttnArgs& part, unsigned grid) {
    k_mx4_attn_join<T, NB><<<grid, 256, 0, stream>>>(part);
  });
}

template <typename T>
int launch_attn(const Mx4AttnArgs& a, hipStream_t stream) {
  switch (a.cache.blocks) {
    case 1: return launch_attn_nb<T, 1>(a, stream);
    case 2: return launch_attn_nb<T, 2>(a, stream);
    case 3: return launch_attn_nb<T, 3>(a, stream);
    case 4: return launch_attn_nb<T, 4>(a, stream);
    case 5: return launch_attn_nb<T, 5>(a, stream);
    case 6: return launch_attn_nb<T, 6>(a, stream);
    case 7: return launch_attn_nb<T, 7>(a, stream);
    default: return launch_attn_nb<T, 8>(a, stream);
  }
}

template <typename T>
int launch_append(Mx4AppendArgs a, hipStream_t stream) {
  const int64_t items = a.max_len * a.cache.heads * a.cache.blocks * 2;
  a.chunks = (items + kAppendThreads / 4 - 1) / (kAppendThreads / 4);
  return launch_blocks(a, &Mx4AppendArgs::block0, a.seq.batch * a.chunks, [&](const Mx4AppendArgs& part, unsigned grid) {
    k_mx4_append<T><<<grid, kAppendThreads, 0, stream>>>(part);
  });
}

}  // namespace

Mx4AttnPlan mx4_attn_plan(int64_t batch, int64_t max_len, int heads, int kv_heads, int blocks, int64_t room) {
  Mx4AttnPlan p{};
  const int64_t rows = max_len * (heads / kv_heads);
  p.tile_rows = rows <= kAttnFewRows ? 16 : kAttnTileRows;
  p.tiles = (rows + p.tile_rows - 1) / p.tile_rows;
  const int64_t items = batch * kv_heads * p.tiles;
  // As many parts of the tokens as fill the CUs, each of 256 tokens or more.
  const int64_t want = p.tile_rows == 16 ? 1024 : 512;
  int64_t splits = items == 0 ? 1 : want / items;
  const int64_t most = (room + 255) / 256;
  splits = splits > most ? most : splits;
  p.splits = (int)(splits < 1 ? 1 : splits > 512 ? 512 : splits);
  p.parts = p.splits == 1 ? 0 : items * p.splits * p.tile_rows;
  p.bytes = (size_t)p.parts * (size_t)(32 * blocks + 2) * 4;
  return p;
}

int launch_mx4_append(const Mx4AppendArgs& a, int dtype, hipStream_t stream) {
  timing_begin(K_MX4_APPEND, stream);
  const int rc = dtype == SF_F16    ? launch_append<__half>(a, stream)
                 : dtype == SF_BF16 ? launch_append<__hip_bfloat16>(a, stream)
                                    : launch_append<float>(a, stream);
  timing_end(K_MX4_APPEND, stream);
  return rc;
}

int launch_mx4_attn(const Mx4AttnArgs& a, int dtype, hipStream_t stream) {
  timing_begin(K_MX4_ATTN, stream);
  const int rc = dtype == SF_F16    ? launch_attn<__half>(a, stream)
                 : dtype == SF_BF16 ? launch_attn<__hip_bfloat16>(a, stream)
                                    : launch_attn<float>(a, stream);
  timing_end(K_MX4_ATTN, stream);
  return rc;
}

}  // namespace sf
