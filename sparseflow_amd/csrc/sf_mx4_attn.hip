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
//
// Sequences differ in length, and a workgroup takes some 5 us to begin and to end: so there
// are as many as the CUs hold, and the units (128 tokens of a tile of rows) of all sequences,
// one after another, are cut into as many even shares.  A share's ends may lie inside a tile's
// tokens: those parts go to the workspace, two at most of a workgroup, and k_mx4_attn_join
// puts them together.  (64 x 8192 tokens, with bf16 weights in one part: 119 us; in two equal parts
// a tile 138, in four 160, in eight 189.)
constexpr int kAttnWaves = 4;
constexpr int kAttnTokens = 32;
constexpr int kAttnUnit = kAttnWaves;   // chunks of kAttnTokens: one to a wavefront
constexpr int kAttnShare = 2;           // units that a workgroup takes at least, where they are parts of tiles

// A sequence's part of the work: tiles of 16 query rows of each shared head, of `units` each.
struct SeqWork {
  int64_t first, n, slot, length;  // its rows, its row of the tables, its tokens
  int64_t keys;                    // tokens that its last query sees
  int64_t tiles, units;
  __device__ __forceinline__ int64_t all(int heads) const { return tiles * units * heads; }
};
__device__ __forceinline__ SeqWork seq_work(const Mx4AttnArgs& a, int64_t b) {
  SeqWork w;
  if (a.seq.offsets == nullptr) {
    w.first = 0;
    w.n = a.seq.tokens;
  } else {
    const int64_t lo = a.seq.offsets[b], hi = a.seq.offsets[b + 1];
    w.first = lo < 0 ? 0 : lo > a.seq.tokens ? a.seq.tokens : lo;
    const int64_t end = hi > a.seq.tokens ? a.seq.tokens : hi;
    w.n = end > w.first ? end - w.first : 0;
  }
  w.slot = seq_slot(a.seq, b);
  w.length = w.slot < 0 ? 0 : a.cache.lengths[w.slot];
  const int64_t room = cache_room(a.cache);
  w.keys = w.length < 0 ? 0 : w.length > room ? room : w.length;
  w.tiles = ((w.n < a.max_len ? w.n : a.max_len) * a.group + 15) / 16;
  const int64_t chunks = (w.keys + kAttnTokens - 1) / kAttnTokens;
  w.units = chunks <= kAttnUnit * a.unit ? 1 : (chunks + kAttnUnit * a.unit - 1) / (kAttnUnit * a.unit);
  return w;
}

// The sum of the threads' values before this one's, and of all (256 threads).
__device__ __forceinline__ int64_t work_before(int64_t v, int64_t& total) {
  __shared__ int64_t part[4];
  const int lane = lane_id(), wave = threadIdx.x / kWave;
  int64_t in = v;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int64_t o = __shfl_up(in, d, kWave);
    if (lane >= d) in += o;
  }
  if (lane == kWave - 1) part[wave] = in;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    before += w < wave ? part[w] : 0;
    total += part[w];
  }
  return before + in - v;
}

// Where this thread's sequences begin, and the units of all; the sequences are dealt to the
// threads in runs.
__device__ __forceinline__ int64_t run_of_sequences(const Mx4AttnArgs& a) { return (a.seq.batch + 255) / 256; }
__device__ __forceinline__ int64_t work_of_run(const Mx4AttnArgs& a, int64_t& total) {
  const int64_t run = run_of_sequences(a), b0 = threadIdx.x * run;
  int64_t mine = 0;
  for (int64_t b = b0; b < b0 + run && b < a.seq.batch; ++b) mine += seq_work(a, b).all(a.cache.heads);
  return work_before(mine, total);
}

// at[0]: the sequence of a unit, at[1]: where the sequence begins (`before`: where this
// thread's do).
__device__ __forceinline__ void find_unit(const Mx4AttnArgs& a, int64_t unit, int64_t before, int64_t (&at)[2]) {
  const int64_t run = run_of_sequences(a), b0 = threadIdx.x * run;
  for (int64_t b = b0; b < b0 + run && b < a.seq.batch; ++b) {
    const int64_t all = seq_work(a, b).all(a.cache.heads);
    if (unit >= before && unit < before + all) at[0] = b, at[1] = before;
    before += all;
  }
  __syncthreads();
}

// Shares: workgroup k of `count` takes the units from share_begin(k) to share_begin(k + 1).
__device__ __forceinline__ int64_t shares(const Mx4AttnArgs& a, int64_t total) {
  const int64_t most = a.parts_o == nullptr ? total : total / kAttnShare;
  return most < 1 ? 1 : most < a.shares ? most : a.shares;
}
__device__ __forceinline__ int64_t share_begin(int64_t k, int64_t count, int64_t total) { return total * k / count; }
__device__ __forceinline__ int64_t share_of(int64_t unit, int64_t count, int64_t total) {
  return ((unit + 1) * count + total - 1) / total - 1;
}

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
  bool large, far;  // some value's scale is kLargeScale, kFarScale or more

  // pages: lane t's is token t0 + t's, or -1 (t < 32).
  __device__ __forceinline__ void load(const CacheView& c, int64_t t0, int kvh, int32_t pages, int lane) {
    const int r = lane & 15, g = lane >> 4;
    have = (uint32_t)__ballot(pages >= 0);
    int32_t kp[2], vp[VU];
#pragma unroll
    for (int u = 0; u < 2; ++u) kp[u] = __shfl(pages, 16 * u + r, kWave);
#pragma unroll
    for (int u = 0; u < VU; ++u) vp[u] = __shfl(pages, (lane + kWave * u) / NB & 31, kWave);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int64_t at = cache_place(c, kp[u], kvh, t0 + 16 * u + r);
      load_codes<NB>(c.k + at * (16 * NB) + 4 * NB * g, k[u]);
      ks[u] = load_scales<NB>(c.k_scales + at * NB);
    }
#pragma unroll
    for (int u = 0; u < VU; ++u) {
      const int at = lane + kWave * u, tok = at / NB & 31, blk = at % NB;
      const int64_t row = cache_place(c, vp[u], kvh, t0 + tok) * NB + blk;
      v[u] = reinterpret_cast<const u32x4*>(c.v)[row];
      vs[u] = c.v_scales[row];
    }
  }

  // The values as bf16 into LDS.
  __device__ __forceinline__ void put(uint16_t* vt, int lane) {
    large = far = false;
#pragma unroll
    for (int u = 0; u < VU; ++u) {
      const int at = lane + kWave * u, tok = at / NB, blk = at - tok * NB;
      // (Of a token without a page scale 0: numbers, which get the weight 0.)
      const bool there = have >> (tok & 31) & 1, off = there && vs[u] >= kFarScale;
      large |= there && vs[u] >= kLargeScale;
      far |= off;
      const float scale = mx4_scale(there && !off ? vs[u] : 0);
      if (off) v[u] = u32x4{0, 0, 0, 0};
      if (NB % 2 == 0 || at < kAttnTokens * NB) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<bf16x8*>(vt + tok * value_stride(NB) + blk * 32 + 8 * value_unit(j, tok)) = mx4_bf16(v[u][j], scale);
      }
    }
  }
};

// Rows of a tile, and the chunks of their tokens that a workgroup takes.
struct TileWork {
  SeqWork seq;
  int64_t b, row0, begin, end;
  int64_t part;  // of the workspace, or -1: the tile's tokens are all there
  int kvh;
};

template <typename T, int NB>
__device__ __forceinline__ void attend_tile(const Mx4AttnArgs& a, const TileWork& work_of, AttnLds<NB>& lds) {
  constexpr int NP = Parts<T>::n;
  constexpr int stride = AttnLds<NB>::stride;
  const CacheView& c = a.cache;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), r = lane & 15, g = lane >> 4;
  const int64_t b = work_of.b, first = work_of.seq.first, n = work_of.seq.n, slot = work_of.seq.slot, length = work_of.seq.length;
  const int64_t row0 = work_of.row0, rows = n * a.group, begin = work_of.begin, end = work_of.end;
  const int kvh = work_of.kvh, group = a.group;

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

  const int64_t keys = work_of.seq.keys;
  const int64_t place0 = length - n + row0 / group;  // the tile's first row's
  const int32_t* table = slot < 0 ? nullptr : c.tables + slot * c.width;
  auto pages_at = [&](int64_t ch) {
    const int64_t t = ch * kAttnTokens + (lane & 31);
    const int32_t p = cache_page(c, table, t < keys ? t : keys - 1);
    return ch < end && t < keys ? p : -1;
  };

  float ref = -INFINITY, l = 0.f;
  bool roomy = false;
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
    const bool more = !roomy && __any(raw.large);
    if (more || ref_passed(top, ref, roomy)) {
      const float was = ref;
      roomy |= more;
      ref = ref_moved(ref, top, roomy, more);
      const float back = exp2_hw(was - (ref == -INFINITY ? 0.f : ref));  // (was = -inf: 0)
      l *= back;
#pragma unroll
      for (int d = 0; d < 2 * NB; ++d) o[d] *= back;
    }
    const float from = ref_from<NP>(ref, roomy);
    float pr[8], sum = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      pr[k] = weight_of<NP>(s[k >> 2][k & 3], c2, from, roomy);
      sum += pr[k];
    }
    l += sum;
    constexpr int WP = kWeightParts<T>;
    bf16x8 pf[WP];
    weight_parts<WP>(pr, pf);
    constexpr int DG = NB < 4 ? 2 * NB : 8;  // tiles of columns at a time
#pragma unroll
    for (int d0 = 0; d0 < 2 * NB; d0 += DG) {
      bf16x4v vf[DG][2];
#pragma unroll
      for (int d = d0; d < d0 + DG && d < 2 * NB; ++d) {
        const int tok = 4 * g + (r >> 2);
        const uint16_t* at = vt + tok * stride + 32 * (d >> 1) + 8 * value_unit(2 * (d & 1) + (r >> 1 & 1), tok) + 4 * (r & 1);
        vf[d - d0][0] = lds_transposed(at);
        vf[d - d0][1] = lds_transposed(at + 16 * stride);
      }
#pragma unroll
      for (int p = 0; p < WP; ++p)
#pragma unroll
        for (int d = d0; d < d0 + DG && d < 2 * NB; ++d)
          o[d] = mfma16(__builtin_shufflevector(vf[d - d0][0], vf[d - d0][1], 0, 1, 2, 3, 4, 5, 6, 7), pf[p], o[d]);
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
  ref = ref_of_seen(c, table, begin * kAttnTokens, end * kAttnTokens < keys ? end * kAttnTokens : keys, place, ref, l);

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
  if (work_of.part >= 0) {
    const int64_t base = work_of.part * 16 + wr;
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
  const bool none = nothing_seen(top, total);
  const float inv = 1.f / total;
  const int64_t oi = orow / group;
  T* y = reinterpret_cast<T*>(a.y) + b * a.y_strides[0] + (first + oi) * a.y_strides[1] +
         (int64_t)(kvh * group + (int)(orow - oi * group)) * a.y_strides[2];
#pragma unroll
  for (int k = 0; k < 2 * NB; ++k) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kAttnWaves; ++w) v += f[w] * lds.o[w][wr][16 * k + wc];
    if (16 * k + wc < a.head_dim) y[16 * k + wc] = from_f32<T>(none ? 0.f : v * inv);
  }
}

template <typename T, int NB>
__global__ __launch_bounds__(kAttnWaves* kWave, NB * kWeightParts<T> <= 8 ? 2 : 1) void k_mx4_attn_rows(Mx4AttnArgs a) {
  __shared__ AttnLds<NB> lds;
  __shared__ int64_t at[2];
  const int heads = a.cache.heads;
  int64_t total;
  const int64_t before = work_of_run(a, total);
  const int64_t count = shares(a, total), k = a.block0 + blockIdx.x;
  if (a.cuts != nullptr && threadIdx.x == 0) a.cuts[k].parts = 0;
  if (total == 0 || k >= count) return;
  int64_t unit = share_begin(k, count, total);
  const int64_t stop = share_begin(k + 1, count, total);
  find_unit(a, unit, before, at);
  TileWork w;
  w.b = __builtin_amdgcn_readfirstlane((int)at[0]);
  int64_t from = at[1];
  w.seq = seq_work(a, w.b);
  while (unit < stop) {
    while (unit >= from + w.seq.all(heads)) {
      from += w.seq.all(heads);
      w.seq = seq_work(a, ++w.b);
    }
    const int64_t in = unit - from, item = in / w.seq.units, u0 = in - item * w.seq.units;
    const int64_t left = stop - unit, u1 = u0 + left < w.seq.units ? u0 + left : w.seq.units;
    w.kvh = (int)(item / w.seq.tiles);
    w.row0 = (item - w.kvh * w.seq.tiles) * 16;
    const int64_t chunks = (w.seq.keys + kAttnTokens - 1) / kAttnTokens, per = kAttnUnit * a.unit;
    w.begin = u0 * per;
    w.end = u1 * per < chunks ? u1 * per : chunks;
    w.part = u0 == 0 && u1 == w.seq.units ? -1 : 2 * k + (u0 == 0);
    // (A tile that the workgroup before is the first to have a part of is this one's to report.)
    if (u0 > 0 && threadIdx.x == 0 && share_of(unit - u0, count, total) == k - 1) {
      AttnCut& cut = a.cuts[k];
      cut.b = w.b;
      cut.first = w.seq.first;
      cut.row0 = w.row0;
      cut.rows = w.seq.n * a.group;
      cut.kvh = w.kvh;
      cut.parts = (int)(share_of(unit - u0 + w.seq.units - 1, count, total) - k + 2);
    }
    attend_tile<T, NB>(a, w, lds);
    unit += u1 - u0;
    __syncthreads();
  }
}

// A row's parts together: W wavefronts to a row (of a workgroup's four), a lane to its columns, F
// parts under way; place(j) is part j's row of the workspace.  W = 1 where there are few parts
// and many rows (32 / 8 heads of 128, the call in us: 4 x 100 queries after 6000 tokens 115, with
// W = 4 152; 32 x 4 after 3000 45 and 61), W = 4 otherwise (one after 100,000: 48, with W = 1 60).
template <typename T, int NB, int W, typename Place>
__device__ __forceinline__ void join_row(const Mx4AttnArgs& a, int64_t parts, Place&& place, T* y) {
  constexpr int C = (32 * NB + kWave - 1) / kWave, F = C <= 2 ? 16 : 8;
  __shared__ float sums[W == 1 ? 1 : 4][kWave * C + 1];
  const int lane = lane_id(), wave = threadIdx.x / kWave % W;
  float top = -INFINITY;
  for (int64_t s = lane; s < parts; s += kWave) top = fmaxf(top, a.parts_ml[2 * place(s)]);
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) top = fmaxf(top, __shfl_xor(top, d, kWave));
  const float from = top == -INFINITY ? 0.f : top;
  float total = 0.f, v[C] = {};
  for (int64_t s0 = wave; s0 < parts; s0 += W * F) {
    float f[F], q[F], p[F][C];
#pragma unroll
    for (int k = 0; k < F; ++k) {
      const bool in = s0 + W * k < parts;
      const int64_t at = place(in ? s0 + W * k : s0);
      f[k] = a.parts_ml[2 * at];
      q[k] = a.parts_ml[2 * at + 1];
#pragma unroll
      for (int e = 0; e < C; ++e) p[k][e] = a.parts_o[at * (32 * NB) + (kWave * e + lane < 32 * NB ? kWave * e + lane : 0)];
    }
#pragma unroll
    for (int k = 0; k < F; ++k) {
      // (A part where nothing is seen has 0 times its zeros; NaN has -infinity for a maximum too, and stays.)
      if (s0 + W * k >= parts) continue;
      const float g = exp2_hw(f[k] - from);
      total += g * q[k];
#pragma unroll
      for (int e = 0; e < C; ++e) v[e] += g * p[k][e];
    }
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int e = 0; e < C; ++e) sums[wave][kWave * e + lane] = v[e];
    if (lane == 0) sums[wave][kWave * C] = total;
    __syncthreads();
    if (wave > 0) return;
    total = (sums[0][kWave * C] + sums[1][kWave * C]) + (sums[2][kWave * C] + sums[3][kWave * C]);
#pragma unroll
    for (int e = 0; e < C; ++e)
      v[e] = (sums[0][kWave * e + lane] + sums[1][kWave * e + lane]) + (sums[2][kWave * e + lane] + sums[3][kWave * e + lane]);
  }
#pragma unroll
  for (int e = 0; e < C; ++e)
    if (kWave * e + lane < a.head_dim) y[kWave * e + lane] = from_f32<T>(nothing_seen(top, total) ? 0.f : v[e] / total);
}
template <typename T>
__device__ __forceinline__ T* row_of_y(const Mx4AttnArgs& a, int64_t b, int64_t first, int kvh, int64_t row) {
  const int64_t i = row / a.group;
  return reinterpret_cast<T*>(a.y) + b * a.y_strides[0] + (first + i) * a.y_strides[1] +
         (int64_t)(kvh * a.group + (int)(row - i * a.group)) * a.y_strides[2];
}

// Tiles of 16 rows whose tokens several workgroups had: join_rows rows of each.
template <typename T, int NB, int W>
__global__ __launch_bounds__(256) void k_mx4_attn_join_cuts(Mx4AttnArgs a, int join_rows) {
  const int64_t id = (a.block0 + blockIdx.x) * (4 / W) + threadIdx.x / kWave / W, k = id / join_rows + 1;
  if (k >= a.shares) return;
  const AttnCut cut = a.cuts[k];
  const int wr = (int)(id % join_rows);
  const int64_t row = cut.row0 + wr;
  if (cut.parts == 0 || row >= cut.rows) return;
  // (The first part is a share's second one, the others are the first of theirs.)
  join_row<T, NB, W>(a, cut.parts, [&](int64_t j) { return (2 * (k - 1 + j) + (j == 0)) * 16 + wr; },
                     row_of_y<T>(a, cut.b, cut.first, cut.kvh, row));
}

// Tiles of kAttnTileRows rows.
template <typename T, int NB, int W>
__global__ __launch_bounds__(256) void k_mx4_attn_join(Mx4AttnArgs a) {
  const int64_t id = (a.block0 + blockIdx.x) * (4 / W) + threadIdx.x / kWave / W;  // (b, kvh, tile, row of it)
  const int64_t tile_id = id / kAttnTileRows;
  const int wr = (int)(id - tile_id * kAttnTileRows);
  const int64_t tile = tile_id % a.tiles, bh = tile_id / a.tiles, b = bh / a.cache.heads;
  int64_t first, n;
  seq_rows(a.seq, b, first, n);
  const int64_t row = tile * kAttnTileRows + wr;
  if (row >= n * a.group) return;
  join_row<T, NB, W>(a, a.splits, [&](int64_t j) { return (tile_id * a.splits + j) * kAttnTileRows + wr; },
                     row_of_y<T>(a, b, first, (int)(bh % a.cache.heads), row));
}

template <typename T>
struct DType {
  static constexpr int code = sizeof(T) == 4 ? SF_F32 : std::is_same<T, __half>::value ? SF_F16 : SF_BF16;
};

template <typename T, int NB>
int launch_attn_nb(const Mx4AttnArgs& a, hipStream_t stream) {
  const int64_t tiles = a.seq.batch * a.cache.heads * a.tiles;
  if (a.tile_rows == 16) {
    const int rc = launch_blocks(a, &Mx4AttnArgs::block0, a.shares, [&](const Mx4AttnArgs& part, unsigned grid) {
      k_mx4_attn_rows<T, NB><<<grid, kAttnWaves * kWave, 0, stream>>>(part);
    });
    if (rc != (int)hipSuccess || a.parts_o == nullptr) return rc;
    const int join_rows = (int)(a.max_len * a.group < 16 ? a.max_len * a.group : 16);
    const int64_t rows = (a.shares - 1) * join_rows;
    const bool few = tiles * 4 >= a.shares;  // parts of a tile
    return launch_blocks(a, &Mx4AttnArgs::block0, few ? (rows + 3) / 4 : rows, [&](const Mx4AttnArgs& part, unsigned grid) {
      if (few) k_mx4_attn_join_cuts<T, NB, 1><<<grid, 256, 0, stream>>>(part, join_rows);
      else k_mx4_attn_join_cuts<T, NB, 4><<<grid, 256, 0, stream>>>(part, join_rows);
    });
  }
  const int rc = launch_mx4_attn_tiles(a, DType<T>::code, stream);
  if (rc != (int)hipSuccess || a.parts_o == nullptr) return rc;
  const bool few = a.splits <= 16;
  return launch_blocks(a, &Mx4AttnArgs::block0, tiles * kAttnTileRows / (few ? 4 : 1), [&](const Mx4AttnArgs& part, unsigned grid) {
    if (few) k_mx4_attn_join<T, NB, 1><<<grid, 256, 0, stream>>>(part);
    else k_mx4_attn_join<T, NB, 4><<<grid, 256, 0, stream>>>(part);
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

Mx4AttnPlan mx4_attn_plan(int64_t batch, int64_t max_len, int heads, int kv_heads, int blocks, int dtype, int64_t room) {
  Mx4AttnPlan p{};
  const int64_t rows = max_len * (heads / kv_heads);
  p.tile_rows = rows <= kAttnFewRows ? 16 : kAttnTileRows;
  p.tiles = (rows + p.tile_rows - 1) / p.tile_rows;
  p.splits = 1;
  const int64_t items = batch * kv_heads * p.tiles;
  const int parts = dtype == SF_F32 ? 3 : dtype == SF_F16 ? 2 : 1;
  if (p.tile_rows == 16) {
    // Workgroups: what the CUs hold of them (by registers).  Short tables: a tile is one unit.
    p.unit = room <= 512 ? 4 : 1;
    const int64_t tokens = kAttnTokens * kAttnUnit * p.unit, units = room <= tokens ? 1 : (room + tokens - 1) / tokens;
    const int64_t hold = blocks * parts <= 2 ? 768 : blocks * (parts == 1 ? 2 : parts) <= 8 ? 512 : 256;
    const int64_t most = units > hold || items > hold ? hold : items * units;  // (no product of large numbers)
    p.shares = units == 1 ? (items < 4 * hold ? items : 4 * hold) : most < hold ? most : hold;
    p.shares = p.shares < 1 ? 1 : p.shares;
    p.parts = units == 1 ? 0 : 2 * p.shares * 16;
  } else {
    // Parts of the tokens only while all of them are on the CUs at once (of what they hold, by
    // registers), and where a part is long enough to be worth its rows' way through memory (bf16,
    // 32 / 8 heads of 128 in us: 1024 tokens 44 whole, 70 in two parts; 128 tiles of 4096 130 whole,
    // 97 in two, 84 in the four that fit, 92 in eight; 192 of 8000 261, 236 in the two that fit; but
    // 256 of 4000 146 and 153, of 2078 79 and 102).
    const int64_t hold = blocks <= 4 && blocks * parts <= 8 ? 512 : 256;
    int64_t splits = items == 0 || room < 2048 ? 1 : hold / items;
    const int64_t most = room / 256;
    splits = splits > most ? most : splits;
    p.splits = (int)(splits < 1 ? 1 : splits);
    p.parts = p.splits == 1 ? 0 : items * p.splits * p.tile_rows;
  }
  p.cuts_at = (size_t)p.parts * (size_t)(32 * blocks + 2) * 4;
  p.bytes = p.cuts_at + (p.tile_rows == 16 && p.parts > 0 ? (size_t)p.shares * sizeof(AttnCut) : 0);
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
