// Attention over the microscaled 4-bit cache for many query rows (see sf_mx4_attn.hip for the
// mathematics and for few rows).
//
// A workgroup takes 128 rows of one sequence and shared head, a wavefront 32; C tokens at a
// time, whose keys and values the workgroup turns into bf16 rows in LDS once for all of them,
// while the codes after those are under way.  S = K Q^T has a lane's column the query row and
// its sixteen elements tokens 8 (e / 4) + 4 h + e % 4 of 32, which is what the second product
// wants of its depth when its tokens are counted like that; V^T comes by transposing loads.
// Tiles with the most tokens begin first, and those of one sequence and shared head are a
// multiple of their number apart: on one XCD where that is a multiple of eight.
//
// Bound by its instructions: of 64 tokens a wavefront has 48 products of bf16 (32 cycles each; 32 of
// them take the weights' two parts) and some 420 vector instructions (4 cycles), of which the softmax
// is 220 and the widening of the codes 80.  2 x 8192 tokens, 32 / 8 heads of 128: bf16 1500 us (730
// TFLOP/s; with weights of one part 1200), f16 1950, float32 4000; 4 x 4096, 16 heads of 64: 282 us
// (490).
#include "sf_mx4_cache.h"

namespace sf {
namespace {

constexpr int kTileWaves = kAttnTileRows / 32;
constexpr int kTileThreads = kTileWaves * kWave;

// Tokens at a time: a 16-byte block of keys and one of values to a thread at most, and half of
// that where the queries' parts leave no registers for as many scores.
constexpr int tile_tokens(int nb, int np) { return nb * np <= 4 ? 64 : 32; }

template <int NB, int C>
struct TileLds {
  static constexpr int stride = value_stride(NB);
  struct Buf {
    uint16_t k[C][32 * NB + 8];   // bf16 rows: 16 bytes on, another bank
    uint16_t v[C][stride];
    uint32_t there[C];            // whether the token has a page
    // Of what each wavefront brought: 1 values from kFarScale on, 2 tokens without a page, 4 values from kLargeScale on.
    uint32_t flags[kTileWaves];
  };
  union {
    Buf buf[2];
    float o[kTileWaves][32][132];    // 128 columns at a time on their way out
  };
};

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

template <typename T, int NB>
__global__ __launch_bounds__(kTileThreads, NB <= 4 && Parts<T>::n < 3 ? 2 : 1) void k_mx4_attn_tile(Mx4AttnArgs a) {
  constexpr int NP = Parts<T>::n, C = tile_tokens(NB, NP), U = C / 32;
  using Lds = TileLds<NB, C>;
  constexpr int stride = Lds::stride;
  extern __shared__ __align__(16) char smem[];
  Lds& lds = *reinterpret_cast<Lds*>(smem);
  const CacheView& c = a.cache;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), r = lane & 31, h = lane >> 5;

  // Which rows, sequence, shared head and part of the tokens.
  int64_t id = a.block0 + blockIdx.x;
  const int64_t items = a.seq.batch * c.heads, item = id % items;
  id /= items;
  const int split = (int)(id % a.splits);
  const int64_t tile = a.tiles - 1 - id / a.splits;
  const int kvh = (int)(item % c.heads);
  const int64_t b = item / c.heads;
  int64_t first, n;
  seq_rows(a.seq, b, first, n);
  const int64_t slot = seq_slot(a.seq, b);
  const int group = a.group;
  const int64_t row0 = tile * kAttnTileRows, rows = n * group;
  if (row0 >= rows) return;
  const int64_t length = slot < 0 ? 0 : c.lengths[slot];

  // This lane's query row.
  const int64_t wrow0 = row0 + 32 * wave, row = wrow0 + r < rows ? wrow0 + r : rows - 1;
  const int64_t i = row / group;
  const int64_t last_place = slot < 0 ? -1 : cache_room(c) - 1;  // (tokens past the table are seen by nobody)
  auto place_in = [&](int64_t at) { return length - n + at < last_place ? length - n + at : last_place; };
  const int64_t place = place_in(i);
  bf16x8 qf[2 * NB][NP];
  {
    const T* q = reinterpret_cast<const T*>(a.q) + b * a.q_strides[0] + (first + i) * a.q_strides[1] +
                 (kvh * group + (row - i * group)) * a.q_strides[2];
#pragma unroll
    for (int j = 0; j < 2 * NB; ++j) load_query<T, NP>(q, 16 * j + 8 * h, a.head_dim, a.scale, qf[j]);
  }

  // The keys that any of the workgroup's rows sees, this part's share of them, and up to where
  // every row of the wavefront sees all, or one sees any.
  auto place_of = [&](int64_t at) { return place_in((at < rows ? at : rows - 1) / group); };
  int64_t keys = place_of(row0 + kAttnTileRows - 1) + 1;
  keys = keys < 0 ? 0 : keys;
  const int64_t all = place_of(wrow0) + 1, any = place_of(wrow0 + 31) + 1;
  const int64_t chunks = (keys + C - 1) / C, begin = chunks * split / a.splits, end = chunks * (split + 1) / a.splits;
  const int32_t* table = slot < 0 ? nullptr : c.tables + slot * c.width;

  // This thread's block of the tokens that are on their way: block `blk` of token `tok`.
  const int tok = threadIdx.x / NB, blk = threadIdx.x - tok * NB;
  const bool mine = threadIdx.x < C * NB;
  auto page_at = [&](int64_t ch) {
    const int64_t t = ch * C + tok;
    const int32_t p = cache_page(c, table, t < keys ? t : keys - 1);
    return mine && ch < end && t < keys ? p : -1;
  };
  u32x4 kc, vc;
  uint32_t ks, vs;
  bool there;
  auto load = [&](int64_t ch, int32_t page) {
    there = page >= 0;
    const int64_t at = cache_place(c, page, kvh, ch * C + tok) * NB + (mine ? blk : 0);
    kc = reinterpret_cast<const u32x4*>(c.k)[at];
    vc = reinterpret_cast<const u32x4*>(c.v)[at];
    ks = c.k_scales[at];
    vs = c.v_scales[at];
  };
  auto put = [&](int64_t ch, typename Lds::Buf& to) {
    // (Of a token without a page scale 0: numbers, which get the weight 0.)
    const bool far = there && vs >= kFarScale, large = there && vs >= kLargeScale;
    if (far) vc = u32x4{0, 0, 0, 0};
    if (far || !there) vs = 0;
    if (mine) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        *reinterpret_cast<bf16x8*>(&to.k[tok][32 * blk + 8 * j]) = mx4_bf16(kc[j], mx4_scale(ks));
        *reinterpret_cast<bf16x8*>(&to.v[tok][32 * blk + 8 * value_unit(j, tok)]) = mx4_bf16(vc[j], mx4_scale(vs));
      }
      if (blk == 0) to.there[tok] = there;
    }
    const uint32_t flags = (__any(far) ? 1 : 0) | (__any(mine && !there && ch * C + tok < keys) ? 2 : 0) | (__any(large) ? 4 : 0);
    if (lane == 0) to.flags[wave] = flags;
  };

  float ref = -INFINITY, l = 0.f;
  bool roomy = false;
  f32x16 o[NB];
#pragma unroll
  for (int d = 0; d < NB; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
  const float c2 = score_factor(a.scale);

  int32_t page = -1;
  if (begin < end) {
    const int32_t now = page_at(begin);
    page = page_at(begin + 1);
    load(begin, now);
    put(begin, lds.buf[begin & 1]);
    const int32_t after = page_at(begin + 2);
    load(begin + 1, page);
    page = after;
  }
  __syncthreads();
  for (int64_t ch = begin; ch < end; ++ch) {
    const typename Lds::Buf& t = lds.buf[ch & 1];
    put(ch + 1, lds.buf[~ch & 1]);
    // (The page first: loads come back in order, and the codes need not be waited for when the
    // page is needed.)
    const int32_t after = page_at(ch + 3);
    load(ch + 2, page);
    page = after;
    const int64_t t0 = ch * C;
    if (t0 < any) {
      f32x16 s[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[u][e] = 0.f;
#pragma unroll
        for (int j = 0; j < 2 * NB; ++j) {
          const bf16x8 kf = *reinterpret_cast<const bf16x8*>(&t.k[32 * u + r][16 * j + 8 * h]);
#pragma unroll
          for (int p = 0; p < NP; ++p) s[u] = mfma32(kf, qf[j][p], s[u]);
        }
      }
      uint32_t flags = 0;
#pragma unroll
      for (int w = 0; w < kTileWaves; ++w) flags |= t.flags[w];
      flags = __builtin_amdgcn_readfirstlane(flags);
      const int last = (int)(place - t0 < -1 ? -1 : place - t0 > C ? C : place - t0);  // the row's last token of these
      if (t0 + C > all || (flags & 2) != 0) {
        uint64_t see = last < 0 ? 0 : last >= 63 ? ~0ull : (2ull << last) - 1;
        if (flags & 2) {
          for (int at = 0; at < C; ++at)
            if (!t.there[at]) see &= ~(1ull << at);
        }
        see >>= 4 * h;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            s[u][e] = (uint32_t)(see >> (32 * u)) >> (8 * (e >> 2) + (e & 3)) & 1 ? s[u][e] : -INFINITY;
      }
      float top = s[0][0];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, s[u][e]);
      top = fmaxf(top, __shfl_xor(top, 32, kWave)) * c2;
      const bool more = !roomy && (flags & 4) != 0;
      if (more || ref_passed(top, ref, roomy)) {
        const float was = ref;
        roomy |= more;
        ref = ref_moved(ref, top, roomy, more);
        const float back = exp2_hw(was - (ref == -INFINITY ? 0.f : ref));  // (was = -inf: 0)
        l *= back;
#pragma unroll
        for (int d = 0; d < NB; ++d) o[d] *= back;
      }
      const float from = ref_from<NP>(ref, roomy);
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          s[u][e] = weight_of<NP>(s[u][e], c2, from, roomy);
          sum[e & 3] += s[u][e];
        }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
      for (int k = 0; k < C / 16; ++k) {
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = s[k >> 1][8 * (k & 1) + e];
        constexpr int WP = kWeightParts<T>;
        bf16x8 pf[WP];
        weight_parts<WP>(w, pf);
        const int tk = 4 * h + (lane >> 2 & 3), unit = value_unit(2 * (lane >> 4 & 1) + (lane >> 1 & 1), tk);
        const uint16_t* at = &t.v[16 * k + tk][8 * unit + 4 * (lane & 1)];
#pragma unroll
        for (int d = 0; d < NB; ++d) {
          const bf16x8 vf = __builtin_shufflevector(lds_transposed(at + 32 * d), lds_transposed(at + 32 * d + 8 * stride), 0, 1, 2,
                                                    3, 4, 5, 6, 7);
#pragma unroll
          for (int p = 0; p < WP; ++p) o[d] = mfma32(vf, pf[p], o[d]);
        }
      }
      if (flags & 1) {
        for (int at = 0; at < C && t0 + at < keys; ++at) {
          if (!t.there[at]) continue;
          const int64_t place_of_it = cache_place(c, cache_page(c, table, t0 + at), kvh, t0 + at) * NB;
          const int lane_of = r + 32 * (at >> 2 & 1), k = 16 * (at >> 5) + 4 * (at >> 3 & 3) + (at & 3);
          float p = 0.f;
#pragma unroll
          for (int e = 0; e < 16 * U; ++e)
            if (e == k) p = s[e >> 4][e & 15];
          p = __shfl(p, lane_of, kWave);
          if (at > last) continue;
#pragma unroll
          for (int d = 0; d < NB; ++d) {
            const uint32_t byte = c.v_scales[place_of_it + d];
            if (byte < kFarScale) continue;
#pragma unroll
            for (int e = 0; e < 16; ++e)
              o[d][e] += p * far_value(reinterpret_cast<const uint32_t*>(c.v) + (place_of_it + d) * 4, byte, 8 * (e >> 2) + 4 * h + (e & 3));
          }
        }
      }
    }
    __syncthreads();
  }
  l += __shfl_xor(l, 32, kWave);
  ref = ref_of_seen(c, table, begin * C, end * C < keys ? end * C : keys, place, ref, l);

  // Out by way of LDS, 128 columns at a time, the wavefront's own: two rows of 32 lanes x four
  // columns an access.
  const float inv = a.splits > 1 || nothing_seen(ref, l) ? 1.f : 1.f / l;
  const int64_t base = (((b * c.heads + kvh) * a.tiles + tile) * a.splits + split) * kAttnTileRows + 32 * wave;
  if (a.splits > 1 && h == 0 && wrow0 + r < rows) a.parts_ml[2 * (base + r)] = ref, a.parts_ml[2 * (base + r) + 1] = l;
#pragma unroll
  for (int d0 = 0; d0 < NB; d0 += 4) {
    wave_lds_sync();
#pragma unroll
    for (int d = d0; d < NB && d < d0 + 4; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = o[d][4 * q + e] * inv;
        *reinterpret_cast<f32x4*>(&lds.o[wave][r][32 * (d - d0) + 8 * q + 4 * h]) = v;
      }
    wave_lds_sync();
    const int col = 32 * d0 + 4 * r;
#pragma unroll 4
    for (int k = 0; k < 16; ++k) {
      const int wr = 2 * k + h;
      const int64_t at = wrow0 + wr;
      if (at >= rows || col >= 32 * NB) continue;
      float v[4];
      load_f32<float, 4>(&lds.o[wave][wr][4 * r], v);
      if (a.splits > 1) {
        store_f32<float, 4>(a.parts_o + (base + wr) * (32 * NB) + col, v);
        continue;
      }
      const int64_t oi = at / group;
      T* y = reinterpret_cast<T*>(a.y) + b * a.y_strides[0] + (first + oi) * a.y_strides[1] +
             (kvh * group + (at - oi * group)) * a.y_strides[2] + col;
      if (col + 4 <= a.head_dim) {
        store_any_f32<T, 4>(y, v);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < a.head_dim) y[e] = from_f32<T>(v[e]);
      }
    }
  }
}

template <typename T, int NB>
int launch_tile_nb(const Mx4AttnArgs& a, hipStream_t stream) {
  constexpr int lds = (int)sizeof(TileLds<NB, tile_tokens(NB, Parts<T>::n)>);
  static_assert(lds <= kMaxLdsBytes, "LDS");
  const int rc = set_lds_limit_once<k_mx4_attn_tile<T, NB>>(lds);
  if (rc != (int)hipSuccess) return rc;
  return launch_blocks(a, &Mx4AttnArgs::block0, a.seq.batch * a.cache.heads * a.tiles * a.splits,
                       [&](const Mx4AttnArgs& part, unsigned grid) { k_mx4_attn_tile<T, NB><<<grid, kTileThreads, lds, stream>>>(part); });
}

template <typename T>
int launch_tile(const Mx4AttnArgs& a, hipStream_t stream) {
  switch (a.cache.blocks) {
    case 1: return launch_tile_nb<T, 1>(a, stream);
    case 2: return launch_tile_nb<T, 2>(a, stream);
    case 3: return launch_tile_nb<T, 3>(a, stream);
    case 4: return launch_tile_nb<T, 4>(a, stream);
    case 5: return launch_tile_nb<T, 5>(a, stream);
    case 6: return launch_tile_nb<T, 6>(a, stream);
    case 7: return launch_tile_nb<T, 7>(a, stream);
    default: return launch_tile_nb<T, 8>(a, stream);
  }
}

}  // namespace

int launch_mx4_attn_tiles(const Mx4AttnArgs& a, int dtype, hipStream_t stream) {
  return dtype == SF_F16 ? launch_tile<__half>(a, stream) : dtype == SF_BF16 ? launch_tile<__hip_bfloat16>(a, stream) : launch_tile<float>(a, stream);
}

}  // namespace sf
