// The paged cache in the microscaled 4-bit format on the device.  gfx950 only.
#pragma once

#include "sf_mx4.h"

namespace sf {
namespace {

// log2(e): scores are kept as exponents of 2.
constexpr float kLog2e = 1.44269504088896340736f;

// The page of token t, or -1.
__device__ __forceinline__ int32_t cache_page(const CacheView& c, const int32_t* __restrict__ table, int64_t t) {
  const int32_t p = table[t >> c.page_shift];
  return p >= 0 && p < c.pages ? p : -1;
}
// Where a head's row of keys or values lies: token t is row t % page of its page, and a page
// holds [heads, page] rows.  Without a page: the pool's first
// row, which is read and left out: behind loads that only some lanes make the compiler waits
// for all that are under way.
__device__ __forceinline__ int64_t cache_place(const CacheView& c, int32_t page, int head, int64_t t) {
  const int64_t at = (((int64_t)page * c.heads + head) << c.page_shift) + (t & ((1 << c.page_shift) - 1));
  return page >= 0 ? at : 0;
}

// 16 lanes point at 4 rows' 16 columns of bf16, four to a row, and lane l gets column l of
// the four rows.
__device__ __forceinline__ bf16x4v lds_transposed(const uint16_t* p) {
  typedef __attribute__((address_space(3))) bf16x4v Lds;
  return __builtin_bit_cast(bf16x4v, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((Lds*)(const_cast<uint16_t*>(p))));
}

// Columns k .. k + 7 of a query row as bf16 parts.  (Scores are taken with |scale|.)
template <typename T, int NP>
__device__ __forceinline__ void load_query(const T* __restrict__ q, int k, int head_dim, float scale, bf16x8 (&p)[NP]) {
  float v[8];
  load8<T>(q, k, head_dim, v);
  if (scale < 0.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = -v[i];
  }
  split8<NP>(v, p);
}

// V's rows in LDS as bf16: an odd number of 64-byte blocks to a row, and the 16-byte units of a
// block (32 columns) changed about by the token, so that what the transposing loads and the
// stores touch at once lies in different banks.
constexpr int value_stride(int nb) { return 32 * (nb | 1); }  // bf16 elements
__device__ __forceinline__ int value_unit(int unit, int tok) { return unit ^ (tok & 3) ^ (tok >> 1 & 2); }

// Softmax weights for the second product, in bf16 parts: three for float32, which lose nothing, and
// two for f16 and bf16, the second rounded: off by 2^-16 of a weight.  (One part, rounded, is off by
// 2^-9: as much as a bf16 result's own rounding, and a third more error against 64 bits.)
template <typename T>
constexpr int kWeightParts = Parts<T>::n == 3 ? 3 : 2;
template <int NP>
__device__ __forceinline__ void weight_parts(const float (&w)[8], bf16x8 (&p)[NP]) {
  if constexpr (NP == 2) {
    u32x4 high, low;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float rest[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        rest[k] = w[2 * i + k] - __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, w[2 * i + k]) & 0xffff0000u);
      high[i] = pack_high(w[2 * i], w[2 * i + 1]);
      low[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{rest[0], rest[1]}), bf16x2));
    }
    p[0] = __builtin_bit_cast(bf16x8, high);
    p[1] = __builtin_bit_cast(bf16x8, low);
  } else {
    split8<NP>(w, p);
  }
}

// The factor of a score that makes it an exponent of 2.  (Where scale is 0, so little that
// it is nothing: what is hidden, -infinity, has to stay that.)
__device__ __forceinline__ float score_factor(float scale) { return fmaxf(fabsf(scale) * kLog2e, 1e-44f); }

// Exponents are taken against a row's `ref`, a whole number at its running maximum or above; it moves
// only where the maximum would pass it by more than kRefSlack, so that the sums are seldom rescaled.
// Weights are at most 2^8 then, and up to 2^22 of them times values of scales below kLargeScale (less
// than 2^97) stay in float32's range.  From the first chunk on that holds a larger value the
// wavefront's refs have kRefRoom more room, and weights are 2^-22 at most: values at the end of float32
// stay in range too.  (Beside those, float32's smallest product, 2^-149, is one of 2^-119 and a weight
// of 1; with the room from the start values of 2^-118 had one bit left.)
constexpr float kRefSlack = 8.f, kRefRoom = 30.f;
constexpr uint32_t kLargeScale = 222;
__device__ __forceinline__ bool ref_passed(float top, float ref, bool roomy) {
  return __any(top > ref + (roomy ? kRefSlack - kRefRoom : kRefSlack));
}
// Of a chunk with the maximum `top`; `more`: with the room from here on.
__device__ __forceinline__ float ref_moved(float ref, float top, bool roomy, bool more) {
  return fmaxf(ref + (more ? kRefRoom : 0.f), ceilf(top) + (roomy ? kRefRoom : 0.f));
}

// A weight: with the queries in one part in one rounding of its exponent (2^-19 of it at 38); where
// they are held in more the exponent stays small, and the room is a factor.
template <int NP>
__device__ __forceinline__ float ref_from(float ref, bool roomy) {
  return ref == -INFINITY ? 0.f : NP > 1 && roomy ? ref - kRefRoom : ref;  // (a row that has seen nothing yet)
}
template <int NP>
__device__ __forceinline__ float weight_of(float score, float c2, float from, bool roomy) {
  const float w = exp2_hw(fmaf(score, c2, -from));
  return NP == 1 ? w : w * (roomy ? 0x1p-30f : 1.f);
}

// Values from scale kFarScale on are no numbers or beyond a float's range at times, and 0 times such
// a one is no 0: they lie in LDS as zeros, and each row adds those that it sees itself.  Column
// `col` of a block with its codes and scale:
constexpr uint32_t kFarScale = 253;
__device__ __forceinline__ float far_value(const uint32_t* codes, uint32_t byte, int col) {
  const f32x2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[col >> 3] >> (4 * (col & 7)) & 15, mx4_scale(byte), 0);
  return v.x;
}

// A row that sees no token is zeros; one that sees tokens whose scores are all -infinity has a
// softmax of 0 / 0.  Both have no sum and -infinity for a maximum after the tokens from `begin` to
// `end` - 1: the maximum of the latter, which any other score passes, becomes the lowest number.
__device__ __forceinline__ bool nothing_seen(float ref, float sum) { return ref == -INFINITY && sum == 0.f; }
__device__ __forceinline__ float ref_of_seen(const CacheView& c, const int32_t* __restrict__ table, int64_t begin, int64_t end,
                                             int64_t place, float ref, float sum) {
  if (!__any(nothing_seen(ref, sum) && place >= begin)) return ref;
  for (int64_t p0 = begin >> c.page_shift; p0 << c.page_shift < end; p0 += kWave) {
    const int64_t at = (p0 + lane_id()) << c.page_shift, t = at > begin ? at : begin;
    const uint64_t there = __ballot(t < end && cache_page(c, table, t < end ? t : end - 1) >= 0);
    if (there == 0) continue;
    const int64_t first = (p0 + __builtin_ctzll(there)) << c.page_shift;  // (the first page there is)
    return nothing_seen(ref, sum) && place >= begin && place >= first ? -__FLT_MAX__ : ref;
  }
  return ref;
}

// The tokens that a sequence's table has room for.
__device__ __forceinline__ int64_t cache_room(const CacheView& c) { return (int64_t)c.width << c.page_shift; }

}  // namespace
}  // namespace sf
