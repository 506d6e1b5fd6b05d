// Rows of a key / value cache held in 4 bits, shared by the kernels that write, read and attend over one.
//
// A layer's cache: codes [B, Hkv, max_len, D / 2] (two's-complement nibbles, element 2 j in the low half of byte j) and one fp16 scale per row
// [B, Hkv, max_len], for keys and for values.  A key is held as it is after the rotary embedding and the orthonormal Hadamard rotation of its
// head (queries are rotated alike, which leaves q . k as it is and spreads channels that stick out over all of them).
//
//   r = x cos + rotate_half(x) sin,  y = H r / sqrt(D)      float32, butterflies over strides 1, 2, 4, ..., then the factor
//   s = fp16(max |y| / 7) (0: 1),  c = clamp(rint(y / s), -8, 7)
//
// with one IEEE operation per step of float32 arithmetic, so the codes are those of the same expression anywhere else.  A row that is not
// finite, or whose scale is not, has the scale NaN and codes of zero: queries that see it get NaN, the others nothing of it.
#pragma once
#include "group_codes.h"

namespace flh {
namespace {

// One head vector of D channels in D / 16 adjacent lanes: the lane of chunk c holds channels 8 c .. 8 c + 7 in v[0 .. 7] and D / 2 + 8 c .. in
// v[8 .. 15], each one's rotary partner beside it.
template <int D>
struct HeadRow {
  static_assert(D == 128 || D == 64, "head dimension");
  static constexpr int kLanes = D / 16;
  float v[16];

  __device__ __forceinline__ static int chunk_of(int pos) { return group_chunk<kLanes>(pos); }

  __device__ __forceinline__ void set(h8 lo, h8 hi) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)lo[e], v[8 + e] = (float)hi[e];
  }
  // (products of two fp16 values are exact: the sum is the only rounding, fused or not)
  __device__ __forceinline__ void turn(h8 cl, h8 ch, h8 sl, h8 sh) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = v[e], b = v[8 + e];
      v[e] = __builtin_fmaf(a, (float)cl[e], -(b * (float)sl[e]));
      v[8 + e] = __builtin_fmaf(b, (float)ch[e], a * (float)sh[e]);
    }
  }
  template <int CTRL>
  __device__ __forceinline__ void across(bool upper) {
    const int sign = upper ? (int)0x80000000 : 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float o = dpp_f<CTRL>(v[e]);
      v[e] = o + __int_as_float(__float_as_int(v[e]) ^ sign);
    }
  }
  // the rows' unnormalised Hadamard transform
  __device__ __forceinline__ void hadamard(int chunk) {
#pragma unroll
    for (int s = 1; s < 8; s *= 2)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (!(e & s)) {
          const float a = v[e], b = v[e + s];
          v[e] = a + b, v[e + s] = a - b;
        }
    across<kDppQuadXor1>(chunk & 1);
    across<kDppQuadXor2>(chunk & 2);
    if constexpr (kLanes == 8) across<kDppRowHalfMirror>(chunk & 4);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = v[e], b = v[8 + e];
      v[e] = a + b, v[8 + e] = a - b;
    }
  }
  __device__ __forceinline__ static constexpr float norm() { return D == 128 ? 0.08838834764831845f : 0.125f; }   // 1 / sqrt(D)
  __device__ __forceinline__ void scale(float f) {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = round_here(v[e] * f);
  }
  // bit pattern of the row's largest |value|, in which infinities and NaN come last
  __device__ __forceinline__ unsigned top() const {
    unsigned m = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) m = max(m, (unsigned)__float_as_int(v[e]) & 0x7FFFFFFFu);
    m = max(m, (unsigned)dpp_i<kDppQuadXor1>((int)m));
    m = max(m, (unsigned)dpp_i<kDppQuadXor2>((int)m));
    if constexpr (kLanes == 8) m = max(m, (unsigned)dpp_i<kDppRowHalfMirror>((int)m));
    return m;
  }
};

struct RowCodes {
  unsigned lo, hi;   // of v[0 .. 7] and v[8 .. 15]
  _Float16 scale;
};

template <int D>
__device__ __forceinline__ RowCodes quantise(const HeadRow<D>& row) {
  const unsigned m = row.top();
  RowCodes r;
  r.scale = (_Float16)round_here(__int_as_float((int)m) * (1.0f / 7.0f));
  if (r.scale == (_Float16)0.0f) r.scale = (_Float16)1.0f;
  const bool finite = m < 0x7F800000u && (float)r.scale < INFINITY;
  if (!finite) r.scale = __builtin_bit_cast(_Float16, (unsigned short)0x7E00);
  const float s = (float)r.scale, inv = __builtin_amdgcn_rcpf(s);
  // the quotient by the reciprocal is off by less than 1e-5 (it is 10.6 at most, for a scale that is subnormal): only next to a border
  // does the code need the division itself, and rows whose values are fp16 meet borders exactly
  float c[16];
  bool near = false;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float t = row.v[e] * inv;
    c[e] = __builtin_rintf(t);
    near |= __builtin_fabsf(t - c[e]) > 0.49995f;
  }
  if (__builtin_amdgcn_ballot_w64(near) != 0) {
#pragma unroll
    for (int e = 0; e < 16; ++e) c[e] = __builtin_rintf(row.v[e] / s);
  }
  r.lo = r.hi = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int a = (int)__builtin_fminf(__builtin_fmaxf(c[e], -8.f), 7.f), b = (int)__builtin_fminf(__builtin_fmaxf(c[8 + e], -8.f), 7.f);
    r.lo |= (unsigned)(a & 15) << (4 * e), r.hi |= (unsigned)(b & 15) << (4 * e);
  }
  if (!finite) r.lo = r.hi = 0;
  return r;
}

// Eight codes as an operand of the fp16 matrix instructions, without a conversion: code + 8 in bits 4 .. 7 of a half is the subnormal
// (code + 8) 2^-20, which they multiply exactly; what the 8 adds, eight times the sum of the other operand, is taken off in float32.  Elements are
// codes 0, 4 | 1, 5 | 2, 6 | 3, 7.  (Bits 0 .. 3 take two shifts less.  But products are lined up by the exponents of their operands, which for
// a subnormal is that of 2^-14 whatever its bits: the sums lost the last ten bits of 24, in bits 4 .. 7 six.)
constexpr unsigned kNibbles = 0x00F000F0u, kEight = 0x00800080u;
__device__ __forceinline__ h8 code_halves(unsigned w) {
  const v4i r = {(int)(((w << 4) & kNibbles) ^ kEight), (int)((w & kNibbles) ^ kEight), (int)(((w >> 4) & kNibbles) ^ kEight),
                 (int)(((w >> 8) & kNibbles) ^ kEight)};
  return __builtin_bit_cast(h8, r);
}
// the place of code e of eight among the elements of an operand
__device__ __forceinline__ constexpr int code_element(int e) { return 2 * (e & 3) + (e >> 2); }

constexpr float kFromSubnormal = 1048576.0f;           // 2^20
// What the 8 adds to an output's sums grows with the number of keys, a sum of signed codes with its root: every so many of its tiles a wave takes it
// off its accumulators, so that their rounding does not grow with the length (keys of nearly one weight, heads of 128, one wave: 16000 off by 3.6e-4
// of the result, 60000 by 6.6e-4, 250000 by 2.4e-3 when it was taken off at the end alone; 3.0e-4 at any of them now, what the weights' and the result's
// own roundings come to, for 1 % of a prompt's time: 4096 tokens 195 -> 197 us).
constexpr int kTakeOff = 16;
constexpr float kLowestRef = -1e30f;                   // reference of a query that has seen nothing: finite, far below every score
constexpr int kTileKeys = 64;

// the fp16 value in the low half of a dword (a mixed-precision multiply-add takes it as it is; left to the compiler, which knows what has to lie
// between a matrix instruction, or an exponential, and the use of its result)
__device__ __forceinline__ float low_half(unsigned v) { return (float)__builtin_bit_cast(_Float16, (unsigned short)v); }
// {fp16(a * x), fp16(b * y)} of fp16 x, y in the low halves
__device__ __forceinline__ h2 pair_times_halves(float a, unsigned x, float b, unsigned y) {
  return h2{(_Float16)__builtin_fmaf(a, low_half(x), 0.0f), (_Float16)__builtin_fmaf(b, low_half(y), 0.0f)};
}

// The reference of a softmax whose largest weight, in powers of two, is `top` (a score's plus its value's scale's exponent, 25 for a factor of 2^10):
// weights stay below 2^12.  A weight's exponent is one multiply-add, score x factor - reference, and so sees the reference's own rounding: it is
// put more than that below the largest (2^-22 of it, less than 1 for scores below 2^22), and where the weights of a tile leave fp16's range all the
// same they are bounded: scores of 10^8 and more, where what lies within their rounding weighs the same.
__device__ __forceinline__ float reference_for(float top) {
  const float r = top - 25.0f;
  return r * (r > 0.f ? 1.0f - 0x1p-22f : 1.0f + 0x1p-22f);
}
__device__ __forceinline__ float exponent_of(unsigned half) { return (float)((half >> 10) & 31u); }
__device__ __forceinline__ float bounded(float x, unsigned half) {
  const float most = 26.0f - exponent_of(half);
  return x > most ? most : x;                          // (NaN stays)
}

// Loads that go straight to LDS, lane i's 16 (4) bytes to lds_base + 16 i (4 i); beyond the descriptor's range they bring zeros
__device__ __forceinline__ void rows_to_lds(const v4i& d, unsigned voff, unsigned lds_base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds_base), "v"(voff), "s"(d) : "memory", "m0");
}
__device__ __forceinline__ void halves_to_lds(const v4i& d, unsigned voff, unsigned lds_base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_ushort %1, %2, 0 offen lds" ::"s"(lds_base), "v"(voff), "s"(d) : "memory", "m0");
}

// Tokens of a block of T that sequence b takes, all or counts[b] of them, in the slots from its length on: none where they do not fit the cache, or
// the length or the count is out of range
__device__ __forceinline__ uint32_t tokens_of(const long long* counts, uint32_t b, uint32_t T, long long length, uint32_t max_len) {
  const long long n = counts ? counts[b] : (long long)T;
  return n < 0 || n > (long long)T || length < 0 || length > (long long)max_len - n ? 0u : (uint32_t)n;
}

// what is made of it here is not made in front of the branch that it is needed behind
__device__ __forceinline__ int opaque(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// every LDS operation of this wave has completed, and no memory operation crosses
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

typedef __attribute__((address_space(3))) v2i lds_v2i;
typedef unsigned short __attribute__((may_alias)) packed_u16;   // a half among dwords

}  // namespace

inline bool bad_scale(float scale) { return !(scale > 0.f) || scale > 1e15f; }

}  // namespace flh
