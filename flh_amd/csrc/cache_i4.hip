// A block of new tokens into a key / value cache held in 4 bits, and rows of one back as fp16 (the format and its arithmetic: cache_i4.h).
#include "cache_i4.h"

namespace flh {
namespace {

struct Write {
  const __half *q, *k, *v, *cos, *sin;
  const long long *lengths, *counts;                   // (counts: of padded rows; null where all T tokens count)
  __half* q_out;
  uint8_t *k_codes, *v_codes;
  __half *k_scales, *v_scales;
  uint32_t items, T, Hq, Hkv, max_len;
};

// D / 16 lanes per head vector; item order: all query heads of a token, then its key heads, then its value heads.  A lane holds both pieces
// of a rotary pair and reads them before it writes either, so q_out may be q.  Bound by the bytes: 8192 tokens of 32 / 8 heads of 128 read 105 MB and
// write 76 (queries and codes), 37.5 us = 4.8 TB/s; 21 tokens: 4 us.
template <int D>
__global__ __launch_bounds__(256) void rope_quant_kernel(Write a) {
  constexpr uint32_t kLanes = HeadRow<D>::kLanes;
  const uint32_t gl = blockIdx.x * 256u + threadIdx.x;
  const uint32_t item = gl / kLanes, chunk = HeadRow<D>::chunk_of(gl % kLanes);
  if (item >= a.items) return;
  const uint32_t heads = a.Hq + 2 * a.Hkv;
  const uint32_t token = item / heads, hh = item % heads, b = token / a.T, t = token % a.T;
  const bool is_q = hh < a.Hq, is_v = hh >= a.Hq + a.Hkv;
  const uint32_t head = is_q ? hh : is_v ? hh - a.Hq - a.Hkv : hh - a.Hq;
  const uint32_t lo = chunk * 8, hi = lo + D / 2;
  const __half* src = (is_q ? a.q + ((size_t)token * a.Hq + head) * D : (is_v ? a.v : a.k) + ((size_t)token * a.Hkv + head) * D);
  HeadRow<D> row;
  row.set(*(const h8*)(src + lo), *(const h8*)(src + hi));
  if (!is_v) {
    const __half *cs = a.cos + (size_t)token * D, *sn = a.sin + (size_t)token * D;
    row.turn(*(const h8*)(cs + lo), *(const h8*)(cs + hi), *(const h8*)(sn + lo), *(const h8*)(sn + hi));
    row.hadamard(chunk);
    row.scale(HeadRow<D>::norm());
  }
  if (is_q) {
    h8 ylo, yhi;
#pragma unroll
    for (int e = 0; e < 8; ++e) ylo[e] = (_Float16)row.v[e], yhi[e] = (_Float16)row.v[8 + e];
    __half* dst = a.q_out + ((size_t)token * a.Hq + head) * D;
    *(h8*)(dst + lo) = ylo;
    *(h8*)(dst + hi) = yhi;
    return;
  }
  const RowCodes r = quantise(row);
  const long long first = a.lengths[b];
  if (t >= tokens_of(a.counts, b, a.T, first, a.max_len)) return;
  const size_t at = ((size_t)b * a.Hkv + head) * a.max_len + (size_t)first + t;
  uint8_t* codes = (is_v ? a.v_codes : a.k_codes) + at * (D / 2);
  *(unsigned*)(codes + chunk * 4) = r.lo;
  *(unsigned*)(codes + D / 4 + chunk * 4) = r.hi;
  if (chunk == 0) ((_Float16*)(is_v ? a.v_scales : a.k_scales))[at] = r.scale;
}

struct Read {
  const uint8_t* codes[2];
  const __half* scales[2];
  const long long* first;
  __half* out[2];
  uint32_t items, rows, Hkv, max_len;
};

// y = fp16(H c s / sqrt(D)) for keys, fp16(c s) for values: sums of codes are whole numbers and their product with the scale has 22 bits.  Bound by the
// bytes: 4 x 1875 slots of 32 heads of 128: 155 MB in 27.4 us, 5.6 TB/s (more than a 2 GiB copy's 4.9: it fits the last-level cache, as a copy of 77 MiB
// does, which runs at 7.0); 900 slots of 8 heads: 3.7 us.
template <int D>
__global__ __launch_bounds__(256) void dequant_kernel(Read a) {
  constexpr uint32_t kLanes = HeadRow<D>::kLanes;
  const uint32_t gl = blockIdx.x * 256u + threadIdx.x;
  const uint32_t item = gl / kLanes, chunk = HeadRow<D>::chunk_of(gl % kLanes);
  if (item >= a.items) return;
  const bool keys = blockIdx.y == 0;
  const uint32_t bh = item / a.rows, i = item % a.rows;
  const long long first = a.first[bh / a.Hkv];
  // (a start far outside must not wrap into the range)
  const bool in = first > -(1ll << 40) && first < (1ll << 40) && first + i >= 0 && first + i < (long long)a.max_len;
  unsigned lo = 0, hi = 0;
  float s = 0.f;
  if (in) {
    const size_t at = (size_t)bh * a.max_len + (size_t)(first + i);
    const uint8_t* codes = a.codes[blockIdx.y] + at * (D / 2);
    lo = *(const unsigned*)(codes + chunk * 4);
    hi = *(const unsigned*)(codes + D / 4 + chunk * 4);
    s = (float)((const _Float16*)a.scales[blockIdx.y])[at];
  }
  HeadRow<D> row;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    row.v[e] = (float)((int)(lo << (28 - 4 * e)) >> 28);
    row.v[8 + e] = (float)((int)(hi << (28 - 4 * e)) >> 28);
  }
  if (keys) row.hadamard(chunk);
  row.scale(s);
  if (keys) row.scale(HeadRow<D>::norm());
  h8 ylo, yhi;
#pragma unroll
  for (int e = 0; e < 8; ++e) ylo[e] = (_Float16)row.v[e], yhi[e] = (_Float16)row.v[8 + e];
  __half* dst = a.out[blockIdx.y] + (size_t)item * D;
  *(h8*)(dst + chunk * 8) = ylo;
  *(h8*)(dst + D / 2 + chunk * 8) = yhi;
}

}  // namespace
}  // namespace flh

using namespace flh;

extern "C" int flh_rope_quant_kv_cache_i4(const flh_half* q, const flh_half* k, const flh_half* v, const flh_half* cos, const flh_half* sin,
                                          const int64_t* lengths, flh_half* q_out, uint8_t* k_codes, flh_half* k_scales, uint8_t* v_codes,
                                          flh_half* v_scales, uint32_t B, uint32_t T, uint32_t Hq, uint32_t Hkv, uint32_t head_dim,
                                          uint32_t max_len, void* stream) {
  return flh_rope_quant_kv_cache_i4_counts(q, k, v, cos, sin, lengths, nullptr, q_out, k_codes, k_scales, v_codes, v_scales, B, T, Hq, Hkv, head_dim,
                                           max_len, stream);
}

extern "C" int flh_rope_quant_kv_cache_i4_counts(const flh_half* q, const flh_half* k, const flh_half* v, const flh_half* cos, const flh_half* sin,
                                                 const int64_t* lengths, const int64_t* counts, flh_half* q_out, uint8_t* k_codes,
                                                 flh_half* k_scales, uint8_t* v_codes, flh_half* v_scales, uint32_t B, uint32_t T, uint32_t Hq,
                                                 uint32_t Hkv, uint32_t head_dim, uint32_t max_len, void* stream) {
  const char* what = "rope_quant_kv_cache";
  if (!q || !k || !v || !cos || !sin || !lengths || !q_out || !k_codes || !k_scales || !v_codes || !v_scales)
    return fail(FLH_EINVAL, "%s: null pointer", what);
  if (misaligned16(q, k, v, cos, sin, q_out, k_codes, v_codes)) return fail(FLH_EINVAL, "%s: tensors must be 16-byte aligned", what);
  if (head_dim != 128 && head_dim != 64) return fail(FLH_EINVAL, "%s: head_dim (%u) must be 64 or 128", what, head_dim);
  if (Hq == 0 || Hkv == 0 || max_len == 0) return fail(FLH_EINVAL, "%s: heads and cache length must be positive", what);
  if (B == 0 || T == 0) return FLH_OK;
  const uint64_t tokens = (uint64_t)B * T, heads = (uint64_t)Hq + 2ull * Hkv;
  if (tokens > 0xFFFFFFFFull || heads > 0xFFFFFFull || tokens * heads > 0xFFFFFF00ull / (head_dim / 16) || (uint64_t)B * Hkv > 0xFFFFFFFFull)
    return fail(FLH_EINVAL, "%s: too many elements for one launch", what);
  const uint64_t slots = (uint64_t)B * Hkv * max_len, queries = tokens * Hq * head_dim * 2, rows = tokens * Hkv * head_dim * 2;
  if (slots > 1ull << 40) return fail(FLH_EINVAL, "%s: problem too large", what);
  const struct { const void* at; uint64_t bytes; } out[5] = {{k_codes, slots * (head_dim / 2)}, {k_scales, slots * 2}, {v_codes, slots * (head_dim / 2)},
                                                             {v_scales, slots * 2}, {q_out, queries}},
      in[7] = {{k, rows}, {v, rows}, {cos, tokens * head_dim * 2}, {sin, tokens * head_dim * 2}, {lengths, (uint64_t)B * 8}, {q, queries},
               {counts, counts ? (uint64_t)B * 8 : 0}};
  for (int i = 0; i < 5; ++i) {
    for (int j = 0; j < i; ++j)
      if (overlap(out[i].at, out[i].bytes, out[j].at, out[j].bytes)) return fail(FLH_EINVAL, "%s: two outputs share memory", what);
    for (const auto& x : in)
      if (overlap(out[i].at, out[i].bytes, x.at, x.bytes) && !(i == 4 && out[i].at == x.at && x.at == (const void*)q))
        return fail(FLH_EINVAL, "%s: an output shares memory with an input", what);
  }
  Write a = {(const __half*)q, (const __half*)k, (const __half*)v, (const __half*)cos, (const __half*)sin, (const long long*)lengths, (const long long*)counts,
             (__half*)q_out, k_codes, v_codes, (__half*)k_scales, (__half*)v_scales, (uint32_t)(tokens * heads), T, Hq, Hkv, max_len};
  const unsigned groups = (unsigned)((tokens * heads * (head_dim / 16) + 255) / 256);
  if (head_dim == 128) hipLaunchKernelGGL(rope_quant_kernel<128>, dim3(groups), dim3(256), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL(rope_quant_kernel<64>, dim3(groups), dim3(256), 0, (hipStream_t)stream, a);
  return check_launch(what);
}

extern "C" int flh_dequant_kv_cache_i4(const uint8_t* k_codes, const flh_half* k_scales, const uint8_t* v_codes, const flh_half* v_scales,
                                       const int64_t* first, flh_half* keys, flh_half* values, uint32_t B, uint32_t rows, uint32_t Hkv,
                                       uint32_t head_dim, uint32_t max_len, void* stream) {
  const char* what = "dequant_kv_cache";
  if (!k_codes || !k_scales || !v_codes || !v_scales || !first || !keys || !values) return fail(FLH_EINVAL, "%s: null pointer", what);
  if (misaligned16(k_codes, v_codes, keys, values)) return fail(FLH_EINVAL, "%s: tensors must be 16-byte aligned", what);
  if (head_dim != 128 && head_dim != 64) return fail(FLH_EINVAL, "%s: head_dim (%u) must be 64 or 128", what, head_dim);
  if (Hkv == 0 || max_len == 0) return fail(FLH_EINVAL, "%s: heads and cache length must be positive", what);
  if (B == 0 || rows == 0) return FLH_OK;
  const uint64_t heads = (uint64_t)B * Hkv;
  if (heads > 0xFFFFFFFFull || heads * rows > 0xFFFFFF00ull / (head_dim / 16)) return fail(FLH_EINVAL, "%s: too many elements for one launch", what);
  const uint64_t slots = heads * max_len, bytes = heads * rows * head_dim * 2;
  if (slots > 1ull << 40) return fail(FLH_EINVAL, "%s: problem too large", what);
  if (overlap(keys, bytes, values, bytes)) return fail(FLH_EINVAL, "%s: two outputs share memory", what);
  const struct { const void* at; uint64_t bytes; } in[5] = {{k_codes, slots * (head_dim / 2)}, {k_scales, slots * 2}, {v_codes, slots * (head_dim / 2)},
                                                            {v_scales, slots * 2}, {first, (uint64_t)B * 8}};
  for (const auto& x : in)
    if (overlap(keys, bytes, x.at, x.bytes) || overlap(values, bytes, x.at, x.bytes))
      return fail(FLH_EINVAL, "%s: an output shares memory with an input", what);
  Read a = {{k_codes, v_codes}, {(const __half*)k_scales, (const __half*)v_scales}, (const long long*)first, {(__half*)keys, (__half*)values},
            (uint32_t)(heads * rows), rows, Hkv, max_len};
  const dim3 grid((unsigned)((heads * rows * (head_dim / 16) + 255) / 256), 2);
  if (head_dim == 128) hipLaunchKernelGGL(dequant_kernel<128>, grid, dim3(256), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL(dequant_kernel<64>, grid, dim3(256), 0, (hipStream_t)stream, a);
  return check_launch(what);
}
