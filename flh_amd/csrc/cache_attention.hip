// Attention over a key / value cache whose sequences have lengths of their own, read on the device:
//
//   tree attention     T drafted tokens per sequence, rotated and written into the slots lengths[b] .. lengths[b] + T - 1; a token
//                      sees the lengths[b] slots before them and those of the tree that its row of the mask names
//   attention weights  attention (one token per sequence over lengths[b] slots, or the causal one of a prompt) that also adds every
//                      slot's probabilities, summed over the queries of its key / value head, to a running float32 sum
//
//   out[r] = sum_j p[r, j] V[j],  p[r, j] = exp(s[r, j] - m[r]) / l[r],  s = scale q[r] . K[j],  m = max_j s,  l = sum_j exp(s - m)
//   weights[j] += sum_r p[r, j]
//
// A wave per query: 64 keys at a time, a lane scores one of them, then holds two channels of the output.
#include "lane_ops.h"

namespace flh {

// prefill_attention.hip
int prefill_attention(const __half* q, const __half* k_cache, const __half* v_cache, __half* out, float* stats, uint32_t B, uint32_t T,
                      uint32_t Hq, uint32_t Hkv, uint32_t head_dim, uint32_t past, uint32_t max_len, float scale, hipStream_t stream);

namespace {

// The drafted keys (rotated in float32, rounded once) and values into their slots: one lane per pair of channels d / 2 apart.
__global__ __launch_bounds__(256) void tree_write_kernel(const __half* __restrict__ k, const __half* __restrict__ v,
                                                         const __half* __restrict__ cos, const __half* __restrict__ sin,
                                                         const long long* __restrict__ lengths, __half* __restrict__ k_cache,
                                                         __half* __restrict__ v_cache, uint32_t B, uint32_t T, uint32_t Hkv, uint32_t d,
                                                         uint32_t max_len) {
  const uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint32_t half = d / 2, c = (uint32_t)(at % half);
  const uint64_t item = at / half;                     // (b, t, head)
  if (item >= (uint64_t)B * T * Hkv) return;
  const uint32_t head = (uint32_t)(item % Hkv), token = (uint32_t)(item / Hkv), b = token / T, t = token % T;
  const long long n = lengths[b];
  if (n < 0 || n + T > max_len) return;
  const _Float16 *kn = (const _Float16*)k + item * d, *vn = (const _Float16*)v + item * d;
  const _Float16 *cf = (const _Float16*)cos + (size_t)token * d, *sf = (const _Float16*)sin + (size_t)token * d;
  const size_t to = (((size_t)b * Hkv + head) * max_len + (size_t)n + t) * d;
  const float x0 = kn[c], x1 = kn[c + half];
  ((_Float16*)k_cache)[to + c] = (_Float16)round_here(x0 * (float)cf[c] - x1 * (float)sf[c]);
  ((_Float16*)k_cache)[to + c + half] = (_Float16)round_here(x1 * (float)cf[c + half] + x0 * (float)sf[c + half]);
  ((_Float16*)v_cache)[to + c] = vn[c];
  ((_Float16*)v_cache)[to + c + half] = vn[c + half];
}

// what a query sees: the slots below `before`, and of the T behind them those that its row of the mask (if there is one) names
struct Seen {
  const uint8_t* mask;
  uint32_t before, T;
  __device__ bool operator()(uint32_t j) const { return j < before || (mask && j - before < T && mask[j - before]); }
};

template <int D>
__device__ __forceinline__ float score(const float* q, const __half* key, float scale) {
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < D; c += 8) {
    const h8 x = *(const h8*)(key + c);
#pragma unroll
    for (int e = 0; e < 8; ++e) s = __builtin_fmaf(q[c + e], (float)x[e], s);
  }
  return s * scale;
}

// One wave per query (b, t, h).  With cos / sin the query is rotated first.  stats (may be null): [B, Hq, T] log2 of
// the sum of exponentials.
template <int D>
__global__ __launch_bounds__(64) void query_attention_kernel(const __half* __restrict__ q, const __half* __restrict__ cos,
                                                             const __half* __restrict__ sin, const __half* __restrict__ k_cache,
                                                             const __half* __restrict__ v_cache, const long long* __restrict__ lengths,
                                                             const uint8_t* __restrict__ mask, uint32_t mask_stride, __half* __restrict__ out,
                                                             float* __restrict__ stats, uint32_t T, uint32_t Hq, uint32_t Hkv,
                                                             uint32_t max_len, float scale) {
  __shared__ float qs[D], ps[64];
  const int lane = threadIdx.x;
  const uint32_t item = blockIdx.x, h = item % Hq, token = item / Hq, b = token / T, t = token % T;
  const _Float16* row = (const _Float16*)q + (size_t)item * D;
  for (int c = lane; c < D; c += 64) {
    float x = row[c];
    if (cos) {
      const float other = row[c ^ (D / 2)];
      const float cf = ((const _Float16*)cos)[(size_t)token * D + c], sf = ((const _Float16*)sin)[(size_t)token * D + c];
      x = c < D / 2 ? x * cf - other * sf : x * cf + other * sf;
    }
    qs[c] = x;
  }
  __syncthreads();
  // the length: of the cache in front of a tree, or all of it
  uint32_t n = 0, end = 0;
  if (const long long all = lengths[b]; all >= 0 && all + (mask ? T : 0) <= max_len) n = (uint32_t)all, end = n + (mask ? T : 0);
  const Seen seen{mask ? mask + (size_t)b * mask_stride + (size_t)t * T : nullptr, n, mask && end ? T : 0};
  const size_t base = ((size_t)b * Hkv + h / (Hq / Hkv)) * max_len * D;
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (uint32_t j0 = 0; j0 < end; j0 += 64) {
    const uint32_t j = j0 + lane;
    const float s = j < end && seen(j) ? score<D>(qs, k_cache + base + (size_t)j * D, scale) : -INFINITY;
    const float m_new = fmaxf(m, wave_max(s));
    const float safe = m_new == -INFINITY ? 0.f : m_new;
    const float p = __expf(s - safe), keep = __expf(m - safe);
    l = l * keep + wave_sum(p);
    o0 *= keep, o1 *= keep;
    m = m_new;
    ps[lane] = p;
    __syncthreads();
    for (uint32_t i = 0; i < 64 && j0 + i < end; ++i) {
      const float w = ps[i];
      if (w == 0.f) continue;                          // (what a query does not see adds nothing, whatever it holds)
      const _Float16* v = (const _Float16*)v_cache + base + (size_t)(j0 + i) * D;
      o0 = __builtin_fmaf(w, (float)v[lane], o0);
      if constexpr (D == 128) o1 = __builtin_fmaf(w, (float)v[lane + 64], o1);
    }
    __syncthreads();
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  _Float16* to = (_Float16*)out + (size_t)item * D;
  to[lane] = (_Float16)(o0 * inv);
  if constexpr (D == 128) to[lane + 64] = (_Float16)(o1 * inv);
  if (stats && lane == 0) stats[((size_t)b * Hq + h) * T + t] = m * 1.4426950408889634f + __builtin_amdgcn_logf(l);
}

// weights[b, g, j] += the probabilities of slot j over all queries of key / value head g: one lane per slot
template <int D>
__global__ __launch_bounds__(64) void slot_weights_kernel(const __half* __restrict__ q, const __half* __restrict__ k_cache,
                                                          const long long* __restrict__ lengths, const float* __restrict__ stats,
                                                          float* __restrict__ weights, uint32_t T, uint32_t Hq, uint32_t Hkv, uint32_t past,
                                                          uint32_t max_len, uint32_t blocks, float scale) {
  __shared__ float qs[D];
  const uint32_t bg = blockIdx.x / blocks, b = bg / Hkv, g = bg % Hkv, rep = Hq / Hkv;
  const uint32_t j = blockIdx.x % blocks * 64 + threadIdx.x;
  const long long n = lengths ? lengths[b] : (long long)past + T;
  if (n <= 0 || n > max_len || blockIdx.x % blocks * 64 >= n) return;
  const __half* key = k_cache + ((size_t)bg * max_len + min(j, max_len - 1)) * D;
  float sum = 0.f, part = 0.f;                         // (in two levels: thousands of small terms one by one lose digits)
  for (uint32_t t = 0; t < T; ++t) {
    if (t % 32 == 0) sum += part, part = 0.f;
    for (uint32_t r = 0; r < rep; ++r) {
      const size_t item = ((size_t)b * T + t) * Hq + g * rep + r;
      __syncthreads();
      for (int c = threadIdx.x; c < D; c += 64) qs[c] = (float)((const _Float16*)q)[item * D + c];
      __syncthreads();
      if (lengths ? j < n : j <= past + t) {
        part += __builtin_amdgcn_exp2f(score<D>(qs, key, scale * 1.4426950408889634f) - stats[((size_t)b * Hq + g * rep + r) * T + t]);
      }
    }
  }
  if (j < n) weights[(size_t)bg * max_len + j] += sum + part;
}

int check_heads(const char* what, uint32_t Hq, uint32_t Hkv, uint32_t head_dim, float scale) {
  if (head_dim != 128 && head_dim != 64) return fail(FLH_EINVAL, "%s: head_dim (%u) must be 64 or 128", what, head_dim);
  if (Hq == 0 || Hkv == 0 || Hq % Hkv) return fail(FLH_EINVAL, "%s: %u query heads do not divide over %u key / value heads", what, Hq, Hkv);
  if (!(scale > 0.f) || scale > 1e30f) return fail(FLH_EINVAL, "%s: the scale must be positive and finite", what);
  return FLH_OK;
}

}  // namespace
}  // namespace flh

using namespace flh;

constexpr uint32_t kMaxNodes = 256;

extern "C" size_t flh_tree_attention_workspace_bytes(uint32_t B, uint32_t T, uint32_t Hq, uint32_t Hkv, uint32_t head_dim) {
  return 16;
}

extern "C" int flh_tree_attention_f16(const flh_half* q, const flh_half* k_new, const flh_half* v_new, const flh_half* cos,
                                      const flh_half* sin, const int64_t* lengths, const uint8_t* mask, int mask_per_sequence,
                                      flh_half* k_cache, flh_half* v_cache, flh_half* out, uint32_t B, uint32_t T, uint32_t Hq,
                                      uint32_t Hkv, uint32_t head_dim, uint32_t max_len, float scale, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  if (!q || !k_new || !v_new || !cos || !sin || !lengths || !mask || !k_cache || !v_cache || !out)
    return fail(FLH_EINVAL, "tree_attention: null pointer");
  if (misaligned16(q, k_new, v_new, cos, sin, k_cache, v_cache, out)) return fail(FLH_EINVAL, "tree_attention: tensors must be 16-byte aligned");
  if (int rc = check_heads("tree_attention", Hq, Hkv, head_dim, scale)) return rc;
  if (T > kMaxNodes) return fail(FLH_EINVAL, "tree_attention: %u nodes (at most %u)", T, kMaxNodes);
  if (B == 0 || T == 0) return FLH_OK;
  const size_t need = flh_tree_attention_workspace_bytes(B, T, Hq, Hkv, head_dim);
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)
    return fail(FLH_EINVAL, "tree_attention: a 16-byte aligned workspace of %zu bytes is required", need);
  if ((uint64_t)B * T * Hq * head_dim > 0x7FFFFFFFull || (uint64_t)B * Hkv * max_len * head_dim > (1ull << 40) || max_len > (1u << 30))
    return fail(FLH_EINVAL, "tree_attention: problem too large");
  const hipStream_t st = (hipStream_t)stream;
  const uint64_t lanes = (uint64_t)B * T * Hkv * (head_dim / 2);
  hipLaunchKernelGGL(tree_write_kernel, dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, st, (const __half*)k_new, (const __half*)v_new,
                     (const __half*)cos, (const __half*)sin, (const long long*)lengths, (__half*)k_cache, (__half*)v_cache, B, T, Hkv,
                     head_dim, max_len);
  if (int rc = check_launch("tree_attention (write)")) return rc;
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3(B * T * Hq), dim3(64), 0, st, (const __half*)q, (const __half*)cos, (const __half*)sin, (const __half*)k_cache,
                       (const __half*)v_cache, (const long long*)lengths, mask, mask_per_sequence ? T * T : 0u, (__half*)out, (float*)nullptr,
                       T, Hq, Hkv, max_len, scale);
  };
  if (head_dim == 128) go(query_attention_kernel<128>);
  else go(query_attention_kernel<64>);
  return check_launch("tree_attention");
}

extern "C" size_t flh_decode_attention_weights_workspace_bytes(uint32_t B, uint32_t Hq, uint32_t Hkv, uint32_t head_dim, uint32_t max_len) {
  return (size_t)B * Hq * 4 + 16;
}

extern "C" size_t flh_prefill_attention_weights_workspace_bytes(uint32_t B, uint32_t T, uint32_t Hq) { return (size_t)B * T * Hq * 4 + 16; }

namespace {
template <int D>
int launch_weights(const __half* q, const __half* k, const __half* v, const long long* lengths, __half* out, float* weights, uint32_t B,
                   uint32_t T, uint32_t Hq, uint32_t Hkv, uint32_t past, uint32_t max_len, float scale, void* ws, hipStream_t st) {
  if (lengths) {
    hipLaunchKernelGGL(query_attention_kernel<D>, dim3(B * T * Hq), dim3(64), 0, st, q, (const __half*)nullptr, (const __half*)nullptr, k, v,
                       lengths, (const uint8_t*)nullptr, 0u, out, (float*)ws, T, Hq, Hkv, max_len, scale);
    if (int rc = check_launch("attention_weights")) return rc;
  } else if (int rc = prefill_attention(q, k, v, out, (float*)ws, B, T, Hq, Hkv, D, past, max_len, scale, st)) {
    return rc;
  }
  const uint32_t blocks = (max_len + 63) / 64;
  hipLaunchKernelGGL(slot_weights_kernel<D>, dim3(B * Hkv * blocks), dim3(64), 0, st, q, k, lengths, (const float*)ws, weights, T, Hq, Hkv, past,
                     max_len, blocks, scale);
  return check_launch("attention_weights (sums)");
}
}  // namespace

extern "C" int flh_decode_attention_weights_f16(const flh_half* q, const flh_half* k_cache, const flh_half* v_cache, const int64_t* lengths,
                                                flh_half* out, float* weights, uint32_t B, uint32_t Hq, uint32_t Hkv, uint32_t head_dim,
                                                uint32_t max_len, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !k_cache || !v_cache || !lengths || !out || !weights) return fail(FLH_EINVAL, "decode_attention_weights: null pointer");
  if (misaligned16(q, k_cache, v_cache, out, weights)) return fail(FLH_EINVAL, "decode_attention_weights: tensors must be 16-byte aligned");
  if (int rc = check_heads("decode_attention_weights", Hq, Hkv, head_dim, scale)) return rc;
  if (B == 0 || max_len == 0) return FLH_OK;
  if ((uint64_t)B * Hq * head_dim > 0x7FFFFFFFull || (uint64_t)B * Hkv * ((max_len + 63) / 64) > 0x7FFFFFFFull || max_len > (1u << 30))
    return fail(FLH_EINVAL, "decode_attention_weights: problem too large");
  const size_t need = flh_decode_attention_weights_workspace_bytes(B, Hq, Hkv, head_dim, max_len);
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)
    return fail(FLH_EINVAL, "decode_attention_weights: a 16-byte aligned workspace of %zu bytes is required", need);
  auto go = [&](auto d) {
    return launch_weights<decltype(d)::value>((const __half*)q, (const __half*)k_cache, (const __half*)v_cache, (const long long*)lengths,
                                              (__half*)out, weights, B, 1, Hq, Hkv, 0, max_len, scale, workspace, (hipStream_t)stream);
  };
  return head_dim == 128 ? go(std::integral_constant<int, 128>{}) : go(std::integral_constant<int, 64>{});
}

extern "C" int flh_prefill_attention_weights_f16(const flh_half* q, const flh_half* k_cache, const flh_half* v_cache, flh_half* out,
                                                 float* weights, uint32_t B, uint32_t T, uint32_t Hq, uint32_t Hkv, uint32_t head_dim,
                                                 uint32_t past, uint32_t max_len, float scale, void* workspace, size_t workspace_bytes,
                                                 void* stream) {
  if (!q || !k_cache || !v_cache || !out || !weights) return fail(FLH_EINVAL, "prefill_attention_weights: null pointer");
  if (misaligned16(q, k_cache, v_cache, out, weights)) return fail(FLH_EINVAL, "prefill_attention_weights: tensors must be 16-byte aligned");
  if (int rc = check_heads("prefill_attention_weights", Hq, Hkv, head_dim, scale)) return rc;
  if (head_dim != 128) return fail(FLH_EINVAL, "prefill_attention_weights: head_dim (%u) must be 128", head_dim);
  if ((uint64_t)past + T > max_len) return fail(FLH_EINVAL, "prefill_attention_weights: past (%u) + T (%u) exceeds the cache length %u", past, T, max_len);
  if (B == 0 || T == 0) return FLH_OK;
  if ((uint64_t)B * T * Hq > 0x7FFFFFFFull || (uint64_t)B * Hkv * ((max_len + 63) / 64) > 0x7FFFFFFFull || max_len > (1u << 30))
    return fail(FLH_EINVAL, "prefill_attention_weights: problem too large");
  const size_t need = flh_prefill_attention_weights_workspace_bytes(B, T, Hq);
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)
    return fail(FLH_EINVAL, "prefill_attention_weights: a 16-byte aligned workspace of %zu bytes is required", need);
  return launch_weights<128>((const __half*)q, (const __half*)k_cache, (const __half*)v_cache, nullptr, (__half*)out, weights, B, T, Hq, Hkv, past,
                             max_len, scale, workspace, (hipStream_t)stream);
}
