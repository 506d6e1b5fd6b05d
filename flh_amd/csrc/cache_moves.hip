// Rows of a key / value cache moved inside it, in every layer's caches at once:
//
//   tree commit   the drafted tokens that the model agrees with, from their slots in the tree to the slots behind the sequence
//   eviction      the slots with the largest attention weights, and the latest, to the front of the cache in their order
//
// Both are bound by the rows' bytes (each read and written once) and, for one sequence, by the launches.  Caches are compacted in
// place: a copy would take as much memory again.
#include <algorithm>
#include <new>
#include <vector>

#include "lane_ops.h"

namespace flh {
namespace {

constexpr int kMaxLayers = 128;                        // caches of one launch: 2 KiB of its arguments
constexpr uint32_t kMaxNodes = 256;

struct Caches {
  __half *k[kMaxLayers], *v[kMaxLayers];
};

// ---- tree commit ---------------------------------------------------------------------------------------------------
// One wave per sequence walks the tree from node 0: the next node is the lowest child whose token the model has chosen.  Lane i looks
// at the nodes i, i + 64, ...; children come behind their parent, so the walk ends after at most T steps.
__global__ __launch_bounds__(64) void tree_walk_kernel(const long long* __restrict__ tokens, const long long* __restrict__ parents,
                                                       uint32_t parents_stride, const long long* __restrict__ chosen,
                                                       const long long* __restrict__ lengths, long long* __restrict__ path,
                                                       long long* __restrict__ accepted, long long* __restrict__ next,
                                                       long long* __restrict__ new_lengths, uint32_t T, uint32_t max_len) {
  constexpr int N = kMaxNodes / 64;
  const uint32_t b = blockIdx.x;
  const int lane = threadIdx.x;
  const long long n = lengths[b];
  const bool active = n >= 0 && n + T <= max_len;
  long long tok[N], par[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t c = i * 64 + lane;
    tok[i] = c < T ? tokens[(size_t)b * T + c] : 0;
    par[i] = c < T ? parents[(size_t)b * parents_stride + c] : -1;
  }
  uint32_t node = 0, count = 0;
  long long want = active ? chosen[(size_t)b * T] : -1;
  if (active) {
    for (;;) {
      if (lane == 0) path[(size_t)b * T + count] = node;
      ++count;
      uint32_t found = T;
#pragma unroll
      for (int i = N - 1; i >= 0; --i) {
        const uint32_t c = i * 64 + lane;
        const unsigned long long hit = __ballot(c < T && c > node && par[i] == (long long)node && tok[i] == want);
        if (hit) found = i * 64 + __builtin_ctzll(hit);
      }
      if (found == T) break;
      node = found;
      want = chosen[(size_t)b * T + node];
    }
  }
  for (uint32_t i = count + lane; i < T; i += 64) path[(size_t)b * T + i] = -1;
  if (lane == 0) accepted[b] = count, next[b] = want, new_lengths[b] = n + count;
}

// One workgroup per (layer, key or value, sequence, head): the accepted rows through LDS, so that no row is overwritten unread.
__global__ __launch_bounds__(256) void tree_move_kernel(Caches caches, const long long* __restrict__ path,
                                                        const long long* __restrict__ accepted, const long long* __restrict__ lengths,
                                                        uint32_t T, uint32_t Hkv, uint32_t pieces, uint32_t max_len) {
  extern __shared__ __align__(16) v4i rows[];
  const uint32_t bg = blockIdx.x, b = bg / Hkv, layer = blockIdx.y;
  const uint32_t count = (uint32_t)accepted[b];
  if (count < 2) return;
  v4i* cache = (v4i*)(blockIdx.z ? caches.v[layer] : caches.k[layer]) + ((size_t)bg * max_len + (size_t)lengths[b]) * pieces;
  // node 0 stays where it is
  for (uint32_t i = threadIdx.x; i < (count - 1) * pieces; i += 256)
    rows[i] = cache[(size_t)path[(size_t)b * T + 1 + i / pieces] * pieces + i % pieces];
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < (count - 1) * pieces; i += 256) cache[pieces + i] = rows[i];
}

// ---- eviction ------------------------------------------------------------------------------------------------------
// A total order of floats as unsigned numbers: larger first when sorted downwards, NaN above everything, -0 with 0.
__device__ __forceinline__ unsigned rank_of(float w) {
  if (w != w) return 0xFFFFFFFFu;
  const unsigned u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One workgroup per (layer, sequence, head): the (budget - recent)-th largest weight of the slots in front of the latest, digit by
// digit, then the slots above it and the first of those at it, in order.
__global__ __launch_bounds__(256) void evict_select_kernel(const float* __restrict__ weights, const long long* __restrict__ lengths,
                                                           long long* __restrict__ kept, float* __restrict__ new_weights,
                                                           long long* __restrict__ new_lengths, uint32_t Hkv, uint32_t max_len,
                                                           uint32_t budget, uint32_t recent) {
  __shared__ unsigned count[256], part[2][4];
  __shared__ unsigned s_digit, s_rest;
  const uint32_t bg = blockIdx.x, b = bg / Hkv;
  const size_t unit = (size_t)blockIdx.y * gridDim.x + bg;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long long len = lengths[b];
  const bool valid = len >= 0 && len <= max_len;
  const uint32_t n = valid ? (uint32_t)len : 0;
  const float* w = weights + unit * max_len;
  float* nw = new_weights + unit * max_len;
  long long* list = kept + unit * budget;
  if (blockIdx.y == 0 && bg % Hkv == 0 && tid == 0) new_lengths[b] = valid && n > budget ? budget : len;
  if (n <= budget) {                                   // (a length that is none: as it is, nothing kept)
    for (uint32_t i = tid; i < budget; i += 256) list[i] = i < n ? (long long)i : -1;
    for (uint32_t i = tid; i < max_len; i += 256) nw[i] = i < n ? w[i] : 0.f;
    return;
  }
  const uint32_t old = n - recent;                     // slots that are chosen from
  unsigned prefix = 0, mask = 0, rest = budget - recent;
  for (int shift = 24; shift >= 0 && rest; shift -= 8) {
    count[tid] = 0;
    __syncthreads();
    for (uint32_t i = tid; i < old; i += 256) {
      const unsigned r = rank_of(w[i]);
      if ((r & mask) == prefix) atomicAdd(&count[(r >> shift) & 255], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      unsigned left = rest;
      int d = 255;
      while (count[d] < left) left -= count[d], --d;
      s_digit = d, s_rest = left;
    }
    __syncthreads();
    prefix |= s_digit << shift, mask |= 255u << shift, rest = s_rest;
  }
  // above the threshold, or one of the first `rest` at it, or one of the latest
  const bool none = budget == recent;
  unsigned above = 0, equal = 0;                       // of the slots so far
  for (uint32_t i0 = 0; i0 < n; i0 += 256) {
    const uint32_t i = i0 + tid;
    const float wi = i < n ? w[i] : 0.f;
    const unsigned r = rank_of(wi);
    const bool late = i >= old && i < n, up = late || (i < old && !none && r > prefix), at = i < old && !none && r == prefix;
    const unsigned long long ups = __ballot(up), ats = __ballot(at);
    __syncthreads();
    if (lane == 0) part[0][wave] = __popcll(ups), part[1][wave] = __popcll(ats);
    __syncthreads();
    unsigned a = above, e = equal;
    for (int k = 0; k < wave; ++k) a += part[0][k], e += part[1][k];
    const unsigned long long below = (1ull << lane) - 1;
    a += __popcll(ups & below), e += __popcll(ats & below);
    if (up || (at && e < rest)) {
      const unsigned to = a + min(e, rest);
      list[to] = i, nw[to] = wi;
    }
    for (int k = 0; k < 4; ++k) above += part[0][k], equal += part[1][k];
  }
  for (uint32_t i = budget + tid; i < max_len; i += 256) nw[i] = 0.f;
}

// One workgroup per (layer, sequence, head) of keys or values; slots move down only, in order, 16 rows at a time.
__global__ __launch_bounds__(256) void evict_move_kernel(Caches caches, const long long* __restrict__ lengths,
                                                         const long long* __restrict__ kept, uint32_t Hkv, uint32_t pieces,
                                                         uint32_t max_len, uint32_t budget) {
  const uint32_t bg = blockIdx.x, layer = blockIdx.y;
  const long long len = lengths[bg / Hkv];
  if (len <= budget || len > max_len) return;
  const long long* list = kept + ((size_t)layer * gridDim.x + bg) * budget;
  v4i* cache = (v4i*)(blockIdx.z ? caches.v[layer] : caches.k[layer]) + (size_t)bg * max_len * pieces;
  const uint64_t all = (uint64_t)budget * pieces;
  for (uint64_t i0 = 0; i0 < all; i0 += 256) {
    const uint64_t i = i0 + threadIdx.x;
    v4i x = {0, 0, 0, 0};
    if (i < all) x = cache[(size_t)list[i / pieces] * pieces + i % pieces];
    asm volatile("" : "+v"(x));                        // (the row has arrived)
    __syncthreads();                                   // every row of these is read before one of them is written
    if (i < all) cache[i] = x;
  }
}

int take_caches(Caches& c, int from, int n, flh_half* const* k, flh_half* const* v, const char* what) {
  for (int i = 0; i < n; ++i) {
    c.k[i] = (__half*)k[from + i], c.v[i] = (__half*)v[from + i];
    if (!c.k[i] || !c.v[i]) return fail(FLH_EINVAL, "%s: null pointer", what);
    if (misaligned16(c.k[i], c.v[i])) return fail(FLH_EINVAL, "%s: caches must be 16-byte aligned", what);
  }
  return FLH_OK;
}

int check_caches(int layers, flh_half* const* k, flh_half* const* v, uint32_t B, uint32_t Hkv, uint32_t head_dim, uint32_t max_len,
                 const char* what) {
  if (layers < 0 || (layers && (!k || !v))) return fail(FLH_EINVAL, "%s: null pointer", what);
  if (Hkv == 0 || max_len == 0) return fail(FLH_EINVAL, "%s: heads and cache length must be positive", what);
  if (head_dim == 0 || head_dim % 8 || head_dim > 512) return fail(FLH_EINVAL, "%s: head_dim (%u) must be a multiple of 8, at most 512", what, head_dim);
  if ((uint64_t)B * Hkv > 0x7FFFFFFFull || max_len > (1u << 30)) return fail(FLH_EINVAL, "%s: problem too large", what);
  Caches c;
  for (int l = 0; l < layers; l += kMaxLayers)
    if (int rc = take_caches(c, l, layers - l < kMaxLayers ? layers - l : kMaxLayers, k, v, what)) return rc;
  // rows of one cache move while those of the others do
  std::vector<uintptr_t> at;
  try {
    at.reserve(2 * (size_t)layers);
  } catch (const std::bad_alloc&) {
    return fail(FLH_EINVAL, "%s: no host memory", what);
  }
  for (int l = 0; l < layers; ++l) at.push_back((uintptr_t)k[l]), at.push_back((uintptr_t)v[l]);
  std::sort(at.begin(), at.end());
  for (size_t i = 1; i < at.size(); ++i)
    if (at[i] - at[i - 1] < (uint64_t)B * Hkv * max_len * head_dim * 2) return fail(FLH_EINVAL, "%s: two caches share memory", what);
  return FLH_OK;
}

}  // namespace
}  // namespace flh

using namespace flh;

extern "C" int flh_tree_commit(const int64_t* tokens, const int64_t* parents, int parents_per_sequence, const int64_t* chosen,
                               const int64_t* lengths, int64_t* path, int64_t* accepted, int64_t* next, int64_t* new_lengths, int layers,
                               flh_half* const* k_caches, flh_half* const* v_caches, uint32_t B, uint32_t T, uint32_t Hkv, uint32_t head_dim,
                               uint32_t max_len, void* stream) {
  if (!tokens || !parents || !chosen || !lengths || !path || !accepted || !next || !new_lengths)
    return fail(FLH_EINVAL, "tree_commit: null pointer");
  if (T == 0 || T > kMaxNodes) return fail(FLH_EINVAL, "tree_commit: %u nodes (1 to %u)", T, kMaxNodes);
  if (lengths == new_lengths) return fail(FLH_EINVAL, "tree_commit: the new lengths need memory of their own");
  if (int rc = check_caches(layers, k_caches, v_caches, B, Hkv, head_dim, max_len, "tree_commit")) return rc;
  if (B == 0) return FLH_OK;
  const hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(tree_walk_kernel, dim3(B), dim3(64), 0, st, (const long long*)tokens, (const long long*)parents,
                     parents_per_sequence ? T : 0u, (const long long*)chosen, (const long long*)lengths, (long long*)path,
                     (long long*)accepted, (long long*)next, (long long*)new_lengths, T, max_len);
  if (int rc = check_launch("tree_commit (walk)")) return rc;
  if (T == 1) return FLH_OK;
  const size_t smem = (size_t)(T - 1) * head_dim * 2;
  static LdsGrant grant;
  if (int rc = reserve_lds((const void*)tree_move_kernel, smem, grant, "tree_commit")) return rc;
  for (int l = 0; l < layers; l += kMaxLayers) {
    Caches c;
    const int n = layers - l < kMaxLayers ? layers - l : kMaxLayers;
    if (int rc = take_caches(c, l, n, k_caches, v_caches, "tree_commit")) return rc;
    hipLaunchKernelGGL(tree_move_kernel, dim3(B * Hkv, n, 2), dim3(256), smem, st, c, (const long long*)path, (const long long*)accepted,
                       (const long long*)lengths, T, Hkv, head_dim / 8, max_len);
    if (int rc = check_launch("tree_commit")) return rc;
  }
  return FLH_OK;
}

extern "C" int flh_evict_kv_cache(int layers, flh_half* const* k_caches, flh_half* const* v_caches, const float* weights,
                                  const int64_t* lengths, int64_t* kept, float* new_weights, int64_t* new_lengths, uint32_t B, uint32_t Hkv,
                                  uint32_t head_dim, uint32_t max_len, uint32_t budget, uint32_t recent, void* stream) {
  if (!weights || !lengths || !kept || !new_weights || !new_lengths) return fail(FLH_EINVAL, "evict_kv_cache: null pointer");
  if (layers == 0) return fail(FLH_EINVAL, "evict_kv_cache: no layers");
  if (budget == 0 || budget > max_len || recent > budget)
    return fail(FLH_EINVAL, "evict_kv_cache: the budget (%u) must be in 1 .. max_len (%u), recent (%u) at most that", budget, max_len, recent);
  if (weights == new_weights || lengths == new_lengths) return fail(FLH_EINVAL, "evict_kv_cache: the new weights and lengths need memory of their own");
  if (int rc = check_caches(layers, k_caches, v_caches, B, Hkv, head_dim, max_len, "evict_kv_cache")) return rc;
  if (B == 0) return FLH_OK;
  const hipStream_t st = (hipStream_t)stream;
  const size_t units = (size_t)B * Hkv;
  for (int l = 0; l < layers; l += kMaxLayers) {
    Caches c;
    const int n = layers - l < kMaxLayers ? layers - l : kMaxLayers;
    if (int rc = take_caches(c, l, n, k_caches, v_caches, "evict_kv_cache")) return rc;
    hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)units, n), dim3(256), 0, st, weights + l * units * max_len, (const long long*)lengths,
                       (long long*)kept + l * units * budget, new_weights + l * units * max_len, (long long*)new_lengths, Hkv, max_len, budget,
                       recent);
    if (int rc = check_launch("evict_kv_cache (select)")) return rc;
    hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)units, n, 2), dim3(256), 0, st, c, (const long long*)lengths,
                       (const long long*)kept + l * units * budget, Hkv, head_dim / 8, max_len, budget);
    if (int rc = check_launch("evict_kv_cache")) return rc;
  }
  return FLH_OK;
}
