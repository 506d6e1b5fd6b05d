// Rows of a key / value cache moved inside it, in every layer's caches at once:
//
//   tree commit   the drafted tokens that the model agrees with, from their slots in the tree to the slots behind the sequence
//   eviction      the slots with the largest attention weights, and the latest, to the front of the cache in their order
//
// Both are bound by the rows' bytes (each read and written once) and, for one sequence, by the launches.  Caches are compacted in
// place: a copy would take as much memory again.
#include <algorithm>
#include <initializer_list>
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
// A wave walks the tree of its sequence from node 0: the next node is the lowest child whose token the model has chosen.  Lane i holds
// the nodes i, i + 64, ... in registers; children come behind their parent, so the walk ends after at most T steps.
struct Tree {
  const long long *tokens, *parents, *chosen, *lengths;
  long long *path, *accepted, *next, *new_lengths;
  uint32_t parents_stride, T, max_len;
};

__device__ __forceinline__ long long of_lane(long long v, int l) {
  return (long long)((uint64_t)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 | (unsigned)__builtin_amdgcn_readlane((int)v, l));
}

// The accepted nodes into `path` (LDS), their number back; `want` is the token behind the last.
__device__ __forceinline__ uint32_t walk(const Tree& t, uint32_t b, uint16_t* path, long long& want) {
  constexpr int N = kMaxNodes / 64;
  const int lane = threadIdx.x & 63;
  long long tok[N], par[N], cho[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t c = i * 64 + lane;
    const bool have = c < t.T;
    tok[i] = have ? t.tokens[(size_t)b * t.T + c] : 0;
    par[i] = have ? t.parents[(size_t)b * t.parents_stride + c] : -1;
    cho[i] = have ? t.chosen[(size_t)b * t.T + c] : 0;
  }
  uint32_t node = 0, count = 0;
  for (;;) {
    if (lane == 0) path[count] = (uint16_t)node;
    ++count;
    const int l = (int)(node & 63);
    want = of_lane(cho[0], l);
#pragma unroll
    for (int i = 1; i < N; ++i)
      if (node >> 6 == (uint32_t)i) want = of_lane(cho[i], l);
    uint32_t found = t.T;
#pragma unroll
    for (int i = N - 1; i >= 0; --i) {
      const uint32_t c = i * 64 + lane;
      const unsigned long long hit = __ballot(c < t.T && c > node && par[i] == (long long)node && tok[i] == want);
      if (hit) found = i * 64 + __builtin_ctzll(hit);
    }
    if (found == t.T) return count;
    node = (uint32_t)__builtin_amdgcn_readfirstlane((int)found);
  }
}

// What moves at once: (keys or values, head, up to 16 chunks of 16 bytes of a row).  One workgroup has sixteen of them, of one sequence and
// layer: it walks the tree for itself (one launch instead of two; the walk is a microsecond), then reads the accepted rows of as many as fit
// its registers, and writes them when all have arrived, so that none is overwritten unread.
constexpr uint32_t kMoves = 16, kHeld = 16;            // of a workgroup; chunks in a thread's registers

__global__ __launch_bounds__(256) void tree_commit_kernel(Caches caches, Tree t, bool first, uint32_t Hkv, uint32_t pieces) {
  __shared__ uint16_t path[kMaxNodes];
  __shared__ uint32_t s_count;
  const uint32_t b = blockIdx.x, layer = blockIdx.y;
  const long long n = t.lengths[b];
  const bool active = n >= 0 && n <= (long long)t.max_len - t.T;
  const bool tells = first && layer == 0 && blockIdx.z == 0;
  if (threadIdx.x < 64) {
    long long want = -1;
    const uint32_t count = active ? walk(t, b, path, want) : 0;
    if (threadIdx.x == 0) {
      s_count = count;
      if (tells) t.accepted[b] = count, t.next[b] = want, t.new_lengths[b] = n + count;
    }
  }
  __syncthreads();
  const uint32_t count = s_count;
  if (tells)
    for (uint32_t i = threadIdx.x; i < t.T; i += 256) t.path[(size_t)b * t.T + i] = i < count ? (long long)path[i] : -1;
  if (count < 2 || !caches.k[layer]) return;
  const uint32_t slices = (pieces + 15) / 16, end = min((blockIdx.z + 1) * kMoves, 2 * Hkv * slices);
  const uint32_t rows = count - 1, width = min(16u, pieces), each = rows * width;   // (node 0 stays where it is)
  const uint32_t batch = max(1u, kHeld * 256 / each);  // (255 rows of 16 chunks fit)
  for (uint32_t u0 = blockIdx.z * kMoves; u0 < end; u0 += batch) {
    const uint32_t all = min(batch, end - u0) * each;
    v4i x[kHeld];
    v4i* to[kHeld];
#pragma unroll
    for (uint32_t k = 0; k < kHeld; ++k) {
      const uint32_t i = k * 256 + threadIdx.x;
      to[k] = nullptr;
      if (i >= all) continue;
      const uint32_t u = u0 + i / each, r = i % each / width, head = (u >> 1) / slices, c = (u >> 1) % slices * 16 + i % width;
      if (c >= pieces) continue;
      v4i* cache = (v4i*)(u & 1 ? caches.v[layer] : caches.k[layer]) + (((size_t)b * Hkv + head) * t.max_len + (size_t)n) * pieces + c;
      to[k] = cache + (size_t)(r + 1) * pieces;
      x[k] = cache[(size_t)path[r + 1] * pieces];
    }
#pragma unroll
    for (uint32_t k = 0; k < kHeld; ++k) asm volatile("" : "+v"(x[k]));   // (the rows have arrived)
    barrier_no_fence();
#pragma unroll
    for (uint32_t k = 0; k < kHeld; ++k)
      if (to[k]) *to[k] = x[k];
  }
}

// ---- eviction ------------------------------------------------------------------------------------------------------
// A total order of floats as unsigned numbers: larger first when sorted downwards, NaN above everything, -0 with 0.
__device__ __forceinline__ unsigned rank_of(float w) {
  if (w != w) return 0xFFFFFFFFu;
  const unsigned u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelectThreads = 512, kSelectWaves = kSelectThreads / 64, kDigits = 2048;
constexpr uint32_t kStagedSlots = 16384;               // weights of a head that are read once, into LDS

// One workgroup per (layer, sequence, head): the (budget - recent)-th largest weight of the slots in front of the latest, in three digits
// of eleven bits (the first holds the sign, the exponent and two bits of the fraction: few weights share one), then the slots above
// it and the first of those at it, in order: every wave counts those of its own range of slots, then writes them.
template <bool STAGED>
__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(const float* __restrict__ weights, const long long* __restrict__ lengths,
                                                                      long long* __restrict__ kept, float* __restrict__ new_weights,
                                                                      long long* __restrict__ new_lengths, uint32_t Hkv, uint32_t max_len,
                                                                      uint32_t budget, uint32_t recent) {
  extern __shared__ float staged[];
  __shared__ unsigned count[kDigits], part[2][kSelectWaves];
  __shared__ unsigned s_digit, s_rest;
  const uint32_t bg = blockIdx.x, b = bg / Hkv;
  const size_t unit = (size_t)blockIdx.y * gridDim.x + bg;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const long long len = lengths[b];
  const bool valid = len >= 0 && len <= max_len;
  const uint32_t n = valid ? (uint32_t)len : 0;
  const float* from = weights + unit * max_len;
  float* nw = new_weights + unit * max_len;
  long long* list = kept + unit * budget;
  if (blockIdx.y == 0 && bg % Hkv == 0 && tid == 0) new_lengths[b] = valid && n > budget ? budget : len;
  if (n <= budget) {                                   // (a length that is none: as it is, nothing kept)
    for (uint32_t i = tid; i < budget; i += kSelectThreads) list[i] = i < n ? (long long)i : -1;
    for (uint32_t i = tid; i < max_len; i += kSelectThreads) nw[i] = i < n ? from[i] : 0.f;
    return;
  }
  if constexpr (STAGED) {
    for (uint32_t i0 = 0; i0 < n; i0 += 8 * kSelectThreads) {   // eight on their way at a time
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = from[min(i0 + k * kSelectThreads + tid, n - 1)];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (const uint32_t i = i0 + k * kSelectThreads + tid; i < n) staged[i] = x[k];
    }
  }
  auto w = [&](uint32_t i) { return STAGED ? staged[i] : from[i]; };
  const uint32_t old = n - recent;                     // slots that are chosen from
  unsigned prefix = 0, mask = 0, rest = budget - recent;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const unsigned digits = pass == 2 ? 1023 : 2047;
    if (rest == 0) break;                              // (nothing but the latest)
    for (int i = tid; i < kDigits; i += kSelectThreads) count[i] = 0;
    __syncthreads();
    for (uint32_t i = tid; i < old; i += kSelectThreads) {
      const unsigned r = rank_of(w(i));
      if ((r & mask) == prefix) atomicAdd(&count[(r >> shift) & digits], 1u);
    }
    __syncthreads();
    // sums from the largest digit down: thread t has the four digits below 2048 - 4 t
    unsigned c[4], sum = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) sum += c[k] = count[kDigits - 1 - 4 * tid - k];
    unsigned up = wave_scan(sum);
    if (lane == 63) part[0][wave] = up;
    __syncthreads();
    for (int k = 0; k < wave; ++k) up += part[0][k];
    unsigned before = up - sum;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (before < rest && before + c[k] >= rest) s_digit = kDigits - 1 - 4 * tid - k, s_rest = rest - before;
      before += c[k];
    }
    __syncthreads();
    prefix |= s_digit << shift, mask |= digits << shift, rest = s_rest;
  }
  // above the threshold, or one of the first `rest` at it, or one of the latest
  const bool none = budget == recent;
  const uint32_t share = ((n + kSelectWaves - 1) / kSelectWaves + 63) / 64 * 64, i0 = wave * share, i1 = min(n, i0 + share);
  auto look = [&](uint32_t i, unsigned long long& ups, unsigned long long& ats) {
    const unsigned r = i < i1 ? rank_of(w(i)) : 0;
    ups = __ballot(i < i1 && (i >= old || (!none && r > prefix)));
    ats = __ballot(i < i1 && i < old && !none && r == prefix);
  };
  unsigned long long ups, ats;
  unsigned above = 0, equal = 0;
  for (uint32_t i = i0; i < i1; i += 64) {
    look(i + lane, ups, ats);
    above += __popcll(ups), equal += __popcll(ats);
  }
  __syncthreads();
  if (lane == 0) part[0][wave] = above, part[1][wave] = equal;
  __syncthreads();
  above = equal = 0;
  for (int k = 0; k < wave; ++k) above += part[0][k], equal += part[1][k];
  const unsigned long long mine = 1ull << lane, below = mine - 1;
  for (uint32_t i = i0; i < i1; i += 64) {
    look(i + lane, ups, ats);
    const unsigned a = above + __popcll(ups & below), e = equal + __popcll(ats & below);
    if ((ups & mine) || ((ats & mine) && e < rest)) {
      const unsigned to = a + min(e, rest);
      list[to] = i + lane, nw[to] = w(i + lane);
    }
    above += __popcll(ups), equal += __popcll(ats);
  }
  for (uint32_t i = budget + tid; i < max_len; i += kSelectThreads) nw[i] = 0.f;
}

// One workgroup per (layer, sequence, head) of keys or values, or per slice of their rows' chunks where those alone are few workgroups.  A
// row moves to a lower slot, and rows keep their order: a batch of rows may be written once it and those before it are read, by all
// waves, and the next batch may be requested before that (its rows lie behind everything that is written until then).
constexpr int kMovePieces = 8;                         // of a thread per batch

__global__ __launch_bounds__(256) void evict_move_kernel(Caches caches, const long long* __restrict__ lengths,
                                                         const long long* __restrict__ kept, uint32_t Hkv, uint32_t pieces, uint32_t width,
                                                         uint32_t max_len, uint32_t budget) {
  const uint32_t bg = blockIdx.x, layer = blockIdx.y, slice = blockIdx.z >> 1;
  const long long len = lengths[bg / Hkv];
  if (len <= (long long)budget || len > max_len) return;
  const long long* list = kept + ((size_t)layer * gridDim.x + bg) * budget;
  v4i* cache = (v4i*)(blockIdx.z & 1 ? caches.v[layer] : caches.k[layer]) + (size_t)bg * max_len * pieces + slice * width;
  const uint32_t all = budget * width;
  constexpr uint32_t BATCH = 256 * kMovePieces;
  v4i x[2][kMovePieces];
  auto request = [&](uint32_t first, v4i(&y)[kMovePieces]) __attribute__((always_inline)) {
    uint32_t row[kMovePieces];
#pragma unroll
    for (int k = 0; k < kMovePieces; ++k) {
      const uint32_t i = min(first + k * 256 + threadIdx.x, all - 1);
      row[k] = (uint32_t)list[i / width];
    }
#pragma unroll
    for (int k = 0; k < kMovePieces; ++k) {
      const uint32_t i = min(first + k * 256 + threadIdx.x, all - 1);
      y[k] = cache[(size_t)row[k] * pieces + i % width];
    }
  };
  auto store = [&](uint32_t first, v4i(&y)[kMovePieces]) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < kMovePieces; ++k) asm volatile("" : "+v"(y[k]));   // (the rows have arrived)
    barrier_no_fence();
#pragma unroll
    for (int k = 0; k < kMovePieces; ++k) {
      const uint32_t i = first + k * 256 + threadIdx.x;
      if (i < all) cache[(size_t)(i / width) * pieces + i % width] = y[k];
    }
  };
  request(0, x[0]);
  for (uint32_t i = 0; i < all; i += 2 * BATCH) {
    if (i + BATCH < all) request(i + BATCH, x[1]);
    store(i, x[0]);
    if (i + BATCH >= all) break;
    if (i + 2 * BATCH < all) request(i + 2 * BATCH, x[0]);
    store(i + BATCH, x[1]);
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
  if ((uint64_t)B * Hkv > 0x7FFFFFFFull || max_len > (1u << 30) || (uint64_t)max_len * (head_dim / 8) > (1u << 31)) return fail(FLH_EINVAL, "%s: problem too large", what);
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

// Outputs in memory of their own: workgroups read the inputs while others write.
struct Piece {
  const void* at;
  uint64_t bytes;
};
int check_outputs(std::initializer_list<Piece> outputs, std::initializer_list<Piece> inputs, const char* what) {
  for (const Piece* o = outputs.begin(); o != outputs.end(); ++o) {
    for (const Piece& i : inputs)
      if (overlap(o->at, o->bytes, i.at, i.bytes)) return fail(FLH_EINVAL, "%s: an output shares memory with an input", what);
    for (const Piece* p = outputs.begin(); p != o; ++p)
      if (overlap(o->at, o->bytes, p->at, p->bytes)) return fail(FLH_EINVAL, "%s: two outputs share memory", what);
  }
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
  if (too_many_items(B, 256)) return fail(FLH_EINVAL, "tree_commit: problem too large");
  const uint64_t nodes = (uint64_t)B * T * 8, each = (uint64_t)B * 8;
  if (int rc = check_outputs({{path, nodes}, {accepted, each}, {next, each}, {new_lengths, each}},
                             {{tokens, nodes}, {parents, parents_per_sequence ? nodes : T * 8ull}, {chosen, nodes}, {lengths, each}}, "tree_commit"))
    return rc;
  if (B == 0) return FLH_OK;
  const uint32_t pieces = head_dim / 8, moves = 2 * Hkv * ((pieces + 15) / 16);
  const Tree t = {(const long long*)tokens, (const long long*)parents, (const long long*)chosen, (const long long*)lengths, (long long*)path,
                  (long long*)accepted,     (long long*)next,          (long long*)new_lengths,  parents_per_sequence ? T : 0u, T, max_len};
  for (int l = 0; l == 0 || l < layers; l += kMaxLayers) {
    Caches c = {};
    const int n = layers - l < kMaxLayers ? layers - l : kMaxLayers;
    if (int rc = take_caches(c, l, n, k_caches, v_caches, "tree_commit")) return rc;
    hipLaunchKernelGGL(tree_commit_kernel, dim3(B, n ? n : 1, n ? (moves + kMoves - 1) / kMoves : 1), dim3(256), 0, (hipStream_t)stream, c, t, l == 0,
                       Hkv, pieces);
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
  if (too_many_items(units, kSelectThreads)) return fail(FLH_EINVAL, "evict_kv_cache: problem too large");
  const uint64_t heads = (uint64_t)layers * units;
  if (int rc = check_outputs({{kept, heads * budget * 8}, {new_weights, heads * max_len * 4}, {new_lengths, B * 8ull}},
                             {{weights, heads * max_len * 4}, {lengths, B * 8ull}}, "evict_kv_cache"))
    return rc;
  for (int l = 0; l < layers; l += kMaxLayers) {
    Caches c;
    const int n = layers - l < kMaxLayers ? layers - l : kMaxLayers;
    if (int rc = take_caches(c, l, n, k_caches, v_caches, "evict_kv_cache")) return rc;
    auto select = [&](auto kern, size_t smem) {
      hipLaunchKernelGGL(kern, dim3((unsigned)units, n), dim3(kSelectThreads), smem, st, weights + l * units * max_len, (const long long*)lengths,
                         (long long*)kept + l * units * budget, new_weights + l * units * max_len, (long long*)new_lengths, Hkv, max_len,
                         budget, recent);
    };
    if (max_len <= kStagedSlots) {
      static LdsGrant grant;
      if (int rc = reserve_lds((const void*)evict_select_kernel<true>, max_len * sizeof(float), grant, "evict_kv_cache")) return rc;
      select(evict_select_kernel<true>, max_len * sizeof(float));
    } else {
      select(evict_select_kernel<false>, 0);
    }
    if (int rc = check_launch("evict_kv_cache (select)")) return rc;
    // Whole rows, or four slices of them where a launch would have fewer than two workgroups per compute unit.  us for both launches, other
    // sides: halves of rows up to four workgroups per unit 157 -> 260 (20 layers x 3 x 3000 slots, 8 heads of 64 channels), eighths and
    // sixteenths up to half a workgroup 28.4 -> 24.8 and 26.0 (1 layer x 4000, heads of 128), 14.0 -> 15.0 and 15.0 (4 x 1100)
    const uint32_t pieces = head_dim / 8, slices = pieces % 4 == 0 && units * n * 2 < 512 ? 4 : 1;
    hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)units, n, 2 * slices), dim3(256), 0, st, c, (const long long*)lengths,
                       (const long long*)kept + l * units * budget, Hkv, pieces, pieces / slices, max_len, budget);
    if (int rc = check_launch("evict_kv_cache")) return rc;
  }
  return FLH_OK;
}
