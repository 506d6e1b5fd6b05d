// Attention over a key / value cache whose sequences have lengths of their own, read on the device:
//
//   tree attention     T drafted tokens per sequence, rotated and written into the slots lengths[b] .. lengths[b] + T - 1; a token
//                      sees the lengths[b] slots before them and those of the tree that its row of the mask names
//   attention weights  attention (one token per sequence over lengths[b] slots, or the causal one of a prompt) that also adds every
//                      slot's probabilities, summed over the queries of its key / value head, to a running float32 sum
//
//   out[r] = sum_j p[r, j] V[j],  p[r, j] = exp(s[r, j] - m[r]) / l[r],  s = scale q[r] . K[j],  m = max_j s,  l = sum_j exp(s - m)
//   weights[j] += sum_r p[r, j]
#include "lane_ops.h"

namespace flh {

// prefill_attention.hip
int prefill_attention(const __half* q, const __half* k_cache, const __half* v_cache, __half* out, float* stats, uint32_t B, uint32_t T,
                      uint32_t Hq, uint32_t Hkv, uint32_t head_dim, uint32_t past, uint32_t max_len, float scale, hipStream_t stream);

namespace {

constexpr uint32_t kMaxNodes = 256;
constexpr float kLowest = -1e30f;                      // running maximum of a query that has seen nothing yet: finite, so that
                                                       // differences from it are no NaN; scores stay far above it

typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 lds_s4;

// What the kernels of one call share
struct Call {
  const __half *q, *k_new, *v_new, *cos, *sin;         // k_new .. sin, mask: trees only
  const long long* lengths;
  const uint8_t* mask;
  __half *k_cache, *v_cache, *out;
  float *partials, *scores, *weights;                  // scores, weights: attention weights only
  uint32_t mask_stride, B, T, Hq, Hkv, rep, rows, row_blocks, max_len, score_pitch, groups, few;
  float scale_log2;
};

// The work of a call is one list of tiles of KT keys: for every sequence and every key / value head, the tiles of the cache and then
// those of the tree.  Workgroup g takes the tiles [g c, g c + c): no workgroup has more than another by more than the rounding of c,
// however the lengths differ, and nothing of it has to be known on the host.  More than 32 WR query rows of a head are blocks of that
// many with a workgroup each, next to each other, so that the second one finds the keys and values in its die's L2 (8 x 64 nodes of 32
// / 8 heads behind 8192 tokens, two blocks, with the queries' high halves alone: 131 us with the blocks as units of the list, whose
// keys and values then come from memory twice, 126 so).
template <int KT, bool TREE>
__device__ __forceinline__ uint32_t tiles_for(const Call& a, long long n) {
  if (TREE) return n < 0 || n > (long long)a.max_len - a.T ? 0 : ((uint32_t)n + KT - 1) / KT + (a.T + KT - 1) / KT;
  return n <= 0 || n > a.max_len ? 0 : ((uint32_t)n + KT - 1) / KT;
}

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
__device__ __forceinline__ uint32_t from_lane(uint32_t v, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); }

// A sequence: its slots taken, the tiles of one of its heads, and those of all sequences before it
struct Place {
  uint32_t b, length, tiles, before;
};

// The sequences' tiles, 64 of them in the lanes at a time (the usual batch: one load and one scan for everything below)
template <int KT, bool TREE>
struct Plan {
  uint32_t c, total;                                   // tiles of a workgroup, of all
  long long n;                                         // of the last 64 sequences looked at: lane's length, tiles, inclusive sum
  uint32_t tiles, up, first, before;                   // .. the first of them, tiles before it

  __device__ __forceinline__ void look(const Call& a, uint32_t b0) {
    const uint32_t b = b0 + (threadIdx.x & 63);
    n = b < a.B ? a.lengths[b] : -1;
    tiles = tiles_for<KT, TREE>(a, n);
    up = wave_scan(tiles * a.Hkv);
    first = b0;
  }
  __device__ __forceinline__ explicit Plan(const Call& a) {
    total = 0;
    for (uint32_t b0 = 0; b0 < a.B; b0 += 64) {
      look(a, b0);
      before = total;
      total += from_lane(up, 63);
    }
    const uint32_t groups = total <= a.few * 8 ? a.few : a.groups;
    c = max(1u, (total + groups - 1) / groups);
  }
  __device__ __forceinline__ Place in_lane(const Call& a, int l) const {
    const uint32_t t = from_lane(tiles, l);
    return {first + l, from_lane((uint32_t)n, l), t, before + from_lane(up, l) - t * a.Hkv};
  }
  // the sequence b
  __device__ __forceinline__ Place of(const Call& a, uint32_t b) {
    if (b - first >= 64) {
      before = 0;
      for (uint32_t b0 = 0;; b0 += 64) {
        look(a, b0);
        if (b - b0 < 64) break;
        before += from_lane(up, 63);
      }
    }
    return in_lane(a, b - first);
  }
  // the sequence that holds tile `pos` (below total)
  __device__ __forceinline__ Place at(const Call& a, uint32_t pos) {
    if (a.B > 64) {
      before = 0;
      for (uint32_t b0 = 0; b0 < a.B; b0 += 64) {
        look(a, b0);
        if (before + from_lane(up, 63) > pos) break;
        before += from_lane(up, 63);
      }
    }
    return in_lane(a, __builtin_ctzll(__ballot(before + up > pos)));
  }
};

// floats of one piece of partial results: 32 WR rows of D sums, their maxima and sums
template <int D, int WR>
constexpr uint32_t kPiece = 32 * WR * (D + 2);

// The thread's index anew: addresses that are made of it here are not computed in front of the loops and kept in registers across them
__device__ __forceinline__ int thread_again() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// 1 KiB: lane i's 16 bytes at voff go to lds_base + 16 i (NT: past the caches)
template <bool NT>
__device__ __forceinline__ void load_rows_to_lds(const v4i& d, unsigned voff, unsigned lds_base) {
  if constexpr (NT)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds" ::"s"(lds_base), "v"(voff), "s"(d) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds_base), "v"(voff), "s"(d) : "memory", "m0");
}

// Rows of D channels in LDS, 16-byte chunks XOR-swizzled by the row: K so that the 16 rows of a fragment read fall into different
// bank groups, V so that the four rows of a transpose load (64 bytes of each) do.
template <int D>
struct Tile {
  static constexpr int PITCH = D * 2, CHUNKS = D / 8;
  static __device__ __forceinline__ int k_swizzle(int r) { return D == 128 ? r & 15 : (r >> 1) & 7; }
  static __device__ __forceinline__ int v_swizzle(int r) { return D == 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2; }
  static __device__ __forceinline__ int k_at(int r, int c) { return r * PITCH + ((c ^ k_swizzle(r)) << 4); }
  static __device__ __forceinline__ int v_at(int r, int c) { return r * PITCH + ((c ^ v_swizzle(r)) << 4); }
};

// (x0, x1): eight channels and their partners half a head further; the rotary embedding in float32, rounded once
// (LOW: and what that leaves, rounded as well)
template <bool LOW>
__device__ __forceinline__ void rotate8(h8& x0, h8& x1, h8& l0, h8& l1, const __half* cos, const __half* sin, int c, int half) {
  const h8 c0 = *(const h8*)(cos + c), c1 = *(const h8*)(cos + c + half), s0 = *(const h8*)(sin + c), s1 = *(const h8*)(sin + c + half);
  const h8 a = x0, b = x1;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float y0 = round_here((float)a[e] * (float)c0[e] - (float)b[e] * (float)s0[e]);
    const float y1 = round_here((float)b[e] * (float)c1[e] + (float)a[e] * (float)s1[e]);
    x0[e] = (_Float16)y0, x1[e] = (_Float16)y1;
    if constexpr (LOW) l0[e] = (_Float16)(y0 - (float)x0[e]), l1[e] = (_Float16)(y1 - (float)x1[e]);
  }
}

// zero for every value that is infinite or a NaN; whether there was one
__device__ __forceinline__ bool finite8(h8& x) {
  bool odd = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float v = (float)x[e];
    const bool is = !(v - v == 0.f);
    odd |= is;
    x[e] = is ? (_Float16)0.f : x[e];
  }
  return odd;
}

// The four waves of a workgroup are WR groups of 32 query rows (the queries of a key / value head: row t rep + i is head i of token t) times
// WK = 4 / WR groups of the tile's keys.  Both products run transposed, so that a lane owns one query:
//   S^T[key, query] = K Q^T (A: rows of K from LDS, B: the queries in registers),  O^T[d, query] += V^T P^T (A: transpose loads of V, B: P
//   as it sits in the scores' accumulators),  v_mfma_f32_32x32x16_f16, softmax in base 2 with float32 statistics per lane, probabilities
//   rounded to fp16 for the second product.
// K and V of the cache come by direct-to-LDS loads, the next tile during the present one.  The tree's own tiles are staged by hand:
// the keys have to be rotated, and go to the cache as well.
//
// A rotated query is rounded to fp16 as the cached keys are, but its rounding is kept as a second fp16 value with MFMAs of its own (ql): it
// moves every score by 2^-11 of its size, twice the error of the result's own rounding (4.3e-4 against 2.1e-4 of the 2-norm).  That costs
// 26.7 -> 28.6 us (2 x 63 nodes of 64 channels behind 5001 tokens), 126 -> 141 (8 x 64 of 128 behind 8192, where the MFMAs bound the launch).
//
// Probabilities are rounded to fp16 without a low half: independent errors of 2^-11 each, which a sum over many slots averages, next to the
// result's own rounding of as much (2.104e-4 of the 2-norm against 2.069e-4 with float32 probabilities, 8 x 64 behind 8192; 2.144e-4
// against 2.093e-4 over the 128 slots of 1 x 8 behind 120).  Low halves with MFMAs of their own give the float32 figure for 144 -> 164 us
// (in a graph; 2 x 63: 26.8 -> 29.7, 4 x 26 behind 1500: 30.9 -> 31.5, decode 16 x 4000: 49.7 -> 50.4), and make an infinite cached value
// NaN where a low half is zero.
//
// What bounds it: memory up to about 64 rows of a head (decode with weights, 16 x up to 4000 slots of 32 / 8 heads: 209 MB in 41 us,
// 5.1 TB/s, where a large copy reads and writes 4.9), the MFMAs from there on (8 x 64 behind 8192: 104 Gflop with the low halves in
// 128 us = 0.81 PFLOP/s, where an 8192^3 product of the vendor's reaches 1.14).  Short shares are ramps as much as tiles.  By a clock in
// the kernel, us: 2 x 63 of 64 channels, five tiles of 64 keys a workgroup: workgroups start over 4.2, lengths and list 0.9, queries and
// their rotation 1.7, the tiles 7.5, the piece 0.7; a share that ends one head and begins the next pays queries and piece again (the last
// ends at 19).  1 x 8 behind 120: starts 2.4, list 0.7, queries 2.4, a cached tile 1.0, the tree's 1.9, the piece 1.2; then the second
// launch (9 + 4 traced).  Not taken: fragments read during the MFMAs before them, as in the prefill kernel (no gain, 131 against 130 us,
// or spills); tiles of a wave of its own two ahead without barriers (58.4 against 58.9 us).
template <int D, int WR, bool TREE, bool NT>
__global__ __launch_bounds__(256, D == 128 && WR == 1 ? 1 : 2) void cache_attention_kernel(const Call a) {
  constexpr int WK = 4 / WR, NKT = WR == 4 ? 2 : 1, KT = 32 * NKT * WK;
  constexpr int PITCH = D * 2, TILE = KT * PITCH, NI = TILE / 4096, RPI = 1024 / PITCH;   // loads of a wave per tile, rows of one load
  constexpr int KS = D / 16, DT = D / 32, NF = NKT * KS;   // NF: fragments of K, and of V, that a wave reads per tile
  using L = Tile<D>;
  extern __shared__ __align__(1024) uint8_t lds[];     // K[2], V[2]; the waves' sums at the end of a segment
  __shared__ float s_m[4][32], s_l[4][32];
  __shared__ unsigned s_odd[2][4];                     // rows of a tree's tile whose values are not all finite, by the tile's parity
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wave / WK, wk = wave % WK;
  const unsigned lds0 = (unsigned)(size_t)lds;

  Plan<KT, TREE> plan(a);
  const uint32_t used = (plan.total + plan.c - 1) / plan.c * a.row_blocks;   // workgroups that have work: the first ones, on all dies
  if (blockIdx.x >= used) return;
  const uint32_t index = xcd_contiguous(blockIdx.x, used), g = index / a.row_blocks, block = index % a.row_blocks;
  uint32_t pos = g * plan.c;
  const uint32_t end = min(pos + plan.c, plan.total);
  Place at = plan.at(a, pos);
  uint32_t head = (pos - at.before) / at.tiles, tile = (pos - at.before) % at.tiles;

  // addresses inside a tile: row wave NI RPI + lane / CHUNKS of the first load, RPI rows further each (V's swizzle is the same there, K's
  // differs in the bits of 4 i)
  const int first_row = wave * NI * RPI + lane / L::CHUNKS;
  const unsigned k_off = L::k_at(first_row, lane % L::CHUNKS), v_off = L::v_at(first_row, lane % L::CHUNKS);
  const int k_at = L::k_at(wk * NKT * 32 + n, h);      // + 32 PITCH per 32 keys; step s of 16 channels enters by XOR
  // transpose loads: lane i of 16 addresses the 8-byte piece i % 4 of the 32-byte run of channels that its group will own, in row i / 4
  const int grp = lane >> 4, gi = lane & 15;
  int tr_off[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
    tr_off[dt] = L::v_at(wk * NKT * 32 + 4 * (grp >> 1) + (gi >> 2), 4 * dt + ((grp & 1) << 1) + ((gi & 3) >> 1)) + ((gi & 1) << 3);

  for (;;) {
    // ---- one segment: tiles [tile, last) of this sequence and head
    const uint32_t b = at.b, length = at.length, last = min(at.tiles, tile + (end - pos));
    const uint32_t cached = (length + KT - 1) / KT;    // tiles of the cache
    const size_t cache = ((size_t)b * a.Hkv + head) * a.max_len * D;
    auto rows_from = [&](const __half* from, uint32_t t) {   // (rows past the length arrive as zeros)
      return buffer_of((const uint8_t*)(from + cache + (size_t)t * KT * D), uniform(min((uint32_t)KT, length - t * KT)) * PITCH);
    };
    auto issue = [&](uint32_t t, int buf) {
      const v4i dk = rows_from(a.k_cache, t), dv = rows_from(a.v_cache, t);
      unsigned k = k_off, v = v_off;
      asm volatile("" : "+v"(k), "+v"(v));             // (offsets kept across the tiles are registers there are not)
#pragma unroll
      for (int i = 0; i < NI; ++i)
        load_rows_to_lds<NT>(dk, (k ^ ((i & (D == 128 ? 3 : 1)) << 6)) + i * 1024, lds0 + buf * TILE + (wave * NI + i) * 1024);
#pragma unroll
      for (int i = 0; i < NI; ++i) load_rows_to_lds<NT>(dv, v + i * 1024, lds0 + (2 + buf) * TILE + (wave * NI + i) * 1024);
    };
    const uint32_t cached_last = min(last, cached);
    if (tile < cached_last) issue(tile, 0);

    // this lane's query as B operand: channels 16 s + 8 h .. + 7 (rows past the last repeat it; they are not used)
    auto row_of = [&](int thread) { return min((block * WR + wr) * 32 + (thread & 31), a.rows - 1); };
    h8 qf[KS], ql[TREE ? KS : 1];
    {
      const int me = thread_again();
      const uint32_t row = row_of(me), h = me >> 5 & 1;
      const size_t at_token = (size_t)b * a.T + row / a.rep;
      const __half* src = a.q + (at_token * a.Hq + head * a.rep + row % a.rep) * D + 8 * h;
#pragma unroll
      for (int s = 0; s < KS; ++s) qf[s] = *(const h8*)(src + 16 * s);
      if constexpr (TREE) {
#pragma unroll
        for (int s = 0; s < KS / 2; ++s) {
          rotate8<true>(qf[s], qf[s + KS / 2], ql[s], ql[s + KS / 2], a.cos + at_token * D, a.sin + at_token * D, 16 * s + 8 * h, D / 2);
        }
      }
    }

    v16f o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
    float m_run = kLowest, sum = 0.f;                  // running maximum (scaled, base 2) and this lane's share of the sum

    // register r of 32-key tile kt: key key0 + 32 kt + 8 (r / 4) + r % 4 of the tile
    const uint32_t key0 = wk * NKT * 32 + 4 * h;
    v16f st[NKT];
    h8 pb[NKT][2];
    auto read_k = [&](int j, int buf) { return *(const h8*)(lds + buf * TILE + j % NKT * 32 * PITCH + (k_at ^ ((j / NKT) << 5))); };
    auto read_v = [&](int j, int buf) {                // (channel tile j % DT of the 16 keys j / DT)
      const uint8_t* v = lds + (2 + buf) * TILE + tr_off[j % DT] + j / DT * (16 * PITCH);
      const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)v);
      const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(v + 8 * PITCH));
      return __builtin_bit_cast(h8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    auto clear = [&]() {
#pragma unroll
      for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) st[kt][r] = 0.f;
    };
    auto score = [&](int j, h8 kf) {
      st[j % NKT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[j / NKT], st[j % NKT], 0, 0, 0);
      if constexpr (TREE) st[j % NKT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, ql[j / NKT], st[j % NKT], 0, 0, 0);
    };
    auto weigh = [&](int j, h8 vf) {
      o[j % DT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pb[j / DT / 2][j / DT % 2], o[j % DT], 0, 0, 0);
    };
    // scores that the queries do not see: those behind the cache's last slot
    auto mask_cached = [&](uint32_t t) {
      if ((t + 1) * KT <= length) return;
      asm volatile("" ::: "memory");                   // (a branch of its own: few tiles need it)
#pragma unroll
      for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (t * KT + key0 + 32 * kt + 8 * (r >> 2) + (r & 3) >= length) st[kt][r] = -INFINITY;
    };
    auto keep_scores = [&](uint32_t t) {               // for the weights' launch
      if ((block * WR + wr) * 32 + n < a.rows) {
        float* to = a.scores + ((size_t)b * a.Hq + head * a.rep + row_of(thread_again())) * a.score_pitch;
#pragma unroll
        for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4) {
            const uint32_t j = t * KT + key0 + 32 * kt + 8 * q4;
            const v4f x = {st[kt][4 * q4] * a.scale_log2, st[kt][4 * q4 + 1] * a.scale_log2, st[kt][4 * q4 + 2] * a.scale_log2,
                           st[kt][4 * q4 + 3] * a.scale_log2};
            if (j < length) *(v4f*)(to + j) = x;
          }
      }
    };
    auto softmax = [&]() {                             // st -> pb; running maximum and sum, and the sums of values with them
      float mx[2 * NKT];
#pragma unroll
      for (int c = 0; c < 2 * NKT; ++c) {
        mx[c] = fmaxf(st[c >> 1][8 * (c & 1)], st[c >> 1][8 * (c & 1) + 1]);
#pragma unroll
        for (int r = 2; r < 8; ++r) mx[c] = fmaxf(mx[c], st[c >> 1][8 * (c & 1) + r]);
      }
      float top = fmaxf(mx[0], mx[1]);
      if constexpr (NKT == 2) top = fmaxf(top, fmaxf(mx[2], mx[3]));
      const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_int(top), __float_as_int(top), false, false);
      top = fmaxf(__int_as_float(halves[0]), __int_as_float(halves[1])) * a.scale_log2;   // (the scale is positive)
      const float m_new = fmaxf(m_run, top);
      // rescale what has been added up -- unless no lane's maximum moved (the common case after the first tiles)
      if (__builtin_amdgcn_ballot_w64(m_new != m_run) != 0) {
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
        sum *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
        m_run = m_new;
      }
#pragma unroll
      for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(st[kt][r], a.scale_log2, -m_run));
          sum += p;
          pb[kt][r >> 3][r & 7] = (_Float16)p;
        }
    };
    auto compute = [&](int buf, auto mask) {
      clear();
#pragma unroll
      for (int j = 0; j < NF; ++j) score(j, read_k(j, buf));
      mask();
      softmax();
#pragma unroll
      for (int j = 0; j < NF; ++j) weigh(j, read_v(j, buf));
    };

    for (uint32_t t = tile; t < cached_last; ++t) {
      const int buf = (t - tile) & 1;
      wait_vmcnt<0>();
      __syncthreads();                                 // this tile has landed, and everybody has read the one before it
      if (t + 1 < cached_last) issue(t + 1, buf ^ 1);
      compute(buf, [&]() { mask_cached(t); });
      if constexpr (!TREE) keep_scores(t);
    }
    if constexpr (TREE) {
      for (uint32_t t = max(tile, cached); t < last; ++t) {
        if (tid < 4) s_odd[t & 1][tid] = 0;            // (last read two tiles ago)
        __syncthreads();                               // (the buffers have been read)
        // the mask's bytes of this lane's query and keys, requested in front of what takes their time to arrive
        uint8_t seen[NKT][16];
        {
          const int me = thread_again();
          const uint8_t* from = a.mask + (size_t)b * a.mask_stride + (size_t)(row_of(me) / a.rep) * a.T;
          const uint32_t first = (t - cached) * KT + wk * NKT * 32 + 4 * (me >> 5 & 1);
#pragma unroll
          for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
            for (int r = 0; r < 16; ++r) seen[kt][r] = from[min(first + 32 * kt + 8 * (r >> 2) + (r & 3), a.T - 1)];
        }
        constexpr int PAIRS = L::CHUNKS / 2;
        for (uint32_t i = thread_again(); i < KT * PAIRS; i += 256) {
          const uint32_t r = i / PAIRS, c = i % PAIRS, j = (t - cached) * KT + r;
          h8 k0 = {}, k1 = {}, v0 = {}, v1 = {};
          if (j < a.T) {
            const size_t at_token = (size_t)b * a.T + j, src = (at_token * a.Hkv + head) * D + 8 * c;
            k0 = *(const h8*)(a.k_new + src), k1 = *(const h8*)(a.k_new + src + D / 2);
            v0 = *(const h8*)(a.v_new + src), v1 = *(const h8*)(a.v_new + src + D / 2);
            h8 none;
            rotate8<false>(k0, k1, none, none, a.cos + at_token * D, a.sin + at_token * D, 8 * c, D / 2);
            if (block == 0) {
              const size_t to = cache + ((size_t)length + j) * D + 8 * c;
              *(h8*)(a.k_cache + to) = k0, *(h8*)(a.k_cache + to + D / 2) = k1;
              *(h8*)(a.v_cache + to) = v0, *(h8*)(a.v_cache + to + D / 2) = v1;
            }
          }
          // an infinite value or a NaN times the zero of a query that does not see it is a NaN: zero here, and added below
          if (finite8(v0) | finite8(v1)) atomicOr(&s_odd[t & 1][r >> 5], 1u << (r & 31));
          *(h8*)(lds + L::k_at(r, c)) = k0, *(h8*)(lds + L::k_at(r, c + PAIRS)) = k1;
          *(h8*)(lds + 2 * TILE + L::v_at(r, c)) = v0, *(h8*)(lds + 2 * TILE + L::v_at(r, c + PAIRS)) = v1;
        }
        __syncthreads();
        compute(0, [&]() {
#pragma unroll
          for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (!seen[kt][r] || (t - cached) * KT + key0 + 32 * kt + 8 * (r >> 2) + (r & 3) >= a.T) st[kt][r] = -INFINITY;
        });
#pragma unroll
        for (int w = 0; w < KT / 32; ++w)
          for (unsigned odd = uniform(s_odd[t & 1][w]); odd && w / NKT == wk; odd &= odd - 1) {
            const uint32_t j = (t - cached) * KT + 32 * w + __builtin_ctz(odd);
            const int me = thread_again();
            if (!a.mask[(size_t)b * a.mask_stride + (size_t)(row_of(me) / a.rep) * a.T + j]) continue;
            const _Float16* v = (const _Float16*)a.v_new + (((size_t)b * a.T + j) * a.Hkv + head) * D + 4 * (me >> 5 & 1);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                const float x = (float)v[32 * dt + 8 * (r >> 2) + (r & 3)];
                o[dt][r] += x - x == 0.f ? 0.f : x;
              }
          }
      }
    }

    // ---- the waves that share rows meet, then the segment's piece goes out: [row group][register quad][lane], maxima and sums behind
    const int me = thread_again(), lane = me & 63, n = me & 31, h = me >> 5 & 1;
    float l_all = sum + lane_xor_f<32>(sum);
    float* piece = a.partials + ((size_t)(g + b * a.Hkv + head) * a.row_blocks + block) * kPiece<D, WR>;
    __syncthreads();
    if constexpr (WK > 1) {
      if (h == 0) s_m[wave][n] = m_run, s_l[wave][n] = l_all;
      __syncthreads();
      float m_all = s_m[wr * WK][n];
#pragma unroll
      for (int k = 1; k < WK; ++k) m_all = fmaxf(m_all, s_m[wr * WK + k][n]);
      l_all = 0.f;
#pragma unroll
      for (int k = 0; k < WK; ++k) l_all += s_l[wr * WK + k][n] * __builtin_amdgcn_exp2f(s_m[wr * WK + k][n] - m_all);
      const float mine = __builtin_amdgcn_exp2f(m_run - m_all);
      v4f* all = (v4f*)lds;                            // [wave][quad][lane]
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
          all[(wave * DT * 4 + dt * 4 + q4) * 64 + lane] =
              v4f{o[dt][4 * q4] * mine, o[dt][4 * q4 + 1] * mine, o[dt][4 * q4 + 2] * mine, o[dt][4 * q4 + 3] * mine};
      __syncthreads();
      constexpr int QUADS = DT * 4 / WK;               // of this wave
#pragma unroll
      for (int i = 0; i < QUADS; ++i) {
        const int quad = wk * QUADS + i;
        v4f x = all[(wr * WK * DT * 4 + quad) * 64 + lane];
#pragma unroll
        for (int k = 1; k < WK; ++k) x += all[((wr * WK + k) * DT * 4 + quad) * 64 + lane];
        ((v4f*)piece)[(wr * DT * 4 + quad) * 64 + lane] = x;
      }
      m_run = m_all;
    } else {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
          ((v4f*)piece)[(wr * DT * 4 + dt * 4 + q4) * 64 + lane] = v4f{o[dt][4 * q4], o[dt][4 * q4 + 1], o[dt][4 * q4 + 2], o[dt][4 * q4 + 3]};
    }
    if (wk == 0 && h == 0) ((v2f*)(piece + 32 * WR * D))[wr * 32 + n] = v2f{m_run, l_all};

    // ---- the next head
    pos += last - tile;
    if (pos >= end) return;
    tile = 0;
    if (++head == a.Hkv) {
      head = 0;
      do {
        if (at.b + 1 == a.B) return;                   // (not reached: there are tiles left)
        at = plan.of(a, at.b + 1);
      } while (at.tiles == 0);
    }
    __syncthreads();                                   // the sums have been read: the buffers are free
  }
}

// The segments of a sequence's head: pieces first .. first + count - 1, each as often as there are row blocks
struct Segments {
  uint32_t first, count;
};
template <int KT, bool TREE>
__device__ __forceinline__ Segments segments_of(const Call& a, const Plan<KT, TREE>& plan, const Place& at, uint32_t head) {
  if (at.tiles == 0) return {0, 0};
  const uint32_t from = at.before + head * at.tiles, first = from / plan.c, last = (from + at.tiles - 1) / plan.c;
  return {first + at.b * a.Hkv + head, last - first + 1};   // (piece g + b Hkv + head: either grows from one piece to the next)
}

// Workgroup (b, head, row block, row group, 32 channels): the pieces' sums weighted and added, out as fp16.  For attention weights, workgroups
// behind those: (b, head, 256 slots), the stored scores -> probabilities, summed over the rows, added to the weights.
template <int D, int WR, bool TREE>
__global__ __launch_bounds__(256) void cache_combine_kernel(const Call a) {
  constexpr int WK = 4 / WR, NKT = WR == 4 ? 2 : 1, KT = 32 * NKT * WK, DT = D / 32;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t outs = a.B * a.Hkv * a.row_blocks * WR * DT;
  const size_t stride = (size_t)a.row_blocks * kPiece<D, WR>;   // from one piece of a row block to its next
  Plan<KT, TREE> plan(a);
  if (blockIdx.x < outs) {
    const uint32_t dt = blockIdx.x % DT, wr = blockIdx.x / DT % WR, block = blockIdx.x / (DT * WR) % a.row_blocks;
    const uint32_t bg = blockIdx.x / (DT * WR * a.row_blocks), b = bg / a.Hkv, head = bg % a.Hkv, row = (block * WR + wr) * 32 + n;
    const Place at = plan.of(a, b);
    const Segments seg = segments_of(a, plan, at, head);
    const float* piece = a.partials + (size_t)seg.first * stride + block * kPiece<D, WR>;
    const uint32_t of_row = 32 * WR * D + (wr * 32 + n) * 2, of_sum = ((wr * DT * 4 + dt * 4 + wave) * 64 + lane) * 4;
    float m = kLowest, l = 0.f;
    v4f x = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t i0 = 0; i0 < seg.count; i0 += 8) {   // eight pieces on their way at a time
      v2f ml[8];
      v4f y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float* p = piece + min(i0 + i, seg.count - 1) * stride;
        ml[i] = *(const v2f*)(p + of_row);
        y[i] = *(const v4f*)(p + of_sum);
      }
      float top = m;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i0 + i >= seg.count) ml[i] = v2f{kLowest, 0.f}, y[i] = v4f{0.f, 0.f, 0.f, 0.f};
        top = fmaxf(top, ml[i][0]);
      }
      const float keep = __builtin_amdgcn_exp2f(m - top);
      l *= keep, x *= keep;
      m = top;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float w = __builtin_amdgcn_exp2f(ml[i][0] - m);
        l = __builtin_fmaf(w, ml[i][1], l);
        x += y[i] * w;
      }
    }
    if (row < a.rows) {
      const float inv = l > 0.f ? 1.f / l : 0.f;       // (a query that sees nothing: zeros)
      const h4 y = {(_Float16)(x[0] * inv), (_Float16)(x[1] * inv), (_Float16)(x[2] * inv), (_Float16)(x[3] * inv)};
      __half* to = a.out + (((size_t)b * a.T + row / a.rep) * a.Hq + head * a.rep + row % a.rep) * D;
      *(h4*)(to + 32 * dt + 8 * wave + 4 * h) = y;
    }
    return;
  }
  if constexpr (!TREE) {
    __shared__ v2f stats[64];
    const uint32_t blocks = (a.max_len + 255) / 256, bg = (blockIdx.x - outs) / blocks, j = (blockIdx.x - outs) % blocks * 256 + tid;
    const uint32_t b = bg / a.Hkv, head = bg % a.Hkv;
    const Place at = plan.of(a, b);
    const uint32_t length = at.length;
    if (at.tiles == 0 || j - tid >= length) return;
    float* to = a.weights + (size_t)bg * a.max_len + min(j, a.max_len - 1);
    const float old = *to;
    const Segments seg = segments_of(a, plan, at, head);
    float sum = 0.f;
    for (uint32_t r0 = 0; r0 < a.rows; r0 += 64) {
      __syncthreads();
      // a wave takes every fourth row, a lane of it every 64th segment
      for (uint32_t r = r0 + wave; r < min(a.rows, r0 + 64); r += 4) {
        const float* piece = a.partials + (size_t)seg.first * stride + r / (32 * WR) * kPiece<D, WR> + 32 * WR * D + r % (32 * WR) * 2;
        float m = kLowest, l = 0.f;
        for (uint32_t i = lane; i < seg.count; i += 64) {
          const v2f ml = *(const v2f*)(piece + i * stride);
          const float top = fmaxf(m, ml[0]);
          l = l * __builtin_amdgcn_exp2f(m - top) + ml[1] * __builtin_amdgcn_exp2f(ml[0] - top);
          m = top;
        }
        const float top = wave_max(m);
        l = wave_sum(l * __builtin_amdgcn_exp2f(m - top));
        m = top;
        if (lane == 0) stats[r - r0] = v2f{m, l == 0.f ? 0.f : 1.f / l};   // (a sum of NaN: no weight of the row is a number)
      }
      __syncthreads();
      if (j < length) {
        const float* s = a.scores + ((size_t)b * a.Hq + head * a.rep + r0) * a.score_pitch + j;
        const uint32_t rows = min(a.rows - r0, 64u);
        for (uint32_t r = 0; r < rows; r += 4) {
          float x[4];
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) x[i] = s[(size_t)min(r + i, rows - 1) * a.score_pitch];
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i)
            if (r + i < rows) sum = __builtin_fmaf(__builtin_amdgcn_exp2f(x[i] - stats[r + i][0]), stats[r + i][1], sum);
        }
      }
    }
    if (j < length) *to = old + sum;
  }
}

// ---- the weights of a prompt -----------------------------------------------------------------------------------------
// weights[b, g, j] += sum over heads of g and queries t of exp2(scale_log2 q . K[j] - lse): the scores of one more product, whose rows
// are queries and whose columns are slots, S = Q K^T on v_mfma_f32_32x32x16_f16 -- a lane owns a column, so that the sum over the queries
// stays in its registers.  A workgroup has 256 slots (64 per wave, whose keys it keeps in registers) and a chunk of the queries, 64 of
// one head at a time through LDS; of several chunks each writes its sums, and a second launch adds them in their order.
// Bound by the exponentials next to the MFMAs: one per 128 multiply-adds.
constexpr int kSlots = 256, kQueries = 64;

struct Columns {
  const __half *q, *k;
  const float* lse;                                    // [B, Hq, T]
  float *weights, *parts;                              // parts [chunk][b][g][pitch]
  uint32_t T, Hq, Hkv, rep, past, max_len, blocks, chunks, chunk, pitch, pairs;   // chunk: queries of one, a multiple of 64
  float scale_log2;
  // blocks of slots that some query of chunk c sees; pairs: their sum over the chunks
  __host__ __device__ uint32_t live_blocks(uint32_t c) const {
    const uint32_t last = c + 1 < chunks ? (c + 1) * chunk : T;
    return (past + last - 1) / kSlots + 1;
  }
};

// A query whose log2 sum is no number has no probabilities either: every slot that it sees gets NaN.  In the kernel's tiles so do
// slots that it does not see (-inf less NaN).  Columns that are NaN come here, which a launch without such a query never does: slot j's
// sum over the queries t0 .. t_end - 1, two lanes a slot.  (Told apart in the loop's tiles it is 1-2 % of every launch -- 285 -> 288.5 us
// for 4096 tokens, 79 -> 80.7 for 4 x 700 behind 100 -- or registers that spill.)
__device__ __forceinline__ float numbers_of_column(const Columns& a, uint32_t b, uint32_t g, uint32_t j, uint32_t t0, uint32_t t_end) {
  constexpr int D = 128;
  const int lane = threadIdx.x & 63, h = lane >> 5;
  const float* lse = a.lse + ((size_t)b * a.Hq + g * a.rep) * a.T;
  uint32_t seen = 0;                                   // past the latest such query
  for (uint32_t head = 0; head < a.rep; ++head)
    for (uint32_t t = t0 + lane; t < t_end; t += 64) {
      const float x = lse[(size_t)head * a.T + t];
      if (!(x - x == 0.f)) seen = max(seen, t + 1);
    }
  for (int o = 32; o; o >>= 1) seen = max(seen, (uint32_t)__shfl_xor((int)seen, o));
  if (j < a.past + seen || j >= a.past + a.T) return NAN;   // (past the last slot: not used)
  const __half* key = a.k + (((size_t)b * a.Hkv + g) * a.max_len + j) * D;
  float sum = 0.f;
  for (uint32_t head = 0; head < a.rep; ++head)
    for (uint32_t t = max(t0, j > a.past ? j - a.past : 0) + h; t < t_end; t += 2) {
      const __half* query = a.q + (((size_t)b * a.T + t) * a.Hq + g * a.rep + head) * D;
      float s = 0.f;
      for (int c = 0; c < D; c += 8) {
        const h8 x = *(const h8*)(query + c), y = *(const h8*)(key + c);
#pragma unroll
        for (int i = 0; i < 8; ++i) s = __builtin_fmaf((float)x[i], (float)y[i], s);
      }
      sum += __builtin_amdgcn_exp2f(__builtin_fmaf(s, a.scale_log2, -lse[(size_t)head * a.T + t]));
    }
  return sum + __shfl_xor(sum, 32);
}

__global__ __launch_bounds__(256, 2) void column_weights_kernel(const Columns a) {
  constexpr int D = 128, PITCH = 2 * D, TILE = kQueries * PITCH, KS = D / 16;
  using L = Tile<D>;
  __shared__ __align__(1024) uint8_t lds[2 * TILE];
  __shared__ __align__(16) float lse[4][kQueries];      // (a tile's are read one tile later)
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // (a die takes a contiguous range, whose workgroups share queries and keys in its L2)
  const uint32_t at = xcd_contiguous(blockIdx.x, gridDim.x), units = gridDim.x / a.pairs, bg = at / a.pairs, b = bg / a.Hkv, g = bg % a.Hkv;
  uint32_t chunk = 0, block = at % a.pairs;
  for (; block >= a.live_blocks(chunk); ++chunk) block -= a.live_blocks(chunk);
  const uint32_t total = a.past + a.T, j0 = block * kSlots, mine = j0 + wave * 64;
  // queries of the chunk that see a slot of the block: from the first tile of 64 that ends behind its first slot
  const uint32_t t_end = min(a.T, (chunk + 1) * a.chunk);
  uint32_t t0 = chunk * a.chunk;
  if (j0 > a.past) t0 = max(t0, (j0 - a.past) / kQueries * kQueries);
  const uint32_t steps = (t_end - t0 + kQueries - 1) / kQueries * a.rep;   // (not zero: the chunk sees the block)
  float sum[2] = {0.f, 0.f};
  {
    // this lane's slots as B operand: channels 16 s + 8 h .. + 7 (slots past the last repeat it; they are not used)
    h8 kf[2][KS];
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
      const __half* src = a.k + ((size_t)bg * a.max_len + min(mine + ct * 32 + n, total - 1)) * D + 8 * h;
#pragma unroll
      for (int s = 0; s < KS; ++s) kf[ct][s] = *(const h8*)(src + 16 * s);
    }
    // loads of a tile: four rows each, four of a wave
    const size_t stride = (size_t)a.Hq * PITCH;        // bytes from one token's query to the next
    const uint32_t my_row = wave * 16 + lane / L::CHUNKS;   // + 4 i
    const unsigned my_off = ((lane % L::CHUNKS) ^ (lane / L::CHUNKS)) << 4;   // (the swizzle by row 16 wave + 4 i + lane / 16: XOR 4 i)
    const unsigned lds0 = (unsigned)(size_t)lds, lse0 = (unsigned)(size_t)&lse[0][0];
    const uint8_t* queries = (const uint8_t*)(a.q + ((size_t)b * a.T * a.Hq + g * a.rep) * D);
    const float* of_heads = a.lse + ((size_t)b * a.Hq + g * a.rep) * a.T;
    auto issue = [&](uint32_t step, int buf) {         // (rows past the last query repeat it; their probabilities are dropped)
      const uint32_t t = t0 + step / a.rep * kQueries, head = step % a.rep;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        load_to_lds16(queries + min(t + my_row + 4 * i, a.T - 1) * stride + head * PITCH + (my_off ^ (i << 6)), lds0 + buf * TILE + (wave * 4 + i) * 1024);
      if (wave == 0) load_to_lds4(of_heads + (size_t)head * a.T + min(t + lane, a.T - 1), lse0 + (step & 3) * kQueries * 4);
    };
    // A tile of 32 queries: the MFMAs of its scores, and between them the exponentials of the tile before it (P: parity of the scores'
    // registers).  Four fragments of Q are on their way or in use at a time, those of the next tile among them.
    const int q_at = L::k_at(n, h);
    v16f st[2][2];
    v4f e[4];                                          // log2 sums of the tile before
    h8 f[4];
    auto read_q = [&](int s, int buf, int rt) { return *(const h8*)(lds + buf * TILE + rt * 32 * PITCH + (q_at ^ (s << 5))); };
    auto read_e = [&](uint32_t step, int rt) {         // register r of a tile: query 8 (r / 4) + 4 h + r % 4
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) e[q4] = *(const v4f*)&lse[step & 3][rt * 32 + 8 * q4 + 4 * h];
    };
    auto mask = [&](auto p_, uint32_t q0) {            // scores of the tile from query q0 on that are none
      constexpr int P = decltype(p_)::value;
      if (q0 + 32 <= t_end && mine + 63 <= a.past + q0) return;
      asm volatile("" ::: "memory");                   // (a branch of its own: few tiles need it)
#pragma unroll
      for (int ct = 0; ct < 2; ++ct)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const uint32_t q = q0 + 8 * (r >> 2) + 4 * h + (r & 3);
          if (q >= t_end || mine + ct * 32 + n > a.past + q) st[P][ct][r] = -INFINITY;
        }
    };
    auto tile = [&](auto p_, auto products_, uint32_t step) {
      constexpr int P = decltype(p_)::value;
      constexpr bool PRODUCTS = decltype(products_)::value;
      float part[4] = {0.f, 0.f, 0.f, 0.f};            // (sums in levels: thousands of small terms one by one lose digits)
      static_for<16>([&](auto j_) {
        constexpr int j = decltype(j_)::value, s = j >> 1, ct = j & 1;
        if constexpr (PRODUCTS) {
          if constexpr (P == 1 && j == 8) {            // the second half has its fragments; from here on the next tiles' are read
            wait_vmcnt<0>();
            wait_lgkmcnt0();
            __syncthreads();                           // the next 64 queries have landed, and everybody has read these
            if (step + 2 < steps) issue(step + 2, step & 1);
          }
          const v16f zero = {};
          st[P][ct] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[s & 3], kf[ct][s], j < 2 ? zero : st[P][ct], 0, 0, 0);
          if constexpr (ct == 1) f[s & 3] = s < 4 ? read_q(s + 4, step & 1, P) : read_q(s - 4, (step + P) & 1, P ^ 1);
        }
        constexpr int c = j >> 3, r = (2 * j) & 15;
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(st[P ^ 1][c][r], a.scale_log2, -e[r >> 2][r & 3]));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(st[P ^ 1][c][r + 1], a.scale_log2, -e[r >> 2][(r & 3) + 1]));
        part[2 * c] += p0, part[2 * c + 1] += p1;
        __builtin_amdgcn_sched_barrier(0);
      });
      sum[0] += part[0] + part[1], sum[1] += part[2] + part[3];
    };
    constexpr std::integral_constant<int, 0> first{};
    constexpr std::integral_constant<int, 1> second{};
#pragma unroll
    for (int r = 0; r < 16; ++r) st[1][0][r] = st[1][1][r] = -INFINITY;   // (in front of the first tile: nothing)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) e[q4] = v4f{0.f, 0.f, 0.f, 0.f};
    issue(0, 0);
    wait_vmcnt<0>();
    __syncthreads();
    if (steps > 1) issue(1, 1);
#pragma unroll
    for (int s = 0; s < 4; ++s) f[s] = read_q(s, 0, 0);
    for (uint32_t step = 0; step < steps; ++step) {
      const uint32_t t = t0 + step / a.rep * kQueries;
      tile(first, std::true_type{}, step);
      mask(first, t);
      read_e(step, 0);
      tile(second, std::true_type{}, step);
      mask(second, t + 32);
      read_e(step, 1);
    }
    tile(first, std::false_type{}, 0);
  }
#pragma unroll
  for (int ct = 0; ct < 2; ++ct) {
    float all = sum[ct] + lane_xor_f<32>(sum[ct]);
    const uint32_t j = mine + ct * 32 + n;
    if (__ballot(all != all)) {
      const float number = numbers_of_column(a, b, g, j, chunk * a.chunk, t_end);
      all = all != all ? number : all;
    }
    if (h == 0 && j < total) {
      if (a.chunks == 1) a.weights[(size_t)bg * a.max_len + j] += all;
      else a.parts[((size_t)chunk * units + bg) * a.pitch + j] = all;
    }
  }
}

__global__ __launch_bounds__(256) void column_sums_kernel(const Columns a, uint32_t units) {
  const uint32_t bg = blockIdx.x / a.blocks, j = blockIdx.x % a.blocks * kSlots + threadIdx.x;
  if (j >= a.past + a.T) return;
  float sum = 0.f;
  uint32_t c = 0;
  while (blockIdx.x % a.blocks >= a.live_blocks(c)) ++c;   // (the first that sees the block; the last sees all)
  for (; c < a.chunks; ++c) sum += a.parts[((size_t)c * units + bg) * a.pitch + j];
  a.weights[(size_t)bg * a.max_len + j] += sum;
}

int check_heads(const char* what, uint32_t Hq, uint32_t Hkv, uint32_t head_dim, float scale) {
  if (head_dim != 128 && head_dim != 64) return fail(FLH_EINVAL, "%s: head_dim (%u) must be 64 or 128", what, head_dim);
  if (Hq == 0 || Hkv == 0 || Hq % Hkv) return fail(FLH_EINVAL, "%s: %u query heads do not divide over %u key / value heads", what, Hq, Hkv);
  if (!(scale > 0.f) || scale > 1e15f) return fail(FLH_EINVAL, "%s: the scale must be positive and at most 1e15", what);
  return FLH_OK;
}

// How many groups of 32 rows a workgroup holds: all of the rows up to 128, so that K and V are read once.
int row_groups(uint64_t rows) { return rows <= 32 ? 1 : rows <= 64 ? 2 : 4; }

// Workgroups of the first launch that have work: as many as are resident (one per compute unit where the tiles fill its LDS, else two), so
// that every piece of work ends at about the same time -- but one per compute unit up to eight tiles each: two hide each other's waits
// only over several tiles, and more of them write more pieces.  us, two -> one: 2 x 32 nodes of 32 / 8 heads behind 4000 (4 tiles) 31.5 ->
// 25.6, 4 x 40 behind 300 (2) 26.2 -> 22.9, 1 x 16 behind 2000 (2) 24.3 -> 20.3, 8 x 20 of 64 channels behind 700 20.3 -> 19.5;  2 x 63 of
// 64 channels behind 5001 (9) 26.7 -> 28.5, 8 x 64 behind 8192 (65) 140 -> 151.
constexpr uint32_t kUnits = 256;
uint32_t work_groups(uint32_t head_dim, int wr) { return head_dim == 128 && wr == 1 ? kUnits : 2 * kUnits; }

uint32_t row_blocks_of(uint64_t rows) { return (uint32_t)((rows + 32 * row_groups(rows) - 1) / (32 * row_groups(rows))); }
uint32_t groups_of(uint32_t head_dim, uint64_t rows) {   // of one row block
  return (work_groups(head_dim, row_groups(rows)) + row_blocks_of(rows) - 1) / row_blocks_of(rows);
}

size_t partial_bytes(uint32_t B, uint64_t rows, uint32_t Hkv, uint32_t head_dim) {
  const int wr = row_groups(rows);
  return rows ? (groups_of(head_dim, rows) + (size_t)B * Hkv) * row_blocks_of(rows) * (32 * wr) * (head_dim + 2) * sizeof(float) : 0;
}

template <int D, int WR, bool TREE>
int launch_rows(Call& a, hipStream_t stream) {
  constexpr int WK = 4 / WR, NKT = WR == 4 ? 2 : 1, KT = 32 * NKT * WK;
  constexpr size_t smem = 4 * (size_t)KT * D * 2;
  static_assert(WK == 1 || smem >= 4 * 32 * D * 4, "the waves' sums reuse the tiles");
  a.row_blocks = row_blocks_of(a.rows);
  a.groups = groups_of(D, a.rows);
  a.few = (kUnits + a.row_blocks - 1) / a.row_blocks;
  auto go = [&](auto kern, LdsGrant& grant) {
    if (int rc = reserve_lds((const void*)kern, smem, grant, "cache attention")) return rc;
    hipLaunchKernelGGL(kern, dim3(a.groups * a.row_blocks), dim3(256), smem, stream, a);
    return check_launch("cache attention");
  };
  static LdsGrant grant, grant_nt;
  // A decode step reads its caches once: past the last-level cache (256 MB) if they do not fit it beside what else a step reads.  us: 16 x 4000
  // slots of 32 / 8 heads (268 MB of caches) 55.4 -> 49.8; 8 x 1000 of 32 / 32 (134 MB) 32.2 -> 32.7
  if (!TREE && WR == 1 && (uint64_t)a.B * a.Hkv * a.max_len * D * 4 > (192ull << 20)) {
    if (int rc = go(cache_attention_kernel<D, WR, TREE, !TREE && WR == 1>, grant_nt)) return rc;
  } else if (int rc = go(cache_attention_kernel<D, WR, TREE, false>, grant)) {
    return rc;
  }
  const uint64_t outs = (uint64_t)a.B * a.Hkv * a.row_blocks * WR * (D / 32), sums = TREE ? 0 : (uint64_t)a.B * a.Hkv * ((a.max_len + 255) / 256);
  hipLaunchKernelGGL((cache_combine_kernel<D, WR, TREE>), dim3((unsigned)(outs + sums)), dim3(256), 0, stream, a);
  return check_launch("cache attention (combine)");
}

template <bool TREE>
int launch_call(Call& a, uint32_t head_dim, hipStream_t stream) {
  auto go = [&](auto d) {
    constexpr int D = decltype(d)::value;
    switch (row_groups(a.rows)) {
      case 1: return launch_rows<D, 1, TREE>(a, stream);
      case 2: return launch_rows<D, 2, TREE>(a, stream);
      default: return launch_rows<D, 4, TREE>(a, stream);
    }
  };
  return head_dim == 128 ? go(std::integral_constant<int, 128>{}) : go(std::integral_constant<int, 64>{});
}

// tiles, rows and elements that fit the kernels' 32-bit counts
bool too_large(uint32_t B, uint32_t T, uint32_t Hq, uint32_t Hkv, uint32_t head_dim, uint32_t max_len) {
  const uint64_t rows = (uint64_t)T * (Hq / Hkv);
  if (rows > (1u << 24) || (uint64_t)B * Hkv > (1u << 24)) return true;   // (the products below then fit 64 bits)
  const uint64_t units = (uint64_t)B * Hkv * row_blocks_of(rows);
  // the joining launch: workgroups of 32 rows and channels, and (attention weights) of 256 slots
  if (too_many_items(units * row_groups(rows) * (head_dim / 32) + (uint64_t)B * Hkv * (((uint64_t)max_len + 255) / 256), 256)) return true;
  return max_len > (1u << 30) || units > (1u << 24) || units * ((uint64_t)max_len / 64 + 8) > 0x7FFFFFFFull ||
         (uint64_t)B * Hkv * max_len * head_dim > (1ull << 40) || (uint64_t)B * T * Hq * head_dim > (1ull << 36);
}

}  // namespace
}  // namespace flh

using namespace flh;

// (sizes that the call itself refuses need no bytes: their counts do not fit the arithmetic)
extern "C" size_t flh_tree_attention_workspace_bytes(uint32_t B, uint32_t T, uint32_t Hq, uint32_t Hkv, uint32_t head_dim) {
  if (Hkv == 0 || head_dim > 128 || too_large(B, T, Hq, Hkv, head_dim, 0)) return 0;
  return partial_bytes(B, (uint64_t)T * (Hq / Hkv), Hkv, head_dim);
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
  if (too_large(B, T, Hq, Hkv, head_dim, max_len)) return fail(FLH_EINVAL, "tree_attention: problem too large");
  const size_t need = flh_tree_attention_workspace_bytes(B, T, Hq, Hkv, head_dim);
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)
    return fail(FLH_EINVAL, "tree_attention: a 16-byte aligned workspace of %zu bytes is required", need);
  const uint64_t cache = (uint64_t)B * Hkv * max_len * head_dim * 2;
  if (overlap(k_cache, cache, v_cache, cache)) return fail(FLH_EINVAL, "tree_attention: the caches share memory");
  Call a = {};
  a.q = (const __half*)q, a.k_new = (const __half*)k_new, a.v_new = (const __half*)v_new, a.cos = (const __half*)cos, a.sin = (const __half*)sin;
  a.lengths = (const long long*)lengths, a.mask = mask, a.mask_stride = mask_per_sequence ? T * T : 0;
  a.k_cache = (__half*)k_cache, a.v_cache = (__half*)v_cache, a.out = (__half*)out, a.partials = (float*)workspace;
  a.B = B, a.T = T, a.Hq = Hq, a.Hkv = Hkv, a.rep = Hq / Hkv, a.rows = T * a.rep, a.max_len = max_len;
  a.scale_log2 = scale * 1.4426950408889634f;
  return launch_call<true>(a, head_dim, (hipStream_t)stream);
}

namespace {
uint32_t score_pitch(uint32_t max_len) { return (max_len + 3) / 4 * 4; }
}  // namespace

extern "C" size_t flh_decode_attention_weights_workspace_bytes(uint32_t B, uint32_t Hq, uint32_t Hkv, uint32_t head_dim, uint32_t max_len) {
  if (Hkv == 0 || head_dim > 128 || too_large(B, 1, Hq, Hkv, head_dim, max_len)) return 0;
  return partial_bytes(B, Hq / Hkv, Hkv, head_dim) + (size_t)B * Hq * score_pitch(max_len) * sizeof(float);
}

extern "C" int flh_decode_attention_weights_f16(const flh_half* q, const flh_half* k_cache, const flh_half* v_cache, const int64_t* lengths,
                                                flh_half* out, float* weights, uint32_t B, uint32_t Hq, uint32_t Hkv, uint32_t head_dim,
                                                uint32_t max_len, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !k_cache || !v_cache || !lengths || !out || !weights) return fail(FLH_EINVAL, "decode_attention_weights: null pointer");
  if (misaligned16(q, k_cache, v_cache, out)) return fail(FLH_EINVAL, "decode_attention_weights: tensors must be 16-byte aligned");
  if ((uintptr_t)weights & 3) return fail(FLH_EINVAL, "decode_attention_weights: the weights must be 4-byte aligned");
  if (int rc = check_heads("decode_attention_weights", Hq, Hkv, head_dim, scale)) return rc;
  if (max_len == 0) return fail(FLH_EINVAL, "decode_attention_weights: the caches have no slots");
  if (B == 0) return FLH_OK;
  if (too_large(B, 1, Hq, Hkv, head_dim, max_len)) return fail(FLH_EINVAL, "decode_attention_weights: problem too large");
  const size_t need = flh_decode_attention_weights_workspace_bytes(B, Hq, Hkv, head_dim, max_len);
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)
    return fail(FLH_EINVAL, "decode_attention_weights: a 16-byte aligned workspace of %zu bytes is required", need);
  Call a = {};
  a.q = (const __half*)q, a.lengths = (const long long*)lengths, a.out = (__half*)out, a.weights = weights;
  a.k_cache = (__half*)k_cache, a.v_cache = (__half*)v_cache;   // (only read)
  a.partials = (float*)workspace, a.scores = (float*)workspace + partial_bytes(B, Hq / Hkv, Hkv, head_dim) / sizeof(float);
  a.B = B, a.T = 1, a.Hq = Hq, a.Hkv = Hkv, a.rep = Hq / Hkv, a.rows = a.rep, a.max_len = max_len, a.score_pitch = score_pitch(max_len);
  a.scale_log2 = scale * 1.4426950408889634f;
  return launch_call<false>(a, head_dim, (hipStream_t)stream);
}

namespace {
// Chunks of queries: enough that the launch has about eight workgroups per compute unit (half of them see nothing of their slots).
void cut_columns(Columns& a, uint32_t B) {
  a.blocks = (a.past + a.T + kSlots - 1) / kSlots;
  const uint64_t units = (uint64_t)B * a.Hkv * a.blocks, tiles = (a.T + kQueries - 1) / kQueries;
  const uint64_t wanted = units >= 2048 ? 1 : (2048 + units - 1) / units, chunks = wanted < tiles ? wanted : tiles;
  a.chunk = (uint32_t)((tiles + chunks - 1) / chunks) * kQueries;
  a.chunks = (a.T + a.chunk - 1) / a.chunk;
  a.pitch = a.blocks * kSlots;
  a.pairs = 0;
  for (uint32_t c = 0; c < a.chunks; ++c) a.pairs += a.live_blocks(c);
}
size_t lse_floats(uint32_t B, uint32_t T, uint32_t Hq) { return ((size_t)B * T * Hq + 3) / 4 * 4; }

// queries, and blocks of slots of a cache of `slots`, that fit the kernels' 32-bit counts
bool too_many_columns(uint32_t B, uint32_t T, uint32_t Hq, uint32_t Hkv, uint64_t slots) {
  const uint64_t rows = (uint64_t)B * T, units = (uint64_t)B * Hkv;
  return rows > 0x7FFFFFFFull || rows * Hq > 0x7FFFFFFFull || slots > (1u << 30) || units > (1u << 24) || too_many_items(units * (slots / kSlots + 1), 256);
}
}  // namespace

extern "C" size_t flh_prefill_attention_weights_workspace_bytes(uint32_t B, uint32_t T, uint32_t Hq, uint32_t Hkv, uint32_t past) {
  if (B == 0 || T == 0 || Hkv == 0 || too_many_columns(B, T, Hq, Hkv, (uint64_t)past + T)) return 0;
  Columns a = {};
  a.T = T, a.Hkv = Hkv, a.past = past;
  cut_columns(a, B);
  return (lse_floats(B, T, Hq) + (a.chunks > 1 ? (size_t)a.chunks * B * Hkv * a.pitch : 0)) * sizeof(float);
}

extern "C" int flh_prefill_attention_weights_f16(const flh_half* q, const flh_half* k_cache, const flh_half* v_cache, flh_half* out,
                                                 float* weights, uint32_t B, uint32_t T, uint32_t Hq, uint32_t Hkv, uint32_t head_dim,
                                                 uint32_t past, uint32_t max_len, float scale, void* workspace, size_t workspace_bytes,
                                                 void* stream) {
  if (!q || !k_cache || !v_cache || !out || !weights) return fail(FLH_EINVAL, "prefill_attention_weights: null pointer");
  if (misaligned16(q, k_cache, v_cache, out)) return fail(FLH_EINVAL, "prefill_attention_weights: tensors must be 16-byte aligned");
  if ((uintptr_t)weights & 3) return fail(FLH_EINVAL, "prefill_attention_weights: the weights must be 4-byte aligned");
  if (int rc = check_heads("prefill_attention_weights", Hq, Hkv, head_dim, scale)) return rc;
  if (head_dim != 128) return fail(FLH_EINVAL, "prefill_attention_weights: head_dim (%u) must be 128", head_dim);
  if ((uint64_t)past + T > max_len) return fail(FLH_EINVAL, "prefill_attention_weights: past (%u) + T (%u) exceeds the cache length %u", past, T, max_len);
  if (B == 0 || T == 0) return FLH_OK;
  if (too_many_columns(B, T, Hq, Hkv, max_len)) return fail(FLH_EINVAL, "prefill_attention_weights: problem too large");
  const size_t need = flh_prefill_attention_weights_workspace_bytes(B, T, Hq, Hkv, past);
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)
    return fail(FLH_EINVAL, "prefill_attention_weights: a 16-byte aligned workspace of %zu bytes is required", need);
  const uint64_t queries = (uint64_t)B * T * Hq * head_dim * 2;
  if (overlap(q, queries, out, queries))               // (the sums read the queries behind the attention)
    return fail(FLH_EINVAL, "prefill_attention_weights: the output needs memory of its own");
  Columns a = {};
  a.q = (const __half*)q, a.k = (const __half*)k_cache, a.weights = weights;
  a.T = T, a.Hq = Hq, a.Hkv = Hkv, a.rep = Hq / Hkv, a.past = past, a.max_len = max_len, a.scale_log2 = scale * 1.4426950408889634f;
  a.lse = (float*)workspace, a.parts = (float*)workspace + lse_floats(B, T, Hq);
  cut_columns(a, B);
  const hipStream_t st = (hipStream_t)stream;
  if (int rc = prefill_attention(a.q, a.k, (const __half*)v_cache, (__half*)out, (float*)workspace, B, T, Hq, Hkv, head_dim, past, max_len, scale, st))
    return rc;
  const uint32_t units = B * Hkv;
  hipLaunchKernelGGL(column_weights_kernel, dim3(units * a.pairs), dim3(256), 0, st, a);
  if (int rc = check_launch("prefill_attention_weights")) return rc;
  if (a.chunks == 1) return FLH_OK;
  hipLaunchKernelGGL(column_sums_kernel, dim3(units * a.blocks), dim3(256), 0, st, a, units);
  return check_launch("prefill_attention_weights (sums)");
}
