// Causal attention of a block of T new tokens per sequence over a key / value cache held in 4 bits (cache_i4.h) that holds them already: token
// t sits in slot lengths[b] + t and sees the slots up to its own.  Queries as the cache's writer leaves them (rotated like the keys), token-major
// [B, T, Hq, D]; output [B, T, Hq * D].
//
// The rows of a key / value head are its T x rep queries, token by token, in blocks of 32, so that heads that share keys share the work of bringing
// them.  The tiles of 64 keys that a block sees are taken by four, two or one of a workgroup's waves in turn (waves_of), each by itself, without a
// barrier.  Both products run on v_mfma_f32_32x32x16_f16 in transposed form (a lane owns one query):
//
//   S^T[key, query] = sum_d ck[key, d] Q[query, d]      O^T[d, query] += sum_key cv[key, d] (p vs)[query, key]
//
// with the codes as they are held (code_halves), keys' scales multiplied into the scores and values' into the probabilities.  A tile comes to
// LDS as packed codes (8 KiB) by direct-to-LDS loads, the next one while it is worked on; values are transposed by the LDS load for 4 bits.
//
// Few rows: the tiles of a block are split over several workgroups, whose pieces (reference, sum, weighted codes) a second launch joins.
//
// What bounds it: many rows, the work around the products.  A tile of 64 keys and 32 queries is 16 + 16 matrix instructions, and 7 vector instructions for
// eight codes, twice, and about 5 for a probability: 4096 tokens of a prompt, 32 / 8 heads of 128: 193 us (passes among others; traced, one by one, 200
// to 217), 712 TFLOP/s of the products below the diagonal, the vector units busy in 71 % of the cycles and the matrix units in 32 %; 4096 behind 16000: 1400
// us, 870 TFLOP/s, at the clock that the card then holds.  The unpacking is each wave's own, about 900 of a tile's 2000 vector clocks: this library's
// kernel over an fp16 cache, which has none, takes 50 us for a prompt of 2048 tokens with its write, this one 76.  64 rows to a wave, whose codes are unpacked
// once for both halves, took 1370 us there and 238 for the prompt (one wave a SIMD, and the diagonal's pairs of a long and a short block leave it alone).
// Few rows: the start and the end of a workgroup (4 x 17 tokens behind 8000 .. 16000: 41 us, of which the codes' bytes are 11) and the blocks' last
// rows (68 rows are three blocks).
#include <algorithm>
#include <type_traits>

#include "cache_i4.h"

namespace flh {
namespace {

constexpr int kThreads = 256, kWaves = 4, kBlockRows = 32, kStages = 2;

struct Prefill {
  const __half* q;
  const long long *lengths, *counts;                                        // (counts: of padded rows; null where all T tokens count)
  const uint8_t *k_codes, *v_codes;
  const __half *k_scales, *v_scales;
  __half* out;
  float* pieces;
  uint32_t B, T, Hq, Hkv, rep, max_len, rows, blocks, splits;   // rows of a key / value head, blocks of 32 of them
  float scale_log2;
};

// tiles with a slot that a query of the block sees, of a sequence of which `count` tokens count (none: it takes no part, or none of them is in the block)
__device__ __forceinline__ uint32_t tiles_of(const Prefill& a, long long length, uint32_t count, uint32_t block) {
  if (block * kBlockRows / a.rep >= count) return 0;
  return ((uint32_t)length + min((min((block + 1) * kBlockRows, a.rows) - 1) / a.rep, count - 1)) / kTileKeys + 1;
}

// How few rows are shared: a block's tiles go in equal parts over several workgroups, as many as its share of the tiles of all gets it of kParts (two
// workgroups a compute unit, one round) and none of fewer than kPartTiles tiles.  That is known on the device alone, like the lengths: the parts are
// one list, and a workgroup takes the entry of its index, parts of a block one after the other, so that a long sequence's lie on all dies.  The same
// number for every sequence took 59 us for 17 tokens each behind 16000 and three times 200 cached ones (4 sequences, 32 / 8 heads of 128), the list
// 36; equal lengths lose nothing (4 x 16000: 42 us either way), but where the rounding gives more than kParts (576: 46 us), hence the floor.  A die's
// entries in one range: 42 us for the ragged batch.  256 of them: 72 in place of 62 us (4 x 17 behind 16000, with the joining launch), 1024: 67.  Parts of
// 4 tiles at least: 34 in place of 27 us for 4 tokens behind 16000; 5 behind 4000 take 21.5 us with parts of 8, 23.5 of 16, 29 of 32 tiles (of which the
// host's two launches are about 20 by themselves).  64 sequences lie in the lanes at a time.
constexpr uint32_t kParts = 512, kPartTiles = 8;
struct Parts {
  uint32_t total, heads, all;                          // entries of the list, blocks of all heads of a sequence, tiles of all of them
  uint32_t entries, up, first, before;                 // of the 64 sequences last looked at

  __device__ __forceinline__ uint32_t longest(const Prefill& a, uint32_t b) const {
    if (b >= a.B) return 0;
    const long long length = a.lengths[b];
    const uint32_t count = tokens_of(a.counts, b, a.T, length, a.max_len);
    return count ? ((uint32_t)length + count - 1) / kTileKeys + 1 : 0;
  }
  __device__ __forceinline__ void look(const Prefill& a, uint32_t b0, uint32_t tiles) {
    // (a sequence that takes no part has its zeros to write: one entry a block)
    entries = b0 + (threadIdx.x & 63) < a.B ? max(1u, min(min(a.splits, (tiles + kPartTiles - 1) / kPartTiles), tiles * kParts / all)) : 0u;
    up = wave_scan(entries * heads);
    first = b0;
  }
  __device__ __forceinline__ explicit Parts(const Prefill& a) {
    heads = a.Hkv * a.blocks;
    uint32_t tiles = 0;
    all = 0;                                           // (below 2^28: the caches' slots are bounded, and B x heads is at most kParts / 2)
    for (uint32_t b0 = 0; b0 < a.B; b0 += 64) {
      tiles = longest(a, b0 + (threadIdx.x & 63));
      all += from_lane(wave_scan(tiles), 63);
    }
    all = max(1u, all * heads);
    total = before = 0;
    if (a.B <= 64) {
      look(a, 0, tiles);
      total = from_lane(up, 63);
      return;
    }
    for (uint32_t b0 = 0; b0 < a.B; b0 += 64) {
      look(a, b0, longest(a, b0 + (threadIdx.x & 63)));
      before = total;
      total += from_lane(up, 63);
    }
  }
  __device__ __forceinline__ static uint32_t from_lane(uint32_t v, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); }
  // sequence b: its parts a block, and the entries in front of it
  __device__ __forceinline__ void of(const Prefill& a, uint32_t b, uint32_t& parts, uint32_t& start) {
    if (b - first >= 64) {
      before = 0;
      for (uint32_t b0 = 0;; b0 += 64) {
        look(a, b0, longest(a, b0 + (threadIdx.x & 63)));
        if (b - b0 < 64) break;
        before += from_lane(up, 63);
      }
    }
    parts = from_lane(entries, b - first);
    start = before + from_lane(up, b - first) - parts * heads;
  }
  // the sequence that holds entry `pos` (below total)
  __device__ __forceinline__ uint32_t at(const Prefill& a, uint32_t pos) {
    if (a.B > 64) {
      before = 0;
      for (uint32_t b0 = 0; b0 < a.B; b0 += 64) {
        look(a, b0, longest(a, b0 + (threadIdx.x & 63)));
        if (before + from_lane(up, 63) > pos) break;
        before += from_lane(up, 63);
      }
    }
    return first + (uint32_t)__builtin_ctzll(__ballot(before + up > pos));
  }
};

// floats of a piece: 32 rows of D sums, their references and sums of exponentials
template <int D>
constexpr uint32_t kPieceFloats = kBlockRows * (D + 2);

template <int D>
struct Layout {
  static constexpr int kRowBytes = D / 2, kTile = kTileKeys * kRowBytes, kLoads = kTile / 1024;
  static constexpr int kStage = 2 * kTile + 2 * kTileKeys * 4;
  // a wave's result: rows of D floats and their reference and sum, 16 bytes further each so that the lanes of a store meet other banks
  static constexpr int kPitch = D + 4;
  static constexpr int kWave = kStages * kStage > (kBlockRows * kPitch + 2 * kBlockRows) * 4 ? kStages * kStage : (kBlockRows * kPitch + 2 * kBlockRows) * 4;
  static constexpr int kBytes = kWaves * kWave;
};

// KW: waves that share 32 rows and take every KW-th tile: all four, two, or one with rows of its own.  Heads of 64: three waves a SIMD where they need
// 168 registers (1111 rows behind 600 slots, 16 / 16 heads: 34 us; 38 at the 172 that two leave room for).
template <int D, int KW>
__global__ __launch_bounds__(kThreads, D == 64 ? 3 : 2) void prefill_i4_kernel(Prefill a) {
  using L = Layout<D>;
  extern __shared__ __align__(1024) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint8_t* const mine = lds + wave * L::kWave;
  const unsigned mine0 = (unsigned)(size_t)mine;
  // The long blocks (late queries) of all heads come first, whatever their number: the launch ends with short ones.  Where the (sequence, key / value
  // head) pairs are a multiple of the dies, each stays on one.  (A die's pairs one after the other, the last one's long blocks late: 4 x 2048 tokens of
  // 16 heads of 64 98 us in place of 78, 8 x 2048 of 32 heads of 128 460 in place of 420; nothing was slower this way.)
  constexpr uint32_t kBlocks = kWaves / KW;            // of a workgroup
  uint32_t split = 0, splits = 1, block, bh;
  if (KW < 4 || a.splits == 1) {
    const uint32_t pairs = a.B * a.Hkv;
    bh = blockIdx.x % pairs, block = ((a.blocks - 1) / kBlocks - blockIdx.x / pairs) * kBlocks + wave / KW;
  } else {
    Parts parts(a);
    if (blockIdx.x >= parts.total) return;
    const uint32_t b = parts.at(a, blockIdx.x);
    uint32_t start;
    parts.of(a, b, splits, start);
    const uint32_t at = blockIdx.x - start, unit = at / splits;
    split = at % splits, block = unit % a.blocks, bh = b * a.Hkv + unit / a.blocks;
  }
  const uint32_t b = bh / a.Hkv, hkv = bh % a.Hkv;
  const long long len = a.lengths[b];
  const bool behind = block >= a.blocks;               // (waves without a block; they wait for the others)
  if (behind) block = a.blocks - 1;
  const uint32_t count = tokens_of(a.counts, b, a.T, len, a.max_len), tiles = tiles_of(a, len, count, block);
  const uint32_t length = tiles ? (uint32_t)len : 0u;

  const uint32_t first_row = block * kBlockRows, live_rows = min((uint32_t)kBlockRows, a.rows - first_row);
  const uint32_t row = first_row + min((uint32_t)n, live_rows - 1);    // (rows past the end repeat the last one; never stored)
  const uint32_t t = row / a.rep, head = hkv * a.rep + row % a.rep;
  const size_t q_at = (((size_t)b * a.T + t) * a.Hq + head) * D;
  // the last slot that the lane's query sees (rows behind those that count see what the last of these does, and are stored as zeros)
  const int limit = (int)(length + min(t, count - 1));
  const uint32_t slots = length + min((first_row + live_rows - 1) / a.rep, count - 1) + 1;   // slots that any of them sees
  const uint32_t tile0 = (uint32_t)((uint64_t)tiles * split / splits), tile1 = behind ? 0 : (uint32_t)((uint64_t)tiles * (split + 1) / splits);
  const uint32_t whole = (length + first_row / a.rep + 1) / kTileKeys;       // tiles that all of them see whole

  const v4i k_rows = buffer_of(a.k_codes + (size_t)bh * a.max_len * L::kRowBytes, slots * L::kRowBytes);
  const v4i v_rows = buffer_of(a.v_codes + (size_t)bh * a.max_len * L::kRowBytes, slots * L::kRowBytes);
  const v4i k_sc = buffer_of((const uint8_t*)(a.k_scales + (size_t)bh * a.max_len), slots * 2);
  const v4i v_sc = buffer_of((const uint8_t*)(a.v_scales + (size_t)bh * a.max_len), slots * 2);
  // chunks of sixteen bytes are permuted so that neither the rows of a score operand nor the sixteen keys of a transpose load fall on the
  // same banks
  unsigned k_src, v_src;
  if constexpr (D == 128) {
    k_src = (lane >> 2) * 64 + (((lane & 3) ^ (lane >> 4)) << 4);
    v_src = (lane >> 2) * 64 + (((lane & 3) ^ (lane >> 5)) << 4);      // (and 2 i of load i)
  } else {
    k_src = v_src = (lane >> 1) * 32 + (((lane & 1) ^ ((lane >> 4) & 1)) << 4);
  }
  auto k_at = [](int r, int c) { return D == 128 ? r * 64 + ((c ^ ((r >> 2) & 3)) << 4) : r * 32 + ((c ^ ((r >> 3) & 1)) << 4); };
  auto v_at = [](int r, int c) { return D == 128 ? r * 64 + ((c ^ ((r >> 3) & 3)) << 4) : r * 32 + ((c ^ ((r >> 3) & 1)) << 4); };
  auto request = [&](uint32_t tile, int stage) {
    const unsigned to = mine0 + stage * L::kStage, from = tile * L::kTile;
#pragma unroll
    for (int i = 0; i < L::kLoads; ++i) rows_to_lds(k_rows, from + i * 1024 + k_src, to + i * 1024);
    halves_to_lds(k_sc, (tile * kTileKeys + lane) * 2, to + 2 * L::kTile);
    halves_to_lds(v_sc, (tile * kTileKeys + lane) * 2, to + 2 * L::kTile + kTileKeys * 4);
#pragma unroll
    for (int i = 0; i < L::kLoads; ++i)
      rows_to_lds(v_rows, from + i * 1024 + (D == 128 ? v_src ^ ((2 * i & 3) << 4) : v_src), to + L::kTile + i * 1024);
  };

  // this lane's query as operand: half h holds the channels of its half of a row's bytes, eight a step
  constexpr int kSteps = D / 16;
  h8 x[kSteps];
#pragma unroll
  for (int j = 0; j < kSteps; ++j) x[j] = *(const h8*)(a.q + q_at + h * (D / 2) + 8 * j);
  asm volatile("" ::: "memory");
  uint32_t tile = tile0 + wave % KW;
  if (tile < tile1) request(tile, 0);
  if (tile + KW < tile1) request(tile + KW, 1);
  h8 qf[kSteps];
  float bias = 0.f;
#pragma unroll
  for (int j = 0; j < kSteps; ++j) {
    qf[j] = __builtin_shufflevector(x[j], x[j], 0, 4, 1, 5, 2, 6, 3, 7);
#pragma unroll
    for (int e = 0; e < 4; ++e) bias = __builtin_amdgcn_fdot2(h2{qf[j][2 * e], qf[j][2 * e + 1]}, h2{(_Float16)1.0f, (_Float16)1.0f}, bias, false);
  }
  bias = -8.0f / kFromSubnormal * (bias + lane_xor_f<32>(bias));
  const float factor = kFromSubnormal * a.scale_log2;

  v16f o[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
  float ref = kLowestRef, l = 0.f, weights = 0.f;      // .. and the sum of the weights as the second product takes them
  const int g = lane >> 4, gi = lane & 15;
  const int key = 8 * (gi >> 2) + 4 * (g >> 1) + (gi & 3);             // the row that the lane addresses in a transpose load

  // eight times the weights, off the sums (of all keys: a query's are in two lanes)
  auto take_off = [&]() __attribute__((always_inline)) {
    const float eight = -8.0f / kFromSubnormal * (weights + lane_xor_f<32>(weights));
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] += eight;
    weights = 0.f;
  };
  bool set_reference = true;
  int taken = 0;
  for (int stage = 0; tile < tile1; tile += KW, stage ^= 1) {
    if (tile + KW < tile1) wait_vmcnt<2 * L::kLoads + 2>();
    else wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    const uint8_t* const kt = mine + stage * L::kStage;
    const uint8_t* const vt = kt + L::kTile;
    unsigned* const ks = (unsigned*)(mine + stage * L::kStage + 2 * L::kTile);
    unsigned* const vs = ks + kTileKeys;
    // ---- scores of two tiles of 32 keys: element r of tile i: key 32 i + 8 (r / 4) + 4 h + r % 4
    v16f st[2];
    unsigned c[2][kSteps];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int r = 0; r < 16; ++r) st[i][r] = bias;
#pragma unroll
      for (int j = 0; j < kSteps / 4; ++j) *(v4i*)(c[i] + 4 * j) = *(const v4i*)(kt + k_at(32 * i + n, h * (kSteps / 4) + j));
    }
    // the scales for all queries at once: keys' as the scores take them, values' in pairs of keys 8 apart, as the weights are packed
    const unsigned k_raw = ks[lane], v_raw = vs[lane];
    ks[lane] = __builtin_bit_cast(unsigned, low_half(k_raw) * factor);
    ((packed_u16*)vs)[2 * (lane >> 4) * 8 + 2 * (lane & 7) + ((lane >> 3) & 1)] = (unsigned short)v_raw;
#pragma unroll
    for (int j = 0; j < kSteps; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) st[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(code_halves(c[i][j]), qf[j], st[i], 0, 0, 0);
    v2i cv[2][D / 32];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
        cv[i][dt] = __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_v2i*)(vt + v_at(32 * i + key, dt) + (g & 1) * 8));
    const int key0 = (int)(tile * kTileKeys) + 4 * h;
    // ---- probabilities, then weights, in pairs (r, r + 4) as the codes' halves come: p[i][u] is slots 16 u .. of tile i
    h8 p[2][2];
    float sum, added;
    auto weigh = [&](auto masked_, auto bounded_) __attribute__((always_inline)) {
      constexpr bool MASKED = decltype(masked_)::value, BOUNDED = decltype(bounded_)::value;
      sum = added = 0.f;
      const int from = opaque(key0);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const v4i k0 = *(const v4i*)(ks + 32 * i + 16 * u + 4 * h), k1 = *(const v4i*)(ks + 32 * i + 16 * u + 8 + 4 * h);
          const v4i v2 = *(const v4i*)(vs + 16 * i + 8 * u + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int a0 = k0[e], a1 = k1[e], vv = v2[e];
            float p0 = __builtin_fmaf(st[i][8 * u + e], __int_as_float(a0), -ref);
            float p1 = __builtin_fmaf(st[i][8 * u + 4 + e], __int_as_float(a1), -ref);
            if constexpr (BOUNDED) p0 = bounded(p0, (unsigned)vv), p1 = bounded(p1, (unsigned)vv >> 16);
            p0 = __builtin_amdgcn_exp2f(p0), p1 = __builtin_amdgcn_exp2f(p1);
            h2 w2 = pair_times_halves(p0, (unsigned)vv & 0xFFFFu, p1, (unsigned)vv >> 16);
            if constexpr (MASKED) {                    // (a value that a query does not see may be NaN)
              const int at = from + 32 * i + 16 * u + e;
              if (at > limit) p0 = 0.f, w2[0] = (_Float16)0.0f;
              if (at + 8 > limit) p1 = 0.f, w2[1] = (_Float16)0.0f;
            }
            sum += p0 + p1;
            p[i][u][2 * e] = w2[0], p[i][u][2 * e + 1] = w2[1];
            added = __builtin_amdgcn_fdot2(w2, h2{(_Float16)1.0f, (_Float16)1.0f}, added, false);
          }
        }
    };
    // A reference that holds the largest weight back, p vs < 2^12 when it is set, in the first tile and again where a weight leaves fp16's range, which
    // few tiles' do.  Of the keys that the query sees alone: what it does not see may be NaN or as large as it likes.
    for (;;) {
      if (set_reference) {
        float top = -INFINITY;
        const int from = opaque(key0);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const v4i k0 = *(const v4i*)(ks + 32 * i + 16 * u + 4 * h), k1 = *(const v4i*)(ks + 32 * i + 16 * u + 8 + 4 * h);
            const v4i v2 = *(const v4i*)(vs + 16 * i + 8 * u + 4 * h);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int a0 = k0[e], a1 = k1[e], vv = v2[e], at = from + 32 * i + 16 * u + e;
              const float y0 = __builtin_fmaf(st[i][8 * u + e], __int_as_float(a0), exponent_of((unsigned)vv));
              const float y1 = __builtin_fmaf(st[i][8 * u + 4 + e], __int_as_float(a1), exponent_of((unsigned)vv >> 16));
              top = __builtin_fmaxf(top, __builtin_fmaxf(at > limit ? -INFINITY : y0, at + 8 > limit ? -INFINITY : y1));
            }
          }
        top = __builtin_fmaxf(top, lane_xor_f<32>(top));
        const float now = __builtin_fmaxf(ref, reference_for(top));
        const float alpha = __builtin_amdgcn_exp2f(ref - now);
        l *= alpha, weights *= alpha;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] *= alpha;
        ref = now;
      }
      if (tile >= whole) weigh(std::true_type{}, std::false_type{});
      else weigh(std::false_type{}, std::false_type{});
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(__builtin_fabsf(added) < INFINITY)) == 0, 1)) break;
      if (set_reference) {                              // (scores of 10^8, or NaN)
        weigh(std::true_type{}, std::true_type{});
        break;
      }
      set_reference = true;
    }
    set_reference = false;
    l += sum, weights += added;
    // ---- output: 32 channels as rows; the lane's sixteen keys 8 (r / 4) + 4 h + r % 4 of a tile of 32 in nibble r
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) {
          const int w8 = cv[i][dt][u];
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(code_halves((unsigned)w8), p[i][u], o[dt], 0, 0, 0);
        }
    if (++taken == kTakeOff) take_off(), taken = 0;
    if (tile + 2 * KW < tile1) {
      wait_lds();                                      // (what was read of this stage)
      request(tile + 2 * KW, stage);
    }
  }

  // ---- the waves' results together
  l += lane_xor_f<32>(l);
  take_off();
  wait_lds();
  float* const there = (float*)mine;                   // (its own stages: everything asked for has come)
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v4f y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = o[dt][4 * k + e] * kFromSubnormal;
      *(v4f*)(there + n * L::kPitch + 32 * dt + 8 * k + 4 * h) = y;
    }
  if constexpr (KW == 1) {
    if (behind) return;
    // its own rows: normalised on the way to the output, in whole rows
    if (h == 0) there[kBlockRows * L::kPitch + n] = tiles ? 1.0f / l : 0.f;   // (a sequence that takes no part: zeros)
    wait_lds();
    constexpr int kChunks = D / 8;
#pragma unroll 2
    for (uint32_t i = lane; i < live_rows * kChunks; i += 64) {
      const uint32_t r = i / kChunks, ch = i % kChunks * 8, at = first_row + r;
      const float inv = there[kBlockRows * L::kPitch + r];
      const bool counts = at / a.rep < count;
      h8 z;
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = (_Float16)(there[r * L::kPitch + ch + e] * inv);
      if (!counts) z = h8{};
      *(h8*)(a.out + (((size_t)b * a.T + at / a.rep) * a.Hq + hkv * a.rep + at % a.rep) * D + ch) = z;
    }
    return;
  }
  if (h == 0) there[kBlockRows * L::kPitch + n] = ref, there[kBlockRows * L::kPitch + kBlockRows + n] = l;
  __syncthreads();
  if (behind) return;
  // a thread: eight channels of a row at a time
  constexpr int kChunks = D / 8;
  const uint8_t* const first_wave = lds + wave / KW * KW * L::kWave;
  for (uint32_t i = tid % (KW * 64); i < live_rows * kChunks; i += KW * 64) {
    const uint32_t r = i / kChunks, ch = i % kChunks * 8;
    float m = kLowestRef, wt[KW], sum = 0.f;
#pragma unroll
    for (int k = 0; k < KW; ++k) m = __builtin_fmaxf(m, ((const float*)(first_wave + k * L::kWave))[kBlockRows * L::kPitch + r]);
    float y[8] = {};
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      const float* from = (const float*)(first_wave + k * L::kWave);
      const float lk = from[kBlockRows * L::kPitch + kBlockRows + r];
      wt[k] = __builtin_amdgcn_exp2f(from[kBlockRows * L::kPitch + r] - m);
      if (lk == 0.f) continue;                         // (a wave without a tile, or one whose keys the query does not see)
      sum += wt[k] * lk;
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const v4f v = *(const v4f*)(from + r * L::kPitch + ch + e);
#pragma unroll
        for (int k4 = 0; k4 < 4; ++k4) y[e + k4] += wt[k] * v[k4];
      }
    }
    if (KW == 4 && splits > 1) {
      float* piece = a.pieces + (size_t)blockIdx.x * kPieceFloats<D>;
      *(v4f*)(piece + r * D + ch) = v4f{y[0], y[1], y[2], y[3]};
      *(v4f*)(piece + r * D + ch + 4) = v4f{y[4], y[5], y[6], y[7]};
      if (ch == 0) piece[kBlockRows * D + r] = m, piece[kBlockRows * (D + 1) + r] = sum;
    } else {
      const float inv = tiles ? 1.0f / sum : 0.f;      // (a sequence that takes no part: zeros)
      const uint32_t at = first_row + r;
      const bool counts = at / a.rep < count;
      h8 z;
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = (_Float16)(y[e] * inv);
      if (!counts) z = h8{};
      *(h8*)(a.out + (((size_t)b * a.T + at / a.rep) * a.Hq + hkv * a.rep + at % a.rep) * D + ch) = z;
    }
  }
}

// one wave per row: its pieces in their order, four at a time on the way
template <int D>
__global__ __launch_bounds__(256) void prefill_i4_join_kernel(Prefill a) {
  const int lane = threadIdx.x & 63;
  const uint32_t item = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= a.B * a.Hkv * a.rows) return;
  const uint32_t bh = item / a.rows, row = item % a.rows, b = bh / a.Hkv, hkv = bh % a.Hkv;
  const uint32_t block = row / kBlockRows, r = row % kBlockRows;
  const bool counts = row / a.rep < tokens_of(a.counts, b, a.T, a.lengths[b], a.max_len);
  Parts parts(a);
  uint32_t splits, start;
  parts.of(a, b, splits, start);
  if (splits == 1) return;                             // (its workgroup has stored the output)
  const float* base = a.pieces + (size_t)(start + (hkv * a.blocks + block) * splits) * kPieceFloats<D>;
  const size_t next = kPieceFloats<D>;
  // lane s: piece s
  const float* at = base + min((uint32_t)lane, splits - 1) * next + kBlockRows * D + r;
  const bool have = (uint32_t)lane < splits;
  const float pl = have ? at[kBlockRows] : 0.f;
  const float pm = pl == 0.f ? kLowestRef : at[0];     // (nothing of it is seen)
  const float m = wave_max(pm);
  const float w = pl == 0.f ? 0.f : __builtin_amdgcn_exp2f(pm - m);
  const float l = wave_sum(w * pl);
  float o[D / 64] = {};
#pragma unroll 4
  for (uint32_t s = 0; s < splits; ++s) {
    const float ws = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), (int)s));
    const bool seen = __builtin_amdgcn_readlane(__float_as_int(pl), (int)s) != 0;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const float v = base[s * next + r * D + lane + 64 * i];
      o[i] += seen ? ws * v : 0.f;
    }
  }
  _Float16* dst = (_Float16*)(a.out + (((size_t)b * a.T + row / a.rep) * a.Hq + hkv * a.rep + row % a.rep) * D);
#pragma unroll
  for (int i = 0; i < D / 64; ++i) dst[lane + 64 * i] = (_Float16)(counts ? o[i] / l : 0.f);
}

// Waves that share a block: all four where the blocks are few (a short tail, but a joint end for each), two from `pairs` blocks on, one from twice as
// many.  us, four / two / one (traced, random codes): heads of 128, 32 / 8 of them, prompts of 512 tokens (512 blocks) 13.1 / 13.9 / 18.6, 1024 26.7 / 23.7 / 31.7,
// 2048 69 / 61 / 66, 4096 223 / 206 / 191, 2048 behind 2048 (2048) 153 / 144 / 148, 64 x 64 tokens behind 1000 (4096) 141 / 117 / 105; heads of 64, 16 / 16 of
// them, whose tiles are less work: 2 x 1111 behind 600 (1120) 28.8 / 30.5 / 37.7, 4096 (2048) 68 / 66 / 86, 4 x 2048 (4096) 81 / 69 / 66, 4 x 4096 (8192)
// 255 / 247 / 220.
uint32_t waves_of(uint64_t blocks, uint32_t head_dim) {
  const uint64_t pairs = head_dim == 128 ? 1024 : 2048;
  return blocks < pairs ? 4 : blocks < 2 * pairs ? 2 : 1;
}

// Parts that a block can have: one from half a round of workgroups on, whatever the lengths.  That is right for lengths that are alike and not for a batch
// with a single long one: 2 tokens each, 32 / 8 heads of 128, 32 sequences (256 blocks) and 33: 8000 slots each 61 and 86 us, 500 each 9 and 11, down from
// 16000 80 and 102, but 60000 and the others 200 42 and 338 (the long one's eight blocks are eight workgroups' then).  64 at most, which the joining launch has
// a lane each for: a sequence with four key / value heads of one block fills half the workgroups.
uint32_t splits_of(uint64_t B, uint64_t heads, uint32_t max_len) {
  const uint64_t tiles = ((uint64_t)max_len + kTileKeys - 1) / kTileKeys, most = (tiles + kPartTiles - 1) / kPartTiles;
  uint64_t s = 2 * B * heads > kParts ? 1 : kParts / heads;
  if (s > 64) s = 64;
  if (s > most) s = most;
  return s < 1 ? 1 : (uint32_t)s;
}
// entries of the list at most: `splits` a block, and in all the parts that kParts workgroups take and one a block
uint64_t entries_of(uint64_t B, uint64_t heads, uint32_t splits) { return std::min<uint64_t>(B * heads * splits, kParts + B * heads); }

uint64_t blocks_of(uint64_t T, uint64_t rep) { return (T * rep + kBlockRows - 1) / kBlockRows; }

bool too_large(uint64_t B, uint64_t T, uint64_t Hq, uint64_t Hkv, uint64_t max_len) {
  const uint64_t rep = Hq / Hkv;
  return B > 0x7FFFFFFFull || Hq > 0xFFFFull || T > 1u << 25 || max_len > (1u << 25) || T * rep > 0x7FFFFF00ull || B * Hkv > 0x7FFFFFFFull ||
         B * Hkv * blocks_of(T, rep) > 0x7FFFFFull || B * T * Hq > 1ull << 33 || B * Hkv * max_len > 1ull << 40;
}

}  // namespace
}  // namespace flh

using namespace flh;

extern "C" size_t flh_prefill_attention_i4_workspace_bytes(uint32_t B, uint32_t T, uint32_t Hq, uint32_t Hkv, uint32_t head_dim, uint32_t max_len) {
  if (Hq == 0 || Hkv == 0 || Hq % Hkv || (head_dim != 128 && head_dim != 64) || max_len == 0 || B == 0 || T == 0 || too_large(B, T, Hq, Hkv, max_len)) return 0;
  const uint64_t heads = (uint64_t)Hkv * blocks_of(T, Hq / Hkv);
  const uint32_t splits = splits_of(B, heads, max_len);
  return splits == 1 ? 0 : (size_t)entries_of(B, heads, splits) * kBlockRows * (head_dim + 2) * sizeof(float);
}

extern "C" int flh_prefill_attention_i4(const flh_half* q, const int64_t* lengths, const uint8_t* k_codes, const flh_half* k_scales,
                                        const uint8_t* v_codes, const flh_half* v_scales, flh_half* out, uint32_t B, uint32_t T, uint32_t Hq,
                                        uint32_t Hkv, uint32_t head_dim, uint32_t max_len, float scale, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  return flh_prefill_attention_i4_counts(q, lengths, nullptr, k_codes, k_scales, v_codes, v_scales, out, B, T, Hq, Hkv, head_dim, max_len, scale,
                                         workspace, workspace_bytes, stream);
}

extern "C" int flh_prefill_attention_i4_counts(const flh_half* q, const int64_t* lengths, const int64_t* counts, const uint8_t* k_codes,
                                               const flh_half* k_scales, const uint8_t* v_codes, const flh_half* v_scales, flh_half* out, uint32_t B,
                                               uint32_t T, uint32_t Hq, uint32_t Hkv, uint32_t head_dim, uint32_t max_len, float scale,
                                               void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "prefill_attention (4-bit cache)";
  if (!q || !lengths || !k_codes || !k_scales || !v_codes || !v_scales || !out) return fail(FLH_EINVAL, "%s: null pointer", what);
  if (misaligned16(q, k_codes, v_codes, out)) return fail(FLH_EINVAL, "%s: tensors must be 16-byte aligned", what);
  if (head_dim != 128 && head_dim != 64) return fail(FLH_EINVAL, "%s: head_dim (%u) must be 64 or 128", what, head_dim);
  if (Hq == 0 || Hkv == 0 || Hq % Hkv) return fail(FLH_EINVAL, "%s: %u query heads do not divide over %u key / value heads", what, Hq, Hkv);
  if (max_len == 0) return fail(FLH_EINVAL, "%s: the caches have no slots", what);
  if (bad_scale(scale)) return fail(FLH_EINVAL, "%s: the scale must be positive and at most 1e15", what);
  if (B == 0 || T == 0) return FLH_OK;
  if (too_large(B, T, Hq, Hkv, max_len)) return fail(FLH_EINVAL, "%s: problem too large", what);
  const uint64_t slots = (uint64_t)B * Hkv * max_len, queries = (uint64_t)B * T * Hq * head_dim * 2;
  const size_t need = flh_prefill_attention_i4_workspace_bytes(B, T, Hq, Hkv, head_dim, max_len);
  if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need))
    return fail(FLH_EINVAL, "%s: a 16-byte aligned workspace of %zu bytes is required", what, need);
  const struct { const void* at; uint64_t bytes; } in[7] = {{k_codes, slots * (head_dim / 2)}, {k_scales, slots * 2}, {v_codes, slots * (head_dim / 2)},
                                                            {v_scales, slots * 2}, {lengths, (uint64_t)B * 8}, {q, queries},
                                                            {counts, counts ? (uint64_t)B * 8 : 0}};
  for (const auto& x : in)
    if (overlap(out, queries, x.at, x.bytes) || overlap(workspace, need, x.at, x.bytes))
      return fail(FLH_EINVAL, "%s: an output shares memory with an input", what);
  if (overlap(out, queries, workspace, need)) return fail(FLH_EINVAL, "%s: the output shares memory with the workspace", what);
  Prefill a = {};
  a.q = (const __half*)q, a.lengths = (const long long*)lengths, a.counts = (const long long*)counts, a.k_codes = k_codes, a.v_codes = v_codes;
  a.k_scales = (const __half*)k_scales, a.v_scales = (const __half*)v_scales, a.out = (__half*)out, a.pieces = (float*)workspace;
  a.B = B, a.T = T, a.Hq = Hq, a.Hkv = Hkv, a.rep = Hq / Hkv, a.max_len = max_len, a.rows = T * a.rep, a.blocks = (uint32_t)blocks_of(T, a.rep);
  a.scale_log2 = scale * 1.4426950408889634f;
  const uint64_t heads = (uint64_t)Hkv * a.blocks, blocks = B * heads;
  a.splits = splits_of(B, heads, max_len);
  const uint32_t shared = waves_of(blocks, head_dim), each = kWaves / shared;   // blocks of a workgroup
  const uint64_t groups = a.splits > 1 ? entries_of(B, heads, a.splits) : (uint64_t)B * Hkv * ((a.blocks + each - 1) / each);
  auto go = [&](auto kern, auto join, size_t smem, LdsGrant& grant) {
    if (int rc = reserve_lds((const void*)kern, smem, grant, what)) return rc;
    hipLaunchKernelGGL(kern, dim3((unsigned)groups), dim3(kThreads), smem, (hipStream_t)stream, a);
    if (int rc = check_launch(what)) return rc;
    if (a.splits == 1) return FLH_OK;
    hipLaunchKernelGGL(join, dim3((unsigned)(((uint64_t)B * Hkv * a.rows + 3) / 4)), dim3(256), 0, (hipStream_t)stream, a);
    return check_launch(what);
  };
  static LdsGrant grants[2][3];
  auto form = [&](auto d) {
    constexpr int D = decltype(d)::value;
    LdsGrant* g = grants[D == 64];
    return shared == 4   ? go(prefill_i4_kernel<D, 4>, prefill_i4_join_kernel<D>, Layout<D>::kBytes, g[0])
           : shared == 2 ? go(prefill_i4_kernel<D, 2>, prefill_i4_join_kernel<D>, Layout<D>::kBytes, g[1])
                         : go(prefill_i4_kernel<D, 1>, prefill_i4_join_kernel<D>, Layout<D>::kBytes, g[2]);
  };
  return head_dim == 128 ? form(std::integral_constant<int, 128>{}) : form(std::integral_constant<int, 64>{});
}
