// Attention of ONE new token per sequence over a key / value cache held in 4 bits (cache_i4.h) whose sequences have lengths of their own, with
// the rotary embedding, the Hadamard rotation, the quantisation and the cache write of the new token inside:
//
//   s[j] = scale ks[j] (q . ck[j]),  p[j] = exp(s[j] - max s),  out = sum_j p[j] vs[j] cv[j] / sum_j p[j]
//
// over the slots 0 .. lengths[b], the new token's among them as it is held.  Codes enter both products as they are: a row's scale is one
// factor of its score, or of its probability.
//
// Work: for every sequence and key / value head (or sixteen of its queries) the tiles of 64 keys form one list, cut into equal shares on the
// device, one a workgroup, whose four waves take every fourth tile.  A share that spans two heads writes two pieces (reference, sum,
// weighted codes); piece number = workgroup + head, unique because one of them grows from a piece to the next.  A second launch joins them.
//
// A wave works by itself: a tile's codes and scales come straight to LDS, the next tile's while it is worked on.  Matrix tiles have keys
// (scores) or channels (output) as rows and the queries of the key / value head as their sixteen columns.  A lane's sixteen scores of a tile
// are those that its operand of the second product takes, and the values' nibbles are read to match by the LDS transpose load for 4 bits.
//
// What bounds it: long caches, the bytes (32 sequences of up to 8000 slots, 32 / 8 heads of 128: 206 MB, 42 us at a large copy's 4.9 TB/s; 48 us + 4.8 of
// the joining launch); one long cache, the way of a workgroup before and after its tiles as well (60000 slots: 63 MB, 12.9 us; 19 + 3.9: the list 0.8, the
// queries 2.3, the waves' results together 1.6 us); short ones, that way and the two launches (300 slots: 8.5 + 3.5 us).  Heads of 64: 14 + 3.9, 28 + 4.0 and
// 8.0 + 3.1 us for the same slots and numbers of heads, 9.3 + 3.1 for 5 x 777 of 32 / 32.  Requesting two tiles ahead was
// slower (the other workgroup of the compute unit hides the latency), and queries brought by direct-to-LDS loads gave nothing.
#include "cache_i4.h"

namespace flh {
namespace {

constexpr int kThreads = 256, kWaves = 4, kCols = 16, kStages = 2;
constexpr uint32_t kHeadTiles = 12;

struct Decode {
  const __half *q, *k_new, *v_new, *cos, *sin;
  const long long* lengths;
  uint8_t *k_codes, *v_codes;
  __half *k_scales, *v_scales, *out;
  float* partials;
  uint32_t B, Hq, Hkv, rep, blocks, max_len, groups;   // blocks: of sixteen queries, per key / value head
  float scale_log2;
};

// tiles of a sequence whose new token takes slot n (none: it takes no part)
__device__ __forceinline__ uint32_t tiles_of(const Decode& a, long long n) {
  return n < 0 || n >= (long long)a.max_len ? 0u : (uint32_t)n / kTileKeys + 1;
}
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); }

struct Place {
  uint32_t b, length, tiles, entries, before;          // a sequence, its slots taken, tiles of a head, entries of a head, those of the sequences before
};

// How the work is shared.  Usually: the tiles of all heads are one list, each head's with kHeadTiles empty entries in front, for what a further head
// costs a workgroup (its queries, the first tile's latency, a piece), and a workgroup takes `c` entries of it.  us, 0 / 4 / 8 / 12 / 16 of them: 1 x
// 60000 slots of 8 heads 23.8 / 21.5 / 19.4 / 19.1 / 19.2, 32 x up to 8000 51.2 / 49.0 / 48.4 / 49.2 / 47.6, 5 x 778 of 32 heads 13.8 / 13.0 / 12.7 /
// 13.0 / 14.6; heads of 64: 1 x 60000 of 8 17.0 / 16.7 / 13.7 / 13.9 / 13.4, 32 x up to 8000 28.5 / 28.7 / 27.9 / 27.9 / 26.8, 16 x up to 3000 of 16
// 18.7 / 18.9 / 17.8 / 18.0 / 17.3, 5 x 777 of 32 9.0 / 9.3 / 9.1 / 9.4 / 10.6.  With few tiles to a workgroup each head is cut into equal parts of at most c
// tiles, and the parts are the list, of which a workgroup takes one (5 x 778: 17.4 -> 13.8).  64 sequences in the lanes at a time.
struct Shares {
  uint32_t c, total, heads;                            // .., entries of the list, heads of a sequence
  bool parts;
  uint32_t length, tiles, entries, up, first, before;  // of the 64 last looked at

  __device__ __forceinline__ void look(const Decode& a, uint32_t b0) {
    const uint32_t b = b0 + (threadIdx.x & 63);
    const long long n = b < a.B ? a.lengths[b] : -1;
    tiles = tiles_of(a, n);
    entries = tiles ? tiles + kHeadTiles : 0;
    length = (uint32_t)n;
    up = wave_scan(entries * heads);
    first = b0;
  }
  __device__ __forceinline__ explicit Shares(const Decode& a) {
    heads = a.Hkv * a.blocks;
    total = 0;
    parts = false;
    for (uint32_t b0 = 0; b0 < a.B; b0 += 64) {
      look(a, b0);
      before = total;
      total += lane_value(up, 63);
    }
    c = max((uint32_t)kWaves, (total + a.groups - 1) / a.groups);
    const uint32_t all_heads = a.B * heads;
    if (a.B <= 64 && all_heads < a.groups) {
      // at most total / most + all_heads parts, which are no more than the workgroups
      const uint32_t most = max((uint32_t)kWaves, (total + a.groups - all_heads - 1) / (a.groups - all_heads));
      if (most <= 2 * kWaves) {
        entries = (tiles + most - 1) / most;
        up = wave_scan(entries * heads);
        total = lane_value(up, 63), c = 1, parts = true;
        return;
      }
    }
    c = (c + kWaves - 1) / kWaves * kWaves;
  }
  __device__ __forceinline__ Place in_lane(int l) const {
    const uint32_t n = lane_value(entries, l);
    return {first + l, lane_value(length, l), lane_value(tiles, l), n, before + lane_value(up, l) - n * heads};
  }
  __device__ __forceinline__ Place of(const Decode& a, uint32_t b) {
    if (b - first >= 64) {
      before = 0;
      for (uint32_t b0 = 0;; b0 += 64) {
        look(a, b0);
        if (b - b0 < 64) break;
        before += lane_value(up, 63);
      }
    }
    return in_lane(b - first);
  }
  // the sequence that holds entry `pos` (below total)
  __device__ __forceinline__ Place at(const Decode& a, uint32_t pos) {
    if (a.B > 64) {
      before = 0;
      for (uint32_t b0 = 0; b0 < a.B; b0 += 64) {
        look(a, b0);
        if (before + lane_value(up, 63) > pos) break;
        before += lane_value(up, 63);
      }
    }
    return in_lane(__builtin_ctzll(__ballot(before + up > pos)));
  }
};

template <int D>
struct Layout {
  static constexpr int kRowBytes = D / 2, kTile = kTileKeys * kRowBytes;      // a tile's codes
  static constexpr int kLoads = kTile / 1024;                                // direct-to-LDS loads for them
  static constexpr int kStage = 2 * kTile + 2 * kTileKeys * 4;               // K, V, their scales (a dword each)
  static constexpr int kQPitch = D * 2 + 16;                                 // bytes of a query's halves
  static constexpr int kPiece = D + 2;                                       // floats of a piece and query, as the joining launch reads them
  static constexpr int kPitch = D + 4;                                       // .. and in LDS, where four at a time lie on 16 bytes
  static constexpr int kWave = kStages * kStage;
  // the waves' stages; the queries' high and low halves; what their scores begin with, and are multiplied by; the new row's codes and scales
  static constexpr int kQ = kWaves * kWave, kBias = kQ + 2 * kCols * kQPitch, kUp = kBias + kCols * 4, kNew = kUp + kCols * 4,
                       kBytes = kNew + 2 * kRowBytes + 16;
  static_assert(kCols * kPitch * 4 <= kWave, "a wave's result takes the place of its stages");
  static_assert(kPitch * 4 % 16 == 0 && kWave % 16 == 0, "rows are stored four floats at a time");
};

template <int D>
__global__ __launch_bounds__(kThreads, 2) void decode_i4_kernel(Decode a) {
  using L = Layout<D>;
  extern __shared__ __align__(1024) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, kb = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned lds0 = (unsigned)(size_t)lds;
  uint8_t* const mine = lds + wave * L::kWave;
  const unsigned mine0 = lds0 + wave * L::kWave;
  Shares shares(a);
  uint32_t pos = blockIdx.x * shares.c;
  const uint32_t end = min(shares.total, pos + shares.c);

  // where a lane's sixteen bytes of a load come from (1 KiB of rows): chunks of sixteen bytes are permuted so that neither the rows of a
  // score operand nor the sixteen keys of a transpose load fall on the same banks
  unsigned k_src[L::kLoads], v_src[L::kLoads];
#pragma unroll
  for (int i = 0; i < L::kLoads; ++i) {
    if constexpr (D == 128) {
      k_src[i] = i * 1024 + (lane >> 2) * 64 + (((lane & 3) ^ (lane >> 4)) << 4);
      v_src[i] = i * 1024 + (lane >> 2) * 64 + (((lane & 3) ^ i) << 4);
    } else {
      k_src[i] = i * 1024 + (lane >> 1) * 32 + (((lane & 1) ^ ((lane >> 4) & 1)) << 4);
      v_src[i] = i * 1024 + (lane >> 1) * 32 + (((lane & 1) ^ ((lane >> 5) & 1)) << 4);
    }
  }
  // byte of chunk `c` in row `r` of a tile as it lies in LDS
  auto k_at = [](int r, int c) { return D == 128 ? r * 64 + ((c ^ ((r >> 2) & 3)) << 4) : r * 32 + ((c ^ ((r >> 3) & 1)) << 4); };
  auto v_at = [](int r, int c) { return D == 128 ? r * 64 + ((c ^ ((r >> 4) & 3)) << 4) : r * 32 + ((c ^ ((r >> 4) & 1)) << 4); };

  while (pos < end) {
    const Place place = shares.at(a, pos);
    const uint32_t unit = (pos - place.before) / place.entries;                 // of the sequence's heads x blocks
    const uint32_t entry = pos - place.before - unit * place.entries;
    const uint32_t behind = min(place.entries, entry + (end - pos));            // entries of the head that are this workgroup's: entry .. behind
    const uint32_t first = shares.parts ? (uint32_t)((uint64_t)place.tiles * entry / place.entries) : max(entry, kHeadTiles) - kHeadTiles;
    const uint32_t stop = shares.parts ? (uint32_t)((uint64_t)place.tiles * (entry + 1) / place.entries) : max(behind, kHeadTiles) - kHeadTiles;
    if (first == stop) {                               // (its first entries alone)
      pos += behind - entry;
      continue;
    }
    const uint32_t hkv = unit / a.blocks, q0 = (unit % a.blocks) * kCols, cols = min((uint32_t)kCols, a.rep - q0);
    const uint32_t bh = place.b * a.Hkv + hkv, slot = place.length;
    const bool has_new = stop == place.tiles;

    // ---- the rows that are turned here: sixteen queries, the new key, the new value
    constexpr int kLanes = HeadRow<D>::kLanes;
    const uint32_t r = tid / kLanes, chunk = HeadRow<D>::chunk_of(tid % kLanes);
    const bool is_q = r < cols, is_new = has_new && (r == kCols || r == kCols + 1), is_v = r == kCols + 1;
    h8 x[2] = {}, c[2] = {}, s[2] = {};
    if (is_q || is_new) {
      const __half* src = is_q ? a.q + ((size_t)place.b * a.Hq + hkv * a.rep + q0 + r) * D : (is_v ? a.v_new : a.k_new) + (size_t)bh * D;
      const __half *cs = a.cos + (size_t)place.b * D, *sn = a.sin + (size_t)place.b * D;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        x[i] = *(const h8*)(src + chunk * 8 + i * (D / 2));
        c[i] = *(const h8*)(cs + chunk * 8 + i * (D / 2));
        s[i] = *(const h8*)(sn + chunk * 8 + i * (D / 2));
      }
    }

    const uint8_t* const k_base = a.k_codes + (size_t)bh * a.max_len * L::kRowBytes;
    const uint8_t* const v_base = a.v_codes + (size_t)bh * a.max_len * L::kRowBytes;
    const v4i k_rows = buffer_of(k_base, (slot + 1) * L::kRowBytes), v_rows = buffer_of(v_base, (slot + 1) * L::kRowBytes);
    const v4i k_sc = buffer_of((const uint8_t*)(a.k_scales + (size_t)bh * a.max_len), (slot + 1) * 2);
    const v4i v_sc = buffer_of((const uint8_t*)(a.v_scales + (size_t)bh * a.max_len), (slot + 1) * 2);
    auto request = [&](uint32_t tile, int stage) {
      const unsigned to = mine0 + stage * L::kStage, from = tile * L::kTile;
#pragma unroll
      for (int i = 0; i < L::kLoads; ++i) rows_to_lds(k_rows, from + k_src[i], to + i * 1024);
#pragma unroll
      for (int i = 0; i < L::kLoads; ++i) rows_to_lds(v_rows, from + v_src[i], to + L::kTile + i * 1024);
      halves_to_lds(k_sc, (tile * kTileKeys + lane) * 2, to + 2 * L::kTile);
      halves_to_lds(v_sc, (tile * kTileKeys + lane) * 2, to + 2 * L::kTile + kTileKeys * 4);
    };
    uint32_t tile = first + wave;
    if (tile < stop) request(tile, 0);

    HeadRow<D> row;
    row.set(x[0], x[1]);
    if (!is_v) {
      row.turn(c[0], c[1], s[0], s[1]);
      row.hadamard(chunk);
      row.scale(HeadRow<D>::norm());
    }
    if (r < kCols) {
      // a query as two fp16 values, by a power of two below what it is where the rotation has taken it out of their range (sums of D channels
      // over sqrt(D)): its scores are multiplied by that
      float sum = 0.f, up = 1.f;
      const unsigned most = row.top();
      if (most > 0x477FE000u && most < 0x7F800000u) {  // (65504; and finite)
        const int e = (int)(most >> 23) - (127 + 14);
        up = __int_as_float((127 + e) << 23);
        row.scale(__int_as_float((127 - e) << 23));
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        h8 high, low;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float y = row.v[8 * i + k];
          const _Float16 hi = (_Float16)y, lo = (_Float16)(y - (float)hi);
          high[code_element(k)] = hi, low[code_element(k)] = lo;
          sum += (float)hi + (float)lo;
        }
        *(h8*)(lds + L::kQ + r * L::kQPitch + (chunk + i * (D / 16)) * 16) = high;
        *(h8*)(lds + L::kQ + (kCols + r) * L::kQPitch + (chunk + i * (D / 16)) * 16) = low;
      }
      sum += dpp_f<kDppQuadXor1>(sum);
      sum += dpp_f<kDppQuadXor2>(sum);
      if constexpr (kLanes == 8) sum += dpp_f<kDppRowHalfMirror>(sum);
      if (chunk == 0) ((float*)(lds + L::kBias))[r] = -8.0f / kFromSubnormal * sum, ((float*)(lds + L::kUp))[r] = up;
    } else if (is_new) {
      const RowCodes codes = quantise(row);
      uint8_t* there = lds + L::kNew + (is_v ? L::kRowBytes : 0);
      *(unsigned*)(there + chunk * 4) = codes.lo;
      *(unsigned*)(there + D / 4 + chunk * 4) = codes.hi;
      if (chunk == 0) *(unsigned*)(lds + L::kNew + 2 * L::kRowBytes + (is_v ? 4 : 0)) = __builtin_bit_cast(unsigned short, codes.scale);
      if (q0 == 0) {
        uint8_t* to = (is_v ? a.v_codes : a.k_codes) + ((size_t)bh * a.max_len + slot) * L::kRowBytes;
        *(unsigned*)(to + chunk * 4) = codes.lo;
        *(unsigned*)(to + D / 4 + chunk * 4) = codes.hi;
        if (chunk == 0) ((_Float16*)(is_v ? a.v_scales : a.k_scales))[(size_t)bh * a.max_len + slot] = codes.scale;
      }
    }
    __syncthreads();

    // this lane's column: query `col`, channels of its quarter of the rows
    constexpr int kSteps = D / 32;
    h8 qh[kSteps], ql[kSteps];
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      qh[j] = *(const h8*)(lds + L::kQ + col * L::kQPitch + (kb * kSteps + j) * 16);
      ql[j] = *(const h8*)(lds + L::kQ + (kCols + col) * L::kQPitch + (kb * kSteps + j) * 16);
    }
    const float bias = ((const float*)(lds + L::kBias))[col], factor = kFromSubnormal * a.scale_log2;
    const bool any_up = __builtin_amdgcn_ballot_w64(((const float*)(lds + L::kUp))[col] != 1.f) != 0;
    const int key = 16 * (col >> 2) + 4 * kb + (col & 3);   // the row that the lane addresses in a transpose load

    float ref = kLowestRef, l = 0.f, weights = 0.f;    // .. and the sum of the weights as the second product takes them
    v4f o[D / 16];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[i] = v4f{0.f, 0.f, 0.f, 0.f};
    // eight times the weights, off the sums (of all keys: a query's are in four lanes)
    auto take_off = [&]() __attribute__((always_inline)) {
      float eight = weights + lane_xor_f<16>(weights);
      eight = -8.0f / kFromSubnormal * (eight + lane_xor_f<32>(eight));
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[i] += eight;
      weights = 0.f;
    };
    bool set_reference = true;
    int taken = 0;
    for (int stage = 0; tile < stop; tile += kWaves, stage ^= 1) {
      if (tile + kWaves < stop) {
        wait_lds();                                    // (what was read of the stage before)
        request(tile + kWaves, stage ^ 1);
        wait_vmcnt<2 * L::kLoads + 2>();
      } else {
        wait_vmcnt<0>();
      }
      asm volatile("" ::: "memory");
      uint8_t* const kt = mine + stage * L::kStage;
      uint8_t* const vt = kt + L::kTile;
      unsigned* const ks = (unsigned*)(vt + L::kTile);
      unsigned* const vs = ks + kTileKeys;
      const bool last = tile + 1 == place.tiles;
      if (last) {                                      // the new row takes the place of what the cache held
        const int n = slot % kTileKeys;
        if (lane < L::kRowBytes / 16) *(v4i*)(kt + k_at(n, lane)) = *(const v4i*)(lds + L::kNew + lane * 16);
        else if (lane >= 32 && lane < 32 + L::kRowBytes / 16)
          *(v4i*)(vt + v_at(n, lane - 32)) = *(const v4i*)(lds + L::kNew + L::kRowBytes + (lane - 32) * 16);
        else if (lane == 63) ks[n] = *(const unsigned*)(lds + L::kNew + 2 * L::kRowBytes), vs[n] = *(const unsigned*)(lds + L::kNew + 2 * L::kRowBytes + 4);
        wait_lds();
      }
      // the scales for all queries at once: keys' as the scores take them, values' in pairs of keys 16 apart, as the weights are packed
      const unsigned k_raw = ks[lane], v_raw = vs[lane];
      ks[lane] = __builtin_bit_cast(unsigned, low_half(k_raw) * factor);
      ((packed_u16*)vs)[(lane >> 5) * 32 + (lane & 15) * 2 + ((lane >> 4) & 1)] = (unsigned short)v_raw;
      // ---- scores: tile t of sixteen keys as rows, key 16 t + 4 kb + i in element i
      v4f st[4];
      unsigned w[4][kSteps];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        st[t] = v4f{bias, bias, bias, bias};
        if constexpr (D == 128) *(v4i*)w[t] = *(const v4i*)(kt + k_at(16 * t + col, kb));
        else *(v2i*)w[t] = *(const v2i*)(kt + k_at(16 * t + col, kb >> 1) + (kb & 1) * 8);
      }
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {               // (four sums side by side: one's next product waits for its last)
        h8 k[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          k[t] = code_halves(w[t][j]);
          st[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[t], qh[j], st[t], 0, 0, 0);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) st[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[t], ql[j], st[t], 0, 0, 0);
      }
      if (__builtin_expect(any_up, 0)) {
        const float up = ((const float*)(lds + L::kUp))[col];
#pragma unroll
        for (int t = 0; t < 4; ++t) st[t] *= up;
      }
      v2i cv[D / 16];
#pragma unroll
      for (int i = 0; i < D / 16; ++i) cv[i] = __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_v2i*)(vt + v_at(key, i >> 1) + (i & 1) * 8));
      // ---- probabilities, then weights, in pairs (2 u, 2 u + 1) of tiles as the codes' halves come
      h8 p[2];
      float sum, added;
      auto weigh = [&](auto masked_, auto bounded_) __attribute__((always_inline)) {
        constexpr bool MASKED = decltype(masked_)::value, BOUNDED = decltype(bounded_)::value;
        sum = added = 0.f;
        const int left = MASKED ? opaque((int)(slot - tile * kTileKeys) - 4 * kb) : 0;   // the last of the lane's keys there is
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const v4i k0 = *(const v4i*)(ks + 32 * u + 4 * kb), k1 = *(const v4i*)(ks + 32 * u + 16 + 4 * kb);
          const v4i v2 = *(const v4i*)(vs + 16 * u + 4 * kb);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int a0 = k0[i], a1 = k1[i], vv = v2[i];
            float p0 = __builtin_fmaf(st[2 * u][i], __int_as_float(a0), -ref), p1 = __builtin_fmaf(st[2 * u + 1][i], __int_as_float(a1), -ref);
            if constexpr (BOUNDED) p0 = bounded(p0, (unsigned)vv), p1 = bounded(p1, (unsigned)vv >> 16);
            p0 = __builtin_amdgcn_exp2f(p0), p1 = __builtin_amdgcn_exp2f(p1);
            if constexpr (MASKED) {                    // (scales behind the sequence come as zeros: so do the weights)
              if (32 * u + i > left) p0 = 0.f;
              if (32 * u + 16 + i > left) p1 = 0.f;
            }
            const h2 w2 = pair_times_halves(p0, (unsigned)vv & 0xFFFFu, p1, (unsigned)vv >> 16);
            sum += p0 + p1;
            p[u][2 * i] = w2[0], p[u][2 * i + 1] = w2[1];
            added = __builtin_amdgcn_fdot2(w2, h2{(_Float16)1.0f, (_Float16)1.0f}, added, false);
          }
        }
      };
      // A reference that holds the largest weight back, p vs < 2^12 when it is set, in the first tile and again where a weight leaves fp16's range,
      // which few tiles' do
      for (;;) {
        if (set_reference) {
          float top = -INFINITY;
          const int left = opaque((int)(slot - tile * kTileKeys) - 4 * kb);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const v4i k0 = *(const v4i*)(ks + 32 * u + 4 * kb), k1 = *(const v4i*)(ks + 32 * u + 16 + 4 * kb);
            const v4i v2 = *(const v4i*)(vs + 16 * u + 4 * kb);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int a0 = k0[i], a1 = k1[i], vv = v2[i];
              const float y0 = __builtin_fmaf(st[2 * u][i], __int_as_float(a0), exponent_of((unsigned)vv));
              const float y1 = __builtin_fmaf(st[2 * u + 1][i], __int_as_float(a1), exponent_of((unsigned)vv >> 16));
              top = __builtin_fmaxf(top, __builtin_fmaxf(32 * u + i > left ? -INFINITY : y0, 32 * u + 16 + i > left ? -INFINITY : y1));
            }
          }
          top = __builtin_fmaxf(top, lane_xor_f<16>(top));
          top = __builtin_fmaxf(top, lane_xor_f<32>(top));
          const float now = __builtin_fmaxf(ref, reference_for(top));
          const float alpha = __builtin_amdgcn_exp2f(ref - now);
          l *= alpha, weights *= alpha;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) o[i] *= alpha;
          ref = now;
        }
        if (last) weigh(std::true_type{}, std::false_type{});
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
      // ---- output: sixteen channels as rows; a lane's sixteen keys 16 t + 4 kb + i in nibble 4 t + i
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const int w8 = cv[i][u];
          o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(code_halves((unsigned)w8), p[u], o[i], 0, 0, 0);
        }
      if (++taken == kTakeOff) take_off(), taken = 0;
    }

    // ---- the waves' results into one piece
    l += lane_xor_f<16>(l);
    l += lane_xor_f<32>(l);
    take_off();
    wait_lds();
    float* const there = (float*)mine;                 // (its own stages: everything asked for has come)
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      v4f y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = o[i][e] * kFromSubnormal;
      *(v4f*)(there + col * L::kPitch + 16 * i + 4 * kb) = y;
    }
    if (kb == 0) there[col * L::kPitch + D] = ref, there[col * L::kPitch + D + 1] = l;
    __syncthreads();
    float* const piece = a.partials + ((size_t)(blockIdx.x + (size_t)place.b * shares.heads + unit) * kCols) * L::kPiece;
    for (uint32_t i = tid; i < cols * D; i += kThreads) {
      const uint32_t h = i / D, ch = i % D;
      float m = kLowestRef, w[kWaves], sum = 0.f, total = 0.f;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) m = __builtin_fmaxf(m, ((const float*)(lds + k * L::kWave))[h * L::kPitch + D]);
#pragma unroll
      for (int k = 0; k < kWaves; ++k) {
        const float* from = (const float*)(lds + k * L::kWave) + h * L::kPitch;
        w[k] = first + k < stop ? __builtin_amdgcn_exp2f(from[D] - m) : 0.f;
        total += first + k < stop ? w[k] * from[ch] : 0.f;
        sum += first + k < stop ? w[k] * from[D + 1] : 0.f;
      }
      piece[h * L::kPiece + ch] = total;
      if (ch == 0) piece[h * L::kPiece + D] = m, piece[h * L::kPiece + D + 1] = sum;
    }
    __syncthreads();
    pos += behind - entry;
  }
}

// n pieces, 4 K of them at a time: their references and sums one a lane, the weighted codes of every fourth one by this wave, all requested at once
// (what is behind the last one is its again, and taken with no weight: with a way out of the loop between them the loads came one after another, 7.0
// us in place of 3.9 for 59 pieces of 32 heads)
template <int D, int K>
__device__ __forceinline__ void join_pieces(const float* base, uint32_t n, int wave, float (&o)[D / 64], float& l) {
  constexpr size_t kStride = (size_t)kCols * (D + 2);
  const int lane = threadIdx.x & 63;
  float m = kLowestRef;
  for (uint32_t s0 = 0; s0 < n; s0 += 4 * K) {
    const bool have = lane < 4 * K && s0 + lane < n;
    const float* at = base + min(s0 + lane, n - 1) * kStride + D;
    const float pm = at[0], pl = at[1];
    float v[K][D / 64];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < D / 64; ++i) v[k][i] = base[min(s0 + wave + 4 * k, n - 1) * kStride + lane + 64 * i];
    const float now = __builtin_fmaxf(m, wave_max(have ? pm : kLowestRef)), old = __builtin_amdgcn_exp2f(m - now);
    const float w = have ? __builtin_amdgcn_exp2f(pm - now) : 0.f;
    l = l * old + (have ? w * pl : 0.f);
#pragma unroll
    for (int i = 0; i < D / 64; ++i) o[i] *= old;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float wk = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), wave + 4 * k));
#pragma unroll
      for (int i = 0; i < D / 64; ++i) o[i] += s0 + wave + 4 * k < n ? wk * v[k][i] : 0.f;
    }
    m = now;
  }
}

// one workgroup of four waves per (sequence, query head): every wave its share of the pieces, then the waves' sums in a fixed order
template <int D>
__global__ __launch_bounds__(256) void decode_i4_join_kernel(Decode a) {
  __shared__ float sums[4][D];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t b = blockIdx.x / a.Hq, hq = blockIdx.x % a.Hq;
  Shares shares(a);
  const Place place = shares.of(a, b);
  const uint32_t hkv = hq / a.rep, in_head = hq % a.rep, unit = hkv * a.blocks + in_head / kCols, h = in_head % kCols;
  float l = 0.f, o[D / 64] = {};
  if (place.tiles) {
    // (from the workgroup with its first tile on)
    const uint32_t start = place.before + unit * place.entries;
    const uint32_t g0 = (start + (shares.parts ? 0 : kHeadTiles)) / shares.c, n = (start + place.entries - 1) / shares.c - g0 + 1;
    const float* base = a.partials + ((size_t)(g0 + (size_t)b * shares.heads + unit) * kCols + h) * (D + 2);
    if (n <= 16) join_pieces<D, 4>(base, n, wave, o, l);
    else join_pieces<D, 16>(base, n, wave, o, l);
    l = wave_sum(l);
  }
#pragma unroll
  for (int i = 0; i < D / 64; ++i) sums[wave][lane + 64 * i] = o[i];
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    const int ch = lane + 64 * i;
    const float sum = (sums[0][ch] + sums[1][ch]) + (sums[2][ch] + sums[3][ch]);
    ((_Float16*)a.out)[(size_t)blockIdx.x * D + ch] = (_Float16)(place.tiles ? sum / l : 0.f);
  }
}

constexpr uint32_t kGroups = 512;                      // two workgroups on each compute unit
// Sequences of a pair of launches: each workgroup looks through the list of them, and one list for all takes time that grows with their square (8 heads
// of 64, 41 slots: 2048 sequences 479 us, 16384 22.8 ms, a million would take a minute and a half; 335 us and 2.8 ms in pairs of launches for 1024 each)
constexpr uint32_t kSequences = 1024;

uint32_t blocks_of(uint32_t rep) { return (rep + kCols - 1) / kCols; }

bool too_large(uint64_t B, uint64_t Hq, uint64_t Hkv, uint32_t head_dim, uint64_t max_len) {
  const uint64_t heads = B * Hkv * blocks_of((uint32_t)(Hq / Hkv));
  return B > 0x7FFFFFFFull || B * Hq > 0x7FFFFFull || heads > 0x7FFFFFull || max_len > (1u << 25) || heads * (max_len / kTileKeys + 1) > 0x7FFFFFFFull ||
         B * Hkv * max_len > 1ull << 40;
}

}  // namespace
}  // namespace flh

using namespace flh;

extern "C" size_t flh_decode_attention_i4_workspace_bytes(uint32_t B, uint32_t Hq, uint32_t Hkv, uint32_t head_dim, uint32_t max_len) {
  if (Hq == 0 || Hkv == 0 || Hq % Hkv || (head_dim != 128 && head_dim != 64) || max_len == 0 || too_large(B, Hq, Hkv, head_dim, max_len)) return 0;
  const uint64_t heads = (uint64_t)B * Hkv * blocks_of(Hq / Hkv);
  return (size_t)(kGroups + heads) * kCols * (head_dim + 2) * sizeof(float);
}

extern "C" int flh_decode_attention_rope_i4(const flh_half* q, const flh_half* k_new, const flh_half* v_new, const flh_half* cos,
                                            const flh_half* sin, const int64_t* lengths, uint8_t* k_codes, flh_half* k_scales,
                                            uint8_t* v_codes, flh_half* v_scales, flh_half* out, uint32_t B, uint32_t Hq, uint32_t Hkv,
                                            uint32_t head_dim, uint32_t max_len, float scale, void* workspace, size_t workspace_bytes,
                                            void* stream) {
  const char* what = "decode_attention (4-bit cache)";
  if (!q || !k_new || !v_new || !cos || !sin || !lengths || !k_codes || !k_scales || !v_codes || !v_scales || !out)
    return fail(FLH_EINVAL, "%s: null pointer", what);
  if (misaligned16(q, k_new, v_new, cos, sin, k_codes, v_codes, out)) return fail(FLH_EINVAL, "%s: tensors must be 16-byte aligned", what);
  if (head_dim != 128 && head_dim != 64) return fail(FLH_EINVAL, "%s: head_dim (%u) must be 64 or 128", what, head_dim);
  if (Hq == 0 || Hkv == 0 || Hq % Hkv) return fail(FLH_EINVAL, "%s: %u query heads do not divide over %u key / value heads", what, Hq, Hkv);
  if (max_len == 0) return fail(FLH_EINVAL, "%s: the caches have no slots", what);
  if (bad_scale(scale)) return fail(FLH_EINVAL, "%s: the scale must be positive and at most 1e15", what);
  if (B == 0) return FLH_OK;
  if (too_large(B, Hq, Hkv, head_dim, max_len)) return fail(FLH_EINVAL, "%s: problem too large", what);
  const size_t need = flh_decode_attention_i4_workspace_bytes(B, Hq, Hkv, head_dim, max_len);
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)
    return fail(FLH_EINVAL, "%s: a 16-byte aligned workspace of %zu bytes is required", what, need);
  const uint64_t slots = (uint64_t)B * Hkv * max_len, queries = (uint64_t)B * Hq * head_dim * 2, rows = (uint64_t)B * Hkv * head_dim * 2;
  const struct { const void* at; uint64_t bytes; } held[6] = {{k_codes, slots * (head_dim / 2)}, {k_scales, slots * 2}, {v_codes, slots * (head_dim / 2)},
                                                              {v_scales, slots * 2}, {workspace, need}, {out, queries}},
      in[6] = {{k_new, rows}, {v_new, rows}, {cos, (uint64_t)B * head_dim * 2}, {sin, (uint64_t)B * head_dim * 2}, {lengths, (uint64_t)B * 8}, {q, queries}};
  for (int i = 0; i < 6; ++i) {
    for (int j = 0; j < i; ++j)
      if (overlap(held[i].at, held[i].bytes, held[j].at, held[j].bytes)) return fail(FLH_EINVAL, "%s: outputs, caches or workspace share memory", what);
    // (the joining launch alone writes `out`, behind everything that reads the queries, keys and values; it reads the lengths itself)
    // (of large batches, in its own pair of launches: the queries' own place will do)
    for (int j = 0; j < 6; ++j)
      if (overlap(held[i].at, held[i].bytes, in[j].at, in[j].bytes) && (i < 5 || j == 4 || (B > kSequences && !(j == 5 && out == q))))
        return fail(FLH_EINVAL, "%s: an output shares memory with an input", what);
  }
  Decode a = {};
  a.partials = (float*)workspace;
  a.Hq = Hq, a.Hkv = Hkv, a.rep = Hq / Hkv, a.blocks = blocks_of(a.rep), a.max_len = max_len;
  a.scale_log2 = scale * 1.4426950408889634f;
  auto go = [&](auto kern, auto join, size_t smem, LdsGrant& grant) {
    if (int rc = reserve_lds((const void*)kern, smem, grant, what)) return rc;
    for (uint32_t done = 0; done < B; done += a.B) {   // (launches of a stream run in order: the pieces are joined before the next ones are written)
      const size_t q_at = (size_t)done * Hq * head_dim, new_at = (size_t)done * Hkv * head_dim, row = (size_t)done * Hkv * max_len;
      a.B = B - done < kSequences ? B - done : kSequences;
      a.q = (const __half*)q + q_at, a.k_new = (const __half*)k_new + new_at, a.v_new = (const __half*)v_new + new_at;
      a.cos = (const __half*)cos + (size_t)done * head_dim, a.sin = (const __half*)sin + (size_t)done * head_dim;
      a.lengths = (const long long*)lengths + done, a.out = (__half*)out + q_at;
      a.k_codes = k_codes + row * (head_dim / 2), a.v_codes = v_codes + row * (head_dim / 2);
      a.k_scales = (__half*)k_scales + row, a.v_scales = (__half*)v_scales + row;
      const uint64_t most = (uint64_t)a.B * Hkv * a.blocks * ((max_len - 1) / kTileKeys + 1);
      a.groups = (uint32_t)(most < kGroups ? most : kGroups);
      hipLaunchKernelGGL(kern, dim3(a.groups), dim3(kThreads), smem, (hipStream_t)stream, a);
      if (int rc = check_launch(what)) return rc;
      hipLaunchKernelGGL(join, dim3(a.B * Hq), dim3(256), 0, (hipStream_t)stream, a);
      if (int rc = check_launch(what)) return rc;
    }
    return FLH_OK;
  };
  static LdsGrant grant128, grant64;
  return head_dim == 128 ? go(decode_i4_kernel<128>, decode_i4_join_kernel<128>, Layout<128>::kBytes, grant128)
                         : go(decode_i4_kernel<64>, decode_i4_join_kernel<64>, Layout<64>::kBytes, grant64);
}
