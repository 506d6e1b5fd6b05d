// Causal attention of a block of T new tokens per sequence over a key / value cache held in 4 bits (cache_i4.h) that holds them already: token
// t sits in slot lengths[b] + t and sees the slots up to its own.  Queries as the cache's writer leaves them (rotated like the keys), token-major
// [B, T, Hq, D]; output [B, T, Hq * D].
//
// The rows of a key / value head are its T x rep queries, token by token: one workgroup = 4 waves = 128 of them, 32 per wave, so that heads that
// share keys share the work of bringing them.  Both products run on v_mfma_f32_32x32x16_f16 in transposed form (a lane owns one query):
//
//   S^T[key, query] = sum_d ck[key, d] Q[query, d]      O^T[d, query] += sum_key cv[key, d] (p vs)[query, key]
//
// with the codes as they are held (code_halves), keys' scales multiplied into the scores and values' into the probabilities.  Tiles of 64 keys,
// three in LDS as packed codes (8 KiB each) by direct-to-LDS loads; values are transposed by the LDS load for 4 bits.
//
// Few rows: the tiles of a block are split over several workgroups, whose pieces (reference, sum, weighted codes) a second launch joins.
#include "cache_i4.h"

namespace flh {
namespace {

constexpr int kThreads = 256, kBlockRows = 128, kStages = 3;

struct Prefill {
  const __half* q;
  const long long* lengths;
  const uint8_t *k_codes, *v_codes;
  const __half *k_scales, *v_scales;
  __half* out;
  float* pieces;
  uint32_t B, T, Hq, Hkv, rep, max_len, rows, blocks, splits;   // rows of a key / value head, blocks of 128 of them
  float scale_log2;
};

// floats of a piece: 128 rows of D sums, their references and sums of exponentials
template <int D>
constexpr uint32_t kPieceFloats = kBlockRows * (D + 2);

template <int D>
struct Layout {
  static constexpr int kRowBytes = D / 2, kTile = kTileKeys * kRowBytes, kStage = 2 * kTile + 2 * kTileKeys * 4;
  static constexpr int kOutPitch = D * 2 + 16;
  static constexpr int kBig = kStages * kStage, kBytes0 = kBig + 16;
  static constexpr int kBytes = kBytes0 > kBlockRows * kOutPitch ? kBytes0 : kBlockRows * kOutPitch;
};

template <int D>
__global__ __launch_bounds__(kThreads, 2) void prefill_i4_kernel(Prefill a) {
  using L = Layout<D>;
  extern __shared__ __align__(1024) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned lds0 = (unsigned)(size_t)lds;
  // every die takes a contiguous range of (sequence, key / value head) pairs; within one the long blocks (late queries) come first
  const unsigned w = xcd_contiguous(blockIdx.x, gridDim.x);
  const uint32_t split = w % a.splits, block = a.blocks - 1 - w / a.splits % a.blocks, bh = w / a.splits / a.blocks;
  const uint32_t b = bh / a.Hkv, hkv = bh % a.Hkv;
  const long long len = a.lengths[b];
  const bool takes_part = len >= 0 && len <= (long long)a.max_len - (long long)a.T;
  const uint32_t length = takes_part ? (uint32_t)len : 0u;

  const uint32_t first_row = block * kBlockRows + wave * 32;
  const uint32_t row = min(first_row + n, a.rows - 1);                 // (rows past the end repeat the last one; never stored)
  const uint32_t t = row / a.rep, head = hkv * a.rep + row % a.rep;
  const size_t q_at = (((size_t)b * a.T + t) * a.Hq + head) * D;
  const int limit = (int)(length + t);                                 // the last slot that the lane's query sees
  const uint32_t last_row = min(block * kBlockRows + kBlockRows, a.rows) - 1;
  const uint32_t slots = length + last_row / a.rep + 1;                // slots that any query of the block sees
  const uint32_t all_tiles = takes_part ? (slots + kTileKeys - 1) / kTileKeys : 0;
  const uint32_t tile0 = (uint32_t)((uint64_t)all_tiles * split / a.splits), tile1 = (uint32_t)((uint64_t)all_tiles * (split + 1) / a.splits);
  // tiles with a slot that some query of the wave sees
  const uint32_t wave_slots = length + min(first_row + 31, a.rows - 1) / a.rep + 1;
  const uint32_t live = __builtin_amdgcn_readfirstlane(first_row < a.rows ? (wave_slots + kTileKeys - 1) / kTileKeys : 0);
  const uint32_t whole = __builtin_amdgcn_readfirstlane((length + min(first_row, a.rows - 1) / a.rep + 1) / kTileKeys);   // tiles all of them see whole

  const v4i k_rows = buffer_of(a.k_codes + (size_t)bh * a.max_len * L::kRowBytes, slots * L::kRowBytes);
  const v4i v_rows = buffer_of(a.v_codes + (size_t)bh * a.max_len * L::kRowBytes, slots * L::kRowBytes);
  const v4i k_sc = buffer_of((const uint8_t*)(a.k_scales + (size_t)bh * a.max_len), slots * 2);
  const v4i v_sc = buffer_of((const uint8_t*)(a.v_scales + (size_t)bh * a.max_len), slots * 2);

  // codes: 1 KiB a load, wave w takes its 16 rows of either (D = 64: 32 rows, two waves for keys, two for values); chunks of sixteen bytes are
  // permuted so that neither the rows of a score operand nor the sixteen keys of a transpose load fall on the same banks
  unsigned k_src, v_src;
  if constexpr (D == 128) {
    k_src = wave * 1024 + (lane >> 2) * 64 + (((lane & 3) ^ (lane >> 4)) << 4);
    v_src = wave * 1024 + (lane >> 2) * 64 + (((lane & 3) ^ ((2 * wave + (lane >> 5)) & 3)) << 4);
  } else {
    k_src = v_src = (wave & 1) * 1024 + (lane >> 1) * 32 + (((lane & 1) ^ ((lane >> 4) & 1)) << 4);
  }
  auto k_at = [](int r, int c) { return D == 128 ? r * 64 + ((c ^ ((r >> 2) & 3)) << 4) : r * 32 + ((c ^ ((r >> 3) & 1)) << 4); };
  auto v_at = [](int r, int c) { return D == 128 ? r * 64 + ((c ^ ((r >> 3) & 3)) << 4) : r * 32 + ((c ^ ((r >> 3) & 1)) << 4); };
  auto request = [&](uint32_t tile, uint32_t stage) {
    const unsigned to = lds0 + stage * L::kStage, from = tile * L::kTile;
    if constexpr (D == 128) {
      rows_to_lds(k_rows, from + k_src, to + wave * 1024);
      rows_to_lds(v_rows, from + v_src, to + L::kTile + wave * 1024);
    } else {
      if (wave < 2) rows_to_lds(k_rows, from + k_src, to + wave * 1024);
      else rows_to_lds(v_rows, from + v_src, to + L::kTile + (wave - 2) * 1024);
    }
    if (wave == 0) halves_to_lds(k_sc, (tile * kTileKeys + lane) * 2, to + 2 * L::kTile);
    if (wave == 1) halves_to_lds(v_sc, (tile * kTileKeys + lane) * 2, to + 2 * L::kTile + kTileKeys * 4);
  };
  // the exponent of a tile's largest value scale, into LDS by one wave, a step ahead of its use
  float* const bigs = (float*)(lds + L::kBig);
  auto find_big = [&](uint32_t stage, uint32_t slot_of_it) {
    const unsigned v = *(const unsigned*)(lds + stage * L::kStage + 2 * L::kTile + kTileKeys * 4 + lane * 4) & 0x7FFFu;
    const float e = wave_max((float)(min(v, 0x7C00u) >> 10));
    if (lane == 0) bigs[slot_of_it] = e - 29.0f;
  };

  // this lane's query as operand: half h holds the channels of its half of a row's bytes, eight a step
  constexpr int kSteps = D / 16;
  h8 qf[kSteps];
  float factor, bias;
  {
    const __half* src = a.q + q_at + h * (D / 2);
    h8 x[kSteps];
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      x[j] = *(const h8*)(src + 8 * j);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, (unsigned)__float_as_int((float)x[j][e]) & 0x7FFFFFFFu);
    }
    top = max(top, (unsigned)lane_xor_i<32>((int)top));
    // largest between 2^8 and 2^9 (a power of two: exact)
    const unsigned e2 = min(254u, 262u - (top >> 23));
    const float f = __int_as_float((int)(e2 << 23));
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < kSteps; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const _Float16 y = (_Float16)((float)x[j][e] * f);
        qf[j][code_element(e)] = y;
        sum += (float)y;
      }
    sum += lane_xor_f<32>(sum);
    bias = -8.0f / kFromSubnormal * sum;
    factor = __builtin_fmaxf(__int_as_float((int)((254u - e2) << 23)) * kFromSubnormal * a.scale_log2, 1e-37f);   // (never zero: it meets -inf)
  }

  v16f o[D / 32], ob;
#pragma unroll
  for (int r = 0; r < 16; ++r) ob[r] = 0.f;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) o[i] = ob;
  float ref = kLowestRef, l = 0.f;

  if (tile0 < tile1) {
    request(tile0, 0);
    if (tile0 + 1 < tile1) request(tile0 + 1, 1);
    wait_vmcnt<0>();
    __syncthreads();
    if (wave == 2) find_big(0, 0);
  }
  uint32_t stage = 0;
  for (uint32_t tile = tile0; tile < tile1; ++tile) {
    wait_vmcnt<0>();
    __syncthreads();   // this tile and the next have come, everybody is done with the one before
    const uint32_t next = stage == 2 ? 0 : stage + 1, third = next == 2 ? 0 : next + 1;
    if (tile + 2 < tile1) request(tile + 2, third);
    if (tile + 1 < tile1 && wave == 2) find_big(next, (tile + 1 - tile0) & 1);
    const uint8_t* const kt = lds + stage * L::kStage;
    const uint8_t* const vt = kt + L::kTile;
    const unsigned* const ks = (const unsigned*)(vt + L::kTile);
    const unsigned* const vs = ks + kTileKeys;
    stage = next;
    if (tile >= live) continue;
    // ---- scores of two tiles of 32 keys: element r of tile kt: key 32 kt + 8 (r / 4) + 4 h + r % 4
    v16f st[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int r = 0; r < 16; ++r) st[i][r] = bias;
      unsigned c[kSteps];
#pragma unroll
      for (int j = 0; j < kSteps / 4; ++j) *(v4i*)(c + 4 * j) = *(const v4i*)(kt + k_at(32 * i + n, h * (kSteps / 4) + j));
#pragma unroll
      for (int j = 0; j < kSteps; ++j) st[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(code_halves(c[j]), qf[j], st[i], 0, 0, 0);
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const v4i k4 = *(const v4i*)(ks + 32 * i + 8 * g + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) st[i][4 * g + e] = times_half(st[i][4 * g + e], (unsigned)k4[e]);
      }
    const bool masked = tile >= whole;
    const int key0 = (int)(tile * kTileKeys) + 4 * h;
    if (masked) {
      asm volatile("" ::: "memory");
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (key0 + 32 * i + 8 * (r >> 2) + (r & 3) > limit) st[i][r] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = __builtin_fmaxf(top, st[i][r]);
    top = __builtin_fmaxf(top, lane_xor_f<32>(top));
    const float now = __builtin_fmaxf(ref, __builtin_fmaf(top, factor, bigs[(tile - tile0) & 1]));
    if (__builtin_amdgcn_ballot_w64(now != ref) != 0) {
      const float alpha = __builtin_amdgcn_exp2f(ref - now);
      l *= alpha;
      ob *= alpha;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) o[i] *= alpha;
      ref = now;
    }
    // ---- probabilities with the values' scales, in pairs (r, r + 4) as the codes' halves come: p[i][u] is slots 16 u .. of tile i
    h8 p[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const v4i v0 = *(const v4i*)(vs + 32 * i + 16 * u + 4 * h), v1 = *(const v4i*)(vs + 32 * i + 16 * u + 8 + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(st[i][8 * u + e], factor, -ref));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(st[i][8 * u + 4 + e], factor, -ref));
          l += p0 + p1;
          const h2 x = pair_times_halves(p0, (unsigned)v0[e], p1, (unsigned)v1[e]);
          p[i][u][2 * e] = x[0], p[i][u][2 * e + 1] = x[1];
        }
      }
    if (masked) {      // (a value that a query does not see may be NaN)
      asm volatile("" ::: "memory");
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (key0 + 32 * i + 8 * (r >> 2) + (r & 3) > limit) p[i][r >> 3][2 * (r & 3) + ((r >> 2) & 1)] = (_Float16)0.0f;
    }
    // ---- output: 32 channels as rows; the lane's sixteen keys 8 (r / 4) + 4 h + r % 4 of a tile of 32 in nibble r
    const int g = lane >> 4, gi = lane & 15;
    const int key = 8 * (gi >> 2) + 4 * (g >> 1) + (gi & 3);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int u = 0; u < 2; ++u) ob = __builtin_amdgcn_mfma_f32_32x32x16_f16(bias_halves(), p[i][u], ob, 0, 0, 0);
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) {
        const v2i c = __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_v2i*)(vt + v_at(32 * i + key, dt) + (g & 1) * 8));
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(code_halves((unsigned)c[0]), p[i][0], o[dt], 0, 0, 0);
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(code_halves((unsigned)c[1]), p[i][1], o[dt], 0, 0, 0);
      }
    }
  }

  l += lane_xor_f<32>(l);
  if (a.splits > 1) {
    float* piece = a.pieces + (((size_t)bh * a.blocks + block) * a.splits + split) * kPieceFloats<D>;
    const uint32_t r0 = wave * 32 + n;
    if (first_row + n < a.rows) {
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          v4f x;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = (o[dt][4 * g + e] - ob[4 * g + e]) * kFromSubnormal;
          *(v4f*)(piece + r0 * D + 32 * dt + 8 * g + 4 * h) = x;
        }
      if (h == 0) piece[kBlockRows * D + r0] = ref, piece[kBlockRows * (D + 1) + r0] = l;
    }
    return;
  }
  // ---- normalise, transpose through LDS, store whole rows (none for a sequence that takes no part: zeros)
  const float inv = takes_part ? kFromSubnormal / l : 0.f;
  __syncthreads();
  uint8_t* stage_out = lds + wave * (32 * L::kOutPitch);
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      h4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (_Float16)((o[dt][4 * g + e] - ob[4 * g + e]) * inv);
      *(h4*)(stage_out + n * L::kOutPitch + (32 * dt + 8 * g + 4 * h) * 2) = v;
    }
  wait_lgkmcnt0();
  __builtin_amdgcn_wave_barrier();
  constexpr int kChunks = D / 8, kPerLoad = 64 / kChunks;
#pragma unroll
  for (int it = 0; it < 32 / kPerLoad; ++it) {
    const uint32_t r = it * kPerLoad + lane / kChunks, c = lane % kChunks, global = first_row + r;
    const v4i v = *(const v4i*)(stage_out + r * L::kOutPitch + c * 16);
    if (global < a.rows)
      *(v4i*)(a.out + (((size_t)b * a.T + global / a.rep) * a.Hq + hkv * a.rep + global % a.rep) * D + c * 8) = v;
  }
}

// one wave per row: its pieces in their order
template <int D>
__global__ __launch_bounds__(256) void prefill_i4_join_kernel(Prefill a) {
  const int lane = threadIdx.x & 63;
  const uint64_t item = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (item >= (uint64_t)a.B * a.Hkv * a.rows) return;
  const uint32_t bh = (uint32_t)(item / a.rows), row = (uint32_t)(item % a.rows), b = bh / a.Hkv, hkv = bh % a.Hkv;
  const uint32_t block = row / kBlockRows, r0 = row % kBlockRows;
  const long long len = a.lengths[b];
  const bool takes_part = len >= 0 && len <= (long long)a.max_len - (long long)a.T;
  float m = kLowestRef, l = 0.f, o[D / 64] = {};
  const float* base = a.pieces + ((size_t)bh * a.blocks + block) * a.splits * kPieceFloats<D>;
  for (uint32_t s = 0; s < a.splits; ++s) {
    const float* piece = base + (size_t)s * kPieceFloats<D>;
    const float pm = piece[kBlockRows * D + r0], pl = piece[kBlockRows * (D + 1) + r0];
    if (pl == 0.f) continue;                           // nothing of it is seen
    const float now = __builtin_fmaxf(m, pm);
    const float old = __builtin_amdgcn_exp2f(m - now), w = __builtin_amdgcn_exp2f(pm - now);
    l = l * old + w * pl;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) o[i] = o[i] * old + w * piece[r0 * D + lane + 64 * i];
    m = now;
  }
  __half* dst = a.out + (((size_t)b * a.T + row / a.rep) * a.Hq + hkv * a.rep + row % a.rep) * D;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) ((_Float16*)dst)[lane + 64 * i] = (_Float16)(takes_part ? o[i] / l : 0.f);
}

// Workgroups over which a block's tiles are split: as many as fill the chip, two a compute unit
uint32_t splits_of(uint64_t groups, uint32_t max_len) {
  const uint64_t tiles = ((uint64_t)max_len + kTileKeys - 1) / kTileKeys;
  uint64_t s = 512 / groups;
  if (s > 16) s = 16;
  if (s > tiles) s = tiles;
  return s < 1 ? 1 : (uint32_t)s;
}

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
  const uint64_t groups = (uint64_t)B * Hkv * blocks_of(T, Hq / Hkv);
  const uint32_t splits = splits_of(groups, max_len);
  return splits == 1 ? 0 : (size_t)(groups * splits) * kBlockRows * (head_dim + 2) * sizeof(float);
}

extern "C" int flh_prefill_attention_i4(const flh_half* q, const int64_t* lengths, const uint8_t* k_codes, const flh_half* k_scales,
                                        const uint8_t* v_codes, const flh_half* v_scales, flh_half* out, uint32_t B, uint32_t T, uint32_t Hq,
                                        uint32_t Hkv, uint32_t head_dim, uint32_t max_len, float scale, void* workspace,
                                        size_t workspace_bytes, void* stream) {
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
  const struct { const void* at; uint64_t bytes; } in[6] = {{k_codes, slots * (head_dim / 2)}, {k_scales, slots * 2}, {v_codes, slots * (head_dim / 2)},
                                                            {v_scales, slots * 2}, {lengths, (uint64_t)B * 8}, {q, queries}};
  for (const auto& x : in)
    if (overlap(out, queries, x.at, x.bytes) || overlap(workspace, need, x.at, x.bytes))
      return fail(FLH_EINVAL, "%s: an output shares memory with an input", what);
  if (overlap(out, queries, workspace, need)) return fail(FLH_EINVAL, "%s: the output shares memory with the workspace", what);
  Prefill a = {};
  a.q = (const __half*)q, a.lengths = (const long long*)lengths, a.k_codes = k_codes, a.v_codes = v_codes;
  a.k_scales = (const __half*)k_scales, a.v_scales = (const __half*)v_scales, a.out = (__half*)out, a.pieces = (float*)workspace;
  a.B = B, a.T = T, a.Hq = Hq, a.Hkv = Hkv, a.rep = Hq / Hkv, a.max_len = max_len, a.rows = T * a.rep, a.blocks = (uint32_t)blocks_of(T, a.rep);
  a.scale_log2 = scale * 1.4426950408889634f;
  const uint64_t groups = (uint64_t)B * Hkv * a.blocks;
  a.splits = splits_of(groups, max_len);
  auto go = [&](auto kern, auto join, size_t smem, LdsGrant& grant) {
    if (int rc = reserve_lds((const void*)kern, smem, grant, what)) return rc;
    hipLaunchKernelGGL(kern, dim3((unsigned)(groups * a.splits)), dim3(kThreads), smem, (hipStream_t)stream, a);
    if (int rc = check_launch(what)) return rc;
    if (a.splits == 1) return FLH_OK;
    hipLaunchKernelGGL(join, dim3((unsigned)(((uint64_t)B * Hkv * a.rows + 3) / 4)), dim3(256), 0, (hipStream_t)stream, a);
    return check_launch(what);
  };
  static LdsGrant grant128, grant64;
  return head_dim == 128 ? go(prefill_i4_kernel<128>, prefill_i4_join_kernel<128>, Layout<128>::kBytes, grant128)
                         : go(prefill_i4_kernel<64>, prefill_i4_join_kernel<64>, Layout<64>::kBytes, grant64);
}
