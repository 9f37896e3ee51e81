// Paged attention with masked and shaped scores: scores capped by a tanh, a bias that falls with distance, a sliding
// window, a prefix that every query of a sequence sees, and a first token per query (documents packed into a sequence).
//
// Row r = (query i, head h G + g) of KV head h sits at position p = len - Q + i. It sees token j of its sequence when
//   j < len  and  (j < prefix  or  (max(start_i, p - window + 1) <= j <= p)),
// and with t = sm_scale q.k its score is t, or cap tanh(t / cap), less slope_h |p - j|. Scores are held in float32 in units
// of log2 e, so that weights are 2^(score - max); with E = 2^(2 log2e t / cap) the cap is A - 2 A / (1 + E), A = cap log2e.
// That form loses about A 2^-23 absolutely, 7e-5 of a weight at the largest cap that uses it (kMaskedPlainCap); beyond, small
// arguments take tanh's series.
//
// Products run on the matrix cores in bf16, transposed: S^T (16 tokens x 16 rows) = K Q^T, O^T (16 channels x 16 rows) +=
// V^T P^T. All three formats' codes are exact in bf16 (8 significant bits); an f16 q is split into two bf16 parts (exact) and
// the weights into two (16 bits: a weight's error is 2^-17, under the 2^-12 of an f16 output's half step). In the
// 16x16x32 layout a lane holds row n = lane % 16 and, with g = lane / 16, the scores of tokens 4 g + i and 16 + 4 g + i of 32;
// they are taken as elements 8 g + e of the second product's contraction, so weights never leave their lane. A V operand
// then needs 8 tokens of one channel per lane: a lane loads 8 channels (8 lane % 16 ..) of its 8 tokens, whole rows by 16
// lanes, and transposes them in registers. Output channel 8 (4 g + i) + c of row n is element i of O^T's block c.
//
// Work is cut into steps of 32 tokens; a tile (rows of one (sequence, KV head)) lists the steps that some row of it sees:
// those of the prefix, then those from its lowest first token to its last position. Steps are dealt out in pieces of a fixed
// number of steps, one per workgroup: ragged batches balance by themselves, and windows cost no launch over the tokens
// before them. The pieces of a tile meet in float32 partials, which the last workgroup to arrive combines in order.
//
// Two kernels:
//  * few rows (up to 48 of a KV head, in tiles of 16): the waves of a workgroup take steps in turn, straight from memory into
//    registers (keys on through LDS), and merge through LDS at the end. Bound by the cache's bytes, short calls by the latency
//    of a piece: FP8, 32 sequences of 256 to 4096 tokens, 8 KV heads, 37.8 us (143 MB, 3.8 TB/s); a window of 4096 of 32768
//    tokens, 8 sequences, 21 us.
//  * many rows: a workgroup's four waves hold 64 or 128 rows; each of two steps' keys and values is loaded and converted by
//    one wave and read by all from LDS, where operands lie in the order lanes take them (no bank conflicts, no swizzle).
//    Bound by the vector units, about 16 operations and 3 transcendentals (a quarter of the rate) a score: BF16, 2048 queries
//    after 2049 tokens, 16 heads on 8, capped, window 2500, 113 us (41 GFLOP).
//
// Tokens a row does not see must add nothing to it, but 0 times an infinity is a NaN: a wave whose result is not finite does
// its piece again with values that are not finite taken out of the products and added one by one to the rows that see them.
// Finite data pays one look at the result.
#pragma once

#include <type_traits>

#include "decode_common.h"

namespace bpt {

typedef __bf16 mbf16x8 __attribute__((ext_vector_type(8)));
typedef float mf32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t mu32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t mu32x4 __attribute__((ext_vector_type(4)));

constexpr int kMaskedStep = 32;
constexpr int kMaskedRowPad = kHeadDim + 4;  // floats of a row in LDS: 16 rows spread over the banks
constexpr int kMaskedItem = 8 * 64;  // 16-byte units of one step's K or V operands in LDS
constexpr float kMaskedSlack = 8.0f;  // a row's reference point may lag its maximum by this (log2): weights stay below 2^8

// ---- conversions ------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t masked_fp8_pair(uint32_t w, bool high) {
  return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
}
// Four int8 codes -> bf16, through float32 (exact).
__device__ __forceinline__ mu32x2 masked_int8x4(uint32_t w) {
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = (float)(int8_t)((w >> (8 * i)) & 0xffu);
  return mu32x2{__builtin_amdgcn_perm(__float_as_uint(f[1]), __float_as_uint(f[0]), 0x07060302u),
                __builtin_amdgcn_perm(__float_as_uint(f[3]), __float_as_uint(f[2]), 0x07060302u)};
}
// Eight codes (two dwords) -> bf16.
template <int KV>
__device__ __forceinline__ mu32x4 masked_codes8(uint32_t w0, uint32_t w1) {
  if constexpr (KV == kKvFp8) {
    return mu32x4{masked_fp8_pair(w0, false), masked_fp8_pair(w0, true), masked_fp8_pair(w1, false), masked_fp8_pair(w1, true)};
  } else {
    const mu32x2 a = masked_int8x4(w0), b = masked_int8x4(w1);
    return mu32x4{a.x, a.y, b.x, b.y};
  }
}
// 4 x 4 byte transpose: w[i] byte j -> out[j] byte i.
__device__ __forceinline__ void masked_transpose4(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t* o) {
  const uint32_t t0 = __builtin_amdgcn_perm(w1, w0, 0x05010400u), t1 = __builtin_amdgcn_perm(w3, w2, 0x05010400u);
  const uint32_t t2 = __builtin_amdgcn_perm(w1, w0, 0x07030602u), t3 = __builtin_amdgcn_perm(w3, w2, 0x07030602u);
  o[0] = __builtin_amdgcn_perm(t1, t0, 0x05040100u);
  o[1] = __builtin_amdgcn_perm(t1, t0, 0x07060302u);
  o[2] = __builtin_amdgcn_perm(t3, t2, 0x05040100u);
  o[3] = __builtin_amdgcn_perm(t3, t2, 0x07060302u);
}
// Two bf16 values with those that are not finite replaced by zeros.
__device__ __forceinline__ uint32_t masked_finite2(uint32_t x) {
  if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u;
  if ((x & 0x7f800000u) == 0x7f800000u) x &= 0xffffu;
  return x;
}
__device__ __forceinline__ mf32x4 masked_mfma(mu32x4 a, mu32x4 b, mf32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mbf16x8, a), __builtin_bit_cast(mbf16x8, b), c, 0, 0, 0);
}

// ---- one step's codes -------------------------------------------------------------------------------------------

template <int KV>
struct MaskedRaw {
  static constexpr int kWords = KV == kKvBf16 ? 32 : 16;
  uint32_t w[kWords];
};

// The pages of a step's two 16-token groups, for page sizes of at least 16.
struct MaskedPages {
  int e[2];
};
__device__ __forceinline__ int masked_clamp_page(const MaskedParams& p, int e) {
  return e < 0 ? 0 : (e >= p.num_blocks ? p.num_blocks - 1 : e);
}
// Byte offset of a token's row of head h in the pools (any page size). Tokens past the last one read it instead.
__device__ __forceinline__ int64_t masked_row(const MaskedParams& p, int b, int h, int token, int len) {
  const int tok = min(token, len - 1);
  const int e = masked_clamp_page(p, ((const int32_t*)p.table)[((int64_t)b * p.table_sb + (tok >> p.logP)) << p.table_i64]);
  return (int64_t)e * p.kv_sblk + (int64_t)(tok & (p.P - 1)) * p.kv_stok + (int64_t)h * p.kv_shead;
}
// Where a step's two 16-token groups lie (pages of at least 16 tokens): byte offsets of their first rows, and from there of the
// last row that holds a token of the sequence, up to which the others are cut. A group behind the sequence reads the first one.
struct MaskedSpot {
  int64_t base[2];
  uint32_t last[2];
  int page[2], rows[2];  // the page, and the last row's number
};
template <bool PU>
__device__ __forceinline__ MaskedSpot masked_spot(const MaskedParams& p, int h, MaskedPages pages, int token0, int len) {
  MaskedSpot s{};
  if constexpr (PU) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const bool in = token0 + 16 * t < len;
      const int token = in ? token0 + 16 * t : token0;
      s.page[t] = masked_clamp_page(p, in ? pages.e[t] : pages.e[0]);
      s.rows[t] = min(len - 1 - token, 15);
      s.base[t] = (int64_t)s.page[t] * p.kv_sblk + (int64_t)(token & (p.P - 1)) * p.kv_stok + (int64_t)h * p.kv_shead;
      s.last[t] = (uint32_t)s.rows[t] * (uint32_t)p.kv_stok;
    }
  }
  return s;
}

// ONCE: read by this workgroup alone (past the caches), else by the other tiles of the head too.
template <int W, bool ONCE>
__device__ __forceinline__ void masked_load(const uint8_t* src, uint32_t* w) {
  typedef uint32_t words __attribute__((ext_vector_type(W)));
  const words x = ONCE ? __builtin_nontemporal_load((const words*)src) : *(const words*)src;
#pragma unroll
  for (int i = 0; i < W; ++i) w[i] = x[i];
}

// Keys: whole rows, 16 bytes a lane (of codes, 8 lanes to a token and 8 tokens to a load; of bf16, 16 and 4), which the memory
// pipeline serves faster than the operands' own order. They get into that order through LDS.
template <int KV, bool PU, bool ONCE>
__device__ __forceinline__ void masked_issue_k(const MaskedParams& p, int b, int h, int token0, int len, const MaskedSpot& s, int lane,
                                               MaskedRaw<KV>& r) {
  constexpr int S = KV == kKvBf16 ? 16 : 8, PER = 64 / S;  // 16-byte segments of a row, rows of a load
  const int row = lane / S;
  const uint32_t x = 16 * (lane % S), stok = (uint32_t)p.kv_stok;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const uint32_t last = s.last[t] + x;
#pragma unroll
    for (int j = 0; j < 16 / PER; ++j) {
      const uint8_t* src = PU ? p.k + s.base[t] + min((uint32_t)(PER * j + row) * stok + x, last)
                              : p.k + masked_row(p, b, h, token0 + 16 * t + PER * j + row, len) + x;
      masked_load<4, ONCE>(src, r.w + 4 * (16 / PER * t + j));
    }
  }
}
// Values: lane (n, g) takes channels 8 n .. + 7 of tokens 4 g + i and 16 + 4 g + i.
template <int KV, bool PU, bool ONCE>
__device__ __forceinline__ void masked_issue_v(const MaskedParams& p, int b, int h, int token0, int len, const MaskedSpot& s, int lane,
                                               MaskedRaw<KV>& r) {
  constexpr int W = KV == kKvBf16 ? 4 : 2;
  const int g = lane >> 4;
  const uint32_t x = 4 * W * (lane & 15), stok = (uint32_t)p.kv_stok;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const uint32_t last = s.last[t] + x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* src = PU ? p.v + s.base[t] + min((uint32_t)(4 * g + i) * stok + x, last)
                              : p.v + masked_row(p, b, h, token0 + 16 * t + 4 * g + i, len) + x;
      masked_load<W, ONCE>(src, r.w + W * (4 * t + i));
    }
  }
}
// Per-token scales: lane l < 32 takes the key's scale of token l, the others the value's of token l - 32.
template <bool PU>
__device__ __forceinline__ float masked_issue_scale(const MaskedParams& p, int b, int h, int token0, int len, const MaskedSpot& s,
                                                    int lane) {
  const float* src = lane < 32 ? p.ks : p.vs;
  if constexpr (PU) {
    int64_t base[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
      base[t] = (int64_t)s.page[t] * p.sc_sblk + (int64_t)((token0 + 16 * t < len ? token0 + 16 * t : token0) & (p.P - 1)) * p.sc_stok +
                (int64_t)h * p.sc_shead;
    const int row = min(lane & 15, (lane & 16) ? s.rows[1] : s.rows[0]);
    return src[((lane & 16) ? base[1] : base[0]) + (uint32_t)row * (uint32_t)p.sc_stok];
  } else {
    const int tok = min(token0 + (lane & 31), len - 1);
    const int e = ((const int32_t*)p.table)[((int64_t)b * p.table_sb + (tok >> p.logP)) << p.table_i64];
    return src[(int64_t)masked_clamp_page(p, e) * p.sc_sblk + (int64_t)(tok & (p.P - 1)) * p.sc_stok + (int64_t)h * p.sc_shead];
  }
}

// Loaded key rows into LDS as the first product's operands: operand s of 16-token group t is 64 units of 16 bytes, unit 16 g + n
// for lane (n, g), from `dst` + 64 (4 t + s) on. Product s takes channels 32 s + 8 g .. + 7 of bf16 rows (segment 4 s + g), of codes
// 64 (s / 2) + 16 g + 8 (s % 2) .. + 7 (halves of segment 4 (s / 2) + g). Units are permuted within their eights by segment, so
// that the 8 lanes that store a row's segments, and the 8 that read one of 8 rows, touch all banks.
__device__ __forceinline__ int masked_k_unit(int t, int s, int g, int n, int twist) {
  return 64 * (4 * t + s) + ((16 * g + n) ^ (g + 4 * twist));
}
template <int KV>
__device__ __forceinline__ void masked_k_place(const MaskedRaw<KV>& r, int lane, mu32x4* dst) {
  constexpr int S = KV == kKvBf16 ? 16 : 8, PER = 64 / S;
  const int row = lane / S, seg = lane % S;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int j = 0; j < 16 / PER; ++j) {
      const uint32_t* w = r.w + 4 * (16 / PER * t + j);
      const int n = PER * j + row, g = seg & 3, s = seg >> 2;
      if constexpr (KV == kKvBf16) {
        dst[masked_k_unit(t, s, g, n, s & 1)] = mu32x4{w[0], w[1], w[2], w[3]};
      } else {
        dst[masked_k_unit(t, 2 * s, g, n, s)] = masked_codes8<KV>(w[0], w[1]);
        dst[masked_k_unit(t, 2 * s + 1, g, n, s)] = masked_codes8<KV>(w[2], w[3]);
      }
    }
}
template <int KV>
__device__ __forceinline__ mu32x4 masked_k_frag(const mu32x4* src, int t, int s, int lane) {
  return src[masked_k_unit(t, s, lane >> 4, lane & 15, KV == kKvBf16 ? s & 1 : s >> 1)];
}
// The same within one wave, which converts after reading: rows as loaded, segments permuted within their eights by row (the 8 lanes
// that store a row's segments, and the 8 that read one segment of 8 rows, touch all banks).
template <int KV>
__device__ __forceinline__ void masked_k_keep(const MaskedRaw<KV>& r, int lane, mu32x4* tile) {
  constexpr int S = KV == kKvBf16 ? 16 : 8, PER = 64 / S;
#pragma unroll
  for (int j = 0; j < 32 / PER; ++j) {
    const int row = PER * j + lane / S;
    tile[S * row + ((lane % S) ^ (row & 7))] = mu32x4{r.w[4 * j], r.w[4 * j + 1], r.w[4 * j + 2], r.w[4 * j + 3]};
  }
}
// Segment c of the lane's operands: of bf16 those of product c, of codes those of products 2 c and 2 c + 1.
template <int KV>
__device__ __forceinline__ mu32x4 masked_k_take(const mu32x4* tile, int t, int c, int lane) {
  const int n = lane & 15, g = lane >> 4;
  return tile[(KV == kKvBf16 ? 16 : 8) * (16 * t + n) + ((4 * c + g) ^ (n & 7))];
}

// The value operands of four channel blocks c = 4 q .. 4 q + 3: channel 8 n + c of the lane's 8 tokens. CAREFUL: with values
// that are not finite replaced by zeros.
template <int KV, bool CAREFUL>
__device__ __forceinline__ void masked_v_frags(const MaskedRaw<KV>& r, int q, mu32x4 (&f)[4]) {
  if constexpr (KV == kKvBf16) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t sel = (c & 1) ? 0x07060302u : 0x05040100u;
      const int d = 2 * q + (c >> 1);  // the dword of a token's channels that holds channel 4 q + c
#pragma unroll
      for (int e = 0; e < 4; ++e) f[c][e] = __builtin_amdgcn_perm(r.w[4 * (2 * e + 1) + d], r.w[4 * (2 * e) + d], sel);
    }
  } else {
    uint32_t lo[4], hi[4];
    masked_transpose4(r.w[q], r.w[2 + q], r.w[4 + q], r.w[6 + q], lo);
    masked_transpose4(r.w[8 + q], r.w[10 + q], r.w[12 + q], r.w[14 + q], hi);
#pragma unroll
    for (int c = 0; c < 4; ++c) f[c] = masked_codes8<KV>(lo[c], hi[c]);
  }
  if constexpr (CAREFUL && KV != kKvInt8) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) f[c][e] = masked_finite2(f[c][e]);
  }
}

// ---- rows -------------------------------------------------------------------------------------------------------

// What one lane knows of row n of each of its RT row tiles.
template <int RT>
struct MaskedRows {
  int pos[RT];         // the row's position
  int lo[RT], hi[RT];  // tokens lo .. hi - 1 are seen behind the prefix
  float slope[RT];     // times log2 e
  float m[RT], l[RT];  // reference point, and this lane's share of the weights' sum
  mf32x4 o[RT][8];     // channels 8 (4 g + i) + c of block c
};

// The steps of a tile, and which of them all of its rows see whole.
struct MaskedRange {
  int len, prefix;
  int sa, sb, n;        // steps 0 .. sa - 1, then sb ..; n in all
  int max_lo, min_hi;   // every row sees tokens max_lo .. min_hi - 1
  int min_lo, max_hi;   // some row sees tokens min_lo .. max_hi - 1 behind the prefix
};
__device__ __forceinline__ int masked_token0(const MaskedRange& r, int t) { return kMaskedStep * (t < r.sa ? t : r.sb + t - r.sa); }

// The page ids of step t's two 16-token groups, in lanes 0 and 1, and of step t + stride's, in lanes 2 and 3 (both clamped to the
// piece's last step), on their way for masked_pages. (Scalar loads would share their counter with LDS: every read of that would
// wait for the page table.)
template <bool PU>
__device__ __forceinline__ int masked_page_list(const MaskedParams& p, const MaskedRange& r, int b, int t, int stride, int t1, int lane) {
  if (!PU) return 0;
  const int token = masked_token0(r, min(t + (lane & 2 ? stride : 0), t1 - 1)) + 16 * (lane & 1);
  return ((const int32_t*)p.table)[((int64_t)b * p.table_sb + (min(token, r.len - 1) >> p.logP)) << p.table_i64];
}
__device__ __forceinline__ MaskedPages masked_pages(int list, int which = 0) {
  return MaskedPages{{__builtin_amdgcn_readlane(list, 2 * which), __builtin_amdgcn_readlane(list, 2 * which + 1)}};
}

// Row r's query, r / G by a multiplication (the host checks that it is exact).
__device__ __forceinline__ int masked_query(const MaskedParams& p, int r) { return p.G == 1 ? r : (int)__umulhi((unsigned)r, p.G_inv); }

__device__ __forceinline__ void masked_bounds(const MaskedParams& p, int b, int qi, int len, int& pos, int& lo, int& hi) {
  pos = len - p.Q + qi;
  lo = p.window > 0 ? max(pos - p.window + 1, 0) : 0;
  if (p.starts) lo = max(lo, p.starts[(int64_t)b * p.st_sb + (int64_t)qi * p.st_sq]);
  hi = min(pos + 1, len);
  if (hi <= lo) hi = lo = 0;  // nothing behind the prefix
}

// Lowest / highest bounds over rows r0 .. r1 - 1 of a KV head, the same in every lane.
__device__ __forceinline__ void masked_extent(const MaskedParams& p, int b, int r0, int r1, int lane, MaskedRange& r) {
  r.min_lo = 0x7fffffff, r.max_lo = 0, r.min_hi = 0x7fffffff, r.max_hi = 0;
  const int q0 = masked_query(p, r0), q1 = masked_query(p, r1 - 1);
  int pos, lo, hi;
  const bool scan = p.starts != nullptr;  // else both bounds rise with the query: the first and the last one tell
  for (int q = scan ? q0 + lane : q0; q <= q1; q += scan ? 64 : max(q1 - q0, 1)) {
    masked_bounds(p, b, q, r.len, pos, lo, hi);
    r.max_lo = max(r.max_lo, lo), r.min_hi = min(r.min_hi, hi), r.max_hi = max(r.max_hi, hi);
    if (hi > lo) r.min_lo = min(r.min_lo, lo);
    else if (!scan) r.min_lo = 0;  // positions below 0: the first row that sees anything sees token 0
  }
  if (scan) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
      r.min_lo = min(r.min_lo, __shfl_xor(r.min_lo, m, 64)), r.max_lo = max(r.max_lo, __shfl_xor(r.max_lo, m, 64));
      r.min_hi = min(r.min_hi, __shfl_xor(r.min_hi, m, 64)), r.max_hi = max(r.max_hi, __shfl_xor(r.max_hi, m, 64));
    }
  }
  r.min_lo = sread(r.min_lo), r.max_lo = sread(r.max_lo), r.min_hi = sread(r.min_hi), r.max_hi = sread(r.max_hi);
}
// The sequence's length and prefix, and the tile's steps.
__device__ __forceinline__ MaskedRange masked_range(const MaskedParams& p, int b, int r0, int r1, int lane) {
  MaskedRange r;
  int len = p.lens ? load_uniform(p.lens + b) : p.len_cap;
  r.len = min(max(len, 0), p.len_cap);
  r.prefix = p.prefix_lens ? min(min(max(load_uniform(p.prefix_lens + b), 0), p.max_prefix), r.len) : 0;
  masked_extent(p, b, r0, r1, lane, r);
  r.sa = (r.prefix + kMaskedStep - 1) / kMaskedStep;
  r.sb = r.sa;
  r.n = r.sa;
  if (r.max_hi > 0) {
    r.sb = max(r.min_lo / kMaskedStep, r.sa);
    r.n = r.sa + max((r.max_hi + kMaskedStep - 1) / kMaskedStep - r.sb, 0);
  }
  return r;
}
__device__ __forceinline__ bool masked_whole(const MaskedRange& r, int token0) {
  const int end = token0 + kMaskedStep;
  return end <= r.prefix || (token0 >= r.max_lo && end <= r.min_hi);
}
__device__ __forceinline__ bool masked_unseen(const MaskedRange& r, int token0) {
  return token0 >= r.prefix && (token0 >= r.max_hi || token0 + kMaskedStep <= r.min_lo);
}

template <int RT>
__device__ __forceinline__ void masked_rows_init(const MaskedParams& p, int b, int h, int first, int rows, int len, int lane,
                                                 MaskedRows<RT>& s) {
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = min(first + 16 * t + (lane & 15), rows - 1);  // lanes past the last row repeat it
    const int qi = masked_query(p, r);
    masked_bounds(p, b, qi, len, s.pos[t], s.lo[t], s.hi[t]);
    s.slope[t] = p.slopes ? p.slopes[h * p.G + r - qi * p.G] * kLog2e : 0.0f;
  }
}
template <int RT>
__device__ __forceinline__ void masked_rows_reset(MaskedRows<RT>& s) {
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    s.m[t] = kNegInf, s.l[t] = 0.0f;
#pragma unroll
    for (int c = 0; c < 8; ++c) s.o[t][c] = mf32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
}

// Queries as the first product's B operands: q[rt][s], and with an f16 q the remainders behind them.
template <int KV, bool QS, int RT>
__device__ __forceinline__ void masked_load_q(const MaskedParams& p, int b, int h, int first, int rows, int lane,
                                              mu32x4 (&q)[RT][QS ? 8 : 4]) {
  const int g = lane >> 4;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = min(first + 16 * t + (lane & 15), rows - 1);
    const int qi = masked_query(p, r);
    const uint16_t* src = (const uint16_t*)p.q + (int64_t)b * p.q_sb + (int64_t)qi * p.q_sq + (int64_t)(h * p.G + r - qi * p.G) * p.q_sh;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int c = KV == kKvBf16 ? 32 * s + 8 * g : 64 * (s >> 1) + 16 * g + 8 * (s & 1);
      const mu32x4 w = *(const mu32x4*)(src + c);
      if constexpr (!QS) {
        q[t][s] = w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x0 = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[e] & 0xffffu));
          const float x1 = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[e] >> 16));
          const bf16x2 hi = pack_bf16(x0, x1);
          q[t][s][e] = __builtin_bit_cast(uint32_t, hi);
          const float h0 = (float)hi[0], h1 = (float)hi[1];  // of an infinity nothing remains
          q[t][4 + s][e] = __builtin_bit_cast(uint32_t, pack_bf16(x0 == h0 ? 0.0f : x0 - h0, x1 == h1 ? 0.0f : x1 - h1));
        }
      }
    }
  }
}

// Values that are not finite, of the step's tokens, added to the row's outputs where it sees them (weights: each token's
// weight before its value's scale, at weights[16 token + n], -1 for tokens that row n does not see).
template <int KV, int SK>
__device__ __forceinline__ void masked_add_nonfinite(const MaskedParams& p, int b, int h, int token0, int len, int lane,
                                                     const float* weights, mf32x4 (&o)[8]) {
  const int n = lane & 15, g = lane >> 4;
  for (int j = 0; j < kMaskedStep; ++j) {
    const int tok = min(token0 + j, len - 1);
    const uint8_t* src = p.v + masked_row(p, b, h, tok, len);
    float vs = 1.0f;
    if constexpr (SK == kScaleTokenHead) {
      const int e = masked_clamp_page(p, ((const int32_t*)p.table)[((int64_t)b * p.table_sb + (tok >> p.logP)) << p.table_i64]);
      vs = p.vs[(int64_t)e * p.sc_sblk + (int64_t)(tok & (p.P - 1)) * p.sc_stok + (int64_t)h * p.sc_shead];
    }
    const bool scale_bad = !(fabsf(vs) <= __FLT_MAX__);
    const float w = weights[16 * j + n];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const int ch = 32 * g + 8 * i + c;
        float v;
        if constexpr (KV == kKvBf16) {
          v = bf16_bits_to_f32(((const uint16_t*)src)[ch]);
        } else if constexpr (KV == kKvFp8) {
          float f[4];
          fp8x4_to_f32(src[ch], f);
          v = f[0];
        } else {
          v = (float)(int8_t)src[ch];
        }
        if ((scale_bad || !(fabsf(v) <= __FLT_MAX__)) && w >= 0.0f) o[c][i] += w * (v * vs);
      }
  }
}

// cap tanh(t / cap) from u = 2 log2e t / cap.
__device__ __forceinline__ float masked_cap(float cap, float u) {
  return fmaf(-2.0f * cap, __builtin_amdgcn_rcpf(1.0f + fast_exp2(u)), cap);
}

// Per-token scales of the lane's tokens, of a step's (keys' 32, then values' 32): keys' times qs.
template <int SK>
__device__ __forceinline__ void masked_scales(const float* sc, int lane, float qs, float (&kf)[8], float (&vf)[8]) {
  if constexpr (SK == kScaleTokenHead) {
    const int g = lane >> 4;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        kf[4 * t + i] = sc[16 * t + 4 * g + i] * qs;
        vf[4 * t + i] = sc[32 + 16 * t + 4 * g + i];
      }
  }
}

// Tile r's raw products S[t] (token 16 t + 4 g + i) -> scores x in log2 units, those that its row does not see (seen) at minus
// infinity, with the row's reference point and sums brought up to date.
template <int SK, int RT>
__device__ __forceinline__ void masked_scores(const MaskedParams& p, const MaskedRange& rg, int token0, bool whole, int lane, float qs,
                                              const float (&kf)[8], const mf32x4 (&S)[2], int r, MaskedRows<RT>& st, float (&x)[8],
                                              uint32_t& seen) {
  const int g = lane >> 4;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = S[e >> 2][e & 3] * (SK == kScaleTokenHead ? kf[e] : qs);
  if (p.cap > kMaskedPlainCap) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {  // tanh z = z (1 - z^2 / 3 + 2 z^4 / 15 - 17 z^6 / 315) near 0, z = u ln2 / 2
      const float z = x[e] * (0.5f * kLn2), z2 = z * z;
      const float series = fmaf(z2, fmaf(z2, fmaf(z2, -17.0f / 315.0f, 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
      const float y = masked_cap(p.cap, x[e]);
      x[e] = fabsf(z) < 0.25f ? p.cap * z * series : y;
    }
  } else if (p.cap > 0.0f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = masked_cap(p.cap, x[e]);
  }
  if (p.slopes) {
    const float d0 = (float)(st.pos[r] - token0 - 4 * g);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf(-st.slope[r], fabsf(d0 - (float)(16 * (e >> 2) + (e & 3))), x[e]);
  }
  seen = 0xffu;
  if (!whole) {
    seen = 0u;
    const int j0 = token0 + 4 * g;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int j = j0 + 16 * (e >> 2) + (e & 3);
      const bool s = j < rg.prefix || (unsigned)(j - st.lo[r]) < (unsigned)(st.hi[r] - st.lo[r]);
      seen |= s ? 1u << e : 0u;
      x[e] = s ? x[e] : kNegInf;
    }
  }
  float mx = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) mx = fmaxf(mx, x[e]);
  mx = max_xor<32>(max_xor<16>(mx));
  if (__any(mx > st.m[r] + kMaskedSlack)) {  // some row's maximum left its reference point behind
    const float m = fmaxf(st.m[r], mx);
    const float a = st.m[r] == kNegInf ? 0.0f : fast_exp2(st.m[r] - m);
    st.m[r] = m;
    st.l[r] *= a;
#pragma unroll
    for (int c = 0; c < 8; ++c) st.o[r][c] *= a;
  }
}

// Tile r's scores -> weights' two bf16 parts. CAREFUL (uniform): values that are not finite stay out of the products and are added
// here instead (weights: this wave's 512 floats of LDS for that).
template <int KV, int SK, int RT, bool CAREFUL>
__device__ __forceinline__ void masked_weights(const MaskedParams& p, const MaskedRange& rg, int b, int h, int token0, bool whole, int lane,
                                               const float (&vf)[8], int r, MaskedRows<RT>& st, float (&x)[8], uint32_t seen,
                                               mu32x4 (&w)[2], float* weights) {
  const float m = st.m[r] == kNegInf ? 0.0f : st.m[r];
  float sum = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = fast_exp2(x[e] - m);
    sum += x[e];
  }
  st.l[r] += sum;
  if constexpr (CAREFUL) {
    const int n = lane & 15, g = lane >> 4;
#pragma unroll
    for (int e = 0; e < 8; ++e) weights[(16 * (e >> 2) + 4 * g + (e & 3)) * 16 + n] = (seen >> e) & 1u ? x[e] : -1.0f;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's lanes read one another's
    masked_add_nonfinite<KV, SK>(p, b, h, token0, rg.len, lane, weights, st.o[r]);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  if constexpr (SK == kScaleTokenHead) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] *= vf[e];
      if (!whole && !((seen >> e) & 1u)) x[e] = 0.0f;  // an unseen token's scale may be anything
      if (CAREFUL && !(fabsf(vf[e]) <= __FLT_MAX__)) x[e] = 0.0f;
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bf16x2 hi = pack_bf16(x[2 * e], x[2 * e + 1]);
    w[0][e] = __builtin_bit_cast(uint32_t, hi);
    w[1][e] = __builtin_bit_cast(uint32_t, pack_bf16(x[2 * e] - (float)hi[0], x[2 * e + 1] - (float)hi[1]));
  }
}

// Whether this lane's sums hold anything that is not finite.
template <int RT>
__device__ __forceinline__ bool masked_nonfinite(const MaskedRows<RT>& st) {
  float z = 0.0f;
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) z = fmaf(st.o[r][c][i], 0.0f, z);
  return z != 0.0f;
}

// The multiplier of raw products that gives scores in log2 units, or with a cap the argument of its exponential.
template <int SK>
__device__ __forceinline__ float masked_qscale(const MaskedParams& p, int h) {
  return SK == kScaleHead ? p.qscale * p.ks[h] : p.qscale;
}

// Sixteen lanes to a row from here on: lane c of them takes channel pairs 2 c + 32 i, so that every store and load of theirs is
// one piece of memory.
struct MaskedPairs {
  float x[4][2];
};
__device__ __forceinline__ void masked_store_pairs(const MaskedParams& p, int b, int h, int r, int c, const MaskedPairs& o, float lse2) {
  const int qi = masked_query(p, r), hq = h * p.G + r - qi * p.G;
  const int64_t at = (int64_t)b * p.o_sb + (int64_t)qi * p.o_sq + (int64_t)hq * p.o_sh + 2 * c;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (!p.out_pairs || p.out_dtype == kFF32) {
      store_float(p.out, at + 32 * i, p.out_dtype, o.x[i][0]);
      store_float(p.out, at + 32 * i + 1, p.out_dtype, o.x[i][1]);
    } else {
      const uint32_t w = p.out_dtype == kFBf16 ? __builtin_bit_cast(uint32_t, pack_bf16(o.x[i][0], o.x[i][1]))
                                               : __builtin_bit_cast(uint32_t, f16x2{(_Float16)o.x[i][0], (_Float16)o.x[i][1]});
      *(uint32_t*)((uint16_t*)p.out + at + 32 * i) = w;
    }
  }
  if (p.lse_out && c == 0) p.lse_out[((int64_t)b * p.Q + qi) * p.Hq + hq] = lse2 == kNegInf ? kNegInf : lse2 * kLn2;
}
__device__ __forceinline__ void masked_store_partial(const MaskedParams& p, int64_t slot, int row, int c, const MaskedPairs& o, float lse2) {
  float* dst = p.ws_out + (slot * p.live_rows + row) * kHeadDim + 2 * c;
#pragma unroll
  for (int i = 0; i < 4; ++i) ws_store2(dst + 32 * i, o.x[i][0], o.x[i][1]);
  if (c == 0) ws_store(p.ws_lse + slot * p.live_rows + row, lse2);
}

// A tile's n pieces (slots slot0 ..) combined by the last of them to arrive, in an order that n and the rows alone set, so that
// the sum does not depend on who came last: the whole workgroup of NT threads. A round trip to the memory side takes a
// microsecond, so NP pieces' loads are under way together (four for the few-row kernel; eight for the many-row one, which has the
// registers: 100 rows, 16 pieces, 53.3 -> 46.9 us), and where rows leave threads over, `parts` of their 16 lanes take every
// parts-th NP of a row's pieces and meet in LDS (`lds`, 130 floats for each 16 threads): FP8, one query, 1 x 16000 tokens, 125
// pieces of 2 rows, 45.8 -> 26.8 us.
template <int NT, int NP>
__device__ __forceinline__ void masked_combine(const MaskedParams& p, int b, int h, int r0, int live, int64_t slot0, int n, int tid,
                                               float* lds) {
  ws_acquire();
  constexpr int GROUPS = NT / 16;
  const int c = tid & 15, group = tid >> 4;
  float M, W;
  MaskedPairs o;
  // Pieces j0 .. j0 + NP - 1 of every `step`, from `from` on: their weights' sum W and products o relative to 2^M.
  auto fold = [&](int row, int from, int step) {
    const float* lse = p.ws_lse + slot0 * p.live_rows + row;
    const float* prt = p.ws_out + (slot0 * p.live_rows + row) * kHeadDim + 2 * c;
    M = kNegInf, W = 0.0f, o = MaskedPairs{};
    for (int j0 = from; j0 < n; j0 += step) {
      float lv[NP], top = kNegInf;
      MaskedPairs ov[NP];
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        lv[j] = kNegInf;
        if (j0 + j < n) {
          lv[j] = ws_load(lse + (int64_t)(j0 + j) * p.live_rows);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            ws_load2(prt + (int64_t)(j0 + j) * p.live_rows * kHeadDim + 32 * i, ov[j].x[i][0], ov[j].x[i][1]);
        }
      }
#pragma unroll
      for (int j = 0; j < NP; ++j) top = fmaxf(top, lv[j]);
      const float nm = fmaxf(M, top), mu = nm == kNegInf ? 0.0f : nm;
      const float a = W > 0.0f ? fast_exp2(M - mu) : (W != W ? W : 0.0f);
      W *= a;
#pragma unroll
      for (int i = 0; i < 4; ++i) o.x[i][0] *= a, o.x[i][1] *= a;
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        if (lv[j] == kNegInf) continue;  // an empty piece
        const float e = fast_exp2(lv[j] - mu);
        W += e;
#pragma unroll
        for (int i = 0; i < 4; ++i) o.x[i][0] = fmaf(e, ov[j].x[i][0], o.x[i][0]), o.x[i][1] = fmaf(e, ov[j].x[i][1], o.x[i][1]);
      }
      M = nm;
    }
  };
  auto finish = [&](int row) {
    const float inv = W == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(W);
#pragma unroll
    for (int i = 0; i < 4; ++i) o.x[i][0] *= inv, o.x[i][1] *= inv;
    masked_store_pairs(p, b, h, r0 + row, c, o, W == 0.0f ? kNegInf : M + __log2f(W));
  };
  int parts = 1;
  while (2 * parts * live <= GROUPS && parts * NP < n) parts *= 2;
  if (parts == 1) {
    for (int row = group; row < live; row += GROUPS) {
      fold(row, 0, NP);
      finish(row);
    }
    return;
  }
  const int row = group / parts, part = group % parts;
  float* s_mw = lds + GROUPS * kHeadDim;
  if (row < live) {
    fold(row, NP * part, NP * parts);
    if (c == 0) s_mw[2 * group] = M, s_mw[2 * group + 1] = W;
#pragma unroll
    for (int i = 0; i < 4; ++i) *(float2*)(lds + group * kHeadDim + 32 * i + 2 * c) = make_float2(o.x[i][0], o.x[i][1]);
  }
  __syncthreads();
  if (row >= live || part != 0) return;
  for (int s = 1; s < parts; ++s) M = fmaxf(M, s_mw[2 * (group + s)]);
  const float mu = M == kNegInf ? 0.0f : M;
  W = 0.0f, o = MaskedPairs{};
  for (int s = 0; s < parts; ++s) {
    const float m = s_mw[2 * (group + s)], w = s_mw[2 * (group + s) + 1];
    const float a = w > 0.0f ? fast_exp2(m - mu) : (w != w ? w : 0.0f);
    W = fmaf(a, w, W);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = *(const float2*)(lds + (group + s) * kHeadDim + 32 * i + 2 * c);
      o.x[i][0] = fmaf(a, x.x, o.x[i][0]), o.x[i][1] = fmaf(a, x.y, o.x[i][1]);
    }
  }
  finish(row);
}

// A workgroup's place: XCD-major (workgroups go to the 8 XCDs in turn, each with its own L2), so that the heads of a page
// (few rows) or the tiles of a head (many rows) meet in one L2.
__device__ __forceinline__ int masked_index() {
  const int x = blockIdx.x, n = gridDim.x;
  const int q = n >> 3, r = n & 7, k = x & 7;
  return k * q + min(k, r) + (x >> 3);
}

constexpr int masked_key_units(int kv) { return kMaskedStep * (kv == kKvBf16 ? 16 : 8); }  // 16-byte units of a step's key rows

// ---- few rows ---------------------------------------------------------------------------------------------------

// One wave's steps t, t + 4, ... < t1 folded into its rows (list: the page ids of the first two). The next step's keys are requested
// once this one's have gone to LDS, its values once this one's are multiplied, and the page ids of the step after that in between:
// no request stands behind a branch, so that each is waited for by itself.
template <int KV, int SK, bool PU, bool QS, bool ONCE, bool CAREFUL>
__device__ __forceinline__ void masked_few_steps(const MaskedParams& p, const MaskedRange& rg, int b, int h, int t, int t1, int lane,
                                                 float qs, const mu32x4 (&q)[1][QS ? 8 : 4], int list, mu32x4* w_keys,
                                                 float* w_scale, float* w_weights, MaskedRows<1>& st) {
  masked_rows_reset(st);
  if (t >= t1) return;
  MaskedRaw<KV> k, v;
  float sc = 0.0f;
  int token0 = masked_token0(rg, t);
  MaskedPages pages = masked_pages(list, 1);  // the next step's
  {
    const MaskedSpot spot = masked_spot<PU>(p, h, masked_pages(list), token0, rg.len);
    masked_issue_k<KV, PU, ONCE>(p, b, h, token0, rg.len, spot, lane, k);
    if constexpr (SK == kScaleTokenHead) sc = masked_issue_scale<PU>(p, b, h, token0, rg.len, spot, lane);
    masked_issue_v<KV, PU, ONCE>(p, b, h, token0, rg.len, spot, lane, v);
  }
  auto step = [&](auto last) {
    masked_k_keep<KV>(k, lane, w_keys);
    if constexpr (SK == kScaleTokenHead) w_scale[lane] = sc;
    const int next = last ? 0 : masked_token0(rg, t + 4);
    MaskedSpot spot{};
    if constexpr (!last) {
      spot = masked_spot<PU>(p, h, pages, next, rg.len);
      masked_issue_k<KV, PU, ONCE>(p, b, h, next, rg.len, spot, lane, k);
      if constexpr (SK == kScaleTokenHead) sc = masked_issue_scale<PU>(p, b, h, next, rg.len, spot, lane);
      list = masked_page_list<PU>(p, rg, b, t + 8, 0, t1, lane);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's lanes read one another's
    mf32x4 S[1][2] = {{mf32x4{0.0f, 0.0f, 0.0f, 0.0f}, mf32x4{0.0f, 0.0f, 0.0f, 0.0f}}};
    constexpr int C = KV == kKvBf16 ? 4 : 2;  // segments of a lane, each for 4 / C products
    mu32x4 seg[2][C];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int c = 0; c < C; ++c) seg[u][c] = masked_k_take<KV>(w_keys, u, c, lane);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        mu32x4 f;
        if constexpr (KV == kKvBf16) f = seg[u][s];
        else f = masked_codes8<KV>(seg[u][s >> 1][2 * (s & 1)], seg[u][s >> 1][2 * (s & 1) + 1]);
        if constexpr (QS) S[0][u] = masked_mfma(f, q[0][4 + s], S[0][u]);
        S[0][u] = masked_mfma(f, q[0][s], S[0][u]);
      }
    const bool whole = masked_whole(rg, token0);
    float kf[8], vf[8], x[8];
    uint32_t seen;
    mu32x4 w[2];
    masked_scales<SK>(w_scale, lane, qs, kf, vf);
    masked_scores<SK, 1>(p, rg, token0, whole, lane, qs, kf, S[0], 0, st, x, seen);
    masked_weights<KV, SK, 1, CAREFUL>(p, rg, b, h, token0, whole, lane, vf, 0, st, x, seen, w, w_weights);
#pragma unroll
    for (int c4 = 0; c4 < 2; ++c4) {
      mu32x4 f[4];
      masked_v_frags<KV, CAREFUL>(v, c4, f);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        st.o[0][4 * c4 + c] = masked_mfma(f[c], w[1], st.o[0][4 * c4 + c]);
        st.o[0][4 * c4 + c] = masked_mfma(f[c], w[0], st.o[0][4 * c4 + c]);
      }
    }
    if constexpr (!last) {
      masked_issue_v<KV, PU, ONCE>(p, b, h, next, rg.len, spot, lane, v);
      pages = masked_pages(list);
      token0 = next;
    }
  };
  for (; t + 4 < t1; t += 4) step(std::false_type{});
  step(std::true_type{});
}

template <int KV, int SK, bool PU, bool QS, bool ONCE>
__global__ __launch_bounds__(256, KV == kKvBf16 ? 2 : 3) void masked_few_kernel(const MaskedParams p) {
  // [4 waves][live][kMaskedRowPad], then [live][4] m and l; on the way there key operands, scales and weights. Vectors, so that it
  // lies on a 16-byte boundary whatever other LDS there is: 16-byte accesses off it take eight times as long.
  extern __shared__ mf32x4 s_dyn[];
  float* smem = (float*)s_dyn;
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 63, wave = sread(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  // Workgroups go to the 8 XCDs in turn: the heads of a piece, whose rows share pages and lines of scales, go to one, and the
  // pieces are dealt out to the XCDs in turn, the first ones of all sequences before the second ones.
  const int heads = p.Hkv * p.tiles, ht = (blockIdx.x >> 3) % heads;
  const int turn = (blockIdx.x >> 3) / heads * 8 + (blockIdx.x & 7), h = ht / p.tiles, tile = ht - h * p.tiles;
  const int piece = turn / p.B, b = turn % p.B;
  if (piece >= p.max_pieces) return;
  const int rows = p.Q * p.G, r0 = 16 * tile, live = min(rows - r0, 16), t0 = piece * p.piece;
  mu32x4 q[1][QS ? 8 : 4];
  masked_load_q<KV, QS, 1>(p, b, h, r0, rows, lane, q);
  // Where steps follow one another from the sequence's first token on, the first page ids are known ahead of its length.
  const bool plain = PU && p.window == 0 && !p.starts;
  int list = 0;
  if (plain) {
    const int group = 2 * (t0 + wave + (lane & 2 ? 4 : 0)) + (lane & 1);
    list = ((const int32_t*)p.table)[((int64_t)b * p.table_sb + min(group >> (p.logP - 4), p.max_blocks - 1)) << p.table_i64];
  }
  const MaskedRange rg = masked_range(p, b, r0, r0 + live, lane);
  const int pieces = max((rg.n + p.piece - 1) / p.piece, 1);
  if (piece >= pieces) return;
  const int t1 = min(t0 + p.piece, rg.n);
  if (!plain && t0 + wave < t1) list = masked_page_list<PU>(p, rg, b, t0 + wave, 4, t1, lane);
  const float vscale = SK == kScaleHead ? p.vs[h] : 1.0f, qs = masked_qscale<SK>(p, h);

  MaskedRows<1> st;
  masked_rows_init<1>(p, b, h, r0, rows, rg.len, lane, st);
  mu32x4* w_keys = (mu32x4*)smem + wave * masked_key_units(KV);  // this wave's key rows,
  float* w_scale = smem + 16 * masked_key_units(KV) + wave * 64;  // per-token scales
  float* w_weights = smem + 16 * masked_key_units(KV) + 4 * 64 + wave * kMaskedStep * 16;  // and, where needed, weights
  masked_few_steps<KV, SK, PU, QS, ONCE, false>(p, rg, b, h, t0 + wave, t1, lane, qs, q, list, w_keys, w_scale, w_weights, st);
  if (__any(masked_nonfinite(st))) {
    if (t0 + wave < t1) list = masked_page_list<PU>(p, rg, b, t0 + wave, 4, t1, lane);
    masked_few_steps<KV, SK, PU, QS, ONCE, true>(p, rg, b, h, t0 + wave, t1, lane, qs, q, list, w_keys, w_scale, w_weights, st);
  }

  // The waves' shares of each row, brought to the row's maximum and added.
  float* s_o = smem;                             // [4 waves][live][kMaskedRowPad]
  float* s_m = smem + 4 * live * kMaskedRowPad;  // [live][4 waves]
  float* s_l = s_m + 4 * live;
  __syncthreads();  // keys, scales and weights lay where the rows go
  const float lsum = sum_xor<32>(sum_xor<16>(st.l[0]));
  if (n < live) {
    if (g == 0) s_m[4 * n + wave] = st.m[0], s_l[4 * n + wave] = lsum;
    float* dst = s_o + (wave * live + n) * kMaskedRowPad + 32 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < 8; c += 4)
        *(mf32x4*)(dst + 8 * i + c) = mf32x4{st.o[0][c][i], st.o[0][c + 1][i], st.o[0][c + 2][i], st.o[0][c + 3][i]};
  }
  __syncthreads();
  const int64_t seg = ((int64_t)b * p.Hkv + h) * p.tiles + tile, slot = seg * p.max_pieces + piece;
  const int row = tid >> 4, c = tid & 15;
  if (row < live) {
    const mf32x4 m = *(const mf32x4*)(s_m + 4 * row), l = *(const mf32x4*)(s_l + 4 * row);
    const float M = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
    float L = 0.0f;
    MaskedPairs o{};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      // Waves that saw nothing have no maximum, nor have those whose scores were all NaN, whose sums carry that on.
      const float a = m[w] == kNegInf ? (l[w] == 0.0f ? 0.0f : 1.0f) : fast_exp2(m[w] - M);
      const float* src = s_o + (w * live + row) * kMaskedRowPad + 2 * c;
      L = fmaf(a, l[w], L);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = *(const float2*)(src + 32 * i);
        o.x[i][0] = fmaf(a, x.x, o.x[i][0]), o.x[i][1] = fmaf(a, x.y, o.x[i][1]);
      }
    }
    const float inv = L == 0.0f ? 0.0f : vscale * __builtin_amdgcn_rcpf(L);
#pragma unroll
    for (int i = 0; i < 4; ++i) o.x[i][0] *= inv, o.x[i][1] *= inv;
    const float lse2 = L == 0.0f ? kNegInf : (M == kNegInf ? 0.0f : M) + __log2f(L);
    if (pieces == 1) masked_store_pairs(p, b, h, r0 + row, c, o, lse2);
    else masked_store_partial(p, slot, row, c, o, lse2);
  }
  if (pieces == 1) return;
  ws_publish();
  __syncthreads();
  if (tid == 0) s_last = ws_arrive(p.counters + seg) == (unsigned)pieces - 1u;
  __syncthreads();
  if (!s_last) return;
  masked_combine<256, 4>(p, b, h, r0, live, seg * p.max_pieces, pieces, tid, smem);
  if (tid == 0) __hip_atomic_store(p.counters + seg, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---- many rows --------------------------------------------------------------------------------------------------

constexpr int kMaskedChunk = 4 * kMaskedItem;         // two steps: K, K, V, V
// Two chunks, their per-token scales, and the waves' weights of a careful pass.
constexpr int kMaskedManyLds = 2 * kMaskedChunk * 16 + (2 * 2 * 64 + 4 * kMaskedStep * 16) * 4;
static_assert(2 * (kMaskedManyLds + 64) <= 160 << 10, "two workgroups to a CU");
static_assert(128 * (kMaskedRowPad + 1) * 4 <= kMaskedManyLds, "the rows fit where the operands lay");

// The piece's steps t0 .. t1 - 1, two at a time, folded into each wave's rows (mine: what they see).
template <int KV, int SK, bool PU, bool QS, int RT, bool CAREFUL>
__device__ __forceinline__ void masked_many_steps(const MaskedParams& p, const MaskedRange& rg, const MaskedRange& mine, int b, int h,
                                                  int t0, int t1, int lane, int wave, bool idle, float qs,
                                                  const mu32x4 (&q)[RT][QS ? 8 : 4], mu32x4* s_op, float* s_scale,
                                                  MaskedRows<RT>& st) {
  const int my_step = wave & 1;  // this wave's share of a chunk: keys (waves 0, 1) or values (2, 3) of one step
  masked_rows_reset(st);
  MaskedRaw<KV> raw;
  float sc = 0.0f;
  int list = t0 < t1 ? masked_page_list<PU>(p, rg, b, t0 + my_step, 0, t1, lane) : 0;
  auto issue = [&](int t) {  // chunk at step t of the list; steps past the piece's last repeat it
    const int token0 = masked_token0(rg, min(t + my_step, t1 - 1));
    const MaskedSpot spot = masked_spot<PU>(p, h, masked_pages(list), token0, rg.len);
    list = masked_page_list<PU>(p, rg, b, t + 2 + my_step, 0, t1, lane);
    if (wave < 2) {
      masked_issue_k<KV, PU, false>(p, b, h, token0, rg.len, spot, lane, raw);
      if constexpr (SK == kScaleTokenHead) sc = masked_issue_scale<PU>(p, b, h, token0, rg.len, spot, lane);
    } else {
      masked_issue_v<KV, PU, false>(p, b, h, token0, rg.len, spot, lane, raw);
    }
  };
  if (t0 < t1) issue(t0);
  for (int t = t0, buf = 0; t < t1; t += 2, buf ^= 1) {
    mu32x4* dst = s_op + buf * kMaskedChunk + wave * kMaskedItem;
    if (wave < 2) {
      masked_k_place<KV>(raw, lane, dst);
      if constexpr (SK == kScaleTokenHead) s_scale[(2 * buf + wave) * 64 + lane] = sc;
    } else {
#pragma unroll
      for (int c4 = 0; c4 < 2; ++c4) {
        mu32x4 f[4];
        masked_v_frags<KV, CAREFUL>(raw, c4, f);
#pragma unroll
        for (int c = 0; c < 4; ++c) dst[64 * (4 * c4 + c) + lane] = f[c];
      }
    }
    __syncthreads();
    if (t + 2 < t1) issue(t + 2);
    const mu32x4* src = s_op + buf * kMaskedChunk;
#pragma unroll
    for (int u2 = 0; u2 < 2; ++u2) {
      const int token0 = masked_token0(rg, min(t + u2, t1 - 1));
      if (t + u2 >= t1 || idle || masked_unseen(mine, token0)) continue;
      mf32x4 S[RT][2];
#pragma unroll
      for (int r = 0; r < RT; ++r) S[r][0] = S[r][1] = mf32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const mu32x4 f = masked_k_frag<KV>(src + u2 * kMaskedItem, u, s, lane);
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            if constexpr (QS) S[r][u] = masked_mfma(f, q[r][4 + s], S[r][u]);
            S[r][u] = masked_mfma(f, q[r][s], S[r][u]);
          }
        }
      float* weights = s_scale + 256 + wave * kMaskedStep * 16;
      const bool whole = masked_whole(mine, token0);
      float kf[8], vf[8], x[8];
      uint32_t seen;
      mu32x4 w[RT][2];
      masked_scales<SK>(s_scale + (2 * buf + u2) * 64, lane, qs, kf, vf);
      const mu32x4* values = src + (2 + u2) * kMaskedItem + lane;
      auto product = [&](int r, const mu32x4& v, int c) {
        st.o[r][c] = masked_mfma(v, w[r][1], st.o[r][c]);
        st.o[r][c] = masked_mfma(v, w[r][0], st.o[r][c]);
      };
      masked_scores<SK, RT>(p, mine, token0, whole, lane, qs, kf, S[0], 0, st, x, seen);
      masked_weights<KV, SK, RT, CAREFUL>(p, mine, b, h, token0, whole, lane, vf, 0, st, x, seen, w[0], weights);
      if constexpr (RT == 2) masked_scores<SK, RT>(p, mine, token0, whole, lane, qs, kf, S[1], 1, st, x, seen);
      if constexpr (RT == 2 && !QS) {
        // The first tile's products run on the matrix units while the vector units take the second's exponentials: BF16, 2048
        // queries after 2049, capped, 122.7 -> 119 us, not capped 107.6 -> 99.3. An f16 q leaves no registers to hold the values.
        mu32x4 v[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = values[64 * c];
#pragma unroll
        for (int c = 0; c < 8; ++c) product(0, v[c], c);
        masked_weights<KV, SK, RT, CAREFUL>(p, mine, b, h, token0, whole, lane, vf, 1, st, x, seen, w[1], weights);
#pragma unroll
        for (int c = 0; c < 8; ++c) product(1, v[c], c);
      } else {
        if constexpr (RT == 2) masked_weights<KV, SK, RT, CAREFUL>(p, mine, b, h, token0, whole, lane, vf, 1, st, x, seen, w[1], weights);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const mu32x4 v = values[64 * c];
#pragma unroll
          for (int r = 0; r < RT; ++r) product(r, v, c);
        }
      }
    }
  }
}

template <int KV, int SK, bool PU, bool QS, int RT>
__global__ __launch_bounds__(256, 2) void masked_many_kernel(const MaskedParams p) {
  extern __shared__ mu32x4 s_op[];  // [2 chunks][K0 K1 V0 V1][8 operands][64 lanes]
  __shared__ int s_last, s_bad;
  constexpr int BM = 64 * RT;
  const int tid = threadIdx.x, lane = tid & 63, wave = sread(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  float* s_scale = (float*)(s_op + 2 * kMaskedChunk);  // [2 chunks][2 steps][64]
  int v = masked_index();
  const int piece = v % p.max_pieces;
  v /= p.max_pieces;
  const int tile = p.tiles - 1 - v % p.tiles;  // the last rows see the most: they start first
  v /= p.tiles;
  const int h = v % p.Hkv, b = v / p.Hkv;
  const int rows = p.Q * p.G, r0 = tile * BM, live = min(BM, rows - r0);
  const MaskedRange rg = masked_range(p, b, r0, r0 + live, lane);
  const int pieces = max((rg.n + p.piece - 1) / p.piece, 1);
  if (piece >= pieces) return;
  const int t0 = piece * p.piece, t1 = min(t0 + p.piece, rg.n);
  const int first = r0 + 16 * RT * wave;  // this wave's rows
  const bool idle = first >= rows;
  MaskedRange mine = rg;  // what they see
  if (!idle) masked_extent(p, b, first, min(first + 16 * RT, rows), lane, mine);

  MaskedRows<RT> st;
  masked_rows_init<RT>(p, b, h, first, rows, rg.len, lane, st);
  mu32x4 q[RT][QS ? 8 : 4];
  masked_load_q<KV, QS, RT>(p, b, h, first, rows, lane, q);
  const float qs = masked_qscale<SK>(p, h);

  masked_many_steps<KV, SK, PU, QS, RT, false>(p, rg, mine, b, h, t0, t1, lane, wave, idle, qs, q, s_op, s_scale, st);
  if (tid == 0) s_bad = 0;
  __syncthreads();
  if (masked_nonfinite(st)) s_bad = 1;
  __syncthreads();
  if (s_bad) masked_many_steps<KV, SK, PU, QS, RT, true>(p, rg, mine, b, h, t0, t1, lane, wave, idle, qs, q, s_op, s_scale, st);

  // Rows go out through LDS (the operands' place), so that whole pieces of them are stored.
  float* s_o = (float*)s_op;  // [BM][kMaskedRowPad], then each row's log2-sum-exp
  float* s_lse = s_o + BM * kMaskedRowPad;
  const int64_t seg = ((int64_t)b * p.Hkv + h) * p.tiles + tile, slot = seg * p.max_pieces + piece;
  const float vscale = SK == kScaleHead ? p.vs[h] : 1.0f;
  __syncthreads();  // the operands are read
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const float l = sum_xor<32>(sum_xor<16>(st.l[r]));
    const int row = 16 * RT * wave + 16 * r + n;
    const float inv = l == 0.0f ? 0.0f : vscale * __builtin_amdgcn_rcpf(l);
    if (g == 0) s_lse[row] = l == 0.0f ? kNegInf : (st.m[r] == kNegInf ? 0.0f : st.m[r]) + __log2f(l);
    float* dst = s_o + row * kMaskedRowPad + 32 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < 8; c += 4)
        *(mf32x4*)(dst + 8 * i + c) =
            mf32x4{st.o[r][c][i] * inv, st.o[r][c + 1][i] * inv, st.o[r][c + 2][i] * inv, st.o[r][c + 3][i] * inv};
  }
  __syncthreads();
  for (int row = tid >> 4; row < live; row += 16) {
    MaskedPairs o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = *(const float2*)(s_o + row * kMaskedRowPad + 2 * (tid & 15) + 32 * i);
      o.x[i][0] = x.x, o.x[i][1] = x.y;
    }
    if (pieces == 1) masked_store_pairs(p, b, h, r0 + row, tid & 15, o, s_lse[row]);
    else masked_store_partial(p, slot, row, tid & 15, o, s_lse[row]);
  }
  if (pieces == 1) return;
  ws_publish();
  __syncthreads();
  if (tid == 0) s_last = ws_arrive(p.counters + seg) == (unsigned)pieces - 1u;
  __syncthreads();
  if (!s_last) return;
  masked_combine<256, 8>(p, b, h, r0, live, seg * p.max_pieces, pieces, tid, s_o);
  if (tid == 0) __hip_atomic_store(p.counters + seg, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---- launches ---------------------------------------------------------------------------------------------------

template <int KV, int SK, bool PU, bool QS>
static hipError_t launch_masked_t(const MaskedParams& p, int rt, bool many, int grid, hipStream_t stream) {
  const int live = p.live_rows;
  // The merge's rows, or the operands, scales and weights that lie there before it.
  const size_t merge = (size_t)4 * live * (kMaskedRowPad + 2) * sizeof(float);
  const size_t early = (size_t)(16 * masked_key_units(KV) + 4 * 64 + 4 * kMaskedStep * 16) * sizeof(float);
  const size_t few = merge > early ? merge : early;
  static_assert((16 * masked_key_units(KV) + 4 * 64) >= 16 * (kHeadDim + 2), "the combine's shares fit");
  hipError_t e = hipSuccess;
  auto run = [&](auto kernel, size_t lds) {
    if (lds > (64u << 10))  // has to be asked for, once per device
      e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e == hipSuccess) hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), lds, stream, p);
  };
  if (rt == 2) run(masked_many_kernel<KV, SK, PU, QS, 2>, kMaskedManyLds);
  else if (many) run(masked_many_kernel<KV, SK, PU, QS, 1>, kMaskedManyLds);
  else if (p.tiles > 1) run(masked_few_kernel<KV, SK, PU, QS, false>, few);
  else run(masked_few_kernel<KV, SK, PU, QS, true>, few);
  return e == hipSuccess ? hipGetLastError() : e;
}

// PU: pages of at least 16 tokens, so that the 16 tokens of a group lie in one, whose id the whole wave reads.
template <int KV, int SK>
static hipError_t launch_masked(const MaskedParams& p, bool q_split, int rt, bool many, int grid, hipStream_t stream) {
  if (p.logP >= 4)
    return q_split ? launch_masked_t<KV, SK, true, true>(p, rt, many, grid, stream)
                   : launch_masked_t<KV, SK, true, false>(p, rt, many, grid, stream);
  return q_split ? launch_masked_t<KV, SK, false, true>(p, rt, many, grid, stream)
                 : launch_masked_t<KV, SK, false, false>(p, rt, many, grid, stream);
}

}  // namespace bpt
