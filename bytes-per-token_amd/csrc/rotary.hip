// Rotary positions: queries and keys [B, Q, H, D] normalised per head (optional) and rotated by their positions, and on
// request the rotated keys and the values quantized straight into their slots of the paged pools.
//
// Per row x of D channels: r = rsqrt(mean x^2 + eps), x_c <- x_c r w_c (with norm weights), then for each pair i of the
// rotary_dim / 2 leading ones, with t = position[axis(i)] * inv_freq[i]:
//   (a, b) <- scaling * (a cos t - b sin t, a sin t + b cos t)
// in float32, rounded once to the output's type or quantized as quant_append does (IEEE divisions, the same formulas).
// Channels past rotary_dim are only normalised.
//
// A workgroup takes a few tokens with all of their heads: the angles of a token are computed once, by one thread per
// pair, and shared through LDS. They need more than 24 bits (position 10^6 times frequency 1 leaves 1/16 radian to
// float32), so turns t / 2 pi are computed in float64 and reduced exactly to an eighth of a turn around the nearest
// quarter; sine and cosine of what is left are Taylor polynomials in float32 (truncation below 2^-28).
//
// A row is held by a group of 2^k lanes, 16 channels (8 pairs) a lane: a pair's channels lie in one lane, so that the
// rotation needs no exchange, and 16-bit rows are loaded and stored 16 bytes at a time, their codes 8. Row sums and maxima are
// butterflies over the group.
//
// Bound by memory: 4 x 4097 tokens of 16 + 16 bf16 heads of 80 channels 46 us (168 MB, 3.6 TB/s), 4 x 4096 tokens of 32 + 8 heads
// of 128 into FP8 pools 96 us (369 MB, 3.8 TB/s). Calls of a few tokens take 5 to 7 us: launch, two memory round trips, the angles.
#include "bpt_device.h"
#include "bpt_internal.h"

namespace bpt {

constexpr int kRotaryThreads = 256;
constexpr int kKvNone = -1;  // no pool: keys are written like the queries

template <int X>
__device__ __forceinline__ void rotary_load8(const void* base, int64_t idx, float* v) {
  if constexpr (X == kFF32) {
    typedef float f4 __attribute__((ext_vector_type(4)));
    const f4 lo = *(const f4*)((const float*)base + idx), hi = *(const f4*)((const float*)base + idx + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = lo[j], v[4 + j] = hi[j];
  } else {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    const u4 w = *(const u4*)((const uint16_t*)base + idx);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (X == kFBf16) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      } else {
        v[2 * j] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[j] & 0xffffu));
        v[2 * j + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[j] >> 16));
      }
    }
  }
}

typedef __bf16 rbf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 rf16x2 __attribute__((ext_vector_type(2)));
template <int X>
__device__ __forceinline__ uint32_t rotary_pack2(float a, float b) {  // rounded to nearest, ties to even
  if constexpr (X == kFBf16) return __builtin_bit_cast(uint32_t, rbf16x2{(__bf16)a, (__bf16)b});
  else return __builtin_bit_cast(uint32_t, rf16x2{(_Float16)a, (_Float16)b});
}

template <int X>
__device__ __forceinline__ void rotary_store8(void* base, int64_t idx, const float* v) {
  if constexpr (X == kFF32) {
    typedef float f4 __attribute__((ext_vector_type(4)));
    *(f4*)((float*)base + idx) = f4{v[0], v[1], v[2], v[3]};
    *(f4*)((float*)base + idx + 4) = f4{v[4], v[5], v[6], v[7]};
  } else {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    *(u4*)((uint16_t*)base + idx) = u4{rotary_pack2<X>(v[0], v[1]), rotary_pack2<X>(v[2], v[3]),
                                       rotary_pack2<X>(v[4], v[5]), rotary_pack2<X>(v[6], v[7])};
  }
}

// cos and sin of position * frequency.
__device__ __forceinline__ float2 rotary_angle(int64_t position, float freq) {
  const double turns = (double)position * (double)freq * 0.15915494309189535;
  double f = turns - rint(turns);        // [-1/2, 1/2], exact
  const double quarter = rint(4.0 * f);  // -2 .. 2
  f = fma(-0.25, quarter, f);            // [-1/8, 1/8], exact
  const float a = (float)(f * 6.283185307179586), s = a * a;
  float sn = fmaf(s, 2.7557319e-6f, -1.9841270e-4f);
  sn = fmaf(s, sn, 8.3333333e-3f);
  sn = fmaf(s, sn, -1.6666667e-1f);
  sn = fmaf(a * s, sn, a);
  float cs = fmaf(s, -2.7557319e-7f, 2.4801587e-5f);
  cs = fmaf(s, cs, -1.3888889e-3f);
  cs = fmaf(s, cs, 4.1666667e-2f);
  cs = fmaf(s, cs, -0.5f);
  cs = fmaf(s, cs, 1.0f);
  const int n = (int)quarter & 3;
  const float c = n & 1 ? sn : cs, d = n & 1 ? cs : sn;
  return make_float2(n == 1 || n == 2 ? -c : c, n >= 2 ? -d : d);
}

// Eight norm weights, of any type.
__device__ __forceinline__ void rotary_load_weights(const void* w, int c, int dtype, float* v) {
  if (dtype == kFBf16) rotary_load8<kFBf16>(w, c, v);
  else if (dtype == kFF16) rotary_load8<kFF16>(w, c, v);
  else rotary_load8<kFF32>(w, c, v);
}

// x / s to where it rounds to the same e4m3 code, given inv = 1 / s to an ulp: the product is within 2^-22 of the quotient, and
// midpoints of normal codes (magnitudes from 2^-6 on) have nothing below the mantissa's bit 19. Products within 4 ulps of one, and
// those below the normal range, take the IEEE division, as do NaN and (rotary_store_codes) scales past 2^+-100.
__device__ __forceinline__ bool rotary_fp8_sure(float q) {
  const uint32_t u = __float_as_uint(q);
  return (u & 0x7fffffffu) >= 0x3c800000u && (u & 0x7fffffffu) < 0x7f000000u && ((u & 0xfffffu) - 0x7fffcu) > 8u;
}

// Chunk of 8 values quantized and stored (n of them; vec: all 8 at once).
template <int KV, int SK>
__device__ __forceinline__ void rotary_store_codes(uint8_t* dst, const float* x, float s, float inv, int n, bool vec) {
  if constexpr (KV == kKvBf16) {
    if (vec) {
      rotary_store8<kFBf16>(dst, 0, x);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n) ((uint16_t*)dst)[j] = f32_to_bf16_bits(x[j]);
    }
  } else {
    uint32_t code[8];
    const bool normal = s >= 0x1p-100f && s <= 0x1p100f;  // far enough inside that the reciprocal is a normal number too
    if constexpr (KV == kKvFp8) {
      float y[8];
      bool sure = normal;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y[j] = x[j] * inv;
        sure &= rotary_fp8_sure(y[j]) || x[j] == 0.0f;
      }
      if (!sure) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = __fdiv_rn(x[j], s);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) code[j] = f32_to_fp8(clamp_fp8_range(y[j]));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float r = normal ? rint_quotient(x[j], s, inv) : rintf(__fdiv_rn(x[j], s));
        r = r > 127.0f ? 127.0f : (r < -128.0f ? -128.0f : r);
        code[j] = (uint32_t)(int32_t)r & 0xffu;
      }
    }
    if (vec) {
      typedef uint32_t u2 __attribute__((ext_vector_type(2)));
      *(u2*)dst = u2{code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24, code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24};
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n) dst[j] = (uint8_t)code[j];
    }
  }
}

template <int X, int KV, int SK>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(const RotaryParams p) {
  __shared__ float2 s_angle[kRotaryMaxAngles];
  const int tid = threadIdx.x;
  const int half = p.rot >> 1;
  const unsigned first = blockIdx.x * (unsigned)p.tokens_per_group;
  const int tokens = (int)min((unsigned)p.tokens_per_group, (unsigned)p.tokens - first);
  const int lanes = 1 << p.log_lanes;  // lanes to a row
  const int u = tid & (lanes - 1);
  const int rot_units = p.interleaved ? (p.rot + 15) >> 4 : (half + 7) >> 3;
  const int rows = p.Hq + p.Hk + (KV == kKvNone ? 0 : p.Hk);
  const int stride = kRotaryThreads >> p.log_lanes, last = tokens * rows;
  const bool vec = p.vec != 0;

  // Row `task`: its token (t of this workgroup, (b, qi) of the call) and head (what: 0 q, 1 k, 2 v), and this lane's two chunks of
  // up to 8 channels: na from ca on, nb from cb on. Of rotated channels the lane has pairs 8 u ..: the chunks hold their
  // first and second channels, or (interleaved) both of four pairs each.
  struct Row {
    int t, what, h, ca, cb, na, nb;
    unsigned b, qi;
    bool turned;
  };
  auto row_of = [&](int task) {
    Row r;
    r.t = task / rows;
    r.h = task - r.t * rows;
    const unsigned tok = first + r.t;
    r.b = tok / (unsigned)p.Q, r.qi = tok - r.b * (unsigned)p.Q;
    r.what = r.h < p.Hq ? 0 : (r.h < p.Hq + p.Hk ? 1 : 2);
    r.h -= r.what == 0 ? 0 : (r.what == 1 ? p.Hq : p.Hq + p.Hk);
    r.turned = r.what != 2 && u < rot_units;
    if (r.turned && !p.interleaved) {
      r.ca = 8 * u, r.cb = half + 8 * u;
      r.na = r.nb = min(8, half - 8 * u);
    } else {
      r.ca = r.what == 2 || r.turned ? 16 * u : p.rot + 16 * (u - rot_units), r.cb = r.ca + 8;
      const int end = r.turned ? p.rot : p.D;
      r.na = max(min(8, end - r.ca), 0), r.nb = max(min(8, end - r.cb), 0);
    }
    return r;
  };
  auto load = [&](const Row& r, float* a, float* b) {
    const void* src = r.what == 0 ? p.q : (r.what == 1 ? p.k : p.v);
    const int64_t xi = r.what == 0 ? r.b * p.q_sb + r.qi * p.q_sq + r.h * p.q_sh : r.b * p.k_sb + r.qi * p.k_sq + r.h * p.k_sh;
    if (vec) {
      if (r.na > 0) {
        rotary_load8<X>(src, xi + r.ca, a);
        rotary_load8<X>(src, xi + r.cb, b);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j < r.na) a[j] = load_float(src, xi + r.ca + j, X);
        if (j < r.nb) b[j] = load_float(src, xi + r.cb + j, X);
      }
    }
  };

  // The first row's channels are on their way while the angles are computed.
  int task = tid >> p.log_lanes;
  Row r = row_of(min(task, last - 1));
  float a[8], b[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] = b[j] = 0.0f;
  load(r, a, b);
  for (int i = tid; i < tokens * half; i += kRotaryThreads) {
    const int t = i / half, f = i - t * half;
    const unsigned tok = first + t, tb = tok / (unsigned)p.Q, tq = tok - tb * (unsigned)p.Q;
    const int64_t pos = load_index(p.positions, p.axis[f] * p.pos_sa + tb * p.pos_sb + tq * p.pos_sq, p.pos_i64 != 0);
    const float2 cs = rotary_angle(pos, p.inv_freq[f]);
    s_angle[i] = make_float2(cs.x * p.scaling, cs.y * p.scaling);
  }
  __syncthreads();

  while (task < last) {
    const void* weight = r.what == 0 ? p.q_norm : p.k_norm;
    if (r.what != 2 && weight) {
      float wa[8], wb[8], sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) wa[j] = wb[j] = 0.0f;
      if (vec) {
        if (r.na > 0) {
          rotary_load_weights(weight, r.ca, p.norm_dtype, wa);
          rotary_load_weights(weight, r.cb, p.norm_dtype, wb);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j < r.na) wa[j] = load_float(weight, r.ca + j, p.norm_dtype);
          if (j < r.nb) wb[j] = load_float(weight, r.cb + j, p.norm_dtype);
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(a[j], a[j], fmaf(b[j], b[j], sum));
      for (int m = lanes >> 1; m >= 1; m >>= 1) sum += __shfl_xor(sum, m, 64);
      const float scale = 1.0f / sqrtf(sum / (float)p.D + p.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] = a[j] * scale * wa[j], b[j] = b[j] * scale * wb[j];
    }
    if (r.turned) {
      const float2* angle = s_angle + r.t * half + 8 * u;
      if (!p.interleaved) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j >= r.na) continue;
          const float2 cs = angle[j];
          const float x = a[j], y = b[j];
          a[j] = fmaf(-y, cs.y, x * cs.x);
          b[j] = fmaf(y, cs.x, x * cs.y);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (2 * (j & 3) >= (j < 4 ? r.na : r.nb)) continue;
          float* c = (j < 4 ? a : b) + 2 * (j & 3);
          const float2 cs = angle[j];
          const float x = c[0], y = c[1];
          c[0] = fmaf(-y, cs.y, x * cs.x);
          c[1] = fmaf(y, cs.x, x * cs.y);
        }
      }
    }

    if (KV == kKvNone || r.what == 0) {
      void* dst = r.what == 0 ? p.q_out : p.k_out;
      const int64_t yi = r.what == 0 ? r.b * p.qo_sb + r.qi * p.qo_sq + r.h * p.qo_sh : r.b * p.ko_sb + r.qi * p.ko_sq + r.h * p.ko_sh;
      if (vec) {
        if (r.na > 0) {
          rotary_store8<X>(dst, yi + r.ca, a);
          rotary_store8<X>(dst, yi + r.cb, b);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j < r.na) store_float(dst, yi + r.ca + j, X, a[j]);
          if (j < r.nb) store_float(dst, yi + r.cb + j, X, b[j]);
        }
      }
    } else if constexpr (KV != kKvNone) {  // into the pool: the row's slot, then its codes
      const int64_t si = r.b * p.s_sb + r.qi * p.s_sq;
      const int64_t blk = load_index(p.blocks, si, p.slot_i64 != 0), off = load_index(p.offsets, si, p.slot_i64 != 0);
      const bool live = blk >= 0 && blk < p.num_blocks && off >= 0 && off < p.P;
      float* scales = r.what == 1 ? p.ks : p.vs;
      float s = 1.0f;
      if constexpr (SK == kScaleHead) {
        s = scales[r.h];
      } else if constexpr (SK == kScaleTokenHead) {
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fmaxf(fabsf(a[j]), fabsf(b[j])));
        for (int m = lanes >> 1; m >= 1; m >>= 1) amax = fmaxf(amax, __shfl_xor(amax, m, 64));
        s = __fdiv_rn(amax, KV == kKvFp8 ? 448.0f : 127.0f);
        s = s < 1e-12f ? 1e-12f : s;
        if (live && u == 0) scales[blk * p.sc_sblk + off * p.sc_stok + r.h * p.sc_shead] = s;
      }
      if (live) {
        const float inv = __builtin_amdgcn_rcpf(s);
        const int eb = KV == kKvBf16 ? 2 : 1;
        uint8_t* dst = (r.what == 1 ? p.kc : p.vc) + blk * p.kv_sblk + off * p.kv_stok + r.h * p.kv_shead;
        if (r.na > 0) rotary_store_codes<KV, SK>(dst + eb * r.ca, a, s, inv, r.na, p.vec_pool && r.na == 8);
        if (r.nb > 0) rotary_store_codes<KV, SK>(dst + eb * r.cb, b, s, inv, r.nb, p.vec_pool && r.nb == 8);
      }
    }
    task += stride;
    if (task < last) {
      r = row_of(task);
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] = b[j] = 0.0f;
      load(r, a, b);
    }
  }
}

template <int KV, int SK>
static hipError_t launch_rotary_t(const RotaryParams& p, int x_dtype, hipStream_t stream) {
  const dim3 grid((unsigned)((p.tokens + p.tokens_per_group - 1) / p.tokens_per_group)), block(kRotaryThreads);
  if (x_dtype == kFBf16) hipLaunchKernelGGL((rotary_kernel<kFBf16, KV, SK>), grid, block, 0, stream, p);
  else if (x_dtype == kFF16) hipLaunchKernelGGL((rotary_kernel<kFF16, KV, SK>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((rotary_kernel<kFF32, KV, SK>), grid, block, 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_rotary(const RotaryParams& p, int x_dtype, bool pool, int kv_dtype, int scale_kind, hipStream_t stream) {
  if (!pool) return launch_rotary_t<kKvNone, kScaleNone>(p, x_dtype, stream);
  if (kv_dtype == kKvBf16) return launch_rotary_t<kKvBf16, kScaleNone>(p, x_dtype, stream);
  if (kv_dtype == kKvFp8 && scale_kind == kScaleHead) return launch_rotary_t<kKvFp8, kScaleHead>(p, x_dtype, stream);
  if (kv_dtype == kKvFp8 && scale_kind == kScaleTokenHead) return launch_rotary_t<kKvFp8, kScaleTokenHead>(p, x_dtype, stream);
  if (kv_dtype == kKvInt8 && scale_kind == kScaleHead) return launch_rotary_t<kKvInt8, kScaleHead>(p, x_dtype, stream);
  if (kv_dtype == kKvInt8 && scale_kind == kScaleTokenHead) return launch_rotary_t<kKvInt8, kScaleTokenHead>(p, x_dtype, stream);
  return hipErrorInvalidValue;
}

}  // namespace bpt
