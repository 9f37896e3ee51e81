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
// rotation needs no exchange, and 16-bit rows are loaded and stored 16 bytes at a time. Row sums and maxima are
// butterflies over the group.
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

template <int X>
__device__ __forceinline__ uint32_t rotary_pack2(float a, float b) {
  if constexpr (X == kFBf16) return (uint32_t)f32_to_bf16_bits(a) | ((uint32_t)f32_to_bf16_bits(b) << 16);
  else return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16);
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

template <int X, int KV, int SK>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(const RotaryParams p) {
  __shared__ float2 s_angle[kRotaryMaxAngles];
  const int tid = threadIdx.x;
  const int half = p.rot >> 1;
  const int64_t first = (int64_t)blockIdx.x * p.tokens_per_group;
  const int tokens = (int)min((int64_t)p.tokens_per_group, p.tokens - first);
  for (int i = tid; i < tokens * half; i += kRotaryThreads) {
    const int t = i / half, f = i - t * half;
    const int64_t tok = first + t, b = tok / p.Q, qi = tok - b * p.Q;
    const int64_t pos = load_index(p.positions, p.axis[f] * p.pos_sa + b * p.pos_sb + qi * p.pos_sq, p.pos_i64 != 0);
    const float2 cs = rotary_angle(pos, p.inv_freq[f]);
    s_angle[i] = make_float2(cs.x * p.scaling, cs.y * p.scaling);
  }
  __syncthreads();

  const int lanes = 1 << p.log_lanes;  // lanes to a row
  const int u = tid & (lanes - 1);
  const int rot_units = (half + 7) >> 3;
  const bool turned = u < rot_units;
  const int rows = p.Hq + p.Hk + (KV == kKvNone ? 0 : p.Hk);
  const int stride = kRotaryThreads >> p.log_lanes;
  for (int task = tid >> p.log_lanes; task < tokens * rows; task += stride) {
    const int t = task / rows;
    int h = task - t * rows;
    const int64_t tok = first + t, b = tok / p.Q, qi = tok - b * p.Q;
    const int what = h < p.Hq ? 0 : (h < p.Hq + p.Hk ? 1 : 2);  // 0: q, 1: k, 2: v
    h -= what == 0 ? 0 : (what == 1 ? p.Hq : p.Hq + p.Hk);
    const void* src = what == 0 ? p.q : (what == 1 ? p.k : p.v);
    const int64_t xi = what == 0 ? b * p.q_sb + qi * p.q_sq + h * p.q_sh : b * p.k_sb + qi * p.k_sq + h * p.k_sh;
    const bool rotate = what != 2;

    // This lane's 16 channels as a[j], b_[j], and where they lie: a[j] at ca + j * step, b_[j] at cb + j * step.
    int ca, cb, step = 1, na, nb;
    if (rotate && turned) {
      na = nb = min(8, half - 8 * u);
      ca = p.interleaved ? 16 * u : 8 * u;
      cb = p.interleaved ? ca + 1 : half + ca;
      step = p.interleaved ? 2 : 1;
    } else {
      ca = rotate ? p.rot + 16 * (u - rot_units) : 16 * u;
      cb = ca + 8;
      na = min(8, p.D - ca);
      nb = min(8, p.D - cb);
    }
    float a[8], b_[8];
    if (p.vec) {
      if (na > 0) {
        if (step == 1) {
          rotary_load8<X>(src, xi + ca, a);
          rotary_load8<X>(src, xi + cb, b_);
        } else {
          float v[16];
          rotary_load8<X>(src, xi + ca, v);
          rotary_load8<X>(src, xi + ca + 8, v + 8);
#pragma unroll
          for (int j = 0; j < 8; ++j) a[j] = v[2 * j], b_[j] = v[2 * j + 1];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = b_[j] = 0.0f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        a[j] = j < na ? load_float(src, xi + ca + j * step, X) : 0.0f;
        b_[j] = j < nb ? load_float(src, xi + cb + j * step, X) : 0.0f;
      }
    }

    const void* weight = what == 0 ? p.q_norm : p.k_norm;
    if (rotate && weight) {
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(a[j], a[j], fmaf(b_[j], b_[j], sum));
      for (int m = lanes >> 1; m >= 1; m >>= 1) sum += __shfl_xor(sum, m, 64);
      const float r = 1.0f / sqrtf(sum / (float)p.D + p.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j < na) a[j] = a[j] * r * load_float(weight, ca + j * step, p.norm_dtype);
        if (j < nb) b_[j] = b_[j] * r * load_float(weight, cb + j * step, p.norm_dtype);
      }
    }
    if (rotate && turned) {
      const float2* angle = s_angle + t * half + 8 * u;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j < na) {
          const float2 cs = angle[j];
          const float x = a[j], y = b_[j];
          a[j] = fmaf(-y, cs.y, x * cs.x);
          b_[j] = fmaf(y, cs.x, x * cs.y);
        }
      }
    }

    if (KV == kKvNone || what == 0) {
      void* dst = what == 0 ? p.q_out : p.k_out;
      const int64_t yi = what == 0 ? b * p.qo_sb + qi * p.qo_sq + h * p.qo_sh : b * p.ko_sb + qi * p.ko_sq + h * p.ko_sh;
      if (p.vec) {
        if (na > 0) {
          if (step == 1) {
            rotary_store8<X>(dst, yi + ca, a);
            rotary_store8<X>(dst, yi + cb, b_);
          } else {
            float v[16];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[2 * j] = a[j], v[2 * j + 1] = b_[j];
            rotary_store8<X>(dst, yi + ca, v);
            rotary_store8<X>(dst, yi + ca + 8, v + 8);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j < na) store_float(dst, yi + ca + j * step, X, a[j]);
          if (j < nb) store_float(dst, yi + cb + j * step, X, b_[j]);
        }
      }
      continue;
    }

    if constexpr (KV != kKvNone) {  // into the pool: the row's slot, then its codes
      const int64_t si = b * p.s_sb + qi * p.s_sq;
      const int64_t blk = load_index(p.blocks, si, p.slot_i64 != 0), off = load_index(p.offsets, si, p.slot_i64 != 0);
      const bool live = blk >= 0 && blk < p.num_blocks && off >= 0 && off < p.P;
      const int64_t ci = blk * p.kv_sblk + off * p.kv_stok + h * p.kv_shead;
      uint8_t* pool = what == 1 ? p.kc : p.vc;
      float* scales = what == 1 ? p.ks : p.vs;
      float s = 1.0f;
      if constexpr (SK == kScaleHead) {
        s = scales[h];
      } else if constexpr (SK == kScaleTokenHead) {
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fmaxf(fabsf(a[j]), fabsf(b_[j])));
        for (int m = lanes >> 1; m >= 1; m >>= 1) amax = fmaxf(amax, __shfl_xor(amax, m, 64));
        s = __fdiv_rn(amax, KV == kKvFp8 ? 448.0f : 127.0f);
        s = s < 1e-12f ? 1e-12f : s;
        if (live && u == 0) scales[blk * p.sc_sblk + off * p.sc_stok + h * p.sc_shead] = s;
      }
      if (!live) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (j >= (k ? nb : na)) continue;
          const float x = k ? b_[j] : a[j];
          const int c = (k ? cb : ca) + j * step;
          if constexpr (KV == kKvBf16) {
            ((uint16_t*)(pool + ci))[c] = f32_to_bf16_bits(x);
          } else {
            const float y = __fdiv_rn(x, s);
            uint32_t code;
            if constexpr (KV == kKvFp8) {
              code = f32_to_fp8(clamp_fp8_range(y));
            } else {
              float r = rintf(y);
              r = r > 127.0f ? 127.0f : (r < -128.0f ? -128.0f : r);
              code = (uint32_t)(int32_t)r & 0xffu;
            }
            pool[ci + c] = (uint8_t)code;
          }
        }
      }
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
