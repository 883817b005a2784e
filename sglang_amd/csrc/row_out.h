// Rows of 16-bit activations to rows of 8-bit codes with one scale per row, fused with what produces the row: a residual
// addition and RMSNorm, SiLU(gate) * up, or nothing.  Nothing is rounded between the loads and the codes.
//
//   RMS:   v = x + residual;  u = v * w;  y = u * r,  r = 1 / sqrt(mean(v^2) + eps)
//   SILU:  y = gate / (1 + exp(-gate)) * up
//   PLAIN: y = x
//   e4m3:       scale = max|y| / 448 or as given;  code = e4m3(clamp(y * (1 / scale), +-448)), zeros for a scale of zero
//   int8:       amax = max(max|y|, 1e-10);  scale = amax / 127;  code = round_half_away(y * (127 / amax))
//   asymmetric: lo = min(0, min y), hi = max(0, max y);  scale = max(hi - lo, 1e-10) / 255;  zp = rint(-128 - lo / scale);
//               code = clamp(rint(y * (1 / scale)) + zp, -128, 127)
//
// The extremes of y are r times those of u (r > 0), so the sum of squares and the extremes meet in ONE exchange between a
// row's lanes, and r enters the codes as a factor of their multiplier: a row is read once, stays in registers, and its
// workgroup waits for one barrier.
//
// A row that holds a NaN or an infinity (RMS: whose sum of squares is not finite) gets a scale that is NaN or infinite, so
// that it cannot pass for numbers behind the product.  The extremes are compared as the bits of non-negative floats, in
// whose order infinity and then NaN come last; fmaxf would drop a NaN.
#pragma once
#include "quant_core.h"

namespace sglamd {

enum { ROW_RMS = 0, ROW_SILU = 1, ROW_PLAIN = 2 };
enum { ROW_TO_FP8 = 0, ROW_TO_INT8 = 1, ROW_TO_ASYM = 2 };

struct RowOutArgs {
  const void* x;     // rows of `hidden` values, SILU: of [gate | up], 2 * hidden
  int64_t x_stride;  // elements between rows
  const void* res;   // RMS: optional
  int64_t res_stride;
  void* res_out;     // RMS: x + res in the activations' type, [rows, hidden]
  const void* w;     // RMS: [hidden]
  float eps;
  void* y;             // RMS: optional, the row before its codes, in the activations' type, [rows, hidden]
  uint8_t* q;          // [rows, hidden]
  float* s;            // [rows]
  int32_t* zp;         // asymmetric: [rows]
  const float* fixed;  // e4m3: optional, the one scale
  int64_t hidden, rows;
};

// Sum and maximum over the wave, in all lanes: rows of 16 lanes by DPP, the four rows by v_readlane.
template <int CTRL>
__device__ __forceinline__ float dpp_f(float v) {
  const int x = __float_as_int(v);
  return __int_as_float(__builtin_amdgcn_update_dpp(x, x, CTRL, 0xf, 0xf, false));
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
}
__device__ __forceinline__ float lanes16_sum(float v) {
  v += dpp_f<0xB1>(v);   // quad_perm [1, 0, 3, 2]
  v += dpp_f<0x4E>(v);   // quad_perm [2, 3, 0, 1]
  v += dpp_f<0x141>(v);  // row_half_mirror
  v += dpp_f<0x140>(v);  // row_mirror
  return v;
}
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t lanes8_umax(uint32_t v) {
  v = umax(v, dpp_u<0xB1>(v));
  v = umax(v, dpp_u<0x4E>(v));
  return umax(v, dpp_u<0x141>(v));
}
__device__ __forceinline__ uint32_t lanes16_umax(uint32_t v) {
  v = lanes8_umax(v);
  return umax(v, dpp_u<0x140>(v));
}
__device__ __forceinline__ float wave_sum(float v) {
  const int x = __float_as_int(lanes16_sum(v));
  const float a = __int_as_float(__builtin_amdgcn_readlane(x, 0)), b = __int_as_float(__builtin_amdgcn_readlane(x, 16));
  const float c = __int_as_float(__builtin_amdgcn_readlane(x, 32)), d = __int_as_float(__builtin_amdgcn_readlane(x, 48));
  return (a + b) + (c + d);
}
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
  const int x = (int)lanes16_umax(v);
  return umax(umax((uint32_t)__builtin_amdgcn_readlane(x, 0), (uint32_t)__builtin_amdgcn_readlane(x, 16)),
              umax((uint32_t)__builtin_amdgcn_readlane(x, 32), (uint32_t)__builtin_amdgcn_readlane(x, 48)));
}

// What a row's lanes exchange: the sum of squares, the largest value (symmetric codes: magnitude) and the largest of the
// negated ones, the last two as the bits of non-negative floats.
struct RowStats {
  float ss;
  uint32_t hi, lo;
};
template <int SRC, int QK>
__device__ __forceinline__ RowStats row_stats_wave(RowStats t) {
  if (SRC == ROW_RMS) t.ss = wave_sum(t.ss);
  t.hi = wave_umax(t.hi & 0x7fffffffu);  // (the larger of two zeros may be the negative one)
  if (QK == ROW_TO_ASYM) t.lo = wave_umax(t.lo & 0x7fffffffu);
  return t;
}
// Over the workgroup's waves (at most 16).
template <int SRC, int QK>
__device__ __forceinline__ RowStats row_stats_block(RowStats t, uint32_t* red) {
  t = row_stats_wave<SRC, QK>(t);
  const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6, l = threadIdx.x & 15;
  if ((threadIdx.x & 63) == 0) {
    red[wave] = __float_as_uint(t.ss);
    red[16 + wave] = t.hi;
    red[32 + wave] = t.lo;
  }
  __syncthreads();
  const bool mine = l < waves;
  if (SRC == ROW_RMS) t.ss = lanes16_sum(mine ? __uint_as_float(red[l]) : 0.f);
  t.hi = lanes16_umax(mine ? red[16 + l] : 0u);
  if (QK == ROW_TO_ASYM) t.lo = lanes16_umax(mine ? red[32 + l] : 0u);
  return t;
}

// One value into its lane's statistics.
template <int SRC, int QK>
__device__ __forceinline__ void row_stats_add(RowStats& t, float y) {
  if (QK == ROW_TO_ASYM) {
    // (a NaN compares as neither, and is caught by row_stats_poison)
    t.hi = __float_as_uint(fmaxf(__uint_as_float(t.hi), y));
    t.lo = __float_as_uint(fmaxf(__uint_as_float(t.lo), -y));
  } else {
    t.hi = umax(t.hi, __float_as_uint(y) & 0x7fffffffu);
  }
}
// Asymmetric codes: `poison` is a sum of 0 * y, NaN exactly where a value is not finite.
__device__ __forceinline__ void row_stats_poison(RowStats& t, float poison) {
  if (poison != 0.f) t.hi = 0x7fc00000u;
}

// What turns a value into an e4m3 code's: finite, so that a zero in a row whose scale has no reciprocal in 32 bits (values below
// 1e-36) stays a zero.
__device__ __forceinline__ float fp8_row_multiplier(float r, float scale) {
  const float mul = scale == 0.f ? 0.f : r / scale;
  return mul > 3.4028234664e38f ? 3.4028234664e38f : mul;  // (a NaN stays one)
}

// How the values of a row become codes: code = convert(value * mul) (asymmetric: + zp).
struct RowScale {
  float scale, mul, zp, r;  // r: RMS, what turns u into y
};
template <int SRC, int QK>
__device__ __forceinline__ RowScale row_scale(const RowOutArgs& a, const RowStats& t) {
  RowScale o;
  o.r = 1.f;
  o.zp = 0.f;
  float bad = 0.f;
  if (SRC == ROW_RMS) {
    o.r = rsqrtf(t.ss / (float)a.hidden + a.eps);
    if (!(t.ss < INFINITY)) bad = NAN;
  }
  const float hi = __uint_as_float(t.hi) * o.r;
  if constexpr (QK == ROW_TO_FP8) {
    o.scale = a.fixed ? *a.fixed : hi / 448.0f;
    o.mul = fp8_row_multiplier(o.r, o.scale);
  } else if constexpr (QK == ROW_TO_INT8) {
    const float amax = hi > 1e-10f || hi != hi ? hi : 1e-10f;
    o.scale = amax / 127.0f;
    o.mul = o.r * (127.0f / amax);
  } else {
    // (half the span: that of finite values may be beyond fp32; halves round as the whole does)
    const float lo = __uint_as_float(t.lo) * o.r, half = 0.5f * hi + 0.5f * lo;
    o.scale = (half > 0.5e-10f || half != half ? half : 0.5e-10f) / 127.5f;
    o.mul = o.r / o.scale;
    o.zp = __builtin_amdgcn_fmed3f(rintf(-128.0f + lo / o.scale), -128.f, 127.f);
  }
  // (a scale that is given stays what it is; there the codes become NaN, which e4m3 has)
  if (QK == ROW_TO_FP8 && a.fixed) o.mul += bad;
  else o.scale += bad;
  return o;
}

template <int QK>
__device__ __forceinline__ uint32_t row_codes4(const float* v, const RowScale& o) {
  float x[4];
#pragma unroll
  for (int j = 0; j < 4; j++) x[j] = v[j] * o.mul;
  if constexpr (QK == ROW_TO_FP8) {
    // the clamp of a NaN would be -448
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = x[j] != x[j] ? x[j] : __builtin_amdgcn_fmed3f(x[j], -448.f, 448.f);
    return pack4_e4m3(x[0], x[1], x[2], x[3]);
  } else if constexpr (QK == ROW_TO_INT8) {
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = __builtin_amdgcn_fmed3f(x[j], -127.f, 127.f);
    return pack4_low(round_away(x[0]), round_away(x[1]), round_away(x[2]), round_away(x[3]));
  } else {
    int c[4];
#pragma unroll
    for (int j = 0; j < 4; j++) c[j] = (int)__builtin_amdgcn_fmed3f(rintf(x[j]) + o.zp, -128.f, 127.f);
    return pack4_low(c[0], c[1], c[2], c[3]);
  }
}

}  // namespace sglamd
