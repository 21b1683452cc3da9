// Rotary positions: y = (a cos t - b sin t, b cos t + a sin t) * factor for
// the pairs (a, b) of the first rotary_dim columns, t = position * frequency.
// Pairs are columns (i, i + rotary_dim / 2) ("half") or (2 i, 2 i + 1)
// ("interleaved").  The frequencies come from the caller in 64 bits, already
// scaled for a long context.
//
// Angles are formed and reduced in 64 bits: at position 10^6 an f32 product is
// off by 0.06 rad.  After the reduction to [-pi/4, pi/4] sine and cosine are
// their Taylor sums, in f32 to the terms r^9 and r^10 (the next are 2e-9) or in
// f64 to r^15 and r^16 (5e-17).
//
// Products and sums are written as the fused operations they become, so that every
// kernel rounds a rotation alike.
//
// A wave holds one head of 256 columns, lane l the columns 4 l .. 4 l + 3; an
// angle is computed once, in one lane, and fetched from it.
#pragma once

#include "common.h"

namespace mi {

struct RotaryPlan {
  double freq[MI_ROPE_MAX_DIM / 2];
  double factor;
  int32_t half;         // rotary_dim / 2
  int32_t interleaved;
};

// Heads of a token that a wave takes in turn, with their angles once: for many rows,
// where a wave's instructions are what counts (105k f16 rows, 64 pairs, 108 MB: one head 24.9
// us, four 17.2); with few rows the chain of one wave does.
constexpr int kRotaryHeads = 4;
inline int rotary_heads(int64_t rows) { return rows < 16384 ? 1 : kRotaryHeads; }

// Checks and copies the caller's plan (host_freq may be null when rotary_dim
// is 0).
mi_status rotary_plan(const double* host_freq, int32_t rotary_dim, int32_t interleaved,
                      double factor, RotaryPlan* out);

// sin and cos of t (64 bits), as T.
template <typename T>
__device__ __forceinline__ void turn(double t, T& s, T& c) {
  constexpr double kHi = 1.5707963267948966, kLo = 6.123233995736766e-17;  // pi / 2
  const double k = rint(t * 0.63661977236758134308);
  const T r = (T)fma(-k, kLo, fma(-k, kHi, t));
  const T r2 = r * r;
  T ps, pc;
  if constexpr (sizeof(T) == 8) {
    ps = fma(r2, -1.0 / 1307674368000.0, 1.0 / 6227020800.0);
    ps = fma(r2, ps, -1.0 / 39916800.0);
    ps = fma(r2, ps, 1.0 / 362880.0);
    ps = fma(r2, ps, -1.0 / 5040.0);
    ps = fma(r2, ps, 1.0 / 120.0);
    ps = fma(r2, ps, -1.0 / 6.0);
    pc = fma(r2, 1.0 / 20922789888000.0, -1.0 / 87178291200.0);
    pc = fma(r2, pc, 1.0 / 479001600.0);
    pc = fma(r2, pc, -1.0 / 3628800.0);
    pc = fma(r2, pc, 1.0 / 40320.0);
    pc = fma(r2, pc, -1.0 / 720.0);
    pc = fma(r2, pc, 1.0 / 24.0);
    pc = fma(r2, pc, -0.5);
  } else {
    ps = fmaf(r2, 1.f / 362880.f, -1.f / 5040.f);
    ps = fmaf(r2, ps, 1.f / 120.f);
    ps = fmaf(r2, ps, -1.f / 6.f);
    pc = fmaf(r2, -1.f / 3628800.f, 1.f / 40320.f);
    pc = fmaf(r2, pc, -1.f / 720.f);
    pc = fmaf(r2, pc, 1.f / 24.f);
    pc = fmaf(r2, pc, -0.5f);
  }
  const T sr = fma(r * r2, ps, r), cr = fma(r2, pc, (T)1);
  const int quadrant = (int)(k - 4.0 * rint(k * 0.25)) & 3;  // -2 .. 2
  const T a = quadrant & 1 ? cr : sr, b = quadrant & 1 ? sr : cr;
  s = quadrant & 2 ? -a : a;
  c = (quadrant + 1) & 2 ? -b : b;
}

// The rotation of one position for a wave: the lane's (cos, sin) pairs, up to
// four (half) or two (interleaved), times the plan's factor.
template <typename T, bool ILV>
struct LaneTurn {
  static constexpr int N = ILV ? 2 : 4;
  T c[N], s[N];

  __device__ __forceinline__ void set(const RotaryPlan& p, double pos, int lane) {
    T ct[2] = {}, st[2] = {};
#pragma unroll
    for (int k = 0; k < 2; k++)
      if (lane + 64 * k < p.half) {
        turn<T>(pos * p.freq[lane + 64 * k], st[k], ct[k]);
        ct[k] *= (T)p.factor;
        st[k] *= (T)p.factor;
      }
    // first pair of the lane's columns
    const int p0 = ILV ? 2 * lane : (4 * lane < p.half ? 4 * lane : 4 * lane - p.half);
#pragma unroll
    for (int e = 0; e < N; e++) {
      c[e] = __shfl(ct[0], (p0 + e) & 63, 64);
      s[e] = __shfl(st[0], (p0 + e) & 63, 64);
      if (p.half > 64) {  // uniform
        const T c1 = __shfl(ct[1], (p0 + e) & 63, 64), s1 = __shfl(st[1], (p0 + e) & 63, 64);
        if (p0 + e >= 64) {
          c[e] = c1;
          s[e] = s1;
        }
      }
    }
  }

  // Rotates the lane's columns y of a head.
  __device__ __forceinline__ void apply(const RotaryPlan& p, T (&y)[4], int lane) const {
    if constexpr (ILV) {
      if (4 * lane < 2 * p.half) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const T a = y[2 * e], b = y[2 * e + 1];
          y[2 * e] = fma(a, c[e], -(b * s[e]));
          y[2 * e + 1] = fma(b, c[e], a * s[e]);
        }
      }
    } else {
      const bool lower = 4 * lane < p.half;
      const int partner = lower ? lane + (p.half >> 2) : lane - (p.half >> 2);
      T o[4];
#pragma unroll
      for (int e = 0; e < 4; e++) o[e] = __shfl(y[e], partner & 63, 64);
      if (4 * lane < 2 * p.half) {
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = fma(y[e], c[e], lower ? -(o[e] * s[e]) : o[e] * s[e]);
      }
    }
  }
};

// The value N lanes on in the lane's row of 16 (a data-parallel-primitive move, no LDS).
template <int N, typename T>
__device__ __forceinline__ T row_turn(T x) {
  if constexpr (sizeof(T) == 8) {
    const u32x2 w = __builtin_bit_cast(u32x2, x);
    const uint32_t lo = w[0], hi = w[1];
    return __builtin_bit_cast(T, u32x2{(uint32_t)__builtin_amdgcn_mov_dpp((int)lo, 0x120 + N, 0xf, 0xf, true),
                                       (uint32_t)__builtin_amdgcn_mov_dpp((int)hi, 0x120 + N, 0xf, 0xf, true)});
  } else {
    return __builtin_bit_cast(T, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x120 + N, 0xf, 0xf, true));
  }
}
// f over the lane's row of 16, in every lane of it.
template <typename T, typename F>
__device__ __forceinline__ T over_row(T x, F f) {
  x = f(x, row_turn<8>(x));
  x = f(x, row_turn<4>(x));
  x = f(x, row_turn<2>(x));
  return f(x, row_turn<1>(x));
}
// Sum over a wave.
template <typename T>
__device__ __forceinline__ T wave_sum(T x) {
  x = over_row(x, [](T a, T b) { return a + b; });
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}

// RMS norm of a head with bf16 weights, in T.
template <typename T>
__device__ __forceinline__ void rms_norm(T (&y)[4], const uint16_t* w, double eps, int lane) {
  const T ss = wave_sum<T>(fma(y[0], y[0], fma(y[1], y[1], fma(y[2], y[2], y[3] * y[3]))));
  T inv;
  if constexpr (sizeof(T) == 8) inv = 1.0 / sqrt(ss / kHeadDim + eps);
  else inv = 1.f / sqrtf(ss / (float)kHeadDim + (float)eps);
  const ushort4 wb = *(const ushort4*)(w + 4 * lane);
  y[0] = y[0] * inv * (T)bf16_to_f32(wb.x);
  y[1] = y[1] * inv * (T)bf16_to_f32(wb.y);
  y[2] = y[2] * inv * (T)bf16_to_f32(wb.z);
  y[3] = y[3] * inv * (T)bf16_to_f32(wb.w);
}

// Four consecutive values of an f32, f16 or bf16 (uint16_t) row.
struct bf16 { uint16_t bits; };
__device__ __forceinline__ float4 load4(const float* p) { return *(const float4*)p; }
__device__ __forceinline__ float4 load4(const _Float16* p) {
  const f16x4 v = *(const f16x4*)p;
  return {(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
}
__device__ __forceinline__ float4 load4(const bf16* p) {
  const ushort4 v = *(const ushort4*)p;
  return {bf16_to_f32(v.x), bf16_to_f32(v.y), bf16_to_f32(v.z), bf16_to_f32(v.w)};
}
__device__ __forceinline__ uint16_t f32_to_bf16(float x) {  // nearest, ties to even
  const uint32_t u = __float_as_uint(x);
  if (x != x) return (uint16_t)((u >> 16) | 0x40);
  return (uint16_t)((u + 0x7fff + ((u >> 16) & 1)) >> 16);
}
// PAST: past the caches, for more rows than they keep (4099 tokens of 16 heads 18.6 us
// without and 17.9; prompts of 6580 tokens appended 31.4 and 29.1: the calls alone, without
// the one that reads the rows next).
template <bool PAST, typename V>
__device__ __forceinline__ void put(V* p, V x) {
  if constexpr (PAST) __builtin_nontemporal_store(x, p);
  else *p = x;
}
template <bool PAST>
__device__ __forceinline__ void store4(float* p, const float (&y)[4]) {
  put<PAST>((f32x4*)p, f32x4{y[0], y[1], y[2], y[3]});
}
template <bool PAST>
__device__ __forceinline__ void store4(_Float16* p, const float (&y)[4]) {
  put<PAST>((f16x4*)p, f16x4{(_Float16)y[0], (_Float16)y[1], (_Float16)y[2], (_Float16)y[3]});
}
template <bool PAST>
__device__ __forceinline__ void store4(bf16* p, const float (&y)[4]) {
  typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
  put<PAST>((u16x4*)p, u16x4{f32_to_bf16(y[0]), f32_to_bf16(y[1]), f32_to_bf16(y[2]), f32_to_bf16(y[3])});
}

}  // namespace mi
