// What the kernels of attention over the paged 4-bit cache share: their
// arguments, the walk over a ragged batch, the output.
#pragma once

#include "paged.h"

namespace mi {

constexpr float kNegBig = -1e30f;  // below every score's base-2 exponent

struct AttnArgs {
  PagedView pv;
  const _Float16* q;
  int64_t q_ts, q_hs;
  const void* gate;  // f16, or f32 (gate32), or null
  int64_t g_ts, g_hs;
  _Float16* out;     // [n][G R][D]
  float* part_o;     // [2 workgroups][16 CT][D]
  float* part_ml;    // [2 workgroups][16 CT][2]
  int2* seg;         // [batch G]: first slot and last workgroup of an item, or -1
  int32_t n, R, max_q, max_len, wgs, gate32, dsplit;
};

// Four values of the gate, from element gi on.
__device__ __forceinline__ f32x4 gate4(const AttnArgs& a, int64_t gi) {
  if (a.gate32) return *(const f32x4*)((const float*)a.gate + gi);
  const f16x4 h = *(const f16x4*)((const _Float16*)a.gate + gi);
  return f32x4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
}

// out of four columns: their sums x times inv, the weights' sum's inverse, the gate, then
// f16.  inv is 0 for a token that attends nothing: zeros, whatever its gate holds.
__device__ __forceinline__ void put4(const AttnArgs& a, int64_t tok, int head, int d, f32x4 x, float inv) {
  x *= inv;
  if (a.gate && inv != 0.f) {
    const f32x4 g = gate4(a, tok * a.g_ts + head * a.g_hs + d);
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = gate_mul(x[e], g[e]);
  }
  *(f16x4*)(a.out + (tok * a.pv.G * a.R + head) * kHeadDim + d) =
      f16x4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
  return (int64_t)((uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32 | (uint32_t)uniform((int)x));
}

// Sum over the workgroup and the exclusive prefix of each thread's x.
template <int NT, typename T>
__device__ __forceinline__ T block_scan(T x, T& before, T* lds) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  T run = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const T y = __shfl_up(run, d, 64);
    if (lane >= d) run += y;
  }
  __syncthreads();  // lds may hold an earlier scan's
  if (lane == 63) lds[w] = run;
  __syncthreads();
  T base = 0, total = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; i++) {
    if (i < w) base += lds[i];
    total += lds[i];
  }
  before = base + run - x;
  return uniform(total);
}

// The sequence s that holds weight unit `unit(total weight)` of weight(s), and the
// weight before it; s = 0 where no sequence does.  (The weights' sum fits T.)
template <int NT, typename T, typename W, typename F>
__device__ __forceinline__ void find_seq(int batch, W weight, F unit, int& s, T& before) {
  __shared__ T lds[NT / 64 + 2];
  const int t = threadIdx.x;
  s = 0;
  before = 0;
  if (batch == 1) {
    unit(uniform(weight(0)));
    return;
  }
  T total = 0, pre = 0, x = 0;
  for (int c = 0; c < batch; c += NT) {
    x = c + t < batch ? weight(c + t) : T(0);
    total += block_scan<NT>(x, pre, lds);
  }
  const T want = unit(total);
  if (want >= total) return;
  T base = 0;
  for (int c = 0; c < batch; c += NT) {
    if (batch > NT) {  // one pass of a small batch has them already
      x = c + t < batch ? weight(c + t) : T(0);
      const T sum = block_scan<NT>(x, pre, lds);
      if (want >= base + sum) {  // uniform
        base += sum;
        continue;
      }
    }
    if (base + pre <= want && want < base + pre + x) {
      lds[NT / 64] = c + t;
      lds[NT / 64 + 1] = base + pre;
    }
    break;
  }
  __syncthreads();
  s = uniform((int)lds[NT / 64]);
  before = uniform(lds[NT / 64 + 1]);
}

// Eight columns of Q in dequant_row's order.
__device__ __forceinline__ f16x8 in_order(f16x8 x) {
  return f16x8{x[0], x[4], x[1], x[5], x[2], x[6], x[3], x[7]};
}

// The prompts' form (paged_prefill.hip): workspace bytes, and the launches.
size_t paged_prefill_workspace();
mi_status paged_prefill(AttnArgs& a, void* workspace, hipStream_t s);

}  // namespace mi
