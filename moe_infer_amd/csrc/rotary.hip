// Rotary positions of one tensor, with an optional RMS norm before.
//
// Bound: memory for many tokens; the chain of one wave for few.  A wave takes
// one head of a token, or four with their angles once (mi::LaneTurn).
#include "rotary.h"

#include <algorithm>
#include <cmath>
#include <cstring>

namespace {

struct RopeApplyArgs {
  const void* x;
  int64_t ts, hs;         // token and head stride of x, in elements
  const void* positions;  // int32 or int64 [n]
  const uint16_t* norm_w;  // bf16 [D] or null
  void* out;              // [n][heads][D]
  int32_t n, heads, pos64;
  double eps;
  mi::RotaryPlan plan;
};

template <typename TI, typename TO, bool ILV, int EACH>
__global__ void __launch_bounds__(256) rope_apply_kernel(const RopeApplyArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t item = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 4 +
                       __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int groups = (a.heads + EACH - 1) / EACH;
  const int64_t tok = item / groups;
  if (tok >= a.n) return;
  const int h0 = (int)(item - tok * groups) * EACH;
  float4 x[EACH];
#pragma unroll
  for (int i = 0; i < EACH; i++)
    x[i] = mi::load4((const TI*)a.x + tok * a.ts + min(h0 + i, a.heads - 1) * a.hs + 4 * lane);
  const double pos = a.pos64 ? (double)((const int64_t*)a.positions)[tok]
                             : (double)((const int32_t*)a.positions)[tok];
  mi::LaneTurn<float, ILV> t;
  t.set(a.plan, pos, lane);
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    if (h0 + i >= a.heads) break;  // uniform
    float y[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    if (a.norm_w) mi::rms_norm<float>(y, a.norm_w, a.eps, lane);
    t.apply(a.plan, y, lane);
    mi::store4<EACH != 1>((TO*)a.out + (tok * a.heads + h0 + i) * mi::kHeadDim + 4 * lane, y);
  }
}

template <typename TI, typename TO>
hipError_t run(const RopeApplyArgs& a, hipStream_t s) {
  const int each = mi::rotary_heads((int64_t)a.n * a.heads);
  const int64_t wgs = ((int64_t)a.n * ((a.heads + each - 1) / each) + 3) / 4;
  const int64_t gx = std::min<int64_t>(wgs, 1 << 22);
  const auto f = each == 1 ? (a.plan.interleaved ? rope_apply_kernel<TI, TO, true, 1>
                                                 : rope_apply_kernel<TI, TO, false, 1>)
                           : (a.plan.interleaved ? rope_apply_kernel<TI, TO, true, mi::kRotaryHeads>
                                                 : rope_apply_kernel<TI, TO, false, mi::kRotaryHeads>);
  return mi::launch("rope_apply", f, dim3((unsigned)gx, (unsigned)((wgs + gx - 1) / gx)), dim3(256), 0, s,
                    a);
}
template <typename TI>
hipError_t run(const RopeApplyArgs& a, int32_t out_type, hipStream_t s) {
  if (out_type == MI_F32) return run<TI, float>(a, s);
  if (out_type == MI_F16) return run<TI, _Float16>(a, s);
  return run<TI, mi::bf16>(a, s);
}

}  // namespace

namespace mi {

mi_status rotary_plan(const double* host_freq, int32_t rotary_dim, int32_t interleaved,
                      double factor, RotaryPlan* out) {
  if (rotary_dim < 0 || rotary_dim % 8 || rotary_dim > kHeadDim || rotary_dim > MI_ROPE_MAX_DIM)
    return fail(MI_ERR_INVALID_ARG, "rotary_dim=%d (multiple of 8, at most %d)", rotary_dim,
                std::min<int>(kHeadDim, MI_ROPE_MAX_DIM));
  if (rotary_dim && !host_freq) return fail(MI_ERR_INVALID_ARG, "null rotation frequencies");
  if (!std::isfinite(factor)) return fail(MI_ERR_INVALID_ARG, "rotation factor %g", factor);
  for (int i = 0; i < rotary_dim / 2; i++)
    if (!std::isfinite(host_freq[i]))
      return fail(MI_ERR_INVALID_ARG, "rotation frequency %d is %g", i, host_freq[i]);
  if (rotary_dim) memcpy(out->freq, host_freq, sizeof(double) * (rotary_dim / 2));
  out->factor = factor;
  out->half = rotary_dim / 2;
  out->interleaved = interleaved != 0;
  return MI_OK;
}

mi_status check_rows(const char* name, const void* p, int32_t type, int64_t ts, int64_t hs,
                     int64_t heads) {
  const int64_t size = type == MI_F32 ? 4 : 2;
  if (type < MI_F32 || type > MI_BF16) return fail(MI_ERR_INVALID_ARG, "%s: type %d", name, type);
  if (!p) return fail(MI_ERR_INVALID_ARG, "%s is null", name);
  if (((uintptr_t)p | (uint64_t)(ts * size) | (uint64_t)(hs * size)) & 15)
    return fail(MI_ERR_INVALID_ARG, "%s: rows must be 16-byte aligned", name);
  if (hs < kHeadDim || (heads > 1 && ts < kHeadDim) || ts < 0)
    return fail(MI_ERR_INVALID_ARG, "%s: strides %lld, %lld", name, (long long)ts, (long long)hs);
  return MI_OK;
}

bool overlaps(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  const char *x = (const char*)a, *y = (const char*)b;
  return x && y && x < y + b_bytes && y < x + a_bytes;
}

}  // namespace mi

extern "C" mi_status mi_rope_apply(const void* x, int32_t x_type, int64_t token_stride,
                                   int64_t head_stride, int32_t n, int32_t heads, int32_t head_dim,
                                   const void* positions, int32_t positions_64,
                                   const uint16_t* norm_w, float eps, const double* host_freq,
                                   int32_t rotary_dim, int32_t interleaved, double factor,
                                   void* out, int32_t out_type, mi_stream stream) {
  mi::clear_error();
  if (head_dim != mi::kHeadDim)
    return mi::fail(MI_ERR_UNSUPPORTED, "head_dim=%d (the kernels are built for %d)", head_dim,
                    mi::kHeadDim);
  if (n <= 0 || heads <= 0) return mi::fail(MI_ERR_INVALID_ARG, "n=%d heads=%d", n, heads);
  MI_TRY(mi::check_rows("x", x, x_type, token_stride, head_stride, heads));
  MI_TRY(mi::check_rows("out", out, out_type, (int64_t)heads * mi::kHeadDim, mi::kHeadDim, heads));
  if (!positions) return mi::fail(MI_ERR_INVALID_ARG, "null positions");
  if (!(eps >= 0.f)) return mi::fail(MI_ERR_INVALID_ARG, "eps=%g", (double)eps);
  RopeApplyArgs a{};
  MI_TRY(mi::rotary_plan(host_freq, rotary_dim, interleaved, factor, &a.plan));
  const int64_t xs = x_type == MI_F32 ? 4 : 2, os = out_type == MI_F32 ? 4 : 2;
  const bool same = x == out && x_type == out_type && head_stride == mi::kHeadDim &&
                    token_stride == (int64_t)heads * mi::kHeadDim;
  if (!same &&
      mi::overlaps(x, xs * mi::rows_extent(n, heads, token_stride, head_stride), out,
                   os * n * heads * mi::kHeadDim))
    return mi::fail(MI_ERR_INVALID_ARG, "out overlaps x (it may only be x itself)");
  a.x = x;
  a.ts = token_stride;
  a.hs = head_stride;
  a.positions = positions;
  a.pos64 = positions_64;
  a.norm_w = norm_w;
  a.out = out;
  a.n = n;
  a.heads = heads;
  a.eps = eps;
  const hipStream_t s = (hipStream_t)stream;
  MI_HIP(x_type == MI_F32   ? run<float>(a, out_type, s)
         : x_type == MI_F16 ? run<_Float16>(a, out_type, s)
                            : run<mi::bf16>(a, out_type, s));
  return MI_OK;
}
