// Attention over the paged 4-bit cache (paged.h): decode steps, drafts to
// verify, chunks and prompts.
//
// The columns of a (sequence, KV head) are its (token, query head of the
// group) pairs, token-major; a workgroup takes CT blocks of 16 of them and a
// range of 32-row tiles, which its four waves take in turn.  A wave's tile:
//   S [32 keys x 16 CT] = K Q^T    16x16x32 MFMA, K dequantised in registers
//   running maximum and sum per column (f32), P = 2^(S - max) in f16
//   O^T [256 x 16 CT] += V^T P     V dequantised in registers
// The row order within a tile (paged.h) makes S's accumulator layout the
// operand layout of P, so nothing goes through LDS between the products.  K of
// the next tile is loaded into K's registers while P V runs, V into V's while
// K Q^T runs.
#include <algorithm>
#include <cmath>

#include "paged.h"

namespace {

constexpr int D = mi::kHeadDim;
constexpr float kNegBig = -1e30f;
constexpr int kWaves = 4;
constexpr int kColPitch = D + 4;  // f32 per column of the merge buffer

struct AttnArgs {
  mi::PagedView pv;
  const _Float16* q;
  int64_t q_ts, q_hs;
  const void* gate;  // f16, or f32 (gate32), or null
  int64_t g_ts, g_hs;
  _Float16* out;     // [n][G R][D]
  float* part_o;     // [item][split][16 CT][D]
  float* part_ml;    // [item][split][16 CT][2]
  int32_t n, R, max_q, max_len, splits, ncb, gate32;
};

// One item: a block of columns of a sequence and KV head.
struct Item {
  int s, h, q0, nq, len;
  int c0;       // first column
  int ntiles;   // tiles that some column of it sees
  bool bad;     // beyond max_q or max_len
};

template <int CT>
__device__ __forceinline__ Item get_item(const AttnArgs& a, int64_t item) {
  Item it;
  const int cb = (int)(item % a.ncb);
  const int64_t sh = item / a.ncb;
  it.s = (int)(sh / a.pv.G);
  it.h = (int)(sh - (int64_t)it.s * a.pv.G);
  a.pv.tokens(it.s, it.q0, it.nq);
  it.len = a.pv.kv_len[it.s];
  it.bad = it.len < 0 || it.len > a.max_len || it.nq > a.max_q;
  if (it.nq <= 0 || it.q0 < 0 || (int64_t)it.q0 + it.nq > a.n) it.nq = 0;
  it.c0 = cb * 16 * CT;
  const int last = min(it.nq - 1, (it.c0 + 16 * CT - 1) / a.R);
  const int end = it.len - it.nq + last + 1;
  it.ntiles = it.bad || it.c0 >= it.nq * a.R || end <= 0 ? 0 : (end + 31) / 32;
  return it;
}

// out of one value: the gate, then f16.
__device__ __forceinline__ void put(const AttnArgs& a, int64_t tok, int head, int d, float x) {
  if (a.gate) {
    const int64_t gi = tok * a.g_ts + head * a.g_hs + d;
    x = mi::gate_mul(x, a.gate32 ? ((const float*)a.gate)[gi] : (float)((const _Float16*)a.gate)[gi]);
  }
  a.out[(tok * a.pv.G * a.R + head) * D + d] = (_Float16)x;
}

template <int CT>
__global__ void __launch_bounds__(256, CT == 1 ? 2 : 1) paged_attn_kernel(const AttnArgs a) {
  extern __shared__ float lds[];
  // merge buffer [wave][16][kColPitch], maxima and sums [wave][16 CT][2], and
  // for CT > 1 the Q operands [CT][8][64] of 16 bytes
  float* const mbuf = lds;
  float* const mlbuf = lds + kWaves * 16 * kColPitch;
  f16x8* const qbuf = (f16x8*)(mlbuf + kWaves * 16 * CT * 2);

  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m16 = lane & 15, quad = lane >> 4;
  const int64_t bid = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  const int64_t item = bid / a.splits;
  const int split = (int)(bid - item * a.splits);
  if (item >= (int64_t)a.pv.batch * a.pv.G * a.ncb) return;
  const Item it = get_item<CT>(a, item);
  if (it.bad) {  // every token of the sequence, by its first workgroup
    if (it.c0 == 0 && split == 0)
      for (int64_t i = threadIdx.x; i < (int64_t)it.nq * a.R * D; i += 256) {
        const int64_t tok = it.q0 + i / (a.R * D);
        a.out[(tok * a.pv.G + it.h) * a.R * D + i % (a.R * D)] = (_Float16)__builtin_nanf("");
      }
    return;
  }
  const int ncols = it.nq * a.R;
  if (it.c0 >= ncols) return;
  const int t0 = (int)((int64_t)it.ntiles * split / a.splits);
  const int t1 = (int)((int64_t)it.ntiles * (split + 1) / a.splits);
  if (t0 == t1 && a.splits > 1) return;

  // the lane's columns: their rows of Q, and the rows they see
  int lim[CT];
  f16x8 q1[8];  // CT == 1: the Q operands
#pragma unroll
  for (int ct = 0; ct < CT; ct++) {
    const int c = it.c0 + 16 * ct + m16;
    const bool in = c < ncols;
    const int tok = in ? c / a.R : 0, head = it.h * a.R + (in ? c - tok * a.R : 0);
    lim[ct] = in ? it.len - it.nq + tok + 1 : 0;
    const _Float16* qp = a.q + (it.q0 + tok) * a.q_ts + head * a.q_hs + 16 * quad;
    if (CT == 1 || w == ct % kWaves) {
#pragma unroll
      for (int f = 0; f < 8; f++) {  // group f / 2, step f % 2
        f16x8 x = {};
        if (in) x = *(const f16x8*)(qp + 64 * (f >> 1) + 8 * (f & 1));
        x = f16x8{x[0], x[4], x[1], x[5], x[2], x[6], x[3], x[7]};
        if constexpr (CT == 1) q1[f] = x;
        else qbuf[(ct * 8 + f) * 64 + lane] = x;
      }
    }
  }
  if constexpr (CT > 1) __syncthreads();
  const int lim0 = it.len - it.nq + it.c0 / a.R + 1;                                 // first column's
  const int lim1 = it.len - it.nq + min(it.nq - 1, (it.c0 + 16 * CT - 1) / a.R) + 1;  // last column's

  const float c2 = mi::kLog2e / 16.f;  // softmax scale 1 / sqrt(256), in base 2
  f32x4 o[CT][16];
  float m[CT], l[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ct++) {
    m[ct] = kNegBig;
    l[ct] = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) o[ct][i] = f32x4{};
  }
  u32x4 k[4], v[4];
  f16x8 ks[2], vs[4], vo[4];
  auto load_k = [&](const uint8_t* p) {
#pragma unroll
    for (int i = 0; i < 4; i++) k[i] = ((const u32x4*)p)[64 * i + lane];
#pragma unroll
    for (int i = 0; i < 2; i++) ks[i] = ((const f16x8*)(p + mi::kKScale))[16 * i + m16];
  };
  auto load_v = [&](const uint8_t* p) {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = ((const u32x4*)(p + mi::kVCodes))[64 * i + lane];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      vs[i] = ((const f16x8*)(p + mi::kVScale))[2 * (4 * i + quad)];
      vo[i] = ((const f16x8*)(p + mi::kVScale))[2 * (4 * i + quad) + 1];
    }
  };
  bool lost = false;  // a page of the range is not there
  int t = t0 + w;
  const uint8_t* cur = t < t1 ? a.pv.tile(it.s, it.h, t) : nullptr;
  const uint8_t* next = t + kWaves < t1 ? a.pv.tile(it.s, it.h, t + kWaves) : nullptr;
  if (cur) {
    load_k(cur);
    load_v(cur);
  }
  for (; t < t1; t += kWaves) {
    const uint8_t* after = t + 2 * kWaves < t1 ? a.pv.tile(it.s, it.h, t + 2 * kWaves) : nullptr;
    if (!cur) {
      lost = true;
      if (next) {
        load_k(next);
        load_v(next);
      }
      cur = next;
      next = after;
      continue;
    }
    f32x4 sc[CT][2];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) sc[ct][0] = sc[ct][1] = f32x4{};
#pragma unroll
    for (int f = 0; f < 8; f++) {
      const int g = f >> 1, step = f & 1;
      f16x8 ka[2];
#pragma unroll
      for (int sub = 0; sub < 2; sub++)
        ka[sub] = mi::dequant_row(k[2 * sub + (g >> 1)][2 * (g & 1) + step],
                                  f16x2{ks[sub][2 * g], ks[sub][2 * g]},
                                  f16x2{ks[sub][2 * g + 1], ks[sub][2 * g + 1]});
#pragma unroll
      for (int ct = 0; ct < CT; ct++) {
        f16x8 qf;
        if constexpr (CT == 1) qf = q1[f];
        else qf = qbuf[(ct * 8 + f) * 64 + lane];
#pragma unroll
        for (int sub = 0; sub < 2; sub++)
          sc[ct][sub] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[sub], qf, sc[ct][sub], 0, 0, 0);
      }
    }
    if (next) load_k(next);
    const int row0 = 32 * t;
    uint32_t poison[CT] = {};  // groups whose values a column must take for not a number
    if (row0 + 32 > lim0) {    // some column does not see some row (uniform)
      // Keys out of sight weigh nothing whatever they hold: their scores are
      // replaced, and V, whose MFMA would make NaN of 0 * NaN, is cleared where
      // no column sees the row or where it is not finite; columns that do see
      // such a row get their NaN below.
#pragma unroll
      for (int ct = 0; ct < CT; ct++)
#pragma unroll
        for (int sub = 0; sub < 2; sub++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (row0 + 16 * sub + 4 * quad + i >= lim[ct]) sc[ct][sub][i] = -__builtin_inff();
#pragma unroll
      for (int g = 0; g < 4; g++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int row = row0 + 16 * (e & 1) + 4 * quad + (e >> 1);
          const bool odd = !(__builtin_fabsf16(vs[g][e]) < (_Float16)__builtin_inff()) ||
                           !(__builtin_fabsf16(vo[g][e]) < (_Float16)__builtin_inff());
          if (odd || row >= lim1) {
#pragma unroll
            for (int ct = 0; ct < CT; ct++)
              if (odd && row < lim[ct]) poison[ct] |= 1u << g;
            vs[g][e] = (_Float16)0.f;
            vo[g][e] = (_Float16)0.f;
          }
        }
    }
    f16x8 p[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
      float x[8], top = -__builtin_inff();
#pragma unroll
      for (int e = 0; e < 8; e++) {
        x[e] = sc[ct][e & 1][e >> 1] * c2;
        top = fmaxf(top, x[e]);
      }
      top = mi::max_rows(top);
      const float mn = fmaxf(m[ct], top);
      if (__any(mn > m[ct])) {
        const float f = __builtin_amdgcn_exp2f(m[ct] - mn);
        l[ct] *= f;
#pragma unroll
        for (int i = 0; i < 16; i++) o[ct][i] *= f;
        m[ct] = mn;
      }
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float y = __builtin_amdgcn_exp2f(x[e] - mn);
        l[ct] += y;
        p[ct][e] = (_Float16)y;  // the MFMA's operand: off by 2^-11 of itself at most
      }
    }
#pragma unroll
    for (int g = 0; g < 4; g++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const f16x8 va = mi::dequant_col(v[g][j], vs[g], vo[g]);
#pragma unroll
        for (int ct = 0; ct < CT; ct++)
          o[ct][4 * g + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, p[ct], o[ct][4 * g + j], 0, 0, 0);
      }
    if (next) load_v(next);
    if (row0 + 32 > lim0) {
#pragma unroll
      for (int ct = 0; ct < CT; ct++)
        if (__any(poison[ct] != 0)) {
          uint32_t all = poison[ct] | __shfl_xor(poison[ct], 16, 64);
          all |= __shfl_xor(all, 32, 64);
#pragma unroll
          for (int i = 0; i < 16; i++)
            if (all >> (i >> 2) & 1) o[ct][i] += __builtin_nanf("");
        }
    }
    cur = next;
    next = after;
  }

  // the waves' maxima and sums, then their O by 16 columns
#pragma unroll
  for (int ct = 0; ct < CT; ct++) {
    l[ct] = mi::sum_rows(l[ct]);
    if (lost) l[ct] = __builtin_nanf("");
    if (quad == 0) {
      float* const ml = mlbuf + ((w * CT + ct) * 16 + m16) * 2;
      ml[0] = m[ct];
      ml[1] = l[ct];
    }
  }
  __syncthreads();
  const int64_t slot = (item * a.splits + split) * (16 * CT);
#pragma unroll
  for (int ct = 0; ct < CT; ct++) {
    float top = kNegBig;
#pragma unroll
    for (int i = 0; i < kWaves; i++) top = fmaxf(top, mlbuf[((i * CT + ct) * 16 + m16) * 2]);
    const float f = __builtin_amdgcn_exp2f(m[ct] - top);
    float* const mb = mbuf + (w * 16 + m16) * kColPitch + 16 * quad;
#pragma unroll
    for (int g = 0; g < 4; g++)
#pragma unroll
      for (int i = 0; i < 4; i++)  // columns 64 g + 16 quad + 4 i + j of O
        *(f32x4*)(mb + 64 * g + 4 * i) =
            f32x4{o[ct][4 * g][i], o[ct][4 * g + 1][i], o[ct][4 * g + 2][i], o[ct][4 * g + 3][i]} * f;
    __syncthreads();
    const int d = threadIdx.x;
    for (int c = 0; c < 16; c++) {
      const int col = it.c0 + 16 * ct + c;
      if (col >= ncols) break;
      float top_c = kNegBig, sum = 0.f, x = 0.f;
#pragma unroll
      for (int i = 0; i < kWaves; i++) top_c = fmaxf(top_c, mlbuf[((i * CT + ct) * 16 + c) * 2]);
#pragma unroll
      for (int i = 0; i < kWaves; i++) {
        const float* const ml = mlbuf + ((i * CT + ct) * 16 + c) * 2;
        sum += ml[1] * __builtin_amdgcn_exp2f(ml[0] - top_c);
        x += mbuf[(i * 16 + c) * kColPitch + d];
      }
      if (a.splits == 1) {
        const int tok = col / a.R;
        put(a, it.q0 + tok, it.h * a.R + col - tok * a.R, d, sum == 0.f ? 0.f : x / sum);
      } else {
        a.part_o[(slot + 16 * ct + c) * D + d] = x;
        if (d == 0) {
          a.part_ml[(slot + 16 * ct + c) * 2] = top_c;
          a.part_ml[(slot + 16 * ct + c) * 2 + 1] = sum;
        }
      }
    }
    if (ct + 1 < CT) __syncthreads();
  }
}

// Joins the splits of an item: a workgroup per (item, column), a thread per
// output column.
template <int CT>
__global__ void __launch_bounds__(D) paged_merge_kernel(const AttnArgs a) {
  const int64_t bid = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  const int64_t item = bid / (16 * CT);
  const int c = (int)(bid - item * (16 * CT)), d = threadIdx.x;
  if (item >= (int64_t)a.pv.batch * a.pv.G * a.ncb) return;
  const Item it = get_item<CT>(a, item);
  if (it.bad || it.c0 + c >= it.nq * a.R) return;
  float top = kNegBig, sum = 0.f, x = 0.f;
  for (int i = 0; i < a.splits; i++) {
    const int t0 = (int)((int64_t)it.ntiles * i / a.splits);
    const int t1 = (int)((int64_t)it.ntiles * (i + 1) / a.splits);
    if (t0 == t1) continue;
    const int64_t slot = (item * a.splits + i) * (16 * CT) + c;
    const float mi_ = a.part_ml[slot * 2], li = a.part_ml[slot * 2 + 1];
    const float xi = a.part_o[slot * D + d];
    const float mn = fmaxf(top, mi_), f = __builtin_amdgcn_exp2f(top - mn),
                g = __builtin_amdgcn_exp2f(mi_ - mn);
    sum = sum * f + li * g;
    x = x * f + xi * g;
    top = mn;
  }
  const int col = it.c0 + c, tok = col / a.R;
  put(a, it.q0 + tok, it.h * a.R + col - tok * a.R, d, sum == 0.f ? 0.f : x / sum);
}

// Column blocks of 16 a workgroup takes: those of one sequence's tokens, up to 4.
int column_blocks(int32_t max_q, int R) {
  const int64_t cols = (int64_t)max_q * R;
  return cols <= 16 ? 1 : cols <= 32 ? 2 : 4;
}

struct Plan {
  int ct, ncb, splits;
  int64_t items;
  size_t o_bytes, ml_bytes;
};

Plan make_plan(int32_t batch, int32_t max_q, int32_t max_len, int H, int G) {
  Plan p;
  const int R = H / G;
  p.ct = column_blocks(max_q, R);
  p.ncb = (int)(((int64_t)max_q * R + 16 * p.ct - 1) / (16 * p.ct));
  p.items = (int64_t)batch * G * p.ncb;
  const int64_t tiles = std::max<int64_t>(1, ((int64_t)max_len + 31) / 32);
  const int64_t want = (1024 + p.items - 1) / p.items;
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({want, (tiles + 7) / 8, 256}));
  const int64_t cols = p.splits > 1 ? p.items * p.splits * 16 * p.ct : 0;
  p.o_bytes = cols * D * sizeof(float);
  p.ml_bytes = cols * 2 * sizeof(float);
  return p;
}

template <int CT>
mi_status run(const AttnArgs& a, const Plan& p, hipStream_t s) {
  static std::atomic<uint64_t> done{0};
  const int lds = (kWaves * 16 * kColPitch + kWaves * 16 * CT * 2) * (int)sizeof(float) +
                  (CT > 1 ? CT * 8 * 64 * 16 : 0);
  MI_TRY(mi::set_lds_limit((const void*)paged_attn_kernel<CT>, lds, done));
  const int64_t wgs = p.items * p.splits, gx = std::min<int64_t>(wgs, 1 << 22);
  MI_HIP(mi::launch("paged_attn", paged_attn_kernel<CT>,
                    dim3((unsigned)gx, (unsigned)((wgs + gx - 1) / gx)), dim3(256), lds, s, a));
  if (p.splits > 1) {
    const int64_t ms = p.items * 16 * CT, mx = std::min<int64_t>(ms, 1 << 22);
    MI_HIP(mi::launch("paged_merge", paged_merge_kernel<CT>,
                      dim3((unsigned)mx, (unsigned)((ms + mx - 1) / mx)), dim3(D), 0, s, a));
  }
  return MI_OK;
}

mi_status check_heads(int32_t H, int32_t G) {
  if (H <= 0 || G <= 0 || H % G)
    return mi::fail(MI_ERR_INVALID_ARG, "num_q_heads=%d num_kv_heads=%d", H, G);
  if (H / G > mi::kPagedRatioMax)
    return mi::fail(MI_ERR_UNSUPPORTED, "%d query heads per KV head (at most %d)", H / G,
                    mi::kPagedRatioMax);
  return MI_OK;
}

}  // namespace

extern "C" size_t mi_attn_paged_workspace_size(int32_t batch, int32_t n, int32_t max_q,
                                               int32_t max_len, int32_t num_q_heads,
                                               int32_t num_kv_heads) {
  mi::clear_error();
  if (check_heads(num_q_heads, num_kv_heads) != MI_OK || batch <= 0 || n <= 0 || max_q <= 0 ||
      max_len < 0)
    return 0;
  const Plan p = make_plan(batch, std::min(max_q, n), max_len, num_q_heads, num_kv_heads);
  return std::max<size_t>(256, p.o_bytes + p.ml_bytes);
}

extern "C" mi_status mi_attn_paged(
    const void* pages, int64_t num_pages, int32_t page_rows, const int32_t* block_table,
    int32_t table_cols, const int32_t* kv_len, const int32_t* cu_q, int32_t batch, int32_t n,
    int32_t max_q, int32_t max_len, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    const mi_f16* q, int64_t q_token_stride, int64_t q_head_stride, const void* gate,
    int32_t gate_type, int64_t gate_token_stride, int64_t gate_head_stride, mi_f16* out,
    void* workspace, size_t workspace_bytes, mi_stream stream) {
  mi::clear_error();
  AttnArgs a{};
  MI_TRY(mi::paged_view((void*)pages, num_pages, page_rows, block_table, table_cols, kv_len, cu_q,
                        batch, num_kv_heads, head_dim, &a.pv));
  MI_TRY(check_heads(num_q_heads, num_kv_heads));
  if (n <= 0 || max_q <= 0 || max_len < 0 || (!cu_q && (n != batch || max_q != 1)))
    return mi::fail(MI_ERR_INVALID_ARG, "n=%d batch=%d max_q=%d max_len=%d", n, batch, max_q,
                    max_len);
  if (max_len > INT32_MAX - 4096)
    return mi::fail(MI_ERR_OUT_OF_RANGE, "max_len=%d", max_len);
  MI_TRY(mi::check_rows("q", q, MI_F16, q_token_stride, q_head_stride, num_q_heads));
  const int64_t out_ts = (int64_t)num_q_heads * D, out_bytes = (int64_t)n * out_ts * 2;
  MI_TRY(mi::check_rows("out", out, MI_F16, out_ts, D, num_q_heads));
  auto clash = [&](const void* p, int64_t size, int64_t ts, int64_t hs) {
    const bool same = p == out && size == 2 && hs == D && ts == out_ts;
    return !same && mi::overlaps(p, size * mi::rows_extent(n, num_q_heads, ts, hs), out, out_bytes);
  };
  if (clash(q, 2, q_token_stride, q_head_stride))
    return mi::fail(MI_ERR_INVALID_ARG, "out overlaps q (it may only be q itself)");
  if (gate) {
    if (gate_type == MI_BF16) return mi::fail(MI_ERR_INVALID_ARG, "gate must be f16 or f32");
    MI_TRY(mi::check_rows("gate", gate, gate_type, gate_token_stride, gate_head_stride, num_q_heads));
    if (clash(gate, gate_type == MI_F32 ? 4 : 2, gate_token_stride, gate_head_stride))
      return mi::fail(MI_ERR_INVALID_ARG, "out overlaps gate (it may only be gate itself)");
  }
  max_q = std::min(max_q, n);
  const Plan p = make_plan(batch, max_q, max_len, num_q_heads, num_kv_heads);
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < p.o_bytes + p.ml_bytes)
    return mi::fail(MI_ERR_INVALID_ARG, "workspace of %zu bytes, %zu needed", workspace_bytes,
                    p.o_bytes + p.ml_bytes);
  a.q = (const _Float16*)q;
  a.q_ts = q_token_stride;
  a.q_hs = q_head_stride;
  a.gate = gate;
  a.gate32 = gate && gate_type == MI_F32;
  a.g_ts = gate_token_stride;
  a.g_hs = gate_head_stride;
  a.out = (_Float16*)out;
  a.part_o = (float*)workspace;
  a.part_ml = (float*)((char*)workspace + p.o_bytes);
  a.n = n;
  a.R = num_q_heads / num_kv_heads;
  a.max_q = max_q;
  a.max_len = max_len;
  a.splits = p.splits;
  a.ncb = p.ncb;
  const hipStream_t s = (hipStream_t)stream;
  return p.ct == 1 ? run<1>(a, p, s) : p.ct == 2 ? run<2>(a, p, s) : run<4>(a, p, s);
}
