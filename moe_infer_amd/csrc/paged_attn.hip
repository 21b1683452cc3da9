// Attention over the paged 4-bit cache (paged.h): decode steps and drafts to verify, up
// to 32 columns a sequence and KV head.
//
// The columns are its (token, query head of the group) pairs, token-major; a workgroup
// takes all of them, in CT blocks of 16, and a range of 32-row tiles, which its waves
// take in turn.  A wave's tile:
//   S [32 keys x 16 CT] = K Q^T    16x16x32 MFMA, K dequantised in registers
//   running maximum and sum per column (f32), P = 2^(S - max) in f16
//   O^T [256 x 16 CT] += V^T P     V dequantised in registers
// The row order within a tile (paged.h) makes S's accumulator layout the
// operand layout of P, so nothing goes through LDS between the products.  K of
// the next tile is loaded into K's registers while P V runs, V into V's while
// K Q^T runs.
//
// A workgroup's waves join through LDS, workgroups that share an item through
// partials that paged_merge_kernel joins.
//
// Bound: for one column block, the page bytes and what a wave issues for them (64
// sequences of up to 32768 rows, 640 MB: 126 us, 5.1 TB/s; a wave's
// tile is 5300 clocks, two waves to a SIMD, of which 680 wait for memory and 13 % of the
// walk goes to waiting at the join for the SIMD's other wave).  For two, one wave's
// instructions (16 sequences of 4 tokens behind up to 32768 rows, 188 MB: 72 us and 5 of
// merge; 4850 clocks a tile, 990 of them waiting).  For few tiles, the chain from the tables
// to a page's id, its tile and the join: 8 sequences of up to 512 rows 10.4 us, one of
// 32768 rows 13.3 and 4.8 of merge (both as traced).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "paged_attn.h"

namespace {

using mi::AttnArgs;
using mi::kNegBig;

constexpr int D = mi::kHeadDim;
constexpr int kColPitch = D + 4;  // f32 per column of the merge buffer

// Waves of a workgroup, and the tiles that each has under way: two waves to a SIMD where
// the accumulators leave room, else two tiles.
constexpr int waves(int ct) { return ct == 1 ? 8 : 4; }
constexpr int ahead(int ct) { return ct == 1 ? 1 : 2; }
// Tiles below which a workgroup is not split further: one to a wave.
constexpr int kMinTiles = 8;

// A sequence as its work: ntiles tiles of 32 rows for each KV head, its items.
struct Seq {
  int q0, nq, len, ntiles;
  bool bad;  // beyond max_q or max_len
};
template <bool UNIFORM>
__device__ __forceinline__ Seq get_seq(const AttnArgs& a, int s) {
  auto load = [](const int32_t* p) { return UNIFORM ? mi::uniform_load(p) : *p; };
  Seq r;
  r.q0 = a.pv.cu_q ? load(a.pv.cu_q + s) : s;
  r.nq = a.pv.cu_q ? load(a.pv.cu_q + s + 1) - r.q0 : 1;
  r.len = load(a.pv.kv_len + s);
  r.bad = r.len < 0 || r.len > a.max_len || r.nq > a.max_q;
  if (r.nq <= 0 || r.q0 < 0 || (int64_t)r.q0 + r.nq > a.n) r.nq = 0;
  r.ntiles = r.bad || r.nq == 0 ? 0 : (r.len + 31) >> 5;
  return r;
}

// A tile in registers, on its way from memory: the words and scales that a lane's
// operands are made of.  (Scales by way of LDS, a sixteenth of the registers, cost
// a decode step 5 %: their reads wait where these are there.)
struct Tile {
  u32x4 k[4], v[4];
  f16x8 ks[2], vs[4], vo[4];
  // A tile as a buffer of its size, or of none: then the loads below return zeros
  // and move nothing, so the last tile of a wave prefetches without a branch
  // (whose two ways would need the loaded registers copied, and waited for).
  static __device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const uint8_t* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, p ? mi::kTileBytes : 0,
                                             0x00020000);
  }
  // (Past the caches, bit 1: a call reads a sequence's page bytes once.  64 sequences 126.5
  // us, 133.7 without; the same for the small ones.  A page that sequences share is read
  // by each of them, which was not timed.)
  static __device__ __forceinline__ u32x4 load(__amdgpu_buffer_rsrc_t b, int lane_at, int at) {
    return __builtin_amdgcn_raw_buffer_load_b128(b, lane_at + at, 0, 2);
  }
  __device__ __forceinline__ void load_k(__amdgpu_buffer_rsrc_t b, int lane) {
#pragma unroll
    for (int i = 0; i < 4; i++) k[i] = load(b, 16 * lane, 1024 * i);
#pragma unroll
    for (int i = 0; i < 2; i++)
      ks[i] = __builtin_bit_cast(f16x8, load(b, 16 * (lane & 15), mi::kKScale + 256 * i));
  }
  __device__ __forceinline__ void load_v(__amdgpu_buffer_rsrc_t b, int lane) {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = load(b, 16 * lane, mi::kVCodes + 1024 * i);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      vs[i] = __builtin_bit_cast(f16x8, load(b, 32 * (lane >> 4), mi::kVScale + 128 * i));
      vo[i] = __builtin_bit_cast(f16x8, load(b, 32 * (lane >> 4), mi::kVScale + 128 * i + 16));
    }
  }
};

// One wave's state over the tiles of an item.
template <int CT>
struct Wave {
  f32x4 o[CT][16];
  float m[CT], l[CT];
  f16x8 q[CT][8];  // Q^T operands, group f / 2, step f % 2
  int lim[CT];     // rows that the lane's columns see
  uint32_t x16;

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
      m[ct] = kNegBig;
      l[ct] = 0.f;
#pragma unroll
      for (int i = 0; i < 16; i++) o[ct][i] = f32x4{};
    }
  }

  // One tile, rows row0 .. row0 + 31; `next` is loaded in its place on the way.
  // MASKED: some column may not see some row; lim1: rows that some column sees.
  template <bool MASKED>
  __device__ __forceinline__ void tile(Tile& b, __amdgpu_buffer_rsrc_t next, int row0, int lim1, int lane) {
    const int quad = lane >> 4;
    // the words as they are here: without this, their shifts move up to the loads,
    // three registers more for each
#pragma unroll
    for (int i = 0; i < 4; i++) asm volatile("" : "+v"(b.k[i]));
    f32x4 sc[CT][2];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) sc[ct][0] = sc[ct][1] = f32x4{};
#pragma unroll
    for (int f = 0; f < 8; f++) {
      const int g = f >> 1, step = f & 1;
      f16x8 ka[2];
#pragma unroll
      for (int sub = 0; sub < 2; sub++)
        ka[sub] = mi::dequant_row(b.k[2 * sub + (g >> 1)][2 * (g & 1) + step],
                                  f16x2{b.ks[sub][2 * g], b.ks[sub][2 * g]},
                                  f16x2{b.ks[sub][2 * g + 1], b.ks[sub][2 * g + 1]}, x16);
#pragma unroll
      for (int ct = 0; ct < CT; ct++) {
#pragma unroll
        for (int sub = 0; sub < 2; sub++)
          sc[ct][sub] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[sub], q[ct][f], sc[ct][sub], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);  // a few operands at a time
    }
    b.load_k(next, lane);
    __builtin_amdgcn_sched_barrier(0);
    uint32_t in1[4] = {};
    if constexpr (MASKED) {
      // Keys out of sight weigh nothing whatever they hold: their scores are replaced
#pragma unroll
      for (int ct = 0; ct < CT; ct++)
#pragma unroll
        for (int sub = 0; sub < 2; sub++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (row0 + 16 * sub + 4 * quad + i >= lim[ct]) sc[ct][sub][i] = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < 4; i++) in1[i] = seen(row0 + 4 * quad + i, lim1);
    }
    constexpr float c2 = mi::kLog2e / 16.f;  // softmax scale 1 / sqrt(256), in base 2
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
      // The reference point moves only when weights would pass 2^8 (f16 holds
      // them to 2^15, the sums are f32), so after the first tile hardly ever.
      if (__any(top > m[ct] + 8.f)) {
        const float mn = fmaxf(m[ct], top), f = __builtin_amdgcn_exp2f(m[ct] - mn);
        l[ct] *= f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
          // four at a time, in ordinary registers and back: all would not fit
          if constexpr (CT > 1) asm volatile("" : "+a"(o[ct][i]));
          o[ct][i] *= f;
          if constexpr (CT > 1) asm volatile("" : "+a"(o[ct][i]));
        }
        m[ct] = mn;
      }
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float y = __builtin_amdgcn_exp2f(x[e] - m[ct]);
        l[ct] += y;
        p[ct][e] = (_Float16)y;  // the MFMA's operand: off by 2^-11 of itself at most
      }
    }
#pragma unroll
    for (int g = 0; g < 4; g++) {
      f16x8 vs = b.vs[g], vo = b.vo[g];
      bool odd_group = false;
      uint32_t poison = 0;  // columns that see a row whose values of this group may not be finite
      if constexpr (MASKED) {
        // V is cleared where no column sees the row or where it may not be finite (its MFMA
        // would make NaN of 0 * NaN); columns that do see such a row get their NaN
        // here.  What tells is the value of code 15, the furthest of the sixteen from
        // 0 once one of them is past f16.  In pairs of rows (4 quad + i, 16 more), as the
        // scales lie; a half whose exponent is all ones carries into its top bit.
        u32x4 ws = __builtin_bit_cast(u32x4, vs), wo = __builtin_bit_cast(u32x4, vo);
        uint32_t top[4], odd = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          ws[i] &= in1[i];
          wo[i] &= in1[i];
          const uint32_t s = ws[i], o = wo[i];
          top[i] = mi::past_f16(s, o);
          odd |= top[i];
        }
        odd_group = __any(odd != 0);
        if (odd_group) {
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint32_t halves = (top[i] >> 15) * 0xffffu;
#pragma unroll
            for (int ct = 0; ct < CT; ct++)
              if (halves & seen(row0 + 4 * quad + i, lim[ct])) poison |= 1u << ct;
            ws[i] &= ~halves;
            wo[i] &= ~halves;
          }
        }
        vs = __builtin_bit_cast(f16x8, ws);
        vo = __builtin_bit_cast(f16x8, wo);
      }
      asm volatile("" : "+v"(b.v[g]));
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const f16x8 va = mi::dequant_col(b.v[g][j], vs, vo, x16);
#pragma unroll
        for (int ct = 0; ct < CT; ct++)
          o[ct][4 * g + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, p[ct], o[ct][4 * g + j], 0, 0, 0);
      }
      if constexpr (MASKED)
        if (odd_group) {
          uint32_t all = poison | __shfl_xor(poison, 16, 64);
          all |= __shfl_xor(all, 32, 64);
#pragma unroll
          for (int ct = 0; ct < CT; ct++)
#pragma unroll
            for (int j = 0; j < 4; j++)
              o[ct][4 * g + j] += all >> ct & 1 ? __builtin_nanf("") : 0.f;
        }
      __builtin_amdgcn_sched_barrier(0);  // not all sixteen operands at once
    }
    b.load_v(next, lane);
    __builtin_amdgcn_sched_barrier(0);
  }
  // Halves of a pair of rows (r, r + 16) that lie before `end`.
  static __device__ __forceinline__ uint32_t seen(int r, int end) {
    return (r < end ? 0xffffu : 0u) | (r + 16 < end ? 0xffff0000u : 0u);
  }
};

// SINGLE: an item to a workgroup, and nothing to join.  (A kernel of its own: with one for
// both, the long walk was a fifth slower.)
template <int CT, bool SINGLE>
__global__ void __launch_bounds__(64 * waves(CT), CT == 1 ? 2 : 1) paged_attn_kernel(const AttnArgs a) {
  constexpr int NW = waves(CT), NT = 64 * NW;
  extern __shared__ float lds[];
  // maxima [wave][16 CT], sums [wave][16], largest maxima [16]; merge buffer
  // [wave][min(16, columns)][kColPitch]
  float* const mbox = lds;
  float* const lbox = mbox + NW * 16 * CT;
  float* const tbox = lbox + NW * 16;
  float* const mbuf = tbox + 16;
  const int mcols = min(16, a.max_q * a.R);

  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int bid = blockIdx.x;

  // By chunks: every item in chunks of up to kMinTiles tiles, one to a workgroup,
  // where the grid has that many.  Else a flat line of tiles, [sequence][KV
  // head][tile], in even pieces, one to a workgroup.
  int s = 0, before = 0, f = 0, f1 = 0;
  const int G = a.pv.G;
  bool chunks = true;
  auto parts = [](int ntiles) { return (ntiles + kMinTiles - 1) / kMinTiles; };
  if constexpr (SINGLE) {
    f = bid;
    f1 = bid + 1;
  } else {
    mi::find_seq<NT>(
        a.pv.batch,
        [&](int i) { return parts(get_seq<false>(a, i).ntiles); },
        [&](int total) {
          chunks = (uint32_t)total * G <= (uint32_t)a.wgs;
          f = bid;
          f1 = min(bid + 1, total * G);
          return chunks ? (int)((uint32_t)f / (uint32_t)G) : total;
        },
        s, before);
    if (!chunks)
      mi::find_seq<NT>(
          a.pv.batch,
          [&](int i) { return get_seq<false>(a, i).ntiles; },
          [&](int total) {
            const uint32_t all = (uint32_t)total * G, each = all / a.wgs, more = all - each * a.wgs;
            f = (int)(each * bid + min((uint32_t)bid, more));
            f1 = f + (int)each + ((uint32_t)bid < more);
            return (int)((uint32_t)f / (uint32_t)G);
          },
          s, before);
  }
  if (f >= f1) return;
  int slot = 2 * bid;

  Wave<CT> st;
  st.x16 = mi::sixteens();
  while (f < f1) {
    int h, t0, t1;
    Seq sq;
    if constexpr (SINGLE) {
      s = (int)((uint32_t)f / (uint32_t)G);
      h = f - s * G;
      sq = get_seq<true>(a, s);
      t0 = 0;
      t1 = sq.ntiles;
      f = f1;
      if (sq.bad) {
        const int width = a.R * D;
        for (int tok = 0; tok < sq.nq; tok++)
          for (int i = threadIdx.x; i < width; i += NT)
            a.out[((int64_t)(sq.q0 + tok) * G + h) * width + i] = (_Float16)__builtin_nanf("");
        return;
      }
      if (sq.nq == 0) return;
    } else {
      sq = get_seq<true>(a, s);
      const int per = chunks ? parts(sq.ntiles) : sq.ntiles;
      if (f >= G * (before + per)) {
        before += per;
        s++;
        continue;
      }
      const uint32_t local = f - G * before, head = local / (uint32_t)per, at = local - head * per;
      h = (int)head;
      if (chunks) {
        t0 = (int)(at * (uint32_t)sq.ntiles / (uint32_t)per);
        t1 = (int)((at + 1) * (uint32_t)sq.ntiles / (uint32_t)per);
        f = f1;
      } else {
        t0 = (int)at;
        t1 = min(sq.ntiles, t0 + (f1 - f));
        f += t1 - t0;
      }
    }
    const int ncols = sq.nq * a.R, first = sq.len - sq.nq;

    // the lane's columns: their rows of Q, and the rows they see (columns past the
    // last take the first's, which nothing reads)
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
      const int c = 16 * ct + (lane & 15);
      const bool in = c < ncols;
      const int tok = in ? c / a.R : 0, head = h * a.R + (in ? c - tok * a.R : 0);
      st.lim[ct] = in ? first + tok + 1 : 0;
      const _Float16* qp = a.q + (sq.q0 + tok) * a.q_ts + head * a.q_hs + 16 * (lane >> 4);
#pragma unroll
      for (int i = 0; i < 8; i++) st.q[ct][i] = *(const f16x8*)(qp + 64 * (i >> 1) + 8 * (i & 1));
    }
    const int lim0 = first + 1, lim1 = sq.len;  // first and last token's
    // tiles [t0, tm) are seen whole, [tm, t1) not
    const int tm = max(t0, min(t1, lim0 >> 5));

    st.clear();
    // A page that is not there is read as no bytes and the sums of the columns that see it
    // become not a number.
    // kAhead tiles are under way, in turn; pages are looked up another one ahead.
    constexpr int kAhead = ahead(CT);
    int lost = INT32_MAX;  // least row in sight whose page is not there
    auto buffer = [&](int32_t id, int t) {
      const uint8_t* p = t < t1 ? a.pv.at(id, h, t) : nullptr;
      if (t < t1 && !p) lost = min(lost, 32 * t);
      return Tile::buffer(p);
    };
    auto page = [&](int t) { return t < t1 ? a.pv.page(s, t) : -1; };
    int t = t0 + w;
    if (t < t1) {
      Tile tiles[kAhead];
      int32_t id[kAhead + 1];
#pragma unroll
      for (int i = 0; i <= kAhead; i++) id[i] = page(t + i * NW);
#pragma unroll
      for (int i = 0; i < kAhead; i++) {
        const auto b = buffer(id[i], t + i * NW);
        tiles[i].load_k(b, lane);
        tiles[i].load_v(b, lane);
      }
      __builtin_amdgcn_sched_barrier(0);  // behind the tiles' loads: it waits for Q's
#pragma unroll
      for (int ct = 0; ct < CT; ct++)
#pragma unroll
        for (int i = 0; i < 8; i++) st.q[ct][i] = mi::in_order(st.q[ct][i]);
      int32_t ahead_id = id[kAhead];
      auto step = [&](Tile& x, auto masked) {
        const auto next = buffer(ahead_id, t + kAhead * NW);
        ahead_id = page(t + (kAhead + 1) * NW);
        st.template tile<decltype(masked)::value>(x, next, 32 * t, lim1, lane);
        t += NW;
      };
      while (t + (kAhead - 1) * NW < tm) {
#pragma unroll
        for (int i = 0; i < kAhead; i++) step(tiles[i], std::false_type{});
      }
      while (t < t1) {  // what some column may not see
#pragma unroll
        for (int i = 0; i < kAhead; i++)
          if (i == 0 || t < t1) step(tiles[i], std::true_type{});
      }
    }

    // The waves' maxima, then their sums and O relative to the largest, 16 columns
    // at a time; a thread joins four output columns.
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
      st.l[ct] = mi::sum_rows(st.l[ct]);
      if (lost < st.lim[ct]) st.l[ct] = __builtin_nanf("");
      if (lane < 16) mbox[(w * CT + ct) * 16 + lane] = st.m[ct];
    }
    // from here on the lane's addresses are formed anew: hoisted out of the loop
    // over items they would be spilled across the tiles
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int m16 = tid & 15, quad = (tid >> 4) & 3;
    __syncthreads();
    const bool whole = t0 == 0 && t1 == sq.ntiles;
    const int64_t col0 = (int64_t)slot * (16 * CT);
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
      float top = kNegBig;
#pragma unroll
      for (int i = 0; i < NW; i++) top = fmaxf(top, mbox[(i * CT + ct) * 16 + m16]);
      const float scale = __builtin_amdgcn_exp2f(st.m[ct] - top);
      if (quad == 0) {
        lbox[w * 16 + m16] = st.l[ct] * scale;
        tbox[m16] = top;  // the same from every wave
      }
      float* const mb = mbuf + (w * mcols + m16) * kColPitch + 16 * quad;
      if (m16 < mcols) {
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
          for (int i = 0; i < 4; i++)  // columns 64 g + 16 quad + 4 i + j of O
            *(f32x4*)(mb + 64 * g + 4 * i) = f32x4{st.o[ct][4 * g][i], st.o[ct][4 * g + 1][i],
                                                   st.o[ct][4 * g + 2][i], st.o[ct][4 * g + 3][i]} *
                                             scale;
      }
      __syncthreads();
      const int d = 4 * (tid & 63);
      for (int c = w; c < mcols; c += NW) {
        const int col = 16 * ct + c;
        if (col >= ncols) break;
        float sum = 0.f;
        f32x4 x = {};
#pragma unroll
        for (int i = 0; i < NW; i++) {
          sum += lbox[i * 16 + c];
          x += *(const f32x4*)(mbuf + (i * mcols + c) * kColPitch + d);
        }
        if (whole) {
          const int tok = col / a.R;
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          mi::put4(a, sq.q0 + tok, h * a.R + col - tok * a.R, d, x, inv);
        } else {
          *(f32x4*)(a.part_o + (col0 + 16 * ct + c) * D + d) = x;
          if (d == 0) *(float2*)(a.part_ml + (col0 + 16 * ct + c) * 2) = float2{tbox[c], sum};
        }
      }
      __syncthreads();
    }
    if (!SINGLE && threadIdx.x == 0) {  // where the merge finds the item's pieces
      int2* const sg = a.seg + (int64_t)s * G + h;
      if (whole) {
        sg->x = -1;
      } else {
        if (t0 == 0) sg->x = slot;
        if (t1 == sq.ntiles) sg->y = bid;
      }
    }
    slot = 2 * bid + 1;  // only the first and the last item of a workgroup are not whole
  }
}

// Joins the pieces of an item: a workgroup per (item, column, part of the 256
// output columns); its first piece is in slot seg.x, the others in slot 2 x of the
// workgroups x behind.  Items without rows become zero, those beyond max_q or
// max_len NaN.
template <int CT>
__global__ void __launch_bounds__(256) paged_merge_kernel(const AttnArgs a) {
  __shared__ f32x4 acc[256];
  __shared__ float ml[256][2];
  const uint32_t parts = a.dsplit, d4 = 64 / parts, groups = 256 / d4;
  const uint32_t bid = blockIdx.y * gridDim.x + blockIdx.x;  // below 2^31 (make_plan)
  const uint32_t ic = bid / parts, part = bid - ic * parts;
  const uint32_t item = ic / (16 * CT);
  const int col = ic % (16 * CT);
  if (item >= (uint32_t)a.pv.batch * a.pv.G) return;
  const int s = item / a.pv.G, h = item - s * a.pv.G;
  const Seq sq = get_seq<true>(a, s);
  const uint32_t t = threadIdx.x, lane4 = t % d4, grp = t / d4, d = 4 * (part * d4 + lane4);
  if (sq.bad || sq.ntiles == 0) {  // every token of the sequence, by its items' first workgroup
    if (col || part) return;
    const _Float16 x = sq.bad ? (_Float16)__builtin_nanf("") : (_Float16)0.f;
    const int width = a.R * D;
    for (int tok = 0; tok < sq.nq; tok++)
      for (int i = t; i < width; i += 256)
        a.out[((int64_t)(sq.q0 + tok) * a.pv.G + h) * width + i] = x;
    return;
  }
  if (col >= sq.nq * a.R) return;
  const int2 sg = a.seg[item];
  if (sg.x < 0) return;
  const int first = sg.x >> 1, count = sg.y - first + 1;
  auto slot = [&](int i) { return (i ? 2 * (first + i) : sg.x) * (16 * CT) + col; };
  float top = kNegBig, sum = 0.f;
  f32x4 x = {};
  for (int i0 = grp; i0 < count; i0 += 4 * (int)groups) {
    float mi_[4], li[4];
    f32x4 xi[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int i = i0 + u * (int)groups;
      const bool in = i < count;
      const int sl = slot(in ? i : i0);
      mi_[u] = in ? a.part_ml[sl * 2] : kNegBig;
      li[u] = in ? a.part_ml[sl * 2 + 1] : 0.f;
      xi[u] = *(const f32x4*)(a.part_o + (int64_t)sl * D + d);
    }
    const float mn = fmaxf(top, fmaxf(fmaxf(mi_[0], mi_[1]), fmaxf(mi_[2], mi_[3])));
    const float f = __builtin_amdgcn_exp2f(top - mn);
    sum *= f;
    x *= f;
    top = mn;
#pragma unroll
    for (int u = 0; u < 4; u++) {
      if (i0 + u * (int)groups >= count) continue;
      const float g = __builtin_amdgcn_exp2f(mi_[u] - mn);
      sum += li[u] * g;
      x += xi[u] * g;
    }
  }
  acc[t] = x;
  if (lane4 == 0) {
    ml[grp][0] = top;
    ml[grp][1] = sum;
  }
  __syncthreads();
  if (t >= d4) return;  // a thread per four output columns of the part
  const int used = min((int)groups, count);
  float m = kNegBig, total = 0.f;
  f32x4 y = {};
  for (int g = 0; g < used; g++) m = fmaxf(m, ml[g][0]);
  for (int g = 0; g < used; g++) {
    const float f = __builtin_amdgcn_exp2f(ml[g][0] - m);
    total += ml[g][1] * f;
    y += acc[g * d4 + t] * f;
  }
  const int tok = col / a.R;
  mi::put4(a, sq.q0 + tok, h * a.R + col - tok * a.R, d, y, total == 0.f ? 0.f : 1.f / total);
}

// Columns of a sequence and KV head that the decode kernels take at most: a workgroup
// takes them all.
constexpr int kManyColumns = 32;

// Column blocks of 16 a workgroup takes.
static_assert(kManyColumns == 2 * 16, "a workgroup of two blocks takes every column");
int column_blocks(int32_t max_q, int R) { return (int64_t)max_q * R <= 16 ? 1 : 2; }

// Whether the prompts' form serves a call: 16 sequences of 4 tokens, 8 heads a group,
// behind 500 / 8192 / 20000 rows 20 / 56 / 81 us here and 34 / 72 / 136 there.
bool many_columns(int32_t max_q, int R) { return (int64_t)max_q * R > kManyColumns; }

struct Plan {
  int ct, wgs, dsplit;
  bool single;
  int64_t items, tiles;
  size_t o_bytes, ml_bytes, seg_bytes;
  size_t bytes() const { return o_bytes + ml_bytes + seg_bytes; }
};

Plan make_plan(int32_t batch, int32_t max_q, int32_t max_len, int H, int G) {
  Plan p;
  const int R = H / G;
  p.ct = column_blocks(max_q, R);
  p.items = (int64_t)batch * G;
  p.tiles = p.items * (((int64_t)max_len + 31) / 32);
  const int64_t per_item = (((int64_t)max_len + 31) / 32 + kMinTiles - 1) / kMinTiles;
  p.wgs = (int)std::max<int64_t>(1, std::min<int64_t>(256, p.items * per_item));
  // An item to a workgroup, and no merge, where that is four tiles to a wave, or more where
  // items fill the card (one KV head's group of 8, two heads a sequence): 8 sequences of
  // 512 rows 10.3 us against 16.5, of 1024 14.0 against 16.4, of 2048 22 against 16.5; 64 of
  // 2048 23 against 26; 128 of 1 to 4000 42 against 68, 256 83 against 103.
  p.single = max_len <= (p.items >= 256 ? 4096 : p.items >= 64 ? 2048 : 1024);
  p.dsplit = p.items * std::min(16 * p.ct, max_q * R) <= 256 ? 4 : 1;
  if (p.items * 16 * p.ct * p.dsplit > INT32_MAX) p.tiles = INT32_MAX;  // refused
  const int64_t cols = (int64_t)2 * p.wgs * 16 * p.ct;
  p.o_bytes = cols * D * sizeof(float);
  p.ml_bytes = cols * 2 * sizeof(float);
  p.seg_bytes = (p.items * sizeof(int2) + 15) & ~(size_t)15;
  return p;
}

// A prompt's workspace also serves the smaller calls that the decode kernels take.
size_t plan_bytes(const Plan& p, int32_t batch, int32_t max_q, int32_t max_len, int H, int G) {
  if (!many_columns(max_q, H / G)) return p.bytes();
  const Plan few = make_plan(batch, std::max(1, kManyColumns / (H / G)), max_len, H, G);
  return std::max(mi::paged_prefill_workspace(), few.bytes());
}

template <int CT, bool SINGLE>
mi_status run(AttnArgs& a, const Plan& p, hipStream_t s) {
  static std::atomic<uint64_t> done{0};
  constexpr int NW = waves(CT);
  const int fixed = (NW * 16 * (CT + 1) + 16) * (int)sizeof(float);
  const int per_col = NW * kColPitch * (int)sizeof(float);
  MI_TRY(mi::set_lds_limit((const void*)paged_attn_kernel<CT, SINGLE>, fixed + 16 * per_col, done));
  MI_HIP(mi::launch("paged_attn", paged_attn_kernel<CT, SINGLE>, dim3((unsigned)(SINGLE ? p.items : p.wgs)),
                    dim3(64 * NW), fixed + std::min(16, a.max_q * a.R) * per_col, s, a));
  if (SINGLE) return MI_OK;
  const int64_t ms = p.items * 16 * CT * p.dsplit, mx = std::min<int64_t>(ms, 1 << 22);
  MI_HIP(mi::launch("paged_merge", paged_merge_kernel<CT>,
                    dim3((unsigned)mx, (unsigned)((ms + mx - 1) / mx)), dim3(256), 0, s, a));
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
  max_q = std::min(max_q, n);
  const Plan p = make_plan(batch, max_q, max_len, num_q_heads, num_kv_heads);
  if (p.tiles >= INT32_MAX && !many_columns(max_q, num_q_heads / num_kv_heads)) return 0;
  return plan_bytes(p, batch, max_q, max_len, num_q_heads, num_kv_heads);
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
  const bool many = many_columns(max_q, num_q_heads / num_kv_heads);
  if (p.tiles >= INT32_MAX && !many)  // the decode kernels count them in 32 bits
    return mi::fail(MI_ERR_UNSUPPORTED, "%d sequences of %d tokens and %d rows in one call", batch, max_q,
                    max_len);
  const size_t need = plan_bytes(p, batch, max_q, max_len, num_q_heads, num_kv_heads);
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)
    return mi::fail(MI_ERR_INVALID_ARG, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
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
  a.seg = (int2*)((char*)workspace + p.o_bytes + p.ml_bytes);
  a.wgs = p.wgs;
  a.dsplit = p.dsplit;
  const hipStream_t s = (hipStream_t)stream;
  if (many) return mi::paged_prefill(a, workspace, s);
  if (p.single) return p.ct == 1 ? run<1, true>(a, p, s) : run<2, true>(a, p, s);
  return p.ct == 1 ? run<1, false>(a, p, s) : run<2, false>(a, p, s);
}
