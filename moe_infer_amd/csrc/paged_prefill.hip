// Attention over the paged 4-bit cache for many tokens: prompts, and chunks
// behind cached rows.
//
// A workgroup takes 128 rows, the (token, query head of the group) pairs of
// 128 / R consecutive tokens of one sequence and KV head, and walks the keys
// that they see in tiles of 64.  The four waves dequantise a tile once into
// LDS as f16, in MFMA operand order; wave (qb, kp) multiplies rows 64 qb .. + 63
// with keys 32 kp .. + 31 of it (v_mfma_f32_32x32x16_f16, S^T = K Q^T, O^T += V^T
// P^T), so that every operand read from LDS feeds two products, and the two
// key halves join at the end.
//
// Bound: the matrix units.  A tile is 64 MFMAs of 32 clocks to a wave, one wave
// to a SIMD; what else it needs is issued between them: the next tile's
// dequantisation (16 words a thread) between those of K Q^T, the softmax of tile t
// between those of P V of tile t - 1.  O^T of 64 rows takes the 256 accumulation
// registers, so the scores have to come out in ordinary ones: their MFMAs are
// asm, which the compiler would otherwise give the accumulation form as well.
//
// The keys of a block of rows are cut into pieces where one walk would outlast an
// even share of the call (a few tokens behind a long context): pieces leave
// partials, paged_prefill_merge_kernel joins them.
#include <algorithm>
#include <cmath>

#include "paged_attn.h"

namespace {

using mi::AttnArgs;
using mi::kNegBig;

constexpr int D = mi::kHeadDim;
constexpr int kRows = 128;   // rows of a workgroup
constexpr int kKeys = 64;    // keys of a tile
constexpr int kHalf = 16384;  // bytes of 32 keys, K or V, as f16
constexpr int kShare = 256;  // even shares of a call: one per CU
constexpr int kMinPiece = 8;  // tiles below which keys are not cut further
constexpr int kSplitBlocks = 256, kSlots = 512;  // most blocks that are cut, and pieces of them

struct PrefillExtra {
  float* part_o;    // [kSlots][kRows][D]
  float* part_ml;   // [kSlots][kRows][2]
  int4* blocks;     // [kSplitBlocks]: sequence, KV head, block, index of its second piece
  int2* count;      // blocks that are cut, tiles of a piece
};

// A sequence as blocks of tb tokens.
struct Blocks {
  int q0, nq, len, nb, tb;
  bool bad;
  __device__ __forceinline__ int first() const { return len - nq; }
  // rows that block b's last token sees, and tiles of them
  __device__ __forceinline__ int end(int b) const { return first() + min(nq, tb * (b + 1)); }
  __device__ __forceinline__ int tiles(int b) const { return max(end(b) + kKeys - 1, 0) / kKeys; }
  // First block with more than x tiles; nb where none has.
  __device__ __forceinline__ int past(int64_t x) const {
    if (nb == 0 || len <= x * kKeys) return nb;
    const int64_t y = x * kKeys - first();
    return y <= 0 ? 0 : (int)((uint32_t)y / (uint32_t)tb);
  }
};
__device__ __forceinline__ Blocks get_blocks(const AttnArgs& a, int s) {
  Blocks r;
  a.pv.tokens(s, r.q0, r.nq);
  r.len = a.pv.kv_len[s];
  r.bad = r.len < 0 || r.len > a.max_len || r.nq > a.max_q;
  if (r.nq <= 0 || r.q0 < 0 || (int64_t)r.q0 + r.nq > a.n) r.nq = 0;
  r.tb = kRows / a.R;
  r.nb = r.bad ? 0 : (r.nq + r.tb - 1) / r.tb;
  return r;
}
// Pieces of a sequence's blocks (one KV head), each of at most `piece` tiles:
// piece k of block b exists where b >= past(k piece), piece 0 always.  Those of
// k >= 1 alone with `more`.
__device__ __forceinline__ int pieces(const Blocks& q, int piece, bool more) {
  int n = more ? 0 : q.nb;
  if (q.nb == 0) return 0;
  const int most = q.tiles(q.nb - 1);
  for (int64_t x = piece; x < most; x += piece) n += q.nb - q.past(x);
  return n;
}

template <int NT>
__device__ __forceinline__ double block_sum(double x, double* lds) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < NT / 64; i++) sum += lds[i];
  return sum;
}

// Tiles of a piece: an even share of the call's tiles (at least, so that no more
// than kShare pieces come on top of one per block), or kMinPiece.
__device__ __forceinline__ int piece_tiles(const AttnArgs& a, double* lds) {
  double mine = 0.0;
  for (int s = threadIdx.x; s < a.pv.batch; s += 256) {
    const Blocks q = get_blocks(a, s);
    if (q.nb) mine += (double)q.nb * (0.5 * (q.tiles(0) + q.tiles(q.nb - 1)) + 1.0);
  }
  const double all = block_sum<256>(mine, lds) * a.pv.G;
  return __builtin_amdgcn_readfirstlane(max(kMinPiece, (int)ceil(all / kShare)));
}

__device__ __forceinline__ void mfma_s(f32x16& c, f16x8 a, f16x8 b) {
  asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
}
__device__ __forceinline__ void mfma_s0(f32x16& c, f16x8 a, f16x8 b) {
  asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "v"(b));
}

__global__ void __launch_bounds__(256, 1) paged_prefill_kernel(const AttnArgs a, const PrefillExtra x) {
  extern __shared__ char lds[];  // K, V [2][2 halves], their scales; then the join of the key halves
  __shared__ double sums[4];
  __shared__ int odd_row[4];  // least masked row whose V group is not finite
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, hl = lane >> 5;
  const int qb = w & 1, kp = w >> 1;
  const int bid = blockIdx.y * gridDim.x + blockIdx.x;
  const int G = a.pv.G;

  // ---- which block of which sequence, and which of its tiles
  const int piece = piece_tiles(a, sums);
  int s, before, local = -1;
  mi::find_seq<256>(
      a.pv.batch, [&](int i) { return pieces(get_blocks(a, i), piece, false); },
      [&](int total) {
        local = (uint32_t)bid < (uint32_t)total * (uint32_t)G ? bid : -1;
        return local < 0 ? total : (int)((uint32_t)bid / (uint32_t)G);
      },
      s, before);
  if (bid == 0) {  // for the merge
    double cut = 0.0;
    for (int i = tid; i < a.pv.batch; i += 256) {
      const Blocks q = get_blocks(a, i);
      cut += q.nb - q.past(piece);
    }
    cut = block_sum<256>(cut, sums);
    if (tid == 0) *x.count = int2{(int)cut * G, piece};
  }
  if (local < 0) return;
  Blocks q = get_blocks(a, s);
  q.q0 = __builtin_amdgcn_readfirstlane(q.q0);
  q.nq = __builtin_amdgcn_readfirstlane(q.nq);
  q.len = __builtin_amdgcn_readfirstlane(q.len);
  q.nb = __builtin_amdgcn_readfirstlane(q.nb);
  const int per = __builtin_amdgcn_readfirstlane(pieces(q, piece, false));
  local -= G * before;
  const int h = (int)((uint32_t)local / (uint32_t)per);
  local -= h * per;
  int k = 0, b0 = 0;  // piece k of the blocks from b0 on, the last (longest) first
  while (local >= q.nb - b0) {
    local -= q.nb - b0;
    k++;
    b0 = __builtin_amdgcn_readfirstlane(q.past((int64_t)k * piece));
  }
  const int b = q.nb - 1 - local;
  const int tok0 = b * q.tb, ntok = min(q.tb, q.nq - tok0), nrows = ntok * a.R;
  const int nt_all = q.tiles(b), cuts = max(1, (nt_all + piece - 1) / piece);
  const int first = q.first() + tok0;  // row of the block's first token
  const int end = first + ntok;
  const int ta = (int)((int64_t)nt_all * k / cuts), tz = (int)((int64_t)nt_all * (k + 1) / cuts);

  if (tid < 4) odd_row[tid] = INT32_MAX;

  // ---- a tile's words: those of the 32-row tiles 2 t and 2 t + 1.  A thread takes a
  // 16-byte piece of K and of V of each, and one word of the scales of one of them,
  // which go through LDS a tile earlier (in registers every thread would hold 20
  // words of them).
  u32x4 rk[2], rv[2];
  uint32_t sk, sv;
  bool lost = false;
  // Where tiles t + 1, t + 2 and t + 3 lie (at[i][u]: tile 2 (t + i) + u), looked up a tile
  // before their loads; the page's id is loaded two tiles before that, by a vector load
  // (a scalar one would hold up every wait for LDS until it has come).  What has no
  // place (behind the last row; a page that the pool does not have, which is lost)
  // reads page 0, and counts for nothing.
  const uint8_t* at[4][2];
  const int pt = a.pv.page_shift - 5;
  const int tend = (end + 31) >> 5;  // 32-row tiles
  const int tlim = (int)min((int64_t)tend, (int64_t)a.pv.cols << pt);
  const uint32_t npages = (uint32_t)a.pv.num_pages;
  const uint64_t page_bytes = ((uint64_t)a.pv.G << pt) * mi::kTileBytes;
  const uint8_t* const pages = a.pv.pages + ((uint64_t)h << pt) * mi::kTileBytes;
  const int32_t* const table = a.pv.table + (int64_t)s * a.pv.cols;
  auto ids = [&](int t) {  // lane u's: page of tile 2 t + u, or any where there is none
    return table[min((2 * t + (lane & 1)) >> pt, a.pv.cols - 1)];
  };
  auto place = [&](const uint8_t* (&p)[2], int32_t idv, int t) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const uint32_t id = __builtin_amdgcn_readlane(idv, u);
      const int ok = (2 * t + u < tlim) & (id < npages);
      lost = lost | ((2 * t + u < tend) & (ok ^ 1));
      const uint64_t off = id * page_bytes + (uint32_t)(((2 * t + u) & ((1 << pt) - 1)) * mi::kTileBytes);
      p[u] = pages + (ok ? off : 0);
    }
  };
  const int m16 = lane & 15, quad = lane >> 4;
  const int su = w >> 1, sat = 4 * (tid & 127);  // the thread's word of scales: tile, offset
  auto buffer = [&](const uint8_t* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, mi::kTileBytes, 0x00020000);
  };
  auto load_k = [&](u32x4 (&r)[2], int i) {
#pragma unroll
    for (int u = 0; u < 2; u++) r[u] = __builtin_amdgcn_raw_buffer_load_b128(buffer(at[i][u]), 16 * tid, 0, 0);
  };
  auto load_v = [&](u32x4 (&r)[2], int i) {
#pragma unroll
    for (int u = 0; u < 2; u++)
      r[u] = __builtin_amdgcn_raw_buffer_load_b128(buffer(at[i][u]), 16 * tid, mi::kVCodes, 0);
  };
  auto load_sk = [&](int i) {
    return __builtin_amdgcn_raw_buffer_load_b32(buffer(su ? at[i][1] : at[i][0]), sat, mi::kKScale, 0);
  };
  auto load_sv = [&](int i) {
    return __builtin_amdgcn_raw_buffer_load_b32(buffer(su ? at[i][1] : at[i][0]), sat, mi::kVScale, 0);
  };
  const uint32_t x16 = mi::sixteens();
  char* const kbuf = lds;
  char* const vbuf = lds + 4 * kHalf;
  char* const ksc = lds + 8 * kHalf;  // [2][2 tiles][512]
  char* const vsc = ksc + 2048;
  auto put_sk = [&](int t, uint32_t y) { *(uint32_t*)(ksc + (t & 1) * 1024 + 4 * tid) = y; };
  // V's word: scale or offset of rows 4 quad + i and 16 more, of group g.  Rows that no
  // token of the block sees read as zero, and so does what is not finite in rows that
  // some token does not see (the MFMA would make NaN of 0 * NaN for it); the
  // tokens that do see such a row get their NaN at the end.
  auto put_sv = [&](int t, uint32_t y) {
    if (kKeys * (t + 1) > first + 1) {  // uniform: not seen whole
      int x = tid;
      asm volatile("" : "+v"(x));  // nothing of this is kept in registers over the tiles
      const int i = x & 3, sq = (x >> 3) & 3, g = (x >> 5) & 3;
      const int row = kKeys * t + 32 * su + 4 * sq + i;
      y &= (row < end ? 0xffffu : 0u) | (row + 16 < end ? 0xffff0000u : 0u);
      const uint32_t odd = ((y & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
      if (odd) {
        atomicMin(&odd_row[g], odd & 0x8000u ? row : row + 16);
        y &= ~((odd >> 15) * 0xffffu);
      }
    }
    *(uint32_t*)(vsc + (t & 1) * 1024 + 4 * tid) = y;
  };
  // The wave's pieces of K: rows 16 (w / 2) + m16, groups 2 (w % 2) and the next.  Word j:
  // operand 4 (2 (w % 2) + j / 2) + quad, lane half j % 2, and the slot whose score lands
  // where P wants the key (slot 16 s + 8 (e / 4) + 4 l + e % 4 of lane half l is key
  // 16 (e % 2) + 4 (2 s + l) + e / 2)
  // Slot x of an operand is stored as x ^ (x >> 3 & 1): the eight lanes that store together
  // would meet in half of the banks.
  auto slot_of = [](int x) { return x ^ ((x >> 3) & 1); };
  const int kslot = 16 * (m16 >> 3) + 8 * ((m16 >> 1) & 1) + 4 * ((m16 >> 2) & 1) + 2 * (m16 & 1) + (w >> 1);
  const int kdst = ((8 * (w & 1) + quad) * 2 * 32 + slot_of(kslot)) * 16;
  const int ksrc = 16 * (16 * (w >> 1) + m16) + 8 * (w & 1);
  // V word j: product quad / 2, block 2 w + j / 2, lane half quad % 2, slot 16 (j % 2) + n
  const int vdst = (((quad >> 1) * 8 + 2 * w) * 2 * 32 + (quad & 1) * 32 + slot_of(m16)) * 16;
  const int opnd = 16 * slot_of(lane);
  const int vsrc = 32 * (4 * w + quad);
  f16x2 kso[2];
  auto get_ks = [&](int t, int u) {  // a piece's scales, ahead of its words
#pragma unroll
    for (int i = 0; i < 2; i++)
      kso[i] = *(const f16x2*)(ksc + (t & 1) * 1024 + 512 * u + ksrc + 4 * i);
  };
  // A word in two halves of six instructions, for the two products of a step.
  f16x2 half[2];
  auto half_k = [&](uint32_t y, int j) {
    const f16x2 so = kso[j >> 1], sc = f16x2{so[0], so[0]}, of = f16x2{so[1], so[1]};
    half[0] = mi::pk_fma(mi::codes16<0>(y, x16), sc, of);
    half[1] = mi::pk_fma(mi::codes16<1>(y, x16), sc, of);
  };
  auto put_k = [&](uint32_t y, int t, int u, int j) {
    const f16x2 so = kso[j >> 1], sc = f16x2{so[0], so[0]}, of = f16x2{so[1], so[1]};
    const f16x2 c = mi::pk_fma(mi::codes16<2>(y, x16), sc, of);
    const f16x2 d = mi::pk_fma(mi::codes16<3>(y, x16), sc, of);
    *(f16x8*)(kbuf + ((t & 1) * 2 + u) * kHalf + kdst + (((j >> 1) * 4 * 2 + (j & 1)) * 32) * 16) =
        f16x8{half[0][0], half[0][1], half[1][0], half[1][1], c[0], c[1], d[0], d[1]};
  };
  f16x8 vs, vo;
  auto get_vs = [&](int t, int u) {
    vs = *(const f16x8*)(vsc + (t & 1) * 1024 + 512 * u + vsrc);
    vo = *(const f16x8*)(vsc + (t & 1) * 1024 + 512 * u + vsrc + 16);
  };
  auto half_v = [&](uint32_t y) {
    half[0] = mi::pk_fma(mi::codes16<0>(y, x16), f16x2{vs[0], vs[1]}, f16x2{vo[0], vo[1]});
    half[1] = mi::pk_fma(mi::codes16<1>(y, x16), f16x2{vs[2], vs[3]}, f16x2{vo[2], vo[3]});
  };
  auto put_v = [&](uint32_t y, int t, int u, int j) {
    const f16x2 c = mi::pk_fma(mi::codes16<2>(y, x16), f16x2{vs[4], vs[5]}, f16x2{vo[4], vo[5]});
    const f16x2 d = mi::pk_fma(mi::codes16<3>(y, x16), f16x2{vs[6], vs[7]}, f16x2{vo[6], vo[7]});
    *(f16x8*)(vbuf + ((t & 1) * 2 + u) * kHalf + vdst + ((j >> 1) * 64 + 16 * (j & 1)) * 16) =
        f16x8{half[0][0], half[0][1], half[1][0], half[1][1], c[0], c[1], d[0], d[1]};
  };

  constexpr float c2 = mi::kLog2e / 16.f;  // softmax scale 1 / sqrt(256), in base 2
  f32x16 acc[2][8];
  float m[2] = {kNegBig, kNegBig}, l[2] = {0.f, 0.f};
  // ---- the first tiles, and Q^T operands of the wave's 64 rows (those first that it
  // finishes), by way of LDS: read row by row, a quarter of the rows a wave
  f16x8 qf[2][16];
  int lim[2];  // rows of the cache that they see
  int32_t id[4], idn = 0;  // pages of tile t + 4
  u32x4 k0[2];
  uint32_t sk0 = 0, sk1 = 0, sv0 = 0;
  if (ta < tz) {
#pragma unroll
    for (int i = 0; i < 4; i++) id[i] = ids(ta + i);
    idn = ids(ta + 4);
  }
  const float rinv = 1.f / (float)a.R;
  auto token = [&](int r) { return (int)(((float)r + 0.5f) * rinv); };  // r / R: r < 128
  {
    f16x8 y[16];
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const int r = 32 * w + 2 * i + hl, rr = r < nrows ? r : 0, tok = token(rr);
      y[i] = *(const f16x8*)(a.q + (int64_t)(q.q0 + tok0 + tok) * a.q_ts +
                             (h * a.R + rr - tok * a.R) * a.q_hs + 8 * col);
    }
    if (ta < tz) {
#pragma unroll
      for (int i = 0; i < 4; i++) place(at[i], id[i], ta + i);
      sk0 = load_sk(0);
      sk1 = load_sk(1);
      sv0 = load_sv(0);
      load_k(k0, 0);
      load_v(rv, 0);
      load_k(rk, 1);
      sk = load_sk(2);
      sv = load_sv(1);
    }
    // the first walk's products with no weights read a buffer of zeros
    for (int i = tid; i < 2 * kHalf / 16; i += 256)
      ((u32x4*)(vbuf + ((ta - 1) & 1) * 2 * kHalf))[i] = u32x4{};
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const int r = 32 * w + 2 * i + hl;
      *(f16x8*)(kbuf + 512 * r + 16 * (col ^ (r & 7))) = mi::in_order(y[i]);
    }
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < 2; c++) {
    const int r = 64 * qb + 32 * (c ^ kp) + col;
    lim[c] = r < nrows ? first + token(r) + 1 : 0;
#pragma unroll
    for (int ks = 0; ks < 16; ks++)
      qf[c][ks] = *(const f16x8*)(kbuf + 512 * r + 16 * ((2 * ks + hl) ^ (r & 7)));
  }
#pragma unroll
  for (int c = 0; c < 2; c++)
#pragma unroll
    for (int i = 0; i < 8; i++) acc[c][i] = f32x16{};
  f16x8 p[2][2];
#pragma unroll
  for (int c = 0; c < 2; c++)
#pragma unroll
    for (int i = 0; i < 2; i++) p[c][i] = f16x8{};

  put_sk(ta, sk0);
  put_sk(ta + 1, sk1);
  __syncthreads();
  put_sv(ta, sv0);
#pragma unroll
  for (int u = 0; u < 2; u++) {
    get_ks(ta, u);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      half_k(k0[u][j], j);
      put_k(k0[u][j], ta, u, j);
    }
  }
  __syncthreads();
  // A ring of four operands: a tile's 16 of K, then the last tile's 16 of V.
  constexpr int kRing = 4;
  f16x8 ring[kRing];
  auto get = [&](const char* buf, int t, int i) {
    ring[i % kRing] = *(const f16x8*)(buf + ((t & 1) * 2 + kp) * kHalf + opnd + 1024 * i);
  };
  for (int t = ta; t < tz; t++) {
    // K Q^T of tile t; between its products the next tile's K and this tile's V go
    // to LDS (what lies behind the last tile is read as zeros)
    f32x16 sc[2];
    get_ks(t + 1, 0);
#pragma unroll
    for (int i = 0; i < kRing; i++) get(kbuf, t, i);
    {
#pragma unroll
      for (int ks = 0; ks < 16; ks++) {
        if (ks == 0) mfma_s0(sc[0], ring[0], qf[0][0]);
        else mfma_s(sc[0], ring[ks % kRing], qf[0][ks]);
        __builtin_amdgcn_sched_barrier(0);
        const uint32_t y = ks < 8 ? rk[ks >> 2][ks & 3] : rv[(ks - 8) >> 2][ks & 3];
        if (ks < 8) half_k(y, ks & 3);
        else half_v(y);
        __builtin_amdgcn_sched_barrier(0);
        if (ks == 0) mfma_s0(sc[1], ring[0], qf[1][0]);
        else mfma_s(sc[1], ring[ks % kRing], qf[1][ks]);
        if (ks + kRing < 16) get(kbuf, t, ks + kRing);
        else get(vbuf, t - 1, ks + kRing - 16);
        if (ks < 8) put_k(y, t + 1, ks >> 2, ks & 3);
        else put_v(y, t, (ks - 8) >> 2, ks & 3);
        if (ks == 3) get_ks(t + 1, 1);
        if (ks == 7) {
          get_vs(t, 0);
          load_k(rk, 2);
        }
        if (ks == 11) get_vs(t, 1);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    // V^T P of tile t - 1: two products an iteration, i, between which go the loads of the
    // tiles ahead, then tile t's weights
    auto product = [&](int i, int c) {  // keys 16 (i / 8) .. of the half, block i % 8
      acc[c][i & 7] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[i % kRing], p[c][i >> 3], acc[c][i & 7], 0, 0, 0);
      if (c == 1 && i + kRing < 16) get(vbuf, t - 1, i + kRing);
      __builtin_amdgcn_sched_barrier(0);
    };
    product(0, 0);
    put_sk(t + 2, sk);  // its buffer held tile t's, which the last walk read
    put_sv(t + 1, sv);
    load_v(rv, 1);
    product(0, 1);
    sk = load_sk(3);
    sv = load_sv(2);
#pragma unroll
    for (int u = 0; u < 2; u++) {
      at[1][u] = at[2][u];
      at[2][u] = at[3][u];
    }
    place(at[3], idn, t + 4);
    idn = ids(t + 5);
    // the scores are read by ordinary instructions from here on
    asm volatile("s_nop 10" : "+v"(sc[0]), "+v"(sc[1]));
    const int row0 = kKeys * t + 32 * kp;
    if (row0 + 32 > first + 1) {  // some row of the block does not see some key (uniform)
      int x = lane;
      asm volatile("" : "+v"(x));
      const int key0 = row0 + 4 * (x >> 5);
#pragma unroll
      for (int c = 0; c < 2; c++)
#pragma unroll
        for (int e = 0; e < 16; e++)
          sc[c][e] = key0 + 16 * (e & 1) + 8 * (e >> 3) + ((e & 7) >> 1) >= lim[c] ? -__builtin_inff() : sc[c][e];
    }
    // The reference point moves only when weights would pass 2^8.
    float shift[2], top[2];
    bool moved = false;
#pragma unroll
    for (int c = 0; c < 2; c++) {
      product(1 + c, 0);
      top[c] = fmaxf(sc[c][0], sc[c][1]);
#pragma unroll
      for (int e = 2; e < 8; e += 2) top[c] = fmaxf(fmaxf(top[c], sc[c][e]), sc[c][e + 1]);
      product(1 + c, 1);
#pragma unroll
      for (int e = 8; e < 16; e += 2) top[c] = fmaxf(fmaxf(top[c], sc[c][e]), sc[c][e + 1]);
    }
    product(3, 0);
#pragma unroll
    for (int c = 0; c < 2; c++) {
      top[c] = mi::max_xor32(top[c]) * c2;
      const bool any = __any(top[c] > m[c] + 8.f);
      const float mn = any ? fmaxf(m[c], top[c]) : m[c];
      shift[c] = __builtin_amdgcn_exp2f(m[c] - mn);
      m[c] = mn;
      l[c] *= shift[c];
      moved = moved || any;
      if (c == 0) product(3, 1);
    }
    uint32_t pn[2][8];  // weights as pairs
#pragma unroll
    for (int i = 4; i < 16; i++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
        product(i, c);
        const int k0 = (2 * (i - 4) + c) * 2 / 3, k1 = (2 * (i - 4) + c + 1) * 2 / 3;
#pragma unroll
        for (int k = k0; k < k1; k++) {  // 16 pairs over 24 products
          const int cc = k >> 3, e = 2 * (k & 7);
          const float ya = __builtin_amdgcn_exp2f(fmaf(sc[cc][e], c2, -m[cc]));
          const float yb = __builtin_amdgcn_exp2f(fmaf(sc[cc][e + 1], c2, -m[cc]));
          l[cc] += ya + yb;
          // the MFMA's operand: off by 2^-11 of itself at most
          pn[cc][k & 7] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)ya, (_Float16)yb});
          asm volatile("" : "+v"(pn[cc][k & 7]), "+v"(l[cc]));  // here, not where it is used
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    if (moved) {  // uniform
#pragma unroll
      for (int c = 0; c < 2; c++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
          // sixteen at a time, in ordinary registers and back: all would not fit
          asm volatile("" : "+a"(acc[c][i]));
          acc[c][i] *= shift[c];
          asm volatile("" : "+a"(acc[c][i]));
        }
    }
#pragma unroll
    for (int c = 0; c < 2; c++)
#pragma unroll
      for (int i = 0; i < 2; i++)
      {
        p[c][i] = __builtin_bit_cast(
            f16x8, u32x4{pn[c][4 * i], pn[c][4 * i + 1], pn[c][4 * i + 2], pn[c][4 * i + 3]});
        asm volatile("" : "+v"(p[c][i]));
      }
    mi::sync_lds();
  }
  // The rows that the wave finishes, and their gates: f16 gates are loaded here, ahead of
  // the stores that a later load would wait for.
  const int r0 = 64 * qb + 32 * kp;
  auto out_row = [&](int i, int64_t& tok, int& head) {
    const int rr = max(0, min(r0 + i, nrows - 1));
    const int at = __builtin_amdgcn_readfirstlane(token(rr));
    tok = q.q0 + tok0 + at;
    head = h * a.R + rr - at * a.R;
  };
  const bool early = cuts == 1 && a.gate && !a.gate32;
  f16x4 gates[32];
  if (early) {
#pragma unroll
    for (int i = 0; i < 32; i++) {
      int64_t tok;
      int head;
      out_row(i, tok, head);
      gates[i] = *(const f16x4*)((const _Float16*)a.gate + tok * a.g_ts + head * a.g_hs + 4 * lane);
    }
  }
  if (ta < tz) {
    const char* const vr = vbuf + (((tz - 1) & 1) * 2 + kp) * kHalf + opnd;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const f16x8 vf = *(const f16x8*)(vr + 1024 * i);
#pragma unroll
      for (int c = 0; c < 2; c++)
        acc[c][i & 7] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, p[c][i >> 3], acc[c][i & 7], 0, 0, 0);
    }
  }

  // ---- the key halves join: wave (qb, kp) finishes rows 32 kp of its 64 and hands
  // the others to its partner.
#pragma unroll
  for (int c = 0; c < 2; c++) {
    l[c] = mi::sum_xor32(l[c]);
    if (lost) l[c] = __builtin_nanf("");
  }
  __syncthreads();  // every wave is done with the tiles
  f32x4* const box = (f32x4*)lds;                    // [2 qb][2 kp][32][64]
  float2* const mlbox = (float2*)(box + 4 * 32 * 64);  // [2][2][32]
  {
    f32x4* const dst = box + (2 * qb + 1 - kp) * 32 * 64;
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
      for (int e4 = 0; e4 < 4; e4++)
        dst[(i * 4 + e4) * 64 + lane] = f32x4{acc[1][i][4 * e4], acc[1][i][4 * e4 + 1],
                                              acc[1][i][4 * e4 + 2], acc[1][i][4 * e4 + 3]};
    if (hl == 0) mlbox[(2 * qb + 1 - kp) * 32 + col] = float2{m[1], l[1]};
  }
  mi::sync_lds();
  const f32x4* const src = box + (2 * qb + kp) * 32 * 64;
  const float2 ml = mlbox[(2 * qb + kp) * 32 + col];
  const float top = fmaxf(m[0], ml.x);
  float fa = __builtin_amdgcn_exp2f(m[0] - top), fb = __builtin_amdgcn_exp2f(ml.x - top);
  const float sum = l[0] * fa + ml.y * fb;
  const int r = 64 * qb + 32 * kp + col;
  if (cuts == 1) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    fa *= inv;
    fb *= inv;
  }
  int64_t slot = 0;
  if (cuts > 1) {  // slots: the first pieces of the blocks that are cut, then the others
    double cut = 0.0, more = 0.0;
    for (int i = tid; i < s; i += 256) {
      const Blocks o = get_blocks(a, i);
      cut += o.nb - o.past(piece);
      more += pieces(o, piece, true);
    }
    const int cut0 = (int)block_sum<256>(cut, sums), more0 = (int)block_sum<256>(more, sums);
    const int b1 = q.past(piece), mine = q.nb - b1;
    const int at = cut0 * G + h * mine + (q.nb - 1 - b);                 // of the blocks
    const int second = more0 * G + h * (per - q.nb) + (q.nb - 1 - b);    // of the pieces k >= 1
    if (k == 0) {
      slot = at;
      if (tid == 0 && at < kSplitBlocks) x.blocks[at] = int4{s, h, b, second};
    } else {
      int add = 0;
      for (int kk = 1; kk < k; kk++) add += q.nb - q.past((int64_t)kk * piece);
      slot = kSplitBlocks + second + add;
    }
    if (slot >= kSlots || (k == 0 && slot >= kSplitBlocks)) return;  // cannot be: piece_tiles
    if (hl == 0 && r < nrows)
      ((float2*)x.part_ml)[slot * kRows + r] = float2{top, sum};
  }
  // The rows go through LDS once more, to be written whole: a wave's own 32, in what it
  // has read of the box.
#pragma unroll
  for (int i = 0; i < 8; i++)
#pragma unroll
    for (int e4 = 0; e4 < 4; e4++) {
      const f32x4 o = src[(i * 4 + e4) * 64 + lane];
#pragma unroll
      for (int n = 0; n < 4; n++) acc[0][i][4 * e4 + n] = acc[0][i][4 * e4 + n] * fa + o[n] * fb;
    }
  f32x4* const rows = box + (2 * qb + kp) * 32 * 64;  // [32][64], row r's piece x at x ^ (r & 7)
#pragma unroll
  for (int g = 0; g < 4; g++) {
    const bool odd = odd_row[g] < lim[0];
#pragma unroll
    for (int x = 0; x < 8; x++) {
      // columns 64 g + 32 (x / 4) + 16 hl + 4 (x % 4) ..: value j is block 2 g + j / 2,
      // element 8 (j % 2) + x
      f32x4 y;
#pragma unroll
      for (int j = 0; j < 4; j++) y[j] = odd ? __builtin_nanf("") : acc[0][2 * g + (j >> 1)][8 * (j & 1) + x];
      rows[64 * col + ((16 * g + 8 * (x >> 2) + 4 * hl + (x & 3)) ^ (col & 7))] = y;
    }
  }
  // (Few instructions: code that runs once a workgroup costs what its fetching does.)
  if (cuts > 1) {
    for (int i = 0; i < min(32, nrows - r0); i++)
      *(f32x4*)(x.part_o + (slot * kRows + r0 + i) * D + 4 * lane) = rows[64 * i + (lane ^ (i & 7))];
    return;
  }
  if (early) {
#pragma unroll
    for (int i = 0; i < 32; i++) {
      f32x4 y = rows[64 * i + (lane ^ (i & 7))];
      int64_t tok;
      int head;
      out_row(i, tok, head);
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] = mi::gate_mul(y[e], (float)gates[i][e]);
      if (r0 + i < nrows) mi::store4(a, tok, head, 4 * lane, y);
    }
  } else {
    for (int i = 0; i < min(32, nrows - r0); i++) {
      int64_t tok;
      int head;
      out_row(i, tok, head);
      mi::put4(a, tok, head, 4 * lane, rows[64 * i + (lane ^ (i & 7))]);
    }
  }
}

// Joins the pieces of the blocks that are cut: a workgroup per (block, 16 rows), a
// wave per row and four columns a thread.  A workgroup per sequence behind them
// makes every token NaN of one beyond max_q or max_len.
__global__ void __launch_bounds__(256) paged_prefill_merge_kernel(const AttnArgs a, const PrefillExtra x) {
  if (blockIdx.x >= 8 * kSplitBlocks) {
    const Blocks q = get_blocks(a, blockIdx.x - 8 * kSplitBlocks);
    const int width = a.pv.G * a.R * D;
    for (int tok = 0; tok < (q.bad ? q.nq : 0); tok++)
      for (int i = threadIdx.x; i < width; i += 256)
        a.out[(int64_t)(q.q0 + tok) * width + i] = (_Float16)__builtin_nanf("");
    return;
  }
  const int at = blockIdx.x >> 3, part = blockIdx.x & 7;
  const int2 c = *x.count;
  if (at >= min(c.x, kSplitBlocks)) return;
  const int4 blk = x.blocks[at];
  const int s = blk.x, h = blk.y, b = blk.z, second = blk.w, piece = c.y;
  const Blocks q = get_blocks(a, s);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int nrows = min(q.tb, q.nq - b * q.tb) * a.R, cuts = (q.tiles(b) + piece - 1) / piece;
  for (int r = 16 * part + w; r < min(16 * part + 16, nrows); r += 4) {
    float top = kNegBig, sum = 0.f;
    f32x4 y = {};
    int add = 0;
    for (int k = 0; k < cuts; k++) {
      const int64_t slot = k ? kSplitBlocks + second + add : at;
      if (k) add += q.nb - q.past((int64_t)k * piece);
      const float2 ml = ((const float2*)x.part_ml)[slot * kRows + r];
      const f32x4 o = *(const f32x4*)(x.part_o + (slot * kRows + r) * D + 4 * lane);
      const float mn = fmaxf(top, ml.x), f = __builtin_amdgcn_exp2f(top - mn),
                  g = __builtin_amdgcn_exp2f(ml.x - mn);
      sum = sum * f + ml.y * g;
      y = y * f + o * g;
      top = mn;
    }
    const int tok = r / a.R;
    mi::put4(a, q.q0 + b * q.tb + tok, h * a.R + r - tok * a.R, 4 * lane,
             y * (sum == 0.f ? 0.f : 1.f / sum));
  }
}

constexpr int kLds = 8 * kHalf + 2 * 2048;

}  // namespace

namespace mi {

size_t paged_prefill_workspace(int32_t, int32_t, int32_t, int32_t, int, int) {
  return (size_t)kSlots * kRows * (D + 2) * sizeof(float) + kSplitBlocks * sizeof(int4) + 64;
}

mi_status paged_prefill(AttnArgs& a, void* workspace, hipStream_t s) {
  static std::atomic<uint64_t> done{0};
  MI_TRY(set_lds_limit((const void*)paged_prefill_kernel, kLds, done));
  PrefillExtra x;
  x.part_o = (float*)workspace;
  x.part_ml = x.part_o + (size_t)kSlots * kRows * D;
  x.blocks = (int4*)(x.part_ml + (size_t)kSlots * kRows * 2);
  x.count = (int2*)(x.blocks + kSplitBlocks);
  const int tb = kRows / a.R;
  // blocks of the batch's sequences, and the pieces that come on top
  const int64_t wgs = ((int64_t)a.n / tb + a.pv.batch) * a.pv.G + kShare;
  const int64_t gx = std::min<int64_t>(wgs, 1 << 22);
  MI_HIP(launch("paged_prefill", paged_prefill_kernel,
                dim3((unsigned)gx, (unsigned)((wgs + gx - 1) / gx)), dim3(256), kLds, s, a, x));
  MI_HIP(launch("paged_merge", paged_prefill_merge_kernel, dim3((unsigned)(8 * kSplitBlocks + a.pv.batch)),
                dim3(256), 0, s, a, x));
  return MI_OK;
}

}  // namespace mi
