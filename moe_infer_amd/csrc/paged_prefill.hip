// Attention over the paged 4-bit cache for many tokens: prompts, and chunks
// behind cached rows.
//
// A workgroup takes blocks of 256 / KP rows, the (token, query head of the group) pairs
// of consecutive tokens of one sequence and KV head, and walks the keys that they see
// in tiles of 32 KP.  The four waves dequantise a tile once into LDS as f16, in MFMA
// operand order; wave (qb, kp) multiplies rows 64 qb .. + 63 with keys 32 kp .. + 31 of
// it (v_mfma_f32_32x32x16_f16, S^T = K Q^T, O^T += V^T P^T), so that every operand read
// from LDS feeds two products.  KP = 1: four waves use what is dequantised, 3600 clocks
// a tile to a wave, 2048 of them MFMA; KP = 2: two do, 4600 clocks, and the two halves of
// the keys join at the end, but a block is half as long, which is what small calls and
// sequences of up to 128 rows want (16 sequences of 128 rows behind 8192: 75 us against 88 for KP = 1; 16 of
// 160: 113 against 90; a prompt of 4096 tokens, 8 heads a group: 232 against 194).
//
// Bound: the instructions that a wave alone on its SIMD issues (535 of four clocks a tile
// for KP = 1 and 690 for KP = 2, 64 of them MFMAs of 32 clocks).  What a tile needs besides
// its products is issued between them, each half of a word's dequantisation behind a
// product of K Q^T, the softmax of tile t behind those of P V of tile t - 1.  O^T of 64
// rows takes the 256 accumulation registers, so the scores have to come out in ordinary
// ones: their MFMAs are asm, which the compiler would otherwise give the accumulation form
// as well.
//
// The keys of all blocks, in the order in which Blocks pairs them, are dealt evenly to one
// workgroup a CU: ragged batches and causal prompts cost what they hold (chunks behind
// 2000 to 16000 rows: 366 us against 430 where whole pieces were dealt).  What a share
// begins and another ends, the merge kernel joins: it reads and writes as much as the
// partials are, 22 us for 128 blocks of 256 rows.
#include <algorithm>

#include "paged_attn.h"

namespace {

using mi::AttnArgs;
using mi::kNegBig;

constexpr int D = mi::kHeadDim;
constexpr int kHalf = 16384;  // bytes of 32 keys, K or V, as f16
constexpr int kShares = 256;  // workgroups of a call, one per CU, with an even share each
constexpr int kOver = 384;    // what starting and ending a block takes, in keys
// Keys below which shares are not made smaller: 256 against 512, 100 tokens behind 2000
// rows 40 us and 45, 8 prompts of 100 38 and 48; less than a block's kOver gains nothing.
constexpr int kMinShare = 256;

// KP: parts of a tile's keys, each another wave's.  256 / KP rows of a block, 32 KP
// keys of a tile.
constexpr int rows_of(int kp) { return 256 / kp; }

// What a share leaves to the merge.
struct Share {
  int32_t rows, token, head;  // of a block that it begins and does not end: rows (or 0), first
                              // token, KV head
  int32_t last, slot;         // the share that ends it, where its own part is
  int32_t joins;              // its first piece continues a block (in slot 2 share)
};
struct PrefillExtra {
  float* part_o;   // [2 kShares][rows][D]
  float* part_ml;  // [2 kShares][rows][2]
  Share* shares;   // [kShares]
};

// A sequence as blocks of tb tokens.  The walk takes them in pairs, the last with the
// first and so on inwards: each pair costs the same.
template <int KP>
struct Blocks {
  int q0, nq, len, nb, tb;
  bool bad;
  __device__ __forceinline__ int first() const { return len - nq; }
  // rows that block b's last token sees, and tiles of them
  __device__ __forceinline__ int end(int b) const { return first() + min(nq, tb * (b + 1)); }
  __device__ __forceinline__ int tiles(int b) const { return max(end(b) + 32 * KP - 1, 32 * KP) / (32 * KP); }
  // Costs in keys: a block's, a pair's, those of one KV head.
  __device__ __forceinline__ int64_t cost(int b) const { return (int64_t)max(first(), 0) + kOver + (int64_t)tb * (b + 1); }
  __device__ __forceinline__ int64_t pair() const { return cost(0) + cost(nb - 1); }
  __device__ __forceinline__ int64_t all() const { return nb * pair() / 2; }
  // tiles before x of a block's cost
  __device__ __forceinline__ int upto(int b, int64_t x) const {
    const int t = tiles(b);
    return x >= cost(b) ? t : (int)min((int64_t)t, max(x - kOver, (int64_t)0) / (32 * KP));
  }
};
template <int KP>
__device__ __forceinline__ Blocks<KP> get_blocks(const AttnArgs& a, int s) {
  Blocks<KP> r;
  a.pv.tokens(s, r.q0, r.nq);
  r.len = a.pv.kv_len[s];
  r.bad = r.len < 0 || r.len > a.max_len || r.nq > a.max_q;
  if (r.nq <= 0 || r.q0 < 0 || (int64_t)r.q0 + r.nq > a.n) r.nq = 0;
  r.tb = rows_of(KP) / a.R;
  r.nb = r.bad ? 0 : (r.nq + r.tb - 1) / r.tb;
  return r;
}
__device__ __forceinline__ int64_t divide(int64_t x, int64_t y) {  // of what is not negative
  return (x | y) >> 32 ? x / y : (int64_t)((uint32_t)x / (uint32_t)y);
}

__device__ __forceinline__ void mfma_s(f32x16& c, f16x8 a, f16x8 b) {
  asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
}
__device__ __forceinline__ void mfma_s0(f32x16& c, f16x8 a, f16x8 b) {
  asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "v"(b));
}

template <int KP>
__global__ void __launch_bounds__(256, 1) paged_prefill_kernel(const AttnArgs a, const PrefillExtra x) {
  extern __shared__ char lds[];  // K, V [2][2 halves], their scales; then the join of the key halves
  __shared__ int odd_row[4];  // least masked row whose V group may not be finite
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int kRows = rows_of(KP), kKeys = 32 * KP;
  const int qb = KP == 1 ? w : w & 1, kp = KP == 1 ? 0 : w >> 1;
  const int G = a.pv.G;
  // Neighbouring shares, which read the same keys, to the CUs of one XCD.
  const int share = (blockIdx.x & 7) * (kShares / 8) + (blockIdx.x >> 3);

  int s;
  int64_t before, at_cost = 0, size = 0, stop = 0;
  mi::find_seq<256>(
      a.pv.batch,
      [&](int i) {
        const auto q = get_blocks<KP>(a, i);
        return q.nb ? G * q.all() : (int64_t)0;
      },
      [&](int64_t total) {
        size = max((total + kShares - 1) / kShares, (int64_t)kMinShare);
        at_cost = min(share * size, total);
        stop = min(at_cost + size, total);
        return at_cost;
      },
      s, before);
  const int64_t start = at_cost;
  Share left{0, 0, 0, 0, 0, 0};
  while (at_cost < stop) {
    // ---- the next block, and which of its tiles
    auto q = get_blocks<KP>(a, s);
    q.q0 = mi::uniform(q.q0);
    q.nq = mi::uniform(q.nq);
    q.len = mi::uniform(q.len);
    q.nb = mi::uniform(q.nb);
    const int64_t all = q.nb ? q.all() : 0;
    if (at_cost - before >= G * all) {
      before += G * all;
      s++;
      continue;
    }
    const int h = (int)divide(at_cost - before, all);
    int64_t x0 = at_cost - before - h * all;  // of the head's cost, then of the block's
    const int pair = (int)divide(x0, q.pair());
    x0 -= pair * q.pair();
    int b = q.nb - 1 - pair;
    if (x0 >= q.cost(b)) {
      x0 -= q.cost(b);
      b = pair;
    }
    const int64_t begin = at_cost - x0, full = q.cost(b);
    at_cost = min(stop, begin + full);
    const int ta = q.upto(b, x0), tz = q.upto(b, at_cost - begin);
    if (ta == tz) continue;
    const bool whole = ta == 0 && tz == q.tiles(b);
    const int slot = 2 * share + (begin + x0 != start);
    const int tok0 = b * q.tb, ntok = min(q.tb, q.nq - tok0), nrows = ntok * a.R;
    if (ta != 0) left.joins = 1;
    else if (!whole) left = Share{nrows, q.q0 + tok0, h, (int)divide(begin + full - 1, size), slot, left.joins};
    const int first = q.first() + tok0;  // row of the block's first token
    const int end = first + ntok;

    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // nothing that hangs on it is kept in registers over blocks
    const int lane = tid & 63, col = lane & 31, hl = lane >> 5;
    __syncthreads();  // the last block is out of LDS
    if (tid < 4) odd_row[tid] = INT32_MAX;

    // ---- a tile's words: those of KP 32-row tiles.  A thread takes a 16-byte piece of K
    // and of V of each, and a word of the scales of one of them (of K and of V each, or of
    // K in the lower waves and of V in the upper), which go through LDS a tile earlier (in
    // registers every thread would hold 20 words of them).
    u32x4 rk[KP], rv[KP];
    uint32_t sk, sv;
    int lost = INT32_MAX;  // least row in sight whose page is not there
    // Where tiles t + 1, t + 2 and t + 3 lie (at[i][u]: 32-row tile KP (t + i) + u), looked up a tile
    // before their loads; the page's id is loaded two tiles before that, by a vector load
    // (a scalar one would hold up every wait for LDS until it has come).  What has no
    // place (behind the last row; a page that the pool does not have, which is lost)
    // reads page 0, and counts for nothing.
    const uint8_t* at[4][KP];
    const int pt = a.pv.page_shift - 5;
    const int tend = (end + 31) >> 5;  // 32-row tiles
    const int tlim = (int)min((int64_t)tend, (int64_t)a.pv.cols << pt);
    const uint32_t npages = (uint32_t)a.pv.num_pages;
    const uint64_t page_bytes = ((uint64_t)a.pv.G << pt) * mi::kTileBytes;
    const uint8_t* const pages = a.pv.pages + ((uint64_t)h << pt) * mi::kTileBytes;
    const int32_t* const table = a.pv.table + (int64_t)s * a.pv.cols;
    auto ids = [&](int t) {  // lane u's: page of tile KP t + u, or any where there is none
      return table[min((KP * t + (lane & (KP - 1))) >> pt, a.pv.cols - 1)];
    };
    auto place = [&](const uint8_t* (&p)[KP], int32_t idv, int t) {
#pragma unroll
      for (int u = 0; u < KP; u++) {
        const uint32_t id = __builtin_amdgcn_readlane(idv, u);
        const int ok = (KP * t + u < tlim) & (id < npages);
        if ((KP * t + u < tend) & (ok ^ 1)) lost = min(lost, 32 * (KP * t + u));
        const uint64_t off = id * page_bytes + (uint32_t)(((KP * t + u) & ((1 << pt) - 1)) * mi::kTileBytes);
        p[u] = pages + (ok ? off : 0);
      }
    };
    const int m16 = lane & 15, quad = lane >> 4;
    const int su = w >> 1, sat = 4 * (tid & 127);  // the thread's word of scales: tile, offset
    auto buffer = [&](const uint8_t* p) {
      return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, mi::kTileBytes, 0x00020000);
    };
    auto load_k = [&](u32x4 (&r)[KP], int i) {
#pragma unroll
      for (int u = 0; u < KP; u++) r[u] = __builtin_amdgcn_raw_buffer_load_b128(buffer(at[i][u]), 16 * tid, 0, 0);
    };
    auto load_v = [&](u32x4 (&r)[KP], int i) {
#pragma unroll
      for (int u = 0; u < KP; u++)
        r[u] = __builtin_amdgcn_raw_buffer_load_b128(buffer(at[i][u]), 16 * tid, mi::kVCodes, 0);
    };
    auto load_sk = [&](int i) {
      return __builtin_amdgcn_raw_buffer_load_b32(buffer(KP == 2 && su ? at[i][KP - 1] : at[i][0]), sat,
                                                  mi::kKScale, 0);
    };
    auto load_sv = [&](int i) {
      return __builtin_amdgcn_raw_buffer_load_b32(buffer(KP == 2 && su ? at[i][KP - 1] : at[i][0]), sat,
                                                  mi::kVScale, 0);
    };
    const uint32_t x16 = mi::sixteens();
    char* const kbuf = lds;
    char* const vbuf = lds + 2 * KP * kHalf;
    char* const ksc = lds + 8 * kHalf;  // [2][KP][512]
    char* const vsc = ksc + 1024 * KP;
    auto put_sk = [&](int t, uint32_t y) { *(uint32_t*)(ksc + (t & 1) * 512 * KP + (KP == 2 ? 4 * tid : sat)) = y; };
    // V's word: scale or offset of rows 4 quad + i and 16 more, of group g.  Rows that no
    // token of the block sees read as zero, and so do values that may not be finite in rows that
    // some token does not see (the MFMA would make NaN of 0 * NaN for it); the
    // tokens that do see such a row get their NaN at the end.
    auto put_sv = [&](int t, uint32_t y) {
      if (kKeys * (t + 1) > first + 1) {  // uniform: not seen whole
        int x = tid;
        asm volatile("" : "+v"(x));  // nothing of this is kept in registers over the tiles
        const int i = x & 3, sq = (x >> 3) & 3, g = (x >> 5) & 3;
        const int row = kKeys * t + (KP == 2 ? 32 * su : 0) + 4 * sq + i;
        y &= (row < end ? 0xffffu : 0u) | (row + 16 < end ? 0xffff0000u : 0u);
        const bool is_offset = x & 4;  // the scale's or the offset's other word is four lanes away
        const uint32_t other = __shfl_xor((int)y, 4, 64);
        const uint32_t odd = mi::past_f16(is_offset ? other : y, is_offset ? y : other);
        if (odd) {
          atomicMin(&odd_row[g], odd & 0x8000u ? row : row + 16);
          y &= ~((odd >> 15) * 0xffffu);
        }
      }
      *(uint32_t*)(vsc + (t & 1) * 512 * KP + (KP == 2 ? 4 * tid : sat)) = y;
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
        kso[i] = *(const f16x2*)(ksc + (t & 1) * 512 * KP + 512 * u + ksrc + 4 * i);
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
      *(f16x8*)(kbuf + ((t & 1) * KP + u) * kHalf + kdst + (((j >> 1) * 4 * 2 + (j & 1)) * 32) * 16) =
          f16x8{half[0][0], half[0][1], half[1][0], half[1][1], c[0], c[1], d[0], d[1]};
    };
    f16x8 vs, vo;
    auto get_vs = [&](int t, int u) {
      vs = *(const f16x8*)(vsc + (t & 1) * 512 * KP + 512 * u + vsrc);
      vo = *(const f16x8*)(vsc + (t & 1) * 512 * KP + 512 * u + vsrc + 16);
    };
    auto half_v = [&](uint32_t y) {
      half[0] = mi::pk_fma(mi::codes16<0>(y, x16), f16x2{vs[0], vs[1]}, f16x2{vo[0], vo[1]});
      half[1] = mi::pk_fma(mi::codes16<1>(y, x16), f16x2{vs[2], vs[3]}, f16x2{vo[2], vo[3]});
    };
    auto put_v = [&](uint32_t y, int t, int u, int j) {
      const f16x2 c = mi::pk_fma(mi::codes16<2>(y, x16), f16x2{vs[4], vs[5]}, f16x2{vo[4], vo[5]});
      const f16x2 d = mi::pk_fma(mi::codes16<3>(y, x16), f16x2{vs[6], vs[7]}, f16x2{vo[6], vo[7]});
      *(f16x8*)(vbuf + ((t & 1) * KP + u) * kHalf + vdst + ((j >> 1) * 64 + 16 * (j & 1)) * 16) =
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
    u32x4 k0[KP];
    uint32_t sk0 = 0, sk1 = 0, sv0 = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) id[i] = ids(ta + i);
    idn = ids(ta + 4);
    const float rinv = 1.f / (float)a.R;
    auto token = [&](int r) { return (int)(((float)r + 0.5f) * rinv); };  // r / R: r < 256
    {
      f16x8 y[kRows / 8];
#pragma unroll
      for (int i = 0; i < kRows / 8; i++) {
        const int r = kRows / 4 * w + 2 * i + hl, rr = r < nrows ? r : 0, tok = token(rr);
        y[i] = *(const f16x8*)(a.q + (int64_t)(q.q0 + tok0 + tok) * a.q_ts +
                               (h * a.R + rr - tok * a.R) * a.q_hs + 8 * col);
      }
#pragma unroll
      for (int i = 0; i < 4; i++) place(at[i], id[i], ta + i);
      if (KP == 2 || !su) {
        sk0 = load_sk(0);
        sk1 = load_sk(1);
      }
      if (KP == 2 || su) sv0 = load_sv(0);
      load_k(k0, 0);
      load_v(rv, 0);
      load_k(rk, 1);
      if (KP == 2 || !su) sk = load_sk(2);
      if (KP == 2) sv = load_sv(1);
      else if (su) sk = load_sv(1);
#pragma unroll
      for (int i = 0; i < kRows / 8; i++) {
        const int r = kRows / 4 * w + 2 * i + hl;
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
      for (int i = 0; i < 8; i++) {
        acc[c][i] = f32x16{};
        asm volatile("" : "+a"(acc[c][i]));
      }
    f16x8 p[2][2];
#pragma unroll
    for (int c = 0; c < 2; c++)
#pragma unroll
      for (int i = 0; i < 2; i++) p[c][i] = f16x8{};

    if (KP == 2 || !su) {
      put_sk(ta, sk0);
      put_sk(ta + 1, sk1);
    }
    __syncthreads();
    // the first walk's products with no weights read a buffer of zeros
    for (int i = tid; i < KP * kHalf / 16; i += 256)
      ((u32x4*)(vbuf + ((ta - 1) & 1) * KP * kHalf))[i] = u32x4{};
    if (KP == 2 || su) put_sv(ta, sv0);
#pragma unroll
    for (int u = 0; u < KP; u++) {
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
      ring[i % kRing] = *(const f16x8*)(buf + ((t & 1) * KP + kp) * kHalf + opnd + 1024 * i);
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
          // half of a word here and half behind the other product, or a word every other step
          const int x = KP == 2 ? ks : ks >> 1, u = x / 4 % KP;
          const bool isk = x < 4 * KP, one = KP == 2 || ks % 2 == 0, two = KP == 2 || ks % 2 == 1;
          const uint32_t y = isk ? rk[u][x & 3] : rv[u][x & 3];
          if (one) {
            if (isk) half_k(y, x & 3);
            else half_v(y);
          }
          if (KP == 1 && two) {
            if (isk) put_k(y, t + 1, u, x & 3);
            else put_v(y, t, u, x & 3);
          }
          __builtin_amdgcn_sched_barrier(0);
          if (ks == 0) mfma_s0(sc[1], ring[0], qf[1][0]);
          else mfma_s(sc[1], ring[ks % kRing], qf[1][ks]);
          if (ks + kRing < 16) get(kbuf, t, ks + kRing);
          else get(vbuf, t - 1, ks + kRing - 16);
          if (KP == 2) {
            if (isk) put_k(y, t + 1, u, x & 3);
            else put_v(y, t, u, x & 3);
            if (ks == 3) get_ks(t + 1, KP - 1);
          }
          if (ks == 7) {
            get_vs(t, 0);
            load_k(rk, 2);
          }
          if (KP == 2 && ks == 11) get_vs(t, KP - 1);
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
      if (KP == 2 || !su) put_sk(t + 2, sk);  // its buffer held tile t's, which the last walk read
      if (KP == 2) put_sv(t + 1, sv);
      else if (su) put_sv(t + 1, sk);
      load_v(rv, 1);
      product(0, 1);
      if constexpr (KP == 2) {
        sk = load_sk(3);
        sv = load_sv(2);
      } else {
        sk = __builtin_amdgcn_raw_buffer_load_b32(buffer(su ? at[2][0] : at[3][0]), sat,
                                                  su ? mi::kVScale : mi::kKScale, 0);
      }
#pragma unroll
      for (int u = 0; u < KP; u++) {
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
    // (Tokens without a row, whose gates may hold anything, are zero whatever those are.)
    const bool early = whole && a.gate && !a.gate32 && first >= 0;
    int r0 = 64 * qb + 32 * kp;
    // Lane i's: where row r0 + i (or the last one) lies in the gate and in the output.
    int64_t gate_at, out_at;
    auto find_rows = [&] {
      const int r = max(0, min(r0 + col, nrows - 1)), tok = token(r), head = h * a.R + r - tok * a.R;
      gate_at = (q.q0 + tok0 + tok) * a.g_ts + head * a.g_hs;
      out_at = ((int64_t)(q.q0 + tok0 + tok) * G * a.R + head) * D;
    };
    auto lane64 = [](int64_t x, int i) {
      return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), i) << 32 |
                       (uint32_t)__builtin_amdgcn_readlane((int)x, i));
    };
    f16x4 gates[32];
    // f16 gates are loaded ahead of the stores that a later load would wait for.
    auto load_gates = [&] {
      find_rows();
      if (early) {
#pragma unroll
        for (int i = 0; i < 32; i++)
          gates[i] = *(const f16x4*)((const _Float16*)a.gate + lane64(gate_at, i) + 4 * lane);
      } else {
#pragma unroll
        for (int i = 0; i < 32; i++) asm("" : "=v"(gates[i]));  // or the last block's would be kept
      }
    };
    load_gates();
    {
      const char* const vr = vbuf + (((tz - 1) & 1) * KP + kp) * kHalf + opnd;
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const f16x8 vf = *(const f16x8*)(vr + 1024 * i);
#pragma unroll
        for (int c = 0; c < 2; c++)
          acc[c][i & 7] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, p[c][i >> 3], acc[c][i & 7], 0, 0, 0);
      }
    }
#pragma unroll
    for (int c = 0; c < 2; c++) {
      l[c] = mi::sum_xor32(l[c]);
      if (lost < lim[c]) l[c] = __builtin_nanf("");
    }
    __syncthreads();  // every wave is done with the tiles

    // ---- the parts of the keys join: wave (qb, kp) finishes rows 32 kp of its 64 and hands
    // the others to its partner.
    f32x4* const box = (f32x4*)lds;  // a wave's [32][64]
    f32x4* const mine = box + (KP * qb + kp) * 32 * 64;
    if constexpr (KP == 2) {
      float2* const mlbox = (float2*)(box + 4 * 32 * 64);  // [2][2][32]
      f32x4* const dst = box + (2 * qb + 1 - kp) * 32 * 64;
#pragma unroll
      for (int i = 0; i < 8; i++) asm volatile("" : "+a"(acc[0][i]), "+a"(acc[1][i]));
#pragma unroll
      for (int i = 0; i < 8; i++)
#pragma unroll
        for (int e4 = 0; e4 < 4; e4++)
          dst[(i * 4 + e4) * 64 + lane] = f32x4{acc[1][i][4 * e4], acc[1][i][4 * e4 + 1],
                                                acc[1][i][4 * e4 + 2], acc[1][i][4 * e4 + 3]};
      if (hl == 0) mlbox[(2 * qb + 1 - kp) * 32 + col] = float2{m[1], l[1]};
      mi::sync_lds();
      const float2 ml = mlbox[(2 * qb + kp) * 32 + col];
      const float top = fmaxf(m[0], ml.x);
      const float fa = __builtin_amdgcn_exp2f(m[0] - top), fb = __builtin_amdgcn_exp2f(ml.x - top);
      l[0] = l[0] * fa + ml.y * fb;
      m[0] = top;
#pragma unroll
      for (int i = 0; i < 8; i++) {
#pragma unroll
        for (int e4 = 0; e4 < 4; e4++) {
          const f32x4 o = mine[(i * 4 + e4) * 64 + lane];
#pragma unroll
          for (int n = 0; n < 4; n++) acc[0][i][4 * e4 + n] = acc[0][i][4 * e4 + n] * fa + o[n] * fb;
        }
        asm volatile("" : "+a"(acc[0][i]));
      }
    }
    // ---- rows to memory: 32 at a time go through LDS once more, to be written whole; what is
    // written there is only read by its own wave.
#pragma unroll
    for (int c = 0; c < 2 / KP; c++) {
      if (c) {
        r0 += 32;
        load_gates();
      }
      const float f = !whole ? 1.f : l[c] == 0.f ? 0.f : 1.f / l[c];
#pragma unroll
      for (int i = 0; i < 8; i++) asm volatile("" : "+a"(acc[0][i]), "+a"(acc[1][i]));  // there until used
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const bool odd = odd_row[g] < lim[c];
#pragma unroll
        for (int x = 0; x < 8; x++) {
          // columns 64 g + 32 (x / 4) + 16 hl + 4 (x % 4) ..: value j is block 2 g + j / 2,
          // element 8 (j % 2) + x; row r's piece y at y ^ (r & 7)
          f32x4 y;
#pragma unroll
          for (int j = 0; j < 4; j++)
            y[j] = odd ? __builtin_nanf("") : acc[c][2 * g + (j >> 1)][8 * (j & 1) + x] * f;
          mine[64 * col + ((16 * g + 8 * (x >> 2) + 4 * hl + (x & 3)) ^ (col & 7))] = y;
        }
      }
      if (!whole) {
        if (hl == 0 && r0 + col < nrows)
          ((float2*)x.part_ml)[(int64_t)slot * kRows + r0 + col] = float2{m[c], l[c]};
        for (int i = 0; i < min(32, nrows - r0); i++)
          *(f32x4*)(x.part_o + ((int64_t)slot * kRows + r0 + i) * D + 4 * lane) = mine[64 * i + (lane ^ (i & 7))];
      } else {
        // (the loops stay short: code that runs once a workgroup costs what its fetching does)
        auto write = [&](int i, f32x4 y) {
          if (r0 + i < nrows)
            *(f16x4*)(a.out + lane64(out_at, i) + 4 * lane) =
                f16x4{(_Float16)y[0], (_Float16)y[1], (_Float16)y[2], (_Float16)y[3]};
        };
        if (early) {
#pragma unroll
          for (int i = 0; i < 32; i++) {
            f32x4 y = mine[64 * i + (lane ^ (i & 7))];
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = mi::gate_mul(y[e], (float)gates[i][e]);
            write(i, y);
          }
        } else {
#pragma unroll 1
          for (int i = 0; i < 32; i++) {
            f32x4 y = mine[64 * i + (lane ^ (i & 7))];
            if (a.gate && first + mi::uniform(token(r0 + i)) >= 0) {
              const f32x4 g = mi::gate4(a, lane64(gate_at, i) + 4 * lane);
#pragma unroll
              for (int e = 0; e < 4; e++) y[e] = mi::gate_mul(y[e], g[e]);
            }
            write(i, y);
          }
        }
      }
    }
  }
  if (threadIdx.x == 0) x.shares[share] = left;
}

// Joins the parts of the blocks that are cut: a workgroup per (share that begins one, 8
// rows), four columns a thread; wave w takes four of the rows and every other part from
// w / 2 on, and two waves join through LDS.  A workgroup per sequence behind them makes
// every token NaN of one beyond max_q or max_len.
constexpr int kMergeRows = 8;
template <int KP>
__global__ void __launch_bounds__(256) paged_prefill_merge_kernel(const AttnArgs a, const PrefillExtra x) {
  constexpr int kRows = rows_of(KP), kParts = kRows / kMergeRows;
  if (blockIdx.x >= kParts * kShares) {
    const auto q = get_blocks<KP>(a, blockIdx.x - kParts * kShares);
    const int width = a.pv.G * a.R * D;
    for (int tok = 0; tok < (q.bad ? q.nq : 0); tok++)
      for (int i = threadIdx.x; i < width; i += 256)
        a.out[(int64_t)(q.q0 + tok) * width + i] = (_Float16)__builtin_nanf("");
    return;
  }
  __shared__ f32x4 box[2][4][64];
  __shared__ float2 mlbox[2][4];
  const int share = blockIdx.x / kParts, part = blockIdx.x % kParts;
  const Share c = x.shares[share];
  if (kMergeRows * part >= c.rows) return;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r0 = kMergeRows * part + 4 * (w & 1), half = w >> 1;
  // the two rows that the wave writes, and their gates
  int64_t out_at[2];
  f32x4 gate[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int r = min(r0 + 2 * half + i, c.rows - 1), tok = r / a.R, head = c.head * a.R + r - tok * a.R;
    out_at[i] = ((int64_t)(c.token + tok) * a.pv.G * a.R + head) * D + 4 * lane;
    if (a.gate) gate[i] = mi::gate4(a, (int64_t)(c.token + tok) * a.g_ts + head * a.g_hs + 4 * lane);
  }
  float top[4], sum[4];
  f32x4 y[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    top[i] = kNegBig;
    sum[i] = 0.f;
    y[i] = f32x4{};
  }
  // Two parts at a time; what is not one weighs nothing, in the place of the first.
  for (int k0 = share + half; k0 <= c.last; k0 += 4) {
    float2 ml[2][4];
    f32x4 o[2][4];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int k = min(k0 + 2 * u, kShares - 1);
      const bool in = k == share || (k0 + 2 * u <= c.last && x.shares[k].joins);
      const int64_t row = (int64_t)(in && k > share ? 2 * k : c.slot) * kRows + r0;  // (of a slot's own)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        ml[u][i] = ((const float2*)x.part_ml)[row + i];
        o[u][i] = *(const f32x4*)(x.part_o + (row + i) * D + 4 * lane);
        if (!in) ml[u][i] = float2{kNegBig, 0.f};
      }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float mn = fmaxf(top[i], fmaxf(ml[0][i].x, ml[1][i].x));
      const float f = __builtin_amdgcn_exp2f(top[i] - mn), g0 = __builtin_amdgcn_exp2f(ml[0][i].x - mn),
                  g1 = __builtin_amdgcn_exp2f(ml[1][i].x - mn);
      sum[i] = sum[i] * f + ml[0][i].y * g0 + ml[1][i].y * g1;
      y[i] = y[i] * f + o[0][i] * g0 + o[1][i] * g1;
      top[i] = mn;
    }
  }
  // wave (w & 1, half) hands rows 2 (1 - half) .. of its four to the other half's
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int j = 2 * (1 - half) + i;
    const f32x4 mine = half ? y[i] : y[2 + i];
    box[w & 1][j][lane] = mine;
    if (lane == 0) mlbox[w & 1][j] = half ? float2{top[i], sum[i]} : float2{top[2 + i], sum[2 + i]};
  }
  mi::sync_lds();
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int j = 2 * half + i;
    if (r0 + j >= c.rows) break;
    const float2 ml = mlbox[w & 1][j];
    const float t = half ? top[2 + i] : top[i], l = half ? sum[2 + i] : sum[i], mn = fmaxf(t, ml.x);
    const float f = __builtin_amdgcn_exp2f(t - mn), g = __builtin_amdgcn_exp2f(ml.x - mn);
    const float all = l * f + ml.y * g, inv = all == 0.f ? 0.f : 1.f / all;
    f32x4 z = ((half ? y[2 + i] : y[i]) * f + box[w & 1][j][lane] * g) * inv;
    if (a.gate && inv != 0.f)  // zeros where a token attends nothing
#pragma unroll
      for (int e = 0; e < 4; e++) z[e] = mi::gate_mul(z[e], gate[i][e]);
    *(f16x4*)(a.out + out_at[i]) = f16x4{(_Float16)z[0], (_Float16)z[1], (_Float16)z[2], (_Float16)z[3]};
  }
}

constexpr int kLds = 8 * kHalf + 2 * 2048;

template <int KP>
mi_status run(const AttnArgs& a, const PrefillExtra& x, hipStream_t s) {
  static std::atomic<uint64_t> done{0};
  MI_TRY(mi::set_lds_limit((const void*)paged_prefill_kernel<KP>, kLds, done));
  MI_HIP(mi::launch("paged_prefill", paged_prefill_kernel<KP>, dim3(kShares), dim3(256), kLds, s, a, x));
  MI_HIP(mi::launch("paged_merge", paged_prefill_merge_kernel<KP>,
                    dim3((unsigned)(rows_of(KP) / kMergeRows * kShares + a.pv.batch)), dim3(256), 0, s, a, x));
  return MI_OK;
}

}  // namespace

namespace mi {

size_t paged_prefill_workspace() {
  return (size_t)2 * kShares * rows_of(1) * (D + 2) * sizeof(float) + kShares * sizeof(Share);
}

mi_status paged_prefill(AttnArgs& a, void* workspace, hipStream_t s) {
  PrefillExtra x;
  x.part_o = (float*)workspace;
  x.part_ml = x.part_o + (size_t)2 * kShares * rows_of(1) * D;
  x.shares = (Share*)(x.part_ml + (size_t)2 * kShares * rows_of(1) * 2);
  // Short blocks for sequences of up to 128 rows (measured at the top) and for calls too
  // small to fill the card, by rows times the longest sequence (at 2.6 M 35 us against
  // 43.5, at 5.1 M 38 and 44, at 17.9 M 54 and 56.5; at 32 M 84 and 75, at 67 M 92 and 77).
  const bool few = (double)a.n * a.R * a.pv.G * a.max_len < 20e6;
  return few || a.max_q * (int64_t)a.R <= rows_of(2) ? run<2>(a, x, s) : run<1>(a, x, s);
}

}  // namespace mi
