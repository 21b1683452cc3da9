// Paged 4-bit KV cache: the layout of a tile and what the kernels that fill
// it, read it and attend over it share.
//
// A page holds page_rows rows (a power of two, 32 to 1024) of every KV head;
// pages is [num_pages][G][page_rows / 32][kTileBytes].  A tile is 32 rows of
// one KV head: 4-bit codes of K and of V, then their scales and offsets in
// f16, one pair per row and group of 64 columns.  A value is
//   f16((16 + code) * scale + offset),
// one rounding: a 4-bit code put into bits 6..9 of an f16 whose exponent is
// that of 16 reads 16 + code, so a pair of values costs a shift, an and-or
// and a packed fma.  (Codes in the low mantissa bits, 1024 + code, need an
// exact subtraction more per pair; an offset for code 0 at 1024 times the
// scale would lose 6 bits of it, at 16 times it is exact to 1/150 of a step.)
//
// Row r = 16 sub + m = 16 sub + 4 quad + i of a tile, which is where the
// 16x16x32 MFMA wants its operands:
//   K, column 64 g + 16 quad + 8 step + e: nibble e of word
//       ((2 sub + g / 2) * 64 + 16 quad + m) * 4 + 2 (g % 2) + step
//     (lane 16 quad + m reads 16 bytes: its A operands of two groups);
//   V, column 64 g + 4 n + j: nibble i + 4 sub of word
//       (64 g + 16 quad + n) * 4 + j
//     (eight keys of a column to a word: a lane's A operand of V^T);
//   K scale and offset of (row, g): half 2 (4 row + g), +1, from kKScale;
//   V scale of (row, g): half (4 g + quad) * 16 + 2 i + sub from kVScale, its
//     offset 8 halves on.
#pragma once

#include "common.h"

namespace mi {

constexpr int kTileRows = 32;
constexpr int kTileBytes = 9216;
constexpr int kVCodes = 4096, kKScale = 8192, kVScale = 8704;
constexpr int kQuantGroup = 64;
constexpr int kPageRowsMin = 32, kPageRowsMax = 1024;
constexpr int kPagedRatioMax = 16;  // query heads per KV head

// A load through the scalar cache of a table that no kernel writes while it is
// read; the address is the same for the whole wave.
__device__ __forceinline__ int32_t uniform_load(const int32_t* p) {
  return *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)p;
}

// The pages of one layer and the rows of a batch of sequences in them.
struct PagedView {
  uint8_t* pages;
  const int32_t* table;   // [batch][cols] page of rows [j page_rows, (j+1) page_rows)
  const int32_t* kv_len;  // [batch] rows of a sequence, the call's tokens included
  const int32_t* cu_q;    // [batch + 1] first token of a sequence; null: one token each
  int64_t num_pages;
  int32_t cols, page_shift, batch, G;

  // Page of tile t (32-row index) of sequence s, the same for a whole wave; -1
  // past the table.
  __device__ __forceinline__ int32_t page(int s, int t) const {
    const int j = t >> (page_shift - 5);
    return j < cols ? uniform_load(table + (int64_t)s * cols + j) : -1;
  }
  // Base of tile t of KV head h in page id; null where the pool has no such page.
  __device__ __forceinline__ uint8_t* at(int32_t id, int h, int t) const {
    if (id < 0 || id >= num_pages) return nullptr;
    const int pt = page_shift - 5;  // tiles per page, as a shift
    return pages + (((int64_t)id * G + h) * ((int64_t)1 << pt) + (t & ((1 << pt) - 1))) * kTileBytes;
  }
  __device__ __forceinline__ uint8_t* tile(int s, int h, int t) const { return at(page(s, t), h, t); }
  // Tokens [q0, q0 + nq) of the call belong to sequence s (nq may be <= 0 for
  // a table that does not ascend; tokens are bounded by n in the kernels).
  __device__ __forceinline__ void tokens(int s, int& q0, int& nq) const {
    q0 = cu_q ? cu_q[s] : s;
    nq = cu_q ? cu_q[s + 1] - q0 : 1;
  }
};

// The arguments that every paged entry point shares.
mi_status paged_view(void* pages, int64_t num_pages, int32_t page_rows, const int32_t* table,
                     int32_t cols, const int32_t* kv_len, const int32_t* cu_q, int32_t batch,
                     int32_t num_kv_heads, int32_t head_dim, PagedView* out);

// A pair of codes of word w, its nibbles k (low half) and k + 4 (high half),
// as 16 + code in f16.  `sixteens` is 0x4c004c00 in a vector register
// (mi::sixteens()): and-or is one instruction only if no more than one of its
// operands is a constant or a scalar register.
template <int K>
__device__ __forceinline__ f16x2 codes16(uint32_t w, uint32_t sixteens) {
  constexpr int sh = 6 - 4 * K;
  const uint32_t x = sh >= 0 ? w << (sh & 31) : w >> (-sh & 31);
  return __builtin_bit_cast(f16x2, (x & 0x03c003c0u) | sixteens);
}
__device__ __forceinline__ uint32_t sixteens() {
  uint32_t v;
  asm("v_mov_b32 %0, 0x4c004c00" : "=v"(v));
  return v;
}

__device__ __forceinline__ f16x2 pk_fma(f16x2 a, f16x2 b, f16x2 c) {
  return __builtin_elementwise_fma(a, b, c);
}

// The top bits of the halves (rows) of scales s and offsets o whose code 15, the one
// furthest out, stands for no finite value (an exponent that is all ones carries there).
__device__ __forceinline__ uint32_t past_f16(uint32_t s, uint32_t o) {
  const f16x2 top = pk_fma(f16x2{31, 31}, __builtin_bit_cast(f16x2, s), __builtin_bit_cast(f16x2, o));
  return ((__builtin_bit_cast(uint32_t, top) & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
}

// Eight values of one scale and offset, in the order {0,4,1,5,2,6,3,7} of the
// word's nibbles.
__device__ __forceinline__ f16x8 dequant_row(uint32_t w, f16x2 scale, f16x2 offset,
                                             uint32_t x16) {
  const f16x2 a = pk_fma(codes16<0>(w, x16), scale, offset);
  const f16x2 b = pk_fma(codes16<1>(w, x16), scale, offset);
  const f16x2 c = pk_fma(codes16<2>(w, x16), scale, offset);
  const f16x2 d = pk_fma(codes16<3>(w, x16), scale, offset);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// Eight keys of one V column; scale, offset: in the same order {0,4,1,5,..}.
__device__ __forceinline__ f16x8 dequant_col(uint32_t w, f16x8 s, f16x8 o, uint32_t x16) {
  const f16x2 a = pk_fma(codes16<0>(w, x16), f16x2{s[0], s[1]}, f16x2{o[0], o[1]});
  const f16x2 b = pk_fma(codes16<1>(w, x16), f16x2{s[2], s[3]}, f16x2{o[2], o[3]});
  const f16x2 c = pk_fma(codes16<2>(w, x16), f16x2{s[4], s[5]}, f16x2{o[4], o[5]});
  const f16x2 d = pk_fma(codes16<3>(w, x16), f16x2{s[6], s[7]}, f16x2{o[6], o[7]});
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

}  // namespace mi
