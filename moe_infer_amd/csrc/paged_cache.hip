// Filling and reading the paged 4-bit cache (paged.h).
//
// Append: Q and K are RMS-normed (optional) and rotated at the row they take,
// Q leaves as f16, K and V leave as 4-bit codes.  The arithmetic from the
// inputs to the codes is in 64 bits: a code is the nearest of sixteen, and a
// value next to the border of two would land on either side of it by the last
// bit of an f32 intermediate, a whole step away.  It is memory bound all the
// same for many tokens (gfx950 runs f64 at the f32 rate).
//
// A call whose sequences hold any number of tokens goes by tile: a workgroup
// takes one tile of one sequence and KV head, quantises the rows that the call
// brings, four to a wave, and stores whole words; rows of the tile that are
// not the call's keep their codes (K by 16-byte pieces of one row, V by merging
// nibbles; no other workgroup holds the same words).  A call of one token per
// sequence goes by row: a wave takes K or V of one row.
#include <algorithm>

#include "paged.h"
#include "rotary.h"

namespace mi {

mi_status paged_view(void* pages, int64_t num_pages, int32_t page_rows, const int32_t* table,
                     int32_t cols, const int32_t* kv_len, const int32_t* cu_q, int32_t batch,
                     int32_t num_kv_heads, int32_t head_dim, PagedView* out) {
  if (head_dim != kHeadDim)
    return fail(MI_ERR_UNSUPPORTED, "head_dim=%d (the kernels are built for %d)", head_dim,
                kHeadDim);
  if (!pages || !table || !kv_len) return fail(MI_ERR_INVALID_ARG, "null pointer argument");
  if ((uintptr_t)pages & 15) return fail(MI_ERR_INVALID_ARG, "pages must be 16-byte aligned");
  if (page_rows < kPageRowsMin || page_rows > kPageRowsMax || (page_rows & (page_rows - 1)))
    return fail(MI_ERR_INVALID_ARG, "page_rows=%d (a power of two, %d to %d)", page_rows,
                kPageRowsMin, kPageRowsMax);
  if (num_pages <= 0 || num_pages > INT32_MAX || cols <= 0 || batch <= 0 || num_kv_heads <= 0)
    return fail(MI_ERR_INVALID_ARG, "num_pages=%lld table columns=%d batch=%d num_kv_heads=%d",
                (long long)num_pages, cols, batch, num_kv_heads);
  if (batch > 65535) return fail(MI_ERR_UNSUPPORTED, "batch=%d above 65535 sequences", batch);
  *out = PagedView{(uint8_t*)pages, table, kv_len, cu_q, num_pages, cols,
                   __builtin_ctz((unsigned)page_rows), batch, num_kv_heads};
  return MI_OK;
}

}  // namespace mi

namespace {

constexpr int D = mi::kHeadDim;
// Waves to a tile of the append by tile: the chain of a row is long, so rows go side by
// side (prompts of 6580 tokens, two KV heads, without Q: 4 waves 28.8 us, 8 waves 20.5).
constexpr int kTileWaves = 8;

struct AppendArgs {
  mi::PagedView pv;
  const void *q, *k, *v;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
  const uint16_t *q_w, *k_w;  // bf16 [D] or null
  _Float16* q_out;            // [n][H][D]
  double eps;
  int32_t n, H;
  int64_t kv_items;           // workgroups of K and V before those of Q
  int32_t each;               // heads of Q a wave
  mi::RotaryPlan plan;
};

// x rounded once to f16, to the nearest or down (the conversion goes by way of f32 and
// rounds twice).
template <bool DOWN = false>
__device__ __forceinline__ _Float16 f64_to_f16(double x) {
  const int bits = 11 - max(__builtin_amdgcn_frexp_exp(x), -13);
  const double y = ldexp(x, bits);
  return (_Float16)(float)ldexp(DOWN ? floor(y) : rint(y), -bits);
}

struct Quant {
  uint32_t codes;  // four codes, one to a byte
  f16x2 so;        // scale, offset of the lane's group
};

// Codes of the lane's four columns z of a row, a group being 16 lanes whose least
// and largest values are lo and hi and which are all finite (`fine`).
__device__ __forceinline__ Quant quantise(const double (&z)[4], double lo, double hi, bool fine) {
  // (hi - lo) / 15, as a division rounds it: the second product makes up what the
  // reciprocal lacks
  const double range = hi - lo, q = range * (1.0 / 15.0);
  const double scale = (double)f64_to_f16(fma(fma(-15.0, q, range), 1.0 / 15.0, q));
  double offset = (double)f64_to_f16(lo - 16.0 * scale);
  // Code 15 stands for a value of f16: next to the end of its range the roundings of scale
  // and offset, which move it by less than 50, would put it past, an infinity from values
  // that are none.
  if (__any(hi > 64000.0)) {
    if (fma(31.0, scale, offset) >= 65520.0) offset = (double)f64_to_f16<true>(fma(-31.0, scale, 65504.0));
    fine = fine && hi < 65520.0;
  }
  const uint64_t ok = __ballot(fine) >> (threadIdx.x & 48);
  if ((ok & 0xffff) != 0xffff || !(fabs(offset) < __builtin_inf()) || !(scale < __builtin_inf())) {
    const _Float16 bad = (_Float16)__builtin_nanf("");
    return Quant{0, f16x2{bad, bad}};
  }
  // (z - offset) / scale rounded: by the reciprocal, which is off by less than 2^-40,
  // and where that could be the other side of a tie by the sign of what lies beyond it
  double inv = __builtin_amdgcn_rcp(scale);
  inv = fma(fma(-scale, inv, 1.0), inv, inv);
  inv = fma(fma(-scale, inv, 1.0), inv, inv);
  double c[4];
  double far = 0.0;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const double t = (z[e] - offset) * inv;
    c[e] = rint(t);
    far = fmax(far, fabs(t - c[e]));
  }
  if (__any(far > 0.5 - 0x1p-36)) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const double d = z[e] - offset, low = floor(d * inv), beyond = fma(-(low + 0.5), scale, d);
      if (fabs(beyond) < 0x1p-30 * scale)
        c[e] = beyond > 0.0 || (beyond == 0.0 && 0.5 * low != floor(0.5 * low)) ? low + 1.0 : low;
    }
  }
  Quant r;
  r.codes = 0;
#pragma unroll
  for (int e = 0; e < 4; e++)
    r.codes |= (uint32_t)min(max((int)c[e] - 16, 0), 15) << (8 * e);
  if (scale == 0.0) r.codes = 0;
  r.so = f16x2{(_Float16)(float)scale, (_Float16)(float)offset};
  return r;
}
template <typename T>
__device__ __forceinline__ Quant quantise(const T (&x)[4]) {
  T lo = fmin(fmin(x[0], x[1]), fmin(x[2], x[3])), hi = fmax(fmax(x[0], x[1]), fmax(x[2], x[3]));
  bool fine = true;
#pragma unroll
  for (int e = 0; e < 4; e++) fine = fine && __builtin_isfinite(x[e]);
  lo = mi::over_row(lo, [](T a, T b) { return fmin(a, b); });
  hi = mi::over_row(hi, [](T a, T b) { return fmax(a, b); });
  const double z[4] = {(double)x[0], (double)x[1], (double)x[2], (double)x[3]};
  return quantise(z, (double)lo, (double)hi, fine);
}

// Four bytes of codes as 16 bits of nibbles.
__device__ __forceinline__ uint32_t nibbles(uint32_t b) {
  b |= b >> 4;
  return (b & 0xff) | ((b >> 8) & 0xff00);
}

// Word index of a K row's columns 8 c .. 8 c + 7.
__device__ __forceinline__ int k_word(int row, int c) {
  const int sub = row >> 4, m = row & 15, g = c >> 3, quad = (c >> 1) & 3, step = c & 1;
  return ((2 * sub + (g >> 1)) * 64 + 16 * quad + m) * 4 + 2 * (g & 1) + step;
}

template <bool ILV>
__device__ __forceinline__ void finish_k(const AppendArgs& a, double (&z)[4], double pos, int lane) {
  mi::LaneTurn<double, ILV> t;
  t.set(a.plan, pos, lane);
  if (a.k_w) mi::rms_norm<double>(z, a.k_w, a.eps, lane);
  t.apply(a.plan, z, lane);
}

template <typename T>
__device__ __forceinline__ float4 load_row(const void* p, int64_t ts, int64_t hs, int64_t tok, int h,
                                           int lane) {
  return mi::load4((const T*)p + tok * ts + h * hs + 4 * lane);
}

// Sequence of token tok; its first token and count.
__device__ __forceinline__ int find_token(const mi::PagedView& pv, int tok, int& q0, int& nq) {
  int s = tok;
  if (pv.cu_q) {
    int lo = 0, hi = pv.batch;  // cu_q[lo] <= tok < cu_q[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pv.cu_q[mid] <= tok) lo = mid;
      else hi = mid;
    }
    s = lo;
  }
  pv.tokens(s, q0, nq);
  return s;
}

// EACH query heads of one token.
template <typename T, bool ILV, int EACH>
__device__ __forceinline__ void q_rows(const AppendArgs& a, int64_t item) {
  const int lane = threadIdx.x & 63;
  const int groups = (a.H + EACH - 1) / EACH;
  const int64_t tok = item / groups;
  if (tok >= a.n) return;
  const int h0 = (int)(item - tok * groups) * EACH;
  float4 x[EACH];
#pragma unroll
  for (int i = 0; i < EACH; i++) x[i] = load_row<T>(a.q, a.q_ts, a.q_hs, tok, min(h0 + i, a.H - 1), lane);
  int q0, nq;
  const int s = find_token(a.pv, (int)tok, q0, nq);
  if (s >= a.pv.batch || tok - q0 < 0 || tok - q0 >= nq) return;  // behind the last sequence
  const int pos = a.pv.kv_len[s] - nq + (int)(tok - q0);
  mi::LaneTurn<float, ILV> t;
  t.set(a.plan, (double)pos, lane);
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    if (h0 + i >= a.H) break;  // uniform
    float y[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    if (a.q_w) mi::rms_norm<float>(y, a.q_w, a.eps, lane);
    t.apply(a.plan, y, lane);
    mi::store4<EACH != 1>(a.q_out + (tok * a.H + h0 + i) * D + 4 * lane, y);
  }
}

// K (kv 0) or V (1) of the one row that sequence s brings.
template <typename T, bool ILV>
__device__ __forceinline__ void one_row(const AppendArgs& a, int64_t item) {
  const int lane = threadIdx.x & 63;
  const int kv = (int)(item & 1);
  const int sh = (int)(item >> 1), s = sh / a.pv.G, h = sh - s * a.pv.G;
  if (s >= a.pv.batch || s >= a.n) return;
  const float4 x = kv ? load_row<T>(a.v, a.v_ts, a.v_hs, s, h, lane)
                      : load_row<T>(a.k, a.k_ts, a.k_hs, s, h, lane);
  const int pos = a.pv.kv_len[s] - 1;
  if (pos < 0) return;  // an empty sequence
  uint8_t* tile = a.pv.tile(s, h, pos >> 5);
  if (!tile) return;
  const int row = pos & 31, g = lane >> 4;
  if (!kv) {
    double z[4] = {x.x, x.y, x.z, x.w};
    finish_k<ILV>(a, z, (double)pos, lane);
    const Quant r = quantise(z);
    const uint32_t half = nibbles(r.codes), other = __shfl_xor(half, 1, 64);
    if (!(lane & 1)) ((uint32_t*)tile)[k_word(row, lane >> 1)] = half | (other << 16);
    if (!(lane & 15)) ((f16x2*)(tile + mi::kKScale))[4 * row + g] = r.so;
  } else {
    const int sub = row >> 4, quad = (row >> 2) & 3, i = row & 3, p = 4 * (i + 4 * sub);
    u32x4* const w = (u32x4*)(tile + mi::kVCodes) + g * 64 + 16 * quad + (lane & 15);
    const u32x4 old = *w;
    const float y[4] = {x.x, x.y, x.z, x.w};
    const Quant r = quantise(y);
    u32x4 now;
#pragma unroll
    for (int j = 0; j < 4; j++)
      now[j] = (old[j] & ~(15u << p)) | (((r.codes >> (8 * j)) & 15u) << p);
    *w = now;
    if (!(lane & 15)) {
      _Float16* const so = (_Float16*)(tile + mi::kVScale) + (4 * g + quad) * 16 + 2 * i + sub;
      so[0] = r.so[0];
      so[8] = r.so[1];
    }
  }
}

template <typename T, bool ILV>
__global__ void __launch_bounds__(256) append_rows_kernel(const AppendArgs a) {
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t wg = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  if (wg < a.kv_items) one_row<T, ILV>(a, wg * 4 + w);
  else q_rows<T, ILV, 1>(a, (wg - a.kv_items) * 4 + w);
}

// The tile that item x of a call stands for: sequence s takes items from
// cu_q[s] / 32 + 2 s on, which leaves room for every tile its tokens can lie in
// (q / 32 + 2 at most).
struct TileItem {
  int s, q0, nq;
  int first;  // row of token q0; negative where the sequence is shorter than its tokens
  int end;    // rows of the sequence
  int local;  // tile of those that the tokens lie in
  int tile;
  __device__ __forceinline__ bool has_tile() const { return local >= 0 && (int64_t)tile * 32 < end; }
};
__device__ __forceinline__ bool find_tile(const mi::PagedView& pv, int32_t n, int64_t x, TileItem& it) {
  int lo = 0, hi = pv.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    const int64_t base = ((int64_t)(pv.cu_q ? pv.cu_q[mid] : mid) >> 5) + 2 * (int64_t)mid;
    if (base <= x) lo = mid;
    else hi = mid;
  }
  it.s = lo;
  pv.tokens(lo, it.q0, it.nq);
  if (it.nq <= 0 || it.q0 < 0 || (int64_t)it.q0 + it.nq > n) return false;
  it.end = max(pv.kv_len[lo], 0);
  it.first = it.end - it.nq;
  it.local = (int)(x - ((it.q0 >> 5) + 2 * (int64_t)lo));
  it.tile = it.local + (max(it.first, 0) >> 5);
  return true;
}

template <typename T, bool ILV>
__device__ void one_tile(const AppendArgs& a, int64_t item) {
  __shared__ u32x4 kw[256];
  __shared__ uint32_t vc[32][64];  // codes of V, one to a byte
  __shared__ f16x2 ks[32][4], vs[32][4];
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int64_t x = item / a.pv.G;
  const int h = (int)(item - x * a.pv.G);
  TileItem it;
  if (!find_tile(a.pv, a.n, x, it) || !it.has_tile()) return;
  uint8_t* const tile = a.pv.tile(it.s, h, it.tile);
  if (!tile) return;
  const int row0 = it.tile * 32;                  // row of the sequence at row 0 of the tile
  const int r0 = max(it.first - row0, 0);         // the call's rows of the tile: [r0, r1)
  const int r1 = min(it.end - row0, 32);
  constexpr int kEach = 32 / kTileWaves;  // rows of a wave
  float4 xk[kEach], xv[kEach];
#pragma unroll
  for (int i = 0; i < kEach; i++) {  // rows outside read the nearest inside
    const int r = min(max(kEach * w + i, r0), r1 - 1);
    const int64_t tok = it.q0 + (row0 + r - it.first);
    xk[i] = load_row<T>(a.k, a.k_ts, a.k_hs, tok, h, lane);
    xv[i] = load_row<T>(a.v, a.v_ts, a.v_hs, tok, h, lane);
  }
#pragma unroll
  for (int i = 0; i < kEach; i++) {
    const int r = kEach * w + i;
    if (r < r0 || r >= r1) continue;  // uniform
    double z[4] = {xk[i].x, xk[i].y, xk[i].z, xk[i].w};
    finish_k<ILV>(a, z, (double)(row0 + r), lane);
    const Quant k = quantise(z);
    const uint32_t half = nibbles(k.codes), other = __shfl_xor(half, 1, 64);
    if (!(lane & 1)) ((uint32_t*)kw)[k_word(r, lane >> 1)] = half | (other << 16);
    const float u[4] = {xv[i].x, xv[i].y, xv[i].z, xv[i].w};
    const Quant v = quantise(u);
    vc[r][lane] = v.codes;
    if (!(lane & 15)) {
      ks[r][lane >> 4] = k.so;
      vs[r][lane >> 4] = v.so;
    }
  }
  __syncthreads();
  auto mine = [&](int r) { return r >= r0 && r < r1; };
  if (t >= 256) return;
  if (mine(16 * (t >> 7) + (t & 15))) ((u32x4*)tile)[t] = kw[t];
  if (t < 32 && mine(t)) ((u32x4*)(tile + mi::kKScale))[t] = *(const u32x4*)&ks[t][0];
  {  // V word (g, quad, n, j): t = 64 g + 16 quad + n
    const int quad = (t >> 4) & 3, col = 16 * (t >> 6) + (t & 15);
    u32x4 now = {};
    uint32_t mask = 0;
#pragma unroll
    for (int p = 0; p < 8; p++) {
      const int r = 16 * (p >> 2) + 4 * quad + (p & 3);
      if (!mine(r)) continue;
      mask |= 15u << (4 * p);
      const uint32_t b = vc[r][col];
#pragma unroll
      for (int j = 0; j < 4; j++) now[j] |= ((b >> (8 * j)) & 15u) << (4 * p);
    }
    u32x4* const dst = (u32x4*)(tile + mi::kVCodes) + t;
    if (mask != 0xffffffffu) {
      const u32x4 old = *dst;
#pragma unroll
      for (int j = 0; j < 4; j++) now[j] |= old[j] & ~mask;
    }
    if (mask) *dst = now;
  }
  {  // V scales and offsets: half t of (g, quad, scale or offset, 2 i + sub)
    const int g = t >> 6, quad = (t >> 4) & 3, o = (t >> 3) & 1, i = (t >> 1) & 3, sub = t & 1;
    const int r = 16 * sub + 4 * quad + i;
    if (mine(r)) ((_Float16*)(tile + mi::kVScale))[t] = vs[r][g][o];
  }
}

template <typename T, bool ILV>
__global__ void __launch_bounds__(64 * kTileWaves) append_tiles_kernel(const AppendArgs a) {
  const int64_t wg = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (wg < a.kv_items) one_tile<T, ILV>(a, wg);
  else if (a.each == 1) q_rows<T, ILV, 1>(a, (wg - a.kv_items) * kTileWaves + w);
  else q_rows<T, ILV, mi::kRotaryHeads>(a, (wg - a.kv_items) * kTileWaves + w);
}

template <typename T>
hipError_t run_append(AppendArgs& a, hipStream_t s) {
  const bool rows = !a.pv.cu_q;
  a.kv_items = rows ? ((int64_t)a.pv.batch * a.pv.G * 2 + 3) / 4
                    : ((int64_t)(a.n >> 5) + 2 * a.pv.batch) * a.pv.G;
  const int waves = rows ? 4 : kTileWaves;
  a.each = rows ? 1 : mi::rotary_heads((int64_t)a.n * a.H);
  const int64_t q_items = a.q ? (int64_t)a.n * ((a.H + a.each - 1) / a.each) : 0;
  const int64_t wgs = a.kv_items + (q_items + waves - 1) / waves;
  const int64_t gx = std::min<int64_t>(wgs, 1 << 22);
  const auto f = rows ? (a.plan.interleaved ? append_rows_kernel<T, true> : append_rows_kernel<T, false>)
                      : (a.plan.interleaved ? append_tiles_kernel<T, true>
                                            : append_tiles_kernel<T, false>);
  return mi::launch("paged_append", f, dim3((unsigned)gx, (unsigned)((wgs + gx - 1) / gx)),
                    dim3(64 * waves), 0, s, a);
}

// ------------------------------------------------------------------- read --

struct ReadArgs {
  mi::PagedView pv;
  _Float16 *k, *v;  // [n][G][D]
  int32_t n;
};

// Rows of one tile of one sequence and KV head as f16: waves 0 and 1 take K, a
// thread eight words of rows 16 apart in steps of 4; waves 2 and 3 take V, a thread eight
// rows of eight columns.  Bound: memory (66,000 rows of two KV heads, 38 MB in and 135
// out, 31 us; the rows are stored past the caches, which they would only sweep: 42.2
// without, for the call alone; small calls take the same way).
__global__ void __launch_bounds__(256) paged_read_kernel(const ReadArgs a) {
  const int t = threadIdx.x;
  const int64_t item = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  const int64_t x = item / a.pv.G;
  const int h = (int)(item - x * a.pv.G);
  TileItem it;
  if (!find_tile(a.pv, a.n, x, it)) return;
  if (it.local == 0 && it.first < 0) {  // tokens whose row does not exist read as zero
    const int none = min(it.nq, -it.first);
    for (int i = t; i < none * 32; i += 256) {
      const int64_t o = (((int64_t)it.q0 + (i >> 5)) * a.pv.G + h) * D + 8 * (i & 31);
      *(f16x8*)(a.k + o) = f16x8{};
      *(f16x8*)(a.v + o) = f16x8{};
    }
  }
  if (!it.has_tile()) return;
  const uint8_t* const tile = a.pv.tile(it.s, h, it.tile);
  const int row0 = it.tile * 32;
  const int r0 = max(it.first - row0, 0), r1 = min(it.end - row0, 32);
  const int64_t tok0 = (int64_t)it.q0 + row0 - it.first;  // token of row 0
  auto out = [&](_Float16* p, int r, int c) {
    return (f16x8*)(p + ((tok0 + r) * a.pv.G + h) * D + 8 * c);
  };
  if (!tile) {  // no such page: the rows are not a number
    const _Float16 nan = (_Float16)__builtin_nanf("");
    const f16x8 bad = {nan, nan, nan, nan, nan, nan, nan, nan};
    for (int i = t; i < 32 * 32; i += 256)
      if ((i >> 5) >= r0 && (i >> 5) < r1) {
        *out(a.k, i >> 5, i & 31) = bad;
        *out(a.v, i >> 5, i & 31) = bad;
      }
    return;
  }
  const int c = t & 31;  // columns 8 c .. 8 c + 7
  const uint32_t x16 = mi::sixteens();
  if (t < 128) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int r = 4 * i + (t >> 5);
      const uint32_t wd = ((const uint32_t*)tile)[k_word(r, c)];
      const f16x2 so = ((const f16x2*)(tile + mi::kKScale))[4 * r + (c >> 3)];
      const f16x8 y = mi::dequant_row(wd, f16x2{so[0], so[0]}, f16x2{so[1], so[1]}, x16);
      if (r >= r0 && r < r1)
        __builtin_nontemporal_store(f16x8{y[0], y[2], y[4], y[6], y[1], y[3], y[5], y[7]}, out(a.k, r, c));
    }
  } else {
    const int quad = (t >> 5) & 3, g = c >> 3;
    const u32x4* const wp = (const u32x4*)(tile + mi::kVCodes) + g * 64 + 16 * quad + 2 * (c & 7);
    const u32x4 w0 = wp[0], w1 = wp[1];
    const f16x8* const sp = (const f16x8*)(tile + mi::kVScale) + 2 * (4 * g + quad);
    const f16x8 s = sp[0], o = sp[1];
    f16x8 col[8];  // column e of the eight rows, in dequant_col's order
#pragma unroll
    for (int e = 0; e < 8; e++) col[e] = mi::dequant_col(e < 4 ? w0[e] : w1[e - 4], s, o, x16);
#pragma unroll
    for (int p = 0; p < 8; p++) {  // element p: row 16 (p % 2) + 4 quad + p / 2
      const int r = 16 * (p & 1) + 4 * quad + (p >> 1);
      if (r >= r0 && r < r1)
        __builtin_nontemporal_store(f16x8{col[0][p], col[1][p], col[2][p], col[3][p], col[4][p], col[5][p],
                                          col[6][p], col[7][p]}, out(a.v, r, c));
    }
  }
}

}  // namespace

extern "C" mi_status mi_paged_append(
    void* pages, int64_t num_pages, int32_t page_rows, const int32_t* block_table,
    int32_t table_cols, const int32_t* kv_len, const int32_t* cu_q, int32_t batch, int32_t n,
    int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t type, const void* q,
    int64_t q_token_stride, int64_t q_head_stride, const void* k, int64_t k_token_stride,
    int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride,
    const uint16_t* q_norm_w, const uint16_t* k_norm_w, float eps, const double* host_freq,
    int32_t rotary_dim, int32_t interleaved, double factor, mi_f16* q_out, mi_stream stream) {
  mi::clear_error();
  AppendArgs a{};
  MI_TRY(mi::paged_view(pages, num_pages, page_rows, block_table, table_cols, kv_len, cu_q, batch,
                        num_kv_heads, head_dim, &a.pv));
  if (n <= 0 || (!cu_q && n != batch))
    return mi::fail(MI_ERR_INVALID_ARG, "n=%d batch=%d", n, batch);
  MI_TRY(mi::check_rows("k", k, type, k_token_stride, k_head_stride, num_kv_heads));
  MI_TRY(mi::check_rows("v", v, type, v_token_stride, v_head_stride, num_kv_heads));
  if (!(eps >= 0.f)) return mi::fail(MI_ERR_INVALID_ARG, "eps=%g", (double)eps);
  MI_TRY(mi::rotary_plan(host_freq, rotary_dim, interleaved, factor, &a.plan));
  if (q) {
    if (num_q_heads <= 0) return mi::fail(MI_ERR_INVALID_ARG, "num_q_heads=%d", num_q_heads);
    MI_TRY(mi::check_rows("q", q, type, q_token_stride, q_head_stride, num_q_heads));
    MI_TRY(mi::check_rows("q_out", q_out, MI_F16, (int64_t)num_q_heads * D, D, num_q_heads));
    const int64_t size = type == MI_F32 ? 4 : 2, out_bytes = (int64_t)n * num_q_heads * D * 2;
    const bool same = q == q_out && type == MI_F16 && q_head_stride == D &&
                      q_token_stride == (int64_t)num_q_heads * D;
    if ((!same && mi::overlaps(q, size * mi::rows_extent(n, num_q_heads, q_token_stride,
                                                         q_head_stride),
                               q_out, out_bytes)) ||
        mi::overlaps(k, size * mi::rows_extent(n, num_kv_heads, k_token_stride, k_head_stride),
                     q_out, out_bytes) ||
        mi::overlaps(v, size * mi::rows_extent(n, num_kv_heads, v_token_stride, v_head_stride),
                     q_out, out_bytes))
      return mi::fail(MI_ERR_INVALID_ARG, "q_out overlaps an input (it may only be q itself)");
  }
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_ts = q_token_stride;
  a.q_hs = q_head_stride;
  a.k_ts = k_token_stride;
  a.k_hs = k_head_stride;
  a.v_ts = v_token_stride;
  a.v_hs = v_head_stride;
  a.q_w = q_norm_w;
  a.k_w = k_norm_w;
  a.q_out = (_Float16*)q_out;
  a.eps = eps;
  a.n = n;
  a.H = num_q_heads;
  const hipStream_t s = (hipStream_t)stream;
  MI_HIP(type == MI_F32   ? run_append<float>(a, s)
         : type == MI_F16 ? run_append<_Float16>(a, s)
                          : run_append<mi::bf16>(a, s));
  return MI_OK;
}

extern "C" mi_status mi_paged_read(const void* pages, int64_t num_pages, int32_t page_rows,
                                   const int32_t* block_table, int32_t table_cols,
                                   const int32_t* kv_len, const int32_t* cu_q, int32_t batch,
                                   int32_t n, int32_t num_kv_heads, int32_t head_dim, mi_f16* k_out,
                                   mi_f16* v_out, mi_stream stream) {
  mi::clear_error();
  ReadArgs a{};
  MI_TRY(mi::paged_view((void*)pages, num_pages, page_rows, block_table, table_cols, kv_len, cu_q,
                        batch, num_kv_heads, head_dim, &a.pv));
  if (n <= 0 || (!cu_q && n != batch))
    return mi::fail(MI_ERR_INVALID_ARG, "n=%d batch=%d", n, batch);
  if (!k_out || !v_out || (((uintptr_t)k_out | (uintptr_t)v_out) & 15))
    return mi::fail(MI_ERR_INVALID_ARG, "k_out and v_out must be 16-byte aligned");
  const int64_t bytes = (int64_t)n * num_kv_heads * D * 2;
  if (mi::overlaps(k_out, bytes, v_out, bytes))
    return mi::fail(MI_ERR_INVALID_ARG, "k_out and v_out overlap");
  a.k = (_Float16*)k_out;
  a.v = (_Float16*)v_out;
  a.n = n;
  const int64_t wgs = ((int64_t)(n >> 5) + 2 * batch) * num_kv_heads;
  const int64_t gx = std::min<int64_t>(wgs, 1 << 22);
  MI_HIP(mi::launch("paged_read", paged_read_kernel,
                    dim3((unsigned)gx, (unsigned)((wgs + gx - 1) / gx)), dim3(256), 0,
                    (hipStream_t)stream, a));
  return MI_OK;
}
