// What the kernels of attention over packed documents share (doc_attn.hip, doc_attn_bwd.hip): element types, LDS tiles, the map from a
// workgroup to its rows, the masks, and the score.
//
// Rows: query head h = kvh * G + g reads key head kvh.  A document's queries x the G heads of one key head are ONE axis of "shared rows",
// row = i * G + g: a tile of shared rows reads its key blocks once for all G heads, and the tiles of a causal mask hug the diagonal.
#pragma once
#include "attn_frag.h"

namespace osud {

struct DocAttnP {
  const void *q, *k, *v, *o, *d_o;
  void *out, *dq, *dk, *dv;
  float* lse;     // [heads][rows_q], natural logarithm
  float* delta;   // [heads][rows_q]: sum_d d_out * out (backward)
  float* ws_o;    // forward split: [split][rows_q][heads][head_dim]; backward split: see doc_attn_bwd.hip
  float* ws_ml;   // forward split: [split][rows_q][heads][2] = maximum (log2 domain), sum
  size_t ld_q, ld_k, ld_v, ld_o, ld_do, ld_dq, ld_dk, ld_dv;  // elements between rows
  const int32_t *q_begin, *k_begin, *prefix;
  const float* slopes;
  // n_docs = n_real documents, and one more where the rows behind them are to be cleared: queries without keys, keys without queries
  int rows_q, rows_k, n_docs, n_real, heads, kv_heads, G, hd, left, right, slots, split, cus;
  float scale, c1 /* scale * log2(e) */, cap, c2 /* 2 scale log2(e) / cap */, cap2 /* cap * log2(e) */;
  float small;                // cap / 2 scale: up to this q.k the series serves
  float tanh1[5], tanh2[5];   // its coefficients for q.k -> tanh(scale q.k / cap), and that times cap2
};

constexpr float kLog2e = 1.4426950408889634f;
// logarithms of sums between the two bases, once per row: in 64 bits, one rounding (a relative error of 2^-24 of a logarithm of 10 is one of 6e-7 in
// every weight of the row)
__device__ __forceinline__ float doc_lse(float m, float l) { return l == 0.f ? -INFINITY : (float)(((double)m + (double)__builtin_amdgcn_logf(l)) * 0.6931471805599453094); }
__device__ __forceinline__ float doc_lse2(float lse) { return lse == -INFINITY ? INFINITY : (float)((double)lse * 1.4426950408889634074); }  // (no key seen: every p is 0)
// kShapeFixed (forward, bf16 and fp32, capped, no slopes, cap <= 60): scores lie within +- 87 binary orders, so 2^score, its sum over 2^30 keys and
// its products with v stay inside the types' ranges without a running maximum (cap 30, with the sum of the rounded weights that bf16 needs then: 2
// documents of 8191 positions, 12 / 4 heads of 128 columns, causal: 515 us, 528 with the maximum; 4 of 8192, 12 heads of 64: 1193, 1248)
enum { kShapeCap = 1, kShapeSlope = 2, kShapeFixed = 4 };
constexpr float kFixedCap = 60.0f;

// ---- element types: 16-byte operand fragments (8 halves or 4 floats per lane), one fragment pair = one contraction step
struct DocBf16 {
  typedef bf16_t E;
  static constexpr int ES = 2, STEP = 16 /* rows of a transposed fragment */, BK = 64 /* keys per block */;
  static constexpr bool kExact = false;
  static __device__ __forceinline__ f32x16 mma(const u32x4& a, const u32x4& b, f32x16 c) { return mfma_h<false>(a, b, c); }
  static __device__ __forceinline__ u32x4 pack(const f32x16& v, int s) { return pack8_h<false>(v, 8 * s); }
  static __device__ __forceinline__ u32x4 pack_rest(const f32x16& v, int s, const u32x4& hi) { return pack8_lo(v, 8 * s, hi); }  // what pack rounded away
  static __device__ __forceinline__ float sum(const u32x4& a, float r) {  // r + the eight elements, two per instruction
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; ++i) r = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf2, (uint32_t)a[i]), __builtin_bit_cast(bf2, 0x3f803f80u), r, false);
    return r;
  }
  static __device__ __forceinline__ float dot(const u32x4& a, const u32x4& b) {
    float r = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r = fmaf(__uint_as_float(a[i] << 16), __uint_as_float(b[i] << 16), r);
      r = fmaf(__uint_as_float(a[i] & 0xffff0000u), __uint_as_float(b[i] & 0xffff0000u), r);
    }
    return r;
  }
};
struct DocF16 {
  typedef f16_t E;
  static constexpr int ES = 2, STEP = 16, BK = 64;
  static constexpr bool kExact = false;
  static __device__ __forceinline__ f32x16 mma(const u32x4& a, const u32x4& b, f32x16 c) { return mfma_h<true>(a, b, c); }
  static __device__ __forceinline__ u32x4 pack(const f32x16& v, int s) { return pack8_h<true>(v, 8 * s); }
};
struct DocF32 {
  typedef float E;
  static constexpr int ES = 4, STEP = 8, BK = 32;
  static constexpr bool kExact = true;
  static __device__ __forceinline__ f32x16 mma(const u32x4& a, const u32x4& b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ u32x4 pack(const f32x16& v, int s) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(v[4 * s + i]);
    return r;
  }
  static __device__ __forceinline__ u32x4 pack_rest(const f32x16&, int, const u32x4& hi) { return hi; }
  static __device__ __forceinline__ float dot(const u32x4& a, const u32x4& b) {
    float r = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) r = fmaf(__uint_as_float(a[i]), __uint_as_float(b[i]), r);
    return r;
  }
};

// ---- LDS tiles: row-major rows of RB bytes, 16-byte chunks XOR-swizzled with the row so that both kinds of read spread over the 64
// banks: 16 rows of one chunk (rowfrag: 16 different 4-bank groups) and 4 rows x 64 bytes (one transposing read: 4 different 16-bank
// groups).  The LDS-DMA writes lanes one after the other, so the swizzle is applied to the source address.
template <typename T, int HDP> struct DocTile {
  static constexpr int RB = HDP * T::ES, CPR = RB / 16;
  static_assert(RB == 128 || RB == 192 || RB == 256 || RB == 384 || RB == 512, "tile rows of 64, 96 or 128 columns");
  static __device__ __forceinline__ int swz(int row) {
    if constexpr (RB == 128) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);  // (row & 1 is bank bit 5 already)
    else if constexpr (RB == 192) return (row >> 2) & 3;                         // (rows 0..3 start 48 banks apart; 12 chunks: XOR inside fours)
    else if constexpr (RB == 384) return (row >> 1) & 7;                         // (24 chunks: XOR inside eights)
    else return ((row & 3) << 2) | ((row >> 2) & 3);
  }
  static __device__ __forceinline__ int off(int row, int chunk) { return row * RB + ((chunk ^ swz(row)) << 4); }
  // The swizzle touches XB bits of the chunk, and row * RB has zeros there: the address of another chunk of the same row is an exclusive or of a
  // constant and an addition that goes into the instruction's offset.  LDS addresses, per lane; a tile starts at a multiple of 256 bytes.
  static constexpr int XB = RB == 192 ? 2 : (RB == 128 || RB == 384 ? 3 : 4), XM = (1 << XB) - 1;
  static __device__ __forceinline__ uint32_t at_chunk(uint32_t base, int c) { return (base ^ (uint32_t)((c & XM) << 4)) + (uint32_t)((c >> XB) << (4 + XB)); }
  // a row fragment = 16 bytes of row r0 + (lane & 31): contraction step ks, this lane's half of it
  static __device__ __forceinline__ uint32_t row_base(int lane) { return (uint32_t)off(lane & 31, lane >> 5); }
  static __device__ __forceinline__ u32x4 row_read(uint32_t base, int r0, int ks) {
    typedef const __attribute__((address_space(3))) u32x4 lds_v;
    return *(lds_v*)(size_t)(at_chunk(base, 2 * ks) + (uint32_t)(r0 * RB));
  }
  // a transposed fragment = contraction over the rows r0 .. r0 + STEP - 1 for column 32 dt + (lane & 31), in the order in which T::pack leaves
  // the score registers (16-bit types: two transposing reads of 4 rows x 16 columns per 16 lanes; fp32: four words)
  static __device__ __forceinline__ uint32_t tr_base(int lane) {
    if constexpr (T::ES == 2) {
      const int row = 4 * (lane >> 5) + ((lane & 15) >> 2), colb = 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
      return (uint32_t)(off(row, colb >> 4) + (colb & 15));
    } else {
      return (uint32_t)(4 * (lane >> 5) * RB);
    }
  }
  static __device__ __forceinline__ u32x4 tr_read(uint32_t base, int r0, int dt, int lane) {
    u32x4 v;
    if constexpr (T::ES == 2) {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      const uint32_t lo_at = at_chunk(base, 4 * dt), hi_at = at_chunk(base ^ 32u, 4 * dt);  // (rows + 8: bit 1 of the swizzled chunk)
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(size_t)(lo_at + (uint32_t)(r0 * RB)));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(size_t)(hi_at + (uint32_t)((r0 + 8) * RB)));
      const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
      v[0] = l2[0]; v[1] = l2[1]; v[2] = h2[0]; v[3] = h2[1];
    } else {
      typedef const __attribute__((address_space(3))) uint32_t lds_w;
      const int colb = (dt * 32 + (lane & 31)) * 4, row = 4 * (lane >> 5);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = *(lds_w*)(size_t)(base + (uint32_t)((r0 + i) * RB + (((colb >> 4) ^ swz(r0 + row + i)) << 4) + (colb & 15)));
    }
    return v;
  }
};

// ---- LDS-DMA of `rows` (a multiple of 4 per wave) tile rows by one workgroup of W waves: rows first + r, r >= 0, of a matrix with row stride
// ldb bytes; source rows past `last` read row `last` again (they are masked by index; the data stays finite where the document's is).
// Chunks behind the head's columns are not loaded: their LDS bytes were cleared once by clear_pads.
// A wave instruction moves 64 chunks = 1024 bytes; DocTile rows are whole numbers of chunks, so lane -> (row, chunk) is fixed per piece.
template <typename T, int HDP, int ROWS, int W> struct DocStage {
  using TL = DocTile<T, HDP>;
  static constexpr int BYTES = ROWS * TL::RB, PIECES = BYTES / 1024, PER = PIECES / W;
  static_assert(BYTES % 1024 == 0 && PIECES % W == 0, "whole pieces per wave");
  static __device__ __forceinline__ void row_chunk(int piece, int lane, int& row, int& chunk) {
    const int c = piece * 64 + lane;
    row = c / TL::CPR;
    chunk = (c - row * TL::CPR) ^ TL::swz(row);
  }
  // per-lane byte offsets of this wave's pieces from the tile's first row (whole tiles)
  static __device__ __forceinline__ void offsets(int wave, int lane, uint32_t ldb, uint32_t (&vo)[PER]) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      int row, chunk;
      row_chunk(wave * PER + i, lane, row, chunk);
      vo[i] = (uint32_t)row * ldb + (uint32_t)(chunk << 4);
    }
  }
  // (cols: chunks of a head's row that are data)
  static __device__ __forceinline__ void load(const char* first /* wave-uniform: the tile's first row, this head's columns */, int valid /* rows there are, >= 1 */,
                                              uint32_t ldb, int cols, uint32_t lds /* tile */, int wave, int lane, const uint32_t (&vo)[PER]) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int piece = wave * PER + i;
      int row, chunk;
      row_chunk(piece, lane, row, chunk);
      uint32_t off = vo[i];
      if (valid < ROWS) off = (uint32_t)(row < valid ? row : valid - 1) * ldb + (uint32_t)(chunk << 4);
      const uint32_t dst = lds + (uint32_t)piece * 1024u;
      if (cols == TL::CPR || chunk < cols)
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(first), "s"(dst) : "memory");
    }
  }
  // the same with the offsets worked out anew: nothing is held in registers between two calls
  static __device__ __forceinline__ void load_fresh(const char* first, int valid, uint32_t ldb, int cols, uint32_t lds, int wave, int lane) {
    asm volatile("" : "+v"(lane));
    uint32_t vo[PER];
    offsets(wave, lane, ldb, vo);
    load(first, valid, ldb, cols, lds, wave, lane, vo);
  }
  static __device__ __forceinline__ void clear_pads(char* tile, int cols, int tid, int threads) {
    if (cols == TL::CPR) return;
    for (int c = tid; c < ROWS * TL::CPR; c += threads) {
      const int row = c / TL::CPR, chunk = c - row * TL::CPR;
      if (chunk >= cols) *reinterpret_cast<uint4*>(tile + TL::off(row, chunk)) = make_uint4(0, 0, 0, 0);
    }
  }
};

// ---- a workgroup's document and rows.  Tile t of document d sits in slot floor(begin[d] * m / BM) + d + t (m shared rows per query): distinct for
// every tile without a table, at most one unused slot per document.  64 documents are looked at per step.
struct DocRange {
  int q0, nq, k0, nk, pre;  // first query / key row, how many, length of the prefix
};
__device__ __forceinline__ int doc_clamp(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }
template <int bm> __device__ __forceinline__ int doc_find(const int32_t* begin, int n_docs, int rows, int m, int slot, int lane, int& tile) {
  auto start = [&](int d) { return (int)((unsigned)(doc_clamp(begin[d], 0, rows) * m) / (unsigned)bm) + d; };  // (rows * m < 2^31)
  int lo = 0, len = n_docs;
  while (len > 1) {
    const int step = (len + 63) >> 6, i = lane * step;
    int n = __popcll(__ballot(i < len && start(lo + (i < len ? i : 0)) <= slot));
    n = n < 1 ? 1 : n;
    const int skip = (n - 1) * step;
    lo += skip;
    len = len - skip < step ? len - skip : step;
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  tile = __builtin_amdgcn_readfirstlane(slot - start(lo));
  return lo;
}
// (offsets that are not in order or out of range give wrong results for their documents and nothing else: every row stays inside the tensors)
__device__ __forceinline__ DocRange doc_range(const DocAttnP& p, int d, bool query_side) {
  DocRange r;
  r.q0 = doc_clamp(p.q_begin[d], 0, p.rows_q);
  r.k0 = doc_clamp(p.k_begin[d], 0, p.rows_k);
  r.pre = 0;
  if (d == p.n_real) {  // the rows behind the last document
    r.nq = query_side ? p.rows_q - r.q0 : 0;
    r.nk = query_side ? 0 : p.rows_k - r.k0;
    return r;
  }
  r.nq = doc_clamp(p.q_begin[d + 1], r.q0, p.rows_q) - r.q0;
  r.nk = doc_clamp(p.k_begin[d + 1], r.k0, p.rows_k) - r.k0;
  if (p.prefix != nullptr) r.pre = doc_clamp(p.prefix[d], 0, r.nk);
  return r;
}
// max / sum over lane and lane ^ 32 (v_permlane32_swap: the halves of two registers change places)
__device__ __forceinline__ float doc_half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float doc_half_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Workgroup b's unit: parts of a split fastest, then key heads, then slots, from the last one (`down`) or the first: each document's longest
// tiles under a causal mask come first (the last of its query tiles, the first of its key tiles), so that a launch ends on short ones.
// Consecutive workgroups sit on consecutive XCDs, so the tiles of a key head stay on the XCDs of its remainder mod 8 and read its keys
// through their L2s.  (One contiguous eighth of the units per XCD reads each key head through one L2, but where a document's tiles
// straddle two eighths the later one ends on the longest tile: 2 documents of 8191 positions, 12 / 4 heads of 128 columns, causal: 605 us, in this order 443.)
struct DocUnit {
  int part, kvh, slot;
};
__device__ __forceinline__ DocUnit doc_unit(const DocAttnP& p, bool down) {
  DocUnit u;
  int b = blockIdx.x;
  u.part = 0;
  if (p.split > 1) {
    u.part = b % p.split;
    b /= p.split;
  }
  const int s = b / p.kv_heads;
  u.kvh = b - s * p.kv_heads;
  u.slot = down ? p.slots - 1 - s : s;
  return u;
}

// ---- masks: key j is visible to position i if j < pre or i - left <= j <= i + right (a negative bound: none)
struct DocBand {
  int lo, hi;
};
__device__ __forceinline__ DocBand doc_band(const DocAttnP& p, int pos, int nk) {  // keys [lo, hi] of one position; hi < lo: none
  DocBand b;
  b.lo = p.left < 0 || pos - p.left < 0 ? 0 : pos - p.left;
  b.hi = p.right < 0 || pos + p.right > nk - 1 ? nk - 1 : pos + p.right;
  return b;
}
// the same as a start and a length, so that one comparison of unsigned numbers asks for both ends (nothing visible: a start that no key reaches)
struct DocSpan {
  int lo;
  unsigned len;
};
__device__ __forceinline__ DocSpan doc_span(int lo, int hi) { return hi < lo ? DocSpan{1 << 30, 0u} : DocSpan{lo, (unsigned)(hi - lo)}; }
// s[r] of the keys key0 + 8 (r / 4) + r % 4 outside of the span and behind the prefix becomes `none`.  APART: documents without a prefix have a way of
// their own.  (What it is worth is the compiler's registers: without caps one way keeps four waves per SIMD at 64 columns, 32 documents of 1024
// positions 130 us against 142; under a cap it takes scalar registers that are not there, 8 documents of 4096 390 us against 350.)
template <bool APART> __device__ __forceinline__ void doc_mask(f32x16& s, int key0, DocSpan span, int pre, float none) {
  const int rel = key0 - span.lo;
  if (APART && pre == 0) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = (unsigned)(rel + 8 * (r >> 2) + (r & 3)) <= span.len ? s[r] : none;
    return;
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int off = 8 * (r >> 2) + (r & 3);
    const bool seen = (key0 + off < pre) | ((unsigned)(rel + off) <= span.len);
    s[r] = seen ? s[r] : none;
  }
}
// 0: no pair of the positions [i0, i1] and the keys [j0, j1] (cut off at nk) is visible; 2: every one is, and j1 < nk; 1: some
__device__ __forceinline__ int doc_class(const DocAttnP& p, int i0, int i1, int j0, int j1, int nk, int pre) {
  if (j0 >= nk) return 0;
  const bool before = p.left >= 0 && j1 < i0 - p.left, behind = p.right >= 0 && j0 > i1 + p.right;
  if (j0 >= pre && (before || behind)) return 0;
  const bool band = (p.left < 0 || j0 >= i1 - p.left) && (p.right < 0 || j1 <= i0 + p.right);
  return j1 < nk && (band || j1 < pre) ? 2 : 1;
}

// ---- capped scores.  tanh(x) = 1 - 2 / (1 + e^(2x)) takes two transcendental instructions (16 cycles each; a multiply-add 4).  Where no score of a
// wave's tile passes half the cap -- the rule outside of outliers -- an odd polynomial of x does: relative error 5.4e-7 with four terms
// (1.3e-8 with the fifth, for the fp32 tier), a least-maximum fit of tanh(x) / x in x^2 over |x| <= 1/2.  2 documents of 8191 positions, 12 / 4
// heads of 128 columns, causal: the polynomial takes 44 us less of 542.
template <typename T> __device__ __forceinline__ float doc_tanh_series(const float (&t)[5], float s) {
  const float y = s * s;
  if constexpr (T::kExact) return s * fmaf(y, fmaf(y, fmaf(y, fmaf(y, t[4], t[3]), t[2]), t[1]), t[0]);
  else return s * fmaf(y, fmaf(y, fmaf(y, t[3], t[2]), t[1]), t[0]);
}
// s[0 .. 15] (q.k) -> gain * tanh(scale s / cap); t = the series for that gain.  `small`: no |s| of the wave passes p.small
template <typename T> __device__ __forceinline__ void doc_tanh(const DocAttnP& p, const float (&t)[5], float gain, bool small, f32x16& s) {
  if (small) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = doc_tanh_series<T>(t, s[r]);
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float e = fmaf(-2.0f * gain, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(s[r] * p.c2)), gain);
      // (fp32 tier: below half the cap that form loses relative accuracy)
      s[r] = T::kExact && fabsf(s[r]) <= p.small ? doc_tanh_series<T>(t, s[r]) : e;
    }
  }
}
__device__ __forceinline__ float doc_largest(const f32x16& s, float m) {
#pragma unroll
  for (int r = 0; r < 16; ++r) m = fmaxf(m, fabsf(s[r]));
  return m;
}

template <typename T> __device__ __forceinline__ void doc_store4(char* p, const f32x16& v, int g, float f) {  // registers 4 g .. 4 g + 3, times f
  if constexpr (T::ES == 4) *reinterpret_cast<float4*>(p) = make_float4(v[4 * g] * f, v[4 * g + 1] * f, v[4 * g + 2] * f, v[4 * g + 3] * f);
  else store4(reinterpret_cast<typename T::E*>(p), v[4 * g] * f, v[4 * g + 1] * f, v[4 * g + 2] * f, v[4 * g + 3] * f);
}
// 32 accumulator columns of a wave (lane & 31 = row of the result, d = 32 dt + 8 g + 4 half + i) -> rows of the result through a patch of LDS,
// stored as whole 16-byte chunks, neighbouring lanes on neighbouring chunks.  row(r) = address of result row r, nullptr: not stored.
template <typename T, int HDP, typename ROW>
__device__ __forceinline__ void doc_store_rows(char* patch, const f32x16 (&acc)[HDP / 32], float f, int hd, int lane, ROW row) {
  using TL = DocTile<T, HDP>;
  const int fr = lane & 31, half = lane >> 5;
#pragma unroll
  for (int dt = 0; dt < HDP / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int b = (dt * 32 + 8 * g + 4 * half) * T::ES;
      doc_store4<T>(patch + TL::off(fr, b >> 4) + (b & 15), acc[dt], g, f);
    }
  asm volatile("" ::: "memory");  // (the LDS operations of a wave execute in order)
  const int cols = hd * T::ES / 16;
#pragma unroll
  for (int it = 0; it < TL::CPR / 2; ++it) {
    const int c = it * 64 + lane, r = c / TL::CPR, chunk = c - r * TL::CPR;
    char* dst = row(r);
    if (dst != nullptr && chunk < cols) *reinterpret_cast<u32x4*>(dst + chunk * 16) = *reinterpret_cast<const u32x4*>(patch + TL::off(r, chunk));
  }
  asm volatile("" ::: "memory");
}

size_t doc_attn_ws(const DocAttnP& p, int prec, int max_k);   // floats of the forward's workspace (0: no split)
size_t doc_attn_bwd_ws(const DocAttnP& p, int prec, int max_q);  // floats of the backward's: delta, lse2, parts of a split
int launch_doc_attn(int prec, DocAttnP& p, int max_k, size_t ws_floats, hipStream_t st);
int launch_doc_attn_bwd(int prec, DocAttnP& p, int max_q, size_t ws_floats, hipStream_t st);

}  // namespace osud
