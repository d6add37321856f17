// Attention over packed documents, backward.  With p = exp(s - lse), dp = d_out . v, delta = sum_d d_out out (= sum_j p dp):
//   ds = p (dp - delta) (1 - tanh^2 where capped);  dq = scale ds k;  dk = scale ds^T q;  dv = p^T d_out;  dk, dv summed over the shared heads.
// (Reference: autograd of nn.MultiheadAttention, train.py:257.)
//
// Two kernels, each recomputing s and dp: the first owns query rows and walks key blocks (dq; it also writes delta and lse * log2(e) for the
// second), the second owns keys and walks query blocks (dk, dv).  Seven products instead of the five of a single pass, but every sum
// is taken in a fixed order: no atomics, two runs give the same bits.
//
// Rounding: p and ds go into p^T d_out and ds^T q in the element type (at most 2^-8 of each in bf16, the size of the results' own rounding).  The
// delta that the forward's rounded out gives carries that rounding once more, so the first kernel sums p dp on its way and the second uses
// that; its own product ds k takes ds as two parts, the element type and what that rounded away, to keep the sum of both errors where
// the other gradients' is (8192 positions with distance penalties, error of dq against 64 bits: 2.3e-3, 2.8e-3 with one part; one rounding: 1.7e-3).
//
// Bound: matrix pipe (48 % busy in the first kernel) and the waits for LDS fragments.  8192 positions, 8 / 2 heads of 128 columns, causal: 336 us the first
// kernel, 320 the second, 20 the join of its parts; 32 documents of 1024 positions, 12 heads of 64: 465 us both.
#include "doc_attn.h"
#include "kernels.h"

namespace osud {
namespace {

// s[0 .. 15] (q.k) -> p = exp(score - lse); capped: dsc = 1 - tanh^2.  dist(r), lse2(r): position - key, lse * log2(e) of element r
template <typename T, int SHAPE, typename DIST, typename LSE>
__device__ __forceinline__ void doc_weights(const DocAttnP& p, f32x16& s, float (&dsc)[16], float slope2, DIST dist, LSE lse2) {
  constexpr bool kCap = (SHAPE & kShapeCap) != 0, kSlope = (SHAPE & kShapeSlope) != 0;
  if constexpr (kCap) {
    const bool small = !__any(doc_largest(s, 0.f) > p.small);
    doc_tanh<T>(p, p.tanh1, 1.0f, small, s);
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    dsc[r] = kCap ? fmaf(-s[r], s[r], 1.0f) : 1.0f;
    float v = fmaf(s[r], kCap ? p.cap2 : p.c1, -lse2(r));
    if constexpr (kSlope) v = fmaf(-slope2, fabsf(dist(r)), v);
    s[r] = __builtin_amdgcn_exp2f(v);
  }
}
template <int SHAPE> __device__ __forceinline__ float doc_ds(float prob, float dp, float delta, float dsc) {
  const float ds = prob * (dp - delta);
  return (SHAPE & kShapeCap) != 0 ? ds * dsc : ds;
}

template <typename T, int HDP, int KS, int SHAPE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(T::ES == 2 ? (HDP == 64 && (SHAPE & kShapeCap) == 0 ? 3 : 2) : (HDP == 128 ? 1 : 2)))) void doc_attn_dq_kernel(DocAttnP p) {
  using TL = DocTile<T, HDP>;
  constexpr int BK = T::BK, KT = BK / 32, DT = HDP / 32;
  using ST = DocStage<T, HDP, BK, 4>;
  constexpr int TILE = ST::BYTES, STAGE = 2 * TILE;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const uint32_t lds0 = (uint32_t)(size_t)(const __attribute__((address_space(3))) void*)smem;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int frow = lane & 31, half = lane >> 5;

  const DocUnit u = doc_unit(p, true);
  const int kvh = u.kvh;
  int tile;
  const DocRange d = doc_range(p, doc_find<128>(p.q_begin, p.n_docs, p.rows_q, p.G, u.slot, lane, tile), true);
  const int vrows = d.nq * p.G, row0 = tile * 128;
  if (tile < 0 || row0 >= vrows) return;
  const int vr = row0 + wave * 32 + frow;
  const int vrc = vr < vrows ? vr : vrows - 1;
  const int qi = (int)((unsigned)vrc / (unsigned)p.G), head = kvh * p.G + vrc - qi * p.G;
  const int shift = d.nk - d.nq, pos = shift + qi;
  const size_t qrow = (size_t)d.q0 + qi;
  auto pos_of = [&](int r) { return shift + (int)((unsigned)(r < vrows ? r : vrows - 1) / (unsigned)p.G); };
  const int wg0 = pos_of(row0), wg1 = pos_of(row0 + 127);
  const int wv0 = __builtin_amdgcn_readlane(pos, 0), wv1 = __builtin_amdgcn_readlane(pos, 31);
  const bool alive = row0 + wave * 32 < vrows;

  const int npre = (d.pre + BK - 1) / BK;
  int bl = doc_band(p, wg0, d.nk).lo / BK;
  const int hi = doc_band(p, wg1, d.nk).hi;
  if (bl < npre) bl = npre;
  const int nblk = npre + (hi < 0 || hi / BK < bl ? 0 : hi / BK - bl + 1);

  const int cols = p.hd * T::ES / 16;
  const uint32_t ldkb = (uint32_t)(p.ld_k * T::ES), ldvb = (uint32_t)(p.ld_v * T::ES);
  const char* const kbase = reinterpret_cast<const char*>(p.k) + ((size_t)d.k0 * p.ld_k + (size_t)kvh * p.hd) * T::ES;
  const char* const vbase = reinterpret_cast<const char*>(p.v) + ((size_t)d.k0 * p.ld_v + (size_t)kvh * p.hd) * T::ES;
  uint32_t vok[ST::PER], vov[ST::PER];
  ST::offsets(wave, lane, ldkb, vok);
  ST::offsets(wave, lane, ldvb, vov);
  auto block_of = [&](int i) { return i < npre ? i : i - npre + bl; };
  auto issue = [&](int i, int stage) {
    const int j0 = block_of(i) * BK;
    ST::load(kbase + (size_t)j0 * ldkb, d.nk - j0, ldkb, cols, lds0 + stage * STAGE, wave, lane, vok);
    ST::load(vbase + (size_t)j0 * ldvb, d.nk - j0, ldvb, cols, lds0 + stage * STAGE + TILE, wave, lane, vov);
  };
  for (int i = 0; i < 4; ++i) ST::clear_pads(smem + i * TILE, cols, tid, 256);
  if (nblk > 0) issue(0, 0);

  u32x4 qf[KS], gf[KS];
  float delta = 0.f;
  {
    const size_t col = (size_t)head * p.hd;
    const char* qp = reinterpret_cast<const char*>(p.q) + (qrow * p.ld_q + col) * T::ES;
    const char* gp = reinterpret_cast<const char*>(p.d_o) + (qrow * p.ld_do + col) * T::ES;
    const char* op = reinterpret_cast<const char*>(p.o) + (qrow * p.ld_o + col) * T::ES;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[ks] = gf[ks] = u32x4{0u, 0u, 0u, 0u};
      const int c = 2 * ks + half;
      if (c < cols) {
        qf[ks] = *reinterpret_cast<const u32x4*>(qp + c * 16);
        gf[ks] = *reinterpret_cast<const u32x4*>(gp + c * 16);
        delta += T::dot(gf[ks], *reinterpret_cast<const u32x4*>(op + c * 16));
      }
    }
  }
  delta = doc_half_sum(delta);
  const size_t at = (size_t)head * p.rows_q + qrow, n_at = (size_t)p.heads * p.rows_q;
  const float lse2 = doc_lse2(p.lse[at]);
  float slope2 = 0.f;
  if constexpr ((SHAPE & kShapeSlope) != 0) slope2 = p.slopes[head] * kLog2e;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[ks]), "+v"(gf[ks]));  // (waited for here, not inside the loop, where it would drain the DMA)

  const DocBand band = doc_band(p, pos, d.nk);
  const DocSpan span = doc_span(band.lo, band.hi);
  f32x16 dq[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[i][r] = 0.f;
  float exact = 0.f;  // sum_j p dp
  const uint32_t kb = lds0 + TL::row_base(lane), tb = lds0 + TL::tr_base(lane);
  for (int it = 0; it < nblk; ++it) {
    const int stage = it & 1;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (it + 1 < nblk) issue(it + 1, stage ^ 1);
    const int j0 = block_of(it) * BK;
    const uint32_t ka = kb + stage * STAGE, va = ka + TILE, ta = tb + stage * STAGE;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const int cls = alive ? doc_class(p, wv0, wv1, j0 + kt * 32, j0 + kt * 32 + 31, d.nk, d.pre) : 0;
      if (cls == 0) continue;
      f32x16 s, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s = T::mma(TL::row_read(ka, kt * 32, ks), qf[ks], s);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) dp = T::mma(TL::row_read(va, kt * 32, ks), gf[ks], dp);
      const int key_lane = j0 + kt * 32 + 4 * half;
      const float dist0 = (float)(pos - key_lane);
      float dsc[16];
      doc_weights<T, SHAPE>(p, s, dsc, slope2, [&](int r) { return dist0 - (float)(8 * (r >> 2) + (r & 3)); }, [&](int) { return lse2; });
      if (cls == 1) doc_mask<(SHAPE & kShapeCap) != 0>(s, key_lane, span, d.pre, 0.f);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        exact = fmaf(s[r], dp[r], exact);
        s[r] = doc_ds<SHAPE>(s[r], dp[r], delta, dsc[r]);
      }
#pragma unroll
      for (int ss = 0; ss < 32 / T::STEP; ++ss) {
        const u32x4 f = T::pack(s, ss), lo = T::pack_rest(s, ss, f);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const u32x4 kf = TL::tr_read(ta, kt * 32 + T::STEP * ss, dt, lane);
          dq[dt] = T::mma(kf, f, dq[dt]);
          if constexpr (!T::kExact) dq[dt] = T::mma(kf, lo, dq[dt]);
        }
      }
    }
  }
  exact = doc_half_sum(exact);
  if (half == 0 && vr < vrows) {
    p.delta[at] = exact;
    p.delta[n_at + at] = lse2;
  }
  __syncthreads();
  if (!alive) return;
  doc_store_rows<T, HDP>(smem + wave * 32 * TL::RB, dq, p.scale, p.hd, lane, [&](int r) -> char* {
    const int v = row0 + wave * 32 + r;
    if (v >= vrows) return nullptr;
    const int i = (int)((unsigned)v / (unsigned)p.G);
    return reinterpret_cast<char*>(p.dq) + (((size_t)d.q0 + i) * p.ld_dq + (size_t)(kvh * p.G + v - i * p.G) * p.hd) * T::ES;
  });
}

// 128 columns of 16-bit elements: dk, dv and the fragments of k and v are 192 registers, one wave per SIMD.  v's fragments stay in LDS then and the
// query blocks are halved to make room: two workgroups per CU (8192 positions, 8 / 2 heads, causal: 343 us; 486 with one wave per SIMD).  64
// columns: three instead of two (256 ragged windows, backward 196 us instead of 209; capped and sloped scores need the registers: 1268 instead of 1232).
template <typename T, int HDP, int SHAPE> constexpr bool doc_v_in_lds = T::ES == 2 && (HDP == 128 || (HDP == 64 && SHAPE == 0));
template <typename T, int HDP> constexpr int doc_bq = HDP == 128 && T::ES == 2 ? 32 : T::BK;

// One workgroup = 128 keys of one document and key head (a wave owns 32: lane = key); the shared heads one after the other, for each the
// query blocks that see the keys.  With a split (few key tiles), part `sp` takes its share of the (head, block) list and leaves fp32 sums.
template <typename T, int HDP, int KS, int SHAPE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(T::ES == 4 ? 1 : HDP == 64 && SHAPE == 0 ? 3 : 2))) void doc_attn_dkv_kernel(DocAttnP p) {
  using TL = DocTile<T, HDP>;
  constexpr bool VL = doc_v_in_lds<T, HDP, SHAPE>;
  constexpr int BQ = doc_bq<T, HDP>, QT = BQ / 32, DT = HDP / 32;
  using ST = DocStage<T, HDP, BQ, 4>;
  constexpr int TILE = ST::BYTES, STAGE = 2 * TILE + 2 * BQ * 4;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const uint32_t lds0 = (uint32_t)(size_t)(const __attribute__((address_space(3))) void*)smem;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int frow = lane & 31, half = lane >> 5;

  const DocUnit u = doc_unit(p, false);
  const int sp = u.part, kvh = u.kvh;
  int tile;
  const DocRange d = doc_range(p, doc_find<128>(p.k_begin, p.n_docs, p.rows_k, 1, u.slot, lane, tile), false);
  const int j0 = tile * 128;
  if (tile < 0 || j0 >= d.nk) return;
  const int jw = j0 + wave * 32;  // this wave's first key
  const bool alive = jw < d.nk;
  const int key = jw + frow, keyc = key < d.nk ? key : d.nk - 1;
  const int shift = d.nk - d.nq;

  // queries that may see a key of the tile
  int i_lo = 0, i_hi = d.nq - 1;
  if (j0 >= d.pre) {
    const int j1 = j0 + 127 < d.nk ? j0 + 127 : d.nk - 1;
    if (p.right >= 0 && j0 - p.right - shift > i_lo) i_lo = j0 - p.right - shift;
    if (p.left >= 0 && j1 + p.left - shift < i_hi) i_hi = j1 + p.left - shift;
  }
  const int b0 = i_lo / BQ, nb = i_hi < i_lo ? 0 : i_hi / BQ - b0 + 1;
  const int total = nb * p.G;
  int it = p.split > 1 ? (int)((long)sp * total / p.split) : 0;
  const int it_end = p.split > 1 ? (int)((long)(sp + 1) * total / p.split) : total;

  const int cols = p.hd * T::ES / 16;
  const uint32_t ldqb = (uint32_t)(p.ld_q * T::ES), ldgb = (uint32_t)(p.ld_do * T::ES);
  uint32_t voq[VL ? 1 : ST::PER], vog[VL ? 1 : ST::PER];
  if constexpr (!VL) {
    ST::offsets(wave, lane, ldqb, voq);
    ST::offsets(wave, lane, ldgb, vog);
  }
  const size_t n_at = (size_t)p.heads * p.rows_q;
  // (head of the group, query block) of a part's turns, one after the other
  struct Turn {
    int g, b;
  };
  auto turn_of = [&](int i) { return Turn{nb > 0 ? i / nb : 0, nb > 0 ? i % nb : 0}; };
  auto after = [&](Turn t) { return t.b + 1 < nb ? Turn{t.g, t.b + 1} : Turn{t.g + 1, 0}; };
  auto issue = [&](Turn t, int stage) {
    const int i0 = (b0 + t.b) * BQ, head = kvh * p.G + t.g;
    const size_t row = (size_t)d.q0 + i0;
    const uint32_t lds = lds0 + stage * STAGE;
    const char* const qp = reinterpret_cast<const char*>(p.q) + (row * p.ld_q + (size_t)head * p.hd) * T::ES;
    const char* const gp = reinterpret_cast<const char*>(p.d_o) + (row * p.ld_do + (size_t)head * p.hd) * T::ES;
    if constexpr (VL) {
      ST::load_fresh(qp, d.nq - i0, ldqb, cols, lds, wave, lane);
      ST::load_fresh(gp, d.nq - i0, ldgb, cols, lds + TILE, wave, lane);
    } else {
      ST::load(qp, d.nq - i0, ldqb, cols, lds, wave, lane, voq);
      ST::load(gp, d.nq - i0, ldgb, cols, lds + TILE, wave, lane, vog);
    }
    if (wave < 2 && lane < BQ) {  // wave 0: delta, wave 1: lse2 of the block's rows
      const float* src = p.delta + (wave == 1 ? n_at : 0) + (size_t)head * p.rows_q + row;
      const uint32_t off = (uint32_t)(i0 + lane < d.nq ? lane : d.nq - 1 - i0) * 4u;
      asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" : : "v"(off), "s"(src), "s"(lds + 2 * TILE + wave * BQ * 4) : "memory");
    }
  };
  for (int i = 0; i < 2; ++i) {
    ST::clear_pads(smem + i * STAGE, cols, tid, 256);
    ST::clear_pads(smem + i * STAGE + TILE, cols, tid, 256);
  }
  const uint32_t ldvb = (uint32_t)(p.ld_v * T::ES);
  if constexpr (VL) {
    using SV = DocStage<T, HDP, 128, 4>;
    SV::clear_pads(smem + 2 * STAGE, cols, tid, 256);
    SV::load_fresh(reinterpret_cast<const char*>(p.v) + (((size_t)d.k0 + j0) * p.ld_v + (size_t)kvh * p.hd) * T::ES, d.nk - j0, ldvb, cols, lds0 + 2 * STAGE, wave, lane);
  }
  Turn now = turn_of(it), next = now;
  if (it < it_end) issue(now, 0);

  u32x4 kf[KS], vf[VL ? 1 : KS];
  {
    const char* kp = reinterpret_cast<const char*>(p.k) + (((size_t)d.k0 + keyc) * p.ld_k + (size_t)kvh * p.hd) * T::ES;
    const char* vp = reinterpret_cast<const char*>(p.v) + (((size_t)d.k0 + keyc) * p.ld_v + (size_t)kvh * p.hd) * T::ES;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int c = 2 * ks + half;
      kf[ks] = u32x4{0u, 0u, 0u, 0u};
      if (c < cols) kf[ks] = *reinterpret_cast<const u32x4*>(kp + c * 16);
      if constexpr (!VL) {
        vf[ks] = u32x4{0u, 0u, 0u, 0u};
        if (c < cols) vf[ks] = *reinterpret_cast<const u32x4*>(vp + c * 16);
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    asm volatile("" : "+v"(kf[ks]));
    if constexpr (!VL) asm volatile("" : "+v"(vf[ks]));
  }

  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[i][r] = dv[i][r] = 0.f;
  if (!alive) {  // (a wave behind the last key only fetches)
    for (int stage = 1; it < it_end; ++it, stage ^= 1) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      now = after(now);
      if (it + 1 < it_end) issue(now, stage);
    }
    __syncthreads();
    return;
  }
  const uint32_t qb = lds0 + TL::row_base(lane), tb = lds0 + TL::tr_base(lane);
  [[maybe_unused]] const uint32_t vb = qb + 2 * STAGE + wave * 32 * TL::RB;
  // queries that see this lane's key
  DocSpan span;
  {
    int lo = 0, hi = d.nq - 1;
    if (key >= d.pre) {
      if (p.right >= 0 && key - p.right - shift > lo) lo = key - p.right - shift;
      if (p.left >= 0 && key + p.left - shift < hi) hi = key + p.left - shift;
    }
    span = doc_span(lo, key < d.nk ? hi : -1);
  }
  int stage = 0;
  for (; it < it_end; ++it) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    next = after(now);
    if (it + 1 < it_end) issue(next, stage ^ 1);
    const int g = now.g, i0 = (b0 + now.b) * BQ;
    now = next;
    float slope2 = 0.f;
    if constexpr ((SHAPE & kShapeSlope) != 0) slope2 = p.slopes[kvh * p.G + g] * kLog2e;
    const uint32_t qa = qb + stage * STAGE, ga = qa + TILE, tq = tb + stage * STAGE, tg = tq + TILE;
    const float* rows = reinterpret_cast<const float*>(smem + stage * STAGE + 2 * TILE);  // delta [BQ], lse2 [BQ]
    stage ^= 1;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int i = i0 + qt * 32;  // this sub-block's first query
      int cls = doc_class(p, shift + i, shift + (i + 31 < d.nq ? i + 31 : d.nq - 1), jw, jw + 31, d.nk, d.pre);
      if constexpr (!VL) {  // (VL: no way round the products of a sub-block that sees nothing, the branch would cost registers)
        if (i >= d.nq || cls == 0) continue;
      }
      if (i + 31 >= d.nq) cls = 1;
      f32x16 s, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.f;
      if constexpr (VL) {  // one step's fragments ahead of the products and no more: 256 registers hold (left to itself the compiler fetches all and spills k)
        u32x4 qn = TL::row_read(qa, qt * 32, 0), gn = TL::row_read(ga, qt * 32, 0), vn = TL::row_read(vb, 0, 0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const u32x4 qc = qn, gc = gn, vc = vn;
          if (ks + 1 < KS) {
            qn = TL::row_read(qa, qt * 32, ks + 1);
            gn = TL::row_read(ga, qt * 32, ks + 1);
            vn = TL::row_read(vb, 0, ks + 1);
          }
          __builtin_amdgcn_sched_barrier(0);
          s = T::mma(qc, kf[ks], s);
          dp = T::mma(gc, vc, dp);
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s = T::mma(TL::row_read(qa, qt * 32, ks), kf[ks], s);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) dp = T::mma(TL::row_read(ga, qt * 32, ks), vf[ks], dp);
      }
      const int qi0 = i + 4 * half;
      const float dist0 = (float)(shift + qi0 - key);
      float dsc[16];
      f32x4 ls[4];
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) ls[q4] = *reinterpret_cast<const f32x4*>(rows + BQ + qt * 32 + 8 * q4 + 4 * half);
      doc_weights<T, SHAPE>(p, s, dsc, slope2, [&](int r) { return dist0 + (float)(8 * (r >> 2) + (r & 3)); }, [&](int r) { return ls[r >> 2][r & 3]; });
      if (cls != 2) doc_mask<true>(s, qi0, span, 0, 0.f);
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const f32x4 de = *reinterpret_cast<const f32x4*>(rows + qt * 32 + 8 * q4 + 4 * half);
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[4 * q4 + e] = doc_ds<SHAPE>(s[4 * q4 + e], dp[4 * q4 + e], de[e], dsc[4 * q4 + e]);
      }
      if constexpr (VL) {
        constexpr int N = 32 / T::STEP * DT;
        u32x4 gn = TL::tr_read(tg, qt * 32, 0, lane), qn = TL::tr_read(tq, qt * 32, 0, lane), pf, df;
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const int ss = n / DT, dt = n % DT;
          const u32x4 gc = gn, qc = qn;
          if (dt == 0) {
            pf = T::pack(s, ss);
            df = T::pack(dp, ss);
          }
          if (n + 1 < N) {
            gn = TL::tr_read(tg, qt * 32 + T::STEP * ((n + 1) / DT), (n + 1) % DT, lane);
            qn = TL::tr_read(tq, qt * 32 + T::STEP * ((n + 1) / DT), (n + 1) % DT, lane);
          }
          __builtin_amdgcn_sched_barrier(0);
          dv[dt] = T::mma(gc, pf, dv[dt]);
          dk[dt] = T::mma(qc, df, dk[dt]);
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
#pragma unroll
        for (int ss = 0; ss < 32 / T::STEP; ++ss) {
          const u32x4 pf = T::pack(s, ss), df = T::pack(dp, ss);
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) dv[dt] = T::mma(TL::tr_read(tg, qt * 32 + T::STEP * ss, dt, lane), pf, dv[dt]);
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) dk[dt] = T::mma(TL::tr_read(tq, qt * 32 + T::STEP * ss, dt, lane), df, dk[dt]);
        }
      }
    }
  }
  __syncthreads();
  if (p.split == 1) {
    char* const patch = smem + wave * 32 * TL::RB;
    auto row = [&](void* base, size_t ld) {
      return [=](int r) -> char* {
        return jw + r >= d.nk ? nullptr : reinterpret_cast<char*>(base) + (((size_t)d.k0 + jw + r) * ld + (size_t)kvh * p.hd) * T::ES;
      };
    };
    doc_store_rows<T, HDP>(patch, dk, p.scale, p.hd, lane, row(p.dk, p.ld_dk));
    doc_store_rows<T, HDP>(patch, dv, 1.0f, p.hd, lane, row(p.dv, p.ld_dv));
  } else if (key < d.nk) {
    float* w = p.ws_o + (((size_t)sp * p.rows_k + d.k0 + key) * p.kv_heads + kvh) * 2 * p.hd;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = dt * 32 + 8 * g + 4 * half;
        if (c < p.hd) {
          *reinterpret_cast<float4*>(w + c) = make_float4(dk[dt][4 * g], dk[dt][4 * g + 1], dk[dt][4 * g + 2], dk[dt][4 * g + 3]);
          *reinterpret_cast<float4*>(w + p.hd + c) = make_float4(dv[dt][4 * g], dv[dt][4 * g + 1], dv[dt][4 * g + 2], dv[dt][4 * g + 3]);
        }
      }
  }
}

// sums the parts of a split, in order: one thread per 8 columns of dk | dv of one (key row, key head)
template <typename T> __global__ __launch_bounds__(256) void doc_dkv_join_kernel(DocAttnP p) {
  const int cpr = p.hd / 4;  // 8-column pieces of dk and dv
  const size_t idx = (size_t)blockIdx.x * 256 + threadIdx.x, n = (size_t)p.rows_k * p.kv_heads;
  const size_t at = idx / cpr;
  int c = (int)(idx - at * cpr) * 8;
  if (at >= n) return;
  const size_t row = at / p.kv_heads;
  const int kvh = (int)(at - row * p.kv_heads);
  const int end = p.n_docs > p.n_real ? p.rows_k : doc_clamp(p.k_begin[p.n_real], 0, p.rows_k);
  if ((int)row >= end || (int)row < doc_clamp(p.k_begin[0], 0, p.rows_k)) return;
  float acc[8] = {};
  for (int s = 0; s < p.split; ++s) {
    float v[8];
    load8(p.ws_o + (s * n + at) * 2 * p.hd + c, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] += v[e];
  }
  const bool is_k = c < p.hd;
  if (is_k) {
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= p.scale;
  } else {
    c -= p.hd;
  }
  store8(reinterpret_cast<typename T::E*>(is_k ? p.dk : p.dv) + row * (is_k ? p.ld_dk : p.ld_dv) + (size_t)kvh * p.hd + c, acc);
}

template <typename T, int HDP, int KS, int SHAPE> int run_doc_bwd(const DocAttnP& p0, hipStream_t st) {
  using TL = DocTile<T, HDP>;
  DocAttnP p = p0;
  constexpr int tiles = 4 * DocStage<T, HDP, T::BK, 4>::BYTES, patch = 4 * 32 * TL::RB;
  constexpr int BQ = doc_bq<T, HDP>, stages = 4 * DocStage<T, HDP, BQ, 4>::BYTES + 4 * BQ * 4 + (doc_v_in_lds<T, HDP, SHAPE> ? 128 * TL::RB : 0);
  constexpr int bytes_q = tiles > patch ? tiles : patch, bytes_k = stages > patch ? stages : patch;
  const auto kq = doc_attn_dq_kernel<T, HDP, KS, SHAPE>;
  const auto kk = doc_attn_dkv_kernel<T, HDP, KS, SHAPE>;
  if (bytes_q > 64 * 1024) OSUD_BIG_LDS_ONCE(kq);
  if (bytes_k > 64 * 1024) OSUD_BIG_LDS_ONCE(kk);
  p.slots = (int)((long)p.rows_q * p.G / 128) + p.n_docs;
  const int split = p.split;
  p.split = 1;
  kq<<<dim3((unsigned)(p.slots * p.kv_heads)), 256, bytes_q, st>>>(p);
  OSUD_HIP(hipGetLastError());
  p.slots = p.rows_k / 128 + p.n_docs;
  p.split = split;
  kk<<<dim3((unsigned)(p.slots * p.kv_heads * p.split)), 256, bytes_k, st>>>(p);
  OSUD_HIP(hipGetLastError());
  if (p.split > 1) {
    const size_t items = (size_t)p.rows_k * p.kv_heads * (p.hd / 4);
    doc_dkv_join_kernel<T><<<dim3((unsigned)((items + 255) / 256)), 256, 0, st>>>(p);
    OSUD_HIP(hipGetLastError());
  }
  return OSUD_OK;
}
template <typename T, int HDP, int KS> int run_doc_bwd_shape(const DocAttnP& p, hipStream_t st) {
  switch ((p.cap > 0.f ? kShapeCap : 0) | (p.slopes != nullptr ? kShapeSlope : 0)) {
    case 0: return run_doc_bwd<T, HDP, KS, 0>(p, st);
    case kShapeCap: return run_doc_bwd<T, HDP, KS, kShapeCap>(p, st);
    case kShapeSlope: return run_doc_bwd<T, HDP, KS, kShapeSlope>(p, st);
    default: return run_doc_bwd<T, HDP, KS, kShapeCap | kShapeSlope>(p, st);
  }
}
template <typename T> int run_doc_bwd_hd(const DocAttnP& p, hipStream_t st) {
  constexpr int N = T::ES == 2 ? 16 : 8;
  if (p.hd <= 64) return run_doc_bwd_shape<T, 64, 64 / N>(p, st);
  if (p.hd <= 80) return run_doc_bwd_shape<T, 96, 80 / N>(p, st);
  if (p.hd <= 96) return run_doc_bwd_shape<T, 96, 96 / N>(p, st);
  return run_doc_bwd_shape<T, 128, 128 / N>(p, st);
}

// Parts of the query axis of the key kernel: as in the forward pass, where its tiles do not give every CU four workgroups (the parts also even out
// a causal mask); at least 512 query rows per part (fp32: 128), at most 16 parts.
int doc_bwd_split(const DocAttnP& p, int prec, int max_q) {
  const int tiles = (p.rows_k / 128 + p.n_docs) * p.kv_heads, least = prec == OSUD_PREC_F32 ? 128 : 512;
  const long rows = (long)(max_q > 0 ? max_q : p.rows_q / (p.n_docs > 0 ? p.n_docs : 1)) * p.G;
  if (p.rows_k == 0 || tiles <= 0 || tiles > 2 * p.cus) return 1;  // (no keys: nothing to join)
  long n = 4L * p.cus / tiles;
  if (n > rows / least) n = rows / least;
  if (n > 16) n = 16;
  return n < 1 ? 1 : (int)n;
}

}  // namespace

size_t doc_attn_bwd_ws(const DocAttnP& p, int prec, int max_q) {
  const size_t n = doc_bwd_split(p, prec, max_q), rows = 2 * (size_t)p.heads * p.rows_q;
  return (rows + 3) / 4 * 4 + (n > 1 ? n * p.rows_k * p.kv_heads * 2 * p.hd : 0);
}

int launch_doc_attn_bwd(int prec, DocAttnP& p, int max_q, size_t ws_floats, hipStream_t st) {
  const size_t rows = (2 * (size_t)p.heads * p.rows_q + 3) / 4 * 4, part = (size_t)p.rows_k * p.kv_heads * 2 * p.hd;
  p.split = doc_bwd_split(p, prec, max_q);
  if (p.split > 1 && rows + p.split * part > ws_floats) p.split = ws_floats < rows + 2 * part ? 1 : (int)((ws_floats - rows) / part);
  p.ws_o = p.delta + rows;
  return prec == OSUD_PREC_BF16 ? run_doc_bwd_hd<DocBf16>(p, st) : run_doc_bwd_hd<DocF32>(p, st);
}

}  // namespace osud
