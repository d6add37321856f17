// Attention over packed documents, forward:  s = scale q.k;  s = cap tanh(s / cap);  s -= slope_h |pos_q - pos_k|;  masks;  o = softmax(s) v.
// (Reference: nn.MultiheadAttention inside DiTBlock.forward, models.py:130-135,164-170, with the (T, T) boolean mask of sample.py:81-84.)
//
// One workgroup = 128 shared rows (queries x the heads of one key head, see doc_attn.h) of one document, four waves of 32 rows.  S^T = K.Q^T on
// the 32 x 32 matrix instructions, so a lane owns one row and the softmax needs one exchange with lane ^ 32; P goes back into the matrix
// pipe as the B operand without leaving registers; the K | V rows of the next block travel by LDS-DMA into the other half of a double
// buffer while this block is computed, one barrier per block.  Statistics, sums and accumulators are fp32; P is rounded to the
// element type for its product (at most 2^-8 of it in bf16, 2^-11 in fp16: the size of the output's own rounding), the sum of lse is taken before.
//
// Bound: the matrix pipe together with the exponentials (16 cycles each, a matrix instruction of 32 x 32 x 16 takes 32).  2 documents of 8192 positions, 12 / 4
// heads of 128 columns, causal: 443 us, 930 TFLOP/s (a large bf16 product: 1225); 4 documents of 8192, 12 heads of 64: 897 us, 919; one query against
// 16 x ~8000 keys: 52-60 us, 4.6-5.3 TB/s.
#include <type_traits>

#include "doc_attn.h"
#include "kernels.h"

namespace osud {
namespace {

template <typename T, int HDP, int KS, int SHAPE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(T::ES == 2 ? (HDP == 64 && SHAPE == 0 ? 4 : HDP == 64 || (HDP == 96 && (KS == 5 || (SHAPE & kShapeSlope) == 0)) ? 3 : 2) : (HDP == 64 ? 2 : 1)))) void doc_attn_kernel(DocAttnP p) {
  using TL = DocTile<T, HDP>;
  constexpr int BK = T::BK, KT = BK / 32, DT = HDP / 32;
  using ST = DocStage<T, HDP, BK, 4>;
  constexpr int TILE = ST::BYTES, STAGE = 2 * TILE;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const uint32_t lds0 = (uint32_t)(size_t)(const __attribute__((address_space(3))) void*)smem;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int frow = lane & 31, half = lane >> 5;

  const DocUnit u = doc_unit(p, true);
  const int sp = u.part, kvh = u.kvh;
  int tile;
  const DocRange d = doc_range(p, doc_find<128>(p.q_begin, p.n_docs, p.rows_q, p.G, u.slot, lane, tile), true);
  const int vrows = d.nq * p.G, row0 = tile * 128;
  if (tile < 0 || row0 >= vrows) return;

  // this lane's row; positions of the workgroup's and of this wave's rows
  const int vr = row0 + wave * 32 + frow;
  const int vrc = vr < vrows ? vr : vrows - 1;
  const int qi = (int)((unsigned)vrc / (unsigned)p.G), head = kvh * p.G + vrc - qi * p.G;
  const int shift = d.nk - d.nq, pos = shift + qi;
  const size_t qrow = (size_t)d.q0 + qi;
  auto pos_of = [&](int r) { return shift + (int)((unsigned)(r < vrows ? r : vrows - 1) / (unsigned)p.G); };
  const int wg0 = pos_of(row0), wg1 = pos_of(row0 + 127);
  const int wv0 = __builtin_amdgcn_readlane(pos, 0), wv1 = __builtin_amdgcn_readlane(pos, 31);
  const bool alive = row0 + wave * 32 < vrows;

  // the blocks to visit: those of the prefix, then those of the band
  const int npre = (d.pre + BK - 1) / BK;
  int bl = doc_band(p, wg0, d.nk).lo / BK;
  const int hi = doc_band(p, wg1, d.nk).hi;
  if (bl < npre) bl = npre;
  const int nband = hi < 0 || hi / BK < bl ? 0 : hi / BK - bl + 1;
  const int nblk = npre + nband;
  int it = p.split > 1 ? (int)((long)sp * nblk / p.split) : 0;
  const int it_end = p.split > 1 ? (int)((long)(sp + 1) * nblk / p.split) : nblk;

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
  if (it < it_end) issue(it, 0);

  u32x4 qf[KS];
  {
    const char* qp = reinterpret_cast<const char*>(p.q) + (qrow * p.ld_q + (size_t)head * p.hd) * T::ES;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[ks] = u32x4{0u, 0u, 0u, 0u};
      if (2 * ks + half < cols) qf[ks] = *reinterpret_cast<const u32x4*>(qp + (2 * ks + half) * 16);
    }
  }
  float slope2 = 0.f;
  if constexpr ((SHAPE & kShapeSlope) != 0) slope2 = p.slopes[head] * kLog2e;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[ks]));  // (waited for here, not inside the loop, where it would drain the DMA)

  const DocBand band = doc_band(p, pos, d.nk);
  const DocSpan span = doc_span(band.lo, band.hi);
  f32x16 o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
  float m_run = (SHAPE & kShapeFixed) != 0 ? 0.f : -INFINITY, l_run = 0.f;
  // Without a running maximum a row's largest weight is no power of two and gets rounded, also where it is the only one: the rounded weights' own sum
  // divides then, and a row that sees one key returns its v
  constexpr bool kOwnSum = (SHAPE & kShapeFixed) != 0 && !T::kExact;
  [[maybe_unused]] float l_own = 0.f;
  [[maybe_unused]] const bool onesided = p.right == 0 && d.pre == 0;

  const uint32_t kb = lds0 + TL::row_base(lane), vb = lds0 + TILE + TL::tr_base(lane);
  int stage = 0;
  for (; it < it_end; ++it) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (it + 1 < it_end) issue(it + 1, stage ^ 1);
    const int j0 = block_of(it) * BK;
    const uint32_t ka = kb + stage * STAGE, va = vb + stage * STAGE;
    stage ^= 1;
    const int cls = alive ? doc_class(p, wv0, wv1, j0, j0 + BK - 1, d.nk, d.pre) : 0;
    if (cls == 0) continue;
    f32x16 s[KT];
    const int key_lane = j0 + 4 * half;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[kt][r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s[kt] = T::mma(TL::row_read(ka, kt * 32, ks), qf[ks], s[kt]);
    }
    // scores in the log2 domain: k1 * s + base (base: this block's and row's part of a distance that has one sign)
    constexpr bool kCap = (SHAPE & kShapeCap) != 0, kSlope = (SHAPE & kShapeSlope) != 0, kFixed = (SHAPE & kShapeFixed) != 0;
    if constexpr (kCap) {
      float big = 0.f;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) big = doc_largest(s[kt], big);
      const bool small = !__any(big > p.small);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) doc_tanh<T>(p, p.tanh2, p.cap2, small, s[kt]);
    }
    const float k1 = kCap || kSlope ? 1.0f : p.c1;
    float base = 0.f;
    if constexpr (kSlope) {
      const float dist0 = (float)(pos - key_lane);
      if (onesided) {  // every visible key is at or before the position: -slope |pos - key| = -slope dist0 + slope off
        base = -slope2 * dist0;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[kt][r] = fmaf(s[kt][r], kCap ? 1.0f : p.c1, slope2 * (float)(kt * 32 + 8 * (r >> 2) + (r & 3)));
      } else {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[kt][r] = fmaf(-slope2, fabsf(dist0 - (float)(kt * 32 + 8 * (r >> 2) + (r & 3))), kCap ? s[kt][r] : s[kt][r] * p.c1);
      }
    }
    if (cls == 1) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) doc_mask<kCap>(s[kt], key_lane + kt * 32, span, d.pre, -INFINITY);
    }
    float shift = 0.f;
    if constexpr (!kFixed) {
      float mx = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[kt][r]);
      mx = doc_half_max(fmaf(mx, k1, base));
      // The reference point moves only when a score passes it by 8 binary orders: p <= 2^8 stays far inside every type's range, and the
      // accumulators are rescaled a few times per row instead of once per block
      const bool up = mx > m_run + 8.0f || (m_run == -INFINITY && mx > -INFINITY);
      if (__any(up)) {
        const float m_new = fmaxf(m_run, mx);
        const float alpha = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - m_new);
        m_run = m_new;
        l_run *= alpha;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) asm volatile("v_mul_f32 %0, %1, %0" : "+v"(o[i][r]) : "v"(alpha));  // (in place: as plain products the compiler copies all of o on every block)
      }
      shift = base - (m_run == -INFINITY ? 0.f : m_run);
    }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int ss = 0; ss < 32 / T::STEP; ++ss) {
#pragma unroll
        for (int r = ss * T::STEP / 2; r < (ss + 1) * T::STEP / 2; ++r) {
          const float e = __builtin_amdgcn_exp2f(kFixed ? s[kt][r] : kCap || kSlope ? s[kt][r] + shift : fmaf(s[kt][r], k1, shift));
          s[kt][r] = e;
          l_run += e;
        }
        const u32x4 pf = T::pack(s[kt], ss);
        if constexpr (kOwnSum) l_own = T::sum(pf, l_own);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] = T::mma(TL::tr_read(va, kt * 32 + T::STEP * ss, dt, lane), pf, o[dt]);
      }
  }
  __syncthreads();  // (the stages are idle: they become the waves' patches)
  if (!alive) return;
  const float l = doc_half_sum(l_run);
  float own = l;
  if constexpr (kOwnSum) own = doc_half_sum(l_own);
  char* const patch = smem + wave * 32 * TL::RB;
  if (p.split == 1) {
    const float inv = own > 0.f || own != own ? 1.0f / own : 0.f;  // (no key seen: zeros)
    if (p.lse != nullptr && half == 0 && vr < vrows)
      p.lse[(size_t)head * p.rows_q + qrow] = doc_lse(m_run, l);
    doc_store_rows<T, HDP>(patch, o, inv, p.hd, lane, [&](int r) -> char* {
      const int v = row0 + wave * 32 + r;
      if (v >= vrows) return nullptr;
      const int i = (int)((unsigned)v / (unsigned)p.G);
      return reinterpret_cast<char*>(p.out) + (((size_t)d.q0 + i) * p.ld_o + (size_t)(kvh * p.G + v - i * p.G) * p.hd) * T::ES;
    });
  } else {
    if (vr < vrows) {
      const size_t at = ((size_t)sp * p.rows_q + qrow) * p.heads + head;
      if (half == 0) *reinterpret_cast<float2*>(p.ws_ml + 2 * at) = make_float2(m_run, l);
      if constexpr (kOwnSum) {  // (the parts are joined by l)
        const float f = own > 0.f ? l / own : 1.0f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[dt][r] *= f;
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int c = dt * 32 + 8 * g + 4 * half;
          if (c < p.hd) *reinterpret_cast<float4*>(p.ws_o + at * p.hd + c) = make_float4(o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]);
        }
    }
  }
}

// joins the parts of a split (at most 64): one wave per (row, head); lane s takes part s's weight, then every lane 2 columns of all parts, in order
template <typename T> __global__ __launch_bounds__(256) void doc_join_kernel(DocAttnP p) {
  const int lane = threadIdx.x & 63;
  const size_t n = (size_t)p.rows_q * p.heads, at = (size_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (at >= n) return;
  const int row = (int)(at / p.heads), head = (int)(at - (size_t)row * p.heads);
  const int end = p.n_docs > p.n_real ? p.rows_q : doc_clamp(p.q_begin[p.n_real], 0, p.rows_q);
  if (row >= end || row < doc_clamp(p.q_begin[0], 0, p.rows_q)) return;  // (no document's: nothing was written)
  float2 ml = make_float2(-INFINITY, 0.f);
  if (lane < p.split) ml = *reinterpret_cast<const float2*>(p.ws_ml + 2 * (lane * n + at));
  const float m = wave_max(ml.x), mu = m == -INFINITY ? 0.f : m;
  const float w = ml.x == -INFINITY && ml.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml.x - mu);
  const float l = wave_sum(ml.y * w);
  float a0 = 0.f, a1 = 0.f;
  const float* src = p.ws_o + at * p.hd + 2 * lane;
  if (2 * lane < p.hd) {
#pragma unroll 8
    for (int s = 0; s < p.split; ++s) {
      const float2 v = *reinterpret_cast<const float2*>(src + s * n * p.hd);
      const float ws = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), s));
      a0 = fmaf(v.x, ws, a0);
      a1 = fmaf(v.y, ws, a1);
    }
    const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
    store2(reinterpret_cast<typename T::E*>(p.out) + (size_t)row * p.ld_o + (size_t)head * p.hd + 2 * lane, a0 * inv, a1 * inv);
  }
  if (lane == 0 && p.lse != nullptr) p.lse[(size_t)head * p.rows_q + row] = doc_lse(m, l);
}

template <typename T, int HDP, int KS, int SHAPE> int run_doc_attn(const DocAttnP& p, hipStream_t st) {
  constexpr int lds = 4 * DocStage<T, HDP, T::BK, 4>::BYTES, patch = 4 * 32 * DocTile<T, HDP>::RB;
  constexpr int bytes = lds > patch ? lds : patch;
  const auto kernel = doc_attn_kernel<T, HDP, KS, SHAPE>;
  if (bytes > 64 * 1024) OSUD_BIG_LDS_ONCE(kernel);
  kernel<<<dim3((unsigned)(p.slots * p.kv_heads * p.split)), 256, bytes, st>>>(p);
  OSUD_HIP(hipGetLastError());
  if (p.split > 1) {
    doc_join_kernel<T><<<dim3((unsigned)(((size_t)p.rows_q * p.heads + 3) / 4)), 256, 0, st>>>(p);
    OSUD_HIP(hipGetLastError());
  }
  return OSUD_OK;
}
template <typename T, int HDP, int KS> int run_doc_attn_shape(const DocAttnP& p, hipStream_t st) {
  switch ((p.cap > 0.f ? kShapeCap : 0) | (p.slopes != nullptr ? kShapeSlope : 0)) {
    case 0: return run_doc_attn<T, HDP, KS, 0>(p, st);
    case kShapeCap:
      if constexpr (!std::is_same<T, DocF16>::value) {
        if (p.cap <= kFixedCap) return run_doc_attn<T, HDP, KS, kShapeCap | kShapeFixed>(p, st);
      }
      return run_doc_attn<T, HDP, KS, kShapeCap>(p, st);
    case kShapeSlope: return run_doc_attn<T, HDP, KS, kShapeSlope>(p, st);
    default: return run_doc_attn<T, HDP, KS, kShapeCap | kShapeSlope>(p, st);
  }
}
// widths of 64, 96 and 128 columns; 65 .. 80 columns skip the contraction steps of the last sixteen pad columns
template <typename T> int run_doc_attn_hd(const DocAttnP& p, hipStream_t st) {
  constexpr int N = T::ES == 2 ? 16 : 8;
  if (p.hd <= 64) return run_doc_attn_shape<T, 64, 64 / N>(p, st);
  if (p.hd <= 80) return run_doc_attn_shape<T, 96, 80 / N>(p, st);
  if (p.hd <= 96) return run_doc_attn_shape<T, 96, 96 / N>(p, st);
  return run_doc_attn_shape<T, 128, 128 / N>(p, st);
}

// Parts of the key axis: few tiles (no more than one per CU) of long documents leave most of the chip idle; up to four workgroups per CU then, each
// with at least 512 keys (a part leaves and re-reads 128 rows x head_dim floats: as much as 128 keys).  fp32 keys take sixteen times as long: 128.
int doc_split(const DocAttnP& p, int prec, int max_k) {
  const int tiles = p.slots * p.kv_heads;
  const long keys = max_k > 0 ? max_k : p.rows_k / (p.n_docs > 0 ? p.n_docs : 1);
  if (tiles <= 0 || tiles > p.cus) return 1;
  long n = 4L * p.cus / tiles;
  const int least = prec == OSUD_PREC_F32 ? 128 : 512;
  if (n > keys / least) n = keys / least;
  if (n > 64) n = 64;
  return n < 1 ? 1 : (int)n;
}

}  // namespace

size_t doc_attn_ws(const DocAttnP& p, int prec, int max_k) {
  const size_t n = doc_split(p, prec, max_k);
  return n > 1 ? n * p.rows_q * p.heads * (p.hd + 2) : 0;
}

int launch_doc_attn(int prec, DocAttnP& p, int max_k, size_t ws_floats, hipStream_t st) {
  p.split = doc_split(p, prec, max_k);
  const size_t part = (size_t)p.rows_q * p.heads * (p.hd + 2);
  if (p.split > 1 && (size_t)p.split * part > ws_floats) p.split = ws_floats / part < 2 ? 1 : (int)(ws_floats / part);
  p.ws_ml = p.ws_o;
  if (p.split > 1) p.ws_ml += (size_t)p.split * p.rows_q * p.heads * p.hd;
  if (prec == OSUD_PREC_BF16) return run_doc_attn_hd<DocBf16>(p, st);
  if (prec == OSUD_PREC_F16) return run_doc_attn_hd<DocF16>(p, st);
  return run_doc_attn_hd<DocF32>(p, st);
}

}  // namespace osud
