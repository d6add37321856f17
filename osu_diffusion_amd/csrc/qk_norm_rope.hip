// Norms of queries and keys for each head and the rotation by position, in one pass over the rows, forward and backward.
// (No counterpart in the reference: its positions enter through the sinusoidal features of models.py:199-225.)
//   r = 1 / sqrt(mean x^2 + eps),  z = x r w;   pair (a, b) of z, angle th = position * f:  a' = gain (a cos th - b sin th),  b' = gain (a sin th + b cos th)
//   backward: dz = the transposed rotation of the gradient;  dw = sum dz x r;  u = dz w;  dx = r (u - x r mean(u x r))
// Memory bound: forward reads and writes every head once, backward reads x and the gradient and writes dx (r is computed again).
//
// A group of lanes owns one head of one row; a lane holds two chunks of W columns that form W whole pairs (half layout: columns i and
// R + i; interleaved: 2 W neighbouring columns), so the rotation needs no exchange and the norm a few lane shuffles.  A workgroup takes
// TPB rows: their angles first, one per lane, into LDS -- each serves all heads of its row.  position * f / 2 pi is taken in 64 bits and
// reduced to a fraction of a turn there: at 10^6 positions a product in 32 bits is off by 0.06 radians.
#include <type_traits>

#include "attn_frag.h"
#include "kernels.h"

namespace osud {
namespace {

constexpr int kMaxHd = 128;
// rows per workgroup and turn; heads in flight per group of lanes; workgroups per CU of the backward pass.  Two heads and what registers they
// leave: 32768 rows of 16 + 16 heads of 72 columns backward (453 MB) 115 us; one head and five workgroups 121, two and three 145; fp32 one head
// (5003 rows, 25 us against 32).
constexpr int kTpb = 8;
template <typename E, bool BACK> constexpr int kFlight = BACK && sizeof(E) == 4 ? 1 : 2;
template <int W> constexpr int kBackPerCu = W == 8 ? 3 : 4;

template <int W, typename E> __device__ __forceinline__ void load_chunk(const E* p, float (&v)[W]) {
  if constexpr (W == 8) load8(p, v);
  else if constexpr (W == 1) v[0] = load_elem(p);
  else loadw<W>(p, v);
}
template <int W, typename E> __device__ __forceinline__ void store_chunk(E* p, const float (&v)[W]) {
  if constexpr (W == 8) store8(p, v);
  else if constexpr (W == 1) store_elem(p, v[0]);
  else storew<W>(p, v);
}

// cos and sin (times gain) of the rows t0 .. t0 + n - 1 into LDS, [row][R]
__device__ __forceinline__ void rope_angles(const RopeP& p, long t0, int n, float2* table) {
  const int R = p.rot / 2;
  for (int i = threadIdx.x; i < n * R; i += 256) {
    const int t = i / R, f = i - t * R;
    const double pos = p.float_positions ? (double)reinterpret_cast<const float*>(p.positions)[t0 + t] : (double)reinterpret_cast<const int32_t*>(p.positions)[t0 + t];
    double turn = pos * p.freqs[f] * 0.15915494309189533577;
    turn -= rint(turn);
    float s, c;
    sincospif(2.0f * (float)turn, &s, &c);
    table[i] = make_float2(c * p.gain, s * p.gain);
  }
}

// one lane's two chunks of a head: columns ca .. ca + W - 1 and cb .. cb + W - 1 (INTER: cb = ca + W)
template <int W, bool INTER> struct RopeLane {
  int ca, cb, pair;
  bool a, b, turn;
  __device__ __forceinline__ RopeLane(const RopeP& p, int l) {
    const int R = p.rot / 2, np = R / W;
    turn = l < np;
    pair = turn ? l * W : 0;
    if (INTER || !turn) {
      ca = (INTER ? 0 : p.rot) + 2 * W * (l - (INTER ? 0 : np));
      cb = ca + W;
    } else {
      ca = pair;
      cb = R + pair;
    }
    a = ca < p.hd;
    b = cb < p.hd;
  }
};
// (x[0 .. 2 W - 1] = chunk a, chunk b)  the rotation, or its transpose
template <int W, bool INTER, bool BACK> __device__ __forceinline__ void rope_turn(const float2* cs, float (&x)[2 * W]) {
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const int ia = INTER ? 2 * i : i, ib = INTER ? 2 * i + 1 : W + i;
    float2 t = cs[i];
    if (BACK) t.y = -t.y;
    const float a = x[ia], b = x[ib];
    x[ia] = a * t.x - b * t.y;
    x[ib] = a * t.y + b * t.x;
  }
}
// N neighbouring elements as they lie in memory: loaded long before they are unpacked
template <typename E, int N> struct RawChunk {
  static constexpr int B = N * (int)sizeof(E);
  static constexpr bool F = std::is_same<E, float>::value;
  typedef typename std::conditional<F, float4, uint4>::type V16;
  typedef typename std::conditional<F, float2, uint2>::type V8;
  typedef typename std::conditional<F, float, uint32_t>::type V4;
  typedef typename std::conditional<B >= 16, V16, typename std::conditional<B == 8, V8, typename std::conditional<B == 4, V4, uint16_t>::type>::type>::type V;
  V v[B >= 16 ? B / 16 : 1];
  __device__ __forceinline__ void load(const E* p, bool there) {
#pragma unroll
    for (int i = 0; i < (B >= 16 ? B / 16 : 1); ++i) v[i] = there ? reinterpret_cast<const V*>(p)[i] : V{};
  }
  __device__ __forceinline__ void unpack(float (&x)[N]) const { load_chunk<N>(reinterpret_cast<const E*>(v), x); }
};
// both chunks of a head (INTER: they are one)
template <typename E, int W, bool INTER> struct RawLane {
  static constexpr bool kOne = INTER && W <= 4;
  RawChunk<E, kOne ? 2 * W : W> c[kOne ? 1 : 2];
  __device__ __forceinline__ void load(const E* p, const RopeLane<W, INTER>& ln, bool there) {
    c[0].load(p + ln.ca, there && ln.a);
    if constexpr (!kOne) c[1].load(p + ln.cb, there && ln.b);
  }
  __device__ __forceinline__ void unpack(float (&x)[2 * W]) const {
    if constexpr (kOne) {
      c[0].unpack(x);
    } else {
      float a[W], b[W];
      c[0].unpack(a);
      c[1].unpack(b);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        x[i] = a[i];
        x[W + i] = b[i];
      }
    }
  }
};
template <int W, bool INTER, typename E> __device__ __forceinline__ void store_lane(E* p, const RopeLane<W, INTER>& ln, const float (&x)[2 * W]) {
  if constexpr (INTER && W <= 4) {
    if (ln.a) store_chunk<2 * W>(p + ln.ca, x);
  } else {
    float a[W], b[W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
      a[i] = x[i];
      b[i] = x[W + i];
    }
    if (ln.a) store_chunk<W>(p + ln.ca, a);
    if (ln.b) store_chunk<W>(p + ln.cb, b);
  }
}
// sum over the GL lanes of a group, every lane gets it: exchanges inside 16 lanes are modifiers of the addition
template <int GL> __device__ __forceinline__ float group_sum(float v) {
  auto add = [&](auto CTRL) { v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), decltype(CTRL)::value, 0xf, 0xf, true)); };
  add(std::integral_constant<int, 0xb1>{});                           // lane ^ 1
  add(std::integral_constant<int, 0x4e>{});                           // lane ^ 2
  if constexpr (GL >= 8) add(std::integral_constant<int, 0x141>{});   // 7 - lane in eights: the other four
  if constexpr (GL >= 16) add(std::integral_constant<int, 0x140>{});  // 15 - lane in sixteens: the other eight
  if constexpr (GL >= 32) v += __shfl_xor(v, 16, 64);
  if constexpr (GL >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}

// one head in registers: x becomes the result (BACK: the gradient, from the upstream gradient g; dw gains this head's share)
template <int W, int GL, bool INTER, bool BACK>
__device__ __forceinline__ void head(const RopeP& p, bool turn, const float2* cs, float inv_hd, const float (&wt)[2 * W], float (&x)[2 * W], float (&g)[2 * W],
                                     float (&dw)[2 * W]) {
  float r = 1.f;
  if (p.norm) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * W; ++i) ss = fmaf(x[i], x[i], ss);
    r = __builtin_amdgcn_rsqf(fmaf(group_sum<GL>(ss), inv_hd, p.eps));  // (one unit in the last place)
  }
  if constexpr (!BACK) {
#pragma unroll
    for (int i = 0; i < 2 * W; ++i) x[i] = x[i] * r * wt[i];
    if (turn) rope_turn<W, INTER, false>(cs, x);
  } else {
    if (turn) rope_turn<W, INTER, true>(cs, g);
    if (p.norm) {
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < 2 * W; ++i) {
        x[i] *= r;
        dw[i] = fmaf(g[i], x[i], dw[i]);
        g[i] *= wt[i];
        dot = fmaf(g[i], x[i], dot);
      }
      dot = group_sum<GL>(dot) * inv_hd;
#pragma unroll
      for (int i = 0; i < 2 * W; ++i) x[i] = r * fmaf(-x[i], dot, g[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 2 * W; ++i) x[i] = g[i];
    }
  }
}

// A turn's heads of q, then of k, go by in batches of FL per group of lanes; the next batch is on its way while one is computed, and the first is
// before the angles are taken (32768 rows of 12 + 12 heads of 64 columns, 201 MB not in the caches: 44.7 us, 55.8 with loads where they are used).
template <typename E, int W, int GL /* lanes per head */, bool INTER, bool BACK>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(BACK ? kBackPerCu<W> : 4))) void qk_norm_rope_kernel(RopeP p) {
  constexpr int TPB = kTpb, FL = kFlight<E, BACK>, NG = 256 / GL;
  __shared__ float2 table[TPB * (kMaxHd / 2)];
  __shared__ float weights[2][kMaxHd];
  __shared__ float red[BACK ? 256 * 2 * W : 1];
  typedef RawLane<E, W, INTER> Raw;
  const int l = threadIdx.x % GL, grp = threadIdx.x / GL;
  const RopeLane<W, INTER> ln(p, l);
  float dw[2][2 * W] = {};
  const float inv_hd = 1.0f / (float)p.hd;
  for (int c = threadIdx.x; c < 2 * p.hd; c += 256) {
    const int part = c >= p.hd, i = c - part * p.hd;
    const float* w = part ? p.kw : p.qw;
    weights[part][i] = w != nullptr ? w[i] : 1.f;
  }
  const uint32_t magic[2] = {0xffffffffu / (uint32_t)p.heads + 1u, 0xffffffffu / (uint32_t)(p.kv_heads > 0 ? p.kv_heads : 1) + 1u};
  struct Batch {
    Raw x[FL], g[BACK ? FL : 1];
  };
  struct Turn {
    long t0;        // first row
    int n, nq, nb;  // rows; batches of q, of both
  };
  auto turn_of = [&](long c) {
    Turn u;
    u.t0 = c * TPB;
    u.n = p.rows - u.t0 < TPB ? (p.rows > u.t0 ? (int)(p.rows - u.t0) : 0) : TPB;
    u.nq = (u.n * p.heads + FL * NG - 1) / (FL * NG);
    u.nb = u.nq + (u.n * p.kv_heads + FL * NG - 1) / (FL * NG);
    return u;
  };
  // token and first column of head-row j of batch b; false: none  (i < 8 heads and 8 heads^2 < 2^32: the multiplication by 2^32 / heads, rounded up, divides exactly)
  auto where = [&](auto PART, const Turn& u, int b, int j, uint32_t& t, uint32_t& col) -> bool {
    constexpr int part = decltype(PART)::value;
    const uint32_t heads = part ? p.kv_heads : p.heads, i = ((uint32_t)(part ? b - u.nq : b) * FL + j) * NG + grp;
    const bool there = i < u.n * heads;
    t = there ? (heads == 1 ? i : __umulhi(i, magic[part])) : 0;
    col = there ? (i - t * heads) * p.hd : 0;
    return there;
  };
  auto load = [&](auto PART, const Turn& u, int b, Batch& s) {
    constexpr int part = decltype(PART)::value;
    const size_t ld = part ? p.ld_k : p.ld_q, ldg = part ? p.ld_gk : p.ld_gq;
    const E* const src = reinterpret_cast<const E*>(part ? p.k : p.q) + u.t0 * ld;
    const E* const up = BACK ? reinterpret_cast<const E*>(part ? p.gk : p.gq) + u.t0 * ldg : nullptr;
#pragma unroll
    for (int j = 0; j < FL; ++j) {
      uint32_t t, col;
      const bool there = where(PART, u, b, j, t, col);
      s.x[j].load(src + (t * (uint32_t)ld + col), ln, there);  // (row strides stay below 2^27 elements)
      if constexpr (BACK) s.g[j].load(up + (t * (uint32_t)ldg + col), ln, there);
    }
  };
  auto compute = [&](auto PART, const Turn& u, int b, const Batch& s) {
    constexpr int part = decltype(PART)::value;
    const size_t ldo = part ? p.ld_ko : p.ld_qo;
    E* const dst = reinterpret_cast<E*>(part ? p.ko : p.qo) + u.t0 * ldo;
    float wt[2 * W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
      wt[i] = weights[part][ln.a ? ln.ca + i : 0];
      wt[W + i] = weights[part][ln.b ? ln.cb + i : 0];
    }
#pragma unroll
    for (int j = 0; j < FL; ++j) {
      uint32_t t, col;
      if (!where(PART, u, b, j, t, col)) continue;  // (a group of lanes is alive or not as one)
      float x[2 * W], g[2 * W];
      s.x[j].unpack(x);
      if constexpr (BACK) s.g[j].unpack(g);
      head<W, GL, INTER, BACK>(p, ln.turn, table + t * (p.rot / 2) + ln.pair, inv_hd, wt, x, g, dw[part]);
      store_lane<W, INTER>(dst + (t * (uint32_t)ldo + col), ln, x);
    }
  };
  constexpr std::integral_constant<int, 0> Q{};
  constexpr std::integral_constant<int, 1> K{};
  Batch now, next;
  for (long c = blockIdx.x; c * TPB < p.rows; c += gridDim.x) {
    const Turn u = turn_of(c);
    load(Q, u, 0, now);
    __syncthreads();
    rope_angles(p, u.t0, u.n, table);
    __syncthreads();
    for (int b = 0; b < u.nb; ++b) {
      if (b + 1 < u.nq) load(Q, u, b + 1, next);
      else if (b + 1 < u.nb) load(K, u, b + 1, next);
      if (b < u.nq) compute(Q, u, b, now);
      else compute(K, u, b, now);
      now = next;
    }
  }
  if constexpr (BACK) {  // this workgroup's sums of the weight gradients, groups added in order: one row of ws
    if (p.ws == nullptr) return;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 2 * W; ++i) red[i * 256 + threadIdx.x] = dw[part][i];
      __syncthreads();
      for (int c = threadIdx.x; c < 2 * W * GL; c += 256) {  // (value i of lane q of every group)
        const int i = c / GL, q = c - i * GL;
        const RopeLane<W, INTER> of(p, q);
        if (!(i < W ? of.a : of.b)) continue;
        float s = 0.f;
#pragma unroll 8
        for (int g = 0; g < NG; ++g) s += red[i * 256 + g * GL + q];
        p.ws[((size_t)blockIdx.x * 2 + part) * p.hd + (i < W ? of.ca + i : of.cb + i - W)] = s;
      }
    }
  }
}

// dw[c] = sum over the workgroups' rows, in a fixed order: 4 columns x 64 row lanes per workgroup
__global__ __launch_bounds__(256) void rope_dw_kernel(const float* ws, int parts, int hd, float* dqw, float* dkw) {
  __shared__ float red[256];
  const int c = blockIdx.x * 4 + (threadIdx.x & 3), rl = threadIdx.x >> 2;
  float s = 0.f;
  if (c < 2 * hd) {
#pragma unroll 8
    for (int r = rl; r < parts; r += 64) s += ws[(size_t)r * 2 * hd + c];
  }
  red[threadIdx.x] = s;
  __syncthreads();
  if (rl != 0 || c >= 2 * hd) return;
  for (int i = 1; i < 64; ++i) s += red[4 * i + threadIdx.x];
  float* out = c < hd ? dqw : dkw;
  if (out != nullptr) out[c < hd ? c : c - hd] = s;
}

constexpr int kBackGroups = 4 * 256;  // at most so many workgroups in the backward pass: rows of ws

template <typename E, int W, int GL, bool INTER, bool BACK> int run_rope(const RopeP& p, hipStream_t st) {
  constexpr int TPB = kTpb;
  const long chunks = p.rows > TPB ? (p.rows + TPB - 1) / TPB : 1;  // (no rows: one workgroup that leaves zeros for the weights)
  long most = 1L << 23;  // (a launch has fewer than 2^32 threads; a workgroup takes several turns then)
  if (BACK) {
    most = (long)kBackPerCu<W> * device_cus();
    if (most > kBackGroups) most = kBackGroups;
  }
  const long grid = chunks < most ? chunks : most;
  qk_norm_rope_kernel<E, W, GL, INTER, BACK><<<dim3((unsigned)grid), 256, 0, st>>>(p);
  OSUD_HIP(hipGetLastError());
  if (BACK && p.ws != nullptr) {
    rope_dw_kernel<<<dim3((2 * p.hd + 3) / 4), 256, 0, st>>>(p.ws, (int)grid, p.hd, p.dqw, p.dkw);
    OSUD_HIP(hipGetLastError());
  }
  return OSUD_OK;
}
template <typename E, bool BACK> int run_rope_width(const RopeP& p, hipStream_t st) {
  // the widest chunk that divides the pairs, the head, the rows' strides and the pointers; a head of hd columns takes at most hd / 2 W + 1 lanes
  size_t all = (size_t)p.hd | p.ld_q | p.ld_qo | reinterpret_cast<size_t>(p.q) / sizeof(E) | reinterpret_cast<size_t>(p.qo) / sizeof(E);
  if (p.kv_heads) all |= p.ld_k | p.ld_ko | reinterpret_cast<size_t>(p.k) / sizeof(E) | reinterpret_cast<size_t>(p.ko) / sizeof(E);
  if (BACK) all |= p.ld_gq | reinterpret_cast<size_t>(p.gq) / sizeof(E);
  if (BACK && p.kv_heads) all |= p.ld_gk | reinterpret_cast<size_t>(p.gk) / sizeof(E);
  if (p.interleaved) {  // (a lane's chunks are 2 W neighbouring columns)
    all |= (size_t)p.rot;
    if (all % 8 == 0) return p.hd <= 64 ? run_rope<E, 4, 8, true, BACK>(p, st) : run_rope<E, 4, 16, true, BACK>(p, st);
    if (all % 4 == 0) return run_rope<E, 2, 32, true, BACK>(p, st);
    return run_rope<E, 1, 64, true, BACK>(p, st);
  }
  all |= (size_t)(p.rot / 2);
  if constexpr (sizeof(E) == 2) {
    if (all % 8 == 0) return p.hd <= 64 ? run_rope<E, 8, 4, false, BACK>(p, st) : run_rope<E, 8, 8, false, BACK>(p, st);
  }
  if (all % 4 == 0) return p.hd <= 64 ? run_rope<E, 4, 8, false, BACK>(p, st) : run_rope<E, 4, 16, false, BACK>(p, st);
  if (all % 2 == 0) return run_rope<E, 2, 32, false, BACK>(p, st);
  return run_rope<E, 1, 64, false, BACK>(p, st);
}

}  // namespace

size_t rope_ws_floats(int hd) { return (size_t)kBackGroups * 2 * hd; }

int launch_qk_norm_rope(int prec, const RopeP& p, bool back, hipStream_t st) {
  if (back) return prec == OSUD_PREC_BF16 ? run_rope_width<bf16_t, true>(p, st) : run_rope_width<float, true>(p, st);
  if (prec == OSUD_PREC_BF16) return run_rope_width<bf16_t, false>(p, st);
  if (prec == OSUD_PREC_F16) return run_rope_width<f16_t, false>(p, st);
  return run_rope_width<float, false>(p, st);
}

}  // namespace osud
