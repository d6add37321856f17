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
// rows per workgroup and turn, head-rows in flight per group of lanes, workgroups per CU of the backward pass (what its registers allow)
template <bool BACK> constexpr int kTpb = BACK ? 4 : 8;
template <bool BACK> constexpr int kFlight = BACK ? 1 : 2;
template <int W> constexpr int kBackPerCu = W == 8 ? 4 : 5;

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
// both chunks of a head (INTER: they are one)
template <int W, bool INTER, typename E> __device__ __forceinline__ void load_lane(const E* p, const RopeLane<W, INTER>& ln, float (&x)[2 * W]) {
  if constexpr (INTER && W <= 4) {
    float v[2 * W] = {};
    if (ln.a) load_chunk<2 * W>(p + ln.ca, v);
#pragma unroll
    for (int i = 0; i < 2 * W; ++i) x[i] = v[i];
  } else {
    float a[W] = {}, b[W] = {};
    if (ln.a) load_chunk<W>(p + ln.ca, a);
    if (ln.b) load_chunk<W>(p + ln.cb, b);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      x[i] = a[i];
      x[W + i] = b[i];
    }
  }
}
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
__device__ __forceinline__ void head(const RopeP& p, const RopeLane<W, INTER>& ln, const float2* cs, float inv_hd, const float (&wt)[2 * W], float (&x)[2 * W],
                                     float (&g)[BACK ? 2 * W : 1], float (&dw)[2 * W]) {
  float r = 1.f;
  if (p.norm) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * W; ++i) ss = fmaf(x[i], x[i], ss);
    r = 1.0f / sqrtf(fmaf(group_sum<GL>(ss), inv_hd, p.eps));
  }
  if constexpr (!BACK) {
#pragma unroll
    for (int i = 0; i < 2 * W; ++i) x[i] = x[i] * r * wt[i];
    if (ln.turn) rope_turn<W, INTER, false>(cs, x);
  } else {
    if (ln.turn) rope_turn<W, INTER, true>(cs, g);
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

template <typename E, int W, int GL /* lanes per head */, bool INTER, bool BACK>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(BACK ? kBackPerCu<W> : 4))) void qk_norm_rope_kernel(RopeP p) {
  constexpr int TPB = kTpb<BACK>, FL = kFlight<BACK>;
  __shared__ float2 table[TPB * (kMaxHd / 2)];
  __shared__ float red[BACK ? 256 * 2 * W : 1];
  const int l = threadIdx.x % GL, grp = threadIdx.x / GL;
  constexpr int NG = 256 / GL;
  const RopeLane<W, INTER> ln(p, l);
  float dw[2][2 * W] = {};
  const float inv_hd = 1.0f / (float)p.hd;
  for (long c = blockIdx.x; c * TPB < p.rows; c += gridDim.x) {
    const long t0 = c * TPB;
    const int n = p.rows - t0 < TPB ? (int)(p.rows - t0) : TPB;
    __syncthreads();
    rope_angles(p, t0, n, table);
    __syncthreads();
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const int heads = part ? p.kv_heads : p.heads;
      if (heads == 0) continue;
      const E* const src = reinterpret_cast<const E*>(part ? p.k : p.q);
      const E* const up = reinterpret_cast<const E*>(part ? p.gk : p.gq);
      E* const dst = reinterpret_cast<E*>(part ? p.ko : p.qo);
      const size_t ld = part ? p.ld_k : p.ld_q, ldg = part ? p.ld_gk : p.ld_gq, ldo = part ? p.ld_ko : p.ld_qo;
      const float* const w = part ? p.kw : p.qw;
      float wt[2 * W];
#pragma unroll
      for (int i = 0; i < W; ++i) {
        wt[i] = w != nullptr && ln.a ? w[ln.ca + i] : 1.f;
        wt[W + i] = w != nullptr && ln.b ? w[ln.cb + i] : 1.f;
      }
      // head-rows grp, grp + NG, ... of the n * heads: FL at a time, all loaded before the first is computed
      for (int i0 = grp; i0 < n * heads; i0 += FL * NG) {
        float x[FL][2 * W], g[FL][BACK ? 2 * W : 1];
        int t[FL];
        size_t out[FL];
        bool live[FL];
#pragma unroll
        for (int j = 0; j < FL; ++j) {
          const int i = i0 + j * NG;
          live[j] = i < n * heads;
          t[j] = live[j] ? (int)((unsigned)i / (unsigned)heads) : 0;
          const size_t row = (size_t)(t0 + t[j]), col = live[j] ? (size_t)(i - t[j] * heads) * p.hd : 0;
          out[j] = row * ldo + col;
          if (live[j]) load_lane<W, INTER>(src + row * ld + col, ln, x[j]);
          if constexpr (BACK) {
            if (live[j]) load_lane<W, INTER>(up + row * ldg + col, ln, g[j]);
          }
        }
#pragma unroll
        for (int j = 0; j < FL; ++j) {
          if (!live[j]) continue;  // (a group of lanes is alive or not as one)
          head<W, GL, INTER, BACK>(p, ln, table + t[j] * (p.rot / 2) + ln.pair, inv_hd, wt, x[j], g[j], dw[part]);
          store_lane<W, INTER>(dst + out[j], ln, x[j]);
        }
      }
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

constexpr int kBackGroups = 5 * 256;  // at most so many workgroups in the backward pass: rows of ws

template <typename E, int W, int GL, bool INTER, bool BACK> int run_rope(const RopeP& p, hipStream_t st) {
  constexpr int TPB = kTpb<BACK>;
  const long chunks = p.rows > TPB ? (p.rows + TPB - 1) / TPB : 1;  // (no rows: one workgroup that leaves zeros for the weights)
  long most = 1L << 30;
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
  if (all % 8 == 0) return p.hd <= 64 ? run_rope<E, 8, 4, false, BACK>(p, st) : run_rope<E, 8, 8, false, BACK>(p, st);
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
