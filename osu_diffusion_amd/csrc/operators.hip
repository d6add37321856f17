// C entries of the query / key norm with rotary positions and of attention over packed documents: checks of the arguments, launches.
#include "doc_attn.h"
#include "kernels.h"

using namespace osud;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<size_t>(p) & 15) == 0; }
size_t type_size(int prec) { return prec == OSUD_PREC_F32 ? 4 : 2; }

int check_precision(const char* who, int prec, bool back) {
  if (prec == OSUD_PREC_BF16 || prec == OSUD_PREC_F32 || (prec == OSUD_PREC_F16 && !back)) return OSUD_OK;
  if (prec == OSUD_PREC_F16) set_error("%s: the fp16 tier has no backward pass", who);
  else set_error("%s: precision %d not built (bf16, fp32; fp16 forward)", who, prec);
  return OSUD_ERR_UNSUPPORTED;
}

int rope_params(const char* who, const osud_rope* r, bool back, const void* q, const void* k, const void* qo, const void* ko, const void* gq, const void* gk, RopeP* p) {
  OSUD_CHECK_ARG(r != nullptr, "%s: null argument", who);
  OSUD_TRY(check_precision(who, r->precision, back));
  OSUD_CHECK_ARG(r->heads >= 1 && r->kv_heads >= 0 && r->heads <= 16384 && r->kv_heads <= 16384, "%s: heads %d, kv_heads %d", who, r->heads, r->kv_heads);
  OSUD_CHECK_ARG(r->head_dim >= 2 && r->head_dim % 2 == 0 && r->head_dim <= 128, "%s: head_dim %d is not an even number up to 128", who, r->head_dim);
  OSUD_CHECK_ARG(r->rot_dim >= 0 && r->rot_dim % 2 == 0 && r->rot_dim <= r->head_dim, "%s: rot_dim %d is not an even number up to head_dim", who, r->rot_dim);
  OSUD_CHECK_ARG(!r->norm || r->eps > 0.f, "%s: eps must be positive", who);
  OSUD_CHECK_ARG(r->rows >= 0 && r->rows < (1L << 32), "%s: rows %ld", who, (long)r->rows);
  const int64_t wq = (int64_t)r->heads * r->head_dim, wk = (int64_t)r->kv_heads * r->head_dim;
  OSUD_CHECK_ARG(r->ld_q >= wq && r->ld_q_out >= wq && (!back || r->ld_dq >= wq), "%s: a row stride of the queries is shorter than their heads", who);
  OSUD_CHECK_ARG(r->ld_k >= wk && r->ld_k_out >= wk && (!back || r->ld_dk >= wk), "%s: a row stride of the keys is shorter than their heads", who);
  for (int64_t ld : {r->ld_q, r->ld_k, r->ld_q_out, r->ld_k_out, back ? r->ld_dq : 0, back ? r->ld_dk : 0})
    OSUD_CHECK_ARG(ld < (1L << 27), "%s: a row stride of %ld elements", who, (long)ld);
  if (r->rows > 0) {
    const size_t es = type_size(r->precision);
    const bool kv = r->kv_heads > 0;
    OSUD_CHECK_ARG(q && qo && (!back || gq) && (!kv || (k && ko && (!back || gk))), "%s: null argument", who);
    OSUD_CHECK_ARG(r->rot_dim == 0 || (r->positions && r->freqs), "%s: positions and freqs are needed to rotate", who);
    for (const void* x : {q, qo, gq, k, ko, gk}) OSUD_CHECK_ARG(reinterpret_cast<size_t>(x) % es == 0, "%s: a pointer is not aligned to its elements", who);
  }
  *p = RopeP{q, k, gq, gk, const_cast<void*>(qo), const_cast<void*>(ko), (size_t)r->ld_q, (size_t)r->ld_k, (size_t)r->ld_dq, (size_t)r->ld_dk, (size_t)r->ld_q_out,
             (size_t)r->ld_k_out, r->positions, r->freqs, r->norm ? r->q_weight : nullptr, r->norm ? r->k_weight : nullptr, nullptr, nullptr, nullptr, (long)r->rows,
             r->heads, r->kv_heads, r->head_dim, r->rot_dim, r->interleaved != 0, r->norm != 0, r->float_positions != 0, r->eps, r->gain};
  return OSUD_OK;
}

int doc_params(const char* who, const osud_doc_attention* a, bool back, DocAttnP* p) {
  OSUD_CHECK_ARG(a != nullptr, "%s: null argument", who);
  OSUD_TRY(check_precision(who, a->precision, back));
  OSUD_CHECK_ARG(a->heads >= 1 && a->kv_heads >= 1 && a->heads % a->kv_heads == 0 && a->heads <= 65536, "%s: heads %d is not a multiple of kv_heads %d", who, a->heads, a->kv_heads);
  OSUD_CHECK_ARG(a->head_dim >= 8 && a->head_dim % 8 == 0 && a->head_dim <= 128, "%s: head_dim %d is not a multiple of 8 up to 128", who, a->head_dim);
  OSUD_CHECK_ARG(a->cap == 0.f || a->cap * 1e4f >= a->scale, "%s: cap %g is below scale %g / 10^4", who, a->cap, a->scale);
  OSUD_CHECK_ARG(a->n_docs >= 0 && a->n_docs < (1 << 24) && a->rows_q >= 0 && a->rows_k >= 0 && a->rows_q < (1 << 30) && a->rows_k < (1 << 30), "%s: %d documents, %d query and %d key rows",
                 who, a->n_docs, a->rows_q, a->rows_k);
  OSUD_CHECK_ARG(a->scale > 0.f && a->scale < 1e18f && a->cap >= 0.f && a->cap < 1e18f, "%s: scale %g must be positive, cap %g not negative", who, a->scale, a->cap);
  OSUD_CHECK_ARG((a->n_docs == 0 && a->clear_rest == 0) || (a->q_begin && a->k_begin), "%s: null offsets", who);
  const int64_t unit = 16 / (int64_t)type_size(a->precision), wq = (int64_t)a->heads * a->head_dim, wk = (int64_t)a->kv_heads * a->head_dim;
  auto stride = [&](int64_t ld, int64_t w) { return ld >= w && ld % unit == 0 && ld < (1 << 23); };
  OSUD_CHECK_ARG(stride(a->ld_q, wq) && stride(a->ld_k, wk) && stride(a->ld_v, wk) && stride(a->ld_out, wq), "%s: a row stride is shorter than its heads or not a multiple of 16 bytes", who);
  OSUD_CHECK_ARG(!back || (stride(a->ld_d_out, wq) && stride(a->ld_dq, wq) && stride(a->ld_dk, wk) && stride(a->ld_dv, wk)),
                 "%s: a row stride is shorter than its heads or not a multiple of 16 bytes", who);
  const int G = a->heads / a->kv_heads;
  const int docs = a->n_docs + (a->clear_rest != 0);
  const int64_t tiles = ((int64_t)a->rows_q * G / 128 + docs) * a->kv_heads, ktiles = ((int64_t)a->rows_k / 128 + docs) * a->kv_heads;
  OSUD_CHECK_ARG((int64_t)a->rows_q * G < (1L << 31) - 128, "%s: %d query rows of %d shared heads", who, a->rows_q, G);
  OSUD_CHECK_ARG(tiles < (1 << 24) && ktiles < (1 << 24), "%s: too many tiles for one launch", who);
  DocAttnP z = {};
  z.ld_q = a->ld_q; z.ld_k = a->ld_k; z.ld_v = a->ld_v; z.ld_o = a->ld_out;
  z.ld_do = a->ld_d_out; z.ld_dq = a->ld_dq; z.ld_dk = a->ld_dk; z.ld_dv = a->ld_dv;
  z.q_begin = a->q_begin; z.k_begin = a->k_begin; z.prefix = a->prefix; z.slopes = a->slopes;
  z.rows_q = a->rows_q; z.rows_k = a->rows_k; z.n_real = a->n_docs; z.n_docs = docs; z.heads = a->heads; z.kv_heads = a->kv_heads; z.G = G; z.hd = a->head_dim;
  const int far = 1 << 30;  // (positions are smaller: no bound, and position +- bound stays inside 32 bits)
  z.left = a->left < 0 || a->left >= far ? -1 : a->left;
  z.right = a->right < 0 || a->right >= far ? -1 : a->right;
  z.slots = (int)((int64_t)a->rows_q * G / 128) + docs;
  z.split = 1;
  z.cus = device_cus();
  z.scale = a->scale;
  z.c1 = a->scale * kLog2e;
  z.cap = a->cap;
  if (a->cap > 0.f) {
    const double x = (double)a->scale / a->cap;
    z.c2 = (float)(2.0 * x * 1.4426950408889634);
    z.cap2 = a->cap * kLog2e;
    z.small = (float)(0.5 / x);
    const double four[5] = {0.999999463558197, -0.33326318860054016, 0.13190296292304993, -0.04440222680568695, 0.0};
    const double five[5] = {1.0, -0.3333306908607483, 0.13324779272079468, -0.05298607423901558, 0.017135007306933403};
    double power = x;
    for (int i = 0; i < 5; ++i, power *= x * x) {
      const double c = (a->precision == OSUD_PREC_F32 ? five : four)[i] * power;
      z.tanh1[i] = (float)c;
      z.tanh2[i] = (float)(c * a->cap * 1.4426950408889634);
    }
  }
  *p = z;
  return OSUD_OK;
}

}  // namespace

extern "C" size_t osud_op_qk_norm_rope_ws(int head_dim) { return head_dim > 0 && head_dim <= 128 ? rope_ws_floats(head_dim) : 0; }

extern "C" int osud_op_qk_norm_rope(const osud_rope* r, const void* q, const void* k, void* q_out, void* k_out, osud_stream stream) {
  RopeP p;
  OSUD_TRY(rope_params("op_qk_norm_rope", r, false, q, k, q_out, k_out, nullptr, nullptr, &p));
  if (p.rows == 0) return OSUD_OK;
  return launch_qk_norm_rope(r->precision, p, false, (hipStream_t)stream);
}

extern "C" int osud_op_qk_norm_rope_bwd(const osud_rope* r, const void* d_q_out, const void* d_k_out, const void* q, const void* k, void* dq, void* dk,
                                        float* dq_weight, float* dk_weight, float* ws, size_t ws_floats, osud_stream stream) {
  RopeP p;
  OSUD_TRY(rope_params("op_qk_norm_rope_bwd", r, true, q, k, dq, dk, d_q_out, d_k_out, &p));
  OSUD_CHECK_ARG(ws != nullptr || (dq_weight == nullptr && dk_weight == nullptr), "op_qk_norm_rope_bwd: weight gradients need a workspace");
  OSUD_CHECK_ARG(ws == nullptr || ws_floats >= rope_ws_floats(r->head_dim), "op_qk_norm_rope_bwd: workspace of %zu floats, %zu needed", ws_floats, rope_ws_floats(r->head_dim));
  if (p.rows == 0 && ws == nullptr) return OSUD_OK;
  if (dq_weight != nullptr || dk_weight != nullptr) p.ws = ws;
  p.dqw = dq_weight;
  p.dkw = dk_weight;
  if (p.rows == 0 && p.ws == nullptr) return OSUD_OK;
  return launch_qk_norm_rope(r->precision, p, true, (hipStream_t)stream);
}

extern "C" size_t osud_op_doc_attention_ws(const osud_doc_attention* a, int backward) {
  DocAttnP p;
  if (doc_params("op_doc_attention_ws", a, backward != 0, &p) != OSUD_OK) return 0;
  return backward ? doc_attn_bwd_ws(p, a->precision, a->max_q) : doc_attn_ws(p, a->precision, a->max_k);
}

extern "C" int osud_op_doc_attention(const osud_doc_attention* a, const void* q, const void* k, const void* v, void* out, float* lse, float* ws,
                                     size_t ws_floats, osud_stream stream) {
  DocAttnP p;
  OSUD_TRY(doc_params("op_doc_attention", a, false, &p));
  if (p.rows_q == 0 || p.n_docs == 0) return OSUD_OK;
  OSUD_CHECK_ARG(q && out && (p.rows_k == 0 || (k && v)), "op_doc_attention: null argument");
  OSUD_CHECK_ARG(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out) && aligned16(ws), "op_doc_attention: a pointer is not 16-byte aligned");
  p.q = q; p.k = k; p.v = v; p.out = out; p.lse = lse; p.ws_o = ws;
  return launch_doc_attn(a->precision, p, a->max_k, ws == nullptr ? 0 : ws_floats, (hipStream_t)stream);
}

extern "C" int osud_op_doc_attention_bwd(const osud_doc_attention* a, const void* q, const void* k, const void* v, const void* out, const float* lse,
                                         const void* d_out, void* dq, void* dk, void* dv, float* ws, size_t ws_floats, osud_stream stream) {
  DocAttnP p;
  OSUD_TRY(doc_params("op_doc_attention_bwd", a, true, &p));
  if (p.n_docs == 0 || (p.rows_q == 0 && p.rows_k == 0)) return OSUD_OK;
  OSUD_CHECK_ARG(p.rows_q == 0 || (q && out && lse && d_out && dq && ws), "op_doc_attention_bwd: null argument");
  OSUD_CHECK_ARG(p.rows_k == 0 || (k && v && dk && dv), "op_doc_attention_bwd: null argument");
  for (const void* x : {q, k, v, out, d_out, (const void*)dq, (const void*)dk, (const void*)dv, (const void*)ws})
    OSUD_CHECK_ARG(aligned16(x), "op_doc_attention_bwd: a pointer is not 16-byte aligned");
  const size_t need = 2 * (size_t)p.heads * p.rows_q;
  OSUD_CHECK_ARG(ws_floats >= need, "op_doc_attention_bwd: workspace of %zu floats, %zu needed", ws_floats, need);
  p.q = q; p.k = k; p.v = v; p.o = out; p.lse = const_cast<float*>(lse); p.d_o = d_out;
  p.dq = dq; p.dk = dk; p.dv = dv; p.delta = ws;
  return launch_doc_attn_bwd(a->precision, p, a->max_q, ws_floats, (hipStream_t)stream);
}
