// C ABI of the transformer-block operators (include/gradtts.h): argument checks and parameter blocks for
// battn_fwd.hip, battn_bwd.hip and rnorm.hip.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>
#include <vector>

#include "battn.h"
#include "decoder_internal.h"
#include "gradtts.h"
#include "rnorm.h"

using namespace gt;

namespace {

// whole number of any size as 32-bit digits, enough for products of small factors
struct Big {
  std::vector<uint32_t> d{1};
  void times(uint32_t m, int power) {
    for (; power > 0; --power) {
      uint64_t carry = 0;
      for (auto& x : d) {
        carry += (uint64_t)x * m;
        x = (uint32_t)carry;
        carry >>= 32;
      }
      if (carry) d.push_back((uint32_t)carry);
    }
  }
  bool at_least(const Big& o) const {
    if (d.size() != o.d.size()) return d.size() > o.d.size();
    for (size_t i = d.size(); i-- > 0;)
      if (d[i] != o.d[i]) return d[i] > o.d[i];
    return true;
  }
};

// first distance of the k-th far bucket, k >= 1: the least d with (d / exact)^far >= (max_distance / exact)^k. The
// floating-point root decides except within 1e-9 of a whole number (its own error is below 1e-12), where whole
// numbers do.
int border_of(int k, int exact, int far, int max_distance) {
  const double x = exact * std::pow((double)max_distance / exact, (double)k / far);
  const double n = std::nearbyint(x);
  if (std::fabs(x - n) > 1e-9 * x) return (int)std::ceil(x);
  Big a, b;
  a.times((uint32_t)n, far);
  a.times((uint32_t)exact, k);
  b.times((uint32_t)max_distance, k);
  b.times((uint32_t)exact, far);
  return a.at_least(b) ? (int)n : (int)n + 1;
}

const char* plan_buckets(int causal, int n_buckets, int max_distance, BaParams& p) {
  if (n_buckets < (causal ? 2 : 4) || n_buckets > BA_MAX_BUCKETS || (!causal && n_buckets % 2))
    return "n_buckets must lie in [2, 128] (bidirectional: even, >= 4)";
  p.nb = n_buckets;
  p.side = causal ? n_buckets : n_buckets / 2;
  p.exact = p.side / 2;
  const int far = p.side - p.exact;
  if (max_distance <= p.exact || max_distance > BA_MAX_DISTANCE)
    return "max_distance must exceed the buckets of single distances and be at most 1024";
  p.nborder = far - 1;
  for (int& x : p.border) x = INT32_MAX;
  for (int k = 1; k < far; ++k) p.border[k - 1] = border_of(k, p.exact, far, max_distance);
  p.dsat = p.nborder ? p.border[p.nborder - 1] : p.exact;
  return nullptr;
}

BaStride st(const gt_stride& s) { return {(long)s.b, (long)s.t, (long)s.h}; }
// rows on the 16-byte grid, 128 of them within 32-bit offsets
bool aligned(const void* p, const gt_stride& s, int es) {
  return s.t >= 0 && s.t < (1 << 21) && ((uintptr_t)p & 15) == 0 && (s.b * es) % 16 == 0 && (s.t * es) % 16 == 0 && (s.h * es) % 16 == 0;
}

constexpr int64_t kMaxT = 1 << 28;

const char* plan_attention(const gt_bucket_attention* a, BaParams& p) {
  if (a->dtype < GT_ELEM_F32 || a->dtype > GT_ELEM_F16) return "dtype must be GT_ELEM_F32, GT_ELEM_BF16 or GT_ELEM_F16";
  if (a->B < 0 || a->Tq < 0 || a->Tk < 0 || a->Tq > kMaxT || a->Tk > kMaxT || a->B > kMaxT)
    return "B, Tq, Tk must lie in [0, 2^28]";
  if (a->Hkv < 1 || a->Hq < 1 || a->Hq % a->Hkv || a->Hq > 65536) return "Hq must be a positive multiple of Hkv";
  if (a->D < 1 || a->D > BA_MAX_D) return "head size must lie in [1, 128]";
  if (!(a->scale >= 0x1p-20f && a->scale <= 0x1p20f)) return "scale must lie in [2^-20, 2^20]";
  p = BaParams{};
  if (const char* e = plan_buckets(a->causal != 0, a->n_buckets, a->max_distance, p)) return e;
  const int64_t rows_q = a->B * a->Tq, rows_k = a->B * a->Tk;
  if (!a->table || (rows_q && !a->q) || (rows_k && (!a->k || !a->v))) return "null tensor";
  p.q = a->q; p.k = a->k; p.v = a->v; p.table = a->table;
  p.qs = st(a->q_stride); p.ks = st(a->k_stride); p.vs = st(a->v_stride); p.os = st(a->out_stride);
  p.B = (int)a->B; p.Tq = (int)a->Tq; p.Tk = (int)a->Tk; p.Hq = (int)a->Hq; p.Hkv = (int)a->Hkv;
  p.G = (int)(a->Hq / a->Hkv); p.D = (int)a->D;
  p.causal = a->causal != 0;
  p.scale = a->scale; p.c = a->scale * 1.44269504088896341f; p.inv_scale = 1.f / a->scale;
  p.len = a->lengths; p.qlen = a->q_lengths; p.qstart = a->q_start;
  const int es = a->dtype == GT_ELEM_F32 ? 4 : 2;
  p.vec = a->D % 8 == 0 && aligned(a->q, a->q_stride, es) && aligned(a->k, a->k_stride, es) && aligned(a->v, a->v_stride, es);
  return nullptr;
}

const char* plan_norm(const gt_residual_norm* a, RnParams& p) {
  if (a->dtype < GT_ELEM_F32 || a->dtype > GT_ELEM_F16) return "dtype must be GT_ELEM_F32, GT_ELEM_BF16 or GT_ELEM_F16";
  if (a->B < 0 || a->T < 0 || a->B > 65535 || a->T > kMaxT) return "B must lie in [0, 65535], T in [0, 2^28]";
  if (a->C < 1 || a->C > RN_MAX_C) return "C must lie in [1, 8192]";
  if (!(a->eps >= 0.f) || !std::isfinite(a->eps) || !std::isfinite(a->scale)) return "eps must be >= 0, eps and scale finite";
  if (!a->post_weight || !a->pre_weight || (a->B * a->T && (!a->x || !a->y))) return "null tensor";
  if (a->gate_per_batch && !a->gate && a->B) return "gate_per_batch without a gate";
  p = RnParams{};
  p.x = a->x; p.y = a->y; p.gate = a->gate; p.w1 = a->post_weight; p.b1 = a->post_bias; p.w2 = a->pre_weight;
  p.b2 = a->pre_bias; p.B = (int)a->B; p.T = (int)a->T; p.C = (int)a->C; p.rms = a->rms != 0;
  p.gate_batch = a->gate_per_batch != 0; p.scale = a->scale; p.eps = a->eps; p.len = a->lengths;
  p.vec = a->C % 8 == 0 && (((uintptr_t)a->x | (uintptr_t)a->y) & 15) == 0;
  return nullptr;
}

int bad(const char* fn, const char* msg) { return gt_internal_fail(GT_ERR_ARG, std::string(fn) + ": " + msg); }
int done(const char* fn, hipError_t e) {
  return e == hipSuccess ? GT_OK : gt_internal_fail(GT_ERR_HIP, std::string(fn) + ": " + hipGetErrorString(e));
}

}  // namespace

extern "C" {

int gt_relative_bucket(int causal, int n_buckets, int max_distance, int64_t offset) try {
  BaParams p{};
  if (plan_buckets(causal != 0, n_buckets, max_distance, p)) return -1;
  const int64_t far = 1 << 20, o = offset < -far ? -far : offset > far ? far : offset;
  const int dist = causal ? (o < 0 ? (int)-o : 0) : (int)(o < 0 ? -o : o);
  int b = dist < p.exact ? dist : p.exact;
  for (int k = 0; k < p.nborder; ++k) b += dist >= p.border[k];
  return b + (!causal && o > 0 ? p.side : 0);
} catch (...) { return -1; }

size_t gt_bucket_attention_workspace_bytes(const gt_bucket_attention* a) try {
  BaParams p;
  return !a || plan_attention(a, p) ? 0 : ba_forward_ws(p, a->dtype);
} catch (...) { return 0; }

int gt_bucket_attention_forward(const gt_bucket_attention* a, void* out, float* lse, void* workspace,
                                size_t workspace_bytes, void* stream) try {
  const char* fn = "gt_bucket_attention_forward";
  if (!a) return bad(fn, "null argument");
  BaParams p;
  if (const char* e = plan_attention(a, p)) return bad(fn, e);
  if (a->B * a->Tq == 0) return GT_OK;
  if (!out) return bad(fn, "null tensor");
  const size_t need = ba_forward_ws(p, a->dtype);
  if (workspace_bytes < need || (need && !workspace)) return gt_internal_fail(GT_ERR_WORKSPACE, "workspace too small");
  p.out = out;
  p.lse = lse;
  p.vec = p.vec && aligned(out, a->out_stride, a->dtype == GT_ELEM_F32 ? 4 : 2);
  return done(fn, launch_ba_forward(p, a->dtype, workspace, (hipStream_t)stream));
} catch (...) { return GT_ERR_ARG; }

size_t gt_bucket_attention_backward_workspace_bytes(const gt_bucket_attention* a) try {
  BaParams p;
  return !a || plan_attention(a, p) ? 0 : ba_backward_ws(p, a->dtype);
} catch (...) { return 0; }

int gt_bucket_attention_backward(const gt_bucket_attention* a, const void* out, const float* lse,
                                 const gt_bucket_attention_grads* g, void* workspace, size_t workspace_bytes,
                                 void* stream) try {
  const char* fn = "gt_bucket_attention_backward";
  if (!a || !g) return bad(fn, "null argument");
  BaParams p;
  if (const char* e = plan_attention(a, p)) return bad(fn, e);
  if (!g->dtable || (a->B * a->Tq && (!out || !lse || !g->dout || !g->dq)) || (a->B * a->Tk && (!g->dk || !g->dv)))
    return bad(fn, "null tensor");
  if (!workspace || workspace_bytes < ba_backward_ws(p, a->dtype)) return gt_internal_fail(GT_ERR_WORKSPACE, "workspace too small");
  const int es = a->dtype == GT_ELEM_F32 ? 4 : 2;
  p.vec = p.vec && aligned(out, a->out_stride, es) && aligned(g->dout, g->dout_stride, es) && aligned(g->dq, g->dq_stride, es) &&
          aligned(g->dk, g->dk_stride, es) && aligned(g->dv, g->dv_stride, es);
  p.o = out; p.lse = const_cast<float*>(lse); p.dout = g->dout; p.dos = st(g->dout_stride);
  p.dq = g->dq; p.dk = g->dk; p.dv = g->dv; p.dtable = g->dtable;
  p.dqs = st(g->dq_stride); p.dks = st(g->dk_stride); p.dvs = st(g->dv_stride);
  return done(fn, launch_ba_backward(p, a->dtype, workspace, (hipStream_t)stream));
} catch (...) { return GT_ERR_ARG; }

int gt_residual_norm_forward(const gt_residual_norm* a, void* out, void* h, float* stats, void* stream) try {
  const char* fn = "gt_residual_norm_forward";
  if (!a) return bad(fn, "null argument");
  RnParams p;
  if (const char* e = plan_norm(a, p)) return bad(fn, e);
  if (a->B * a->T == 0) return GT_OK;
  if (!out || !h) return bad(fn, "null tensor");
  p.out = out; p.h = h; p.stats = stats;
  p.vec = p.vec && (((uintptr_t)out | (uintptr_t)h) & 15) == 0;
  return done(fn, launch_rn_forward(p, a->dtype, (hipStream_t)stream));
} catch (...) { return GT_ERR_ARG; }

size_t gt_residual_norm_backward_workspace_bytes(const gt_residual_norm* a) try {
  RnParams p;
  return !a || plan_norm(a, p) ? 0 : rn_backward_ws(p);
} catch (...) { return 0; }

int gt_residual_norm_backward(const gt_residual_norm* a, const float* stats, const gt_residual_norm_grads* g,
                              void* workspace, size_t workspace_bytes, void* stream) try {
  const char* fn = "gt_residual_norm_backward";
  if (!a || !g) return bad(fn, "null argument");
  RnParams p;
  if (const char* e = plan_norm(a, p)) return bad(fn, e);
  if (!g->dpost_weight || !g->dpre_weight || (a->B * a->T && (!stats || !g->dout || !g->dh || !g->dx || !g->dy)))
    return bad(fn, "null tensor");
  if ((g->dgate && !a->gate) || (g->dpost_bias && !a->post_bias) || (g->dpre_bias && !a->pre_bias))
    return bad(fn, "gradient of an absent parameter");
  if (!workspace || workspace_bytes < rn_backward_ws(p)) return gt_internal_fail(GT_ERR_WORKSPACE, "workspace too small");
  p.stats = const_cast<float*>(stats);
  p.dout = g->dout; p.dh = g->dh; p.dx = g->dx; p.dy = g->dy; p.dgate = g->dgate; p.dw1 = g->dpost_weight;
  p.db1 = g->dpost_bias; p.dw2 = g->dpre_weight; p.db2 = g->dpre_bias;
  p.vec = p.vec && (((uintptr_t)g->dout | (uintptr_t)g->dh | (uintptr_t)g->dx | (uintptr_t)g->dy) & 15) == 0;
  return done(fn, launch_rn_backward(p, a->dtype, workspace, (hipStream_t)stream));
} catch (...) { return GT_ERR_ARG; }

}  // extern "C"
