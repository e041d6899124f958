// C ABI of the attention layers' operators: block tables, rotary positions, cache writes and
// attention over a paged cache (the parts of attentionForward, src/model.zig:918-979, between
// its projections).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <vector>

#include "../../include/qmm.h"
#include "qmm_internal.h"
#include "qmm_launch.h"

using namespace qmm;

namespace {

Arr *arr(qmm_array a) { return (Arr *)a.ctx; }

// An int32 array of `dims` sizes (-1: any).
int check_int(const char *op, const char *name, const Arr *a, const std::vector<int> &dims) {
  if (!a) return fail("[%s] missing %s", op, name);
  if (a->dtype != QMM_INT32) return fail("[%s] %s must be int32", op, name);
  bool same = a->ndim == (int)dims.size();
  for (int i = 0; same && i < a->ndim; ++i) same = dims[i] < 0 || a->shape[i] == dims[i];
  if (!same) {
    std::string want;
    for (size_t i = 0; i < dims.size(); ++i)
      want += (i ? ", " : "") + (dims[i] < 0 ? std::string("any") : std::to_string(dims[i]));
    return fail("[%s] %s must be an array of shape [%s]", op, name, want.c_str());
  }
  return 0;
}

bool misaligned(const Arr *a) { return ((uintptr_t)a->data & 15) != 0; }

bool floating(const Arr *a) { return a->dtype == QMM_BFLOAT16 || a->dtype == QMM_FLOAT32; }

// [pages, heads, block, D] bfloat16, 16-byte aligned.
int check_cache(const char *op, const char *name, const Arr *a) {
  if (!a) return fail("[%s] missing %s", op, name);
  if (a->dtype != QMM_BFLOAT16 || a->ndim != 4)
    return fail("[%s] %s must be a bfloat16 array [pages, heads, block, D]", op, name);
  if (a->shape[1] < 1 || a->shape[2] < 1) return fail("[%s] %s needs heads and a block size", op, name);
  if ((double)a->shape[0] * a->shape[1] * a->shape[2] > UINT32_MAX)  // (they are counted in 32 bits)
    return fail("[%s] %s has over 2^32 - 1 keys", op, name);
  if (misaligned(a)) return fail("[%s] %s must be 16-byte aligned", op, name);
  return 0;
}

int check_head_dim(const char *op, int D) {
  if (D < 8 || D > 256 || D % 8)
    return fail("[%s] the head dimension must be a multiple of 8 from 8 to 256, got %d", op, D);
  return 0;
}

int check_freqs(const char *op, const Arr *f, int D) {
  if (!f) return fail("[%s] missing freqs", op);
  if (f->dtype != QMM_FLOAT32 || f->ndim != 1) return fail("[%s] freqs must be a 1D float32 array", op);
  if (2 * (int64_t)f->shape[0] > D)
    return fail("[%s] %d frequencies rotate more than the head's %d values", op, f->shape[0], D);
  return 0;
}

// [D] weights of a head norm, or the null handle.
int check_norm(const char *op, const char *name, const Arr *a, int D) {
  if (!a) return 0;
  if (!floating(a) || a->ndim != 1 || a->shape[0] != D)
    return fail("[%s] %s must be [%d], bfloat16 or float32", op, name, D);
  if (misaligned(a)) return fail("[%s] %s must be 16-byte aligned", op, name);
  return 0;
}

struct Shape {
  int ndim, dims[QMM_MAX_DIM];
};

// An array and the bytes that it takes.
struct Span {
  const Arr *a;
  uintptr_t lo, hi;
  Span(const Arr *x) : a(x), lo(x ? (uintptr_t)x->data : 0), hi(lo ? lo + x->nbytes() : 0) {}
};
bool overlap(const Span &x, const Span &y) { return x.lo < y.hi && y.lo < x.hi; }

// A result's handle before the call: none, one whose array serves as it is (see alloc_arr), or one that is replaced.
struct Result {
  const char *name;
  const qmm_array *res;
  Span cur;
  bool kept;
  Result(const char *n, const qmm_array *r, const Shape &s, qmm_dtype dtype) : name(n), res(r), cur(arr(*r)) {
    const Arr *a = cur.a;
    kept = cur.lo && a->dtype == dtype && a->ndim == s.ndim && std::equal(s.dims, s.dims + s.ndim, a->shape);
  }
};

// A result may not be the handle of an input that it would replace (the input would be freed before it is read), nor lie
// over an input, except exactly over one of `same`, which the kernels read before they write.
int check_result(const char *op, const Result &r, std::initializer_list<Span> inputs, std::initializer_list<const Arr *> same) {
  if (!r.cur.a) return 0;
  for (const Span &in : inputs) {
    if (!in.a) continue;
    if (!r.kept) {
      if (r.cur.a == in.a) return fail("[%s] %s is the handle of an input of another shape or type", op, r.name);
      continue;
    }
    if (!overlap(r.cur, in)) continue;
    bool ok = false;
    for (const Arr *x : same) ok = ok || (in.a == x && in.lo == r.cur.lo && in.hi == r.cur.hi);
    if (!ok) return fail("[%s] %s lies over an input", op, r.name);
  }
  return 0;
}

}  // namespace

extern "C" {

int qmm_rope_frequencies(float *out, float *amplitude, int rotary_dim, double base, qmm_rope_scaling sc) {
  const char *op = "rope_frequencies";
  if (!out) return finish(fail("[%s] null result pointer", op));
  if (rotary_dim < 2 || rotary_dim % 2) return finish(fail("[%s] the rotated part must be an even size, got %d", op, rotary_dim));
  if (!(base > 1)) return finish(fail("[%s] the base must be over 1", op));
  const bool scaled = sc.kind != QMM_ROPE_PLAIN;
  if (sc.kind < QMM_ROPE_PLAIN || sc.kind > QMM_ROPE_BANDS) return finish(fail("[%s] unknown scaling kind %d", op, (int)sc.kind));
  if (scaled && !(sc.factor >= 1)) return finish(fail("[%s] the scaling factor must be at least 1", op));
  const bool ramped = sc.kind == QMM_ROPE_RAMP || sc.kind == QMM_ROPE_BANDS;
  if (ramped && !(sc.original_len > 0)) return finish(fail("[%s] original_len must be positive", op));
  if (ramped && !(sc.fast > sc.slow && sc.slow > 0)) return finish(fail("[%s] needs fast > slow > 0", op));
  if (sc.kind == QMM_ROPE_BASE && rotary_dim == 2) return finish(fail("[%s] one pair has no base to change", op));
  const double tau = 6.283185307179586476925;
  const int half = rotary_dim / 2;
  if (sc.kind == QMM_ROPE_BASE) base *= std::pow(sc.factor, (double)rotary_dim / (rotary_dim - 2));
  // the pair (as a real number) that turns n times over the original length
  auto pair_of = [&](double n) { return half * std::log(sc.original_len / (n * tau)) / std::log(base); };
  double lo = 0, hi = 0;
  if (sc.kind == QMM_ROPE_RAMP) {
    lo = std::fmax(std::floor(pair_of(sc.fast)), 0.0);
    hi = std::fmin(std::ceil(pair_of(sc.slow)), (double)(rotary_dim - 1));
    if (hi <= lo) hi = lo + 0.001;
  }
  for (int i = 0; i < half; ++i) {
    double f = std::pow(base, -(double)i / half);
    if (sc.kind == QMM_ROPE_LINEAR) {
      f /= sc.factor;
    } else if (sc.kind == QMM_ROPE_RAMP) {
      const double u = std::fmin(std::fmax((i - lo) / (hi - lo), 0.0), 1.0);
      f = f * (1 - u) + f / sc.factor * u;
    } else if (sc.kind == QMM_ROPE_BANDS) {
      const double turns = sc.original_len * f / tau;
      const double u = std::fmin(std::fmax((turns - sc.slow) / (sc.fast - sc.slow), 0.0), 1.0);
      f = f / sc.factor * (1 - u) + f * u;
    }
    out[i] = (float)f;
  }
  if (amplitude) *amplitude = sc.kind == QMM_ROPE_RAMP ? (float)(0.1 * std::log(sc.factor) + 1) : 1.f;
  return finish(0);
}

int qmm_block_tables(qmm_array *table_out, qmm_array *head_out, qmm_array *q_starts, qmm_array *kv_lens,
                     qmm_array *positions, qmm_array *slots, qmm_array table, qmm_array head, qmm_array cached_lens,
                     qmm_array new_lens, qmm_array free_blocks, int block_size, int n_tokens, qmm_stream s) {
  begin_op();
  const char *op = "block_tables";
  if (!table_out || !head_out || !q_starts || !kv_lens || !positions || !slots)
    return finish(fail("[%s] null result pointer", op));
  Arr *ta = arr(table), *ha = arr(head), *ca = arr(cached_lens), *na = arr(new_lens), *fa = arr(free_blocks);
  if (check_int(op, "table", ta, {-1, -1})) return finish(1);
  const int R = ta->shape[0], W = ta->shape[1];
  if (check_int(op, "head", ha, {1}) || check_int(op, "cached_lens", ca, {R}) || check_int(op, "new_lens", na, {R}) ||
      check_int(op, "free_blocks", fa, {-1}))
    return finish(1);
  if (block_size < 1) return finish(fail("[%s] block_size must be positive, got %d", op, block_size));
  if (n_tokens < 0) return finish(fail("[%s] n_tokens must not be negative", op));
  if (R > BLOCK_TABLES_MAX_R) return finish(fail("[%s] %d requests: at most %d", op, R, BLOCK_TABLES_MAX_R));
  const Result out[] = {{"table_out", table_out, {2, {R, W}}, QMM_INT32}, {"head_out", head_out, {1, {1}}, QMM_INT32},
                        {"q_starts", q_starts, {1, {R + 1}}, QMM_INT32}, {"kv_lens", kv_lens, {1, {R}}, QMM_INT32},
                        {"positions", positions, {1, {n_tokens}}, QMM_INT32}, {"slots", slots, {1, {n_tokens}}, QMM_INT32}};
  const std::initializer_list<Span> inputs = {ta, ha, ca, na, fa};
  if (check_result(op, out[0], inputs, {ta}) || check_result(op, out[1], inputs, {ha}) ||
      check_result(op, out[2], inputs, {}) || check_result(op, out[3], inputs, {ca, na}) ||
      check_result(op, out[4], inputs, {}) || check_result(op, out[5], inputs, {}))
    return finish(1);
  for (const Result &o : out)
    for (const Result *p = out; p != &o; ++p)
      if (p->res == o.res || (o.cur.a && o.cur.a == p->cur.a) || (o.kept && p->kept && overlap(o.cur, p->cur)))
        return finish(fail("[%s] %s lies over %s", op, o.name, p->name));
  hipStream_t st = stream_of(s);
  Arr *to, *ho, *qo, *ko, *po, *so;
  if (alloc_arr(table_out, {R, W}, QMM_INT32, st, &to) || alloc_arr(head_out, {1}, QMM_INT32, st, &ho) ||
      alloc_arr(q_starts, {R + 1}, QMM_INT32, st, &qo) || alloc_arr(kv_lens, {R}, QMM_INT32, st, &ko) ||
      alloc_arr(positions, {n_tokens}, QMM_INT32, st, &po) || alloc_arr(slots, {n_tokens}, QMM_INT32, st, &so))
    return finish(1);
  BlockTableArgs a;
  a.R = R, a.W = W, a.T = n_tokens, a.F = fa->shape[0], a.block = block_size;
  a.table = (const int *)ta->data, a.head = (const int *)ha->data, a.cached = (const int *)ca->data;
  a.fresh = (const int *)na->data, a.free_blocks = (const int *)fa->data;
  a.table_out = (int *)to->data, a.head_out = (int *)ho->data, a.q_starts = (int *)qo->data;
  a.kv_lens = (int *)ko->data, a.positions = (int *)po->data, a.slots = (int *)so->data;
  hipError_t e = launch_block_tables(a, st);
  if (e != hipSuccess) return finish(fail_hip(e, op));
  return finish(0);
}

int qmm_rope(qmm_array *res, qmm_array x, qmm_array positions, qmm_array freqs, float amplitude, bool interleaved,
             bool transpose, qmm_stream s) {
  begin_op();
  const char *op = "rope";
  if (!res) return finish(fail("[%s] null result pointer", op));
  Arr *xa = arr(x), *pa = arr(positions), *fa = arr(freqs);
  if (!xa) return finish(fail("[%s] missing x", op));
  if (!floating(xa)) return finish(fail("[%s] x must be bfloat16 or float32", op));
  if (xa->ndim < 3) return finish(fail("[%s] x must be [..., T, H, D]", op));
  const int D = xa->shape[xa->ndim - 1], H = xa->shape[xa->ndim - 2];
  if (check_head_dim(op, D) || check_freqs(op, fa, D)) return finish(1);
  if (misaligned(xa)) return finish(fail("[%s] x must be 16-byte aligned", op));
  int64_t T = 1;
  for (int i = 0; i < xa->ndim - 2; ++i) T *= xa->shape[i];
  if (T > INT32_MAX) return finish(fail("[%s] too many tokens", op));
  if (check_int(op, "positions", pa, {(int)T})) return finish(1);
  Shape shape{xa->ndim, {}};
  std::copy(xa->shape, xa->shape + xa->ndim, shape.dims);
  if (check_result(op, {"the result", res, shape, xa->dtype}, {xa, pa, fa}, {xa})) return finish(1);
  hipStream_t st = stream_of(s);
  Arr *ya;
  if (alloc_arr(res, std::vector<int>(xa->shape, xa->shape + xa->ndim), xa->dtype, st, &ya)) return finish(1);
  if (misaligned(ya)) return finish(fail("[%s] the result must be 16-byte aligned", op));
  if (T == 0 || H == 0) return finish(0);
  RopeArgs a{};
  a.set[0] = RopeHeads{xa->data, ya->data, nullptr, H, D, 0, 1, 0};
  a.sets = 1, a.T = (int)T, a.D = D, a.half = fa->shape[0];
  a.in_f32 = a.out_f32 = xa->dtype == QMM_FLOAT32;
  a.interleaved = interleaved;
  a.amplitude = amplitude, a.sign = transpose ? -1.f : 1.f, a.eps = 0.f;
  a.positions = (const int *)pa->data, a.freqs = (const float *)fa->data;
  a.slots = nullptr, a.NB = 0, a.block = 1;
  hipError_t e = launch_rope(a, st);
  if (e != hipSuccess) return finish(fail_hip(e, op));
  return finish(0);
}

int qmm_rope_cache(qmm_array *q_out, qmm_array k_cache, qmm_array v_cache, qmm_array q, qmm_array k, qmm_array v,
                   qmm_array positions, qmm_array slots, qmm_array freqs, float amplitude, bool interleaved,
                   qmm_array q_norm, qmm_array k_norm, float norm_eps, qmm_stream s) {
  begin_op();
  const char *op = "rope_cache";
  if (!q_out) return finish(fail("[%s] null result pointer", op));
  Arr *kc = arr(k_cache), *vc = arr(v_cache), *qa = arr(q), *ka = arr(k), *va = arr(v), *pa = arr(positions),
      *sa = arr(slots), *fa = arr(freqs), *qn = arr(q_norm), *kn = arr(k_norm);
  if (check_cache(op, "k_cache", kc) || check_cache(op, "v_cache", vc)) return finish(1);
  const int NB = kc->shape[0], Hkv = kc->shape[1], block = kc->shape[2], D = kc->shape[3];
  for (int i = 0; i < 4; ++i)
    if (kc->shape[i] != vc->shape[i]) return finish(fail("[%s] k_cache and v_cache shapes differ", op));
  if (check_head_dim(op, D) || check_freqs(op, fa, D)) return finish(1);
  if (!qa || !ka || !va) return finish(fail("[%s] missing input", op));
  if (!floating(qa) || ka->dtype != qa->dtype || va->dtype != qa->dtype)
    return finish(fail("[%s] q, k, v must all be bfloat16 or all float32", op));
  if (qa->ndim != 3 || qa->shape[2] < D || qa->shape[2] % 8)
    return finish(fail("[%s] q must be [T, Hq, %d or more, a multiple of 8]", op, D));
  const int T = qa->shape[0], Hq = qa->shape[1];
  for (const Arr *x : {ka, va})
    if (x->ndim != 3 || x->shape[0] != T || x->shape[1] != Hkv || x->shape[2] != D)
      return finish(fail("[%s] k and v must be [%d, %d, %d]", op, T, Hkv, D));
  if (check_int(op, "positions", pa, {T}) || check_int(op, "slots", sa, {T})) return finish(1);
  if (check_norm(op, "q_norm", qn, D) || check_norm(op, "k_norm", kn, D)) return finish(1);
  if (misaligned(qa) || misaligned(ka) || misaligned(va))
    return finish(fail("[%s] q, k and v must be 16-byte aligned", op));
  const Arr *qc = arr(*q_out);
  if (qc && (qc == qa || (qc->data && qc->data == qa->data)) && (qa->shape[2] != D || qa->dtype != QMM_BFLOAT16))
    return finish(fail("[%s] q_out can be q's own array only at q's layout", op));
  if (check_result(op, {"q_out", q_out, {3, {T, Hq, D}}, QMM_BFLOAT16}, {qa, ka, va, kc, vc, pa, sa, fa, qn, kn}, {qa}))
    return finish(1);
  hipStream_t st = stream_of(s);
  Arr *qo;
  if (alloc_arr(q_out, {T, Hq, D}, QMM_BFLOAT16, st, &qo)) return finish(1);
  if (misaligned(qo)) return finish(fail("[%s] the result must be 16-byte aligned", op));
  if (T == 0) return finish(0);
  RopeArgs a{};
  a.set[0] = RopeHeads{qa->data, qo->data, qn ? qn->data : nullptr, Hq, qa->shape[2], qn && qn->dtype == QMM_FLOAT32, 1, 0};
  a.set[1] = RopeHeads{ka->data, kc->data, kn ? kn->data : nullptr, Hkv, D, kn && kn->dtype == QMM_FLOAT32, 1, 1};
  a.set[2] = RopeHeads{va->data, vc->data, nullptr, Hkv, D, 0, 0, 1};
  a.sets = 3, a.T = T, a.D = D, a.half = fa->shape[0];
  a.in_f32 = qa->dtype == QMM_FLOAT32, a.out_f32 = 0;
  a.interleaved = interleaved;
  a.amplitude = amplitude, a.sign = 1.f, a.eps = norm_eps;
  a.positions = (const int *)pa->data, a.slots = (const int *)sa->data, a.freqs = (const float *)fa->data;
  a.NB = NB, a.block = block;
  hipError_t e = launch_rope(a, st);
  if (e != hipSuccess) return finish(fail_hip(e, op));
  return finish(0);
}

int qmm_paged_attention(qmm_array *res, qmm_array q, qmm_array k_cache, qmm_array v_cache, qmm_array table,
                        qmm_array q_starts, qmm_array kv_lens, qmm_array gate, float scale, int window, qmm_stream s) {
  begin_op();
  const char *op = "paged_attention";
  if (!res) return finish(fail("[%s] null result pointer", op));
  Arr *qa = arr(q), *kc = arr(k_cache), *vc = arr(v_cache), *ta = arr(table), *sa = arr(q_starts), *la = arr(kv_lens),
      *ga = arr(gate);
  if (check_cache(op, "k_cache", kc) || check_cache(op, "v_cache", vc)) return finish(1);
  for (int i = 0; i < 4; ++i)
    if (kc->shape[i] != vc->shape[i]) return finish(fail("[%s] k_cache and v_cache shapes differ", op));
  const int NB = kc->shape[0], Hkv = kc->shape[1], block = kc->shape[2], D = kc->shape[3];
  if (check_head_dim(op, D)) return finish(1);
  if (!qa) return finish(fail("[%s] missing q", op));
  if (qa->dtype != QMM_BFLOAT16 || qa->ndim != 3 || qa->shape[2] != D)
    return finish(fail("[%s] q must be a bfloat16 array [T, Hq, %d]", op, D));
  const int T = qa->shape[0], Hq = qa->shape[1];
  if (Hq < 1 || Hq % Hkv) return finish(fail("[%s] %d query heads do not share %d key heads evenly", op, Hq, Hkv));
  if (check_int(op, "table", ta, {-1, -1})) return finish(1);
  const int R = ta->shape[0], W = ta->shape[1];
  if (check_int(op, "q_starts", sa, {R + 1}) || check_int(op, "kv_lens", la, {R})) return finish(1);
  if (R > ATTN_MAX_R) return finish(fail("[%s] %d requests: at most %d", op, R, ATTN_MAX_R));
  if (ga && (ga->dtype != QMM_BFLOAT16 || ga->ndim != 3 || ga->shape[0] != T || ga->shape[1] != Hq ||
             ga->shape[2] < D || ga->shape[2] % 8 || misaligned(ga)))
    return finish(fail("[%s] gate must be a 16-byte aligned bfloat16 array [%d, %d, %d or more, a multiple of 8]", op, T,
                       Hq, D));
  if (window < 0) return finish(fail("[%s] window must not be negative, got %d", op, window));
  if (!std::isfinite(scale)) return finish(fail("[%s] scale must be finite", op));
  if (misaligned(qa)) return finish(fail("[%s] q must be 16-byte aligned", op));
  AttnArgs a;
  a.q = (const uint16_t *)qa->data, a.k = (const uint16_t *)kc->data, a.v = (const uint16_t *)vc->data;
  a.gate = ga ? (const uint16_t *)ga->data : nullptr;
  a.table = (const int *)ta->data, a.q_starts = (const int *)sa->data, a.kv_lens = (const int *)la->data;
  a.T = T, a.R = R, a.W = W, a.Hq = Hq, a.Hkv = Hkv, a.D = D, a.Dg = ga ? ga->shape[2] : 0;
  a.NB = NB, a.block = block, a.window = window, a.scale = scale;
  const char *too_much = attention_limits(a);
  if (too_much) return finish(fail("[%s] too many %s", op, too_much));
  if (check_result(op, {"the result", res, {3, {T, Hq, D}}, QMM_BFLOAT16}, {qa, kc, vc, ta, sa, la, ga}, {qa, ga}))
    return finish(1);
  hipStream_t st = stream_of(s);
  Arr *oa;
  if (alloc_arr(res, {T, Hq, D}, QMM_BFLOAT16, st, &oa)) return finish(1);
  if (misaligned(oa)) return finish(fail("[%s] the result must be 16-byte aligned", op));
  if (T == 0) return finish(0);
  a.o = (uint16_t *)oa->data;
  Scratch scratch;
  const size_t need = attention_workspace(a);
  if (need && scratch.take(st, need)) return finish(1);
  hipError_t e = launch_attention(a, scratch.get(), st);
  if (e != hipSuccess) return finish(fail_hip(e, op));
  return finish(0);
}

}  // extern "C"
