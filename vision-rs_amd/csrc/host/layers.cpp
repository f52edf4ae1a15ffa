// C-ABI entry points of the transformer-layer operators (include/vrs.h): RMS
// norm, rotary positions, attention over packed sequences.  Each checks its
// arguments, picks a kernel instance and launches it on the caller's stream.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <tuple>

#include "layers.h"

using namespace vrs;

extern "C" {

int vrs_rms_norm(vrs_ctx* ctx, const vrs_rms_desc* d, const void* x, const void* res, const float* weight, void* sum,
                 void* y, float* scales, void* stream) {
  const char* me = "vrs_rms_norm";
  if (!ctx || !d) return fail(VRS_EINVAL, "%s: null argument", me);
  int rc = check_type(d->dtype, me);
  if (rc) return rc;
  const bool f8 = d->y_dtype == VRS_FP8;
  if (!f8 && d->y_dtype != d->dtype)
    return fail(VRS_EUNSUPPORTED, "%s: y_dtype %d (dtype %d or VRS_FP8)", me, d->y_dtype, d->dtype);
  if (d->rows < 0 || d->cols < 1) return fail(VRS_EBADSHAPE, "%s: %d rows of %d columns", me, d->rows, d->cols);
  if (d->cols > 32768) return fail(VRS_EUNSUPPORTED, "%s: %d columns (up to 32768)", me, d->cols);
  if (!(d->eps > 0.f) || std::isinf(d->eps)) return fail(VRS_EINVAL, "%s: eps %g", me, (double)d->eps);
  if (d->rows == 0) return VRS_OK;      // empty tensors may have null addresses
  const size_t es = elt_size(d->dtype);
  if ((rc = check_ptr(x, es, me, "x")) || (rc = check_ptr(weight, 4, me, "weight")) ||
      (rc = check_ptr(y, f8 ? 1 : es, me, "y")))
    return rc;
  if ((res && (rc = check_ptr(res, es, me, "res"))) || (sum && (rc = check_ptr(sum, es, me, "sum")))) return rc;
  if (sum == y) return fail(VRS_EINVAL, "%s: sum and y are one buffer", me);
  if (f8 && (x == y || res == y)) return fail(VRS_EINVAL, "%s: an e4m3 y over an input", me);
  // outputs must not fold rows onto each other; inputs may (a stride of 0 repeats a row)
  for (int64_t s : {d->x_ld, d->res_ld, d->sum_ld, d->y_ld})
    if (s < 0 || s >> 40) return fail(VRS_EBADSHAPE, "%s: row stride %lld", me, (long long)s);
  if (d->y_ld < d->cols || (sum && d->sum_ld < d->cols))
    return fail(VRS_EBADSHAPE, "%s: row strides", me);
  for (const auto& [p, ld, name] : {std::tuple<const void*, int64_t, const char*>{x, d->x_ld, "x"}, {res, d->res_ld, "res"}})
    if (p && ((p == y && ld != d->y_ld) || (p == sum && ld != d->sum_ld)))
      return fail(VRS_EBADSHAPE, "%s: %s is an output with another row stride", me, name);
  const int vec = 16 / (int)es;
  auto fits = [&](const void* p, int64_t ld) { return !p || (aligned(p, 16) && ld % vec == 0); };
  bool wide = d->cols % vec == 0 && fits(x, d->x_ld) && fits(res, d->res_ld) && fits(sum, d->sum_ld);
  if (f8) {
    if (d->group == 0) {
      int e;
      if (!(d->out_step >= 1e-30f && d->out_step <= 1e30f) || std::frexp(d->out_step, &e) != 0.5f)
        return fail(VRS_EINVAL, "%s: out_step %g must be a positive power of two", me, (double)d->out_step);
    } else {
      if (d->group != d->cols && d->group != 32 && d->group != 64 && d->group != 128)
        return fail(VRS_EUNSUPPORTED, "%s: group %d (0, 32, 64, 128 or all %d columns)", me, d->group, d->cols);
      if (d->cols % d->group) return fail(VRS_EBADSHAPE, "%s: %d columns in groups of %d", me, d->cols, d->group);
      if ((rc = check_ptr(scales, 4, me, "scales"))) return rc;
    }
    if (!wide || d->cols % 16 || !aligned(y, 16) || d->y_ld % 16)
      return fail(VRS_EBADSHAPE, "%s: e4m3 needs 16-byte aligned rows and a multiple of 16 columns", me);
  } else {
    if (d->group) return fail(VRS_EINVAL, "%s: group %d without VRS_FP8", me, d->group);
    wide = wide && fits(y, d->y_ld);
  }

  // The fewest threads that hold a row in at most four vectors each: a row up to 256 vectors (bf16
  // 2048, float32 1024 columns) in one wave, whose sums need no barrier; over 1024 vectors in LDS.
  struct Shape { int tpr, nv; };
  static const Shape kWide[] = {{64, 1}, {64, 2}, {64, 4}, {256, 2}, {256, 4}, {0, 0}};
  static const Shape kOne[] = {{64, 4}, {256, 4}, {0, 0}};
  const int v = wide ? vec : 1, chunks = (d->cols + v - 1) / v;
  const Shape* sh = wide ? kWide : kOne;
  while (sh->tpr && sh->tpr * sh->nv < chunks) ++sh;
  char name[64];
  const char* out = f8 ? "e4m3" : "same";
  if (sh->tpr) snprintf(name, sizeof name, "vrs_rms_%s_%s_%dx%d_v%d", dsuffix(d->dtype), out, sh->tpr, sh->nv, v);
  else snprintf(name, sizeof name, "vrs_rms_%s_%s_wide%dk_v%d", dsuffix(d->dtype), out, d->cols <= 16384 ? 16 : 32, v);
  vrs_rms_args a{};
  a.x = x; a.res = res; a.weight = weight; a.sum = sum; a.y = y; a.scales = scales;
  a.x_ld = d->x_ld; a.res_ld = d->res_ld; a.sum_ld = d->sum_ld; a.y_ld = d->y_ld;
  a.rows = d->rows; a.cols = d->cols; a.eps = d->eps;
  a.group = f8 ? d->group : 0;
  a.inv_step = f8 && d->group == 0 ? 1.f / d->out_step : 1.f;
  const int wg = sh->tpr ? 256 : 1024, rpw = sh->tpr ? wg / sh->tpr : 1;
  const int64_t steps = ((int64_t)d->rows + rpw - 1) / rpw;
  // workgroups that walk the rows: four to a CU (8192 rows of 4096: 42.4 us; three 42.0, eight 45.3)
  const int64_t resident = sh->tpr ? 1024 : 512;
  return launch(ctx, name, dim3((unsigned)std::min(steps, resident)), dim3(wg), 0, &a, stream);
}

int vrs_rope_freqs(int32_t pairs, double base, int32_t scaling, double factor, double low, double high,
                   double orig_len, double* out) {
  const char* me = "vrs_rope_freqs";
  if (!out) return fail(VRS_EINVAL, "%s: null out", me);
  if (pairs < 1 || pairs > 256) return fail(VRS_EBADSHAPE, "%s: %d pairs (1..256)", me, pairs);
  if (!(base > 1.0) || std::isinf(base)) return fail(VRS_EINVAL, "%s: base %g", me, base);
  if (scaling < VRS_ROPE_PLAIN || scaling > VRS_ROPE_BY_INDEX) return fail(VRS_EINVAL, "%s: scaling %d", me, scaling);
  if (scaling != VRS_ROPE_PLAIN && (!(factor > 0.0) || std::isinf(factor)))
    return fail(VRS_EINVAL, "%s: factor %g", me, factor);
  if (scaling >= VRS_ROPE_BY_TURNS && (!(low > 0.0) || !(high > low) || std::isinf(high) || !(orig_len >= 1.0) || std::isinf(orig_len)))
    return fail(VRS_EINVAL, "%s: turns %g .. %g over %g positions", me, low, high, orig_len);
  // pair index whose frequency makes t turns over orig_len positions
  auto index_of = [&](double t) { return pairs * std::log(orig_len / (t * 2.0 * M_PI)) / std::log(base); };
  for (int i = 0; i < pairs; ++i) {
    const double f = std::pow(base, -(double)i / pairs) / (2.0 * M_PI);
    double keep = 1.0;      // share of the unscaled frequency
    if (scaling == VRS_ROPE_LINEAR) keep = 0.0;
    if (scaling == VRS_ROPE_BY_TURNS) keep = std::clamp((f * orig_len - low) / (high - low), 0.0, 1.0);
    if (scaling == VRS_ROPE_BY_INDEX) {
      const double from = std::max(std::floor(index_of(high)), 0.0);
      const double to = std::max(std::min(std::ceil(index_of(low)), 2.0 * pairs - 1.0), from + 1e-3);
      keep = 1.0 - std::clamp((i - from) / (to - from), 0.0, 1.0);
    }
    out[i] = f * keep + f / (scaling == VRS_ROPE_PLAIN ? 1.0 : factor) * (1.0 - keep);
  }
  return VRS_OK;
}

int vrs_rope(vrs_ctx* ctx, const vrs_rope_desc* d, const vrs_seqs* seqs, const double* freq, const int32_t* positions,
             const void* q, const void* k, const void* v, void* q_out, void* k_out, void* v_out, void* stream) {
  const char* me = "vrs_rope";
  if (!ctx || !d) return fail(VRS_EINVAL, "%s: null argument", me);
  int rc = check_type(d->dtype, me);
  if (rc) return rc;
  if (d->rows < 0 || d->heads < 0 || d->kv_heads < 0 || d->heads + (int64_t)d->kv_heads < 1 || d->k_out_rows < 0)
    return fail(VRS_EBADSHAPE, "%s: %d rows, %d + %d heads", me, d->rows, d->heads, d->kv_heads);
  if (d->head_dim < 1 || d->head_dim > 4096 || d->rot < 2 || d->rot % 2 || d->rot > d->head_dim || d->rot > 512)
    return fail(VRS_EBADSHAPE, "%s: rot %d of head_dim %d", me, d->rot, d->head_dim);
  if (d->layout != VRS_ROPE_HALF && d->layout != VRS_ROPE_PAIRS) return fail(VRS_EINVAL, "%s: layout %d", me, d->layout);
  if (!std::isfinite(d->scale)) return fail(VRS_EINVAL, "%s: scale", me);
  if (d->axes < 1 || d->axes > 4 || (d->axes > 1 && !positions))
    return fail(VRS_EINVAL, "%s: %d axes%s", me, d->axes, positions ? "" : " without positions");
  vrs_rope_args a{};
  int64_t end = 0;
  for (int i = 0; i < d->axes; ++i) {
    if (d->axis_pairs[i] < 0) return fail(VRS_EBADSHAPE, "%s: axis_pairs", me);
    end += d->axis_pairs[i];
    if (i < 3) a.axis_end[i] = i + 1 < d->axes ? (int32_t)std::min<int64_t>(end, d->rot) : d->rot;
  }
  for (int i = d->axes; i < 3; ++i) a.axis_end[i] = d->rot;
  if (end != d->rot / 2) return fail(VRS_EBADSHAPE, "%s: axes of %lld pairs, rot %d", me, (long long)end, d->rot);
  if (seqs && (rc = check_seqs(seqs, me))) return rc;
  if (d->rows == 0 || (seqs && seqs->n == 0)) return VRS_OK;      // empty tensors may have null addresses
  const size_t es = elt_size(d->dtype);
  if ((rc = check_ptr(freq, 8, me, "freq"))) return rc;
  if (positions && (rc = check_ptr(positions, 4, me, "positions"))) return rc;
  if (positions && d->pos_ld < d->rows) return fail(VRS_EBADSHAPE, "%s: pos_ld", me);
  if (d->heads && ((rc = check_ptr(q, es, me, "q")) || (rc = check_ptr(q_out, es, me, "q_out")))) return rc;
  if (d->kv_heads && ((rc = check_ptr(k, es, me, "k")) || (rc = check_ptr(k_out, es, me, "k_out")))) return rc;
  if (v && (!d->kv_heads || (rc = check_ptr(v, es, me, "v")) || (rc = check_ptr(v_out, es, me, "v_out"))))
    return rc ? rc : fail(VRS_EINVAL, "%s: v without kv_heads", me);
  if (d->kv_heads && !seqs && d->k_out_rows < d->rows)
    return fail(VRS_EBADSHAPE, "%s: %d rows into k_out's %d", me, d->rows, d->k_out_rows);
  for (int64_t s : {d->q_ld, d->q_hd, d->k_ld, d->k_hd, d->v_ld, d->v_hd, d->qo_ld, d->qo_hd, d->ko_ld, d->ko_hd,
                    d->vo_ld, d->vo_hd})
    if (s < 0 || s >> 40) return fail(VRS_EBADSHAPE, "%s: stride %lld", me, (long long)s);
  // Rows that go where k_start says may leave gaps between sequences in which other heads lie (a cache with
  // the heads outside each sequence's rows): there the strides alone show no fold, but of one row or one head.
  auto folds = [&](int64_t ld, int64_t hd) {
    if (seqs && seqs->k_start)
      return (d->k_out_rows > 1 && ld < d->head_dim) || (d->kv_heads > 1 && hd < d->head_dim);
    return !apart(ld, hd, d->k_out_rows, d->kv_heads, d->head_dim);
  };
  if ((d->heads && !apart(d->qo_ld, d->qo_hd, d->rows, d->heads, d->head_dim)) ||
      (d->kv_heads && folds(d->ko_ld, d->ko_hd)) || (v && folds(d->vo_ld, d->vo_hd)))
    return fail(VRS_EBADSHAPE, "%s: output strides fold rows or heads onto each other", me);
  if (d->heads && q == q_out && (d->q_ld != d->qo_ld || d->q_hd != d->qo_hd))
    return fail(VRS_EBADSHAPE, "%s: q_out is q with other strides", me);
  const bool moves = seqs && (seqs->k_start || seqs->k_len);
  if (d->kv_heads && k == k_out && (moves || d->k_ld != d->ko_ld || d->k_hd != d->ko_hd))
    return fail(VRS_EBADSHAPE, "%s: k_out is k, but rows move or strides differ", me);
  if (v && v == v_out) return fail(VRS_EINVAL, "%s: v_out is v", me);

  // the widest vector that divides the pairs, the head and every stride
  int vec = 16 / (int)es;
  auto fits = [&](int n) {
    const size_t bytes = n * es;
    bool ok = d->rot / 2 % n == 0 && d->head_dim % n == 0;
    auto one = [&](const void* p, int64_t ld, int64_t hd) { ok = ok && aligned(p, bytes) && ld % n == 0 && hd % n == 0; };
    if (d->heads) one(q, d->q_ld, d->q_hd), one(q_out, d->qo_ld, d->qo_hd);
    if (d->kv_heads) one(k, d->k_ld, d->k_hd), one(k_out, d->ko_ld, d->ko_hd);
    if (v) one(v, d->v_ld, d->v_hd), one(v_out, d->vo_ld, d->vo_hd);
    return ok;
  };
  while (vec > 1 && !fits(vec)) vec = vec == 8 ? 4 : 1;
  a.q = q; a.k = k; a.v = v; a.qo = q_out; a.ko = k_out; a.vo = v_out;
  a.freq = freq; a.pos = positions;
  if (seqs) a.s.q_start = seqs->q_start, a.s.k_start = seqs->k_start, a.s.k_len = seqs->k_len, a.s.n = seqs->n;
  a.s.q_rows = d->rows; a.s.k_rows = d->kv_heads ? d->k_out_rows : 0x7fffffff;
  a.q_ld = d->q_ld; a.q_hd = d->q_hd; a.k_ld = d->k_ld; a.k_hd = d->k_hd; a.v_ld = d->v_ld; a.v_hd = d->v_hd;
  a.qo_ld = d->qo_ld; a.qo_hd = d->qo_hd; a.ko_ld = d->ko_ld; a.ko_hd = d->ko_hd; a.vo_ld = d->vo_ld; a.vo_hd = d->vo_hd;
  a.pos_ld = d->pos_ld;
  a.rows = d->rows; a.heads = d->heads; a.kv = d->kv_heads; a.dim = d->head_dim; a.rot = d->rot;
  a.pairs_layout = d->layout == VRS_ROPE_PAIRS;
  a.scale = d->scale;
  if ((int64_t)std::max(d->heads, d->kv_heads) * d->head_dim >= 1 << 24)    // the kernels' divisions are exact below
    return fail(VRS_EUNSUPPORTED, "%s: heads of %d elements", me, d->head_dim);
  // a wave to a row once they fill the card twice, else four
  const int wpr = d->rows >= 2048 ? 1 : 4, rpw = 4 / wpr;
  const int64_t blocks = ((int64_t)d->rows + rpw - 1) / rpw;
  if (blocks >= (1ll << 32) / 256) return fail(VRS_EBADSHAPE, "%s: %d rows", me, d->rows);
  char name[64];
  snprintf(name, sizeof name, "vrs_rope_%s_v%d_w%d", dsuffix(d->dtype), vec, wpr);
  return launch(ctx, name, dim3((unsigned)blocks), dim3(256), 0, &a, stream);
}

}  // extern "C"

namespace vrs {

int check_attention(const vrs_attention_desc* d, const vrs_seqs* seqs, const char* me) {
  if (!d || !seqs) return fail(VRS_EINVAL, "%s: null argument", me);
  int rc = check_type(d->dtype, me);
  if (rc || (rc = check_seqs(seqs, me))) return rc;
  if (d->q_rows < 0 || d->k_rows < 0 || d->heads < 1 || d->kv_heads < 1 || d->heads % d->kv_heads)
    return fail(VRS_EBADSHAPE, "%s: %d and %d rows, %d heads on %d", me, d->q_rows, d->k_rows, d->heads, d->kv_heads);
  // the kernels' key numbers run on to the end of the tiles ahead, 512 at most past the last key
  if (d->k_rows > 0x7fffffff - 1023) return fail(VRS_EUNSUPPORTED, "%s: %d key rows", me, d->k_rows);
  if (d->head_dim < 8 || d->head_dim % 8 || d->head_dim > 128)
    return fail(VRS_EUNSUPPORTED, "%s: head_dim %d (a multiple of 8 up to 128)", me, d->head_dim);
  if (!(d->scale >= 0.f && d->scale <= 1e30f)) return fail(VRS_EINVAL, "%s: scale %g", me, (double)d->scale);
  const int vec = 16 / (int)elt_size(d->dtype);
  for (int64_t s : {d->q_ld, d->q_hd, d->k_ld, d->k_hd, d->v_ld, d->v_hd, d->o_ld, d->o_hd})
    if (s < 0 || s >> 40 || s % vec) return fail(VRS_EBADSHAPE, "%s: stride %lld (multiples of 16 bytes)", me, (long long)s);
  for (int64_t s : {d->q_ld, d->k_ld, d->v_ld, d->o_ld})
    if (s >= (1 << 22)) return fail(VRS_EUNSUPPORTED, "%s: row stride %lld", me, (long long)s);
  if (!apart(d->o_ld, d->o_hd, d->q_rows, d->heads, d->head_dim))
    return fail(VRS_EBADSHAPE, "%s: output strides fold rows or heads onto each other", me);
  return VRS_OK;
}

int check_attention_buffers(const vrs_attention_desc* d, const void* q, const void* k, const void* v, const void* out,
                            const char* me) {
  for (const auto& [p, name] : {std::pair<const void*, const char*>{q, "q"}, {k, "k"}, {v, "v"}, {out, "out"}}) {
    if (!p && (d->k_rows || name[0] == 'q' || name[0] == 'o')) return fail(VRS_EINVAL, "%s: null %s", me, name);
    if (!aligned(p, 16)) return fail(VRS_EBADSHAPE, "%s: %s must be 16-byte aligned", me, name);
  }
  if ((d->k_rows && (out == k || out == v)) || (out == q && (d->o_ld != d->q_ld || d->o_hd != d->q_hd)))
    return fail(VRS_EINVAL, "%s: out is an input", me);
  return VRS_OK;
}

}  // namespace vrs

namespace {

// Which kernel, and into how many parts the keys are split.
struct AttentionPlan {
  bool few;
  int qt, waves;          // 32-row tiles of a wave (prompts), waves of a workgroup
  int parts;
  int64_t row_tiles;      // few: 32-row tiles of the longest sequence; prompts: ids of row tiles
};
AttentionPlan plan_attention(const vrs_attention_desc* d, const vrs_seqs* s) {
  const int64_t group = d->heads / d->kv_heads;
  // (unknown: as if all sequences were of one length)
  const int64_t n = std::max(s->n, 1);
  const int64_t mq = std::max<int64_t>(1, s->max_q > 0 ? std::min(s->max_q, d->q_rows) : (d->q_rows + n - 1) / n);
  const int64_t mk = s->max_k > 0 ? std::min(s->max_k, d->k_rows) : (d->k_rows + n - 1) / n;
  AttentionPlan p;
  p.qt = 1;
  p.waves = 4;
  // Rows of a key head that fit one row tile, or two of them where that still leaves workgroups few, or in
  // float32; the prompts' kernel takes 128 rows and more.  Measured against it, 8 key heads of 128, bfloat16:
  // one token of 64 sequences over 500 .. 8000 keys 250 us against 305, over 8000 each 425 against 509, over
  // 2000 each 121 against 94; of one over 2000 17.1 against 17.7.  64 rows (16 queries of 4 heads) over 2000
  // keys: one sequence 17.5 against 18.2, 8 30.5 against 26.2, 64 281 against 97.  float32: the 64 tokens 537
  // against 2418, 64 rows of 64 sequences 496 against 532.
  p.few = mq * group <= 32 || (mq * group <= 64 && (n * d->kv_heads <= 64 || d->dtype == VRS_F32));
  if (p.few) {
    p.row_tiles = (mq * group + 31) / 32;
    // Workgroups of four waves, two on a CU at once: two of each wherever there are enough keys for 192
    // a part.  bfloat16, bound by memory, takes four parts beyond that, so that long and short sequences
    // even out; float32, bound by the matrix instructions that most of a row tile spends on no row, does
    // not gain.  Measured, head_dim 128, 8 key heads: bfloat16, 64 tokens over 500 .. 8000 keys, 512
    // workgroups: 1 part 278 us, 2 246, 4 236, 8 254; one token, 4000 keys: 192 keys a part 14.5 us, 256
    // 16.5, 384 16.8.  float32, the same 64 tokens: 1 part 475 us, 2 516, 4 574; 64 over 500 .. 2000: 1 183,
    // 2 209, 4 246; 16 over 500 .. 8000: 2 208, 4 158, 8 166; one, 4000 keys: 128 keys a part 36 us, 192 30.
    const int64_t wgs = std::max<int64_t>(1, n * d->kv_heads * p.row_tiles);
    const int64_t least = d->dtype == VRS_BF16 ? 4 : 1;
    p.parts = (int)std::clamp<int64_t>(std::min(std::max(least, 512 / wgs), mk / 192), 1, 64);
    // short ones: eight waves and no second launch (head_dim 128, 300 keys: 9.6 us against 10.2, 700:
    // 13.7 against 12.6; head_dim 64, 700: 8.5 against 9.5)
    if (d->dtype == VRS_BF16 && wgs <= 256 && mk * (d->head_dim <= 64 ? 64 : 128) <= 1 << 16) p.waves = 8, p.parts = 1;
  } else {
    // row tiles at most: whole ones of all rows and a part of one to each sequence
    auto count = [&](int64_t bm) {
      return std::min(d->q_rows * group / bm + s->n, s->n * ((mq * group + bm - 1) / bm));
    };
    // 256 rows to a workgroup where key tiles are many (fewer reads of them; measured at head_dim 128,
    // causal 8192 keys: 516 us against 545; causal up to 2800 keys, where more of a tile is masked:
    // 198 against 189) and there are such workgroups for every CU.
    const int64_t keys = std::max<int64_t>(1, d->causal ? mk - mq / 2 : mk);    // of a row, in the mean
    const bool f32 = d->dtype == VRS_F32, small = d->head_dim <= 64;
    if (keys >= 2048 && count(256) * d->kv_heads >= (small ? 512 : 256)) {
      if (!f32 && small) p.qt = 2;
      else p.waves = 8;
    }
    const int64_t bm = 32 * p.qt * p.waves;
    p.row_tiles = d->q_rows * group / bm + (int64_t)s->n;
    // Parts: CUs take whole workgroups, so few of them leave CUs idle in the last round; a CU with one
    // workgroup of 4 waves is slower than its share of two (bfloat16: 0.6, where a wave waits for
    // itself; float32, bound by its matrix instructions, 0.95); each part more costs its unfinished
    // rows' way through memory, and the first a second launch.  Times in us: 32 keys of a workgroup at
    // the rates measured, 4 TB/s, 4 us.  Measured, four pieces of 100 .. 300 queries over 2000 .. 9000
    // keys: 1 part 207, 2 165, 3 192, 4 175; two maps of 1369 in float32: 1 101, 2 107, 3 84, 4 92.
    const double wgs = std::max(1.0, (double)count(bm) * (double)d->kv_heads);
    const double step = bm / 128.0 * (f32 ? (small ? 2.1 : 4.1) : (small ? 0.32 : 0.51));
    const double alone = p.waves * p.qt > 4 ? 1.0 : f32 ? 0.95 : 0.6;
    const double rows = (double)std::min((int64_t)d->q_rows, s->n * mq) * d->heads;
    double best = 0;
    for (int i = 1; i <= 16 && (i == 1 || keys / i >= 128); ++i) {
      const double on_cu = std::ceil(wgs * i / 256.0), odd = std::fmod(on_cu, 2.0);
      const double t = (on_cu - odd + odd / alone) * std::ceil((double)keys / i / 32.0) * step +
                       (i > 1 ? 4.0 + 2.0 * i * rows * (d->head_dim + 2) * 4 / 4e6 : 0.0);
      if (i == 1 || t < best) best = t, p.parts = i;
    }
  }
  return p;
}
size_t attention_bytes(const vrs_attention_desc* d, const AttentionPlan& p) {
  return p.parts == 1 ? 0 : (size_t)p.parts * d->q_rows * d->heads * (d->head_dim + 2) * 4;
}

}  // namespace

extern "C" {

size_t vrs_attention_workspace_size(const vrs_attention_desc* d, const vrs_seqs* seqs) {
  if (check_attention(d, seqs, "vrs_attention") || d->q_rows == 0 || seqs->n == 0) return 0;
  return attention_bytes(d, plan_attention(d, seqs));
}

int vrs_attention(vrs_ctx* ctx, const vrs_attention_desc* d, const vrs_seqs* seqs, const void* q, const void* k,
                  const void* v, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  const char* me = "vrs_attention";
  if (!ctx) return fail(VRS_EINVAL, "%s: null ctx", me);
  int rc = check_attention(d, seqs, me);
  if (rc) return rc;
  if (d->q_rows == 0 || seqs->n == 0) return VRS_OK;
  if ((rc = check_attention_buffers(d, q, k, v, out, me))) return rc;
  const AttentionPlan p = plan_attention(d, seqs);
  const size_t need = attention_bytes(d, p);
  if (need) {
    if (!workspace || workspace_bytes < need)
      return fail(VRS_EINVAL, "%s: workspace of %zu bytes, %zu needed", me, workspace ? workspace_bytes : (size_t)0, need);
    if (!aligned(workspace, 16)) return fail(VRS_EINVAL, "%s: workspace alignment", me);
  }
  vrs_attention_args a{};
  a.q = q; a.k = k; a.v = v; a.out = out;
  a.s.q_start = seqs->q_start; a.s.k_start = seqs->k_start; a.s.k_len = seqs->k_len; a.s.n = seqs->n;
  a.s.q_rows = d->q_rows; a.s.k_rows = d->k_rows;
  a.q_ld = d->q_ld; a.q_hd = d->q_hd; a.k_ld = d->k_ld; a.k_hd = d->k_hd;
  a.v_ld = d->v_ld; a.v_hd = d->v_hd; a.o_ld = d->o_ld; a.o_hd = d->o_hd;
  a.heads = d->heads; a.kv = d->kv_heads; a.dim = d->head_dim; a.causal = d->causal != 0;
  a.parts = p.parts;
  a.c = (float)((d->scale > 0.f ? (double)d->scale : 1.0 / std::sqrt((double)d->head_dim)) * 1.4426950408889634);
  if (need) {
    const int64_t rows = (int64_t)p.parts * d->q_rows * d->heads;
    a.part_o = static_cast<float*>(workspace);
    a.part_rl = reinterpret_cast<float2*>(a.part_o + rows * d->head_dim);
  }
  const int64_t blocks = p.parts * (p.few ? (int64_t)seqs->n : p.row_tiles) * d->kv_heads;
  const int64_t joins = ((int64_t)d->q_rows * d->heads * (d->head_dim / 4) + 255) / 256;
  if (p.row_tiles >= (1ll << 31) || blocks >= (1ll << 32) / 512 || joins >= (1ll << 32) / 256)
    return fail(VRS_EBADSHAPE, "%s: grid too large", me);
  const int D = d->head_dim <= 64 ? 64 : 128;
  char name[64];
  if (p.few) {
    snprintf(name, sizeof name, "vrs_attention_few_%s_d%d_w%d", dsuffix(d->dtype), D, p.waves);
    rc = launch(ctx, name, dim3((unsigned)blocks, (unsigned)p.row_tiles), dim3(64 * p.waves), 0, &a, stream);
  } else {
    snprintf(name, sizeof name, "vrs_attention_prompt_%s_d%d_q%d_w%d", dsuffix(d->dtype), D, p.qt, p.waves);
    rc = launch(ctx, name, dim3((unsigned)blocks), dim3(64 * p.waves), 0, &a, stream);
  }
  if (rc) return rc;
  if (p.parts == 1) return VRS_OK;
  snprintf(name, sizeof name, "vrs_attention_join_%s", dsuffix(d->dtype));
  return launch(ctx, name, dim3((unsigned)joins), dim3(256), 0, &a, stream);
}

}  // extern "C"
