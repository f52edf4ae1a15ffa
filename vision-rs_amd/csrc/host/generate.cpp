// C-ABI entry points of the operators that generate from a cache (include/vrs.h):
// attention over shared prefixes, beam search's step, attention that keys receive,
// eviction.  Each checks its arguments, picks kernels and launches them on the
// caller's stream.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <initializer_list>

#include "layers.h"

using namespace vrs;

namespace {

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Whether p, if not null, is one of the others.
bool one_of(const void* p, std::initializer_list<const void*> others) {
  return p && std::find(others.begin(), others.end(), p) != others.end();
}

int check_workspace(const void* ws, size_t have, size_t need, const char* me) {
  if (!need) return VRS_OK;
  if (!ws || have < need) return fail(VRS_EINVAL, "%s: workspace of %zu bytes, %zu needed", me, ws ? have : (size_t)0, need);
  if (!aligned(ws, 16)) return fail(VRS_EINVAL, "%s: workspace alignment", me);
  return VRS_OK;
}

// ---- attention over shared prefixes ------------------------------------------

int check_prefixes(const vrs_prefixes* p, const char* me) {
  if (!p) return fail(VRS_EINVAL, "%s: null prefixes", me);
  if (p->n < 0) return fail(VRS_EBADSHAPE, "%s: %d prefixes", me, p->n);
  if (p->max_rows < 0 || p->max_k < 0) return fail(VRS_EINVAL, "%s: negative max_rows or max_k", me);
  int rc;
  if (p->n && ((rc = check_ptr(p->first, 4, me, "first")) || (rc = check_ptr(p->k_start, 4, me, "prefix k_start")) ||
               (rc = check_ptr(p->k_len, 4, me, "prefix k_len"))))
    return rc;
  return VRS_OK;
}

// Kernels and parts of the prefixes' keys and of the own ones.
struct PrefixPlan {
  bool pre_few, own_few;
  bool finish;                      // the own keys' launch finishes; else all parts are joined by a third kernel
  int pre_parts, own_parts, part_len;
  int64_t pre_rows, own_rows;       // few: row tiles of the longest; else ids of row tiles
};
PrefixPlan plan_prefix(const vrs_attention_desc* d, const vrs_seqs* s, const vrs_prefixes* x) {
  const int64_t group = d->heads / d->kv_heads, n = s->n, g = x->n;
  // (unknown: as if all were of one length)
  const int64_t mq = std::max<int64_t>(1, s->max_q > 0 ? std::min(s->max_q, d->q_rows) : up(d->q_rows, n));
  const int64_t mk = s->max_k > 0 ? std::min(s->max_k, d->k_rows) : up(d->k_rows, n);
  const int64_t mr = std::max<int64_t>(1, x->max_rows > 0 ? std::min(x->max_rows, d->q_rows) : up(d->q_rows, g));
  const int64_t mp = std::max<int64_t>(1, x->max_k > 0 ? std::min(x->max_k, d->k_rows) : up(d->k_rows, g));
  PrefixPlan p;
  // one 32-row tile a key head, as vrs_attention's single tokens; more rows share LDS tiles of the keys
  p.pre_few = mr * group <= 32;
  p.own_few = mq * group <= 32;
  auto tiles = [&](int64_t count, int64_t rows) { return std::min(d->q_rows * group / 128 + count, count * up(rows * group, 128)); };
  const int64_t pre = (p.pre_few ? g * up(mr * group, 32) : tiles(g, mr)) * d->kv_heads;
  const int64_t own = (p.own_few ? n * up(mq * group, 32) : tiles(n, mq)) * d->kv_heads;
  // Parts of a prefix, all of one length but the last: 384 workgroups as long as there are 128 keys for each (64
  // tokens on four prefixes of 1500 .. 6000 keys: 256 52.1 us, 384 51.4, 512 52.8, 768 53.3).
  const int64_t parts = std::clamp<int64_t>(std::min(up(384, pre), up(mp, 128)), 1, 64);
  p.part_len = (int)(up(up(mp, parts), p.pre_few ? 128 : 32) * (p.pre_few ? 128 : 32));     // (few rows: a tile to each wave)
  p.pre_parts = (int)up(mp, p.part_len);
  p.own_parts = (int)std::clamp<int64_t>(std::min(512 / own, mk / 192), 1, 16);
  p.finish = !p.own_few && p.own_parts == 1;
  p.pre_rows = p.pre_few ? up(mr * group, 32) : d->q_rows * group / 128 + g;
  p.own_rows = p.own_few ? up(mq * group, 32) : d->q_rows * group / 128 + n;
  return p;
}
size_t prefix_bytes(const vrs_attention_desc* d, const PrefixPlan& p) {
  return (size_t)(p.pre_parts + (p.finish ? 0 : p.own_parts)) * d->q_rows * d->heads * (d->head_dim + 2) * 4;
}

}  // namespace

extern "C" {

size_t vrs_prefix_attention_workspace_size(const vrs_attention_desc* d, const vrs_seqs* seqs,
                                           const vrs_prefixes* prefixes) {
  const char* me = "vrs_prefix_attention";
  if (check_attention(d, seqs, me) || check_prefixes(prefixes, me) || d->q_rows == 0 || seqs->n == 0) return 0;
  if (prefixes->n == 0) return vrs_attention_workspace_size(d, seqs);
  return prefix_bytes(d, plan_prefix(d, seqs, prefixes));
}

int vrs_prefix_attention(vrs_ctx* ctx, const vrs_attention_desc* d, const vrs_seqs* seqs, const vrs_prefixes* prefixes,
                         const void* q, const void* k, const void* v, void* out, void* workspace,
                         size_t workspace_bytes, void* stream) {
  const char* me = "vrs_prefix_attention";
  if (!ctx) return fail(VRS_EINVAL, "%s: null ctx", me);
  int rc = check_attention(d, seqs, me);
  if (rc || (rc = check_prefixes(prefixes, me))) return rc;
  if (d->q_rows == 0 || seqs->n == 0) return VRS_OK;
  if (prefixes->n == 0) return vrs_attention(ctx, d, seqs, q, k, v, out, workspace, workspace_bytes, stream);
  if ((rc = check_attention_buffers(d, q, k, v, out, me))) return rc;
  const PrefixPlan p = plan_prefix(d, seqs, prefixes);
  if ((rc = check_workspace(workspace, workspace_bytes, prefix_bytes(d, p), me))) return rc;
  vrs_prefix_args x{};
  vrs_attention_args& a = x.a;
  a.q = q; a.k = k; a.v = v; a.out = out;
  a.s.q_start = seqs->q_start; a.s.k_start = seqs->k_start; a.s.k_len = seqs->k_len; a.s.n = seqs->n;
  a.s.q_rows = d->q_rows; a.s.k_rows = d->k_rows;
  a.q_ld = d->q_ld; a.q_hd = d->q_hd; a.k_ld = d->k_ld; a.k_hd = d->k_hd;
  a.v_ld = d->v_ld; a.v_hd = d->v_hd; a.o_ld = d->o_ld; a.o_hd = d->o_hd;
  a.heads = d->heads; a.kv = d->kv_heads; a.dim = d->head_dim; a.causal = d->causal != 0;
  a.parts = p.pre_parts + (p.finish ? 0 : p.own_parts);
  a.c = (float)((d->scale > 0.f ? (double)d->scale : 1.0 / std::sqrt((double)d->head_dim)) * 1.4426950408889634);
  a.part_o = static_cast<float*>(workspace);
  a.part_rl = reinterpret_cast<float2*>(a.part_o + (int64_t)a.parts * d->q_rows * d->heads * d->head_dim);
  x.first = prefixes->first; x.p_start = prefixes->k_start; x.p_len = prefixes->k_len; x.groups = prefixes->n;
  x.pre_parts = p.pre_parts; x.own_parts = p.own_parts; x.part_len = p.part_len; x.finish = p.finish;
  const int64_t pre = (int64_t)d->kv_heads * p.pre_parts * (p.pre_few ? (int64_t)prefixes->n : p.pre_rows);
  const int64_t own = (int64_t)d->kv_heads * p.own_parts * (p.own_few ? (int64_t)seqs->n : p.own_rows);
  const int64_t per_row = up((int64_t)d->heads * (d->head_dim / 4), 256);
  if (p.pre_rows >= (1 << 16) * 256ll || p.own_rows >= (1 << 16) * 256ll || pre + own >= (1ll << 32) / 512 ||
      d->q_rows >= (1 << 24) || per_row > 65535)
    return fail(VRS_EBADSHAPE, "%s: grid too large", me);
  const int D = d->head_dim <= 64 ? 64 : 128;
  char name[64];
  // (row tiles past the grid's are taken in turn)
  x.pre_rows = (int32_t)std::min<int64_t>(p.pre_rows, 65535); x.own_rows = (int32_t)std::min<int64_t>(p.own_rows, 65535);
  auto go = [&](const char* kind, int64_t pre_blocks, int64_t own_blocks) {
    x.pre_blocks = (int32_t)pre_blocks;
    const int y = std::max(pre_blocks && p.pre_few ? x.pre_rows : 1, own_blocks && p.own_few ? x.own_rows : 1);
    snprintf(name, sizeof name, "vrs_prefix_%s_%s_d%d", kind, dsuffix(d->dtype), D);
    return launch(ctx, name, dim3((unsigned)(pre_blocks + own_blocks), (unsigned)y), dim3(256), 0, &x, stream);
  };
  if (p.own_few) {
    rc = go(p.pre_few ? "few" : "mixed", pre, own);
  } else {
    rc = go(p.pre_few ? "few" : "prompt", pre, 0);
    if (!rc) rc = go("own", 0, own);
  }
  if (rc || p.finish) return rc;
  snprintf(name, sizeof name, "vrs_prefix_join_%s", dsuffix(d->dtype));
  return launch(ctx, name, dim3((unsigned)d->q_rows, (unsigned)per_row), dim3(256), 0, &x, stream);
}

}  // extern "C"

// ---- beam search ---------------------------------------------------------------

namespace {

int check_beam(const vrs_beam_desc* d, const char* me) {
  if (!d) return fail(VRS_EINVAL, "%s: null argument", me);
  if (int rc = check_type(d->dtype, me)) return rc;
  if (d->batch < 0 || d->beams < 1 || d->vocab < 1)
    return fail(VRS_EBADSHAPE, "%s: %d requests of %d beams, %d tokens", me, d->batch, d->beams, d->vocab);
  if (d->beams > 64 || d->k > 128) return fail(VRS_EUNSUPPORTED, "%s: %d beams (up to 64), k %d (up to 128)", me, d->beams, d->k);
  if ((int64_t)d->beams * d->vocab >= 0x7fffffff) return fail(VRS_EUNSUPPORTED, "%s: %d beams of %d tokens", me, d->beams, d->vocab);
  if ((int64_t)d->batch * d->beams > 65535) return fail(VRS_EUNSUPPORTED, "%s: %d requests of %d beams (65535 rows)", me, d->batch, d->beams);
  if (d->k < 1 || d->k > (int64_t)d->beams * d->vocab) return fail(VRS_EBADSHAPE, "%s: k %d", me, d->k);
  if (d->ld < 0 || d->ld >> 40) return fail(VRS_EBADSHAPE, "%s: row stride %lld", me, (long long)d->ld);
  return VRS_OK;
}

struct BeamPlan { int vt, chunk, chunks; };
// Chunks of 8192 logits where these give two workgroups to a CU (32 elements a thread, fewer lists to join), else of
// 2048 (latency: four beams over 32000 tokens, 64 workgroups instead of 16).
BeamPlan plan_beam(const vrs_beam_desc* d) {
  const int v = 16 / (int)elt_size(d->dtype), rows = d->batch * d->beams;
  BeamPlan p;
  const bool large = (int64_t)rows * up(d->vocab, 8192) >= 512;
  p.vt = (large ? 8192 : 2048) / 256 / v;
  p.chunk = 256 * v * p.vt;
  p.chunks = (int)up(d->vocab, p.chunk);
  return p;
}
size_t beam_part_bytes(const vrs_beam_desc* d, const BeamPlan& p) { return (size_t)d->batch * d->beams * p.chunks * 16; }
size_t beam_bytes(const vrs_beam_desc* d, const BeamPlan& p) {
  return beam_part_bytes(d, p) + (size_t)d->batch * d->beams * p.chunks * d->k * 8;
}

// Whether three dimensions of `bytes` long rows, n[i] times stride[i], keep rows apart: each stride passes over
// all that the smaller ones reach.
bool rows_apart(int64_t bytes, const int64_t (&n)[3], const int64_t (&stride)[3]) {
  int o[3] = {0, 1, 2};
  std::sort(o, o + 3, [&](int i, int j) { return stride[i] < stride[j]; });
  int64_t reach = bytes;
  for (int i : o) {
    if (n[i] <= 1) continue;
    if (stride[i] < reach) return false;
    reach += (n[i] - 1) * stride[i];
  }
  return true;
}

}  // namespace

extern "C" {

size_t vrs_beam_select_workspace_size(const vrs_beam_desc* d) {
  if (check_beam(d, "vrs_beam_select") || d->batch == 0) return 0;
  return beam_bytes(d, plan_beam(d));
}

int vrs_beam_select(vrs_ctx* ctx, const vrs_beam_desc* d, const void* logits, const float* scores, const uint8_t* done,
                    float* out_scores, int32_t* out_parents, int32_t* out_tokens, void* workspace,
                    size_t workspace_bytes, void* stream) {
  const char* me = "vrs_beam_select";
  if (!ctx) return fail(VRS_EINVAL, "%s: null ctx", me);
  int rc = check_beam(d, me);
  if (rc) return rc;
  if (done && (d->eos < 0 || d->eos >= d->vocab)) return fail(VRS_EINVAL, "%s: eos %d of %d tokens", me, d->eos, d->vocab);
  if (d->batch == 0) return VRS_OK;      // empty tensors may have null addresses
  if ((rc = check_ptr(logits, elt_size(d->dtype), me, "logits")) || (rc = check_ptr(scores, 4, me, "scores")) ||
      (rc = check_ptr(out_scores, 4, me, "out_scores")) || (rc = check_ptr(out_parents, 4, me, "out_parents")) ||
      (rc = check_ptr(out_tokens, 4, me, "out_tokens")))
    return rc;
  if (one_of(out_scores, {logits, scores, done, out_parents, out_tokens}) || one_of(out_parents, {logits, scores, done, out_tokens}) ||
      one_of(out_tokens, {logits, scores, done}))
    return fail(VRS_EINVAL, "%s: an output is another buffer", me);
  const BeamPlan p = plan_beam(d);
  if ((rc = check_workspace(workspace, workspace_bytes, beam_bytes(d, p), me))) return rc;
  vrs_beam_args a{};
  a.logits = logits; a.scores = scores; a.done = done;
  a.part = static_cast<double2*>(workspace);
  a.list = reinterpret_cast<uint2*>(static_cast<char*>(workspace) + beam_part_bytes(d, p));
  a.out_scores = out_scores; a.out_parents = out_parents; a.out_tokens = out_tokens;
  a.ld = d->ld;
  a.batch = d->batch; a.beams = d->beams; a.vocab = d->vocab; a.k = d->k; a.eos = d->eos;
  a.chunks = p.chunks; a.chunk = p.chunk;
  char name[64];
  snprintf(name, sizeof name, "vrs_beam_part_%s_v%d", dsuffix(d->dtype), p.vt);
  rc = launch(ctx, name, dim3((unsigned)p.chunks, (unsigned)(d->batch * d->beams)), dim3(256), 0, &a, stream);
  if (rc) return rc;
  snprintf(name, sizeof name, "vrs_beam_join_%s", dsuffix(d->dtype));
  return launch(ctx, name, dim3((unsigned)d->batch), dim3(256), 0, &a, stream);
}

int vrs_beam_reorder(vrs_ctx* ctx, const vrs_reorder_desc* d, const int32_t* parents, const int32_t* len, void* state,
                     void* stream) {
  const char* me = "vrs_beam_reorder";
  if (!ctx || !d) return fail(VRS_EINVAL, "%s: null argument", me);
  if (d->batch < 0 || d->beams < 1 || d->layers < 0 || d->rows < 0 || d->row_bytes < 0)
    return fail(VRS_EBADSHAPE, "%s: %d requests of %d beams, %d layers of %d rows of %lld bytes", me, d->batch, d->beams,
                d->layers, d->rows, (long long)d->row_bytes);
  if (d->beams > 64) return fail(VRS_EUNSUPPORTED, "%s: %d beams (up to 64)", me, d->beams);
  for (int64_t s : {d->row_bytes, d->row_ld, d->slot_ld, d->layer_ld})
    if (s < 0 || s >> 42) return fail(VRS_EBADSHAPE, "%s: stride %lld", me, (long long)s);
  if (d->batch == 0 || d->layers == 0 || d->rows == 0 || d->row_bytes == 0) return VRS_OK;
  int rc;
  if ((rc = check_ptr(parents, 4, me, "parents")) || (len && (rc = check_ptr(len, 4, me, "len"))) ||
      (rc = check_ptr(state, 1, me, "state")))
    return rc;
  if (one_of(state, {parents, len})) return fail(VRS_EINVAL, "%s: the state is parents or len", me);
  if (!rows_apart(d->row_bytes, {d->rows, (int64_t)d->batch * d->beams, d->layers}, {d->row_ld, d->slot_ld, d->layer_ld}))
    return fail(VRS_EBADSHAPE, "%s: strides fold rows onto each other", me);
  if (d->batch > 65535 || d->layers > 65535) return fail(VRS_EUNSUPPORTED, "%s: %d requests, %d layers (up to 65535)", me, d->batch, d->layers);
  auto fits = [&](int64_t v) {
    return aligned(state, v) && d->row_bytes % v == 0 && (d->rows == 1 || d->row_ld % v == 0) && d->slot_ld % v == 0 &&
           (d->layers == 1 || d->layer_ld % v == 0);
  };
  const int v = fits(16) ? 16 : fits(4) ? 4 : 1;
  if (d->row_bytes / v >= (1ll << 31)) return fail(VRS_EUNSUPPORTED, "%s: rows of %lld bytes", me, (long long)d->row_bytes);
  vrs_reorder_args a{};
  a.state = static_cast<char*>(state); a.parents = parents; a.len = len;
  a.row_ld = d->row_ld; a.slot_ld = d->slot_ld; a.layer_ld = d->layer_ld;
  a.batch = d->batch; a.beams = d->beams; a.rows = d->rows; a.cols = (int32_t)(d->row_bytes / v);
  const int64_t units = up((int64_t)d->rows * a.cols, 256), pairs = (int64_t)d->batch * d->layers;
  const unsigned x = (unsigned)std::clamp<int64_t>(up(8192, pairs), 1, units);
  char name[64];
  snprintf(name, sizeof name, "vrs_beam_reorder_b%d_n%d", v, d->beams <= 4 ? 4 : d->beams <= 8 ? 8 : d->beams <= 16 ? 16 : 64);
  return launch(ctx, name, dim3(x, (unsigned)d->batch, (unsigned)d->layers), dim3(256), 0, &a, stream);
}

}  // extern "C"

// ---- attention that keys receive -------------------------------------------------

namespace {

int check_weights(const vrs_weights_desc* d, const vrs_seqs* seqs, const char* me) {
  if (!d || !seqs) return fail(VRS_EINVAL, "%s: null argument", me);
  vrs_attention_desc t{};                 // what vrs_attention asks of queries and keys
  t.q_rows = d->q_rows; t.k_rows = d->k_rows; t.heads = d->heads; t.kv_heads = d->kv_heads; t.head_dim = d->head_dim;
  t.dtype = d->dtype; t.causal = d->causal; t.scale = d->scale;
  t.q_ld = d->q_ld; t.q_hd = d->q_hd; t.k_ld = d->k_ld; t.k_hd = d->k_hd; t.v_ld = d->k_ld; t.v_hd = d->k_hd;
  t.q_rows = std::min(t.q_rows, 1);       // no output of that kind
  t.o_hd = t.o_ld = 128;
  int rc = check_attention(&t, seqs, me);
  if (rc) return rc;
  if (!(d->decay >= 0.f && d->decay <= 1.f)) return fail(VRS_EINVAL, "%s: decay %g", me, (double)d->decay);
  for (int64_t s : {d->acc_ld, d->acc_hd})
    if (s < 0 || s >> 40) return fail(VRS_EBADSHAPE, "%s: stride %lld", me, (long long)s);
  // (the kernels' offsets from a row tile's first query)
  if ((d->heads / d->kv_heads) * d->q_hd + 65 * d->q_ld >= (1ll << 31) / 4)
    return fail(VRS_EUNSUPPORTED, "%s: query strides %lld and %lld", me, (long long)d->q_ld, (long long)d->q_hd);
  if ((d->k_rows > 1 && d->acc_ld < 1) || (d->kv_heads > 1 && d->acc_hd < 1))
    return fail(VRS_EBADSHAPE, "%s: acc strides fold rows or heads onto each other", me);
  return VRS_OK;
}

struct WeightsPlan {
  bool few;
  int parts, key_parts;
  int64_t row_tiles;       // few: 32-row tiles of the longest sequence; else ids of 128-row tiles
  int64_t s_ld, key_tiles; // keys counted on, in whole tiles; tiles of them
};
WeightsPlan plan_weights(const vrs_weights_desc* d, const vrs_seqs* s) {
  const int64_t group = d->heads / d->kv_heads, n = s->n;
  const int64_t mq = std::max<int64_t>(1, s->max_q > 0 ? std::min(s->max_q, d->q_rows) : up(d->q_rows, n));
  const int64_t mk = std::max<int64_t>(1, s->max_k > 0 ? std::min(s->max_k, d->k_rows) : up(d->k_rows, n));
  WeightsPlan p;
  // Few rows leave their scores: one 32-row tile a key head, whose scores are at most half of a key's bytes in
  // bfloat16 at a head of 128.  Single tokens go in four parts at least, so that long and short caches even out (64
  // over 500 .. 8000 keys: 128 us; one part 197).
  p.few = mq * group <= 32;
  p.key_parts = 1;
  if (p.few) {
    p.row_tiles = up(mq * group, 32);
    const int64_t wgs = n * d->kv_heads * p.row_tiles;
    p.parts = (int)std::clamp<int64_t>(std::min(std::max<int64_t>(4, up(512, wgs)), mk / 192), 1, 64);
    p.key_tiles = up(mk, 1024);
    p.s_ld = p.key_tiles * 1024;
  } else {
    p.row_tiles = d->q_rows * group / 128 + n;
    const int64_t wgs = std::min(p.row_tiles, n * up(mq * group, 128)) * d->kv_heads;
    p.parts = (int)std::clamp<int64_t>(std::min(1024 / wgs, mk / 256), 1, 32);
    p.key_tiles = up(mk, 128);
    p.s_ld = p.key_tiles * 128;
    // (a prompt of 4096 queries, 8 key heads: 1024 workgroups 132 us, 2048 127, 4096 137)
    p.key_parts = (int)std::clamp<int64_t>(std::min(2048 / (n * d->kv_heads * p.key_tiles), mq * group / 256), 1, 16);
  }
  return p;
}
size_t weights_rl_bytes(const vrs_weights_desc* d, const WeightsPlan& p) { return (size_t)up((int64_t)p.parts * d->q_rows * d->heads, 2) * 16; }
size_t weights_bytes(const vrs_weights_desc* d, int32_t n, const WeightsPlan& p) {
  const size_t rows = p.few ? (size_t)d->q_rows * d->heads : p.key_parts > 1 ? (size_t)p.key_parts * n * d->kv_heads : 0;
  return weights_rl_bytes(d, p) + rows * p.s_ld * 4;
}

}  // namespace

extern "C" {

size_t vrs_attention_weights_workspace_size(const vrs_weights_desc* d, const vrs_seqs* seqs) {
  if (check_weights(d, seqs, "vrs_attention_weights") || d->k_rows == 0 || seqs->n == 0) return 0;
  return weights_bytes(d, seqs->n, plan_weights(d, seqs));
}

int vrs_attention_weights(vrs_ctx* ctx, const vrs_weights_desc* d, const vrs_seqs* seqs, const void* q, const void* k,
                          float* acc, void* workspace, size_t workspace_bytes, void* stream) {
  const char* me = "vrs_attention_weights";
  if (!ctx) return fail(VRS_EINVAL, "%s: null ctx", me);
  int rc = check_weights(d, seqs, me);
  if (rc) return rc;
  if (d->k_rows == 0 || seqs->n == 0) return VRS_OK;
  if ((d->q_rows && (rc = check_ptr(q, 16, me, "q"))) || (rc = check_ptr(k, 16, me, "k")) || (rc = check_ptr(acc, 4, me, "acc"))) return rc;
  if ((const void*)acc == q || (const void*)acc == k) return fail(VRS_EINVAL, "%s: acc is an input", me);
  const WeightsPlan p = plan_weights(d, seqs);
  if ((rc = check_workspace(workspace, workspace_bytes, weights_bytes(d, seqs->n, p), me))) return rc;
  vrs_weights_args a{};
  a.q = q; a.k = k; a.acc = acc;
  a.rl = static_cast<float2*>(workspace);
  a.scores = reinterpret_cast<float*>(static_cast<char*>(workspace) + weights_rl_bytes(d, p));
  a.s.q_start = seqs->q_start; a.s.k_start = seqs->k_start; a.s.k_len = seqs->k_len; a.s.n = seqs->n;
  a.s.q_rows = d->q_rows; a.s.k_rows = d->k_rows;
  a.q_ld = d->q_ld; a.q_hd = d->q_hd; a.k_ld = d->k_ld; a.k_hd = d->k_hd; a.acc_ld = d->acc_ld; a.acc_hd = d->acc_hd;
  a.s_ld = p.s_ld;
  a.heads = d->heads; a.kv = d->kv_heads; a.dim = d->head_dim; a.causal = d->causal != 0; a.parts = p.parts;
  a.key_parts = p.key_parts;
  a.c = (float)((d->scale > 0.f ? (double)d->scale : 1.0 / std::sqrt((double)d->head_dim)) * 1.4426950408889634);
  a.decay = d->decay;
  const int64_t pairs = (int64_t)seqs->n * d->kv_heads;
  const int64_t first = (p.few ? pairs : p.row_tiles * d->kv_heads) * p.parts;
  if (p.row_tiles >= (1ll << 30) || first >= (1ll << 32) / 256 || pairs * p.key_parts >= (1ll << 32) / 256)
    return fail(VRS_EBADSHAPE, "%s: grid too large", me);
  const int D = d->head_dim <= 64 ? 64 : 128;
  char name[64];
  if (d->q_rows) {
    snprintf(name, sizeof name, "vrs_weights_%s_%s_d%d", p.few ? "scores" : "stats", dsuffix(d->dtype), D);
    const unsigned y = p.few ? (unsigned)std::min<int64_t>(p.row_tiles, 65535) : 1;
    rc = launch(ctx, name, dim3((unsigned)first, y), dim3(256), 0, &a, stream);
    if (rc) return rc;
    // (q_rows * heads < 2^31, as the first launch's grid has it)
    if (!p.few && p.parts > 1 &&
        (rc = launch(ctx, "vrs_weights_rows", dim3((unsigned)up((int64_t)d->q_rows * d->heads, 256)), dim3(256), 0, &a, stream)))
      return rc;
  }
  if (p.few) snprintf(name, sizeof name, "vrs_weights_sum_%s", dsuffix(d->dtype));
  else snprintf(name, sizeof name, "vrs_weights_keys_%s_d%d", dsuffix(d->dtype), D);
  const unsigned tiles = (unsigned)std::min<int64_t>(p.key_tiles, 65535);
  rc = launch(ctx, name, dim3((unsigned)(pairs * p.key_parts), tiles), dim3(256), 0, &a, stream);
  if (rc || p.key_parts == 1) return rc;
  return launch(ctx, "vrs_weights_join", dim3((unsigned)pairs, (unsigned)up(p.s_ld, 256)), dim3(256), 0, &a, stream);
}

// ---- eviction ----------------------------------------------------------------------

int vrs_cache_evict(vrs_ctx* ctx, const vrs_evict_desc* d, const int32_t* k_start, const int32_t* k_len,
                    const int32_t* out_start, const void* k, const void* v, const float* acc, void* k_out, void* v_out,
                    float* acc_out, int32_t* len_out, int32_t* kept, void* stream) {
  const char* me = "vrs_cache_evict";
  if (!ctx || !d) return fail(VRS_EINVAL, "%s: null argument", me);
  int rc = check_type(d->dtype, me);
  if (rc) return rc;
  if (d->n < 0 || d->k_rows < 0 || d->out_rows < 0 || d->kv_heads < 1 || d->head_dim < 1 || d->head_dim > 4096)
    return fail(VRS_EBADSHAPE, "%s: %d sequences, %d and %d rows, %d heads of %d", me, d->n, d->k_rows, d->out_rows, d->kv_heads, d->head_dim);
  if (d->budget < 1 || d->first < 0 || d->recent < 0 || (int64_t)d->first + d->recent > d->budget)
    return fail(VRS_EINVAL, "%s: first %d and recent %d of a budget of %d", me, d->first, d->recent, d->budget);
  if (d->max_k < 0) return fail(VRS_EINVAL, "%s: negative max_k", me);
  for (int64_t s : {d->k_ld, d->k_hd, d->v_ld, d->v_hd, d->acc_ld, d->acc_hd, d->ko_ld, d->ko_hd, d->vo_ld, d->vo_hd,
                    d->acco_ld, d->acco_hd})
    if (s < 0 || s >> 40) return fail(VRS_EBADSHAPE, "%s: stride %lld", me, (long long)s);
  if (d->n == 0) return VRS_OK;
  // the kernels' numbers of keys and of kept places run on to the end of the tiles ahead
  if (std::max(d->k_rows, d->budget) > 0x7fffffff - (1 << 20))
    return fail(VRS_EUNSUPPORTED, "%s: %d key rows, a budget of %d", me, d->k_rows, d->budget);
  const size_t es = elt_size(d->dtype);
  if ((rc = check_ptr(k_start, 4, me, "k_start")) || (rc = check_ptr(k_len, 4, me, "k_len")) || (rc = check_ptr(kept, 4, me, "kept")) ||
      (out_start && (rc = check_ptr(out_start, 4, me, "out_start"))) || (len_out && (rc = check_ptr(len_out, 4, me, "len_out"))))
    return rc;
  if (d->k_rows && ((rc = check_ptr(k, es, me, "k")) || (rc = check_ptr(v, es, me, "v")) || (rc = check_ptr(acc, 4, me, "acc")))) return rc;
  if (d->out_rows && ((rc = check_ptr(k_out, es, me, "k_out")) || (rc = check_ptr(v_out, es, me, "v_out")) ||
                      (rc = check_ptr(acc_out, 4, me, "acc_out"))))
    return rc;
  if (d->k_rows && d->out_rows && (k_out == v_out || k_out == v || v_out == k)) return fail(VRS_EINVAL, "%s: k and v are one buffer", me);
  // in place, rows must not move but down their own sequence
  const bool moved = out_start && out_start != k_start;
  if ((k_out == k && k && (moved || d->ko_ld != d->k_ld || d->ko_hd != d->k_hd)) ||
      (v_out == v && v && (moved || d->vo_ld != d->v_ld || d->vo_hd != d->v_hd)) ||
      (acc_out == acc && acc && (moved || d->acco_ld != d->acc_ld || d->acco_hd != d->acc_hd)))
    return fail(VRS_EBADSHAPE, "%s: an output is its input with other strides or rows", me);
  auto folds = [&](int64_t ld, int64_t hd, int64_t dim) {
    return (d->out_rows > 1 && ld < dim) || (d->kv_heads > 1 && hd < dim);
  };
  if (folds(d->ko_ld, d->ko_hd, d->head_dim) || folds(d->vo_ld, d->vo_hd, d->head_dim) || folds(d->acco_ld, d->acco_hd, 1))
    return fail(VRS_EBADSHAPE, "%s: output strides fold rows or heads onto each other", me);
  const void *k_in = d->k_rows ? k : nullptr, *v_in = d->k_rows ? v : nullptr, *acc_in = d->k_rows ? acc : nullptr;
  const void *k_to = d->out_rows ? k_out : nullptr, *v_to = d->out_rows ? v_out : nullptr, *acc_to = d->out_rows ? acc_out : nullptr;
  if (one_of(kept, {k_start, k_len, out_start, k_in, v_in, acc_in, k_to, v_to, acc_to})) return fail(VRS_EINVAL, "%s: kept is another array", me);
  if (one_of(len_out, {k_start, out_start, kept, k_in, v_in, acc_in, k_to, v_to, acc_to}))
    return fail(VRS_EINVAL, "%s: len_out is another array", me);
  if (one_of(acc_to, {k_in, v_in, k_to, v_to}) || one_of(acc_in, {k_to, v_to})) return fail(VRS_EINVAL, "%s: acc is another buffer", me);

  auto fits = [&](int64_t bytes) {
    const int64_t n = bytes / (int64_t)es;
    auto of = [&](const void* p, int64_t ld, int64_t hd) { return aligned(p, bytes) && ld % n == 0 && hd % n == 0; };
    // (an empty buffer may have any address)
    return d->head_dim % n == 0 && (d->k_rows == 0 || (of(k, d->k_ld, d->k_hd) && of(v, d->v_ld, d->v_hd))) &&
           (d->out_rows == 0 || (of(k_out, d->ko_ld, d->ko_hd) && of(v_out, d->vo_ld, d->vo_hd)));
  };
  const int b = fits(16) ? 16 : fits(4) ? 4 : 2;
  const int64_t per = b / (int64_t)es;
  vrs_evict_args a{};
  a.k = k; a.v = v; a.acc = acc; a.ko = k_out; a.vo = v_out; a.acco = acc_out;
  a.k_start = k_start; a.k_len = k_len; a.o_start = out_start; a.len_out = len_out; a.kept = kept;
  a.k_ld = d->k_ld / per; a.k_hd = d->k_hd / per; a.v_ld = d->v_ld / per; a.v_hd = d->v_hd / per;
  a.ko_ld = d->ko_ld / per; a.ko_hd = d->ko_hd / per; a.vo_ld = d->vo_ld / per; a.vo_hd = d->vo_hd / per;
  a.acc_ld = d->acc_ld; a.acc_hd = d->acc_hd; a.acco_ld = d->acco_ld; a.acco_hd = d->acco_hd;
  a.n = d->n; a.k_rows = d->k_rows; a.o_rows = d->out_rows; a.kv = d->kv_heads; a.dim = d->head_dim;
  a.budget = d->budget; a.first = d->first; a.recent = d->recent;
  a.cols = (int32_t)(d->head_dim / per);
  const int64_t pairs = (int64_t)d->n * d->kv_heads;
  // Workgroups of the move: two to a CU.  Slices of 128 bytes of a row (half a cache line costs its whole), of 32
  // where workgroups would be few; blocks of rows where nothing moves in place.
  const bool in_place = (k_out == k && k) || (v_out == v && v);
  const int64_t want = up(512, 2 * pairs), row = (int64_t)d->head_dim * (int64_t)es;
  a.slices = (int32_t)std::clamp<int64_t>(want, 1, std::max<int64_t>(1, row / (want > 4 && in_place ? 32 : 128)));
  a.slices = std::min(std::max(a.slices, (int32_t)up(a.cols, 256)), a.cols);      // (a thread to a vector of a slice)
  const int64_t blocks = in_place ? 1 : std::clamp<int64_t>(want / a.slices, 1, std::max<int64_t>(1, d->budget / 32));
  if (pairs * a.slices >= (1ll << 32) / 1024) return fail(VRS_EBADSHAPE, "%s: grid too large", me);
  // the choice holds 16 keys of a thread in registers, and waits for fewer waves where 256 threads are enough
  const int threads = (d->max_k > 0 ? d->max_k : d->k_rows / d->n) <= 4096 ? 256 : 1024;
  char name[64];
  snprintf(name, sizeof name, "vrs_evict_choose_t%d", threads);
  if ((rc = launch(ctx, name, dim3((unsigned)pairs), dim3(threads), 0, &a, stream))) return rc;
  snprintf(name, sizeof name, "vrs_evict_move_b%d", b);
  return launch(ctx, name, dim3((unsigned)(pairs * a.slices), 2, (unsigned)std::min<int64_t>(blocks, 65535)), dim3(256), 0, &a, stream);
}

}  // extern "C"
