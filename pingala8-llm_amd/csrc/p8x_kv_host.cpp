// p8x_kv_host.cpp -- entry points of the calls between the linears (norm, cache, attention of drafted tokens): argument
// checks, and the structs of p8x.h as kernel arguments.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "p8x_kv.h"

namespace p8x {
namespace {

bool is_float(int dtype) { return dtype == P8X_F32 || dtype == P8X_F16 || dtype == P8X_BF16; }
bool aligned(const void *p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }
size_t elem_size(int dtype) { return dtype == P8X_F32 ? 4 : 2; }

int check_cache(const char *fn, const p8x_kv_cache *c, KvDev &o) {
    if (!c) return set_error(P8X_ERR_ARG, "%s: null cache", fn);
    if (c->dtype != P8X_F16 && c->dtype != P8X_BF16) return set_error(P8X_ERR_ARG, "%s: cache dtype %d (P8X_F16 or P8X_BF16)", fn, c->dtype);
    if (c->n_seq < 1 || c->n_kv < 1 || c->max_len < 1) return set_error(P8X_ERR_ARG, "%s: n_seq %d n_kv %d max_len %d", fn, c->n_seq, c->n_kv, c->max_len);
    if (c->n_seq > 65535 || c->n_kv > 65535) return set_error(P8X_ERR_UNSUPPORTED, "%s: n_seq %d n_kv %d (at most 65535)", fn, c->n_seq, c->n_kv);
    if (c->max_len > (1 << 30)) return set_error(P8X_ERR_UNSUPPORTED, "%s: max_len %d (at most 2^30)", fn, c->max_len);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return set_error(P8X_ERR_UNSUPPORTED, "%s: head_dim %d (64, 128 or 256)", fn, c->head_dim);
    if (!c->k || !c->v || !c->len) return set_error(P8X_ERR_ARG, "%s: null k, v or len", fn);
    if (!aligned(c->k, 16) || !aligned(c->v, 16)) return set_error(P8X_ERR_ARG, "%s: k and v 16-byte aligned", fn);
    if ((c->page_stride | c->head_stride | c->slot_stride) & 7 || c->slot_stride < (size_t)c->head_dim || (c->n_kv > 1 && c->head_stride < (size_t)c->head_dim))
        return set_error(P8X_ERR_ARG, "%s: strides %zu %zu %zu (multiples of 8, rows of %d apart)", fn, c->page_stride, c->head_stride, c->slot_stride, c->head_dim);
    if (c->page_size < 1 || c->n_pages < 1) return set_error(P8X_ERR_ARG, "%s: page_size %d n_pages %d", fn, c->page_size, c->n_pages);
    if (c->pages) {
        if (c->page_size % 16) return set_error(P8X_ERR_ARG, "%s: page_size %d (a multiple of 16)", fn, c->page_size);
        if (c->ld_pages * (size_t)c->page_size < (size_t)c->max_len)
            return set_error(P8X_ERR_ARG, "%s: %zu pages of %d slots for max_len %d", fn, c->ld_pages, c->page_size, c->max_len);
    } else if (c->n_pages < c->n_seq || c->page_size < c->max_len) {
        return set_error(P8X_ERR_ARG, "%s: without a page table n_pages %d >= n_seq %d and page_size %d >= max_len %d", fn, c->n_pages, c->n_seq, c->page_size, c->max_len);
    }
    o = {(uint16_t *)c->k, (uint16_t *)c->v, c->page_stride, c->head_stride, c->slot_stride, c->pages, c->ld_pages, c->len,
         c->page_size, c->n_pages, c->max_len, c->n_seq, c->n_kv, c->dtype == P8X_BF16};
    return P8X_OK;
}

// rows of `heads` heads of D elements, 16-byte pieces
bool rows_ok(const void *p, int dtype, size_t ld, size_t hs, int heads, int D) {
    return aligned(p, 16) && (ld | hs) % (16 / elem_size(dtype)) == 0 && ld >= (size_t)D && (heads == 1 || hs >= (size_t)D);
}

// kv, q: what the call reads of them
int check_drafts(const char *fn, const p8x_kv_cache *c, const p8x_drafts *d, bool k, bool v, bool q, int most, DraftDev &o) {
    if (!d) return set_error(P8X_ERR_ARG, "%s: null drafts", fn);
    if (d->n_tokens < 0 || d->max_tokens < 0) return set_error(P8X_ERR_ARG, "%s: n_tokens %d max_tokens %d", fn, d->n_tokens, d->max_tokens);
    if (most && d->max_tokens > most) return set_error(P8X_ERR_UNSUPPORTED, "%s: max_tokens %d (at most %d)", fn, d->max_tokens, most);
    if (!d->first) return set_error(P8X_ERR_ARG, "%s: null first", fn);
    const size_t hkv = d->head_stride_kv ? d->head_stride_kv : (size_t)c->head_dim, hq = d->head_stride_q ? d->head_stride_q : (size_t)c->head_dim;
    o = {d->first, d->k, d->v, d->ld_kv, hkv, d->kv_dtype == P8X_F32, d->mask, d->q, d->ld_q, hq, d->q_dtype == P8X_F32,
         d->n_tokens, d->max_tokens, 1, d->scale};
    if (d->n_tokens == 0 || d->max_tokens == 0) return P8X_OK;
    if ((k && !d->k) || (v && !d->v)) return set_error(P8X_ERR_ARG, "%s: null draft k or v", fn);
    if (d->kv_dtype != P8X_F32 && d->kv_dtype != c->dtype) return set_error(P8X_ERR_ARG, "%s: draft k, v dtype %d (P8X_F32 or the cache's)", fn, d->kv_dtype);
    if ((k && !rows_ok(d->k, d->kv_dtype, d->ld_kv, hkv, c->n_kv, c->head_dim)) || (v && !rows_ok(d->v, d->kv_dtype, d->ld_kv, hkv, c->n_kv, c->head_dim)))
        return set_error(P8X_ERR_ARG, "%s: draft k, v rows 16-byte aligned, strides %zu %zu", fn, d->ld_kv, hkv);
    if (q) {
        if (d->n_heads < 1 || d->n_heads % c->n_kv) return set_error(P8X_ERR_ARG, "%s: n_heads %d of n_kv %d", fn, d->n_heads, c->n_kv);
        if (d->n_heads > 65535) return set_error(P8X_ERR_UNSUPPORTED, "%s: n_heads %d (at most 65535)", fn, d->n_heads);
        if (!d->q) return set_error(P8X_ERR_ARG, "%s: null q", fn);
        if (d->q_dtype != P8X_F32 && d->q_dtype != c->dtype) return set_error(P8X_ERR_ARG, "%s: q dtype %d (P8X_F32 or the cache's)", fn, d->q_dtype);
        if (!rows_ok(d->q, d->q_dtype, d->ld_q, hq, d->n_heads, c->head_dim))
            return set_error(P8X_ERR_ARG, "%s: q rows 16-byte aligned, strides %zu %zu", fn, d->ld_q, hq);
        if (!(d->scale - d->scale == 0.0f)) return set_error(P8X_ERR_ARG, "%s: scale is not finite", fn);
        o.G = d->n_heads / c->n_kv;
    }
    return P8X_OK;
}

constexpr int kMostTokens = 1 << 30;   // of a sequence: slots are counted in 31 bits

// the rotation of heads of D elements
int check_rotation(const char *fn, const p8x_rotation *r, int D, TurnDev &o) {
    if (!r) return set_error(P8X_ERR_ARG, "%s: null rotation", fn);
    if (r->layout != P8X_ROPE_HALF && r->layout != P8X_ROPE_PAIRS) return set_error(P8X_ERR_ARG, "%s: layout %d", fn, r->layout);
    if (r->n_rot < 0 || r->n_rot > D) return set_error(P8X_ERR_ARG, "%s: n_rot %d of head_dim %d", fn, r->n_rot, D);
    if (r->n_rot % 8) return set_error(P8X_ERR_UNSUPPORTED, "%s: n_rot %d (a multiple of 8)", fn, r->n_rot);
    if (r->n_rot && !r->freq) return set_error(P8X_ERR_ARG, "%s: null freq", fn);
    if (!aligned(r->freq, 16) || !aligned(r->w_q, 16) || !aligned(r->w_k, 16)) return set_error(P8X_ERR_ARG, "%s: freq, w_q and w_k 16-byte aligned", fn);
    if (!(r->amplitude - r->amplitude == 0.0f)) return set_error(P8X_ERR_ARG, "%s: amplitude is not finite", fn);
    o = {r->freq, r->w_q, r->w_k, r->amplitude, r->eps, r->layout == P8X_ROPE_PAIRS, r->n_rot};
    return P8X_OK;
}

// head rows in and out; null: none
int check_heads(const char *fn, const p8x_heads *h, int D, HeadsDev &o) {
    o = {};
    if (!h || h->n == 0) return P8X_OK;
    if (h->n < 0) return set_error(P8X_ERR_ARG, "%s: %d heads", fn, h->n);
    if (h->n > 65535) return set_error(P8X_ERR_UNSUPPORTED, "%s: %d heads (at most 65535)", fn, h->n);
    if (!h->x || !h->out) return set_error(P8X_ERR_ARG, "%s: null heads x or out", fn);
    if (!is_float(h->dtype) || !is_float(h->out_dtype)) return set_error(P8X_ERR_ARG, "%s: heads dtypes %d %d", fn, h->dtype, h->out_dtype);
    o = {h->x, h->ld, h->head_stride ? h->head_stride : (size_t)D, h->out, h->ld_out, h->head_stride_out ? h->head_stride_out : (size_t)D, h->n, h->dtype, h->out_dtype};
    if (!rows_ok(o.x, o.dtype, o.ld, o.hs, o.n, D) || !rows_ok(o.out, o.out_dtype, o.ldo, o.hso, o.n, D))
        return set_error(P8X_ERR_ARG, "%s: heads' rows 16-byte aligned, strides %zu %zu to %zu %zu", fn, o.ld, o.hs, o.ldo, o.hso);
    if (o.x == o.out && (o.dtype != o.out_dtype || o.ld != o.ldo || o.hs != o.hso))
        return set_error(P8X_ERR_ARG, "%s: heads in place with another type or strides", fn);
    return P8X_OK;
}

}  // namespace
}  // namespace p8x

using namespace p8x;

extern "C" {

int p8x_norm_residual(const p8x_norm_args *a, void *stream) {
    const char *fn = "p8x_norm_residual";
    if (!a) return set_error(P8X_ERR_ARG, "%s: null arguments", fn);
    if (a->n < 0 || a->C < 1) return set_error(P8X_ERR_ARG, "%s: n %d C %d", fn, a->n, a->C);
    if (a->C > P8X_NORM_MAX_C) return set_error(P8X_ERR_UNSUPPORTED, "%s: C %d (at most %d)", fn, a->C, P8X_NORM_MAX_C);
    if (!a->h) return set_error(P8X_ERR_ARG, "%s: null h", fn);
    if (!a->h_out && !a->x) return set_error(P8X_ERR_ARG, "%s: neither h_out nor x", fn);
    if (!is_float(a->h_dtype) || (a->y && !is_float(a->y_dtype)) || (a->x && !is_float(a->x_dtype)) || (a->y && a->gate && !is_float(a->gate_dtype)))
        return set_error(P8X_ERR_ARG, "%s: dtypes y %d h %d x %d gate %d", fn, a->y_dtype, a->h_dtype, a->x_dtype, a->gate_dtype);
    if (a->post < P8X_NORM_NONE || a->post > P8X_NORM_LAYER || a->pre < P8X_NORM_NONE || a->pre > P8X_NORM_LAYER)
        return set_error(P8X_ERR_ARG, "%s: norms %d %d", fn, a->post, a->pre);
    if (a->gate && a->gate_act != P8X_GATE_LINEAR && a->gate_act != P8X_GATE_SIGMOID) return set_error(P8X_ERR_ARG, "%s: gate_act %d", fn, a->gate_act);
    const size_t C = (size_t)a->C;
    if (a->n > 1 && (a->ldh < C || (a->y && a->ldy < C) || (a->h_out && a->ldho < C) || (a->x && a->ldx < C) || (a->y && a->gate && a->ld_gate && a->ld_gate < C)))
        return set_error(P8X_ERR_ARG, "%s: a row stride below C %d", fn, a->C);
    const struct { const void *p; size_t to; } al[] = {{a->y, elem_size(a->y_dtype)}, {a->h, elem_size(a->h_dtype)}, {a->h_out, elem_size(a->h_dtype)},
                                                     {a->x, elem_size(a->x_dtype)}, {a->gate, elem_size(a->gate_dtype)}, {a->w_post, 4},
                                                     {a->b_post, 4}, {a->w_pre, 4}, {a->b_pre, 4}};
    for (const auto &e : al)
        if (!aligned(e.p, e.to)) return set_error(P8X_ERR_ARG, "%s: a pointer is not aligned to its elements", fn);
    if (a->n == 0) return P8X_OK;
    return launch_norm_residual(*a, (hipStream_t)stream);
}

int p8x_attn_tree(const p8x_kv_cache *c, const p8x_drafts *d, void *out, size_t ld_out, size_t head_stride_out, float *lse, void *workspace,
                  size_t workspace_bytes, void *stream) {
    const char *fn = "p8x_attn_tree";
    KvDev k;
    DraftDev q;
    int rc = check_cache(fn, c, k);
    if (!rc) rc = check_drafts(fn, c, d, true, true, true, P8X_MAX_DRAFT, q);
    if (rc) return rc;
    if (!d->n_tokens || !d->max_tokens) return P8X_OK;
    const size_t hs = head_stride_out ? head_stride_out : (size_t)c->head_dim;
    if (!out || !rows_ok(out, d->q_dtype, ld_out, hs, d->n_heads, c->head_dim))
        return set_error(P8X_ERR_ARG, "%s: out rows 16-byte aligned, strides %zu %zu", fn, ld_out, hs);
    if (workspace && !aligned(workspace, 16)) return set_error(P8X_ERR_ARG, "%s: workspace 16-byte aligned", fn);
    return launch_attn_tree(k, q, c->head_dim, out, ld_out, hs, lse, workspace, workspace ? workspace_bytes : 0, (hipStream_t)stream);
}

size_t p8x_attn_workspace(const p8x_kv_cache *c, const p8x_drafts *d) {
    KvDev k;
    DraftDev q;
    if (check_cache("p8x_attn_workspace", c, k) || check_drafts("p8x_attn_workspace", c, d, false, false, false, P8X_MAX_DRAFT, q)) return 0;
    if (d->n_heads < 1 || d->n_heads % c->n_kv || !d->n_tokens || !d->max_tokens) return 0;
    q.G = d->n_heads / c->n_kv;
    return attn_workspace(k, q, c->head_dim);
}

int p8x_kv_score(const p8x_kv_cache *c, const p8x_drafts *d, const uint64_t *accept, const float *lse, float decay, const float *score,
                 float *score_out, void *stream) {
    const char *fn = "p8x_kv_score";
    KvDev k;
    DraftDev q;
    int rc = check_cache(fn, c, k);
    if (!rc) rc = check_drafts(fn, c, d, true, false, true, P8X_MAX_DRAFT, q);
    if (rc) return rc;
    if (!lse || !score || !score_out) return set_error(P8X_ERR_ARG, "%s: null lse, score or score_out", fn);
    if (!(decay - decay == 0.0f)) return set_error(P8X_ERR_ARG, "%s: decay is not finite", fn);
    return launch_kv_score(k, q, c->head_dim, accept, lse, decay, score, score_out, (hipStream_t)stream);
}

int p8x_kv_append(const p8x_kv_cache *c, const p8x_drafts *d, const uint64_t *accept, const int32_t *at, int32_t *pos, int32_t *len_out,
                  void *stream) {
    const char *fn = "p8x_kv_append";
    KvDev k;
    DraftDev q;
    int rc = check_cache(fn, c, k);
    if (!rc) rc = check_drafts(fn, c, d, true, true, false, accept ? P8X_MAX_DRAFT : 0, q);
    if (rc) return rc;
    return launch_kv_append(k, q, c->head_dim, accept, at, pos, len_out, (hipStream_t)stream);
}

int p8x_rope_frequencies(const p8x_rope_scaling *s, int n_rot, uint64_t *freq, float *amplitude) {
    const char *fn = "p8x_rope_frequencies";
    if (!s || (n_rot && !freq)) return set_error(P8X_ERR_ARG, "%s: null arguments", fn);
    if (n_rot < 0 || n_rot % 2) return set_error(P8X_ERR_ARG, "%s: n_rot %d", fn, n_rot);
    auto positive = [](double v) { return v > 0 && v - v == 0; };
    const bool ends = s->kind == P8X_ROPE_BANDS || s->kind == P8X_ROPE_YARN;
    if (s->kind < P8X_ROPE_PLAIN || s->kind > P8X_ROPE_YARN || !positive(s->base) || (s->kind == P8X_ROPE_YARN && s->base <= 1) ||
        (s->kind != P8X_ROPE_PLAIN && !positive(s->factor)) || (ends && (!positive(s->original) || !positive(s->low) || !positive(s->high) || s->low >= s->high)))
        return set_error(P8X_ERR_ARG, "%s: kind %d base %g factor %g original %g low %g high %g", fn, s->kind, s->base, s->factor, s->original, s->low, s->high);
    const double pi2 = 6.283185307179586476925;
    // the (fractional) pair that makes so many turns in the original length: original theta_i = 2 pi turns
    auto pair_of = [&](double turns) { return n_rot * std::log(s->original / (turns * pi2)) / (2 * std::log(s->base)); };
    double lo = 0, hi = 0;
    if (s->kind == P8X_ROPE_YARN) {
        lo = std::fmax(0.0, std::floor(pair_of(s->high)));
        hi = std::fmin(n_rot - 1.0, std::ceil(pair_of(s->low)));
    }
    for (int i = 0; i < n_rot / 2; ++i) {
        double th = std::pow(s->base, -2.0 * i / n_rot);
        if (s->factors) {
            if (!positive(s->factors[i])) return set_error(P8X_ERR_ARG, "%s: factors[%d] %g", fn, i, s->factors[i]);
            th /= s->factors[i];
        }
        double far = 0;   // how much of the pair is divided by the factor
        if (s->kind == P8X_ROPE_LINEAR) far = 1;
        else if (s->kind == P8X_ROPE_BANDS) far = (s->high - s->original * th / pi2) / (s->high - s->low);
        else if (s->kind == P8X_ROPE_YARN) far = (i - lo) / std::fmax(hi - lo, 0.001);
        far = std::fmin(1.0, std::fmax(0.0, far));
        if (far > 0) th = far * (th / s->factor) + (1 - far) * th;
        const double turns = th / pi2, part = turns - std::floor(turns);   // whole turns do nothing
        if (!(turns - turns == 0)) return set_error(P8X_ERR_ARG, "%s: pair %d turns %g a position", fn, i, turns);
        const double scaled = std::nearbyint(std::ldexp(part, 64));
        freq[i] = scaled >= 18446744073709551616.0 ? 0 : (uint64_t)scaled;
    }
    if (amplitude) *amplitude = s->kind == P8X_ROPE_YARN && s->factor > 1 ? (float)(0.1 * std::log(s->factor) + 1) : 1.0f;
    return P8X_OK;
}

int p8x_rope(const p8x_rotation *r, int n_tokens, int head_dim, const int32_t *pos, const p8x_heads *q, const p8x_heads *k, void *stream) {
    const char *fn = "p8x_rope";
    TurnDev t;
    HeadsDev hq, hk;
    if (n_tokens < 0) return set_error(P8X_ERR_ARG, "%s: n_tokens %d", fn, n_tokens);
    if (head_dim < 8 || head_dim > 256 || head_dim % 8) return set_error(P8X_ERR_UNSUPPORTED, "%s: head_dim %d (a multiple of 8, 8 .. 256)", fn, head_dim);
    int rc = check_rotation(fn, r, head_dim, t);
    if (!rc) rc = check_heads(fn, q, head_dim, hq);
    if (!rc) rc = check_heads(fn, k, head_dim, hk);
    if (rc) return rc;
    if (!hq.n && !hk.n) return set_error(P8X_ERR_ARG, "%s: neither q nor k", fn);
    if (n_tokens == 0) return P8X_OK;
    if (!pos) return set_error(P8X_ERR_ARG, "%s: null pos", fn);
    return launch_rope(t, n_tokens, head_dim, pos, hq, hk, (hipStream_t)stream);
}

int p8x_kv_append_rope(const p8x_kv_cache *c, const p8x_drafts *d, const p8x_rotation *r, const int32_t *at, const p8x_heads *q, int32_t *pos,
                       int32_t *len_out, void *stream) {
    const char *fn = "p8x_kv_append_rope";
    KvDev k;
    DraftDev t;
    TurnDev turn;
    HeadsDev h;
    int rc = check_cache(fn, c, k);
    if (!rc) rc = check_drafts(fn, c, d, true, true, false, kMostTokens, t);
    if (!rc) rc = check_rotation(fn, r, c->head_dim, turn);
    if (!rc) rc = check_heads(fn, q, c->head_dim, h);
    if (rc) return rc;
    return launch_kv_append_rope(k, t, c->head_dim, turn, at, h, d->kv_dtype, pos, len_out, (hipStream_t)stream);
}

int p8x_attn_prompt(const p8x_kv_cache *c, const p8x_drafts *d, void *out, int out_dtype, size_t ld_out, size_t head_stride_out, float *lse,
                    void *workspace, size_t workspace_bytes, void *stream) {
    const char *fn = "p8x_attn_prompt";
    KvDev k;
    DraftDev q;
    int rc = check_cache(fn, c, k);
    if (!rc) rc = check_drafts(fn, c, d, false, false, true, kMostTokens, q);
    if (rc) return rc;
    if (d->mask) return set_error(P8X_ERR_ARG, "%s: a mask (its tokens see all before them)", fn);
    if (!is_float(out_dtype)) return set_error(P8X_ERR_ARG, "%s: out dtype %d", fn, out_dtype);
    if (!d->n_tokens || !d->max_tokens) return P8X_OK;
    // row tiles of 128 at least, 512 threads each: a launch has less than 2^32 (and rows of a sequence stay below 2^31)
    if (((int64_t)d->n_tokens * q.G / 128 + std::min(c->n_seq, d->n_tokens)) * c->n_kv >= 1 << 23)
        return set_error(P8X_ERR_UNSUPPORTED, "%s: %d tokens of %d sequences, %d heads (row tiles of 128: below 2^23)", fn, d->n_tokens, c->n_seq, d->n_heads);
    if (out_dtype == P8X_F32 && d->q_dtype != P8X_F32) return set_error(P8X_ERR_UNSUPPORTED, "%s: f32 out of 16-bit queries", fn);
    const size_t hs = head_stride_out ? head_stride_out : (size_t)c->head_dim;
    if (!out || !rows_ok(out, out_dtype, ld_out, hs, d->n_heads, c->head_dim))
        return set_error(P8X_ERR_ARG, "%s: out rows 16-byte aligned, strides %zu %zu", fn, ld_out, hs);
    if (workspace && !aligned(workspace, 16)) return set_error(P8X_ERR_ARG, "%s: workspace 16-byte aligned", fn);
    return launch_attn_prompt(k, q, c->head_dim, out, out_dtype, ld_out, hs, lse, workspace, workspace ? workspace_bytes : 0, (hipStream_t)stream);
}

size_t p8x_attn_prompt_workspace(const p8x_kv_cache *c, const p8x_drafts *d) {
    KvDev k;
    DraftDev q;
    if (check_cache("p8x_attn_prompt_workspace", c, k) || check_drafts("p8x_attn_prompt_workspace", c, d, false, false, false, 0, q)) return 0;
    if (d->n_heads < 1 || d->n_heads % c->n_kv || !d->n_tokens || !d->max_tokens) return 0;
    q.G = d->n_heads / c->n_kv;
    return attn_prompt_workspace(k, q, c->head_dim);
}

size_t p8x_kv_evict_workspace(const p8x_kv_cache *c, int budget) {
    KvDev k;
    if (check_cache("p8x_kv_evict_workspace", c, k) || budget < 1) return 0;
    return kv_evict_workspace(k, budget);
}

int p8x_kv_evict(const p8x_kv_cache *c, const p8x_evict_args *a, void *stream) {
    const char *fn = "p8x_kv_evict";
    KvDev k;
    if (int rc = check_cache(fn, c, k)) return rc;
    if (!a) return set_error(P8X_ERR_ARG, "%s: null arguments", fn);
    if (a->budget < 1 || a->n_sink < 0 || a->n_recent < 0 || a->n_sink > a->budget - a->n_recent)
        return set_error(P8X_ERR_ARG, "%s: budget %d n_sink %d n_recent %d", fn, a->budget, a->n_sink, a->n_recent);
    if (!a->score || !a->score_out || !a->len_out) return set_error(P8X_ERR_ARG, "%s: null score, score_out or len_out", fn);
    if (a->pos && !a->pos_out) return set_error(P8X_ERR_ARG, "%s: null pos_out", fn);
    if (!a->pos && (a->n_sink || a->n_recent)) return set_error(P8X_ERR_ARG, "%s: n_sink %d n_recent %d need pos", fn, a->n_sink, a->n_recent);
    const size_t need = kv_evict_workspace(k, a->budget);
    if (!a->workspace || !aligned(a->workspace, 16) || a->workspace_bytes < need)
        return set_error(P8X_ERR_ARG, "%s: workspace of %zu bytes, 16-byte aligned (given %zu)", fn, need, a->workspace ? a->workspace_bytes : 0);
    return launch_kv_evict(k, c->head_dim, *a, (hipStream_t)stream);
}

}  // extern "C"
