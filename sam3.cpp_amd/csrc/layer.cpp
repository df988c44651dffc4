// C-ABI entry points of the nodes around a layer's products: RMS norm with the residual and an 8-bit
// output, dequantized rows, rotary positions, the 8-bit key/value cache and its attention.
#include <climits>
#include <cmath>

#include "context.h"

using namespace mi355;

namespace {

bool is_float(int t) { return t == T_F32 || t == T_F16; }

// an empty tensor needs no data
bool empty(const mi355_tensor* t) { return t->ne[0] == 0 || t->ne[1] == 0 || t->ne[2] == 0 || t->ne[3] == 0; }
bool has_data(const mi355_tensor* t) { return t->data || empty(t); }
// every row of t starts on `bytes`
bool rows_on(const mi355_tensor* t, uintptr_t bytes) {
    return ((reinterpret_cast<uintptr_t>(t->data) | (uintptr_t)t->nb[1] | (uintptr_t)t->nb[2] | (uintptr_t)t->nb[3]) &
            (bytes - 1)) == 0;
}
// rows of contiguous elements, on the element's own size (blocks: on that of their fields)
bool rows_ok(const mi355_tensor* t) {
    return t->nb[0] == type_size(t->type) && rows_on(t, t->type == T_F32 || t->type == T_Q8_1 ? 4 : 2);
}
bool same_ne(const mi355_tensor* a, const mi355_tensor* b) {
    for (int i = 0; i < 4; ++i)
        if (a->ne[i] != b->ne[i]) return false;
    return true;
}
bool int32_dims(const mi355_tensor* t) {
    for (int i = 0; i < 4; ++i)
        if (t->ne[i] > INT_MAX) return false;
    return true;
}
// rows times anything below stays within int64 and a launch within its limit
bool rows_fit(const mi355_tensor* t) {
    return int32_dims(t) && (double)t->ne[1] * (double)t->ne[2] * (double)t->ne[3] < 2147483647.0;
}
RowSpan span_of(const mi355_tensor* t) {
    RowSpan s{nullptr, {0, 0, 0}};
    if (!t) return s;
    s.base = static_cast<char*>(t->data);
    for (int i = 0; i < 3; ++i) s.nb[i] = t->nb[i + 1];
    return s;
}
void strides(const mi355_tensor* t, int64_t nb[3]) {
    for (int i = 0; i < 3; ++i) nb[i] = t->nb[i + 1];
}

mi355_status check_rms_norm(mi355_context* ctx, const mi355_tensor* x, const mi355_tensor* add, const mi355_tensor* sum,
                            const mi355_tensor* dst) {
    if (!x || !dst || !has_data(x) || !has_data(dst) || (add && !has_data(add)) || (sum && !has_data(sum)))
        return fail(ctx, MI355_STATUS_INVALID_ARG, "rms_norm: null argument");
    const mi355_tensor* all[4] = {x, dst, add, sum};
    for (const mi355_tensor* t : all)
        if (t && !dims_ok(t)) return fail(ctx, MI355_STATUS_INVALID_ARG, "rms_norm: negative ne/nb or not the ggml layout");
    if (!is_float(x->type)) return fail(ctx, MI355_STATUS_UNSUPPORTED, "rms_norm: x must be F32 or F16");
    if (!(is_float(dst->type) || dst->type == T_Q8_0 || dst->type == T_Q8_1))
        return fail(ctx, MI355_STATUS_UNSUPPORTED, "rms_norm: dst type %d not supported", dst->type);
    if ((add && add->type != x->type) || (sum && sum->type != x->type))
        return fail(ctx, MI355_STATUS_UNSUPPORTED, "rms_norm: add and sum must have x's type");
    for (const mi355_tensor* t : all)
        if (t && !same_ne(t, x)) return fail(ctx, MI355_STATUS_INVALID_ARG, "rms_norm: shape mismatch");
    if (!is_float(dst->type) && x->ne[0] % 32 != 0)
        return fail(ctx, MI355_STATUS_INVALID_ARG, "rms_norm: ne0 not a multiple of the block size");
    for (const mi355_tensor* t : all)
        if (t && !rows_ok(t)) return fail(ctx, MI355_STATUS_UNSUPPORTED, "rms_norm: rows must be contiguous and aligned to their type");
    if (x->ne[0] > RMS_MAX || !rows_fit(x))
        return fail(ctx, MI355_STATUS_UNSUPPORTED, "rms_norm: rows longer than %d, or too many", RMS_MAX);
    return MI355_STATUS_SUCCESS;
}

// The axis and turns a position of every pair; false: the parameters do not fit together.
bool rope_table(const mi355_rope_params* p, RopeArgs* a) {
    if (p->n_dims < 2 || p->n_dims % 2 != 0 || p->n_dims > 2 * ROPE_PAIRS) return false;
    if (p->pairs != MI355_ROPE_ADJACENT && p->pairs != MI355_ROPE_HALVES) return false;
    if (p->order != MI355_ROPE_CONSECUTIVE && p->order != MI355_ROPE_INTERLEAVED) return false;
    if ((p->restart | 1) != 1 || (p->inverse | 1) != 1) return false;
    if (!(p->freq_base > 0.0f) || !std::isfinite(p->freq_base) || !std::isfinite(p->freq_scale)) return false;
    const int n = p->n_dims / 2;
    int64_t total = 0;
    for (int s : p->sections) {
        if (s < 0) return false;
        total += s;
    }
    if (total != n || (p->order == MI355_ROPE_INTERLEAVED && p->sections[3] != 0)) return false;
    // freq_base ^ (-2^k / size) by squaring, of one size or each axis's: a power is a product of at most seven.
    // The 64-bit mantissas' error doubles with every squaring and is a relative e 2^-63 at pair e, which bases far from one
    // make small beside what follows; the products below one are made in 64-bit fixed point (eight truncations: 2^-61 of a
    // turn, 2^-30 at the ends of int32's positions), a tenth of the time of the floating ones.
    long double root[4][7];
    uint64_t fixed[4][7];
    const long double unit = (long double)p->freq_scale / 6.283185307179586476925286766559L, two64 = 18446744073709551616.0L;
    bool below = unit >= 0.0L && unit < 1.0L;
    if (a)
        for (int s = 0; s < (p->restart ? 4 : 1); ++s) {
            const int size = p->restart ? p->sections[s] : n;
            if (size == 0) continue;
            root[s][0] = powl((long double)p->freq_base, -1.0L / (long double)size);
            for (int k = 1; k < 7; ++k) root[s][k] = root[s][k - 1] * root[s][k - 1];
            below = below && root[s][0] < 1.0L;
            for (int k = 0; below && k < 7; ++k) fixed[s][k] = (uint64_t)(root[s][k] * two64);
        }
    const uint64_t unit64 = below ? (uint64_t)(unit * two64) : 0;
    int count[4] = {0, 0, 0, 0}, axis = 0;
    for (int i = 0; i < n; ++i) {
        if (p->order == MI355_ROPE_INTERLEAVED) {
            axis = i % 3;
            if (axis != 0 && i >= 3 * p->sections[axis]) axis = 0;
        } else {
            while (count[axis] == p->sections[axis]) ++axis;  // total == n: an axis with room is left
        }
        const int e = p->restart ? count[axis] : i;
        ++count[axis];
        if (!a) continue;
        const int s = p->restart ? axis : 0;
        uint64_t turn = unit64;
        if (below) {
            for (int k = 0, b = e; b; ++k, b >>= 1)
                if (b & 1) turn = (uint64_t)(((unsigned __int128)turn * fixed[s][k]) >> 64);
        } else {
            long double f = unit;
            for (int k = 0; k < 7; ++k)
                if (e >> k & 1) f *= root[s][k];
            f -= floorl(f);
            turn = f < 1.0L ? (uint64_t)(f * two64) : 0;
        }
        a->turn[i] = p->inverse ? 0 - turn : turn;
        a->axis[i] = (uint8_t)axis;
    }
    for (int s = 0; s < 4; ++s)
        if (count[s] != p->sections[s]) return false;
    return true;
}

mi355_status check_rope(mi355_context* ctx, const mi355_tensor* src, const mi355_rope_params* p, const mi355_tensor* dst,
                        RopeArgs* a) {
    if (!src || !p || !dst || !has_data(src) || !has_data(dst)) return fail(ctx, MI355_STATUS_INVALID_ARG, "rope_multi: null argument");
    if (!dims_ok(src) || !dims_ok(dst)) return fail(ctx, MI355_STATUS_INVALID_ARG, "rope_multi: negative ne/nb or not the ggml layout");
    if (!rope_table(p, a)) return fail(ctx, MI355_STATUS_INVALID_ARG, "rope_multi: parameters out of range, or sections that do not make n_dims / 2 pairs");
    if (!is_float(src->type) || dst->type != src->type) return fail(ctx, MI355_STATUS_UNSUPPORTED, "rope_multi: src and dst must both be F32 or F16");
    if (!same_ne(src, dst)) return fail(ctx, MI355_STATUS_INVALID_ARG, "rope_multi: shape mismatch");
    if (p->n_dims > src->ne[0]) return fail(ctx, MI355_STATUS_INVALID_ARG, "rope_multi: n_dims %d beyond ne0", p->n_dims);
    if (!rows_ok(src) || !rows_ok(dst)) return fail(ctx, MI355_STATUS_UNSUPPORTED, "rope_multi: rows must be contiguous and aligned to their type");
    if (!rows_fit(src) || src->ne[0] > 65536 || (double)src->ne[2] * src->ne[3] * ((src->ne[1] + 3) / 4) * (src->ne[0] / 8 + 2) > 2147483000.0)
        return fail(ctx, MI355_STATUS_UNSUPPORTED, "rope_multi: sizes beyond the launch limits");
    return MI355_STATUS_SUCCESS;
}

mi355_status check_cache(mi355_context* ctx, const char* op, const mi355_kv_cache* c, const mi355_kv_seqs* s) {
    if (!c || !s || (c->n_blocks && (!c->k || !c->v || !c->k_scale || !c->v_scale)) || (!s->table && s->n_seq && s->max_blocks) ||
        (!s->n_kv && s->n_seq))
        return fail(ctx, MI355_STATUS_INVALID_ARG, "%s: null argument", op);
    if (c->n_blocks < 0 || c->n_head_kv < 1 || s->n_seq < 0 || s->max_blocks < 0)
        return fail(ctx, MI355_STATUS_INVALID_ARG, "%s: negative cache or sequence sizes, or no heads", op);
    if (!(c->block_tokens == 16 || c->block_tokens == 32 || c->block_tokens == 64 || c->block_tokens == 128))
        return fail(ctx, MI355_STATUS_UNSUPPORTED, "%s: block_tokens %d (supported: 16, 32, 64, 128)", op, c->block_tokens);
    if (!(c->head_dim == 64 || c->head_dim == 96 || c->head_dim == 128))
        return fail(ctx, MI355_STATUS_UNSUPPORTED, "%s: head size %d (supported: 64, 96, 128)", op, c->head_dim);
    if (((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) ||
        ((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale) | reinterpret_cast<uintptr_t>(s->table) |
          reinterpret_cast<uintptr_t>(s->n_kv)) & 3))
        return fail(ctx, MI355_STATUS_INVALID_ARG, "%s: the cache must be 16-byte aligned, scales, table and lengths 4-byte", op);
    if (c->n_head_kv > 65535 || s->n_seq > 65535 || (int64_t)s->max_blocks * c->block_tokens > 1 << 30)
        return fail(ctx, MI355_STATUS_UNSUPPORTED, "%s: sizes beyond the launch limits", op);
    return MI355_STATUS_SUCCESS;
}

KvView kv_view(const mi355_kv_cache* c, const mi355_kv_seqs* s) {
    KvView v;
    v.k = c->k; v.v = c->v; v.k_scale = c->k_scale; v.v_scale = c->v_scale;
    v.n_blocks = c->n_blocks; v.heads = c->n_head_kv; v.bt = c->block_tokens;
    v.bt_log2 = __builtin_ctz((unsigned)c->block_tokens);
    v.table = s->table; v.n_kv = s->n_kv; v.n_seq = s->n_seq; v.max_blocks = s->max_blocks;
    return v;
}

// k and v [head_dim, n_tokens, n_head_kv, n_seq] of a write or read (either null only when reading)
mi355_status kv_rows(mi355_context* ctx, const char* op, const mi355_kv_cache* c, const mi355_kv_seqs* s, const mi355_tensor* k,
                     const mi355_tensor* v, const int32_t* idx, KvRows* r) {
    const mi355_tensor* one = k ? k : v;
    r->k = r->v = nullptr;
    for (const mi355_tensor* t : {k, v}) {
        if (!t) continue;
        if (!has_data(t)) return fail(ctx, MI355_STATUS_INVALID_ARG, "%s: null data pointer", op);
        if (!dims_ok(t)) return fail(ctx, MI355_STATUS_INVALID_ARG, "%s: negative ne/nb or not the ggml layout", op);
        if (!is_float(t->type) || t->type != one->type) return fail(ctx, MI355_STATUS_UNSUPPORTED, "%s: k and v must both be F32 or F16", op);
        if (!same_ne(t, one) || t->ne[0] != c->head_dim || t->ne[2] != c->n_head_kv || t->ne[3] != s->n_seq)
            return fail(ctx, MI355_STATUS_INVALID_ARG, "%s: k and v must be [head_dim, n_tokens, n_head_kv, n_seq]", op);
        if (!rows_ok(t)) return fail(ctx, MI355_STATUS_UNSUPPORTED, "%s: rows must be contiguous and aligned to their type", op);
        if (!rows_fit(t)) return fail(ctx, MI355_STATUS_UNSUPPORTED, "%s: sizes beyond the launch limits", op);
    }
    if (reinterpret_cast<uintptr_t>(idx) & 3) return fail(ctx, MI355_STATUS_INVALID_ARG, "%s: counts and positions must be 4-byte aligned", op);
    if (k) { r->k = static_cast<char*>(k->data); strides(k, r->k_nb); }
    if (v) { r->v = static_cast<char*>(v->data); strides(v, r->v_nb); }
    r->n_tok = (int)one->ne[1];
    r->f16 = one->type == T_F16;
    r->idx = idx;
    return MI355_STATUS_SUCCESS;
}

mi355_status check_attn(mi355_context* ctx, const mi355_kv_cache* c, const mi355_kv_seqs* s, const mi355_tensor* q,
                        const mi355_tensor* dst) {
    const mi355_status st = check_cache(ctx, "kv_cache_attn", c, s);
    if (st != MI355_STATUS_SUCCESS) return st;
    if (!q || !dst || !has_data(q) || !has_data(dst)) return fail(ctx, MI355_STATUS_INVALID_ARG, "kv_cache_attn: null argument");
    if (!dims_ok(q) || !dims_ok(dst)) return fail(ctx, MI355_STATUS_INVALID_ARG, "kv_cache_attn: negative ne/nb or not the ggml layout");
    if (!is_float(q->type) || !is_float(dst->type)) return fail(ctx, MI355_STATUS_UNSUPPORTED, "kv_cache_attn: q and dst must be F32 or F16");
    if (q->ne[0] != c->head_dim || q->ne[3] != s->n_seq || q->ne[2] < 1 || q->ne[2] % c->n_head_kv != 0)
        return fail(ctx, MI355_STATUS_INVALID_ARG, "kv_cache_attn: q must be [head_dim, n_q, n_head, n_seq], n_head a multiple of n_head_kv");
    if (dst->ne[0] != q->ne[0] || dst->ne[1] != q->ne[2] || dst->ne[2] != q->ne[1] || dst->ne[3] != q->ne[3])
        return fail(ctx, MI355_STATUS_INVALID_ARG, "kv_cache_attn: dst must be [head_dim, n_head, n_q, n_seq]");
    if (!rows_ok(q) || !rows_ok(dst)) return fail(ctx, MI355_STATUS_UNSUPPORTED, "kv_cache_attn: rows must be contiguous and aligned to their type");
    if (!rows_fit(q) || q->ne[2] > 65535 || q->ne[1] > INT_MAX / 2) return fail(ctx, MI355_STATUS_UNSUPPORTED, "kv_cache_attn: sizes beyond the launch limits");
    return MI355_STATUS_SUCCESS;
}

KvAttnPlan attn_plan(const mi355_context* ctx, const mi355_kv_cache* c, const mi355_kv_seqs* s, const mi355_tensor* q,
                     int window) {
    return kv_attn_plan((int)q->ne[1], (int)q->ne[2], c->n_head_kv, s->n_seq, (int64_t)s->max_blocks * c->block_tokens, window, c->head_dim,
                        q->type == T_F16, ctx->cus);
}

}  // namespace

extern "C" {

int mi355_supports_rms_norm(const mi355_tensor* x, const mi355_tensor* add, const mi355_tensor* sum, const mi355_tensor* dst) {
    return check_rms_norm(nullptr, x, add, sum, dst) == MI355_STATUS_SUCCESS;
}

mi355_status mi355_rms_norm(mi355_context* ctx, const mi355_tensor* x, const mi355_tensor* add, const float* w, float eps,
                            const mi355_tensor* sum, const mi355_tensor* dst) {
    const mi355_status st = check_rms_norm(ctx, x, add, sum, dst);
    if (st != MI355_STATUS_SUCCESS) return st;
    if (reinterpret_cast<uintptr_t>(w) & 3) return fail(ctx, MI355_STATUS_INVALID_ARG, "rms_norm: w must be 4-byte aligned");
    if (!(eps >= 0.0f)) return fail(ctx, MI355_STATUS_INVALID_ARG, "rms_norm: eps must not be negative");
    if (!ctx) return fail(nullptr, MI355_STATUS_INVALID_ARG, "rms_norm: null context");
    (void)hipSetDevice(ctx->device);
    RmsArgs a;
    a.x = span_of(x); a.add = span_of(add); a.sum = span_of(sum); a.dst = span_of(dst);
    a.w = w;
    a.ne1 = x->ne[1]; a.ne2 = x->ne[2];
    a.rows = x->ne[1] * x->ne[2] * x->ne[3];
    a.n = (int)x->ne[0];
    a.eps = eps;
    a.xf16 = x->type == T_F16;
    a.out = dst->type;
    Timed tm(ctx, "rms_norm");
    return hip_check(ctx, tm.done(launch_rms_norm(a, ctx->stream)), "rms_norm launch");
}

mi355_status mi355_dequantize_rows(mi355_context* ctx, int type, const void* src, const mi355_tensor* dst) {
    if (!dst || !has_data(dst) || (!src && !empty(dst))) return fail(ctx, MI355_STATUS_INVALID_ARG, "dequantize_rows: null argument");
    if (!dims_ok(dst)) return fail(ctx, MI355_STATUS_INVALID_ARG, "dequantize_rows: negative ne/nb or not the ggml layout");
    if (!(type == T_Q8_0 || type == T_Q8_1 || type == T_Q4_0 || type == T_Q4_1))
        return fail(ctx, MI355_STATUS_UNSUPPORTED, "dequantize_rows: type %d not supported", type);
    if (!is_float(dst->type)) return fail(ctx, MI355_STATUS_UNSUPPORTED, "dequantize_rows: dst must be F32 or F16");
    if (dst->ne[0] % 32 != 0) return fail(ctx, MI355_STATUS_INVALID_ARG, "dequantize_rows: ne0 not a multiple of the block size");
    if (!rows_ok(dst)) return fail(ctx, MI355_STATUS_UNSUPPORTED, "dequantize_rows: rows must be contiguous and aligned to their type");
    if (reinterpret_cast<uintptr_t>(src) & (type == T_Q8_1 ? 3 : 1))
        return fail(ctx, MI355_STATUS_INVALID_ARG, "dequantize_rows: src must be 2-byte (Q8_1: 4-byte) aligned");
    if (!rows_fit(dst) || dst->ne[0] > INT_MAX) return fail(ctx, MI355_STATUS_UNSUPPORTED, "dequantize_rows: sizes beyond the launch limits");
    if (!ctx) return fail(nullptr, MI355_STATUS_INVALID_ARG, "dequantize_rows: null context");
    (void)hipSetDevice(ctx->device);
    Timed tm(ctx, "dequantize_rows");
    return hip_check(ctx, tm.done(launch_dequantize_rows(src, type, span_of(dst), dst->type == T_F16, dst->ne[0],
                                                         dst->ne[1] * dst->ne[2] * dst->ne[3], dst->ne[1], dst->ne[2], ctx->stream)),
                     "dequantize_rows launch");
}

int mi355_supports_rope_multi(const mi355_tensor* src, const mi355_rope_params* p, const mi355_tensor* dst) {
    return check_rope(nullptr, src, p, dst, nullptr) == MI355_STATUS_SUCCESS;
}

mi355_status mi355_rope_multi(mi355_context* ctx, const mi355_tensor* src, const int32_t* pos, const mi355_rope_params* p,
                              const mi355_tensor* dst) {
    RopeArgs a;
    const mi355_status st = check_rope(ctx, src, p, dst, &a);
    if (st != MI355_STATUS_SUCCESS) return st;
    if ((!pos && !empty(src)) || (reinterpret_cast<uintptr_t>(pos) & 3)) return fail(ctx, MI355_STATUS_INVALID_ARG, "rope_multi: pos null or not 4-byte aligned");
    if (!ctx) return fail(nullptr, MI355_STATUS_INVALID_ARG, "rope_multi: null context");
    (void)hipSetDevice(ctx->device);
    a.src = static_cast<const char*>(src->data);
    a.dst = static_cast<char*>(dst->data);
    strides(src, a.s_nb);
    strides(dst, a.d_nb);
    a.ne0 = (int)src->ne[0]; a.heads = (int)src->ne[1]; a.tokens = (int)src->ne[2]; a.batch = (int)src->ne[3];
    a.pairs = p->n_dims / 2;
    a.f16 = src->type == T_F16;
    a.halves = p->pairs == MI355_ROPE_HALVES;
    a.pos = pos;
    Timed tm(ctx, "rope_multi");
    return hip_check(ctx, tm.done(launch_rope_multi(a, ctx->stream)), "rope_multi launch");
}

mi355_status mi355_kv_cache_write(mi355_context* ctx, const mi355_kv_cache* cache, const mi355_kv_seqs* seqs, const mi355_tensor* k,
                                  const mi355_tensor* v, const int32_t* n_new) {
    mi355_status st = check_cache(ctx, "kv_cache_write", cache, seqs);
    if (st != MI355_STATUS_SUCCESS) return st;
    if (!k || !v) return fail(ctx, MI355_STATUS_INVALID_ARG, "kv_cache_write: null argument");
    KvRows r;
    st = kv_rows(ctx, "kv_cache_write", cache, seqs, k, v, n_new, &r);
    if (st != MI355_STATUS_SUCCESS) return st;
    if (!ctx) return fail(nullptr, MI355_STATUS_INVALID_ARG, "kv_cache_write: null context");
    (void)hipSetDevice(ctx->device);
    Timed tm(ctx, "kv_cache_write");
    return hip_check(ctx, tm.done(launch_kv_write(kv_view(cache, seqs), r, cache->head_dim, ctx->stream)), "kv_cache_write launch");
}

mi355_status mi355_kv_cache_read(mi355_context* ctx, const mi355_kv_cache* cache, const mi355_kv_seqs* seqs, const int32_t* pos,
                                 const mi355_tensor* k, const mi355_tensor* v) {
    mi355_status st = check_cache(ctx, "kv_cache_read", cache, seqs);
    if (st != MI355_STATUS_SUCCESS) return st;
    if (!k && !v) return fail(ctx, MI355_STATUS_INVALID_ARG, "kv_cache_read: neither k nor v");
    KvRows r;
    st = kv_rows(ctx, "kv_cache_read", cache, seqs, k, v, pos, &r);
    if (st != MI355_STATUS_SUCCESS) return st;
    if (!ctx) return fail(nullptr, MI355_STATUS_INVALID_ARG, "kv_cache_read: null context");
    (void)hipSetDevice(ctx->device);
    Timed tm(ctx, "kv_cache_read");
    return hip_check(ctx, tm.done(launch_kv_read(kv_view(cache, seqs), r, cache->head_dim, ctx->stream)), "kv_cache_read launch");
}

int mi355_supports_kv_cache_attn(const mi355_kv_cache* cache, const mi355_kv_seqs* seqs, const mi355_tensor* q, const mi355_tensor* dst) {
    return check_attn(nullptr, cache, seqs, q, dst) == MI355_STATUS_SUCCESS;
}

size_t mi355_kv_cache_attn_workspace_size(const mi355_context* ctx, const mi355_kv_cache* cache, const mi355_kv_seqs* seqs,
                                          const mi355_tensor* q, int32_t window) {
    if (!ctx || !cache || !seqs || !q || q->ne[0] * q->ne[1] * q->ne[2] * q->ne[3] == 0 || cache->n_head_kv < 1) return 0;
    return attn_plan(ctx, cache, seqs, q, window).bytes;
}

mi355_status mi355_kv_cache_attn(mi355_context* ctx, const mi355_kv_cache* cache, const mi355_kv_seqs* seqs, const mi355_tensor* q,
                                 const int32_t* n_q, float scale, int causal, int32_t window, const mi355_tensor* dst) {
    const mi355_status st = check_attn(ctx, cache, seqs, q, dst);
    if (st != MI355_STATUS_SUCCESS) return st;
    if (reinterpret_cast<uintptr_t>(n_q) & 3) return fail(ctx, MI355_STATUS_INVALID_ARG, "kv_cache_attn: n_q must be 4-byte aligned");
    if (!std::isfinite(scale) || window < 0 || (causal | 1) != 1)
        return fail(ctx, MI355_STATUS_INVALID_ARG, "kv_cache_attn: scale must be finite, window not negative, causal 0 or 1");
    if (!ctx) return fail(nullptr, MI355_STATUS_INVALID_ARG, "kv_cache_attn: null context");
    (void)hipSetDevice(ctx->device);
    KvAttnArgs a;
    a.c = kv_view(cache, seqs);
    a.q = static_cast<const char*>(q->data);
    a.dst = static_cast<char*>(dst->data);
    strides(q, a.q_nb);
    strides(dst, a.d_nb);
    a.n_q = (int)q->ne[1]; a.heads = (int)q->ne[2];
    a.group = a.heads / cache->n_head_kv;
    a.nq = n_q;
    a.scale = scale; a.causal = causal;
    a.window = window < 1 << 30 ? window : 1 << 30;
    a.q16 = q->type == T_F16; a.d16 = dst->type == T_F16;
    if (cache->n_blocks == 0) a.c.max_blocks = 0;  // nothing to attend to
    if ((int64_t)a.n_q * a.heads * a.c.n_seq == 0) return MI355_STATUS_SUCCESS;
    const KvAttnPlan p = attn_plan(ctx, cache, seqs, q, a.window);
    mi355_status ws = p.nt && p.splits > 1 ? ensure_arrived(ctx) : MI355_STATUS_SUCCESS;
    if (ws == MI355_STATUS_SUCCESS) ws = ensure_ws(ctx, p.bytes, false);
    if (ws != MI355_STATUS_SUCCESS) return ws;
    a.part = static_cast<float*>(ctx->ws);
    a.arrived = static_cast<uint32_t*>(ctx->arrived);
    Timed tm(ctx, p.nt == 0 ? "kv_cache_attn_128" : p.nt == 2 ? "kv_cache_attn_32" : "kv_cache_attn_16");  // by the rows of a workgroup
    return hip_check(ctx, tm.done(launch_kv_attn(a, p, cache->head_dim, ctx->stream)), "kv_cache_attn launch");
}

}  // extern "C"
