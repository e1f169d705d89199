// C entry points of the paged key/value cache (include/q3c.h, q3c_kv_*): every check that the host can make, then one launcher call.
// No context: nothing is allocated, nothing throws, and an error is its status code alone.
#include "kv.h"

namespace {

bool aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

int view(const q3c_kv* kv, KvView* c) {
    if (!kv || kv->struct_size != (int32_t)sizeof(q3c_kv)) return Q3C_ERR_INVALID_ARGUMENT;
    if (kv->dtype < Q3C_KV_F32 || kv->dtype > Q3C_KV_INT4) return Q3C_ERR_INVALID_ARGUMENT;
    if (kv->layers < 1 || kv->pages < 1 || kv->kv_heads < 1 || kv->rows < 1 || kv->pages_per_row < 1 || kv->head_dim < 1 || kv->page_size < 1)
        return Q3C_ERR_INVALID_ARGUMENT;
    if (!kv->k || !kv->v || !kv->table || !kv->lens || !kv->refs || !kv->status || !aligned(kv->k, 16) || !aligned(kv->v, 16))
        return Q3C_ERR_INVALID_ARGUMENT;
    int shift = 3;
    while (shift < 8 && (1 << shift) != kv->page_size) ++shift;
    if ((1 << shift) != kv->page_size || kv->head_dim % 16 || kv->head_dim > 256) return Q3C_ERR_UNSUPPORTED;
    const bool four = kv->dtype == Q3C_KV_INT4;
    if (four && kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256) return Q3C_ERR_UNSUPPORTED;
    if (four && (!kv->k_scale || !kv->v_scale || !aligned(kv->k_scale, 16) || !aligned(kv->v_scale, 16))) return Q3C_ERR_INVALID_ARGUMENT;
    if (kv->kv_heads > 65535 || (long long)kv->pages_per_row * kv->page_size > 0x40000000ll) return Q3C_ERR_UNSUPPORTED;   // grid y; int32 positions
    if ((long long)kv->kv_heads * kv->page_size * kv->head_dim * 4 >= 0x80000000ll) return Q3C_ERR_UNSUPPORTED;            // a page of one layer
    c->dtype = kv->dtype;
    c->layers = kv->layers; c->pages = kv->pages; c->heads = kv->kv_heads; c->ps_shift = shift; c->dim = kv->head_dim;
    c->rows = kv->rows; c->width = kv->pages_per_row;
    c->k = kv->k; c->v = kv->v; c->ks = (bf16*)kv->k_scale; c->vs = (bf16*)kv->v_scale;
    c->table = kv->table; c->lens = kv->lens; c->refs = kv->refs; c->status = kv->status;
    return 0;
}
int batch(const int32_t* rows, const int32_t* offsets, int32_t sequences, int32_t tokens, KvBatch* b) {
    if (sequences < 0 || tokens < 0 || (sequences > 0 && !rows)) return Q3C_ERR_INVALID_ARGUMENT;
    if (!offsets && tokens != sequences) return Q3C_ERR_INVALID_ARGUMENT;
    if (!sequences && tokens) return Q3C_ERR_INVALID_ARGUMENT;
    if (tokens > (1 << 24) || sequences > (1 << 24)) return Q3C_ERR_UNSUPPORTED;
    b->rows = rows; b->offsets = offsets; b->sequences = sequences; b->tokens = tokens;
    return 0;
}
// [token][head][dim] activations: read and written four elements at a time
bool strided(const void* p, int64_t ts, int64_t hs, size_t elem) { return p && aligned(p, 4 * elem) && ts % 4 == 0 && hs % 4 == 0 && ts >= 0 && hs >= 0; }
int done(hipError_t e) { return e == hipSuccess ? 0 : Q3C_ERR_HIP; }
size_t act_bytes(const KvView& c) { return c.dtype == Q3C_KV_F32 ? 4 : 2; }
// A launch has fewer than 2^32 threads along x: below 2^24 workgroups of 256.
constexpr long long MOST_BLOCKS = 1 << 24;
bool pieces_fit(const KvView& c, int count) {      // one workgroup per 16 KB of a pair
    const long long page = ((long long)c.heads << c.ps_shift) * c.dim * (c.dtype == Q3C_KV_F32 ? 4 : 2);
    return ((page + 16383) / 16384 * 4 * c.layers + 1) * count < MOST_BLOCKS;
}
bool heads_fit(int tokens, long long heads) {      // append, gather: at most a wave per head while tokens are few, per four of them beyond
    return tokens * heads < 8 * MOST_BLOCKS;
}

}  // namespace

extern "C" {

int q3c_kv_reserve(const q3c_kv* kv, const int32_t* rows, const int32_t* offsets, int32_t sequences, int32_t tokens, void* stream) {
    KvView c; KvBatch b;
    int rc = view(kv, &c);
    if (rc || (rc = batch(rows, offsets, sequences, tokens, &b))) return rc;
    return done(q3_launch_kv_reserve(c, b, (hipStream_t)stream));
}

int q3c_kv_append(const q3c_kv* kv, int32_t layer, const void* q, int64_t q_ts, int64_t q_hs, const void* k, int64_t k_ts, int64_t k_hs,
                  const void* v, int64_t v_ts, int64_t v_hs, int32_t q_heads, const int32_t* rows, const int32_t* offsets, int32_t sequences,
                  int32_t tokens, const float* q_weight, const float* k_weight, const float* cos_table, const float* sin_table, int64_t positions,
                  int32_t rot_dim, float eps, void* q_out, void* stream) {
    KvAppendArgs a = {};
    int rc = view(kv, &a.c);
    if (rc || (rc = batch(rows, offsets, sequences, tokens, &a.b))) return rc;
    if (layer < 0 || layer >= a.c.layers || q_heads < 1) return Q3C_ERR_INVALID_ARGUMENT;
    if (!tokens) return 0;
    const size_t e = act_bytes(a.c);
    if (!strided(q, q_ts, q_hs, e) || !strided(k, k_ts, k_hs, e) || !strided(v, v_ts, v_hs, e) || !q_out || !aligned(q_out, 16)) return Q3C_ERR_INVALID_ARGUMENT;
    if ((q_weight || k_weight) && !(eps > 0.f)) return Q3C_ERR_INVALID_ARGUMENT;
    if (!aligned(q_weight, 16) || !aligned(k_weight, 16)) return Q3C_ERR_INVALID_ARGUMENT;
    if (rot_dim < 0 || rot_dim > a.c.dim || rot_dim % 8) return Q3C_ERR_UNSUPPORTED;
    if (a.c.dtype == Q3C_KV_INT4 && rot_dim && rot_dim != a.c.dim) return Q3C_ERR_UNSUPPORTED;
    if (rot_dim && (!cos_table || !sin_table || !aligned(cos_table, 16) || !aligned(sin_table, 16))) return Q3C_ERR_INVALID_ARGUMENT;
    if (rot_dim && positions < ((int64_t)a.c.width << a.c.ps_shift)) return Q3C_ERR_INVALID_ARGUMENT;
    if (!heads_fit(tokens, q_heads + 2ll * a.c.heads)) return Q3C_ERR_UNSUPPORTED;
    a.layer = layer;
    a.q = {q, q_ts, q_hs}; a.k = {k, k_ts, k_hs}; a.v = {v, v_ts, v_hs};
    a.q_heads = q_heads;
    a.qw = q_weight; a.kw = k_weight; a.cos_t = cos_table; a.sin_t = sin_table;
    a.rot = rot_dim; a.eps = eps; a.inv_dim = 1.0f / (float)a.c.dim; a.q_out = q_out;
    return done(q3_launch_kv_append(a, (hipStream_t)stream));
}

int q3c_kv_gather(const q3c_kv* kv, int32_t layer, const int32_t* rows, const int32_t* offsets, int32_t sequences, int32_t tokens, void* k_out,
                  void* v_out, int32_t out_precision, void* stream) {
    KvView c; KvBatch b;
    int rc = view(kv, &c);
    if (rc || (rc = batch(rows, offsets, sequences, tokens, &b))) return rc;
    if (layer < 0 || layer >= c.layers || (out_precision != Q3C_PRECISION_F32 && out_precision != Q3C_PRECISION_BF16)) return Q3C_ERR_INVALID_ARGUMENT;
    if (!tokens) return 0;
    if (!k_out || !v_out || !aligned(k_out, 16) || !aligned(v_out, 16)) return Q3C_ERR_INVALID_ARGUMENT;
    if (!heads_fit(tokens, 2ll * c.heads)) return Q3C_ERR_UNSUPPORTED;
    return done(q3_launch_kv_gather(c, b, layer, k_out, v_out, out_precision == Q3C_PRECISION_F32 ? Q3_F32 : Q3_BF16, (hipStream_t)stream));
}

static int attend_shape(const q3c_kv* kv, int32_t q_heads, int32_t sequences, int32_t tokens, int32_t window, int32_t sinks, int32_t max_len, KvView* c) {
    const int rc = view(kv, c);
    if (rc) return rc;
    if (q_heads < 1 || q_heads % c->heads || sequences < 0 || tokens < 0 || window < 0 || sinks < 0 || max_len < 0) return Q3C_ERR_INVALID_ARGUMENT;
    // a workgroup per 16 columns along x, per 128 columns and kv head, or a wave per 16 columns and kv head
    const long long columns = (long long)tokens * (q_heads / c->heads), tiles = columns / 16 + sequences;
    if (tiles >= MOST_BLOCKS || (columns / 128 + sequences) * c->heads >= MOST_BLOCKS || tiles * c->heads >= 4 * MOST_BLOCKS) return Q3C_ERR_UNSUPPORTED;
    return 0;
}

int q3c_kv_attend_workspace_bytes(const q3c_kv* kv, int32_t q_heads, int32_t sequences, int32_t tokens, int32_t window, int32_t sinks,
                                  int32_t max_len, size_t* bytes) {
    KvView c;
    if (!bytes) return Q3C_ERR_INVALID_ARGUMENT;
    const int rc = attend_shape(kv, q_heads, sequences, tokens, window, sinks, max_len, &c);
    if (rc) return rc;
    size_t most = 0;                       // with offsets and, where there can be none, without
    for (int ragged = tokens == sequences ? 0 : 1; ragged < 2; ++ragged) {
        const size_t n = q3_kv_attend_ws(c, tokens, sequences, q_heads, ragged, q3_kv_attend_split(c, tokens, sequences, q_heads, ragged, window, sinks, max_len).splits);
        if (n > most) most = n;
    }
    *bytes = most;
    return 0;
}

int q3c_kv_attend(const q3c_kv* kv, int32_t layer, const void* q, int64_t q_ts, int64_t q_hs, int32_t q_heads, const int32_t* rows,
                  const int32_t* offsets, int32_t sequences, int32_t tokens, int32_t window, int32_t sinks, float scale, int32_t max_len, void* out,
                  void* workspace, size_t workspace_bytes, void* stream) {
    KvAttendArgs a = {};
    int rc = attend_shape(kv, q_heads, sequences, tokens, window, sinks, max_len, &a.c);
    if (rc || (rc = batch(rows, offsets, sequences, tokens, &a.b))) return rc;
    if (layer < 0 || layer >= a.c.layers || !(scale > 0.f) || !(scale < 1e37f)) return Q3C_ERR_INVALID_ARGUMENT;
    if (!tokens) return 0;
    if (!strided(q, q_ts, q_hs, act_bytes(a.c)) || !out || !aligned(out, 16)) return Q3C_ERR_INVALID_ARGUMENT;
    const KvSplit cut = q3_kv_attend_split(a.c, tokens, sequences, q_heads, offsets != nullptr, window, sinks, max_len);
    a.splits = cut.splits;
    a.share = cut.share;
    a.most = cut.most;
    const size_t need = q3_kv_attend_ws(a.c, tokens, sequences, q_heads, offsets != nullptr, a.splits);
    if (need && (!workspace || !aligned(workspace, 16))) return Q3C_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < need) return Q3C_ERR_WORKSPACE;
    a.layer = layer;
    a.q = {q, q_ts, q_hs};
    a.q_heads = q_heads; a.group = q_heads / a.c.heads; a.window = window; a.sinks = sinks;
    a.scale_log2e = scale * 1.44269504088896340736f;
    a.out = out;
    a.ws = (float*)workspace;
    return done(q3_launch_kv_attend(a, (hipStream_t)stream));
}

int q3c_kv_fork(const q3c_kv* kv, const int32_t* parents, const int32_t* children, int32_t count, void* workspace, size_t workspace_bytes, void* stream) {
    KvView c;
    const int rc = view(kv, &c);
    if (rc) return rc;
    if (count < 0 || (count && (!parents || !children || !workspace || !aligned(workspace, 4)))) return Q3C_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < 12ull * count) return Q3C_ERR_WORKSPACE;
    if (!pieces_fit(c, count)) return Q3C_ERR_UNSUPPORTED;
    return done(q3_launch_kv_fork(c, parents, children, count, (int*)workspace, (hipStream_t)stream));
}
int q3c_kv_release(const q3c_kv* kv, const int32_t* rows, int32_t count, void* stream) {
    KvView c;
    const int rc = view(kv, &c);
    if (rc) return rc;
    if (count < 0 || (count && !rows)) return Q3C_ERR_INVALID_ARGUMENT;
    if (count >= MOST_BLOCKS) return Q3C_ERR_UNSUPPORTED;
    return done(q3_launch_kv_release(c, rows, count, 0, 0, 0, (hipStream_t)stream));
}
int q3c_kv_trim(const q3c_kv* kv, const int32_t* rows, int32_t count, int32_t window, int32_t sinks, void* stream) {
    KvView c;
    const int rc = view(kv, &c);
    if (rc) return rc;
    if (count < 0 || (count && !rows) || window < 1 || sinks < 0) return Q3C_ERR_INVALID_ARGUMENT;
    if (count >= MOST_BLOCKS) return Q3C_ERR_UNSUPPORTED;
    return done(q3_launch_kv_release(c, rows, count, 1, window, sinks, (hipStream_t)stream));
}
int q3c_kv_copy_pages(const q3c_kv* kv, const int32_t* src, const int32_t* dst, int32_t count, void* workspace, size_t workspace_bytes, void* stream) {
    KvView c;
    const int rc = view(kv, &c);
    if (rc) return rc;
    if (count < 0 || (count && (!src || !dst || !workspace || !aligned(workspace, 4)))) return Q3C_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < 4ull * count) return Q3C_ERR_WORKSPACE;
    if (!pieces_fit(c, count)) return Q3C_ERR_UNSUPPORTED;
    return done(q3_launch_kv_copy(c, src, dst, count, (int*)workspace, (hipStream_t)stream));
}
int q3c_kv_compact(const q3c_kv* kv, int32_t* live_dev, void* workspace, size_t workspace_bytes, void* stream) {
    KvView c;
    const int rc = view(kv, &c);
    if (rc) return rc;
    if (!live_dev || !workspace || !aligned(workspace, 4)) return Q3C_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < 8ull * c.pages + 16) return Q3C_ERR_WORKSPACE;
    return done(q3_launch_kv_compact(c, live_dev, (int*)workspace, (hipStream_t)stream));
}

}  // extern "C"
