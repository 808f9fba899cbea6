// Attention: argument checks and workspaces of tvl_attention, tvl_attention_backward and tvl_cached_attention.  See include/tvl.h.
#include "attention_tiles.h"

namespace tvl {

// rows of a written tensor must not share elements: strides sorted, each at least the extent of what lies inside it
static bool rows_apart(int64_t dim, int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t n2, int64_t s2) {
    int64_t n[3] = {n0, n1, n2}, s[3] = {s0, s1, s2}, extent = dim;
    for (int x = 0; x < 3; ++x)
        for (int y = 0; y + 1 < 3; ++y)
            if (s[y] > s[y + 1]) {
                const int64_t ts = s[y], tn = n[y];
                s[y] = s[y + 1]; n[y] = n[y + 1];
                s[y + 1] = ts; n[y + 1] = tn;
            }
    for (int x = 0; x < 3; ++x) {
        if (n[x] <= 1) continue;
        if (s[x] < extent) return false;
        extent = s[x] * (n[x] - 1) + extent;
    }
    return true;
}

// the checks that the three entry points share
static int check(const tvl_attention_args* a, const char* who, bool cached) {
    TVL_REQUIRE(a && a->struct_bytes == sizeof(tvl_attention_args), "%s: NULL argument block or one of another size than %zu bytes", who, sizeof(tvl_attention_args));
    TVL_REQUIRE(a->dtype == TVL_F32 || a->dtype == TVL_F16 || a->dtype == TVL_BF16, "%s: dtype must be f32/f16/bf16, got %d", who, a->dtype);
    TVL_REQUIRE(a->batch >= 0 && a->queries >= 0 && a->keys >= 0, "%s: negative shape", who);
    TVL_REQUIRE(a->heads > 0 && a->kv_heads > 0 && a->heads % a->kv_heads == 0, "%s: heads=%lld must be a multiple of kv_heads=%lld", who, (long long)a->heads, (long long)a->kv_heads);
    TVL_REQUIRE(a->dim >= 1 && a->dim <= ATTENTION_MAX_DIM, "%s: head dim %lld outside [1, %d]", who, (long long)a->dim, ATTENTION_MAX_DIM);
    TVL_REQUIRE(a->heads <= (1 << 16) && a->batch <= (1 << 20) && a->queries <= (1 << 30) && a->keys <= (1 << 30), "%s: batch, heads or tokens too large", who);
    // every launch stays under 2^32 threads: at least 64 rows for each 256 of them, a cache's steps 16 rows for 512, the gradient kernels 128 rows for up
    // to 512, which a forward call that is asked for the log-sums is held to as well
    const int64_t most = cached || a->queries > a->keys ? a->queries : a->keys, pairs = a->batch * a->heads;
    TVL_REQUIRE(pairs * ceil_div(most, cached ? 16 : 64) < ((int64_t)1 << (cached ? 23 : 24)) && (cached || a->lse == nullptr || pairs * ceil_div(most, 128) < ((int64_t)1 << 23)),
                "%s: too many rows for one launch", who);
    TVL_REQUIRE(a->scale == a->scale && a->scale - a->scale == 0.0f, "%s: scale must be finite", who);
    TVL_REQUIRE(a->softcap >= 0.0f && a->softcap - a->softcap == 0.0f, "%s: softcap must be finite and not negative", who);
    TVL_REQUIRE(cached || a->documents == nullptr || a->queries == a->keys, "%s: documents need as many queries as keys", who);
    if (a->batch == 0) return TVL_OK;
    const size_t z = dtype_size(a->dtype);
    TVL_REQUIRE(a->queries == 0 || (a->q && a->out), "%s: NULL query or output pointer", who);
    TVL_REQUIRE(a->keys == 0 || (a->k && a->v), "%s: NULL key or value pointer", who);
    TVL_REQUIRE(aligned(a->q, z) && aligned(a->k, z) && aligned(a->v, z) && aligned(a->out, z) && aligned(a->lse, 4) && aligned(a->slopes, 4) && aligned(a->prefix, 8) &&
                    aligned(a->documents, 8) && aligned(a->cache_len, 8) && aligned(a->count, 8), "%s: misaligned pointer", who);
    TVL_REQUIRE(a->q_token >= 0 && a->k_token >= 0 && a->v_token >= 0, "%s: negative token stride", who);      // lane offsets inside a tile are unsigned
    TVL_REQUIRE(rows_apart(a->dim, a->batch, a->o_batch, a->queries, a->o_token, a->heads, a->o_head), "%s: rows of the output overlap", who);
    return TVL_OK;
}

// whether the sizes of a block make sense: a caller asks for its workspace before any entry point has checked them
static bool sized(const tvl_attention_args* a) {
    return a && a->struct_bytes == sizeof(tvl_attention_args) && a->batch > 0 && a->queries >= 0 && a->keys >= 0 && a->heads > 0 && a->kv_heads > 0 && a->heads % a->kv_heads == 0 &&
           a->dim >= 1 && a->dim <= ATTENTION_MAX_DIM;
}

// A cap so far above every score that it bends none by a bit (its share of a score below 2^87 is under 2^-26 of it) is no cap: the quotient and the product with it
// would leave float32's range.
static tvl_attention_args without_far_cap(const tvl_attention_args& a) {
    tvl_attention_args b = a;
    if (b.softcap > 0x1p100f) b.softcap = 0.0f;
    return b;
}

// parts of a workspace, each a multiple of 256 bytes
static size_t round256(size_t v) { return (v + 255) & ~size_t(255); }
static bool any_rows(const tvl_attention_args& a) { return a.queries > 0; }
static size_t span_bytes(const tvl_attention_args& a) {
    return a.documents && any_rows(a) ? round256((size_t)a.batch * (size_t)ceil_div(a.queries, SPAN) * sizeof(DocumentSpan)) : 0;
}
static size_t delta_bytes(const tvl_attention_args& a) { return any_rows(a) ? round256((size_t)a.batch * a.heads * a.queries * 4) : 0; }
static size_t slab_bytes(const tvl_attention_args& a) {
    if (!any_rows(a) || a.keys == 0) return 0;
    const int parts = attention_backward_parts(a);
    return parts > 1 ? (size_t)parts * 2 * a.batch * a.keys * a.kv_heads * a.dim * 4 : 0;
}

static int check_workspace(const char* who, size_t need, const void* workspace, size_t bytes) {
    TVL_REQUIRE(need == 0 || (workspace && bytes >= need && aligned(workspace, 256)), "%s: needs %zu bytes of 256-byte aligned workspace", who, need);
    return TVL_OK;
}

}  // namespace tvl

using namespace tvl;

extern "C" {

size_t tvl_attention_workspace_bytes(const tvl_attention_args* a) { return sized(a) ? span_bytes(*a) : 0; }

int tvl_attention(const tvl_attention_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check(a, "attention", false); rc != TVL_OK) return rc;
    if (a->batch == 0 || a->queries == 0) return TVL_OK;
    if (const int rc = check_workspace("attention", span_bytes(*a), workspace, workspace_bytes); rc != TVL_OK) return rc;
    hipStream_t st = (hipStream_t)stream;
    DocumentSpan* spans = a->documents ? static_cast<DocumentSpan*>(workspace) : nullptr;
    if (spans)
        if (const int rc = launch_document_spans(*a, spans, st); rc != TVL_OK) return rc;
    return launch_attention_forward(without_far_cap(*a), false, spans, st);
}

size_t tvl_attention_backward_workspace_bytes(const tvl_attention_args* a) {
    return sized(a) ? span_bytes(*a) + delta_bytes(*a) + slab_bytes(*a) : 0;
}

int tvl_attention_backward(const tvl_attention_args* a, const tvl_attention_grads* g, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check(a, "attention_backward", false); rc != TVL_OK) return rc;
    TVL_REQUIRE(g && g->struct_bytes == sizeof(tvl_attention_grads), "attention_backward: NULL gradient block or one of another size than %zu bytes", sizeof(tvl_attention_grads));
    if (a->batch == 0 || (a->queries == 0 && a->keys == 0)) return TVL_OK;
    const size_t z = dtype_size(a->dtype);
    TVL_REQUIRE(a->queries == 0 || (a->lse && g->grad_out), "attention_backward: NULL lse or grad_out pointer");
    TVL_REQUIRE(g->g_token >= 0, "attention_backward: negative token stride");
    TVL_REQUIRE((g->dk != nullptr) == (g->dv != nullptr), "attention_backward: dk and dv go together");
    TVL_REQUIRE(aligned(g->grad_out, z) && aligned(g->dq, z) && aligned(g->dk, z) && aligned(g->dv, z), "attention_backward: misaligned pointer");
    if (const int rc = check_workspace("attention_backward", tvl_attention_backward_workspace_bytes(a), workspace, workspace_bytes); rc != TVL_OK) return rc;
    hipStream_t st = (hipStream_t)stream;
    char* at = static_cast<char*>(workspace);
    DocumentSpan* spans = a->documents ? reinterpret_cast<DocumentSpan*>(at) : nullptr;
    float* delta = reinterpret_cast<float*>(at + span_bytes(*a));
    float* slabs = reinterpret_cast<float*>(at + span_bytes(*a) + delta_bytes(*a));
    if (spans)
        if (const int rc = launch_document_spans(*a, spans, st); rc != TVL_OK) return rc;
    return launch_attention_backward(without_far_cap(*a), *g, spans, delta, slabs, st);
}

size_t tvl_cached_attention_workspace_bytes(const tvl_attention_args* a) {
    return sized(a) && any_rows(*a) && attention_step_serves(*a) ? round256(attention_step_bytes(*a)) : 0;
}

int tvl_cached_attention(const tvl_attention_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check(a, "cached_attention", true); rc != TVL_OK) return rc;
    if (a->batch == 0 || a->queries == 0) return TVL_OK;
    if (const int rc = check_workspace("cached_attention", tvl_cached_attention_workspace_bytes(a), workspace, workspace_bytes); rc != TVL_OK) return rc;
    hipStream_t st = (hipStream_t)stream;
    const tvl_attention_args b = without_far_cap(*a);
    return attention_step_serves(b) ? launch_attention_step(b, static_cast<float*>(workspace), st) : launch_attention_forward(b, true, nullptr, st);
}

}  // extern "C"
