// Attention: argument checks of tvl_attention, tvl_attention_backward, tvl_cached_attention and their kernels.  See include/tvl.h.
#include "tvl_common.h"

namespace tvl {

constexpr int MAX_DIM = 128;

// what a query sees
struct Sight {
    int64_t place;        // of the query among the keys
    int64_t end;          // keys that exist
    int64_t prefix;
    int64_t doc;
    const int64_t* docs;
    bool causal, nan, none;
    __device__ bool sees(int64_t j) const {
        if (none || j >= end || (causal && j > place && j >= prefix)) return false;
        return docs == nullptr || (doc >= 0 && docs[j] == doc);
    }
};

template <bool CACHED>
__device__ Sight sight_of(const tvl_attention_args& a, int64_t b, int64_t i) {
    Sight s;
    s.prefix = a.prefix ? a.prefix[b] : a.prefix_value;
    s.docs = nullptr;
    s.doc = 0;
    s.nan = s.none = false;
    if (CACHED) {
        const int64_t before = a.cache_len ? a.cache_len[b * a.cache_len_stride] : a.cache_len_value;
        int64_t n = a.count ? a.count[b] : a.queries;
        n = n < 0 ? 0 : (n > a.queries ? a.queries : n);
        s.causal = true;
        s.none = i >= n;
        s.nan = !s.none && !(before >= 0 && before < a.keys - i);
        s.place = before + i;
        s.end = s.nan || s.none ? 0 : (before + n < a.keys ? before + n : a.keys);
    } else {
        s.causal = a.causal != 0;
        s.place = i + a.keys - a.queries;
        s.end = a.keys;
        if (a.documents) { s.docs = a.documents + b * a.documents_batch; s.doc = s.docs[i]; }
    }
    return s;
}

__device__ __forceinline__ float wave_max(float v) {
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// score of one key: scaled, capped, biased; `th` = tanh of the cap (0 without one)
template <typename T>
__device__ __forceinline__ float score(const tvl_attention_args& a, const float* q, const T* k, float slope, int64_t away, float& th) {
    float s = 0.0f;
    for (int e = 0; e < a.dim; ++e) s += q[e] * to_float(k[e]);
    s *= a.scale;
    th = 0.0f;
    if (a.softcap > 0.0f) { th = tanhf(s / a.softcap); s = a.softcap * th; }
    return s - slope * (float)(away < 0 ? -away : away);
}

// One wave per query: lanes take 64 keys at a time for the scores, then two elements of the head each for the sum over values.
template <typename T, bool CACHED>
__global__ void __launch_bounds__(256) attention_row_kernel(tvl_attention_args a) {
    __shared__ float rows[4][MAX_DIM];
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int64_t row = (int64_t)blockIdx.x * 4 + wave, total = a.batch * a.heads * a.queries;
    const bool live = row < total;
    const int64_t r = live ? row : 0, i = r % a.queries, h = r / a.queries % a.heads, b = r / a.queries / a.heads, hk = h / (a.heads / a.kv_heads);
    float* q = rows[wave];
    const T* qp = (const T*)a.q + b * a.q_batch + i * a.q_token + h * a.q_head;
    for (int e = lane; e < a.dim; e += 64) q[e] = to_float(qp[e]);
    __syncthreads();
    if (!live) return;
    const T* kp = (const T*)a.k + b * a.k_batch + hk * a.k_head;
    const T* vp = (const T*)a.v + b * a.v_batch + hk * a.v_head;
    const Sight sight = sight_of<CACHED>(a, b, i);
    const float slope = a.slopes ? a.slopes[h] : 0.0f;
    float m = -INFINITY, l = 0.0f, acc[2] = {0.0f, 0.0f};
    for (int64_t j0 = 0; j0 < sight.end; j0 += 64) {
        const int64_t j = j0 + lane;
        const bool sees = sight.sees(j);
        const uint64_t any = __ballot(sees);
        if (any == 0) continue;
        float th, s = -INFINITY;
        if (sees) s = score(a, q, kp + j * a.k_token, slope, sight.place - j, th);
        const float top = fmaxf(m, wave_max(s)), base = top == -INFINITY ? 0.0f : top;
        const float shrink = expf(m - base), w = sees ? expf(s - base) : 0.0f;
        m = top;
        l = l * shrink + wave_sum(w);
        acc[0] *= shrink; acc[1] *= shrink;
        for (int x = 0; x < 64; ++x) {
            if (!((any >> x) & 1)) continue;
            const float wx = __shfl(w, x);
            for (int y = 0; y < 2; ++y)
                if (lane + 64 * y < a.dim) acc[y] += wx * to_float(vp[(j0 + x) * a.v_token + lane + 64 * y]);
        }
    }
    T* op = (T*)a.out + b * a.o_batch + i * a.o_token + h * a.o_head;
    for (int y = 0; y < 2; ++y)
        if (lane + 64 * y < a.dim) op[lane + 64 * y] = from_float<T>(sight.nan ? __builtin_nanf("") : (l == 0.0f ? 0.0f : acc[y] / l));
    if (!CACHED && a.lse && lane == 0) a.lse[r] = l == 0.0f ? -INFINITY : m + logf(l);
}

// delta_i = out_i . grad_i
template <typename T>
__global__ void __launch_bounds__(256) attention_delta_kernel(tvl_attention_args a, tvl_attention_grads g, float* __restrict__ delta) {
    const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
    const int lane = threadIdx.x % 64;
    if (row >= a.batch * a.heads * a.queries) return;
    const int64_t i = row % a.queries, h = row / a.queries % a.heads, b = row / a.queries / a.heads;
    const T* op = (const T*)a.out + b * a.o_batch + i * a.o_token + h * a.o_head;
    const T* gp = (const T*)g.grad_out + b * g.g_batch + i * g.g_token + h * g.g_head;
    float s = 0.0f;
    for (int e = lane; e < a.dim; e += 64) s += to_float(op[e]) * to_float(gp[e]);
    s = wave_sum(s);
    if (lane == 0) delta[row] = s;
}

// One wave per query: dq_i = scale * sum_j p_ij (g_i . v_j - delta_i) (1 - tanh^2) k_j
template <typename T>
__global__ void __launch_bounds__(256) attention_dq_kernel(tvl_attention_args a, tvl_attention_grads g, const float* __restrict__ delta) {
    __shared__ float rows[4][2][MAX_DIM];
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int64_t row = (int64_t)blockIdx.x * 4 + wave, total = a.batch * a.heads * a.queries;
    const bool live = row < total;
    const int64_t r = live ? row : 0, i = r % a.queries, h = r / a.queries % a.heads, b = r / a.queries / a.heads, hk = h / (a.heads / a.kv_heads);
    float *q = rows[wave][0], *go = rows[wave][1];
    const T* qp = (const T*)a.q + b * a.q_batch + i * a.q_token + h * a.q_head;
    const T* gp = (const T*)g.grad_out + b * g.g_batch + i * g.g_token + h * g.g_head;
    for (int e = lane; e < a.dim; e += 64) { q[e] = to_float(qp[e]); go[e] = to_float(gp[e]); }
    __syncthreads();
    if (!live) return;
    const T* kp = (const T*)a.k + b * a.k_batch + hk * a.k_head;
    const T* vp = (const T*)a.v + b * a.v_batch + hk * a.v_head;
    const Sight sight = sight_of<false>(a, b, i);
    const float slope = a.slopes ? a.slopes[h] : 0.0f, lse = a.lse[r], dl = delta[r];
    float acc[2] = {0.0f, 0.0f};
    for (int64_t j0 = 0; j0 < sight.end; j0 += 64) {
        const int64_t j = j0 + lane;
        const bool sees = sight.sees(j);
        const uint64_t any = __ballot(sees);
        float ds = 0.0f;
        if (sees) {
            float th, dp = 0.0f;
            const float w = expf(score(a, q, kp + j * a.k_token, slope, sight.place - j, th) - lse);
            for (int e = 0; e < a.dim; ++e) dp += go[e] * to_float(vp[j * a.v_token + e]);
            ds = a.scale * w * (dp - dl) * (1.0f - th * th);
        }
        for (int x = 0; x < 64; ++x) {
            if (!((any >> x) & 1)) continue;
            const float dx = __shfl(ds, x);
            for (int y = 0; y < 2; ++y)
                if (lane + 64 * y < a.dim) acc[y] += dx * to_float(kp[(j0 + x) * a.k_token + lane + 64 * y]);
        }
    }
    T* op = (T*)g.dq + ((b * a.queries + i) * a.heads + h) * a.dim;
    for (int y = 0; y < 2; ++y)
        if (lane + 64 * y < a.dim) op[lane + 64 * y] = from_float<T>(acc[y]);
}

// One wave per key: dv_j = sum_i p_ij g_i, dk_j = scale * sum_i p_ij (g_i . v_j - delta_i) (1 - tanh^2) q_i over the queries of all heads that share it
template <typename T>
__global__ void __launch_bounds__(256) attention_dkv_kernel(tvl_attention_args a, tvl_attention_grads g, const float* __restrict__ delta) {
    __shared__ float rows[4][2][MAX_DIM];
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int64_t row = (int64_t)blockIdx.x * 4 + wave, total = a.batch * a.kv_heads * a.keys;
    const bool live = row < total;
    const int64_t r = live ? row : 0, j = r % a.keys, hk = r / a.keys % a.kv_heads, b = r / a.keys / a.kv_heads, group = a.heads / a.kv_heads;
    float *k = rows[wave][0], *v = rows[wave][1];
    const T* kp = (const T*)a.k + b * a.k_batch + j * a.k_token + hk * a.k_head;
    const T* vp = (const T*)a.v + b * a.v_batch + j * a.v_token + hk * a.v_head;
    for (int e = lane; e < a.dim; e += 64) { k[e] = to_float(kp[e]); v[e] = to_float(vp[e]); }
    __syncthreads();
    if (!live) return;
    float dk[2] = {0.0f, 0.0f}, dv[2] = {0.0f, 0.0f};
    for (int64_t h = hk * group; h < (hk + 1) * group; ++h) {
        const T* qp = (const T*)a.q + b * a.q_batch + h * a.q_head;
        const T* gp = (const T*)g.grad_out + b * g.g_batch + h * g.g_head;
        const float slope = a.slopes ? a.slopes[h] : 0.0f;
        for (int64_t i0 = 0; i0 < a.queries; i0 += 64) {
            const int64_t i = i0 + lane;
            bool sees = false;
            float w = 0.0f, ds = 0.0f;
            if (i < a.queries) {
                const Sight sight = sight_of<false>(a, b, i);
                sees = sight.sees(j);
                if (sees) {
                    const int64_t at = (b * a.heads + h) * a.queries + i;
                    float th, dp = 0.0f;
                    w = expf(score(a, k, qp + i * a.q_token, slope, sight.place - j, th) - a.lse[at]);
                    for (int e = 0; e < a.dim; ++e) dp += v[e] * to_float(gp[i * g.g_token + e]);
                    ds = a.scale * w * (dp - delta[at]) * (1.0f - th * th);
                }
            }
            const uint64_t any = __ballot(sees);
            for (int x = 0; x < 64; ++x) {
                if (!((any >> x) & 1)) continue;
                const float wx = __shfl(w, x), dx = __shfl(ds, x);
                for (int y = 0; y < 2; ++y)
                    if (lane + 64 * y < a.dim) {
                        dv[y] += wx * to_float(gp[(i0 + x) * g.g_token + lane + 64 * y]);
                        dk[y] += dx * to_float(qp[(i0 + x) * a.q_token + lane + 64 * y]);
                    }
            }
        }
    }
    const int64_t at = ((b * a.keys + j) * a.kv_heads + hk) * a.dim;
    for (int y = 0; y < 2; ++y)
        if (lane + 64 * y < a.dim) { ((T*)g.dk)[at + lane + 64 * y] = from_float<T>(dk[y]); ((T*)g.dv)[at + lane + 64 * y] = from_float<T>(dv[y]); }
}

template <typename T>
static int run_forward(const tvl_attention_args& a, bool cached, hipStream_t st) {
    const unsigned g = (unsigned)ceil_div(a.batch * a.heads * a.queries, 4);
    if (cached) hipLaunchKernelGGL((attention_row_kernel<T, true>), dim3(g), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((attention_row_kernel<T, false>), dim3(g), dim3(256), 0, st, a);
    TVL_LAUNCH_CHECK();
    return TVL_OK;
}

template <typename T>
static int run_backward(const tvl_attention_args& a, const tvl_attention_grads& g, float* delta, hipStream_t st) {
    const unsigned gq = (unsigned)ceil_div(a.batch * a.heads * a.queries, 4), gk = (unsigned)ceil_div(a.batch * a.kv_heads * a.keys, 4);
    if (gq) {
        hipLaunchKernelGGL((attention_delta_kernel<T>), dim3(gq), dim3(256), 0, st, a, g, delta);
        TVL_LAUNCH_CHECK();
        if (g.dq) hipLaunchKernelGGL((attention_dq_kernel<T>), dim3(gq), dim3(256), 0, st, a, g, delta);
        TVL_LAUNCH_CHECK();
    }
    if (gk && g.dk) {
        hipLaunchKernelGGL((attention_dkv_kernel<T>), dim3(gk), dim3(256), 0, st, a, g, delta);
        TVL_LAUNCH_CHECK();
    }
    return TVL_OK;
}

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
    TVL_REQUIRE(a->dim >= 1 && a->dim <= MAX_DIM, "%s: head dim %lld outside [1, %d]", who, (long long)a->dim, MAX_DIM);
    TVL_REQUIRE(a->heads <= (1 << 16) && a->batch <= (1 << 20) && a->queries <= (1 << 30) && a->keys <= (1 << 30), "%s: batch, heads or tokens too large", who);
    // a launch holds fewer than 2^32 threads
    TVL_REQUIRE(a->batch * a->heads * (cached || a->queries > a->keys ? a->queries : a->keys) < ((int64_t)1 << 26), "%s: too many rows for one launch", who);
    TVL_REQUIRE(a->scale == a->scale && a->scale - a->scale == 0.0f, "%s: scale must be finite", who);
    TVL_REQUIRE(a->softcap >= 0.0f && a->softcap - a->softcap == 0.0f, "%s: softcap must be finite and not negative", who);
    TVL_REQUIRE(cached || a->documents == nullptr || a->queries == a->keys, "%s: documents need as many queries as keys", who);
    if (a->batch == 0) return TVL_OK;
    const size_t z = dtype_size(a->dtype);
    TVL_REQUIRE(a->queries == 0 || (a->q && a->out), "%s: NULL query or output pointer", who);
    TVL_REQUIRE(a->keys == 0 || (a->k && a->v), "%s: NULL key or value pointer", who);
    TVL_REQUIRE(aligned(a->q, z) && aligned(a->k, z) && aligned(a->v, z) && aligned(a->out, z) && aligned(a->lse, 4) && aligned(a->slopes, 4) && aligned(a->prefix, 8) &&
                    aligned(a->documents, 8) && aligned(a->cache_len, 8) && aligned(a->count, 8), "%s: misaligned pointer", who);
    TVL_REQUIRE(rows_apart(a->dim, a->batch, a->o_batch, a->queries, a->o_token, a->heads, a->o_head), "%s: rows of the output overlap", who);
    return TVL_OK;
}

}  // namespace tvl

using namespace tvl;

extern "C" {

size_t tvl_attention_workspace_bytes(const tvl_attention_args* a) { (void)a; return 0; }

int tvl_attention(const tvl_attention_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check(a, "attention", false); rc != TVL_OK) return rc;
    if (a->batch == 0 || a->queries == 0) return TVL_OK;
    (void)workspace; (void)workspace_bytes;
    hipStream_t st = (hipStream_t)stream;
    if (a->dtype == TVL_F32) return run_forward<float>(*a, false, st);
    if (a->dtype == TVL_F16) return run_forward<f16>(*a, false, st);
    return run_forward<bf16_t>(*a, false, st);
}

size_t tvl_attention_backward_workspace_bytes(const tvl_attention_args* a) {
    return a && a->batch > 0 && a->heads > 0 && a->queries > 0 ? (size_t)(a->batch * a->heads * a->queries) * 4 : 0;
}

int tvl_attention_backward(const tvl_attention_args* a, const tvl_attention_grads* g, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check(a, "attention_backward", false); rc != TVL_OK) return rc;
    TVL_REQUIRE(g && g->struct_bytes == sizeof(tvl_attention_grads), "attention_backward: NULL gradient block or one of another size than %zu bytes", sizeof(tvl_attention_grads));
    if (a->batch == 0 || (a->queries == 0 && a->keys == 0)) return TVL_OK;
    const size_t z = dtype_size(a->dtype), need = tvl_attention_backward_workspace_bytes(a);
    TVL_REQUIRE(a->queries == 0 || (a->lse && g->grad_out), "attention_backward: NULL lse or grad_out pointer");
    TVL_REQUIRE((g->dk != nullptr) == (g->dv != nullptr), "attention_backward: dk and dv go together");
    TVL_REQUIRE(aligned(g->grad_out, z) && aligned(g->dq, z) && aligned(g->dk, z) && aligned(g->dv, z), "attention_backward: misaligned pointer");
    TVL_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 256)), "attention_backward: needs %zu bytes of 256-byte aligned workspace", need);
    hipStream_t st = (hipStream_t)stream;
    if (a->dtype == TVL_F32) return run_backward<float>(*a, *g, (float*)workspace, st);
    if (a->dtype == TVL_F16) return run_backward<f16>(*a, *g, (float*)workspace, st);
    return run_backward<bf16_t>(*a, *g, (float*)workspace, st);
}

size_t tvl_cached_attention_workspace_bytes(const tvl_attention_args* a) { (void)a; return 0; }

int tvl_cached_attention(const tvl_attention_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check(a, "cached_attention", true); rc != TVL_OK) return rc;
    if (a->batch == 0 || a->queries == 0) return TVL_OK;
    (void)workspace; (void)workspace_bytes;
    hipStream_t st = (hipStream_t)stream;
    if (a->dtype == TVL_F32) return run_forward<float>(*a, true, st);
    if (a->dtype == TVL_F16) return run_forward<f16>(*a, true, st);
    return run_forward<bf16_t>(*a, true, st);
}

}  // extern "C"
