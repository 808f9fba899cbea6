// Rotary positions: tvl_rotary (any tensor of heads, forward and transposed) and tvl_rotary_cache (the joint projection's
// output straight into a key / value cache).  See include/tvl.h for the map.
#include "tvl_common.h"

namespace tvl {

// where a head's row goes and how much of it is turned
struct RotaryParams {
    const void* x;
    int64_t x_batch, x_token, x_head;
    void* y;                                 // turned heads [0, heads)
    int64_t y_batch, y_token, y_head;
    void* kc;                                // cache form: heads [heads, heads + kv_heads) turned, the next kv_heads copied
    void* vc;
    int64_t k_batch, k_head, k_slot, v_batch, v_head, v_slot;
    const float* table;
    int64_t ld_table, table_rows;
    const int64_t* positions;                // plain form
    int64_t pos_batch, pos_token;
    const int64_t* cache_len;                // cache form
    const int64_t* count;
    int64_t cache_len_stride, cache_len_value, slots;
    int64_t rows;                            // batch * tokens
    int tokens, heads, kv_heads, dim, rd;
    float sign;                              // +1, or -1 for the transposed map
};

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack { T e[VEC]; };

// One thread moves 2 * VEC elements of one head: VEC pairs (both halves, or 2 * VEC neighbours), or 2 * VEC elements behind the
// rotated part.  Each element is read and written once and each angle row once per head out of the cache, so the pass is bound
// by HBM; VEC is 16 bytes where strides, pointers and the rotated part allow it.
// 4 x 2048 tokens, 64 heads of 64, half turned, bf16: 36.7 us, 3.65 TB/s (a large copy reaches 4.9); the cache write of 8 prompts of up to 745 tokens, 96 heads of
// 64, f16: 31.5 us; one token: 3.2 us, the launch.  What is likely between this and a copy: places by 64-bit division, angles
// by 4-byte loads.
template <typename T, int VEC, bool CACHE, bool NEIGHBOURS>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryParams p) {
    using V = Pack<T, VEC>;
    const int half = p.rd / 2, turn_units = half / VEC, copy_units = (p.dim - p.rd + 2 * VEC - 1) / (2 * VEC), units = turn_units + copy_units;
    const int all_heads = CACHE ? p.heads + 2 * p.kv_heads : p.heads;
    const uint32_t per_row = (uint32_t)(units * all_heads);
    const int64_t total = p.rows * per_row;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < total; at += (int64_t)gridDim.x * 256) {
        const int64_t row = at / per_row;
        const uint32_t rest = (uint32_t)(at - row * per_row);
        const int head = rest / units, unit = rest - head * units;
        const int64_t b = row / p.tokens;
        const int t = (int)(row - b * p.tokens);
        int64_t pos;
        bool pad = false, inside;
        if constexpr (CACHE) {
            const int64_t before = p.cache_len ? p.cache_len[b * p.cache_len_stride] : p.cache_len_value;
            pad = p.count && t >= p.count[b];
            inside = before >= 0 && before < p.slots - t && before < p.table_rows - t;
            pos = before + t;
        } else {
            pos = p.positions[b * p.pos_batch + t * p.pos_token];
            inside = pos >= 0 && pos < p.table_rows;
        }
        T* dst;
        bool turned = true;
        if (head < p.heads) {
            dst = (T*)p.y + b * p.y_batch + t * p.y_token + head * p.y_head;
        } else {
            if (pad || !inside) continue;    // the caches keep what they hold
            turned = head < p.heads + p.kv_heads;
            dst = turned ? (T*)p.kc + b * p.k_batch + (head - p.heads) * p.k_head + pos * p.k_slot
                         : (T*)p.vc + b * p.v_batch + (head - p.heads - p.kv_heads) * p.v_head + pos * p.v_slot;
        }
        const T* src = (const T*)p.x + b * p.x_batch + t * p.x_token + head * p.x_head;
        const bool fill = pad || !inside;
        const T value = from_float<T>(pad ? 0.0f : __builtin_nanf(""));
        if (unit < turn_units) {
            const int i = unit * VEC;        // first pair of this thread
            const int lo = NEIGHBOURS ? 2 * i : i, hi = NEIGHBOURS ? 2 * i + VEC : half + i;
            V a, c;
            if (fill) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) a.e[e] = c.e[e] = value;
            } else {
                a = *reinterpret_cast<const V*>(src + lo);
                c = *reinterpret_cast<const V*>(src + hi);
                if (turned) {
                    const float* angle = p.table + pos * p.ld_table + i;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float cs = angle[e], sn = p.sign * angle[half + e];
                        // pair e: (a[e], c[e]), or elements 2e and 2e + 1 of the 2 * VEC neighbours
                        T& first = NEIGHBOURS ? (2 * e < VEC ? a.e[2 * e % VEC] : c.e[2 * e % VEC]) : a.e[e];
                        T& second = NEIGHBOURS ? (2 * e + 1 < VEC ? a.e[(2 * e + 1) % VEC] : c.e[(2 * e + 1) % VEC]) : c.e[e];
                        const float u = to_float(first), w = to_float(second);
                        // one rounded product, one fused multiply-add: the same bits on every path
                        first = from_float<T>(__builtin_fmaf(u, cs, -(w * sn)));
                        second = from_float<T>(__builtin_fmaf(w, cs, u * sn));
                    }
                }
            }
            *reinterpret_cast<V*>(dst + lo) = a;
            *reinterpret_cast<V*>(dst + hi) = c;
        } else {
            const int lo = p.rd + (unit - turn_units) * 2 * VEC;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int c0 = lo + h * VEC;
                if (c0 < p.dim) {
                    V a;
                    if (fill) {
#pragma unroll
                        for (int e = 0; e < VEC; ++e) a.e[e] = value;
                    } else {
                        a = *reinterpret_cast<const V*>(src + c0);
                    }
                    *reinterpret_cast<V*>(dst + c0) = a;
                }
            }
        }
    }
}

template <typename T, int VEC, bool CACHE>
static int launch_rotary_v(const RotaryParams& p, bool neighbours, hipStream_t st) {
    const int64_t units = p.rd / 2 / VEC + ceil_div(p.dim - p.rd, 2 * VEC);
    const int64_t total = p.rows * units * (CACHE ? p.heads + 2 * p.kv_heads : p.heads);
    const int64_t blocks = ceil_div(total, 256);
    const unsigned g = (unsigned)(blocks < 65536 ? blocks : 65536);
    if (neighbours) hipLaunchKernelGGL((rotary_kernel<T, VEC, CACHE, true>), dim3(g), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((rotary_kernel<T, VEC, CACHE, false>), dim3(g), dim3(256), 0, st, p);
    TVL_LAUNCH_CHECK();
    return TVL_OK;
}

template <typename T, bool CACHE>
static int launch_rotary_t(const RotaryParams& p, bool neighbours, hipStream_t st) {
    constexpr int VEC = 16 / sizeof(T);
    auto fits = [&](const void* ptr, int64_t a, int64_t b, int64_t c) { return ptr == nullptr || (aligned(ptr, 16) && a % VEC == 0 && b % VEC == 0 && c % VEC == 0); };
    const bool wide = (p.rd / 2) % VEC == 0 && p.dim % VEC == 0 && fits(p.x, p.x_batch, p.x_token, p.x_head) && fits(p.y, p.y_batch, p.y_token, p.y_head) &&
                      fits(p.kc, p.k_batch, p.k_head, p.k_slot) && fits(p.vc, p.v_batch, p.v_head, p.v_slot);
    return wide ? launch_rotary_v<T, VEC, CACHE>(p, neighbours, st) : launch_rotary_v<T, 1, CACHE>(p, neighbours, st);
}

template <bool CACHE>
static int launch_rotary(const RotaryParams& p, int dtype, bool neighbours, hipStream_t st) {
    if (dtype == TVL_F32) return launch_rotary_t<float, CACHE>(p, neighbours, st);
    if (dtype == TVL_F16) return launch_rotary_t<f16, CACHE>(p, neighbours, st);
    return launch_rotary_t<bf16_t, CACHE>(p, neighbours, st);
}

}  // namespace tvl

using namespace tvl;

extern "C" {

int tvl_rotary(const tvl_rotary_args* a, void* stream) {
    TVL_REQUIRE(a && a->struct_bytes == sizeof(tvl_rotary_args), "rotary: NULL argument block or one of another size than %zu bytes", sizeof(tvl_rotary_args));
    TVL_REQUIRE(a->dtype == TVL_F32 || a->dtype == TVL_F16 || a->dtype == TVL_BF16, "rotary: dtype must be f32/f16/bf16, got %d", a->dtype);
    TVL_REQUIRE(a->batch >= 0 && a->tokens >= 0 && a->heads >= 0 && a->dim >= 0 && a->table_rows >= 0, "rotary: negative shape");
    TVL_REQUIRE(a->tokens <= (1 << 30) && a->heads <= (1 << 16) && a->dim <= (1 << 12), "rotary: tokens, heads or dim too large");
    TVL_REQUIRE(a->rotary_dim >= 0 && a->rotary_dim % 2 == 0 && a->rotary_dim <= a->dim, "rotary: rotary_dim=%lld must be even and at most dim=%lld",
                (long long)a->rotary_dim, (long long)a->dim);
    TVL_REQUIRE(a->ld_table >= a->rotary_dim, "rotary: table rows hold %lld values, rotary_dim=%lld", (long long)a->ld_table, (long long)a->rotary_dim);
    if (a->batch == 0 || a->tokens == 0 || a->heads == 0 || a->dim == 0) return TVL_OK;
    TVL_REQUIRE(a->batch <= (1 << 30), "rotary: batch too large");
    TVL_REQUIRE(a->x && a->y && a->positions && (a->table || a->table_rows == 0 || a->rotary_dim == 0), "rotary: NULL pointer");
    TVL_REQUIRE(aligned(a->x, dtype_size(a->dtype)) && aligned(a->y, dtype_size(a->dtype)) && aligned(a->positions, 8) && aligned(a->table, 4), "rotary: misaligned pointer");
    RotaryParams p{};
    p.x = a->x; p.x_batch = a->x_batch; p.x_token = a->x_token; p.x_head = a->x_head;
    p.y = a->y; p.y_batch = a->y_batch; p.y_token = a->y_token; p.y_head = a->y_head;
    p.table = a->table; p.ld_table = a->ld_table; p.table_rows = a->table_rows;
    p.positions = a->positions; p.pos_batch = a->pos_batch; p.pos_token = a->pos_token;
    p.rows = a->batch * a->tokens;
    p.tokens = (int)a->tokens; p.heads = (int)a->heads; p.dim = (int)a->dim; p.rd = (int)a->rotary_dim;
    p.sign = a->inverse ? -1.0f : 1.0f;
    return launch_rotary<false>(p, a->dtype, a->interleaved != 0, (hipStream_t)stream);
}

int tvl_rotary_cache(const tvl_rotary_cache_args* a, void* stream) {
    TVL_REQUIRE(a && a->struct_bytes == sizeof(tvl_rotary_cache_args), "rotary_cache: NULL argument block or one of another size than %zu bytes",
                sizeof(tvl_rotary_cache_args));
    TVL_REQUIRE(a->dtype == TVL_F32 || a->dtype == TVL_F16 || a->dtype == TVL_BF16, "rotary_cache: dtype must be f32/f16/bf16, got %d", a->dtype);
    TVL_REQUIRE(a->batch >= 0 && a->tokens >= 0 && a->heads >= 0 && a->kv_heads >= 0 && a->dim >= 0 && a->slots >= 0 && a->table_rows >= 0, "rotary_cache: negative shape");
    TVL_REQUIRE(a->tokens <= (1 << 30) && a->heads <= (1 << 16) && a->kv_heads <= (1 << 16) && a->dim <= (1 << 12), "rotary_cache: tokens, heads or dim too large");
    TVL_REQUIRE(a->rotary_dim >= 0 && a->rotary_dim % 2 == 0 && a->rotary_dim <= a->dim, "rotary_cache: rotary_dim=%lld must be even and at most dim=%lld",
                (long long)a->rotary_dim, (long long)a->dim);
    TVL_REQUIRE(a->ld_table >= a->rotary_dim, "rotary_cache: table rows hold %lld values, rotary_dim=%lld", (long long)a->ld_table, (long long)a->rotary_dim);
    if (a->batch == 0 || a->tokens == 0 || a->heads + a->kv_heads == 0 || a->dim == 0) return TVL_OK;
    TVL_REQUIRE(a->batch <= (1 << 30), "rotary_cache: batch too large");
    TVL_REQUIRE(a->qkv && (a->q || a->heads == 0) && (a->table || a->table_rows == 0 || a->rotary_dim == 0) && ((a->k_cache && a->v_cache) || a->slots == 0 || a->kv_heads == 0), "rotary_cache: NULL pointer");
    const size_t z = dtype_size(a->dtype);
    TVL_REQUIRE(aligned(a->qkv, z) && aligned(a->q, z) && aligned(a->k_cache, z) && aligned(a->v_cache, z) && aligned(a->table, 4) && aligned(a->cache_len, 8) &&
                    aligned(a->count, 8), "rotary_cache: misaligned pointer");
    RotaryParams p{};
    p.x = a->qkv; p.x_batch = a->x_batch; p.x_token = a->x_token; p.x_head = a->dim;
    p.y = a->q; p.y_head = a->dim; p.y_token = a->heads * a->dim; p.y_batch = a->tokens * p.y_token;
    p.kc = a->k_cache; p.vc = a->v_cache;
    p.k_batch = a->k_batch; p.k_head = a->k_head; p.k_slot = a->k_slot;
    p.v_batch = a->v_batch; p.v_head = a->v_head; p.v_slot = a->v_slot;
    p.table = a->table; p.ld_table = a->ld_table; p.table_rows = a->table_rows;
    p.cache_len = a->cache_len; p.count = a->count; p.cache_len_stride = a->cache_len_stride; p.cache_len_value = a->cache_len_value; p.slots = a->slots;
    p.rows = a->batch * a->tokens;
    p.tokens = (int)a->tokens; p.heads = (int)a->heads; p.kv_heads = (int)a->kv_heads; p.dim = (int)a->dim; p.rd = (int)a->rotary_dim;
    p.sign = 1.0f;
    return launch_rotary<true>(p, a->dtype, a->interleaved != 0, (hipStream_t)stream);
}

}  // extern "C"
