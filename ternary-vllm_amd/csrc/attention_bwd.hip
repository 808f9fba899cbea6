// Backward attention: delta = rowsum(out * grad_out), then dq per query tile and dk, dv per key tile.  The scores are formed again from
// q, k and the saved log-sum, twice (14 instead of 10 operations per pair, head and element, 16 for 16-bit operands): every gradient is then summed in
// the registers of one workgroup, in a fixed order, without atomics.
// GPU times below: A = 4 x 2048 causal tokens, 32 heads of 64, bf16; B = 8191 tokens in 7 documents, 16 / 4 heads of 128, capped, bf16; C = 128 x 197 tokens,
// 12 heads of 64, f16.
#include "attention_tiles.h"

namespace tvl {

constexpr int GT = 64;    // rows of a staged tile
constexpr int PIECE = 32; // of them at a time
// N values of a piece that a lane holds: row of value x (of lane group 0)
template <int R> constexpr int VALUES = PIECE * R / 64;
template <int R> __device__ __forceinline__ constexpr int piece_row(int x) { return x / REGS<R> * R + result_row<R>(x % REGS<R>, 0); }

// Shape of a gradient kernel: W waves of R queries or keys each, 128 in all, its registers limited to OCCUPANCY waves per SIMD.  16-bit heads of 64
// fit two waves per SIMD at R = 32, whose products read LDS half as often: the pass over 4 x 2048 causal tokens, 32 heads, bf16, takes 530 us, at R = 16
// 730.  Longer rows and float32 fit them at R = 16 only (16-bit rows of 128 but for 1 to 3 registers of dk / dv, float32 ones but for 6 to 69): 8192 tokens, 16 heads of 128, f16
// 2500 us, at R = 32 with one wave 3655 (bf16 2510 and 2690); float32 (4 x 2048 causal, 16 heads) of 64 1520 against 1556, of 128 2850 against 3014.
template <typename T, int DP> struct Shape {
    static constexpr int R = DP == 64 && sizeof(T) == 2 ? 32 : 16, W = 128 / R, OCCUPANCY = 2;
};

// float16 score gradients (2^BACKWARD_LIFT times as large, as their weights are) are rounded in a range of their own for every column, a query of dq or a
// key of dk, that follows the largest one of the column so far.  They stay as they are while that one lies in [1, 2^15]; else a power of two `fit` brings
// it to [2^7, 2^8), and the column's sum is rescaled when that moves, as a softmax's maximum is.  Nothing overflows however large values and output
// gradients are, a small one is off by at most 2^-25 of its column's largest, and no column depends on what another one holds.  (A power of two for
// a whole sequence, from its largest output gradient, made infinities of large values and zeros of the gradients of small documents beside large ones.)
// What is not finite spoils its own column.
struct Range {
    float fit = 1.0f, most = 0.0f;      // most: the largest one that fits
    bool scaled = false;                // whether any lane's fit is not 1
    template <int R, int N, int D> __device__ __forceinline__ void follow(const float (&ds)[N], Acc<R> (&acc)[D]) {
        float top = 0.0f;
#pragma unroll
        for (int x = 0; x < N; ++x) top = fmaxf(top, fabsf(ds[x]));
        if (__any(top > most)) {
            top = column_max<R>(top);
            float now = fit;
            if (top > most) {
                const int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127 - 7;      // fit 2^-e, from 2^-100 to 2^100
                now = top >= 1.0f && top <= 32768.0f ? 1.0f : __builtin_bit_cast(float, (uint32_t)(127 - (e < -100 ? -100 : (e > 100 ? 100 : e))) << 23);
                most = __builtin_bit_cast(float, (269u << 23) - __builtin_bit_cast(uint32_t, now));      // 2^15 / fit
            }
            const float shrink = now * __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, fit));
            fit = now;
            scaled = __any(fit != 1.0f);
#pragma unroll
            for (int d = 0; d < D; ++d) acc[d] *= shrink;
        }
    }
};

// delta[row] = sum over the head of out * grad_out, with the rounded output: one pass over two tensors in place of one over keys and values.  16 lanes per row, 16 bytes each: one read of both tensors, bound by HBM (A: 12.4 us, 5.4 TB/s; B: 12.3; C: 15.8).
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256) attention_delta_kernel(tvl_attention_args a, tvl_attention_grads gr, float* __restrict__ delta, int blocks) {
    constexpr int PER = 16 / (int)sizeof(T);
    const int bh = blockIdx.x / blocks, n = blockIdx.x % blocks, h = bh % (int)a.heads, b = bh / (int)a.heads;
    const int lane = threadIdx.x % 16, row = threadIdx.x / 16, dim = (int)a.dim, queries = (int)a.queries;
#pragma unroll
    for (int p = 0; p < GT / 16; ++p) {
        const int i = n * GT + p * 16 + row;
        float sum = 0.0f;
        if (i < queries) {
            const T* op = (const T*)a.out + b * a.o_batch + (int64_t)i * a.o_token + h * a.o_head;
            const T* gp = (const T*)gr.grad_out + b * gr.g_batch + (int64_t)i * gr.g_token + h * gr.g_head;
            for (int u = lane; u * PER < dim; u += 16) {
                const u32x4 x = load_unit<T, WIDE>(op, u, dim), y = load_unit<T, WIDE>(gp, u, dim);
                const T *xe = reinterpret_cast<const T*>(&x), *ye = reinterpret_cast<const T*>(&y);
#pragma unroll
                for (int e = 0; e < PER; ++e) sum += to_float(xe[e]) * to_float(ye[e]);
            }
        }
        for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        if (i < queries && lane == 0) delta[(int64_t)bh * queries + i] = sum;
    }
}

// dq.  W waves x R queries; per 32 keys: S^T = K Q^T, dP^T = V dO^T, dS^T = P (dP - delta) bend (a lane holds one query), dQ^T += K^T dS^T.  Six operations per
// pair and element, eight for 16-bit operands (`mean` below).  A: 222 us (620 TFLOP/s), B: 383, C: 118.  The matrix cores are busy 41 % of the time at heads of 64 and 43 %
// at 128: exponentials and conversions on the vector ALU and the operands' way out of LDS (no bank conflicts) wait for each other with two waves per SIMD.
// float16's range costs a maximum per score and a branch in front of the last product: 4 x 2048 causal, 32 heads of 64 257 us.
//
// delta' of the rounded output is off by its two roundings (weights, result), for rows whose weight lies on few keys as far as a score gradient's own rounding,
// and all in one direction.  For 16-bit operands the sum of P (dP - delta') over a row, zero but for that error, is formed beside (`rest`, float32), and
// sum of P bend K with it (`mean`, a product more out of the same operands): dq = scale (sum of dS K - rest mean), and delta = delta' + rest goes to the
// pass over keys.
// BARE: delta alone, for calls that want dk and dv only, so that they get the same bits.
template <typename T, int DP, Form FORM, bool BARE>
__global__ void __launch_bounds__((64 * Shape<T, DP>::W), (Shape<T, DP>::OCCUPANCY)) attention_dq_kernel(tvl_attention_args a, tvl_attention_grads gr, const DocumentSpan* __restrict__ spans, float* __restrict__ delta,
                                                           int tiles) {
    constexpr bool WIDE = FORM != ODD, MEND = sizeof(T) == 2;
    constexpr int R = Shape<T, DP>::R, THREADS = 64 * Shape<T, DP>::W, QB = 128, CK = CHUNK<R>, N = VALUES<R>;
    typedef Tile<T, DP> L;
    typedef typename Operand<T>::elem E;
    extern __shared__ __align__(16) char lds[];
    constexpr int TILE = GT * L::ROW, BUFFER = 2 * TILE + (FORM == PLAIN ? 0 : GT * 8);     // keys, values, documents

    const int group = (int)(a.heads / a.kv_heads), pairs = (int)(a.batch * a.kv_heads);
    const Place at = place_of(blockIdx.x, pairs, group, tiles);
    const int b = at.pair / (int)a.kv_heads, hk = at.pair % (int)a.kv_heads, h = hk * group + at.head;
    const int wave = wave_number(), lane = threadIdx.x % 64, r = lane % R, g = lane / R;
    const int q0 = at.tile * QB, qw = q0 + wave * R, i = qw + r;
    const int dim = (int)a.dim, queries = (int)a.queries;
    bool lost;
    const Sequence seq = sequence_of<false>(a, b, lost);
    const int last = q0 + QB < queries ? q0 + QB : queries, reach = seq.limit(last - 1);
    const int all = seq.limit(q0);      // keys every query of the block sees
    const int wlast = qw + R < queries ? qw + R : queries;
    const int wreach = wlast > qw ? seq.limit(wlast - 1) : 0, wall = wlast > qw ? seq.limit(qw) : 0;
    const int mine = i < queries ? seq.limit(i) : 0;
    const T* kp = (const T*)a.k + b * a.k_batch + hk * a.k_head;
    const T* vp = (const T*)a.v + b * a.v_batch + hk * a.v_head;
    const int64_t* docs = FORM == PLAIN ? nullptr : a.documents;
    int64_t doc = -1;
    DocumentWindow docw;
    if (docs) {
        docs += b * a.documents_batch;
        if (i < queries) doc = docs[i];
        docw.start(spans + (int64_t)b * ((queries + SPAN - 1) / SPAN), queries, q0, QB);
    }
    Frag<T> qf[DP / CK], gf[DP / CK];
    constexpr float UP = BACKWARD_LIFT<T>, DOWN = 1.0f / (float)(1 << (int)UP);      // weights and score gradients are formed 2^UP times as large
    float lse = 0.0f, dl = 0.0f;
#pragma unroll
    for (int c = 0; c < DP / CK; ++c) {
        qf[c] = gf[c] = Frag<T>{};
        if (i < queries) {
            qf[c] = load_frag<T, WIDE>((const T*)a.q + b * a.q_batch + (int64_t)i * a.q_token + h * a.q_head, g + (64 / R) * c, dim);
            gf[c] = load_frag<T, WIDE>((const T*)gr.grad_out + b * gr.g_batch + (int64_t)i * gr.g_token + h * gr.g_head, g + (64 / R) * c, dim);
        }
    }
    if (i < queries) {
        const int64_t row = ((int64_t)b * a.heads + h) * queries + i;
        lse = a.lse[row] * LOG2E - UP;
        dl = delta[row];
    }
    Range range;
    const float slope = a.slopes ? a.slopes[h] * LOG2E : 0.0f;
    const bool capped = FORM != PLAIN && a.softcap > 0.0f, biased = FORM != PLAIN && a.slopes != nullptr;
    const float to_log2 = a.scale * LOG2E, to_cap = capped ? a.scale / a.softcap : 0.0f, from_cap = a.softcap * LOG2E;
    const float pre = capped ? 1.0f : to_log2, unit = capped || biased ? 1.0f : to_log2;
    Acc<R> acc[DP / R] = {}, mean[MEND && !BARE ? DP / R : 1] = {};
    float rest = 0.0f;

    auto next = [&](int j) { return docs && j < reach ? docw.next(j / SPAN, (reach + SPAN - 1) / SPAN, lane) * SPAN : j; };
    const int lane_row = L::template lane_row<R>(lane), lane_col = L::template lane_column<R>(lane);
    // one set of staging registers: the next keys are on their way during the first half of a tile, the next values during the second
    Stage<T, DP, GT, THREADS, WIDE> stage;
    int64_t side = -1;
    auto fetch_keys = [&](int j) {
        stage.load(kp, a.k_token, j, seq.end, dim);
        if (docs && threadIdx.x < GT) side = j + (int)threadIdx.x < seq.end ? docs[j + threadIdx.x] : -1;
    };
    auto put_keys = [&](char* to) {
        stage.store(to);
        if (docs && threadIdx.x < GT) reinterpret_cast<int64_t*>(to + 2 * TILE)[threadIdx.x] = side;
    };
    int j0 = next(0), buf = 0;
    if (j0 < reach) {
        fetch_keys(j0);
        put_keys(lds);
        stage.load(vp, a.v_token, j0, seq.end, dim);
        stage.store(lds + TILE);
    }
    __syncthreads();
    // MASKED: some query of the block does not see some key of the tile
    auto step = [&](auto masked) __attribute__((always_inline)) {
        constexpr bool MASKED = decltype(masked)::value;
        const int j1 = next(j0 + GT);
        char* ahead = lds + (buf ^ 1) * BUFFER;
        if (j1 < reach) fetch_keys(j1);
        const char *kt = lds + buf * BUFFER, *vt = kt + TILE;
        const int64_t* kdocs = reinterpret_cast<const int64_t*>(kt + 2 * TILE);
        const bool one_document = !MASKED || !docs || docw.one(j0 / SPAN, lane);
        auto piece = [&](int t) __attribute__((always_inline)) {
            const int jt = j0 + t;
            if (MASKED && jt >= wreach) return;
            float s[N], dp[N], bend[FORM == PLAIN ? 1 : N];
#pragma unroll
            for (int n = 0; n < PIECE / R; ++n) {
                Acc<R> u = {}, w = {};
#pragma unroll
                for (int c = 0; c < DP / CK; ++c) {
                    u = mma(L::template read<R>(kt + t * L::ROW, lane_row, n * R, c), qf[c], u);
                    w = mma(L::template read<R>(vt + t * L::ROW, lane_row, n * R, c), gf[c], w);
                }
#pragma unroll
                for (int x = 0; x < REGS<R>; ++x) { s[n * REGS<R> + x] = u[x]; dp[n * REGS<R> + x] = w[x]; }
            }
            [[maybe_unused]] Frag<T> df[PIECE / CK], pf[PIECE / CK];
            if (capped) {
#pragma unroll
                for (int x = 0; x < N; ++x) s[x] *= to_cap;
                cap_tanh<T, FORM, N>(s, a.softcap);
#pragma unroll
                for (int x = 0; x < N; ++x) {
                    bend[x] = __builtin_fmaf(-s[x], s[x], 1.0f);
                    dp[x] -= dl;
                    if constexpr (!MEND) dp[x] = product(dp[x], bend[x]);
                    s[x] *= from_cap;
                }
            } else {
#pragma unroll
                for (int x = 0; x < N; ++x) dp[x] -= dl;
            }
            if (biased) {
                const int here = i + seq.shift - jt - 4 * g;
#pragma unroll
                for (int x = 0; x < N; ++x) s[x] = __builtin_fmaf(-slope, fabsf((float)(here - piece_row<R>(x))), s[x] * pre);
            }
#pragma unroll
            for (int x = 0; x < N; ++x) {
                s[x] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x], unit, -lse));
                dp[x] = product(dp[x], s[x]);
            }
            if (MASKED && (jt + PIECE > wall || !one_document)) {
                auto hide = [&](int x) __attribute__((always_inline)) {
                    dp[x] = 0.0f;
                    if constexpr (MEND && !BARE) s[x] = 0.0f;
                    if constexpr (MEND && !BARE && FORM != PLAIN) bend[x] = 0.0f;
                };
                const int left = mine - jt - 4 * g;
#pragma unroll
                for (int x = 0; x < N; ++x)
                    if (piece_row<R>(x) >= left) hide(x);
                if (!one_document) {
#pragma unroll
                    for (int x = 0; x < N; ++x)
                        if (!same_document(kdocs + t + 4 * g + piece_row<R>(x), doc)) hide(x);
                }
            }
            if constexpr (MEND) {
#pragma unroll
                for (int x = 0; x < N; ++x) rest += dp[x];
                if constexpr (BARE) return;
                if constexpr (FORM != PLAIN) {
                    if (capped) {
#pragma unroll
                        for (int x = 0; x < N; ++x) {
                            dp[x] = product(dp[x], bend[x]);
                            s[x] = product(s[x], bend[x]);
                        }
                    }
                }
            }
            // keys across, for both products; what is not finite in them must not reach queries that do not see it
            const bool spoilt = MASKED && (!one_document || (jt + PIECE > wall && wall < seq.end)) && holds_not_finite<T, DP, PIECE>(kt + t * L::ROW, lane);
            Frag<T> across[PIECE / CK][DP / R];
#pragma unroll
            for (int c = 0; c < PIECE / CK; ++c)
#pragma unroll
                for (int d = 0; d < DP / R; ++d) across[c][d] = L::template read_across<R>(kt + t * L::ROW, lane_col, c * CK, d);
            if (MASKED && spoilt) {
#pragma unroll
                for (int c = 0; c < PIECE / CK; ++c)
#pragma unroll
                    for (int d = 0; d < DP / R; ++d) across[c][d] = finite_part<T>(across[c][d]);
            }
            // weights and score gradients are rounded to the operands' type for the last products; their sums are float32
            if constexpr (MEND) {
#pragma unroll
                for (int x = 0; x < N; ++x) pf[x / 8][x % 8] = (E)s[x];
#pragma unroll
                for (int c = 0; c < PIECE / CK; ++c)
#pragma unroll
                    for (int d = 0; d < DP / R; ++d) mean[d] = mma(across[c][d], pf[c], mean[d]);
            }
            if constexpr (__is_same(T, f16)) {
                range.follow<R>(dp, acc);
                if (range.scaled) {
#pragma unroll
                    for (int x = 0; x < N; ++x) dp[x] = product(dp[x], range.fit);
                }
            }
#pragma unroll
            for (int x = 0; x < N; ++x) df[x / 8][x % 8] = (E)dp[x];
#pragma unroll
            for (int c = 0; c < PIECE / CK; ++c)
#pragma unroll
                for (int d = 0; d < DP / R; ++d) acc[d] = mma(across[c][d], df[c], acc[d]);
            if (MASKED && spoilt) {
#pragma unroll 1
                for (int row = 0; row < PIECE && jt + row < reach; ++row)
                    add_not_finite<T, DP, R>(kt, t + row, jt + row < mine && (one_document || (doc >= 0 && kdocs[t + row] == doc)), true, g, acc);
            }
        };
        piece(0);
        if (j1 < reach) {
            put_keys(ahead);
            stage.load(vp, a.v_token, j1, seq.end, dim);
        }
        piece(PIECE);
        if (j1 < reach) stage.store(ahead + TILE);
        __syncthreads();
        buf ^= 1;
        j0 = j1;
    };
    auto clean = [&](int j) { return j + GT <= all && (!docs || docw.one(j / SPAN, lane)); };
    while (j0 < reach) {
        while (j0 < reach && clean(j0)) step(std::false_type{});
        while (j0 < reach && !clean(j0)) step(std::true_type{});
    }
    if constexpr (MEND) {
        rest = column_sum<R>(rest) * DOWN;
        if (i < queries && g == 0) delta[((int64_t)b * a.heads + h) * queries + i] = dl + rest;
    }
    if (BARE || i >= queries) return;
    const float back = a.scale / range.fit * DOWN, off = -rest * a.scale * DOWN;
    T* op = (T*)gr.dq + (((int64_t)b * queries + i) * a.heads + h) * dim;
#pragma unroll
    for (int d = 0; d < DP / R; ++d)
#pragma unroll
        for (int x = 0; x < REGS<R>; ++x) {
            const int col = d * R + result_row<R>(x, g);
            float v = product(acc[d][x], back);
            if constexpr (MEND && !BARE) v = __builtin_fmaf(off, mean[d][x], v);
            if (mine <= 1) v = 0.0f;      // a softmax over one key has no slope
            if (col < dim) op[col] = from_float<T>(v);
        }
}

// dk, dv.  W waves x R keys; over the heads that share them and tiles of 64 queries: S = Q K^T, dP = dO V^T (a lane holds one key, K and V stay in
// registers), dV^T += dO^T P, dK^T += Q^T dS.  Eight operations per pair and element.  A: 292 us (471 TFLOP/s), C: 181, B: 630 in two parts;
// bound as dq is, matrix cores busy 31 %.
template <typename T, int DP, Form FORM>
__global__ void __launch_bounds__((64 * Shape<T, DP>::W), (Shape<T, DP>::OCCUPANCY)) attention_dkv_kernel(tvl_attention_args a, tvl_attention_grads gr, const DocumentSpan* __restrict__ spans, const float* __restrict__ delta,
                                                            int tiles, int parts, float* __restrict__ slabs) {
    constexpr bool WIDE = FORM != ODD;
    constexpr int R = Shape<T, DP>::R, THREADS = 64 * Shape<T, DP>::W, KB = 128, CK = CHUNK<R>, N = VALUES<R>;
    typedef Tile<T, DP> L;
    typedef typename Operand<T>::elem E;
    extern __shared__ __align__(16) char lds[];
    constexpr int TILE = GT * L::ROW, STEP = 2 * TILE + 2 * GT * 4 + (FORM == PLAIN ? 0 : GT * 8);     // q, grad_out, log-sums, deltas, documents

    const int group = (int)(a.heads / a.kv_heads), pairs = (int)(a.batch * a.kv_heads);
    // `parts` workgroups share the heads of a group
    const Place at = place_of(blockIdx.x, pairs, parts, tiles);
    const int share = group / parts, head0 = at.head * share;
    const int b = at.pair / (int)a.kv_heads, hk = at.pair % (int)a.kv_heads;
    const int wave = wave_number(), lane = threadIdx.x % 64, r = lane % R, g = lane / R;
    const int k0 = (tiles - 1 - at.tile) * KB, kw = k0 + wave * R, j = kw + r;    // with a causal mask the first keys have the most queries
    const int dim = (int)a.dim, queries = (int)a.queries, keys = (int)a.keys;
    bool lost;
    const Sequence seq = sequence_of<false>(a, b, lost);
    const int64_t* docs = FORM == PLAIN ? nullptr : a.documents;
    int64_t doc = -1;
    DocumentWindow docw;
    if (docs) {
        docs += b * a.documents_batch;
        if (j < keys) doc = docs[j];
        docw.start(spans + (int64_t)b * ((queries + SPAN - 1) / SPAN), queries, k0, KB);
    }
    Frag<T> kf[DP / CK], vf[DP / CK];
#pragma unroll
    for (int c = 0; c < DP / CK; ++c) {
        kf[c] = vf[c] = Frag<T>{};
        if (j < keys) {
            kf[c] = load_frag<T, WIDE>((const T*)a.k + b * a.k_batch + (int64_t)j * a.k_token + hk * a.k_head, g + (64 / R) * c, dim);
            vf[c] = load_frag<T, WIDE>((const T*)a.v + b * a.v_batch + (int64_t)j * a.v_token + hk * a.v_head, g + (64 / R) * c, dim);
        }
    }
    Range range;
    constexpr float UP = BACKWARD_LIFT<T>;
    const bool capped = FORM != PLAIN && a.softcap > 0.0f, biased = FORM != PLAIN && a.slopes != nullptr;
    const float to_log2 = a.scale * LOG2E, to_cap = capped ? a.scale / a.softcap : 0.0f, from_cap = a.softcap * LOG2E;
    const float pre = capped ? 1.0f : to_log2, unit = capped || biased ? 1.0f : to_log2;
    Acc<R> dk[DP / R] = {}, dv[DP / R] = {};

    // queries in front of this one see key 0 at most: a softmax over one key has no slope
    const int lone = keys <= 1 ? queries : (seq.causal && seq.prefix <= 1 ? 1 - seq.shift : 0);
    // query i sees key j from i = j - shift on (all of them for keys in the prefix)
    int begin = seq.causal && k0 >= seq.prefix ? k0 - seq.shift : 0;
    begin = begin < 0 ? 0 : begin / GT * GT;
    const int steps = begin < queries ? (queries - begin + GT - 1) / GT : 0, total = steps * share;
    // steps in order: tiles of the first head, then of the next; tiles without a document of the block's are skipped
    auto next = [&](int n) {
        if (!docs) return n;
        while (n < total) {
            const int from = n / steps * steps, at = begin / SPAN, m = docw.next(at + n - from, at + steps, lane) - at;
            if (m < steps) return from + m;
            n = from + steps;
        }
        return n;
    };
    const int lane_row = L::template lane_row<R>(lane), lane_col = L::template lane_column<R>(lane);
    Stage<T, DP, GT, THREADS, WIDE> stage;
    float side = 0.0f;      // threads 0..63: a log-sum (less UP: weights and score gradients come out 2^UP times as large), 64..127: a delta
    int64_t qdoc = -1;      // threads 0..63
    auto fetch_queries = [&](int n) {
        const int h = hk * group + head0 + n / steps, i0 = begin + (n % steps) * GT;
        stage.load((const T*)a.q + b * a.q_batch + h * a.q_head, a.q_token, i0, queries, dim);
        const int i = i0 + (threadIdx.x & 63);
        const int64_t row = ((int64_t)b * a.heads + h) * queries + i;
        // a query behind the last gets weights exp(-inf) = 0
        if (threadIdx.x < 64) side = i < queries ? a.lse[row] * LOG2E - UP : __builtin_inff();
        else if (threadIdx.x < 128) side = i < queries ? delta[row] : 0.0f;
        if (docs && threadIdx.x < GT) qdoc = i < queries ? docs[i] : -1;
    };
    auto put_queries = [&](char* to) {
        stage.store(to);
        if (threadIdx.x < 128) *reinterpret_cast<float*>(to + 2 * TILE + 4 * threadIdx.x) = side;
        if (docs && threadIdx.x < GT) reinterpret_cast<int64_t*>(to + 2 * TILE + 2 * GT * 4)[threadIdx.x] = qdoc;
    };
    auto fetch_grads = [&](int n) {
        stage.load((const T*)gr.grad_out + b * gr.g_batch + (hk * group + head0 + n / steps) * gr.g_head, gr.g_token, begin + (n % steps) * GT, queries, dim);
    };
    int n = next(0), buf = 0;
    if (n < total) {
        fetch_queries(n);
        put_queries(lds);
        fetch_grads(n);
        stage.store(lds + TILE);
    }
    __syncthreads();
    // MASKED: some query of the tile does not see some key of the block
    auto step = [&](auto masks) __attribute__((always_inline)) {
        constexpr bool MASKED = decltype(masks)::value;
        const int n1 = next(n + 1);
        char* ahead = lds + (buf ^ 1) * STEP;
        if (n1 < total) fetch_queries(n1);
        const char *qt = lds + buf * STEP, *gt = qt + TILE;
        const float *lses = reinterpret_cast<const float*>(qt + 2 * TILE), *deltas = lses + GT;
        const int64_t* qdocs = reinterpret_cast<const int64_t*>(deltas + GT);
        const int h = hk * group + head0 + n / steps, i0 = begin + (n % steps) * GT;
        const float slope = biased ? a.slopes[h] * LOG2E : 0.0f;
        const bool one_document = !MASKED || !docs || docw.one(i0 / SPAN, lane);
        auto piece = [&](int t) __attribute__((always_inline)) {
            const int it = i0 + t;
            const int ilast = it + PIECE < queries ? it + PIECE - 1 : queries - 1;
            if (MASKED && (it >= queries || kw >= keys)) return;
            if (MASKED && seq.limit(ilast) <= kw) return;                              // none of these queries sees a key of the wave
            float s[N], dp[N];
#pragma unroll
            for (int n = 0; n < PIECE / R; ++n) {
                Acc<R> u = {}, w = {};
#pragma unroll
                for (int c = 0; c < DP / CK; ++c) {
                    u = mma(L::template read<R>(qt + t * L::ROW, lane_row, n * R, c), kf[c], u);
                    w = mma(L::template read<R>(gt + t * L::ROW, lane_row, n * R, c), vf[c], w);
                }
#pragma unroll
                for (int x = 0; x < REGS<R>; ++x) { s[n * REGS<R> + x] = u[x]; dp[n * REGS<R> + x] = w[x]; }
            }
            const bool masked = MASKED && (seq.limit(it) < kw + R || !one_document);
            Frag<T> pf[PIECE / CK], df[PIECE / CK];
            const float *ls = lses + t + 4 * g, *dl = deltas + t + 4 * g;
            if (capped) {
#pragma unroll
                for (int x = 0; x < N; ++x) s[x] *= to_cap;
                cap_tanh<T, FORM, N>(s, a.softcap);
#pragma unroll
                for (int x = 0; x < N; ++x) {
                    dp[x] = product(dp[x] - dl[piece_row<R>(x)], __builtin_fmaf(-s[x], s[x], 1.0f));
                    s[x] *= from_cap;
                }
            } else {
#pragma unroll
                for (int x = 0; x < N; ++x) dp[x] -= dl[piece_row<R>(x)];
            }
            if (biased) {
                const int here = it + 4 * g + seq.shift - j;
#pragma unroll
                for (int x = 0; x < N; ++x) s[x] = __builtin_fmaf(-slope, fabsf((float)(here + piece_row<R>(x))), s[x] * pre);
            }
#pragma unroll
            for (int x = 0; x < N; ++x) {
                s[x] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x], unit, -ls[piece_row<R>(x)]));
                dp[x] = product(dp[x], s[x]);
            }
            if (MASKED && masked) {
                // query i = it + 4 g + row sees key j if j is in its sequence's prefix or not behind its place
                const int from = j >= seq.end ? PIECE : (!seq.causal || j < seq.prefix ? -PIECE : j - seq.shift - it - 4 * g);
                const int slope_from = kw == 0 && lone - it - 4 * g > from ? lone - it - 4 * g : from;
#pragma unroll
                for (int x = 0; x < N; ++x) {
                    if (piece_row<R>(x) < from) s[x] = 0.0f;
                    if (piece_row<R>(x) < slope_from) dp[x] = 0.0f;
                }
                if (!one_document) {
#pragma unroll
                    for (int x = 0; x < N; ++x)
                        if (!same_document(qdocs + t + 4 * g + piece_row<R>(x), doc)) s[x] = dp[x] = 0.0f;
                }
            }
            // weights and score gradients are rounded to the operands' type for the last products; their sums are float32
            const bool spoilt = MASKED && masked && (holds_not_finite<T, DP, PIECE>(gt + t * L::ROW, lane) || holds_not_finite<T, DP, PIECE>(qt + t * L::ROW, lane));
            auto across = [&](const char* tile, int c, int d) __attribute__((always_inline)) {
                Frag<T> f = L::template read_across<R>(tile + t * L::ROW, lane_col, c * CK, d);
                if (MASKED && spoilt) f = finite_part<T>(f);
                return f;
            };
#pragma unroll
            for (int x = 0; x < N; ++x) pf[x / 8][x % 8] = (E)s[x];
#pragma unroll
            for (int c = 0; c < PIECE / CK; ++c)
#pragma unroll
                for (int d = 0; d < DP / R; ++d) dv[d] = mma(across(gt, c, d), pf[c], dv[d]);
            if constexpr (__is_same(T, f16)) {
                range.follow<R>(dp, dk);
                if (range.scaled) {
#pragma unroll
                    for (int x = 0; x < N; ++x) dp[x] = product(dp[x], range.fit);
                }
            }
#pragma unroll
            for (int x = 0; x < N; ++x) df[x / 8][x % 8] = (E)dp[x];
#pragma unroll
            for (int c = 0; c < PIECE / CK; ++c)
#pragma unroll
                for (int d = 0; d < DP / R; ++d) dk[d] = mma(across(qt, c, d), df[c], dk[d]);
            if (MASKED && spoilt) {
#pragma unroll 1
                for (int row = 0; row < PIECE && it + row < queries; ++row) {
                    const bool sees = j < seq.limit(it + row) && (one_document || (doc >= 0 && qdocs[t + row] == doc));
                    add_not_finite<T, DP, R>(gt, t + row, sees, false, g, dv);
                    add_not_finite<T, DP, R>(qt, t + row, sees, true, g, dk);
                }
            }
        };
        piece(0);
        if (n1 < total) {
            put_queries(ahead);
            fetch_grads(n1);
        }
        piece(PIECE);
        if (n1 < total) stage.store(ahead + TILE);
        __syncthreads();
        buf ^= 1;
        n = n1;
    };
    auto clean = [&](int m) {
        const int i0 = begin + (m % steps) * GT;
        return seq.limit(i0) >= k0 + KB && (!docs || docw.one(i0 / SPAN, lane));
    };
    while (n < total) {
        while (n < total && !clean(n)) step(std::true_type{});
        while (n < total && clean(n)) step(std::false_type{});
    }
    if (j >= keys) return;
    const float down = 1.0f / (float)(1 << (int)UP), back = a.scale / range.fit * down;
    const int64_t row = (((int64_t)b * keys + j) * a.kv_heads + hk) * dim;
#pragma unroll
    for (int d = 0; d < DP / R; ++d)
#pragma unroll
        for (int x = 0; x < REGS<R>; ++x) {
            const int col = d * R + result_row<R>(x, g);
            if (col >= dim) continue;
            if (parts > 1) {
                const int64_t all = (int64_t)a.batch * keys * a.kv_heads * dim;
                slabs[at.head * 2 * all + row + col] = dk[d][x] * back;
                slabs[(at.head * 2 + 1) * all + row + col] = dv[d][x] * down;
            } else {
                ((T*)gr.dk)[row + col] = from_float<T>(product(dk[d][x], back));
                ((T*)gr.dv)[row + col] = from_float<T>(product(dv[d][x], down));
            }
        }
}

// dk and dv from the parts of a group's heads, added in order: bound by HBM
template <typename T>
__global__ void __launch_bounds__(256) attention_gather_kernel(const float* __restrict__ slabs, int parts, int64_t n, T* __restrict__ dk, T* __restrict__ dv) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float x = 0.0f, y = 0.0f;
        for (int p = 0; p < parts; ++p) {
            x += slabs[p * 2 * n + i];
            y += slabs[(p * 2 + 1) * n + i];
        }
        dk[i] = from_float<T>(x);
        dv[i] = from_float<T>(y);
    }
}

// Parts of a group's heads: a key tile whose workgroup takes all heads in turn is the longest chain of the pass, so where the key tiles alone do not
// give two workgroups per compute unit the heads are divided (float32 sums through memory, added in order by a second launch of 13 us).  The backward pass in one part and
// as divided, us: B 1351 and 1084; 8192 causal tokens, 16 / 4 heads of 128, bf16 2060 and 1424; 2048 tokens, 32 / 8 heads of 128 492 and 259; 1024 tokens, 32 heads of 64 over one
// key head, f16 1120 and 100; 2 x 512 tokens, 16 / 4 heads of 64 100-120 and 85-119; 4 x 2048 tokens, 32 / 8 heads of 128, bf16, not divided further, 1112 and 1095.
int attention_backward_parts(const tvl_attention_args& a) {
    if (a.queries == 0) return 1;      // sums of nothing: no workspace either
    const int64_t tiles = a.batch * a.kv_heads * ceil_div(a.keys, 128);
    const int group = (int)(a.heads / a.kv_heads);
    for (int p = 1; p < group; ++p)
        if (group % p == 0 && tiles * p >= 512) return p;
    return group;
}

template <typename T, int DP, Form FORM, bool BARE>
static int launch_dq(const tvl_attention_args& a, const tvl_attention_grads& g, const DocumentSpan* spans, float* delta, hipStream_t st) {
    const int64_t tiles = ceil_div(a.queries, 128);
    const size_t bytes = 4 * GT * (size_t)Tile<T, DP>::ROW + (FORM == PLAIN ? 0 : 2 * GT * 8);
    if (bytes > 65536) TVL_HIP_CHECK(hipFuncSetAttribute((const void*)attention_dq_kernel<T, DP, FORM, BARE>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    hipLaunchKernelGGL((attention_dq_kernel<T, DP, FORM, BARE>), dim3((unsigned)(a.batch * a.heads * tiles)), dim3(64 * Shape<T, DP>::W), bytes, st, a, g, spans, delta, (int)tiles);
    TVL_LAUNCH_CHECK();
    return TVL_OK;
}

template <typename T, int DP, Form FORM>
static int launch_gradients(const tvl_attention_args& a, const tvl_attention_grads& g, const DocumentSpan* spans, float* delta, float* slabs, hipStream_t st) {
    if (g.dq && a.queries > 0) {
        if (const int rc = launch_dq<T, DP, FORM, false>(a, g, spans, delta, st); rc != TVL_OK) return rc;
    }
    if constexpr (sizeof(T) == 2)
        if (!g.dq && g.dk && a.queries > 0 && a.keys > 0)
            if (const int rc = launch_dq<T, DP, FORM, true>(a, g, spans, delta, st); rc != TVL_OK) return rc;
    if (g.dk && a.keys > 0) {
        const int blocks = (int)ceil_div(a.keys, 128), parts = attention_backward_parts(a);
        const size_t bytes = 2 * (2 * GT * (size_t)Tile<T, DP>::ROW + 2 * GT * 4 + (FORM == PLAIN ? 0 : GT * 8));
        if (bytes > 65536) TVL_HIP_CHECK(hipFuncSetAttribute((const void*)attention_dkv_kernel<T, DP, FORM>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
        hipLaunchKernelGGL((attention_dkv_kernel<T, DP, FORM>), dim3((unsigned)(a.batch * a.kv_heads * blocks * parts)), dim3(64 * Shape<T, DP>::W), bytes, st, a, g, spans, delta,
                           blocks, parts, slabs);
        TVL_LAUNCH_CHECK();
        if (parts > 1) {
            const int64_t n = a.batch * a.keys * a.kv_heads * a.dim, most = ceil_div(n, 256);
            hipLaunchKernelGGL((attention_gather_kernel<T>), dim3((unsigned)(most < 4096 ? most : 4096)), dim3(256), 0, st, slabs, parts, n, (T*)g.dk, (T*)g.dv);
            TVL_LAUNCH_CHECK();
        }
    }
    return TVL_OK;
}

template <typename T>
static int launch_backward(const tvl_attention_args& a, const tvl_attention_grads& g, const DocumentSpan* spans, float* delta, float* slabs, hipStream_t st) {
    const size_t z = sizeof(T);
    const bool grad = wide_rows(g.grad_out, a.dim, g.g_batch, g.g_token, g.g_head, z);
    const bool wide = grad && wide_rows(a.q, a.dim, a.q_batch, a.q_token, a.q_head, z) && wide_rows(a.k, a.dim, a.k_batch, a.k_token, a.k_head, z) &&
                      wide_rows(a.v, a.dim, a.v_batch, a.v_token, a.v_head, z);
    if (a.queries > 0) {
        const int blocks = (int)ceil_div(a.queries, GT);
        const unsigned n = (unsigned)(a.batch * a.heads * blocks);
        if (grad && wide_rows(a.out, a.dim, a.o_batch, a.o_token, a.o_head, z)) hipLaunchKernelGGL((attention_delta_kernel<T, true>), dim3(n), dim3(256), 0, st, a, g, delta, blocks);
        else hipLaunchKernelGGL((attention_delta_kernel<T, false>), dim3(n), dim3(256), 0, st, a, g, delta, blocks);
        TVL_LAUNCH_CHECK();
    }
    // odd rows take the same shapes: the same sums in the same order
    return with_form<T>(a, wide, [&](auto form) {
        constexpr Form FORM = decltype(form)::value;
        return a.dim <= 64 ? launch_gradients<T, 64, FORM>(a, g, spans, delta, slabs, st) : launch_gradients<T, 128, FORM>(a, g, spans, delta, slabs, st);
    });
}

int launch_attention_backward(const tvl_attention_args& a, const tvl_attention_grads& g, const DocumentSpan* spans, float* delta, float* slabs, hipStream_t st) {
    if (a.dtype == TVL_F32) return launch_backward<float>(a, g, spans, delta, slabs, st);
    if (a.dtype == TVL_F16) return launch_backward<f16>(a, g, spans, delta, slabs, st);
    return launch_backward<bf16_t>(a, g, spans, delta, slabs, st);
}

}  // namespace tvl
