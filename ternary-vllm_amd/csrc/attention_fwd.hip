// Forward attention over tiles: tvl_attention, and tvl_cached_attention for chunks of many tokens.
#include "attention_tiles.h"

namespace tvl {

// One workgroup: 4 waves x 32 queries of one head; keys and values come in tiles of 64 through LDS, two buffers, the next tile's loads in
// flight while this one is used: its keys during the scores, its values during the rest, through one set of registers (two sets spill at heads of 128).  Per wave and tile: S^T = K Q^T (a lane holds 32 scores of ONE query: maximum and sum are plain loops
// over its registers plus one exchange with the other half), weights 2^(s - m) rounded to the operands' type as the second product's operand,
// O^T += V^T P^T.  m is kept until a score exceeds it by 8 (in powers of two): the weights stay below 2^8 (float16: 2^15, see LIFT), and the
// accumulator is almost never rescaled.  Tiles that every query sees whole run in a loop without masks.
// Heads of 128: 8192 x 8192, 16 heads, f16 645 us (850 TFLOP/s), causal bf16 16 / 4 heads 340 us (810), capped 540; heads of 64: 4 x 2048, 32 heads, bf16
// 207 us (660 TFLOP/s), causal 152 us (452), 128 x 197, 12 heads, f16 64 us (238).  A score costs an exponential and about four other vector instructions
// whatever the head's length, so heads of 64 are bound by the vector ALU; heads of 128 reach 76 % of the rate of a large library product.  One set of registers
// instead of two, and banks without conflicts, took them from 883 to below 700 us; 16-bit forms of heads of 128 still keep some registers in scratch memory (19 to 22 in PLAIN, 60 to 168 in the others).
template <typename T, int DP, bool CACHED, Form FORM>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) attention_forward_kernel(tvl_attention_args a, const DocumentSpan* __restrict__ spans, int tiles) {
    constexpr bool WIDE = FORM != ODD;
    constexpr int R = 32, KT = 64, QB = 128, CK = CHUNK<R>;
    typedef Tile<T, DP> L;
    extern __shared__ __align__(16) char lds[];
    constexpr int TILE = KT * L::ROW, BUFFER = 2 * TILE + (FORM == PLAIN ? 0 : KT * 8);     // keys, values, documents

    const int group = (int)(a.heads / a.kv_heads), pairs = (int)(a.batch * a.kv_heads);
    const Place at = place_of(blockIdx.x, pairs, group, tiles);
    const int b = at.pair / (int)a.kv_heads, hk = at.pair % (int)a.kv_heads, h = hk * group + at.head;
    const int wave = wave_number(), lane = threadIdx.x % 64, r = lane % R, g = lane / R;
    const int q0 = at.tile * QB, qw = q0 + wave * R, i = qw + r;
    const int dim = (int)a.dim, queries = (int)a.queries;

    bool lost;
    const Sequence seq = sequence_of<CACHED>(a, b, lost);
    const int last = q0 + QB < seq.real ? q0 + QB : seq.real;                  // real queries of this block end here
    const int reach = last > q0 ? seq.limit(last - 1) : 0;                      // limits grow with the query
    const int all = last > q0 ? seq.limit(q0) : 0;                              // keys every real query of the block sees
    const int wlast = qw + R < seq.real ? qw + R : seq.real;
    const int wreach = wlast > qw ? seq.limit(wlast - 1) : 0, wall = wlast > qw ? seq.limit(qw) : 0;   // keys some / every query of the wave sees
    const int mine = i < seq.real ? seq.limit(i) : 0;

    const T* kp = (const T*)a.k + b * a.k_batch + hk * a.k_head;
    const T* vp = (const T*)a.v + b * a.v_batch + hk * a.v_head;
    const T* qp = (const T*)a.q + b * a.q_batch + h * a.q_head + (int64_t)i * a.q_token;
    const int64_t* docs = CACHED || FORM == PLAIN ? nullptr : a.documents;
    int64_t doc = -1;
    DocumentWindow docw;
    if (docs) {
        docs += b * a.documents_batch;
        if (i < queries) doc = docs[i];
        docw.start(spans + (int64_t)b * ((queries + SPAN - 1) / SPAN), queries, q0, QB);
    }

    // a negative scale goes into the queries' sign, so that the largest product is the largest score
    const float scale = fabsf(a.scale);
    Frag<T> qf[DP / CK];
#pragma unroll
    for (int c = 0; c < DP / CK; ++c) {
        qf[c] = Frag<T>{};
        if (i < seq.real) qf[c] = load_frag<T, WIDE>(qp, g + (64 / R) * c, dim);
        if (a.scale < 0.0f) qf[c] = -qf[c];
    }
    const float slope = a.slopes ? a.slopes[h] * LOG2E : 0.0f;
    const bool capped = FORM != PLAIN && a.softcap > 0.0f, biased = FORM != PLAIN && (a.slopes != nullptr || a.scale == 0.0f);
    const float to_log2 = scale * LOG2E, to_cap = capped ? scale / a.softcap : 0.0f, from_cap = a.softcap * LOG2E;
    // without cap and bias the scaling is part of the exponential's argument (a zero scale would make NaN of -infinity there)
    const float pre = capped ? 1.0f : to_log2, unit = capped || biased ? 1.0f : to_log2;

    Acc<R> acc[DP / R] = {};
    float m = -__builtin_inff(), base = 0.0f, sum = 0.0f;

    // tiles whose documents no query of the block has are skipped
    auto next = [&](int j) { return docs && j < reach ? docw.next(j / SPAN, (reach + SPAN - 1) / SPAN, lane) * SPAN : j; };
    // one set of staging registers: the next keys are on their way while the scores are formed, the next values during the rest
    Stage<T, DP, KT, 256, WIDE> stage;
    int64_t side = -1;
    auto fetch_keys = [&](int j) {
        stage.load(kp, a.k_token, j, seq.end, dim);
        if (docs && threadIdx.x < KT) side = j + (int)threadIdx.x < seq.end ? docs[j + threadIdx.x] : -1;
    };
    auto put_keys = [&](char* to) {
        stage.store(to);
        if (docs && threadIdx.x < KT) reinterpret_cast<int64_t*>(to + 2 * TILE)[threadIdx.x] = side;
    };
    const int lane_row = L::template lane_row<R>(lane), lane_col = L::template lane_column<R>(lane);
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
        const int j1 = next(j0 + KT);
        if (j1 < reach) fetch_keys(j1);
        char* ahead = lds + (buf ^ 1) * BUFFER;
        const char *kt = lds + buf * BUFFER, *vt = kt + TILE;
        const int64_t* kdocs = reinterpret_cast<const int64_t*>(kt + 2 * TILE);
        const bool busy = !MASKED || j0 < wreach;
        Acc<R> s[KT / R];
        if (busy) {
#pragma unroll
            for (int t = 0; t < KT / R; ++t) {
                s[t] = Acc<R>{};
#pragma unroll
                for (int c = 0; c < DP / CK; ++c) s[t] = mma(L::template read<R>(kt, lane_row, t * R, c), qf[c], s[t]);
            }
        }
        if (j1 < reach) {
            put_keys(ahead);
            stage.load(vp, a.v_token, j1, seq.end, dim);
        }
        if (busy) {
            // scores: units of `unit` powers of two
            const bool one_document = !MASKED || !docs || docw.one(j0 / SPAN, lane);
            if (capped) {
#pragma unroll
                for (int t = 0; t < KT / R; ++t) {
                    s[t] *= to_cap;
                    cap_tanh<T, FORM, REGS<R>>(s[t], a.softcap);
                    s[t] *= from_cap;
                }
            }
            if (biased) {
                const int here = i + seq.shift - j0 - 4 * g;
#pragma unroll
                for (int t = 0; t < KT / R; ++t)
#pragma unroll
                    for (int x = 0; x < REGS<R>; ++x) {
                        const float away = fabsf((float)(here - (t * R + result_row<R>(x, 0))));
                        s[t][x] = __builtin_fmaf(-slope, away, s[t][x] * pre);
                    }
            }
            if (MASKED && (j0 + KT > wall || !one_document)) {
                const int left = mine - j0 - 4 * g;
#pragma unroll
                for (int t = 0; t < KT / R; ++t)
#pragma unroll
                    for (int x = 0; x < REGS<R>; ++x)
                        if (t * R + result_row<R>(x, 0) >= left) s[t][x] = -__builtin_inff();
                if (!one_document) {
#pragma unroll
                    for (int t = 0; t < KT / R; ++t)
#pragma unroll
                        for (int x = 0; x < REGS<R>; ++x)
                            if (!same_document(kdocs + t * R + result_row<R>(x, g), doc)) s[t][x] = -__builtin_inff();
                }
            }
            float top = s[0][0];
#pragma unroll
            for (int t = 0; t < KT / R; ++t)
#pragma unroll
                for (int x = 0; x < REGS<R>; ++x) top = fmaxf(top, s[t][x]);
            top = column_max<R>(top) * unit;
            const bool grow = top > m + 8.0f;
            if (__any(grow)) {
                const float now = grow ? top : m, shrink = grow ? __builtin_amdgcn_exp2f(m - now) : 1.0f;
                m = now;
                base = m == -__builtin_inff() ? 0.0f : m - LIFT<T>;
                sum *= shrink;
#pragma unroll
                for (int d = 0; d < DP / R; ++d) acc[d] *= shrink;
            }
            Frag<T> pf[KT / CK];
#pragma unroll
            for (int t = 0; t < KT / R; ++t)
#pragma unroll
                for (int x = 0; x < REGS<R>; ++x) {
                    const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][x], unit, -base));
                    sum += w;
                    // weights are rounded to the operands' type for the second product (relative 2^-11 / 2^-8 each, the sum stays float32)
                    pf[(t * REGS<R> + x) / 8][x % 8] = (typename Operand<T>::elem)w;
                }
            // keys of this tile that some query of the wave does not see (a prefix may end here for all of them): an infinity or NaN in their values must not reach it
            if (MASKED && (!one_document || (j0 + KT > wall && wall < seq.end)) && holds_not_finite<T, DP, KT>(vt, lane)) {
#pragma unroll
                for (int c = 0; c < KT / CK; ++c)
#pragma unroll
                    for (int d = 0; d < DP / R; ++d) acc[d] = mma(finite_part<T>(L::template read_across<R>(vt, lane_col, c * CK, d)), pf[c], acc[d]);
#pragma unroll 1
                for (int row = 0; row < KT && j0 + row < reach; ++row)
                    add_not_finite<T, DP, R>(vt, row, j0 + row < mine && (one_document || (doc >= 0 && kdocs[row] == doc)), false, g, acc);
            } else {
#pragma unroll
                for (int c = 0; c < KT / CK; ++c)
#pragma unroll
                    for (int d = 0; d < DP / R; ++d) acc[d] = mma(L::template read_across<R>(vt, lane_col, c * CK, d), pf[c], acc[d]);
            }
        }
        if (j1 < reach) stage.store(ahead + TILE);
        __syncthreads();
        buf ^= 1;
        j0 = j1;
    };
    auto clean = [&](int j) { return j + KT <= all && (!docs || docw.one(j / SPAN, lane)); };
    while (j0 < reach) {
        while (j0 < reach && clean(j0)) step(std::false_type{});
        while (j0 < reach && !clean(j0)) step(std::true_type{});
    }

    sum = column_sum<R>(sum);
    if (i >= queries) return;
    const bool empty = sum == 0.0f || i >= seq.real;      // sees nothing, or padding (whose registers hold what unmasked tiles gave it)
    const float inv = 1.0f / sum;
    const bool nan = CACHED && i < seq.real && (lost || seq.shift + i >= (int)a.keys);
    T* op = (T*)a.out + b * a.o_batch + (int64_t)i * a.o_token + h * a.o_head;
#pragma unroll
    for (int d = 0; d < DP / R; ++d)
#pragma unroll
        for (int x = 0; x < REGS<R>; x += 4) {
            const int col = d * R + result_row<R>(x, g);
            T v[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) v[y] = from_float<T>(nan ? __builtin_nanf("") : (empty ? 0.0f : product(acc[d][x + y], inv)));
            if constexpr (WIDE) {
                typedef uint32_t quad __attribute__((ext_vector_type(sizeof(T))));
                if (col < dim) *reinterpret_cast<quad*>(op + col) = *reinterpret_cast<const quad*>(v);
            } else {
#pragma unroll
                for (int y = 0; y < 4; ++y)
                    if (col + y < dim) op[col + y] = v[y];
            }
        }
    if (!CACHED && a.lse && g == 0) a.lse[((int64_t)b * a.heads + h) * queries + i] = sum == 0.0f ? -__builtin_inff() : (base + __builtin_amdgcn_logf(sum)) * LN2;
}

// spans[b][n] of tokens 64 n .. 64 n + 63: 64 KB for 8191 tokens, bound by the launch (4.9 us)
__global__ void __launch_bounds__(64) document_spans_kernel(const int64_t* __restrict__ documents, int64_t stride, int tokens, int blocks, DocumentSpan* __restrict__ spans) {
    const int b = blockIdx.x / blocks, n = blockIdx.x % blocks, i = n * SPAN + threadIdx.x;
    const int64_t doc = documents[b * stride + (i < tokens ? i : n * SPAN)];
    int64_t lo = doc < 0 ? INT64_MAX : doc, hi = doc < 0 ? -1 : doc;
    for (int o = 32; o > 0; o >>= 1) {
        const int64_t l = __shfl_xor((long long)lo, o), u = __shfl_xor((long long)hi, o);
        lo = l < lo ? l : lo;
        hi = u > hi ? u : hi;
    }
    const bool whole = __all(doc >= 0);
    if (threadIdx.x == 0) spans[blockIdx.x] = DocumentSpan{lo, hi, whole};
}

int launch_document_spans(const tvl_attention_args& a, DocumentSpan* spans, hipStream_t st) {
    const int blocks = (int)ceil_div(a.queries, SPAN);
    hipLaunchKernelGGL(document_spans_kernel, dim3((unsigned)(a.batch * blocks)), dim3(64), 0, st, a.documents, a.documents_batch, (int)a.queries, blocks, spans);
    TVL_LAUNCH_CHECK();
    return TVL_OK;
}

template <typename T, int DP, bool CACHED, Form FORM>
static int launch_forward(const tvl_attention_args& a, const DocumentSpan* spans, hipStream_t st) {
    const int tiles = (int)ceil_div(a.queries, 128);
    const size_t bytes = 4 * 64 * (size_t)Tile<T, DP>::ROW + (FORM == PLAIN ? 0 : 2 * 64 * 8);
    if (bytes > 65536) TVL_HIP_CHECK(hipFuncSetAttribute((const void*)attention_forward_kernel<T, DP, CACHED, FORM>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    hipLaunchKernelGGL((attention_forward_kernel<T, DP, CACHED, FORM>), dim3((unsigned)(a.batch * a.heads * tiles)), dim3(256), bytes, st, a, spans, tiles);
    TVL_LAUNCH_CHECK();
    return TVL_OK;
}

template <typename T, bool CACHED>
static int launch_forward_t(const tvl_attention_args& a, const DocumentSpan* spans, hipStream_t st) {
    const size_t z = sizeof(T);
    const bool wide = wide_rows(a.q, a.dim, a.q_batch, a.q_token, a.q_head, z) && wide_rows(a.k, a.dim, a.k_batch, a.k_token, a.k_head, z) &&
                      wide_rows(a.v, a.dim, a.v_batch, a.v_token, a.v_head, z) && wide_rows(a.out, a.dim, a.o_batch, a.o_token, a.o_head, z);
    return with_form<T>(a, wide, [&](auto form) {
        constexpr Form FORM = decltype(form)::value;
        return a.dim <= 64 ? launch_forward<T, 64, CACHED, FORM>(a, spans, st) : launch_forward<T, 128, CACHED, FORM>(a, spans, st);
    });
}

int launch_attention_forward(const tvl_attention_args& a, bool cached, const DocumentSpan* spans, hipStream_t st) {
    if (a.dtype == TVL_F32) return cached ? launch_forward_t<float, true>(a, spans, st) : launch_forward_t<float, false>(a, spans, st);
    if (a.dtype == TVL_F16) return cached ? launch_forward_t<f16, true>(a, spans, st) : launch_forward_t<f16, false>(a, spans, st);
    return cached ? launch_forward_t<bf16_t, true>(a, spans, st) : launch_forward_t<bf16_t, false>(a, spans, st);
}

}  // namespace tvl
