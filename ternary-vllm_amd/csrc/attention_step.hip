// Attention of few new tokens over a cache: tvl_cached_attention for decode steps and drafted tokens.
#include "attention_tiles.h"

namespace tvl {

constexpr int WAVES = 8;      // of a workgroup, each on its own keys
constexpr int STEP = 32;      // keys a wave takes at a time
constexpr int ROWS = 16;      // rows (token, head of the group) of a workgroup

// Where the range of keys is cut: S parts of whole steps, by the sequence's own length
__device__ __forceinline__ void part_of(int reach, int splits, int n, int& lo, int& hi) {
    const int per = ((reach + splits - 1) / splits + STEP - 1) / STEP * STEP;
    lo = per * n < reach ? per * n : reach;
    hi = lo + per < reach ? lo + per : reach;
}

// One workgroup: all rows that share a key head (tokens x heads of the group, 16 at a time as the columns of 16 x 16 products) over one part of
// the keys.  The cache is read once, so the pass is bound by HBM; the products ride along at 1/16 .. 16/16 use.  Each wave
// takes 32 keys at a time: keys straight into operand registers, values through a piece of LDS of its own (no barrier in the loop), the
// next 32 keys' loads in flight.  The waves' running maxima, sums and accumulators are joined in LDS at the end, parts of a long
// cache by a second small launch.
// 256 sequences x 600 x 32 heads of 64, f16: 246 us, 5.1 TB/s; 4 x 28000 x 32 / 8 heads of 128, bf16, capped: 90 us, 5.1 TB/s (a large copy reaches 4.9); one sequence x 745:
// 8.3 us, of which 4 are an empty launch.
template <typename T, int DP, Form FORM>
__global__ void __launch_bounds__(64 * WAVES) attention_step_kernel(tvl_attention_args a, int tiles, int splits, float* __restrict__ parts) {
    constexpr bool WIDE = FORM != ODD;
    constexpr int R = 16, CK = CHUNK<R>;
    typedef Tile<T, DP> L;
    typedef typename Operand<T>::elem E;
    extern __shared__ __align__(16) char lds[];
    constexpr int UNITS = STEP * L::UNITS / 64;

    const int group = (int)(a.heads / a.kv_heads), pairs = (int)(a.batch * a.kv_heads), rows = (int)a.queries * group;
    // row tiles of one (sequence, key head) next to each other on one XCD: they read the same keys
    const Place at = place_of(blockIdx.x, pairs, tiles, splits);
    const int b = at.pair / (int)a.kv_heads, hk = at.pair % (int)a.kv_heads, first = at.head * ROWS, split = splits - 1 - at.tile;
    const int wave = wave_number(), lane = threadIdx.x % 64, r = lane % R, g = lane / R;
    const int row = first + r, i = row / group, h = hk * group + row % group;
    const int dim = (int)a.dim;
    bool lost;
    const Sequence seq = sequence_of<true>(a, b, lost);
    const int end = first + ROWS < rows ? first + ROWS : rows;                       // rows of this tile end here
    const int ilast = (end - 1) / group < seq.real ? (end - 1) / group : seq.real - 1, ifirst = first / group;
    const int reach = ilast >= ifirst ? seq.limit(ilast) : 0, all = ilast >= ifirst ? seq.limit(ifirst) : 0;
    const bool real = row < rows && i < seq.real;
    const int mine = real ? seq.limit(i) : 0;
    int lo, hi;
    part_of(reach, splits, split, lo, hi);

    Frag<T> qf[DP / CK];
    const float scale = fabsf(a.scale);
#pragma unroll
    for (int c = 0; c < DP / CK; ++c) {
        qf[c] = Frag<T>{};
        if (real) qf[c] = load_frag<T, WIDE>((const T*)a.q + b * a.q_batch + (int64_t)i * a.q_token + h * a.q_head, g + (64 / R) * c, dim);
        if (a.scale < 0.0f) qf[c] = -qf[c];
    }
    const bool capped = FORM != PLAIN && a.softcap > 0.0f, biased = FORM != PLAIN && (a.slopes != nullptr || a.scale == 0.0f);
    const float slope = biased && a.slopes && real ? a.slopes[h] * LOG2E : 0.0f;
    const float to_log2 = scale * LOG2E, to_cap = capped ? scale / a.softcap : 0.0f, from_cap = a.softcap * LOG2E;
    const float pre = capped ? 1.0f : to_log2, unit = capped || biased ? 1.0f : to_log2;

    const T* kp = (const T*)a.k + b * a.k_batch + hk * a.k_head;
    const T* vp = (const T*)a.v + b * a.v_batch + hk * a.v_head;
    char* vt = lds + wave * STEP * L::ROW;
    Frag<T> kf[STEP / R][DP / CK];
    u32x4 vv[UNITS];
    auto fetch = [&](int j0) {
#pragma unroll
        for (int t = 0; t < STEP / R; ++t) {
            const int j = j0 + t * R + r;
#pragma unroll
            for (int c = 0; c < DP / CK; ++c) {
                kf[t][c] = Frag<T>{};
                if (j < hi) kf[t][c] = load_frag<T, WIDE>(kp + (int64_t)j * a.k_token, g + (64 / R) * c, dim);
            }
        }
#pragma unroll
        for (int x = 0; x < UNITS; ++x) {
            const int u = lane + 64 * x, j = j0 + u / L::UNITS;
            vv[x] = u32x4{0, 0, 0, 0};
            if (j < hi) vv[x] = load_unit<T, WIDE>(vp + (int64_t)j * a.v_token, u % L::UNITS, dim);
        }
    };
    const int lane_col = L::template lane_column<R>(lane);
    Acc<R> acc[DP / R] = {};
    float m = -__builtin_inff(), base = 0.0f, sum = 0.0f;
    int j0 = lo + wave * STEP;
    if (j0 < hi) fetch(j0);
    while (j0 < hi) {
        Acc<R> s[STEP / R];
#pragma unroll
        for (int t = 0; t < STEP / R; ++t) {
            s[t] = Acc<R>{};
#pragma unroll
            for (int c = 0; c < DP / CK; ++c) s[t] = mma(kf[t][c], qf[c], s[t]);
        }
#pragma unroll
        for (int x = 0; x < UNITS; ++x) {
            const int u = lane + 64 * x;
            *reinterpret_cast<u32x4*>(vt + L::at(u / L::UNITS, u % L::UNITS)) = vv[x];
        }
        __builtin_amdgcn_wave_barrier();
        const int here = j0;
        j0 += WAVES * STEP;
        if (j0 < hi) fetch(j0);
        if (capped) {
#pragma unroll
            for (int t = 0; t < STEP / R; ++t) {
                s[t] *= to_cap;
                cap_tanh<T, FORM, REGS<R>>(s[t], a.softcap);
                s[t] *= from_cap;
            }
        }
        if (biased) {
            const int away = i + seq.shift - here - 4 * g;
#pragma unroll
            for (int t = 0; t < STEP / R; ++t)
#pragma unroll
                for (int x = 0; x < REGS<R>; ++x) s[t][x] = __builtin_fmaf(-slope, fabsf((float)(away - (t * R + result_row<R>(x, 0)))), s[t][x] * pre);
        }
        const bool masked = here + STEP > all || here + STEP > hi;
        const int left = (mine < hi ? mine : hi) - here - 4 * g;
        if (masked) {
#pragma unroll
            for (int t = 0; t < STEP / R; ++t)
#pragma unroll
                for (int x = 0; x < REGS<R>; ++x)
                    if (t * R + result_row<R>(x, 0) >= left) s[t][x] = -__builtin_inff();
        }
        float top = s[0][0];
#pragma unroll
        for (int t = 0; t < STEP / R; ++t)
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
        Frag<T> pf;
#pragma unroll
        for (int t = 0; t < STEP / R; ++t)
#pragma unroll
            for (int x = 0; x < REGS<R>; ++x) {
                const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][x], unit, -base));
                sum += w;
                pf[t * REGS<R> + x] = (E)w;      // rounded to the operands' type for the second product; the sum stays float32
            }
        // tokens of a chunk see different keys: an infinity or NaN in a later token's value must not reach an earlier token
        if (here + STEP > all && all < reach && holds_not_finite<T, DP, STEP>(vt, lane)) {
#pragma unroll
            for (int d = 0; d < DP / R; ++d) acc[d] = mma(finite_part<T>(L::template read_across<R>(vt, lane_col, 0, d)), pf, acc[d]);
#pragma unroll 1
            for (int x = 0; x < STEP && here + x < hi; ++x) add_not_finite<T, DP, R>(vt, x, here + x < mine, false, g, acc);
        } else {
#pragma unroll
            for (int d = 0; d < DP / R; ++d) acc[d] = mma(L::template read_across<R>(vt, lane_col, 0, d), pf, acc[d]);
        }
        __builtin_amdgcn_wave_barrier();
    }
    sum = column_sum<R>(sum);

    // join the waves: per wave [row][dim], then maxima and sums
    __syncthreads();
    float* joined = reinterpret_cast<float*>(lds);
    float* stats = joined + WAVES * ROWS * DP;
    const int used = end - first;
    if (r < used) {
#pragma unroll
        for (int d = 0; d < DP / R; ++d) *reinterpret_cast<f32x4*>(joined + (wave * ROWS + r) * DP + d * R + 4 * g) = acc[d];
        if (g == 0) { stats[wave * ROWS + r] = m; stats[(WAVES + wave) * ROWS + r] = sum; }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < used * DP; x += 64 * WAVES) {
        const int y = x / DP, col = x % DP, ry = first + y, iy = ry / group, hy = hk * group + ry % group;
        float top = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) top = fmaxf(top, stats[w * ROWS + y]);
        const float from = top == -__builtin_inff() ? 0.0f : top;
        float total = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float ws = stats[(WAVES + w) * ROWS + y];
            if (ws == 0.0f) continue;           // a wave that saw nothing
            const float f = __builtin_amdgcn_exp2f((stats[w * ROWS + y] == -__builtin_inff() ? 0.0f : stats[w * ROWS + y]) - from);
            total += f * ws;
            o += f * joined[(w * ROWS + y) * DP + col];
        }
        if (splits > 1) {
            float* part = parts + ((int64_t)(at.pair * (int64_t)splits + split) * rows + ry) * (DP + 2);
            part[2 + col] = o;
            if (col == 0) { part[0] = top; part[1] = total; }
        } else if (col < dim) {
            const bool empty = total == 0.0f || iy >= seq.real, nan = iy < seq.real && (lost || seq.shift + iy >= (int)a.keys);
            ((T*)a.out)[b * a.o_batch + (int64_t)iy * a.o_token + hy * a.o_head + col] = from_float<T>(nan ? __builtin_nanf("") : (empty ? 0.0f : o / total));
        }
    }
}

// out of the parts of a long cache: one workgroup per row; the parts' maxima and sums first, then every wave adds its share of the accumulators.
// Few kilobytes from L2, bound by the launch (4.7 us); one workgroup per sequence and key head took 74 us with its step for one pair x 32000 keys, now 20
constexpr int MOST_PARTS = 512;
template <typename T, int DP>
__global__ void __launch_bounds__(256) attention_join_kernel(tvl_attention_args a, int splits, const float* __restrict__ parts) {
    __shared__ float factor[MOST_PARTS], side[4], sums[4][DP];
    const int group = (int)(a.heads / a.kv_heads), rows = (int)a.queries * group, lane = threadIdx.x % 64, wave = wave_number();
    const int pair = (int)(blockIdx.x / (unsigned)rows), row = (int)(blockIdx.x % (unsigned)rows), i = row / group, b = pair / (int)a.kv_heads, h = pair % (int)a.kv_heads * group + row % group;
    const float* part = parts + ((int64_t)pair * splits * rows + row) * (DP + 2);
    const int64_t stride = (int64_t)rows * (DP + 2);
    float m[MOST_PARTS / 256], ws[MOST_PARTS / 256], top = -__builtin_inff();
#pragma unroll
    for (int x = 0; x < MOST_PARTS / 256; ++x) {
        const int s = threadIdx.x + 256 * x;
        m[x] = -__builtin_inff();
        ws[x] = 0.0f;
        if (s < splits) { m[x] = part[s * stride]; ws[x] = part[s * stride + 1]; }
        top = fmaxf(top, m[x]);
    }
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if (lane == 0) side[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(side[0], side[1]), fmaxf(side[2], side[3]));
    const float from = top == -__builtin_inff() ? 0.0f : top;
    float total = 0.0f;
#pragma unroll
    for (int x = 0; x < MOST_PARTS / 256; ++x) {
        // a part that saw nothing adds nothing
        const float f = ws[x] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f((m[x] == -__builtin_inff() ? 0.0f : m[x]) - from);
        if (ws[x] != 0.0f) total += f * ws[x];
        const int s = threadIdx.x + 256 * x;
        if (s < splits) factor[s] = f;
    }
    for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o);
    __syncthreads();
    if (lane == 0) side[wave] = total;
    float acc[DP / 64] = {};
#pragma unroll 4
    for (int s = wave; s < splits; s += 4) {
        const float f = factor[s];
#pragma unroll
        for (int d = 0; d < DP / 64; ++d) {
            const float v = part[s * stride + 2 + lane + 64 * d];
            acc[d] += f == 0.0f ? 0.0f : f * v;
        }
    }
#pragma unroll
    for (int d = 0; d < DP / 64; ++d) sums[wave][lane + 64 * d] = acc[d];
    __syncthreads();
    bool lost;
    const Sequence seq = sequence_of<true>(a, b, lost);
    total = (side[0] + side[1]) + (side[2] + side[3]);
    const int col = threadIdx.x;
    if (col >= (int)a.dim) return;
    const float o = (sums[0][col] + sums[1][col]) + (sums[2][col] + sums[3][col]);
    const bool empty = total == 0.0f || i >= seq.real, nan = i < seq.real && (lost || seq.shift + i >= (int)a.keys);
    ((T*)a.out)[b * a.o_batch + (int64_t)i * a.o_token + h * a.o_head + col] = from_float<T>(nan ? __builtin_nanf("") : (empty ? 0.0f : o / total));
}

static bool step_wide(const tvl_attention_args& a) {
    const size_t z = dtype_size(a.dtype);
    return wide_rows(a.q, a.dim, a.q_batch, a.q_token, a.q_head, z) && wide_rows(a.k, a.dim, a.k_batch, a.k_token, a.k_head, z) && wide_rows(a.v, a.dim, a.v_batch, a.v_token, a.v_head, z);
}

// Rows (tokens x heads of a group) that the cache kernel takes; more go to the tile kernel, which takes one head per workgroup and never cuts the keys.  Measured (us, us): 4
// sequences, 4 key heads of 128, 64 rows here, 72 there: 1000 keys 18, 35; 4000 keys 25, 121; 28000 keys 77, 778; one sequence, 32 heads of 64, 64 rows here, 65 there: 14.8, 22.9;
// 22, 71; 74, 456.  The bound keeps whole prompts with the tile kernel (8 x 745 over a fresh cache 56); long caches would be served by this one far beyond it, and are not yet.
bool attention_step_serves(const tvl_attention_args& a) {
    const int64_t rows = a.queries * (a.heads / a.kv_heads);
    return rows <= 64;
}

// Parts the keys are cut into: enough for one workgroup per compute unit, none shorter than 512 keys; a cache of up to 1024 slots stays whole, its
// second launch costs more than the parts gain.  Measured (us, us): 32 pairs x 745 of 1024 slots whole 8.3, 4 parts 9.3; 256 pairs x 745 whole 11.9,
// 2 parts 17.3; 32 pairs x 28000 x 128 in 8 parts 89.6, 16 parts 92.6; one pair x 32000 in 62 parts 20.5, 31 parts 23.8, 125 parts 20.1; one
// pair x 1000 of 1024 slots whole 9.1, of 1025 in 3 parts 9.5; 4 pairs 9.3 and 9.4.
int attention_step_splits(const tvl_attention_args& a) {
    const int64_t work = a.batch * a.kv_heads * ceil_div(a.queries * (a.heads / a.kv_heads), ROWS);
    const int64_t want = ceil_div(256, work), most = a.keys <= 1024 ? 1 : ceil_div(a.keys, 512);
    int64_t n = want < most ? want : most;
    n = n < MOST_PARTS ? n : MOST_PARTS;
    return (int)(n < 1 ? 1 : n);
}

size_t attention_step_bytes(const tvl_attention_args& a) {
    const int splits = attention_step_splits(a);
    // rows of the padded head dim whatever the form: the odd form pads to the largest
    return splits > 1 ? (size_t)a.batch * a.kv_heads * splits * (size_t)(a.queries * (a.heads / a.kv_heads)) * (ATTENTION_MAX_DIM + 2) * 4 : 0;
}

template <typename T, int DP, Form FORM>
static int launch_step(const tvl_attention_args& a, float* parts, hipStream_t st) {
    const int64_t rows = a.queries * (a.heads / a.kv_heads), pairs = a.batch * a.kv_heads;
    const int tiles = (int)ceil_div(rows, ROWS), splits = attention_step_splits(a);
    const size_t values = (size_t)WAVES * STEP * Tile<T, DP>::ROW, join = (size_t)WAVES * ROWS * (DP + 2) * 4, bytes = values > join ? values : join;
    if (bytes > 65536) TVL_HIP_CHECK(hipFuncSetAttribute((const void*)attention_step_kernel<T, DP, FORM>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    hipLaunchKernelGGL((attention_step_kernel<T, DP, FORM>), dim3((unsigned)(pairs * tiles * splits)), dim3(64 * WAVES), bytes, st, a, tiles, splits, parts);
    TVL_LAUNCH_CHECK();
    if (splits > 1) {
        hipLaunchKernelGGL((attention_join_kernel<T, DP>), dim3((unsigned)(pairs * rows)), dim3(256), 0, st, a, splits, parts);
        TVL_LAUNCH_CHECK();
    }
    return TVL_OK;
}

template <typename T>
static int launch_step_t(const tvl_attention_args& a, float* parts, hipStream_t st) {
    return with_form<T>(a, step_wide(a), [&](auto form) {
        constexpr Form FORM = decltype(form)::value;
        if constexpr (FORM == ODD) return launch_step<T, 128, ODD>(a, parts, st);
        else return a.dim <= 64 ? launch_step<T, 64, FORM>(a, parts, st) : launch_step<T, 128, FORM>(a, parts, st);
    });
}

int launch_attention_step(const tvl_attention_args& a, float* parts, hipStream_t st) {
    if (a.dtype == TVL_F32) return launch_step_t<float>(a, parts, st);
    if (a.dtype == TVL_F16) return launch_step_t<f16>(a, parts, st);
    return launch_step_t<bf16_t>(a, parts, st);
}

}  // namespace tvl
