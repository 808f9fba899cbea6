// Shared parts of the attention kernels: matrix-core fragments, tiles in LDS, what a query sees, scores.
//
// All products run on the matrix cores in R x R output tiles (R = 32: v_mfma_f32_32x32x16, R = 16: v_mfma_f32_16x16x32; float32
// operands: v_mfma_f32_32x32x2 / 16x16x4, eight of them in place of one 16-bit instruction).  Lane l of a wave is r = l % R, g = l / R:
//   an operand fragment is 8 elements of row r at 8 g .. 8 g + 7 of a chunk of K = 512 / R contracted elements;
//   register x of the result holds row 4 (64 / R) (x / 4) + 4 g + x % 4 of column r.
// A product's result therefore feeds the next product's second operand from the registers it is in, if the first operand
// lists the contracted elements in the same order: fragment element 4 u + y of chunk c is element K c + (K / 2) u + 4 g + y.  read_across() reads
// a tile of LDS in that order down its rows; the scores never leave the registers of the lanes that hold them.
#pragma once
#include "tvl_common.h"

#include <type_traits>

namespace tvl {

constexpr int ATTENTION_MAX_DIM = 128;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Operand;
template <> struct Operand<f16> { typedef f16x8 frag; typedef _Float16 elem; };
template <> struct Operand<bf16_t> { typedef bf16x8 frag; typedef __bf16 elem; };
template <> struct Operand<float> { typedef f32x8 frag; typedef float elem; };
template <typename T> using Frag = typename Operand<T>::frag;

template <int R> struct Result;
template <> struct Result<32> { typedef f32x16 type; };
template <> struct Result<16> { typedef f32x4 type; };
template <int R> using Acc = typename Result<R>::type;
template <int R> constexpr int REGS = R * R / 64;       // result registers of a lane
template <int R> constexpr int CHUNK = 512 / R;         // contracted elements of one fragment pair

__device__ __forceinline__ f32x16 mma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(f32x8 a, f32x8 b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
}

// row of result register x (of lane group g)
template <int R> __device__ __forceinline__ constexpr int result_row(int x, int g) { return 4 * (64 / R) * (x >> 2) + 4 * g + (x & 3); }

__device__ __forceinline__ bool not_finite(float v) { return (__builtin_bit_cast(uint32_t, v) & 0x7F800000u) == 0x7F800000u; }

// the fragment with zeros in place of infinities and NaN
template <typename T> __device__ __forceinline__ Frag<T> finite_part(Frag<T> a) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (not_finite((float)a[e])) a[e] = (typename Operand<T>::elem)0.0f;
    return a;
}

// ---- tiles in LDS ------------------------------------------------------------------------------
// Rows of DP elements in 16-byte units.  LDS has 64 banks of 4 bytes: 16 lanes of a b128 read, 32 lanes of a transposing b64 read, go together.  A
// unit lies at its place with its low bits exchanged by the row's, so that 16 rows at one place of a row, and 4 rows x 4 neighbouring
// units, all fall on different banks.  The exchange is an exclusive-or of bits of the row's number: a lane works out its offset
// once, and what the compiler knows (chunk, tile, half) is an exclusive-or or an immediate.
template <typename T, int DP> struct Tile {
    static constexpr int UNITS = DP * (int)sizeof(T) / 16;
    static constexpr int PER = 16 / (int)sizeof(T);          // elements of a unit
    static constexpr int ROW = DP * (int)sizeof(T);
    static constexpr int LOW = UNITS % 16 == 0 ? 15 : 7;     // unit bits that are exchanged
    static_assert(UNITS % 8 == 0, "rows are multiples of 128 bytes");
    // rows of 128 bytes: two fill the banks, so 8 pairs; longer rows: each fills them.  Products of 16 rows read two units of rows 4 apart together across, and
    // neighbouring units of rows 4 and 8 apart together along (a b128 read takes lanes 0..3, 12..15, 20..27 at a time): groups of four rows differ by 2, 3 and 1.
    // By 1, 2 and 3 dq and dk / dv of heads of 128 spent 45 % of their LDS cycles in conflicts (8192 x 16 heads, f16: backward 2710 us, now 2500).
    __device__ static __forceinline__ constexpr int swap_bits(int row) {
        return LOW == 7 ? ((row >> 1) & 1) << 2 | ((row >> 3) & 1) << 1 | ((row >> 2) & 1) : (row & 3) << 2 | (((row >> 2) ^ (row >> 3)) & 1) << 1 | ((row >> 3) & 1);
    }
    __device__ static __forceinline__ int at(int row, int unit) { return row * ROW + ((unit ^ swap_bits(row)) << 4); }
    // a lane's offset moved by `unit` units and `rows` rows (bits that the lane's own unit and row do not use)
    __device__ static __forceinline__ int moved(int lane_at, int unit, int rows) {
        return (lane_at ^ (((unit ^ swap_bits(rows)) & LOW) << 4)) + ((unit & ~LOW) << 4) + rows * ROW;
    }

    // fragments of row `row0 + r`, elements 8 (g + (64 / R) c) ..: a lane's offset, and the read  (row0 a multiple of 32)
    template <int R> __device__ static __forceinline__ int lane_row(int lane) { return at(lane % R, (lane / R) * (8 / PER)); }
    template <int R> __device__ static __forceinline__ Frag<T> read(const char* tile, int lane_at, int row0, int c) {
        if constexpr (sizeof(T) == 2) {
            return __builtin_bit_cast(Frag<T>, *reinterpret_cast<const u32x4*>(tile + moved(lane_at, 64 / R * c, 0) + row0 * ROW));
        } else {
            const f32x4 lo = *reinterpret_cast<const f32x4*>(tile + moved(lane_at, 128 / R * c, 0) + row0 * ROW);
            const f32x4 hi = *reinterpret_cast<const f32x4*>(tile + moved(lane_at, 128 / R * c + 1, 0) + row0 * ROW);
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }

    // fragments down the rows: element 4 u + y is row row0 + (K / 2) u + 4 g + y, column R d + r  (K = CHUNK<R>, row0 a multiple of 16)
    template <int R> __device__ static __forceinline__ int lane_column(int lane) {
        const int r = lane % R, g = lane / R, i = lane & 15;
        // ds_read_b64_tr_b16: 16 lanes point at 4 rows x 4 pieces of 4 elements and get the 16 columns
        if constexpr (sizeof(T) == 2) return at(4 * g + (i >> 2), ((r & ~15) >> 3) + ((i & 3) >> 1)) + 8 * (i & 1);
        return at(4 * g, r >> 2) + 4 * (r & 3);
    }
    template <int R> __device__ static __forceinline__ Frag<T> read_across(const char* tile, int lane_at, int row0, int d) {
        if constexpr (sizeof(T) == 2) {
            i16x4 v[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const char* p = tile + moved(lane_at, d * R / PER, CHUNK<R> / 2 * u) + row0 * ROW;
                v[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(p));
            }
            return __builtin_bit_cast(Frag<T>, __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            Frag<T> f;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int y = 0; y < 4; ++y)
                    f[4 * u + y] = *reinterpret_cast<const float*>(tile + moved(lane_at, d * R / PER, CHUNK<R> / 2 * u + y) + row0 * ROW);
            return f;
        }
    }
};

// A masked weight is zero, and zero times an infinity or NaN is NaN: where rows of a tile are seen by some columns of a wave's product and not by
// others, the wave looks for such rows first.  If there are any it multiplies the finite part of the tile and adds what is not finite to
// the columns that see it.
template <typename T, int DP, int ROWS> __device__ __forceinline__ bool holds_not_finite(const char* tile, int lane) {
    bool bad = false;
#pragma unroll
    for (int u = lane; u < ROWS * Tile<T, DP>::UNITS; u += 64) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(tile + 16 * u);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t w = v[e];
            if constexpr (sizeof(T) == 4) {
                bad |= (w & 0x7F800000u) == 0x7F800000u;
            } else {
                constexpr uint32_t EXP = __is_same(T, f16) ? 0x7C00u : 0x7F80u;
                bad |= (w & EXP) == EXP || (w & (EXP << 16)) == (EXP << 16);
            }
        }
    }
    return __any(bad);
}
// acc += the infinities and NaN of row `row`, where the lane's column sees it (`spoil`: NaN whatever the element is)
template <typename T, int DP, int R>
__device__ __forceinline__ void add_not_finite(const char* tile, int row, bool sees, bool spoil, int g, Acc<R>* acc) {
#pragma unroll
    for (int d = 0; d < DP / R; ++d)
#pragma unroll
        for (int x = 0; x < REGS<R>; ++x) {
            const int col = d * R + result_row<R>(x, g);
            constexpr int PER = Tile<T, DP>::PER;
            const float v = to_float(*reinterpret_cast<const T*>(tile + Tile<T, DP>::at(row, col / PER) + (int)sizeof(T) * (col % PER)));
            if (sees && not_finite(v)) acc[d][x] += spoil ? __builtin_nanf("") : v;
        }
}

// 16 bytes of a row of `dim` elements, zeros behind them; WIDE: rows are 16-byte aligned and dim a multiple of the unit
template <typename T, bool WIDE>
__device__ __forceinline__ u32x4 load_unit(const T* row, int unit, int dim) {
    constexpr int PER = 16 / (int)sizeof(T);
    u32x4 v = {0, 0, 0, 0};
    const int c = unit * PER;
    if constexpr (WIDE) {
        if (c < dim) v = *reinterpret_cast<const u32x4*>(row + c);
    } else {
        T e[PER] = {};
#pragma unroll
        for (int x = 0; x < PER; ++x)
            if (c + x < dim) e[x] = row[c + x];
        v = *reinterpret_cast<const u32x4*>(e);
    }
    return v;
}

// fragment of a row straight from global memory (elements 8 c8 ..)
template <typename T, bool WIDE>
__device__ __forceinline__ Frag<T> load_frag(const T* row, int c8, int dim) {
    if constexpr (sizeof(T) == 2) {
        return __builtin_bit_cast(Frag<T>, load_unit<T, WIDE>(row, c8, dim));
    } else {
        const f32x4 lo = __builtin_bit_cast(f32x4, load_unit<T, WIDE>(row, 2 * c8, dim)), hi = __builtin_bit_cast(f32x4, load_unit<T, WIDE>(row, 2 * c8 + 1, dim));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
}

// A tile's way from global memory to LDS through the registers of THREADS threads.  Offsets inside a tile are 32-bit bytes (wide_rows() sees to it for
// the wide forms), tiles lie at 64-bit places.
template <typename T, int DP, int ROWS, int THREADS, bool WIDE> struct Stage {
    typedef Tile<T, DP> L;
    static constexpr int N = ROWS * L::UNITS / THREADS, APART = THREADS / L::UNITS;
    static_assert(ROWS * L::UNITS % THREADS == 0 && THREADS % L::UNITS == 0 && APART % 8 == 0 && (APART % 16 == 0 || APART == 8), "every thread moves the same unit of rows APART apart");
    u32x4 v[N];
    // rows row0 .. row0 + ROWS - 1 of a matrix; rows from `end` on are zero and not read.  One 32-bit offset per lane, the rest is in scalar
    // registers: per-row offsets get spilled, and a reload waits for the loads in front of it
    __device__ __forceinline__ void load(const T* base, int64_t stride, int row0, int end, int dim) {
        const int row = threadIdx.x / L::UNITS, unit = threadIdx.x % L::UNITS;
        const T* tile = base + (int64_t)row0 * stride;
#pragma unroll
        for (int x = 0; x < N; ++x) v[x] = u32x4{0, 0, 0, 0};
        if constexpr (WIDE) {
            const uint32_t at = (uint32_t)row * (uint32_t)(stride * (int64_t)sizeof(T)) + 16u * unit;
            if (unit * L::PER >= dim) return;
            if (row0 + ROWS <= end) {
#pragma unroll
                for (int x = 0; x < N; ++x) v[x] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(tile + (int64_t)(x * APART) * stride) + at);
            } else {
#pragma unroll
                for (int x = 0; x < N; ++x)
                    if (row0 + x * APART + row < end) v[x] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(tile + (int64_t)(x * APART) * stride) + at);
            }
        } else {
#pragma unroll
            for (int x = 0; x < N; ++x)
                if (row0 + row + x * APART < end) v[x] = load_unit<T, false>(tile + (int64_t)(row + x * APART) * stride, unit, dim);
        }
    }
    __device__ __forceinline__ void store(char* tile) const {
        const int at = L::at(threadIdx.x / L::UNITS, threadIdx.x % L::UNITS);
#pragma unroll
        for (int x = 0; x < N; ++x) *reinterpret_cast<u32x4*>(tile + L::moved(at, 0, x * APART)) = v[x];
    }
};

// the values of lanes l % 32 and l % 32 + 32: v_permlane32_swap exchanges the halves of two registers
__device__ __forceinline__ void both_halves(float v, float& lo, float& hi) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t x = a[0], y = a[1];
    lo = __builtin_bit_cast(float, x);
    hi = __builtin_bit_cast(float, y);
}
// the wave's number in its workgroup, known to be the same for all its lanes
__device__ __forceinline__ int wave_number() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64); }

// whether a token is of document `doc` (none if negative): its document is staged beside its tile in LDS
__device__ __forceinline__ bool same_document(const int64_t* staged, int64_t doc) { return (*staged == doc) & (doc >= 0); }

// maximum / sum over the lanes that hold one column (the groups g)
template <int R> __device__ __forceinline__ float column_max(float v) {
    float lo, hi;
    both_halves(v, lo, hi);
    v = fmaxf(lo, hi);
    if constexpr (R == 16) v = fmaxf(v, __shfl_xor(v, 16));
    return v;
}
template <int R> __device__ __forceinline__ float column_sum(float v) {
    float lo, hi;
    both_halves(v, lo, hi);
    v = lo + hi;
    if constexpr (R == 16) v = v + __shfl_xor(v, 16);
    return v;
}

// Forms of a kernel.  PLAIN: wide rows, no cap, no bias, no documents.  GENERAL: wide rows, all of them.  CAP_FAR: the same for 16-bit operands under a cap
// above SHORT_CAP.  ODD: any rows.  (Both ways to cap in one form
// spill more: 8192 causal tokens, 16 / 4 heads of 128, bf16, forward, capped at 50, 731 us against 543; capped at 65 758.)
enum Form { PLAIN, GENERAL, CAP_FAR, ODD };

// ---- what a query sees, and its scores ---------------------------------------------------------

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// x = tanh(x) for N scores divided by the cap.  float32: the library's.  16-bit operands: 1 - 2 / (e^2x + 1) from one hardware
// exponential and reciprocal, off by 2^-21 at most wherever x lies; times a cap of up to 64 that is 2^-15 of a power of e, a sixteenth of the
// rounding of a float16 weight.  Larger caps meet scores that are small beside them, where only a relative error is small enough:
// (1 - e) / (1 + e) with e = exp(-2 |x|) from 1 on, and below it the continued fraction x / (1 + x^2 / (3 + x^2 / (5 + x^2 / (7 + x^2 / 9)))), 2^-24 off
// at 1.
constexpr float SHORT_CAP = 64.0f;
template <typename T, Form FORM, int N, typename V> __device__ __forceinline__ void cap_tanh(V& x, float cap) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = tanhf(x[i]);
    } else if (FORM == GENERAL || (FORM == ODD && cap <= SHORT_CAP)) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = 1.0f - 2.0f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x[i] * (2.0f * LOG2E)) + 1.0f);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float a = fabsf(x[i]), y = a * a, e = __builtin_amdgcn_exp2f(a * (-2.0f * LOG2E));
            const bool low = a < 1.0f;
            const float above = low ? a * __builtin_fmaf(y, y + 105.0f, 945.0f) : 1.0f - e, below = low ? __builtin_fmaf(y, __builtin_fmaf(15.0f, y, 420.0f), 945.0f) : 1.0f + e;
            x[i] = copysignf(above * __builtin_amdgcn_rcpf(below), x[i]);
        }
    }
}

// float16 holds 2^15 and no digits below 2^-25: softmax weights rounded to it are formed 2^LIFT times as large, so that a long row's many small ones,
// which the float32 sum counts, count in the products too.  In the forward pass the largest weight of a row then lies in [2^7, 2^15] (its
// running maximum may lag by 2^8) and a weight is off by at most 2^-32 of it; the backward pass lifts weights relative to their sum, at most 1 but for the
// log-sum's rounding.  The other types have float32's range.
template <typename T> constexpr float LIFT = __is_same(T, f16) ? 7.0f : 0.0f;
template <typename T> constexpr float BACKWARD_LIFT = __is_same(T, f16) ? 12.0f : 0.0f;

// a product that is rounded to float32 before anything else happens to it: never part of a fused or mixed-precision instruction, so the same bits
// in every form of a kernel
__device__ __forceinline__ float product(float x, float y) {
#pragma clang fp contract(off)
    return x * y;
}

// Sequence b of a call.  Places and limits fit 32 bits: tokens are at most 2^30.
struct Sequence {
    int real;          // queries that are real
    int end;           // keys that exist
    int shift;         // place of query 0 among the keys
    int prefix;
    bool causal;
    // query i sees keys j < limit(i)
    __device__ __forceinline__ int limit(int i) const {
        int v = end;
        if (causal) {
            const int p = i + shift + 1, q = p > prefix ? p : prefix;
            v = q < end ? q : end;
        }
        return v < 0 ? 0 : v;
    }
};

template <bool CACHED>
__device__ __forceinline__ Sequence sequence_of(const tvl_attention_args& a, int b, bool& lost) {
    Sequence s;
    const int64_t p = a.prefix ? a.prefix[b] : a.prefix_value;
    s.prefix = (int)(p < 0 ? 0 : (p < a.keys ? p : a.keys));
    lost = false;
    if constexpr (CACHED) {
        const int64_t before = a.cache_len ? a.cache_len[b * a.cache_len_stride] : a.cache_len_value;
        const int64_t n = a.count ? a.count[b] : a.queries;
        s.real = (int)(n < 0 ? 0 : (n < a.queries ? n : a.queries));
        s.causal = true;
        lost = before < 0 || before >= a.keys;                   // no query of this sequence has a slot
        s.shift = lost ? (int)a.keys : (int)before;              // query i's slot is shift + i: outside from a.keys on
        const int64_t e = (int64_t)s.shift + s.real;
        s.end = lost ? 0 : (int)(e < a.keys ? e : a.keys);
    } else {
        s.real = (int)a.queries;
        s.causal = a.causal != 0;
        s.shift = (int)(a.keys - a.queries);
        s.end = (int)a.keys;
    }
    return s;
}

// smallest and largest document of every block of 64 tokens, without the padding (lo > hi: nothing but padding), and whether there is none:
// blocks that cannot meet are skipped, blocks of one document need no test
struct DocumentSpan { int64_t lo, hi, whole; };
constexpr int SPAN = 64;

// The documents of 64 blocks of tokens against those of a workgroup's own tokens [lo, hi], as two bit masks that stay in scalar registers:
// blocks that cannot meet them, and blocks that hold the one document they all are: one trip to memory per 4096 tokens.
struct DocumentWindow {
    const DocumentSpan* spans;
    int blocks, window;
    int64_t lo, hi;
    bool whole;
    uint64_t skip, single;
    __device__ __forceinline__ void start(const DocumentSpan* s, int tokens, int first, int rows) {
        spans = s;
        blocks = (tokens + SPAN - 1) / SPAN;
        window = -1;
        lo = INT64_MAX;
        hi = -1;
        whole = true;
        for (int i = first / SPAN; i < blocks && i * SPAN < first + rows; ++i) {
            lo = s[i].lo < lo ? s[i].lo : lo;
            hi = s[i].hi > hi ? s[i].hi : hi;
            whole = whole && s[i].whole;
        }
    }
    __device__ __forceinline__ void look(int block, int lane) {
        if (block / 64 == window) return;
        window = block / 64;
        DocumentSpan s{INT64_MAX, -1, 0};
        if (window * 64 + lane < blocks) s = spans[window * 64 + lane];
        skip = __ballot(s.hi < lo || s.lo > hi);
        single = __ballot(s.whole && whole && s.lo == s.hi && lo == hi && s.lo == lo);
    }
    // first block from `block` on, below `end`, that is not skipped
    __device__ __forceinline__ int next(int block, int end, int lane) {
        while (block < end) {
            look(block, lane);
            const uint64_t rest = ~skip >> (block & 63);
            if (rest != 0) return block + __builtin_ctzll(rest);
            block = (block / 64 + 1) * 64;
        }
        return block;
    }
    __device__ __forceinline__ bool one(int block, int lane) {
        look(block, lane);
        return (single >> (block & 63)) & 1;
    }
};

// Sequence and head of a workgroup.  Workgroups with equal blockIdx % 8 share an L2 (8 XCDs): where the (sequence, key head) pairs divide by 8,
// each pair's query tiles and heads stay on one of them, so its keys and values are fetched into one L2.  Tiles come last first: with a
// causal mask those are the long ones; few pairs take turns, so that all their long tiles start first.
struct Place { int pair, head, tile; };
__device__ __forceinline__ Place place_of(uint32_t id, int pairs, int group, int tiles) {
    const uint32_t per = (uint32_t)group * tiles;
    uint32_t pair, rest;
    if (pairs % 8 == 0) {
        const uint32_t local = id >> 3;
        pair = (local / per) * 8 + (id & 7);
        rest = local % per;
    } else {
        pair = id % (uint32_t)pairs;
        rest = id / (uint32_t)pairs;
    }
    return Place{(int)pair, (int)(rest % group), tiles - 1 - (int)(rest / group)};
}

// host side
static inline bool featureless(const tvl_attention_args& a) { return a.softcap == 0.0f && a.slopes == nullptr && a.documents == nullptr && a.scale != 0.0f; }
// launch(form) for the call, the form as a compile-time value
template <typename T, typename F> static inline int with_form(const tvl_attention_args& a, bool wide, F launch) {
    if (!wide) return launch(std::integral_constant<Form, ODD>{});
    if (featureless(a)) return launch(std::integral_constant<Form, PLAIN>{});
    if constexpr (sizeof(T) == 2)
        if (a.softcap > SHORT_CAP) return launch(std::integral_constant<Form, CAP_FAR>{});
    return launch(std::integral_constant<Form, GENERAL>{});
}
static inline bool wide_rows(const void* p, int64_t dim, int64_t batch, int64_t token, int64_t head, size_t z) {
    const int64_t per = (int64_t)(16 / z);
    return aligned(p, 16) && dim % per == 0 && batch % per == 0 && token % per == 0 && head % per == 0 && token * (int64_t)z < (int64_t)1 << 25;
}

int launch_attention_forward(const tvl_attention_args& a, bool cached, const DocumentSpan* spans, hipStream_t st);
int launch_attention_backward(const tvl_attention_args& a, const tvl_attention_grads& g, const DocumentSpan* spans, float* delta, float* slabs, hipStream_t st);
int attention_backward_parts(const tvl_attention_args& a);
bool attention_step_serves(const tvl_attention_args& a);
size_t attention_step_bytes(const tvl_attention_args& a);
int launch_attention_step(const tvl_attention_args& a, float* parts, hipStream_t st);
int launch_document_spans(const tvl_attention_args& a, DocumentSpan* spans, hipStream_t st);

}  // namespace tvl
