// libstag_train.so: C ABI (include/stag_train.h) and kernels of the operators that learn node classifiers.
// gfx950 only; no CPU fallback.
#include "stag_train.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <type_traits>

namespace {

thread_local char g_err[512];

int fail(int code, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof g_err, fmt, ap);
    va_end(ap);
    return code;
}

#define HIP_TRY(expr)                                                                                          \
    do {                                                                                                       \
        hipError_t e_ = (expr);                                                                                \
        if (e_ != hipSuccess) return fail(STAG_E_HIP, "%s: %s (%s:%d)", #expr, hipGetErrorString(e_), __FILE__, __LINE__); \
    } while (0)

#define REQUIRE(cond, ...)                                        \
    do {                                                          \
        if (!(cond)) return fail(STAG_E_INVALID, __VA_ARGS__);    \
    } while (0)

typedef _Float16 f16;
typedef __bf16 bf16;

int type_bytes(int type) { return type == STAG_F32 ? 4 : 2; }
bool type_known(int type) { return type == STAG_F32 || type == STAG_BF16 || type == STAG_F16; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned(const void *p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

// the packed row of batch position i: its words, or null for padding
__device__ __forceinline__ const uint32_t *row_of(const uint32_t *bits, int64_t n, int64_t row_stride, const int32_t *rows, int64_t i) {
    const int64_t r = rows ? (int64_t)rows[i] : i;
    return r >= 0 && r < n ? bits + r * row_stride : nullptr;
}

// ------------------------------------------------------------------------------------------------------------------
// scores and their gradient
// ------------------------------------------------------------------------------------------------------------------
// Both are products of a matrix of zeros and ones, held as bits, with a matrix of coefficients or gradients:
//   scores  S[i][c] = sum_f x[i][f] T[f][c]        rows of the result: batch rows,  summed over: features
//   grad    D[f][c] = sum_i x[i][f] G[i][c]        rows of the result: features,    summed over: batch rows
// and run on the matrix cores although four of five bits are 0: 1,500 additions a score fed from LDS or L2 one by one take longer than
// 7,500 multiply-adds at the matrix cores' rate.  A bit becomes a 16-bit operand by one shift and one mask: bit 14 alone is 2.0, in bf16
// and in f16, and a mask of two such bits makes a pair; the factor 2 is taken out of the result.  A zero or one is exact
// in 16 bits; a 32-bit coefficient is cut into three bf16 pieces of 8 bits each, which together are the coefficient (to 2^-133, the
// smallest step of bf16: below 2^-110 that is less than 24 bits), and multiplied piece by piece into the same 32-bit sums.  16-bit
// coefficients go in as they are.
//
// What bounds them: the matrix cores for 32-bit coefficients (8,192 rows x 7,500 features x 1,000 columns: 218 us, 1.7 PFLOP/s of bf16
// operations counted densely; a library's bf16 product of 8,192^3 reaches 1.19 on the same card), the making of operands
// beside them for 16-bit ones (that size's gradient in bf16: 105 us, 1.2 PFLOP/s), latency for one node's batch (4,096 x
// 7,500 x 13: 10 us and 3 for adding up its parts).
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
typedef __attribute__((ext_vector_type(4))) float f32x4;

struct ProductArgs {
    const uint32_t *bits;
    int64_t n, row_stride;
    const int32_t *rows;
    int64_t m;
    const void *mat;            // table or gradient
    int64_t mat_stride;
    const float *bias;          // scores: added
    float *out, *bias_out;      // bias_out: grad: column sums
    int64_t out_stride;
    const uint32_t *turned;     // TURNED: the bits by feature, see k_turn
    float *part;                // more than one part: their sums [parts][result rows][k], then column sums [parts][k]
    int32_t n_features, words, k;       // words of a row of bits (TURNED: of a turned row)
    int32_t row_blocks, col_blocks, parts;
    int32_t steps, steps_per_part;      // in units of 4 K-steps (TURN: of 1)
    float scale;
};

template <int TYPE> struct Raw { typedef uint16_t type; };
template <> struct Raw<STAG_F32> { typedef uint32_t type; };

template <int TYPE> __device__ __forceinline__ bool not_finite(uint32_t raw) {
    constexpr uint32_t ONES = TYPE == STAG_F32 ? 0x7f800000u : TYPE == STAG_BF16 ? 0x7f80u : 0x7c00u;
    return (raw & ONES) == ONES;
}
template <int TYPE> __device__ __forceinline__ float value_of(uint32_t raw) {
    return TYPE == STAG_F32 ? __uint_as_float(raw) : TYPE == STAG_BF16 ? __uint_as_float(raw << 16) : (float)__builtin_bit_cast(f16, (uint16_t)raw);
}

// A buffer of up to 2^31 - 1 bytes: loads behind its end give zero, stores there are dropped.
constexpr uint32_t NOWHERE = 0x80000000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void *p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, (int)(bytes < 0 ? 0 : bytes > 0x7fffffff ? 0x7fffffff : bytes), 0x00020000);
}
template <typename raw_t> __device__ __forceinline__ uint32_t load_raw(__amdgpu_buffer_rsrc_t from, uint32_t at) {
    if constexpr (sizeof(raw_t) == 4)
        return __builtin_amdgcn_raw_buffer_load_b32(from, at, 0, 0);
    else
        return __builtin_amdgcn_raw_buffer_load_b16(from, at, 0, 0);
}

__device__ __forceinline__ uint32_t low_halves(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x05040100u); }
__device__ __forceinline__ uint32_t high_halves(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }

// the 8 operands of K-step part s: bits 4s .. 4s+3 and 4s+16 .. 4s+19 of x, as 2.0 or 0
__device__ __forceinline__ u32x4 operands(uint32_t x, int s) {
    u32x4 a;
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = __builtin_amdgcn_alignbit(x, x, (4 * s + j + 18) & 31) & 0x40004000u;
    return a;
}

// 32 x 32 bits in each half of the wave: lane r held row r, lane f comes to hold column f (bit r = row r)
__device__ __forceinline__ uint32_t transposed(uint32_t x, int lane) {
#define STAG_EXCHANGE(J, LOW)                                                                    \
    {                                                                                            \
        const uint32_t y = (uint32_t)__builtin_amdgcn_ds_swizzle((int)x, (J) << 10 | 0x1f);      \
        const uint32_t keep = lane & (J) ? ~(LOW) : (LOW);                                       \
        const uint32_t z = __builtin_amdgcn_alignbit(y, y, lane & (J) ? (J) : 32 - (J));         \
        x = (x & keep) | (z & ~keep);                                                            \
    }
    STAG_EXCHANGE(16, 0x0000ffffu)
    STAG_EXCHANGE(8, 0x00ff00ffu)
    STAG_EXCHANGE(4, 0x0f0f0f0fu)
    STAG_EXCHANGE(2, 0x33333333u)
    STAG_EXCHANGE(1, 0x55555555u)
#undef STAG_EXCHANGE
    return x;
}

// Where the bits of a result row come from: ROWS: a batch row (scores); TURN: a feature, whose bits in 64 batch rows the wave
// turns out of their packed rows as it goes; TURNED: a feature, from bits that k_turn has laid out by feature before.
enum Source { ROWS, TURN, TURNED };

typedef const uint32_t __attribute__((address_space(4))) *const_words;      // read through the scalar cache

constexpr int W = 8;      // waves of a workgroup
constexpr int NOTES = 1024;      // words of the notes of k_product

// A workgroup of W waves makes W MT x 32 rows of the result by NT x 32 columns; a wave its own MT row tiles.  A K-step
// is 64 terms of the sum: two words of bits, one for each half of the wave (the matrix instruction takes 8 terms from
// each half), in four instructions of 16 terms.  The workgroup loads the coefficients of U K-steps, 64 U x 32 NT, cuts them into pieces
// and stores them to LDS in operand order; the next ones are in flight while the matrix cores work on these.
//
// Why these tiles: 2 x 2 tiles a wave make 8 (or 24) matrix instructions of the 4 (or 6) operands loaded from LDS and two made
// from bits, and 8 waves share what the workgroup cuts, at two waves a SIMD (150 to 190 registers).  Measured at the level's size, scores in
// 32 bits and gradient in bf16, in us: 4 waves of 4 x 2 tiles with the sum in two parts 273 and 157; 8 of 2 x 2, one K-step a barrier 290
// and 164, two 275 and 142, four 260 and 135.  Then: operands, bits and loads in turns with the matrix instructions (in_turns) and WIDE
// loads 242 -> 222 and 121 -> 108; what is left of it without the coefficients' way into LDS is 199 and 94.  Two buffers in LDS and one
// barrier, with half of the waves cutting coefficients while the others multiply: 235 and 113, the matrix cores then run slower.
// One tile a wave where there are few.
//
// WIDE: rows of coefficients that all begin at a multiple of 16 bytes (32-bit ones) or 8 are loaded four columns at a time.
template <int TYPE, Source SRC, int MT, int NT, bool WIDE>
__global__ __launch_bounds__(64 * W, 2) void k_product(ProductArgs a) {
    typedef typename Raw<TYPE>::type raw_t;
    constexpr bool GRAD = SRC != ROWS;
    constexpr int P = TYPE == STAG_F32 ? 3 : 1, COLS = 32 * NT, U = SRC == TURN ? 2 : 4;
    // a thread's share of the 8 x COLS groups of 8 terms of U K-steps; PASSES of them are of one K-step
    constexpr int ITEMS = U * 8 * COLS / (64 * W), PASSES = 8 * COLS > 64 * W ? 8 * COLS / (64 * W) : 1;
    static_assert(ITEMS >= 1 && (!WIDE || ITEMS == 4), "a group for every thread, or one of four columns");
    constexpr int QUADS = COLS / 4, SUMS = WIDE ? 4 : 1;
    typedef __attribute__((ext_vector_type(MT))) uint32_t words_t;          // TURN: a lane loads the words of its wave's row tiles at once
    __shared__ u32x4 lds[U][P][8][COLS];
    __shared__ float sums[GRAD ? 64 * W * SUMS : 1];
    __shared__ uint32_t note[NOTES];
    __shared__ int met, bad;
    // Workgroups go round the card's 8 dies in turn; each die is given neighbours in row blocks of the same columns and terms, which share the
    // coefficients in its L2 (HBM reads of the level's scores 248 -> 85 MB, of its gradient 193 -> 85; 221 -> 218 and 107.5 -> 104.7 us).
    const int per_die = gridDim.x / 8, tile = (int)(blockIdx.x % 8) * per_die + (int)(blockIdx.x / 8);
    if (tile >= a.row_blocks * a.col_blocks * a.parts) return;
    const int block_x = tile % a.row_blocks, block_y = tile / a.row_blocks % a.col_blocks, block_z = tile / a.row_blocks / a.col_blocks;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int64_t tile0 = ((int64_t)block_x * W + wave) * MT;           // this wave's first row tile
    const int64_t out_rows = GRAD ? a.n_features : a.m;
    const int col = WIDE ? 4 * (threadIdx.x % QUADS) : threadIdx.x % COLS, c0 = block_y * COLS, c = c0 + col;
    const bool c_ok = c < a.k;
    const int64_t limit = GRAD ? a.m : a.n_features;                       // terms of the sum
    constexpr int UNIT = SRC == TURN ? 1 : 4;                              // K-steps of a step of the plan
    const int first = block_z * a.steps_per_part * UNIT, last = min((int)(block_z + 1) * a.steps_per_part, a.steps) * UNIT;
    uint32_t padding[MT] = {}, any_padding = 0;                             // ROWS: which rows of a tile are padding

    // the term that stands at place r (0..63) of K-step ks
    auto term = [&](int ks, int r) -> int64_t {
        if constexpr (GRAD) return (int64_t)ks * 64 + r;
        return 32 * ((int64_t)(ks >> 2) * 8 + (r >> 5) * 4 + (ks & 3)) + (r & 31);
    };

    f32x16 acc[MT][NT];
    float column_sum[SUMS];
    // An infinity or NaN that met a zero bit has made NaN of a sum that it has no part in.  If a sum is not finite after the first
    // sweep, a second one takes such coefficients for zeros and notes the groups of U K-steps that have them (a bit for one group, or for 2, 4, 8 ..
    // of sums that are very long); afterwards it is found out there which sums have them.
    if (threadIdx.x == 0) met = bad = 0;
    int note_shift = 0;

    // Buffer loads: one 32-bit offset a lane, and what lies behind the last term or column reads as zero.  A thread's items: its
    // column in ITEMS groups of terms, or (WIDE) four columns in one group, as they lie in memory.
    constexpr int WORDS = WIDE && TYPE != STAG_F32 ? 2 : 4;
    uint32_t b[WIDE ? 8 : ITEMS][WIDE ? WORDS : 8];
    auto step_of = [&](int i) { return WIDE ? wave * 64 / (8 * QUADS) : PASSES * 64 * W == 8 * COLS ? i / PASSES : (i * 64 * W + wave * 64) / (8 * COLS); };      // the same for a whole wave
    auto group_of = [&](int i) -> int { return WIDE ? threadIdx.x % (8 * QUADS) / QUADS : (i * 64 * W + threadIdx.x) % (8 * COLS) / COLS; };
    uint32_t at_b[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int g = group_of(i), r0 = 4 * (g >> 1) + (g & 1) * (GRAD ? 32 : 128);
        at_b[i] = c_ok ? (uint32_t)((r0 * (int)a.mat_stride + c) * (int)sizeof(raw_t)) : NOWHERE;
    }
    const uint32_t row_b = (uint32_t)a.mat_stride * sizeof(raw_t);
    auto load_b = [&](int ks, bool there = true) {
#pragma unroll
        for (int i = 0; i < (WIDE ? 1 : ITEMS); ++i) {
            const int64_t t0 = term(ks + step_of(i), 0);
            const auto from = buffer((const raw_t *)a.mat + t0 * a.mat_stride, there ? (limit - t0) * row_b : 0);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const uint32_t at = at_b[i % PASSES] + ((q >> 1) + 16 * (q & 1)) * row_b;
                if constexpr (!WIDE) {
                    b[i][q] = load_raw<raw_t>(from, at);
                } else if constexpr (TYPE == STAG_F32) {
                    const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(from, at, 0, 0);
                    b[q][0] = v[0], b[q][1] = v[1], b[q][2] = v[2], b[q][3] = v[3];
                } else {
                    const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(from, at, 0, 0);
                    b[q][0] = v[0], b[q][1] = v[1];
                }
            }
        }
    };
    // term q of item i, as its type's bits
    auto raw_of = [&](int i, int q) -> uint32_t {
        if constexpr (!WIDE) return b[i][q];
        if constexpr (TYPE == STAG_F32) return b[q][i];
        return i & 1 ? b[q][i >> 1] >> 16 : b[q][i >> 1] & 0xffffu;
    };
    auto clear = [&](int i, int q) {
        if constexpr (!WIDE)
            b[i][q] = 0;
        else if constexpr (TYPE == STAG_F32)
            b[q][i] = 0;
        else
            b[q][i >> 1] &= i & 1 ? 0xffffu : 0xffff0000u;
    };
    // Where a column's operands lie among the COLS of LDS: turned a little, so that neither four columns a thread nor one meet in a bank
    auto place = [](int col) { return (col & ~7) | ((col + (col >> 3)) & 7); };
    // `real_at`: which of a K-step's rows are no padding (GRAD); the others are zeros, whatever the memory holds
    auto store_b = [&](auto careful, auto real_at) {
        if constexpr (WIDE && GRAD) {
            const uint64_t real = a.rows ? real_at(0) : ~0ull;
            if (real != ~0ull) {
                const uint32_t there = (uint32_t)(real >> (32 * (group_of(0) & 1) + 4 * (group_of(0) >> 1)));
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (!(there >> ((q >> 1) + 16 * (q & 1)) & 1u)) {
#pragma unroll
                        for (int j = 0; j < WORDS; ++j) b[q][j] = 0;
                    }
            }
        }
        if constexpr (WIDE) {
            if (c + 4 > a.k) {      // what lies behind the last column
#pragma unroll
                for (int i = 1; i < ITEMS; ++i)
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        if (c + i >= a.k) clear(i, q);
            }
        }
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int u = step_of(i), g = group_of(i);
            if constexpr (GRAD && !WIDE) {
                const uint64_t real = SRC == TURN || a.rows ? real_at(u) : ~0ull;      // TURN: a part may end inside the U K-steps
                if (real != ~0ull) {
                    const uint32_t there = (uint32_t)(real >> (32 * (g & 1) + 4 * (g >> 1)));
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        if (!(there >> ((q >> 1) + 16 * (q & 1)) & 1u)) clear(i, q);
                }
            }
            if constexpr (GRAD) {
                if (block_x == 0) {
                    float s = 0.f;
#pragma unroll
                    for (int q = 0; q < 8; ++q) s += value_of<TYPE>(raw_of(i, q));
                    column_sum[WIDE ? i : 0] += s;
                }
            }
            if constexpr (careful.value) {
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (not_finite<TYPE>(raw_of(i, q))) {
                        met = 1;
                        clear(i, q);
                    }
            }
            const int to = place(WIDE ? col + i : col);
            if constexpr (TYPE == STAG_F32) {
                uint32_t v[8], y[8], z[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    v[q] = raw_of(i, q);
                    const float left = __uint_as_float(v[q]) - __uint_as_float(v[q] & 0xffff0000u);        // exact: the low 16 bits
                    y[q] = __float_as_uint(left);
                    z[q] = __float_as_uint(left - __uint_as_float(y[q] & 0xffff0000u));                    // exact: the low 8 bits
                }
                u32x4 p0, p1, p2;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    p0[j] = high_halves(v[2 * j], v[2 * j + 1]);
                    p1[j] = high_halves(y[2 * j], y[2 * j + 1]);
                    p2[j] = high_halves(z[2 * j], z[2 * j + 1]);
                }
                lds[u][0][g][to] = p0;
                lds[u][P > 1 ? 1 : 0][g][to] = p1;
                lds[u][P > 2 ? 2 : 0][g][to] = p2;
            } else {
                u32x4 p0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (WIDE) {
                        const uint32_t lo = b[2 * j][i >> 1], hi = b[2 * j + 1][i >> 1];
                        p0[j] = i & 1 ? high_halves(lo, hi) : low_halves(lo, hi);
                    } else {
                        // Kept in registers of their own up to here: a load into the upper half of one that another load is to fill waits
                        // for that load, and 32 loads one after the other took 236 us where these take 130.
                        asm("" : "+v"(b[i][2 * j]), "+v"(b[i][2 * j + 1]));
                        p0[j] = b[i][2 * j] | b[i][2 * j + 1] << 16;
                    }
                }
                lds[u][0][g][to] = p0;
            }
        }
    };
    int operand_at[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) operand_at[n] = place(32 * n + (lane & 31));
    auto multiply = [&](int u, const uint32_t *x) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            u32x4 w[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) w[t] = operands(x[t], s);
#pragma unroll
            for (int p = P - 1; p >= 0; --p)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const u32x4 v = lds[u][p][2 * s + half][operand_at[n]];
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        if constexpr (TYPE == STAG_F16)
                            acc[t][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, w[t]), __builtin_bit_cast(f16x8, v), acc[t][n], 0, 0, 0);
                        else
                            acc[t][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, w[t]), __builtin_bit_cast(bf16x8, v), acc[t][n], 0, 0, 0);
                    }
                }
        }
    };

    // The order that keeps the matrix cores fed: operands leave LDS AHEAD turns before their own, those of the bits are made and
    // the next coefficients asked for in between.  Left to itself the compiler loads an operand where it is needed and waits.
    auto in_turns = [&] {
        constexpr int READS = U * 4 * P * NT, AHEAD = P == 1 ? 2 : 3;
        __builtin_amdgcn_sched_group_barrier(0x2, 8 * MT, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
        for (int r = 0; r < READS; ++r) {
            __builtin_amdgcn_sched_group_barrier(0x8, MT, 0);
            if (r < READS - AHEAD) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x2, (8 * MT + P * NT - 1) / (P * NT) + 1, 0);
            if (r % 3 == 0) __builtin_amdgcn_sched_group_barrier(0x20, 1, 0);
        }
    };

    auto sweep = [&](auto careful) -> bool {
#pragma unroll
        for (int i = 0; i < SUMS; ++i) column_sum[i] = 0.f;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[t][n] = (f32x16)(0.f);
        if constexpr (SRC != TURN) {
            const uint32_t *row[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const int64_t i = (tile0 + t) * 32 + (lane & 31);
                if constexpr (SRC == ROWS) {
                    row[t] = i < a.m ? row_of(a.bits, a.n, a.row_stride, a.rows, i) : nullptr;
                    padding[t] = (uint32_t)__ballot(row[t] == nullptr);
                    any_padding |= padding[t];
                } else {
                    row[t] = i < out_rows ? a.turned + i * a.words : nullptr;
                }
            }
            const auto valid = (const_words)(uintptr_t)(SRC == TURNED ? a.turned + out_rows * a.words : nullptr);
            auto load_x = [&](int sb, u32x4 *x) {
                const int w = sb * 8 + half * 4;
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    x[t] = (u32x4)(0u);
                    if (row[t] && w < a.words) x[t] = *(const u32x4 *)(row[t] + w);
                }
            };
            uint32_t real[8];                                                   // TURNED: which of the U K-steps' rows are no padding
            auto load_real = [&](int sb) {
                if constexpr (SRC == TURNED) {
#pragma unroll
                    for (int q = 0; q < (WIDE ? 2 : 8); ++q) real[q] = valid[sb * 8 + (WIDE ? 4 * q + step_of(0) : q)];
                }
            };
            auto real_at = [&](int u) -> uint64_t {
                if constexpr (SRC != TURNED) return ~0ull;
                uint32_t lo = real[0], hi = real[WIDE ? 1 : 4];
#pragma unroll
                for (int i = 1; i < (WIDE ? 1 : U); ++i) lo = u == i ? real[i] : lo, hi = u == i ? real[4 + i] : hi;
                return (uint32_t)__builtin_amdgcn_readfirstlane(lo) | (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane(hi) << 32;
            };
            u32x4 x[MT], next[MT];
            load_b(first);
            load_x(first >> 2, x);
            load_real(first >> 2);
#pragma unroll 1
            for (int ks = first; ks < last; ks += U) {
                const bool more = ks + U < last;
                store_b(careful, real_at);
                __syncthreads();
                if (careful.value && threadIdx.x == 0 && met) {
                    const int at = ((ks - first) / U) >> note_shift;
                    note[at >> 5] |= 1u << (at & 31);
                    met = 0;
                }
                if (more) {
                    load_x((ks + U) >> 2, next);
                    load_real((ks + U) >> 2);
                }
                load_b(ks + U, more);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    uint32_t w[MT];
#pragma unroll
                    for (int t = 0; t < MT; ++t) w[t] = x[t][u];
                    multiply(u, w);
                }
                in_turns();
                __syncthreads();
#pragma unroll
                for (int t = 0; t < MT; ++t) x[t] = next[t];
            }
        } else {
            const int64_t w0 = tile0 < a.words ? tile0 : a.words - MT;
            const uint32_t *row[U];
            words_t x[U];
            uint64_t real[U];
            auto load_row = [&](int u, int ks) {
                const int64_t i = (int64_t)ks * 64 + lane;
                row[u] = ks < last && i < a.m ? row_of(a.bits, a.n, a.row_stride, a.rows, i) : nullptr;
            };
            auto load_x = [&](int u) {
                real[u] = __ballot(row[u] != nullptr);
                x[u] = row[u] ? *(const words_t *)(row[u] + w0) : (words_t)(0u);
            };
            auto real_at = [&](int u) {
                uint64_t r = real[0];
#pragma unroll
                for (int i = 1; i < U; ++i) r = u == i ? real[i] : r;
                return r;
            };
#pragma unroll
            for (int u = 0; u < U; ++u) load_row(u, first + u);
            load_b(first);
#pragma unroll
            for (int u = 0; u < U; ++u) load_x(u);
#pragma unroll
            for (int u = 0; u < U; ++u) load_row(u, first + U + u);
#pragma unroll 1
            for (int ks = first; ks < last; ks += U) {
                const bool more = ks + U < last;
                store_b(careful, real_at);
                __syncthreads();
                if (careful.value && threadIdx.x == 0 && met) {
                    const int at = ((ks - first) / U) >> note_shift;
                    note[at >> 5] |= 1u << (at & 31);
                    met = 0;
                }
                words_t now[U];
#pragma unroll
                for (int u = 0; u < U; ++u) now[u] = x[u];
                if (more) {
                    load_b(ks + U);
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        load_x(u);
                        load_row(u, ks + 2 * U + u);
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    uint32_t w[MT];
#pragma unroll
                    for (int t = 0; t < MT; ++t) w[t] = transposed(now[u][t], lane);
                    multiply(u, w);
                }
                __syncthreads();
            }
        }
        float probe = 0.f;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) probe = fmaf(acc[t][n][i], 0.f, probe);
        return probe == 0.f;
    };
    if (!sweep(std::false_type())) bad = 1;
    __syncthreads();
    const bool careful = bad;
    bool overflowed = false;
    if (careful) {
        const int groups = (last - first + U - 1) / U;
        while (((groups - 1) >> note_shift) >= 32 * NOTES) ++note_shift;
        for (int i = threadIdx.x; i < NOTES; i += 64 * W) note[i] = 0;
        overflowed = !sweep(std::true_type());
        __syncthreads();
        // Which of a tile's 32 rows of sums have a term that takes them up (+infinity or NaN) or down (-infinity or NaN), a bit each; a lane looks
        // at its column; both make NaN, in whatever order.  A level's scores in 32 bits and gradient in bf16 take 0.6 and 0.3 ms with one row of
        // infinities, 2.3 and 2.1 ms when all is NaN.
        uint32_t up[MT][NT] = {}, down[MT][NT] = {};
        for (int noted = 0; noted < groups; noted += 1 << note_shift) {
            const int n_at = noted >> note_shift;
            if (!(note[n_at >> 5] >> (n_at & 31) & 1u)) continue;
            for (int h = 2 * (first + noted * U); h < 2 * min(last, first + (noted + (1 << note_shift)) * U); ++h) {
                // 32 terms; lane j (or j + 32) finds out which of the rows have term j
                const int64_t t0 = term(h >> 1, 32 * (h & 1));
                uint32_t has[MT];
                if constexpr (GRAD) {
                    const int64_t at = t0 + (lane & 31);
                    const uint32_t *words = at < limit ? row_of(a.bits, a.n, a.row_stride, a.rows, at) : nullptr;
#pragma unroll
                    for (int t = 0; t < MT; ++t) has[t] = words && (tile0 + t) * 32 < out_rows ? words[tile0 + t] : 0u;
                } else {
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        const int64_t r = (tile0 + t) * 32 + (lane & 31);
                        const uint32_t *words = r < out_rows && t0 < limit ? row_of(a.bits, a.n, a.row_stride, a.rows, r) : nullptr;
                        has[t] = transposed(words ? words[t0 >> 5] : 0u, lane);
                    }
                }
#pragma unroll 1
                for (int j0 = 0; j0 < 32; j0 += 8) {
                    uint32_t v[8][NT];
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const int cc = c0 + 32 * n + (lane & 31);
                            v[j][n] = cc < a.k && t0 + j0 + j < limit ? ((const raw_t *)a.mat)[(t0 + j0 + j) * a.mat_stride + cc] : 0u;
                        }
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int t = 0; t < MT; ++t) {
                            const uint32_t rows = __builtin_amdgcn_readlane(has[t], j0 + j);
#pragma unroll
                            for (int n = 0; n < NT; ++n)
                                if (not_finite<TYPE>(v[j][n])) {
                                    const float x = value_of<TYPE>(v[j][n]);
                                    up[t][n] |= x != -INFINITY ? rows : 0u;
                                    down[t][n] |= x != INFINITY ? rows : 0u;
                                }
                        }
                }
            }
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int r = 8 * (i >> 2) + 4 * half + (i & 3);
                    const bool u = up[t][n] >> r & 1u, d = down[t][n] >> r & 1u;
                    if (u || d) acc[t][n][i] = !d ? INFINITY : !u ? -INFINITY : NAN;
                }
    }

    const bool whole = a.parts == 1;
    float *to = whole ? a.out : a.part + (int64_t)block_z * out_rows * a.k;
    const int64_t stride = whole ? a.out_stride : a.k;
    const float scale = whole ? 0.5f * a.scale : 0.5f;
    const auto into = buffer(to + tile0 * 32 * stride, to ? (out_rows - tile0 * 32) * stride * 4 : 0);
    const uint32_t row_to = (uint32_t)stride * 4;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int cc = c0 + 32 * n + (lane & 31);
        const uint32_t at = cc < a.k ? (uint32_t)(4 * half * (int)stride + cc) * 4 : NOWHERE;
        const float bias = !GRAD && whole && a.bias && cc < a.k ? a.bias[cc] : 0.f;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const uint32_t pad = padding[t] >> (4 * half);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int r = 8 * (i >> 2) + (i & 3);
                float v = acc[t][n][i] * scale;
                if constexpr (!GRAD) {
                    if (any_padding)
                        v += pad >> r & 1u ? 0.f : bias;
                    else
                        v += bias;
                }
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), into, at + (32 * t + r) * row_to, 0, 0);
            }
        }
    }
    if constexpr (GRAD) {
        if (block_x == 0) {
#pragma unroll
            for (int i = 0; i < SUMS; ++i) sums[threadIdx.x * SUMS + i] = column_sum[i];
            __syncthreads();
            const int cc = c0 + threadIdx.x;
            if (threadIdx.x < COLS && cc < a.k) {
                float s = 0.f;
#pragma unroll
                for (int g = 0; g < 64 * W * SUMS / COLS; ++g) s += sums[g * COLS + threadIdx.x];
                if (!whole)
                    a.part[(int64_t)a.parts * out_rows * a.k + (int64_t)block_z * a.k + cc] = s;
                else if (a.bias_out)
                    a.bias_out[cc] = s;
            }
        }
    }
    // Not finite without the infinities and NaN: twice the sum, which is what the matrix cores make, may be too large where the sum is
    // not.  Added up term by term, which is slow (a level with one such column: scores 17 ms, gradient 89).
    if (!to || !overflowed) return;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int cc = c0 + 32 * n + (lane & 31);
        float probe = 0.f;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) probe = fmaf(acc[t][n][i], 0.f, probe);
        if (probe == 0.f || cc >= a.k) continue;
        const int64_t end = min(limit, term(last, 0));
        for (int e = 0; e < 16 * MT; ++e) {
            const int64_t r = tile0 * 32 + 32 * (e >> 4) + 8 * (e >> 2 & 3) + 4 * half + (e & 3);
            if (r >= out_rows) break;
            float s = 0.f;
            if constexpr (GRAD) {
                for (int64_t at = term(first, 0); at < end && s == s; ++at) {
                    const uint32_t *words = row_of(a.bits, a.n, a.row_stride, a.rows, at);
                    if (words && (words[r >> 5] >> (r & 31) & 1u)) s += value_of<TYPE>(((const raw_t *)a.mat)[at * a.mat_stride + cc]);
                }
            } else {
                const uint32_t *words = row_of(a.bits, a.n, a.row_stride, a.rows, r);
                if (!words) continue;
                for (int64_t w = term(first, 0) >> 5; 32 * w < end && s == s; ++w)
                    for (uint32_t bits = words[w]; bits; bits &= bits - 1) {
                        const int64_t at = 32 * w + __builtin_ctz(bits);
                        if (at < end) s += value_of<TYPE>(((const raw_t *)a.mat)[at * a.mat_stride + cc]);
                    }
            }
            to[r * stride + cc] = whole ? s * a.scale + (!GRAD && a.bias ? a.bias[cc] : 0.f) : s;
        }
    }
}

// The batch's bits by feature: turned[f][w], w < words = 8 * ceil(m / 256), with the words in the order in which k_product
// takes them: word 8 s + 4 h + q holds batch rows 64 (4 s + q) + 32 h + (0..31).  Row n_features says which batch rows are no padding.
// A wave turns 256 rows by 4 words of features; a lane loads 16 bytes of four rows and stores 16 bytes of four features.
// 32 x 32 bits are turned in five exchanges between lanes.  8,192 rows of 7,500 features: 8 us, 1.9 TB/s in and out; latency bounds it.
__global__ __launch_bounds__(256) void k_turn(ProductArgs a, uint32_t *turned, int row_words, int word_blocks) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int64_t s = blockIdx.x / word_blocks;
    const int w0 = (blockIdx.x % word_blocks * 4 + wave) * 4;
    if (w0 >= row_words) return;
    u32x4 x[4], real;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int64_t i = 64 * (4 * s + q) + lane;
        const uint32_t *row = i < a.m ? row_of(a.bits, a.n, a.row_stride, a.rows, i) : nullptr;
        x[q] = row ? *(const u32x4 *)(row + w0) : (u32x4)(0u);
        const uint64_t mask = __ballot(row != nullptr);
        real[q] = half ? (uint32_t)(mask >> 32) : (uint32_t)mask;
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        u32x4 y;
#pragma unroll
        for (int q = 0; q < 4; ++q) y[q] = transposed(x[q][t], lane);
        const int64_t f = (int64_t)(w0 + t) * 32 + (lane & 31);
        if (f < a.n_features) *(u32x4 *)(turned + f * a.words + 8 * s + 4 * half) = y;
    }
    if (w0 == 0 && (lane & 31) == 0) *(u32x4 *)(turned + (int64_t)a.n_features * a.words + 8 * s + 4 * half) = real;
}

// Adds up the parts, in order, eight loads in flight; no parts (an empty batch) make zeros.  Launch and memory latency bound it: 3 us
// for one node's 4,096 x 13 scores of 15 parts.
template <bool GRAD>
__global__ __launch_bounds__(256) void k_join(ProductArgs a, int parts, int64_t out_rows) {
    const int64_t all = out_rows * a.k;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < all + (GRAD ? a.k : 0); at += (int64_t)gridDim.x * 256) {
        const bool bias = GRAD && at >= all;
        const float *part = bias ? a.part + parts * all + (at - all) : a.part + at;
        const int64_t step = bias ? a.k : all;
        float s = 0.f;
        for (int p = 0; p < parts; p += 8) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = p + u < parts ? part[(p + u) * step] : 0.f;
#pragma unroll
            for (int u = 0; u < 8; ++u) s += v[u];
        }
        if (bias) {
            if (a.bias_out) a.bias_out[at - all] = s;
            continue;
        }
        const int64_t r = at / a.k;
        const int c = (int)(at - r * a.k);
        const bool padding = !GRAD && a.rows && !row_of(a.bits, a.n, a.row_stride, a.rows, r);
        if (a.out) a.out[r * a.out_stride + c] = padding ? 0.f : s * a.scale + (!GRAD && a.bias ? a.bias[c] : 0.f);
    }
}

// Few rows: the lookups themselves.  A workgroup makes one row of scores, `cw` columns of it (a power of two up to 64): it
// lists the row's tokens in LDS, 256 words at a time, and its 1024 / cw column groups take the tokens in turn, four loads in flight.
// Latency bounds it: the row, the list, the loads and the halving of the groups' sums take 4.2 us for a row of 7,500 features and 8 columns.
constexpr int LOOKUP_WORDS = 256;
template <typename T>
__global__ __launch_bounds__(1024) void k_lookup(ProductArgs a, int cw_log) {
    __shared__ uint16_t token[LOOKUP_WORDS * 32];
    __shared__ int before[4];
    __shared__ float part[1024];
    const int64_t i = blockIdx.x;
    const int cw = 1 << cw_log, c = blockIdx.y * cw + (threadIdx.x & (cw - 1)), slot = threadIdx.x >> cw_log, slots = 1024 >> cw_log;
    const uint32_t *row = row_of(a.bits, a.n, a.row_stride, a.rows, i);
    float s = 0.f;
    if (row) {
        const int words = (a.n_features + 31) / 32;
        for (int w0 = 0; w0 < words; w0 += LOOKUP_WORDS) {
            __syncthreads();
            uint32_t x = 0;
            int count = 0, inside = 0;
            if (threadIdx.x < LOOKUP_WORDS) {
                const int w = w0 + threadIdx.x;
                if (w < words) x = row[w];
                if (32 * (w + 1) > a.n_features) x &= w < words ? 0xffffffffu >> (32 * words - a.n_features) : 0u;
                count = __builtin_popcount(x);
                inside = count;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const int y = __shfl_up(inside, o);
                    if ((threadIdx.x & 63) >= o) inside += y;
                }
                if ((threadIdx.x & 63) == 63) before[threadIdx.x >> 6] = inside;
            }
            __syncthreads();
            const int b0 = before[0], b1 = before[1], b2 = before[2], total = b0 + b1 + b2 + before[3];
            if (threadIdx.x < LOOKUP_WORDS) {
                const int wv = threadIdx.x >> 6;
                int at = inside - count + (wv > 0 ? b0 : 0) + (wv > 1 ? b1 : 0) + (wv > 2 ? b2 : 0);
                for (; x; x &= x - 1) token[at++] = (uint16_t)(threadIdx.x * 32 + __builtin_ctz(x));
            }
            __syncthreads();
            if (c < a.k) {
                const T *from = (const T *)a.mat + (int64_t)w0 * 32 * a.mat_stride + c;
                int t = slot;
                for (; t + 3 * slots < total; t += 4 * slots) {
                    float v[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) v[u] = (float)from[(int64_t)token[t + u * slots] * a.mat_stride];
                    s += (v[0] + v[1]) + (v[2] + v[3]);
                }
                for (; t < total; t += slots) s += (float)from[(int64_t)token[t] * a.mat_stride];
            }
        }
    }
    part[threadIdx.x] = s;
    for (int half = slots / 2; half; half >>= 1) {
        __syncthreads();
        if (slot < half) part[threadIdx.x] += part[threadIdx.x + (half << cw_log)];
    }
    if (slot == 0 && c < a.k) a.out[i * a.out_stride + c] = row ? part[threadIdx.x] * a.scale + (a.bias ? a.bias[c] : 0.f) : 0.f;
}

// ------------------------------------------------------------------------------------------------------------------
// loss of siblings
// ------------------------------------------------------------------------------------------------------------------
// e = exp(-|s|): 2^t with the rounding of t = -|s| log2(e) put back in; below 2^-126 by way of 2^(t + 64)
__device__ __forceinline__ float exp_minus_abs(float s) {
#pragma clang fp contract(off)
    float x = fabsf(s);
    x = x > 110.f ? 110.f : x;
    const float t = -x * 0x1.715476p+0f, lost = fmaf(-x, 0x1.715476p+0f, -t) - x * 0x1.4ae0bep-26f;
    const bool low = t < -120.f;
    const float y = __builtin_amdgcn_exp2f(low ? t + 64.f : t);
    return fmaf(y, lost * 0x1.62e430p-1f, y) * (low ? 0x1p-64f : 1.f);
}

// log(1 + e) for 0 <= e <= 1: 2 artanh(z), z = e / (2 + e) <= 1/3, by its series; what is left out is below 2^-26 of it.  For
// small e it is e, whose halves may not be numbers of 32 bits.
__device__ __forceinline__ float log_one_plus(float e) {
    const float d = 2.f + e, r = __builtin_amdgcn_rcpf(d), z0 = e * r, z = fmaf(fmaf(-z0, d, e), r, z0), q = z * z;
    float p = 1.f / 15.f;
    p = fmaf(p, q, 1.f / 13.f);
    p = fmaf(p, q, 1.f / 11.f);
    p = fmaf(p, q, 1.f / 9.f);
    p = fmaf(p, q, 1.f / 7.f);
    p = fmaf(p, q, 1.f / 5.f);
    p = fmaf(p, q, 1.f / 3.f);
    return e < 0x1p-26f ? e : 2.f * fmaf(p * q, z, z);
}

struct LossArgs {
    const float *scores, *weight;
    const int32_t *label, *siblings;
    float *loss;                // one partial row of sums a workgroup row
    void *grad;
    int64_t score_stride, grad_stride, m;
    int32_t k, ct;              // ct: column vectors of a workgroup
    float scale;
};

// one score's loss and slope, times w
__device__ __forceinline__ void loss_of(float z, bool positive, float w, float &term, float &slope) {
    const float s = positive ? -z : z;
    const float e = exp_minus_abs(s), d = 1.f + e, r = __builtin_amdgcn_rcpf(d);
    term = w * ((s < 0.f ? 0.f : s) + log_one_plus(e));                              // softplus(s); NaN stays NaN
    const float p = (s >= 0.f ? 1.f : e) * fmaf(fmaf(-d, r, 1.f), r, r) * w;         // sigmoid(s)
    slope = positive ? -p : p;
}

// part[cv] = the sums of the rp threads of column cv, by halves (a single column's 1,024 one after the other took 6 us)
template <int V> __device__ __forceinline__ void add_rows(float *part, const float *sum, int r, int rp, int cv, int ct) {
#pragma unroll
    for (int j = 0; j < V; ++j) part[threadIdx.x * V + j] = sum[j];
    for (int n = rp; n > 1;) {
        const int half = (n + 1) / 2;
        __syncthreads();
        if (r + half < n) {
#pragma unroll
            for (int j = 0; j < V; ++j) part[threadIdx.x * V + j] += part[(threadIdx.x + half * ct) * V + j];
        }
        n = half;
    }
}

// A thread owns V neighbouring columns and goes down the rows of its workgroup, four at a time so that their loads are in
// flight together; loss sums stay in its registers until the workgroup adds them up in a fixed order and stores one
// partial row of K sums.  Scores are read only where the row trains.  Every score is read and every gradient written once: HBM bounds large
// ones, the launch small ones (300 x 8 in 4.7 us).
template <typename T, int V, int THREADS>
__global__ __launch_bounds__(THREADS) void k_loss(LossArgs a) {
    const float *const scores = a.scores, *const weight = a.weight;
    const int32_t *const label = a.label, *const siblings = a.siblings;
    float *const loss = a.loss;
    T *const grad = (T *)a.grad;
    const int64_t score_stride = a.score_stride, grad_stride = a.grad_stride, m = a.m;
    const int k = a.k, ct = a.ct;
    const float scale = a.scale;
    constexpr int ROWS_AT_ONCE = 4;
    typedef __attribute__((ext_vector_type(V))) T out_t;
    __shared__ float part[THREADS * V];
    const int cv = threadIdx.x % ct, r = threadIdx.x / ct, rp = THREADS / ct;
    const int c0 = (blockIdx.y * ct + cv) * V;
    float sum[V] = {};
    if (r < rp && c0 < k) {
        const int64_t step = (int64_t)gridDim.x * rp;
        for (int64_t i0 = (int64_t)blockIdx.x * rp + r; i0 < m; i0 += ROWS_AT_ONCE * step) {
            int lo[ROWS_AT_ONCE], hi[ROWS_AT_ONCE], lab[ROWS_AT_ONCE];
            float w[ROWS_AT_ONCE], z[ROWS_AT_ONCE][V];
#pragma unroll
            for (int u = 0; u < ROWS_AT_ONCE; ++u) {
                const int64_t i = i0 + u * step < m ? i0 + u * step : m - 1;
                lo[u] = siblings ? siblings[2 * i] : 0;
                hi[u] = siblings ? siblings[2 * i + 1] : k;
                lab[u] = label[i];
                w[u] = weight ? weight[i] : 1.f;
            }
#pragma unroll
            for (int u = 0; u < ROWS_AT_ONCE; ++u) {
                const int64_t i = i0 + u * step;
                if (i < m && c0 + V > lo[u] && c0 < hi[u]) {
                    const float *src = scores + i * score_stride + c0;
                    if constexpr (V == 1) {
                        z[u][0] = src[0];
                    } else {
#pragma unroll
                        for (int q = 0; q < V; q += 4) {
                            const float4 f = *(const float4 *)(src + q);
                            z[u][q] = f.x, z[u][q + 1] = f.y, z[u][q + 2] = f.z, z[u][q + 3] = f.w;
                        }
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < ROWS_AT_ONCE; ++u) {
                const int64_t i = i0 + u * step;
                if (i >= m) break;
                out_t g = (out_t)(T)0.f;
                if (c0 + V > lo[u] && c0 < hi[u]) {
                    const float wu = scale * w[u];
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const int c = c0 + j;
                        if (c < lo[u] || c >= hi[u]) continue;
                        float term, slope;
                        loss_of(z[u][j], c == lab[u], wu, term, slope);
                        sum[j] += term;
                        g[j] = (T)slope;
                    }
                }
                if (grad) __builtin_nontemporal_store(g, (out_t *)(grad + i * grad_stride + c0));
            }
        }
    }
    if (!loss) return;
    add_rows<V>(part, sum, r, rp, cv, ct);
    if (r == 0 && c0 < k) {
#pragma unroll
        for (int j = 0; j < V; ++j) loss[(int64_t)blockIdx.x * k + c0 + j] = part[cv * V + j];
    }
}

// The same where rows train ranges of columns: a place of the tree has a handful of siblings among the thousands of a level,
// so a row's gradient is zeros but for them, and what bounds the loss is writing those.  A workgroup takes ROWS rows at once: 256 / ROWS
// threads to a row compute its siblings (if they are no more) into LDS, then the owners of columns put them into the vectors
// of zeros that they store and into their sums.  Wider ranges are computed by the owners.  65,536 x 1,000 in bf16: 39 us a
// pass with 8 rows, 45 with 16, 49 with 32; each owner computing its own, one lane in 64 busy: 65.  Narrow tables, where an
// owner's next row is many rows on, take 32.
template <typename T, int V, int ROWS>
__global__ __launch_bounds__(256) void k_loss_siblings(LossArgs a) {
    const float *const scores = a.scores, *const weight = a.weight;
    const int32_t *const label = a.label, *const siblings = a.siblings;
    float *const loss = a.loss;
    T *const grad = (T *)a.grad;
    const int64_t score_stride = a.score_stride, grad_stride = a.grad_stride, m = a.m;
    const int k = a.k, ct = a.ct;
    const float scale = a.scale;
    constexpr int NARROW = 256 / ROWS;
    typedef __attribute__((ext_vector_type(V))) T out_t;
    __shared__ int s_lo[ROWS], s_hi[ROWS], s_label[ROWS];
    __shared__ float s_weight[ROWS], s_term[ROWS][NARROW], s_slope[ROWS][NARROW];
    __shared__ float part[256 * V];
    const int cv = threadIdx.x % ct, r = threadIdx.x / ct, rp = 256 / ct;
    const int c0 = (blockIdx.y * ct + cv) * V;
    float sum[V] = {};
    for (int64_t i0 = (int64_t)blockIdx.x * ROWS; i0 < m; i0 += (int64_t)gridDim.x * ROWS) {
        {
            const int q = threadIdx.x / NARROW, j = threadIdx.x % NARROW;
            const int64_t i = i0 + q;
            int lo = 0, hi = 0, lab = -1;
            float w = 0.f;
            if (i < m) {
                lo = max(siblings[2 * i], 0);
                hi = max(min(siblings[2 * i + 1], k), 0);
                lab = label[i];
                w = scale * (weight ? weight[i] : 1.f);
            }
            if (hi - lo <= NARROW && j < hi - lo) loss_of(scores[i * score_stride + lo + j], lo + j == lab, w, s_term[q][j], s_slope[q][j]);
            if (j == 0) {
                s_lo[q] = lo;
                s_hi[q] = hi;
                s_label[q] = lab;
                s_weight[q] = w;
            }
        }
        __syncthreads();
        if (r < rp && c0 < k) {
            for (int q = r; q < ROWS; q += rp) {
                const int64_t i = i0 + q;
                if (i >= m) break;
                const int lo = s_lo[q], hi = s_hi[q];
                out_t g = (out_t)(T)0.f;
                if (c0 + V > lo && c0 < hi) {
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const int c = c0 + j;
                        if (c < lo || c >= hi) continue;
                        float term, slope;
                        if (hi - lo <= NARROW) {
                            term = s_term[q][c - lo];
                            slope = s_slope[q][c - lo];
                        } else {
                            loss_of(scores[i * score_stride + c], c == s_label[q], s_weight[q], term, slope);
                        }
                        sum[j] += term;
                        g[j] = (T)slope;
                    }
                }
                if (grad) __builtin_nontemporal_store(g, (out_t *)(grad + i * grad_stride + c0));
            }
        }
        __syncthreads();
    }
    if (!loss) return;
    add_rows<V>(part, sum, r, rp, cv, ct);
    if (r == 0 && c0 < k) {
#pragma unroll
        for (int j = 0; j < V; ++j) loss[(int64_t)blockIdx.x * k + c0 + j] = part[cv * V + j];
    }
}

// adds up the partial rows: 32 columns a workgroup, every 32nd row to a thread, then the 32 sums in order (1,024 rows of 1,000: 4.4 us)
__global__ __launch_bounds__(1024) void k_loss_join(const float *part, int n_parts, int k, float *loss) {
    __shared__ double sums[32][33];
    const int col = threadIdx.x & 31, g = threadIdx.x >> 5, c = blockIdx.x * 32 + col;
    double s = 0.0;
    if (c < k) {
#pragma unroll 8
        for (int p = g; p < n_parts; p += 32) s += part[(int64_t)p * k + c];
    }
    sums[g][col] = s;
    __syncthreads();
    if (g == 0 && c < k) {
        for (int q = 1; q < 32; ++q) s += sums[q][col];
        loss[c] = (float)s;
    }
}

// ------------------------------------------------------------------------------------------------------------------
// AdamW over many tensors
// ------------------------------------------------------------------------------------------------------------------
constexpr int STEP_COUNTERS = 32, STEP_LINE = 32;
static_assert(STAG_ADAMW_STEP_WORDS == STEP_LINE * (2 + STEP_COUNTERS), "the words of d_step");

struct AdamwArgs {
    const stag_adamw_tensor_t *tensors;
    const stag_adamw_tile_t *tiles;
    int64_t n_tiles;
    int split;                  // waves to a tile: 1, or 4 (a block each) when there are few
    void *m, *v;
    float *m_scale, *v_scale;
    int32_t *step;
    float lr, beta1, beta2, one_minus_beta1, one_minus_beta2, log_beta1, log_beta2, eps;
};

// Four neighbouring values as they lie in memory (16-bit ones in the first two words), past the caches: a step touches each once.
// `whole`: all there and aligned; otherwise one by one up to `count`, zeros behind it.
__device__ __forceinline__ u32x4 load4(const void *p, int type, int64_t at, int64_t count, bool whole) {
    u32x4 x = (u32x4)(0u);
    if (whole) {
        if (type == STAG_F32) return __builtin_nontemporal_load((const u32x4 *)((const uint32_t *)p + at));
        const u32x2 q = __builtin_nontemporal_load((const u32x2 *)((const uint16_t *)p + at));
        x[0] = q[0], x[1] = q[1];
        return x;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (at + j < count) {
            if (type == STAG_F32)
                x[j] = ((const uint32_t *)p)[at + j];
            else
                x[j >> 1] |= (uint32_t)((const uint16_t *)p)[at + j] << (16 * (j & 1));
        }
    return x;
}

__device__ __forceinline__ void values4(u32x4 raw, int type, float *x) {
    if (type == STAG_F32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(raw[j]);
    } else if (type == STAG_BF16) {
#pragma unroll
        for (int j = 0; j < 2; ++j) x[2 * j] = __uint_as_float(raw[j] << 16), x[2 * j + 1] = __uint_as_float(raw[j] & 0xffff0000u);
    } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) x[2 * j] = (float)__builtin_bit_cast(f16, (uint16_t)raw[j]), x[2 * j + 1] = (float)__builtin_bit_cast(f16, (uint16_t)(raw[j] >> 16));
    }
}

__device__ __forceinline__ void store4(void *p, int type, int64_t at, int64_t count, bool whole, const float *x) {
    if (type == STAG_F32) {
        if (whole) {
            __builtin_nontemporal_store((f32x4){x[0], x[1], x[2], x[3]}, (f32x4 *)((float *)p + at));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (at + j < count) ((float *)p)[at + j] = x[j];
        }
        return;
    }
    uint16_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = type == STAG_BF16 ? __builtin_bit_cast(uint16_t, (bf16)x[j]) : __builtin_bit_cast(uint16_t, (f16)x[j]);
    if (whole) {
        __builtin_nontemporal_store((u32x2){h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16}, (u32x2 *)((uint16_t *)p + at));
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (at + j < count) ((uint16_t *)p)[at + j] = h[j];
    }
}

// the largest of the wave's x and of its y, the same for every lane; both at once, since a lane's neighbour can be read two instructions on
__device__ __forceinline__ void wave_max(uint32_t &x, uint32_t &y) {
#define STAG_MAX_DPP(CONTROL)                                                              \
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CONTROL, 0xf, 0xf, true)); \
    y = max(y, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)y, CONTROL, 0xf, 0xf, true));
    STAG_MAX_DPP(0x111)      // row_shr 1, 2, 4, 8: the last lane of each 16 has their maximum
    STAG_MAX_DPP(0x112)
    STAG_MAX_DPP(0x114)
    STAG_MAX_DPP(0x118)
    STAG_MAX_DPP(0x142)      // row_bcast 15, 31: the last lane has all
    STAG_MAX_DPP(0x143)
#undef STAG_MAX_DPP
    x = (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
    y = (uint32_t)__builtin_amdgcn_readlane((int)y, 63);
}

// The exponents (biased) of the smallest powers of two s with max|x| <= 448 s over the wave's 256 values x, and y >= 0; 448 = 1.75 * 2^8
// is the largest e4m3 value.  A power of two, so that dividing by it rounds nothing.  Infinities and NaN have no say.
__device__ __forceinline__ void scale_exponents(const float *x, const float *y, int &x_exponent, int &y_exponent) {
    constexpr float LEAST = 0x1p-117f;      // biased exponent 10
    uint32_t top_x = __float_as_uint(fmaxf(fmaxf(fmaxf(LEAST, fabsf(x[0])), fmaxf(fabsf(x[1]), fabsf(x[2]))), fabsf(x[3])));
    uint32_t top_y = __float_as_uint(fmaxf(fmaxf(fmaxf(LEAST, fabsf(y[0])), fmaxf(fabsf(y[1]), fabsf(y[2]))), fabsf(y[3])));
    wave_max(top_x, top_y);
    if (max(top_x, top_y) >= 0x7f800000u) {
        asm volatile("");                   // seldom: not to be computed beforehand
        top_x = top_y = __float_as_uint(LEAST);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t a = __float_as_uint(x[j]) & 0x7fffffffu, b = __float_as_uint(y[j]) & 0x7fffffffu;
            top_x = max(top_x, a < 0x7f800000u ? a : 0u);
            top_y = max(top_y, b < 0x7f800000u ? b : 0u);
        }
        wave_max(top_x, top_y);
    }
    x_exponent = (int)(top_x >> 23) - 8 + ((top_x & 0x7fffffu) > 0x600000u);
    y_exponent = (int)(top_y >> 23) - 8 + ((top_y & 0x7fffffu) > 0x600000u);
}

// x's e4m3 code as byte J of `codes`, rounded up or down by `chance` (the upper 16 bits of it).  From 2^-6 on a code has 3 bits behind the
// leading one: adding 20 random bits below them and cutting them off goes up with the probability of what is cut.  Below 2^-6
// codes are 2^-9 apart, as they are from 2^-6 to 2^-5: such a value is moved there (what is below 2^-29 of it is dropped), rounded and moved back.
// That is what the conversion instruction does; written out it took 9 instructions.
template <int J> __device__ __forceinline__ uint32_t with_e4m3(float x, uint32_t chance, uint32_t codes) {
    return (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(x, (int)((chance & 0xffff0000u) | 0x8000u), (int)codes, J);
}

// The roots of four values >= 0.  32 bits: by the instruction.  8 bits: from x / sqrt(x) and one step of Newton's method, which puts the
// rounding right.  The instructions take what is below 2^-126 for zero, and what Newton's step subtracts below 2^-96 is no normal
// number; such values (zero among them) are multiplied by 2^64 first, in a branch that a wave seldom takes.
template <int BITS> __device__ __forceinline__ void roots_of(const float *x, float *root) {
    auto plain = [](float x) {
        if constexpr (BITS == 32) return __builtin_amdgcn_sqrtf(x);
        const float s = __builtin_amdgcn_rsqf(x), y = x * s;
        return x == 0.f || x == INFINITY ? x : fmaf(fmaf(-y, y, x), 0.5f * s, y);
    };
    constexpr uint32_t SMALL = 0x0f800000u;      // 2^-96
    const uint32_t least = min(min(__float_as_uint(x[0]), __float_as_uint(x[1])), min(__float_as_uint(x[2]), __float_as_uint(x[3])));
    if (least >= SMALL) {
#pragma unroll
        for (int j = 0; j < 4; ++j) root[j] = plain(x[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool small = __float_as_uint(x[j]) < SMALL;
            const float y = plain(small ? x[j] * 0x1p64f : x[j]);
            root[j] = small ? y * 0x1p-32f : y;
        }
    }
}

__device__ __forceinline__ void unpack_e4m3(uint32_t q, float *x) {
    x[0] = __builtin_amdgcn_cvt_f32_fp8((int)q, 0);
    x[1] = __builtin_amdgcn_cvt_f32_fp8((int)q, 1);
    x[2] = __builtin_amdgcn_cvt_f32_fp8((int)q, 2);
    x[3] = __builtin_amdgcn_cvt_f32_fp8((int)q, 3);
}

// A wave takes a tile of four blocks of 256 values, four neighbouring values a lane, and has the loads of GROUP blocks in
// flight before it computes.  Everything is read once and written once; what bounds it with 32-bit states is HBM (the 54 million
// values of 1,600 tables in 32 bits, 1.5 GB: 253 us, 6.0 TB/s), with 8-bit ones the 60 instructions a value (as bf16: 126 us, 4.3 TB/s).  m, v and the root are rounded after
// every operation (no fused multiply-add), so that the 8-bit codes are a function of the inputs that any other 32-bit
// implementation can restate.
template <int BITS>
__global__ __launch_bounds__(256) void k_adamw(AdamwArgs a) {
#pragma clang fp contract(off)
    constexpr int GROUP = BITS == 32 ? 4 : 2;
    const int lane = threadIdx.x & 63;
    const int t = __hip_atomic_load(a.step, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1;
    // 1 - beta^t = -expm1(t log beta)
    const float c1 = a.lr / -expm1f((float)t * a.log_beta1);
    const float c2 = 1.f / sqrtf(-expm1f((float)t * a.log_beta2));
    const uint32_t salt = (uint32_t)t * 0x9E3779B9u;
    for (int64_t w = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); w < a.n_tiles * a.split; w += (int64_t)gridDim.x * 4) {
        const stag_adamw_tile_t tile = a.tiles[a.split == 1 ? w : w / 4];
        const stag_adamw_tensor_t d = a.tensors[tile.tensor];
        const int64_t at0 = (int64_t)tile.tile * STAG_ADAMW_TILE, s0 = d.state_at + at0;
        const bool vec_p = ((uintptr_t)d.param & (d.param_type == STAG_F32 ? 15 : 7)) == 0;
        const bool vec_g = ((uintptr_t)d.grad & (d.grad_type == STAG_F32 ? 15 : 7)) == 0;
        const float keep = 1.f - a.lr * d.weight_decay, shrink = a.lr * d.l1;
        const int from = a.split == 1 ? 0 : (int)(w & 3);
        const int blocks = (int)min((int64_t)(a.split == 1 ? STAG_ADAMW_TILE / STAG_ADAMW_BLOCK : from + 1), (d.count - at0 + STAG_ADAMW_BLOCK - 1) / STAG_ADAMW_BLOCK);
        const bool inside = at0 + STAG_ADAMW_TILE <= d.count;
#pragma unroll 1
        for (int b0 = from; b0 < blocks; b0 += GROUP) {
            u32x4 raw_p[GROUP], raw_g[GROUP], raw_m[GROUP], raw_v[GROUP];
            float ms[GROUP], vs[GROUP];
#pragma unroll
            for (int b = 0; b < GROUP; ++b) {
                if (b0 + b >= blocks) continue;
                const int64_t at = at0 + (b0 + b) * STAG_ADAMW_BLOCK + lane * 4, s = s0 + (b0 + b) * STAG_ADAMW_BLOCK + lane * 4;
                const bool full = inside || at + 4 <= d.count;
                raw_p[b] = load4(d.param, d.param_type, at, d.count, full && vec_p);
                raw_g[b] = load4(d.grad, d.grad_type, at, d.count, full && vec_g);
                if constexpr (BITS == 32) {
                    raw_m[b] = load4(a.m, STAG_F32, s, 0, true);
                    raw_v[b] = load4(a.v, STAG_F32, s, 0, true);
                } else {
                    raw_m[b][0] = __builtin_nontemporal_load((const uint32_t *)((const uint8_t *)a.m + s));
                    raw_v[b][0] = __builtin_nontemporal_load((const uint32_t *)((const uint8_t *)a.v + s));
                    ms[b] = a.m_scale[s0 / STAG_ADAMW_BLOCK + b0 + b];
                    vs[b] = a.v_scale[s0 / STAG_ADAMW_BLOCK + b0 + b];
                }
            }
#pragma unroll
            for (int b = 0; b < GROUP; ++b) {
                if (b0 + b >= blocks) continue;
                const int64_t at = at0 + (b0 + b) * STAG_ADAMW_BLOCK + lane * 4, s = s0 + (b0 + b) * STAG_ADAMW_BLOCK + lane * 4;
                const bool full = inside || at + 4 <= d.count;
                float p[4], g[4], m[4], v[4], root[4];
                values4(raw_p[b], d.param_type, p);
                values4(raw_g[b], d.grad_type, g);
                if constexpr (BITS == 32) {
                    values4(raw_m[b], STAG_F32, m);
                    values4(raw_v[b], STAG_F32, v);
                } else {
                    unpack_e4m3(raw_m[b][0], m);
                    unpack_e4m3(raw_v[b][0], v);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        m[j] = m[j] * ms[b];
                        v[j] = v[j] * vs[b];
                        v[j] = v[j] * v[j];
                    }
                }
                if (!inside) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (at + j >= d.count) m[j] = v[j] = 0.f;      // places between tensors hold nothing
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    m[j] = m[j] * a.beta1 + g[j] * a.one_minus_beta1;
                    v[j] = v[j] * a.beta2 + (g[j] * g[j]) * a.one_minus_beta2;
                }
                roots_of<BITS>(v, root);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float r = __builtin_amdgcn_rcpf(fmaf(root[j], c2, a.eps));
                    p[j] = fmaf(-c1 * m[j], r, p[j] * keep);
                    if (shrink > 0.f) {
                        const float left = fmaf(-shrink, r, fabsf(p[j]));
                        p[j] = copysignf(left < 0.f ? 0.f : left, p[j]);
                    }
                }
                store4(d.param, d.param_type, at, d.count, full && vec_p, p);
                if constexpr (BITS == 32) {
                    store4(a.m, STAG_F32, s, 0, true, m);
                    store4(a.v, STAG_F32, s, 0, true, v);
                } else {
                    int me, ve;
                    scale_exponents(m, root, me, ve);
                    const float mi = __int_as_float((254 - me) << 23), vi = __int_as_float((254 - ve) << 23);
                    uint32_t m_codes = 0, v_codes = 0;
                    auto code = [&](auto place) {
                        constexpr int j = place.value;
                        // Two rounds of shift, exclusive or and multiply, with the constants that C. Wellons published ("Prospecting for Hash
                        // Functions", 2018)
                        uint32_t x = (uint32_t)(s + j) ^ salt;
                        x = (x ^ x >> 16) * 0x7FEB352Du;
                        x = (x ^ x >> 15) * 0x846CA68Bu;
                        x ^= x >> 16;
                        // a root of zero would divide by eps alone: what is not zero stays so
                        uint32_t q = __float_as_uint(root[j] * vi);
                        if (q - 1u < 0x3b000000u - 1u) q = 0x3b000000u;      // 2^-9
                        m_codes = with_e4m3<j>(m[j] * mi, x, m_codes);
                        v_codes = with_e4m3<j>(__uint_as_float(q), x << 16, v_codes);
                    };
                    code(std::integral_constant<int, 0>());
                    code(std::integral_constant<int, 1>());
                    code(std::integral_constant<int, 2>());
                    code(std::integral_constant<int, 3>());
                    __builtin_nontemporal_store(m_codes, (uint32_t *)((uint8_t *)a.m + s));
                    __builtin_nontemporal_store(v_codes, (uint32_t *)((uint8_t *)a.v + s));
                    if (lane == 0) {
                        a.m_scale[s >> 8] = __int_as_float(me << 23);
                        a.v_scale[s >> 8] = __int_as_float(ve << 23);
                    }
                }
            }
        }
    }
    // The last workgroup to come here, when all have read t, counts the step.  2,048 atomics on one address took 120 us, so
    // the workgroups come in by 32 counters in lines of their own, and the last of each goes on to the one of all.  Nothing
    // else is ordered by this, so it is relaxed: a release would write back the L2 for every workgroup.
    __syncthreads();
    if (threadIdx.x == 0) {
        const int groups = min((int)gridDim.x, STEP_COUNTERS), g = blockIdx.x % STEP_COUNTERS;
        int32_t *mine = a.step + STEP_LINE * (1 + g), *all = a.step + STEP_LINE * (1 + STEP_COUNTERS);
        if (__hip_atomic_fetch_add(mine, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == ((int)gridDim.x - 1 - g) / STEP_COUNTERS) {
            __hip_atomic_store(mine, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (__hip_atomic_fetch_add(all, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == groups - 1) {
                __hip_atomic_store(all, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_store(a.step, t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------------------------
constexpr int64_t MAX_M = (int64_t)1 << 31;      // rows of a batch
constexpr int32_t MAX_K = 1 << 20;               // classifiers of a table
constexpr int32_t MAX_FEATURES = 1 << 27;
constexpr int64_t MAX_THREADS = (int64_t)1 << 32;      // a launch has fewer than this along x
constexpr int64_t MAX_STRIDE = 1 << 21;          // 160 rows of it stay under 2^31 bytes, a buffer's reach

int check_rows(const uint32_t *d_bits, int64_t n, int64_t row_stride, int32_t n_features, const int32_t *d_rows, int64_t m, int32_t k, int type) {
    REQUIRE(type_known(type), "unknown type %d", type);
    REQUIRE(n_features >= 1 && n_features <= MAX_FEATURES, "n_features = %d is not in 1..%d", n_features, MAX_FEATURES);
    REQUIRE(k >= 1 && k <= MAX_K, "k = %d is not in 1..%d", k, MAX_K);
    REQUIRE(m >= 0 && m < MAX_M, "m = %lld is not in 0..2^31-1", (long long)m);
    REQUIRE(n >= 0, "n = %lld is negative", (long long)n);
    REQUIRE(d_rows || m <= n, "m = %lld rows of %lld, without d_rows", (long long)m, (long long)n);
    REQUIRE(row_stride % 4 == 0 && row_stride * 32 >= n_features, "row_stride = %lld words: a multiple of 4 that holds %d features is wanted",
            (long long)row_stride, n_features);
    REQUIRE(n == 0 || (d_bits && aligned(d_bits, 16)), "d_bits is null or not 16-byte aligned");
    REQUIRE(aligned(d_rows, 4), "d_rows is not 4-byte aligned");
    return STAG_OK;
}

int check_matrix(const char *name, const void *p, int type, int64_t stride, int32_t k) {
    REQUIRE(p && aligned(p, type_bytes(type)), "%s is null or not aligned to its type", name);
    REQUIRE(stride >= k, "%s's stride %lld is less than its %d columns", name, (long long)stride, k);
    REQUIRE(stride <= MAX_STRIDE, "%s's stride %lld is over %lld", name, (long long)stride, (long long)MAX_STRIDE);
    return STAG_OK;
}

#define TRY(expr)                 \
    do {                          \
        const int rc_ = (expr);   \
        if (rc_ != STAG_OK) return rc_; \
    } while (0)

// how a product is cut up
struct Plan {
    bool lookup;
    Source src;
    int mt, nt, steps, per_part, parts;
    int64_t row_blocks, col_blocks, out_rows, turned_words, turned_bytes, work_bytes;
};

// In how many parts the sum is cut, so that few result tiles still fill the card: of 1, 2, 3, 4, 6, 8, 12 .. 256 and those that fill it once,
// the one whose time is the least by what was measured on the card, in ns -- `step` for each step of a workgroup that has its CU to
// itself, half as much again where two share one (`shared`: they fit), and for more than one part 5,000 for the second launch and the parts'
// sums once out and once in at 4 TB/s.  (628 small and medium sizes: 3,000 instead 1.1 % slower on the mean, up to 4 us a pass; 7,000 0.4 %, up to 14.)
struct Cut {
    int parts;
    double time;
};
Cut best_cut(int64_t blocks, int steps, int step, bool shared, int64_t values) {
    Cut best = {1, 0.0};
    auto look = [&](int parts) {
        if (parts < 1 || parts > steps || parts > 256) return;
        const int per = (steps + parts - 1) / parts;
        const double all = (double)blocks * ((steps + per - 1) / per);
        const double load = !shared ? std::ceil(all / 256) : all <= 256 ? 1.0 : 1.5 * std::ceil(all / 512);
        const double time = per * (double)step * load + (parts > 1 ? 5000.0 + 8.0 * parts * (double)values / 4000.0 : 0.0);
        if (parts == 1 || time < best.time) best = {parts, time};
    };
    for (int parts = 1; parts <= 256; parts *= 2) {
        look(parts);
        look(parts + parts / 2);
    }
    look((int)(256 / blocks));
    look((int)(512 / blocks));
    return best;
}

Plan product_plan(bool grad, int64_t m, int32_t n_features, int32_t k, int type) {
    Plan p = {};
    p.out_rows = grad ? n_features : m;
    if (m == 0) return p;
    // Few lookups are done one by one: 4.3 us for a row of 7,500 features and 8 columns, where the product and its join take 8;
    // 512 rows 7.5 against 8.9, 32 columns 10.0 against 9.4; 16 rows of 1,000 columns 16 against 19, 32 rows 23 against 19.
    // A row is one workgroup's: 100,000 features keep it 25 us, the product 16.
    p.lookup = !grad && m * ceil_div(k, 64) <= 512 && n_features <= 32768 && m * k * n_features <= 120000000;
    if (p.lookup) return p;
    p.nt = k <= 32 ? 1 : 2;
    p.col_blocks = ceil_div(k, 32 * p.nt);
    // Turning the bits beforehand pays when many column blocks would each turn them (us beforehand against as they go, 32 bits and 7,500
    // features: 3,000 rows x 400 columns 65 against 76, x 200 43 against 42, 1,800 x 1,000 75 against 81, 1,100 x 400 43 against 32; bf16 and
    // 2,500 features: 3,000 x 1,000 36 against 52, x 400 26 against 26, x 200 24 against 20; 750 features, 5,000 x 1,000: 30 against 29)
    p.src = !grad ? ROWS : k > 128 && n_features >= 2048 && m * k >= 800000 ? TURNED : TURN;
    if (p.src == TURNED) {
        p.turned_words = 8 * ceil_div(m, 256);
        p.turned_bytes = ceil_div(((int64_t)n_features + 1) * p.turned_words * 4, 256) * 256;
    }
    p.steps = (int)(p.src == ROWS ? ceil_div(n_features, 256) : p.src == TURN ? ceil_div(m, 64) : ceil_div(m, 256));
    // One row tile a wave or two: two share what they load, one fills the card with fewer rows.  Over 149 sizes of 300 to 8,192 rows, 40 to 1,000
    // columns and 750 to 30,000 features the choice comes out 1 % above the better of both, two tiles always 14 % above it.
    double least = 0;
    for (int mt = p.src == TURNED ? 2 : 1; mt <= (p.src == TURN || p.nt == 1 ? 1 : 2); ++mt) {
        const int64_t row_blocks = ceil_div(p.out_rows, 32 * W * mt);
        const int step = type == STAG_F32 ? (p.src == TURN ? (p.nt == 2 ? 1100 : 800) : p.nt == 1 ? 2200 : mt == 1 ? 4600 : 7600)
                                          : (p.src == TURN ? (p.nt == 2 ? 700 : 500) : p.nt == 1 ? 1300 : mt == 1 ? 2400 : 2900);
        const Cut cut = best_cut(row_blocks * p.col_blocks, p.steps, step, p.src == TURN || p.nt == 1, p.out_rows * k);
        if (p.mt && cut.time >= least) continue;
        least = cut.time;
        p.mt = mt;
        p.row_blocks = row_blocks;
        p.per_part = (int)ceil_div(p.steps, cut.parts);
        p.parts = (int)ceil_div(p.steps, p.per_part);
    }
    p.work_bytes = p.turned_bytes + (p.parts > 1 ? ((int64_t)p.parts * (p.out_rows + (grad ? 1 : 0)) * k) * 4 : 0);
    return p;
}

// launches k_product<TYPE, SRC, MT, NT, WIDE> if that is what the plan says and the coefficients lie so
template <int TYPE, Source SRC, int MT, int NT, bool WIDE>
bool launched(const Plan &p, const ProductArgs &a, hipStream_t st) {
    if (p.src != SRC || p.mt != MT || p.nt != NT || (WIDE && (a.mat_stride % 4 || !aligned(a.mat, 4 * type_bytes(TYPE))))) return false;
    k_product<TYPE, SRC, MT, NT, WIDE><<<8 * (unsigned)ceil_div(p.row_blocks * p.col_blocks * p.parts, 8), 64 * W, 0, st>>>(a);
    return true;
}

template <int TYPE, bool GRAD>
int product(const Plan &p, ProductArgs a, void *work, hipStream_t st) {
    a.words = (int32_t)ceil_div(a.n_features, 128) * 4;
    a.steps = p.steps;
    a.steps_per_part = p.per_part;
    a.part = (float *)((char *)work + p.turned_bytes);
    a.row_blocks = (int32_t)p.row_blocks;
    a.col_blocks = (int32_t)p.col_blocks;
    a.parts = p.parts;
    REQUIRE((p.row_blocks * p.col_blocks * p.parts + 8) * 64 * W < MAX_THREADS, "%lld rows of %d columns are too many", (long long)p.out_rows, a.k);
    if (p.parts) {
        bool done;
        if constexpr (GRAD) {
            if (p.src == TURNED) {
                const int row_words = a.words;
                a.turned = (const uint32_t *)work;
                a.words = (int32_t)p.turned_words;
                const int64_t word_blocks = ceil_div(row_words, 16), turns = ceil_div(a.m, 256) * word_blocks;
                REQUIRE(turns * 256 < MAX_THREADS, "%lld rows of %d features are too many", (long long)a.m, a.n_features);
                k_turn<<<(unsigned)turns, 256, 0, st>>>(a, (uint32_t *)work, row_words, (int)word_blocks);
            }
            done = launched<TYPE, TURNED, 2, 2, true>(p, a, st) || launched<TYPE, TURNED, 2, 2, false>(p, a, st) || launched<TYPE, TURN, 1, 2, false>(p, a, st) ||
                   launched<TYPE, TURN, 1, 1, false>(p, a, st);
        } else {
            done = launched<TYPE, ROWS, 2, 2, true>(p, a, st) || launched<TYPE, ROWS, 2, 2, false>(p, a, st) || launched<TYPE, ROWS, 1, 2, true>(p, a, st) || launched<TYPE, ROWS, 1, 2, false>(p, a, st) ||
                   launched<TYPE, ROWS, 1, 1, false>(p, a, st);
        }
        REQUIRE(done, "no kernel for %d x %d tiles", p.mt, p.nt);
        HIP_TRY(hipGetLastError());
    }
    if (p.parts != 1) {      // an empty sum has no parts
        const int64_t blocks = ceil_div((p.out_rows + (GRAD ? 1 : 0)) * a.k, 256);
        k_join<GRAD><<<(unsigned)(blocks < 1 << 20 ? blocks : 1 << 20), 256, 0, st>>>(a, p.parts, p.out_rows);
        HIP_TRY(hipGetLastError());
    }
    return STAG_OK;
}

template <typename T>
int lookup(const ProductArgs &a, hipStream_t st) {
    int cw_log = 0;
    while (cw_log < 6 && (1 << cw_log) < a.k) ++cw_log;
    k_lookup<T><<<dim3((unsigned)a.m, (unsigned)ceil_div(a.k, 1 << cw_log)), 1024, 0, st>>>(a, cw_log);
    HIP_TRY(hipGetLastError());
    return STAG_OK;
}

// how k_loss is laid over [m][k]
struct LossPlan {
    int v, ct, threads;
    unsigned gx, gy;
};

LossPlan loss_plan(int64_t m, int32_t k, int v, bool siblings) {
    LossPlan p;
    // few values: one workgroup a column tile, whose sums are the result without a second launch; the more threads, the
    // fewer values one after the other (300 x 8: 9.3 us with 256 threads of four columns, 4.7 with 1,024 of one)
    const bool few = m * (int64_t)k <= 16384;
    p.threads = few ? 1024 : 256;
    p.v = few ? 1 : v;
    const int64_t cols = ceil_div(k, p.v);
    p.ct = (int)(cols < p.threads ? cols : p.threads);
    p.gy = (unsigned)ceil_div(cols, p.ct);
    // 1,024 workgroups, or 512 where each writes rows of siblings' gradients over nearly all of its threads (65,536 x 1,000 in 32 bits 60
    // against 71 us, x 4,000 in bf16 97 against 112; over half of the threads, x 1,000 and x 520 in bf16, 52 against 36 and 47 against 30).
    // A last tile of few columns takes as many workgroups as a full one, which costs most just above one tile (x 256 24 us, x 257 69).
    const unsigned all = siblings && p.ct >= 192 ? 512 : 1024;
    const int64_t passes = ceil_div(m, p.threads / p.ct), wanted = all / p.gy > 0 ? all / p.gy : 1;
    p.gx = (unsigned)(few ? 1 : passes < wanted ? passes : wanted);
    return p;
}

template <typename T>
int loss_typed(const LossPlan &p, LossArgs a, float *parts, hipStream_t st) {
    float *const d_loss = a.loss;
    const bool d_siblings = a.siblings != nullptr, join = d_loss && p.gx > 1;
    if (join) a.loss = parts;
    a.ct = p.ct;
    auto launch = [&](auto kernel) { kernel<<<dim3(p.gx, p.gy), p.threads, 0, st>>>(a); };
    constexpr int MOST = sizeof(T) == 4 ? 4 : 8;
    if (p.threads == 1024)
        launch(k_loss<T, 1, 1024>);
    else if (d_siblings && p.ct >= 64)
        p.v == 1 ? launch(k_loss_siblings<T, 1, 8>) : p.v == 4 ? launch(k_loss_siblings<T, 4, 8>) : launch(k_loss_siblings<T, MOST, 8>);
    else if (d_siblings)
        p.v == 1 ? launch(k_loss_siblings<T, 1, 32>) : p.v == 4 ? launch(k_loss_siblings<T, 4, 32>) : launch(k_loss_siblings<T, MOST, 32>);
    else if (p.v == 1)
        launch(k_loss<T, 1, 256>);
    else if (p.v == 4)
        launch(k_loss<T, 4, 256>);
    else
        launch(k_loss<T, MOST, 256>);
    HIP_TRY(hipGetLastError());
    if (join) {
        k_loss_join<<<(unsigned)ceil_div(a.k, 32), 1024, 0, st>>>(parts, (int)p.gx, a.k, d_loss);
        HIP_TRY(hipGetLastError());
    }
    return STAG_OK;
}

}  // namespace

extern "C" {

const char *stag_train_last_error(void) { return g_err; }

int64_t stag_row_scores_workspace(int64_t m, int32_t n_features, int32_t k, int32_t type) {
    TRY(check_rows(nullptr, 0, (((int64_t)n_features + 127) / 128) * 4, n_features, (const int32_t *)16, m, k, type));
    return product_plan(false, m, n_features, k, type).work_bytes;
}

int64_t stag_row_scores_grad_workspace(int64_t m, int32_t n_features, int32_t k, int32_t type) {
    TRY(check_rows(nullptr, 0, (((int64_t)n_features + 127) / 128) * 4, n_features, (const int32_t *)16, m, k, type));
    return product_plan(true, m, n_features, k, type).work_bytes;
}

int stag_row_scores_dev(const uint32_t *d_bits, int64_t n, int64_t row_stride, int32_t n_features, const int32_t *d_rows, int64_t m, const void *d_table,
                        int32_t type, int64_t table_stride, const float *d_bias, int32_t k, float scale, float *d_scores, int64_t score_stride,
                        void *d_work, int64_t work_bytes, void *stream) {
    TRY(check_rows(d_bits, n, row_stride, n_features, d_rows, m, k, type));
    TRY(check_matrix("d_table", d_table, type, table_stride, k));
    if (m == 0) return STAG_OK;
    TRY(check_matrix("d_scores", d_scores, STAG_F32, score_stride, k));
    REQUIRE(aligned(d_bias, 4), "d_bias is not aligned to its type");
    const Plan p = product_plan(false, m, n_features, k, type);
    REQUIRE(work_bytes >= p.work_bytes && (p.work_bytes == 0 || (d_work && aligned(d_work, 256))), "d_work: %lld bytes, 256-byte aligned, are wanted",
            (long long)p.work_bytes);
    ProductArgs a = {};
    a.bits = d_bits, a.n = n, a.row_stride = row_stride, a.rows = d_rows, a.m = m, a.n_features = n_features;
    a.mat = d_table, a.mat_stride = table_stride, a.bias = d_bias, a.k = k, a.scale = scale, a.out = d_scores, a.out_stride = score_stride;
    hipStream_t st = (hipStream_t)stream;
    switch (type) {
    case STAG_F32:
        return p.lookup ? lookup<float>(a, st) : product<STAG_F32, false>(p, a, d_work, st);
    case STAG_BF16:
        return p.lookup ? lookup<bf16>(a, st) : product<STAG_BF16, false>(p, a, d_work, st);
    default:
        return p.lookup ? lookup<f16>(a, st) : product<STAG_F16, false>(p, a, d_work, st);
    }
}

int stag_row_scores_grad_dev(const uint32_t *d_bits, int64_t n, int64_t row_stride, int32_t n_features, const int32_t *d_rows, int64_t m,
                             const void *d_grad, int32_t type, int64_t grad_stride, int32_t k, float scale, float *d_table_grad,
                             int64_t table_grad_stride, float *d_bias_grad, void *d_work, int64_t work_bytes, void *stream) {
    TRY(check_rows(d_bits, n, row_stride, n_features, d_rows, m, k, type));
    if (m > 0) TRY(check_matrix("d_grad", d_grad, type, grad_stride, k));
    if (d_table_grad) TRY(check_matrix("d_table_grad", d_table_grad, STAG_F32, table_grad_stride, k));
    REQUIRE(aligned(d_bias_grad, 4), "d_bias_grad is not aligned to its type");
    if (!d_table_grad && !d_bias_grad) return STAG_OK;
    const Plan p = product_plan(true, m, n_features, k, type);
    REQUIRE(work_bytes >= p.work_bytes && (p.work_bytes == 0 || (d_work && aligned(d_work, 256))), "d_work: %lld bytes, 256-byte aligned, are wanted",
            (long long)p.work_bytes);
    ProductArgs a = {};
    a.bits = d_bits, a.n = n, a.row_stride = row_stride, a.rows = d_rows, a.m = m, a.n_features = n_features;
    a.mat = d_grad, a.mat_stride = grad_stride, a.k = k, a.scale = scale, a.out = d_table_grad, a.out_stride = table_grad_stride, a.bias_out = d_bias_grad;
    hipStream_t st = (hipStream_t)stream;
    switch (type) {
    case STAG_F32:
        return product<STAG_F32, true>(p, a, d_work, st);
    case STAG_BF16:
        return product<STAG_BF16, true>(p, a, d_work, st);
    default:
        return product<STAG_F16, true>(p, a, d_work, st);
    }
}

int64_t stag_sibling_loss_workspace(int64_t m, int32_t k) {
    REQUIRE(m >= 0 && m < MAX_M, "m = %lld is not in 0..2^31-1", (long long)m);
    REQUIRE(k >= 1 && k <= MAX_K, "k = %d is not in 1..%d", k, MAX_K);
    unsigned most = 1;
    for (int v : {1, 4, 8}) {
        const unsigned gx = loss_plan(m, k, v, false).gx;      // siblings take no more
        if (gx > most) most = gx;
    }
    return most > 1 ? (int64_t)most * k * 4 : 0;
}

int stag_sibling_loss_dev(const float *d_scores, int64_t score_stride, int64_t m, int32_t k, const int32_t *d_label, const int32_t *d_siblings,
                          const float *d_weight, float scale, float *d_loss, void *d_grad, int32_t type, int64_t grad_stride, void *d_work,
                          int64_t work_bytes, void *stream) {
    REQUIRE(type_known(type), "unknown type %d", type);
    const int64_t need = stag_sibling_loss_workspace(m, k);
    if (need < 0) return (int)need;
    if (m > 0) {
        TRY(check_matrix("d_scores", d_scores, STAG_F32, score_stride, k));
        REQUIRE(d_label && aligned(d_label, 4), "d_label is null or not aligned to its type");
        REQUIRE(aligned(d_siblings, 4) && aligned(d_weight, 4) && aligned(d_loss, 4), "d_siblings, d_weight or d_loss is not aligned to its type");
        if (d_grad) TRY(check_matrix("d_grad", d_grad, type, grad_stride, k));
    }
    if (!d_loss && (!d_grad || m == 0)) return STAG_OK;
    REQUIRE(!d_loss || (work_bytes >= need && (need == 0 || (d_work && aligned(d_work, 256)))), "d_work: %lld bytes, 256-byte aligned, are wanted", (long long)need);
    // 16 bytes of gradient at once, if all rows of both matrices allow it
    auto fits = [&](int v) {
        return k % v == 0 && score_stride % v == 0 && aligned(d_scores, 16) && (!d_grad || (grad_stride % v == 0 && aligned(d_grad, v * type_bytes(type))));
    };
    const LossPlan p = loss_plan(m, k, type != STAG_F32 && fits(8) ? 8 : fits(4) ? 4 : 1, d_siblings != nullptr);
    LossArgs a = {};
    a.scores = d_scores, a.weight = d_weight, a.label = d_label, a.siblings = d_siblings, a.loss = d_loss, a.grad = d_grad;
    a.score_stride = score_stride, a.grad_stride = grad_stride, a.m = m, a.k = k, a.scale = scale;
    hipStream_t st = (hipStream_t)stream;
    switch (type) {
    case STAG_F32:
        return loss_typed<float>(p, a, (float *)d_work, st);
    case STAG_BF16:
        return loss_typed<bf16>(p, a, (float *)d_work, st);
    default:
        return loss_typed<f16>(p, a, (float *)d_work, st);
    }
}

int stag_adamw_dev(const stag_adamw_tensor_t *d_tensors, const stag_adamw_tile_t *d_tiles, int64_t n_tiles, int32_t state_bits, void *d_m, void *d_v,
                   float *d_m_scale, float *d_v_scale, int32_t *d_step, double lr, double beta1, double beta2, double eps, void *stream) {
    REQUIRE(state_bits == 32 || state_bits == 8, "state_bits = %d: 32 or 8 are wanted", state_bits);
    REQUIRE(n_tiles >= 0 && n_tiles < (int64_t)1 << 40, "n_tiles = %lld", (long long)n_tiles);
    REQUIRE(lr >= 0 && std::isfinite(lr), "lr = %g", lr);
    REQUIRE(beta1 > 0 && beta1 < 1 && beta2 > 0 && beta2 < 1, "beta1 = %g, beta2 = %g: not inside (0, 1)", beta1, beta2);
    REQUIRE(eps >= 0 && std::isfinite(eps), "eps = %g", eps);
    REQUIRE(d_step && aligned(d_step, 4), "d_step is null or not aligned");
    if (n_tiles > 0) {
        REQUIRE(d_tensors && d_tiles && aligned(d_tensors, 8) && aligned(d_tiles, 8), "d_tensors or d_tiles is null or not aligned");
        REQUIRE(d_m && d_v && aligned(d_m, 16) && aligned(d_v, 16), "d_m or d_v is null or not 16-byte aligned");
        REQUIRE(state_bits == 32 || (d_m_scale && d_v_scale && aligned(d_m_scale, 4) && aligned(d_v_scale, 4)), "8-bit states have scales");
    }
    AdamwArgs a;
    a.tensors = d_tensors;
    a.tiles = d_tiles;
    a.n_tiles = n_tiles;
    a.m = d_m;
    a.v = d_v;
    a.m_scale = d_m_scale;
    a.v_scale = d_v_scale;
    a.step = d_step;
    a.lr = (float)lr;
    a.beta1 = (float)beta1;
    a.beta2 = (float)beta2;
    a.one_minus_beta1 = (float)(1.0 - beta1);
    a.one_minus_beta2 = (float)(1.0 - beta2);
    a.log_beta1 = (float)std::log(beta1);
    a.log_beta2 = (float)std::log(beta2);
    a.eps = (float)eps;
    a.split = n_tiles <= 2048 ? 4 : 1;
    const int64_t waves = n_tiles * a.split;
    // A tile a wave with 32-bit states; with 8-bit ones a few, since a wave's start costs as much as half a tile's arithmetic (1,600
    // tables, up to 4,096, 8,192, 16,384 workgroups: 270, 259, 254 us and 133, 125, 131).  A step of nothing is counted too.
    const int64_t most = state_bits == 32 ? 1 << 20 : 8192;
    const unsigned grid = (unsigned)(waves < 4 * most ? ceil_div(waves + (waves == 0), 4) : most);
    if (state_bits == 32)
        k_adamw<32><<<grid, 256, 0, (hipStream_t)stream>>>(a);
    else
        k_adamw<8><<<grid, 256, 0, (hipStream_t)stream>>>(a);
    HIP_TRY(hipGetLastError());
    return STAG_OK;
}

}  // extern "C"
