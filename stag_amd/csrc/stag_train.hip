// libstag_train.so: C ABI (include/stag_train.h) and kernels of the operators that learn node classifiers.
// gfx950 only; no CPU fallback.
#include "stag_train.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>

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

template <int TYPE> struct Of;
template <> struct Of<STAG_F32> { typedef float type; };
template <> struct Of<STAG_BF16> { typedef bf16 type; };
template <> struct Of<STAG_F16> { typedef f16 type; };

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
// one thread per score
template <typename T>
__global__ __launch_bounds__(256) void k_scores(const uint32_t *bits, int64_t n, int64_t row_stride, int n_features, const int32_t *rows,
                                                int64_t m, const T *table, int64_t table_stride, const float *bias, int k,
                                                float scale, float *scores, int64_t score_stride) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= m * k) return;
    const int64_t i = at / k;
    const int c = (int)(at - i * k);
    const uint32_t *row = row_of(bits, n, row_stride, rows, i);
    float s = 0.f;
    if (row) {
        for (int w = 0; 32 * w < n_features; ++w) {
            float part = 0.f;
            for (uint32_t x = row[w]; x; x &= x - 1) {
                const int f = 32 * w + __builtin_ctz(x);
                if (f < n_features) part += (float)table[(int64_t)f * table_stride + c];
            }
            s += part;
        }
        s = s * scale + (bias ? bias[c] : 0.f);
    }
    scores[i * score_stride + c] = s;
}

// one thread per coefficient; feature n_features stands for the bias, which every row has
template <typename T>
__global__ __launch_bounds__(256) void k_grad(const uint32_t *bits, int64_t n, int64_t row_stride, int n_features, const int32_t *rows,
                                              int64_t m, const T *grad, int64_t grad_stride, int k, float scale, float *table_grad,
                                              int64_t table_grad_stride, float *bias_grad) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= ((int64_t)n_features + 1) * k) return;
    const int f = (int)(at / k), c = (int)(at - (int64_t)f * k);
    float s = 0.f, part = 0.f;
    for (int64_t i = 0; i < m; ++i) {
        const uint32_t *row = row_of(bits, n, row_stride, rows, i);
        if (row && (f == n_features || (row[f >> 5] >> (f & 31) & 1u))) part += (float)grad[i * grad_stride + c];
        if ((i & 31) == 31) {
            s += part;
            part = 0.f;
        }
    }
    s += part;
    if (f < n_features) {
        if (table_grad) table_grad[(int64_t)f * table_grad_stride + c] = s * scale;
    } else if (bias_grad) {
        bias_grad[c] = s;
    }
}

// ------------------------------------------------------------------------------------------------------------------
// loss of siblings
// ------------------------------------------------------------------------------------------------------------------
// A thread owns V neighbouring columns and goes down the rows of its workgroup; loss sums stay in its registers until the
// workgroup adds them up in a fixed order and stores one partial row of K sums.  Scores are read only where the row
// trains (a place of the tree has a handful of siblings among the thousands of a level); the rest of the gradient is
// zeros, so what bounds a level's loss is writing the gradient.
template <typename T, int V>
__global__ __launch_bounds__(256) void k_loss(const float *scores, int64_t score_stride, int64_t m, int k, const int32_t *label,
                                              const int32_t *siblings, const float *weight, float scale, float *loss, T *grad,
                                              int64_t grad_stride, int ct) {
    __shared__ float part[256 * V];
    const int cv = threadIdx.x % ct, r = threadIdx.x / ct, rp = 256 / ct;
    const int c0 = (blockIdx.y * ct + cv) * V;
    float sum[V] = {};
    if (r < rp && c0 < k) {
        for (int64_t i = (int64_t)blockIdx.x * rp + r; i < m; i += (int64_t)gridDim.x * rp) {
            int lo = 0, hi = k;
            if (siblings) {
                lo = siblings[2 * i];
                hi = siblings[2 * i + 1];
            }
            float g[V] = {};
            if (c0 + V > lo && c0 < hi) {
                const int lab = label[i];
                const float w = scale * (weight ? weight[i] : 1.f);
                const float *src = scores + i * score_stride + c0;
                float z[V];
                if constexpr (V == 4) {
                    const float4 q = *(const float4 *)src;
                    z[0] = q.x, z[1] = q.y, z[2] = q.z, z[3] = q.w;
                } else {
                    z[0] = src[0];
                }
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const int c = c0 + j;
                    if (c < lo || c >= hi) continue;
                    const float s = c == lab ? -z[j] : z[j];
                    const float e = expf(-fabsf(s));
                    sum[j] += w * ((s < 0.f ? 0.f : s) + log1pf(e));      // softplus(s); NaN stays NaN
                    const float p = (s >= 0.f ? 1.f : e) / (1.f + e) * w;  // sigmoid(s)
                    g[j] = c == lab ? -p : p;
                }
            }
            if (grad) {
                T *dst = grad + i * grad_stride + c0;
                if constexpr (V == 4) {
                    T out[4] = {(T)g[0], (T)g[1], (T)g[2], (T)g[3]};
                    if constexpr (sizeof(T) == 4)
                        *(float4 *)dst = *(const float4 *)out;
                    else
                        *(uint2 *)dst = *(const uint2 *)out;
                } else {
                    dst[0] = (T)g[0];
                }
            }
        }
    }
    if (!loss) return;
#pragma unroll
    for (int j = 0; j < V; ++j) part[threadIdx.x * V + j] = sum[j];
    __syncthreads();
    if (r == 0 && c0 < k) {
        for (int j = 0; j < V; ++j) {
            float s = 0.f;
            for (int q = 0; q < rp; ++q) s += part[(q * ct + cv) * V + j];
            loss[(int64_t)blockIdx.x * k + c0 + j] = s;
        }
    }
}

__global__ __launch_bounds__(256) void k_loss_join(const float *part, int n_parts, int k, float *loss) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= k) return;
    double s = 0.0;
    for (int p = 0; p < n_parts; ++p) s += part[(int64_t)p * k + c];
    loss[c] = (float)s;
}

// ------------------------------------------------------------------------------------------------------------------
// AdamW over many tensors
// ------------------------------------------------------------------------------------------------------------------
struct AdamwArgs {
    const stag_adamw_tensor_t *tensors;
    const stag_adamw_tile_t *tiles;
    int64_t n_tiles;
    void *m, *v;
    float *m_scale, *v_scale;
    int32_t *step;
    float lr, beta1, beta2, one_minus_beta1, one_minus_beta2, log_beta1, log_beta2, eps;
};

__device__ __forceinline__ float4 load4(const void *p, int type, int64_t at, int64_t count, bool whole) {
    float x[4];
    if (whole) {
        if (type == STAG_F32) return *(const float4 *)((const float *)p + at);
        const uint2 q = *(const uint2 *)((const uint16_t *)p + at);
        const uint32_t h[4] = {q.x & 0xffffu, q.x >> 16, q.y & 0xffffu, q.y >> 16};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            x[j] = type == STAG_BF16 ? __uint_as_float(h[j] << 16) : (float)__builtin_bit_cast(f16, (uint16_t)h[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[j] = 0.f;
            if (at + j < count)
                x[j] = type == STAG_F32 ? ((const float *)p)[at + j] : type == STAG_BF16 ? (float)((const bf16 *)p)[at + j]
                                                                                         : (float)((const f16 *)p)[at + j];
        }
    }
    return make_float4(x[0], x[1], x[2], x[3]);
}

__device__ __forceinline__ void store4(void *p, int type, int64_t at, int64_t count, bool whole, const float *x) {
    uint16_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = type == STAG_BF16 ? __builtin_bit_cast(uint16_t, (bf16)x[j]) : __builtin_bit_cast(uint16_t, (f16)x[j]);
    if (whole) {
        if (type == STAG_F32)
            *(float4 *)((float *)p + at) = make_float4(x[0], x[1], x[2], x[3]);
        else
            *(uint2 *)((uint16_t *)p + at) = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (at + j < count) {
                if (type == STAG_F32)
                    ((float *)p)[at + j] = x[j];
                else
                    ((uint16_t *)p)[at + j] = h[j];
            }
    }
}

// The exponent (biased) of the smallest power of two s with max|x| <= 448 s over the wave's 256 values; 448 = 1.75 * 2^8 is
// the largest e4m3 value.  A power of two, so that dividing by it rounds nothing.  Infinities and NaN have no say.
__device__ __forceinline__ int scale_exponent(const float *x) {
    int top = 10 << 23;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int a = __float_as_int(x[j]) & 0x7fffffff;
        if (a < 0x7f800000) top = max(top, a);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) top = max(top, __shfl_xor(top, o));
    return (top >> 23) - 8 + ((top & 0x7fffff) > 0x600000);
}

// x / s as the value of an e4m3 code, up or down by `chance` (16 bits).  From 2^-6 on a code has 3 bits behind the leading
// one: adding 20 random bits below them and cutting them off goes up with the probability of what is cut; below, codes
// are 2^-9 apart.
__device__ __forceinline__ float rounded(float x, float inv, uint32_t chance) {
#pragma clang fp contract(off)
    const float y = x * inv, a = fabsf(y);
    const float normal = __uint_as_float((__float_as_uint(a) + (chance << 4 | 8u)) & 0xfff00000u);
    const float small = floorf(a * 512.f + ((float)chance + 0.5f) * 0x1p-16f) * 0x1p-9f;
    return copysignf(a < 0x1p-6f ? small : normal, y);
}

__device__ __forceinline__ uint32_t pack_e4m3(const float *x) {
    int q = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], q, true);
}

__device__ __forceinline__ void unpack_e4m3(uint32_t q, float *x) {
    x[0] = __builtin_amdgcn_cvt_f32_fp8((int)q, 0);
    x[1] = __builtin_amdgcn_cvt_f32_fp8((int)q, 1);
    x[2] = __builtin_amdgcn_cvt_f32_fp8((int)q, 2);
    x[3] = __builtin_amdgcn_cvt_f32_fp8((int)q, 3);
}

// A wave takes a tile of four blocks of 256 values, four neighbouring values a lane.  Everything is read once and written
// once; what bounds it is HBM.  m, v and the root are rounded after every operation (no fused multiply-add), so that the 8-bit codes are a
// function of the inputs that any other 32-bit implementation can restate.
template <int BITS>
__global__ __launch_bounds__(256) void k_adamw(AdamwArgs a) {
#pragma clang fp contract(off)
    const int lane = threadIdx.x & 63;
    const int t = __hip_atomic_load(a.step, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1;
    // 1 - beta^t = -expm1(t log beta)
    const float c1 = a.lr / -expm1f((float)t * a.log_beta1);
    const float c2 = 1.f / sqrtf(-expm1f((float)t * a.log_beta2));
    const uint32_t salt = (uint32_t)t * 0x9E3779B9u;
    for (int64_t w = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); w < a.n_tiles; w += (int64_t)gridDim.x * 4) {
        const stag_adamw_tile_t tile = a.tiles[w];
        const stag_adamw_tensor_t d = a.tensors[tile.tensor];
        const int64_t at0 = (int64_t)tile.tile * STAG_ADAMW_TILE + lane * 4;
        const int vec_p = ((uintptr_t)d.param & (d.param_type == STAG_F32 ? 15 : 7)) == 0;
        const int vec_g = ((uintptr_t)d.grad & (d.grad_type == STAG_F32 ? 15 : 7)) == 0;
        const float keep = 1.f - a.lr * d.weight_decay, shrink = a.lr * d.l1;
#pragma unroll
        for (int b = 0; b < STAG_ADAMW_TILE / 256; ++b) {
            const int64_t at = at0 + b * 256, s = d.state_at + at;
            if (at - lane * 4 >= d.count) break;
            const bool full = at + 4 <= d.count;
            const float4 p4 = load4(d.param, d.param_type, at, d.count, full && vec_p);
            const float4 g4 = load4(d.grad, d.grad_type, at, d.count, full && vec_g);
            float p[4] = {p4.x, p4.y, p4.z, p4.w}, g[4] = {g4.x, g4.y, g4.z, g4.w}, m[4], v[4], root[4];
            if constexpr (BITS == 32) {
                const float4 m4 = *(const float4 *)((const float *)a.m + s), v4 = *(const float4 *)((const float *)a.v + s);
                m[0] = m4.x, m[1] = m4.y, m[2] = m4.z, m[3] = m4.w;
                v[0] = v4.x, v[1] = v4.y, v[2] = v4.z, v[3] = v4.w;
            } else {
                unpack_e4m3(*(const uint32_t *)((const uint8_t *)a.m + s), m);
                unpack_e4m3(*(const uint32_t *)((const uint8_t *)a.v + s), v);
                const float ms = a.m_scale[s >> 8], vs = a.v_scale[s >> 8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    m[j] = m[j] * ms;
                    v[j] = v[j] * vs;
                    v[j] = v[j] * v[j];
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (at + j >= d.count) m[j] = v[j] = 0.f;      // places between tensors hold nothing
                m[j] = m[j] * a.beta1 + g[j] * a.one_minus_beta1;
                v[j] = v[j] * a.beta2 + (g[j] * g[j]) * a.one_minus_beta2;
                root[j] = sqrtf(v[j]);
                const float r = __builtin_amdgcn_rcpf(root[j] * c2 + a.eps);
                p[j] = p[j] * keep - c1 * m[j] * r;
                const float left = fabsf(p[j]) - shrink * r;
                if (shrink > 0.f) p[j] = copysignf(left < 0.f ? 0.f : left, p[j]);
            }
            store4(d.param, d.param_type, at, d.count, full && vec_p, p);
            if constexpr (BITS == 32) {
                *(float4 *)((float *)a.m + s) = make_float4(m[0], m[1], m[2], m[3]);
                *(float4 *)((float *)a.v + s) = make_float4(v[0], v[1], v[2], v[3]);
            } else {
                const int me = scale_exponent(m), ve = scale_exponent(root);
                const float mi = __int_as_float((254 - me) << 23), vi = __int_as_float((254 - ve) << 23);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t x = (uint32_t)(s + j) ^ salt;
                    x = (x ^ x >> 16) * 0x7FEB352Du;
                    x = (x ^ x >> 15) * 0x846CA68Bu;
                    x ^= x >> 16;
                    m[j] = rounded(m[j], mi, x >> 16);
                    const float q = rounded(root[j], vi, x & 0xffffu);
                    v[j] = root[j] > 0.f && q == 0.f ? 0x1p-9f : q;      // a root of zero would divide by eps alone: what is not zero stays so
                }
                *(uint32_t *)((uint8_t *)a.m + s) = pack_e4m3(m);
                *(uint32_t *)((uint8_t *)a.v + s) = pack_e4m3(v);
                if (lane == 0) {
                    a.m_scale[s >> 8] = __int_as_float(me << 23);
                    a.v_scale[s >> 8] = __int_as_float(ve << 23);
                }
            }
        }
    }
    // the last workgroup to come here, when all have read t, counts the step
    __syncthreads();
    if (threadIdx.x == 0) {
        const int before = __hip_atomic_fetch_add(a.step + 1, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        if (before == (int)gridDim.x - 1) {
            __hip_atomic_store(a.step + 1, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(a.step, t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------------------------
constexpr int64_t MAX_M = (int64_t)1 << 31;      // rows of a batch
constexpr int32_t MAX_K = 1 << 20;               // classifiers of a table
constexpr int32_t MAX_FEATURES = 1 << 27;

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
    return STAG_OK;
}

#define TRY(expr)                 \
    do {                          \
        const int rc_ = (expr);   \
        if (rc_ != STAG_OK) return rc_; \
    } while (0)

template <typename T>
int scores_typed(const uint32_t *d_bits, int64_t n, int64_t row_stride, int32_t n_features, const int32_t *d_rows, int64_t m, const void *d_table,
                 int64_t table_stride, const float *d_bias, int32_t k, float scale, float *d_scores, int64_t score_stride, hipStream_t st) {
    REQUIRE(m * k < (int64_t)1 << 39, "m * k is too large");
    k_scores<T><<<(unsigned)ceil_div(m * k, 256), 256, 0, st>>>(d_bits, n, row_stride, n_features, d_rows, m, (const T *)d_table, table_stride, d_bias, k,
                                                               scale, d_scores, score_stride);
    HIP_TRY(hipGetLastError());
    return STAG_OK;
}

template <typename T>
int grad_typed(const uint32_t *d_bits, int64_t n, int64_t row_stride, int32_t n_features, const int32_t *d_rows, int64_t m, const void *d_grad,
               int64_t grad_stride, int32_t k, float scale, float *d_table_grad, int64_t table_grad_stride, float *d_bias_grad, hipStream_t st) {
    const int64_t blocks = ceil_div(((int64_t)n_features + 1) * k, 256);
    REQUIRE(blocks < (int64_t)1 << 31, "n_features * k is too large");
    k_grad<T><<<(unsigned)blocks, 256, 0, st>>>(d_bits, n, row_stride, n_features, d_rows, m, (const T *)d_grad, grad_stride, k, scale, d_table_grad,
                                               table_grad_stride, d_bias_grad);
    HIP_TRY(hipGetLastError());
    return STAG_OK;
}

// how k_loss is laid over [m][k]
struct LossPlan {
    int v, ct;
    unsigned gx, gy;
};

LossPlan loss_plan(int64_t m, int32_t k, bool vectors) {
    LossPlan p;
    p.v = vectors ? 4 : 1;
    const int64_t cols = ceil_div(k, p.v);
    p.ct = (int)(cols < 256 ? cols : 256);
    p.gy = (unsigned)ceil_div(cols, p.ct);
    const int64_t passes = ceil_div(m, 256 / p.ct), wanted = 2048 / p.gy > 0 ? 2048 / p.gy : 1;
    // few values: one workgroup a column tile, whose sums are the result without a second launch
    p.gx = (unsigned)(m * (int64_t)k <= 16384 ? 1 : passes < wanted ? passes : wanted);
    return p;
}

template <typename T>
int loss_typed(const LossPlan &p, const float *d_scores, int64_t score_stride, int64_t m, int32_t k, const int32_t *d_label, const int32_t *d_siblings,
               const float *d_weight, float scale, float *d_loss, void *d_grad, int64_t grad_stride, float *parts, hipStream_t st) {
    float *to = d_loss && p.gx > 1 ? parts : d_loss;
    const dim3 grid(p.gx, p.gy);
    if (p.v == 4)
        k_loss<T, 4><<<grid, 256, 0, st>>>(d_scores, score_stride, m, k, d_label, d_siblings, d_weight, scale, to, (T *)d_grad, grad_stride, p.ct);
    else
        k_loss<T, 1><<<grid, 256, 0, st>>>(d_scores, score_stride, m, k, d_label, d_siblings, d_weight, scale, to, (T *)d_grad, grad_stride, p.ct);
    HIP_TRY(hipGetLastError());
    if (d_loss && p.gx > 1) {
        k_loss_join<<<(unsigned)ceil_div(k, 256), 256, 0, st>>>(parts, (int)p.gx, k, d_loss);
        HIP_TRY(hipGetLastError());
    }
    return STAG_OK;
}

}  // namespace

extern "C" {

const char *stag_train_last_error(void) { return g_err; }

int64_t stag_row_scores_workspace(int64_t m, int32_t n_features, int32_t k, int32_t type) {
    TRY(check_rows(nullptr, 0, (((int64_t)n_features + 127) / 128) * 4, n_features, (const int32_t *)16, m, k, type));
    return 0;
}

int64_t stag_row_scores_grad_workspace(int64_t m, int32_t n_features, int32_t k, int32_t type) {
    TRY(check_rows(nullptr, 0, (((int64_t)n_features + 127) / 128) * 4, n_features, (const int32_t *)16, m, k, type));
    return 0;
}

int stag_row_scores_dev(const uint32_t *d_bits, int64_t n, int64_t row_stride, int32_t n_features, const int32_t *d_rows, int64_t m, const void *d_table,
                        int32_t type, int64_t table_stride, const float *d_bias, int32_t k, float scale, float *d_scores, int64_t score_stride,
                        void *d_work, int64_t work_bytes, void *stream) {
    TRY(check_rows(d_bits, n, row_stride, n_features, d_rows, m, k, type));
    TRY(check_matrix("d_table", d_table, type, table_stride, k));
    if (m == 0) return STAG_OK;
    TRY(check_matrix("d_scores", d_scores, STAG_F32, score_stride, k));
    REQUIRE(aligned(d_bias, 4), "d_bias is not aligned to its type");
    const int64_t need = stag_row_scores_workspace(m, n_features, k, type);
    REQUIRE(work_bytes >= need && (need == 0 || (d_work && aligned(d_work, 256))), "d_work: %lld bytes, 256-byte aligned, are wanted", (long long)need);
    hipStream_t st = (hipStream_t)stream;
    switch (type) {
    case STAG_F32:
        return scores_typed<float>(d_bits, n, row_stride, n_features, d_rows, m, d_table, table_stride, d_bias, k, scale, d_scores, score_stride, st);
    case STAG_BF16:
        return scores_typed<bf16>(d_bits, n, row_stride, n_features, d_rows, m, d_table, table_stride, d_bias, k, scale, d_scores, score_stride, st);
    default:
        return scores_typed<f16>(d_bits, n, row_stride, n_features, d_rows, m, d_table, table_stride, d_bias, k, scale, d_scores, score_stride, st);
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
    const int64_t need = stag_row_scores_grad_workspace(m, n_features, k, type);
    REQUIRE(work_bytes >= need && (need == 0 || (d_work && aligned(d_work, 256))), "d_work: %lld bytes, 256-byte aligned, are wanted", (long long)need);
    hipStream_t st = (hipStream_t)stream;
    switch (type) {
    case STAG_F32:
        return grad_typed<float>(d_bits, n, row_stride, n_features, d_rows, m, d_grad, grad_stride, k, scale, d_table_grad, table_grad_stride, d_bias_grad, st);
    case STAG_BF16:
        return grad_typed<bf16>(d_bits, n, row_stride, n_features, d_rows, m, d_grad, grad_stride, k, scale, d_table_grad, table_grad_stride, d_bias_grad, st);
    default:
        return grad_typed<f16>(d_bits, n, row_stride, n_features, d_rows, m, d_grad, grad_stride, k, scale, d_table_grad, table_grad_stride, d_bias_grad, st);
    }
}

int64_t stag_sibling_loss_workspace(int64_t m, int32_t k) {
    REQUIRE(m >= 0 && m < MAX_M, "m = %lld is not in 0..2^31-1", (long long)m);
    REQUIRE(k >= 1 && k <= MAX_K, "k = %d is not in 1..%d", k, MAX_K);
    const unsigned a = loss_plan(m, k, true).gx, b = loss_plan(m, k, false).gx, most = a > b ? a : b;
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
    const bool vectors = k % 4 == 0 && score_stride % 4 == 0 && aligned(d_scores, 16) && (!d_grad || (grad_stride % 4 == 0 && aligned(d_grad, 4 * type_bytes(type))));
    const LossPlan p = loss_plan(m, k, vectors);
    hipStream_t st = (hipStream_t)stream;
    float *parts = (float *)d_work;
    switch (type) {
    case STAG_F32:
        return loss_typed<float>(p, d_scores, score_stride, m, k, d_label, d_siblings, d_weight, scale, d_loss, d_grad, grad_stride, parts, st);
    case STAG_BF16:
        return loss_typed<bf16>(p, d_scores, score_stride, m, k, d_label, d_siblings, d_weight, scale, d_loss, d_grad, grad_stride, parts, st);
    default:
        return loss_typed<f16>(p, d_scores, score_stride, m, k, d_label, d_siblings, d_weight, scale, d_loss, d_grad, grad_stride, parts, st);
    }
}

int stag_adamw_dev(const stag_adamw_tensor_t *d_tensors, const stag_adamw_tile_t *d_tiles, int64_t n_tiles, int32_t state_bits, void *d_m, void *d_v,
                   float *d_m_scale, float *d_v_scale, int32_t *d_step, double lr, double beta1, double beta2, double eps, void *stream) {
    REQUIRE(state_bits == 32 || state_bits == 8, "state_bits = %d: 32 or 8 are wanted", state_bits);
    REQUIRE(n_tiles >= 0 && n_tiles < (int64_t)1 << 40, "n_tiles = %lld", (long long)n_tiles);
    REQUIRE(lr >= 0 && std::isfinite(lr), "lr = %g", lr);
    REQUIRE(beta1 > 0 && beta1 < 1 && beta2 > 0 && beta2 < 1, "beta1 = %g, beta2 = %g: not inside (0, 1)", beta1, beta2);
    REQUIRE(eps >= 0 && std::isfinite(eps), "eps = %g", eps);
    if (n_tiles == 0) return STAG_OK;
    REQUIRE(d_tensors && d_tiles && d_step && aligned(d_tensors, 8) && aligned(d_tiles, 8) && aligned(d_step, 4), "d_tensors, d_tiles or d_step is null or not aligned");
    REQUIRE(d_m && d_v && aligned(d_m, 16) && aligned(d_v, 16), "d_m or d_v is null or not 16-byte aligned");
    REQUIRE(state_bits == 32 || (d_m_scale && d_v_scale && aligned(d_m_scale, 4) && aligned(d_v_scale, 4)), "8-bit states have scales");
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
    const unsigned grid = (unsigned)(n_tiles < 4 * 2048 ? ceil_div(n_tiles, 4) : 2048);
    if (state_bits == 32)
        k_adamw<32><<<grid, 256, 0, (hipStream_t)stream>>>(a);
    else
        k_adamw<8><<<grid, 256, 0, (hipStream_t)stream>>>(a);
    HIP_TRY(hipGetLastError());
    return STAG_OK;
}

}  // extern "C"
