// Shared pieces of the fine-tuning operators (matmul.hip, finetune.hip): the counter-based dropout
// generator, the activations with their derivatives and the epilogue of a matrix product.
#pragma once
#include <type_traits>

#include "common.h"

namespace clipvit {

// ---- dropout ----
// Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2, 3",
// SC 2011): ten rounds of two 32 x 32 -> 64-bit products on a 128-bit counter. The counter of element
// (row m, column n) is (n / 4, m, offset), its word n % 4, the key is the 64-bit seed, so the mask is a
// function of the element's place and never stored: the backward pass computes it again. An element is
// kept when its word exceeds `drop_max` = round(p 2^32) - 1 (so p = 1 keeps nothing).
struct Dropout {
    unsigned k0, k1;         // seed
    unsigned o0, o1;         // offset (when offset_dev is null)
    const uint2* offset_dev; // offset read on the device: a captured graph draws a new mask per replay
    unsigned drop_max;
    float scale;             // 1 / (1 - p), 0 for p = 1
    int on;                  // 0: no dropout (p rounds to 0)
};

__device__ __forceinline__ uint4 philox4(unsigned quad, unsigned row, unsigned o0, unsigned o1, unsigned k0, unsigned k1) {
    unsigned c0 = quad, c1 = row, c2 = o0, c3 = o1;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = (unsigned)(b >> 32) ^ c1 ^ k0;
        c1 = (unsigned)b;
        c2 = (unsigned)(a >> 32) ^ c3 ^ k1;
        c3 = (unsigned)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}
__device__ __forceinline__ uint2 drop_offset(const Dropout& d) {
    return d.offset_dev ? *d.offset_dev : make_uint2(d.o0, d.o1);
}
// four consecutive columns (n % 4 == 0) of row m: kept values scaled, dropped ones exactly 0 (whatever
// they held, NaN included)
__device__ __forceinline__ void drop4(const Dropout& d, const uint2& o, int m, int n, float scale, float& a, float& b, float& c, float& e) {
    const uint4 w = philox4((unsigned)n >> 2, (unsigned)m, o.x, o.y, d.k0, d.k1);
    a = w.x > d.drop_max ? a * scale : 0.f;
    b = w.y > d.drop_max ? b * scale : 0.f;
    c = w.z > d.drop_max ? c * scale : 0.f;
    e = w.w > d.drop_max ? e * scale : 0.f;
}

// ---- activations ----
// z Phi-like gates: quick_gelu z s(1.702 z), silu z s(z) (s the logistic function by v_exp_f32 and
// v_rcp_f32: relative error a few 2^-23), gelu z (1 + erf(z / sqrt 2)) / 2, gelu_tanh with the tanh written
// as a logistic: (1 + tanh t) / 2 = s(2 t).
enum Act { ACT_NONE = 0, ACT_QUICK_GELU = 1, ACT_GELU = 2, ACT_GELU_TANH = 3, ACT_SILU = 4, ACT_RELU = 5 };

__device__ __forceinline__ float logistic(float t) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * t));
}
// value and derivative; the derivative's z factors are clamped so that it reaches its limit (0 or 1) at
// +-inf instead of inf * 0 (a NaN z gives NaN through the gate)
template <bool SLOPE, int ACT>
__device__ __forceinline__ float act_one(float beta, float z, float& slope) {
    const float zc = SLOPE ? fminf(fmaxf(z, -100.f), 100.f) : z;
    if constexpr (ACT == ACT_SILU) {  // also quick_gelu: beta 1.702
        const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(beta * z));  // beta = -log2(e) beta
        if (SLOPE) slope = s * (1.0f - 0.69314718055994531f * beta * zc * (1.0f - s));
        return z * s;
    } else if constexpr (ACT == ACT_GELU) {
        // Phi(-|z|) = t P(t) e^(-z^2 / 2), t = 1 / (1 + 0.29 |z|), P of degree 5 fitted for |z| <= 14 (minimax, linear
        // programme) to 7.1e-8 absolute and 2^-13.5 relative: the tail has to keep its leading digits for bf16, which holds
        // it. Evaluated in fp32 it is off by at most 2.3e-7 near 0 and 2^-13.4 relative. It shares the exponential with the
        // derivative (erff and its own exponential: 70 instructions an element against 30, 4928 x 512 x 2048 with the
        // derivative 52 us against 38).
        const float az = fabsf(z), t = __builtin_amdgcn_rcpf(1.0f + 0.29f * az);
        const float e = __builtin_amdgcn_exp2f(-0.72134752044448170f * az * az);
        const float q = t * (0.116854535f + t * (0.100881662f + t * (0.178990770f + t * (-0.0923373715f + t * (0.284243027f + t * -0.0886325613f))))) * e;
        const float c = z < 0.f ? q : 1.0f - q;
        if (SLOPE) slope = c + 0.39894228040143268f * zc * e;
        return z * c;
    } else if constexpr (ACT == ACT_GELU_TANH) {
        const float s = logistic(1.5957691216057308f * (z + 0.044715f * z * (z * z)));
        if (SLOPE) slope = s + zc * s * (1.0f - s) * (1.5957691216057308f * (1.0f + 0.134145f * (zc * zc)));
        return z * s;
    } else {
        if (SLOPE) slope = z != z ? z : (z > 0.f ? 1.f : 0.f);
        return z != z ? z : fmaxf(z, 0.f);
    }
}
// C values at once: one uniform branch on the kind, not one an element
template <bool SLOPE, int C>
__device__ __forceinline__ void act_cols(int act, float (&v)[C], float (&g)[C]) {
    if (act == ACT_QUICK_GELU || act == ACT_SILU) {
        const float beta = act == ACT_SILU ? -1.4426950408889634f : -2.4554669595930157f;
#pragma unroll
        for (int j = 0; j < C; ++j) v[j] = act_one<SLOPE, ACT_SILU>(beta, v[j], g[j]);
    } else if (act == ACT_GELU) {
#pragma unroll
        for (int j = 0; j < C; ++j) v[j] = act_one<SLOPE, ACT_GELU>(0.f, v[j], g[j]);
    } else if (act == ACT_GELU_TANH) {
#pragma unroll
        for (int j = 0; j < C; ++j) v[j] = act_one<SLOPE, ACT_GELU_TANH>(0.f, v[j], g[j]);
    } else {
#pragma unroll
        for (int j = 0; j < C; ++j) v[j] = act_one<SLOPE, ACT_RELU>(0.f, v[j], g[j]);
    }
}
// The derivative as the forward saves it: sign and 15 bits of magnitude, all of these derivatives lying in (-0.13, 1.13).
// From 2^(M - 14) up the magnitude is fixed point in steps of 2^-14; below it is a float of M mantissa bits, whose steps
// join those: off by at most 2^-15 absolute and 2^-(M + 1) relative. bf16 operands: M = 7, half a bf16 step (2^-8), down to
// 2^-118; fp16 operands: M = 9, half of 2^-9, down to 2^-33, under what an fp16 dz resolves (2^-24 for |dy| up to 2^8); less
// is 0. (Fixed point alone loses the derivative of a saturated unit altogether: quick_gelu is 9 % off at z = -6 and 0 past
// -7.6. A plain 16-bit float is as far off near 1 as dz's own rounding is.) 0x7fff stands for NaN.
template <typename T>
struct SlopeCode {
    static constexpr int M = std::is_same<T, BF16>::value ? 7 : 9, LOW = std::is_same<T, BF16>::value ? -118 : -33;
    static constexpr unsigned OFF = ((127 + LOW) << M) - 1;          // float bits >> (23 - M) minus this: 1 at 2^LOW
    static constexpr unsigned JOIN = ((M - 14 - LOW) << M) + 1;      // code of 2^(M - 14)
    // 512 + magnitude is a float in steps of 2^-14: its bits minus this are the fixed-point part's codes
    static constexpr unsigned FIXED = 0x44000000u - (JOIN - (1u << M));
    static_assert(JOIN - (1u << M) + 18678 < 0x7fff, "1.14, more than any magnitude, stays below NaN");
    static __device__ __forceinline__ short encode(float g) {
        const unsigned bits = __float_as_uint(g), mag = bits & 0x7fffffffu;
        const float a = __uint_as_float(mag);
        const unsigned fixed = __float_as_uint(a + 512.f) - FIXED;
        const unsigned tail = __builtin_elementwise_sub_sat(mag, (OFF << (23 - M)) - (1u << (22 - M))) >> (23 - M);
        const unsigned m = min(a < 1.0f / (1 << (14 - M)) ? tail : fixed, 0x7fffu);
        return (short)(m | (bits >> 16 & 0x8000u));
    }
    static __device__ __forceinline__ float decode(short q) {
        const unsigned m = q & 0x7fff;
        const float tail = m ? __uint_as_float((m + OFF) << (23 - M)) : 0.f;
        const float fixed = m == 0x7fff ? __builtin_nanf("") : __uint_as_float(m + FIXED) - 512.f;
        const float a = m < JOIN ? tail : fixed;
        return __uint_as_float(__float_as_uint(a) | ((unsigned)q & 0x8000u) << 16);
    }
};

// ---- epilogue of C = A B^T ----
//   z = acc + bias + low-rank term;  y = residual + dropout(act(z));  slope = act'(z)
struct Epilogue {
    void* y;               // [M, N] 16-bit, row stride ldy
    const void* bias;      // [N] or null
    const void* res;       // [M, N] 16-bit or null, row stride ldr
    short* slope;          // [M, N] contiguous (row stride N) or null
    int64_t ldy, ldr;
    int M, N;
    int m_base;            // row of the whole operand that row 0 is (the dropout counter's)
    int bias_f32, act;
    int vec;               // every 8-column group of y, res and slope rows is 16-byte aligned
    int nt;                // store y and slope past the caches' retention (outputs far larger than the L2s)
    Dropout drop;
    // low-rank term u v^T (u [M, R], v [N, R], both zero-padded to R % 32 == 0 columns); low_mask: the
    // dropout mask (scale 1) is applied to this term instead of the activation's value
    const u16 *lu, *lv;
    int R, low_mask;
};

// the bias of C columns from n, zeros past N or without one
template <typename T, int C>
__device__ __forceinline__ void bias_cols(const Epilogue& e, int n, float (&b)[C]) {
#pragma unroll
    for (int j = 0; j < C; ++j) {
        b[j] = 0.f;
        if (e.bias && n + j < e.N) b[j] = e.bias_f32 ? ((const float*)e.bias)[n + j] : T::to_f32(((const u16*)e.bias)[n + j]);
    }
}

// C consecutive columns n .. n + C - 1 (n % C == 0) of row m: v = acc (+ the low-rank term), b their bias. Columns at or
// past N are not touched.
template <typename T, int C>
__device__ __forceinline__ void epilogue_cols(const Epilogue& e, const uint2& off, int m, int n, float (&v)[C], const float (&b)[C]) {
    const int nc = min(C, e.N - n);
    if (m >= e.M || nc <= 0) return;
    const bool whole = nc == C && e.vec;
#pragma unroll
    for (int j = 0; j < C; ++j) v[j] += b[j];
    if (e.act != ACT_NONE) {
        float gr[C];
        if (e.slope) {
            short q[C];
            act_cols<true, C>(e.act, v, gr);
#pragma unroll
            for (int j = 0; j < C; ++j) q[j] = SlopeCode<T>::encode(gr[j]);
            short* s = e.slope + (int64_t)m * e.N + n;
            if (whole) {
                if constexpr (C % 8 == 0) {
#pragma unroll
                    for (int j = 0; j < C; j += 8) {
                        uint4 w;
                        __builtin_memcpy(&w, q + j, 16);
                        *(uint4*)(s + j) = w;
                    }
                } else {
                    uint2 w;
                    __builtin_memcpy(&w, q, 8);
                    *(uint2*)s = w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < C; ++j)
                    if (j < nc) s[j] = q[j];
            }
        } else {
            act_cols<false, C>(e.act, v, gr);
        }
    }
    if (e.drop.on && !e.low_mask) {
#pragma unroll
        for (int j = 0; j < C; j += 4) drop4(e.drop, off, e.m_base + m, n + j, e.drop.scale, v[j], v[j + 1], v[j + 2], v[j + 3]);
    }
    u16* y = (u16*)e.y + (int64_t)m * e.ldy + n;
    const u16* r = e.res ? (const u16*)e.res + (int64_t)m * e.ldr + n : nullptr;
    if (whole) {
        if (r) {
            u16 rr[C];
            if constexpr (C % 8 == 0) {
#pragma unroll
                for (int j = 0; j < C; j += 8) {
                    const uint4 w = *(const uint4*)(r + j);
                    __builtin_memcpy(rr + j, &w, 16);
                }
            } else {
                const uint2 w = *(const uint2*)r;
                __builtin_memcpy(rr, &w, 8);
            }
#pragma unroll
            for (int j = 0; j < C; ++j) v[j] += T::to_f32(rr[j]);
        }
        if constexpr (C % 8 == 0) {
#pragma unroll
            for (int j = 0; j < C; j += 8)
                *(uint4*)(y + j) = make_uint4(pack2<T>(v[j], v[j + 1]), pack2<T>(v[j + 2], v[j + 3]),
                                              pack2<T>(v[j + 4], v[j + 5]), pack2<T>(v[j + 6], v[j + 7]));
        } else {
            *(uint2*)y = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
        }
    } else {
#pragma unroll
        for (int j = 0; j < C; ++j)
            if (j < nc) y[j] = T::from_f32(r ? v[j] + T::to_f32(r[j]) : v[j]);
    }
}

// ---- matrix product C = A B^T (matmul.hip) ----
// A(m, k) at A + m * lda + k (a_k) or A + k * lda + m; B(n, k) likewise. Any M, N, K >= 0.
struct Matmul {
    const u16 *A, *B;
    int64_t lda, ldb;
    int a_k, b_k;
    int M, N, K;
    Epilogue e;
};
// One launch: tile (0 = 64 x 64, 1 = 128 x 128, 2 = 256 x 256), slices of k, and its estimated time.
struct MatmulPart {
    int rows, tile, S, kslice;
    double us;
};
struct MatmulPlan {
    size_t a_bytes, b_bytes, part_bytes;
    int N4, parts;
    MatmulPart part[2];  // rows [0, part[0].rows), then the rest
};
// the launches for this shape, strides and alignment; `chosen`: with these parts' rows, tiles and slices (rows of the first
// of two a multiple of 256)
MatmulPlan matmul_plan(const Matmul& a, const MatmulPart* chosen = nullptr, int parts = 0);
// bytes of device workspace that launch_matmul needs
size_t matmul_workspace(const MatmulPlan& p);
inline size_t matmul_workspace(const Matmul& a) { return matmul_workspace(matmul_plan(a)); }
// 0, or -1 when the workspace is too small
int launch_matmul(hipStream_t s, int dtype, const Matmul& a, const MatmulPlan& p, void* ws, size_t ws_bytes);
inline int launch_matmul(hipStream_t s, int dtype, const Matmul& a, void* ws, size_t ws_bytes) {
    return launch_matmul(s, dtype, a, matmul_plan(a), ws, ws_bytes);
}

// largest row stride (elements) the tiles' 32-bit in-tile offsets allow
constexpr int64_t MATMUL_MAX_LD = 1 << 22;

}  // namespace clipvit
