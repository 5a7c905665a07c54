// Fine-tuning operators: counter-based dropout, a Linear's dz and bias gradient, the low-rank adapter's
// thin products, and the C entry points of all of them (the matrix product itself is matmul.hip).
//
// A Linear with an adapter (main.py:19-59): y = x W^T + b + s (dropout(x) A) B. The reference runs the
// adapter as a side branch while it trains (train_lora.py, without dropout) and this library merges it for inference
// (clipvit_load_lora); these operators are the unmerged form with its gradients.
#include <cmath>
#include <string>

#include "clipvit.h"
#include "finetune.h"

namespace clipvit {

extern thread_local std::string g_err;

namespace {

// ---- element access: 32- or 16-bit storage, fp32 arithmetic ----
struct F32T {
    typedef float store;
    static __device__ __forceinline__ float to_f32(float v) { return v; }
    static __device__ __forceinline__ float from_f32(float v) { return v; }
};
struct BF16T {
    typedef u16 store;
    typedef BF16 half;
    static __device__ __forceinline__ float to_f32(u16 v) { return BF16::to_f32(v); }
    static __device__ __forceinline__ u16 from_f32(float v) { return BF16::from_f32(v); }
};
struct F16T {
    typedef u16 store;
    typedef F16 half;
    static __device__ __forceinline__ float to_f32(u16 v) { return F16::to_f32(v); }
    static __device__ __forceinline__ u16 from_f32(float v) { return F16::from_f32(v); }
};
// C consecutive elements, nc of them valid; 16 bytes at a time where `vec` says so and all are valid
template <class E, int C>
__device__ __forceinline__ void load_cols(const typename E::store* p, int nc, bool vec, float (&v)[C]) {
    constexpr int PER = 16 / sizeof(typename E::store);
    if (vec && nc >= C) {
#pragma unroll
        for (int j = 0; j < C; j += PER) {
            typename E::store t[PER];
            const uint4 w = *(const uint4*)(p + j);
            __builtin_memcpy(t, &w, 16);
#pragma unroll
            for (int i = 0; i < PER; ++i) v[j + i] = E::to_f32(t[i]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < C; ++j) v[j] = j < nc ? E::to_f32(p[j]) : 0.f;
    }
}
template <class E, int C>
__device__ __forceinline__ void store_cols(typename E::store* p, int nc, bool vec, const float (&v)[C]) {
    constexpr int PER = 16 / sizeof(typename E::store);
    if (vec && nc >= C) {
#pragma unroll
        for (int j = 0; j < C; j += PER) {
            typename E::store t[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) t[i] = E::from_f32(v[j + i]);
            uint4 w;
            __builtin_memcpy(&w, t, 16);
            *(uint4*)(p + j) = w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < C; ++j)
            if (j < nc) p[j] = E::from_f32(v[j]);
    }
}

// ---- dropout: y = residual + mask(x) scale; eight columns a thread ----
struct DropArgs {
    const void *x, *res;
    void* y;
    int64_t ldx, ldr, ldy;
    int rows, cols, vec, tx;  // tx threads cover tx * 8 columns, 256 / tx rows a step
    Dropout d;
};
template <class E>
__global__ __launch_bounds__(256) void dropout_kernel(DropArgs a) {
    typedef typename E::store S;
    const int c = ((int)blockIdx.x * a.tx + (int)threadIdx.x % a.tx) * 8;
    const int ty = (int)threadIdx.x / a.tx, ny = 256 / a.tx;
    if (c >= a.cols) return;
    const int nc = min(8, a.cols - c);
    const uint2 off = drop_offset(a.d);
    for (int64_t m = (int64_t)blockIdx.y * ny + ty; m < a.rows; m += (int64_t)gridDim.y * ny) {
        float v[8];
        load_cols<E, 8>((const S*)a.x + m * a.ldx + c, nc, a.vec, v);
        if (a.d.on) {
            drop4(a.d, off, (int)m, c, a.d.scale, v[0], v[1], v[2], v[3]);
            drop4(a.d, off, (int)m, c + 4, a.d.scale, v[4], v[5], v[6], v[7]);
        }
        if (a.res) {
            float r[8];
            load_cols<E, 8>((const S*)a.res + m * a.ldr + c, nc, a.vec, r);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += r[j];
        }
        store_cols<E, 8>((S*)a.y + m * a.ldy + c, nc, a.vec, v);
    }
}

// The same for rows that 16-byte accesses cannot address (an odd width, a slice): a wave takes 256 columns of a row, lane l
// computes the mask of the four columns 4 l .. 4 l + 3, four ballots make it a 256-bit mask in scalar registers, and every
// access is one element a lane, 64 consecutive ones an instruction (eight scattered elements a lane: 12611 x 2049 fp32 100 us,
// 2.0 TB/s).
template <class E>
__global__ __launch_bounds__(256) void dropout_rows_kernel(DropArgs a) {
    typedef typename E::store S;
    const int lane = threadIdx.x & 63;
    const int c0 = ((int)blockIdx.x * a.tx + (int)(threadIdx.x >> 6) % a.tx) * 256;
    const int ty = (int)(threadIdx.x >> 6) / a.tx, ny = 4 / a.tx;
    if (c0 >= a.cols) return;
    const uint2 off = drop_offset(a.d);
    for (int64_t m = (int64_t)blockIdx.y * ny + ty; m < a.rows; m += (int64_t)gridDim.y * ny) {
        unsigned long long keep[4] = {~0ull, ~0ull, ~0ull, ~0ull};
        if (a.d.on) {
            const uint4 w = philox4(((unsigned)c0 >> 2) + lane, (unsigned)m, off.x, off.y, a.d.k0, a.d.k1);
            keep[0] = __ballot(w.x > a.d.drop_max);
            keep[1] = __ballot(w.y > a.d.drop_max);
            keep[2] = __ballot(w.z > a.d.drop_max);
            keep[3] = __ballot(w.w > a.d.drop_max);
        }
        const int q = lane & 3;
        const unsigned long long mine = q & 2 ? (q & 1 ? keep[3] : keep[2]) : (q & 1 ? keep[1] : keep[0]);
        const S* x = (const S*)a.x + m * a.ldx;
        const S* r = (const S*)a.res + m * a.ldr;
        S* y = (S*)a.y + m * a.ldy;
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = c0 + 64 * j + lane;
            v[j] = c < a.cols ? E::to_f32(x[c]) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = c0 + 64 * j + lane;
            if (c >= a.cols) continue;
            // column 64 j + lane is word lane & 3 of quad 16 j + lane / 4
            float o = a.d.on ? ((mine >> (16 * j + (lane >> 2))) & 1 ? v[j] * a.d.scale : 0.f) : v[j];
            if (a.res) o += E::to_f32(r[c]);
            y[c] = E::from_f32(o);
        }
    }
}

// ---- dz = dropout(dy) * act'(z), and the column sums of the unrounded dz for the bias gradient ----
struct DzArgs {
    const void* dy;
    const short* slope;  // [M, N] or null
    void* dz;            // [M, lddz] or null
    float* part;         // [gridDim.y][N] column sums of a block's rows, or null
    void* db;            // the bias gradient itself where one block has all the rows (part null), or null
    int64_t lddy, lddz;
    int M, N, rows, vec, db_f32;  // rows of a block
    Dropout d;
};
template <class E>
__global__ __launch_bounds__(256) void dz_kernel(DzArgs a) {
    typedef typename E::store S;
    __shared__ float sums[8][32][9];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int c = ((int)blockIdx.x * 32 + tx) * 8;
    const int nc = min(8, a.N - c);
    float s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = 0.f;
    if (nc > 0) {
        const uint2 off = drop_offset(a.d);
        const int64_t m1 = min((int64_t)a.M, ((int64_t)blockIdx.y + 1) * a.rows);
        for (int64_t m = (int64_t)blockIdx.y * a.rows + ty; m < m1; m += 8) {
            float v[8];
            load_cols<E, 8>((const S*)a.dy + m * a.lddy + c, nc, a.vec, v);
            if (a.d.on) {
                drop4(a.d, off, (int)m, c, a.d.scale, v[0], v[1], v[2], v[3]);
                drop4(a.d, off, (int)m, c + 4, a.d.scale, v[4], v[5], v[6], v[7]);
            }
            if (a.slope) {
                const short* q = a.slope + m * a.N + c;
                short t[8];
                if (a.vec && nc == 8) {
                    const uint4 w = *(const uint4*)q;
                    __builtin_memcpy(t, &w, 16);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) t[j] = j < nc ? q[j] : (short)0;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] *= SlopeCode<typename E::half>::decode(t[j]);
            }
            if (a.dz) store_cols<E, 8>((S*)a.dz + m * a.lddz + c, nc, a.vec, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) s[j] += v[j];
        }
    }
    if (!a.part && !a.db) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) sums[ty][tx][j] = s[j];
    __syncthreads();
    if (ty == 0 && nc > 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float t = 0.f;
#pragma unroll
            for (int y = 0; y < 8; ++y) t += sums[y][tx][j];
            if (j >= nc) continue;
            if (a.part) a.part[(int64_t)blockIdx.y * a.N + c + j] = t;
            else if (a.db_f32) ((float*)a.db)[c + j] = t;
            else ((S*)a.db)[c + j] = E::from_f32(t);
        }
    }
}
// db = the blocks' column sums in a fixed order; 32 columns a block, eight slices of the blocks each
template <class E>
__global__ __launch_bounds__(256) void db_kernel(const float* __restrict__ part, int blocks, int N, void* db, int db_f32) {
    __shared__ float sums[8][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int n = blockIdx.x * 32 + tx;
    float s = 0.f;
    if (n < N) {
#pragma unroll 8
        for (int b = ty; b < blocks; b += 8) s += part[(int64_t)b * N + n];
    }
    sums[ty][tx] = s;
    __syncthreads();
    if (ty || n >= N) return;
    float t = 0.f;
#pragma unroll
    for (int y = 0; y < 8; ++y) t += sums[y][tx];
    if (db_f32) ((float*)db)[n] = t;
    else ((typename E::store*)db)[n] = E::from_f32(t);
}

// ---- low-rank factors, zero padded: dst[i][j] = src(i, j), i < I (zeros past ri), j < J (zeros past rj), J a multiple of 8 ----
// A thread writes eight j of a row in one store; neighbours take neighbouring i where those are contiguous in src (one
// element a thread, j fastest, read a line for each: 4096 x 16 transposed 6.7 us).
struct PadArgs {
    const u16* src;
    int64_t s0, s1;
    int ri, rj, I, J;
    u16* dst;
};
__global__ __launch_bounds__(256) void pad_kernel(PadArgs a, PadArgs b, int blocks_a) {
    const bool first = (int)blockIdx.x < blocks_a;
    const PadArgs& p = first ? a : b;
    const int64_t t = ((int64_t)blockIdx.x - (first ? 0 : blocks_a)) * 256 + threadIdx.x, along = p.s0 == 1 ? p.I : p.J >> 3;
    const int64_t hi = t / along, lo = t - hi * along;
    const int64_t r = p.s0 == 1 ? lo : hi, c = (p.s0 == 1 ? hi : lo) * 8;
    if (r >= p.I || c >= p.J) return;
    const u16* s = p.src + r * p.s0 + c * p.s1;
    u16 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = r < p.ri && c + j < p.rj ? s[j * p.s1] : (u16)0;
    uint4 w;
    __builtin_memcpy(&w, v, 16);
    *(uint4*)(p.dst + r * p.J + c) = w;
}

// ---- thin product u[m, r] = alpha sum_k mask(x)[m, k] f[r, k], 32 ranks a launch row ----
// One workgroup: RG groups of 16 rows of x, its four waves a quarter of k each, so x is read once, by 16-byte loads straight
// into the MFMA fragment (lane: row lane & 15). Steps are 64 deep: lane group g takes k 16 g .. 16 g + 15 of it as two
// fragments (the order of k inside a step is free, f is read in the same one), so a step touches whole 128-byte lines.
// f's fragments, read from the caches, serve all RG row groups: with one group they were twice x's bytes (18464 x 4096,
// rank 16: 73 us, 2 TB/s). The quarters meet in LDS.
struct DownArgs {
    const u16 *x, *f;  // x [M, K] row stride ldx; f [R, K] row stride ldf, rows past r and columns past K (to 64) zero
    u16* u;            // [M, R]
    int64_t ldx, ldf;
    int M, K, R, rank, vec;
    float alpha;
    Dropout d;
};
template <typename T, int RG>
__global__ __launch_bounds__(256) void lora_down_kernel(DownArgs a) {
    typedef typename T::vec8 vec8;
    __shared__ float red[3][RG][64][9];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int li = lane & 15, g = lane >> 4;
    const int m0 = blockIdx.x * (16 * RG) + li, r0 = blockIdx.y * 32;
    const bool two = a.rank > r0 + 16;  // (the second 16 ranks are all padding otherwise)
    const int nk = (a.K + 63) >> 6, k0 = nk * wave / 4, k1 = nk * (wave + 1) / 4;
    const u16* xr[RG];
#pragma unroll
    for (int i = 0; i < RG; ++i) xr[i] = a.x + (int64_t)min(m0 + 16 * i, a.M - 1) * a.ldx;  // (rows past M are not stored)
    const u16* f0 = a.f + (int64_t)(r0 + li) * a.ldf;
    const u16* f1 = f0 + 16 * a.ldf;
    const uint2 off = drop_offset(a.d);
    f32x4 c0[RG], c1[RG];
#pragma unroll
    for (int i = 0; i < RG; ++i) c0[i] = c1[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto masked = [&](uint4 x, int m, int k) -> vec8 {
        u16 v[8];
        __builtin_memcpy(v, &x, 16);
        if (a.d.on) {
            const uint4 p = philox4((unsigned)k >> 2, (unsigned)m, off.x, off.y, a.d.k0, a.d.k1);
            const uint4 q = philox4(((unsigned)k >> 2) + 1, (unsigned)m, off.x, off.y, a.d.k0, a.d.k1);
            const unsigned w[8] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = w[j] > a.d.drop_max ? v[j] : (u16)0;
        }
        vec8 r;
        __builtin_memcpy(&r, v, 16);
        return r;
    };
    const int whole = a.vec ? a.K >> 6 : 0;  // steps of 64 whole columns
    int kt = k0;
#pragma unroll 2
    for (; kt < min(k1, whole); ++kt) {
        const int k = kt * 64 + 16 * g;
        uint4 x[RG][2];
#pragma unroll
        for (int i = 0; i < RG; ++i) {
            x[i][0] = *(const uint4*)(xr[i] + k);
            x[i][1] = *(const uint4*)(xr[i] + k + 8);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const vec8 fa = *(const vec8*)(f0 + k + 8 * h);
            const vec8 fb = two ? *(const vec8*)(f1 + k + 8 * h) : fa;
#pragma unroll
            for (int i = 0; i < RG; ++i) {
                const vec8 xf = masked(x[i][h], m0 + 16 * i, k + 8 * h);
                c0[i] = T::mfma16(fa, xf, c0[i]);  // lane: row m, ranks 4 g .. 4 g + 3
                if (two) c1[i] = T::mfma16(fb, xf, c1[i]);
            }
        }
    }
    for (; kt < k1; ++kt) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = kt * 64 + 16 * g + 8 * h;
            const vec8 fa = *(const vec8*)(f0 + k), fb = *(const vec8*)(f1 + k);
#pragma unroll
            for (int i = 0; i < RG; ++i) {
                u16 v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = k + j < a.K ? xr[i][k + j] : (u16)0;
                uint4 x;
                __builtin_memcpy(&x, v, 16);
                const vec8 xf = masked(x, m0 + 16 * i, k);
                c0[i] = T::mfma16(fa, xf, c0[i]);
                c1[i] = T::mfma16(fb, xf, c1[i]);
            }
        }
    }
    if (wave) {
#pragma unroll
        for (int i = 0; i < RG; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                red[wave - 1][i][lane][j] = c0[i][j];
                red[wave - 1][i][lane][4 + j] = c1[i][j];
            }
    }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int i = 0; i < RG; ++i) {
        const int m = m0 + 16 * i;
        if (m >= a.M) continue;
        for (int w = 0; w < 3; ++w)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                c0[i][j] += red[w][i][lane][j];
                c1[i][j] += red[w][i][lane][4 + j];
            }
        // a padded rank is zero whatever the row holds (the zero factor times an infinity is not)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            c0[i][j] = r0 + 4 * g + j < a.rank ? c0[i][j] * a.alpha : 0.f;
            c1[i][j] = r0 + 16 + 4 * g + j < a.rank ? c1[i][j] * a.alpha : 0.f;
        }
        u16* u = a.u + (int64_t)m * a.R + r0 + 4 * g;
        *(uint2*)u = make_uint2(pack2<T>(c0[i][0], c0[i][1]), pack2<T>(c0[i][2], c0[i][3]));
        *(uint2*)(u + 16) = make_uint2(pack2<T>(c1[i][0], c1[i][1]), pack2<T>(c1[i][2], c1[i][3]));
    }
}

// ---- thin gradient g[c, r] = sum_m mask(x)[m, c] u[m, r]: 128 columns x 32 ranks a workgroup, slices of rows ----
// x passes through registers once (16-byte loads, masked, eight columns of a row a thread) into an LDS tile of
// 32 rows, which the four waves read transposed (32 columns each) against u's 32 ranks.
struct GradArgs {
    const u16 *x, *u;  // x [M, C] row stride ldx, u [M, R] contiguous
    float* part;       // [gridDim.z][R][C4]
    int64_t ldx;
    int M, C, C4, R, rows, vec;  // rows of a slice, a multiple of 32
    Dropout d;
};
typedef unsigned u32x2f __attribute__((ext_vector_type(2)));
template <typename T>
__global__ __launch_bounds__(256) void lora_grad_kernel(GradArgs a) {
    typedef typename T::vec8 vec8;
    // rows of 128 columns (256 B) / 32 ranks (64 B), 32-B units swizzled by the row (see matmul.hip)
    __shared__ __attribute__((aligned(16))) u16 xs[2][32 * 128], us[2][32 * 32];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int li = lane & 15, g = lane >> 4, q = li >> 2, p = li & 3;
    const int c0 = blockIdx.x * 128, r0 = blockIdx.y * 32;
    const int64_t ms = (int64_t)blockIdx.z * a.rows;
    const int steps = (int)((min((int64_t)a.M - ms, (int64_t)a.rows) + 31) >> 5);
    const uint2 off = drop_offset(a.d);
    const int xk = threadIdx.x >> 4, xc = threadIdx.x & 15;  // this thread's rows xk, xk + 16, chunk xc
    const int cc = c0 + xc * 8, nc = min(8, a.C - cc);
    const int uk = threadIdx.x >> 2, uc = threadIdx.x & 3;   // threads 0 .. 127: row uk of u, chunk uc
    u16 xv[2][8];
    uint4 uv;
    auto fetch = [&](int st) {
        const int64_t mb = ms + st * 32;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t m = mb + xk + 16 * h;
            const int n = m < a.M ? nc : 0;
            const u16* s = a.x + m * a.ldx + cc;
            if (a.vec && n == 8) {
                const uint4 w = *(const uint4*)s;
                __builtin_memcpy(xv[h], &w, 16);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) xv[h][j] = j < n ? s[j] : (u16)0;
            }
        }
        if (threadIdx.x < 128) {
            const int64_t m = mb + uk;
            uv = m < a.M ? *(const uint4*)(a.u + m * a.R + r0 + uc * 8) : make_uint4(0, 0, 0, 0);
        }
    };
    auto put = [&](int st) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = xk + 16 * h;
            if (a.d.on && nc > 0) {
                const unsigned m = (unsigned)(ms + st * 32 + k);
                const uint4 w0 = philox4((unsigned)cc >> 2, m, off.x, off.y, a.d.k0, a.d.k1);
                const uint4 w1 = philox4(((unsigned)cc >> 2) + 1, m, off.x, off.y, a.d.k0, a.d.k1);
                const unsigned w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                for (int j = 0; j < 8; ++j) xv[h][j] = w[j] > a.d.drop_max ? xv[h][j] : (u16)0;
            }
            const int f = (k & 3) | ((k >> 1) & 4);
            uint4 w;
            __builtin_memcpy(&w, xv[h], 16);
            *(uint4*)(&xs[st & 1][k * 128 + ((xc ^ (f << 1)) << 3)]) = w;
        }
        if (threadIdx.x < 128) *(uint4*)(&us[st & 1][uk * 32 + uc * 8]) = uv;
    };
    f32x4 acc[2][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i >> 1][i & 1] = f32x4{0.f, 0.f, 0.f, 0.f};
    fetch(0);
    for (int st = 0; st < steps; ++st) {
        put(st);
        if (st + 1 < steps) fetch(st + 1);
        __syncthreads();
        vec8 xf[2], uf[2];
        {
            const int k = 8 * g + q, f = (k & 3) | ((k >> 1) & 4);
            const unsigned xb = (unsigned)(size_t)(LDS_AS u16*)xs[st & 1], ub = (unsigned)(size_t)(LDS_AS u16*)us[st & 1];
            const unsigned x0 = xb + k * 256 + (((wave * 2) ^ f) << 5) + p * 8, x1 = xb + k * 256 + (((wave * 2 + 1) ^ f) << 5) + p * 8;
            const unsigned u0 = ub + k * 64 + p * 8;
            u32x2f r[8];
            asm volatile(
                "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:1024\n\t"
                "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:1024\n\t"
                "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:256\n\t"
                "ds_read_b64_tr_b16 %6, %10 offset:32\n\tds_read_b64_tr_b16 %7, %10 offset:288\n\ts_waitcnt lgkmcnt(0)"
                : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
                : "v"(x0), "v"(x1), "v"(u0)
                : "memory");
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                xf[i] = __builtin_bit_cast(vec8, (u32x4){r[2 * i].x, r[2 * i].y, r[2 * i + 1].x, r[2 * i + 1].y});
                uf[i] = __builtin_bit_cast(vec8, (u32x4){r[4 + 2 * i].x, r[4 + 2 * i].y, r[5 + 2 * i].x, r[5 + 2 * i].y});
            }
        }
        // lane: rank r0 + 16 i + li, columns 16 j + 4 g .. + 3 of the wave's 32
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = T::mfma16(xf[j], uf[i], acc[i][j]);
        // two LDS buffers: the next put writes the other one, and a wave passes the next barrier only
        // after its reads above
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int c = c0 + wave * 32 + 16 * j + 4 * g;
            if (c < a.C4) *(f32x4*)(a.part + ((int64_t)blockIdx.z * a.R + r0 + 16 * i + li) * a.C4 + c) = acc[i][j];
        }
}
// the slices' sums in order; out[c, r] (or [r, c]) by strides, r < rank; four columns a thread
template <typename T>
__global__ __launch_bounds__(256) void lora_grad_join_kernel(const float* __restrict__ part, int slices, int R, int C, int C4, int rank,
                                                             u16* out, int64_t so_c, int64_t so_r) {
    const int q = C4 >> 2;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int r = (int)(i / q), c = (int)(i - (int64_t)r * q) * 4;
    if (r >= rank) return;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    const float* p = part + (int64_t)r * C4 + c;
#pragma unroll 8
    for (int z = 0; z < slices; ++z) s += *(const f32x4*)(p + (int64_t)z * R * C4);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (c + j < C) out[(c + j) * so_c + r * so_r] = T::from_f32(s[j]);
}

// ---- host side ----
#define FT_FAIL(code, msg) \
    do {                   \
        g_err = (msg);     \
        return (code);     \
    } while (0)
#define FT_LAUNCHED()                                                                            \
    do {                                                                                         \
        const hipError_t e_ = hipGetLastError();                                                 \
        if (e_ != hipSuccess) FT_FAIL(CLIPVIT_E_HIP, std::string("launch: ") + hipGetErrorString(e_)); \
    } while (0)

bool is16(int dtype) { return dtype == CLIPVIT_BF16 || dtype == CLIPVIT_F16; }
bool aligned16(const void* p) { return ((size_t)p & 15) == 0; }
int64_t up(int64_t v, int64_t q) { return (v + q - 1) / q * q; }
constexpr int64_t MAX_DIM = 1 << 30;

bool bad_dropout(const clipvit_dropout_args& d) { return !(d.p >= 0.0 && d.p <= 1.0); }
Dropout make_dropout(const clipvit_dropout_args& d) {
    Dropout r{};
    const double t = std::floor(d.p * 4294967296.0 + 0.5);
    r.on = t >= 1.0;
    if (!r.on) return r;
    r.k0 = (unsigned)d.seed;
    r.k1 = (unsigned)(d.seed >> 32);
    r.o0 = (unsigned)d.offset;
    r.o1 = (unsigned)(d.offset >> 32);
    r.offset_dev = (const uint2*)d.offset_dev;
    r.drop_max = (unsigned)(t - 1.0);
    r.scale = d.p < 1.0 ? (float)(1.0 / (1.0 - d.p)) : 0.f;
    return r;
}

// a [rows, cols] view with one unit stride -> (contiguous along columns?, row stride); false: refused. A single column has
// no second k row: any stride does that puts one outside a tile's resource (at most 512 bytes) in 32 bits.
bool panel_of(int64_t s0, int64_t s1, int64_t rows, int64_t cols, int& contig, int64_t& ld) {
    if (s1 == 1 || cols == 1) {
        contig = 1;
        ld = rows <= 1 ? up(cols, 8) : s0;
        if (cols == 1 && rows > 1 && s0 == 1) {  // one column of consecutive elements
            contig = 0;
            ld = 4096;
            return true;
        }
        return rows <= 1 || (ld >= cols && ld < MATMUL_MAX_LD);
    }
    if (s0 == 1 || rows == 1) {
        contig = 0;
        ld = cols <= 1 ? 4096 : s1;
        return cols <= 1 || (ld >= rows && ld < MATMUL_MAX_LD);
    }
    return false;
}

// C [M, N] = A(m, k) B(n, k)^T with the given strides; false: an operand is refused
bool make_matmul(Matmul& m, const void* A, int64_t a0, int64_t a1, const void* B, int64_t b0, int64_t b1, int64_t M, int64_t N, int64_t K,
                 void* y, int64_t ldy) {
    m = Matmul{};
    m.A = (const u16*)A;
    m.B = (const u16*)B;
    m.M = (int)M;
    m.N = (int)N;
    m.K = (int)K;
    m.e.M = m.M;
    m.e.N = m.N;
    m.e.y = y;
    m.e.ldy = M > 1 ? ldy : up(N, 8);
    if (!M || !N || !K) return true;
    return panel_of(a0, a1, M, K, m.a_k, m.lda) && panel_of(b0, b1, N, K, m.b_k, m.ldb);
}

// A workspace as consecutive 256-byte aligned parts; with a null base it only counts.
struct Arena {
    unsigned char* base;
    size_t used = 0;
    void* take(size_t bytes) {
        void* p = base ? base + used : nullptr;
        used += (bytes + 255) / 256 * 256;
        return p;
    }
};

struct Db {  // dz / bias-gradient launch
    DzArgs d;
    void* db;
    int db_f32, blocks;
};
Db make_dz(const void* dy, int64_t dy_stride, const int16_t* slope, void* dz, int64_t lddz, void* db, int db_f32, int64_t M, int64_t N,
           const Dropout& drop) {
    Db b{};
    DzArgs& d = b.d;
    b.db = db;
    b.db_f32 = db_f32;
    // about 4096 workgroups of 256 columns and at least 8 rows (fewer rows a block fill the chip on small products:
    // 1237 x 437 21 -> 8 us; fewer blocks shorten the join: 36928 x 4096 23 -> 6 us)
    const int64_t most = 4096 / ((N + 255) / 256 ? (N + 255) / 256 : 1), need = (M + 7) / 8;
    b.blocks = (int)(need < most ? need : most > 1 ? most : (M ? 1 : 0));
    if (db && M && M <= 128) b.blocks = 1;  // few rows: one block writes db, no join launch
    d.rows = b.blocks ? (int)up((M + b.blocks - 1) / b.blocks, 8) : 8;
    d.dy = dy;
    d.slope = slope;
    d.dz = dz;
    d.lddy = M > 1 ? dy_stride : up(N, 8);
    d.lddz = lddz;
    d.M = (int)M;
    d.N = (int)N;
    d.d = drop;
    d.vec = aligned16(dy) && d.lddy % 8 == 0 && (!dz || (aligned16(dz) && lddz % 8 == 0)) && (!slope || (aligned16(slope) && N % 8 == 0));
    return b;
}
size_t dz_part_bytes(const Db& b) { return b.db && b.blocks > 1 ? (size_t)b.blocks * b.d.N * 4 : 0; }
void launch_dz(hipStream_t s, bool bf, Db& b, void* part) {
    b.d.part = b.db && b.blocks > 1 ? (float*)part : nullptr;
    b.d.db = b.blocks == 1 ? b.db : nullptr;
    b.d.db_f32 = b.db_f32;
    if (b.blocks) {
        const dim3 grid((b.d.N + 255) / 256, b.blocks);
        if (bf) dz_kernel<BF16T><<<grid, 256, 0, s>>>(b.d);
        else dz_kernel<F16T><<<grid, 256, 0, s>>>(b.d);
    }
    if (b.db && b.blocks != 1) {
        const int g = (b.d.N + 31) / 32;
        if (bf) db_kernel<BF16T><<<g, 256, 0, s>>>(b.d.part, b.blocks, b.d.N, b.db, b.db_f32);
        else db_kernel<F16T><<<g, 256, 0, s>>>(b.d.part, b.blocks, b.d.N, b.db, b.db_f32);
    }
}

// ---- Linear ----
int check_sizes(const char* what, int dtype, int bias_dtype, int64_t M, int64_t N, int64_t K) {
    if (!is16(dtype)) FT_FAIL(CLIPVIT_E_INVALID, std::string(what) + ": dtype must be BF16 or F16");
    if (bias_dtype != CLIPVIT_F32 && bias_dtype != dtype) FT_FAIL(CLIPVIT_E_INVALID, std::string(what) + ": bias must be F32 or of the operands' type");
    if (M < 0 || N < 0 || K < 0 || M > MAX_DIM || N > MAX_DIM || K > MAX_DIM)
        FT_FAIL(CLIPVIT_E_INVALID, std::string(what) + ": M, N and K must lie in [0, 2^30]");
    return CLIPVIT_OK;
}
const char* const OPERANDS = "x and w need one unit stride, rows that do not overlap and a stride below 2^22";

int linear_of(const clipvit_linear_args* a, Matmul& m) {
    if (!a) FT_FAIL(CLIPVIT_E_INVALID, "null arguments");
    if (const int rc = check_sizes("linear", a->dtype, a->bias_dtype, a->M, a->N, a->K)) return rc;
    if (a->activation < 0 || a->activation > ACT_RELU) FT_FAIL(CLIPVIT_E_INVALID, "linear: unknown activation");
    if (bad_dropout(a->dropout)) FT_FAIL(CLIPVIT_E_INVALID, "dropout: p must lie in [0, 1]");
    if (a->M && a->N) {
        if (!a->y || (a->K && (!a->x || !a->w))) FT_FAIL(CLIPVIT_E_INVALID, "linear: null operand");
        if (a->y_stride < a->N && a->M > 1) FT_FAIL(CLIPVIT_E_INVALID, "linear: y rows overlap");
        if (a->residual && a->residual_stride < 0) FT_FAIL(CLIPVIT_E_INVALID, "linear: residual stride");
    }
    if (!make_matmul(m, a->x, a->x_stride[0], a->x_stride[1], a->w, a->w_stride[0], a->w_stride[1], a->M, a->N, a->K, a->y, a->y_stride))
        FT_FAIL(CLIPVIT_E_INVALID, std::string("linear: ") + OPERANDS);
    Epilogue& e = m.e;
    e.bias = a->bias;
    e.bias_f32 = a->bias_dtype == CLIPVIT_F32;
    e.res = a->residual;
    e.ldr = a->M > 1 ? a->residual_stride : up(a->N, 8);
    e.slope = a->activation ? a->slope : nullptr;
    e.act = a->activation;
    e.drop = make_dropout(a->dropout);
    return CLIPVIT_OK;
}

struct LinearGrad {
    Matmul dx, dw;
    Db dz;
    bool want_dx, want_dw, changed;
};
int linear_grad_of(const clipvit_linear_grad_args* a, LinearGrad& g, Arena& ws, void*& part, void*& mm, size_t& mm_bytes) {
    if (!a) FT_FAIL(CLIPVIT_E_INVALID, "null arguments");
    if (const int rc = check_sizes("linear_grad", a->dtype, a->bias_dtype, a->M, a->N, a->K)) return rc;
    if (bad_dropout(a->dropout)) FT_FAIL(CLIPVIT_E_INVALID, "dropout: p must lie in [0, 1]");
    g.want_dx = a->dx && a->M && a->K;
    g.want_dw = a->dw && a->N && a->K;
    if (a->M && a->N && !a->dy) FT_FAIL(CLIPVIT_E_INVALID, "linear_grad: null dy");
    if ((g.want_dx && a->N && !a->w) || (g.want_dw && a->M && !a->x)) FT_FAIL(CLIPVIT_E_INVALID, "linear_grad: null operand");
    if (a->M > 1 && a->N && (a->dy_stride < a->N || a->dy_stride >= MATMUL_MAX_LD)) FT_FAIL(CLIPVIT_E_INVALID, "linear_grad: dy stride");
    const Dropout drop = make_dropout(a->dropout);
    g.changed = (a->slope || drop.on) && (g.want_dx || g.want_dw) && a->M && a->N;
    const int64_t ld = g.changed ? up(a->N, 8) : a->dy_stride;
    if (ld >= MATMUL_MAX_LD && (g.want_dx || g.want_dw) && a->M > 1) FT_FAIL(CLIPVIT_E_INVALID, "linear_grad: N too large");
    void* dz = g.changed ? ws.take((size_t)a->M * ld * 2) : nullptr;
    g.dz = make_dz(a->dy, a->dy_stride, a->slope, dz, ld, a->N ? a->db : nullptr, a->bias_dtype == CLIPVIT_F32, a->M, a->N, drop);
    if (g.changed && !dz) g.dz.d.dz = (void*)256;  // counting the workspace: an aligned stand-in
    part = ws.take(dz_part_bytes(g.dz));
    const void* z = g.changed ? g.dz.d.dz : a->dy;
    mm_bytes = 0;
    if (g.want_dx) {
        if (!make_matmul(g.dx, z, ld, 1, a->w, a->w_stride[1], a->w_stride[0], a->M, a->K, a->N, a->dx, a->K))
            FT_FAIL(CLIPVIT_E_INVALID, std::string("linear_grad: ") + OPERANDS);
        mm_bytes = matmul_workspace(g.dx);
    }
    if (g.want_dw) {
        if (!make_matmul(g.dw, z, 1, ld, a->x, a->x_stride[1], a->x_stride[0], a->N, a->K, a->M, a->dw, a->K))
            FT_FAIL(CLIPVIT_E_INVALID, std::string("linear_grad: ") + OPERANDS);
        const size_t b = matmul_workspace(g.dw);
        if (b > mm_bytes) mm_bytes = b;  // the two products run one after the other and share it
    }
    mm = ws.take(mm_bytes);
    return CLIPVIT_OK;
}

// ---- LoRA Linear ----
int64_t rank32(int64_t r) { return up(r, 32); }
int check_lora(const char* what, int dtype, int bias_dtype, int64_t M, int64_t N, int64_t K, int64_t rank, const clipvit_dropout_args& d) {
    if (const int rc = check_sizes(what, dtype, bias_dtype, M, N, K)) return rc;
    if (rank < 1 || rank > 65536) FT_FAIL(CLIPVIT_E_INVALID, std::string(what) + ": rank must lie in [1, 65536]");
    if (bad_dropout(d)) FT_FAIL(CLIPVIT_E_INVALID, "dropout: p must lie in [0, 1]");
    return CLIPVIT_OK;
}
void launch_pad(hipStream_t s, const PadArgs& a, const PadArgs& b) {
    const int64_t na = ((int64_t)a.I * (a.J / 8) + 255) / 256, nb = ((int64_t)b.I * (b.J / 8) + 255) / 256;
    if (na + nb) pad_kernel<<<(unsigned)(na + nb), 256, 0, s>>>(a, b, (int)na);
}
void launch_down(hipStream_t s, bool bf, const void* x, int64_t ldx, const void* f, int64_t ldf, void* u, int64_t M, int64_t K, int64_t R,
                 int64_t rank, float alpha, const Dropout& drop) {
    if (!M) return;
    DownArgs d{};
    d.x = (const u16*)x;
    d.f = (const u16*)f;
    d.u = (u16*)u;
    d.ldx = M > 1 ? ldx : 0;
    d.ldf = ldf;
    d.M = (int)M;
    d.K = (int)K;
    d.R = (int)R;
    d.rank = (int)rank;
    d.vec = aligned16(x) && d.ldx % 8 == 0;
    d.alpha = alpha;
    d.d = drop;
    // two row groups a workgroup once that still gives every CU one; single groups spread few rows wider
    const int rg = M >= 8192 ? 2 : 1;
    const dim3 grid((unsigned)((M + 16 * rg - 1) / (16 * rg)), (unsigned)(R / 32));
    if (bf && rg == 2) lora_down_kernel<BF16, 2><<<grid, 256, 0, s>>>(d);
    else if (bf) lora_down_kernel<BF16, 1><<<grid, 256, 0, s>>>(d);
    else if (rg == 2) lora_down_kernel<F16, 2><<<grid, 256, 0, s>>>(d);
    else lora_down_kernel<F16, 1><<<grid, 256, 0, s>>>(d);
}
int grad_slices(int64_t M, int64_t C, int64_t R) {
    const int64_t wg = ((C + 127) / 128) * (R / 32);
    int64_t s = (1024 + wg - 1) / wg;
    const int64_t most = (M + 127) / 128;  // at least four 32-row steps a slice
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s);
}
size_t grad_bytes(int64_t M, int64_t C, int64_t R) { return C ? (size_t)grad_slices(M, C, R) * (size_t)R * (size_t)up(C, 4) * 4 : 0; }
// out(c, r) = sum_m mask(x)[m, c] u[m, r], r < rank, at out + c so_c + r so_r
void launch_grad(hipStream_t s, bool bf, const void* x, int64_t ldx, const void* u, void* out, int64_t so_c, int64_t so_r, int64_t M, int64_t C,
                 int64_t R, int64_t rank, const Dropout& drop, void* part) {
    if (!C) return;
    GradArgs d{};
    d.x = (const u16*)x;
    d.u = (const u16*)u;
    d.part = (float*)part;
    d.ldx = M > 1 ? ldx : 0;
    d.M = (int)M;
    d.C = (int)C;
    d.C4 = (int)up(C, 4);
    d.R = (int)R;
    d.vec = aligned16(x) && d.ldx % 8 == 0;
    d.d = drop;
    int slices = grad_slices(M, C, R);
    d.rows = (int)up((M + slices - 1) / slices, 32);
    slices = M ? (int)((M + d.rows - 1) / d.rows) : 0;
    if (slices) {
        const dim3 grid((unsigned)((C + 127) / 128), (unsigned)(R / 32), slices);
        if (bf) lora_grad_kernel<BF16><<<grid, 256, 0, s>>>(d);
        else lora_grad_kernel<F16><<<grid, 256, 0, s>>>(d);
    }
    const unsigned g = (unsigned)((rank * (up(C, 4) / 4) + 255) / 256);
    if (bf) lora_grad_join_kernel<BF16><<<g, 256, 0, s>>>(d.part, slices, d.R, d.C, d.C4, (int)rank, (u16*)out, so_c, so_r);
    else lora_grad_join_kernel<F16><<<g, 256, 0, s>>>(d.part, slices, d.R, d.C, d.C4, (int)rank, (u16*)out, so_c, so_r);
}
PadArgs pad_of(const void* src, int64_t s0, int64_t s1, int64_t ri, int64_t rj, int64_t I, int64_t J, void* dst) {
    return PadArgs{(const u16*)src, s0, s1, (int)ri, (int)rj, (int)I, (int)J, (u16*)dst};
}

struct Lora {
    Matmul y;
    void *f, *v, *mm;
    size_t mm_bytes;
};
int lora_of(const clipvit_lora_args* a, Lora& l, Arena& ws) {
    if (!a) FT_FAIL(CLIPVIT_E_INVALID, "null arguments");
    if (const int rc = check_lora("lora_linear", a->dtype, a->bias_dtype, a->M, a->N, a->K, a->rank, a->dropout)) return rc;
    const int64_t R = rank32(a->rank);
    if (a->M && a->N) {
        if (!a->y || !a->u || !aligned16(a->u) || !a->b || (a->K && (!a->x || !a->w || !a->a)))
            FT_FAIL(CLIPVIT_E_INVALID, "lora_linear: null or misaligned operand");
        if (a->M > 1 && a->x_stride < a->K) FT_FAIL(CLIPVIT_E_INVALID, "lora_linear: x rows overlap");
    }
    if (!make_matmul(l.y, a->x, a->x_stride, 1, a->w, a->w_stride[0], a->w_stride[1], a->M, a->N, a->K, a->y, a->N))
        FT_FAIL(CLIPVIT_E_INVALID, std::string("lora_linear: ") + OPERANDS);
    l.f = ws.take((size_t)R * up(a->K, 64) * 2);
    l.v = ws.take((size_t)a->N * R * 2);
    Epilogue& e = l.y.e;
    e.bias = a->bias;
    e.bias_f32 = a->bias_dtype == CLIPVIT_F32;
    e.lu = (const u16*)a->u;
    e.lv = (const u16*)l.v;
    e.R = (int)R;
    l.mm_bytes = matmul_workspace(l.y);
    l.mm = ws.take(l.mm_bytes);
    return CLIPVIT_OK;
}

struct LoraGrad {
    Matmul dx, dw;
    Db db;
    bool want_dx, want_dw, want_du;
    void *f, *v, *du, *grad, *part, *mm;
    size_t mm_bytes;
};
int lora_grad_of(const clipvit_lora_grad_args* a, LoraGrad& g, Arena& ws) {
    if (!a) FT_FAIL(CLIPVIT_E_INVALID, "null arguments");
    if (const int rc = check_lora("lora_linear_grad", a->dtype, a->bias_dtype, a->M, a->N, a->K, a->rank, a->dropout)) return rc;
    const int64_t R = rank32(a->rank);
    g.want_dx = a->dx && a->M && a->K;
    g.want_dw = a->dw && a->N && a->K;
    g.want_du = g.want_dx || (a->da && a->K);
    if (a->M && a->N && !a->dy) FT_FAIL(CLIPVIT_E_INVALID, "lora_linear_grad: null dy");
    if ((g.want_dx && a->N && !a->w) || (g.want_dx && !a->a) || (g.want_du && a->N && !a->b) || ((g.want_dw || a->da) && a->M && a->K && !a->x) ||
        (a->db_factor && a->M && (!a->u || !aligned16(a->u))))
        FT_FAIL(CLIPVIT_E_INVALID, "lora_linear_grad: null or misaligned operand");
    if (a->M > 1 && ((a->N && (a->dy_stride < a->N || a->dy_stride >= MATMUL_MAX_LD)) || ((g.want_dw || a->da) && a->x_stride < a->K)))
        FT_FAIL(CLIPVIT_E_INVALID, "lora_linear_grad: row stride");
    const Dropout none{};
    if (g.want_du) {
        g.f = ws.take((size_t)R * up(a->N, 64) * 2);
        g.v = ws.take((size_t)a->K * R * 2);
        g.du = ws.take((size_t)a->M * R * 2);
    }
    const size_t ga = a->da ? grad_bytes(a->M, a->K, R) : 0, gb = a->db_factor ? grad_bytes(a->M, a->N, R) : 0;
    g.grad = ws.take(ga > gb ? ga : gb);
    g.db = make_dz(a->dy, a->dy_stride, nullptr, nullptr, 8, a->N ? a->dbias : nullptr, a->bias_dtype == CLIPVIT_F32, a->M, a->N, none);
    g.part = ws.take(dz_part_bytes(g.db));
    g.mm_bytes = 0;
    if (g.want_dx) {
        if (!make_matmul(g.dx, a->dy, a->dy_stride, 1, a->w, a->w_stride[1], a->w_stride[0], a->M, a->K, a->N, a->dx, a->K))
            FT_FAIL(CLIPVIT_E_INVALID, std::string("lora_linear_grad: ") + OPERANDS);
        Epilogue& e = g.dx.e;
        e.lu = (const u16*)g.du;
        e.lv = (const u16*)g.v;
        e.R = (int)R;
        e.drop = make_dropout(a->dropout);
        e.low_mask = e.drop.on;
        g.mm_bytes = matmul_workspace(g.dx);
    }
    if (g.want_dw) {
        if (!make_matmul(g.dw, a->dy, 1, a->dy_stride, a->x, 1, a->x_stride, a->N, a->K, a->M, a->dw, a->K))
            FT_FAIL(CLIPVIT_E_INVALID, std::string("lora_linear_grad: ") + OPERANDS);
        const size_t b = matmul_workspace(g.dw);
        if (b > g.mm_bytes) g.mm_bytes = b;
    }
    g.mm = ws.take(g.mm_bytes);
    return CLIPVIT_OK;
}

bool bad_workspace(const Arena& need, const void* ws, size_t bytes) { return need.used > bytes || (need.used && (!ws || ((size_t)ws & 255))); }
const char* const WORKSPACE = "workspace too small or not 256-byte aligned (ask the call's _workspace)";

template <typename F>
int guarded(F&& f) noexcept {
    try {
        g_err.clear();
        return f();
    } catch (...) {
        try {
            g_err = "host allocation failed";
        } catch (...) {
        }
        return CLIPVIT_E_NOMEM;
    }
}

}  // namespace
}  // namespace clipvit

using namespace clipvit;

extern "C" {

int clipvit_linear_workspace(const clipvit_linear_args* a, size_t* bytes) {
    return guarded([&]() -> int {
        Matmul m;
        if (!bytes) FT_FAIL(CLIPVIT_E_INVALID, "null argument");
        if (const int rc = linear_of(a, m)) return rc;
        *bytes = matmul_workspace(m);
        return CLIPVIT_OK;
    });
}

int clipvit_linear(void* stream, const clipvit_linear_args* a, void* workspace, size_t bytes) {
    return guarded([&]() -> int {
        Matmul m;
        if (const int rc = linear_of(a, m)) return rc;
        if (!m.M || !m.N) return CLIPVIT_OK;
        if ((bytes && !workspace) || ((size_t)workspace & 255) || launch_matmul((hipStream_t)stream, a->dtype, m, workspace, bytes))
            FT_FAIL(CLIPVIT_E_INVALID, std::string("linear: ") + WORKSPACE);
        FT_LAUNCHED();
        return CLIPVIT_OK;
    });
}

int clipvit_matmul_plan_test(int64_t M, int64_t N, int64_t K, clipvit_matmul_part* parts, int* count) {
    return guarded([&]() -> int {
        if (!parts || !count) FT_FAIL(CLIPVIT_E_INVALID, "null argument");
        if (const int rc = check_sizes("matmul plan", CLIPVIT_F16, CLIPVIT_F16, M, N, K)) return rc;
        Matmul m{};
        m.M = (int)M;
        m.N = (int)N;
        m.K = (int)K;
        const MatmulPlan p = matmul_plan(m);
        *count = p.parts;
        for (int i = 0; i < p.parts; ++i) parts[i] = clipvit_matmul_part{p.part[i].rows, 64 << p.part[i].tile, p.part[i].S, p.part[i].kslice};
        return CLIPVIT_OK;
    });
}

int clipvit_linear_test(void* stream, const clipvit_linear_args* a, const clipvit_matmul_part* parts, int count, void* workspace, size_t bytes,
                        size_t* need) {
    return guarded([&]() -> int {
        Matmul m;
        if (const int rc = linear_of(a, m)) return rc;
        if (!parts || count < 1 || count > 2 || !m.M || !m.N) FT_FAIL(CLIPVIT_E_INVALID, "linear_test: one or two parts of a product");
        MatmulPart chosen[2];
        int64_t rows = 0;
        for (int i = 0; i < count; ++i) {
            const clipvit_matmul_part& p = parts[i];
            if (p.rows < 1 || (p.tile != 64 && p.tile != 128 && p.tile != 256) || p.slices < 1 || p.slices > 64 || (i + 1 < count && p.rows % 256))
                FT_FAIL(CLIPVIT_E_INVALID, "linear_test: rows (the first part's a multiple of 256), tile 64, 128 or 256, 1 to 64 slices");
            chosen[i] = MatmulPart{p.rows, p.tile >> 7, p.slices, 0, 0};
            rows += p.rows;
        }
        if (rows != m.M) FT_FAIL(CLIPVIT_E_INVALID, "linear_test: the parts' rows are not M");
        const MatmulPlan p = matmul_plan(m, chosen, count);
        if (need) {
            *need = matmul_workspace(p);
            return CLIPVIT_OK;
        }
        if ((bytes && !workspace) || ((size_t)workspace & 255) || launch_matmul((hipStream_t)stream, a->dtype, m, p, workspace, bytes))
            FT_FAIL(CLIPVIT_E_INVALID, std::string("linear_test: ") + WORKSPACE);
        FT_LAUNCHED();
        return CLIPVIT_OK;
    });
}

int clipvit_linear_grad_workspace(const clipvit_linear_grad_args* a, size_t* bytes) {
    return guarded([&]() -> int {
        if (!bytes) FT_FAIL(CLIPVIT_E_INVALID, "null argument");
        LinearGrad g{};
        Arena count{nullptr};
        void *part, *mm;
        size_t mm_bytes;
        if (const int rc = linear_grad_of(a, g, count, part, mm, mm_bytes)) return rc;
        *bytes = count.used;
        return CLIPVIT_OK;
    });
}

int clipvit_linear_grad(void* stream, const clipvit_linear_grad_args* a, void* workspace, size_t bytes) {
    return guarded([&]() -> int {
        LinearGrad g{};
        Arena ws{(unsigned char*)workspace};
        void *part, *mm;
        size_t mm_bytes;
        if (const int rc = linear_grad_of(a, g, ws, part, mm, mm_bytes)) return rc;
        if (bad_workspace(ws, workspace, bytes)) FT_FAIL(CLIPVIT_E_INVALID, std::string("linear_grad: ") + WORKSPACE);
        hipStream_t s = (hipStream_t)stream;
        bool any = false;
        if (g.changed || g.dz.db) {
            launch_dz(s, a->dtype == CLIPVIT_BF16, g.dz, part);
            any = true;
        }
        if ((g.want_dx && launch_matmul(s, a->dtype, g.dx, mm, mm_bytes)) || (g.want_dw && launch_matmul(s, a->dtype, g.dw, mm, mm_bytes)))
            FT_FAIL(CLIPVIT_E_INVALID, std::string("linear_grad: ") + WORKSPACE);
        if (any || g.want_dx || g.want_dw) FT_LAUNCHED();
        return CLIPVIT_OK;
    });
}

int clipvit_dropout(void* stream, int dtype, const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, void* y,
                    int64_t y_stride, int64_t rows, int64_t cols, const clipvit_dropout_args* dropout) {
    return guarded([&]() -> int {
        if (!dropout) FT_FAIL(CLIPVIT_E_INVALID, "null arguments");
        if (dtype != CLIPVIT_F32 && !is16(dtype)) FT_FAIL(CLIPVIT_E_INVALID, "dropout: dtype must be F32, BF16 or F16");
        if (bad_dropout(*dropout)) FT_FAIL(CLIPVIT_E_INVALID, "dropout: p must lie in [0, 1]");
        if (rows < 0 || cols < 0 || rows > MAX_DIM || cols > MAX_DIM) FT_FAIL(CLIPVIT_E_INVALID, "dropout: rows and columns must lie in [0, 2^30]");
        if (!rows || !cols) return CLIPVIT_OK;
        if (!x || !y) FT_FAIL(CLIPVIT_E_INVALID, "dropout: null argument");
        if (rows > 1 && (x_stride < 0 || residual_stride < 0 || y_stride < cols)) FT_FAIL(CLIPVIT_E_INVALID, "dropout: row stride");
        DropArgs d{};
        d.x = x;
        d.res = residual;
        d.y = y;
        d.ldx = rows > 1 ? x_stride : 0;
        d.ldr = rows > 1 ? residual_stride : 0;
        d.ldy = rows > 1 ? y_stride : 0;
        d.rows = (int)rows;
        d.cols = (int)cols;
        d.d = make_dropout(*dropout);
        const int per = dtype == CLIPVIT_F32 ? 4 : 8;
        d.vec = aligned16(x) && aligned16(y) && aligned16(residual) && d.ldx % per == 0 && d.ldy % per == 0 && (!residual || d.ldr % per == 0);
        // tx threads (waves) cover a row's groups of 8 (256) columns: the widest that leaves at most an eighth of them idle
        const int per_group = d.vec ? 8 : 256, most = d.vec ? 64 : 4, all = d.vec ? 256 : 4;
        const int groups = (int)((cols + per_group - 1) / per_group);
        d.tx = most;
        while (d.tx > 1 && ((groups + d.tx - 1) / d.tx) * (int64_t)d.tx * 8 > (int64_t)groups * 9) d.tx >>= 1;
        const int ny = all / d.tx, gx = (groups + d.tx - 1) / d.tx;
        int64_t gy = (rows + ny - 1) / ny;
        const int64_t cap = (16384 + gx - 1) / gx;
        if (gy > cap) gy = cap;
        if (gy > 65535) gy = 65535;
        const dim3 grid(gx, (unsigned)gy);
        hipStream_t s = (hipStream_t)stream;
        if (d.vec) {
            if (dtype == CLIPVIT_F32) dropout_kernel<F32T><<<grid, 256, 0, s>>>(d);
            else if (dtype == CLIPVIT_BF16) dropout_kernel<BF16T><<<grid, 256, 0, s>>>(d);
            else dropout_kernel<F16T><<<grid, 256, 0, s>>>(d);
        } else {
            if (dtype == CLIPVIT_F32) dropout_rows_kernel<F32T><<<grid, 256, 0, s>>>(d);
            else if (dtype == CLIPVIT_BF16) dropout_rows_kernel<BF16T><<<grid, 256, 0, s>>>(d);
            else dropout_rows_kernel<F16T><<<grid, 256, 0, s>>>(d);
        }
        FT_LAUNCHED();
        return CLIPVIT_OK;
    });
}

int clipvit_lora_linear_workspace(const clipvit_lora_args* a, size_t* bytes) {
    return guarded([&]() -> int {
        if (!bytes) FT_FAIL(CLIPVIT_E_INVALID, "null argument");
        Lora l{};
        Arena count{nullptr};
        if (const int rc = lora_of(a, l, count)) return rc;
        *bytes = count.used;
        return CLIPVIT_OK;
    });
}

int clipvit_lora_linear(void* stream, const clipvit_lora_args* a, void* workspace, size_t bytes) {
    return guarded([&]() -> int {
        Lora l{};
        Arena ws{(unsigned char*)workspace};
        if (const int rc = lora_of(a, l, ws)) return rc;
        if (!a->M || !a->N) return CLIPVIT_OK;
        if (bad_workspace(ws, workspace, bytes)) FT_FAIL(CLIPVIT_E_INVALID, std::string("lora_linear: ") + WORKSPACE);
        hipStream_t s = (hipStream_t)stream;
        const int64_t R = rank32(a->rank), Kp = up(a->K, 64);
        const Dropout drop = make_dropout(a->dropout);
        launch_pad(s, pad_of(a->a, a->a_stride[1], a->a_stride[0], a->rank, a->K, R, Kp, l.f),
                   pad_of(a->b, a->b_stride[1], a->b_stride[0], a->N, a->rank, a->N, R, l.v));
        launch_down(s, a->dtype == CLIPVIT_BF16, a->x, a->x_stride, l.f, Kp, a->u, a->M, a->K, R, a->rank, a->scaling * (drop.on ? drop.scale : 1.f), drop);
        if (launch_matmul(s, a->dtype, l.y, l.mm, l.mm_bytes)) FT_FAIL(CLIPVIT_E_INVALID, std::string("lora_linear: ") + WORKSPACE);
        FT_LAUNCHED();
        return CLIPVIT_OK;
    });
}

int clipvit_lora_linear_grad_workspace(const clipvit_lora_grad_args* a, size_t* bytes) {
    return guarded([&]() -> int {
        if (!bytes) FT_FAIL(CLIPVIT_E_INVALID, "null argument");
        LoraGrad g{};
        Arena count{nullptr};
        if (const int rc = lora_grad_of(a, g, count)) return rc;
        *bytes = count.used;
        return CLIPVIT_OK;
    });
}

int clipvit_lora_linear_grad(void* stream, const clipvit_lora_grad_args* a, void* workspace, size_t bytes) {
    return guarded([&]() -> int {
        LoraGrad g{};
        Arena ws{(unsigned char*)workspace};
        if (const int rc = lora_grad_of(a, g, ws)) return rc;
        if (bad_workspace(ws, workspace, bytes)) FT_FAIL(CLIPVIT_E_INVALID, std::string("lora_linear_grad: ") + WORKSPACE);
        hipStream_t s = (hipStream_t)stream;
        const bool bf = a->dtype == CLIPVIT_BF16;
        const int64_t R = rank32(a->rank), Np = up(a->N, 64);
        const Dropout drop = make_dropout(a->dropout), none{};
        if (g.want_du) {
            launch_pad(s, pad_of(a->b, a->b_stride[0], a->b_stride[1], a->rank, a->N, R, Np, g.f),
                       pad_of(a->a, a->a_stride[0], a->a_stride[1], a->K, a->rank, g.want_dx ? a->K : 0, R, g.v));
            launch_down(s, bf, a->dy, a->dy_stride, g.f, Np, g.du, a->M, a->N, R, a->rank, a->scaling * (drop.on ? drop.scale : 1.f), none);
            if (g.want_dx && launch_matmul(s, a->dtype, g.dx, g.mm, g.mm_bytes)) FT_FAIL(CLIPVIT_E_INVALID, std::string("lora_linear_grad: ") + WORKSPACE);
            if (a->da) launch_grad(s, bf, a->x, a->x_stride, g.du, a->da, a->rank, 1, a->M, a->K, R, a->rank, drop, g.grad);
        }
        if (a->db_factor) launch_grad(s, bf, a->dy, a->dy_stride, a->u, a->db_factor, 1, a->N, a->M, a->N, R, a->rank, none, g.grad);
        if (g.want_dw && launch_matmul(s, a->dtype, g.dw, g.mm, g.mm_bytes)) FT_FAIL(CLIPVIT_E_INVALID, std::string("lora_linear_grad: ") + WORKSPACE);
        if (g.db.db) launch_dz(s, bf, g.db, g.part);
        FT_LAUNCHED();
        return CLIPVIT_OK;
    });
}

}  // extern "C"
