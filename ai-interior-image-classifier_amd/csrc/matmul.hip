// Matrix product of the fine-tuning operators: C[m, n] = sum_k A(m, k) B(n, k) on 16-bit operands, fp32
// accumulation, with the epilogue of finetune.h. Each operand is contiguous along k (a "row panel") or along
// its own index (a "column panel"): a Linear's forward is (k, k), its input gradient (k, column) and its
// weight gradient (column, column), all on the tensors as the user's program holds them.
//
// Tile: WM x WN waves, each FM 16-row fragments x 64 columns, in 32-deep k-steps through a ring of four LDS
// stages filled by buffer loads straight to LDS. The MFMA runs with swapped operands (B rows as its A), so
// a lane holds consecutive columns of one row.
//
// LDS image of a stage: A then B.
//  * row panel (R rows x 32 k, 64 B a row): 16-B chunk c of row r at chunk c ^ ((r >> 2) & 2); fragments by
//    ds_read_b128. B's rows are staged permuted inside each group of 64 (LDS row 16 f + i holds column
//    16 (i >> 2) + 4 f + (i & 3)), which leaves 16 consecutive columns in a lane.
//  * column panel (32 k x R columns, 2 R bytes a k): fragments by ds_read_b64_tr_b16 (lane 4 q + p of a
//    16-lane group supplies k row q, columns 4 p .. 4 p + 3; lane i receives column i of the four k). The
//    32-B unit of a row is XORed with f(k), which makes the eight k rows that a half wave reads distinct in
//    their banks. B's columns stay in order; four lane groups exchange their fragments in the epilogue
//    (permlane32_swap, permlane16_swap) for the same 16 consecutive columns.
// Ragged edges: rows past the matrix and k past K lie outside the buffer resource (or get an offset that
// does) and read as zeros.
#include <type_traits>

#include "finetune.h"

namespace clipvit {
namespace {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
constexpr unsigned OOB = 0xFFFFFFF0u;
constexpr int NS = 4;  // LDS stages

template <int N>
using ic = std::integral_constant<int, N>;

// k-row swizzle of a column panel in 32-B units: R >= 128 columns (rows of at least 256 B) need 8 distinct
// units, 64 columns (two rows per 256 B) 4
template <int R>
__device__ __forceinline__ int col_swz(int k) {
    return R >= 128 ? (k & 3) | ((k >> 1) & 4) : ((k >> 1) & 1) | ((k >> 2) & 2);
}

// One operand's panel of a tile: staging offsets and the per-step resource.
// R rows (row panel) or columns (column panel) from index i0 of `count`; NW waves share its R / 16 pieces of 1 KB.
template <bool KC, int R, int NW, bool PERM>
struct Panel {
    static constexpr int NP = R / 16 / NW;
    const unsigned char* base;
    unsigned long long kstep;  // column panel: bytes of 32 k rows
    unsigned range;            // row panel: bytes; column panel: bytes of its last valid row from the first column
    unsigned ld2;
    int K, chunk;
    unsigned voff[NP];

    __device__ __forceinline__ void init(const u16* p, int64_t ld, int i0, int count, int K_, int w, int lane) {
        const int valid = min(R, count - i0);
        K = K_;
        ld2 = (unsigned)(ld * 2);
        if constexpr (KC) {
            base = (const unsigned char*)(p + (int64_t)i0 * ld);
            range = (unsigned)(valid - 1) * ld2 + (unsigned)((K + 7) & ~7) * 2;  // (rows are padded to 8 elements)
            kstep = 0;
            const int r = lane >> 2;
            chunk = (lane & 3) ^ ((r >> 2) & 2);
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                int row = (w * NP + i) * 16 + r;  // LDS row
                if constexpr (PERM) row = (row & ~63) + 16 * ((row & 15) >> 2) + 4 * ((row >> 4) & 3) + (row & 3);
                voff[i] = row < valid ? (unsigned)row * ld2 + chunk * 16 : OOB;
            }
        } else {
            base = (const unsigned char*)(p + i0);
            range = (unsigned)((valid + 7) & ~7) * 2;
            kstep = (unsigned long long)ld2 * 32;
            chunk = 0;
            constexpr int CPR = R / 8;  // 16-B chunks per k row
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int idx = (w * NP + i) * 64 + lane;
                const int k = idx / CPR, c = (idx % CPR) ^ (col_swz<R>(k) << 1);
                voff[i] = c * 8 < valid ? (unsigned)k * ld2 + c * 16 : OOB;
            }
        }
    }
    // stage k-step kt (32 deep) into dst (this operand's part of a stage, the wave's first piece)
    __device__ __forceinline__ void stage(int kt, int w, unsigned char* dst) const {
        const int left = K - kt * 32;
        unsigned char* d = dst + w * NP * 1024;
        if constexpr (KC) {
            const i32x4_t rs = buf_rsrc(base, left > 0 ? range : 0u);
            const bool in = chunk * 8 < left;
#pragma unroll
            for (int i = 0; i < NP; ++i) blds16(rs, in ? voff[i] : OOB, left > 0 ? kt * 64 : 0, d + i * 1024);
        } else {
            const i32x4_t rs = buf_rsrc(base + (left > 0 ? kstep * (unsigned)kt : 0ull),
                                        left > 0 ? (unsigned)(min(left, 32) - 1) * ld2 + range : 0u);
#pragma unroll
            for (int i = 0; i < NP; ++i) blds16(rs, voff[i], 0, d + i * 1024);
        }
    }
};

template <typename T>
__device__ __forceinline__ typename T::vec8 vec_of(const u32x2& a, const u32x2& b) {
    return __builtin_bit_cast(typename T::vec8, (u32x4){a.x, a.y, b.x, b.y});
}

// Fragment reads: four fragments per asm block, which ends with its own wait (hipcc does not see these
// reads, and a plain LDS read would make it drain the LDS-DMA loads in flight).
template <typename T>
__device__ __forceinline__ void read_rows4(typename T::vec8 (&d)[4], unsigned a) {
    asm volatile(
        "ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:1024\n\tds_read_b128 %2, %4 offset:2048\n\t"
        "ds_read_b128 %3, %4 offset:3072\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(d[0]), "=&v"(d[1]), "=&v"(d[2]), "=&v"(d[3])
        : "v"(a)
        : "memory");
}
template <typename T>
__device__ __forceinline__ void read_rows1(typename T::vec8& d, unsigned a) {
    asm volatile("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(d) : "v"(a) : "memory");
}
// HS = bytes of four k rows
template <typename T, int HS>
__device__ __forceinline__ void read_cols4(typename T::vec8 (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3) {
    u32x2 r[8];
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%12\n\t"
        "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:%12\n\t"
        "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:%12\n\t"
        "ds_read_b64_tr_b16 %6, %11\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
        : "v"(a0), "v"(a1), "v"(a2), "v"(a3), "i"(HS)
        : "memory");
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = vec_of<T>(r[2 * i], r[2 * i + 1]);
}
template <typename T, int HS>
__device__ __forceinline__ void read_cols1(typename T::vec8& d, unsigned a) {
    u32x2 r0, r1;
    asm volatile("ds_read_b64_tr_b16 %0, %2\n\tds_read_b64_tr_b16 %1, %2 offset:%3\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(r0), "=&v"(r1)
                 : "v"(a), "i"(HS)
                 : "memory");
    d = vec_of<T>(r0, r1);
}

// four lane groups exchange their four 4-column fragments: group b then holds columns 16 b .. 16 b + 15
__device__ __forceinline__ void group_transpose(f32x4 (&a)[4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        unsigned x[4];
#pragma unroll
        for (int f = 0; f < 4; ++f) x[f] = __float_as_uint(a[f][r]);
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            const auto s = __builtin_amdgcn_permlane32_swap(x[f], x[f + 2], false, false);
            x[f] = s[0];
            x[f + 2] = s[1];
        }
#pragma unroll
        for (int f = 0; f < 4; f += 2) {
            const auto s = __builtin_amdgcn_permlane16_swap(x[f], x[f + 1], false, false);
            x[f] = s[0];
            x[f + 1] = s[1];
        }
#pragma unroll
        for (int f = 0; f < 4; ++f) a[f][r] = __uint_as_float(x[f]);
    }
}

// part != null: split-k, slice z writes its fp32 partial sums to part + z * M * N4 (row stride N4)
template <typename T, bool AK, bool BK, int WM, int WN, int FM, bool PP>
__global__ __launch_bounds__(64 * WM * WN, PP ? 1 : 2) void matmul_kernel(Matmul a, float* part, int N4, int ksteps) {
    typedef typename T::vec8 vec8;
    constexpr int BM = WM * FM * 16, BN = WN * 64, W = WM * WN;
    constexpr int A_ST = BM * 64, STAGE = (BM + BN) * 64;
    static_assert(!PP || (WM == 2 && WN == 4), "ping-pong: two groups of four waves");
    static_assert(FM == 1 || FM % 4 == 0, "fragment reads come in fours");
    constexpr int NA = PP ? 4 : W;  // waves that stage A (PP: group 0 stages A, group 1 B)
    using PA = Panel<AK, BM, NA, false>;
    using PB = Panel<BK, BN, NA, BK>;
    __shared__ __attribute__((aligned(16))) unsigned char smem[NS * STAGE];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int nM = (a.M + BM - 1) / BM, nN = (a.N + BN - 1) / BN;
    int mt, nt;
    if (!tile_of_block(blockIdx.x, nM, nN, 0, mt, nt)) return;
    const int m0 = mt * BM, n0 = nt * BN;
    // this slice's k range
    const int nk_all = (a.K + 31) >> 5;
    const int kt0 = blockIdx.y * ksteps, nk = min(ksteps, nk_all - kt0);

    PA pa;
    PB pb;
    const int sw = PP ? wn : wave;
    if (!PP || wm == 0) pa.init(a.A, a.lda, m0, a.M, a.K, sw, lane);
    if (!PP || wm == 1) pb.init(a.B, a.ldb, n0, a.N, a.K, sw, lane);
    auto stage = [&](int t) {
        unsigned char* d = smem + (t & (NS - 1)) * STAGE;
        // steps past the slice's end fill a stage that is not read (kept, so that the counted waits hold)
        const int kt = t < nk ? kt0 + t : nk_all;
        if (!PP || wm == 0) pa.stage(kt, sw, d);
        if (!PP || wm == 1) pb.stage(kt, sw, d + A_ST);
    };

    // fragment addresses within a stage
    const int li = lane & 15, g = lane >> 4, q = li >> 2, p = li & 3;
    const unsigned lds0 = (unsigned)(size_t)(LDS_AS unsigned char*)smem;
    unsigned aaddr[AK ? 1 : FM], baddr[BK ? 1 : 4];
    if constexpr (AK) {
        aaddr[0] = lds0 + (wm * FM * 16 + li) * 64 + ((g ^ ((li >> 2) & 2)) << 4);
    } else {
        const int k = 8 * g + q, f = col_swz<BM>(k);
#pragma unroll
        for (int i = 0; i < FM; ++i) aaddr[i] = lds0 + k * (BM * 2) + (((wm * FM + i) ^ f) << 5) + p * 8;
    }
    if constexpr (BK) {
        baddr[0] = lds0 + A_ST + (wn * 64 + li) * 64 + ((g ^ ((li >> 2) & 2)) << 4);
    } else {
        const int k = 8 * g + q, f = col_swz<BN>(k);
#pragma unroll
        for (int i = 0; i < 4; ++i) baddr[i] = lds0 + A_ST + k * (BN * 2) + (((wn * 4 + i) ^ f) << 5) + p * 8;
    }
    vec8 af[FM], bf[4];
    f32x4 acc[FM][4];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto reads = [&](int t) {
        const unsigned so = (unsigned)(t & (NS - 1)) * STAGE;
        if constexpr (BK) read_rows4<T>(bf, baddr[0] + so);
        else read_cols4<T, BN * 8>(bf, baddr[0] + so, baddr[1] + so, baddr[2] + so, baddr[3] + so);
        if constexpr (FM == 1) {
            if constexpr (AK) read_rows1<T>(af[0], aaddr[0] + so);
            else read_cols1<T, BM * 8>(af[0], aaddr[0] + so);
        } else {
#pragma unroll
            for (int i = 0; i < FM; i += 4) {
                vec8 d[4];
                if constexpr (AK) read_rows4<T>(d, aaddr[0] + so + i * 1024);
                else read_cols4<T, BM * 8>(d, aaddr[i] + so, aaddr[i + 1] + so, aaddr[i + 2] + so, aaddr[i + 3] + so);
#pragma unroll
                for (int j = 0; j < 4; ++j) af[i + j] = d[j];
            }
        }
    };
    auto mfmas = [&]() {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = T::mfma16(bf[j], af[i], acc[i][j]);
        __builtin_amdgcn_s_setprio(0);
    };
    auto bar = [&]() {
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };

    if (nk > 0) {
        stage(0);
        stage(1);
        stage(2);
        if constexpr (PP) {
            // Two groups of four waves, one barrier apart: while one issues its 32 MFMAs the other stages
            // k-step t + 3 and reads its fragments. A wave waits for its own pieces of step t + 1 (two
            // younger groups may be in flight) before the barrier that ends slot 2 t + 1.
            constexpr int AHEAD_A = 2 * PA::NP, AHEAD_B = 2 * PB::NP;
            if (wm == 0) {
                vm_wait<AHEAD_A>();
                bar();
                for (int t = 0; t < nk; ++t) {
                    stage(t + 3);
                    reads(t);
                    bar();
                    mfmas();
                    __builtin_amdgcn_sched_barrier(0);
                    vm_wait<AHEAD_A>();
                    bar();
                }
                bar();
            } else {
                vm_wait<AHEAD_B>();
                bar();
                bar();
                for (int t = 0; t < nk; ++t) {
                    stage(t + 3);
                    vm_wait<AHEAD_B>();
                    reads(t);
                    bar();
                    mfmas();
                    bar();
                }
            }
        } else {
            constexpr int AHEAD = 2 * (PA::NP + PB::NP);
            for (int t = 0; t < nk; ++t) {
                vm_wait<AHEAD>();  // this wave's pieces of step t
                bar();             // every wave's; and step t - 1 is read by all
                stage(t + 3);
                reads(t);
                mfmas();
            }
        }
        vm_wait<0>();  // no load into LDS outlives the workgroup
    }

    // ---- epilogue ----
    const uint2 off = a.e.drop.on ? drop_offset(a.e.drop) : make_uint2(0, 0);
    const bool low = !part && a.e.R > 0;
    const int nw = n0 + wn * 64;  // the wave's first column
#pragma unroll 1
    for (int i0 = 0; i0 < FM; ++i0) {
        // (a rolled loop over a register array: the switch below selects the fragment row)
        f32x4 c[4];
#pragma unroll
        for (int i = 0; i < FM; ++i)
            if (i == i0) {
#pragma unroll
                for (int j = 0; j < 4; ++j) c[j] = acc[i][j];
            }
        const int m = m0 + (wm * FM + i0) * 16 + li;
        f32x4 tl[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) tl[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (low) {
            // rank-R term: fragments straight from global memory (u and v rows are padded to 32 columns)
            for (int r = 0; r < a.e.R; r += 32) {
                const u32x4 z = {0u, 0u, 0u, 0u};
                const u32x4 uf = m < a.M ? *(const u32x4*)(a.e.lu + (int64_t)m * a.e.R + r + 8 * g) : z;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int n = nw + (BK ? 16 * (li >> 2) + 4 * j + (li & 3) : 16 * j + li);
                    const u32x4 vf = n < a.N ? *(const u32x4*)(a.e.lv + (int64_t)n * a.e.R + r + 8 * g) : z;
                    tl[j] = T::mfma16(__builtin_bit_cast(vec8, vf), __builtin_bit_cast(vec8, uf), tl[j]);
                }
            }
        }
        if constexpr (!BK) {
            group_transpose(c);
            if (low) group_transpose(tl);
        }
        const int n = nw + 16 * g;
        if (part) {
            if (m < a.M) {
                float* o = part + ((int64_t)blockIdx.y * a.M + m) * N4 + n;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (n + 4 * j < N4) *(f32x4*)(o + 4 * j) = c[j];
            }
            continue;
        }
        float v[16], t[16];
        const bool masked = low && a.e.low_mask;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            v[j] = c[j >> 2][j & 3];
            t[j] = tl[j >> 2][j & 3];
            if (!masked) v[j] += t[j];
        }
        if (masked) epilogue_cols<T, 16, true>(a.e, off, m, n, v, t);
        else epilogue_cols<T, 16, false>(a.e, off, m, n, v, t);
    }
}

// join of a split product: the slices' partial sums in order, then the epilogue; four columns a thread
template <typename T>
__global__ __launch_bounds__(256) void matmul_join_kernel(Epilogue e, const float* __restrict__ part, int N4, int S) {
    const int nq = N4 >> 2;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int m = (int)(i / nq), n = (int)(i - (int64_t)m * nq) * 4;
    if (m >= e.M) return;
    const int64_t sl = (int64_t)e.M * N4;
    const float* p = part + (int64_t)m * N4 + n;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    for (int z = 0; z < S; ++z) s += *(const f32x4*)(p + z * sl);
    float v[4] = {s[0], s[1], s[2], s[3]}, t[4] = {0.f, 0.f, 0.f, 0.f};
    const uint2 off = e.drop.on ? drop_offset(e.drop) : make_uint2(0, 0);
    if (e.R > 0) {
        const u16 *u = e.lu + (int64_t)m * e.R;
        for (int j = 0; j < 4; ++j) {
            if (n + j >= e.N) break;
            const u16* w = e.lv + (int64_t)(n + j) * e.R;
            float d = 0.f;
            for (int r = 0; r < e.R; ++r) d += T::to_f32(u[r]) * T::to_f32(w[r]);
            if (e.low_mask) t[j] = d;
            else v[j] += d;
        }
    }
    if (e.R > 0 && e.low_mask) epilogue_cols<T, 4, true>(e, off, m, n, v, t);
    else epilogue_cols<T, 4, false>(e, off, m, n, v, t);
}

// an operand whose rows the 16-byte loads cannot address (odd length, stride or base): copied to rows of
// `cp` elements (a multiple of 8), zero padded; 8 elements a thread
__global__ __launch_bounds__(256) void repack_kernel(const u16* __restrict__ src, int64_t ld, int rows, int cols, u16* __restrict__ dst, int cp) {
    const int cq = cp >> 3;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t r = i / cq;
    const int c = (int)(i - r * cq) * 8;
    if (r >= rows) return;
    const u16* s = src + r * ld + c;
    u16 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? s[j] : (u16)0;
    uint4 w;
    __builtin_memcpy(&w, v, 16);
    *(uint4*)(dst + r * cp + c) = w;
}

bool loadable(const u16* p, int64_t ld, int len) { return ((size_t)p & 15) == 0 && ld % 8 == 0 && len % 8 == 0; }

struct Plan {
    size_t a_bytes, b_bytes, part_bytes;
    int tile, S, ksteps, N4;  // tile: 0 = 64 x 64, 1 = 128 x 128, 2 = 256 x 256
};

int tiles(int M, int N, int t) { return ((M + t - 1) / t) * ((N + t - 1) / t); }

Plan plan_of(const Matmul& a) {
    Plan p{};
    const int al = a.a_k ? a.K : a.M, ar = a.a_k ? a.M : a.K, bl = a.b_k ? a.K : a.N, br = a.b_k ? a.N : a.K;
    auto up = [](int64_t v, int64_t q) { return (v + q - 1) / q * q; };
    if (a.K > 0 && !loadable(a.A, a.lda, al)) p.a_bytes = (size_t)up((int64_t)ar * up(al, 8) * 2, 256);
    if (a.K > 0 && !loadable(a.B, a.ldb, bl)) p.b_bytes = (size_t)up((int64_t)br * up(bl, 8) * 2, 256);
    p.tile = tiles(a.M, a.N, 256) >= 128 ? 2 : tiles(a.M, a.N, 128) >= 128 ? 1 : 0;
    const int nk = (a.K + 31) / 32;
    p.S = 1;
    p.ksteps = nk > 0 ? nk : 1;
    p.N4 = (int)up(a.N, 4);
    const int nt = p.tile == 2 ? tiles(a.M, a.N, 256) : p.tile == 1 ? tiles(a.M, a.N, 128) : tiles(a.M, a.N, 64);
    if (nt < 256 && nk >= 16) {  // few tiles and a long k: slices of at least 8 k-steps, about 512 workgroups
        int S = min(min(512 / nt, nk / 8), 64);
        if (S > 1) {
            p.ksteps = (nk + S - 1) / S;
            p.S = (nk + p.ksteps - 1) / p.ksteps;
        }
    }
    if (p.S > 1) p.part_bytes = (size_t)p.S * a.M * p.N4 * 4;
    return p;
}

template <typename T, bool AK, bool BK>
void launch_tile(hipStream_t s, const Matmul& a, const Plan& p, float* part) {
    const int bm = p.tile == 2 ? 256 : p.tile == 1 ? 128 : 64;
    const dim3 grid(tiles(a.M, a.N, bm), p.S);
    if (p.tile == 2) matmul_kernel<T, AK, BK, 2, 4, 8, true><<<grid, 512, 0, s>>>(a, part, p.N4, p.ksteps);
    else if (p.tile == 1) matmul_kernel<T, AK, BK, 2, 2, 4, false><<<grid, 256, 0, s>>>(a, part, p.N4, p.ksteps);
    else matmul_kernel<T, AK, BK, 4, 1, 1, false><<<grid, 256, 0, s>>>(a, part, p.N4, p.ksteps);
}

template <typename T>
void launch_typed(hipStream_t s, const Matmul& a, const Plan& p, float* part) {
    if (a.a_k && a.b_k) launch_tile<T, true, true>(s, a, p, part);
    else if (a.a_k) launch_tile<T, true, false>(s, a, p, part);
    else if (a.b_k) launch_tile<T, false, true>(s, a, p, part);
    else launch_tile<T, false, false>(s, a, p, part);
    if (p.S > 1) {
        const int64_t n = (int64_t)a.M * (p.N4 >> 2);
        matmul_join_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(a.e, part, p.N4, p.S);
    }
}

void repack(hipStream_t s, const u16*& p, int64_t& ld, int rows, int len, void* dst) {
    const int cp = (len + 7) / 8 * 8;
    const int64_t n = (int64_t)rows * (cp / 8);
    repack_kernel<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(p, ld, rows, len, (u16*)dst, cp);
    p = (const u16*)dst;
    ld = cp;
}

}  // namespace

size_t matmul_workspace(const Matmul& a) {
    if (a.M <= 0 || a.N <= 0) return 0;
    const Plan p = plan_of(a);
    return p.a_bytes + p.b_bytes + p.part_bytes;
}

int launch_matmul(hipStream_t s, int dtype, const Matmul& a0, void* ws, size_t ws_bytes) {
    if (a0.M <= 0 || a0.N <= 0) return 0;
    Matmul a = a0;
    const Plan p = plan_of(a);
    if (p.a_bytes + p.b_bytes + p.part_bytes > ws_bytes) return -1;
    unsigned char* w = (unsigned char*)ws;
    if (p.a_bytes) {
        repack(s, a.A, a.lda, a.a_k ? a.M : a.K, a.a_k ? a.K : a.M, w);
        w += p.a_bytes;
    }
    if (p.b_bytes) {
        repack(s, a.B, a.ldb, a.b_k ? a.N : a.K, a.b_k ? a.K : a.N, w);
        w += p.b_bytes;
    }
    float* part = p.S > 1 ? (float*)w : nullptr;
    a.e.vec = ((size_t)a.e.y & 15) == 0 && a.e.ldy % 8 == 0 &&
              (!a.e.res || (((size_t)a.e.res & 15) == 0 && a.e.ldr % 8 == 0)) &&
              (!a.e.slope || (((size_t)a.e.slope & 15) == 0 && a.N % 8 == 0));
    if (dtype == 1) launch_typed<BF16>(s, a, p, part);
    else launch_typed<F16>(s, a, p, part);
    return 0;
}

}  // namespace clipvit
