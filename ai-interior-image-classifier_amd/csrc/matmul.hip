// Matrix product of the fine-tuning operators: C[m, n] = sum_k A(m, k) B(n, k) on 16-bit operands, fp32
// accumulation, with the epilogue of finetune.h. Each operand is contiguous along k (a "row panel") or along
// its own index (a "column panel"): a Linear's forward is (k, k), its input gradient (k, column) and its
// weight gradient (column, column), all on the tensors as the user's program holds them.
//
// Every k-tile is 64 deep, so that a row panel's loads are whole 128-byte lines: at 64 bytes a row the products
// of two row panels ran at 873 TFLOP/s where two column panels reached 1213 (8192^3, bf16; the delivered rate is
// requests in flight times their size). Loads go from global memory straight to LDS (buffer_load ... lds). The
// MFMA runs with swapped operands (B rows as its A), so a lane holds four consecutive columns of one row.
//
// LDS image:
//  * row panel (R rows x 64 k, 128 B a row): 16-B chunk c of row r at chunk c ^ (r & 7); fragments by ds_read_b128;
//  * column panel (64 k x R columns, 2 R bytes a k): fragments by ds_read_b64_tr_b16 (lane 4 q + p of a 16-lane
//    group supplies k row q, columns 4 p .. 4 p + 3; lane i receives column i of the four k). The 32-B unit of a
//    row is XORed with a function of k that sends the eight k rows that a half wave reads to distinct banks.
// Ragged edges: rows past the matrix and k past K lie outside the buffer resource (or get an offset that
// does) and read as zeros.
//
// Epilogue: each wave passes its accumulators, 64 rows x 64 columns at a time, through a part of the stages' LDS of its
// own (chunks XORed with the row: no conflicts), and continues with eight consecutive columns a lane: 128 contiguous
// bytes a row for the 16-bit residual, slope and output, whole groups of four for the dropout counter.
#include <type_traits>

#include "finetune.h"

namespace clipvit {
namespace {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
constexpr unsigned OOB = 0xFFFFFFF0u;

// k-row swizzle of a column panel in 32-B units: R >= 128 columns (rows of at least 256 B) need 8 distinct
// units, 64 columns (two rows per 256 B) 4
template <int R>
__device__ __forceinline__ int col_swz(int k) {
    return R >= 128 ? (k & 3) | ((k >> 1) & 4) : ((k >> 1) & 1) | ((k >> 2) & 2);
}

// Position in a panel's LDS image -> row (column) of the tile. Whole: the panel is the tile's operand. Half<H, W>: the
// W-wide halves H of every 2 W rows.
struct Whole {
    static __device__ __forceinline__ int at(int i) { return i; }
};
template <int H, int W>
struct Half {
    static __device__ __forceinline__ int at(int i) { return (i & ~(W - 1)) * 2 + W * H + (i & (W - 1)); }
};

// One operand's panel of a tile: R rows (KC) or columns, staged by NW waves, NP pieces of 1 KB each.
template <bool KC, int R, int NW, class Map>
struct Panel {
    static constexpr int NP = R / 8 / NW;
    const unsigned char* base;
    unsigned long long kstep;  // column panel: bytes of 64 k rows
    unsigned range;            // row panel: bytes; column panel: bytes of its last valid row from the first column
    unsigned ld2;
    int K, chunk;
    unsigned voff[NP];

    // the operand's rows (columns) i0 .. of `count`; this wave is number w of NW
    __device__ __forceinline__ void init(const u16* p, int64_t ld, int i0, int count, int K_, int w, int lane) {
        const int valid = min(count - i0, 1 << 12);
        K = K_;
        ld2 = (unsigned)(ld * 2);
        if constexpr (KC) {
            base = (const unsigned char*)(p + (int64_t)i0 * ld);
            range = (unsigned)(min(valid, 256) - 1) * ld2 + (unsigned)((K + 7) & ~7) * 2;  // (rows are padded to 8 elements)
            kstep = 0;
            const int r = lane >> 3;
            chunk = (lane & 7) ^ r;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int row = Map::at((w * NP + i) * 8 + r);
                voff[i] = row < valid ? (unsigned)row * ld2 + chunk * 16 : OOB;
            }
        } else {
            base = (const unsigned char*)(p + i0);
            range = (unsigned)((min(valid, 256) + 7) & ~7) * 2;
            kstep = (unsigned long long)ld2 * 64;
            chunk = 0;
            constexpr int CPR = R / 8;  // 16-B chunks per k row
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int idx = (w * NP + i) * 64 + lane;
                const int k = idx / CPR, c = Map::at(((idx % CPR) ^ (col_swz<R>(k) << 1)) * 8);
                voff[i] = c < valid ? (unsigned)k * ld2 + c * 2 : OOB;
            }
        }
    }
    // stage k-tile kt into dst (the panel's part of a stage)
    __device__ __forceinline__ void stage(int kt, int w, unsigned char* dst) const {
        const int left = K - kt * 64;
        unsigned char* d = dst + w * NP * 1024;
        if constexpr (KC) {
            const i32x4_t rs = buf_rsrc(base, left > 0 ? range : 0u);
            const bool in = chunk * 8 < left;
#pragma unroll
            for (int i = 0; i < NP; ++i) blds16(rs, in ? voff[i] : OOB, left > 0 ? kt * 128 : 0, d + i * 1024);
        } else {
            const i32x4_t rs = buf_rsrc(base + (left > 0 ? kstep * (unsigned)kt : 0ull),
                                        left > 0 ? (unsigned)(min(left, 64) - 1) * ld2 + range : 0u);
#pragma unroll
            for (int i = 0; i < NP; ++i) blds16(rs, voff[i], 0, d + i * 1024);
        }
    }
};

// k-tile j of a low-rank factor [count, rank] (contiguous rows, rank % 32 == 0), as a row panel from row i0
template <int R, int NW, class Map>
__device__ __forceinline__ void stage_low(const u16* low, int rank, int i0, int count, int j, int w, int lane, unsigned char* dst) {
    const int valid = min(count - i0, 256), r = lane >> 3, chunk = (lane & 7) ^ r;
    const i32x4_t rs = buf_rsrc(low + (int64_t)i0 * rank, (unsigned)valid * (unsigned)rank * 2);
#pragma unroll
    for (int i = 0; i < R / 8 / NW; ++i) {
        const int piece = w * (R / 8 / NW) + i, row = Map::at(piece * 8 + r);
        const bool in = row < valid && j * 64 + chunk * 8 < rank;
        blds16(rs, in ? (unsigned)(row * rank + j * 64 + chunk * 8) * 2 : OOB, 0, dst + piece * 1024);
    }
}

// 32 ranks (from 32 j on) of rows i0 .. i0 + 255 of a low-rank factor: 64 bytes a row, its four chunks swizzled by the row
__device__ __forceinline__ void stage_low32(const u16* low, int rank, int i0, int count, int j, int w, int lane, unsigned char* dst) {
    const int valid = min(count - i0, 256);
    const i32x4_t rs = buf_rsrc(low + (int64_t)i0 * rank, (unsigned)valid * (unsigned)rank * 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int piece = w * 4 + i, row = piece * 16 + (lane >> 2), chunk = (lane & 3) ^ ((row >> 2) & 3);
        blds16(rs, row < valid ? (unsigned)(row * rank + j * 32 + chunk * 8) * 2 : OOB, 0, dst + piece * 1024);
    }
}

// Fragment reads of FR (1, 2 or 4) 16-row fragments x 64 k from position i0 of a panel. Each asm block ends with its own
// wait (hipcc does not see these reads, and a plain LDS read would make it drain the LDS-DMA loads in flight).
template <typename T, bool KC, int R, int FR>
struct Frags {
    typedef typename T::vec8 vec8;
    unsigned addr[KC ? 2 : FR];  // row panel: k halves 0, 1; column panel: one per fragment
    __device__ __forceinline__ void init(unsigned lds, int i0, int lane) {
        const int li = lane & 15, g = lane >> 4;
        if constexpr (KC) {
            addr[0] = lds + (i0 + li) * 128 + ((g ^ (li & 7)) << 4);
            addr[1] = lds + (i0 + li) * 128 + (((4 + g) ^ (li & 7)) << 4);
        } else {
            const int k = 8 * g + (li >> 2), f = col_swz<R>(k);
#pragma unroll
            for (int i = 0; i < FR; ++i) addr[i] = lds + k * (R * 2) + (((i0 / 16 + i) ^ f) << 5) + (li & 3) * 8;
        }
    }
    __device__ __forceinline__ void read(vec8 (&d)[2][FR], unsigned so) const {
        if constexpr (KC && FR == 4) {
            asm volatile(
                "ds_read_b128 %0, %8\n\tds_read_b128 %1, %8 offset:2048\n\tds_read_b128 %2, %8 offset:4096\n\t"
                "ds_read_b128 %3, %8 offset:6144\n\tds_read_b128 %4, %9\n\tds_read_b128 %5, %9 offset:2048\n\t"
                "ds_read_b128 %6, %9 offset:4096\n\tds_read_b128 %7, %9 offset:6144\n\ts_waitcnt lgkmcnt(0)"
                : "=&v"(d[0][0]), "=&v"(d[0][1]), "=&v"(d[0][2]), "=&v"(d[0][3]), "=&v"(d[1][0]), "=&v"(d[1][1]),
                  "=&v"(d[1][2]), "=&v"(d[1][3])
                : "v"(addr[0] + so), "v"(addr[1] + so)
                : "memory");
        } else if constexpr (KC && FR == 2) {
            asm volatile(
                "ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:2048\n\tds_read_b128 %2, %5\n\t"
                "ds_read_b128 %3, %5 offset:2048\n\ts_waitcnt lgkmcnt(0)"
                : "=&v"(d[0][0]), "=&v"(d[0][1]), "=&v"(d[1][0]), "=&v"(d[1][1])
                : "v"(addr[0] + so), "v"(addr[1] + so)
                : "memory");
        } else if constexpr (KC) {
            asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %3\n\ts_waitcnt lgkmcnt(0)"
                         : "=&v"(d[0][0]), "=&v"(d[1][0])
                         : "v"(addr[0] + so), "v"(addr[1] + so)
                         : "memory");
        } else if constexpr (FR == 4) {
            u32x2 r[16];
            asm volatile(
                "ds_read_b64_tr_b16 %0, %16\n\tds_read_b64_tr_b16 %1, %16 offset:%20\n\t"
                "ds_read_b64_tr_b16 %2, %17\n\tds_read_b64_tr_b16 %3, %17 offset:%20\n\t"
                "ds_read_b64_tr_b16 %4, %18\n\tds_read_b64_tr_b16 %5, %18 offset:%20\n\t"
                "ds_read_b64_tr_b16 %6, %19\n\tds_read_b64_tr_b16 %7, %19 offset:%20\n\t"
                "ds_read_b64_tr_b16 %8, %16 offset:%21\n\tds_read_b64_tr_b16 %9, %16 offset:%22\n\t"
                "ds_read_b64_tr_b16 %10, %17 offset:%21\n\tds_read_b64_tr_b16 %11, %17 offset:%22\n\t"
                "ds_read_b64_tr_b16 %12, %18 offset:%21\n\tds_read_b64_tr_b16 %13, %18 offset:%22\n\t"
                "ds_read_b64_tr_b16 %14, %19 offset:%21\n\tds_read_b64_tr_b16 %15, %19 offset:%22\n\ts_waitcnt lgkmcnt(0)"
                : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7]),
                  "=&v"(r[8]), "=&v"(r[9]), "=&v"(r[10]), "=&v"(r[11]), "=&v"(r[12]), "=&v"(r[13]), "=&v"(r[14]), "=&v"(r[15])
                : "v"(addr[0] + so), "v"(addr[1] + so), "v"(addr[2] + so), "v"(addr[3] + so), "i"(R * 8), "i"(R * 64), "i"(R * 72)
                : "memory");
#pragma unroll
            for (int i = 0; i < 8; ++i)
                d[i >> 2][i & 3] = __builtin_bit_cast(vec8, (u32x4){r[2 * i].x, r[2 * i].y, r[2 * i + 1].x, r[2 * i + 1].y});
        } else if constexpr (FR == 2) {
            u32x2 r[8];
            asm volatile(
                "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%10\n\t"
                "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:%10\n\t"
                "ds_read_b64_tr_b16 %4, %8 offset:%11\n\tds_read_b64_tr_b16 %5, %8 offset:%12\n\t"
                "ds_read_b64_tr_b16 %6, %9 offset:%11\n\tds_read_b64_tr_b16 %7, %9 offset:%12\n\ts_waitcnt lgkmcnt(0)"
                : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
                : "v"(addr[0] + so), "v"(addr[1] + so), "i"(R * 8), "i"(R * 64), "i"(R * 72)
                : "memory");
#pragma unroll
            for (int i = 0; i < 4; ++i)
                d[i >> 1][i & 1] = __builtin_bit_cast(vec8, (u32x4){r[2 * i].x, r[2 * i].y, r[2 * i + 1].x, r[2 * i + 1].y});
        } else {
            u32x2 r[4];
            asm volatile(
                "ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %4 offset:%5\n\t"
                "ds_read_b64_tr_b16 %2, %4 offset:%6\n\tds_read_b64_tr_b16 %3, %4 offset:%7\n\ts_waitcnt lgkmcnt(0)"
                : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
                : "v"(addr[0] + so), "i"(R * 8), "i"(R * 64), "i"(R * 72)
                : "memory");
#pragma unroll
            for (int i = 0; i < 2; ++i)
                d[i][0] = __builtin_bit_cast(vec8, (u32x4){r[2 * i].x, r[2 * i].y, r[2 * i + 1].x, r[2 * i + 1].y});
        }
    }
};

// Block -> tile. Blocks b, b + 8, .. share an XCD (speed only): each XCD takes a contiguous range of an order that
// walks bands of six tile rows column by column, so the 32 tiles it runs at a time are about 6 x 5 and share their
// operand panels in its L2 (against tiles in row-major order: 18464 x 1024 x 4096 forward 200 -> 167 us,
// 36928 x 1024 x 4096 370 -> 330 us; bands of 4 and 8 rows measure the same within 1 %).
__device__ __forceinline__ void tile_at(int bid, int nM, int nN, int& mt, int& nt) {
    constexpr int G = 6;
    const int nwg = nM * nN;
    const int q = nwg >> 3, r = nwg & 7, x = bid & 7;
    const int t = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (bid >> 3);
    const int band = t / (G * nN), m0 = band * G, gm = min(G, nM - m0), rr = t - band * G * nN;
    nt = rr / gm;
    mt = m0 + rr - nt * gm;
}

__device__ __forceinline__ void bar() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
}

// KS times 32 ranks of the low-rank term from their fragments; masked, in the accumulators' layout, where a lane's four
// columns are one counter of the generator (a fragment at a time: the scheduler would otherwise spill)
template <typename T, int FR, int FB, int J0, int KS, int FM>
__device__ __forceinline__ void low_acc(const Epilogue& e, const uint2& off, const typename T::vec8 (&a)[KS][FR], const typename T::vec8 (&b)[KS][FB],
                                        f32x4 (&acc)[FM][4], int i0, int m, int n) {
    if (!e.low_mask) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int i = 0; i < FR; ++i)
#pragma unroll
                for (int j = 0; j < FB; ++j) acc[i0 + i][J0 + j] = T::mfma16(b[ks][j], a[ks][i], acc[i0 + i][J0 + j]);
        return;
    }
#pragma unroll
    for (int i = 0; i < FR; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j) {
            f32x4 t = T::mfma16(b[0][j], a[0][i], f32x4{0.f, 0.f, 0.f, 0.f});
            if constexpr (KS == 2) t = T::mfma16(b[1][j], a[1][i], t);
            float t0 = t[0], t1 = t[1], t2 = t[2], t3 = t[3];
            drop4(e.drop, off, e.m_base + m + 16 * i, n + 16 * (J0 + j), 1.0f, t0, t1, t2, t3);
            acc[i0 + i][J0 + j] += f32x4{t0, t1, t2, t3};
            __builtin_amdgcn_sched_barrier(0);
        }
}

// acc[i][j]: rows mw + 16 i .., columns nw + 16 j .. of C, in the MFMA's layout (lane: row lane & 15, columns
// 4 (lane >> 4) .. + 3). eb: LDS of this wave's own, 4 KB for each of up to four fragment rows. part != null: the
// slice's fp32 sums, row stride N4.
template <typename T, int FM>
__device__ __forceinline__ void store_tile(const Matmul& a, f32x4 (&acc)[FM][4], int mw, int nw, float* eb, float* part, int N4, int lane) {
    const Epilogue& e = a.e;
    constexpr int H = FM < 4 ? FM : 4;
    const int li = lane & 15, g = lane >> 4, er = lane >> 3, ec = lane & 7;
    const int n = nw + 8 * ec;
    if (mw >= a.M || nw >= (part ? N4 : a.N)) return;
    const uint2 off = e.drop.on ? drop_offset(e.drop) : make_uint2(0, 0);
    auto get = [&](int row, float (&v)[8]) {
        const f32x4 x = *(const f32x4*)(eb + row * 64 + (((2 * ec) ^ (row & 15)) << 2));
        const f32x4 y = *(const f32x4*)(eb + row * 64 + (((2 * ec + 1) ^ (row & 15)) << 2));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = x[j];
            v[4 + j] = y[j];
        }
    };
    float b[8];
    if (!part) bias_cols<T, 8>(e, n, b);
    const bool full = !part && e.vec && mw + 16 * FM <= a.M && nw + 64 <= a.N;
    const int64_t r0 = mw + er;
    u16* y = (u16*)e.y + r0 * e.ldy + n;
    const u16* res = (const u16*)e.res + r0 * e.ldr + n;
    short* sl = e.slope + r0 * e.N + n;
    const bool drop = e.drop.on && !e.low_mask;
#pragma unroll
    for (int i0 = 0; i0 < FM; i0 += H) {
#pragma unroll
        for (int i = 0; i < H; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) *(f32x4*)(eb + (i * 16 + li) * 64 + (((4 * j + g) ^ li) << 2)) = acc[i0 + i][j];
        const int mr = mw + 16 * i0;
        if (part) {
#pragma unroll 1
            for (int s = 0; s < 2 * H; ++s) {
                const int m = mr + 8 * s + er;
                float v[8];
                get(8 * s + er, v);
                if (m < a.M && n < N4) {
                    float* o = part + (int64_t)m * N4 + n;
                    *(f32x4*)o = f32x4{v[0], v[1], v[2], v[3]};
                    if (n + 4 < N4) *(f32x4*)(o + 4) = f32x4{v[4], v[5], v[6], v[7]};
                }
            }
        } else if (full) {
            // every row and column of the wave's part is inside C and 16-byte aligned
#pragma unroll 2
            for (int s = 0; s < 2 * H; ++s) {
                float v[8], gr[8];
                get(8 * s + er, v);
                u32x4 rw;
                if (e.res) {
                    rw = *(const u32x4*)res;
                    res += 8 * e.ldr;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += b[j];
                if (e.act != ACT_NONE) {
                    if (e.slope) {
                        act_cols<true, 8>(e.act, v, gr);
                        short q[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) q[j] = SlopeCode<T>::encode(gr[j]);
                        u32x4 w;
                        __builtin_memcpy(&w, q, 16);
                        if (e.nt) __builtin_nontemporal_store(w, (u32x4*)sl);
                        else *(u32x4*)sl = w;
                        sl += 8 * (int64_t)e.N;
                    } else {
                        act_cols<false, 8>(e.act, v, gr);
                    }
                }
                if (drop) {
                    const int m = e.m_base + mr + 8 * s + er;
                    drop4(e.drop, off, m, n, e.drop.scale, v[0], v[1], v[2], v[3]);
                    drop4(e.drop, off, m, n + 4, e.drop.scale, v[4], v[5], v[6], v[7]);
                }
                if (e.res) {
                    u16 rr[8];
                    __builtin_memcpy(rr, &rw, 16);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] += T::to_f32(rr[j]);
                }
                const u32x4 w = {pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7])};
                if (e.nt) __builtin_nontemporal_store(w, (u32x4*)y);
                else *(u32x4*)y = w;
                y += 8 * e.ldy;
            }
        } else {
#pragma unroll 1
            for (int s = 0; s < 2 * H; ++s) {
                float v[8];
                get(8 * s + er, v);
                epilogue_cols<T, 8>(e, off, mr + 8 * s + er, n, v, b);
            }
        }
    }
}

// One step's fragment reads of the 256 x 256 tile: A's four fragments and B's two, 64 k each, from 128-wide half panels,
// then TAIL (the barrier) and only then the wait: the reads land while the wave waits at the barrier. All of it is one
// asm block, so no register of a read in flight is visible to the compiler.
#define STEP_A_ROWS                                                                                       \
    "ds_read_b128 %[a0], %[pa0]\n\tds_read_b128 %[a1], %[pa0] offset:2048\n\t"                            \
    "ds_read_b128 %[a2], %[pa0] offset:4096\n\tds_read_b128 %[a3], %[pa0] offset:6144\n\t"                \
    "ds_read_b128 %[a4], %[pa1]\n\tds_read_b128 %[a5], %[pa1] offset:2048\n\t"                            \
    "ds_read_b128 %[a6], %[pa1] offset:4096\n\tds_read_b128 %[a7], %[pa1] offset:6144\n\t"
#define STEP_B_ROWS                                                                                       \
    "ds_read_b128 %[b0], %[pb0]\n\tds_read_b128 %[b1], %[pb0] offset:2048\n\t"                            \
    "ds_read_b128 %[b2], %[pb1]\n\tds_read_b128 %[b3], %[pb1] offset:2048\n\t"
// column panels of 128 columns: four k rows are 1024 bytes, 32 are 8192
#define STEP_COL(d, e, f, g, p)                                                                           \
    "ds_read_b64_tr_b16 %[" d "], %[" p "]\n\tds_read_b64_tr_b16 %[" e "], %[" p "] offset:1024\n\t"      \
    "ds_read_b64_tr_b16 %[" f "], %[" p "] offset:8192\n\tds_read_b64_tr_b16 %[" g "], %[" p "] offset:9216\n\t"
#define STEP_A_COLS                                                                                       \
    STEP_COL("a0", "a1", "a8", "a9", "pa0") STEP_COL("a2", "a3", "aa", "ab", "pa1")                       \
    STEP_COL("a4", "a5", "ac", "ad", "pa2") STEP_COL("a6", "a7", "ae", "af", "pa3")
#define STEP_B_COLS STEP_COL("b0", "b1", "b4", "b5", "pb0") STEP_COL("b2", "b3", "b6", "b7", "pb1")
#define OUT_A_ROWS                                                                                        \
    [a0] "=&v"(a[0][0]), [a1] "=&v"(a[0][1]), [a2] "=&v"(a[0][2]), [a3] "=&v"(a[0][3]), [a4] "=&v"(a[1][0]),  \
    [a5] "=&v"(a[1][1]), [a6] "=&v"(a[1][2]), [a7] "=&v"(a[1][3])
#define OUT_B_ROWS [b0] "=&v"(b[0][0]), [b1] "=&v"(b[0][1]), [b2] "=&v"(b[1][0]), [b3] "=&v"(b[1][1])
#define OUT_A_COLS                                                                                        \
    [a0] "=&v"(ra[0]), [a1] "=&v"(ra[1]), [a2] "=&v"(ra[2]), [a3] "=&v"(ra[3]), [a4] "=&v"(ra[4]),       \
    [a5] "=&v"(ra[5]), [a6] "=&v"(ra[6]), [a7] "=&v"(ra[7]), [a8] "=&v"(ra[8]), [a9] "=&v"(ra[9]),       \
    [aa] "=&v"(ra[10]), [ab] "=&v"(ra[11]), [ac] "=&v"(ra[12]), [ad] "=&v"(ra[13]), [ae] "=&v"(ra[14]),  \
    [af] "=&v"(ra[15])
#define OUT_B_COLS                                                                                        \
    [b0] "=&v"(rb[0]), [b1] "=&v"(rb[1]), [b2] "=&v"(rb[2]), [b3] "=&v"(rb[3]), [b4] "=&v"(rb[4]),       \
    [b5] "=&v"(rb[5]), [b6] "=&v"(rb[6]), [b7] "=&v"(rb[7])
#define IN_A_ROWS [pa0] "v"(fa.addr[0] + sa), [pa1] "v"(fa.addr[1] + sa)
#define IN_A_COLS [pa0] "v"(fa.addr[0] + sa), [pa1] "v"(fa.addr[1] + sa), [pa2] "v"(fa.addr[2] + sa), [pa3] "v"(fa.addr[3] + sa)
#define IN_B [pb0] "v"(fb.addr[0] + sb), [pb1] "v"(fb.addr[1] + sb)
#define STEP_ASM(READS, TAIL, OUTS, INS) asm volatile(READS TAIL "s_barrier\n\ts_waitcnt lgkmcnt(0)" : OUTS : INS : "memory")
#define COMMA ,
#define STEP(TAIL)                                                                                                           \
    if constexpr (AK && BK) STEP_ASM(STEP_B_ROWS STEP_A_ROWS, TAIL, OUT_B_ROWS COMMA OUT_A_ROWS, IN_B COMMA IN_A_ROWS);        \
    else if constexpr (AK) STEP_ASM(STEP_B_COLS STEP_A_ROWS, TAIL, OUT_B_COLS COMMA OUT_A_ROWS, IN_B COMMA IN_A_ROWS);         \
    else if constexpr (BK) STEP_ASM(STEP_B_ROWS STEP_A_COLS, TAIL, OUT_B_ROWS COMMA OUT_A_COLS, IN_B COMMA IN_A_COLS);         \
    else STEP_ASM(STEP_B_COLS STEP_A_COLS, TAIL, OUT_B_COLS COMMA OUT_A_COLS, IN_B COMMA IN_A_COLS);
// VM8: also waits until at most eight of the wave's loads are in flight before the barrier
template <typename T, bool AK, bool BK, bool VM8>
__device__ __forceinline__ void read_step(const Frags<T, AK, 128, 4>& fa, unsigned sa, typename T::vec8 (&a)[2][4], const Frags<T, BK, 128, 2>& fb,
                                          unsigned sb, typename T::vec8 (&b)[2][2]) {
    typedef typename T::vec8 vec8;
    u32x2 ra[AK ? 1 : 16], rb[BK ? 1 : 8];
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (VM8) {
        STEP("s_waitcnt vmcnt(8)\n\t")
    } else {
        STEP("")
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (!AK) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            a[i >> 2][i & 3] = __builtin_bit_cast(vec8, (u32x4){ra[2 * i].x, ra[2 * i].y, ra[2 * i + 1].x, ra[2 * i + 1].y});
    }
    if constexpr (!BK) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            b[i >> 1][i & 1] = __builtin_bit_cast(vec8, (u32x4){rb[2 * i].x, rb[2 * i].y, rb[2 * i + 1].x, rb[2 * i + 1].y});
    }
}

// 256 x 256 tiles. Eight waves in two groups of four, one barrier apart: while one group issues 32 MFMAs the other
// reads its next fragments. A k-tile T is two steps: step (T, 0) computes the group's first 64 rows, (T, 1) its other
// 64. B's fragments stay in registers for both; to balance the reads, step (T, 0) reads A's first half and B's second
// 32 columns of T, step (T, 1) A's second half and B's first 32 columns of T + 1. Slot = barrier interval; group g
// issues the reads of step (T, h) in slot 4 T + 2 h + g, has them at the start of the next slot and computes there.
// LDS holds two k-tiles. A part read in slots s (group 0) and s + 1 (group 1) is out of every wave's reads before the
// barrier that ends slot s + 2, and is refilled from slot s + 3 on:
//  * A0(T), read in 4 T and 4 T + 1, by A0(T + 2) in slot 4 T + 3; A1(T - 1), read in 4 T - 2 and 4 T - 1, by A1(T + 1) in
//    slot 4 T + 1: group 0, at the start of its MFMA segments. At their end it waits for its four oldest pieces (eight
//    younger ones may fly): five slots after their issue, one before their first read.
//  * B0(T), read in 4 T - 2 and 4 T - 1, by B0(T + 2) in slot 4 T + 1; B1(T), read in 4 T and 4 T + 1, by B1(T + 2) in
//    slot 4 T + 3: group 1, in its read segments, where it also waits, five slots after the issue.
// Steps past the last k-tile stage zeros into parts nobody reads (kept, so that the counted waits hold).
// Bound by the MFMA segments and what a slot adds to their 512 cycles (barrier, waits, staging): at 8192^3 bf16 805 us,
// 1360 TFLOP/s, for the forward's layouts, 795 us for dx's, 820 us for dw's (a library product of that size: 700 us). With
// the reads waited for before the barrier and refills a slot earlier it was 874 us; issuing the staging between the
// MFMAs instead of before them changed nothing (778-794 against 789-791 us on one card). A tile costs 8.5 us besides its
// k-tiles' 1.4 us each, of which the epilogue is 6 (11 with quick_gelu, whose exponential and reciprocal are quarter rate).
template <typename T, bool AK, bool BK>
__global__ __launch_bounds__(512, 1) void matmul256_kernel(Matmul a, float* part, int N4, int kslice) {
    typedef typename T::vec8 vec8;
    using PA0 = Panel<AK, 128, 4, Half<0, 64>>;
    using PA1 = Panel<AK, 128, 4, Half<1, 64>>;
    using PB0 = Panel<BK, 128, 4, Half<0, 32>>;
    using PB1 = Panel<BK, 128, 4, Half<1, 32>>;
    constexpr int HALF = 16384, ST = 32768, B_OFF = 65536, LOW = 131072;
    __shared__ __attribute__((aligned(16))) unsigned char smem[163840];  // two k-tiles, 32 ranks of the low-rank factors
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 2, wn = wave & 3;
    const int nM = (a.M + 255) / 256, nN = (a.N + 255) / 256;
    int mt, nt;
    tile_at(blockIdx.x, nM, nN, mt, nt);
    const int m0 = mt * 256, n0 = nt * 256;
    const int nk_all = (a.K + 63) >> 6;
    const int kt0 = blockIdx.y * kslice, nk = min(kslice, nk_all - kt0);
    auto kt_of = [&](int t) { return t < nk ? kt0 + t : nk_all; };

    const unsigned lds = (unsigned)(size_t)(LDS_AS unsigned char*)smem;
    Frags<T, AK, 128, 4> fa;
    Frags<T, BK, 128, 2> fb;
    fa.init(lds, wm * 64, lane);
    fb.init(lds + B_OFF, wn * 32, lane);
    vec8 af[2][4], b0[2][2], b1[2][2], bn[2][2];
    f32x4 acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto mfmas = [&](auto half) {
        constexpr int H = decltype(half)::value * 4;
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[H + i][j] = T::mfma16(j < 2 ? b0[ks][j & 1] : b1[ks][j & 1], af[ks][i], acc[H + i][j]);
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto next_b0 = [&]() {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int j = 0; j < 2; ++j) b0[ks][j] = bn[ks][j];
    };
    using H0 = std::integral_constant<int, 0>;
    using H1 = std::integral_constant<int, 1>;
    const bool low = a.e.R > 0 && blockIdx.y == 0;
    auto low_stage = [&](int j) {
        if (wm == 0) stage_low32(a.e.lu, a.e.R, m0, a.M, j, wn, lane, smem + LOW);
        else stage_low32(a.e.lv, a.e.R, n0, a.N, j, wn, lane, smem + LOW + 16384);
    };
    if (low) low_stage(0);  // (the oldest loads: the counted waits below include them)
    if (nk > 0) {
        if (wm == 0) {
            PA0 p0;
            PA1 p1;
            p0.init(a.A, a.lda, m0, a.M, a.K, wn, lane);
            p1.init(a.A, a.lda, m0, a.M, a.K, wn, lane);
            p0.stage(kt_of(0), wn, smem);
            p1.stage(kt_of(0), wn, smem + HALF);
            p0.stage(kt_of(1), wn, smem + ST);
            vm_wait<8>();
            bar();
            fb.read(b0, 0);
            bar();
            for (int t = 0; t < nk; ++t) {
                const int so = (t & 1) * ST;
                read_step<T, AK, BK, false>(fa, so, af, fb, so + HALF, b1);
                p1.stage(kt_of(t + 1), wn, smem + (so ^ ST) + HALF);
                mfmas(H0{});
                vm_wait<8>();
                bar();
                read_step<T, AK, BK, false>(fa, so + HALF, af, fb, so ^ ST, bn);
                p0.stage(kt_of(t + 2), wn, smem + so);
                mfmas(H1{});
                next_b0();
                vm_wait<8>();
                bar();
            }
            bar();
        } else {
            PB0 p0;
            PB1 p1;
            p0.init(a.B, a.ldb, n0, a.N, a.K, wn, lane);
            p1.init(a.B, a.ldb, n0, a.N, a.K, wn, lane);
            p0.stage(kt_of(0), wn, smem + B_OFF);
            p1.stage(kt_of(0), wn, smem + B_OFF + HALF);
            p0.stage(kt_of(1), wn, smem + B_OFF + ST);
            p1.stage(kt_of(1), wn, smem + B_OFF + ST + HALF);
            vm_wait<8>();
            bar();
            fb.read(b0, 0);
            bar();
            bar();
            for (int t = 0; t < nk; ++t) {
                const int so = (t & 1) * ST;
                p0.stage(kt_of(t + 2), wn, smem + B_OFF + so);
                read_step<T, AK, BK, true>(fa, so, af, fb, so + HALF, b1);
                mfmas(H0{});
                bar();
                p1.stage(kt_of(t + 2), wn, smem + B_OFF + so + HALF);
                read_step<T, AK, BK, true>(fa, so + HALF, af, fb, so ^ ST, bn);
                mfmas(H1{});
                next_b0();
                bar();
            }
        }
        vm_wait<0>();  // no load into LDS outlives the k loop: the epilogue takes the stages over
        bar();
    }
    if (low) {
        // rank-R term, 32 ranks at a time, the first ones staged before the k loop. (All staged after it like k-tiles, 64 a
        // step: training step of 18464 x 1024 x 4096, rank 16, 492 against 481 us on one card. Fragments straight from global
        // memory cost 14 us a round of tiles; as further k-tiles of the loop, their branch slowed the loop by a quarter.)
        const uint2 off = a.e.drop.on ? drop_offset(a.e.drop) : make_uint2(0, 0);
        const int li = lane & 15, g = lane >> 4;
        const unsigned char* pa = smem + LOW + (wm * 128 + li) * 64 + ((g ^ (li >> 2)) << 4);
        const unsigned char* pb = smem + LOW + 16384 + (wn * 64 + li) * 64 + ((g ^ (li >> 2)) << 4);
        vm_wait<0>();
        bar();
#pragma unroll 1
        for (int j = 0; j * 32 < a.e.R; ++j) {
            if (j) {
                bar();  // every wave has read the ranks before
                low_stage(j);
                vm_wait<0>();
                bar();
            }
            asm volatile("" ::: "memory");
            vec8 u[1][4], v[1][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[0][i] = *(const vec8*)(pb + i * 1024);
#pragma unroll
            for (int i = 0; i < 4; ++i) u[0][i] = *(const vec8*)(pa + i * 1024);
            low_acc<T, 4, 4, 0>(a.e, off, u, v, acc, 0, m0 + wm * 128 + li, n0 + wn * 64 + 4 * g);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 4; ++i) u[0][i] = *(const vec8*)(pa + 4096 + i * 1024);
            low_acc<T, 4, 4, 0>(a.e, off, u, v, acc, 4, m0 + wm * 128 + 64 + li, n0 + wn * 64 + 4 * g);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }
    store_tile<T, 8>(a, acc, m0 + wm * 128, n0 + wn * 64, (float*)smem + wave * 4096,
                     part ? part + (int64_t)blockIdx.y * a.M * N4 : nullptr, N4, lane);
}

// Smaller tiles: WM x WN waves of FM x 16 rows x 64 columns, NS stages, one barrier a k-tile. (Eight stages of the 64 x 64
// tile where there is at most one workgroup a CU measured slower than three: 1 x 512 x 2048 7.1 against 6.6 us.)
template <typename T, bool AK, bool BK, int WM, int WN, int FM, int NS>
__global__ __launch_bounds__(64 * WM * WN, 2) void matmul_kernel(Matmul a, float* part, int N4, int kslice) {
    typedef typename T::vec8 vec8;
    constexpr int BM = WM * FM * 16, BN = WN * 64, W = WM * WN;
    constexpr int A_ST = BM * 128, STAGE = (BM + BN) * 128;
    using PA = Panel<AK, BM, W, Whole>;
    using PB = Panel<BK, BN, W, Whole>;
    __shared__ __attribute__((aligned(16))) unsigned char smem[NS * STAGE];
    static_assert(NS * STAGE >= W * 4096 * FM, "the epilogue's LDS");
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int nM = (a.M + BM - 1) / BM, nN = (a.N + BN - 1) / BN;
    int mt, nt;
    tile_at(blockIdx.x, nM, nN, mt, nt);
    const int m0 = mt * BM, n0 = nt * BN;
    const int nk_all = (a.K + 63) >> 6;
    const int kt0 = blockIdx.y * kslice, nk = min(kslice, nk_all - kt0);

    PA pa;
    PB pb;
    pa.init(a.A, a.lda, m0, a.M, a.K, wave, lane);
    pb.init(a.B, a.ldb, n0, a.N, a.K, wave, lane);
    auto stage = [&](int t, int st) {
        const int kt = t < nk ? kt0 + t : nk_all;  // past the slice: zeros into a stage nobody reads
        pa.stage(kt, wave, smem + st * STAGE);
        pb.stage(kt, wave, smem + st * STAGE + A_ST);
    };
    const unsigned lds = (unsigned)(size_t)(LDS_AS unsigned char*)smem;
    Frags<T, AK, BM, FM> fa;
    Frags<T, BK, BN, 4> fb;
    fa.init(lds, wm * FM * 16, lane);
    fb.init(lds + A_ST, wn * 64, lane);
    vec8 af[2][FM], bf[2][4];
    f32x4 acc[FM][4];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (nk > 0) {
        constexpr int NP = PA::NP + PB::NP;
#pragma unroll
        for (int t = 0; t < NS - 1; ++t) stage(t, t);
        int st = 0;
        for (int t = 0; t < nk; ++t) {
            vm_wait<(NS - 2) * NP>();  // this wave's pieces of k-tile t
            bar();                     // every wave's; and k-tile t - 1 is read by all
            stage(t + NS - 1, st == 0 ? NS - 1 : st - 1);
            fb.read(bf, st * STAGE);
            fa.read(af, st * STAGE);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = T::mfma16(bf[ks][j], af[ks][i], acc[i][j]);
            __builtin_amdgcn_s_setprio(0);
            st = st == NS - 1 ? 0 : st + 1;
        }
        vm_wait<0>();  // no load into LDS outlives the k loop: the epilogue takes the stages over
        bar();
    }
    if (a.e.R > 0 && blockIdx.y == 0) {  // as above
        const uint2 off = a.e.drop.on ? drop_offset(a.e.drop) : make_uint2(0, 0);
        Frags<T, true, BM, FM> la;
        Frags<T, true, BN, 4> lb;
        la.init(lds, wm * FM * 16, lane);
        lb.init(lds + A_ST, wn * 64, lane);
#pragma unroll 1
        for (int j = 0; j * 64 < a.e.R; ++j) {
            stage_low<BM, W, Whole>(a.e.lu, a.e.R, m0, a.M, j, wave, lane, smem);
            stage_low<BN, W, Whole>(a.e.lv, a.e.R, n0, a.N, j, wave, lane, smem + A_ST);
            vm_wait<0>();
            bar();
            lb.read(bf, 0);
            la.read(af, 0);
            low_acc<T, FM, 4, 0>(a.e, off, af, bf, acc, 0, m0 + wm * FM * 16 + (lane & 15), n0 + wn * 64 + 4 * (lane >> 4));
            bar();
        }
    }
    store_tile<T, FM>(a, acc, m0 + wm * FM * 16, n0 + wn * 64, (float*)smem + wave * FM * 1024,
                      part ? part + (int64_t)blockIdx.y * a.M * N4 : nullptr, N4, lane);
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
    float v[4] = {s[0], s[1], s[2], s[3]};
    const uint2 off = e.drop.on ? drop_offset(e.drop) : make_uint2(0, 0);
    float b[4];
    bias_cols<T, 4>(e, n, b);
    epilogue_cols<T, 4>(e, off, m, n, v, b);
}

// operands whose rows the 16-byte loads cannot address (odd length, stride or base), up to two a launch: copied to
// rows of `cp` elements (a multiple of 8), zero padded; 8 elements a thread
struct RepackArgs {
    const u16* src;
    int64_t ld;
    int rows, cols;
    u16* dst;
    int cp;
};
__global__ __launch_bounds__(256) void repack_kernel(RepackArgs a, RepackArgs b, int blocks_a) {
    const bool first = (int)blockIdx.x < blocks_a;
    const RepackArgs& p = first ? a : b;
    const int cq = p.cp >> 3;
    const int64_t i = ((int64_t)blockIdx.x - (first ? 0 : blocks_a)) * 256 + threadIdx.x;
    const int64_t r = i / cq;
    const int c = (int)(i - r * cq) * 8;
    if (r >= p.rows) return;
    const u16* s = p.src + r * p.ld + c;
    u16 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < p.cols ? s[j] : (u16)0;
    uint4 w;
    __builtin_memcpy(&w, v, 16);
    *(uint4*)(p.dst + r * p.cp + c) = w;
}

bool loadable(const u16* p, int64_t ld, int len) { return ((size_t)p & 15) == 0 && ld % 8 == 0 && len % 8 == 0; }

typedef MatmulPart Part;

int tiles(int M, int N, int t) { return ((M + t - 1) / t) * ((N + t - 1) / t); }

// Estimated time of a launch: rounds of workgroups times (k-tiles of a slice x time of one + start and epilogue),
// and the join of a split. Fitted to products measured at every (tile, slices) on 12 shapes, M x K x N: e.g.
// 12608 x 4096 x 1024 64 / 128 / 256-wide tiles 170 / 107 / 95 us, 256 in two slices 144; 4928 x 512 x 2048 27 / 23 / 22 us;
// 4096 x 36928 x 1024 256 in 1 / 2 / 4 / 8 slices 864 / 452 / 272 / 297 us; 2048 x 4928 x 512 64 in 1 / 2 / 4 slices 27.5 / 24.0 / 26.9
// us; 1237 x 768 x 440 7 / 13 / 26 us.
double cost_us(int tile, int nt, int S, int ks, double out) {
    // one 256-wide workgroup a CU; two of the smaller ones, each slower beside the other than alone
    static const double alone[3] = {0.30, 0.83, 1.42}, beside[3] = {0.43, 1.13, 1.42}, fixed[3] = {2.5, 4.0, 8.5};
    const int64_t wgs = (int64_t)nt * S, slots = tile == 2 ? 256 : 512, full = wgs / slots, rest = wgs % slots;
    double t = full * (ks * beside[tile] + fixed[tile]);
    if (rest) t += ks * (rest <= 256 ? alone[tile] : beside[tile]) + fixed[tile];
    if (S > 1) t += 5.0 + (S * 8.0 + 2.0) * out / 4.5e6;
    return t;
}

Part best_part(int M, int N, int nk, int N4) {
    Part b{M, 0, 1, nk > 0 ? nk : 1, 1e30};
    for (int t = 0; t < 3; ++t) {
        const int nt = tiles(M, N, 64 << t);
        for (int S = 1; S <= 64 && (S == 1 || (nk >= 2 * S && (int64_t)nt * S <= 1024)); ++S) {
            const int ks = nk > 0 ? (nk + S - 1) / S : 1;
            const double c = cost_us(t, nt, S, ks, (double)M * N4);
            if (c < b.us) b = Part{M, t, nk > 0 ? (nk + ks - 1) / ks : 1, ks, c};
        }
    }
    return b;
}

template <typename T, bool AK, bool BK>
void launch_tile(hipStream_t s, const Matmul& a, const Part& p, int N4, float* part) {
    const dim3 grid(tiles(a.M, a.N, 64 << p.tile), p.S);
    if (p.tile == 2) matmul256_kernel<T, AK, BK><<<grid, 512, 0, s>>>(a, part, N4, p.kslice);
    else if (p.tile == 1) matmul_kernel<T, AK, BK, 2, 2, 4, 2><<<grid, 256, 0, s>>>(a, part, N4, p.kslice);
    else matmul_kernel<T, AK, BK, 4, 1, 1, 3><<<grid, 256, 0, s>>>(a, part, N4, p.kslice);
}

template <typename T>
void launch_part(hipStream_t s, const Matmul& a, const Part& p, int N4, float* part) {
    if (a.a_k && a.b_k) launch_tile<T, true, true>(s, a, p, N4, part);
    else if (a.a_k) launch_tile<T, true, false>(s, a, p, N4, part);
    else if (a.b_k) launch_tile<T, false, true>(s, a, p, N4, part);
    else launch_tile<T, false, false>(s, a, p, N4, part);
    if (p.S > 1) {
        const int64_t n = (int64_t)a.M * (N4 >> 2);
        matmul_join_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(a.e, part, N4, p.S);
    }
}

// rows [m0, m0 + rows) of the product
Matmul rows_of(const Matmul& a, int m0, int rows) {
    Matmul r = a;
    r.M = rows;
    r.A = a.A + (int64_t)m0 * (a.a_k ? a.lda : 1);
    Epilogue& e = r.e;
    e.M = rows;
    e.m_base = a.e.m_base + m0;
    e.y = (u16*)a.e.y + (int64_t)m0 * a.e.ldy;
    if (e.res) e.res = (const u16*)a.e.res + (int64_t)m0 * a.e.ldr;
    if (e.slope) e.slope = a.e.slope + (int64_t)m0 * a.e.N;
    if (e.lu) e.lu = a.e.lu + (int64_t)m0 * a.e.R;
    return r;
}

// rows whose length or stride or base the 16-byte loads cannot take, as rows of the length rounded up to 8. A single row may
// be longer than a stride that the tiles' 32-bit offsets hold (a multiple of 2^26 elements wraps to row 0): it gets one that
// puts the k rows after it outside a tile's resource.
RepackArgs repack_of(const u16*& p, int64_t& ld, int rows, int len, void* dst) {
    const int cp = (len + 7) / 8 * 8;
    const RepackArgs r{p, ld, rows, len, (u16*)dst, cp};
    p = (const u16*)dst;
    ld = rows > 1 ? cp : 4096;
    return r;
}

}  // namespace

MatmulPlan matmul_plan(const Matmul& a, const MatmulPart* chosen, int parts) {
    MatmulPlan p{};
    if (a.M <= 0 || a.N <= 0) return p;
    const int al = a.a_k ? a.K : a.M, ar = a.a_k ? a.M : a.K, bl = a.b_k ? a.K : a.N, br = a.b_k ? a.N : a.K;
    auto up = [](int64_t v, int64_t q) { return (v + q - 1) / q * q; };
    if (a.K > 0 && !loadable(a.A, a.lda, al)) p.a_bytes = (size_t)up((int64_t)ar * up(al, 8) * 2, 256);
    if (a.K > 0 && !loadable(a.B, a.ldb, bl)) p.b_bytes = (size_t)up((int64_t)br * up(bl, 8) * 2, 256);
    const int nk = (a.K + 63) / 64, nN = (a.N + 255) / 256, nM = (a.M + 255) / 256;
    p.N4 = (int)up(a.N, 4);
    p.parts = chosen ? parts : 1;
    for (int i = 0; i < parts && chosen; ++i) {
        const int ks = nk > 0 ? (nk + chosen[i].S - 1) / chosen[i].S : 1;
        p.part[i] = Part{chosen[i].rows, chosen[i].tile, nk > 0 ? (nk + ks - 1) / ks : 1, ks, 0};
    }
    if (!chosen) p.part[0] = best_part(a.M, a.N, nk, p.N4);
    // whole rounds of 256-wide tiles as one launch and the remaining rows as another with tiles of its own, where
    // that is estimated faster (the launch itself 3 us): 36928 x 4096 x 1024 is 580 tiles, 2.3 rounds in the time of 3
    const int round_rows = nN <= 256 ? 256 / nN : 0;  // tile rows of one round
    if (!chosen && round_rows && (256 % nN) * 16 <= 256 && nM > round_rows) {
        const int rows = nM / round_rows * round_rows * 256;
        if (rows < a.M) {
            const Part main{rows, 2, 1, nk > 0 ? nk : 1, cost_us(2, tiles(rows, a.N, 256), 1, nk, 0)};
            const Part rest = best_part(a.M - rows, a.N, nk, p.N4);
            if (main.us + rest.us + 3.0 < p.part[0].us) {
                p.parts = 2;
                p.part[0] = main;
                p.part[1] = rest;
            }
        }
    }
    for (int i = 0; i < p.parts; ++i) {
        const Part& q = p.part[i];
        const size_t bytes = q.S > 1 ? (size_t)q.S * q.rows * p.N4 * 4 : 0;
        if (bytes > p.part_bytes) p.part_bytes = bytes;
    }
    return p;
}

size_t matmul_workspace(const MatmulPlan& p) { return p.a_bytes + p.b_bytes + p.part_bytes; }

int launch_matmul(hipStream_t s, int dtype, const Matmul& a0, const MatmulPlan& p, void* ws, size_t ws_bytes) {
    if (a0.M <= 0 || a0.N <= 0) return 0;
    Matmul a = a0;
    if (p.a_bytes + p.b_bytes + p.part_bytes > ws_bytes) return -1;
    unsigned char* w = (unsigned char*)ws;
    if (p.a_bytes || p.b_bytes) {
        RepackArgs r[2]{};
        if (p.a_bytes) r[0] = repack_of(a.A, a.lda, a.a_k ? a.M : a.K, a.a_k ? a.K : a.M, w);
        if (p.b_bytes) r[1] = repack_of(a.B, a.ldb, a.b_k ? a.N : a.K, a.b_k ? a.K : a.N, w + p.a_bytes);
        const int64_t na = ((int64_t)r[0].rows * (r[0].cp / 8) + 255) / 256, nb = ((int64_t)r[1].rows * (r[1].cp / 8) + 255) / 256;
        repack_kernel<<<(unsigned)(na + nb), 256, 0, s>>>(r[0], r[1], (int)na);
    }
    float* part = (float*)(w + p.a_bytes + p.b_bytes);
    a.e.vec = ((size_t)a.e.y & 15) == 0 && a.e.ldy % 8 == 0 &&
              (!a.e.res || (((size_t)a.e.res & 15) == 0 && a.e.ldr % 8 == 0)) &&
              (!a.e.slope || (((size_t)a.e.slope & 15) == 0 && a.N % 8 == 0));
    // y past the L2s' and most of the Infinity Cache's size is not kept there for a later reader anyway: stored past
    // them it leaves the operand panels (36928 x 1024 x 4096 forward 301 -> 293 us)
    a.e.nt = (int64_t)a.M * a.N * 2 >= (int64_t)64 << 20;
    int m0 = 0;
    for (int i = 0; i < p.parts; ++i) {
        const Part& q = p.part[i];
        const Matmul r = rows_of(a, m0, q.rows);
        if (dtype == 1) launch_part<BF16>(s, r, q, p.N4, q.S > 1 ? part : nullptr);
        else launch_part<F16>(s, r, q, p.N4, q.S > 1 ? part : nullptr);
        m0 += q.rows;
    }
    return 0;
}

}  // namespace clipvit
