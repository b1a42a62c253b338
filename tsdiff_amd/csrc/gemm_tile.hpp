// gemm_tile.hpp -- C[m][n] = sum_k M(m, k) N(n, k) on operand tiles in LDS (block_tile.hpp), for the kernels of the gated
// linear layer.  An operand is a matrix whose rows are the output's (k contiguous: RowOperand) or whose rows are the
// contraction's (ColOperand); its tiles are copied as they lie and read along or across.
// The instruction's first operand is the n side: a lane then holds four neighbouring n of one m, which is how a
// row-major result is stored and how the epilogues read what belongs to it.
#pragma once
#include "block_tile.hpp"

namespace tsd {
namespace blk {

// Waves over one side of the output tile: two, or four of 64 rows or columns each over a side of 256
constexpr int gemm_waves(int n) { return n > 128 ? n / 64 : 2; }
constexpr int gemm_wg(int bm, int bn) { return 64 * gemm_waves(bm) * gemm_waves(bn); }
constexpr int GEMM_K = 32;    // steps of the contraction a tile

// Tile row r is matrix row first + r (r < split) or, TWO, row first2 + r - split of a second matrix; k along the rows
template <class T, bool TWO> struct RowOperand {
    static constexpr bool ACROSS = false, BASES = TWO;
    const T *p, *p2;
    int64_t ld;
    int rows, kmax, first, split, first2;
    int vw;  // load_raw's
    template <int N> using TileOf = Tile<T, N, GEMM_K / 8>;
    __device__ __forceinline__ void load(Raw<T>& raw, int r, int c, int k) const {
        const bool two = TWO && r >= split;
        const int row = two ? first2 + r - split : first + r, kk = k + c * 8, n = row < rows ? kmax - kk : 0;
        load_raw(raw, (two ? p2 : p) + (n > 0 ? (int64_t)row * ld + kk : 0), n < 0 ? 0 : n > 8 ? 8 : n, vw);
    }
    // bytes from the tile's first matrix (both matrices' tiles fit 2 GiB: the caller has seen to it)
    __device__ __forceinline__ uint32_t offset(int r, int c) const {
        const bool two = TWO && r >= split;
        return (two ? first2 + r - split : first + r) < rows ? (uint32_t)(((two ? r - split : r) * ld + c * 8) * (int)sizeof(T))
                                                              : DMA_NOWHERE;
    }
    // the first value of the tile at k that a load of rows `row` .. reads from, and how many k's its matrix has from there on
    __device__ __forceinline__ const T* base(int row, int k, int& left) const {
        left = kmax - k;
        return (TWO && row >= split ? p2 + (int64_t)first2 * ld : p + (int64_t)first * ld) + k;
    }
    // from the tile at k to the result they follow each other in memory and lie inside of one matrix
    __device__ __forceinline__ int whole_until(int) const { return kmax; }
    __device__ __forceinline__ int64_t step() const { return GEMM_K; }
    // is k + r (or chunk c of row r at k) there
    __device__ __forceinline__ static bool has(int, int c, int left) { return c * 8 < left; }
};
// Rows of the contraction, from `ksplit` on those of a second matrix (kmax rows each), from `wrap` on all of them once more
// (wrap: a multiple of 16); columns first ..
template <class T> struct ColOperand {
    static constexpr bool ACROSS = true, BASES = false;
    const T *p, *p2;
    int64_t ld;
    int cols, kmax, first, ksplit, wrap;
    int vw;  // load_raw's
    template <int N> using TileOf = Tile<T, GEMM_K, N / 8>;
    __device__ __forceinline__ void load(Raw<T>& raw, int r, int c, int k) const {
        const int kr = k + r - (k + r >= wrap ? wrap : 0);
        const bool two = kr >= ksplit;
        const int kk = kr - (two ? ksplit : 0), col = first + c * 8, n = kk < kmax ? cols - col : 0;
        load_raw(raw, (two ? p2 : p) + (n > 0 ? (int64_t)kk * ld + col : 0), n < 0 ? 0 : n > 8 ? 8 : n, vw);
    }
    __device__ __forceinline__ uint32_t offset(int r, int c) const {
        return first + c * 8 < cols ? (uint32_t)((r * ld + c * 8) * (int)sizeof(T)) : DMA_NOWHERE;
    }
    // ksplit and wrap are multiples of 8, as few rows as a wave's load may hold: it lies on one side
    __device__ __forceinline__ const T* base(int row, int k, int& left) const {
        const int kw = k - (k + row >= wrap ? wrap : 0);
        const bool two = kw + row >= ksplit;
        const int kk = kw - (two ? ksplit : 0);
        left = kmax - kk;
        return (two ? p2 : p) + (int64_t)kk * ld + first;
    }
    __device__ __forceinline__ int whole_until(int k) const {
        const bool again = k >= wrap;
        const int kw = again ? k - wrap : k, kk = kw < ksplit ? kw : kw - ksplit;
        const int edge = kw < ksplit ? ksplit - kw : again ? 1 << 30 : wrap - k, rows = kmax - kk;
        return k + (edge < rows ? edge : rows);
    }
    __device__ __forceinline__ int64_t step() const { return GEMM_K * ld; }
    __device__ __forceinline__ static bool has(int r, int, int left) { return r < left; }
};

// Where the chunks of a tile of N output rows (or columns) lie, for 32-bit offsets from a base that is the same for a wave;
// places outside of the matrix are NOWHERE.  LDS places for loads straight to LDS (PERMUTED): a wave's 64 lanes fill 64
// neighbouring places, so the lane of place p of row r fetches chunk p ^ swizzle(r).
template <class T, int N, int WG, class Op, bool PERMUTED> struct Places {
    using Lds = typename Op::template TileOf<N>;
    static constexpr int UNITS = Lds::ROWS * Lds::C, U = UNITS < WG ? 1 : UNITS / WG;
    // (a tile smaller than the workgroup is loaded by several waves alike: every wave counts the same loads)
    static_assert(UNITS % WG == 0 || (WG % UNITS == 0 && UNITS % 64 == 0), "whole loads");
    static constexpr int B = Op::BASES ? U : 1;  // bases of a wave's loads
    uint32_t off[U];
    int row[U], chunk[U];
    // The tiles of a whole part of the operand (most of them) follow each other by the same distance, with no bounds to look
    // at: `left` of them are still to come.  (Not for f32, where a second way to the registers costs more than it saves:
    // forward of 3600 x 256 -> 2 x 1024 34 us against 31.)
    i32x4 at[B];
    int left;
    __device__ __forceinline__ void init(const Op& op) {
        left = 0;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = (threadIdx.x + i * WG) % UNITS;
            row[i] = u / Lds::C;
            chunk[i] = PERMUTED ? (u % Lds::C) ^ Lds::swizzle(row[i]) : u % Lds::C;
            off[i] = op.offset(row[i], chunk[i]);
        }
    }
    // The tile at k; the one before it was at k - GEMM_K.  One matrix a load: the 64 places of a wave lie on one side of the
    // operand's split.
    template <class F> __device__ __forceinline__ void each(const Op& op, int k, F f) {
        if constexpr (PERMUTED) {
            if (--left >= 0) {
#pragma unroll
                for (int b = 0; b < B; ++b) dma_advance(at[b], op.step() * (int64_t)sizeof(T));
#pragma unroll
                for (int i = 0; i < U; ++i) f(i, at[Op::BASES ? i : 0], off[i]);
                return;
            }
            left = (op.whole_until(k) - k) / GEMM_K - 1;
            left = left < 0 ? 0 : left;
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            int rest;
            const i32x4 buf = dma_buffer(op.base(__builtin_amdgcn_readfirstlane(row[i]), k, rest));
            if (i < B) at[i] = buf;  // (of a tile in one matrix: all are the same)
            f(i, buf, Op::has(row[i], chunk[i], rest) ? off[i] : DMA_NOWHERE);
        }
    }
};

// A tile by way of registers, DEPTH tiles under way.  FAST (f32): branch-free loads with the bounds in the buffer.
template <class T, int N, int WG, class Op, int DEPTH, bool FAST> struct RegStage {
    using Lds = typename Op::template TileOf<N>;
    static constexpr int UNITS = Lds::ROWS * Lds::C, U = (UNITS + WG - 1) / WG;
    Raw<T> raw[DEPTH][U];
    Places<T, N, WG, Op, false> places;
    __device__ __forceinline__ void init(const Op& op) {
        if constexpr (FAST) places.init(op);
    }
    __device__ __forceinline__ void load(int d, const Op& op, int k) {
        if constexpr (FAST) {
            places.each(op, k, [&](int i, i32x4 buf, uint32_t off) {
                raw[d][i].a = buffer_load(buf, off);
                raw[d][i].b = buffer_load(buf, off + 16);
            });
        } else {
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int u = threadIdx.x + i * WG;
                if (UNITS % WG == 0 || u < UNITS) op.load(raw[d][i], u / Lds::C, u % Lds::C, k);
            }
        }
    }
    __device__ __forceinline__ void store(int d, char* lds) const {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = threadIdx.x + i * WG;
            if (UNITS % WG == 0 || u < UNITS) Lds::put(lds, u / Lds::C, u % Lds::C, raw_chunk(raw[d][i]));
        }
    }
};
// Straight to LDS
template <class T, int N, int WG, class Op> struct DmaStage {
    using At = Places<T, N, WG, Op, true>;
    static constexpr int U = At::U;
    At places;
    int at[U];  // LDS bytes of a wave's load
    __device__ __forceinline__ void init(const Op& op) {
        places.init(op);
#pragma unroll
        for (int i = 0; i < U; ++i)
            at[i] = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / 64 * 64 + i * WG) % At::UNITS * 16);
    }
    __device__ __forceinline__ void issue(const Op& op, int k, uint32_t lds) {
        places.each(op, k, [&](int i, i32x4 buf, uint32_t off) { dma_load(buf, off, lds + at[i]); });
    }
};

template <class T, int BM, int BN, class NS, class MS> struct GemmTile {
    using NT = typename NS::template TileOf<BN>;
    using MT = typename MS::template TileOf<BM>;
    static constexpr int BUF = NT::BYTES + MT::BYTES;
    static constexpr int WG = gemm_wg(BM, BN), MI = BM / gemm_waves(BM) / 16, NJ = BN / gemm_waves(BN) / 16;  // subtiles of a wave
    using Acc = f32x4[NJ][MI];

    template <class NRow>
    __device__ __forceinline__ static void products(const char* nb, int mrow, NRow nrow, Acc& acc) {
        const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
        const char* mb = nb + NT::BYTES;
        Chunk<T> mf[MI];
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            if constexpr (MS::ACROSS) mf[i] = MT::get_across(mb, 0, mrow / 16 + i);
            else mf[i] = MT::get(mb, mrow + i * 16 + r, c);
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            Chunk<T> nf;
            if constexpr (NS::ACROSS) nf = NT::get_across(nb, 0, nrow(j) / 16);
            else nf = NT::get(nb, nrow(j) + r, c);
#pragma unroll
            for (int i = 0; i < MI; ++i) acc[j][i] = mma(nf, mf[i], acc[j][i]);
        }
    }
    __device__ __forceinline__ static void clear(Acc& acc) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int i = 0; i < MI; ++i) acc[j][i] = f32x4{0, 0, 0, 0};
    }
    // One output tile: acc[jn][im] of the calling wave, n rows nrow(jn) and m rows mrow + im * 16 of the tile; ends behind a
    // barrier.  The next DEPTH tiles' values are on their way into registers.  BUFS 2: two LDS buffers, one barrier a tile;
    // 1: one buffer, two barriers, and twice the workgroups on a CU where LDS is what limits them.
    template <int DEPTH, int BUFS, bool FAST, class NRow>
    __device__ __forceinline__ static void by_registers(char* lds, const NS& ns, const MS& ms, int kbegin, int kend, int mrow,
                                                        NRow nrow, Acc& acc) {
        RegStage<T, BN, WG, NS, DEPTH, FAST> nst;
        RegStage<T, BM, WG, MS, DEPTH, FAST> mst;
        nst.init(ns);
        mst.init(ms);
        clear(acc);
#pragma unroll
        for (int d = 0; d < DEPTH; ++d)
            if (kbegin + d * GEMM_K < kend) {
                nst.load(d, ns, kbegin + d * GEMM_K);
                mst.load(d, ms, kbegin + d * GEMM_K);
            }
        nst.store(0, lds);
        mst.store(0, lds + NT::BYTES);
        __syncthreads();
        int cur = 0;
        for (int k0 = kbegin; k0 < kend; k0 += DEPTH * GEMM_K) {
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) {
                const int k = k0 + d * GEMM_K;
                if (k >= kend) break;
                if (k + DEPTH * GEMM_K < kend) {
                    nst.load(d, ns, k + DEPTH * GEMM_K);
                    mst.load(d, ms, k + DEPTH * GEMM_K);
                }
                products(lds + cur * BUF, mrow, nrow, acc);
                if constexpr (BUFS == 2) cur ^= 1;
                else __syncthreads();
                if (k + GEMM_K < kend) {
                    nst.store((d + 1) % DEPTH, lds + cur * BUF);
                    mst.store((d + 1) % DEPTH, lds + cur * BUF + NT::BYTES);
                }
                __syncthreads();
            }
        }
    }
    // The same with loads straight to LDS: STAGES buffers, STAGES - 1 tiles under way, one barrier a tile.
    template <int STAGES, class NRow>
    __device__ __forceinline__ static void by_dma(char* lds, const NS& ns, const MS& ms, int kbegin, int kend, int mrow, NRow nrow,
                                                  Acc& acc) {
        DmaStage<T, BN, WG, NS> nst;
        DmaStage<T, BM, WG, MS> mst;
        constexpr int LOADS = DmaStage<T, BN, WG, NS>::U + DmaStage<T, BM, WG, MS>::U;
        nst.init(ns);
        mst.init(ms);
        clear(acc);
        const uint32_t base = lds_offset(lds);
#pragma unroll
        for (int d = 0; d < STAGES - 1; ++d) {  // (tiles past the end load zeros: the count of loads stays the same)
            nst.issue(ns, kbegin + d * GEMM_K, base + d * BUF);
            mst.issue(ms, kbegin + d * GEMM_K, base + d * BUF + NT::BYTES);
        }
        int buf = 0, ahead = STAGES - 1;
        for (int k = kbegin; k < kend; k += GEMM_K) {
            dma_wait<(STAGES - 2) * LOADS>();
            lds_barrier();
            nst.issue(ns, k + (STAGES - 1) * GEMM_K, base + ahead * BUF);
            mst.issue(ms, k + (STAGES - 1) * GEMM_K, base + ahead * BUF + NT::BYTES);
            products(lds + buf * BUF, mrow, nrow, acc);
            buf = buf + 1 == STAGES ? 0 : buf + 1;
            ahead = ahead + 1 == STAGES ? 0 : ahead + 1;
        }
        dma_wait<0>();  // nothing may land in LDS that is used otherwise, or belongs to the next workgroup
        lds_barrier();
    }
};

// Workgroup b of a grid over (long side) x (short side) tiles: consecutive workgroups go to the eight XCDs in turn, so the
// tiles of one long-side row are given to one XCD, whose L2 then holds that row's operand once.
struct TileAt {
    int lo, sh;
};
__device__ __forceinline__ TileAt tile_at(int b, int nshort) {
    const int xcd = b & 7, l = b >> 3;
    return {xcd + 8 * (l / nshort), l % nshort};
}
inline int tile_grid(int nlong, int nshort) { return (nlong + 7) / 8 * 8 * nshort; }

}  // namespace blk
}  // namespace tsd
