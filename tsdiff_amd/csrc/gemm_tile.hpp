// gemm_tile.hpp -- C[m][n] = sum_k M(m, k) N(n, k) on operand tiles in LDS (block_tile.hpp), for the kernels of the gated
// linear layer.  Either operand is read as it lies (k contiguous) or turned (the tile's rows contiguous) on its way to LDS.
// The instruction's first operand is the n side: a lane then holds four neighbouring n of one m, which is how a
// row-major result is stored and how the epilogues read what belongs to it.
#pragma once
#include "block_tile.hpp"

namespace tsd {
namespace blk {

constexpr int GEMM_WG = 256;  // four waves, two by two over the output tile
constexpr int GEMM_K = 32;    // steps of the contraction a tile

// rows x kmax values, k contiguous; rows from `split` on are rows of a second matrix
template <class T> struct RowSource {
    const T *p, *p2;
    int64_t ld;
    int rows, kmax, first, split, first2;  // tile row r < split: row first + r of p; else row first2 + r - split of p2
    bool vec;
    __device__ __forceinline__ void load(Raw<T>& raw, int r, int k) const {
        const bool two = r >= split;
        const int row = two ? first2 + r - split : first + r;
        const int n = row < rows ? kmax - k : 0;
        load_raw(raw, (two ? p2 : p) + (n > 0 ? (int64_t)row * ld + k : 0), n < 0 ? 0 : n > 8 ? 8 : n, vec);
    }
};
// kmax x cols values, columns contiguous; k from `ksplit` on are rows k - ksplit of a second matrix
template <class T> struct ColSource {
    const T *p, *p2;
    int64_t ld;
    int cols, kmax, first, ksplit;  // kmax: rows of either matrix
    bool vec;                       // two columns a load: even ld and first, 4-byte aligned
    __device__ __forceinline__ void load(ColRaw<T>& raw, int c, int k) const {
        const bool two = k >= ksplit;
        const int kk = two ? k - ksplit : k, col = first + c;
        const T* q = (two ? p2 : p) + col;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            raw.w[j] = 0;
            if (col < cols && kk + j < kmax) col_load(raw.w[j], q + (int64_t)(kk + j) * ld, cols - col, vec && col + 1 < cols);
        }
    }
};

template <class T, int ROWS> struct RowStage {
    static constexpr int UNITS = ROWS * 4, U = (UNITS + GEMM_WG - 1) / GEMM_WG;
    using Lds = Tile<T, ROWS, 4>;
    Raw<T> raw[U];
    __device__ __forceinline__ void load(const RowSource<T>& s, int k) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = threadIdx.x + i * GEMM_WG;
            if (UNITS % GEMM_WG == 0 || u < UNITS) s.load(raw[i], u >> 2, k + (u & 3) * 8);
        }
    }
    __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = threadIdx.x + i * GEMM_WG;
            if (UNITS % GEMM_WG == 0 || u < UNITS) Lds::put(lds, u >> 2, u & 3, raw_chunk(raw[i]));
        }
    }
};
template <class T, int ROWS> struct ColStage {
    static constexpr int W = ColRaw<T>::W, COLS = ROWS / W, UNITS = COLS * 4, U = (UNITS + GEMM_WG - 1) / GEMM_WG;
    using Lds = Tile<T, ROWS, 4>;
    ColRaw<T> raw[U];
    __device__ __forceinline__ void load(const ColSource<T>& s, int k) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = threadIdx.x + i * GEMM_WG;
            if (UNITS % GEMM_WG == 0 || u < UNITS) s.load(raw[i], (u % COLS) * W, k + (u / COLS) * 8);
        }
    }
    __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = threadIdx.x + i * GEMM_WG;
            if (UNITS % GEMM_WG == 0 || u < UNITS)
#pragma unroll
                for (int c = 0; c < W; ++c) Lds::put(lds, (u % COLS) * W + c, u / COLS, col_chunk<T>(raw[i], c));
        }
    }
};
template <class T, int ROWS, class Source> struct StageOf;
template <class T, int ROWS> struct StageOf<T, ROWS, RowSource<T>> { using type = RowStage<T, ROWS>; };
template <class T, int ROWS> struct StageOf<T, ROWS, ColSource<T>> { using type = ColStage<T, ROWS>; };

template <class T, int BM, int BN> constexpr int gemm_lds() { return 2 * (Tile<T, BM, 4>::BYTES + Tile<T, BN, 4>::BYTES); }

// One output tile: acc[jn][im] of the calling wave, n rows nrow(jn) and m rows mrow + im * 16 of the tile.
// The next tile's values are on their way into registers while this tile's products run; two LDS buffers, one barrier a tile.
template <class T, int BM, int BN, class NS, class MS, class NRow>
__device__ __forceinline__ void gemm_tile(char* lds, const NS& ns, const MS& ms, int kbegin, int kend, int mrow, NRow nrow,
                                          f32x4 (&acc)[BN / 32][BM / 32]) {
    using NT = Tile<T, BN, 4>;
    using MT = Tile<T, BM, 4>;
    constexpr int BUF = NT::BYTES + MT::BYTES;
    const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
    typename StageOf<T, BN, NS>::type nst;
    typename StageOf<T, BM, MS>::type mst;
#pragma unroll
    for (int j = 0; j < BN / 32; ++j)
#pragma unroll
        for (int i = 0; i < BM / 32; ++i) acc[j][i] = f32x4{0, 0, 0, 0};
    if (kbegin >= kend) return;
    nst.load(ns, kbegin);
    mst.load(ms, kbegin);
    nst.store(lds);
    mst.store(lds + NT::BYTES);
    __syncthreads();
    int cur = 0;
    for (int k = kbegin; k < kend; k += GEMM_K) {
        const bool more = k + GEMM_K < kend;
        if (more) {
            nst.load(ns, k + GEMM_K);
            mst.load(ms, k + GEMM_K);
        }
        const char* nb = lds + cur * BUF;
        const char* mb = nb + NT::BYTES;
        Chunk<T> mf[BM / 32];
#pragma unroll
        for (int i = 0; i < BM / 32; ++i) mf[i] = MT::get(mb, mrow + i * 16 + r, c);
#pragma unroll
        for (int j = 0; j < BN / 32; ++j) {
            const Chunk<T> nf = NT::get(nb, nrow(j) + r, c);
#pragma unroll
            for (int i = 0; i < BM / 32; ++i) acc[j][i] = mma(nf, mf[i], acc[j][i]);
        }
        if (more) {
            char* next = lds + (cur ^ 1) * BUF;
            nst.store(next);
            mst.store(next + NT::BYTES);
        }
        __syncthreads();
        cur ^= 1;
    }
}

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
