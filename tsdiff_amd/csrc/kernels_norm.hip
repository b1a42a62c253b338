// kernels_norm.hip -- layer norm over the last dimension, forward and backward (f32, bf16, f16; statistics in fp32).
//
//   y = xh w + b,  xh = (x - m) r,  m = mean x,  r = (mean (x - m)^2 + eps)^(-1/2)
//   g = dy w:  dx = r (g - mean g - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// HBM-bound: x in, y out (forward), x and dy in, dx out (backward).  A group of LANES lanes holds a whole row in
// registers (E values a lane, VE neighbouring ones a load), so the mean and the centred squares are two passes over
// registers and one over memory.  The backward's groups go over many rows each and keep their columns' share of dw
// and db in registers; a workgroup adds its groups' shares in LDS and writes one row of partial sums, and a second
// launch adds those in a fixed order (no atomics: the same bits on every run).
//
// Widths that are no multiple of a 16-byte load: a group's rows are a multiple of 8 apart, so all of them start at the same
// place between two 16-byte borders.  The group's columns are shifted by that much once, and its loads and stores are
// 16 bytes on their borders again, but for the pieces at a row's two ends, which go value by value.
//
// Measured (GPU time): bf16, 262144 x 256: forward 50 us (5.3 TB/s), backward 82 us (4.9 TB/s), sums of the parts 5.5 us.
// f16, 4099 x 1030 (rows between borders, out of L2): 14, 25 and 4 us.  f32, 3600 x 256: 4, 6 and 4 us; 17 x 256: 3 us.
#include <initializer_list>

#include "block_tile.hpp"

namespace tsd {
namespace blk {

constexpr int NORM_WG = 256;
constexpr int NORM_MAX_DIM = 8192;
constexpr int NORM_MAX_PARTS = 1024;

template <int LANES> __device__ __forceinline__ float norm_sum(float v, float* red) {
#pragma unroll
    for (int m = 1; m < (LANES < 64 ? LANES : 64); m *= 2) v += __shfl_xor(v, m, 64);
    if constexpr (LANES > 64) {
        __syncthreads();  // the last sum's readers are done
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int w = 1; w < LANES / 64; ++w) v += red[w];
    }
    return v;
}

template <int N> struct alignas(N) Bytes {
    char b[N];
};

// VE neighbouring values, one load of VE * sizeof(T) bytes
template <class T, int VE> __device__ __forceinline__ void norm_load(float* x, const T* __restrict__ p) {
    const Bytes<VE * sizeof(T)> raw = *reinterpret_cast<const Bytes<VE * sizeof(T)>*>(p);
    T t[VE];
    __builtin_memcpy(t, &raw, sizeof(raw));
#pragma unroll
    for (int j = 0; j < VE; ++j) x[j] = to_f(t[j]);
}
template <class T, int VE> __device__ __forceinline__ void norm_store(T* __restrict__ p, const float* x) {
    T t[VE];
#pragma unroll
    for (int j = 0; j < VE; ++j) t[j] = (T)x[j];
    Bytes<VE * sizeof(T)> raw;
    __builtin_memcpy(&raw, t, sizeof(raw));
    *reinterpret_cast<Bytes<VE * sizeof(T)>*>(p) = raw;
}

// Values v * VE + j of a lane are columns (v * LANES + lane) * VE - s + j; places without a column hold `fill`.
// SHIFT false: s is 0 and dim a multiple of VE.
template <class T, int VE, int LANES, int E, bool SHIFT> struct NormRow {
    static constexpr int NV = E / VE;
    __device__ __forceinline__ static int col(int v, int lane, int s) { return (v * LANES + lane) * VE - (SHIFT ? s : 0); }
    __device__ __forceinline__ static bool has(int e, int lane, int s, int dim) {
        if constexpr (!SHIFT) return col(e / VE, lane, s) < dim;
        return (unsigned)(col(e / VE, lane, s) + e % VE) < (unsigned)dim;
    }
    // a row as it lies in memory: on its way while the row before it is worked on
    using Raw = Bytes<VE * sizeof(T)>[NV];
    // (EDGE false: where a row starts or ends between two borders, the neighbouring row's values come along)
    template <bool EDGE> __device__ __forceinline__ static void fetch(Raw& raw, const T* p, int dim, int lane, int s) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = col(v, lane, s);
            if constexpr (EDGE) {
                T t[VE];
#pragma unroll
                for (int j = 0; j < VE; ++j) t[j] = (unsigned)(c + j) < (unsigned)dim ? p[c + j] : (T)0.f;
                __builtin_memcpy(&raw[v], t, sizeof(t));
            } else {
                raw[v] = {};
                if ((!SHIFT || c + VE > 0) && c < dim) raw[v] = *reinterpret_cast<const Bytes<VE * sizeof(T)>*>(p + c);
            }
        }
    }
    __device__ __forceinline__ static void values(float (&x)[E], const Raw& raw, int dim, int lane, int s) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            T t[VE];
            __builtin_memcpy(t, &raw[v], sizeof(t));
#pragma unroll
            for (int j = 0; j < VE; ++j) x[v * VE + j] = !SHIFT || has(v * VE + j, lane, s, dim) ? to_f(t[j]) : 0.f;
        }
    }
    // weight or bias (null: `fill`)
    __device__ __forceinline__ static void load_param(float (&x)[E], const T* p, int dim, int lane, int s, float fill) {
        if (p == nullptr) {
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = fill;
            return;
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = col(v, lane, s);
            if constexpr (SHIFT) {  // (every load at once: no column is looked at twice, and none waits for another)
#pragma unroll
                for (int j = 0; j < VE; ++j) x[v * VE + j] = to_f(p[c + j < 0 ? 0 : c + j < dim ? c + j : dim - 1]);
            } else if (c < dim) {
                norm_load<T, VE>(x + v * VE, p + c);
            } else {
#pragma unroll
                for (int j = 0; j < VE; ++j) x[v * VE + j] = fill;
            }
        }
    }
    __device__ __forceinline__ static void store(T* p, const float (&x)[E], int dim, int lane, int s) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = col(v, lane, s);
            if (SHIFT ? c >= 0 && c + VE <= dim : c < dim) {
                norm_store<T, VE>(p + c, x + v * VE);
            } else if constexpr (SHIFT) {
                if (c + VE > 0 && c < dim) store_piece(p + c, x + v * VE, c < 0 ? -c : 0, c + VE > dim ? dim - c : VE);
            }
        }
    }
    // values j0 .. j1 of a piece between two borders, in stores of 8, 4 and 2 bytes that lie on theirs
    __device__ __forceinline__ static void store_piece(T* p, const float* x, int j0, int j1) {
        T t[VE];
#pragma unroll
        for (int j = 0; j < VE; ++j) t[j] = (T)x[j];
        if (j0 > 0 && j1 < VE) {  // a row inside of one piece
#pragma unroll
            for (int j = 0; j < VE; ++j)
                if (j >= j0 && j < j1) p[j] = t[j];
            return;
        }
        u32x4 w;
        __builtin_memcpy(&w, t, 16);
        auto word = [&](int i) { return i == 0 ? w[0] : i == 1 ? w[1] : i == 2 ? w[2] : w[3]; };
        char* b = reinterpret_cast<char*>(p);
        const int size = (j1 - j0) * (int)sizeof(T);
        int at = j0 * (int)sizeof(T);
        if (j0 > 0) {  // its end: the small stores first
            if (size & 2) *reinterpret_cast<uint16_t*>(b + at) = (uint16_t)(word(at >> 2) >> 16);
            at += size & 2;
            if (size & 4) *reinterpret_cast<uint32_t*>(b + at) = word(at >> 2);
            if (size & 8) *reinterpret_cast<uint2*>(b + 8) = uint2{w[2], w[3]};
        } else {       // its beginning: the large stores first
            if (size & 8) *reinterpret_cast<uint2*>(b) = uint2{w[0], w[1]};
            at = size & 8;
            if (size & 4) *reinterpret_cast<uint32_t*>(b + at) = word(at >> 2);
            at += size & 4;
            if (size & 2) *reinterpret_cast<uint16_t*>(b + at) = (uint16_t)word(at >> 2);
        }
    }
};
// where row r of x starts between two borders of VE values
template <class T, int VE, bool SHIFT> __device__ __forceinline__ int norm_shift(const T* x, int64_t start) {
    return SHIFT ? (int)((reinterpret_cast<uintptr_t>(x + start) / sizeof(T)) % VE) : 0;
}

// A group's rows first, first + step, ..: each is fetched while the one before it is worked on.  With SHIFT the first and the
// last row of all go by themselves: what lies beside them need not be theirs to read.  work(r, next): next >= rows: none.
template <bool SHIFT, class Fetch, class Edge, class Work>
__device__ __forceinline__ void norm_rows(int64_t first, int64_t step, int64_t rows, Fetch fetch, Edge edge, Work work) {
    const int64_t none = (int64_t)1 << 62;
    if constexpr (SHIFT) {
        const int64_t last = rows - 1;
        if (first == 0 && first < last) {
            edge(first);
            work(first, none);
            first += step;
        }
        if (first < last) fetch(first);
        int64_t r = first;
        for (; r < last; r += step) work(r, r + step < last ? r + step : none);
        if (r == last) {
            edge(r);
            work(r, none);
        }
    } else {
        if (first < rows) fetch(first);
        for (int64_t r = first; r < rows; r += step) work(r, r + step);
    }
}

template <class T, int VE, int LANES, int E, bool SHIFT>
__global__ __launch_bounds__(NORM_WG) void norm_fwd_kernel(int rows, int dim, const T* __restrict__ x, int64_t ldx,
                                                           const T* __restrict__ w, const T* __restrict__ b, float eps,
                                                           T* __restrict__ y, float* __restrict__ mean,
                                                           float* __restrict__ rstd) {
    using R = NormRow<T, VE, LANES, E, SHIFT>;
    __shared__ float red[4];
    constexpr int GROUPS = NORM_WG / LANES;
    const int lane = threadIdx.x % LANES;
    const int64_t first = (int64_t)blockIdx.x * GROUPS + threadIdx.x / LANES;
    const int s = norm_shift<T, VE, SHIFT>(x, first * ldx);
    float wv[E], bv[E];
    R::load_param(wv, w, dim, lane, s, 1.f);
    R::load_param(bv, b, dim, lane, s, 0.f);
    const float inv = 1.f / (float)dim;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    typename R::Raw raw;
    auto work = [&](int64_t r, int64_t next) {
        float v[E];
        R::values(v, raw, dim, lane, s);
        if (next < rows) R::template fetch<false>(raw, x + next * ldx, dim, lane, s);
        float t = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) t += v[e];
        const float m = norm_sum<LANES>(t, red) * inv;
        float q = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            v[e] = R::has(e, lane, s, dim) ? v[e] - m : 0.f;
            q += v[e] * v[e];
        }
        const float rs = 1.f / sqrtf(norm_sum<LANES>(q, red) * inv + eps);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = v[e] * rs * wv[e] + bv[e];
        R::store(y + r * dim, v, dim, lane, s);
        if (mean != nullptr && lane == 0) {
            mean[r] = m;
            rstd[r] = rs;
        }
    };
    norm_rows<SHIFT>(first, step, rows, [&](int64_t r) { R::template fetch<false>(raw, x + r * ldx, dim, lane, s); },
                     [&](int64_t r) { R::template fetch<true>(raw, x + r * ldx, dim, lane, s); }, work);
}

template <class T, int VE, int LANES, int E, bool SHIFT>
__global__ __launch_bounds__(NORM_WG) void norm_bwd_kernel(int rows, int dim, const T* __restrict__ x, int64_t ldx,
                                                           const T* __restrict__ w, const T* __restrict__ dy,
                                                           int64_t lddy, const float* __restrict__ mean,
                                                           const float* __restrict__ rstd, T* __restrict__ dx,
                                                           float* __restrict__ part) {
    using R = NormRow<T, VE, LANES, E, SHIFT>;
    __shared__ float red[4];
    extern __shared__ float sums[];  // [2][W]
    constexpr int GROUPS = NORM_WG / LANES;
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const int64_t first = (int64_t)blockIdx.x * GROUPS + group;
    const int s = norm_shift<T, VE, SHIFT>(x, first * ldx);
    float wv[E], dw[E], db[E];
    R::load_param(wv, w, dim, lane, s, 1.f);
#pragma unroll
    for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.f;
    const float inv = 1.f / (float)dim;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    typename R::Raw rawx, rawg;
    float next_m = 0.f, next_r = 0.f;
    auto fetch = [&](int64_t r) {
        R::template fetch<false>(rawx, x + r * ldx, dim, lane, s);
        R::template fetch<false>(rawg, dy + r * lddy, dim, lane, s);
        next_m = mean[r];
        next_r = rstd[r];
    };
    auto edge = [&](int64_t r) {
        R::template fetch<true>(rawx, x + r * ldx, dim, lane, s);
        R::template fetch<true>(rawg, dy + r * lddy, dim, lane, s);
        next_m = mean[r];
        next_r = rstd[r];
    };
    auto work = [&](int64_t r, int64_t next) {
        float v[E], g[E];
        R::values(v, rawx, dim, lane, s);
        R::values(g, rawg, dim, lane, s);
        const float m = next_m, rs = next_r;
        if (next < rows) fetch(next);
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            v[e] = R::has(e, lane, s, dim) ? (v[e] - m) * rs : 0.f;
            dw[e] += g[e] * v[e];
            db[e] += g[e];
            g[e] *= wv[e];
            s0 += g[e];
            s1 += g[e] * v[e];
        }
        s0 = norm_sum<LANES>(s0, red) * inv;
        s1 = norm_sum<LANES>(s1, red) * inv;
        if (dx != nullptr) {
#pragma unroll
            for (int e = 0; e < E; ++e) g[e] = rs * (g[e] - s0 - v[e] * s1);
            R::store(dx + r * dim, g, dim, lane, s);
        }
    };
    norm_rows<SHIFT>(first, step, rows, fetch, edge, work);
    if (part == nullptr) return;
    constexpr int W = LANES * E;  // columns that a group has room for
    if constexpr (GROUPS > 1) {
        for (int k = 0; k < GROUPS; ++k) {  // one group after the other: the order is fixed
            if (group == k) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int c = R::col(e / VE, lane, s) + e % VE;
                    if (R::has(e, lane, s, dim)) {
                        sums[c] = k ? sums[c] + dw[e] : dw[e];
                        sums[W + c] = k ? sums[W + c] + db[e] : db[e];
                    }
                }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < 2 * W; c += NORM_WG) {
            const int col = c % W;
            if (col < dim) part[(size_t)blockIdx.x * 2 * dim + (c / W) * dim + col] = sums[c];
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int c = R::col(e / VE, lane, s) + e % VE;
            if (R::has(e, lane, s, dim)) {
                part[(size_t)blockIdx.x * 2 * dim + c] = dw[e];
                part[(size_t)blockIdx.x * 2 * dim + dim + c] = db[e];
            }
        }
    }
}

// out[c] = sum over `parts` rows of part[.][c], c < 2 dim: 16 columns a workgroup, 16 threads a column
template <class T>
__global__ __launch_bounds__(256) void norm_reduce_kernel(int parts, int dim, const float* __restrict__ part,
                                                          T* __restrict__ dw, T* __restrict__ db) {
    __shared__ float red[16][17];
    const int cx = threadIdx.x & 15, k = threadIdx.x >> 4, c = blockIdx.x * 16 + cx;
    float s = 0.f;
    if (c < 2 * dim) {
#pragma unroll 8
        for (int p = k; p < parts; p += 16) s += part[(size_t)p * 2 * dim + c];
    }
    red[k][cx] = s;
    __syncthreads();
    if (k == 0 && c < 2 * dim) {
        s = red[0][cx];
#pragma unroll
        for (int j = 1; j < 16; ++j) s += red[j][cx];
        if (c < dim) {
            if (dw != nullptr) dw[c] = (T)s;
        } else if (db != nullptr) {
            db[c - dim] = (T)s;
        }
    }
}

struct NormCall {
    int rows, dim;
    int64_t ldx, lddy;
    const void *x, *w, *b, *dy;
    float eps;
    void *y, *dx;
    float *mean, *rstd, *part;
    int parts;
    hipStream_t st;
};

// workgroups of the backward = rows of partial sums: about 4 a CU, >= 16 rows each; a multiple of 8 (see above)
static int norm_parts(int rows) {
    const int n = (int)(((int64_t)rows + 8 * 16 - 1) / (8 * 16)) * 8;
    return n < 8 ? 8 : n < NORM_MAX_PARTS ? n : NORM_MAX_PARTS;
}

template <class T, int VE, bool SHIFT, int LANES, int E> static int norm_launch(const NormCall& c) {
    constexpr int GROUPS = NORM_WG / LANES;
    if (c.dy == nullptr) {
        // 8 workgroups a CU at most; with SHIFT two rows a group at least, for the weights that come value by value
        constexpr int RG = GROUPS * (SHIFT ? 2 : 1);
        int64_t blocks = ((int64_t)c.rows + RG - 1) / RG;
        blocks = blocks < 2048 ? (blocks + 7) / 8 * 8 : 2048;
        hipLaunchKernelGGL((norm_fwd_kernel<T, VE, LANES, E, SHIFT>), dim3((unsigned)blocks), dim3(NORM_WG), 0, c.st, c.rows, c.dim,
                           (const T*)c.x, c.ldx, (const T*)c.w, (const T*)c.b, c.eps, (T*)c.y, c.mean, c.rstd);
    } else {
        const size_t lds = c.part != nullptr && GROUPS > 1 ? (size_t)2 * LANES * E * sizeof(float) : 0;
        hipLaunchKernelGGL((norm_bwd_kernel<T, VE, LANES, E, SHIFT>), dim3(c.parts), dim3(NORM_WG), lds, c.st, c.rows, c.dim,
                           (const T*)c.x, c.ldx, (const T*)c.w, (const T*)c.dy, c.lddy, c.mean, c.rstd, (T*)c.dx, c.part);
    }
    TSD_LAUNCH_CHECK("layer_norm");
    return TSD_OK;
}

// The smallest group that holds a row: a wave (or part of one) up to 32 values a lane (2048 columns), four waves beyond.
template <class T, int VE, bool SHIFT> static int norm_by_dim(const NormCall& c) {
    const int n = (c.dim + (SHIFT ? VE - 1 : 0) + VE - 1) / VE;  // loads a row
    if constexpr (VE > 1) {
        if (n <= 16) return norm_launch<T, VE, SHIFT, 16, VE>(c);
        if (n <= 32) return norm_launch<T, VE, SHIFT, 32, VE>(c);
    }
    if (n <= 64) return norm_launch<T, VE, SHIFT, 64, VE>(c);
    if (n <= 128) return norm_launch<T, VE, SHIFT, 64, 2 * VE>(c);
    if (n <= 192) return norm_launch<T, VE, SHIFT, 64, 3 * VE>(c);
    if (n <= 256) return norm_launch<T, VE, SHIFT, 64, 4 * VE>(c);
    if constexpr (VE <= 4) {
        if (n <= 512) return norm_launch<T, VE, SHIFT, 64, 8 * VE>(c);
    }
    if constexpr (VE == 1) {
        if (n <= 1024) return norm_launch<T, VE, SHIFT, 64, 16>(c);
        if (n <= 2048) return norm_launch<T, VE, SHIFT, 64, 32>(c);
    }
    if (n * VE <= 256 * 16) return norm_launch<T, VE, SHIFT, 256, 16>(c);
    if (n * VE <= 256 * 32) return norm_launch<T, VE, SHIFT, 256, 32>(c);
    return norm_launch<T, 1, false, 256, 32>(c);  // (8192 columns and a shift)
}

// 16-byte loads where every row of every tensor starts and ends on a border, or where all start equally far from one;
// value by value otherwise
struct NormPlace {
    const void* p;
    int64_t ld;
};
template <class T> static int norm_dispatch(const NormCall& c, std::initializer_list<NormPlace> rows, uintptr_t params) {
    constexpr int V = 16 / sizeof(T);
    const uintptr_t first = reinterpret_cast<uintptr_t>(rows.begin()->p);
    bool alike = true, whole = c.dim % V == 0 && params % 16 == 0;
    for (const NormPlace& r : rows) {
        if (r.p == nullptr) continue;
        const uintptr_t p = reinterpret_cast<uintptr_t>(r.p);
        alike = alike && (p - first) % 16 == 0 && (r.ld - rows.begin()->ld) % V == 0;
        whole = whole && p % 16 == 0 && r.ld % V == 0;
    }
    if (whole) return norm_by_dim<T, V, false>(c);
    if (alike && first % sizeof(T) == 0) return norm_by_dim<T, V, true>(c);
    return norm_by_dim<T, 1, false>(c);
}

static int norm_check(const char* name, int32_t dtype, int32_t rows, int32_t dim, int64_t ldx, const void* x) {
    TSD_REQUIRE(dtype == TSD_F32 || dtype == TSD_BF16 || dtype == TSD_F16, "%s: unknown type %d", name, dtype);
    TSD_REQUIRE(rows >= 0 && dim >= 1 && ldx >= dim, "%s: bad sizes rows %d dim %d row stride %lld", name, rows, dim,
                (long long)ldx);
    TSD_REQUIRE(x != nullptr || rows == 0, "%s: null pointer", name);
    if (dim > NORM_MAX_DIM) {
        set_error("%s: dim %d > %d", name, dim, NORM_MAX_DIM);
        return TSD_ERR_UNSUPPORTED;
    }
    return TSD_OK;
}

}  // namespace blk
}  // namespace tsd

using namespace tsd;
using namespace tsd::blk;

extern "C" {

int tsd_layer_norm_fwd(int32_t dtype, int32_t rows, int32_t dim, const void* x, int64_t ldx, const void* weight,
                       const void* bias, float eps, void* y, float* mean, float* rstd, void* stream) {
    const int rc = norm_check("tsd_layer_norm_fwd", dtype, rows, dim, ldx, x);
    if (rc != TSD_OK) return rc;
    if (rows == 0) return TSD_OK;
    TSD_REQUIRE(y != nullptr && (mean == nullptr) == (rstd == nullptr), "tsd_layer_norm_fwd: null pointer");
    NormCall c = {};
    c.rows = rows;
    c.dim = dim;
    c.ldx = ldx;
    c.x = x;
    c.w = weight;
    c.b = bias;
    c.eps = eps;
    c.y = y;
    c.mean = mean;
    c.rstd = rstd;
    c.st = (hipStream_t)stream;
    TSD_BY_DTYPE(dtype, T, return norm_dispatch<T>(c, {{x, ldx}, {y, dim}}, (uintptr_t)weight | (uintptr_t)bias));
    return TSD_OK;
}

size_t tsd_layer_norm_scratch_floats(int32_t rows, int32_t dim) {
    return rows < 1 || dim < 1 ? 0 : (size_t)norm_parts(rows) * 2 * dim;
}

int tsd_layer_norm_bwd(int32_t dtype, int32_t rows, int32_t dim, const void* x, int64_t ldx, const void* weight,
                       const void* dy, int64_t lddy, const float* mean, const float* rstd, void* dx, void* dweight,
                       void* dbias, float* scratch, size_t scratch_floats, void* stream) {
    const int rc = norm_check("tsd_layer_norm_bwd", dtype, rows, dim, ldx, x);
    if (rc != TSD_OK) return rc;
    const bool sums = dweight != nullptr || dbias != nullptr;
    if (rows > 0) {
        TSD_REQUIRE(dy != nullptr && mean != nullptr && rstd != nullptr && lddy >= dim, "tsd_layer_norm_bwd: null pointer");
        TSD_REQUIRE(!sums || (scratch != nullptr && scratch_floats >= tsd_layer_norm_scratch_floats(rows, dim)),
                    "tsd_layer_norm_bwd: scratch of %zu floats, %zu needed", scratch_floats,
                    tsd_layer_norm_scratch_floats(rows, dim));
    }
    NormCall c = {};
    c.rows = rows;
    c.dim = dim;
    c.ldx = ldx;
    c.lddy = lddy;
    c.x = x;
    c.w = weight;
    c.dy = dy;
    c.mean = const_cast<float*>(mean);
    c.rstd = const_cast<float*>(rstd);
    c.dx = dx;
    c.part = sums ? scratch : nullptr;
    c.parts = rows > 0 ? norm_parts(rows) : 0;
    c.st = (hipStream_t)stream;
    if (rows > 0 && (dx != nullptr || sums)) {
        int r = TSD_OK;
        TSD_BY_DTYPE(dtype, T, r = norm_dispatch<T>(c, {{x, ldx}, {dy, lddy}, {dx, dim}}, (uintptr_t)weight));
        if (r != TSD_OK) return r;
    }
    if (sums) {
        TSD_BY_DTYPE(dtype, T, hipLaunchKernelGGL((norm_reduce_kernel<T>), dim3((2 * dim + 15) / 16), dim3(256), 0, c.st,
                                                  c.parts, dim, scratch, (T*)dweight, (T*)dbias));
        TSD_LAUNCH_CHECK("layer_norm_reduce");
    }
    return TSD_OK;
}

}  // extern "C"
