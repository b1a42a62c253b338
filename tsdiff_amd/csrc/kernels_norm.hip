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

// values v * VE + j of a lane are columns (v * LANES + lane) * VE + j; columns past `dim` hold zeros
template <class T, int VE, int LANES, int E> struct NormRow {
    static constexpr int NV = E / VE;
    __device__ __forceinline__ static int col(int v, int lane) { return (v * LANES + lane) * VE; }
    __device__ __forceinline__ static void load(float (&x)[E], const T* p, int dim, int lane, float fill) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (p != nullptr && col(v, lane) < dim) {
                norm_load<T, VE>(x + v * VE, p + col(v, lane));
            } else {
#pragma unroll
                for (int j = 0; j < VE; ++j) x[v * VE + j] = fill;
            }
        }
    }
    __device__ __forceinline__ static void store(T* p, const float (&x)[E], int dim, int lane) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (col(v, lane) < dim) norm_store<T, VE>(p + col(v, lane), x + v * VE);
    }
};

template <class T, int VE, int LANES, int E>
__global__ __launch_bounds__(NORM_WG) void norm_fwd_kernel(int rows, int dim, const T* __restrict__ x, int64_t ldx,
                                                           const T* __restrict__ w, const T* __restrict__ b, float eps,
                                                           T* __restrict__ y, float* __restrict__ mean,
                                                           float* __restrict__ rstd) {
    using R = NormRow<T, VE, LANES, E>;
    __shared__ float red[4];
    constexpr int GROUPS = NORM_WG / LANES;
    const int lane = threadIdx.x % LANES;
    float wv[E], bv[E];
    R::load(wv, w, dim, lane, 1.f);
    R::load(bv, b, dim, lane, 0.f);
    const float inv = 1.f / (float)dim;
    for (int64_t r = (int64_t)blockIdx.x * GROUPS + threadIdx.x / LANES; r < rows; r += (int64_t)gridDim.x * GROUPS) {
        float v[E];
        R::load(v, x + r * ldx, dim, lane, 0.f);
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) s += v[e];
        const float m = norm_sum<LANES>(s, red) * inv;
        float q = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            v[e] = R::col(e / VE, lane) < dim ? v[e] - m : 0.f;
            q += v[e] * v[e];
        }
        const float rs = 1.f / sqrtf(norm_sum<LANES>(q, red) * inv + eps);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = v[e] * rs * wv[e] + bv[e];
        R::store(y + r * dim, v, dim, lane);
        if (mean != nullptr && lane == 0) {
            mean[r] = m;
            rstd[r] = rs;
        }
    }
}

template <class T, int VE, int LANES, int E>
__global__ __launch_bounds__(NORM_WG) void norm_bwd_kernel(int rows, int dim, const T* __restrict__ x, int64_t ldx,
                                                           const T* __restrict__ w, const T* __restrict__ dy,
                                                           int64_t lddy, const float* __restrict__ mean,
                                                           const float* __restrict__ rstd, T* __restrict__ dx,
                                                           float* __restrict__ part) {
    using R = NormRow<T, VE, LANES, E>;
    __shared__ float red[4];
    extern __shared__ float sums[];  // [GROUPS][2][dim padded to LANES * E]
    constexpr int GROUPS = NORM_WG / LANES;
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    float wv[E], dw[E], db[E];
    R::load(wv, w, dim, lane, 1.f);
#pragma unroll
    for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.f;
    const float inv = 1.f / (float)dim;
    for (int64_t r = (int64_t)blockIdx.x * GROUPS + group; r < rows; r += (int64_t)gridDim.x * GROUPS) {
        float v[E], g[E];
        R::load(v, x + r * ldx, dim, lane, 0.f);
        R::load(g, dy + r * lddy, dim, lane, 0.f);
        const float m = mean[r], rs = rstd[r];
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            v[e] = R::col(e / VE, lane) < dim ? (v[e] - m) * rs : 0.f;
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
            R::store(dx + r * dim, g, dim, lane);
        }
    }
    if (part == nullptr) return;
    constexpr int W = LANES * E;
    if constexpr (GROUPS > 1) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int c = R::col(e / VE, lane) + e % VE;
            sums[(group * 2) * W + c] = dw[e];
            sums[(group * 2 + 1) * W + c] = db[e];
        }
        __syncthreads();
        for (int c = threadIdx.x; c < 2 * W; c += NORM_WG) {
            const int col = c % W;
            if (col >= dim) continue;
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < GROUPS; ++k) s += sums[k * 2 * W + c];
            part[(size_t)blockIdx.x * 2 * dim + (c / W) * dim + col] = s;
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int c = R::col(e / VE, lane) + e % VE;
            if (c < dim) {
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

static int norm_parts(int rows) {  // workgroups of the backward = rows of partial sums: about 4 a CU, >= 16 rows each
    const int n = (rows + 15) / 16;
    return n < 1 ? 1 : n < NORM_MAX_PARTS ? n : NORM_MAX_PARTS;
}

template <class T, int VE, int LANES, int E> static int norm_launch(const NormCall& c) {
    constexpr int GROUPS = NORM_WG / LANES;
    if (c.dy == nullptr) {
        int64_t blocks = ((int64_t)c.rows + GROUPS - 1) / GROUPS;
        blocks = blocks < 16384 ? blocks : 16384;
        hipLaunchKernelGGL((norm_fwd_kernel<T, VE, LANES, E>), dim3((unsigned)blocks), dim3(NORM_WG), 0, c.st, c.rows, c.dim,
                           (const T*)c.x, c.ldx, (const T*)c.w, (const T*)c.b, c.eps, (T*)c.y, c.mean, c.rstd);
    } else {
        const size_t lds = c.part != nullptr && GROUPS > 1 ? (size_t)GROUPS * 2 * LANES * E * sizeof(float) : 0;
        static_assert(GROUPS == 1 || GROUPS * 2 * LANES * E * 4 <= 48 * 1024, "partial sums fit the default LDS limit");
        hipLaunchKernelGGL((norm_bwd_kernel<T, VE, LANES, E>), dim3(c.parts), dim3(NORM_WG), lds, c.st, c.rows, c.dim,
                           (const T*)c.x, c.ldx, (const T*)c.w, (const T*)c.dy, c.lddy, c.mean, c.rstd, (T*)c.dx, c.part);
    }
    TSD_LAUNCH_CHECK("layer_norm");
    return TSD_OK;
}

// the smallest group that holds a row: a wave (or part of one) up to 16 values a lane, four waves up to 32
template <class T, int VE> static int norm_by_dim(const NormCall& c) {
    const int n = (c.dim + VE - 1) / VE;  // loads a row
    if constexpr (VE * sizeof(T) == 16) {
        if (n <= 16) return norm_launch<T, VE, 16, VE>(c);
        if (n <= 32) return norm_launch<T, VE, 32, VE>(c);
    }
    if (n <= 64) return norm_launch<T, VE, 64, VE>(c);
    if (n <= 128) return norm_launch<T, VE, 64, 2 * VE>(c);
    if constexpr (VE <= 4) {
        if (n <= 256) return norm_launch<T, VE, 64, 4 * VE>(c);
    }
    if constexpr (VE <= 2) {
        if (n <= 512) return norm_launch<T, VE, 64, 8 * VE>(c);
    }
    if (c.dim <= 256 * 8) return norm_launch<T, VE, 256, 8>(c);
    if (c.dim <= 256 * 16) return norm_launch<T, VE, 256, 16>(c);
    return norm_launch<T, VE, 256, 32>(c);
}

template <class T> static int norm_by_width(const NormCall& c, int ve) {
    if constexpr (sizeof(T) == 2) {
        if (ve == 8) return norm_by_dim<T, 8>(c);
        if (ve >= 2) return norm_by_dim<T, 2>(c);
    } else {
        if (ve == 4) return norm_by_dim<T, 4>(c);
    }
    return norm_by_dim<T, 1>(c);
}

// values a load may take: 16 bytes where every row of every tensor starts on such a border and ends on one
static int norm_width(size_t size, int dim, int64_t ldx, int64_t lddy, uintptr_t any) {
    const int most = (int)(16 / size);
    for (int ve = most; ve > 1; ve /= 2)
        if (dim % ve == 0 && ldx % ve == 0 && lddy % ve == 0 && any % (ve * size) == 0) return ve;
    return 1;
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
    const uintptr_t any = (uintptr_t)x | (uintptr_t)y | (uintptr_t)weight | (uintptr_t)bias;
    TSD_BY_DTYPE(dtype, T, return norm_by_width<T>(c, norm_width(sizeof(T), dim, ldx, dim, any)));
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
        const uintptr_t any = (uintptr_t)x | (uintptr_t)dy | (uintptr_t)dx | (uintptr_t)weight;
        int r = TSD_OK;
        TSD_BY_DTYPE(dtype, T, r = norm_by_width<T>(c, norm_width(sizeof(T), dim, ldx, lddy, any)));
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
