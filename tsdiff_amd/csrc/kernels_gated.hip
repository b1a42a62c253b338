// kernels_gated.hip -- the gated linear layer h = act(x Wg^T + bg) * (x Wu^T + bu), forward and backward.
//
//   g = x Wg^T + bg, u = x Wu^T + bu, h = a(g) u
//   dg = dh u a'(g), du = dh a(g);  dx = dg Wg + du Wu;  dWg = dg^T x, dWu = du^T x;  dbg, dbu = column sums
//
// Forward: one launch; a workgroup multiplies a tile of rows with the same columns of both weights, so a lane holds g and u
// of one place and the product leaves the kernel as h.  Backward: launch 1 computes g and u again (they are not kept: at 256
// inputs reading them back in f32 costs more than the products) and writes D = [dg | du] in the tensors' type -- the one
// rounding of an intermediate, since D is the next two products' matrix operand -- with each row tile's column sums in fp32;
// launch 2 is dx = D [Wg; Wu]; launch 3 dW = D^T x, the rows split over workgroups; launch 4 adds the parts in a fixed order.
#include "gemm_tile.hpp"

namespace tsd {
namespace blk {

// a(g) and a'(g), kinds of tsd_act_fwd
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.f + fast_exp(-g)); }
__device__ __forceinline__ float softplus(float g) { return fmaxf(g, 0.f) + log1pf(fast_exp(-fabsf(g))); }
__device__ __forceinline__ float act_value(int kind, float g) {
    if (kind == 0) return g * sigmoid(g);
    if (kind == 2) return g < 0.f ? 0.f : g;
    return softplus(g) - (kind == 1 ? 0.693147180559945309f : 0.f);
}
__device__ __forceinline__ float act_slope(int kind, float g) {
    if (kind == 2) return g > 0.f ? 1.f : 0.f;
    const float s = sigmoid(g);
    return kind == 0 ? s * (1.f + g * (1.f - s)) : s;
}

struct GatedDims {
    int rows, in, out, outp;  // outp: out rounded up to 8, the width of each half of D
    int64_t ldx, lddh;
    int kind;
    bool xvec, wvec, hvec, dhvec;
};

template <class T, int BM, int BN, bool BWD>
__global__ __launch_bounds__(GEMM_WG) void gated_kernel(GatedDims d, int ftiles, int mtiles, const T* __restrict__ x,
                                                        const T* __restrict__ wg, const T* __restrict__ wu,
                                                        const T* __restrict__ bg, const T* __restrict__ bu,
                                                        const T* __restrict__ dh, T* __restrict__ h, T* __restrict__ D,
                                                        float* __restrict__ part) {
    extern __shared__ __align__(16) char lds[];
    constexpr int FT = BN / 2, TN = BN / 64, TM = BM / 32;  // columns a tile; gate (and up) subtiles, row subtiles of a wave
    const TileAt at = tile_at(blockIdx.x, ftiles);
    if (at.lo >= mtiles) return;
    const int m0 = at.lo * BM, f0 = at.sh * FT;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wn = wave & 1, wm = wave >> 1;
    const int nbase = wn * (FT / 2), mrow = wm * (BM / 2);
    const RowSource<T> ns = {wg, wu, d.in, d.out, d.in, f0, FT, f0, d.wvec};
    const RowSource<T> ms = {x, x, d.ldx, d.rows, d.in, m0, BM, 0, d.xvec};
    f32x4 acc[2 * TN][TM];
    gemm_tile<T, BM, BN>(lds, ns, ms, 0, d.in, mrow,
                         [&](int j) { return j < TN ? nbase + j * 16 : FT + nbase + (j - TN) * 16; }, acc);
    const int r = lane & 15, c4 = (lane >> 4) * 4;
    float* red = reinterpret_cast<float*>(lds);  // [2 (wm)][2][FT] column sums
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const int fl = nbase + j * 16 + c4, f = f0 + fl, nf = d.out - f;
        const f32x4 zero = {0, 0, 0, 0};
        const f32x4 vbg = bg != nullptr ? load4(bg + f, nf, false) : zero;
        const f32x4 vbu = bu != nullptr ? load4(bu + f, nf, false) : zero;
        f32x4 sg = zero, su = zero;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const int m = m0 + mrow + i * 16 + r;
            const f32x4 g = acc[j][i] + vbg, u = acc[j + TN][i] + vbu;
            if constexpr (!BWD) {
                f32x4 o;
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = act_value(d.kind, g[e]) * u[e];
                if (m < d.rows) store4(h + (int64_t)m * d.out + f, o, nf, d.hvec);
            } else {
                f32x4 og = zero, ou = zero;
                if (m < d.rows) {
                    const f32x4 v = load4(dh + (int64_t)m * d.lddh + f, nf, d.dhvec);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (e < nf) {
                            ou[e] = v[e] * act_value(d.kind, g[e]);
                            og[e] = v[e] * u[e] * act_slope(d.kind, g[e]);
                        }
                    T* o = D + (int64_t)m * 2 * d.outp + f;
                    store4(o, og, d.outp - f, true);
                    store4(o + d.outp, ou, d.outp - f, true);
                }
                sg += og;
                su += ou;
            }
        }
        if constexpr (BWD) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
#pragma unroll
                for (int s = 1; s < 16; s *= 2) {
                    sg[e] += __shfl_xor(sg[e], s, 64);
                    su[e] += __shfl_xor(su[e], s, 64);
                }
                if (r == 0) {  // (gemm_tile ends behind a barrier: the operand tiles are free)
                    red[(wm * 2) * FT + fl + e] = sg[e];
                    red[(wm * 2 + 1) * FT + fl + e] = su[e];
                }
            }
        }
    }
    if constexpr (BWD) {
        if (part == nullptr) return;
        __syncthreads();
        for (int t = threadIdx.x; t < 2 * FT; t += GEMM_WG) {
            const int f = f0 + t % FT;
            if (f < d.outp) part[(int64_t)at.lo * 2 * d.outp + (t / FT) * d.outp + f] = red[t] + red[2 * FT + t];
        }
    }
}

// dx[m][k] = sum over f < 2 outp of D[m][f] [Wg; Wu][f][k]
template <class T, int BM, int BN>
__global__ __launch_bounds__(GEMM_WG) void gated_dx_kernel(GatedDims d, int ktiles, int mtiles, const T* __restrict__ D,
                                                           const T* __restrict__ wg, const T* __restrict__ wu,
                                                           T* __restrict__ dx) {
    extern __shared__ __align__(16) char lds[];
    const TileAt at = tile_at(blockIdx.x, ktiles);
    if (at.lo >= mtiles) return;
    const int m0 = at.lo * BM, k0 = at.sh * BN;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int nbase = (wave & 1) * (BN / 2), mrow = (wave >> 1) * (BM / 2);
    const ColSource<T> ns = {wg, wu, d.in, d.in, d.out, k0, d.outp, d.wvec};
    const RowSource<T> ms = {D, D, 2 * d.outp, d.rows, 2 * d.outp, m0, BM, 0, true};
    f32x4 acc[BN / 32][BM / 32];
    gemm_tile<T, BM, BN>(lds, ns, ms, 0, 2 * d.outp, mrow, [&](int j) { return nbase + j * 16; }, acc);
    const int r = lane & 15, c4 = (lane >> 4) * 4;
#pragma unroll
    for (int j = 0; j < BN / 32; ++j)
#pragma unroll
        for (int i = 0; i < BM / 32; ++i) {
            const int m = m0 + mrow + i * 16 + r, k = k0 + nbase + j * 16 + c4;
            if (m < d.rows) store4(dx + (int64_t)m * d.in + k, acc[j][i], d.in - k, d.wvec);
        }
}

// part[s][f][k] = sum over the rows of split s of D[m][f] x[m][k]
template <class T, int BM, int BN>
__global__ __launch_bounds__(GEMM_WG) void gated_dw_kernel(GatedDims d, int ktiles, int ftiles, int rows_a_split,
                                                           const T* __restrict__ D, const T* __restrict__ x,
                                                           float* __restrict__ part) {
    extern __shared__ __align__(16) char lds[];
    const int k0 = (blockIdx.x % ktiles) * BN, f0 = (blockIdx.x / ktiles) * BM;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int nbase = (wave & 1) * (BN / 2), mrow = (wave >> 1) * (BM / 2);
    const int64_t rb = (int64_t)blockIdx.y * rows_a_split;
    const int n = (int)(d.rows - rb < rows_a_split ? d.rows - rb : rows_a_split);
    const ColSource<T> ns = {x + rb * d.ldx, x, d.ldx, d.in, n, k0, 1 << 30, d.xvec};
    const ColSource<T> ms = {D + rb * 2 * d.outp, D, 2 * d.outp, 2 * d.outp, n, f0, 1 << 30, true};
    f32x4 acc[BN / 32][BM / 32];
    gemm_tile<T, BM, BN>(lds, ns, ms, 0, n, mrow, [&](int j) { return nbase + j * 16; }, acc);
    const int r = lane & 15, c4 = (lane >> 4) * 4;
    float* o = part + (int64_t)blockIdx.y * 2 * d.outp * d.in;
#pragma unroll
    for (int j = 0; j < BN / 32; ++j)
#pragma unroll
        for (int i = 0; i < BM / 32; ++i) {
            const int f = f0 + mrow + i * 16 + r, k = k0 + nbase + j * 16 + c4;
            if (f < 2 * d.outp) store4(o + (int64_t)f * d.in + k, acc[j][i], d.in - k, d.in % 4 == 0);
        }
}

// the parts of dW (workgroups below wblocks) and of the column sums, added in order
template <class T>
__global__ __launch_bounds__(256) void gated_reduce_kernel(GatedDims d, int wblocks, int splits, int mtiles,
                                                           const float* __restrict__ wpart, const float* __restrict__ bpart,
                                                           T* __restrict__ dwg, T* __restrict__ dwu, T* __restrict__ dbg,
                                                           T* __restrict__ dbu) {
    if ((int)blockIdx.x < wblocks) {
        const int64_t size = (int64_t)2 * d.outp * d.in, i = ((int64_t)blockIdx.x * 256 + threadIdx.x);
        if (i >= size) return;
        const int f = (int)(i / d.in), k = (int)(i % d.in), half = f >= d.outp, ff = f - half * d.outp;
        if (ff >= d.out) return;
        float s = 0.f;
#pragma unroll 8
        for (int p = 0; p < splits; ++p) s += wpart[p * size + i];
        T* o = half ? dwu : dwg;
        if (o != nullptr) o[(int64_t)ff * d.in + k] = (T)s;
        return;
    }
    __shared__ float red[16][17];
    const int cx = threadIdx.x & 15, q = threadIdx.x >> 4, c = ((int)blockIdx.x - wblocks) * 16 + cx, W = 2 * d.outp;
    float s = 0.f;
    if (c < W) {
#pragma unroll 8
        for (int p = q; p < mtiles; p += 16) s += bpart[(int64_t)p * W + c];
    }
    red[q][cx] = s;
    __syncthreads();
    if (q == 0 && c < W) {
        s = red[0][cx];
#pragma unroll
        for (int j = 1; j < 16; ++j) s += red[j][cx];
        const int half = c >= d.outp, ff = c - half * d.outp;
        T* o = half ? dbu : dbg;
        if (o != nullptr && ff < d.out) o[ff] = (T)s;
    }
}

constexpr int GATED_BM = 128, GATED_BN = 128;

static int gated_splits(int rows, int in, int outp, int* rows_a_split) {
    const int tiles = ((2 * outp + GATED_BM - 1) / GATED_BM) * ((in + GATED_BN - 1) / GATED_BN);
    int s = (512 + tiles - 1) / tiles;
    const int most = (rows + 255) / 256;
    s = s < most ? s : most;
    s = s < 1 ? 1 : s;
    int per = (rows + s - 1) / s;
    per = (per + GEMM_K - 1) / GEMM_K * GEMM_K;
    per = per < GEMM_K ? GEMM_K : per;
    if (rows_a_split) *rows_a_split = per;
    return rows > 0 ? (rows + per - 1) / per : 0;
}

struct GatedScratch {  // bytes from the start
    size_t D, bpart, wpart, total;
    int mtiles, splits, rows_a_split;
};
static GatedScratch gated_scratch(int dtype, int rows, int in, int out) {
    GatedScratch s = {};
    const size_t outp = ((size_t)out + 7) / 8 * 8, es = dtype == TSD_F32 ? 4 : 2;
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    s.mtiles = (rows + GATED_BM - 1) / GATED_BM;
    s.splits = gated_splits(rows, in, (int)outp, &s.rows_a_split);
    s.D = 0;
    s.bpart = up((size_t)rows * 2 * outp * es);
    s.wpart = s.bpart + up((size_t)s.mtiles * 2 * outp * 4);
    s.total = s.wpart + up((size_t)s.splits * 2 * outp * in * 4);
    return s;
}

static int gated_check(const char* name, int32_t dtype, int32_t act, int32_t rows, int32_t in, int32_t out, int64_t ldx,
                       const void* x, const void* wg, const void* wu) {
    TSD_REQUIRE(dtype == TSD_F32 || dtype == TSD_BF16 || dtype == TSD_F16, "%s: unknown type %d", name, dtype);
    TSD_REQUIRE(act >= 0 && act <= 3, "%s: unknown activation %d", name, act);
    TSD_REQUIRE(rows >= 0 && in >= 1 && out >= 1 && ldx >= in, "%s: bad sizes rows %d in %d out %d row stride %lld", name, rows,
                in, out, (long long)ldx);
    TSD_REQUIRE(rows == 0 || (x != nullptr && wg != nullptr && wu != nullptr), "%s: null pointer", name);
    if (in > (1 << 20) || out > (1 << 20) || ldx > (1ll << 31)) {
        set_error("%s: in %d out %d row stride %lld: at most 2^20 features", name, in, out, (long long)ldx);
        return TSD_ERR_UNSUPPORTED;
    }
    return TSD_OK;
}

template <class T>
static GatedDims gated_dims(int rows, int in, int out, int act, const void* x, int64_t ldx, const void* wg, const void* wu,
                            const void* dx) {
    const int v = (int)(16 / sizeof(T)) > 8 ? 8 : 8;  // chunks of 8 values: a row of a whole number of them
    GatedDims d = {};
    d.rows = rows;
    d.in = in;
    d.out = out;
    d.outp = (out + 7) / 8 * 8;
    d.ldx = ldx;
    d.kind = act;
    d.xvec = in % v == 0 && ldx % v == 0 && aligned16(x);
    d.wvec = in % v == 0 && aligned16(wg) && aligned16(wu) && aligned16(dx);
    return d;
}

template <class T>
static int gated_fwd(GatedDims d, const void* x, const void* wg, const void* wu, const void* bg, const void* bu, void* h,
                     hipStream_t st) {
    static DeviceOnce once;
    constexpr int lds = gemm_lds<T, GATED_BM, GATED_BN>();
    auto k = gated_kernel<T, GATED_BM, GATED_BN, false>;
    const int rc = allow_lds(k, lds, once);
    if (rc != TSD_OK) return rc;
    const int ft = (d.out + GATED_BN / 2 - 1) / (GATED_BN / 2), mt = (d.rows + GATED_BM - 1) / GATED_BM;
    d.hvec = d.out % 4 == 0 && aligned16(h);
    hipLaunchKernelGGL(k, dim3(tile_grid(mt, ft)), dim3(GEMM_WG), lds, st, d, ft, mt, (const T*)x, (const T*)wg, (const T*)wu,
                       (const T*)bg, (const T*)bu, (const T*)nullptr, (T*)h, (T*)nullptr, (float*)nullptr);
    TSD_LAUNCH_CHECK("gated_fwd");
    return TSD_OK;
}

template <class T>
static int gated_bwd(GatedDims d, const GatedScratch& s, const void* x, const void* wg, const void* wu, const void* bg,
                     const void* bu, const void* dh, int64_t lddh, void* dx, void* dwg, void* dwu, void* dbg, void* dbu,
                     char* scratch, hipStream_t st) {
    static DeviceOnce once_d, once_x, once_w;
    constexpr int lds = gemm_lds<T, GATED_BM, GATED_BN>();
    T* D = reinterpret_cast<T*>(scratch + s.D);
    float* bpart = reinterpret_cast<float*>(scratch + s.bpart);
    float* wpart = reinterpret_cast<float*>(scratch + s.wpart);
    const bool sums = dbg != nullptr || dbu != nullptr, weights = dwg != nullptr || dwu != nullptr;
    int rc;
    if (d.rows > 0) {
        d.lddh = lddh;
        d.dhvec = d.out % 4 == 0 && lddh % 4 == 0 && aligned16(dh);
        auto k1 = gated_kernel<T, GATED_BM, GATED_BN, true>;
        if ((rc = allow_lds(k1, lds, once_d)) != TSD_OK) return rc;
        const int ft = (d.outp + GATED_BN / 2 - 1) / (GATED_BN / 2);
        hipLaunchKernelGGL(k1, dim3(tile_grid(s.mtiles, ft)), dim3(GEMM_WG), lds, st, d, ft, s.mtiles, (const T*)x, (const T*)wg,
                           (const T*)wu, (const T*)bg, (const T*)bu, (const T*)dh, (T*)nullptr, D, sums ? bpart : nullptr);
        TSD_LAUNCH_CHECK("gated_bwd");
        const int kt = (d.in + GATED_BN - 1) / GATED_BN;
        if (dx != nullptr) {
            auto k2 = gated_dx_kernel<T, GATED_BM, GATED_BN>;
            if ((rc = allow_lds(k2, lds, once_x)) != TSD_OK) return rc;
            hipLaunchKernelGGL(k2, dim3(tile_grid(s.mtiles, kt)), dim3(GEMM_WG), lds, st, d, kt, s.mtiles, D, (const T*)wg,
                               (const T*)wu, (T*)dx);
            TSD_LAUNCH_CHECK("gated_dx");
        }
        if (weights) {
            auto k3 = gated_dw_kernel<T, GATED_BM, GATED_BN>;
            if ((rc = allow_lds(k3, lds, once_w)) != TSD_OK) return rc;
            const int f2 = (2 * d.outp + GATED_BM - 1) / GATED_BM;
            hipLaunchKernelGGL(k3, dim3(kt * f2, s.splits), dim3(GEMM_WG), lds, st, d, kt, f2, s.rows_a_split, D, (const T*)x,
                               wpart);
            TSD_LAUNCH_CHECK("gated_dw");
        }
    }
    if (weights || sums) {
        const int wb = weights ? (int)(((int64_t)2 * d.outp * d.in + 255) / 256) : 0, bb = sums ? (2 * d.outp + 15) / 16 : 0;
        hipLaunchKernelGGL(gated_reduce_kernel<T>, dim3(wb + bb), dim3(256), 0, st, d, wb, s.splits, s.mtiles, wpart, bpart,
                           (T*)dwg, (T*)dwu, (T*)dbg, (T*)dbu);
        TSD_LAUNCH_CHECK("gated_reduce");
    }
    return TSD_OK;
}

}  // namespace blk
}  // namespace tsd

using namespace tsd;
using namespace tsd::blk;

extern "C" {

int tsd_gated_linear_fwd(int32_t dtype, int32_t act, int32_t rows, int32_t in, int32_t out, const void* x, int64_t ldx,
                         const void* w_gate, const void* w_up, const void* b_gate, const void* b_up, void* h, void* stream) {
    const int rc = gated_check("tsd_gated_linear_fwd", dtype, act, rows, in, out, ldx, x, w_gate, w_up);
    if (rc != TSD_OK) return rc;
    if (rows == 0) return TSD_OK;
    TSD_REQUIRE(h != nullptr, "tsd_gated_linear_fwd: null pointer");
    TSD_BY_DTYPE(dtype, T, return gated_fwd<T>(gated_dims<T>(rows, in, out, act, x, ldx, w_gate, w_up, nullptr), x, w_gate,
                                               w_up, b_gate, b_up, h, (hipStream_t)stream));
    return TSD_OK;
}

size_t tsd_gated_linear_scratch_floats(int32_t dtype, int32_t rows, int32_t in, int32_t out) {
    if (rows < 1 || in < 1 || out < 1) return 0;
    return gated_scratch(dtype, rows, in, out).total / 4;
}

int tsd_gated_linear_bwd(int32_t dtype, int32_t act, int32_t rows, int32_t in, int32_t out, const void* x, int64_t ldx,
                         const void* w_gate, const void* w_up, const void* b_gate, const void* b_up, const void* dh,
                         int64_t lddh, void* dx, void* dw_gate, void* dw_up, void* db_gate, void* db_up, float* scratch,
                         size_t scratch_floats, void* stream) {
    const int rc = gated_check("tsd_gated_linear_bwd", dtype, act, rows, in, out, ldx, x, w_gate, w_up);
    if (rc != TSD_OK) return rc;
    const GatedScratch s = gated_scratch(dtype, rows, in, out);
    TSD_REQUIRE(rows == 0 || (dh != nullptr && lddh >= out), "tsd_gated_linear_bwd: null pointer or row stride");
    TSD_REQUIRE(rows == 0 || (scratch != nullptr && aligned16(scratch) && scratch_floats * 4 >= s.total),
                "tsd_gated_linear_bwd: scratch of %zu floats, %zu needed (16-byte aligned)", scratch_floats, s.total / 4);
    TSD_BY_DTYPE(dtype, T, return gated_bwd<T>(gated_dims<T>(rows, in, out, act, x, ldx, w_gate, w_up, dx), s, x, w_gate, w_up,
                                               b_gate, b_up, dh, lddh, dx, dw_gate, dw_up, db_gate, db_up, (char*)scratch,
                                               (hipStream_t)stream));
    return TSD_OK;
}

}  // extern "C"
