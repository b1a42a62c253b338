// kernels_gated.hip -- the gated linear layer h = act(x Wg^T + bg) * (x Wu^T + bu), forward and backward.
//
//   g = x Wg^T + bg, u = x Wu^T + bu, h = a(g) u
//   dg = dh u a'(g), du = dh a(g);  dx = dg Wg + du Wu;  dWg = dg^T x, dWu = du^T x;  dbg, dbu = column sums
//
// Forward: one launch; a workgroup multiplies a tile of rows with the same columns of both weights, so a lane holds g and u
// of one place and the product leaves the kernel as h.  Backward: launch 1 computes g and u again (they are not kept, which saves
// 2 rows out values between the passes; in time that is the cheaper choice in 16 bits up to about 460 inputs, where writing and
// reading them costs as much as the products, in f32 only up to about 120) and writes D = [dg | du] in the tensors' type -- the
// one rounding of an intermediate, since D is the next two products' matrix operand; a small D (at most 2^18 values of 16 bits) is
// written with what the rounding left as a second half of twice the width, which the products go over too, since sums of few
// terms show one rounding more than large ones, and time is no matter there -- with each row tile's column sums in fp32;
// f16 gradients put a launch in front, by which D lies in the middle of f16's range whatever the size of dh (GatedMaxes);
// launch 2 is dx = D [Wg; Wu]; launch 3 dW = D^T x, the rows split over workgroups; launch 4 adds the parts in a fixed order.
//
// Measured (GPU time a launch; each product is 4 rows in out operations):
//   bf16, 65536 x 256 -> 2 x 1024: forward 121 us (568 TFLOP/s, h and x are 170 MB of it), first of the backward 178 us (it
//   writes D, 268 MB, and reads dh, 134 MB), dx 85 us (809 TFLOP/s), dW 90 us (764 TFLOP/s), sums 13 us.  Bound by what a CU
//   draws from L2 (about 10 TB/s over the chip: each row of x goes to 16 column tiles), the two first ones by that and by memory.
//   f32, 3600 x 256 -> 2 x 1024: 30, 36, 32, 32 and 11 us; six plane products each: 118 to 124 TFLOP/s of f32 are 710 to 743 of
//   bf16.
//   f16, 5003 x 204 -> 2 x 530: 14 us and 3 for the copies of odd rows, then 10 (gated_max_kernel), 18, 13, 14 and 8 us.
//   f32, 17 x 256 -> 2 x 512, forward: 8 us: a chain of eight steps in 16 workgroups.
#include <type_traits>

#include "gemm_tile.hpp"

namespace tsd {
namespace blk {

// a(g) and a'(g), kinds of tsd_act_fwd
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.f + fast_exp(-g)); }
__device__ __forceinline__ float softplus(float g) { return fmaxf(g, 0.f) + log1pf(fast_exp(-fabsf(g))); }
// KIND < 0: any of them, by `kind` (the same in all lanes)
template <int KIND> __device__ __forceinline__ float act_value(int kind, float g) {
    if constexpr (KIND >= 0) kind = KIND;
    if (kind == 0) return g * sigmoid(g);
    if (kind == 2) return g < 0.f ? 0.f : g;
    return softplus(g) - (kind == 1 ? 0.693147180559945309f : 0.f);
}
template <int KIND> __device__ __forceinline__ float act_slope(int kind, float g) {
    if constexpr (KIND >= 0) kind = KIND;
    if (kind == 2) return g > 0.f ? 1.f : 0.f;
    const float s = sigmoid(g);
    return kind == 0 ? s + g * s * (1.f - s) : s;
}

// sum over the 16 lanes l / 16 * 16 ..: neighbours, pairs, halves of 8, halves of 16, inside of the vector pipe
template <int CTRL> __device__ __forceinline__ float from_lane(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float over_16(float v) {
    v += from_lane<0xB1>(v);   // quad_perm 1 0 3 2
    v += from_lane<0x4E>(v);   // quad_perm 2 3 0 1
    v += from_lane<0x141>(v);  // row_half_mirror
    return v + from_lane<0x140>(v);  // row_mirror
}

struct GatedDims {
    int rows, in, out, outp;  // outp: out rounded up to 8, the width of each half of D
    int planes;               // of D: 1, or 2 with what the rounding left
    int inw;                  // values a row of x and the weights as the products read them: in, or in rounded up to 8 (packed)
    int64_t ldx, lddh, ldw;
    int kind;
    bool bvec;  // both biases: four values a load
    int xvw, wvw, dhvw, hvw, dxvw;  // values a load or store of x, the weights, dh, h, dx may take
};

// f16: D = [dg | du] times a power of two s, by which neither small gradients fall among the subnormal numbers (steps of 2^-24)
// nor large products beyond 65504 (4096 x 256 -> 2 x 512, dh of 1e-5: dW off by 1.8e-3 without s, by 2.9e-4 with it, as for dh
// of 1; rounding dW alone: 2.1e-4).  One s for all of D, since its rows and its columns are both summed over; it takes the bound
//   |D| <= max |dh| (X W + max |b| + 1) 1.25   (|a'| < 1.1, |a(g)| < |g| + 0.7, the rest is room for roundings)
// into 2^14 .. 2^15, X and W being the largest norms of a row of x and of a row of the weights.  The bound lies above D's ordinary
// values by about 5 sqrt(in), which leaves them 16 to 26 powers of two above the subnormal numbers; with norms a single large
// value in x or the weights costs what it may make of u, not in times that.  What is not finite is left out: its rows are lost
// either way.
template <class T> constexpr bool gated_scaled() { return std::is_same<T, f16>::value; }
struct GatedScale {
    float by, undo;
};
using u16x2 = unsigned short __attribute__((ext_vector_type(2)));
constexpr int GATED_MAX_WG = 1024, GATED_MAX_WGS = 256;
struct GatedMax {  // bits that compare like the values: norms of x and the weights (bf16, rounded up), biases and dh (f16)
    u16x2 xw, bd;
};
__device__ __forceinline__ u16x2 larger(u16x2 a, u16x2 b) { return __builtin_elementwise_max(a, b); }
template <int CTRL> __device__ __forceinline__ u16x2 from_lane(u16x2 v) {
    return __builtin_bit_cast(u16x2, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ u16x2 largest_of_wave(u16x2 v) {
    v = larger(v, from_lane<0xB1>(v));  // neighbours, pairs, halves of 8 and of 16 lanes, as over_16
    v = larger(v, from_lane<0x4E>(v));
    v = larger(v, from_lane<0x141>(v));
    v = larger(v, from_lane<0x140>(v));
    uint32_t a = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    const uint32_t x = r[0], y = r[1];
    a = __builtin_bit_cast(uint32_t, larger(__builtin_bit_cast(u16x2, x), __builtin_bit_cast(u16x2, y)));
    const auto q = __builtin_amdgcn_permlane32_swap(a, a, false, false);
    const uint32_t z = q[0], w = q[1];
    return larger(__builtin_bit_cast(u16x2, z), __builtin_bit_cast(u16x2, w));
}
// (the list is asked for where other loads are waited for too)
template <class T> struct GatedMaxes {
    u32x4 raw[2];
    __device__ __forceinline__ void load(const GatedMax* __restrict__ maxes) {
        if constexpr (gated_scaled<T>()) {
            const u32x4* p = reinterpret_cast<const u32x4*>(maxes) + 2 * (threadIdx.x & 63);
            static_assert(GATED_MAX_WGS == 4 * 64, "two loads a lane");
            raw[0] = p[0];
            raw[1] = p[1];
        }
    }
    __device__ __forceinline__ GatedScale scale() const {
        if constexpr (!gated_scaled<T>()) return {1.f, 1.f};
        auto two = [&](int i, int j) { return __builtin_bit_cast(u16x2, (uint32_t)raw[i][j]); };
        const u16x2 xw = largest_of_wave(larger(larger(two(0, 0), two(0, 2)), larger(two(1, 0), two(1, 2))));
        const u16x2 bd = largest_of_wave(larger(larger(two(0, 1), two(0, 3)), larger(two(1, 1), two(1, 3))));
        auto value = [](unsigned short b) { return (float)__builtin_bit_cast(f16, b); };
        auto norm = [](unsigned short b) { return __builtin_bit_cast(float, (uint32_t)b << 16); };
        // 2^-24 .. 2^70, or 0
        const float bound = value(bd[1]) * 1.25f * (norm(xw[0]) * norm(xw[1]) + value(bd[0]) + 1.f);
        const int e = (int)(__builtin_bit_cast(uint32_t, bound) >> 23);  // 2^(e - 127) <= bound
        const int to = bound > 0.f ? 127 + 14 + 127 - e : 127;
        return {__builtin_bit_cast(float, (uint32_t)to << 23), __builtin_bit_cast(float, (uint32_t)(254 - to) << 23)};
    }
};

// A tile of BM rows x BC columns in LDS on its way to (from) memory, so that neighbouring lanes touch neighbouring bytes
template <class T, int BM, int BC, int WG> struct OutTile {
    static constexpr int LD = BC * (int)sizeof(T) + 16, BYTES = BM * LD, CH = BC / 8, UNITS = BM * CH;
    static constexpr int U = (UNITS + WG - 1) / WG;
    __device__ __forceinline__ static T* at(char* lds, int row, int col) { return reinterpret_cast<T*>(lds + row * LD) + col; }
    __device__ __forceinline__ static void fetch(Raw<T> (&raw)[U], const T* p, int64_t ld, int rows, int cols, int vw) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = threadIdx.x + i * WG, r = u / CH, c = (u % CH) * 8, n = u < UNITS && r < rows ? cols - c : 0;
            load_raw(raw[i], p + (n > 0 ? r * ld + c : 0), n < 0 ? 0 : n > 8 ? 8 : n, vw);
        }
    }
    __device__ __forceinline__ static void keep(const Raw<T> (&raw)[U], char* lds) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = threadIdx.x + i * WG;
            if (UNITS % WG == 0 || u < UNITS)
                __builtin_memcpy(__builtin_assume_aligned(at(lds, u / CH, (u % CH) * 8), 16), &raw[i], sizeof(Raw<T>));
        }
    }
    __device__ __forceinline__ static void write(char* lds, T* p, int64_t ld, int rows, int cols, int vw) {
        if (vw * sizeof(T) >= 16) {
            constexpr int V = 16 / sizeof(T), CV = BC / V;
            for (int u = threadIdx.x; u < BM * CV; u += WG) {
                const int r = u / CV, c = (u % CV) * V;
                if (r < rows && c < cols)
                    *reinterpret_cast<u32x4*>(p + r * ld + c) = *reinterpret_cast<const u32x4*>(at(lds, r, c));
            }
            return;
        }
        for (int u = threadIdx.x; u < BM * BC; u += WG) {
            const int r = u / BC, c = u % BC;
            if (r < rows && c < cols) p[r * ld + c] = *at(lds, r, c);
        }
    }
};

// FAST: 16-byte loads with bounds in the buffer, straight to LDS for the 16-bit types, by way of registers for f32 (its planes
// are made there).  Otherwise guarded loads of what width the rows allow.
template <int BM> constexpr int gated_depth() { return BM == 128 ? 1 : BM == 64 ? 2 : 4; }
constexpr int GATED_STAGES = 3;
template <class T, int BM> constexpr int gated_bufs() { return sizeof(T) == 4 && BM == 128 ? 1 : 2; }
template <class T, int BM, int BN, bool FAST, class NS, class MS, class NRow>
__device__ __forceinline__ void gated_gemm(char* lds, const NS& ns, const MS& ms, int kb, int ke, int mrow, NRow nrow,
                                           typename GemmTile<T, BM, BN, NS, MS>::Acc& acc) {
    using G = GemmTile<T, BM, BN, NS, MS>;
    if constexpr (FAST && sizeof(T) == 2) G::template by_dma<GATED_STAGES>(lds, ns, ms, kb, ke, mrow, nrow, acc);
    else G::template by_registers<gated_depth<BM>(), gated_bufs<T, BM>(), FAST>(lds, ns, ms, kb, ke, mrow, nrow, acc);
}
template <class T, int BM, int BN, bool FAST> constexpr int gated_lds(int behind) {
    const int g = (BM + BN) * 64 * Elem<T>::P * (FAST && sizeof(T) == 2 ? GATED_STAGES : gated_bufs<T, BM>());
    return g > behind ? g : behind;
}
template <class T, int BM> constexpr bool gated_rest() { return sizeof(T) == 2 && BM == 32; }  // instances that can write it
template <class T, int BM, int BN> constexpr int gated_behind(bool bwd) {
    return (bwd ? gated_rest<T, BM>() ? 4 : 2 : 1) * OutTile<T, BM, BN / 2, 64>::BYTES +
           (bwd ? gemm_waves(BM) * 2 * (BN / 2) * 4 : 0);
}

template <class T, int BM, int BN, bool FAST, bool BWD>
__global__ __launch_bounds__(gemm_wg(BM, BN), sizeof(T) == 4 ? 2 : BM > 128 ? 4 : 3) void gated_kernel(
    GatedDims d, int ftiles, int mtiles, const T* __restrict__ x, const T* __restrict__ wg, const T* __restrict__ wu,
    const T* __restrict__ bg, const T* __restrict__ bu, const T* __restrict__ dh, T* __restrict__ h, T* __restrict__ D,
    float* __restrict__ part, const GatedMax* __restrict__ maxes) {
    extern __shared__ __align__(16) char lds[];
    constexpr int WG = gemm_wg(BM, BN), WM = gemm_waves(BM), WN = gemm_waves(BN);
    constexpr int FT = BN / 2, TN = FT / WN / 16, TM = BM / WM / 16;  // columns a tile; gate (and up) subtiles, row subtiles of a wave
    using Out = OutTile<T, BM, FT, WG>;
    const TileAt at = tile_at(blockIdx.x, ftiles);
    if (at.lo >= mtiles) return;
    const int m0 = at.lo * BM, f0 = at.sh * FT;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wn = wave % WN, wm = wave / WN;
    const int nbase = wn * (FT / WN), mrow = wm * (BM / WM);
    const RowOperand<T, true> ns = {wg, wu, d.ldw, d.out, d.inw, f0, FT, f0, d.wvw};
    const RowOperand<T, false> ms = {x, x, d.ldx, d.rows, d.inw, m0, BM, 0, d.xvw};
    f32x4 acc[2 * TN][TM];
    const int r = lane & 15, c4 = (lane >> 4) * 4;
    Raw<T> dhr[BWD ? Out::U : 1];
    gated_gemm<T, BM, BN, FAST>(lds, ns, ms, 0, d.inw, mrow,
                               [&](int j) { return j < TN ? nbase + j * 16 : FT + nbase + (j - TN) * 16; }, acc);
    GatedMaxes<T> most;
    if constexpr (BWD) most.load(maxes);
    f32x4 vbg[TN], vbu[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const int f = f0 + nbase + j * 16 + c4, nf = d.out - f;
        const f32x4 zero = {0, 0, 0, 0};
        vbg[j] = bg != nullptr ? load4(bg + f, nf, d.bvec) : zero;
        vbu[j] = bu != nullptr ? load4(bu + f, nf, d.bvec) : zero;
    }
    char* second = lds + Out::BYTES;
    constexpr bool REST = BWD && gated_rest<T, BM>();
    float* red = reinterpret_cast<float*>(lds + (REST ? 4 : 2) * Out::BYTES);  // [WM][2][FT] column sums
    if constexpr (BWD) {
        Out::fetch(dhr, dh + (int64_t)m0 * d.lddh + f0, d.lddh, d.rows - m0, d.out - f0, d.dhvw);
        Out::keep(dhr, lds);
        __syncthreads();
    }
    const GatedScale scale = BWD ? most.scale() : GatedScale{1.f, 1.f};
    const bool whole = m0 + BM <= d.rows && f0 + FT <= d.out;
    // (a tile without edges needs no looks at them; swish has code of its own: with all kinds' in every place of the unrolled
    // loops the code outgrows its cache)
    auto epilogue = [&](auto kind) {
        constexpr int KIND = decltype(kind)::value;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int fl = nbase + j * 16 + c4, f = f0 + fl, nf = d.out - f;
            f32x4 sg = {0, 0, 0, 0}, su = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const int ml = mrow + i * 16 + r;
                const f32x4 g = acc[j][i] + vbg[j], u = acc[j + TN][i] + vbu[j];
                T* o = Out::at(lds, ml, fl);
                if constexpr (!BWD) {
                    f32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = act_value<KIND>(d.kind, g[e]) * u[e];
                    store4(o, v, 4, true);
                } else {  // dh's place takes dg; columns and rows outside hold zeros, whatever g and u are there
                    const f32x4 v = load4(o, 4, true);
                    f32x4 og, ou;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        ou[e] = v[e] * act_value<KIND>(d.kind, g[e]);
                        og[e] = v[e] * u[e] * act_slope<KIND>(d.kind, g[e]);
                    }
                    if (!whole) {
                        const bool real = m0 + ml < d.rows;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            ou[e] = real && e < nf ? ou[e] : 0.f;
                            og[e] = real && e < nf ? og[e] : 0.f;
                        }
                    }
                    sg += og;
                    su += ou;
                    if constexpr (gated_scaled<T>()) {
                        og *= scale.by;
                        ou *= scale.by;
                    }
                    store4(o, og, 4, true);
                    store4(Out::at(second, ml, fl), ou, 4, true);
                    if constexpr (REST) {
                        f32x4 rg, ru;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            rg[e] = og[e] - to_f((T)og[e]);
                            ru[e] = ou[e] - to_f((T)ou[e]);
                        }
                        store4(Out::at(second + Out::BYTES, ml, fl), rg, 4, true);
                        store4(Out::at(second + 2 * Out::BYTES, ml, fl), ru, 4, true);
                    }
                }
            }
            if constexpr (BWD) {
                if (part != nullptr) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float a = over_16(sg[e]), b = over_16(su[e]);
                        if (r == 0) {
                            red[(wm * 2) * FT + fl + e] = a;
                            red[(wm * 2 + 1) * FT + fl + e] = b;
                        }
                    }
                }
            }
        }
    };
    if (d.kind == 0) epilogue(std::integral_constant<int, 0>());
    else epilogue(std::integral_constant<int, -1>());
    __syncthreads();
    if constexpr (!BWD) {
        Out::write(lds, h + (int64_t)m0 * d.out + f0, d.out, d.rows - m0, d.out - f0, d.hvw);
    } else {
        const int64_t ldd = (int64_t)d.planes * 2 * d.outp;
        T* o = D + m0 * ldd + f0;
        Out::write(lds, o, ldd, d.rows - m0, d.outp - f0, 8);
        Out::write(second, o + d.outp, ldd, d.rows - m0, d.outp - f0, 8);
        if (REST && d.planes == 2) {
            Out::write(second + Out::BYTES, o + 2 * d.outp, ldd, d.rows - m0, d.outp - f0, 8);
            Out::write(second + 2 * Out::BYTES, o + 3 * d.outp, ldd, d.rows - m0, d.outp - f0, 8);
        }
        if (part == nullptr) return;
        for (int t = threadIdx.x; t < 2 * FT; t += WG) {
            const int f = f0 + t % FT;
            float s = red[t];
#pragma unroll
            for (int w = 1; w < WM; ++w) s += red[2 * FT * w + t];
            if (f < d.outp) part[(int64_t)at.lo * 2 * d.outp + (t / FT) * d.outp + f] = s;
        }
    }
}

template <class T, int NJ, int MI>
__device__ __forceinline__ void gated_undo(f32x4 (&acc)[NJ][MI], const GatedMax* __restrict__ maxes) {
    if constexpr (gated_scaled<T>()) {
        GatedMaxes<T> most;
        most.load(maxes);
        const GatedScale scale = most.scale();
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int i = 0; i < MI; ++i) acc[j][i] *= scale.undo;
    }
}

// dx[m][k] = sum over f < 2 outp of D[m][f] [Wg; Wu][f][k]; several shares of f (blockIdx.y): their sums in fp32 to part
template <class T, int BM, int BN, bool FAST>
__global__ __launch_bounds__(gemm_wg(BM, BN)) void gated_dx_kernel(GatedDims d, int ktiles, int mtiles, const T* __restrict__ D,
                                                           const T* __restrict__ wg, const T* __restrict__ wu,
                                                           T* __restrict__ dx, int share, float* __restrict__ part,
                                                           const GatedMax* __restrict__ maxes) {
    extern __shared__ __align__(16) char lds[];
    using Out = OutTile<T, BM, BN, gemm_wg(BM, BN)>;
    const TileAt at = tile_at(blockIdx.x, ktiles);
    if (at.lo >= mtiles) return;
    const int m0 = at.lo * BM, k0 = at.sh * BN;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    constexpr int WM = gemm_waves(BM), WN = gemm_waves(BN), MI = BM / WM / 16, NJ = BN / WN / 16;
    const int nbase = wave % WN * (BN / WN), mrow = wave / WN * (BM / WM);
    const int width = d.planes * 2 * d.outp;  // of D
    const ColOperand<T> ns = {wg, wu, d.ldw, d.inw, d.out, k0, d.outp, 2 * d.outp, d.wvw};
    const RowOperand<T, false> ms = {D, D, width, d.rows, width, m0, BM, 0, 8};
    f32x4 acc[NJ][MI];
    const int fb = blockIdx.y * share, fe = fb + share < width ? fb + share : width;
    gated_gemm<T, BM, BN, FAST>(lds, ns, ms, fb, fe, mrow, [&](int j) { return nbase + j * 16; }, acc);
    gated_undo<T, NJ, MI>(acc, maxes);
    const int r = lane & 15, c4 = (lane >> 4) * 4;
    if (gridDim.y > 1) {
        float* o = part + (int64_t)blockIdx.y * d.rows * d.in;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                const int m = m0 + mrow + i * 16 + r, k = k0 + nbase + j * 16 + c4;
                if (m < d.rows) store4(o + (int64_t)m * d.in + k, acc[j][i], d.in - k, d.in % 4 == 0);
            }
        return;
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < MI; ++i) store4(Out::at(lds, mrow + i * 16 + r, nbase + j * 16 + c4), acc[j][i], 4, true);
    __syncthreads();
    Out::write(lds, dx + (int64_t)m0 * d.in + k0, d.in, d.rows - m0, d.in - k0, d.dxvw);
}

// From part to part of dW, floats: powers of two apart, a place's parts would all lie on the same memory channels (their sum,
// 32 parts of 2048 x 256: 21 us, with these 4 KB between them 14)
__host__ __device__ constexpr int64_t gated_part(int outp, int in) { return (int64_t)2 * outp * in + 1088; }

// part[s][f][k] = sum over the rows of split s of D[m][f] x[m][k]
template <class T, int BM, int BN, bool FAST>
__global__ __launch_bounds__(gemm_wg(BM, BN)) void gated_dw_kernel(GatedDims d, int ktiles, int rows_a_split, const T* __restrict__ D,
                                                           const T* __restrict__ x, float* __restrict__ part,
                                                           const GatedMax* __restrict__ maxes) {
    extern __shared__ __align__(16) char lds[];
    const int k0 = (blockIdx.x % ktiles) * BN, f0 = (blockIdx.x / ktiles) * BM;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    constexpr int WM = gemm_waves(BM), WN = gemm_waves(BN), MI = BM / WM / 16, NJ = BN / WN / 16;
    const int nbase = wave % WN * (BN / WN), mrow = wave / WN * (BM / WM);
    const int64_t rb = (int64_t)blockIdx.y * rows_a_split;
    const int n = (int)(d.rows - rb < rows_a_split ? d.rows - rb : rows_a_split);
    // the rows of both halves of D, one behind the other, and x's rows twice
    const int width = d.planes * 2 * d.outp, half = d.planes == 2 ? (n + 7) / 8 * 8 : 1 << 30;
    const T *xb = x + rb * d.ldx, *db = D + rb * width;
    const ColOperand<T> ns = {xb, xb, d.ldx, d.inw, n, k0, half, 1 << 30, d.xvw};
    const ColOperand<T> ms = {db, db + 2 * d.outp, width, 2 * d.outp, n, f0, half, 1 << 30, 8};
    f32x4 acc[NJ][MI];
    gated_gemm<T, BM, BN, FAST>(lds, ns, ms, 0, d.planes == 2 ? half + n : n, mrow, [&](int j) { return nbase + j * 16; },
                                acc);
    gated_undo<T, NJ, MI>(acc, maxes);
    const int r = lane & 15, c4 = (lane >> 4) * 4;
    float* o = part + blockIdx.y * gated_part(d.outp, d.in);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int f = f0 + mrow + i * 16 + r, k = k0 + nbase + j * 16 + c4;
            if (f < 2 * d.outp) store4(o + (int64_t)f * d.in + k, acc[j][i], d.in - k, d.in % 4 == 0);
        }
}

// x and the weights with rows of `inw` values, zeros behind the first `in`: a thread a chunk of 8
template <class T>
__global__ __launch_bounds__(256) void gated_pack_kernel(GatedDims d, const T* __restrict__ x, const T* __restrict__ wg,
                                                         const T* __restrict__ wu, T* __restrict__ xp, T* __restrict__ wp) {
    const int chunks = d.inw / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / chunks;
    const int c = (int)(i % chunks) * 8, n = d.in - c;
    if (row >= d.rows + 2 * (int64_t)d.out) return;
    Raw<T> raw;
    if (row < d.rows) load_raw(raw, x + row * d.ldx + c, n > 8 ? 8 : n, d.xvw);
    else if (row < d.rows + (int64_t)d.out) load_raw(raw, wg + (row - d.rows) * d.in + c, n > 8 ? 8 : n, d.wvw);
    else load_raw(raw, wu + (row - d.rows - d.out) * d.in + c, n > 8 ? 8 : n, d.wvw);
    T* to = row < d.rows ? xp + row * d.inw + c : wp + (row - d.rows) * d.inw + c;
    __builtin_memcpy(__builtin_assume_aligned(to, 16), &raw, sizeof(raw));
}

// What GatedMaxes reads: of each workgroup's share the largest norm of a row of x or the weights, the largest |bias| or |dh|.  A
// pass over them, by memory (65536 x 256 -> 2 x 1024, 169 MB: 42 us; 5003 x 204 -> 2 x 530, with the copies: 10 us): 16 waves, four
// loads a lane under way.
struct GatedScan {  // an array of one kind
    const f16* p;
    int64_t rows, ld, cols;  // (biases and dh: where rows follow each other they are one)
    f16* copy;               // what gated_pack_kernel writes, on the way (or null)
    int64_t share;           // rows (biases and dh: chunks of 8 values) a workgroup
    int vw, last;            // the last of its workgroups + 1
};
enum { SCAN_X, SCAN_WG, SCAN_WU, SCAN_BG, SCAN_BU, SCAN_DH, SCANS };
struct GatedScans {
    GatedScan s[SCANS];
};
__device__ __forceinline__ bool gated_has_norms(int k) { return k <= SCAN_WU; }
// rows at .. end - 1: G lanes a row, four rows of a group at once
__device__ __forceinline__ unsigned short gated_norms(const GatedScan& s, int64_t at, int64_t end) {
    const int chunks = (int)((s.cols + 7) / 8);
    int G = 1;
    while (G < chunks && G < 64) G *= 2;
    const int64_t groups = GATED_MAX_WG / G;
    float top = 0.f;
    for (int64_t row = at + threadIdx.x / G; row < end; row += 4 * groups) {  // (the same in all lanes of a group)
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        for (int c = threadIdx.x % G; c < chunks; c += G) {
            const int n = (int)s.cols - c * 8;
            Raw<f16> raw[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t r = row + u * groups;
                load_raw(raw[u], s.p + (r < end ? r * s.ld + c * 8 : 0), r >= end ? 0 : n > 8 ? 8 : n, s.vw);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t r = row + u * groups;
                if (s.copy != nullptr && r < end) *reinterpret_cast<u32x4*>(s.copy + (r * chunks + c) * 8) = raw[u].a;
                const f16x8 v = __builtin_bit_cast(f16x8, raw[u].a);
#pragma unroll
                for (int j = 0; j < 8; ++j) sum[u] += (float)v[j] * (float)v[j];
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            for (int k = 1; k < G; k *= 2) sum[u] += __shfl_xor(sum[u], k, 64);
            top = sum[u] < INFINITY && sum[u] > top ? sum[u] : top;
        }
    }
    // (past the bf16 below it, by one or two of its steps)
    return top > 0.f ? (unsigned short)((__builtin_bit_cast(uint32_t, sqrtf(top)) >> 16) + 1) : 0;
}
// chunks at .. end - 1
__device__ __forceinline__ unsigned short gated_largest(const GatedScan& s, int64_t at, int64_t end) {
    const int64_t chunks = (s.cols + 7) / 8, dr = GATED_MAX_WG / chunks, dc = GATED_MAX_WG % chunks;
    int64_t i = at + threadIdx.x, row = i / chunks, c = i % chunks;
    u16x2 m = {0, 0};
    while (i < end) {
        Raw<f16> raw[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t n = i < end ? s.cols - c * 8 : 0;
            load_raw(raw[u], s.p + (n > 0 ? row * s.ld + c * 8 : 0), n > 8 ? 8 : (int)n, n < 8 ? 1 : s.vw);  // (a whole array's end)
            i += GATED_MAX_WG;
            row += dr;
            c += dc;
            if (c >= chunks) {
                c -= chunks;
                ++row;
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            u16x2 w[4], t = {0, 0};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j] = __builtin_bit_cast(u16x2, (uint32_t)raw[u].a[j] & 0x7fff7fffu);
                t = larger(t, w[j]);
            }
            if (t[0] >= 0x7c00 || t[1] >= 0x7c00) {  // infinities and NaN are left out
                t = u16x2{0, 0};
                for (int j = 0; j < 4; ++j)
                    for (int h = 0; h < 2; ++h)
                        if (w[j][h] < 0x7c00 && w[j][h] > t[0]) t[0] = w[j][h];
            }
            m = larger(m, t);
        }
    }
    return m[0] > m[1] ? m[0] : m[1];
}
__global__ __launch_bounds__(GATED_MAX_WG) void gated_max_kernel(GatedScans all, GatedMax* __restrict__ maxes) {
    int k = 0, first = 0;
    for (; k < SCANS - 1 && (int)blockIdx.x >= all.s[k].last; ++k) first = all.s[k].last;
    const GatedScan s = all.s[k];
    const int64_t total = gated_has_norms(k) ? s.rows : s.rows * ((s.cols + 7) / 8);
    const int64_t at = ((int)blockIdx.x - first) * s.share, end = at + s.share < total ? at + s.share : total;
    const unsigned short mine = gated_has_norms(k) ? gated_norms(s, at, end) : gated_largest(s, at, end);
    __shared__ unsigned short red[GATED_MAX_WG / 64];
    const u16x2 m = largest_of_wave(u16x2{mine, 0});
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m[0];
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned short v = 0;
        for (int w = 0; w < GATED_MAX_WG / 64; ++w) v = red[w] > v ? red[w] : v;
        const unsigned short none = 0;
        maxes[blockIdx.x] = {u16x2{k == SCAN_X ? v : none, k == SCAN_WG || k == SCAN_WU ? v : none},
                             u16x2{k == SCAN_BG || k == SCAN_BU ? v : none, k == SCAN_DH ? v : none}};
    }
    if (blockIdx.x == 0 && gridDim.x + threadIdx.x < GATED_MAX_WGS) maxes[gridDim.x + threadIdx.x] = {};
}

// the parts of dx (workgroups below xblocks), of dW (wblocks more) and of the column sums, added in order
template <class T>
__global__ __launch_bounds__(256) void gated_reduce_kernel(GatedDims d, int xblocks, int xsplits, const float* __restrict__ xpart,
                                                           T* __restrict__ dx, int wblocks, int splits, int mtiles,
                                                           const float* __restrict__ wpart, const float* __restrict__ bpart,
                                                           T* __restrict__ dwg, T* __restrict__ dwu, T* __restrict__ dbg,
                                                           T* __restrict__ dbu) {
    int b = blockIdx.x;
    if (b < xblocks) {
        const int64_t size = (int64_t)d.rows * d.in, i = (int64_t)b * 256 + threadIdx.x;
        if (i >= size) return;
        float s = 0.f;
#pragma unroll 8
        for (int p = 0; p < xsplits; ++p) s += xpart[p * size + i];
        dx[i] = (T)s;
        return;
    }
    b -= xblocks;
    __shared__ f32x4 red4[4][64];
    if (b < wblocks) {  // 256 places a workgroup, four a load, four threads share the parts (whole f32x4: size is a multiple of 8)
        const int lane = threadIdx.x & 63, q = threadIdx.x >> 6;
        const int64_t size = (int64_t)2 * d.outp * d.in, i = (int64_t)b * 256 + lane * 4;
        f32x4 s = {0, 0, 0, 0};
        if (i < size) {
#pragma unroll 8
            for (int p = q; p < splits; p += 4) s += *reinterpret_cast<const f32x4*>(wpart + p * gated_part(d.outp, d.in) + i);
        }
        red4[q][lane] = s;
        __syncthreads();
        const int64_t at = (int64_t)b * 256 + threadIdx.x;
        if (at >= size) return;
        const int f = (int)(at / d.in), k = (int)(at % d.in), half = f >= d.outp, ff = f - half * d.outp;
        const int l = threadIdx.x >> 2, e = threadIdx.x & 3;
        T* o = half ? dwu : dwg;
        if (ff < d.out && o != nullptr) o[(int64_t)ff * d.in + k] = (T)(red4[0][l][e] + red4[1][l][e] + red4[2][l][e] + red4[3][l][e]);
        return;
    }
    b -= wblocks;
    __shared__ float red[16][17];
    const int cx = threadIdx.x & 15, q = threadIdx.x >> 4, c = b * 16 + cx, W = 2 * d.outp;
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

// Tiles of an output.  A tile of 128 x 128 draws 16 KB from L2 for 16 instructions of each of its four waves, and that is what
// bounds the long products: 65536 x 256 -> 2 x 1024 in bf16, the same time with two, three or four tiles under way.  So the
// 16-bit types take 256 x 256 (dx 106 -> 83 us, dW 106 -> 91) or, where an epilogue wants a second workgroup on the CU,
// 256 x 128 (forward 127 -> 119; the backward's first launch 188 -> 180, with dh and the biases fetched behind the product:
// eight waves have no registers for them before), as long as their rounds over the chip and their edges leave little idle.
// Else 128 x 128 where they fill the 256 CUs, else 64 x 64, else 32 x 64; guarded loads: 32 x 64.
enum { TILE_256, TILE_TALL, TILE_128, TILE_64, TILE_32, TILE_GUARDED };
static const int TILE_M[6] = {256, 256, 128, 64, 32, 32}, TILE_N[6] = {256, 128, 128, 64, 64, 64};
static int div_up(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }
static int64_t gated_tiles(int64_t m, int64_t n, int t) { return (int64_t)div_up(m, TILE_M[t]) * div_up(n, TILE_N[t]); }
static bool gated_fills(int64_t m, int64_t n, int t, int64_t times) {
    const int64_t tiles = gated_tiles(m, n, t), slots = t == TILE_256 ? 256 : 512, wgs = tiles * times;
    if (t > TILE_TALL) return wgs >= 256;
    return 5 * wgs >= 4 * slots * div_up(wgs, slots) && 4 * tiles * TILE_M[t] * TILE_N[t] <= 5 * m * n;
}
#define GATED_BY_TILE(tile, BM, BN, ...)                                               \
    switch (tile) {                                                                    \
        case TILE_256:                                                                 \
            if constexpr (sizeof(T) == 2) { constexpr int BM = 256, BN = 256; __VA_ARGS__; } break; \
        case TILE_TALL:                                                                \
            if constexpr (sizeof(T) == 2) { constexpr int BM = 256, BN = 128; __VA_ARGS__; } break; \
        case TILE_128: { constexpr int BM = 128, BN = 128; __VA_ARGS__; } break;       \
        case TILE_64: { constexpr int BM = 64, BN = 64; __VA_ARGS__; } break;          \
        case TILE_32: { constexpr int BM = 32, BN = 64; __VA_ARGS__; } break;          \
        default: break;                                                                \
    }

struct GatedScratch {  // bytes from the start
    size_t pack, D, bpart, wpart, xpart, maxes, total;
    int tile, mtiles;                  // of the first launch, whose row tiles have a row of column sums each
    int wtile, splits, rows_a_split;   // of dW (TILE_256 of 16 bits, TILE_128, TILE_64, TILE_GUARDED)
    int xtile, xsplits, share;         // of dx
    int planes;                        // of D
};
// Rows that no 16-byte load fits are copied to rows that it does where the products are long enough to pay for the launch;
// below, their tiles come in by narrower, guarded loads (2066 rows of 965 -> 1292 f16, forward and backward: 572 us by guarded
// loads, 197 with the copies).
static bool gated_packed(int rows, int in, int out) { return (int64_t)rows * in * out >= (1 << 22); }
static GatedScratch gated_scratch(int dtype, int rows, int in, int out, bool fast, bool bwd) {
    GatedScratch s = {};
    const size_t outp = ((size_t)out + 7) / 8 * 8, inp = ((size_t)in + 7) / 8 * 8, es = dtype == TSD_F32 ? 4 : 2;
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const bool guarded = !fast && !gated_packed(rows, in, out);
    const int first = guarded ? TILE_GUARDED : es == 4 ? TILE_128 : TILE_TALL;
    for (s.tile = first; s.tile < TILE_32 && !gated_fills(rows, 2 * outp, s.tile, 1);) ++s.tile;
    s.mtiles = div_up(rows, TILE_M[s.tile]);
    s.planes = es == 2 && s.tile >= TILE_32 && (int64_t)rows * 2 * outp <= (1 << 18) ? 2 : 1;
    const size_t width = s.planes * 2 * outp;
    // dW: the rows in shares: one workgroup a CU of the largest tiles, 1024 rows each at least; else about two, of at least 256
    // rows.  The large tiles save time a row and cost more parts to add, 4 us.  bf16, launch and sum of the parts in us, at
    // 512 / 768 / 1024 / 1536 / 2048 rows a share:
    //   256 -> 2 x 1024: 256 x 256 44 / 54 / 62 / 83 / 106, 128 x 128 39 / 52 / 64 / 88 / 115
    //   512 -> 2 x 512:  43 / 52 / 62 / 82 / 101, 39 / 51 / 64 / 90 / 121
    //   1024 -> 2 x 2048: 47 / 53 / 62 / 74 / 90, 42 / 52 / 61 / 81 / 101
    const int most = div_up(rows, 256), large = guarded ? TILE_GUARDED : es == 4 ? TILE_128 : TILE_256;
    int n = 0;
    for (s.wtile = large;; s.wtile += s.wtile == TILE_256 ? 2 : 1) {
        const int64_t tiles = gated_tiles(2 * outp, in, s.wtile);
        n = s.wtile == TILE_256 ? (int)(256 / tiles) : (int)((511 + tiles) / tiles);
        n = n < most ? n : most;
        n = n < 1 ? 1 : n;
        if (s.wtile == TILE_GUARDED || s.wtile == TILE_64) break;
        if (s.wtile == TILE_256 ? gated_fills(2 * outp, in, s.wtile, n) && rows / n >= 1024
                                : gated_fills(2 * outp, in, s.wtile, most))
            break;
    }
    s.rows_a_split = div_up(div_up(rows > 0 ? rows : 1, n), GEMM_K) * GEMM_K;
    s.splits = div_up(rows, s.rows_a_split);
    // dx: the largest tiles that fill the chip; where fewer than 128 of them are to do, with shares of at least eight steps of
    // the contraction (16300 x 250 -> 2 x 600, 256 tiles: in two shares 33 + 16 us with the sum of the parts, in one 25 + 7;
    // 10000 x 256 -> 2 x 512: 15 + 14 us, 64 x 64 tiles without shares 16 + 7)
    const int steps = div_up(width, GEMM_K);
    for (s.xtile = large;; ++s.xtile) {
        const int64_t t = gated_tiles(rows, in, s.xtile);
        int x = t >= 128 || s.xtile <= TILE_TALL ? 1 : (int)(512 / (t > 0 ? t : 1));
        x = x < steps / 8 ? x : steps / 8;
        x = x < 1 ? 1 : x;
        s.share = div_up(steps, x) * GEMM_K;
        s.xsplits = div_up(width, s.share);
        if (s.xtile >= TILE_32 || gated_fills(rows, in, s.xtile, s.xsplits)) break;
    }
    s.pack = 0;
    s.D = up(!fast && gated_packed(rows, in, out) ? ((size_t)rows + 2 * (size_t)out) * inp * es : 0);
    if (!bwd) {
        s.total = s.D;
        return s;
    }
    s.bpart = s.D + up((size_t)rows * width * es);
    s.wpart = s.bpart + up((size_t)s.mtiles * 2 * outp * 4);
    s.xpart = s.wpart + up((size_t)s.splits * (size_t)gated_part((int)outp, in) * 4);
    s.maxes = s.xpart + (s.xsplits > 1 ? up((size_t)s.xsplits * rows * in * 4) : 0);
    s.total = s.maxes + (dtype == TSD_F16 ? up(GATED_MAX_WGS * sizeof(GatedMax)) : 0);
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
                            const void* bg, const void* bu) {
    GatedDims d = {};
    d.rows = rows;
    d.in = in;
    d.out = out;
    d.outp = (out + 7) / 8 * 8;
    d.ldx = ldx;
    d.planes = 1;
    d.inw = in;
    d.ldw = in;
    d.kind = act;
    d.xvw = load_width(sizeof(T), in, ldx, x);
    const int a = load_width(sizeof(T), in, in, wg), b = load_width(sizeof(T), in, in, wu);
    d.wvw = a < b ? a : b;
    d.bvec = aligned16(bg) && aligned16(bu);
    return d;
}
// 16-byte loads everywhere, and a tile's rows within the 2 GiB that a buffer's offsets reach
static bool gated_fast(const GatedDims& d) { return d.xvw == 8 && d.wvw == 8 && d.ldx <= (1 << 21); }

// Where the copies in scratch lie; null: there are none
template <class T> static T* gated_copies(const GatedDims& d, char* scratch) {
    return gated_fast(d) || !gated_packed(d.rows, d.in, d.out) ? nullptr : reinterpret_cast<T*>(scratch);
}
// x, wg and wu become the copies
template <class T> static void gated_use_copies(GatedDims& d, const void*& x, const void*& wg, const void*& wu, T* xp) {
    d.inw = (d.in + 7) / 8 * 8;
    T* wp = xp + (int64_t)d.rows * d.inw;
    x = xp;
    wg = wp;
    wu = wp + (int64_t)d.out * d.inw;
    d.ldx = d.ldw = d.inw;
    d.xvw = d.wvw = 8;
}
template <class T>
static int gated_pack(GatedDims& d, const void*& x, const void*& wg, const void*& wu, char* scratch, hipStream_t st) {
    T* xp = gated_copies<T>(d, scratch);
    if (xp == nullptr) return TSD_OK;
    d.inw = (d.in + 7) / 8 * 8;
    const int64_t chunks = ((int64_t)d.rows + 2 * (int64_t)d.out) * (d.inw / 8);
    hipLaunchKernelGGL(gated_pack_kernel<T>, dim3((unsigned)((chunks + 255) / 256)), dim3(256), 0, st, d, (const T*)x,
                       (const T*)wg, (const T*)wu, xp, xp + (int64_t)d.rows * d.inw);
    TSD_LAUNCH_CHECK("gated_pack");
    gated_use_copies(d, x, wg, wu, xp);
    return TSD_OK;
}

template <class T, int BM, int BN, bool FAST, bool BWD>
static int gated_first(GatedDims d, const void* x, const void* wg, const void* wu, const void* bg, const void* bu, const void* dh,
                       void* h, void* D, float* part, const GatedMax* maxes, hipStream_t st) {
    static DeviceOnce once;
    constexpr int lds = gated_lds<T, BM, BN, FAST>(gated_behind<T, BM, BN>(BWD));
    auto k = gated_kernel<T, BM, BN, FAST, BWD>;
    const int rc = allow_lds(k, lds, once);
    if (rc != TSD_OK) return rc;
    const int ft = div_up(BWD ? d.outp : d.out, BN / 2), mt = div_up(d.rows, BM);
    hipLaunchKernelGGL(k, dim3(tile_grid(mt, ft)), dim3(gemm_wg(BM, BN)), lds, st, d, ft, mt, (const T*)x, (const T*)wg, (const T*)wu,
                       (const T*)bg, (const T*)bu, (const T*)dh, (T*)h, (T*)D, part, maxes);
    TSD_LAUNCH_CHECK("gated_linear");
    return TSD_OK;
}
template <class T, int BM, int BN, bool FAST>
static int gated_dx(GatedDims d, const GatedScratch& s, const T* D, const void* wg, const void* wu, void* dx, float* part,
                    const GatedMax* maxes, hipStream_t st) {
    static DeviceOnce once;
    constexpr int lds = gated_lds<T, BM, BN, FAST>(OutTile<T, BM, BN, 64>::BYTES);
    auto k = gated_dx_kernel<T, BM, BN, FAST>;
    const int rc = allow_lds(k, lds, once);
    if (rc != TSD_OK) return rc;
    const int kt = div_up(d.in, BN), mt = div_up(d.rows, BM);
    hipLaunchKernelGGL(k, dim3(tile_grid(mt, kt), s.xsplits), dim3(gemm_wg(BM, BN)), lds, st, d, kt, mt, D, (const T*)wg,
                       (const T*)wu, (T*)dx, s.share, part, maxes);
    TSD_LAUNCH_CHECK("gated_dx");
    return TSD_OK;
}
template <class T, int BM, int BN, bool FAST>
static int gated_dw(GatedDims d, const GatedScratch& s, const T* D, const void* x, float* wpart, const GatedMax* maxes,
                    hipStream_t st) {
    static DeviceOnce once;
    constexpr int lds = gated_lds<T, BM, BN, FAST>(0);
    auto k = gated_dw_kernel<T, BM, BN, FAST>;
    const int rc = allow_lds(k, lds, once);
    if (rc != TSD_OK) return rc;
    const int kt = div_up(d.in, BN), ft = div_up(2 * d.outp, BM);
    hipLaunchKernelGGL(k, dim3(kt * ft, s.splits), dim3(gemm_wg(BM, BN)), lds, st, d, kt, s.rows_a_split, D, (const T*)x, wpart,
                       maxes);
    TSD_LAUNCH_CHECK("gated_dw");
    return TSD_OK;
}
// The list of the largest values, one launch, with the copies of gated_pack where xp is not null: at most 250 shares of all
// chunks, and one more for each array
static int gated_maxes(const GatedDims& d, const void* x, const void* wg, const void* wu, const void* bg, const void* bu, const void* dh,
                       f16* xp, f16* wp, GatedMax* maxes, hipStream_t st) {
    const int64_t rows = d.rows, in = d.in, out = d.out, inw = (in + 7) / 8 * 8;
    f16* wp2 = wp != nullptr ? wp + out * inw : nullptr;
    GatedScans all = {{{(const f16*)x, rows, d.ldx, in, xp, 0, d.xvw, 0},
                       {(const f16*)wg, out, in, in, wp, 0, d.wvw, 0},
                       {(const f16*)wu, out, in, in, wp2, 0, d.wvw, 0},
                       {(const f16*)bg, bg != nullptr ? 1 : 0, out, out, nullptr, 0, 1, 0},
                       {(const f16*)bu, bu != nullptr ? 1 : 0, out, out, nullptr, 0, 1, 0},
                       {(const f16*)dh, rows, d.lddh, out, nullptr, 0, d.dhvw, 0}}};
    int64_t chunks = 0;
    for (int k = 0; k < SCANS; ++k) {
        GatedScan& s = all.s[k];
        if (k > SCAN_WU && s.ld == s.cols) {
            s.cols *= s.rows;
            s.rows = s.cols > 0 ? 1 : 0;
            s.vw = load_width(sizeof(f16), 8, 8, s.p);
        }
        chunks += s.rows * ((s.cols + 7) / 8);
    }
    const int64_t share = chunks / 250 + 1 < 4096 ? 4096 : chunks / 250 + 1;
    int wgs = 0;
    for (int k = 0; k < SCANS; ++k) {
        GatedScan& s = all.s[k];
        const int64_t c = (s.cols + 7) / 8, parts = s.rows > 0 ? div_up(s.rows * c, share) : 0;
        s.share = k > SCAN_WU ? share : parts > 0 ? div_up(s.rows, parts) : 0;
        wgs += (int)parts;
        s.last = wgs;
    }
    hipLaunchKernelGGL(gated_max_kernel, dim3(wgs), dim3(GATED_MAX_WG), 0, st, all, maxes);
    TSD_LAUNCH_CHECK("gated_max");
    return TSD_OK;
}
template <class T, bool BWD, class... A> static int gated_first_by(int tile, const GatedDims& d, A... a) {
    GATED_BY_TILE(tile, BM, BN, {
        if constexpr (BN <= 128) return gated_first<T, BM, BN, true, BWD>(d, a...);
    });
    return gated_first<T, 32, 64, false, BWD>(d, a...);
}

template <class T>
static int gated_bwd(GatedDims d, const void* x, const void* wg, const void* wu, const void* bg, const void* bu,
                     const void* dh, int64_t lddh, void* dx, void* dwg, void* dwu, void* dbg, void* dbu,
                     const GatedScratch& s, char* scratch, hipStream_t st) {
    T* D = reinterpret_cast<T*>(scratch + s.D);
    float* bpart = reinterpret_cast<float*>(scratch + s.bpart);
    float* wpart = reinterpret_cast<float*>(scratch + s.wpart);
    float* xpart = reinterpret_cast<float*>(scratch + s.xpart);
    GatedMax* maxes = reinterpret_cast<GatedMax*>(scratch + s.maxes);
    const bool sums = dbg != nullptr || dbu != nullptr, weights = dwg != nullptr || dwu != nullptr;
    int rc = TSD_OK;
    d.planes = s.planes;
    if (d.rows > 0) {
        d.lddh = lddh;
        d.dhvw = load_width(sizeof(T), d.out, lddh, dh);
        d.dxvw = load_width(sizeof(T), d.in, d.in, dx);
        if constexpr (gated_scaled<T>()) {
            T* xp = gated_copies<T>(d, scratch + s.pack);
            rc = gated_maxes(d, x, wg, wu, bg, bu, dh, xp, xp != nullptr ? xp + d.rows * (((int64_t)d.in + 7) / 8 * 8) : nullptr, maxes, st);
            if (xp != nullptr) gated_use_copies(d, x, wg, wu, xp);
        } else {
            rc = gated_pack<T>(d, x, wg, wu, scratch + s.pack, st);
        }
        if (rc != TSD_OK) return rc;
        rc = gated_first_by<T, true>(s.tile, d, x, wg, wu, bg, bu, dh, (void*)nullptr, (void*)D, sums ? bpart : (float*)nullptr,
                                     (const GatedMax*)maxes, st);
        if (rc == TSD_OK && dx != nullptr) {
            GATED_BY_TILE(s.xtile, BM, BN, { rc = gated_dx<T, BM, BN, true>(d, s, D, wg, wu, dx, xpart, maxes, st); });
            if (s.xtile == TILE_GUARDED) rc = gated_dx<T, 32, 64, false>(d, s, D, wg, wu, dx, xpart, maxes, st);
        }
        if (rc == TSD_OK && weights) {
            if (s.wtile == TILE_GUARDED) rc = gated_dw<T, 32, 64, false>(d, s, D, x, wpart, maxes, st);
            else if (s.wtile == TILE_64) rc = gated_dw<T, 64, 64, true>(d, s, D, x, wpart, maxes, st);
            else if (s.wtile == TILE_128) rc = gated_dw<T, 128, 128, true>(d, s, D, x, wpart, maxes, st);
            else if constexpr (sizeof(T) == 2) rc = gated_dw<T, 256, 256, true>(d, s, D, x, wpart, maxes, st);
        }
    }
    const bool parts = d.rows > 0 && dx != nullptr && s.xsplits > 1;
    if (rc == TSD_OK && (weights || sums || parts)) {
        const int xb = parts ? (int)(((int64_t)d.rows * d.in + 255) / 256) : 0;
        const int wb = weights ? (int)(((int64_t)2 * d.outp * d.in + 255) / 256) : 0, bb = sums ? (2 * d.outp + 15) / 16 : 0;
        hipLaunchKernelGGL(gated_reduce_kernel<T>, dim3(xb + wb + bb), dim3(256), 0, st, d, xb, s.xsplits, xpart, (T*)dx, wb, s.splits,
                           s.mtiles, wpart, bpart, (T*)dwg, (T*)dwu, (T*)dbg, (T*)dbu);
        TSD_LAUNCH_CHECK("gated_reduce");
    }
    return rc;
}

}  // namespace blk
}  // namespace tsd

using namespace tsd;
using namespace tsd::blk;

extern "C" {

size_t tsd_gated_linear_scratch_floats(int32_t dtype, int32_t rows, int32_t in, int32_t out, const void* x, int64_t ldx,
                                       const void* w_gate, const void* w_up, int32_t backward) {
    if (rows < 1 || in < 1 || out < 1) return 0;
    TSD_BY_DTYPE(dtype, T, {
        const GatedDims d = gated_dims<T>(rows, in, out, 0, x, ldx, w_gate, w_up, nullptr, nullptr);
        return gated_scratch(dtype, rows, in, out, gated_fast(d), backward != 0).total / 4;
    });
    return 0;
}

int tsd_gated_linear_fwd(int32_t dtype, int32_t act, int32_t rows, int32_t in, int32_t out, const void* x, int64_t ldx,
                         const void* w_gate, const void* w_up, const void* b_gate, const void* b_up, void* h, float* scratch,
                         size_t scratch_floats, void* stream) {
    int rc = gated_check("tsd_gated_linear_fwd", dtype, act, rows, in, out, ldx, x, w_gate, w_up);
    if (rc != TSD_OK) return rc;
    if (rows == 0) return TSD_OK;
    TSD_REQUIRE(h != nullptr, "tsd_gated_linear_fwd: null pointer");
    TSD_BY_DTYPE(dtype, T, {
        GatedDims d = gated_dims<T>(rows, in, out, act, x, ldx, w_gate, w_up, b_gate, b_up);
        const GatedScratch s = gated_scratch(dtype, rows, in, out, gated_fast(d), false);
        TSD_REQUIRE(s.total == 0 || (scratch != nullptr && aligned16(scratch) && scratch_floats * 4 >= s.total),
                    "tsd_gated_linear_fwd: scratch of %zu floats, %zu needed (16-byte aligned)", scratch_floats, s.total / 4);
        d.hvw = load_width(sizeof(T), out, out, h);
        if ((rc = gated_pack<T>(d, x, w_gate, w_up, (char*)scratch, (hipStream_t)stream)) != TSD_OK) return rc;
        return gated_first_by<T, false>(s.tile, d, x, w_gate, w_up, b_gate, b_up, (const void*)nullptr, h, (void*)nullptr,
                                        (float*)nullptr, (const GatedMax*)nullptr, (hipStream_t)stream);
    });
    return TSD_OK;
}

int tsd_gated_linear_bwd(int32_t dtype, int32_t act, int32_t rows, int32_t in, int32_t out, const void* x, int64_t ldx,
                         const void* w_gate, const void* w_up, const void* b_gate, const void* b_up, const void* dh,
                         int64_t lddh, void* dx, void* dw_gate, void* dw_up, void* db_gate, void* db_up, float* scratch,
                         size_t scratch_floats, void* stream) {
    const int rc = gated_check("tsd_gated_linear_bwd", dtype, act, rows, in, out, ldx, x, w_gate, w_up);
    if (rc != TSD_OK) return rc;
    TSD_REQUIRE(rows == 0 || (dh != nullptr && lddh >= out), "tsd_gated_linear_bwd: null pointer or row stride");
    TSD_BY_DTYPE(dtype, T, {
        const GatedDims d = gated_dims<T>(rows, in, out, act, x, ldx, w_gate, w_up, b_gate, b_up);
        const GatedScratch s = gated_scratch(dtype, rows, in, out, gated_fast(d), true);
        TSD_REQUIRE(rows == 0 || (scratch != nullptr && aligned16(scratch) && scratch_floats * 4 >= s.total),
                    "tsd_gated_linear_bwd: scratch of %zu floats, %zu needed (16-byte aligned)", scratch_floats, s.total / 4);
        return gated_bwd<T>(d, x, w_gate, w_up, b_gate, b_up, dh, lddh, dx, dw_gate, dw_up, db_gate, db_up, s, (char*)scratch,
                            (hipStream_t)stream);
    });
    return TSD_OK;
}

}  // extern "C"
