// kernels_attention.hip -- attention inside the graphs of a ragged batch, forward and backward.
//
//   S = scale Q K^T over the open keys of the row's graph, P = softmax S, O = P V, L = log2 sum exp2(S log2 e)
//   delta = sum_d dO O;  dP = dO V^T;  dS = P (dP - delta);  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
//
// One pass over the keys: the running maximum and sum of each row stay in registers and the scores never leave them.  The
// scores are computed turned, S^T = K Q^T, so that a lane holds one row's scores (their statistics are a lane's own, two
// shuffles join the four lanes of a row) AND the result registers are the operand of the next product as they stand: the
// contraction's order is free, so the keys of V are laid out in LDS in the order in which S^T leaves the matrix pipes.
// The backward computes the scores again from L: one launch over row tiles for dQ (and delta), one over key tiles for dK and
// dV; every gradient is summed by one workgroup in a fixed order, without atomics.
//
// Rows are (query, query head of the key head's group), so heads that share keys share their tiles.  Tiles never cross a
// graph: workgroup s looks its graph up, tile slot(v) = floor(start_v / T) + v being where graph v's tiles begin -- a bound
// on the tiles before it that needs no prefix sum and no lengths on the host, at most one idle workgroup a graph.  Offsets
// are clamped into the tensors.  Rows and keys outside of every graph count as graphs without keys / rows: they are written
// as zeros.  Masked and missing keys are zeros in LDS whatever memory holds there, so that no NaN meets a zero weight.
#include "block_tile.hpp"

namespace tsd {
namespace blk {

constexpr int ATT_KT = 64;  // keys (forward, dQ) a tile in LDS
constexpr float LOG2E = 1.44269504088896341f;

struct AttDims {
    int graphs, rows_q, rows_k, heads, kv_heads, group, dim;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, do_row, do_head;
    float scale, scale2;  // scale2 = scale * log2 e
    int splits;
    bool qvec, kvec, vvec, dovec, ovec;
    const int32_t *q_ptr, *k_ptr;
    const uint8_t* mask;
};

struct Span {
    int qs, qe, ks, ke;  // queries and keys of the graph
    int tile;            // which of its tiles
};
__device__ __forceinline__ int clamp_to(int v, int n) { return v < 0 ? 0 : v > n ? n : v; }
// boundary v of the list 0, ptr[0], .., ptr[G], n
__device__ __forceinline__ int bound_at(const int32_t* ptr, int graphs, int n, int v) {
    return v == 0 ? 0 : v > graphs + 1 ? n : clamp_to(ptr[v - 1], n);
}
// the graph whose tiles hold slot s (64 lanes look at a time); tiles of T rows, `times` rows an entry
__device__ __forceinline__ Span find_span(const AttDims& d, bool by_key, int T, int times, int s) {
    const int32_t* ptr = by_key ? d.k_ptr : d.q_ptr;
    const int n = by_key ? d.rows_k : d.rows_q, lane = threadIdx.x & 63;
    int lo = 0, count = d.graphs + 2;  // slot(lo) <= s, and the answer is below lo + count
    while (count > 1) {
        const int step = (count + 63) / 64, v = lo + lane * step;
        const bool in = lane * step < count && (int64_t)bound_at(ptr, d.graphs, n, v) * times / T + v <= s;
        const unsigned long long m = __ballot(in);
        const int last = 63 - __builtin_clzll(m | 1);
        lo += last * step;
        count = count - last * step < step ? count - last * step : step;
    }
    Span sp;
    const int start = bound_at(ptr, d.graphs, n, lo);
    sp.tile = s - (int)((int64_t)start * times / T) - lo;
    const bool real = lo >= 1 && lo <= d.graphs;
    const int end = bound_at(ptr, d.graphs, n, lo + 1);
    const int ostart = real ? bound_at(by_key ? d.q_ptr : d.k_ptr, d.graphs, by_key ? d.rows_q : d.rows_k, lo) : 0;
    const int oend = real ? bound_at(by_key ? d.q_ptr : d.k_ptr, d.graphs, by_key ? d.rows_q : d.rows_k, lo + 1) : 0;
    sp.qs = by_key ? ostart : start;
    sp.qe = by_key ? oend : end;
    sp.ks = by_key ? start : ostart;
    sp.ke = by_key ? end : oend;
    if (sp.qe < sp.qs) sp.qe = sp.qs;
    if (sp.ke < sp.ks) sp.ke = sp.ks;
    return sp;
}

// Values (row, d) of a graph's rows or keys
template <class T> struct Rows {
    const T* p;        // row 0 of the graph, this head (the first of the group)
    int64_t row, head; // strides
    int n, group, dim; // rows
    const uint8_t* mask;
    bool vec;
    __device__ __forceinline__ bool has(int r) const { return r < n && (mask == nullptr || mask[r] != 0); }
    __device__ __forceinline__ const T* at(int r) const {
        if (group == 1) return p + (int64_t)r * row;
        const int q = r / group;
        return p + (int64_t)q * row + (r - q * group) * head;
    }
};

// tile rows r0 .. r0 + ROWS as they lie: chunk c of row r
template <class T, int ROWS, int DP, int NT>
__device__ __forceinline__ void stage_rows(char* lds, const Rows<T>& s, int r0) {
    constexpr int C = DP / 8;
    for (int u = threadIdx.x; u < ROWS * C; u += NT) {
        const int r = u / C, c = u % C, n = s.dim - c * 8;
        Raw<T> raw;
        if (n > 0 && s.has(r0 + r)) load_raw(raw, s.at(r0 + r) + c * 8, n > 8 ? 8 : n, s.vec);
        else raw_zero(raw);
        Tile<T, ROWS, C>::put(lds, r, c, raw_chunk(raw));
    }
}
// The same values turned: row d, the tile's rows along it.  Chunk 4 b + g of a row holds rows 32 b + 4 g .. + 3 and
// 32 b + 16 + 4 g .. + 3: the order in which two neighbouring 16 x 16 results leave lane group g.
template <class T, int ROWS, int DP, int NT>
__device__ __forceinline__ void stage_cols(char* lds, const Rows<T>& s, int r0) {
    constexpr int W = ColRaw<T>::W, COLS = DP / W, C = ROWS / 8;
    for (int u = threadIdx.x; u < COLS * C; u += NT) {
        const int d = (u % COLS) * W, c = u / COLS, base = r0 + (c >> 2) * 32 + (c & 3) * 4;
        ColRaw<T> raw;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int r = base + (j & 3) + (j >> 2) * 16;
            raw.w[j] = 0;
            if (d < s.dim && s.has(r)) col_load(raw.w[j], s.at(r) + d, s.dim - d, s.vec);
        }
#pragma unroll
        for (int k = 0; k < W; ++k) Tile<T, DP, C>::put(lds, d + k, c, col_chunk<T>(raw, k));
    }
}
// one row's operand, kept in registers: chunk (lane / 16) of each 32 values
template <class T, int DP> __device__ __forceinline__ void row_chunks(Chunk<T> (&f)[DP / 32], const Rows<T>& s, int r) {
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) {
        const int d0 = b * 32 + g * 8, n = s.dim - d0;
        Raw<T> raw;
        if (n > 0 && s.has(r)) load_raw(raw, s.at(r) + d0, n > 8 ? 8 : n, s.vec);
        else raw_zero(raw);
        f[b] = raw_chunk(raw);
    }
}
// two 16 x 16 results of neighbouring subtiles as the operand of the next product
template <class T> __device__ __forceinline__ Chunk<T> joined(const f32x4& a, const f32x4& b) {
    const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return to_chunk(x, T());
}
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float over_groups_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float over_groups_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}
template <class T>
__device__ __forceinline__ Rows<T> rows_of(const T* p, int64_t row, int64_t head, int start, int n, int first_head, int group,
                                           int dim, const uint8_t* mask, bool vec) {
    return {p + (int64_t)start * row + (int64_t)first_head * head, row, head, n, group, dim,
            mask == nullptr ? nullptr : mask + start, vec};
}
// keys of split z: whole tiles, in equal shares
__device__ __forceinline__ void split_range(int n, int tile, int splits, int z, int* b, int* e) {
    const int tiles = (n + tile - 1) / tile, per = (tiles + splits - 1) / splits;
    *b = z * per * tile;
    *e = (z + 1) * per * tile;
    if (*b > n) *b = n;
    if (*e > n) *e = n;
}

// ---------------------------------------------------------------------------------------------
// forward: WAVES waves of 16 rows each share the key tiles
// ---------------------------------------------------------------------------------------------
template <class T, int DP, int WAVES, int KT>
__global__ __launch_bounds__(WAVES * 64) void att_fwd_kernel(AttDims d, const T* __restrict__ q, const T* __restrict__ k,
                                                             const T* __restrict__ v, T* __restrict__ out,
                                                             float* __restrict__ lse, float* __restrict__ part) {
    constexpr int NT = WAVES * 64, TR = WAVES * 16;
    using KTile = Tile<T, KT, DP / 8>;
    using VTile = Tile<T, DP, KT / 8>;
    extern __shared__ __align__(16) char lds[];
    char* kl = lds;
    char* vl = kl + KTile::BYTES;
    const Span sp = find_span(d, false, TR, d.group, blockIdx.x);
    const int hk = blockIdx.y, r0 = sp.tile * TR, nrows = (sp.qe - sp.qs) * d.group;
    if (r0 >= nrows) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const int row = r0 + wave * 16 + c;
    const uint8_t* mask = d.mask;
    const Rows<T> qr = rows_of(q, d.q_row, d.q_head, sp.qs, nrows, hk * d.group, d.group, d.dim, nullptr, d.qvec);
    const Rows<T> kr = rows_of(k, d.k_row, d.k_head, sp.ks, sp.ke - sp.ks, hk, 1, d.dim, mask, d.kvec);
    const Rows<T> vr = rows_of(v, d.v_row, d.v_head, sp.ks, sp.ke - sp.ks, hk, 1, d.dim, mask, d.vvec);
    Chunk<T> qf[DP / 32];
    row_chunks<T, DP>(qf, qr, row);
    f32x4 o[DP / 16];
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) o[t] = f32x4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.f;
    int kb, ke;
    split_range(kr.n, KT, d.splits, blockIdx.z, &kb, &ke);
    for (int k0 = kb; k0 < ke; k0 += KT) {
        __syncthreads();
        stage_rows<T, KT, DP, NT>(kl, kr, k0);
        stage_cols<T, KT, DP, NT>(vl, vr, k0);
        __syncthreads();
        f32x4 s[KT / 16];
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < KT / 16; ++t) {
            s[t] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int b = 0; b < DP / 32; ++b) s[t] = mma(KTile::get(kl, t * 16 + c, b * 4 + g), qf[b], s[t]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[t][e] = kr.has(k0 + t * 16 + g * 4 + e) ? s[t][e] * d.scale2 : -INFINITY;
                top = fmaxf(top, s[t][e]);
            }
        }
        top = fmaxf(m, over_groups_max(top));
        const float safe = top == -INFINITY ? 0.f : top, a = exp2_fast(m - safe);
        m = top;
        l *= a;
#pragma unroll
        for (int t = 0; t < KT / 16; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[t][e] = exp2_fast(s[t][e] - safe);
                l += s[t][e];
            }
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) o[t] *= a;
#pragma unroll
        for (int b = 0; b < KT / 32; ++b) {
            const Chunk<T> p = joined<T>(s[2 * b], s[2 * b + 1]);
#pragma unroll
            for (int t = 0; t < DP / 16; ++t) o[t] = mma(VTile::get(vl, t * 16 + c, b * 4 + g), p, o[t]);
        }
    }
    l = over_groups_sum(l);
    if (row >= nrows) return;
    const int qi = sp.qs + row / d.group, h = hk * d.group + row % d.group;
    const int64_t at = (int64_t)qi * d.heads + h;
    if (d.splits > 1) {  // unnormalised sums and their statistics: att_join_kernel ends the work
        const int64_t all = (int64_t)d.rows_q * d.heads, i = blockIdx.z * all + at;
        float* po = part + i * d.dim;
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) store4(po + t * 16 + g * 4, o[t], d.dim - t * 16 - g * 4, d.dim % 4 == 0);
        if (g == 0) {
            float* ps = part + d.splits * all * d.dim + 2 * i;
            ps[0] = m;
            ps[1] = l;
        }
        return;
    }
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) store4(out + at * d.dim + t * 16 + g * 4, o[t] * inv, d.dim - t * 16 - g * 4, d.ovec);
    if (lse != nullptr && g == 0) lse[at] = l == 0.f ? -INFINITY : m + log2f(l);
}

// The parts of a row: out = sum_z 2^(m_z - m) O_z / sum_z 2^(m_z - m) l_z, 64 rows' values a workgroup
template <class T>
__global__ __launch_bounds__(256) void att_join_kernel(int64_t all, int dim, int splits, const float* __restrict__ part,
                                                       T* __restrict__ out, float* __restrict__ lse) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, at = i / dim;
    if (at >= all) return;
    const int e = (int)(i % dim);
    const float* stat = part + splits * all * dim;
    float m = -INFINITY;
    for (int z = 0; z < splits; ++z) m = fmaxf(m, stat[2 * (z * all + at)]);
    const float safe = m == -INFINITY ? 0.f : m;
    float l = 0.f, o = 0.f;
    for (int z = 0; z < splits; ++z) {
        const float a = exp2_fast(stat[2 * (z * all + at)] - safe);
        l += a * stat[2 * (z * all + at) + 1];
        o += a * part[(z * all + at) * dim + e];
    }
    out[i] = (T)(l == 0.f ? 0.f : o / l);
    if (lse != nullptr && e == 0) lse[at] = l == 0.f ? -INFINITY : m + log2f(l);
}

// out[i] = sum_z part[z][i]
template <class T>
__global__ __launch_bounds__(256) void att_sum_kernel(int64_t n, int splits, const float* __restrict__ part, T* __restrict__ a,
                                                      const float* __restrict__ part2, T* __restrict__ a2) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const float* p = blockIdx.y ? part2 : part;
    T* o = blockIdx.y ? a2 : a;
    float s = 0.f;
    for (int z = 0; z < splits; ++z) s += p[z * n + i];
    o[i] = (T)s;
}

// ---------------------------------------------------------------------------------------------
// dQ: the forward's tiles again; delta on the way
// ---------------------------------------------------------------------------------------------
template <class T, int DP, int WAVES, int KT>
__global__ __launch_bounds__(WAVES * 64) void att_dq_kernel(AttDims d, const T* __restrict__ q, const T* __restrict__ k,
                                                            const T* __restrict__ v, const T* __restrict__ out,
                                                            const T* __restrict__ dout, const float* __restrict__ lse,
                                                            float* __restrict__ delta, T* __restrict__ dq,
                                                            float* __restrict__ part) {
    constexpr int NT = WAVES * 64, TR = WAVES * 16;
    using KTile = Tile<T, KT, DP / 8>;
    using KCols = Tile<T, DP, KT / 8>;
    extern __shared__ __align__(16) char lds[];
    char* kl = lds;
    char* vl = kl + KTile::BYTES;
    char* kc = vl + KTile::BYTES;
    const Span sp = find_span(d, false, TR, d.group, blockIdx.x);
    const int hk = blockIdx.y, r0 = sp.tile * TR, nrows = (sp.qe - sp.qs) * d.group;
    if (r0 >= nrows) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const int row = r0 + wave * 16 + c;
    const Rows<T> qr = rows_of(q, d.q_row, d.q_head, sp.qs, nrows, hk * d.group, d.group, d.dim, nullptr, d.qvec);
    const Rows<T> gr = rows_of(dout, d.do_row, d.do_head, sp.qs, nrows, hk * d.group, d.group, d.dim, nullptr, d.dovec);
    const Rows<T> orow = rows_of(out, (int64_t)d.heads * d.dim, d.dim, sp.qs, nrows, hk * d.group, d.group, d.dim, nullptr, d.ovec);
    const Rows<T> kr = rows_of(k, d.k_row, d.k_head, sp.ks, sp.ke - sp.ks, hk, 1, d.dim, d.mask, d.kvec);
    const Rows<T> vr = rows_of(v, d.v_row, d.v_head, sp.ks, sp.ke - sp.ks, hk, 1, d.dim, d.mask, d.vvec);
    Chunk<T> qf[DP / 32], gf[DP / 32];
    row_chunks<T, DP>(qf, qr, row);
    row_chunks<T, DP>(gf, gr, row);
    const bool mine = row < nrows;
    const int qi = sp.qs + (mine ? row / d.group : 0), h = hk * d.group + (mine ? row % d.group : 0);
    const int64_t at = (int64_t)qi * d.heads + h;
    float del = 0.f;
    if (mine) {
        const T *po = orow.at(row), *pg = gr.at(row);
#pragma unroll
        for (int b = 0; b < DP / 32; ++b)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int x = b * 32 + g * 8 + e;
                if (x < d.dim) del += to_f(po[x]) * to_f(pg[x]);
            }
    }
    del = over_groups_sum(del);
    const float L = mine ? lse[at] : INFINITY, safe = L == -INFINITY ? INFINITY : L;  // no open key: every weight is 0
    if (mine && g == 0 && blockIdx.z == 0) delta[at] = del;
    f32x4 acc[DP / 16];
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) acc[t] = f32x4{0, 0, 0, 0};
    int kb, ke;
    split_range(kr.n, KT, d.splits, blockIdx.z, &kb, &ke);
    for (int k0 = kb; k0 < ke; k0 += KT) {
        __syncthreads();
        stage_rows<T, KT, DP, NT>(kl, kr, k0);
        stage_rows<T, KT, DP, NT>(vl, vr, k0);
        stage_cols<T, KT, DP, NT>(kc, kr, k0);
        __syncthreads();
#pragma unroll
        for (int p = 0; p < KT / 32; ++p) {
            f32x4 ds[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int t = 2 * p + u;
                f32x4 s = {0, 0, 0, 0}, dp = {0, 0, 0, 0};
#pragma unroll
                for (int b = 0; b < DP / 32; ++b) {
                    s = mma(KTile::get(kl, t * 16 + c, b * 4 + g), qf[b], s);
                    dp = mma(KTile::get(vl, t * 16 + c, b * 4 + g), gf[b], dp);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float w = kr.has(k0 + t * 16 + g * 4 + e) ? exp2_fast(s[e] * d.scale2 - safe) : 0.f;
                    ds[u][e] = w * (dp[e] - del);
                }
            }
            const Chunk<T> f = joined<T>(ds[0], ds[1]);
#pragma unroll
            for (int t = 0; t < DP / 16; ++t) acc[t] = mma(KCols::get(kc, t * 16 + c, p * 4 + g), f, acc[t]);
        }
    }
    if (!mine) return;
    // a row without an open key has dQ = 0 whatever dO and O hold
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) {
        const f32x4 r = L == -INFINITY ? f32x4{0, 0, 0, 0} : acc[t] * d.scale;
        const int n = d.dim - t * 16 - g * 4;
        if (d.splits > 1)
            store4(part + (blockIdx.z * (int64_t)d.rows_q * d.heads + at) * d.dim + t * 16 + g * 4, r, n, d.dim % 4 == 0);
        else
            store4(dq + at * d.dim + t * 16 + g * 4, r, n, d.ovec);
    }
}

// ---------------------------------------------------------------------------------------------
// dK, dV: WAVES waves of 16 keys each; all rows (of all heads that read the keys) go by in tiles of RT
// ---------------------------------------------------------------------------------------------
template <class T, int DP, int WAVES, int RT>
__global__ __launch_bounds__(WAVES * 64) void att_dkv_kernel(AttDims d, const T* __restrict__ q, const T* __restrict__ k,
                                                             const T* __restrict__ v, const T* __restrict__ dout,
                                                             const float* __restrict__ lse, const float* __restrict__ delta,
                                                             T* __restrict__ dk, T* __restrict__ dv, float* __restrict__ part) {
    constexpr int NT = WAVES * 64, TK = WAVES * 16;
    using RTile = Tile<T, RT, DP / 8>;
    using CTile = Tile<T, DP, RT / 8>;
    extern __shared__ __align__(16) char lds[];
    char* ql = lds;
    char* gl = ql + RTile::BYTES;
    char* qc = gl + RTile::BYTES;
    char* gc = qc + CTile::BYTES;
    float* stat = reinterpret_cast<float*>(gc + CTile::BYTES);  // [2][RT]: L, delta
    const Span sp = find_span(d, true, TK, 1, blockIdx.x);
    const int hk = blockIdx.y, k0 = sp.tile * TK, nkeys = sp.ke - sp.ks, nrows = (sp.qe - sp.qs) * d.group;
    if (k0 >= nkeys) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const int key = k0 + wave * 16 + c;
    const Rows<T> qr = rows_of(q, d.q_row, d.q_head, sp.qs, nrows, hk * d.group, d.group, d.dim, nullptr, d.qvec);
    const Rows<T> gr = rows_of(dout, d.do_row, d.do_head, sp.qs, nrows, hk * d.group, d.group, d.dim, nullptr, d.dovec);
    const Rows<T> kr = rows_of(k, d.k_row, d.k_head, sp.ks, nkeys, hk, 1, d.dim, d.mask, d.kvec);
    const Rows<T> vr = rows_of(v, d.v_row, d.v_head, sp.ks, nkeys, hk, 1, d.dim, d.mask, d.vvec);
    Chunk<T> kf[DP / 32], vf[DP / 32];
    row_chunks<T, DP>(kf, kr, key);
    row_chunks<T, DP>(vf, vr, key);
    const bool open = kr.has(key);
    f32x4 ak[DP / 16], av[DP / 16];
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) ak[t] = av[t] = f32x4{0, 0, 0, 0};
    int rb, re;
    split_range(nrows, RT, d.splits, blockIdx.z, &rb, &re);
    for (int r0 = rb; r0 < re; r0 += RT) {
        __syncthreads();
        stage_rows<T, RT, DP, NT>(ql, qr, r0);
        stage_rows<T, RT, DP, NT>(gl, gr, r0);
        stage_cols<T, RT, DP, NT>(qc, qr, r0);
        stage_cols<T, RT, DP, NT>(gc, gr, r0);
        for (int u = threadIdx.x; u < RT; u += NT) {
            const int r = r0 + u;
            float L = INFINITY, del = 0.f;  // a missing row's weights are 0
            if (r < nrows) {
                const int64_t at = (int64_t)(sp.qs + r / d.group) * d.heads + hk * d.group + r % d.group;
                L = lse[at];
                L = L == -INFINITY ? INFINITY : L;
                del = delta[at];
            }
            stat[u] = L;
            stat[RT + u] = del;
        }
        __syncthreads();
#pragma unroll
        for (int p = 0; p < RT / 32; ++p) {
            f32x4 w[2], ds[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int t = 2 * p + u;
                f32x4 s = {0, 0, 0, 0}, dp = {0, 0, 0, 0};
#pragma unroll
                for (int b = 0; b < DP / 32; ++b) {
                    s = mma(RTile::get(ql, t * 16 + c, b * 4 + g), kf[b], s);
                    dp = mma(RTile::get(gl, t * 16 + c, b * 4 + g), vf[b], dp);
                }
                const f32x4 L = *reinterpret_cast<const f32x4*>(stat + t * 16 + g * 4);
                const f32x4 del = *reinterpret_cast<const f32x4*>(stat + RT + t * 16 + g * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    w[u][e] = open ? exp2_fast(s[e] * d.scale2 - L[e]) : 0.f;
                    ds[u][e] = open ? w[u][e] * (dp[e] - del[e]) : 0.f;
                }
            }
            const Chunk<T> pf = joined<T>(w[0], w[1]), df = joined<T>(ds[0], ds[1]);
#pragma unroll
            for (int t = 0; t < DP / 16; ++t) {
                av[t] = mma(CTile::get(gc, t * 16 + c, p * 4 + g), pf, av[t]);
                ak[t] = mma(CTile::get(qc, t * 16 + c, p * 4 + g), df, ak[t]);
            }
        }
    }
    if (key >= nkeys) return;
    const int64_t all = (int64_t)d.rows_k * d.kv_heads, at = (int64_t)(sp.ks + key) * d.kv_heads + hk;
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) {
        const int x = t * 16 + g * 4, n = d.dim - x;
        // a masked key's gradients are 0 whatever the rows that do not read it hold
        const f32x4 rk = open ? ak[t] * d.scale : f32x4{0, 0, 0, 0}, rv = open ? av[t] : f32x4{0, 0, 0, 0};
        if (d.splits > 1) {
            store4(part + (blockIdx.z * all + at) * d.dim + x, rk, n, d.dim % 4 == 0);
            store4(part + ((d.splits + blockIdx.z) * all + at) * d.dim + x, rv, n, d.dim % 4 == 0);
        } else {
            store4(dk + at * d.dim + x, rk, n, d.ovec);
            store4(dv + at * d.dim + x, rv, n, d.ovec);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
// One wave a tile where the graphs are small (its 16 rows fill it at least as well as 64 would), four otherwise.
static int att_waves(int64_t rows, int graphs) { return rows <= 32 * (int64_t)(graphs < 1 ? 1 : graphs) ? 1 : 4; }
static int att_slots(int64_t rows, int graphs, int tile) { return (int)(rows / tile) + graphs + 2; }
// Shares of the other side's tiles: enough workgroups for the 256 CUs, and four tiles of 64 a share at least.
static int att_splits(int64_t workgroups, int64_t other, int graphs) {
    const int64_t want = 1024 / (workgroups < 1 ? 1 : workgroups), most = other / (graphs < 1 ? 1 : graphs) / 256;
    const int64_t s = want < most ? want : most;
    return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

struct AttPlan {
    int wq, wk, splits_q, splits_k;  // waves a tile; shares of the keys (forward, dQ) and of the rows (dK, dV)
    size_t fwd, bwd;                 // scratch floats
    size_t part;                     // where the backward's parts begin (behind delta)
};
static AttPlan att_plan(const tsd_attention& a) {
    AttPlan p = {};
    const int group = a.heads / a.kv_heads;
    const int64_t rows = (int64_t)a.num_queries * group, keys = a.num_keys;
    p.wq = att_waves(rows, a.num_graphs);
    p.wk = att_waves(keys, a.num_graphs);
    p.splits_q = att_splits((rows / (16 * p.wq) + a.num_graphs) * a.kv_heads, keys, a.num_graphs);
    p.splits_k = att_splits((keys / (16 * p.wk) + a.num_graphs) * a.kv_heads, rows, a.num_graphs);
    const size_t nq = (size_t)a.num_queries * a.heads, nk = (size_t)keys * a.kv_heads;
    p.fwd = p.splits_q > 1 ? p.splits_q * nq * (a.dim + 2) : 0;
    const size_t q = p.splits_q > 1 ? p.splits_q * nq * a.dim : 0, k = p.splits_k > 1 ? 2 * p.splits_k * nk * a.dim : 0;
    p.part = (nq + 3) / 4 * 4;
    p.bwd = p.part + (q > k ? q : k);  // dQ's parts are joined before dK's and dV's are written
    return p;
}

static int att_check(const char* name, const tsd_attention* a) {
    TSD_REQUIRE(a != nullptr, "%s: null pointer", name);
    TSD_REQUIRE(a->dtype == TSD_F32 || a->dtype == TSD_BF16 || a->dtype == TSD_F16, "%s: unknown type %d", name, a->dtype);
    TSD_REQUIRE(a->num_graphs >= 0 && a->num_queries >= 0 && a->num_keys >= 0 && a->heads >= 1 && a->kv_heads >= 1 &&
                    a->heads % a->kv_heads == 0 && a->dim >= 1,
                "%s: bad sizes: %d graphs, %d queries, %d keys, %d heads, %d key heads, dim %d", name, a->num_graphs,
                a->num_queries, a->num_keys, a->heads, a->kv_heads, a->dim);
    if (a->dim > TSD_ATTENTION_MAX_DIM || a->kv_heads > 65535 || (int64_t)a->num_queries * a->heads > (1 << 30) ||
        (int64_t)a->num_keys * a->heads > (1 << 30) || a->num_graphs > (1 << 22)) {
        set_error("%s: head dim %d (at most %d), %d queries, %d keys, %d heads, %d graphs", name, a->dim, TSD_ATTENTION_MAX_DIM,
                  a->num_queries, a->num_keys, a->heads, a->num_graphs);
        return TSD_ERR_UNSUPPORTED;
    }
    TSD_REQUIRE(a->q_ptr != nullptr && a->k_ptr != nullptr, "%s: null offsets", name);
    TSD_REQUIRE(a->num_queries == 0 || a->q != nullptr, "%s: null pointer", name);
    TSD_REQUIRE(a->num_keys == 0 || (a->k != nullptr && a->v != nullptr), "%s: null pointer", name);
    return TSD_OK;
}
static bool att_vec(const void* p, int64_t row, int64_t head, int dim, int es) {
    const int v = 16 / es;
    return dim % 8 == 0 && row % v == 0 && head % v == 0 && aligned16(p);
}
static AttDims att_dims(const tsd_attention& a) {
    AttDims d = {};
    const int es = a.dtype == TSD_F32 ? 4 : 2;
    d.graphs = a.num_graphs;
    d.rows_q = a.num_queries;
    d.rows_k = a.num_keys;
    d.heads = a.heads;
    d.kv_heads = a.kv_heads;
    d.group = a.heads / a.kv_heads;
    d.dim = a.dim;
    d.q_row = a.q_row;
    d.q_head = a.q_head;
    d.k_row = a.k_row;
    d.k_head = a.k_head;
    d.v_row = a.v_row;
    d.v_head = a.v_head;
    d.scale = a.scale;
    d.scale2 = a.scale * LOG2E;
    d.qvec = att_vec(a.q, a.q_row, a.q_head, a.dim, es);
    d.kvec = att_vec(a.k, a.k_row, a.k_head, a.dim, es);
    d.vvec = att_vec(a.v, a.v_row, a.v_head, a.dim, es);
    d.q_ptr = a.q_ptr;
    d.k_ptr = a.k_ptr;
    d.mask = a.key_mask;
    return d;
}

template <class T, int DP, int WAVES>
static int att_launch_fwd(AttDims d, const tsd_attention& a, T* out, float* lse, float* scratch, hipStream_t st) {
    constexpr int KT = WAVES == 1 ? 32 : ATT_KT;
    constexpr int lds = Tile<T, KT, DP / 8>::BYTES + Tile<T, DP, KT / 8>::BYTES;
    static DeviceOnce once;
    auto k = att_fwd_kernel<T, DP, WAVES, KT>;
    const int rc = allow_lds(k, lds, once);
    if (rc != TSD_OK) return rc;
    hipLaunchKernelGGL(k, dim3(att_slots((int64_t)d.rows_q * d.group, d.graphs, WAVES * 16), d.kv_heads, d.splits),
                       dim3(WAVES * 64), lds, st, d, (const T*)a.q, (const T*)a.k, (const T*)a.v, out, lse, scratch);
    TSD_LAUNCH_CHECK("attention_fwd");
    if (d.splits > 1) {
        const int64_t all = (int64_t)d.rows_q * d.heads;
        hipLaunchKernelGGL(att_join_kernel<T>, dim3((unsigned)((all * d.dim + 255) / 256)), dim3(256), 0, st, all, d.dim, d.splits,
                           scratch, out, lse);
        TSD_LAUNCH_CHECK("attention_join");
    }
    return TSD_OK;
}
template <class T, int DP, int WAVES>
static int att_launch_dq(AttDims d, const tsd_attention& a, const T* out, const T* dout, const float* lse, float* delta, T* dq,
                         float* part, hipStream_t st) {
    constexpr int KT = WAVES == 1 || DP == 128 ? 32 : ATT_KT;
    constexpr int lds = 2 * Tile<T, KT, DP / 8>::BYTES + Tile<T, DP, KT / 8>::BYTES;
    static DeviceOnce once;
    auto k = att_dq_kernel<T, DP, WAVES, KT>;
    const int rc = allow_lds(k, lds, once);
    if (rc != TSD_OK) return rc;
    hipLaunchKernelGGL(k, dim3(att_slots((int64_t)d.rows_q * d.group, d.graphs, WAVES * 16), d.kv_heads, d.splits),
                       dim3(WAVES * 64), lds, st, d, (const T*)a.q, (const T*)a.k, (const T*)a.v, out, dout, lse, delta, dq, part);
    TSD_LAUNCH_CHECK("attention_dq");
    if (d.splits > 1) {
        const int64_t n = (int64_t)d.rows_q * d.heads * d.dim;
        hipLaunchKernelGGL(att_sum_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, n, d.splits, part, dq,
                           (const float*)nullptr, (T*)nullptr);
        TSD_LAUNCH_CHECK("attention_dq_sum");
    }
    return TSD_OK;
}
template <class T, int DP, int WAVES>
static int att_launch_dkv(AttDims d, const tsd_attention& a, const T* dout, const float* lse, const float* delta, T* dk, T* dv,
                          float* part, hipStream_t st) {
    constexpr int RT = 32;
    constexpr int lds = 2 * Tile<T, RT, DP / 8>::BYTES + 2 * Tile<T, DP, RT / 8>::BYTES + 2 * RT * 4;
    static DeviceOnce once;
    auto k = att_dkv_kernel<T, DP, WAVES, RT>;
    const int rc = allow_lds(k, lds, once);
    if (rc != TSD_OK) return rc;
    hipLaunchKernelGGL(k, dim3(att_slots(d.rows_k, d.graphs, WAVES * 16), d.kv_heads, d.splits), dim3(WAVES * 64), lds, st, d,
                       (const T*)a.q, (const T*)a.k, (const T*)a.v, dout, lse, delta, dk, dv, part);
    TSD_LAUNCH_CHECK("attention_dkv");
    if (d.splits > 1) {
        const int64_t n = (int64_t)d.rows_k * d.kv_heads * d.dim;
        hipLaunchKernelGGL(att_sum_kernel<T>, dim3((unsigned)((n + 255) / 256), 2), dim3(256), 0, st, n, d.splits, part, dk,
                           part + d.splits * n, dv);
        TSD_LAUNCH_CHECK("attention_dkv_sum");
    }
    return TSD_OK;
}

template <class T, int DP>
static int att_fwd(AttDims d, const AttPlan& p, const tsd_attention& a, void* out, float* lse, float* scratch, hipStream_t st) {
    d.splits = p.splits_q;
    d.ovec = d.dim % 4 == 0 && aligned16(out);
    return p.wq == 1 ? att_launch_fwd<T, DP, 1>(d, a, (T*)out, lse, scratch, st)
                     : att_launch_fwd<T, DP, 4>(d, a, (T*)out, lse, scratch, st);
}
template <class T, int DP>
static int att_bwd(AttDims d, const AttPlan& p, const tsd_attention& a, const void* out, const void* dout, int64_t do_row,
                   int64_t do_head, const float* lse, void* dq, void* dk, void* dv, float* scratch, hipStream_t st) {
    float *delta = scratch, *part = scratch + p.part;
    d.do_row = do_row;
    d.do_head = do_head;
    d.dovec = att_vec(dout, do_row, do_head, d.dim, sizeof(T));
    d.ovec = d.dim % 8 == 0 && aligned16(out) && aligned16(dq) && aligned16(dk) && aligned16(dv);
    int rc = TSD_OK;
    if (d.rows_q > 0) {
        d.splits = p.splits_q;
        rc = p.wq == 1 ? att_launch_dq<T, DP, 1>(d, a, (const T*)out, (const T*)dout, lse, delta, (T*)dq, part, st)
                       : att_launch_dq<T, DP, 4>(d, a, (const T*)out, (const T*)dout, lse, delta, (T*)dq, part, st);
    }
    if (rc == TSD_OK && d.rows_k > 0) {
        d.splits = p.splits_k;
        rc = p.wk == 1 ? att_launch_dkv<T, DP, 1>(d, a, (const T*)dout, lse, delta, (T*)dk, (T*)dv, part, st)
                       : att_launch_dkv<T, DP, 4>(d, a, (const T*)dout, lse, delta, (T*)dk, (T*)dv, part, st);
    }
    return rc;
}

}  // namespace blk
}  // namespace tsd

using namespace tsd;
using namespace tsd::blk;

extern "C" {

size_t tsd_graph_attention_scratch_floats(const tsd_attention* a, int32_t backward) {
    if (att_check("tsd_graph_attention_scratch_floats", a) != TSD_OK) return 0;
    const AttPlan p = att_plan(*a);
    return backward ? p.bwd : p.fwd;
}

int tsd_graph_attention_fwd(const tsd_attention* a, void* out, float* lse, float* scratch, size_t scratch_floats, void* stream) {
    const int rc = att_check("tsd_graph_attention_fwd", a);
    if (rc != TSD_OK) return rc;
    if (a->num_queries == 0) return TSD_OK;
    const AttPlan p = att_plan(*a);
    TSD_REQUIRE(out != nullptr, "tsd_graph_attention_fwd: null pointer");
    TSD_REQUIRE(p.fwd == 0 || (scratch != nullptr && aligned16(scratch) && scratch_floats >= p.fwd),
                "tsd_graph_attention_fwd: scratch of %zu floats, %zu needed (16-byte aligned)", scratch_floats, p.fwd);
    const AttDims d = att_dims(*a);
    hipStream_t st = (hipStream_t)stream;
    TSD_BY_DTYPE(a->dtype, T, {
        if (d.dim <= 32) return att_fwd<T, 32>(d, p, *a, out, lse, scratch, st);
        if (d.dim <= 64) return att_fwd<T, 64>(d, p, *a, out, lse, scratch, st);
        return att_fwd<T, 128>(d, p, *a, out, lse, scratch, st);
    });
    return TSD_OK;
}

int tsd_graph_attention_bwd(const tsd_attention* a, const void* out, const float* lse, const void* dout, int64_t do_row,
                            int64_t do_head, void* dq, void* dk, void* dv, float* scratch, size_t scratch_floats, void* stream) {
    const int rc = att_check("tsd_graph_attention_bwd", a);
    if (rc != TSD_OK) return rc;
    const AttPlan p = att_plan(*a);
    TSD_REQUIRE(a->num_queries == 0 || (out != nullptr && lse != nullptr && dout != nullptr && dq != nullptr),
                "tsd_graph_attention_bwd: null pointer");
    TSD_REQUIRE(a->num_keys == 0 || (dk != nullptr && dv != nullptr), "tsd_graph_attention_bwd: null pointer");
    TSD_REQUIRE(scratch != nullptr ? aligned16(scratch) && scratch_floats >= p.bwd : p.bwd == 0,
                "tsd_graph_attention_bwd: scratch of %zu floats, %zu needed (16-byte aligned)", scratch_floats, p.bwd);
    const AttDims d = att_dims(*a);
    hipStream_t st = (hipStream_t)stream;
    TSD_BY_DTYPE(a->dtype, T, {
        if (d.dim <= 32) return att_bwd<T, 32>(d, p, *a, out, dout, do_row, do_head, lse, dq, dk, dv, scratch, st);
        if (d.dim <= 64) return att_bwd<T, 64>(d, p, *a, out, dout, do_row, do_head, lse, dq, dk, dv, scratch, st);
        return att_bwd<T, 128>(d, p, *a, out, dout, do_row, do_head, lse, dq, dk, dv, scratch, st);
    });
    return TSD_OK;
}

}  // extern "C"
