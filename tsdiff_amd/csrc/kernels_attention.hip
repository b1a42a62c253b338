// kernels_attention.hip -- attention inside the graphs of a ragged batch, forward and backward.
//
//   S = scale Q K^T over the open keys of the row's graph, P = softmax S, O = P V, L = log2 sum exp2(S log2 e)
//   (L = +inf for a row without keys: every 2^(S - L) of it is 0)
//   delta = sum_d dO O;  dP = dO V^T;  dS = P (dP - delta);  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
//
// One pass over the keys: the running maximum and sum of each row stay in registers and the scores never leave them.  The
// scores are computed turned, S^T = K Q^T, so that a lane holds one row's scores (their statistics are a lane's own, two
// swaps join the four lanes of a row) AND the result registers are the operand of the next product as they stand: the rows
// of a tile are taken in the order (sub_row) in which a lane's eight scores are eight consecutive keys.  Every tile lies in
// LDS as it lies in memory, for both products: S reads it along its rows, P V and dS K by the LDS's transposing read.
// The backward computes the scores again from L: one launch over row tiles for dQ (and delta), one over key tiles for dK and
// dV.  Without atomics: a gradient is summed by one workgroup in a fixed order or, where few workgroups have long sums, in parts
// that a further launch adds in order.
//
// Rows are (query, query head of the key head's group), so heads that share keys share their tiles.  Tiles never cross a
// graph: workgroup s looks its graph up, slot(v) = floor((start_v + v (T - 1)) / T) being where graph v's tiles begin -- a
// bound on the tiles before it that needs no prefix sum and no lengths on the host, less than one idle workgroup a graph.
// The key heads of a slot are neighbouring workgroups: they go to the eight XCDs in turn, and share lines of memory in time.
// Offsets are clamped into the tensors.  Rows and keys outside of every graph count as graphs without keys / rows: they are written
// as zeros.  Masked and missing keys are zeros in LDS whatever memory holds there, so that no NaN meets a zero weight.
//
// Measured (GPU time a launch):
//   f32, 1024 graphs of 64, 8 heads of 32: forward 77 us (3.5 TB/s of 268 MB), dQ 104 us (3.9 TB/s), dK and dV 120 us
//   (3.4 TB/s): by memory, and by the six plane products of each f32 one, which take as long.
//   bf16, 3 graphs of 1888, 1493 and 2405, 8 heads on 2 key heads of 64, the first closed and a fifth of the others' keys:
//   forward 57 us, dQ 67 us, dK and dV 81 us: 286, 367 and 407 TFLOP/s of the pairs in open graphs, a quarter to a third of the
//   pipes' rate: the two open graphs are 490 workgroups of the forward, under two waves a SIMD, and a wave's chain S, maximum,
//   exp2, P V has nothing of the next tile to work on while it waits.
//   f16, 8 graphs of 2000 .. 8192, one query, 8 heads of 64: 20 us (3.5 TB/s of the keys and values that are read) and 4 us to
//   join the parts.
//   f32, 100 graphs of 6 .. 30, 8 heads of 32, forward: 7 us, two of them a kernel's launch.
#include "block_tile.hpp"

namespace tsd {
namespace blk {

constexpr float LOG2E = 1.44269504088896341f;
constexpr float LAG = 6.f;  // (in powers of two: weights up to 64 times 1, far from the end of every type)
// f16: the weights and dS become matrix operands as powers of two of themselves.  As they are, small ones fall among the
// subnormal numbers (steps of 2^-24), where a long list of them is lost as a whole, and a dS beyond 65504 becomes infinite
// (2000 nodes, 2 heads of 64, dO of 1e-3: dQ and dK off by 2.6e-3 so, by 5.1e-4 with these, the rounding of dQ itself 4.7e-4;
// for 4 to 6 % of the time of a training step of long graphs).
// Forward: 2^(S - m + 9), up to 2^15 with LAG; dK / dV: 2^(S - L + 15); dS: DsScale.
template <class T> constexpr bool att_scaled() { return __is_same(T, f16); }
template <class T> constexpr float att_fwd_shift() { return att_scaled<T>() ? 9.f : 0.f; }
template <class T> constexpr float att_dkv_shift() { return att_scaled<T>() ? 15.f : 0.f; }

struct AttDims {
    int graphs, rows_q, rows_k, heads, kv_heads, group, dim;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, do_row, do_head;
    float scale, scale2;  // scale2 = scale * log2 e
    int splits;
    int heads_a_wg;       // key heads that a workgroup goes over, one after the other
    float graph_of_slot;  // where equal graphs would have a slot's graph
    int qvw, kvw, vvw, dovw;  // values a load of each may take (load_raw)
    bool ovec;
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
    return v <= 0 ? 0 : v > graphs + 1 ? n : clamp_to(ptr[v - 1], n);
}
// The graph whose tiles (T rows, `times` rows an entry) hold slot s.  slot(v) = floor((start_v times + v (T - 1)) / T) leaves
// every graph the tiles it needs.  64 lanes look at a time, first where equal graphs would have it.
__device__ __forceinline__ Span find_span(const AttDims& d, bool by_key, int T, int times, int s) {
    const int32_t* ptr = by_key ? d.k_ptr : d.q_ptr;
    const int32_t* other = by_key ? d.q_ptr : d.k_ptr;
    const int n = by_key ? d.rows_k : d.rows_q, on = by_key ? d.rows_q : d.rows_k, lane = threadIdx.x & 63, all = d.graphs + 2;
    // (32 bits: at most 2^29 rows and 2^22 graphs)
    auto slot = [&](int b, int v) { return (int)(((uint32_t)b * (uint32_t)times + (uint32_t)v * (uint32_t)(T - 1)) / (uint32_t)T); };
    int lo = (int)((float)s * d.graph_of_slot) - 32;
    lo = lo > all - 64 ? all - 64 : lo;
    lo = lo < 0 ? 0 : lo;
    int b = bound_at(ptr, d.graphs, n, lo + lane);
    unsigned long long m = __ballot(lo + lane < all && slot(b, lo + lane) <= s);
    if (!(m & 1) || (m == ~0ull && lo + 64 < all)) {  // not here: narrow the whole list down
        lo = 0;
        int count = all;  // slot(lo) <= s < slot(lo + count)
        while (count > 64) {
            const int step = (count + 63) / 64, v = lo + lane * step;
            m = __ballot(lane * step < count && slot(bound_at(ptr, d.graphs, n, v), v) <= s);
            const int last = 63 - __builtin_clzll(m | 1);
            lo += last * step;
            count = count - last * step < step ? count - last * step : step;
        }
        b = bound_at(ptr, d.graphs, n, lo + lane);
        m = __ballot(lane < count && slot(b, lo + lane) <= s);
    }
    const int last = 63 - __builtin_clzll(m | 1), v = lo + last;
    const int start = __builtin_amdgcn_readlane(b, last);
    int end = last < 63 ? __builtin_amdgcn_readlane(b, last < 63 ? last + 1 : 63) : bound_at(ptr, d.graphs, n, v + 1);
    int os = 0, oe = 0;
    if (v >= 1 && v <= d.graphs) {
        if (other == ptr && on == n) {
            os = start;
            oe = end;
        } else {
            os = bound_at(other, d.graphs, on, v);
            oe = bound_at(other, d.graphs, on, v + 1);
        }
    }
    Span sp;
    sp.tile = s - slot(start, v);
    end = end < start ? start : end;
    oe = oe < os ? os : oe;
    sp.qs = by_key ? os : start;
    sp.qe = by_key ? oe : end;
    sp.ks = by_key ? start : os;
    sp.ke = by_key ? end : oe;
    return sp;
}

// row = query * group + head of the group
__device__ __forceinline__ int query_of(int row, int group) { return group == 1 ? row : row / group; }

// Values (row, d) of a graph's rows or keys
template <class T> struct Rows {
    const T* p;         // row 0 of the graph, this head (the first of the group)
    int64_t row, head;  // strides
    int n, group, dim;  // n: rows
    const uint8_t* mask;
    int vw;
    __device__ __forceinline__ bool has(int r) const { return r < n && (mask == nullptr || mask[r] != 0); }
    __device__ __forceinline__ const T* at(int r) const {
        if (group == 1) return p + (int64_t)r * row;
        const int q = r / group;
        return p + (int64_t)q * row + (r - q * group) * head;
    }
    // bit i: row r0 + i (i < 64) is there
    __device__ __forceinline__ uint64_t there(int r0) const { return n - r0 >= 64 ? ~0ull : n > r0 ? (1ull << (n - r0)) - 1 : 0; }
    // ... and open (i < ROWS); the same in every lane
    template <int ROWS> __device__ __forceinline__ uint64_t open(int r0) const {
        if (mask == nullptr) return there(r0);
        const int lane = threadIdx.x & 63;
        return __ballot(lane < ROWS && has(r0 + lane));
    }
};
// Is exactly one key open (the same in every lane)?  Its weight is then 1 whatever its score, dS = 0, and what is left of
// dP - delta in 24 bits is no gradient: dQ and dK are their sums times 0 (a NaN stays one).
template <class T> __device__ __forceinline__ bool one_open(const Rows<T>& s) {
    if (s.mask == nullptr) return s.n == 1;
    int count = 0;
    for (int r0 = 0; r0 < s.n && count < 2; r0 += 64) count += __popcll(s.template open<64>(r0));
    return count == 1;
}
// Which keys are open, a word a tile, MASK_TILES tiles at a time in LDS: looked up tile by tile, the mask's bytes would be
// waited for in front of every tile's loads.
constexpr int MASK_TILES = 128, MASK_BYTES = MASK_TILES * 8;
template <int WAVES, int KT, class T>
__device__ __forceinline__ void mask_words(const Rows<T>& s, int tb, int te, uint64_t* words) {
    if (s.mask == nullptr) return;
    __syncthreads();
#pragma unroll 4
    for (int t = tb + (int)(threadIdx.x >> 6); t < te; t += WAVES) {
        const uint64_t w = s.template open<KT>(t * KT);
        if ((threadIdx.x & 63) == 0) words[t - tb] = w;
    }
    __syncthreads();
}
template <int KT, class T> __device__ __forceinline__ uint64_t mask_word(const Rows<T>& s, int t, int tb, const uint64_t* words) {
    if (s.mask == nullptr) return s.there(t * KT);
    const uint64_t w = words[t - tb];
    return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)w) |
           (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(w >> 32)) << 32;
}

// A tile of ROWS rows on its way to LDS; rows that are not open become zeros.  FAST: 16-byte loads with bounds in the buffer,
// straight to LDS (DMA) for the 16-bit types, by way of registers for f32; otherwise guarded loads.  QUERIES (DMA): rows of
// several heads; where the group divides ROWS a lane's places are the same in every tile, and the tiles follow each other by
// the same distance (dK and dV of 3 graphs of 1200 .. 2600 nodes, 4 heads a key head: 103 -> 79 us).
template <class T, bool FAST> constexpr bool att_dma() { return FAST && sizeof(T) == 2; }
template <class T, int ROWS, int DP, int NT, bool FAST, bool QUERIES> struct RowStage {
    using Lds = Tile<T, ROWS, DP / 8>;
    static constexpr bool DMA = att_dma<T, FAST>();
    static constexpr int C = DP / 8, UNITS = ROWS * C, U = (UNITS + NT - 1) / NT;
    static_assert(UNITS % NT == 0 || (NT % UNITS == 0 && UNITS % 64 == 0), "whole loads");
    Raw<T> raw[DMA ? 1 : U];
    static constexpr bool KEEP = DMA && QUERIES;
    uint32_t off[KEEP ? U : 1];
    int place[DMA ? U : 1];  // LDS bytes of a wave's load
    int queries;             // of a tile; 0: no whole number
    i32x4 at;                // tile `next` - 1
    int next;
    __device__ __forceinline__ static int row(int i) { return (threadIdx.x + i * NT) % UNITS / C; }  // (a small tile is
    __device__ __forceinline__ static int chunk(int i) {                                     //  loaded by several waves alike)
        const int c = (threadIdx.x + i * NT) % C;
        return DMA ? c ^ Lds::swizzle(row(i)) : c;
    }
    __device__ __forceinline__ void init(const Rows<T>& s) {
        queries = 0;
        if constexpr (KEEP) {
            next = -1;
            queries = ROWS % s.group == 0 ? ROWS / s.group : 0;
#pragma unroll
            for (int i = 0; i < U; ++i) {
                off[i] = chunk(i) * 8 < s.dim ? (uint32_t)((int)(s.at(row(i)) - s.p) + chunk(i) * 8) * (uint32_t)sizeof(T) : DMA_NOWHERE;
            }
        }
        if constexpr (DMA) {
#pragma unroll
            for (int i = 0; i < U; ++i)
                place[i] = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / 64 * 64 + i * NT) % UNITS * 16);
        }
    }
    template <bool ALL> __device__ __forceinline__ void fast(i32x4 buf, const uint32_t (&from)[U], uint64_t open, uint32_t lds) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const uint32_t o = ALL || (open >> row(i) & 1) ? from[i] : DMA_NOWHERE;
            if constexpr (DMA) {
                dma_load(buf, o, lds + place[i]);
            } else {
                raw[i].a = buffer_load(buf, o);
                raw[i].b = buffer_load(buf, o + 16);
            }
        }
    }
    __device__ __forceinline__ void load(const Rows<T>& s, int tile, uint64_t open, uint32_t lds) {
        if constexpr (FAST) {
            constexpr uint64_t ALL = ROWS == 64 ? ~0ull : (1ull << (ROWS % 64)) - 1;
            if (KEEP && queries > 0) {
                if (tile == next) dma_advance(at, queries * s.row * (int64_t)sizeof(T));
                else at = dma_buffer(s.p + (int64_t)(tile * queries) * s.row);
                next = tile + 1;
                if constexpr (KEEP) {
                    if ((open & ALL) == ALL) fast<true>(at, off, open, lds);
                    else fast<false>(at, off, open, lds);
                }
            } else {
                const int r0 = tile * ROWS;
                const T* base = s.p + (int64_t)query_of(r0, s.group) * s.row;
                uint32_t from[U];
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const int d = s.group == 1 ? row(i) * (int)s.row : (int)(s.at(r0 + row(i)) - base);
                    from[i] = chunk(i) * 8 < s.dim ? (uint32_t)(d + chunk(i) * 8) * (uint32_t)sizeof(T) : DMA_NOWHERE;
                }
                fast<false>(dma_buffer(base), from, open, lds);
            }
        } else {
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int r = row(i), c = chunk(i), n = open >> r & 1 ? s.dim - c * 8 : 0;
                load_raw(raw[i], n > 0 ? s.at(tile * ROWS + r) + c * 8 : s.p, n < 0 ? 0 : n > 8 ? 8 : n, s.vw);
            }
        }
    }
    __device__ __forceinline__ void store(char* lds) const {
        if constexpr (!DMA) {
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int u = threadIdx.x + i * NT;
                if (UNITS % NT == 0 || u < UNITS) Lds::put(lds, u / C, u % C, raw_chunk(raw[i]));
            }
        }
    }
};

template <class T, int N> __device__ __forceinline__ void in_registers(const Chunk<T> (&f)[N]) {
#pragma unroll
    for (int b = 0; b < N; ++b)
#pragma unroll
        for (int p = 0; p < Elem<T>::P; ++p) {
            const u32x4 v = __builtin_bit_cast(u32x4, f[b].p[p]);
            asm volatile("" : : "v"(v));
        }
}
// one row's operand, kept in registers: chunk (lane / 16) of each 32 values
template <class T> __device__ __forceinline__ void row_raw(Raw<T>& raw, const Rows<T>& s, int r, bool has, int b) {
    const int d0 = b * 32 + ((threadIdx.x & 63) >> 4) * 8, n = has ? s.dim - d0 : 0;
    load_raw(raw, n > 0 ? s.at(r) + d0 : s.p, n < 0 ? 0 : n > 8 ? 8 : n, s.vw);
}
template <class T, int DP> __device__ __forceinline__ void row_chunks(Chunk<T> (&f)[DP / 32], const Rows<T>& s, int r) {
    const bool has = s.has(r);
    Raw<T> raw[DP / 32];
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) row_raw(raw[b], s, r, has, b);
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) f[b] = raw_chunk(raw[b]);
}
__device__ __forceinline__ float raw_dot(const Raw<float>& a, const Raw<float>& b) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) s += a.a[j] * b.a[j] + a.b[j] * b.b[j];
    return s;
}
template <class T> __device__ __forceinline__ float raw_dot(const Raw<T>& a, const Raw<T>& b) {
    T x[8], y[8];
    __builtin_memcpy(x, &a, 16);
    __builtin_memcpy(y, &b, 16);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s += to_f(x[j]) * to_f(y[j]);
    return s;
}
// Of a block of 32 tile rows, row i of 16 x 16 subtile t is row 8 (i / 4) + 4 t + i % 4: lane group g then holds rows
// 8 g .. + 7 of the block, in order, in the results of t = 0 and 1 -- chunk g of the next product's operand.
__device__ __forceinline__ int sub_row(int t) {
    const int i = threadIdx.x & 15;
    return 32 * (t >> 1) + 8 * (i >> 2) + 4 * (t & 1) + (i & 3);
}
template <class T> __device__ __forceinline__ Chunk<T> joined(const f32x4& a, const f32x4& b) {
    const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return to_chunk(x, T());
}
// The weights as a matrix operand: rounded to the tensors' type where a wave has many products to do (f32: its three
// planes); for the small graphs of one wave with what the rounding leaves as a second operand, at no cost that shows.
template <class T, bool REST> struct Weights {
    Chunk<T> c, rest;
    __device__ __forceinline__ Weights() = default;
    __device__ __forceinline__ Weights(const f32x4& a, const f32x4& b) {
        c = joined<T>(a, b);
        if constexpr (REST) {
            f32x4 x = a, y = b;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] -= (float)c.p[0][e];
                y[e] -= (float)c.p[0][4 + e];
            }
            rest = joined<T>(x, y);
        }
    }
    __device__ __forceinline__ f32x4 times(const Chunk<T>& v, f32x4 acc) const {
        if constexpr (REST) acc = mma(v, rest, acc);
        return mma(v, c, acc);
    }
};
template <class T, int WAVES> constexpr bool att_rest() { return sizeof(T) == 2 && WAVES == 1; }
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// over the four lanes l % 16 + 0, 16, 32, 48
template <class F> __device__ __forceinline__ float over_groups(float v, F f) {
    uint32_t a = __builtin_bit_cast(uint32_t, v);
    auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    uint32_t x = r[0], y = r[1];
    a = __builtin_bit_cast(uint32_t, f(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y)));
    r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
    x = r[0], y = r[1];
    return f(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}
__device__ __forceinline__ float over_groups_max(float v) {
    return over_groups(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float over_groups_sum(float v) {
    return over_groups(v, [](float a, float b) { return a + b; });
}
// The power of two that a lane's dS (of one row or one key: the four lanes of it go together) are multiplied by: the largest so
// far lies in 2^14 .. 2^15, or below where it is less than 2^-86.  A larger one lowers it, and what is summed up so far with it.
struct DsScale {
    float by = 0x1p100f;
    __device__ __forceinline__ static float inverse(float power) {
        return __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, power));
    }
    template <int D> __device__ __forceinline__ void take(f32x4& a, f32x4& b, f32x4 (&acc)[D]) {
        float hi = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) hi = fmaxf(hi, fmaxf(fabsf(a[e]), fabsf(b[e])));
        if (__any(hi * by > 0x1p15f)) {
            const float top = over_groups_max(hi);
            const int e = 127 + 14 + 127 - (int)(__builtin_bit_cast(uint32_t, top) >> 23);  // 2^14 <= top 2^(e - 127) < 2^15
            const float to = __builtin_bit_cast(float, (uint32_t)(e < 27 ? 27 : e > 227 ? 227 : e) << 23);
            const float next = top * by > 0x1p15f ? to : by, ratio = next * inverse(by);
            by = next;
#pragma unroll
            for (int t = 0; t < D; ++t) acc[t] *= ratio;
        }
        a *= by;
        b *= by;
    }
};
template <class T>
__device__ __forceinline__ Rows<T> rows_of(const T* p, int64_t row, int64_t head, int start, int n, int first_head, int group,
                                           int dim, const uint8_t* mask, int vw) {
    return {p + (int64_t)start * row + (int64_t)first_head * head, row, head, n, group, dim,
            mask == nullptr ? nullptr : mask + start, vw};
}
// tiles of split z, in equal shares
__device__ __forceinline__ void split_range(int n, int tile, int splits, int z, int* b, int* e) {
    const int tiles = (n + tile - 1) / tile, per = (tiles + splits - 1) / splits;
    *b = z * per < tiles ? z * per : tiles;
    *e = (z + 1) * per < tiles ? (z + 1) * per : tiles;
}

// The tiles b .. e - 1 of one pair of row sets, one after the other in LDS: load(i, open, buffer) starts tile i's loads,
// step(i, open, buffer) is its work.  DMA: three buffers, two tiles under way; registers: one buffer (the planes of f32 take
// three times the room, and workgroups on a CU are worth more than the barrier saved), one tile under way.
// LOADS: the loads of a wave a tile.  ready() uses what was loaded to registers in front of the loop: the compiler would
// otherwise wait for it inside, and with it, every time, for the tiles under way.
template <int LOADS, bool DMA, class Open, class Load, class Store, class Ready, class Step>
__device__ __forceinline__ void over_tiles(int b, int e, Open open, Load load, Store store, Ready ready, Step step) {
    if (b >= e) return;
    if constexpr (DMA) {
        uint64_t m0 = open(b), m1 = b + 1 < e ? open(b + 1) : 0;
        load(b, m0, 0);
        if (b + 1 < e) load(b + 1, m1, 1);
        ready();
        int buf = 0;
        for (int i = b; i < e; ++i) {
            const uint64_t m2 = i + 2 < e ? open(i + 2) : 0;
            if (i + 1 < e) dma_wait<LOADS>();
            else dma_wait<0>();
            lds_barrier();
            if (i + 2 < e) load(i + 2, m2, buf == 0 ? 2 : buf - 1);
            step(i, m0, buf);
            m0 = m1;
            m1 = m2;
            buf = buf == 2 ? 0 : buf + 1;
        }
    } else {
        uint64_t m0 = open(b);
        load(b, m0, 0);
        for (int i = b; i < e; ++i) {
            if (i > b) __syncthreads();
            store(0);
            __syncthreads();
            const uint64_t m1 = i + 1 < e ? open(i + 1) : 0;
            if (i + 1 < e) load(i + 1, m1, 0);
            step(i, m0, 0);
            m0 = m1;
        }
    }
}
template <class T, bool FAST> constexpr int att_buffers() { return att_dma<T, FAST>() ? 3 : 1; }

// ---------------------------------------------------------------------------------------------
// forward: WAVES waves of 16 rows each share the key tiles (64 keys for the 16-bit types: three workgroups on a CU)
// ---------------------------------------------------------------------------------------------
template <class T, int DP, int WAVES, int KT, bool FAST>
__global__ __launch_bounds__(WAVES * 64) void att_fwd_kernel(AttDims d, const T* __restrict__ q, const T* __restrict__ k,
                                                             const T* __restrict__ v, T* __restrict__ out,
                                                             T* __restrict__ rest, float* __restrict__ lse,
                                                             float* __restrict__ part) {
    constexpr int NT = WAVES * 64, TR = WAVES * 16;
    using Stage = RowStage<T, KT, DP, NT, FAST, false>;
    using KTile = typename Stage::Lds;
    constexpr int BUF = 2 * KTile::BYTES;
    extern __shared__ __align__(16) char lds[];
    const int hgroups = (d.kv_heads + d.heads_a_wg - 1) / d.heads_a_wg;
    const Span sp = find_span(d, false, TR, d.group, blockIdx.x / hgroups);
    const int r0 = sp.tile * TR, nrows = (sp.qe - sp.qs) * d.group;
    if (r0 >= nrows) return;
    const int h0 = blockIdx.x % hgroups * d.heads_a_wg, h1 = h0 + d.heads_a_wg < d.kv_heads ? h0 + d.heads_a_wg : d.kv_heads;
    for (int hk = h0; hk < h1; ++hk) {
        if (hk > h0) lds_barrier();  // the tiles of the last head have been read
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
        const int row = r0 + wave * 16 + c;
        const Rows<T> qr = rows_of(q, d.q_row, d.q_head, sp.qs, nrows, hk * d.group, d.group, d.dim, (const uint8_t*)nullptr, d.qvw);
        const Rows<T> kr = rows_of(k, d.k_row, d.k_head, sp.ks, sp.ke - sp.ks, hk, 1, d.dim, d.mask, d.kvw);
        const Rows<T> vr = rows_of(v, d.v_row, d.v_head, sp.ks, sp.ke - sp.ks, hk, 1, d.dim, d.mask, d.vvw);
        Chunk<T> qf[DP / 32];
        f32x4 o[DP / 16];
        row_chunks<T, DP>(qf, qr, row);
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) o[t] = f32x4{0, 0, 0, 0};
        float m = -INFINITY, l = 0.f;
        Stage ks, vs;
        ks.init(kr);
        vs.init(vr);
        const uint32_t at_lds = lds_offset(lds);
        int first, last;
        split_range(kr.n, KT, d.splits, blockIdx.z, &first, &last);
        uint64_t* words = reinterpret_cast<uint64_t*>(lds + att_buffers<T, FAST>() * BUF);
        for (int tb = first; tb < last; tb += MASK_TILES) {
            const int te = tb + MASK_TILES < last ? tb + MASK_TILES : last;
            if (tb > first) lds_barrier();  // the last tiles have been read
            mask_words<WAVES, KT>(kr, tb, te, words);
            over_tiles<2 * Stage::U, Stage::DMA>(
                tb, te, [&](int i) { return mask_word<KT>(kr, i, tb, words); },
                [&](int i, uint64_t open, int buf) {
                    ks.load(kr, i, open, at_lds + buf * BUF);
                    vs.load(vr, i, open, at_lds + buf * BUF + KTile::BYTES);
                },
                [&](int buf) {
                    ks.store(lds + buf * BUF);
                    vs.store(lds + buf * BUF + KTile::BYTES);
                },
                [&]() { in_registers<T>(qf); },
                [&](int, uint64_t open, int buf) {
                    if (open == 0) return;  // nothing to attend to
                    const char* kl = lds + buf * BUF;
                    const char* vl = kl + KTile::BYTES;
                    f32x4 s[KT / 16];
#pragma unroll
                    for (int t = 0; t < KT / 16; ++t) {
                        s[t] = f32x4{0, 0, 0, 0};
#pragma unroll
                        for (int b = 0; b < DP / 32; ++b) {
                            const Chunk<T> kf = KTile::get(kl, sub_row(t), b * 4 + g);
                            s[t] = mma(kf, qf[b], s[t]);
                        }
                    }
                    if (KT == 64 ? open != ~0ull : (uint32_t)open != 0xffffffffu) {
                        // a closed key's score is as low as it gets: a sign-extended bit picks it (the scale may be negative)
                        const uint32_t closed = d.scale2 < 0.f ? 0x7f800000u : 0xff800000u;
#pragma unroll
                        for (int t = 0; t < KT / 16; ++t) {
                            const int bits = (int)(uint32_t)(open >> (32 * (t >> 1) + 8 * g + 4 * (t & 1)));
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe(bits, e, 1);
                                const float v = s[t][e];
                                s[t][e] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, v) & m) | (closed & ~m));
                            }
                        }
                    }
                    const float sc = d.scale2;
                    float hi = -INFINITY;
                    if (sc >= 0.f) {
#pragma unroll
                        for (int t = 0; t < KT / 16; ++t)
#pragma unroll
                            for (int e = 0; e < 4; ++e) hi = fmaxf(hi, s[t][e]);
                    } else {
#pragma unroll
                        for (int t = 0; t < KT / 16; ++t)
#pragma unroll
                            for (int e = 0; e < 4; ++e) hi = fmaxf(hi, -s[t][e]);
                    }
                    hi *= fabsf(sc);
                    // The weights are taken from a maximum that may lag behind by a factor of 2^LAG, which neither they nor their
                    // sum notice: most tiles then need no look at the other lanes and no scaling of what is summed up.
                    if (__any(hi > m + LAG)) {
                        const float top = fmaxf(m, over_groups_max(hi)), a = exp2_fast(m - (top == -INFINITY ? 0.f : top));
                        m = top;
                        l *= a;
#pragma unroll
                        for (int t = 0; t < DP / 16; ++t) o[t] *= a;
                    }
                    const float safe = (m == -INFINITY ? 0.f : m) - att_fwd_shift<T>();
#pragma unroll
                    for (int t = 0; t < KT / 16; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s[t][e] = exp2_fast(__builtin_fmaf(s[t][e], sc, -safe));
                            l += s[t][e];
                        }
#pragma unroll
                    for (int b = 0; b < KT / 32; ++b) {
                        const Weights<T, att_rest<T, WAVES>()> p = {s[2 * b], s[2 * b + 1]};
#pragma unroll
                        for (int t = 0; t < DP / 16; ++t) {
                            const Chunk<T> vf = KTile::get_across(vl, b * 32, t);
                            o[t] = p.times(vf, o[t]);
                        }
                    }
                });
        }
        const float ls = over_groups_sum(l);
        m -= att_fwd_shift<T>();  // (what the weights were taken from)
        if (row >= nrows) continue;
        const int qi = query_of(row, d.group);
        const int64_t at = (int64_t)(sp.qs + qi) * d.heads + hk * d.group + row - qi * d.group;
        if (d.splits > 1) {  // unnormalised sums and their statistics: att_join_kernel ends the work
            const int64_t all = (int64_t)d.rows_q * d.heads, i = blockIdx.z * all + at;
            float* po = part + i * d.dim;
#pragma unroll
            for (int t = 0; t < DP / 16; ++t) store4(po + t * 16 + g * 4, o[t], d.dim - t * 16 - g * 4, d.dim % 4 == 0);
            if (g == 0) {
                float* ps = part + d.splits * all * d.dim + 2 * i;
                ps[0] = m;
                ps[1] = ls;
            }
            continue;
        }
        const float inv = ls > 0.f ? __builtin_amdgcn_rcpf(ls) : ls == 0.f ? 0.f : ls;
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) {
            f32x4 v = o[t] * inv;
            store4(out + at * d.dim + t * 16 + g * 4, v, d.dim - t * 16 - g * 4, d.ovec);
            if (rest != nullptr) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] -= to_f((T)v[e]);
                store4(rest + at * d.dim + t * 16 + g * 4, v, d.dim - t * 16 - g * 4, d.ovec);
            }
        }
        if (lse != nullptr && g == 0) lse[at] = ls == 0.f ? INFINITY : m + __builtin_amdgcn_logf(ls);
    }
}

// The parts of a row: out = sum_z 2^(m_z - m) O_z / sum_z 2^(m_z - m) l_z, a thread a value, 256 a workgroup
template <class T>
__global__ __launch_bounds__(256) void att_join_kernel(int64_t all, int dim, int splits, const float* __restrict__ part,
                                                        T* __restrict__ out, T* __restrict__ rest, float* __restrict__ lse) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, at = i / dim;
    if (at >= all) return;
    const int e = (int)(i % dim);
    const float* stat = part + splits * all * dim;
    float m = -INFINITY;
#pragma unroll 8
    for (int z = 0; z < splits; ++z) m = fmaxf(m, stat[2 * (z * all + at)]);
    const float safe = m == -INFINITY ? 0.f : m;
    float l = 0.f, o = 0.f;
#pragma unroll 8
    for (int z = 0; z < splits; ++z) {
        const float a = exp2_fast(stat[2 * (z * all + at)] - safe);
        l += a * stat[2 * (z * all + at) + 1];
        o += a * part[(z * all + at) * dim + e];
    }
    const float v = l == 0.f ? 0.f : o / l;
    out[i] = (T)v;
    if (rest != nullptr) rest[i] = (T)(v - to_f((T)v));
    if (lse != nullptr && e == 0) lse[at] = l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
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
#pragma unroll 8
    for (int z = 0; z < splits; ++z) s += p[z * n + i];
    o[i] = (T)s;
}

// ---------------------------------------------------------------------------------------------
// dQ: the forward's tiles again, S and dP along their rows, dS K across them; delta = sum dO O on the way, of O and what its
// rounding left (of a rounded O alone, delta is off by up to 2^-9 sum |dO O| in bf16: as much as dS on rows with one large weight)
// ---------------------------------------------------------------------------------------------
template <class T, int DP, int WAVES, int KT, bool FAST>
__global__ __launch_bounds__(WAVES * 64) void att_dq_kernel(AttDims d, const T* __restrict__ q, const T* __restrict__ k,
                                                            const T* __restrict__ v, const T* __restrict__ out,
                                                            const T* __restrict__ rest, const T* __restrict__ dout,
                                                            const float* __restrict__ lse, float* __restrict__ delta,
                                                            T* __restrict__ dq, float* __restrict__ part) {
    constexpr int NT = WAVES * 64, TR = WAVES * 16;
    using Stage = RowStage<T, KT, DP, NT, FAST, false>;
    using KTile = typename Stage::Lds;
    constexpr int BUF = 2 * KTile::BYTES;
    extern __shared__ __align__(16) char lds[];
    const int hgroups = (d.kv_heads + d.heads_a_wg - 1) / d.heads_a_wg;
    const Span sp = find_span(d, false, TR, d.group, blockIdx.x / hgroups);
    const int r0 = sp.tile * TR, nrows = (sp.qe - sp.qs) * d.group;
    if (r0 >= nrows) return;
    const int h0 = blockIdx.x % hgroups * d.heads_a_wg, h1 = h0 + d.heads_a_wg < d.kv_heads ? h0 + d.heads_a_wg : d.kv_heads;
    for (int hk = h0; hk < h1; ++hk) {
        if (hk > h0) lds_barrier();  // the tiles of the last head have been read
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
        const int row = r0 + wave * 16 + c;
        const uint8_t* no = nullptr;
        const Rows<T> qr = rows_of(q, d.q_row, d.q_head, sp.qs, nrows, hk * d.group, d.group, d.dim, no, d.qvw);
        const Rows<T> gr = rows_of(dout, d.do_row, d.do_head, sp.qs, nrows, hk * d.group, d.group, d.dim, no, d.dovw);
        const Rows<T> orow = rows_of(out, (int64_t)d.heads * d.dim, d.dim, sp.qs, nrows, hk * d.group, d.group, d.dim, no,
                                     d.ovec ? 8 : 1);
        const Rows<T> kr = rows_of(k, d.k_row, d.k_head, sp.ks, sp.ke - sp.ks, hk, 1, d.dim, d.mask, d.kvw);
        const Rows<T> vr = rows_of(v, d.v_row, d.v_head, sp.ks, sp.ke - sp.ks, hk, 1, d.dim, d.mask, d.vvw);
        Chunk<T> qf[DP / 32], gf[DP / 32];
        f32x4 acc[DP / 16];
        const bool mine = row < nrows;
        row_chunks<T, DP>(qf, qr, row);
        float s = 0.f;
#pragma unroll
        for (int b = 0; b < DP / 32; ++b) {
            Raw<T> a, o;
            row_raw(a, gr, row, mine, b);
            row_raw(o, orow, row, mine, b);
            gf[b] = raw_chunk(a);
            s += raw_dot(a, o);
            if (rest != nullptr) {
                Rows<T> more = orow;
                more.p = rest + (orow.p - out);
                row_raw(o, more, row, mine, b);
                s += raw_dot(a, o);
            }
        }
        const float del = over_groups_sum(s);
        const int qi = mine ? query_of(row, d.group) : 0;
        const int64_t at = (int64_t)(sp.qs + qi) * d.heads + hk * d.group + (mine ? row - qi * d.group : 0);
        const float L = mine ? lse[at] : INFINITY;
        if (mine && g == 0 && blockIdx.z == 0) delta[at] = del;
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) acc[t] = f32x4{0, 0, 0, 0};
        DsScale scale;
        Stage ks, vs;
        ks.init(kr);
        vs.init(vr);
        const uint32_t at_lds = lds_offset(lds);
        int first, last;
        split_range(kr.n, KT, d.splits, blockIdx.z, &first, &last);
        uint64_t* words = reinterpret_cast<uint64_t*>(lds + att_buffers<T, FAST>() * BUF);
        int opened = 0;  // open keys of this share
        for (int tb = first; tb < last; tb += MASK_TILES) {
            const int te = tb + MASK_TILES < last ? tb + MASK_TILES : last;
            if (tb > first) lds_barrier();  // the last tiles have been read
            mask_words<WAVES, KT>(kr, tb, te, words);
            over_tiles<2 * Stage::U, Stage::DMA>(
                tb, te, [&](int i) { return mask_word<KT>(kr, i, tb, words); },
                [&](int i, uint64_t open, int buf) {
                    ks.load(kr, i, open, at_lds + buf * BUF);
                    vs.load(vr, i, open, at_lds + buf * BUF + KTile::BYTES);
                },
                [&](int buf) {
                    ks.store(lds + buf * BUF);
                    vs.store(lds + buf * BUF + KTile::BYTES);
                },
                [&]() {
                    in_registers<T>(qf);
                    in_registers<T>(gf);
                    asm volatile("" : : "v"(L));
                },
                [&](int, uint64_t open, int buf) {
                    if (open == 0) return;  // nothing to attend to
                    opened += __popcll(open);
                    const char* kl = lds + buf * BUF;
                    const char* vl = kl + KTile::BYTES;
#pragma unroll
                    for (int p = 0; p < KT / 32; ++p) {
                        f32x4 s[2], dp[2];
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            s[u] = dp[u] = f32x4{0, 0, 0, 0};
#pragma unroll
                            for (int b = 0; b < DP / 32; ++b) {
                                const Chunk<T> kf = KTile::get(kl, sub_row(2 * p + u), b * 4 + g);
                                const Chunk<T> vf = KTile::get(vl, sub_row(2 * p + u), b * 4 + g);
                                s[u] = mma(kf, qf[b], s[u]);
                                dp[u] = mma(vf, gf[b], dp[u]);
                            }
                        }
                        const int bits = (int)(uint32_t)(open >> (32 * p + 8 * g));
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float w = exp2_fast(__builtin_fmaf(s[u][e], d.scale2, -L)) * (dp[u][e] - del);
                                s[u][e] = __builtin_bit_cast(
                                    float, __builtin_bit_cast(uint32_t, w) & (uint32_t)__builtin_amdgcn_sbfe(bits, 4 * u + e, 1));
                            }
                        if constexpr (att_scaled<T>()) scale.take(s[0], s[1], acc);
                        const Weights<T, att_rest<T, WAVES>()> f = {s[0], s[1]};
#pragma unroll
                        for (int t = 0; t < DP / 16; ++t) {
                            const Chunk<T> kc = KTile::get_across(kl, p * 32, t);
                            acc[t] = f.times(kc, acc[t]);
                        }
                    }
                });
        }
        const float times = opened == 1 && (d.splits == 1 || one_open(kr)) ? 0.f : d.scale;
        if (!mine) continue;
        // a row without an open key has dQ = 0 whatever dO and O hold
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) {
            if constexpr (att_scaled<T>()) acc[t] *= DsScale::inverse(scale.by);
            const f32x4 r = L == INFINITY ? f32x4{0, 0, 0, 0} : acc[t] * times;
            const int n = d.dim - t * 16 - g * 4;
            if (d.splits > 1)
                store4(part + (blockIdx.z * (int64_t)d.rows_q * d.heads + at) * d.dim + t * 16 + g * 4, r, n, d.dim % 4 == 0);
            else
                store4(dq + at * d.dim + t * 16 + g * 4, r, n, d.ovec);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// dK, dV: WAVES waves of 16 keys each; all rows (of all heads that read the keys) go by in tiles of RT, with their L and delta
// ---------------------------------------------------------------------------------------------
template <class T, int DP, int WAVES, int RT, bool FAST>
__global__ __launch_bounds__(WAVES * 64) void att_dkv_kernel(AttDims d, const T* __restrict__ q, const T* __restrict__ k,
                                                             const T* __restrict__ v, const T* __restrict__ dout,
                                                             const float* __restrict__ lse, const float* __restrict__ delta,
                                                             T* __restrict__ dk, T* __restrict__ dv, float* __restrict__ part) {
    constexpr int NT = WAVES * 64, TK = WAVES * 16;
    using Stage = RowStage<T, RT, DP, NT, FAST, true>;
    using RTile = typename Stage::Lds;
    constexpr int STAT = 2 * RTile::BYTES, BUF = STAT + 2 * 64 * 4;  // Q, dO, then 64 values of L and of delta each
    constexpr int STATS = WAVES > 1 ? 1 : 2;                         // stat loads of a wave a tile
    extern __shared__ __align__(16) char lds[];
    const int hgroups = (d.kv_heads + d.heads_a_wg - 1) / d.heads_a_wg;
    const Span sp = find_span(d, true, TK, 1, blockIdx.x / hgroups);
    const int k0 = sp.tile * TK, nkeys = sp.ke - sp.ks, nrows = (sp.qe - sp.qs) * d.group;
    if (k0 >= nkeys) return;
    const int h0 = blockIdx.x % hgroups * d.heads_a_wg, h1 = h0 + d.heads_a_wg < d.kv_heads ? h0 + d.heads_a_wg : d.kv_heads;
    for (int hk = h0; hk < h1; ++hk) {
        if (hk > h0) lds_barrier();  // the tiles of the last head have been read
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
        const int key = k0 + wave * 16 + c;
        const uint8_t* no = nullptr;
        const Rows<T> qr = rows_of(q, d.q_row, d.q_head, sp.qs, nrows, hk * d.group, d.group, d.dim, no, d.qvw);
        const Rows<T> gr = rows_of(dout, d.do_row, d.do_head, sp.qs, nrows, hk * d.group, d.group, d.dim, no, d.dovw);
        const Rows<T> kr = rows_of(k, d.k_row, d.k_head, sp.ks, nkeys, hk, 1, d.dim, d.mask, d.kvw);
        const Rows<T> vr = rows_of(v, d.v_row, d.v_head, sp.ks, nkeys, hk, 1, d.dim, d.mask, d.vvw);
        // row r's statistics lie at (qs + r / group) heads + hk group + r % group
        const int64_t stat0 = (int64_t)sp.qs * d.heads + hk * d.group;
        auto stat_at = [&](int r) {
            const int qi = query_of(r, d.group);
            return (int64_t)qi * d.heads + r - qi * d.group;
        };
        Chunk<T> kf[DP / 32], vf[DP / 32];
        f32x4 ak[DP / 16], av[DP / 16];
        row_chunks<T, DP>(kf, kr, key);
        row_chunks<T, DP>(vf, vr, key);
        const bool open_key = kr.has(key);
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) ak[t] = av[t] = f32x4{0, 0, 0, 0};
        DsScale scale;
        Stage qs, gs;
        qs.init(qr);
        gs.init(gr);
        const uint32_t stat_off = (uint32_t)stat_at(lane % RT) * 4;  // in a tile of whole queries
        float stat_reg = 0.f;
        const uint32_t at_lds = lds_offset(lds);
        int tb, te;
        split_range(nrows, RT, d.splits, blockIdx.z, &tb, &te);
        static_assert(TK <= 64, "a word");
        const uint64_t any = kr.template open<TK>(k0);
        if (any == 0) te = tb;  // nobody attends to these keys
        over_tiles<2 * Stage::U + STATS, Stage::DMA>(
            tb, te, [&](int i) { return qr.there(i * RT); },
            [&](int i, uint64_t open, int buf) {
                qs.load(qr, i, open, at_lds + buf * BUF);
                gs.load(gr, i, open, at_lds + buf * BUF + RTile::BYTES);
                // a missing row: its Q, dO, L and delta are zeros, and so is what it adds
                if constexpr (Stage::DMA) {
                    const int64_t first = qs.queries > 0 ? (int64_t)(i * qs.queries) * d.heads : stat_at(i * RT);
                    uint32_t off = qs.queries > 0 ? stat_off : (uint32_t)((stat_at(i * RT + lane % RT) - first) * 4);
                    off = (open >> lane & 1) && lane < RT ? off : DMA_NOWHERE;
#pragma unroll
                    for (int w = 0; w < STATS; ++w) {
                        const int which = STATS == 2 ? w : wave & 1;
                        dma_load4(dma_buffer((which ? delta : lse) + stat0 + first), off, at_lds + buf * BUF + STAT + which * 256);
                    }
                } else {
                    // Without a branch: at the join behind one the compiler has put a register away while the lanes that stay
                    // out of it were still switched off (tools/check_spills.py).
                    // Two waves load one of the two each; one wave loads both (both in each of four waves: dK and dV of 1024 graphs
                    // of 64, 8 heads of 32, 131 -> 121 us).
                    static_assert(RT == 32, "half a wave");
                    const int r = lane % RT;
                    const int64_t first = stat_at(i * RT);
                    const uint32_t gone = (uint32_t)(~open >> r) << 31;  // DMA_NOWHERE and beyond
                    const uint32_t off = (uint32_t)((stat_at(i * RT + r) - first) * 4) | gone;
                    if constexpr (STATS == 1) {
                        stat_reg = buffer_load1(dma_buffer((wave & 1 ? delta : lse) + stat0 + first), off);
                    } else {
                        const float l = buffer_load1(dma_buffer(lse + stat0 + first), off);
                        const float del = buffer_load1(dma_buffer(delta + stat0 + first), off);
                        stat_reg = lane / RT ? del : l;
                    }
                }
            },
            [&](int buf) {
                qs.store(lds + buf * BUF);
                gs.store(lds + buf * BUF + RTile::BYTES);
                if (!Stage::DMA && wave < 2)
                    reinterpret_cast<float*>(lds + buf * BUF + STAT)[STATS == 1 ? threadIdx.x : lane / RT * 64 + lane % RT] = stat_reg;
            },
            [&]() {
                in_registers<T>(kf);
                in_registers<T>(vf);
            },
            [&](int, uint64_t open, int buf) {
                const char* ql = lds + buf * BUF;
                const char* gl = ql + RTile::BYTES;
                const float* stat = reinterpret_cast<const float*>(ql + STAT);
#pragma unroll
                for (int p = 0; p < RT / 32; ++p) {
                    f32x4 s[2], dp[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        s[u] = dp[u] = f32x4{0, 0, 0, 0};
#pragma unroll
                        for (int b = 0; b < DP / 32; ++b) {
                            const Chunk<T> qf = RTile::get(ql, sub_row(2 * p + u), b * 4 + g);
                            const Chunk<T> gf = RTile::get(gl, sub_row(2 * p + u), b * 4 + g);
                            s[u] = mma(qf, kf[b], s[u]);
                            dp[u] = mma(gf, vf[b], dp[u]);
                        }
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const f32x4 L = *reinterpret_cast<const f32x4*>(stat + 32 * p + 8 * g + 4 * u);
                        const f32x4 del = *reinterpret_cast<const f32x4*>(stat + 64 + 32 * p + 8 * g + 4 * u);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float from = att_scaled<T>() ? att_dkv_shift<T>() - L[e] : -L[e];
                            const float w = exp2_fast(__builtin_fmaf(s[u][e], d.scale2, from));
                            s[u][e] = w;
                            dp[u][e] = w * (dp[u][e] - del[e]);
                        }
                    }
                    if ((uint32_t)(open >> (32 * p)) != 0xffffffffu) {  // what zeros make of infinite keys is no row's
                        const int bits = (int)(uint32_t)(open >> (32 * p + 8 * g));
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe(bits, 4 * u + e, 1);
                                const float w = s[u][e], ds = dp[u][e];
                                s[u][e] = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, w) & m);
                                dp[u][e] = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, ds) & m);
                            }
                    }
                    if constexpr (att_scaled<T>()) scale.take(dp[0], dp[1], ak);
                    const Weights<T, att_rest<T, WAVES>()> pf = {s[0], s[1]}, df = {dp[0], dp[1]};
#pragma unroll
                    for (int t = 0; t < DP / 16; ++t) {
                        const Chunk<T> gc = RTile::get_across(gl, p * 32, t);
                        av[t] = pf.times(gc, av[t]);
                        const Chunk<T> qc = RTile::get_across(ql, p * 32, t);
                        ak[t] = df.times(qc, ak[t]);
                    }
                }
            });
        const int64_t all = (int64_t)d.rows_k * d.kv_heads;
        const float times = any != 0 && (any & (any - 1)) == 0 && one_open(kr) ? 0.f : d.scale;
        if (key >= nkeys) continue;
        const int64_t at = (int64_t)(sp.ks + key) * d.kv_heads + hk;
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) {
            const int y = t * 16 + g * 4, n = d.dim - y;
            if constexpr (att_scaled<T>()) {
                av[t] *= 0x1p-15f;  // 2^-att_dkv_shift, which dS has too
                ak[t] *= DsScale::inverse(scale.by) * 0x1p-15f;
            }
            // a masked key's gradients are 0 whatever the rows that do not read it hold (a lane's sums are one key's)
            const f32x4 zero = {0, 0, 0, 0}, rk = open_key ? ak[t] * times : zero, rv = open_key ? av[t] : zero;
            if (d.splits > 1) {
                store4(part + (blockIdx.z * all + at) * d.dim + y, rk, n, d.dim % 4 == 0);
                store4(part + ((d.splits + blockIdx.z) * all + at) * d.dim + y, rv, n, d.dim % 4 == 0);
            } else {
                store4(dk + at * d.dim + y, rk, n, d.ovec);
                store4(dv + at * d.dim + y, rv, n, d.ovec);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
// How a side (queries of all heads of a group, or keys) is cut into tiles
enum { SIDE_16, SIDE_64 };
static const int SIDE_ROWS[2] = {16, 64};
// One wave of 16 rows where the graphs are small (its tile is filled at least as well as one of 64 rows), four waves that share
// the other side's tiles otherwise.  (32 rows a wave read a tile half as often, but two workgroups less fit a CU: 145 us
// against 105 for the forward of 4 graphs of 1000 .. 2000 nodes, 8 heads of 128 bf16 values.)  Values that no 16-byte load
// fits have the second instance alone.
static int att_side(int64_t rows, int graphs, bool aligned) {
    return aligned && rows <= 32 * (int64_t)(graphs < 1 ? 1 : graphs) ? SIDE_16 : SIDE_64;
}
// Workgroups of a launch.  Where there are many, each goes over several key heads: looking the graph up, and the workgroups
// that find no tile, are then paid for less often.
static int att_grid(AttDims& d, int64_t rows, int tile) {
    const int64_t slots = (rows + (int64_t)(d.graphs + 2) * (tile - 1)) / tile;
    d.graph_of_slot = (float)(d.graphs + 2) / (float)(slots > 0 ? slots : 1);
    d.heads_a_wg = 1;
    while (d.heads_a_wg < d.kv_heads && slots * d.splits * (d.kv_heads / (2 * d.heads_a_wg)) >= 2048) d.heads_a_wg *= 2;
    return (int)(slots * ((d.kv_heads + d.heads_a_wg - 1) / d.heads_a_wg));
}
// Shares of the other side's tiles: so many waves for the 1024 SIMDs as `target`, and 256 rows a share at least.
static int att_splits(int64_t waves, int64_t other, int graphs, int target) {
    const int64_t want = target / (waves < 1 ? 1 : waves), most = other / (graphs < 1 ? 1 : graphs) / 256;
    const int64_t s = want < most ? want : most;
    return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

static int att_width(const void* p, int64_t row, int64_t head, int dim, int es) {
    int w = load_width(es, dim, row, p);
    while (w > 1 && head % w != 0) w /= 2;
    return w;
}
// 16-byte loads, and what a tile spans within the 2 GiB that a buffer's offsets reach
static bool att_aligned(const tsd_attention& a, const void* dout, int64_t do_row, int64_t do_head) {
    const int es = a.dtype == TSD_F32 ? 4 : 2, group = a.heads / a.kv_heads;
    auto near = [&](int64_t row, int64_t head) { return row >= 0 && head >= 0 && 65 * row + group * head < (1ll << 29); };
    return att_width(a.q, a.q_row, a.q_head, a.dim, es) == 8 && att_width(a.k, a.k_row, a.k_head, a.dim, es) == 8 &&
           att_width(a.v, a.v_row, a.v_head, a.dim, es) == 8 && near(a.q_row, a.q_head) && near(a.k_row, a.k_head) &&
           near(a.v_row, a.v_head) &&
           (dout == nullptr || (att_width(dout, do_row, do_head, a.dim, es) == 8 && near(do_row, do_head)));
}

struct AttPlan {
    int side_q, side_k, splits_q, splits_k;  // tiles; shares of the keys (forward, dQ) and of the rows (dK, dV)
    size_t fwd, bwd;                         // scratch floats
    size_t part;                             // where the backward's parts begin (behind delta)
};
// (the sizes of the scratch do not depend on strides or addresses: the query function sees the same)
static AttPlan att_plan(const tsd_attention& a, bool aligned) {
    AttPlan p = {};
    const int group = a.heads / a.kv_heads;
    const int64_t rows = (int64_t)a.num_queries * group, keys = a.num_keys;
    auto waves = [&](int64_t n) {
        const int side = att_side(n, a.num_graphs, true);
        return (n / SIDE_ROWS[side] + a.num_graphs) * a.kv_heads * (side == SIDE_16 ? 1 : 4);
    };
    p.side_q = att_side(rows, a.num_graphs, aligned);
    p.side_k = att_side(keys, a.num_graphs, aligned);
    p.splits_q = att_splits(waves(rows), keys, a.num_graphs, 2048);
    p.splits_k = att_splits(waves(keys), rows, a.num_graphs, 4096);
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
    if (a->dim > TSD_ATTENTION_MAX_DIM || (int64_t)a->num_queries * a->heads > (1 << 29) ||
        (int64_t)a->num_keys * a->heads > (1 << 29) || (int64_t)a->num_graphs * a->kv_heads > (1 << 22) || a->heads > (1 << 16)) {
        set_error("%s: head dim %d (at most %d), %d queries, %d keys, %d heads, %d graphs", name, a->dim, TSD_ATTENTION_MAX_DIM,
                  a->num_queries, a->num_keys, a->heads, a->num_graphs);
        return TSD_ERR_UNSUPPORTED;
    }
    TSD_REQUIRE(a->q_ptr != nullptr && a->k_ptr != nullptr, "%s: null offsets", name);
    TSD_REQUIRE(a->num_queries == 0 || a->q != nullptr, "%s: null pointer", name);
    TSD_REQUIRE(a->num_keys == 0 || (a->k != nullptr && a->v != nullptr), "%s: null pointer", name);
    return TSD_OK;
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
    if (d.scale2 == 0.f) d.scale2 = 0x1p-126f;  // (a closed key's infinite score stays one, every other score vanishes)
    d.qvw = att_width(a.q, a.q_row, a.q_head, a.dim, es);
    d.kvw = att_width(a.k, a.k_row, a.k_head, a.dim, es);
    d.vvw = att_width(a.v, a.v_row, a.v_head, a.dim, es);
    d.q_ptr = a.q_ptr;
    d.k_ptr = a.k_ptr;
    d.mask = a.key_mask;
    return d;
}

// rows of a tile of the other side: what keeps three workgroups on a CU
template <class T, int DP, int WAVES> constexpr int att_tile() { return WAVES == 1 || DP == 128 || sizeof(T) == 4 ? 32 : 64; }
template <class T, int DP, int WAVES, bool FAST>
static int att_launch_fwd(AttDims d, const tsd_attention& a, T* out, T* rest, float* lse, float* scratch, hipStream_t st) {
    constexpr int KT = att_tile<T, DP, WAVES>();
    constexpr int lds = att_buffers<T, FAST>() * 2 * Tile<T, KT, DP / 8>::BYTES + MASK_BYTES;
    static DeviceOnce once;
    auto k = att_fwd_kernel<T, DP, WAVES, KT, FAST>;
    const int rc = allow_lds(k, lds, once);
    if (rc != TSD_OK) return rc;
    hipLaunchKernelGGL(k, dim3(att_grid(d, (int64_t)d.rows_q * d.group, WAVES * 16), 1, d.splits), dim3(WAVES * 64), lds, st, d,
                       (const T*)a.q, (const T*)a.k, (const T*)a.v, out, rest, lse, scratch);
    TSD_LAUNCH_CHECK("attention_fwd");
    return TSD_OK;
}
template <class T, int DP, int WAVES, bool FAST>
static int att_launch_dq(AttDims d, const tsd_attention& a, const T* out, const T* rest, const T* dout, const float* lse,
                         float* delta, T* dq, float* part, hipStream_t st) {
    constexpr int KT = att_tile<T, DP, WAVES>();
    constexpr int lds = att_buffers<T, FAST>() * 2 * Tile<T, KT, DP / 8>::BYTES + MASK_BYTES;
    static DeviceOnce once;
    auto k = att_dq_kernel<T, DP, WAVES, KT, FAST>;
    const int rc = allow_lds(k, lds, once);
    if (rc != TSD_OK) return rc;
    hipLaunchKernelGGL(k, dim3(att_grid(d, (int64_t)d.rows_q * d.group, WAVES * 16), 1, d.splits), dim3(WAVES * 64), lds, st, d,
                       (const T*)a.q, (const T*)a.k, (const T*)a.v, out, rest, dout, lse, delta, dq, part);
    TSD_LAUNCH_CHECK("attention_dq");
    return TSD_OK;
}
template <class T, int DP, int WAVES, bool FAST>
static int att_launch_dkv(AttDims d, const tsd_attention& a, const T* dout, const float* lse, const float* delta, T* dk, T* dv,
                          float* part, hipStream_t st) {
    constexpr int RT = 32;
    constexpr int lds = att_buffers<T, FAST>() * (2 * Tile<T, RT, DP / 8>::BYTES + 512);
    static DeviceOnce once;
    auto k = att_dkv_kernel<T, DP, WAVES, RT, FAST>;
    const int rc = allow_lds(k, lds, once);
    if (rc != TSD_OK) return rc;
    hipLaunchKernelGGL(k, dim3(att_grid(d, d.rows_k, WAVES * 16), 1, d.splits), dim3(WAVES * 64), lds, st, d,
                       (const T*)a.q, (const T*)a.k, (const T*)a.v, dout, lse, delta, dk, dv, part);
    TSD_LAUNCH_CHECK("attention_dkv");
    return TSD_OK;
}
// launch<T, DP, waves, FAST> of a side
#define ATT_BY_SIDE(rc, side, aligned, launch, ...)                           \
    if (!(aligned)) rc = launch<T, DP, 4, false>(__VA_ARGS__);                \
    else if (side == SIDE_16) rc = launch<T, DP, 1, true>(__VA_ARGS__);       \
    else rc = launch<T, DP, 4, true>(__VA_ARGS__);

template <class T, int DP>
static int att_fwd(AttDims d, const tsd_attention& a, void* out, void* rest, float* lse, float* scratch, hipStream_t st) {
    const bool aligned = att_aligned(a, nullptr, 0, 0);
    const AttPlan p = att_plan(a, aligned);
    d.splits = p.splits_q;
    d.ovec = d.dim % 4 == 0 && aligned16(out) && aligned16(rest);
    int rc;
    ATT_BY_SIDE(rc, p.side_q, aligned, att_launch_fwd, d, a, (T*)out, (T*)rest, lse, scratch, st);
    if (rc == TSD_OK && d.splits > 1) {
        const int64_t all = (int64_t)d.rows_q * d.heads;
        hipLaunchKernelGGL(att_join_kernel<T>, dim3((unsigned)((all * d.dim + 255) / 256)), dim3(256), 0, st, all, d.dim, d.splits,
                           scratch, (T*)out, (T*)rest, lse);
        TSD_LAUNCH_CHECK("attention_join");
    }
    return rc;
}
template <class T, int DP>
static int att_bwd(AttDims d, const tsd_attention& a, const void* out, const void* rest, const void* dout, int64_t do_row,
                   int64_t do_head, const float* lse, void* dq, void* dk, void* dv, float* scratch, hipStream_t st) {
    const bool aligned = att_aligned(a, dout, do_row, do_head);
    const AttPlan p = att_plan(a, aligned);
    float *delta = scratch, *part = scratch + p.part;
    d.do_row = do_row;
    d.do_head = do_head;
    d.dovw = att_width(dout, do_row, do_head, d.dim, sizeof(T));
    d.ovec = d.dim % 8 == 0 && aligned16(out) && aligned16(rest) && aligned16(dq) && aligned16(dk) && aligned16(dv);
    int rc = TSD_OK;
    if (d.rows_q > 0) {
        d.splits = p.splits_q;
        ATT_BY_SIDE(rc, p.side_q, aligned, att_launch_dq, d, a, (const T*)out, (const T*)rest, (const T*)dout, lse, delta, (T*)dq, part,
                    st);
        if (rc == TSD_OK && d.splits > 1) {
            const int64_t n = (int64_t)d.rows_q * d.heads * d.dim;
            hipLaunchKernelGGL(att_sum_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, n, d.splits, part, (T*)dq,
                               (const float*)nullptr, (T*)nullptr);
            TSD_LAUNCH_CHECK("attention_dq_sum");
        }
    }
    if (rc == TSD_OK && d.rows_k > 0) {
        d.splits = p.splits_k;
        ATT_BY_SIDE(rc, p.side_k, aligned, att_launch_dkv, d, a, (const T*)dout, lse, delta, (T*)dk, (T*)dv, part, st);
        if (rc == TSD_OK && d.splits > 1) {
            const int64_t n = (int64_t)d.rows_k * d.kv_heads * d.dim;
            hipLaunchKernelGGL(att_sum_kernel<T>, dim3((unsigned)((n + 255) / 256), 2), dim3(256), 0, st, n, d.splits, part, (T*)dk,
                               part + d.splits * n, (T*)dv);
            TSD_LAUNCH_CHECK("attention_dkv_sum");
        }
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
    const AttPlan p = att_plan(*a, true);
    return backward ? p.bwd : p.fwd;
}

int tsd_graph_attention_fwd(const tsd_attention* a, void* out, void* out_rest, float* lse, float* scratch, size_t scratch_floats,
                            void* stream) {
    const int rc = att_check("tsd_graph_attention_fwd", a);
    if (rc != TSD_OK) return rc;
    if (a->num_queries == 0) return TSD_OK;
    const AttPlan p = att_plan(*a, true);
    TSD_REQUIRE(out != nullptr, "tsd_graph_attention_fwd: null pointer");
    TSD_REQUIRE(p.fwd == 0 || (scratch != nullptr && aligned16(scratch) && scratch_floats >= p.fwd),
                "tsd_graph_attention_fwd: scratch of %zu floats, %zu needed (16-byte aligned)", scratch_floats, p.fwd);
    const AttDims d = att_dims(*a);
    hipStream_t st = (hipStream_t)stream;
    TSD_BY_DTYPE(a->dtype, T, {
        if (d.dim <= 32) return att_fwd<T, 32>(d, *a, out, out_rest, lse, scratch, st);
        if (d.dim <= 64) return att_fwd<T, 64>(d, *a, out, out_rest, lse, scratch, st);
        return att_fwd<T, 128>(d, *a, out, out_rest, lse, scratch, st);
    });
    return TSD_OK;
}

int tsd_graph_attention_bwd(const tsd_attention* a, const void* out, const void* out_rest, const float* lse, const void* dout,
                            int64_t do_row, int64_t do_head, void* dq, void* dk, void* dv, float* scratch, size_t scratch_floats, void* stream) {
    const int rc = att_check("tsd_graph_attention_bwd", a);
    if (rc != TSD_OK) return rc;
    const AttPlan p = att_plan(*a, true);
    TSD_REQUIRE(a->num_queries == 0 || (out != nullptr && lse != nullptr && dout != nullptr && dq != nullptr),
                "tsd_graph_attention_bwd: null pointer");
    TSD_REQUIRE(a->num_keys == 0 || (dk != nullptr && dv != nullptr), "tsd_graph_attention_bwd: null pointer");
    TSD_REQUIRE(scratch != nullptr ? aligned16(scratch) && scratch_floats >= p.bwd : p.bwd == 0,
                "tsd_graph_attention_bwd: scratch of %zu floats, %zu needed (16-byte aligned)", scratch_floats, p.bwd);
    const AttDims d = att_dims(*a);
    hipStream_t st = (hipStream_t)stream;
    TSD_BY_DTYPE(a->dtype, T, {
        if (d.dim <= 32) return att_bwd<T, 32>(d, *a, out, out_rest, dout, do_row, do_head, lse, dq, dk, dv, scratch, st);
        if (d.dim <= 64) return att_bwd<T, 64>(d, *a, out, out_rest, dout, do_row, do_head, lse, dq, dk, dv, scratch, st);
        return att_bwd<T, 128>(d, *a, out, out_rest, dout, do_row, do_head, lse, dq, dk, dv, scratch, st);
    });
    return TSD_OK;
}

}  // extern "C"
