// block_tile.hpp -- element types, operand tiles and the MFMA step shared by the kernels of an attention block
// (kernels_gated.hip, kernels_attention.hip): f32, bf16 and f16 tensors, fp32 accumulation everywhere.
//
// One matrix instruction takes 16 x 16 outputs and 32 steps of the contraction: lane l holds 8 consecutive steps
// (l / 16) * 8 .. + 7 of row l % 16 of either operand, and of the result the four rows (l / 16) * 4 .. + 3 of column
// l % 16.  bf16 and f16 operands go in as they are.  An f32 operand goes in as THREE bf16 planes, x = hi + mid + lo
// (8 + 8 + 8 bits, each the rounded rest of the one before): six of the nine plane products, smallest first, leave
// 2^-24 of a product out.  bf16 has the exponents of f32, so nothing has to be scaled, unlike f16 planes, and the largest
// values, which would round to infinity, have the largest bf16 as their first plane; a rate of 1/6 of the bf16 pipes is 2.6
// times that of the f32 matrix instruction.  (A non-finite f32 operand comes out as NaN: inf - inf in the split.)
#pragma once
#include "common.hpp"

namespace tsd {
namespace blk {

using bf16 = __bf16;
using f16 = _Float16;
using bf16x8 = bf16 __attribute__((ext_vector_type(8)));
using f16x8 = f16 __attribute__((ext_vector_type(8)));
using u32x4 = uint32_t __attribute__((ext_vector_type(4)));
using f32x2 = float __attribute__((ext_vector_type(2)));
using bf16x2 = bf16 __attribute__((ext_vector_type(2)));

// Chunk<T>: 8 values of the contraction, as matrix operands (P planes of 16 bytes)
template <class T> struct Elem;
template <> struct Elem<bf16> {
    static constexpr int P = 1;
    using vec = bf16x8;
};
template <> struct Elem<f16> {
    static constexpr int P = 1;
    using vec = f16x8;
};
template <> struct Elem<float> {
    static constexpr int P = 3;
    using vec = bf16x8;
};
template <class T> struct Chunk {
    typename Elem<T>::vec p[Elem<T>::P];
};

__device__ __forceinline__ Chunk<bf16> to_chunk(const float (&x)[8], bf16) {
    Chunk<bf16> c;
#pragma unroll
    for (int j = 0; j < 8; ++j) c.p[0][j] = (bf16)x[j];
    return c;
}
__device__ __forceinline__ Chunk<f16> to_chunk(const float (&x)[8], f16) {
    Chunk<f16> c;
#pragma unroll
    for (int j = 0; j < 8; ++j) c.p[0][j] = (f16)x[j];
    return c;
}
constexpr float BF16_MAX = 0x1.FEp127f;
// (ANY: values as they come from memory; weights and their gradients are far from the largest.  The limit on the first plane
// costs 1 to 2 % of the f32 launches: gated 30000 x 256 -> 2 x 1024, training, 716 -> 732 us.)
template <bool ANY> __device__ __forceinline__ Chunk<float> to_planes(const float (&x)[8]) {
    Chunk<float> c;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        f32x2 r = {x[j], x[j + 1]};
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            f32x2 v = r;
            if (ANY && p == 0) v = {__builtin_amdgcn_fmed3f(r[0], -BF16_MAX, BF16_MAX), __builtin_amdgcn_fmed3f(r[1], -BF16_MAX, BF16_MAX)};
            const bf16x2 h = __builtin_convertvector(v, bf16x2);
            c.p[p][j] = h[0];
            c.p[p][j + 1] = h[1];
            r[0] -= (float)h[0];
            r[1] -= (float)h[1];
        }
    }
    return c;
}

__device__ __forceinline__ Chunk<float> to_chunk(const float (&x)[8], float) { return to_planes<false>(x); }

__device__ __forceinline__ f32x4 mma(const Chunk<bf16>& a, const Chunk<bf16>& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[0], b.p[0], c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(const Chunk<f16>& a, const Chunk<f16>& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.p[0], b.p[0], c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(const Chunk<float>& a, const Chunk<float>& b, f32x4 c) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[2], b.p[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[0], b.p[2], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[1], b.p[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[1], b.p[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[0], b.p[1], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[0], b.p[0], c, 0, 0, 0);
}

// ---------------------------------------------------------------------------------------------
// Raw<T>: 8 values as they come from memory.  load_raw reads `n` of them (0 .. 8) and leaves zeros behind.
// ---------------------------------------------------------------------------------------------
template <class T> struct Raw;
template <> struct Raw<float> {
    f32x4 a, b;
};
template <> struct Raw<bf16> {
    u32x4 a;
};
template <> struct Raw<f16> {
    u32x4 a;
};
__device__ __forceinline__ void raw_zero(Raw<float>& r) { r.a = r.b = f32x4{0, 0, 0, 0}; }
__device__ __forceinline__ void raw_zero(Raw<bf16>& r) { r.a = u32x4{0, 0, 0, 0}; }
__device__ __forceinline__ void raw_zero(Raw<f16>& r) { r.a = u32x4{0, 0, 0, 0}; }
__device__ __forceinline__ void raw_load8(Raw<float>& r, const float* p) {
    r.a = *reinterpret_cast<const f32x4*>(p);
    r.b = *reinterpret_cast<const f32x4*>(p + 4);
}
__device__ __forceinline__ void raw_load8(Raw<bf16>& r, const bf16* p) { r.a = *reinterpret_cast<const u32x4*>(p); }
__device__ __forceinline__ void raw_load8(Raw<f16>& r, const f16* p) { r.a = *reinterpret_cast<const u32x4*>(p); }
__device__ __forceinline__ void raw_put(Raw<float>& r, int j, float v) { (j < 4 ? r.a : r.b)[j & 3] = v; }
template <class T> __device__ __forceinline__ uint32_t bits16(T v) {
    uint16_t b;
    __builtin_memcpy(&b, &v, 2);
    return b;
}
template <class T> __device__ __forceinline__ void raw_put16(u32x4& a, int j, T v) {
    a[j >> 1] |= bits16(v) << (16 * (j & 1));
}
__device__ __forceinline__ void raw_put(Raw<bf16>& r, int j, bf16 v) { raw_put16(r.a, j, v); }
__device__ __forceinline__ void raw_put(Raw<f16>& r, int j, f16 v) { raw_put16(r.a, j, v); }

// vw: values a load may take (p aligned to as many, n a multiple of it): 8, 4, 2 or 1
template <class T> __device__ __forceinline__ void load_raw(Raw<T>& r, const T* __restrict__ p, int n, int vw) {
    raw_zero(r);
    if constexpr (sizeof(T) == 2) {
        if (vw == 8) {
            if (n > 0) raw_load8(r, p);
        } else if (vw == 4) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (4 * j < n) {
                    const uint2 v = *reinterpret_cast<const uint2*>(p + 4 * j);
                    r.a[2 * j] = v.x;
                    r.a[2 * j + 1] = v.y;
                }
        } else if (vw == 2) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (2 * j < n) r.a[j] = *reinterpret_cast<const uint32_t*>(p + 2 * j);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < n) raw_put(r, j, p[j]);
        }
    } else {
        if (vw >= 4) {
            if (n > 0) r.a = *reinterpret_cast<const f32x4*>(p);
            if (n > 4) r.b = *reinterpret_cast<const f32x4*>(p + 4);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < n) raw_put(r, j, p[j]);
        }
    }
}
// the widest such load for rows of `n` values `ld` apart from p on (strides of further dimensions: any common factor of ld)
inline int load_width(size_t size, int64_t n, int64_t ld, const void* p) {
    for (int v = 8; v > 1; v /= 2)
        if (n % v == 0 && ld % v == 0 && (reinterpret_cast<uintptr_t>(p) & (v * size < 16 ? v * size - 1 : 15)) == 0) return v;
    return 1;
}
__device__ __forceinline__ Chunk<bf16> raw_chunk(const Raw<bf16>& r) {
    Chunk<bf16> c;
    c.p[0] = __builtin_bit_cast(bf16x8, r.a);
    return c;
}
__device__ __forceinline__ Chunk<f16> raw_chunk(const Raw<f16>& r) {
    Chunk<f16> c;
    c.p[0] = __builtin_bit_cast(f16x8, r.a);
    return c;
}
__device__ __forceinline__ Chunk<float> raw_chunk(const Raw<float>& r) {
    const float x[8] = {r.a[0], r.a[1], r.a[2], r.a[3], r.b[0], r.b[1], r.b[2], r.b[3]};
    return to_planes<true>(x);
}

// ---------------------------------------------------------------------------------------------
// An operand tile in LDS: P planes of ROWS rows of C chunks (16 bytes each).  It is read along its rows (get: chunk c of
// row r) or across them (get_across: 8 rows of one column, by the LDS's transposing read), so a tensor is brought in as it
// lies in memory whichever way a product goes over it.  Chunk c of row r lies at place c ^ swizzle(r): 16 lanes that read
// one chunk of 16 rows (consecutive ones, or 0-3, 8-11, 16-19, 24-27) touch all 64 banks once, and so do the 32 lanes
// that read two chunks of rows 0-3 and 8-11 across.
// ---------------------------------------------------------------------------------------------
using s16x4 = short __attribute__((ext_vector_type(4)));
using s16x8 = short __attribute__((ext_vector_type(8)));
template <class T, int ROWS_, int C_> struct Tile {
    static constexpr int ROWS = ROWS_, C = C_;
    static_assert(C == 4 || C == 8 || C == 16 || C == 32, "chunks of a row");
    static constexpr int P = Elem<T>::P;
    static constexpr int PLANE = ROWS * C * 16, BYTES = P * PLANE;
    using vec = typename Elem<T>::vec;
    __device__ __forceinline__ static int swizzle(int r) {
        const int low = ((r >> 2) ^ (r >> 4)) & 1, b3 = (r >> 3) & 1;
        if constexpr (C >= 16) return low | (r & 3) << 1 | b3 << 3;
        if constexpr (C == 8) return low | ((r >> 1) & 1) << 1 | b3 << 2;
        return low | b3 << 1;
    }
    __device__ __forceinline__ static int at(int row, int c) { return (row * C + (c ^ swizzle(row))) * 16; }
    __device__ __forceinline__ static void put(char* lds, int row, int c, const Chunk<T>& v) {
        const int o = at(row, c);
#pragma unroll
        for (int p = 0; p < P; ++p) *reinterpret_cast<vec*>(lds + p * PLANE + o) = v.p[p];
    }
    __device__ __forceinline__ static Chunk<T> get(const char* lds, int row, int c) {
        Chunk<T> v;
        const int o = at(row, c);
#pragma unroll
        for (int p = 0; p < P; ++p) v.p[p] = *reinterpret_cast<const vec*>(lds + p * PLANE + o);
        return v;
    }
    // rows row0 + 8 (lane / 16) .. + 7 of column 16 t + lane % 16; row0 a multiple of 32
    __device__ __forceinline__ static Chunk<T> get_across(const char* lds, int row0, int t) {
        typedef __attribute__((address_space(3))) s16x4* lds4;
        const int lane = threadIdx.x & 63, i = lane & 15, r = row0 + (lane >> 4) * 8 + (i >> 2), c = 2 * t + ((i & 3) >> 1);
        const int o0 = at(r, c) + (i & 1) * 8, o1 = at(r + 4, c) + (i & 1) * 8;
        Chunk<T> v;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(lds + p * PLANE + o0));
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(lds + p * PLANE + o1));
            v.p[p] = __builtin_bit_cast(vec, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        }
        return v;
    }
};

// ---------------------------------------------------------------------------------------------
// Loads from memory to LDS that pass no register (16-bit types): lane l of a wave writes 16 bytes at the wave's base +
// 16 l (m0 holds the base: nothing else in these kernels uses it); an offset past the buffer's end (NOWHERE) writes zeros.
// The buffer's address may come from a vector instruction (v_readfirstlane) right in front, and the compiler's hazard recognizer
// does not look into the statement: it lets the five wait states pass itself that the load needs then (s_mov 1, s_nop 3 4).
// The compiler does not see them: dma_wait<N> waits until at most the N youngest loads of the wave are under way, behind it
// stands a barrier.
// ---------------------------------------------------------------------------------------------
using i32x4 = int __attribute__((ext_vector_type(4)));
constexpr uint32_t DMA_NOWHERE = 0x80000000u;
__device__ __forceinline__ i32x4 dma_buffer(const void* p) {  // 2 GiB from p on; p (48 bits) the same in all lanes
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    return i32x4{__builtin_amdgcn_readfirstlane((int)(uint32_t)a), __builtin_amdgcn_readfirstlane((int)(a >> 32)), 0x7fffffff,
                 0x00027000};
}
__device__ __forceinline__ void dma_advance(i32x4& buf, int64_t bytes) {
    const int lo = buf[0], hi = buf[1];
    const uint64_t a = ((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo) + (uint64_t)bytes;
    buf[0] = (int)(uint32_t)a;
    buf[1] = (int)(a >> 32);
}
// the same bounds for loads to registers
__device__ __forceinline__ f32x4 buffer_load(i32x4 buf, uint32_t off) {
    return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(
        __builtin_amdgcn_make_buffer_rsrc((void*)((uint64_t)(uint32_t)buf[0] | (uint64_t)(uint32_t)buf[1] << 32), 0, buf[2], buf[3]),
        (int)off, 0, 0));
}
__device__ __forceinline__ float buffer_load1(i32x4 buf, uint32_t off) {
    return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(
        __builtin_amdgcn_make_buffer_rsrc((void*)((uint64_t)(uint32_t)buf[0] | (uint64_t)(uint32_t)buf[1] << 32), 0, buf[2], buf[3]),
        (int)off, 0, 0));
}
__device__ __forceinline__ void dma_load(i32x4 buf, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(off), "s"(buf)
                 : "memory");
}
// 4 bytes a lane: lane l writes the wave's base + 4 l
__device__ __forceinline__ void dma_load4(i32x4 buf, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dword %1, %2, 0 offen lds"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(off), "s"(buf)
                 : "memory");
}
template <int N> __device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory"); }
// every wave's LDS reads are done and its awaited loads have landed
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory"); }
__device__ __forceinline__ uint32_t lds_offset(const char* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

// ---------------------------------------------------------------------------------------------
// stores of four neighbouring outputs, rounded once
// ---------------------------------------------------------------------------------------------
template <class T> __device__ __forceinline__ void store4(T* p, f32x4 v, int n, bool vec) {
    if (vec && n >= 4) {
        T t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = (T)v[i];
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<f32x4*>(p) = v;
        } else {
            uint2 u;
            u.x = bits16(t[0]) | bits16(t[1]) << 16;
            u.y = bits16(t[2]) | bits16(t[3]) << 16;
            *reinterpret_cast<uint2*>(p) = u;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < n) p[i] = (T)v[i];
}

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return (float)v; }
__device__ __forceinline__ float to_f(f16 v) { return (float)v; }

template <class T> __device__ __forceinline__ f32x4 load4(const T* p, int n, bool vec) {
    f32x4 r = {0, 0, 0, 0};
    if (vec && n >= 4) {
        if constexpr (sizeof(T) == 4) return *reinterpret_cast<const f32x4*>(p);
        T t[4];
        __builtin_memcpy(t, __builtin_assume_aligned(p, 8), 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = to_f(t[i]);
        return r;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < n) r[i] = to_f(p[i]);
    return r;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// C entry -> instance: TSD_F32 / TSD_BF16 / TSD_F16
#define TSD_BY_DTYPE(dtype, T, ...)                                          \
    switch (dtype) {                                                         \
        case TSD_F32: { using T = float; __VA_ARGS__; } break;               \
        case TSD_BF16: { using T = ::tsd::blk::bf16; __VA_ARGS__; } break;   \
        case TSD_F16: { using T = ::tsd::blk::f16; __VA_ARGS__; } break;     \
        default: break;                                                      \
    }

}  // namespace blk
}  // namespace tsd
