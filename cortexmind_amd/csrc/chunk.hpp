// Rows of fp32, bf16 or fp16 elements as 16-byte chunks, for kernels that
// take any element type, any length and any element-aligned address.
//
// gfx950 takes a 128-bit global access at any element's address, so a row
// keeps 128-bit accesses whatever its length; what is left at its end is
// read once more from the last whole chunk's place (Span) with the elements
// that another chunk has already taken counted as zero, so no load needs a
// branch and every load is in bounds.
#pragma once

#include "half.hpp"

namespace cxm {
namespace {

typedef unsigned u32x4e __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4e __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <int DT>
struct Elem {
    using S = uint16_t;
    static constexpr int kVec = 8;
    __device__ static float load(S v) { return H<DT>::load(v); }
    __device__ static S store(float v) { return H<DT>::store(v); }
};
template <>
struct Elem<CXM_DT_F32> {
    using S = float;
    static constexpr int kVec = 4;
    __device__ static float load(S v) { return v; }
    __device__ static S store(float v) { return v; }
};

// Two floats rounded to nearest even in one word (v_cvt_pk_bf16_f32 on
// gfx950; NaN stays a quiet NaN).
template <int DT>
__device__ __forceinline__ unsigned pack2(float a, float b) {
    if constexpr (DT == CXM_DT_BF16) return __builtin_bit_cast(unsigned, bf16x2{static_cast<__bf16>(a), static_cast<__bf16>(b)});
    else return __builtin_bit_cast(unsigned, f16x2{static_cast<_Float16>(a), static_cast<_Float16>(b)});
}

// VE consecutive elements in registers: kVec (one 128-bit access) or 1.
// load_nt sets the non-temporal hint, for what is touched once.
template <int DT, int VE>
struct Chunk;
template <int VE>
struct Chunk<CXM_DT_F32, VE> {
    float r[VE];
    __device__ __forceinline__ void load(const float *p) {
        if constexpr (VE == 4) {
            const f32x4e v = *reinterpret_cast<const f32x4e *>(p);
            r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
        } else {
            r[0] = *p;
        }
    }
    __device__ __forceinline__ void load_nt(const float *p) {
        if constexpr (VE == 4) {
            const f32x4e v = __builtin_nontemporal_load(reinterpret_cast<const f32x4e *>(p));
            r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
        } else {
            r[0] = *p;
        }
    }
    __device__ __forceinline__ float get(int e) const { return r[e]; }
    __device__ __forceinline__ void set(const float (&v)[VE]) {
#pragma unroll
        for (int e = 0; e < VE; ++e) r[e] = v[e];
    }
    __device__ __forceinline__ void store(float *p) const {
        if constexpr (VE == 4) *reinterpret_cast<f32x4e *>(p) = f32x4e{r[0], r[1], r[2], r[3]};
        else *p = r[0];
    }
    __device__ __forceinline__ float raw(int e) const { return r[e]; }
};
template <int DT, int VE>
struct Chunk {
    unsigned r[(VE + 1) / 2];
    __device__ __forceinline__ void load(const uint16_t *p) {
        if constexpr (VE == 8) {
            const u32x4e v = *reinterpret_cast<const u32x4e *>(p);
            r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
        } else {
            r[0] = *p;
        }
    }
    __device__ __forceinline__ void load_nt(const uint16_t *p) {
        if constexpr (VE == 8) {
            const u32x4e v = __builtin_nontemporal_load(reinterpret_cast<const u32x4e *>(p));
            r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
        } else {
            r[0] = *p;
        }
    }
    __device__ __forceinline__ uint16_t raw(int e) const { return static_cast<uint16_t>(r[e / 2] >> (16 * (e & 1))); }
    __device__ __forceinline__ float get(int e) const { return H<DT>::load(raw(e)); }
    __device__ __forceinline__ void set(const float (&v)[VE]) {
        if constexpr (VE == 8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = pack2<DT>(v[2 * i], v[2 * i + 1]);
        } else {
            r[0] = pack2<DT>(v[0], 0.0f);
        }
    }
    __device__ __forceinline__ void store(uint16_t *p) const {
        if constexpr (VE == 8) *reinterpret_cast<u32x4e *>(p) = u32x4e{r[0], r[1], r[2], r[3]};
        else *p = static_cast<uint16_t>(r[0]);
    }
};

// Where chunk number c of a row of n elements (n >= VE) lies: `off`, moved
// back to the row's last VE elements where the chunk reaches past its end,
// and `dup`, how many of those belong to earlier chunks (VE or more: none is
// this chunk's own).  Elements e < dup are neither counted nor stored.
struct Span {
    unsigned off, dup;
};
template <int VE>
__device__ __forceinline__ Span span_of(unsigned c, unsigned n) {
    const unsigned col = c * VE, last = n - VE;
    const unsigned off = col < last ? col : last;
    return {off, col - off};
}
// Stores a chunk's own elements.
template <int DT, int VE>
__device__ __forceinline__ void store_span(typename Elem<DT>::S *row, Span s, const Chunk<DT, VE> &v) {
    if (s.dup == 0) {
        v.store(row + s.off);
    } else if (s.dup < VE) {
#pragma unroll
        for (int e = 1; e < VE; ++e)
            if (e >= static_cast<int>(s.dup)) row[s.off + e] = v.raw(e);
    }
}

// ------------------------------------------------------- 8-bit (e4m3) rows

// Four floats within +-448 as e4m3, rounded to nearest even (NaN: NaN).
__device__ __forceinline__ unsigned pack_e4m3(float a, float b, float c, float d) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return static_cast<unsigned>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true));
}
// Eight e4m3 bytes' values.
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void unpack_e4m3(unsigned w, float *v) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
    const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    v[0] = lo.x; v[1] = lo.y; v[2] = hi.x; v[3] = hi.y;
}

constexpr float kE4M3Max = 448.0f;

// Scale of values whose largest magnitude is `amax`, and its reciprocal:
// amax times the rounded 1 / 448 (the largest is held as 448, within an fp32
// rounding; the correctly rounded amax / 448 is one away for half of all values,
// an error of 2^-24 beside the codes' 2^-4), or 0 and 0 where that is no normal
// float; NaN and infinity stay.
struct Scale8 {
    float scale, inv;
};
__device__ __forceinline__ Scale8 scale_e4m3(float amax) {
    const float s = amax * (1.0f / kE4M3Max);
    if (s < FLT_MIN) return {0.0f, 0.0f};
    return {s, 1.0f / s};
}

}  // namespace

// ---------------------------------------------------------- host

// Workgroups of `threads` that one launch can have: fewer than 2^32 threads.
constexpr size_t most_wgs(size_t threads) { return 0xffffffffu / threads; }

// out[j] = sum of part[i][j] over i < n (rows `ld` floats apart), rounded to
// `dtype`; the order is fixed (colsum.hip).
int col_sum(const float *part, size_t n, size_t cols, size_t ld, void *out, int dtype, hipStream_t s);

// Whether [a, a + an) and [b, b + bn) share a byte (null or empty: no).
inline bool overlap(const void *a, size_t an, const void *b, size_t bn) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x && y && an && bn && x < y + bn && y < x + an;
}
// The same, but one being exactly the other is allowed (in place).
inline bool overlap_not_same(const void *a, size_t an, const void *b, size_t bn) {
    return a != b && overlap(a, an, b, bn);
}
inline bool is_float_dtype(int dt) { return dt == CXM_DT_F32 || dt == CXM_DT_BF16 || dt == CXM_DT_F16; }
inline size_t dtype_bytes(int dt) { return dt == CXM_DT_F32 ? 4 : dt == CXM_DT_E4M3 ? 1 : 2; }

}  // namespace cxm
