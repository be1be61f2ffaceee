// What the norms of rows share (norm.hip, layernorm.hip): reductions of a row
// over the lanes that hold it, its 8-bit form, and the sizes of their launches.
#pragma once

#include "chunk.hpp"

namespace cxm {

// Two sums that meet together.
struct Pair {
    float a, b;
};
struct PairSumOp {
    using T = Pair;
    __device__ static T identity() { return {0.0f, 0.0f}; }
    __device__ static T combine(T x, T y) { return {x.a + y.a, x.b + y.b}; }
};
template <int CTRL>
__device__ __forceinline__ Pair dpp(Pair p) {
    return {dpp<CTRL>(p.a), dpp<CTRL>(p.b)};
}
__device__ __forceinline__ Pair readlane(Pair p, int lane) { return {readlane(p.a, lane), readlane(p.b, lane)}; }
__device__ __forceinline__ Pair swap16(Pair p) { return {swap16(p.a), swap16(p.b)}; }

namespace {

// Largest magnitude, NaN if any is NaN.
struct AmaxOp : MaxOp {
    __device__ static T identity() { return 0.0f; }
};

template <bool ONCE, int DT, int VE>
__device__ __forceinline__ void load_once(Chunk<DT, VE> &c, const typename Elem<DT>::S *p) {
    if constexpr (ONCE) c.load_nt(p);
    else c.load(p);
}

template <class Op, int G, int NT>
__device__ __forceinline__ typename Op::T row_reduce(typename Op::T v, typename Op::T *lds) {
    if constexpr (G <= kWave) return group_reduce<Op, G>(v);
    else return block_reduce<Op, NT>(v, lds);
}

// Eight (four, one) e4m3 bytes of a chunk's own elements.
template <int VE>
__device__ __forceinline__ void store_q(uint8_t *row, Span s, const float (&v)[VE], float inv) {
    float t[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) t[e] = v[e] * inv;
    if constexpr (VE == 1) {
        if (s.dup == 0) row[s.off] = static_cast<uint8_t>(pack_e4m3(t[0], 0.0f, 0.0f, 0.0f));
    } else {
        unsigned w[VE / 4];
#pragma unroll
        for (int i = 0; i < VE / 4; ++i) w[i] = pack_e4m3(t[4 * i], t[4 * i + 1], t[4 * i + 2], t[4 * i + 3]);
        if (s.dup == 0) {
            typedef unsigned u32b __attribute__((aligned(1)));
            typedef unsigned u32x2b __attribute__((ext_vector_type(2), aligned(1)));
            if constexpr (VE == 8) *reinterpret_cast<u32x2b *>(row + s.off) = u32x2b{w[0], w[1]};
            else *reinterpret_cast<u32b *>(row + s.off) = w[0];
        } else if (s.dup < VE) {
#pragma unroll
            for (int e = 1; e < VE; ++e)
                if (e >= static_cast<int>(s.dup)) row[s.off + e] = static_cast<uint8_t>(w[e / 4] >> (8 * (e & 3)));
        }
    }
}

inline hipStream_t hs(cxm_stream_t s) { return reinterpret_cast<hipStream_t>(s); }

// Rows of whole 128-byte lines (null: yes).
inline bool whole_lines(const void *p, size_t cols, size_t bytes) {
    return (reinterpret_cast<uintptr_t>(p) | cols * bytes) % 128 == 0;
}

// Workgroups of the backward: enough to fill the chip, few enough that their
// shares of dw are a small part of the traffic.
size_t bwd_wgs(size_t rows, int per_wg, size_t per_cu = 2) {
    const size_t need = (rows + per_wg - 1) / per_wg, most = device_cus() * per_cu;
    return need < most ? need : most;
}

// Row lengths stay below 2^31, so that an element's place in its row is 32 bits.
bool row_shape_ok(size_t rows, size_t cols) {
    return cols < (size_t(1) << 31) && (rows == 0 || cols == 0 || rows <= (size_t(1) << 46) / cols);
}

}  // namespace
}  // namespace cxm
