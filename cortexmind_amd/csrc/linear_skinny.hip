// Layer products of one to a few rows with the weight stored [N, K], bound by
// the one read of the weight.
//  * one row (two of 16 bits): a wave reads whole rows of the weight, 1 KiB per
//    load, and multiplies on the vector units (1x4096x8192 bf16 13.2 us; the
//    form below 15.3, the ring 14.2; two rows 14.5, 15.8 and 14.0);
//  * up to 16 rows by a weight of up to 8 MiB: the weight goes straight from
//    memory to the matrix cores' registers as the MFMA's row operand (16
//    outputs n per 16x16 step) and the rows of x are its columns; the waves of
//    a workgroup share K and meet in LDS in wave order; K is split over
//    workgroups too, the last one of a tile adding the splits in their order
//    (16x1024x4096 bf16 5.1 us, the ring 5.6; larger weights are the ring's:
//    16x4096x4096 17.4 and 10.4, as every lane's row of x is read with each step).
// Rows past the end re-read the last one; what is not the tile's is not
// stored.  Non-temporal loads of the weight were slower (13.9 against 13.2 us).
#include "gemm16.hpp"
#include "linear.hpp"
#include "linear_act.hpp"

namespace cxm {
namespace {

typedef int i32x8s __attribute__((ext_vector_type(8)));
typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef unsigned u32x4b __attribute__((ext_vector_type(4), aligned(1)));

constexpr int kSW = 8;  // waves per workgroup

struct SkinnyArgs {
    const uint8_t *x, *w;
    unsigned M, N;
    size_t kb;       // bytes of a row of K
    unsigned tiles, splits;
    unsigned per;    // steps per split
    float *part;
    unsigned *counters;
    LinEpi e;
};

template <int DT>
__device__ __forceinline__ f32x4v mfma_16x16(u32x4 a, u32x4 b, f32x4v c) {
    if constexpr (DT == CXM_DT_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                       0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                      0);
}
__device__ __forceinline__ f32x4v mfma_16x16_8(u32x4 a0, u32x4 a1, u32x4 b0, u32x4 b1, f32x4v c) {
    const i32x8s a = {static_cast<int>(a0.x), static_cast<int>(a0.y), static_cast<int>(a0.z), static_cast<int>(a0.w),
                      static_cast<int>(a1.x), static_cast<int>(a1.y), static_cast<int>(a1.z), static_cast<int>(a1.w)};
    const i32x8s b = {static_cast<int>(b0.x), static_cast<int>(b0.y), static_cast<int>(b0.z), static_cast<int>(b0.w),
                      static_cast<int>(b1.x), static_cast<int>(b1.y), static_cast<int>(b1.z), static_cast<int>(b1.w)};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
}

// 16 bytes at p of which `n` (0 to 16) count, the others zero; bytes by bytes.
__device__ __forceinline__ u32x4 ld16_part(const uint8_t *p, int n) {
    u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const unsigned b = i < n ? p[i] : 0u;
        v[i / 4] |= b << (8 * (i & 3));
    }
    return v;
}
__device__ __forceinline__ u32x4 ld16(const uint8_t *p) {
    const u32x4b v = *reinterpret_cast<const u32x4b *>(p);
    return u32x4{v.x, v.y, v.z, v.w};
}

// One output element's epilogue.
template <int OT>
__device__ __forceinline__ void skinny_store(const LinEpi &e, float v, unsigned m, unsigned n, unsigned N) {
    const size_t o = static_cast<size_t>(m) * N + n;
    if (e.rs) v = v * e.rs[m] * e.cs[n];
    if (e.bias) v += H<OT>::load(static_cast<const uint16_t *>(e.bias)[n]);
    if (e.z) static_cast<uint16_t *>(e.z)[o] = H<OT>::store(v);
    float t[1] = {v};
    act_apply<false, 1>(e.act, t);
    if (e.res) t[0] += H<OT>::load(static_cast<const uint16_t *>(e.res)[o]);
    static_cast<uint16_t *>(e.y)[o] = H<OT>::store(t[0]);
}

// Adds the waves' sums (sums[wave][E] for E elements), meets the other splits,
// and gives every finished element to `put(element, value)`.
template <int E, class F>
__device__ __forceinline__ void skinny_join(const SkinnyArgs &a, unsigned tile, unsigned split, const float *sums,
                                            int *flag, const F &put) {
    constexpr int NT = kSW * kWave, PT = (E + NT - 1) / NT;
    float v[PT];
#pragma unroll
    for (int p = 0; p < PT; ++p) {
        const int q = threadIdx.x + p * NT;
        v[p] = q < E ? combine_pairwise<SumOp, kSW>(sums + q, E) : 0.0f;
    }
    if (a.splits > 1) {
        float *my = a.part + (static_cast<size_t>(tile) * a.splits + split) * E;
#pragma unroll
        for (int p = 0; p < PT; ++p) {
            const int q = threadIdx.x + p * NT;
            if (q < E) st_dev(my + q, v[p]);
        }
        if (!last_block_ticket(ctr(a.counters, tile), a.splits, flag)) return;
        const float *base = a.part + static_cast<size_t>(tile) * a.splits * E;
#pragma unroll
        for (int p = 0; p < PT; ++p) {
            const int q = threadIdx.x + p * NT;
            if (q < E) v[p] = combine_partials<SumOp>(base + q, a.splits, E, 0.0f);
        }
    }
#pragma unroll
    for (int p = 0; p < PT; ++p) {
        const int q = threadIdx.x + p * NT;
        if (q < E) put(q, v[p]);
    }
}

// 16 columns n per workgroup, a step of 128 bytes along K.  The two 16-byte
// loads of a step take its halves, so that the four lanes of a row read 64
// contiguous bytes.
template <int DT, int OT>
__global__ __launch_bounds__(kSW *kWave) void k_linear_rows(SkinnyArgs a) {
    constexpr int D = 4;  // steps in flight
    constexpr int E = 256;
    __shared__ float sums[kSW * E];
    __shared__ int flag;
    const unsigned tile = blockIdx.x / a.splits, split = blockIdx.x - tile * a.splits;
    const unsigned n0 = tile * 16;
    const int lane = threadIdx.x & (kWave - 1), r16 = lane & 15, q = lane >> 4;
    const unsigned w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint8_t *wp = a.w + static_cast<size_t>(n0 + r16 < a.N ? n0 + r16 : a.N - 1) * a.kb + 16 * q;
    const uint8_t *xp = a.x + static_cast<size_t>(static_cast<unsigned>(r16) < a.M ? r16 : a.M - 1) * a.kb + 16 * q;
    f32x4v acc = {0.f, 0.f, 0.f, 0.f};
    auto mul = [&](const u32x4 (&u)[2], const u32x4 (&v)[2]) {
        if constexpr (DT == CXM_DT_E4M3) {
            acc = mfma_16x16_8(u[0], u[1], v[0], v[1], acc);
        } else {
            acc = mfma_16x16<DT>(u[0], v[0], acc);
            acc = mfma_16x16<DT>(u[1], v[1], acc);
        }
    };
    // wave w's share of this split's whole steps [s0, s1), one after the other
    // from a place that moves with the tile: rows a power of two apart, read by
    // every workgroup at the same k, meet in few of the memory channels
    const unsigned whole = static_cast<unsigned>(a.kb / 128);
    const unsigned s0 = split * a.per, s1 = s0 + a.per < whole ? s0 + a.per : whole;
    const unsigned all = s1 > s0 ? s1 - s0 : 0, each = (all + kSW - 1) / kSW;
    const unsigned T = all > w * each ? (all - w * each < each ? all - w * each : each) : 0;
    const unsigned turn = T ? tile % T : 0;
    auto at = [&](unsigned t) {
        const unsigned u = (t < T ? t : T - 1) + turn;
        return static_cast<size_t>(s0 + w * each + (u < T ? u : u - T)) * 128;
    };
    u32x4 fw[D][2], fx[D][2];
    auto load = [&](int d, unsigned t) {
        const size_t o = at(t);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            fw[d][h] = ld16(wp + o + 64 * h);
            fx[d][h] = ld16(xp + o + 64 * h);
        }
    };
    if (T > 0) {
#pragma unroll
        for (int d = 0; d < D; ++d) load(d, d);
        unsigned t = 0;
        for (; t + D <= T; t += D) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                mul(fw[d], fx[d]);
                load(d, t + d + D);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (t + d < T) mul(fw[d], fx[d]);
    }
    const int rest = static_cast<int>(a.kb % 128);
    if (rest != 0 && split == a.splits - 1 && w == kSW - 1) {  // the last wave's share is the shortest
        const size_t o = static_cast<size_t>(whole) * 128;
        u32x4 u[2], v[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u[h] = ld16_part(wp + o + 64 * h, rest - 16 * q - 64 * h);
            v[h] = ld16_part(xp + o + 64 * h, rest - 16 * q - 64 * h);
        }
        mul(u, v);
    }
    // accumulator register r of lane l: n = 4 (l / 16) + r, m = l % 16
#pragma unroll
    for (int r = 0; r < 4; ++r) sums[w * E + r16 * 16 + 4 * q + r] = acc[r];
    __syncthreads();
    skinny_join<E>(a, tile, split, sums, &flag, [&](int p, float v) {
        const unsigned m = p / 16, c = n0 + p % 16;
        if (m < a.M && c < a.N) skinny_store<OT>(a.e, v, m, c, a.N);
    });
}

// One or two rows: a wave takes kDotRows rows of the weight whole.
constexpr int kDotRows = 2, kDotDepth = 4;
// (two rows of e4m3 take the ring: 8192x8192 17.9 us here, 14.3 there)
inline bool dot_takes(size_t M, size_t kb, int dtype) {
    return kb >= 16 && (M == 1 || (M == 2 && dtype != CXM_DT_E4M3));
}

template <int DT>
struct DotElems {
    static constexpr int kVec = DT == CXM_DT_E4M3 ? 16 : 8;
    __device__ static void get(u32x4 r, float (&v)[kVec]) {
        if constexpr (DT == CXM_DT_E4M3) {
#pragma unroll
            for (int i = 0; i < 4; ++i) unpack_e4m3(r[i], v + 4 * i);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = H<DT>::load(static_cast<uint16_t>(r[i / 2] >> (16 * (i & 1))));
        }
    }
};

template <int DT, int OT, int M>
__global__ __launch_bounds__(kBlock) void k_linear_dot(SkinnyArgs a) {
    constexpr int VE = DotElems<DT>::kVec, RW = kDotRows, D = kDotDepth;
    const unsigned lane = threadIdx.x % kWave;
    const unsigned n0 = (blockIdx.x * (kBlock / kWave) + threadIdx.x / kWave) * RW;
    if (n0 >= a.N) return;  // whole waves
    const uint8_t *wp[RW];
#pragma unroll
    for (int j = 0; j < RW; ++j) wp[j] = a.w + static_cast<size_t>(n0 + j < a.N ? n0 + j : a.N - 1) * a.kb;
    const unsigned T = static_cast<unsigned>((a.kb + 1023) / 1024), bytes = static_cast<unsigned>(a.kb);
    float acc[RW][M];
#pragma unroll
    for (int j = 0; j < RW; ++j)
#pragma unroll
        for (int i = 0; i < M; ++i) acc[j][i] = 0.0f;
    u32x4 fw[D][RW], fx[D][M];
    // piece t of a row: 16 bytes per lane, those past its end moved back to it
    auto off = [&](unsigned t) {
        const unsigned o = t * 1024 + lane * 16;
        return o < bytes - 16 ? o : bytes - 16;
    };
    auto load = [&](int d, unsigned t) {
        const unsigned o = off(t < T ? t : T - 1);
#pragma unroll
        for (int j = 0; j < RW; ++j) fw[d][j] = ld16(wp[j] + o);
#pragma unroll
        for (int i = 0; i < M; ++i) fx[d][i] = ld16(a.x + static_cast<size_t>(i) * a.kb + o);
    };
    auto mul = [&](int d, unsigned t) {
        float w[RW][VE];
#pragma unroll
        for (int j = 0; j < RW; ++j) DotElems<DT>::get(fw[d][j], w[j]);
        const bool last = t == T - 1;  // the only one with elements of another lane's
        const int dup = static_cast<int>(t * 1024 + lane * 16 - off(t)) / (16 / VE);
#pragma unroll
        for (int i = 0; i < M; ++i) {
            float x[VE];
            DotElems<DT>::get(fx[d][i], x);
            if (last) {
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    x[e] = e >= dup ? x[e] : 0.0f;
#pragma unroll
                    for (int j = 0; j < RW; ++j) w[j][e] = e >= dup ? w[j][e] : 0.0f;
                }
            }
#pragma unroll
            for (int j = 0; j < RW; ++j)
#pragma unroll
                for (int e = 0; e < VE; ++e) acc[j][i] = fmaf(w[j][e], x[e], acc[j][i]);
        }
    };
#pragma unroll
    for (int d = 0; d < D; ++d) load(d, d);
    for (unsigned t = 0; t < T; t += D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            if (t + d < T) mul(d, t + d);
            load(d, t + d + D);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
#pragma unroll
    for (int j = 0; j < RW; ++j)
#pragma unroll
        for (int i = 0; i < M; ++i) {
            const float v = group_reduce<SumOp, kWave>(acc[j][i]);
            if (lane == static_cast<unsigned>(j * M + i) && n0 + j < a.N) skinny_store<OT>(a.e, v, i, n0 + j, a.N);
        }
}

template <int DT, int OT>
int skinny_launch(const SkinnyArgs &a, hipStream_t s) {
    if (dot_takes(a.M, a.kb, DT)) {
        constexpr unsigned R = kBlock / kWave * kDotRows;
        const dim3 grid((a.N + R - 1) / R), block(kBlock);
        if (a.M == 1) hipLaunchKernelGGL((k_linear_dot<DT, OT, 1>), grid, block, 0, s, a);
        else if constexpr (DT != CXM_DT_E4M3) hipLaunchKernelGGL((k_linear_dot<DT, OT, 2>), grid, block, 0, s, a);
        return launch_status();
    }
    hipLaunchKernelGGL((k_linear_rows<DT, OT>), dim3(a.tiles * a.splits), dim3(kSW * kWave), 0, s, a);
    return launch_status();
}

}  // namespace

// Whether these kernels take the product; fills in the plan (kernel 0).
bool linear_skinny_plan(const LinProduct &p, LinPlan *l) {
    const size_t kb = p.K * dtype_bytes(p.dtype);
    if (p.ta || !p.tb || p.M > 16 || kb >= (size_t(1) << 31) || p.N >= (size_t(1) << 28)) return false;
    const bool dot = dot_takes(p.M, kb, p.dtype);
    if (!dot && kb * p.N > (size_t(8) << 20)) return false;
    *l = LinPlan{};
    l->splits = l->per = 1;
    l->tiles = (p.N + 15) / 16;
    if (dot) return true;
    const size_t whole = kb / 128, target = 2 * device_cus();
    if (l->tiles < target) {
        l->splits = target / l->tiles;
        const size_t most = whole / (2 * kSW);  // two steps per wave at least
        if (l->splits > most) l->splits = most;
        if (l->splits < 1) l->splits = 1;
    }
    l->per = whole ? (whole + l->splits - 1) / l->splits : 1;
    if (whole) l->splits = (whole + l->per - 1) / l->per;
    if (l->splits > 1) l->bytes_part = (l->tiles * l->splits * 256 * sizeof(float) + 255) / 256 * 256;
    return true;
}

int linear_skinny_run(const LinProduct &p, const LinPlan &l, float *part, unsigned *counters, hipStream_t s) {
    const SkinnyArgs a{static_cast<const uint8_t *>(p.a),
                       static_cast<const uint8_t *>(p.b),
                       static_cast<unsigned>(p.M),
                       static_cast<unsigned>(p.N),
                       p.K * dtype_bytes(p.dtype),
                       static_cast<unsigned>(l.tiles),
                       static_cast<unsigned>(l.splits),
                       static_cast<unsigned>(l.per),
                       part,
                       counters,
                       p.e};
    if (p.dtype == CXM_DT_E4M3) {
        if (p.out == CXM_DT_BF16) return skinny_launch<CXM_DT_E4M3, CXM_DT_BF16>(a, s);
        return skinny_launch<CXM_DT_E4M3, CXM_DT_F16>(a, s);
    }
    if (p.dtype == CXM_DT_BF16) return skinny_launch<CXM_DT_BF16, CXM_DT_BF16>(a, s);
    return skinny_launch<CXM_DT_F16, CXM_DT_F16>(a, s);
}

}  // namespace cxm
