// Layer products of few rows (M up to 64: new tokens), bound by the one read
// of the weight.
//
// The weight goes straight from memory to the matrix cores' registers as the
// MFMA's row operand (16 outputs n per 16x16 step) and the rows of x are its
// columns, 16 at a time; the waves of a workgroup take K in turns, several
// steps of 128-bit loads in flight, and meet in LDS in wave order; K is
// split over workgroups too until the chip is full, the last workgroup of a
// tile adding the splits in their order.
//  * weight [N, K]: a lane reads 32 bytes of one row per step of 128 bytes
//    along K: two 16x16x32 16-bit steps, or one 16x16x128 e4m3 step;
//  * weight [K, N]: a lane reads 8 columns of 8 rows (16 bytes each), and
//    32 byte permutes turn them into the operands of 8 tiles of 16 columns.
// Rows past the end re-read the last one, a ragged row's last columns are
// read from its end (chunk.hpp); what is not the tile's is not stored.
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
    size_t kb;       // bytes of K (weight [N, K]) or K (weight [K, N])
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

// Weight [N, K], k along its rows: 16 NR columns n per workgroup.  The two
// 16-byte loads of a step take the halves of its 128 bytes, so that the four
// lanes of a row read 64 contiguous bytes.
template <int DT, int OT, int MT, int NR>
__global__ __launch_bounds__(kSW *kWave) void k_linear_rows(SkinnyArgs a) {
    constexpr int D = MT == 4 ? 2 : 4;  // steps in flight
    constexpr int NC = 16 * NR, E = MT * 16 * NC;
    __shared__ float sums[kSW * E];
    __shared__ int flag;
    const unsigned tile = blockIdx.x / a.splits, split = blockIdx.x - tile * a.splits;
    const unsigned n0 = tile * NC;
    const int lane = threadIdx.x & (kWave - 1), r16 = lane & 15, q = lane >> 4;
    const unsigned w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint8_t *wp[NR], *xp[MT];
#pragma unroll
    for (int j = 0; j < NR; ++j) {
        const unsigned n = n0 + 16 * j + r16 < a.N ? n0 + 16 * j + r16 : a.N - 1;
        wp[j] = a.w + static_cast<size_t>(n) * a.kb + 16 * q;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const unsigned m = 16 * i + r16 < a.M ? 16 * i + r16 : a.M - 1;
        xp[i] = a.x + static_cast<size_t>(m) * a.kb + 16 * q;
    }
    f32x4v acc[MT][NR];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NR; ++j) acc[i][j] = f32x4v{0.f, 0.f, 0.f, 0.f};
    auto mul = [&](const u32x4 (&u)[NR][2], const u32x4 (&v)[MT][2]) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NR; ++j) {
                if constexpr (DT == CXM_DT_E4M3) {
                    acc[i][j] = mfma_16x16_8(u[j][0], u[j][1], v[i][0], v[i][1], acc[i][j]);
                } else {
                    acc[i][j] = mfma_16x16<DT>(u[j][0], v[i][0], acc[i][j]);
                    acc[i][j] = mfma_16x16<DT>(u[j][1], v[i][1], acc[i][j]);
                }
            }
    };
    // whole steps of 128 bytes: wave w's share of this split's [s0, s1), one
    // after the other from a place that moves with the tile: rows a power of
    // two apart, read by every workgroup at the same k, meet in few of the
    // memory channels
    const unsigned whole = static_cast<unsigned>(a.kb / 128);
    const unsigned s0 = split * a.per, s1 = s0 + a.per < whole ? s0 + a.per : whole;
    const unsigned all = s1 > s0 ? s1 - s0 : 0, each = (all + kSW - 1) / kSW;
    const unsigned T = all > w * each ? (all - w * each < each ? all - w * each : each) : 0;
    const unsigned turn = T ? tile % T : 0;
    auto at = [&](unsigned t) {
        const unsigned u = (t < T ? t : T - 1) + turn;
        return static_cast<size_t>(s0 + w * each + (u < T ? u : u - T)) * 128;
    };
    u32x4 fw[D][NR][2], fx[D][MT][2];
    auto load = [&](int d, unsigned t) {
        const size_t o = at(t);
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            fw[d][j][0] = ld16(wp[j] + o);
            fw[d][j][1] = ld16(wp[j] + o + 64);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            fx[d][i][0] = ld16(xp[i] + o);
            fx[d][i][1] = ld16(xp[i] + o + 64);
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
        u32x4 u[NR][2], v[MT][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int j = 0; j < NR; ++j) u[j][h] = ld16_part(wp[j] + o + 64 * h, rest - 16 * q - 64 * h);
#pragma unroll
            for (int i = 0; i < MT; ++i) v[i][h] = ld16_part(xp[i] + o + 64 * h, rest - 16 * q - 64 * h);
        }
        mul(u, v);
    }
    // accumulator register r of lane l: n = 4 (l / 16) + r, m = l % 16
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NR; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) sums[w * E + (16 * i + r16) * NC + 16 * j + 4 * q + r] = acc[i][j][r];
    __syncthreads();
    skinny_join<E>(a, tile, split, sums, &flag, [&](int p, float v) {
        const unsigned m = p / NC, c = n0 + p % NC;
        if (m < a.M && c < a.N) skinny_store<OT>(a.e, v, m, c, a.N);
    });
}

// Weight [K, N]: 128 columns per workgroup, N >= 8.
template <int DT, int OT, int MT>
__global__ __launch_bounds__(kSW *kWave) void k_linear_cols(SkinnyArgs a) {
    constexpr int D = MT == 1 ? 2 : 1;
    constexpr int E = 16 * 128;  // one 16-row tile of x at a time
    __shared__ float sums[kSW * E / 2];
    __shared__ int flag;
    const unsigned tile = blockIdx.x / a.splits, split = blockIdx.x - tile * a.splits;
    const int lane = threadIdx.x & (kWave - 1), r16 = lane & 15, q = lane >> 4;
    const unsigned w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const Span sp = span_of<8>(tile * 16 + r16, a.N);
    const uint16_t *W = reinterpret_cast<const uint16_t *>(a.w) + sp.off;
    const uint16_t *X = reinterpret_cast<const uint16_t *>(a.x);
    const size_t K = a.kb;
    const uint16_t *xp[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) xp[i] = X + static_cast<size_t>(16 * i + r16 < a.M ? 16 * i + r16 : a.M - 1) * K + 8 * q;
    f32x4v acc[MT][8];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[i][c] = f32x4v{0.f, 0.f, 0.f, 0.f};
    auto mul = [&](const u32x4 (&f)[8], const u32x4 (&x)[MT]) {
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            u32x4 v;
#pragma unroll
            for (int p = 0; p < 4; ++p)
                v[p] = __builtin_amdgcn_perm(f[2 * p + 1][c / 2], f[2 * p][c / 2], (c & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i][c] = mfma_16x16<DT>(v, x[i], acc[i][c]);
        }
    };
    const unsigned whole = static_cast<unsigned>(K / 32);
    const unsigned s0 = split * a.per, s1 = s0 + a.per < whole ? s0 + a.per : whole;
    const unsigned T = s1 > s0 + w ? (s1 - s0 - w + kSW - 1) / kSW : 0;
    u32x4 fw[D][8], fx[D][MT];
    auto load = [&](int d, unsigned t) {
        const size_t k = static_cast<size_t>(s0 + w + (t < T ? t : T - 1) * kSW) * 32;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const u32x4e v = *reinterpret_cast<const u32x4e *>(W + (k + 8 * q + e) * a.N);
            fw[d][e] = u32x4{v.x, v.y, v.z, v.w};
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const u32x4e v = *reinterpret_cast<const u32x4e *>(xp[i] + k);
            fx[d][i] = u32x4{v.x, v.y, v.z, v.w};
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
    const unsigned rest = static_cast<unsigned>(K % 32);
    if (rest != 0 && split == a.splits - 1 && w == whole % kSW) {
        const size_t k = static_cast<size_t>(whole) * 32;
        u32x4 f[8], x[MT];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const unsigned kk = 8 * q + e;
            const u32x4e v = *reinterpret_cast<const u32x4e *>(W + (k + (kk < rest ? kk : rest - 1)) * a.N);
            f[e] = kk < rest ? u32x4{v.x, v.y, v.z, v.w} : u32x4{0u, 0u, 0u, 0u};
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
            x[i] = ld16_part(reinterpret_cast<const uint8_t *>(xp[i] + k), 2 * (static_cast<int>(rest) - 8 * q));
        mul(f, x);
    }
    // Tile c's accumulator register r of lane l: column chunk 4 (l / 16) + r,
    // element c of it, row l % 16.  Eight rows of 128 columns at a time.
    constexpr int EH = E / 2;
#pragma unroll
    for (int h = 0; h < 2 * MT; ++h) {
        if (h > 0) __syncthreads();
        if (r16 / 8 == (h & 1)) {
#pragma unroll
            for (int c = 0; c < 8; ++c)
#pragma unroll
                for (int r = 0; r < 4; ++r) sums[w * EH + (r16 % 8) * 128 + 8 * (4 * q + r) + c] = acc[h / 2][c][r];
        }
        __syncthreads();
        SkinnyArgs b = a;
        b.part = a.part ? a.part + static_cast<size_t>(h) * a.tiles * a.splits * EH : nullptr;
        b.counters = a.counters ? ctr(a.counters, static_cast<size_t>(h) * a.tiles) : nullptr;
        if (8u * h < a.M)
            skinny_join<EH>(b, tile, split, sums, &flag, [&](int p, float v) {
                const unsigned m = 8 * h + p / 128, chunk = tile * 16 + (p % 128) / 8, e = p % 8;
                const Span s = span_of<8>(chunk, a.N);
                if (m < a.M && e >= s.dup && s.dup < 8) skinny_store<OT>(a.e, v, m, s.off + e, a.N);
            });
    }
}

template <int DT, int OT>
int skinny_launch(const SkinnyArgs &a, bool tb, int nr, hipStream_t s) {
    const dim3 grid(a.tiles * a.splits), block(kSW * kWave);
    if (tb) {
        if (a.M <= 16 && nr == 1) hipLaunchKernelGGL((k_linear_rows<DT, OT, 1, 1>), grid, block, 0, s, a);
        else if (a.M <= 16) hipLaunchKernelGGL((k_linear_rows<DT, OT, 1, 2>), grid, block, 0, s, a);
        else if (a.M <= 32) hipLaunchKernelGGL((k_linear_rows<DT, OT, 2, 2>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((k_linear_rows<DT, OT, 4, 1>), grid, block, 0, s, a);
    } else if constexpr (DT != CXM_DT_E4M3) {
        if (a.M <= 16) hipLaunchKernelGGL((k_linear_cols<DT, OT, 1>), grid, block, 0, s, a);
        else if (a.M <= 32) hipLaunchKernelGGL((k_linear_cols<DT, OT, 2>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((k_linear_cols<DT, OT, 4>), grid, block, 0, s, a);
    }
    return launch_status();
}

// Tiles of 16 outputs per workgroup, weight [N, K].
int rows_tiles(size_t M, size_t N) {
    if (M > 32) return 1;
    if (M > 16) return 2;
    (void)N;
    return 1;
}

}  // namespace

// CXM_OK with plan->kernel = 0, or kDeclined.
int linear_skinny_plan(const LinProduct &p, LinPlan *l) {
    constexpr size_t kMax = size_t(1) << 28;
    const size_t kb = p.tb ? p.K * dtype_bytes(p.dtype) : p.K;
    if (p.M > 64 || p.ta || (!p.tb && p.N < 8) || kb >= (size_t(1) << 31) || p.N >= kMax) return kDeclined;
    *l = LinPlan{};
    l->kernel = 0;
    const size_t width = p.tb ? 16 * rows_tiles(p.M, p.N) : 128, step = p.tb ? 128 : 32;
    l->tiles = (p.N + width - 1) / width;
    const size_t whole = kb / step, target = 2 * device_cus();
    l->splits = 1;
    if (l->tiles < target) {
        l->splits = target / l->tiles;
        const size_t most = whole / (2 * kSW);  // two steps per wave at least
        if (l->splits > most) l->splits = most;
        if (l->splits < 1) l->splits = 1;
    }
    l->per = whole ? (whole + l->splits - 1) / l->splits : 1;
    if (whole) l->splits = (whole + l->per - 1) / l->per;
    if (l->tiles * l->splits > 0x7fffffu) return kDeclined;
    const size_t mt = p.M <= 16 ? 1 : p.M <= 32 ? 2 : 4;
    if (l->splits > 1)
        l->bytes_part = (l->tiles * l->splits * mt * 16 * width * sizeof(float) + 255) / 256 * 256;
    l->tiles_n = l->tiles;  // one ticket per tile (and per 8 rows, weight [K, N])
    if (!p.tb) l->tiles *= 2 * mt;
    return CXM_OK;
}

int linear_skinny_run(const LinProduct &p, const LinPlan &l, float *part, unsigned *counters, hipStream_t s) {
    const SkinnyArgs a{static_cast<const uint8_t *>(p.a),
                       static_cast<const uint8_t *>(p.b),
                       static_cast<unsigned>(p.M),
                       static_cast<unsigned>(p.N),
                       p.tb ? p.K * dtype_bytes(p.dtype) : p.K,
                       static_cast<unsigned>(l.tiles_n),
                       static_cast<unsigned>(l.splits),
                       static_cast<unsigned>(l.per),
                       part,
                       counters,
                       p.e};
    const int nr = rows_tiles(p.M, p.N);
    if (p.dtype == CXM_DT_E4M3) {
        if (p.out == CXM_DT_BF16) return skinny_launch<CXM_DT_E4M3, CXM_DT_BF16>(a, true, nr, s);
        return skinny_launch<CXM_DT_E4M3, CXM_DT_F16>(a, true, nr, s);
    }
    if (p.dtype == CXM_DT_BF16) return skinny_launch<CXM_DT_BF16, CXM_DT_BF16>(a, p.tb, nr, s);
    return skinny_launch<CXM_DT_F16, CXM_DT_F16>(a, p.tb, nr, s);
}

}  // namespace cxm
