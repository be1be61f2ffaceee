// Layer products on the matrix cores: bf16 / fp16 (v_mfma_f32_32x32x16) and
// e4m3 (v_mfma_f32_32x32x64), fp32 accumulation, and the layer's epilogue
// (scales, bias, activation, residual) before the only rounding.
//
// The ring of gemm16_ring.hpp (stages of 64 bytes per row) with these changes:
//  * eight waves, two per SIMD, on tiles of 256 and 128: one hides the
//    other's barriers and the epilogue's latency (four waves of 128x128 ran
//    4096x1024x4096 in 46.3 us against 37.5, 8192^3 at 1200 TFLOP/s against
//    1320; 2500x1024x1504 on 128 tiles 15.1 against 13.3, two K groups of
//    four 14.8);
//  * few rows: 32x64 tiles by four K groups of two waves;
//  * any M and N: rows and columns past the end re-read the last ones, their
//    sums are not stored;
//  * either operand stored with k along its rows or across them (the
//    transposing LDS reads serve both sides), so no product transposes first;
//  * few tiles split K over workgroups; the last one to finish a tile adds
//    the splits' partial sums in their order;
//  * the epilogue goes through LDS, 32 rows at a time, so that a lane has 8
//    consecutive elements of a row: 128-bit reads of the residual and writes
//    of z and y, and the activation's code once per 8 elements.
// An e4m3 product is the same ring over 16-bit units (two bytes of k): a stage
// of 64 bytes per row is one 32x32x64 step, to which each lane gives the two
// 16-byte pieces that the 16-bit form takes as two steps.  (Which k a lane
// holds does not matter as long as both operands agree.)
// The e4m3 steps align their products to the step's largest and drop what lies
// below 2^-13 of it before the fp32 sum (measured: 2^16 - 2^16 + p keeps p =
// 2^3 and loses 2^2; the 16-byte forms of the instruction do the same): 1e-5 of
// the sum of magnitudes at K = 64 and 2e-6 at K = 1024, far below the
// half step of the 16-bit result (4.9e-4 and 3.9e-3) and of the operands (6e-2).
#include <type_traits>

#include "gemm16_ring.hpp"
#include "linear.hpp"
#include "linear_act.hpp"

namespace cxm {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

struct RingArgs {
    const uint16_t *A, *B;
    size_t lda, ldb;  // of a stored row: units, staged bytes
    size_t M, N, K;
    unsigned tiles_m, tiles_n, splits, stages, per, gm;
    float *part;
    unsigned *counters;
    LinEpi e;
};

// A TM x TN tile by KG groups of WM x WN waves.  The groups take the stages
// of K in turns, each with a ring of its own, and add their sums in LDS at the
// end (in their order): more waves and loads in flight where the tiles are few
// and small.
// One load instruction of a wave brings 1 KiB; a group of more waves than
// an operand has such pieces loads some of them twice (the same bytes to the
// same place).
template <int TM_, int TN_, int WM_, int WN_, int KG_>
struct Geo {
    static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, KG = KG_;
    static constexpr int GW = WM * WN, WAVES = KG * GW, NT = WAVES * kWave;
    static constexpr int HM = TM / WM, HN = TN / WN;         // a wave's rows and columns
    static constexpr int MB = HM / 32, NB = HN / 32;         // its 32x32 blocks
    static constexpr int IA = TM >= 16 * GW ? TM / (16 * GW) : 1, IB = TN >= 16 * GW ? TN / (16 * GW) : 1;
    static constexpr int PS = IA + IB;                       // loads of a wave per stage
    static constexpr int TA = TM * kR_BK, STAGE = (TM + TN) * kR_BK;  // 16-bit units
    static constexpr int OWN = MB % KG == 0 ? MB / KG : MB;  // row blocks that a group finishes (else group 0 all)
    static constexpr int EPI = 32 * (HN + 8);                // floats of a wave's epilogue rows
    static_assert(MB >= 1 && NB >= 1, "every wave multiplies");
    static constexpr int PER = WAVES / 4;                    // waves whose epilogue rows share a stage's array
    static_assert(PER * EPI * 4 <= KG * STAGE * 2, "the epilogue fits the rings");
    static_assert(KG <= 5 && (KG == 1 || GW * MB * NB * 1024 * 4 <= KG * STAGE * 2), "the groups' sums fit the rings");
};

// Byte offsets of this lane's loads of an operand's stage (T rows of 64 bytes
// where k runs along the rows, else 32 k rows of T columns), rows (or chunks
// of 8 columns) past the operand's last clamped to it: `left` of them count
// from the tile's first.
template <int T, int ISSUES, bool KC>
struct SideLoads {
    unsigned o[ISSUES];
    unsigned to;  // byte offset of the wave's first piece in the operand's stage
    // w: the wave in its group
    __device__ __forceinline__ void init(size_t ld, size_t left, unsigned w) {
        constexpr unsigned PARTS = T / (16 * ISSUES);  // waves that share the stage
        w %= PARTS;
        to = w * (ISSUES * kWave * 16);
        const int lane = threadIdx.x & (kWave - 1);
        if constexpr (KC) {
            const int rr = lane >> 2, p = lane & 3;
#pragma unroll
            for (int s = 0; s < ISSUES; ++s) {
                const int row = static_cast<int>(w * ISSUES + s) * 16 + rr;
                const size_t r = static_cast<size_t>(row) < left ? row : left - 1;
                o[s] = static_cast<unsigned>((r * ld + 8 * (p ^ rkey(row))) * sizeof(uint16_t));
            }
        } else {
            constexpr int CPR = T / 8, RPI = kWave / CPR;
            const int rr = lane / CPR, p = lane % CPR;
            const size_t last = (left + 7) / 8 - 1;  // rows are stored in whole chunks
#pragma unroll
            for (int s = 0; s < ISSUES; ++s) {
                const int row = static_cast<int>(w * ISSUES + s) * RPI + rr;
                const size_t c = p ^ nkey<T>(row);
                o[s] = static_cast<unsigned>((row * ld + 8 * (c < last ? c : last)) * sizeof(uint16_t));
            }
        }
    }
    __device__ __forceinline__ void issue(const uint16_t *X, size_t r0, size_t k, size_t ld, uint16_t *stage) const {
        const uint16_t *base = KC ? X + r0 * ld + k : X + k * ld + r0;
        const unsigned l0 = lds_addr(stage) + __builtin_amdgcn_readfirstlane(to);
#pragma unroll
        for (int s = 0; s < ISSUES; ++s) lds_load16_at(base, o[s], l0 + s * kWave * 16);
    }
};

// Fragments of k block kb (16 units) of one operand's stage of T rows (or
// columns): rows w0 + 32 i + l32, eight k at 16 kb + 8 lhi.
template <int T, bool KC, int N>
__device__ __forceinline__ void side_frags(const uint16_t *st, int kb, int w0, int l32, int lhi, u32x4 (&f)[N]) {
    if constexpr (KC) {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = *reinterpret_cast<const u32x4 *>(st + roff(w0 + i * 32 + l32, 2 * kb + lhi));
    } else {
        const int lane = threadIdx.x & (kWave - 1);
        const int g = lane >> 4, jj = lane & 15;
        const int r = 16 * kb + 8 * (g >> 1) + (jj >> 2);
        const int c = 16 * (g & 1) + 4 * (jj & 3);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int n = w0 + i * 32 + c;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4 *)(st + noff<T>(r, n)));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4 *)(st + noff<T>(r + 4, n)));
            const u32x2 ul = __builtin_bit_cast(u32x2, lo), uh = __builtin_bit_cast(u32x2, hi);
            f[i] = u32x4{ul.x, ul.y, uh.x, uh.y};
        }
    }
}

template <class G, bool KA, bool KB>
struct RingLoads {
    const uint16_t *A, *B;
    size_t lda, ldb, m0, n0;
    SideLoads<G::TM, G::IA, KA> oa;
    SideLoads<G::TN, G::IB, KB> ob;
    __device__ __forceinline__ void issue(size_t k, uint16_t *stage) const {
        oa.issue(A, m0, k, lda, stage);
        ob.issue(B, n0, k, ldb, stage + G::TA);
    }
};

// The same stages filled through registers, for operands whose rows the
// direct loads cannot take (no multiple of 16 bytes, another base, or a K
// that ends inside a stage): unaligned 128-bit loads, D stages before their
// LDS writes.  What lies past K is zero; a piece across a row's end is read as
// the row's last 16 bytes and shifted down (rows of 16 bytes at least).
__device__ __forceinline__ u32x4 shift_down(u32x4 v, unsigned bytes) {
    const unsigned b = bytes * 8;
    const uint64_t x = static_cast<uint64_t>(v.y) << 32 | v.x, y = static_cast<uint64_t>(v.w) << 32 | v.z;
    const uint64_t lo = b == 0 ? x : b < 64 ? x >> b | y << (64 - b) : b < 128 ? y >> (b - 64) : 0;
    const uint64_t hi = b < 64 ? y >> b : 0;
    return u32x4{static_cast<unsigned>(lo), static_cast<unsigned>(lo >> 32), static_cast<unsigned>(hi),
                 static_cast<unsigned>(hi >> 32)};
}
typedef unsigned u32x4p __attribute__((ext_vector_type(4), aligned(1)));

template <int T, int ISSUES, bool KC>
struct SideStage {
    const char *x;   // KC: the tile's first row; else the operand
    size_t ld;       // bytes of a row
    size_t end;      // KC: the same; else rows of k
    unsigned o[ISSUES], row0, c, sh, to;
    __device__ __forceinline__ void init(const void *X, size_t row_bytes, size_t k_rows, size_t r0, size_t left,
                                         unsigned w) {
        constexpr unsigned PARTS = T / (16 * ISSUES);
        w %= PARTS;
        const unsigned lane = threadIdx.x & (kWave - 1);
        to = w * (ISSUES * kWave * 16) + lane * 16;
        ld = row_bytes;
        if constexpr (KC) {
            x = static_cast<const char *>(X) + r0 * ld;
            end = row_bytes;
            row0 = w * ISSUES * 16 + (lane >> 2);
            c = 16 * ((lane & 3) ^ rkey(static_cast<int>(row0)));  // 16 rows on, the key is the same
            sh = 0;
#pragma unroll
            for (int s = 0; s < ISSUES; ++s) {
                const size_t r = row0 + 16 * s;
                o[s] = static_cast<unsigned>((r < left ? r : left - 1) * ld);
            }
        } else {
            constexpr unsigned CPR = T / 8, RPI = kWave / CPR;
            x = static_cast<const char *>(X);
            end = k_rows;
            row0 = w * ISSUES * RPI + lane / CPR;
            sh = 0;
            c = 0;
#pragma unroll
            for (int s = 0; s < ISSUES; ++s) {
                // the chunk of a row differs with its key; its place in the row as well
                const unsigned r = row0 + RPI * s;
                const size_t at = r0 * 2 + 16 * ((lane % CPR) ^ nkey<T>(static_cast<int>(r)));
                const size_t in = at < ld - 16 ? at : ld - 16;
                o[s] = static_cast<unsigned>(in);
                const unsigned d = at - in < 16 ? static_cast<unsigned>(at - in) : 16u;
                sh |= d << (8 * s);  // up to four issues
            }
        }
    }
    __device__ __forceinline__ void load(size_t tile, u32x4 (&v)[ISSUES]) const {
        if constexpr (KC) {
            const size_t at = tile * 64 + c, in = at < end - 16 ? at : end - 16;
#pragma unroll
            for (int s = 0; s < ISSUES; ++s) {
                const u32x4p t = *reinterpret_cast<const u32x4p *>(x + o[s] + in);
                v[s] = u32x4{t.x, t.y, t.z, t.w};
            }
        } else {
            constexpr unsigned RPI = kWave / (T / 8);
#pragma unroll
            for (int s = 0; s < ISSUES; ++s) {
                const size_t k = tile * 32 + row0 + RPI * s;
                const u32x4p t = *reinterpret_cast<const u32x4p *>(x + (k < end ? k : end - 1) * ld + o[s]);
                v[s] = u32x4{t.x, t.y, t.z, t.w};
            }
        }
    }
    __device__ __forceinline__ void store(size_t tile, const u32x4 (&v)[ISSUES], uint16_t *stage) const {
        char *p = reinterpret_cast<char *>(stage) + to;
        if constexpr (KC) {
            const size_t at = tile * 64 + c;
            const bool cut = tile * 64 + 64 > end;  // the same in every lane
            const unsigned d = at + 16 <= end ? 0u : at - (end - 16) < 16 ? static_cast<unsigned>(at - (end - 16)) : 16u;
#pragma unroll
            for (int s = 0; s < ISSUES; ++s)
                *reinterpret_cast<u32x4 *>(p + s * kWave * 16) = cut ? shift_down(v[s], d) : v[s];
        } else {
            constexpr unsigned RPI = kWave / (T / 8);
            const bool cut = tile * 32 + 32 > end;
#pragma unroll
            for (int s = 0; s < ISSUES; ++s) {
                u32x4 u = v[s];
                if (__builtin_expect(__any(sh != 0), 0)) u = shift_down(u, (sh >> (8 * s)) & 0xffu);
                if (cut && tile * 32 + row0 + RPI * s >= end) u = u32x4{0u, 0u, 0u, 0u};
                *reinterpret_cast<u32x4 *>(p + s * kWave * 16) = u;
            }
        }
    }
};

// Both sides; D register sets (D divides the four steps of a turn).
template <class G, bool KA, bool KB>
struct StageLoads {
    static constexpr int D = 2;
    SideStage<G::TM, G::IA, KA> a;
    SideStage<G::TN, G::IB, KB> b;
    u32x4 va[D][G::IA], vb[D][G::IB];
    __device__ __forceinline__ void load(int d, size_t tile) {
        a.load(tile, va[d]);
        b.load(tile, vb[d]);
    }
    __device__ __forceinline__ void store(int d, size_t tile, uint16_t *stage) const {
        a.store(tile, va[d], stage);
        b.store(tile, vb[d], stage + G::TA);
    }
};

// The barrier of a staged ring: this wave's LDS reads and writes are done.
__device__ __forceinline__ void stage_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ f32x16 mfma8(u32x4 a0, u32x4 a1, u32x4 b0, u32x4 b1, f32x16 c) {
    const i32x8 a = {static_cast<int>(a0.x), static_cast<int>(a0.y), static_cast<int>(a0.z), static_cast<int>(a0.w),
                     static_cast<int>(a1.x), static_cast<int>(a1.y), static_cast<int>(a1.z), static_cast<int>(a1.w)};
    const i32x8 b = {static_cast<int>(b0.x), static_cast<int>(b0.y), static_cast<int>(b0.z), static_cast<int>(b0.w),
                     static_cast<int>(b1.x), static_cast<int>(b1.y), static_cast<int>(b1.z), static_cast<int>(b1.w)};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
}

template <class G>
struct Frags {
    u32x4 a[2][G::MB], b[2][G::NB];  // two k blocks of a stage
};
template <class G>
using Acc = f32x16[G::MB][G::NB];

// Interleaves NM MFMAs with the ND LDS reads of the next fragments.
template <int NM, int ND>
__device__ __forceinline__ void lin_interleave() {
    constexpr int P = NM < ND ? NM : ND, M = NM / P, D = ND / P;
#pragma unroll
    for (int t = 0; t < P; ++t) {
        __builtin_amdgcn_sched_group_barrier(0x008, M, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, D, 0);
    }
    if constexpr (NM > P * M) __builtin_amdgcn_sched_group_barrier(0x008, NM - P * M, 0);
    if constexpr (ND > P * D) __builtin_amdgcn_sched_group_barrier(0x100, ND - P * D, 0);
}

template <int DT, class G>
__device__ __forceinline__ void lin_mfma(const u32x4 (&a)[G::MB], const u32x4 (&b)[G::NB], Acc<G> &acc) {
#pragma unroll
    for (int i = 0; i < G::MB; ++i)
#pragma unroll
        for (int j = 0; j < G::NB; ++j) acc[i][j] = mfma16<DT>(a[i], b[j], acc[i][j]);
}

// 16-bit step on stage cur, as ring_step; f[0] holds block 0 of cur.  LAST:
// one of the steps after the unrolled loop, where a group may have no stage
// left (`live` false) and only keeps the barrier.
// `feed` fills a stage ahead, after the barrier (STG: through registers).
template <int DT, class G, bool KA, bool KB, bool STG, bool LAST, class F>
__device__ __forceinline__ void lin_step16(const F &feed, uint16_t *cur, const uint16_t *nxt, Frags<G> &f, Acc<G> &acc,
                                           int am, int bn, int l32, int lhi, bool live) {
    auto barrier = [] {
        if constexpr (STG) stage_barrier();
        else ring_barrier<2 * G::PS>();
    };
    if constexpr (LAST) {
        side_frags<G::TM, KA>(cur, 1, am, l32, lhi, f.a[1]);
        side_frags<G::TN, KB>(cur + G::TA, 1, bn, l32, lhi, f.b[1]);
        if (live) {
            lin_mfma<DT, G>(f.a[0], f.b[0], acc);
            lin_mfma<DT, G>(f.a[1], f.b[1], acc);
        }
        barrier();
        side_frags<G::TM, KA>(nxt, 0, am, l32, lhi, f.a[0]);
        side_frags<G::TN, KB>(nxt + G::TA, 0, bn, l32, lhi, f.b[0]);
        feed();
        return;
    }
    constexpr int NM = G::MB * G::NB, ND = G::MB * (KA ? 1 : 2) + G::NB * (KB ? 1 : 2);
    side_frags<G::TM, KA>(cur, 1, am, l32, lhi, f.a[1]);
    side_frags<G::TN, KB>(cur + G::TA, 1, bn, l32, lhi, f.b[1]);
    lin_mfma<DT, G>(f.a[0], f.b[0], acc);
    lin_interleave<NM, ND>();
    barrier();
    side_frags<G::TM, KA>(nxt, 0, am, l32, lhi, f.a[0]);
    side_frags<G::TN, KB>(nxt + G::TA, 0, bn, l32, lhi, f.b[0]);
    feed();
    lin_mfma<DT, G>(f.a[1], f.b[1], acc);
    if constexpr (!STG) {
        lin_interleave<NM, ND>();
        __builtin_amdgcn_sched_group_barrier(0x020, G::PS, 0);
    }
}

// e4m3 step: f holds all of cur's stage and is refilled from nxt as its parts
// have had their last product, the columns before the last ones before the
// barrier: one set of fragments, where a second one spilled (the same 66 us at
// 4096^3).
template <class G, bool STG, bool LAST, class F>
__device__ __forceinline__ void lin_step8(const F &feed, const uint16_t *nxt, Frags<G> &f, Acc<G> &acc, int am, int bn,
                                          int l32, int lhi, bool live) {
    constexpr int J = G::NB - 1;
    const uint16_t *nb = nxt + G::TA;
    auto mul = [&](int i, int j) { acc[i][j] = mfma8(f.a[0][i], f.a[1][i], f.b[0][j], f.b[1][j], acc[i][j]); };
    if (!LAST || live) {
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int i = 0; i < G::MB; ++i) mul(i, j);
        if constexpr (!LAST) __builtin_amdgcn_sched_group_barrier(0x008, J * G::MB, 0);
    }
    if constexpr (STG) stage_barrier();
    else ring_barrier<2 * G::PS>();
    feed();
    auto read_b = [&](int j) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
            f.b[kb][j] = *reinterpret_cast<const u32x4 *>(nb + roff(bn + j * 32 + l32, 2 * kb + lhi));
    };
#pragma unroll
    for (int j = 0; j < J; ++j) read_b(j);
#pragma unroll
    for (int i = 0; i < G::MB; ++i) {
        if (!LAST || live) mul(i, J);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
            f.a[kb][i] = *reinterpret_cast<const u32x4 *>(nxt + roff(am + i * 32 + l32, 2 * kb + lhi));
    }
    read_b(J);
    if constexpr (!LAST && !STG) {
        __builtin_amdgcn_sched_group_barrier(0x100, 2 * J, 0);
#pragma unroll
        for (int i = 0; i < G::MB; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
}

// The tile's sums through the wave's LDS to rows of 8 elements per lane.
template <int OT, class G>
__device__ __forceinline__ void lin_epilogue(const LinEpi &e, const Acc<G> &acc, float *lds, size_t m0, size_t n0,
                                             size_t M, size_t N, int l32, int lhi, int group) {
    constexpr int W = G::HN, LP = W + 8;  // row stride: 4 rows on distinct halves of the banks
    constexpr int LPR = W / 8, RPP = kWave / LPR;             // lanes per row, rows per pass
    const int lane = threadIdx.x & (kWave - 1);
    const int cl = 8 * (lane % LPR);
    const size_t col = n0 + cl;
    const int own = col >= N ? 0 : N - col < 8 ? static_cast<int>(N - col) : 8;  // elements of this lane's rows
    const auto *res = static_cast<const uint16_t *>(e.res);
    auto *z = static_cast<uint16_t *>(e.z);
    auto *y = static_cast<uint16_t *>(e.y);
    float bias[8], cs[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) bias[i] = 0.0f, cs[i] = 1.0f;
    // columns past the end: the last one's values, whose results are not stored
    if (e.bias) {
#pragma unroll
        for (int i = 0; i < 8; ++i) bias[i] = H<OT>::load(static_cast<const uint16_t *>(e.bias)[col + i < N ? col + i : N - 1]);
    }
    if (e.cs) {
#pragma unroll
        for (int i = 0; i < 8; ++i) cs[i] = e.cs[col + i < N ? col + i : N - 1];
    }
#pragma unroll
    for (int i = 0; i < G::MB; ++i) {
        if (i / G::OWN != group) continue;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < G::NB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) lds[(8 * (r / 4) + 4 * lhi + (r % 4)) * LP + 32 * j + l32] = acc[i][j][r];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int p = 0; p < 32 / RPP; ++p) {
            const int rl = p * RPP + lane / LPR;
            const size_t row = m0 + 32 * i + rl;
            if (row >= M || own == 0) continue;
            float v[8];
            const float4 lo = *reinterpret_cast<const float4 *>(&lds[rl * LP + cl]);
            const float4 hi = *reinterpret_cast<const float4 *>(&lds[rl * LP + cl + 4]);
            v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w;
            v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
            const size_t o = row * N + col;
            Chunk<OT, 8> c;
            if (e.res) {
                if (own == 8) {
                    c.load(res + o);
                } else {
                    uint16_t t[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) t[k] = res[o + (k < own ? k : own - 1)];
#pragma unroll
                    for (int k = 0; k < 4; ++k) c.r[k] = t[2 * k] | static_cast<unsigned>(t[2 * k + 1]) << 16;
                }
            }
            const float rs = e.rs ? e.rs[row] : 1.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (e.rs) v[k] = v[k] * rs * cs[k];
                v[k] += bias[k];
            }
            auto put = [&](uint16_t *q) {
                Chunk<OT, 8> d;
                d.set(v);
                if (own == 8) {
                    d.store(q + o);
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (k < own) q[o + k] = d.raw(k);
                }
            };
            if (e.z) put(z);
            act_apply<false, 8>(e.act, v);
            if (e.res) {
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] += c.get(k);
            }
            put(y);
        }
    }
}

template <int DT, int OT, class G, bool KA, bool KB, bool STG>
__global__ __launch_bounds__(G::NT) void k_linear_ring(RingArgs a) {
    // an array per stage of the rings, each holding the groups'
    constexpr int RS = G::KG * G::STAGE;
    __shared__ __attribute__((aligned(16))) uint16_t r0[RS], r1[RS], r2[RS], r3[RS];
    __shared__ int flag;
    const unsigned wg = xcd_remap16(blockIdx.x, gridDim.x);
    const unsigned tile = wg / a.splits, split = wg - tile * a.splits;
    unsigned tm, tn;
    group_tile(tile, a.tiles_m, a.tiles_n, a.gm, &tm, &tn);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int group = G::KG > 1 ? wave / G::GW : 0, gw = G::KG > 1 ? wave % G::GW : wave;
    const int am = gw / G::WN * G::HM, bn = gw % G::WN * G::HN;
    const int lane = threadIdx.x & (kWave - 1), l32 = lane & 31, lhi = lane >> 5;

    Acc<G> acc;
#pragma unroll
    for (int i = 0; i < G::MB; ++i)
#pragma unroll
        for (int j = 0; j < G::NB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    {
        uint16_t *s0 = r0 + group * G::STAGE, *s1 = r1 + group * G::STAGE, *s2 = r2 + group * G::STAGE,
                 *s3 = r3 + group * G::STAGE;
        const size_t first = static_cast<size_t>(split) * a.per;
        const size_t T = a.stages - first < a.per ? a.stages - first : a.per;  // this split's stages, at least 1
        // group g takes stages g, g + KG, ...; all make the same number of steps
        const size_t all = T / G::KG, steps = G::KG > 1 ? (T + G::KG - 1) / G::KG : T;
        const size_t mine = G::KG > 1 ? (T + G::KG - 1 - group) / G::KG : T;
        // stages past the last reload it into places whose fragments are not used
        auto tile_of = [&](size_t t) {
            const size_t u = t < mine ? t : mine - 1;
            if constexpr (G::KG > 1) return first + (mine ? group + u * G::KG : 0);
            else return first + u;
        };
        const size_t m0 = static_cast<size_t>(tm) * G::TM, n0 = static_cast<size_t>(tn) * G::TN;
        Frags<G> f;
        size_t t = 0;
        auto loop = [&](const auto &feed) {
            // feed(i, stage cur of step t + i, the stage two on)
            side_frags<G::TM, KA>(s0, 0, am, l32, lhi, f.a[0]);
            side_frags<G::TN, KB>(s0 + G::TA, 0, bn, l32, lhi, f.b[0]);
            if constexpr (DT == CXM_DT_E4M3) {
                side_frags<G::TM, true>(s0, 1, am, l32, lhi, f.a[1]);
                side_frags<G::TN, true>(s0 + G::TA, 1, bn, l32, lhi, f.b[1]);
            }
            auto step = [&](auto last, auto index, uint16_t *cur, uint16_t *nxt, uint16_t *two, bool live) {
                constexpr bool L = decltype(last)::value;
                auto fill = [&] { feed(index, cur, two); };
                if constexpr (DT == CXM_DT_E4M3) lin_step8<G, STG, L>(fill, nxt, f, acc, am, bn, l32, lhi, live);
                else lin_step16<DT, G, KA, KB, STG, L>(fill, cur, nxt, f, acc, am, bn, l32, lhi, live);
            };
            using No = std::false_type;
            using Yes = std::true_type;
            const std::integral_constant<int, 0> i0{};
            const std::integral_constant<int, 1> i1{};
            const std::integral_constant<int, 2> i2{};
            const std::integral_constant<int, 3> i3{};
            for (; t + 4 <= all; t += 4) {
                step(No{}, i0, s0, s1, s2, true);
                step(No{}, i1, s1, s2, s3, true);
                step(No{}, i2, s2, s3, s0, true);
                step(No{}, i3, s3, s0, s1, true);
            }
            if (t < steps) step(Yes{}, i0, s0, s1, s2, G::KG == 1 || t < mine);
            if (t + 1 < steps) step(Yes{}, i1, s1, s2, s3, G::KG == 1 || t + 1 < mine);
            if (t + 2 < steps) step(Yes{}, i2, s2, s3, s0, G::KG == 1 || t + 2 < mine);
            if (G::KG > 1 && t + 3 < steps) step(Yes{}, i3, s3, s0, s1, t + 3 < mine);
        };
        if constexpr (STG) {
            StageLoads<G, KA, KB> ld;
            constexpr int D = StageLoads<G, KA, KB>::D;
            ld.a.init(a.A, a.lda, a.K, m0, a.M - m0, gw);
            ld.b.init(a.B, a.ldb, a.K, n0, a.N - n0, gw);
            for (int i = 0; i < 2; ++i) {
                ld.load(0, tile_of(i));
                ld.store(0, tile_of(i), i ? s1 : s0);
            }
#pragma unroll
            for (int d = 0; d < D; ++d) ld.load(d, tile_of(2 + d));
            stage_barrier();
            loop([&](auto index, uint16_t *, uint16_t *two) {
                constexpr int d = decltype(index)::value % D;
                const size_t at = t + decltype(index)::value;
                ld.store(d, tile_of(at + 2), two);
                ld.load(d, tile_of(at + 2 + D));
            });
        } else {
            RingLoads<G, KA, KB> ld;
            ld.A = a.A;
            ld.B = a.B;
            ld.lda = a.lda;
            ld.ldb = a.ldb;
            ld.m0 = m0;
            ld.n0 = n0;
            ld.oa.init(a.lda, a.M - m0, gw);
            ld.ob.init(a.ldb, a.N - n0, gw);
            ld.issue(tile_of(0) * kR_BK, s0);
            ld.issue(tile_of(1) * kR_BK, s1);
            ld.issue(tile_of(2) * kR_BK, s2);
            ld.issue(tile_of(3) * kR_BK, s3);
            ring_barrier<3 * G::PS>();
            loop([&](auto index, uint16_t *cur, uint16_t *) {
                ld.issue(tile_of(t + 4 + decltype(index)::value) * kR_BK, cur);
            });
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load into LDS is left
    __syncthreads();  // every wave's fragment reads are done: the rings become scratch
    auto scratch = [&](int i) { return reinterpret_cast<float *>(i == 0 ? r0 : i == 1 ? r1 : i == 2 ? r2 : r3); };
    if constexpr (G::KG > 1) {
        // a group's sums of the row blocks that another one finishes, by the
        // sender's rank among the others
        auto slot = [&](int i, int sender, int owner) {
            const int rank = sender < owner ? sender : sender - 1;
            return scratch(rank) + (gw * G::MB + i) * (G::NB * 16 * kWave) + lane;
        };
#pragma unroll
        for (int i = 0; i < G::MB; ++i) {
            const int owner = i / G::OWN;
            if (owner == group) continue;
            float *p = slot(i, group, owner);
#pragma unroll
            for (int j = 0; j < G::NB; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) p[(j * 16 + r) * kWave] = acc[i][j][r];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < G::MB; ++i) {
            constexpr int O = G::OWN;
            const int owner = i / O;
            if (owner != group) continue;
#pragma unroll
            for (int j = 0; j < G::NB; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float v = 0.0f;
#pragma unroll
                    for (int s = 0; s < G::KG; ++s) {
                        const float u = s == i / O ? acc[i][j][r] : slot(i, s, i / O)[(j * 16 + r) * kWave];
                        v = s == 0 ? u : v + u;
                    }
                    acc[i][j][r] = v;
                }
        }
        __syncthreads();
    }
    if (a.splits > 1) {
        const unsigned ws = xcd_remap16(blockIdx.x, gridDim.x);
        const unsigned ti = ws / a.splits, sp = ws - ti * a.splits;
        float *base = a.part + static_cast<size_t>(ti) * a.splits * (G::TM * G::TN) + gw * kWave + lane;
        float *my = base + static_cast<size_t>(sp) * (G::TM * G::TN);
#pragma unroll
        for (int i = 0; i < G::MB; ++i) {
            if (i / G::OWN != group) continue;
#pragma unroll
            for (int j = 0; j < G::NB; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) st_dev(my + ((i * G::NB + j) * 16 + r) * (G::GW * kWave), acc[i][j][r]);
        }
        if (!last_block_ticket(ctr(a.counters, ti), a.splits, &flag)) return;
#pragma unroll
        for (int i = 0; i < G::MB; ++i) {
            if (i / G::OWN != group) continue;
#pragma unroll
            for (int j = 0; j < G::NB; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
            for (unsigned q = 0; q < a.splits; ++q) {
                const float *p = base + static_cast<size_t>(q) * (G::TM * G::TN);
#pragma unroll
                for (int j = 0; j < G::NB; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[i][j][r] += ld_dev(p + ((i * G::NB + j) * 16 + r) * (G::GW * kWave));
            }
        }
    }
    // the tile origin again, from the workgroup index, so that it need not live across the K loop
    group_tile(xcd_remap16(blockIdx.x, gridDim.x) / a.splits, a.tiles_m, a.tiles_n, a.gm, &tm, &tn);
    lin_epilogue<OT, G>(a.e, acc, scratch(wave / G::PER) + wave % G::PER * G::EPI, static_cast<size_t>(tm) * G::TM + am,
                        static_cast<size_t>(tn) * G::TN + bn, a.M, a.N, l32, lhi, group);
}

template <int DT, int OT, class G, bool STG>
int ring_layout(const RingArgs &a, unsigned wgs, bool ta, bool tb, hipStream_t s) {
    const dim3 grid(wgs), block(G::NT);
    if constexpr (DT == CXM_DT_E4M3) {
        hipLaunchKernelGGL((k_linear_ring<DT, OT, G, true, true, STG>), grid, block, 0, s, a);
    } else {
        if (!ta && !tb) hipLaunchKernelGGL((k_linear_ring<DT, OT, G, true, false, STG>), grid, block, 0, s, a);
        else if (!ta) hipLaunchKernelGGL((k_linear_ring<DT, OT, G, true, true, STG>), grid, block, 0, s, a);
        else if constexpr (G::TM >= 64)
            hipLaunchKernelGGL((k_linear_ring<DT, OT, G, false, false, STG>), grid, block, 0, s, a);
        else return CXM_E_INVALID;  // (no plan: a stage's rows of 32 columns are too short for the chunk keys)
    }
    return launch_status();
}

template <int DT, int OT, bool STG>
int ring_tile(const RingArgs &a, unsigned wgs, int tm, bool ta, bool tb, hipStream_t s) {
    if constexpr (!STG) {  // (staged: linear_plan)
        if (tm == 256) return ring_layout<DT, OT, Geo<256, 256, 2, 4, 1>, STG>(a, wgs, ta, tb, s);
        if (tm == 128) return ring_layout<DT, OT, Geo<128, 128, 2, 4, 1>, STG>(a, wgs, ta, tb, s);
    }
    if (tm == 64) return ring_layout<DT, OT, Geo<64, 64, 2, 2, 1>, STG>(a, wgs, ta, tb, s);
    if (tm == 32) return ring_layout<DT, OT, Geo<32, 64, 1, 2, 4>, STG>(a, wgs, ta, tb, s);
    return CXM_E_INVALID;
}

template <bool STG>
int ring_dtype(const LinProduct &p, const RingArgs &a, unsigned n, int tm, hipStream_t s) {
    if (p.dtype == CXM_DT_E4M3) {
        if (p.out == CXM_DT_BF16) return ring_tile<CXM_DT_E4M3, CXM_DT_BF16, STG>(a, n, tm, false, true, s);
        return ring_tile<CXM_DT_E4M3, CXM_DT_F16, STG>(a, n, tm, false, true, s);
    }
    if (p.dtype == CXM_DT_BF16) return ring_tile<CXM_DT_BF16, CXM_DT_BF16, STG>(a, n, tm, p.ta, p.tb, s);
    return ring_tile<CXM_DT_F16, CXM_DT_F16, STG>(a, n, tm, p.ta, p.tb, s);
}

}  // namespace

int linear_ring_run(const LinProduct &p, const LinPlan &l, const void *A, const void *B, float *part,
                    unsigned *counters, hipStream_t s) {
    const size_t wgs = l.tiles * l.splits;
    const size_t row_a = (p.ta ? p.M : p.K) * dtype_bytes(p.dtype), row_b = (p.tb ? p.K : p.N) * dtype_bytes(p.dtype);
    if (l.stages == 0 || l.stages > 0x7fffffffu || l.per * (l.splits - 1) >= l.stages || l.per * l.splits < l.stages ||
        wgs > most_wgs(1024) || (p.ta && p.tb))
        return CXM_E_TOO_LARGE;
    // what the kernels assume: direct loads, 16-byte aligned rows and whole stages;
    // staged ones, rows of 16 bytes at least; both, a tile's lane offsets within 32 bits
    // (255 rows of 2^24 bytes)
    if (l.staged ? row_a < 16 || row_b < 16 || row_a >= (size_t(1) << 24) || row_b >= (size_t(1) << 24)
                 : !aligned16(A) || !aligned16(B) || l.lda % 8 != 0 || l.ldb % 8 != 0 || l.lda > (size_t(1) << 23) ||
                       l.ldb > (size_t(1) << 23))
        return CXM_E_TOO_LARGE;
    const RingArgs a{static_cast<const uint16_t *>(A),
                     static_cast<const uint16_t *>(B),
                     l.staged ? row_a : l.lda,
                     l.staged ? row_b : l.ldb,
                     p.M,
                     p.N,
                     p.K,
                     static_cast<unsigned>(l.tiles_m),
                     static_cast<unsigned>(l.tiles_n),
                     static_cast<unsigned>(l.splits),
                     static_cast<unsigned>(l.stages),
                     static_cast<unsigned>(l.per),
                     4,
                     part,
                     counters,
                     p.e};
    const unsigned n = static_cast<unsigned>(wgs);
    return l.staged ? ring_dtype<true>(p, a, n, l.kernel, s) : ring_dtype<false>(p, a, n, l.kernel, s);
}

}  // namespace cxm
