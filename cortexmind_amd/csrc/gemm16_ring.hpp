// The ring shared by the 16-bit GEMM (gemm16.hip) and the layer products
// (linear.hip): tiles in four LDS stages filled by direct global-to-LDS
// loads, and the order in which workgroups take the tiles.
#pragma once

#include "gemm16.hpp"

namespace cxm {
namespace {

constexpr int kHThreads = 256;

__device__ __forceinline__ unsigned xcd_remap16(unsigned b, unsigned g) {
    if (g % 8 != 0) return b;
    return (b % 8) * (g / 8) + b / 8;
}

// ----------------------------------------------- ring: four LDS stages of BK 32
//
// A TM x TM workgroup tile (TM = 256 or 128), four waves of TM/2 x TM/2
// (NB x NB MFMA blocks of 32x32, NB = TM/64), interior tiles only (M, N
// multiples of TM, K a multiple of 128).  The k loop runs over a ring of
// four LDS stages of 32 k, filled by direct global-to-LDS loads
// (lds_load16_at) four steps ahead (three tiles in flight); the loop is
// unrolled over the ring so that stage addresses are constants.
// A step on stage t: MFMAs of k block 0 with block 1's fragments read
// between them; the ring barrier (this wave's loads of stage t+1 landed,
// every wave done reading stage t); the next stage's block-0 fragments;
// loads of tile t+4 into stage t; MFMAs of k block 1.
//
// A is stored [M,K] (k contiguous).  Its stage holds TM rows of 64 bytes,
// the four 16-byte groups of row r XOR-keyed by (r / 4) % 4: 16
// consecutive rows, one group each, land on 16 distinct 16-byte slots of
// the 64 banks, so a ds_read_b128 fragment read is conflict-free.
// B is either stored as B^T [N,K] (KB, same stage layout as A) or as
// [K,N] (n contiguous).  The [K,N] stage holds 32 k rows of TM columns as
// loaded, 16-byte chunk c of row r at c ^ 4*(r % 4), and fragments come
// from ds_read_b64_tr_b16: in each 16-lane group, result lane i element e
// is element i % 4 of the 64 bits addressed by lane i / 4 + 4 e.  Lane j
// of a group addresses row k0 + j / 4, columns n0 + 4 (j % 4) .. +3, so
// lane i receives B[k0 .. k0+3][n0 + i]: four consecutive k of one column,
// half of a 32x32x16 operand; two reads give the eight.  The chunk key puts
// the four rows one read touches (64 bytes each) on distinct banks.
constexpr int kR_BK = 32;

template <int TM>
struct Ring {
    static constexpr int NB = TM / 64;            // 32x32 blocks per wave side
    static constexpr int TILE = TM * kR_BK;       // elements per operand stage
    static constexpr int ISSUES = TM / 64;        // load instructions per wave per operand per stage
    static constexpr int PER_STAGE = 2 * ISSUES;  // loads a wave has in flight per stage
};

__device__ __forceinline__ int rkey(int r) { return (r >> 2) & 3; }
__device__ __forceinline__ int roff(int row, int g) { return row * kR_BK + 8 * (g ^ rkey(row)); }
// Chunk key of k row r in a [K,N] stage of TM columns.  Rows of 64 columns
// take half the banks each, so that rows 0 and 2 (1 and 3) meet there.
template <int TM>
__device__ __forceinline__ int nkey(int r) {
    return TM == 64 ? 4 * ((r >> 1) & 1) : 4 * (r & 3);
}
// element offset of (k row r, column n) in a [K,N] stage of TM columns
template <int TM>
__device__ __forceinline__ int noff(int r, int n) {
    return r * TM + (((n >> 3) ^ nkey<TM>(r)) << 3) + (n & 7);
}

// Stage fills.  A TM x 32 stage of X k-contiguous (row stride Kd) at rows
// r0.., k0..: each wave fills TM/4 rows, 16 per instruction (lane L: row
// L/4, LDS group L%4, global group (L%4) ^ key).  A 32 x TM stage of B
// stored [K,N] (row stride N) at k rows k0.., columns n0..: each wave
// fills 8 rows; an instruction covers 1 KiB, i.e. 64 / (TM/8) rows (lane
// L: row L / (TM/8), LDS chunk L % (TM/8), global chunk
// (L % (TM/8)) ^ 4*(row % 4)).  Each load reads from a base uniform across
// the workgroup (X + r0 Kd + k0, or B + k0 N + n0) plus a 32-bit lane
// offset fixed for the whole K loop (RingOffs16), into an LDS destination
// computed on the scalar unit: no 64-bit vector address arithmetic per load.
template <int TM>
struct RingOffs16 {
    unsigned o[Ring<TM>::ISSUES];
};
template <int TM>
__device__ __forceinline__ RingOffs16<TM> ring_offs_k(size_t Kd) {
    const int lane = threadIdx.x & (kWave - 1), w = threadIdx.x / kWave;
    const int rr = lane >> 2, p = lane & 3;
    RingOffs16<TM> f;
#pragma unroll
    for (int s = 0; s < Ring<TM>::ISSUES; ++s) {
        const int row = w * (TM / 4) + s * 16 + rr;
        f.o[s] = static_cast<unsigned>((row * Kd + 8 * (p ^ rkey(row))) * sizeof(uint16_t));
    }
    return f;
}
template <int TM>
__device__ __forceinline__ RingOffs16<TM> ring_offs_n(size_t N) {
    constexpr int CPR = TM / 8, RPI = kWave / CPR;
    const int lane = threadIdx.x & (kWave - 1), w = threadIdx.x / kWave;
    const int rr = lane / CPR, p = lane % CPR;
    RingOffs16<TM> f;
#pragma unroll
    for (int s = 0; s < Ring<TM>::ISSUES; ++s) {
        const int row = w * 8 + s * RPI + rr;
        f.o[s] = static_cast<unsigned>((row * N + 8 * (p ^ nkey<TM>(row))) * sizeof(uint16_t));
    }
    return f;
}
// k-contiguous stage (KC) at rows r0.., k0..; else a [K,N] stage at k rows
// k0.., columns r0..
template <int TM, bool KC>
__device__ __forceinline__ void ring_issue_at(const uint16_t *__restrict__ X, size_t r0, size_t k0, size_t ld,
                                              const RingOffs16<TM> &f, uint16_t *stage) {
    const unsigned w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint16_t *base = KC ? X + r0 * ld + k0 : X + k0 * ld + r0;
    const unsigned l0 = lds_addr(stage) + (KC ? w * (TM / 4) * kR_BK : w * 8 * TM) * sizeof(uint16_t);
#pragma unroll
    for (int s = 0; s < Ring<TM>::ISSUES; ++s) lds_load16_at(base, f.o[s], l0 + s * kWave * 16);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// Fragments of k block kb (16 k) of a stage: A rows wm*TM/2 + 32 i + l32,
// eight k at 16 kb + 8 lhi; B likewise from the k-contiguous or the [K,N]
// stage.
template <int TM, bool KB>
__device__ __forceinline__ void ring_frags(const uint16_t *sa, const uint16_t *sb, int kb, int wm, int wn, int l32,
                                           int lhi, u32x4 (&fa)[Ring<TM>::NB], u32x4 (&fb)[Ring<TM>::NB]) {
    constexpr int NB = Ring<TM>::NB;
#pragma unroll
    for (int i = 0; i < NB; ++i)
        fa[i] = *reinterpret_cast<const u32x4 *>(sa + roff(wm * (TM / 2) + i * 32 + l32, 2 * kb + lhi));
    if constexpr (KB) {
#pragma unroll
        for (int j = 0; j < NB; ++j)
            fb[j] = *reinterpret_cast<const u32x4 *>(sb + roff(wn * (TM / 2) + j * 32 + l32, 2 * kb + lhi));
    } else {
        const int lane = threadIdx.x & (kWave - 1);
        const int g = lane >> 4, jj = lane & 15;
        const int r = 16 * kb + 8 * (g >> 1) + (jj >> 2);
        const int c = 16 * (g & 1) + 4 * (jj & 3);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int n = wn * (TM / 2) + j * 32 + c;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4 *)(sb + noff<TM>(r, n)));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4 *)(sb + noff<TM>(r + 4, n)));
            const u32x2 ul = __builtin_bit_cast(u32x2, lo), uh = __builtin_bit_cast(u32x2, hi);
            fb[j] = u32x4{ul.x, ul.y, uh.x, uh.y};
        }
    }
}

template <int DT, int NB>
__device__ __forceinline__ void ring_mfma(const u32x4 (&fa)[NB], const u32x4 (&fb)[NB], f32x16 (&acc)[NB][NB]) {
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = mfma16<DT>(fa[i], fb[j], acc[i][j]);
}

// Interleaves a k block's MFMAs with the fragment reads of the next block:
// two MFMAs per read for the 256 tile with k-contiguous B (eight reads),
// otherwise one MFMA per read until either runs out.
template <int TM, bool KB>
__device__ __forceinline__ void ring_interleave() {
    constexpr int NM = Ring<TM>::NB * Ring<TM>::NB;
    constexpr int ND = Ring<TM>::NB * (KB ? 2 : 3);
    if constexpr (TM == 256 && KB) {
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
    } else {
        constexpr int P = NM < ND ? NM : ND;
#pragma unroll
        for (int t = 0; t < P; ++t) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        if constexpr (NM > P) __builtin_amdgcn_sched_group_barrier(0x008, NM - P, 0);
        if constexpr (ND > P) __builtin_amdgcn_sched_group_barrier(0x100, ND - P, 0);
    }
}

// Fills a B stage: k-contiguous (B^T [N,K], rows n0..) or [K,N] (k rows k0..).
template <int TM, bool KB>
__device__ __forceinline__ void ring_issue_b(const uint16_t *__restrict__ B, size_t n0, size_t kf, size_t K, size_t N,
                                             const RingOffs16<TM> &ob, uint16_t *stage) {
    if constexpr (KB) ring_issue_at<TM, true>(B, n0, kf, K, ob, stage);
    else ring_issue_at<TM, false>(B, n0, kf, N, ob, stage);
}

// Step t on stage cur (A tile at +0, B tile at +TILE, tile t); nxt holds
// tile t+1.  After the barrier every wave has read all of cur, which is
// refilled at once with tile t+4 (k offset kf): three tiles stay in flight.
template <int DT, int TM, bool KB>
__device__ __forceinline__ void ring_step(const uint16_t *__restrict__ A, const uint16_t *__restrict__ B, size_t K,
                                          size_t N, size_t m0, size_t n0, size_t kf, uint16_t *cur,
                                          const uint16_t *nxt, u32x4 (&fa)[Ring<TM>::NB], u32x4 (&fb)[Ring<TM>::NB],
                                          f32x16 (&acc)[Ring<TM>::NB][Ring<TM>::NB], int wm, int wn, int l32,
                                          int lhi, const RingOffs16<TM> &oa, const RingOffs16<TM> &ob) {
    constexpr int NB = Ring<TM>::NB, TILE = Ring<TM>::TILE;
    u32x4 ga[NB], gb[NB];
    ring_frags<TM, KB>(cur, cur + TILE, 1, wm, wn, l32, lhi, ga, gb);  // block 1, during block 0's MFMAs
    ring_mfma<DT, NB>(fa, fb, acc);
    ring_interleave<TM, KB>();
    ring_barrier<2 * Ring<TM>::PER_STAGE>();  // tile t+1 has landed; tiles t+2, t+3 may be in flight
    ring_frags<TM, KB>(nxt, nxt + TILE, 0, wm, wn, l32, lhi, fa, fb);  // next step's block 0
    ring_issue_at<TM, true>(A, m0, kf, K, oa, cur);
    ring_issue_b<TM, KB>(B, n0, kf, K, N, ob, cur + TILE);
    ring_mfma<DT, NB>(ga, gb, acc);
    ring_interleave<TM, KB>();
    __builtin_amdgcn_sched_group_barrier(0x020, Ring<TM>::PER_STAGE, 0);
}

// Tile order: the XCD remap gives each XCD a contiguous range of tile ids;
// inside it, ids walk down GM tile rows before moving one tile column, so
// the tiles an XCD runs at once share GM row blocks of A and a few column
// blocks of B in its L2 (one tile row would share 1 and all of them).
__device__ __forceinline__ void group_tile(unsigned id, unsigned tiles_m, unsigned tiles_n, unsigned gm, unsigned *tm,
                                           unsigned *tn) {
    const unsigned per_group = gm * tiles_n;
    const unsigned group = id / per_group;
    const unsigned first = group * gm;
    const unsigned rows = tiles_m - first < gm ? tiles_m - first : gm;
    const unsigned in = id - group * per_group;
    *tm = first + in % rows;
    *tn = in / rows;
}

}  // namespace
}  // namespace cxm
