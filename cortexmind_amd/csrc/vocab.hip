// What a model's logits say about tokens, and the logits' gradients: log
// probabilities of given tokens, the entropy, the likeliest tokens, and the
// divergence from a teacher's distribution over its top tokens.
//
// With z = scale x, m the row's largest x, u = (x - m) scale log2(e):
//   S = sum 2^u,  T = sum u 2^u
//   lse = scale m + ln S,  log p = (x - m) scale - ln S,
//   entropy = ln S - ln 2 T / S
//   d x = scale (d logp ([token] - p) - d entropy p (log p + entropy)),
//   d x = scale d loss (p - q) with p = exp(z - lse)
// Logits are read once.  A row belongs to a wave, or is cut into segments of a
// workgroup each, which the lanes hold in registers between the largest value,
// the sums and the selection of the top tokens; the last workgroup of a row to
// arrive joins the segments' m, S, T and tokens (in the segments' order).
// x - m comes before the product with the scale, so that a row of the type's
// lowest values is a row of equal ones, and u is kept at or above -1000, where
// 2^u is zero as it is at -infinity, so that u 2^u is no NaN there.
#include "chunk.hpp"

namespace cxm {
namespace {

inline hipStream_t hs(cxm_stream_t s) { return reinterpret_cast<hipStream_t>(s); }

constexpr float kLog2e = 0x1.715476p+0f, kLn2 = 0x1.62e430p-1f, kLow = -1000.0f;
constexpr unsigned kTopMost = 64;       // tokens that a call returns
constexpr unsigned kTeacherMost = 256;  // entries of a teacher's row
constexpr size_t kTicket = 16;          // words between two rows' tickets
constexpr int kStatChunks = 8, kStatFew = 7, kGradChunks = 4;  // (kStatFew: held to 64 registers, 8 waves of a SIMD)

__device__ __forceinline__ float fmax3(float a, float b) { return __builtin_elementwise_maximum(a, b); }

struct IntSumOp {
    using T = int;
    __device__ static T identity() { return 0; }
    __device__ static T combine(T a, T b) { return a + b; }
};
struct InfMaxOp : MaxOp {
    __device__ static T identity() { return -INFINITY; }
};

// m, S and T of some of a row's elements.
struct Part {
    float m, s, t;
};
// S and T with u counted from M instead.
__device__ __forceinline__ Part rebase(Part p, float M, float c) {
    const float base = M == -INFINITY ? 0.0f : M;
    const float d = fmax3((p.m - base) * c, kLow), f = __builtin_amdgcn_exp2f(d);
    return {M, p.s * f, fmaf(d, p.s, p.t) * f};
}

struct Logits {
    const void *x;
    size_t ld, rows;
    unsigned vocab, nseg, seglen;  // seglen: a multiple of 64
    float scale, c;                // c = scale log2(e)
    unsigned odd;                  // 1: some row's chunks begin an element earlier (shift_of)
};
// A chunk's place in its row, and which of its elements are its own: lo <= e < hi.
struct Own {
    unsigned off;
    int lo, hi;
    __device__ bool has(int e) const { return e >= lo && e < hi; }
};
// The chunk at column col - shift of a row, in a segment that ends at column
// end: moved back to the segment's last VE elements where it reaches past its
// end (which may lie before the segment), and on to the row's first where it
// begins before it.
template <int VE>
__device__ __forceinline__ Own own_of(unsigned col, unsigned shift, unsigned end) {
    const int c = static_cast<int>(col - shift), last = static_cast<int>(end) - VE;
    int off = c < last ? c : last;
    off = off > 0 ? off : 0;
    return {static_cast<unsigned>(off), c - off, c < 0 ? c + VE : VE};
}
// 1 for 16-bit rows that begin between two dwords: their chunks then begin an
// element earlier, at a dword (2500 fp16 rows of 50001 took 55 us at any element's
// address, of 50002 45).
template <int DT, int VE>
__device__ __forceinline__ unsigned shift_of(const void *row) {
    return DT == CXM_DT_F32 || VE == 1 ? 0u : static_cast<unsigned>(reinterpret_cast<uintptr_t>(row) >> 1 & 1);
}
// The elements that are not the chunk's own become -infinity.
template <int DT, int VE>
__device__ __forceinline__ void drop_others(Chunk<DT, VE> &c, Own o) {
    if (o.lo <= 0 && o.hi == VE) return;
    if constexpr (DT == CXM_DT_F32) {
#pragma unroll
        for (int e = 0; e < VE; ++e) c.r[e] = o.has(e) ? c.r[e] : -INFINITY;
    } else {
        constexpr unsigned inf = DT == CXM_DT_BF16 ? 0xff80u : 0xfc00u;
#pragma unroll
        for (int e = 0; e < VE; ++e)
            if (!o.has(e)) c.r[e / 2] = e & 1 ? (c.r[e / 2] & 0xffffu) | inf << 16 : (c.r[e / 2] & 0xffff0000u) | inf;
    }
}
// Stores a chunk's own elements; with the non-temporal hint, since a gradient that
// is no longer than the cache is rare (into memory that is not in the cache, bf16
// 2048x65500 96.1 -> 90.7 us, fp32 1000x30011 47.6 -> 45.2; into the same buffer over
// and over, 86.0 -> 91.1 and 42.9 -> 45.5).
template <int DT, int VE>
__device__ __forceinline__ void store_own(typename Elem<DT>::S *row, Own o, const Chunk<DT, VE> &c) {
    if (o.lo <= 0 && o.hi == VE) {
        c.store_nt(row + o.off);
    } else {
#pragma unroll
        for (int e = 0; e < VE; ++e)
            if (o.has(e)) row[o.off + e] = c.raw(e);
    }
}
// A segment of a row: its chunks begin at columns s0 - shift, s0 - shift + VE, ...
struct Seg {
    unsigned s0, end, shift;
    int its;  // chunks that some lane of this wave has, G lanes' VE elements apart
    __device__ unsigned begin() const { return s0 < shift ? 0 : s0 - shift; }
    template <int VE, int G>
    __device__ Own own(int i, unsigned lane) const {
        return own_of<VE>(s0 + (i * G + lane) * VE, shift, end);
    }
};
template <int DT, int VE, int G>
__device__ __forceinline__ Seg seg_of(const Logits &in, const void *row, unsigned number, unsigned lane) {
    Seg s;
    s.shift = shift_of<DT, VE>(row);
    s.s0 = number * in.seglen;
    const unsigned all = in.vocab + s.shift, to = all - s.s0 < in.seglen ? all : s.s0 + in.seglen;
    s.end = to - s.shift;
    const unsigned first = s.s0 + (__builtin_amdgcn_readfirstlane(lane / kWave) * kWave) * VE;
    s.its = first >= to ? 0 : static_cast<int>((to - first + G * VE - 1) / (G * VE));
    return s;
}

// The same value, which the compiler takes for a new one: what is computed from it
// is computed anew and not kept in registers (64 unpacked values, 64 masks) from
// one pass over a lane's chunks to the next.
__device__ __forceinline__ unsigned again(unsigned v) {
    asm volatile("" : "+v"(v));
    return v;
}
template <int DT, int VE>
__device__ __forceinline__ void again(Chunk<DT, VE> &c) {
    for (auto &r : c.r) asm volatile("" : "+v"(r));
}

// Barrier of G threads: a workgroup's, or a wave's own LDS accesses in order.
template <int G>
__device__ __forceinline__ void group_sync() {
    if constexpr (G == kBlock) __syncthreads();
    else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}
// Reduction over G threads, valid in all of them.  lds: one per wave of the workgroup.
template <class Op, int G>
__device__ __forceinline__ typename Op::T group_all(typename Op::T v, typename Op::T *lds) {
    if constexpr (G == kBlock) return block_reduce<Op, kBlock>(v, lds);
    else return wave_reduce<Op>(v);
}

struct StatArgs {
    Logits in;
    // log probabilities (kind 0)
    const int32_t *tokens;
    float *logp, *entropy, *lse;
    float *top_logp;
    int32_t *top_ids;
    unsigned top;
    // distillation (kind 1)
    const int32_t *ids;
    const float *teacher;
    float *loss;
    unsigned k;
    int kind;
    // segments
    Part *parts;      // [rows, nseg]
    ArgPair *cands;   // [rows, nseg, keep]
    float *bars;      // [rows, nseg, 2]: values that `top`, and `rth`, of the segment's tokens are not below
    unsigned rth, need;  // need segments' rth tokens are at least `top`
    unsigned keep;    // tokens a segment hands on, its `top` among them
    unsigned *tickets;
};

__device__ __forceinline__ bool better(ArgPair a, ArgPair b) { return a.v > b.v || (a.v == b.v && a.i < b.i); }

// The value whose bits, made ascending in the value's order, are `key` (no
// number's key: NaN, which compares false).
__device__ __forceinline__ float value_of(unsigned key) {
    return __builtin_bit_cast(float, key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// Bits of a 32-bit value that its type can have set: the others are all alike.
template <int DT>
constexpr int kLowBit = DT == CXM_DT_F32 ? 0 : DT == CXM_DT_BF16 ? 16 : 13;
// A value's bits, ascending in the value's order; zeros alike.
__device__ __forceinline__ unsigned key_of(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// A value that at least `n` of a wave's 64 J values are not below: the n-th
// largest, bit by bit, or less, where those not below it are at most `most`.
template <int DT, int J>
__device__ __forceinline__ float threshold(const float (&v)[J], unsigned n, unsigned most) {
    unsigned k[J], key = 0;
#pragma unroll
    for (int j = 0; j < J; ++j) k[j] = key_of(v[j]);
    auto step = [&](int b) {  // whether that is enough
        const unsigned t = key | 1u << b;
        unsigned c = 0;
#pragma unroll
        for (int j = 0; j < J; ++j) c += __popcll(__ballot(k[j] >= t));
        key = c >= n ? t : key;
        return c >= n && c <= most;
    };
#pragma nounroll
    for (int b = 31; b >= kLowBit<DT>; --b)
        if (step(b)) break;
    // (a negative value whose last bits are open stands for the lowest that begins so: nothing is lost)
    return key < 0x007fffffu ? -INFINITY : value_of(key);
}

// Chunk number i of a lane's, i known only when it runs: a few selections, where
// an indexed register array would go through memory, and loops over i stay small
// (the top tokens' code was 65 KB with all of them unrolled, past the instruction
// cache).
template <int DT, int VE, int C>
__device__ __forceinline__ Chunk<DT, VE> pick(const Chunk<DT, VE> (&c)[C], int i) {
    Chunk<DT, VE> r = c[0];
#pragma unroll
    for (int k = 1; k < C; ++k)
#pragma unroll
        for (int w = 0; w < static_cast<int>(sizeof(r.r) / sizeof(r.r[0])); ++w) r.r[w] = i == k ? c[k].r[w] : r.r[w];
    return r;
}

// LDS of a group.
struct Room {
    ArgPair *list, *best;  // room for kCap<G> and kTopMost tokens
    int *count;
    float *bar;
};
template <int J>
struct Width {
    static constexpr int value = J;
};
template <int G>
constexpr unsigned kCap = G == kBlock ? 512 : 128;

// Room for one more token in the list (the place may lie past it).  Each lane
// for itself: few have any, and the compiler's joint form is long.
__device__ __forceinline__ unsigned next_place(const Room &r) { return atomicAdd(r.count + again(0u), 1); }

// Sorts list[0 .. n) and keeps the first min(n, top) in it, in order: each
// token's place is the number of better ones.  Where there are many more than
// `top`, those below a value that `top` are not below leave first (512 tokens
// ranked among each other took 20 us).
template <int DT, int G, unsigned CAP>
__device__ __forceinline__ unsigned keep_top(const Room &r, unsigned n, unsigned top, unsigned lane) {
    group_sync<G>();
    if (n > top + top / 4 + 8) {
        constexpr int E = CAP / G;
        if (G != kBlock || lane < kWave) {
            // (as few values a lane as hold the list)
            auto bar = [&](auto width) {
                constexpr int J = decltype(width)::value;
                float v[J];
#pragma unroll
                for (int j = 0; j < J; ++j) v[j] = j * kWave + lane < n ? r.list[j * kWave + lane].v : -INFINITY;
                return threshold<DT, J>(v, top, top + top / 8);
            };
            const float t = n <= kWave ? bar(Width<1>{}) : n <= 2 * kWave ? bar(Width<2>{}) : bar(Width<CAP / kWave>{});
            if (lane == 0) {
                *r.bar = t;
                *r.count = 0;
            }
        }
        ArgPair mine[E];
#pragma unroll
        for (int e = 0; e < E; ++e) mine[e] = r.list[e * G + lane];  // (past n: not looked at)
        group_sync<G>();
        const float t = *r.bar;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e * G + lane < n && mine[e].v >= t) r.list[next_place(r)] = mine[e];
        group_sync<G>();
        n = *r.count;
    }
    for (unsigned i = lane; i < n; i += G) {
        const ArgPair mine = r.list[i];
        unsigned rank = 0;
#pragma unroll 8
        for (unsigned j = 0; j < n; ++j) rank += better(r.list[j], mine);
        if (rank < top) r.best[rank] = mine;
    }
    group_sync<G>();
    const unsigned kept = n < top ? n : top;
    for (unsigned i = lane; i < kept; i += G) r.list[i] = r.best[i];
    group_sync<G>();
    return kept;
}

// A teacher's row in a wave: entry j 64 + lane in place j, negative ids where there is none.
struct Teacher {
    static constexpr int E = kTeacherMost / kWave;
    int id[E];
    float v[E];
    __device__ __forceinline__ void load(const int32_t *ids, const float *values, unsigned k, unsigned lane) {
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const unsigned i = j * kWave + lane;
            id[j] = -1;
            if (i < k) {
                id[j] = ids[i];
                v[j] = values[i];
            }
        }
    }
};

// Log probabilities of a row whose sums are known, with its top tokens in r.list;
// or its divergence from the teacher.  By one wave.
template <int DT, bool ENT, bool TOP>
__device__ __forceinline__ void finish_row(const StatArgs &a, size_t row, Part p, const Room &r, const Teacher &t, unsigned lane) {
    using S = typename Elem<DT>::S;
    const S *x = static_cast<const S *>(a.in.x) + row * a.in.ld;
    if (!TOP && a.kind == 1) {
        // the teacher's tokens' logits, at once
        float at[Teacher::E], tm = -INFINITY;
#pragma unroll
        for (int j = 0; j < Teacher::E; ++j) {
            at[j] = 0.0f;
            if (t.id[j] < 0) continue;
            if (static_cast<unsigned>(t.id[j]) < a.in.vocab) at[j] = Elem<DT>::load(x[t.id[j]]);
            tm = fmax3(tm, static_cast<unsigned>(t.id[j]) < a.in.vocab ? t.v[j] : __builtin_nanf(""));
        }
        tm = wave_reduce<InfMaxOp>(tm);
        const float log_s = logf(p.s);
        float z = 0.0f, w = 0.0f;
        if (tm != -INFINITY && !__builtin_isnan(tm)) {
#pragma unroll
            for (int j = 0; j < Teacher::E; ++j) {
                if (t.id[j] < 0) continue;
                const float l = (t.v[j] - tm) * a.in.scale, e = expf(l);
                if (e == 0.0f) continue;
                z += e;
                w = fmaf(e, l - ((at[j] - p.m) * a.in.scale - log_s), w);
            }
        }
        z = wave_reduce<SumOp>(z);
        w = wave_reduce<SumOp>(w);
        if (lane == 0) {
            a.loss[row] = tm == -INFINITY ? 0.0f : __builtin_isnan(tm) ? tm : w / z - logf(z);
            if (a.lse) a.lse[row] = fmaf(a.in.scale, p.m, log_s);
        }
        return;
    }
    const float log_s = logf(p.s);
    auto logp = [&](float v) { return (v - p.m) * a.in.scale - log_s; };
    if constexpr (TOP) {
        const bool bad = __builtin_isnan(p.m);
        if (lane < a.top) {
            const ArgPair v = r.list[lane];
            a.top_ids[row * a.top + lane] = bad ? -1 : v.i;
            a.top_logp[row * a.top + lane] = bad ? __builtin_nanf("") : logp(v.v);
        }
    }
    if (lane == 0) {
        if (a.lse) a.lse[row] = fmaf(a.in.scale, p.m, log_s);
        if constexpr (ENT) {
            const float h = log_s - kLn2 * (p.t / p.s);
            a.entropy[row] = h < 0.0f ? 0.0f : h;
        }
        if (a.logp) {
            const int tok = a.tokens[row];
            a.logp[row] = tok < 0                                       ? 0.0f
                          : static_cast<unsigned>(tok) < a.in.vocab ? logp(Elem<DT>::load(x[tok]))
                                                                        : __builtin_nanf("");
        }
    }
}

// m, S and T of what a wave holds, from its largest value.
template <int DT, int VE, int C, bool ENT>
__device__ __forceinline__ Part again_from_the_largest(Chunk<DT, VE> (&c)[C], int its, float scale) {
    float m = -INFINITY, s = 0.0f, t = 0.0f;
#pragma nounroll
    for (int i = 0; i < its; ++i) {
        const Chunk<DT, VE> v = pick(c, i);
#pragma unroll
        for (int e = 0; e < VE; ++e) m = fmax3(m, v.get(e));
    }
    m = wave_reduce<InfMaxOp>(m);
    const float base = m == -INFINITY ? 0.0f : m;
#pragma nounroll
    for (int i = 0; i < its; ++i) {
        const Chunk<DT, VE> v = pick(c, i);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const float u = fmax3((v.get(e) - base) * scale, kLow), p = __builtin_amdgcn_exp2f(u);
            s += p;
            if constexpr (ENT) t = fmaf(u, p, t);
        }
    }
    return Part{m, wave_reduce<SumOp>(s), ENT ? wave_reduce<SumOp>(t) : 0.0f};
}

// The n best tokens of a segment whose lanes hold c exactly, where too many are
// not below the bar because they are equal: the value of the n-th bit by bit,
// then, of those equal to it, the last place that is taken.  Into the list.
template <int DT, int VE, int G, int C>
__device__ __forceinline__ void exact_top(const Chunk<DT, VE> (&c)[C], const Seg &seg, unsigned n, const Room &room,
                                          unsigned lane, int *lds) {
    // tokens above t, and those equal to it before place `to`: into the list with `keep`, else counted
    auto count = [&](float t, unsigned to, bool keep) {
        int k = 0;
#pragma nounroll
        for (int i = 0; i < seg.its; ++i) {
            const Own own = seg.own<VE, G>(i, lane);
            const Chunk<DT, VE> v = pick(c, i);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float x = v.get(e);
                const unsigned j = own.off + e;
                const bool in = own.has(e) && (x > t || (x == t && j < to));
                k += in;
                if (in && keep) room.list[next_place(room)] = ArgPair{x, static_cast<int>(j)};
            }
        }
        return static_cast<unsigned>(group_all<IntSumOp, G>(k, lds));
    };
    constexpr int places = 15;  // a segment has at most 2^14
    unsigned key = 0, place = 0;
    float t = 0.0f;
#pragma nounroll
    for (int step = 31; step >= kLowBit<DT> - places - 1; --step) {
        const bool value = step >= kLowBit<DT>, last = step == kLowBit<DT> - places - 1;
        const unsigned bit = value ? 1u << step : last ? 0u : 1u << (step - kLowBit<DT> + places);
        if (!value && step == kLowBit<DT> - 1) {  // all bits of the value are known
            if (!(key & 0x80000000u)) key |= (1u << kLowBit<DT>) - 1;  // a negative value's are counted from its other end
            t = key < 0x007fffffu ? -INFINITY : value_of(key);
        }
        if (last && lane == 0) *room.count = 0;
        if (last) group_sync<G>();
        const unsigned got = count(value ? value_of(key | bit) : t, value ? ~0u : last ? seg.begin() + place + 1 : seg.begin() + (place | bit), last);
        if (value && got >= n) key |= bit;
        if (!value && got < n) place |= bit;  // (before the last place that is taken there are fewer)
    }
    group_sync<G>();
}

// A row's top tokens, in order, from its segments' lists: those below the
// highest bar are left out as they are read.
template <int DT, int G, unsigned CAP>
__device__ __forceinline__ void join_top(const StatArgs &a, size_t row, const Room &room, unsigned lane, float *lds_f,
                                         int *lds_i) {
    constexpr int U = 4, J = 4;
    const float *bars = a.bars + row * a.in.nseg * 2;
    const size_t total = static_cast<size_t>(a.in.nseg) * a.keep;
    const ArgPair *cands = a.cands + row * total;
    ArgPair v[U];
    auto load = [&](size_t b) {
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = b + u * G + lane < total ? ld_dev(cands + b + u * G + lane) : ArgPair{-INFINITY, 0x7fffffff};
    };
    load(0);
    float low = -INFINITY;
    for (unsigned i = lane; i < a.in.nseg; i += G) low = fmax3(low, ld_dev(bars + 2 * i));
    low = group_all<InfMaxOp, G>(low, lds_f);
    // each of `need` segments has `rth` tokens not below its second bar
    if (a.in.nseg >= 16 && a.in.nseg <= J * kWave) {
        float second[J];
        if (lane < kWave) {
#pragma unroll
            for (int j = 0; j < J; ++j) second[j] = j * kWave + lane < a.in.nseg ? ld_dev(bars + 2 * (j * kWave + lane) + 1) : -INFINITY;
            const float t = threshold<DT, J>(second, a.need, 0);
            if (lane == 0) *room.bar = t;
        }
        group_sync<G>();
        low = fmax3(low, *room.bar);
    }
    unsigned have = 0;
    if (lane == 0) *room.count = 0;
    group_sync<G>();
    auto counted = [&] {
        group_sync<G>();
        have = *room.count;
        group_sync<G>();
    };
    bool fits = true;
    size_t b = 0;
    int u = 0;
    for (;;) {
        const bool done = b >= total;
        if (u == 0 && !done) {
            if (b) load(b);
            auto passing = [&] {
                int k = 0;
#pragma unroll
                for (int j = 0; j < U; ++j) k += v[j].v >= low && v[j].i != 0x7fffffff;
                return static_cast<unsigned>(group_all<IntSumOp, G>(k, lds_i));
            };
            fits = have + passing() <= CAP;
            if (!fits) {  // without those that the wave's own best ones leave out
                float w[U];
#pragma unroll
                for (int j = 0; j < U; ++j) w[j] = v[j].v;
                low = fmax3(low, threshold<DT, U>(w, a.top, a.top + a.top / 8));
                fits = have + passing() <= CAP;
            }
        }
        if (!fits && !done) counted();
        if (done || (!fits && have + G > CAP)) {  // (at most G more each time)
            have = keep_top<DT, G, CAP>(room, have, a.top, lane);
            if (done) break;
            if (lane == 0) *room.count = static_cast<int>(have);
            group_sync<G>();
        }
        ArgPair mine = v[0];
#pragma unroll
        for (int j = 1; j < U; ++j) {
            mine.v = u == j ? v[j].v : mine.v;
            mine.i = u == j ? v[j].i : mine.i;
        }
        if (mine.v >= low && mine.i != 0x7fffffff) room.list[next_place(room)] = mine;
        if (++u == U || b + u * G >= total) {
            counted();
            b += U * G;
            u = 0;
        }
    }
}

// A row per G lanes (nseg 1, G = 64) or a segment per workgroup; C chunks a lane.
// One read of the logits and the exponentials' issue bound it: 2048 rows of 131072
// bf16 distilled from 64 tokens 93.6 us (5.7 TB/s; over half of the cycles are vector
// work), 2500 of 50001 fp16 with entropy and 5 tokens 66.2 (3.8 TB/s; 46 without tokens),
// 16 of 131072 bf16 with 20 tokens 14.9, which is latency.  Rows with fewer unmasked
// logits than tokens wanted in a segment take the search of exact_top in each of
// them, and waves of -infinity (or of values far from zero) a second look at their
// values: with 10 logits of a row unmasked 174 us (16 of 131072), 2050 (2500 of 50001),
// and without tokens 172 for 87 (2048 of 131072); with 1000 unmasked no more than usual.
template <int DT, int VE, int G, int C, bool ENT, bool TOP>
__global__ __launch_bounds__(kBlock, C == kStatFew ? 8 : 1) void k_vocab_stats(StatArgs a) {
    using S = typename Elem<DT>::S;
    constexpr int NG = kBlock / G;
    __shared__ float lds_f[kBlock / kWave];
    __shared__ int lds_i[kBlock / kWave];
    __shared__ Part lds_p[kBlock / kWave];
    constexpr unsigned CAP = kCap<G>;
    __shared__ ArgPair lists[TOP ? NG : 1][TOP ? CAP : 1], bests[TOP ? NG : 1][TOP ? kTopMost : 1];
    __shared__ float peaks[TOP && G == kBlock ? kBlock : 1], bars[NG];  // peaks: each lane's largest value
    __shared__ int counts[NG], flag;
    const unsigned lane = threadIdx.x % G, grp = threadIdx.x / G;
    const Room room{lists[TOP ? grp : 0], bests[TOP ? grp : 0], &counts[grp], &bars[grp]};
    const size_t row = G == kBlock ? blockIdx.x / a.in.nseg : static_cast<size_t>(blockIdx.x) * NG + grp;
    if (row >= a.in.rows) return;  // a whole wave of a workgroup whose waves have rows of their own
    const unsigned number = G == kBlock ? blockIdx.x % a.in.nseg : 0;
    const S *x = static_cast<const S *>(a.in.x) + row * a.in.ld;
    const Seg seg = seg_of<DT, VE, G>(a.in, x, number, lane);
    Chunk<DT, VE> c[C];
    Teacher teacher;
    if (!TOP && a.kind == 1 && lane < kWave) teacher.load(a.ids + row * a.k, a.teacher + row * a.k, a.k, lane);
#pragma unroll
    for (int i = 0; i < C; ++i)
        if (i < seg.its) c[i].load_nt(x + seg.own<VE, G>(i, lane).off);
    // Without the top tokens one pass, with the largest of the wave's first chunks as m, which the others need
    // not be below: S then says whether they are by too much, and the sums are taken again from the largest of
    // all.  With them the largest values come first, and a wave finds the bar while the others go on.  z's product
    // with c is not rounded on its own; what m c lost is made up for where it is small (half a last place of m c:
    // with far logits that is more octaves than an exponential holds), else the sums are taken again too.
    [[maybe_unused]] const unsigned held = seg.end - seg.begin(), n0 = held < a.top ? held : a.top;
    [[maybe_unused]] float low = -INFINITY;  // the bar: at least `top` tokens are not below it, so none below it is wanted
    float cm[C], from = -INFINITY;           // each chunk's largest, all of them's
#pragma unroll
    for (int i = 0; i < C; ++i) cm[i] = -INFINITY;
    auto prepare = [&](int i) {
        // (only a wave's first and last chunks are shared with another)
        if (i == 0 || i + 1 >= seg.its) drop_others<DT, VE>(c[i], seg.own<VE, G>(i, again(lane)));
        if (!TOP && i) return;
        float a0 = -INFINITY, a1 = -INFINITY;
#pragma unroll
        for (int e = 0; e < VE; ++e) (e & 1 ? a1 : a0) = fmax3(e & 1 ? a1 : a0, c[i].get(e));
        cm[i] = fmax3(a0, a1);
        from = fmax3(from, cm[i]);
    };
    if constexpr (TOP) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
            if (i >= seg.its) break;
            prepare(i);
        }
        if (lane == 0) *room.count = 0;
        // (where most of the lanes that hold anything are wanted, stopping early would tell nothing)
        const unsigned near = 2 * n0 * VE <= held && 2 * n0 <= G ? n0 + n0 / 8 + 4 : 0;
        if constexpr (G == kBlock) {
            constexpr int NW = kBlock / kWave;
            // Few tokens: of the largest values of 64 groups of four lanes, as good a bar for a quarter of the work,
            // which the workgroup waits for (each instruction of one wave costs the turns of the SIMD's others).
            const bool few = a.top <= 24;
            float m = fmax3(from, dpp<kQuadXor1>(from));
            m = fmax3(m, dpp<kQuadXor2>(m));
            if (!few) peaks[lane] = from;
            else if (lane % 4 == 0) peaks[lane / 4] = m;
            __syncthreads();
            if (lane / kWave == number % NW) {
                float t, second = -INFINITY;
                const bool join = a.in.nseg >= 16;
                if (few) {
                    const float v[1] = {peaks[lane % kWave]};
                    t = threshold<DT, 1>(v, n0, 2 * n0 * 4 * VE <= held ? n0 + n0 / 8 + 2 : 0);
                    if (join) second = threshold<DT, 1>(v, a.rth, a.rth);
                } else {
                    float v[NW];
#pragma unroll
                    for (int j = 0; j < NW; ++j) v[j] = peaks[j * kWave + lane % kWave];
                    t = threshold<DT, NW>(v, n0, near);
                    if (join) second = threshold<DT, NW>(v, a.rth, a.rth);
                }
                if (lane % kWave == 0) {
                    bars[0] = t;
                    if (a.in.nseg > 1) {
                        st_dev(a.bars + 2 * (row * a.in.nseg + number), n0 < a.top ? -INFINITY : t);
                        st_dev(a.bars + 2 * (row * a.in.nseg + number) + 1, second);
                    }
                }
            }
        } else {
            const float v[1] = {from};
            low = threshold<DT, 1>(v, n0, near);
        }
    }
    Part p{-INFINITY, 0.0f, 0.0f};
    if (seg.its > 0) {
        float mc = 0.0f;
        float sum[2] = {0.0f, 0.0f}, ent[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < C; ++i) {
            if (i >= seg.its) break;
            if constexpr (TOP) again(c[i]);
            else prepare(i);
            if (i == 0) {
                from = wave_reduce<InfMaxOp>(from);
                mc = from * a.in.c;
            }
            float u[VE], q[VE];
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                u[e] = fmaf(c[i].get(e), a.in.c, -mc);
                if constexpr (ENT) u[e] = fmax3(u[e], kLow);
            }
#pragma unroll
            for (int e = 0; e < VE; ++e) q[e] = __builtin_amdgcn_exp2f(u[e]);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                sum[e & 1] += q[e];
                if constexpr (ENT) ent[e & 1] = fmaf(u[e], q[e], ent[e & 1]);
            }
        }
        p = Part{from, wave_reduce<SumOp>(sum[0] + sum[1]), ENT ? wave_reduce<SumOp>(ent[0] + ent[1]) : 0.0f};
        // 64: S keeps what lies up to 60 octaves below m, and the rounding of u, 2^-19, is 22 of S's own.  T, a sum of
        // terms as large as lost, would lose as many times its own roundings: 1.  (NaN, and an infinite m: not below.)
        const float lost = -fmaf(from, a.in.c, -mc);
        if (fabsf(lost) < (ENT ? 1.0f : 64.0f) && p.s < 0x1p20f) {
            const float f = __builtin_amdgcn_exp2f(lost);
            p = Part{from, p.s * f, fmaf(lost, p.s, p.t) * f};
        } else {
            p = again_from_the_largest<DT, VE, C, ENT>(c, seg.its, a.in.c);
        }
    }
    if constexpr (G == kBlock) {
        constexpr int NW = kBlock / kWave;
        if (lane % kWave == 0) lds_p[lane / kWave] = p;
        __syncthreads();
        const Part one = lds_p[lane % NW];  // every four lanes for themselves
        static_assert(NW == 4, "the sums below are over four lanes");
        const float top = group_reduce<InfMaxOp, NW>(one.m);
        const Part v = rebase(one, top, a.in.c);
        const Part q{top, group_reduce<SumOp, NW>(v.s), ENT ? group_reduce<SumOp, NW>(v.t) : 0.0f};
        p = q;
    }
    unsigned n = 0;  // tokens in the list
    if constexpr (TOP) {
        if constexpr (G == kBlock) low = bars[0];
        if (!__builtin_isnan(p.m)) {
            if constexpr (G != kBlock) group_sync<G>();
            // the chunks that have such tokens, one per lane at a time
            unsigned hits = 0;
#pragma unroll
            for (int i = 0; i < C; ++i) hits |= i < seg.its && cm[i] >= low ? 1u << i : 0u;
#pragma nounroll
            while (__any(hits != 0)) {
                const int i = hits ? __builtin_ctz(hits) : 0;
                const Own own = seg.own<VE, G>(i, lane);
                const Chunk<DT, VE> v = pick(c, i);
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    if (hits && v.get(e) >= low && own.has(e)) {
                        const unsigned at = next_place(room);
                        if (at < CAP) room.list[at] = ArgPair{v.get(e), static_cast<int>(own.off + e)};
                    }
                }
                hits &= hits - 1;
            }
            group_sync<G>();
            n = *room.count;
            if (n > CAP) {
                exact_top<DT, VE, G, C>(c, seg, n0, room, lane, lds_i);
                n = n0;
            }
            if (G != kBlock || a.in.nseg == 1 || n > a.keep) n = keep_top<DT, G, CAP>(room, n, n0, lane);
        }
    }
    if constexpr (G == kBlock) {
        if (a.in.nseg > 1) {
            const size_t at = row * a.in.nseg + number;
            if (lane == 0) {
                float *to = &a.parts[at].m;
                st_dev(to, p.m);
                st_dev(to + 1, p.s);
                st_dev(to + 2, p.t);
            }
            if constexpr (TOP) {
                for (unsigned i = lane; i < a.keep; i += G)
                    st_dev(a.cands + at * a.keep + i, i < n ? room.list[i] : ArgPair{-INFINITY, 0x7fffffff});
            }
            if (!last_block_ticket(a.tickets + row * kTicket, a.in.nseg, &flag)) return;
            if (!TOP && lane >= kWave) return;
            // every wave for itself
            const float *parts = &a.parts[row * a.in.nseg].m;
            const unsigned l = lane % kWave;
            const Part one = l < a.in.nseg ? Part{ld_dev(parts + 3 * l), ld_dev(parts + 3 * l + 1), ld_dev(parts + 3 * l + 2)}
                                           : Part{-INFINITY, 0.0f, 0.0f};
            float top = one.m;
            for (unsigned i = l + kWave; i < a.in.nseg; i += kWave) top = fmax3(top, ld_dev(parts + 3 * i));
            top = wave_reduce<InfMaxOp>(top);
            Part q = rebase(one, top, a.in.c);
            for (unsigned i = l + kWave; i < a.in.nseg; i += kWave) {
                const Part v = rebase(Part{ld_dev(parts + 3 * i), ld_dev(parts + 3 * i + 1), ld_dev(parts + 3 * i + 2)}, top, a.in.c);
                q.s += v.s;
                q.t += v.t;
            }
            p = Part{top, wave_reduce<SumOp>(q.s), wave_reduce<SumOp>(q.t)};
            if constexpr (TOP) {
                if (a.in.nseg * a.keep <= 512) {  // few enough for one wave, without barriers
                    if (lane >= kWave) return;
                    if (!__builtin_isnan(p.m)) join_top<DT, kWave, CAP>(a, row, room, lane, lds_f, lds_i);
                } else {
                    if (!__builtin_isnan(p.m)) join_top<DT, G, CAP>(a, row, room, lane, lds_f, lds_i);
                }
            }
        }
    }
    if (lane < kWave) finish_row<DT, ENT, TOP>(a, row, p, room, teacher, lane);
}

struct GradArgs {
    Logits in;
    const float *lse;
    void *dx;
    size_t ldd;
    // log probabilities
    const int32_t *tokens;
    const float *entropy, *dlogp, *dentropy;
    // distillation
    const int32_t *ids;
    const float *teacher, *dloss;
    unsigned k;
};

// What a row's log probabilities are counted from: log p = scale (x - from) - less.
struct Base {
    float from, less;
};
// lse is fp32: its rounding moves every p = exp(scale x - lse) of the row by up to 2^-24 |lse| of itself, past 2^24 by
// factors (a row of a mask's value alone, or of the type's lowest, would have p = 1 everywhere, not 1 / vocab).
// From 2^12 on, where that is more than the roundings of fp16, a row is counted from its own largest value, as in
// the forward pass, by one workgroup alone: in place the others' parts are gone once they have stored.  Such rows are
// read three times.
constexpr float kFarLse = 4096.0f;

// The base of a row by G lanes: its largest value and the log of its sum, if lse is theirs, else lse (which is
// then of more logits than these).  The same row's, summed otherwise, differ by less than 4 of lse's last places.
template <int DT, int VE, int G, int U>
__device__ __forceinline__ Base far_base(const Logits &in, const typename Elem<DT>::S *x, float lse, unsigned lane, float *lds) {
    auto each = [&](auto &&take) {
#pragma nounroll
        for (unsigned n = 0; n < in.nseg; ++n) {
            const Seg seg = seg_of<DT, VE, G>(in, x, n, lane);
#pragma nounroll
            for (int from = 0; from < seg.its; from += U) {
                Chunk<DT, VE> c[U];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (from + u < seg.its) c[u].load(x + seg.own<VE, G>(from + u, lane).off);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (from + u >= seg.its) break;
                    drop_others<DT, VE>(c[u], seg.own<VE, G>(from + u, again(lane)));
                    take(c[u]);
                }
            }
        }
    };
    float m = -INFINITY, s = 0.0f;
    each([&](const Chunk<DT, VE> &c) {
#pragma unroll
        for (int e = 0; e < VE; ++e) m = fmax3(m, c.get(e));
    });
    m = group_all<InfMaxOp, G>(m, lds);
    each([&](const Chunk<DT, VE> &c) {
        float t = 0.0f;
#pragma unroll
        for (int e = 0; e < VE; ++e) t += __builtin_amdgcn_exp2f((c.get(e) - m) * in.c);
        s += t;
    });
    const float log_s = logf(group_all<SumOp, G>(s, lds)), own = fmaf(in.scale, m, log_s);
    const bool same = own == lse || (__builtin_isfinite(lse) && fabsf(own - lse) <= fabsf(lse) * 0x1p-22f);
    return same ? Base{m, log_s} : Base{0.0f, lse};
}

// A row per G lanes or a segment per workgroup, as above.  Each wave finds out by
// itself whether the row has a gradient; the teacher's probabilities and the
// gradients of its tokens in the segment are the first wave's, which stores them
// over the others'.  One read and one write bound it: bf16 2048x65500 with entropy
// 91.0 us (5.9 TB/s), fp32 1000x30011 from 17 tokens 45.4 (5.3), bf16 2048x131072
// from 64 178 (6.0).
template <int DT, int VE, int G, int C, bool DISTILL, bool ENT>
__global__ __launch_bounds__(kBlock) void k_vocab_grad(GradArgs a) {
    using S = typename Elem<DT>::S;
    constexpr int NG = kBlock / G, E = Teacher::E;
    __shared__ float qs[DISTILL ? NG : 1][DISTILL ? kTeacherMost : 1];
    __shared__ alignas(16) int qi[DISTILL ? NG : 1][DISTILL ? kTeacherMost : 1];
    [[maybe_unused]] __shared__ float ql[DISTILL ? NG : 1][DISTILL ? kTeacherMost : 1];  // (of a far row)
    __shared__ float lds[kBlock / kWave];
    const unsigned lane = threadIdx.x % G, grp = threadIdx.x / G;
    const size_t row = G == kBlock ? blockIdx.x / a.in.nseg : static_cast<size_t>(blockIdx.x) * NG + grp;
    if (row >= a.in.rows) return;  // a whole wave of a workgroup whose waves have rows of their own
    const S *x = static_cast<const S *>(a.in.x) + row * a.in.ld;
    S *dx = static_cast<S *>(a.dx) + row * a.ldd;
    const unsigned number = G == kBlock ? blockIdx.x % a.in.nseg : 0;
    const Seg seg = seg_of<DT, VE, G>(a.in, x, number, lane);
    Chunk<DT, VE> c[C];
    Own own[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
        own[i] = seg.own<VE, G>(i, lane);
        if (i < seg.its) c[i].load_nt(x + own[i].off);
    }
    const float lse = a.lse[row];
    // d x = p (slope + bend (log p)) + what the tokens get
    float slope, bend = 0.0f, given = 0.0f;
    unsigned token = ~0u;
    [[maybe_unused]] float late[E], tm = -INFINITY;  // the gradient at the teacher's tokens of this segment
    [[maybe_unused]] Teacher t;
    if constexpr (DISTILL) {
        t.load(a.ids + row * a.k, a.teacher + row * a.k, a.k, lane % kWave);
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (t.id[j] >= 0) tm = fmax3(tm, static_cast<unsigned>(t.id[j]) < a.in.vocab ? t.v[j] : __builtin_nanf(""));
        tm = wave_reduce<InfMaxOp>(tm);
        slope = tm == -INFINITY ? 0.0f : __builtin_isnan(tm) ? tm : a.dloss[row] * a.in.scale;
    } else {
        const int tok = a.tokens ? a.tokens[row] : -1;
        const float g = tok < 0 || !a.dlogp ? 0.0f : static_cast<unsigned>(tok) < a.in.vocab ? a.dlogp[row] : __builtin_nanf("");
        slope = -g * a.in.scale;
        if (tok >= 0) {
            token = tok;
            given = g * a.in.scale;
        }
        if constexpr (ENT) {
            bend = -a.dentropy[row] * a.in.scale;
            slope = bend == 0.0f ? slope : fmaf(bend, a.entropy[row], slope);
        }
    }
    const bool none = slope == 0.0f && bend == 0.0f && given == 0.0f;  // zeros, whatever the logits are
    // a chunk's gradient, in its place
    auto grad_of = [&](Chunk<DT, VE> &c, const Own &own, auto &&log_p) {
        float l[VE], p[VE], v[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            l[e] = log_p(c.get(e));
            if constexpr (ENT) l[e] = fmax3(l[e], kLow);
        }
#pragma unroll
        for (int e = 0; e < VE; ++e) p[e] = __builtin_amdgcn_exp2f(l[e] * kLog2e);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            if constexpr (ENT) v[e] = p[e] * fmaf(bend, l[e], slope);
            else v[e] = p[e] * slope;
            if constexpr (!DISTILL) v[e] += own.off + e == token ? given : 0.0f;
            v[e] = none ? 0.0f : v[e];
        }
        c.set(v);
        store_own<DT, VE>(dx, own, c);
    };
    auto usual = [&]() __attribute__((always_inline)) {
        if constexpr (DISTILL) {
            if (lane < kWave) {
                float at[E], q[E], z = 0.0f;
                bool mine[E];
#pragma unroll
                for (int j = 0; j < E; ++j) {  // what the dense gradient may be stored over
                    mine[j] = t.id[j] >= static_cast<int>(seg.begin()) && t.id[j] < static_cast<int>(seg.end);
                    at[j] = mine[j] ? Elem<DT>::load(x[t.id[j]]) : 0.0f;
                    q[j] = t.id[j] < 0 ? 0.0f : expf((t.v[j] - (tm == -INFINITY ? 0.0f : tm)) * a.in.scale);
                    z += q[j];
                }
                z = wave_reduce<SumOp>(z);
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    q[j] /= z;
                    qs[grp][j * kWave + lane] = q[j];
                    qi[grp][j * kWave + lane] = mine[j] ? t.id[j] : -1;
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    if (!__any(mine[j])) continue;
                    // a token may be there more than once
                    int times = 0;
                    for (unsigned i = 0; i < (a.k + 3) / 4; ++i) {
                        const int4 v = reinterpret_cast<const int4 *>(qi[grp])[i];
                        times += (v.x == t.id[j]) + (v.y == t.id[j]) + (v.z == t.id[j]) + (v.w == t.id[j]);
                    }
                    float all = q[j];
                    if (__any(mine[j] && times > 1)) {
                        all = 0.0f;
                        for (unsigned i = 0; i < a.k; ++i) all += qi[grp][i] == t.id[j] ? qs[grp][i] : 0.0f;
                    }
                    const float p = __builtin_amdgcn_exp2f(fmaf(a.in.scale, at[j], -lse) * kLog2e);
                    late[j] = slope == 0.0f ? 0.0f : slope * (p - all);
                    if (!mine[j]) t.id[j] = -1;
                }
            }
        }
        if (DISTILL && a.dx == a.in.x) {  // not before the teacher's tokens have been read
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            group_sync<G>();
        }
#pragma unroll
        for (int i = 0; i < C; ++i) {
            if (i >= seg.its) break;
            // (with a teacher the chunks' places are found anew: 64 registers, 70 where they are kept)
            grad_of(c[i], DISTILL ? seg.own<VE, G>(i, again(lane)) : own[i], [&](float v) { return fmaf(a.in.scale, v, -lse); });
        }
        if constexpr (DISTILL) {
            // over what was stored above, by whichever lane
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            group_sync<G>();
            if (lane < kWave) {
#pragma unroll
                for (int j = 0; j < E; ++j)
                    if (t.id[j] >= static_cast<int>(seg.begin()) && t.id[j] < static_cast<int>(seg.end))
                        dx[t.id[j]] = Elem<DT>::store(__builtin_isnan(slope) ? slope : late[j]);
            }
        }
    };
    auto far_row = [&]() __attribute__((always_inline)) {
        // one of the row's workgroups, and the chip's XCDs, which take workgroups in turn, in turn (always the first: 864 us
        // for 2048 rows of 65500 bf16 in 8 segments, all of them on one XCD)
        if (number != row * (a.in.nseg < 8 ? a.in.nseg : 8) / 8 % a.in.nseg) return;
        const unsigned l = again(lane);
        const Base base = far_base<DT, VE, G, DISTILL || C == 1 ? 1 : C>(a.in, x, lse, l, lds);
        auto log_p = [&](float v) { return fmaf(a.in.scale, v - base.from, -base.less); };
        auto entry = [&](unsigned i) {  // the id of the teacher's entry i, negative where there is none
            const int id = a.ids[row * a.k + i];
            return static_cast<unsigned>(id) < a.in.vocab ? id : -1;
        };
        if constexpr (DISTILL) {
            if (l < kWave) {
                float z = 0.0f;
#pragma nounroll
                for (unsigned i = l; i < a.k; i += kWave) {
                    const int id = entry(i);
                    const float q = id < 0 ? 0.0f : expf((a.teacher[row * a.k + i] - tm) * a.in.scale);
                    qi[grp][i] = id;
                    qs[grp][i] = q;
                    z += q;
                }
                z = wave_reduce<SumOp>(z);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma nounroll
                for (unsigned i = l; i < a.k; i += kWave) {
                    const int id = qi[grp][i];
                    if (id < 0) continue;
                    float all = 0.0f;
#pragma nounroll
                    for (unsigned j = 0; j < a.k; ++j) all += qi[grp][j] == id ? qs[grp][j] : 0.0f;
                    const float p = __builtin_amdgcn_exp2f(log_p(Elem<DT>::load(x[id])) * kLog2e);
                    ql[grp][i] = slope * (p - all / z);
                }
            }
            group_sync<G>();  // the teacher's tokens have been read
        }
#pragma nounroll
        for (unsigned n = 0; n < a.in.nseg; ++n) {
            const Seg each = seg_of<DT, VE, G>(a.in, x, n, l);
#pragma nounroll
            for (int i = 0; i < each.its; ++i) {
                const Own at = each.own<VE, G>(i, l);
                Chunk<DT, VE> v;
                v.load(x + at.off);
                grad_of(v, at, log_p);
            }
        }
        if constexpr (DISTILL) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            group_sync<G>();
            if (l < kWave)
#pragma nounroll
                for (unsigned i = l; i < a.k; i += kWave)
                    if (qi[grp][i] >= 0) dx[qi[grp][i]] = Elem<DT>::store(ql[grp][i]);
        }
    };
    // The same for all of a wave.  Said so, and asked in the way that keeps each path's registers out of the other (64 at
    // most, 8 waves of a SIMD; the other way round up to 72).
    if constexpr (DISTILL) {
        if (__builtin_amdgcn_readfirstlane(none || !(fabsf(lse) >= kFarLse))) return usual();
        far_row();
    } else {
        if (__builtin_amdgcn_readfirstlane(!none && fabsf(lse) >= kFarLse)) return far_row();
        usual();
    }
}

// ----------------------------------------------------------------- launch

// Cuts rows into segments of at most `most` elements, and of fewer (but a chunk
// for every lane) where there would be fewer workgroups than fill the chip.
void cut(Logits *in, unsigned most, unsigned least, size_t wgs) {
    const size_t all = static_cast<size_t>(in->vocab) + in->odd;
    size_t nseg = (all + most - 1) / most;
    const size_t want = (wgs + in->rows - 1) / in->rows, can = (all + least - 1) / least;
    if (nseg < want) nseg = want < can ? want : can;
    const size_t len = (all + nseg - 1) / nseg;
    in->seglen = static_cast<unsigned>((len + 63) / 64 * 64);
    in->nseg = static_cast<unsigned>((all + in->seglen - 1) / in->seglen);
}

// Whether a wave holds a row of C chunks a lane, and there are rows enough to give each wave one.
bool wave_rows(const Logits &in, unsigned chunk, unsigned chunks) {
    return in.vocab + in.odd <= 64 * chunk * chunks && (in.vocab <= 64 * chunk || in.rows >= 4 * device_cus());
}

template <int DT, int VE, int G, bool ENT, bool TOP, int C = VE == 1 ? 1 : kStatChunks>
int stats_launch(const StatArgs &a, hipStream_t s) {
    const size_t wgs = G == kBlock ? a.in.rows * a.in.nseg : (a.in.rows + kBlock / G - 1) / (kBlock / G);
    hipLaunchKernelGGL((k_vocab_stats<DT, VE, G, C, ENT, TOP>), dim3(static_cast<unsigned>(wgs)), dim3(kBlock), 0, s, a);
    return launch_status();
}

template <int DT, bool ENT, bool TOP>
int stats(StatArgs a, cxm_stream_t st) {
    constexpr int VE = Elem<DT>::kVec;
    a.in.nseg = 1;
    a.in.seglen = (a.in.vocab + a.in.odd + 63) / 64 * 64;
    const bool wave = a.in.vocab < static_cast<unsigned>(VE) || wave_rows(a.in, VE, kStatChunks);
    // with top tokens fewer and larger segments, since joining them takes longer: 16 rows of 131072 bf16 and 64
    // tokens 22.9 us on 256 workgroups, 25.7 on 512
    if (!wave) cut(&a.in, kBlock * VE * kStatChunks, kBlock * VE * (TOP ? 2 : 1), (TOP ? 1 : 4) * device_cus());
    if (a.in.nseg > most_wgs(kBlock) / a.in.rows) return CXM_E_TOO_LARGE;
    if (wave) {
        return a.in.vocab < static_cast<unsigned>(VE) ? stats_launch<DT, 1, 64, ENT, TOP>(a, hs(st))
                                                      : stats_launch<DT, VE, 64, ENT, TOP>(a, hs(st));
    }
    if (a.in.nseg > 1) {
        const size_t segs = a.in.rows * a.in.nseg, o_bars = (segs * sizeof(Part) + 255) / 256 * 256;
        const size_t o_cands = o_bars + (TOP ? (segs * 2 * sizeof(float) + 255) / 256 * 256 : 0);
        a.keep = a.top + a.top / 2 + 12;
        a.rth = (2 * a.top + a.in.nseg - 1) / a.in.nseg;
        a.need = TOP ? (a.top + a.rth - 1) / a.rth : 0;
        Workspace ws;
        const int rc = get_workspace(st, (a.in.rows * kTicket + kCtr - 1) / kCtr,
                                     o_cands + (TOP ? segs * a.keep * sizeof(ArgPair) : 0), &ws);
        if (rc) return rc;
        a.tickets = ws.counters;
        a.parts = static_cast<Part *>(ws.scratch);
        a.bars = reinterpret_cast<float *>(static_cast<char *>(ws.scratch) + o_bars);
        a.cands = reinterpret_cast<ArgPair *>(static_cast<char *>(ws.scratch) + o_cands);
    }
    // 16-bit segments of 8 chunks a lane take 71 registers, 7 waves of a SIMD; of 7 chunks, where that holds them, 64
    // and 8 waves: 2500 rows of 50001 fp16 and 5 tokens 66.0 us instead of 73.2 (68.3 at 66 registers and 7 waves; held
    // to 64 registers, 8 chunks spill: 71.8 there, but 512 rows of 131072 bf16 and 20 tokens 46.3 instead of 43.8).  The
    // cut does not aim at 7: with many rows 50001 is 4 segments of 12544, but 32000, 65536 and 131072 are segments of 16000
    // to 16384, which have 7 waves; fewer chunks and more segments there have not been timed.
    if constexpr (VE == 8 && ENT && TOP) {
        if (a.in.seglen <= kBlock * VE * kStatFew) return stats_launch<DT, VE, kBlock, ENT, TOP, kStatFew>(a, hs(st));
    }
    return stats_launch<DT, VE, kBlock, ENT, TOP>(a, hs(st));
}

template <int DT>
int stats_any(const StatArgs &a, cxm_stream_t st) {
    if (a.top) return a.entropy ? stats<DT, true, true>(a, st) : stats<DT, false, true>(a, st);
    return a.entropy ? stats<DT, true, false>(a, st) : stats<DT, false, false>(a, st);
}
int stats_any(const StatArgs &a, int dtype, cxm_stream_t st) {
    switch (dtype) {
        case CXM_DT_F32: return stats_any<CXM_DT_F32>(a, st);
        case CXM_DT_BF16: return stats_any<CXM_DT_BF16>(a, st);
        default: return stats_any<CXM_DT_F16>(a, st);
    }
}

template <int DT, int VE, int G, bool DISTILL, bool ENT>
int grad_launch(const GradArgs &a, hipStream_t s) {
    constexpr int C = VE == 1 ? 1 : kGradChunks;
    const size_t wgs = G == kBlock ? a.in.rows * a.in.nseg : (a.in.rows + kBlock / G - 1) / (kBlock / G);
    hipLaunchKernelGGL((k_vocab_grad<DT, VE, G, C, DISTILL, ENT>), dim3(static_cast<unsigned>(wgs)), dim3(kBlock), 0, s, a);
    return launch_status();
}

template <int DT, bool DISTILL, bool ENT>
int grad(GradArgs a, cxm_stream_t st) {
    constexpr int VE = Elem<DT>::kVec;
    a.in.nseg = 1;
    a.in.seglen = (a.in.vocab + a.in.odd + 63) / 64 * 64;
    const bool wave = a.in.vocab < static_cast<unsigned>(VE) || wave_rows(a.in, VE, kGradChunks);
    if (!wave) cut(&a.in, kBlock * VE * kGradChunks, kBlock * VE, 4 * device_cus());
    if (a.in.nseg > most_wgs(kBlock) / a.in.rows) return CXM_E_TOO_LARGE;
    if (a.in.vocab < static_cast<unsigned>(VE)) return grad_launch<DT, 1, 64, DISTILL, ENT>(a, hs(st));
    return wave ? grad_launch<DT, VE, 64, DISTILL, ENT>(a, hs(st)) : grad_launch<DT, VE, kBlock, DISTILL, ENT>(a, hs(st));
}

template <bool DISTILL, bool ENT>
int grad_any(const GradArgs &a, int dtype, cxm_stream_t st) {
    switch (dtype) {
        case CXM_DT_F32: return grad<CXM_DT_F32, DISTILL, ENT>(a, st);
        case CXM_DT_BF16: return grad<CXM_DT_BF16, DISTILL, ENT>(a, st);
        default: return grad<CXM_DT_F16, DISTILL, ENT>(a, st);
    }
}

// Bytes from the first element to past the last of rows of `vocab` elements, ld apart.
size_t span_bytes(size_t rows, size_t ld, size_t vocab, size_t e) { return rows ? ((rows - 1) * ld + vocab) * e : 0; }

// What all four entries ask of the logits.
int check_logits(const void *x, size_t ld, float scale, size_t rows, size_t vocab, int dtype) {
    if (!is_float_dtype(dtype) || !(scale > 0.0f) || !__builtin_isfinite(scale) || vocab == 0 || ld < vocab) return CXM_E_INVALID;
    if (rows && !x) return CXM_E_INVALID;
    // a row's columns are numbered in 32 bits, past its end too
    if (vocab > 0x7fff0000u || (rows && ld > (size_t(1) << 46) / rows) || rows > most_wgs(kBlock)) return CXM_E_TOO_LARGE;
    return CXM_OK;
}

struct Region {
    const void *p;
    size_t n;
};
// Whether an output meets an input or another output.
template <int NO, int NI>
bool any_overlap(const Region (&out)[NO], const Region (&in)[NI]) {
    for (int i = 0; i < NO; ++i) {
        for (int j = 0; j < NI; ++j)
            if (overlap(out[i].p, out[i].n, in[j].p, in[j].n)) return true;
        for (int j = 0; j < i; ++j)
            if (overlap(out[i].p, out[i].n, out[j].p, out[j].n)) return true;
    }
    return false;
}

Logits logits_of(const void *x, size_t ld, float scale, size_t rows, size_t vocab, int dtype) {
    const unsigned odd = dtype != CXM_DT_F32 && ((reinterpret_cast<uintptr_t>(x) >> 1 | ld) & 1);
    return Logits{x, ld, rows, static_cast<unsigned>(vocab), 1, 0, scale, scale * kLog2e, odd};
}

}  // namespace
}  // namespace cxm

extern "C" {

int cxm_logprob_fwd_t(const void *logits, size_t ld, const int32_t *tokens, float scale, float *logp, float *entropy,
                      float *lse, float *top_logp, int32_t *top_ids, size_t top, size_t rows, size_t vocab, int dtype,
                      cxm_stream_t s) {
    const int rc = cxm::check_logits(logits, ld, scale, rows, vocab, dtype);
    if (rc) return rc;
    if (top > cxm::kTopMost || top > vocab || (logp && !tokens) || (top && (!top_logp || !top_ids)) ||
        (!logp && !entropy && !lse && !top))
        return CXM_E_INVALID;
    if (rows == 0) return CXM_OK;
    const size_t r4 = rows * 4;
    const cxm::Region out[5] = {{logp, r4}, {entropy, r4}, {lse, r4}, {top ? top_logp : nullptr, r4 * top},
                                {top ? top_ids : nullptr, r4 * top}};
    const cxm::Region in[2] = {{logits, cxm::span_bytes(rows, ld, vocab, cxm::dtype_bytes(dtype))}, {tokens, r4}};
    if (cxm::any_overlap(out, in)) return CXM_E_INVALID;
    cxm::StatArgs a{};
    a.in = cxm::logits_of(logits, ld, scale, rows, vocab, dtype);
    a.tokens = tokens;
    a.logp = logp;
    a.entropy = entropy;
    a.lse = lse;
    a.top_logp = top_logp;
    a.top_ids = top_ids;
    a.top = static_cast<unsigned>(top);
    return cxm::stats_any(a, dtype, s);
}

int cxm_distill_fwd_t(const void *logits, size_t ld, const int32_t *ids, const float *teacher, size_t k, float scale,
                      float *loss, float *lse, size_t rows, size_t vocab, int dtype, cxm_stream_t s) {
    const int rc = cxm::check_logits(logits, ld, scale, rows, vocab, dtype);
    if (rc) return rc;
    if (k == 0 || k > cxm::kTeacherMost) return CXM_E_INVALID;
    if (rows == 0) return CXM_OK;
    if (!ids || !teacher || !loss) return CXM_E_INVALID;
    const size_t r4 = rows * 4;
    const cxm::Region out[2] = {{loss, r4}, {lse, r4}};
    const cxm::Region in[3] = {{logits, cxm::span_bytes(rows, ld, vocab, cxm::dtype_bytes(dtype))}, {ids, r4 * k}, {teacher, r4 * k}};
    if (cxm::any_overlap(out, in)) return CXM_E_INVALID;
    cxm::StatArgs a{};
    a.in = cxm::logits_of(logits, ld, scale, rows, vocab, dtype);
    a.ids = ids;
    a.teacher = teacher;
    a.loss = loss;
    a.lse = lse;
    a.k = static_cast<unsigned>(k);
    a.kind = 1;
    return cxm::stats_any(a, dtype, s);
}

int cxm_logprob_bwd_t(const void *logits, size_t ld, const int32_t *tokens, float scale, const float *lse,
                      const float *entropy, const float *dlogp, const float *dentropy, void *dlogits, size_t ldd,
                      size_t rows, size_t vocab, int dtype, cxm_stream_t s) {
    const int rc = cxm::check_logits(logits, ld, scale, rows, vocab, dtype);
    if (rc) return rc;
    if (ldd < vocab || (dlogp && !tokens) || (dentropy && !entropy) || (!dlogp && !dentropy)) return CXM_E_INVALID;
    if (rows == 0) return CXM_OK;
    if (ldd > (size_t(1) << 46) / rows) return CXM_E_TOO_LARGE;
    if (!lse || !dlogits) return CXM_E_INVALID;
    const size_t r4 = rows * 4, e = cxm::dtype_bytes(dtype), n = cxm::span_bytes(rows, ld, vocab, e);
    const cxm::Region out[1] = {{dlogits, cxm::span_bytes(rows, ldd, vocab, e)}};
    const bool in_place = dlogits == logits && ldd == ld;
    const cxm::Region in[6] = {{in_place ? nullptr : logits, n}, {tokens, r4}, {lse, r4}, {entropy, r4}, {dlogp, r4}, {dentropy, r4}};
    if (cxm::any_overlap(out, in)) return CXM_E_INVALID;
    cxm::GradArgs a{};
    a.in = cxm::logits_of(logits, ld, scale, rows, vocab, dtype);
    a.lse = lse;
    a.dx = dlogits;
    a.ldd = ldd;
    a.tokens = tokens;
    a.entropy = entropy;
    a.dlogp = dlogp;
    a.dentropy = dentropy;
    return dentropy ? cxm::grad_any<false, true>(a, dtype, s) : cxm::grad_any<false, false>(a, dtype, s);
}

int cxm_distill_bwd_t(const void *logits, size_t ld, const int32_t *ids, const float *teacher, size_t k, float scale,
                      const float *lse, const float *dloss, void *dlogits, size_t ldd, size_t rows, size_t vocab,
                      int dtype, cxm_stream_t s) {
    const int rc = cxm::check_logits(logits, ld, scale, rows, vocab, dtype);
    if (rc) return rc;
    if (ldd < vocab || k == 0 || k > cxm::kTeacherMost) return CXM_E_INVALID;
    if (rows == 0) return CXM_OK;
    if (ldd > (size_t(1) << 46) / rows) return CXM_E_TOO_LARGE;
    if (!ids || !teacher || !lse || !dloss || !dlogits) return CXM_E_INVALID;
    const size_t r4 = rows * 4, e = cxm::dtype_bytes(dtype), n = cxm::span_bytes(rows, ld, vocab, e);
    const cxm::Region out[1] = {{dlogits, cxm::span_bytes(rows, ldd, vocab, e)}};
    const bool in_place = dlogits == logits && ldd == ld;
    const cxm::Region in[5] = {{in_place ? nullptr : logits, n}, {ids, r4 * k}, {teacher, r4 * k}, {lse, r4}, {dloss, r4}};
    if (cxm::any_overlap(out, in)) return CXM_E_INVALID;
    cxm::GradArgs a{};
    a.in = cxm::logits_of(logits, ld, scale, rows, vocab, dtype);
    a.lse = lse;
    a.dx = dlogits;
    a.ldd = ldd;
    a.ids = ids;
    a.teacher = teacher;
    a.dloss = dloss;
    a.k = static_cast<unsigned>(k);
    return cxm::grad_any<true, false>(a, dtype, s);
}

}  // extern "C"
