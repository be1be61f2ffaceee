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
constexpr int kStatChunks = 8, kGradChunks = 4;

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
};
// A segment's chunk that begins at column col: moved back to the segment's last
// VE elements where it reaches past its end (which may lie before the segment:
// never before the row).
template <int VE>
__device__ __forceinline__ Span seg_span(unsigned col, unsigned end) {
    const unsigned last = end - VE, off = col < last ? col : last;
    return {off, col - off};
}
// The first `dup` elements become -infinity.
template <int DT, int VE>
__device__ __forceinline__ void drop_dup(Chunk<DT, VE> &c, unsigned dup) {
    if (dup == 0) return;
    if constexpr (DT == CXM_DT_F32) {
#pragma unroll
        for (int e = 0; e < VE; ++e) c.r[e] = e < static_cast<int>(dup) ? -INFINITY : c.r[e];
    } else {
        constexpr unsigned inf = DT == CXM_DT_BF16 ? 0xff80u : 0xfc00u;
#pragma unroll
        for (int e = 0; e < VE; ++e)
            if (e < static_cast<int>(dup)) c.r[e / 2] = e & 1 ? (c.r[e / 2] & 0xffffu) | inf << 16 : (c.r[e / 2] & 0xffff0000u) | inf;
    }
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
    ArgPair *cands;   // [rows, nseg, top]
    unsigned *tickets;
};

__device__ __forceinline__ bool better(ArgPair a, ArgPair b) { return a.v > b.v || (a.v == b.v && a.i < b.i); }

// The value whose bits, made ascending in the value's order, are `key` (no
// number's key: NaN, which compares false).
__device__ __forceinline__ float value_of(unsigned key) {
    return __builtin_bit_cast(float, key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// LDS of a group.
struct Room {
    ArgPair *list, *best;  // kList and kTopMost entries
    int *count;
};
constexpr unsigned kList = 512;

// Sorts list[0 .. n) (n <= kList) and keeps the first min(n, top) in it, in order.
template <int G>
__device__ __forceinline__ unsigned keep_top(const Room &r, unsigned n, unsigned top, unsigned lane) {
    group_sync<G>();
    for (unsigned i = lane; i < n; i += G) {
        const ArgPair mine = r.list[i];
        unsigned rank = 0;
        for (unsigned j = 0; j < n; ++j) rank += better(r.list[j], mine);
        if (rank < top) r.best[rank] = mine;
    }
    group_sync<G>();
    const unsigned kept = n < top ? n : top;
    for (unsigned i = lane; i < kept; i += G) r.list[i] = r.best[i];
    group_sync<G>();
    return kept;
}

// Log probabilities of a row whose sums are known, with its `n` top tokens in
// r.list; or its divergence from the teacher.
template <int DT, int G, bool ENT, bool TOP>
__device__ __forceinline__ void finish_row(const StatArgs &a, size_t row, Part p, const Room &r, unsigned lane, float *lds) {
    using S = typename Elem<DT>::S;
    const S *x = static_cast<const S *>(a.in.x) + row * a.in.ld;
    const float log_s = logf(p.s);
    auto logp = [&](float v) { return (v - p.m) * a.in.scale - log_s; };
    if (lane == 0) {
        if (a.lse) a.lse[row] = fmaf(a.in.scale, p.m, log_s);
        if constexpr (ENT) {
            const float h = log_s - kLn2 * (p.t / p.s);
            a.entropy[row] = h < 0.0f ? 0.0f : h;
        }
        if (a.kind == 0 && a.logp) {
            const int tok = a.tokens[row];
            a.logp[row] = tok < 0                                       ? 0.0f
                          : static_cast<unsigned>(tok) < a.in.vocab ? logp(Elem<DT>::load(x[tok]))
                                                                        : __builtin_nanf("");
        }
    }
    if constexpr (TOP) {
        const bool bad = __builtin_isnan(p.m);
        for (unsigned i = lane; i < a.top; i += G) {
            const ArgPair v = r.list[i];
            a.top_ids[row * a.top + i] = bad ? -1 : v.i;
            a.top_logp[row * a.top + i] = bad ? __builtin_nanf("") : logp(v.v);
        }
    }
    if (a.kind == 1) {
        const int32_t *ids = a.ids + row * a.k;
        const float *tv = a.teacher + row * a.k;
        float tm = -INFINITY, bad = 0.0f;
        for (unsigned i = lane; i < a.k; i += G) {
            if (ids[i] < 0) continue;
            if (static_cast<unsigned>(ids[i]) >= a.in.vocab) bad = __builtin_nanf("");
            tm = fmax3(tm, tv[i]);
        }
        tm = group_all<InfMaxOp, G>(fmax3(tm, bad == 0.0f ? -INFINITY : bad), lds);
        float z = 0.0f, w = 0.0f;
        if (tm != -INFINITY && !__builtin_isnan(tm)) {
            for (unsigned i = lane; i < a.k; i += G) {
                if (ids[i] < 0) continue;
                const float l = (tv[i] - tm) * a.in.scale, e = expf(l);
                if (e == 0.0f) continue;
                z += e;
                w = fmaf(e, l - logp(Elem<DT>::load(x[ids[i]])), w);
            }
        }
        z = group_all<SumOp, G>(z, lds);
        w = group_all<SumOp, G>(w, lds);
        if (lane == 0) a.loss[row] = tm == -INFINITY ? 0.0f : __builtin_isnan(tm) ? tm : w / z - logf(z);
    }
}

// A row per G lanes (nseg 1, G = 64) or a segment per workgroup; C chunks a lane.
template <int DT, int VE, int G, int C, bool ENT, bool TOP>
__global__ __launch_bounds__(kBlock) void k_vocab_stats(StatArgs a) {
    using S = typename Elem<DT>::S;
    constexpr int NG = kBlock / G;
    __shared__ float lds_f[kBlock / kWave];
    __shared__ int lds_i[kBlock / kWave];
    __shared__ Part lds_p[kBlock / kWave];
    __shared__ ArgPair lists[TOP ? NG : 1][TOP ? (G == kBlock ? kList : kTopMost) : 1], bests[TOP ? NG : 1][TOP ? kTopMost : 1];
    __shared__ int counts[NG], flag;
    const unsigned lane = threadIdx.x % G, grp = threadIdx.x / G;
    const Room room{lists[TOP ? grp : 0], bests[TOP ? grp : 0], &counts[grp]};
    const size_t row = G == kBlock ? blockIdx.x / a.in.nseg : static_cast<size_t>(blockIdx.x) * NG + grp;
    if (row >= a.in.rows) return;  // a whole wave of a workgroup whose waves have rows of their own
    const unsigned seg = G == kBlock ? blockIdx.x % a.in.nseg : 0;
    const unsigned s0 = seg * a.in.seglen, s1 = a.in.vocab - s0 < a.in.seglen ? a.in.vocab : s0 + a.in.seglen;
    const S *x = static_cast<const S *>(a.in.x) + row * a.in.ld;
    // chunks that some lane of this wave has
    const unsigned first = s0 + (__builtin_amdgcn_readfirstlane(lane / kWave) * kWave) * VE;
    const int its = first >= s1 ? 0 : static_cast<int>((s1 - first + G * VE - 1) / (G * VE));
    Chunk<DT, VE> c[C];
    Span sp[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
        sp[i] = seg_span<VE>(s0 + (i * G + lane) * VE, s1);
        if (i < its) c[i].load_nt(x + sp[i].off);
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        if (i >= its) break;
        drop_dup<DT, VE>(c[i], sp[i].dup);
#pragma unroll
        for (int e = 0; e < VE; ++e) m = fmax3(m, c[i].get(e));
    }
    m = wave_reduce<InfMaxOp>(m);
    const float base = m == -INFINITY ? 0.0f : m;
    float sum[2] = {0.0f, 0.0f}, ent[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < C; ++i) {
        if (i >= its) break;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            float u = (c[i].get(e) - base) * a.in.c;
            if constexpr (ENT) u = fmax3(u, kLow);
            const float p = __builtin_amdgcn_exp2f(u);
            sum[e & 1] += p;
            if constexpr (ENT) ent[e & 1] = fmaf(u, p, ent[e & 1]);
        }
    }
    Part p{m, wave_reduce<SumOp>(sum[0] + sum[1]), ENT ? wave_reduce<SumOp>(ent[0] + ent[1]) : 0.0f};
    if constexpr (G == kBlock) {
        constexpr int NW = kBlock / kWave;
        if (lane % kWave == 0) lds_p[lane / kWave] = p;
        __syncthreads();
        float top = lds_p[0].m;
#pragma unroll
        for (int w = 1; w < NW; ++w) top = fmax3(top, lds_p[w].m);
        Part q{top, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const Part v = rebase(lds_p[w], top, a.in.c);
            q.s += v.s;
            q.t += v.t;
        }
        p = q;
    }
    unsigned n = 0;  // tokens selected
    if constexpr (TOP) {
        // The segment's top tokens exactly: the value of the last of them bit by bit, then, of those equal to
        // it, the last place that is taken.
        n = s1 - s0 < a.top ? s1 - s0 : a.top;
        if (!__builtin_isnan(p.m)) {
            auto count = [&](auto &&f) {
                int k = 0;
#pragma unroll
                for (int i = 0; i < C; ++i) {
                    if (i >= its) break;
#pragma unroll
                    for (int e = 0; e < VE; ++e) k += f(c[i].get(e), sp[i].off + e, e >= static_cast<int>(sp[i].dup));
                }
                return static_cast<unsigned>(group_all<IntSumOp, G>(k, lds_i));
            };
            unsigned key = 0;
            constexpr int low = DT == CXM_DT_F32 ? 0 : DT == CXM_DT_BF16 ? 16 : 13;  // bits below are all alike
            for (int b = 31; b >= low; --b) {
                const float t = value_of(key | 1u << b);
                if (count([&](float v, unsigned, bool own) { return own && v >= t; }) >= n) key |= 1u << b;
            }
            if (!(key & 0x80000000u)) key |= (1u << low) - 1;  // a negative value's bits are counted from its other end
            const float t = key < 0x007fffffu ? -INFINITY : value_of(key);
            const unsigned above = count([&](float v, unsigned, bool own) { return own && v > t; }), ties = n - above;
            unsigned place = 0;  // the ties below s0 + place are fewer than `ties`
            for (unsigned b = 1u << 14; b; b >>= 1) {
                const unsigned to = s0 + (place | b);
                if (count([&](float v, unsigned j, bool own) { return own && v == t && j < to; }) < ties) place |= b;
            }
            if (lane == 0) *room.count = 0;
            group_sync<G>();
#pragma unroll
            for (int i = 0; i < C; ++i) {
                if (i >= its) break;
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const float v = c[i].get(e);
                    const unsigned j = sp[i].off + e;
                    if (e >= static_cast<int>(sp[i].dup) && (v > t || (v == t && j <= s0 + place)))
                        room.list[atomicAdd(room.count, 1)] = ArgPair{v, static_cast<int>(j)};
                }
            }
            group_sync<G>();
        }
    }
    if constexpr (G == kBlock) {
        if (a.in.nseg > 1) {
            const size_t at = row * a.in.nseg + seg;
            if (lane == 0) {
                float *to = &a.parts[at].m;
                st_dev(to, p.m);
                st_dev(to + 1, p.s);
                st_dev(to + 2, p.t);
            }
            if constexpr (TOP) {
                // (a NaN segment's are not looked at)
                for (unsigned i = lane; i < a.top; i += G)
                    st_dev(a.cands + at * a.top + i, i < n && !__builtin_isnan(p.m) ? room.list[i] : ArgPair{-INFINITY, 0x7fffffff});
            }
            if (!last_block_ticket(a.tickets + row * kTicket, a.in.nseg, &flag)) return;
            const float *from = &a.parts[row * a.in.nseg].m;
            float top = -INFINITY;
            for (unsigned i = lane; i < a.in.nseg; i += G) top = fmax3(top, ld_dev(from + 3 * i));
            top = block_reduce<InfMaxOp, kBlock>(top, lds_f);
            Part q{top, 0.0f, 0.0f};
            for (unsigned i = lane; i < a.in.nseg; i += G) {
                const Part v = rebase(Part{ld_dev(from + 3 * i), ld_dev(from + 3 * i + 1), ld_dev(from + 3 * i + 2)}, top, a.in.c);
                q.s += v.s;
                q.t += v.t;
            }
            q.s = block_reduce<SumOp, kBlock>(q.s, lds_f);
            q.t = block_reduce<SumOp, kBlock>(q.t, lds_f);
            p = q;
            if constexpr (TOP) {
                const size_t total = static_cast<size_t>(a.in.nseg) * a.top;
                const ArgPair *cands = a.cands + row * total;
                unsigned have = 0;
                for (size_t b = 0; b < total;) {
                    const unsigned take = total - b < kList - have ? static_cast<unsigned>(total - b) : kList - have;
                    for (unsigned i = lane; i < take; i += G) room.list[have + i] = ld_dev(cands + b + i);
                    b += take;
                    have = keep_top<G>(room, have + take, a.top, lane);
                }
                n = have;
            }
        } else if constexpr (TOP) {
            keep_top<G>(room, n, a.top, lane);
        }
    } else if constexpr (TOP) {
        keep_top<G>(room, n, a.top, lane);
    }
    finish_row<DT, G, ENT, TOP>(a, row, p, room, lane, lds_f);
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

template <int DT, int VE, int G, int C, bool DISTILL, bool ENT>
__global__ __launch_bounds__(kBlock) void k_vocab_grad(GradArgs a) {
    using S = typename Elem<DT>::S;
    constexpr int NG = kBlock / G, KE = kTeacherMost / G;
    __shared__ float lds_f[kBlock / kWave];
    __shared__ float qs[DISTILL ? NG : 1][DISTILL ? kTeacherMost : 1];
    __shared__ int qi[DISTILL ? NG : 1][DISTILL ? kTeacherMost : 1];
    const unsigned lane = threadIdx.x % G, grp = threadIdx.x / G;
    const size_t row = G == kBlock ? blockIdx.x / a.in.nseg : static_cast<size_t>(blockIdx.x) * NG + grp;
    if (row >= a.in.rows) return;  // a whole wave of a workgroup whose waves have rows of their own
    const unsigned seg = G == kBlock ? blockIdx.x % a.in.nseg : 0;
    const unsigned s0 = seg * a.in.seglen, s1 = a.in.vocab - s0 < a.in.seglen ? a.in.vocab : s0 + a.in.seglen;
    const S *x = static_cast<const S *>(a.in.x) + row * a.in.ld;
    S *dx = static_cast<S *>(a.dx) + row * a.ldd;
    const unsigned first = s0 + (__builtin_amdgcn_readfirstlane(lane / kWave) * kWave) * VE;
    const int its = first >= s1 ? 0 : static_cast<int>((s1 - first + G * VE - 1) / (G * VE));
    Chunk<DT, VE> c[C];
    Span sp[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
        sp[i] = seg_span<VE>(s0 + (i * G + lane) * VE, s1);
        if (i < its) c[i].load_nt(x + sp[i].off);
    }
    const float lse = a.lse[row];
    // d x = p (slope + bend (log p)) + what the tokens get
    float slope, bend = 0.0f, given = 0.0f;
    unsigned token = ~0u;
    float late_v[KE];  // distillation: the gradient at the teacher's tokens of this segment
    bool late[KE];
    if constexpr (DISTILL) {
        const int32_t *ids = a.ids + row * a.k;
        const float *tv = a.teacher + row * a.k;
        int id[KE];
        float t[KE], tm = -INFINITY;
#pragma unroll
        for (int j = 0; j < KE; ++j) {
            const unsigned i = j * G + lane;
            id[j] = i < a.k ? ids[i] : -1;
            t[j] = i < a.k && id[j] >= 0 ? tv[i] : -INFINITY;
            if (id[j] >= 0 && static_cast<unsigned>(id[j]) >= a.in.vocab) t[j] = __builtin_nanf("");
            tm = fmax3(tm, t[j]);
        }
        tm = group_all<InfMaxOp, G>(tm, lds_f);
        float z = 0.0f, q[KE];
        const float from = tm == -INFINITY ? 0.0f : tm;
#pragma unroll
        for (int j = 0; j < KE; ++j) {
            q[j] = expf((t[j] - from) * a.in.scale);
            z += q[j];
        }
        z = group_all<SumOp, G>(z, lds_f);
        slope = tm == -INFINITY ? 0.0f : a.dloss[row] * a.in.scale;
#pragma unroll
        for (int j = 0; j < KE; ++j) {
            q[j] /= z;
            qs[grp][j * G + lane] = q[j];
            qi[grp][j * G + lane] = id[j];
        }
        group_sync<G>();
#pragma unroll
        for (int j = 0; j < KE; ++j) {
            late[j] = id[j] >= static_cast<int>(s0) && id[j] < static_cast<int>(s1);
            late_v[j] = 0.0f;
            if (late[j]) {
                float all = 0.0f;  // a token may be there more than once
                for (unsigned i = 0; i < a.k; ++i) all += qi[grp][i] == id[j] ? qs[grp][i] : 0.0f;
                const float p = __builtin_amdgcn_exp2f(fmaf(a.in.scale, Elem<DT>::load(x[id[j]]), -lse) * kLog2e);
                late_v[j] = slope == 0.0f ? 0.0f : slope * (p - all);
            }
        }
        if (__builtin_isnan(tm)) slope = tm;
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
    if constexpr (DISTILL) {  // every teacher's token has been read (dx may be x)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        group_sync<G>();
    }
#pragma unroll
    for (int i = 0; i < C; ++i) {
        if (i >= its) break;
        float v[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            float l = fmaf(a.in.scale, c[i].get(e), -lse);
            if constexpr (ENT) l = fmax3(l, kLow);
            const float p = __builtin_amdgcn_exp2f(l * kLog2e);
            if constexpr (ENT) v[e] = p * fmaf(bend, l, slope);
            else v[e] = p * slope;
            if constexpr (!DISTILL) v[e] += sp[i].off + e == token ? given : 0.0f;
            v[e] = none ? 0.0f : v[e];
        }
        c[i].set(v);
        store_span<DT, VE>(dx, sp[i], c[i]);
    }
    if constexpr (DISTILL) {
        // over what was stored above, by whichever lane
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        group_sync<G>();
#pragma unroll
        for (int j = 0; j < KE; ++j)
            if (late[j]) dx[qi[grp][j * G + lane]] = Elem<DT>::store(__builtin_isnan(slope) ? slope : late_v[j]);
    }
}

// ----------------------------------------------------------------- launch

// Cuts rows into segments of at most `most` elements, and of fewer (but a chunk
// for every lane) where there would be fewer workgroups than fill the chip.
void cut(Logits *in, unsigned most, unsigned least) {
    size_t nseg = (in->vocab + most - 1) / most;
    const size_t want = (4 * device_cus() + in->rows - 1) / in->rows, can = (in->vocab + least - 1) / least;
    if (nseg < want) nseg = want < can ? want : can;
    const size_t len = (in->vocab + nseg - 1) / nseg;
    in->seglen = static_cast<unsigned>((len + 63) / 64 * 64);
    in->nseg = (in->vocab + in->seglen - 1) / in->seglen;
}

// Whether a wave holds a row of C chunks a lane, and there are rows enough to give each wave one.
bool wave_rows(const Logits &in, unsigned chunk, unsigned chunks) {
    return in.vocab <= 64 * chunk * chunks && (in.vocab <= 64 * chunk || in.rows >= 4 * device_cus());
}

template <int DT, int VE, int G, bool ENT, bool TOP>
int stats_launch(const StatArgs &a, hipStream_t s) {
    constexpr int C = VE == 1 ? 1 : kStatChunks;
    const size_t wgs = G == kBlock ? a.in.rows * a.in.nseg : (a.in.rows + kBlock / G - 1) / (kBlock / G);
    hipLaunchKernelGGL((k_vocab_stats<DT, VE, G, C, ENT, TOP>), dim3(static_cast<unsigned>(wgs)), dim3(kBlock), 0, s, a);
    return launch_status();
}

template <int DT, bool ENT, bool TOP>
int stats(StatArgs a, cxm_stream_t st) {
    constexpr int VE = Elem<DT>::kVec;
    a.in.nseg = 1;
    a.in.seglen = (a.in.vocab + 63) / 64 * 64;
    const bool wave = a.in.vocab < static_cast<unsigned>(VE) || wave_rows(a.in, VE, kStatChunks);
    if (!wave) cut(&a.in, kBlock * VE * kStatChunks, kBlock * VE);
    if (a.in.nseg > most_wgs(kBlock) / a.in.rows) return CXM_E_TOO_LARGE;
    if (wave) {
        return a.in.vocab < static_cast<unsigned>(VE) ? stats_launch<DT, 1, 64, ENT, TOP>(a, hs(st))
                                                      : stats_launch<DT, VE, 64, ENT, TOP>(a, hs(st));
    }
    if (a.in.nseg > 1) {
        const size_t segs = a.in.rows * a.in.nseg, o_cands = (segs * sizeof(Part) + 255) / 256 * 256;
        Workspace ws;
        const int rc = get_workspace(st, (a.in.rows * kTicket + kCtr - 1) / kCtr,
                                     o_cands + (TOP ? segs * a.top * sizeof(ArgPair) : 0), &ws);
        if (rc) return rc;
        a.tickets = ws.counters;
        a.parts = static_cast<Part *>(ws.scratch);
        a.cands = reinterpret_cast<ArgPair *>(static_cast<char *>(ws.scratch) + o_cands);
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
    a.in.seglen = (a.in.vocab + 63) / 64 * 64;
    const bool wave = a.in.vocab < static_cast<unsigned>(VE) || wave_rows(a.in, VE, kGradChunks);
    if (!wave) cut(&a.in, kBlock * VE * kGradChunks, kBlock * VE);
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

Logits logits_of(const void *x, size_t ld, float scale, size_t rows, size_t vocab) {
    return Logits{x, ld, rows, static_cast<unsigned>(vocab), 1, 0, scale, scale * kLog2e};
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
    a.in = cxm::logits_of(logits, ld, scale, rows, vocab);
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
    a.in = cxm::logits_of(logits, ld, scale, rows, vocab);
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
    a.in = cxm::logits_of(logits, ld, scale, rows, vocab);
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
    a.in = cxm::logits_of(logits, ld, scale, rows, vocab);
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
