// Layer norm of the rows of [rows, cols], with the residual's addition before
// it and an optional 8-bit output, and its backward.
//
//   h = x + res (rounded to the type; h = x without a residual)
//   mean = sum(h) / cols,  rstd = 1 / sqrt(sum((h - mean)^2) / cols + eps)
//   y = (h - mean) rstd w + bias;  8 bits: as in norm.hip
// Backward, with n = (h - mean) rstd and g = dy w:
//   dx = rstd (g - mean(g) - n mean(g n)) (+ dh)
//   dw[j] = sum over rows of dy n,  db[j] = sum over rows of dy
//
// Bound by memory: one read of each input and one write of each output.  The
// row stays in registers between the sum that gives its mean, the sum of its
// squared distances from it (which the one-pass sum of squares would lose to
// cancellation where the mean is large) and its output.  A row belongs to 16
// or 64 lanes of a wave or to a whole workgroup; sums are fp32.  fp16 20001x1003
// 14.3 us (5.6 TB/s).  Backward with dh bf16 8192x2048 27 us (5 TB/s) and 4 for the sums
// of dw and db; vector work is a third of its cycles, so neither bounds it: its
// workgroups are one wave per SIMD, in which a row's reduction and stores follow each
// other with only the next row's loads beside them.
#include "norm.hpp"

namespace cxm {
namespace {

struct LnFwd {
    const void *x, *res, *w, *bias;
    void *h, *y;
    uint8_t *q;
    float *scale, *mean, *rstd;
    size_t rows;
    unsigned cols;
    float eps;
};

struct LnBwd {
    const void *h, *w, *dy, *dh;
    const float *mean, *rstd;
    void *dx;
    float *part;  // [workgroups, 2 ld] sums of dw, and of db ld floats on
    size_t rows;
    unsigned cols, ld;
};

__device__ __forceinline__ float ln_rstd(float ss, unsigned cols, float eps) {
    return 1.0f / __builtin_sqrtf(ss / static_cast<float>(cols) + eps);
}

// G lanes per row, C chunks of VE elements per lane, NT threads.  AL: rows of
// whole 128-byte lines, read with the non-temporal hint; other rows are written
// with it (5000 rows of 1003 floats 10.5 -> 8.1 us, 20001 of 1003 fp16 20.7 -> 18.7;
// whole lines 4096x8192 44.6 -> 47.4).
template <int DT, int VE, int G, int C, int NT, bool AL>
__global__ __launch_bounds__(NT) void k_ln_fwd(LnFwd a) {
    using S = typename Elem<DT>::S;
    constexpr int R = G <= kWave ? NT / G : 1;
    __shared__ float lds[NT / kWave];
    const size_t mine = static_cast<size_t>(blockIdx.x) * R + (R > 1 ? threadIdx.x / G : 0);
    const bool live = mine < a.rows;  // lanes past the last row take it again and store nothing
    const size_t base = (live ? mine : a.rows - 1) * a.cols;
    const unsigned lane = threadIdx.x % G;
    const S *x = static_cast<const S *>(a.x) + base;
    const S *res = static_cast<const S *>(a.res) + (a.res ? base : 0);
    const S *w = static_cast<const S *>(a.w), *bias = static_cast<const S *>(a.bias);

    Span s[C];
    Chunk<DT, VE> cx[C], cr[C], cw[C], cb[C];
#pragma unroll
    for (int i = 0; i < C; ++i) s[i] = span_of<VE>(i * G + lane, a.cols);
#pragma unroll
    for (int i = 0; i < C; ++i) load_once<AL>(cx[i], x + s[i].off);
    if (a.res) {
#pragma unroll
        for (int i = 0; i < C; ++i) load_once<AL>(cr[i], res + s[i].off);
    }
#pragma unroll
    for (int i = 0; i < C; ++i) cw[i].load(w + s[i].off);
    if (a.bias) {
#pragma unroll
        for (int i = 0; i < C; ++i) cb[i].load(bias + s[i].off);
    }
    if (a.res) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
            float t[VE];
#pragma unroll
            for (int e = 0; e < VE; ++e) t[e] = cx[i].get(e) + cr[i].get(e);
            cx[i].set(t);
        }
        if (a.h && live) {
            S *h = static_cast<S *>(a.h) + base;
#pragma unroll
            for (int i = 0; i < C; ++i) store_span<DT, VE, !AL>(h, s[i], cx[i]);
        }
    }
    float v[C][VE];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < C; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            v[i][e] = cx[i].get(e);
            sum += e >= static_cast<int>(s[i].dup) ? v[i][e] : 0.0f;
        }
    const float mean = row_reduce<SumOp, G, NT>(sum, lds) / static_cast<float>(a.cols);
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < C; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            v[i][e] -= mean;
            const float d = e >= static_cast<int>(s[i].dup) ? v[i][e] : 0.0f;
            ss = fmaf(d, d, ss);
        }
    const float rstd = ln_rstd(row_reduce<SumOp, G, NT>(ss, lds), a.cols, a.eps);
    if (live && lane == 0) {
        if (a.mean) a.mean[mine] = mean;
        if (a.rstd) a.rstd[mine] = rstd;
    }
#pragma unroll
    for (int i = 0; i < C; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const float n = v[i][e] * rstd;
            v[i][e] = fmaf(n, cw[i].get(e), a.bias ? cb[i].get(e) : 0.0f);
        }
    if (a.y && live) {
        S *y = static_cast<S *>(a.y) + base;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            cx[i].set(v[i]);
            store_span<DT, VE, !AL>(y, s[i], cx[i]);
        }
    }
    if (a.q) {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
            for (int e = 0; e < VE; ++e) m = AmaxOp::combine(m, e >= static_cast<int>(s[i].dup) ? fabsf(v[i][e]) : 0.0f);
        m = row_reduce<AmaxOp, G, NT>(m, lds);
        const Scale8 k = scale_e4m3(m);
        if (live) {
            if (lane == 0) a.scale[mine] = k.scale;
#pragma unroll
            for (int i = 0; i < C; ++i) store_q<VE>(a.q + base, s[i], v[i], k.inv);
        }
    }
}

// A workgroup per row of any length: the row is read again for each of the sum
// of squares, the 8-bit scale and the output.
template <int DT, int NT>
__global__ __launch_bounds__(NT) void k_ln_fwd_long(LnFwd a) {
    using S = typename Elem<DT>::S;
    constexpr int VE = Elem<DT>::kVec;
    __shared__ float lds[NT / kWave];
    const size_t row = blockIdx.x, base = row * a.cols;
    const S *x = static_cast<const S *>(a.x) + base, *res = static_cast<const S *>(a.res) + (a.res ? base : 0);
    const S *w = static_cast<const S *>(a.w), *bias = static_cast<const S *>(a.bias);
    S *h = a.h ? static_cast<S *>(a.h) + base : nullptr;
    const unsigned whole = a.cols / VE, tail = whole * VE + threadIdx.x;
    auto chunk = [&](unsigned off) {  // h's chunk
        Chunk<DT, VE> c;
        c.load(x + off);
        if (a.res) {
            Chunk<DT, VE> r;
            r.load(res + off);
            float t[VE];
#pragma unroll
            for (int e = 0; e < VE; ++e) t[e] = c.get(e) + r.get(e);
            c.set(t);
        }
        return c;
    };
    auto single = [&](unsigned j) {  // h's element
        S hv = x[j];
        if (a.res) hv = Elem<DT>::store(Elem<DT>::load(hv) + Elem<DT>::load(res[j]));
        return hv;
    };
    float sum = 0.0f, ss = 0.0f;
    for (unsigned i = threadIdx.x; i < whole; i += NT) {
        const Chunk<DT, VE> c = chunk(i * VE);
        float t = 0.0f;
#pragma unroll
        for (int e = 0; e < VE; ++e) t += c.get(e);
        sum += t;
    }
    if (tail < a.cols) sum += Elem<DT>::load(single(tail));
    const float mean = block_reduce<SumOp, NT>(sum, lds) / static_cast<float>(a.cols);
    for (unsigned i = threadIdx.x; i < whole; i += NT) {
        const Chunk<DT, VE> c = chunk(i * VE);
        float t = 0.0f;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const float d = c.get(e) - mean;
            t = fmaf(d, d, t);
        }
        ss += t;
    }
    if (tail < a.cols) {
        const float d = Elem<DT>::load(single(tail)) - mean;
        ss = fmaf(d, d, ss);
    }
    const float rstd = ln_rstd(block_reduce<SumOp, NT>(ss, lds), a.cols, a.eps);
    if (threadIdx.x == 0) {
        if (a.mean) a.mean[row] = mean;
        if (a.rstd) a.rstd[row] = rstd;
    }
    auto one = [&](float hv, float wv, float bv) { return fmaf((hv - mean) * rstd, wv, bv); };
    auto out = [&](unsigned off, const Chunk<DT, VE> &c, float (&v)[VE]) {  // y's chunk
        Chunk<DT, VE> cw, cb;
        cw.load(w + off);
        if (a.bias) cb.load(bias + off);
#pragma unroll
        for (int e = 0; e < VE; ++e) v[e] = one(c.get(e), cw.get(e), a.bias ? cb.get(e) : 0.0f);
    };
    auto out1 = [&](unsigned j, S hv) {
        return one(Elem<DT>::load(hv), Elem<DT>::load(w[j]), a.bias ? Elem<DT>::load(bias[j]) : 0.0f);
    };
    Scale8 k{0.0f, 0.0f};
    if (a.q) {
        float m = 0.0f;
        for (unsigned i = threadIdx.x; i < whole; i += NT) {
            float v[VE];
            out(i * VE, chunk(i * VE), v);
#pragma unroll
            for (int e = 0; e < VE; ++e) m = AmaxOp::combine(m, fabsf(v[e]));
        }
        if (tail < a.cols) m = AmaxOp::combine(m, fabsf(out1(tail, single(tail))));
        m = block_reduce<AmaxOp, NT>(m, lds);
        k = scale_e4m3(m);
        if (threadIdx.x == 0) a.scale[row] = k.scale;
    }
    for (unsigned i = threadIdx.x; i < whole; i += NT) {
        const unsigned off = i * VE;
        const Chunk<DT, VE> c = chunk(off);
        float v[VE];
        out(off, c, v);
        if (h) c.store(h + off);
        if (a.y) {
            Chunk<DT, VE> cy;
            cy.set(v);
            cy.store(static_cast<S *>(a.y) + base + off);
        }
        if (a.q) store_q<VE>(a.q + base, Span{off, 0}, v, k.inv);
    }
    if (tail < a.cols) {
        const S hv = single(tail);
        const float v = out1(tail, hv);
        if (h) h[tail] = hv;
        if (a.y) static_cast<S *>(a.y)[base + tail] = Elem<DT>::store(v);
        if (a.q) a.q[base + tail] = static_cast<uint8_t>(pack_e4m3(v * k.inv, 0.0f, 0.0f, 0.0f));
    }
}

// Backward: workgroup b takes rows b R, b R + 1, ... of every gridDim.x R, loads
// a row while the one before it is reduced, and keeps its shares of dw and db in
// registers; the workgroups' shares meet in col_sum2 in a fixed order.
template <int DT, int VE, int G, int C, int NT, bool AL>
__global__ __launch_bounds__(NT) void k_ln_bwd(LnBwd a) {
    using S = typename Elem<DT>::S;
    constexpr int R = G <= kWave ? NT / G : 1;
    constexpr int W = G * C * VE;  // columns held
    __shared__ Pair lds[NT / kWave];
    __shared__ float sums[R > 1 ? R : 1][R > 1 ? W : 1];
    const unsigned lane = threadIdx.x % G, grp = R > 1 ? threadIdx.x / G : 0;
    Span s[C];
    Chunk<DT, VE> cw[C], ch[C], cd[C], ca[C];
    float aw[C][VE], ab[C][VE];
#pragma unroll
    for (int i = 0; i < C; ++i) {
        s[i] = span_of<VE>(i * G + lane, a.cols);
        cw[i].load(static_cast<const S *>(a.w) + s[i].off);
#pragma unroll
        for (int e = 0; e < VE; ++e) aw[i][e] = ab[i][e] = 0.0f;
    }
    const size_t step = static_cast<size_t>(gridDim.x) * R;
    size_t first = static_cast<size_t>(blockIdx.x) * R;
    float rstd = 0.0f, mean = 0.0f;
    auto load = [&](size_t r) {
        const size_t row = r < a.rows ? r : a.rows - 1, base = row * a.cols;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            load_once<AL>(ch[i], static_cast<const S *>(a.h) + base + s[i].off);
            load_once<AL>(cd[i], static_cast<const S *>(a.dy) + base + s[i].off);
        }
        if (a.dh) {
#pragma unroll
            for (int i = 0; i < C; ++i) load_once<AL>(ca[i], static_cast<const S *>(a.dh) + base + s[i].off);
        }
        rstd = a.rstd[row];
        mean = a.mean[row];
    };
    load(first + grp);
    for (; first < a.rows; first += step) {  // the same count for every thread of the workgroup
        const size_t row = first + grp;
        const bool live = row < a.rows;
        const float rs = rstd, mu = mean;
        float n[C][VE], g[C][VE];
        Chunk<DT, VE> past[C];
        Pair dot{0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < C; ++i) {
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float dy = live && e >= static_cast<int>(s[i].dup) ? cd[i].get(e) : 0.0f;
                n[i][e] = (ch[i].get(e) - mu) * rs;
                g[i][e] = dy * cw[i].get(e);
                aw[i][e] = live ? fmaf(dy, n[i][e], aw[i][e]) : aw[i][e];
                ab[i][e] += dy;
                dot.a += g[i][e];
                dot.b = fmaf(g[i][e], n[i][e], dot.b);
            }
            past[i] = ca[i];
        }
        if (first + step < a.rows) load(row + step);
        dot = row_reduce<PairSumOp, G, NT>(dot, lds);
        const float mg = dot.a / static_cast<float>(a.cols), mgn = dot.b / static_cast<float>(a.cols);
        if (live) {
            S *dx = static_cast<S *>(a.dx) + row * a.cols;
#pragma unroll
            for (int i = 0; i < C; ++i) {
                float t[VE];
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const float r = rs * (fmaf(-n[i][e], mgn, g[i][e]) - mg);
                    t[e] = a.dh ? r + past[i].get(e) : r;
                }
                Chunk<DT, VE> c;
                c.set(t);
                store_span<DT, VE, !AL>(dx, s[i], c);
            }
        }
    }
    float *part = a.part + static_cast<size_t>(blockIdx.x) * 2 * a.ld;
    auto share = [&](const float(&acc)[C][VE], float *to) {
        if constexpr (R > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < C; ++i)
#pragma unroll
                for (int e = 0; e < VE; ++e) sums[grp][(i * G + lane) * VE + e] = acc[i][e];
            __syncthreads();
            // a chunk moved back holds column off + e where its own place would be col + e
            for (unsigned j = threadIdx.x; j < a.cols; j += NT) {
                const unsigned c = j / VE;
                const Span t = span_of<VE>(c, a.cols);
                to[j] = combine_pairwise<SumOp, R>(&sums[0][c * VE + (j - t.off)], W);
            }
        } else {
#pragma unroll
            for (int i = 0; i < C; ++i)
#pragma unroll
                for (int e = 0; e < VE; ++e)
                    if (e >= static_cast<int>(s[i].dup)) to[s[i].off + e] = acc[i][e];
        }
    };
    share(aw, part);
    share(ab, part + a.ld);
}

// The same for rows of up to 2048 chunks, a workgroup of 1024 per row, whose
// registers are half as many: chunks stay packed until the output, the weights are
// read for each use (from L1 or L2), places are computed anew, and only in fp32 is
// the next row loaded ahead (16-bit then spills 17 registers: 2000x12288 94 us).
// fp32 2000x6001 53.5 us (k_ln_bwd_long 66.3), bf16 2000x12288 69.4 (76.0),
// 2000x12001 85.5 (92.1); but 100x16000, fewer rows than CUs, 32.8 (29.1).
template <int DT, int C, bool AL>
__global__ __launch_bounds__(1024) void k_ln_bwd_wide(LnBwd a) {
    using S = typename Elem<DT>::S;
    constexpr int VE = Elem<DT>::kVec, NT = 1024;
    constexpr bool AHEAD = DT == CXM_DT_F32;
    __shared__ Pair lds[NT / kWave];
    const S *w = static_cast<const S *>(a.w);
    float aw[C][VE], ab[C][VE];
#pragma unroll
    for (int i = 0; i < C; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) aw[i][e] = ab[i][e] = 0.0f;
    auto span = [&](int i) {
        unsigned c = i * NT + threadIdx.x;
        asm volatile("" : "+v"(c));
        return span_of<VE>(c, a.cols);
    };
    struct Row {
        Chunk<DT, VE> h[C], d[C], a[C];
        float rs, mu;
    };
    auto load = [&](Row &q, size_t row) {
        const size_t base = row * a.cols;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const unsigned off = span(i).off;
            load_once<AL>(q.h[i], static_cast<const S *>(a.h) + base + off);
            load_once<AL>(q.d[i], static_cast<const S *>(a.dy) + base + off);
            if (a.dh) load_once<AL>(q.a[i], static_cast<const S *>(a.dh) + base + off);
        }
        q.rs = a.rstd[row];
        q.mu = a.mean[row];
    };
    Row cur, next;
    size_t row = blockIdx.x;
    if constexpr (AHEAD) load(next, row);
    for (; row < a.rows; row += gridDim.x) {
        if constexpr (AHEAD) {
            cur = next;
            if (row + gridDim.x < a.rows) load(next, row + gridDim.x);
        } else {
            load(cur, row);
        }
        Pair dot{0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < C; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            const Span s = span(i);
            Chunk<DT, VE> cw;
            cw.load(w + s.off);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float n = (cur.h[i].get(e) - cur.mu) * cur.rs;
                const float dy = e >= static_cast<int>(s.dup) ? cur.d[i].get(e) : 0.0f, g = dy * cw.get(e);
                aw[i][e] = fmaf(dy, n, aw[i][e]);
                ab[i][e] += dy;
                dot.a += g;
                dot.b = fmaf(g, n, dot.b);
            }
        }
        dot = block_reduce<PairSumOp, NT>(dot, lds);
        const float mg = dot.a / static_cast<float>(a.cols), mgn = dot.b / static_cast<float>(a.cols);
        S *dx = static_cast<S *>(a.dx) + row * a.cols;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            // one chunk at a time, and what it unpacks to not kept from above: else 30 registers spill
            __builtin_amdgcn_sched_barrier(0);
            for (auto &r : cur.h[i].r) asm volatile("" : "+v"(r));
            for (auto &r : cur.d[i].r) asm volatile("" : "+v"(r));
            const Span s = span(i);
            Chunk<DT, VE> cw;
            cw.load(w + s.off);
            float t[VE];
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float n = (cur.h[i].get(e) - cur.mu) * cur.rs, g = cur.d[i].get(e) * cw.get(e);
                const float r = cur.rs * (fmaf(-n, mgn, g) - mg);
                t[e] = a.dh ? r + cur.a[i].get(e) : r;
            }
            cw.set(t);
            store_span<DT, VE, !AL>(dx, s, cw);
        }
    }
    float *part = a.part + static_cast<size_t>(blockIdx.x) * 2 * a.ld;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const Span s = span(i);
#pragma unroll
        for (int e = 0; e < VE; ++e)
            if (e >= static_cast<int>(s.dup)) {
                part[s.off + e] = aw[i][e];
                part[a.ld + s.off + e] = ab[i][e];
            }
    }
}

// Rows longer than these hold: dx by a workgroup per row, which reads the row
// twice; dw and db by k_ln_dw_part, run before it (dx may be dy or h).
template <int DT, int NT>
__global__ __launch_bounds__(NT) void k_ln_bwd_long(LnBwd a) {
    using S = typename Elem<DT>::S;
    constexpr int VE = Elem<DT>::kVec;
    __shared__ Pair lds[NT / kWave];
    const size_t row = blockIdx.x, base = row * a.cols;
    const S *h = static_cast<const S *>(a.h) + base, *dy = static_cast<const S *>(a.dy) + base;
    const S *dh = static_cast<const S *>(a.dh) + (a.dh ? base : 0), *w = static_cast<const S *>(a.w);
    S *dx = static_cast<S *>(a.dx) + base;
    const float rs = a.rstd[row], mu = a.mean[row];
    const unsigned whole = a.cols / VE, tail = whole * VE + threadIdx.x;
    Pair dot{0.0f, 0.0f};
    for (unsigned i = threadIdx.x; i < whole; i += NT) {
        Chunk<DT, VE> ch, cd, cw;
        ch.load(h + i * VE);
        cd.load(dy + i * VE);
        cw.load(w + i * VE);
        Pair t{0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const float n = (ch.get(e) - mu) * rs, g = cd.get(e) * cw.get(e);
            t.a += g;
            t.b = fmaf(g, n, t.b);
        }
        dot = PairSumOp::combine(dot, t);
    }
    if (tail < a.cols) {
        const float n = (Elem<DT>::load(h[tail]) - mu) * rs, g = Elem<DT>::load(dy[tail]) * Elem<DT>::load(w[tail]);
        dot = PairSumOp::combine(dot, Pair{g, g * n});
    }
    dot = block_reduce<PairSumOp, NT>(dot, lds);
    const float mg = dot.a / static_cast<float>(a.cols), mgn = dot.b / static_cast<float>(a.cols);
    auto one = [&](float hv, float dv, float wv) {
        const float n = (hv - mu) * rs, g = dv * wv;
        return rs * (fmaf(-n, mgn, g) - mg);
    };
    for (unsigned i = threadIdx.x; i < whole; i += NT) {
        Chunk<DT, VE> ch, cd, cw, ca;
        ch.load(h + i * VE);
        cd.load(dy + i * VE);
        cw.load(w + i * VE);
        if (a.dh) ca.load(dh + i * VE);
        float t[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const float r = one(ch.get(e), cd.get(e), cw.get(e));
            t[e] = a.dh ? r + ca.get(e) : r;
        }
        ch.set(t);
        ch.store(dx + i * VE);
    }
    if (tail < a.cols) {
        const float r = one(Elem<DT>::load(h[tail]), Elem<DT>::load(dy[tail]), Elem<DT>::load(w[tail]));
        dx[tail] = Elem<DT>::store(a.dh ? r + Elem<DT>::load(dh[tail]) : r);
    }
}

// dw and db over the rows r0, r0 + gridDim.y, ... of a tile of columns.
template <int DT>
__global__ __launch_bounds__(kBlock) void k_ln_dw_part(LnBwd a) {
    using S = typename Elem<DT>::S;
    constexpr int VE = Elem<DT>::kVec;
    const unsigned c = blockIdx.x * kBlock + threadIdx.x;
    if (c * VE >= a.cols) return;
    const Span s = span_of<VE>(c, a.cols);
    float aw[VE], ab[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) aw[e] = ab[e] = 0.0f;
    for (size_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
        Chunk<DT, VE> ch, cd;
        ch.load(static_cast<const S *>(a.h) + r * a.cols + s.off);
        cd.load(static_cast<const S *>(a.dy) + r * a.cols + s.off);
        const float rs = a.rstd[r], mu = a.mean[r];
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            aw[e] = fmaf(cd.get(e), (ch.get(e) - mu) * rs, aw[e]);
            ab[e] += cd.get(e);
        }
    }
    float *part = a.part + static_cast<size_t>(blockIdx.y) * 2 * a.ld;
#pragma unroll
    for (int e = 0; e < VE; ++e)
        if (e >= static_cast<int>(s.dup)) {
            part[s.off + e] = aw[e];
            part[a.ld + s.off + e] = ab[e];
        }
}

// ----------------------------------------------------------------- launch

template <int DT, int VE, int G, int C, int NT>
int fwd_launch(const LnFwd &a, hipStream_t s) {
    constexpr int R = G <= kWave ? NT / G : 1;
    constexpr size_t E = sizeof(typename Elem<DT>::S);
    const size_t wgs = (a.rows + R - 1) / R;
    if (wgs > most_wgs(NT)) return CXM_E_TOO_LARGE;
    const dim3 grid(static_cast<unsigned>(wgs));
    if (whole_lines(a.x, a.cols, E) && whole_lines(a.res, a.cols, E))
        hipLaunchKernelGGL((k_ln_fwd<DT, VE, G, C, NT, true>), grid, dim3(NT), 0, s, a);
    else
        hipLaunchKernelGGL((k_ln_fwd<DT, VE, G, C, NT, false>), grid, dim3(NT), 0, s, a);
    return launch_status();
}

template <int DT>
int fwd_dispatch(const LnFwd &a, hipStream_t s) {
    constexpr int VE = Elem<DT>::kVec;
    if (a.cols < static_cast<unsigned>(VE)) return fwd_launch<DT, 1, 16, 1, 256>(a, s);
    const unsigned chunks = (a.cols + VE - 1) / VE;
    const bool few = a.rows < 4 * device_cus();  // a wave per row would leave most of the chip idle
    if (chunks <= 16) return fwd_launch<DT, VE, 16, 1, 256>(a, s);
    if (chunks <= 64) return fwd_launch<DT, VE, 64, 1, 256>(a, s);
    if (chunks <= 128 && !few) return fwd_launch<DT, VE, 64, 2, 256>(a, s);
    if (chunks <= 256) return few ? fwd_launch<DT, VE, 256, 1, 256>(a, s) : fwd_launch<DT, VE, 64, 4, 256>(a, s);
    if (chunks <= 512) return few ? fwd_launch<DT, VE, 512, 1, 512>(a, s) : fwd_launch<DT, VE, 256, 2, 256>(a, s);
    if (chunks <= 1024) return few ? fwd_launch<DT, VE, 1024, 1, 1024>(a, s) : fwd_launch<DT, VE, 256, 4, 256>(a, s);
    if (chunks <= 2048) return fwd_launch<DT, VE, 1024, 2, 1024>(a, s);
    if (a.rows > most_wgs(1024)) return CXM_E_TOO_LARGE;
    hipLaunchKernelGGL((k_ln_fwd_long<DT, 1024>), dim3(static_cast<unsigned>(a.rows)), dim3(1024), 0, s, a);
    return launch_status();
}

int bwd_parts(LnBwd *a, size_t parts, cxm_stream_t st) {
    a->ld = (a->cols + 3) / 4 * 4;
    Workspace ws;
    const int rc = get_workspace(st, 0, parts * 2 * a->ld * sizeof(float), &ws);
    if (rc) return rc;
    a->part = static_cast<float *>(ws.scratch);
    return CXM_OK;
}

// The workgroups' shares into dw and (null: not wanted) db.
int bwd_sums(const LnBwd &a, size_t parts, void *dw, void *db, int dtype, cxm_stream_t st) {
    return col_sum2(a.part, parts, a.cols, 2 * static_cast<size_t>(a.ld), dw, a.ld, db, dtype, hs(st));
}

template <int DT, int VE, int G, int C, int NT>
int bwd_launch(LnBwd a, void *dw, void *db, cxm_stream_t st) {
    constexpr int R = G <= kWave ? NT / G : 1;
    constexpr size_t E = sizeof(typename Elem<DT>::S);
    // A workgroup's shares are 8 bytes a column, which it writes and col_sum2 reads: from 128 chunks a row on, one
    // workgroup per CU instead of two (bf16 8192x2048 31.7 us instead of 36.7, 4096x8192 57.7 instead of 73.3, fp32
    // 2048x4096 29.8 instead of 34.2; but bf16 30001x771 51.9 instead of 45.5).
    const size_t wgs = bwd_wgs(a.rows, R, G * C > 128 ? 1 : 2);
    const int rc = bwd_parts(&a, wgs, st);
    if (rc) return rc;
    const dim3 grid(static_cast<unsigned>(wgs));
    const bool lines = whole_lines(a.h, a.cols, E) && whole_lines(a.dy, a.cols, E) && whole_lines(a.dh, a.cols, E);
    if constexpr (G > 512) {
        if (lines) hipLaunchKernelGGL((k_ln_bwd_wide<DT, C, true>), grid, dim3(NT), 0, hs(st), a);
        else hipLaunchKernelGGL((k_ln_bwd_wide<DT, C, false>), grid, dim3(NT), 0, hs(st), a);
    } else {
        if (lines) hipLaunchKernelGGL((k_ln_bwd<DT, VE, G, C, NT, true>), grid, dim3(NT), 0, hs(st), a);
        else hipLaunchKernelGGL((k_ln_bwd<DT, VE, G, C, NT, false>), grid, dim3(NT), 0, hs(st), a);
    }
    const int r = launch_status();
    return r ? r : bwd_sums(a, wgs, dw, db, DT, st);
}

template <int DT>
int bwd_dispatch(LnBwd a, void *dw, void *db, cxm_stream_t st) {
    constexpr int VE = Elem<DT>::kVec;
    if (a.cols < static_cast<unsigned>(VE)) return bwd_launch<DT, 1, 16, 1, 256>(a, dw, db, st);
    const unsigned chunks = (a.cols + VE - 1) / VE;
    const bool few = a.rows <= static_cast<size_t>(device_cus());  // 64x2048: 7.5 us with a workgroup per row, 9.2 with a wave
    if (chunks <= 16) return bwd_launch<DT, VE, 16, 1, 256>(a, dw, db, st);
    if (chunks <= 64) return bwd_launch<DT, VE, 64, 1, 256>(a, dw, db, st);
    if (chunks <= 128) return bwd_launch<DT, VE, 64, 2, 256>(a, dw, db, st);
    if (chunks <= 256) return few ? bwd_launch<DT, VE, 256, 1, 256>(a, dw, db, st) : bwd_launch<DT, VE, 64, 4, 256>(a, dw, db, st);
    if (chunks <= 512) return bwd_launch<DT, VE, 256, 2, 256>(a, dw, db, st);
    if (chunks <= 1024) return bwd_launch<DT, VE, 512, 2, 512>(a, dw, db, st);
    if (chunks <= 2048 && !few) return bwd_launch<DT, VE, 1024, 2, 1024>(a, dw, db, st);
    if (a.rows > most_wgs(1024)) return CXM_E_TOO_LARGE;
    const size_t tiles = (chunks + kBlock - 1) / kBlock;
    size_t parts = 4 * device_cus() / tiles;
    parts = parts < 1 ? 1 : parts > a.rows ? a.rows : parts;
    const int rc = bwd_parts(&a, parts, st);
    if (rc) return rc;
    hipLaunchKernelGGL((k_ln_dw_part<DT>), dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(parts)), dim3(kBlock),
                       0, hs(st), a);
    int r = launch_status();
    if (r == CXM_OK) r = bwd_sums(a, parts, dw, db, DT, st);
    if (r) return r;
    hipLaunchKernelGGL((k_ln_bwd_long<DT, 1024>), dim3(static_cast<unsigned>(a.rows)), dim3(1024), 0, hs(st), a);
    return launch_status();
}

}  // namespace
}  // namespace cxm

extern "C" {

int cxm_layernorm_fwd_t(const void *x, const void *res, const void *w, const void *bias, float eps, void *h, void *y,
                        uint8_t *q, float *scale, float *mean, float *rstd, size_t rows, size_t cols, int dtype,
                        cxm_stream_t s) {
    using cxm::overlap;
    using cxm::overlap_not_same;
    if (!cxm::is_float_dtype(dtype) || !(eps >= 0.0f)) return CXM_E_INVALID;
    if (rows == 0) return CXM_OK;
    if (!x || !w || cols == 0 || (!y && !q) || (q && !scale) || (h && !res)) return CXM_E_INVALID;
    if (!cxm::row_shape_ok(rows, cols)) return CXM_E_TOO_LARGE;
    const size_t e = cxm::dtype_bytes(dtype), n = rows * cols * e;
    // h and y may each be x or res itself; no other output meets an input or another output
    const struct {
        const void *p;
        size_t n;
    } out[6] = {{h, n}, {y, n}, {q, q ? rows * cols : 0}, {scale, q ? rows * 4 : 0}, {mean, rows * 4}, {rstd, rows * 4}};
    for (int i = 0; i < 6; ++i) {
        const bool in_place = i < 2;
        if (in_place ? overlap_not_same(out[i].p, out[i].n, x, n) || overlap_not_same(out[i].p, out[i].n, res, n)
                     : overlap(out[i].p, out[i].n, x, n) || overlap(out[i].p, out[i].n, res, n))
            return CXM_E_INVALID;
        if (overlap(out[i].p, out[i].n, w, cols * e) || overlap(out[i].p, out[i].n, bias, cols * e)) return CXM_E_INVALID;
        for (int j = 0; j < i; ++j)
            if (overlap(out[i].p, out[i].n, out[j].p, out[j].n)) return CXM_E_INVALID;
    }
    const cxm::LnFwd a{x, res, w, bias, h, y, q, scale, mean, rstd, rows, static_cast<unsigned>(cols), eps};
    switch (dtype) {
        case CXM_DT_F32: return cxm::fwd_dispatch<CXM_DT_F32>(a, cxm::hs(s));
        case CXM_DT_BF16: return cxm::fwd_dispatch<CXM_DT_BF16>(a, cxm::hs(s));
        default: return cxm::fwd_dispatch<CXM_DT_F16>(a, cxm::hs(s));
    }
}

int cxm_layernorm_bwd_t(const void *h, const float *mean, const float *rstd, const void *w, const void *dy,
                        const void *dh, void *dx, void *dw, void *db, size_t rows, size_t cols, int dtype,
                        cxm_stream_t s) {
    using cxm::overlap;
    using cxm::overlap_not_same;
    if (!cxm::is_float_dtype(dtype) || !dw || cols == 0) return CXM_E_INVALID;
    if (!cxm::row_shape_ok(rows, cols) || cols >= (size_t(1) << 26)) return CXM_E_TOO_LARGE;  // (col_sum2's grid)
    const size_t e = cxm::dtype_bytes(dtype), n = rows * cols * e, c = cols * e;
    if (overlap(dw, c, db, c)) return CXM_E_INVALID;
    if (rows == 0) return cxm::col_sum2(nullptr, 0, cols, 0, dw, 0, db, dtype, cxm::hs(s));  // empty sums
    if (!h || !mean || !rstd || !w || !dy || !dx) return CXM_E_INVALID;
    // dx may be h, dy or dh itself
    for (const void *in : {h, dy, dh})
        if (overlap_not_same(dx, n, in, n) || overlap(dw, c, in, n) || overlap(db, c, in, n)) return CXM_E_INVALID;
    for (const float *in : {mean, rstd})
        if (overlap(dx, n, in, rows * 4) || overlap(dw, c, in, rows * 4) || overlap(db, c, in, rows * 4))
            return CXM_E_INVALID;
    for (const void *o : {dw, db})
        if (overlap(dx, n, o, c) || overlap(o, c, w, c)) return CXM_E_INVALID;
    if (overlap(dx, n, w, c)) return CXM_E_INVALID;
    const cxm::LnBwd a{h, w, dy, dh, mean, rstd, dx, nullptr, rows, static_cast<unsigned>(cols), 0};
    switch (dtype) {
        case CXM_DT_F32: return cxm::bwd_dispatch<CXM_DT_F32>(a, dw, db, s);
        case CXM_DT_BF16: return cxm::bwd_dispatch<CXM_DT_BF16>(a, dw, db, s);
        default: return cxm::bwd_dispatch<CXM_DT_F16>(a, dw, db, s);
    }
}

}  // extern "C"
