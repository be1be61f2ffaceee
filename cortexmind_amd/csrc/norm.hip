// Root-mean-square norm of the rows of [rows, cols], with the residual's
// addition before it and an optional 8-bit output, its backward, and the
// 8-bit form of rows on its own.
//
//   h = x + res (rounded to the type; h = x without a residual)
//   rstd = 1 / sqrt(mean(h^2) + eps),  y = h rstd w
//   8 bits: scale = max |y| / 448, q = e4m3(y / scale)
// Backward, with n = h rstd and g = dy w:
//   dx = rstd (g - n mean(g n)) (+ dh),  dw[j] = sum over rows of dy n
//
// Bound by memory: one read of each input and one write of each output, the
// row staying in registers between its sum of squares and its output.  A row
// belongs to 16 or 64 lanes of a wave or to a whole workgroup, so that a
// lane holds one to four chunks of 16 bytes; rows beyond that are read twice
// (the second time mostly from L2).  All sums are fp32.
#include "norm.hpp"

namespace cxm {
namespace {

struct RmsFwd {
    const void *x, *res, *w;
    void *h, *y;
    uint8_t *q;
    float *scale, *rstd;
    size_t rows;
    unsigned cols;
    float eps;
    int norm;  // 0: y = x, for the 8-bit form of rows alone
};

struct RmsBwd {
    const void *h, *w, *dy, *dh;
    const float *rstd;
    void *dx;
    float *part;  // [workgroups, ld] sums of dw
    size_t rows;
    unsigned cols, ld;
};

__device__ __forceinline__ float rms_rstd(float ss, unsigned cols, float eps) {
    return 1.0f / __builtin_sqrtf(ss / static_cast<float>(cols) + eps);
}

// G lanes per row, C chunks of VE elements per lane, NT threads.  AL: rows of
// whole 128-byte lines, read with the non-temporal hint (4096x4096 bf16 to 8
// bits 23.3 -> 21.2 us; rows of 1003 floats, whose waves share lines, 7.4 ->
// 8.6, so those do without).  Outputs are what the next call reads: no hint.
template <int DT, int VE, int G, int C, int NT, bool AL>
__global__ __launch_bounds__(NT) void k_rms_fwd(RmsFwd a) {
    using S = typename Elem<DT>::S;
    constexpr int R = G <= kWave ? NT / G : 1;
    __shared__ float lds[NT / kWave];
    const size_t mine = static_cast<size_t>(blockIdx.x) * R + (R > 1 ? threadIdx.x / G : 0);
    const bool live = mine < a.rows;  // lanes past the last row take it again and store nothing
    const size_t base = (live ? mine : a.rows - 1) * a.cols;
    const unsigned lane = threadIdx.x % G;
    const S *x = static_cast<const S *>(a.x) + base;
    const S *res = static_cast<const S *>(a.res) + (a.res ? base : 0);
    const S *w = static_cast<const S *>(a.w);

    Span s[C];
    Chunk<DT, VE> cx[C], cr[C], cw[C];
#pragma unroll
    for (int i = 0; i < C; ++i) s[i] = span_of<VE>(i * G + lane, a.cols);
#pragma unroll
    for (int i = 0; i < C; ++i) load_once<AL>(cx[i], x + s[i].off);
    if (a.res) {
#pragma unroll
        for (int i = 0; i < C; ++i) load_once<AL>(cr[i], res + s[i].off);
    }
    if (a.norm) {
#pragma unroll
        for (int i = 0; i < C; ++i) cw[i].load(w + s[i].off);
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
            for (int i = 0; i < C; ++i) store_span<DT, VE>(h, s[i], cx[i]);
        }
    }
    float v[C][VE];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < C; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            v[i][e] = e >= static_cast<int>(s[i].dup) ? cx[i].get(e) : 0.0f;
            ss = fmaf(v[i][e], v[i][e], ss);
        }
    if (a.norm) {
        ss = row_reduce<SumOp, G, NT>(ss, lds);
        const float rstd = rms_rstd(ss, a.cols, a.eps);
        if (a.rstd && live && lane == 0) a.rstd[mine] = rstd;
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float t = v[i][e] * rstd;
                v[i][e] = t * cw[i].get(e);
            }
    }
    if (a.y && live) {
        S *y = static_cast<S *>(a.y) + base;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            cx[i].set(v[i]);
            store_span<DT, VE>(y, s[i], cx[i]);
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

// A workgroup per row of any length: the row is read again for its output
// (and once more for the 8-bit one, whose scale needs every y).
template <int DT, int NT>
__global__ __launch_bounds__(NT) void k_rms_fwd_long(RmsFwd a) {
    using S = typename Elem<DT>::S;
    constexpr int VE = Elem<DT>::kVec;
    __shared__ float lds[NT / kWave];
    const size_t row = blockIdx.x, base = row * a.cols;
    const S *x = static_cast<const S *>(a.x) + base, *res = static_cast<const S *>(a.res) + (a.res ? base : 0);
    const S *w = static_cast<const S *>(a.w);
    S *h = a.h ? static_cast<S *>(a.h) + base : nullptr;
    const unsigned chunks = (a.cols + VE - 1) / VE;
    auto sum = [&](Span s) {  // h's chunk
        Chunk<DT, VE> c;
        c.load(x + s.off);
        if (a.res) {
            Chunk<DT, VE> r;
            r.load(res + s.off);
            float t[VE];
#pragma unroll
            for (int e = 0; e < VE; ++e) t[e] = c.get(e) + r.get(e);
            c.set(t);
        }
        return c;
    };
    float rstd = 1.0f;
    if (a.norm) {
        float ss = 0.0f;
        for (unsigned i = threadIdx.x; i < chunks; i += NT) {
            const Span s = span_of<VE>(i, a.cols);
            const Chunk<DT, VE> c = sum(s);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float v = e >= static_cast<int>(s.dup) ? c.get(e) : 0.0f;
                ss = fmaf(v, v, ss);
            }
        }
        ss = block_reduce<SumOp, NT>(ss, lds);
        rstd = rms_rstd(ss, a.cols, a.eps);
        if (a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
    }
    auto out = [&](Span s, const Chunk<DT, VE> &c, float (&v)[VE]) {  // y's chunk
        Chunk<DT, VE> cw;
        if (a.norm) cw.load(w + s.off);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const float t = c.get(e) * rstd;
            v[e] = a.norm ? t * cw.get(e) : c.get(e);
        }
    };
    Scale8 k{0.0f, 0.0f};
    if (a.q) {
        float m = 0.0f;
        for (unsigned i = threadIdx.x; i < chunks; i += NT) {
            const Span s = span_of<VE>(i, a.cols);
            float v[VE];
            out(s, sum(s), v);
#pragma unroll
            for (int e = 0; e < VE; ++e) m = AmaxOp::combine(m, e >= static_cast<int>(s.dup) ? fabsf(v[e]) : 0.0f);
        }
        m = block_reduce<AmaxOp, NT>(m, lds);
        k = scale_e4m3(m);
        if (threadIdx.x == 0) a.scale[row] = k.scale;
    }
    // The last chunk shares elements with the one before it, which may be
    // stored over them (h on x, y on x or res): the tail's elements are read
    // one by one.
    const unsigned whole = a.cols / VE;
    for (unsigned i = threadIdx.x; i < whole; i += NT) {
        const Span s{i * VE, 0};
        const Chunk<DT, VE> c = sum(s);
        float v[VE];
        out(s, c, v);
        if (h) c.store(h + s.off);
        if (a.y) {
            Chunk<DT, VE> cy;
            cy.set(v);
            cy.store(static_cast<S *>(a.y) + base + s.off);
        }
        if (a.q) store_q<VE>(a.q + base, s, v, k.inv);
    }
    const unsigned j = whole * VE + threadIdx.x;
    if (j < a.cols) {
        S hv = x[j];
        if (a.res) hv = Elem<DT>::store(Elem<DT>::load(hv) + Elem<DT>::load(res[j]));
        const float hf = Elem<DT>::load(hv), n = hf * rstd;
        const float v = a.norm ? n * Elem<DT>::load(w[j]) : hf;
        if (h) h[j] = hv;
        if (a.y) static_cast<S *>(a.y)[base + j] = Elem<DT>::store(v);
        if (a.q) a.q[base + j] = static_cast<uint8_t>(pack_e4m3(v * k.inv, 0.0f, 0.0f, 0.0f));
    }
}

// Backward: workgroup b takes rows b R, b R + 1, ... of every gridDim.x R,
// loads a row while the one before it is reduced, and keeps its share of dw
// in registers; the workgroups' shares meet in col_sum in a fixed order.
template <int DT, int VE, int G, int C, int NT, bool AL>
__global__ __launch_bounds__(NT) void k_rms_bwd(RmsBwd a) {
    using S = typename Elem<DT>::S;
    constexpr int R = G <= kWave ? NT / G : 1;
    constexpr int W = G * C * VE;  // columns held
    __shared__ float lds[NT / kWave];
    __shared__ float dws[R > 1 ? R : 1][R > 1 ? W : 1];
    const unsigned lane = threadIdx.x % G, grp = R > 1 ? threadIdx.x / G : 0;
    Span s[C];
    Chunk<DT, VE> cw[C], ch[C], cd[C], ca[C];
    float acc[C][VE];
#pragma unroll
    for (int i = 0; i < C; ++i) {
        s[i] = span_of<VE>(i * G + lane, a.cols);
        cw[i].load(static_cast<const S *>(a.w) + s[i].off);
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[i][e] = 0.0f;
    }
    const size_t step = static_cast<size_t>(gridDim.x) * R;
    size_t first = static_cast<size_t>(blockIdx.x) * R;
    float rstd = 0.0f;
    auto load = [&](size_t r) {
        const size_t base = (r < a.rows ? r : a.rows - 1) * a.cols;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            load_once<AL>(ch[i], static_cast<const S *>(a.h) + base + s[i].off);
            load_once<AL>(cd[i], static_cast<const S *>(a.dy) + base + s[i].off);
        }
        if (a.dh) {
#pragma unroll
            for (int i = 0; i < C; ++i) load_once<AL>(ca[i], static_cast<const S *>(a.dh) + base + s[i].off);
        }
        rstd = a.rstd[r < a.rows ? r : a.rows - 1];
    };
    load(first + grp);
    for (; first < a.rows; first += step) {  // the same count for every thread of the workgroup
        const size_t row = first + grp;
        const bool live = row < a.rows;
        const float rs = rstd;
        float n[C][VE], g[C][VE], d[C][VE];
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const bool keep = live && e >= static_cast<int>(s[i].dup);
                n[i][e] = ch[i].get(e) * rs;
                const float dy = cd[i].get(e);
                g[i][e] = dy * cw[i].get(e);
                const float t = dy * n[i][e];
                acc[i][e] += keep ? t : 0.0f;
                dot += keep ? g[i][e] * n[i][e] : 0.0f;
                d[i][e] = a.dh ? ca[i].get(e) : 0.0f;
            }
        if (first + step < a.rows) load(row + step);
        dot = row_reduce<SumOp, G, NT>(dot, lds);
        const float mean = dot / static_cast<float>(a.cols);
        if (live) {
            S *dx = static_cast<S *>(a.dx) + row * a.cols;
#pragma unroll
            for (int i = 0; i < C; ++i) {
                float t[VE];
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const float u = n[i][e] * mean;
                    const float r = rs * (g[i][e] - u);
                    t[e] = a.dh ? r + d[i][e] : r;
                }
                Chunk<DT, VE> c;
                c.set(t);
                store_span<DT, VE>(dx, s[i], c);
            }
        }
    }
    float *part = a.part + static_cast<size_t>(blockIdx.x) * a.ld;
    if constexpr (R > 1) {
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
            for (int e = 0; e < VE; ++e) dws[grp][(i * G + lane) * VE + e] = acc[i][e];
        __syncthreads();
        // a chunk moved back holds column off + e where its own place would be col + e
        for (unsigned j = threadIdx.x; j < a.cols; j += NT) {
            const unsigned c = j / VE;
            const Span t = span_of<VE>(c, a.cols);
            part[j] = combine_pairwise<SumOp, R>(&dws[0][c * VE + (j - t.off)], W);
        }
    } else {
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if (e >= static_cast<int>(s[i].dup)) part[s[i].off + e] = acc[i][e];
    }
}

// The same for rows of 2048 chunks (C = 2; fp32 4096, C = 4), a workgroup of 1024
// per row, whose registers are half as many: the chunks stay packed until the
// output, the weights are read for each use (from L1 or L2), and with C = 4 the
// next row is not loaded ahead.  fp16 4096x8448 61.5 us and bf16 2048x12288 with
// dh 54.8 (held as k_rms_bwd does, spilling 31 registers, 141.6 and 104.3), fp32
// 1024x16000 66.6 (k_rms_bwd_long 87.3); 16-bit C = 4 spills 40 registers
// (448x30656 78.5 us; k_rms_bwd_long 45.6).
template <int DT, int C, bool AL>
__global__ __launch_bounds__(1024) void k_rms_bwd_wide(RmsBwd a) {
    using S = typename Elem<DT>::S;
    constexpr int VE = Elem<DT>::kVec, NT = 1024;
    constexpr bool AHEAD = C <= 2;
    __shared__ float lds[NT / kWave];
    const S *w = static_cast<const S *>(a.w);
    float acc[C][VE];
#pragma unroll
    for (int i = 0; i < C; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[i][e] = 0.0f;
    auto span = [&](int i) {  // computed anew in each place: else 60 registers spill
        unsigned c = i * NT + threadIdx.x;
        asm volatile("" : "+v"(c));
        return span_of<VE>(c, a.cols);
    };
    // the wave's first chunk of its i-th ones, and the chunks there are: past them there is nothing to do
    const unsigned chunks = (a.cols + VE - 1) / VE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    auto first = [&](int i) { return i * NT + wave * kWave; };
    struct Row {
        Chunk<DT, VE> h[C], d[C], a[C];
        float rs;
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
    };
    Row cur, next;
    size_t row = blockIdx.x;
    if constexpr (AHEAD) load(next, row);
    for (; row < a.rows; row += gridDim.x) {
        const size_t base = row * a.cols, then = row + gridDim.x;
        if constexpr (AHEAD) {
            cur = next;
            if (then < a.rows) load(next, then);
        } else {
            load(cur, row);
        }
        auto &ch = cur.h, &cd = cur.d, &ca = cur.a;
        const float rs = cur.rs;
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            if (first(i) >= chunks) break;
            const Span s = span(i);
            Chunk<DT, VE> cw;
            cw.load(w + s.off);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float n = ch[i].get(e) * rs, dy = e >= static_cast<int>(s.dup) ? cd[i].get(e) : 0.0f;
                acc[i][e] = fmaf(dy, n, acc[i][e]);
                dot = fmaf(dy * cw.get(e), n, dot);
            }
        }
        const float mean = block_reduce<SumOp, NT>(dot, lds) / static_cast<float>(a.cols);
        S *dx = static_cast<S *>(a.dx) + base;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            if (first(i) >= chunks) break;
            // one chunk at a time, and what it unpacks to not kept from above: else 60 registers spill
            __builtin_amdgcn_sched_barrier(0);
            for (auto &r : ch[i].r) asm volatile("" : "+v"(r));
            for (auto &r : cd[i].r) asm volatile("" : "+v"(r));
            const Span s = span(i);
            Chunk<DT, VE> cw;
            cw.load(w + s.off);
            float t[VE];
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float n = ch[i].get(e) * rs, g = cd[i].get(e) * cw.get(e), u = n * mean;
                const float r = rs * (g - u);
                t[e] = a.dh ? r + ca[i].get(e) : r;
            }
            ch[i].set(t);
            store_span<DT, VE>(dx, s, ch[i]);
        }
    }
    float *part = a.part + static_cast<size_t>(blockIdx.x) * a.ld;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const Span s = span(i);
#pragma unroll
        for (int e = 0; e < VE; ++e)
            if (e >= static_cast<int>(s.dup)) part[s.off + e] = acc[i][e];
    }
}

// Rows longer than these hold: dx by a workgroup per row, which reads
// the row twice; dw by k_rms_dw_part, run before it (dx may be dy or h).
template <int DT, int NT>
__global__ __launch_bounds__(NT) void k_rms_bwd_long(RmsBwd a) {
    using S = typename Elem<DT>::S;
    constexpr int VE = Elem<DT>::kVec;
    __shared__ float lds[NT / kWave];
    const size_t row = blockIdx.x, base = row * a.cols;
    const S *h = static_cast<const S *>(a.h) + base, *dy = static_cast<const S *>(a.dy) + base;
    const S *dh = static_cast<const S *>(a.dh) + (a.dh ? base : 0), *w = static_cast<const S *>(a.w);
    S *dx = static_cast<S *>(a.dx) + base;
    const float rs = a.rstd[row];
    const unsigned whole = a.cols / VE, tail = whole * VE + threadIdx.x;
    float dot = 0.0f;
    for (unsigned i = threadIdx.x; i < whole; i += NT) {
        Chunk<DT, VE> ch, cd, cw;
        ch.load(h + i * VE);
        cd.load(dy + i * VE);
        cw.load(w + i * VE);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const float n = ch.get(e) * rs, g = cd.get(e) * cw.get(e);
            dot += g * n;
        }
    }
    if (tail < a.cols) {
        const float n = Elem<DT>::load(h[tail]) * rs, g = Elem<DT>::load(dy[tail]) * Elem<DT>::load(w[tail]);
        dot += g * n;
    }
    const float mean = block_reduce<SumOp, NT>(dot, lds) / static_cast<float>(a.cols);
    auto one = [&](float hv, float dv, float wv) {
        const float n = hv * rs, g = dv * wv, u = n * mean;
        return rs * (g - u);
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

// dw over the rows r0, r0 + gridDim.y, ... of a tile of columns.
template <int DT>
__global__ __launch_bounds__(kBlock) void k_rms_dw_part(RmsBwd a) {
    using S = typename Elem<DT>::S;
    constexpr int VE = Elem<DT>::kVec;
    const unsigned c = blockIdx.x * kBlock + threadIdx.x;
    if (c * VE >= a.cols) return;
    const Span s = span_of<VE>(c, a.cols);
    float acc[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) acc[e] = 0.0f;
    for (size_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
        Chunk<DT, VE> ch, cd;
        ch.load(static_cast<const S *>(a.h) + r * a.cols + s.off);
        cd.load(static_cast<const S *>(a.dy) + r * a.cols + s.off);
        const float rs = a.rstd[r];
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const float n = ch.get(e) * rs, t = cd.get(e) * n;
            acc[e] += t;
        }
    }
    float *part = a.part + static_cast<size_t>(blockIdx.y) * a.ld;
#pragma unroll
    for (int e = 0; e < VE; ++e)
        if (e >= static_cast<int>(s.dup)) part[s.off + e] = acc[e];
}

// ----------------------------------------------------------------- launch

template <int DT, int VE, int G, int C, int NT>
int fwd_launch(const RmsFwd &a, hipStream_t s) {
    constexpr int R = G <= kWave ? NT / G : 1;
    const size_t wgs = (a.rows + R - 1) / R;
    if (wgs > most_wgs(NT)) return CXM_E_TOO_LARGE;
    const dim3 grid(static_cast<unsigned>(wgs));
    if (whole_lines(a.x, a.cols, sizeof(typename Elem<DT>::S)) && whole_lines(a.res, a.cols, sizeof(typename Elem<DT>::S)))
        hipLaunchKernelGGL((k_rms_fwd<DT, VE, G, C, NT, true>), grid, dim3(NT), 0, s, a);
    else
        hipLaunchKernelGGL((k_rms_fwd<DT, VE, G, C, NT, false>), grid, dim3(NT), 0, s, a);
    return launch_status();
}

template <int DT>
int fwd_dispatch(const RmsFwd &a, hipStream_t s) {
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
    if (chunks <= 4096) return fwd_launch<DT, VE, 1024, 4, 1024>(a, s);
    if (a.rows > most_wgs(1024)) return CXM_E_TOO_LARGE;
    hipLaunchKernelGGL((k_rms_fwd_long<DT, 1024>), dim3(static_cast<unsigned>(a.rows)), dim3(1024), 0, s, a);
    return launch_status();
}

int fwd_any(const RmsFwd &a, int dtype, hipStream_t s) {
    switch (dtype) {
        case CXM_DT_F32: return fwd_dispatch<CXM_DT_F32>(a, s);
        case CXM_DT_BF16: return fwd_dispatch<CXM_DT_BF16>(a, s);
        default: return fwd_dispatch<CXM_DT_F16>(a, s);
    }
}

int bwd_parts(RmsBwd *a, size_t parts, cxm_stream_t st) {
    a->ld = (a->cols + 3) / 4 * 4;
    Workspace ws;
    const int rc = get_workspace(st, 0, parts * a->ld * sizeof(float), &ws);
    if (rc) return rc;
    a->part = static_cast<float *>(ws.scratch);
    return CXM_OK;
}

template <int DT, int VE, int G, int C, int NT>
int bwd_launch(RmsBwd a, void *dw, cxm_stream_t st) {
    constexpr int R = G <= kWave ? NT / G : 1;
    const size_t wgs = bwd_wgs(a.rows, R);
    const int rc = bwd_parts(&a, wgs, st);
    if (rc) return rc;
    const dim3 grid(static_cast<unsigned>(wgs));
    constexpr size_t E = sizeof(typename Elem<DT>::S);
    if (whole_lines(a.h, a.cols, E) && whole_lines(a.dy, a.cols, E) && whole_lines(a.dh, a.cols, E))
        hipLaunchKernelGGL((k_rms_bwd<DT, VE, G, C, NT, true>), grid, dim3(NT), 0, hs(st), a);
    else
        hipLaunchKernelGGL((k_rms_bwd<DT, VE, G, C, NT, false>), grid, dim3(NT), 0, hs(st), a);
    const int r = launch_status();
    return r ? r : col_sum(a.part, wgs, a.cols, a.ld, dw, DT, hs(st));
}

template <int DT, int C>
int bwd_wide(RmsBwd a, void *dw, cxm_stream_t st) {
    const size_t wgs = a.rows < device_cus() ? a.rows : device_cus();
    const int rc = bwd_parts(&a, wgs, st);
    if (rc) return rc;
    const dim3 grid(static_cast<unsigned>(wgs));
    constexpr size_t E = sizeof(typename Elem<DT>::S);
    if (whole_lines(a.h, a.cols, E) && whole_lines(a.dy, a.cols, E) && whole_lines(a.dh, a.cols, E))
        hipLaunchKernelGGL((k_rms_bwd_wide<DT, C, true>), grid, dim3(1024), 0, hs(st), a);
    else
        hipLaunchKernelGGL((k_rms_bwd_wide<DT, C, false>), grid, dim3(1024), 0, hs(st), a);
    const int r = launch_status();
    return r ? r : col_sum(a.part, wgs, a.cols, a.ld, dw, DT, hs(st));
}

template <int DT>
int bwd_dispatch(RmsBwd a, void *dw, cxm_stream_t st) {
    constexpr int VE = Elem<DT>::kVec;
    if (a.cols < static_cast<unsigned>(VE)) return bwd_launch<DT, 1, 16, 1, 256>(a, dw, st);
    const unsigned chunks = (a.cols + VE - 1) / VE;
    if (chunks <= 16) return bwd_launch<DT, VE, 16, 1, 256>(a, dw, st);
    if (chunks <= 64) return bwd_launch<DT, VE, 64, 1, 256>(a, dw, st);
    if (chunks <= 128) return bwd_launch<DT, VE, 64, 2, 256>(a, dw, st);
    if (chunks <= 256) return bwd_launch<DT, VE, 64, 4, 256>(a, dw, st);
    if (chunks <= 512) return bwd_launch<DT, VE, 256, 2, 256>(a, dw, st);
    if (chunks <= 1024) return bwd_launch<DT, VE, 512, 2, 512>(a, dw, st);
    if (chunks <= 2048) return bwd_wide<DT, 2>(a, dw, st);
    if constexpr (DT == CXM_DT_F32) {
        if (chunks <= 4096) return bwd_wide<DT, 4>(a, dw, st);
    }
    if (a.rows > most_wgs(1024)) return CXM_E_TOO_LARGE;
    const size_t tiles = (chunks + kBlock - 1) / kBlock;
    size_t parts = 4 * device_cus() / tiles;
    parts = parts < 1 ? 1 : parts > a.rows ? a.rows : parts;
    const int rc = bwd_parts(&a, parts, st);
    if (rc) return rc;
    hipLaunchKernelGGL((k_rms_dw_part<DT>), dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(parts)), dim3(kBlock),
                       0, hs(st), a);
    int r = launch_status();
    if (r == CXM_OK) r = col_sum(a.part, parts, a.cols, a.ld, dw, DT, hs(st));
    if (r) return r;
    hipLaunchKernelGGL((k_rms_bwd_long<DT, 1024>), dim3(static_cast<unsigned>(a.rows)), dim3(1024), 0, hs(st), a);
    return launch_status();
}

}  // namespace
}  // namespace cxm

extern "C" {

int cxm_rmsnorm_fwd_t(const void *x, const void *res, const void *w, float eps, void *h, void *y, uint8_t *q,
                      float *scale, float *rstd, size_t rows, size_t cols, int dtype, cxm_stream_t s) {
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
    } out[5] = {{h, n}, {y, n}, {q, q ? rows * cols : 0}, {scale, q ? rows * 4 : 0}, {rstd, rows * 4}};
    for (int i = 0; i < 5; ++i) {
        const bool in_place = i < 2;
        if (in_place ? overlap_not_same(out[i].p, out[i].n, x, n) || overlap_not_same(out[i].p, out[i].n, res, n)
                     : overlap(out[i].p, out[i].n, x, n) || overlap(out[i].p, out[i].n, res, n))
            return CXM_E_INVALID;
        if (overlap(out[i].p, out[i].n, w, cols * e)) return CXM_E_INVALID;
        for (int j = 0; j < i; ++j)
            if (overlap(out[i].p, out[i].n, out[j].p, out[j].n)) return CXM_E_INVALID;
    }
    const cxm::RmsFwd a{x, res, w, h, y, q, scale, rstd, rows, static_cast<unsigned>(cols), eps, 1};
    return cxm::fwd_any(a, dtype, cxm::hs(s));
}

int cxm_quant_rows_t(const void *x, uint8_t *q, float *scale, size_t rows, size_t cols, int dtype, cxm_stream_t s) {
    if (!cxm::is_float_dtype(dtype)) return CXM_E_INVALID;
    if (rows == 0) return CXM_OK;
    if (!x || !q || !scale || cols == 0) return CXM_E_INVALID;
    if (!cxm::row_shape_ok(rows, cols)) return CXM_E_TOO_LARGE;
    const size_t n = rows * cols;
    if (cxm::overlap(q, n, x, n * cxm::dtype_bytes(dtype)) || cxm::overlap(scale, rows * 4, x, n * cxm::dtype_bytes(dtype)) ||
        cxm::overlap(scale, rows * 4, q, n))
        return CXM_E_INVALID;
    const cxm::RmsFwd a{x,     nullptr, nullptr, nullptr, nullptr, q, scale, nullptr, rows, static_cast<unsigned>(cols),
                        0.0f, 0};
    return cxm::fwd_any(a, dtype, cxm::hs(s));
}

int cxm_rmsnorm_bwd_t(const void *h, const float *rstd, const void *w, const void *dy, const void *dh, void *dx,
                      void *dw, size_t rows, size_t cols, int dtype, cxm_stream_t s) {
    using cxm::overlap;
    using cxm::overlap_not_same;
    if (!cxm::is_float_dtype(dtype) || !dw || cols == 0) return CXM_E_INVALID;
    if (!cxm::row_shape_ok(rows, cols) || cols >= (size_t(1) << 26)) return CXM_E_TOO_LARGE;  // (col_sum's grid)
    const size_t e = cxm::dtype_bytes(dtype), n = rows * cols * e;
    cxm::RmsBwd a{h, w, dy, dh, rstd, dx, nullptr, rows, static_cast<unsigned>(cols), 0};
    if (rows == 0) return cxm::col_sum(nullptr, 0, cols, cols, dw, dtype, cxm::hs(s));  // an empty sum
    if (!h || !rstd || !w || !dy || !dx) return CXM_E_INVALID;
    // dx may be h, dy or dh itself
    for (const void *in : {h, dy, dh})
        if (overlap_not_same(dx, n, in, n) || overlap(dw, cols * e, in, n)) return CXM_E_INVALID;
    if (overlap(dx, n, w, cols * e) || overlap(dx, n, rstd, rows * 4) || overlap(dx, n, dw, cols * e) ||
        overlap(dw, cols * e, w, cols * e) || overlap(dw, cols * e, rstd, rows * 4))
        return CXM_E_INVALID;
    switch (dtype) {
        case CXM_DT_F32: return cxm::bwd_dispatch<CXM_DT_F32>(a, dw, s);
        case CXM_DT_BF16: return cxm::bwd_dispatch<CXM_DT_BF16>(a, dw, s);
        default: return cxm::bwd_dispatch<CXM_DT_F16>(a, dw, s);
    }
}

}  // extern "C"
