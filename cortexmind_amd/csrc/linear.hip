// A dense layer: y = act(x W + bias) + residual in fp32, bf16, fp16 or from
// e4m3 operands with scales, and its backward
//   dz = dy act'(z),  db = column sums of dz,  dx = dz W^T,  dW = x^T dz.
// The host side (plan, workspace, argument checks), the copies that bring
// ragged operands into the ring's form, the backward's first kernel and the
// fp32 epilogue.  The products are linear_ring.hip's and linear_skinny.hip's;
// in fp32 they are cxm_gemm_f32's, and the activation and the residual a
// pass over the result.
#include "linear.hpp"
#include "linear_act.hpp"

namespace cxm {
namespace {

inline hipStream_t hs(cxm_stream_t s) { return reinterpret_cast<hipStream_t>(s); }
inline size_t up(size_t v, size_t m) { return (v + m - 1) / m * m; }

// ------------------------------------------------ operands for the ring
//
// The ring's direct-to-LDS loads take 16-byte aligned pieces and whole stages
// of 64 bytes of k.  Where that fails and the staged form is the slower
// (linear_plan), an operand is copied once, its rows extended by zeros; one
// read and one write of it, against the product's many.
typedef unsigned u32x4b1 __attribute__((ext_vector_type(4), aligned(1)));

struct PadSide {
    const uint8_t *x;
    uint8_t *y;
    size_t rows, bytes, out_rows;  // stored rows and their length; rows of the copy, zero past them
    size_t row0;                   // the launch's first row
    unsigned pieces, tiles;        // 16-byte pieces of a row of the copy; workgroups per kPadRows rows
    unsigned wgs;
};

// A wave takes 1 KiB of kPadRows / 4 rows, its loads in flight together: no
// load stands in a branch, where the compiler would wait for it (2500x1003 and
// 1003x1499 8.3 us so).  A row's last piece is read as its last 16 bytes and
// shifted down; rows shorter than 16 bytes go byte by byte.
constexpr int kPadRows = 8;
__global__ __launch_bounds__(kBlock) void k_pad(PadSide a, PadSide b) {
    constexpr int R = kPadRows / (kBlock / kWave);
    const bool first = blockIdx.x < a.wgs;
    const PadSide &p = first ? a : b;
    const unsigned id = first ? blockIdx.x : blockIdx.x - a.wgs;
    const unsigned lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
    const unsigned piece = id % p.tiles * kWave + lane;
    const size_t r0 = p.row0 + static_cast<size_t>(id / p.tiles) * kPadRows + w * R, at = static_cast<size_t>(piece) * 16;
    if (piece >= p.pieces) return;
    uint64_t lo[R], hi[R];
    if (p.bytes >= 16) {
        const size_t o = at < p.bytes - 16 ? at : p.bytes - 16;
        const unsigned sh = at - o < 16 ? static_cast<unsigned>(at - o) * 8 : 128u;  // bits that belong to the piece before
        u32x4b1 v[R];
#pragma unroll
        for (int i = 0; i < R; ++i)
            v[i] = *reinterpret_cast<const u32x4b1 *>(p.x + (r0 + i < p.rows ? r0 + i : p.rows - 1) * p.bytes + o);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const uint64_t x = static_cast<uint64_t>(v[i].y) << 32 | v[i].x, y = static_cast<uint64_t>(v[i].w) << 32 | v[i].z;
            lo[i] = sh == 0 ? x : sh < 64 ? x >> sh | y << (64 - sh) : sh < 128 ? y >> (sh - 64) : 0;
            hi[i] = sh < 64 ? y >> sh : 0;
        }
    } else {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            lo[i] = hi[i] = 0;
            const uint8_t *q = p.x + (r0 + i < p.rows ? r0 + i : p.rows - 1) * p.bytes;
            for (size_t k = 0; at == 0 && k < p.bytes; ++k) {
                if (k < 8) lo[i] |= static_cast<uint64_t>(q[k]) << (8 * k);
                else hi[i] |= static_cast<uint64_t>(q[k]) << (8 * (k - 8));
            }
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (r0 + i >= p.out_rows) break;
        const bool in = r0 + i < p.rows;
        const uint64_t x = in ? lo[i] : 0, y = in ? hi[i] : 0;
        *reinterpret_cast<u32x4 *>(p.y + ((r0 + i) * p.pieces + piece) * 16) =
            u32x4{static_cast<unsigned>(x), static_cast<unsigned>(x >> 32), static_cast<unsigned>(y),
                  static_cast<unsigned>(y >> 32)};
    }
}

PadSide pad_side(const void *x, void *y, size_t rows, size_t bytes, size_t out_rows, size_t out_bytes) {
    const size_t pieces = out_bytes / 16;
    return PadSide{static_cast<const uint8_t *>(x), static_cast<uint8_t *>(y), rows, bytes, out_rows, 0,
                   static_cast<unsigned>(pieces), static_cast<unsigned>((pieces + kWave - 1) / kWave), 0};
}

// Both sides in one launch (out_rows 0: no such side); rows past what a grid holds,
// 2^23 workgroups a side, in launches of their own.
int pad_launch(PadSide a, PadSide b, hipStream_t s) {
    size_t next[2] = {0, 0};
    while (next[0] < a.out_rows || next[1] < b.out_rows) {
        for (int i = 0; i < 2; ++i) {
            PadSide &p = i ? b : a;
            p.row0 = next[i];
            p.wgs = 0;
            if (next[i] >= p.out_rows) continue;
            const size_t need = (p.out_rows - next[i] + kPadRows - 1) / kPadRows, most = most_wgs(kBlock) / 2 / p.tiles;
            const size_t groups = need < most ? need : most;
            p.wgs = static_cast<unsigned>(groups * p.tiles);
            next[i] += groups * kPadRows;
        }
        hipLaunchKernelGGL(k_pad, dim3(a.wgs + b.wgs), dim3(kBlock), 0, s, a, b);
        const int r = launch_status();
        if (r) return r;
    }
    return CXM_OK;
}

// ------------------------------------------------------------ fp32 layer

// y = act(z) + res over z = x W + bias, which gemm_ex left in `from`.
__global__ __launch_bounds__(kBlock) void k_linear_f32(const float *from, const float *res, float *y, size_t n, int act) {
    const size_t i = (static_cast<size_t>(blockIdx.x) * kBlock + threadIdx.x) * 4;
    if (i >= n) return;
    const int own = n - i < 4 ? static_cast<int>(n - i) : 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f}, r[4] = {0.f, 0.f, 0.f, 0.f};
    if (own == 4) {
        Chunk<CXM_DT_F32, 4> c;
        c.load(from + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = c.get(e);
        if (res) {
            c.load(res + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] = c.get(e);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < own) {
                v[e] = from[i + e];
                r[e] = res ? res[i + e] : 0.0f;
            }
    }
    act_apply<true, 4>(act, v);
    if (res) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += r[e];
    }
    if (own == 4) {
        Chunk<CXM_DT_F32, 4> c;
        c.set(v);
        c.store(y + i);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < own) y[i + e] = v[e];
    }
}

int linear_f32(const float *x, const float *w, const float *bias, const float *res, float *z, float *y, size_t m,
               size_t k, size_t n, int tw, int act, cxm_stream_t st) {
    // without z, y holds x W + bias for a moment (so a residual in y itself is refused)
    const bool fused = !z && !res && (act == CXM_ACT_NONE || act == CXM_ACT_RELU);
    float *to = z ? z : y;
    const size_t wgs = (m * n + 4 * kBlock - 1) / (4 * kBlock);
    if (wgs > most_wgs(kBlock)) return CXM_E_TOO_LARGE;
    const Epilogue e{bias, nullptr, fused ? act : CXM_ACT_NONE, 0, 0.0f};
    const int rc = gemm_ex(x, w, to, m, k, n, 0, tw, e, st);
    if (rc || fused || (to == y && !res && act == CXM_ACT_NONE)) return rc;
    hipLaunchKernelGGL(k_linear_f32, dim3(static_cast<unsigned>(wgs)), dim3(kBlock), 0, hs(st), to, res, y, m * n, act);
    return launch_status();
}

// ------------------------------------------------------- backward, first
//
// dz = dy act'(z) and the column sums of dz (unrounded, fp32): each of a
// workgroup's waves takes rows of one tile of 64 chunks; the waves meet in
// LDS, the workgroups' shares in k_col_sum, both in a fixed order (for few rows
// the last workgroup of a tile adding them costs what the launch does: 512x1024
// 21.5 -> 23.8 us for the whole backward, 98x86 13.5 -> 12.3).  bf16
// 4096x4096 with GELU: 19.6 us, 5.1 TB/s; 26 vector instructions an element, by
// the counters 12.5 us of the vector units beside 14.6 us of memory, and the
// two overlap only across waves.  Two
// and four rows in flight per wave (20.0, 21.9 us) and the next row loaded
// ahead of the slope (20.5, 19.6 with half the workgroups) gain nothing.
struct ActBwd {
    const void *z, *dy;
    void *dz;
    float *part;  // null: no sums wanted
    size_t rows;
    unsigned cols, ld;
    int act;
};

template <int DT, int VE>
__global__ __launch_bounds__(kBlock) void k_act_bwd(ActBwd a) {
    using S = typename Elem<DT>::S;
    constexpr bool FINE = DT == CXM_DT_F32;
    constexpr int W = kBlock / kWave;
    __shared__ float lds[W][kWave * VE];
    const unsigned lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
    const unsigned c = blockIdx.x * kWave + lane;
    const Span s = span_of<VE>(c, a.cols);
    float acc[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) acc[e] = 0.0f;
    const size_t step = static_cast<size_t>(gridDim.y) * W;
    for (size_t r = static_cast<size_t>(blockIdx.y) * W + w; r < a.rows; r += step) {
        const size_t o = r * a.cols;
        Chunk<DT, VE> cz, cd;
        float z[VE], d[VE];
        cd.load_nt(static_cast<const S *>(a.dy) + o + s.off);
        if (a.act != CXM_ACT_NONE) {
            cz.load_nt(static_cast<const S *>(a.z) + o + s.off);
#pragma unroll
            for (int e = 0; e < VE; ++e) z[e] = cz.get(e);
        }
        act_slope<FINE, VE>(a.act, z, d);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            d[e] *= cd.get(e);
            acc[e] += d[e];
        }
        if (a.dz) {
            cd.set(d);
            store_span<DT, VE>(static_cast<S *>(a.dz) + o, s, cd);
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int e = 0; e < VE; ++e) lds[w][e * kWave + lane] = acc[e];
    __syncthreads();
    if (w == 0) {
        float *part = a.part + static_cast<size_t>(blockIdx.y) * a.ld;
#pragma unroll
        for (int e = 0; e < VE; ++e)
            if (e >= static_cast<int>(s.dup))
                part[s.off + e] = combine_pairwise<SumOp, W>(&lds[0][e * kWave + lane], kWave * VE);
    }
}

// Row shares of the column sums.
size_t act_bwd_parts(size_t rows, size_t cols, int dtype) {
    const size_t ve = cols < (dtype == CXM_DT_F32 ? 4u : 8u) ? 1 : dtype == CXM_DT_F32 ? 4 : 8;
    const size_t tiles = (cols + kWave * ve - 1) / (kWave * ve), need = (rows + kBlock / kWave - 1) / (kBlock / kWave);
    size_t n = 8 * device_cus() / tiles;
    n = n < 1 ? 1 : n;
    n = n < need ? n : need;
    return n < 65535 ? n : 65535;
}

template <int DT, int VE>
int act_bwd_launch(const ActBwd &a, size_t parts, void *db, hipStream_t s) {
    const size_t tiles = (a.cols + kWave * VE - 1) / (kWave * VE);
    hipLaunchKernelGGL((k_act_bwd<DT, VE>), dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(parts)), dim3(kBlock),
                       0, s, a);
    const int r = launch_status();
    if (r || !db) return r;
    return col_sum(a.part, parts, a.cols, a.ld, db, DT, s);
}
template <int DT>
int act_bwd(const ActBwd &a, size_t parts, void *db, hipStream_t s) {
    if (a.cols < static_cast<unsigned>(Elem<DT>::kVec)) return act_bwd_launch<DT, 1>(a, parts, db, s);
    return act_bwd_launch<DT, Elem<DT>::kVec>(a, parts, db, s);
}

bool act_ok(int act) { return act == CXM_ACT_NONE || act == CXM_ACT_RELU || act == CXM_ACT_SIGMOID || act == CXM_ACT_TANH ||
                              act == CXM_ACT_GELU || act == CXM_ACT_SILU; }

// Sizes whose element and byte counts stay far within 64 bits, and whose rows
// the kernels number in 32.
bool dims_ok(size_t m, size_t k, size_t n) {
    constexpr size_t kRow = size_t(1) << 23;
    return m < (size_t(1) << 31) && k < kRow && n < kRow;
}

int run_one(const LinProduct &p, cxm_stream_t st) {
    LinPlan l;
    int rc = linear_plan(p, &l);
    if (rc) return rc;
    Workspace ws{};
    if (l.bytes() || l.counters()) {
        rc = get_workspace(st, l.counters(), l.bytes(), &ws);
        if (rc) return rc;
    }
    return linear_run(p, l, static_cast<char *>(ws.scratch), ws.counters, hs(st));
}

}  // namespace

// The ring's tile and K splits.
int linear_plan(const LinProduct &p, LinPlan *l) {
    if (linear_skinny_plan(p, l)) return CXM_OK;
    *l = LinPlan{};
    const size_t unit = 2, es = dtype_bytes(p.dtype), kb = p.K * es;
    // rows of k: whole stages of 64 bytes; rows across k: whole chunks of 16 bytes, and whole stages of rows
    const size_t kpad = up(kb, 64) / unit;  // units along K
    l->stages = kpad / 32;
    l->copy_a = !aligned16(p.a) || (p.ta ? p.M % 8 != 0 || p.K % 32 != 0 : kb % 64 != 0);
    l->copy_b = !aligned16(p.b) || (p.tb ? kb % 64 != 0 : p.N % 8 != 0 || p.K % 32 != 0);
    l->lda = p.ta ? up(p.M, 8) : kpad;
    l->ldb = p.tb ? kpad : up(p.N, 8);
    if (l->lda > (size_t(1) << 23) || l->ldb > (size_t(1) << 23)) return CXM_E_TOO_LARGE;  // (never, by dims_ok)
    const size_t cus = device_cus();
    auto tiles = [&](size_t tm, size_t tn) { return ((p.M + tm - 1) / tm) * ((p.N + tn - 1) / tn); };
    // The tile, by what these cost at K = 1024 (us; CUs of 256):
    //  * 256: a round of up to one tile per CU about 37 (64 of them 27);
    //  * 128: 10 and 11 for each 256 of them (64 of them 9.8, 240 13.3, 1024 45);
    //  * 64, several on a CU: 3 and 3.9 for each 256 (256 of them 6.8, 960 19.2),
    //    so 128 from half as many tiles as CUs.  By tiles alone, this misses with
    //    B [K, N], whose rows a 64 tile takes in 128-byte pieces: 225x1024x5000
    //    18.0 us (on 128 10.2), 282x8256x4128 92.7 (74.8), at short K the other
    //    way (3389x64x686 8.8, on 64 6.6); within 2% on average with B [N, K];
    //  * 32x64 up to 32 rows (16x4096x4096 10.1, on 64s 10.5; x8192 18.7 / 20.6).
    const size_t t256 = tiles(256, 256), t128 = tiles(128, 128);
    const double c256 = 3.4 * static_cast<double>((t256 + cus - 1) / cus), c128 = 1.0 + static_cast<double>(t128) / cus;
    const bool few = p.M <= 32 && !p.ta;
    l->kernel = few ? 32 : c256 <= c128 ? 256 : t128 >= cus / 2 ? 128 : 64;
    const size_t tm = static_cast<size_t>(l->kernel), tn = few ? 64 : tm;
    l->tiles_m = (p.M + tm - 1) / tm;
    l->tiles_n = (p.N + tn - 1) / tn;
    l->tiles = l->tiles_m * l->tiles_n;
    // K over up to one workgroup per CU, each split worth its meeting: 32
    // stages where four groups share them, else 8 (16x1024x4096 on 64 tiles 5.8,
    // in two 6.7; 512x4096x512 on 64 tiles 15.9, in four 10.0, in eight 10.6)
    l->splits = 1;
    if (tm <= 64 && l->tiles < cus) {
        l->splits = cus / l->tiles;
        const size_t most = l->stages / (few ? 32 : 8);
        if (l->splits > most) l->splits = most;
        if (l->splits < 1) l->splits = 1;
    }
    l->per = (l->stages + l->splits - 1) / l->splits;
    l->splits = (l->stages + l->per - 1) / l->per;
    if (l->tiles > most_wgs(1024) / l->splits) return CXM_E_TOO_LARGE;
    // Operands that the direct loads cannot take go through registers as they
    // are, or are copied first.  A copy costs about 6 us and its bytes at 3
    // TB/s, a stage through registers 0.15 us more on tiles of 64 (301x4001x301
    // 14.8 us / copied 18.8, 100x4001x4001 22.9 / 28.6, but 701x8001x1201 85 /
    // 52) and, its waves reading each weight once, nothing on 32x64 (20x4001x4001
    // 16.1 / 26.9, e4m3 20x8001x8001 17.9 / 37.6); larger tiles gain nothing
    // (128: 2500x1003x1499 22.5 / 22.3; 256: 4001^3 204 / 146).
    const size_t copy_a = (p.ta ? kpad : p.M) * l->lda * unit, copy_b = (p.tb ? p.N : kpad) * l->ldb * unit;
    if ((l->copy_a || l->copy_b) && tm <= 64 && (p.ta ? p.M : p.K) * es >= 16 && (p.tb ? p.K : p.N) * es >= 16) {
        const double rounds = static_cast<double>((l->tiles * l->splits + cus - 1) / cus);
        const double staged = few ? 0.0 : 0.15 * static_cast<double>(l->per) * rounds;
        const double copied = 6.0 + (static_cast<double>(l->copy_a ? copy_a : 0) + static_cast<double>(l->copy_b ? copy_b : 0)) / 3e6;
        l->staged = staged < copied;
        if (l->staged) l->copy_a = l->copy_b = false;
        // Staged 16-bit tiles wait for their own loads more than for the CU: two
        // of them per CU from 40 stages each (100x4001x4001 [K,N] 26.8 -> 20.4 us,
        // 127x5887x1818 [N,K] 19.6 -> 18.9, three 24.2; e4m3 200x8001x2001 22.7
        // -> 23.2; direct loads 128x5888x1792 13.1 -> 14.8)
        if (l->staged && !few && es == 2 && l->per >= 40 && l->tiles * l->splits <= cus) {
            l->splits *= 2;
            l->per = (l->stages + l->splits - 1) / l->splits;
            l->splits = (l->stages + l->per - 1) / l->per;
        }
    }
    if (l->copy_a) l->bytes_a = up(copy_a, 256);
    if (l->copy_b) l->bytes_b = up(copy_b, 256);
    if (l->splits > 1) l->bytes_part = up(l->tiles * l->splits * tm * tn * sizeof(float), 256);
    return CXM_OK;
}

int linear_run(const LinProduct &p, const LinPlan &l, char *scratch, unsigned *counters, hipStream_t s) {
    if (l.kernel == 0)
        return linear_skinny_run(p, l, l.bytes_part ? reinterpret_cast<float *>(scratch) : nullptr,
                                 l.splits > 1 ? counters : nullptr, s);
    const size_t es = dtype_bytes(p.dtype);
    const void *a = p.a, *b = p.b;
    const size_t krows = l.stages * 32;
    PadSide pa{}, pb{};
    if (l.copy_a) {
        a = scratch;
        pa = p.ta ? pad_side(p.a, scratch, p.K, p.M * es, krows, l.lda * 2)
                  : pad_side(p.a, scratch, p.M, p.K * es, p.M, l.lda * 2);
    }
    if (l.copy_b) {
        b = scratch + l.bytes_a;
        pb = p.tb ? pad_side(p.b, scratch + l.bytes_a, p.N, p.K * es, p.N, l.ldb * 2)
                  : pad_side(p.b, scratch + l.bytes_a, p.K, p.N * es, krows, l.ldb * 2);
    }
    const int rc = pad_launch(pa, pb, s);
    if (rc) return rc;
    return linear_ring_run(p, l, a, b, reinterpret_cast<float *>(scratch + l.bytes_a + l.bytes_b), counters, s);
}

}  // namespace cxm

extern "C" {

int cxm_linear_fwd_t(const void *x, const void *w, const void *bias, const void *res, void *z, void *y, size_t m,
                     size_t k, size_t n, int trans_w, int act, int dtype, cxm_stream_t s) {
    using namespace cxm;
    if (!is_float_dtype(dtype) || !act_ok(act)) return CXM_E_INVALID;
    if (m == 0 || n == 0) return CXM_OK;
    if (!x || !w || !y || k == 0) return CXM_E_INVALID;
    if (!dims_ok(m, k, n)) return CXM_E_TOO_LARGE;
    const size_t e = dtype_bytes(dtype), out = m * n * e;
    const bool in_place = dtype != CXM_DT_F32 || z;  // y may be res itself
    if ((in_place ? overlap_not_same(y, out, res, out) : overlap(y, out, res, out)) || overlap(z, out, res, out) ||
        overlap(y, out, z, out))
        return CXM_E_INVALID;
    for (const void *o : {static_cast<const void *>(y), static_cast<const void *>(z)})
        if (overlap(o, out, x, m * k * e) || overlap(o, out, w, k * n * e) || overlap(o, out, bias, n * e)) return CXM_E_INVALID;
    if (dtype == CXM_DT_F32)
        return linear_f32(static_cast<const float *>(x), static_cast<const float *>(w), static_cast<const float *>(bias),
                          static_cast<const float *>(res), static_cast<float *>(z), static_cast<float *>(y), m, k, n,
                          trans_w != 0, act, s);
    const LinProduct p{x, w, m, k, n, false, trans_w != 0, dtype, dtype, {bias, res, z, y, nullptr, nullptr, act}};
    return run_one(p, s);
}

int cxm_linear_q8_fwd(const uint8_t *x, const float *x_scale, const uint8_t *w, const float *w_scale, const void *bias,
                      const void *res, void *z, void *y, size_t m, size_t k, size_t n, int act, int dtype,
                      cxm_stream_t s) {
    using namespace cxm;
    if ((dtype != CXM_DT_BF16 && dtype != CXM_DT_F16) || !act_ok(act)) return CXM_E_INVALID;
    if (m == 0 || n == 0) return CXM_OK;
    if (!x || !w || !x_scale || !w_scale || !y || k == 0) return CXM_E_INVALID;
    if (!dims_ok(m, k, n)) return CXM_E_TOO_LARGE;
    const size_t out = m * n * 2;
    if (overlap_not_same(y, out, res, out) || overlap(z, out, res, out) || overlap(y, out, z, out)) return CXM_E_INVALID;
    for (const void *o : {static_cast<const void *>(y), static_cast<const void *>(z)})
        if (overlap(o, out, x, m * k) || overlap(o, out, w, k * n) || overlap(o, out, bias, n * 2) ||
            overlap(o, out, x_scale, m * 4) || overlap(o, out, w_scale, n * 4))
            return CXM_E_INVALID;
    const LinProduct p{x, w, m, k, n, false, true, CXM_DT_E4M3, dtype, {bias, res, z, y, x_scale, w_scale, act}};
    return run_one(p, s);
}

int cxm_linear_bwd_t(const void *x, const void *w, const void *z, const void *dy, void *dz, void *dx, void *dw, void *db,
                     size_t m, size_t k, size_t n, int trans_w, int act, int dtype, cxm_stream_t s) {
    using namespace cxm;
    if (!is_float_dtype(dtype) || !act_ok(act)) return CXM_E_INVALID;
    if (m == 0 || n == 0 || k == 0) return CXM_E_INVALID;
    if (!dims_ok(m, k, n) || m >= (size_t(1) << 23)) return CXM_E_TOO_LARGE;
    const bool none = act == CXM_ACT_NONE;
    if (!dy || (!none && (!z || !dz)) || (dx && !w) || (dw && !x)) return CXM_E_INVALID;
    const size_t e = dtype_bytes(dtype), mn = m * n * e, mk = m * k * e, kn = k * n * e;
    // dz may be z or dy itself; no other output meets an input or another output
    if (overlap_not_same(dz, mn, z, mn) || overlap_not_same(dz, mn, dy, mn)) return CXM_E_INVALID;
    const struct {
        const void *p;
        size_t n;
    } out[4] = {{dz, mn}, {dx, mk}, {dw, kn}, {db, n * e}}, in[4] = {{x, mk}, {w, kn}, {z, mn}, {dy, mn}};
    for (int i = 0; i < 4; ++i) {
        for (int j = 0; j < 4; ++j)
            if (!(i == 0 && j >= 2) && overlap(out[i].p, out[i].n, in[j].p, in[j].n)) return CXM_E_INVALID;
        for (int j = 0; j < i; ++j)
            if (overlap(out[i].p, out[i].n, out[j].p, out[j].n)) return CXM_E_INVALID;
    }
    const bool f32 = dtype == CXM_DT_F32;
    const bool first = db || dz;  // dz to write or sums to make
    const void *g = dz ? dz : dy;
    const LinEpi plain{nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, CXM_ACT_NONE};
    // dx [m, k] = dz W^T; dW [k, n] = x^T dz, or stored [n, k]: dz^T x
    LinProduct px{g, w, m, n, k, false, trans_w == 0, dtype, dtype, plain};
    LinProduct pw = trans_w ? LinProduct{g, x, n, m, k, true, false, dtype, dtype, plain}
                            : LinProduct{x, g, k, m, n, true, false, dtype, dtype, plain};
    px.e.y = dx;
    pw.e.y = dw;
    LinPlan lx{}, lw{};
    size_t bytes = 0, counters = 0;
    const size_t parts = act_bwd_parts(m, n, dtype), ld = (n + 3) / 4 * 4;
    if (db) bytes = parts * ld * sizeof(float);
    if (!f32) {
        for (int i = 0; i < 2; ++i) {
            if (!(i ? dw : dx)) continue;
            LinPlan &l = i ? lw : lx;
            const int rc = linear_plan(i ? pw : px, &l);
            if (rc) return rc;
            bytes = l.bytes() > bytes ? l.bytes() : bytes;
            counters = l.counters() > counters ? l.counters() : counters;
        }
    }
    Workspace ws{};
    if (bytes || counters) {  // once, before the first launch
        const int rc = get_workspace(s, counters, bytes, &ws);
        if (rc) return rc;
    }
    if (first) {
        const ActBwd a{z, dy, dz, db ? static_cast<float *>(ws.scratch) : nullptr, m, static_cast<unsigned>(n),
                       static_cast<unsigned>(ld), act};
        const int rc = f32 ? act_bwd<CXM_DT_F32>(a, parts, db, hs(s))
                       : dtype == CXM_DT_BF16 ? act_bwd<CXM_DT_BF16>(a, parts, db, hs(s))
                                              : act_bwd<CXM_DT_F16>(a, parts, db, hs(s));
        if (rc) return rc;
    }
    if (f32) {
        const auto *gf = static_cast<const float *>(g), *xf = static_cast<const float *>(x);
        if (dx) {
            const int rc = cxm_gemm_f32(gf, static_cast<const float *>(w), static_cast<float *>(dx), m, n, k, 0, !trans_w,
                                        nullptr, CXM_ACT_NONE, nullptr, s);
            if (rc) return rc;
        }
        if (!dw) return CXM_OK;
        return trans_w ? cxm_gemm_f32(gf, xf, static_cast<float *>(dw), n, m, k, 1, 0, nullptr, CXM_ACT_NONE, nullptr, s)
                       : cxm_gemm_f32(xf, gf, static_cast<float *>(dw), k, m, n, 1, 0, nullptr, CXM_ACT_NONE, nullptr, s);
    }
    if (dx) {
        const int rc = linear_run(px, lx, static_cast<char *>(ws.scratch), ws.counters, hs(s));
        if (rc) return rc;
    }
    return dw ? linear_run(pw, lw, static_cast<char *>(ws.scratch), ws.counters, hs(s)) : CXM_OK;
}

}  // extern "C"
