// Rows of a table looked up by token and scaled, and the table's gradient.
//
//   y[t] = table[ids[t]] * scale
//   dw[v] = scale * sum over t with ids[t] == v of dy[t]  (+ dw[v])
//
// Both are bound by memory.  The gradient's tokens are sorted by id first, so
// that every row of dw is one sum in the order of the tokens (no atomics on
// floats: the same bits every time) and is written once.  Two launches:
//  * k_embed_sort: a workgroup owns a range of ids.  It reads all ids twice
//    (they lie in L2), counts those below its range, which says where its part
//    of the sorted list begins, and places those in it in order; the rows that
//    no token has become zero in the same launch.
//  * k_embed_sum: a wave takes up to L neighbours of the sorted list and a tile
//    of columns, and writes the rows of ids that lie within its part; what an
//    id's tokens give in several waves meets in LDS, in several workgroups in
//    scratch, added up by the last of them to arrive, in the list's order.
#include "chunk.hpp"

namespace cxm {
namespace {

inline hipStream_t hs(cxm_stream_t s) { return reinterpret_cast<hipStream_t>(s); }

// ---------------------------------------------------------------- forward

// G lanes per row piece of G chunks, U tokens per group of lanes.
template <int DT, int VE, int G, int U>
__global__ __launch_bounds__(kBlock) void k_embed(const typename Elem<DT>::S *table, const int32_t *ids, float scale,
                                                  typename Elem<DT>::S *y, size_t tokens, size_t vocab, unsigned cols,
                                                  unsigned tiles) {
    constexpr int R = kBlock / G;
    const size_t blk = blockIdx.x / tiles;
    const unsigned tile = blockIdx.x - static_cast<unsigned>(blk) * tiles;
    const Span s = span_of<VE>(tile * G + threadIdx.x % G, cols);
    const size_t first = (blk * R + threadIdx.x / G) * U;
    int id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) id[u] = ids[first + u < tokens ? first + u : tokens - 1];
    Chunk<DT, VE> c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const bool in = id[u] >= 0 && static_cast<size_t>(id[u]) < vocab;
        c[u].load(table + (in ? static_cast<size_t>(id[u]) * cols : 0) + s.off);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (first + u >= tokens) break;
        const bool in = id[u] >= 0 && static_cast<size_t>(id[u]) < vocab;
        const float other = id[u] < 0 ? 0.0f : __builtin_nanf("");
        float v[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) v[e] = in ? c[u].get(e) * scale : other;
        c[u].set(v);
        store_span<DT, VE>(y + (first + u) * cols, s, c[u]);
    }
}

template <int DT, int VE, int G, int U>
int fwd_launch(const void *table, const int32_t *ids, float scale, void *y, size_t tokens, size_t vocab, unsigned cols,
               hipStream_t s) {
    using S = typename Elem<DT>::S;
    const unsigned tiles = ceil_div(ceil_div(cols, VE), G);
    const size_t blks = (tokens + static_cast<size_t>(kBlock / G) * U - 1) / (static_cast<size_t>(kBlock / G) * U);
    if (blks > most_wgs(kBlock) / tiles) return CXM_E_TOO_LARGE;
    hipLaunchKernelGGL((k_embed<DT, VE, G, U>), dim3(static_cast<unsigned>(blks * tiles)), dim3(kBlock), 0, s,
                       static_cast<const S *>(table), ids, scale, static_cast<S *>(y), tokens, vocab, cols, tiles);
    return launch_status();
}

template <int DT>
int fwd_dispatch(const void *table, const int32_t *ids, float scale, void *y, size_t tokens, size_t vocab, unsigned cols,
                 hipStream_t s) {
    constexpr int VE = Elem<DT>::kVec;
    if (cols < static_cast<unsigned>(VE)) return fwd_launch<DT, 1, 16, 1>(table, ids, scale, y, tokens, vocab, cols, s);
    const unsigned chunks = ceil_div(cols, VE);
    if (chunks <= 16) return fwd_launch<DT, VE, 16, 1>(table, ids, scale, y, tokens, vocab, cols, s);
    if (tokens < 4 * device_cus()) return fwd_launch<DT, VE, 64, 1>(table, ids, scale, y, tokens, vocab, cols, s);
    return fwd_launch<DT, VE, 64, 4>(table, ids, scale, y, tokens, vocab, cols, s);
}

// --------------------------------------------------------------- backward

struct Place {
    int id, token;
};

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr unsigned kSortIds = 512;  // most ids of a workgroup
constexpr int kSortAhead = 8;       // groups of 64 ids in flight

struct SortArgs {
    const int32_t *ids;
    size_t tokens, vocab;
    unsigned range;        // ids per workgroup, at most kSortIds
    Place *sorted;         // [tokens]
    unsigned *starts;      // [vocab + 1]: where each id's tokens begin
    char *dw;              // null: accumulating, nothing becomes zero
    size_t row_bytes;
};

// Zeros over a row of n bytes at 2-byte alignment, by one wave.
__device__ __forceinline__ void zero_row(char *p, size_t n, unsigned lane) {
    const size_t whole = n / 16;
    for (size_t i = lane; i < whole; i += kWave) *reinterpret_cast<u32x4e *>(p + i * 16) = u32x4e{0, 0, 0, 0};
    const size_t at = whole * 16 + lane * 2;
    if (at < n) *reinterpret_cast<uint16_t *>(p + at) = 0;
}

__global__ __launch_bounds__(kSortThreads) void k_embed_sort(SortArgs a) {
    __shared__ unsigned hist[kSortWaves][kSortIds];
    __shared__ unsigned wsum[kSortWaves], below_all;
    __shared__ unsigned long long absent[kSortIds / kWave];  // a bit for each id that no token has
    const unsigned lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const size_t v0 = static_cast<size_t>(blockIdx.x) * a.range;
    const unsigned range = static_cast<unsigned>(a.vocab - v0 < a.range ? a.vocab - v0 : a.range);
    const size_t per = (a.tokens + kSortThreads - 1) / kSortThreads * kWave;  // a wave's tokens, in a row
    const size_t t0 = wave * per < a.tokens ? wave * per : a.tokens, t1 = t0 + per < a.tokens ? t0 + per : a.tokens;
    for (unsigned i = threadIdx.x; i < kSortWaves * kSortIds; i += kSortThreads) (&hist[0][0])[i] = 0;
    if (threadIdx.x == 0) below_all = 0;
    __syncthreads();
    // ids[i], or -1 (no id) past the wave's part
    auto batch = [&](size_t at, int(&id)[kSortAhead]) {
#pragma unroll
        for (int k = 0; k < kSortAhead; ++k) {
            const size_t i = at + k * kWave + lane;
            id[k] = i < t1 ? a.ids[i] : -1;
        }
    };
    unsigned below = 0;
    for (size_t at = t0; at < t1; at += kSortAhead * kWave) {
        int id[kSortAhead];
        batch(at, id);
#pragma unroll
        for (int k = 0; k < kSortAhead; ++k) {
            const long long r = static_cast<long long>(id[k]) - static_cast<long long>(v0);
            below += id[k] >= 0 && r < 0;
            if (r >= 0 && r < range) atomicAdd(&hist[wave][r], 1u);
        }
    }
    atomicAdd(&below_all, below);
    __syncthreads();
    // where each wave's tokens of each id go: ids in turn, within one the waves in turn
    const unsigned r = threadIdx.x;
    unsigned total = 0;
    if (r < range) {
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) total += hist[w][r];
    }
    unsigned incl = total;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const unsigned o = __shfl_up(incl, d);
        if (lane >= static_cast<unsigned>(d)) incl += o;
    }
    if (lane == kWave - 1) wsum[wave] = incl;
    __syncthreads();
    unsigned at = below_all + incl - total;
    for (unsigned w = 0; w < wave; ++w) at += wsum[w];
    if (r < range) {
        a.starts[v0 + r] = at;
        if (v0 + r + 1 == a.vocab) a.starts[a.vocab] = at + total;
        for (int w = 0; w < kSortWaves; ++w) {
            const unsigned n = hist[w][r];
            hist[w][r] = at;
            at += n;
        }
    }
    const unsigned long long none = __ballot(r < range && total == 0);
    if (lane == 0 && wave < kSortIds / kWave) absent[wave] = none;
    __syncthreads();
    const int bits = 32 - __clz((range - 1) | 1);
    for (size_t base = t0; base < t1; base += kSortAhead * kWave) {
        int id[kSortAhead];
        batch(base, id);
#pragma unroll
        for (int k = 0; k < kSortAhead; ++k) {
            const long long d = static_cast<long long>(id[k]) - static_cast<long long>(v0);
            const bool in = d >= 0 && d < range;
            unsigned long long same = __ballot(in);
            if (same == 0) continue;
            const unsigned key = in ? static_cast<unsigned>(d) : 0;
            for (int b = 0; b < bits; ++b) {  // the lanes that have this lane's id
                const unsigned long long one = __ballot(key >> b & 1);
                same &= key >> b & 1 ? one : ~one;
            }
            if (in) {
                const unsigned rank = __popcll(same & ((1ull << lane) - 1));
                const unsigned to = hist[wave][key] + rank;
                a.sorted[to] = Place{id[k], static_cast<int>(base + k * kWave + lane)};
                // one lane moves the place on, after all have read it and before the next group does
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                if (rank == 0) hist[wave][key] = to + __popcll(same);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
        }
    }
    if (a.dw) {
        for (unsigned i = wave; i < range; i += kSortWaves)
            if (absent[i / kWave] >> (i % kWave) & 1) zero_row(a.dw + (v0 + i) * a.row_bytes, a.row_bytes, lane);
    }
}

constexpr int kSumThreads = 512, kSumWaves = kSumThreads / kWave;
constexpr size_t kTicket = 16;  // words between two of its tickets

struct SumArgs {
    const void *dy;
    void *dw;
    const Place *sorted;
    const unsigned *starts;
    float *part;        // [spans][2][tiles * 64 * VE]: what an id's tokens give in a span, of the id that
                        // began before it and of the one that goes on after it
    unsigned *tickets;  // [spans * tiles], kTicket apart
    size_t vocab;
    unsigned cols, tiles, per;  // per: a wave's places
    float scale;
    int accumulate;
};

template <int DT, int GT, int VE>
__global__ __launch_bounds__(kSumThreads) void k_embed_sum(SumArgs a) {
    using S = typename Elem<DT>::S;
    using SG = typename Elem<GT>::S;
    constexpr int AH = 8;  // rows in flight
    __shared__ float head[kSumWaves][VE][kWave], tail[kSumWaves][VE][kWave];
    // of each wave: 1 its first id began before it, 2 that id also goes on after it, 4 its last id began in it and goes on
    __shared__ int kind[kSumWaves];
    __shared__ int last_id[kSumWaves], flag;
    const unsigned lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const unsigned span = blockIdx.x / a.tiles, tile = blockIdx.x - span * a.tiles;
    const unsigned all = a.starts[a.vocab];
    const unsigned from = span * (kSumWaves * a.per);
    if (from >= all) return;
    const unsigned p0 = from + wave * a.per < all ? from + wave * a.per : all, p1 = p0 + a.per < all ? p0 + a.per : all;
    const unsigned col = tile * kWave + lane;
    const Span s = span_of<VE>(col, a.cols);
    const S *dy = static_cast<const S *>(a.dy) + s.off;
    auto finish = [&](int id, const float(&sum)[VE]) {
        SG *row = static_cast<SG *>(a.dw) + static_cast<size_t>(id) * a.cols;
        float v[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) v[e] = sum[e] * a.scale;
        // dw's element may be wider than dy's: its chunks are then halves
        constexpr int VG = VE == 1 ? 1 : Elem<GT>::kVec;
#pragma unroll
        for (int h = 0; h < VE / VG; ++h) {
            Chunk<GT, VG> c;
            float t[VG];
            if (a.accumulate) c.load(row + s.off + h * VG);
#pragma unroll
            for (int e = 0; e < VG; ++e) t[e] = a.accumulate ? c.get(e) + v[h * VG + e] : v[h * VG + e];
            c.set(t);
            const unsigned dup = s.dup > static_cast<unsigned>(h * VG) ? s.dup - h * VG : 0;
            store_span<GT, VG>(row, Span{s.off + h * VG, dup}, c);
        }
    };
    float acc[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) acc[e] = 0.0f;
    int k = 0, cur = -1;
    if (p0 < p1) {
        const unsigned n = p1 - p0;
        bool began = true;  // whether the id being added up began in this wave
        for (unsigned b0 = 0; b0 < n; b0 += kWave) {
            const unsigned m = n - b0 < kWave ? n - b0 : kWave;
            const Place mine = a.sorted[p0 + b0 + (lane < m ? lane : m - 1)];
            if (b0 == 0) {
                cur = readlane(mine.id, 0);
                began = a.starts[cur] == p0;
            }
            for (unsigned i0 = 0; i0 < m; i0 += AH) {
                Chunk<DT, VE> c[AH];
#pragma unroll
                for (int u = 0; u < AH; ++u) {
                    const unsigned i = i0 + u < m ? i0 + u : m - 1;
                    c[u].load(dy + static_cast<size_t>(static_cast<unsigned>(readlane(mine.token, i))) * a.cols);
                }
#pragma unroll
                for (int u = 0; u < AH; ++u) {
                    if (i0 + u >= m) break;
                    const int id = readlane(mine.id, i0 + u);
                    if (id != cur) {
                        if (began) {
                            finish(cur, acc);
                        } else {
                            k |= 1;
#pragma unroll
                            for (int e = 0; e < VE; ++e) head[wave][e][lane] = acc[e];
                        }
#pragma unroll
                        for (int e = 0; e < VE; ++e) acc[e] = 0.0f;
                        cur = id;
                        began = true;
                    }
#pragma unroll
                    for (int e = 0; e < VE; ++e) acc[e] += c[u].get(e);
                }
            }
        }
        const bool ends = a.starts[cur + 1] <= p1;
        if (began && ends) {
            finish(cur, acc);
        } else if (began) {
            k |= 4;
#pragma unroll
            for (int e = 0; e < VE; ++e) tail[wave][e][lane] = acc[e];
        } else {
            k |= ends ? 1 : 3;
#pragma unroll
            for (int e = 0; e < VE; ++e) head[wave][e][lane] = acc[e];
        }
    }
    if (lane == 0) {
        kind[wave] = k;
        last_id[wave] = cur;
    }
    __syncthreads();
    // What the waves share: each wave with a tail adds the heads behind it; the first wave the heads of an
    // id that began before the workgroup.
    const size_t width = static_cast<size_t>(a.tiles) * kWave * VE;
    float *part = a.part + static_cast<size_t>(span) * 2 * width + static_cast<size_t>(tile) * kWave * VE;
    auto chain = [&](unsigned w, float(&sum)[VE]) {  // adds heads from wave w on; whether the id ends within the workgroup
        for (; w < kSumWaves; ++w) {
#pragma unroll
            for (int e = 0; e < VE; ++e) sum[e] += head[w][e][lane];
            if (!(kind[w] & 2)) return true;
        }
        return false;
    };
    auto publish = [&](int slot, const float(&sum)[VE]) {
#pragma unroll
        for (int e = 0; e < VE; ++e) st_dev(part + slot * width + e * kWave + lane, sum[e]);
    };
    if (kind[wave] & 4) {
        float sum[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) sum[e] = tail[wave][e][lane];
        if (chain(wave + 1, sum)) finish(last_id[wave], sum);
        else publish(1, sum);
    }
    if (wave == 0 && (kind[0] & 1)) {
        float sum[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) sum[e] = 0.0f;
        chain(0, sum);
        publish(0, sum);
    }
    // An id in several workgroups: the last of them to have stored its part adds them up.
    const unsigned places = kSumWaves * a.per, to = from + places < all ? from + places : all;
    const int ids[2] = {a.sorted[from].id, a.sorted[to - 1].id};
    for (int which = 0; which < 2; ++which) {
        const unsigned s0 = a.starts[ids[which]], s1 = a.starts[ids[which] + 1];
        const unsigned g0 = s0 / places, g1 = (s1 - 1) / places;
        // 0: it began before this workgroup; 1: it began here and goes on
        if (which == 0 ? g0 == span : (g0 != span || g1 == span)) continue;
        const bool last = last_block_ticket(a.tickets + (static_cast<size_t>(g0) * a.tiles + tile) * kTicket, g1 - g0 + 1, &flag);
        if (!last) continue;
        // each wave a run of the parts, one after the other
        const unsigned count = g1 - g0 + 1, each = (count + kSumWaves - 1) / kSumWaves;
        const unsigned c0 = wave * each < count ? wave * each : count, c1 = c0 + each < count ? c0 + each : count;
        float sum[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) sum[e] = 0.0f;
        for (unsigned c = c0; c < c1; c += 2) {
            float v[2][VE];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const unsigned cc = c + u < c1 ? c + u : c;
                const float *p = a.part + (static_cast<size_t>(g0 + cc) * 2 + (cc == 0 ? 1 : 0)) * width +
                                 static_cast<size_t>(tile) * kWave * VE + lane;
#pragma unroll
                for (int e = 0; e < VE; ++e) v[u][e] = ld_dev(p + e * kWave);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if (c + u >= c1) break;
#pragma unroll
                for (int e = 0; e < VE; ++e) sum[e] += v[u][e];
            }
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < VE; ++e) head[wave][e][lane] = sum[e];
        __syncthreads();
        if (wave == 0) {
            for (int w = 1; w < kSumWaves; ++w)
#pragma unroll
                for (int e = 0; e < VE; ++e) sum[e] += head[w][e][lane];
            finish(ids[which], sum);
        }
        __syncthreads();
    }
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

template <int DT, int GT, int VE>
int sum_launch(SumArgs a, size_t wgs, hipStream_t s) {
    hipLaunchKernelGGL((k_embed_sum<DT, GT, VE>), dim3(static_cast<unsigned>(wgs)), dim3(kSumThreads), 0, s, a);
    return launch_status();
}

template <int DT, int GT>
int bwd(const int32_t *ids, const void *dy, float scale, void *dw, int accumulate, size_t tokens, size_t vocab,
        unsigned cols, cxm_stream_t st) {
    constexpr int VE = Elem<DT>::kVec;
    const bool narrow = cols < static_cast<unsigned>(VE);
    const unsigned ve = narrow ? 1 : VE, tiles = ceil_div(ceil_div(cols, ve), kWave);
    // ids per workgroup of the sort: one round of workgroups on the chip
    const size_t cus = device_cus();
    size_t range = (vocab + cus - 1) / cus;
    range = range < kSortIds ? range : kSortIds;
    const size_t sorters = (vocab + range - 1) / range;
    // a wave's places: enough waves to fill the chip, few enough that ids seldom meet in scratch
    size_t per = tokens * tiles / (cus * 16);
    per = per < 8 ? 8 : per > 128 ? 128 : per;
    const size_t spans = (tokens + per * kSumWaves - 1) / (per * kSumWaves);
    if (sorters > most_wgs(kSortThreads) || spans > most_wgs(kSumThreads) / tiles) return CXM_E_TOO_LARGE;
    const size_t o_starts = align256(tokens * sizeof(Place)), o_part = o_starts + align256((vocab + 1) * sizeof(unsigned));
    const size_t bytes = o_part + spans * 2 * tiles * kWave * ve * sizeof(float);
    Workspace ws;
    const int rc = get_workspace(st, (spans * tiles * kTicket + kCtr - 1) / kCtr, bytes, &ws);
    if (rc) return rc;
    char *base = static_cast<char *>(ws.scratch);
    const SortArgs so{ids,
                      tokens,
                      vocab,
                      static_cast<unsigned>(range),
                      reinterpret_cast<Place *>(base),
                      reinterpret_cast<unsigned *>(base + o_starts),
                      accumulate ? nullptr : static_cast<char *>(dw),
                      cols * sizeof(typename Elem<GT>::S)};
    hipLaunchKernelGGL(k_embed_sort, dim3(static_cast<unsigned>(sorters)), dim3(kSortThreads), 0, hs(st), so);
    int r = launch_status();
    if (r || tokens == 0) return r;
    const SumArgs sa{dy,    dw,   so.sorted, so.starts, reinterpret_cast<float *>(base + o_part), ws.counters, vocab, cols,
                     tiles, static_cast<unsigned>(per), scale, accumulate};
    return narrow ? sum_launch<DT, GT, 1>(sa, spans * tiles, hs(st)) : sum_launch<DT, GT, VE>(sa, spans * tiles, hs(st));
}

// Sizes that the kernels number in 32 bits, and whose bytes fit 64.
bool sizes_ok(size_t tokens, size_t vocab, size_t cols) {
    constexpr size_t k31 = size_t(1) << 31, k46 = size_t(1) << 46;
    return tokens < k31 && vocab < k31 && cols < k31 && tokens <= k46 / cols && vocab <= k46 / cols;
}

}  // namespace
}  // namespace cxm

extern "C" {

int cxm_embedding_fwd_t(const void *table, const int32_t *ids, float scale, void *y, size_t tokens, size_t vocab,
                        size_t cols, int dtype, cxm_stream_t s) {
    using cxm::overlap;
    if (!cxm::is_float_dtype(dtype) || !__builtin_isfinite(scale) || vocab == 0 || cols == 0) return CXM_E_INVALID;
    if (tokens == 0) return CXM_OK;
    if (!table || !ids || !y) return CXM_E_INVALID;
    if (!cxm::sizes_ok(tokens, vocab, cols)) return CXM_E_TOO_LARGE;
    const size_t e = cxm::dtype_bytes(dtype), n = tokens * cols * e;
    if (overlap(y, n, table, vocab * cols * e) || overlap(y, n, ids, tokens * 4)) return CXM_E_INVALID;
    const unsigned c = static_cast<unsigned>(cols);
    switch (dtype) {
        case CXM_DT_F32: return cxm::fwd_dispatch<CXM_DT_F32>(table, ids, scale, y, tokens, vocab, c, cxm::hs(s));
        case CXM_DT_BF16: return cxm::fwd_dispatch<CXM_DT_BF16>(table, ids, scale, y, tokens, vocab, c, cxm::hs(s));
        default: return cxm::fwd_dispatch<CXM_DT_F16>(table, ids, scale, y, tokens, vocab, c, cxm::hs(s));
    }
}

int cxm_embedding_bwd_t(const int32_t *ids, const void *dy, float scale, void *dw, int accumulate, size_t tokens,
                        size_t vocab, size_t cols, int dtype, int g_dtype, cxm_stream_t s) {
    using cxm::overlap;
    if (!cxm::is_float_dtype(dtype) || (g_dtype != dtype && g_dtype != CXM_DT_F32) || (accumulate != 0 && accumulate != 1) ||
        !__builtin_isfinite(scale) || vocab == 0 || cols == 0 || !dw || (tokens && (!ids || !dy)))
        return CXM_E_INVALID;
    if (!cxm::sizes_ok(tokens, vocab, cols)) return CXM_E_TOO_LARGE;
    const size_t n = vocab * cols * cxm::dtype_bytes(g_dtype);
    if (tokens && (overlap(dw, n, dy, tokens * cols * cxm::dtype_bytes(dtype)) || overlap(dw, n, ids, tokens * 4)))
        return CXM_E_INVALID;
    if (tokens == 0 && accumulate) return CXM_OK;
    const unsigned c = static_cast<unsigned>(cols);
    switch (dtype) {
        case CXM_DT_F32: return cxm::bwd<CXM_DT_F32, CXM_DT_F32>(ids, dy, scale, dw, accumulate, tokens, vocab, c, s);
        case CXM_DT_BF16:
            return g_dtype == dtype ? cxm::bwd<CXM_DT_BF16, CXM_DT_BF16>(ids, dy, scale, dw, accumulate, tokens, vocab, c, s)
                                    : cxm::bwd<CXM_DT_BF16, CXM_DT_F32>(ids, dy, scale, dw, accumulate, tokens, vocab, c, s);
        default:
            return g_dtype == dtype ? cxm::bwd<CXM_DT_F16, CXM_DT_F16>(ids, dy, scale, dw, accumulate, tokens, vocab, c, s)
                                    : cxm::bwd<CXM_DT_F16, CXM_DT_F32>(ids, dy, scale, dw, accumulate, tokens, vocab, c, s);
    }
}

}  // extern "C"
