// Rows of a table looked up by token and scaled, and the table's gradient.
//
//   y[t] = table[ids[t]] * scale
//   dw[v] = scale * sum over t with ids[t] == v of dy[t]  (+ dw[v])
//
// Both are bound by memory.  The gradient's tokens are sorted by id first, so
// that every row of dw is one sum in the order of the tokens (no atomics on
// floats: the same bits every time) and is written once.  Two launches:
//  * k_embed_sort: a workgroup owns every 2^n-th id.  It reads all ids twice
//    (they lie in L2), counts those of the owners before it, which says where its
//    part of the sorted list begins, and places its own in order; the rows
//    that no token has become zero in the same launch.
//  * k_embed_sum: a wave takes up to 16 neighbours of the sorted list and a tile
//    of columns, and writes the rows of ids that lie within its part; what an
//    id's tokens give in several waves meets in LDS, in several workgroups in
//    scratch, added up by the last of them to arrive, in the list's order.
// 32768 tokens of 2048 bf16 into 65536 rows: 48 us with 216 MB of zeros, and 46 us of
// sums, whose rows are read at random (3.9 TB/s with what they write); accumulating,
// without the zeros, 71 us in all.
#include "chunk.hpp"

namespace cxm {
namespace {

inline hipStream_t hs(cxm_stream_t s) { return reinterpret_cast<hipStream_t>(s); }

// Workgroup b of a grid goes to XCD b mod 8.  The pieces of a row that is not whole
// lines share lines, which then meet in several L2s: number the workgroups so
// that an XCD's take neighbouring pieces (20001 rows of 1003 floats looked up in
// 30.7 us instead of 33.4; whole lines 42.5 and 41.3).
struct Spread {
    unsigned n, xcds, each;  // pieces, XCDs, pieces of an XCD
    __device__ unsigned piece() const { return blockIdx.x % xcds * each + blockIdx.x / xcds; }  // n or more: none
};
// The grid is xcds * each workgroups.
Spread spread_of(unsigned n) {
    DevLayout l{0, 1};
    const unsigned xcds = device_layout(&l) == CXM_OK && l.xccs > 0 ? static_cast<unsigned>(l.xccs) : 1;
    return {n, xcds, (n + xcds - 1) / xcds};
}

// ---------------------------------------------------------------- forward

// G lanes per row piece of G chunks, U tokens per group of lanes.  Stores carry the
// non-temporal hint (20001 rows of 1003 floats 30.7 -> 22.7 us, 32768 of 2048 bf16
// 42.4 -> 31.5).  The gradient's rows are stored without it: 32768x2048 bf16 took 92
// with it where 94 without into memory that is not in the cache, but 92 for 80 where it is.
template <int DT, int VE, int G, int U>
__global__ __launch_bounds__(kBlock) void k_embed(const typename Elem<DT>::S *table, const int32_t *ids, float scale,
                                                  typename Elem<DT>::S *y, size_t tokens, size_t vocab, unsigned cols,
                                                  unsigned tiles, Spread spread) {
    constexpr int R = kBlock / G;
    const unsigned piece = spread.piece();
    if (piece >= spread.n) return;
    const size_t blk = piece / tiles;
    const unsigned tile = piece - static_cast<unsigned>(blk) * tiles;
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
        store_span<DT, VE, true>(y + (first + u) * cols, s, c[u]);
    }
}

template <int DT, int VE, int G, int U>
int fwd_launch(const void *table, const int32_t *ids, float scale, void *y, size_t tokens, size_t vocab, unsigned cols,
               hipStream_t s) {
    using S = typename Elem<DT>::S;
    const unsigned tiles = ceil_div(ceil_div(cols, VE), G);
    const size_t blks = (tokens + static_cast<size_t>(kBlock / G) * U - 1) / (static_cast<size_t>(kBlock / G) * U);
    if (blks > (most_wgs(kBlock) - kCtr) / tiles) return CXM_E_TOO_LARGE;  // (fewer than 64 XCDs round the grid up)
    const Spread spread = spread_of(static_cast<unsigned>(blks * tiles));
    hipLaunchKernelGGL((k_embed<DT, VE, G, U>), dim3(spread.xcds * spread.each), dim3(kBlock), 0, s,
                       static_cast<const S *>(table), ids, scale, static_cast<S *>(y), tokens, vocab, cols, tiles, spread);
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
constexpr unsigned kSortIds = 256;  // most ids of a workgroup
constexpr unsigned kPending = 256 + kWave;  // tokens that a wave holds back until it has 64
constexpr int kSortAhead = 4;       // groups of 256 ids in flight
typedef int i32x4e __attribute__((ext_vector_type(4), aligned(4)));

// The sorted list's order: owner by owner (the id's low `bits` bits), an
// owner's ids in turn.  The ids that a text uses most are neighbours (small, as
// a rule), and so have an owner each.
struct Order {
    unsigned bits, range;  // 2^bits owners of at most `range` ids
    __host__ __device__ unsigned number(unsigned id) const { return (id & ((1u << bits) - 1)) * range + (id >> bits); }
};

struct SortArgs {
    const int32_t *ids;
    size_t tokens;
    unsigned vocab;
    Order order;
    Place *sorted;     // [tokens]
    unsigned *starts;  // [owners * range + 1]: where each id's tokens begin
    char *dw;          // null: accumulating, nothing becomes zero
    size_t row_bytes;
};

// Zeros over a row of n bytes at 2-byte alignment, by one wave.
__device__ __forceinline__ void zero_row(char *p, size_t n, unsigned lane) {
    const size_t whole = n / 16;
    for (size_t i = lane; i < whole; i += kWave) *reinterpret_cast<u32x4e *>(p + i * 16) = u32x4e{0, 0, 0, 0};
    const size_t at = whole * 16 + lane * 2;
    if (at < n) *reinterpret_cast<uint16_t *>(p + at) = 0;
}

// Half of the waves write the zeros of absent ids while the other half place the
// tokens; without zeros all of them place (the zeros between the sums, in their
// launch, took 111 us instead of 94: 32768 tokens of 2048 bf16, 65536 ids).
__global__ __launch_bounds__(kSortThreads) void k_embed_sort(SortArgs a) {
    __shared__ unsigned hist[kSortWaves * kSortIds];  // [wave][id]
    __shared__ unsigned wsum[kSortWaves], below_all;
    __shared__ unsigned long long absent[kSortIds / kWave];  // a bit for each id that no token has
    __shared__ Place pending[kSortWaves][kPending];
    const unsigned lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const unsigned owner = blockIdx.x, mask = (1u << a.order.bits) - 1, shift = a.order.bits, cap = a.order.range;
    const unsigned range = owner < a.vocab ? ((a.vocab - owner - 1) >> shift) + 1 : 0;  // its ids: owner, owner + owners, ...
    // a wave's tokens, in a row: whole groups of 4 for all lanes but the last ones
    const size_t per = (a.tokens + 4 * kSortThreads - 1) / (4 * kSortThreads) * 4 * kWave;
    for (unsigned i = threadIdx.x; i < kSortWaves * cap; i += kSortThreads) hist[i] = 0;
    if (threadIdx.x == 0) below_all = 0;
    __syncthreads();
    // four ids a lane, -1 (no id) past a wave's part
    auto batch = [&](size_t at, size_t end, int(&id)[kSortAhead][4]) {
#pragma unroll
        for (int k = 0; k < kSortAhead; ++k) {
            const size_t i = at + (k * kWave + lane) * 4;
            if (i + 4 <= end) {
                const i32x4e v = *reinterpret_cast<const i32x4e *>(a.ids + i);
                id[k][0] = v.x; id[k][1] = v.y; id[k][2] = v.z; id[k][3] = v.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) id[k][j] = i + j < end ? a.ids[i + j] : -1;
            }
        }
    };
    auto end_of = [&](size_t from) { return from + per < a.tokens ? from + per : a.tokens; };
    // an id's owner (of no id: none)
    auto owner_of = [&](int id) { return static_cast<unsigned>(id) < a.vocab ? static_cast<unsigned>(id) & mask : ~0u; };
    unsigned below = 0;
    for (size_t t0 = wave * per, t1 = end_of(t0), at = t0; at < t1; at += kSortAhead * kWave * 4) {
        int id[kSortAhead][4];
        batch(at, t1, id);
#pragma unroll
        for (int k = 0; k < kSortAhead; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned o = owner_of(id[k][j]);
                below += o < owner;
                const bool mine = o == owner;
                const unsigned long long in = __ballot(mine);
                if (in == 0) continue;
                const unsigned key = static_cast<unsigned>(id[k][j]) >> shift;
                if (__popcll(in) < 24) {
                    if (mine) atomicAdd(&hist[wave * cap + key], 1u);
                } else {  // those of the first one's id together: a text that is mostly one id would queue up here
                    const unsigned one = readlane(static_cast<int>(key), __builtin_ctzll(in));
                    const unsigned long long same = __ballot(mine && key == one);
                    if (mine && key != one) atomicAdd(&hist[wave * cap + key], 1u);
                    if (lane == __builtin_ctzll(same)) atomicAdd(&hist[wave * cap + one], static_cast<unsigned>(__popcll(same)));
                }
            }
    }
    for (int d = 1; d < kWave; d *= 2) below += __shfl_xor(below, d);
    if (lane == 0) atomicAdd(&below_all, below);
    __syncthreads();
    // where each wave's tokens of each id go: ids in turn, within one the waves in turn
    const unsigned r = threadIdx.x;
    unsigned total = 0;
    if (r < range) {
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) total += hist[w * cap + r];
    }
    unsigned incl = total;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const unsigned o = __shfl_up(incl, d);
        if (lane >= static_cast<unsigned>(d)) incl += o;
    }
    if (lane == kWave - 1) wsum[wave] = incl;
    const unsigned long long none = __ballot(r < range && total == 0);
    if (lane == 0 && wave < kSortIds / kWave) absent[wave] = none;
    __syncthreads();
    unsigned at = below_all + incl - total;
    for (unsigned w = 0; w < wave; ++w) at += wsum[w];
    if (r < cap) {  // (past its last id: where the next owner's begin)
        a.starts[owner * cap + r] = at;
        if (owner == mask && r + 1 == cap) a.starts[owner * cap + cap] = at + total;
    }
    if (r < range) {
        for (int w = 0; w < kSortWaves; ++w) {
            const unsigned n = hist[w * cap + r];
            hist[w * cap + r] = at;
            at += n;
        }
    }
    __syncthreads();
    const unsigned placers = a.dw ? kSortWaves / 2 : kSortWaves;
    if (wave >= placers) {
        for (unsigned i = wave - placers; i < range; i += kSortWaves - placers)
            if (absent[i / kWave] >> (i % kWave) & 1)
                zero_row(a.dw + (owner + (static_cast<size_t>(i) << shift)) * a.row_bytes, a.row_bytes, lane);
        return;
    }
    // A wave's own tokens are first put together, in order, and placed 64 at a time: the owner of a text's
    // most frequent ids has them in every group (placed group by group, one id after the other, the gradient of
    // 131072 tokens took 133 us, so 100).
    const unsigned parts = kSortWaves / placers;
    Place *held = pending[wave];
    const int key_bits = 32 - __clz((cap - 1) | 1);
    for (unsigned w = wave * parts; w < (wave + 1) * parts; ++w) {
        unsigned have = 0;
        auto place = [&](unsigned at, unsigned n) {  // held[at .. at + n), n <= 64
            const Place mine = held[at + (lane < n ? lane : 0)];
            const unsigned key = static_cast<unsigned>(mine.id) >> shift;
            unsigned long long same = __ballot(lane < n);
            if (__any(key != static_cast<unsigned>(readlane(static_cast<int>(key), 0)))) {
                for (int b = 0; b < key_bits; ++b) {  // the lanes that have this lane's id
                    const unsigned long long one = __ballot(key >> b & 1);
                    same &= key >> b & 1 ? one : ~one;
                }
            }
            const unsigned rank = __popcll(same & ((1ull << lane) - 1)), to = hist[w * cap + key];
            // every lane has read the place before it moves on, and the next reader sees it moved
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (lane < n) {
                a.sorted[to + rank] = mine;
                if (rank == 0) hist[w * cap + key] = to + __popcll(same);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        };
        for (size_t t0 = w * per, t1 = end_of(t0), base = t0; base < t1; base += kSortAhead * kWave * 4) {
            int id[kSortAhead][4];
            batch(base, t1, id);
#pragma unroll
            for (int k = 0; k < kSortAhead; ++k) {
                unsigned long long in[4], any = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) any |= in[j] = __ballot(owner_of(id[k][j]) == owner);
                if (!any) continue;
                unsigned rank = have, more = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    rank += __popcll(in[j] & ((1ull << lane) - 1));
                    more += __popcll(in[j]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (in[j] >> lane & 1) held[rank++] = Place{id[k][j], static_cast<int>(base + (k * kWave + lane) * 4 + j)};
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                have += more;
                if (have < kWave) continue;
                unsigned at = 0;
                for (; have - at >= kWave; at += kWave) place(at, kWave);
                have -= at;
                const Place rest = held[at + (lane < have ? lane : 0)];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                if (lane < have) held[lane] = rest;
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
        }
        if (have) place(0, have);
    }
}

constexpr int kSumThreads = 512, kSumWaves = kSumThreads / kWave;
constexpr int kPlaces = 16;     // most places of a wave, all of their rows in flight
constexpr size_t kTicket = 16;  // words between two of its tickets

struct SumArgs {
    const void *dy;
    void *dw;
    const Place *sorted;
    const unsigned *starts;
    float *part;        // [spans][2][tiles * 64 * VE]: what an id's tokens give in a span, of the id that
                        // began before it and of the one that goes on after it
    unsigned *tickets;  // [spans * tiles], kTicket apart
    Order order;
    unsigned ends;  // owners * range: starts[ends] places are in the list
    unsigned tokens, cols, tiles, per;  // per: a wave's places
    float scale;
    int accumulate;
    Spread spread;
};

template <int DT, int GT, int VE>
__global__ __launch_bounds__(kSumThreads) void k_embed_sum(SumArgs a) {
    using S = typename Elem<DT>::S;
    using SG = typename Elem<GT>::S;
    __shared__ float head[kSumWaves][VE][kWave], tail[kSumWaves][VE][kWave];
    // of each wave: 1 its first id began before it, 2 that id also goes on after it, 4 its last id began in it and goes on
    __shared__ int kind[kSumWaves];
    __shared__ int first_id[kSumWaves], last_id[kSumWaves], flag;
    const unsigned lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const unsigned piece = a.spread.piece();
    if (piece >= a.spread.n) return;
    const unsigned span = piece / a.tiles, tile = piece - span * a.tiles;
    const unsigned places = kSumWaves * a.per, from = span * places, begin = from + wave * a.per;
    // the wave's places, with one before them (lane 0) and one behind
    const unsigned p = begin + lane - 1;
    const Place mine = a.sorted[p < a.tokens ? p : 0];
    const unsigned all = a.starts[a.ends];
    if (from >= all) return;
    const unsigned p0 = begin < all ? begin : all, p1 = p0 + a.per < all ? p0 + a.per : all, n = p1 - p0;
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
            // (reading a wave's rows of dw with its rows of dy took no less time, in half as many waves)
            if (a.accumulate) c.load(row + s.off + h * VG);
#pragma unroll
            for (int e = 0; e < VG; ++e) t[e] = a.accumulate ? c.get(e) + v[h * VG + e] : v[h * VG + e];
            c.set(t);
            const unsigned dup = s.dup > static_cast<unsigned>(h * VG) ? s.dup - h * VG : 0;
            store_span<GT, VG>(row, Span{s.off + h * VG, dup}, c);
        }
    };
    int k = 0, cur = -1;
    if (n) {
        Chunk<DT, VE> c[kPlaces];
        // all row numbers before the first branch: after one the compiler waits for every load in flight before
        // it reads the places again (32768 tokens of 2048 bf16 took 70 us instead of 43)
        unsigned row[kPlaces];
        int ids[kPlaces];
#pragma unroll
        for (int u = 0; u < kPlaces; ++u) {
            row[u] = static_cast<unsigned>(readlane(mine.token, u + 1));
            ids[u] = readlane(mine.id, u + 1);
        }
#pragma unroll
        for (int u = 0; u < kPlaces; ++u)
            if (u < static_cast<int>(n)) c[u].load_nt(dy + static_cast<size_t>(row[u]) * a.cols);
        float acc[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[e] = 0.0f;
        cur = readlane(mine.id, 1);
        if (lane == 0) first_id[wave] = cur;
        bool began = p0 == 0 || readlane(mine.id, 0) != cur;  // whether the id being added up began in this wave
#pragma unroll
        for (int u = 0; u < kPlaces; ++u) {
            if (u >= static_cast<int>(n)) continue;
            const int id = ids[u];
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
        const bool ends = p1 >= all || readlane(mine.id, n + 1) != cur;
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
    // An id in several workgroups: the last of them to have stored its part adds them up.  (0: it began before
    // this workgroup; 1: it began here and goes on.)
    const int last_wave = static_cast<int>(((from + places < all ? from + places : all) - from - 1) / a.per);
    int w0 = last_wave;  // where the last id began
    while (w0 >= 0 && (kind[w0] & 2)) --w0;
    const bool before = kind[0] & 1, after = w0 >= 0 && (kind[w0] & 4);
    for (int which = 0; which < 2; ++which) {
        if (!(which == 0 ? before : after)) continue;
        const int id = which == 0 ? first_id[0] : last_id[last_wave];
        const unsigned q = a.order.number(static_cast<unsigned>(id));
        const unsigned s0 = a.starts[q], s1 = a.starts[q + 1];
        const unsigned g0 = s0 / places, count = (s1 - 1) / places - g0 + 1;
        const bool last = last_block_ticket(a.tickets + (static_cast<size_t>(g0) * a.tiles + tile) * kTicket, count, &flag);
        if (!last) continue;
        // each wave a run of the parts, one after the other
        const unsigned each = (count + kSumWaves - 1) / kSumWaves;
        const unsigned c0 = wave * each < count ? wave * each : count, c1 = c0 + each < count ? c0 + each : count;
        float sum[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) sum[e] = 0.0f;
        constexpr int U = 8;
        for (unsigned c = c0; c < c1; c += U) {
            float v[U][VE];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const unsigned cc = c + u < c1 ? c + u : c;
                const float *at = a.part + (static_cast<size_t>(g0 + cc) * 2 + (cc == 0 ? 1 : 0)) * width +
                                  static_cast<size_t>(tile) * kWave * VE + lane;
#pragma unroll
                for (int e = 0; e < VE; ++e) v[u][e] = ld_dev(at + e * kWave);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (c + u >= c1) continue;
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
            finish(id, sum);
        }
        __syncthreads();
    }
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

template <int DT, int GT, int VE>
int sum_launch(const SumArgs &a, hipStream_t s) {
    hipLaunchKernelGGL((k_embed_sum<DT, GT, VE>), dim3(a.spread.xcds * a.spread.each), dim3(kSumThreads), 0, s, a);
    return launch_status();
}

template <int DT, int GT>
int bwd(const int32_t *ids, const void *dy, float scale, void *dw, int accumulate, size_t tokens, size_t vocab,
        unsigned cols, cxm_stream_t st) {
    constexpr int VE = Elem<DT>::kVec;
    const bool narrow = cols < static_cast<unsigned>(VE);
    const unsigned ve = narrow ? 1 : VE, tiles = ceil_div(ceil_div(cols, ve), kWave);
    // owners: a power of two of them, one round of workgroups on the chip unless each would have too many ids
    const size_t cus = device_cus();
    Order order{0, 0};
    while ((size_t(2) << order.bits) <= vocab &&
           ((size_t(2) << order.bits) <= cus || (vocab + (size_t(1) << order.bits) - 1) >> order.bits > kSortIds))
        ++order.bits;
    const size_t owners = size_t(1) << order.bits;
    order.range = static_cast<unsigned>((vocab + owners - 1) >> order.bits);
    // a wave's places: as many as are in flight at once, fewer where that leaves CUs without work
    size_t per = kPlaces;
    while (per > 4 && tokens * tiles < per * kSumWaves * cus) per /= 2;
    const size_t spans = (tokens + per * kSumWaves - 1) / (per * kSumWaves);
    if (owners > most_wgs(kSortThreads) || spans > (most_wgs(kSumThreads) - kCtr) / tiles) return CXM_E_TOO_LARGE;
    const size_t ends = owners * order.range;
    const size_t o_starts = align256(tokens * sizeof(Place)), o_part = o_starts + align256((ends + 1) * sizeof(unsigned));
    const size_t bytes = o_part + spans * 2 * tiles * kWave * ve * sizeof(float);
    Workspace ws;
    const int rc = get_workspace(st, (spans * tiles * kTicket + kCtr - 1) / kCtr, bytes, &ws);
    if (rc) return rc;
    char *base = static_cast<char *>(ws.scratch);
    const SortArgs so{ids,
                      tokens,
                      static_cast<unsigned>(vocab),
                      order,
                      reinterpret_cast<Place *>(base),
                      reinterpret_cast<unsigned *>(base + o_starts),
                      accumulate ? nullptr : static_cast<char *>(dw),
                      cols * sizeof(typename Elem<GT>::S)};
    hipLaunchKernelGGL(k_embed_sort, dim3(static_cast<unsigned>(owners)), dim3(kSortThreads), 0, hs(st), so);
    int r = launch_status();
    if (r || tokens == 0) return r;
    const SumArgs sa{dy,
                     dw,
                     so.sorted,
                     so.starts,
                     reinterpret_cast<float *>(base + o_part),
                     ws.counters,
                     order,
                     static_cast<unsigned>(ends),
                     static_cast<unsigned>(tokens),
                     cols,
                     tiles,
                     static_cast<unsigned>(per),
                     scale,
                     accumulate,
                     spread_of(static_cast<unsigned>(spans * tiles))};
    return narrow ? sum_launch<DT, GT, 1>(sa, hs(st)) : sum_launch<DT, GT, VE>(sa, hs(st));
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
