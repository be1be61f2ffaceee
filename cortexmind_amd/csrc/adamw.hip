// One AdamW step over all tensors of a model in one launch, with the moments
// in fp32 or in 8 bits.  Stands beside cxm_sgd_f32.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2      (g times the factor)
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound by memory (each value read and written once).  The tensors are cut
// into pieces of kPiece values, a workgroup each; a table on the device, made
// once per optimizer, says which piece belongs to which tensor.
//
// 8-bit moments: m and r = sqrt(v) (the root halves the range that e4m3's 18
// octaves have to cover) as e4m3 with an fp32 scale per kBlock8 values, the
// largest magnitude / 448.  Rounding is stochastic: to the upper neighbour
// with the probability of the distance to the lower one, so the expected
// stored value is the exact one.  Rounded to nearest, an average whose step
// changes it by 1 - b2 = 0.1% would never leave a value (half a step is 3 to
// 6%).  A root above zero is never stored as zero, which would divide a
// moment by eps alone.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>
#include <new>
#include <type_traits>
#include <vector>

#include "chunk.hpp"

struct cxm_adamw;

namespace cxm {
namespace {

typedef unsigned u32x2a __attribute__((ext_vector_type(2)));

constexpr unsigned kBlock8 = 256;                   // values per scale: 64 lanes of 4
constexpr unsigned kLane = 4, kUnits = 2;           // values of a thread: kUnits times kLane, a wave's lanes side by side
constexpr unsigned kPiece = kBlock * kLane * kUnits;  // values per workgroup

struct AdamTensor {
    void *p;
    const void *g;
    float *w;  // fp32 master or null
    void *m, *v;
    float *ms, *vs;
    size_t n;
    unsigned long long first;  // the number of its value 0, for the random bits
    unsigned piece0;           // its first piece
    float decay;
    int vec;  // every pointer 16-byte aligned (8-bit moments: 8)
};

struct AdamStep {
    const AdamTensor *tensors;
    const unsigned *owner;  // piece -> tensor
    const float *scalars;   // null, or {lr, step, factor} on the device
    double lr;
    float c1, c2;           // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
    float log_b1, log_b2;
    float b1, b1c, b2, b2c, eps;
    unsigned key;
};

// 32 random bits of value number c: two multiply-and-shift rounds.
__device__ __forceinline__ unsigned noise32(unsigned long long c, unsigned key) {
    unsigned x = static_cast<unsigned>(c) ^ key ^ (static_cast<unsigned>(c >> 32) * 0xC2B2AE35u);
    x ^= x >> 16;
    x *= 0x85EBCA6Bu;
    x ^= x >> 16;
    x *= 0xC2B2AE35u;
    return x ^ (x >> 16);
}

// Byte SEL of `w` becomes v (|v| up to 448) as e4m3, its magnitude rounded to
// the neighbour above with the probability of the distance to the one below:
// v_cvt_sr_fp8_f32 adds the upper 20 bits of `rnd` below the 3 kept mantissa
// bits and cuts the rest off (below 2^-6 below the even steps of 2^-9).  Its
// last 4 bits are zero, so a block's largest value, 448 but for an fp32
// rounding of the scale or two, never carries past 448 into the NaN.
template <int SEL>
__device__ __forceinline__ unsigned round_e4m3(float v, unsigned rnd, unsigned w) {
    return static_cast<unsigned>(__builtin_amdgcn_cvt_sr_fp8_f32(v, static_cast<int>(rnd), static_cast<int>(w), SEL));
}
// The largest of |v| that is finite, over the wave (a block).
__device__ __forceinline__ float block_amax(const float (&v)[kLane]) {
    float m = 0.0f;
#pragma unroll
    for (unsigned e = 0; e < kLane; ++e) m = fmaxf(m, fabsf(v[e]));  // a NaN is passed over
    m = group_reduce<MaxOp, kWave>(m);
    if (__builtin_expect(m > FLT_MAX, 0)) {  // the same in every lane
        m = 0.0f;
#pragma unroll
        for (unsigned e = 0; e < kLane; ++e) m = fabsf(v[e]) <= FLT_MAX ? fmaxf(m, fabsf(v[e])) : m;
        m = group_reduce<MaxOp, kWave>(m);
    }
    return m;
}

// Four elements of a type in registers, whole or one by one.
template <int DT>
struct Quad {
    float v[kLane];
    __device__ __forceinline__ void load(const typename Elem<DT>::S *p) {
        if constexpr (DT == CXM_DT_F32) {
            const float4 x = ld4_stream(p);
            v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
        } else {
            const u32x2a x = __builtin_nontemporal_load(reinterpret_cast<const u32x2a *>(p));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = H<DT>::load(static_cast<uint16_t>(x[e / 2] >> (16 * (e & 1))));
        }
    }
    __device__ __forceinline__ void store(typename Elem<DT>::S *p) const {
        if constexpr (DT == CXM_DT_F32) st4_stream(p, make_float4(v[0], v[1], v[2], v[3]));
        else
            __builtin_nontemporal_store(u32x2a{pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3])},
                                        reinterpret_cast<u32x2a *>(p));
    }
};

template <int PD, int GD, bool MASTER, bool Q8>
__global__ __launch_bounds__(kBlock) void k_adamw(AdamStep a) {
    using PS = typename Elem<PD>::S;
    using GS = typename Elem<GD>::S;
    const AdamTensor t = a.tensors[a.owner[blockIdx.x]];
    PS *p = static_cast<PS *>(t.p);
    const GS *g = static_cast<const GS *>(t.g);
    auto *m8 = static_cast<uint8_t *>(t.m), *v8 = static_cast<uint8_t *>(t.v);
    auto *m32 = static_cast<float *>(t.m), *v32 = static_cast<float *>(t.v);
    const unsigned lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
    const size_t i00 = static_cast<size_t>(blockIdx.x - t.piece0) * kPiece + w * (kBlock8 * kUnits) + lane * kLane;

    Quad<CXM_DT_F32> m[kUnits], v[kUnits], wt[kUnits];
    Quad<GD> gr[kUnits];
    Quad<PD> pp[kUnits];
    unsigned qm[kUnits], qv[kUnits];
    float sm[kUnits], sv[kUnits];
    bool whole[kUnits];
    size_t blk[kUnits];
    const size_t blocks = (t.n + kBlock8 - 1) / kBlock8;
#pragma unroll
    for (unsigned u = 0; u < kUnits; ++u) {
        const size_t i = i00 + u * kBlock8;
        whole[u] = t.vec && i + kLane <= t.n;
        blk[u] = i / kBlock8;
        if constexpr (Q8) {  // a wave past the end takes the last block's scales and stores nothing
            const size_t b = blk[u] < blocks ? blk[u] : blocks - 1;
            sm[u] = t.ms[b];
            sv[u] = t.vs[b];
        }
        if (whole[u]) {
            if constexpr (MASTER) wt[u].load(t.w + i);
            else pp[u].load(p + i);
            gr[u].load(g + i);
            if constexpr (Q8) {
                qm[u] = __builtin_nontemporal_load(reinterpret_cast<const unsigned *>(m8 + i));
                qv[u] = __builtin_nontemporal_load(reinterpret_cast<const unsigned *>(v8 + i));
            } else {
                m[u].load(m32 + i);
                v[u].load(v32 + i);
            }
        } else {
            qm[u] = qv[u] = 0;
#pragma unroll
            for (unsigned e = 0; e < kLane; ++e) {
                const bool in = i + e < t.n;
                wt[u].v[e] = MASTER && in ? t.w[i + e] : 0.0f;
                pp[u].v[e] = !MASTER && in ? Elem<PD>::load(p[i + e]) : 0.0f;
                gr[u].v[e] = in ? Elem<GD>::load(g[i + e]) : 0.0f;
                if constexpr (Q8) {
                    qm[u] |= (in ? static_cast<unsigned>(m8[i + e]) : 0u) << (8 * e);
                    qv[u] |= (in ? static_cast<unsigned>(v8[i + e]) : 0u) << (8 * e);
                } else {
                    m[u].v[e] = in ? m32[i + e] : 0.0f;
                    v[u].v[e] = in ? v32[i + e] : 0.0f;
                }
            }
        }
    }

    // the step's factors, from the host in 64 bits, or from the device's
    // scalars: 1 - b^t as -expm1(t log b), which loses no digits in 32 bits
    // at small t (1 - powf would)
    double lr = a.lr;
    float c1 = a.c1, c2 = a.c2, factor = 1.0f;
    if (a.scalars) {
        const float l = a.scalars[0], step = a.scalars[1];
        lr = l;
        c1 = -l / expm1f(step * a.log_b1);
        c2 = 1.0f / __builtin_sqrtf(-expm1f(step * a.log_b2));
        factor = a.scalars[2];
    }
    const float keep = static_cast<float>(1.0 - lr * static_cast<double>(t.decay));

#pragma unroll
    for (unsigned u = 0; u < kUnits; ++u) {
        const size_t i = i00 + u * kBlock8;
        if constexpr (Q8) {
            unpack_e4m3(qm[u], m[u].v);
            unpack_e4m3(qv[u], v[u].v);
        }
        float pn[kLane];
#pragma unroll
        for (unsigned e = 0; e < kLane; ++e) {
            const float gv = a.scalars ? gr[u].v[e] * factor : gr[u].v[e];
            float m0 = m[u].v[e], v0 = v[u].v[e];
            if constexpr (Q8) {
                m0 *= sm[u];
                v0 *= sv[u];
                v0 *= v0;
            }
            const float m1 = a.b1 * m0, m2 = a.b1c * gv, gg = gv * gv, v1 = a.b2 * v0, v2 = a.b2c * gg;
            const float mn = m1 + m2, vn = v1 + v2, r = __builtin_sqrtf(vn);
            const float d = r * c2 + a.eps, q = (MASTER ? wt[u].v[e] : pp[u].v[e]) * keep;
            // the quotient by the reciprocal estimate (1 ulp) of a normal divisor: its
            // error is 2^-23 of an update that is itself a small part of p
            const float up = c1 * mn * (d >= FLT_MIN ? __builtin_amdgcn_rcpf(d) : 1.0f / d);
            pn[e] = q - up;
            m[u].v[e] = mn;
            v[u].v[e] = Q8 ? r : vn;
        }
        if constexpr (Q8) {
            const Scale8 km = scale_e4m3(block_amax(m[u].v)), kv = scale_e4m3(block_amax(v[u].v));
            if (lane == 0 && blk[u] < blocks) {
                t.ms[blk[u]] = km.scale;
                t.vs[blk[u]] = kv.scale;
            }
            // NaN and infinity are stored as NaN, where they are alone
            auto put = [&](auto sel) {
                constexpr int S = decltype(sel)::value;
                const unsigned bits = noise32(t.first + i + S, a.key);
                const float x = m[u].v[S] * km.inv, y = v[u].v[S] * kv.inv;
                // a root above zero that would be 0 or 2^-9 is 2^-9
                const float yy = y > 0.0f && y < 0x1p-9f ? 0x1p-9f : y;
                qm[u] = round_e4m3<S>(fabsf(m[u].v[S]) <= FLT_MAX ? x : __builtin_nanf(""), bits << 16, qm[u]);
                qv[u] = round_e4m3<S>(v[u].v[S] <= FLT_MAX ? yy : __builtin_nanf(""), bits & 0xFFFF0000u, qv[u]);
            };
            put(std::integral_constant<int, 0>{});
            put(std::integral_constant<int, 1>{});
            put(std::integral_constant<int, 2>{});
            put(std::integral_constant<int, 3>{});
        }
#pragma unroll
        for (unsigned e = 0; e < kLane; ++e) wt[u].v[e] = pp[u].v[e] = pn[e];
        if (whole[u]) {
            if constexpr (MASTER) wt[u].store(t.w + i);
            pp[u].store(p + i);
            if constexpr (Q8) {
                __builtin_nontemporal_store(qm[u], reinterpret_cast<unsigned *>(m8 + i));
                __builtin_nontemporal_store(qv[u], reinterpret_cast<unsigned *>(v8 + i));
            } else {
                m[u].store(m32 + i);
                v[u].store(v32 + i);
            }
        } else {
#pragma unroll
            for (unsigned e = 0; e < kLane; ++e) {
                if (i + e >= t.n) break;
                if constexpr (MASTER) t.w[i + e] = pn[e];
                p[i + e] = Elem<PD>::store(pn[e]);
                if constexpr (Q8) {
                    m8[i + e] = static_cast<uint8_t>(qm[u] >> (8 * e));
                    v8[i + e] = static_cast<uint8_t>(qv[u] >> (8 * e));
                } else {
                    m32[i + e] = m[u].v[e];
                    v32[i + e] = v[u].v[e];
                }
            }
        }
    }
}

inline int hip_status(hipError_t e) { return e == hipSuccess ? CXM_OK : static_cast<int>(e); }

}  // namespace
}  // namespace cxm

struct cxm_adamw {
    cxm::AdamTensor *tensors = nullptr;  // device
    unsigned *owner = nullptr;           // device
    unsigned pieces = 0;
    int device = 0, p_dtype = 0, g_dtype = 0;
    bool master = false, q8 = false;
};

namespace {

using namespace cxm;

template <int PD, int GD, bool MASTER>
void adam_launch(const cxm_adamw &h, const AdamStep &a, hipStream_t s) {
    if (h.q8) hipLaunchKernelGGL((k_adamw<PD, GD, MASTER, true>), dim3(h.pieces), dim3(kBlock), 0, s, a);
    else hipLaunchKernelGGL((k_adamw<PD, GD, MASTER, false>), dim3(h.pieces), dim3(kBlock), 0, s, a);
}
template <int PD>
void adam_launch16(const cxm_adamw &h, const AdamStep &a, hipStream_t s) {
    if (h.g_dtype == CXM_DT_F32) {
        if (h.master) adam_launch<PD, CXM_DT_F32, true>(h, a, s);
        else adam_launch<PD, CXM_DT_F32, false>(h, a, s);
    } else {
        if (h.master) adam_launch<PD, PD, true>(h, a, s);
        else adam_launch<PD, PD, false>(h, a, s);
    }
}

struct Range {
    uintptr_t at;
    size_t n;
    bool written;
};

int adam_create(cxm_adamw **out, const cxm_adamw_tensor_t *tensors, size_t count, int p_dtype, int g_dtype,
                int state_dtype) {
    const bool q8 = state_dtype == CXM_DT_E4M3;
    const size_t pb = dtype_bytes(p_dtype), gb = dtype_bytes(g_dtype), sb = q8 ? 1 : 4;
    std::vector<AdamTensor> table;
    std::vector<unsigned> owner;
    std::vector<Range> ranges;
    unsigned long long first = 0;
    bool master = false, seen = false;
    for (size_t i = 0; i < count; ++i) {
        const cxm_adamw_tensor_t &t = tensors[i];
        if (t.n == 0) continue;
        if (t.n > (size_t(1) << 46)) return CXM_E_TOO_LARGE;
        if (!t.p || !t.g || !t.m || !t.v || (q8 && (!t.m_scale || !t.v_scale)) || !(t.decay >= 0.0f && t.decay <= FLT_MAX))
            return CXM_E_INVALID;
        if (seen && master != (t.master != nullptr)) return CXM_E_INVALID;  // masters: all tensors or none
        seen = true;
        master = t.master != nullptr;
        if (master && p_dtype == CXM_DT_F32) return CXM_E_INVALID;
        const size_t blocks = (t.n + kBlock8 - 1) / kBlock8, pieces = (t.n + kPiece - 1) / kPiece;
        if (owner.size() + pieces > most_wgs(kBlock)) return CXM_E_TOO_LARGE;
        AdamTensor d{};
        d.p = t.p;
        d.g = t.g;
        d.w = t.master;
        d.m = t.m;
        d.v = t.v;
        d.ms = q8 ? t.m_scale : nullptr;
        d.vs = q8 ? t.v_scale : nullptr;
        d.n = t.n;
        d.first = first;
        d.piece0 = static_cast<unsigned>(owner.size());
        d.decay = t.decay;
        d.vec = aligned16(t.p) && aligned16(t.g) && (!master || aligned16(t.master)) &&
                (q8 ? (reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.v)) % 8 == 0
                    : aligned16(t.m) && aligned16(t.v));
        first += static_cast<unsigned long long>(blocks) * kBlock8;
        owner.insert(owner.end(), pieces, static_cast<unsigned>(table.size()));
        table.push_back(d);
        const struct {
            const void *at;
            size_t n;
            bool written;
        } r[] = {{t.p, t.n * pb, true},          {t.g, t.n * gb, false},
                 {t.master, master ? t.n * 4 : 0, true}, {t.m, t.n * sb, true},
                 {t.v, t.n * sb, true},          {d.ms, q8 ? blocks * 4 : 0, true},
                 {d.vs, q8 ? blocks * 4 : 0, true}};
        for (const auto &x : r)
            if (x.n) ranges.push_back({reinterpret_cast<uintptr_t>(x.at), x.n, x.written});
    }
    // nothing that is written meets anything else (a tensor listed twice, a
    // gradient in its parameter's place); gradients may be shared
    std::sort(ranges.begin(), ranges.end(), [](const Range &x, const Range &y) { return x.at < y.at; });
    uintptr_t end = 0, wend = 0;
    for (const Range &r : ranges) {
        if (r.at < wend || (r.written && r.at < end)) return CXM_E_INVALID;
        if (r.at + r.n > end) end = r.at + r.n;
        if (r.written && r.at + r.n > wend) wend = r.at + r.n;
    }

    std::unique_ptr<cxm_adamw> h(new cxm_adamw);
    h->pieces = static_cast<unsigned>(owner.size());
    h->p_dtype = p_dtype;
    h->g_dtype = g_dtype;
    h->master = master;
    h->q8 = q8;
    if (h->pieces) {
        hipError_t e = hipGetDevice(&h->device);
        if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void **>(&h->tensors), table.size() * sizeof(AdamTensor));
        if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void **>(&h->owner), owner.size() * sizeof(unsigned));
        if (e == hipSuccess) e = hipMemcpy(h->tensors, table.data(), table.size() * sizeof(AdamTensor), hipMemcpyHostToDevice);
        if (e == hipSuccess) e = hipMemcpy(h->owner, owner.data(), owner.size() * sizeof(unsigned), hipMemcpyHostToDevice);
        if (e != hipSuccess) {
            (void)hipGetLastError();
            if (h->tensors) (void)hipFree(h->tensors);
            if (h->owner) (void)hipFree(h->owner);
            return hip_status(e);
        }
    }
    *out = h.release();
    return CXM_OK;
}

}  // namespace

extern "C" {

int cxm_adamw_create(cxm_adamw **handle, const cxm_adamw_tensor_t *tensors, size_t count, int p_dtype, int g_dtype,
                     int state_dtype) {
    if (!handle) return CXM_E_INVALID;
    *handle = nullptr;
    if ((count && !tensors) || !is_float_dtype(p_dtype) || (g_dtype != p_dtype && g_dtype != CXM_DT_F32) ||
        (state_dtype != CXM_DT_F32 && state_dtype != CXM_DT_E4M3))
        return CXM_E_INVALID;
    try {
        return adam_create(handle, tensors, count, p_dtype, g_dtype, state_dtype);
    } catch (const std::bad_alloc &) {
        return static_cast<int>(hipErrorOutOfMemory);
    } catch (...) {
        return CXM_E_INVALID;
    }
}

int cxm_adamw_step(cxm_adamw *h, double lr, double beta1, double beta2, double eps, size_t step,
                   const float *scalars, uint64_t seed, cxm_stream_t s) {
    if (!h || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0)) return CXM_E_INVALID;
    if (!scalars && (step == 0 || !std::isfinite(lr))) return CXM_E_INVALID;
    if (h->pieces == 0) return CXM_OK;
    int dev = 0;
    const hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return hip_status(e);
    if (dev != h->device) return CXM_E_INVALID;  // the table and the tensors are on another device
    AdamStep a{};
    a.tensors = h->tensors;
    a.owner = h->owner;
    a.scalars = scalars;
    a.lr = lr;
    a.c1 = static_cast<float>(lr / (1.0 - std::pow(beta1, static_cast<double>(step))));
    a.c2 = static_cast<float>(1.0 / std::sqrt(1.0 - std::pow(beta2, static_cast<double>(step))));
    a.log_b1 = static_cast<float>(std::log(beta1));
    a.log_b2 = static_cast<float>(std::log(beta2));
    a.b1 = static_cast<float>(beta1);
    a.b1c = static_cast<float>(1.0 - beta1);
    a.b2 = static_cast<float>(beta2);
    a.b2c = static_cast<float>(1.0 - beta2);
    a.eps = static_cast<float>(eps);
    a.key = static_cast<unsigned>(seed * 0x9E3779B1ull) ^ static_cast<unsigned>(seed >> 32);
    hipStream_t hs = reinterpret_cast<hipStream_t>(s);
    if (h->p_dtype == CXM_DT_F32) adam_launch<CXM_DT_F32, CXM_DT_F32, false>(*h, a, hs);
    else if (h->p_dtype == CXM_DT_BF16) adam_launch16<CXM_DT_BF16>(*h, a, hs);
    else adam_launch16<CXM_DT_F16>(*h, a, hs);
    return launch_status();
}

int cxm_adamw_destroy(cxm_adamw *h) {
    if (!h) return CXM_E_INVALID;
    int rc = CXM_OK;
    for (void *p : {static_cast<void *>(h->tensors), static_cast<void *>(h->owner)}) {
        const hipError_t e = p ? hipFree(p) : hipSuccess;
        if (e != hipSuccess && rc == CXM_OK) rc = hip_status(e);
    }
    delete h;
    return rc;
}

}  // extern "C"
