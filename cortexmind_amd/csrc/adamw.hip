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
#include <cmath>
#include <cstring>
#include <memory>
#include <new>
#include <vector>
#include <algorithm>

#include "chunk.hpp"

struct cxm_adamw;

namespace cxm {
namespace {

constexpr unsigned kLane = 8;                // values per thread
constexpr unsigned kPiece = kBlock * kLane;  // values per workgroup
constexpr unsigned kBlock8 = 256;            // values per scale: 32 lanes

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

// a in [0, 448] to e4m3's neighbour above with the probability of a's distance
// to the one below: 16 random bits are added below the 3 kept mantissa bits and
// the rest cut off.  Below 2^-6 the steps are even (2^-9): 2^-6 is added
// first and taken off after.
__device__ __forceinline__ float round_e4m3(float a, unsigned bits) {
    const float low = a < 0x1p-6f ? 0x1p-6f : 0.0f;
    const float b = a + low;
    const unsigned u = (__builtin_bit_cast(unsigned, b) + (bits << 4)) & ~0xFFFFFu;
    return __builtin_bit_cast(float, u) - low;
}

template <int PD, int GD, bool MASTER, bool Q8>
__global__ __launch_bounds__(kBlock) void k_adamw(AdamStep a) {
    using PS = typename Elem<PD>::S;
    using GS = typename Elem<GD>::S;
    const AdamTensor t = a.tensors[a.owner[blockIdx.x]];
    const size_t i0 = static_cast<size_t>(blockIdx.x - t.piece0) * kPiece + threadIdx.x * kLane;
    const bool whole = t.vec && i0 + kLane <= t.n;
    PS *p = static_cast<PS *>(t.p);
    const GS *g = static_cast<const GS *>(t.g);

    float vp[kLane], vg[kLane], vm[kLane], vv[kLane];
    size_t blk = i0 / kBlock8;
    const size_t blocks = (t.n + kBlock8 - 1) / kBlock8;
    const bool leads = Q8 && blk < blocks && i0 % kBlock8 == 0;
    if (blk >= blocks) blk = blocks - 1;
    float sm = 0.0f, sv = 0.0f;
    if constexpr (Q8) {
        sm = t.ms[blk];
        sv = t.vs[blk];
    }
    auto load_f = [](const float *q, float (&o)[kLane]) {
        const float4 x = ld4(q), y = ld4(q + 4);
        o[0] = x.x; o[1] = x.y; o[2] = x.z; o[3] = x.w;
        o[4] = y.x; o[5] = y.y; o[6] = y.z; o[7] = y.w;
    };
    if (whole) {
        if constexpr (MASTER) {
            load_f(t.w + i0, vp);
        } else if constexpr (PD == CXM_DT_F32) {
            load_f(p + i0, vp);
        } else {
            Chunk<PD, 8> c;
            c.load(p + i0);
#pragma unroll
            for (int e = 0; e < 8; ++e) vp[e] = c.get(e);
        }
        if constexpr (GD == CXM_DT_F32) {
            load_f(g + i0, vg);
        } else {
            Chunk<GD, 8> c;
            c.load(g + i0);
#pragma unroll
            for (int e = 0; e < 8; ++e) vg[e] = c.get(e);
        }
        if constexpr (Q8) {
            const uint2 qm = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(t.m) + i0);
            const uint2 qv = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(t.v) + i0);
            unpack_e4m3(qm.x, vm);
            unpack_e4m3(qm.y, vm + 4);
            unpack_e4m3(qv.x, vv);
            unpack_e4m3(qv.y, vv + 4);
        } else {
            load_f(static_cast<const float *>(t.m) + i0, vm);
            load_f(static_cast<const float *>(t.v) + i0, vv);
        }
    } else {
#pragma unroll
        for (unsigned e = 0; e < kLane; ++e) {
            const size_t i = i0 + e;
            vp[e] = vg[e] = vm[e] = vv[e] = 0.0f;
            if (i < t.n) {
                if constexpr (MASTER) vp[e] = t.w[i];
                else vp[e] = Elem<PD>::load(p[i]);
                vg[e] = Elem<GD>::load(g[i]);
                if constexpr (Q8) {
                    float u[4];
                    unpack_e4m3(static_cast<const uint8_t *>(t.m)[i], u);
                    vm[e] = u[0];
                    unpack_e4m3(static_cast<const uint8_t *>(t.v)[i], u);
                    vv[e] = u[0];
                } else {
                    vm[e] = static_cast<const float *>(t.m)[i];
                    vv[e] = static_cast<const float *>(t.v)[i];
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

    float am = 0.0f, av = 0.0f;
#pragma unroll
    for (unsigned e = 0; e < kLane; ++e) {
        const float gr = a.scalars ? vg[e] * factor : vg[e];
        float m0 = vm[e], v0 = vv[e];
        if constexpr (Q8) {
            m0 *= sm;
            v0 *= sv;
            v0 *= v0;
        }
        const float m1 = a.b1 * m0, m2 = a.b1c * gr, gg = gr * gr, v1 = a.b2 * v0, v2 = a.b2c * gg;
        const float m = m1 + m2, v = v1 + v2, r = __builtin_sqrtf(v);
        const float d = r * c2 + a.eps, u = c1 * m / d, q = vp[e] * keep;
        vp[e] = q - u;
        vm[e] = m;
        vv[e] = Q8 ? r : v;
        if constexpr (Q8) {  // the largest finite magnitudes
            am = fabsf(m) <= FLT_MAX && fabsf(m) > am ? fabsf(m) : am;
            av = r <= FLT_MAX && r > av ? r : av;
        }
    }
    uint2 qm{0, 0}, qv{0, 0};
    if constexpr (Q8) {
        am = group_reduce<MaxOp, 32>(am);
        av = group_reduce<MaxOp, 32>(av);
        const Scale8 km = scale_e4m3(am), kv = scale_e4m3(av);
        if (leads) {
            t.ms[blk] = km.scale;
            t.vs[blk] = kv.scale;
        }
        float em[kLane], ev[kLane];
#pragma unroll
        for (unsigned e = 0; e < kLane; ++e) {
            const unsigned bits = noise32(t.first + i0 + e, a.key);
            const float x = fabsf(vm[e]) * km.inv, y = vv[e] * kv.inv;
            // NaN and infinity are stored as NaN, where they are alone
            const float qx = round_e4m3(x < kE4M3Max ? x : kE4M3Max, bits & 0xFFFFu);
            float qy = round_e4m3(y < kE4M3Max ? y : kE4M3Max, bits >> 16);
            qy = qy == 0.0f && y > 0.0f ? 0x1p-9f : qy;
            em[e] = fabsf(vm[e]) <= FLT_MAX ? __builtin_copysignf(qx, vm[e]) : __builtin_nanf("");
            ev[e] = vv[e] <= FLT_MAX ? qy : __builtin_nanf("");
        }
        qm = uint2{pack_e4m3(em[0], em[1], em[2], em[3]), pack_e4m3(em[4], em[5], em[6], em[7])};
        qv = uint2{pack_e4m3(ev[0], ev[1], ev[2], ev[3]), pack_e4m3(ev[4], ev[5], ev[6], ev[7])};
    }

    auto store_f = [](float *q, const float (&o)[kLane]) {
        st4(q, make_float4(o[0], o[1], o[2], o[3]));
        st4(q + 4, make_float4(o[4], o[5], o[6], o[7]));
    };
    if (whole) {
        if constexpr (MASTER) store_f(t.w + i0, vp);
        if constexpr (PD == CXM_DT_F32) {
            store_f(p + i0, vp);
        } else {
            Chunk<PD, 8> c;
            c.set(vp);
            c.store(p + i0);
        }
        if constexpr (Q8) {
            *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(t.m) + i0) = qm;
            *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(t.v) + i0) = qv;
        } else {
            store_f(static_cast<float *>(t.m) + i0, vm);
            store_f(static_cast<float *>(t.v) + i0, vv);
        }
    } else {
#pragma unroll
        for (unsigned e = 0; e < kLane; ++e) {
            const size_t i = i0 + e;
            if (i < t.n) {
                if constexpr (MASTER) t.w[i] = vp[e];
                p[i] = Elem<PD>::store(vp[e]);
                if constexpr (Q8) {
                    static_cast<uint8_t *>(t.m)[i] = static_cast<uint8_t>((e < 4 ? qm.x : qm.y) >> (8 * (e & 3)));
                    static_cast<uint8_t *>(t.v)[i] = static_cast<uint8_t>((e < 4 ? qv.x : qv.y) >> (8 * (e & 3)));
                } else {
                    static_cast<float *>(t.m)[i] = vm[e];
                    static_cast<float *>(t.v)[i] = vv[e];
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
        if (owner.size() + pieces > 0x7fffffu * size_t(16)) return CXM_E_TOO_LARGE;
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
