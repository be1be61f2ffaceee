// Column sums of fp32 partials, the second half of the weight and bias
// gradients (norm.hip, layernorm.hip, linear.hip).
#include "chunk.hpp"

namespace cxm {
namespace {

// out[j] = the sum of part[0 .. n - 1][j] (and, of a second grid row, out2[j] that
// of the columns `second` floats on): 16 columns per workgroup (64-byte
// pieces of a row), its 64 groups of 16 lanes taking every 64th partial, eight
// loads in flight; the groups meet pairwise in LDS.  With 64 columns per
// workgroup 2048 columns of 1024 partials ran on 32 CUs, 6.2 us.
constexpr int kSumThreads = 1024, kSumCols = 16;
template <int DT>
__global__ __launch_bounds__(kSumThreads) void k_col_sum(const float *part, unsigned n, unsigned cols, size_t ld,
                                                         typename Elem<DT>::S *out, size_t second,
                                                         typename Elem<DT>::S *out2) {
    constexpr unsigned W = kSumThreads / kSumCols, U = 8;
    __shared__ float lds[W][kSumCols];
    const unsigned c = threadIdx.x % kSumCols, g = threadIdx.x / kSumCols;
    const unsigned j = blockIdx.x * kSumCols + c;
    const float *p = part + (j < cols ? j : cols - 1);
    if (blockIdx.y) {
        p += second;
        out = out2;
    }
    float s = 0.0f;
    for (unsigned i = g; i < n; i += W * U) {
        float v[U];
#pragma unroll
        for (unsigned u = 0; u < U; ++u) v[u] = i + u * W < n ? p[(i + u * W) * ld] : 0.0f;
#pragma unroll
        for (unsigned u = 0; u < U; ++u) s += v[u];
    }
    lds[g][c] = s;
    __syncthreads();
    if (g == 0 && j < cols) out[j] = Elem<DT>::store(combine_pairwise<SumOp, W>(&lds[0][c], kSumCols));
}

template <int DT>
void launch(const float *part, unsigned n, unsigned cols, size_t ld, void *out, size_t second, void *out2, hipStream_t s) {
    using S = typename Elem<DT>::S;
    hipLaunchKernelGGL((k_col_sum<DT>), dim3((cols + kSumCols - 1) / kSumCols, out2 ? 2 : 1), dim3(kSumThreads), 0, s,
                       part, n, cols, ld, static_cast<S *>(out), second, static_cast<S *>(out2));
}

}  // namespace

// (Columns past what a grid holds, 2^26 - 16 of them, in a launch of their own:
// the callers have launched their first half and must not be refused here.)
int col_sum2(const float *part, size_t n, size_t cols, size_t ld, void *out, size_t second, void *out2, int dtype,
             hipStream_t s) {
    if (n > 0x7fffffffu || cols > 0x7fffffffu) return CXM_E_TOO_LARGE;
    constexpr size_t kMost = most_wgs(kSumThreads) * kSumCols;
    const unsigned nn = static_cast<unsigned>(n);
    for (size_t j = 0; j < cols; j += kMost) {
        const unsigned nc = static_cast<unsigned>(cols - j < kMost ? cols - j : kMost);
        const float *p = part ? part + j : nullptr;
        char *o = static_cast<char *>(out) + j * dtype_bytes(dtype);
        char *o2 = out2 ? static_cast<char *>(out2) + j * dtype_bytes(dtype) : nullptr;
        if (dtype == CXM_DT_F32) launch<CXM_DT_F32>(p, nn, nc, ld, o, second, o2, s);
        else if (dtype == CXM_DT_BF16) launch<CXM_DT_BF16>(p, nn, nc, ld, o, second, o2, s);
        else launch<CXM_DT_F16>(p, nn, nc, ld, o, second, o2, s);
        const int r = launch_status();
        if (r) return r;
    }
    return CXM_OK;
}

int col_sum(const float *part, size_t n, size_t cols, size_t ld, void *out, int dtype, hipStream_t s) {
    return col_sum2(part, n, cols, ld, out, 0, nullptr, dtype, s);
}

}  // namespace cxm
