// Column sums of fp32 partials, the second half of the weight and bias
// gradients (norm.hip, linear.hip).
#include "chunk.hpp"

namespace cxm {
namespace {

// out[j] = the sum of part[0 .. n - 1][j]: 16 columns per workgroup (64-byte
// pieces of a row), its 64 groups of 16 lanes taking every 64th partial, eight
// loads in flight; the groups meet pairwise in LDS.  With 64 columns per
// workgroup 2048 columns of 1024 partials ran on 32 CUs, 6.2 us.
constexpr int kSumThreads = 1024, kSumCols = 16;
template <int DT>
__global__ __launch_bounds__(kSumThreads) void k_col_sum(const float *part, unsigned n, unsigned cols, size_t ld,
                                                         typename Elem<DT>::S *out) {
    constexpr unsigned W = kSumThreads / kSumCols, U = 8;
    __shared__ float lds[W][kSumCols];
    const unsigned c = threadIdx.x % kSumCols, g = threadIdx.x / kSumCols;
    const unsigned j = blockIdx.x * kSumCols + c;
    const float *p = part + (j < cols ? j : cols - 1);
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
void launch(const float *part, unsigned n, unsigned cols, size_t ld, void *out, hipStream_t s) {
    hipLaunchKernelGGL((k_col_sum<DT>), dim3((cols + kSumCols - 1) / kSumCols), dim3(kSumThreads), 0, s, part, n, cols, ld,
                       static_cast<typename Elem<DT>::S *>(out));
}

}  // namespace

int col_sum(const float *part, size_t n, size_t cols, size_t ld, void *out, int dtype, hipStream_t s) {
    if (n > 0x7fffffffu || cols > 0x7fffffffu || (cols + kSumCols - 1) / kSumCols > most_wgs(kSumThreads)) return CXM_E_TOO_LARGE;
    const unsigned nn = static_cast<unsigned>(n), nc = static_cast<unsigned>(cols);
    if (dtype == CXM_DT_F32) launch<CXM_DT_F32>(part, nn, nc, ld, out, s);
    else if (dtype == CXM_DT_BF16) launch<CXM_DT_BF16>(part, nn, nc, ld, out, s);
    else launch<CXM_DT_F16>(part, nn, nc, ld, out, s);
    return launch_status();
}

}  // namespace cxm
