// What the layer products' files share: the epilogue, the product's
// description and the engine's plan (linear.hip: host side and small
// kernels; linear_ring.hip: the tiled kernels; linear_skinny.hip: few rows).
#pragma once

#include "chunk.hpp"
#include "gemm_epi.hpp"

namespace cxm {

// z = v (row scale) (column scale) + bias, y = act(z) + res; every pointer
// but y may be null.  z, y, res: [m, n] of the output type.
struct LinEpi {
    const void *bias, *res;
    void *z, *y;
    const float *rs, *cs;
    int act;
};

// y = epilogue(op(A) op(B)): A [M, K] ([K, M] with ta), B [K, N] ([N, K] with
// tb).  dtype CXM_DT_E4M3 (A [M, K], B [N, K] only): bytes; else out == dtype.
struct LinProduct {
    const void *a, *b;
    size_t M, K, N;
    bool ta, tb;
    int dtype, out;
    LinEpi e;
};

struct LinPlan {
    int kernel;       // 0 skinny, else the rows of the ring's tile
    bool copy_a, copy_b, staged;
    size_t lda, ldb;  // of what the ring reads, in its 16-bit units
    size_t stages;    // of 32 units along K
    size_t splits, per;
    size_t tiles_m, tiles_n, tiles;
    size_t bytes_a, bytes_b, bytes_part;  // workspace, multiples of 256
    size_t bytes() const { return bytes_a + bytes_b + bytes_part; }
    size_t counters() const { return splits > 1 ? tiles : 0; }
};

int linear_plan(const LinProduct &p, LinPlan *plan);
// `scratch` holds plan.bytes() (256-byte aligned), `counters` plan.counters().
int linear_run(const LinProduct &p, const LinPlan &plan, char *scratch, unsigned *counters, hipStream_t s);

bool linear_skinny_plan(const LinProduct &p, LinPlan *plan);
int linear_skinny_run(const LinProduct &p, const LinPlan &plan, float *part, unsigned *counters, hipStream_t s);
int linear_ring_run(const LinProduct &p, const LinPlan &plan, const void *a, const void *b, float *part,
                    unsigned *counters, hipStream_t s);

}  // namespace cxm
