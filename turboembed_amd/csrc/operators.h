// Launchers of the operators on device memory (operators.cpp checks their
// arguments). As the launchers of kernels.h: each enqueues on the given
// stream and returns the launch's error; none allocates, waits or copies.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kernels.h"

namespace rocm {

// Rows at most this wide are held in one workgroup's registers (row_codes.hip).
constexpr uint64_t ROW_COLS_MAX = 65536;

// Row strides are in elements. Absent arrays are NULL (codes are wanted where
// scales is given: rows of no columns have scales alone).
struct RowArgs {
    const void *x, *res, *w;
    void *sum, *out;
    int8_t *codes;
    float *scales;
    uint64_t ldx, ldr, lds, ldo, ldc;
    Dt xt, rt, wt, ot;   // rt: the residual's, and v's (xt without one)
    int rows, cols;
    double eps;
};
// rms_norm (with w), or quantize_tokens (w NULL: codes and scales alone).
hipError_t row_codes(hipStream_t s, const RowArgs &a);

// The widest inner width of an int8 product: 131071 * 128 * 128 < 2^31.
constexpr uint64_t I8_INNER_MAX = 131071;

struct LinearArgs {
    const int8_t *a, *w;
    const float *as, *ws, *bias;
    void *out;
    uint64_t lda, ldw, ldo;
    Dt ot;
    int m, n, k;
};
hipError_t linear_i8(hipStream_t s, const LinearArgs &a);
// The kernel that linear_i8 takes for an inner width of 16 or more: 1 to 4,
// pieces of so many 16 rows, or 64, 128 or 256, tiles of that edge. aligned:
// operands of whole aligned 16-byte chunks.
int linear_i8_kernel(int m, int n, int k, bool aligned);

// Cross attention's work, as a plan holds it on the device. The rows of a
// (sequence, key head) are its query tokens' heads that read the key head:
// row r is token r / share of the sequence's, head kv * share + r % share.
// An item is up to part_rows of them (32, a wave's, or 128, four waves')
// against keys k0 .. k0 + nk - 1; where a row's keys are cut over several
// items, each leaves its part (`part`) in the workspace and a join adds them
// up; part -1 writes the output itself.
struct CrossItem {
    int32_t q0;           // the sequence's first token
    int32_t row0, rows;
    int32_t k0, nk;
    int32_t kv;
    int32_t part;
    int32_t pad;
};
// The rows whose keys were cut: parts part0 .. part0 + parts - 1.
struct CrossJoin {
    int32_t q0, row0, rows, kv, part0, parts, pad[2];
};

struct CrossArgs {
    const void *q, *k, *v;
    void *out;
    const int32_t *mask;
    float *ws;               // parts
    const CrossItem *items;
    const CrossJoin *joins;
    uint64_t qs[2], ks[2], vs[2], os[2];   // strides of tokens and heads, elements
    Dt dt;
    int n_items, n_joins, part_rows, most_rows, share, width;   // (most_rows: of one join)
    bool one_wave;           // no item has more than 32 rows, a wave's
    float scale;             // of a score, times log2(e); positive...
    float turn;              // ...with 1, -1 or 0 times q
};
hipError_t cross_attention(hipStream_t s, const CrossArgs &a);

// A part's floats, of the most rows that a join has: its rows' sums, four columns of every row after another,
// then each row's maximum (base 2) and sum of weights; a row without a finite
// maximum leaves 1 for that sum if it had a live key.
inline __host__ __device__ uint64_t cross_part_floats(int most_rows, int width) {
    return ((uint64_t)most_rows * ((width + 3) / 4 * 4 + 2) + 3) / 4 * 4;   // (16-byte stores)
}

}  // namespace rocm
