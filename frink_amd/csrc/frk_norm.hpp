// What the norm and the runtime share: a norm's operands, and the forms of quantized activations that it can leave.
#pragma once

#include "frk_f8.hpp"
#include "frk_mx4.hpp"

namespace frk {

enum { ACTS_NONE = -1, ACTS_Q8_K = FRK_ACTS_Q8_K, ACTS_FP8 = FRK_ACTS_FP8, ACTS_MXFP4 = FRK_ACTS_MXFP4 };

struct NormArgs {
    const void *x, *residual;  // [batch][cols] of one type; residual: or null
    const void *weight;        // [cols] of weight_type, or null: ones
    int weight_type;
    double eps, inverse_cols;
    size_t batch, rows;  // rows: the batch, or more of a form whose last tile's rows are to be zeros
    int cols, chunks, waves;  // (chunks, waves, inverse_cols: the launch's own)
    void *sum, *y;       // of x's type; or null
};
struct NormOut {  // (of one form; null pointers: not wanted)
    F8Acts f8, f8_strips;
    int f8_blocks;
    Q8KActsOut plain;
    Q8KTiled tiled;
    int q8k_blocks;
    Mx4Acts mx4;
};
int launch_rms_norm(int type, NormArgs a, int form, const NormOut &out, hipStream_t s);
// the numbers that a batch in one form (its pointers set) stands for
int launch_acts_values(int form, const NormOut &in, size_t rows, size_t cols, float *out, hipStream_t s);

}  // namespace frk
