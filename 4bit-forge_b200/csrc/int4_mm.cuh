// Arguments of the int4 product kernels, shared by their translation units.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

namespace forge {

struct Int4Fwd {
    const void *x;
    int64_t ldx;
    const uint32_t *packed[2];   // [R, C/8]; the second matrix only in the gated form
    const float *scales[2];      // [R, G]
    int gs;
    int64_t T, C, R, G;
    const void *bias;            // [R] or NULL (linear form)
    int act;
    const void *res;             // [T, ldres >= R] or NULL (linear form)
    int64_t ldres;
    void *y;                     // [T, R]
    void *pre0, *pre1;           // pre-activations [T, R] or NULL (pre1: gated form)
    int32_t *status;
};

struct Int4Dgrad {
    const __half *a;             // [T, ldk]: dz times powers of two
    int64_t ldk;
    const float *unscale;        // [T]
    const uint32_t *packed[2];
    const __half2 *pairs;        // [mats * R, G]: normalised scales, hi and lo part
    int gs, mats;
    int64_t T, C, R, G;
    void *dx;                    // [T, C]
    int32_t *status;
};

}  // namespace forge
