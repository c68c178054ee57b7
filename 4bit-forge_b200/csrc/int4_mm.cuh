// Arguments of the int4 product kernels, shared by their translation units.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
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
    bool vec8, vec16;            // rows of packed words start on 8 (16) bytes
};

struct Int4Dgrad {
    const __half *a;             // [T, ldk + lo]: dz times powers of two, in fp16, and behind it what that rounds off
    int64_t ldk, lo;             // lo: 0, or ldk when the low parts are there (fp16 gradients only)
    const float *unscale;        // [T]
    const uint32_t *packed[2];
    const __half2 *pairs;        // [mats * R, G]: normalised scales, hi and lo part
    const float *group;          // [ceil(mats * R / kKBlock), G]: powers of two that the sums of a block of rows take
    int gs, mats;
    int64_t T, C, R, G;
    void *dx;                    // [T, C]
    int32_t *status;
    bool vec8;                   // rows of packed words start on 8 bytes
};

constexpr int kKBlock = 512;           // weight rows whose products are summed up before they enter dx
// Most tokens that int4_decode takes.  16 tokens there and in the tensor-memory kernel, groups of 128: 7168 -> 2048 9.6 and
// 15.4 us, 2048 -> 7168 10.4 and 11.8, 2048 -> 768 3.9 and 8.5, 7168 -> 18432 50.0 and 49.7 (gated 99.6 and 88.9, but 96.8 and
// 107.5 at 9 tokens); groups of 32: 7168 -> 18432 58.5 and 92.8.  24 tokens, 7168 -> 2048: 16.9 and 14.5.
constexpr int kDecodeTokens = 16;
// more tokens than int4_decode takes; the backward product
int int4_fwd_tc(const Int4Fwd &P, bool bf16, bool gated, cudaStream_t st);
int int4_dgrad_tc(const Int4Dgrad &P, bool bf16, const char *who, cudaStream_t st);
int int4_decode(const Int4Fwd &P, bool bf16, bool gated, cudaStream_t st);

}  // namespace forge
