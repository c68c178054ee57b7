// Second step of the column sums of the backward passes (a norm's gain, a bias): partial sums of row shares, joined.
#pragma once
#include "common.cuh"
#include "elem.cuh"

namespace forge {

// out[c] = sum over n rows of partial[n, C], in a fixed order: 32 columns x 32 row strands per CTA
template <typename T>
__global__ void __launch_bounds__(1024) column_sum_kernel(const float *__restrict__ partial, int n, int64_t C, T *out) {
    __shared__ float s[32][33];
    const int64_t c = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
    const int k = threadIdx.x >> 5;
    float v = 0.0f;
    if (c < C)
#pragma unroll 4
        for (int r = k; r < n; r += 32) v += partial[(int64_t)r * C + c];
    s[k][threadIdx.x & 31] = v;
    __syncthreads();
    v = s[threadIdx.x & 31][k];              // column k of the block, strand = lane
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int64_t co = (int64_t)blockIdx.x * 32 + k;
    if ((threadIdx.x & 31) == 0 && co < C) out[co] = Elem<T>::from_f(v);
}
// out [C] of type `dtype`; n = 0 gives zeros
inline void launch_column_sum(const float *partial, int n, int64_t C, void *out, int dtype, cudaStream_t st) {
    const unsigned blocks = (unsigned)cdiv(C, (int64_t)32);
    if (dtype == FORGE_DTYPE_F32) column_sum_kernel<float><<<blocks, 1024, 0, st>>>(partial, n, C, (float *)out);
    else if (dtype == FORGE_DTYPE_BF16) column_sum_kernel<__nv_bfloat16><<<blocks, 1024, 0, st>>>(partial, n, C, (__nv_bfloat16 *)out);
    else column_sum_kernel<__half><<<blocks, 1024, 0, st>>>(partial, n, C, (__half *)out);
    FORGE_NOTE_LAUNCH();
}

}  // namespace forge
