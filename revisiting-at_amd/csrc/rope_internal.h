// What the attention's backward pass shares with qk_norm_rope (host side).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

// Cosines and sines of every token's pairs: cs [(B,) N, d / 2] (cos, sin); the samples' own where pos_b != 0.  Checks its arguments.
int rope_table(const void* positions, int pos_dtype, int64_t pos_b, int32_t axes, const int32_t* sections, const float* inv_freq, int64_t B,
               int64_t N, int32_t d, float2* cs, hipStream_t s);
// cnx_qk_norm_rope_fwd; half: bf16 heads, results in fp16 (norm only), beyond its range its largest number
int rope_forward(const void* q, const void* k, void* yq, void* yk, int dtype, bool half, const int64_t* strides, const void* wq, const void* wk,
                 int w_dtype, const void* positions, int pos_dtype, int64_t pos_batch_stride, int32_t axes, const int32_t* sections,
                 const float* inv_freq, int64_t B, int64_t N, int32_t Hq, int32_t Hk, int32_t d, float eps, int32_t norm, int32_t interleaved,
                 hipStream_t s);
// dwq, dwk [d] (either may be NULL) = sums over the rows of pq [nq][d], pk [nk][d], in a fixed order
int rope_dw(const float* pq, int nq, const float* pk, int nk, int32_t d, float* dwq, float* dwk, hipStream_t s);
