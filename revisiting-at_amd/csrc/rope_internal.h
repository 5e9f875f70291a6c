// What the attention's backward pass shares with qk_norm_rope (host side).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

// Cosines and sines of every token's pairs: cs [(B,) N, d / 2] (cos, sin); the samples' own where pos_b != 0.  Checks its arguments.
int rope_table(const void* positions, int pos_dtype, int64_t pos_b, int32_t axes, const int32_t* sections, const float* inv_freq, int64_t B,
               int64_t N, int32_t d, float2* cs, hipStream_t s);
// dwq, dwk [d] (either may be NULL) = sums over the rows of part [2][rows][d], in a fixed order
int rope_dw(const float* part, int rows, int32_t d, float* dwq, float* dwk, hipStream_t s);
