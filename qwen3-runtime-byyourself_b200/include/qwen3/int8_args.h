/* qwen3/int8_args.h - the arguments of the kernels of 8-bit integer rows (kernels.h), handed over as a structure in host memory that the call
   reads before it returns.  All pointers are device pointers; `stream` is a cudaStream_t.
   Rows in 8 bits: codes [rows, width] (-128 to 127), rows `stride` bytes apart, a multiple of 16 that is at least the width, from a 16-byte
   boundary on; scales float32 [rows].  A code stands for code * scale of its row. */
#pragma once

#include <stdint.h>

/* q3_quantize_rows_*: rows of x as codes and scales.  q3_rms_norm_int8_*: the same of rms-normed rows, of x + delta if delta is given (that sum
   goes to `total`, rounded to x's type).  Strides in elements. */
typedef struct q3_int8_rows_args {
    const void *x, *delta, *weight;                   /* weight: float32 [width] (the norm's) */
    void *total, *codes, *scales, *stream;
    int64_t rows, x_stride, delta_stride, total_stride, codes_stride;
    double eps;
    int width, reserved;
} q3_int8_rows_args;

/* q3_gemm_int8_*: y[m, n] = (sum over k of x[m, k] w[n, k]) * x_scales[m] * w_scales[n], the sum in whole numbers (width at most 131,071, so
   that 32 bits hold it); y [rows, channels], dense, in bfloat16 or float32.  activation 0: that; 1 (SiLU) and 2 (the tanh form of GELU): the
   channels are gate[8] up[8] in turns (their number a multiple of 16) and y [rows, channels / 2] = act(gate) * up in 32 bits, rounded once.  `status`: see
   the tcgen05 products. */
typedef struct q3_gemm_int8_args {
    const void *x, *x_scales, *w, *w_scales;
    void *y, *status, *stream;
    int64_t x_stride, w_stride;                       /* bytes, multiples of 16 */
    int rows, channels, width, out_is_f32, activation, splits;
} q3_gemm_int8_args;
