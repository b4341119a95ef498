// What the int8 row quantisation and the int8 product share: the second is launched while the first still runs.
#pragma once

#include "dependent_launch.cuh"

namespace fp8gmm {

// The product of rows that `fp8gmm_quantize_rows_int8` has just been enqueued for on the same stream: its CTAs may start, and
// load weights, before the codes are there (after_quantize).
int int8_gemm_launch(const fp8gmm_int8_gemm_args* a, void* stream, bool after_quantize);

}  // namespace fp8gmm
