// What the int8 row quantisation and the int8 product share: the second is launched while the first still runs.
#pragma once

#include "common.cuh"

namespace fp8gmm {

// The product of rows that `fp8gmm_quantize_rows_int8` has just been enqueued for on the same stream: its CTAs may start, and
// load weights, before the codes are there.
int int8_gemm_launch(const fp8gmm_int8_gemm_args* a, void* stream, bool after_quantize);

#ifdef __CUDACC__
// Lets the next kernel of the stream start its CTAs as soon as all CTAs of this one have come here (programmatic dependent
// launch); it reads this kernel's results only behind grid_dependency_wait.
__device__ __forceinline__ void let_dependents_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
#endif

}  // namespace fp8gmm
