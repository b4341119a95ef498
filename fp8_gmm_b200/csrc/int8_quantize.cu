// Rows of bf16 -> int8 codes with one fp32 scale per row, optionally gathered by the router's sort and behind the expert's
// activation (HBM-bound: two bytes read, one written per element; four read with SwiGLU).
//
//   v[r, :] = act(x[src(r), :]),  top = max_k |v[r, k]|,  scale[r] = top / 127,  code[r, k] = round_half_even(127 v[r, k] / top)
//
// The code is the correctly rounded quotient, not v * (1 / scale): with bf16 inputs 127 v / top is exactly half-way between
// two codes quite often (v = top / 2 already is), and a reciprocal's error would send such values either way.  With t = 127 v
// (exact: 8 + 7 significant bits), y = t * (1 / top) is off by less than 2 ulp and one residual step, y + (t - y top) / top
// with a fused multiply-add for the exact residual, gives the representable half-way values exactly; any other quotient of a
// 15-bit by an 8-bit number is further from half-way than fp32's rounding.  Both are scaled by a power of two first, so that
// neither the reciprocal nor the product leaves fp32's range.
// A row of zeros has scale 0 and codes 0.  A row that holds an infinity or a NaN has scale NaN and codes 0: all its products
// come out NaN, no other row's do.
#include "common.cuh"

namespace fp8gmm {
namespace {

constexpr int kThreads = 256;
constexpr int kStatusBadIndex = 0x200;   // as in routing.cu: an index that names no row

struct QuantRowsParams {
  const uint16_t* in;
  int64_t in_ld;       // row pitch in elements
  const int32_t* indices;
  int top_k;
  int64_t in_rows;
  int64_t rows, cols;  // of the codes
  int8_t* codes;
  float* scales;
  int* status;
};

__device__ __forceinline__ float bf16_at(const uint16_t* p, int64_t i) { return __uint_as_float(static_cast<uint32_t>(p[i]) << 16); }

template <int kAct>
__device__ __forceinline__ float activated(float a, float b) {
  if constexpr (kAct == FP8GMM_ACT_SWIGLU) return a / (1.f + expf(-a)) * b;
  // 0.5 (1 + tanh u) = 1 / (1 + exp(-2u)): without the cancellation of 1 + tanh u at negative u
  if constexpr (kAct == FP8GMM_ACT_GELU) return a / (1.f + expf(-2.f * 0.79788456f * a * (1.f + 0.044715f * a * a)));
  return a;
}

// Factors of one row: t = v * pre, y = t * inv, residual against `top`.
struct RowScale {
  float pre, inv, top, scale;
};
__device__ __forceinline__ RowScale row_scale(uint32_t top_bits) {
  RowScale s;
  const float top = __uint_as_float(top_bits);
  if (top_bits >= 0x7F800000u) {          // infinity or NaN
    s = {0.f, 0.f, 0.f, __uint_as_float(0x7FC00000u)};
  } else if (top_bits == 0u) {
    s = {0.f, 0.f, 0.f, 0.f};
  } else {
    int e = 127 - static_cast<int>(top_bits >> 23);   // 2^e * top is in [1, 2) for normal numbers
    e = max(-126, min(e, 120));
    const float two_e = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
    s.pre = 127.f * two_e;
    s.top = top * two_e;
    s.inv = __frcp_rn(s.top);
    s.scale = __fdiv_rn(top, 127.f);
  }
  return s;
}
__device__ __forceinline__ int code_of(float v, const RowScale& s) {
  const float t = v * s.pre;
  float y = t * s.inv;
  y = fmaf(fmaf(-y, s.top, t), s.inv, y);
  return __float2int_rn(y);
}

__device__ __forceinline__ uint32_t block_max(uint32_t v) {
  __shared__ uint32_t warp_max_[kThreads / 32];
  v = __reduce_max_sync(0xFFFFFFFFu, v);
  if ((threadIdx.x & 31) == 0) warp_max_[threadIdx.x >> 5] = v;
  __syncthreads();
  uint32_t m = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) m = max(m, warp_max_[w]);
  __syncthreads();
  return m;
}

template <int kAct>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const QuantRowsParams p) {
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    int64_t src = r;
    if (p.indices != nullptr) {
      const int32_t slot = p.indices[r];
      src = slot / p.top_k;
      if (slot < 0 || src >= p.in_rows) {   // names no row: zeros, reported
        if (threadIdx.x == 0) {
          atomicOr(p.status, kStatusBadIndex);
          p.scales[r] = 0.f;
        }
        for (int64_t c = threadIdx.x; c < p.cols; c += kThreads) p.codes[r * p.cols + c] = 0;
        continue;
      }
    }
    const uint16_t* a = p.in + src * p.in_ld;
    const uint16_t* b = a + p.cols;   // SwiGLU: [gate | up]
    uint32_t top = 0;
    for (int64_t c = threadIdx.x; c < p.cols; c += kThreads) {
      const float v = activated<kAct>(bf16_at(a, c), kAct == FP8GMM_ACT_SWIGLU ? bf16_at(b, c) : 0.f);
      top = max(top, __float_as_uint(v) & 0x7FFFFFFFu);   // ordered as integers, with NaN above infinity
    }
    const RowScale s = row_scale(block_max(top));
    if (threadIdx.x == 0) p.scales[r] = s.scale;
    const bool zero = s.pre == 0.f;
    for (int64_t c = threadIdx.x; c < p.cols; c += kThreads) {
      const float v = activated<kAct>(bf16_at(a, c), kAct == FP8GMM_ACT_SWIGLU ? bf16_at(b, c) : 0.f);
      p.codes[r * p.cols + c] = static_cast<int8_t>(zero ? 0 : code_of(v, s));
    }
  }
}

}  // namespace
}  // namespace fp8gmm

extern "C" {

int fp8gmm_quantize_rows_int8(const fp8gmm_quantize_rows_args* a, void* stream) {
  using namespace fp8gmm;
  FP8GMM_CHECK_ARG(a != nullptr, "quantize_rows_int8: NULL arguments");
  FP8GMM_CHECK_ARG(a->rows >= 0 && a->cols >= 0 && a->in_rows >= 0, "quantize_rows_int8: negative size");
  FP8GMM_CHECK_ARG(a->activation == FP8GMM_ACT_NONE || a->activation == FP8GMM_ACT_GELU || a->activation == FP8GMM_ACT_SWIGLU,
                   "quantize_rows_int8: unknown activation %d", a->activation);
  const int64_t width = a->activation == FP8GMM_ACT_SWIGLU ? 2 * a->cols : a->cols;
  FP8GMM_CHECK_ARG(a->in_ld >= width, "quantize_rows_int8: a row pitch of %lld is shorter than a row of %lld", (long long)a->in_ld, (long long)width);
  if (a->rows == 0) return FP8GMM_OK;   // `indices` may then be a NULL that stands for an empty array
  FP8GMM_CHECK_ARG(a->indices != nullptr ? a->top_k > 0 : a->in_rows == a->rows, "quantize_rows_int8: %s",
                   a->indices != nullptr ? "top_k must be positive" : "row counts differ");
  FP8GMM_CHECK_ARG(a->cols > 0, "quantize_rows_int8: rows of no columns");
  FP8GMM_CHECK_ARG((a->in != nullptr || a->in_rows == 0) && a->codes && a->scales, "quantize_rows_int8: NULL pointer");
  QuantRowsParams p;
  p.in = static_cast<const uint16_t*>(a->in);
  p.in_ld = a->in_ld;
  p.indices = a->indices;
  p.top_k = a->top_k;
  p.in_rows = a->in_rows;
  p.rows = a->rows;
  p.cols = a->cols;
  p.codes = static_cast<int8_t*>(a->codes);
  p.scales = a->scales;
  p.status = device_status_word();
  FP8GMM_CHECK_ARG(p.status != nullptr, "quantize_rows_int8: cannot resolve the device status word");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t cap = static_cast<int64_t>(sm_count()) * 8;
  const int grid = static_cast<int>(a->rows < cap ? a->rows : cap);
  if (a->activation == FP8GMM_ACT_SWIGLU) quantize_rows_kernel<FP8GMM_ACT_SWIGLU><<<grid, kThreads, 0, s>>>(p);
  else if (a->activation == FP8GMM_ACT_GELU) quantize_rows_kernel<FP8GMM_ACT_GELU><<<grid, kThreads, 0, s>>>(p);
  else quantize_rows_kernel<FP8GMM_ACT_NONE><<<grid, kThreads, 0, s>>>(p);
  FP8GMM_CHECK_CUDA(cudaGetLastError());
  count_launch();
  return FP8GMM_OK;
}

}  // extern "C"
