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
//
// Two kernels.  quantize_rows_kernel: a block for one row or several short ones, the row in registers between the maximum and the
// codes, so it is read once; 16-byte loads, 8-byte stores.  quantize_long_rows_kernel: rows that are too long for that, or not
// aligned to 16 bytes, are walked twice (the second time out of L2 or L1).
#include "int8.cuh"

namespace fp8gmm {
namespace {

constexpr int kLongThreads = 256;
constexpr int kMaxThreads = 512;
constexpr int kMaxVecs = 4;              // 8-element vectors a thread holds: rows of up to 512 * 4 * 8 = 16384 elements
constexpr int kStatusBadIndex = 0x200;   // as in routing.cu: an index that names no row

struct QuantRowsParams {
  const uint16_t* in;
  int64_t in_ld;       // row pitch in elements
  const int32_t* indices;
  int top_k;
  int64_t in_rows;
  int64_t rows, cols;  // of the codes
  int8_t* codes;
  int64_t codes_ld;
  float* scales;
  int* status;
};

__device__ __forceinline__ float bf16_at(const uint16_t* p, int64_t i) { return __uint_as_float(static_cast<uint32_t>(p[i]) << 16); }

// a / (1 + 2^p) from the hardware's exp2 and reciprocal, a few ulp (the rounding of exp2's argument, |p| 2^-24, is larger from
// |p| = 4 on).  Both instructions flush subnormal numbers, so the quotient is taken 16 times as large, 16 / (1 + e) =
// 1 / (1/16 + 2^(p - 4)): it then stays normal for every e = 2^p in fp32's range.  An exp that overflows gives 0.
constexpr float kLog2E = 1.44269504f;
__device__ __forceinline__ float over_one_plus_exp2(float a, float power_minus_4) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(power_minus_4));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e + 0.0625f));
  return a * 0.0625f * r;
}
template <int kAct>
__device__ __forceinline__ float activated(float a, float b) {
  if constexpr (kAct == FP8GMM_ACT_SWIGLU) return over_one_plus_exp2(a, fmaf(a, -kLog2E, -4.f)) * b;
  if constexpr (kAct == FP8GMM_ACT_GELU) {
    // 0.5 (1 + tanh u) = 1 / (1 + exp(-2u)), without the cancellation of 1 + tanh u at
    // negative u; the power of two is -2u log2(e) = a (c + 0.044715 c a^2)
    constexpr float kC = -2.f * 0.79788456f * kLog2E;
    return over_one_plus_exp2(a, fmaf(a, fmaf(a * a, 0.044715f * kC, kC), -4.f));
  }
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
// The code in the low byte: adding 1.5 * 2^23 rounds to the nearest integer, ties to even, and leaves it in the low bits.  Behind
// an activation there are no exact ties to respect (v itself is rounded), and the quotient is not corrected.
template <int kAct>
__device__ __forceinline__ uint32_t code_of(float v, const RowScale& s) {
  constexpr float kMagic = 12582912.f;
  const float t = v * s.pre;
  if constexpr (kAct != FP8GMM_ACT_NONE) return __float_as_uint(fmaf(t, s.inv, kMagic));
  float y = t * s.inv;
  y = fmaf(fmaf(-y, s.top, t), s.inv, y);
  return __float_as_uint(y + kMagic);
}
// max(a, |b|), NaN if either is
__device__ __forceinline__ float max_abs(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
  return r;
}

// Maximum over the threads of one row (blockDim.x of them, whole warps) of bits of non-negative floats (ordered like them, NaN
// above infinity); `warp_max` has a place for every warp of the row.
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* warp_max) {
  v = __reduce_max_sync(0xFFFFFFFFu, v);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return __reduce_max_sync(0xFFFFFFFFu, lane < warps ? warp_max[lane] : 0u);
}

// Source row of row r, or -1 (reported) if the index names none.
__device__ __forceinline__ int64_t source_row(const QuantRowsParams& p, int64_t r) {
  if (p.indices == nullptr) return r;
  const int32_t slot = p.indices[r];
  const int64_t src = slot / p.top_k;
  if (slot >= 0 && src < p.in_rows) return src;
  if (threadIdx.x == 0) atomicOr(p.status, kStatusBadIndex);
  return -1;
}

template <int kAct, int kVecs>
__global__ void __launch_bounds__(kMaxThreads, kVecs == 2 ? 4 : kAct == FP8GMM_ACT_SWIGLU ? 2 : 3) quantize_rows_kernel(const QuantRowsParams p) {
  __shared__ uint32_t warp_max[kMaxThreads / 32];
  let_dependents_start();
  const int64_t r = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  const bool live = r < p.rows;
  const int64_t src = live ? source_row(p, r) : -1;
  const int vecs = static_cast<int>(p.cols >> 3);
  const uint4* a = reinterpret_cast<const uint4*>(p.in + (src < 0 ? 0 : src) * p.in_ld);
  uint4 raw[kVecs], raw2[kAct == FP8GMM_ACT_SWIGLU ? kVecs : 1];
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    const int c = threadIdx.x + u * blockDim.x;
    const bool in = c < vecs && src >= 0;
    raw[u] = in ? __ldg(a + c) : make_uint4(0, 0, 0, 0);
    if constexpr (kAct == FP8GMM_ACT_SWIGLU) raw2[u] = in ? __ldg(a + vecs + c) : make_uint4(0, 0, 0, 0);   // [gate | up]
  }
  float v[kVecs][8];
  float top = 0.f;
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
    uint32_t w2[4] = {0, 0, 0, 0};
    if constexpr (kAct == FP8GMM_ACT_SWIGLU) w2[0] = raw2[u].x, w2[1] = raw2[u].y, w2[2] = raw2[u].z, w2[3] = raw2[u].w;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[u][2 * j] = activated<kAct>(bf16_lo(w[j]), bf16_lo(w2[j]));
      v[u][2 * j + 1] = activated<kAct>(bf16_hi(w[j]), bf16_hi(w2[j]));
      top = max_abs(max_abs(top, v[u][2 * j]), v[u][2 * j + 1]);
    }
  }
  const RowScale s = row_scale(row_max(__float_as_uint(top), warp_max + threadIdx.y * (blockDim.x >> 5)));
  if (!live) return;
  if (threadIdx.x == 0) p.scales[r] = s.scale;
  const bool zero = s.pre == 0.f;
  uint2* out = reinterpret_cast<uint2*>(p.codes + r * p.codes_ld);
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    const int c = threadIdx.x + u * blockDim.x;
    if (c >= vecs) break;
    uint32_t q[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float* x = &v[u][4 * h];
      const uint32_t lo = __byte_perm(code_of<kAct>(x[0], s), code_of<kAct>(x[1], s), 0x0040);
      const uint32_t hi = __byte_perm(code_of<kAct>(x[2], s), code_of<kAct>(x[3], s), 0x0040);
      q[h] = zero ? 0u : __byte_perm(lo, hi, 0x5410);
    }
    out[c] = make_uint2(q[0], q[1]);
  }
}

template <int kAct>
__global__ void __launch_bounds__(kLongThreads) quantize_long_rows_kernel(const QuantRowsParams p) {
  __shared__ uint32_t warp_max[2][kLongThreads / 32];
  let_dependents_start();
  int turn = 0;   // two sets of places: a warp may be one row ahead of another
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x, turn ^= 1) {
    const int64_t src = source_row(p, r);
    const uint16_t* a = p.in + (src < 0 ? 0 : src) * p.in_ld;
    const uint16_t* b = a + p.cols;   // SwiGLU: [gate | up]
    uint32_t top = 0;
    if (src >= 0)
      for (int64_t c = threadIdx.x; c < p.cols; c += kLongThreads) {
        const float v = activated<kAct>(bf16_at(a, c), kAct == FP8GMM_ACT_SWIGLU ? bf16_at(b, c) : 0.f);
        top = max(top, __float_as_uint(v) & 0x7FFFFFFFu);
      }
    const RowScale s = row_scale(row_max(top, warp_max[turn]));
    if (threadIdx.x == 0) p.scales[r] = s.scale;
    const bool zero = s.pre == 0.f;
    for (int64_t c = threadIdx.x; c < p.cols; c += kLongThreads) {
      uint32_t q = 0;
      if (!zero) q = code_of<kAct>(activated<kAct>(bf16_at(a, c), kAct == FP8GMM_ACT_SWIGLU ? bf16_at(b, c) : 0.f), s);
      p.codes[r * p.codes_ld + c] = static_cast<int8_t>(q & 0xFFu);
    }
  }
}

template <int kAct>
void launch_rows(const QuantRowsParams& p, cudaStream_t s) {
  const int64_t vecs = p.cols / 8;
  const bool aligned = p.cols % 8 == 0 && p.codes_ld % 8 == 0 && p.in_ld % 8 == 0 && reinterpret_cast<uintptr_t>(p.in) % 16 == 0 && reinterpret_cast<uintptr_t>(p.codes) % 8 == 0;
  if (aligned && vecs <= kMaxThreads * kMaxVecs && p.rows <= INT32_MAX) {
    // Four vectors per thread keep more bytes in flight (measured against two: 32768 rows of 4096 69 / 81 us, behind SwiGLU
    // 14336 wide 384 / 434 us = 6.1 TB/s); two answer sooner where all rows run at once, and fill a warp with a short row
    // (100000 rows of 272: 29 / 37 us).  Short rows share a block, since starting a block takes about 1 ns of the GPU's
    // time (one row per block: 262144 rows of 1024 took 272 us, now 126).
    const int per = vecs <= 64 || (vecs <= 2 * kMaxThreads && p.rows <= 4 * sm_count()) ? 2 : 4;
    const int threads = static_cast<int>(((vecs + per - 1) / per + 31) / 32 * 32);
    const int rows_per_block = threads < 256 ? 256 / threads : 1;
    const dim3 block(threads, rows_per_block);
    const unsigned int grid = static_cast<unsigned int>((p.rows + rows_per_block - 1) / rows_per_block);
    if (per == 2) quantize_rows_kernel<kAct, 2><<<grid, block, 0, s>>>(p);
    else quantize_rows_kernel<kAct, 4><<<grid, block, 0, s>>>(p);
    return;
  }
  const int64_t cap = static_cast<int64_t>(sm_count()) * 8;
  quantize_long_rows_kernel<kAct><<<static_cast<int>(p.rows < cap ? p.rows : cap), kLongThreads, 0, s>>>(p);
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
  FP8GMM_CHECK_ARG(a->codes_ld == 0 || a->codes_ld >= a->cols, "quantize_rows_int8: a row pitch of %lld is shorter than the codes' %lld",
                   (long long)a->codes_ld, (long long)a->cols);
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
  p.codes_ld = a->codes_ld != 0 ? a->codes_ld : a->cols;
  p.scales = a->scales;
  p.status = device_status_word();
  FP8GMM_CHECK_ARG(p.status != nullptr, "quantize_rows_int8: cannot resolve the device status word");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->activation == FP8GMM_ACT_SWIGLU) launch_rows<FP8GMM_ACT_SWIGLU>(p, s);
  else if (a->activation == FP8GMM_ACT_GELU) launch_rows<FP8GMM_ACT_GELU>(p, s);
  else launch_rows<FP8GMM_ACT_NONE>(p, s);
  FP8GMM_CHECK_CUDA(cudaGetLastError());
  count_launch();
  return FP8GMM_OK;
}

}  // extern "C"
