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

// Two floats in a register pair: one instruction for both where there is a packed form, each rounded as on its own.  The kernel is
// bound by its instructions as much as by HBM: 32768 rows of 4096 took 69 us with single ones and 61.5 with these; behind GELU 89
// and 77, behind SwiGLU 106 and 102.  (Behind an activation the special function unit is next, two operations an element at an
// eighth of the rate; one reciprocal shared by two elements saved a quarter of them and cost more in the test for its range: 93.)
struct Pair {
  uint64_t v;
};
__device__ __forceinline__ Pair pair_of(float a, float b) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ Pair both(float a) { return pair_of(a, a); }
__device__ __forceinline__ float2 split(Pair p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p.v));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// a / (1 + 2^p) from the hardware's exp2 and reciprocal, a few ulp (the rounding of exp2's argument, |p| 2^-24, is larger from
// |p| = 4 on).  Both instructions flush subnormal numbers, so the quotient is taken 16 times as large, 16 / (1 + e) =
// 1 / (1/16 + 2^(p - 4)): it then stays normal for every e = 2^p in fp32's range.  An exp that overflows gives 0.
// The two share a reciprocal, 1 / d = d' / (d d'), unless d d' leaves the range in which that stays normal: the special function
// unit, at an eighth of the others' rate, is what limits this kernel behind an activation.
constexpr float kLog2E = 1.44269504f;
__device__ __forceinline__ Pair over_one_plus_exp2(Pair a, Pair powers_minus_4) {
  const float2 p = split(powers_minus_4);
  const float2 d = split(add2(pair_of(exp2_approx(p.x), exp2_approx(p.y)), both(0.0625f)));
  const Pair inv = pair_of(rcp_approx(d.x), rcp_approx(d.y));
  return mul2(mul2(a, both(0.0625f)), inv);
}
template <int kAct>
__device__ __forceinline__ Pair activated(Pair a, Pair b) {
  if constexpr (kAct == FP8GMM_ACT_SWIGLU) return mul2(over_one_plus_exp2(a, fma2(a, both(-kLog2E), both(-4.f))), b);
  if constexpr (kAct == FP8GMM_ACT_GELU) {
    // 0.5 (1 + tanh u) = 1 / (1 + exp(-2u)), without the cancellation of 1 + tanh u at
    // negative u; the power of two is -2u log2(e) = a (c + 0.044715 c a^2)
    constexpr float kC = -2.f * 0.79788456f * kLog2E;
    return over_one_plus_exp2(a, fma2(a, fma2(mul2(a, a), both(0.044715f * kC), both(kC)), both(-4.f)));
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
// The codes in the low bytes: adding 1.5 * 2^23 rounds to the nearest integer, ties to even, and leaves it in the low bits.  Behind
// an activation there are no exact ties to respect (v itself is rounded), and the quotient is not corrected.
template <int kAct>
__device__ __forceinline__ uint2 codes_of(Pair v, const RowScale& s) {
  const Pair magic = both(12582912.f), t = mul2(v, both(s.pre));
  Pair y;
  if constexpr (kAct != FP8GMM_ACT_NONE) {
    y = fma2(t, both(s.inv), magic);
  } else {
    y = mul2(t, both(s.inv));
    y = add2(fma2(fma2(y, both(-s.top), t), both(s.inv), y), magic);
  }
  const float2 r = split(y);
  return make_uint2(__float_as_uint(r.x), __float_as_uint(r.y));
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
  Pair v[kVecs][4];
  float top = 0.f;
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
    uint32_t w2[4] = {0, 0, 0, 0};
    if constexpr (kAct == FP8GMM_ACT_SWIGLU) w2[0] = raw2[u].x, w2[1] = raw2[u].y, w2[2] = raw2[u].z, w2[3] = raw2[u].w;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[u][j] = activated<kAct>(pair_of(bf16_lo(w[j]), bf16_hi(w[j])), pair_of(bf16_lo(w2[j]), bf16_hi(w2[j])));
      const float2 x = split(v[u][j]);
      top = max_abs(max_abs(top, x.x), x.y);
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
      const uint2 a2 = codes_of<kAct>(v[u][2 * h], s), b2 = codes_of<kAct>(v[u][2 * h + 1], s);
      q[h] = zero ? 0u : __byte_perm(__byte_perm(a2.x, a2.y, 0x0040), __byte_perm(b2.x, b2.y, 0x0040), 0x5410);
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
    // columns c (even) and c + 1, in the pairs of the other kernel
    auto activated_at = [&](int64_t c) {
      const bool two = c + 1 < p.cols;
      return activated<kAct>(pair_of(bf16_at(a, c), two ? bf16_at(a, c + 1) : 0.f),
                             kAct == FP8GMM_ACT_SWIGLU ? pair_of(bf16_at(b, c), two ? bf16_at(b, c + 1) : 0.f) : both(0.f));
    };
    uint32_t top = 0;
    if (src >= 0)
      for (int64_t c = 2 * threadIdx.x; c < p.cols; c += 2 * kLongThreads) {
        const float2 v = split(activated_at(c));
        top = max(top, max(__float_as_uint(v.x) & 0x7FFFFFFFu, __float_as_uint(v.y) & 0x7FFFFFFFu));
      }
    const RowScale s = row_scale(row_max(top, warp_max[turn]));
    if (threadIdx.x == 0) p.scales[r] = s.scale;
    const bool zero = s.pre == 0.f;
    for (int64_t c = 2 * threadIdx.x; c < p.cols; c += 2 * kLongThreads) {
      const uint2 q = zero ? make_uint2(0u, 0u) : codes_of<kAct>(activated_at(c), s);
      int8_t* out = p.codes + r * p.codes_ld + c;
      out[0] = static_cast<int8_t>(q.x & 0xFFu);
      if (c + 1 < p.cols) out[1] = static_cast<int8_t>(q.y & 0xFFu);
    }
  }
}

template <int kAct>
void launch_rows(const QuantRowsParams& p, cudaStream_t s) {
  const int64_t vecs = p.cols / 8;
  const bool aligned = p.cols % 8 == 0 && p.codes_ld % 8 == 0 && p.in_ld % 8 == 0 && reinterpret_cast<uintptr_t>(p.in) % 16 == 0 && reinterpret_cast<uintptr_t>(p.codes) % 8 == 0;
  if (aligned && vecs <= kMaxThreads * kMaxVecs && p.rows <= INT32_MAX) {
    // Four vectors per thread keep more bytes in flight (measured against two: 32768 rows of 4096 61 / 71 us, 262144 rows of 1024
    // 117 / 138); two answer sooner where all rows run at once (300 rows of 4096 2.5 / 2.9 us), and fill a warp with a short row
    // (100000 rows of 272: 25 / 32 us).  Short rows share a block, since starting a block takes about 1 ns of the GPU's time
    // (one row per block: 262144 rows of 1024 took 271 us, 100000 of 272 105), but no more than that needs: blocks of 128 threads
    // against 256, 32768 rows of 4096 60 / 61.5, behind SwiGLU 98 / 103, 1200 behind GELU 5.1 / 5.4, 100000 rows of 272 29 / 25.
    const int per = vecs <= 64 || (vecs <= 2 * kMaxThreads && p.rows <= 4 * sm_count()) ? 2 : 4;
    const int threads = static_cast<int>(((vecs + per - 1) / per + 31) / 32 * 32);
    const int block_threads = vecs <= 64 ? 256 : 128;
    const int rows_per_block = threads < block_threads ? block_threads / threads : 1;
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
