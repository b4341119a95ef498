// Rows of bf16 -> int8 codes with one fp32 scale per row, optionally gathered by the router's sort and behind the expert's
// activation (HBM-bound: two bytes read, one written per element; four read with SwiGLU).
//
//   v[r, :] = act(x[src(r), :]),  top = max_k |v[r, k]|,  scale[r] = top / 127,  code[r, k] = round_half_even(127 v[r, k] / top)
//
// The code is the correctly rounded quotient of the fp32 number v, not v * (1 / scale): with bf16 inputs 127 v / top is exactly
// half-way between two codes quite often (v = top / 2 already is), and a reciprocal's error would send such values either way.
// Without an activation t = 127 v is exact (8 + 7 significant bits), y = t * (1 / top) is off by less than 2 ulp and one residual
// step, y + (t - y top) / top with a fused multiply-add for the exact residual, gives the representable half-way values exactly;
// any other quotient of a 15-bit by an 8-bit number is further from half-way than fp32's rounding.  Behind an activation there are
// half-way quotients too (GELU returns its argument above 6), and v has 24 bits: see codes_of.  t and top are scaled by a power of
// two first, so that neither the reciprocal nor the product leaves fp32's range.
// A row of zeros has scale 0 and codes 0.  A row that holds an infinity or a NaN has scale NaN and codes 0: all its products
// come out NaN, no other row's do.
//
// Two kernels.  quantize_rows_kernel: a block for one row or several short ones, the row in registers between the maximum and the
// codes, so it is read once; 16-byte loads, 8-byte stores; 64 registers behind an activation (with 40 the values spill: 131 us
// instead of 116 for 32768 rows of 4096 behind SwiGLU).  quantize_long_rows_kernel: rows that are too long for that, or not
// aligned to 16 bytes, are walked twice (the second time out of L2 or L1).
#include "int8.cuh"

namespace fp8gmm {
namespace {

constexpr int kLongThreads = 256;
constexpr int kMaxThreads = 512;
constexpr int kMaxVecs = 4;              // 8-element vectors a thread holds: rows of up to 512 * 4 * 8 = 16384 elements
constexpr int kStatusBadIndex = FP8GMM_STATUS_BAD_INDEX;

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
// bound by its instructions as much as by HBM: 32768 rows of 4096 took 69 us with single ones and 61.5 with these.  (Behind an
// activation the special function unit is next, two operations an element at an eighth of the rate.)
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

// v = a / (1 + e), e = 2^p: exp2 and reciprocal of the special function unit (relative errors 2^-22 and 2^-23), then one
// residual step that takes the quotient to the rounding of v itself.  The sum is taken half as large: the reciprocal flushes
// subnormal results, and this keeps it normal up to p = 127; beyond, e is at most fp32's largest number and v comes out as 0.
// Against 64 bits 25 codes of 2 * 10^8 differ behind SiLU and 21 behind GELU (normal rows with a few large values), as many as
// with IEEE division and expf; without the residual steps here and in codes_of it was 772 behind GELU.  32768 rows of 4096 take
// 93 us behind GELU and 116 behind SwiGLU, 75 and 97 without those steps.  Tried: 2^p from a polynomial and the sum in two floats,
// 21 and 21 codes, but 141 and 155 us.
constexpr float kRound = 12582912.f;   // 1.5 * 2^23: adding it rounds to the nearest integer, ties to even, into the low bits
__device__ __forceinline__ Pair exp2_approx(Pair p) {
  const float2 x = split(p);
  return pair_of(exp2_approx(x.x), exp2_approx(x.y));
}
__device__ __forceinline__ Pair over_one_plus(Pair a, Pair e) {
  const float2 es = split(e);   // the smaller number, also of a NaN: those of `a` come back through the product with it
  const Pair minus_d = fma2(pair_of(fminf(es.x, 3.4028235e38f), fminf(es.y, 3.4028235e38f)), both(-0.5f), both(-0.5f));
  const float2 ds = split(minus_d);
  const Pair inv = pair_of(rcp_approx(-ds.x), rcp_approx(-ds.y)), half = mul2(a, both(0.5f)), v = mul2(half, inv);
  return fma2(fma2(v, minus_d, half), inv, v);
}
template <int kAct>
__device__ __forceinline__ Pair activated(Pair a, Pair b) {
  if constexpr (kAct == FP8GMM_ACT_SWIGLU) {
    // p = -a log2(e): log2(e) in 16 bits, whose product with a bf16 number is exact, and 2^x = 1 + x ln 2 for the rest
    constexpr float kHigh = 0x1.7154p0f, kRest = 7.0526075e-06f * 0.69314718f;
    const Pair e = exp2_approx(mul2(a, both(-kHigh)));
    return mul2(over_one_plus(a, fma2(e, mul2(a, both(-kRest)), e)), b);
  }
  if constexpr (kAct == FP8GMM_ACT_GELU) {
    // 0.5 (1 + tanh u) = 1 / (1 + exp(-2u)), without the cancellation of 1 + tanh u at
    // negative u; the power of two is -2u log2(e) = a (k + 0.044715 k a^2)
    constexpr float k = static_cast<float>(-2 * 0.79788456 * 1.4426950408889634), k3 = static_cast<float>(-2 * 0.79788456 * 1.4426950408889634 * 0.044715);
    return over_one_plus(a, exp2_approx(mul2(a, fma2(mul2(a, a), both(k3), both(k)))));
  }
  return a;
}

// Factors of one row: t = v * pre, y = t * inv, residuals against `top`; a residual of `limit` or more calls for a closer look.
struct RowScale {
  float pre, inv, top, limit, scale;
};
__device__ __forceinline__ RowScale row_scale(uint32_t top_bits) {
  RowScale s;
  const float top = __uint_as_float(top_bits), inf = __uint_as_float(0x7F800000u);
  if (top_bits >= 0x7F800000u) {          // infinity or NaN
    s = {0.f, 0.f, 0.f, inf, __uint_as_float(0x7FC00000u)};
  } else if (top_bits == 0u) {
    s = {0.f, 0.f, 0.f, inf, 0.f};
  } else {
    int e = 127 - static_cast<int>(top_bits >> 23);   // 2^e * top is in [1, 2) for normal numbers
    e = max(-126, min(e, 120));
    const float two_e = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
    s.pre = 127.f * two_e;
    s.top = top * two_e;
    s.inv = __frcp_rn(s.top);
    s.limit = 0.49999f * s.top;
    s.scale = __fdiv_rn(top, 127.f);
  }
  return s;
}
// max(a, |b|), NaN if either is
__device__ __forceinline__ float max_abs(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
  return r;
}

// The codes of a pair in the low bytes (kRound + code).  `worst` collects the largest residual |t - code top| behind an activation:
// t is off by up to 2^-24 of 127.5 top there, so a residual below 0.49999 top proves the code to be the nearest integer.
template <int kAct>
__device__ __forceinline__ uint2 codes_of(Pair v, const RowScale& s, float& worst) {
  const Pair t = mul2(v, both(s.pre));
  float2 r;
  if constexpr (kAct != FP8GMM_ACT_NONE) {
    const Pair z = fma2(t, both(s.inv), both(kRound));
    const float2 left = split(fma2(add2(z, both(-kRound)), both(-s.top), t));
    worst = max_abs(max_abs(worst, left.x), left.y);
    r = split(z);
  } else {
    const Pair y = mul2(t, both(s.inv));
    r = split(add2(fma2(fma2(y, both(-s.top), t), both(s.inv), y), both(kRound)));
  }
  return make_uint2(__float_as_uint(r.x), __float_as_uint(r.y));
}
// The code of a value whose vector of eight holds a residual of `limit` or more (one in 6000), from the quotient in 64 bits: 127 v
// has 31 bits and top 24, so its distance from half-way is 0 or far more than the quotient's rounding.
__device__ __forceinline__ uint32_t exact_code(float v, float top) {
  return static_cast<uint32_t>(__double2int_rn(__ddiv_rn(127.0 * static_cast<double>(v), static_cast<double>(top))));
}
__device__ __forceinline__ uint32_t exact_codes(Pair v, float top) {
  const float2 x = split(v);
  return (exact_code(x.x, top) & 0xFFu) | (exact_code(x.y, top) & 0xFFu) << 8;
}
__device__ __noinline__ uint2 exact_codes(Pair a, Pair b, Pair c, Pair d, float top) {
  return make_uint2(exact_codes(a, top) | exact_codes(b, top) << 16, exact_codes(c, top) | exact_codes(d, top) << 16);
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
__global__ void __launch_bounds__(kMaxThreads, kAct != FP8GMM_ACT_NONE ? 2 : kVecs == 2 ? 4 : 3) quantize_rows_kernel(const QuantRowsParams p) {
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
  const uint32_t top_bits = row_max(__float_as_uint(top), warp_max + threadIdx.y * (blockDim.x >> 5));
  const RowScale s = row_scale(top_bits);
  if (!live) return;
  if (threadIdx.x == 0) p.scales[r] = s.scale;
  const bool zero = s.pre == 0.f;
  uint2* out = reinterpret_cast<uint2*>(p.codes + r * p.codes_ld);
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    const int c = threadIdx.x + u * blockDim.x;
    if (c >= vecs) break;
    uint32_t q[2];
    float worst = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint2 a2 = codes_of<kAct>(v[u][2 * h], s, worst), b2 = codes_of<kAct>(v[u][2 * h + 1], s, worst);
      q[h] = zero ? 0u : __byte_perm(__byte_perm(a2.x, a2.y, 0x0040), __byte_perm(b2.x, b2.y, 0x0040), 0x5410);
    }
    out[c] = kAct != FP8GMM_ACT_NONE && worst >= s.limit ? exact_codes(v[u][0], v[u][1], v[u][2], v[u][3], __uint_as_float(top_bits)) : make_uint2(q[0], q[1]);
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
    top = row_max(top, warp_max[turn]);
    const RowScale s = row_scale(top);
    if (threadIdx.x == 0) p.scales[r] = s.scale;
    const bool zero = s.pre == 0.f;
    for (int64_t c = 2 * threadIdx.x; c < p.cols; c += 2 * kLongThreads) {
      const Pair v = activated_at(c);
      float worst = 0.f;
      uint2 q = codes_of<kAct>(v, s, worst);
      if (kAct != FP8GMM_ACT_NONE && worst >= s.limit) q = make_uint2(exact_code(split(v).x, __uint_as_float(top)), exact_code(split(v).y, __uint_as_float(top)));
      if (zero) q = make_uint2(0u, 0u);
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
    // against 256, 32768 rows of 4096 60 / 61.5, behind SwiGLU 116 / 121, 1200 behind GELU 6.0 / 6.5, 100000 rows of 272 29 / 25.
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
