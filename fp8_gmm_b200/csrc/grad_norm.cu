// Global 2-norm over a list of gradients, and their clipping (HBM-bound).
//
//   norm = sqrt(sum_i sum_j g_i[j]^2),   out_i = g_i * min(1, max_norm / (norm + 1e-6))
//
// Every CTA of the first launch writes one partial sum of squares, in double, into a workspace slot of its own; all slots are
// added up in the same fixed order (no atomics, the same bits on every run), by every CTA of the clipping launch while there are
// few, by a launch in between otherwise.  Clipping takes one tile of 8192 elements per CTA: a grid that stays resident and loops
// keeps loads and stores of all its CTAs in step and reached 5.6 TB/s where this reaches 6.9 (2 bytes read, 4 written per
// element).  A tensor list travels in the kernel parameter block, as in pointwise.cu.
// Squares: 8 elements are summed in fp32 and these sums added up in double.  An fp32 square overflows above 1.8e19 and loses
// bits below 1e-19, both inside bf16's range; a thread whose fp32 sum of 32 elements is not in [2^-100, inf) therefore adds
// them up again in double, out of registers (all zeros excepted, which empty experts leave).  (Eight fp32 additions are off by 4.5 *
// 2^-24 at most; with every square in double the norm of 1.4 G bf16 elements takes 573 us instead of 435.)  A clipping factor that is
// no normal fp32 number multiplies in double.
// Clipping walks the elements backwards: what the first one read last is still in L2, and its own results are stored
// so that they leave L2 first.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "dependent_launch.cuh"

#include <cuda_fp16.h>

namespace fp8gmm {
namespace {

constexpr int kThreads = 256;
constexpr int kPerThread = 32;                         // elements of a tile that a thread has in flight
constexpr int kTileElems = kThreads * kPerThread;      // 8192
// A thread handles kUnit neighbouring elements at a time: 8 (16 bytes) where everything is 16 bits wide, 4 where fp32 takes part,
// so that a warp's widest accesses are 512 contiguous bytes.
template <int kType, int kOther = kType>
constexpr int kUnitOf = kType == FP8GMM_F32 || kOther == FP8GMM_F32 ? 4 : 8;
constexpr int kMaxTensors = 320;
constexpr int kFewTensors = 24;  // lists up to this length travel in a parameter block of 1 KiB instead of 11
constexpr int kCtasPerSm = 4;
constexpr int kMaxGrid = 1024;  // workspace slots of one launch

struct GradDesc {
  const void* in;
  void* out;
  int64_t numel;
  int8_t in_type, out_type;
  int8_t shift;    // elements by which `in` lies behind a 16-byte boundary: tiles start on the boundary
  int8_t out_vec;  // `out` has 16-byte boundaries at the same elements
};

template <int kMax>
struct GradArgs {
  int num;
  int tile_start[kMax + 1];
  GradDesc d[kMax];
};

// kBytes contiguous bytes (8 or 16) as 32-bit words.
template <int kBytes>
__device__ __forceinline__ void load_words(const uint32_t* p, uint32_t* w) {
  if constexpr (kBytes == 16) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
  } else {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x, w[1] = x.y;
  }
}

// The raw bits of a thread's elements of a tile; those outside the tensor are 0.  Unit u holds elements
// first + u * kThreads * kUnit + [0, kUnit).  All loads are issued before the first use.
template <int kType, int kUnit>
struct Units {
  static constexpr int kCount = kPerThread / kUnit;
  static constexpr int kBytes = kUnit * (kType == FP8GMM_F32 ? 4 : 2);
  static constexpr int kWords = kBytes / 4;
  uint32_t w[kCount][kWords];

  __device__ __forceinline__ void load(const GradDesc& d, int64_t first) {
#pragma unroll
    for (int u = 0; u < kCount; ++u) {
      const int64_t i = first + u * (kThreads * kUnit);
      const uint32_t* p = reinterpret_cast<const uint32_t*>(static_cast<const char*>(d.in) + i * (kBytes / kUnit));
      if (i >= 0 && i + kUnit <= d.numel) {
        load_words<kBytes>(p, w[u]);
      } else {
#pragma unroll
        for (int h = 0; h < kWords; ++h) w[u][h] = 0u;
#pragma unroll
        for (int j = 0; j < kUnit; ++j)
          if (i + j >= 0 && i + j < d.numel) {
            if constexpr (kType == FP8GMM_F32) w[u][j] = p[j];
            else w[u][j / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[j]) << (16 * (j & 1));
          }
      }
    }
  }
  __device__ __forceinline__ void unpack(int u, float (&v)[kUnit]) const {
#pragma unroll
    for (int h = 0; h < kWords; ++h) {
      if constexpr (kType == FP8GMM_F32) {
        v[h] = __uint_as_float(w[u][h]);
      } else if constexpr (kType == FP8GMM_BF16) {
        v[2 * h] = bf16_lo(w[u][h]);
        v[2 * h + 1] = bf16_hi(w[u][h]);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[u][h]));
        v[2 * h] = f.x;
        v[2 * h + 1] = f.y;
      }
    }
  }
};

// Stores elements i + [0, kUnit), those that lie in the tensor.
template <int kType, int kUnit>
__device__ __forceinline__ void store_unit(const GradDesc& d, int64_t i, const float (&v)[kUnit]) {
  constexpr int kSize = kType == FP8GMM_F32 ? 4 : 2, kWords = kUnit * kSize / 4;
  uint32_t w[kWords];
#pragma unroll
  for (int h = 0; h < kWords; ++h) {
    if constexpr (kType == FP8GMM_F32) {
      w[h] = __float_as_uint(v[h]);
    } else if constexpr (kType == FP8GMM_BF16) {
      w[h] = pack_bf16x2(v[2 * h], v[2 * h + 1]);
    } else {
      const __half2 x = __floats2half2_rn(v[2 * h], v[2 * h + 1]);
      w[h] = *reinterpret_cast<const uint32_t*>(&x);
    }
  }
  uint32_t* p = reinterpret_cast<uint32_t*>(static_cast<char*>(d.out) + i * kSize);
  if (d.out_vec && i >= 0 && i + kUnit <= d.numel) {
    if constexpr (kWords == 4) st_stream16(p, make_uint4(w[0], w[1], w[2], w[3]));
    else st_stream8(p, make_uint2(w[0], w[1]));
  } else {
#pragma unroll
    for (int j = 0; j < kUnit; ++j)
      if (i + j >= 0 && i + j < d.numel) {
        if constexpr (kType == FP8GMM_F32) p[j] = w[j];
        else reinterpret_cast<uint16_t*>(p)[j] = static_cast<uint16_t>(w[j / 2] >> (16 * (j & 1)));
      }
  }
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double warp_sums[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  if ((threadIdx.x & 31) == 0) warp_sums[threadIdx.x >> 5] = v;
  __syncthreads();
  double total = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) total += warp_sums[w];
  return total;
}

// First element of the tile, counted from the 16-byte boundary at or in front of the tensor.
template <int kMax>
__device__ __forceinline__ int64_t tile_base(const GradArgs<kMax>& args, int t, int tile) {
  return static_cast<int64_t>(tile - args.tile_start[t]) * kTileElems - args.d[t].shift;
}

template <int kType>
__device__ __forceinline__ double tile_squares(const GradDesc& d, int64_t base) {
  constexpr int kUnit = kUnitOf<kType>;
  using X = Units<kType, kUnit>;
  X x;
  x.load(d, base + threadIdx.x * kUnit);
  float s[4] = {0.f, 0.f, 0.f, 0.f}, v[kUnit];   // eight elements each
#pragma unroll
  for (int u = 0; u < X::kCount; ++u) {
    x.unpack(u, v);
#pragma unroll
    for (int j = 0; j < kUnit; ++j) s[u * kUnit / 8] = fmaf(v[j], v[j], s[u * kUnit / 8]);
  }
  const float all = (s[0] + s[1]) + (s[2] + s[3]);
  // 2^-100 <= all < inf: no square overflowed, and what vanished is below 2^-45 of it
  if (all >= 7.9e-31f && all <= 3.4e38f) return (static_cast<double>(s[0]) + s[1]) + (static_cast<double>(s[2]) + s[3]);
  uint32_t any = 0;
#pragma unroll
  for (int u = 0; u < X::kCount; ++u)
#pragma unroll
    for (int h = 0; h < X::kWords; ++h) any |= x.w[u][h];
  double sum = 0.0;
  if (any != 0u) {
#pragma unroll
    for (int u = 0; u < X::kCount; ++u) {
      x.unpack(u, v);
#pragma unroll
      for (int j = 0; j < kUnit; ++j) sum = fma(static_cast<double>(v[j]), static_cast<double>(v[j]), sum);
    }
  }
  return sum;
}

template <int kMax>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) sum_squares_kernel(const __grid_constant__ GradArgs<kMax> args, double* __restrict__ partials) {
  let_dependents_start();
  double sum = 0.0;
  const int tiles = args.tile_start[args.num];
  int t = 0;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    while (args.tile_start[t + 1] <= tile) ++t;
    const GradDesc& d = args.d[t];
    const int64_t base = tile_base(args, t, tile);
    if (d.in_type == FP8GMM_BF16) sum += tile_squares<FP8GMM_BF16>(d, base);
    else if (d.in_type == FP8GMM_F32) sum += tile_squares<FP8GMM_F32>(d, base);
    else sum += tile_squares<FP8GMM_F16>(d, base);
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

__device__ __forceinline__ double total_of(const double* __restrict__ sums, int num_sums) {
  double v = 0.0;
  for (int i = threadIdx.x; i < num_sums; i += kThreads) v += sums[i];
  return block_sum(v);
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const double* __restrict__ partials, int num_partials,
                                                        double* __restrict__ sum, float* __restrict__ norm) {
  let_dependents_start();
  grid_dependency_wait();
  const double total = total_of(partials, num_partials);
  if (threadIdx.x == 0) {
    if (sum != nullptr) *sum = total;
    if (norm != nullptr) *norm = static_cast<float>(sqrt(total));
  }
}

template <int kIn, int kOut>
__device__ __forceinline__ void clip_tile(const GradDesc& d, int64_t base, float coef) {
  constexpr int kUnit = kUnitOf<kIn, kOut>;
  Units<kIn, kUnit> x;
  const int64_t first = base + threadIdx.x * kUnit;
  x.load(d, first);
#pragma unroll
  for (int u = 0; u < kPerThread / kUnit; ++u) {
    float v[kUnit];
    x.unpack(u, v);
#pragma unroll
    for (int j = 0; j < kUnit; ++j) v[j] *= coef;
    store_unit<kOut, kUnit>(d, first + u * (kThreads * kUnit), v);
  }
}
template <int kIn>
__device__ __forceinline__ void clip_tile(const GradDesc& d, int64_t base, float coef) {
  if (d.out_type == FP8GMM_BF16) clip_tile<kIn, FP8GMM_BF16>(d, base, coef);
  else if (d.out_type == FP8GMM_F32) clip_tile<kIn, FP8GMM_F32>(d, base, coef);
  else clip_tile<kIn, FP8GMM_F16>(d, base, coef);
}

__device__ __forceinline__ float load_one(const GradDesc& d, int64_t i) {
  if (d.in_type == FP8GMM_F32) return static_cast<const float*>(d.in)[i];
  if (d.in_type == FP8GMM_BF16) return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(d.in)[i]) << 16);
  return __half2float(static_cast<const __half*>(d.in)[i]);
}
// With a factor below fp32's normal range, where it would lose bits that ordinary results need (a norm of 1e41 and a limit of 1:
// elements of 1e38 become 1e-3): products in 64 bits, one element at a time.
__device__ __noinline__ void clip_tile_by_double(const GradDesc& d, int64_t base, double c) {
  for (int u = threadIdx.x; u < kTileElems; u += kThreads) {
    const int64_t i = base + u;
    if (i < 0 || i >= d.numel) continue;
    const float v = static_cast<float>(static_cast<double>(load_one(d, i)) * c);
    if (d.out_type == FP8GMM_F32) static_cast<float*>(d.out)[i] = v;
    else if (d.out_type == FP8GMM_BF16) static_cast<__nv_bfloat16*>(d.out)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(d.out)[i] = __float2half_rn(v);
  }
}

// One tile per CTA, from the last one to the first.
template <int kMax>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) clip_kernel(const __grid_constant__ GradArgs<kMax> args, const double* __restrict__ sums,
                                                                    int num_sums, float max_norm, float* __restrict__ norm) {
  const int tile = args.tile_start[args.num] - 1 - static_cast<int>(blockIdx.x);
  const int t = upper_slot(args.tile_start, args.num, tile);
  const GradDesc& d = args.d[t];
  const int64_t base = tile_base(args, t, tile);
  grid_dependency_wait();
  const double n = sqrt(num_sums == 1 ? *sums : total_of(sums, num_sums));
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(n);
  const double c = static_cast<double>(max_norm) / (n + 1e-6);
  const float coef = c >= 1.0 ? 1.f : static_cast<float>(c);  // a NaN norm keeps its NaN
  if (coef == 1.f && d.in == d.out) return;   // in place and within the limit: nothing changes
  if (c > 0.0 && c < 0x1p-126) clip_tile_by_double(d, base, c);
  else if (d.in_type == FP8GMM_BF16) clip_tile<FP8GMM_BF16>(d, base, coef);
  else if (d.in_type == FP8GMM_F32) clip_tile<FP8GMM_F32>(d, base, coef);
  else clip_tile<FP8GMM_F16>(d, base, coef);
}

int64_t elem_size(int type) { return type == FP8GMM_F32 ? 4 : 2; }
bool type_ok(int type) { return type == FP8GMM_BF16 || type == FP8GMM_F16 || type == FP8GMM_F32; }

int check_descs(const fp8gmm_grad_desc* descs, int count, const char* name, bool with_out) {
  FP8GMM_CHECK_ARG(count >= 0 && (count == 0 || descs != nullptr), "%s: bad descriptor list", name);
  for (int i = 0; i < count; ++i) {
    const fp8gmm_grad_desc& d = descs[i];
    FP8GMM_CHECK_ARG(d.numel >= 0, "%s: tensor %d has a negative size", name, i);
    FP8GMM_CHECK_ARG(type_ok(d.in_type) && (!with_out || type_ok(d.out_type)), "%s: tensor %d has an unknown type", name, i);
    FP8GMM_CHECK_ARG(d.numel <= (int64_t{1} << 42), "%s: tensor %d is too large", name, i);
    if (d.numel == 0) continue;
    FP8GMM_CHECK_ARG(d.in != nullptr && (!with_out || d.out != nullptr), "%s: tensor %d has a NULL pointer", name, i);
    FP8GMM_CHECK_ARG(reinterpret_cast<uintptr_t>(d.in) % elem_size(d.in_type) == 0 &&
                         (!with_out || reinterpret_cast<uintptr_t>(d.out) % elem_size(d.out_type) == 0),
                     "%s: tensor %d is not aligned to its type", name, i);
  }
  return FP8GMM_OK;
}

// An element that two list entries write, or that one entry writes while another reads it, would be scaled once, twice or
// in parts, by chance: refused.  An entry may read what it writes when both are the same array of the same type.
struct Range {
  uintptr_t begin, end;
  int owner;
};
int check_overlap(const fp8gmm_grad_desc* descs, int count, const char* name) {
  try {
    std::vector<Range> outs;
    outs.reserve(static_cast<size_t>(count));
    for (int i = 0; i < count; ++i)
      if (descs[i].numel > 0) {
        const uintptr_t b = reinterpret_cast<uintptr_t>(descs[i].out);
        outs.push_back({b, b + static_cast<uintptr_t>(descs[i].numel * elem_size(descs[i].out_type)), i});
      }
    std::sort(outs.begin(), outs.end(), [](const Range& x, const Range& y) { return x.begin < y.begin; });
    for (size_t j = 1; j < outs.size(); ++j)
      FP8GMM_CHECK_ARG(outs[j - 1].end <= outs[j].begin, "%s: outputs %d and %d share memory", name, outs[j - 1].owner, outs[j].owner);
    for (int i = 0; i < count; ++i) {
      const fp8gmm_grad_desc& d = descs[i];
      if (d.numel == 0 || (d.in == d.out && d.in_type == d.out_type)) continue;
      const uintptr_t b = reinterpret_cast<uintptr_t>(d.in), e = b + static_cast<uintptr_t>(d.numel * elem_size(d.in_type));
      // the first output that ends behind the input's first byte is the only one that can begin the overlap
      const auto it = std::upper_bound(outs.begin(), outs.end(), b, [](uintptr_t v, const Range& r) { return v < r.end; });
      FP8GMM_CHECK_ARG(it == outs.end() || it->begin >= e, "%s: input %d and output %d share memory", name, i, it->owner);
    }
  } catch (const std::bad_alloc&) {
    set_error("%s: out of host memory", name);
    return FP8GMM_INVALID_ARGUMENT;
  }
  return FP8GMM_OK;
}

// Fills `args` with the next descriptors, as many as one launch takes; returns the index of the first one left.
template <int kMax>
int fill(GradArgs<kMax>& args, const fp8gmm_grad_desc* descs, int i, int count) {
  args.num = 0;
  args.tile_start[0] = 0;
  for (; i < count && args.num < kMax; ++i) {
    const fp8gmm_grad_desc& t = descs[i];
    if (t.numel == 0) continue;
    const int size = static_cast<int>(elem_size(t.in_type));
    const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(t.in) % 16) / size;
    const int64_t tiles = (t.numel + shift + kTileElems - 1) / kTileElems;
    if (tiles + args.tile_start[args.num] > INT32_MAX) break;
    GradDesc& d = args.d[args.num];
    d = {t.in, t.out, t.numel, static_cast<int8_t>(t.in_type), static_cast<int8_t>(t.out_type), static_cast<int8_t>(shift), 0};
    // as integers: `out` may be a NULL that is not used
    if (type_ok(t.out_type)) d.out_vec = (reinterpret_cast<uintptr_t>(t.out) - static_cast<uintptr_t>(shift) * elem_size(t.out_type)) % 16 == 0;
    args.tile_start[args.num + 1] = args.tile_start[args.num] + static_cast<int>(tiles);
    ++args.num;
  }
  return i;
}

template <int kMax>
int grid_of(const GradArgs<kMax>& args) {
  const int cap = std::min(kMaxGrid, sm_count() * kCtasPerSm);
  return std::min(args.tile_start[args.num], cap);
}

// Partial sums of squares of all tensors into `partials`; *used = number of slots written.
template <int kMax>
int launch_sum_squares(const fp8gmm_grad_desc* descs, int count, double* partials, int slots, int* used, cudaStream_t s) {
  GradArgs<kMax> args;
  *used = 0;
  for (int i = 0; i < count;) {
    i = fill(args, descs, i, count);
    if (args.num == 0) continue;
    const int grid = grid_of(args);
    FP8GMM_CHECK_ARG(*used + grid <= slots, "sum_squares: workspace too small");
    sum_squares_kernel<kMax><<<grid, kThreads, 0, s>>>(args, partials + *used);
    FP8GMM_CHECK_CUDA(cudaGetLastError());
    count_launch();
    *used += grid;
  }
  return FP8GMM_OK;
}

template <int kMax>
int launch_clip(const fp8gmm_grad_desc* descs, int count, const double* sums, int num_sums, float max_norm, float* norm, bool after_sums, cudaStream_t s) {
  GradArgs<kMax> args;
  for (int i = 0; i < count;) {
    i = fill(args, descs, i, count);
    if (args.num == 0) continue;
    // the first launch may follow the sums directly; a later one writes what the one before it may not have read yet only if
    // an entry's output were another's input, which is refused
    FP8GMM_CHECK_CUDA(launch_dependent(clip_kernel<kMax>, args.tile_start[args.num], kThreads, 0, s, after_sums, args, sums, num_sums, max_norm, norm));
    count_launch();
    after_sums = false;
    norm = nullptr;
  }
  if (norm != nullptr) {  // nothing to clip: the norm is still wanted
    FP8GMM_CHECK_CUDA(launch_dependent(norm_kernel, 1, kThreads, 0, s, false, sums, num_sums, static_cast<double*>(nullptr), norm));
    count_launch();
  }
  return FP8GMM_OK;
}

int launch_sum_squares(const fp8gmm_grad_desc* descs, int count, void* workspace, size_t bytes, int* used, cudaStream_t s) {
  double* partials = static_cast<double*>(workspace);
  const int slots = static_cast<int>(bytes / sizeof(double));
  return count <= kFewTensors ? launch_sum_squares<kFewTensors>(descs, count, partials, slots, used, s)
                              : launch_sum_squares<kMaxTensors>(descs, count, partials, slots, used, s);
}
int launch_clip(const fp8gmm_grad_desc* descs, int count, const double* sums, int num_sums, float max_norm, float* norm, bool after_sums,
                cudaStream_t s) {
  return count <= kFewTensors ? launch_clip<kFewTensors>(descs, count, sums, num_sums, max_norm, norm, after_sums, s)
                              : launch_clip<kMaxTensors>(descs, count, sums, num_sums, max_norm, norm, after_sums, s);
}

int check_workspace(const void* workspace, size_t bytes, int count, const char* name) {
  FP8GMM_CHECK_ARG(workspace != nullptr && bytes >= fp8gmm_sum_squares_workspace_bytes(count) && reinterpret_cast<uintptr_t>(workspace) % 8 == 0,
                   "%s: the workspace needs %zu bytes, aligned to 8", name, fp8gmm_sum_squares_workspace_bytes(count));
  return FP8GMM_OK;
}

}  // namespace
}  // namespace fp8gmm

extern "C" {

size_t fp8gmm_sum_squares_workspace_bytes(int count) {
  using namespace fp8gmm;
  const size_t launches = count <= 0 ? 1 : (static_cast<size_t>(count) + kMaxTensors - 1) / kMaxTensors;
  return (launches * kMaxGrid + 1) * sizeof(double);   // a place for every CTA's sum, and for their total
}

int fp8gmm_multi_sum_squares(const fp8gmm_grad_desc* descs, int count, void* workspace, size_t workspace_bytes, double* sum,
                             float* norm, void* stream) {
  using namespace fp8gmm;
  int rc = check_descs(descs, count, "multi_sum_squares", false);
  if (rc != FP8GMM_OK) return rc;
  FP8GMM_CHECK_ARG(sum != nullptr || norm != nullptr, "multi_sum_squares: NULL output");
  rc = check_workspace(workspace, workspace_bytes, count, "multi_sum_squares");
  if (rc != FP8GMM_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int used = 0;
  rc = launch_sum_squares(descs, count, workspace, workspace_bytes, &used, s);
  if (rc != FP8GMM_OK) return rc;
  FP8GMM_CHECK_CUDA(launch_dependent(norm_kernel, 1, kThreads, 0, s, used > 0, static_cast<const double*>(workspace), used, sum, norm));
  count_launch();
  return FP8GMM_OK;
}

int fp8gmm_multi_clip(const fp8gmm_grad_desc* descs, int count, const double* sum, float max_norm, float* norm, void* stream) {
  using namespace fp8gmm;
  int rc = check_descs(descs, count, "multi_clip", true);
  if (rc != FP8GMM_OK) return rc;
  FP8GMM_CHECK_ARG(sum != nullptr, "multi_clip: NULL sum");
  FP8GMM_CHECK_ARG(max_norm >= 0.f, "multi_clip: max_norm must not be negative");
  rc = check_overlap(descs, count, "multi_clip");
  if (rc != FP8GMM_OK) return rc;
  return launch_clip(descs, count, sum, 1, max_norm, norm, false, static_cast<cudaStream_t>(stream));
}

int fp8gmm_multi_clip_grad_norm(const fp8gmm_grad_desc* descs, int count, float max_norm, void* workspace, size_t workspace_bytes,
                                float* norm, void* stream) {
  using namespace fp8gmm;
  int rc = check_descs(descs, count, "multi_clip_grad_norm", true);
  if (rc != FP8GMM_OK) return rc;
  FP8GMM_CHECK_ARG(max_norm >= 0.f, "multi_clip_grad_norm: max_norm must not be negative");
  rc = check_workspace(workspace, workspace_bytes, count, "multi_clip_grad_norm");
  if (rc != FP8GMM_OK) return rc;
  rc = check_overlap(descs, count, "multi_clip_grad_norm");
  if (rc != FP8GMM_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int used = 0;
  rc = launch_sum_squares(descs, count, workspace, workspace_bytes, &used, s);
  if (rc != FP8GMM_OK) return rc;
  double* sums = static_cast<double*>(workspace);
  if (used < std::min(kMaxGrid, sm_count() * kCtasPerSm)) return launch_clip(descs, count, sums, used, max_norm, norm, used > 0, s);
  // many tiles: one more launch (2 us) adds the partial sums up once instead of in every CTA
  FP8GMM_CHECK_CUDA(launch_dependent(norm_kernel, 1, kThreads, 0, s, true, sums, used, sums + used, static_cast<float*>(nullptr)));
  count_launch();
  return launch_clip(descs, count, sums + used, 1, max_norm, norm, true, s);
}

}  // extern "C"
