// Global 2-norm over a list of gradients, and their clipping (HBM-bound).
//
//   norm = sqrt(sum_i sum_j g_i[j]^2),   out_i = g_i * min(1, max_norm / (norm + 1e-6))
//
// Two launches: every CTA of the first writes one partial sum of squares, in double, into a workspace slot of its own;
// every CTA of the second adds up all slots in the same fixed order (so no atomics, and the same bits on every run) and
// scales its share of the elements.  A tensor list travels in the kernel parameter block, as in pointwise.cu.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "common.cuh"

#include <cuda_fp16.h>

namespace fp8gmm {
namespace {

constexpr int kThreads = 256;
constexpr int kTileElems = 8192;
constexpr int kMaxTensors = 320;
constexpr int kMaxGrid = 1024;  // workspace slots of one launch

struct GradDesc {
  const void* in;
  void* out;
  int64_t numel;
  int in_type, out_type;
};

struct GradArgs {
  int num;
  int tile_start[kMaxTensors + 1];
  GradDesc d[kMaxTensors];
};

__device__ __forceinline__ float load_elem(const void* p, int type, int64_t i) {
  if (type == FP8GMM_F32) return static_cast<const float*>(p)[i];
  if (type == FP8GMM_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_elem(void* p, int type, int64_t i, float v) {
  if (type == FP8GMM_F32) static_cast<float*>(p)[i] = v;
  else if (type == FP8GMM_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
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
  __syncthreads();
  return total;
}

// Squares in double: an fp32 square overflows above 1.8e19 and vanishes below 1e-23, both inside bf16's range.
__global__ void __launch_bounds__(kThreads) sum_squares_kernel(const __grid_constant__ GradArgs args, double* __restrict__ partials) {
  double sum = 0.0;
  const int tiles = args.tile_start[args.num];
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int t = upper_slot(args.tile_start, args.num, tile);
    const GradDesc& d = args.d[t];
    const int64_t base = static_cast<int64_t>(tile - args.tile_start[t]) * kTileElems;
    const int64_t end = min(base + kTileElems, d.numel);
    for (int64_t i = base + threadIdx.x; i < end; i += kThreads) {
      const double v = load_elem(d.in, d.in_type, i);
      sum += v * v;
    }
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
  const double total = total_of(partials, num_partials);
  if (threadIdx.x == 0) {
    if (sum != nullptr) *sum = total;
    if (norm != nullptr) *norm = static_cast<float>(sqrt(total));
  }
}

__global__ void __launch_bounds__(kThreads) clip_kernel(const __grid_constant__ GradArgs args, const double* __restrict__ sums,
                                                        int num_sums, float max_norm, float* __restrict__ norm) {
  const double n = sqrt(total_of(sums, num_sums));
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(n);
  const double c = static_cast<double>(max_norm) / (n + 1e-6);
  const float coef = c >= 1.0 ? 1.f : static_cast<float>(c);  // a NaN norm keeps its NaN
  const int tiles = args.tile_start[args.num];
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int t = upper_slot(args.tile_start, args.num, tile);
    const GradDesc& d = args.d[t];
    const int64_t base = static_cast<int64_t>(tile - args.tile_start[t]) * kTileElems;
    const int64_t end = min(base + kTileElems, d.numel);
    for (int64_t i = base + threadIdx.x; i < end; i += kThreads)
      store_elem(d.out, d.out_type, i, load_elem(d.in, d.in_type, i) * coef);
  }
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
int fill(GradArgs& args, const fp8gmm_grad_desc* descs, int i, int count) {
  args.num = 0;
  args.tile_start[0] = 0;
  for (; i < count && args.num < kMaxTensors; ++i) {
    const fp8gmm_grad_desc& t = descs[i];
    if (t.numel == 0) continue;
    const int64_t tiles = (t.numel + kTileElems - 1) / kTileElems;
    if (tiles + args.tile_start[args.num] > INT32_MAX) break;
    args.d[args.num] = {t.in, t.out, t.numel, t.in_type, t.out_type};
    args.tile_start[args.num + 1] = args.tile_start[args.num] + static_cast<int>(tiles);
    ++args.num;
  }
  return i;
}

int grid_of(const GradArgs& args) {
  const int cap = std::min(kMaxGrid, sm_count() * 4);
  return std::min(args.tile_start[args.num], cap);
}

// Partial sums of squares of all tensors into `partials`; *used = number of slots written.
int launch_sum_squares(const fp8gmm_grad_desc* descs, int count, double* partials, int slots, int* used, cudaStream_t s) {
  GradArgs args;
  *used = 0;
  for (int i = 0; i < count;) {
    i = fill(args, descs, i, count);
    if (args.num == 0) continue;
    const int grid = grid_of(args);
    FP8GMM_CHECK_ARG(*used + grid <= slots, "sum_squares: workspace too small");
    sum_squares_kernel<<<grid, kThreads, 0, s>>>(args, partials + *used);
    FP8GMM_CHECK_CUDA(cudaGetLastError());
    count_launch();
    *used += grid;
  }
  return FP8GMM_OK;
}

int launch_clip(const fp8gmm_grad_desc* descs, int count, const double* sums, int num_sums, float max_norm, float* norm, cudaStream_t s) {
  GradArgs args;
  for (int i = 0; i < count;) {
    i = fill(args, descs, i, count);
    if (args.num == 0) continue;
    clip_kernel<<<grid_of(args), kThreads, 0, s>>>(args, sums, num_sums, max_norm, norm);
    FP8GMM_CHECK_CUDA(cudaGetLastError());
    count_launch();
    norm = nullptr;
  }
  if (norm != nullptr) {  // nothing to clip: the norm is still wanted
    norm_kernel<<<1, kThreads, 0, s>>>(sums, num_sums, nullptr, norm);
    FP8GMM_CHECK_CUDA(cudaGetLastError());
    count_launch();
  }
  return FP8GMM_OK;
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
  return launches * kMaxGrid * sizeof(double);
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
  rc = launch_sum_squares(descs, count, static_cast<double*>(workspace), static_cast<int>(workspace_bytes / sizeof(double)), &used, s);
  if (rc != FP8GMM_OK) return rc;
  norm_kernel<<<1, kThreads, 0, s>>>(static_cast<const double*>(workspace), used, sum, norm);
  FP8GMM_CHECK_CUDA(cudaGetLastError());
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
  return launch_clip(descs, count, sum, 1, max_norm, norm, static_cast<cudaStream_t>(stream));
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
  rc = launch_sum_squares(descs, count, static_cast<double*>(workspace), static_cast<int>(workspace_bytes / sizeof(double)), &used, s);
  if (rc != FP8GMM_OK) return rc;
  return launch_clip(descs, count, static_cast<const double*>(workspace), used, max_norm, norm, s);
}

}  // extern "C"
