// Grouped product of 8-bit integers with one scale per row (token) and per output channel.
//
//   C[r, n] = bf16( float( sum_k a[r, k] * b[g, n, k] ) * (a_scale[r] * b_scale[g, n]) ),   row r in group g
//
// The sum is an exact 32-bit integer (|a|, |b| <= 128 and K < 2^17), so every tile shape and every split of the contraction
// gives the same bits; the conversion to float, the product of the scales and the final bf16 are the only roundings.
#include "common.cuh"

namespace fp8gmm {
namespace {

constexpr int kMaxGroups = 512;
constexpr int kStatusBadSizes = 0x400;   // group sizes that are negative or reach behind the last row
constexpr int kTile = 64, kStepK = 64, kThreads = 256;

struct Int8GemmParams {
  const int8_t* a;
  const int8_t* b;
  uint16_t* c;
  const float* a_scales;
  const float* b_scales;
  const int64_t* device_sizes;        // group sizes on the device, or NULL: row_start holds their prefix sums
  int num_groups;
  int rows, n, k;
  int* status;
  int row_start[kMaxGroups + 1];
};

// One CTA per (row tile, channel tile); the row tiles are numbered group by group.
__global__ void __launch_bounds__(kThreads) int8_gemm_kernel(const __grid_constant__ Int8GemmParams p) {
  __shared__ int32_t as[kTile][kStepK / 4 + 1], bs[kTile][kStepK / 4 + 1];
  __shared__ int sh_group, sh_row0, sh_rows;
  if (threadIdx.x == 0) {
    int tile = blockIdx.x, row = 0, g = 0, found = -1, m = 0;
    for (; g < p.num_groups; ++g) {
      m = p.row_start[g + 1] - p.row_start[g];
      if (p.device_sizes != nullptr) {
        const int64_t want = p.device_sizes[g];
        m = static_cast<int>(want < 0 ? 0 : want > p.rows - row ? p.rows - row : want);
        if (m != want) atomicOr(p.status, kStatusBadSizes);
      }
      const int tiles = (m + kTile - 1) / kTile;
      if (tile < tiles) {
        found = g;
        break;
      }
      tile -= tiles;
      row += m;
    }
    sh_group = found;
    sh_row0 = row + tile * kTile;
    sh_rows = min(kTile, m - tile * kTile);
  }
  __syncthreads();
  if (sh_group < 0) return;
  const int64_t row0 = sh_row0, n0 = static_cast<int64_t>(blockIdx.y) * kTile;
  const int rows = sh_rows, cols = min(static_cast<int64_t>(kTile), p.n - n0);
  const int8_t* b = p.b + (static_cast<int64_t>(sh_group) * p.n + n0) * p.k;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < p.k; k0 += kStepK) {
    for (int i = threadIdx.x; i < kTile * kStepK / 4; i += kThreads) {
      const int r = i / (kStepK / 4), c = i % (kStepK / 4);
      const bool in = k0 + 4 * c < p.k;
      as[r][c] = in && r < rows ? *reinterpret_cast<const int32_t*>(p.a + (row0 + r) * p.k + k0 + 4 * c) : 0;
      bs[r][c] = in && r < cols ? *reinterpret_cast<const int32_t*>(b + static_cast<int64_t>(r) * p.k + k0 + 4 * c) : 0;
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kStepK / 4; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(as[ty + 16 * i][c], bs[tx + 16 * j][c], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = ty + 16 * i, n = tx + 16 * j;
      if (r < rows && n < cols) {
        const float s = p.a_scales[row0 + r] * p.b_scales[static_cast<int64_t>(sh_group) * p.n + n0 + n];
        const __nv_bfloat16 v = __float2bfloat16_rn(static_cast<float>(acc[i][j]) * s);
        p.c[(row0 + r) * p.n + n0 + n] = *reinterpret_cast<const uint16_t*>(&v);
      }
    }
}

}  // namespace
}  // namespace fp8gmm

extern "C" {

int fp8gmm_int8_grouped_gemm(const fp8gmm_int8_gemm_args* a, void* stream) {
  using namespace fp8gmm;
  FP8GMM_CHECK_ARG(a != nullptr, "int8_grouped_gemm: NULL arguments");
  FP8GMM_CHECK_ARG(a->num_groups >= 0 && a->num_groups <= kMaxGroups, "int8_grouped_gemm: num_groups %d outside [0, %d]", a->num_groups, kMaxGroups);
  FP8GMM_CHECK_ARG(a->n > 0 && a->k > 0 && a->n % 16 == 0 && a->k % 16 == 0, "int8_grouped_gemm: N (%lld) and K (%lld) must be positive multiples of 16",
                   (long long)a->n, (long long)a->k);
  FP8GMM_CHECK_ARG(a->k < (1 << 17), "int8_grouped_gemm: K = %lld could overflow the 32-bit sums (K < 131072)", (long long)a->k);
  FP8GMM_CHECK_ARG(a->n <= INT32_MAX / (a->num_groups > 0 ? a->num_groups : 1) - 1024, "int8_grouped_gemm: too many weight rows");
  FP8GMM_CHECK_ARG(a->rows >= 0 && a->rows <= INT32_MAX - 1024, "int8_grouped_gemm: bad number of rows");
  FP8GMM_CHECK_ARG(a->num_groups == 0 || (a->m_sizes != nullptr) != (a->device_m_sizes != nullptr),
                   "int8_grouped_gemm: group sizes are given on the host or on the device, not both");
  Int8GemmParams p;
  p.row_start[0] = 0;
  for (int g = 0; g < a->num_groups; ++g) {
    const int64_t m = a->m_sizes != nullptr ? a->m_sizes[g] : 0;
    FP8GMM_CHECK_ARG(m >= 0 && m <= a->rows - p.row_start[g], "int8_grouped_gemm: group %d has a bad size of %lld", g, (long long)m);
    p.row_start[g + 1] = p.row_start[g] + static_cast<int>(m);
  }
  FP8GMM_CHECK_ARG(a->m_sizes == nullptr || p.row_start[a->num_groups] == a->rows, "int8_grouped_gemm: the group sizes sum to %d, not to the %lld rows",
                   p.row_start[a->num_groups], (long long)a->rows);
  if (a->rows == 0 || a->num_groups == 0) return FP8GMM_OK;
  FP8GMM_CHECK_ARG(a->a && a->b && a->c && a->a_scales && a->b_scales, "int8_grouped_gemm: NULL pointer");
  FP8GMM_CHECK_ARG((reinterpret_cast<uintptr_t>(a->a) | reinterpret_cast<uintptr_t>(a->b) | reinterpret_cast<uintptr_t>(a->c)) % 16 == 0,
                   "int8_grouped_gemm: operand pointers must be 16-byte aligned");
  p.a = static_cast<const int8_t*>(a->a);
  p.b = static_cast<const int8_t*>(a->b);
  p.c = static_cast<uint16_t*>(a->c);
  p.a_scales = a->a_scales;
  p.b_scales = a->b_scales;
  p.device_sizes = a->device_m_sizes;
  p.num_groups = a->num_groups;
  p.rows = static_cast<int>(a->rows);
  p.n = static_cast<int>(a->n);
  p.k = static_cast<int>(a->k);
  p.status = device_status_word();
  FP8GMM_CHECK_ARG(p.status != nullptr, "int8_grouped_gemm: cannot resolve the device status word");
  // each group adds at most one partial row tile to rows / kTile
  const int row_tiles = (p.rows + kTile - 1) / kTile + p.num_groups;
  const dim3 grid(row_tiles, (p.n + kTile - 1) / kTile);
  FP8GMM_CHECK_ARG(grid.y <= 65535, "int8_grouped_gemm: N too large");
  int8_gemm_kernel<<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  FP8GMM_CHECK_CUDA(cudaGetLastError());
  count_launch();
  return FP8GMM_OK;
}

}  // extern "C"
