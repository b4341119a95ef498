// Grouped product of 8-bit integers with one scale per row (token) and per output channel (sm_100a, tcgen05 / TMEM).
//
//   C[r, n] = bf16( float( sum_k a[r, k] * b[g, n, k] ) * (a_scale[r] * b_scale[g, n]) ),   row r in group g
//
// The sum is an exact 32-bit integer (|a|, |b| <= 128 and K < 2^17), so every tile shape and every split of the contraction
// gives the same bits; the conversion to float, the product of the scales, the product with them and the final bf16 are the
// only roundings.
//
// The operands are swapped against gemm_sm100.cu: output channels are the M dimension of the MMA (TMEM lanes), rows the N
// dimension (TMEM columns).  A group of any number of rows then costs an MMA only as wide as its rows, and a warp's 32 lanes
// hold 32 neighbouring channels of one output row.
// Two kernels:
//   * int8_pair_kernel (many rows per group, tensor bound): persistent CTA pairs, tiles of 256 channels x up to 256 rows,
//     accumulators double-buffered in TMEM, results transposed through shared memory and written as 256-byte runs;
//   * int8_stream_kernel (few rows per group, bound by reading the weights): one tile of 128 channels x kT rows per CTA, the
//     contraction optionally split over a cluster whose CTAs add their partial sums through distributed shared memory.
// Group sizes come from the host (parameter block) or are read on the device; either way every CTA builds the prefix sums of
// rows and tiles in shared memory.  Waits on mbarriers are bounded as in gemm_sm100.cu.
#include <cstdlib>
#include <cstring>

#include "int8.cuh"
#include "sm100_ptx.cuh"

namespace fp8gmm {
namespace {

constexpr int kMaxGroups = 512;
constexpr int kStatusBadSizes = 0x400;   // group sizes that are negative or reach behind the last row
constexpr int kThreads = 192;            // TMA producer warp, MMA warp, four epilogue warps
constexpr int kChannels = 128;           // channels of one CTA's tile
constexpr int kBlockK = 128;             // bytes of contraction per stage: one 128-byte swizzle atom
constexpr int kWBytes = kChannels * kBlockK;

struct Int8GemmParams {
  CUtensorMap map_w;                     // weights (G*N, K), box 128 rows x 128 bytes
  CUtensorMap map_x;                     // codes (rows, K), box of the tile's rows (per CTA) x 128 bytes
  uint16_t* c;
  const float* a_scales;
  const float* b_scales;
  const int64_t* device_sizes;           // group sizes on the device, or NULL: row_start holds their prefix sums
  int* status;
  unsigned long long wait_ns;
  int num_groups, rows, n, k;
  int tile_rows, tiles_n, super_tiles;
  int row_start[kMaxGroups + 1];
};

// D[tmem] (+)= W[smem] X[smem]^T in 8-bit integers, issued by one thread.
template <int kCtas>
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t desc_w, uint64_t desc_x, uint32_t idesc, uint32_t accumulate) {
  if constexpr (kCtas == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_w), "l"(desc_x), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_w), "l"(desc_x), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Instruction descriptor of kind::i8: [4,6) D format (2 = s32), [7,10) / [10,13) A / B format (1 = signed), [17,23) N >> 3,
// [24,29) M >> 4; both operands K-major.
__device__ __forceinline__ uint32_t idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ uint32_t tmem_ld1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr) : "memory");
  return r;
}
__device__ __forceinline__ void st_cluster32(uint32_t cluster_addr, uint32_t v) {
  asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t ld_shared32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ uint16_t result_bf16(uint32_t acc, float scale) {
  const __nv_bfloat16 v = __float2bfloat16_rn(__fmul_rn(__int2float_rn(static_cast<int>(acc)), scale));
  return *reinterpret_cast<const uint16_t*>(&v);
}

// Prefix sums of rows and tiles over the groups, by one warp.  Sizes read on the device are cut off at the last row.
__device__ __forceinline__ void build_groups(const Int8GemmParams& p, int* row_start, int* tile_start, int lane) {
  long long rows = 0;
  int tiles = 0;
  bool bad = false;
  for (int g0 = 0; g0 < p.num_groups; g0 += 32) {
    const int g = g0 + lane;
    long long m = 0;
    if (g < p.num_groups) {
      if (p.device_sizes != nullptr) {
        const long long want = p.device_sizes[g];
        m = want < 0 ? 0 : want > p.rows ? p.rows : want;
        bad |= m != want;
      } else {
        m = p.row_start[g + 1] - p.row_start[g];
      }
    }
    long long incl = m;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xFFFFFFFFu, incl, o);
      if (lane >= o) incl += up;
    }
    const long long limit = p.rows;
    const int lo = static_cast<int>(min(rows + incl - m, limit)), hi = static_cast<int>(min(rows + incl, limit));
    bad |= rows + incl > limit;
    int t = (hi - lo + p.tile_rows - 1) / p.tile_rows * p.tiles_n;
    const int mine = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xFFFFFFFFu, t, o);
      if (lane >= o) t += up;
    }
    if (g < p.num_groups) {
      row_start[g] = lo;
      tile_start[g] = tiles + t - mine;
    }
    rows += __shfl_sync(0xFFFFFFFFu, incl, 31);
    tiles += __shfl_sync(0xFFFFFFFFu, t, 31);
  }
  if (lane == 0) {
    row_start[p.num_groups] = static_cast<int>(min(rows, static_cast<long long>(p.rows)));
    tile_start[p.num_groups] = tiles;
  }
  if (blockIdx.x == 0 && __any_sync(0xFFFFFFFFu, bad) && lane == 0) atomicOr(p.status, kStatusBadSizes);
}

struct Tile {
  int group, row0, rows, n0;
};
// Tiles of a group: super-rows of `super_tiles` row tiles, row tiles fastest inside one, so that the tiles in flight share
// weights and codes through L2.
__device__ __forceinline__ Tile decode_tile(const Int8GemmParams& p, const int* row_start, const int* tile_start, int tile, int channels) {
  Tile t;
  const int g = upper_slot(tile_start, p.num_groups, tile);
  const int local = tile - tile_start[g], m = row_start[g + 1] - row_start[g];
  const int row_tiles = (m + p.tile_rows - 1) / p.tile_rows;
  const int per_super = p.super_tiles * p.tiles_n;
  const int s = local / per_super, rem = local - s * per_super;
  const int h = min(p.super_tiles, row_tiles - s * p.super_tiles);
  const int mt = s * p.super_tiles + rem % h;
  t.group = g;
  t.n0 = rem / h * channels;
  t.row0 = row_start[g] + mt * p.tile_rows;
  t.rows = min(p.tile_rows, m - mt * p.tile_rows);
  return t;
}

// =============================================================================================
// Few rows per group: one tile of 128 channels x kT rows per CTA
// =============================================================================================
template <int kT>
struct StreamCfg {
  static constexpr int kXBytes = kT * kBlockK;
  static constexpr int kStageBytes = kWBytes + kXBytes;
  // two CTAs per SM, so that one streams weights while the other starts or ends: at most 110 KiB each
  static constexpr int kStages = 108 * 1024 / kStageBytes;
  static constexpr int kTmemCols = kT < 32 ? 32 : kT;
  static constexpr int kTableBytes = 2 * (kMaxGroups + 1) * 4;
  static constexpr int kSmemBytes = kStages * kStageBytes + 1024 + 256;
};

template <int kT>
__global__ void __launch_bounds__(kThreads, 2) int8_stream_kernel(const __grid_constant__ Int8GemmParams p, int splits) {
  using C = StreamCfg<kT>;
  constexpr int kStages = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t tiles_addr = (raw_addr + 1023u) & ~1023u;
  uint8_t* tiles_ptr = smem_raw + (tiles_addr - raw_addr);
  uint64_t* bars = reinterpret_cast<uint64_t*>(tiles_ptr + kStages * C::kStageBytes);
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (kStages + s); };
  const uint32_t done_bar = bar0 + 8u * (2 * kStages);
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_slot + 1);
  // the group table is needed for the decoding alone: it lies in the first stage, before any load goes there
  int* row_start = reinterpret_cast<int*>(tiles_ptr);
  int* tile_start = row_start + kMaxGroups + 1;
  static_assert(C::kTableBytes <= C::kStageBytes, "the group table has to fit into a stage");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  if (threadIdx.x == 32) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    prefetch_tensormap(&p.map_w);
    prefetch_tensormap(&p.map_x);
  }
  if (warp == 2) {
    tmem_alloc(smem_u32(tmem_base_slot), C::kTmemCols);
    tmem_relinquish();
  }
  if (warp == 0) build_groups(p, row_start, tile_start, lane);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_base_slot;
  const int tile = blockIdx.x / splits;
  const bool live = tile < tile_start[p.num_groups];      // the same for all CTAs of a cluster
  Tile t = {0, 0, 0, 0};
  if (live) t = decode_tile(p, row_start, tile_start, tile, kChannels);
  const int num_kb = (p.k + kBlockK - 1) / kBlockK;
  const int kb0 = num_kb * rank / splits, kb1 = live ? num_kb * (rank + 1) / splits : kb0;
  __syncthreads();                                        // everybody has read the table: loads may overwrite it
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {
      fence_async_smem();   // the table's generic-proxy writes come before the loads into the same memory
      const int yw = t.group * p.n + t.n0, first = min(kb1 - kb0, kStages);
      // weights do not depend on the kernel before this one (the quantisation of the rows): their first loads go ahead of it
      for (int i = 0; i < first; ++i) {
        mbar_expect_tx(full_bar(i), C::kStageBytes);
        tma_load_2d(tiles_addr + i * C::kStageBytes, &p.map_w, full_bar(i), (kb0 + i) * kBlockK, yw);
      }
      grid_dependency_wait();
      for (int i = 0; i < first; ++i)
        tma_load_2d(tiles_addr + i * C::kStageBytes + kWBytes, &p.map_x, full_bar(i), (kb0 + i) * kBlockK, t.row0);
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0 + first; kb < kb1 && ok; ++kb) {
        ok = mbar_wait(empty_bar(stage), phase, abort_flag, p.status, 0x1, p.wait_ns);
        if (ok) {
          const uint32_t sw = tiles_addr + stage * C::kStageBytes;
          mbar_expect_tx(full_bar(stage), C::kStageBytes);
          tma_load_2d(sw, &p.map_w, full_bar(stage), kb * kBlockK, yw);
          tma_load_2d(sw + kWBytes, &p.map_x, full_bar(stage), kb * kBlockK, t.row0);
        }
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && live) {
      const uint32_t idesc = idesc_i8(kChannels, kT);
      const uint64_t desc_w0 = make_smem_desc(tiles_addr), desc_x0 = make_smem_desc(tiles_addr + kWBytes);
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = mbar_wait(full_bar(stage), phase, abort_flag, p.status, 0x4, p.wait_ns);
        if (!ok) break;
        const uint64_t dw = desc_w0 + static_cast<uint64_t>(stage * (C::kStageBytes >> 4));
        const uint64_t dx = desc_x0 + static_cast<uint64_t>(stage * (C::kStageBytes >> 4));
#pragma unroll
        for (int k = 0; k < kBlockK / 32; ++k) umma_i8<1>(tmem_base, dw + 2 * k, dx + 2 * k, idesc, (kb != kb0 || k != 0) ? 1u : 0u);
        umma_commit(empty_bar(stage));
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (ok) umma_commit(done_bar);
    }
    __syncwarp();
  }

  const int quad = warp & 3;
  const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
  const int channel = t.n0 + quad * 32 + lane;
  const bool epilogue = warp >= 2 && live;
  const bool col_ok = channel < p.n;
  float sb = 0.f;
  if (epilogue) {
    grid_dependency_wait();
    if (col_ok) sb = p.b_scales[static_cast<int64_t>(t.group) * p.n + channel];
    if (lane == 0) ok = mbar_wait(done_bar, 0, abort_flag, p.status, 0x8, p.wait_ns);
    ok = __shfl_sync(0xFFFFFFFFu, ok, 0);
    tc_fence_after();
  }
  uint16_t* dst = p.c + static_cast<int64_t>(t.row0) * p.n + channel;
  if (splits == 1) {
    if (epilogue && ok) {
#pragma unroll
      for (int c0 = 0; c0 < kT; c0 += 16) {
        if (c0 >= t.rows) break;
        const float my_sa = lane < 16 && c0 + lane < t.rows ? p.a_scales[t.row0 + c0 + lane] : 0.f;
        uint32_t r[16];
        tmem_ld16(taddr + c0, r);
        tc_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float s = __fmul_rn(__shfl_sync(0xFFFFFFFFu, my_sa, j), sb);
          if (col_ok && c0 + j < t.rows) dst[static_cast<int64_t>(c0 + j) * p.n] = result_bf16(r[j], s);
        }
      }
    }
  } else {
    // Each CTA of the cluster finishes kT / splits of the rows: it receives the other CTAs' partial sums of them in its (now
    // idle) stages, [sender][row][channel].
    const int width = kT / splits;
    __syncwarp();
    cluster_sync_all();
    if (epilogue && ok) {
#pragma unroll
      for (int c0 = 0; c0 < kT; c0 += 16) {
        uint32_t r[16];
        tmem_ld16(taddr + c0, r);
        tc_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int to = (c0 + j) / width, row = c0 + j - to * width;
          if (to != rank) {
            const int slot = rank < to ? rank : rank - 1;
            const uint32_t at = tiles_addr + static_cast<uint32_t>(((slot * width + row) * kChannels + quad * 32 + lane) * 4);
            st_cluster32(map_to_cta(at, static_cast<uint32_t>(to)), r[j]);
          }
        }
      }
    }
    __syncwarp();
    cluster_sync_all();
    if (epilogue && ok) {
      for (int row = 0; row < width; ++row) {
        const int token = rank * width + row;
        if (token >= t.rows) break;
        uint32_t acc = tmem_ld1(taddr + token);
        tc_wait_ld();
        for (int slot = 0; slot < splits - 1; ++slot)
          acc += ld_shared32(tiles_addr + static_cast<uint32_t>(((slot * width + row) * kChannels + quad * 32 + lane) * 4));
        const float s = __fmul_rn(p.a_scales[t.row0 + token], sb);
        if (col_ok) dst[static_cast<int64_t>(token) * p.n] = result_bf16(acc, s);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {  // copies and MMAs still in flight get time to land before shared memory and TMEM go away
    const unsigned long long t0 = global_ns();
    while (global_ns() - t0 < 200000ull) {
    }
  }
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::kTmemCols);
  }
}

// =============================================================================================
// Many rows per group: persistent CTA pairs, 256 channels x up to 256 rows per tile
// =============================================================================================
struct PairCfg {
  static constexpr int kRows = 256;
  static constexpr int kStages = 6;
  static constexpr int kStageBytes = kWBytes + kRows / 2 * kBlockK;   // 32 KiB per CTA
  static constexpr int kTmemCols = 512;
  static constexpr int kStagingBytes = 2 * 32 * kChannels * 2;        // two boxes of 32 rows x 128 channels of bf16
  static constexpr int kScaleBytes = 2 * kRows * 4;
  static constexpr int kTableBytes = (2 * (kMaxGroups + 1) * 4 + 15) / 16 * 16;
  static constexpr int kSmemBytes = kStages * kStageBytes + kStagingBytes + kScaleBytes + kTableBytes + 1024 + 256;
};

__device__ __forceinline__ void epilogue_barrier() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) int8_pair_kernel(const __grid_constant__ Int8GemmParams p) {
  using C = PairCfg;
  constexpr int kStages = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t tiles_addr = (raw_addr + 1023u) & ~1023u;
  uint8_t* staging = smem_raw + (tiles_addr - raw_addr) + kStages * C::kStageBytes;
  float* scale_buf = reinterpret_cast<float*>(staging + C::kStagingBytes);
  int* row_start = reinterpret_cast<int*>(staging + C::kStagingBytes + C::kScaleBytes);
  int* tile_start = row_start + kMaxGroups + 1;
  uint64_t* bars = reinterpret_cast<uint64_t*>(staging + C::kStagingBytes + C::kScaleBytes + C::kTableBytes);
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (kStages + s); };
  auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * kStages + a); };
  auto tempty_bar = [&](int a) { return bar0 + 8u * (2 * kStages + 2 + a); };
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const bool leader = rank == 0;
  const int worker = blockIdx.x >> 1, num_workers = gridDim.x >> 1;

  if (threadIdx.x == 32) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), 8);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    prefetch_tensormap(&p.map_w);
    prefetch_tensormap(&p.map_x);
  }
  if (warp == 2) {
    tmem_alloc_pair(smem_u32(tmem_base_slot), C::kTmemCols);
    tmem_relinquish_pair();
  }
  if (warp == 0) build_groups(p, row_start, tile_start, lane);
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  grid_dependency_wait();
  const uint32_t tmem_base = *tmem_base_slot;
  const int total_tiles = tile_start[p.num_groups];
  const int num_kb = (p.k + kBlockK - 1) / kBlockK;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint32_t full0_leader = map_to_cta(full_bar(0), 0);
      for (int tile = worker; tile < total_tiles && ok; tile += num_workers) {
        const Tile t = decode_tile(p, row_start, tile_start, tile, 2 * kChannels);
        const int width = (t.rows + 31) & ~31;                       // columns of this tile's MMAs, half of them from each CTA
        const int yw = t.group * p.n + t.n0 + rank * kChannels, yx = t.row0 + rank * (width / 2);
        for (int kb = 0; kb < num_kb && ok; ++kb) {
          ok = mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, 0x1, p.wait_ns);
          if (ok) {
            const uint32_t sw = tiles_addr + stage * C::kStageBytes, bar = full0_leader + 8u * stage;
            if (leader) mbar_expect_tx(full_bar(stage), 2 * C::kStageBytes);   // both CTAs credit the leader's barrier
            tma_load_2d_pair(sw, &p.map_w, bar, kb * kBlockK, yw);
            tma_load_2d_pair(sw + kWBytes, &p.map_x, bar, kb * kBlockK, yx);
          }
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (leader && lane == 0) {
      const uint64_t desc_w0 = make_smem_desc(tiles_addr), desc_x0 = make_smem_desc(tiles_addr + kWBytes);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int tile = worker; tile < total_tiles && ok; tile += num_workers) {
        const Tile t = decode_tile(p, row_start, tile_start, tile, 2 * kChannels);
        const uint32_t idesc = idesc_i8(2 * kChannels, (t.rows + 31) & ~31);
        ok = mbar_wait(tempty_bar(acc), acc_phase ^ 1u, abort_flag, p.status, 0x2, p.wait_ns);
        if (!ok) break;
        tc_fence_after();
        const uint32_t tmem_d = tmem_base + static_cast<uint32_t>(acc * C::kRows);
        for (int kb = 0; kb < num_kb; ++kb) {
          ok = mbar_wait(full_bar(stage), phase, abort_flag, p.status, 0x4, p.wait_ns);
          if (!ok) break;
          const uint64_t dw = desc_w0 + static_cast<uint64_t>(stage * (C::kStageBytes >> 4));
          const uint64_t dx = desc_x0 + static_cast<uint64_t>(stage * (C::kStageBytes >> 4));
#pragma unroll
          for (int k = 0; k < kBlockK / 32; ++k) umma_i8<2>(tmem_d, dw + 2 * k, dx + 2 * k, idesc, (kb | k) != 0 ? 1u : 0u);
          umma_commit_pair(empty_bar(stage));
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        umma_commit_pair(tfull_bar(acc));
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
    }
    __syncwarp();
  } else {
    const int quad = warp & 3, thread = threadIdx.x - 64;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int tile = worker; tile < total_tiles; tile += num_workers) {
      const Tile t = decode_tile(p, row_start, tile_start, tile, 2 * kChannels);
      const int n0 = t.n0 + rank * kChannels;
      const int channel = n0 + quad * 32 + lane;
      const float sb = channel < p.n ? p.b_scales[static_cast<int64_t>(t.group) * p.n + channel] : 0.f;
      float* scales = scale_buf + acc * C::kRows;
      for (int i = thread; i < t.rows; i += 128) scales[i] = p.a_scales[t.row0 + i];
      if (lane == 0 && ok) ok = mbar_wait(tfull_bar(acc), acc_phase, abort_flag, p.status, 0x8, p.wait_ns);
      ok = __shfl_sync(0xFFFFFFFFu, ok, 0);
      epilogue_barrier();     // the scales are there; every warp goes on, also one that gave up, as the barriers count all four
      tc_fence_after();
      const uint32_t taddr = tmem_base + static_cast<uint32_t>(acc * C::kRows) + (static_cast<uint32_t>(quad * 32) << 16);
      for (int c0 = 0; c0 < t.rows; c0 += 32) {
        uint16_t* box = reinterpret_cast<uint16_t*>(staging) + ((c0 >> 5) & 1) * 32 * kChannels;
        if (ok) {
          uint32_t r[32];
          tmem_ld32(taddr + c0, r);
          tc_wait_ld();
          uint16_t* mine = box + quad * 32 + lane;
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 sa = *reinterpret_cast<const float4*>(scales + c0 + j);
            mine[(j + 0) * kChannels] = result_bf16(r[j + 0], __fmul_rn(sa.x, sb));
            mine[(j + 1) * kChannels] = result_bf16(r[j + 1], __fmul_rn(sa.y, sb));
            mine[(j + 2) * kChannels] = result_bf16(r[j + 2], __fmul_rn(sa.z, sb));
            mine[(j + 3) * kChannels] = result_bf16(r[j + 3], __fmul_rn(sa.w, sb));
          }
        }
        epilogue_barrier();
        // 16 threads write the 256 bytes of a row; the box is free again after the next barrier
        const int chunk = thread & 15;
        if (ok && n0 + chunk * 8 < p.n) {
#pragma unroll
          for (int it = 0; it < 4; ++it) {
            const int row = it * 8 + (thread >> 4);
            if (c0 + row < t.rows)
              *reinterpret_cast<uint4*>(p.c + static_cast<int64_t>(t.row0 + c0 + row) * p.n + n0 + chunk * 8) =
                  *reinterpret_cast<const uint4*>(box + row * kChannels + chunk * 8);
          }
        }
      }
      epilogue_barrier();     // the last box is read before the next tile writes into it
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(map_to_cta(tempty_bar(acc), 0));
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
  }
  tc_fence_before();
  cluster_sync_all();
  if (*abort_flag) {
    const unsigned long long t0 = global_ns();
    while (global_ns() - t0 < 200000ull) {
    }
  }
  cluster_sync_all();   // a CTA must not leave while its peer can still touch its shared memory or barriers
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, C::kTmemCols);
  }
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
// (rows x cols) bytes, row pitch cols, box of box_rows x 128 bytes, SWIZZLE_128B.
int encode_rows(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int box_rows) {
  auto fn = get_encode_fn();
  if (!fn) {
    set_error("cuTensorMapEncodeTiled is not available from this driver");
    return FP8GMM_CUDA_ERROR;
  }
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(cols)};
  const cuuint32_t box[2] = {kBlockK, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t elem[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed with %d (base %p, rows %lld, cols %lld)", static_cast<int>(r), base, (long long)rows, (long long)cols);
    return FP8GMM_CUDA_ERROR;
  }
  return FP8GMM_OK;
}

// Process-wide override for tests (fp8gmm_set_int8_variant): 0 = chosen per call.
int g_tile_rows = 0, g_splits = 0;

template <typename... Args>
int launch(void (*kernel)(Args...), int grid, int cluster, int smem, cudaStream_t s, bool early, Args... args) {
  FP8GMM_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  if (early) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = cluster;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  cfg.attrs = attr;
  FP8GMM_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
  count_launch();
  return FP8GMM_OK;
}

template <int kT>
int launch_stream(Int8GemmParams& p, int64_t row_tiles, int splits, cudaStream_t s, bool early) {
  const int64_t grid = row_tiles * p.tiles_n * splits;
  FP8GMM_CHECK_ARG(grid <= INT32_MAX, "int8_grouped_gemm: problem too large");
  return launch<Int8GemmParams, int>(int8_stream_kernel<kT>, static_cast<int>(grid), splits, StreamCfg<kT>::kSmemBytes, s, early, p, splits);
}

}  // namespace
// Argument checks; nothing is launched and no CUDA call made.
int int8_gemm_check(const fp8gmm_int8_gemm_args* a) {
  FP8GMM_CHECK_ARG(a != nullptr, "int8_grouped_gemm: NULL arguments");
  FP8GMM_CHECK_ARG(a->num_groups >= 0 && a->num_groups <= kMaxGroups, "int8_grouped_gemm: num_groups %d outside [0, %d]", a->num_groups, kMaxGroups);
  FP8GMM_CHECK_ARG(a->n > 0 && a->k > 0 && a->n % 16 == 0 && a->k % 16 == 0, "int8_grouped_gemm: N (%lld) and K (%lld) must be positive multiples of 16",
                   (long long)a->n, (long long)a->k);
  FP8GMM_CHECK_ARG(a->k < (1 << 17), "int8_grouped_gemm: K = %lld could overflow the 32-bit sums (K < 131072)", (long long)a->k);
  FP8GMM_CHECK_ARG(a->n <= INT32_MAX / (a->num_groups > 0 ? a->num_groups : 1) - 1024, "int8_grouped_gemm: too many weight rows");
  FP8GMM_CHECK_ARG(a->rows >= 0 && a->rows <= INT32_MAX - 1024, "int8_grouped_gemm: bad number of rows");
  FP8GMM_CHECK_ARG(a->num_groups == 0 || (a->m_sizes != nullptr) != (a->device_m_sizes != nullptr),
                   "int8_grouped_gemm: group sizes are given on the host or on the device, not both");
  int64_t sum = 0;
  for (int g = 0; a->m_sizes != nullptr && g < a->num_groups; ++g) {
    const int64_t m = a->m_sizes[g];
    FP8GMM_CHECK_ARG(m >= 0 && m <= a->rows - sum, "int8_grouped_gemm: group %d has a bad size of %lld", g, (long long)m);
    sum += m;
  }
  FP8GMM_CHECK_ARG(a->m_sizes == nullptr || sum == a->rows, "int8_grouped_gemm: the group sizes sum to %lld, not to the %lld rows",
                   (long long)sum, (long long)a->rows);
  if (a->rows == 0 || a->num_groups == 0) return FP8GMM_OK;
  FP8GMM_CHECK_ARG(a->a && a->b && a->c && a->a_scales && a->b_scales, "int8_grouped_gemm: NULL pointer");
  FP8GMM_CHECK_ARG((reinterpret_cast<uintptr_t>(a->a) | reinterpret_cast<uintptr_t>(a->b) | reinterpret_cast<uintptr_t>(a->c)) % 16 == 0,
                   "int8_grouped_gemm: operand pointers must be 16-byte aligned");
  return FP8GMM_OK;
}

int int8_gemm_launch(const fp8gmm_int8_gemm_args* a, void* stream, bool after_quantize) {
  int rc = int8_gemm_check(a);
  if (rc != FP8GMM_OK || a->rows == 0 || a->num_groups == 0) return rc;
  Int8GemmParams p;
  memset(&p, 0, sizeof(p));
  for (int g = 0; a->m_sizes != nullptr && g < a->num_groups; ++g) p.row_start[g + 1] = p.row_start[g] + static_cast<int>(a->m_sizes[g]);
  p.c = static_cast<uint16_t*>(a->c);
  p.a_scales = a->a_scales;
  p.b_scales = a->b_scales;
  p.device_sizes = a->device_m_sizes;
  p.num_groups = a->num_groups;
  p.rows = static_cast<int>(a->rows);
  p.n = static_cast<int>(a->n);
  p.k = static_cast<int>(a->k);
  p.wait_ns = gemm_wait_limit_ns();
  p.status = device_status_word();
  FP8GMM_CHECK_ARG(p.status != nullptr, "int8_grouped_gemm: cannot resolve the device status word");
  // The rule goes by the mean rows of a group that can have any, so that sizes on the host and on the device take the same path.
  const int groups = p.rows < p.num_groups ? p.rows : p.num_groups;
  const int mean = (p.rows + groups - 1) / groups;
  int tile_rows = g_tile_rows;
  if (tile_rows == 0) tile_rows = mean <= 16 ? 16 : mean <= 32 ? 32 : mean <= 64 ? 64 : mean <= 128 ? 128 : 256;
  p.tile_rows = tile_rows;
  rc = encode_rows(&p.map_w, a->b, a->num_groups * a->n, a->k, kChannels);
  if (rc != FP8GMM_OK) return rc;
  rc = encode_rows(&p.map_x, a->a, a->rows, a->k, tile_rows == 256 ? 128 : tile_rows);
  if (rc != FP8GMM_OK) return rc;
  // each group adds at most one partial row tile to rows / tile_rows
  const int64_t row_tiles = p.rows / tile_rows + groups;
  const int channels = tile_rows == 256 ? 2 * kChannels : kChannels;
  p.tiles_n = (p.n + channels - 1) / channels;
  FP8GMM_CHECK_ARG(row_tiles * p.tiles_n <= INT32_MAX / 2, "int8_grouped_gemm: problem too large");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (tile_rows == 256) {
    p.super_tiles = (p.k > 8192 ? 2048 : 4096) / PairCfg::kRows;
    int sms = sm_count() / 2;
    const int64_t most = row_tiles * p.tiles_n;
    return launch<Int8GemmParams>(int8_pair_kernel, 2 * static_cast<int>(most < sms ? most : sms), 1, PairCfg::kSmemBytes, s, after_quantize, p);
  }
  p.super_tiles = INT32_MAX / 2 / p.tiles_n;   // row tiles fastest: the CTAs that share weights run side by side
  int splits = g_splits;
  const int num_kb = (p.k + kBlockK - 1) / kBlockK;
  if (splits == 0) {
    splits = 1;
    const int64_t tiles = row_tiles * p.tiles_n;
    while (splits < 8 && tiles * splits < 2 * sm_count() && num_kb >= 8 * splits) splits *= 2;
  }
  while (splits > num_kb || splits > tile_rows) splits /= 2;
  switch (tile_rows) {
    case 16: return launch_stream<16>(p, row_tiles, splits, s, after_quantize);
    case 32: return launch_stream<32>(p, row_tiles, splits, s, after_quantize);
    case 64: return launch_stream<64>(p, row_tiles, splits, s, after_quantize);
    default: return launch_stream<128>(p, row_tiles, splits, s, after_quantize);
  }
}
}  // namespace fp8gmm

extern "C" {

int fp8gmm_set_int8_variant(int tile_rows, int splits) {
  using namespace fp8gmm;
  FP8GMM_CHECK_ARG(tile_rows == 0 || tile_rows == 16 || tile_rows == 32 || tile_rows == 64 || tile_rows == 128 || tile_rows == 256,
                   "set_int8_variant: tile_rows must be 0, 16, 32, 64, 128 or 256");
  FP8GMM_CHECK_ARG(splits == 0 || splits == 1 || splits == 2 || splits == 4 || splits == 8, "set_int8_variant: splits must be 0, 1, 2, 4 or 8");
  g_tile_rows = tile_rows;
  g_splits = splits;
  return FP8GMM_OK;
}

int fp8gmm_int8_grouped_gemm(const fp8gmm_int8_gemm_args* a, void* stream) { return fp8gmm::int8_gemm_launch(a, stream, false); }

int fp8gmm_int8_linear(const fp8gmm_quantize_rows_args* q, const fp8gmm_int8_gemm_args* g, void* stream) {
  FP8GMM_CHECK_ARG(q != nullptr && g != nullptr, "int8_linear: NULL arguments");
  FP8GMM_CHECK_ARG(q->codes == g->a && q->scales == g->a_scales && q->rows == g->rows && q->cols == g->k,
                   "int8_linear: the product has to take the codes, scales, rows and columns of the quantisation");
  int rc = fp8gmm::int8_gemm_check(g);   // before anything is launched
  if (rc != FP8GMM_OK) return rc;
  rc = fp8gmm_quantize_rows_int8(q, stream);
  return rc != FP8GMM_OK ? rc : fp8gmm::int8_gemm_launch(g, stream, q->rows > 0);
}

}  // extern "C"
