// Grouped product of 8-bit integers with one scale per row (token) and per output channel (sm_100a, tcgen05 / TMEM).
//
//   C[r, n] = bf16( float( sum_k a[r, k] * b[g, n, k] ) * (a_scale[r] * b_scale[g, n]) ),   row r in group g
//
// The sum is an exact 32-bit integer (|a|, |b| <= 128 and K < 2^17), so every tile shape and every split of the contraction
// gives the same bits; the conversion to float, the product of the scales, the product with them and the final bf16 are the
// only roundings.  Where the product of the two scales leaves fp32's normal range the three factors are multiplied in 64 bits.
//
// The operands are swapped against gemm_sm100.cu: output channels are the M dimension of the MMA (TMEM lanes), rows the N
// dimension (TMEM columns).  A group of any number of rows then costs an MMA only as wide as its rows, and a warp's 32 lanes
// hold 32 neighbouring channels of one output row.
//   * Persistent CTA pairs (cta_group::2): a tile is 256 channels x up to 128 or 256 rows; each CTA loads its half of the channels'
//     weights and half of the tile's rows, 256 contraction bytes per stage, into a ring of 4 or 3 stages.  Where such tiles would
//     keep less than half of the GPU loading weights (few experts, few channels, few rows), a tile is 128 channels: the MMA stays
//     256 wide and its other rows, whatever lies in shared memory behind the weights, are not looked at.
//   * Accumulators are double-buffered in TMEM.  A chunk of 32 rows is read as 16 x 8 fragments, transposed by stmatrix into a
//     box in shared memory and written as 256-byte runs; two groups of four warps take the chunks in turns.  This bounds products
//     with short contractions (8 x 4096 rows, 28672 channels, 512 contraction bytes, 1.9 GB written: 560 us; with one group that
//     stored 2 bytes per lane into the box 1123, with two 787, with fragments and stmatrix 690, with the arrival that does not
//     wait for the stores 599, with the rows' addresses carried along 560, with the look at the scales' sizes 570; HBM's floor is 308).  With 4096 contraction bytes it
//     is hidden behind the MMAs.
// Group sizes come from the host (parameter block) or are read on the device; either way every CTA builds the prefix sums of
// rows and tiles in shared memory.  Waits on mbarriers are bounded as in gemm_sm100.cu.
#include <atomic>
#include <cstring>

#include "int8.cuh"
#include "sm100_ptx.cuh"

namespace fp8gmm {
namespace {

constexpr int kMaxGroups = 512;
constexpr int kStatusBadSizes = FP8GMM_STATUS_BAD_SIZES;   // group sizes that are negative or reach behind the last row
constexpr int kThreads = 320;            // TMA producer warp, MMA warp, two groups of four epilogue warps
constexpr int kChannels = 128;           // channels of one CTA's half of the MMA
constexpr int kAtomK = 128;              // bytes of contraction in one box: a 128-byte swizzle atom
constexpr int kAtoms = 2;                // boxes along the contraction per stage
constexpr int kBlockK = kAtoms * kAtomK;
constexpr int kBoxPitch = kChannels * 2 + 16;   // bytes of a row in the epilogue's box: the 16-byte pieces of eight rows lie in different banks

struct Int8GemmParams {
  CUtensorMap map_w;                     // weights (G*N, K), box of `channels` rows x 128 bytes
  CUtensorMap map_x[4];                  // codes (rows, K), boxes of 16, 32, 64 and 128 rows x 128 bytes (up to half of tile_rows): a
                                         // tile with few rows loads no more than it needs
  uint16_t* c;
  const float* a_scales;
  const float* b_scales;
  const int64_t* device_sizes;           // group sizes on the device, or NULL: row_start holds their prefix sums
  int* status;
  unsigned long long wait_ns;
  int num_groups, rows, n, k;
  int channels;                          // of one CTA's half of a tile: 128 or 64
  int tile_rows, tiles_n, super_tiles;
  int x_maps;                            // entries of map_x that a tile can need
  int stages, stage_bytes;
  int row_start[kMaxGroups + 1];
};

// D[tmem] (+)= W[smem] X[smem]^T in 8-bit integers over both CTAs of the pair, issued by one thread of the leader.
__device__ __forceinline__ void umma_i8_pair(uint32_t tmem_d, uint64_t desc_w, uint64_t desc_x, uint32_t idesc, uint32_t accumulate) {
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

// 16 lanes x 32 columns of a warp's quarter of TMEM as four 16 x 8 fragments: registers 4n, 4n + 1 hold lane i / 4, columns
// 8n + 2 (i % 4) and the next; 4n + 2, 4n + 3 the same of lane 8 + i / 4.
__device__ __forceinline__ void tmem_ld_16x32(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// Stores four 8 x 8 matrices of 16-bit elements transposed: lane 8m + i gives the address of matrix m's column i.
__device__ __forceinline__ void store_transposed(uint32_t addr, uint32_t m0, uint32_t m1, uint32_t m2, uint32_t m3) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(m0), "r"(m1), "r"(m2), "r"(m3) : "memory");
}

// Arrival behind tc_fence_before, which orders the reads of tensor memory against it.  Nothing else has to be visible to the
// MMA warp; the release of mbar_arrive_cluster would wait for the warp's stores to C.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

__device__ __forceinline__ float result(uint32_t acc, float row_scale, float channel_scale) {
  return __fmul_rn(__int2float_rn(static_cast<int>(acc)), __fmul_rn(row_scale, channel_scale));
}
// With any scales.  A product of scales that is subnormal has lost bits, one that overflows makes a NaN of a sum of 0, though the
// result may be a normal number.  A tile whose scales are all `ordinary` takes `result`, which then gives the same bits.
__device__ __forceinline__ float result_of_any(uint32_t sum, float row_scale, float channel_scale) {
  const int acc = static_cast<int>(sum);
  const float s = __fmul_rn(row_scale, channel_scale);
  if (fabsf(s) >= 1.17549435e-38f && fabsf(s) <= 3.4028235e38f) return __fmul_rn(__int2float_rn(acc), s);
  return __double2float_rn(static_cast<double>(acc) * static_cast<double>(row_scale) * static_cast<double>(channel_scale));
}
// The product of two such scales is 0 or a normal number.
__device__ __forceinline__ bool ordinary(float scale) {
  const float size = fabsf(scale);   // no branches: every tile starts with this
  return (size <= 0x1p63f) & ((size >= 0x1p-62f) | (size == 0.f));
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

// 32 rows of a warp's 32 channels through the scales into the box.  `row_scales`: of rows 2 (lane % 4) and the next, and every
// eighth from there; `out`: where this lane's pieces of the transposed fragments go.
template <bool kOrdinary>
__device__ __forceinline__ void transpose_chunk(const uint32_t (&lo)[16], const uint32_t (&hi)[16], const float* row_scales, const float (&sb)[4], uint32_t out) {
  auto value = [](uint32_t acc, float row_scale, float channel_scale) {
    return kOrdinary ? result(acc, row_scale, channel_scale) : result_of_any(acc, row_scale, channel_scale);
  };
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const float2 sa = *reinterpret_cast<const float2*>(row_scales + 8 * n);
    store_transposed(out + 8 * n * kBoxPitch,
                     pack_bf16x2(value(lo[4 * n], sa.x, sb[0]), value(lo[4 * n + 1], sa.y, sb[0])),
                     pack_bf16x2(value(lo[4 * n + 2], sa.x, sb[1]), value(lo[4 * n + 3], sa.y, sb[1])),
                     pack_bf16x2(value(hi[4 * n], sa.x, sb[2]), value(hi[4 * n + 1], sa.y, sb[2])),
                     pack_bf16x2(value(hi[4 * n + 2], sa.x, sb[3]), value(hi[4 * n + 3], sa.y, sb[3])));
  }
}
// Reads the fragments again: the loop over ordinary chunks keeps its code and registers.
__device__ __noinline__ void transpose_chunk_of_any(uint32_t taddr, const float* row_scales, float s0, float s1, float s2, float s3, uint32_t out) {
  uint32_t lo[16], hi[16];
  tmem_ld_16x32(taddr, lo);
  tmem_ld_16x32(taddr + (16u << 16), hi);
  tc_wait_ld();
  const float sb[4] = {s0, s1, s2, s3};
  transpose_chunk<false>(lo, hi, row_scales, sb, out);
}

struct Tile {
  int group, row0, rows, n0;
};
// Tiles of a group: super-rows of `super_tiles` row tiles, row tiles fastest inside one, so that the tiles in flight share
// weights and codes through L2.
__device__ __forceinline__ Tile decode_tile(const Int8GemmParams& p, const int* row_start, const int* tile_start, int tile) {
  Tile t;
  const int g = upper_slot(tile_start, p.num_groups, tile);
  const int local = tile - tile_start[g], m = row_start[g + 1] - row_start[g];
  const int row_tiles = (m + p.tile_rows - 1) / p.tile_rows;
  const int per_super = p.super_tiles * p.tiles_n;
  const int s = local / per_super, rem = local - s * per_super;
  const int h = min(p.super_tiles, row_tiles - s * p.super_tiles);
  const int mt = s * p.super_tiles + rem % h;
  t.group = g;
  t.n0 = rem / h * (2 * p.channels);
  t.row0 = row_start[g] + mt * p.tile_rows;
  t.rows = min(p.tile_rows, m - mt * p.tile_rows);
  return t;
}

constexpr int kMaxRows = 256;                 // rows of the larger tile
constexpr int kMaxStages = 12 / kAtoms;
constexpr int kRingBytes = 6 * 32 * 1024;
constexpr int kTmemCols = 512;
constexpr int kBoxBytes = 32 * kBoxPitch;     // 32 rows x 128 channels of bf16
constexpr int kStagingBytes = 2 * kBoxBytes;
constexpr int kScaleBytes = 2 * kMaxRows * 4;
constexpr int kTableBytes = (2 * (kMaxGroups + 1) * 4 + 15) / 16 * 16;
constexpr int kSmemBytes = kRingBytes + kStagingBytes + kScaleBytes + kTableBytes + 1024 + 256;

// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// Columns of a tile's MMAs; half of its rows come from each CTA.
__device__ __forceinline__ int mma_width(int rows) { return (rows + 31) & ~31; }

// Barrier of one group of epilogue warps.
__device__ __forceinline__ void epilogue_barrier(int group) { asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory"); }
// The same, and whether `mine` is true in all threads of the group.
__device__ __forceinline__ bool epilogue_barrier_all(int group, bool mine) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbar.red.and.pred p, %2, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(all)
      : "r"(mine ? 1u : 0u), "r"(1 + group)
      : "memory");
  return all != 0;
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) int8_gemm_kernel(const __grid_constant__ Int8GemmParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t tiles_addr = (raw_addr + 1023u) & ~1023u;
  uint8_t* staging = smem_raw + (tiles_addr - raw_addr) + kRingBytes;
  float* scale_buf = reinterpret_cast<float*>(staging + kStagingBytes);
  int* row_start = reinterpret_cast<int*>(staging + kStagingBytes + kScaleBytes);
  int* tile_start = row_start + kMaxGroups + 1;
  uint64_t* bars = reinterpret_cast<uint64_t*>(staging + kStagingBytes + kScaleBytes + kTableBytes);
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (kMaxStages + s); };
  auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * kMaxStages + a); };
  auto tempty_bar = [&](int a) { return bar0 + 8u * (2 * kMaxStages + 2 + a); };
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(bars + 2 * kMaxStages + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const bool leader = rank == 0;
  const int stages = p.stages, stage_bytes = p.stage_bytes, w_bytes = p.channels * kAtomK, x_bytes = p.tile_rows / 2 * kAtomK;

  if (threadIdx.x == 32) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), 16);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    prefetch_tensormap(&p.map_w);
    for (int i = 0; i < p.x_maps; ++i) prefetch_tensormap(&p.map_x[i]);
  }
  if (warp == 2) {
    tmem_alloc_pair(smem_u32(tmem_base_slot), kTmemCols);
    tmem_relinquish_pair();
  }
  if (warp == 0) build_groups(p, row_start, tile_start, lane);
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_base_slot;
  const int worker = blockIdx.x >> 1, num_workers = gridDim.x >> 1;
  const int total_tiles = tile_start[p.num_groups];
  // whole stages, then 32-byte steps of a last one that ends with the contraction: no box of zeros, no MMAs on zeros (8 x 2000
  // rows, 3520 channels: K = 544 44.7 -> 41.4 us; tests for it inside the loops made K = 2048 1 - 4 % slower)
  const int num_kb = (p.k + kBlockK - 1) / kBlockK, full_kb = p.k / kBlockK;
  const int last_steps = (p.k - full_kb * kBlockK + 31) / 32, last_atoms = (last_steps + kAtomK / 32 - 1) / (kAtomK / 32);

  if (warp == 0) {
    // ===================== TMA producer: both CTAs credit the leader's barriers =====================
    // The whole warp walks the loop and one elected lane issues: code under a test of the lane number cannot keep its operands in
    // uniform registers, and the MMA warp's loop took 300 ns per 128 bytes of contraction that way instead of 190 (one tile of 256
    // channels and few rows).  Waiting for barriers and signalling them accounts for most of that, so a stage is two boxes deep: 97 ns.
    const bool issue = elect_one();
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t full0_leader = map_to_cta(full_bar(0), 0);
    for (int tile = worker; tile < total_tiles && ok; tile += num_workers) {
      const Tile t = decode_tile(p, row_start, tile_start, tile);
      const int width = mma_width(t.rows);
      const int yw = t.group * p.n + t.n0 + rank * p.channels, yx = t.row0 + rank * (width / 2);
      const int box = width <= 32 ? 0 : width <= 64 ? 1 : width <= 128 ? 2 : 3;   // box of 16 << box rows: one CTA's half
      const CUtensorMap* map_x = &p.map_x[box];
      const int bytes = 2 * (w_bytes + (16 << box) * kAtomK);                             // of one box along K, in both CTAs
      int kb = 0;
      if (tile == worker) {
        // Weights do not depend on the kernel before this one (the quantisation of the rows): a ring full of them goes ahead.
        const int first = min(num_kb, stages);
        for (int i = 0; i < first; ++i) {
          const int atoms = i < full_kb ? kAtoms : last_atoms;
          if (leader && issue) mbar_expect_tx(full_bar(i), atoms * bytes);
#pragma unroll
          for (int h = 0; h < kAtoms; ++h)
            if (issue && h < atoms) tma_load_2d_pair(tiles_addr + i * stage_bytes + h * w_bytes, &p.map_w, full0_leader + 8u * i, i * kBlockK + h * kAtomK, yw);
        }
        grid_dependency_wait();
        for (int i = 0; i < first; ++i)
#pragma unroll
          for (int h = 0; h < kAtoms; ++h)
            if (issue && (h < last_atoms || i < full_kb)) tma_load_2d_pair(tiles_addr + i * stage_bytes + kAtoms * w_bytes + h * x_bytes, map_x, full0_leader + 8u * i, i * kBlockK + h * kAtomK, yx);
        kb = first;
        stage = first == stages ? 0 : first;
        phase = first == stages ? 1u : 0u;
      }
      for (; kb < full_kb && ok; ++kb) {
        ok = mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, 0x1, p.wait_ns);
        if (ok) {
          const uint32_t sw = tiles_addr + stage * stage_bytes, bar = full0_leader + 8u * stage;
          if (leader && issue) mbar_expect_tx(full_bar(stage), kAtoms * bytes);
#pragma unroll
          for (int h = 0; h < kAtoms; ++h) {
            if (issue) tma_load_2d_pair(sw + h * w_bytes, &p.map_w, bar, kb * kBlockK + h * kAtomK, yw);
            if (issue) tma_load_2d_pair(sw + kAtoms * w_bytes + h * x_bytes, map_x, bar, kb * kBlockK + h * kAtomK, yx);
          }
        }
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (kb < num_kb && ok) {
        ok = mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, 0x1, p.wait_ns);
        if (ok) {
          const uint32_t sw = tiles_addr + stage * stage_bytes, bar = full0_leader + 8u * stage;
          if (leader && issue) mbar_expect_tx(full_bar(stage), last_atoms * bytes);
#pragma unroll
          for (int h = 0; h < kAtoms; ++h) {
            if (issue && h < last_atoms) tma_load_2d_pair(sw + h * w_bytes, &p.map_w, bar, kb * kBlockK + h * kAtomK, yw);
            if (issue && h < last_atoms) tma_load_2d_pair(sw + kAtoms * w_bytes + h * x_bytes, map_x, bar, kb * kBlockK + h * kAtomK, yx);
          }
        }
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ===================== MMA issuer: one lane of the leader =====================
    if (leader) {
      const bool issue = elect_one();
      const uint64_t desc_w0 = make_smem_desc(tiles_addr), desc_x0 = make_smem_desc(tiles_addr + kAtoms * w_bytes);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      grid_dependency_wait();   // the limit of the waits below is for this kernel's own copies, not for the quantisation in front
      for (int tile = worker; tile < total_tiles; tile += num_workers) {
        const Tile t = decode_tile(p, row_start, tile_start, tile);
        const uint32_t idesc = idesc_i8(2 * kChannels, mma_width(t.rows));
        ok = mbar_wait(tempty_bar(acc), acc_phase ^ 1u, abort_flag, p.status, 0x2, p.wait_ns);
        if (!ok) break;
        tc_fence_after();
        const uint32_t tmem_d = tmem_base + static_cast<uint32_t>(acc * kMaxRows);
        for (int kb = 0; kb < full_kb; ++kb) {
          ok = mbar_wait(full_bar(stage), phase, abort_flag, p.status, 0x4, p.wait_ns);
          if (!ok) break;
          const uint64_t dw = desc_w0 + static_cast<uint64_t>(stage * (stage_bytes >> 4));
          const uint64_t dx = desc_x0 + static_cast<uint64_t>(stage * (stage_bytes >> 4));
#pragma unroll
          for (int k = 0; k < kBlockK / 32; ++k)
            if (issue)
              umma_i8_pair(tmem_d, dw + (k >> 2) * (w_bytes >> 4) + 2 * (k & 3), dx + (k >> 2) * (x_bytes >> 4) + 2 * (k & 3), idesc, (kb | k) != 0 ? 1u : 0u);
          if (issue) umma_commit_pair(empty_bar(stage));
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        if (full_kb < num_kb) {
          ok = mbar_wait(full_bar(stage), phase, abort_flag, p.status, 0x4, p.wait_ns);
          if (!ok) break;
          const uint64_t dw = desc_w0 + static_cast<uint64_t>(stage * (stage_bytes >> 4));
          const uint64_t dx = desc_x0 + static_cast<uint64_t>(stage * (stage_bytes >> 4));
#pragma unroll
          for (int k = 0; k < kBlockK / 32; ++k)
            if (issue && k < last_steps)
              umma_i8_pair(tmem_d, dw + (k >> 2) * (w_bytes >> 4) + 2 * (k & 3), dx + (k >> 2) * (x_bytes >> 4) + 2 * (k & 3), idesc, (full_kb | k) != 0 ? 1u : 0u);
          if (issue) umma_commit_pair(empty_bar(stage));
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (issue) umma_commit_pair(tfull_bar(acc));
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
    }
    __syncwarp();
  } else {
    // ===================== epilogue: two groups of four warps, 32 channels each, 32 rows at a time in turns =====================
    // A warp that gave up on a wait goes on through its group's barriers, which count all four.
    const int quad = warp & 3, group = (warp - 2) >> 2, thread = (threadIdx.x - 64) & 127;
    const int my_row = ((thread >> 5) * 2 + group) * 32 + lane;   // the row of a tile whose scale this thread fetches
    const uint8_t* box = staging + group * kBoxBytes;
    // where this lane's pieces of the transposed fragments go: row lane % 8 of eight, channels 8 (lane / 8) of the warp's 32
    const uint32_t box_out = smem_u32(box) + (lane & 7) * kBoxPitch + (quad * 32 + (lane >> 3) * 8) * 2;
    const uint8_t* box_in = box + (thread >> 4) * kBoxPitch + (thread & 15) * 16;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    grid_dependency_wait();
    Tile next;
    float next_sa = 0.f, next_sb[4] = {0.f, 0.f, 0.f, 0.f};   // of the row my_row, of channels lane / 4 + 8 j of the warp's
    // the scales of a tile are fetched while the one before it is written
    auto fetch = [&](int tile) {
      if (tile >= total_tiles) return;
      next = decode_tile(p, row_start, tile_start, tile);
      const int n0 = next.n0 + rank * p.channels, channel = n0 + quad * 32 + (lane >> 2), n_end = min(n0 + p.channels, p.n);
      const float* sb = p.b_scales + static_cast<int64_t>(next.group) * p.n + channel;
#pragma unroll
      for (int j = 0; j < 4; ++j) next_sb[j] = channel + 8 * j < n_end ? sb[8 * j] : 0.f;
      if (my_row < next.rows) next_sa = p.a_scales[next.row0 + my_row];
    };
    fetch(worker);
    for (int tile = worker; tile < total_tiles; tile += num_workers) {
      const Tile t = next;
      const float sb[4] = {next_sb[0], next_sb[1], next_sb[2], next_sb[3]};
      const int n0 = t.n0 + rank * p.channels, n_end = min(n0 + p.channels, p.n);
      float* scales = scale_buf + acc * kMaxRows;
      scales[my_row] = next_sa;
      const bool mine = ((my_row >= t.rows) | ordinary(next_sa)) & ordinary(sb[0]) & ordinary(sb[1]) & ordinary(sb[2]) & ordinary(sb[3]);
      fetch(tile + num_workers);
      if (lane == 0 && ok) ok = mbar_wait(tfull_bar(acc), acc_phase, abort_flag, p.status, 0x8, p.wait_ns);
      ok = __shfl_sync(0xFFFFFFFFu, ok, 0);
      const bool all_ordinary = epilogue_barrier_all(group, mine);
      tc_fence_after();
      const uint32_t taddr = tmem_base + static_cast<uint32_t>(acc * kMaxRows) + (static_cast<uint32_t>(quad * 32) << 16);

      // 16 threads write the 256 bytes of a row
      uint16_t* out = p.c + static_cast<int64_t>(t.row0 + group * 32 + (thread >> 4)) * p.n + n0 + (thread & 15) * 8;
      const bool writes = n0 + (thread & 15) * 8 < n_end;
      for (int c0 = group * 32; c0 < t.rows; c0 += 64) {
        if (ok) {
          uint32_t lo[16], hi[16];   // lanes 0-15 and 16-31
          tmem_ld_16x32(taddr + c0, lo);
          tmem_ld_16x32(taddr + c0 + (16u << 16), hi);
          tc_wait_ld();
          if (all_ordinary) transpose_chunk<true>(lo, hi, scales + c0 + 2 * (lane & 3), sb, box_out);
          else transpose_chunk_of_any(taddr + c0, scales + c0 + 2 * (lane & 3), sb[0], sb[1], sb[2], sb[3], box_out);
        }
        epilogue_barrier(group);
        if (ok && writes) {
          if (c0 + 32 <= t.rows) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<uint4*>(out + static_cast<int64_t>(i) * 8 * p.n) = *reinterpret_cast<const uint4*>(box_in + i * 8 * kBoxPitch);
          } else {
            for (int row = thread >> 4, i = 0; c0 + row < t.rows; row += 8, ++i)
              *reinterpret_cast<uint4*>(out + static_cast<int64_t>(i) * 8 * p.n) = *reinterpret_cast<const uint4*>(box_in + i * 8 * kBoxPitch);
          }
        }
        out += static_cast<int64_t>(64) * p.n;
        epilogue_barrier(group);   // the box is read before it is written again
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster_relaxed(map_to_cta(tempty_bar(acc), 0));
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
  }
  tc_fence_before();
  cluster_sync_all();
  if (*abort_flag) {  // copies and MMAs still in flight get time to land before shared memory and TMEM go away
    const unsigned long long t0 = global_ns();
    while (global_ns() - t0 < 200000ull) {
    }
  }
  cluster_sync_all();   // a CTA must not leave while its peer can still touch its shared memory or barriers
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
// (rows x cols) bytes, row pitch `pitch`, box of box_rows x 128 bytes, SWIZZLE_128B.
int encode_rows(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t pitch, int box_rows) {
  auto fn = get_encode_fn();
  if (!fn) {
    set_error("cuTensorMapEncodeTiled is not available from this driver");
    return FP8GMM_CUDA_ERROR;
  }
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch)};
  const cuuint32_t box[2] = {kAtomK, static_cast<cuuint32_t>(box_rows)};
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
int g_tile_rows = 0, g_channels = 0;

// Once per device: the attribute stays.
int allow_shared_memory() {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  FP8GMM_CHECK_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = uint64_t{1} << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit) != 0) return FP8GMM_OK;
  FP8GMM_CHECK_CUDA(cudaFuncSetAttribute(int8_gemm_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
  done.fetch_or(bit, std::memory_order_relaxed);
  return FP8GMM_OK;
}

int pairs() { return gemm_sms() > 1 ? gemm_sms() / 2 : 1; }

// Time of a tile of up to `rows` rows, in that of one of 128: the weights' loads and the MMAs bound it up to there (204 - 250 ns per
// 128 bytes of contraction, 380 - 440 with 256 rows; 64 rows 0.9 of 128).
double tile_time(int64_t rows) { return rows <= 64 ? 0.9 : rows <= 128 ? 1.0 : 1.0 + 0.7 * static_cast<double>(rows - 128) / 128; }
// Time of the pair with the most tiles: `groups` groups of `mean` rows each in tiles of tile_rows.
double worker_time(int64_t groups, int64_t mean, int64_t tiles_n, int64_t tile_rows) {
  const int64_t row_tiles = (mean + tile_rows - 1) / tile_rows;
  const int64_t most = (groups * row_tiles * tiles_n + pairs() - 1) / pairs();
  const double full = tile_time(mean < tile_rows ? mean : tile_rows), last = tile_time(mean - (row_tiles - 1) * tile_rows);
  return full + (most - 1) * ((row_tiles - 1) * full + last) / row_tiles;
}

// Rows and channels of a tile.  256 rows read the weights least often; 128 are for groups of up to 128 rows (one more stage in
// flight), for tiles that all fit one wave of the grid, and where the pair with the most tiles is done sooner with them.  128
// channels where tiles of 256 would fill less than half of the grid (a third with more than 128 rows a group) and the time goes
// into loading weights.  The rule goes by the mean rows of a group that can have any, so that sizes on the host and on the device
// take the same tile; the results are the same bits with all.  Measured, us, product alone.  128 / 256 rows: three experts of
// 3520 x 4096 with 300 rows 17.6 / 26.0, eight of 1536 x 4096 with 300 rows 19.0 / 26.5, with 1000 rows 46.4 / 41.6, eight of 8192 x 4096 with 300 rows
// 89.4 / 92.6, with 2000 rows 458 / 387.  128 / 256 channels, 128 rows: two rows of 4096 x 14336 24.8 / 27.6, one expert of 256 x 1040 with 300
// rows 7.3 / 7.9, of 768 x 4096 with 200 rows 9.8 / 10.1, three of 1536 x 4096 with 200 rows 11.4 / 10.6.  Over 405 shapes (1 to 8
// experts of equally many rows, 64 to 2000, 256 to 8192 channels, 256 to 4096 bytes) the rule takes 0.6 % more than the best tile on
// average; with uneven groups it can miss the better one, by up to 18 % of the estimate above.
// (Splitting the contraction of a partial wave's tiles between pairs, with sums handed on through L2, cost about 8 us a
// tile: dropped.)
struct TileShape {
  int rows, channels;
};
TileShape choose_tile(const fp8gmm_int8_gemm_args* a) {
  const int64_t tiles_n = (a->n + 2 * kChannels - 1) / (2 * kChannels);
  const int64_t groups = a->rows < a->num_groups ? a->rows : a->num_groups;
  const int64_t mean = (a->rows + groups - 1) / groups;
  const int64_t small = groups * ((mean + 127) / 128) * tiles_n;   // tiles of 128 rows and 256 channels
  const bool few = mean <= 128 || small <= pairs() || worker_time(groups, mean, tiles_n, 128) < worker_time(groups, mean, tiles_n, 256);
  const bool narrow = few && (mean <= 128 ? 2 : 3) * small <= pairs();
  TileShape t;
  t.rows = g_tile_rows != 0 ? g_tile_rows : few ? 128 : 256;
  t.channels = g_channels != 0 ? g_channels / 2 : narrow ? kChannels / 2 : kChannels;
  return t;
}

}  // namespace

// Argument checks; nothing is launched and no CUDA call made.
int int8_gemm_check(const fp8gmm_int8_gemm_args* a) {
  FP8GMM_CHECK_ARG(a != nullptr, "int8_grouped_gemm: NULL arguments");
  FP8GMM_CHECK_ARG(a->num_groups >= 0 && a->num_groups <= kMaxGroups, "int8_grouped_gemm: num_groups %d outside [0, %d]", a->num_groups, kMaxGroups);
  FP8GMM_CHECK_ARG(a->n > 0 && a->k > 0 && a->n % 16 == 0 && a->k % 16 == 0, "int8_grouped_gemm: N (%lld) and K (%lld) must be positive multiples of 16",
                   (long long)a->n, (long long)a->k);
  FP8GMM_CHECK_ARG(a->a_ld == 0 || (a->a_ld >= a->k && a->a_ld <= INT32_MAX && a->a_ld % 16 == 0),
                   "int8_grouped_gemm: a row pitch of %lld is not a multiple of 16 from K = %lld to 2^31", (long long)a->a_ld, (long long)a->k);
  FP8GMM_CHECK_ARG(a->k < (1 << 17), "int8_grouped_gemm: K = %lld could overflow the 32-bit sums (K < 131072)", (long long)a->k);
  FP8GMM_CHECK_ARG(a->n <= INT32_MAX / (a->num_groups > 0 ? a->num_groups : 1) - 1024, "int8_grouped_gemm: too many weight rows");
  FP8GMM_CHECK_ARG(a->rows >= 0 && a->rows <= INT32_MAX - 1024, "int8_grouped_gemm: bad number of rows");
  FP8GMM_CHECK_ARG(a->num_groups == 0 || (a->m_sizes != nullptr) != (a->device_m_sizes != nullptr),
                   "int8_grouped_gemm: group sizes are given on the host or on the device, not both");
  FP8GMM_CHECK_ARG(a->num_groups > 0 || a->rows == 0, "int8_grouped_gemm: %lld rows, but no groups", (long long)a->rows);
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
  const TileShape tile = choose_tile(a);
  const int tile_rows = p.tile_rows = tile.rows;
  p.channels = tile.channels;
  rc = encode_rows(&p.map_w, a->b, a->num_groups * a->n, a->k, a->k, p.channels);
  if (rc != FP8GMM_OK) return rc;
  for (; p.x_maps < 4 && (p.x_maps == 0 || (32 << p.x_maps <= tile_rows && 16 << p.x_maps < p.rows)); ++p.x_maps) {
    rc = encode_rows(&p.map_x[p.x_maps], a->a, a->rows, a->k, a->a_ld != 0 ? a->a_ld : a->k, 16 << p.x_maps);
    if (rc != FP8GMM_OK) return rc;
  }
  // with 64 channels the MMA reads 16 KiB from the start of each half of the weights all the same: into what lies behind them
  p.stage_bytes = kAtoms * (p.channels + tile_rows / 2) * kAtomK;
  p.stages = kRingBytes / p.stage_bytes < kMaxStages ? kRingBytes / p.stage_bytes : kMaxStages;
  p.tiles_n = (p.n + 2 * p.channels - 1) / (2 * p.channels);
  // a band of codes of 4096 rows (2048 with a long contraction) stays in L2 while the channel tiles sweep past it
  p.super_tiles = (p.k > 8192 ? 2048 : 4096) / tile_rows;
  // each group adds at most one partial row tile to rows / tile_rows
  const int64_t most = (p.rows / tile_rows + (p.rows < p.num_groups ? p.rows : p.num_groups)) * static_cast<int64_t>(p.tiles_n);
  FP8GMM_CHECK_ARG(most <= INT32_MAX / 2, "int8_grouped_gemm: problem too large");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int workers = most < pairs() ? static_cast<int>(most) : pairs();
  rc = allow_shared_memory();
  if (rc != FP8GMM_OK) return rc;
  FP8GMM_CHECK_CUDA(launch_dependent(int8_gemm_kernel, 2 * workers, kThreads, kSmemBytes, s, after_quantize, p));
  count_launch();
  return FP8GMM_OK;
}

}  // namespace fp8gmm

extern "C" {

int fp8gmm_set_int8_variant(int tile_rows, int tile_channels) {
  using namespace fp8gmm;
  FP8GMM_CHECK_ARG(tile_rows == 0 || tile_rows == 128 || tile_rows == 256, "set_int8_variant: tile_rows must be 0, 128 or 256");
  FP8GMM_CHECK_ARG(tile_channels == 0 || tile_channels == 128 || tile_channels == 256, "set_int8_variant: tile_channels must be 0, 128 or 256");
  g_tile_rows = tile_rows;
  g_channels = tile_channels;
  return FP8GMM_OK;
}

int fp8gmm_int8_grouped_gemm(const fp8gmm_int8_gemm_args* a, void* stream) { return fp8gmm::int8_gemm_launch(a, stream, false); }

int fp8gmm_int8_linear(const fp8gmm_quantize_rows_args* q, const fp8gmm_int8_gemm_args* g, void* stream) {
  FP8GMM_CHECK_ARG(q != nullptr && g != nullptr, "int8_linear: NULL arguments");
  FP8GMM_CHECK_ARG(q->codes == g->a && q->scales == g->a_scales && q->rows == g->rows && q->cols == g->k && q->codes_ld == g->a_ld,
                   "int8_linear: the product has to take the codes, scales, rows, columns and row pitch of the quantisation");
  int rc = fp8gmm::int8_gemm_check(g);   // before anything is launched
  if (rc != FP8GMM_OK) return rc;
  rc = fp8gmm_quantize_rows_int8(q, stream);
  return rc != FP8GMM_OK ? rc : fp8gmm::int8_gemm_launch(g, stream, q->rows > 0);
}

}  // extern "C"
