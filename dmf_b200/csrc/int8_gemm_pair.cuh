// The 8-bit product for many rows, on CTA pairs:
//
//   out[m, n] = (sum_k x[m, k] w[n, k]) x_scale[m] w_scale[n] + bias[n],    the sum in int32
//
// Persistent clusters of two CTAs walk tiles of 256 x BN outputs; a tile's products are tcgen05.mma.cta_group::2 of kind::i8,
// M = 256, N = BN, 32 bytes of k each.  CTA r holds 128 of the tile's rows of x and half of its rows of w, so a 128-byte step of
// k costs each SM 16 KB + BN / 2 * 128 bytes of loads for 256 x BN x 128 products of the pair.
//
// With BN = 256 a last stretch of at most 128 columns is done in tiles of half the width (N = 1152: 4.5 tiles a row instead of 5).
//
// Warps: 0 TMA producer (both CTAs), 1 MMA issuer (leader CTA), 2.. epilogue (both CTAs).  Two accumulators of BN columns
// alternate in tensor memory, so the epilogue of a tile runs under the products of the next one.  An epilogue warp takes 32 rows
// (its quarter of the lanes) and 64 or 128 columns, 64 at a time; the rounded results go through 4 KB of its own to a TMA store.
//
// What bounds it: shared memory.  At full rate the loads write 64 bytes per cycle and SM and the products read as much, of the
// 128 it has, so the epilogue has to be sparing: it reads the accumulators in the layout of matrix fragments, where a thread has
// two columns of each eight and so reads 16 bytes of scales and bias for eight results.  (In the row layout, where every thread
// reads those of all columns, that alone took 6 us of 59 at 16384 x 1152 x 3456.)
//
// In bursts: 16384 x 1152 x 3456 51 us (2.5 Pop/s; 63 call after call, at the power limit), x 4608 63 us (2.7), 16384 x 4608 x 1152 66 us
// (2.6; 5.2 or 4.3 rounds of tiles), 8192^3 345 us (3.2); a larger tile would need less of the L2, but 256 x 256 twice is all the tensor memory there is.
//
// Every wait is bounded (see sm100_ptx.cuh); a role whose wait gives up leaves its loop, the others follow at their next wait,
// all meet at the end.
#pragma once

#include <cuda.h>
#include <stdint.h>

#include <type_traits>

#include "int8_types.cuh"
#include "sm100_ptx.cuh"

namespace dmf {

struct Int8GemmParams {
  CUtensorMap x_map, w_map;     // boxes of 128 bytes of k; x: 128 rows (pair) / the tile's tokens, w: BN / 2 rows (pair) / 128
  CUtensorMap w_half_map;       // pair, narrow: boxes of 64 rows of w
  CUtensorMap out_map;          // pair, out_vec: boxes of 128 bytes x 32 rows
  const float *x_scale, *w_scale;
  const void* bias;
  void* out;
  int32_t* status_word;
  int64_t out_stride;
  int m, n, k;
  int tiles_m, tiles_n;         // pair: without the narrow ones
  int narrow;                   // pair: the columns end in tiles of half the width
  int out_dtype, bias_dtype;
  int out_vec;                  // rows of out start at multiples of 16 bytes
};

constexpr int kRoleInt8Producer = 600, kRoleInt8Mma = 700, kRoleInt8Epilogue = 800;

// After a wait gave up: loads that were issued land before anybody reuses or leaves the shared memory (they need microseconds;
// the wait that gave up has taken seconds).
__device__ __forceinline__ void int8_drain(volatile int* abort_flag) {
  if (*abort_flag == 0) return;
  const long long t0 = clock64();
  while (clock64() - t0 < 2000000ll) {
  }
}

template <int BN>
struct Int8PairTraits {
  static constexpr int kXBytes = 128 * 128, kWBytes = BN / 2 * 128, kStageBytes = kXBytes + kWBytes;
  static constexpr int kStages = BN == 256 ? 5 : (BN == 192 ? 6 : 7);
  static constexpr int kRingBytes = kStages * kStageBytes;
  static constexpr int kCols = BN == 256 ? 128 : 64;                   // columns of an epilogue warp
  static constexpr int kWarps = BN / kCols * 4, kThreads = 64 + 32 * kWarps;   // epilogue warps; all threads
  static constexpr int kWarpStage = 4096, kWarpVec = kCols * 8;        // per epilogue warp: staged results; scales and bias
  static constexpr int kBarFull = 0, kBarEmpty = kStages, kBarAccFull = 2 * kStages, kBarAccEmpty = kBarAccFull + 2,
                       kNumBars = kBarAccEmpty + 2;
  static constexpr int kSmemBytes = 1024 + kRingBytes + kWarps * (kWarpStage + kWarpVec) + kNumBars * 8 + 16;
  static_assert(kSmemBytes <= 227 * 1024, "shared memory of one CTA");
  static constexpr uint32_t kTmemCols = BN == 128 ? 256 : 512;
};

constexpr int kInt8GroupM = 8;   // tiles run over w within groups of 8 row tiles: w is read from HBM once per 2048 rows at most

// The tiles of a cluster, in order: its share of the whole tiles, then of the narrow ones (the last 128 columns or fewer), which
// go to the clusters that had one whole tile less, twice, before everybody gets them in turn.
struct Int8TileWalk {
  int whole, tiles_m, tiles_n, narrow, clusters, id;
  int t, turn;
  __device__ __forceinline__ Int8TileWalk(const Int8GemmParams& p, int id_, int clusters_)
      : whole(p.tiles_m * p.tiles_n), tiles_m(p.tiles_m), tiles_n(p.tiles_n), narrow(p.narrow ? p.tiles_m : 0), clusters(clusters_), id(id_),
        t(id_), turn(id_ >= whole % clusters_ ? 0 : 2) {}
  // the next tile, false after the last
  __device__ __forceinline__ bool next(int& tm, int& tn, bool& is_narrow) {
    if (t < whole) {
      const int per_group = kInt8GroupM * tiles_n;
      const int g = t / per_group, r = t % per_group;
      const int rows = min(kInt8GroupM, tiles_m - g * kInt8GroupM);
      tm = g * kInt8GroupM + r % rows;
      tn = r / rows;
      is_narrow = false;
      t += clusters;
      return true;
    }
    const int busy = whole % clusters, free = clusters - busy;
    const int slot = turn < 2 ? turn * free + id - busy : 2 * free + id + (turn - 2) * clusters;
    ++turn;
    tm = slot;
    tn = tiles_n;
    is_narrow = true;
    return slot < narrow;
  }
};

template <int BN, typename T>
__global__ void __launch_bounds__(Int8PairTraits<BN>::kThreads, 1) int8_gemm_pair_kernel(const __grid_constant__ Int8GemmParams p) {
  using TR = Int8PairTraits<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t s_ring = smem_u32(smem);
  uint8_t* out_stage = smem + TR::kRingBytes;
  uint8_t* vecs = out_stage + TR::kWarps * TR::kWarpStage;
  uint64_t* bars = reinterpret_cast<uint64_t*>(vecs + TR::kWarps * TR::kWarpVec);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + TR::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](int i) -> uint32_t { return bar0 + 8u * static_cast<uint32_t>(i); };
  auto lbar = [&](int i) -> uint32_t { return map_to_cta(bar(i), 0); };  // the leader's barrier

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int cluster_id = blockIdx.x >> 1, num_clusters = gridDim.x >> 1;
  const int k_steps = (p.k + 127) >> 7;
  Int8TileWalk walk(p, cluster_id, num_clusters);

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < TR::kNumBars; ++i) {
      uint32_t count = 1;                          // tcgen05.commit, multicast from the leader
      if (i < TR::kBarEmpty) count = 2;            // the producers' arrivals with their bytes (used in the leader)
      if (i >= TR::kBarAccEmpty) count = 2 * TR::kWarps;  // the epilogue warps of both CTAs (used in the leader)
      mbar_init(bar(i), count);
    }
    fence_mbar_init();
  }
  if (warp == 0) {
    __syncwarp();
    tmem_alloc_pair(smem_u32(tmem_slot), TR::kTmemCols);
    tmem_relinquish_alloc_permit_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers are initialised before anybody arrives remotely
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  grid_dependency_wait();
  grid_launch_dependents();

  if (warp == 0) {
    // =========================== TMA producer (each CTA) ====================
    if (lane == 0) {
      prefetch_tensor_map(&p.x_map);
      prefetch_tensor_map(&p.w_map);
      uint32_t cnt = 0;
      bool ok = true;
      int tm, tn;
      bool narrow;
      while (ok && walk.next(tm, tn, narrow)) {
        const int x_row = tm * 256 + static_cast<int>(rank) * 128, w_row = tn * BN + static_cast<int>(rank) * (narrow ? 64 : BN / 2);
        for (int kk = 0; kk < k_steps; ++kk, ++cnt) {
          const uint32_t s = cnt % TR::kStages, ph = (cnt / TR::kStages) & 1u;
          ok = mbar_wait(bar(TR::kBarEmpty + s), ph ^ 1u, abort_flag, p.status_word, kRoleInt8Producer + TR::kBarEmpty + s);
          if (!ok) break;
          const uint32_t dst = s_ring + s * TR::kStageBytes, fb = lbar(TR::kBarFull + s);
          mbar_arrive_expect_tx_cluster(fb, narrow ? TR::kXBytes + 64 * 128 : TR::kStageBytes);
          tma_load_2d_pair(dst, &p.x_map, fb, kk * 128, x_row);
          tma_load_2d_pair(dst + TR::kXBytes, narrow ? &p.w_half_map : &p.w_map, fb, kk * 128, w_row);
        }
      }
    }
  } else if (warp == 1) {
    // ===================== MMA issuer (leader CTA only) =======================
    if (rank == 0) {
      const bool leader = elect_one();
      uint32_t cnt = 0, tcnt = 0;
      bool ok = true, narrow;
      int tm, tn;
      for (; ok && walk.next(tm, tn, narrow); ++tcnt) {
        const uint32_t a = tcnt & 1u, idesc = narrow ? make_idesc_i8(256, 128) : make_idesc_i8(256, BN);
        // the epilogue of the tile before the last has read this accumulator (both CTAs)
        ok = mbar_wait(bar(TR::kBarAccEmpty + a), ((tcnt >> 1) & 1u) ^ 1u, abort_flag, p.status_word,
                       kRoleInt8Mma + TR::kBarAccEmpty + a);
        if (!ok) break;
        tc_fence_after_sync();
        for (int kk = 0; kk < k_steps; ++kk, ++cnt) {
          const uint32_t s = cnt % TR::kStages, ph = (cnt / TR::kStages) & 1u;
          ok = mbar_wait(bar(TR::kBarFull + s), ph, abort_flag, p.status_word, kRoleInt8Mma + TR::kBarFull + s);
          if (!ok) break;
          tc_fence_after_sync();
          const uint32_t xs = s_ring + s * TR::kStageBytes, ws = xs + TR::kXBytes;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            mma_i8_pair(tmem + a * BN, make_smem_desc(xs + i * 32, 16, 1024, kSwizzle128),
                        make_smem_desc(ws + i * 32, 16, 1024, kSwizzle128), idesc, (kk > 0 || i > 0) ? 1u : 0u, leader);
          tc_commit_pair(bar(TR::kBarEmpty + s), leader);
        }
        if (!ok) break;
        tc_commit_pair(bar(TR::kBarAccFull + a), leader);
      }
    }
  } else {
    // =========================== epilogue (each CTA) ==========================
    constexpr int kCols = TR::kCols, kPer = kCols / 32;
    constexpr int kWide = 128 / sizeof(T);             // results per 128 bytes: 64 or 32
    const int ew = warp - 2, quarter = warp & 3, col0 = (ew >> 2) * kCols;
    float* s_w = reinterpret_cast<float*>(vecs + ew * TR::kWarpVec);
    float* s_b = s_w + kCols;
    uint8_t* stage = out_stage + ew * TR::kWarpStage;
    const uint32_t s_stage = smem_u32(stage);
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + col0;
    const int frow = lane >> 2, fcol = 2 * (lane & 3);  // this lane's first row and column of a fragment
    // scales and bias of a tile's columns and the scales of this lane's rows: in registers a tile ahead
    float next_w[kPer], next_b[kPer], next_x[4];
    int tm, tn, next_tm, next_tn;
    bool narrow, next_narrow, more;
    auto fetch = [&] {
      more = walk.next(next_tm, next_tn, next_narrow);
      if (!more) return;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int n = next_tn * BN + col0 + i * 32 + lane;
        next_w[i] = n < p.n ? p.w_scale[n] : 0.f;
        next_b[i] = n < p.n && p.bias != nullptr ? row_load(p.bias, p.bias_dtype, n) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t m = static_cast<int64_t>(next_tm) * 256 + rank * 128 + quarter * 32 + frow + 8 * i;
        next_x[i] = m < p.m ? p.x_scale[m] : 0.f;
      }
    };
    auto slot = [](int row, int piece) -> int { return row * 128 + ((piece ^ (row & 7)) << 4); };   // the store map's swizzle
    fetch();
    for (uint32_t tcnt = 0; more; ++tcnt) {
      tm = next_tm;
      tn = next_tn;
      narrow = next_narrow;
      const int n0 = tn * BN + col0;
      const int m0 = tm * 256 + static_cast<int>(rank) * 128 + quarter * 32;
      const uint32_t a = tcnt & 1u;
      const float xs[4] = {next_x[0], next_x[1], next_x[2], next_x[3]};
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        s_w[i * 32 + lane] = next_w[i];
        s_b[i * 32 + lane] = next_b[i];
      }
      fetch();
      __syncwarp();
      const bool ok = __all_sync(0xffffffffu, mbar_wait(bar(TR::kBarAccFull + a), (tcnt >> 1) & 1u, abort_flag, p.status_word,
                                                        kRoleInt8Epilogue + TR::kBarAccFull + a));
      if (!ok) break;
      tc_fence_after_sync();
      if (narrow && col0 >= 128) {                     // no columns of this warp's
        mbar_arrive_warp_cluster(lbar(TR::kBarAccEmpty + a));
        continue;
      }
#pragma unroll
      for (int c0 = 0; c0 < kCols; c0 += 32) {
        uint32_t lo[16], hi[16];                       // rows frow, + 8 and + 16, + 24
        tmem_ld_16x256b_x4(lane_base + a * BN + c0, lo);
        tmem_ld_16x256b_x4(lane_base + (16u << 16) + a * BN + c0, hi);
        if (c0 % kWide == 0) {                         // the stage: its last store has read it
          if (lane == 0) tma_store_wait_read();
          __syncwarp();
        }
        tmem_wait_ld();
        if (c0 + 32 == kCols) {                        // the accumulator may be written again
          tc_fence_before_sync();
          mbar_arrive_warp_cluster(lbar(TR::kBarAccEmpty + a));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 w = *reinterpret_cast<const float2*>(s_w + c0 + 8 * j + fcol), b = *reinterpret_cast<const float2*>(s_b + c0 + 8 * j + fcol);
          float f[4][2];                               // rows frow + 8 i
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t* v = (i < 2 ? lo : hi) + 4 * j + 2 * (i & 1);
            f[i][0] = fmaf(static_cast<float>(static_cast<int>(v[0])) * xs[i], w.x, b.x);
            f[i][1] = fmaf(static_cast<float>(static_cast<int>(v[1])) * xs[i], w.y, b.y);
          }
          if constexpr (sizeof(T) == 2) {
            stmatrix_x4(s_stage + slot(lane, (c0 % kWide) / 8 + j), Pack2<T>::pack(f[0][0], f[0][1]), Pack2<T>::pack(f[1][0], f[1][1]),
                        Pack2<T>::pack(f[2][0], f[2][1]), Pack2<T>::pack(f[3][0], f[3][1]));
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<float2*>(stage + slot(frow + 8 * i, 2 * j + (fcol >> 2)) + (fcol & 2) * 4) = make_float2(f[i][0], f[i][1]);
          }
        }
        if ((c0 + 32) % kWide == 0) {                  // 128 bytes of every row are staged
          const int n = n0 + c0 + 32 - kWide;
          if (p.out_vec) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&p.out_map, s_stage, n, m0);   // clipped at the matrix's ends
              tma_store_commit();
            }
          } else {
            // rows that start anywhere: a row at a time, 32 bits per lane; in rows that start between two words the words are
            // put together from two lanes'
            __syncwarp();
            const int rows = min(32, p.m - m0), cols = min(kWide, p.n - n);
            T* dst = static_cast<T*>(p.out) + static_cast<int64_t>(m0) * p.out_stride + n;
#pragma unroll 1
            for (int row0 = 0; row0 < rows; row0 += 8) {
              uint32_t v[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const uint32_t*>(stage + slot(row0 + i, lane >> 2) + (lane & 3) * 4);
#pragma unroll
              for (int i = 0; i < 8; ++i, dst += p.out_stride) {
                if (row0 + i >= rows) break;
                if constexpr (sizeof(T) == 4) {
                  if (lane < cols) *reinterpret_cast<uint32_t*>(dst + lane) = v[i];
                } else {
                  uint16_t* d = reinterpret_cast<uint16_t*>(dst);
                  const uint32_t odd = reinterpret_cast<uintptr_t>(dst) >> 1 & 1u;   // (the whole warp alike)
                  const uint32_t next = __shfl_down_sync(0xffffffffu, v[i], 1);
                  const int c = 2 * lane + static_cast<int>(odd);
                  const uint32_t u = odd != 0u ? __funnelshift_r(v[i], next, 16) : v[i];
                  if (odd != 0u && lane == 0 && cols > 0) d[0] = static_cast<uint16_t>(v[i]);
                  if (c + 1 < cols) *reinterpret_cast<uint32_t*>(d + c) = u;
                  else if (c < cols) d[c] = static_cast<uint16_t>(u);
                }
              }
            }
          }
          __syncwarp();
        }
      }
    }
    if (p.out_vec && lane == 0) tma_store_wait_all();
  }

  // ============================== teardown ==================================
  __syncwarp();
  int8_drain(abort_flag);
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // nobody leaves (or frees tensor memory) while the other CTA may still touch this one
  tc_fence_after_sync();
  if (warp == 0) tmem_dealloc_pair(tmem, TR::kTmemCols);
}

}  // namespace dmf
