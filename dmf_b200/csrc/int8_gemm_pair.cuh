// The 8-bit product for many rows, on CTA pairs:
//
//   out[m, n] = (sum_k x[m, k] w[n, k]) x_scale[m] w_scale[n] + bias[n],    the sum in int32
//
// Persistent clusters of two CTAs walk tiles of 256 x BN outputs; a tile's products are tcgen05.mma.cta_group::2 of kind::i8,
// M = 256, N = BN, 32 bytes of k each.  CTA r holds 128 of the tile's rows of x and half of its rows of w, so a 128-byte step of
// k costs each SM 16 KB + BN / 2 * 128 bytes of loads for 256 x BN x 128 products of the pair.
//
// Warps: 0 TMA producer (both CTAs), 1 MMA issuer (leader CTA), 2..9 epilogue (both CTAs).  Two accumulators of BN columns
// alternate in tensor memory, so the epilogue of a tile runs under the products of the next one.  An epilogue warp takes 32 rows
// (its quarter of the lanes) and half of the columns: scales and bias from a copy of its own in shared memory, the rounded
// results through 4 KB of its own to whole 16-byte pieces of rows, 128 bytes of a row at a time.
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
  const float *x_scale, *w_scale;
  const void* bias;
  void* out;
  int32_t* status_word;
  int64_t out_stride;
  int m, n, k;
  int tiles_m, tiles_n;
  int out_dtype, bias_dtype;
  int out_vec;                  // rows of out start at multiples of 16 bytes
};

constexpr int kRoleInt8Producer = 600, kRoleInt8Mma = 700, kRoleInt8Epilogue = 800;

// the output type's vectors: 16 bytes of results
template <typename T>
struct OutVec {
  static constexpr int kElems = 8;
  __device__ __forceinline__ static uint4 pack(const float* v) {
    return make_uint4(Pack2<T>::pack(v[0], v[1]), Pack2<T>::pack(v[2], v[3]), Pack2<T>::pack(v[4], v[5]), Pack2<T>::pack(v[6], v[7]));
  }
};
template <>
struct OutVec<float> {
  static constexpr int kElems = 4;
  __device__ __forceinline__ static uint4 pack(const float* v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};

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
  static constexpr int kWarpStage = 4096, kWarpVec = BN / 2 * 8;       // per epilogue warp: staged results; scales and bias
  static constexpr int kBarFull = 0, kBarEmpty = kStages, kBarAccFull = 2 * kStages, kBarAccEmpty = kBarAccFull + 2,
                       kNumBars = kBarAccEmpty + 2;
  static constexpr int kSmemBytes = 1024 + kRingBytes + 8 * (kWarpStage + kWarpVec) + kNumBars * 8 + 16;
  static_assert(kSmemBytes <= 227 * 1024, "shared memory of one CTA");
  static constexpr uint32_t kTmemCols = BN == 128 ? 256 : 512;
};

constexpr int kInt8PairThreads = 320;
constexpr int kInt8GroupM = 8;   // tiles run over w within groups of 8 row tiles: w is read from HBM once per 2048 rows at most

__device__ __forceinline__ void int8_tile(int t, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int per_group = kInt8GroupM * tiles_n;
  const int g = t / per_group, r = t % per_group;
  const int rows = min(kInt8GroupM, tiles_m - g * kInt8GroupM);
  tm = g * kInt8GroupM + r % rows;
  tn = r / rows;
}

template <int BN, typename T>
__global__ void __launch_bounds__(kInt8PairThreads, 1) int8_gemm_pair_kernel(const __grid_constant__ Int8GemmParams p) {
  using TR = Int8PairTraits<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t s_ring = smem_u32(smem);
  uint8_t* out_stage = smem + TR::kRingBytes;
  uint8_t* vecs = out_stage + 8 * TR::kWarpStage;
  uint64_t* bars = reinterpret_cast<uint64_t*>(vecs + 8 * TR::kWarpVec);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + TR::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](int i) -> uint32_t { return bar0 + 8u * static_cast<uint32_t>(i); };
  auto lbar = [&](int i) -> uint32_t { return map_to_cta(bar(i), 0); };  // the leader's barrier

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int cluster_id = blockIdx.x >> 1, num_clusters = gridDim.x >> 1;
  const int tiles = p.tiles_m * p.tiles_n, k_steps = (p.k + 127) >> 7;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < TR::kNumBars; ++i) {
      uint32_t count = 1;                          // tcgen05.commit, multicast from the leader
      if (i < TR::kBarEmpty) count = 2;            // the producers' arrivals with their bytes (used in the leader)
      if (i >= TR::kBarAccEmpty) count = 16;       // the epilogue warps of both CTAs (used in the leader)
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

  if (warp == 0) {
    // =========================== TMA producer (each CTA) ====================
    if (lane == 0) {
      prefetch_tensor_map(&p.x_map);
      prefetch_tensor_map(&p.w_map);
      uint32_t cnt = 0;
      bool ok = true;
      for (int t = cluster_id; ok && t < tiles; t += num_clusters) {
        int tm, tn;
        int8_tile(t, p.tiles_m, p.tiles_n, tm, tn);
        const int x_row = tm * 256 + static_cast<int>(rank) * 128, w_row = tn * BN + static_cast<int>(rank) * (BN / 2);
        for (int kk = 0; kk < k_steps; ++kk, ++cnt) {
          const uint32_t s = cnt % TR::kStages, ph = (cnt / TR::kStages) & 1u;
          ok = mbar_wait(bar(TR::kBarEmpty + s), ph ^ 1u, abort_flag, p.status_word, kRoleInt8Producer + TR::kBarEmpty + s);
          if (!ok) break;
          const uint32_t dst = s_ring + s * TR::kStageBytes, fb = lbar(TR::kBarFull + s);
          mbar_arrive_expect_tx_cluster(fb, TR::kStageBytes);
          tma_load_2d_pair(dst, &p.x_map, fb, kk * 128, x_row);
          tma_load_2d_pair(dst + TR::kXBytes, &p.w_map, fb, kk * 128, w_row);
        }
      }
    }
  } else if (warp == 1) {
    // ===================== MMA issuer (leader CTA only) =======================
    if (rank == 0) {
      const bool leader = elect_one();
      constexpr uint32_t idesc = make_idesc_i8(256, BN);
      uint32_t cnt = 0, tcnt = 0;
      bool ok = true;
      for (int t = cluster_id; ok && t < tiles; t += num_clusters, ++tcnt) {
        const uint32_t a = tcnt & 1u;
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
    constexpr int kCols = BN / 2;                      // columns of a warp
    constexpr int kVec = OutVec<T>::kElems;            // results per 16 bytes
    constexpr int kPer = kCols / 32;                   // columns of a lane's scales
    const int ew = warp - 2, quarter = warp & 3, half = ew >> 2;
    float* s_w = reinterpret_cast<float*>(vecs + ew * TR::kWarpVec);
    float* s_b = s_w + kCols;
    uint8_t* stage = out_stage + ew * TR::kWarpStage;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + half * kCols;
    // scales and bias of a tile's columns and the scale of this lane's row: in registers a tile ahead
    float next_w[kPer], next_b[kPer], next_x = 0.f;
    auto fetch = [&](int t) {
      if (t >= tiles) return;
      int tm, tn;
      int8_tile(t, p.tiles_m, p.tiles_n, tm, tn);
      const int n0 = tn * BN + half * kCols;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int n = n0 + i * 32 + lane;
        next_w[i] = n < p.n ? p.w_scale[n] : 0.f;
        next_b[i] = n < p.n && p.bias != nullptr ? row_load(p.bias, p.bias_dtype, n) : 0.f;
      }
      const int64_t m = static_cast<int64_t>(tm) * 256 + rank * 128 + quarter * 32 + lane;
      next_x = m < p.m ? p.x_scale[m] : 0.f;
    };
    fetch(cluster_id);
    uint32_t tcnt = 0;
    for (int t = cluster_id; t < tiles; t += num_clusters, ++tcnt) {
      int tm, tn;
      int8_tile(t, p.tiles_m, p.tiles_n, tm, tn);
      const int n0 = tn * BN + half * kCols;
      const int64_t m0 = static_cast<int64_t>(tm) * 256 + rank * 128 + quarter * 32;
      const uint32_t a = tcnt & 1u;
      const float xs = next_x;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        s_w[i * 32 + lane] = next_w[i];
        s_b[i * 32 + lane] = next_b[i];
      }
      fetch(t + num_clusters);
      __syncwarp();
      const bool ok = __all_sync(0xffffffffu, mbar_wait(bar(TR::kBarAccFull + a), (tcnt >> 1) & 1u, abort_flag, p.status_word,
                                                        kRoleInt8Epilogue + TR::kBarAccFull + a));
      if (!ok) break;
      tc_fence_after_sync();
      const bool whole = p.out_vec && m0 + 32 <= p.m && n0 + kCols <= p.n;
      // W columns from column c0 of this warp: at most 128 bytes of each row go through shared memory at a time
      auto emit = [&](int c0, auto width) {
        constexpr int W = decltype(width)::value;
        constexpr int kPieces = W / kVec;              // 16-byte pieces of a row, 8 or 4
        constexpr int kRows = 32 / kPieces;            // rows per warp-wide store
        auto slot = [](int row, int piece) -> int {
          return row * (kPieces * 16) + ((piece ^ (kPieces == 8 ? row & 7 : (row >> 1) & 3)) << 4);
        };
#pragma unroll
        for (int h = 0; h < W / 32; ++h) {
          const int c = c0 + h * 32;
          uint32_t v[32];
          tmem_ld_x32(lane_base + a * BN + c, v);
          float4 w4[8], b4[8];                         // under the load: all before the stores, which could alias them
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            w4[i] = *reinterpret_cast<const float4*>(s_w + c + 4 * i);
            b4[i] = *reinterpret_cast<const float4*>(s_b + c + 4 * i);
          }
          tmem_wait_ld();
          if (c + 32 == kCols) {                       // the tile's last read: the accumulator may be written again
            tc_fence_before_sync();
            mbar_arrive_warp_cluster(lbar(TR::kBarAccEmpty + a));
          }
          float f[32];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            f[4 * i] = fmaf(static_cast<float>(static_cast<int>(v[4 * i])) * xs, w4[i].x, b4[i].x);
            f[4 * i + 1] = fmaf(static_cast<float>(static_cast<int>(v[4 * i + 1])) * xs, w4[i].y, b4[i].y);
            f[4 * i + 2] = fmaf(static_cast<float>(static_cast<int>(v[4 * i + 2])) * xs, w4[i].z, b4[i].z);
            f[4 * i + 3] = fmaf(static_cast<float>(static_cast<int>(v[4 * i + 3])) * xs, w4[i].w, b4[i].w);
          }
#pragma unroll
          for (int j = 0; j < 32; j += kVec)
            *reinterpret_cast<uint4*>(stage + slot(lane, (h * 32 + j) / kVec)) = OutVec<T>::pack(f + j);
        }
        __syncwarp();
        const int row0 = lane / kPieces, piece = lane % kPieces;
        T* dst = static_cast<T*>(p.out) + (m0 + row0) * p.out_stride + n0 + c0 + piece * kVec;
        if (whole) {
          uint4 v[kPieces];
#pragma unroll
          for (int it = 0; it < kPieces; ++it) v[it] = *reinterpret_cast<const uint4*>(stage + slot(it * kRows + row0, piece));
#pragma unroll
          for (int it = 0; it < kPieces; ++it) *reinterpret_cast<uint4*>(dst + it * kRows * p.out_stride) = v[it];
        } else {
          const int n = n0 + c0 + piece * kVec;
#pragma unroll 1
          for (int it = 0; it < kPieces; ++it, dst += kRows * p.out_stride) {
            const uint4 v = *reinterpret_cast<const uint4*>(stage + slot(it * kRows + row0, piece));
            if (m0 + it * kRows + row0 >= p.m) continue;
            if (p.out_vec && n + kVec <= p.n) {
              *reinterpret_cast<uint4*>(dst) = v;
            } else {
              const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
              for (int i = 0; i < kVec; ++i)
                if (n + i < p.n) dst[i] = e[i];
            }
          }
        }
        __syncwarp();
      };
      constexpr int kWide = 8 * kVec;                  // 128 bytes of a row: 64 or 32 columns
#pragma unroll
      for (int c0 = 0; c0 + kWide <= kCols; c0 += kWide) emit(c0, std::integral_constant<int, kWide>{});
      if constexpr (kCols % kWide != 0) emit(kCols / kWide * kWide, std::integral_constant<int, kCols % kWide>{});
    }
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
