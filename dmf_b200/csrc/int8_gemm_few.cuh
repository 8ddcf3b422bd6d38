// The 8-bit product for few rows: the weight is the wide operand of the tensor cores.
//
// A CTA computes 128 output channels of TB tokens as D[channel, token] = w x^T (tcgen05.mma of kind::i8, M = 128, N = TB); the
// CTAs of a cluster share such a tile and split k among them, so that even one token's product has every SM read its part of the
// weight.  Each CTA sends the other CTAs their columns of its sums (int32: exact, the order does not matter) through distributed
// shared memory; after one cluster barrier CTA r adds up columns [r TB / S, (r + 1) TB / S), scales them and writes them, 32
// consecutive channels of a token per warp instruction.
//
// What bounds it: latency.  Of the 4.5 us that 1 x 1152 x 6912 takes, 1.2 are the weight's 8 MB at the HBM's rate; 2.9 us is what 3
// steps of k take in one tile, and every further step 0.21 (18 to 24 KB at the 90 to 115 GB/s that an SM takes in from the L2).  A split k costs 1 to 4 us, so only long
// sums are split: 16 x 4608 x 1152 takes 10.0 us in one piece and 4.6 in eight.  With wide tiles most of that is bank conflicts: `sums`
// holds the columns of a channel side by side, so the lanes of a warp, a channel each, read and send at a stride of `cols` words - 2-way
// conflicts at 16 tokens in eight pieces, 16-way at 32 in two, 32-way at 64 in two (shared-memory wavefronts of a CTA's reads, and those
// that conflicts add: 157 and 64, 2133 and 1920, 8179 and 7826).  (Bulk copies between the CTAs instead of stores: 2
// us more; CTAs of a cluster on SMs of their own: clusters of four do not fill the GPU, 6.3 -> 11.3 us at 64 x 4608 x 1152.)
#pragma once

#include <type_traits>

#include "int8_gemm_pair.cuh"

namespace dmf {

template <int TB>
struct Int8FewTraits {
  static constexpr int kWBytes = 128 * 128, kXBytes = TB * 128, kStageBytes = kWBytes + kXBytes;
  static constexpr int kStages = TB == 16 ? 5 : (TB == 32 ? 4 : 3);     // two CTAs per SM
  static constexpr int kRingBytes = kStages * kStageBytes;
  static constexpr int kSumBytes = TB * 128 * 4;
  static constexpr int kBarFull = 0, kBarEmpty = kStages, kBarAcc = 2 * kStages, kNumBars = kBarAcc + 1;
  static constexpr int kSmemBytes = 1024 + kRingBytes + kSumBytes + TB * 4 + kNumBars * 8 + 16;
  static constexpr uint32_t kTmemCols = TB < 32 ? 32 : TB;
};

constexpr int kInt8FewThreads = 192;

template <int TB, typename T>
__global__ void __launch_bounds__(kInt8FewThreads) int8_gemm_few_kernel(const __grid_constant__ Int8GemmParams p, int splits) {
  using TR = Int8FewTraits<TB>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t s_ring = smem_u32(smem);
  int* sums = reinterpret_cast<int*>(smem + TR::kRingBytes);     // [source CTA][channel][column of mine]
  float* s_x = reinterpret_cast<float*>(smem + TR::kRingBytes + TR::kSumBytes);   // the tokens' scales (16-byte aligned)
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + TR::kRingBytes + TR::kSumBytes + TB * 4);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + TR::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](int i) -> uint32_t { return bar0 + 8u * static_cast<uint32_t>(i); };

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x) % splits, tile = static_cast<int>(blockIdx.x) / splits;
  const int tn = tile % p.tiles_n, tm = tile / p.tiles_n;
  const int k_steps = (p.k + 127) >> 7;
  const int k0 = static_cast<int>(static_cast<int64_t>(k_steps) * rank / splits);
  const int k1 = static_cast<int>(static_cast<int64_t>(k_steps) * (rank + 1) / splits);   // splits <= k_steps: never empty

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < TR::kNumBars; ++i) mbar_init(bar(i), 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    __syncwarp();
    tmem_alloc(smem_u32(tmem_slot), TR::kTmemCols);
    tmem_relinquish_alloc_permit();
  }
  tc_fence_before_sync();
  __syncthreads();
  if (splits > 1) cluster_sync_all();  // the others' shared memory is theirs from here on
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  grid_dependency_wait();
  grid_launch_dependents();

  if (warp == 0) {
    if (lane == 0) {
      prefetch_tensor_map(&p.w_map);
      prefetch_tensor_map(&p.x_map);
      for (int kk = k0, cnt = 0; kk < k1; ++kk, ++cnt) {
        const uint32_t s = cnt % TR::kStages, ph = (cnt / TR::kStages) & 1u;
        if (!mbar_wait(bar(TR::kBarEmpty + s), ph ^ 1u, abort_flag, p.status_word, kRoleInt8Producer + TR::kBarEmpty + s)) break;
        const uint32_t dst = s_ring + s * TR::kStageBytes;
        mbar_arrive_expect_tx(bar(TR::kBarFull + s), TR::kStageBytes);
        tma_load_2d(dst, &p.w_map, bar(TR::kBarFull + s), kk * 128, tn * 128);
        tma_load_2d(dst + TR::kWBytes, &p.x_map, bar(TR::kBarFull + s), kk * 128, tm * TB);
      }
    }
  } else if (warp == 1) {
    const bool leader = elect_one();
    constexpr uint32_t idesc = make_idesc_i8(128, TB);
    bool ok = true;
    for (int kk = k0, cnt = 0; kk < k1; ++kk, ++cnt) {
      const uint32_t s = cnt % TR::kStages, ph = (cnt / TR::kStages) & 1u;
      ok = mbar_wait(bar(TR::kBarFull + s), ph, abort_flag, p.status_word, kRoleInt8Mma + TR::kBarFull + s);
      if (!ok) break;
      tc_fence_after_sync();
      const uint32_t ws = s_ring + s * TR::kStageBytes, xs = ws + TR::kWBytes;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        mma_i8(tmem, make_smem_desc(ws + i * 32, 16, 1024, kSwizzle128), make_smem_desc(xs + i * 32, 16, 1024, kSwizzle128), idesc,
               (kk > k0 || i > 0) ? 1u : 0u, leader);
      tc_commit(bar(TR::kBarEmpty + s), leader);
    }
    if (ok) tc_commit(bar(TR::kBarAcc), leader);
  }

  // warps 2..5: a lane has one channel
  const int quarter = warp & 3;
  const int channel = quarter * 32 + lane;
  const int64_t n = static_cast<int64_t>(tn) * 128 + channel;
  const int m0 = tm * TB;
  T* out = static_cast<T*>(p.out) + n;
  const bool mine = warp >= 2 && n < p.n;
  float ws = 0.f, b = 0.f;
  bool ok = false;
  if (warp >= 2) {
    if (mine) {
      ws = p.w_scale[n];
      b = p.bias != nullptr ? row_load(p.bias, p.bias_dtype, n) : 0.f;
    }
    if (threadIdx.x - 64 < TB) s_x[threadIdx.x - 64] = m0 + static_cast<int>(threadIdx.x) - 64 < p.m ? p.x_scale[m0 + threadIdx.x - 64] : 0.f;
    named_bar_sync(1, 128);
    ok = __all_sync(0xffffffffu, mbar_wait(bar(TR::kBarAcc), 0, abort_flag, p.status_word, kRoleInt8Epilogue + TR::kBarAcc));
    tc_fence_after_sync();
  }
  auto scaled = [&](int sum, float x_scale) { return fmaf(static_cast<float>(sum) * x_scale, ws, b); };
  auto store = [&](T* dst, float y) {
    if constexpr (std::is_same<T, float>::value) *dst = y;
    else *dst = T(y);
  };
  constexpr int kChunk = TB < 32 ? TB : 32;
  const int cols = TB / splits, shift = __ffs(cols) - 1;   // columns of a CTA: a power of two, 2 at least
  const uint32_t lane_base = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  if (ok) {
#pragma unroll
    for (int c0 = 0; c0 < TB; c0 += kChunk) {
      if (m0 + c0 >= p.m) break;
      uint32_t v[kChunk];
      if constexpr (kChunk == 16) tmem_ld_x16(lane_base + c0, v);
      else tmem_ld_x32(lane_base + c0, v);
      tmem_wait_ld();
      if (splits == 1) {
        // all scales before the first store, which they would otherwise wait for (64 tokens: 3.2 us of epilogue)
        float y[kChunk];
#pragma unroll
        for (int j = 0; j < kChunk; j += 4) {
          const float4 x = *reinterpret_cast<const float4*>(s_x + c0 + j);
          y[j] = scaled(static_cast<int>(v[j]), x.x);
          y[j + 1] = scaled(static_cast<int>(v[j + 1]), x.y);
          y[j + 2] = scaled(static_cast<int>(v[j + 2]), x.z);
          y[j + 3] = scaled(static_cast<int>(v[j + 3]), x.w);
        }
        if (mine) {
          T* dst = out + static_cast<int64_t>(m0 + c0) * p.out_stride;
          const int count = min(kChunk, p.m - m0 - c0);
#pragma unroll
          for (int j = 0; j < kChunk; ++j, dst += p.out_stride)
            if (j < count) store(dst, y[j]);
        }
      } else {
        // to the column's owner, columns of one channel side by side; tokens that are none travel too, nobody reads them
        auto at = [&](int c) -> uint32_t {
          return map_to_cta(smem_u32(sums + (rank * 128 + channel) * cols + (c & (cols - 1))), c >> shift);
        };
        if (cols >= 4) {
#pragma unroll
          for (int j = 0; j < kChunk; j += 4) st_shared_cluster_v4(at(c0 + j), v[j], v[j + 1], v[j + 2], v[j + 3]);
        } else {
#pragma unroll
          for (int j = 0; j < kChunk; j += 2) st_shared_cluster_v2(at(c0 + j), v[j], v[j + 1]);
        }
      }
    }
  }
  if (splits > 1) {
    __syncwarp();
    cluster_sync_all();                          // everybody's sums have arrived
    if (ok)
      for (int c = 0; c < cols && m0 + rank * cols + c < p.m; ++c) {
        int s = 0;
        for (int r = 0; r < splits; ++r) s += sums[(r * 128 + channel) * cols + c];
        if (mine) store(out + static_cast<int64_t>(m0 + rank * cols + c) * p.out_stride, scaled(s, s_x[rank * cols + c]));
      }
  }
  __syncwarp();
  int8_drain(abort_flag);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 1) tmem_dealloc(tmem, TR::kTmemCols);
}

}  // namespace dmf
