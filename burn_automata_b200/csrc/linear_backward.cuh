// linear_backward.cuh -- the linear layer's whole backward pass in one walk over
// the rows, for layers whose weights fit a block's memory.
//
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz
// With few weights and many rows this is bound by memory: dy, z and x have to
// be read and dx written, once.  A block walks tiles of 128 rows: TMA brings
// the tile's dy, z and x; eight warps turn dy into dz in place (and add up
// db); one thread issues both products; four warps write dx.  The tile of dz
// lies in shared memory as 128-byte lines of 64 outputs per row, which the
// tensor core reads as A (rows x outputs, k along a line) for dx and as A^T
// (outputs x rows, k across lines) for dW, so it is written once.  dW stays in
// TMEM over all tiles of the block; the blocks' sums meet in
// product_reduce_kernel in a fixed order.
// 1048576 rows of a 64 -> 128 relu layer in bf16: 139 us, 5.8 TB/s; the
// whole call, with the sums' kernel, 152 (separate passes for dz, dx and dW
// take 131 + 67 + 63).
#pragma once

#include "linear_product.cuh"

namespace npa {
namespace linear_tc {

constexpr int kFusedThreads = 512;     // 4 dx warps, 4 control, 8 for dz
constexpr int kFusedStages = 2;  // at most
// Tiles to a block at most: 512 accumulating steps of dW, as long as any sum
// stays in one accumulator (terms of one sign lose 1.1e-7 of it at each).
constexpr int kFusedTiles = kLongBlocks * kBK / kBM;

// A position in a ring of `slots` slots and the parity of its current phase.
struct RingCursor {
  int slots;
  uint32_t slot = 0, parity = 0;
  __device__ __forceinline__ void advance() {
    if (++slot == uint32_t(slots)) {
      slot = 0;
      parity ^= 1;
    }
  }
};

struct FusedBackward {
  int64_t rows;
  int inputs, outputs;
  int out_blocks, in_blocks;  // of 64 columns
  int k_pad, n_pad;           // outputs and inputs in whole 16s
  int m_blocks;               // of 128 outputs
  int stages;  // two where they fit, else one
  uint32_t stage_bytes, weight_bytes;
  uint32_t tmem_columns;
  uint32_t dx_idesc, dw_idesc;
  int act, has_z, want_dx, want_dw, want_db;
  float* dw_partials;  // [blocks][m_blocks * 128][pitch]
  int64_t pitch;
  float* db_partials;  // [blocks][outputs]
};

// Shared memory of a block: the stages (dy, z, x), the weights, dx's staging
// buffers and the barriers.
inline size_t fused_smem(const FusedBackward& f) {
  return size_t(f.stages) * f.stage_bytes + f.weight_bytes + 4 * 4096 + 1024 + 256;
}
// Static shared memory beside it (the column sums).
constexpr size_t kFusedStaticSmem = kLoaderWarps * 32 * 8 * sizeof(float);
inline bool fused_fits(const FusedBackward& f) {
  return fused_smem(f) + kFusedStaticSmem + 1024 <= kSmemLimit &&
         (f.m_blocks + 2) * f.n_pad <= 512 && f.k_pad <= 256 && f.n_pad <= 256;
}

template <class T>
__global__ void __launch_bounds__(kFusedThreads, 1)
fused_backward_kernel(const __grid_constant__ CUtensorMap map_dy, const __grid_constant__ CUtensorMap map_z,
                      const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                      const __grid_constant__ CUtensorMap map_dx, const __grid_constant__ FusedBackward f) {
  constexpr uint32_t kBlockBytes = kBM * 128;  // 128 rows of 64 columns
  extern __shared__ char smem_raw[];
  __shared__ float db_sums[kLoaderWarps * 32 * 8];
  const uint32_t raw = tc::smem_addr(smem_raw);
  const uint32_t base = (raw + 1023) & ~1023u;
  const uint32_t weights = base + f.stages * f.stage_bytes;
  const uint32_t out_base = weights + f.weight_bytes;
  const uint32_t full = out_base + 4 * 4096, ready = full + 8 * kFusedStages;
  const uint32_t empty = ready + 8 * kFusedStages, acc_full = empty + 8 * kFusedStages;
  const uint32_t acc_empty = acc_full + 16, weights_full = acc_empty + 16, dw_done = weights_full + 8;
  const uint32_t tmem_at = dw_done + 8;
  // within a stage
  const uint32_t z_off = f.out_blocks * kBlockBytes;
  const uint32_t x_off = (f.has_z ? 2 : 1) * f.out_blocks * kBlockBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kTma = 4, kMma = 5, kFirstSlope = 8;
  const int64_t tiles = (f.rows + kBM - 1) / kBM;

  let_next_launch();
  if (warp == kMma) {
    if (lane == 0) {
      for (int s = 0; s < kFusedStages; ++s) {
        tc::bar_init(full + 8 * s, 1);
        tc::bar_init(ready + 8 * s, kLoaderWarps);
        tc::bar_init(empty + 8 * s, 1);
        tc::bar_init(acc_full + 8 * s, 1);
        tc::bar_init(acc_empty + 8 * s, 4);
      }
      tc::bar_init(weights_full, 1);
      tc::bar_init(dw_done, 1);
      asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    __syncwarp();
    tc::tmem_alloc(tmem_at, f.tmem_columns);
    tc::fence_before();
  }
  __syncthreads();
  tc::fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(tmem) : "r"(tmem_at) : "memory");
  const uint32_t tmem_dx = tmem + f.m_blocks * f.n_pad;  // after dW's columns
  bool ok = true;

  if (warp == kTma) {
    if (lane == 0) {
      if (f.want_dx) {
        tc::bar_expect(weights_full, f.weight_bytes);
        for (int i = 0; i < f.in_blocks; ++i)
          tc::tma_load(weights + i * f.k_pad * 128, &map_w, i * 64, 0, weights_full);
      }
      RingCursor at{f.stages};
      uint32_t issued = 0;
      for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x, at.advance()) {
        ok = tc::bar_wait(empty + 8 * at.slot, at.parity ^ 1);
        if (!ok) break;
        if (issued < uint32_t(f.stages)) ++issued;
        const uint32_t bar = full + 8 * at.slot, stage = base + at.slot * f.stage_bytes;
        const int row = int(t * kBM);
        tc::bar_expect(bar, f.stage_bytes);
        for (int i = 0; i < f.out_blocks; ++i) {
          tc::tma_load(stage + i * kBlockBytes, &map_dy, i * 64, row, bar);
          if (f.has_z) tc::tma_load(stage + z_off + i * kBlockBytes, &map_z, i * 64, row, bar);
        }
        for (int i = 0; i < f.in_blocks; ++i)
          tc::tma_load(stage + x_off + i * kBlockBytes, &map_x, i * 64, row, bar);
      }
      if (!ok)  // copies in flight must land before the block may leave
        for (uint32_t j = 0; j < issued; ++j) {
          const uint32_t slot = (at.slot + f.stages - 1 - j) % f.stages;
          tc::bar_wait(full + 8 * slot, slot < at.slot ? at.parity : at.parity ^ 1);
        }
    }
  } else if (warp == kMma) {
    const uint32_t issue = tc::elected();
    RingCursor at{f.stages};
    Cursor<2> acc;
    if (f.want_dx) ok = __all_sync(0xffffffffu, tc::bar_wait(weights_full, 0));
    bool first = true;
    for (int64_t t = blockIdx.x; t < tiles && ok; t += gridDim.x, at.advance()) {
      ok = __all_sync(0xffffffffu, tc::bar_wait(ready + 8 * at.slot, at.parity));
      if (!ok) break;
      tc::fence_after();
      const uint32_t dz = base + at.slot * f.stage_bytes, x = dz + x_off;
      if (f.want_dx) {
        ok = __all_sync(0xffffffffu, tc::bar_wait(acc_empty + 8 * acc.slot, acc.parity ^ 1));
        if (!ok) break;
        tc::fence_after();
        const uint64_t a0 = tc::operand_desc(dz, false, 0);
        const uint64_t b0 = tc::operand_desc(weights, true, f.k_pad * 128);
        for (int k = 0; k < f.k_pad / 16; ++k)
          tc::mma_f16(tmem_dx + acc.slot * f.n_pad, a0 + ((k / 4 * kBlockBytes + k % 4 * 32) >> 4),
                      b0 + (k * 2048 >> 4), f.dx_idesc, k > 0, issue);
        tc::mma_commit(acc_full + 8 * acc.slot, issue);
        acc.advance();
      }
      if (f.want_dw) {
        const uint64_t b0 = tc::operand_desc(x, true, kBlockBytes);
        for (int m = 0; m < f.m_blocks; ++m) {
          const uint64_t a0 = tc::operand_desc(dz + m * 2 * kBlockBytes, true, kBlockBytes);
#pragma unroll
          for (int k = 0; k < kBM / 16; ++k)
            tc::mma_f16(tmem + m * f.n_pad, a0 + (k * 2048 >> 4), b0 + (k * 2048 >> 4), f.dw_idesc,
                        !first || k > 0, issue);
        }
      }
      first = false;
      tc::mma_commit(empty + 8 * at.slot, issue);
    }
    // dW is whole (and nothing is in flight) when this completes
    tc::mma_commit(dw_done, issue);
    if (!__all_sync(0xffffffffu, tc::bar_wait(dw_done, 0))) ok = false;
  } else if (warp >= kFirstSlope) {
    // dz in place of dy, and the columns' sums: a thread keeps eight columns
    const int tid = threadIdx.x - kFirstSlope * 32;
    const int chunks = f.out_blocks * 8, rows_at_once = kLoaderWarps * 32 / chunks;
    const int chunk = tid % chunks, row0 = tid / chunks;
    const uint32_t column = (chunk >> 3) * kBlockBytes;
    float sums[8] = {};
    RingCursor at{f.stages};
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x, at.advance()) {
      ok = __all_sync(0xffffffffu, tc::bar_wait(full + 8 * at.slot, at.parity));
      if (!ok) break;
      const uint32_t stage = base + at.slot * f.stage_bytes + column;
      if (row0 < rows_at_once && (f.has_z || f.want_db)) {
#pragma unroll 2
        for (int r = row0; r < kBM; r += rows_at_once) {
          const uint32_t where = stage + swizzled(r, chunk & 7);
          const uint4 g = load_shared16(where);
          const uint32_t gw[4] = {g.x, g.y, g.z, g.w};
          float d[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 p = unpack2<T>(gw[j]);
            d[2 * j] = p.x;
            d[2 * j + 1] = p.y;
          }
          if (f.has_z) {
            const uint4 zz = load_shared16(where + z_off);
            const uint32_t zw[4] = {zz.x, zz.y, zz.z, zz.w};
            float zf[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 p = unpack2<T>(zw[j]);
              zf[2 * j] = p.x;
              zf[2 * j + 1] = p.y;
            }
            times_slope<true>(f.act, d, zf);
            store_shared16(where, make_uint4(pack2<T>(d[0], d[1]), pack2<T>(d[2], d[3]),
                                             pack2<T>(d[4], d[5]), pack2<T>(d[6], d[7])));
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) sums[j] += d[j];
        }
      }
      tc::fence_async_shared();
      __syncwarp();
      if (lane == 0) tc::bar_arrive(ready + 8 * at.slot);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) db_sums[tid * 8 + j] = row0 < rows_at_once ? sums[j] : 0.0f;
    asm volatile("bar.sync 1, %0;\n" ::"n"(kLoaderWarps * 32) : "memory");  // these warps only
    if (f.want_db)
      for (int c = tid; c < f.outputs; c += kLoaderWarps * 32) {
        float s = 0.0f;
        for (int q = 0; q < rows_at_once; ++q) s += db_sums[(q * chunks + c / 8) * 8 + c % 8];
        f.db_partials[int64_t(blockIdx.x) * f.outputs + c] = s;
      }
  } else if (warp < 4) {
    const uint32_t lanes = uint32_t(warp * 32) << 16, buf = out_base + warp * 4096;
    if (f.want_dx) {
      Cursor<2> acc;
      for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x, acc.advance()) {
        ok = __all_sync(0xffffffffu, tc::bar_wait(acc_full + 8 * acc.slot, acc.parity));
        if (!ok) break;
        tc::fence_after();
        const int row = int(t * kBM) + warp * 32;
        for (int c = 0; c < f.in_blocks; ++c) {
          float v[64];
#pragma unroll
          for (int h = 0; h < 64; h += 16) {
            float part[16] = {};
            if (c * 64 + h < f.n_pad)
              tc::tmem_load(tmem_dx + lanes + acc.slot * f.n_pad + c * 64 + h, part);
#pragma unroll
            for (int j = 0; j < 16; ++j) v[h + j] = part[j];
          }
          if (c + 1 == f.in_blocks) {
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tc::bar_arrive(acc_empty + 8 * acc.slot);
          }
          if (lane == 0) tc::bulk_wait_read<0>();
          __syncwarp();
          stage_values<T>(buf, lane, v, 0);
          tc::fence_async_shared();
          __syncwarp();
          if (lane == 0) {
            tc::tma_store(&map_dx, c * 64, row, buf);
            tc::bulk_commit();
          }
        }
      }
      if (lane == 0) tc::bulk_wait_all();
    }
    if (f.want_dw && ok) {
      ok = __all_sync(0xffffffffu, tc::bar_wait(dw_done, 0));
      tc::fence_after();
      for (int m = 0; m < f.m_blocks && ok; ++m) {
        float* const to = f.dw_partials +
                          ((int64_t(blockIdx.x) * f.m_blocks + m) * kBM + warp * 32 + lane) * f.pitch;
        for (int c = 0; c < f.n_pad; c += 16) {
          float v[16];
          tc::tmem_load(tmem + lanes + m * f.n_pad + c, v);
#pragma unroll
          for (int j = 0; j < 16; j += 4)
            if (c + j < f.pitch)
              *reinterpret_cast<float4*>(to + c + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
        }
      }
    }
  }
  if (!ok && lane == 0) atomicAdd(&g_timeouts, 1ull);
  tc::fence_before();
  __syncthreads();
  if (warp == kMma) {
    tc::fence_after();
    tc::tmem_free(tmem, f.tmem_columns);
  }
}

}  // namespace linear_tc
}  // namespace npa
