// linear.cu -- matrix product with bias, activation and residual, and its
// backward pass.
//
//   z = x W^T + b,  y = act(z) + r;  dz = dy act'(z),
//   dx = dz W,  dW = dz^T x,  db = sum over rows of dz.
// The three products run on product_kernel (linear_product.cuh); the sums over
// rows that give db, and dz itself, come from slope_kernel.
#include <algorithm>
#include <atomic>

#include "linear_backward.cuh"

namespace npa {
namespace {

using linear_tc::FusedBackward;
using linear_tc::load_ragged;
using linear_tc::Operand;
using linear_tc::Product;

// ---- the split product's layers, summed in order, with the epilogue ----
// Column sums that wait to be added: [count][outputs].
struct BiasSums {
  const float* partials;  // null: none
  int count, outputs;
  void* dbias;
};
// 32 outputs by a block; its eight warps each add every eighth partial in order.
template <class T>
__device__ __forceinline__ void reduce_bias(const BiasSums& b, int block) {
  __shared__ float acc[8][32];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int col = block * 32 + tx;
  float s = 0.0f;
  if (col < b.outputs)
#pragma unroll 8
    for (int p = ty; p < b.count; p += 8) s += b.partials[int64_t(p) * b.outputs + col];
  acc[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && col < b.outputs)
    static_cast<T*>(b.dbias)[col] =
        from_f32<T>(((acc[0][tx] + acc[1][tx]) + (acc[2][tx] + acc[3][tx])) +
                    ((acc[4][tx] + acc[5][tx]) + (acc[6][tx] + acc[7][tx])));
}
// A block has 32 groups of four columns; its eight warps each add every eighth
// layer, and the first adds the eight sums in order.  The blocks past `blocks`
// add a bias gradient on the way: a launch less.
template <class T>
__global__ void __launch_bounds__(256) product_reduce_kernel(const __grid_constant__ Product p, int blocks,
                                                             const __grid_constant__ BiasSums bias) {
  let_next_launch();
  wait_for_previous();
  if (int(blockIdx.x) >= blocks) {
    reduce_bias<T>(bias, int(blockIdx.x) - blocks);
    return;
  }
  __shared__ float4 sums[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t quads = (p.n + 3) / 4;
  const int64_t e = int64_t(blockIdx.x) * 32 + lane;
  const bool mine = e < int64_t(p.m) * quads;
  const int64_t row = e / quads, col = e % quads * 4;
  const int64_t layer = p.layer_rows * p.partial_pitch;
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (mine) {
    const float* const at = p.partials + row * p.partial_pitch + col;
#pragma unroll 8
    for (int s = warp; s < p.splits; s += 8) {
      const float4 f = *reinterpret_cast<const float4*>(at + s * layer);
      v.x += f.x;
      v.y += f.y;
      v.z += f.z;
      v.w += f.w;
    }
  }
  sums[warp][lane] = v;
  __syncthreads();
  if (warp != 0 || !mine) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) {
    const float4 f = sums[w][lane];
    v.x += f.x;
    v.y += f.y;
    v.z += f.z;
    v.w += f.w;
  }
  const float total[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (col + j >= p.n) break;
    float z = total[j];
    if (p.bias) z += to_f32(static_cast<const T*>(p.bias)[col + j]);
    if (p.z) static_cast<T*>(p.z)[row * p.z_stride + col + j] = from_f32<T>(z);
    float y = linear_tc::activation<sizeof(T) == 2>(p.act, z);
    if (p.residual)
      y += to_f32(static_cast<const T*>(p.residual)[row * p.residual_stride + col + j]);
    static_cast<T*>(p.y)[row * p.y_stride + col + j] = from_f32<T>(y);
  }
}

// ---- a few rows: bound by reading the weights once ----
constexpr int kFewRows = 8;

// A warp has OUTS outputs of all R rows and walks k with 16-byte loads (VEC
// values; single values where a row does not start on 16 bytes).  Plain f32
// products: at eight rows a weight read from memory still costs more than its
// eight multiply-adds.  One row of a 1024 -> 4096 bf16 layer: 4.0 us on the device
// with the weights in memory, against 8.2 for split tiles and their sum.
template <class T, int R, int OUTS, int VEC>
__global__ void __launch_bounds__(256) few_rows_kernel(const __grid_constant__ LinearArgs a) {
  using P = Pack<T, VEC>;
  const int lane = threadIdx.x & 31;
  const int64_t first = (int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5)) * OUTS;
  if (first >= a.outputs) return;
  const T* const w = static_cast<const T*>(a.weight);
  const T* const x = static_cast<const T*>(a.x);
  float acc[R][OUTS];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int o = 0; o < OUTS; ++o) acc[r][o] = 0.0f;
  const int rows = int(a.rows);
#pragma unroll 2
  for (int k = lane * VEC; k < a.inputs; k += 32 * VEC) {
    P wv[OUTS];
#pragma unroll
    for (int o = 0; o < OUTS; ++o)  // past the last output: the last one again
      wv[o] = *reinterpret_cast<const P*>(w + min(first + o, int64_t(a.outputs) - 1) * a.weight_stride + k);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const P xv = *reinterpret_cast<const P*>(x + int64_t(min(r, rows - 1)) * a.x_stride + k);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float xf = to_f32(xv.v[j]);
#pragma unroll
        for (int o = 0; o < OUTS; ++o) acc[r][o] += xf * to_f32(wv[o].v[j]);
      }
    }
  }
  float mine = 0.0f;  // lane r * OUTS + o keeps (r, o)
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int o = 0; o < OUTS; ++o) {
      float s = acc[r][o];
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      if (lane == r * OUTS + o) mine = s;
    }
  const int r = lane / OUTS;
  const int64_t col = first + lane % OUTS;
  if (r >= R || r >= rows || col >= a.outputs) return;
  float z = mine;
  if (a.bias) z += to_f32(static_cast<const T*>(a.bias)[col]);
  if (a.z) static_cast<T*>(a.z)[r * a.z_stride + col] = from_f32<T>(z);
  float y = linear_tc::activation<sizeof(T) == 2>(a.activation, z);
  if (a.residual) y += to_f32(static_cast<const T*>(a.residual)[r * a.residual_stride + col]);
  static_cast<T*>(a.y)[r * a.y_stride + col] = from_f32<T>(y);
}
template <class T, int R>
npa_status launch_few_rows(const LinearArgs& a, bool vec, cudaStream_t s) {
  constexpr int kVec = 16 / int(sizeof(T));
  // One output to a warp, or four for two rows or more whose outputs would take
  // more than three quarters of a wave of such warps: a weight is then read for
  // several rows, and x for four outputs at once (bf16 2 x 1024 -> 4096 4.9 us, four
  // 5.2; -> 8192 8.1 and 6.4; 8 x 1024 -> 2560 7.0 and 7.4; -> 3584 8.8 and 7.5; but
  // 1 x 1024 -> 4096 4.0 and 6.3, -> 32768 14.2 and 15.4).
  bool four = false;
  if (R > 1 && a.outputs > 2048) {
    int per_sm = 0, sms = 0;
    const void* const one = vec ? reinterpret_cast<const void*>(few_rows_kernel<T, R, 1, kVec>)
                                : reinterpret_cast<const void*>(few_rows_kernel<T, R, 1, 1>);
    NPA_TRY(kernel_occupancy(one, 256, 0, &per_sm, &sms));
    four = a.outputs > int64_t(per_sm) * sms * 8 * 3 / 4;
  }
  if (four) {
    const unsigned grid = unsigned((a.outputs + 31) / 32);
    if (vec)
      few_rows_kernel<T, R, 4, kVec><<<grid, 256, 0, s>>>(a);
    else
      few_rows_kernel<T, R, 4, 1><<<grid, 256, 0, s>>>(a);
  } else {
    const unsigned grid = unsigned((a.outputs + 7) / 8);
    if (vec)
      few_rows_kernel<T, R, 1, kVec><<<grid, 256, 0, s>>>(a);
    else
      few_rows_kernel<T, R, 1, 1><<<grid, 256, 0, s>>>(a);
  }
  return after_launch("linear few_rows_kernel");
}

// The backward pass of a few rows as one kernel.  A block has a slab of inputs
// and all outputs: LANES threads side by side have the slab (VEC inputs each),
// the block's groups of them share the outputs out.  W's slab is read once (dx)
// and dW's written on the way; the groups' shares of dx meet in shared memory.
template <class T, int R, int VEC, int LANES>
__global__ void __launch_bounds__(256) few_rows_backward_kernel(const __grid_constant__ LinearBackwardArgs a) {
  using P = Pack<T, VEC>;
  constexpr int kGroups = 256 / LANES, kSlab = LANES * VEC;
  __shared__ float sums[8][R][kSlab];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int in_group = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int64_t col = int64_t(blockIdx.x) * kSlab + in_group * VEC;
  const bool mine = col < a.inputs;
  const int rows = int(a.rows);
  const T* const w = static_cast<const T*>(a.weight);
  float acc[R][VEC];
  P x[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[r][j] = 0.0f;
    x[r] = P{};
    if (a.dweight && mine && r < rows)
      x[r] = *reinterpret_cast<const P*>(static_cast<const T*>(a.x) + r * a.x_stride + col);
  }
  // every lane of a warp makes the same number of turns: they exchange dz
#pragma unroll 2
  for (int o0 = 0; o0 < a.outputs; o0 += kGroups) {
    const int64_t o = o0 + group;
    const bool there = o < a.outputs;
    P wv{};
    if (a.dx && there && mine) wv = *reinterpret_cast<const P*>(w + o * a.weight_stride + col);
    // lane r of every eight has row r's dz
    float d = 0.0f;
    if (there && (lane & 7) < rows) {
      const int64_t r = lane & 7;
      d = to_f32(static_cast<const T*>(a.dy)[r * a.dy_stride + o]);
      if (a.z)
        d *= linear_tc::activation_slope<sizeof(T) == 2>(
            a.activation, to_f32(static_cast<const T*>(a.z)[r * a.z_stride + o]));
    }
    float dw[VEC], db = 0.0f;
#pragma unroll
    for (int j = 0; j < VEC; ++j) dw[j] = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float dr = __shfl_sync(0xffffffffu, d, (lane & ~7) | r);
      if (r < rows) {
        db += dr;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          acc[r][j] += dr * to_f32(wv.v[j]);
          dw[j] += dr * to_f32(x[r].v[j]);
        }
      }
    }
    if (there && mine && a.dweight) {
      P out;
#pragma unroll
      for (int j = 0; j < VEC; ++j) out.v[j] = from_f32<T>(dw[j]);
      *reinterpret_cast<P*>(static_cast<T*>(a.dweight) + o * a.inputs + col) = out;
    }
    if (there && a.dbias && blockIdx.x == 0 && in_group == 0)
      static_cast<T*>(a.dbias)[o] = from_f32<T>(db);
  }
  if (!a.dx) return;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      float s = acc[r][j];
#pragma unroll
      for (int d = LANES; d < 32; d <<= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      if (lane < LANES) sums[warp][r][in_group * VEC + j] = s;
    }
  __syncthreads();
  for (int e = threadIdx.x; e < R * kSlab; e += 256) {
    const int r = e / kSlab, c = e % kSlab;
    const int64_t at = int64_t(blockIdx.x) * kSlab + c;
    if (r >= rows || at >= a.inputs) continue;
    float s = 0.0f;
#pragma unroll
    for (int q = 0; q < 8; ++q) s += sums[q][r][c];
    static_cast<T*>(a.dx)[r * a.dx_stride + at] = from_f32<T>(s);
  }
}
template <class T, int R>
npa_status launch_few_rows_backward(const LinearBackwardArgs& a, bool vec, cudaStream_t s) {
  constexpr int kVec = 16 / int(sizeof(T));
  if (vec)
    few_rows_backward_kernel<T, R, kVec, 8>
        <<<unsigned((a.inputs + 8 * kVec - 1) / (8 * kVec)), 256, 0, s>>>(a);
  else
    few_rows_backward_kernel<T, R, 1, 32><<<unsigned((a.inputs + 31) / 32), 256, 0, s>>>(a);
  return after_launch("linear few_rows_backward_kernel");
}
// Few enough that a block's walk over all outputs stays short (a kernel or
// three less to launch than the tiles' way, which is what such calls cost).
bool few_rows_backward(int64_t rows, int outputs) {
  return rows <= kFewRows && rows * outputs <= 4096;
}

// ---- dz and the bias gradient ----
struct SlopeArgs {
  const void* dy;
  int64_t dy_stride;
  const void* z;  // null: dz = dy
  int64_t z_stride;
  int64_t rows;
  int outputs;
  int64_t rows_per_block;
  int act;
  void* dz;  // optional
  int64_t dz_stride;
  float* partials;  // [gridDim.y][outputs]
  int tx;           // column groups per block, a power of two
};
// dz = dy act'(z) rounded to the storage type, and each block's column sums of
// the unrounded values.  A thread has 16 bytes of every (256 / tx)th row; RAGGED:
// of rows that start anywhere or end within them (dz's rows are whole, zero past
// the outputs).
// Blocks to an SM, all in one wave: three, but two of the aligned bf16 kernel, which
// spills at 80 registers (16384 x 1024 -> 4096 backward, us with three and two: bf16
// silu 321 and 275, gelu 372 and 333, relu 342 and 304; f16 silu 315 and 321; with
// four f16 took a second wave, 31 more).
template <class T, bool RAGGED>
constexpr int kSlopeBlocks = std::is_same<T, __nv_bfloat16>::value && !RAGGED ? 2 : 3;
template <class T, bool RAGGED>
__global__ void __launch_bounds__(256, (kSlopeBlocks<T, RAGGED>)) slope_kernel(const __grid_constant__ SlopeArgs a) {
  let_next_launch();
  wait_for_previous();
  constexpr int VEC = 16 / int(sizeof(T));
  using P = Pack<T, VEC>;
  __shared__ float sums[256 * VEC];
  constexpr int kAhead = RAGGED ? 2 : 4;  // rows in flight per thread
  const int tx = threadIdx.x & (a.tx - 1), ty = threadIdx.x / a.tx, rows_at_once = 256 / a.tx;
  const int64_t col = (int64_t(blockIdx.x) * a.tx + tx) * VEC;
  const bool mine = col < a.outputs;
  const int valid = mine ? int(min(int64_t(VEC), a.outputs - col)) : 0;
  const int64_t begin = int64_t(blockIdx.y) * a.rows_per_block;
  const int64_t end = min(begin + a.rows_per_block, a.rows);
  const T* const dy = static_cast<const T*>(a.dy) + col;
  const T* const z = static_cast<const T*>(a.z) + col;
  T* const dz = static_cast<T*>(a.dz) + col;
  auto read = [&](const T* p, int64_t r) -> P {
    if (!RAGGED) return *reinterpret_cast<const P*>(p);
    return load_ragged<T>(p, valid, (r > 0 || col > 0) && r + 1 < a.rows);
  };
  float s[VEC] = {};
  if (mine) {
    for (int64_t r0 = begin + ty; r0 < end; r0 += int64_t(kAhead) * rows_at_once) {
      P g[kAhead], zz[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int64_t r = r0 + int64_t(i) * rows_at_once;
        if (r < end) {
          g[i] = read(dy + r * a.dy_stride, r);
          if (a.z) zz[i] = read(z + r * a.z_stride, r);
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int64_t r = r0 + int64_t(i) * rows_at_once;
        if (r >= end) break;
        float d[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) d[j] = to_f32(g[i].v[j]);
        if (a.z) {
          float zf[VEC];
#pragma unroll
          for (int j = 0; j < VEC; ++j) zf[j] = to_f32(zz[i].v[j]);
          linear_tc::times_slope<sizeof(T) == 2>(a.act, d, zf);
        }
        P out;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          s[j] += d[j];
          out.v[j] = from_f32<T>(d[j]);
        }
        if (a.dz) *reinterpret_cast<P*>(dz + r * a.dz_stride) = out;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) sums[j * 256 + threadIdx.x] = s[j];
  __syncthreads();
  for (int c = threadIdx.x; c < a.tx * VEC; c += 256) {
    const int64_t at = int64_t(blockIdx.x) * a.tx * VEC + c;
    if (at >= a.outputs) continue;
    float t = 0.0f;
    for (int q = 0; q < rows_at_once; ++q) t += sums[(c % VEC) * 256 + q * a.tx + c / VEC];
    a.partials[int64_t(blockIdx.y) * a.outputs + at] = t;
  }
}
template <class T>
__global__ void __launch_bounds__(256) bias_reduce_kernel(const __grid_constant__ BiasSums bias) {
  let_next_launch();
  wait_for_previous();
  reduce_bias<T>(bias, int(blockIdx.x));
}
template <class T>
npa_status launch_bias_reduce(const BiasSums& b, cudaStream_t s) {
  NPA_CUDA(launch_kernel(true, bias_reduce_kernel<T>, dim3(grid_for(b.outputs, 32)), 256, 0, s, b),
           "bias_reduce_kernel");
  return after_launch("bias_reduce_kernel");
}
template <class T>
npa_status launch_product_reduce(const Product& p, const BiasSums& b, cudaStream_t s) {
  const unsigned blocks = grid_for(uint64_t(p.m) * ((p.n + 3) / 4), 32);
  const unsigned more = b.partials ? grid_for(b.outputs, 32) : 0;
  NPA_CUDA(launch_kernel(true, product_reduce_kernel<T>, dim3(blocks + more), 256, 0, s, p, int(blocks), b),
           "product_reduce_kernel");
  return after_launch("product_reduce_kernel");
}

// ---- rows of odd widths, copied to rows that start on 16 bytes ----
// A thread writes 16 bytes; past the width they are zero.
template <class T>
__global__ void __launch_bounds__(256) pack_kernel(const T* __restrict__ from, int64_t stride, int64_t rows,
                                                   int width, T* __restrict__ to, int64_t pitch) {
  constexpr int kChunk = 16 / int(sizeof(T));
  let_next_launch();
  wait_for_previous();
  const int64_t chunks = pitch / kChunk;
  const int64_t e = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (e >= rows * chunks) return;
  const int64_t row = e / chunks;
  const int col = int(e % chunks) * kChunk;
  Pack<T, kChunk> out{};
  if (col < width)
    out = load_ragged<T>(from + row * stride + col, min(kChunk, width - col),
                         (row > 0 || col > 0) && row + 1 < rows);
  *reinterpret_cast<Pack<T, kChunk>*>(to + row * pitch + col) = out;
}
int64_t packed_pitch(int width) { return (int64_t(width) + 7) / 8 * 8; }
// Replaces an operand's rows by a packed copy in `to`.
template <class T>
npa_status pack_rows(Operand& o, void* to, bool after, cudaStream_t s) {
  const int64_t pitch = packed_pitch(o.width), rows = o.rows;
  const T* const from = static_cast<const T*>(o.p);
  const dim3 grid(grid_for(uint64_t(rows) * (pitch * sizeof(T) / 16), 256));
  NPA_CUDA(launch_kernel(after, pack_kernel<T>, grid, 256, 0, s, from, o.ld, rows, o.width,
                         static_cast<T*>(to), pitch),
           "linear pack_kernel");
  o.p = to;
  o.ld = pitch;
  o.width = int(pitch);  // zeros past the width
  return after_launch("linear pack_kernel");
}
// Whether operands with rows of an odd width are packed: where the loader warps
// would lose more than the copies take.  bf16: 65536 x 130 x 128 takes 27 us
// unpacked and 21 packed, 8192 x 1001 x 1000 190 and 28.  f32 goes through the
// loader warps either way and gains only what aligned loads save, once for each
// tile of outputs: 8192 x 1001 x 1000 takes 203 us unpacked and 135 packed,
// 70000 x 131 x 600 186 and 146.
bool packs(size_t size, int width, int64_t rows, int inputs, int outputs) {
  return width * size % 16 != 0 && rows > kFewRows &&
         double(rows) * inputs * outputs >= double(1 << 29) &&
         (size == 2 || outputs >= 384);
}

// ---- host side ----
constexpr int kSms = 148;             // the plans' block count: B200's SMs
constexpr int kBiasBlocks = 3 * kSms;  // of slope_kernel at most

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) !=
            cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      p = nullptr;
    }
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

template <class T>
constexpr CUtensorMapDataType tma_type() {
  return sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                        : (std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                          : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
}

// Rows that TMA can address: 16-byte aligned starts, strides below 2^40 bytes.
bool tma_rows(const void* p, int64_t stride, int64_t rows, size_t size) {
  if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  return rows <= 1 || (stride * int64_t(size) % 16 == 0 && stride * int64_t(size) < (int64_t(1) << 40));
}

// A map of `rows` rows of `width` values in boxes of box_rows x 128 bytes,
// 128-byte swizzled; values outside read as zero and are not written.
template <class T>
npa_status make_map(CUtensorMap* map, const void* p, int64_t width, int64_t rows, int64_t stride,
                    int box_rows) {
  const EncodeTiled encode = encode_tiled();
  if (!encode) return fail(NPA_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[2] = {cuuint64_t(width), cuuint64_t(rows)};
  const cuuint64_t pitch =
      rows <= 1 ? cuuint64_t((width * sizeof(T) + 15) / 16 * 16) : cuuint64_t(stride * sizeof(T));
  const cuuint32_t box[2] = {cuuint32_t(128 / sizeof(T)), cuuint32_t(box_rows)};
  const cuuint32_t step[2] = {1, 1};
  const CUresult r = encode(map, tma_type<T>(), 2, const_cast<void*>(p), dims, &pitch, box, step,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(NPA_ERR_CUDA, "cuTensorMapEncodeTiled failed with " + std::to_string(int(r)));
  return NPA_OK;
}

int ceil_div(int64_t a, int64_t b) { return int((a + b - 1) / b); }

// Tile shape and k splits of an m x n x k product.
struct Plan {
  int bn;
  bool pair;
  int m_tiles, n_tiles, k_blocks, splits, split_blocks;
  int64_t layer_rows, partial_pitch;
  size_t partial_bytes() const {
    return splits > 1 ? size_t(splits) * layer_rows * partial_pitch * 4 : 0;
  }
};
Plan plan_product(size_t size, bool tma, int64_t m, int64_t n, int64_t k) {
  Plan p{};
  p.k_blocks = ceil_div(k, linear_tc::kBK);
  p.partial_pitch = (n + 3) / 4 * 4;
  // The shape with the least time on the fullest SM, in units of 100 cycles: a
  // tile takes its k blocks or its epilogue, whichever is longer, as measured
  // (8192 x 4096 x 4096: 7 units a block in a pair's tile; 607399 x 48 x 192:
  // 109 us in pairs' tiles of 256 columns, 98 in tiles of 128), and a split sum
  // another pass.  The loader warps' blocks cost more than their products.
  struct Shape {
    int bn, block, epilogue;
    bool pair;
  };
  constexpr Shape kTmaShapes[] = {{256, 7, 66, true}, {256, 10, 70, false}, {128, 5, 28, false}, {64, 4, 16, false}};
  constexpr Shape kF32Shapes[] = {{128, 30, 35, false}, {64, 20, 20, false}};
  constexpr Shape kLoaderShapes[] = {{128, 40, 28, false}, {64, 26, 16, false}};
  const Shape* shapes = size == 4 ? kF32Shapes : tma ? kTmaShapes : kLoaderShapes;
  const int shape_count = size == 2 && tma ? 4 : 2;
  int64_t best = INT64_MAX;
  for (int i = 0; i < shape_count; ++i) {
    const Shape& shape = shapes[i];
    if (shape.bn > 64 && shape.bn / 2 >= n) continue;
    if (shape.pair && m <= linear_tc::kBM) continue;
    const int rows = shape.pair ? 2 * linear_tc::kBM : linear_tc::kBM;
    const int walkers = shape.pair ? kSms / 2 : kSms;
    const int64_t tiles = int64_t(ceil_div(m, rows)) * ceil_div(n, shape.bn);
    int splits = int(std::max<int64_t>(1, std::min<int64_t>(walkers / tiles, p.k_blocks / 4)));
    const int blocks = ceil_div(p.k_blocks, splits);
    splits = ceil_div(p.k_blocks, blocks);
    const int64_t cost =
        int64_t(ceil_div(tiles * splits, walkers)) * (std::max(blocks * shape.block, shape.epilogue) + 8) +
        (splits > 1 ? 40 : 0);
    if (cost < best) {
      best = cost;
      p.bn = shape.bn;
      p.pair = shape.pair;
      p.m_tiles = ceil_div(m, rows);
      p.n_tiles = ceil_div(n, shape.bn);
      p.splits = splits;
      p.split_blocks = blocks;
      p.layer_rows = int64_t(p.m_tiles) * rows;
    }
  }
  return p;
}
size_t product_workspace(size_t size, int64_t m, int64_t n, int64_t k) {
  return std::max(plan_product(size, true, m, n, k).partial_bytes(),
                  plan_product(size, false, m, n, k).partial_bytes());
}

template <class T>
int vector_width(const void* p, int64_t stride, int64_t rows) {
  int vec = 16 / int(sizeof(T));
  while (vec > 1 && (reinterpret_cast<uintptr_t>(p) % (vec * sizeof(T)) ||
                     (rows > 1 && stride % vec)))
    vec /= 2;
  return vec;
}

// Blocks of the pair kernel KERNEL that run at once on the current device; one
// answer per kernel and device is kept.
template <auto KERNEL>
npa_status pair_blocks(int threads, size_t smem, int sms, int* blocks) {
  static std::atomic<int> cached[64];
  int dev = 0;
  NPA_CUDA(cudaGetDevice(&dev), "cudaGetDevice");
  const int known = dev < 64 ? cached[dev].load() : 0;
  if (known) {
    *blocks = known;
    return NPA_OK;
  }
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(unsigned(sms / 2 * 2));
  config.blockDim = dim3(unsigned(threads));
  config.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  int clusters = 0;
  NPA_CUDA(cudaOccupancyMaxActiveClusters(&clusters, KERNEL, &config),
           "cudaOccupancyMaxActiveClusters");
  if (clusters < 1) return fail(NPA_ERR_UNSUPPORTED, "linear pair kernel cannot be resident");
  *blocks = 2 * clusters;
  if (dev < 64) cached[dev].store(*blocks);
  return NPA_OK;
}

template <class T, bool LOADER, int BN, bool PAIR, linear_tc::Form FORM>
npa_status launch_product_as(const CUtensorMap (&maps)[4], const Product& p, bool after,
                          cudaStream_t stream) {
  using C = linear_tc::Config<T, LOADER, BN, PAIR>;
  const auto kernel = linear_tc::product_kernel<T, LOADER, BN, PAIR, FORM>;
  int per_sm = 0, sms = 0;
  NPA_TRY(kernel_occupancy(reinterpret_cast<const void*>(kernel), C::kThreads, C::kSmemBytes,
                           &per_sm, &sms));
  if (per_sm < 1) return fail(NPA_ERR_UNSUPPORTED, "linear kernel cannot be resident");
  const int64_t tiles = int64_t(p.m_tiles) * p.n_tiles * p.splits;
  if constexpr (PAIR) {
    int blocks = 0;
    NPA_TRY((pair_blocks<linear_tc::product_kernel<T, LOADER, BN, PAIR, FORM>>(C::kThreads, C::kSmemBytes, sms,
                                                                             &blocks)));
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(unsigned(std::min<int64_t>(2 * tiles, blocks)));
    config.blockDim = dim3(C::kThreads);
    config.dynamicSmemBytes = C::kSmemBytes;
    config.stream = stream;
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attr;
    config.numAttrs = after ? 2 : 1;
    NPA_CUDA(cudaLaunchKernelEx(&config, kernel, maps[0], maps[1], maps[2], maps[3], p),
             "linear product_kernel");
  } else {
    NPA_CUDA(launch_kernel(after, kernel, dim3(unsigned(std::min<int64_t>(tiles, sms))), C::kThreads,
                           C::kSmemBytes, stream, maps[0], maps[1], maps[2], maps[3], p),
             "linear product_kernel");
  }
  return after_launch("linear product_kernel");
}

template <class T, bool LOADER, int BN, bool PAIR = false>
npa_status launch_product(const CUtensorMap (&maps)[4], const Product& p, bool after,
                          cudaStream_t stream) {
  using linear_tc::kLong, linear_tc::kRagged, linear_tc::kWhole;
  if constexpr (sizeof(T) == 2)
    if (p.long_k) return launch_product_as<T, LOADER, BN, PAIR, kLong>(maps, p, after, stream);
  const bool whole = p.partials || (p.y_tma && (!p.z || p.z_tma) &&
                                    (!p.residual || (p.residual_vec && p.n * sizeof(T) % 16 == 0)));
  return whole ? launch_product_as<T, LOADER, BN, PAIR, kWhole>(maps, p, after, stream)
               : launch_product_as<T, LOADER, BN, PAIR, kRagged>(maps, p, after, stream);
}

// Runs the product; p holds operands, sizes and the epilogue's buffers.  A bias
// gradient that waits is added behind it.
template <class T>
npa_status run_product(Product p, float* partials, bool after, BiasSums bias, cudaStream_t stream) {
  constexpr bool kSplitParts = sizeof(T) == 4;
  const int64_t a_rows = p.a.rows, b_rows = p.b.rows;
  const bool tma = !kSplitParts && tma_rows(p.a.p, p.a.ld, a_rows, sizeof(T)) &&
                   tma_rows(p.b.p, p.b.ld, b_rows, sizeof(T));
  const Plan plan = plan_product(sizeof(T), tma, p.m, p.n, p.k);
  if (int64_t(plan.m_tiles) * plan.n_tiles * plan.splits >= int64_t(1) << 31)
    return fail(NPA_ERR_UNSUPPORTED, "linear product of 2^31 tiles or more");
  p.m_tiles = plan.m_tiles;
  p.n_tiles = plan.n_tiles;
  p.k_blocks = plan.k_blocks;
  p.splits = plan.splits;
  p.split_blocks = plan.split_blocks;
  p.layer_rows = plan.layer_rows;
  p.partial_pitch = plan.partial_pitch;
  p.partials = plan.splits > 1 ? partials : nullptr;
  p.long_k = sizeof(T) == 2 && plan.split_blocks > linear_tc::kLongBlocks;
  p.idesc = tc::instruction_desc(!std::is_same<T, __half>::value, p.a.mn_major, p.b.mn_major,
                                 plan.pair ? 2 * linear_tc::kBM : linear_tc::kBM, plan.bn);
  p.a_vec = vector_width<T>(p.a.p, p.a.ld, a_rows);
  p.b_vec = vector_width<T>(p.b.p, p.b.ld, b_rows);
  constexpr int kWhole = 16 / int(sizeof(T));
  p.whole_chunks = p.a_vec == kWhole && p.b_vec == kWhole && p.a.width % kWhole == 0 &&
                   p.b.width % kWhole == 0;
  p.y_tma = tma_rows(p.y, p.y_stride, p.m, sizeof(T));
  p.z_tma = p.z && tma_rows(p.z, p.z_stride, p.m, sizeof(T));
  p.residual_vec = p.residual && tma_rows(p.residual, p.residual_stride, p.m, sizeof(T));
  CUtensorMap maps[4] = {};
  if (tma) {
    NPA_TRY(p.a.mn_major ? make_map<T>(&maps[0], p.a.p, p.m, p.k, p.a.ld, linear_tc::kBK)
                         : make_map<T>(&maps[0], p.a.p, p.k, p.m, p.a.ld, linear_tc::kBM));
    NPA_TRY(p.b.mn_major ? make_map<T>(&maps[1], p.b.p, p.n, p.k, p.b.ld, linear_tc::kBK)
                         : make_map<T>(&maps[1], p.b.p, p.k, p.n, p.b.ld,
                                       plan.pair ? plan.bn / 2 : plan.bn));
  }
  if (p.partials)
    NPA_TRY(make_map<float>(&maps[2], p.partials, p.n,
                            int64_t(p.splits) * p.layer_rows, p.partial_pitch, 32));
  else if (p.y_tma)
    NPA_TRY(make_map<T>(&maps[2], p.y, p.n, p.m, p.y_stride, 32));
  if (p.z_tma && !p.partials) NPA_TRY(make_map<T>(&maps[3], p.z, p.n, p.m, p.z_stride, 32));
  if constexpr (kSplitParts) {
    NPA_TRY(plan.bn == 128 ? (launch_product<T, true, 128>(maps, p, after, stream))
                           : (launch_product<T, true, 64>(maps, p, after, stream)));
  } else if (tma) {
    NPA_TRY(plan.pair        ? (launch_product<T, false, 256, true>(maps, p, after, stream))
            : plan.bn == 256 ? (launch_product<T, false, 256>(maps, p, after, stream))
            : plan.bn == 128 ? (launch_product<T, false, 128>(maps, p, after, stream))
                             : (launch_product<T, false, 64>(maps, p, after, stream)));
  } else {
    NPA_TRY(plan.bn == 128 ? (launch_product<T, true, 128>(maps, p, after, stream))
                           : (launch_product<T, true, 64>(maps, p, after, stream)));
  }
  if (p.partials) return launch_product_reduce<T>(p, bias, stream);
  return bias.partials ? launch_bias_reduce<T>(bias, stream) : NPA_OK;
}

// The one-walk backward pass's shape, or stage_bytes = 0 where it has none:
// 16-bit layers whose weights, two stages of rows and accumulators fit an SM.
constexpr int64_t kFusedRows = 2048;  // at least: fewer rows leave most SMs idle
FusedBackward plan_fused(size_t size, int activation, int64_t rows, int inputs, int outputs) {
  FusedBackward f{};
  if (size != 2 || rows < kFusedRows || inputs > 256 || outputs > 256) return f;
  f.rows = rows;
  f.inputs = inputs;
  f.outputs = outputs;
  f.out_blocks = ceil_div(outputs, 64);
  f.in_blocks = ceil_div(inputs, 64);
  f.k_pad = ceil_div(outputs, 16) * 16;
  f.n_pad = ceil_div(inputs, 16) * 16;
  f.m_blocks = ceil_div(outputs, 128);
  f.act = activation;
  f.has_z = activation != NPA_ACTIVATION_IDENTITY;
  f.stage_bytes = uint32_t(f.out_blocks * (f.has_z ? 2 : 1) + f.in_blocks) * linear_tc::kBM * 128;
  f.weight_bytes = uint32_t(f.in_blocks) * f.k_pad * 128;
  f.tmem_columns = 32;
  while (int(f.tmem_columns) < (f.m_blocks + 2) * f.n_pad) f.tmem_columns *= 2;
  f.pitch = (int64_t(inputs) + 3) / 4 * 4;
  for (f.stages = linear_tc::kFusedStages; f.stages >= 1; --f.stages)
    if (linear_tc::fused_fits(f)) return f;
  return FusedBackward{};
}
// A block for each SM, or several one after another where a block would walk more
// than kFusedTiles tiles: dW's accumulator takes a step for every 16 rows (each
// start costs about 7 us: 1300000 x 64 x 128 186 us, 174 in one walk whose sums
// would lose up to 6e-5 of them).
int fused_blocks(const FusedBackward& f) {
  const int64_t tiles = (f.rows + linear_tc::kBM - 1) / linear_tc::kBM, a_wave = kSms * linear_tc::kFusedTiles;
  return int(std::min<int64_t>(tiles, kSms * ((tiles + a_wave - 1) / a_wave)));
}
size_t fused_partial_bytes(const FusedBackward& f) {
  return f.stage_bytes ? size_t(fused_blocks(f)) * f.m_blocks * linear_tc::kBM * f.pitch * 4 : 0;
}

struct BackwardCarve {
  void* dz;  // where dz is not dy as it lies
  int64_t dz_stride;
  void *x, *weight;  // packed, where they are
  float* bias_partials;
  float* product_partials;
  size_t bytes;
};
BackwardCarve carve_backward(void* ws, int dtype, int activation, int64_t rows, int inputs,
                             int outputs) {
  const size_t size = dtype_bytes(dtype);
  Carve c(ws, 0);
  BackwardCarve b{};
  b.dz_stride = (int64_t(outputs) + 7) / 8 * 8;  // rows of 16-byte multiples
  b.dz = activation != NPA_ACTIVATION_IDENTITY || outputs * size % 16 != 0
             ? static_cast<void*>(c.take<char>(size_t(rows) * b.dz_stride * size))
             : nullptr;
  if (packs(size, inputs, rows, inputs, outputs)) {
    const size_t pitch = size_t(packed_pitch(inputs));
    b.x = c.take<char>(size_t(rows) * pitch * size);
    b.weight = c.take<char>(size_t(outputs) * pitch * size);
  }
  const FusedBackward fused = plan_fused(size, activation, rows, inputs, outputs);
  b.bias_partials = c.take<float>(size_t(std::max(kBiasBlocks, fused.stage_bytes ? fused_blocks(fused) : 0)) * outputs);
  size_t partial = std::max(product_workspace(size, rows, inputs, outputs),
                                  product_workspace(size, outputs, inputs, rows));
  partial = std::max(partial, fused_partial_bytes(fused));
  b.product_partials = c.take<float>(partial / 4);
  b.bytes = c.used;
  return b;
}

struct ForwardCarve {
  void *x, *weight;  // packed, where they are
  float* product_partials;
  size_t bytes;
};
ForwardCarve carve_forward(void* ws, size_t size, int64_t rows, int inputs, int outputs) {
  Carve c(ws, 0);
  ForwardCarve f{};
  f.product_partials = c.take<float>(product_workspace(size, rows, outputs, inputs) / 4);
  if (packs(size, inputs, rows, inputs, outputs)) {
    const size_t pitch = size_t(packed_pitch(inputs));
    f.x = c.take<char>(size_t(rows) * pitch * size);
    f.weight = c.take<char>(size_t(outputs) * pitch * size);
  }
  f.bytes = c.used;
  return f;
}

template <class T>
npa_status forward_typed(const LinearArgs& a, void* workspace, cudaStream_t s) {
  if (a.rows <= kFewRows) {
    constexpr int kVec = 16 / int(sizeof(T));
    const bool vec = a.inputs % kVec == 0 && vector_width<T>(a.x, a.x_stride, a.rows) == kVec &&
                     vector_width<T>(a.weight, a.weight_stride, a.outputs) == kVec;
    if (a.rows == 1) return launch_few_rows<T, 1>(a, vec, s);
    if (a.rows == 2) return launch_few_rows<T, 2>(a, vec, s);
    return a.rows <= 4 ? launch_few_rows<T, 4>(a, vec, s) : launch_few_rows<T, 8>(a, vec, s);
  }
  Product p{};
  p.a = {a.x, a.x_stride, 0, int(a.rows), a.inputs};
  p.b = {a.weight, a.weight_stride, 0, a.outputs, a.inputs};
  p.m = int(a.rows);
  p.n = a.outputs;
  p.k = a.inputs;
  p.bias = a.bias;
  p.residual = a.residual;
  p.residual_stride = a.residual_stride;
  p.y = a.y;
  p.y_stride = a.y_stride;
  p.z = a.z;
  p.z_stride = a.z_stride;
  p.act = a.activation;
  const ForwardCarve ws = carve_forward(workspace, sizeof(T), a.rows, a.inputs, a.outputs);
  if (ws.x) {
    NPA_TRY(pack_rows<T>(p.a, ws.x, false, s));
    NPA_TRY(pack_rows<T>(p.b, ws.weight, true, s));
  }
  return run_product<T>(p, ws.product_partials, ws.x != nullptr, {}, s);
}

template <class T, bool RAGGED>
npa_status launch_slope(SlopeArgs s, int* parts, cudaStream_t stream) {
  const int groups = ceil_div(s.outputs, 16 / int(sizeof(T)));
  s.tx = 1;
  while (s.tx < 32 && s.tx < groups) s.tx *= 2;
  const int grid_x = ceil_div(groups, s.tx);
  const int64_t at_once = 256 / s.tx;
  const int64_t most = std::max(1, kSlopeBlocks<T, RAGGED> * kSms / grid_x);
  *parts = int(std::max<int64_t>(1, std::min<int64_t>(most, (s.rows + at_once * 4 - 1) / (at_once * 4))));
  s.rows_per_block = (s.rows + *parts - 1) / *parts;
  *parts = int((s.rows + s.rows_per_block - 1) / s.rows_per_block);
  slope_kernel<T, RAGGED><<<dim3(unsigned(grid_x), unsigned(*parts)), 256, 0, stream>>>(s);
  return after_launch("slope_kernel");
}

template <class T>
npa_status launch_fused(const LinearBackwardArgs& a, FusedBackward f, const BackwardCarve& ws,
                        cudaStream_t s) {
  f.want_dx = a.dx != nullptr;
  f.want_dw = a.dweight != nullptr;
  f.want_db = a.dbias != nullptr;
  f.dw_partials = ws.product_partials;
  f.db_partials = ws.bias_partials;
  constexpr bool kBf16 = !std::is_same<T, __half>::value;
  f.dx_idesc = tc::instruction_desc(kBf16, false, true, linear_tc::kBM, f.n_pad);
  f.dw_idesc = tc::instruction_desc(kBf16, true, true, linear_tc::kBM, f.n_pad);
  CUtensorMap maps[5] = {};
  NPA_TRY(make_map<T>(&maps[0], a.dy, a.outputs, a.rows, a.dy_stride, linear_tc::kBM));
  if (a.z) NPA_TRY(make_map<T>(&maps[1], a.z, a.outputs, a.rows, a.z_stride, linear_tc::kBM));
  NPA_TRY(make_map<T>(&maps[2], a.x, a.inputs, a.rows, a.x_stride, linear_tc::kBM));
  NPA_TRY(make_map<T>(&maps[3], a.weight, a.inputs, a.outputs, a.weight_stride, f.k_pad));
  if (a.dx) NPA_TRY(make_map<T>(&maps[4], a.dx, a.inputs, a.rows, a.dx_stride, 32));
  const auto kernel = linear_tc::fused_backward_kernel<T>;
  // the whole of an SM's memory whatever the shape: one launch shape, one block
  const size_t smem = linear_tc::kSmemLimit - linear_tc::kFusedStaticSmem - 1024;
  int per_sm = 0, sms = 0;
  NPA_TRY(kernel_occupancy(reinterpret_cast<const void*>(kernel), linear_tc::kFusedThreads, smem,
                           &per_sm, &sms));
  if (per_sm < 1) return fail(NPA_ERR_UNSUPPORTED, "linear backward kernel cannot be resident");
  const int blocks = fused_blocks(f);
  kernel<<<unsigned(blocks), linear_tc::kFusedThreads, smem, s>>>(maps[0], maps[1], maps[2], maps[3],
                                                                  maps[4], f);
  NPA_TRY(after_launch("linear fused_backward_kernel"));
  BiasSums bias{};
  if (a.dbias) bias = {ws.bias_partials, blocks, a.outputs, a.dbias};
  if (a.dweight) {
    Product p{};
    p.m = a.outputs;
    p.n = a.inputs;
    p.splits = blocks;
    p.layer_rows = int64_t(f.m_blocks) * linear_tc::kBM;
    p.partial_pitch = f.pitch;
    p.partials = f.dw_partials;
    p.y = a.dweight;
    p.y_stride = a.inputs;
    return launch_product_reduce<T>(p, bias, s);
  }
  if (a.dbias) return launch_bias_reduce<T>(bias, s);
  return NPA_OK;
}

template <class T>
npa_status backward_typed(const LinearBackwardArgs& a, const BackwardCarve& ws, cudaStream_t s) {
  if (a.rows == 0) {
    if (a.dweight)
      NPA_CUDA(cudaMemsetAsync(a.dweight, 0, size_t(a.inputs) * a.outputs * sizeof(T), s),
               "cudaMemsetAsync");
    if (a.dbias)
      NPA_CUDA(cudaMemsetAsync(a.dbias, 0, size_t(a.outputs) * sizeof(T), s), "cudaMemsetAsync");
    return NPA_OK;
  }
  if (few_rows_backward(a.rows, a.outputs)) {
    if (!a.dx && !a.dweight && !a.dbias) return NPA_OK;
    constexpr int kVec = 16 / int(sizeof(T));
    const bool vec = a.inputs % kVec == 0 &&
                     (!a.dx || (vector_width<T>(a.weight, a.weight_stride, a.outputs) == kVec &&
                                vector_width<T>(a.dx, a.dx_stride, a.rows) == kVec)) &&
                     (!a.dweight || (vector_width<T>(a.x, a.x_stride, a.rows) == kVec &&
                                     vector_width<T>(a.dweight, a.inputs, a.outputs) == kVec));
    if (a.rows == 1) return launch_few_rows_backward<T, 1>(a, vec, s);
    if (a.rows == 2) return launch_few_rows_backward<T, 2>(a, vec, s);
    return a.rows <= 4 ? launch_few_rows_backward<T, 4>(a, vec, s)
                       : launch_few_rows_backward<T, 8>(a, vec, s);
  }
  if constexpr (sizeof(T) == 2) {
    const FusedBackward f = plan_fused(sizeof(T), a.activation, a.rows, a.inputs, a.outputs);
    if (f.stage_bytes && (a.dx || a.dweight) && tma_rows(a.dy, a.dy_stride, a.rows, 2) &&
        (!a.z || tma_rows(a.z, a.z_stride, a.rows, 2)) && a.x &&
        tma_rows(a.x, a.x_stride, a.rows, 2) && a.weight &&
        tma_rows(a.weight, a.weight_stride, a.outputs, 2) &&
        (!a.dx || tma_rows(a.dx, a.dx_stride, a.rows, 2)))
      return launch_fused<T>(a, f, ws, s);
  }
  const T* dz = static_cast<const T*>(a.dy);
  int64_t dz_stride = a.dy_stride;
  int dz_width = a.outputs;
  bool after = false;  // a kernel of this call precedes
  BiasSums bias{};     // waits for the last product
  // dz is written where it is not dy, and where dy's odd rows are worth copying:
  // by the pass that sums them for dbias, or for much work
  const bool write_dz =
      ws.dz && (a.dx || a.dweight) &&
      (a.z || a.dbias || packs(sizeof(T), a.outputs, a.rows, a.inputs, a.outputs));
  if (a.dbias || write_dz) {
    SlopeArgs g{};
    g.dy = a.dy;
    g.dy_stride = a.dy_stride;
    g.z = a.z;
    g.z_stride = a.z_stride;
    g.rows = a.rows;
    g.outputs = a.outputs;
    g.act = a.activation;
    g.dz = write_dz ? ws.dz : nullptr;
    g.dz_stride = ws.dz_stride;
    g.partials = ws.bias_partials;
    int parts = 0;
    constexpr int kVec = 16 / int(sizeof(T));
    if (a.outputs % kVec == 0 && vector_width<T>(a.dy, a.dy_stride, a.rows) == kVec &&
        (!a.z || vector_width<T>(a.z, a.z_stride, a.rows) == kVec))
      NPA_TRY((launch_slope<T, false>(g, &parts, s)));
    else
      NPA_TRY((launch_slope<T, true>(g, &parts, s)));
    after = true;
    if (a.dbias) bias = {ws.bias_partials, parts, a.outputs, a.dbias};
    if (g.dz) {
      dz = static_cast<const T*>(ws.dz);
      dz_stride = ws.dz_stride;
      dz_width = int((a.outputs + kVec - 1) / kVec * kVec);  // zeros past outputs
    }
  }
  Operand weight{a.weight, a.weight_stride, 1, a.outputs, a.inputs};
  Operand x{a.x, a.x_stride, 1, int(a.rows), a.inputs};
  if (ws.x) {
    if (a.dweight) {
      NPA_TRY(pack_rows<T>(x, ws.x, after, s));
      after = true;
    }
    if (a.dx) {
      NPA_TRY(pack_rows<T>(weight, ws.weight, after, s));
      after = true;
    }
  }
  if (a.dx) {
    Product p{};
    p.a = {dz, dz_stride, 0, int(a.rows), dz_width};
    p.b = weight;
    p.m = int(a.rows);
    p.n = a.inputs;
    p.k = a.outputs;
    p.y = a.dx;
    p.y_stride = a.dx_stride;
    NPA_TRY(run_product<T>(p, ws.product_partials, after, a.dweight ? BiasSums{} : bias, s));
    after = true;
  }
  if (a.dweight) {
    Product p{};
    p.a = {dz, dz_stride, 1, int(a.rows), dz_width};
    p.b = x;
    p.m = a.outputs;
    p.n = a.inputs;
    p.k = int(a.rows);
    p.y = a.dweight;
    p.y_stride = a.inputs;
    return run_product<T>(p, ws.product_partials, after, bias, s);
  }
  return !a.dx && bias.partials ? launch_bias_reduce<T>(bias, s) : NPA_OK;
}

}  // namespace

size_t linear_workspace(int dtype, int64_t rows, int inputs, int outputs) {
  return rows <= kFewRows
             ? 0
             : carve_forward(nullptr, dtype_bytes(dtype), rows, inputs, outputs).bytes;
}

npa_status launch_linear(int dtype, const LinearArgs& a, void* workspace, cudaStream_t stream) {
  switch (dtype) {
    case NPA_DTYPE_F32: return forward_typed<float>(a, workspace, stream);
    case NPA_DTYPE_F16: return forward_typed<__half>(a, workspace, stream);
    default: return forward_typed<__nv_bfloat16>(a, workspace, stream);
  }
}

size_t linear_backward_workspace(int dtype, int activation, int64_t rows, int inputs, int outputs) {
  if (rows == 0) return 0;
  // A few rows' kernel uses none, but every call with rows takes a workspace: what
  // a caller has to pass does not hang on which kernels a row count gets.
  if (few_rows_backward(rows, outputs)) return 256;
  return carve_backward(nullptr, dtype, activation, rows, inputs, outputs).bytes;
}

npa_status launch_linear_backward(int dtype, const LinearBackwardArgs& a, void* workspace,
                                  cudaStream_t stream) {
  const BackwardCarve ws =
      a.rows == 0 || few_rows_backward(a.rows, a.outputs)
          ? BackwardCarve{}
                  : carve_backward(workspace, dtype, a.activation, a.rows, a.inputs, a.outputs);
  switch (dtype) {
    case NPA_DTYPE_F32: return backward_typed<float>(a, ws, stream);
    case NPA_DTYPE_F16: return backward_typed<__half>(a, ws, stream);
    default: return backward_typed<__nv_bfloat16>(a, ws, stream);
  }
}

uint64_t linear_timeouts() {
  unsigned long long v = 0;
  if (cudaMemcpyFromSymbol(&v, linear_tc::g_timeouts, sizeof(v)) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return v;
}

}  // namespace npa
