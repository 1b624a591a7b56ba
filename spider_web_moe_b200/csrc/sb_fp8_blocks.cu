// Quantisation to e4m3 with one fp32 scale per block of 128 columns and 1 or
// 128 rows.
//
//   a = max(amax |x|, 2^-100), scale = a / 448, q = e4m3(x * (448 / a))
//
// The floor keeps 448 / a finite and makes a block of zeros quantise to zeros.
// amax is taken over the bit patterns of |x|, so that an inf or NaN reaches the
// scale and the block dequantises to NaN instead of to plausible numbers.
//
// Both kernels are bound by memory: cols * (2 or 4) bytes read and cols bytes
// written per row.
#include "sb_common.cuh"
#include "sb_fp8.cuh"
#include "sb_internal.h"

namespace sb {

// ---------------------------------------------------------------- rows
// block_rows 1, unit column stride: 16 lanes hold one block, 8 elements each
// (16-byte loads of bf16), and walk kRowsBlocks consecutive blocks of their row,
// whose loads are all in flight together.  A CTA covers 16 rows, so the scales
// of one column of blocks, which are row-contiguous, leave 64 bytes at a time.
constexpr int kRowsBlocks = 4;
constexpr int kRowsPerCta = 16;
constexpr int kMaxCols = 1 << 24;  // the column blocks are a grid's y extent

template <typename T, bool kVec>
SB_DEVINL void load8(const T* __restrict__ p, int64_t col_stride, int valid, float (&v)[8]) {
  if (kVec && valid >= 8) {
    if constexpr (sizeof(T) == 2) {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    } else {
      const float4 a = *reinterpret_cast<const float4*>(p);
      const float4 b = *reinterpret_cast<const float4*>(p + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < valid ? to_f32<T>(p[i * col_stride]) : 0.f;
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(256) fp8_quantize_rows_kernel(const sb_fp8_quantize_args p) {
  pdl_wait();
  pdl_trigger();
  const int lane16 = threadIdx.x & 15;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * kRowsPerCta + (threadIdx.x >> 4);
  const int cb0 = blockIdx.y * kRowsBlocks;
  int64_t rows = p.rows;
  if (p.row_count) rows = min(rows, static_cast<int64_t>(*p.row_count));
  const bool live = r < rows;  // uniform over the 16 lanes; the shuffles below need the whole warp
  const int64_t src = live ? (p.row_index ? p.row_index[r] : r) : 0;
  const T* x = static_cast<const T*>(p.x) + blockIdx.z * p.x_batch + src * p.x_row;
  uint8_t* q = static_cast<uint8_t*>(p.q) + blockIdx.z * p.q_batch + r * p.ldq;
  float* scale = p.scale + blockIdx.z * p.scale_batch + r * p.scale_row;
  float v[kRowsBlocks][8];
#pragma unroll
  for (int i = 0; i < kRowsBlocks; ++i) {
    const int c = (cb0 + i) * 128 + lane16 * 8;
    load8<T, kVec>(x + c * p.x_col, p.x_col, live ? p.cols - c : 0, v[i]);
  }
#pragma unroll
  for (int i = 0; i < kRowsBlocks; ++i) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, abs_bits(v[i][j]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const int c = (cb0 + i) * 128 + lane16 * 8;
    if (!live || c >= p.cols) continue;
    const Fp8Scale s = fp8_scale(m);
    if (lane16 == 0) scale[static_cast<int64_t>(cb0 + i) * p.scale_col] = s.scale;
    uint2 o8;
    o8.x = fp8_pack4(v[i][0] * s.inv, v[i][1] * s.inv, v[i][2] * s.inv, v[i][3] * s.inv);
    o8.y = fp8_pack4(v[i][4] * s.inv, v[i][5] * s.inv, v[i][6] * s.inv, v[i][7] * s.inv);
    if (c + 8 <= p.cols) {
      *reinterpret_cast<uint2*>(q + c) = o8;
    } else {
      for (int j = 0; c + j < p.cols; ++j) q[c + j] = static_cast<uint8_t>((j < 4 ? o8.x >> (8 * j) : o8.y >> (8 * (j - 4))));
    }
  }
}

// The same for bf16 rows on 16-byte boundaries with whole 8-column chunks: 8 lanes
// hold a block, 16 elements each, as loaded (two elements per register): the
// maximum of two is one 16-bit-pair instruction, two blocks share a register in
// the shuffles, and the few registers leave room for more loads in flight.
constexpr int kBf16Blocks = 4;

__global__ void __launch_bounds__(256, 4) fp8_quantize_rows_bf16_kernel(const sb_fp8_quantize_args p) {
  pdl_wait();
  pdl_trigger();
  const int lane8 = threadIdx.x & 7;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x >> 3);
  const int cb0 = blockIdx.y * kBf16Blocks;
  int64_t rows = p.rows;
  if (p.row_count) rows = min(rows, static_cast<int64_t>(*p.row_count));
  const bool live = r < rows;
  const int64_t src = live ? (p.row_index ? p.row_index[r] : r) : 0;
  const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(p.x) + blockIdx.z * p.x_batch + src * p.x_row;
  uint8_t* q = static_cast<uint8_t*>(p.q) + blockIdx.z * p.q_batch + r * p.ldq;
  float* scale = p.scale + blockIdx.z * p.scale_batch + r * p.scale_row;
  // a lane's 16 elements are 8 at lane8 * 8 and 8 at 64 + lane8 * 8: each load of
  // the 8 lanes is 128 consecutive bytes
  uint4 v[kBf16Blocks][2];
#pragma unroll
  for (int i = 0; i < kBf16Blocks; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = (cb0 + i) * 128 + h * 64 + lane8 * 8;
      v[i][h] = live && c < p.cols ? *reinterpret_cast<const uint4*>(x + c) : make_uint4(0, 0, 0, 0);
    }
  uint32_t amax[kBf16Blocks];
#pragma unroll
  for (int i = 0; i < kBf16Blocks; i += 2) {
    uint32_t m[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint4 a = v[i + k][0], b = v[i + k][1];
      constexpr uint32_t kAbs = 0x7fff7fffu;
      m[k] = __vmaxu2(__vmaxu2(__vmaxu2(a.x & kAbs, a.y & kAbs), __vmaxu2(a.z & kAbs, a.w & kAbs)),
                      __vmaxu2(__vmaxu2(b.x & kAbs, b.y & kAbs), __vmaxu2(b.z & kAbs, b.w & kAbs)));
    }
    // low halves: block i, high halves: block i + 1
    uint32_t w = __vmaxu2(__byte_perm(m[0], m[1], 0x5410), __byte_perm(m[0], m[1], 0x7632));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) w = __vmaxu2(w, __shfl_xor_sync(0xffffffffu, w, o));
    amax[i] = w << 16;
    amax[i + 1] = w & 0xffff0000u;
  }
  if (!live) return;
#pragma unroll
  for (int i = 0; i < kBf16Blocks; ++i) {
    const int cb = cb0 + i;
    if (cb * 128 >= p.cols) break;
    const Fp8Scale s = fp8_scale(amax[i]);
    if (lane8 == 0) scale[static_cast<int64_t>(cb) * p.scale_col] = s.scale;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = cb * 128 + h * 64 + lane8 * 8;
      if (c >= p.cols) continue;
      *reinterpret_cast<uint2*>(q + c) =
          make_uint2(fp8_pack4_bf16(v[i][h].x, v[i][h].y, s.inv), fp8_pack4_bf16(v[i][h].z, v[i][h].w, s.inv));
    }
  }
}

// ---------------------------------------------------------------- tiles
// 128 x 128 tile per CTA through shared memory: block_rows 128 (one scale per
// tile), and block_rows 1 of a matrix whose rows, not columns, are contiguous
// (a transposed view).  Shared memory keeps the order of the contiguous
// direction: [row][col] or, for kColMajor, [col][row]; the loads are coalesced
// and the reads below (32 consecutive rows per warp) meet no bank conflict.
template <typename T, bool kColMajor, bool kVec>
__global__ void __launch_bounds__(256) fp8_quantize_tile_kernel(const sb_fp8_quantize_args p) {
  constexpr int kPitch = kColMajor ? 128 + 16 / sizeof(T) : 128 + 4 / sizeof(T);
  extern __shared__ __align__(16) uint8_t tile_raw[];
  T* tile = reinterpret_cast<T*>(tile_raw);
  __shared__ uint32_t s_max[256];
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x;
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * 128;
  const int64_t c0 = static_cast<int64_t>(blockIdx.x) * 128;
  const int nr = static_cast<int>(min(static_cast<int64_t>(128), p.rows - r0));
  const int nc = static_cast<int>(min(static_cast<int64_t>(128), p.cols - c0));
  const T* x = static_cast<const T*>(p.x) + blockIdx.z * p.x_batch + r0 * p.x_row + c0 * p.x_col;
  // i: the contiguous direction (8 elements per thread), o: the other one
  const int ni = kColMajor ? nr : nc, no = kColMajor ? nc : nr;
  const int64_t si = kColMajor ? p.x_row : p.x_col, so = kColMajor ? p.x_col : p.x_row;
#pragma unroll
  for (int it = 0; it < 8; ++it) {
    const int o = it * 16 + (tid >> 4), i = (tid & 15) * 8;
    float v[8];
    load8<T, kVec>(x + o * so + i * si, si, o < no ? ni - i : 0, v);
    T* dst = tile + o * kPitch + i;
#pragma unroll
    for (int j = 0; j < 8; ++j) dst[j] = from_f32<T>(v[j]);  // exact: v holds values of T
  }
  __syncthreads();
  // one row and half of its columns per thread: a warp's lanes sit in 32
  // consecutive rows
  const int r = tid & 127, half = tid >> 7, h = half * 64;
  float v[64];
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 64; ++j) {
    v[j] = to_f32<T>(kColMajor ? tile[(h + j) * kPitch + r] : tile[r * kPitch + h + j]);
    m = max(m, abs_bits(v[j]));
  }
  if (p.block_rows == 1) {
    s_max[tid] = m;
    __syncthreads();
    m = max(m, s_max[tid ^ 128]);
  } else {
    m = __reduce_max_sync(0xffffffffu, m);
    if ((tid & 31) == 0) s_max[tid >> 5] = m;
    __syncthreads();
    m = s_max[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) m = max(m, s_max[w]);
  }
  const Fp8Scale s = fp8_scale(m);
  float* scale = p.scale + blockIdx.z * p.scale_batch + blockIdx.x * p.scale_col;
  if (p.block_rows == 1) {
    if (half == 0 && r < nr) scale[(r0 + r) * p.scale_row] = s.scale;
  } else if (tid == 0) {
    scale[blockIdx.y * p.scale_row] = s.scale;
  }
  if (r >= nr) return;
  uint8_t* q = static_cast<uint8_t*>(p.q) + blockIdx.z * p.q_batch + (r0 + r) * p.ldq + c0 + h;
#pragma unroll
  for (int j = 0; j < 64; j += 16) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      w[k] = fp8_pack4(v[j + 4 * k] * s.inv, v[j + 4 * k + 1] * s.inv, v[j + 4 * k + 2] * s.inv,
                       v[j + 4 * k + 3] * s.inv);
    if (h + j + 16 <= nc) {
      *reinterpret_cast<uint4*>(q + j) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (h + j + i < nc) q[j + i] = static_cast<uint8_t>(w[i >> 2] >> (8 * (i & 3)));
    }
  }
}

// 128 x 128 blocks of bf16 rows on 16-byte boundaries (whole 8-column chunks): the
// CTA's 8 x 16 bytes per thread stay in registers between the maximum and the
// rounding; no tile in shared memory.
__global__ void __launch_bounds__(256, 4) fp8_quantize_block_bf16_kernel(const sb_fp8_quantize_args p) {
  __shared__ uint32_t s_max[8];
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane16 = tid & 15;
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * 128 + (tid >> 4);
  const int c = blockIdx.x * 128 + lane16 * 8;
  const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(p.x) + blockIdx.z * p.x_batch + c;
  uint4 v[8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = r0 + 16 * i;
    v[i] = r < p.rows && c < p.cols ? *reinterpret_cast<const uint4*>(x + r * p.x_row) : make_uint4(0, 0, 0, 0);
  }
  constexpr uint32_t kAbs = 0x7fff7fffu;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    m = __vmaxu2(m, __vmaxu2(__vmaxu2(v[i].x & kAbs, v[i].y & kAbs), __vmaxu2(v[i].z & kAbs, v[i].w & kAbs)));
  m = __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16));
  if ((tid & 31) == 0) s_max[tid >> 5] = m;
  __syncthreads();
  m = s_max[0];
#pragma unroll
  for (int w = 1; w < 8; ++w) m = max(m, s_max[w]);
  const Fp8Scale s = fp8_scale(m << 16);
  if (tid == 0)
    p.scale[blockIdx.z * p.scale_batch + blockIdx.y * p.scale_row + blockIdx.x * p.scale_col] = s.scale;
  if (c >= p.cols) return;
  uint8_t* q = static_cast<uint8_t*>(p.q) + blockIdx.z * p.q_batch + c;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = r0 + 16 * i;
    if (r < p.rows) *reinterpret_cast<uint2*>(q + r * p.ldq) = make_uint2(fp8_pack4_bf16(v[i].x, v[i].y, s.inv), fp8_pack4_bf16(v[i].z, v[i].w, s.inv));
  }
}

// bf16 matrices whose rows are contiguous (transposed views), rows a multiple of 8
// and columns on 16-byte boundaries: the tile lies in shared memory as [col][row]
// and a thread takes two neighbouring rows, one 32-bit word per column, and a
// quarter of the columns.  kBoth: the matrix itself (d: 1 x 128 blocks of p's
// transpose) is quantised from the same loads, before they go to shared memory.
template <bool kBoth>
__global__ void __launch_bounds__(256, 4)
fp8_quantize_transposed_bf16_kernel(const sb_fp8_quantize_args p, const sb_fp8_quantize_args d) {
  constexpr int kPitch = 136;  // elements; 68 words, so a warp's 32 row pairs meet no bank conflict
  __shared__ __align__(16) __nv_bfloat16 tile[128 * kPitch];
  __shared__ uint32_t s_max[256];
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x;
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * 128;
  const int64_t c0 = static_cast<int64_t>(blockIdx.x) * 128;
  const int nr = static_cast<int>(min(static_cast<int64_t>(128), p.rows - r0));
  const int nc = static_cast<int>(min(static_cast<int64_t>(128), p.cols - c0));
  const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(p.x) + blockIdx.z * p.x_batch + r0 + c0 * p.x_col;
  {
    const int r = (tid & 15) * 8;
    uint4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = i * 16 + (tid >> 4);
      v[i] = r < nr && c < nc ? *reinterpret_cast<const uint4*>(x + c * p.x_col + r) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(tile + (i * 16 + (tid >> 4)) * kPitch + r) = v[i];
    if constexpr (kBoth) {
      // 16 lanes hold a block of the untransposed matrix; two of them share a
      // register in the shuffles
      constexpr uint32_t kAbs = 0x7fff7fffu;
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        uint32_t m[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint4 u = v[i + k];
          m[k] = __vmaxu2(__vmaxu2(u.x & kAbs, u.y & kAbs), __vmaxu2(u.z & kAbs, u.w & kAbs));
        }
        uint32_t w = __vmaxu2(__byte_perm(m[0], m[1], 0x5410), __byte_perm(m[0], m[1], 0x7632));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) w = __vmaxu2(w, __shfl_xor_sync(0xffffffffu, w, o));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int c = (i + k) * 16 + (tid >> 4);
          if (c >= nc || r >= nr) continue;
          const Fp8Scale s = fp8_scale(k ? w & 0xffff0000u : w << 16);
          if ((tid & 15) == 0) d.scale[(c0 + c) * d.scale_row + blockIdx.y * d.scale_col] = s.scale;
          *reinterpret_cast<uint2*>(static_cast<uint8_t*>(d.q) + (c0 + c) * d.ldq + r0 + r) =
              make_uint2(fp8_pack4_bf16(v[i + k].x, v[i + k].y, s.inv), fp8_pack4_bf16(v[i + k].z, v[i + k].w, s.inv));
        }
      }
    }
  }
  __syncthreads();
  const int pair = tid & 63, quarter = tid >> 6;
  uint32_t v[32];
  uint32_t m = 0;
  constexpr uint32_t kAbs = 0x7fff7fffu;
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    v[j] = *reinterpret_cast<const uint32_t*>(tile + (quarter * 32 + j) * kPitch + pair * 2);
    m = __vmaxu2(m, v[j] & kAbs);
  }
  s_max[tid] = m;
  __syncthreads();
  float* scale = p.scale + blockIdx.z * p.scale_batch + blockIdx.x * p.scale_col;
  float inv[2];
  if (p.block_rows == 1) {
    m = __vmaxu2(__vmaxu2(s_max[pair], s_max[pair + 64]), __vmaxu2(s_max[pair + 128], s_max[pair + 192]));
    const Fp8Scale lo = fp8_scale(m << 16), hi = fp8_scale(m & 0xffff0000u);
    inv[0] = lo.inv;
    inv[1] = hi.inv;
    if (quarter == 0 && pair * 2 < nr) {  // nr is even
      scale[(r0 + pair * 2) * p.scale_row] = lo.scale;
      scale[(r0 + pair * 2 + 1) * p.scale_row] = hi.scale;
    }
  } else {
    m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = __vmaxu2(m, s_max[(tid & 31) + 32 * i]);
    m = __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16));
    const Fp8Scale s = fp8_scale(m << 16);
    inv[0] = inv[1] = s.inv;
    if (tid == 0) scale[blockIdx.y * p.scale_row] = s.scale;
  }
  if (pair * 2 >= nr) return;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint8_t* q = static_cast<uint8_t*>(p.q) + blockIdx.z * p.q_batch + (r0 + pair * 2 + h) * p.ldq + c0 + quarter * 32;
#pragma unroll
    for (int j = 0; j < 32; j += 16) {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t* u = v + j + 4 * k;
        const uint32_t sel = h ? 0x7632 : 0x5410;
        w[k] = fp8_pack4_bf16(__byte_perm(u[0], u[1], sel), __byte_perm(u[2], u[3], sel), inv[h]);
      }
      const int left = nc - quarter * 32 - j;
      if (left >= 16) {
        *reinterpret_cast<uint4*>(q + j) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (i < left) q[j + i] = static_cast<uint8_t>(w[i >> 2] >> (8 * (i & 3)));
      }
    }
  }
}

template <typename T, bool kColMajor, bool kVec>
static int launch_tile(const sb_fp8_quantize_args& p, cudaStream_t st) {
  constexpr int kPitch = kColMajor ? 128 + 16 / sizeof(T) : 128 + 4 / sizeof(T);
  constexpr int kSmem = 128 * kPitch * sizeof(T);
  auto kern = fp8_quantize_tile_kernel<T, kColMajor, kVec>;
  static int configured_device = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (configured_device != dev) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return cuda_status(e);
    configured_device = dev;
  }
  return launch(kern, dim3((p.cols + 127) / 128, (p.rows + 127) / 128, p.batch), dim3(256), kSmem, st, p);
}

template <typename T>
static int quantize_typed(const sb_fp8_quantize_args& p, cudaStream_t st) {
  constexpr int64_t kAlign = 16 / sizeof(T);  // elements of a 16-byte load
  const bool base = reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && p.x_batch % kAlign == 0;
  if (p.block_rows == 1 && (p.x_row != 1 || p.x_col == 1 || p.row_index || p.row_count)) {
    const dim3 grid((p.rows + kRowsPerCta - 1) / kRowsPerCta, (p.cols + 128 * kRowsBlocks - 1) / (128 * kRowsBlocks),
                    p.batch);
    if (sizeof(T) == 2 && p.x_col == 1 && base && p.x_row % 8 == 0 && p.cols % 8 == 0)
      return launch(fp8_quantize_rows_bf16_kernel,
                    dim3((p.rows + 31) / 32, (p.cols + 128 * kBf16Blocks - 1) / (128 * kBf16Blocks), p.batch), dim3(256), 0,
                    st, p);
    if (p.x_col == 1 && base && p.x_row % kAlign == 0)
      return launch(fp8_quantize_rows_kernel<T, true>, grid, dim3(256), 0, st, p);
    return launch(fp8_quantize_rows_kernel<T, false>, grid, dim3(256), 0, st, p);
  }
  if (p.rows > 65535 * 128) return SB_ERR_UNSUPPORTED;  // a grid's y extent
  const dim3 tiles((p.cols + 127) / 128, (p.rows + 127) / 128, p.batch);
  if (sizeof(T) == 2 && p.x_row == 1 && p.x_col != 1 && base && p.x_col % 8 == 0 && p.rows % 8 == 0)
    return launch(fp8_quantize_transposed_bf16_kernel<false>, tiles, dim3(256), 0, st, p, p);
  if (sizeof(T) == 2 && p.x_col == 1 && base && p.x_row % 8 == 0 && p.cols % 8 == 0)
    return launch(fp8_quantize_block_bf16_kernel, tiles, dim3(256), 0, st, p);
  if (p.x_row == 1 && p.x_col != 1)
    return base && p.x_col % kAlign == 0 ? launch_tile<T, true, true>(p, st) : launch_tile<T, true, false>(p, st);
  return p.x_col == 1 && base && p.x_row % kAlign == 0 ? launch_tile<T, false, true>(p, st)
                                                       : launch_tile<T, false, false>(p, st);
}

int fp8_quantize_both(const sb_fp8_quantize_args& d, const sb_fp8_quantize_args& t, cudaStream_t st) {
  if (d.dtype != SB_BF16 || d.block_rows != 1 || d.batch != 1 || d.row_index || d.x_col != 1 || d.x_row % 8 ||
      d.cols % 8 || reinterpret_cast<uintptr_t>(d.x) % 16 || d.cols > 65535 * 128 || d.rows <= 0)
    return SB_ERR_UNSUPPORTED;
  return launch(fp8_quantize_transposed_bf16_kernel<true>, dim3((t.cols + 127) / 128, (t.rows + 127) / 128), dim3(256), 0,
                st, t, d);
}

}  // namespace sb

using namespace sb;

extern "C" SB_API int sb_fp8_quantize_blocks(const sb_fp8_quantize_args* args, void* stream) {
  if (!args) return SB_ERR_ARG;
  const sb_fp8_quantize_args& p = *args;
  if ((p.dtype != SB_F32 && p.dtype != SB_BF16) || (p.block_rows != 1 && p.block_rows != 128) || p.batch < 0 ||
      p.batch > 65535 || p.rows < 0 || p.rows > kMaxExtent || p.cols < 0 || p.cols > kMaxCols ||
      p.ldq % 16 || p.q_batch % 16 || p.ldq < p.cols ||
      ((p.row_index || p.row_count) && (p.block_rows != 1 || p.batch != 1)))
    return SB_ERR_ARG;
  if (p.batch == 0 || p.rows == 0 || p.cols == 0) return SB_OK;
  if (!p.x || !p.q || !p.scale || reinterpret_cast<uintptr_t>(p.q) % 16) return SB_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return p.dtype == SB_F32 ? quantize_typed<float>(p, st) : quantize_typed<__nv_bfloat16>(p, st);
}
