// e4m3 blocks: quantisation of matrices by rows, by tiles and transposed (layout
// and rounding in al_fp8.h). Bound by memory: each value is read once.

#include "al_fp8.h"

namespace {

// --------------------------------------------------------------------------
// quantisation
// --------------------------------------------------------------------------

// 1x128 blocks of a matrix whose rows may be any distance apart (and whose
// columns may be, with STRIDED): sixteen lanes a block
template <typename T, int KIND, bool STRIDED>
__launch_bounds__(256)
__global__ void quant_rows_kernel(const T* __restrict__ x, long row_stride, long col_stride,
                                  unsigned char* __restrict__ q, void* __restrict__ scale,
                                  long blocks, int dim, int pitch, int scale_stride) {
  const int per_row = pitch / kQB, lane = threadIdx.x & 15;
  for (long b = (long)blockIdx.x * 16 + (threadIdx.x >> 4); b < blocks; b += (long)gridDim.x * 16) {
    const long r = b / per_row;
    const int kb = (int)(b - r * per_row), c = kb * kQB + lane * 8;
    f32x8 f = {0, 0, 0, 0, 0, 0, 0, 0};
    if (STRIDED) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < dim) f[i] = (float)x[r * row_stride + (c + i) * col_stride];
    } else {
      f = load8_upto(x + r * row_stride + c, dim - c);
    }
    const BlockScale s = block_scale<KIND>(max_over_16(amax8(f)));
    *(i32x2*)(q + r * pitch + c) = keep_upto(to_fp8(f, s.inv), dim - c);
    if (lane == 0) store_scale<KIND>(scale, r * scale_stride + kb, s.code);
  }
}

// One 128x128 tile a workgroup, read once: 8x8 values a thread. Writes the
// tile's codes by rows (q), and transposed (qt), with blocks along the rows
// that each is stored in; with TILE one scale serves all of it. part: sums of
// each column over the tile's rows, for the gradient of a bias.
template <typename T, int KIND, bool TILE>
__launch_bounds__(256)
__global__ void quant_tile_kernel(const T* __restrict__ x, long row_stride, int rows, int cols,
                                  unsigned char* __restrict__ q, void* __restrict__ scale,
                                  int pitch, int scale_stride,
                                  unsigned char* __restrict__ qt, void* __restrict__ scale_t,
                                  int pitch_t, int scale_t_stride, float* __restrict__ part) {
  __shared__ unsigned words[16][kQB];  // column maxima or sums of each 8 rows
  __shared__ float col_inv[kQB];
  __shared__ __align__(16) unsigned char bytes[kQB][144];
  const int t = threadIdx.x, c8 = t & 15, rg = t >> 4;
  const int r0 = blockIdx.y * kQB, c0 = blockIdx.x * kQB;
  const int row = r0 + rg * 8, col = c0 + c8 * 8;
  f32x8 f[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    f[j] = f32x8{0, 0, 0, 0, 0, 0, 0, 0};
    if (row + j < rows) f[j] = load8_upto(x + (long)(row + j) * row_stride + col, cols - col);
  }
  BlockScale all;
  if (TILE) {
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, amax8(f[j]));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
    if ((t & 63) == 0) words[0][t >> 6] = m;
    __syncthreads();
    m = max(max(words[0][0], words[0][1]), max(words[0][2], words[0][3]));
    all = block_scale<KIND>(m);
    if (t == 0) {
      if (q) store_scale<KIND>(scale, (long)blockIdx.y * scale_stride + blockIdx.x, all.code);
      if (qt) store_scale<KIND>(scale_t, (long)blockIdx.x * scale_t_stride + blockIdx.y, all.code);
    }
    __syncthreads();
  }
  if (q) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      BlockScale s = all;
      if (!TILE) s = block_scale<KIND>(max_over_16(amax8(f[j])));
      if (row + j < rows) {
        *(i32x2*)(q + (long)(row + j) * pitch + col) = keep_upto(to_fp8(f[j], s.inv), cols - col);
        if (!TILE && c8 == 0)
          store_scale<KIND>(scale, (long)(row + j) * scale_stride + blockIdx.x, s.code);
      }
    }
  }
  if (part) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) s += f[j][i];
      words[rg][c8 * 8 + i] = __float_as_uint(s);
    }
    __syncthreads();
    if (t < kQB && c0 + t < cols) {
      float s = 0.f;
#pragma unroll
      for (int g = 0; g < 16; ++g) s += __uint_as_float(words[g][t]);
      part[(long)blockIdx.y * cols + c0 + t] = s;
    }
    __syncthreads();
  }
  if (!qt) return;
  if (!TILE) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      unsigned m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, abs_bits(f[j][i]));
      words[rg][c8 * 8 + i] = m;
    }
    __syncthreads();
    if (t < kQB) {
      unsigned m = 0;
#pragma unroll
      for (int g = 0; g < 16; ++g) m = max(m, words[g][t]);
      const BlockScale s = block_scale<KIND>(m);
      col_inv[t] = s.inv;
      if (c0 + t < cols)
        store_scale<KIND>(scale_t, (long)(c0 + t) * scale_t_stride + blockIdx.y, s.code);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    f32x8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = f[j][i];
    const float inv = TILE ? all.inv : col_inv[c8 * 8 + i];
    *(i32x2*)&bytes[c8 * 8 + i][rg * 8] = keep_upto(to_fp8(v, inv), rows - row);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = (t >> 3) + i * 32, at = (t & 7) * 16;
    if (c0 + c < cols)
      *(i32x4*)(qt + (long)(c0 + c) * pitch_t + r0 + at) = *(const i32x4*)&bytes[c][at];
  }
}

template <typename F> void with_type(int type, F f) {
  if (type == kTypeF32) f((float*)0);
  else if (type == kTypeBF16) f((__bf16*)0);
  else f((_Float16*)0);
}
template <typename F> void with_kind(int kind, F f) {
  if (kind == kE8M0) f(std::integral_constant<int, kE8M0>{});
  else f(std::integral_constant<int, kF32>{});
}

}  // namespace

extern "C" void al_quant_rows(int type, int kind, const void* x, long row_stride,
                              long col_stride, void* q, void* scale, long rows, int dim,
                              int pitch, int scale_stride, hipStream_t stream) {
  const long blocks = rows * (pitch / kQB);
  const int grid = (int)std::min((blocks + 15) / 16, 8192l);
  with_type(type, [&](auto* t) {
    with_kind(kind, [&](auto k) {
      typedef std::remove_pointer_t<decltype(t)> T;
      constexpr int KIND = decltype(k)::value;
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, stream, (const T*)x, row_stride,
                           col_stride, (unsigned char*)q, scale, blocks, dim, pitch, scale_stride);
      };
      col_stride == 1 ? go(quant_rows_kernel<T, KIND, false>) : go(quant_rows_kernel<T, KIND, true>);
    });
  });
}

extern "C" void al_quant_tile(int type, int kind, int tile, const void* x, long row_stride,
                              int rows, int cols, void* q, void* scale, int pitch,
                              int scale_stride, void* qt, void* scale_t, int pitch_t,
                              int scale_t_stride, float* part, hipStream_t stream) {
  const dim3 grid((cols + kQB - 1) / kQB, (rows + kQB - 1) / kQB);
  with_type(type, [&](auto* t) {
    with_kind(kind, [&](auto k) {
      typedef std::remove_pointer_t<decltype(t)> T;
      constexpr int KIND = decltype(k)::value;
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, (const T*)x, row_stride, rows, cols,
                           (unsigned char*)q, scale, pitch, scale_stride, (unsigned char*)qt,
                           scale_t, pitch_t, scale_t_stride, part);
      };
      tile ? go(quant_tile_kernel<T, KIND, true>) : go(quant_tile_kernel<T, KIND, false>);
    });
  });
}
