// e4m3 blocks: quantisation of matrices by rows, by tiles and transposed (layout
// and rounding in al_fp8.h). Bound by memory: each value is read once.

#include "al_fp8.h"

#include <algorithm>

namespace {

// --------------------------------------------------------------------------
// quantisation
// --------------------------------------------------------------------------

// 1x128 blocks of a matrix whose rows may be any distance apart (and whose
// columns may be, with STRIDED): sixteen lanes a block. 65536x2048 in bf16 takes 76 us,
// 5.3 TB/s.
template <typename T, int KIND, bool STRIDED>
__launch_bounds__(256)
__global__ void quant_rows_kernel(const T* __restrict__ x, long row_stride, long col_stride,
                                  unsigned char* __restrict__ q, void* __restrict__ scale,
                                  long blocks, int dim, int pitch, int scale_stride) {
  const int per_row = pitch / kQB, lane = threadIdx.x & 15;
  for (long b = (long)blockIdx.x * 16 + (threadIdx.x >> 4); b < blocks; b += (long)gridDim.x * 16) {
    const long r = b / per_row;
    const int kb = (int)(b - r * per_row), c = kb * kQB + lane * 8;
    typename Raw8<T>::V v;
    if (STRIDED) {
      typename Vec8<T>::V e = (typename Vec8<T>::V)(T)0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < dim) e[i] = x[r * row_stride + (c + i) * col_stride];
      v = __builtin_bit_cast(typename Raw8<T>::V, e);
    } else {
      v = raw8_upto(x + r * row_stride + c, dim - c);
    }
    Top<T> top;
    top.add(v);
    const BlockScale s = block_scale<KIND>(max_over_16(top.bits()));
    *(i32x2*)(q + r * pitch + c) = keep_upto(raw_to_fp8<T, KIND>(v, s), dim - c);
    if (lane == 0) store_scale<KIND>(scale, r * scale_stride + kb, s.code);
  }
}

// 128x128 tiles, each read once, 8x8 values a thread, the next one's while this one is
// worked on. Writes a tile's codes by rows (q), and transposed (qt), with blocks along
// the rows that each is stored in; with TILE one scale serves all of it. part: sums of
// each column over the tile's rows in 64 bits, for the gradient of a bias. By rows and transposed
// 8192x4096 in bf16 takes 23 us (its bytes at a copy's rate: 25), 16384x8192 121 (100),
// with 32-bit scales 27 and 128; with the sums 29 and 128.
template <typename T, int KIND, bool TILE>
__launch_bounds__(256)
__global__ void quant_tile_kernel(const T* __restrict__ x, long row_stride, int rows, int cols,
                                  unsigned char* __restrict__ q, void* __restrict__ scale,
                                  int pitch, int scale_stride,
                                  unsigned char* __restrict__ qt, void* __restrict__ scale_t,
                                  int pitch_t, int scale_t_stride, double* __restrict__ part,
                                  int across, int tiles) {
  constexpr bool WIDE = std::is_same<T, float>::value;
  // column maxima (16-bit types: of two columns a word) of each 8 rows
  __shared__ unsigned words[16][kQB];
  __shared__ unsigned col_code[kQB];
  // a column's eight bytes of rows 8u .. 8u + 7 lie at u ^ (column >> 3): lanes that
  // write eight columns apart then fall on different banks
  __shared__ __align__(16) unsigned char bytes[kQB][kQB];
  const int t = threadIdx.x, c8 = t & 15, rg = t >> 4;
  typedef typename Raw8<T>::V Raw;
  auto load = [&](Raw (&v)[8], int tile) {
    const int row = tile / across * kQB + rg * 8, col = tile % across * kQB + c8 * 8;
    if (row + 8 <= rows && col + 8 <= cols) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = raw8(x + (long)(row + j) * row_stride + col);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = row + j < rows ? raw8_upto(x + (long)(row + j) * row_stride + col, cols - col) : (Raw)0;
    }
  };
  // the next tile's values are on their way while this one's are worked on
  Raw v[8], next[8];
  load(v, blockIdx.x);
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int by = tile / across, bx = tile % across;
    const int r0 = by * kQB, c0 = bx * kQB, row = r0 + rg * 8, col = c0 + c8 * 8;
    if (tile + (int)gridDim.x < tiles) load(next, tile + gridDim.x);
    BlockScale all;
    if (TILE) {
      Top<T> top;
#pragma unroll
      for (int j = 0; j < 8; ++j) top.add(v[j]);
      unsigned m = top.bits();
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
      if ((t & 63) == 0) words[0][t >> 6] = m;
      __syncthreads();
      m = max(max(words[0][0], words[0][1]), max(words[0][2], words[0][3]));
      all = block_scale<KIND>(m);
      if (t == 0) {
        if (q) store_scale<KIND>(scale, (long)by * scale_stride + bx, all.code);
        if (qt) store_scale<KIND>(scale_t, (long)bx * scale_t_stride + by, all.code);
      }
      __syncthreads();
    }
    if (q) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        BlockScale s = all;
        if (!TILE) {
          Top<T> top;
          top.add(v[j]);
          s = block_scale<KIND>(max_over_16(top.bits()));
        }
        if (row + j < rows) {
          *(i32x2*)(q + (long)(row + j) * pitch + col) = keep_upto(raw_to_fp8<T, KIND>(v[j], s), cols - col);
          if (!TILE && c8 == 0)
            store_scale<KIND>(scale, (long)(row + j) * scale_stride + bx, s.code);
        }
      }
    }
    if (part) {
      double* sums = (double*)bytes;  // of each 8 rows, in the codes' place
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        double s = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) s += (double)(float)__builtin_bit_cast(typename Vec8<T>::V, v[j])[i];
        sums[rg * kQB + c8 * 8 + i] = s;
      }
      __syncthreads();
      if (t < kQB && c0 + t < cols) {
        double s = 0;
#pragma unroll
        for (int g = 0; g < 16; ++g) s += sums[g * kQB + t];
        part[(long)by * cols + c0 + t] = s;
      }
      __syncthreads();
    }
    if (qt) {
      if (!TILE) {
        if constexpr (WIDE) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            unsigned m = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, abs_bits(v[j][i]));
            words[rg][c8 * 8 + i] = m;
          }
        } else {
          i32x4 m;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            Top<T> top;
#pragma unroll
            for (int j = 0; j < 8; ++j) top.add(v[j][i]);
            m[i] = __builtin_bit_cast(int, top.m);
          }
          *(i32x4*)&words[rg][c8 * 4] = m;
        }
        __syncthreads();
        if (t < kQB) {
          unsigned m = 0;
          if constexpr (WIDE) {
#pragma unroll
            for (int g = 0; g < 16; ++g) m = max(m, words[g][t]);
          } else {
#pragma unroll
            for (int g = 0; g < 16; ++g) m = max(m, words[g][t >> 1] >> (16 * (t & 1)) & 0xffffu);
            m = Top<T>::bits((unsigned short)m);
          }
          const BlockScale s = block_scale<KIND>(m);
          col_code[t] = KIND == kE8M0 ? s.code : __float_as_uint(s.inv);
          if (c0 + t < cols)
            store_scale<KIND>(scale_t, (long)(c0 + t) * scale_t_stride + by, s.code);
        }
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        BlockScale s = all;
        if (!TILE) {
          const unsigned c = col_code[c8 * 8 + i];
          s.code = c;
          s.inv = __uint_as_float(c);
        }
        i32x2 codes;
        if constexpr (WIDE || KIND == kF32) {
          f32x8 f;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if constexpr (WIDE) f[j] = v[j][i];
            else f[j] = (float)__builtin_bit_cast(typename Vec8<T>::V, v[j])[i];
          }
          codes = to_fp8<KIND>(f, s);
        } else {
          // two rows of a column side by side, as the conversion takes them
          const float scale_by = e8m0_value(s.code);
          int two[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            two[j] = (int)__builtin_amdgcn_perm((unsigned)v[2 * j + 1][i >> 1], (unsigned)v[2 * j][i >> 1],
                                                i & 1 ? 0x07060302u : 0x05040100u);
          codes[0] = two_codes<T, true>(two_codes<T, false>(0, two[0], scale_by), two[1], scale_by);
          codes[1] = two_codes<T, true>(two_codes<T, false>(0, two[2], scale_by), two[3], scale_by);
        }
        *(i32x2*)&bytes[c8 * 8 + i][(rg ^ c8) * 8] = keep_upto(codes, rows - row);
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = (t >> 3) + i * 32, at = t & 7, turn = c >> 3;
        i32x4 two = *(const i32x4*)&bytes[c][(at ^ turn >> 1) * 16];
        if (turn & 1) two = i32x4{two[2], two[3], two[0], two[1]};
        if (c0 + c < cols) *(i32x4*)(qt + (long)(c0 + c) * pitch_t + r0 + at * 16) = two;
      }
      __syncthreads();  // the bytes have been read
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = next[j];
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
                              int scale_t_stride, double* part, hipStream_t stream) {
  const int across = (cols + kQB - 1) / kQB, tiles = across * ((rows + kQB - 1) / kQB);
  // as many as are resident, 32-bit scales' registers leaving three blocks a unit (fp32
  // input, two: 1024 blocks are two even rounds)
  const dim3 grid(std::min(tiles, kind == kF32 && type != kTypeF32 ? 768 : 1024));
  with_type(type, [&](auto* t) {
    with_kind(kind, [&](auto k) {
      typedef std::remove_pointer_t<decltype(t)> T;
      constexpr int KIND = decltype(k)::value;
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, (const T*)x, row_stride, rows, cols,
                           (unsigned char*)q, scale, pitch, scale_stride, (unsigned char*)qt,
                           scale_t, pitch_t, scale_t_stride, part, across, tiles);
      };
      tile ? go(quant_tile_kernel<T, KIND, true>) : go(quant_tile_kernel<T, KIND, false>);
    });
  });
}
