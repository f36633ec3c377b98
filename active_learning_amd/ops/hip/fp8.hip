// e4m3 blocks: quantisation and matrix products with a scale for each block of
// 128 (layout and rounding in al_fp8.h).
//
//   C[m,n] = sum over blocks b of sa[m,b] * sb[n,b] * (sum over k in b of a[m,k] * b[n,k]) + bias[n]
//
// Both operands have the contraction along their rows. The 8-bit matrix
// instruction adds its products in groups of eight and drops what lies more
// than 13 bits under a group's largest product: relative errors of 1e-5 to 7e-5
// of a result (normal and heavy-tailed data, 2048 deep), far under a 16-bit
// output's rounding (2^-9, 2^-12) and over a 32-bit one's. 32-bit outputs are therefore
// computed with bf16 instructions, into which e4m3 codes convert exactly.

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

// --------------------------------------------------------------------------
// products
// --------------------------------------------------------------------------

struct Gemm {
  const unsigned char *a, *b;
  const void *sa, *sb;        // scales: a by row and block, b by row (or tile) and block
  long lda, ldb;              // bytes from row to row, 128 for each block
  int sa_stride, sb_stride;   // scales from row to row
  int m, n, blocks;           // blocks: of 128 along the contraction
  int b_tile;                 // b's scales are those of 128x128 tiles
  const void* bias;
  int bias_type;
  void* out;
  int out_type;
  float* split_out;           // partial sums [split][m][n] where the contraction is split
  int splits;
};

AL_DEV float bias_at(const void* p, int type, int n) {
  return type == kTypeF32 ? ((const float*)p)[n]
         : type == kTypeBF16 ? (float)((const __bf16*)p)[n] : (float)((const _Float16*)p)[n];
}
AL_DEV void store_out(void* p, int type, long at, float v) {
  if (type == kTypeF32) ((float*)p)[at] = v;
  else if (type == kTypeBF16) ((__bf16*)p)[at] = (__bf16)v;
  else ((_Float16*)p)[at] = (_Float16)v;
}

// one block's 16x16 products, unscaled; EXACT: in bf16 instructions
template <bool EXACT> AL_DEV f32x4 block_product(i32x8 x, i32x8 y) {
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  if (!EXACT) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, zero, 0, 0, 0, 0, 0, 0);
  f32x4 d = zero;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bf16x8v u, v;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bf16x2v u0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[2 * i + h], 1.f, false);
      const bf16x2v u1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[2 * i + h], 1.f, true);
      const bf16x2v v0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y[2 * i + h], 1.f, false);
      const bf16x2v v1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y[2 * i + h], 1.f, true);
      u[4 * h] = u0[0]; u[4 * h + 1] = u0[1]; u[4 * h + 2] = u1[0]; u[4 * h + 3] = u1[1];
      v[4 * h] = v0[0]; v[4 * h + 1] = v0[1]; v[4 * h + 2] = v1[0]; v[4 * h + 3] = v1[1];
    }
    d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(u, v, d, 0, 0, 0);
  }
  return d;
}

// 128x128 outputs a workgroup, four waves of 64x64, one block of 128 a step
// through 32 KB of LDS. Rows of b are the first operand, so that a lane holds
// four neighbouring columns of an output row.
template <bool EXACT, int KIND>
__launch_bounds__(256)
__global__ void gemm_kernel(Gemm g) {
  __shared__ __align__(16) unsigned char lds_a[128 * 128], lds_b[128 * 128];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int l15 = lane & 15, l4 = lane >> 4;
  const int m0 = blockIdx.x * 128, n0 = blockIdx.y * 128;
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // chunk c of a row lies at c ^ ((row >> 1) & 7): 16 rows' chunks fall on
  // different banks
  const int lrow = t >> 3, lchunk = t & 7;
  const int first = (int)((long)g.blocks * blockIdx.z / g.splits);
  const int last = (int)((long)g.blocks * (blockIdx.z + 1) / g.splits);
  for (int kb = first; kb < last; ++kb) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = lrow + i * 32;
      const long ra = min(m0 + r, g.m - 1), rb = min(n0 + r, g.n - 1);
      const int at = r * 128 + ((lchunk ^ ((r >> 1) & 7)) << 4);
      *(i32x4*)(lds_a + at) = *(const i32x4*)(g.a + ra * g.lda + (long)kb * kQB + lchunk * 16);
      *(i32x4*)(lds_b + at) = *(const i32x4*)(g.b + rb * g.ldb + (long)kb * kQB + lchunk * 16);
    }
    __syncthreads();
    auto fragment = [&](const unsigned char* lds, int r) {
      const int s = (r >> 1) & 7;
      const i32x4 lo = *(const i32x4*)(lds + r * 128 + (((2 * l4) ^ s) << 4));
      const i32x4 hi = *(const i32x4*)(lds + r * 128 + (((2 * l4 + 1) ^ s) << 4));
      return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    i32x8 fa[4];
    float sa[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      fa[i] = fragment(lds_a, wm + i * 16 + l15);
      sa[i] = load_scale<KIND>(g.sa, (long)min(m0 + wm + i * 16 + l15, g.m - 1) * g.sa_stride + kb);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const i32x8 fb = fragment(lds_b, wn + j * 16 + l15);
      f32x4 sb;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = min(n0 + wn + j * 16 + l4 * 4 + r, g.n - 1);
        sb[r] = load_scale<KIND>(g.sb, (long)(g.b_tile ? n / kQB : n) * g.sb_stride + kb);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 d = block_product<EXACT>(fb, fa[i]);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = fmaf(d[r], sa[i] * sb[r], acc[i][j][r]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + wm + i * 16 + l15;
    if (m >= g.m) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = n0 + wn + j * 16 + l4 * 4 + r;
        if (n >= g.n) continue;
        if (g.splits > 1)
          g.split_out[((long)blockIdx.z * g.m + m) * g.n + n] = acc[i][j][r];
        else
          store_out(g.out, g.out_type, (long)m * g.n + n,
                    acc[i][j][r] + (g.bias ? bias_at(g.bias, g.bias_type, n) : 0.f));
      }
  }
}

// joins the partial sums of a split contraction, in order
__launch_bounds__(256)
__global__ void gemm_join_kernel(Gemm g) {
  const long count = (long)g.m * g.n;
  for (long i = grid_stride_begin(); i < count; i += grid_stride_step()) {
    float s = 0.f;
    for (int z = 0; z < g.splits; ++z) s += g.split_out[z * count + i];
    store_out(g.out, g.out_type, i, s + (g.bias ? bias_at(g.bias, g.bias_type, (int)(i % g.n)) : 0.f));
  }
}

// Up to 16 rows, straight from the values: a workgroup computes 16 columns, its
// eight waves take every eighth block of the contraction, quantise x's block as
// they read it, and join through LDS in order. What it costs is b's bytes.
template <typename T, bool EXACT, int KIND>
__launch_bounds__(512)
__global__ void few_rows_kernel(const T* __restrict__ x, long x_stride, int dim, Gemm g) {
  __shared__ f32x4 lds[8][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l15 = lane & 15, l4 = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const unsigned char* b = g.b + (long)min(n0 + l15, g.n - 1) * g.ldb + l4 * 32;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int kb = wave; kb < g.blocks; kb += 8) {
    const i32x4 lo = *(const i32x4*)(b + (long)kb * kQB), hi = *(const i32x4*)(b + (long)kb * kQB + 16);
    const i32x8 fb = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    const int c = kb * kQB + l4 * 32;
    f32x8 f[4];
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = f32x8{0, 0, 0, 0, 0, 0, 0, 0};
      if (l15 < g.m) f[i] = load8_upto(x + l15 * x_stride + c + i * 8, dim - c - i * 8);
      top = max(top, amax8(f[i]));
    }
    top = max(top, (unsigned)__shfl_xor((int)top, 16, 64));
    top = max(top, (unsigned)__shfl_xor((int)top, 32, 64));
    const BlockScale s = block_scale<KIND>(top);
    i32x8 fa;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const i32x2 codes = keep_upto(to_fp8(f[i], s.inv), dim - c - i * 8);
      fa[2 * i] = codes[0];
      fa[2 * i + 1] = codes[1];
    }
    const float sa = KIND == kF32 ? __uint_as_float(s.code)
                                  : __uint_as_float(s.code == 255u ? 0x7fc00000u : s.code << 23);
    const f32x4 d = block_product<EXACT>(fb, fa);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = min(n0 + l4 * 4 + r, g.n - 1);
      const float sb = load_scale<KIND>(g.sb, (long)(g.b_tile ? n / kQB : n) * g.sb_stride + kb);
      acc[r] = fmaf(d[r], sa * sb, acc[r]);
    }
  }
  lds[wave][lane] = acc;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) acc += lds[w][lane];
  if (l15 >= g.m) return;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int n = n0 + l4 * 4 + r;
    if (n < g.n)
      store_out(g.out, g.out_type, (long)l15 * g.n + n,
                acc[r] + (g.bias ? bias_at(g.bias, g.bias_type, n) : 0.f));
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

// how many parts the contraction is split into; the caller gives that many
// [m][n] matrices of floats where there are more than one
extern "C" int al_fp8_gemm_splits(int m, int n, int blocks) {
  const long tiles = (long)((m + 127) / 128) * ((n + 127) / 128);
  int s = (int)std::min((long)blocks / 4, 256 / std::max(tiles, 1l));
  return std::max(1, std::min(s, 16));
}

extern "C" void al_fp8_gemm(int kind, const void* a, const void* sa, long lda, int sa_stride,
                            const void* b, const void* sb, long ldb, int sb_stride, int b_tile,
                            int m, int n, int blocks, const void* bias, int bias_type, void* out,
                            int out_type, float* split_out, int splits, hipStream_t stream) {
  Gemm g = {(const unsigned char*)a, (const unsigned char*)b, sa, sb, lda, ldb, sa_stride,
            sb_stride, m, n, blocks, b_tile, bias, bias_type, out, out_type, split_out, splits};
  const dim3 grid((m + 127) / 128, (n + 127) / 128, splits);
  with_kind(kind, [&](auto k) {
    constexpr int KIND = decltype(k)::value;
    if (out_type == kTypeF32) hipLaunchKernelGGL((gemm_kernel<true, KIND>), grid, dim3(256), 0, stream, g);
    else hipLaunchKernelGGL((gemm_kernel<false, KIND>), grid, dim3(256), 0, stream, g);
  });
  if (splits > 1) {
    const int join = (int)std::min(((long)m * n + 255) / 256, 2048l);
    hipLaunchKernelGGL(gemm_join_kernel, dim3(join), dim3(256), 0, stream, g);
  }
}

extern "C" void al_fp8_few_rows(int kind, int type, const void* x, long x_stride, int dim,
                                const void* b, const void* sb, long ldb, int sb_stride, int b_tile,
                                int m, int n, int blocks, const void* bias, int bias_type,
                                void* out, hipStream_t stream) {
  Gemm g = {nullptr, (const unsigned char*)b, nullptr, sb, 0, ldb, 0, sb_stride, m, n, blocks,
            b_tile, bias, bias_type, out, type, nullptr, 1};
  with_type(type, [&](auto* t) {
    with_kind(kind, [&](auto k) {
      typedef std::remove_pointer_t<decltype(t)> T;
      constexpr int KIND = decltype(k)::value;
      hipLaunchKernelGGL((few_rows_kernel<T, std::is_same<T, float>::value, KIND>),
                         dim3((n + 15) / 16), dim3(512), 0, stream, (const T*)x, x_stride, dim, g);
    });
  });
}
