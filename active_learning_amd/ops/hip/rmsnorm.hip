// Root-mean-square norm over the last axis, with an optional residual's
// addition in front of it and an optional output in e4m3 blocks.
//
//   s = x + r (rounded to their type, stored)      rstd = 1 / sqrt(mean(s^2) + eps)
//   y = s * rstd * w
//   ds = rstd * (w dy - u * mean(w dy u)) + ds_out,   u = s * rstd
//   dw = sum over rows of dy * u
//
// The norm is that of the stored, rounded sum: the backward pass reads the same
// numbers and differentiates what the forward pass computed. Squares, and dw over its
// partial rows, are summed in 64 bits, the rest is in 32, rounded to the type on the store.

#include "al_fp8.h"

namespace {

enum { kOutPlain = 0, kOutE8M0 = 1, kOutF32 = 2 };

// sum over the TPR threads of a row; every thread gets it
template <int TPR, typename F> AL_DEV F row_sum(F v, F* lds) {
  v = wave_total(v);
  if (TPR == 64) return v;
  constexpr int W = TPR / 64;
  __syncthreads();  // the last row's sums have been read
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  F s = 0;
#pragma unroll
  for (int i = 0; i < W; ++i) s += lds[i];
  return s;
}

constexpr int block_of(int tpr) { return tpr < 256 ? 256 : tpr; }

// One row per TPR threads, VPT vectors of eight values each, rows strided over
// the grid so that the weight stays in registers. VPT == 0: rows of any length,
// read twice.
//
// Squares are summed in 64 bits: those of values over 1.8e19 leave the range of 32, and a
// row of finite values would become zeros. (Where the root is over 2^126, 1 / root is below
// the normal range and has 21 bits.) 16383x4096 in bf16 with a residual, traced: 93 us,
// with 32 bits 88.
//
// In front of an e4m3 output 1 / root and the first product are held as pairs of floats: y
// is then the exact value rounded once, and a value next to a border between two codes or
// scales falls on its own side of it (with 32 bits throughout, 50 codes in 123 million did
// not). At 130000x2048 in bf16 with a residual that and the sum cost 355 us against 336, at
// 5.3 and 5.5 TB/s; the reductions go through lane permutations
// of the vector unit (LDS shuffles: 187 us for 160 without a residual).
//
// One vector a thread: no more registers than let eight waves share a SIMD, as the
// grid counts on (with seven the last eighth of the blocks runs alone: 426 us for 355).
template <typename T, typename W, int TPR, int VPT, bool RES, int OUT>
__launch_bounds__(block_of(TPR), VPT == 1 ? 8 : 1)
__global__ void rms_fwd_kernel(const T* __restrict__ x, long x_stride,
                               const T* __restrict__ res, long res_stride,
                               const W* __restrict__ w, T* __restrict__ y,
                               T* __restrict__ total, float* __restrict__ rstd_out,
                               unsigned char* __restrict__ q, void* __restrict__ scale,
                               long rows, int dim, int pitch, int scale_stride,
                               float eps) {
  __shared__ double lds[16];
  constexpr int RPB = block_of(TPR) / TPR;
  constexpr int N = VPT ? VPT : 1;
  const int t = threadIdx.x % TPR;
  const int sweeps = VPT ? VPT : (max(dim, pitch) + TPR * 8 - 1) / (TPR * 8);
  f32x8 wv[N];
  if (VPT) {
#pragma unroll
    for (int i = 0; i < N; ++i) wv[i] = load8_upto(w + (i * TPR + t) * 8, dim - (i * TPR + t) * 8);
  }
  const double per_value = 1.0 / (double)dim;
  const long first = (long)blockIdx.x * RPB;
  for (long r0 = first; r0 < rows; r0 += (long)gridDim.x * RPB) {
    const long r = r0 + threadIdx.x / TPR;
    if (RPB > 1 && r >= rows) break;  // whole waves; no barrier when RPB > 1
    f32x8 v[N];
    double ss = 0;
    auto take = [&](int c) {
      f32x8 f = load8_upto(x + r * x_stride + c, dim - c);
      if (RES) {
        f += load8_upto(res + r * res_stride + c, dim - c);
        if (c < dim) store8_upto(total + r * dim + c, f, dim - c);
        f = __builtin_convertvector(__builtin_convertvector(f, typename Vec8<T>::V), f32x8);
      }
      return f;
    };
#pragma unroll
    for (int i = 0; i < N; ++i) {
      for (int k = i; k < sweeps; k += N) {
        v[i] = take((k * TPR + t) * 8);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += (double)v[i][j] * (double)v[i][j];
      }
    }
    ss = row_sum<TPR>(ss, lds);
    // the hardware's root has 23 bits; a step of Newton's method doubles them
    const double mean = ss * per_value + (double)eps;
    double root = __builtin_amdgcn_rsq(mean);
    if (!isinf(mean)) root *= 1.5 - 0.5 * mean * root * root;
    const float rstd = (float)root, rstd_low = (float)(root - (double)rstd);
    if (rstd_out && t == 0) rstd_out[r] = rstd;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      for (int k = i; k < sweeps; k += N) {
        const int c = (k * TPR + t) * 8;
        f32x8 f, ww;
        if (VPT) { f = v[i]; ww = wv[i]; }
        else {
          ww = load8_upto(w + c, dim - c);
          // the stored sum, where there is one: this thread wrote it
          f = RES ? load8_upto(total + r * dim + c, dim - c)
                  : load8_upto(x + r * x_stride + c, dim - c);
        }
        if (OUT == kOutPlain) {
          f = f * rstd * ww;
          if (c < dim) store8_upto(y + r * dim + c, f, dim - c);
        } else {
          constexpr int KIND = OUT == kOutE8M0 ? kE8M0 : kF32;
          // the exact value's nearest, and what the exact value is over it
          auto product = [&](int j, float& over) {
#pragma clang fp contract(off)
            const float u = f[j] * rstd;
            const float low = fmaf(f[j], rstd_low, fmaf(f[j], rstd, -u)) * ww[j];
            const float nearest = fmaf(u, ww[j], low);
            over = fmaf(u, ww[j], -nearest) + low;
            return nearest;
          };
          f32x8 out;
          float over;
#pragma unroll
          for (int j = 0; j < 8; ++j) out[j] = product(j, over);
          unsigned top = amax8(out);
          // the largest value a block's scale can hold, by its nearest: a little more
          // than that takes the next scale
          if (KIND == kE8M0 && (top & 0x7fffffu) == 0x600000u) {
            bool more = false;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float nearest = product(j, over);
              more |= abs_bits(nearest) == top && (nearest > 0.f ? over > 0.f : over < 0.f);
            }
            top += more;
          }
          const BlockScale b = block_scale<KIND>(max_over_16(top));
          if (c < pitch) {
            *(i32x2*)(q + r * pitch + c) = keep_upto(to_fp8<KIND>(out, b), dim - c);
            if ((t & 15) == 0 && c < dim)
              store_scale<KIND>(scale, r * scale_stride + c / kQB, b.code);
          }
        }
      }
    }
  }
}

// The same walk over the rows; dw is summed in registers over a block's rows,
// joined over its waves in order, and written as one partial row for each block. Bound by
// memory: 16383x4096 in bf16 with the sum's gradient 103 us, 5.2 TB/s.
template <typename T, typename W, int TPR, int VPT, bool DSUM>
__launch_bounds__(block_of(TPR))
__global__ void rms_bwd_kernel(const T* __restrict__ s, long s_stride,
                               const T* __restrict__ dy, const T* __restrict__ dsum,
                               const W* __restrict__ w, const float* __restrict__ rstd_in,
                               T* __restrict__ dx, float* __restrict__ part,
                               long rows, int dim) {
  __shared__ float lds[16];
  extern __shared__ float dw_lds[];
  constexpr int RPB = block_of(TPR) / TPR;
  constexpr int N = VPT ? VPT : 1;
  const int t = threadIdx.x % TPR;
  const int sweeps = VPT ? VPT : (dim + TPR * 8 - 1) / (TPR * 8);
  f32x8 wv[N], dw[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    dw[i] = f32x8{0, 0, 0, 0, 0, 0, 0, 0};
    if (VPT) wv[i] = load8_upto(w + (i * TPR + t) * 8, dim - (i * TPR + t) * 8);
  }
  for (long r0 = (long)blockIdx.x * RPB; r0 < rows; r0 += (long)gridDim.x * RPB) {
    const long r = r0 + threadIdx.x / TPR;
    if (RPB > 1 && r >= rows) break;
    const float rstd = rstd_in[r];
    f32x8 u[N], g[N], add[N];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      for (int k = i; k < sweeps; k += N) {
        const int c = (k * TPR + t) * 8;
        u[i] = load8_upto(s + r * s_stride + c, dim - c) * rstd;
        g[i] = load8_upto(dy + r * dim + c, dim - c);
        if (DSUM && VPT) add[i] = load8_upto(dsum + r * dim + c, dim - c);
        if (VPT) dw[i] += g[i] * u[i];
        g[i] *= VPT ? wv[i] : load8_upto(w + c, dim - c);
#pragma unroll
        for (int j = 0; j < 8; ++j) dot += g[i][j] * u[i][j];
      }
    }
    dot = row_sum<TPR>(dot, lds) / (float)dim;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      for (int k = i; k < sweeps; k += N) {
        const int c = (k * TPR + t) * 8;
        if (!VPT) {
          u[i] = load8_upto(s + r * s_stride + c, dim - c) * rstd;
          g[i] = load8_upto(dy + r * dim + c, dim - c) * load8_upto(w + c, dim - c);
        }
        f32x8 d = (g[i] - u[i] * dot) * rstd;
        if (DSUM) d += VPT ? add[i] : load8_upto(dsum + r * dim + c, dim - c);
        if (c < dim) store8_upto(dx + r * dim + c, d, dim - c);
      }
    }
  }
  if (!VPT || !part) return;
  if (RPB == 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * TPR + t) * 8;
      if (c < dim) store8_upto(part + (long)blockIdx.x * dim + c, dw[i], dim - c);
    }
  } else {
    for (int wave = 0; wave < RPB; ++wave) {
      if ((int)(threadIdx.x / TPR) == wave) {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int c = (i * TPR + t) * 8 + j;
            if (c < dim) {
              const float v = (wave ? dw_lds[c] : 0.f) + dw[i][j];
              if (wave == RPB - 1) part[(long)blockIdx.x * dim + c] = v;
              else dw_lds[c] = v;
            }
          }
      }
      __syncthreads();
    }
  }
}

// dw's partial rows for lengths that do not fit in registers: one column a
// thread, a strip of rows a block
template <typename T>
__global__ void rms_dw_kernel(const T* __restrict__ s, long s_stride,
                              const T* __restrict__ dy, const float* __restrict__ rstd,
                              float* __restrict__ part, long rows, int dim) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= dim) return;
  float sum = 0.f;
  for (long r = blockIdx.y; r < rows; r += gridDim.y)
    sum += (float)dy[r * dim + c] * ((float)s[r * s_stride + c] * rstd[r]);
  part[(long)blockIdx.y * dim + c] = sum;
}

// out[c] = sum over p of part[p][c] in 64 bits: 16 columns a block, the partial rows over
// 64 threads each, joined in order
template <typename P, typename W>
__launch_bounds__(1024)
__global__ void col_sum_kernel(const P* __restrict__ part, W* __restrict__ out,
                               int parts, int dim) {
  __shared__ double lds[64][17];
  const int x = threadIdx.x & 15, y = threadIdx.x >> 4, c = blockIdx.x * 16 + x;
  double s = 0;
  if (c < dim)
    for (int p = y; p < parts; p += 64) s += (double)part[(long)p * dim + c];
  lds[y][x] = s;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    __syncthreads();
    if (y < o) lds[y][x] += lds[y + o][x];
  }
  if (y == 0 && c < dim) out[c] = (W)(float)lds[0][x];
}

struct Shape { int tpr, vpt; };

// The forward pass. Up to 1024 values a wave holds a row and needs no barrier, longer
// rows are spread with one vector a thread, up to 32768 with a few: beyond that a row is
// read twice. Measured on 266 million values in bf16, us with the residual / without (of
// the plain form's shapes those that are not taken with sums in 32 bits):
//   1024 values, plain:  64 threads x 2 vectors 462 / 190, x 4 (half of them idle, fewer
//                        waves at once) 404 / 211; to e4m3, x 2, 355 / 165
//   2048 values:         64 x 4 plain 384 / 206, to e4m3 411; 256 x 1 389 / 192, 356 / 166
//   4096 values, plain:  256 x 2 460 / 191, 512 x 1 399 / 193
//   8192 values, e4m3:   256 x 4 403 / 167, 1024 x 1 340 / 179; plain 388 / 209, 387 / 185
// (their bytes at a copy's rate: plain 396 / 198, e4m3 346 / 148). The rule does not ask
// for the number of rows, so a row's numbers do not depend on the rows beside it.
Shape fwd_shape(int dim, bool res, int out) {
  const bool plain = out == kOutPlain;
  if (dim <= 512) return {64, 1};
  if (dim <= 1024) return {64, res && plain ? 4 : 2};
  if (dim <= 2048) return {256, 1};
  if (dim <= 4096) return {512, 1};
  if (dim <= 8192) return {1024, 1};
  if (dim <= 16384) return {1024, 2};
  if (dim <= 32768) return {1024, 4};
  return {1024, 0};
}
// The backward pass holds four times as much for each value: one vector a thread, or
// two where a wave holds a row. As many blocks as are resident at once (of 512 threads
// three a unit). Measured on 67 million values, us with the sum's gradient / without:
//   1000 values, bf16:  64 threads x 2 108 / 83, 256 x 1 170 / 129; fp32: 212 / 161, 206 / 148
//   4096 values, bf16:  768 blocks 103 / 79, 1024 blocks 120 / 92
// (their bytes at a copy's rate: bf16 100 / 75, fp32 200 / 150). Eight waves a SIMD by
// spilling registers: 4096 values 134.
Shape bwd_shape(bool wide, int dim) {
  if (dim <= 512) return {64, 1};
  if (dim <= 1024 && !wide) return {64, 2};
  if (dim <= 2048) return {256, 1};
  if (dim <= 4096) return {512, 1};
  if (dim <= 8192) return {1024, 1};
  if (dim <= 16384) return {1024, 2};
  return {1024, 0};
}

template <int N> using Int = std::integral_constant<int, N>;
template <typename F> void with_fwd_shape(Shape s, F f) {
  if (s.tpr == 64) s.vpt == 1 ? f(Int<64>{}, Int<1>{}) : s.vpt == 2 ? f(Int<64>{}, Int<2>{}) : f(Int<64>{}, Int<4>{});
  else if (s.tpr == 256) f(Int<256>{}, Int<1>{});
  else if (s.tpr == 512) f(Int<512>{}, Int<1>{});
  else s.vpt == 1 ? f(Int<1024>{}, Int<1>{}) : s.vpt == 2 ? f(Int<1024>{}, Int<2>{}) : s.vpt == 4 ? f(Int<1024>{}, Int<4>{}) : f(Int<1024>{}, Int<0>{});
}
template <typename F> void with_bwd_shape(Shape s, F f) {
  if (s.tpr == 64) s.vpt == 1 ? f(Int<64>{}, Int<1>{}) : f(Int<64>{}, Int<2>{});
  else if (s.tpr == 256) f(Int<256>{}, Int<1>{});
  else if (s.tpr == 512) f(Int<512>{}, Int<1>{});
  else s.vpt == 1 ? f(Int<1024>{}, Int<1>{}) : s.vpt == 2 ? f(Int<1024>{}, Int<2>{}) : f(Int<1024>{}, Int<0>{});
}

int blocks_for(Shape s, long rows, long most) {
  const int rpb = block_of(s.tpr) / s.tpr;
  return (int)std::min((rows + rpb - 1) / rpb, most);
}

template <typename T, typename W>
void fwd(const void* x, long x_stride, const void* res, long res_stride, const void* w,
         void* y, void* total, float* rstd, void* q, void* scale, int out, long rows,
         int dim, int pitch, int scale_stride, float eps, hipStream_t stream) {
  const Shape shape = fwd_shape(dim, res != nullptr, out);
  const int blocks = blocks_for(shape, rows, 2048);
  with_fwd_shape(shape, [&](auto tpr, auto vpt) {
    constexpr int TPR = decltype(tpr)::value, VPT = decltype(vpt)::value;
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(blocks), dim3(block_of(TPR)), 0, stream, (const T*)x,
                         x_stride, (const T*)res, res_stride, (const W*)w, (T*)y, (T*)total,
                         rstd, (unsigned char*)q, scale, rows, dim, pitch, scale_stride, eps);
    };
    if (out == kOutPlain) res ? go(rms_fwd_kernel<T, W, TPR, VPT, true, kOutPlain>) : go(rms_fwd_kernel<T, W, TPR, VPT, false, kOutPlain>);
    else if (out == kOutE8M0) res ? go(rms_fwd_kernel<T, W, TPR, VPT, true, kOutE8M0>) : go(rms_fwd_kernel<T, W, TPR, VPT, false, kOutE8M0>);
    else res ? go(rms_fwd_kernel<T, W, TPR, VPT, true, kOutF32>) : go(rms_fwd_kernel<T, W, TPR, VPT, false, kOutF32>);
  });
}

template <typename T, typename W>
void bwd(const void* s, long s_stride, const void* dy, const void* dsum, const void* w,
         const float* rstd, void* dx, float* part, void* dw, int parts, long rows, int dim,
         hipStream_t stream) {
  with_bwd_shape(bwd_shape(std::is_same<T, float>::value, dim), [&](auto tpr, auto vpt) {
    constexpr int TPR = decltype(tpr)::value, VPT = decltype(vpt)::value;
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(parts), dim3(block_of(TPR)), TPR < 256 ? dim * 4 : 0,
                         stream, (const T*)s, s_stride, (const T*)dy, (const T*)dsum,
                         (const W*)w, rstd, (T*)dx, part, rows, dim);
    };
    dsum ? go(rms_bwd_kernel<T, W, TPR, VPT, true>) : go(rms_bwd_kernel<T, W, TPR, VPT, false>);
    if (VPT == 0 && part)
      hipLaunchKernelGGL(rms_dw_kernel<T>, dim3((dim + 255) / 256, parts), dim3(256), 0, stream,
                         (const T*)s, s_stride, (const T*)dy, rstd, part, rows, dim);
  });
  if (dw)
    hipLaunchKernelGGL((col_sum_kernel<float, W>), dim3((dim + 15) / 16), dim3(1024), 0, stream, part,
                       (W*)dw, parts, dim);
}

template <typename F> void with_types(int type, int wtype, F f) {
  // the weight has 32 bits, or the input's type
  if (type == kTypeF32) f((float*)0, (float*)0);
  else if (type == kTypeBF16) wtype == kTypeF32 ? f((__bf16*)0, (float*)0) : f((__bf16*)0, (__bf16*)0);
  else wtype == kTypeF32 ? f((_Float16*)0, (float*)0) : f((_Float16*)0, (_Float16*)0);
}

}  // namespace

extern "C" void al_rms_fwd(int type, int wtype, const void* x, long x_stride,
                           const void* res, long res_stride, const void* w, void* y,
                           void* total, float* rstd, void* q, void* scale, int out,
                           long rows, int dim, int pitch, int scale_stride, float eps,
                           hipStream_t stream) {
  with_types(type, wtype, [&](auto* t, auto* wt) {
    fwd<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(wt)>>(
        x, x_stride, res, res_stride, w, y, total, rstd, q, scale, out, rows, dim, pitch,
        scale_stride, eps, stream);
  });
}

// how many partial rows of dw the backward pass writes
extern "C" int al_rms_bwd_parts(int type, long rows, int dim) {
  const Shape shape = bwd_shape(type == kTypeF32, dim);
  return blocks_for(shape, rows, shape.tpr == 512 ? 768 : 1024);
}

extern "C" void al_rms_bwd(int type, int wtype, const void* s, long s_stride,
                           const void* dy, const void* dsum, const void* w,
                           const float* rstd, void* dx, float* part, void* dw, int parts,
                           long rows, int dim, hipStream_t stream) {
  with_types(type, wtype, [&](auto* t, auto* wt) {
    bwd<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(wt)>>(
        s, s_stride, dy, dsum, w, rstd, dx, part, dw, parts, rows, dim, stream);
  });
}

extern "C" void al_col_sum(const double* part, void* out, int type, int parts, int dim,
                           hipStream_t stream) {
  const dim3 grid((dim + 15) / 16), block(1024);
  if (type == kTypeF32)
    hipLaunchKernelGGL((col_sum_kernel<double, float>), grid, block, 0, stream, part, (float*)out, parts, dim);
  else if (type == kTypeBF16)
    hipLaunchKernelGGL((col_sum_kernel<double, __bf16>), grid, block, 0, stream, part, (__bf16*)out, parts, dim);
  else
    hipLaunchKernelGGL((col_sum_kernel<double, _Float16>), grid, block, 0, stream, part, (_Float16*)out, parts, dim);
}
