// Fused optimizer updates (fp32 master params).
// SGD: p -= lr * (momentum-buffered (g + wd*p)); one read-modify-write pass
// (reference reaches torch.optim.SGD, arg_pools/default.py:39-40).
// Adam for VAAL's VAE/discriminator (vaal_sampler.py:139-140).

#include "al_fp8.h"

#include <algorithm>

template <bool SHADOW>
__global__ void sgd_kernel(float* __restrict__ p, const float* __restrict__ g,
                           float* __restrict__ buf, float lr, float momentum,
                           float wd, long n, bf16* __restrict__ shadow) {
  for (long i = grid_stride_begin(); i < n; i += grid_stride_step()) {
    float grad = g[i] + wd * p[i];
    if (momentum != 0.f) {
      const float b = buf[i] * momentum + grad;
      buf[i] = b;
      grad = b;
    }
    const float np = p[i] - lr * grad;
    p[i] = np;
    if (SHADOW) shadow[i] = f2bf(np);  // refresh the bf16 weight copy in-pass
  }
}

extern "C" void al_sgd_step(float* p, const float* g, float* buf, float lr,
                            float momentum, float wd, long n, void* shadow,
                            hipStream_t stream) {
  int blocks = (int)min((n + 255) / 256, (long)2048);
  if (shadow)
    hipLaunchKernelGGL((sgd_kernel<true>), dim3(blocks), dim3(256), 0, stream, p, g,
                       buf, lr, momentum, wd, n, (bf16*)shadow);
  else
    hipLaunchKernelGGL((sgd_kernel<false>), dim3(blocks), dim3(256), 0, stream, p, g,
                       buf, lr, momentum, wd, n, nullptr);
}

// ---------------------------------------------------------------------------
// Multi-tensor SGD: ONE launch updates every parameter (the per-tensor
// variant cost 161 launches/step on ResNet-50, profiles/
// r50_b256_step_breakdown_final.md). The host packs a chunk table
// (6 int64 per chunk: p, g, momentum-buf, bf16-shadow pointers + element
// offset + count); each workgroup owns one chunk. Scalar fp32 accesses:
// grads may be element-aligned views into a DDP bucket, so 16-byte vector
// loads are not safe, and the pass is HBM-bound anyway.
struct SgdChunk {
  float* p;
  const float* g;
  float* buf;
  bf16* shadow;
  long off;
  long n;
};

// ZG (persistent-grad mode): zero the gradient in the same pass after
// consuming it — the training step then needs NO zero_grad / grad realloc,
// which keeps gradient storage stable so a hipGraph-captured step contains
// no allocations and the chunk table never rebuilds inside capture.
template <bool ZG>
__global__ void sgd_mt_kernel(const SgdChunk* __restrict__ table, float lr,
                              float momentum, float wd) {
  SgdChunk e = table[blockIdx.x];
  float* p = e.p + e.off;
  float* g = const_cast<float*>(e.g) + e.off;
  float* buf = e.buf ? e.buf + e.off : nullptr;
  bf16* sh = e.shadow ? e.shadow + e.off : nullptr;
  const int n = (int)e.n;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    float grad = g[i] + wd * p[i];
    if (ZG) g[i] = 0.f;
    if (momentum != 0.f) {
      const float b = buf[i] * momentum + grad;
      buf[i] = b;
      grad = b;
    }
    const float np = p[i] - lr * grad;
    p[i] = np;
    if (sh) sh[i] = f2bf(np);
  }
}

extern "C" void al_sgd_step_multi(const void* table, int nchunks, float lr,
                                  float momentum, float wd, int zero_grad,
                                  hipStream_t stream) {
  if (zero_grad)
    hipLaunchKernelGGL((sgd_mt_kernel<true>), dim3(nchunks), dim3(256), 0, stream,
                       (const SgdChunk*)table, lr, momentum, wd);
  else
    hipLaunchKernelGGL((sgd_mt_kernel<false>), dim3(nchunks), dim3(256), 0, stream,
                       (const SgdChunk*)table, lr, momentum, wd);
}

// Variant reading (lr, momentum, wd) from device memory: lets a hipGraph-
// captured training step track the LR schedule — the host updates the
// 3-float hyper buffer between replays instead of re-capturing. A step that was
// captured without momentum has no buffers, whatever the hyper buffer says later:
// the kernels that read it look for both.
template <bool ZG>
__global__ void sgd_mt_kernel_dev(const SgdChunk* __restrict__ table,
                                  const float* __restrict__ hyper) {
  const float lr = hyper[0], momentum = hyper[1], wd = hyper[2];
  SgdChunk e = table[blockIdx.x];
  float* p = e.p + e.off;
  float* g = const_cast<float*>(e.g) + e.off;
  float* buf = e.buf ? e.buf + e.off : nullptr;
  bf16* sh = e.shadow ? e.shadow + e.off : nullptr;
  const int n = (int)e.n;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    float grad = g[i] + wd * p[i];
    if (ZG) g[i] = 0.f;
    if (buf && momentum != 0.f) {
      const float b = buf[i] * momentum + grad;
      buf[i] = b;
      grad = b;
    }
    const float np = p[i] - lr * grad;
    p[i] = np;
    if (sh) sh[i] = f2bf(np);
  }
}

extern "C" void al_sgd_step_multi_dev(const void* table, int nchunks,
                                      const float* hyper, int zero_grad,
                                      hipStream_t stream) {
  if (zero_grad)
    hipLaunchKernelGGL((sgd_mt_kernel_dev<true>), dim3(nchunks), dim3(256), 0,
                       stream, (const SgdChunk*)table, hyper);
  else
    hipLaunchKernelGGL((sgd_mt_kernel_dev<false>), dim3(nchunks), dim3(256), 0,
                       stream, (const SgdChunk*)table, hyper);
}

// ---------------------------------------------------------------------------
// Batched (K,R,S,C) -> (C,R,S,K) bf16 weight transpose: refreshes every
// conv's cached bwd-data permutation in ONE launch right after the fused SGD
// update (the per-conv ATen permute+clone path cost ~53 launches / 0.35 ms
// per step at B=256, tools/fill_audit.py). One workgroup per 64x64 (k, c)
// tile of one rs plane; host enqueues only full tiles (K, C % 64 == 0 —
// the igemm-eligible conv weights). Table row: 4 int64 =
// (src, dst, k0 | c0<<16 | rs<<32, K | C<<16 | RS<<32).
__global__ void wt_refresh_kernel(const long* __restrict__ table) {
  const long* row = table + (long)blockIdx.x * 4;
  const bf16* __restrict__ src = (const bf16*)row[0];
  bf16* __restrict__ dst = (bf16*)row[1];
  const long m1 = row[2], m2 = row[3];
  const int k0 = (int)(m1 & 0xffff), c0 = (int)((m1 >> 16) & 0xffff);
  const int rs = (int)(m1 >> 32);
  const int K = (int)(m2 & 0xffff), C = (int)((m2 >> 16) & 0xffff);
  const int RS = (int)(m2 >> 32);
  __shared__ short tile[64][68];  // 68: de-phase LDS banks across rows
  // load: thread -> (k row = t/4, 16-col strip = (t%4)*16); 2 x 16B per lane
  const int kl = threadIdx.x >> 2, cs = (threadIdx.x & 3) << 4;
  {
    const s16x8* sp =
        (const s16x8*)(src + ((long)(k0 + kl) * RS + rs) * C + c0 + cs);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s16x8 v = sp[u];
#pragma unroll
      for (int j = 0; j < 8; ++j) tile[kl][cs + u * 8 + j] = v[j];
    }
  }
  __syncthreads();
  // store transposed: thread -> (c row = t/4, 16-k strip)
  const int cl = threadIdx.x >> 2, ks = (threadIdx.x & 3) << 4;
  s16x8* dp = (s16x8*)(dst + ((long)(c0 + cl) * RS + rs) * K + k0 + ks);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    s16x8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = tile[ks + u * 8 + j][cl];
    dp[u] = v;
  }
}

extern "C" void al_wt_refresh(const void* table, int nrows, hipStream_t stream) {
  hipLaunchKernelGGL(wt_refresh_kernel, dim3(nrows), dim3(256), 0, stream,
                     (const long*)table);
}

__global__ void adam_kernel(float* __restrict__ p, const float* __restrict__ g,
                            float* __restrict__ m, float* __restrict__ v, float lr,
                            float b1, float b2, float eps, float wd, float bc1,
                            float bc2, long n) {
  for (long i = grid_stride_begin(); i < n; i += grid_stride_step()) {
    const float grad = g[i] + wd * p[i];
    const float mi = m[i] * b1 + (1.f - b1) * grad;
    const float vi = v[i] * b2 + (1.f - b2) * grad * grad;
    m[i] = mi;
    v[i] = vi;
    p[i] -= lr * (mi / bc1) / (sqrtf(vi / bc2) + eps);
  }
}

extern "C" void al_adam_step(float* p, const float* g, float* m, float* v, float lr,
                             float b1, float b2, float eps, float wd, float bc1,
                             float bc2, long n, hipStream_t stream) {
  int blocks = (int)min((n + 255) / 256, (long)2048);
  hipLaunchKernelGGL(adam_kernel, dim3(blocks), dim3(256), 0, stream, p, g, m, v, lr,
                     b1, b2, eps, wd, bc1, bc2, n);
}

// ---------------------------------------------------------------------------
// Norm of all gradients together, and the factor that clips them:
//   norm = sqrt(sum over all tensors of g^2),  factor = min(1, max / (norm + 1e-6))
// The tensors' addresses travel in the kernels' arguments: no table to copy, and
// a captured launch keeps its own (the multi-tensor step below has one). Squares are summed in 64 bits, so that neither
// large nor tiny values leave the range, first by thread, then by block, then
// over the blocks' partial sums, each in a fixed order. Bound by one read of the
// gradients: 301 tensors of 400 million floats together in 286 us, 5.6 TB/s, and as
// bf16 in 148. Four vectors in flight a thread instead of one: 284 and 151.

constexpr int kNormTensors = 160;  // 24 bytes each: the arguments stay under 4 KB
constexpr int kNormChunk = 16384;  // values a block takes at a time

struct NormTensor {
  void* p;
  long n;
  long first;  // its first chunk among the batch's
};
struct NormBatch {
  NormTensor t[kNormTensors];
  long chunks;
  int count;
};

// the values of chunk c: [p, p + n)
template <typename T> AL_DEV T* norm_chunk(const NormBatch& b, long c, int& n) {
  int lo = 0, hi = b.count - 1;  // the last tensor whose first chunk is not after c
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (b.t[mid].first <= c) lo = mid;
    else hi = mid - 1;
  }
  const long off = (c - b.t[lo].first) * kNormChunk, left = b.t[lo].n - off;
  n = (int)(left < kNormChunk ? left : kNormChunk);
  return (T*)b.t[lo].p + off;
}

template <typename T>
__launch_bounds__(256)
__global__ void sq_sum_kernel(NormBatch b, double* __restrict__ part) {
  __shared__ double lds[4];
  double s = 0;
  for (long c = blockIdx.x; c < b.chunks; c += gridDim.x) {
    int n;
    const T* p = norm_chunk<T>(b, c, n);
    int i = threadIdx.x * 8;
    for (; i + 8 <= n; i += 256 * 8) {
      const f32x8 f = load8(p + i);
#pragma unroll
      for (int j = 0; j < 8; ++j) s += (double)f[j] * (double)f[j];
    }
    for (; i < n; ++i) {  // the last, shorter vector: one thread's
      const double v = (float)p[i];
      s += v * v;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = lds[0] + lds[1] + lds[2] + lds[3];
}

// out[0] = norm, out[1] = the clipping factor
__launch_bounds__(256)
__global__ void norm_factor_kernel(const double* __restrict__ part, int parts, float max_norm,
                                   const float* __restrict__ max_dev, float* __restrict__ out) {
  __shared__ double lds[4];
  double s = 0;
  for (int i = threadIdx.x; i < parts; i += 256) s += part[i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    const double norm = sqrt(lds[0] + lds[1] + lds[2] + lds[3]);
    const float bound = max_dev ? *max_dev : max_norm;
    const double f = isinf(bound) ? 1.0 : (double)bound / (norm + 1e-6);  // none: no look at the norm
    out[0] = (float)norm;
    out[1] = f < 1.0 ? (float)f : f >= 1.0 ? 1.f : __builtin_nanf("");
  }
}

// g *= factor in place; nothing is touched where the factor is one
template <typename T>
__launch_bounds__(256)
__global__ void scale_kernel(NormBatch b, const float* __restrict__ norm_factor) {
  const float f = norm_factor[1];
  if (f == 1.f) return;
  for (long c = blockIdx.x; c < b.chunks; c += gridDim.x) {
    int n;
    T* p = norm_chunk<T>(b, c, n);
    int i = threadIdx.x * 8;
    for (; i + 8 <= n; i += 256 * 8) store8(p + i, load8(p + i) * f);
    for (; i < n; ++i) p[i] = (T)((float)p[i] * f);
  }
}

// The multi-tensor SGD step with clipped gradients: the factor is applied as the
// gradient is read, which costs no pass of its own, and p.grad keeps its values.
// Bound by memory: 20 bytes a value with momentum. Norm and step over 301 tensors of
// 400 million floats take 1.87 ms, 24 bytes a value at 5.1 TB/s, while the addresses are
// those of the step before; where one changed the host makes the table anew, 4.2 ms. Four blocks share a
// table row, so that a small network fills the chip.
constexpr int kSgdSub = 4;
template <bool ZG>
__launch_bounds__(256)
__global__ void sgd_mt_clip_kernel(const SgdChunk* __restrict__ table, float lr, float momentum,
                                   float wd, const float* __restrict__ hyper,
                                   const float* __restrict__ norm_factor) {
  if (hyper) { lr = hyper[0]; momentum = hyper[1]; wd = hyper[2]; }
  const float factor = norm_factor[1];
  // from the last row to the first: the norm's pass read the last gradients last,
  // and some of them are still in the cache
  const int at = gridDim.x - 1 - blockIdx.x;
  const SgdChunk e = table[at / kSgdSub];
  const int part = (((int)e.n + kSgdSub - 1) / kSgdSub + 7) & ~7;
  const int begin = part * (at % kSgdSub), end = min(begin + part, (int)e.n);
  float* p = e.p + e.off;
  float* g = const_cast<float*>(e.g) + e.off;
  float* buf = e.buf ? e.buf + e.off : nullptr;
  bf16* sh = e.shadow ? e.shadow + e.off : nullptr;
  for (int i = begin + threadIdx.x * 8; i < end; i += 256 * 8) {
    const int left = end - i;
    f32x8 w = load8_upto(p + i, left);
    f32x8 grad = load8_upto(g + i, left) * factor + wd * w;
    if (ZG) store8_upto(g + i, f32x8{0, 0, 0, 0, 0, 0, 0, 0}, left);
    if (buf && momentum != 0.f) {
      grad = load8_upto(buf + i, left) * momentum + grad;
      store8_upto(buf + i, grad, left);
    }
    w -= lr * grad;
    store8_upto(p + i, w, left);
    if (sh) store8_upto((__bf16*)sh + i, w, left);
  }
}

// The per-tensor updates with a clipping factor, a launch each. Adam reads and writes 28
// bytes a value, the norm 4: 301 tensors of 400 million floats take 3.3 ms, 3.9 TB/s with
// one value a thread at a time; the 62 tensors of a ResNet-18 0.32 ms, which is the calls.
__global__ void sgd_clip_kernel(float* __restrict__ p, const float* __restrict__ g,
                                float* __restrict__ buf, float lr, float momentum, float wd,
                                const float* __restrict__ hyper, long n,
                                bf16* __restrict__ shadow, const float* __restrict__ norm_factor) {
  if (hyper) { lr = hyper[0]; momentum = hyper[1]; wd = hyper[2]; }
  const float factor = norm_factor[1];
  for (long i = grid_stride_begin(); i < n; i += grid_stride_step()) {
    float grad = g[i] * factor + wd * p[i];
    if (buf && momentum != 0.f) {
      grad = buf[i] * momentum + grad;
      buf[i] = grad;
    }
    const float np = p[i] - lr * grad;
    p[i] = np;
    if (shadow) shadow[i] = f2bf(np);
  }
}

__global__ void adam_clip_kernel(float* __restrict__ p, const float* __restrict__ g,
                                 float* __restrict__ m, float* __restrict__ v, float lr,
                                 float b1, float b2, float eps, float wd, float bc1, float bc2,
                                 long n, const float* __restrict__ norm_factor) {
  const float factor = norm_factor[1];
  for (long i = grid_stride_begin(); i < n; i += grid_stride_step()) {
    const float grad = g[i] * factor + wd * p[i];
    const float mi = m[i] * b1 + (1.f - b1) * grad;
    const float vi = v[i] * b2 + (1.f - b2) * grad * grad;
    m[i] = mi;
    v[i] = vi;
    p[i] -= lr * (mi / bc1) / (sqrtf(vi / bc2) + eps);
  }
}

// batch: built by norm_batch_add; part: one double a block
extern "C" int al_norm_batch_bytes() { return (int)sizeof(NormBatch); }
extern "C" void al_norm_batch_clear(void* batch) {
  ((NormBatch*)batch)->chunks = 0;
  ((NormBatch*)batch)->count = 0;
}
// false where the batch is full
extern "C" int al_norm_batch_add(void* batch, void* p, long n) {
  NormBatch* b = (NormBatch*)batch;
  if (b->count == kNormTensors) return 0;
  b->t[b->count++] = NormTensor{p, n, b->chunks};
  b->chunks += (n + kNormChunk - 1) / kNormChunk;
  return 1;
}
extern "C" int al_norm_blocks(const void* batch) {
  return (int)std::min(((const NormBatch*)batch)->chunks, 2048l);
}
extern "C" void al_sq_sum(int type, const void* batch, double* part, hipStream_t stream) {
  const NormBatch& b = *(const NormBatch*)batch;
  const dim3 grid(al_norm_blocks(batch)), block(256);
  if (type == kTypeF32) hipLaunchKernelGGL(sq_sum_kernel<float>, grid, block, 0, stream, b, part);
  else if (type == kTypeBF16) hipLaunchKernelGGL(sq_sum_kernel<__bf16>, grid, block, 0, stream, b, part);
  else hipLaunchKernelGGL(sq_sum_kernel<_Float16>, grid, block, 0, stream, b, part);
}
extern "C" void al_norm_factor(const double* part, int parts, float max_norm, const float* max_dev,
                               float* out, hipStream_t stream) {
  hipLaunchKernelGGL(norm_factor_kernel, dim3(1), dim3(256), 0, stream, part, parts, max_norm,
                     max_dev, out);
}
extern "C" void al_scale_by_factor(int type, const void* batch, const float* norm_factor,
                                   hipStream_t stream) {
  const NormBatch& b = *(const NormBatch*)batch;
  const dim3 grid(al_norm_blocks(batch)), block(256);
  if (type == kTypeF32) hipLaunchKernelGGL(scale_kernel<float>, grid, block, 0, stream, b, norm_factor);
  else if (type == kTypeBF16) hipLaunchKernelGGL(scale_kernel<__bf16>, grid, block, 0, stream, b, norm_factor);
  else hipLaunchKernelGGL(scale_kernel<_Float16>, grid, block, 0, stream, b, norm_factor);
}
extern "C" void al_sgd_step_multi_clip(const void* table, int nchunks, float lr, float momentum,
                                       float wd, const float* hyper, const float* norm_factor,
                                       int zero_grad, hipStream_t stream) {
  const dim3 grid(nchunks * kSgdSub), block(256);
  if (zero_grad)
    hipLaunchKernelGGL((sgd_mt_clip_kernel<true>), grid, block, 0, stream, (const SgdChunk*)table,
                       lr, momentum, wd, hyper, norm_factor);
  else
    hipLaunchKernelGGL((sgd_mt_clip_kernel<false>), grid, block, 0, stream, (const SgdChunk*)table,
                       lr, momentum, wd, hyper, norm_factor);
}
extern "C" void al_sgd_step_clip(float* p, const float* g, float* buf, float lr, float momentum,
                                 float wd, const float* hyper, long n, void* shadow,
                                 const float* norm_factor, hipStream_t stream) {
  const int blocks = (int)std::min((n + 255) / 256, 2048l);
  hipLaunchKernelGGL(sgd_clip_kernel, dim3(blocks), dim3(256), 0, stream, p, g, buf, lr, momentum,
                     wd, hyper, n, (bf16*)shadow, norm_factor);
}
extern "C" void al_adam_step_clip(float* p, const float* g, float* m, float* v, float lr, float b1,
                                  float b2, float eps, float wd, float bc1, float bc2, long n,
                                  const float* norm_factor, hipStream_t stream) {
  const int blocks = (int)std::min((n + 255) / 256, 2048l);
  hipLaunchKernelGGL(adam_clip_kernel, dim3(blocks), dim3(256), 0, stream, p, g, m, v, lr, b1, b2,
                     eps, wd, bc1, bc2, n, norm_factor);
}
