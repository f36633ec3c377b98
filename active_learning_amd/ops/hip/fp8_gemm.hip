// Matrix products of e4m3 blocks, with a scale for each block of 128 (layout in
// al_fp8.h).
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

#include <algorithm>

namespace {

struct Gemm {
  const unsigned char *a, *b;
  const void *sa, *sb;        // scales: a by row and block, b by row (or tile) and block
  long lda, ldb;              // bytes from row to row, 128 for each block
  int sa_stride, sb_stride;   // scales from row to row
  int m, n, blocks;           // blocks: of 128 along the contraction
  const void* bias;
  int bias_type;
  void* out;
  int out_type;
  int ldo;                    // values from row to row of the result
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

AL_DEV void store_four(void* p, int type, long at, f32x4 v, int left) {
  if (left >= 4) {
    if (type == kTypeF32) __builtin_memcpy((float*)p + at, &v, 16);
    else if (type == kTypeBF16) {
      const bf16x4v r = __builtin_convertvector(v, bf16x4v);
      __builtin_memcpy((__bf16*)p + at, &r, 8);
    } else {
      const f16x4v r = __builtin_convertvector(v, f16x4v);
      __builtin_memcpy((_Float16*)p + at, &r, 8);
    }
    return;
  }
  for (int e = 0; e < left; ++e) store_out(p, type, at + e, v[e]);
}

// eight codes times a power of two as bf16, which holds them exactly
AL_DEV bf16x8v to_bf16(int lo, int hi, float scale) {
  const bf16x2v a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const bf16x2v b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2v c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const bf16x2v d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8v{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Both scales of a block, multiplied with each other, leave the range of a float where the
// result does not (operands around 1e-19: 2^-140 times sums around 2^17). So the left one
// is a power of two, which the matrix instruction or the conversion in front of it
// applies, times a factor of 1 to 2, and only the factor is multiplied with the right one.
// Powers are 2^-60 to 2^103: a block's sum, of 2^-18 to 2^25 where it is not zero, stays
// normal, and where the factor takes over beyond them its product leaves the range only
// with a result that does.
struct Scale {
  unsigned code;  // of the power of two, 2^(code - 127)
  float factor;
};
AL_DEV Scale split(float scale) {
  const int e = (int)(__float_as_uint(scale) >> 23 & 255u);
  const int code = e < 127 - 60 ? 127 - 60 : e > 127 + 103 ? 127 + 103 : e;
  return {(unsigned)code, __builtin_ldexpf(scale, 127 - code)};
}
template <int KIND> AL_DEV float scale_value(unsigned code) {
  return __uint_as_float(KIND == kF32 ? code : code == 255u ? 0x7fc00000u : code ? code << 23 : 0x400000u);
}

constexpr int kOne = 127;  // the power 2^0

// one block's 16x16 products times y's power of two; EXACT: in bf16 instructions
template <bool EXACT> AL_DEV f32x4 block_product(i32x8 x, i32x8 y, unsigned power) {
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  if (!EXACT) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, zero, 0, 0, 0, kOne, 0, (int)power);
  const float by = __uint_as_float(power << 23);
  f32x4 d = zero;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16(x[2 * i], x[2 * i + 1], 1.f),
                                                to_bf16(y[2 * i], y[2 * i + 1], by), d, 0, 0, 0);
  return d;
}

template <int KIND> AL_DEV unsigned scale_code(const void* p, long at) {
  return KIND == kF32 ? ((const unsigned*)p)[at] : ((const unsigned char*)p)[at];
}

// --------------------------------------------------------------------------
// few outputs: (16 MT) x (16 NT) a workgroup, straight from memory
// --------------------------------------------------------------------------
//
// Each wave takes every WAVES-th block of the contraction, with fragments read
// into registers a block ahead, so that no wave waits for another; the waves'
// sums meet in LDS and are joined in order. With T a float type a's rows come as
// values, at most 16 of them, and each wave quantises the blocks that it reads:
// a launch less, and b's bytes are what it costs. With T unsigned char they come
// as codes.
//
// 1x1000x2048 with values takes 5.1 us, a launch; 16x8192x8192 21 us for 67 MB of b, which a
// copy moves in 12.5, and 16x16384x8192 31.5 us (24.9): each unit takes 25 KB a microsecond of
// x and b together, with 16 waves (21), three blocks in flight a wave (24) and blocks in an
// order of each workgroup's own (22) too.
template <typename T, bool EXACT, int KIND, bool BTILE, int MT, int NT, int WAVES>
__launch_bounds__(WAVES * 64)
__global__ void direct_kernel(const T* __restrict__ x, long x_stride, int dim, Gemm g, int across) {
  constexpr bool VALUES = !std::is_same<T, unsigned char>::value;
  constexpr bool HW = KIND == kE8M0 && !EXACT;  // the matrix instruction applies the scales
  static_assert(!VALUES || MT == 1, "values: one tile of rows");
  __shared__ f32x4 lds[WAVES][MT * NT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l15 = lane & 15, l4 = lane >> 4;
  const int n0 = blockIdx.x % across * (16 * NT), m0 = blockIdx.x / across * (16 * MT);

  // rows behind the last are the last one again; their outputs are not stored
  const unsigned char *a[MT], *b[NT];
  long sa[MT], sb[NT];  // where the first block's scales are
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const long m = min(m0 + i * 16 + l15, g.m - 1);
    a[i] = VALUES ? (const unsigned char*)(x + m * x_stride + l4 * 16) : g.a + m * g.lda + l4 * 16;
    sa[i] = m * g.sa_stride;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int n = min(n0 + j * 16 + l15, g.n - 1);
    b[j] = g.b + (long)n * g.ldb + l4 * 16;
    sb[j] = (long)(BTILE ? n / kQB : n) * g.sb_stride;
  }
  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  struct Raw {
    i32x8 a[VALUES ? 1 : MT], b[NT];
    typename Raw8<typename std::conditional<VALUES, T, float>::type>::V v[VALUES ? 4 : 1];
    unsigned sa[MT], sb[NT];
  };
  // A lane has 16 values of each half of the block, so that a load takes 64
  // neighbouring bytes of a row: the order within a block is the same on both sides
  // and means nothing to the sum.
  auto load32 = [](const unsigned char* p) {
    const i32x4 lo = *(const i32x4*)p, hi = *(const i32x4*)(p + 64);
    return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  auto place = [](int i) { return (i >> 1) * 64 + (i & 1) * 8; };  // of a lane's i-th eight
  auto load = [&](Raw& r, int kb) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      r.b[j] = load32(b[j] + (long)kb * kQB);
      r.sb[j] = scale_code<KIND>(g.sb, sb[j] + kb);
    }
    if (VALUES) {
      const int left = dim - kb * kQB - l4 * 16;
      const T* p = (const T*)a[0] + (long)kb * kQB;
      if constexpr (VALUES) {
        if ((kb + 1) * kQB <= dim) {
#pragma unroll
          for (int i = 0; i < 4; ++i) r.v[i] = raw8(p + place(i));
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) r.v[i] = raw8_upto(p + place(i), left - place(i));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        r.a[VALUES ? 0 : i] = load32(a[i] + (long)kb * kQB);
        r.sa[i] = scale_code<KIND>(g.sa, sa[i] + kb);
      }
    }
  };
  auto compute = [&](Raw& r, int kb) {
    if constexpr (VALUES) {
      Top<T> most;
#pragma unroll
      for (int i = 0; i < 4; ++i) most.add(r.v[i]);
      unsigned top = most.bits();
      top = max(top, (unsigned)__shfl_xor((int)top, 16, 64));
      top = max(top, (unsigned)__shfl_xor((int)top, 32, 64));
      const BlockScale s = block_scale<KIND>(top);
      r.sa[0] = s.code;
      const int left = dim - kb * kQB - l4 * 16;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const i32x2 codes = keep_upto(raw_to_fp8<T, KIND>(r.v[i], s), left - place(i));
        r.a[0][2 * i] = codes[0];
        r.a[0][2 * i + 1] = codes[1];
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      f32x4 by;
      if (!HW) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          by[e] = scale_value<KIND>(BTILE ? r.sb[j] : (unsigned)__shfl((int)r.sb[j], l4 * 4 + e, 64));
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const i32x8 fa = r.a[VALUES ? 0 : i];
        if (HW) {
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(r.b[j], fa, acc[i][j], 0, 0, 0,
                                                                      (int)r.sb[j], 0, (int)r.sa[i]);
        } else {
          const Scale s = split(scale_value<KIND>(r.sa[i]));
          const f32x4 d = block_product<EXACT>(r.b[j], fa, s.code);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[e], s.factor * by[e], acc[i][j][e]);
        }
      }
    }
  };
  Raw r[2];
  if (wave < g.blocks) load(r[0], wave);
  for (int kb = wave; kb < g.blocks; kb += 2 * WAVES) {
    if (kb + WAVES < g.blocks) load(r[1], kb + WAVES);
    compute(r[0], kb);
    if (kb + WAVES >= g.blocks) break;
    if (kb + 2 * WAVES < g.blocks) load(r[0], kb + 2 * WAVES);
    compute(r[1], kb + WAVES);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) lds[wave][i * NT + j][lane] = acc[i][j];
  __syncthreads();
#pragma unroll
  for (int f = 0; f < MT * NT; f += WAVES) {
    if (f + wave >= MT * NT) break;
    const int i = (f + wave) / NT, j = (f + wave) % NT;
    f32x4 v = lds[0][f + wave][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v += lds[w][f + wave][lane];
    const int m = m0 + i * 16 + l15;
    if (m >= g.m) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = n0 + j * 16 + l4 * 4 + e;
      if (n < g.n)
        store_out(g.out, g.out_type, (long)m * g.ldo + n,
                  v[e] + (g.bias ? bias_at(g.bias, g.bias_type, n) : 0.f));
    }
  }
}

// --------------------------------------------------------------------------
// 256x256 outputs a workgroup
// --------------------------------------------------------------------------
//
// Eight waves, two on each SIMD, in two groups that run half a phase apart: while
// one group's matrix instructions run, the other reads its fragments from LDS and
// asks for tiles to come. A step is one block of 128 (64 KB of operands) and has
// two phases, one for each half of a's rows. All rows go straight to LDS (no
// registers): a's 128-row halves through a ring of five, b's tiles through a ring
// of two, scales through a ring of two that hold four steps each; what a phase
// asks for is used six or seven phases later. A wave computes 2 x 64 rows by 64
// columns in 32x32 tiles; b's rows are the first operand, so that a lane holds
// neighbouring columns of one output row.
//
// With e8m0 scales the matrix instruction applies them, or, in the EXACT form (bf16
// instructions), the conversion to bf16. 32-bit scales multiply each block's sum as
// it is added to the total, but for the left one's power of two.
//
// 8192x8192x8192: e8m0 384 to 407 us, 2.7 to 2.86 PFLOP/s, the matrix cores busy in 79% of
// the cycles and the clock at 1.66 GHz, which power leaves; 32-bit scales 484 to 501 us, where
// the scaling takes as many vector cycles as the products take matrix cycles (780 where the
// right one's scales differ from row to row and come from LDS for each value); EXACT 751 us,
// 1.46 PFLOP/s. LDS conflicts: 1 cycle in 150.

constexpr int kHalf = 128 * 128;       // bytes of half a tile: 128 rows of a block
constexpr int kRingB = 5 * kHalf;      // where b's ring begins
constexpr int kRingS = kRingB + 4 * kHalf;  // where the scales' ring begins

typedef __amdgpu_buffer_rsrc_t Rsrc;
// a buffer that ends where the operand's rows do: what lies behind reads as zero
AL_DEV Rsrc rsrc_of(const void* p, long bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)(unsigned)min(bytes, 0xffffffffl), 0x00020000);
}
template <int BYTES> AL_DEV void lds_load(Rsrc from, unsigned off, int step, unsigned char* to) {
  typedef __attribute__((address_space(3))) void* Lds;
  static_assert(BYTES == 4 || BYTES == 16, "one or four words a lane");
  if (BYTES == 16) __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (Lds)to, 16, off, step, 0, 0);
  else __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (Lds)to, 4, off, step, 0, 0);
}

// all but the COUNT newest of this wave's loads are done, and all its LDS reads
template <int COUNT> AL_DEV void wait_but() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(COUNT) : "memory");
}
AL_DEV void phase_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

// the workgroup's tile: neighbouring workgroups run on different XCDs, so each XCD
// is given a run of tiles of its own, in patches eight tiles high that share its L2
AL_DEV void tile_of(int id, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int count = tiles_m * tiles_n, per = count / 8, extra = count % 8;
  const int xcd = id & 7, at = id >> 3;
  id = xcd * per + min(xcd, extra) + at;
  const int group = 8 * tiles_n, first = id / group * 8, high = min(8, tiles_m - first);
  tm = first + id % group % high;
  tn = id % group / high;
}

template <int KIND, bool EXACT, bool BTILE>
__launch_bounds__(512, 2)
__global__ void gemm256_kernel(Gemm g, int tiles_m, int tiles_n) {
  static_assert(KIND == kE8M0 || !EXACT, "32-bit scales and results: the direct kernel");
  constexpr bool HW = KIND == kE8M0 && !EXACT;
  constexpr int SB = KIND == kE8M0 ? 4 : 16;  // bytes of four steps' scales
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wid >> 2, wc = wid & 3, l31 = lane & 31, l5 = lane >> 5;
  int tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
  const int m0 = tm * 256, n0 = tn * 256;

  const int steps = g.blocks;

  // A wave's load brings 8 rows of 128 bytes; the chunk that lands at slot s of row
  // r is s ^ (r >> 1 & 7). A read of 16 bytes a lane takes 16 lanes at a time, of
  // rows 0-3, 12-15, 20-23 and 24-27 first: this way they fall on different banks.
  const int rows_a = min(256, g.m - m0), rows_b = min(256, g.n - n0);
  const Rsrc a = rsrc_of(g.a + (long)m0 * g.lda, (long)rows_a * g.lda);
  const Rsrc b = rsrc_of(g.b + (long)n0 * g.ldb, (long)rows_b * g.ldb);
  // Rows behind the operand's last are the last one again, and no output of theirs is
  // stored.
  const int r = wid * 8 + (lane >> 3);  // and 64 rows on, and on
  const unsigned chunk = ((lane & 7) ^ (r >> 1 & 7)) * 16;
  const unsigned off_a = (unsigned)r * (unsigned)g.lda, off_b = (unsigned)r * (unsigned)g.ldb;
  const unsigned step_a = 64 * (unsigned)g.lda, step_b = 64 * (unsigned)g.ldb;
  const unsigned last_a = (unsigned)(rows_a - 1) * (unsigned)g.lda, last_b = (unsigned)(rows_b - 1) * (unsigned)g.ldb;
  // scales: the first four waves bring those of a's rows, the others those of b's
  const int sr = (wid & 3) * 64 + lane;
  const int scale_row = wid < 4 ? g.sa_stride * (SB / 4) : g.sb_stride * (SB / 4);  // bytes
  const int scale_rows = wid < 4 ? rows_a : BTILE ? (rows_b + kQB - 1) / kQB : rows_b;
  const Rsrc scale = rsrc_of(
      (const unsigned char*)(wid < 4 ? g.sa : g.sb) +
          (long)(wid < 4 ? m0 : BTILE ? n0 / kQB : n0) * scale_row,
      (long)scale_rows * scale_row);
  const unsigned off_s =
      (unsigned)min(BTILE && wid >= 4 ? sr / kQB : sr, scale_rows - 1) * (unsigned)scale_row;

  // what lies behind the last step is asked for at the last one: every wave has
  // the same loads in flight in every step
  const int last = steps - 1;
  auto load_a = [&](int k, int h, int ring) __attribute__((always_inline)) {
    unsigned char* to = smem + ring + wid * 1024;
    lds_load<16>(a, min(off_a + 2 * h * step_a, last_a) + chunk, min(k, last) * kQB, to);
    lds_load<16>(a, min(off_a + (2 * h + 1) * step_a, last_a) + chunk, min(k, last) * kQB, to + 8192);
  };
  auto load_b = [&](int k) __attribute__((always_inline)) {
    unsigned char* to = smem + kRingB + (k & 1) * 2 * kHalf + wid * 1024;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      lds_load<16>(b, min(off_b + i * step_b, last_b) + chunk, min(k, last) * kQB, to + i * 8192);
  };
  auto load_scales = [&](int word) __attribute__((always_inline)) {
    lds_load<SB>(scale, off_s, min(word, last >> 2) * SB, smem + kRingS + ((word & 1) * 512 + wid * 64) * SB);
  };

  f32x16 acc[2][2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[h][i][j][r] = 0.f;

  // A lane's row has four 16-byte chunks, two for each half of the block; the other
  // three lie where bits 4 and 6 of the first one's address are turned over. Where
  // registers are short these addresses are computed again for each use.
  auto this_lane = [&]() __attribute__((always_inline)) {
    if (HW) return lane;
    int l = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    asm volatile("" : "+v"(l));
    return l;
  };
  auto first_chunk = [&](int l) __attribute__((always_inline)) {
    return (l & 31) * 128 + (((l >> 5) * 2 ^ (l >> 1 & 7)) << 4);
  };
  auto fragment = [&](unsigned first, int half) __attribute__((always_inline)) {
    typedef const __attribute__((address_space(3))) i32x4* Chunk;
    const i32x4 lo = *(Chunk)(first ^ (half * 64)), hi = *(Chunk)(first ^ (half * 64 + 16));
    return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  const unsigned lds = (unsigned)(unsigned long)(__attribute__((address_space(3))) unsigned char*)smem;

  i32x8 fa[2][2], fb[2][2];
  int sa[2], sb[2];  // e8m0: this step's scales, in the lowest byte; else a's powers and b's bits
  float ga[2];       // 32-bit scales: a's factors
  // where the scales of step k (the s-th of its four) are
  auto scale_of = [&](int row, int k, int s) __attribute__((always_inline)) {
    const unsigned char* p = smem + kRingS + ((k >> 2 & 1) * 512 + row) * SB;
    return KIND == kF32 ? ((const int*)p)[s] : (int)(*(const unsigned*)p >> (8 * s));
  };
  auto read_a = [&](int k, int s, int h, int ring) __attribute__((always_inline)) {
    const int l = this_lane(), l31 = l & 31;
    const unsigned p = lds + ring + wr * 64 * 128 + first_chunk(l);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      fa[i][0] = fragment(p + i * 32 * 128, 0);
      fa[i][1] = fragment(p + i * 32 * 128, 1);
      sa[i] = scale_of(h * 128 + wr * 64 + i * 32 + l31, k, s);
      if (KIND == kF32) {
        const Scale x = split(__int_as_float(sa[i]));
        sa[i] = (int)x.code;
        ga[i] = x.factor;
      }
    }
  };
  auto read_b = [&](int k, int s) __attribute__((always_inline)) {
    const int l = this_lane(), l31 = l & 31;
    const unsigned p = lds + kRingB + (k & 1) * 2 * kHalf + wc * 64 * 128 + first_chunk(l);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      fb[j][0] = fragment(p + j * 32 * 128, 0);
      fb[j][1] = fragment(p + j * 32 * 128, 1);
      if (KIND == kE8M0 || BTILE) sb[j] = scale_of(256 + wc * 64 + j * 32 + l31, k, s);
    }
  };
  auto multiply = [&](int k, int s, f32x16 (&c)[2][2]) __attribute__((always_inline)) {
    __builtin_amdgcn_s_setprio(1);
    if (HW) {
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            c[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                fb[j][half], fa[i][half], c[i][j], 0, 0, 0, sb[j], 0, sa[i]);
    } else if (KIND == kE8M0) {
      // the values themselves, which bf16 holds exactly
      const float ua = __int_as_float(sa[0] << 23), va = __int_as_float(sa[1] << 23);
      const float ub = __int_as_float(sb[0] << 23), vb = __int_as_float(sb[1] << 23);
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int q = 0; q < 8; q += 2) {
          const bf16x8v x0 = to_bf16(fa[0][half][q], fa[0][half][q + 1], ua);
          const bf16x8v x1 = to_bf16(fa[1][half][q], fa[1][half][q + 1], va);
          const bf16x8v y0 = to_bf16(fb[0][half][q], fb[0][half][q + 1], ub);
          const bf16x8v y1 = to_bf16(fb[1][half][q], fb[1][half][q + 1], vb);
          c[0][0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y0, x0, c[0][0], 0, 0, 0);
          c[0][1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y1, x0, c[0][1], 0, 0, 0);
          c[1][0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y0, x1, c[1][0], 0, 0, 0);
          c[1][1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y1, x1, c[1][1], 0, 0, 0);
        }
    } else {
      // three tiles' products ahead of their scaling, as many as registers hold: one ahead
      // takes 12 us more of 8192x8192x8192
      f32x16 d[3];
      auto start = [&](f32x16& d, int t) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) d[r] = 0.f;
#pragma unroll
        for (int half = 0; half < 2; ++half)
          d = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[t >> 1][half], fa[t & 1][half], d, 0, 0, 0,
                                                              kOne, 0, sa[t & 1]);
      };
      auto add = [&](f32x16& d, int t) __attribute__((always_inline)) {
        const int i = t & 1, j = t >> 1;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int by = BTILE ? sb[j] : scale_of(256 + wc * 64 + j * 32 + (r >> 2) * 8 + l5 * 4 + (r & 3), k, s);
          c[i][j][r] = fmaf(d[r], ga[i] * __int_as_float(by), c[i][j][r]);
        }
      };
      start(d[0], 0);
      start(d[1], 1);
      start(d[2], 2);
      __builtin_amdgcn_sched_barrier(0);
      add(d[0], 0);
      start(d[0], 3);
      __builtin_amdgcn_sched_barrier(0);
      add(d[1], 1);
      add(d[2], 2);
      add(d[0], 3);
    }
    __builtin_amdgcn_s_setprio(0);
  };

  load_scales(0);
  load_a(0, 0, 0);
  load_a(0, 1, kHalf);
  load_b(0);
  load_a(1, 0, 2 * kHalf);
  load_a(1, 1, 3 * kHalf);
  load_b(1);
  asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
  phase_barrier();
  if (wr) phase_barrier();
  int read = 0, write = 4 * kHalf;  // places in a's ring
  auto next = [](int at) { return at == 4 * kHalf ? 0 : at + kHalf; };
  // The s-th of four steps, without a branch between its parts: the compiler would
  // move matrix instructions over it.
  auto one_step = [&](auto s_, int k) __attribute__((always_inline)) {
    constexpr int s = decltype(s_)::value;
    read_b(k, s);
    read_a(k, s, 0, read);
    load_a(k + 2, 0, write);
    // not before the second group's last phase of the words' last user is over
    if (s == 1) load_scales((k >> 2) + 1);
    wait_but<63>();
    phase_barrier();
    multiply(k, s, acc[0]);
    phase_barrier();
    read = next(read);
    write = next(write);
    read_a(k, s, 1, read);
    load_a(k + 2, 1, write);
    load_b(k + 2);
    // The next step's tiles are there, in every wave's part: newer are the loads of
    // the step after it.
    wait_but<s == 1 ? 9 : 8>();
    phase_barrier();
    multiply(k, s, acc[1]);
    phase_barrier();
    read = next(read);
    write = next(write);
  };
  int k = 0;
  for (; k + 4 <= steps; k += 4) {
    one_step(std::integral_constant<int, 0>{}, k);
    one_step(std::integral_constant<int, 1>{}, k + 1);
    one_step(std::integral_constant<int, 2>{}, k + 2);
    one_step(std::integral_constant<int, 3>{}, k + 3);
  }
  if (k < steps) {
    one_step(std::integral_constant<int, 0>{}, k);
    if (k + 1 < steps) {
      one_step(std::integral_constant<int, 1>{}, k + 1);
      if (k + 2 < steps) one_step(std::integral_constant<int, 2>{}, k + 2);
    }
  }
  if (!wr) phase_barrier();
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  phase_barrier();

  // computed anew: kept until here they would take registers from the loop
  int own = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
  asm volatile("" : "+v"(own));
  const int e31 = own & 31, e5 = own >> 5, thread = wid * 64 + own;

  // Through LDS, so that rows are written in whole lines; 16-byte chunks again
  // spread over the banks by their row.
  float* bias = (float*)(smem + kRingS);  // the scales' place: 256 floats
  if (thread < 256)
    bias[thread] = g.bias && n0 + thread < g.n
                            ? bias_at(g.bias, g.bias_type, n0 + thread) : 0.f;
  __syncthreads();
  auto each_four = [&](int h, auto put) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = wc * 64 + j * 32 + q * 8 + e5 * 4;
        const f32x4 add = *(const f32x4*)(bias + n);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          f32x4 v;
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = acc[h][i][j][q * 4 + r] + add[r];
          put(h * 128 + wr * 64 + i * 32 + e31, n, v);
        }
      }
  };
  if (!EXACT) {
    const bool halves = g.out_type == kTypeF16;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      each_four(h, [&](int m, int n, f32x4 v) {
        *(s16x4*)(smem + m * 512 + (((n >> 3) ^ e31) << 4) + (n & 4) * 2) =
            halves ? __builtin_bit_cast(s16x4, __builtin_convertvector(v, f16x4v))
                   : __builtin_bit_cast(s16x4, __builtin_convertvector(v, bf16x4v));
      });
    __syncthreads();
    const int c = thread & 31, left = g.n - n0 - c * 8;
    const int high = left > 0 ? min(256, g.m - m0) : 0;
    short* out = (short*)g.out + (long)m0 * g.ldo + n0 + c * 8;
    for (int m = thread >> 5; m < high; m += 16) {
      const s16x8 v = *(const s16x8*)(smem + m * 512 + ((c ^ (m & 31)) << 4));
      short* to = out + (long)m * g.ldo;
      if (left >= 8) __builtin_memcpy(to, &v, 16);
      else
        for (int r = 0; r < left; ++r) to[r] = *(const short*)(smem + m * 512 + ((c ^ (m & 31)) << 4) + r * 2);
    }
    return;
  }
  float* out = (float*)g.out + (long)m0 * g.ldo + n0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (h) __syncthreads();
    each_four(h, [&](int m, int n, f32x4 v) {
      *(f32x4*)(smem + (m & 127) * 1024 + (((n >> 2) ^ e31) << 4)) = v;
    });
    __syncthreads();
    const int c = thread & 63, left = g.n - n0 - c * 4;
    const int high = left > 0 ? min(128, g.m - m0 - h * 128) : 0;
    for (int m = thread >> 6; m < high; m += 8) {
      const float* from = (const float*)(smem + m * 1024 + ((c ^ (m & 31)) << 4));
      float* to = out + (long)(h * 128 + m) * g.ldo + c * 4;
      if (left >= 4) __builtin_memcpy(to, from, 16);
      else
        for (int r = 0; r < left; ++r) to[r] = from[r];
    }
  }
}

// --------------------------------------------------------------------------
// 64x64 and 128x128 outputs a workgroup
// --------------------------------------------------------------------------
//
// Between the two others: waves of WM x WN parts of a TM x TN tile share operands
// through a ring of STAGES steps in LDS. Loads run STAGES - 1 steps ahead and one
// barrier a step serves both ends of the ring: whoever passes it has its part of
// this step's loads there and is done with the last step, whose place is then asked
// for anew. The order of the 16-byte chunks within a block is the same on both
// sides: a lane has chunks l4 and l4 + 4 of its row.
//
// 2048x2048x8192 takes 44 us, and for 32-bit results 72; 4096x2048x8192 for 32-bit results
// 117 (a bf16 product at the library's rate: 97). There the matrix cores are busy in 44% of
// the cycles and the vector units, which convert, in 35%: waves that meet at a barrier each
// step do both at the same times. Fragments read a step ahead, 16 waves of 32x64 and four
// of 64x128 took 119, 128 and 141 us.
// Two stages fit twice: no more registers than let both workgroups run (130 instead of 128
// with 32-bit scales by row: 8192x1000x2048 34.6 us, 30.1 this way).
template <int KIND, bool EXACT, bool BTILE, int TM, int TN, int WM, int WN, int STAGES>
__launch_bounds__(WM * WN * 64, STAGES == 2 ? 4 : 1)
__global__ void gemm_mid_kernel(Gemm g, int tiles_m, int tiles_n) {
  constexpr bool HW = KIND == kE8M0 && !EXACT;
  constexpr int WAVES = WM * WN, MT = TM / WM / 16, NT = TN / WN / 16;
  constexpr int LA = TM / 8 / WAVES, LB = TN / 8 / WAVES, SCALES = (TM + TN) / 64;
  constexpr int LOADS = LA + LB + 1;  // of a wave in a step
  constexpr int STAGE = (TM + TN) * (kQB + 4);
  static_assert(LA * 8 * WAVES == TM && LB * 8 * WAVES == TN && SCALES <= WAVES, "whole loads");
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l15 = lane & 15, l4 = lane >> 4;
  int tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
  const int m0 = tm * TM, n0 = tn * TN;
  const int first = (int)((long)g.blocks * blockIdx.y / g.splits);
  const int steps = (int)((long)g.blocks * (blockIdx.y + 1) / g.splits) - first;

  // Rows behind the operand's last are the last one again, and no output of theirs is
  // stored. The chunk that lands at slot s of row r is s ^ (r & 7).
  const int rows_a = min(TM, g.m - m0), rows_b = min(TN, g.n - n0);
  const Rsrc a = rsrc_of(g.a + (long)m0 * g.lda + (long)first * kQB, (long)rows_a * g.lda - (long)first * kQB);
  const Rsrc b = rsrc_of(g.b + (long)n0 * g.ldb + (long)first * kQB, (long)rows_b * g.ldb - (long)first * kQB);
  const int r8 = lane >> 3;
  const unsigned chunk = ((lane & 7) ^ r8) * 16;
  unsigned off_a[LA], off_b[LB];
#pragma unroll
  for (int i = 0; i < LA; ++i)
    off_a[i] = (unsigned)min((i * WAVES + wid) * 8 + r8, rows_a - 1) * (unsigned)g.lda + chunk;
#pragma unroll
  for (int i = 0; i < LB; ++i)
    off_b[i] = (unsigned)min((i * WAVES + wid) * 8 + r8, rows_b - 1) * (unsigned)g.ldb + chunk;
  // Each wave brings 64 rows' scales, some of them as another wave does too: all have
  // the same loads in flight. e8m0: the word that holds the step's byte.
  const int part = wid % SCALES;
  const bool of_a = part * 64 < TM;
  const int row = part * 64 + lane - (of_a ? 0 : TM);
  const unsigned char* scale =
      (const unsigned char*)(of_a ? g.sa : g.sb) +
      (KIND == kE8M0 ? 1l : 4l) *
          (of_a ? (long)min(m0 + row, g.m - 1) * g.sa_stride
                : (long)(BTILE ? min(n0 + row, g.n - 1) / kQB : min(n0 + row, g.n - 1)) * g.sb_stride);
  const int last = steps - 1;
  auto load = [&](int k) __attribute__((always_inline)) {
    unsigned char* to = smem + k % STAGES * STAGE;
    const int at = min(k, last);  // behind the last step it again
#pragma unroll
    for (int i = 0; i < LA; ++i) lds_load<16>(a, off_a[i], at * kQB, to + (i * WAVES + wid) * 1024);
#pragma unroll
    for (int i = 0; i < LB; ++i) lds_load<16>(b, off_b[i], at * kQB, to + TM * kQB + (i * WAVES + wid) * 1024);
    const unsigned char* p = scale + (KIND == kE8M0 ? (first + at) & ~3 : (first + at) * 4);
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p,
                                     (__attribute__((address_space(3))) void*)(to + (TM + TN) * kQB + part * 256), 4,
                                     0, 0);
  };

  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int wm = wid / WN * (TM / WM), wn = wid % WN * (TN / WN);
  const unsigned char* own = smem + l15 * kQB + ((l4 ^ (l15 & 7)) << 4);
#pragma unroll
  for (int k = 0; k < STAGES - 1; ++k) load(k);
  for (int k = 0; k < steps; ++k) {
    wait_but<LOADS * (STAGES - 2)>();
    phase_barrier();
    load(k + STAGES - 1);
    const int place = k % STAGES * STAGE;
    auto fragment = [&](int r) __attribute__((always_inline)) {
      const unsigned char* p = own + place + r * kQB;
      // chunk l4 + 4 lies where bit 6 is turned over
      const i32x4 lo = *(const i32x4*)p, hi = *(const i32x4*)(smem + ((unsigned)(p - smem) ^ 64u));
      return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    auto scale_of = [&](int r) __attribute__((always_inline)) {
      const unsigned w = *(const unsigned*)(smem + place + (TM + TN) * kQB + r * 4);
      return KIND == kE8M0 ? w >> (((first + k) & 3) * 8) & 255u : w;
    };
    i32x8 fa[MT], fb[NT];
    unsigned sa[MT];
    float xa[MT];  // 32-bit scales: the factors beside the powers
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      fa[i] = fragment(wm + i * 16);
      sa[i] = scale_of(wm + i * 16 + l15);
      if (KIND == kF32) {
        const Scale s = split(__uint_as_float(sa[i]));
        sa[i] = s.code;
        xa[i] = s.factor;
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) fb[j] = fragment(TM + wn + j * 16);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      if (KIND == kE8M0) {
        const unsigned sb = scale_of(TM + wn + j * 16 + l15);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          if (HW) {
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], fa[i], acc[i][j], 0, 0, 0, (int)sb, 0,
                                                                        (int)sa[i]);
          } else {
            const float x = __uint_as_float(sa[i] << 23), y = __uint_as_float(sb << 23);
#pragma unroll
            for (int q = 0; q < 8; q += 2)
              acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16(fb[j][q], fb[j][q + 1], y),
                                                                  to_bf16(fa[i][q], fa[i][q + 1], x), acc[i][j], 0, 0, 0);
          }
        }
      } else {
        f32x4 by;
#pragma unroll
        for (int e = 0; e < 4; ++e) by[e] = __uint_as_float(scale_of(TM + wn + j * 16 + (BTILE ? 0 : l4 * 4 + e)));
        f32x4 d[MT];  // all before the first is used: 2500x2500x8192 80 us, one by one 4 more
#pragma unroll
        for (int i = 0; i < MT; ++i) d[i] = block_product<EXACT>(fb[j], fa[i], sa[i]);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[i][e], xa[i] * by[e], acc[i][j][e]);
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing lands in LDS after the end
  const bool split = g.splits > 1;
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = m0 + wm + i * 16 + l15;
    if (m >= g.m) continue;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int n = n0 + wn + j * 16 + l4 * 4;
      f32x4 v = acc[i][j];
      if (split) {
        float* to = g.split_out + ((long)blockIdx.y * g.m + m) * g.n + n;
        if (n + 4 <= g.n) __builtin_memcpy(to, &v, 16);
        else
          for (int e = 0; e < g.n - n; ++e) to[e] = v[e];
        continue;
      }
      if (g.bias)
        for (int e = 0; e < 4; ++e) v[e] += n + e < g.n ? bias_at(g.bias, g.bias_type, n + e) : 0.f;
      store_four(g.out, g.out_type, (long)m * g.ldo + n, v, g.n - n);
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

// Which kernel computes a product, by how many workgroups its tiles would make (all
// figures in us, on 256 compute units, for 16-bit results unless said otherwise):
//   32x32 direct while each unit has one and a wave has few blocks: 256x1000x2048 7.4
//     against 8.9 of 64x64, but 64x64x8192 22 against 9.9 of 64x64 in eight parts;
//   64x64 while each unit has two: 1024x1000x2048 9.7 against 16 of 32x32 and 13 of
//     128x128; 512x4096x4096 19 against 24;
//   128x128 in four stages while each has one, in two (which fit twice) while each has
//     two and tiles are short: 2048x2048x8192 44 against 54 of 256x256, 8192x1000x2048
//     23 against 25, but 3000x3000x5120 76 against 48;
//   128x256 while each has one, for 32-bit results, 4096x2048x8192 117 against 139, and
//     for 32-bit scales, 2500x2500x8192 80 against 96 (with e8m0 256x256 is as fast: 70
//     and 67); and wherever both have 32 bits, for which 256x256 has no registers;
//   256x256 for the rest: 8192x8192x8192 386 against 575 of 128x128.
enum Tile { kDirect32, kMid64, kMid128Deep, kMid128, kMid128x256, kBig };
static Tile tile_for(int kind, int out_type, int m, int n, int blocks) {
  const bool exact = out_type == kTypeF32;
  auto groups = [&](int tm, int tn) { return (long)((m + tm - 1) / tm) * ((n + tn - 1) / tn); };
  if (groups(32, 32) <= 256 && blocks <= 16) return kDirect32;
  if (groups(64, 64) <= 512) return kMid64;
  if (groups(128, 128) <= 256) return kMid128Deep;
  if (exact && kind == kF32) return kMid128x256;
  if (!exact && groups(128, 128) <= 512 && blocks <= 16) return kMid128;
  if ((exact || kind == kF32) && groups(128, 256) <= 256) return kMid128x256;
  return kBig;
}

// How many columns 256x256 tiles take where their last round on the 256 units would be
// the shorter part of one: whole rounds, if smaller tiles compute the rest in less than
// the round that it saves (a half with 128x128, three quarters with 128x256), and a
// round is long enough for another launch. 4096x4452x4096 89 us in one launch, 76 in
// two; 8192x4608x8192 258 and 248; with 32-bit scales 117 and 89, 340 and 308.
static int columns_of_rounds(int kind, int out_type, int m, int n, int blocks) {
  const int down = (m + 255) / 256, rounds = (int)((long)down * ((n + 255) / 256) / 256);
  const int columns = rounds * 256 / down * 256;
  if (blocks < 16 || columns == 0 || columns >= n) return n;
  const Tile rest = tile_for(kind, out_type, m, n - columns, blocks);
  return rest == kBig || rest == kMid128 ? n : columns;
}

// How many parts the contraction is split into; the caller gives that many [m][n]
// matrices of floats where there are more than one. Only 64x64 tiles are split, to
// one workgroup a unit and eight steps each: 500x500x8192 26 us in one part, 14 in
// four; 32x8192x8192 27 and, in two, 19.
extern "C" int al_fp8_gemm_splits(int kind, int out_type, int m, int n, int blocks) {
  if (tile_for(kind, out_type, m, n, blocks) != kMid64) return 1;
  const long tiles = (long)((m + 63) / 64) * ((n + 63) / 64);
  return (int)std::max(1l, std::min({(long)blocks / 8, 256 / std::max(tiles, 1l), 8l}));
}

// a launch with more than 64 KB of LDS, which is asked for once on each device
template <auto KERNEL>
static void launch_lds(int groups, int splits, int threads, int bytes, hipStream_t stream, Gemm g, int tiles_m,
                       int tiles_n) {
  static bool allowed[64];
  int device = 0;
  (void)hipGetDevice(&device);
  if (!allowed[device & 63]) {
    (void)hipFuncSetAttribute((const void*)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    allowed[device & 63] = true;
  }
  hipLaunchKernelGGL(KERNEL, dim3(groups, splits), dim3(threads), bytes, stream, g, tiles_m, tiles_n);
}

template <int KIND, bool EXACT, bool BTILE, int TM, int TN, int WM, int WN, int STAGES>
static void launch_mid(const Gemm& g, hipStream_t stream) {
  const int down = (g.m + TM - 1) / TM, across = (g.n + TN - 1) / TN;
  launch_lds<gemm_mid_kernel<KIND, EXACT, BTILE, TM, TN, WM, WN, STAGES>>(
      down * across, g.splits, WM * WN * 64, STAGES * (TM + TN) * (kQB + 4), stream, g, down, across);
}

template <int KIND, bool EXACT, bool BTILE>
static void gemm(Tile tile, const Gemm& g, hipStream_t stream) {
  auto across = [&](int t) { return (g.n + t - 1) / t; };
  auto down = [&](int t) { return (g.m + t - 1) / t; };
  if (tile == kDirect32) {
    hipLaunchKernelGGL((direct_kernel<unsigned char, EXACT, KIND, BTILE, 2, 2, 4>), dim3(across(32) * down(32)),
                       dim3(256), 0, stream, (const unsigned char*)nullptr, 0l, 0, g, across(32));
  } else if (tile == kMid64) {
    launch_mid<KIND, EXACT, BTILE, 64, 64, 2, 2, 4>(g, stream);
  } else if (tile == kMid128Deep) {
    launch_mid<KIND, EXACT, BTILE, 128, 128, 2, 4, 4>(g, stream);
  }
  if constexpr (EXACT || KIND == kF32) {
    if (tile == kMid128x256) launch_mid<KIND, EXACT, BTILE, 128, 256, 2, 4, 3>(g, stream);
  }
  if constexpr (!EXACT) {
    if (tile == kMid128) launch_mid<KIND, false, BTILE, 128, 128, 2, 4, 2>(g, stream);
  }
  if constexpr (!(EXACT && KIND == kF32)) {
    if (tile == kBig)
      launch_lds<gemm256_kernel<KIND, EXACT, BTILE>>(
          down(256) * across(256), 1, 512, kRingS + 2 * 512 * (KIND == kE8M0 ? 4 : 16), stream, g, down(256),
          across(256));
  }
}

extern "C" void al_fp8_gemm(int kind, const void* a, const void* sa, long lda, int sa_stride,
                            const void* b, const void* sb, long ldb, int sb_stride, int b_tile,
                            int m, int n, int blocks, const void* bias, int bias_type, void* out,
                            int out_type, float* split_out, int splits, hipStream_t stream) {
  const Gemm g = {(const unsigned char*)a, (const unsigned char*)b, sa, sb, lda, ldb, sa_stride,
                  sb_stride, m, n, blocks, bias, bias_type, out, out_type, n, split_out, splits};
  auto run = [&](const Gemm& g) {
    const Tile tile = tile_for(kind, out_type, g.m, g.n, blocks);
    with_kind(kind, [&](auto k) {
      constexpr int KIND = decltype(k)::value;
      if (out_type == kTypeF32) b_tile ? gemm<KIND, true, true>(tile, g, stream) : gemm<KIND, true, false>(tile, g, stream);
      else b_tile ? gemm<KIND, false, true>(tile, g, stream) : gemm<KIND, false, false>(tile, g, stream);
    });
  };
  const int columns = tile_for(kind, out_type, m, n, blocks) == kBig ? columns_of_rounds(kind, out_type, m, n, blocks) : n;
  Gemm part = g;
  part.n = columns;
  run(part);
  if (columns < n) {  // a multiple of 256
    const int bytes = out_type == kTypeF32 ? 4 : 2;
    part.n = n - columns;
    part.b = g.b + (long)columns * ldb;
    part.sb = (const unsigned char*)sb + (long)(b_tile ? columns / kQB : columns) * sb_stride * (kind == kE8M0 ? 1 : 4);
    part.out = (unsigned char*)out + (long)columns * bytes;
    if (bias) part.bias = (const unsigned char*)bias + (long)columns * (bias_type == kTypeF32 ? 4 : 2);
    run(part);
  }
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
            bias, bias_type, out, type, n, nullptr, 1};
  with_type(type, [&](auto* t) {
    with_kind(kind, [&](auto k) {
      typedef std::remove_pointer_t<decltype(t)> T;
      constexpr int KIND = decltype(k)::value;
      constexpr bool EXACT = std::is_same<T, float>::value;
      auto go = [&](auto kernel, int columns) {
        const int across = (n + columns - 1) / columns;
        hipLaunchKernelGGL(kernel, dim3(across), dim3(512), 0, stream, (const T*)x, x_stride, dim, g, across);
      };
      // as many columns as still give each compute unit a workgroup: the more of
      // them share the quantisation of x the better
      if (n >= 64 * 256) b_tile ? go(direct_kernel<T, EXACT, KIND, true, 1, 4, 8>, 64) : go(direct_kernel<T, EXACT, KIND, false, 1, 4, 8>, 64);
      else if (n >= 32 * 256) b_tile ? go(direct_kernel<T, EXACT, KIND, true, 1, 2, 8>, 32) : go(direct_kernel<T, EXACT, KIND, false, 1, 2, 8>, 32);
      else b_tile ? go(direct_kernel<T, EXACT, KIND, true, 1, 1, 8>, 16) : go(direct_kernel<T, EXACT, KIND, false, 1, 1, 8>, 16);
    });
  });
}
