// y = x W^T with W in 4 bits: w = (code - zero) * scale, codes 0 .. 15, a scale and a zero for a row's group of 32, 64 or 128 k.
// bf16 x, fp32 sums.  (The reference has no weights of fewer bits than its activations'.)
//
// W comes in blocks of 16 rows x 128 k of 1 KB, as the waves read them: int32 [ceil(N / 16)][ceil(K / 128)][64][4]; lane 16 g + r holds row r,
// its word s the k 32 s + 8 g + i, i = 0 .. 7, at nibble i / 2 + 4 (i % 2), which is one operand of v_mfma_f32_16x16x32_bf16 (W as A, x^T as
// B).  Groups have a word each, int32 [ceil(N / 16)][ceil(K / 128) * 128 / group][16]: the scale in bfloat16 in the upper half, 16 + zero in
// bfloat16 (exactly) in the lower.  Rows and k behind the last are zero words.
//
// A code becomes an operand in two instructions for two of them: the bfloat16 number 16 + code has the code in the upper four bits of its mantissa, so a
// word's nibbles are shifted into place, masked and joined with the exponent.  Of a group the matrix cores then sum
//   D = sum_k (16 + code) x   and   S = sum_k x   (a product with ones, shared by the blocks of 16 rows that a wave holds),
// exactly but for the rounding of fp32 sums, and the group adds scale * (D - (16 + zero) S) to the result in fp32: the weights are never rounded.
//
//  * w4_rows: up to 16 rows of x.  A workgroup owns NT blocks of 16 rows of W; its waves share K in stretches of U blocks; their sums are added in
//    LDS in wave order.  Bound by the stream of W (0.53 bytes a weight with groups of 128).
//  * w4_wide: more rows, 16 MB a workgroup.  Its waves have NT blocks of W each and share x, which goes through LDS; where there are few of them K is cut
//    over workgroups, whose sums w4_add adds in order.
//  * many rows go through the large tiles (gemm_large.hip), which round the weights to fp16 in their registers; w4_half makes fp16 of x for them, and their sums
//    of a cut K come to w4_add, too.
#include "common.h"
#include "row_scale.h"

#include <type_traits>

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// eight codes of a word as 16 + code
__device__ __forceinline__ bf16x8 operand_of(uint32_t w) {
  u32x4 v;
  v[0] = ((w << 3) & 0x00780078u) | 0x41804180u;
  v[1] = ((w >> 1) & 0x00780078u) | 0x41804180u;
  v[2] = ((w >> 5) & 0x00780078u) | 0x41804180u;
  v[3] = ((w >> 9) & 0x00780078u) | 0x41804180u;
  return __builtin_bit_cast(bf16x8, v);
}
__device__ __forceinline__ float scale_of(uint32_t word) { return __uint_as_float(word & 0xffff0000u); }
__device__ __forceinline__ float zero_of(uint32_t word) { return __uint_as_float(word << 16); }  // 16 + zero
__device__ __forceinline__ bf16x8 all_ones() {
  bf16x8 v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (__bf16)1.f;
  return v;
}
__device__ __forceinline__ float silu_times(float gate, float up) { return gate / (1.f + expf(-gate)) * up; }
// gate and up rows in turns of 8: what a result is
enum { W4_STORE = 0, W4_GATED = 1, W4_PART = 2, W4_RESIDUAL = 3 };

struct W4Args {
  const bf16_t* x;
  const u32x4* data;
  const u32x4* words;
  void* y;
  int ldx, ldy, M, N, K;
};

// ------------------------------------------------------------------ up to 16 rows
// NT, U, WAVES and AHEAD (the loads of a wave's next stretch fly while it multiplies the one before) as rows_shape says, which measured them.
//
// The rows of x may be without their norm (RowScale), and the result may go into the residual stream with the norm that follows (W4_RESIDUAL): two launches
// fewer a layer of a decode step.
template <int NT, int U, int WAVES, bool AHEAD, int GROUP, int EPI, class OUT>
__global__ __launch_bounds__(WAVES * FG_WAVE) void w4_rows_kernel(const W4Args a, const RowScale sc, const Residual rs) {
  constexpr bool GATED = EPI == W4_GATED;
  constexpr int COLS = GATED ? 8 : 16, OUTS = NT * 16 * COLS, THREADS = WAVES * FG_WAVE, TURNS = (OUTS + THREADS - 1) / THREADS;
  constexpr int GPB = 128 / GROUP;  // groups in a block of 128 k
  constexpr int SPG = GROUP / 32;   // steps of 32 k in a group
  __shared__ __attribute__((aligned(16))) float red[WAVES][NT][256];
  __shared__ float rscale[16];
  const int lane = threadIdx.x % FG_WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / FG_WAVE);
  const int r16 = lane & 15, g = lane >> 4;
  const int kb = (a.K + 127) / 128, nb = (a.N + 15) / 16;
  const int t0 = blockIdx.x * NT;
  const bf16_t* xrow = a.x + (size_t)min(r16, a.M - 1) * a.ldx;  // (rows that are clamped are not stored)
  const u32x4* w_at[NT];
  const u32x4* s_at[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const size_t block = (size_t)min(t0 + t, nb - 1) * kb;
    w_at[t] = a.data + block * 64 + lane;
    s_at[t] = a.words + block * (GPB * 4) + g;  // the words of rows 4g .. 4g + 3
  }
  // What the result needs beside the sums is asked for here and there when they are.
  const RowScaleLoads squares = row_scale_ask<THREADS>(sc, a.M);
  float h[TURNS], norm_w[TURNS];
  if (EPI == W4_RESIDUAL) {
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      const int e = threadIdx.x + i * THREADS, m = min(e / (COLS * NT), a.M - 1), col = min((t0 + e / COLS % NT) * COLS + e % COLS, a.N - 1);
      h[i] = rs.h[(size_t)m * rs.ldh + col];
      norm_w[i] = rs.norm_w_f32 ? ((const float*)rs.norm_w)[col] : (float)((const bf16_t*)rs.norm_w)[col];
    }
  }
  const bf16x8 ones = all_ones();
  f32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};

  struct Stretch {
    u32x4 w[U][NT], s[U][NT][GPB], x[U][4];
  };
  // Loads are never conditional: a block behind the last is the last one again, and its x is zero.
  auto load = [&](Stretch& b, int c0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = min(c0 + u, kb - 1);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        b.w[u][t] = w_at[t][(size_t)c * 64];
#pragma unroll
        for (int j = 0; j < GPB; ++j) b.s[u][t][j] = s_at[t][(c * GPB + j) * 4];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        const int k = (c0 + u) * 128 + 32 * st + 8 * g;
        b.x[u][st] = *(const u32x4*)(xrow + (k < a.K ? k : 0));
      }
  };
  auto multiply = [&](const Stretch& b, int c0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      bf16x8 x[4];
#pragma unroll
      for (int st = 0; st < 4; ++st)
        x[st] = __builtin_bit_cast(bf16x8, (c0 + u) * 128 + 32 * st + 8 * g < a.K ? b.x[u][st] : u32x4{0, 0, 0, 0});
#pragma unroll
      for (int j = 0; j < GPB; ++j) {
        f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < SPG; ++st) sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, x[j * SPG + st], sum, 0, 0, 0);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          f32x4 d = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int st = 0; st < SPG; ++st)
            d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand_of(b.w[u][t][j * SPG + st]), x[j * SPG + st], d, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            acc[t][i] = fmaf(scale_of(b.s[u][t][j][i]), fmaf(-zero_of(b.s[u][t][j][i]), sum[i], d[i]), acc[t][i]);
        }
      }
    }
  };
  constexpr int STEP = WAVES * U;
  if constexpr (AHEAD) {
    Stretch a0, a1;
    load(a0, wave * U);
    for (int c0 = wave * U; c0 < kb; c0 += 2 * STEP) {
      load(a1, c0 + STEP);
      multiply(a0, c0);
      if (c0 + STEP >= kb) break;  // uniform
      load(a0, c0 + 2 * STEP);
      multiply(a1, c0 + STEP);
    }
  } else {
    for (int c0 = wave * U; c0 < kb; c0 += STEP) {
      Stretch b;
      load(b, c0);
      multiply(b, c0);
    }
  }
  // lane (row of x r16, rows of W 4g .. 4g + 3): a block's 16 x 16 sums as [row of x][row of W]
#pragma unroll
  for (int t = 0; t < NT; ++t) *(f32x4*)&red[wave][t][16 * r16 + 4 * g] = acc[t];
  row_scale_end<THREADS>(sc, row_scale_sum<THREADS>(sc, a.M, squares), rscale);
  __syncthreads();
#pragma unroll
  for (int turn = 0; turn < TURNS; ++turn) {
    const int e = threadIdx.x + turn * THREADS;
    if (e >= OUTS) break;  // whole waves
    const int n = e % COLS, t = e / COLS % NT, m = e / (COLS * NT);
    const int col = (t0 + t) * COLS + n, at = m * 16 + n;
    float v = 0.f, up = 0.f;
#pragma unroll
    for (int wv = 0; wv < WAVES; ++wv) {
      v += red[wv][t][at];
      if (GATED) up += red[wv][t][at + 8];
    }
    v *= rscale[m];
    up *= rscale[m];
    const bool there = m < a.M && col < (GATED ? a.N / 2 : a.N);
    if constexpr (EPI == W4_RESIDUAL) {
      const float sum = h[turn] + v;
      if (there) {
        rs.h[(size_t)m * rs.ldh + col] = sum;
        rs.x_out[(size_t)m * rs.ldxo + col] = (bf16_t)(sum * norm_w[turn]);
      }
      float square = there ? sum * sum : 0.f;  // (16 lanes beside one another have a block's 16 columns of a row)
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) square += __shfl_xor(square, w, FG_WAVE);
      if (n == 0 && m < a.M && t0 + t < nb) rs.ssq_out[(size_t)m * nb + t0 + t] = square;
    } else if (there) {
      ((OUT*)a.y)[(size_t)m * a.ldy + col] = from_f<OUT>(GATED ? silu_times(v, up) : v);
    }
  }
}

// ------------------------------------------------------------------ more rows
// Eight waves, each with NT blocks of 16 rows of W, whose words and codes go from memory into its registers three blocks of 128 k ahead; the waves' common
// 16 MB rows of x go straight into LDS as far ahead, through a ring of four stages with one bare barrier a stage.  A row of a stage is 256 bytes, and
// its 16-byte chunk c lies at place c ^ (row % 16), so that a load brings whole lines and 16 lanes that read the same chunk of 16 rows use all banks.
//
// With every wave reading x for itself (the form for up to 16 rows) x was the bound, by the requests: 16 rows' half lines a load.  us, that form and this one:
// 48 rows of 4,096 x 14,336 43 / 19.6, 64 rows of 28,672 x 4,096 48 / 34, 64 of 4,096 x 14,336 57 / 23, 32 of 4,096 x 14,336 31 / 17.
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  constexpr int n = N < 63 ? N : 63;
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((n & 15) | ((n >> 4) << 14) | (7 << 4));  // (and no read of LDS in flight)
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void bare_barrier() {  // (__syncthreads would wait for every load in flight)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// A lane's offset behind the end of any buffer (they have at most 4,000,000,000 bytes): the load gives zeros, also with the scalar offset added.
#define W4_NOWHERE 0xf0000000u
#define W4_WAVES 8

template <int MB, int NT, int GROUP, int EPI, class OUT>
__global__ __launch_bounds__(W4_WAVES * FG_WAVE) void w4_wide_kernel(const W4Args a, int stages_per_split, size_t part_stride) {
  constexpr int GPB = 128 / GROUP, SPG = GROUP / 32, RING = 4;
  constexpr int LOAD_ROWS = W4_WAVES * 4;                    // rows of x that one load of every wave brings
  constexpr int XL = (16 * MB + LOAD_ROWS - 1) / LOAD_ROWS;  // loads of x a wave issues a stage
  constexpr int STAGE = XL * LOAD_ROWS * 128;                // elements
  constexpr int LOADS = XL + NT * (1 + GPB);
  __shared__ __attribute__((aligned(16))) bf16_t ring[RING][STAGE];
  const int lane = threadIdx.x % FG_WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / FG_WAVE);
  const int r16 = lane & 15, g = lane >> 4;
  const int kb = (a.K + 127) / 128, nb = (a.N + 15) / 16;
  const int t0 = (blockIdx.x * W4_WAVES + wave) * NT, m0 = blockIdx.y * (16 * MB);
  const int first = blockIdx.z * stages_per_split, n_stages = min(stages_per_split, kb - first);
  const int rows = min(16 * MB, a.M - m0);
  const __amdgpu_buffer_rsrc_t x_rows = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(a.x + (size_t)m0 * a.ldx), 0, 2u * (unsigned)((rows - 1) * a.ldx + a.K), 0x20000);
  unsigned xo[XL];
  int xk[XL];
#pragma unroll
  for (int j = 0; j < XL; ++j) {
    const int q = j * W4_WAVES * FG_WAVE + threadIdx.x, row = q / 16, c = (q % 16) ^ (row & 15);
    xo[j] = row < rows ? 2u * (unsigned)row * (unsigned)a.ldx + 16u * c : W4_NOWHERE;
    xk[j] = 8 * c;
  }
  const u32x4* w_at[NT];
  const u32x4* s_at[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const size_t block = (size_t)min(t0 + t, nb - 1) * kb;
    w_at[t] = a.data + block * 64 + lane;
    s_at[t] = a.words + block * (GPB * 4) + g;
  }
  u32x4 w[RING][NT], s[RING][NT][GPB];
  // Every stage is LOADS loads of a wave, also one behind the last (zeros, and the last blocks of W again): wait_vmcnt counts them.
  auto load = [&](int i, int slot) {
    const int c = first + min(i, n_stages - 1);
#pragma unroll
    for (int j = 0; j < XL; ++j) {
      const unsigned off = i < n_stages && c * 128 + xk[j] < a.K ? xo[j] : W4_NOWHERE;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(x_rows, (__attribute__((address_space(3))) void*)(&ring[slot][(j * W4_WAVES + wave) * 512]), 16,
                                               off, 256u * (unsigned)c, 0, 0);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      w[slot][t] = w_at[t][(size_t)c * 64];
#pragma unroll
      for (int j = 0; j < GPB; ++j) s[slot][t][j] = s_at[t][(c * GPB + j) * 4];
    }
    asm volatile("" ::: "memory");  // (a stage's loads stay together, in front of the next one's)
    __builtin_amdgcn_sched_barrier(0);
  };
  const bf16x8 ones = all_ones();
  f32x4 acc[NT][MB];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) acc[t][mb] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](int slot) {
    const bf16_t* mine = ring[slot] + r16 * 128;
#pragma unroll
    for (int j = 0; j < GPB; ++j) {
      bf16x8 op[NT][SPG];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int st = 0; st < SPG; ++st) op[t][st] = operand_of(w[slot][t][j * SPG + st]);
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f}, d[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) d[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < SPG; ++st) {
          const bf16x8 x = *(const bf16x8*)(mine + mb * 2048 + (((4 * (j * SPG + st) + g) ^ r16) * 8));
#pragma unroll
          for (int t = 0; t < NT; ++t) d[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(op[t][st], x, d[t], 0, 0, 0);
          sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, x, sum, 0, 0, 0);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            acc[t][mb][i] = fmaf(scale_of(s[slot][t][j][i]), fmaf(-zero_of(s[slot][t][j][i]), sum[i], d[t][i]), acc[t][mb][i]);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < RING - 1; ++i) load(i, i);
  for (int i0 = 0; i0 < n_stages; i0 += RING) {
#pragma unroll
    for (int u = 0; u < RING; ++u) {
      if (i0 + u >= n_stages) break;     // uniform over the workgroup
      wait_vmcnt<(RING - 2) * LOADS>();  // this wave's part of the stage has landed, and behind the barrier everyone's
      bare_barrier();                    // and nobody reads the place of the stage before any more
      load(i0 + u + RING - 1, (u + RING - 1) % RING);
      multiply(u);
    }
  }
  wait_vmcnt<0>();  // (what was asked for behind the end has landed before the LDS is given up)
  // lane (row of x r16, rows of W 4g .. 4g + 3)
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int n = 16 * (t0 + t) + 4 * g;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      const int m = m0 + 16 * mb + r16;
      if constexpr (EPI == W4_GATED) {
        // the gates' lanes get their ups from 32 lanes on
        bf16x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (__bf16)silu_times(acc[t][mb][i], __shfl_xor(acc[t][mb][i], 32, FG_WAVE));
        if (m < a.M && n < a.N && g < 2) *(bf16x4*)((bf16_t*)a.y + (size_t)m * a.ldy + 8 * (t0 + t) + 4 * g) = v;
      } else if constexpr (EPI == W4_PART) {  // (rows of a multiple of 16 numbers)
        if (m < a.M && n < a.ldy) *(f32x4*)((float*)a.y + blockIdx.z * part_stride + (size_t)m * a.ldy + n) = acc[t][mb];
      } else if (m < a.M) {
        OUT* to = (OUT*)a.y + (size_t)m * a.ldy + n;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n + i < a.N) to[i] = from_f<OUT>(acc[t][mb][i]);
      }
    }
  }
}

// y from partial sums [splits][M][ld], ld a multiple of 16, added in order: a thread four numbers.
template <bool GATED, class OUT>
__global__ __launch_bounds__(256) void w4_add_kernel(const float* __restrict__ part, size_t part_stride, int splits, int ld, OUT* __restrict__ y,
                                                     int ldy, int M, int N) {
  const int per_row = ld / 4;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)M * per_row) return;  // (four threads of a block of 16 stay or go together)
  const int m = (int)(i / per_row), n = (int)(i % per_row) * 4;
  const float* p = part + (size_t)m * ld + n;
  f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; ++s) v += *(const f32x4*)(p + s * part_stride);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (GATED) {
      const float up = __shfl_xor(v[e], 2, FG_WAVE);
      if (n % 16 < 8) y[(size_t)m * ldy + n / 16 * 8 + n % 16 + e] = from_f<OUT>(silu_times(v[e], up));
    } else if (n + e < N) {
      y[(size_t)m * ldy + n + e] = from_f<OUT>(v[e]);
    }
  }
}

// x in fp16 for the large tiles, each row divided by a power of two, so that its largest number lies below 2^15 (exact, but for numbers below 2^-29 of the
// largest); and what the scales of a row of W are divided by there: their largest comes to lie below 2^11, a weight below 2^15.  A workgroup a row of x, then one a
// block of 16 rows of W.  exponents: of M rows of x, and from the next multiple of 4 on of the rows of W.
__global__ __launch_bounds__(256) void w4_half_kernel(const bf16_t* __restrict__ x, int ldx, _Float16* __restrict__ xh, int* __restrict__ exponents,
                                                      const uint32_t* __restrict__ words, int M, int K, int groups) {
  typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
  __shared__ uint32_t largest[4][16];
  const int tid = threadIdx.x, lane = tid % FG_WAVE, wave = tid / FG_WAVE;
  if ((int)blockIdx.x < M) {  // uniform
    const bf16_t* row = x + (size_t)blockIdx.x * ldx;
    uint32_t size = 0;
    for (int k = 8 * tid; k < K; k += 8 * 256) {
      const u32x4 v = *(const u32x4*)(row + k);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = v[i] & 0x7fff0000u, b = (v[i] << 16) & 0x7fff0000u;
        if (a < 0x7f800000u) size = max(size, a);  // (numbers that are not finite stay what they are)
        if (b < 0x7f800000u) size = max(size, b);
      }
    }
#pragma unroll
    for (int n = 32; n > 0; n >>= 1) size = max(size, (uint32_t)__shfl_xor((int)size, n, FG_WAVE));
    if (lane == 0) largest[wave][0] = size;
    __syncthreads();
    size = max(max(largest[0][0], largest[1][0]), max(largest[2][0], largest[3][0]));
    const int e = max((int)(size >> 23), 1) - 127 - 14;
    if (tid == 0) exponents[blockIdx.x] = e;
    for (int k = 8 * tid; k < K; k += 8 * 256) {
      float v[8];
      load8<bf16_t>(row + k, v);
      f16x8 h;
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = (_Float16)ldexpf(v[i], -e);
      *(f16x8*)(xh + (size_t)blockIdx.x * K + k) = h;
    }
  } else {
    const int block = blockIdx.x - M;
    uint32_t size = 0;
    for (int j = tid / 16; j < groups; j += 16) size = max(size, words[((size_t)block * groups + j) * 16 + tid % 16] & 0x7fff0000u);
    size = max(size, (uint32_t)__shfl_xor((int)size, 16, FG_WAVE));
    size = max(size, (uint32_t)__shfl_xor((int)size, 32, FG_WAVE));
    if (lane < 16) largest[wave][lane] = size;
    __syncthreads();
    if (tid < 16) {
      size = max(max(largest[0][tid], largest[1][tid]), max(largest[2][tid], largest[3][tid]));
      exponents[(M + 3) / 4 * 4 + 16 * block + tid] = max((int)(size >> 23), 1) - 127 - 10;
    }
  }
}

// Up to 16 rows.  A workgroup has one block of 16 rows of W up to as many workgroups as there are compute units (256), with groups of 32 up to three a unit, two blocks up to
// 1,024 blocks, then four.  us at 1 / 8 / 16 rows with one block and with two, groups of 128: 256 blocks x 5,120 k 6.2 / 6.8 / 8.3 and 8.2 / 9.0 / 10.2, 288 8.2 / 9.8 / 13.5 and 8.3 / 9.0 /
// 10.2, 512 8.8 / 10.1 / 13.8 and 8.9 / 9.4 / 10.6; x 2,048 k 256 3.6 / 4.0 / 4.6 and 4.0 / 4.3 / 4.9, 288 4.5 / 5.3 / 6.6 and 4.1 / 4.3 / 4.9; x 8,192 k 256 8.2 / 9.0 / 10.9 and 11.5 / 11.8 / 13.6,
// 288 12.0 / 14.4 / 19.0 and 11.8 / 11.9 / 13.7.  Groups of 64: 256 x 5,120 k 6.3 / 7.1 / 9.0 and 7.5 / 8.3 / 10.3, 288 10.0 / 11.5 / 15.4 and 7.6 / 8.5 / 10.6.  Groups of 32: 256 x 5,120 k 7.1 / 7.6 / 9.3
// and 15.4 / 16.4 / 17.6, 768 17.8 / 19.2 / 24.0 and 20.1 / 21.5 / 23.9, 896 21.9 / 23.9 / 30.1 and 20.3 / 21.8 / 24.1 (768 x 2,048 k 9.9 / 10.7 / 12.4 and 9.7 / 10.2 / 11.3).  Two and four blocks: 1,792 x 4,096 k
// 16.9 and 17.3 at 8 rows, 21 and 19.1 at 16, whose x the blocks share; 512 x 28,672 k 34.9 and 39 at 8.
// Two blocks a workgroup with 16 waves of one block of k and with 8 of two, 1 / 8 / 16 rows: 384 x 4,096 k 5.8 / 6.3 / 7.6 and 6.0 / 6.3 / 7.5, 704 x 2,048 k 6.9 / 7.7 / 8.9 and 5.5 / 6.2 / 7.4, 1,024 x
// 2,048 k 7.7 / 8.4 / 9.7 and 6.2 / 6.8 / 8.0.  One block a workgroup with two blocks of k a wave and with one: 256 x 4,096 k 5.3 / 6.0 / 7.2 and 5.3 / 5.7 / 6.9, x 8,192 k 8.0 / 8.9 / 11.9 and
// 8.1 / 8.9 / 10.9, x 14,336 k 11.3 / 12.9 / 18.8 and 12.2 / 13.3 / 16.9 (that in groups of 64 13.6 / 15.1 / 19.9 and 12.9 / 13.9 / 19.5).  (The number of rows picks nothing: a row has the same bits whatever
// is beside it.)
template <int GROUP, int EPI, class OUT>
static void launch_rows(const W4Args& a, const RowScale& sc, const Residual& rs, hipStream_t stream) {
  const int nb = (a.N + 15) / 16;
  constexpr int WAVES = GROUP == 64 ? 16 : 8;  // (with groups of 64 two stretches of two blocks do not fit the registers, with 32 not two of one)
  if constexpr (GROUP == 128)
    if (nb <= 256 && a.K > 8192) {
      w4_rows_kernel<1, 2, 16, false, GROUP, EPI, OUT><<<nb, 1024, 0, stream>>>(a, sc, rs);
      return;
    }
  if (nb <= (GROUP == 32 ? 768 : 256)) w4_rows_kernel<1, 1, 16, false, GROUP, EPI, OUT><<<nb, 1024, 0, stream>>>(a, sc, rs);
  else if (nb <= 1024) w4_rows_kernel<2, GROUP == 128 ? 2 : 1, WAVES, GROUP != 32, GROUP, EPI, OUT><<<(nb + 1) / 2, WAVES * FG_WAVE, 0, stream>>>(a, sc, rs);
  else w4_rows_kernel<4, 1, 8, GROUP != 32, GROUP, EPI, OUT><<<(nb + 3) / 4, 512, 0, stream>>>(a, sc, rs);
}
template <class GO>
static void with_group(int group, GO go) {
  if (group == 32) go(std::integral_constant<int, 32>{});
  else if (group == 64) go(std::integral_constant<int, 64>{});
  else go(std::integral_constant<int, 128>{});
}
static bool product_ok(const void* x, int ldx, const void* data, const void* words, int N, int K, int group) {
  return x && data && words && N > 0 && K > 0 && (group == 32 || group == 64 || group == 128) && K % group == 0 && ldx >= K && ldx % 8 == 0;
}
static bool scale_ok(const float* ssq, int n_parts, int dim, float eps) { return !ssq || (n_parts >= 1 && dim >= 1 && eps >= 0.f); }

template <int GROUP, bool GATED, class OUT, int MB, int NT>
static void launch_wide_of(const W4Args& a, int splits, float* part, bool add, hipStream_t stream) {
  const dim3 grid((a.N + 16 * NT * W4_WAVES - 1) / (16 * NT * W4_WAVES), (a.M + 16 * MB - 1) / (16 * MB), splits);
  const int kb = (a.K + 127) / 128;
  if (splits == 1) {
    w4_wide_kernel<MB, NT, GROUP, GATED ? W4_GATED : W4_STORE, OUT><<<grid, W4_WAVES * FG_WAVE, 0, stream>>>(a, kb, 0);
    return;
  }
  W4Args p = a;
  p.y = part;
  p.ldy = (a.N + 15) / 16 * 16;
  const size_t stride = (size_t)a.M * p.ldy;
  w4_wide_kernel<MB, NT, GROUP, W4_PART, float><<<grid, W4_WAVES * FG_WAVE, 0, stream>>>(p, (kb + splits - 1) / splits, stride);
  if (!add) return;
  const long long threads = (long long)a.M * (p.ldy / 4);
  w4_add_kernel<GATED, OUT><<<(unsigned)((threads + 255) / 256), 256, 0, stream>>>(part, stride, splits, p.ldy, (OUT*)a.y, a.ldy, a.M, a.N);
}
template <int GROUP, bool GATED, class OUT>
static bool launch_wide(const W4Args& a, int mb, int nt, int splits, float* part, bool add, hipStream_t stream) {
  if (mb == 2 && nt == 1) launch_wide_of<GROUP, GATED, OUT, 2, 1>(a, splits, part, add, stream);
  else if (mb == 3 && nt == 1) launch_wide_of<GROUP, GATED, OUT, 3, 1>(a, splits, part, add, stream);
  else if (mb == 4 && nt == 1) launch_wide_of<GROUP, GATED, OUT, 4, 1>(a, splits, part, add, stream);
  else if constexpr (GROUP == 32) return false;  // (the words of four groups a block: two blocks a wave do not fit its registers)
  else if (mb == 2 && nt == 2) launch_wide_of<GROUP, GATED, OUT, 2, 2>(a, splits, part, add, stream);
  else if (mb == 3 && nt == 2) launch_wide_of<GROUP, GATED, OUT, 3, 2>(a, splits, part, add, stream);
  else if constexpr (GROUP == 64) return false;
  else if (mb == 4 && nt == 2) launch_wide_of<GROUP, GATED, OUT, 4, 2>(a, splits, part, add, stream);
  else return false;
  return true;
}

// x: bf16 [M, ldx], rows 16-byte aligned; data, words: as above, 16-byte aligned.  y: [M, ldy], fp32 or bf16; gated (bf16, N % 16 == 0, ldy % 4 == 0): W is
// a gate and an up matrix in turns of 8 rows, y = silu(gate) * up of N / 2 columns.  mb, nt: blocks of 16 rows of x a workgroup (2 to 4) and of W a wave (1 or 2; 1
// with groups of 32, and with groups of 64 and mb 4) of w4_wide, or 0 for w4_rows (M <= 16).  splits > 1: K is cut, none of them empty, and part holds fp32 [splits][M][N rounded up to 16],
// which are added into y, or left as they are where y is null.  ssq [M, n_parts] (null: x is taken as it is; else w4_rows): the sums of squares, over dim
// columns, of the rows' norm.
extern "C" int fg_gemm_w4(const void* x, int ldx, const void* data, const void* words, void* y, int ldy, int M, int N, int K, int group,
                          int gated, int out_dtype, int mb, int nt, int splits, float* part, const float* ssq, int n_parts, int dim, float eps,
                          hipStream_t stream) {
  if (M <= 0) return FG_OK;
  if (!product_ok(x, ldx, data, words, N, K, group) || !scale_ok(ssq, n_parts, dim, eps) || ldy < (gated ? N / 2 : N) ||
      (gated && (N % 16 || ldy % 4 || out_dtype != FG_BF16)) || (out_dtype != FG_F32 && out_dtype != FG_BF16) || (!y && (splits < 2 || gated)))
    return FG_ERR_ARG;
  const W4Args a{(const bf16_t*)x, (const u32x4*)data, (const u32x4*)words, y, ldx, ldy, M, N, K};
  const int kb = (K + 127) / 128;
  if (mb == 0) {
    if (M > 16 || splits != 1) return FG_ERR_ARG;
  } else if (mb < 2 || mb > 4 || splits < 1 || splits > 64 || (kb + splits - 1) / splits * (splits - 1) >= kb || (splits > 1 && !part) || ssq ||
             128LL * ldx + 2LL * K > 4000000000LL || M > 32 * 65535 || (long long)M * ((N + 15) / 16 * 4) > 512LL * 2147483647LL) {
    return FG_ERR_ARG;
  }
  bool ok = true;
  with_group(group, [&](auto kernel_group) {
    constexpr int GROUP = decltype(kernel_group)::value;
    if (mb == 0) {
      const RowScale sc{ssq, n_parts, ssq ? 1.f / (float)dim : 0.f, eps};
      if (gated) launch_rows<GROUP, W4_GATED, bf16_t>(a, sc, {}, stream);
      else if (out_dtype == FG_F32) launch_rows<GROUP, W4_STORE, float>(a, sc, {}, stream);
      else launch_rows<GROUP, W4_STORE, bf16_t>(a, sc, {}, stream);
    } else {
      if (gated) ok = launch_wide<GROUP, true, bf16_t>(a, mb, nt, splits, part, true, stream);
      else if (out_dtype == FG_F32) ok = launch_wide<GROUP, false, float>(a, mb, nt, splits, part, y != nullptr, stream);
      else ok = launch_wide<GROUP, false, bf16_t>(a, mb, nt, splits, part, y != nullptr, stream);
    }
  });
  return ok ? fg_launch_status() : FG_ERR_ARG;
}

// Up to 16 rows: h [M, ldh] += the product, x_out [M, ldxo] = h * norm_w in bf16, ssq_out [M, ceil(N / 16)] = the sums of squares of h (row_scale.h).
extern "C" int fg_gemm_w4_residual(const void* x, int ldx, const void* data, const void* words, int M, int N, int K, int group, const float* ssq,
                                   int n_parts, int dim, float eps, float* h, int ldh, const void* norm_w, int norm_w_dtype, void* x_out, int ldxo,
                                   float* ssq_out, hipStream_t stream) {
  if (M <= 0) return FG_OK;
  if (!product_ok(x, ldx, data, words, N, K, group) || !scale_ok(ssq, n_parts, dim, eps) || M > 16 || !h || !norm_w || !x_out || !ssq_out || ldh < N ||
      ldxo < N || (norm_w_dtype != FG_F32 && norm_w_dtype != FG_BF16))
    return FG_ERR_ARG;
  const W4Args a{(const bf16_t*)x, (const u32x4*)data, (const u32x4*)words, nullptr, ldx, 0, M, N, K};
  const RowScale sc{ssq, n_parts, ssq ? 1.f / (float)dim : 0.f, eps};
  const Residual rs{h, ldh, norm_w, norm_w_dtype == FG_F32, (bf16_t*)x_out, ldxo, ssq_out};
  with_group(group, [&](auto kernel_group) { launch_rows<decltype(kernel_group)::value, W4_RESIDUAL, bf16_t>(a, sc, rs, stream); });
  return fg_launch_status();
}

// xh: fp16 [M, K]; exponents: int32 [M rounded up to 4, then N rounded up to 16], 16-byte aligned (w4_half_kernel).
extern "C" int fg_w4_half(const void* x, int ldx, void* xh, int* exponents, const void* words, int M, int N, int K, int group, hipStream_t stream) {
  if (M <= 0) return FG_OK;
  const long long blocks = (long long)M + (N + 15) / 16;
  if (!product_ok(x, ldx, words, words, N, K, group) || !xh || !exponents || K % 8 || blocks > 2147483647LL) return FG_ERR_ARG;
  w4_half_kernel<<<(unsigned)blocks, 256, 0, stream>>>((const bf16_t*)x, ldx, (_Float16*)xh, exponents, (const uint32_t*)words, M, K,
                                                       (K + 127) / 128 * (128 / group));
  return fg_launch_status();
}

// y [M, ldy] = the sums part [splits][M][ld] (ld: N rounded up to 16), added in order; gated as above (then bf16).
extern "C" int fg_w4_add(const float* part, int splits, int ld, void* y, int ldy, int M, int N, int gated, int out_dtype, hipStream_t stream) {
  if (M <= 0) return FG_OK;
  const long long groups = ((long long)M * (ld / 4) + 255) / 256;
  if (!part || !y || splits < 1 || N <= 0 || ld % 16 || ld < N || ldy < (gated ? N / 2 : N) || groups > 2147483647LL ||
      (gated && (N % 16 || out_dtype != FG_BF16)) || (out_dtype != FG_F32 && out_dtype != FG_BF16))
    return FG_ERR_ARG;
  const size_t stride = (size_t)M * ld;
  if (gated) w4_add_kernel<true, bf16_t><<<(unsigned)groups, 256, 0, stream>>>(part, stride, splits, ld, (bf16_t*)y, ldy, M, N);
  else if (out_dtype == FG_F32) w4_add_kernel<false, float><<<(unsigned)groups, 256, 0, stream>>>(part, stride, splits, ld, (float*)y, ldy, M, N);
  else w4_add_kernel<false, bf16_t><<<(unsigned)groups, 256, 0, stream>>>(part, stride, splits, ld, (bf16_t*)y, ldy, M, N);
  return fg_launch_status();
}
