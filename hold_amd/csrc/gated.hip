// The gated layer  h = act(x Wg^T + bg) * (x Wu^T + bu)  in one kernel, and its backward pass.
//
//   dg = dh * u * act'(g)      du = dh * act(g)      (g, u: the two projections)
//   dx = dg Wg + du Wu         dWg = dg^T x
//   dWu = du^T x               dbg = sum_t dg, dbu = sum_t du
//
// u act'(g) and act(g) are kept from the forward pass where that is less time, and computed again, 4 T D H operations, where D is
// short or the rows are few (`keeps` has the measurements).
//
// KERNELS.  gated_mma_kernel: both projections of a tile share the x tile in LDS, the epilogue applies bias, activation and product
// (forward) or forms dg, du from dh and the recomputed g, u (backward), with the column sums for the bias gradients from the
// unrounded values.  gated_short_kernel: the same for D <= 256 in bf16.  gated_kept_kernel: dg, du from what was kept.  gated_dx_kernel: [dg | du]
// times [Wg; Wu] as one sum.  gated_dw_kernel: both weight gradients, the sum over tokens split over blocks into fp32 partial tiles that
// gated_finish_kernel adds in a fixed order.  gated_rows_kernel, gated_few_kernel: T <= 4, T <= 64.
//
// ROUNDINGS.  fp32: fp32 products and sums on v_mfma_f32_16x16x4_f32, for any number of rows.  Two fp16 limbs a value under a row's common
// scale take half the time (131072 x 256 -> 256 125 against 276 us, a step of 16384 x 768 -> 4096 2.35 against 5.24 ms) and lose digits
// without a sign where a row of x, of a weight or of dg spans more than some four decades (3e-3 relative at ten, 512 features); three bf16
// limbs keep every exponent, but an infinity times a limb of zero is NaN.
// bf16: dg and du are rounded to bf16 once, as the operands of the next matrix instructions (gradients 2.35e-3 from the
// exact ones, 1.66e-3 with that rounding left out and only the result's own; a second limb of each would double both products, two
// thirds of a training step); before, what is kept is cut to 24 bits, and everything else is fp32.
#include "tile16.h"

#include "../../include/hold_hip.h"

using namespace t16;

namespace {

enum { ACT_SILU = 0, ACT_GELU = 1, ACT_RELU = 2, ACT_SIGMOID = 3 };

// e^x by v_exp_f32 (2^x to 1 ulp).  EXACT: the product x log2 e in two parts, 2^-23 relative; else its rounding alone, |x| 2^-24, which is
// nothing to a result in bf16
template <bool EXACT>
__device__ __forceinline__ float exp_of(float x) {
  const float p = x * 1.44269504088896341f;
  if (!EXACT) return __builtin_amdgcn_exp2f(p);
  const float lo = fmaf(x, 1.44269504088896341f, -p) + x * 1.925962989e-8f;  // log2 e = 1.4426950216... + 1.926e-8 in float32
  const float e = __builtin_amdgcn_exp2f(p);
  return fabsf(p) < 200.f ? e * fmaf(lo, 0.693147180559945f, 1.f) : e;  // beyond: 0 or infinity
}
// 1 / x for x in [1, inf], by v_rcp_f32 (1 ulp) and, EXACT, a Newton step; 1 / inf = 0
template <bool EXACT>
__device__ __forceinline__ float recip(float x) {
  const float r = __builtin_amdgcn_rcpf(x);
  return EXACT && r > 0.f ? fmaf(fmaf(-x, r, 1.f), r, r) : r;
}
// the normal distribution function, 0.5 erfc(-g / sqrt 2).  erfc(z), z >= 0, by W. H. Press et al., "Numerical Recipes" (6.2, erfcc): t e^(-z^2 +
// P(t)), t = 1 / (1 + z / 2), fractional error below 1.2e-7 everywhere
template <bool EXACT>
__device__ __forceinline__ float normal_cdf(float g) {
  const float z = 0.70710678118654752f * fabsf(g), t = recip<EXACT>(fmaf(0.5f, z, 1.f));
  float p = 0.17087277f;
  p = fmaf(p, t, -0.82215223f);
  p = fmaf(p, t, 1.48851587f);
  p = fmaf(p, t, -1.13520398f);
  p = fmaf(p, t, 0.27886807f);
  p = fmaf(p, t, -0.18628806f);
  p = fmaf(p, t, 0.09678418f);
  p = fmaf(p, t, 0.37409196f);
  p = fmaf(p, t, 1.00002368f);
  p = fmaf(p, t, -1.26551223f);
  const float e = 0.5f * t * exp_of<EXACT>(fmaf(-z, z, p));
  return g > 0.f ? 1.f - e : e;
}

// act(g) and act'(g)
template <bool DERIV, bool EXACT>
__device__ __forceinline__ void activate(int act, float g, float& a, float& da) {
  if (act == ACT_RELU) {
    a = g > 0.f ? g : (g == g ? 0.f : g);
    da = g > 0.f ? 1.f : (g == g ? 0.f : g);
  } else if (act == ACT_GELU) {
    const float phi = normal_cdf<EXACT>(g);
    a = g * phi;
    if (DERIV) da = phi + g * (0.39894228040143268f * exp_of<EXACT>(-0.5f * g * g));
  } else {
    const float s = recip<EXACT>(1.f + exp_of<EXACT>(-g));
    if (act == ACT_SIGMOID) {
      a = s;
      if (DERIV) da = s * (1.f - s);
    } else {
      a = g * s;
      if (DERIV) da = s * (1.f + g * (1.f - s));
    }
  }
}

// ---- element access in the caller's type -------------------------------------------------------------------------------------------
template <int MODE>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  return MODE == MODE_BF16 ? bf16_value(((const uint16_t*)p)[i]) : ((const float*)p)[i];
}
template <int MODE>
__device__ __forceinline__ void store1(void* p, int64_t i, float v) {
  if (MODE == MODE_BF16) ((uint16_t*)p)[i] = bf16_bits(v);
  else ((float*)p)[i] = v;
}
// four consecutive elements of which the first n exist; rows may start anywhere (the memory takes 16 bytes on any element's boundary)
template <int MODE>
__device__ __forceinline__ f32x4 load4(const void* p, int64_t i, int n) {
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (n >= 4) {
    if (MODE == MODE_BF16) {
      u32x2 w;
      __builtin_memcpy(&w, (const uint16_t*)p + i, 8);
      const uint32_t w0 = w[0], w1 = w[1];
      v = f32x4{bf16_value((uint16_t)w0), bf16_value((uint16_t)(w0 >> 16)), bf16_value((uint16_t)w1), bf16_value((uint16_t)(w1 >> 16))};
    } else {
      __builtin_memcpy(&v, (const float*)p + i, 16);
    }
  } else {
#pragma unroll
    for (int r = 0; r < 3; ++r)
      if (r < n) v[r] = load1<MODE>(p, i + r);
  }
  return v;
}
template <int MODE>
__device__ __forceinline__ void store4(void* p, int64_t i, int n, f32x4 v) {
  if (n >= 4) {
    if (MODE == MODE_BF16) {
      const u32x2 w = {(uint32_t)bf16_bits(v[0]) | (uint32_t)bf16_bits(v[1]) << 16, (uint32_t)bf16_bits(v[2]) | (uint32_t)bf16_bits(v[3]) << 16};
      __builtin_memcpy((uint16_t*)p + i, &w, 8);
    } else {
      __builtin_memcpy((float*)p + i, &v, 16);
    }
  } else {
#pragma unroll
    for (int r = 0; r < 3; ++r)
      if (r < n) store1<MODE>(p, i + r, v[r]);
  }
}

// eight, on a 16-byte boundary
template <int MODE>
__device__ __forceinline__ void store8(void* p, int64_t i, const float (&v)[8]) {
  if constexpr (MODE == MODE_BF16) {
    u32x4 w;
#pragma unroll
    for (int r = 0; r < 4; ++r) w[r] = bf16_bits(v[2 * r]) | (uint32_t)bf16_bits(v[2 * r + 1]) << 16;
    *(u32x4*)((uint16_t*)p + i) = w;
  } else {
    *(f32x4*)((float*)p + i) = f32x4{v[0], v[1], v[2], v[3]};
    *(f32x4*)((float*)p + i + 4) = f32x4{v[4], v[5], v[6], v[7]};
  }
}

template <int MODE> constexpr int chunk_k() { return MODE == MODE_BF16 ? 8 : 4; }  // elements in 16 bytes

// 16 bytes of a row from element c on, zeros from element K on
template <int MODE>
__device__ __forceinline__ u32x4 chunk16(const void* p, int64_t at, int c, int K) {
  constexpr int N = chunk_k<MODE>();
  u32x4 v = {0u, 0u, 0u, 0u};
  if (c + N <= K) {
    __builtin_memcpy(&v, (const char*)p + (at + c) * (16 / N), 16);
    return v;
  }
#pragma unroll
  for (int i = 0; i < N - 1; ++i)
    if (c + i < K) {
      if (MODE == MODE_BF16) v[i >> 1] |= (uint32_t)((const uint16_t*)p)[at + c + i] << (16 * (i & 1));
      else v[i] = ((const uint32_t*)p)[at + c + i];
    }
  return v;
}
template <int MODE>
__device__ __forceinline__ float lane_value(u32x4 v, int i) {
  const uint32_t w = MODE == MODE_BF16 ? v[i >> 1] : v[i];  // a copy: __builtin_bit_cast of a vector's element reads element 0
  return __builtin_bit_cast(float, MODE == MODE_BF16 ? (i & 1 ? w & 0xffff0000u : w << 16) : w);
}

// rows whose base, stride or length the tile loads cannot take -> [rows][Kp], zeros behind K; up to three matrices of equal length
struct CopyArgs {
  const void* x[3]; int64_t ld[3], rows[3];
  void* out[3];
  int K, Kp;
};
template <int MODE>
__global__ __launch_bounds__(256) void gated_copy_rows_kernel(CopyArgs a) {
  constexpr int N = chunk_k<MODE>();
  const int lane = threadIdx.x & 63;
  const int64_t all = a.rows[0] + a.rows[1] + a.rows[2];
  for (int64_t q = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); q < all; q += (int64_t)gridDim.x * 4) {
    const int w = q < a.rows[0] ? 0 : q < a.rows[0] + a.rows[1] ? 1 : 2;
    const int64_t r = q - (w > 0 ? a.rows[0] : 0) - (w > 1 ? a.rows[1] : 0);
    u32x4* o = (u32x4*)a.out[w] + r * (a.Kp / N);
    for (int c = lane; c < a.Kp / N; c += 64) o[c] = chunk16<MODE>(a.x[w], r * a.ld[w], c * N, a.K);
  }
}

// element i of an operand of the tile loads
template <int MODE>
__device__ __forceinline__ const uint16_t* element(const void* p, int64_t i) { return (const uint16_t*)p + i * halves<MODE>(); }

// ---- both projections and what follows them (fp32, 131072 x 256 -> 256: 277 us, 124 TFLOP/s, the matrix cores 78 % busy, no bank conflict;
// the rest is tiles of eight steps starting and ending, two blocks a unit) ----
struct MmaArgs {
  const void* x; int64_t ldx;                    // operands as the tile loads take them: [T][K]
  const void* wg; const void* wu; int64_t ldwg, ldwu;
  const void* bg; const void* bu;
  int64_t T; int H; int K; int act;
  void* h; int64_t ldh;                          // forward
  const void* dh; int64_t lddh;                  // backward
  void* dg; void* du; int64_t Hp;                // [T][Hp] dg and du
  float* dbpart;                                 // [row tiles][2][H] column sums, or null
  int tm, tn;
  void* kept;                                    // forward: [T][Hp / 4] times p and s of four columns
};

// What the forward pass leaves for the backward one, for four columns side by side: p = u act'(g) and s = act(g).  fp32: as they are, 32
// bytes.  bf16: 24 bits of each, as four upper halves of p, of s and four pairs of their third bytes (p's below), 24 bytes: cut off,
// not rounded, an error below 2^-15 of the value before dg and du are rounded to 2^-8.
__device__ __forceinline__ void cut(f32x4 p, f32x4 s, u32x2 (&w)[3]) {
  uint32_t a[4], b[4], v[6];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const float x = p[r], y = s[r];
    a[r] = __builtin_bit_cast(uint32_t, x);
    b[r] = __builtin_bit_cast(uint32_t, y);
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const uint32_t l0 = (a[2 * r] >> 8 & 0xff) | (b[2 * r] & 0xff00), l1 = (a[2 * r + 1] >> 8 & 0xff) | (b[2 * r + 1] & 0xff00);
    v[r] = a[2 * r] >> 16 | (a[2 * r + 1] & 0xffff0000u);
    v[2 + r] = b[2 * r] >> 16 | (b[2 * r + 1] & 0xffff0000u);
    v[4 + r] = l0 | l1 << 16;
  }
#pragma unroll
  for (int r = 0; r < 3; ++r) w[r] = u32x2{v[2 * r], v[2 * r + 1]};
}

template <int MODE, bool BWD, int BM, int BN, int WM, int WN, bool PHASED, int S = 2, bool KEEP = false>
__global__ __launch_bounds__(64 * WM * WN) void gated_mma_kernel(MmaArgs a) {
  using Cr = Core<MODE, KC, KC, BM, BN, 2, WM, WN, S>;
  __shared__ __align__(1024) char smem[Cr::LDS];
  int tm, tn;
  tile_of(blockIdx.x, gridDim.x, a.tm, a.tn, 8, tm, tn);
  const int64_t m0 = (int64_t)tm * BM;
  const int n0 = tn * BN;
  typename Cr::Acc acc;
  Cr::zero(acc);
  const Operand A = {element<MODE>(a.x, m0 * a.ldx), 0, a.ldx, a.T - m0, a.K};
  const Operand B[2] = {{element<MODE>(a.wg, (int64_t)n0 * a.ldwg), 0, a.ldwg, a.H - n0, a.K},
                        {element<MODE>(a.wu, (int64_t)n0 * a.ldwu), 0, a.ldwu, a.H - n0, a.K}};
  if constexpr (PHASED) Cr::run_phased(smem, A, B, acc);
  else Cr::run(smem, A, B, acc);

  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
  float* sums = (float*)smem;  // [WM][2][BN]
  f32x4 dhs[BWD ? Cr::NI : 1][BWD ? Cr::MI : 1];  // all of them requested before the first store
  if (BWD) {
#pragma unroll
    for (int ni = 0; ni < Cr::NI; ++ni)
#pragma unroll
      for (int mi = 0; mi < Cr::MI; ++mi) {
        const int j = n0 + wn * (BN / WN) + 16 * ni + 4 * (lane >> 4), n = a.H - j;
        const int64_t i = m0 + wm * (BM / WM) + 16 * mi + (lane & 15);
        dhs[BWD ? ni : 0][BWD ? mi : 0] = i < a.T && n > 0 ? load4<MODE>(a.dh, i * a.lddh + j, n) : f32x4{0.f, 0.f, 0.f, 0.f};
      }
  }
  // Where much is kept the tiles of 256 rows, alone on their unit, send p and s through LDS, half of each wave's rows at a time, so that
  // whole lines leave: 16384 x 2048 -> 8192 in bf16 1300 -> 1064 us (916 with nothing kept); h alone is as fast from the registers.
  // 16-byte chunks of a row are exchanged by its place among 16, which spreads a column's writes over the banks
  constexpr bool CUT = KEEP && MODE == MODE_BF16, STAGED = PHASED && CUT;
  constexpr int PITCH = CUT ? BN * 6 : 0;
  constexpr int PARTS = STAGED ? 2 : 1, MH = Cr::MI / PARTS, ROWS = WM * MH * 16;
  static_assert(!STAGED || (ROWS * PITCH <= Cr::LDS && PITCH % 256 == 0), "the rows of a part fit");
  auto place = [&](int row, int byte) { return smem + row * PITCH + (byte ^ (row & 15) << 4); };
#pragma unroll
  for (int part = 0; part < PARTS; ++part) {
  if (STAGED) __syncthreads();
#pragma unroll
  for (int ni = 0; ni < Cr::NI; ++ni) {
    const int jt = wn * (BN / WN) + 16 * ni + 4 * (lane >> 4), j = n0 + jt, n = a.H - j;
    f32x4 bg = {0.f, 0.f, 0.f, 0.f}, bu = {0.f, 0.f, 0.f, 0.f};
    if (a.bg && n > 0) bg = load4<MODE>(a.bg, j, n);
    if (a.bu && n > 0) bu = load4<MODE>(a.bu, j, n);
    f32x4 sg = {0.f, 0.f, 0.f, 0.f}, su = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int mi = part * MH; mi < (part + 1) * MH; ++mi) {
      const int64_t i = m0 + wm * (BM / WM) + 16 * mi + (lane & 15);
      const bool row = i < a.T;
      const f32x4 g = acc[0][mi][ni] + bg, u = acc[1][mi][ni] + bu;
      if (!BWD) {
        f32x4 h, p, z;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float s, d;
          activate<KEEP, MODE == MODE_F32>(a.act, g[r], s, d);
          h[r] = s * u[r];
          if (KEEP) { p[r] = d * u[r]; z[r] = s; }
        }
        if (row && n > 0) {
          const int q = wm * MH * 16 + 16 * (mi - part * MH) + (lane & 15);
          store4<MODE>(a.h, i * a.ldh + j, n, h);
          if constexpr (CUT) {
            u32x2 w[3];
            cut(p, z, w);
#pragma unroll
            for (int r = 0; r < 3; ++r) *(u32x2*)(STAGED ? place(q, jt * 6 + 8 * r) : (char*)a.kept + (i * a.Hp + j) * 6 + 8 * r) = w[r];
          } else if constexpr (KEEP) {
            float* o = (float*)a.kept + (i * a.Hp + j) * 2;
            *(f32x4*)o = p;
            *(f32x4*)(o + 4) = z;
          }
        }
      } else {
        f32x4 dg = {0.f, 0.f, 0.f, 0.f}, du = dg;
        if (row && n > 0) {
          const f32x4 dh = dhs[ni][mi];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float s, d;
            activate<true, MODE == MODE_F32>(a.act, g[r], s, d);
            dg[r] = r < n ? dh[r] * u[r] * d : 0.f;
            du[r] = r < n ? dh[r] * s : 0.f;
          }
        }
        sg += dg;
        su += du;
        if (row && j < a.Hp) {  // Hp is a multiple of 8: all four columns are inside, the ones behind H as zeros
          const int64_t o = i * a.Hp + j;
          store4<MODE>(a.dg, o, 4, dg);
          store4<MODE>(a.du, o, 4, du);
        }
      }
    }
    if (BWD && a.dbpart) {  // over the wave's rows: the 16 lanes of equal j
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
          sg[r] += __shfl_xor(sg[r], o, 64);
          su[r] += __shfl_xor(su[r], o, 64);
        }
      if ((lane & 15) == 0) {
        *(f32x4*)(sums + (wm * 2 + 0) * BN + jt) = sg;
        *(f32x4*)(sums + (wm * 2 + 1) * BN + jt) = su;
      }
    }
  }
  if (STAGED) {
    __syncthreads();
    constexpr int CHUNKS = STAGED ? PITCH / 16 : 1;
    for (int e = threadIdx.x; e < ROWS * CHUNKS; e += 64 * WM * WN) {
      const int q = e / CHUNKS, c = e % CHUNKS * 16;
      const int64_t i = m0 + q / (MH * 16) * (BM / WM) + part * MH * 16 + q % (MH * 16);
      if (i >= a.T) continue;
      if (n0 * 6 + c < a.Hp * 6) *(u32x4*)((char*)a.kept + (i * a.Hp + n0) * 6 + c) = *(const u32x4*)place(q, c);
    }
  }
  }
  if (BWD && a.dbpart) {
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * BN; c += Cr::THREADS) {
      const int w = c / BN, j = c % BN;
      if (n0 + j < a.H) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < WM; ++k) v += sums[(k * 2 + w) * BN + j];
        a.dbpart[((int64_t)tm * 2 + w) * a.H + n0 + j] = v;
      }
    }
  }
}

// ---- dg and du from what was kept --------------------------------------------------------------------------------------------------------
// Bound by its bytes: 12 a value in bf16, 20 in fp32.  A lane takes eight columns, a wave 512 of a row, a block 64 rows; four rows are
// requested before the first is used.
constexpr int KEPT_ROWS = 64;
struct KeptArgs {
  const void* kept; const void* dh; int64_t lddh;
  int64_t T; int H; int64_t Hp;
  void* dg; void* du;
  float* dbpart;
  int cols;  // blocks side by side
};
template <int MODE>
__global__ __launch_bounds__(256) void gated_kept_kernel(KeptArgs a) {
  constexpr int W = MODE == MODE_BF16 ? 3 : 4, U = 4;  // 16-byte words of eight columns; rows in flight
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), tile = blockIdx.x / a.cols, j = (blockIdx.x % a.cols * 64 + lane) * 8;
  const int64_t i0 = (int64_t)tile * KEPT_ROWS + wave;
  const int n = a.H - j;
  __shared__ __align__(16) float sums[2][4][512];
  float sg[8], su[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) sg[r] = su[r] = 0.f;
  if (n > 0)  // Hp ends less than eight columns behind H
    for (int q = 0; q < KEPT_ROWS / 4; q += U) {
      u32x4 w[U][W];
      f32x4 dh[U][2];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int64_t i = i0 + 4 * (q + k);
        if (i >= a.T) continue;
        const u32x4* src = (const u32x4*)((const char*)a.kept + (i * a.Hp + j) * (MODE == MODE_BF16 ? 6 : 8));
#pragma unroll
        for (int v = 0; v < W; ++v) w[k][v] = src[v];
        dh[k][0] = load4<MODE>(a.dh, i * a.lddh + j, n);
        dh[k][1] = load4<MODE>(a.dh, i * a.lddh + j + 4, n - 4);
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int64_t i = i0 + 4 * (q + k);
        if (i >= a.T) continue;
        float dg[8], du[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          float p, s;
          if constexpr (MODE == MODE_BF16) {
            const int at = r / 4 * 6 + r % 4 / 2, sh = 16 * (r & 1);
            const uint32_t l = w[k][(at + 4) / 4][(at + 4) % 4] >> sh;
            p = __builtin_bit_cast(float, (w[k][at / 4][at % 4] >> sh) << 16 | (l & 0xff) << 8);
            s = __builtin_bit_cast(float, (w[k][(at + 2) / 4][(at + 2) % 4] >> sh) << 16 | (l & 0xff00));
          } else {
            const uint32_t x = w[k][r / 4 * 2][r % 4], y = w[k][r / 4 * 2 + 1][r % 4];
            p = __builtin_bit_cast(float, x);
            s = __builtin_bit_cast(float, y);
          }
          const float t = dh[k][r / 4][r % 4];
          dg[r] = r < n ? t * p : 0.f;  // the columns behind H are zeros
          du[r] = r < n ? t * s : 0.f;
          sg[r] += dg[r];
          su[r] += du[r];
        }
        const int64_t o = i * a.Hp + j;
        store8<MODE>(a.dg, o, dg);
        store8<MODE>(a.du, o, du);
      }
    }
  if (a.dbpart) {  // the four waves' rows
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      sums[0][wave][lane * 8 + r] = sg[r];
      sums[1][wave][lane * 8 + r] = su[r];
    }
    __syncthreads();
    const int first = blockIdx.x % a.cols * 512;
    for (int c = threadIdx.x; c < 1024; c += 256) {
      const int t = c >> 9, col = c & 511;
      if (first + col < a.H)
        a.dbpart[((int64_t)tile * 2 + t) * a.H + first + col] = sums[t][0][col] + sums[t][1][col] + (sums[t][2][col] + sums[t][3][col]);
    }
  }
}

// ---- short rows in bf16: D <= 256 ----------------------------------------------------------------------------------------------------------
// With a sum this short a tile is mostly its start and its end.  So: a block keeps 64 columns of both weight matrices in LDS for its whole
// life, as fragments in the order of their reads, and its eight waves run over rows without meeting again: a wave loads 16 MI whole rows as
// they are (128 bytes of a row at a time), multiplies, and stores.  One launch, x read once a panel, nothing written but the result: rows off
// the 16-byte boundaries need no copy (131072 x 250 -> 256 71 us, copied and in tiles 94; 65536 x 100 -> 256 30 against 47); aligned ones
// take the tiles' time forward (131072 x 256 -> 256 61 us both, 2.2 TB/s) and steps up to 6 % less (333 against 347 us).
// (In fp32 the matrix instructions take sixteen times as long, and the tiles' start and end are nothing beside them.)
constexpr int PANEL = 64, SHORT_WAVES = 8, SHORT_ROW = 256;

struct ShortArgs {
  const void* x; int64_t ldx;
  const void* w[2]; int64_t ldw[2];
  const void* b[2];
  int64_t T, chunk;          // rows of a block: chunk, a multiple of 16 MI waves
  int D, H, act, panels, parts;
  void* h; int64_t ldh;      // forward
  const void* dh; int64_t lddh;  // backward, as MmaArgs
  void* dg; void* du; int64_t Hp;
  float* dbpart;             // [parts waves][2][H], or null
};

// 16 rows x 32 KS of k as fragments: a lane holds row lane % 16 (clamped to the last), 8 k's of every 32
// FULL: D = 32 KS, no chunk ends inside a row
template <int KS, bool FULL>
__device__ __forceinline__ void short_rows(const void* p, int64_t ld, int64_t row, int64_t rows, int D, s16x8 (&f)[KS]) {
  const int lane = threadIdx.x & 63, kl = 8 * (lane >> 4);
  int64_t r = row + (lane & 15);
  r = r < rows ? r : rows - 1;
#pragma unroll
  for (int k = 0; k < KS; ++k) f[k] = __builtin_bit_cast(s16x8, chunk16<MODE_BF16>(p, r * ld, 32 * k + kl, FULL ? 32 * KS + 8 : D));
}

template <bool BWD, int KS, int MI, bool FULL>
__global__ __launch_bounds__(64 * SHORT_WAVES) void gated_short_kernel(ShortArgs a) {
  constexpr int NF = PANEL / 16;
  __shared__ __align__(16) s16x8 panel[KS][2 * NF][64];
  __shared__ __align__(16) float bias[2][PANEL];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  // all panels of a part's rows on one XCD (blocks go to the XCDs in turn): its L2 serves the rows after the first
  const int x8 = blockIdx.x % 8, i8 = blockIdx.x / 8;
  const bool even = a.parts % 8 == 0;
  const int part = even ? x8 + 8 * (i8 / a.panels) : (int)blockIdx.x / a.panels, pan = even ? i8 % a.panels : (int)blockIdx.x % a.panels;
  const int n0 = pan * PANEL;
  {  // a wave: 16 columns of one of the matrices
    const int w = wave / NF, q = wave % NF;
    s16x8 f[KS];
    short_rows<KS, FULL>(a.w[w], a.ldw[w], n0 + 16 * q, a.H, a.D, f);
#pragma unroll
    for (int k = 0; k < KS; ++k) panel[k][wave][lane] = f[k];
    if (lane < 16) {
      const int j = n0 + 16 * q + lane;
      bias[w][16 * q + lane] = a.b[w] && j < a.H ? load1<MODE_BF16>(a.b[w], j) : 0.f;
    }
  }
  static_assert(SHORT_WAVES == 2 * NF, "a wave for each 16 columns of the panel");
  __syncthreads();
  const int jl = 4 * (lane >> 4);  // of 16 columns the lane's four
  f32x4 sum[2][BWD ? NF : 1];
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int f = 0; f < (BWD ? NF : 1); ++f) sum[w][f] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int64_t begin = part * a.chunk, end = begin + a.chunk < a.T ? begin + a.chunk : a.T;
  for (int64_t row = begin + wave * 16 * MI; row < end; row += SHORT_WAVES * 16 * MI) {
    s16x8 x[MI][KS];
#pragma unroll
    for (int m = 0; m < MI; ++m) {
      short_rows<KS, FULL>(a.x, a.ldx, row + 16 * m, a.T, a.D, x[m]);
      __builtin_amdgcn_sched_barrier(0);
    }
    f32x4 dhs[MI][BWD ? NF : 1];  // on their way while the products run
    if (BWD) {
#pragma unroll
      for (int m = 0; m < MI; ++m) {
        const int64_t i = row + 16 * m + (lane & 15);
#pragma unroll
        for (int f = 0; f < NF; ++f) {
          const int j = n0 + 16 * f + jl;
          dhs[m][BWD ? f : 0] = i < a.T && j < a.H ? load4<MODE_BF16>(a.dh, i * a.lddh + j, a.H - j) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
      }
    }
    f32x4 acc[2][MI][NF];
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int f = 0; f < NF; ++f) acc[w][m][f] = f32x4{0.f, 0.f, 0.f, 0.f};
    asm volatile("" ::: "memory");  // the panel is the same for every round: it would be hoisted out of the loop, into scratch
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        __builtin_amdgcn_sched_barrier(0);  // and read a matrix at a time
        s16x8 b[NF];
#pragma unroll
        for (int f = 0; f < NF; ++f) b[f] = panel[k][w * NF + f][lane];
#pragma unroll
        for (int m = 0; m < MI; ++m)
#pragma unroll
          for (int f = 0; f < NF; ++f) acc[w][m][f] = mfma<MODE_BF16>(b[f], x[m][k], acc[w][m][f]);
      }
#pragma unroll
    for (int m = 0; m < MI; ++m) {
      const int64_t i = row + 16 * m + (lane & 15);
      const bool live = i < a.T;
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const int j = n0 + 16 * f + jl, n = a.H - j;
        const f32x4 g = acc[0][m][f] + *(const f32x4*)&bias[0][16 * f + jl], u = acc[1][m][f] + *(const f32x4*)&bias[1][16 * f + jl];
        if (!BWD) {
          f32x4 h;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float s, d;
            activate<false, false>(a.act, g[r], s, d);
            h[r] = s * u[r];
          }
          if (live && n > 0) store4<MODE_BF16>(a.h, i * a.ldh + j, n, h);
        } else {
          f32x4 dg = {0.f, 0.f, 0.f, 0.f}, du = dg;
          if (live) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              float s, d;
              activate<true, false>(a.act, g[r], s, d);
              if (r < n) {
                dg[r] = dhs[m][BWD ? f : 0][r] * u[r] * d;
                du[r] = dhs[m][BWD ? f : 0][r] * s;
              }
            }
          }
          sum[0][BWD ? f : 0] += dg;
          sum[1][BWD ? f : 0] += du;
          if (live && j < a.Hp) {  // as the tiles' epilogue
            const int64_t o = i * a.Hp + j;
            store4<MODE_BF16>(a.dg, o, 4, dg);
            store4<MODE_BF16>(a.du, o, 4, du);
          }
        }
      }
    }
  }
  if (BWD && a.dbpart) {  // a wave's own column sums, over the 16 lanes of equal columns
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        f32x4 v = sum[w][BWD ? f : 0];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int o = 1; o < 16; o <<= 1) v[r] += __shfl_xor(v[r], o, 64);
        const int j = n0 + 16 * f + jl;
        if ((lane & 15) == 0 && j < a.H) store4<MODE_F32>(a.dbpart, (((int64_t)part * SHORT_WAVES + wave) * 2 + w) * a.H + j, a.H - j, v);
      }
  }
}

// ---- dx = dg Wg + du Wu (fp32, 65536 x 256 <- 512: 264 us, 130 TFLOP/s, the matrix cores 82 % busy) ----
struct DxArgs {
  const void* dg; const void* du; int64_t Hp;
  const void* wg; const void* wu; int64_t ldwg, ldwu;
  int64_t T; int H, D;
  void* dx;
  int64_t chunk; int splits;  // the sum over H is split, `chunk` each
  float* part;                // [split][T][D], where splits > 1
  int tm, tn;
};

template <int MODE, int BM, int BN, int WM, int WN, bool PHASED>
__global__ __launch_bounds__(64 * WM * WN) void gated_dx_kernel(DxArgs a) {
  using Cr = Core<MODE, KC, KS, BM, BN, 1, WM, WN>;
  __shared__ __align__(1024) char smem[Cr::LDS];
  const int per = a.tm * a.tn, sp = (int)(blockIdx.x / per);
  int tm, tn;
  tile_of(blockIdx.x % per, per, a.tm, a.tn, 8, tm, tn);
  const int64_t m0 = (int64_t)tm * BM, k0 = sp * a.chunk, ka = a.Hp - k0 < a.chunk ? a.Hp - k0 : a.chunk, kb = a.H - k0 < a.chunk ? a.H - k0 : a.chunk;
  const int n0 = tn * BN;
  typename Cr::Acc acc;
  Cr::zero(acc);
  const int64_t cols = (a.D + chunk_k<MODE>() - 1) / chunk_k<MODE>() * chunk_k<MODE>() - n0;
#pragma unroll 1
  for (int up = 0; up < 2; ++up) {
    const int64_t ld = up ? a.ldwu : a.ldwg;
    const Operand A = {element<MODE>(up ? a.du : a.dg, m0 * a.Hp + k0), 0, a.Hp, a.T - m0, ka};
    const Operand B[1] = {{element<MODE>(up ? a.wu : a.wg, k0 * ld + n0), 0, ld, cols, kb}};
    if constexpr (PHASED) Cr::run_phased(smem, A, B, acc);
    else Cr::run(smem, A, B, acc);
  }
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
#pragma unroll
  for (int mi = 0; mi < Cr::MI; ++mi) {
    const int64_t i = m0 + wm * (BM / WM) + 16 * mi + (lane & 15);
    if (i >= a.T) continue;
#pragma unroll
    for (int ni = 0; ni < Cr::NI; ++ni) {
      const int j = n0 + wn * (BN / WN) + 16 * ni + 4 * (lane >> 4);
      const f32x4 v = acc[0][mi][ni];
      if (j >= a.D) continue;
      if (a.splits == 1) store4<MODE>(a.dx, i * a.D + j, a.D - j, v);
      else store4<MODE_F32>(a.part, (sp * a.T + i) * a.D + j, a.D - j, v);
    }
  }
}

// ---- dWg = dg^T x, dWu = du^T x (fp32, the same layer: 256 us, 134 TFLOP/s, 85 % busy) ----
struct DwArgs {
  const void* d[2]; int64_t Hp;
  const void* x; int64_t ldx;
  int64_t T; int H, D;
  int64_t chunk; int splits;
  void* out[2];   // the results, where splits == 1
  float* part;    // [split][2][H][D], elsewhere
  int tm, tn;
};

template <int MODE, int BM, int BN, int WM, int WN, bool PHASED>
__global__ __launch_bounds__(64 * WM * WN) void gated_dw_kernel(DwArgs a) {
  using Cr = Core<MODE, KS, KS, BM, BN, 1, WM, WN>;
  __shared__ __align__(1024) char smem[Cr::LDS];
  const int per = a.tm * a.tn, sp = (int)(blockIdx.x / (2 * per)), rest = (int)(blockIdx.x % (2 * per)), w = rest / per;
  int tm, tn;
  tile_of(rest % per, per, a.tm, a.tn, 8, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  const int64_t t0 = (int64_t)sp * a.chunk, K = a.T - t0 < a.chunk ? a.T - t0 : a.chunk;
  typename Cr::Acc acc;
  Cr::zero(acc);
  const Operand A = {element<MODE>(a.d[w], t0 * a.Hp + m0), 0, a.Hp, a.Hp - m0, K};
  const Operand B[1] = {{element<MODE>(a.x, t0 * a.ldx + n0), 0, a.ldx, (a.D + chunk_k<MODE>() - 1) / chunk_k<MODE>() * chunk_k<MODE>() - n0, K}};
  if constexpr (PHASED) Cr::run_phased(smem, A, B, acc);
  else Cr::run(smem, A, B, acc);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
#pragma unroll
  for (int mi = 0; mi < Cr::MI; ++mi) {
    const int i = m0 + wm * (BM / WM) + 16 * mi + (lane & 15);
    if (i >= a.H) continue;
#pragma unroll
    for (int ni = 0; ni < Cr::NI; ++ni) {
      const int j = n0 + wn * (BN / WN) + 16 * ni + 4 * (lane >> 4);
      if (j >= a.D) continue;
      const f32x4 v = acc[0][mi][ni];
      if (a.splits == 1) store4<MODE>(a.out[w], (int64_t)i * a.D + j, a.D - j, v);
      else store4<MODE_F32>(a.part, (((int64_t)sp * 2 + w) * a.H + i) * a.D + j, a.D - j, v);
    }
  }
}

// ---- what is left: the parts of dx and dW in the order of their splits, the column sums of the bias gradients -----------------------------------
struct FinishArgs {
  const float* part[2]; int splits[2], sets[2]; int64_t n[2];  // dx, dW: `sets` results of n lie side by side in a split's part
  void* out[2][2];
  const float* db; int tiles, H;                               // [tiles][2][H]
  void* dbg; void* dbu;
  int first[3];                                                // first block of dW, of db; blocks
};
template <int MODE>
__global__ __launch_bounds__(256) void gated_finish_kernel(FinishArgs a) {
  const int id = blockIdx.x;
  if (id >= a.first[1]) {  // 16 columns, 16 interleaved chains each, joined in a fixed order
    const int cols = (a.H + 15) / 16, q = id - a.first[1], w = q / cols, c = threadIdx.x & 15, j = q % cols * 16 + c, t0 = threadIdx.x >> 4;
    __shared__ float s[16][16];
    float v = 0.f;
    if (j < a.H)
#pragma unroll 4
      for (int t = t0; t < a.tiles; t += 16) v += a.db[((int64_t)t * 2 + w) * a.H + j];
    s[t0][c] = v;
    __syncthreads();
    void* out = w ? a.dbu : a.dbg;
    if (t0 == 0 && j < a.H && out) {
#pragma unroll
      for (int k = 8; k > 0; k >>= 1)
#pragma unroll
        for (int i = 0; i < k; ++i) s[i][c] += s[i + k][c];
      store1<MODE>(out, j, s[0][c]);
    }
    return;
  }
  const int r = id >= a.first[0];
  const int64_t n = a.n[r], per = (n + 1023) / 1024, q = id - (r ? a.first[0] : 0), w = q / per, i = (q % per * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const int m = n - i < 4 ? (int)(n - i) : 4;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < a.splits[r]; ++s) v += load4<MODE_F32>(a.part[r], ((int64_t)s * a.sets[r] + w) * n + i, m);
  store4<MODE>(a.out[r][w], i, m, v);
}

// ---- few rows ------------------------------------------------------------------------------------------------------------------------------
// T <= 64: bound by the weights' bytes, which are read once, 16 a lane, as they are.
constexpr int ROWS_MAX = 64;
struct RowsArgs {
  const void* x; int64_t ldx;
  const void* w[2]; int64_t ldw[2];
  const void* b[2];
  void* h; int64_t ldh;
  int T, D, H, act;
};

// T <= 4: dot products, a wave computes NC columns of both projections for all rows, its lanes along k (4 x 4096 -> 8192 in bf16, 134 MB of
// weights: 26 us; one column a wave reads x as often as the weights and took 56)
template <int MODE, int NT, int NC>
__global__ __launch_bounds__(256) void gated_rows_kernel(RowsArgs a) {
  constexpr int N = chunk_k<MODE>();
  const int lane = threadIdx.x & 63, j0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * NC;
  if (j0 >= a.H) return;
  float s[2][NC][NT];
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int t = 0; t < NT; ++t) s[w][n][t] = 0.f;
  for (int c = lane * N; c < a.D; c += 64 * N) {
    u32x4 v[2][NC], x[NT];
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int w = 0; w < 2; ++w) v[w][n] = chunk16<MODE>(a.w[w], (j0 + n < a.H ? j0 + n : a.H - 1) * a.ldw[w], c, a.D);
#pragma unroll
    for (int t = 0; t < NT; ++t) x[t] = chunk16<MODE>(a.x, (t < a.T ? t : a.T - 1) * a.ldx, c, a.D);
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const float y = lane_value<MODE>(v[w][n], i);
#pragma unroll
          for (int t = 0; t < NT; ++t) s[w][n][t] = fmaf(y, lane_value<MODE>(x[t], i), s[w][n][t]);
        }
  }
  float g = 0.f, u = 0.f;  // lane n NT + t keeps column n of row t
#pragma unroll
  for (int n = 0; n < NC; ++n)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) s[w][n][t] += __shfl_xor(s[w][n][t], o, 64);
      if (lane == n * NT + t) {
        g = s[0][n][t];
        u = s[1][n][t];
      }
    }
  const int j = j0 + lane / NT, t = lane % NT;
  if (lane < NC * NT && j < a.H && t < a.T) {
    if (a.b[0]) g += load1<MODE>(a.b[0], j);
    if (a.b[1]) u += load1<MODE>(a.b[1], j);
    float f, d;
    activate<false, MODE == MODE_F32>(a.act, g, f, d);
    store1<MODE>(a.h, t * a.ldh + j, f * u);
  }
}

// 4 < T <= 64: 16 columns a block on the matrix cores (bf16: 16x16x32; fp32: 16x16x4, fp32 operands), the weights' chunks going straight from
// memory into the first operand's registers; the block's four waves take every fourth group of k, their sums meet in LDS.
// In fp32 a lane's four k's feed four instructions: k runs in another order, the same for both operands.
template <int MODE, int NB>
__global__ __launch_bounds__(256) void gated_few_kernel(RowsArgs a) {
  constexpr int N = chunk_k<MODE>(), STEP = 4 * N, U = 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j0 = blockIdx.x * 16, r = lane & 15, kl = (lane >> 4) * N;
  const int jr = j0 + r < a.H ? j0 + r : a.H - 1;
  f32x4 acc[2][NB];
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int n = 0; n < NB; ++n) acc[w][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int k0 = wave * STEP * U; k0 < a.D; k0 += 4 * STEP * U) {
    u32x4 v[U][2], x[U][NB];
#pragma unroll
    for (int i = 0; i < U; ++i) {
#pragma unroll
      for (int w = 0; w < 2; ++w) v[i][w] = chunk16<MODE>(a.w[w], jr * a.ldw[w], k0 + i * STEP + kl, a.D);
#pragma unroll
      for (int n = 0; n < NB; ++n) x[i][n] = chunk16<MODE>(a.x, (16 * n + r < a.T ? 16 * n + r : a.T - 1) * a.ldx, k0 + i * STEP + kl, a.D);
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          if (MODE == MODE_BF16) {
            acc[w][n] = mfma<MODE_BF16>(__builtin_bit_cast(s16x8, v[i][w]), __builtin_bit_cast(s16x8, x[i][n]), acc[w][n]);
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              acc[w][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(lane_value<MODE>(v[i][w], q), lane_value<MODE>(x[i][n], q), acc[w][n], 0, 0, 0);
          }
        }
  }
  __shared__ f32x4 part[3][2][NB][64];
  if (wave) {
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int n = 0; n < NB; ++n) part[wave - 1][w][n][lane] = acc[w][n];
  }
  __syncthreads();
  if (wave) return;
  const int j = j0 + 4 * (lane >> 4), n4 = a.H - j;  // a lane: four columns of row 16 n + r
  if (n4 <= 0) return;
  f32x4 bias[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) bias[w] = a.b[w] ? load4<MODE>(a.b[w], j, n4) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int t = 16 * n + r;
    f32x4 h;
#pragma unroll
    for (int w = 0; w < 2; ++w) acc[w][n] = ((acc[w][n] + part[0][w][n][lane]) + part[1][w][n][lane]) + part[2][w][n][lane] + bias[w];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float f, d;
      activate<false, MODE == MODE_F32>(a.act, acc[0][n][q], f, d);
      h[q] = f * acc[1][n][q];
    }
    if (t < a.T) store4<MODE>(a.h, t * a.ldh + j, n4, h);
  }
}

inline int ok() { return hipGetLastError() == hipSuccess ? HOLD_OK : HOLD_E_LAUNCH; }
inline int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
inline int64_t rows_grid(int64_t rows, int64_t most = 2048) {  // a row a wave; eight blocks a unit
  const int64_t b = (rows + 3) / 4;
  return b < 1 ? 1 : (b > most ? most : b);
}

// (bf16) Tiles of 256 rows, one block a compute unit, or of 128, two a unit: by the time of the launch in rounds over the 256 units.  The
// small tiles' lower rate (1135 against 1310 TFLOP/s at 4096^3, more LDS reads and loads a product) counts little against a part-filled
// round.  65536 x 1024 -> 2048: 493 against 574 us.  In fp32 the matrix instructions bound the tiles of 128 already.
bool large_tiles(int64_t n256, int64_t n128) {
  const double large = (double)((n256 + 255) / 256);
  double small = 0.58 * (double)((n128 + 511) / 512);
  if (n128 <= 512) small = 0.58 * (n128 <= 256 ? 0.68 : 1.);
  return large <= small;
}
// in the products with dg and du, two blocks a unit hide their ends behind each other's products where the sum is short
constexpr int64_t SHORT_SUM = 16;
inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// where everything of one call lies in its workspace (bytes; every part starts on a multiple of 256)
struct Plan {
  bool copy_x, copy_w[2];
  bool brief, big, little, keep, dx_big, dw_big;  // brief: the kernel for short rows; big, little: tiles of 256 and of 64 rows
  int64_t parts, part_rows;
  int64_t Dp, Hp, row_tiles;
  int64_t dx_splits, dx_chunk, dw_splits, dw_chunk;
  int64_t x, w, dg, dbpart, dx_sums, dw_sums, bytes;
};

bool aligned16(const void* p, int64_t ld, int es) { return (uintptr_t)p % 16 == 0 && (ld * es) % 16 == 0; }

// a sum over K is split until some 512 blocks of `tiles` tiles have work, each at least `least` long
void split_sum(int64_t tiles, int64_t K, int64_t least, int64_t& splits, int64_t& chunk) {
  int64_t s = tiles >= 384 ? 1 : cdiv(512, tiles);
  const int64_t most = cdiv(K, least);
  s = s > most ? most : s;
  chunk = up(cdiv(K, s), 64);
  splits = cdiv(K, chunk);
}

// Whether the forward pass keeps u act'(g) and act(g) where a backward one may follow.  Whole steps, kept against computed again: fp32
// 16384 x 768 -> 4096 5.24 against 6.54 ms, 65536 x 288 -> 512 1.38 against 1.58, 65536 x 256 -> 512 0.98 against 1.15, x 128 -> 512 0.63
// against 0.67; bf16 16384 x 2048 -> 8192 3.46 against 4.16 ms, 65536 x 640 -> 512 556 against 590 us, x 512 431 against 427; with less
// than some 2^21 values a step is its launches (700 x 1024 -> 1024 in fp32: 192 against 192 us).  Up to 256 features and 2^23 values
// the 8 bytes a value are not spent for the rest (70000 x 256 -> 48 in fp32: 239 against 264).  16384 x 8192 values are 0.8 GB in bf16, 1.1 in fp32
bool keeps(const hold_gated_desc& d) {
  const int64_t n = d.T * d.H;
  if (d.T <= ROWS_MAX || n < (1 << 21)) return false;
  return d.dtype == HOLD_GATED_F32 ? d.D > 256 || (d.D > 128 && n >= (1 << 23)) : d.D > 512;
}
int64_t kept_bytes(const hold_gated_desc& d) { return d.T * up(d.H, 8) * (d.dtype == HOLD_GATED_F32 ? 8 : 6); }

Plan plan(const hold_gated_desc& d, bool bwd) {
  Plan p = {};
  const bool f32 = d.dtype == HOLD_GATED_F32;
  const int es = f32 ? 4 : 2, step = f32 ? 32 : 64, whole = 16 / es;
  p.Dp = up(d.D, whole);
  p.Hp = up(d.H, 8);
  p.copy_x = d.D % whole || !aligned16(d.x, d.ldx, es);
  p.copy_w[0] = d.D % whole || !aligned16(d.w_gate, d.ldwg, es);
  p.copy_w[1] = d.D % whole || !aligned16(d.w_up, d.ldwu, es);
  int64_t o = 0;
  auto take = [&](int64_t bytes) { const int64_t at = o; o += up(bytes, 256); return at; };
  p.brief = !f32 && d.D <= SHORT_ROW;
  // some 256 blocks; a part's rows are whole rounds of its waves, and all panels of a part go to one XCD where the parts divide
  const int64_t panels = cdiv(d.H, PANEL), round = SHORT_WAVES * 16 * (bwd ? 1 : 2), rounds = cdiv(d.T, round);
  int64_t parts = cdiv(256, panels);
  parts = parts > rounds ? rounds : parts >= 8 ? (parts + 7) / 8 * 8 : parts;
  p.part_rows = cdiv(rounds, parts) * round;
  p.parts = cdiv(d.T, p.part_rows);
  p.big = !f32 && !bwd && large_tiles(cdiv(d.T, 256) * cdiv(d.H, 128), cdiv(d.T, 128) * cdiv(d.H, 64));
  // (backward: only for what is not kept, sums or results too short for large tiles)
  // up to half a block a unit of 128 x (64 + 64): tiles a quarter of that, four stages deep, their loads three steps ahead (2019 x 2816 ->
  // 32 in fp32: 180 -> 100 us; 1000 x 1000 -> 1000, 128 blocks: 72 -> 46, in bf16 17 -> 13; 2000 x 700 -> 600, 160: fp32 59 against 67, bf16
  // 25 against 32)
  p.little = !p.big && cdiv(d.T, 128) * cdiv(d.H, 64) <= 128;
  p.keep = d.kept != nullptr;
  p.row_tiles = p.keep ? cdiv(d.T, KEPT_ROWS) : p.brief ? p.parts * SHORT_WAVES : cdiv(d.T, p.big ? 256 : p.little ? 64 : 128);
  if (p.brief && !bwd) return p;  // takes everything as it is
  p.x = p.copy_x ? take(d.T * p.Dp * es) : 0;
  // (fp32 rows beyond the short ones: room for the weights' copies in any case, so that a call with weights of other strides finds it too)
  p.w = p.copy_w[0] || p.copy_w[1] || (f32 && d.D > SHORT_ROW) ? take(2 * (int64_t)d.H * p.Dp * es) : 0;
  if (bwd) {
    p.dg = take(2 * d.T * p.Hp * es);
    if (d.db_gate || d.db_up) p.dbpart = take(p.row_tiles * 2 * d.H * 4);
    const int64_t x256 = cdiv(d.T, 256) * cdiv(d.D, 256), x128 = cdiv(d.T, 128) * cdiv(d.D, 128);
    p.dx_big = !f32 && x256 >= 150 && 2 * cdiv(p.Hp, step) > SHORT_SUM && large_tiles(x256, x128);
    split_sum(p.dx_big ? 512 : x128, p.Hp, 512, p.dx_splits, p.dx_chunk);
    const int64_t w256 = 2 * cdiv(d.H, 256) * cdiv(d.D, 256), w128 = 2 * cdiv(d.H, 128) * cdiv(d.D, 128);
    p.dw_big = !f32 && w256 >= 200 && cdiv(d.T, step) > SHORT_SUM && large_tiles(w256, w128);
    split_sum(p.dw_big ? 512 : w128, d.T, 512, p.dw_splits, p.dw_chunk);
    if (p.dx_splits > 1) p.dx_sums = take(p.dx_splits * d.T * d.D * 4);
    if (p.dw_splits > 1) p.dw_sums = take(p.dw_splits * 2 * (int64_t)d.H * d.D * 4);
  }
  p.bytes = o;
  return p;
}

int check(const hold_gated_desc* d) {
  if (!d || !d->x || !d->w_gate || !d->w_up || d->T < 1 || d->D < 1 || d->H < 1 || d->act < 0 || d->act > 3) return HOLD_E_ARG;
  if (d->dtype != HOLD_GATED_F32 && d->dtype != HOLD_GATED_BF16) return HOLD_E_ARG;
  if (d->kept && (!keeps(*d) || (uintptr_t)d->kept % 16)) return HOLD_E_ARG;
  if (d->ldx < d->D || d->ldwg < d->D || d->ldwu < d->D) return HOLD_E_ARG;
  // the tile loads' 32-bit offsets: 256 rows of an operand, 64 rows of dg
  if (d->ldx > (1 << 21) || d->ldwg > (1 << 21) || d->ldwu > (1 << 21) || d->H > (1 << 21) || d->T > (1ll << 31)) return HOLD_E_ARG;
  // a launch has less than 2^32 threads: 512 a tile of 128 x 64 of h or dx, or of 128 x 128 of both weights' gradients
  if (((d->T + 127) / 128) * (((d->H > d->D ? d->H : d->D) + 63) / 64) >= (1ll << 23)) return HOLD_E_ARG;
  if (((int64_t)d->H + 127) / 128 * (((int64_t)d->D + 127) / 128) >= (1ll << 22)) return HOLD_E_ARG;
  return HOLD_OK;
}

template <int MODE>
void operands(const hold_gated_desc& d, const Plan& p, char* ws, hipStream_t st, MmaArgs& a) {
  a.x = d.x; a.ldx = d.ldx;
  a.wg = d.w_gate; a.ldwg = d.ldwg;
  a.wu = d.w_up; a.ldwu = d.ldwu;
  a.Hp = p.Hp;
  if (p.copy_x || p.copy_w[0] || p.copy_w[1]) {
    CopyArgs c = {};
    c.K = d.D; c.Kp = (int)p.Dp;
    int n = 0;
    auto add = [&](const void*& from, int64_t& ld, int64_t rows, char* to) {
      c.x[n] = from; c.ld[n] = ld; c.rows[n] = rows; c.out[n] = to;
      from = to;
      ld = p.Dp;
      ++n;
    };
    if (p.copy_x) add(a.x, a.ldx, d.T, ws + p.x);
    if (p.copy_w[0]) add(a.wg, a.ldwg, d.H, ws + p.w);
    if (p.copy_w[1]) add(a.wu, a.ldwu, d.H, ws + p.w + (int64_t)d.H * p.Dp * 2 * halves<MODE>());
    hipLaunchKernelGGL(gated_copy_rows_kernel<MODE>, dim3((unsigned)rows_grid(c.rows[0] + c.rows[1] + c.rows[2])), dim3(256), 0, st, c);
  }
  a.bg = d.b_gate; a.bu = d.b_up;
  a.T = d.T; a.H = d.H; a.K = (int)p.Dp; a.act = d.act;
}

template <bool BWD>
void launch_short(const hold_gated_desc& d, const MmaArgs& m, const Plan& p, hipStream_t st) {
  ShortArgs a = {};
  a.x = d.x; a.ldx = d.ldx;
  a.w[0] = d.w_gate; a.w[1] = d.w_up; a.ldw[0] = d.ldwg; a.ldw[1] = d.ldwu;
  a.b[0] = d.b_gate; a.b[1] = d.b_up;
  a.T = d.T; a.chunk = p.part_rows; a.D = d.D; a.H = d.H; a.act = d.act;
  a.panels = (int)cdiv(d.H, PANEL); a.parts = (int)p.parts;
  a.h = m.h; a.ldh = m.ldh;
  a.dh = m.dh; a.lddh = m.lddh;
  a.dg = m.dg; a.du = m.du; a.Hp = p.Hp;
  a.dbpart = m.dbpart;
  const dim3 grid((unsigned)(a.panels * p.parts)), block(64 * SHORT_WAVES);
  constexpr int MI = BWD ? 1 : 2;
  const int ks = (d.D + 31) / 32;
  const bool full = d.D % 64 == 0;
#define HOLD_SHORT(KS)                                                                                             \
  if (full) hipLaunchKernelGGL((gated_short_kernel<BWD, KS, MI, true>), grid, block, 0, st, a);               \
  else hipLaunchKernelGGL((gated_short_kernel<BWD, KS, MI, false>), grid, block, 0, st, a)
  if (ks <= 2) { HOLD_SHORT(2); }
  else if (ks <= 4) { HOLD_SHORT(4); }
  else if (ks <= 6) { HOLD_SHORT(6); }
  else { HOLD_SHORT(8); }
#undef HOLD_SHORT
}

template <int MODE, bool BWD>
void launch_mma(const hold_gated_desc& d, MmaArgs a, const Plan& p, hipStream_t st) {
  if (p.keep && BWD) {
    KeptArgs k = {};
    k.kept = d.kept; k.dh = d.dh; k.lddh = d.lddh;
    k.T = d.T; k.H = d.H; k.Hp = p.Hp;
    k.dg = a.dg; k.du = a.du;
    k.dbpart = a.dbpart;
    k.cols = (int)cdiv(d.H, 512);
    hipLaunchKernelGGL(gated_kept_kernel<MODE>, dim3((unsigned)(p.row_tiles * k.cols)), dim3(256), 0, st, k);
  } else if (p.keep) {
    a.kept = d.kept;
    const int t = p.big ? 256 : 128;
    a.tm = (int)cdiv(a.T, t); a.tn = (int)cdiv(a.H, t / 2);
    if constexpr (MODE == MODE_BF16) {
      if (p.big) hipLaunchKernelGGL((gated_mma_kernel<MODE, false, 256, 128, 4, 4, true, 2, true>), dim3((unsigned)(a.tm * a.tn)), dim3(1024), 0, st, a);
    }
    if (!p.big) hipLaunchKernelGGL((gated_mma_kernel<MODE, false, 128, 64, 4, 2, false, 2, true>), dim3((unsigned)(a.tm * a.tn)), dim3(512), 0, st, a);
  } else if (p.brief) {
    launch_short<BWD>(d, a, p, st);
  } else if (!BWD && p.big) {
    a.tm = (int)cdiv(a.T, 256); a.tn = (int)cdiv(a.H, 128);
    if constexpr (MODE == MODE_BF16)
      hipLaunchKernelGGL((gated_mma_kernel<MODE, false, 256, 128, 4, 4, true>), dim3((unsigned)(a.tm * a.tn)), dim3(1024), 0, st, a);
  } else if (p.little) {
    a.tm = (int)cdiv(a.T, 64); a.tn = (int)cdiv(a.H, 32);
    hipLaunchKernelGGL((gated_mma_kernel<MODE, BWD, 64, 32, 2, 1, false, 4>), dim3((unsigned)(a.tm * a.tn)), dim3(128), 0, st, a);
  } else {
    a.tm = (int)cdiv(a.T, 128); a.tn = (int)cdiv(a.H, 64);
    hipLaunchKernelGGL((gated_mma_kernel<MODE, BWD, 128, 64, 4, 2, false>), dim3((unsigned)(a.tm * a.tn)), dim3(512), 0, st, a);
  }
}

template <int MODE>
void rows(const hold_gated_desc& d, hipStream_t st) {
  RowsArgs a = {};
  a.x = d.x; a.ldx = d.ldx;
  a.w[0] = d.w_gate; a.w[1] = d.w_up; a.ldw[0] = d.ldwg; a.ldw[1] = d.ldwu;
  a.b[0] = d.b_gate; a.b[1] = d.b_up;
  a.h = d.h; a.ldh = d.ldh;
  a.T = (int)d.T; a.D = d.D; a.H = d.H; a.act = d.act;
  // four columns a wave where that still leaves two waves a SIMD, one elsewhere
#define HOLD_ROWS(NT, NC) hipLaunchKernelGGL((gated_rows_kernel<MODE, NT, NC>), dim3((unsigned)cdiv(d.H, 4 * NC)), dim3(256), 0, st, a)
#define HOLD_FEW(NB) hipLaunchKernelGGL((gated_few_kernel<MODE, NB>), dim3((unsigned)cdiv(d.H, 16)), dim3(256), 0, st, a)
  const bool wide = d.H >= 4096;
  if (d.T == 1) { if (wide) HOLD_ROWS(1, 4); else HOLD_ROWS(1, 1); }
  else if (d.T == 2) { if (wide) HOLD_ROWS(2, 4); else HOLD_ROWS(2, 1); }
  else if (d.T <= 4) { if (wide) HOLD_ROWS(4, 4); else HOLD_ROWS(4, 1); }
  else if (d.T <= 16) HOLD_FEW(1);
  else if (d.T <= 32) HOLD_FEW(2);
  else HOLD_FEW(4);
#undef HOLD_ROWS
#undef HOLD_FEW
}

template <int MODE>
int fwd(const hold_gated_desc& d, hipStream_t st) {
  if (d.T <= ROWS_MAX) {
    rows<MODE>(d, st);
    return ok();
  }
  const Plan p = plan(d, false);
  if (p.bytes > d.workspace_bytes || (p.bytes && !d.workspace)) return HOLD_E_ARG;
  MmaArgs a = {};
  if (!p.brief) operands<MODE>(d, p, (char*)d.workspace, st, a);
  a.h = d.h; a.ldh = d.ldh;
  launch_mma<MODE, false>(d, a, p, st);
  return ok();
}

template <int MODE>
int bwd(const hold_gated_desc& d, hipStream_t st) {
  const Plan p = plan(d, true);
  if (p.bytes > d.workspace_bytes || !d.workspace) return HOLD_E_ARG;
  char* ws = (char*)d.workspace;
  MmaArgs a = {};
  operands<MODE>(d, p, ws, st, a);
  a.dh = d.dh; a.lddh = d.lddh;
  a.dg = ws + p.dg; a.du = ws + p.dg + d.T * p.Hp * 2 * halves<MODE>();
  a.dbpart = d.db_gate || d.db_up ? (float*)(ws + p.dbpart) : nullptr;
  launch_mma<MODE, true>(d, a, p, st);
  FinishArgs f = {};
  if (d.dx) {
    DxArgs x = {};
    x.dg = a.dg; x.du = a.du; x.Hp = p.Hp;
    x.wg = a.wg; x.wu = a.wu; x.ldwg = a.ldwg; x.ldwu = a.ldwu;
    x.T = d.T; x.H = d.H; x.D = d.D;
    x.dx = d.dx; x.chunk = p.dx_chunk; x.splits = (int)p.dx_splits; x.part = (float*)(ws + p.dx_sums);
    const int t = p.dx_big ? 256 : 128;
    x.tm = (int)cdiv(d.T, t); x.tn = (int)cdiv(d.D, t);
    const unsigned blocks = (unsigned)(x.tm * x.tn * x.splits);
    if constexpr (MODE == MODE_BF16) {
      if (p.dx_big) hipLaunchKernelGGL((gated_dx_kernel<MODE, 256, 256, 4, 4, true>), dim3(blocks), dim3(1024), 0, st, x);
    }
    if (!p.dx_big) hipLaunchKernelGGL((gated_dx_kernel<MODE, 128, 128, 2, 4, false>), dim3(blocks), dim3(512), 0, st, x);
    if (x.splits > 1) {
      f.part[0] = x.part; f.splits[0] = x.splits; f.sets[0] = 1; f.n[0] = d.T * d.D;
      f.out[0][0] = d.dx;
      f.first[0] = (int)cdiv(f.n[0], 1024);
    }
  }
  if (d.dw_gate) {
    DwArgs w = {};
    w.d[0] = a.dg; w.d[1] = a.du; w.Hp = p.Hp;
    w.x = a.x; w.ldx = a.ldx;
    w.T = d.T; w.H = d.H; w.D = d.D;
    w.chunk = p.dw_chunk; w.splits = (int)p.dw_splits;
    w.out[0] = d.dw_gate; w.out[1] = d.dw_up; w.part = (float*)(ws + p.dw_sums);
    const int t = p.dw_big ? 256 : 128;
    w.tm = (int)cdiv(d.H, t); w.tn = (int)cdiv(d.D, t);
    const unsigned blocks = (unsigned)(2 * w.tm * w.tn * w.splits);
    if constexpr (MODE == MODE_BF16) {
      if (p.dw_big) hipLaunchKernelGGL((gated_dw_kernel<MODE, 256, 256, 4, 4, true>), dim3(blocks), dim3(1024), 0, st, w);
    }
    if (!p.dw_big) hipLaunchKernelGGL((gated_dw_kernel<MODE, 128, 128, 2, 4, false>), dim3(blocks), dim3(512), 0, st, w);
    if (w.splits > 1) {
      f.part[1] = w.part; f.splits[1] = w.splits; f.sets[1] = 2; f.n[1] = (int64_t)d.H * d.D;
      f.out[1][0] = d.dw_gate; f.out[1][1] = d.dw_up;
    }
  }
  f.first[1] = f.first[0] + (int)(2 * cdiv(f.n[1], 1024));
  f.first[2] = f.first[1];
  if (a.dbpart) {
    f.db = a.dbpart; f.tiles = (int)p.row_tiles; f.H = d.H; f.dbg = d.db_gate; f.dbu = d.db_up;
    f.first[2] += (int)(2 * cdiv(d.H, 16));
  }
  if (f.first[2]) hipLaunchKernelGGL(gated_finish_kernel<MODE>, dim3((unsigned)f.first[2]), dim3(256), 0, st, f);
  return ok();
}

}  // namespace

extern "C" int hold_gated_workspace(const hold_gated_desc* d, int32_t backward, int64_t* bytes) {
  if (check(d) != HOLD_OK || !bytes) return HOLD_E_ARG;
  *bytes = !backward && d->T <= ROWS_MAX ? 0 : plan(*d, backward != 0).bytes;
  return HOLD_OK;
}

extern "C" int hold_gated_kept(const hold_gated_desc* d, int64_t* bytes) {
  if (check(d) != HOLD_OK || !bytes) return HOLD_E_ARG;
  *bytes = keeps(*d) ? kept_bytes(*d) : 0;
  return HOLD_OK;
}

extern "C" int hold_gated_fwd(const hold_gated_desc* d, hold_stream_t st) {
  if (check(d) != HOLD_OK || !d->h || d->ldh < d->H) return HOLD_E_ARG;
  return d->dtype == HOLD_GATED_F32 ? fwd<MODE_F32>(*d, (hipStream_t)st) : fwd<MODE_BF16>(*d, (hipStream_t)st);
}

extern "C" int hold_gated_bwd(const hold_gated_desc* d, hold_stream_t st) {
  if (check(d) != HOLD_OK || !d->dh || d->lddh < d->H || (!d->dw_gate != !d->dw_up)) return HOLD_E_ARG;
  if (((uintptr_t)d->dx | (uintptr_t)d->dw_gate | (uintptr_t)d->dw_up) % 16) return HOLD_E_ARG;
  return d->dtype == HOLD_GATED_F32 ? bwd<MODE_F32>(*d, (hipStream_t)st) : bwd<MODE_BF16>(*d, (hipStream_t)st);
}
