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
// unrounded values.  gated_short_kernel: the same for D <= 256.  gated_kept_kernel: dg, du from what was kept.  gated_dx_kernel: [dg | du]
// times [Wg; Wu] as one sum.  gated_dw_kernel: both weight gradients, the sum over tokens split over blocks into fp32 partial tiles that
// gated_finish_kernel adds in a fixed order.  gated_rows_kernel, gated_few_kernel: T <= 4, T <= 64.
//
// ROUNDINGS.  bf16: dg and du are rounded to bf16 once, as the operands of the next matrix instructions; before, what is kept
// is cut to 24 bits, and everything else is fp32.
// fp32: every operand is split into two fp16 limbs (tile16.h) after an exact power-of-two scale: a row of x by its own largest
// magnitude; the two weight matrices by one exponent each (the same limbs serve the product over D and the one over H); a row of dg,
// du by a bound of its magnitude from the row maxima of x and dh and the weights' maximum (some log2 D bits above the typical value, of
// the 39 that the limbs span), du's 2^(eu - eg) times dg's, the ratio of the weight matrices' scales: so both halves of dx meet at one
// scale.  For dW the rows' scales are taken back on the x side: x_t 2^(R - r_t), R from the largest row.
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

template <int K>
__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
  for (int o = K / 2; o > 0; o >>= 1) {
    const int u = __shfl_xor(v, o, 64);
    v = u > v ? u : v;
  }
  return v;
}
__device__ __forceinline__ float wave_fmax(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}

constexpr int NPART = 256;  // blocks that look for the weights' maxima
// exponents kept by a backward call in fp32 (ints): [0] Wg, [1] Wu, [2] bg, [3] bu (exp_above of the largest magnitude, NONE of nothing),
// [4] R, [5] and [6] the exponents by which Wg and Wu are scaled (a matrix of zeros takes the other's)
constexpr int NONE = -100000;
__device__ __forceinline__ int exp_or_none(float m) { return m > 0.f ? exp_above(m) : NONE; }

// a wave's rows: 4 consecutive elements a lane, 256 a piece
__device__ __forceinline__ f32x4 row4(const float* p, int c, int K) { return load4<MODE_F16X3>(p, c, K - c); }

__device__ __forceinline__ float row_max(const float* p, int K) {
  const int lane = threadIdx.x & 63;
  float m = 0.f;
  for (int c = 4 * lane; c < K; c += 256) {
    const f32x4 v = row4(p, c, K);
#pragma unroll
    for (int r = 0; r < 4; ++r) m = fmaxf(m, finite_abs(v[r]));
  }
  return wave_fmax(m);
}

// largest finite magnitude of the weights and biases, per block of the grid: part[which][block]
__global__ __launch_bounds__(256) void gated_amax_kernel(const float* wg, int64_t ldg, const float* wu, int64_t ldu, const float* bg,
                                                         const float* bu, int H, int D, float* part) {
  const int which = blockIdx.y;
  float m = 0.f;
  if (which < 2) {
    const float* p = which ? wu : wg;
    const int64_t ld = which ? ldu : ldg;
    for (int r = blockIdx.x * 4 + (threadIdx.x >> 6); r < H; r += gridDim.x * 4) m = fmaxf(m, row_max(p + r * ld, D));
  } else {
    const float* p = which == 2 ? bg : bu;
    if (p)
      for (int c = blockIdx.x * 256 + threadIdx.x; c < H; c += gridDim.x * 256) m = fmaxf(m, finite_abs(p[c]));
    m = wave_fmax(m);
  }
  __shared__ float s[4];
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) part[which * NPART + blockIdx.x] = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
}

__device__ __forceinline__ float part_max(const float* part, int which) {  // every wave of a block by itself; NPART values
  const int lane = threadIdx.x & 63;
  const f32x4 v = *(const f32x4*)(part + which * NPART + 4 * lane);
  static_assert(NPART == 256, "four values a lane");
  return wave_fmax(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])));
}

// 4 scaled values as limbs; columns behind K up to Kp as zeros
__device__ __forceinline__ void put_limbs(uint16_t* o, int64_t limb, f32x4 v, int k) {
  Split y[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) y[r] = split16(ldexpf(v[r], k));
  *(u32x2*)o = u32x2{y[0].hi | (uint32_t)y[1].hi << 16, y[2].hi | (uint32_t)y[3].hi << 16};
  *(u32x2*)(o + limb) = u32x2{y[0].lo | (uint32_t)y[1].lo << 16, y[2].lo | (uint32_t)y[3].lo << 16};
}
// one row to limbs by 2^k
__device__ __forceinline__ void pack_row(const float* p, int K, int Kp, int k, uint16_t* o, int64_t limb) {
  const int lane = threadIdx.x & 63;
  for (int c = 4 * lane; c < Kp; c += 256) put_limbs(o + c, limb, row4(p, c, K), k);
}

struct PackArgs {
  const float* x; int64_t ldx, T;
  const float* w[2]; int64_t ldw[2];
  int H, D, Dp;
  uint16_t* ox; int64_t xlimb;  // null: x's rows are only measured
  uint16_t* ow; int64_t wlimb, second;
  int* rowexp;       // [T]
  int* colexp;       // [2][Hp]: the exponent of a weight row's scale
  int64_t Hp;
  // backward
  const float* part; // the weights' maxima: one scale a matrix, and the exponents below
  int* exps;
  const float* dh; int64_t lddh; int act;
  int* rscale; int* rpart;
};

// All rows to limbs [rows][Dp], a wave a row: x's scaled to [2^14, 2^15) by their own exponents, the weights' too (forward, where they only
// meet x) or by one a matrix (backward, where the sum also runs over H).  Backward: also the scale exponent r_t of a row of dg and du and
// the block's largest exponent of x_t 2^-r_t:
//   |g| <= D max|x_t| max|Wg| + max|bg|, |u| likewise; |act(g)| <= |g| (sigmoid: 1); |act'| < 2 (relu: 1, sigmoid: 1/4)
template <bool BWD>
__global__ __launch_bounds__(256) void gated_pack_kernel(PackArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int e[4] = {NONE, NONE, NONE, NONE}, ws[2] = {0, 0}, ld2 = 0, top = NONE;
  if (BWD) {
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = exp_or_none(part_max(a.part, i));
    ws[0] = e[0] != NONE ? e[0] : e[1] != NONE ? e[1] : 15;
    ws[1] = e[1] != NONE ? e[1] : e[0] != NONE ? e[0] : 15;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      a.exps[5] = ws[0];
      a.exps[6] = ws[1];
    }
    while ((1 << ld2) < a.D) ++ld2;
  }
  const int64_t rows = a.T + 2 * (int64_t)a.H;
  for (int64_t r = (int64_t)blockIdx.x * 4 + wave; r < rows; r += (int64_t)gridDim.x * 4) {
    if (r >= a.T) {
      const int w = r - a.T >= a.H, j = (int)(r - a.T) - w * a.H;
      const float* p = a.w[w] + j * a.ldw[w];
      int ex = BWD ? ws[w] : 0;
      if (!BWD) {
        ex = exp_or_none(row_max(p, a.D));
        ex = ex == NONE ? 15 : ex;
      }
      if (lane == 0) a.colexp[w * a.Hp + j] = ex;
      pack_row(p, a.D, a.Dp, 15 - ex, a.ow + w * a.second + (int64_t)j * a.Dp, a.wlimb);
      continue;
    }
    const float* p = a.x + r * a.ldx;
    uint16_t* o = a.ox + r * a.Dp;
    int ex;
    if (a.Dp <= 256) {  // the row stays in registers
      const f32x4 v = row4(p, 4 * lane, a.D);
      ex = exp_or_none(wave_fmax(fmaxf(fmaxf(finite_abs(v[0]), finite_abs(v[1])), fmaxf(finite_abs(v[2]), finite_abs(v[3])))));
      if (4 * lane < a.Dp && a.ox) put_limbs(o + 4 * lane, a.xlimb, v, ex == NONE ? 0 : 15 - ex);
    } else {
      ex = exp_or_none(row_max(p, a.D));
      if (a.ox) pack_row(p, a.D, a.Dp, ex == NONE ? 0 : 15 - ex, o, a.xlimb);
    }
    if (lane == 0) a.rowexp[r] = ex;
    if (BWD) {
      const int ed = exp_or_none(row_max(a.dh + r * a.lddh, a.H));
      auto proj = [&](int w) {  // exponent above a projection's magnitude
        const int m = (ex == NONE || e[w] == NONE) ? NONE : ex + e[w] + ld2, b = e[2 + w];
        return (m > b ? m : b) == NONE ? NONE : (m > b ? m : b) + 1;
      };
      const int eg = proj(0), eu = proj(1);
      const int ea = a.act == ACT_SIGMOID ? 0 : eg, edg = eu + (a.act == ACT_SIGMOID ? -2 : a.act == ACT_RELU ? 0 : 1);
      // r_t of dg such that dg 2^r_t and du 2^(r_t + shift) both stay below 2^15
      const int shift = ws[1] - ws[0], top2 = edg > ea + shift ? edg : ea + shift;
      const bool none = ed == NONE || top2 < -50000;
      const int k = none ? NONE : 15 - (ed + top2);
      if (lane == 0) a.rscale[r] = k;
      if (!none && ex != NONE && ex - k > top) top = ex - k;
    }
  }
  if (BWD) {
    __shared__ int s[4];
    if (lane == 0) s[wave] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
      const int u = s[0] > s[1] ? s[0] : s[1], v = s[2] > s[3] ? s[2] : s[3];
      a.rpart[blockIdx.x] = u > v ? u : v;
    }
  }
}

// x_t 2^(R - r_t) as limbs for the sum over tokens; rows without a gradient are zeros (where finite).  exps[4] = R
__global__ __launch_bounds__(256) void gated_pack_tokens_kernel(const float* x, int64_t ld, int64_t T, int D, int Dp, const int* rscale,
                                                                const int* part, int nparts, uint16_t* out, int64_t limb, int* exps) {
  const int lane = threadIdx.x & 63;
  __shared__ int tops[4];
  int top = NONE;
#pragma unroll 8
  for (int i = threadIdx.x; i < nparts; i += 256) top = part[i] > top ? part[i] : top;
  top = wave_max<64>(top);
  if (lane == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) top = tops[i] > top ? tops[i] : top;
  const int R = top == NONE ? 0 : 15 - top;
  if (blockIdx.x == 0 && threadIdx.x == 0) exps[4] = R;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < T; r += (int64_t)gridDim.x * 4) {
    const int k = rscale[r];
    for (int c = 4 * lane; c < Dp; c += 256) {
      f32x4 v = row4(x + r * ld, c, D);
      if (k == NONE) v *= 0.f;
      put_limbs(out + r * Dp + c, limb, v, k == NONE ? 0 : R - k);
    }
  }
}

// bf16 rows whose base, stride or length the tile loads cannot take -> [rows][Kp], zeros behind K; up to three matrices of equal length
struct CopyArgs {
  const uint16_t* x[3]; int64_t ld[3], rows[3];
  uint16_t* out[3];
  int K, Kp;
};
__global__ __launch_bounds__(256) void gated_copy_rows_kernel(CopyArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t all = a.rows[0] + a.rows[1] + a.rows[2];
  for (int64_t q = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); q < all; q += (int64_t)gridDim.x * 4) {
    const int w = q < a.rows[0] ? 0 : q < a.rows[0] + a.rows[1] ? 1 : 2;
    const int64_t r = q - (w > 0 ? a.rows[0] : 0) - (w > 1 ? a.rows[1] : 0);
    const uint16_t* p = a.x[w] + r * a.ld[w];
    uint16_t* o = a.out[w] + r * a.Kp;
    for (int c = 8 * lane; c < a.Kp; c += 512) *(u32x4*)(o + c) = chunk16<MODE_BF16>(p, 0, c, a.K);
  }
}

// ---- both projections and what follows them -------------------------------------------------------------------------------------------
struct MmaArgs {
  const uint16_t* x; int64_t ldx, xlimb;         // operands as the tile loads take them: [T][Dp]
  const uint16_t* wg; const uint16_t* wu; int64_t ldwg, ldwu, wlimb;
  const void* bg; const void* bu;
  int64_t T; int H; int K; int act;
  const int* rowexp; const int* colexp; const int* exps;  // fp32: the scales of x's rows, of the weights' rows; backward's exponents
  void* h; int64_t ldh;                          // forward
  const void* dh; int64_t lddh;                  // backward
  uint16_t* dg; uint16_t* du; int64_t Hp, dlimb; // [T][Hp] limbs of dg and du
  const int* rscale;
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
  const Operand A = {a.x + m0 * a.ldx, a.xlimb, a.ldx, a.T - m0, a.K};
  const Operand B[2] = {{a.wg + (int64_t)n0 * a.ldwg, a.wlimb, a.ldwg, a.H - n0, a.K}, {a.wu + (int64_t)n0 * a.ldwu, a.wlimb, a.ldwu, a.H - n0, a.K}};
  if constexpr (PHASED) Cr::run_phased(smem, A, B, acc);
  else Cr::run(smem, A, B, acc);

  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
  const int shift = MODE == MODE_F16X3 && BWD ? a.exps[6] - a.exps[5] : 0;
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
  // Where much is kept the tiles of 256 rows, alone on their unit, send bf16's p and s or fp32's h (fp32's p and s are whole lines as they
  // are) through LDS, half of each wave's rows at a time, so that whole lines leave: 16384 x 2048 -> 8192 in bf16 1300 -> 1064 us
  // (916 with nothing kept), 16384 x 768 -> 4096 in fp32 690 -> 632 (538).  h alone is as fast from the registers.  16-byte chunks of a
  // row are exchanged by its place among 16, which spreads a column's writes over the banks
  constexpr bool STAGED = PHASED && KEEP;
  constexpr bool CUT = KEEP && MODE == MODE_BF16, STAGED_H = STAGED && !CUT;
  constexpr int ES = MODE == MODE_BF16 ? 2 : 4, HB = STAGED_H ? BN * ES : 0, PITCH = HB + (CUT ? BN * 6 : 0);
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
    int eg[4] = {0, 0, 0, 0}, eu[4] = {0, 0, 0, 0};
    if (MODE == MODE_F16X3 && n > 0) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {  // [2][Hp]: four entries are inside
        eg[r] = a.colexp[j + r] - 15;
        eu[r] = a.colexp[a.Hp + j + r] - 15;
      }
    }
    f32x4 sg = {0.f, 0.f, 0.f, 0.f}, su = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int mi = part * MH; mi < (part + 1) * MH; ++mi) {
      const int64_t i = m0 + wm * (BM / WM) + 16 * mi + (lane & 15);
      const bool row = i < a.T;
      f32x4 g = acc[0][mi][ni], u = acc[1][mi][ni];
      if (MODE == MODE_F16X3) {
        const int e = row ? a.rowexp[i] : NONE, ex = e == NONE ? 0 : e - 15;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          g[r] = ldexpf(g[r], ex + eg[r]);
          u[r] = ldexpf(u[r], ex + eu[r]);
        }
      }
      g += bg;
      u += bu;
      if (!BWD) {
        f32x4 h, p, z;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float s, d;
          activate<KEEP, MODE == MODE_F16X3>(a.act, g[r], s, d);
          h[r] = s * u[r];
          if (KEEP) { p[r] = d * u[r]; z[r] = s; }
        }
        if (row && n > 0) {
          const int q = wm * MH * 16 + 16 * (mi - part * MH) + (lane & 15);
          if (STAGED_H) store4<MODE>(place(q, jt * ES), 0, 4, h);
          else store4<MODE>(a.h, i * a.ldh + j, n, h);
          if constexpr (CUT) {
            u32x2 w[3];
            cut(p, z, w);
#pragma unroll
            for (int r = 0; r < 3; ++r) *(u32x2*)(STAGED ? place(q, HB + jt * 6 + 8 * r) : (char*)a.kept + (i * a.Hp + j) * 6 + 8 * r) = w[r];
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
            activate<true, MODE == MODE_F16X3>(a.act, g[r], s, d);
            dg[r] = r < n ? dh[r] * u[r] * d : 0.f;
            du[r] = r < n ? dh[r] * s : 0.f;
          }
        }
        sg += dg;
        su += du;
        if (row && j < a.Hp) {  // Hp is a multiple of 8: all four columns are inside, the ones behind H as zeros
          const int64_t o = i * a.Hp + j;
          if (MODE == MODE_BF16) {
            store4<MODE>(a.dg, o, 4, dg);
            store4<MODE>(a.du, o, 4, du);
          } else {
            const int k = a.rscale[i] == NONE ? 0 : a.rscale[i], ku = a.rscale[i] == NONE ? 0 : k + shift;
            uint16_t hg[4], lg[4], hu[4], lu[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const Split x = split16(ldexpf(dg[r], k)), y = split16(ldexpf(du[r], ku));
              hg[r] = x.hi; lg[r] = x.lo; hu[r] = y.hi; lu[r] = y.lo;
            }
            auto pack = [](const uint16_t (&v)[4]) { return u32x2{v[0] | (uint32_t)v[1] << 16, v[2] | (uint32_t)v[3] << 16}; };
            *(u32x2*)(a.dg + o) = pack(hg);
            *(u32x2*)(a.dg + a.dlimb + o) = pack(lg);
            *(u32x2*)(a.du + o) = pack(hu);
            *(u32x2*)(a.du + a.dlimb + o) = pack(lu);
          }
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
    for (int e = threadIdx.x; e < ROWS * PITCH / 16; e += 64 * WM * WN) {
      const int q = e / (PITCH / 16), c = e % (PITCH / 16) * 16;
      const int64_t i = m0 + q / (MH * 16) * (BM / WM) + part * MH * 16 + q % (MH * 16);
      if (i >= a.T) continue;
      const u32x4 w = *(const u32x4*)place(q, c);
      if (c >= HB) {
        if (n0 * 6 + c - HB < a.Hp * 6) *(u32x4*)((char*)a.kept + (i * a.Hp + n0) * 6 + c - HB) = w;
      } else {
        const int j = n0 + c / ES;
        char* o = (char*)a.h + (i * a.ldh + j) * ES;
        if (a.H - j >= 16 / ES) {
          __builtin_memcpy(o, &w, 16);
        } else {
#pragma unroll
          for (int r = 0; r < 16 / ES; ++r) {
            const uint32_t v = w[r * ES / 4];
            if (j + r >= a.H) continue;
            if (ES == 4) ((uint32_t*)o)[r] = v;
            else ((uint16_t*)o)[r] = (uint16_t)(v >> 16 * (r & 1));
          }
        }
      }
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
  uint16_t* dg; uint16_t* du; int64_t dlimb;
  const int* rscale; const int* exps;
  float* dbpart;
  int cols;  // blocks side by side
};
template <int MODE>
__global__ __launch_bounds__(256) void gated_kept_kernel(KeptArgs a) {
  constexpr int W = MODE == MODE_BF16 ? 3 : 4, U = 4;  // 16-byte words of eight columns; rows in flight
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), tile = blockIdx.x / a.cols, j = (blockIdx.x % a.cols * 64 + lane) * 8;
  const int64_t i0 = (int64_t)tile * KEPT_ROWS + wave;
  const int n = a.H - j;
  const int shift = MODE == MODE_F16X3 ? a.exps[6] - a.exps[5] : 0;
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
        auto put = [&](uint16_t* to, const uint16_t (&v)[8]) {
          *(u32x4*)(to + o) = u32x4{v[0] | (uint32_t)v[1] << 16, v[2] | (uint32_t)v[3] << 16, v[4] | (uint32_t)v[5] << 16, v[6] | (uint32_t)v[7] << 16};
        };
        uint16_t g0[8], u0[8], g1[8], u1[8];
        const int e = MODE == MODE_F16X3 ? a.rscale[i] : 0, eg = e == NONE ? 0 : e, eu = e == NONE ? 0 : e + shift;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          if constexpr (MODE == MODE_BF16) {
            g0[r] = bf16_bits(dg[r]);
            u0[r] = bf16_bits(du[r]);
          } else {
            const Split x = split16(ldexpf(dg[r], eg)), y = split16(ldexpf(du[r], eu));
            g0[r] = x.hi; g1[r] = x.lo; u0[r] = y.hi; u1[r] = y.lo;
          }
        }
        put(a.dg, g0);
        put(a.du, u0);
        if constexpr (MODE != MODE_BF16) {
          put(a.dg + a.dlimb, g1);
          put(a.du + a.dlimb, u1);
        }
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

// ---- short rows: D <= 256 ------------------------------------------------------------------------------------------------------------------
// With a sum this short a tile is mostly its start and its end, and the limbs' way through memory costs as much as the layer.  So: a block
// keeps 64 columns of both weight matrices in LDS for its whole life, as fragments in the order of their reads, and its eight waves run
// over rows without meeting again: a wave loads 16 MI whole rows as they are (128 bytes of a row at a time), finds their scales and splits
// them in registers, multiplies, and stores.  One launch, x read once a panel, nothing written but the result.
// 131072 x 256 -> 256 in fp32: packing and tiles 177 us, this 124: 278 TFLOP/s (three products a term) and
// 2.2 TB/s, neither near its bound -- a wave's splits, products and activations take turns, and two waves share a SIMD.
constexpr int PANEL = 64, SHORT_WAVES = 8, SHORT_ROW = 256;

struct ShortArgs {
  const void* x; int64_t ldx;
  const void* w[2]; int64_t ldw[2];
  const void* b[2];
  int64_t T, chunk;          // rows of a block: chunk, a multiple of 16 MI waves
  int D, H, act, panels, parts;
  void* h; int64_t ldh;      // forward
  const void* dh; int64_t lddh;  // backward, as MmaArgs
  uint16_t* dg; uint16_t* du; int64_t Hp, dlimb;
  const int* rscale; const int* exps;
  float* dbpart;             // [parts waves][2][H], or null
};

// 16 rows x 32 KS of k as fragments: a lane holds row lane % 16 (clamped to the last), 8 k's of every 32.  fp32: scaled to [2^14, 2^15), `e` = the
// row's exponent, limbs; the largest magnitude ignores NaN, and a row with an infinity, scaled by 1, keeps infinities or NaN
// FULL: D = 32 KS, no chunk ends inside a row
template <int MODE, int KS, bool FULL>
__device__ __forceinline__ void short_rows(const void* p, int64_t ld, int64_t row, int64_t rows, int D, s16x8 (&f)[KS][limbs<MODE>()], int& e) {
  const int lane = threadIdx.x & 63, kl = 8 * (lane >> 4);
  int64_t r = row + (lane & 15);
  r = r < rows ? r : rows - 1;
  if constexpr (MODE == MODE_BF16) {
#pragma unroll
    for (int k = 0; k < KS; ++k) f[k][0] = __builtin_bit_cast(s16x8, chunk16<MODE_BF16>(p, r * ld, 32 * k + kl, FULL ? 32 * KS + 8 : D));
    e = 0;
  } else {
    u32x4 v[KS][2];
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int q = 0; q < 2; ++q) v[k][q] = chunk16<MODE_F16X3>(p, r * ld, 32 * k + kl + 4 * q, FULL ? 32 * KS + 8 : D);
    float m = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) m = fmaxf(m, fabsf(lane_value<MODE_F16X3>(v[k][q], i)));
    m = fmaxf(m, __shfl_xor(m, 16, 64));
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    e = m > 0.f && m < __builtin_inff() ? exp_above(m) : 15;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      u32x4 hi, lo;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float a = ldexpf(lane_value<MODE_F16X3>(v[k][q >> 1], 2 * (q & 1)), 15 - e), b = ldexpf(lane_value<MODE_F16X3>(v[k][q >> 1], 2 * (q & 1) + 1), 15 - e);
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        const f16x2 h = __builtin_convertvector(f32x2{a, b}, f16x2);
        const f16x2 l = __builtin_convertvector(f32x2{a - (float)h[0], b - (float)h[1]}, f16x2);
        hi[q] = __builtin_bit_cast(uint32_t, h);
        lo[q] = __builtin_bit_cast(uint32_t, l);
      }
      f[k][0] = __builtin_bit_cast(s16x8, hi);
      f[k][1] = __builtin_bit_cast(s16x8, lo);
    }
  }
}

template <int MODE, bool BWD, int KS, int MI, bool FULL>
__global__ __launch_bounds__(64 * SHORT_WAVES) void gated_short_kernel(ShortArgs a) {
  constexpr int NL = limbs<MODE>(), NF = PANEL / 16;
  __shared__ __align__(16) s16x8 panel[KS][2 * NF][NL][64];
  __shared__ __align__(16) int colexp[2][PANEL];
  __shared__ __align__(16) float bias[2][PANEL];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  // all panels of a part's rows on one XCD (blocks go to the XCDs in turn): its L2 serves the rows after the first
  const int x8 = blockIdx.x % 8, i8 = blockIdx.x / 8;
  const bool even = a.parts % 8 == 0;
  const int part = even ? x8 + 8 * (i8 / a.panels) : (int)blockIdx.x / a.panels, pan = even ? i8 % a.panels : (int)blockIdx.x % a.panels;
  const int n0 = pan * PANEL;
  {  // a wave: 16 columns of one of the matrices
    const int w = wave / NF, q = wave % NF;
    s16x8 f[KS][NL];
    int e;
    short_rows<MODE, KS, FULL>(a.w[w], a.ldw[w], n0 + 16 * q, a.H, a.D, f, e);
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int l = 0; l < NL; ++l) panel[k][wave][l][lane] = f[k][l];
    if (lane < 16) {
      const int j = n0 + 16 * q + lane;
      colexp[w][16 * q + lane] = e - 15;
      bias[w][16 * q + lane] = a.b[w] && j < a.H ? load1<MODE>(a.b[w], j) : 0.f;
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
  const int shift = MODE == MODE_F16X3 && BWD ? a.exps[6] - a.exps[5] : 0;
  const int64_t begin = part * a.chunk, end = begin + a.chunk < a.T ? begin + a.chunk : a.T;
  for (int64_t row = begin + wave * 16 * MI; row < end; row += SHORT_WAVES * 16 * MI) {
    s16x8 x[MI][KS][NL];
    int ex[MI];
#pragma unroll
    for (int m = 0; m < MI; ++m) {
      short_rows<MODE, KS, FULL>(a.x, a.ldx, row + 16 * m, a.T, a.D, x[m], ex[m]);
      __builtin_amdgcn_sched_barrier(0);
    }
    f32x4 dhs[MI][BWD ? NF : 1];  // on their way while the products run
    int rs[MI];
    if (BWD) {
#pragma unroll
      for (int m = 0; m < MI; ++m) {
        const int64_t i = row + 16 * m + (lane & 15);
#pragma unroll
        for (int f = 0; f < NF; ++f) {
          const int j = n0 + 16 * f + jl;
          dhs[m][BWD ? f : 0] = i < a.T && j < a.H ? load4<MODE>(a.dh, i * a.lddh + j, a.H - j) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
        rs[m] = MODE == MODE_F16X3 ? (i < a.T ? a.rscale[i] : NONE) : 0;
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
        s16x8 b[NF][NL];
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
          for (int l = 0; l < NL; ++l) b[f][l] = panel[k][w * NF + f][l][lane];
#pragma unroll
        for (int p = NL == 2 ? 0 : 2; p < 3; ++p)
#pragma unroll
          for (int m = 0; m < MI; ++m)
#pragma unroll
            for (int f = 0; f < NF; ++f) acc[w][m][f] = mfma<MODE>(b[f][p == 0 ? NL - 1 : 0], x[m][k][p == 1 ? NL - 1 : 0], acc[w][m][f]);
      }
#pragma unroll
    for (int m = 0; m < MI; ++m) {
      const int64_t i = row + 16 * m + (lane & 15);
      const bool live = i < a.T;
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const int j = n0 + 16 * f + jl, n = a.H - j;
        f32x4 g = acc[0][m][f], u = acc[1][m][f];
        if (MODE == MODE_F16X3) {
          const int4 cg = *(const int4*)&colexp[0][16 * f + jl], cu = *(const int4*)&colexp[1][16 * f + jl];
          const int e0 = ex[m] - 15;
          g = f32x4{ldexpf(g[0], e0 + cg.x), ldexpf(g[1], e0 + cg.y), ldexpf(g[2], e0 + cg.z), ldexpf(g[3], e0 + cg.w)};
          u = f32x4{ldexpf(u[0], e0 + cu.x), ldexpf(u[1], e0 + cu.y), ldexpf(u[2], e0 + cu.z), ldexpf(u[3], e0 + cu.w)};
        }
        g += *(const f32x4*)&bias[0][16 * f + jl];
        u += *(const f32x4*)&bias[1][16 * f + jl];
        if (!BWD) {
          f32x4 h;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float s, d;
            activate<false, MODE == MODE_F16X3>(a.act, g[r], s, d);
            h[r] = s * u[r];
          }
          if (live && n > 0) store4<MODE>(a.h, i * a.ldh + j, n, h);
        } else {
          f32x4 dg = {0.f, 0.f, 0.f, 0.f}, du = dg;
          if (live) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              float s, d;
              activate<true, MODE == MODE_F16X3>(a.act, g[r], s, d);
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
            if (MODE == MODE_BF16) {
              store4<MODE>(a.dg, o, 4, dg);
              store4<MODE>(a.du, o, 4, du);
            } else {
              put_limbs(a.dg + o, a.dlimb, dg, rs[m] == NONE ? 0 : rs[m]);
              put_limbs(a.du + o, a.dlimb, du, rs[m] == NONE ? 0 : rs[m] + shift);
            }
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
        if ((lane & 15) == 0 && j < a.H) store4<MODE_F16X3>(a.dbpart, (((int64_t)part * SHORT_WAVES + wave) * 2 + w) * a.H + j, a.H - j, v);
      }
  }
}

// ---- dx = dg Wg + du Wu -----------------------------------------------------------------------------------------------------------------
struct DxArgs {
  const uint16_t* dg; const uint16_t* du; int64_t Hp, dlimb;
  const uint16_t* wg; const uint16_t* wu; int64_t ldwg, ldwu, wlimb;
  int64_t T; int H, D;
  const int* rscale; const int* exps;
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
  const int64_t cols = (a.D + 7) / 8 * 8 - n0;
#pragma unroll 1
  for (int up = 0; up < 2; ++up) {
    const int64_t ld = up ? a.ldwu : a.ldwg;
    const Operand A = {(up ? a.du : a.dg) + m0 * a.Hp + k0, a.dlimb, a.Hp, a.T - m0, ka};
    const Operand B[1] = {{(up ? a.wu : a.wg) + k0 * ld + n0, a.wlimb, ld, cols, kb}};
    if constexpr (PHASED) Cr::run_phased(smem, A, B, acc);
    else Cr::run(smem, A, B, acc);
  }
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
  const int ew = MODE == MODE_F16X3 ? a.exps[5] - 15 : 0;
#pragma unroll
  for (int mi = 0; mi < Cr::MI; ++mi) {
    const int64_t i = m0 + wm * (BM / WM) + 16 * mi + (lane & 15);
    if (i >= a.T) continue;
    const int k = MODE == MODE_F16X3 ? (a.rscale[i] == NONE ? ew : ew - a.rscale[i]) : 0;
#pragma unroll
    for (int ni = 0; ni < Cr::NI; ++ni) {
      const int j = n0 + wn * (BN / WN) + 16 * ni + 4 * (lane >> 4);
      f32x4 v = acc[0][mi][ni];
      if (MODE == MODE_F16X3)
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = ldexpf(v[r], k);
      if (j >= a.D) continue;
      if (a.splits == 1) store4<MODE>(a.dx, i * a.D + j, a.D - j, v);
      else store4<MODE_F16X3>(a.part, (sp * a.T + i) * a.D + j, a.D - j, v);
    }
  }
}

// ---- dWg = dg^T x, dWu = du^T x -----------------------------------------------------------------------------------------------------------
struct DwArgs {
  const uint16_t* d[2]; int64_t Hp, dlimb;
  const uint16_t* x; int64_t ldx, xlimb;
  int64_t T; int H, D;
  int64_t chunk; int splits;
  const int* exps;
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
  const Operand A = {a.d[w] + t0 * a.Hp + m0, a.dlimb, a.Hp, a.Hp - m0, K};
  const Operand B[1] = {{a.x + t0 * a.ldx + n0, a.xlimb, a.ldx, (a.D + 7) / 8 * 8 - n0, K}};
  if constexpr (PHASED) Cr::run_phased(smem, A, B, acc);
  else Cr::run(smem, A, B, acc);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
  const int e = MODE == MODE_F16X3 ? -a.exps[4] - (w ? a.exps[6] - a.exps[5] : 0) : 0;
#pragma unroll
  for (int mi = 0; mi < Cr::MI; ++mi) {
    const int i = m0 + wm * (BM / WM) + 16 * mi + (lane & 15);
    if (i >= a.H) continue;
#pragma unroll
    for (int ni = 0; ni < Cr::NI; ++ni) {
      const int j = n0 + wn * (BN / WN) + 16 * ni + 4 * (lane >> 4);
      if (j >= a.D) continue;
      f32x4 v = acc[0][mi][ni];
      if (MODE == MODE_F16X3)
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = ldexpf(v[r], e);
      if (a.splits == 1) store4<MODE>(a.out[w], (int64_t)i * a.D + j, a.D - j, v);
      else store4<MODE_F16X3>(a.part, (((int64_t)sp * 2 + w) * a.H + i) * a.D + j, a.D - j, v);
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
  for (int s = 0; s < a.splits[r]; ++s) v += load4<MODE_F16X3>(a.part[r], ((int64_t)s * a.sets[r] + w) * n + i, m);
  store4<MODE>(a.out[r][w], i, m, v);
}

// ---- few rows ------------------------------------------------------------------------------------------------------------------------------
// T <= 64: bound by the weights' bytes, which are read once, 16 a lane, as they are; no product of limbs, fp32 keeps fp32 arithmetic.
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
    activate<false, MODE == MODE_F16X3>(a.act, g, f, d);
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
      activate<false, MODE == MODE_F16X3>(a.act, acc[0][n][q], f, d);
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

// Tiles of 256 rows, one block a compute unit, or of 128, two a unit: by the time of the launch in rounds over the 256 units.  The small
// tiles' lower rate (1135 against 1310 TFLOP/s at 4096^3, more LDS reads and loads a product) counts little against a part-filled round.
// Sums of 5 to 16 steps: 65536 x 384 -> 512 in fp32 200 against 219 us, 65536 x 1024 -> 2048 in bf16 493 against 574.
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
  int64_t Dp, Hp, row_tiles, pack_blocks;
  int64_t dx_splits, dx_chunk, dw_splits, dw_chunk;
  int64_t x, w, dg, xt, part, exps, rowexp, colexp, rscale, dbpart, dx_sums, dw_sums, spart, bytes;
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
// 16384 x 768 -> 4096 2.35 against 3.0 ms, 65536 x 264 -> 512 0.94 against 1.03, in the kernel for short rows no less; bf16 16384 x
// 2048 -> 8192 3.46 against 4.16 ms, 65536 x 640 -> 512 556 against 590 us, x 512 431 against 427; with less than some 2^21 values a step
// is its launches (700 x 1024 -> 1024 in fp32: 165 against 161 us).  16384 x 8192 values are 0.8 GB in bf16, 1.1 in fp32
bool keeps(const hold_gated_desc& d) {
  return d.T > ROWS_MAX && d.T * d.H >= (1 << 21) && d.D > (d.dtype == HOLD_GATED_F32 ? SHORT_ROW : 512);
}
int64_t kept_bytes(const hold_gated_desc& d) { return d.T * up(d.H, 8) * (d.dtype == HOLD_GATED_F32 ? 8 : 6); }

Plan plan(const hold_gated_desc& d, bool bwd) {
  Plan p = {};
  const bool f32 = d.dtype == HOLD_GATED_F32;
  const int nl = f32 ? 2 : 1, step = f32 ? 32 : 64;
  p.Dp = up(d.D, 8);
  p.Hp = up(d.H, 8);
  p.copy_x = f32 || d.D % 8 || !aligned16(d.x, d.ldx, 2);
  p.copy_w[0] = f32 || d.D % 8 || !aligned16(d.w_gate, d.ldwg, 2);
  p.copy_w[1] = f32 || d.D % 8 || !aligned16(d.w_up, d.ldwu, 2);
  int64_t o = 0;
  auto take = [&](int64_t bytes) { const int64_t at = o; o += up(bytes, 256); return at; };
  p.brief = d.D <= SHORT_ROW;
  // some 256 blocks; a part's rows are whole rounds of its waves, and all panels of a part go to one XCD where the parts divide
  const int64_t panels = cdiv(d.H, PANEL), round = SHORT_WAVES * 16 * (bwd ? 1 : 2), rounds = cdiv(d.T, round);
  int64_t parts = cdiv(256, panels);
  parts = parts > rounds ? rounds : parts >= 8 ? (parts + 7) / 8 * 8 : parts;
  p.part_rows = cdiv(rounds, parts) * round;
  p.parts = cdiv(d.T, p.part_rows);
  p.big = !bwd && large_tiles(cdiv(d.T, 256) * cdiv(d.H, 128), cdiv(d.T, 128) * cdiv(d.H, 64));
  // (backward: only for what is not kept, sums or results too short for large tiles)
  // up to half a block a unit of 128 x (64 + 64): tiles a quarter of that, four stages deep, their loads three steps ahead (2019 x 2816 ->
  // 32 in fp32: 80.9 -> 57.0 us; 1000 x 1000 -> 1000, 128 blocks: 39 -> 32, in bf16 17 -> 13; 2000 x 700 -> 600, 160: 25 against 32)
  p.little = !p.big && cdiv(d.T, 128) * cdiv(d.H, 64) <= 128;
  p.keep = d.kept != nullptr;
  p.row_tiles = p.keep ? cdiv(d.T, KEPT_ROWS) : p.brief ? p.parts * SHORT_WAVES : cdiv(d.T, p.big ? 256 : p.little ? 64 : 128);
  p.pack_blocks = rows_grid(d.T + 2 * (int64_t)d.H, 4096);
  if (p.brief && !bwd) return p;  // takes everything as it is
  p.x = p.copy_x && !(f32 && (p.brief || (p.keep && bwd))) ? take(d.T * p.Dp * 2 * nl) : 0;
  p.w = p.copy_w[0] || p.copy_w[1] ? take(2 * (int64_t)d.H * p.Dp * 2 * nl) : 0;
  if (f32) {
    p.rowexp = take(d.T * 4);
    p.colexp = take(2 * p.Hp * 4);
  }
  if (bwd) {
    p.dg = take(2 * d.T * p.Hp * 2 * nl);
    if (f32) {
      p.part = take(4 * NPART * 4);
      p.exps = take(8 * 4);
      p.xt = take(d.T * p.Dp * 2 * nl);
      p.rscale = take(d.T * 4);
      p.spart = take(p.pack_blocks * 4);
    }
    if (d.db_gate || d.db_up) p.dbpart = take(p.row_tiles * 2 * d.H * 4);
    const int64_t x256 = cdiv(d.T, 256) * cdiv(d.D, 256), x128 = cdiv(d.T, 128) * cdiv(d.D, 128);
    p.dx_big = x256 >= 150 && 2 * cdiv(p.Hp, step) > SHORT_SUM && large_tiles(x256, x128);
    split_sum(p.dx_big ? 512 : x128, p.Hp, 512, p.dx_splits, p.dx_chunk);
    const int64_t w256 = 2 * cdiv(d.H, 256) * cdiv(d.D, 256), w128 = 2 * cdiv(d.H, 128) * cdiv(d.D, 128);
    p.dw_big = w256 >= 200 && cdiv(d.T, step) > SHORT_SUM && large_tiles(w256, w128);
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

template <int MODE, bool BWD>
void operands(const hold_gated_desc& d, const Plan& p, char* ws, hipStream_t st, MmaArgs& a) {
  const int64_t WX = d.T * p.Dp, WW = (int64_t)d.H * p.Dp;
  a.x = (const uint16_t*)d.x; a.ldx = d.ldx; a.xlimb = 0;
  a.wg = (const uint16_t*)d.w_gate; a.ldwg = d.ldwg;
  a.wu = (const uint16_t*)d.w_up; a.ldwu = d.ldwu; a.wlimb = 0;
  a.Hp = p.Hp;
  if (MODE == MODE_F16X3) {
    PackArgs k = {};
    k.x = (const float*)d.x; k.ldx = d.ldx; k.T = d.T;
    k.w[0] = (const float*)d.w_gate; k.w[1] = (const float*)d.w_up; k.ldw[0] = d.ldwg; k.ldw[1] = d.ldwu;
    k.H = d.H; k.D = d.D; k.Dp = (int)p.Dp;
    k.ox = p.brief || (p.keep && BWD) ? nullptr : (uint16_t*)(ws + p.x); k.xlimb = WX;
    k.ow = (uint16_t*)(ws + p.w); k.wlimb = 2 * WW; k.second = WW;
    k.rowexp = (int*)(ws + p.rowexp); k.colexp = (int*)(ws + p.colexp); k.Hp = p.Hp;
    if (BWD) {
      float* part = (float*)(ws + p.part);
      k.part = part; k.exps = (int*)(ws + p.exps);
      k.dh = (const float*)d.dh; k.lddh = d.lddh; k.act = d.act;
      k.rscale = (int*)(ws + p.rscale); k.rpart = (int*)(ws + p.spart);
      hipLaunchKernelGGL(gated_amax_kernel, dim3(NPART, 4), dim3(256), 0, st, k.w[0], d.ldwg, k.w[1], d.ldwu, (const float*)d.b_gate,
                         (const float*)d.b_up, d.H, d.D, part);
      a.exps = k.exps;
      a.rscale = k.rscale;
    }
    hipLaunchKernelGGL(gated_pack_kernel<BWD>, dim3((unsigned)p.pack_blocks), dim3(256), 0, st, k);
    a.x = k.ox; a.ldx = p.Dp; a.xlimb = WX;
    a.wg = k.ow; a.wu = k.ow + WW; a.ldwg = a.ldwu = p.Dp; a.wlimb = 2 * WW;
    a.rowexp = k.rowexp; a.colexp = k.colexp;
  } else if (p.copy_x || p.copy_w[0] || p.copy_w[1]) {
    CopyArgs c = {};
    c.K = d.D; c.Kp = (int)p.Dp;
    int n = 0;
    auto add = [&](const void* from, int64_t ld, int64_t rows, uint16_t* to) {
      c.x[n] = (const uint16_t*)from; c.ld[n] = ld; c.rows[n] = rows; c.out[n] = to;
      ++n;
    };
    uint16_t* w = (uint16_t*)(ws + p.w);
    if (p.copy_x) { add(d.x, d.ldx, d.T, (uint16_t*)(ws + p.x)); a.x = c.out[n - 1]; a.ldx = p.Dp; }
    if (p.copy_w[0]) { add(d.w_gate, d.ldwg, d.H, w); a.wg = w; a.ldwg = p.Dp; }
    if (p.copy_w[1]) { add(d.w_up, d.ldwu, d.H, w + WW); a.wu = w + WW; a.ldwu = p.Dp; }
    hipLaunchKernelGGL(gated_copy_rows_kernel, dim3((unsigned)rows_grid(c.rows[0] + c.rows[1] + c.rows[2])), dim3(256), 0, st, c);
  }
  a.bg = d.b_gate; a.bu = d.b_up;
  a.T = d.T; a.H = d.H; a.K = (int)p.Dp; a.act = d.act;
}

template <int MODE, bool BWD>
void launch_short(const hold_gated_desc& d, const MmaArgs& m, const Plan& p, hipStream_t st) {
  ShortArgs a = {};
  a.x = d.x; a.ldx = d.ldx;
  a.w[0] = d.w_gate; a.w[1] = d.w_up; a.ldw[0] = d.ldwg; a.ldw[1] = d.ldwu;
  a.b[0] = d.b_gate; a.b[1] = d.b_up;
  a.T = d.T; a.chunk = p.part_rows; a.D = d.D; a.H = d.H; a.act = d.act;
  a.panels = (int)cdiv(d.H, PANEL); a.parts = (int)p.parts;
  a.h = m.h; a.ldh = m.ldh;
  a.dh = m.dh; a.lddh = m.lddh;
  a.dg = m.dg; a.du = m.du; a.Hp = p.Hp; a.dlimb = m.dlimb;
  a.rscale = m.rscale; a.exps = m.exps; a.dbpart = m.dbpart;
  const dim3 grid((unsigned)(a.panels * p.parts)), block(64 * SHORT_WAVES);
  constexpr int MI = BWD ? 1 : 2;
  const int ks = (d.D + 31) / 32;
  const bool full = d.D % 64 == 0;
#define HOLD_SHORT(KS)                                                                                             \
  if (full) hipLaunchKernelGGL((gated_short_kernel<MODE, BWD, KS, MI, true>), grid, block, 0, st, a);               \
  else hipLaunchKernelGGL((gated_short_kernel<MODE, BWD, KS, MI, false>), grid, block, 0, st, a)
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
    k.dg = a.dg; k.du = a.du; k.dlimb = a.dlimb;
    k.rscale = a.rscale; k.exps = a.exps; k.dbpart = a.dbpart;
    k.cols = (int)cdiv(d.H, 512);
    hipLaunchKernelGGL(gated_kept_kernel<MODE>, dim3((unsigned)(p.row_tiles * k.cols)), dim3(256), 0, st, k);
  } else if (p.keep) {
    a.kept = d.kept;
    const int t = p.big ? 256 : 128;
    a.tm = (int)cdiv(a.T, t); a.tn = (int)cdiv(a.H, t / 2);
    if (p.big) hipLaunchKernelGGL((gated_mma_kernel<MODE, false, 256, 128, 4, 4, true, 2, true>), dim3((unsigned)(a.tm * a.tn)), dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((gated_mma_kernel<MODE, false, 128, 64, 4, 2, false, 2, true>), dim3((unsigned)(a.tm * a.tn)), dim3(512), 0, st, a);
  } else if (p.brief) {
    launch_short<MODE, BWD>(d, a, p, st);
  } else if (!BWD && p.big) {
    a.tm = (int)cdiv(a.T, 256); a.tn = (int)cdiv(a.H, 128);
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
  if (!p.brief) operands<MODE, false>(d, p, (char*)d.workspace, st, a);
  a.h = d.h; a.ldh = d.ldh;
  launch_mma<MODE, false>(d, a, p, st);
  return ok();
}

template <int MODE>
int bwd(const hold_gated_desc& d, hipStream_t st) {
  const Plan p = plan(d, true);
  if (p.bytes > d.workspace_bytes || !d.workspace) return HOLD_E_ARG;
  char* ws = (char*)d.workspace;
  constexpr bool F32 = MODE == MODE_F16X3;
  constexpr int NL = limbs<MODE>();
  MmaArgs a = {};
  operands<MODE, true>(d, p, ws, st, a);
  const int64_t XN = d.T * p.Dp, DN = d.T * p.Hp;
  if (F32)
    hipLaunchKernelGGL(gated_pack_tokens_kernel, dim3((unsigned)rows_grid(d.T)), dim3(256), 0, st, (const float*)d.x, d.ldx, d.T, d.D, (int)p.Dp,
                       a.rscale, (const int*)(ws + p.spart), (int)p.pack_blocks, (uint16_t*)(ws + p.xt), XN,
                       (int*)(ws + p.exps));
  a.dh = d.dh; a.lddh = d.lddh;
  a.dg = (uint16_t*)(ws + p.dg); a.du = a.dg + NL * DN; a.dlimb = DN;
  a.dbpart = d.db_gate || d.db_up ? (float*)(ws + p.dbpart) : nullptr;
  launch_mma<MODE, true>(d, a, p, st);
  FinishArgs f = {};
  if (d.dx) {
    DxArgs x = {};
    x.dg = a.dg; x.du = a.du; x.Hp = p.Hp; x.dlimb = DN;
    x.wg = a.wg; x.wu = a.wu; x.ldwg = a.ldwg; x.ldwu = a.ldwu; x.wlimb = a.wlimb;
    x.T = d.T; x.H = d.H; x.D = d.D;
    x.rscale = a.rscale; x.exps = a.exps;
    x.dx = d.dx; x.chunk = p.dx_chunk; x.splits = (int)p.dx_splits; x.part = (float*)(ws + p.dx_sums);
    const int t = p.dx_big ? 256 : 128;
    x.tm = (int)cdiv(d.T, t); x.tn = (int)cdiv(d.D, t);
    const unsigned blocks = (unsigned)(x.tm * x.tn * x.splits);
    if (p.dx_big) hipLaunchKernelGGL((gated_dx_kernel<MODE, 256, 256, 4, 4, true>), dim3(blocks), dim3(1024), 0, st, x);
    else hipLaunchKernelGGL((gated_dx_kernel<MODE, 128, 128, 2, 4, false>), dim3(blocks), dim3(512), 0, st, x);
    if (x.splits > 1) {
      f.part[0] = x.part; f.splits[0] = x.splits; f.sets[0] = 1; f.n[0] = d.T * d.D;
      f.out[0][0] = d.dx;
      f.first[0] = (int)cdiv(f.n[0], 1024);
    }
  }
  if (d.dw_gate) {
    DwArgs w = {};
    w.d[0] = a.dg; w.d[1] = a.du; w.Hp = p.Hp; w.dlimb = DN;
    w.x = F32 ? (const uint16_t*)(ws + p.xt) : a.x; w.ldx = F32 ? p.Dp : a.ldx; w.xlimb = F32 ? XN : 0;
    w.T = d.T; w.H = d.H; w.D = d.D;
    w.chunk = p.dw_chunk; w.splits = (int)p.dw_splits; w.exps = a.exps;
    w.out[0] = d.dw_gate; w.out[1] = d.dw_up; w.part = (float*)(ws + p.dw_sums);
    const int t = p.dw_big ? 256 : 128;
    w.tm = (int)cdiv(d.H, t); w.tn = (int)cdiv(d.D, t);
    const unsigned blocks = (unsigned)(2 * w.tm * w.tn * w.splits);
    if (p.dw_big) hipLaunchKernelGGL((gated_dw_kernel<MODE, 256, 256, 4, 4, true>), dim3(blocks), dim3(1024), 0, st, w);
    else hipLaunchKernelGGL((gated_dw_kernel<MODE, 128, 128, 2, 4, false>), dim3(blocks), dim3(512), 0, st, w);
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
  return d->dtype == HOLD_GATED_F32 ? fwd<MODE_F16X3>(*d, (hipStream_t)st) : fwd<MODE_BF16>(*d, (hipStream_t)st);
}

extern "C" int hold_gated_bwd(const hold_gated_desc* d, hold_stream_t st) {
  if (check(d) != HOLD_OK || !d->dh || d->lddh < d->H || (!d->dw_gate != !d->dw_up)) return HOLD_E_ARG;
  if (((uintptr_t)d->dx | (uintptr_t)d->dw_gate | (uintptr_t)d->dw_up) % 16) return HOLD_E_ARG;
  return d->dtype == HOLD_GATED_F32 ? bwd<MODE_F16X3>(*d, (hipStream_t)st) : bwd<MODE_BF16>(*d, (hipStream_t)st);
}
