// The gated layer  h = act(x Wg^T + bg) * (x Wu^T + bu)  in one kernel, and its backward pass.
//
//   dg = dh * u * act'(g)      du = dh * act(g)      (g, u: the two projections, computed again instead of kept: 4 T D H operations
//   dx = dg Wg + du Wu         dWg = dg^T x          against 16 T H bytes written and read, less time up to D ~ 600 and no memory)
//   dWu = du^T x               dbg = sum_t dg, dbu = sum_t du
//
// KERNELS.  gated_mma_kernel: both projections of a tile share the x tile in LDS, the epilogue applies bias, activation and product
// (forward) or forms dg, du from dh and the recomputed g, u (backward), with the column sums for the bias gradients from the
// unrounded values.  gated_dx_kernel: [dg | du] times [Wg; Wu] as one sum.  gated_dw_kernel: both weight gradients, the sum over
// tokens split over blocks into fp32 partial tiles that gated_dw_reduce_kernel adds in a fixed order.  gated_rows_kernel: T <= 64 rows.
//
// ROUNDINGS.  bf16: dg and du are rounded to bf16 once, as the operands of the next matrix instructions; everything before is fp32.
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

__device__ __forceinline__ float sigmoid_f(float g) { return 1.f / (1.f + expf(-g)); }

// act(g) and act'(g)
template <bool DERIV>
__device__ __forceinline__ void activate(int act, float g, float& a, float& da) {
  if (act == ACT_RELU) {
    a = g > 0.f ? g : (g == g ? 0.f : g);
    da = g > 0.f ? 1.f : (g == g ? 0.f : g);
  } else if (act == ACT_GELU) {
    const float phi = 0.5f * erfcf(-0.70710678118654752f * g);
    a = g * phi;
    if (DERIV) da = phi + g * (0.39894228040143268f * expf(-0.5f * g * g));
  } else {
    const float s = sigmoid_f(g);
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
// four consecutive elements of which the first n exist; VEC: all four do and the address is a multiple of their size
template <int MODE>
__device__ __forceinline__ f32x4 load4(const void* p, int64_t i, int n, bool vec) {
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (vec && n >= 4) {
    if (MODE == MODE_BF16) {
      const u32x2 w = *(const u32x2*)((const uint16_t*)p + i);
      v = f32x4{bf16_value((uint16_t)w[0]), bf16_value((uint16_t)(w[0] >> 16)), bf16_value((uint16_t)w[1]), bf16_value((uint16_t)(w[1] >> 16))};
    } else {
      v = *(const f32x4*)((const float*)p + i);
    }
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < n) v[r] = load1<MODE>(p, i + r);
  }
  return v;
}
template <int MODE>
__device__ __forceinline__ void store4(void* p, int64_t i, int n, bool vec, f32x4 v) {
  if (vec && n >= 4) {
    if (MODE == MODE_BF16)
      *(u32x2*)((uint16_t*)p + i) = u32x2{(uint32_t)bf16_bits(v[0]) | (uint32_t)bf16_bits(v[1]) << 16, (uint32_t)bf16_bits(v[2]) | (uint32_t)bf16_bits(v[3]) << 16};
    else
      *(f32x4*)((float*)p + i) = v;
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < n) store1<MODE>(p, i + r, v[r]);
  }
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
// exponents kept by a call in fp32 (ints): [0] Wg, [1] Wu, [2] bg, [3] bu (all: exp_above of the largest magnitude, NONE of nothing), [4] R,
// [5] and [6] the exponents by which Wg and Wu are scaled (a matrix of zeros takes the other's)
constexpr int NONE = -100000;
__device__ __forceinline__ int exp_or_none(float m) { return m > 0.f ? exp_above(m) : NONE; }

// bits of the largest finite magnitude of a tensor, per block of the grid: part[which][block]
__global__ __launch_bounds__(256) void gated_amax_kernel(const float* wg, int64_t ldg, const float* wu, int64_t ldu, const float* bg,
                                                         const float* bu, int H, int D, float* part) {
  const float* src[4] = {wg, wu, bg, bu};
  const int which = blockIdx.y;
  const float* p = src[which];
  float m = 0.f;
  if (p && which < 2) {
    const int64_t ld = which ? ldu : ldg;
    const int lane = threadIdx.x & 63;
    for (int r = blockIdx.x * 4 + (threadIdx.x >> 6); r < H; r += gridDim.x * 4)
      for (int c = lane; c < D; c += 64) m = fmaxf(m, finite_abs(p[r * ld + c]));
  } else if (p) {
    for (int c = blockIdx.x * 256 + threadIdx.x; c < H; c += gridDim.x * 256) m = fmaxf(m, finite_abs(p[c]));
  }
  __shared__ float s[4];
  m = wave_fmax(m);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) part[which * NPART + blockIdx.x] = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
}

__device__ __forceinline__ float part_max(const float* part, int which) {  // every wave of a block by itself; NPART values
  const int lane = threadIdx.x & 63;
  float m = 0.f;
  for (int i = lane; i < NPART; i += 64) m = fmaxf(m, part[which * NPART + i]);
  return wave_fmax(m);
}

__device__ __forceinline__ void write_limbs(uint16_t* hi, uint16_t* lo, const float (&v)[8]) {
  u32x4 h, l;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const Split a = split16(v[2 * i]), b = split16(v[2 * i + 1]);
    h[i] = a.hi | (uint32_t)b.hi << 16;
    l[i] = a.lo | (uint32_t)b.lo << 16;
  }
  *(u32x4*)hi = h;
  *(u32x4*)lo = l;
}

// fp32 rows -> limbs [R][Kp], each row scaled to [2^14, 2^15) by its own exponent (rowexp: exp_above of the row, NONE of an empty one)
__global__ __launch_bounds__(256) void gated_pack_rows_kernel(const float* x, int64_t ld, int64_t R, int K, int Kp, uint16_t* out, int64_t limb,
                                                              int* rowexp) {
  const int lane = threadIdx.x & 63;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < R; r += (int64_t)gridDim.x * 4) {
    const float* p = x + r * ld;
    float m = 0.f;
    for (int c = lane; c < K; c += 64) m = fmaxf(m, finite_abs(p[c]));
    m = wave_fmax(m);
    const int e = exp_or_none(m), k = e == NONE ? 0 : 15 - e;
    if (lane == 0) rowexp[r] = e;
    for (int c = lane * 8; c < Kp; c += 512) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = c + i < K ? ldexpf(p[c + i], k) : 0.f;
      write_limbs(out + r * Kp + c, out + limb + r * Kp + c, v);
    }
  }
}

// both weight matrices -> limbs [H][Dp], one exponent a matrix; block 0 leaves the exponents in `exps`
__global__ __launch_bounds__(256) void gated_pack_weights_kernel(const float* wg, int64_t ldg, const float* wu, int64_t ldu, int H, int D, int Dp,
                                                                 const float* part, uint16_t* out, int64_t limb, int64_t second, int* exps) {
  const int lane = threadIdx.x & 63, which = blockIdx.y;
  const int e = exp_or_none(part_max(part, which)), other = exp_or_none(part_max(part, 1 - which));
  const int scale = e != NONE ? e : other != NONE ? other : 15, k = 15 - scale;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    exps[which] = e;
    exps[5 + which] = scale;
  }
  if (blockIdx.x == 0 && threadIdx.x < 64) {
    const int eb = exp_or_none(part_max(part, 2 + which));
    if (lane == 0) exps[2 + which] = eb;
  }
  const float* w = which ? wu : wg;
  const int64_t ld = which ? ldu : ldg;
  uint16_t* o = out + which * second;
  for (int r = blockIdx.x * 4 + (threadIdx.x >> 6); r < H; r += gridDim.x * 4)
    for (int c = lane * 8; c < Dp; c += 512) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = c + i < D ? ldexpf(w[r * ld + c + i], k) : 0.f;
      write_limbs(o + (int64_t)r * Dp + c, o + limb + (int64_t)r * Dp + c, v);
    }
}

// backward, fp32: the scale exponent r_t of every row of dg and du, and per block the largest exponent of x_t 2^-r_t.
//   |g| <= D max|x_t| max|Wg| + max|bg|, |u| likewise; |act(g)| <= |g| (sigmoid: 1); |act'| < 2 (relu: 1, sigmoid: 1/4)
__global__ __launch_bounds__(256) void gated_row_scale_kernel(const float* dh, int64_t ld, int64_t T, int H, int D, int act, const int* rowexp,
                                                              const int* exps, int* rscale, int* part) {
  const int lane = threadIdx.x & 63;
  int ld2 = 0;
  while ((1 << ld2) < D) ++ld2;
  int top = NONE;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < T; r += (int64_t)gridDim.x * 4) {
    float m = 0.f;
    for (int c = lane; c < H; c += 64) m = fmaxf(m, finite_abs(dh[r * ld + c]));
    const int ed = exp_or_none(wave_fmax(m)), ex = rowexp[r];
    auto proj = [&](int w) {  // exponent above a projection's magnitude
      const int a = (ex == NONE || exps[w] == NONE) ? NONE : ex + exps[w] + ld2, b = exps[2 + w];
      return (a > b ? a : b) == NONE ? NONE : (a > b ? a : b) + 1;
    };
    const int eg = proj(0), eu = proj(1);
    const int ea = act == ACT_SIGMOID ? 0 : eg, edg = eu + (act == ACT_SIGMOID ? -2 : act == ACT_RELU ? 0 : 1);
    // r_t of dg such that dg 2^r_t and du 2^(r_t + shift) both stay below 2^15
    const int shift = exps[6] - exps[5], top2 = edg > ea + shift ? edg : ea + shift;
    const bool none = ed == NONE || top2 < -50000;
    const int k = none ? NONE : 15 - (ed + top2);
    if (lane == 0) rscale[r] = k;
    if (!none && ex != NONE && ex - k > top) top = ex - k;
  }
  __shared__ int s[4];
  if (lane == 0) s[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    int v = s[0];
    for (int i = 1; i < 4; ++i) v = s[i] > v ? s[i] : v;
    part[blockIdx.x] = v;
  }
}

// x_t 2^(R - r_t) as limbs for the sum over tokens; rows without a gradient are zeros (where finite).  exps[4] = R
__global__ __launch_bounds__(256) void gated_pack_tokens_kernel(const float* x, int64_t ld, int64_t T, int D, int Dp, const int* rscale, const int* part,
                                                                int nparts, uint16_t* out, int64_t limb, int* exps) {
  const int lane = threadIdx.x & 63;
  int top = NONE;
  for (int i = lane; i < nparts; i += 64) top = part[i] > top ? part[i] : top;
  top = wave_max<64>(top);
  const int R = top == NONE ? 0 : 15 - top;
  if (blockIdx.x == 0 && threadIdx.x == 0) exps[4] = R;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < T; r += (int64_t)gridDim.x * 4) {
    const int k = rscale[r];
    for (int c = lane * 8; c < Dp; c += 512) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = c + i < D ? x[r * ld + c + i] : 0.f;
        v[i] = k == NONE ? y * 0.f : ldexpf(y, R - k);
      }
      write_limbs(out + r * Dp + c, out + limb + r * Dp + c, v);
    }
  }
}

// bf16 rows whose base, stride or length the tile loads cannot take -> [R][Kp], zeros behind K
__global__ __launch_bounds__(256) void gated_copy_rows_kernel(const uint16_t* x, int64_t ld, int64_t R, int K, int Kp, uint16_t* out) {
  const int lane = threadIdx.x & 63;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < R; r += (int64_t)gridDim.x * 4)
    for (int c = lane; c < Kp; c += 64) out[r * Kp + c] = c < K ? x[r * ld + c] : (uint16_t)0;
}

// ---- both projections and what follows them -------------------------------------------------------------------------------------------
struct MmaArgs {
  const uint16_t* x; int64_t ldx, xlimb;         // operands as the tile loads take them: [T][Dp]
  const uint16_t* wg; const uint16_t* wu; int64_t ldwg, ldwu, wlimb;
  const void* bg; const void* bu;
  int64_t T; int H; int K; int act;
  const int* rowexp; const int* exps;            // fp32: the scales of x's rows and of the weights
  void* h; int64_t ldh;                          // forward
  const void* dh; int64_t lddh;                  // backward
  uint16_t* dg; uint16_t* du; int64_t Hp, dlimb; // [T][Hp] limbs of dg and du
  const int* rscale;
  float* dbpart;                                 // [row tiles][2][H] column sums, or null
  int tm, tn;
};

template <int MODE, bool BWD, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void gated_mma_kernel(MmaArgs a) {
  using Cr = Core<MODE, KC, KC, BM, BN, 2, WM, WN>;
  __shared__ __align__(1024) char smem[Cr::LDS];
  int tm, tn;
  tile_of(blockIdx.x, gridDim.x, a.tm, a.tn, 8, tm, tn);
  const int64_t m0 = (int64_t)tm * BM;
  const int n0 = tn * BN;
  typename Cr::Acc acc;
  Cr::zero(acc);
  const Operand A = {a.x + m0 * a.ldx, a.xlimb, a.ldx, a.T - m0, a.K};
  const Operand B[2] = {{a.wg + (int64_t)n0 * a.ldwg, a.wlimb, a.ldwg, a.H - n0, a.K}, {a.wu + (int64_t)n0 * a.ldwu, a.wlimb, a.ldwu, a.H - n0, a.K}};
  Cr::run(smem, A, B, acc);

  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
  const int eg = MODE == MODE_F16X3 ? a.exps[5] - 15 : 0, eu = MODE == MODE_F16X3 ? a.exps[6] - 15 : 0;
  constexpr int ES = MODE == MODE_BF16 ? 2 : 4;
  const bool hvec = BWD ? (a.lddh % 4 == 0 && (uintptr_t)a.dh % (4 * ES) == 0) : (a.ldh % 4 == 0 && (uintptr_t)a.h % (4 * ES) == 0);
  const bool bvec = (uintptr_t)a.bg % (4 * ES) == 0 && (uintptr_t)a.bu % (4 * ES) == 0;
  float* sums = (float*)smem;  // [WM][2][BN]
#pragma unroll
  for (int ni = 0; ni < Cr::NI; ++ni) {
    const int jt = wn * (BN / WN) + 16 * ni + 4 * (lane >> 4), j = n0 + jt, n = a.H - j;
    f32x4 bg = {0.f, 0.f, 0.f, 0.f}, bu = {0.f, 0.f, 0.f, 0.f};
    if (a.bg && n > 0) bg = load4<MODE>(a.bg, j, n, bvec);
    if (a.bu && n > 0) bu = load4<MODE>(a.bu, j, n, bvec);
    f32x4 sg = {0.f, 0.f, 0.f, 0.f}, su = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int mi = 0; mi < Cr::MI; ++mi) {
      const int64_t i = m0 + wm * (BM / WM) + 16 * mi + (lane & 15);
      const bool row = i < a.T;
      f32x4 g = acc[0][mi][ni], u = acc[1][mi][ni];
      if (MODE == MODE_F16X3) {
        const int e = row ? a.rowexp[i] : NONE, ex = e == NONE ? 0 : e - 15;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          g[r] = ldexpf(g[r], ex + eg);
          u[r] = ldexpf(u[r], ex + eu);
        }
      }
      g += bg;
      u += bu;
      if (!BWD) {
        f32x4 h;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float s, d;
          activate<false>(a.act, g[r], s, d);
          h[r] = s * u[r];
        }
        if (row && n > 0) store4<MODE>(a.h, i * a.ldh + j, n, hvec, h);
      } else {
        f32x4 dg = {0.f, 0.f, 0.f, 0.f}, du = dg;
        if (row && n > 0) {
          const f32x4 dh = load4<MODE>(a.dh, i * a.lddh + j, n, hvec);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float s, d;
            activate<true>(a.act, g[r], s, d);
            dg[r] = r < n ? dh[r] * u[r] * d : 0.f;
            du[r] = r < n ? dh[r] * s : 0.f;
          }
        }
        sg += dg;
        su += du;
        if (row && j < a.Hp) {  // Hp is a multiple of 8: all four columns are inside, the ones behind H as zeros
          const int64_t o = i * a.Hp + j;
          if (MODE == MODE_BF16) {
            store4<MODE>(a.dg, o, 4, true, dg);
            store4<MODE>(a.du, o, 4, true, du);
          } else {
            const int k = a.rscale[i] == NONE ? 0 : a.rscale[i], ku = a.rscale[i] == NONE ? 0 : k + eu - eg;
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

// db[w][j] = sum over the row tiles, in 4 interleaved chains per column joined in a fixed order
template <int MODE>
__global__ __launch_bounds__(256) void gated_db_kernel(const float* part, int tiles, int H, void* dbg, void* dbu) {
  const int w = blockIdx.y, j = blockIdx.x * 64 + (threadIdx.x & 63), q = threadIdx.x >> 6;
  __shared__ float s[4][64];
  float v = 0.f;
  if (j < H)
    for (int t = q; t < tiles; t += 4) v += part[((int64_t)t * 2 + w) * H + j];
  s[q][threadIdx.x & 63] = v;
  __syncthreads();
  void* out = w ? dbu : dbg;
  if (q == 0 && j < H && out) {
    const int c = threadIdx.x;
    store1<MODE>(out, j, (s[0][c] + s[1][c]) + (s[2][c] + s[3][c]));
  }
}

// ---- dx = dg Wg + du Wu -----------------------------------------------------------------------------------------------------------------
struct DxArgs {
  const uint16_t* dg; const uint16_t* du; int64_t Hp, dlimb;
  const uint16_t* wg; const uint16_t* wu; int64_t ldwg, ldwu, wlimb;
  int64_t T; int H, D;
  const int* rscale; const int* exps;
  void* dx; int64_t lddx;
  int tm, tn;
};

template <int MODE, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void gated_dx_kernel(DxArgs a) {
  using Cr = Core<MODE, KC, KS, BM, BN, 1, WM, WN>;
  __shared__ __align__(1024) char smem[Cr::LDS];
  int tm, tn;
  tile_of(blockIdx.x, gridDim.x, a.tm, a.tn, 8, tm, tn);
  const int64_t m0 = (int64_t)tm * BM;
  const int n0 = tn * BN;
  typename Cr::Acc acc;
  Cr::zero(acc);
  const int64_t cols = (a.D + 7) / 8 * 8 - n0;
#pragma unroll 1
  for (int up = 0; up < 2; ++up) {
    const Operand A = {(up ? a.du : a.dg) + m0 * a.Hp, a.dlimb, a.Hp, a.T - m0, a.Hp};
    const Operand B[1] = {{(up ? a.wu : a.wg) + n0, a.wlimb, up ? a.ldwu : a.ldwg, cols, a.H}};
    Cr::run(smem, A, B, acc);
  }
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
  const int ew = MODE == MODE_F16X3 ? a.exps[5] - 15 : 0;
  const bool vec = a.lddx % 4 == 0;
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
      if (j < a.D) store4<MODE>(a.dx, i * a.lddx + j, a.D - j, vec, v);
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

template <int MODE, int BM, int BN, int WM, int WN>
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
  Cr::run(smem, A, B, acc);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
  const int e = MODE == MODE_F16X3 ? -a.exps[4] - (w ? a.exps[6] - a.exps[5] : 0) : 0;
  const bool vec = a.D % 4 == 0;
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
      if (a.splits == 1) store4<MODE>(a.out[w], (int64_t)i * a.D + j, a.D - j, vec, v);
      else store4<MODE_F16X3>(a.part, (((int64_t)sp * 2 + w) * a.H + i) * a.D + j, a.D - j, vec, v);
    }
  }
}

template <int MODE>
__global__ __launch_bounds__(256) void gated_dw_reduce_kernel(const float* part, int splits, int64_t HD, void* dwg, void* dwu) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  const int w = blockIdx.y;
  if (i >= HD) return;
  const int n = HD - i < 4 ? (int)(HD - i) : 4;
  const bool vec = HD % 4 == 0;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; ++s) v += load4<MODE_F16X3>(part, ((int64_t)s * 2 + w) * HD + i, n, vec);
  store4<MODE>(w ? dwu : dwg, i, n, true, v);
}

// ---- few rows ------------------------------------------------------------------------------------------------------------------------------
// T <= 64: the weights are read once, by fours of lanes along k; a wave holds 4 output columns (2 of each matrix... see RowsGeom) and
// all rows' sums.  fp32 arithmetic throughout: 2 T operations a weight element stay below the time of its bytes up to T = 64 in bf16.
constexpr int ROWS_MAX = 64;

template <int MODE, int NT>
__global__ __launch_bounds__(256) void gated_rows_kernel(const void* x, int64_t ldx, const void* wg, int64_t ldwg, const void* wu, int64_t ldwu,
                                                         const void* bg, const void* bu, int T, int D, int H, int act, void* h, int64_t ldh, int xvec,
                                                         int wvec) {
  const int lane = threadIdx.x & 63, j = blockIdx.x * 4 + (threadIdx.x >> 6), t0 = blockIdx.y * NT;
  if (j >= H) return;
  float g[NT], u[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) g[t] = u[t] = 0.f;
  for (int c = lane * 4; c < D; c += 256) {
    const int n = D - c;
    const f32x4 a = load4<MODE>(wg, j * ldwg + c, n, wvec), b = load4<MODE>(wu, j * ldwu + c, n, wvec);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (t0 + t < T) {
        const f32x4 v = load4<MODE>(x, (t0 + t) * ldx + c, n, xvec);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          g[t] = fmaf(a[r], v[r], g[t]);
          u[t] = fmaf(b[r], v[r], u[t]);
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      g[t] += __shfl_xor(g[t], o, 64);
      u[t] += __shfl_xor(u[t], o, 64);
    }
  const float vg = bg ? load1<MODE>(bg, j) : 0.f, vu = bu ? load1<MODE>(bu, j) : 0.f;
#pragma unroll
  for (int t = 0; t < NT; ++t)
    if (lane == t && t0 + t < T) {
      float s, d;
      activate<false>(act, g[t] + vg, s, d);
      store1<MODE>(h, (t0 + t) * ldh + j, s * (u[t] + vu));
    }
}

inline int ok() { return hipGetLastError() == hipSuccess ? HOLD_OK : HOLD_E_LAUNCH; }
inline int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
inline int64_t rows_grid(int64_t rows) {
  const int64_t b = (rows + 3) / 4;
  return b < 1 ? 1 : (b > 4096 ? 4096 : b);
}

// where everything of one call lies in its workspace (bytes; every part starts on a multiple of 256)
struct Plan {
  bool copy_x, copy_w[2];
  int64_t Dp, Hp, splits, chunk, row_tiles, scale_blocks;
  int64_t x, w, dg, xt, part, exps, rowexp, rscale, dbpart, dwpart, spart, bytes;
  bool big;
};

bool aligned16(const void* p, int64_t ld, int es) { return (uintptr_t)p % 16 == 0 && (ld * es) % 16 == 0; }

Plan plan(const hold_gated_desc& d, bool bwd) {
  Plan p = {};
  const int nl = d.dtype == HOLD_GATED_F32 ? 2 : 1;
  p.Dp = up(d.D, 8);
  p.Hp = up(d.H, 8);
  const bool f32 = d.dtype == HOLD_GATED_F32;
  p.copy_x = f32 || d.D % 8 || !aligned16(d.x, d.ldx, 2);
  p.copy_w[0] = f32 || d.D % 8 || !aligned16(d.w_gate, d.ldwg, 2);
  p.copy_w[1] = f32 || d.D % 8 || !aligned16(d.w_up, d.ldwu, 2);
  int64_t o = 0;
  auto take = [&](int64_t bytes) { const int64_t at = o; o += up(bytes, 256); return at; };
  // 256 x (128 + 128) tiles where they fill the 256 compute units, 128 x (64 + 64) elsewhere
  p.big = ((d.T + 255) / 256) * ((d.H + 127) / 128) >= 256;
  p.row_tiles = p.big ? (d.T + 255) / 256 : (d.T + 127) / 128;
  p.x = p.copy_x ? take(d.T * p.Dp * 2 * nl) : 0;
  p.w = p.copy_w[0] || p.copy_w[1] ? take(2 * (int64_t)d.H * p.Dp * 2 * nl) : 0;
  if (f32) {
    p.part = take(4 * NPART * 4);
    p.exps = take(8 * 4);
    p.rowexp = take(d.T * 4);
  }
  if (bwd) {
    p.dg = take(2 * d.T * p.Hp * 2 * nl);
    p.scale_blocks = rows_grid(d.T);
    if (f32) {
      p.xt = take(d.T * p.Dp * 2 * nl);
      p.rscale = take(d.T * 4);
      p.spart = take(p.scale_blocks * 4);
    }
    if (d.db_gate || d.db_up) p.dbpart = take(p.row_tiles * 2 * d.H * 4);
    // the tokens are split so that some 512 blocks have work, each at least 512 tokens
    const int64_t tiles = 2 * ((d.H + 127) / 128) * ((d.D + 127) / 128);
    int64_t s = tiles >= 512 ? 1 : (512 + tiles - 1) / tiles;
    const int64_t most = (d.T + 511) / 512;
    s = s > most ? most : s;
    p.chunk = up((d.T + s - 1) / s, 64);
    p.splits = (d.T + p.chunk - 1) / p.chunk;
    if (p.splits > 1) p.dwpart = take(p.splits * 2 * (int64_t)d.H * d.D * 4);
  }
  p.bytes = o;
  return p;
}

int check(const hold_gated_desc* d) {
  if (!d || !d->x || !d->w_gate || !d->w_up || d->T < 1 || d->D < 1 || d->H < 1 || d->act < 0 || d->act > 3) return HOLD_E_ARG;
  if (d->dtype != HOLD_GATED_F32 && d->dtype != HOLD_GATED_BF16) return HOLD_E_ARG;
  if (d->ldx < d->D || d->ldwg < d->D || d->ldwu < d->D) return HOLD_E_ARG;
  // the tile loads' 32-bit offsets: 256 rows of an operand, 64 rows of dg, and the tile grids
  if (d->ldx > (1 << 21) || d->ldwg > (1 << 21) || d->ldwu > (1 << 21) || d->H > (1 << 21) || d->T > (1ll << 31)) return HOLD_E_ARG;
  if (((d->T + 127) / 128) * ((d->H + 63) / 64) > (1ll << 30)) return HOLD_E_ARG;
  return HOLD_OK;
}

template <int MODE>
void operands(const hold_gated_desc& d, const Plan& p, char* ws, hipStream_t st, MmaArgs& a) {
  const int64_t WX = d.T * p.Dp, WW = (int64_t)d.H * p.Dp;
  a.x = (const uint16_t*)d.x; a.ldx = d.ldx; a.xlimb = 0;
  a.wg = (const uint16_t*)d.w_gate; a.ldwg = d.ldwg;
  a.wu = (const uint16_t*)d.w_up; a.ldwu = d.ldwu; a.wlimb = 0;
  if (MODE == MODE_F16X3) {
    float* part = (float*)(ws + p.part);
    int* exps = (int*)(ws + p.exps);
    int* rowexp = (int*)(ws + p.rowexp);
    uint16_t* x = (uint16_t*)(ws + p.x);
    uint16_t* w = (uint16_t*)(ws + p.w);
    hipLaunchKernelGGL(gated_amax_kernel, dim3(NPART, 4), dim3(256), 0, st, (const float*)d.w_gate, d.ldwg, (const float*)d.w_up, d.ldwu,
                       (const float*)d.b_gate, (const float*)d.b_up, d.H, d.D, part);
    hipLaunchKernelGGL(gated_pack_rows_kernel, dim3((unsigned)rows_grid(d.T)), dim3(256), 0, st, (const float*)d.x, d.ldx, d.T, d.D, (int)p.Dp, x, WX,
                       rowexp);
    hipLaunchKernelGGL(gated_pack_weights_kernel, dim3((unsigned)rows_grid(d.H), 2), dim3(256), 0, st, (const float*)d.w_gate, d.ldwg,
                       (const float*)d.w_up, d.ldwu, d.H, d.D, (int)p.Dp, part, w, WW * 2, WW, exps);
    a.x = x; a.ldx = p.Dp; a.xlimb = WX;
    a.wg = w; a.wu = w + WW; a.ldwg = a.ldwu = p.Dp; a.wlimb = 2 * WW;
    a.rowexp = rowexp; a.exps = exps;
  } else {
    if (p.copy_x) {
      hipLaunchKernelGGL(gated_copy_rows_kernel, dim3((unsigned)rows_grid(d.T)), dim3(256), 0, st, (const uint16_t*)d.x, d.ldx, d.T, d.D, (int)p.Dp,
                         (uint16_t*)(ws + p.x));
      a.x = (const uint16_t*)(ws + p.x); a.ldx = p.Dp;
    }
    for (int w = 0; w < 2; ++w)
      if (p.copy_w[w]) {
        uint16_t* o = (uint16_t*)(ws + p.w) + w * WW;
        hipLaunchKernelGGL(gated_copy_rows_kernel, dim3((unsigned)rows_grid(d.H)), dim3(256), 0, st, (const uint16_t*)(w ? d.w_up : d.w_gate),
                           w ? d.ldwu : d.ldwg, (int64_t)d.H, d.D, (int)p.Dp, o);
        if (w) { a.wu = o; a.ldwu = p.Dp; } else { a.wg = o; a.ldwg = p.Dp; }
      }
  }
  a.bg = d.b_gate; a.bu = d.b_up;
  a.T = d.T; a.H = d.H; a.K = (int)p.Dp; a.act = d.act;
}

template <int MODE, bool BWD>
void launch_mma(MmaArgs a, bool big, hipStream_t st) {
  if (big) {
    a.tm = (int)((a.T + 255) / 256); a.tn = (a.H + 127) / 128;
    hipLaunchKernelGGL((gated_mma_kernel<MODE, BWD, 256, 128, 2, 4>), dim3((unsigned)(a.tm * a.tn)), dim3(512), 0, st, a);
  } else {
    a.tm = (int)((a.T + 127) / 128); a.tn = (a.H + 63) / 64;
    hipLaunchKernelGGL((gated_mma_kernel<MODE, BWD, 128, 64, 2, 2>), dim3((unsigned)(a.tm * a.tn)), dim3(256), 0, st, a);
  }
}

template <int MODE>
void rows(const hold_gated_desc& d, hipStream_t st) {
  constexpr int ES = MODE == MODE_BF16 ? 2 : 4;
  const int xvec = d.ldx % 4 == 0 && (uintptr_t)d.x % (4 * ES) == 0;
  const int wvec = d.ldwg % 4 == 0 && d.ldwu % 4 == 0 && (uintptr_t)d.w_gate % (4 * ES) == 0 && (uintptr_t)d.w_up % (4 * ES) == 0;
  const dim3 block(256);
  const unsigned gx = (unsigned)((d.H + 3) / 4);
#define HOLD_ROWS(NT) \
  hipLaunchKernelGGL((gated_rows_kernel<MODE, NT>), dim3(gx, (unsigned)((d.T + NT - 1) / NT)), block, 0, st, d.x, d.ldx, d.w_gate, d.ldwg, d.w_up, \
                     d.ldwu, d.b_gate, d.b_up, (int)d.T, d.D, d.H, d.act, d.h, d.ldh, xvec, wvec)
  if (d.T == 1) HOLD_ROWS(1);
  else if (d.T <= 4) HOLD_ROWS(4);
  else HOLD_ROWS(16);
#undef HOLD_ROWS
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
  operands<MODE>(d, p, (char*)d.workspace, st, a);
  a.h = d.h; a.ldh = d.ldh;
  launch_mma<MODE, false>(a, p.big, st);
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
  operands<MODE>(d, p, ws, st, a);
  const int64_t XN = d.T * p.Dp, DN = d.T * p.Hp;
  if (F32) {
    hipLaunchKernelGGL(gated_row_scale_kernel, dim3((unsigned)p.scale_blocks), dim3(256), 0, st, (const float*)d.dh, d.lddh, d.T, d.H, d.D, d.act,
                       a.rowexp, a.exps, (int*)(ws + p.rscale), (int*)(ws + p.spart));
    hipLaunchKernelGGL(gated_pack_tokens_kernel, dim3((unsigned)rows_grid(d.T)), dim3(256), 0, st, (const float*)d.x, d.ldx, d.T, d.D, (int)p.Dp,
                       (const int*)(ws + p.rscale), (const int*)(ws + p.spart), (int)p.scale_blocks, (uint16_t*)(ws + p.xt), XN, (int*)(ws + p.exps));
  }
  a.dh = d.dh; a.lddh = d.lddh;
  a.dg = (uint16_t*)(ws + p.dg); a.du = a.dg + NL * DN; a.Hp = p.Hp; a.dlimb = DN;
  a.rscale = (const int*)(ws + p.rscale);
  a.dbpart = d.db_gate || d.db_up ? (float*)(ws + p.dbpart) : nullptr;
  launch_mma<MODE, true>(a, p.big, st);
  if (a.dbpart)
    hipLaunchKernelGGL(gated_db_kernel<MODE>, dim3((unsigned)((d.H + 63) / 64), 2), dim3(256), 0, st, a.dbpart, (int)p.row_tiles, d.H, d.db_gate, d.db_up);
  if (d.dx) {
    DxArgs x = {};
    x.dg = a.dg; x.du = a.du; x.Hp = p.Hp; x.dlimb = DN;
    x.wg = a.wg; x.wu = a.wu; x.ldwg = a.ldwg; x.ldwu = a.ldwu; x.wlimb = a.wlimb;
    x.T = d.T; x.H = d.H; x.D = d.D;
    x.rscale = a.rscale; x.exps = a.exps;
    x.dx = d.dx; x.lddx = d.D;
    x.tm = (int)((d.T + 127) / 128); x.tn = (d.D + 127) / 128;
    hipLaunchKernelGGL((gated_dx_kernel<MODE, 128, 128, 2, 2>), dim3((unsigned)(x.tm * x.tn)), dim3(256), 0, st, x);
  }
  if (d.dw_gate) {
    DwArgs w = {};
    w.d[0] = a.dg; w.d[1] = a.du; w.Hp = p.Hp; w.dlimb = DN;
    w.x = F32 ? (const uint16_t*)(ws + p.xt) : a.x; w.ldx = F32 ? p.Dp : a.ldx; w.xlimb = F32 ? XN : 0;
    w.T = d.T; w.H = d.H; w.D = d.D;
    w.chunk = p.chunk; w.splits = (int)p.splits; w.exps = a.exps;
    w.out[0] = d.dw_gate; w.out[1] = d.dw_up; w.part = (float*)(ws + p.dwpart);
    w.tm = (d.H + 127) / 128; w.tn = (d.D + 127) / 128;
    hipLaunchKernelGGL((gated_dw_kernel<MODE, 128, 128, 2, 2>), dim3((unsigned)(2 * w.tm * w.tn * w.splits)), dim3(256), 0, st, w);
    if (w.splits > 1) {
      const int64_t HD = (int64_t)d.H * d.D;
      hipLaunchKernelGGL(gated_dw_reduce_kernel<MODE>, dim3((unsigned)((HD + 1023) / 1024), 2), dim3(256), 0, st, w.part, w.splits, HD, d.dw_gate, d.dw_up);
    }
  }
  return ok();
}

}  // namespace

extern "C" int hold_gated_workspace(const hold_gated_desc* d, int32_t backward, int64_t* bytes) {
  if (check(d) != HOLD_OK || !bytes) return HOLD_E_ARG;
  *bytes = !backward && d->T <= ROWS_MAX ? 0 : plan(*d, backward != 0).bytes;
  return HOLD_OK;
}

extern "C" int hold_gated_fwd(const hold_gated_desc* d, hold_stream_t st) {
  if (check(d) != HOLD_OK || !d->h || d->ldh < d->H) return HOLD_E_ARG;
  return d->dtype == HOLD_GATED_F32 ? fwd<MODE_F16X3>(*d, (hipStream_t)st) : fwd<MODE_BF16>(*d, (hipStream_t)st);
}

extern "C" int hold_gated_bwd(const hold_gated_desc* d, hold_stream_t st) {
  if (check(d) != HOLD_OK || !d->dh || d->lddh < d->H || (!d->dw_gate != !d->dw_up)) return HOLD_E_ARG;
  return d->dtype == HOLD_GATED_F32 ? bwd<MODE_F16X3>(*d, (hipStream_t)st) : bwd<MODE_BF16>(*d, (hipStream_t)st);
}
