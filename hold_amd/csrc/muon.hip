// Orthogonalised updates: the polynomial iteration that brings the singular values of a matrix near one without a decomposition, and
// the momentum step that applies it to weight matrices.
//
//   X0 = G / (|G|_F + eps)        A = X X^T        X <- (a I + b A + c A A) X       `steps` times, on the side with fewer rows
//
// Three products a step (GRAM: A; POLY: C = a I + b A + c A A; APPLY: C X) for ALL matrices of a call in one launch each: a list of
// matrices of any shapes (or a batch of equal ones) is cut into tiles, and a block finds its matrix in the tile counts.
//
// Steps are taken one by one for every shape and type.  On wide matrices k steps could be joined into Q X with Q built from m x m products,
// which saves a quarter of the operations; but A's rounding errors then grow by a^2 = 12 a step where X's grow by a, 1.0e-4 of the norm
// against 1.5e-5 for a matrix of rank 64 and noise, and no caller asked for that.
//
// ARITHMETIC.  Small singular values grow by a^steps (485 with the usual coefficients), and with them every rounding of X relative to
// the largest one; bf16's 2^-9 would be the result there.  So X, A and C = a I + b A + c A A are kept as two fp16 limbs (tile16.h,
// 2^-22 each) and multiplied by three limb products with fp32 accumulation.  Their scales need no pass over the data: the singular
// values start at <= 1, the polynomial bounds them after every step (the host follows that bound), and no entry of a matrix is larger
// than its largest singular value.  The norm is summed in fp64: neither huge nor tiny gradients leave its range.
#include "tile16.h"

#include <math.h>

#include "../../include/hold_hip.h"

using namespace t16;

namespace {

constexpr int MAXI = 36;  // items of one launch; its arguments then take up to 4.7 KB (the last APPLY of several shapes)

struct Item {
  const void* g;  // the matrix (orthogonalise), the gradient (step)
  void* m;        // momentum, or null
  void* p;        // the result, or the parameter
  int64_t stride; // elements from one matrix of the item to the next, in all three
  int64_t x;      // this item's first X, in elements of the workspace
  int rows, cols, ldg, ldm, ldp, count;
  int part, nb;   // first partial sum, partial sums a matrix
  float gain;     // the step's factor: learning rate times the scale of the matrix's shape
};
struct Items {
  Item it[MAXI];
  int n;
};
struct Step {
  float mu, rest, decay, grad_mul, clip, eps;  // rest = 1 - mu
  int nesterov, dtype;
  const float* sumsq;
};
// the items' blocks of a launch begin at first[k]
struct Firsts {
  int first[MAXI + 1];
};
// Matrices of equal shape lie one after the other in the workspace: the products in between know them as classes only, and a call
// whose matrices all have one shape (ONE) finds everything in the first bytes of its arguments instead of a chain of loads
struct Class {
  int64_t x, c;      // the class's first X and first A, in elements
  int m, n, mp, np;  // the smaller and the larger side, and both rounded up to 8
  int mats, item;    // matrices, the first one's item
  int tile;          // first tile in the launch
};
struct Classes {
  Class k[MAXI];
  int n;
};
struct OneClass {
  Class k[1];
  int n;
};

template <class F>
__device__ __forceinline__ int last_below(int n, int id, F first) {
  int k = 0;
  while (k + 1 < n && id >= first(k + 1)) ++k;
  return k;
}
__host__ __device__ __forceinline__ int up8(int v) { return (v + 7) / 8 * 8; }

__device__ __forceinline__ float value(const void* p, int64_t i, int dtype) {
  if (dtype == HOLD_MUON_F32) return ((const float*)p)[i];
  const uint16_t b = ((const uint16_t*)p)[i];
  return dtype == HOLD_MUON_BF16 ? bf16_value(b) : (float)__builtin_bit_cast(_Float16, b);
}
__device__ __forceinline__ void put(void* p, int64_t i, int dtype, float v) {
  if (dtype == HOLD_MUON_F32) ((float*)p)[i] = v;
  else ((uint16_t*)p)[i] = dtype == HOLD_MUON_BF16 ? bf16_bits(v) : __builtin_bit_cast(uint16_t, (_Float16)v);
}

// the factor of the gradients: grad_mul and the clip to a global norm, as hold_adam_step has them
__device__ __forceinline__ float grad_scale(const Step& s) {
  float f = s.grad_mul;
  if (s.clip > 0.f && s.sumsq) f *= fminf(1.f, s.clip / (sqrtf(s.sumsq[0]) * fabsf(s.grad_mul) + 1e-6f));
  return f;
}
// the matrix to orthogonalise at element (r, c) once the momentum is updated
__device__ __forceinline__ float update_of(const Item& it, const Step& s, float f, int64_t b, int r, int c) {
  const float g = value(it.g, b + (int64_t)r * it.ldg + c, s.dtype);
  if (!it.m) return g;
  const float m = ((const float*)it.m)[b + (int64_t)r * it.ldm + c];
  return s.nesterov ? s.rest * (g * f) + s.mu * m : m;
}

// Momentum and the partial sums of squares: a block takes an equal share of a matrix's elements, the partial sums are added in a fixed
// order.  Matrices without gaps between rows, on 16-byte boundaries, go by 16 bytes, two of each operand in flight per thread
// (36 matrices of 256 x 256: 46.7 us element by element).
__global__ __launch_bounds__(256) void ns_norm_kernel(Items a, Firsts t, Step s, double* part) {
  const int k = last_below(a.n, blockIdx.x, [&](int i) { return t.first[i]; });
  const Item& it = a.it[k];
  const int q = blockIdx.x - t.first[k], mat = q / it.nb, blk = q % it.nb;
  const int64_t b = mat * it.stride, n = (int64_t)it.rows * it.cols, per = ((n + it.nb - 1) / it.nb + 7) / 8 * 8;
  const int64_t begin = blk * per, end = begin + per < n ? begin + per : n;
  const float f = it.m ? grad_scale(s) : 1.f;
  double sum = 0.;
  auto one = [&](float g, float& m) {
    float u = g;
    if (it.m) {
      const float gf = g * f;
      m = s.mu * m + s.rest * gf;
      u = s.nesterov ? s.rest * gf + s.mu * m : m;
    }
    sum += (double)u * u;
  };
  const bool lin = it.ldg == it.cols && (!it.m || it.ldm == it.cols);
  float* mp = (float*)it.m + b;
  if (lin && s.dtype == HOLD_MUON_F32 && ((uintptr_t)it.g | (uintptr_t)it.m | (uint64_t)(4 * b)) % 16 == 0) {
    const float* gp = (const float*)it.g + b;
    const int64_t whole = end & ~(int64_t)3;
    for (int64_t e = begin + 4 * threadIdx.x; e < whole; e += 2048) {
      const bool two = e + 1024 < whole;
      f32x4 g0 = *(const f32x4*)(gp + e), g1 = two ? *(const f32x4*)(gp + e + 1024) : f32x4{0.f, 0.f, 0.f, 0.f};
      f32x4 m0 = {0.f, 0.f, 0.f, 0.f}, m1 = m0;
      if (it.m) {
        m0 = *(const f32x4*)(mp + e);
        if (two) m1 = *(const f32x4*)(mp + e + 1024);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float x = m0[r], y = m1[r];
        one(g0[r], x);
        if (two) one(g1[r], y);
        m0[r] = x;
        m1[r] = y;
      }
      if (it.m) {
        *(f32x4*)(mp + e) = m0;
        if (two) *(f32x4*)(mp + e + 1024) = m1;
      }
    }
    const int64_t e = whole + threadIdx.x;
    if (e >= begin && e < end) {
      float m = it.m ? mp[e] : 0.f;
      one(gp[e], m);
      if (it.m) mp[e] = m;
    }
  } else if (lin && s.dtype != HOLD_MUON_F32 && ((uintptr_t)it.g | (uint64_t)(2 * b)) % 16 == 0) {
    const uint16_t* gp = (const uint16_t*)it.g + b;
    const int64_t whole = end & ~(int64_t)7;
    for (int64_t e = begin + 8 * threadIdx.x; e < whole; e += 2048) {
      const u32x4 w = *(const u32x4*)(gp + e);
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const uint16_t h = (uint16_t)(w[r >> 1] >> (16 * (r & 1)));
        float m = 0.f;
        one(s.dtype == HOLD_MUON_BF16 ? bf16_value(h) : (float)__builtin_bit_cast(_Float16, h), m);
      }
    }
    const int64_t e = whole + threadIdx.x;
    float m = 0.f;
    if (e >= begin && e < end) one(value(gp, e, s.dtype), m);
  } else {
    for (int64_t e = begin + threadIdx.x; e < end; e += 256) {
      const int64_t r = lin ? 0 : e / it.cols, c = e - r * it.cols;
      float m = it.m ? mp[r * it.ldm + c] : 0.f;
      one(value(it.g, b + r * it.ldg + c, s.dtype), m);
      if (it.m) mp[r * it.ldm + c] = m;
    }
  }
  __shared__ double w[4];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) part[it.part + q] = (w[0] + w[1]) + (w[2] + w[3]);
}

// 2^xs / (|X|_F + eps); a matrix of zeros without eps is divided by one: it stays zero.  (A norm of NaN stays NaN.)
__device__ __forceinline__ double norm_factor(double sumsq, float eps, int xs) {
  const double n = sqrt(sumsq) + (double)eps;
  return ldexp(1. / (n == 0. ? 1. : n), xs);
}

// X0 as limbs [min][max] (rounded up to 8, zeros behind), scaled by 2^xs: 64 x 64 tiles of the source through LDS, transposed where it is tall
__global__ __launch_bounds__(256) void ns_load_kernel(Items a, Firsts t, Step s, const double* part, uint16_t* ws, int64_t limb, int xs) {
  const int k = last_below(a.n, blockIdx.x, [&](int i) { return t.first[i]; });
  const Item& it = a.it[k];
  const bool tall = it.rows > it.cols;
  const int m = tall ? it.cols : it.rows, n = tall ? it.rows : it.cols, mp = up8(m), np = up8(n);
  const int tn = (np + 63) / 64, tm = (mp + 63) / 64;
  const int q = blockIdx.x - t.first[k], mat = q / (tm * tn), tile = q % (tm * tn), i0 = tile / tn * 64, j0 = tile % tn * 64;
  __shared__ float s_tile[64][65];
  __shared__ double s_sum[4];
  double sum = 0.;
  for (int i = threadIdx.x; i < it.nb; i += 256) sum += part[it.part + mat * it.nb + i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum;
  const int64_t b = mat * it.stride;
  const float f = it.m ? grad_scale(s) : 1.f;
  const int r0 = tall ? j0 : i0, c0 = tall ? i0 : j0;  // the tile's place in the source
  const bool whole = r0 + 64 <= it.rows && c0 + 64 <= it.cols && s.dtype == HOLD_MUON_F32 &&
                     (((uintptr_t)it.g | (uintptr_t)it.m | (uint64_t)(4 * b)) % 16 | (uint32_t)(it.ldg | (it.m ? it.ldm : 0)) % 4) == 0;
  if (whole) {  // 16 bytes a lane, all of a thread's loads requested together
    const float* gp = (const float*)it.g + b + c0;
    const float* mp = (const float*)it.m + b + c0;
    f32x4 g[4], m[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int r = r0 + q * 16 + (threadIdx.x >> 4), c = 4 * (threadIdx.x & 15);
      g[q] = *(const f32x4*)(gp + (int64_t)r * it.ldg + c);
      if (it.m) m[q] = *(const f32x4*)(mp + (int64_t)r * it.ldm + c);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float u = !it.m ? g[q][i] : s.nesterov ? s.rest * (g[q][i] * f) + s.mu * m[q][i] : m[q][i];
        s_tile[q * 16 + (threadIdx.x >> 4)][4 * (threadIdx.x & 15) + i] = u;
      }
  } else {
#pragma unroll 4
    for (int e = threadIdx.x; e < 4096; e += 256) {
      const int r = e >> 6, c = e & 63;
      s_tile[r][c] = r0 + r < it.rows && c0 + c < it.cols ? update_of(it, s, f, b, r0 + r, c0 + c) : 0.f;
    }
  }
  __syncthreads();
  const double inv = norm_factor((s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]), s.eps, xs);
  uint16_t* x = ws + it.x + (int64_t)mat * mp * np;
  for (int e = threadIdx.x; e < 512; e += 256) {
    const int i = e >> 3, j = (e & 7) * 8;
    if (i0 + i >= mp || j0 + j >= np) continue;
    u32x4 h, l;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float v = tall ? s_tile[j + 2 * r][i] : s_tile[i][j + 2 * r], w = tall ? s_tile[j + 2 * r + 1][i] : s_tile[i][j + 2 * r + 1];
      const bool in = i0 + i < m;  // behind the last row and column: zeros, also where the norm is not finite
      const Split y = split16(in && j0 + j + 2 * r < n ? (float)(v * inv) : 0.f), z = split16(in && j0 + j + 2 * r + 1 < n ? (float)(w * inv) : 0.f);
      h[r] = y.hi | (uint32_t)z.hi << 16;
      l[r] = y.lo | (uint32_t)z.lo << 16;
    }
    uint16_t* o = x + (int64_t)(i0 + i) * np + j0 + j;
    *(u32x4*)o = h;
    *(u32x4*)(o + limb) = l;
  }
}

__device__ __forceinline__ void store_limbs(uint16_t* o, int64_t limb, f32x4 v) {
  Split y[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) y[r] = split16(v[r]);
  *(u32x2*)o = u32x2{y[0].hi | (uint32_t)y[1].hi << 16, y[2].hi | (uint32_t)y[3].hi << 16};
  *(u32x2*)(o + limb) = u32x2{y[0].lo | (uint32_t)y[1].lo << 16, y[2].lo | (uint32_t)y[3].lo << 16};
}
__device__ __forceinline__ float half_value(uint32_t w, int h) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> (16 * h))); }
__device__ __forceinline__ f32x4 load_limbs(const uint16_t* p, int64_t limb) {
  const u32x2 h = *(const u32x2*)p, l = *(const u32x2*)(p + limb);
  f32x4 v;
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = half_value(h[r >> 1], r & 1) + half_value(l[r >> 1], r & 1);
  return v;
}

enum { GRAM = 0, POLY = 1, APPLY = 2 };
struct NsArgs {
  const uint16_t* x;  // X: hi at the item's place, lo `limb` further
  uint16_t* y;        // the next X
  const uint16_t* l;  // m x m operand: POLY's A; APPLY's C - a I
  uint16_t* o;        // m x m result of GRAM and POLY
  int64_t xlimb, climb;
  float a, b, c;      // the polynomial's, already in the scales of what they are multiplied with and of the result
  int shift;          // exponent from the accumulated sum to the stored limbs
};

static_assert(sizeof(Classes) + sizeof(NsArgs) + sizeof(Step) + sizeof(Items) <= 5120, "a launch's arguments stay small");
struct NoItems {};
template <bool LAST> struct ItemArg { typedef NoItems type; };
template <> struct ItemArg<true> { typedef Items type; };

// Symmetric results (all but APPLY's): only the tiles on and below the diagonal; what is right of it is written as their mirror image, turned in LDS
// rows of a tile: T; columns: as many, but 64 at least where an operand is read by k
template <int KIND>
constexpr int tile_cols(int T) { return KIND == APPLY && T == 32 ? 64 : T; }
template <int KIND, int T, int WM, int WN, int S, bool PHASED, bool LAST, class CLASSES>
__global__ __launch_bounds__(64 * WM * WN) void ns_mma_kernel(CLASSES cl, NsArgs s, Step st, typename ItemArg<LAST>::type items) {
  constexpr int TC = tile_cols<KIND>(T);
  using Cr = Core<MODE_F16X3, KC, KIND == APPLY ? KS : KC, T, TC, 1, WM, WN, S, T == 32 || WM * WN == 8 && T == 64 ? 64 : 32>;
  constexpr int PITCH = T + 8, TURN = KIND == APPLY ? 0 : T * PITCH * 2;
  __shared__ __align__(1024) char smem[Cr::LDS > TURN ? Cr::LDS : TURN];
  // the tile list is cut into an eighth for each XCD, as tile_of does: neighbours share a matrix
  const int total = gridDim.x, qq = total / 8, rr = total % 8, xcd = blockIdx.x % 8, ii = blockIdx.x / 8;
  const int id = xcd * qq + (xcd < rr ? xcd : rr) + ii;
  constexpr bool ONE = sizeof(CLASSES) == sizeof(OneClass);
  const int k = ONE ? 0 : last_below(cl.n, id, [&](int i) { return cl.k[i].tile; });
  const Class& c = cl.k[k];
  const int m = c.m, n = c.n, mp = c.mp, np = c.np, tm = (mp + T - 1) / T, tn = KIND == APPLY ? (np + TC - 1) / TC : tm;
  const int per = KIND == APPLY ? tm * tn : tm * (tm + 1) / 2, q = id - c.tile, mat = q / per, tile = q % per;
  int i0, j0;
  if (KIND == APPLY) {  // bands of 8 row tiles, column by column
    const int w = 8 * tn, band = tile / w, f0 = band * 8, h = tm - f0 < 8 ? tm - f0 : 8;
    i0 = (f0 + (tile - band * w) % h) * T;
    j0 = (tile - band * w) / h * TC;
  } else {  // row bi of the triangle begins at tile bi (bi + 1) / 2
    int bi = (int)((sqrtf(8.f * tile + 1.f) - 1.f) * 0.5f);
    while (bi * (bi + 1) / 2 > tile) --bi;
    while ((bi + 1) * (bi + 2) / 2 <= tile) ++bi;
    i0 = bi * T;
    j0 = (tile - bi * (bi + 1) / 2) * T;
  }
  const int64_t xo = c.x + (int64_t)mat * mp * np, co = c.c + (int64_t)mat * mp * mp;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
  typename Cr::Acc acc;
  Cr::zero(acc);
  Operand A, B[1];
  if (KIND == GRAM) {
    A = Operand{s.x + xo + (int64_t)i0 * np, s.xlimb, np, mp - i0, np};
    B[0] = Operand{s.x + xo + (int64_t)j0 * np, s.xlimb, np, mp - j0, np};
  } else if (KIND != APPLY) {
    A = Operand{s.l + co + (int64_t)i0 * mp, s.climb, mp, mp - i0, mp};
    B[0] = Operand{s.l + co + (int64_t)j0 * mp, s.climb, mp, mp - j0, mp};
  } else {
    A = Operand{s.l + co + (int64_t)i0 * mp, s.climb, mp, mp - i0, mp};
    B[0] = Operand{s.x + xo + j0, s.xlimb, np, np - j0, mp};
  }
  // POLY adds b A, APPLY a X (C comes without a I: X itself, in one rounding, instead of the limbs of a diagonal that is large against
  // the rest of C; in front of the sum every addition would round at its size).  The small tiles' launches are latencies: there the own tile
  // is requested before the products, not behind them
  constexpr bool EARLY = (KIND == POLY || KIND == APPLY) && T <= 64;
  const uint16_t* own = KIND == POLY ? s.l + co : s.x + xo;
  const int64_t olimb = KIND == POLY ? s.climb : s.xlimb;
  const int opitch = KIND == APPLY ? np : mp;
  f32x4 early[EARLY ? Cr::MI : 1][EARLY ? Cr::NI : 1];
  if (EARLY) {
#pragma unroll
    for (int mi = 0; mi < Cr::MI; ++mi)
#pragma unroll
      for (int ni = 0; ni < Cr::NI; ++ni) {
        const int i = i0 + wm * (T / WM) + 16 * mi + (lane & 15), j = j0 + wn * (TC / WN) + 16 * ni + 4 * (lane >> 4);
        early[EARLY ? mi : 0][EARLY ? ni : 0] = i < mp && j < opitch ? load_limbs(own + (int64_t)i * opitch + j, olimb) : f32x4{0.f, 0.f, 0.f, 0.f};
      }
  }
  if constexpr (PHASED) Cr::run_phased(smem, A, B, acc);
  else Cr::run(smem, A, B, acc);
  uint16_t* sym = s.o + co;
  uint16_t* turn = (uint16_t*)smem;
#pragma unroll
  for (int mi = 0; mi < Cr::MI; ++mi) {
    const int it = wm * (T / WM) + 16 * mi + (lane & 15), i = i0 + it;
#pragma unroll
    for (int ni = 0; ni < Cr::NI; ++ni) {
      const int jt = wn * (TC / WN) + 16 * ni + 4 * (lane >> 4), j = j0 + jt;
      f32x4& v = acc[0][mi][ni];
      const bool in = i < mp && j < (KIND == APPLY ? np : mp);
      if (KIND == GRAM) {
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = ldexpf(v[r], s.shift);
        if (in) store_limbs(sym + (int64_t)i * mp + j, s.climb, v);
      } else if (KIND == POLY) {
        if (in) {
          const f32x4 u = EARLY ? early[EARLY ? mi : 0][EARLY ? ni : 0] : load_limbs(own + (int64_t)i * opitch + j, olimb);
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = fmaf(s.c, v[r], s.b * u[r]);
          store_limbs(sym + (int64_t)i * mp + j, s.climb, v);
        }
      } else {
        if (in) v += s.a * (EARLY ? early[EARLY ? mi : 0][EARLY ? ni : 0] : load_limbs(own + (int64_t)i * opitch + j, olimb));
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = ldexpf(v[r], s.shift);
        if constexpr (!LAST) {
          if (in) store_limbs(s.y + xo + (int64_t)i * np + j, s.xlimb, v);
        } else if (i < m) {
          const bool list = items.it[c.item].count == 1;  // a class is a run of single items, or one item of many matrices
          const Item& d = items.it[c.item + (list ? mat : 0)];
          const bool tall = d.rows > d.cols;
          const int64_t b = list ? 0 : mat * d.stride;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (j + r >= n) continue;
            const int64_t at = b + (tall ? (int64_t)(j + r) * d.ldp + i : (int64_t)i * d.ldp + j + r);
            if (d.m) {
              float* p = (float*)d.p + at;
              *p = *p * st.decay - d.gain * v[r];
            } else {
              put(d.p, at, st.dtype, v[r]);
            }
          }
        }
      }
    }
  }
  if (KIND != APPLY && i0 != j0) {  // limb by limb: [j][i] in LDS, whole rows out
#pragma unroll 1
    for (int l = 0; l < 2; ++l) {
#pragma unroll
      for (int mi = 0; mi < Cr::MI; ++mi)
#pragma unroll
        for (int ni = 0; ni < Cr::NI; ++ni)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const Split y = split16(acc[0][mi][ni][r]);
            turn[(wn * (TC / WN) + 16 * ni + 4 * (lane >> 4) + r) * PITCH + wm * (T / WM) + 16 * mi + (lane & 15)] = l ? y.lo : y.hi;
          }
      __syncthreads();
      for (int e = threadIdx.x; e < T * T / 8; e += 64 * WM * WN) {
        const int r = e / (T / 8), q8 = e % (T / 8) * 8;
        if (j0 + r < mp && i0 + q8 < mp) *(u32x4*)(sym + (int64_t)(j0 + r) * mp + i0 + q8 + (l ? s.climb : 0)) = *(const u32x4*)(turn + r * PITCH + q8);
      }
      __syncthreads();
    }
  }
}

// ---- small matrices: a block each, the whole iteration in LDS ----------------------------------------------------------------------------------
// X and A as limbs in LDS; 16 waves take 32 x 32 blocks of each product, results wait in registers until everyone has read.  One launch
// instead of 2 + 3 a step: a 64 x 64 matrix takes 25 us instead of 66, most of it the barriers between products of a few hundred cycles.
constexpr int SMALL_STEPS = 8, SMALL_LDS = 160 * 1024 - 1024, SMALL_BLOCKS = 32;
struct SmallSteps {
  float a[SMALL_STEPS], b[SMALL_STEPS], c[SMALL_STEPS];
  int gram[SMALL_STEPS], apply[SMALL_STEPS], n, xs;
};
inline int up32(int v) { return (v + 31) / 32 * 32; }
// A row's pitch in elements and the exchange of its 16-byte chunks, so that neither a fragment by rows nor one by k meets a bank twice: rows of
// multiples of 256 bytes exchange eight pairs of chunks; others are an odd multiple of 64 bytes long, which spreads 4 rows over the banks, and
// exchange fours
__host__ __device__ __forceinline__ int small_pitch(int n32) { return n32 % 128 == 0 ? n32 : (n32 / 32 | 1) * 32; }
__device__ __forceinline__ int small_swz(int pitch, int r) { return pitch % 128 == 0 ? ((r & 3) | ((r >> 1) & 4)) << 4 : (-(r >> 2) & 3) << 3; }
__device__ __forceinline__ int small_at(int pitch, int r, int c) { return r * pitch + (c ^ small_swz(pitch, r)); }
// elements of the two arrays (one limb); what fits: both limbs of both in LDS, at most two blocks of X a wave
bool small(const Item& it, int steps) {
  const int64_t m = it.rows < it.cols ? it.rows : it.cols, n = it.rows < it.cols ? it.cols : it.rows;
  if (steps > SMALL_STEPS || m > 128 || n > 2048) return false;
  const int64_t mp = up32((int)m), np = up32((int)n);
  return 4 * mp * (small_pitch((int)np) + small_pitch((int)mp)) <= SMALL_LDS && (mp / 32) * (np / 32) <= SMALL_BLOCKS;
}

// acc[mi][ni] of a 32 x 32 block: sum over K of A(i, k) B(j, k); A by rows, B by rows (LB = KC) or by k (KS).  The exchange of chunks depends on
// a row's place among 16 alone: it is the same for every 16 rows and every 32 k's
template <int LB>
__device__ __forceinline__ void small_block(const uint16_t* a, int pa, int la, const uint16_t* b, int pb, int lb, int i0, int j0, int K, f32x4 (&acc)[2][2]) {
  const int lane = threadIdx.x & 63, row = lane & 15, kl = 8 * (lane >> 4), kr = kl + (row >> 2), xa = small_swz(pa, row), xb = small_swz(pb, row);
  const uint16_t* ap = a + (i0 + row) * pa;
  const uint16_t* bp = LB == KC ? b + (j0 + row) * pb : b + kr * pb;
  const int x0 = small_swz(pb, kr), x1 = small_swz(pb, kr + 4), c = j0 + 4 * (lane & 3);
  const int o[2][2] = {{c ^ x0, 4 * pb + (c ^ x1)}, {(c + 16) ^ x0, 4 * pb + ((c + 16) ^ x1)}};  // KS: the two halves of two 16-column fragments
#pragma unroll 1
  for (int k = 0; k < K; k += 32) {
    s16x8 fa[2][2], fb[2][2];
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int l = 0; l < 2; ++l) {
        fa[q][l] = *(const s16x8*)(ap + l * la + 16 * q * pa + ((k + kl) ^ xa));
        if (LB == KC) {
          fb[q][l] = *(const s16x8*)(bp + l * lb + 16 * q * pb + ((k + kl) ^ xb));
        } else {
          const s16x4 u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(bp + l * lb + o[q][0]));
          const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(bp + l * lb + o[q][1]));
          fb[q][l] = __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
        }
      }
#pragma unroll
    for (int p = 0; p < 3; ++p)
#pragma unroll
      for (int mi = 0; mi < 2; ++mi)
#pragma unroll
        for (int ni = 0; ni < 2; ++ni) acc[mi][ni] = mfma<MODE_F16X3>(fb[ni][p == 0], fa[mi][p == 1], acc[mi][ni]);
    if (LB == KS) bp += 32 * pb;
  }
}

__global__ __launch_bounds__(1024) void ns_small_kernel(Items a, Firsts t, Step s, SmallSteps st) {
  __shared__ __align__(16) uint16_t lds[SMALL_LDS / 2];
  __shared__ double red[16];
  const int k = last_below(a.n, blockIdx.x, [&](int i) { return t.first[i]; });
  const Item& it = a.it[k];
  const int64_t base = (int64_t)(blockIdx.x - t.first[k]) * it.stride;
  const bool tall = it.rows > it.cols;
  const int m = tall ? it.cols : it.rows, n = tall ? it.rows : it.cols, mp = (m + 31) / 32 * 32, np = (n + 31) / 32 * 32;
  const int px = small_pitch(np), pa = small_pitch(mp), lx = mp * px, la = mp * pa;
  uint16_t* X = lds;
  uint16_t* A = lds + 2 * lx;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const float f = it.m ? grad_scale(s) : 1.f;
  // momentum and the norm, then X0 from the same thread's elements
  const int count = it.rows * it.cols;
  double sum = 0.;
#pragma unroll 4
  for (int e = threadIdx.x; e < count; e += 1024) {
    const int r = e / it.cols, c = e - r * it.cols;
    const float g = value(it.g, base + (int64_t)r * it.ldg + c, s.dtype);
    float u = g;
    if (it.m) {
      float* p = (float*)it.m + base + (int64_t)r * it.ldm + c;
      const float gf = g * f, mm = s.mu * *p + s.rest * gf;
      *p = mm;
      u = s.nesterov ? s.rest * gf + s.mu * mm : mm;
    }
    sum += (double)u * u;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if (lane == 0) red[wave] = sum;
  for (int e = threadIdx.x; e < lx; e += 1024) ((uint32_t*)X)[e] = 0u;  // both limbs, also behind the last row and column
  __syncthreads();
  sum = 0.;
#pragma unroll
  for (int w = 0; w < 16; ++w) sum += red[w];
  const double inv = norm_factor(sum, s.eps, st.xs);
#pragma unroll 4
  for (int e = threadIdx.x; e < count; e += 1024) {
    const int r = e / it.cols, c = e - r * it.cols;
    const Split y = split16((float)(update_of(it, s, f, base, r, c) * inv));
    uint16_t* x = X + (tall ? small_at(px, c, r) : small_at(px, r, c));
    x[0] = y.hi;
    x[lx] = y.lo;
  }
  __syncthreads();
  const int tm = mp / 32, tn = np / 32;
  auto each = [&](const f32x4 (&acc)[2][2], int i0, int j0, auto put4) {
#pragma unroll
    for (int mi = 0; mi < 2; ++mi)
#pragma unroll
      for (int ni = 0; ni < 2; ++ni) put4(i0 + 16 * mi + (lane & 15), j0 + 16 * ni + 4 * (lane >> 4), acc[mi][ni]);
  };
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  f32x4 x[2][2][2];  // X's blocks of the wave, up to two
#pragma unroll 1
  for (int q = 0; q < st.n; ++q) {
    f32x4 acc[2][2] = {{zero, zero}, {zero, zero}};
    const int ai = wave / tm * 32, aj = wave % tm * 32;  // tm^2 <= 16 blocks of A
    if (wave < tm * tm) {
      small_block<KC>(X, px, lx, X, px, lx, ai, aj, np, acc);
      each(acc, ai, aj, [&](int i, int j, f32x4 v) {
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = ldexpf(v[r], st.gram[q]);
        store_limbs(A + small_at(pa, i, j), la, v);
      });
    }
    __syncthreads();
    f32x4 c[2][2] = {{zero, zero}, {zero, zero}};
    if (wave < tm * tm) small_block<KC>(A, pa, la, A, pa, la, ai, aj, mp, c);
    if (wave < tm * tm) {
#pragma unroll
      for (int mi = 0; mi < 2; ++mi)
#pragma unroll
        for (int ni = 0; ni < 2; ++ni) {
#pragma unroll
          for (int r = 0; r < 4; ++r) c[mi][ni][r] = fmaf(st.c[q], c[mi][ni][r], st.b[q] * ldexpf(acc[mi][ni][r], st.gram[q]));  // C - a I; A before its limbs
        }
    }
    __syncthreads();
    if (wave < tm * tm) each(c, ai, aj, [&](int i, int j, f32x4 v) { store_limbs(A + small_at(pa, i, j), la, v); });
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int b = wave + 16 * h;
#pragma unroll
      for (int mi = 0; mi < 2; ++mi)
#pragma unroll
        for (int ni = 0; ni < 2; ++ni) x[h][mi][ni] = zero;
      if (b < tm * tn) {
        small_block<KS>(A, pa, la, X, px, lx, b / tn * 32, b % tn * 32, mp, x[h]);
#pragma unroll
        for (int mi = 0; mi < 2; ++mi)
#pragma unroll
          for (int ni = 0; ni < 2; ++ni)
            x[h][mi][ni] += st.a[q] * load_limbs(X + small_at(px, b / tn * 32 + 16 * mi + (lane & 15), b % tn * 32 + 16 * ni + 4 * (lane >> 4)), lx);
      }
    }
    if (q + 1 == st.n) break;
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int b = wave + 16 * h;
      if (b < tm * tn)
        each(x[h], b / tn * 32, b % tn * 32, [&](int i, int j, f32x4 v) {
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = ldexpf(v[r], st.apply[q]);
          store_limbs(X + small_at(px, i, j), lx, v);
        });
    }
    __syncthreads();
  }
  const int shift = st.apply[st.n - 1];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int b = wave + 16 * h;
    if (b < tm * tn)
      each(x[h], b / tn * 32, b % tn * 32, [&](int i, int j, f32x4 v) {
        if (i >= m) return;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (j + r >= n) continue;
          const int64_t at = base + (tall ? (int64_t)(j + r) * it.ldp + i : (int64_t)i * it.ldp + j + r);
          const float y = ldexpf(v[r], shift);
          if (it.m) {
            float* p = (float*)it.p + at;
            *p = *p * s.decay - it.gain * y;
          } else {
            put(it.p, at, s.dtype, y);
          }
        }
      });
  }
}

inline int ok() { return hipGetLastError() == hipSuccess ? HOLD_OK : HOLD_E_LAUNCH; }

// The bounds of the singular values of X, and of the entries of A and C, through the iteration; false: they leave the range of the limbs
struct Bounds {
  int xs[33], as[33], cs[33];  // exponents of the scales of X, A, C: largest entry to below 2^14, a factor of 4 under fp16's range
};
bool follow(const float* coef, int steps, Bounds& o) {
  double r = 1.;
  for (int k = 0; k <= steps; ++k) {
    if (!(r < 1e9) || !(r > 1e-9)) return false;
    o.xs[k] = 14 - (int)ceil(log2(r));
    if (k == steps) break;
    o.as[k] = 14 - (int)ceil(2. * log2(r));
    const double a = coef[3 * k], b = coef[3 * k + 1], c = coef[3 * k + 2], S = r * r;
    if (!isfinite(a) || !isfinite(b) || !isfinite(c)) return false;
    auto P = [&](double s) { return fabs(a + b * s + c * s * s); };
    double top = fmax(fmax(P(0.), P(S)), fabs(b * S + c * S * S));  // of a I + C, and of C, which is what is stored
    if (c != 0. && -b / (2. * c) > 0. && -b / (2. * c) < S) top = fmax(fmax(top, P(-b / (2. * c))), fabs(b * b / (4. * c)));
    if (!(top < 1e9) || !(top > 1e-9)) return false;
    o.cs[k] = 14 - (int)ceil(log2(top));
    // the largest |s (a + b s^2 + c s^4)| on [0, r]: its ends and where a + 3 b s^2 + 5 c s^4 = 0
    double next = r * P(S);
    auto at = [&](double s2) {
      if (s2 > 0. && s2 < S) next = fmax(next, sqrt(s2) * P(s2));
    };
    if (c != 0.) {
      const double disc = 9. * b * b - 20. * a * c;
      if (disc >= 0.) {
        at((-3. * b + sqrt(disc)) / (10. * c));
        at((-3. * b - sqrt(disc)) / (10. * c));
      }
    } else if (b != 0.) {
      at(-a / (3. * b));
    }
    r = next;
  }
  return true;
}

inline int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

// the workspace of one group of items: partial sums, X twice, A and C, all limbs
struct Room {
  int64_t part, x, y, mm[2], xn, cn, bytes;
};
// sorts the items by shape, finds the classes and lays out the workspace
Room room(Items& a, Classes& cl) {
  auto small = [](const Item& i) { return i.rows < i.cols ? i.rows : i.cols; };
  auto large = [](const Item& i) { return i.rows < i.cols ? i.cols : i.rows; };
  for (int k = 1; k < a.n; ++k) {  // by insertion: equal shapes keep their order
    const Item it = a.it[k];
    int q = k;
    while (q > 0 && (small(a.it[q - 1]) > small(it) || (small(a.it[q - 1]) == small(it) && large(a.it[q - 1]) > large(it)))) {
      a.it[q] = a.it[q - 1];
      --q;
    }
    a.it[q] = it;
  }
  Room r = {};
  int64_t parts = 0, xn = 0, cn = 0;
  cl.n = 0;
  for (int k = 0; k < a.n; ++k) {
    Item& it = a.it[k];
    const int m = small(it), n = large(it);
    const int64_t mp = up8(m), np = up8(n), nb = ((int64_t)m * n + 4095) / 4096;
    it.nb = (int)(nb > 512 ? 512 : nb);
    it.part = (int)parts;
    it.x = xn;
    if (cl.n && it.count == 1 && a.it[cl.k[cl.n - 1].item].count == 1 && cl.k[cl.n - 1].m == m && cl.k[cl.n - 1].n == n) ++cl.k[cl.n - 1].mats;
    else cl.k[cl.n++] = Class{xn, cn, m, n, (int)mp, (int)np, it.count, k, 0};
    parts += (int64_t)it.nb * it.count;
    xn += mp * np * it.count;
    cn += mp * mp * it.count;
  }
  xn = up256(xn); cn = up256(cn);
  int64_t o = 0;
  auto take = [&](int64_t bytes) { const int64_t at = o; o += up256(bytes); return at; };
  r.part = take(parts * 8);
  r.x = take(xn * 4);
  r.y = take(xn * 4);
  for (int k = 0; k < 2; ++k) r.mm[k] = take(cn * 4);
  r.xn = xn; r.cn = cn;
  r.bytes = o;
  return r;
}

template <int KIND>
int64_t count_tiles(Classes& cl, int T) {
  int64_t n = 0;
  for (int k = 0; k < cl.n; ++k) {
    Class& c = cl.k[k];
    c.tile = (int)n;
    const int64_t tm = (c.mp + T - 1) / T, tn = (c.np + tile_cols<KIND>(T) - 1) / tile_cols<KIND>(T);
    n += (KIND == APPLY ? tm * tn : tm * (tm + 1) / 2) * c.mats;
    if (n > (1 << 30)) return -1;
  }
  return n;
}

template <int KIND, int T, int WM, int WN, int S, bool PHASED, bool LAST>
void launch_tiles(const Classes& cl, const NsArgs& s, const Step& st, const Items& a, unsigned n, hipStream_t stream) {
  typename ItemArg<LAST>::type items;
  if constexpr (LAST) items = a;
  if (cl.n == 1) {
    const OneClass one = {{cl.k[0]}, 1};
    hipLaunchKernelGGL((ns_mma_kernel<KIND, T, WM, WN, S, PHASED, LAST, OneClass>), dim3(n), dim3(64 * WM * WN), 0, stream, one, s, st, items);
  } else {
    hipLaunchKernelGGL((ns_mma_kernel<KIND, T, WM, WN, S, PHASED, LAST, Classes>), dim3(n), dim3(64 * WM * WN), 0, stream, cl, s, st, items);
  }
}

// The tile size by the launch's time, rounds of blocks over the 256 compute units at (per k + fixed) microseconds.  256 and 192: one block a
// unit; 128: two; 64 (three stages of LDS): three; a last round that leaves units with fewer blocks is shorter.  Fitted to launches alone
// on single matrices of 1500 .. 4096 and batches of 256 .. 1024 rows, each with every tile size: 4096^3 takes 255 us in 256 x 256
// tiles, 2 x 154 in 128, 5.3 x 119 in 64; 36 matrices of 256 x 256 in 64 8 us a product, 14 in 128.  Where
// a launch of 64 is latency more than work it takes shorter ways: up to two blocks a unit (APPLY: one) in tiles of 32 x 32 (32 x 64) with
// four stages of 64, sums up to 256 requested at once (a 256 x 256 matrix 110 -> 80 us, 3 x 1531 x 517 in 16 bits 273 -> 232; with more
// blocks the loads count: 1024 x 1024 280 -> 295); else up to two blocks a unit with eight waves in steps of 64 (1024 x 1024 280 -> 245,
// 16 x 256 x 256 123 -> 110; above, three blocks of four waves: 48 x 256 x 256 205 against 210).  Tiles of 128 in phases where both
// operands are read by rows: GRAM of 6 x 1024 x 4096 124 -> 113 us; APPLY's 175 stay 174.
struct TileCost {
  int size, units;                   // rows; blocks of a full round
  double full[2], two[2], alone[2];  // a round: full, of up to 512 blocks (64), of up to 256
};
const TileCost COST[4] = {{256, 256, {.0535, 36.}, {.0535, 36.}, {.0535, 36.}},
                          {192, 256, {.0535, 6.}, {.0535, 6.}, {.0535, 6.}},
                          {128, 512, {.034, 15.}, {.034, 15.}, {.026, 13.}},
                          {64, 768, {.025, 3.}, {.016, 4.}, {.012, 4.}}};

template <int KIND, bool LAST>
int launch(Classes& cl, const NsArgs& s, const Step& st, const Items& a, hipStream_t stream) {
  double K = 0.;  // the longest sum
  for (int k = 0; k < cl.n; ++k) K = fmax(K, KIND == GRAM ? cl.k[k].np : cl.k[k].mp);
  int best = -1;
  double least = 0.;
  for (int k = 0; k < 4; ++k) {
    const TileCost& c = COST[k];
    const int64_t n = count_tiles<KIND>(cl, c.size);
    if (n < 0) continue;
    const int64_t rest = n % c.units;
    const double* last = rest <= 256 ? c.alone : rest <= 512 ? c.two : c.full;
    const double t = (double)(n / c.units) * (K * c.full[0] + c.full[1]) + (rest ? K * last[0] + last[1] : 0.);
    if (best < 0 || t < least) { best = k; least = t; }
  }
  if (best < 0) return HOLD_E_ARG;
  const int64_t few = best == 3 ? count_tiles<KIND>(cl, 32) : -1;
  if (few > 0 && few <= (KIND == APPLY ? 256 : 512)) {
    launch_tiles<KIND, 32, 2, 2, 4, false, LAST>(cl, s, st, a, (unsigned)few, stream);
    return HOLD_OK;
  }
  const unsigned n = (unsigned)count_tiles<KIND>(cl, COST[best].size);
  if (best == 0) launch_tiles<KIND, 256, 4, 4, 2, true, LAST>(cl, s, st, a, n, stream);
  else if (best == 1) launch_tiles<KIND, 192, 3, 4, 2, true, LAST>(cl, s, st, a, n, stream);
  else if (best == 2) launch_tiles<KIND, 128, 2, 4, 2, KIND != APPLY, LAST>(cl, s, st, a, n, stream);
  else if (n <= 512) launch_tiles<KIND, 64, 2, 4, 2, false, LAST>(cl, s, st, a, n, stream);
  else launch_tiles<KIND, 64, 2, 2, 3, false, LAST>(cl, s, st, a, n, stream);
  return HOLD_OK;
}

int run_group(Items& a, const Step& st, const float* coef, int steps, char* ws, hipStream_t stream) {
  Bounds bo;
  if (!follow(coef, steps, bo)) return HOLD_E_ARG;
  Classes cl;
  const Room r = room(a, cl);
  double* part = (double*)(ws + r.part);
  uint16_t* x = (uint16_t*)(ws + r.x);
  uint16_t* y = (uint16_t*)(ws + r.y);
  uint16_t* mm[2] = {(uint16_t*)(ws + r.mm[0]), (uint16_t*)(ws + r.mm[1])};
  Firsts tn = {}, tl = {};
  int64_t nn = 0, nl = 0;
  for (int k = 0; k < a.n; ++k) {
    const Item& it = a.it[k];
    tn.first[k] = (int)nn;
    tl.first[k] = (int)nl;
    nn += (int64_t)it.nb * it.count;
    nl += (int64_t)((up8(it.rows) + 63) / 64) * ((up8(it.cols) + 63) / 64) * it.count;
    if (nn > (1 << 30) || nl > (1 << 30)) return HOLD_E_ARG;
  }
  if (count_tiles<APPLY>(cl, 256) < 0) return HOLD_E_ARG;
  hipLaunchKernelGGL(ns_norm_kernel, dim3((unsigned)nn), dim3(256), 0, stream, a, tn, st, part);
  hipLaunchKernelGGL(ns_load_kernel, dim3((unsigned)nl), dim3(256), 0, stream, a, tl, st, part, x, r.xn, bo.xs[0]);
  NsArgs s = {};
  s.xlimb = r.xn;
  s.climb = r.cn;
  int rc = HOLD_OK;
  auto gram = [&](int k) {
    s.x = x;
    s.o = mm[0];
    s.shift = bo.as[k] - 2 * bo.xs[k];
    if (rc == HOLD_OK) rc = launch<GRAM, false>(cl, s, st, a, stream);
  };
  auto poly = [&](int k) {  // C without a I
    s.l = mm[0];
    s.o = mm[1];
    s.b = (float)ldexp((double)coef[3 * k + 1], bo.cs[k] - bo.as[k]);
    s.c = (float)ldexp((double)coef[3 * k + 2], bo.cs[k] - 2 * bo.as[k]);
    if (rc == HOLD_OK) rc = launch<POLY, false>(cl, s, st, a, stream);
  };
  auto apply = [&](int k) {
    const bool last = k + 1 == steps;
    s.a = (float)ldexp((double)coef[3 * k], bo.cs[k]);
    s.l = mm[1];
    s.x = x;
    s.y = y;
    s.shift = (last ? 0 : bo.xs[k + 1]) - bo.cs[k] - bo.xs[k];
    if (rc == HOLD_OK) rc = last ? launch<APPLY, true>(cl, s, st, a, stream) : launch<APPLY, false>(cl, s, st, a, stream);
    uint16_t* z = x;
    x = y;
    y = z;
  };
  for (int k = 0; k < steps; ++k) {
    gram(k);
    poly(k);
    apply(k);
  }
  return rc == HOLD_OK ? ok() : rc;
}

int run_small(const Items& a, const Step& st, const float* coef, int steps, hipStream_t stream) {
  Bounds bo;
  if (!follow(coef, steps, bo)) return HOLD_E_ARG;
  SmallSteps ss = {};
  ss.n = steps;
  ss.xs = bo.xs[0];
  for (int k = 0; k < steps; ++k) {
    ss.gram[k] = bo.as[k] - 2 * bo.xs[k];
    ss.a[k] = (float)ldexp((double)coef[3 * k], bo.cs[k]);
    ss.b[k] = (float)ldexp((double)coef[3 * k + 1], bo.cs[k] - bo.as[k]);
    ss.c[k] = (float)ldexp((double)coef[3 * k + 2], bo.cs[k] - 2 * bo.as[k]);
    ss.apply[k] = (k + 1 == steps ? 0 : bo.xs[k + 1]) - bo.cs[k] - bo.xs[k];
  }
  Firsts t = {};
  int64_t n = 0;
  for (int k = 0; k < a.n; ++k) {
    t.first[k] = (int)n;
    n += a.it[k].count;
    if (n > (1 << 30)) return HOLD_E_ARG;
  }
  hipLaunchKernelGGL(ns_small_kernel, dim3((unsigned)n), dim3(1024), 0, stream, a, t, st, ss);
  return ok();
}

bool sizes_ok(int64_t rows, int64_t cols, int64_t count) {
  return rows >= 1 && cols >= 1 && count >= 1 && rows <= (1 << 20) && cols <= (1 << 20) && count <= (1 << 24);
}
bool one_item(const hold_ortho_desc* d, Items& a) {
  if (!d || !sizes_ok(d->rows, d->cols, d->batch)) return false;
  a.n = 1;
  Item& it = a.it[0];
  it = Item{};
  it.rows = d->rows;
  it.cols = it.ldg = it.ldm = it.ldp = d->cols;
  it.count = d->batch;
  it.stride = (int64_t)d->rows * d->cols;
  return true;
}
bool read_item(const hold_muon_desc* d, int k, Item& it) {
  const hold_muon_item& i = d->items[k];
  if (!sizes_ok(i.rows, i.cols, 1) || i.ldp < i.cols || i.ldg < i.cols || i.ldm < i.cols) return false;
  it = Item{};
  it.g = i.g; it.m = i.m; it.p = i.p;
  it.rows = i.rows; it.cols = i.cols; it.count = 1;
  it.ldg = i.ldg; it.ldm = i.ldm; it.ldp = i.ldp;
  it.gain = (float)(d->lr * i.scale);
  return true;
}
// a launch has less than 2^32 threads: a batch that would pass 2^21 blocks goes in parts, one after the other in the same workspace
int32_t part_of(const Item& it, int steps) {
  if (small(it, steps)) return 1 << 21;
  const int64_t blocks = ((int64_t)it.rows + 71) / 64 * (((int64_t)it.cols + 71) / 64) + 512, n = (1 << 21) / blocks;
  return n < 1 ? 1 : (int32_t)n;
}
// calls f(items, little) for the groups of a step, up to MAXI items that are computed alike: in one block's LDS each (little), or all in
// every launch; false: a bad item
template <class F>
bool groups_of(const hold_muon_desc* d, F f) {
  for (const bool little : {false, true}) {
    Items a;
    a.n = 0;
    for (int k = 0; k < d->n_items; ++k) {
      Item it;
      if (!read_item(d, k, it)) return false;
      if (small(it, d->steps) != little) continue;
      a.it[a.n++] = it;
      if (a.n == MAXI) {
        if (!f(a, little)) return false;
        a.n = 0;
      }
    }
    if (a.n && !f(a, little)) return false;
  }
  return true;
}

}  // namespace

extern "C" int hold_orthogonalize_workspace(const hold_ortho_desc* d, int64_t* bytes) {
  Items a;
  Classes cl;
  if (!one_item(d, a) || !bytes) return HOLD_E_ARG;
  const int32_t part = part_of(a.it[0], d->steps);
  if (a.it[0].count > part) a.it[0].count = part;
  *bytes = small(a.it[0], d->steps) ? 256 : room(a, cl).bytes;
  return HOLD_OK;
}

extern "C" int hold_orthogonalize(const hold_ortho_desc* d, hold_stream_t stream) {
  Items a;
  int64_t need = 0;
  if (hold_orthogonalize_workspace(d, &need) != HOLD_OK || !d->workspace || need > d->workspace_bytes || !one_item(d, a)) return HOLD_E_ARG;
  if (!d->x || !d->out || !d->coef || d->steps < 1 || d->steps > 32 || d->dtype < 0 || d->dtype > 2 || !(d->eps >= 0.f)) return HOLD_E_ARG;
  Step st = {};
  st.eps = d->eps;
  st.dtype = d->dtype;
  const Item whole = a.it[0];
  const int64_t bytes = whole.stride * (d->dtype == HOLD_MUON_F32 ? 4 : 2);
  const int32_t part = part_of(whole, d->steps);
  for (int32_t k = 0; k < d->batch; k += part) {
    Item& it = a.it[0] = whole;
    it.g = (const char*)d->x + k * bytes;
    it.p = (char*)d->out + k * bytes;
    it.count = d->batch - k < part ? d->batch - k : part;
    const int rc = small(whole, d->steps) ? run_small(a, st, d->coef, d->steps, (hipStream_t)stream)
                                          : run_group(a, st, d->coef, d->steps, (char*)d->workspace, (hipStream_t)stream);
    if (rc != HOLD_OK) return rc;
  }
  return HOLD_OK;
}

extern "C" int hold_muon_workspace(const hold_muon_desc* d, int64_t* bytes) {
  if (!d || !bytes || d->n_items < 1 || !d->items) return HOLD_E_ARG;
  *bytes = 256;
  return groups_of(d, [&](Items& a, bool little) {
    if (little) return true;
    Classes cl;
    const int64_t n = room(a, cl).bytes;
    if (n > *bytes) *bytes = n;
    return true;
  }) ? HOLD_OK : HOLD_E_ARG;
}

extern "C" int hold_muon_step(const hold_muon_desc* d, hold_stream_t stream) {
  int64_t need = 0;
  Bounds bo;
  if (hold_muon_workspace(d, &need) != HOLD_OK || !d->workspace || need > d->workspace_bytes) return HOLD_E_ARG;
  if (!d->coef || d->steps < 1 || d->steps > 32 || !(d->eps >= 0.f) || !follow(d->coef, d->steps, bo)) return HOLD_E_ARG;
  for (int k = 0; k < d->n_items; ++k)
    if (!d->items[k].p || !d->items[k].g || !d->items[k].m) return HOLD_E_ARG;
  Step st = {};
  st.eps = d->eps;
  st.dtype = HOLD_MUON_F32;
  st.mu = (float)d->momentum;
  st.rest = (float)(1.0 - d->momentum);
  st.nesterov = d->nesterov;
  st.decay = (float)(1.0 - d->lr * d->weight_decay);
  st.grad_mul = d->grad_mul;
  st.clip = d->clip_norm;
  st.sumsq = d->sumsq;
  int rc = HOLD_OK;  // groups share the workspace: they run one after the other
  groups_of(d, [&](Items& a, bool little) {
    rc = little ? run_small(a, st, d->coef, d->steps, (hipStream_t)stream)
                : run_group(a, st, d->coef, d->steps, (char*)d->workspace, (hipStream_t)stream);
    return rc == HOLD_OK;
  });
  return rc;
}
