// Tiled products on the matrix cores, the core of gated.hip and muon.hip:   acc[i][j] += sum_k A(i, k) B(j, k).
//
// ARITHMETIC.  MODE_BF16: bf16 operands, v_mfma_f32_16x16x32_bf16.  MODE_F16X3: fp32 operands as two fp16 limbs, x 2^e = hi + lo
// with hi = RN_f16(x 2^e), lo = RN_f16(x 2^e - hi) and the three limb products hi hi + hi lo + lo hi on v_mfma_f32_16x16x32_f16: the
// dropped lo lo and the second rounding are <= 2^-22 of a product each (fp32's own rounding: 2^-24) where both factors are within 2^-17 of
// the largest value that shares their scale; below that the error is 2^-39 of that largest value.  MODE_F32: fp32 operands as they are,
// v_mfma_f32_16x16x4_f32, a sixteenth of the 16-bit rate: every product and sum rounds as fp32 does, whatever the operands' range, and
// infinities and NaN stay where the formula has them.  Accumulation is fp32 in all three.
//
// OPERANDS.  Each of the two may lie in memory with k contiguous (KC: [row][k]) or with the rows contiguous (KS: [k][row]): no
// transposed copy is ever made.  KC fragments are ds_read_b128; KS fragments are a pair of ds_read_b64_tr_b16, each of which hands
// lane c of a 16-lane group column c of the 4 x 16 block that the group's lanes address (fp32: four ds_read_b32).  Both come from LDS tiles that
// buffer_load_dwordx4 ... lds fills directly; the 16-byte chunks of a tile row are permuted (on the global side, since the LDS side is
// linear) so that the 16 rows that a fragment touches spread over all 64 banks.
//
// EDGES.  The buffer descriptor ends at the operand's last element, so rows behind it and k behind K arrive as zeros; a k tail inside
// a KC row is masked per 16-byte chunk.  Required, and ensured by the callers' checks or padded copies: 16-byte aligned bases, leading
// dimensions in multiples of 16 bytes, K (KC) resp. row count (KS) rounded up to 16 bytes inside the allocation.
//
// PIPELINE.  S LDS stages: the loads of the next S - 1 steps are in flight while one is multiplied; one s_waitcnt + s_barrier a step.
#ifndef HOLD_TILE16_H
#define HOLD_TILE16_H
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace t16 {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void lds_void;

enum { MODE_BF16 = 0, MODE_F16X3 = 1, MODE_F32 = 2 };
enum { KC = 0, KS = 1 };
constexpr uint32_t OOB = 0xC0000000u;  // a byte offset behind every descriptor's end

template <int MODE> constexpr int limbs() { return MODE == MODE_F16X3 ? 2 : 1; }
template <int MODE> constexpr int step_k() { return MODE == MODE_BF16 ? 64 : 32; }
template <int MODE> constexpr int halves() { return MODE == MODE_F32 ? 2 : 1; }  // of 16 bits in an element

// one operand of a tile: `p` points at the tile's first row and k = 0 (KC: row-major rows; KS: its first column at k = 0)
struct Operand {
  const uint16_t* p;
  int64_t limb;  // elements from the hi array to the lo array (MODE_F16X3)
  int64_t ld;
  int64_t rows;  // rows of the operand from the tile's first one on (KS: columns, rounded up to 16 bytes)
  int64_t k;     // k's of the operand (KC: rounded up to 16 bytes, the last ones zeros); the shorter of the two ends in zeros
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// LDS tile of R rows x BK k's of one limb, E halves an element
template <int LAY, int R, int BK, int E>
struct Tile {
  static constexpr int RB = (LAY == KC ? BK : R) * 2 * E;  // bytes of a tile row
  static constexpr int NR = LAY == KC ? R : BK;         // tile rows
  static constexpr int C = RB / 16;                     // 16-byte chunks of a tile row
  static constexpr int BYTES = RB * NR;
  static constexpr int PIECES = BYTES / 1024;           // wave-wide 16-byte loads
  static_assert(E == 1 || LAY == KC || C % 16 == 0, "fp32 by k: whole 256 bytes");
  static_assert((LAY == KC ? C == 4 || C == 8 : C % 8 == 0) && BYTES % 1024 == 0, "tile rows of 64 or 128 bytes (KC), multiples of 128 (KS): the exchange of chunks stays inside a row");
  static __device__ __forceinline__ int swz(int row) {
    // a 16-byte read is served 16 lanes at a time: of two neighbouring 16-lane groups (two chunks), rows 0-3 and 12-15 of one with
    // rows 4-11 of the other
    if (LAY == KC) return C == 8 ? ((row >> 1) & 7) : (-(row >> 2) & 3);
    // fp32: a read touches 64 bytes of each of four rows k, four apart: each in another quarter of the banks
    if (E == 2) return 4 * ((row >> 2) & 3);
    // of the 16 rows k that a transposing read touches, 8 at a time: by the whole 256 bytes of the banks where a row is a multiple of
    // that; where it is an odd multiple of 128 its parity already moves it by half of them
    return C % 16 == 0 ? 2 * ((row & 3) | ((row >> 1) & 4)) : 2 * (((row >> 1) & 1) | ((row >> 2) & 2));
  }
};

// loads of one operand's tile; `first` = index of the wave's first piece, `stride` = waves
template <int LAY, int R, int BK, int NW, int E>
struct Loader {
  using T = Tile<LAY, R, BK, E>;
  static_assert(R * E <= 256, "lengths in 32 bits");
  static constexpr int N = (T::PIECES + NW - 1) / NW;
  static constexpr bool EVEN = T::PIECES % NW == 0;
  uint32_t off[N];
  int kk[N];  // first k of the lane's chunk inside the step (KC)

  __device__ __forceinline__ void init(int wave, int lane, int64_t ld) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int q = (wave + i * NW) * 64 + lane, row = q / T::C, chunk = (q % T::C) ^ T::swz(row);
      off[i] = (uint32_t)(row * (int)ld * 2 * E + chunk * 16);
      kk[i] = chunk * 8 / E;
    }
  }
  // k0: first k of the step; lds: the tile's place in LDS
  __device__ __forceinline__ void load(const Operand& o, int limb, int64_t k0, char* lds, int wave) const {
    // lengths in 32 bits: at most 256 / E rows (KC) or BK rows (KS) of at most 2^21 elements
    const uint16_t* p = o.p + (limb * o.limb + (LAY == KC ? k0 : k0 * o.ld)) * E;
    const int64_t left = o.k - k0;
    const int kend = left < BK ? (int)left : BK, rows = o.rows < R ? (int)o.rows : R;
    const int len = (LAY == KC ? (rows - 1) * (int)o.ld + kend : (kend - 1) * (int)o.ld + rows) * 2 * E;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(p), 0, kend > 0 && rows > 0 ? len : 0, 0x00020000);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!EVEN && wave + i * NW >= T::PIECES) break;
      const uint32_t v = (LAY == KC && kk[i] >= kend) ? OOB : off[i];
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(lds + (wave + i * NW) * 1024), 16, v, 0, 0, 0);
    }
  }
};

// the wave's fragments: 16 rows x 32 k's, lane l: row l % 16, k = 8 (l / 16) + 0..7 (fp32: 16 k's, 4 (l / 16) + 0..3)
template <int LAY, int R, int BK, int E>
struct Reader {
  using T = Tile<LAY, R, BK, E>;
  static constexpr int G = BK * E / 32;  // fragments along a step
  int base[LAY == KC ? G : 1];
  int s;
  __device__ __forceinline__ void init(int lane) {
    if (LAY == KC) {
      const int row = lane & 15;
#pragma unroll
      for (int ks = 0; ks < (LAY == KC ? G : 1); ++ks) base[ks] = row * T::RB + (((ks * 4 + (lane >> 4)) ^ T::swz(row)) * 16);
      s = 0;
    } else if (E == 2) {
      const int k = 4 * (lane >> 4);
      base[0] = k * T::RB + (lane & 15) * 4;
      s = T::swz(k) * 16;
    } else {
      const int k = 8 * (lane >> 4) + ((lane & 15) >> 2);
      base[0] = k * T::RB + ((lane & 3) >> 1) * 16 + (lane & 1) * 8;
      s = T::swz(k) * 16;
    }
  }
  __device__ __forceinline__ s16x8 frag(const char* lds, int row0, int ks) const {
    if (LAY == KC) return *(const s16x8*)(lds + base[ks] + row0 * T::RB);
    const char* a = lds + base[0] + ((row0 * 2 * E) ^ s) + ks * (32 / E) * T::RB;
    if (E == 2) {
      f32x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = *(const float*)(a + i * T::RB);
      return __builtin_bit_cast(s16x8, v);
    }
    const s16x4 u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)a);
    const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(a + 4 * T::RB));
    return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

template <int MODE>
__device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
  if (MODE == MODE_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// A block of WM x WN waves computes a BM x BN tile for each of NB operands B that share A.  The matrix instruction's first operand
// is B: a lane then holds FOUR CONSECUTIVE j of ONE row i, so results leave as 8- or 16-byte stores:
//   acc[b][mi][ni][r]:  i = wm BM / WM + 16 mi + lane % 16,   j = wn BN / WN + 16 ni + 4 (lane / 16) + r
template <int MODE, int LA, int LB, int BM, int BN, int NB, int WM, int WN, int S = 2, int BK_ = step_k<MODE>()>
struct Core {
  static constexpr int BK = BK_, NL = limbs<MODE>(), NW = WM * WN, E = halves<MODE>();
  static constexpr int MI = BM / WM / 16, NI = BN / WN / 16;
  using TA = Tile<LA, BM, BK, E>;
  using TB = Tile<LB, BN, BK, E>;
  static constexpr int STAGE = NL * (TA::BYTES + NB * TB::BYTES), LDS = S * STAGE;
  static constexpr int THREADS = 64 * NW;
  typedef f32x4 Acc[NB][MI][NI];

  static __device__ __forceinline__ void zero(Acc& acc) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[b][i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // matrix instructions of rows i0 .. i0 + n - 1 of the tile with all columns; the three limb products one after the other over the
  // columns, the small ones first (they meet the smaller partial sum), so that no instruction waits for the one before it
  template <int N>
  static __device__ __forceinline__ void rows_mfma(const s16x8 (&fa)[N][NL], const s16x8 (&fb)[NB][NI][NL], Acc& acc, int i0) {
    if constexpr (MODE == MODE_F32) {  // the k's 4 (l / 16) + q of the fragments feed instruction q
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < NI; ++j) {
              const f32x4 x = __builtin_bit_cast(f32x4, fa[i][0]), y = __builtin_bit_cast(f32x4, fb[b][j][0]);
              acc[b][i0 + i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(y[q], x[q], acc[b][i0 + i][j], 0, 0, 0);
            }
      return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int p = NL == 2 ? 0 : 2; p < 3; ++p)
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int j = 0; j < NI; ++j) acc[b][i0 + i][j] = mfma<MODE>(fb[b][j][p == 0 ? NL - 1 : 0], fa[i][p == 1 ? NL - 1 : 0], acc[b][i0 + i][j]);
  }

  // The same sums as run(), software-pipelined inside a wave: a step is cut into phases of half the tile's rows and 32 k's; while a
  // phase's matrix instructions run, the next phase's fragments are read.  The last phase of a step already reads the next stage, so the
  // barrier stands in the middle of the arithmetic, and the loads issued behind it have a whole step to arrive.
  // the order of a phase: its LDS reads and its loads spread evenly between its matrix instructions
  template <int M, int D, int V, int g = 0>
  static __device__ __forceinline__ void interleave() {
    constexpr int G = M < 16 ? M : 16;
    if constexpr (g < G) {
      constexpr int m = M * (g + 1) / G - M * g / G, v = V * (g + 1) / G - V * g / G, d = D * (g + 1) / G - D * g / G;
      if constexpr (m > 0) __builtin_amdgcn_sched_group_barrier(0x8, m, 0);
      if constexpr (v > 0) __builtin_amdgcn_sched_group_barrier(0x10, v, 0);
      if constexpr (d > 0) __builtin_amdgcn_sched_group_barrier(0x100, d, 0);
      interleave<M, D, V, g + 1>();
    }
  }

  static __device__ __forceinline__ void run_phased(char* smem, const Operand& A, const Operand (&B)[NB], Acc& acc) {
    static_assert(S == 2 && MI % 2 == 0 && MODE != MODE_F32, "two stages, halves of the rows");
    constexpr int HA = MI / 2, Q = 2 * (BK / 32), P = NL == 2 ? 3 : 1;
    constexpr int RA = LA == KC ? 1 : 2, RB = LB == KC ? 1 : 2;  // LDS reads a fragment
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
    Loader<LA, BM, BK, NW, E> la;
    Loader<LB, BN, BK, NW, E> lb[NB];
    la.init(wave, lane, A.ld);
#pragma unroll
    for (int b = 0; b < NB; ++b) lb[b].init(wave, lane, B[b].ld);
    Reader<LA, BM, BK, E> ra;
    Reader<LB, BN, BK, E> rb;
    ra.init(lane);
    rb.init(lane);
    const int nk = (int)((A.k + BK - 1) / BK);
    auto stage_a = [&](int kt, char* s) {
#pragma unroll
      for (int l = 0; l < NL; ++l) la.load(A, l, (int64_t)kt * BK, s + l * TA::BYTES, wave);
    };
    auto stage_b = [&](int kt, char* s) {
#pragma unroll
      for (int l = 0; l < NL; ++l)
#pragma unroll
        for (int b = 0; b < NB; ++b) lb[b].load(B[b], l, (int64_t)kt * BK, s + NL * TA::BYTES + (b * NL + l) * TB::BYTES, wave);
    };
    constexpr int VA = NL * Loader<LA, BM, BK, NW, E>::N, VB = NL * NB * Loader<LB, BN, BK, NW, E>::N;
    s16x8 fa[2][HA][NL], fb[NB][NI][NL];
    auto read_a = [&](s16x8 (&f)[HA][NL], const char* s, int q) {
#pragma unroll
      for (int i = 0; i < HA; ++i)
#pragma unroll
        for (int l = 0; l < NL; ++l) f[i][l] = ra.frag(s + l * TA::BYTES, wm * (BM / WM) + 16 * (i + (q & 1) * HA), q >> 1);
    };
    auto read_b = [&](int b, int j, const char* s, int ks) {
#pragma unroll
      for (int l = 0; l < NL; ++l) fb[b][j][l] = rb.frag(s + NL * TA::BYTES + (b * NL + l) * TB::BYTES, wn * (BN / WN) + 16 * j, ks);
    };
    stage_a(0, smem);
    stage_b(0, smem);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (nk > 1) stage_a(1, smem + STAGE);
    read_a(fa[0], smem, 0);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int j = 0; j < NI; ++j) read_b(b, j, smem, 0);
    for (int kt = 0; kt < nk; ++kt) {
      char* s = smem + (kt & 1) * STAGE;
      char* t = smem + ((kt + 1) & 1) * STAGE;
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const bool last = q == Q - 1;
        const char* next = last ? t : s;  // behind the last step: leftovers of the other stage, read and never used
        if (last) {
          asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
          stage_a(kt + 2, s);  // behind the last step the descriptor is empty: zeros, waited for below
        }
        if ((q & 1) == 0) {
          if (q == 0) stage_b(kt + 1, t);
          read_a(fa[1], next, q + 1);
          rows_mfma<HA>(fa[0], fb, acc, 0);
          if (q == 0) interleave<HA * NB * NI * P, HA * NL * RA, VB>();
          else interleave<HA * NB * NI * P, HA * NL * RA, 0>();
        } else {
          read_a(fa[0], next, last ? 0 : q + 1);
          // column by column: a column's fragments are read anew as soon as its last product is issued
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < NI; ++j) {
#pragma unroll
              for (int p = NL == 2 ? 0 : 2; p < 3; ++p)
#pragma unroll
                for (int i = 0; i < HA; ++i) acc[b][HA + i][j] = mfma<MODE>(fb[b][j][p == 0 ? NL - 1 : 0], fa[1][i][p == 1 ? NL - 1 : 0], acc[b][HA + i][j]);
              read_b(b, j, next, last ? 0 : (q + 1) >> 1);
            }
          if (last) interleave<HA * NB * NI * P, HA * NL * RA + NB * NI * NL * RB, VA>();
          else interleave<HA * NB * NI * P, HA * NL * RA + NB * NI * NL * RB, 0>();
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    // also the loads behind the last step, which write zeros: the caller may use the stages at once
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }

  // A.k > 0.  Ends with every wave past its last read of the LDS stages.
  static __device__ __forceinline__ void run(char* smem, const Operand& A, const Operand (&B)[NB], Acc& acc) {
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
    Loader<LA, BM, BK, NW, E> la;
    Loader<LB, BN, BK, NW, E> lb[NB];
    la.init(wave, lane, A.ld);
#pragma unroll
    for (int b = 0; b < NB; ++b) lb[b].init(wave, lane, B[b].ld);
    Reader<LA, BM, BK, E> ra;
    Reader<LB, BN, BK, E> rb;
    ra.init(lane);
    rb.init(lane);
    const int nk = (int)((A.k + BK - 1) / BK);
    auto stage = [&](int kt, char* s) {
#pragma unroll
      for (int l = 0; l < NL; ++l) {
        la.load(A, l, (int64_t)kt * BK, s + l * TA::BYTES, wave);
#pragma unroll
        for (int b = 0; b < NB; ++b) lb[b].load(B[b], l, (int64_t)kt * BK, s + NL * TA::BYTES + (b * NL + l) * TB::BYTES, wave);
      }
    };
    // loads a wave issues per stage: the same for every wave, or S == 2
    constexpr int LPS = NL * (Loader<LA, BM, BK, NW, E>::N + NB * Loader<LB, BN, BK, NW, E>::N), AHEAD = (S - 2) * LPS;
    static_assert(S == 2 || (Loader<LA, BM, BK, NW, E>::EVEN && Loader<LB, BN, BK, NW, E>::EVEN && AHEAD < 63), "countable loads");
    const bool all = S > 2 && nk <= S;  // a sum that fits: one wait for everything
#pragma unroll
    for (int i = 0; i < S - 1; ++i)
      if (i < nk) stage(i, smem + i * STAGE);
    if (all && nk == S) stage(S - 1, smem + (S - 1) * STAGE);
    int at = 0, to = S - 1;  // the stage that is read, the stage that is filled
    for (int kt = 0; kt < nk; ++kt) {
      const char* s = smem + at * STAGE;
      if (!all || kt == 0) {
        // (the wave's own reads of the stage that is filled next are done too)
        if (S == 2 || all || kt + S - 1 > nk) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(AHEAD) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      }
      if (!all && kt + S - 1 < nk) stage(kt + S - 1, smem + to * STAGE);
      at = at + 1 == S ? 0 : at + 1;
      to = to + 1 == S ? 0 : to + 1;
      const char* sa = s;
      const char* sb = s + NL * TA::BYTES;
#pragma unroll
      for (int ks = 0; ks < BK * E / 32; ++ks) {
        s16x8 fb[NB][NI][NL];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int l = 0; l < NL; ++l) fb[b][j][l] = rb.frag(sb + (b * NL + l) * TB::BYTES, wn * (BN / WN) + 16 * j, ks);
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          s16x8 fa[1][NL];
#pragma unroll
          for (int l = 0; l < NL; ++l) fa[0][l] = ra.frag(sa + l * TA::BYTES, wm * (BM / WM) + 16 * i, ks);
          rows_mfma<1>(fa, fb, acc, i);
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
};

// Block -> tile.  Consecutive blocks go to the 8 XCDs in turn and each has its own L2: XCD x gets the x-th contiguous eighth of the
// tile list, and the list walks bands of `band` row tiles so that the tiles in flight on an XCD share their operands.
__device__ __forceinline__ void tile_of(int id, int total, int tm, int tn, int band, int& m, int& n) {
  const int q = total / 8, r = total % 8, x = id % 8, i = id / 8;
  const int t = x * q + (x < r ? x : r) + i;
  const int per = band * tn, b = t / per, first = b * band, h = (tm - first) < band ? (tm - first) : band;
  m = first + (t - b * per) % h;
  n = (t - b * per) / h;
}

__device__ __forceinline__ uint16_t bf16_bits(float x) {
  return __builtin_bit_cast(uint16_t, (__bf16)x);
}
__device__ __forceinline__ float bf16_value(uint16_t b) { return __builtin_bit_cast(float, (uint32_t)b << 16); }

struct Split {
  uint16_t hi, lo;
};
// hi + lo of an already scaled value; a value that is not finite has no low limb
__device__ __forceinline__ Split split16(float x) {
  const _Float16 h = (_Float16)x;
  const float r = x - (float)h;
  const _Float16 l = (_Float16)(r == r && fabsf(r) < 65504.f ? r : 0.f);
  return {__builtin_bit_cast(uint16_t, h), __builtin_bit_cast(uint16_t, l)};
}

// exponent e with |x| < 2^e for |x| <= m (m finite and > 0; subnormals count as 2^-126)
__device__ __forceinline__ int exp_above(float m) {
  const int e = (int)((__builtin_bit_cast(uint32_t, m) >> 23) & 0xffu) - 126;
  return e < -125 ? -125 : e;
}
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < __builtin_inff() ? a : 0.f;  // infinities and NaN count as nothing: they pass the limb split by themselves
}

}  // namespace t16
#endif
