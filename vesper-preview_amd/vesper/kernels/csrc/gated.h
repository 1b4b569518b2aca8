// What the gated delta rule's kernels share (gated_scan.hip, gated_backward.hip): matrix operands in
// pieces, their way through LDS, the chunk's coefficients and factors in the workspace.
//
// The rule per head, state H [D, D] (key rows, value columns), log decay g_t:
//   H_t = e^{g_t} H_{t-1} + k_t u_t^T,  u_t = beta_t (v_t - e^{g_t} H_{t-1}^T k_t),  o_t = H_t^T q_t.
// A chunk of C = 64 tokens with G_i = g_1 + .. + g_i, eps_i = e^{G_i}, E_ij = e^{G_i - G_j} (j <= i),
// kap_j = e^{G_C - G_j}, gam = e^{G_C}, A_ij = beta_i E_ij k_i.k_j (j < i), T = (I + A)^-1,
// P_ij = E_ij q_i.k_j:
//   R_i = beta_i (v_i - eps_i H^T k_i),  Delta = T R,  O_i = eps_i H^T q_i + sum_j W_ij R_j with W = P T,
//   H' = gam H + sum_j kap_j k_j Delta_j^T.
// Every exponent is at most zero where g is, so nothing overflows however far a state decays. The sums
// G and their differences are in float64: behind a token that forgets (g of -inf counts as -1e4, whose
// exponential is zero all the same) the sums are large and their differences are not.
//
// Precision: inputs in bf16 are exact MFMA operands. What the kernels compute in float32 and multiply
// again (H, R, Delta, T, their gradients) goes into bf16 MFMA as the sum of kPieces bf16 numbers, each the
// rounding of what the ones before it leave, and a product takes the pairs of pieces whose indices sum to
// less than kPieces. Three pieces hold 24 bits, float32's own; six bf16 MFMAs (three where one operand is
// an input) at 16 cycles a 16x16x32 tile each are 2.7 (5.3) times faster than float32 MFMA's 256 cycles.
// With two pieces the states were off by 4e-6 of their norm and dg by 8e-6, with three by less than 1e-7
// besides the accumulators' float32 rounding. Inputs in float32 go through float32 MFMA.
#pragma once

#include "common.h"

namespace vsp {
namespace gated {

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

constexpr int kChunk = 64;
constexpr int kPieces = 3;
constexpr double kLeastDecay = -1e4;  // log decays below it: their exponentials are zero either way

// ---- operands: 32 of a product's k a step, eight a lane; lane (c, g) = (l % 16, l / 16) holds row or column c. Where
// operands meet accumulators the k run in the order of a pair of accumulator tiles (rows 4 g + r of the first, then of the
// second), so that a pair of tiles is the next product's operand as it lies in the registers; else k 8 g .. 8 g + 7 ----
template <typename T, int NP> struct Operand;
template <int NP> struct Operand<__bf16, NP> { bf16x8 p[NP]; };
template <int NP> struct Operand<float, NP> { f32x4 lo, hi; };

// acc += A B over one step: the pairs of pieces of order below kPieces, the smallest first
template <int NA, int NB>
__device__ __forceinline__ f32x4 mma(const Operand<__bf16, NA>& a, const Operand<__bf16, NB>& b, f32x4 acc) {
#pragma unroll
  for (int s = kPieces - 1; s >= 0; --s)
#pragma unroll
    for (int i = 0; i <= s; ++i)
      if (i < NA && s - i < NB) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i < NA ? i : 0], b.p[s - i < NB ? s - i : 0], acc, 0, 0, 0);
  return acc;
}
template <int NA, int NB>
__device__ __forceinline__ f32x4 mma(const Operand<float, NA>& a, const Operand<float, NB>& b, f32x4 acc) {
#pragma unroll
  for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.lo[e], b.lo[e], acc, 0, 0, 0);
#pragma unroll
  for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.hi[e], b.hi[e], acc, 0, 0, 0);
  return acc;
}

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Float32 values as NP bf16 pieces, each the rounding of what the ones before it leave; the difference (exact) takes one
// instruction, the piece times -1 added.
template <int NP, int N> __device__ __forceinline__ void split(float (&x)[N], __bf16 (&out)[NP][N]) {
  // -1 in the low and in the high half, in registers: as a literal the second is float32's inline constant -1, which
  // the instruction takes for a low half
  unsigned low = 0xbf80u, high = 0xbf800000u;
  asm("" : "+s"(low), "+s"(high));
  const bf16x2 first = __builtin_bit_cast(bf16x2, low), second = __builtin_bit_cast(bf16x2, high);
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const bf16x2 y = {(__bf16)x[e], (__bf16)x[e + 1]};
      out[p][e] = y[0];
      out[p][e + 1] = y[1];
      if (p + 1 < NP) {
        x[e] = __builtin_amdgcn_fdot2_f32_bf16(y, first, x[e], false);
        x[e + 1] = __builtin_amdgcn_fdot2_f32_bf16(y, second, x[e + 1], false);
      }
    }
}
template <int NP> __device__ __forceinline__ void split4(f32x4 v, bf16x4 (&out)[NP]) {
  float x[4] = {v[0], v[1], v[2], v[3]};
  __bf16 y[NP][4];
  split<NP, 4>(x, y);
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int e = 0; e < 4; ++e) out[p][e] = y[p][e];
}

// A pair of accumulator tiles as the operand whose k run down their rows.
template <typename T, int NP>
__device__ __forceinline__ Operand<T, NP> paired(f32x4 a, f32x4 b) {
  Operand<T, NP> o;
  if constexpr (sizeof(T) == 2) {
    float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    __bf16 y[NP][8];
    split<NP, 8>(x, y);
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int e = 0; e < 8; ++e) o.p[p][e] = y[p][e];
  } else {
    o.lo = a;
    o.hi = b;
  }
  return o;
}

// A sum of log decays (in float64) times log2 e as two float32 numbers, and e to the difference of two sums: the first
// parts' difference is rounded by half a step of itself, as a float32 exponent has to be.
struct DecaySum { float hi, lo; };
__device__ __forceinline__ DecaySum decay_sum(double sum) {
  const double x = sum * 1.4426950408889634074;
  const float hi = (float)x;
  return {hi, (float)(x - (double)hi)};
}
__device__ __forceinline__ float decay(DecaySum a, DecaySum b) { return __builtin_amdgcn_exp2f((a.hi - b.hi) + (a.lo - b.lo)); }

__device__ __forceinline__ int lane_col() { return threadIdx.x & 15; }
__device__ __forceinline__ int lane_grp() { return (threadIdx.x & 63) >> 4; }

// ---- one head's rows of a chunk in [B, N, H, D], through a buffer resource: rows past the sequence and features past D
// read zeros and drop writes, so that no load is followed by a select (which would wait for it) and none is conditional
// (a wait for an older load could not count the newer ones) ----
constexpr unsigned kNowhere = 0x7ffffff0u;  // an offset past every range

template <typename T> struct Rows {
  __amdgpu_buffer_rsrc_t r;
  unsigned pitch;  // bytes of a token's H heads
  int D;
  __device__ __forceinline__ unsigned at(int row, int f) const {
    return f < D ? (unsigned)row * pitch + (unsigned)f * (unsigned)sizeof(T) : kNowhere;
  }
  // eight elements of a row, from feature f (a multiple of 8)
  __device__ __forceinline__ Operand<T, 1> row(int row, int f) const {
    const unsigned o = at(row, f);
    Operand<T, 1> x;
    if constexpr (sizeof(T) == 2) {
      x.p[0] = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(r, o, 0, 0));
    } else {
      x.lo = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, o, 0, 0));
      x.hi = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, o + 16, 0, 0));
    }
    return x;
  }
  __device__ __forceinline__ T one(int row, int f) const {
    if constexpr (sizeof(T) == 2) {
      return __builtin_bit_cast(T, (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, at(row, f), 0, 0));
    } else {
      return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, at(row, f), 0, 0));
    }
  }
  // eight elements from feature f (a multiple of 8)
  __device__ __forceinline__ void put_eight(int row, int f, const float (&x)[8]) const {
    const unsigned o = at(row, f);
    if constexpr (sizeof(T) == 2) {
      bf16x8 y;
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = (__bf16)x[i];
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, y), r, o, 0, 0);
    } else {
      const f32x4 lo = {x[0], x[1], x[2], x[3]}, hi = {x[4], x[5], x[6], x[7]};
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, lo), r, o, 0, 0);
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, hi), r, o + 16, 0, 0);
    }
  }
  // four elements from feature f (a multiple of 4)
  __device__ __forceinline__ void put_four(int row, int f, f32x4 x) const {
    if constexpr (sizeof(T) == 2) {
      bf16x4 y;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = (__bf16)x[i];
      __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2_t, y), r, at(row, f), 0, 0);
    } else {
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, x), r, at(row, f), 0, 0);
    }
  }
};

// ---- a chunk's rows in LDS as they come from memory, 16-byte pieces straight into LDS (no registers, no padding): a
// row's pieces are permuted by bits of its number, so that the reads of a step of 16 rows (row operands) and the transposed
// reads of 8 rows at a time (column operands) spread over the 64 banks ----
template <typename T, int W> struct Tile {  // 64 rows of W elements
  static constexpr int kPer = 16 / (int)sizeof(T);  // elements a piece
  static constexpr int kRow = W / kPer;             // pieces a row: a power of two from 2 on
  static constexpr int kElems = kChunk * W;
  static constexpr int kInstr = kRow;               // wave instructions a tile: 64 pieces each
  __device__ __forceinline__ static int permute(int row) {
    if constexpr (kRow >= 16) return ((row >> 3) & 1) | ((row & 7) << 1);
    else if constexpr (kRow == 8) return ((row >> 3) & 1) | (((row >> 1) & 3) << 1);
    else if constexpr (kRow == 4) return ((row >> 3) & 1) | (((row >> 2) & 1) << 1);
    else return 0;
  }
  __device__ __forceinline__ static int at(int row, int f) {
    return row * W + (((f / kPer) ^ permute(row)) * kPer) + (f & (kPer - 1));
  }
  // instruction j of the tile: lane l brings piece 64 j + l of the rows' features from `first` on
  __device__ __forceinline__ static void stage(T* tile, const Rows<T>& rows, int j, int first) {
    const int l = threadIdx.x & 63, p = 64 * j + l, row = p / kRow;
    buffer_load_lds16(rows.r, tile + 64 * kPer * j, rows.at(row, first + ((p & (kRow - 1)) ^ permute(row)) * kPer), 0);
  }
  // eight elements of a row from feature f (a multiple of 8)
  __device__ __forceinline__ static Operand<T, 1> row(const T* tile, int row, int f) {
    Operand<T, 1> x;
    if constexpr (sizeof(T) == 2) {
      x.p[0] = *reinterpret_cast<const bf16x8*>(tile + at(row, f));
    } else {
      x.lo = *reinterpret_cast<const f32x4*>(tile + at(row, f));
      x.hi = *reinterpret_cast<const f32x4*>(tile + at(row, f + 4));
    }
    return x;
  }
  // rows 16 i + 4 g .. + 3 of column f0 + c: an accumulator tile's layout
  __device__ __forceinline__ static f32x4 four(const T* tile, int i, int f0) {
    const int c = lane_col(), r0 = 16 * i + 4 * lane_grp();
    f32x4 x;
    if constexpr (sizeof(T) == 2) {
      const bf16x4 y = read_tr16<bf16x4>(tile + at(r0 + (c >> 2), f0 + 4 * (c & 3)));
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = (float)y[r];
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = tile[at(r0 + r, f0 + c)];
    }
    return x;
  }
  // column f0 + c of the rows of step s, in the order of a pair of accumulator tiles
  __device__ __forceinline__ static Operand<T, 1> columns(const T* tile, int s, int f0) {
    const int c = lane_col(), r0 = 32 * s + 4 * lane_grp();
    Operand<T, 1> x;
    if constexpr (sizeof(T) == 2) {
      const bf16x4 lo = read_tr16<bf16x4>(tile + at(r0 + (c >> 2), f0 + 4 * (c & 3)));
      const bf16x4 hi = read_tr16<bf16x4>(tile + at(r0 + 16 + (c >> 2), f0 + 4 * (c & 3)));
      x.p[0] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x.lo[e] = tile[at(r0 + e, f0 + c)];
        x.hi[e] = tile[at(r0 + 16 + e, f0 + c)];
      }
    }
    return x;
  }
};

// All but the last LEFT of this wave's loads and stores are done: direct loads among them are in LDS.
template <int LEFT = 0> __device__ __forceinline__ void direct_loads_done() {
  static_assert(LEFT < 64);
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0x0F70 | (LEFT & 15) | (LEFT >> 4) << 14);  // vmcnt
  __builtin_amdgcn_sched_barrier(0);
}

// Column f0 + c of rows 32 s + 8 g .. + 7 of a row-major LDS tile [token][feature].
template <typename T>
__device__ __forceinline__ Operand<T, 1> load_columns(const T* tile, int pitch, int s, int f0) {
  const int c = lane_col(), g = lane_grp();
  Operand<T, 1> o;
  if constexpr (sizeof(T) == 2) {
    const T* p = tile + (32 * s + 8 * g + (c >> 2)) * pitch + f0 + 4 * (c & 3);
    const bf16x4 a = read_tr16<bf16x4>(p), b = read_tr16<bf16x4>(p + 4 * pitch);
    o.p[0] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
    const T* p = tile + (32 * s + 8 * g) * pitch + f0 + c;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o.lo[e] = p[e * pitch];
      o.hi[e] = p[(4 + e) * pitch];
    }
  }
  return o;
}

// ---- operands in LDS or in the workspace: a step's pieces one after the other, a piece 16 bytes a lane (float32: the eight values in
// two planes of four) ----
template <typename T, int NP> struct Frags {
  static constexpr int kStep = sizeof(T) == 2 ? NP * 512 : 512;  // elements of a step
  template <int N> __device__ __forceinline__ static void put(T* base, int s, const Operand<T, N>& o) {
    const int l = threadIdx.x & 63;
    T* step = base + s * kStep;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int p = 0; p < NP; ++p) *reinterpret_cast<bf16x8*>(step + (p * 64 + l) * 8) = o.p[p];
    } else {
      *reinterpret_cast<f32x4*>(step + l * 4) = o.lo;
      *reinterpret_cast<f32x4*>(step + (64 + l) * 4) = o.hi;
    }
  }
  // An accumulator tile as half of step t / 2: in the order of pairs of tiles, or (NATURAL) with k 8 g .. 8 g + 7 a lane.
  template <bool NATURAL> __device__ __forceinline__ static void put_tile(T* base, int t, f32x4 acc) {
    const int c = lane_col(), g = lane_grp();
    const int lane = NATURAL ? (2 * (t & 1) + (g >> 1)) * 16 + c : 16 * g + c, half = NATURAL ? g & 1 : t & 1;
    T* step = base + (t >> 1) * kStep;
    if constexpr (sizeof(T) == 2) {
      bf16x4 x[NP];
      split4<NP>(acc, x);
#pragma unroll
      for (int p = 0; p < NP; ++p) *reinterpret_cast<bf16x4*>(step + (p * 64 + lane) * 8 + 4 * half) = x[p];
    } else {
      *reinterpret_cast<f32x4*>(step + (half * 64 + lane) * 4) = acc;
    }
  }
  // the first N pieces of a step
  template <int N = NP> __device__ __forceinline__ static Operand<T, N> get(const T* base, int s) {
    const int l = threadIdx.x & 63;
    const T* step = base + s * kStep;
    Operand<T, N> o;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int p = 0; p < N; ++p) o.p[p] = *reinterpret_cast<const bf16x8*>(step + (p * 64 + l) * 8);
    } else {
      o.lo = *reinterpret_cast<const f32x4*>(step + l * 4);
      o.hi = *reinterpret_cast<const f32x4*>(step + (64 + l) * 4);
    }
    return o;
  }
};

// The six operand steps that cover a lower triangle of 4 x 4 tiles. By rows i (the sums run over j <= i): steps
// 0 .. i / 2; by columns j (over i >= j): steps j / 2 .. 1. The tiles of a step outside the triangle are zeros.
constexpr int kTriSteps = 6;
__host__ __device__ constexpr int row_step(int i, int s) { return i < 2 ? i : 2 * i - 2 + s; }
__host__ __device__ constexpr int col_step(int j, int s) { return j < 2 ? 2 * j + s : j + 2; }

// ---- the workspace of one chunk and head ----
// coefficients: beta, eps, kap, 64 floats each, and behind these both parts of the sums of the decays; of the first three
// in LDS a direct load's 1 KiB (zeros behind them)
constexpr int kCoef = 3 * kChunk, kCoefLds = 256, kCoefAll = 5 * kChunk;
__device__ __forceinline__ void stage_coef(float* dst, const float* coef) {
  buffer_load_lds16(buffer_rsrc(coef, kCoef * sizeof(float)), dst, 16 * (threadIdx.x & 63), 0);
}
template <typename T, int NP> struct Factor {  // elements of a triangular factor
  static constexpr int kElems = kTriSteps * Frags<T, NP>::kStep;
};
template <typename T> struct Pieces { static constexpr int kN = kPieces; };
template <> struct Pieces<float> { static constexpr int kN = 1; };
// Pieces of H, R and W in the outputs' products. The outputs are 1.7e-3 of their norm from float64's, which is their rounding
// to bf16 alone, with two as with three. With two, single values next to a border between two bf16 numbers fall on its other
// side than a float32 computation's: 1.1e-4 of the norm in all, 3e-5 with three, which took 112 us for 94 in the chain of
// B8 T4096 H8 d64 and 51 for 47 in its prep. With one, heads of width 16 were 2.8e-3 off.
template <typename T> struct OutPieces { static constexpr int kN = 2; };
template <> struct OutPieces<float> { static constexpr int kN = 1; };

// A chunk's record of accumulator tiles, 1 KiB each as they lie in a wave's registers: a store of a wave is contiguous (by
// columns of the matrix, 64 bytes at a time, the stores took as long as all else in the chain).
struct Record {
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ void put(int tile, f32x4 x) const {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, x), r, (64 * tile + (threadIdx.x & 63)) * 16, 0, 0);
  }
};
__device__ __forceinline__ Record record(float* base, size_t chunk, int tiles) {
  return {buffer_rsrc(base + chunk * tiles * 256, (unsigned)tiles * 1024u)};
}

// LDS writes before, LDS reads after, for the whole workgroup; loads from memory stay in flight, direct loads into LDS
// among them (a release fence would wait for those: direct_loads_done does, where they are due).
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <typename T>
struct Dims {
  int N, H, D, chunks;
  // element offset of token t of head h in [B, N, H, D]
  __device__ __forceinline__ size_t at(int b, int t, int h) const { return (((size_t)b * N + t) * H + h) * D; }
  // a head's rows of chunk ci, the first of them at `first`, to the end of the chunk or of the sequence
  __device__ __forceinline__ Rows<T> rows_at(const T* first, int ci) const {
    const int left = N - ci * kChunk, count = left < kChunk ? left : kChunk;
    const unsigned pitch = (unsigned)H * D * sizeof(T);
    return {buffer_rsrc(first, (count - 1) * pitch + (unsigned)(D * sizeof(T))), pitch, D};
  }
  // the rows of head h from token t0, a chunk's first
  __device__ __forceinline__ Rows<T> rows(const T* p, int b, int t0, int h) const { return rows_at(p + at(b, t0, h), t0 / kChunk); }
  // the bytes of a chunk's flags; without flags an empty range
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t flags(const uint8_t* p, int b, int t0) const {
    const int count = N - t0 < kChunk ? N - t0 : kChunk;
    return buffer_rsrc(p == nullptr ? p : p + (size_t)b * N + t0, p == nullptr ? 0u : (unsigned)count);
  }
};

// ---- launchers shared between the translation units ----
// The chunks' coefficients and the factors T and P, by rows (the forward's) or by columns (the backward's, P in
// pieces too).
template <typename T>
int launch_prep(const T* q, const T* k, const T* beta, const float* g, float* coef, T* tf, T* pf, int B, int N, int H,
                int D, bool columns, hipStream_t stream);

// `kept`: a forward that keeps records, or the backward, whose last kernel has 512 threads a chunk.
int check_sizes(int B, int N, int H, int D, bool kept, const char* who);

// the records of a forward that a backward follows, float32 accumulator tiles (rows features or tokens, columns values): of
// each chunk its starting state, tile (value tile) * tiles + (feature tile); then of each its Delta, tile (value tile) * 4 +
// (token tile)
__host__ __device__ constexpr int tiles_of(int D) { return (D + 15) / 16; }
__host__ __device__ inline size_t state_floats(size_t total, int D) { return total * tiles_of(D) * tiles_of(D) * 256; }
inline size_t record_bytes(size_t total, int D) { return (state_floats(total, D) + total * tiles_of(D) * 4 * 256) * sizeof(float); }
inline int chunks_of(int N) { return (N + kChunk - 1) / kChunk; }
inline int width_of(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 128 ? 128 : 256; }

}  // namespace gated
}  // namespace vsp
