// The gated delta rule's chunked scan on CDNA4 (gfx950); the mathematics and the operands are in gated.h.
//
//  * gated_prep_kernel: a wave a chunk and head (for few chunks gated_prep_lines_kernel: four), all of them at once:
//    the decays' sums, the products of all pairs of the chunk's tokens (K K^T and Q K^T), the inverse T and W = P T,
//    both written as MFMA operands.
//  * gated_chain_kernel: a workgroup a head and 16 value columns walks the chunks (value columns of the state evolve
//    independently, so a head of width 64 is four chains). Four waves carry the chain, each one tile of 16 tokens
//    (R, Delta) and its share of the state's feature tiles in accumulators; between the three dependent products
//    (K H, T R, K^T Delta) the tiles pass through LDS as operands in pieces. Four more waves bring keys and values
//    straight into LDS two chunks ahead and form the outputs O = eps Q H + W R in the gaps, so that the chain waits
//    for no memory.
#include "gated.h"
#include "vesper_kernels.h"

namespace vsp {
namespace gated {
namespace {

// --------------------------------------------------------------------------------------------
// prep
// --------------------------------------------------------------------------------------------
constexpr int kPad = 20;                   // pitch of a 16 x 16 float32 tile in LDS
constexpr int kTile = 16 * kPad + 4;       // tiles start on other banks
constexpr int kPrepWaves = 4;
// Up to so many chunks prep by lines: a workgroup a CU, in float32, whose products are longer, two.
template <typename T> constexpr int kLineChunks = sizeof(T) == 2 ? 256 : 512;

struct PrepLds {
  float hi[kChunk], lo[kChunk];  // both parts of the decays' sums
  float beta[kChunk];            // -beta
  float a[4 * kTile];            // diagonal tiles of -A, column by column
  float x[4 * kTile];            // their inverses (I + A_bb)^-1, row by row
};

__device__ __forceinline__ void wave_lds_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// x moved along the lanes by the pattern CTRL, in the rows of 16 lanes of ROWS; zero where nothing moves in.
template <int CTRL, int ROWS> __device__ __forceinline__ double moved(double x) {
  const u32x2_t y = __builtin_bit_cast(u32x2_t, x);
  const u32x2_t z = {(unsigned)__builtin_amdgcn_update_dpp(0, (int)y[0], CTRL, ROWS, 0xf, false),
                     (unsigned)__builtin_amdgcn_update_dpp(0, (int)y[1], CTRL, ROWS, 0xf, false)};
  return __builtin_bit_cast(double, z);
}
// Sums of x over the lanes up to each one, moved in registers: through shuffles, by LDS, they
// took 4000 cycles longer.
__device__ __forceinline__ double sums_up_to(double x) {
  x += moved<0x111, 0xf>(x);  // one, two, four and eight lanes up within 16
  x += moved<0x112, 0xf>(x);
  x += moved<0x114, 0xf>(x);
  x += moved<0x118, 0xf>(x);
  x += moved<0x142, 0xa>(x);  // lane 15 of 16 to the next 16, in the odd ones
  x += moved<0x143, 0xc>(x);  // lane 31 to the upper half
  return x;
}

// C[16 x 16] += A B in float32: lane (c, g) holds A[c][4 g + r] and B[4 g + r][c], an accumulator's own layout.
__device__ __forceinline__ f32x4 mm16f(f32x4 a, f32x4 b, f32x4 acc) {
#pragma unroll
  for (int r = 0; r < 4; ++r) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], b[r], acc, 0, 0, 0);
  return acc;
}

// Row (COLS: column) a of a lower triangle of accumulator tiles, tile o at x[o], as its operands of gated.h's six steps;
// tiles outside the triangle are zeros.
template <typename T, int NP, bool COLS>
__device__ __forceinline__ void put_line(T* out, int a, const f32x4 (&x)[4]) {
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    if (COLS ? 2 * s + 1 < a : 2 * s > a) continue;
    const bool first = !COLS || 2 * s >= a, second = COLS || 2 * s + 1 <= a;
    Frags<T, NP>::put(out, COLS ? col_step(a, s - a / 2) : row_step(a, s),
                      paired<T, NP>(first ? x[2 * s] : zero4(), second ? x[2 * s + 1] : zero4()));
  }
}

// Bound by its own arithmetic and its latency, not by memory: of a wave's 20 to 27 thousand cycles alone on its SIMD the 80
// decays a lane take 2500, the substitution 2700, the 144 float32 MFMAs of T and W and their splitting 7000, the loads and
// the decays' sums 5000, and three waves a SIMD share them. B8 T4096 H8 d64 (160 MB in and out) 47 us, B1 T8191 H12 18, 64
// chunks of float32 13 (by lines, below, 8; but 51 and 21 for the large ones: each wave inverts a diagonal tile, where one
// wave has all four in its 64 lanes). Tried: four waves a SIMD (61: the registers spill).
// COLS, for the backward pass: the factors T and P by columns, with accumulator rows i and columns j. Else T and
// W = P T by rows, transposed: rows j, columns i. With X the diagonal tiles' inverses (I + A_bb)^-1, tile by tile:
//   T_ij = -X_i sum_k A_ik T_kj (k = j .. i - 1), or transposed T_ij^T = -X_j^T sum_k A_kj^T T_ik^T (k = j + 1 .. i);
//   W_ij^T = X_j^T (P_ij^T - sum_k A_kj^T W_ik^T) (k = j + 1 .. i), from W (I + A) = P.
// In either form the tile A that multiplies is an accumulator tile of the other form's layout, and what it multiplies is
// one of its own: no tile leaves registers, and a line of T or W is written when it is done.
template <typename T, int DP, bool COLS>
__global__ __launch_bounds__(64 * kPrepWaves, 2) void gated_prep_kernel(
    const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ beta, const float* __restrict__ g,
    float* __restrict__ coef, T* __restrict__ tf, T* __restrict__ pf, Dims<T> dims, int total) {
  __shared__ PrepLds lds[kPrepWaves];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63, c = l & 15, grp = l >> 4;
  const int id = blockIdx.x * kPrepWaves + wave;
  if (id >= total) return;  // whole waves; no workgroup barrier below
  PrepLds& s = lds[wave];
  const int chunk = id % dims.chunks, bh = id / dims.chunks, h = bh % dims.H, b = bh / dims.H;
  const int t0 = chunk * kChunk;
  constexpr int KS = DP / 32;
  constexpr int NT = Pieces<T>::kN, NPP = COLS ? NT : OutPieces<T>::kN;

  // the decays and the first rows are loaded together
  const bool ok = t0 + l < dims.N;
  const size_t at = ((size_t)b * dims.N + (ok ? t0 + l : t0)) * dims.H + h;
  const float gl = g[at], bl = to_f32(beta[at]);
  const Rows<T> krows = dims.rows(k, b, t0, h), qrows = dims.rows(q, b, t0, h);
  struct In {
    Operand<T, 1> k[4], q[4];
  };
  auto load = [&](int st, In& in) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      in.k[i] = krows.row(16 * i + c, 32 * st + 8 * grp);
      in.q[i] = qrows.row(16 * i + c, 32 * st + 8 * grp);
    }
  };
  In in[2];
  load(0, in[0]);
  // lane l is token t0 + l; tokens behind the last decay nothing and write nothing
  {
    const double sum = sums_up_to(ok ? ((double)gl < kLeastDecay ? kLeastDecay : (double)gl) : 0.0);
    const u32x2_t bits = __builtin_bit_cast(u32x2_t, sum);
    const u32x2_t last = {(unsigned)__builtin_amdgcn_readlane((int)bits[0], 63), (unsigned)__builtin_amdgcn_readlane((int)bits[1], 63)};
    const double all = __builtin_bit_cast(double, last);
    const float be = ok ? bl : 0.f;
    const DecaySum parts = decay_sum(sum);
    s.hi[l] = parts.hi;
    s.lo[l] = parts.lo;
    s.beta[l] = -be;
    float* co = coef + (size_t)id * kCoefAll;
    co[l] = be;
    co[kChunk + l] = expf((float)sum);
    co[2 * kChunk + l] = expf((float)(all - sum));
    co[kCoef + l] = parts.hi;
    co[kCoef + kChunk + l] = parts.lo;
  }

  // K K^T and Q K^T of the lower tiles, in both accumulator layouts where both are needed: `mult` multiplies (for
  // COLS rows j, columns i; else rows i, columns j), the diagonal tiles serve both.
  f32x4 mult[10], pp[10];
#pragma unroll
  for (int t = 0; t < 10; ++t) mult[t] = pp[t] = zero4();
#pragma unroll
  for (int st = 0; st < KS; ++st) {
    if (st + 1 < KS) load(st + 1, in[(st + 1) & 1]);
    const In& now = in[st & 1];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j <= i; ++j) {
        const int t = i * (i + 1) / 2 + j;
        mult[t] = COLS ? mma(now.k[j], now.k[i], mult[t]) : mma(now.k[i], now.k[j], mult[t]);
        pp[t] = COLS ? mma(now.q[i], now.k[j], pp[t]) : mma(now.k[j], now.q[i], pp[t]);
      }
  }
  wave_lds_sync();

  // the decays between pairs, -beta and the triangles; the sums are read at once, not each before its use
  T* tout = tf + (size_t)id * Factor<T, NT>::kElems;
  T* pout = pf + (size_t)id * Factor<T, NPP>::kElems;
  f32x4 hi_row[4], lo_row[4], beta_row[4];  // of tokens 16 i + 4 g + r
  DecaySum col[4];                          // of tokens 16 i + c
  float beta_col[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    hi_row[i] = *reinterpret_cast<const f32x4*>(s.hi + 16 * i + 4 * grp);
    lo_row[i] = *reinterpret_cast<const f32x4*>(s.lo + 16 * i + 4 * grp);
    beta_row[i] = *reinterpret_cast<const f32x4*>(s.beta + 16 * i + 4 * grp);
    col[i] = {s.hi[16 * i + c], s.lo[16 * i + c]};
    beta_col[i] = s.beta[16 * i + c];
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j <= i; ++j) {
      const int t = i * (i + 1) / 2 + j;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 4 * grp + r;
        const DecaySum row_i = {hi_row[i][r], lo_row[i][r]}, row_j = {hi_row[j][r], lo_row[j][r]};
        // of mult: i by rows, j by columns (COLS: the other way round); of Q K^T: i by columns, j by rows (COLS: the other way)
        const float em = (COLS ? beta_col[i] : beta_row[i][r]) * (COLS ? decay(col[i], row_j) : decay(row_i, col[j]));
        mult[t][r] *= i > j || (COLS ? row < c : c < row) ? em : 0.f;
        const float ep = COLS ? decay(row_i, col[j]) : decay(col[i], row_j);
        pp[t][r] *= i > j || (COLS ? c <= row : row <= c) ? ep : 0.f;
      }
      if (i == j) {  // -A[ii][jj] of the diagonal tile at jj * kPad + ii
        if constexpr (COLS) {
#pragma unroll
          for (int r = 0; r < 4; ++r) s.a[i * kTile + (4 * grp + r) * kPad + c] = mult[t][r];
        } else {
          *reinterpret_cast<f32x4*>(s.a + i * kTile + c * kPad + 4 * grp) = mult[t];
        }
      }
    }
  wave_lds_sync();

  // X = (I + A_bb)^-1 by forward substitution: lane l solves column l % 16 of block l / 16, column by column of A
  {
    float x[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = r == c ? 1.f : 0.f;
    const float* a = s.a + grp * kTile;
#pragma unroll
    for (int kk = 0; kk < 15; ++kk)
#pragma unroll
      for (int f = (kk + 1) / 4; f < 4; ++f) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(a + kk * kPad + 4 * f);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (4 * f + r > kk) x[4 * f + r] = __builtin_fmaf(y[r], x[kk], x[4 * f + r]);
      }
#pragma unroll
    for (int r = 0; r < 16; ++r) s.x[grp * kTile + r * kPad + c] = x[r];
  }
  wave_lds_sync();

  // the diagonal inverses in this form's accumulator layout and as multipliers, then line by line
  f32x4 xt[4], xm[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float* x = s.x + i * kTile;
    const f32x4 along = *reinterpret_cast<const f32x4*>(x + c * kPad + 4 * grp);  // X[c][4 g + r]
    f32x4 down;                                                                   // X[4 g + r][c]
#pragma unroll
    for (int r = 0; r < 4; ++r) down[r] = x[(4 * grp + r) * kPad + c];
    xt[i] = COLS ? down : along;
    xm[i] = COLS ? along : down;
  }
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    f32x4 t[4], w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = w[i] = zero4();
    t[a] = xt[a];
    if constexpr (COLS) {
#pragma unroll
      for (int i = a; i < 4; ++i) {
        w[i] = pp[i * (i + 1) / 2 + a];
        if (i == a) continue;
        f32x4 m = zero4();
#pragma unroll
        for (int kk = a; kk < i; ++kk) m = mm16f(mult[i * (i + 1) / 2 + kk], t[kk], m);
        t[i] = mm16f(xm[i], m, zero4());
      }
    } else {
#pragma unroll
      for (int j = a; j >= 0; --j) {
        f32x4 m = zero4(), n = pp[a * (a + 1) / 2 + j];
#pragma unroll
        for (int kk = j + 1; kk <= a; ++kk) {
          m = mm16f(mult[kk * (kk + 1) / 2 + j], t[kk], m);
          n = mm16f(mult[kk * (kk + 1) / 2 + j], w[kk], n);
        }
        if (j < a) t[j] = mm16f(xm[j], m, zero4());
        w[j] = mm16f(xm[j], n, zero4());
      }
    }
    put_line<T, NT, COLS>(tout, a, t);
    put_line<T, NPP, COLS>(pout, a, w);
  }
}

struct LinesLds {
  float hi[kChunk], lo[kChunk];  // both parts of the decays' sums
  float beta[kChunk];            // -beta
  f32x4 mult[6][64];    // -A's tiles below the diagonal, (i, j) at i (i - 1) / 2 + j, as they lie in registers
  float a[4 * kTile];   // the diagonal ones, column by column
  float x[4 * kTile];   // their inverses (I + A_bb)^-1, row by row
};

// The same by a workgroup of four waves a chunk and head, for few chunks: a wave has a line (row or column a), its tiles of
// K K^T and Q K^T, its diagonal tile's inverse and its tiles of T and W; the tiles of A and the inverses pass by LDS. Its
// results are the other's bit for bit. Calls of the scan with one and the other for 64, 128, 256, 512 and 1024 chunks of one a
// row, in us: float32 14 and 19, 17 and 21, 24 and 30, 38 and 42, 70 and 66; bf16 12 and 14, 14 and 17, 20 and 23, 32.5 and
// 32.6, 52 and 49.
template <typename T, int DP, bool COLS>
__global__ __launch_bounds__(256) void gated_prep_lines_kernel(
    const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ beta, const float* __restrict__ g,
    float* __restrict__ coef, T* __restrict__ tf, T* __restrict__ pf, Dims<T> dims) {
  __shared__ __attribute__((aligned(16))) LinesLds s;
  const int id = blockIdx.x, l = threadIdx.x & 63, c = l & 15, grp = l >> 4;
  // the lines are of different lengths: the waves of a SIMD shall not all have the same one
  const int a = __builtin_amdgcn_readfirstlane(((threadIdx.x >> 6) + id) & 3);
  const int chunk = id % dims.chunks, bh = id / dims.chunks, h = bh % dims.H, b = bh / dims.H;
  const int t0 = chunk * kChunk;
  constexpr int KS = DP / 32;
  constexpr int NT = Pieces<T>::kN, NPP = COLS ? NT : OutPieces<T>::kN;

  // the line's tiles (tile o of the other index): of K K^T as what multiplies (COLS: rows j, columns i; else rows i,
  // columns j), of Q K^T as what is multiplied; tiles outside the triangle: the diagonal one's rows again, not used
  f32x4 mult[4], pp[4];
#pragma unroll
  for (int o = 0; o < 4; ++o) mult[o] = pp[o] = zero4();
  const Rows<T> krows = dims.rows(k, b, t0, h), qrows = dims.rows(q, b, t0, h);
  struct In {
    Operand<T, 1> ka, qa, kf[4], qf[COLS ? 4 : 1];
  };
  auto load = [&](int st, In& in) {
    const int f = 32 * st + 8 * grp;
    in.ka = krows.row(16 * a + c, f);
    if constexpr (!COLS) in.qa = qrows.row(16 * a + c, f);
#pragma unroll
    for (int o = 0; o < 4; ++o) {
      const int row = 16 * (COLS ? (o < a ? a : o) : (o < a ? o : a)) + c;
      in.kf[o] = krows.row(row, f);
      if constexpr (COLS) in.qf[o] = qrows.row(row, f);
    }
  };
  auto multiply = [&](const In& in) {
#pragma unroll
    for (int o = 0; o < 4; ++o)
      if (COLS ? o >= a : o <= a) {
        mult[o] = mma(in.ka, in.kf[o], mult[o]);
        pp[o] = COLS ? mma(in.qf[COLS ? o : 0], in.ka, pp[o]) : mma(in.kf[o], in.qa, pp[o]);
      }
  };
  // the decays, by the wave with the shortest line: lane l is token t0 + l; tokens behind the last decay nothing and write
  // nothing
  const bool sums = a == (COLS ? 3 : 0), ok = t0 + l < dims.N;
  float gl = 0.f, bl = 0.f;
  if (sums) {
    const size_t at = ((size_t)b * dims.N + (ok ? t0 + l : t0)) * dims.H + h;
    gl = g[at];
    bl = to_f32(beta[at]);
  }
  constexpr int AHEAD = KS < 2 || sizeof(T) == 4 ? 1 : 2;  // steps whose loads are in flight while the decays are summed
  In in[AHEAD];
#pragma unroll
  for (int st = 0; st < AHEAD; ++st) load(st, in[st]);
  double sum = 0.0;
  if (sums) {
    if (!ok) bl = 0.f;
    sum = sums_up_to(ok ? ((double)gl < kLeastDecay ? kLeastDecay : (double)gl) : 0.0);
    const DecaySum parts = decay_sum(sum);
    s.hi[l] = parts.hi;
    s.lo[l] = parts.lo;
    s.beta[l] = -bl;
  }
#pragma unroll
  for (int st = 0; st < AHEAD; ++st) multiply(in[st]);
#pragma unroll
  for (int st = AHEAD; st < KS; ++st) {
    load(st, in[0]);
    multiply(in[0]);
  }
  lds_barrier();
  if (sums) {
    const double all = __shfl(sum, 63);
    const DecaySum parts = decay_sum(sum);
    float* co = coef + (size_t)id * kCoefAll;
    co[l] = bl;
    co[kChunk + l] = expf((float)sum);
    co[2 * kChunk + l] = expf((float)(all - sum));
    co[kCoef + l] = parts.hi;
    co[kCoef + kChunk + l] = parts.lo;
  }

  // the decays between pairs, -beta and the triangles; the sums are read at once, not each before its use
  const f32x4 hi_own = *reinterpret_cast<const f32x4*>(s.hi + 16 * a + 4 * grp), lo_own = *reinterpret_cast<const f32x4*>(s.lo + 16 * a + 4 * grp);
  const f32x4 beta_own = *reinterpret_cast<const f32x4*>(s.beta + 16 * a + 4 * grp);
  const DecaySum col_own = {s.hi[16 * a + c], s.lo[16 * a + c]};
  f32x4 hi_row[4], lo_row[4];
  DecaySum col[4];
  float beta_col[4];
#pragma unroll
  for (int o = 0; o < 4; ++o) {
    hi_row[o] = *reinterpret_cast<const f32x4*>(s.hi + 16 * o + 4 * grp);
    lo_row[o] = *reinterpret_cast<const f32x4*>(s.lo + 16 * o + 4 * grp);
    col[o] = {s.hi[16 * o + c], s.lo[16 * o + c]};
    beta_col[o] = s.beta[16 * o + c];
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int o = 0; o < 4; ++o)
    if (COLS ? o >= a : o <= a) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 4 * grp + r;
        const DecaySum mine = {hi_own[r], lo_own[r]}, other = {hi_row[o][r], lo_row[o][r]};
        // of mult: i the own rows (COLS: columns of tile o), j the columns of tile o (COLS: the own rows)
        const float em = (COLS ? beta_col[o] : beta_own[r]) * (COLS ? decay(col[o], mine) : decay(mine, col[o]));
        mult[o][r] *= o != a || (COLS ? row < c : c < row) ? em : 0.f;
        // of Q K^T: i the own columns (COLS: rows of tile o), j the rows of tile o (COLS: the own columns)
        const float ep = COLS ? decay(other, col_own) : decay(col_own, other);
        pp[o][r] *= o != a || (COLS ? c <= row : row <= c) ? ep : 0.f;
      }
      if (o == a) {
        if constexpr (COLS) {
#pragma unroll
          for (int r = 0; r < 4; ++r) s.a[a * kTile + (4 * grp + r) * kPad + c] = mult[o][r];
        } else {
          *reinterpret_cast<f32x4*>(s.a + a * kTile + c * kPad + 4 * grp) = mult[o];
        }
      } else {
        s.mult[COLS ? o * (o - 1) / 2 + a : a * (a - 1) / 2 + o][l] = mult[o];
      }
    }
  wave_lds_sync();

  // X = (I + A_aa)^-1 by forward substitution: each lane solves column l % 16, column by column of A
  {
    float x[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = r == c ? 1.f : 0.f;
    const float* t = s.a + a * kTile;
#pragma unroll
    for (int kk = 0; kk < 15; ++kk)
#pragma unroll
      for (int q4 = (kk + 1) / 4; q4 < 4; ++q4) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(t + kk * kPad + 4 * q4);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (4 * q4 + r > kk) x[4 * q4 + r] = __builtin_fmaf(y[r], x[kk], x[4 * q4 + r]);
      }
    if (grp == 0) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s.x[a * kTile + r * kPad + c] = x[r];
    }
  }
  lds_barrier();

  // the line, tile by tile from the diagonal on
  f32x4 t[4], w[4];
#pragma unroll
  for (int o = 0; o < 4; ++o) t[o] = w[o] = zero4();
#pragma unroll
  for (int step = 0; step < 4; ++step) {
    const int o = COLS ? step : 3 - step;
    if (COLS ? o < a : o > a) continue;
    const float* x = s.x + o * kTile;
    const f32x4 along = *reinterpret_cast<const f32x4*>(x + c * kPad + 4 * grp);  // X[c][4 g + r]
    f32x4 down;                                                                   // X[4 g + r][c]
#pragma unroll
    for (int r = 0; r < 4; ++r) down[r] = x[(4 * grp + r) * kPad + c];
    f32x4 m = zero4();
    if constexpr (COLS) w[o] = pp[o];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      if constexpr (COLS) {
        if (kk < o && kk >= a) m = mm16f(s.mult[o * (o - 1) / 2 + (kk < o ? kk : 0)][l], t[kk], m);
      } else {
        if (kk > o && kk <= a) {
          const f32x4 y = s.mult[kk * (kk - 1) / 2 + (kk > o ? o : 0)][l];
          m = mm16f(y, t[kk], m);
          pp[o] = mm16f(y, w[kk], pp[o]);
        }
      }
    }
    t[o] = o == a ? (COLS ? down : along) : mm16f(COLS ? along : down, m, zero4());
    if constexpr (!COLS) w[o] = mm16f(down, pp[o], zero4());
  }
  put_line<T, NT, COLS>(tf + (size_t)id * Factor<T, NT>::kElems, a, t);
  put_line<T, NPP, COLS>(pf + (size_t)id * Factor<T, NPP>::kElems, a, w);
}

// --------------------------------------------------------------------------------------------
// chain
// --------------------------------------------------------------------------------------------
template <typename T, int DP> struct ChainShape {
  static constexpr int KS = DP / 32;                    // operand steps over the features
  static constexpr int TILES = DP / 16;                 // feature tiles
  static constexpr int FT = TILES < 4 ? 1 : TILES / 4;  // of them a chain wave's, at most
  static constexpr int NT = Pieces<T>::kN;
  static constexpr int NO = OutPieces<T>::kN;
  using F = Frags<T, NT>;
  using FO = Frags<T, NO>;
  using Keys = Tile<T, DP>;
  using Slice = Tile<T, 16>;
  struct Stage {  // what comes from memory by LDS
    T keys[Keys::kElems];
    T values[Slice::kElems];
    float coef[kCoefLds];
  };
  // How many chunks ahead of the one in hand the loads into LDS go: a chunk is shorter than the memory's latency, so two
  // (with one, B1 T8191 H12 d64 took 10 us longer). Float32 heads of width 256 have room for the chunk in hand only, and
  // wait for each.
  static constexpr size_t kFixed = ((size_t)KS + 4) * F::kStep * sizeof(T), kLds = 160 * 1024;
  static constexpr int LEAD = kFixed + 3 * sizeof(Stage) <= kLds ? 2 : 0;
  static constexpr int RING = LEAD + 1;
  struct Lds {
    Stage ring[RING];
    T state[KS * F::kStep];
    T r[2 * F::kStep];
    T kept[2 * F::kStep];
  };
  static_assert(sizeof(Lds) <= kLds, "more than a CU's LDS");
  // direct loads of one wave for a chunk: keys, a slice of values, coefficients (bf16: two waves each)
  static constexpr int kLoads = Keys::kInstr / 4 + (sizeof(T) == 2 ? 1 : 2);
};

// What a chain wave reads of a chunk from memory: its tokens' rows of T.
template <typename T> struct ChainIn { Operand<T, Pieces<T>::kN> t[2]; };

// What an output wave reads of a chunk: its tokens' queries, its rows of W.
template <typename T, int DP> struct OutIn {
  Operand<T, 1> qf[DP / 32];
  Operand<T, OutPieces<T>::kN> wf[2];
  float eps;
  uint8_t on;
};

// A chunk is three dependent products and three barriers, about 2300 cycles: K H 800 (of it 120 the barrier), T R 850, K^T
// Delta 500, in each the reads of the operands from LDS, the MFMAs of the pieces, and the split of the result into pieces. So
// the time is the chunks' number times 0.9 us (B1 T8191 H12 d64, 48 workgroups) to 1.5 us (B8 T4096 H8 d64, 256 of them: 94 us
// for 64; the clock falls to 2.1 GHz, and one XCD is slower by a fifth). With records the writes bound it: B16 T1024 H12 d64 52 us
// without and 96 with them (290 MB, past what the 256 MB cache behind the L2s holds). What brought it there, at B1: operands
// in pieces through LDS between four waves instead of all in one wave's registers (208 us), direct loads into LDS (150), W
// for the outputs, T into registers, two chunks ahead, loads spread over the spans, reads issued together (118).
// Few long rows leave most CUs without a chain: their sequence is walked in segments. What a segment makes of its starting
// state is affine, H' = M H + U. A first launch walks all segments but the last from zero (its end is U) and, without
// values, from the identity (M), gated_join_kernel carries the state from segment to segment, and a second launch walks
// each from its start: three times the work, on all CUs. Whole and in segments, prep and all, in us (bf16): B1 T8191 H12 d64
// 137 and 87, T4096 H2 d64 68 and 42, T4096 H16 d64 75 and 65, T2048 H8 d64 43 and 40, T4096 H2 d256 157 and 142.
struct Segments {
  int count, chunks;    // segments a row and head, chunks a segment
  const float* states;  // the starting states of the second one and on, [B H][count - 1][D][D]
  float* maps;          // U and M, [B H][count - 1][2][D][D]
};
enum Walk { kOutputs, kRecords, kMaps };  // outputs; outputs and records; only the end state, into maps

template <typename T, int DP, Walk WALK>
__global__ __launch_bounds__(512) void gated_chain_kernel(
    const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, const float* __restrict__ coef,
    const T* __restrict__ tf, const T* __restrict__ pf, const float* __restrict__ s_in, T* __restrict__ o,
    float* __restrict__ s_out, const uint8_t* __restrict__ active, float* __restrict__ rec_h, float* __restrict__ rec_d,
    Dims<T> dims, int slices, Segments segs) {
  using S = ChainShape<T, DP>;
  using F = typename S::F;
  using FO = typename S::FO;
  using Keys = typename S::Keys;
  using Slice = typename S::Slice;
  constexpr int KS = S::KS, FT = S::FT, TILES = S::TILES, NT = S::NT, NO = S::NO, LEAD = S::LEAD, RING = S::RING;
  __shared__ __attribute__((aligned(16))) typename S::Lds lds;

  const int id = xcd_logical_block(blockIdx.x, gridDim.x);
  const int sl = id % slices, walks = WALK == kMaps ? 2 * (segs.count - 1) : segs.count, walk = id / slices % walks;
  const int seg = WALK == kMaps ? walk / 2 : walk, bh = id / slices / walks, h = bh % dims.H, b = bh / dims.H;
  const bool map = WALK == kMaps && walk % 2 == 1;  // M's columns
  // the walk's chunks: nc from chunk `from` on
  const int D = dims.D, from = seg * segs.chunks, nc = dims.chunks - from < segs.chunks ? dims.chunks - from : segs.chunks;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & 3;
  const int c = lane_col(), grp = lane_grp();
  const size_t chunk0 = (size_t)bh * dims.chunks + from;

  // features past D and rows past the end are not brought: zeros, and what an earlier chunk left there, times zeros
  for (int i = threadIdx.x; i < (int)(sizeof(lds.ring) / 16); i += 512) reinterpret_cast<f32x4*>(lds.ring)[i] = zero4();
  lds_barrier();

  if (wave < 4) {
    // ---- the chain: wave w has the 16 tokens w of R and Delta, and of the state's feature tiles each fourth ----
    __builtin_amdgcn_s_setprio(3);
    const int vcol = 16 * sl + c, own = 16 * w + 4 * grp;
    const T* tp = tf + chunk0 * Factor<T, NT>::kElems + row_step(w, 0) * F::kStep;
    auto load = [&](int ci, ChainIn<T>& to) {
      const T* tc = tp + (size_t)(ci < nc ? ci : nc - 1) * Factor<T, NT>::kElems;
      to.t[0] = F::get(tc, 0);
      to.t[1] = F::get(tc, w >= 2 ? 1 : 0);  // always, so that no wait for a chunk's waits for the next one's too
    };
    ChainIn<T> ta, tb;
    load(0, ta);
    f32x4 hs[FT];
    const float* sp = seg == 0 ? s_in + (size_t)bh * D * D : segs.states + ((size_t)bh * (segs.count - 1) + seg - 1) * D * D;
#pragma unroll
    for (int i = 0; i < FT; ++i) {
      const int ft = w + 4 * i;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int f = 16 * ft + 4 * grp + r;
        if constexpr (WALK == kMaps) hs[i][r] = map && f == vcol && f < D ? 1.f : 0.f;
        else hs[i][r] = f < D && vcol < D ? sp[(size_t)f * D + vcol] : 0.f;
      }
      if (ft < TILES) F::template put_tile<true>(lds.state, ft, hs[i]);
    }
    lds_barrier();
    int slot = 0;
    auto step = [&](int ci, const ChainIn<T>& tin, ChainIn<T>& next) {
      const typename S::Stage& in = lds.ring[slot];
      slot = slot + 1 < RING ? slot + 1 : 0;
      if constexpr (LEAD == 0) lds_barrier();
      // R = beta (V - eps K H)
      f32x4 x = zero4();
#pragma unroll
      for (int s0 = 0; s0 < KS; s0 += 2) {
        Operand<T, 1> kr[2];
        Operand<T, NT> st[2];
#pragma unroll
        for (int s = 0; s < 2 && s0 + s < KS; ++s) {
          kr[s] = Keys::row(in.keys, 16 * w + c, 32 * (s0 + s) + 8 * grp);
          st[s] = F::get(lds.state, s0 + s);
        }
        __builtin_amdgcn_sched_barrier(0);  // reads together, not one by one before its product
#pragma unroll
        for (int s = 0; s < 2 && s0 + s < KS; ++s) x = mma(kr[s], st[s], x);
      }
      const f32x4 beta = *reinterpret_cast<const f32x4*>(in.coef + own);
      const f32x4 eps = *reinterpret_cast<const f32x4*>(in.coef + kChunk + own);
      const f32x4 vx = map ? zero4() : Slice::four(in.values, w, 0);
      if constexpr (WALK == kRecords) {
        const Record rh = record(rec_h, chunk0 + ci, slices * slices);
#pragma unroll
        for (int i = 0; i < FT; ++i)
          if (w + 4 * i < slices) rh.put(sl * slices + w + 4 * i, hs[i]);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = beta[r] * (vx[r] - eps[r] * x[r]);
      F::template put_tile<false>(lds.r, w, x);
      lds_barrier();
      // Delta = T R; the next chunk's T and K^T on the way
      const Operand<T, NT> r0 = F::get(lds.r, 0), r1 = F::get(lds.r, 1);
      __builtin_amdgcn_sched_barrier(0);
      load(ci + 1, next);
      f32x4 dl = mma(tin.t[0], r0, zero4());
      if (w >= 2) dl = mma(tin.t[1], r1, dl);
      const f32x4 kap = *reinterpret_cast<const f32x4*>(in.coef + 2 * kChunk + own);
      const float gam = in.coef[2 * kChunk - 1];
      constexpr int AHEAD = FT < 2 ? FT : 2;  // feature tiles whose K^T waits in registers
      Operand<T, 1> kc[AHEAD][2];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
#pragma unroll
        for (int s = 0; s < 2; ++s) kc[i][s] = Keys::columns(in.keys, s, 16 * (TILES < 4 ? w & 1 : w + 4 * i));
#pragma unroll
      for (int i = 0; i < FT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) hs[i][r] *= gam;
      f32x4 kd;
#pragma unroll
      for (int r = 0; r < 4; ++r) kd[r] = kap[r] * dl[r];
      F::template put_tile<false>(lds.kept, w, kd);
      if constexpr (WALK == kRecords) record(rec_d, chunk0 + ci, 4 * slices).put(4 * sl + w, dl);
      lds_barrier();
      // H' = gam H + K^T (kap Delta)
      const Operand<T, NT> k0 = F::get(lds.kept, 0), k1 = F::get(lds.kept, 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < FT; ++i) {
        const int ft = w + 4 * i;
        if (ft < TILES) {
          if (i >= AHEAD) {
            hs[i] = mma(Keys::columns(in.keys, 0, 16 * ft), k0, hs[i]);
            hs[i] = mma(Keys::columns(in.keys, 1, 16 * ft), k1, hs[i]);
          } else {
            hs[i] = mma(kc[i < AHEAD ? i : 0][0], k0, hs[i]);
            hs[i] = mma(kc[i < AHEAD ? i : 0][1], k1, hs[i]);
          }
          F::template put_tile<true>(lds.state, ft, hs[i]);
        }
      }
      lds_barrier();
    };
    for (int ci = 0; ci < nc; ci += 2) {
      step(ci, ta, tb);
      if (ci + 1 < nc) step(ci + 1, tb, ta);
    }
    if (WALK != kMaps && seg + 1 < segs.count) return;  // the next segment's start is there already
    float* so = WALK == kMaps ? segs.maps + (((size_t)bh * (segs.count - 1) + seg) * 2 + map) * D * D : s_out + (size_t)bh * D * D;
#pragma unroll
    for (int i = 0; i < FT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int f = 16 * (w + 4 * i) + 4 * grp + r;
        if (f < D && vcol < D) so[(size_t)f * D + vcol] = hs[i][r];
      }
  } else {
    // ---- memory into LDS ahead, and the outputs: O^T tile of the 16 tokens w (rows values, columns tokens). In a chunk's
    //      three spans: H^T Q^T and this wave's operands of the next chunk; W R, while the chain loads its T; of the chunk
    //      LEAD ahead keys, values and coefficients, and the outputs' store: the loads are spread, for a CU takes 64 bytes a
    //      cycle and who issues waits for its turn. Every wave issues kLoads direct loads a chunk, after its other loads and
    //      unconditionally, so that a wait can leave those of one chunk in flight; past the end they bring the last chunk
    //      again ----
    const size_t stride = (size_t)kChunk * dims.H * D;  // elements from a chunk's rows to the next one's
    const size_t at = dims.at(b, from * kChunk, h);
    const T *kp = k + at, *vp = v + at, *qp = q + at;
    T* op = o + at;
    const T* pp = pf + chunk0 * Factor<T, NO>::kElems + row_step(w, 0) * FO::kStep;
    const float* cp = coef + chunk0 * kCoefAll;
    auto within = [&](int ci) { return ci < nc ? ci : nc - 1; };
    auto stage = [&](int ahead, int slot) {
      const int ci = within(ahead);
      typename S::Stage& to = lds.ring[slot];
      const Rows<T> krows = dims.rows_at(kp + ci * stride, from + ci), vrows = dims.rows_at(vp + ci * stride, from + ci);
      const float* co = cp + (size_t)ci * kCoefAll;
#pragma unroll
      for (int j = 0; j < Keys::kInstr / 4; ++j) Keys::stage(to.keys, krows, 4 * j + w, 0);
      if constexpr (Slice::kInstr == 4) {
        Slice::stage(to.values, vrows, w, 16 * sl);
        stage_coef(to.coef, co);
      } else {
        if (w < 2) Slice::stage(to.values, vrows, w, 16 * sl);
        else stage_coef(to.coef, co);
      }
    };
    auto load = [&](int ahead, OutIn<T, DP>& in) {
      const int ci = within(ahead);
      const Rows<T> qrows = dims.rows_at(qp + ci * stride, from + ci);
#pragma unroll
      for (int s = 0; s < KS; ++s) in.qf[s] = qrows.row(16 * w + c, 32 * s + 8 * grp);
      const T* pb = pp + (size_t)ci * Factor<T, NO>::kElems;
      in.wf[0] = FO::get(pb, 0);
      in.wf[1] = FO::get(pb, w >= 2 ? 1 : 0);
      in.eps = cp[(size_t)ci * kCoefAll + kChunk + 16 * w + c];
      in.on = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(dims.flags(active, b, (from + ci) * kChunk), 16 * w + c, 0, 0);
    };
    int free = LEAD == 0 ? 0 : RING - 1;  // the slot of the chunk LEAD ahead
    auto step = [&](int ci, const OutIn<T, DP>& in, OutIn<T, DP>& next) {
      if constexpr (LEAD == 0) {
        stage(ci, 0);
        direct_loads_done();
        lds_barrier();
      }
      if constexpr (WALK == kMaps) {
        lds_barrier();
        lds_barrier();
        if constexpr (LEAD > 0) stage(ci + LEAD, free);
        direct_loads_done<LEAD == 0 ? 0 : S::kLoads>();
        free = free + 1 < RING ? free + 1 : 0;
        lds_barrier();
        return;
      }
      f32x4 acc = zero4();
#pragma unroll
      for (int s0 = 0; s0 < KS; s0 += 2) {
        Operand<T, NO> st[2];
#pragma unroll
        for (int s = 0; s < 2 && s0 + s < KS; ++s) st[s] = F::template get<NO>(lds.state, s0 + s);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < 2 && s0 + s < KS; ++s) acc = mma(st[s], in.qf[s0 + s], acc);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[r] *= in.eps;
      load(ci + 1, next);
      lds_barrier();
      const Operand<T, NO> r0 = F::template get<NO>(lds.r, 0), r1 = F::template get<NO>(lds.r, 1);
      __builtin_amdgcn_sched_barrier(0);
      acc = mma(r0, in.wf[0], acc);
      if (w >= 2) acc = mma(r1, in.wf[1], acc);
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[r] = active == nullptr || in.on ? acc[r] : 0.f;
      lds_barrier();
      if constexpr (LEAD > 0) stage(ci + LEAD, free);
      direct_loads_done<LEAD == 0 ? 0 : S::kLoads>();
      dims.rows_at(op + ci * stride, from + ci).put_four(16 * w + c, 16 * sl + 4 * grp, acc);
      free = free + 1 < RING ? free + 1 : 0;
      lds_barrier();
    };
    OutIn<T, DP> a, bb;
#pragma unroll
    for (int ci = 0; ci < LEAD; ++ci) stage(ci, ci);
    if constexpr (WALK != kMaps) load(0, a);
    direct_loads_done();
    lds_barrier();
    for (int ci = 0; ci < nc; ci += 2) {
      step(ci, a, bb);
      if (ci + 1 < nc) step(ci + 1, bb, a);
    }
  }
  direct_loads_done();
}

// The segments' starting states: H = M H + U, segment by segment, a workgroup a head and 16 value columns; wave w has the
// feature tiles w, w + 4, .. Serial: about 2 us a segment (the maps come from another XCD's L2).
template <typename T, int DP>
__global__ __launch_bounds__(256) void gated_join_kernel(const float* __restrict__ s_in, float* __restrict__ states, int D,
                                                         int slices, Segments segs) {
  using S = ChainShape<T, DP>;
  using F = typename S::F;
  constexpr int KS = S::KS, FT = S::FT, TILES = S::TILES, NT = S::NT;
  __shared__ __attribute__((aligned(16))) T state[KS * F::kStep];
  const int sl = blockIdx.x % slices, bh = blockIdx.x / slices, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane_col(), grp = lane_grp(), vcol = 16 * sl + c, joins = segs.count - 1;
  const size_t size = (size_t)D * D;
  auto read = [&](const float* p, int ft) {
    f32x4 x;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int f = 16 * ft + 4 * grp + r;
      x[r] = f < D && vcol < D ? p[(size_t)f * D + vcol] : 0.f;
    }
    return x;
  };
  f32x4 hs[FT];
#pragma unroll
  for (int i = 0; i < FT; ++i) hs[i] = read(s_in + bh * size, w + 4 * i);
  for (int s = 0; s < joins; ++s) {
    const float* u = segs.maps + ((size_t)bh * joins + s) * 2 * size;
    const Rows<float> m = {buffer_rsrc(u + size, (unsigned)(size * sizeof(float))), (unsigned)D * 4u, D};
#pragma unroll
    for (int i = 0; i < FT; ++i)
      if (w + 4 * i < TILES) F::template put_tile<true>(state, w + 4 * i, hs[i]);
    lds_barrier();
#pragma unroll
    for (int i = 0; i < FT; ++i) hs[i] = read(u, w + 4 * i);
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const Operand<T, NT> h = F::get(state, k);
#pragma unroll
      for (int i = 0; i < FT; ++i) {
        const Operand<float, 1> x = m.row(16 * (w + 4 * i) + c, 32 * k + 8 * grp);
        hs[i] = mma(paired<T, NT>(x.lo, x.hi), h, hs[i]);
      }
    }
    float* to = states + ((size_t)bh * joins + s) * size;
#pragma unroll
    for (int i = 0; i < FT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int f = 16 * (w + 4 * i) + 4 * grp + r;
        if (f < D && vcol < D) to[(size_t)f * D + vcol] = hs[i][r];
      }
    lds_barrier();
  }
}

// Segments a row and head: what the CUs hold at once of either launch (heads of up to 64 two workgroups a CU, wider ones
// one), 8 chunks each at least, 16 at most (joining them is serial), and no fewer than four.
int segments_of(int B, int N, int H, int D) {
  const size_t groups = (size_t)B * H * tiles_of(D);
  const int chunks = chunks_of(N);
  if (groups > 64) return 1;
  const int most = chunks / 8 < 16 ? chunks / 8 : 16, walks = (int)(256 / groups), maps = 1 + (int)((D <= 64 ? 256 : 128) / groups);
  const int fit = walks < maps ? walks : maps, count = fit < most ? fit : most;
  if (count < 4) return 1;
  const int each = (chunks + count - 1) / count;
  return (chunks + each - 1) / each;
}

template <typename T, int DP>
void launch_prep_width(const T* q, const T* k, const T* beta, const float* g, float* coef, T* tf, T* pf, Dims<T> dims,
                       int total, bool columns, hipStream_t stream) {
  if (total <= kLineChunks<T>) {
    const dim3 grid((unsigned)total), block(256);
    if (columns) hipLaunchKernelGGL((gated_prep_lines_kernel<T, DP, true>), grid, block, 0, stream, q, k, beta, g, coef, tf, pf, dims);
    else hipLaunchKernelGGL((gated_prep_lines_kernel<T, DP, false>), grid, block, 0, stream, q, k, beta, g, coef, tf, pf, dims);
    return;
  }
  const dim3 grid((unsigned)((total + kPrepWaves - 1) / kPrepWaves)), block(64 * kPrepWaves);
  if (columns) hipLaunchKernelGGL((gated_prep_kernel<T, DP, true>), grid, block, 0, stream, q, k, beta, g, coef, tf, pf, dims, total);
  else hipLaunchKernelGGL((gated_prep_kernel<T, DP, false>), grid, block, 0, stream, q, k, beta, g, coef, tf, pf, dims, total);
}

template <typename T, int DP>
void launch_chain(const T* q, const T* k, const T* v, const float* coef, const T* tf, const T* pf, const float* s_in,
                  T* o, float* s_out, const uint8_t* active, float* rec_h, float* rec_d, float* joined, Dims<T> dims, int B,
                  hipStream_t stream) {
  const int slices = tiles_of(dims.D), heads = B * dims.H, count = segments_of(B, dims.N, dims.H, dims.D);
  const dim3 grid((unsigned)(heads * slices * count)), block(512);
  const size_t floats = (size_t)heads * (count - 1) * dims.D * dims.D;
  const Segments segs{count, (dims.chunks + count - 1) / count, joined, joined + floats};
#define VSP_CHAIN(WALK, GRID)                                                                                                     \
  hipLaunchKernelGGL((gated_chain_kernel<T, DP, WALK>), GRID, block, 0, stream, q, k, v, coef, tf, pf, s_in, o, s_out, active,    \
                     rec_h, rec_d, dims, slices, segs)
  if (count > 1) {
    VSP_CHAIN(kMaps, dim3((unsigned)(heads * slices * 2 * (count - 1))));
    hipLaunchKernelGGL((gated_join_kernel<T, DP>), dim3((unsigned)(heads * slices)), dim3(256), 0, stream, s_in, joined, dims.D, slices, segs);
  }
  if (rec_h != nullptr) VSP_CHAIN(kRecords, grid);
  else VSP_CHAIN(kOutputs, grid);
#undef VSP_CHAIN
}

size_t align16(size_t x) { return (x + 15) & ~(size_t)15; }

// the forward's workspace: coefficients, T and W of every chunk and head, and the segments' states and maps
template <typename T> size_t factor_bytes(size_t total) {
  return align16(total * kCoefAll * sizeof(float)) + total * sizeof(T) * (Factor<T, Pieces<T>::kN>::kElems + Factor<T, OutPieces<T>::kN>::kElems);
}
template <typename T> size_t forward_bytes(int B, int N, int H, int D) {
  return factor_bytes<T>((size_t)B * H * chunks_of(N)) + (size_t)B * H * (segments_of(B, N, H, D) - 1) * 3 * D * D * sizeof(float);
}

template <typename T>
int scan(const void* q_, const void* k_, const void* v_, const void* beta_, const float* g, const float* s_in, void* o_,
         float* s_out, void* ws, size_t ws_bytes, float* records, size_t records_bytes, const uint8_t* active, int B,
         int N, int H, int D, hipStream_t stream, const char* who) {
  if (const int st = check_sizes(B, N, H, D, records != nullptr, who); st != OK) return st;
  if (B == 0 || N == 0) return fail(ERR_ARG, "%s: no tokens (B=%d N=%d)", who, B, N);
  const size_t total = (size_t)B * H * chunks_of(N);
  if (!q_ || !k_ || !v_ || !beta_ || !g || !s_in || !o_ || !s_out || !ws) return fail(ERR_ARG, "%s: null pointer", who);
  if ((reinterpret_cast<uintptr_t>(q_) | reinterpret_cast<uintptr_t>(k_) | reinterpret_cast<uintptr_t>(v_) |
       reinterpret_cast<uintptr_t>(o_) | reinterpret_cast<uintptr_t>(ws) | reinterpret_cast<uintptr_t>(records)) & 15)
    return fail(ERR_ARG, "%s: q, k, v, o, the workspace and the records must be 16-byte aligned", who);
  if (ws_bytes < forward_bytes<T>(B, N, H, D))
    return fail(ERR_ARG, "%s: workspace of %zu bytes, needs %zu", who, ws_bytes, forward_bytes<T>(B, N, H, D));
  if (records != nullptr && records_bytes < record_bytes(total, D))
    return fail(ERR_ARG, "%s: records of %zu bytes, need %zu", who, records_bytes, record_bytes(total, D));
  const T *q = static_cast<const T*>(q_), *k = static_cast<const T*>(k_), *v = static_cast<const T*>(v_);
  const T* beta = static_cast<const T*>(beta_);
  T* o = static_cast<T*>(o_);
  float* coef = static_cast<float*>(ws);
  T* tf = reinterpret_cast<T*>(static_cast<char*>(ws) + align16(total * kCoefAll * sizeof(float)));
  T* pf = tf + total * Factor<T, Pieces<T>::kN>::kElems;
  const Dims<T> dims{N, H, D, chunks_of(N)};
  if (const int st = launch_prep<T>(q, k, beta, g, coef, tf, pf, B, N, H, D, false, stream); st != OK) return st;
  float* joined = reinterpret_cast<float*>(static_cast<char*>(ws) + factor_bytes<T>(total));
  float* rec_d = records == nullptr ? nullptr : records + state_floats(total, D);
  switch (width_of(D)) {
    case 32: launch_chain<T, 32>(q, k, v, coef, tf, pf, s_in, o, s_out, active, records, rec_d, joined, dims, B, stream); break;
    case 64: launch_chain<T, 64>(q, k, v, coef, tf, pf, s_in, o, s_out, active, records, rec_d, joined, dims, B, stream); break;
    case 128: launch_chain<T, 128>(q, k, v, coef, tf, pf, s_in, o, s_out, active, records, rec_d, joined, dims, B, stream); break;
    default: launch_chain<T, 256>(q, k, v, coef, tf, pf, s_in, o, s_out, active, records, rec_d, joined, dims, B, stream); break;
  }
  return check_launch(who);
}

}  // namespace

template <typename T>
int launch_prep(const T* q, const T* k, const T* beta, const float* g, float* coef, T* tf, T* pf, int B, int N, int H,
                int D, bool columns, hipStream_t stream) {
  const Dims<T> dims{N, H, D, chunks_of(N)};
  const int total = B * H * dims.chunks;
  switch (width_of(D)) {
    case 32: launch_prep_width<T, 32>(q, k, beta, g, coef, tf, pf, dims, total, columns, stream); break;
    case 64: launch_prep_width<T, 64>(q, k, beta, g, coef, tf, pf, dims, total, columns, stream); break;
    case 128: launch_prep_width<T, 128>(q, k, beta, g, coef, tf, pf, dims, total, columns, stream); break;
    default: launch_prep_width<T, 256>(q, k, beta, g, coef, tf, pf, dims, total, columns, stream); break;
  }
  return check_launch("the gated scan's factors");
}
template int launch_prep<__bf16>(const __bf16*, const __bf16*, const __bf16*, const float*, float*, __bf16*, __bf16*, int, int, int, int, bool, hipStream_t);
template int launch_prep<float>(const float*, const float*, const float*, const float*, float*, float*, float*, int, int, int, int, bool, hipStream_t);

int check_sizes(int B, int N, int H, int D, bool kept, const char* who) {
  if (B < 0 || N < 0 || H < 1) return fail(ERR_ARG, "%s: bad sizes B=%d N=%d H=%d", who, B, N, H);
  if (D < 8 || D > 256 || D % 8 != 0) return fail(ERR_UNSUPPORTED, "%s: head dimension %d (multiples of 8 in 8..256)", who, D);
  if (N > (1 << 30)) return fail(ERR_UNSUPPORTED, "%s: %d tokens a row (at most 2^30)", who, N);
  // a chunk's rows are addressed by 32-bit offsets
  if ((size_t)H * D > (size_t)1 << 22) return fail(ERR_UNSUPPORTED, "%s: tokens of %d x %d features (at most 2^22)", who, H, D);
  // launches of fewer than 2^32 threads, counts in 32 bits: a wave a chunk and head, 512 threads a slice; of the backward
  // 512 a chunk and head
  if ((size_t)B * H * chunks_of(N) > (size_t)1 << 25 || (size_t)B * H * ((D + 15) / 16) > (size_t)1 << 22)
    return fail(ERR_UNSUPPORTED, "%s: B=%d N=%d H=%d (at most 2^25 chunks of 64 tokens, 2^22 slices of 16 value columns)", who, B, N, H);
  if (kept && (size_t)B * H * chunks_of(N) >= (size_t)1 << 23)
    return fail(ERR_UNSUPPORTED, "%s: B=%d N=%d H=%d (fewer than 2^23 chunks of 64 tokens with records)", who, B, N, H);
  return OK;
}

}  // namespace gated
}  // namespace vsp

extern "C" size_t vsp_gated_scan_workspace_bytes(int B, int N, int H, int D, int fp32) {
  using namespace vsp::gated;
  if (B <= 0 || N <= 0 || H <= 0 || D <= 0) return 0;
  return fp32 ? forward_bytes<float>(B, N, H, D) : forward_bytes<__bf16>(B, N, H, D);
}

extern "C" size_t vsp_gated_scan_records_bytes(int B, int N, int H, int D) {
  using namespace vsp::gated;
  if (B <= 0 || N <= 0 || H <= 0 || D <= 0) return 0;
  return record_bytes((size_t)B * H * chunks_of(N), D);
}

extern "C" int vsp_gated_scan_bf16(const void* q, const void* k, const void* v, const void* beta, const float* g,
                                   const float* state_in, void* o, float* state_out, void* workspace,
                                   size_t workspace_bytes, void* records, size_t records_bytes, const uint8_t* active,
                                   int B, int N, int H, int D, void* stream) {
  return vsp::gated::scan<__bf16>(q, k, v, beta, g, state_in, o, state_out, workspace, workspace_bytes,
                                  static_cast<float*>(records), records_bytes, active, B, N, H, D,
                                  reinterpret_cast<hipStream_t>(stream), "vsp_gated_scan_bf16");
}

extern "C" int vsp_gated_scan_f32(const void* q, const void* k, const void* v, const void* beta, const float* g,
                                  const float* state_in, void* o, float* state_out, void* workspace,
                                  size_t workspace_bytes, void* records, size_t records_bytes, const uint8_t* active,
                                  int B, int N, int H, int D, void* stream) {
  return vsp::gated::scan<float>(q, k, v, beta, g, state_in, o, state_out, workspace, workspace_bytes,
                                 static_cast<float*>(records), records_bytes, active, B, N, H, D,
                                 reinterpret_cast<hipStream_t>(stream), "vsp_gated_scan_f32");
}
