// The gated delta rule's backward pass on CDNA4 (gfx950); notation and operands as in gated.h.
//
// With dH' the gradient of a chunk's end state and dO its outputs' gradients (zero where inactive):
//   dDelta = P^T dO + kap (K dH'),  dR = T^T dDelta,  dV = beta dR,
//   dH = gam dH' + Q^T (eps dO) - K^T (beta eps dR).
// With dP_ij = E_ij dO_i.Delta_j (j <= i) and B_ij = E_ij dR_i.Delta_j (j < i):
//   dQ_i = eps_i H dO_i + sum_j dP_ij k_j,    Y_i = -(eps_i H dR_i + sum_j B_ij k_j),
//   C_j = kap_j dH' Delta_j + sum_i dP_ij q_i - sum_i beta_i B_ij k_i,
//   dK_i = beta_i Y_i + C_i,   dbeta_i = dR_i.v_i + k_i.Y_i,
//   dG_i = q_i.dQ_i + beta_i k_i.Y_i - k_i.C_i,  and for the chunk's last sum also
//   gam <dH', H> + sum_j kap_j k_j.(dH' Delta_j);   dg_t = sum of dG_i over the chunk's i >= t.
// (Every exponent is a difference of sums: its derivative adds to the later sum what it takes from the earlier one.)
//
//  * gated_prep_kernel (gated_scan.hip) forms T and P again, as operands by columns.
//  * gated_chain_backward_kernel walks the chunks from the last to the first like the forward's chain, a workgroup a
//    head and 16 value columns: four waves carry dH through three dependent products, four more form P^T dO and
//    Q^T (eps dO) of the chunk that comes next. It writes dV and keeps dH' and dR of each chunk, in float32.
//  * gated_grad_kernel: a workgroup a chunk and head, all at once, for the rest: wave w holds dQ, Y and C of the
//    16 tokens w, sums over the value columns 32 at a time from H, dH', Delta and dR in pieces in LDS, then over
//    the chunk's tokens with accumulator tiles as operands.
#include "gated.h"
#include "vesper_kernels.h"

namespace vsp {
namespace gated {
namespace {

// --------------------------------------------------------------------------------------------
// chain, backwards
// --------------------------------------------------------------------------------------------
template <typename T, int DP> struct BackShape {
  static constexpr int KS = DP / 32;
  static constexpr int TILES = DP / 16;
  static constexpr int FT = TILES < 4 ? 1 : TILES / 4;
  static constexpr int PITCH = DP + (sizeof(T) == 2 ? 8 : 4);
  static constexpr int NT = Pieces<T>::kN;
  // float32 queries are read from memory by columns: both tiles of a head of width 256 would not fit the LDS
  static constexpr bool kStageQ = sizeof(T) == 2;
  using F = Frags<T, NT>;
  using F1 = Frags<T, 1>;
  struct Lds {
    T keys[kChunk * PITCH];
    T queries[kStageQ ? kChunk * PITCH : 8];
    T state[KS * F::kStep];   // dH
    T ddelta[2 * F::kStep];
    T dread[2 * F::kStep];    // -beta eps dR
    T d_o[2 * F1::kStep];
    T edo[2 * F::kStep];      // eps dO
    float z[4 * 64 * 4];      // P^T dO, an accumulator tile after the other
    float qdo[TILES * 64 * 4];  // Q^T (eps dO)
  };
};

template <typename T, int DP> struct BackIn {  // what a chain wave reads of a chunk
  Operand<T, 1> kf[BackShape<T, DP>::KS];
  Operand<T, Pieces<T>::kN> tf[2];
  f32x4 beta, eps, kap;
  float gam;
};

template <typename T, int DP> struct BackTile {  // a quarter of a tile of keys or queries
  Operand<T, 1> x[DP / 32];
};

template <typename T, int DP> struct BackSide {  // what the other waves read of the next chunk, besides the queries
  Operand<T, Pieces<T>::kN> pf[2];
  f32x4 eps;
  T d_o[4];
  uint8_t on[4];
};

template <typename T, int DP>
__global__ __launch_bounds__(512) void gated_chain_backward_kernel(
    const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ d_o, const float* __restrict__ coef,
    const T* __restrict__ tf, const T* __restrict__ pf, const float* __restrict__ d_state, T* __restrict__ dv,
    float* __restrict__ d_state_in, const uint8_t* __restrict__ active, float* __restrict__ rec_dh,
    float* __restrict__ rec_dr, Dims<T> dims, int slices) {
  using S = BackShape<T, DP>;
  using F = typename S::F;
  using F1 = typename S::F1;
  constexpr int KS = S::KS, FT = S::FT, NT = S::NT;
  __shared__ __attribute__((aligned(16))) typename S::Lds lds;

  const int id = xcd_logical_block(blockIdx.x, gridDim.x);
  const int sl = id % slices, bh = id / slices, h = bh % dims.H, b = bh / dims.H;
  const int D = dims.D, nc = dims.chunks;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & 3;
  const int c = lane_col(), grp = lane_grp(), lane = threadIdx.x & 63;
  const int vcol = 16 * sl + c;
  const size_t chunk0 = (size_t)bh * nc;

  if (wave < 4) {
    f32x4 dh[FT];
#pragma unroll
    for (int i = 0; i < FT; ++i) {
      const int ft = w + 4 * i;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int f = 16 * ft + 4 * grp + r;
        dh[i][r] = d_state != nullptr && f < D && vcol < D ? d_state[((size_t)bh * D + f) * D + vcol] : 0.f;
      }
      if (ft < S::TILES) F::put(lds.state, ft, dh[i]);
    }
    auto load = [&](int ci, BackIn<T, DP>& in) {
      const Rows<T> krows = dims.rows(k, b, ci * kChunk, h);
#pragma unroll
      for (int st = 0; st < KS; ++st) in.kf[st] = krows.row(16 * w + c, 32 * st + 8 * grp);
      const T* tb = tf + (chunk0 + ci) * Factor<T, NT>::kElems + col_step(w, 0) * F::kStep;
      in.tf[0] = F::get(tb, 0);
      in.tf[1] = F::get(tb, w < 2 ? 1 : 0);
      const float* co = coef + (chunk0 + ci) * kCoef + 16 * w + 4 * grp;
      in.beta = *reinterpret_cast<const f32x4*>(co);
      in.eps = *reinterpret_cast<const f32x4*>(co + kChunk);
      in.kap = *reinterpret_cast<const f32x4*>(co + 2 * kChunk);
      in.gam = coef[(chunk0 + ci) * kCoef + 2 * kChunk - 1];
    };
    auto step = [&](int ci, const BackIn<T, DP>& in) {
      const Record rh = record(rec_dh, chunk0 + ci, D, D);
#pragma unroll
      for (int i = 0; i < FT; ++i) rh.put(vcol, 16 * (w + 4 * i) + 4 * grp, dh[i]);
      // dDelta = P^T dO + kap (K dH')
      f32x4 x = zero4();
#pragma unroll
      for (int st = 0; st < KS; ++st) x = mma(in.kf[st], F::get(lds.state, st), x);
      const f32x4 z = *reinterpret_cast<const f32x4*>(lds.z + (w * 64 + lane) * 4);
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = in.kap[r] * x[r] + z[r];
      F::put(lds.ddelta, w, x);
      lds_barrier();
      // dR = T^T dDelta
      f32x4 dr;
      if (w < 2) {
        dr = mma(in.tf[0], F::get(lds.ddelta, 0), zero4());
        dr = mma(in.tf[1], F::get(lds.ddelta, 1), dr);
      } else {
        dr = mma(in.tf[0], F::get(lds.ddelta, 1), zero4());
      }
      f32x4 y;
#pragma unroll
      for (int r = 0; r < 4; ++r) y[r] = -(in.beta[r] * in.eps[r]) * dr[r];
      F::put(lds.dread, w, y);
      f32x4 add[FT];
#pragma unroll
      for (int i = 0; i < FT; ++i)
        add[i] = w + 4 * i < S::TILES ? *reinterpret_cast<const f32x4*>(lds.qdo + ((w + 4 * i) * 64 + lane) * 4) : zero4();
      record(rec_dr, chunk0 + ci, kChunk, D).put(vcol, 16 * w + 4 * grp, dr);
      const Rows<T> dvrows = dims.rows(dv, b, ci * kChunk, h);
#pragma unroll
      for (int r = 0; r < 4; ++r) dvrows.put_one(16 * w + 4 * grp + r, vcol, from_f32<T>(in.beta[r] * dr[r]));
      lds_barrier();
      // dH = gam dH' + Q^T (eps dO) - K^T (beta eps dR)
      const Operand<T, NT> y0 = F::get(lds.dread, 0), y1 = F::get(lds.dread, 1);
#pragma unroll
      for (int i = 0; i < FT; ++i) {
        const int ft = w + 4 * i;
        if (ft < S::TILES) {
#pragma unroll
          for (int r = 0; r < 4; ++r) dh[i][r] = in.gam * dh[i][r] + add[i][r];
          dh[i] = mma(load_columns(lds.keys, S::PITCH, 0, 16 * ft), y0, dh[i]);
          dh[i] = mma(load_columns(lds.keys, S::PITCH, 1, 16 * ft), y1, dh[i]);
          F::put(lds.state, ft, dh[i]);
        }
      }
      lds_barrier();
    };
    BackIn<T, DP> a, bb;
    load(nc - 1, a);
    lds_barrier();
    lds_barrier();
    for (int ci = nc - 1; ci >= 0; ci -= 2) {  // past the first chunk it is loaded again, so that no load is conditional
      load(ci >= 1 ? ci - 1 : 0, bb);
      step(ci, a);
      if (ci < 1) break;
      load(ci >= 2 ? ci - 2 : 0, a);
      step(ci - 1, bb);
    }
    float* so = d_state_in + (size_t)bh * D * D;
#pragma unroll
    for (int i = 0; i < FT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int f = 16 * (w + 4 * i) + 4 * grp + r;
        if (f < D && vcol < D) so[(size_t)f * D + vcol] = dh[i][r];
      }
  } else {
    // ---- the keys of the chunk in hand into LDS; of the next chunk the queries, dO and eps dO, then P^T dO, then
    //      Q^T (eps dO), each in one of the three spans between barriers ----
    const int hl = threadIdx.x - 256;
    auto load_tile = [&](const T* src, int ci, BackTile<T, DP>& in) {
      const Rows<T> rows = dims.rows(src, b, ci * kChunk, h);
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {
        const int p = hl + 256 * i;
        in.x[i] = rows.row(p / (DP / 8), 8 * (p % (DP / 8)));
      }
    };
    auto put_tile = [&](T* dst, const BackTile<T, DP>& in) {
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {
        const int p = hl + 256 * i, row = p / (DP / 8), f = 8 * (p % (DP / 8));
        T* at = dst + row * S::PITCH + f;
        if constexpr (sizeof(T) == 2) {
          *reinterpret_cast<bf16x8*>(at) = in.x[i].p[0];
        } else {
          reinterpret_cast<f32x4*>(at)[0] = in.x[i].lo;
          reinterpret_cast<f32x4*>(at)[1] = in.x[i].hi;
        }
      }
    };
    auto load_side = [&](int ci, BackSide<T, DP>& in) {
      const T* pb = pf + (chunk0 + ci) * Factor<T, NT>::kElems + col_step(w, 0) * F::kStep;
      in.pf[0] = F::get(pb, 0);
      in.pf[1] = F::get(pb, w < 2 ? 1 : 0);
      in.eps = *reinterpret_cast<const f32x4*>(coef + (chunk0 + ci) * kCoef + kChunk + 16 * w + 4 * grp);
      const Rows<T> rows = dims.rows(d_o, b, ci * kChunk, h);
      const __amdgpu_buffer_rsrc_t flags = dims.flags(active, b, ci * kChunk);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        in.d_o[r] = rows.one(16 * w + 4 * grp + r, vcol);
        in.on[r] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(flags, 16 * w + 4 * grp + r, 0, 0);
      }
    };
    auto put_side = [&](const BackSide<T, DP>& in) {
      f32x4 x, e;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[r] = active == nullptr || in.on[r] ? to_f32(in.d_o[r]) : 0.f;
        e[r] = in.eps[r] * x[r];
      }
      F1::put(lds.d_o, w, x);
      F::put(lds.edo, w, e);
    };
    auto form_z = [&](const BackSide<T, DP>& in) {
      f32x4 z;
      if (w < 2) {
        z = mma(in.pf[0], F1::get(lds.d_o, 0), zero4());
        z = mma(in.pf[1], F1::get(lds.d_o, 1), z);
      } else {
        z = mma(in.pf[0], F1::get(lds.d_o, 1), zero4());
      }
      *reinterpret_cast<f32x4*>(lds.z + (w * 64 + lane) * 4) = z;
    };
    auto query_columns = [&](int ci, int s, int f0) -> Operand<T, 1> {
      if constexpr (S::kStageQ) {
        return load_columns(lds.queries, S::PITCH, s, f0);
      } else {
        Operand<T, 1> x;
        const Rows<T> rows = dims.rows(q, b, ci * kChunk, h);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x.lo[e] = rows.one(32 * s + 8 * grp + e, f0 + c);
          x.hi[e] = rows.one(32 * s + 8 * grp + 4 + e, f0 + c);
        }
        return x;
      }
    };
    auto form_qdo = [&](int ci) {
      const Operand<T, NT> e0 = F::get(lds.edo, 0), e1 = F::get(lds.edo, 1);
#pragma unroll
      for (int i = 0; i < FT; ++i) {
        const int ft = w + 4 * i;
        if (ft < S::TILES) {
          f32x4 x = mma(query_columns(ci, 0, 16 * ft), e0, zero4());
          x = mma(query_columns(ci, 1, 16 * ft), e1, x);
          *reinterpret_cast<f32x4*>(lds.qdo + (ft * 64 + lane) * 4) = x;
        }
      }
    };
    BackTile<T, DP> keys, queries;
    BackSide<T, DP> side;
    load_tile(k, nc - 1, keys);
    if constexpr (S::kStageQ) load_tile(q, nc - 1, queries);
    load_side(nc - 1, side);
    if constexpr (S::kStageQ) put_tile(lds.queries, queries);
    put_side(side);
    lds_barrier();
    form_z(side);
    form_qdo(nc - 1);
    if constexpr (S::kStageQ) load_tile(q, nc > 1 ? nc - 2 : 0, queries);
    load_side(nc > 1 ? nc - 2 : 0, side);
    lds_barrier();
    for (int ci = nc - 1; ci >= 0; --ci) {  // past the first chunk it is formed again, so that nothing is conditional
      put_tile(lds.keys, keys);
      load_tile(k, ci >= 1 ? ci - 1 : 0, keys);
      if constexpr (S::kStageQ) put_tile(lds.queries, queries);
      put_side(side);
      lds_barrier();
      form_z(side);
      if constexpr (S::kStageQ) load_tile(q, ci >= 2 ? ci - 2 : 0, queries);
      load_side(ci >= 2 ? ci - 2 : 0, side);
      lds_barrier();
      form_qdo(ci >= 1 ? ci - 1 : 0);
      lds_barrier();
    }
  }
}

// --------------------------------------------------------------------------------------------
// the other gradients
// --------------------------------------------------------------------------------------------
// Rows of float32 in LDS as NP planes of pieces (float32 itself: one plane).
template <typename T, int NP, int ROWS, int PITCH> struct Planes {
  static constexpr int kPlane = ROWS * PITCH;
  T x[NP * kPlane];
  __device__ __forceinline__ void put(int row, int col, f32x4 v) {
    if constexpr (sizeof(T) == 2) {
      bf16x4 p[NP];
      split4<NP>(v, p);
#pragma unroll
      for (int i = 0; i < NP; ++i) *reinterpret_cast<bf16x4*>(x + i * kPlane + row * PITCH + col) = p[i];
    } else {
      *reinterpret_cast<f32x4*>(x + row * PITCH + col) = v;
    }
  }
  // column f0 + c of rows 8 g .. 8 g + 7
  __device__ __forceinline__ Operand<T, NP> columns(int f0) const {
    Operand<T, NP> o;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < NP; ++i) o.p[i] = load_columns<T>(x + i * kPlane, PITCH, 0, f0).p[0];
    } else {
      const Operand<T, 1> y = load_columns<T>(x, PITCH, 0, f0);
      o.lo = y.lo;
      o.hi = y.hi;
    }
    return o;
  }
};

// Column f0 + c of a tile's rows 32 s + 4 g + r and 32 s + 16 + 4 g + r: the k order of a pair of accumulator tiles.
template <typename T>
__device__ __forceinline__ Operand<T, 1> load_columns_paired(const T* tile, int pitch, int s, int f0) {
  Operand<T, 1> o;
  if constexpr (sizeof(T) == 2) {
    const bf16x4 a = read_tr16_rows<bf16x4>(tile, pitch, 32 * s, f0), b = read_tr16_rows<bf16x4>(tile, pitch, 32 * s + 16, f0);
    o.p[0] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
    const T* p = tile + (32 * s + 4 * lane_grp()) * pitch + f0 + lane_col();
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o.lo[e] = p[e * pitch];
      o.hi[e] = p[(16 + e) * pitch];
    }
  }
  return o;
}

// A pair of accumulator tiles as the operand whose k run down their rows.
template <typename T, int NP>
__device__ __forceinline__ Operand<T, NP> paired(f32x4 a, f32x4 b) {
  Operand<T, NP> o;
  if constexpr (sizeof(T) == 2) {
    bf16x4 x[NP], y[NP];
    split4<NP>(a, x);
    split4<NP>(b, y);
#pragma unroll
    for (int i = 0; i < NP; ++i) o.p[i] = __builtin_shufflevector(x[i], y[i], 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
    o.lo = a;
    o.hi = b;
  }
  return o;
}

template <typename T, int NP>
__device__ __forceinline__ float operand_dot(const Operand<T, NP>& a, const Operand<T, 1>& b) {
  float s = 0.f;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float x = (float)a.p[NP - 1][e];
#pragma unroll
      for (int i = NP - 2; i >= 0; --i) x += (float)a.p[i][e];
      s += x * (float)b.p[0][e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) s += a.lo[e] * b.lo[e] + a.hi[e] * b.hi[e];
  }
  return s;
}

template <typename T>
__device__ __forceinline__ f32x4 four(const T* p) {
  f32x4 x;
  if constexpr (sizeof(T) == 2) {
    const bf16x4 y = *reinterpret_cast<const bf16x4*>(p);
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = (float)y[r];
  } else {
    x = *reinterpret_cast<const f32x4*>(p);
  }
  return x;
}

template <typename T, int DP> struct GradShape {
  static constexpr int TILES = DP / 16;
  static constexpr int NT = Pieces<T>::kN;
  static constexpr int PAD = sizeof(T) == 2 ? 8 : 4;
  static constexpr int PITCH = DP + PAD;
  using States = Planes<T, NT, 32, DP + PAD>;
  using Tokens = Planes<T, NT, 32, kChunk + PAD>;
  struct Values {  // 32 value columns
    States h, dh;
    Tokens delta, dr;
  };
  struct Rows {
    T keys[kChunk * PITCH];
    T queries[kChunk * PITCH];
  };
  struct Lds {
    union {
      Values values;
      Rows rows;
    } u;
    double sums[kChunk];
    float beta[kChunk], eps[kChunk], kap[kChunk], dsum[kChunk];
    float part[4][2];  // each wave's share of <dH', H> and of the chunk end's other terms
  };
};

template <typename T, int DP>
__global__ __launch_bounds__(256) void gated_grad_kernel(
    const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, const float* __restrict__ g,
    const T* __restrict__ d_o, const float* __restrict__ coef, const float* __restrict__ rec_h,
    const float* __restrict__ rec_d, const float* __restrict__ rec_dh, const float* __restrict__ rec_dr,
    const uint8_t* __restrict__ active, T* __restrict__ dq, T* __restrict__ dk, T* __restrict__ dbeta,
    float* __restrict__ dg, Dims<T> dims) {
  using S = GradShape<T, DP>;
  constexpr int NT = S::NT, TILES = S::TILES;
  __shared__ __attribute__((aligned(16))) typename S::Lds lds;
  const int id = xcd_logical_block(blockIdx.x, gridDim.x);
  const int chunk = id % dims.chunks, bh = id / dims.chunks, h = bh % dims.H, b = bh / dims.H;
  const int D = dims.D, t0 = chunk * kChunk;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63, c = l & 15, grp = l >> 4;

  // the decays' sums, as the prep kernel forms them
  float gl = 0.f;
  if (w == 0) {
    const bool ok = t0 + l < dims.N;
    gl = g[((size_t)b * dims.N + (ok ? t0 + l : t0)) * dims.H + h];
    double sum = ok ? ((double)gl < kLeastDecay ? kLeastDecay : (double)gl) : 0.0;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const double up = __shfl_up(sum, off);
      if (l >= off) sum += up;
    }
    lds.sums[l] = sum;
    const float* co = coef + (size_t)id * kCoef;
    lds.beta[l] = co[l];
    lds.eps[l] = co[kChunk + l];
    lds.kap[l] = co[2 * kChunk + l];
  }

  // ---- sums over the value columns, 32 at a time ----
  f32x4 aq[TILES], ay[TILES], ac[TILES];  // dQ^T, Y^T, C^T: rows features, columns the wave's tokens
#pragma unroll
  for (int i = 0; i < TILES; ++i) aq[i] = ay[i] = ac[i] = zero4();
  // by rows j, columns the wave's tokens i: dP^T, B^T (j <= i); by rows i, columns the wave's tokens j: dP, B (i >= j)
  f32x4 pt[4], bt[4], pr[4], br[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) pt[i] = bt[i] = pr[i] = br[i] = zero4();
  float inner = 0.f, dot_v = 0.f;
  const int token = t0 + 16 * w + c;
  const Rows<T> dorows = dims.rows(d_o, b, t0, h), vrows = dims.rows(v, b, t0, h);
  bool on[4];  // of token 16 i + c
  {
    const __amdgpu_buffer_rsrc_t flags = dims.flags(active, b, t0);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      on[i] = active == nullptr || (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(flags, 16 * i + c, 0, 0) != 0;
  }
  for (int v0 = 0; v0 < D; v0 += 32) {
    if (v0 > 0) __syncthreads();
    constexpr int QUADS = DP / 4;
    for (int p = threadIdx.x; p < 32 * QUADS; p += 256) {
      const int row = p / QUADS, f = 4 * (p % QUADS);
      const bool ok = v0 + row < D && f < D;
      const size_t at = ((size_t)id * D + (ok ? v0 + row : 0)) * D + (ok ? f : 0);
      f32x4 x = *reinterpret_cast<const f32x4*>(rec_h + at), y = *reinterpret_cast<const f32x4*>(rec_dh + at);
      if (!ok) x = y = zero4();
      inner += (x[0] * y[0] + x[1] * y[1]) + (x[2] * y[2] + x[3] * y[3]);
      lds.u.values.h.put(row, f, x);
      lds.u.values.dh.put(row, f, y);
    }
    for (int p = threadIdx.x; p < 32 * (kChunk / 4); p += 256) {
      const int row = p / (kChunk / 4), t = 4 * (p % (kChunk / 4));
      const bool ok = v0 + row < D;
      const size_t at = ((size_t)id * D + (ok ? v0 + row : 0)) * kChunk + t;
      f32x4 x = *reinterpret_cast<const f32x4*>(rec_d + at), y = *reinterpret_cast<const f32x4*>(rec_dr + at);
      if (!ok) x = y = zero4();
      lds.u.values.delta.put(row, t, x);
      lds.u.values.dr.put(row, t, y);
    }
    Operand<T, 1> dof[4];
    const int vc = v0 + 8 * grp;
#pragma unroll
    for (int i = 0; i < 4; ++i) dof[i] = dorows.row(16 * i + c, on[i] ? vc : D);
    const Operand<T, 1> vf = vrows.row(16 * w + c, vc);
    __syncthreads();
    const Operand<T, NT> del_w = lds.u.values.delta.columns(16 * w), dr_w = lds.u.values.dr.columns(16 * w);
    dot_v += operand_dot(dr_w, vf);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i <= w) {
        const Operand<T, NT> x = lds.u.values.delta.columns(16 * i);
        Operand<T, 1> own = dof[0];
        if (w == 1) own = dof[1];
        if (w == 2) own = dof[2];
        if (w == 3) own = dof[3];
        pt[i] = mma(x, own, pt[i]);
        bt[i] = mma(x, dr_w, bt[i]);
      }
      if (i >= w) {
        pr[i] = mma(dof[i], del_w, pr[i]);
        br[i] = mma(lds.u.values.dr.columns(16 * i), del_w, br[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      const Operand<T, NT> x = lds.u.values.h.columns(16 * i);
      Operand<T, 1> own = dof[0];
      if (w == 1) own = dof[1];
      if (w == 2) own = dof[2];
      if (w == 3) own = dof[3];
      aq[i] = mma(x, own, aq[i]);
      ay[i] = mma(x, dr_w, ay[i]);
      ac[i] = mma(lds.u.values.dh.columns(16 * i), del_w, ac[i]);
    }
  }
  __syncthreads();

  // ---- the keys and queries, the decays between pairs, sums over the chunk's tokens ----
  {
    constexpr int PIECES = kChunk * (DP / 8);
    const Rows<T> krows = dims.rows(k, b, t0, h), qrows = dims.rows(q, b, t0, h);
#pragma unroll
    for (int p = threadIdx.x; p < PIECES; p += 256) {
      const int row = p / (DP / 8), f = 8 * (p % (DP / 8));
      const Operand<T, 1> x = krows.row(row, f), y = qrows.row(row, f);
      T *kd = lds.u.rows.keys + row * S::PITCH + f, *qd = lds.u.rows.queries + row * S::PITCH + f;
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<bf16x8*>(kd) = x.p[0];
        *reinterpret_cast<bf16x8*>(qd) = y.p[0];
      } else {
        reinterpret_cast<f32x4*>(kd)[0] = x.lo;
        reinterpret_cast<f32x4*>(kd)[1] = x.hi;
        reinterpret_cast<f32x4*>(qd)[0] = y.lo;
        reinterpret_cast<f32x4*>(qd)[1] = y.hi;
      }
    }
  }
  const int own = 16 * w + c;
  const float beta_own = lds.beta[own], eps_own = lds.eps[own], kap_own = lds.kap[own];
  const double sum_own = lds.sums[own];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 16 * i + 4 * grp + r;
      if (i <= w) {  // row j, column i
        const float e = row <= own ? expf((float)(sum_own - lds.sums[row])) : 0.f;
        pt[i][r] *= e;
        bt[i][r] *= row < own ? e : 0.f;
      }
      if (i >= w) {  // row i, column j
        const float e = row >= own ? expf((float)(lds.sums[row] - sum_own)) : 0.f;
        pr[i][r] *= e;
        br[i][r] *= row > own ? -lds.beta[row] * e : 0.f;
      }
    }
#pragma unroll
  for (int i = 0; i < TILES; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      aq[i][r] *= eps_own;
      ay[i][r] *= eps_own;
      ac[i][r] *= kap_own;
    }
  __syncthreads();
  float end = 0.f;  // sum_j kap_j k_j.(dH' Delta_j)
#pragma unroll
  for (int i = 0; i < TILES; ++i) {
    const f32x4 kx = four(lds.u.rows.keys + own * S::PITCH + 16 * i + 4 * grp);
#pragma unroll
    for (int r = 0; r < 4; ++r) end += kx[r] * ac[i][r];
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    if (2 * s <= w) {
      const Operand<T, NT> x = paired<T, NT>(pt[2 * s], pt[2 * s + 1]), y = paired<T, NT>(bt[2 * s], bt[2 * s + 1]);
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        const Operand<T, 1> kc = load_columns_paired(lds.u.rows.keys, S::PITCH, s, 16 * i);
        aq[i] = mma(kc, x, aq[i]);
        ay[i] = mma(kc, y, ay[i]);
      }
    }
    if (2 * s + 1 >= w) {
      const Operand<T, NT> x = paired<T, NT>(pr[2 * s], pr[2 * s + 1]), y = paired<T, NT>(br[2 * s], br[2 * s + 1]);
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        ac[i] = mma(load_columns_paired(lds.u.rows.queries, S::PITCH, s, 16 * i), x, ac[i]);
        ac[i] = mma(load_columns_paired(lds.u.rows.keys, S::PITCH, s, 16 * i), y, ac[i]);
      }
    }
  }

  // ---- out ----
  float dot_q = 0.f, dot_y = 0.f, dot_c = 0.f;
  const Rows<T> dqrows = dims.rows(dq, b, t0, h), dkrows = dims.rows(dk, b, t0, h);
#pragma unroll
  for (int i = 0; i < TILES; ++i) {
    const int f = 16 * i + 4 * grp;
    const f32x4 kx = four(lds.u.rows.keys + own * S::PITCH + f), qx = four(lds.u.rows.queries + own * S::PITCH + f);
    f32x4 x;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float y = -ay[i][r];
      dot_q += qx[r] * aq[i][r];
      dot_y += kx[r] * y;
      dot_c += kx[r] * ac[i][r];
      x[r] = beta_own * y + ac[i][r];
    }
    dqrows.put_four(own, f, aq[i]);
    dkrows.put_four(own, f, x);
  }
  dot_q = sum_over_rows(dot_q);
  dot_y = sum_over_rows(dot_y);
  dot_c = sum_over_rows(dot_c);
  dot_v = sum_over_rows(dot_v);
  if (grp == 0) {
    lds.dsum[own] = dot_q + beta_own * dot_y - dot_c;
    if (token < dims.N) dbeta[((size_t)b * dims.N + token) * dims.H + h] = from_f32<T>(dot_v + dot_y);
  }
  inner = group_sum<64>(inner);
  end = group_sum<64>(end);
  if (l == 0) {
    lds.part[w][0] = inner;
    lds.part[w][1] = end;
  }
  __syncthreads();
  if (w == 0) {
    float x = lds.dsum[l];  // the sum over this token and those behind it
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const float down = __shfl_down(x, off);
      if (l + off < 64) x += down;
    }
    const float hh = (lds.part[0][0] + lds.part[1][0]) + (lds.part[2][0] + lds.part[3][0]);
    const float ee = (lds.part[0][1] + lds.part[1][1]) + (lds.part[2][1] + lds.part[3][1]);
    x += lds.eps[kChunk - 1] * hh + ee;
    // what forgets the state has no gradient
    if (t0 + l < dims.N) dg[((size_t)b * dims.N + t0 + l) * dims.H + h] = (double)gl < kLeastDecay ? 0.f : x;
  }
}

size_t align16(size_t x) { return (x + 15) & ~(size_t)15; }

// coefficients, T and P by columns, then dH' and dR of every chunk and head
template <typename T> size_t factor_bytes(size_t total) {
  return align16(total * kCoef * sizeof(float)) + 2 * total * sizeof(T) * Factor<T, Pieces<T>::kN>::kElems;
}
template <typename T> size_t backward_bytes(size_t total, int D) { return factor_bytes<T>(total) + record_bytes(total, D); }

template <typename T, int DP>
void launch_back(const T* q, const T* k, const T* v, const float* g, const T* d_o, const float* d_state,
                 const uint8_t* active, const float* rec_h, const float* rec_d, const float* coef, const T* tf,
                 const T* pf, float* rec_dh, float* rec_dr, T* dq, T* dk, T* dv, T* dbeta, float* dg, float* d_state_in,
                 Dims<T> dims, int B, hipStream_t stream) {
  const int slices = (dims.D + 15) / 16;
  hipLaunchKernelGGL((gated_chain_backward_kernel<T, DP>), dim3((unsigned)(B * dims.H * slices)), dim3(512), 0, stream, q, k, d_o,
                     coef, tf, pf, d_state, dv, d_state_in, active, rec_dh, rec_dr, dims, slices);
  hipLaunchKernelGGL((gated_grad_kernel<T, DP>), dim3((unsigned)(B * dims.H * dims.chunks)), dim3(256), 0, stream, q, k, v, g,
                     d_o, coef, rec_h, rec_d, rec_dh, rec_dr, active, dq, dk, dbeta, dg, dims);
}

template <typename T>
int scan_backward(const void* q_, const void* k_, const void* v_, const void* beta_, const float* g,
                  const float* records, size_t records_bytes, const void* d_o_, const float* d_state,
                  const uint8_t* active, void* dq_, void* dk_, void* dv_, void* dbeta_, float* dg, float* d_state_in,
                  void* ws, size_t ws_bytes, int B, int N, int H, int D, hipStream_t stream, const char* who) {
  if (const int st = check_sizes(B, N, H, D, who); st != OK) return st;
  if (B == 0 || N == 0) return fail(ERR_ARG, "%s: no tokens (B=%d N=%d)", who, B, N);
  const size_t total = (size_t)B * H * chunks_of(N);
  if (!q_ || !k_ || !v_ || !beta_ || !g || !records || !d_o_ || !dq_ || !dk_ || !dv_ || !dbeta_ || !dg || !d_state_in || !ws)
    return fail(ERR_ARG, "%s: null pointer", who);
  if ((reinterpret_cast<uintptr_t>(q_) | reinterpret_cast<uintptr_t>(k_) | reinterpret_cast<uintptr_t>(v_) |
       reinterpret_cast<uintptr_t>(d_o_) | reinterpret_cast<uintptr_t>(dq_) | reinterpret_cast<uintptr_t>(dk_) |
       reinterpret_cast<uintptr_t>(dv_) | reinterpret_cast<uintptr_t>(ws) | reinterpret_cast<uintptr_t>(records)) & 15)
    return fail(ERR_ARG, "%s: q, k, v, their gradients, d_o, the workspace and the records must be 16-byte aligned", who);
  if (ws_bytes < backward_bytes<T>(total, D))
    return fail(ERR_ARG, "%s: workspace of %zu bytes, needs %zu", who, ws_bytes, backward_bytes<T>(total, D));
  if (records_bytes < record_bytes(total, D))
    return fail(ERR_ARG, "%s: records of %zu bytes, need %zu", who, records_bytes, record_bytes(total, D));
  const T *q = static_cast<const T*>(q_), *k = static_cast<const T*>(k_), *v = static_cast<const T*>(v_);
  const T *beta = static_cast<const T*>(beta_), *d_o = static_cast<const T*>(d_o_);
  T *dq = static_cast<T*>(dq_), *dk = static_cast<T*>(dk_), *dv = static_cast<T*>(dv_), *dbeta = static_cast<T*>(dbeta_);
  float* coef = static_cast<float*>(ws);
  T* tf = reinterpret_cast<T*>(static_cast<char*>(ws) + align16(total * kCoef * sizeof(float)));
  T* pf = tf + total * Factor<T, Pieces<T>::kN>::kElems;
  float* rec_dh = reinterpret_cast<float*>(static_cast<char*>(ws) + factor_bytes<T>(total));
  float* rec_dr = rec_dh + total * D * D;
  const float* rec_d = records + total * D * D;
  const Dims<T> dims{N, H, D, chunks_of(N)};
  if (const int st = launch_prep<T>(q, k, beta, g, coef, tf, pf, B, N, H, D, true, stream); st != OK) return st;
#define VSP_BACK(DP) launch_back<T, DP>(q, k, v, g, d_o, d_state, active, records, rec_d, coef, tf, pf, rec_dh, rec_dr, dq, dk, \
                                        dv, dbeta, dg, d_state_in, dims, B, stream)
  switch (width_of(D)) {
    case 32: VSP_BACK(32); break;
    case 64: VSP_BACK(64); break;
    case 128: VSP_BACK(128); break;
    default: VSP_BACK(256); break;
  }
#undef VSP_BACK
  return check_launch(who);
}

}  // namespace
}  // namespace gated
}  // namespace vsp

extern "C" size_t vsp_gated_scan_backward_workspace_bytes(int B, int N, int H, int D, int fp32) {
  using namespace vsp::gated;
  if (B <= 0 || N <= 0 || H <= 0 || D <= 0) return 0;
  const size_t total = (size_t)B * H * chunks_of(N);
  return fp32 ? backward_bytes<float>(total, D) : backward_bytes<__bf16>(total, D);
}

extern "C" int vsp_gated_scan_backward_bf16(const void* q, const void* k, const void* v, const void* beta,
                                            const float* g, const void* records, size_t records_bytes, const void* d_o,
                                            const float* d_state, const uint8_t* active, void* dq, void* dk, void* dv,
                                            void* dbeta, float* dg, float* d_state_in, void* workspace,
                                            size_t workspace_bytes, int B, int N, int H, int D, void* stream) {
  return vsp::gated::scan_backward<__bf16>(q, k, v, beta, g, static_cast<const float*>(records), records_bytes, d_o, d_state, active,
                                           dq, dk, dv, dbeta, dg, d_state_in, workspace, workspace_bytes, B, N, H, D,
                                           reinterpret_cast<hipStream_t>(stream), "vsp_gated_scan_backward_bf16");
}

extern "C" int vsp_gated_scan_backward_f32(const void* q, const void* k, const void* v, const void* beta,
                                           const float* g, const void* records, size_t records_bytes, const void* d_o,
                                           const float* d_state, const uint8_t* active, void* dq, void* dk, void* dv,
                                           void* dbeta, float* dg, float* d_state_in, void* workspace,
                                           size_t workspace_bytes, int B, int N, int H, int D, void* stream) {
  return vsp::gated::scan_backward<float>(q, k, v, beta, g, static_cast<const float*>(records), records_bytes, d_o, d_state, active,
                                          dq, dk, dv, dbeta, dg, d_state_in, workspace, workspace_bytes, B, N, H, D,
                                          reinterpret_cast<hipStream_t>(stream), "vsp_gated_scan_backward_f32");
}
