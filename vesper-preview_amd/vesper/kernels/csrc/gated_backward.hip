// The gated delta rule's backward pass on CDNA4 (gfx950); notation and operands as in gated.h.
//
// With dH' the gradient of a chunk's end state and dO its outputs' gradients (zero where inactive):
//   dDelta = P^T dO + kap (K dH'),  dR = T^T dDelta,  dV = beta dR,
//   dH = gam dH' + Q^T (eps dO) - K^T (beta eps dR).
// With dP_ij = E_ij dO_i.Delta_j (j <= i) and B_ij = E_ij dR_i.Delta_j (j < i):
//   dQ_i = eps_i H dO_i + sum_j dP_ij k_j,    Y_i = -(eps_i H dR_i + sum_j B_ij k_j),
//   C_j = kap_j dH' Delta_j + sum_i dP_ij q_i - sum_i beta_i B_ij k_i,
//   dK_i = beta_i Y_i + C_i,   dbeta_i = dR_i.v_i + k_i.Y_i.
// A token's decay is in every exponent that reaches over it, and its gradient is the sum of their terms:
//   dg_t = sum_{i >= t} eps_i (q_i.(H dO_i) - beta_i k_i.(H dR_i)) + sum_{j < t <= i} (dP_ij q_i.k_j - beta_i B_ij k_i.k_j)
//        + sum_{j < t} kap_j k_j.(dH' Delta_j) + gam <dH', H>.
// Every term has e^{g_t} in it. The sums G_i's own gradients, summed over i >= t, are the same number as the
// difference of terms that have not: behind decays of e^-10 and less their rounding was all that was left of it.
//
//  * gated_prep_kernel (gated_scan.hip) forms T and P again, as operands by columns.
//  * gated_chain_backward_kernel walks the chunks from the last to the first like the forward's chain, a workgroup a
//    head and 16 value columns: four waves carry dH through three dependent products, four more bring everything into
//    LDS ahead and form P^T dO and Q^T (eps dO) of the next chunk. It keeps dH' and dR of each chunk.
//  * gated_grad_kernel: a workgroup a chunk and head, all at once, for the rest: wave w holds dQ, Y and C of the
//    16 tokens w, sums over the value columns 32 at a time from H, dH', Delta and dR in pieces in LDS, then over
//    the chunk's tokens with accumulator tiles as operands.
#include <type_traits>

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
  static constexpr int NT = Pieces<T>::kN;
  // float32 queries are read from memory by columns: the LDS has no room for them beside the rest
  static constexpr bool kStageQ = sizeof(T) == 2;
  using F = Frags<T, NT>;
  using Keys = Tile<T, DP>;
  using Slice = Tile<T, 16>;
  // How many chunks ahead of the one in hand the loads of keys into LDS go; heads of width 256 have room for the chunk in
  // hand only, and wait for each.
  static constexpr int LEAD = DP > 128 ? 0 : 2, RING = LEAD + 1, QRING = LEAD == 0 ? 1 : 2;
  struct Lds {
    T keys[RING][Keys::kElems];
    float coef[3][kCoefLds];
    T queries[QRING][kStageQ ? Keys::kElems : 8];
    T d_o[2][Slice::kElems];
    T state[KS * F::kStep];      // dH
    T ddelta[2 * F::kStep];
    T dread[2 * F::kStep];       // -beta eps dR
    float z[4 * 256];            // P^T dO, accumulator tiles one after the other
    float qdo[TILES * 256];      // Q^T (eps dO)
  };
  static_assert(sizeof(Lds) <= 160 * 1024, "more than a CU's LDS");
  // direct loads of one wave for a chunk: queries, keys, a slice of dO and the coefficients (bf16: two waves each)
  static constexpr int kLoads = (kStageQ ? 2 : 1) * Keys::kInstr / 4 + (sizeof(T) == 2 ? 1 : 2);
};

// What a chain wave reads of a chunk from memory: its tokens' columns of T.
template <typename T> struct BackChainIn { Operand<T, Pieces<T>::kN> t[2]; };

template <typename T> struct BackIn {  // what the other waves keep of a chunk in registers
  Operand<T, Pieces<T>::kN> pf[2];
  uint8_t on;  // of token l
};

// As the forward's chain: three dependent products a chunk, then memory. B2 T1500 H8 d128 41 us (24 chunks of 1.7 us on half of
// the CUs), B16 T1024 H12 d64 103 us (310 MB). dV left it for the next kernel (four scattered stores a wave and chunk), the
// operands of T went from LDS into registers, and the loads over the three spans: 52 to 41 us.
template <typename T, int DP>
__global__ __launch_bounds__(512) void gated_chain_backward_kernel(
    const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ d_o, const float* __restrict__ coef,
    const T* __restrict__ tf, const T* __restrict__ pf, const float* __restrict__ d_state,
    float* __restrict__ d_state_in, const uint8_t* __restrict__ active, float* __restrict__ rec_dh,
    float* __restrict__ rec_dr, Dims<T> dims, int slices) {
  using S = BackShape<T, DP>;
  using F = typename S::F;
  using Keys = typename S::Keys;
  using Slice = typename S::Slice;
  constexpr int KS = S::KS, FT = S::FT, TILES = S::TILES, NT = S::NT, LEAD = S::LEAD, RING = S::RING, QRING = S::QRING;
  __shared__ __attribute__((aligned(16))) typename S::Lds lds;

  const int id = xcd_logical_block(blockIdx.x, gridDim.x);
  const int sl = id % slices, bh = id / slices, h = bh % dims.H, b = bh / dims.H;
  const int D = dims.D, nc = dims.chunks;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & 3;
  const int c = lane_col(), grp = lane_grp(), lane = threadIdx.x & 63;
  const size_t chunk0 = (size_t)bh * nc;

  // features past D and rows past the end are not brought: zeros, and what another chunk left there, times zeros
  for (int i = threadIdx.x; i < (int)((sizeof(lds.keys) + sizeof(lds.coef) + sizeof(lds.queries) + sizeof(lds.d_o)) / 16); i += 512)
    reinterpret_cast<f32x4*>(&lds)[i] = zero4();
  lds_barrier();

  if (wave < 4) {
    // ---- the chain: wave w has the 16 tokens w of dDelta and dR, and of dH's feature tiles each fourth ----
    __builtin_amdgcn_s_setprio(3);
    const int vcol = 16 * sl + c, own = 16 * w + 4 * grp;
    const T* tp = tf + chunk0 * Factor<T, NT>::kElems;
    f32x4 dh[FT];
#pragma unroll
    for (int i = 0; i < FT; ++i) {
      const int ft = w + 4 * i;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int f = 16 * ft + 4 * grp + r;
        dh[i][r] = d_state != nullptr && f < D && vcol < D ? d_state[((size_t)bh * D + f) * D + vcol] : 0.f;
      }
      if (ft < TILES) F::template put_tile<true>(lds.state, ft, dh[i]);
    }
    lds_barrier();
    lds_barrier();
    lds_barrier();
    // BOTH: the wave's columns of T have two steps. The code twice, so that no load is conditional
    auto run = [&](auto both) {
      constexpr bool BOTH = decltype(both)::value;
      auto load = [&](int it, BackChainIn<T>& to) {
        const T* tc = tp + (size_t)(it < nc ? nc - 1 - it : 0) * Factor<T, NT>::kElems;
        if constexpr (BOTH) to.t[0] = F::get(tc, col_step(w, 0));
        to.t[1] = F::get(tc, col_step(w, 1));
      };
      BackChainIn<T> ta, tb;
      load(0, ta);
      int slot = 0, cslot = 0;
      auto step = [&](int it, const BackChainIn<T>& tin, BackChainIn<T>& next) {
        const int ci = nc - 1 - it;
        const T* keys = lds.keys[slot];
        const float* co = lds.coef[cslot];
        slot = slot + 1 < RING ? slot + 1 : 0;
        cslot = cslot + 1 < 3 ? cslot + 1 : 0;
        if constexpr (LEAD == 0) lds_barrier();
        // dDelta = P^T dO + kap (K dH')
        f32x4 x = zero4();
#pragma unroll
        for (int s0 = 0; s0 < KS; s0 += 2) {
          Operand<T, 1> kr[2];
          Operand<T, NT> st[2];
#pragma unroll
          for (int s = 0; s < 2 && s0 + s < KS; ++s) {
            kr[s] = Keys::row(keys, 16 * w + c, 32 * (s0 + s) + 8 * grp);
            st[s] = F::get(lds.state, s0 + s);
          }
          __builtin_amdgcn_sched_barrier(0);  // reads together, not one by one before its product
#pragma unroll
          for (int s = 0; s < 2 && s0 + s < KS; ++s) x = mma(kr[s], st[s], x);
        }
        const f32x4 kap = *reinterpret_cast<const f32x4*>(co + 2 * kChunk + own);
        const f32x4 z = *reinterpret_cast<const f32x4*>(lds.z + 256 * w + 4 * lane);
        const Record rh = record(rec_dh, chunk0 + ci, slices * slices);
#pragma unroll
        for (int i = 0; i < FT; ++i)
          if (w + 4 * i < slices) rh.put(sl * slices + w + 4 * i, dh[i]);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = kap[r] * x[r] + z[r];
        F::template put_tile<false>(lds.ddelta, w, x);
        lds_barrier();
        // dR = T^T dDelta; the next chunk's T, K^T and Q^T (eps dO) on the way
        Operand<T, NT> d0;
        if constexpr (BOTH) d0 = F::get(lds.ddelta, 0);
        const Operand<T, NT> d1 = F::get(lds.ddelta, 1);
        __builtin_amdgcn_sched_barrier(0);
        load(it + 1, next);
        f32x4 dr = mma(tin.t[1], d1, zero4());
        if constexpr (BOTH) dr = mma(tin.t[0], d0, dr);
        const f32x4 beta = *reinterpret_cast<const f32x4*>(co + own);
        const f32x4 eps = *reinterpret_cast<const f32x4*>(co + kChunk + own);
        const float gam = co[2 * kChunk - 1];
        constexpr int AHEAD = FT < 2 ? FT : 2;  // feature tiles whose K^T waits in registers
        Operand<T, 1> kc[AHEAD][2];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
#pragma unroll
          for (int s = 0; s < 2; ++s) kc[i][s] = Keys::columns(keys, s, 16 * (TILES < 4 ? w & 1 : w + 4 * i));
#pragma unroll
        for (int i = 0; i < FT; ++i)
          if (w + 4 * i < TILES) {
            const f32x4 add = *reinterpret_cast<const f32x4*>(lds.qdo + 256 * (w + 4 * i) + 4 * lane);
#pragma unroll
            for (int r = 0; r < 4; ++r) dh[i][r] = gam * dh[i][r] + add[r];
          }
        f32x4 y;
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] = -(beta[r] * dr[r] * eps[r]);
        F::template put_tile<false>(lds.dread, w, y);
        record(rec_dr, chunk0 + ci, 4 * slices).put(4 * sl + w, dr);
        lds_barrier();
        // dH = gam dH' + Q^T (eps dO) - K^T (beta eps dR)
        const Operand<T, NT> y0 = F::get(lds.dread, 0), y1 = F::get(lds.dread, 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < FT; ++i) {
          const int ft = w + 4 * i;
          if (ft < TILES) {
            if (i >= AHEAD) {
              dh[i] = mma(Keys::columns(keys, 0, 16 * ft), y0, dh[i]);
              dh[i] = mma(Keys::columns(keys, 1, 16 * ft), y1, dh[i]);
            } else {
              dh[i] = mma(kc[i < AHEAD ? i : 0][0], y0, dh[i]);
              dh[i] = mma(kc[i < AHEAD ? i : 0][1], y1, dh[i]);
            }
            F::template put_tile<true>(lds.state, ft, dh[i]);
          }
        }
        lds_barrier();
      };
      for (int it = 0; it < nc; it += 2) {
        step(it, ta, tb);
        if (it + 1 < nc) step(it + 1, tb, ta);
      }
    };
    if (w < 2) run(std::true_type{});
    else run(std::false_type{});
    float* so = d_state_in + (size_t)bh * D * D;
#pragma unroll
    for (int i = 0; i < FT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int f = 16 * (w + 4 * i) + 4 * grp + r;
        if (f < D && vcol < D) so[(size_t)f * D + vcol] = dh[i][r];
      }
  } else {
    // ---- memory into LDS ahead, and of the next chunk P^T dO (the 16 tokens w) and Q^T (eps dO) (each fourth feature tile).
    //      Chunk number it counts from the last one back; past the first it stays, so that nothing is conditional. In
    //      chunk it's three spans: dO of chunk it + 1 into registers, loads of the queries of it + 2 and the keys of
    //      it + LEAD; P^T dO, loads of the coefficients of it + 2 and dO of it + 3; Q^T (eps dO), loads of this wave's
    //      columns of P of it + 2. Every wave issues the same number of direct loads in the same order, so that the wait
    //      for the last chunk's leaves this one's in flight; the loads are spread, for a CU takes 64 bytes a cycle ----
    const size_t stride = (size_t)kChunk * dims.H * D;
    const T *kp = k + dims.at(b, 0, h), *qp = q + dims.at(b, 0, h), *gp = d_o + dims.at(b, 0, h);
    const T* pp = pf + chunk0 * Factor<T, NT>::kElems + col_step(w, 0) * F::kStep;
    const float* cp = coef + chunk0 * kCoefAll;
    auto chunk_of = [&](int it) { return it < nc ? nc - 1 - it : 0; };
    auto stage = [&](int it, int slot) {
      const int ci = chunk_of(it);
      const Rows<T> rows = dims.rows_at(kp + ci * stride, ci);
#pragma unroll
      for (int j = 0; j < Keys::kInstr / 4; ++j) Keys::stage(lds.keys[slot], rows, 4 * j + w, 0);
    };
    // `slot` as a constant: the reads of one slot then do not wait for the loads into the other
    auto stage_q = [&](int it, auto slot) {
      if constexpr (S::kStageQ) {
        const int ci = chunk_of(it);
        const Rows<T> rows = dims.rows_at(qp + ci * stride, ci);
#pragma unroll
        for (int j = 0; j < Keys::kInstr / 4; ++j) Keys::stage(lds.queries[decltype(slot)::value % QRING], rows, 4 * j + w, 0);
      }
    };
    auto stage_do = [&](int it, auto slot, int coef_it, int coef_slot) {  // and the coefficients of chunk coef_it
      const int ci = chunk_of(it);
      const Rows<T> rows = dims.rows_at(gp + ci * stride, ci);
      T* to = lds.d_o[decltype(slot)::value];
      const float* co = cp + (size_t)chunk_of(coef_it) * kCoefAll;
      if constexpr (Slice::kInstr == 4) {
        Slice::stage(to, rows, w, 16 * sl);
        stage_coef(lds.coef[coef_slot], co);
      } else {
        if (w < 2) Slice::stage(to, rows, w, 16 * sl);
        else stage_coef(lds.coef[coef_slot], co);
      }
    };
    auto run = [&](auto both) {  // as in the chain
      constexpr bool BOTH = decltype(both)::value;
      auto load = [&](int it, BackIn<T>& in) {
        const int ci = chunk_of(it);
        const T* pb = pp + (size_t)ci * Factor<T, NT>::kElems;
        if constexpr (BOTH) in.pf[0] = F::get(pb, 0);
        in.pf[1] = F::get(pb, BOTH ? 1 : 0);
        in.on = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(dims.flags(active, b, ci * kChunk), lane, 0, 0);
      };
      f32x4 x[4];  // dO as accumulator tiles (rows tokens), zero where inactive
      auto read_do = [&](const BackIn<T>& in, auto slot) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = Slice::four(lds.d_o[decltype(slot)::value], j, 0);
        if (active != nullptr) {
          const uint64_t on = __builtin_amdgcn_ballot_w64(in.on != 0) >> (4 * grp);
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) x[j][r] = (on >> (16 * j + r)) & 1 ? x[j][r] : 0.f;
        }
      };
      auto form_z = [&](const BackIn<T>& in) {
        f32x4 z = mma(in.pf[1], paired<T, 1>(x[2], x[3]), zero4());
        if constexpr (BOTH) z = mma(in.pf[0], paired<T, 1>(x[0], x[1]), z);
        *reinterpret_cast<f32x4*>(lds.z + 256 * w + 4 * lane) = z;
      };
      auto form_qdo = [&](int it, auto slot, const float* co) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f32x4 eps = *reinterpret_cast<const f32x4*>(co + kChunk + 16 * j + 4 * grp);
#pragma unroll
          for (int r = 0; r < 4; ++r) x[j][r] *= eps[r];
        }
        const Operand<T, NT> e0 = paired<T, NT>(x[0], x[1]), e1 = paired<T, NT>(x[2], x[3]);
#pragma unroll
        for (int i = 0; i < FT; ++i) {
          const int ft = w + 4 * i;
          if (ft < TILES) {
            f32x4 y;
            if constexpr (S::kStageQ) {
              y = mma(Keys::columns(lds.queries[decltype(slot)::value % QRING], 0, 16 * ft), e0, zero4());
              y = mma(Keys::columns(lds.queries[decltype(slot)::value % QRING], 1, 16 * ft), e1, y);
            } else {
              const int ci = chunk_of(it);
              const Rows<T> rows = dims.rows_at(qp + ci * stride, ci);
              Operand<T, 1> qc[2];
#pragma unroll
              for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  qc[s].lo[e] = rows.one(32 * s + 4 * grp + e, 16 * ft + c);
                  qc[s].hi[e] = rows.one(32 * s + 16 + 4 * grp + e, 16 * ft + c);
                }
              y = mma(qc[0], e0, zero4());
              y = mma(qc[1], e1, y);
            }
            *reinterpret_cast<f32x4*>(lds.qdo + 256 * ft + 4 * lane) = y;
          }
        }
      };
      constexpr std::integral_constant<int, 0> even{};
      constexpr std::integral_constant<int, 1> odd{};
      BackIn<T> in;
      int free = LEAD, c1 = 1, c2 = 2;  // the slots of the keys of chunk it + LEAD, of the coefficients of it + 1 and it + 2
      auto step = [&](int it, auto mine, auto other) {  // `mine` is it's parity
        if constexpr (LEAD == 0) {
          stage(it, 0);
          stage_q(it + 1, other);
          stage_do(it + 2, mine, it + 2, c2);
          direct_loads_done();
          lds_barrier();
        }
        read_do(in, other);
        if constexpr (LEAD > 0) {
          stage_q(it + 2, mine);
          stage(it + LEAD, free);
        }
        lds_barrier();
        if constexpr (LEAD > 0) stage_do(it + 3, other, it + 2, c2);
        form_z(in);
        direct_loads_done<LEAD == 0 ? 0 : S::kLoads>();
        lds_barrier();
        load(it + 2, in);
        form_qdo(it + 1, other, lds.coef[c1]);
        free = free + 1 < RING ? free + 1 : 0;
        c1 = c2;
        c2 = c2 + 1 < 3 ? c2 + 1 : 0;
        lds_barrier();
      };
#pragma unroll
      for (int it = 0; it < LEAD; ++it) stage(it, it);
      stage_q(0, even);
      stage_do(0, even, 0, 0);
      stage_do(1, odd, 1, 1);
      load(0, in);
      direct_loads_done();
      lds_barrier();
      read_do(in, even);
      form_z(in);
      load(1, in);
      form_qdo(0, even, lds.coef[0]);
      lds_barrier();
      if constexpr (LEAD > 0) {
        stage_q(1, odd);
        stage_do(2, even, 1, 1);
      }
      direct_loads_done();
      lds_barrier();
      for (int it = 0; it < nc; it += 2) {
        step(it, even, odd);
        if (it + 1 < nc) step(it + 1, odd, even);
      }
    };
    if (w < 2) run(std::true_type{});
    else run(std::false_type{});
  }
  direct_loads_done();
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

// The pieces' sums.
template <typename T, int NP> __device__ __forceinline__ void whole(const Operand<T, NP>& a, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if constexpr (sizeof(T) == 2) {
      x[e] = (float)a.p[NP - 1][e];
#pragma unroll
      for (int i = NP - 2; i >= 0; --i) x[e] += (float)a.p[i][e];
    } else {
      x[e] = e < 4 ? a.lo[e & 3] : a.hi[e & 3];
    }
  }
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

template <typename T>
__device__ __forceinline__ Operand<T, 1> eight(const T* p) {
  Operand<T, 1> x;
  if constexpr (sizeof(T) == 2) {
    x.p[0] = *reinterpret_cast<const bf16x8*>(p);
  } else {
    x.lo = reinterpret_cast<const f32x4*>(p)[0];
    x.hi = reinterpret_cast<const f32x4*>(p)[1];
  }
  return x;
}

template <typename T, int DP> struct GradShape {
  static constexpr int TILES = DP / 16;
  static constexpr int NT = Pieces<T>::kN;
  static constexpr int PAD = sizeof(T) == 2 ? 8 : 4;
  static constexpr int PITCH = DP + PAD;
  static constexpr int ITEMS = TILES < 4 ? 1 : TILES / 4;  // tiles a wave's of the states' records of 32 columns
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
      float pairs[2][kChunk][kChunk + 4];  // E dO.Delta (j <= i) and E dR.Delta (j < i), [i][j]
      Rows rows;
      f32x4 y[4][TILES][64];  // beta Y as accumulator tiles
    } u;
    float coef[kCoefAll];
    float ends[2][kChunk];          // of dg: each token's terms with the chunk's start, and with its end
    float across[4][kChunk];        // of dg: the terms of the pairs around token t whose first is of tile w, [w][t]
    float part[8];                  // each wave's share of <dH', H>
  };
};

// Bound by memory: 122 KB a chunk and head of width 64 (half of it the four records), B16 T1024 H12 d64 113 us for 375 MB (3.3
// TB/s), B2 T1500 H8 d128 39 us for 160 MB. With four waves for all it was 227 us (286 registers, one workgroup a CU), with
// eight 127, with the pairs' products formed once and no register spilled 107; the decays' gradients by the terms around
// each token, with Q K^T and K K^T of the lower tiles once more, take 6 of the 113 (2.5 of the 39, and 2 of the 10.7 of B32 T88
// H2 d16 in float32).
// Waves 0 to 3 hold dQ and Y of the 16 tokens w, waves 4 to 7 C. What comes from memory for the next 32 value columns is in
// flight while those in LDS are multiplied.
template <typename T, int DP>
__global__ __launch_bounds__(512, DP <= 64 ? 4 : 2) void gated_grad_kernel(
    const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, const float* __restrict__ g,
    const T* __restrict__ d_o, const float* __restrict__ coef, const float* __restrict__ rec_h,
    const float* __restrict__ rec_d, const float* __restrict__ rec_dh, const float* __restrict__ rec_dr,
    const uint8_t* __restrict__ active, T* __restrict__ dq, T* __restrict__ dk, T* __restrict__ dv, T* __restrict__ dbeta,
    float* __restrict__ dg, Dims<T> dims) {
  using S = GradShape<T, DP>;
  constexpr int NT = S::NT, TILES = S::TILES, ITEMS = S::ITEMS;
  __shared__ __attribute__((aligned(16))) typename S::Lds lds;
  const int id = xcd_logical_block(blockIdx.x, gridDim.x);
  const int chunk = id % dims.chunks, bh = id / dims.chunks, h = bh % dims.H, b = bh / dims.H;
  const int D = dims.D, t0 = chunk * kChunk;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & 3;
  const int l = threadIdx.x & 63, c = l & 15, grp = l >> 4, own = 16 * w + c;

  auto body = [&](auto kind) {
    constexpr bool first = decltype(kind)::value;
    // ---- sums over the value columns, 32 at a time ----
    // first: dQ^T and Y^T (rows features, columns the wave's tokens); else C^T, and dP and B (rows i, columns the wave's tokens
    // j <= i), which the others get by LDS, transposed
    f32x4 acc[TILES], ay[first ? TILES : 1], mp[4], mb[4];
#pragma unroll
    for (int i = 0; i < TILES; ++i) acc[i] = ay[first ? i : 0] = zero4();
#pragma unroll
    for (int i = 0; i < 4; ++i) mp[i] = mb[i] = zero4();
    float inner = 0.f, dot_v = 0.f;
    const int tiles = tiles_of(D);
    const unsigned state_bytes = (unsigned)(tiles * tiles) * 1024u, token_bytes = (unsigned)tiles * 4096u;
    const __amdgpu_buffer_rsrc_t rh = buffer_rsrc(rec_h + state_floats(id, D), state_bytes), rdh = buffer_rsrc(rec_dh + state_floats(id, D), state_bytes),
                                 rd = buffer_rsrc(rec_d + (size_t)id * tiles * 1024, token_bytes), rdr = buffer_rsrc(rec_dr + (size_t)id * tiles * 1024, token_bytes);
    const Rows<T> dorows = dims.rows(d_o, b, t0, h), vrows = dims.rows(v, b, t0, h);
    bool on[first ? 1 : 4];  // of the own token; of token 16 i + c
    {
      const __amdgpu_buffer_rsrc_t flags = dims.flags(active, b, t0);
#pragma unroll
      for (int i = 0; i < (first ? 1 : 4); ++i)
        on[i] = active == nullptr || (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(flags, first ? own : 16 * i + c, 0, 0) != 0;
    }
    if (threadIdx.x < kCoefAll / 4)
      reinterpret_cast<f32x4*>(lds.coef)[threadIdx.x] = reinterpret_cast<const f32x4*>(coef + (size_t)id * kCoefAll)[threadIdx.x];

    f32x4 xh[ITEMS], xdh[ITEMS], xd, xdr;  // records of the next value columns
    auto load16 = [](__amdgpu_buffer_rsrc_t r, unsigned at) { return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0)); };
    auto load = [&](int v0) {
#pragma unroll
      for (int n = 0; n < ITEMS; ++n) {
        const int tile = wave + 8 * n, ft = tile % TILES, half = tile / TILES;
        const unsigned at = half < 2 && ft < tiles ? (unsigned)(64 * ((v0 / 16 + half) * tiles + ft) + l) * 16u : kNowhere;
        xh[n] = load16(rh, at);
        xdh[n] = load16(rdh, at);
      }
      const unsigned at = (unsigned)(64 * (4 * (v0 / 16) + wave) + l) * 16u;
      xd = load16(rd, at);
      xdr = load16(rdr, at);
    };
    load(0);
    const float beta_own = coef[(size_t)id * kCoefAll + own];
    const Rows<T> dvrows = dims.rows(dv, b, t0, h);
    for (int v0 = 0; v0 < D; v0 += 32) {
      const int vc = v0 + 8 * grp;
      Operand<T, 1> dof[4];  // dO of all tokens; first: dO and V of its own
      if constexpr (first) {
        dof[0] = dorows.row(own, on[0] ? vc : D);
        dof[1] = vrows.row(own, vc);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) dof[i] = dorows.row(16 * i + c, on[first ? 0 : i] ? vc : D);
      }
#pragma unroll
      for (int n = 0; n < ITEMS; ++n) {
        const int tile = wave + 8 * n, ft = tile % TILES, half = tile / TILES;
        inner += (xh[n][0] * xdh[n][0] + xh[n][1] * xdh[n][1]) + (xh[n][2] * xdh[n][2] + xh[n][3] * xdh[n][3]);
        if (2 * TILES % 8 == 0 || half < 2) {
          lds.u.values.h.put(16 * half + c, 16 * ft + 4 * grp, xh[n]);
          lds.u.values.dh.put(16 * half + c, 16 * ft + 4 * grp, xdh[n]);
        }
      }
      lds.u.values.delta.put(16 * (wave / 4) + c, 16 * w + 4 * grp, xd);
      lds.u.values.dr.put(16 * (wave / 4) + c, 16 * w + 4 * grp, xdr);
      lds_barrier();
      load(v0 + 32);  // past the width: zeros
      if constexpr (first) {
        const Operand<T, NT> dr_w = lds.u.values.dr.columns(16 * w);
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
          const Operand<T, NT> x = lds.u.values.h.columns(16 * i);
          acc[i] = mma(x, dof[0], acc[i]);
          ay[i] = mma(x, dr_w, ay[i]);
        }
        float dr8[8], v8[8];  // dV = beta dR
        whole<T, NT>(dr_w, dr8);
        whole<T, 1>(dof[1], v8);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          dot_v += dr8[e] * v8[e];
          dr8[e] *= beta_own;
        }
        dvrows.put_eight(own, vc, dr8);
      } else {
        const Operand<T, NT> del_w = lds.u.values.delta.columns(16 * w);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i >= w) {
            mp[i] = mma(dof[i], del_w, mp[i]);
            mb[i] = mma(lds.u.values.dr.columns(16 * i), del_w, mb[i]);
          }
#pragma unroll
        for (int i = 0; i < TILES; ++i) acc[i] = mma(lds.u.values.dh.columns(16 * i), del_w, acc[i]);
      }
      lds_barrier();
    }

    // ---- the keys and queries, the decays between pairs, sums over the chunk's tokens ----
    constexpr int PIECES = kChunk * (DP / 8), KQ = (PIECES + 511) / 512;
    Operand<T, 1> kx[KQ], qx[KQ];
    {
      const Rows<T> krows = dims.rows(k, b, t0, h), qrows = dims.rows(q, b, t0, h);
#pragma unroll
      for (int n = 0; n < KQ; ++n) {
        const int p = threadIdx.x + 512 * n, row = p / (DP / 8), f = 8 * (p % (DP / 8));
        kx[n] = krows.row(row, row < kChunk ? f : D);
        qx[n] = qrows.row(row, row < kChunk ? f : D);
      }
    }
    if constexpr (!first) {
      const DecaySum sum_own = {lds.coef[kCoef + own], lds.coef[kCoef + kChunk + own]};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i >= w) {
          const float* co = lds.coef + 16 * i + 4 * grp;
          const f32x4 beta = *reinterpret_cast<const f32x4*>(co), hi = *reinterpret_cast<const f32x4*>(co + kCoef),
                      lo = *reinterpret_cast<const f32x4*>(co + kCoef + kChunk);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int row = 16 * i + 4 * grp + r;
            const float e = decay({hi[r], lo[r]}, sum_own);
            mp[i][r] *= row >= own ? e : 0.f;
            mb[i][r] *= row > own ? e : 0.f;
            lds.u.pairs[0][row][own] = mp[i][r];
            lds.u.pairs[1][row][own] = mb[i][r];
            mb[i][r] *= -beta[r];
          }
        }
    }
    const float scale = lds.coef[(first ? kChunk : 2 * kChunk) + own];  // eps, kap
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        acc[i][r] *= scale;
        if constexpr (first) ay[i][r] *= scale;
      }
    lds_barrier();
    if constexpr (first) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i <= w) {
          mp[i] = *reinterpret_cast<const f32x4*>(&lds.u.pairs[0][own][16 * i + 4 * grp]);
          mb[i] = *reinterpret_cast<const f32x4*>(&lds.u.pairs[1][own][16 * i + 4 * grp]);
        }
    }
    lds_barrier();
#pragma unroll
    for (int n = 0; n < KQ; ++n) {
      const int p = threadIdx.x + 512 * n, row = p / (DP / 8), f = 8 * (p % (DP / 8));
      if (PIECES % 512 == 0 || row < kChunk) {
        T *kd = lds.u.rows.keys + row * S::PITCH + f, *qd = lds.u.rows.queries + row * S::PITCH + f;
        if constexpr (sizeof(T) == 2) {
          *reinterpret_cast<bf16x8*>(kd) = kx[n].p[0];
          *reinterpret_cast<bf16x8*>(qd) = qx[n].p[0];
        } else {
          reinterpret_cast<f32x4*>(kd)[0] = kx[n].lo;
          reinterpret_cast<f32x4*>(kd)[1] = kx[n].hi;
          reinterpret_cast<f32x4*>(qd)[0] = qx[n].lo;
          reinterpret_cast<f32x4*>(qd)[1] = qx[n].hi;
        }
      }
    }
    lds_barrier();
    const T *keys_own = lds.u.rows.keys + own * S::PITCH + 4 * grp, *queries_own = lds.u.rows.queries + own * S::PITCH + 4 * grp;
    float end = 0.f;  // eps_i (q_i.(H dO_i) - beta_i k_i.(H dR_i)), or kap_j k_j.(dH' Delta_j)
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      const f32x4 kf = four(keys_own + 16 * i), qf = first ? four(queries_own + 16 * i) : kf;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        end += qf[r] * acc[i][r];
        if constexpr (first) end -= beta_own * (kf[r] * ay[i][r]);
      }
    }
    end = sum_over_rows(end);
    if (grp == 0) lds.ends[first ? 0 : 1][own] = end;
    if constexpr (!first) {
      // the pairs' terms, rows i, columns j: down each column the sums over i >= t, then over the columns j < t
      float below = 0.f;  // of the tiles below
#pragma unroll
      for (int i = 3; i >= 0; --i)
        if (i >= w) {
          f32x4 qk = zero4(), kk = zero4();
#pragma unroll
          for (int s = 0; s < DP / 32; ++s) {
            const int f = 32 * s + 8 * grp;
            const Operand<T, 1> kj = eight(lds.u.rows.keys + own * S::PITCH + f);
            qk = mma(eight(lds.u.rows.queries + (16 * i + c) * S::PITCH + f), kj, qk);
            kk = mma(eight(lds.u.rows.keys + (16 * i + c) * S::PITCH + f), kj, kk);
          }
          f32x4 x;
#pragma unroll
          for (int r = 3; r >= 0; --r) {
            x[r] = mp[i][r] * qk[r] + mb[i][r] * kk[r];
            if (r < 3) x[r] += x[r + 1];
          }
          // x[0] of the rows' groups behind this one
          const auto p16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(x[0]), __float_as_uint(x[0]), false, false);
          const float odd = __uint_as_float(p16[1]), both = __uint_as_float(p16[0]) + odd;
          const auto p32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(both), __float_as_uint(both), false, false);
          const float upper = __uint_as_float(p32[1]);
          const float behind = ((grp & 1) == 0 ? odd : 0.f) + (grp < 2 ? upper : 0.f) + below;
          below += __uint_as_float(p32[0]) + upper;
#pragma unroll
          for (int r = 0; r < 4; ++r) x[r] = group_sum<16>(i > w || 4 * grp + r > c ? x[r] + behind : 0.f);
          if (c == 0) *reinterpret_cast<f32x4*>(&lds.across[w][16 * i + 4 * grp]) = x;
        }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
      if (first ? 2 * s <= w : 2 * s + 1 >= w) {
        const Operand<T, NT> x = paired<T, NT>(mp[2 * s], mp[2 * s + 1]), y = paired<T, NT>(mb[2 * s], mb[2 * s + 1]);
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
          const Operand<T, 1> kc = load_columns_paired(lds.u.rows.keys, S::PITCH, s, 16 * i);
          if constexpr (first) {
            acc[i] = mma(kc, x, acc[i]);
            ay[i] = mma(kc, y, ay[i]);
          } else {
            acc[i] = mma(load_columns_paired(lds.u.rows.queries, S::PITCH, s, 16 * i), x, acc[i]);
            acc[i] = mma(kc, y, acc[i]);
          }
        }
      }

    // ---- out ----
    if constexpr (first) {
      float dot_y = 0.f;  // k.Y
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        const f32x4 kf = four(keys_own + 16 * i);
#pragma unroll
        for (int r = 0; r < 4; ++r) dot_y -= kf[r] * ay[i][r];
      }
      dot_y = sum_over_rows(dot_y);
      dot_v = sum_over_rows(dot_v);
      if (grp == 0 && t0 + own < dims.N) dbeta[((size_t)b * dims.N + t0 + own) * dims.H + h] = from_f32<T>(dot_v + dot_y);
    }
    inner = group_sum<64>(inner);
    if (l == 0) lds.part[wave] = inner;
    lds_barrier();
    if constexpr (first) {  // dK = beta Y + C
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        f32x4 y;
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] = -(beta_own * ay[i][r]);
        lds.u.y[w][i][l] = y;
      }
    }
    lds_barrier();
    const Rows<T> rows = dims.rows(first ? dq : dk, b, t0, h);
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      if constexpr (!first) {
        const f32x4 y = lds.u.y[w][i][l];
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][r] += y[r];
      }
      rows.put_four(own, 16 * i + 4 * grp, acc[i]);
    }
  };
  if (wave < 4) body(std::true_type{});
  else body(std::false_type{});
  if (wave == 0) {
    const size_t at = ((size_t)b * dims.N + (t0 + l < dims.N ? t0 + l : t0)) * dims.H + h;
    const float gl = g[at];
    float from = lds.ends[0][l], to = l > 0 ? lds.ends[1][l - 1] : 0.f;  // the sums from this token on, and before it
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const float down = __shfl_down(from, off), up = __shfl_up(to, off);
      if (l + off < 64) from += down;
      if (l >= off) to += up;
    }
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) x += lds.part[i];
    x = lds.coef[2 * kChunk - 1] * x + from + to;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (16 * i <= l) x += lds.across[i][l];
    // what forgets the state has no gradient
    if (t0 + l < dims.N) dg[at] = (double)gl < kLeastDecay ? 0.f : x;
  }
}

size_t align16(size_t x) { return (x + 15) & ~(size_t)15; }

// coefficients, T and P by columns, then dH' and dR of every chunk and head
template <typename T> size_t factor_bytes(size_t total) {
  return align16(total * kCoefAll * sizeof(float)) + 2 * total * sizeof(T) * Factor<T, Pieces<T>::kN>::kElems;
}
template <typename T> size_t backward_bytes(size_t total, int D) { return factor_bytes<T>(total) + record_bytes(total, D); }

template <typename T, int DP>
void launch_back(const T* q, const T* k, const T* v, const float* g, const T* d_o, const float* d_state,
                 const uint8_t* active, const float* rec_h, const float* rec_d, const float* coef, const T* tf,
                 const T* pf, float* rec_dh, float* rec_dr, T* dq, T* dk, T* dv, T* dbeta, float* dg, float* d_state_in,
                 Dims<T> dims, int B, hipStream_t stream) {
  const int slices = (dims.D + 15) / 16;
  hipLaunchKernelGGL((gated_chain_backward_kernel<T, DP>), dim3((unsigned)(B * dims.H * slices)), dim3(512), 0, stream, q, k, d_o,
                     coef, tf, pf, d_state, d_state_in, active, rec_dh, rec_dr, dims, slices);
  hipLaunchKernelGGL((gated_grad_kernel<T, DP>), dim3((unsigned)(B * dims.H * dims.chunks)), dim3(512), 0, stream, q, k, v, g,
                     d_o, coef, rec_h, rec_d, rec_dh, rec_dr, active, dq, dk, dv, dbeta, dg, dims);
}

template <typename T>
int scan_backward(const void* q_, const void* k_, const void* v_, const void* beta_, const float* g,
                  const float* records, size_t records_bytes, const void* d_o_, const float* d_state,
                  const uint8_t* active, void* dq_, void* dk_, void* dv_, void* dbeta_, float* dg, float* d_state_in,
                  void* ws, size_t ws_bytes, int B, int N, int H, int D, hipStream_t stream, const char* who) {
  if (const int st = check_sizes(B, N, H, D, true, who); st != OK) return st;
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
  T* tf = reinterpret_cast<T*>(static_cast<char*>(ws) + align16(total * kCoefAll * sizeof(float)));
  T* pf = tf + total * Factor<T, Pieces<T>::kN>::kElems;
  float* rec_dh = reinterpret_cast<float*>(static_cast<char*>(ws) + factor_bytes<T>(total));
  float* rec_dr = rec_dh + state_floats(total, D);
  const float* rec_d = records + state_floats(total, D);
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
