// The looped column's projections in 8-bit integers on CDNA4 (gfx950): every block of a pass's stacked
// weight in one launch, with a scale for each token and each output channel.
//
//   y_j[m, c] = (sum_k z[m, k] w_j[c, k]) (a_m b_jc),  int32 sums (exact: at most 16384 * 127^2 < 2^31),
//
// z [M, d] int8 with scales a (norm_int8.hip), the weights stacked and transposed as the bf16
// projection's (project.hip; vesper/column.py:192-260, vesper/attention.py:269-292), [p, cols, d] int8 with
// scales b [p, cols]. The product of the two scales is rounded to float32, the sum is converted to it, and
// their product is rounded once more to the output's type; the write strength's block may pass through
// the logistic function first.
//
// Two kernels, by the number of tokens:
//
// tile (many tokens): 256 tokens x 256 columns, eight waves of 64 x 128, both operands through LDS in two stages of
// 128 inputs (whole cache lines a row), by a workgroup a CU that goes from tile to tile; or, where that makes few
// workgroups, 128 x 128 or 128 x 64 in waves of 64 x 32 and three stages. global_load_lds_dwordx4 moves eight rows of 128 bytes an
// instruction, each row's 16-byte segments XOR-swizzled so that the fragment reads meet each bank once; 16x16x64 int8
// MFMA formed transposed (weight rows as the A operand); the second half's fragments are read during the first half's
// products. 8192^3: 412 to 473 us among other work, 520 to 540 back to back (2.0 to 2.7 Pop/s; the clock falls under
// them: the matrix units are busy 69 % of the cycles), a library product of the same operands 547. 32767 x 768 to 2316
// columns: 72 us (116 Gop, 1.6 Pop/s). One tile a workgroup needed 96: its first loads and its outputs stood alone, and
// the logistic function, chosen an output at a time, ran for all of them (86 with that block's outputs apart; 78 from
// tile to tile; 72 with the next tile's second stage loading under the outputs too). Stages of 64 inputs, four deep,
// read half cache lines (117 when the present form took 94); three stages of 256 x 128: 108; outputs stored straight
// from the accumulators, 32 bytes a row: 95 to 107.
//
// few (up to 64 tokens, a decode step): bound by reading the weights once. A workgroup takes 16 columns and
// all the tokens; its waves share the inputs, each reading whole 128-byte lines of 16 weight rows straight
// into the MFMA operand's registers; the waves' int32 sums are joined through LDS. Past 16 tokens the tokens'
// own reads count (from L2, by every workgroup): 32 columns a workgroup where there are enough (64 tokens, 8192 to
// 8192: 40 us with 16 columns, 31 with 32, now 26; 64 x 512 to 1544: 4.0 and 4.7), and eight waves in place of four
// (64 x 512: 4.5 -> 4.0; with up to 16 tokens four are as good or better: 16 x 8192 to 8192 16.7 us, 4.0 TB/s of
// weights, against 17.8; two or four steps' loads in flight a wave gave nothing).
#include <type_traits>

#include "common.h"
#include "vesper_kernels.h"

namespace vsp {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kMaxBlocks = 4;
constexpr int kBK = 128;  // inputs a stage
constexpr int kBand = 4;       // row tiles of a band (an XCD's workgroups go down its rows before the next column)
constexpr int kFewTokens = 64; // its most tokens

struct Blocks {
  int nblk;
  int used[kMaxBlocks];       // columns written per block
  int start[kMaxBlocks + 1];  // first column tile of each block
  void* out[kMaxBlocks];      // [M, used] per block
};

struct Args {
  const int8_t* z;
  const float* z_scale;
  const int8_t* wt;
  const float* w_scale;
  int M, d, cols, sig_block;
};

// An output: the sum times both scales, through the logistic function where asked. That is formed with the
// exponential and reciprocal instructions (each within a unit of float32; the exponent's own rounding moves a result
// far below 1 by a relative |y| 2^-23, in float32 outputs too): a thread of the tiles has 32 or 128 outputs, and as
// calls of the library's functions their code outgrew the instruction cache (32767 tokens of 768: 104 us with
// it, 90 without a logistic block).
template <typename T, bool SIG>
__device__ __forceinline__ T finish(int sum, float scale) {
  float y = (float)sum * scale;
  if constexpr (SIG) y = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * y));
  return from_f32<T>(y);
}

__device__ __forceinline__ int block_of(const Blocks& blk, int tile) {
  int nb = 0;
#pragma unroll
  for (int j = 1; j < kMaxBlocks; ++j)
    if (j < blk.nblk && tile >= blk.start[j]) nb = j;
  return nb;
}

// 16 bytes from a buffer (zeros past its range).
__device__ __forceinline__ i32x4 load16(__amdgpu_buffer_rsrc_t r, unsigned off) {
  return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0));
}

// A resource over `rows` rows of d bytes from `base`, in scalar registers: its parts are the same in every lane, but
// the compiler, which formed them from a division, would otherwise run a loop over the lanes for each load.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const int8_t* base, int rows, int d) {
  const uint64_t p = reinterpret_cast<uint64_t>(base);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)p);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(p >> 32));
  const int bytes = __builtin_amdgcn_readfirstlane(rows * d);
  return buffer_rsrc(reinterpret_cast<const int8_t*>((uint64_t)lo | ((uint64_t)hi << 32)), (unsigned)bytes);
}

constexpr unsigned kOutside = 0x80000000u;  // an offset past every resource's range (under 2 GiB)

// The wave's loads but the N newest have arrived in LDS, its LDS reads have returned, and every wave is here.
template <int N>
__device__ __forceinline__ void arrive() {
#if defined(__HIP_DEVICE_COMPILE__)
  // the wait as the builtin, which the compiler's own count of loads takes note of (behind inline assembly it would
  // wait again, for all but the newest loads, before the first read of a stage)
  static_assert(N < 64, "vmcnt has six bits");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | ((N >> 4) << 14));  // vmcnt(N), lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#endif
}

// A wave's tile of sums out: tokens m0 .. and columns c0 .. of block nb, with their scales, which lie in `lds` from
// `zscale` and `wscale` on. Lane (lq, g) holds columns 16 j + 4 g + r of token 16 i + lq. Outputs of 16 bits go through
// LDS (from `room` on, the wave's own), 16 tokens by 64 columns (or the tile's fewer) at a time, so that whole cache
// lines leave; row r's 16-byte segment s is at s ^ (r % the row's segments). Returns how many stores the wave has made
// for certain: tile_stores, or 0 where some may have had nothing to store (or, in float32, are not counted).
template <typename T, int TM, int TN>
constexpr int tile_stores() {
  return sizeof(T) == 2 ? TM * (TN * 16 * 16) / (64 * 8) : 0;  // 64 lanes of eight outputs a store
}
template <typename T, int TM, int TN>
__device__ __forceinline__ int store_tile(const i32x4 (&acc)[TN][TM], const Args& a, const Blocks& blk, int nb, int m0,
                                          int c0, int8_t* lds, int zscale, int wscale, int room) {
  typedef T V4 __attribute__((ext_vector_type(4)));
  typedef T V8 __attribute__((ext_vector_type(8)));
  int l = threadIdx.x & 63;
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" : "+v"(l));  // formed anew for each tile: kept in registers over the products, addresses would spill
#endif
  const int lq = l & 15, g = l >> 4, used = blk.used[nb];
  T* out = static_cast<T*>(blk.out[nb]);
  auto put = [&](auto sig, auto all) {
    constexpr bool SIG = decltype(sig)::value, full = decltype(all)::value;
    if constexpr (sizeof(T) == 2) {
      // TC column tiles a pass: 16-byte segments a row, rows an instruction
      constexpr int TC = TN < 4 ? TN : 4, SEG = 2 * TC, EACH = 64 / SEG;
      static_assert(TM * (TN / TC) * (16 / EACH) == tile_stores<T, TM, TN>(), "a store for each turn of the loops");
      const int seg = l % SEG, r0 = l / SEG;
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const float zs = *reinterpret_cast<const float*>(lds + (zscale + 64 * i + 4 * lq));
#pragma unroll
        for (int j0 = 0; j0 < TN; j0 += TC) {
#pragma unroll
          for (int j = 0; j < TC; ++j) {
            const int c = 16 * j + 4 * g;
            const f32x4 bs = *reinterpret_cast<const f32x4*>(lds + (wscale + 64 * j0 + 4 * c));
            V4 y;
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = finish<T, SIG>(acc[j0 + j][i][r], zs * bs[r]);
            *reinterpret_cast<V4*>(lds + (room + 32 * TC * lq + 16 * ((c >> 3) ^ (lq & (SEG - 1))) + 2 * (c & 7))) = y;
          }
          __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the rows are in LDS
#pragma unroll
          for (int it = 0; it < 16 / EACH; ++it) {
            const int r = EACH * it + r0, m = m0 + 16 * i + r, col = c0 + 16 * j0 + 8 * seg;
            if (!full && (m >= a.M || col >= used)) continue;
            const V8 v = *reinterpret_cast<const V8*>(lds + (room + 32 * TC * r + 16 * (seg ^ (r & (SEG - 1)))));
            T* orow = out + (size_t)m * used + col;
            if (full || (used & 7) == 0) {
              *reinterpret_cast<V8*>(orow) = v;
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (col + e < used) orow[e] = v[e];
            }
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int m = m0 + 16 * i + lq;
        if (m >= a.M) continue;
        const float zs = *reinterpret_cast<const float*>(lds + (zscale + 64 * i + 4 * lq));
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const int col = c0 + 16 * j + 4 * g;
          const f32x4 bs = *reinterpret_cast<const f32x4*>(lds + (wscale + 64 * j + 16 * g));
          float y[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) y[r] = finish<T, SIG>(acc[j][i][r], zs * bs[r]);
          T* orow = out + (size_t)m * used + col;
          if ((used & 3) == 0 && col < used) {
            *reinterpret_cast<float4*>(orow) = make_float4(y[0], y[1], y[2], y[3]);
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (col + r < used) orow[r] = y[r];
          }
        }
      }
    }
  };
  // the logistic block's outputs apart: as a choice an output, its instructions run for all (32767 tokens of 768: 96 us
  // and 86); and a whole tile without a test an output
  if (nb == a.sig_block) {
    put(std::true_type{}, std::false_type{});
    return 0;
  }
  if ((used & 7) == 0 && m0 <= a.M - 16 * TM && c0 <= used - 16 * TN) {  // (sums here could pass 2^31)
    put(std::false_type{}, std::true_type{});
    return tile_stores<T, TM, TN>();
  }
  put(std::false_type{}, std::false_type{});
  return 0;
}

// The products of one stage of 128 inputs: TM x TN tiles from a wave's rows of both operands in LDS. Row r's 16-byte
// segment s is at s ^ 2 ((r >> 1) & 3), so that a fragment read (lanes 0-7 with 16-23: rows 0-7, two segments each)
// meets every bank once.
__device__ __forceinline__ int swizzle(int row) { return 2 * ((row >> 1) & 3); }
template <int TM, int TN>
__device__ __forceinline__ void stage_products(const int8_t* sz, const int8_t* sw, int zrow, int wrow,
                                               i32x4 (&acc)[TN][TM]) {
  const int l = threadIdx.x & 63, lq = l & 15, g = l >> 4;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    i32x4 zf[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int row = zrow + 16 * i + lq;
      zf[i] = *reinterpret_cast<const i32x4*>(sz + row * kBK + 16 * ((4 * s + g) ^ swizzle(row)));
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int row = wrow + 16 * j + lq;
      const i32x4 f = *reinterpret_cast<const i32x4*>(sw + row * kBK + 16 * ((4 * s + g) ^ swizzle(row)));
#pragma unroll
      for (int i = 0; i < TM; ++i) acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f, zf[i], acc[j][i], 0, 0, 0);
    }
  }
}
// Their order, behind LOADS direct loads: the fragments of the second half are read while the first half's products
// run, and the wait for the loads stays behind the products.
template <int TM, int TN, int LOADS>
__device__ __forceinline__ void stage_order() {
  constexpr int AHEAD = TN < 4 ? TN : 4, EACH = (TM + 2 * TN - AHEAD + TN - 1) / TN;
  if constexpr (LOADS > 0) __builtin_amdgcn_sched_group_barrier(0x10, LOADS, 0);
  __builtin_amdgcn_sched_group_barrier(0x100, TM + AHEAD, 0);
#pragma unroll
  for (int u = 0; u < 2 * TN; ++u) {
    __builtin_amdgcn_sched_group_barrier(0x8, TM, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, EACH, 0);
  }
  __builtin_amdgcn_sched_barrier(0);
}

// Direct loads of stages into LDS by NW waves: instruction j of wave w fills rows 8 (w + NW j) .. + 7 of a stage, 128
// bytes each; lane l brings row l / 8's logical segment (l % 8) ^ swizzle(row).
template <int NL, int NW>
struct Loader {
  unsigned off[NL];  // the scalar offset holds the stage only: it stays below every resource's size
  int w, seg, d;
  __device__ __forceinline__ Loader(int w_, int l, int d_) : w(w_), d(d_) {
    const int row = l >> 3;
    seg = (l & 7) ^ swizzle(row);
#pragma unroll
    for (int j = 0; j < NL; ++j) off[j] = (unsigned)(8 * (w + NW * j) + row) * (unsigned)d + 16u * (unsigned)seg;
  }
  // inputs past d (a multiple of 16, so whole segments), and whole stages past the last, are zeros
  template <int ROWS>
  __device__ __forceinline__ void rows(__amdgpu_buffer_rsrc_t r, int st, int stages, int8_t* to) const {
    static_assert(ROWS % (8 * NW) == 0 && ROWS / (8 * NW) <= NL, "whole load instructions");
    const bool in = st * kBK + 16 * seg < d;
    const unsigned so = (unsigned)(min(st, stages - 1) * kBK);
#pragma unroll
    for (int j = 0; j < ROWS / (8 * NW); ++j) buffer_load_lds16(r, to + (w + NW * j) * 1024, in ? off[j] : kOutside, so);
  }
};

// A tile's place: its block, first row and first column; false past the last.
struct Place {
  int nb, m0, c0;
};
// Tiles are numbered in bands of kBand row tiles, down a band's rows before the next column tile: tiles of adjacent
// numbers share rows of z and columns of the weights in an XCD's L2.
template <int BM, int BN>
__device__ __forceinline__ bool place_of(const Blocks& blk, int tile, int ctiles, int mtiles, Place& p) {
  const int top = tile / (kBand * ctiles) * kBand, in_band = tile - top * ctiles, rows = min(kBand, mtiles - top);
  if (rows <= 0) return false;
  const int ct = in_band / rows;
  if (ct >= ctiles) return false;
  p.nb = block_of(blk, ct);
  p.m0 = (top + in_band - ct * rows) * BM;
  p.c0 = (ct - blk.start[p.nb]) * BN;
  return true;
}

// Tiles of 256 x 256, eight waves of 64 tokens x 128 columns, a workgroup a CU that takes tiles until none is left: the
// next tile's first two stages load under the last products and the outputs.
template <typename T>
__global__ __launch_bounds__(512, 1) void project_int8_kernel(const Args a, const Blocks blk, int ctiles, int mtiles,
                                                             int tiles) {
  constexpr int BM = 256, BN = 256, TM = 4, TN = 8, NL = 4;
  // Two stages of [rows][128 inputs] of each operand, as separate variables: the compiler tells the direct loads into
  // one from the reads of the other. It would wait for all of them at an access of a variable that none fills; so the
  // scales ([tile's parity][tokens, columns]: one is written while the last tile's is read) and the waves' room for
  // their outputs lie behind the first stage, whose loads have always arrived by then.
  constexpr int kScale = BM * kBK, kRoom = sizeof(T) == 2 ? 2048 : 0, kStores = tile_stores<T, TM, TN>();
  __shared__ __align__(16) int8_t sZ0[kScale + 4096 + 8 * kRoom], sZ1[BM * kBK];
  __shared__ __align__(16) int8_t sW0[BN * kBK], sW1[BN * kBK];

  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63;
  const int wm = w & 3, wn = w >> 2, d = a.d, stages = (d + kBK - 1) / kBK;
  // XCD x (workgroups x, x + 8, ..) takes the x-th eighth of the tiles, its workgroups adjacent ones at a time; the
  // grid is whole rounds over the 8 XCDs
  const int xcd = blockIdx.x & 7, lane_wg = blockIdx.x >> 3, each = gridDim.x >> 3, share = (tiles + 7) >> 3;
  int at = lane_wg;
  Place p{}, next{};
  auto place = [&](Place& q) {
    const bool more = at < share && place_of<BM, BN>(blk, xcd * share + at, ctiles, mtiles, q);
    at += each;
    return more;
  };
  if (!place(p)) return;

  const Loader<NL, 8> load(w, l, d);
  __amdgpu_buffer_rsrc_t rz, rw;  // of the rows of the tile being loaded: rows past the operands' ends read zeros
  auto aim = [&](const Place& q, bool more) {
    rz = rows_rsrc(a.z + (size_t)q.m0 * d, more ? min(BM, a.M - q.m0) : 0, d);
    rw = rows_rsrc(a.wt + ((size_t)q.nb * a.cols + q.c0) * d, more ? min(BN, a.cols - q.c0) : 0, d);
  };
  auto issue = [&](int st, int8_t* dz, int8_t* dw) {
    load.template rows<BM>(rz, st, stages, dz);
    load.template rows<BN>(rw, st, stages, dw);
  };
  // a thread's one of the tile's 512 scales
  const int si = threadIdx.x & 255;
  auto scale = [&](const Place& q) {
    return threadIdx.x < 256 ? a.z_scale[min(q.m0 + si, a.M - 1)]
                             : a.w_scale[(size_t)q.nb * a.cols + min(q.c0 + si, blk.used[q.nb] - 1)];
  };

  aim(p, true);
  issue(0, sZ0, sW0);
  float sc = scale(p);
  arrive<0>();
  issue(1, sZ1, sW1);
  int stores = 0;
  for (int parity = 0;; parity ^= 1) {
    *reinterpret_cast<float*>(sZ0 + (kScale + 2048 * parity + 4 * threadIdx.x)) = sc;
    const bool more = place(next);
    if (more) sc = scale(next);
    i32x4 acc[TN][TM];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int i = 0; i < TM; ++i) acc[j][i] = i32x4{0, 0, 0, 0};
    // Pairs of stages (the second of the last pair may be all zeros), the first one's loads arrived and the second's on
    // their way: the products of one, a barrier behind which the other has arrived and every wave is here, and the
    // loads into the buffers that were just read.
    int st = 0;
    do {  // there is always one: the compiler then knows that the scale has arrived with them
      stage_products<TM, TN>(sZ0, sW0, 64 * wm, 128 * wn, acc);
      stage_order<TM, TN, 0>();
      // the loads have arrived; the last tile's stores, issued behind them, may still be on their way (memory
      // operations retire in the order of their issue): 72 us in place of 74 for 32767 tokens of 768
      if (stores == kStores) arrive<kStores>();
      else arrive<0>();
      stores = 0;
      const bool last = st + 2 >= stages;
      if (last) aim(next, more);
      issue(last ? 0 : st + 2, sZ0, sW0);
      stage_products<TM, TN>(sZ1, sW1, 64 * wm, 128 * wn, acc);
      stage_order<TM, TN, 2 * NL>();
      arrive<0>();
      issue(last ? 1 : st + 3, sZ1, sW1);
      st += 2;
    } while (st < stages);
    __builtin_amdgcn_sched_barrier(0);  // the stores stay behind the loads
    if (p.c0 + 128 * wn < blk.used[p.nb])
      stores = store_tile<T, TM, TN>(acc, a, blk, p.nb, p.m0 + 64 * wm, p.c0 + 128 * wn, sZ0,
                                     kScale + 2048 * parity + 256 * wm, kScale + 2048 * parity + 1024 + 512 * wn,
                                     kScale + 4096 + kRoom * w);
    __builtin_amdgcn_sched_barrier(0);
    if (!more) {
      arrive<0>();  // the loads (zeros) have landed before the LDS is another workgroup's
      return;
    }
    p = next;
  }
}

// Tiles of 128 x 32 WN, 2 WN waves of 64 tokens x 32 columns, three stages in LDS: for the calls that have few tiles,
// each of which then waits for most of its loads. Bound by LDS (at 128 x 128 the fragments' reads take 768 cycles a stage
// and the loads' writes 256, the products 512), so with few of them narrower tiles on more CUs are faster.
template <typename T, int WN>
__global__ __launch_bounds__(128 * WN, WN == 4 ? 1 : 2) void project_int8_small_kernel(const Args a, const Blocks blk,
                                                                                     int ctiles, int mtiles) {
  constexpr int NW = 2 * WN, BM = 128, BN = 32 * WN, TM = 4, TN = 2, NL = BM / (8 * NW);
  constexpr int PER = NL + BN / (8 * NW);  // a wave's loads of a stage
  constexpr int kScale = BM * kBK;  // the tokens' and the columns' scales behind the first stage
  __shared__ __align__(16) int8_t sZ0[kScale + 4 * (BM + BN)], sZ1[BM * kBK], sZ2[BM * kBK];
  __shared__ __align__(16) int8_t sW0[BN * kBK], sW1[BN * kBK], sW2[BN * kBK];

  Place p{};  // the grid is padded to whole XCD rounds; whole workgroups leave
  if (!place_of<BM, BN>(blk, xcd_logical_block(blockIdx.x, gridDim.x), ctiles, mtiles, p)) return;
  const int used = blk.used[p.nb], d = a.d, stages = (d + kBK - 1) / kBK;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63;
  const int wm = w & 1, wn = w >> 1;

  const __amdgpu_buffer_rsrc_t rz = rows_rsrc(a.z + (size_t)p.m0 * d, min(BM, a.M - p.m0), d);
  const __amdgpu_buffer_rsrc_t rw = rows_rsrc(a.wt + ((size_t)p.nb * a.cols + p.c0) * d, min(BN, a.cols - p.c0), d);
  const Loader<NL, NW> load(w, l, d);
  auto issue = [&](int st, int8_t* dz, int8_t* dw) {
    load.template rows<BM>(rz, st, stages, dz);
    load.template rows<BN>(rw, st, stages, dw);
  };

  i32x4 acc[TN][TM];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int i = 0; i < TM; ++i) acc[j][i] = i32x4{0, 0, 0, 0};
  // A stage: the loads of the one two ahead, into the buffers that were read a stage ago (every wave has passed the
  // barrier behind those reads); the products; then the next stage has to have arrived. Every stage issues the same
  // number of loads (zeros past the last), so that the count of those still out, one stage's, is the same too.
  auto step = [&](const int8_t* sz, const int8_t* sw, int st, int8_t* dz, int8_t* dw) {
    issue(st, dz, dw);
    stage_products<TM, TN>(sz, sw, 16 * TM * wm, 16 * TN * wn, acc);
    stage_order<TM, TN, PER>();
    arrive<PER>();
  };
  issue(0, sZ0, sW0);
  // the scales of the tile's tokens and columns, behind the first stage
  if (threadIdx.x < BM + BN) {
    const int i = threadIdx.x;
    const float* from = i < BM ? a.z_scale + min(p.m0 + i, a.M - 1)
                               : a.w_scale + ((size_t)p.nb * a.cols + min(p.c0 + i - BM, used - 1));
    *reinterpret_cast<float*>(sZ0 + (kScale + 4 * i)) = *from;
  }
  issue(1, sZ1, sW1);
  arrive<PER>();
  for (int st = 0; st < stages; st += 3) {
    step(sZ0, sW0, st + 2, sZ2, sW2);
    if (st + 1 < stages) step(sZ1, sW1, st + 3, sZ0, sW0);
    if (st + 2 < stages) step(sZ2, sW2, st + 4, sZ1, sW1);
  }
  arrive<0>();  // the last loads (zeros) have landed before the LDS is another workgroup's
  if (p.c0 + 16 * TN * wn < used)
    store_tile<T, TM, TN>(acc, a, blk, p.nb, p.m0 + 64 * wm, p.c0 + 32 * wn, sZ0, kScale + 256 * wm,
                          kScale + 512 + 128 * wn, 1024 * w);
}

// MT tiles of 16 tokens and NC of 16 columns, NW waves sharing the inputs.
template <typename T, int MT, int NC, int NW>
__global__ __launch_bounds__(64 * NW) void project_int8_few_kernel(const Args a, const Blocks blk) {
  __shared__ int part[NW][MT][16][16 * NC + 1];  // [token][column], a column more against bank conflicts
  const int nb = block_of(blk, blockIdx.x);
  const int c0 = ((int)blockIdx.x - blk.start[nb]) * (16 * NC);
  const int used = blk.used[nb], d = a.d;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63, lq = l & 15, g = l >> 4;
  const __amdgpu_buffer_rsrc_t rz = rows_rsrc(a.z, a.M, d);
  const __amdgpu_buffer_rsrc_t rw =
      rows_rsrc(a.wt + ((size_t)nb * a.cols + c0) * d, min(16 * NC, a.cols - c0), d);
  i32x4 acc[NC][MT];
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[c][i] = i32x4{0, 0, 0, 0};
  // a step: 128 inputs of 16 weight rows a tile, lane (lq, g) the 32 bytes at 32 g of row lq
  const unsigned row = (unsigned)lq * (unsigned)d + 16u * (unsigned)g, tile = 16u * (unsigned)d;
  const int steps = (d + 127) / 128;
  // Each workgroup begins at a step of its own (the sums are exact, so their order is free): from the first step on
  // together, all of them read the same few lines of every row, which lie in few of the caches' and memory's channels
  // (32 tokens, 8192 to 8192: 28 us together, 18.4 so; 64 tokens 29 and 26; 1 token, 4096 to 6144: 8.4 and 7.5).
  int at = (w + (int)blockIdx.x) % steps;
  for (int n = w; n < steps; n += NW) {
    const int k0 = 128 * at;
    at += NW;
    if (at >= steps) at -= steps;
    i32x4 f[2][NC], zf[2][MT];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = k0 + 64 * h;
      const unsigned o = k + 16 * g < d ? row + (unsigned)k : kOutside;  // d is a multiple of 16
#pragma unroll
      for (int c = 0; c < NC; ++c) f[h][c] = load16(rw, o + tile * (unsigned)c);
#pragma unroll
      for (int i = 0; i < MT; ++i) zf[h][i] = load16(rz, o + tile * (unsigned)i);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < MT; ++i)
          acc[c][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[h][c], zf[h][i], acc[c][i], 0, 0, 0);
  }
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) part[w][i][lq][16 * c + 4 * g + r] = acc[c][i][r];
  __syncthreads();
  const float* ws = a.w_scale + (size_t)nb * a.cols;
  T* out = static_cast<T*>(blk.out[nb]);
  for (int i = threadIdx.x; i < 256 * MT * NC; i += 64 * NW) {
    const int c = i % (16 * NC), m = i / (16 * NC);
    if (m >= a.M || c0 + c >= used) continue;
    int sum = 0;
#pragma unroll
    for (int u = 0; u < NW; ++u) sum += part[u][m >> 4][m & 15][c];
    const float scale = a.z_scale[m] * ws[c0 + c];
    out[(size_t)m * used + c0 + c] = nb == a.sig_block ? finish<T, true>(sum, scale) : finish<T, false>(sum, scale);
  }
}

template <typename T>
int project_int8(const int8_t* z, const float* z_scale, const int8_t* wt, const float* w_scale, int nblk, int cols,
                 int d, int M, const int (&used_in)[kMaxBlocks], void* const (&out_in)[kMaxBlocks], int sigmoid_block,
                 void* stream, const char* who) {
  if (nblk < 1 || nblk > kMaxBlocks) return fail(ERR_ARG, "%s: %d weight blocks (1..%d)", who, nblk, kMaxBlocks);
  if (d < 16 || d > 16384 || d % 16 != 0)
    return fail(ERR_ARG, "%s: width %d (a multiple of 16 in 16..16384)", who, d);
  if (M < 0 || cols < 1) return fail(ERR_ARG, "%s: bad sizes M=%d cols=%d", who, M, cols);
  if (sigmoid_block < -1 || sigmoid_block >= nblk) return fail(ERR_ARG, "%s: sigmoid block %d", who, sigmoid_block);
  // the wide tile where the small one's workgroups would go around the 256 CUs more than twice, the narrow one where
  // the narrow one's do not fill them once (128 x 8192 to 8192: 26.5 us, 128 columns 30.8; 256 x 4096 to 6144: 16.2 and
  // 18.2; 1000 x 2048 to 2048: 10.7 and 11.8; but 512 x 8192 to 8192, 512 narrow ones: 41 and 37)
  const bool few = M <= kFewTokens;
  int64_t small = 0, half = 0;
  for (int j = 0; j < nblk; ++j) {
    small += ((int64_t)(used_in[j] > 0 ? used_in[j] : 0) + 127) / 128;
    half += ((int64_t)(used_in[j] > 0 ? used_in[j] : 0) + 63) / 64;
  }
  const int64_t mt = ((int64_t)M + 127) / 128;
  const int tile = small * mt > 512 ? 256 : 128, tile_cols = tile == 256 ? 256 : half * mt <= 256 ? 64 : 128;
  // the few-token kernel's columns: 32 where 16 would make more than a workgroup a CU (each reads all the tokens)
  int64_t narrow = 0;
  for (int j = 0; j < nblk; ++j) narrow += ((int64_t)(used_in[j] > 0 ? used_in[j] : 0) + 15) / 16;
  const int few_cols = M > 16 && narrow > 256 ? 32 : 16;
  const int width = few ? few_cols : tile_cols;
  Blocks blk{};
  blk.nblk = nblk;
  int64_t tiles = 0;
  for (int j = 0; j < kMaxBlocks; ++j) {
    blk.start[j] = (int)tiles;
    if (j >= nblk) continue;
    if (used_in[j] < 1 || used_in[j] > cols)
      return fail(ERR_ARG, "%s: block %d uses %d of its %d columns", who, j, used_in[j], cols);
    if (M > 0 && out_in[j] == nullptr) return fail(ERR_ARG, "%s: null output for block %d", who, j);
    if (reinterpret_cast<uintptr_t>(out_in[j]) & 15) return fail(ERR_ARG, "%s: output %d must be 16-byte aligned", who, j);
    blk.used[j] = used_in[j];
    blk.out[j] = out_in[j];
    tiles += ((int64_t)used_in[j] + width - 1) / width;
  }
  blk.start[kMaxBlocks] = (int)tiles;
  if (M == 0) return OK;
  if (!z || !z_scale || !wt || !w_scale) return fail(ERR_ARG, "%s: null pointer", who);
  if ((reinterpret_cast<uintptr_t>(z) | reinterpret_cast<uintptr_t>(wt)) & 15)
    return fail(ERR_ARG, "%s: z and the weights must be 16-byte aligned", who);
  const int mtiles = (int)(((int64_t)M + tile - 1) / tile);
  const int64_t n = few ? tiles : (tiles * mtiles + 7) / 8 * 8;  // whole rounds over the 8 XCDs
  if (n >= ((int64_t)1 << 31)) return fail(ERR_ARG, "%s: too many tiles", who);
  const Args a{z, z_scale, wt, w_scale, M, d, cols, sigmoid_block};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (!few) {
    if (tile == 256)
      hipLaunchKernelGGL(project_int8_kernel<T>, dim3((unsigned)(n < 256 ? n : 256)), dim3(512), 0, s, a, blk,
                         (int)tiles, mtiles, (int)(tiles * mtiles));
    else if (tile_cols == 128)
      hipLaunchKernelGGL((project_int8_small_kernel<T, 4>), dim3((unsigned)n), dim3(512), 0, s, a, blk, (int)tiles, mtiles);
    else
      hipLaunchKernelGGL((project_int8_small_kernel<T, 2>), dim3((unsigned)n), dim3(256), 0, s, a, blk, (int)tiles, mtiles);
    return check_launch(who);
  }
  if (n >= ((int64_t)1 << 32) / (M <= 16 ? 256 : 512))  // a launch has less than 2^32 threads
    return fail(ERR_UNSUPPORTED, "%s: %lld workgroups", who, (long long)n);
  auto go = [&](auto kern, int nw) { hipLaunchKernelGGL(kern, dim3((unsigned)n), dim3(64 * nw), 0, s, a, blk); };
  if (M <= 16) go(project_int8_few_kernel<T, 1, 1, 4>, 4);
  else if (M <= 32) few_cols == 16 ? go(project_int8_few_kernel<T, 2, 1, 8>, 8) : go(project_int8_few_kernel<T, 2, 2, 8>, 8);
  else few_cols == 16 ? go(project_int8_few_kernel<T, 4, 1, 8>, 8) : go(project_int8_few_kernel<T, 4, 2, 8>, 8);
  return check_launch(who);
}

}  // namespace
}  // namespace vsp

#define VSP_PROJECT_INT8(SUFFIX, T)                                                                                    \
  extern "C" int vsp_project_int8_##SUFFIX(const int8_t* z, const float* z_scale, const int8_t* weights,               \
                                           const float* weights_scale, int nblk, int cols, int d, int M, int used0,    \
                                           int used1, int used2, int used3, void* out0, void* out1, void* out2,        \
                                           void* out3, int sigmoid_block, void* stream) {                              \
    const int used[4] = {used0, used1, used2, used3};                                                                  \
    void* const out[4] = {out0, out1, out2, out3};                                                                     \
    return vsp::project_int8<T>(z, z_scale, weights, weights_scale, nblk, cols, d, M, used, out, sigmoid_block, stream, \
                                "vsp_project_int8_" #SUFFIX);                                                          \
  }
VSP_PROJECT_INT8(bf16, __bf16)
VSP_PROJECT_INT8(f16, _Float16)
VSP_PROJECT_INT8(f32, float)
