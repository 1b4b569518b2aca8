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
// tile (many tokens): 256 tokens x 256 columns a workgroup of eight waves of 64 x 128, both operands through LDS in
// two stages of 128 inputs (whole cache lines a row), or, where that makes few workgroups, 128 x 128 in waves of
// 64 x 32 and three stages. global_load_lds_dwordx4 moves eight rows of 128 bytes an instruction, each row's
// 16-byte segments XOR-swizzled so that the fragment reads meet each bank once; 16x16x64 int8 MFMA formed
// transposed (weight rows as the A operand); the second half's fragments are read during the first half's products.
// 8192^3: 480 us (2.3 Pop/s; the chip's products clock down under them: the matrix units are busy 58 % of the
// cycles), a library product of the same operands 547. 32767 x 768 to 2316 columns: 94 us, of which the loads into
// LDS take 36 alone (503 MB, 14 TB/s), the products 25 and the outputs 29, with one workgroup a CU nearly one after
// the other; 128 x 128 tiles, two workgroups a CU, need 57, 15 and 22: 98 us. Stages of 64 inputs, four deep, read
// half cache lines: 117 us. Three stages of 256 x 128: 108 us. A workgroup a CU that goes from tile to tile, loading the
// next one's first stage under the last products: 95-107 us (stores and loads retire in one order, so its first wait
// is for the stores too).
//
// few (up to 64 tokens, a decode step): bound by reading the weights once. A workgroup takes 16 columns and
// all the tokens; its waves share the inputs, each reading whole 128-byte lines of 16 weight rows straight
// into the MFMA operand's registers; the waves' int32 sums are joined through LDS. Past 16 tokens the tokens'
// own reads count (from L2, by every workgroup): 32 columns a workgroup where there are enough (64 tokens, 8192 to
// 8192: 40 us with 16 columns, 31 with 32; 64 x 512 to 1544: 4.0 and 4.7), and eight waves in place of four (64 x
// 512: 4.5 -> 4.0; with up to 16 tokens four are as good or better: 16 x 8192 to 8192 17.0 us, 3.9 TB/s of
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
// exponential and reciprocal instructions (each within a unit of float32): a thread has 64 to 128 outputs, and as
// calls of the library's functions their code outgrew the instruction cache (32767 tokens of 768: 104 us with
// it, 90 without a logistic block).
template <typename T>
__device__ __forceinline__ T finish(int sum, float scale, bool sig) {
  float y = (float)sum * scale;
  if (sig) y = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * y));
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

// WM x WN waves of 16 TM tokens x 16 TN columns each, S stages in LDS.
template <typename T, int WM, int WN, int TM, int TN, int S>
__global__ __launch_bounds__(64 * WM * WN, 1) void project_int8_kernel(const Args a, const Blocks blk, int ctiles,
                                                                      int mtiles, int band) {
  constexpr int AHEAD = TN < 4 ? TN : 4;  // weight fragments read ahead of the products
  constexpr int NW = WM * WN, BM = 16 * TM * WM, BN = 16 * TN * WN;
  static_assert(BM == BN && BM % (8 * NW) == 0, "square tiles of whole load instructions");
  static_assert(S == 2 || S == 3, "two or three stages");
  // Stages of the z rows and the weight rows, [rows][128 inputs] each: row r's 16-byte segment s at s ^
  // 2 ((r >> 1) & 3), so that a fragment read (lanes 0-7 with 16-23: rows 0-7, two segments each) meets every
  // bank once. Separate variables: the compiler tells the direct loads into one from the reads of the others.
  __shared__ __align__(16) int8_t sZ0[BM * kBK], sZ1[BM * kBK], sZ2[S == 3 ? BM * kBK : 16];
  __shared__ __align__(16) int8_t sW0[BN * kBK], sW1[BN * kBK], sW2[S == 3 ? BN * kBK : 16];
  __shared__ __align__(16) float sScaleZ[BM], sScaleW[BN];

  // Workgroups of an XCD take runs of tiles, bands of `band` row tiles each, down a band's rows before the next
  // column tile: those that run together share rows of z and columns of the weights in the XCD's L2.
  const int lg = xcd_logical_block(blockIdx.x, gridDim.x);
  const int top = lg / (band * ctiles) * band, in_band = lg - top * ctiles, rows = min(band, mtiles - top);
  if (rows <= 0) return;  // the grid is padded to whole XCD rounds; whole workgroups leave
  const int ct = in_band / rows, mt = top + in_band - ct * rows;
  if (ct >= ctiles) return;
  const int nb = block_of(blk, ct);
  const int c0 = (ct - blk.start[nb]) * BN;
  const int used = blk.used[nb], d = a.d;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63, lq = l & 15, g = l >> 4;
  const int wm = w % WM, wn = w / WM;  // the wave's tokens 16 TM wm .. and columns 16 TN wn ..
  const bool live = c0 + 16 * TN * wn < used;
  const int stages = (d + kBK - 1) / kBK;

  // resources of the tile's own rows (under 256 x 16384 bytes): rows past the operands' ends read zeros
  const int zrows = min(BM, a.M - mt * BM), wrows = min(BN, a.cols - c0);
  const __amdgpu_buffer_rsrc_t rz = rows_rsrc(a.z + (size_t)mt * BM * d, zrows, d);
  const __amdgpu_buffer_rsrc_t rw = rows_rsrc(a.wt + ((size_t)nb * a.cols + c0) * d, wrows, d);
  auto kswz = [](int row) { return 2 * ((row >> 1) & 3); };
  // direct loads: instruction j of wave w fills rows 8 (w + NW j) .. + 7 of a stage, 128 bytes each; lane l brings
  // row l / 8's logical segment (l % 8) ^ kswz(row)
  constexpr int NL = BM / (8 * NW);
  const int lrow = l >> 3, lseg = (l & 7) ^ kswz(lrow);
  unsigned off[NL];  // the scalar offset holds the stage only: it stays below every resource's size
#pragma unroll
  for (int j = 0; j < NL; ++j) off[j] = (unsigned)(8 * (w + NW * j) + lrow) * (unsigned)d + 16u * (unsigned)lseg;
  auto issue = [&](int st, int8_t* dz, int8_t* dw) {
    // inputs past d (d is a multiple of 16, so whole segments), and whole stages past the last, are zeros
    const bool in = st * kBK + 16 * lseg < d;
    const unsigned so = (unsigned)(min(st, stages - 1) * kBK);
#pragma unroll
    for (int j = 0; j < NL; ++j) buffer_load_lds16(rz, dz + (w + NW * j) * 1024, in ? off[j] : kOutside, so);
#pragma unroll
    for (int j = 0; j < NL; ++j) buffer_load_lds16(rw, dw + (w + NW * j) * 1024, in ? off[j] : kOutside, so);
  };

  i32x4 acc[TN][TM];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int i = 0; i < TM; ++i) acc[j][i] = i32x4{0, 0, 0, 0};
  // A stage: the loads of the one S - 1 ahead, into the buffers that were read a stage ago (every wave has passed the
  // barrier behind those reads); the products; then the next stage has to have arrived. Every stage issues the same
  // number of loads (zeros past the last), so that the count of those still out, S - 2 stages', is the same too.
  auto step = [&](const int8_t* sz, const int8_t* sw, int st, int8_t* dz, int8_t* dw) {
    issue(st, dz, dw);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      i32x4 zf[TM];
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int row = 16 * (TM * wm + i) + lq;
        zf[i] = *reinterpret_cast<const i32x4*>(sz + row * kBK + 16 * ((4 * s + g) ^ kswz(row)));
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int row = 16 * (TN * wn + j) + lq;
        const i32x4 f = *reinterpret_cast<const i32x4*>(sw + row * kBK + 16 * ((4 * s + g) ^ kswz(row)));
#pragma unroll
        for (int i = 0; i < TM; ++i) acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f, zf[i], acc[j][i], 0, 0, 0);
      }
    }
    // the fragments of the second half are read while the first half's products run
    constexpr int EACH = (TM + 2 * TN - AHEAD + TN - 1) / TN;
    __builtin_amdgcn_sched_group_barrier(0x10, 2 * NL, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, TM + AHEAD, 0);
#pragma unroll
    for (int u = 0; u < 2 * TN; ++u) {
      __builtin_amdgcn_sched_group_barrier(0x8, TM, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, EACH, 0);
    }
    __builtin_amdgcn_sched_barrier(0);  // the wait stays behind the products
    arrive<2 * NL * (S - 2)>();
  };

  issue(0, sZ0, sW0);
  // the scales of the tile's tokens and columns, behind the first stage
  for (int i = threadIdx.x; i < BM; i += 64 * NW) sScaleZ[i] = a.z_scale[min(mt * BM + i, a.M - 1)];
  for (int i = threadIdx.x; i < BN; i += 64 * NW) sScaleW[i] = a.w_scale[(size_t)nb * a.cols + min(c0 + i, used - 1)];
  if constexpr (S == 3) issue(1, sZ1, sW1);
  arrive<2 * NL * (S - 2)>();
  if constexpr (S == 2) {
    for (int st = 0; st < stages; st += 2) {
      step(sZ0, sW0, st + 1, sZ1, sW1);
      if (st + 1 < stages) step(sZ1, sW1, st + 2, sZ0, sW0);
    }
  } else {
    for (int st = 0; st < stages; st += 3) {
      step(sZ0, sW0, st + 2, sZ2, sW2);
      if (st + 1 < stages) step(sZ1, sW1, st + 3, sZ0, sW0);
      if (st + 2 < stages) step(sZ2, sW2, st + 4, sZ1, sW1);
    }
  }
  arrive<0>();  // the last loads (zeros) have landed before the buffers are used again
  if (!live) return;

  // lane (lq, g) holds columns 16 j + 4 g + r of token 16 i + lq
  const int m0 = mt * BM + 16 * TM * wm, cw = c0 + 16 * TN * wn;
  T* out = static_cast<T*>(blk.out[nb]);
  float zs[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) zs[i] = sScaleZ[16 * (TM * wm + i) + lq];
  if constexpr (sizeof(T) == 2) {
    // through LDS (free behind the last barrier), so that whole rows leave: the wave's tile, row r's 16-byte segment
    // s at s ^ (r % the row's segments), then as whole rows
    typedef T V4 __attribute__((ext_vector_type(4)));
    typedef T V8 __attribute__((ext_vector_type(8)));
    constexpr int SEG = 2 * TN, TILE = 256 * TM * TN, PER = BM * kBK / (TILE * 2);  // PER waves' tiles a buffer
    static_assert(PER >= 1 && 4 * PER >= NW, "the waves' tiles fit two stages");
    int8_t* base = w / PER == 0 ? sZ0 : w / PER == 1 ? sZ1 : w / PER == 2 ? sW0 : sW1;
    T* stile = reinterpret_cast<T*>(base) + (w % PER) * TILE;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int c = 16 * j + 4 * g;
      const f32x4 bs = *reinterpret_cast<const f32x4*>(sScaleW + 16 * TN * wn + c);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int row = 16 * i + lq;
        V4 y;
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] = finish<T>(acc[j][i][r], zs[i] * bs[r], nb == a.sig_block);
        *reinterpret_cast<V4*>(stile + row * (16 * TN) + 8 * ((c >> 3) ^ (row & (SEG - 1))) + (c & 7)) = y;
      }
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the tile is in LDS (only this wave reads it)
    const int seg = l % SEG, col = cw + 8 * seg;
    const bool whole = (used & 7) == 0;
#pragma unroll
    for (int it = 0; it < 16 * TM * SEG / 64; ++it) {
      const int row = (64 / SEG) * it + l / SEG, m = m0 + row;
      if (m >= a.M || col >= used) continue;
      const V8 v = *reinterpret_cast<const V8*>(stile + row * (16 * TN) + 8 * (seg ^ (row & (SEG - 1))));
      T* orow = out + (size_t)m * used + col;
      if (whole) {
        *reinterpret_cast<V8*>(orow) = v;
      } else {
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (col + r < used) orow[r] = v[r];
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int col = cw + 16 * j + 4 * g;
      const f32x4 bs = *reinterpret_cast<const f32x4*>(sScaleW + 16 * TN * wn + 16 * j + 4 * g);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int m = m0 + 16 * i + lq;
        if (m >= a.M) continue;
        float y[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] = finish<T>(acc[j][i][r], zs[i] * bs[r], nb == a.sig_block);
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
  const unsigned row = (unsigned)lq * (unsigned)d + 32u * (unsigned)g, tile = 16u * (unsigned)d;
  for (int k0 = 128 * w; k0 < d; k0 += 128 * NW) {
    i32x4 f[2][NC], zf[2][MT];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = k0 + 16 * h;
      const unsigned o = k + 32 * g < d ? row + (unsigned)k : kOutside;  // d is a multiple of 16
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
    out[(size_t)m * used + c0 + c] = finish<T>(sum, a.z_scale[m] * ws[c0 + c], nb == a.sig_block);
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
  // the wide tile where the small one's workgroups would go around the 256 CUs more than twice
  const bool few = M <= kFewTokens;
  int64_t small = 0;
  for (int j = 0; j < nblk; ++j) small += ((int64_t)(used_in[j] > 0 ? used_in[j] : 0) + 127) / 128;
  const int tile = small * (((int64_t)M + 127) / 128) > 512 ? 256 : 128;
  // the few-token kernel's columns: 32 where 16 would make more than a workgroup a CU (each reads all the tokens)
  int64_t narrow = 0;
  for (int j = 0; j < nblk; ++j) narrow += ((int64_t)(used_in[j] > 0 ? used_in[j] : 0) + 15) / 16;
  const int few_cols = M > 16 && narrow > 256 ? 32 : 16;
  const int width = few ? few_cols : tile;
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
    auto run = [&](auto kern) {
      hipLaunchKernelGGL(kern, dim3((unsigned)n), dim3(512), 0, s, a, blk, (int)tiles, mtiles, kBand);
    };
    if (tile == 256) run(project_int8_kernel<T, 4, 2, 4, 8, 2>);
    else run(project_int8_kernel<T, 2, 4, 4, 2, 3>);
    return check_launch(who);
  }
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
