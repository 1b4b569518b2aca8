// Layer norm on CDNA4 (gfx950), forward and backward, with the residual's addition in it.
//
// Forward, a row s = x + r of d values: y = (s - mu) / sqrt(var + eps) * gain + bias, mu the mean, var the mean of
// (s - mu)^2; the sum s is written too (the residual stream), with mu and 1 / sqrt(var + eps) of each row for the
// backward. Both passes take s in float32: a sum that is kept in 16 bits is formed again from x and r in the backward,
// since the rounding of s would be off from its row's mu and rstd by up to the whole deviation of a narrow row (and
// put 2e-3 on dgain).
// Backward, xh = (s - mu) rstd, w = dy gain: ds = rstd (w - mean(w) - xh mean(w xh)) + dsum, which is dx and dr;
// dgain = sum over rows of dy xh, dbias of dy.
//
// Both are bound by memory: a row is read once into registers (16-byte loads), the two sums a row needs are lane
// reductions, and what is written is written once. Rows of up to 64 lanes' worth belong to a wave, wider ones to a
// workgroup of four (or, past that, sixteen) waves. The sums over rows stay in registers: a workgroup takes rows
// grid apart, each lane adds up the columns that it holds in every row, and leaves one partial row; a second kernel
// adds the partial rows in order. No atomics: results repeat bit for bit. 16384 x 4096 in bf16 with the residual and the
// sum's gradient: forward 100 us (537 MB, 5.4 TB/s), backward 140 (686 MB, 4.9 TB/s: each row waits for its two sums between
// its loads and its stores) and 5 for the columns; 16383 x 768 in float32 30, 35 and 4; 30000 x 513 in bf16 48 and 73 (element by
// element 116 and 173).
//
// A row whose sum passes float32 is summed again in parts of 2^-ceil(log2 d) of its values. A row is scaled by a power of
// two (exact) that brings its largest deviation below 2^32 before it is squared, so that var does not overflow; eps is
// scaled with it. So is, up, a row of small deviations where eps is next to nothing (below 2^-100), so that the squares
// do not vanish; beside a larger eps what is lost of them does not count.
#include <algorithm>
#include <initializer_list>

#include "common.h"
#include "vesper_kernels.h"

namespace vsp {
namespace {

// WAVES waves share a row, SEG pieces of 8 elements a lane; EDGE for odd widths and unaligned memory.
// Reduction over the waves of a row; `slot` alternates so that one barrier a reduction is enough.
template <int WAVES, int N, typename Op>
__device__ __forceinline__ void row_reduce(float (&x)[N], float (*red)[16][N], int slot, Op op) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = group_reduce<64>(x[i], op);
  if constexpr (WAVES > 1) {
    const int w = (threadIdx.x >> 6) % WAVES;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) red[slot][w][i] = x[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = red[slot][0][i];
    for (int j = 1; j < WAVES; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = op(x[i], red[slot][j][i]);
  }
}

// Eight elements of a row from f on. EDGE: rows of any width and alignment; a row's last piece goes element by element, the
// others in 16 bytes at the type's alignment (which the memory path takes). Else the width is a multiple of 8 and all
// memory 16-byte aligned, and a piece past the row reads its first one. What is past the row is masked by `inside`.
template <bool EDGE> __device__ __forceinline__ bool inside(int f, int e, int d) { return EDGE ? f + e < d : f < d; }

// as they come from memory, converted where they are used: 16-bit values take half of the registers
template <typename T> struct Piece {
  typedef T V8 __attribute__((ext_vector_type(8), aligned(16)));  // as the launcher checks it (eight floats of their own: 32)
  typedef T V8u __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  V8 x;
  template <bool EDGE> __device__ __forceinline__ void load(const T* row, int f, int d) {
    if constexpr (!EDGE) {
      x = *reinterpret_cast<const V8*>(row + (f < d ? f : 0));
    } else if (f + 8 <= d) {
      x = *reinterpret_cast<const V8u*>(row + f);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = f + e < d ? row[f + e] : (T)0;
    }
  }
  __device__ __forceinline__ float get(int e) const { return to_f32(x[e]); }
};
template <bool EDGE, typename T>
__device__ __forceinline__ void store_piece(T* row, int f, int d, const float (&x)[8]) {
  typename Piece<T>::V8 y;
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = from_f32<T>(x[e]);
  if constexpr (!EDGE) {
    *reinterpret_cast<typename Piece<T>::V8*>(row + f) = y;
  } else if (f + 8 <= d) {
    *reinterpret_cast<typename Piece<T>::V8u*>(row + f) = y;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (f + e < d) row[f + e] = y[e];
  }
}

template <int WAVES> struct NormShape {
  static constexpr int NT = WAVES == 1 ? 256 : 64 * WAVES;
  static constexpr int ROWS = NT / (64 * WAVES);  // rows a workgroup has in hand at once
};

template <typename TX, typename TR, typename TY, int WAVES, int SEG, bool EDGE>
__global__ __launch_bounds__(NormShape<WAVES>::NT) void layer_norm_kernel(
    const TX* __restrict__ x, const TR* __restrict__ res, const float* __restrict__ gain, const float* __restrict__ bias,
    TX* __restrict__ sum_out, TY* __restrict__ y, float* __restrict__ stats, int rows, int d, float eps) {
  __shared__ float red[4][16][1];
  constexpr int LANES = 64 * WAVES;
  const int t = threadIdx.x % LANES;
  // whole waves, and whole workgroups where a barrier follows; between two uses of a slot are two barriers at least
  for (long row = (long)blockIdx.x * NormShape<WAVES>::ROWS + threadIdx.x / LANES; row < rows;
       row += (long)gridDim.x * NormShape<WAVES>::ROWS) {
    const size_t base = (size_t)row * d;
    float v[SEG][8];
    float sum[1] = {0.f};
#pragma unroll
    for (int j = 0; j < SEG; ++j) {
      const int f = 8 * (t + LANES * j);
      Piece<TX> xs;
      xs.template load<EDGE>(x + base, f, d);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[j][e] = xs.get(e);
      if (res != nullptr) {
        Piece<TR> r;
        r.template load<EDGE>(res + base, f, d);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] += r.get(e);
        if (f < d) store_piece<EDGE>(sum_out + base, f, d, v[j]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[0] += inside<EDGE>(f, e, d) ? v[j][e] : 0.f;
    }
    row_reduce<WAVES, 1>(sum, red, 0, SumOp{});
    float mu = sum[0] / (float)d;
    if (!(fabsf(sum[0]) <= 3.40282347e38f)) {  // the same for all of the row's lanes: its sum overflowed (or a value is none)
      const float part = __builtin_ldexpf(1.f, d > 1 ? __builtin_clz((unsigned)(d - 1)) - 32 : 0);
      float again[1] = {0.f};
#pragma unroll
      for (int j = 0; j < SEG; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) again[0] += inside<EDGE>(8 * (t + LANES * j), e, d) ? v[j][e] * part : 0.f;
      row_reduce<WAVES, 1>(again, red, 3, SumOp{});
      mu = again[0] / ((float)d * part);
    }
    float peak[1] = {0.f};
#pragma unroll
    for (int j = 0; j < SEG; ++j) {
      const int f = 8 * (t + LANES * j);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[j][e] = inside<EDGE>(f, e, d) ? v[j][e] - mu : 0.f;
        peak[0] = __builtin_fmaxf(peak[0], fabsf(v[j][e]));
      }
    }
    row_reduce<WAVES, 1>(peak, red, 1, MaxOp{});
    float scale = 1.f;
    if (peak[0] > 4294967296.f || (eps < 0x1p-100f && peak[0] < 0x1p-32f && peak[0] > 0.f)) {
      const int up = 32 - __builtin_amdgcn_frexp_expf(peak[0]);
      scale = __builtin_ldexpf(1.f, up < 100 ? up : 100);
    }
    float sq[1] = {0.f};
#pragma unroll
    for (int j = 0; j < SEG; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[j][e] *= scale;
        sq[0] += v[j][e] * v[j][e];
      }
    row_reduce<WAVES, 1>(sq, red, 2, SumOp{});
    const float root = 1.f / __builtin_sqrtf(sq[0] / (float)d + eps * scale * scale);
    if (stats != nullptr && t == 0) {
      stats[2 * (size_t)row] = mu;
      stats[2 * (size_t)row + 1] = root * scale;
    }
#pragma unroll
    for (int j = 0; j < SEG; ++j) {
      const int f = 8 * (t + LANES * j);
      if (f >= d) continue;
      Piece<float> gn, bs;
      gn.template load<EDGE>(gain, f, d);
      if (bias != nullptr) bs.template load<EDGE>(bias, f, d);
      float out[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e] = v[j][e] * root * gn.get(e) + (bias != nullptr ? bs.get(e) : 0.f);
      store_piece<EDGE>(y + base, f, d, out);
    }
  }
}

// res as in the forward, or null where x is the float32 sum itself. dres may be null (no residual, or of x's type:
// then dx serves both). partial: [grid][2][d] sums of dy xh and dy.
template <typename TX, typename TR, typename TY, int WAVES, int SEG, bool EDGE>
__global__ __launch_bounds__(NormShape<WAVES>::NT) void layer_norm_backward_kernel(
    const TX* __restrict__ x, const TR* __restrict__ res, const float* __restrict__ gain, const float* __restrict__ stats,
    const TY* __restrict__ dy,
    const TX* __restrict__ dsum, TX* __restrict__ dx, TR* __restrict__ dres, float* __restrict__ partial, int rows, int d) {
  constexpr int LANES = 64 * WAVES, ROWS = NormShape<WAVES>::ROWS;
  // Sixteen waves of two pieces have 128 registers each: the sum's gradient is loaded at the end, the gain at each use.
  constexpr bool TIGHT = WAVES == 16 && SEG > 1;
  __shared__ float red[2][16][2];
  __shared__ float cols[ROWS > 1 ? ROWS : 1][ROWS > 1 ? 64 * SEG * 8 : 1];
  const int t = threadIdx.x % LANES, sub = threadIdx.x / LANES;
  Piece<float> gn[SEG];
  float dg[SEG][8], db[SEG][8];
#pragma unroll
  for (int j = 0; j < SEG; ++j) {
    if (!TIGHT) gn[j].template load<EDGE>(gain, 8 * (t + LANES * j), d);
#pragma unroll
    for (int e = 0; e < 8; ++e) dg[j][e] = db[j][e] = 0.f;
  }
  int slot = 0;
  for (long row = (long)blockIdx.x * ROWS + sub; row < rows; row += (long)gridDim.x * ROWS) {
    const size_t base = (size_t)row * d;
    const float mu = stats[2 * (size_t)row], rstd = stats[2 * (size_t)row + 1];
    float xh[SEG][8];
    Piece<TY> g[SEG];
    Piece<TX> add[SEG];
    float sums[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < SEG; ++j) {
      const int f = 8 * (t + LANES * j);
      Piece<TX> xs;
      xs.template load<EDGE>(x + base, f, d);
#pragma unroll
      for (int e = 0; e < 8; ++e) xh[j][e] = xs.get(e);
      if (res != nullptr) {
        Piece<TR> r;
        r.template load<EDGE>(res + base, f, d);
#pragma unroll
        for (int e = 0; e < 8; ++e) xh[j][e] += r.get(e);
      }
      g[j].template load<EDGE>(dy + base, f, d);
      if (TIGHT) gn[j].template load<EDGE>(gain, f, d);
      if (!TIGHT && dsum != nullptr) add[j].template load<EDGE>(dsum + base, f, d);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool ok = inside<EDGE>(f, e, d);
        xh[j][e] = ok ? (xh[j][e] - mu) * rstd : 0.f;
        const float g0 = ok ? g[j].get(e) : 0.f, w = ok ? g0 * gn[j].get(e) : 0.f;
        db[j][e] += g0;
        dg[j][e] += g0 * xh[j][e];
        sums[0] += w;
        sums[1] += w * xh[j][e];
      }
    }
    row_reduce<WAVES, 2>(sums, red, slot, SumOp{});
    slot ^= 1;
    const float m0 = sums[0] / (float)d, m1 = sums[1] / (float)d;
#pragma unroll
    for (int j = 0; j < SEG; ++j) {
      const int f = 8 * (t + LANES * j);
      if (f >= d) continue;
      float o[8];
      if (TIGHT) gn[j].template load<EDGE>(gain, f, d);
      if (TIGHT && dsum != nullptr) add[j].template load<EDGE>(dsum + base, f, d);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = rstd * (g[j].get(e) * gn[j].get(e) - m0 - xh[j][e] * m1) + (dsum != nullptr ? add[j].get(e) : 0.f);
      store_piece<EDGE>(dx + base, f, d, o);
      if (dres != nullptr) store_piece<EDGE>(dres + base, f, d, o);
    }
  }
  float* out = partial + (size_t)blockIdx.x * 2 * d;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if constexpr (ROWS > 1) {  // the workgroup's waves hold the same columns: their sums in order, through LDS
      __syncthreads();
#pragma unroll
      for (int j = 0; j < SEG; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) cols[sub][8 * (t + LANES * j) + e] = half ? db[j][e] : dg[j][e];
      __syncthreads();
      for (int f = threadIdx.x; f < d; f += NormShape<WAVES>::NT) {
        float x = cols[0][f];
        for (int i = 1; i < ROWS; ++i) x += cols[i][f];
        out[half * d + f] = x;
      }
    } else {
#pragma unroll
      for (int j = 0; j < SEG; ++j) {
        const int f = 8 * (t + LANES * j);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (f + e < d) out[half * d + f + e] = half ? db[j][e] : dg[j][e];
      }
    }
  }
}

// dgain and dbias: the column sums of the partial rows. A workgroup takes 64 columns (of the 2 d); its sixteen waves take
// every sixteenth partial row each, eight of them in flight, then the sixteen sums are added in order.
constexpr int kColumnWaves = 16;
__global__ __launch_bounds__(64 * kColumnWaves) void layer_norm_columns_kernel(const float* __restrict__ partial,
                                                                              float* __restrict__ dgain,
                                                                              float* __restrict__ dbias, int parts, int d) {
  __shared__ float red[kColumnWaves][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
  float a[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = 0.f;
  if (col < 2 * d) {
    int p = w;
    for (; p + 7 * kColumnWaves < parts; p += 8 * kColumnWaves)
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] += partial[(size_t)(p + i * kColumnWaves) * 2 * d + col];
    for (; p < parts; p += kColumnWaves) a[0] += partial[(size_t)p * 2 * d + col];
  }
  red[w][lane] = ((a[0] + a[1]) + (a[2] + a[3])) + ((a[4] + a[5]) + (a[6] + a[7]));
  __syncthreads();
  if (w == 0 && col < 2 * d) {
    float x = red[0][lane];
#pragma unroll
    for (int i = 1; i < kColumnWaves; ++i) x += red[i][lane];
    if (col < d) dgain[col] = x;
    else if (dbias != nullptr) dbias[col - d] = x;
  }
}

// The widest row of a shape: WAVES * 64 lanes, SEG pieces of 8. W4 and W8 are the shapes of rows of up to 4096 and 8192. Rows
// of odd widths take one piece a lane where they can: with two, their element-wise ends take all registers.
#define VSP_NORM_SHAPES(GO, W4, W8)             \
  if (vec) {                                    \
    if (d <= 512) GO(1, 1, false)               \
    else if (d <= 1024) GO(1, 2, false)         \
    else if (d <= 2048) GO(4, 1, false)         \
    else if (d <= 4096) W4(GO)                  \
    else if (d <= 8192) W8(GO)                  \
    else GO(16, 2, false)                       \
  } else {                                      \
    if (d <= 512) GO(1, 1, true)                \
    else if (d <= 2048) GO(4, 1, true)          \
    else if (d <= 8192) GO(16, 1, true)         \
    else GO(16, 2, true)                        \
  }

bool aligned16(std::initializer_list<const void*> ps) {
  uintptr_t x = 0;
  for (const void* p : ps) x |= reinterpret_cast<uintptr_t>(p);
  return (x & 15) == 0;
}

int norm_check(int rows, int d, const char* who) {
  if (rows < 0 || d < 1 || d > 16384) return fail(ERR_ARG, "%s: rows %d, width %d (1..16384)", who, rows, d);
  return OK;
}

template <typename TX, typename TR, typename TY>
int norm_forward(const void* x_, const void* res_, const float* gain, const float* bias, void* sum_, void* y_, float* stats,
                 int rows, int d, float eps, hipStream_t stream, const char* who) {
  const TX* x = static_cast<const TX*>(x_);
  const TR* res = static_cast<const TR*>(res_);
  TX* sum = static_cast<TX*>(sum_);
  TY* y = static_cast<TY*>(y_);
  const bool vec = d % 8 == 0 && aligned16({x, res, gain, bias, sum, y});
  // launches of fewer than 2^32 threads: past 2^20 workgroups each takes several rows
#define VSP_GO(W, S, EDGE)                                                                                              \
  hipLaunchKernelGGL((layer_norm_kernel<TX, TR, TY, W, S, EDGE>),                                                       \
                     dim3((unsigned)std::min<long>(((long)rows + NormShape<W>::ROWS - 1) / NormShape<W>::ROWS, 1 << 20)), \
                     dim3(NormShape<W>::NT), 0, stream, x, res, gain, bias, sum, y, stats, rows, d, eps);
#define VSP_W4(GO) GO(4, 2, false)
#define VSP_W8(GO) GO(4, 4, false)
  VSP_NORM_SHAPES(VSP_GO, VSP_W4, VSP_W8)
#undef VSP_W4
#undef VSP_W8
#undef VSP_GO
  return check_launch(who);
}

// Workgroups of the backward, and so partial rows, at most; as many as the card holds at once are launched, each with
// several rows where there are many: with 1024 of a kernel of which it holds 768, the last quarter ran alone (16384 x
// 4096 in bf16: 195 us against 154).
constexpr int kNormParts = 1024, kCus = 256;
int norm_parts(int rows, int d) {
  const int at_once = d <= 1024 ? 4 : 1;
  const int groups = rows / at_once + (rows % at_once != 0);
  return groups < kNormParts ? groups : kNormParts;
}

int held_at_once(const void* kernel, int threads) {
  int per_cu = 0;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, kernel, threads, 0) != hipSuccess || per_cu < 1) per_cu = 1;
  return per_cu * kCus;
}

template <typename TX, typename TR, typename TY>
int norm_backward(const void* x_, const void* res_, const float* gain, const float* stats, const void* dy_, const void* dsum_, void* dx_,
                  void* dres_, float* dgain, float* dbias, float* ws, int rows, int d, hipStream_t stream, const char* who) {
  const TX *x = static_cast<const TX*>(x_), *dsum = static_cast<const TX*>(dsum_);
  const TR* res = static_cast<const TR*>(res_);
  const TY* dy = static_cast<const TY*>(dy_);
  TX* dx = static_cast<TX*>(dx_);
  TR* dres = static_cast<TR*>(dres_);
  const bool vec = d % 8 == 0 && aligned16({x, res, gain, dy, dsum, dx, dres});
  int parts = norm_parts(rows, d);
#define VSP_GO(W, S, EDGE)                                                                                              \
  {                                                                                                                  \
    static const int held = held_at_once(reinterpret_cast<const void*>(layer_norm_backward_kernel<TX, TR, TY, W, S, EDGE>), NormShape<W>::NT); \
    parts = std::min(parts, held);                                                                                   \
    hipLaunchKernelGGL((layer_norm_backward_kernel<TX, TR, TY, W, S, EDGE>), dim3((unsigned)parts), dim3(NormShape<W>::NT), 0, \
                       stream, x, res, gain, stats, dy, dsum, dx, dres, ws, rows, d);                                \
  }
// one piece a lane: four waves of four pieces have room for one workgroup a CU (4096 x 8192 in bf16: 123 us against 82)
#define VSP_W4(GO) GO(8, 1, false)
#define VSP_W8(GO) GO(16, 1, false)
  VSP_NORM_SHAPES(VSP_GO, VSP_W4, VSP_W8)
#undef VSP_W4
#undef VSP_W8
#undef VSP_GO
  hipLaunchKernelGGL(layer_norm_columns_kernel, dim3((unsigned)((2 * d + 63) / 64)), dim3(64 * kColumnWaves), 0, stream, ws, dgain, dbias, parts, d);
  return check_launch(who);
}

// The types of x (and the sum), the residual and y. Codes: 0 float32, 1 bfloat16, 2 float16.
template <typename F> int by_types(int tx, int tr, int ty, const char* who, F go) {
  struct F32 { using T = float; };
  struct B16 { using T = __bf16; };
  struct H16 { using T = _Float16; };
  if (tx == 1 && tr == 1 && ty == 1) return go(B16{}, B16{}, B16{});
  if (tx == 2 && tr == 2 && ty == 2) return go(H16{}, H16{}, H16{});
  if (tx == 0) switch (3 * tr + ty) {
    case 0: return go(F32{}, F32{}, F32{});
    case 1: return go(F32{}, F32{}, B16{});
    case 2: return go(F32{}, F32{}, H16{});
    case 3: return go(F32{}, B16{}, F32{});
    case 4: return go(F32{}, B16{}, B16{});
    case 5: return go(F32{}, B16{}, H16{});
    case 6: return go(F32{}, H16{}, F32{});
    case 7: return go(F32{}, H16{}, B16{});
    case 8: return go(F32{}, H16{}, H16{});
    default: break;
  }
  return fail(ERR_UNSUPPORTED, "%s: types %d, %d, %d of x, the residual and y", who, tx, tr, ty);
}

}  // namespace
}  // namespace vsp

extern "C" int vsp_layer_norm(const void* x, const void* residual, const float* gain, const float* bias, void* sum_out,
                              void* y, float* stats, int x_type, int residual_type, int y_type, int rows, int d, float eps,
                              void* stream) {
  using namespace vsp;
  const char* who = "vsp_layer_norm";
  if (const int st = norm_check(rows, d, who); st != OK) return st;
  if (rows == 0) return OK;
  if (!x || !gain || !y || (residual && !sum_out)) return fail(ERR_ARG, "%s: null pointer", who);
  return by_types(x_type, residual_type, y_type, who, [&](auto a, auto b, auto c) {
    return norm_forward<typename decltype(a)::T, typename decltype(b)::T, typename decltype(c)::T>(
        x, residual, gain, bias, sum_out, y, stats, rows, d, eps, reinterpret_cast<hipStream_t>(stream), who);
  });
}

extern "C" size_t vsp_layer_norm_backward_workspace_bytes(int rows, int d) {
  if (rows <= 0 || d <= 0) return 0;
  return (size_t)vsp::norm_parts(rows, d) * 2 * d * sizeof(float);
}

extern "C" int vsp_layer_norm_backward(const void* x, const void* residual, const float* gain, const float* stats,
                                       const void* dy, const void* dsum, void* dx, void* dresidual, float* dgain, float* dbias,
                                       void* workspace, size_t workspace_bytes, int x_type, int residual_type, int y_type,
                                       int rows, int d, void* stream) {
  using namespace vsp;
  const char* who = "vsp_layer_norm_backward";
  if (const int st = norm_check(rows, d, who); st != OK) return st;
  if (rows == 0) return fail(ERR_ARG, "%s: no rows", who);
  if (!x || !gain || !stats || !dy || !dx || !dgain || !workspace) return fail(ERR_ARG, "%s: null pointer", who);
  if (workspace_bytes < vsp_layer_norm_backward_workspace_bytes(rows, d))
    return fail(ERR_ARG, "%s: workspace of %zu bytes, needs %zu", who, workspace_bytes, vsp_layer_norm_backward_workspace_bytes(rows, d));
  return by_types(x_type, residual_type, y_type, who, [&](auto a, auto b, auto c) {
    return norm_backward<typename decltype(a)::T, typename decltype(b)::T, typename decltype(c)::T>(
        x, residual, gain, stats, dy, dsum, dx, dresidual, dgain, dbias, static_cast<float*>(workspace), rows, d,
        reinterpret_cast<hipStream_t>(stream), who);
  });
}
