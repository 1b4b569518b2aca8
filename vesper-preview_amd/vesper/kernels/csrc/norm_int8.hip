// RMSNorm with the residual's addition and an output in 8-bit integers, one scale a row, on CDNA4
// (gfx950): the operand of the 8-bit projections (project_int8.hip).
//
//   s = x + r (float32),  y = s / sqrt(mean(s^2) + 1e-6) * g,  a = max |y| / 127,  code = round(y / a)
//
// computed scale-safely as the bf16 norm (norm.hip; vesper/column.py:146-188): the row is first divided by
// its largest magnitude floored at 1e-3. Rounding a row against its own largest value leaves every
// element within half a step, a / 2. A row whose normalized values all stay below 2^-120 (zeros, or a
// gain that small) is stored as zeros with a = 0; a row with an infinity or a NaN, in x, r or the gain's
// product, has a = NaN and codes 0, so what is computed from it is NaN as from the bf16 norm. The quotients are
// products with reciprocals (of the row's magnitude, its root and a), a few float32 roundings away from the exact
// ones: one within 1e-3 of the middle between two codes may become either.
//
// Rows are held in registers between the reductions, so memory is touched once: bound by the bytes, 11
// an element with a bf16 residual, the sum written and float32 x (32767 rows of 768: 50.7 us, 5.5 TB/s, a large
// copy's rate; 64 rows of 512: 3.2 us). Up to 2048 wide a wave takes a row
// (reductions by DPP and lane swaps, no barrier); wider rows take a workgroup.
#include "common.h"
#include "vesper_kernels.h"

namespace vsp {
namespace {

constexpr float kRmsEps = 1e-6f;         // column.py:55
constexpr float kRmsScaleFloor = 1e-3f;  // column.py:56
constexpr float kTinyRow = 0x1p-120f;    // largest magnitude below which a row is stored as zeros

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    typedef T V8 __attribute__((ext_vector_type(8)));
    V8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = from_f32<T>(v[e]);
    *reinterpret_cast<V8*>(p) = y;
  } else {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}

// A reduction over the NT threads of a row: a wave's lanes, then the row's waves through LDS.
template <int NT, typename Op>
__device__ __forceinline__ float row_reduce(float x, Op op, float* slots) {
  x = group_reduce<64>(x, op);
  if constexpr (NT > 64) {
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = x;
    __syncthreads();
    x = slots[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) x = op(x, slots[w]);
  }
  return x;
}

// NT threads a row (64: four rows a workgroup), each with NSEG segments of eight elements.
template <typename T, typename R, int NSEG, int NT>
__global__ __launch_bounds__(NT == 64 ? 256 : NT) void rms_norm_int8_kernel(const T* __restrict__ x,
                                                                            const R* __restrict__ res,
                                                                            const float* __restrict__ gain,
                                                                            T* __restrict__ sum_out,
                                                                            int8_t* __restrict__ out,
                                                                            float* __restrict__ scale_out, int rows,
                                                                            int d) {
  __shared__ float slots[3][NT / 64];  // one set a reduction: none waits for the last one's readers
  const int row = NT == 64 ? blockIdx.x * 4 + (int)(threadIdx.x >> 6) : (int)blockIdx.x;
  const int t = NT == 64 ? (int)threadIdx.x & 63 : (int)threadIdx.x;
  if (row >= rows) return;  // whole waves, and with NT > 64 the grid has no such workgroup
  const size_t base = (size_t)row * d;
  float v[NSEG][8], peak = 0.f;
#pragma unroll
  for (int j = 0; j < NSEG; ++j) {
    const int f = 8 * (t + NT * j);
    const bool ok = f < d;
    float e[8];
    load8_f32(x + base + (ok ? f : 0), e);
    if (res != nullptr) {
      float r[8];
      load8_f32(res + base + (ok ? f : 0), r);
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] += r[i];
      if (ok && sum_out != nullptr) store8(sum_out + base + f, e);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[j][i] = ok ? e[i] : 0.f;
      peak = __builtin_fmaxf(peak, __builtin_fabsf(v[j][i]));
    }
  }
  const float scale = __builtin_fmaxf(row_reduce<NT>(peak, MaxOp{}, slots[0]), kRmsScaleFloor);
  const float inv_scale = 1.f / scale;
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < NSEG; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[j][i] *= inv_scale;
      ss += v[j][i] * v[j][i];
    }
  ss = row_reduce<NT>(ss, SumOp{}, slots[1]);  // NaN where the row holds a NaN, or an infinity (inf * 0)
  const float inv_rms = 1.f / __builtin_sqrtf(ss / (float)d + kRmsEps / (scale * scale));
  float top = ss < __builtin_inff() ? 0.f : __builtin_inff();
#pragma unroll
  for (int j = 0; j < NSEG; ++j) {
    const int f = 8 * (t + NT * j);
    float g[8];
    if (gain != nullptr) load8_f32(gain + (f < d ? f : 0), g);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[j][i] *= inv_rms;
      if (gain != nullptr) v[j][i] *= f < d ? g[i] : 0.f;
      const float y = __builtin_fabsf(v[j][i]);
      top = y < __builtin_inff() ? __builtin_fmaxf(top, y) : __builtin_inff();
    }
  }
  top = row_reduce<NT>(top, MaxOp{}, slots[2]);
  float a = top / 127.f, inv = 0.f;
  if (!(top < __builtin_inff())) a = __builtin_nanf("");
  else if (top < kTinyRow) a = 0.f;
  else inv = 1.f / a;
#pragma unroll
  for (int j = 0; j < NSEG; ++j) {
    const int f = 8 * (t + NT * j);
    if (f >= d) continue;
    uint32_t w[2] = {0, 0};
    if (inv != 0.f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i >> 2] |= ((uint32_t)(int)__builtin_rintf(v[j][i] * inv) & 0xffu) << (8 * (i & 3));
    }
    *reinterpret_cast<uint2*>(out + base + f) = make_uint2(w[0], w[1]);
  }
  if (t == 0) scale_out[row] = a;
}

template <typename T, typename R>
int rms_norm_int8(const T* x, const R* res, T* sum_out, const float* gain, int8_t* out, float* scale, int rows, int d,
                  void* stream, const char* who) {
  if (rows < 0 || d < 8 || d > 16384 || d % 8 != 0)
    return fail(ERR_ARG, "%s: rows %d, width %d (a multiple of 8 in 8..16384)", who, rows, d);
  if (rows == 0) return OK;
  if (!x || !out || !scale) return fail(ERR_ARG, "%s: null pointer", who);
  if (sum_out != nullptr && res == nullptr) return fail(ERR_ARG, "%s: a sum without a residual", who);
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(gain) | reinterpret_cast<uintptr_t>(res) |
       reinterpret_cast<uintptr_t>(sum_out)) & 15)
    return fail(ERR_ARG, "%s: x, the residual, the sum and gain must be 16-byte aligned", who);
  if (reinterpret_cast<uintptr_t>(out) & 7) return fail(ERR_ARG, "%s: out must be 8-byte aligned", who);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  auto go = [&](auto kern, int nt) {
    // a launch has less than 2^32 threads: at most 2^22 rows of 512, 2^25 of 64
    const int most = nt == 64 ? 1 << 25 : 1 << 22;
    for (int64_t r = 0; r < rows; r += most) {
      const int n = (int)(rows - r < most ? rows - r : most);
      const size_t at = (size_t)r * d;
      const unsigned grid = nt == 64 ? (unsigned)(n + 3) / 4 : (unsigned)n;
      hipLaunchKernelGGL(kern, dim3(grid), dim3(nt == 64 ? 256 : nt), 0, s, x + at, res ? res + at : nullptr, gain,
                         sum_out ? sum_out + at : nullptr, out + at, scale + r, n, d);
    }
  };
  if (d <= 512) go(rms_norm_int8_kernel<T, R, 1, 64>, 64);
  else if (d <= 1024) go(rms_norm_int8_kernel<T, R, 2, 64>, 64);
  else if (d <= 2048) go(rms_norm_int8_kernel<T, R, 4, 64>, 64);
  else if (d <= 4096) go(rms_norm_int8_kernel<T, R, 2, 256>, 256);
  else if (d <= 8192) go(rms_norm_int8_kernel<T, R, 4, 256>, 256);
  else go(rms_norm_int8_kernel<T, R, 4, 512>, 512);
  return check_launch(who);
}

}  // namespace
}  // namespace vsp

#define VSP_RMS_NORM_INT8(NAME, T, R)                                                                                \
  extern "C" int vsp_rms_norm_int8_##NAME(const void* x, const void* residual, void* sum_out, const float* gain,     \
                                          int8_t* out, float* scale, int rows, int d, void* stream) {                \
    return vsp::rms_norm_int8<T, R>(static_cast<const T*>(x), static_cast<const R*>(residual),                       \
                                    static_cast<T*>(sum_out), gain, out, scale, rows, d, stream,                     \
                                    "vsp_rms_norm_int8_" #NAME);                                                     \
  }
VSP_RMS_NORM_INT8(f32_bf16, float, __bf16)
VSP_RMS_NORM_INT8(f32_f16, float, _Float16)
VSP_RMS_NORM_INT8(bf16, __bf16, __bf16)
VSP_RMS_NORM_INT8(f16, _Float16, _Float16)
