// The KV ring held in four bits on CDNA4 (gfx950): tokens quantised as they are written, read back by
// position, and the attention of one new token per row over the codes.
//
// The ring is the decoder's (vesper/attention.py:62-139, :298-338): a token at position p lives in slot
// p % W, visibility is decided by positions and flags, slots are in no order of age. Its rows are held
// head by head, [B, HKV, W, dk / 2] codes and [B, HKV, W] pairs (ring4.h): one head's rows are
// contiguous, so the workgroup that attends a head reads whole cache lines (a token's row is only
// dk / 2 bytes: 32 at dk 64; token by token every head's reader would fetch all the heads' bytes).
//
// Attention. Slots with a valid token at a position in (p - W, p] other than slot p % W, and the new
// token from its own argument (not quantised): the slot that the new token is about to take is never
// attended (in the ring's proper use it holds p - W, out of the window, or nothing), so no reader waits
// for a writer and a step that is repeated gives the same result. With codes c, pairs (s, m):
//   score_j = scale (s_j sum_e q_e c_je + m_j sum_e q_e)
//   o_e     = sum_j P_j (s'_j c'_je + m'_j) / sum_j P_j = [sum_j (P_j s'_j) c'_je + sum_j P_j m'_j] / sum_j P_j
// so both products run on the codes themselves and each pair is applied once a token and query head.
// Both are MFMA products (16x16x32), scores formed transposed, S^T = K q^T, so that a lane holds one
// query head's scores of eight tokens, which is the operand layout that O^T = V^T P^T takes: the softmax
// weights go from one product to the next in registers. Codes become bf16 by setting the exponent of
// 128 above the four bits (128 + c is exact in bf16), two codes an instruction; the 128 is taken out with
// the sums (128 sum q, and a product with a row of 128s that gives 128 sum P s'). With fp16 queries the
// scores' codes are 1024 + c less 1024 in fp16, also exact. A group has at most eight query heads and the
// tile sixteen columns, so the columns hold each head twice: P s' rounded to bf16 in the first eight and
// the rest of it, rounded again, in the others, together 16 bits of it. Sums, maxima and weights are
// float32; the running maximum is raised only when a tile's exceeds it by more than 8 (weights up to 2^8
// are as exact), so the accumulators are rarely rescaled.
#include <type_traits>

#include "common.h"
#include "ring4.h"
#include "vesper_kernels.h"

namespace vsp {
namespace {

constexpr int kQuantMaxGroup = 8;
constexpr int kTile = 32;       // tokens a wave takes at a time
constexpr int kAttnWaves = 4;   // waves a workgroup
constexpr float kRaise = 8.f;   // log2: how far a tile's maximum may exceed the running one

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ---- writing and reading ------------------------------------------------------------------------
// L lanes a row of eight features each; a workgroup takes 256 / L tokens of one head, keys or values, so
// the ring's side is contiguous and the tokens' side whole rows of dk elements. The heads of the same
// tokens are consecutive workgroups of one XCD (short rows share their cache lines there).
template <typename T, int L>
__global__ __launch_bounds__(256) void quant_write_kernel(const T* __restrict__ k, const T* __restrict__ v,
                                                          const int64_t* __restrict__ pos,
                                                          const int64_t* __restrict__ lengths, uint32_t* ring_k,
                                                          uint32_t* ring_v, uint32_t* k_scale, uint32_t* v_scale,
                                                          int64_t* ring_pos, uint8_t* ring_valid, int B, int N, int HKV,
                                                          int dk, int W, int blocks) {
  constexpr int TB = 256 / L;
  const int lg = xcd_logical_block(blockIdx.x, gridDim.x);
  const int head2 = lg % (2 * HKV), rest = lg / (2 * HKV);
  const int b = rest / blocks, tb = rest - b * blocks;
  const int head = head2 >> 1;
  const bool values = (head2 & 1) != 0;
  const int part = threadIdx.x % L, t = tb * TB + (int)threadIdx.x / L;
  const int len = lengths == nullptr ? N : (int)min(max(lengths[b], (int64_t)0), (int64_t)N);
  const int i = max(len - W, 0) + t;  // the last W tokens of the row are the ones that stay
  if (i >= len) return;               // whole rows of lanes leave together
  const int64_t p = pos[(size_t)b * N + i];
  if (p < 0) return;  // refused by the host wrapper
  const int slot = (int)(p % W);
  const bool live = 8 * part < dk;
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = 0.f;
  if (live) load8_f32((values ? v : k) + (((size_t)b * N + i) * HKV + head) * dk + 8 * part, x);
  uint32_t pair;
  const uint32_t codes = quantize_row8<T, L>(x, live, pair);
  const size_t row = ((size_t)b * HKV + head) * W + slot;
  if (live) (values ? ring_v : ring_k)[row * (size_t)(dk / 8) + part] = codes;
  if (part == 0) {
    (values ? v_scale : k_scale)[row] = pair;
    if (head2 == 0) {
      ring_pos[(size_t)b * W + slot] = p;
      ring_valid[(size_t)b * W + slot] = 1;
    }
  }
}

template <typename T, int L>
__global__ __launch_bounds__(256) void quant_read_kernel(const uint32_t* __restrict__ ring_k,
                                                         const uint32_t* __restrict__ ring_v,
                                                         const uint32_t* __restrict__ k_scale,
                                                         const uint32_t* __restrict__ v_scale,
                                                         const int64_t* __restrict__ ring_pos,
                                                         const uint8_t* __restrict__ ring_valid,
                                                         const int64_t* __restrict__ pos, T* __restrict__ k,
                                                         T* __restrict__ v, uint8_t* __restrict__ found, int B, int N,
                                                         int HKV, int dk, int W, int blocks) {
  typedef T V8 __attribute__((ext_vector_type(8)));
  constexpr int TB = 256 / L;
  const int lg = xcd_logical_block(blockIdx.x, gridDim.x);
  const int head2 = lg % (2 * HKV), rest = lg / (2 * HKV);
  const int b = rest / blocks, tb = rest - b * blocks;
  const int head = head2 >> 1;
  const bool values = (head2 & 1) != 0;
  const int part = threadIdx.x % L, i = tb * TB + (int)threadIdx.x / L;
  if (i >= N) return;
  const int64_t p = pos[(size_t)b * N + i];
  const int slot = p < 0 ? 0 : (int)(p % W);
  const size_t at = (size_t)b * W + slot;
  const bool here = p >= 0 && ring_valid[at] != 0 && ring_pos[at] == p;
  const size_t row = ((size_t)b * HKV + head) * W + slot;
  if (8 * part < dk) {
    V8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = from_f32<T>(0.f);
    if (here)
      y = dequantize_row8<T, V8>((values ? ring_v : ring_k)[row * (size_t)(dk / 8) + part],
                                 (values ? v_scale : k_scale)[row]);
    *reinterpret_cast<V8*>((values ? v : k) + (((size_t)b * N + i) * HKV + head) * dk + 8 * part) = y;
  }
  if (head2 == 0 && part == 0) found[(size_t)b * N + i] = here ? 1 : 0;
}

// ---- attention ----------------------------------------------------------------------------------
// The codes of a dword as eight elements, in the order 0 4 1 5 2 6 3 7 of the features.
template <typename T> struct Codes;
template <> struct Codes<__bf16> {
  static constexpr float kBias = 128.f;  // 0x4300 | c is 128 + c
  typedef bf16x8 V8;
  __device__ __forceinline__ static V8 unpack(uint32_t w) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
    return __builtin_bit_cast(V8, r);
  }
  __device__ __forceinline__ static f32x4 mma(V8 a, V8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Codes<_Float16> {
  static constexpr float kBias = 0.f;
  typedef f16x8 V8;
  __device__ __forceinline__ static V8 unpack(uint32_t w) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f16x2 x = __builtin_bit_cast(f16x2, ((w >> (4 * i)) & 0x000f000fu) | 0x64006400u);  // 1024 + c
      r[i] = __builtin_bit_cast(uint32_t, x - f16x2{(_Float16)1024.f, (_Float16)1024.f});
    }
    return __builtin_bit_cast(V8, r);
  }
  __device__ __forceinline__ static f32x4 mma(V8 a, V8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
// the k-th feature of a dword's eight in Codes<T>'s order
__device__ __forceinline__ constexpr int code_feature(int k) { return (k >> 1) + 4 * (k & 1); }

// Buffer loads of 1 to 16 bytes a lane; past the resource's range they give zeros.
__device__ __forceinline__ uint32_t load_b8(__amdgpu_buffer_rsrc_t r, unsigned off) {
  return (uint32_t)(uint8_t)__builtin_amdgcn_raw_buffer_load_b8(r, (int)off, 0, 0);
}
__device__ __forceinline__ uint32_t load_b16(__amdgpu_buffer_rsrc_t r, unsigned off) {
  return (uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, (int)off, 0, 0);
}
// WHOLE: every piece of N dwords that starts in the range ends in it; else dword by dword.
template <int N, bool WHOLE>
__device__ __forceinline__ void load_dwords(__amdgpu_buffer_rsrc_t r, unsigned off, uint32_t (&out)[N]) {
  if constexpr (N == 1 || !WHOLE) {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, (int)(off + 4 * i), 0, 0);
  } else if constexpr (N == 2) {
    const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, (int)off, 0, 0));
    out[0] = x[0];
    out[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const u32x4 x = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)(off + 4 * i), 0, 0));
#pragma unroll
      for (int e = 0; e < 4; ++e) out[i + e] = x[e];
    }
  }
}

// The largest of x over the lanes l, l ^ 16, l ^ 32, l ^ 48 (a column of an MFMA result).
__device__ __forceinline__ float max_over_rows(float x) {
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __builtin_fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
  const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __builtin_fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}

struct QuantAttnArgs {
  const int64_t* pos;
  uint32_t* ring_k;
  uint32_t* ring_v;
  uint32_t* k_scale;
  uint32_t* v_scale;
  int64_t* ring_pos;
  uint8_t* ring_valid;
  const uint8_t* active;
  float* partial;  // [B, H, splits, 2 + dk] softmax states, with more than one split
  int B, H, HKV, dk, W, splits, write;
  float scale_log2;
};

// One workgroup: the query heads of one KV head of one row over one of `splits` runs of tiles of 32
// slots, its waves taking the tiles in turn. NS: the head width in units of 32, rounded up to a power of two.
// Lane (c, g) = (l % 16, l / 16). K tile: lane holds dwords g NS .. + NS of the codes of tokens c and
// 16 + c. V tile: lane holds features c M .. + M of tokens 4 g + i and 16 + 4 g + i (i = 0..3), M = 2 NS,
// which are the tokens whose scores it holds; its M accumulators hold features (4 g + r) M + e, r = 0..3.
// Features past dk: K's meet zeros of q, V's are not stored; both lie inside the ring or read as zero.
// WHOLE: dk is a whole number of lanes' pieces (NS dwords), so no piece reaches past the ring's end.
template <typename T, int NS, bool WHOLE>
__global__ __launch_bounds__(64 * kAttnWaves) void quant_attn_kernel(const T* __restrict__ q, const T* __restrict__ knew,
                                                                     const T* __restrict__ vnew, T* __restrict__ o,
                                                                     const QuantAttnArgs a) {
  constexpr int DP = 32 * NS, M = 2 * NS;
  constexpr int NW = kAttnWaves;
  constexpr int VD = M <= 8 ? 1 : M / 8;  // dwords of a lane's piece of a V row
  using C = Codes<T>;
  typedef T V8 __attribute__((ext_vector_type(8)));
  __shared__ __align__(16) float2 stage[NW][2][kTile];  // the tile's pairs as the products take them
  __shared__ float smerge[NW][kQuantMaxGroup][2 + DP];

  const int lg = xcd_logical_block(blockIdx.x, gridDim.x);
  const int kvh = lg % a.HKV, rest = lg / a.HKV;
  const int b = rest / a.splits, split = rest - b * a.splits;
  const int G = a.H / a.HKV, dk = a.dk, W = a.W;
  const int tid = threadIdx.x, l = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), c = l & 15, g = l >> 4;
  const int64_t p = a.pos[b];
  const int slot = p < 0 ? -1 : (int)(p % W);
  const size_t head = (size_t)b * a.HKV + kvh;
  const unsigned rb = (unsigned)dk / 2;  // bytes a row
  const __amdgpu_buffer_rsrc_t rk = buffer_rsrc(a.ring_k + head * W * (dk / 8), (unsigned)W * rb);
  const __amdgpu_buffer_rsrc_t rv = buffer_rsrc(a.ring_v + head * W * (dk / 8), (unsigned)W * rb);
  const uint32_t* pairs = (l < 32 ? a.k_scale : a.v_scale) + head * W;

  // the group's queries: column c holds head c % 8 (columns of heads past G are zero and never stored)
  const int hd = c & 7;
  const bool has = hd < G;
  const size_t qrow = (size_t)b * a.H + (size_t)kvh * G + (has ? hd : 0);
  V8 qf[NS];
  float qsum = 0.f, fresh = 0.f;  // the sum of the query's features, and its product with the new key
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const int f0 = 8 * (g * NS + s);
    V8 x, kn;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = kn[e] = from_f32<T>(0.f);
    if (f0 < dk) {
      if (has) x = *reinterpret_cast<const V8*>(q + qrow * dk + f0);
      kn = *reinterpret_cast<const V8*>(knew + head * dk + f0);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      qf[s][e] = x[code_feature(e)];
      qsum += to_f32(x[e]);
      fresh += to_f32(x[e]) * to_f32(kn[e]);
    }
  }
  qsum = sum_over_rows(qsum);
  fresh = sum_over_rows(fresh) * a.scale_log2;

  float m = -1e30f, lsum = 0.f, low = 0.f;  // the running maximum, the lane's sums of P and of P m'
  f32x4 acc[M], bias = zero4();
#pragma unroll
  for (int e = 0; e < M; ++e) acc[e] = zero4();
  if (split == 0 && w == 0) {  // the new token starts the first wave's state
    m = fresh;
    lsum = g == 0 ? 1.f : 0.f;
    if (c < 8) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < M; ++e) {
          const int f = (4 * g + r) * M + e;
          if (f < dk) acc[e][r] = to_f32(vnew[head * dk + f]);
        }
    }
  }
  const float second = c < 8 ? 0.f : 1.f;
  bf16x8 ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = (__bf16)128.f;

  const int tiles = (W + kTile - 1) / kTile;
  const int first = (int)((int64_t)tiles * split / a.splits), last = (int)((int64_t)tiles * (split + 1) / a.splits);
  for (int t = first + w; t < last; t += NW) {
    const int j0 = kTile * t;
    // the tile's loads
    const int js = j0 + (l & 31), jc = min(js, W - 1);
    const uint32_t pair = pairs[jc];
    const int64_t rp = a.ring_pos[(size_t)b * W + jc];
    const uint8_t flag = a.ring_valid[(size_t)b * W + jc];
    uint32_t kc[2][NS], vc[8][VD];
#pragma unroll
    for (int u = 0; u < 2; ++u) load_dwords<NS, WHOLE>(rk, (unsigned)(j0 + 16 * u + c) * rb + 4u * NS * (unsigned)g, kc[u]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned off = (unsigned)(j0 + 4 * g + (i & 3) + 16 * (i >> 2)) * rb + (unsigned)(c * NS);
      if constexpr (M == 2) vc[i][0] = load_b8(rv, off);
      else if constexpr (M == 4) vc[i][0] = load_b16(rv, off);
      else load_dwords<VD, WHOLE>(rv, off, vc[i]);
    }
    // which tokens are seen, and their pairs: lanes 0..31 the keys', 32..63 the values'
    const bool seen = js < W && flag != 0 && rp <= p && rp > p - W && js != slot && p >= 0;
    const uint32_t mask = (uint32_t)__ballot(seen);
    if (mask == 0) continue;
    const float ps = pair_scale<T>(pair), pl = pair_low<T>(pair);
    float2 st;
    if (l < 32) st = make_float2(ps * a.scale_log2, (pl - C::kBias * ps) * a.scale_log2);
    else st = seen ? make_float2(ps, pl) : make_float2(0.f, 0.f);  // no NaN of an unseen slot meets a zero weight
    __builtin_amdgcn_wave_barrier();
    stage[w][l >> 5][l & 31] = st;
    __builtin_amdgcn_wave_barrier();
    // scores of the lane's eight tokens: 4 g + i in the first tile of 16, then 16 + 4 g + i
    float sc[8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f32x4 d = zero4();
#pragma unroll
      for (int s = 0; s < NS; ++s) d = C::mma(C::unpack(kc[u][s]), qf[s], d);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 ab = stage[w][0][16 * u + 4 * g + i];
        sc[4 * u + i] = ab.x * d[i] + ab.y * qsum;
      }
    }
    if (mask != 0xffffffffu) {
      const uint32_t mine = mask >> (4 * g);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (((mine >> ((i & 3) + 16 * (i >> 2))) & 1u) == 0) sc[i] = -kInf;
    }
    float top = sc[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = __builtin_fmaxf(top, sc[i]);
    top = max_over_rows(top);
    if (__ballot(top > m + kRaise) != 0) {
      const float mn = __builtin_fmaxf(m, top);
      const float f = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      lsum *= f;
      low *= f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        bias[r] *= f;
#pragma unroll
        for (int e = 0; e < M; ++e) acc[e][r] *= f;
      }
    }
    // weights, and the weights times the values' scales as two bf16 parts over the column halves
    bf16x8 pv;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 ab = stage[w][1][16 * (i >> 2) + 4 * g + (i & 3)];
      const float pj = __builtin_amdgcn_exp2f(sc[i] - m);
      lsum += pj;
      low = __builtin_fmaf(pj, ab.y, low);
      const float x = pj * ab.x;
      pv[i] = (__bf16)__builtin_fmaf(-second, (float)(__bf16)x, x);
    }
    bias = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pv, bias, 0, 0, 0);
    // pairs of tokens' codes of one feature: 16 bits a token and four features
    constexpr int PIECES = M <= 4 ? 1 : M / 4, PER = M <= 4 ? M : 4;
#pragma unroll
    for (int h = 0; h < PIECES; ++h) {
      uint32_t two[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t x = vc[2 * i][h / 2], y = vc[2 * i + 1][h / 2];
        two[i] = M <= 4 ? (x | (y << 16)) : (h & 1) == 0 ? ((x & 0xffffu) | (y << 16)) : ((x >> 16) | (y & 0xffff0000u));
      }
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = ((two[i] >> (4 * e)) & 0x000f000fu) | 0x43004300u;
        acc[4 * h + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, r), pv, acc[4 * h + e], 0, 0, 0);
      }
    }
  }

  // the wave's state: sums over the lane groups, the two parts of P s' joined (column c and c + 8)
  lsum = sum_over_rows(lsum);
  low = sum_over_rows(low);
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int e = 0; e < M; ++e) {
      float x = acc[e][r] - bias[r];
      x += dpp_f32<0x128>(x);  // row_ror:8
      if (c < G && (4 * g + r) * M + e < dk) smerge[w][c][2 + (4 * g + r) * M + e] = x + low;
    }
  if (g == 0 && c < G) {
    smerge[w][c][0] = m;
    smerge[w][c][1] = lsum;
  }
  __syncthreads();
  const bool on = a.active == nullptr || a.active[b] != 0;
  for (int i = tid; i < G * dk; i += 64 * NW) {
    const int gi = i / dk, d = i - gi * dk;
    float mx = smerge[0][gi][0];
#pragma unroll
    for (int u = 1; u < NW; ++u) mx = __builtin_fmaxf(mx, smerge[u][gi][0]);
    float ls = 0.f, num = 0.f;
#pragma unroll
    for (int u = 0; u < NW; ++u) {
      const float f = __builtin_amdgcn_exp2f(smerge[u][gi][0] - mx);
      ls += smerge[u][gi][1] * f;
      num += smerge[u][gi][2 + d] * f;
    }
    const size_t row = (size_t)b * a.H + (size_t)kvh * G + gi;
    if (a.splits == 1) {
      o[row * dk + d] = from_f32<T>(on ? num / ls : 0.f);
    } else {
      float* part = a.partial + (row * a.splits + split) * (size_t)(2 + dk);
      part[2 + d] = num;
      if (d == 0) {
        part[0] = mx;
        part[1] = ls;
      }
    }
  }

  // The new token into its slot, which no workgroup attends (a reader of its codes drops them).
  if (!a.write || split != 0 || p < 0) return;
  constexpr int L = DP / 8;
  if (w < 2 && l < L) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
    const bool live = 8 * l < dk;
    if (live) load8_f32((w == 0 ? knew : vnew) + head * dk + 8 * l, x);
    uint32_t pr;
    const uint32_t codes = quantize_row8<T, L>(x, live, pr);
    const size_t row = head * W + slot;
    if (live) (w == 0 ? a.ring_k : a.ring_v)[row * (size_t)(dk / 8) + l] = codes;
    if (l == 0) {
      (w == 0 ? a.k_scale : a.v_scale)[row] = pr;
      if (w == 0 && kvh == 0) {
        a.ring_pos[(size_t)b * W + slot] = p;
        a.ring_valid[(size_t)b * W + slot] = 1;
      }
    }
  }
}

// The splits' softmax states of one query head joined, in the splits' order.
template <typename T>
__global__ __launch_bounds__(256) void quant_join_kernel(const float* __restrict__ partial, T* __restrict__ o,
                                                         const uint8_t* __restrict__ active, int H, int dk, int splits) {
  const size_t row = blockIdx.x;
  const float* part = partial + row * splits * (size_t)(2 + dk);
  const bool on = active == nullptr || active[row / H] != 0;
  float mx = part[0];
  for (int s = 1; s < splits; ++s) mx = __builtin_fmaxf(mx, part[(size_t)s * (2 + dk)]);
  for (int d = threadIdx.x; d < dk; d += 256) {
    float ls = 0.f, num = 0.f;
    for (int s = 0; s < splits; ++s) {
      const float* x = part + (size_t)s * (2 + dk);
      const float f = __builtin_amdgcn_exp2f(x[0] - mx);
      ls += x[1] * f;
      num += x[2 + d] * f;
    }
    o[row * dk + d] = from_f32<T>(on ? num / ls : 0.f);
  }
}

// ---- host side ----------------------------------------------------------------------------------

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// The sizes every entry shares; 0 or an error.
int quant_sizes(int B, int HKV, int D, int W, const char* who) {
  if (B < 0 || HKV < 1 || W < 1) return fail(ERR_ARG, "%s: bad sizes B=%d HKV=%d W=%d", who, B, HKV, W);
  if (D < 8 || D > 256 || D % 8 != 0)
    return fail(ERR_UNSUPPORTED, "%s: head dimension %d (kernels: multiples of 8 up to 256)", who, D);
  if ((int64_t)(W + (int64_t)kTile) * (D / 2) >= ((int64_t)1 << 31))
    return fail(ERR_UNSUPPORTED, "%s: a head's window of %d slots of %d bytes over 2 GiB", who, W, D / 2);
  return OK;
}

int lanes_of(int D) { return D <= 8 ? 1 : D <= 16 ? 2 : D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32; }

// Runs f with the lanes a row takes as a compile-time number.
template <typename F> void by_lanes(int D, F f) {
  switch (lanes_of(D)) {
    case 1: f(std::integral_constant<int, 1>{}); break;
    case 2: f(std::integral_constant<int, 2>{}); break;
    case 4: f(std::integral_constant<int, 4>{}); break;
    case 8: f(std::integral_constant<int, 8>{}); break;
    case 16: f(std::integral_constant<int, 16>{}); break;
    default: f(std::integral_constant<int, 32>{}); break;
  }
}

template <typename T>
int quant_write(const T* k, const T* v, const int64_t* pos, const int64_t* lengths, void* ring_k, void* ring_v,
                void* k_scale, void* v_scale, int64_t* ring_pos, uint8_t* ring_valid, int B, int N, int HKV, int D,
                int W, void* stream, const char* who) {
  const int st = quant_sizes(B, HKV, D, W, who);
  if (st != OK) return st;
  if (N < 0) return fail(ERR_ARG, "%s: N=%d", who, N);
  if (B == 0 || N == 0) return OK;
  if (!k || !v || !pos || !ring_k || !ring_v || !k_scale || !v_scale || !ring_pos || !ring_valid)
    return fail(ERR_ARG, "%s: null pointer", who);
  if (!aligned(k, 16) || !aligned(v, 16)) return fail(ERR_ARG, "%s: k and v must be 16-byte aligned", who);
  if (!aligned(ring_k, 4) || !aligned(ring_v, 4) || !aligned(k_scale, 4) || !aligned(v_scale, 4))
    return fail(ERR_ARG, "%s: the ring's tensors must be 4-byte aligned", who);
  const int tb = 256 / lanes_of(D), blocks = ((N < W ? N : W) + tb - 1) / tb;
  const int64_t grid = (int64_t)B * blocks * 2 * HKV;
  if (grid >= ((int64_t)1 << 31)) return fail(ERR_UNSUPPORTED, "%s: %lld workgroups", who, (long long)grid);
  by_lanes(D, [&](auto lanes) {
    hipLaunchKernelGGL((quant_write_kernel<T, decltype(lanes)::value>), dim3((unsigned)grid), dim3(256), 0,
                       reinterpret_cast<hipStream_t>(stream), k, v, pos, lengths, static_cast<uint32_t*>(ring_k),
                       static_cast<uint32_t*>(ring_v), static_cast<uint32_t*>(k_scale), static_cast<uint32_t*>(v_scale),
                       ring_pos, ring_valid, B, N, HKV, D, W, blocks);
  });
  return check_launch(who);
}

template <typename T>
int quant_read(const void* ring_k, const void* ring_v, const void* k_scale, const void* v_scale,
               const int64_t* ring_pos, const uint8_t* ring_valid, const int64_t* pos, T* k, T* v, uint8_t* found, int B,
               int N, int HKV, int D, int W, void* stream, const char* who) {
  const int st = quant_sizes(B, HKV, D, W, who);
  if (st != OK) return st;
  if (N < 0) return fail(ERR_ARG, "%s: N=%d", who, N);
  if (B == 0 || N == 0) return OK;
  if (!k || !v || !pos || !ring_k || !ring_v || !k_scale || !v_scale || !ring_pos || !ring_valid || !found)
    return fail(ERR_ARG, "%s: null pointer", who);
  if (!aligned(k, 16) || !aligned(v, 16)) return fail(ERR_ARG, "%s: k and v must be 16-byte aligned", who);
  if (!aligned(ring_k, 4) || !aligned(ring_v, 4) || !aligned(k_scale, 4) || !aligned(v_scale, 4))
    return fail(ERR_ARG, "%s: the ring's tensors must be 4-byte aligned", who);
  const int tb = 256 / lanes_of(D), blocks = (int)(((int64_t)N + tb - 1) / tb);
  const int64_t grid = (int64_t)B * blocks * 2 * HKV;
  if (grid >= ((int64_t)1 << 31)) return fail(ERR_UNSUPPORTED, "%s: %lld workgroups", who, (long long)grid);
  by_lanes(D, [&](auto lanes) {
    hipLaunchKernelGGL((quant_read_kernel<T, decltype(lanes)::value>), dim3((unsigned)grid), dim3(256), 0,
                       reinterpret_cast<hipStream_t>(stream), static_cast<const uint32_t*>(ring_k),
                       static_cast<const uint32_t*>(ring_v), static_cast<const uint32_t*>(k_scale),
                       static_cast<const uint32_t*>(v_scale), ring_pos, ring_valid, pos, k, v, found, B, N, HKV, D, W,
                       blocks);
  });
  return check_launch(who);
}

// How many workgroups share a head's window: enough that the card's 256 CUs have four each, and no more
// than there are tiles for their waves.
int attn_splits(int B, int HKV, int W) {
  const int64_t heads = (int64_t)B * HKV;
  const int tiles = (W + kTile - 1) / kTile, most = (tiles + kAttnWaves - 1) / kAttnWaves;
  const int64_t want = heads >= 1024 ? 1 : (1024 + heads - 1) / heads;
  return (int)(want < most ? want : most);
}

size_t attn_workspace(int B, int H, int HKV, int D, int W) {
  const int splits = attn_splits(B, HKV, W);
  return splits == 1 ? 0 : (size_t)B * H * splits * (2 + D) * sizeof(float);
}

template <typename T>
int quant_attn(const T* q, const T* knew, const T* vnew, const int64_t* pos, void* ring_k, void* ring_v, void* k_scale,
               void* v_scale, int64_t* ring_pos, uint8_t* ring_valid, T* o, const uint8_t* active, void* workspace,
               size_t ws_bytes, int B, int H, int HKV, int D, int W, float scale, int write, void* stream_ptr,
               const char* who) {
  const int st = quant_sizes(B, HKV, D, W, who);
  if (st != OK) return st;
  if (H < 1 || H % HKV != 0) return fail(ERR_ARG, "%s: %d query heads are not a multiple of %d KV heads", who, H, HKV);
  if (H / HKV > kQuantMaxGroup)
    return fail(ERR_UNSUPPORTED, "%s: %d query heads per KV head (at most %d)", who, H / HKV, kQuantMaxGroup);
  if (B == 0) return OK;
  if (!q || !knew || !vnew || !pos || !ring_k || !ring_v || !k_scale || !v_scale || !ring_pos || !ring_valid || !o)
    return fail(ERR_ARG, "%s: null pointer", who);
  if (!aligned(q, 16) || !aligned(knew, 16) || !aligned(vnew, 16))
    return fail(ERR_ARG, "%s: q, k and v must be 16-byte aligned", who);
  if (!aligned(ring_k, 4) || !aligned(ring_v, 4) || !aligned(k_scale, 4) || !aligned(v_scale, 4))
    return fail(ERR_ARG, "%s: the ring's tensors must be 4-byte aligned", who);
  const int splits = attn_splits(B, HKV, W);
  const size_t need = attn_workspace(B, H, HKV, D, W);
  if (need > 0 && (workspace == nullptr || ws_bytes < need || !aligned(workspace, 4)))
    return fail(ERR_ARG, "%s: workspace of %zu bytes given, %zu needed", who, workspace ? ws_bytes : (size_t)0, need);
  const int64_t grid = (int64_t)B * HKV * splits;
  if (grid >= ((int64_t)1 << 31) || (int64_t)B * H >= ((int64_t)1 << 31))
    return fail(ERR_UNSUPPORTED, "%s: %lld workgroups", who, (long long)grid);
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_ptr);
  const QuantAttnArgs a{pos, static_cast<uint32_t*>(ring_k), static_cast<uint32_t*>(ring_v),
                        static_cast<uint32_t*>(k_scale), static_cast<uint32_t*>(v_scale), ring_pos, ring_valid, active,
                        static_cast<float*>(workspace), B, H, HKV, D, W, splits, write,
                        scale * 1.4426950408889634f};
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64 * kAttnWaves), 0, stream, q, knew, vnew, o, a);
  };
  if (D <= 32) go(quant_attn_kernel<T, 1, true>);
  else if (D <= 64) D % 16 == 0 ? go(quant_attn_kernel<T, 2, true>) : go(quant_attn_kernel<T, 2, false>);
  else if (D <= 128) D % 32 == 0 ? go(quant_attn_kernel<T, 4, true>) : go(quant_attn_kernel<T, 4, false>);
  else D % 64 == 0 ? go(quant_attn_kernel<T, 8, true>) : go(quant_attn_kernel<T, 8, false>);
  if (splits > 1)
    hipLaunchKernelGGL(quant_join_kernel<T>, dim3((unsigned)(B * H)), dim3(256), 0, stream,
                       static_cast<const float*>(workspace), o, active, H, D, splits);
  return check_launch(who);
}

}  // namespace
}  // namespace vsp

#define VSP_QUANT_RING(SUFFIX, T)                                                                                      \
  extern "C" int vsp_quant_ring_write_##SUFFIX(const void* k, const void* v, const int64_t* pos, const int64_t* lengths,   \
                                               void* ring_k, void* ring_v, void* k_scale, void* v_scale,               \
                                               int64_t* ring_pos, uint8_t* ring_valid, int B, int N, int HKV, int D,   \
                                               int window, void* stream) {                                             \
    return vsp::quant_write<T>(static_cast<const T*>(k), static_cast<const T*>(v), pos, lengths, ring_k, ring_v,       \
                               k_scale, v_scale, ring_pos, ring_valid, B, N, HKV, D, window, stream,                   \
                               "vsp_quant_ring_write_" #SUFFIX);                                                       \
  }                                                                                                                    \
  extern "C" int vsp_quant_ring_read_##SUFFIX(                                                                         \
      const void* ring_k, const void* ring_v, const void* k_scale, const void* v_scale, const int64_t* ring_pos,       \
      const uint8_t* ring_valid, const int64_t* pos, void* k, void* v, uint8_t* found, int B, int N, int HKV, int D,   \
      int window, void* stream) {                                                                                      \
    return vsp::quant_read<T>(ring_k, ring_v, k_scale, v_scale, ring_pos, ring_valid, pos, static_cast<T*>(k),         \
                              static_cast<T*>(v), found, B, N, HKV, D, window, stream, "vsp_quant_ring_read_" #SUFFIX); \
  }                                                                                                                    \
  extern "C" int vsp_quant_ring_attn_##SUFFIX(                                                                         \
      const void* q, const void* k, const void* v, const int64_t* pos, void* ring_k, void* ring_v, void* k_scale,      \
      void* v_scale, int64_t* ring_pos, uint8_t* ring_valid, void* o, const uint8_t* active, void* workspace,          \
      size_t workspace_bytes, int B, int H, int HKV, int D, int window, float scale, int write, void* stream) {        \
    return vsp::quant_attn<T>(static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v), pos,       \
                              ring_k, ring_v, k_scale, v_scale, ring_pos, ring_valid, static_cast<T*>(o), active,      \
                              workspace, workspace_bytes, B, H, HKV, D, window, scale, write, stream,                  \
                              "vsp_quant_ring_attn_" #SUFFIX);                                                         \
  }
VSP_QUANT_RING(bf16, __bf16)
VSP_QUANT_RING(f16, _Float16)

extern "C" size_t vsp_quant_ring_attn_workspace_bytes(int B, int H, int HKV, int D, int window) {
  if (B < 1 || H < 1 || HKV < 1 || D < 1 || window < 1) return 0;
  return vsp::attn_workspace(B, H, HKV, D, window);
}
