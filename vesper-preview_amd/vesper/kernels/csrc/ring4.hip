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
// 128 above the four bits (128 + c is exact in bf16), two codes an instruction; the 128 is taken out in
// the sums (the scores' begin at -128 sum q, which with the scales applied would overflow for keys past 2^121; a product
// with a row of 128s gives 128 sum P s'). With fp16 queries the
// scores' codes are 1024 + c less 1024 in fp16, also exact. A group has at most eight query heads and the
// tile sixteen columns, so the columns hold each head twice: P s' rounded to bf16 in the first eight and
// the rest of it, rounded again, in the others, together 16 bits of it. Sums, maxima and weights are
// float32; the running maximum is raised only when a tile's exceeds it by more than 8 (weights up to 2^8
// are as exact), so the accumulators are rarely rescaled. It is also raised where the values are so large (past 2^72)
// that the sums would overflow: the output then is finite as the values are, unless scores past 2^29 meet them.
//
// Bound by HBM where the ring is long: 8 rows of 65536 slots, four heads of 128 (290 MB): 58.5 us, 5.0 TB/s, and 4.7
// for the join. Short windows are a launch and a wave's chain of loads: 64 rows of 512 slots, 8 heads of 64: 9.7 us,
// 4.8 with nothing to attend. Writing 7 ragged rows of 4097 tokens (8 heads of 64): 16.8 us (14.0 at best), reading them
// back 17.4 (16.3); a bare copy of the write's pattern takes 10.4.
#include <type_traits>

#include "common.h"
#include "ring4.h"
#include "vesper_kernels.h"

namespace vsp {
namespace {

constexpr int kQuantMaxGroup = 8;
constexpr int kTile = 32;       // tokens a wave takes at a time
constexpr int kMaxSplits = 256;  // workgroups that share a window (one thread each in the join)
constexpr int64_t kMaxThreads = (int64_t)1 << 32;  // a launch has fewer
constexpr float kRaise = 8.f;   // log2: how far a tile's maximum may exceed the running one
// Sums of weights up to 2^8 times 143 scales, over at most 2^29 slots, stay below 2^128 while no pair of the values
// exceeds kLargePair. A wave that has met one that does keeps its running maximum kHeadroom (log2) above the scores, so
// that its weights, of which only the ratios count, and its sums are 2^64 times smaller.
constexpr float kLargePair = 0x1p72f, kHeadroom = 64.f;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ---- writing and reading ------------------------------------------------------------------------
// L lanes a row of eight features each, key and value of a token by the same lanes; a workgroup takes 256 / L
// tokens of one head, so the ring's side is contiguous and the tokens' side whole rows of dk elements. The heads
// of the same tokens are consecutive workgroups of one XCD (short rows share their cache lines there). What is
// left is the arithmetic a row (the slot's division by W and the indices), so a lane group takes both rows.
// slot of a position >= 0: most fit 32 bits, where the division is a fraction of the 64-bit one
__device__ __forceinline__ int slot_of(int64_t p, int W) {
  return (uint64_t)p >> 32 == 0 ? (int)((uint32_t)p % (uint32_t)W) : (int)(p % W);
}

template <typename T, int L>
__global__ __launch_bounds__(256) void quant_write_kernel(const T* __restrict__ k, const T* __restrict__ v,
                                                          const int64_t* __restrict__ pos,
                                                          const int64_t* __restrict__ lengths, uint32_t* ring_k,
                                                          uint32_t* ring_v, uint32_t* k_scale, uint32_t* v_scale,
                                                          int64_t* ring_pos, uint8_t* ring_valid, int B, int N, int HKV,
                                                          int dk, int W, int blocks) {
  constexpr int TB = 256 / L;
  const unsigned lg = (unsigned)xcd_logical_block(blockIdx.x, gridDim.x);
  const unsigned head = lg % (unsigned)HKV, rest = lg / (unsigned)HKV;
  const unsigned b = rest / (unsigned)blocks, tb = rest - b * (unsigned)blocks;
  const unsigned part = threadIdx.x % L, t = threadIdx.x / L;
  const int len = lengths == nullptr ? N : (int)min(max(lengths[b], (int64_t)0), (int64_t)N);
  const int kept = min(len, W), i0 = (int)tb * TB;  // the last W tokens of the row are the ones that stay
  if ((int)t >= kept - i0) return;                  // whole rows of lanes leave together
  const size_t token = (size_t)b * N + (len - kept) + i0;  // the workgroup's first; lanes add 32-bit offsets
  const int64_t p = pos[token];                   // positions go up by one: the first gives all
  const bool live = (int)(8 * part) < dk;
  float xk[8], xv[8];
  const size_t base = (token * HKV + head) * dk;
  const unsigned at = t * (unsigned)(HKV * dk) + (live ? 8 * part : 0u);
  load8_f32(k + base + at, xk);
  load8_f32(v + base + at, xv);
  if (p < 0) return;  // refused by the host wrapper
  unsigned slot = (unsigned)slot_of(p, W) + t;  // t is below W, as tokens past it are not kept
  if (slot >= (unsigned)W) slot -= (unsigned)W;
  const size_t first = ((size_t)b * HKV + head) * W;  // the head's rows
  uint32_t pk, pv;
  const uint32_t ck = quantize_row8<T, L>(xk, pk), cv = quantize_row8<T, L>(xv, pv);
  if (live) {
    const unsigned to = slot * (unsigned)(dk / 8) + part;
    (ring_k + first * (dk / 8))[to] = ck;
    (ring_v + first * (dk / 8))[to] = cv;
  }
  if (part == 0) {
    (k_scale + first)[slot] = pk;
    (v_scale + first)[slot] = pv;
    if (head == 0) {
      ring_pos[(size_t)b * W + slot] = p + t;
      ring_valid[(size_t)b * W + slot] = 1;
    }
  }
}

constexpr int kReadTokens = 2;  // tokens a lane group of the read takes
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
  constexpr int TB = 256 / L, R = kReadTokens;
  const unsigned lg = (unsigned)xcd_logical_block(blockIdx.x, gridDim.x);
  const unsigned head = lg % (unsigned)HKV, rest = lg / (unsigned)HKV;
  const unsigned b = rest / (unsigned)blocks, tb = rest - b * (unsigned)blocks;
  const unsigned part = threadIdx.x % L, t0 = threadIdx.x / L;
  const size_t token = (size_t)b * N + tb * (R * TB);  // the workgroup's first; lanes add 32-bit offsets
  const int left = N - (int)(tb * (R * TB));
  const size_t first = ((size_t)b * HKV + head) * W;  // the head's rows
  const bool live = (int)(8 * part) < dk;
  // R tokens a lane group, every load of all of them before any is used; a row's codes are loaded with the flag
  // and position that say whether they count
  int64_t p[R], held[R];
  uint8_t flag[R];
  uint32_t ck[R], cv[R], pk[R], pv[R];
#pragma unroll
  for (int r = 0; r < R; ++r) p[r] = pos[token + (unsigned)min((int)(t0 + r * TB), left - 1)];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const unsigned slot = p[r] < 0 ? 0u : (unsigned)slot_of(p[r], W);
    flag[r] = (ring_valid + (size_t)b * W)[slot];
    held[r] = (ring_pos + (size_t)b * W)[slot];
    const unsigned piece = slot * (unsigned)(dk / 8) + (live ? part : 0u);
    ck[r] = (ring_k + first * (dk / 8))[piece];
    cv[r] = (ring_v + first * (dk / 8))[piece];
    pk[r] = (k_scale + first)[slot];
    pv[r] = (v_scale + first)[slot];
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const unsigned t = t0 + r * TB;
    if ((int)t >= left) break;
    const bool here = p[r] >= 0 && flag[r] != 0 && held[r] == p[r];
    if (live) {
      // a token that is not held: zeros, as codes and pairs of zero give
      const V8 yk = dequantize_row8<T, V8>(here ? ck[r] : 0u, here ? pk[r] : 0u);
      const V8 yv = dequantize_row8<T, V8>(here ? cv[r] : 0u, here ? pv[r] : 0u);
      const size_t base = (token * HKV + head) * dk;
      const unsigned to = t * (unsigned)(HKV * dk) + 8 * part;
      *reinterpret_cast<V8*>(k + base + to) = yk;
      *reinterpret_cast<V8*>(v + base + to) = yv;
    }
    if (head == 0 && part == 0) found[token + t] = here ? 1 : 0;
  }
}

// ---- attention ----------------------------------------------------------------------------------
// The mask and the exponent bits that turn codes into elements, in registers that the compiler cannot see
// through: the and and the or then are one instruction (as literals they would be two, each with its own).
struct CodeBits {
  uint32_t mask, one;
  __device__ __forceinline__ explicit CodeBits(uint32_t exponent) : mask(0x000f000fu), one(exponent) {
#if defined(__HIP_DEVICE_COMPILE__)
    asm("" : "+s"(mask));
    asm("" : "+v"(one));
#endif
  }
  __device__ __forceinline__ uint32_t two(uint32_t w, int nibble) const { return ((w >> (4 * nibble)) & mask) | one; }
};
// The codes of a dword as eight elements, in the order 0 4 1 5 2 6 3 7 of the features.
template <typename T> struct Codes;
template <> struct Codes<__bf16> {
  static constexpr float kBias = 128.f;
  static constexpr uint32_t kOne = 0x43004300u;  // 0x4300 | c is 128 + c
  typedef bf16x8 V8;
  __device__ __forceinline__ static V8 unpack(uint32_t w, const CodeBits& bits) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = bits.two(w, i);
    return __builtin_bit_cast(V8, r);
  }
  __device__ __forceinline__ static f32x4 mma(V8 a, V8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Codes<_Float16> {
  static constexpr float kBias = 0.f;
  static constexpr uint32_t kOne = 0x64006400u;  // 0x6400 | c is 1024 + c
  typedef f16x8 V8;
  __device__ __forceinline__ static V8 unpack(uint32_t w, const CodeBits& bits) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f16x2 x = __builtin_bit_cast(f16x2, bits.two(w, i));
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

// Buffer loads of 1 to 16 bytes a lane at a lane's offset and a scalar one; past the resource's range they give zeros.
__device__ __forceinline__ uint32_t load_b8(__amdgpu_buffer_rsrc_t r, unsigned off, unsigned base) {
  return (uint32_t)(uint8_t)__builtin_amdgcn_raw_buffer_load_b8(r, (int)off, (int)base, 0);
}
__device__ __forceinline__ uint32_t load_b16(__amdgpu_buffer_rsrc_t r, unsigned off, unsigned base) {
  return (uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, (int)off, (int)base, 0);
}
__device__ __forceinline__ u32x2 load_b64(__amdgpu_buffer_rsrc_t r, unsigned off, unsigned base) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, (int)off, (int)base, 0));
}
// WHOLE: every piece of N dwords that starts in the range ends in it; else dword by dword.
template <int N, bool WHOLE>
__device__ __forceinline__ void load_dwords(__amdgpu_buffer_rsrc_t r, unsigned off, unsigned base, uint32_t (&out)[N]) {
  if constexpr (N == 1 || !WHOLE) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      out[i] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, (int)(off + 4 * i), (int)base, 0);
  } else if constexpr (N == 2) {
    const u32x2 x = load_b64(r, off, base);
    out[0] = x[0];
    out[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const u32x4 x =
          __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)(off + 4 * i), (int)base, 0));
#pragma unroll
      for (int e = 0; e < 4; ++e) out[i + e] = x[e];
    }
  }
}

// The greatest of three that are not NaN, without fmaxf's quieting of its inputs.
__device__ __forceinline__ float top3(float x, float y, float z) {
  float r = x;
#if defined(__HIP_DEVICE_COMPILE__)
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
#endif
  return r;
}

// The largest of x over the lanes l, l ^ 16, l ^ 32, l ^ 48 (a column of an MFMA result).
__device__ __forceinline__ float max_over_rows(float x) {
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = top3(__uint_as_float(p[0]), __uint_as_float(p[1]), __uint_as_float(p[1]));
  const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return top3(__uint_as_float(q[0]), __uint_as_float(q[1]), __uint_as_float(q[1]));
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
  int B, H, HKV, dk, W, splits, per, heads;  // per: tiles a split; heads: B HKV
  float scale_log2;
};

// The new tokens into their slots, which no workgroup attends (a reader of their codes drops them): L lanes
// a row, keys then values, in workgroups behind the attention's.
template <typename T, int L>
__device__ __forceinline__ void write_tokens(const T* knew, const T* vnew, const QuantAttnArgs& a, int block, int threads) {
  const int64_t r = ((int64_t)block * threads + threadIdx.x) / L;
  const int part = threadIdx.x % L;
  if (r >= 2 * (int64_t)a.heads) return;  // whole rows of lanes
  const bool values = r >= a.heads;
  const size_t head = (size_t)(values ? r - a.heads : r);
  const int b = (int)(head / a.HKV), kvh = (int)(head - (size_t)b * a.HKV);
  const int64_t p = a.pos[b];
  if (p < 0) return;
  const int slot = slot_of(p, a.W);
  const bool live = 8 * part < a.dk;
  float x[8];
  load8_f32((values ? vnew : knew) + head * a.dk + (live ? 8 * part : 0), x);
  uint32_t pair;
  const uint32_t codes = quantize_row8<T, L>(x, pair);
  const size_t row = head * a.W + slot;
  if (live) (values ? a.ring_v : a.ring_k)[row * (size_t)(a.dk / 8) + part] = codes;
  if (part == 0) {
    (values ? a.v_scale : a.k_scale)[row] = pair;
    if (!values && kvh == 0) {
      a.ring_pos[(size_t)b * a.W + slot] = p;
      a.ring_valid[(size_t)b * a.W + slot] = 1;
    }
  }
}

// One tile's loads: a token's pair, position and flag a lane (lanes 0..31 the keys' pairs, 32..63 the values'),
// and the codes of both products.
template <int NS>
struct QuantTile {
  static constexpr int VD = NS <= 4 ? 1 : NS / 4;  // dwords of a lane's piece of a V row
  uint32_t pair;
  int64_t pos;
  uint32_t flag;
  uint32_t k[2][NS], v[8][VD];
};

// One workgroup: the query heads of one KV head of one row over one of `splits` runs of tiles of 32
// slots, its NW waves taking the tiles in turn, each with the next tile's loads in flight while it works on
// one. NS: the head width in units of 32, rounded up to a power of two.
// Lane (c, g) = (l % 16, l / 16). K tile: lane holds dwords g NS .. + NS of the codes of tokens c and
// 16 + c. V tile: lane holds features c M .. + M of tokens 4 g + i and 16 + 4 g + i (i = 0..3), M = 2 NS,
// which are the tokens whose scores it holds; its M accumulators hold features (4 g + r) M + e, r = 0..3.
// Features past dk: K's meet zeros of q, V's are not stored; both lie inside the ring or read as zero.
// WHOLE: dk is a whole number of lanes' pieces (NS dwords), so no piece reaches past the ring's end.
// (At least two waves a SIMD: the accumulators then stay in the registers that the rescaling reads.)
template <typename T, int NS, bool WHOLE, int NW>
__global__ __launch_bounds__(64 * NW, NW / 4 < 2 ? 2 : NW / 4) void quant_attn_kernel(
    const T* __restrict__ q, const T* __restrict__ knew, const T* __restrict__ vnew, T* __restrict__ o,
    const QuantAttnArgs a) {
  constexpr int DP = 32 * NS, M = 2 * NS;
  using C = Codes<T>;
  typedef T V8 __attribute__((ext_vector_type(8)));
  __shared__ __align__(16) float2 stage[NW][2][kTile];  // the tile's pairs as the products take them
  __shared__ float smerge[NW][kQuantMaxGroup][2 + DP];
  __shared__ float sfresh[kQuantMaxGroup];

  const int grid = a.heads * a.splits;
  if ((int)blockIdx.x >= grid) {
    write_tokens<T, DP / 8>(knew, vnew, a, (int)blockIdx.x - grid, 64 * NW);
    return;
  }
  const int lg = xcd_logical_block(blockIdx.x, grid);
  const int kvh = lg % a.HKV, rest = lg / a.HKV;
  const int b = rest / a.splits, split = rest - b * a.splits;
  const int G = a.H / a.HKV, dk = a.dk, W = a.W;
  const int tid = threadIdx.x, l = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), c = l & 15, g = l >> 4;
  const size_t head = (size_t)b * a.HKV + kvh;
  const unsigned rb = (unsigned)dk / 2;  // bytes a row
  const __amdgpu_buffer_rsrc_t rk = buffer_rsrc(a.ring_k + head * W * (dk / 8), (unsigned)W * rb);
  const __amdgpu_buffer_rsrc_t rv = buffer_rsrc(a.ring_v + head * W * (dk / 8), (unsigned)W * rb);
  const uint32_t* pairs = (l < 32 ? a.k_scale : a.v_scale) + head * W;
  const __amdgpu_buffer_rsrc_t rp = buffer_rsrc(a.ring_pos + (size_t)b * W, 8u * (unsigned)W);
  const __amdgpu_buffer_rsrc_t rf = buffer_rsrc(a.ring_valid + (size_t)b * W, (unsigned)W);

  // A tile's loads; its first slot is below W, so that the scalar offsets stay below the resources' sizes.
  const unsigned koff = (unsigned)c * rb + 4u * NS * (unsigned)g, voff = 4u * (unsigned)g * rb + (unsigned)(c * NS);
  auto fetch = [&](int t, QuantTile<NS>& x) {
    const unsigned j0 = (unsigned)(kTile * t), base = j0 * rb, js = (unsigned)(l & 31);
    x.pos = __builtin_bit_cast(int64_t, load_b64(rp, 8u * js, 8u * j0));
    x.flag = load_b8(rf, js, j0);
    x.pair = pairs[min((int)(j0 + js), W - 1)];
#pragma unroll
    for (int u = 0; u < 2; ++u) load_dwords<NS, WHOLE>(rk, koff + 16u * u * rb, base, x.k[u]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned off = voff + (unsigned)((i & 3) + 16 * (i >> 2)) * rb;
      if constexpr (M == 2) x.v[i][0] = load_b8(rv, off, base);
      else if constexpr (M == 4) x.v[i][0] = load_b16(rv, off, base);
      else load_dwords<QuantTile<NS>::VD, WHOLE>(rv, off, base, x.v[i]);
    }
  };
  const int first = split * a.per, last = min(first + a.per, (W + kTile - 1) / kTile);
  int t = first + w;
  QuantTile<NS> even, odd;
  if (t < last) fetch(t, even);

  const int64_t p = a.pos[b];
  const int slot = p < 0 ? -1 : slot_of(p, W);
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
  f32x4 unbias = zero4();  // where the scores' sums begin: they end as those of the codes alone
  if constexpr (C::kBias != 0.f) unbias = f32x4{-C::kBias * qsum, -C::kBias * qsum, -C::kBias * qsum, -C::kBias * qsum};
  if (w == 0) {
    fresh = sum_over_rows(fresh) * a.scale_log2;
    if (l < kQuantMaxGroup) sfresh[l] = fresh;
  }

  float m = -3.40282347e38f, lsum = 0.f, low = 0.f;  // the running maximum (finite: scores of -inf weigh 0), the lane's sums of P and of P m'
  float room = 0.f;  // how far above the scores the running maximum is kept
  f32x4 acc[M], bias = zero4();
#pragma unroll
  for (int e = 0; e < M; ++e) acc[e] = zero4();
  const float second = c < 8 ? 0.f : 1.f;
  bf16x8 ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = (__bf16)128.f;

  const CodeBits kbits(C::kOne), vbits(Codes<__bf16>::kOne);
  const int64_t oldest = p < 0 ? INT64_MAX : p - W;  // positions past it and up to p are seen
  auto work = [&](int t, const QuantTile<NS>& tile) {
    // which tokens are seen (slots past W read flag 0), and their pairs
    const bool seen = tile.flag != 0 && tile.pos <= p && tile.pos > oldest && kTile * t + (l & 31) != slot;
    const uint32_t mask = (uint32_t)__ballot(seen);
    if (mask != 0) {
      const float ps = pair_scale<T>(tile.pair), pl = pair_low<T>(tile.pair);
      float2 st;
      if (l < 32) st = make_float2(ps * a.scale_log2, pl * a.scale_log2);
      else st = seen ? make_float2(ps, pl) : make_float2(0.f, 0.f);  // no NaN of an unseen slot meets a zero weight
      if constexpr (std::is_same_v<T, __bf16>) {  // fp16's numbers are never that large
        const float size = __builtin_fmaxf(__builtin_fabsf(st.x), __builtin_fabsf(st.y));
        if (__ballot(size > kLargePair) >> 32 != 0) room = kHeadroom;
      }
      __builtin_amdgcn_wave_barrier();
      stage[w][l >> 5][l & 31] = st;
      __builtin_amdgcn_wave_barrier();
      // scores of the lane's eight tokens: 4 g + i in the first tile of 16, then 16 + 4 g + i
      float sc[8];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f32x4 d = unbias;
#pragma unroll
        for (int s = 0; s < NS; ++s) d = C::mma(C::unpack(tile.k[u][s], kbits), qf[s], d);
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
      const float top = max_over_rows(top3(top3(sc[0], sc[1], sc[2]), top3(sc[3], sc[4], sc[5]), top3(sc[6], sc[7], sc[7])));
      if (__ballot(top + room > m + kRaise) != 0) {
        const float mn = __builtin_fmaxf(m, top + room);
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
          const uint32_t x = tile.v[2 * i][h / 2], y = tile.v[2 * i + 1][h / 2];
          two[i] = M <= 4 ? (x | (y << 16)) : (h & 1) == 0 ? ((x & 0xffffu) | (y << 16)) : ((x >> 16) | (y & 0xffff0000u));
        }
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          u32x4 r;
#pragma unroll
          for (int i = 0; i < 4; ++i) r[i] = vbits.two(two[i], e);
          acc[4 * h + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, r), pv, acc[4 * h + e], 0, 0, 0);
        }
      }
    }
  };
  // two tiles a turn, each in registers of its own: a tile's loads are issued before the other's work
  for (; t < last; t += 2 * NW) {
    if (t + NW < last) fetch(t + NW, odd);
    work(t, even);
    if (t + NW < last) {
      if (t + 2 * NW < last) fetch(t + 2 * NW, even);
      work(t + NW, odd);
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
      if (c < G) smerge[w][c][2 + (4 * g + r) * M + e] = x + low;
    }
  if (g == 0 && c < G) {
    smerge[w][c][0] = lsum == 0.f ? -kInf : m;  // a wave that saw nothing has no say in the maximum
    smerge[w][c][1] = lsum;
  }
  __syncthreads();
  // the waves' states, and in the first split the new token's (weight 1 at its score), joined
  const bool on = a.active == nullptr || a.active[b] != 0;
  for (int i = tid; i < G * dk; i += 64 * NW) {
    const int gi = i / dk, d = i - gi * dk;
    float mx = split == 0 ? sfresh[gi] : -kInf;
#pragma unroll
    for (int u = 0; u < NW; ++u) mx = __builtin_fmaxf(mx, smerge[u][gi][0]);
    const float from = mx == -kInf ? 0.f : mx;  // a split that saw nothing: weights of zero
    float ls = 0.f, num = 0.f;
    if (split == 0) {
      ls = __builtin_amdgcn_exp2f(sfresh[gi] - from);
      num = ls * to_f32(vnew[head * dk + d]);
    }
#pragma unroll
    for (int u = 0; u < NW; ++u) {
      const float f = __builtin_amdgcn_exp2f(smerge[u][gi][0] - from);
      ls += smerge[u][gi][1] * f;
      num += smerge[u][gi][2 + d] * f;
    }
    const size_t row = (size_t)b * a.H + (size_t)kvh * G + gi;
    if (a.splits == 1) {
      o[row * dk + d] = from_f32<T>(on ? average<T>(num, ls) : 0.f);
    } else {
      float* part = a.partial + (row * a.splits + split) * (size_t)(2 + dk);
      part[2 + d] = num;
      if (d == 0) {
        part[0] = mx;
        part[1] = ls;
      }
    }
  }
}

// The splits' softmax states of one query head joined (the first holds the new token, so their maximum is one of a
// score): their weights first, one split a thread, then groups of
// dk threads take the splits in turn and the groups' sums are added in order.
template <typename T>
__global__ __launch_bounds__(1024) void quant_join_kernel(const float* __restrict__ partial, T* __restrict__ o,
                                                          const uint8_t* __restrict__ active, int H, int dk,
                                                          int splits) {
  __shared__ float weight[kMaxSplits], sums[1024], red[2][16];
  const size_t row = blockIdx.x;
  const int pitch = 2 + dk;
  const float* part = partial + row * splits * (size_t)pitch;
  const int t = threadIdx.x, w = t >> 6, nw = blockDim.x >> 6;
  const float m = t < splits ? part[(size_t)t * pitch] : -kInf, l = t < splits ? part[(size_t)t * pitch + 1] : 0.f;
  float mx = group_max<64>(m);
  if ((t & 63) == 0) red[0][w] = mx;
  __syncthreads();
  for (int u = 0; u < nw; ++u) mx = __builtin_fmaxf(mx, red[0][u]);
  const float f = __builtin_amdgcn_exp2f(m - mx);
  if (t < splits) weight[t] = f;
  const float ls = group_sum<64>(t < splits ? l * f : 0.f);
  if ((t & 63) == 0) red[1][w] = ls;
  __syncthreads();
  const int groups = (int)blockDim.x / dk, grp = t / dk, d = t - grp * dk;
  float num = 0.f;
  if (grp < groups) {
#pragma unroll 8
    for (int s = grp; s < splits; s += groups) num += part[(size_t)s * pitch + 2 + d] * weight[s];
  }
  sums[t] = num;
  __syncthreads();
  if (t < dk) {
    float total = 0.f, sum = 0.f;
    for (int u = 0; u < nw; ++u) total += red[1][u];
    for (int u = 0; u < groups; ++u) sum += sums[u * dk + t];
    const bool on = active == nullptr || active[row / H] != 0;
    o[row * dk + t] = from_f32<T>(on ? average<T>(sum, total) : 0.f);
  }
}

// ---- host side ----------------------------------------------------------------------------------

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// The sizes every entry shares; 0 or an error.
int quant_sizes(int B, int HKV, int D, int W, const char* who) {
  if (B < 0 || HKV < 1 || W < 1) return fail(ERR_ARG, "%s: bad sizes B=%d HKV=%d W=%d", who, B, HKV, W);
  if (HKV > (1 << 14)) return fail(ERR_UNSUPPORTED, "%s: %d KV heads (at most 16384)", who, HKV);
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
  const int64_t grid = (int64_t)B * blocks * HKV;
  if (grid >= kMaxThreads / 256) return fail(ERR_UNSUPPORTED, "%s: %lld workgroups", who, (long long)grid);
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
  const int tb = kReadTokens * (256 / lanes_of(D)), blocks = (int)(((int64_t)N + tb - 1) / tb);
  const int64_t grid = (int64_t)B * blocks * HKV;
  if (grid >= kMaxThreads / 256) return fail(ERR_UNSUPPORTED, "%s: %lld workgroups", who, (long long)grid);
  by_lanes(D, [&](auto lanes) {
    hipLaunchKernelGGL((quant_read_kernel<T, decltype(lanes)::value>), dim3((unsigned)grid), dim3(256), 0,
                       reinterpret_cast<hipStream_t>(stream), static_cast<const uint32_t*>(ring_k),
                       static_cast<const uint32_t*>(ring_v), static_cast<const uint32_t*>(k_scale),
                       static_cast<const uint32_t*>(v_scale), ring_pos, ring_valid, pos, k, v, found, B, N, HKV, D, W,
                       blocks);
  });
  return check_launch(who);
}

// How a head's window is shared: waves a workgroup, workgroups (splits) a head and tiles a split.
//
// A workgroup costs about 2 us before and after its tiles, a tile 0.35 to 0.8 us of a wave, and a second split
// the launch that joins them, 3.2 to 5 us. So, with tiles for 512 workgroups of four waves and eight tiles
// each, or 256 heads: four waves, as many splits as make 512 workgroups (64 heads of 8191 slots at dk 64: 18.0 us
// with 512, 22.4 with 256, 19.0 with 1024; 512 heads of 512 slots: 9.4 us, with eight waves 9.9, in two splits 15.2).
// Else the workgroup is as wide as its registers allow, 16 waves up to dk 64 and eight beyond, and a window of up
// to 64 tiles stays whole (8 heads of 512 slots at dk 64: 6.7 us, four splits of four waves 8.0; 128 heads with four
// query heads each: 7.1 us, four waves in two splits 9.7); longer ones are split by 32 tiles, wider heads by 16
// (one head of 65536 slots at dk 128: 64 splits 11.0 us, 128 8.3; 32 heads of 4096 at dk 256: four splits 16.2, eight 13.7).
constexpr int kManyGroups = 512;
struct AttnShape {
  int waves, splits, per;
};
AttnShape attn_shape(int B, int HKV, int D, int W) {
  const int64_t heads = (int64_t)B * HKV, tiles = ((int64_t)W + kTile - 1) / kTile;
  const int64_t runs = tiles / (D <= 64 ? 32 : 16), most = runs < 1 ? 1 : runs > kMaxSplits ? kMaxSplits : runs;
  const int64_t share = heads >= kManyGroups ? 1 : (kManyGroups + heads - 1) / heads;
  const bool many = heads >= 256 || heads * most >= kManyGroups;
  const int64_t splits = !many && tiles <= 64 ? 1 : share < most ? share : most;
  const int64_t per = (tiles + splits - 1) / splits;
  return {many ? 4 : D <= 64 ? 16 : 8, (int)((tiles + per - 1) / per), (int)per};
}

size_t attn_workspace(int B, int H, int HKV, int D, int W) {
  const int splits = attn_shape(B, HKV, D, W).splits;
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
  const AttnShape shape = attn_shape(B, HKV, D, W);
  const int splits = shape.splits;
  const size_t need = attn_workspace(B, H, HKV, D, W);
  if (need > 0 && (workspace == nullptr || ws_bytes < need || !aligned(workspace, 4)))
    return fail(ERR_ARG, "%s: workspace of %zu bytes given, %zu needed", who, workspace ? ws_bytes : (size_t)0, need);
  const int threads = 64 * shape.waves, lanes = D <= 32 ? 4 : lanes_of(D);
  const int64_t grid = (int64_t)B * HKV * splits + (write ? ((int64_t)B * HKV * 2 * lanes + threads - 1) / threads : 0);
  if (grid >= kMaxThreads / threads || (int64_t)B * H >= ((int64_t)1 << 31))
    return fail(ERR_UNSUPPORTED, "%s: %lld workgroups", who, (long long)grid);
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_ptr);
  const QuantAttnArgs a{pos, static_cast<uint32_t*>(ring_k), static_cast<uint32_t*>(ring_v),
                        static_cast<uint32_t*>(k_scale), static_cast<uint32_t*>(v_scale), ring_pos, ring_valid, active,
                        static_cast<float*>(workspace), B, H, HKV, D, W, splits, shape.per,
                        B * HKV, scale * 1.4426950408889634f};
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(threads), 0, stream, q, knew, vnew, o, a);
  };
  auto by_width = [&](auto nw) {  // four waves, or the most that the width's registers allow (0)
    constexpr int NW = decltype(nw)::value, N64 = NW == 0 ? 16 : NW, N256 = NW == 0 ? 8 : NW;
    if (D <= 32) go(quant_attn_kernel<T, 1, true, N64>);
    else if (D <= 64) D % 16 == 0 ? go(quant_attn_kernel<T, 2, true, N64>) : go(quant_attn_kernel<T, 2, false, N64>);
    else if (D <= 128) D % 32 == 0 ? go(quant_attn_kernel<T, 4, true, N256>) : go(quant_attn_kernel<T, 4, false, N256>);
    else D % 64 == 0 ? go(quant_attn_kernel<T, 8, true, N256>) : go(quant_attn_kernel<T, 8, false, N256>);
  };
  if (shape.waves == 4) by_width(std::integral_constant<int, 4>{});
  else by_width(std::integral_constant<int, 0>{});
  if (splits > 1)
    hipLaunchKernelGGL(quant_join_kernel<T>, dim3((unsigned)(B * H)), dim3(splits <= 8 ? 256 : 1024), 0,
                       stream, static_cast<const float*>(workspace), o, active, H, D, splits);
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
