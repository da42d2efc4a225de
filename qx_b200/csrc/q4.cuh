// q4.cuh — the 4-bit cache row and the arithmetic of a new token's heads.
//
// A row (one position, all kv heads) is 288 bytes for both models:
//   [0, 256)    codes, kv head after kv head, D / 2 bytes each
//   [256, 288)  fp16 scales [kv head][D / 32]
// A code c in -7..7 of a group of 32 dims stands for c * scale, the values of
// the framework's Q4 weights. Within a head the codes are laid out for the lane
// that reads them in the attention kernel, and in the form that costs it the
// fewest instructions (group j of D / 32, dim 32 j + r):
//   keys    32-bit word t * (D / 32) + j holds dims r = 8 t .. 8 t + 7: lane t of
//           a quad reads its words of all groups at once. Byte i has c of dim
//           8 t + i in its high nibble and c of dim 8 t + 4 + i in its low one, in
//           two's complement, so that w and w << 4, masked with 0xf0 in each byte,
//           are eight 8-bit integers 16 c.
//   values  16-bit half g * (D / 32) + j holds c + 7 of dims r = 8 i + g in nibble
//           i (i = 0..3): lane group g reads its halves of all groups at once
//
// A head is D / 8 neighbouring lanes of eight dims each: lane `c` of a head
// holds dims 8 c .. 8 c + 7, group c / 4, t = c % 4. Rotation pairs dim d with
// d + D / 2, half a head's lanes away.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "q4.h"
#include "qx_math.cuh"
#include "qx_ptx.cuh"

namespace qx {

struct GraniteHeads {
  static constexpr bool QWEN = false;
  static constexpr int HQ = 16, HKV = 8, D = 64, G = 2;
  static constexpr float SCALE = 0.015625f;  // ATTENTION_MULTIPLIER, qx-model lib.rs:20
};
struct Qwen3Heads {
  static constexpr bool QWEN = true;
  static constexpr int HQ = 32, HKV = 4, D = 128, G = 8;
  static constexpr float SCALE = 0.08838834764831845f;  // 1/sqrt(128)
};

constexpr int kQ4CodeBytes = 256;
constexpr int kQ4RowBytes = 288;

template <class M>
struct Q4Row {
  static constexpr int NG = M::D / 32;   // groups per head
  static constexpr int LPH = M::D / 8;   // lanes per head
  static constexpr int HEAD = M::D / 2;  // code bytes per head
  static_assert(M::HKV * HEAD == kQ4CodeBytes, "codes of a row");
  static_assert(kQ4CodeBytes + M::HKV * NG * 2 == kQ4RowBytes, "codes and scales of a row");
  static __device__ __forceinline__ int key_word(int head, int c) { return head * HEAD + 4 * ((c & 3) * NG + (c >> 2)); }
  static __device__ __forceinline__ int value_half(int head, int j, int g) { return head * HEAD + 2 * (g * NG + j); }
  static __device__ __forceinline__ int scale(int head, int j) { return kQ4CodeBytes + 2 * (head * NG + j); }
};

// Eight neighbouring elements as f32 (vec: base + i is 16-byte aligned).
__device__ __forceinline__ void load8(const void* base, long long i, int dtype, bool vec, float* x) {
  if (!vec) {
    load_any_n<8>(base, i, 1, dtype, x);
  } else if (dtype == 1) {
    Vec16<__nv_bfloat16>::load(reinterpret_cast<const __nv_bfloat16*>(base) + i, x);
  } else if (dtype == 2) {
    Vec16<__half>::load(reinterpret_cast<const __half*>(base) + i, x);
  } else {
    Vec16<float>::load(reinterpret_cast<const float*>(base) + i, x);
    Vec16<float>::load(reinterpret_cast<const float*>(base) + i + 4, x + 4);
  }
}

__device__ __forceinline__ void store8(void* base, long long i, int dtype, bool vec, const float* x) {
  if (!vec) {
#pragma unroll
    for (int e = 0; e < 8; ++e) store_any(base, i + e, dtype, x[e]);
  } else if (dtype == 0) {
    float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + i);
    o[0] = make_float4(x[0], x[1], x[2], x[3]);
    o[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (dtype == 1) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
        w[e] = *reinterpret_cast<const uint32_t*>(&b);
      } else {
        const __half2 h = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
        w[e] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(base) + i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// 1 / sqrt(mean + 1e-6) of a head over LANES lanes of N elements each, rounded
// once to f32. The sum of squares is a double (products of two 16-bit inputs and
// their sum are exact in it), so its order does not matter: quantised keys sit next
// to rounding borders, where an ulp of the norm would decide a code. Queries, which
// are not quantised to 4 bits, are summed in f32 and come here where that overflows.
template <class M, int N = 8, int LANES = Q4Row<M>::LPH>
__device__ __forceinline__ float exact_inv_rms(const float* x) {
  double sum = 0.0;
#pragma unroll
  for (int e = 0; e < N; ++e) sum = fma((double)x[e], (double)x[e], sum);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return (float)rsqrt(sum * (1.0 / M::D) + 1.0e-6);
}

// Of key heads: norm (Qwen) and rotation of this lane's eight dims of a head at `position`.
// The operation order is each model's: granite_rope_pair's fused pair
// (qx-consensus-math lib.rs:199-207), cpu_qk_norm_rope's separately rounded
// one (qx-qwen-parity main.rs:1170-1210). tab: the table's entries of these dims
// (rope_of_lane).
template <class M>
__device__ __forceinline__ void rotate_key(float* x, int c, const float* norm, const float2* tab) {
  constexpr int LPH = Q4Row<M>::LPH;
  if constexpr (M::QWEN) {
    const float inv = exact_inv_rms<M>(x);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __fmul_rn(__fmul_rn(x[e], inv), norm ? norm[8 * c + e] : 1.0f);
  }
  const bool right = c >= LPH / 2;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float y = __shfl_xor_sync(0xffffffffu, x[e], LPH / 2);
    const float2 t = tab[e];
    if constexpr (M::QWEN)
      x[e] = right ? __fadd_rn(__fmul_rn(x[e], t.x), __fmul_rn(y, t.y))
                   : __fsub_rn(__fmul_rn(x[e], t.x), __fmul_rn(y, t.y));
    else
      x[e] = right ? __fmaf_rn(x[e], t.y, __fmul_rn(y, t.x)) : __fmaf_rn(-y, t.x, __fmul_rn(x[e], t.y));
  }
}

// The rotation table's entries of lane c's dims at `position`.
template <class M>
__device__ __forceinline__ void rope_of_lane(const float2* rope, int position, int c, float2* tab) {
  const float4* from = reinterpret_cast<const float4*>(rope + (long long)position * (M::D / 2) +
                                                       8 * (c & (Q4Row<M>::LPH / 2 - 1)));
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float4 v = from[e];
    tab[2 * e] = make_float2(v.x, v.y);
    tab[2 * e + 1] = make_float2(v.z, v.w);
  }
}

// The codes of this lane's eight dims, each plus `offset` (0 or 7) in the low byte
// of an integer, and its group's scale. False when the scale is not finite: a value
// above 7 * 65504, an infinity, or a NaN (which fmaxf alone would drop).
__device__ __forceinline__ bool quantise8(const float* x, int offset, uint32_t* codes, __half* scale) {
  float top = 0.0f;
  float2 bad = make_float2(0.0f, 0.0f);  // NaN once a value is not finite
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    top = fmax3f(top, fabsf(x[e]), fabsf(x[e + 1]));
    bad = __ffma2_rn(make_float2(x[e], x[e + 1]), make_float2(0.0f, 0.0f), bad);
  }
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  // top / 7, correctly rounded: one multiplication and a correction by its
  // residual (compared with the division for all 2^23 mantissas)
  constexpr float SEVENTH = 1.0f / 7.0f;
  const float guess = __fmul_rn(top, SEVENTH);
  const __half h = __float2half_rn(__fmaf_rn(__fmaf_rn(-7.0f, guess, top), SEVENTH, guess));
  const float s = __half2float(h);
  // x / s rounded to an integer, by adding 1.5 * 2^23: a product with the
  // approximate reciprocal is off by less than 2^-19 of a step, so only quotients
  // closer than that to a border between two codes need the division itself, and
  // only the scales that fp16 rounds coarsely, its subnormals, need the limits
  float inv;
  asm("rcp.approx.f32 %0, %1;" : "=f"(inv) : "f"(s));
  const float base = 12582912.0f + (float)offset;
  float away = 0.0f;  // the largest distance of a quotient from its integer
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float2 q = __fmul2_rn(make_float2(x[e], x[e + 1]), make_float2(inv, inv));
    const float2 n = __fadd2_rn(q, make_float2(base, base));
    const float2 back = __fadd2_rn(n, make_float2(-base, -base));
    const float2 d = __ffma2_rn(back, make_float2(-1.0f, -1.0f), q);
    away = fmax3f(away, fabsf(d.x), fabsf(d.y));
    codes[e] = __float_as_uint(n.x);
    codes[e + 1] = __float_as_uint(n.y);
  }
  if (away > 0.5f - 3.0e-6f || top * inv > 7.4f) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      codes[e] = (uint32_t)(__float2int_rn(fminf(fmaxf(__fdiv_rn(x[e], s), -7.0f), 7.0f)) + offset);
  }
  if (!(s > 0.0f)) {  // a scale that rounds to zero: every value is zero
#pragma unroll
    for (int e = 0; e < 8; ++e) codes[e] = (uint32_t)offset;
  }
  *scale = h;
  return bad.x + bad.y == 0.0f && isfinite(s);
}

// The low bytes of four words.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// This lane's eight codes (offset 0) as a word of a key row.
__device__ __forceinline__ uint32_t key_codes(const uint32_t* c) {
  const uint32_t high = low_bytes(c[0], c[1], c[2], c[3]), low = low_bytes(c[4], c[5], c[6], c[7]);
  return ((high << 4) & 0xf0f0f0f0u) | (low & 0x0f0f0f0fu);
}

// Store this lane's word and scale as part of a key row.
template <class M>
__device__ __forceinline__ void put_key(char* row, int head, int c, uint32_t codes, __half scale) {
  *reinterpret_cast<uint32_t*>(row + Q4Row<M>::key_word(head, c)) = codes;
  if ((c & 3) == 0) *reinterpret_cast<__half*>(row + Q4Row<M>::scale(head, c >> 2)) = scale;
}

// The halves g = 2 t (low 16 bits) and 2 t + 1 of a value row's group that
// lane t of a quad stores, from its codes (offset 7): nibble i of half g comes from lane i, which holds
// dims 8 i + g. Every lane of the warp takes part.
__device__ __forceinline__ uint32_t value_halves(const uint32_t* c) {
  const int lane = threadIdx.x & 31, t = lane & 3;
  const uint32_t codes = low_bytes(c[0], c[2], c[4], c[6]) + 16u * low_bytes(c[1], c[3], c[5], c[7]);
  uint32_t out = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = __shfl_sync(0xffffffffu, codes, (lane & ~3) + i) >> (8 * t);
    out |= (w & 15u) << (4 * i) | ((w >> 4) & 15u) << (16 + 4 * i);
  }
  return out;
}

// Store this lane's halves (value_halves) and scale as part of a value row.
template <class M>
__device__ __forceinline__ void put_value(char* row, int head, int c, uint32_t halves, __half scale) {
  const int t = c & 3, j = c >> 2;
  *reinterpret_cast<uint16_t*>(row + Q4Row<M>::value_half(head, j, 2 * t)) = (uint16_t)halves;
  *reinterpret_cast<uint16_t*>(row + Q4Row<M>::value_half(head, j, 2 * t + 1)) = (uint16_t)(halves >> 16);
  if (t == 0) *reinterpret_cast<__half*>(row + Q4Row<M>::scale(head, j)) = scale;
}

// The entry of seqs (in rising order of `first`) that holds index i.
__device__ __forceinline__ int find_seq(const Q4Seq* seqs, int n, int i) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (seqs[mid].first <= i) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

}  // namespace qx
