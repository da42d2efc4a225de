// q4_cache.cu — writing a 4-bit cache and reading it back.
//
// qx_q4_append_kernel norms (Qwen) and rotates the queries and keys of many
// new tokens, quantises keys and values and writes them into the arena's
// rows, all in one pass: every input is read once and every output written
// once. qx_q4_read_kernel expands rows into plain tensors.
//
// Measured: 32768 bf16 Qwen3 tokens (norm, rotation, 4-bit rows; 640 MB) written in
// 133.5 us, 4.8 TB/s, 73% of a copy's rate; read back as bf16 in 18 us, 4.8 TB/s.
// 9001 bf16 Granite tokens: 17.3 and 6.4 us; one token: 1.8 and 1.6 us. The writes
// are bound by instructions and latency together: issue slots are busy 68% of the
// time (Granite 70%), DRAM 53%, with 28 of 32 warps an SM active, most of which
// wait for loads. What brought them there from 312 us: inputs of known types, all
// loaded before the first is used; one lane layout for queries that needs no
// exchange for the rotation; the table and the norm weights once a lane for all its
// heads; codes without a division or a conversion. (The check for norms that pass
// f32 is 2 us of the 133.5; by half warps or once for all heads it takes 3 or 4.)
#include "q4.cuh"

namespace qx {
namespace {

constexpr int kThreads = 256;

// N neighbouring elements as loaded, f32 (WIDE) or two 16-bit ones to a word;
// VEC: 16-byte aligned rows (the 32768 tokens above: 133.5 us, 162 where the inputs
// start at an odd element; read back 17 and 55). Types that the compiler knows, so that no load waits
// for another's branch.
template <int N, bool WIDE, bool VEC>
struct Raw {
  uint32_t w[WIDE ? N : N / 2];
  __device__ __forceinline__ void load(const void* base, long long i) {
    if constexpr (WIDE) {
      const float* p = reinterpret_cast<const float*>(base) + i;
#pragma unroll
      for (int e = 0; e < N; e += 4) {
        if constexpr (VEC) {
          const uint4 u = *reinterpret_cast<const uint4*>(p + e);
          w[e] = u.x, w[e + 1] = u.y, w[e + 2] = u.z, w[e + 3] = u.w;
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) w[e + k] = __float_as_uint(p[e + k]);
        }
      }
    } else {
      const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + i;
      if constexpr (VEC && N == 8) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
      } else if constexpr (VEC) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        w[0] = u.x, w[1] = u.y;
      } else {
#pragma unroll
        for (int e = 0; e < N / 2; ++e) w[e] = (uint32_t)p[2 * e] | (uint32_t)p[2 * e + 1] << 16;
      }
    }
  }
  // elements 2 e and 2 e + 1
  __device__ __forceinline__ float2 pair(int e, bool bf16) const {
    if constexpr (WIDE) return make_float2(__uint_as_float(w[2 * e]), __uint_as_float(w[2 * e + 1]));
    if (bf16) return make_float2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
  }
};

__device__ __forceinline__ void store4(void* base, long long i, int dtype, bool vec, const float* x) {
  if (!vec) {
#pragma unroll
    for (int e = 0; e < 4; ++e) store_any(base, i + e, dtype, x[e]);
  } else if (dtype == 0) {
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + i) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
    uint32_t w[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (dtype == 1) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
        w[e] = *reinterpret_cast<const uint32_t*>(&b);
      } else {
        const __half2 h = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
        w[e] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(base) + i) = make_uint2(w[0], w[1]);
  }
}

// Four warps take one (token, layer): each a quarter of the query heads and half
// of the key or value heads, D / 8 lanes a head. A key's or value's lane has eight
// neighbouring dims; a query's has dims 4 c .. 4 c + 3 and the four that they are
// rotated with, so that it needs no other lane but for the norm. A lane has the
// same dims in all its heads: it loads its rotation and norm weights once, and all
// its inputs before it uses the first. (With those of 32-bit inputs in flight it
// has 80 registers, of 16-bit ones 64: three CTAs an SM, four.)
template <class M, bool WIDE, bool VEC>
__global__ void __launch_bounds__(kThreads, WIDE ? 3 : 4) qx_q4_append_kernel(const __grid_constant__ Q4AppendParams p) {
  using R = Q4Row<M>;
  constexpr int HPW = 32 / R::LPH;         // heads per warp at once
  constexpr int PASSES = M::HQ / HPW / 4;  // of query heads per warp
  constexpr int HALF = M::D / 2;
  static_assert(M::HKV == 2 * HPW, "a warp's half of the key or value heads is one pass");
  const int lane = threadIdx.x & 31, c = lane & (R::LPH - 1), sub = lane / R::LPH;
  const int quarter = (threadIdx.x >> 5) & 3;
  const unsigned unit = blockIdx.x * (kThreads / 128) + (threadIdx.x >> 7);
  pdl_wait();
  if (unit >= (unsigned)p.token_count * p.layer_count) return;
  const unsigned step = p.layer_count == 1 ? unit : unit / p.layer_count;
  const int token = p.token_begin + (int)step, l = (int)(unit - step * p.layer_count);
  const bool value = quarter >= 2;
  const int kv = (quarter & 1) * HPW + sub;       // key or value head
  const int q0 = quarter * PASSES * HPW + sub;    // first query head
  const bool bf16 = p.in_dtype == 1;
  Raw<8, WIDE, VEC> y;
  y.load(value ? p.v : p.k, token * (value ? p.v_stride : p.k_stride) + ((long long)l * M::HKV + kv) * M::D + 8 * c);
  Raw<4, WIDE, VEC> x[PASSES][2];
  if (p.q) {
    const long long from = token * p.q_stride + ((long long)l * M::HQ + q0) * M::D + 4 * c;
#pragma unroll
    for (int a = 0; a < PASSES; ++a) {
      x[a][0].load(p.q, from + a * HPW * M::D);
      x[a][1].load(p.q, from + a * HPW * M::D + HALF);
    }
  }
  const Q4Seq s = p.seqs[find_seq(p.seqs, p.n_seq, token)];
  const int position = s.begin + token - s.first;
  const long long row = kv_row(p.arena.paging, p.arena.capacity, p.arena.layers, s.seq, p.layer_begin + l, position);
  const long long cell = (long long)token * p.layer_count + l;
  bool good = true;
  {
    float f[8];
    uint32_t codes[8];
    __half scale;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 z = y.pair(e, bf16);
      f[2 * e] = z.x, f[2 * e + 1] = z.y;
    }
    if (value) {
      good = quantise8(f, 7, codes, &scale);
      put_value<M>(p.arena.v + row * kQ4RowBytes, kv, c, value_halves(codes), scale);
    } else {
      float2 tab[8];
      rope_of_lane<M>(p.rope, position, c, tab);
      rotate_key<M>(f, c, p.k_norm, tab);
      if (p.k_rot) store8(p.k_rot, (cell * M::HKV + kv) * M::D + 8 * c, p.rot_dtype, VEC, f);
      good = quantise8(f, 0, codes, &scale);
      put_key<M>(p.arena.k + row * kQ4RowBytes, kv, c, key_codes(codes), scale);
    }
  }
  if (p.q) {
    // pairs of neighbouring dims: (cos, cos) and (sin, sin), norm weights
    float2 cs[2], sn[2], w[4];
    {
      const float4* from = reinterpret_cast<const float4*>(p.rope + (long long)position * HALF + 4 * c);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float4 v = from[e];
        cs[e] = M::QWEN ? make_float2(v.x, v.z) : make_float2(v.y, v.w);
        sn[e] = M::QWEN ? make_float2(v.y, v.w) : make_float2(v.x, v.z);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = 4 * c + 2 * (e & 1) + (e >> 1) * HALF;
        w[e] = M::QWEN && p.q_norm ? make_float2(p.q_norm[d], p.q_norm[d + 1]) : make_float2(1.0f, 1.0f);
      }
    }
    float2 bad = make_float2(0.0f, 0.0f);  // NaN once a result is not finite
#pragma unroll
    for (int a = 0; a < PASSES; ++a) {
      float2 v[4];  // dims 4 c + 0, 1; + 2, 3; and their partners
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = x[a][e >> 1].pair(e & 1, bf16);
      if constexpr (M::QWEN) {
        const float2 s2 = __fadd2_rn(__ffma2_rn(v[0], v[0], __fmul2_rn(v[1], v[1])), __ffma2_rn(v[2], v[2], __fmul2_rn(v[3], v[3])));
        float sum = s2.x + s2.y;
#pragma unroll
        for (int o = R::LPH / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        float inv = rsqrtf(fmaf(sum, 1.0f / M::D, 1.0e-6f));
        if (__any_sync(0xffffffffu, !isfinite(sum))) {  // elements beyond 1.6e18 may pass f32 in their squares
          const float x8[8] = {v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
          const float exact = exact_inv_rms<M>(x8);
          if (!isfinite(sum)) inv = exact;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __fmul2_rn(__fmul2_rn(v[e], make_float2(inv, inv)), w[e]);
      }
      float out[8];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 minus = make_float2(-sn[e].x, -sn[e].y);
        float2 left, right;
        if constexpr (M::QWEN) {  // each product and sum rounded
          left = __fadd2_rn(__fmul2_rn(v[e], cs[e]), __fmul2_rn(v[2 + e], minus));
          right = __fadd2_rn(__fmul2_rn(v[2 + e], cs[e]), __fmul2_rn(v[e], sn[e]));
        } else {
          left = __ffma2_rn(v[2 + e], minus, __fmul2_rn(v[e], cs[e]));
          right = __ffma2_rn(v[2 + e], cs[e], __fmul2_rn(v[e], sn[e]));
        }
        out[2 * e] = left.x, out[2 * e + 1] = left.y, out[4 + 2 * e] = right.x, out[5 + 2 * e] = right.y;
        bad = __ffma2_rn(left, make_float2(0.0f, 0.0f), bad);
        bad = __ffma2_rn(right, make_float2(0.0f, 0.0f), bad);
      }
      const long long to = (cell * M::HQ + q0 + a * HPW) * M::D + 4 * c;
      store4(p.q_rot, to, p.rot_dtype, VEC, out);
      store4(p.q_rot, to + HALF, p.rot_dtype, VEC, out + 4);
    }
    good &= bad.x + bad.y == 0.0f;
  }
  if (!good) flag_error(p.err, QX_ERR_BIT_NONFINITE);
}

// A lane takes eight dims of a head, of a row's key and value; a head's values are
// spread over its lanes' words (half g of a group holds dim g of each of its four
// lanes), which the lanes pass around.
template <class M>
__global__ void __launch_bounds__(kThreads) qx_q4_read_kernel(const __grid_constant__ Q4ReadParams p) {
  using R = Q4Row<M>;
  constexpr int LANES = M::HKV * R::LPH;  // per row
  static_assert(kThreads % LANES == 0, "whole rows a CTA");
  const int at = threadIdx.x % LANES, head = at / R::LPH, c = at & (R::LPH - 1);
  const unsigned unit = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  pdl_wait();
  if (unit >= (unsigned)p.token_count * p.layer_count) return;
  const unsigned step = p.layer_count == 1 ? unit : unit / p.layer_count;
  const int token = p.token_begin + (int)step, l = (int)(unit - step * p.layer_count);
  const Q4Seq s = p.seqs[find_seq(p.seqs, p.n_seq, token)];
  const long long row = kQ4RowBytes * kv_row(p.arena.paging, p.arena.capacity, p.arena.layers, s.seq,
                                             p.layer_begin + l, s.begin + token - s.first);
  const long long out = (((long long)token * p.layer_count + l) * M::HKV + head) * M::D + 8 * c;
  uint32_t key = 0u, value = 0u;
  float key_scale = 0.0f, value_scale = 0.0f;
  if (p.key_out) {
    key = *reinterpret_cast<const uint32_t*>(p.arena.k + row + R::key_word(head, c));
    key_scale = __half2float(*reinterpret_cast<const __half*>(p.arena.k + row + R::scale(head, c >> 2)));
  }
  if (p.value_out) {
    value = *reinterpret_cast<const uint32_t*>(p.arena.v + row + head * R::HEAD + 4 * c);
    value_scale = __half2float(*reinterpret_cast<const __half*>(p.arena.v + row + R::scale(head, c >> 2)));
  }
  // a nibble in the low bits of 2^23 is 2^23 plus it
  auto put2 = [](float* to, uint32_t a, uint32_t b, float base, float scale) {
    const float2 c = __fadd2_rn(make_float2(__uint_as_float((a & 15u) | 0x4b000000u), __uint_as_float((b & 15u) | 0x4b000000u)),
                                make_float2(-base, -base));
    const float2 y = __fmul2_rn(c, make_float2(scale, scale));
    to[0] = y.x;
    to[1] = y.y;
  };
  float x[8];
  if (p.key_out) {
    const uint32_t turned = key ^ 0x88888888u;  // c + 8
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      put2(x + i, turned >> (8 * i + 4), turned >> (8 * i + 12), 8388616.0f, key_scale);
      put2(x + 4 + i, turned >> (8 * i), turned >> (8 * i + 8), 8388616.0f, key_scale);
    }
    store8(p.key_out, out, p.out_dtype, p.vec, x);
  }
  if (p.value_out) {
    const int base = (threadIdx.x & 31) & ~(R::LPH - 1), j = c >> 2;
    const int shift = 4 * (c & 3) + 16 * (j & 1);  // half g NG + j: NG is even
#pragma unroll
    for (int g = 0; g < 8; g += 2) {
      const uint32_t a = __shfl_sync(0xffffffffu, value, base + ((g * R::NG + j) >> 1));
      const uint32_t b = __shfl_sync(0xffffffffu, value, base + (((g + 1) * R::NG + j) >> 1));
      put2(x + g, a >> shift, b >> shift, 8388615.0f, value_scale);
    }
    store8(p.value_out, out, p.out_dtype, p.vec, x);
  }
}

// Launch as a programmatic dependent of the stream's previous kernel.
template <class P>
cudaError_t launch_dependent(void (*fn)(P), long long blocks, int threads, cudaStream_t stream, const P& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, fn, p);
}

template <class M>
cudaError_t append(const Q4AppendParams& p, cudaStream_t stream) {
  const long long units = (long long)p.token_count * p.layer_count;
  void (*fn)(Q4AppendParams) = p.in_dtype == 0 ? (p.vec ? qx_q4_append_kernel<M, true, true> : qx_q4_append_kernel<M, true, false>)
                                               : (p.vec ? qx_q4_append_kernel<M, false, true> : qx_q4_append_kernel<M, false, false>);
  return launch_dependent(fn, (units + kThreads / 128 - 1) / (kThreads / 128), kThreads, stream, p);
}

template <class M>
cudaError_t read(const Q4ReadParams& p, cudaStream_t stream) {
  constexpr int ROWS = kThreads / (M::HKV * Q4Row<M>::LPH);  // a CTA
  const long long total = (long long)p.token_count * p.layer_count;
  return launch_dependent(qx_q4_read_kernel<M>, (total + ROWS - 1) / ROWS, kThreads, stream, p);
}

}  // namespace

cudaError_t launch_q4_append(bool qwen, const Q4AppendParams& p, cudaStream_t stream) {
  return qwen ? append<Qwen3Heads>(p, stream) : append<GraniteHeads>(p, stream);
}
cudaError_t launch_q4_read(bool qwen, const Q4ReadParams& p, cudaStream_t stream) {
  return qwen ? read<Qwen3Heads>(p, stream) : read<GraniteHeads>(p, stream);
}

}  // namespace qx
