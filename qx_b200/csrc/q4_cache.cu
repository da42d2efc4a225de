// q4_cache.cu — writing a 4-bit cache and reading it back.
//
// qx_q4_append_kernel norms (Qwen) and rotates the queries and keys of many
// new tokens, quantises keys and values and writes them into the arena's
// rows, all in one pass: every input is read once and every output written
// once. qx_q4_read_kernel expands rows into plain tensors.
#include "q4.cuh"

namespace qx {
namespace {

constexpr int kThreads = 256;

// A warp takes 32 / LPH neighbouring heads of one (token, layer), in the
// order query heads, key heads, value heads: D / 8 lanes a head, eight dims a
// lane, 16-byte loads of 16-bit inputs.
template <class M>
__global__ void __launch_bounds__(kThreads) qx_q4_append_kernel(const __grid_constant__ Q4AppendParams p) {
  using R = Q4Row<M>;
  constexpr int HPW = 32 / R::LPH;  // heads per warp
  const int lane = threadIdx.x & 31, c = lane & (R::LPH - 1);
  const int q_heads = p.q ? M::HQ : 0;
  const int warps = (q_heads + 2 * M::HKV) / HPW;  // per (token, layer)
  const long long w = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const long long unit = w / warps;
  pdl_wait();
  if (unit >= (long long)p.token_count * p.layer_count) return;
  int head = (int)(w - unit * warps) * HPW + lane / R::LPH;
  const int token = p.token_begin + (int)(unit / p.layer_count), l = (int)(unit % p.layer_count);
  const Q4Seq s = p.seqs[find_seq(p.seqs, p.n_seq, token)];
  const int position = s.begin + token - s.first;
  float x[8];
  bool good = true;
  if (head < q_heads) {
    load8(p.q, token * p.q_stride + ((long long)l * M::HQ + head) * M::D + 8 * c, p.q_dtype, p.vec, x);
    good = rotate_head<M>(x, c, position, p.q_norm, p.rope);
    store8(p.q_rot, (((long long)token * p.layer_count + l) * M::HQ + head) * M::D + 8 * c, p.rot_dtype, p.vec, x);
  } else {
    head -= q_heads;
    const long long row = kv_row(p.arena.paging, p.arena.capacity, p.arena.layers, s.seq, p.layer_begin + l, position);
    int codes[8];
    __half scale;
    if (head < M::HKV) {
      load8(p.k, token * p.k_stride + ((long long)l * M::HKV + head) * M::D + 8 * c, p.in_dtype, p.vec, x);
      good = rotate_head<M>(x, c, position, p.k_norm, p.rope);
      if (p.k_rot)
        store8(p.k_rot, (((long long)token * p.layer_count + l) * M::HKV + head) * M::D + 8 * c, p.rot_dtype, p.vec, x);
      good &= quantise8(x, codes, &scale);
      put_key<M>(p.arena.k + row * kQ4RowBytes, head, c, key_codes(codes), scale);
    } else {
      head -= M::HKV;
      load8(p.v, token * p.v_stride + ((long long)l * M::HKV + head) * M::D + 8 * c, p.in_dtype, p.vec, x);
      good = quantise8(x, codes, &scale);
      put_value<M>(p.arena.v + row * kQ4RowBytes, head, c, value_halves(codes), scale);
    }
  }
  if (!good) flag_error(p.err, QX_ERR_BIT_NONFINITE);
}

// A lane takes eight dims of a head of one key or value row.
template <class M>
__global__ void __launch_bounds__(kThreads) qx_q4_read_kernel(const __grid_constant__ Q4ReadParams p) {
  using R = Q4Row<M>;
  constexpr int CHUNKS = M::HKV * R::LPH;  // lanes per row
  const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
  const long long unit = i / (2 * CHUNKS);
  pdl_wait();
  if (unit >= (long long)p.token_count * p.layer_count) return;
  const int at = (int)(i - unit * 2 * CHUNKS), side = at / CHUNKS, head = at % CHUNKS / R::LPH, c = at & (R::LPH - 1);
  void* out = side ? p.value_out : p.key_out;
  if (!out) return;
  const int token = p.token_begin + (int)(unit / p.layer_count), l = (int)(unit % p.layer_count);
  const Q4Seq s = p.seqs[find_seq(p.seqs, p.n_seq, token)];
  const long long row = kv_row(p.arena.paging, p.arena.capacity, p.arena.layers, s.seq, p.layer_begin + l,
                               s.begin + token - s.first);
  const char* src = (side ? p.arena.v : p.arena.k) + row * kQ4RowBytes;
  int codes[8];
  if (side == 0) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(src + R::key_word(head, c));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      codes[i] = (int)(w << (24 - 8 * i)) >> 28;
      codes[4 + i] = (int)(w << (28 - 8 * i)) >> 28;
    }
  } else {
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      const uint32_t half = *reinterpret_cast<const uint16_t*>(src + R::value_half(head, c >> 2, g));
      codes[g] = (int)((half >> (4 * (c & 3))) & 15u) - 7;
    }
  }
  const float scale = __half2float(*reinterpret_cast<const __half*>(src + R::scale(head, c >> 2)));
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = __fmul_rn((float)codes[e], scale);
  store8(out, (((long long)token * p.layer_count + l) * M::HKV + head) * M::D + 8 * c, p.out_dtype, p.vec, x);
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
  const int warps = ((p.q ? M::HQ : 0) + 2 * M::HKV) / (32 / Q4Row<M>::LPH);
  const long long total = (long long)p.token_count * p.layer_count * warps;
  return launch_dependent(qx_q4_append_kernel<M>, (total + kThreads / 32 - 1) / (kThreads / 32), kThreads, stream, p);
}

template <class M>
cudaError_t read(const Q4ReadParams& p, cudaStream_t stream) {
  const long long total = (long long)p.token_count * p.layer_count * 2 * M::HKV * Q4Row<M>::LPH;
  return launch_dependent(qx_q4_read_kernel<M>, (total + kThreads - 1) / kThreads, kThreads, stream, p);
}

}  // namespace

cudaError_t launch_q4_append(bool qwen, const Q4AppendParams& p, cudaStream_t stream) {
  return qwen ? append<Qwen3Heads>(p, stream) : append<GraniteHeads>(p, stream);
}
cudaError_t launch_q4_read(bool qwen, const Q4ReadParams& p, cudaStream_t stream) {
  return qwen ? read<Qwen3Heads>(p, stream) : read<GraniteHeads>(p, stream);
}

}  // namespace qx
