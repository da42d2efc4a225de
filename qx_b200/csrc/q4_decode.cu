// q4_decode.cu — attention of new tokens over a 4-bit cache.
//
// First form: a warp takes one query head of one (sequence, layer), a lane
// D / 32 neighbouring dims, row after row with a running maximum and sum.
#include "q4.cuh"

namespace qx {
namespace {

template <class M>
__global__ void __launch_bounds__(128) qx_q4_decode_kernel(const __grid_constant__ Q4DecodeParams p) {
  using R = Q4Row<M>;
  constexpr int N = M::D / 32;
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  pdl_wait();
  if (w >= (long long)p.n_seq * p.layer_count * M::HQ) return;
  const int qh = (int)(w % M::HQ), h = qh / M::G;
  const long long unit = w / M::HQ;
  const int l = (int)(unit % p.layer_count), i = (int)(unit / p.layer_count);
  const Q4Seq s = p.seqs[i];
  const long long base = (((long long)(p.seq_begin + i) * p.layer_count + l) * M::HQ + qh) * M::D;
  float q[N], o[N], m = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    q[e] = p.q[base + N * lane + e];
    o[e] = 0.0f;
  }
  for (int r = 0; r < s.begin; ++r) {
    const long long row = kv_row(p.arena.paging, p.arena.capacity, p.arena.layers, s.seq, p.layer_begin + l, r);
    const unsigned char* kr = reinterpret_cast<const unsigned char*>(p.arena.k) + row * kQ4RowBytes;
    const unsigned char* vr = reinterpret_cast<const unsigned char*>(p.arena.v) + row * kQ4RowBytes;
    float dot = 0.0f, v[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int d = N * lane + e, j = d >> 5, rr = d & 31;
      const int kb = R::key_word(h, d >> 3) + ((rr & 7) >> 1);
      const int kc = (kr[kb] >> (4 * (rr & 1))) & 15;
      dot += q[e] * (float)(kc - 7) * __half2float(*reinterpret_cast<const __half*>(kr + R::scale(h, j)));
      const int vb = R::value_half(h, j, rr & 7) + (rr >> 4);
      const int vc = (vr[vb] >> (4 * ((rr >> 3) & 1))) & 15;
      v[e] = (float)(vc - 7) * __half2float(*reinterpret_cast<const __half*>(vr + R::scale(h, j)));
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
    const float x = dot * M::SCALE, top = fmaxf(m, x), keep = expf(m - top), e0 = expf(x - top);
    m = top;
    sum = sum * keep + e0;
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = o[e] * keep + e0 * v[e];
  }
  bool good = true;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float y = o[e] / sum;
    good &= isfinite(y);
    store_any(p.out, base + N * lane + e, p.out_dtype, y);
  }
  if (!good) flag_error(p.err, QX_ERR_BIT_NONFINITE);
}

}  // namespace

cudaError_t launch_q4_decode(bool qwen, const Q4DecodeParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  const long long warps = (long long)p.n_seq * p.layer_count * (qwen ? Qwen3Heads::HQ : GraniteHeads::HQ);
  cfg.gridDim = dim3((unsigned)((warps + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, qwen ? qx_q4_decode_kernel<Qwen3Heads> : qx_q4_decode_kernel<GraniteHeads>, p);
}

}  // namespace qx
