// packed.cu — causal attention of whole prompts packed one after another.
//
// First form: a warp takes one query head of one token, a lane D / 32
// neighbouring dims, key after key with a running maximum and sum.
#include "q4.cuh"

namespace qx {
namespace {

template <class M>
__global__ void __launch_bounds__(128) qx_packed_kernel(const __grid_constant__ PackedParams p) {
  constexpr int N = M::D / 32;
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  pdl_wait();
  if (w >= (long long)p.token_count * M::HQ) return;
  const int qh = (int)(w % M::HQ), h = qh / M::G;
  const int token = p.token_begin + (int)(w / M::HQ);
  const Q4Seq s = p.seqs[find_seq(p.seqs, p.n_seq, token)];
  float q[N], o[N], m = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    q[e] = load_any(p.q, token * p.q_stride + qh * M::D + N * lane + e, p.dtype);
    o[e] = 0.0f;
  }
  for (int t = s.first; t <= token; ++t) {
    float dot = 0.0f;
#pragma unroll
    for (int e = 0; e < N; ++e) dot += q[e] * load_any(p.k, t * p.k_stride + h * M::D + N * lane + e, p.dtype);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
    const float x = dot * M::SCALE, top = fmaxf(m, x), keep = expf(m - top), e0 = expf(x - top);
    m = top;
    sum = sum * keep + e0;
#pragma unroll
    for (int e = 0; e < N; ++e)
      o[e] = o[e] * keep + e0 * load_any(p.v, t * p.v_stride + h * M::D + N * lane + e, p.dtype);
  }
  bool good = true;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float y = o[e] / sum;
    good &= isfinite(y);
    store_any(p.out, ((long long)token * M::HQ + qh) * M::D + N * lane + e, p.dtype, y);
  }
  if (!good) flag_error(p.err, QX_ERR_BIT_NONFINITE);
}

}  // namespace

cudaError_t launch_packed(bool qwen, const PackedParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  const long long warps = (long long)p.token_count * (qwen ? Qwen3Heads::HQ : GraniteHeads::HQ);
  cfg.gridDim = dim3((unsigned)((warps + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, qwen ? qx_packed_kernel<Qwen3Heads> : qx_packed_kernel<GraniteHeads>, p);
}

}  // namespace qx
