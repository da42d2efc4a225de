// q4.h — launches of the 4-bit KV cache and packed-prompt kernels
// (q4_cache.cu, q4_decode.cu, packed.cu), as qxcuda.cu calls them.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kv_row.cuh"

namespace qx {

// Sequences of one launch: they travel in the parameter block (under 4 KB),
// so a call copies no table and a captured graph keeps its own. Calls with
// more sequences make one launch per kQ4Seqs of them.
constexpr int kQ4Seqs = 200;

// One sequence's rows in a call.
struct Q4Seq {
  int seq;    // sequence index in the arena
  int begin;  // first cache row (append, read) or rows attended (decode)
  int first;  // first packed token of this sequence (append, read) or first work item (decode)
};

// A 4-bit arena as the kernels see it.
struct Q4Arena {
  char* k;
  char* v;
  int capacity;  // rows per (sequence, layer) of a contiguous arena
  int layers;
  KvPaging paging;
};

struct Q4AppendParams {
  Q4Arena arena;
  int layer_begin, layer_count;
  int n_seq;
  int token_begin, token_count;  // packed tokens of this launch
  const void* q;                 // null: only keys and values
  const void* k;
  const void* v;
  void* q_rot;  // rotated queries [token][layer][HQ * D], or null
  void* k_rot;  // rotated keys before quantisation, or null
  long long q_stride, k_stride, v_stride;  // elements between tokens
  const float* q_norm;
  const float* k_norm;
  const float2* rope;  // Granite: (sin, cos); Qwen: (cos, sin); [position][D / 2]
  int in_dtype, rot_dtype;
  int vec;  // q, k, v and their strides allow 16-byte loads, q_rot and k_rot 16-byte stores
  unsigned* err;
  Q4Seq seqs[kQ4Seqs];
};

struct Q4ReadParams {
  Q4Arena arena;
  int layer_begin, layer_count;
  int n_seq;
  int token_begin, token_count;
  void* key_out;    // [token][layer][HKV * D], or null
  void* value_out;  // likewise
  int out_dtype;
  int vec;  // the outputs allow 16-byte stores
  Q4Seq seqs[kQ4Seqs];
};

struct Q4DecodeParams {
  Q4Arena arena;
  int layer_begin, layer_count;
  int n_seq;
  int seq_begin;  // index of seqs[0] among the call's sequences
  // The launch's cells, (sequence, layer) in order, lie one after another on a
  // line of tiles; CTA b attends tiles [b * per_cta, (b + 1) * per_cta) of it.
  int per_cta;
  int total;      // tiles of the line
  int padded;     // a cell's place is rounded up to whole CTAs (a split the caller asked for)
  int max_parts;  // CTAs that share a cell, at most; above 1 qx_q4_merge_kernel follows
  const void* q;  // [sequence][layer][HQ * D]
  const void* k;  // [sequence][layer][HKV * D]
  const void* v;
  void* out;         // [sequence][layer][HQ * D]
  float* q_rot_out;  // rotated queries, or null
  const float* q_norm;
  const float* k_norm;
  const float2* rope;
  uint4* operands;  // rotated queries as MMA operands, per (sequence, layer) of the launch: see q4_operand_bytes
  float* units;     // and [HQ] base-2 logits of their sums
  float* part_o;    // of cells shared by CTAs: [CTA][2][HQ][D] sums (slot 0: the CTA's first cell, 1: its last)
  float2* part_ml;  // and [CTA][2][HQ] (m, l)
  int q_dtype, in_dtype, out_dtype;
  int vec;  // q, k and v allow 16-byte loads
  unsigned* err;
  Q4Seq seqs[kQ4Seqs];  // begin: rows attended, the new token's among them; first: its place on the line
};

constexpr int kQ4Tile = 32;  // cache rows per pipeline stage; pages hold a multiple of it

// One prompt of a packed call: its first packed token, its length, its first
// work item in the launch.
struct PackedSeq {
  int token, length, item;
};

struct PackedParams {
  // tokens x heads x head_dim: boxes of 64 dims, of a query tile's heads and
  // tokens and of 128 keys, 128-byte swizzle
  CUtensorMap tmq, tmk, tmv;
  const void* q;
  const void* k;
  const void* v;
  void* out;  // [token][HQ][D]
  long long q_stride, k_stride, v_stride;  // elements between tokens
  int dtype;
  int tokens;  // of all the call's prompts
  int n_seq;
  int items;
  unsigned* err;
  PackedSeq seqs[kQ4Seqs];  // longest first
};

// Tokens of a query block (two tiles of 128 query rows).
constexpr int packed_block(bool qwen) { return qwen ? 32 : 128; }
constexpr int kPackedKeys = 128;  // keys of a tile

cudaError_t launch_q4_append(bool qwen, const Q4AppendParams& p, cudaStream_t stream);
cudaError_t launch_q4_read(bool qwen, const Q4ReadParams& p, cudaStream_t stream);
// The kernels' attributes on the current device, before the first launch there.
cudaError_t setup_q4_decode();
cudaError_t setup_packed();
// The preparation, the attention and, where CTAs share cells, the merge; the
// kernels launched.
cudaError_t launch_q4_decode(bool qwen, const Q4DecodeParams& p, cudaStream_t stream, int* launched);
// Decode CTAs resident on one SM.
int q4_decode_blocks_per_sm();
// Bytes of the operands of one (sequence, layer): two 7-bit terms of every
// element, four unless the output is bf16.
constexpr size_t q4_operand_bytes(int heads, int d, int out_dtype) { return (size_t)heads * d * (out_dtype == 1 ? 2 : 4); }
cudaError_t launch_packed(bool qwen, const PackedParams& p, cudaStream_t stream);

}  // namespace qx
