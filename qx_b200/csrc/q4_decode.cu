// q4_decode.cu — one decode step over a 4-bit cache.
//
// qx_q4_prepare_kernel writes the new token's rows and the rotated queries as
// MMA operands; qx_q4_decode_kernel attends; where a sequence was split,
// qx_q4_merge_kernel joins the parts. Each is a programmatic dependent of the one
// before.
//
// qx_q4_decode_kernel: all (sequence, layer) cells of a launch lie on one line of
// tiles of 32 rows, and every CTA, two an SM, takes the same length of it: the
// stream of rows never stops between cells, and no CTA has more rows than
// another. A CTA attends all kv heads, so a tile is one contiguous piece of
// memory a side (288 bytes a row). Two groups of four warps take alternate tiles;
// a warp takes a unit of eight query heads, one kv head of Qwen or four of
// Granite (and then half of the tile's rows):
//   copies   by bulk copies into a ring of six stages, three a group; the last
//            warp of a group to finish a tile refills its stage. (A stage belongs
//            to one group: a warp is then never two phases ahead of a barrier,
//            which its parity could not tell from none.)
//   scores   S = Q K^T by mma.m16n8k32 on 8-bit integers, exact: K's codes are
//            8-bit integers as they lie in the row but for a mask, a query is
//            rounded once to an integer of 15 bits (29 unless the output is bf16)
//            against its head's largest element, cut into terms of 7 bits: rows
//            0-7 of an operand hold one term of the unit's heads, rows 8-15 the
//            next. Each group of 32 dims has its own accumulator, multiplied by
//            the row's scale in f32.
//   softmax  in f32, base 2, a running reference m per head and warp
//   output   O^T += V^T P'^T by mma.m16n8k16, V's codes as fp16 integers; P' =
//            P * scale of (row, group), rounded to fp16 (two fp16 terms when the
//            output is f32), one operand per group. P falls out of the score
//            accumulators in exactly the operand layout.
// Granite's four kv heads of a unit share accumulators: a head's operand is
// zero in the rows (columns) of the other heads, so a lane's scores, weights and
// outputs are those of its own query head whichever kv head it has, and the
// softmax runs on full lanes.
//
// Measured (the rows' bytes at a copy's 6.5 TB/s in brackets): 48 ragged Qwen3
// sequences of up to 8190 rows, 2 layers, 68.7 us (38.5); 128 ragged Granite ones of
// up to 4096, 4 layers, 121 us (91.9); one Qwen3 layer of 32768 rows 14.1 us (2.9);
// 24 Granite layers of 4064 rows, f32 in and out, 24.6 us (8.6); one of 512 rows 8.3
// us. The batches are bound by latency at 16 warps an SM: an instruction issues in
// 55% of the cycles, the tensor pipe is busy 23% (Granite 30%), DRAM 46% (60%), and
// a warp's stalls are spread over loads, fixed latencies and full pipes: each walks
// one chain of wait, products, scaling, maximum, exponentials, products. With every
// row in L2 they still take 64 and 110 us, the stream of rows without the work 50
// and 100. In f32 a row takes twice the products (the 24 layers: tensor pipe 29%,
// issue 40%). Single sequences are bound by the chain of three launches and the
// joining of the parts. Steps: f16 products only 117 and 225 us,
// integer scores 102 and 169, masks of one instruction 98 and 156, a grid of their
// own for queries and new rows 92 and 145, one line of tiles 69 and 120.
//
// The tensor instructions take their operands from registers: 4-bit codes
// would have to pass through shared memory a second time to reach tcgen05, and
// the products are a small part of the work (expanding a tile's codes takes
// more instructions than multiplying them).
//
// The row order inside a block of 8 (row_g, row_a, row_b below) makes the
// quads' loads of neighbouring MMA rows fall into different banks: a row is 72
// words, 8 modulo 32, and rows 0, 6, 1, 7, 2, 4, 3, 5 give every 128-byte phase
// of the key loads, of the value loads and of the scale loads distinct banks.
#include "q4.cuh"

namespace qx {
namespace {

constexpr int kThreads = 256;
constexpr int kStages = 6;
constexpr int kSide = kQ4Tile * kQ4RowBytes;  // bytes of a tile's keys, or values
constexpr int kStage = 2 * kSide;

// The next tile a group's stages take: its place on the line and its cell.
struct Cursor {
  int at, seq, layer, tile, tiles;
};

// The largest P' = 2^(x - m) * scale of a step is set to about 2^kTop when the
// reference m moves, and m moves when it would pass 2^(kTop + kSlack), below
// fp16's largest: the smaller weights and the groups of smaller scale then keep
// as much of fp16's range below it as there is.
constexpr float kTop = 7.0f, kSlack = 8.0f;

__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8(int* d, const uint32_t* a, uint32_t b0, uint32_t b1, const int* c) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}

// Integer accumulators start at the bits of 1.5 * 2^23: read as f32, they are
// that number plus the sum (|sum| <= 127 * 112 * 32 < 2^22).
constexpr int kZeroBits = 0x4b400000;
constexpr float kZero = 12582912.0f;
__device__ __forceinline__ float2 sums(int a, int b) {
  return __fadd2_rn(make_float2(__int_as_float(a), __int_as_float(b)), make_float2(-kZero, -kZero));
}

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_half(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// Four integers' parts of `shift` bits and up, rounded, as bytes; y becomes the
// rest.
__device__ __forceinline__ uint32_t take_bytes(int* y, int shift) {
  uint32_t w = 0u;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int part = shift ? (y[e] + (1 << shift >> 1)) >> shift : y[e];
    y[e] -= part << shift;
    w |= ((uint32_t)part & 255u) << (8 * e);
  }
  return w;
}

// Nibbles 0 and 4 of w (low: bits 0 and 16) as fp16 c - 7: 0x6400 | c is 1024 +
// c. `magic` is 0x64006400 in a register, read from memory so that it stays there:
// with two constants the mask and the or are two instructions.
__device__ __forceinline__ uint32_t codes_low(uint32_t w, uint32_t magic) {
  const uint32_t x = (w & 0x000f000fu) | magic;
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), __float2half2_rn(1031.0f));
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Nibbles 1 and 5: 0x6400 | 16 c is 1024 + 16 c.
__device__ __forceinline__ uint32_t codes_high(uint32_t w, uint32_t magic) {
  const uint32_t x = (w & 0x00f000f0u) | magic;
  const __half2 h = __hfma2(*reinterpret_cast<const __half2*>(&x), __float2half2_rn(0.0625f), __float2half2_rn(-71.0f));
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Add one to a shared counter; the caller's reads of the stage are ordered
// before it, those of the others' before the last caller's return.
__device__ __forceinline__ unsigned count_up(unsigned* counter) {
  unsigned old;
  asm volatile("atom.acq_rel.cta.shared::cta.add.u32 %0, [%1], 1;" : "=r"(old) : "r"(smem_addr(counter)) : "memory");
  return old;
}

template <int N>
struct Words {  // N 16-bit halves per row and lane
  uint32_t w[N / 2];
  __device__ __forceinline__ void load(const unsigned char* p) {
    if constexpr (N == 4) {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      w[0] = u.x;
      w[1] = u.y;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
  }
};

template <class M>
struct Dec {
  static constexpr int NG = M::D / 32;
  static constexpr int KVU = 8 / M::G;            // kv heads of a unit of eight query heads
  static constexpr int UNITS = M::HKV / KVU;
  static constexpr int PARTS = 4 / UNITS;         // of a tile's rows, a warp each
  static constexpr int ROWS = kQ4Tile / PARTS, BLOCKS = ROWS / 8;
  static constexpr int WARPS = 2 * PARTS;         // of a unit, both groups
  static constexpr int OWN = 2 * NG / WARPS;      // blocks of 16 dims that a warp of a unit writes out
  static constexpr int OFF_SWAP = kStages * kStage;   // [warp][lane] float4
  static constexpr int OFF_STAT = OFF_SWAP + 8 * 32 * 16;  // [warp][8 heads] (m, l)
  static constexpr int OFF_BAR = OFF_STAT + 8 * 8 * 8;
  static constexpr int OFF_DONE = OFF_BAR + 8 * kStages;
  static constexpr int OFF_CURSOR = OFF_DONE + 4 * kStages;
  static constexpr int OFF_MAGIC = OFF_CURSOR + 2 * (int)sizeof(Cursor);
  static constexpr int SMEM = OFF_MAGIC + 4;
  static_assert(2 * (SMEM + 1024) <= 228 * 1024, "two CTAs an SM");
};

// What an output type asks for: queries of four terms of 7 bits (else two),
// weights of two fp16 terms (else one).
template <int OUT>
struct Need {
  static constexpr bool QUERY = OUT != 1, WEIGHT = OUT == 0;
  static constexpr int PAIRS = QUERY ? 2 : 1;
};

// The rotated queries of a unit as MMA operands: pairs of terms.
template <class M, int PAIRS>
struct Query {
  uint32_t a[M::D / 32][PAIRS][4];
  float unit;  // base-2 logit of the first pair's sum
};

// Lane (g, t) holds dims 32 j + 8 t .. + 7 of query head g of the unit:
// rotation pairs are in the lane, norms in the quad.
template <class M, int PAIRS>
__device__ __forceinline__ bool load_query(const Q4DecodeParams& p, long long first_head, int position,
                                           Query<M, PAIRS>* out) {
  constexpr int NG = M::D / 32;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long base = (first_head + g) * M::D + 8 * t;
  float x[NG * 8];
#pragma unroll
  for (int j = 0; j < NG; ++j) load8(p.q, base + 32 * j, p.q_dtype, p.vec, x + 8 * j);
  if constexpr (M::QWEN) {
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      s[e] = fmaf(x[e], x[e], x[8 + e] * x[8 + e]) + fmaf(x[16 + e], x[16 + e], x[24 + e] * x[24 + e]);
    float sum = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    float inv = __frcp_rn(__fsqrt_rn(fmaf(sum, 1.0f / M::D, 1.0e-6f)));
    if (__any_sync(0xffffffffu, !isfinite(sum))) {
      const float exact = exact_inv_rms<M, NG * 8, 4>(x);
      if (!isfinite(sum)) inv = exact;
    }
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[8 * j + e] = __fmul_rn(__fmul_rn(x[8 * j + e], inv), p.q_norm ? p.q_norm[32 * j + 8 * t + e] : 1.0f);
  }
  const float2* tab = p.rope + (long long)position * (M::D / 2) + 8 * t;
  bool good = true;
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < NG / 2; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float l = x[8 * j + e], r = x[8 * (j + NG / 2) + e];
      const float2 c = tab[32 * j + e];
      float a, b;
      if constexpr (M::QWEN) {
        a = __fsub_rn(__fmul_rn(l, c.x), __fmul_rn(r, c.y));
        b = __fadd_rn(__fmul_rn(r, c.x), __fmul_rn(l, c.y));
      } else {
        a = __fmaf_rn(-r, c.x, __fmul_rn(l, c.y));
        b = __fmaf_rn(r, c.y, __fmul_rn(l, c.x));
      }
      x[8 * j + e] = a;
      x[8 * (j + NG / 2) + e] = b;
      good &= isfinite(a) && isfinite(b);
      top = fmaxf(top, fmaxf(fabsf(a), fabsf(b)));
    }
  if (p.q_rot_out) {
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) p.q_rot_out[base + 32 * j + e] = x[8 * j + e];
  }
  // the head's largest element to 126 * 2^7 (126 * 2^21): its first term, rounded,
  // then stays within a byte; a code counts 16
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)), 1e-30f);
  constexpr float MOST = PAIRS == 2 ? 126.0f * 2097152.0f : 126.0f * 128.0f;
  const float up = MOST / top;
  out->unit = M::SCALE * 1.4426950408889634f / 16.0f * (top / (126.0f * 128.0f));
#pragma unroll
  for (int j = 0; j < NG; ++j)
#pragma unroll
    for (int s = 0; s < 2; ++s) {  // dims 8 t .. + 3, 8 t + 4 .. + 7
      int y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = __float2int_rn(x[8 * j + 4 * s + e] * up);
      if constexpr (PAIRS == 2) {
        out->a[j][0][2 * s] = take_bytes(y, 21);
        out->a[j][0][2 * s + 1] = take_bytes(y, 14);
      }
      out->a[j][PAIRS - 1][2 * s] = take_bytes(y, 7);
      out->a[j][PAIRS - 1][2 * s + 1] = take_bytes(y, 0);
    }
  return good;
}

// Before the attention: per (sequence, layer) the queries normed (Qwen), rotated
// and cut into operands, the new token's rows quantised into the arena. A warp
// per unit of eight query heads, four for the keys' and values' heads.
template <class M, int PAIRS>
__global__ void __launch_bounds__(256) qx_q4_prepare_kernel(const __grid_constant__ Q4DecodeParams p) {
  using C = Dec<M>;
  using R = Q4Row<M>;
  constexpr int NG = C::NG;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i = blockIdx.x / p.layer_count, layer = blockIdx.x - i * p.layer_count;
  const Q4Seq seq = p.seqs[i];
  const int position = seq.begin - 1;
  const long long cell = (long long)p.seq_begin * p.layer_count + blockIdx.x;  // of the call
  pdl_wait();
  // The attention grid may start: every grid before this one has completed, so it
  // may read all rows but the new ones, for which it waits.
  pdl_launch_dependents();
  bool good;
  if (warp < C::UNITS) {
    Query<M, PAIRS> query;
    good = load_query<M, PAIRS>(p, cell * M::HQ + 8 * warp, position, &query);
    uint4* out = p.operands + ((long long)blockIdx.x * C::UNITS + warp) * NG * PAIRS * 32 + lane;
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
      for (int a = 0; a < PAIRS; ++a)
        out[(j * PAIRS + a) * 32] = make_uint4(query.a[j][a][0], query.a[j][a][1], query.a[j][a][2], query.a[j][a][3]);
    if ((lane & 3) == 0) p.units[(long long)blockIdx.x * M::HQ + 8 * warp + (lane >> 2)] = query.unit;
  } else {
    const int at = 32 * (warp - C::UNITS) + lane, c = at & (R::LPH - 1), h = at / R::LPH % M::HKV;
    const bool value = at >= M::HKV * R::LPH;  // the same for a whole warp
    const long long row = kv_row(p.arena.paging, p.arena.capacity, p.arena.layers, seq.seq, p.layer_begin + layer, position);
    float x[8];
    load8(value ? p.v : p.k, (cell * M::HKV + h) * M::D + 8 * c, p.in_dtype, p.vec, x);
    uint32_t codes[8];
    __half scale;
    if (value) {
      good = quantise8(x, 7, codes, &scale);
      put_value<M>(p.arena.v + row * kQ4RowBytes, h, c, value_halves(codes), scale);
    } else {
      float2 tab[8];
      rope_of_lane<M>(p.rope, position, c, tab);
      rotate_key<M>(x, c, p.k_norm, tab);
      good = quantise8(x, 0, codes, &scale);
      put_key<M>(p.arena.k + row * kQ4RowBytes, h, c, key_codes(codes), scale);
    }
  }
  if (!good) flag_error(p.err, QX_ERR_BIT_NONFINITE);
}

template <class M, int OUT>
__global__ void __launch_bounds__(kThreads, 2) qx_q4_decode_kernel(const __grid_constant__ Q4DecodeParams p) {
  using C = Dec<M>;
  using R = Q4Row<M>;
  constexpr int NG = C::NG, KVU = C::KVU, PAIRS = Need<OUT>::PAIRS;
  constexpr bool PRECISE = Need<OUT>::WEIGHT;
  extern __shared__ __align__(128) unsigned char sm[];
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + C::OFF_BAR);
  unsigned* done = reinterpret_cast<unsigned*>(sm + C::OFF_DONE);
  Cursor* cursor = reinterpret_cast<Cursor*>(sm + C::OFF_CURSOR);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int group = warp >> 2, unit = (warp & 3) / C::PARTS, part = warp & (C::PARTS - 1);
  // this CTA's stretch of the line, and the cell it starts in
  const int start = blockIdx.x * p.per_cta;
  auto tiles_of = [&](int i) { return (p.seqs[i].begin + kQ4Tile - 1) / kQ4Tile; };
  int seq = find_seq(p.seqs, p.n_seq, start), tiles = tiles_of(seq);
  const int place = p.padded ? (tiles + p.per_cta - 1) / p.per_cta * p.per_cta : tiles;
  int layer = (start - p.seqs[seq].first) / place, tile = (start - p.seqs[seq].first) - layer * place;
  const int end = p.padded ? start + min(p.per_cta, tiles - tile) : min(start + p.per_cta, p.total);
  bool ok = true;

  // one tile further
  auto advance = [&](Cursor& c) {
    ++c.at;
    if (++c.tile < c.tiles) return;
    c.tile = 0;
    if (++c.layer == p.layer_count) {
      c.layer = 0;
      if (++c.seq < p.n_seq) c.tiles = tiles_of(c.seq);
    }
  };
  auto issue = [&](const Cursor& c) {
    const int s = (c.at - start) % kStages, begin = c.tile * kQ4Tile;
    const long long row = kv_row(p.arena.paging, p.arena.capacity, p.arena.layers, p.seqs[c.seq].seq,
                                 p.layer_begin + c.layer, begin);
    const uint32_t bytes = min(kQ4Tile, p.seqs[c.seq].begin - begin) * kQ4RowBytes;
    mbar_arrive_expect_tx(&full[s], 2u * bytes);
    bulk_load(sm + s * kStage, p.arena.k + row * kQ4RowBytes, bytes, &full[s]);
    bulk_load(sm + s * kStage + kSide, p.arena.v + row * kQ4RowBytes, bytes, &full[s]);
  };
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      done[s] = 0u;
    }
    *reinterpret_cast<volatile uint32_t*>(sm + C::OFF_MAGIC) = 0x64006400u;
    fence_barrier_init();
    // Rows of earlier calls may be read before the wait: qx_q4_prepare_kernel, the
    // grid before this one, lets this one start only when all before it are
    // complete. A cell's last tile has the row which that grid writes.
    Cursor c = {start, seq, layer, tile, tiles};
    bool waited = false;
    for (int k = 0; k < kStages && c.at < end; ++k) {
      if (c.tile == c.tiles - 1 && !waited) {
        pdl_wait();
        waited = true;
      }
      issue(c);
      advance(c);
    }
    cursor[c.at & 1 ^ start & 1] = c;
    advance(c);
    cursor[c.at & 1 ^ start & 1] = c;
  }
  __syncthreads();
  const uint32_t magic = *reinterpret_cast<volatile uint32_t*>(sm + C::OFF_MAGIC);
  pdl_wait();
  pdl_launch_dependents();

  // the cache row that MMA row (or column) g stands for, and those of 2 t and 2 t + 1
  const int row_g = (g & 1) ? 4 + ((g >> 1) ^ 2) : g >> 1, row_a = t, row_b = 4 + (t ^ 2);
  const int own = KVU == 1 ? 0 : g / M::G;  // kv head of query head g within the unit
  const int scale_at = R::scale(unit * KVU + own, 0);
  const int zero[4] = {kZeroBits, kZeroBits, kZeroBits, kZeroBits};
  bool good = true;

  for (int at = start; at < end;) {  // cell by cell
  const int n_tiles = min(end - at, tiles - tile);  // of this cell in this CTA
  const int attend = p.seqs[seq].begin;
  const long long here = (long long)seq * p.layer_count + layer;  // the cell within the launch
  Query<M, PAIRS> query;
  {
    const uint4* in = p.operands + (here * C::UNITS + unit) * NG * PAIRS * 32 + lane;
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
      for (int a = 0; a < PAIRS; ++a) {
        const uint4 w = in[(j * PAIRS + a) * 32];
        query.a[j][a][0] = w.x, query.a[j][a][1] = w.y, query.a[j][a][2] = w.z, query.a[j][a][3] = w.w;
      }
    query.unit = p.units[here * M::HQ + 8 * unit + g];
  }

  float o[2 * NG][4];
#pragma unroll
  for (int m = 0; m < 2 * NG; ++m)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[m][e] = 0.0f;
  float m = -INFINITY;  // of query head g, this lane's rows
  float2 sum = make_float2(0.0f, 0.0f);

  for (int k = (at - start + group) & 1; k < n_tiles; k += 2) {  // this group's tiles
    const int kk = at - start + k, s = kk % kStages;
    unsigned char* data = sm + s * kStage;
    const int valid = min(kQ4Tile, attend - (tile + k) * kQ4Tile);
    if (ok) ok = mbar_wait_bounded(&full[s], (uint32_t)(kk / kStages) & 1u, p.err);
    __syncwarp();
    const int r0 = C::ROWS * part;
    if (r0 < valid) {
      const unsigned char* ks = data + r0 * kQ4RowBytes;
      const unsigned char* vs = ks + kSide;
      // ---- scores: x[n] = rows 8 n + row_a, 8 n + row_b of head g, Granite's two
      // blocks at a time so that its masked operands serve both
      constexpr int NB = KVU == 1 ? 1 : 2;
      float2 x[C::BLOCKS];
#pragma unroll
      for (int n0 = 0; n0 < C::BLOCKS; n0 += NB) {
        int c[NB][NG][PAIRS][4];
#pragma unroll
        for (int kv = 0; kv < KVU; ++kv) {
          uint32_t w[NB][NG];
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            const unsigned char* kr = ks + (8 * (n0 + n) + row_g) * kQ4RowBytes + (unit * KVU + kv) * R::HEAD + 4 * NG * t;
            if constexpr (NG == 4) {
              const uint4 u = *reinterpret_cast<const uint4*>(kr);
              w[n][0] = u.x, w[n][1] = u.y, w[n][2] = u.z, w[n][3] = u.w;
            } else {
              const uint2 u = *reinterpret_cast<const uint2*>(kr);
              w[n][0] = u.x, w[n][1] = u.y;
            }
          }
#pragma unroll
          for (int j = 0; j < NG; ++j) {
            uint32_t a[PAIRS][4];
#pragma unroll
            for (int i2 = 0; i2 < PAIRS; ++i2)
#pragma unroll
              for (int e = 0; e < 4; ++e) a[i2][e] = KVU == 1 || own == kv ? query.a[j][i2][e] : 0u;
#pragma unroll
            for (int n = 0; n < NB; ++n) {
              const uint32_t b0 = w[n][j] & 0xf0f0f0f0u, b1 = (w[n][j] << 4) & 0xf0f0f0f0u;
#pragma unroll
              for (int i2 = 0; i2 < PAIRS; ++i2) mma_s8(c[n][j][i2], a[i2], b0, b1, kv == 0 ? zero : c[n][j][i2]);
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          Words<NG> sa, sb;
          sa.load(ks + (8 * (n0 + n) + row_a) * kQ4RowBytes + scale_at);
          sb.load(ks + (8 * (n0 + n) + row_b) * kQ4RowBytes + scale_at);
          float2 acc = make_float2(0.0f, 0.0f);
#pragma unroll
          for (int j = 0; j < NG; ++j) {
            const float2 fa = unpack_half(sa.w[j / 2]), fb = unpack_half(sb.w[j / 2]);
            float2 dot = __ffma2_rn(sums(c[n][j][0][0], c[n][j][0][1]), make_float2(128.0f, 128.0f),
                                    sums(c[n][j][0][2], c[n][j][0][3]));
            if constexpr (PAIRS == 2) {
              const float2 low = __ffma2_rn(sums(c[n][j][1][0], c[n][j][1][1]), make_float2(128.0f, 128.0f),
                                            sums(c[n][j][1][2], c[n][j][1][3]));
              dot = __ffma2_rn(low, make_float2(1.0f / 16384.0f, 1.0f / 16384.0f), dot);
            }
            acc = __ffma2_rn(make_float2(j & 1 ? fa.y : fa.x, j & 1 ? fb.y : fb.x), dot, acc);
          }
          x[n0 + n] = __fmul2_rn(acc, make_float2(query.unit, query.unit));
        }
      }
      Words<NG> va[C::BLOCKS], vb[C::BLOCKS];  // scales of the values
#pragma unroll
      for (int n = 0; n < C::BLOCKS; ++n) {
        va[n].load(vs + (8 * n + row_a) * kQ4RowBytes + scale_at);
        vb[n].load(vs + (8 * n + row_b) * kQ4RowBytes + scale_at);
      }
      if (r0 + C::ROWS > valid) {  // rows past the last: no weight, and no garbage for a scale
#pragma unroll
        for (int n = 0; n < C::BLOCKS; ++n) {
          if (r0 + 8 * n + row_a >= valid) {
            x[n].x = -INFINITY;
#pragma unroll
            for (int e = 0; e < NG / 2; ++e) va[n].w[e] = 0u;
          }
          if (r0 + 8 * n + row_b >= valid) {
            x[n].y = -INFINITY;
#pragma unroll
            for (int e = 0; e < NG / 2; ++e) vb[n].w[e] = 0u;
          }
        }
      }
      // ---- reference m, from the largest score plus the exponent of the
      // largest scale
      float top = fmaxf(x[0].x, x[0].y);
      uint32_t most = 0u;
#pragma unroll
      for (int n = 1; n < C::BLOCKS; ++n) top = fmax3f(top, x[n].x, x[n].y);
#pragma unroll
      for (int n = 0; n < C::BLOCKS; ++n)
#pragma unroll
        for (int e = 0; e < NG / 2; ++e) most = __vimax3_u16x2(most, va[n].w[e], vb[n].w[e]);
      top += (float)(int)(max(most & 0xffffu, most >> 16) >> 10) - 14.0f;
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)) - kTop;
      const bool raise = top > m + kSlack;  // always in the first step (m = -inf)
      if (__any_sync(0xffffffffu, raise)) {
        const float keep = raise ? fast_exp2(m - top) : 1.0f;
        if (raise) m = top;
        sum = __fmul2_rn(sum, make_float2(keep, keep));
        const float k0 = __shfl_sync(0xffffffffu, keep, 8 * t), k1 = __shfl_sync(0xffffffffu, keep, 8 * t + 4);
#pragma unroll
        for (int e = 0; e < 2 * NG; ++e) {
          o[e][0] *= k0;
          o[e][1] *= k1;
          o[e][2] *= k0;
          o[e][3] *= k1;
        }
      }
#pragma unroll
      for (int n = 0; n < C::BLOCKS; ++n) {
        x[n] = __fadd2_rn(x[n], make_float2(-m, -m));
        x[n] = make_float2(fast_exp2(x[n].x), fast_exp2(x[n].y));
        sum = __fadd2_rn(sum, x[n]);
      }
      // ---- O^T += V^T P'^T, 16 rows at a time
#pragma unroll
      for (int n = 0; n < C::BLOCKS; n += 2) {
        // the operand of group j: rows 2 t, 2 t + 1 of both blocks, head g
        uint32_t h0[NG], h1[NG], l0[NG], l1[NG];
        auto weights = [&](int j) {
          const float2 a0 = unpack_half(va[n].w[j / 2]), b0 = unpack_half(vb[n].w[j / 2]);
          const float2 a1 = unpack_half(va[n + 1].w[j / 2]), b1 = unpack_half(vb[n + 1].w[j / 2]);
          const float2 p0 = __fmul2_rn(x[n], make_float2(j & 1 ? a0.y : a0.x, j & 1 ? b0.y : b0.x));
          const float2 p1 = __fmul2_rn(x[n + 1], make_float2(j & 1 ? a1.y : a1.x, j & 1 ? b1.y : b1.x));
          h0[j] = pack_half(p0.x, p0.y), h1[j] = pack_half(p1.x, p1.y);
          if constexpr (PRECISE) {
            const float2 q0 = unpack_half(h0[j]), q1 = unpack_half(h1[j]);
            l0[j] = pack_half(p0.x - q0.x, p0.y - q0.y), l1[j] = pack_half(p1.x - q1.x, p1.y - q1.y);
          }
        };
        if constexpr (KVU > 1) {
#pragma unroll
          for (int j = 0; j < NG; ++j) weights(j);
        }
#pragma unroll
        for (int kv = 0; kv < KVU; ++kv) {
          const bool mine = KVU == 1 || own == kv;
          Words<NG> ca0, cb0, ca1, cb1;
          const unsigned char* vr = vs + 8 * n * kQ4RowBytes + (unit * KVU + kv) * R::HEAD + 2 * NG * g;
          ca0.load(vr + row_a * kQ4RowBytes);
          cb0.load(vr + row_b * kQ4RowBytes);
          ca1.load(vr + (8 + row_a) * kQ4RowBytes);
          cb1.load(vr + (8 + row_b) * kQ4RowBytes);
#pragma unroll
          for (int j = 0; j < NG; ++j) {
            if constexpr (KVU == 1) weights(j);
            // half j of the rows: low 16 bits row a, high 16 bits row b
            const uint32_t pick = j & 1 ? 0x7632u : 0x5410u;
            const uint32_t z0 = __byte_perm(ca0.w[j / 2], cb0.w[j / 2], pick);
            const uint32_t z1 = __byte_perm(ca1.w[j / 2], cb1.w[j / 2], pick);
            const uint32_t p0 = mine ? h0[j] : 0u, p1 = mine ? h1[j] : 0u;
            const uint32_t c00 = codes_low(z0, magic), c01 = codes_high(z0, magic);
            const uint32_t c02 = codes_low(z0 >> 8, magic), c03 = codes_high(z0 >> 8, magic);
            const uint32_t c10 = codes_low(z1, magic), c11 = codes_high(z1, magic);
            const uint32_t c12 = codes_low(z1 >> 8, magic), c13 = codes_high(z1 >> 8, magic);
            mma_f16(o[2 * j], c00, c01, c10, c11, p0, p1);
            mma_f16(o[2 * j + 1], c02, c03, c12, c13, p0, p1);
            if constexpr (PRECISE) {
              const uint32_t q0 = mine ? l0[j] : 0u, q1 = mine ? l1[j] : 0u;
              mma_f16(o[2 * j], c00, c01, c10, c11, q0, q1);
              mma_f16(o[2 * j + 1], c02, c03, c12, c13, q0, q1);
            }
          }
        }
      }
    }
    // the last warp of the group to finish a tile refills its stage; a warp whose
    // wait ran out neither waits nor counts again, so no stage of its group is
    // refilled from then on
    __syncwarp();
    if (lane == 0 && ok && count_up(&done[s]) == 3u) {
      done[s] = 0u;
      Cursor c = cursor[group];
      if (c.at < end) {
        issue(c);
        advance(c);
        advance(c);
        cursor[group] = c;
      }
    }
  }

  // ---- the sums of a unit's warps meet: each warp of the unit writes OWN blocks of
  // 16 dims and gets the others' shares of them through shared memory, one block a
  // round (a fragment is the same lanes' in every warp)
  {
    const bool whole = n_tiles == tiles;
    const long long slot = 2ll * blockIdx.x + (at == start ? 0 : 1);
    const int w = group * C::PARTS + part;  // this warp among its unit's
    auto warp_of = [&](int i) { return i / C::PARTS * 4 + unit * C::PARTS + i % C::PARTS; };
    float2* stat = reinterpret_cast<float2*>(sm + C::OFF_STAT);
    float4* swap = reinterpret_cast<float4*>(sm + C::OFF_SWAP);
    float all = sum.x + sum.y;
    all += __shfl_xor_sync(0xffffffffu, all, 1);
    all += __shfl_xor_sync(0xffffffffu, all, 2);
    if (t == 0) stat[warp * 8 + g] = make_float2(m, all);
    named_sync(1 + unit, 32 * C::WARPS);
    float top = -INFINITY, den = 0.0f;
#pragma unroll
    for (int i = 0; i < C::WARPS; ++i) top = fmaxf(top, stat[warp_of(i) * 8 + g].x);
#pragma unroll
    for (int i = 0; i < C::WARPS; ++i) {
      const float2 ml = stat[warp_of(i) * 8 + g];
      den = fmaf(fast_exp2(ml.x - top), ml.y, den);
    }
    if (!whole && w == 0 && t == 0) p.part_ml[slot * M::HQ + 8 * unit + g] = make_float2(top, den);
    const float scale = fast_exp2(m - top) * (whole ? 1.0f / den : 1.0f);
    const float k0 = __shfl_sync(0xffffffffu, scale, 8 * t), k1 = __shfl_sync(0xffffffffu, scale, 8 * t + 4);
    auto block = [&](int e) {  // the fragment of dims 16 e .., scaled
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < 2 * NG; ++i)
        if (i == e) v = make_float4(o[i][0] * k0, o[i][1] * k1, o[i][2] * k0, o[i][3] * k1);
      return v;
    };
#pragma unroll
    for (int b = 0; b < C::OWN; ++b) {
      const int mine = w * C::OWN + b;
      float4 v = block(mine);
#pragma unroll
      for (int r = 1; r < C::WARPS; ++r) {
        swap[warp * 32 + lane] = block((w + r) % C::WARPS * C::OWN + b);
        named_sync(1 + unit, 32 * C::WARPS);
        const float4 x = swap[warp_of((w + C::WARPS - r) % C::WARPS) * 32 + lane];
        v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
        named_sync(1 + unit, 32 * C::WARPS);
      }
      // heads 2 t and 2 t + 1, dims 16 mine + g and 8 further
      const long long e = (8 * unit + 2 * t) * M::D + 16 * mine + g;
      if (!whole) {
        float* out = p.part_o + slot * M::HQ * M::D + e;
        out[0] = v.x, out[M::D] = v.y, out[8] = v.z, out[M::D + 8] = v.w;
      } else {
        good &= isfinite(v.x) && isfinite(v.y) && isfinite(v.z) && isfinite(v.w);
        const long long out = ((long long)p.seq_begin * p.layer_count + here) * M::HQ * M::D + e;
        store_any(p.out, out, OUT, v.x);
        store_any(p.out, out + M::D, OUT, v.y);
        store_any(p.out, out + 8, OUT, v.z);
        store_any(p.out, out + M::D + 8, OUT, v.w);
      }
    }
  }
  at += n_tiles;
  tile = 0;
  if (++layer == p.layer_count) {
    layer = 0;
    if (++seq < p.n_seq) tiles = tiles_of(seq);
  }
  }
  if (!ok && lane == 0) {  // what is still on its way to the group's stages lands before the CTA exits
    const int issued = cursor[group].at;
    for (int at = max(start + group, issued - kStages); at < min(issued, end); at += 2)
      mbar_wait_bounded(&full[(at - start) % kStages], (uint32_t)((at - start) / kStages) & 1u, p.err);
  }
  if (!good && ok) flag_error(p.err, QX_ERR_BIT_NONFINITE);
}

// Cells shared by CTAs: a CTA joins 1024 / SHARES outputs of a cell, SHARES
// threads (of neighbouring 256 / SHARES) taking every SHARES-th part of the same
// four. One share where cells have few parts, 32 (then 32 dims of one head)
// where they have many: more than 8 of a Granite cell, 16 of a Qwen3 one, whose 128
// CTAs a cell then cost more. Always one against always 32, the decode as a whole in us:
//   Granite  128 sequences of 2 or 3 parts 120.8 | 149.3; 40 of 9 25.6 | 26.2, 36 of 9
//            25.3 | 25.1, 28 of 12 22.2 | 21.1, 20 of 15 19.8 | 16.3, 8 of 19 15.6 | 12.7
//   Qwen3    48 of 2 to 7 68.5 | 95.3; 40 of 9 30.9 | 41.6, 28 of 12 25.1 | 30.9, 20 of
//            16 52.2 | 55.0, 12 of 17 21.2 | 21.2, 8 of 19 18.8 | 16.7, 10 of 31 36.9 |
//            31.5, one of 32 14.7 | 9.3, of 147 42.2 | 14.2
template <class M, int SHARES>
__global__ void __launch_bounds__(256) qx_q4_merge_kernel(const __grid_constant__ Q4DecodeParams p) {
  constexpr int E = 1024 / SHARES, SLICES = M::HQ * M::D / E, LANES = 256 / SHARES;
  __shared__ float red[SHARES == 1 ? 1 : SHARES][E + 4];
  __shared__ float2 stat[SHARES];
  const int tid = threadIdx.x, slice = blockIdx.x % SLICES, cell = blockIdx.x / SLICES;
  const int i = cell / p.layer_count, layer = cell - i * p.layer_count;
  const int tiles = (p.seqs[i].begin + kQ4Tile - 1) / kQ4Tile;
  const int place = p.padded ? (tiles + p.per_cta - 1) / p.per_cta * p.per_cta : tiles;
  const int first = p.seqs[i].first + layer * place;
  const int b0 = first / p.per_cta, parts = (first + tiles - 1) / p.per_cta - b0 + 1;
  // Before any CTA leaves: cells whose borders are CTA borders are all whole, and a grid
  // that did not wait would be complete while the attention still runs, with nothing to
  // keep the stream's next kernel from its workspace and rows.
  pdl_wait();
  if (parts == 1) return;
  const int share = tid / LANES, e = slice * E + 4 * (tid % LANES), qh = e / M::D;
  // the first part lies in slot 1 of its CTA unless it is the CTA's first cell
  auto slot = [&](int s) { return 2ll * (b0 + s) + (s == 0 && first != b0 * p.per_cta ? 1 : 0); };
  float top = -INFINITY, den = 0.0f;
  for (int s = share; s < parts; s += SHARES) top = fmaxf(top, p.part_ml[slot(s) * M::HQ + qh].x);
  float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int s = share; s < parts; s += SHARES) {
    const float2 ml = p.part_ml[slot(s) * M::HQ + qh];
    const float4 v = *reinterpret_cast<const float4*>(p.part_o + slot(s) * M::HQ * M::D + e);
    const float w = fast_exp2(ml.x - top);
    den = fmaf(w, ml.y, den);
    y.x = fmaf(w, v.x, y.x);
    y.y = fmaf(w, v.y, y.y);
    y.z = fmaf(w, v.z, y.z);
    y.w = fmaf(w, v.w, y.w);
  }
  const long long out = ((long long)p.seq_begin * p.layer_count + cell) * M::HQ * M::D;
  bool good = true;
  if constexpr (SHARES == 1) {
    const float o[4] = {y.x / den, y.y / den, y.z / den, y.w / den};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      good &= isfinite(o[c]);
      store_any(p.out, out + e + c, p.out_dtype, o[c]);
    }
  } else {
    static_assert(SHARES == 1 || M::D % E == 0, "a CTA's outputs are one head's");
    *reinterpret_cast<float4*>(&red[share][4 * (tid % LANES)]) = y;
    if (tid % LANES == 0) stat[share] = make_float2(top, den);
    __syncthreads();
    if (tid < E) {
      float all = -INFINITY, num = 0.0f, sum = 0.0f;
#pragma unroll 8
      for (int s = 0; s < SHARES; ++s) all = fmaxf(all, stat[s].x);
#pragma unroll 8
      for (int s = 0; s < SHARES; ++s) {
        const float w = fast_exp2(stat[s].x - all);
        sum = fmaf(w, stat[s].y, sum);
        num = fmaf(w, red[s][tid], num);
      }
      const float o = num / sum;
      good = isfinite(o);
      store_any(p.out, out + slice * E + tid, p.out_dtype, o);
    }
  }
  if (!good) flag_error(p.err, QX_ERR_BIT_NONFINITE);
}

cudaError_t launch_dependent(void (*fn)(Q4DecodeParams), int blocks, int threads, int smem, cudaStream_t stream,
                             const Q4DecodeParams& p, int* launched) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, p);
  if (e == cudaSuccess) ++*launched;
  return e;
}

template <class M, int OUT>
cudaError_t setup() {
  return cudaFuncSetAttribute(qx_q4_decode_kernel<M, OUT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Dec<M>::SMEM);
}

template <class M, int OUT>
cudaError_t decode(const Q4DecodeParams& p, cudaStream_t stream, int* launched) {
  const int cells = p.n_seq * p.layer_count, ctas = (p.total + p.per_cta - 1) / p.per_cta;
  cudaError_t e = launch_dependent(qx_q4_prepare_kernel<M, Need<OUT>::PAIRS>, cells, 32 * (Dec<M>::UNITS + 4), 0, stream, p, launched);
  if (e == cudaSuccess) e = launch_dependent(qx_q4_decode_kernel<M, OUT>, ctas, kThreads, Dec<M>::SMEM, stream, p, launched);
  if (e != cudaSuccess || p.max_parts == 1) return e;
  constexpr int OUTPUTS = M::HQ * M::D;
  if (p.max_parts <= (M::QWEN ? 16 : 8))
    return launch_dependent(qx_q4_merge_kernel<M, 1>, cells * (OUTPUTS / 1024), 256, 0, stream, p, launched);
  return launch_dependent(qx_q4_merge_kernel<M, 32>, cells * (OUTPUTS / 32), 256, 0, stream, p, launched);
}

}  // namespace

cudaError_t setup_q4_decode() {
  for (cudaError_t e : {setup<Qwen3Heads, 0>(), setup<Qwen3Heads, 1>(), setup<Qwen3Heads, 2>(), setup<GraniteHeads, 0>(),
                        setup<GraniteHeads, 1>(), setup<GraniteHeads, 2>()})
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}

cudaError_t launch_q4_decode(bool qwen, const Q4DecodeParams& p, cudaStream_t stream, int* launched) {
  *launched = 0;
  if (p.out_dtype == 0) return qwen ? decode<Qwen3Heads, 0>(p, stream, launched) : decode<GraniteHeads, 0>(p, stream, launched);
  if (p.out_dtype == 1) return qwen ? decode<Qwen3Heads, 1>(p, stream, launched) : decode<GraniteHeads, 1>(p, stream, launched);
  return qwen ? decode<Qwen3Heads, 2>(p, stream, launched) : decode<GraniteHeads, 2>(p, stream, launched);
}

int q4_decode_blocks_per_sm() { return 2; }

}  // namespace qx
