// packed.cu — causal attention of whole prompts packed one after another, on
// tcgen05 tensor cores.
//
// A work item is a block of a prompt's tokens and one kv head: two query tiles
// of 128 rows, each 128 / G tokens x the kv head's G query heads, so the heads
// of a group share every key and value tile. The grid has one CTA per item, longest
// first; a CTA that is running takes further items by cancelling CTAs that are not
// launched yet, so the next item's loads and first scores are under way while the
// last one's outputs are written, and its set-up is paid once:
//   warp 9      TMA producer, one thread: loads an item's query tiles, each as soon
//               as the last scores of the tile before are done, and its key and
//               value tiles of 128 tokens through one ring in the order of their
//               use, then asks for the next item
//   warp 8      MMA issuer, one lane: for each tile in turn O += P V, then the
//               next scores S = Q K^T, so one tile's products run while the
//               other's softmax does
//   warps 0-3, 4-7  the softmax of the first, the second tile: a thread owns a
//               row, reads its 128 scores from TMEM, writes 128 weights over
//               them as 16-bit pairs (the A operand of P V). The row's
//               reference moves only when its maximum passes it by 2^8; then
//               the thread rescales its row of O in TMEM, which no product
//               uses while the tile's scores are being read.
// S of a tile is issued after its P V, and tensor instructions of one thread
// complete in order: once S is there, P may be overwritten and O is settled. An
// item's first P V starts O afresh; its weights are written after the tile's
// threads have read the last item's O.
//
// Measured, medians: a Qwen3 prompt of 16384 tokens 1.58 to 1.64 ms for a moment (1340
// to 1390 TFLOP/s of the causal half; a library product of bf16 matrices reaches 1646
// for a moment, 1373 for seconds), 1.85 ms call after call at the power cap; 11 ragged
// Qwen3 prompts of together 12345 tokens 165 us (1000), one of 2048 34 to 35 us; 3
// Granite prompts of 8200 tokens 176 to 180 us (765 to 780), 200 to 230 in replays
// back to back, one of 4096 51 to 54 us (635 to 670), 7 of 777 9.3 us. A step,
// both tiles against a key tile, takes 3100 cycles of which the tensor pipe needs 2048: a tile's scores (512, and about 270 to hand them over), its
// row maxima (400), its exponentials (1400) and the products of their last half (256)
// follow one another, and the other tile's do not fill all of the gaps. An item adds
// about 3000 cycles for its outputs. Steps:
//   products issued by a converged warp, operands in uniform registers: a single
//   diverged lane took 105 cycles an instruction of 64     190 -> 172 us (11 prompts)
//   weights handed over by halves, loads in flight together     172 -> 165
//   outputs in 64-byte pieces by an exchange among four lanes   204 -> 193
//   further items by cancelling CTAs                            212 -> 204
//   (asked for at an item's start, not its end: 2048 tokens 43 -> 53, who is last
//   takes two)
//   registers split 216 to 72 between the softmax and the issuing warps, where one
//   size for all spills                                         223 -> 208
//   exponentials against the reference so far, made again where it moves: spills,
//   twice the time; a persistent grid with dealt items: 224 -> 244
//
// A key tile may hold tokens its rows do not attend: later ones of the prompt,
// the next prompt's. Their scores are replaced by -inf, so their weights are
// zero, but a zero weight times an infinite or NaN value is NaN: of a row whose
// sums are finite and whose output is not, the dims that this can have touched are
// computed again over what it attends only (careful_rows).
//
// A wait that runs out (1 s) ends its warp's walk, and the others' with it: they
// wait once more at most for what no longer comes, then for their own copies and
// products, and leave.
#include <type_traits>

#include "q4.cuh"
#include "qx_tc.cuh"

namespace qx {
namespace {

template <class M, typename T>
struct Packed {
  static constexpr int NT = 384;                    // warps 10 and 11 only give up registers
  // registers a thread of the softmax warps (a row's scores and weights without a
  // spill) and of the others, after the split
  static constexpr int REGS = 216, REGS_OTHER = 72;
  static constexpr int HALVES = M::D / 64;          // 64-dim column blocks of a row
  static constexpr int TOKENS = 128 / M::G;         // tokens of a query tile
  static constexpr int BLK = 128 * 128;             // [128 rows][128 B]
  static constexpr int TILE = HALVES * BLK;
  static constexpr int STAGES = M::D == 128 ? 5 : 8;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_RING = 2 * TILE;
  static constexpr int OFF_BAR = OFF_RING + STAGES * TILE;
  // ring full/empty, per tile: queries there, queries done with, scores there,
  // weights there (by halves), output done; answers there/read
  static constexpr int NBAR = 2 * STAGES + 12 + 4;
  static constexpr int OFF_ITEM = OFF_BAR + (8 * NBAR + 15) / 16 * 16;  // two answers of 16 bytes
  static constexpr int SMEM = OFF_ITEM + 32 + 16 + 1024;       // + TMEM slot, + slack to align the base
  static constexpr uint32_t COL_S = 0, COL_O = 256;            // tile u: scores at 128 u, output at 256 + D u
  static constexpr int FMT = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  static constexpr float TAU = 8.0f;
  // Every POLY-th pair of exponentials is made on the FMA pipe (0: none). With 64
  // dims the special-function unit has as many exponentials a product as with 128 but
  // half the time: none, every fourth, every third pair take 187, 180, 178 us for 3
  // Granite prompts of 8200 tokens, 450, 433, 434 for 10 of together 30000, 54.1, 52.8,
  // 52.6 for one of 4096 (every second: 60 there); with 128 dims 1578, 1586, 1591 us for
  // 16384 tokens and 162, 163, 165 for 11 ragged prompts.
  static constexpr int POLY = M::D == 64 ? 3 : 0;
  static constexpr float UNIT = M::SCALE * 1.4426950408889634f;  // base-2 logit of a score
  static_assert(SMEM <= 227 * 1024, "fits one SM");
  static_assert(packed_block(M::QWEN) == 2 * TOKENS, "two tiles a block");
};

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float2 x) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(x.x, x.y);
    return *reinterpret_cast<const uint32_t*>(&b);
  } else {
    const __half2 h = __floats2half2_rn(x.x, x.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// 2^x, x <= TAU, of a pair on the FMA pipe: x = n + f, n rounded by adding and
// taking off 1.5 * 2^23, 2^f by a polynomial of degree 3 (fitted for the smallest
// relative error on [-0.5, 0.5], 7.5e-5; a weight's rounding to fp16 is up to
// 4.9e-4), 2^n through the exponent field. x below -126, -inf among them, gives 0 (so does
// NaN, but a row with such a score has NaN for its reference):
// the value at -126 is taken off, which no larger result notices.
__device__ __forceinline__ float2 exp2_fma(float2 x) {
  constexpr float C0 = 0.9999281167984009f, C1 = 0.6932609677314758f, C2 = 0.24261054396629333f, C3 = 0.05517132207751274f;
  constexpr float ROUND = 12582912.0f;
  const float least = __int_as_float(__float_as_int(C0) - (126 << 23));
  x = make_float2(fmaxf(x.x, -126.0f), fmaxf(x.y, -126.0f));
  const float2 j = __fadd2_rn(x, make_float2(ROUND, ROUND));
  const float2 n = __fadd2_rn(j, make_float2(-ROUND, -ROUND));
  const float2 f = __ffma2_rn(n, make_float2(-1.0f, -1.0f), x);
  float2 y = __ffma2_rn(make_float2(C3, C3), f, make_float2(C2, C2));
  y = __ffma2_rn(y, f, make_float2(C1, C1));
  y = __ffma2_rn(y, f, make_float2(C0, C0));
  y = make_float2(__int_as_float(__float_as_int(y.x) + (__float_as_int(j.x) << 23)),
                  __int_as_float(__float_as_int(y.y) + (__float_as_int(j.y) << 23)));
  return __fadd2_rn(y, make_float2(-least, -least));
}

// Up to eight neighbouring output rows of a tile (those of `rows`, a bit each) again,
// by a whole warp: the dims in which a token that a row does not attend, but its key
// tiles hold (up to `end`), is not finite, over the tokens it does attend only,
// against the row's own reference m and sum, which lane `from` + a holds for row a.
// A dim ends as soon as it is not finite by what a row does attend, so that only the
// rows of one query tile before a dim's first such value walk all their tokens. The
// warps that wait for this one do so for 1 s at most: hence eight rows together, which
// share their loads, and a limit on a prompt's length (140001 tokens: 0.3 s). False
// when a row is not finite.
template <class M, typename T>
__device__ __noinline__ bool careful_rows(const PackedParams& p, int first, int token, int end, int h, unsigned rows,
                                          int from, float m, float sum) {
  constexpr int N = M::D / 32, TG = 8 / M::G, U = 32 / N;
  using P = Packed<M, T>;
  const int lane = threadIdx.x & 31, last = token + (31 - __clz(rows)) / M::G;
  auto value = [&](int t, int e) {
    return Elem<T>::to_f32(static_cast<const T*>(p.v)[t * p.v_stride + h * M::D + 32 * e + lane]);
  };
  float o[8][N];
  bool dirty[TG][N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
#pragma unroll
    for (int j = 0; j < TG; ++j) dirty[j][e] = false;
#pragma unroll
    for (int a = 0; a < 8; ++a) o[a][e] = 0.0f;
  }
  for (int t = token + 1; t < end; ++t)
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const bool bad = !isfinite(value(t, e));
#pragma unroll
      for (int j = 0; j < TG; ++j) dirty[j][e] |= bad && t > token + j;
    }
  for (int t0 = first; t0 <= last; t0 += 32) {
    bool open = false;
#pragma unroll
    for (int e = 0; e < N; ++e)
#pragma unroll
      for (int a = 0; a < 8; ++a) open |= dirty[a / M::G][e] && (rows >> a & 1u) && isfinite(o[a][e]);
    if (!__any_sync(0xffffffffu, open)) break;
    float weight[8];
#pragma unroll
    for (int a = 0; a < 8; ++a) weight[a] = 0.0f;
    if (t0 + lane <= last) {
      const T* k = static_cast<const T*>(p.k) + (t0 + lane) * p.k_stride + h * M::D;
#pragma unroll 4
      for (int d = 0; d < M::D; d += 8) {
        float y[8];
        Vec16<T>::load(k + d, y);
#pragma unroll
        for (int a = 0; a < 8; ++a) {
          if (TG > 1 && !(rows >> a & 1u)) continue;  // a token past the last
          float x[8];
          Vec16<T>::load(static_cast<const T*>(p.q) + (token + a / M::G) * p.q_stride + (h * M::G + a % M::G) * M::D + d, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) weight[a] = fmaf(x[e], y[e], weight[a]);
        }
      }
    }
#pragma unroll
    for (int a = 0; a < 8; ++a) {
      const float ref = __shfl_sync(0xffffffffu, m, from + a);
      weight[a] = t0 + lane <= token + a / M::G ? fast_exp2(fmaf(weight[a], P::UNIT, -ref)) : 0.0f;
    }
    for (int u0 = 0; u0 < 32; u0 += U) {  // 32 loads in flight
      float x[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < N; ++e) x[u][e] = t0 + u0 + u <= last ? value(t0 + u0 + u, e) : 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int a = 0; a < 8; ++a) {
          const float w = __shfl_sync(0xffffffffu, weight[a], u0 + u);
          if (TG > 1 && t0 + u0 + u > token + a / M::G) continue;  // a zero weight would not do
#pragma unroll
          for (int e = 0; e < N; ++e) o[a][e] = fmaf(w, x[u][e], o[a][e]);
        }
    }
  }
  bool good = true;
#pragma unroll
  for (int a = 0; a < 8; ++a) {
    const float all = __shfl_sync(0xffffffffu, sum, from + a);
    if (!(rows >> a & 1u)) continue;
    T* out = static_cast<T*>(p.out) + ((long long)(token + a / M::G) * M::HQ + h * M::G + a % M::G) * M::D;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if (dirty[a / M::G][e]) out[32 * e + lane] = Elem<T>::from_f32(o[a][e] / all);
      good &= isfinite(Elem<T>::to_f32(out[32 * e + lane]));
    }
  }
  return __all_sync(0xffffffffu, good);
}

// A work item of this CTA.
struct Item {
  int token, length;  // the prompt's first packed token, its tokens
  int head;           // kv head
  int q0;             // first token of the block, within the prompt
  int tiles[2];       // key tiles that each query tile attends (0: past the prompt's end)
};

template <class M, int TOKENS>
__device__ __forceinline__ void find_item(const PackedParams& p, int index, Item* out) {
  int lo = 0, hi = p.n_seq - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.seqs[mid].item <= index) lo = mid;
    else hi = mid - 1;
  }
  const PackedSeq seq = p.seqs[lo];
  const int rel = index - seq.item, blocks = (seq.length + 2 * TOKENS - 1) / (2 * TOKENS);
  out->token = seq.token;
  out->length = seq.length;
  out->head = rel % M::HKV;
  out->q0 = (blocks - 1 - rel / M::HKV) * 2 * TOKENS;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int begin = out->q0 + u * TOKENS, end = min(begin + TOKENS, seq.length);
    out->tiles[u] = begin < seq.length ? (end + kPackedKeys - 1) / kPackedKeys : 0;
  }
}

// A place in the ring of N tiles, and its barriers' parity there.
template <int N>
struct Place {
  int at = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void advance() {
    if (++at == N) {
      at = 0;
      parity ^= 1u;
    }
  }
};

// Ask for a CTA of this grid that is not launched yet; the answer, 16 bytes, lands
// in shared memory and completes them on the barrier. Not after an answer of none.
__device__ __forceinline__ void ask_for_cta(void* answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
               ::"r"(smem_addr(answer)), "r"(smem_addr(bar))
               : "memory");
}
// The block index of an answer, -1 for none.
__device__ __forceinline__ int answered_cta(const void* answer) {
  int got, x;
  asm volatile(
      "{\n"
      ".reg .b128 r;\n"
      ".reg .pred p;\n"
      "ld.shared.b128 r, [%2];\n"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n"
      "selp.s32 %0, 1, 0, p;\n"
      "mov.s32 %1, 0;\n"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n"
      "}"
      : "=r"(got), "=r"(x)
      : "r"(smem_addr(answer))
      : "memory");
  return got ? x : -1;
}

template <class M, typename T>
__global__ void __launch_bounds__(Packed<M, T>::NT, 1) qx_packed_kernel(const __grid_constant__ PackedParams p) {
  using C = Packed<M, T>;
  constexpr int NS = C::STAGES;
  extern __shared__ __align__(1024) unsigned char sm_raw[];
  unsigned char* sm = sm_raw + ((1024u - (smem_addr(sm_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + C::OFF_BAR);  // [NS] a key or value tile landed
  uint64_t* empty = full + NS;     // [NS] its products completed
  uint64_t* qfull = empty + NS;    // [tile] queries landed
  uint64_t* qempty = qfull + 2;    // [tile] the item's last scores completed
  uint64_t* sfull = qempty + 2;    // [tile] scores in TMEM (and everything issued before them done)
  uint64_t* pfull = sfull + 2;     // [tile][half] weights of 64 keys in TMEM
  uint64_t* odone = pfull + 4;     // [tile] output in TMEM
  uint64_t* ifull = odone + 2;     // [2] the answer to a request for an item landed
  uint64_t* iempty = ifull + 2;    // [2] all warps have read it
  unsigned char* answers = sm + C::OFF_ITEM;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(answers + 32);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int u = 0; u < 2; ++u) {
      mbar_init(&qfull[u], 1);
      mbar_init(&qempty[u], 1);
      mbar_init(&sfull[u], 1);
      mbar_init(&pfull[2 * u], 4);
      mbar_init(&pfull[2 * u + 1], 4);
      mbar_init(&odone[u], 1);
      mbar_init(&ifull[u], 1);
      mbar_init(&iempty[u], 10);
    }
    fence_barrier_init();
  }
  if (warp == 8) {
    tmem_alloc(tslot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = *tslot;
  pdl_wait();
  pdl_launch_dependents();
  bool ok = true;
  Item item;
  // item k + 1 is the answer of slot k % 2: its block index, -1 past the last, or
  // once a wait of this warp has run out
  auto next_item = [&](int k) {
    if (__all_sync(0xffffffffu, ok)) ok &= mbar_wait_bounded(&ifull[k & 1], (uint32_t)(k >> 1) & 1u, p.err);
    const int index = __all_sync(0xffffffffu, ok) ? answered_cta(answers + 16 * (k & 1)) : -1;
    fence_proxy_async_shared();  // the read above comes before the next answer
    __syncwarp();
    if (lane == 0) mbar_arrive(&iempty[k & 1]);
    return index;
  };

  if (warp >= 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_OTHER));
  if (warp == 9) {
    // ---- TMA producer: of an item, keys of tile i are load 2 i, its values 2 i + 1
    if (lane == 0) {
      prefetch_tmap(&p.tmq);
      prefetch_tmap(&p.tmk);
      prefetch_tmap(&p.tmv);
    }
    Place<NS> place;
    int loads = 0, used[2] = {0, 0};
    for (int k = 0, index = blockIdx.x; index >= 0; index = next_item(k++)) {
      find_item<M, C::TOKENS>(p, index, &item);
      if (lane == 0) {
        const int n = 2 * max(item.tiles[0], item.tiles[1]);
        auto queries = [&](int u) {
          if (!item.tiles[u]) return;
          if (used[u]) ok &= mbar_wait_bounded(&qempty[u], (uint32_t)(used[u] - 1) & 1u, p.err);
          ++used[u];
          mbar_arrive_expect_tx(&qfull[u], C::TILE);
#pragma unroll
          for (int b = 0; b < C::HALVES; ++b)
            tma_load_3d(sm + C::OFF_Q + u * C::TILE + b * C::BLK, &p.tmq, 64 * b, item.head * M::G,
                        item.token + item.q0 + u * C::TOKENS, &qfull[u]);
        };
        queries(0);
        for (int i = 0; i < n && ok; ++i, ++loads, place.advance()) {
          const int s = place.at;
          if (loads >= NS) ok &= mbar_wait_bounded(&empty[s], place.parity ^ 1u, p.err);
          mbar_arrive_expect_tx(&full[s], C::TILE);
#pragma unroll
          for (int b = 0; b < C::HALVES; ++b)
            tma_load_3d(sm + C::OFF_RING + s * C::TILE + b * C::BLK, i & 1 ? &p.tmv : &p.tmk, 64 * b, item.head,
                        item.token + (i >> 1) * kPackedKeys, &full[s]);
          if (i == 0) queries(1);
        }
        // asked for now, not before: who is done first takes the next item
        if (k >= 2) ok &= mbar_wait_bounded(&iempty[k & 1], (uint32_t)((k >> 1) - 1) & 1u, p.err);
        if (ok) {
          mbar_arrive_expect_tx(&ifull[k & 1], 16);
          ask_for_cta(answers + 16 * (k & 1), &ifull[k & 1]);
        }
      }
      __syncwarp();
    }
    // no copy may still be landing when the CTA exits
    if (lane == 0) {
      for (int i = max(0, loads - NS); i < loads; ++i)
        ok &= mbar_wait_bounded(&full[i % NS], (uint32_t)(i / NS) & 1u, p.err);
      for (int u = 0; u < 2; ++u)
        if (used[u]) ok &= mbar_wait_bounded(&qfull[u], (uint32_t)(used[u] - 1) & 1u, p.err);
    }
  } else if (warp == 8) {
    // ---- MMA issuer: the whole warp walks, one lane issues -------------------------
    constexpr uint32_t IDESC_S = umma_idesc_16bit(128, kPackedKeys, C::FMT, false, false);
    constexpr uint32_t IDESC_PV = umma_idesc_16bit(128, M::D, C::FMT, false, true);
    const uint32_t one = one_lane(), tm = __reduce_max_sync(0xffffffffu, tbase);
    // a descriptor counts addresses in units of 16 bytes in its lowest bits
    const uint64_t dq = umma_desc_sw128(smem_addr(sm + C::OFF_Q), 16, 1024);
    const uint64_t dk = umma_desc_sw128(smem_addr(sm + C::OFF_RING), 16, 1024);
    const uint64_t dv = umma_desc_sw128(smem_addr(sm + C::OFF_RING), C::BLK, 1024);
    Place<NS> keys, values;                                // of the step's tiles, of the next step's keys
    int items[2] = {0, 0}, weights[2] = {0, 0};            // per tile: items, weight tiles taken
    for (int k = 0, index = blockIdx.x; index >= 0; index = __reduce_max_sync(0xffffffffu, next_item(k++))) {
      find_item<M, C::TOKENS>(p, index, &item);
      const int n = max(item.tiles[0], item.tiles[1]);
      auto landed = [&](const Place<NS>& s) {
        ok &= mbar_wait_bounded(&full[s.at], s.parity, p.err);
        __syncwarp();
        tc_fence_after();
      };
      auto commit = [&](uint64_t* bar) {
        if (one) tc_commit(bar);
        __syncwarp();
      };
      auto scores = [&](int u, int i) {  // S of query tile u and key tile i
#pragma unroll
        for (int kk = 0; kk < M::D / 16; ++kk) {
          const uint32_t at = ((kk >> 2) * C::BLK + (kk & 3) * 32) >> 4;
          tc_mma_one(one, tm + C::COL_S + 128 * u, dq + (uint32_t)(u * (C::TILE >> 4)) + at,
                     dk + (uint32_t)(keys.at * (C::TILE >> 4)) + at, IDESC_S, kk > 0);
        }
        commit(&sfull[u]);
        if (i + 1 == item.tiles[u]) commit(&qempty[u]);
      };
      auto output = [&](int u, int i) {  // O += P V of query tile u and key tile i
#pragma unroll
        for (int kk = 0; kk < kPackedKeys / 16; ++kk) {
          if (kk % 4 == 0) {
            ok &= mbar_wait_bounded(&pfull[2 * u + kk / 4], (uint32_t)weights[u] & 1u, p.err);
            __syncwarp();
            tc_fence_after();
          }
          tc_mma_ts_one(one, tm + C::COL_O + M::D * u, tm + C::COL_S + 128 * u + 8 * kk,
                        dv + (uint32_t)(values.at * (C::TILE >> 4)) + (uint32_t)(kk * (2048 >> 4)), IDESC_PV,
                        (i > 0 ? 1u : 0u) | (kk > 0 ? 1u : 0u));
        }
        ++weights[u];
      };
      landed(keys);
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (item.tiles[u]) {
          ok &= mbar_wait_bounded(&qfull[u], (uint32_t)items[u] & 1u, p.err);
          ++items[u];
          __syncwarp();
          tc_fence_after();
          scores(u, 0);
        }
      commit(&empty[keys.at]);
      keys.advance();
      for (int i = 0; i < n; ++i) {
        values = keys;  // this step's values, then the next step's keys
        landed(values);
        keys.advance();
        if (i + 1 < n) landed(keys);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (i < item.tiles[u]) output(u, i);
          if (i + 1 < item.tiles[u]) scores(u, i + 1);
          else if (i + 1 == item.tiles[u]) commit(&odone[u]);
        }
        commit(&empty[values.at]);
        if (i + 1 < n) {
          commit(&empty[keys.at]);
          keys.advance();
        }
        if (!__all_sync(0xffffffffu, ok)) break;
      }
    }
    // TMEM is released only after every product completed
    for (int u = 0; u < 2; ++u)
      if (items[u]) ok &= mbar_wait_bounded(&odone[u], (uint32_t)(items[u] - 1) & 1u, p.err);
  } else if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS));
    // ---- softmax of tile u: thread owns row r (token r / G of the tile, head r % G)
    const int u = warp >> 2, r = tid & 127;
    const uint32_t trow = tbase + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t ts = trow + C::COL_S + 128 * u, to = trow + C::COL_O + M::D * u;
    int seen = 0, written = 0;  // score tiles, items of this query tile
    for (int k = 0, index = blockIdx.x; index >= 0; index = next_item(k++)) {
      find_item<M, C::TOKENS>(p, index, &item);
      const int tiles = u ? item.tiles[1] : item.tiles[0];
      if (!tiles) continue;
      const int pos = item.q0 + u * C::TOKENS + r / M::G;  // within the prompt
      float m = -INFINITY;
      float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
      for (int i = 0; i < tiles; ++i, ++seen) {
        ok &= mbar_wait_bounded(&sfull[u], (uint32_t)seen & 1u, p.err);
        __syncwarp();
        tc_fence_after();
        float s[128];
#pragma unroll
        for (int c = 0; c < 128; c += 32) tmem_ld32(ts + c, s + c);
        tmem_wait_ld<128>(s);
        if (i == tiles - 1 || (i + 1) * kPackedKeys > item.q0 + u * C::TOKENS) {  // some key is later than some row
          const int limit = pos - i * kPackedKeys;
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (c > limit) s[c] = -INFINITY;
        }
        float m4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int c = 4; c < 124; c += 8) {
#pragma unroll
          for (int e = 0; e < 4; ++e) m4[e] = fmax3f_nan(m4[e], s[c + 2 * e], s[c + 2 * e + 1]);
        }
        m4[0] = fmax3f_nan(m4[0], s[124], s[125]);
        m4[1] = fmax3f_nan(m4[1], s[126], s[127]);
        const float top = fmax3f_nan(fmax3f_nan(m4[0], m4[1], m4[2]), m4[3], m4[3]) * C::UNIT;
        // true on the first tile (m = -inf), and for a score that is NaN: it becomes the
        // reference and with it the row (exp2_fma would make it a weight of zero)
        const bool raise = !(top <= m + C::TAU);
        if (__any_sync(0xffffffffu, raise)) {
          const float keep = raise ? fast_exp2(m - top) : 1.0f;
          if (i > 0) {
#pragma unroll
            for (int c = 0; c < M::D; c += 16) {
              float o[16];
              uint32_t b[16];
              tmem_ld16_sync(to + c, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) b[e] = __float_as_uint(o[e] * keep);
              tmem_st16u(to + c, b);
            }
          }
          sum[0] = __fmul2_rn(sum[0], make_float2(keep, keep));
          sum[1] = __fmul2_rn(sum[1], make_float2(keep, keep));
          if (raise) m = top;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t w[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int c = 32 * q + 2 * j;
            const float2 x = __ffma2_rn(make_float2(s[c], s[c + 1]), make_float2(C::UNIT, C::UNIT), make_float2(-m, -m));
            float2 e;
            if (C::POLY && j % (C::POLY ? C::POLY : 1) == C::POLY - 1) e = exp2_fma(x);
            else e = make_float2(fast_exp2(x.x), fast_exp2(x.y));
            w[j] = pack_pair<T>(e);
            sum[j & 1] = __fadd2_rn(sum[j & 1], e);
          }
          tmem_st16u(ts + 16 * q, w);
          if (q & 1) {  // the products of the first 64 keys start while the others' weights are made
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&pfull[2 * u + q / 2]);
          }
        }
        if (!__all_sync(0xffffffffu, ok)) break;  // here, while the products run
      }
      // ---- output -------------------------------------------------------------------
      ok &= mbar_wait_bounded(&odone[u], (uint32_t)written & 1u, p.err);
      ++written;
      __syncwarp();
      tc_fence_after();
      const float all = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y), inv = 1.0f / all;
      const bool real = pos < item.length;
      const int token = item.token + pos;
      float2 off = make_float2(0.0f, 0.0f);  // NaN once an output is not finite
      // four lanes exchange their rows' 16-byte pieces, so that a store writes 64
      // bytes of 8 rows and not 16 of 32: lane t of the four ends with piece t of each
      const int r0 = r & ~3, pos0 = item.q0 + u * C::TOKENS + r0 / M::G;
      T* out = static_cast<T*>(p.out) + ((long long)(item.token + pos0) * M::HQ + item.head * M::G + r0 % M::G) * M::D +
               8 * (lane & 3);
      float o[M::D];
#pragma unroll
      for (int c = 0; c < M::D; c += 32) tmem_ld32(to + c, o + c);
      tmem_wait_ld<M::D>(o);
#pragma unroll
      for (int c = 0; c < M::D; c += 32) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float2 y = __fmul2_rn(make_float2(o[c + 2 * e], o[c + 2 * e + 1]), make_float2(inv, inv));
          off = __ffma2_rn(y, make_float2(0.0f, 0.0f), off);
          w[e] = pack_pair<T>(y);
        }
#pragma unroll
        for (int bit = 1; bit < 4; bit <<= 1) {
          const bool upper = lane & bit;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            if ((e >> 2) & bit) continue;
            const int f = e + 4 * bit;
            const uint32_t got = __shfl_xor_sync(0xffffffffu, upper ? w[e] : w[f], bit);
            if (upper) w[e] = got;
            else w[f] = got;
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (pos0 + j / M::G < item.length)
            *reinterpret_cast<uint4*>(out + (j / M::G * M::HQ + j % M::G) * M::D + c) =
                make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
      }
      const bool good = off.x + off.y == 0.0f;
      __syncwarp();  // a row that is recomputed is written after this
      tc_fence_before();  // O was read: the next item's first product may write it once its weights are there
      unsigned redo = __ballot_sync(0xffffffffu, real && ok && !good && isfinite(m) && isfinite(all));
      bool bad = real && !good && !(isfinite(m) && isfinite(all));
      while (redo) {  // eight neighbouring lanes' rows together
        const int from = (__ffs(redo) - 1) & ~7;
        const unsigned rows = redo >> from & 255u;
        redo &= ~(255u << from);
        bad |= !careful_rows<M, T>(p, item.token, __shfl_sync(0xffffffffu, token, from),
                                   min(item.token + tiles * kPackedKeys, p.tokens), item.head, rows, from, m, all);
      }
      if (bad && ok) flag_error(p.err, QX_ERR_BIT_NONFINITE);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tbase, 512);
  }
}

template <class M, typename T>
cudaError_t setup() {
  using C = Packed<M, T>;
  cudaError_t e = cudaFuncSetAttribute(qx_packed_kernel<M, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return e;
  // the kernel's split would wait for registers that a launch with fewer does not have
  cudaFuncAttributes fa;
  e = cudaFuncGetAttributes(&fa, qx_packed_kernel<M, T>);
  if (e != cudaSuccess) return e;
  return fa.numRegs * C::NT < C::REGS * 256 + C::REGS_OTHER * 128 ? cudaErrorLaunchOutOfResources : cudaSuccess;
}

template <class M, typename T>
cudaError_t packed(const PackedParams& p, cudaStream_t stream) {
  using C = Packed<M, T>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.items);
  cfg.blockDim = dim3(C::NT);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, qx_packed_kernel<M, T>, p);
}

}  // namespace

cudaError_t setup_packed() {
  for (cudaError_t e : {setup<Qwen3Heads, __nv_bfloat16>(), setup<Qwen3Heads, __half>(),
                        setup<GraniteHeads, __nv_bfloat16>(), setup<GraniteHeads, __half>()})
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}

cudaError_t launch_packed(bool qwen, const PackedParams& p, cudaStream_t stream) {
  if (p.dtype == 1)
    return qwen ? packed<Qwen3Heads, __nv_bfloat16>(p, stream) : packed<GraniteHeads, __nv_bfloat16>(p, stream);
  return qwen ? packed<Qwen3Heads, __half>(p, stream) : packed<GraniteHeads, __half>(p, stream);
}

}  // namespace qx
