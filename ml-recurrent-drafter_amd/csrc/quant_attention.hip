// Masked attention over a KV cache held in 4 or 8 bits (gfx950; kv_quant.h has the row format).
//
//   O[b,q,h,:] = softmax_k( Q[b,h,q,:] . K[b,hk,k,:] * scale  masked by bits[b,q,k] ) V[b,hk,k,:]
//
// The mask bits and the row shifts are those of rd_verify_attention; a row that attends to nothing is
// written as zeros.  Two kernels behind one entry point:
//   attn_quant_kernel    bf16 and fp16, head_dim 64 and 128, on v_mfma_f32_16x16x32
//   attn_quant_generic_kernel  every other type and head size the cache has
//
// attn_quant_kernel.  The query heads of a kv head are folded into the rows (row = query * group + head in
// group), so that K and V are read once per kv head.  A wave takes 16 * RB rows and goes over units of 32 keys
// with a running maximum, row sums and accumulators in registers:
//   S^T = K Q^T  A operand: lane (key l % 16, chunk l / 16) needs 8 consecutive k-slots per step.  The
//                order of the dims in a dot product is free, so chunk c of the record is dims
//                [c D/4, (c+1) D/4): D/4 contiguous codes per lane, one block of 8 per step.
//   O^T = V^T P^T  A operand: lane (column l % 16, key group l / 16) needs 8 keys of one dim.  Column n
//                is the D/16 dims from n D/16 on, tile j of the output their j-th; the 8 keys are those
//                whose scores the lane already holds (16 t + 4 (l / 16) + i), so P^T goes from the
//                accumulators of the first product into the B operand of the second as it is.
//                Codes of two keys become two dims times two keys: two conversions (code pair x scale
//                to a 16-bit pair, one instruction, exact) and two byte permutes.
// P is rounded to the 16-bit type there (half a step of it, as every 16-bit product of the model rounds: 2^-9 of a
// weight in bf16; in fp16 2^-12, and for weights below 2^-21 of the running maximum's 2^-32 of that one);
// scores, maximum, sums and accumulators are fp32.  The row sums come out of the matrix pipeline too, as
// the product of P with ones: the sum of the rounded weights, the ones that V is multiplied with.
// A query row lives in one column of the accumulators (l % 16), so rescaling is a lane scalar; the running
// maximum is lazy: raised only when some score exceeds it by 2^8 in the exponential, where fp32 has room
// for 2^120 such weights (values times weights are summed before they are divided: 2^8 |v| summed over a row's
// keys has to be a finite number of fp32, which only values beyond 2^97 or so can miss).
// Weights depend on differences of scores alone: where a row's maximum is so large that its rounding in log2 units
// matters (2^22), the keys are gone over once more with the scores subtracted before they are scaled.
//
// Records travel memory -> registers (whole contiguous units, 16 bytes per lane) -> LDS as they lie in
// memory, and are picked apart from there without a bank conflict (rows of 48, 80 and 144 bytes spread 16
// lanes over all banks): picked apart from memory, each unit took 22 scattered loads and the return path of
// the vector memory was busy for 80 to 95 % of the time.  Keys outside the piece and outside the tile's
// attended span read as zeros through the range check of a buffer descriptor, without touching memory.  Mask
// words travel with their unit, and only where the span table does not say that every row attends to it.
//
// Four layouts (shape_of chooses, with both sides measured):
//   rows <= 16      RB 1, eight waves behind each other take the units in turn and are merged through LDS.
//                   Bound by memory: batch 8, 32 heads, one token, 2548 keys in 4 bits: 16 us, 4.4 TB/s of records
//                   (a copy of 1 GiB reaches 5.15); one sequence of 65 537 keys in 8 bits, 8 kv heads: 29 to 32 us
//                   and 4 for the merge of its pieces, 4.5 TB/s.
//   <= 32 a tile    RB 2, two or four waves behind each other.  Bound by the vector ALU, which converts every unit
//                   for 32 rows (about 130 of 230 instructions), and by the matrix pipeline, which runs beside it
//                   for a small part of the time only: batch 8, 32 heads, a tree of 115 over 735 keys: 23 us, 390
//                   TFLOP/s; 16 x 162 rows of 40 heads over 1962 keys in 8 bits: 138 to 152 us.
//   <= 256 a tile   RB 2, eight waves side by side: a unit is converted once for all of them, its operands lie in LDS
//                   in the lanes' order.  8 x 32 heads, 768 rows, 8192 keys: 898 us, 919 TFLOP/s in 4 bits, 854 us in
//                   8 bits, where a large bf16 matrix product of the library reaches 1200; of the rest, conversion
//                   costs about 100 ns of the 585 per unit and SIMD and the operands' way through LDS 60.
// Tried and slower: 48 and 64 rows a wave (registers spill, or one wave on a SIMD: tree of 115 over 735 keys 38 us), two
// and four waves side by side with two buffers (40 and 33 us), the next unit's first product put between the softmax's
// instructions by hand (363 us where priorities gave 347), K's operands of the coming unit read as late as needed.
//
// V and masked keys: a probability of zero does not silence a NaN in V (0 * NaN).  Where the output of a
// workgroup holds a NaN, its waves go over their keys once more: blocks of V that read back as NaN are then
// taken out of the product, and the rows that attend to such a key get their NaN from a second product, of
// the mask with the marks of those blocks.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <type_traits>

#include "attn_plan.h"
#include "kv_quant.h"
#include "rd_common.h"

namespace {

using namespace rd::kvq;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kUnit = 32;        // keys a wave takes at a time
constexpr int kSpanQueries = 16; // queries that share an entry of the span table
constexpr float kFar = 4194304.f;  // 2^22: fp32 has a quarter of a unit there
constexpr int kSpanInts = 4;     // {first key, one past the last, full_lo, full_hi} of those queries

struct QuantArgs {
  const void* q; int64_t q_sb, q_sh, q_ss;       // elements
  const char* k; const char* v; int64_t c_sb, c_sh;  // records, byte strides {batch, head}; rows follow each other
  void* out; int64_t o_sb, o_sh, o_ss;
  const uint64_t* bits; const int32_t* plan; const int32_t* spans; const int32_t* row_start;
  float* part_o;   // [slot][rows][D], slot = (b * Hkv + hk) * max_pieces + piece
  float* part_ml;  // [slot][rows][2]
  int64_t max_len;
  int B, H, Hkv, group, n_q, kv_len, words, D, bits_per_code;
  int span_blocks, max_pieces, piece;
  int sorted;      // workgroups take their tiles by rank (sorted_pair)
  float scale;     // softmax scale; times log2 e for the MFMA kernel
  float inv_scale; // its reciprocal
  float rise;      // how far a score may lie above the running maximum: 8 in log2 units
};

__device__ inline float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

template <typename T> struct Ops;
template <> struct Ops<__hip_bfloat16> {
  using V8 = bf16x8;
  static constexpr bool kF16 = false;
  static constexpr uint32_t kOne = 0x3f80u;
  static constexpr float kLift = 0.f;              // (see weights)
  static __device__ uint32_t fp4(uint32_t w, float s, std::integral_constant<int, 0>) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0)); }
  static __device__ uint32_t fp4(uint32_t w, float s, std::integral_constant<int, 1>) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1)); }
  static __device__ uint32_t fp4(uint32_t w, float s, std::integral_constant<int, 2>) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2)); }
  static __device__ uint32_t fp4(uint32_t w, float s, std::integral_constant<int, 3>) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3)); }
  static __device__ uint32_t fp8_lo(uint32_t w, float s) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false)); }
  static __device__ uint32_t fp8_hi(uint32_t w, float s) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true)); }
  static __device__ uint32_t pack(float a, float b) {
    const bf16x2 p = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
    return __builtin_bit_cast(uint32_t, p);
  }
  static __device__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <> struct Ops<__half> {
  using V8 = f16x8;
  static constexpr bool kF16 = true;
  static constexpr uint32_t kOne = 0x3c00u;
  static constexpr float kLift = 7.f;
  static __device__ uint32_t fp4(uint32_t w, float s, std::integral_constant<int, 0>) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 0)); }
  static __device__ uint32_t fp4(uint32_t w, float s, std::integral_constant<int, 1>) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 1)); }
  static __device__ uint32_t fp4(uint32_t w, float s, std::integral_constant<int, 2>) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 2)); }
  static __device__ uint32_t fp4(uint32_t w, float s, std::integral_constant<int, 3>) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 3)); }
  static __device__ uint32_t fp8_lo(uint32_t w, float s) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, false)); }
  static __device__ uint32_t fp8_hi(uint32_t w, float s) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, true)); }
  static __device__ uint32_t pack(float a, float b) {
    const f16x2 p = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    return __builtin_bit_cast(uint32_t, p);
  }
  static __device__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

// W consecutive 16-bit pairs from the codes of 2 W values: `code` are the dwords that hold them from
// pair 0 on
template <typename T, int BITS, int W>
__device__ inline void convert(const uint32_t* code, float s, uint32_t (&out)[W]) {
  if constexpr (BITS == 4) {
    out[0] = Ops<T>::fp4(code[0], s, std::integral_constant<int, 0>{});
    out[1] = Ops<T>::fp4(code[0], s, std::integral_constant<int, 1>{});
    if constexpr (W == 4) {
      out[2] = Ops<T>::fp4(code[0], s, std::integral_constant<int, 2>{});
      out[3] = Ops<T>::fp4(code[0], s, std::integral_constant<int, 3>{});
    }
  } else {
    out[0] = Ops<T>::fp8_lo(code[0], s);
    out[1] = Ops<T>::fp8_hi(code[0], s);
    if constexpr (W == 4) {
      out[2] = Ops<T>::fp8_lo(code[1], s);
      out[3] = Ops<T>::fp8_hi(code[1], s);
    }
  }
}

// Which rows a workgroup's tile holds and which keys they attend to; the same arithmetic in the
// attention kernel and in the merge of its pieces.
struct Tile {
  int rows;         // rows of the batch row (queries that exist * group)
  int64_t q_off, o_off;
  int lo, hi;       // the tile's attended keys lie in [lo, hi)
  int begin;        // lo rounded down to a unit: pieces are counted from here
  int n_pieces;     // at least 1: piece 0 of a tile that attends to nothing writes its zeros
  int full_lo, full_hi;  // every row attends to every key of [full_lo, full_hi): whole units, maybe none
};
__device__ inline void tile_rows(const QuantArgs& a, int b, Tile& t) {
  int n = a.n_q;
  t.q_off = (int64_t)b * a.q_sb;
  t.o_off = (int64_t)b * a.o_sb;
  if (a.row_start != nullptr) {
    const int r0 = a.row_start[b];
    n = a.row_start[b + 1] - r0;
    n = n < a.n_q ? n : a.n_q;
    t.q_off = (int64_t)r0 * a.q_ss;
    t.o_off = (int64_t)r0 * a.o_ss;
  }
  t.rows = n * a.group;
}
// the keys of the rows from row0 on (kLanes: the span blocks are read by the lanes of a wave, not in turn)
template <bool kLanes = false>
__device__ inline void tile_keys(const QuantArgs& a, int b, int row0, int rows_per_tile, Tile& t) {
  t.lo = a.kv_len; t.hi = 0;
  t.full_lo = 0; t.full_hi = a.kv_len;
  if (row0 < t.rows) {
    const int end = row0 + rows_per_tile < t.rows ? row0 + rows_per_tile : t.rows;
    const int s0 = row0 / a.group / kSpanQueries, s1 = (end - 1) / a.group / kSpanQueries;
    const int32_t* sp = a.spans + kSpanInts * ((int64_t)b * a.span_blocks + s0);
    if constexpr (kLanes) {
      const int lane = threadIdx.x & 63;
      if (lane <= s1 - s0) {
        const int4 x = reinterpret_cast<const int4*>(sp)[lane];
        t.lo = x.x; t.hi = x.y; t.full_lo = x.z; t.full_hi = x.w;
      }
#pragma unroll
      for (int x = 1; x < 64; x *= 2) {
        t.lo = min(t.lo, __shfl_xor(t.lo, x));
        t.hi = max(t.hi, __shfl_xor(t.hi, x));
        t.full_lo = max(t.full_lo, __shfl_xor(t.full_lo, x));
        t.full_hi = min(t.full_hi, __shfl_xor(t.full_hi, x));
      }
      t.lo = __builtin_amdgcn_readfirstlane(t.lo);
      t.hi = __builtin_amdgcn_readfirstlane(t.hi);
      t.full_lo = __builtin_amdgcn_readfirstlane(t.full_lo);
      t.full_hi = __builtin_amdgcn_readfirstlane(t.full_hi);
    } else {
      for (int s = s0; s <= s1; ++s, sp += kSpanInts) {
        t.lo = sp[0] < t.lo ? sp[0] : t.lo;
        t.hi = sp[1] > t.hi ? sp[1] : t.hi;
        t.full_lo = sp[2] > t.full_lo ? sp[2] : t.full_lo;
        t.full_hi = sp[3] < t.full_hi ? sp[3] : t.full_hi;
      }
    }
  }
  t.begin = t.lo / kUnit * kUnit;
  t.n_pieces = t.hi > t.lo ? (t.hi - t.begin + a.piece - 1) / a.piece : 1;
}
// The (batch row, tile) pair of a workgroup's place in the launch, the pairs with the most keys first: every thread
// weighs one pair, and the one whose rank is the place is taken.  `weights` and `pick` are LDS.
constexpr int kMaxSorted = 512;                     // pairs, one per thread of the widest workgroup
__device__ inline int sorted_pair(const QuantArgs& a, int pairs, int tiles, int rows_per_tile, int place, uint32_t* weights, int* pick) {
  const int tid = threadIdx.x;
  uint32_t mine = 0;
  if (tid < pairs) {
    Tile t;
    const int b = tid / tiles, row0 = tid % tiles * rows_per_tile;
    tile_rows(a, b, t);
    int lo = a.kv_len, hi = 0;
    if (row0 < t.rows) {
      const int end = row0 + rows_per_tile < t.rows ? row0 + rows_per_tile : t.rows;
      const int s1 = (end - 1) / a.group / kSpanQueries;
      const int4* const sp = reinterpret_cast<const int4*>(a.spans) + (int64_t)b * a.span_blocks;
      for (int s0 = row0 / a.group / kSpanQueries; s0 <= s1; s0 += 8) {
        int4 x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = sp[min(s0 + i, s1)];
#pragma unroll
        for (int i = 0; i < 8; ++i) { lo = min(lo, x[i].x); hi = max(hi, x[i].y); }
      }
    }
    // (no two are equal: the thread's number is in the low bits, the later tile first)
    mine = (uint32_t)((hi > lo ? (hi - lo + kUnit - 1) / kUnit : 0) * kMaxSorted + tid);
  }
  weights[tid] = mine;
  __syncthreads();
  if (tid < pairs) {
    int rank = 0;
    for (int i = 0; i < pairs; i += 4) {            // (behind the last pair: zeros)
      const u32x4 w = *reinterpret_cast<const u32x4*>(weights + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) rank += w[e] > mine;
    }
    if (rank == place) *pick = tid;
  }
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(*pick);
}
__device__ inline Tile tile_of(const QuantArgs& a, int b, int row0, int rows_per_tile) {
  Tile t;
  tile_rows(a, b, t);
  tile_keys(a, b, row0, rows_per_tile, t);
  return t;
}

// max(a, b) as one instruction, with `inf` a register the compiler knows nothing about (fmaxf first quiets
// each operand that came out of the matrix pipeline, and so does a median with a known infinity); a NaN may
// lose, which is fine for a running maximum: its row ends as NaN whatever the maximum
__device__ inline float larger(float a, float b, float inf) { return __builtin_amdgcn_fmed3f(a, b, inf); }

// the lanes l, l ^ 16, l ^ 32, l ^ 48 share a query row
__device__ inline float row_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}

// ---------------------------------------------------------------------------------------------
// MFMA kernel
// ---------------------------------------------------------------------------------------------
template <typename T, int BITS, int D, int RB, int R, int K>
// (Three waves on a SIMD where head_dim is 64 and R is 1, for which the second sweep keeps 20 to 56 bytes in scratch: batch
// 16, 32 / 8 heads, 46 rows, 1257 keys 24.2 -> 20.3 us, 40 heads, 162 rows, 1962 keys in 8 bits 99 -> 88 us.  At 128 the
// third wave would put most of the accumulators there.)
__global__ __launch_bounds__(R * K * 64, D == 64 && R == 1 ? 3 : 2) void attn_quant_kernel(QuantArgs a) {
  static_assert(R == 1 || K == 1, "waves side by side or behind each other");
  using O = Ops<T>;
  constexpr int kRec = record_bytes(BITS, D), kCodes = code_bytes(BITS, D);
  constexpr int kSteps = D / 32;                    // blocks of 8 dims in a K chunk
  constexpr int kCols = D / 16;                     // dims of a V column = tiles of the output
  constexpr int kColBytes = kCols * BITS / 8;
  constexpr int kWaves = R * K;
  constexpr int kRows = 16 * RB * R;
  constexpr int kPitch = D + 4;                     // floats of a merged row in LDS
  constexpr int kKw = D * BITS / 128;               // dwords of a lane's K chunk (D/4 codes)
  constexpr int kVw = kColBytes > 4 ? 2 : 1;        // dwords of a lane's V column (D/16 codes)
  constexpr int kUnitBytes = kUnit * kRec;          // the records of a unit follow each other
  constexpr int kLoads = (kUnitBytes + 1023) / 1024;  // 16 bytes per lane each
  constexpr int kTail = kUnitBytes / 16 - 64 * (kLoads - 1);  // lanes of the last one that read
  constexpr int kRawBytes = kLoads * 1024;
  // R > 1: two waves bring a unit, one its K and one its V, and what all of them read of it are its operands,
  // converted once: 2 kSteps of K, kCols of V.  Two buffers of a round's units each.
  constexpr bool kShared = R > 1;
  constexpr int kRoundUnits = kShared ? R / 2 : K;  // units of a round
  constexpr int kVAt = kShared ? 2 * kSteps * 1024 : kRawBytes;  // where a slot's V begins, records or operands
  static_assert(kVAt >= kRawBytes && (!kShared || kCols * 1024 >= kRawBytes), "records fit the place of their operands");
  constexpr int kMaskRows = kShared ? kRows / 2 : kRows;  // rows of the tile whose mask words a wave brings
  constexpr int kMaskWords = (kMaskRows + 63) / 64;
  constexpr int kMaskAt = kShared ? kVAt + kCols * 1024 : 2 * kRawBytes;
  constexpr int kSlotBytes = kMaskAt + 4 * kRows;
  // the slots (records of K, then of V, or operands), later the rows that waves behind each other merge
  constexpr int kSlots = kShared ? 2 * kRoundUnits : K;
  constexpr int kMergeBytes = K > 1 ? kWaves * 16 * RB * kPitch * 4 : 0;
  constexpr int kLdsBytes = kSlots * kSlotBytes > kMergeBytes ? kSlots * kSlotBytes : kMergeBytes;
  __shared__ __attribute__((aligned(16))) char s_mem[kLdsBytes];
  __shared__ float s_ml[kWaves * 16 * RB * 2];
  float* const s_o = reinterpret_cast<float*>(s_mem);

  // (a causal prompt's last rows have the most keys: first)
  const int tiles = gridDim.x / a.Hkv, hk = blockIdx.x % a.Hkv;
  int tile = tiles - 1 - blockIdx.x / a.Hkv;
  int b = blockIdx.y / a.max_pieces;
  const int piece = blockIdx.y % a.max_pieces;
  if constexpr (R > 1) {
    static_assert(kWaves * 64 >= kMaxSorted, "a thread per pair");
    if (a.sorted) {
      __shared__ int s_pick;
      const int pair = sorted_pair(a, a.B * tiles, tiles, kRows, blockIdx.y * tiles + blockIdx.x / a.Hkv,
                                   reinterpret_cast<uint32_t*>(s_mem), &s_pick);
      b = pair / tiles; tile = pair % tiles;
    }
  }
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int row_wave = R > 1 ? wave : 0;
  // which unit of a round the wave brings, and (R > 1) whether its K (0) or its V (1)
  const int mine = kShared ? wave % kRoundUnits : wave, part = kShared ? wave / kRoundUnits : 0;
  const int row0 = tile * kRows;
  const int shift = a.plan[RD_PLAN_HDR + 4 * b + 3];  // (requested together with what the tile needs)
  Tile t;
  tile_rows(a, b, t);
  if (row0 >= t.rows) return;

  // queries: B operand of the first product, lane (row l % 16, dims of chunk l / 16)
  u32x4 qf[RB][kSteps];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int r = row0 + 16 * (RB * row_wave + rb) + col;
    const int rc = r < t.rows ? r : t.rows - 1;     // behind the last row: that row again, not written
    const int qi = rc / a.group;
    const int h = hk * a.group + (rc - qi * a.group);
    const T* qp = reinterpret_cast<const T*>(a.q) + t.q_off + (int64_t)h * a.q_sh + (int64_t)qi * a.q_ss + grp * (D / 4);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) qf[rb][s] = *reinterpret_cast<const u32x4*>(qp + 8 * s);
  }

  tile_keys<(kRows > 64)>(a, b, row0, kRows, t);
  if (piece >= t.n_pieces) return;
  const int lo = t.begin + piece * a.piece;
  const int hi = t.hi < lo + a.piece ? t.hi : lo + a.piece;

  // K and V rows of the piece through descriptors that begin at key lo (or at the slab's first row, `skip`
  // keys further, where a shift puts lo in front of it) and end behind the last attended key: rows outside
  // read as zeros without touching memory.
  const int skip = shift > lo ? shift - lo : 0;
  const int64_t end = hi < a.max_len + shift ? hi : a.max_len + shift;
  const bool any = end > (int64_t)lo + skip;
  const int64_t slab = (int64_t)b * a.c_sb + (int64_t)hk * a.c_sh + (any ? ((int64_t)lo + skip - shift) * kRec : 0);
  const int range = any ? (int)((end - lo - skip) * kRec) : 0;
  const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(a.k) + slab, 0, range, 0x00020000);
  const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(a.v) + slab, 0, range, 0x00020000);
  const int q_first = row0 / a.group;               // first query of the tile
  const __amdgpu_buffer_rsrc_t mr = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint64_t*>(a.bits) + ((int64_t)b * a.n_q + q_first) * a.words, 0, 0x7fffffff, 0x00020000);

  int mask_off[kMaskWords];                         // of the rows whose mask words the lane brings
#pragma unroll
  for (int x = 0; x < kMaskWords; ++x) {
    const int r = row0 + kMaskRows * part + (lane + 64 * x) % kMaskRows;
    mask_off[x] = ((r < t.rows ? r : t.rows - 1) / a.group - q_first) * a.words * 8;
  }

  const int n_units = (hi - lo + kUnit - 1) / kUnit;
  const int u0 = skip / kUnit;                      // (0, unless a shift points in front of the slab)
  constexpr uint32_t kStride = kRoundUnits * kUnitBytes, kNowhere = 0x80000000u;  // (beyond every range)
  uint32_t off_at, tail_at;                         // byte offsets of the lane in the coming unit, and in its last load
  u32x4 rk[kLoads], rv[kLoads];                     // (R > 1: rk alone, of K or V)
  const __amdgpu_buffer_rsrc_t first = kShared && part != 0 ? vr : kr;
  uint32_t mask[kMaskWords];
  // which units every row of the tile attends to in full: no mask is read for those
  auto is_full = [&](int i) __attribute__((always_inline)) {
    const int key0 = lo + i * kUnit;
    return key0 >= t.full_lo && key0 + kUnit <= t.full_hi;
  };
  auto fetch_mask = [&](int i) __attribute__((always_inline)) {
    if (i < n_units && !is_full(i)) {
#pragma unroll
      for (int x = 0; x < kMaskWords; ++x) mask[x] = __builtin_amdgcn_raw_buffer_load_b32(mr, mask_off[x], 4 * (lo / kUnit + i), 0);
    }
  };
  auto fetch = [&](int i) __attribute__((always_inline)) {
    fetch_mask(i);
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const uint32_t off = j + 1 < kLoads ? off_at + 1024 * j : tail_at;
      rk[j] = __builtin_amdgcn_raw_buffer_load_b128(first, off, 0, 0);
    }
    if constexpr (!kShared) {
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const uint32_t off = j + 1 < kLoads ? off_at + 1024 * j : tail_at;
        rv[j] = __builtin_amdgcn_raw_buffer_load_b128(vr, off, 0, 0);
      }
    }
    off_at += kStride; tail_at += kStride;
    asm volatile("" : "+v"(off_at), "+v"(tail_at));
  };
  auto fetch_first = [&]() __attribute__((always_inline)) {
    const int base = ((u0 + mine) * kUnit - skip) * kRec + 16 * lane;  // (negative for rows in front of the slab)
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int at = base + 1024 * j;
      const uint32_t off = at < 0 || (j + 1 == kLoads && lane >= kTail) ? kNowhere : (uint32_t)at;
      rk[j] = __builtin_amdgcn_raw_buffer_load_b128(first, off, 0, 0);
      if constexpr (!kShared) rv[j] = __builtin_amdgcn_raw_buffer_load_b128(vr, off, 0, 0);
    }
    fetch_mask(u0 + mine);
    off_at = (uint32_t)base + kStride;
    tail_at = lane < kTail ? (uint32_t)base + 1024 * (kLoads - 1) + kStride : kNowhere;
    asm volatile("" : "+v"(off_at), "+v"(tail_at));
  };
  // Between a wave's own writes and reads: LDS serves a wave's accesses in order, the compiler has to keep
  // that order too.
  auto own_order = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  };
  auto stage = [&](int i, char* slot) __attribute__((always_inline)) {
    char* const at = slot + (kShared ? part * kVAt : 0) + 16 * lane;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) *reinterpret_cast<u32x4*>(at + 1024 * j) = rk[j];
    if constexpr (!kShared) {
#pragma unroll
      for (int j = 0; j < kLoads; ++j) *reinterpret_cast<u32x4*>(at + kVAt + 1024 * j) = rv[j];
    }
    if (i < n_units && !is_full(i)) {
#pragma unroll
      for (int x = 0; x < kMaskWords; ++x)
        if (kMaskRows % 64 == 0 || lane + 64 * x < kMaskRows)
          *reinterpret_cast<uint32_t*>(slot + kMaskAt + 4 * (kMaskRows * part + lane + 64 * x)) = mask[x];
    }
  };
  // the lane's codes and scales of a unit's records, for the operands of the two products
  struct Codes { uint32_t k[2][kKw], ks[2], v[8][kVw], vs[8]; };
  auto k_codes = [&](const char* s_k, Codes& c) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const char* rec = s_k + (16 * h + col) * kRec;
      if constexpr (kKw == 2) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(rec + 8 * grp);
        c.k[h][0] = w[0]; c.k[h][1] = w[1];
      } else {
#pragma unroll
        for (int p = 0; p < kKw / 4; ++p) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(rec + 4 * kKw * grp + 16 * p);
#pragma unroll
          for (int e = 0; e < 4; ++e) c.k[h][4 * p + e] = w[e];
        }
      }
      if constexpr (kSteps == 4) c.ks[h] = *reinterpret_cast<const uint32_t*>(rec + kCodes + 4 * grp);
      else c.ks[h] = *reinterpret_cast<const uint16_t*>(rec + kCodes + 2 * grp);
    }
  };
  auto v_codes = [&](const char* s_v, Codes& c) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const char* rec = s_v + (16 * (j / 4) + 4 * grp + j % 4) * kRec;
      if constexpr (kColBytes == 2) c.v[j][0] = *reinterpret_cast<const uint16_t*>(rec + 2 * col);
      else if constexpr (kColBytes == 4) c.v[j][0] = *reinterpret_cast<const uint32_t*>(rec + 4 * col);
      else {
        const u32x2 w = *reinterpret_cast<const u32x2*>(rec + 8 * col);
        c.v[j][0] = w[0]; c.v[j][1] = w[1];
      }
      c.vs[j] = *reinterpret_cast<const uint8_t*>(rec + kCodes + col * kCols / kBlock);
    }
  };
  // step s of the keys 16 h + col
  auto k_operand = [&](const Codes& c, int s, int h) __attribute__((always_inline)) {
    // byte s of the scales in the exponent field (the conversion looks at nothing else)
    const uint32_t e = s == 0 ? c.ks[h] << 23 : (s == 1 ? c.ks[h] << 15 : (s == 2 ? c.ks[h] << 7 : c.ks[h] >> 1));
    uint32_t w[4];
    convert<T, BITS, 4>(&c.k[h][s * BITS / 4], __uint_as_float(e), w);
    return u32x4{w[0], w[1], w[2], w[3]};
  };
  // pairs of (dim, dim + 1) of one key -> pairs of keys of one dim: dims 2 d and 2 d + 1 of the lane's column
  struct VPairs { uint32_t w[8][kCols / 2]; };
  auto v_pairs = [&](const Codes& c) __attribute__((always_inline)) {
    VPairs p;
#pragma unroll
    for (int j = 0; j < 8; ++j) convert<T, BITS, kCols / 2>(c.v[j], __uint_as_float(c.vs[j] << 23), p.w[j]);
    return p;
  };
  auto v_operand = [&](const VPairs& p, int j) __attribute__((always_inline)) {
    u32x4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      r[e] = __builtin_amdgcn_perm(p.w[2 * e + 1][j / 2], p.w[2 * e][j / 2], j % 2 == 0 ? 0x05040100u : 0x07060302u);
    return r;
  };
  // the wave's part of a slot: records -> operands, in the order the lanes read them back
  auto convert_part = [&](char* slot) __attribute__((always_inline)) {
    Codes c;
    own_order();
    u32x4* const dst = reinterpret_cast<u32x4*>(slot) + lane;
    if (part == 0) {
      k_codes(slot, c);
      own_order();
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        dst[64 * (2 * s)] = k_operand(c, s, 0);
        dst[64 * (2 * s + 1)] = k_operand(c, s, 1);
      }
    } else {
      v_codes(slot + kVAt, c);
      own_order();
      const VPairs p = v_pairs(c);
#pragma unroll
      for (int j = 0; j < kCols; ++j) dst[64 * (2 * kSteps + j)] = v_operand(p, j);
    }
  };
  if (any) fetch_first();

  const bool active = row0 + 16 * RB * row_wave < t.rows;  // (a wave without rows only brings and converts units)

  // o: output tiles, l: row sums (the product of P with ones: every element of a lane's l is its row's sum),
  // m: running maximum in log2 units, over: the score above which it is raised (second sweep: the score of m)
  f32x4 o[RB][kCols], l[RB];
  float m[RB], over[RB];
  float inf = INFINITY;
  asm volatile("" : "+v"(inf));
  const u32x4 ones = {O::kOne * 0x10001u, O::kOne * 0x10001u, O::kOne * 0x10001u, O::kOne * 0x10001u};

  // mask bits of the wave's rows for the unit whose records lie at `here`
  auto read_mask = [&](const char* here, bool full, uint32_t (&on)[RB]) __attribute__((always_inline)) {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      on[rb] = 0xffffffffu;
      if (!full) on[rb] = *reinterpret_cast<const uint32_t*>(here + kMaskAt + 4 * (16 * (RB * row_wave + rb) + col));
    }
  };
  // V of keys that no row of the wave attends to is left out, whatever it holds; blocks that read back as NaN
  // (or that no append wrote: a scale beyond the type's range) are left out too, and rows that attend to
  // one get their NaN from the product of the mask with the marks of those blocks.
  auto part_nan = [&](Codes& c, const uint32_t (&on)[RB]) __attribute__((always_inline)) {
    constexpr uint32_t kCap = (uint32_t)scale_max(BITS, O::kF16);
    uint32_t seen = 0;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) seen |= on[rb];
#pragma unroll
    for (int x = 1; x < 16; x *= 2) seen |= (uint32_t)__shfl_xor((int)seen, x);
    u32x4 bad;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool unseen = ((seen >> (16 * (j / 4) + 4 * grp + j % 4)) & 1) == 0, is_bad = c.vs[j] > kCap;
#pragma unroll
      for (int w = 0; w < kVw; ++w) c.v[j][w] = unseen || is_bad ? 0u : c.v[j][w];
      c.vs[j] = unseen || is_bad ? 127u : c.vs[j];
      const uint32_t mark = is_bad && !unseen ? O::kOne : 0u;
      if (j % 2 == 0) bad[j / 2] = mark; else bad[j / 2] |= mark << 16;
    }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      u32x4 has;
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const uint32_t two = on[rb] >> (16 * (j / 4) + 4 * grp + j % 4);
        has[j / 2] = ((two & 1) ? O::kOne : 0u) | ((two & 2) ? O::kOne << 16 : 0u);
      }
      const f32x4 count = O::mfma(bad, has, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float poison = count[e] > 0.f ? NAN : 0.f;
#pragma unroll
        for (int j = 0; j < kCols; ++j) o[rb][j][e] += poison;
      }
    }
  };
  // Scores to weights.  sc[rb][h] holds keys 16 h + 4 grp + e of row `col`; the weights come out in the order
  // of the second product's B operand.  kCheck: scores are subtracted before they are scaled (one instruction more per
  // weight), so that the rounding of a large m in log2 units is no factor of the row's weights.
  auto weights = [&](auto check_c, f32x4 (&sc)[RB][2], bool full, const uint32_t (&on)[RB], u32x4 (&pf)[RB]) __attribute__((always_inline)) {
    constexpr bool kCheck = decltype(check_c)::value;
    if (!full) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        uint32_t w = on[rb] >> (4 * grp);
        asm volatile("" : "+v"(w));                 // (keeps this a branch: as selects on every unit it would cost 24 instructions per row block)
#pragma unroll
        for (int j = 0; j < 8; ++j) sc[rb][j / 4][j % 4] = (w >> (16 * (j / 4) + j % 4)) & 1 ? sc[rb][j / 4][j % 4] : -INFINITY;
      }
    }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = sc[rb][j / 4][j % 4];
      const float top = fmaxf(fmaxf(larger(x[0], x[1], inf), larger(x[2], x[3], inf)), fmaxf(larger(x[4], x[5], inf), larger(x[6], x[7], inf)));
      if (__ballot(kCheck ? top - over[rb] > a.rise : top > over[rb]) != 0) {
        const float raw = kCheck ? fmaxf(over[rb], row_max(top)) : 0.f;
        const float up = kCheck ? raw * a.scale : fmaxf(m[rb], row_max(top) * a.scale);
        const float keep = up == -INFINITY ? 1.f : fast_exp2(m[rb] - up);
        m[rb] = up;
        over[rb] = kCheck ? raw : (up + 8.f) * a.inv_scale;
        l[rb] *= keep;
#pragma unroll
        for (int j = 0; j < kCols; ++j) o[rb][j] *= keep;
      }
      // nothing attended yet: every p below is exp2(-inf).  fp16 weights are held 2^7 times as large, 2^15 at most: its
      // smallest number is 2^-24, and 2^23 keys of 2^-26 of the largest weight are an eighth of the sum.  The sum has
      // the factor too, and so the quotient has not.
      const float m_use = fmaxf(kCheck ? over[rb] : m[rb], -3.4e38f) - (kCheck ? 0.f : O::kLift);
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = fast_exp2(kCheck ? __builtin_fmaf(x[j] - m_use, a.scale, O::kLift) : __builtin_fmaf(x[j], a.scale, -m_use));
      pf[rb] = u32x4{O::pack(p[0], p[1]), O::pack(p[2], p[3]), O::pack(p[4], p[5]), O::pack(p[6], p[7])};
    }
  };

  // The queries are waited for here, before the next unit's loads go out: left to its first use, the wait sits
  // in the loop, where it waits for those loads too, unit after unit.
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int s = 0; s < kSteps; ++s) asm volatile("" : "+v"(qf[rb][s]));
  auto sweep = [&](auto check_c) __attribute__((always_inline)) {
    constexpr bool kCheck = decltype(check_c)::value;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      m[rb] = -INFINITY; over[rb] = -INFINITY; l[rb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < kCols; ++j) o[rb][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (!any) return;                               // (uniform over the workgroup)
    if constexpr (!kShared) {
      // Every wave by itself.  While unit i is multiplied with V, unit i + kWaves goes to LDS and its K codes
      // come back, and unit i + 2 kWaves is on its way from memory.
      char* const slot = s_mem + wave * kSlotBytes;
      int i = u0 + wave;
      Codes c;
      auto next = [&](int n) __attribute__((always_inline)) {
        own_order();
        stage(n, slot);
        if (n + kWaves < n_units) fetch(n + kWaves);
        own_order();
        k_codes(slot, c);
      };
      if (i < n_units) next(i);
      for (; i < n_units; i += kWaves) {
        const bool full = is_full(i);
        uint32_t on[RB];
        read_mask(slot, full, on);
        v_codes(slot + kVAt, c);
        f32x4 sc[RB][2];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) sc[rb][0] = sc[rb][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          const u32x4 k0 = k_operand(c, s, 0), k1 = k_operand(c, s, 1);
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) {
            sc[rb][0] = O::mfma(k0, qf[rb][s], sc[rb][0]);
            sc[rb][1] = O::mfma(k1, qf[rb][s], sc[rb][1]);
          }
        }
        __builtin_amdgcn_s_setprio(0);
        if constexpr (kCheck) part_nan(c, on);
        u32x4 pf[RB];
        weights(check_c, sc, full, on, pf);
        const VPairs pairs = v_pairs(c);
        if (i + kWaves < n_units) next(i + kWaves);
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);             // (as below: 8 x 32 heads, 128 queries, 1000 keys: 37.5 -> 35.0 us)
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) l[rb] = O::mfma(ones, pf[rb], l[rb]);
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
          const u32x4 vf = v_operand(pairs, j);
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) o[rb][j] = O::mfma(vf, pf[rb], o[rb][j]);
        }
      }
    } else {
      // Rounds of kRoundUnits units, which every wave goes over.  Meanwhile it brings its part of the coming
      // round into the other buffer: those with K before the first unit, those with V, which share their
      // SIMDs, in the middle of the round.
      auto bring = [&](int round, int buffer) __attribute__((always_inline)) {
        char* const slot = s_mem + (buffer * kRoundUnits + mine) * kSlotBytes;
        __builtin_amdgcn_s_setprio(0);
        stage(round + mine, slot);
        if (round + kRoundUnits < n_units) fetch(round + kRoundUnits + mine);
        if constexpr (!kCheck) convert_part(slot);
      };
      __syncthreads();                              // (the first sweep's units are no longer read)
      bring(u0, 0);
      int buffer = 0;
      for (int round = u0; round < n_units; round += kRoundUnits, buffer ^= 1) {
        __syncthreads();
        const int last = n_units - round < kRoundUnits ? n_units - round : kRoundUnits;
        const bool more = round + kRoundUnits < n_units;
        const char* const units = s_mem + buffer * kRoundUnits * kSlotBytes;
        if (more && (part == 0 || !active)) bring(round + kRoundUnits, buffer ^ 1);
        u32x4 kf[2 * kSteps];                       // K operands, requested one unit ahead
        if constexpr (!kCheck) {
#pragma unroll
          for (int f = 0; f < 2 * kSteps; ++f) kf[f] = reinterpret_cast<const u32x4*>(units)[64 * f + lane];
        }
        if (!active) continue;
        for (int slot = 0; slot < last; ++slot) {
          if (more && part != 0 && slot == kRoundUnits / 2) bring(round + kRoundUnits, buffer ^ 1);
          const bool full = is_full(round + slot);
          const char* const here = units + slot * kSlotBytes;
          uint32_t on[RB];
          read_mask(here, full, on);
          Codes c;
          if constexpr (kCheck) {
            k_codes(here, c);
            v_codes(here + kVAt, c);
          }
          f32x4 sc[RB][2];
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) sc[rb][0] = sc[rb][1] = f32x4{0.f, 0.f, 0.f, 0.f};
          // The wave in the matrix products goes before the one in the softmax on the same SIMD, whose
          // exponentials fill the gaps; with equal priorities the two tend to be in the same phase
          // (8 x 32 heads, 768 queries, 8192 keys: 941 -> 919 us, of 64 dims 551 -> 530).
          __builtin_amdgcn_s_setprio(1);
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            if constexpr (kCheck) {
              kf[2 * s] = k_operand(c, s, 0);
              kf[2 * s + 1] = k_operand(c, s, 1);
            }
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
              sc[rb][0] = O::mfma(kf[2 * s], qf[rb][s], sc[rb][0]);
              sc[rb][1] = O::mfma(kf[2 * s + 1], qf[rb][s], sc[rb][1]);
            }
          }
          u32x4 vf[kCols];
          if constexpr (!kCheck) {
            const u32x4* const ready = reinterpret_cast<const u32x4*>(here) + lane;
#pragma unroll
            for (int j = 0; j < kCols / 2; ++j) vf[j] = ready[64 * (2 * kSteps + j)];
            const u32x4* const next = reinterpret_cast<const u32x4*>(units + (slot + 1 < last ? slot + 1 : slot) * kSlotBytes) + lane;
#pragma unroll
            for (int f = 0; f < 2 * kSteps; ++f) kf[f] = next[64 * f];
            __builtin_amdgcn_sched_barrier(0);      // (requested here, so that the softmax covers the way)
          } else {
            part_nan(c, on);
          }
          u32x4 pf[RB];
          __builtin_amdgcn_s_setprio(0);
          weights(check_c, sc, full, on, pf);
          __builtin_amdgcn_s_setprio(1);
          if constexpr (!kCheck) {
            const u32x4* const ready = reinterpret_cast<const u32x4*>(here) + lane;
#pragma unroll
            for (int j = kCols / 2; j < kCols; ++j) vf[j] = ready[64 * (2 * kSteps + j)];
          }
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) l[rb] = O::mfma(ones, pf[rb], l[rb]);
          VPairs pairs;
          if constexpr (kCheck) pairs = v_pairs(c);
#pragma unroll
          for (int j = 0; j < kCols; ++j) {
            if constexpr (kCheck) vf[j] = v_operand(pairs, j);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) o[rb][j] = O::mfma(vf[j], pf[rb], o[rb][j]);
          }
        }
      }
    }
  };
  sweep(std::false_type{});
  // A NaN in the output comes from one that somebody attends to, or from a NaN block of V under a masked
  // key (0 * NaN): the wave goes over its keys once more and keeps the two apart.  So it does where a row's
  // maximum is so large that its rounding, a factor of all the row's weights, can leave the type's range (finite scores of
  // 2^28 in log2 units gave NaN or zeros); in the loop of the first sweep that would cost 2 to 10 % of every launch.
  bool odd_row = false;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) odd_row = odd_row || (fabsf(m[rb]) > kFar && m[rb] != -INFINITY);
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int j = 0; j < kCols; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) odd_row = odd_row || o[rb][j][e] != o[rb][j][e];
  if constexpr (R > 1) odd_row = __syncthreads_or(odd_row);  // (all of them: the rounds have barriers)
  if (__builtin_expect(__ballot(odd_row) != 0, 0)) {
    fetch_first();
    sweep(std::true_type{});
  }

  // A lane holds the dims [4 kCols grp, 4 kCols (grp + 1)) of its rows.
  if constexpr (K == 1) {
    // The finished rows (keys are not cut here) go through LDS, from where the lanes write whole rows one behind
    // the other (the epilogue of 256 rows of 128 dims: 7.9 -> 2.5 us).
    typedef u32x4 u32x4_any __attribute__((aligned(8)));
    constexpr int kOutPitch = 2 * D + 16, kRowLanes = D / 8, kStepRows = 64 / kRowLanes;
    static_assert(kWaves * 16 * RB * kOutPitch <= kLdsBytes, "LDS of the finished rows");
    char* const rows = s_mem + wave * 16 * RB * kOutPitch;
    __syncthreads();                                // (the units are no longer read)
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const float sum = l[rb][0], inv = sum == 0.f ? 0.f : 1.f / sum;  // (a NaN sum stays one)
      float x[4 * kCols];                           // (the lane's dims in their order)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < kCols; ++j) x[kCols * i + j] = o[rb][j][i] * inv;
#pragma unroll
      for (int c = 0; c < 4 * kCols; c += 8)
        *reinterpret_cast<u32x4*>(rows + (16 * rb + col) * kOutPitch + 2 * (4 * kCols * grp + c)) =
            u32x4{O::pack(x[c], x[c + 1]), O::pack(x[c + 2], x[c + 3]), O::pack(x[c + 4], x[c + 5]), O::pack(x[c + 6], x[c + 7])};
    }
    own_order();
#pragma unroll
    for (int r0 = 0; r0 < 16 * RB; r0 += kStepRows) {
      const int rr = r0 + lane / kRowLanes, r = row0 + 16 * RB * row_wave + rr;
      if (r >= t.rows) continue;
      const int qi = r / a.group, h = hk * a.group + (r - qi * a.group);
      T* op = reinterpret_cast<T*>(a.out) + t.o_off + (int64_t)h * a.o_sh + (int64_t)qi * a.o_ss + lane % kRowLanes * 8;
      *reinterpret_cast<u32x4_any*>(op) = *reinterpret_cast<const u32x4*>(rows + rr * kOutPitch + 16 * (lane % kRowLanes));
    }
  } else {
    // four neighbouring dims of row r: the result, or this piece's part of it (m in log2 units)
    auto put = [&](int r, int dq, f32x4 acc, float top, float sum) __attribute__((always_inline)) {
      if (t.n_pieces > 1) {
        const int64_t slot = ((int64_t)b * a.Hkv + hk) * a.max_pieces + piece;
        const int64_t pr = slot * ((int64_t)a.n_q * a.group) + r;
        *reinterpret_cast<f32x4*>(a.part_o + pr * D + dq) = acc;
        if (dq == 0) { a.part_ml[2 * pr] = top; a.part_ml[2 * pr + 1] = sum; }
      } else {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;  // (a NaN sum stays one)
        const int qi = r / a.group, h = hk * a.group + (r - qi * a.group);
        T* op = reinterpret_cast<T*>(a.out) + t.o_off + (int64_t)h * a.o_sh + (int64_t)qi * a.o_ss + dq;
        const u32x2 w = {O::pack(acc[0] * inv, acc[1] * inv), O::pack(acc[2] * inv, acc[3] * inv)};
        *reinterpret_cast<u32x2*>(op) = w;
      }
    };
    // merge the K waves behind each other; row of the merge: (wave * RB + row block) * 16 + col
    constexpr int kThreads = kWaves * 64, kQuads = D / 4, kBlocks = R * RB;
    __syncthreads();                                // (the units are no longer read)
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int at = (wave * RB + rb) * 16 + col;
      float* dst = s_o + at * kPitch + 4 * kCols * grp;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < kCols; j += 4)
          *reinterpret_cast<f32x4*>(dst + kCols * i + j) = f32x4{o[rb][j][i], o[rb][j + 1][i], o[rb][j + 2][i], o[rb][j + 3][i]};
      }
      if (grp == 0) { s_ml[at * 2] = m[rb]; s_ml[at * 2 + 1] = l[rb][0]; }
    }
    __syncthreads();
#pragma unroll
    for (int e0 = 0; e0 < 16 * kBlocks * kQuads; e0 += kThreads) {
      const int rr = (e0 + tid) / kQuads, dq = (e0 + tid) % kQuads * 4;
      const int r = row0 + rr;
      if (r >= t.rows) continue;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < K; ++w) top = fmaxf(top, s_ml[(w * 16 * kBlocks + rr) * 2]);
      const float m_use = fmaxf(top, -3.4e38f);
      float sum = 0.f;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < K; ++w) {
        const int at = w * 16 * kBlocks + rr;
        const float f = fast_exp2(s_ml[at * 2] - m_use);  // a wave without keys: exp2(-inf)
        sum += f * s_ml[at * 2 + 1];
        acc += f * *reinterpret_cast<const f32x4*>(s_o + at * kPitch + dq);
      }
      put(r, dq, acc, top, sum);
    }
  }
}

// Joins the pieces of rows whose keys were cut (32 pieces of 32 rows of 128 dims: 4.0 us, of which the smallest launches
// take 2.4; 18 us with one thread group per row and one piece at a time).  D / 4 threads carry a row's dims; with many pieces `parts`
// such groups of a workgroup share a row (piece p goes to group p % parts) and are joined through LDS.  Four
// pieces are requested at a time: the kernel is the latency of its loads.
constexpr int kMergeThreads = 256, kMergeMaxParts = 8;
struct Partial { float m, l; f32x4 o; };
__device__ inline Partial join(const Partial& a, const Partial& b) {
  const float up = fmaxf(a.m, b.m), m_use = fmaxf(up, -3.4e38f);
  const float fa = fast_exp2(a.m - m_use), fb = fast_exp2(b.m - m_use);
  return {up, fa * a.l + fb * b.l, fa * a.o + fb * b.o};
}
template <typename T>
__global__ __launch_bounds__(kMergeThreads) void attn_quant_merge_kernel(QuantArgs a, int rows_per_tile, int parts) {
  using O = Ops<T>;
  __shared__ Partial s_part[kMergeThreads];
  const int hk = blockIdx.y, b = blockIdx.z;
  const int quads = a.D / 4, per_row = quads * parts, rows_per_wg = kMergeThreads / per_row;
  const int sub = threadIdx.x / per_row, part = threadIdx.x % per_row / quads, dq = threadIdx.x % quads * 4;
  const int64_t r64 = (int64_t)blockIdx.x * rows_per_wg + sub;
  const int64_t all_rows = (int64_t)a.n_q * a.group;
  const int r = r64 < all_rows ? (int)r64 : (int)all_rows - 1;
  const Tile t = tile_of(a, b, r / rows_per_tile * rows_per_tile, rows_per_tile);
  const bool mine = r64 < all_rows && r < t.rows && t.n_pieces > 1;
  const int n = mine ? t.n_pieces : 0;
  Partial acc = {-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f}};
  const int64_t first = ((int64_t)b * a.Hkv + hk) * a.max_pieces;
  for (int p0 = part; p0 < n; p0 += 4 * parts) {
    Partial x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = p0 + i * parts < n ? p0 + i * parts : p0;  // (past the last piece: one that is there, not counted)
      const int64_t pr = (first + p) * all_rows + r;
      x[i].m = a.part_ml[2 * pr];
      x[i].l = a.part_ml[2 * pr + 1];
      x[i].o = *reinterpret_cast<const f32x4*>(a.part_o + pr * a.D + dq);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (p0 + i * parts < n) acc = join(acc, x[i]);
  }
  if (parts > 1) {
    s_part[threadIdx.x] = acc;
    __syncthreads();
    if (part == 0)
      for (int i = 1; i < parts; ++i) acc = join(acc, s_part[threadIdx.x + i * quads]);
  }
  if (!mine || part != 0) return;
  const float inv = acc.l == 0.f ? 0.f : 1.f / acc.l;
  const int qi = r / a.group, h = hk * a.group + (r - qi * a.group);
  T* op = reinterpret_cast<T*>(a.out) + t.o_off + (int64_t)h * a.o_sh + (int64_t)qi * a.o_ss + dq;
  const u32x2 w = {O::pack(acc.o[0] * inv, acc.o[1] * inv), O::pack(acc.o[2] * inv, acc.o[3] * inv)};
  *reinterpret_cast<u32x2*>(op) = w;
}

// ---------------------------------------------------------------------------------------------
// Generic kernel: one workgroup per (query, head, batch row); keys in chunks of 256.  For types and head sizes that
// no workload of this framework decodes with; each key's record is read by one lane.
// ---------------------------------------------------------------------------------------------
constexpr int kGenThreads = 256;

template <typename T> __device__ inline float ld(const T* p);
template <> __device__ inline float ld<float>(const float* p) { return *p; }
template <> __device__ inline float ld<__hip_bfloat16>(const __hip_bfloat16* p) { return __bfloat162float(*p); }
template <> __device__ inline float ld<__half>(const __half* p) { return __half2float(*p); }
template <typename T> __device__ inline void st(T* p, float v);
template <> __device__ inline void st<float>(float* p, float v) { *p = v; }
template <> __device__ inline void st<__hip_bfloat16>(__hip_bfloat16* p, float v) { *p = __float2bfloat16(v); }
template <> __device__ inline void st<__half>(__half* p, float v) { *p = __float2half(v); }

// value d of the record at `rec`
__device__ inline float held(const char* rec, int bits, int dim, int d) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const uint32_t scale = reinterpret_cast<const uint8_t*>(rec)[code_bytes(bits, dim) + d / kBlock];
  const float s = __uint_as_float(scale << 23);
  uint32_t byte = reinterpret_cast<const uint8_t*>(rec)[d * bits / 8];
  const f32x2 p = bits == 4 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(byte, s, 0)
                            : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(byte, s, false);
  return bits == 4 && (d & 1) ? p[1] : p[0];
}

__device__ inline float block_reduce(float v, bool is_max, float* s_tmp) {
  for (int off = 32; off > 0; off >>= 1) {
    const float o = __shfl_xor(v, off);
    v = is_max ? fmaxf(v, o) : v + o;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s_tmp[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = s_tmp[0];
  for (int w = 1; w < kGenThreads / 64; ++w) r = is_max ? fmaxf(r, s_tmp[w]) : r + s_tmp[w];
  return r;
}

template <typename T>
__global__ __launch_bounds__(kGenThreads) void attn_quant_generic_kernel(QuantArgs a) {
  __shared__ float s_q[kMaxDim];
  __shared__ float s_p[kGenThreads];
  __shared__ float s_tmp[kGenThreads / 64];
  const int q = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int hk = h / a.group, D = a.D, bits = a.bits_per_code, tid = threadIdx.x;
  const Tile t = tile_of(a, b, q * a.group, a.group);
  if (q * a.group >= t.rows) return;
  const T* qp = reinterpret_cast<const T*>(a.q) + t.q_off + (int64_t)h * a.q_sh + (int64_t)q * a.q_ss;
  const int shift = a.plan[RD_PLAN_HDR + 4 * b + 3];
  const int rec = record_bytes(bits, D);
  const int64_t slab = (int64_t)b * a.c_sb + (int64_t)hk * a.c_sh;
  if (tid < D) s_q[tid] = ld<T>(qp + tid) * a.scale;
  __syncthreads();
  const uint64_t* brow = a.bits + ((int64_t)b * a.n_q + q) * a.words;
  float m = -INFINITY, l = 0.f, acc = 0.f;
  for (int c0 = t.begin; c0 < t.hi; c0 += kGenThreads) {
    const int j = c0 + tid;
    const int64_t row = (int64_t)j - shift;
    // (a shift that leaves the slab is never followed)
    const bool on = j < t.hi && ((brow[j >> 6] >> (j & 63)) & 1ull) && row >= 0 && row < a.max_len;
    float sc = -INFINITY;
    if (on) {
      const char* kr = a.k + slab + row * rec;
      float dot = 0.f;
      for (int d = 0; d < D; ++d) dot += s_q[d] * held(kr, bits, D, d);
      sc = dot;
    }
    const float up = fmaxf(m, block_reduce(sc, true, s_tmp));
    const float m_use = fmaxf(up, -3.4e38f);
    const float p = on ? __expf(sc - m_use) : 0.f;
    const float csum = block_reduce(p, false, s_tmp);
    const float keep = __expf(m - m_use);
    l = l * keep + csum;
    s_p[tid] = on ? p : -1.f;   // masked: whatever V holds there is left out
    __syncthreads();
    if (tid < D) {
      acc *= keep;
      const int n = (t.hi - c0) < kGenThreads ? (t.hi - c0) : kGenThreads;
      for (int jj = 0; jj < n; ++jj) {
        const float pj = s_p[jj];
        if (pj != -1.f) acc += pj * held(a.v + slab + ((int64_t)(c0 + jj) - shift) * rec, bits, D, tid);
      }
    }
    m = up;
    __syncthreads();
  }
  if (tid < D) {
    T* op = reinterpret_cast<T*>(a.out) + t.o_off + (int64_t)h * a.o_sh + (int64_t)q * a.o_ss;
    st<T>(op + tid, l == 0.f ? 0.f : acc / l);
  }
}

// ---------------------------------------------------------------------------------------------
// Span table: first and one past the last key that 16 consecutive queries of a batch row attend to.
// ---------------------------------------------------------------------------------------------
// Within it, a run of whole units that all of them attend to in full: from the first such unit to the
// first one behind it that is not (looked for among the first 2^15 units).  A unit's words of the queries are
// read by as many neighbouring lanes.  Once per mask; bound by latency (two masks of 1900 x 1900: 5.1 us, one of
// 1 x 65 537: 5.0, 1 x 33: 3.0).
constexpr int kSpanThreads = 256, kSpanBits = 1 << 15;
__global__ __launch_bounds__(kSpanThreads) void attn_spans_kernel(const uint64_t* __restrict__ bits, int n_q, int words,
                                                                  int kv_len, int32_t* __restrict__ spans) {
  __shared__ uint32_t s_full[kSpanBits / 32];
  __shared__ int s_tmp[3][kSpanThreads / 64];
  const int b = blockIdx.y, q0 = blockIdx.x * kSpanQueries, tid = threadIdx.x;
  const int nq = n_q - q0 < kSpanQueries ? n_q - q0 : kSpanQueries;
  const uint32_t* rows = reinterpret_cast<const uint32_t*>(bits + ((int64_t)b * n_q + q0) * words);
  const int units = 2 * words, full_words = ((units < kSpanBits ? units : kSpanBits) + 31) / 32;
  for (int i = tid; i < full_words; i += kSpanThreads) s_full[i] = 0;
  __syncthreads();
  int lanes = 1;                                    // per unit: a power of two
  while (lanes < nq) lanes *= 2;
  const int q = tid % lanes < nq ? tid % lanes : nq - 1, step = kSpanThreads / lanes;
  int lo = kv_len, neg_hi = 0;
  for (int u = tid / lanes; u < (units + step - 1) / step * step; u += 4 * step) {  // (whole waves: shuffles below)
    uint32_t x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = u + i * step < units ? u + i * step : units - 1;
      x[i] = rows[(int64_t)q * units + at];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = u + i * step;
      uint32_t some = x[i], all = x[i];
      for (int o = 1; o < lanes; o *= 2) {
        some |= (uint32_t)__shfl_xor((int)some, o);
        all &= (uint32_t)__shfl_xor((int)all, o);
      }
      if (at >= units) continue;
      if (some != 0) {
        const int f = at * kUnit + __ffs((int)some) - 1, e = at * kUnit + 32 - __clz((int)some);
        lo = f < lo ? f : lo;
        neg_hi = -e < neg_hi ? -e : neg_hi;
      }
      if (all == 0xffffffffu && at < kSpanBits && tid % lanes == 0) atomicOr(&s_full[at / 32], 1u << (at % 32));
    }
  }
  __syncthreads();
  // first full unit, then the first one behind it that is not
  auto block_min = [&](int v, int* tmp) {
    for (int o = 32; o > 0; o >>= 1) {
      const int w = __shfl_xor(v, o);
      v = w < v ? w : v;
    }
    if ((tid & 63) == 0) tmp[tid >> 6] = v;
  };
  auto joined = [&](const int* tmp) {
    int v = tmp[0];
    for (int i = 1; i < kSpanThreads / 64; ++i) v = tmp[i] < v ? tmp[i] : v;
    return v;
  };
  const int none = full_words * 32;
  int full = none;
  for (int i = tid; i < full_words; i += kSpanThreads)
    if (s_full[i] != 0) { full = i * 32 + __ffs((int)s_full[i]) - 1; break; }
  block_min(lo, s_tmp[0]);
  block_min(neg_hi, s_tmp[1]);
  block_min(full, s_tmp[2]);
  __syncthreads();
  lo = joined(s_tmp[0]);
  neg_hi = joined(s_tmp[1]);
  full = joined(s_tmp[2]);
  int stop = none;
  for (int i = full / 32 + tid; i < full_words; i += kSpanThreads) {
    const uint32_t gaps = ~s_full[i] & (i == full / 32 ? ~0u << (full % 32) : ~0u);
    if (gaps != 0) { stop = i * 32 + __ffs((int)gaps) - 1; break; }
  }
  __syncthreads();                                  // (s_tmp is read above)
  block_min(stop, s_tmp[0]);
  __syncthreads();
  if (tid == 0) {
    stop = joined(s_tmp[0]);
    int32_t* out = spans + kSpanInts * ((int64_t)b * gridDim.x + blockIdx.x);
    out[0] = lo;
    out[1] = -neg_hi < kv_len ? -neg_hi : kv_len;
    out[2] = full < none ? full * kUnit : 0;
    out[3] = full < none ? stop * kUnit : 0;
  }
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
constexpr int kComputeUnits = 256;

// The launch of a shape: the workgroup's layout (see attn_quant_kernel) and how the keys are cut.
enum Layout { kNarrow, kMiddle2, kMiddle4, kWide };
constexpr int kTileRows[] = {16, 32, 32, 256}, kLayoutWaves[] = {8, 2, 4, 8};
struct Shape { int layout, tile_rows, tiles, piece, max_pieces, sorted; };
Shape shape_of(int batch, int n_heads, int n_kv_heads, int n_q, int kv_len, int head_dim) {
  Shape s;
  const int64_t rows = (int64_t)n_q * (n_heads / n_kv_heads), slabs = (int64_t)batch * n_kv_heads;
  // kWide converts a unit once for 256 rows, in one workgroup of eight waves on a compute unit.  It is the faster
  // one (batch 2, prompt of 1900, 32 / 8 heads: 87 us against 110 us) where its workgroups come out even, that is
  // where rows fill three quarters of what whole rounds of them hold: batch 8, 32 heads, 1200 keys in 4 bits,
  // 162 rows (0.75) 51 against 63 us, 128 rows (0.5) 42 against 37 us; batch 12, 128 rows over 1500 keys (0.38) 60
  // against 50 us.  Prompts wait for the longest of their tiles, which the first round has; they need a quarter of a
  // round more: batch 2, 32 / 8 heads, 1300 tokens (1.3 rounds) 55 against 62 us, batch 1, 2000 tokens (1 round) 75
  // against 61 us.
  // At head_dim 64, where the other layouts have three waves on a SIMD, it takes 7/8 (batch 8, 32 heads, 1200 keys: 200
  // rows 38 against 48 us, 400 rows (0.81) 72 against 67 us) and half a round (batch 1, 32 / 8 heads, 2500 tokens (1.25)
  // 63 against 57 us; batch 2, 1900 tokens (1.9) 60 against 65 us).
  // Two waves per tile where that alone gives every SIMD two waves (34 against 37 us), else four (batch 8,
  // 32 heads, 48 rows, 1000 keys: 27 against 34 us).
  const int64_t wide = slabs * rd::ceil_div(rows, 256), blocks = slabs * rd::ceil_div(rows, 32);
  const bool prompt = n_q > kv_len / 2;
  if (rows <= 16) s.layout = kNarrow;
  else if (prompt ? 4 * wide >= (head_dim == 64 ? 6 : 5) * kComputeUnits
                  : blocks >= (head_dim == 64 ? 7 : 6) * kComputeUnits * rd::ceil_div(wide, kComputeUnits)) s.layout = kWide;
  else s.layout = blocks >= 4 * kComputeUnits ? kMiddle2 : kMiddle4;
  s.tile_rows = kTileRows[s.layout];
  s.tiles = (int)rd::ceil_div(rows, s.tile_rows);
  // A prompt's large tiles, longest first whatever the mask: its last rows have the most keys, and so have the rows
  // of left padding, which attend to everything where the model asks for that (batch 2, 1900 tokens, such padding:
  // 133 -> 96 us; without padding 2.5 us more than in the order of the rows).
  s.sorted = s.layout == kWide && prompt && (int64_t)batch * s.tiles <= kMaxSorted;
  // Keys are cut into pieces as far as every SIMD needs waves: two with few rows, where the kernel waits for
  // memory (one sequence of 65 536 keys in 8 bits, 8 kv heads: 35 against 44 us), one otherwise (batch 8, 32
  // heads, 20 rows, 1000 keys: 25 against 30 us).  A piece has at least two (four) units per wave, and a cut
  // has to save what the merge of the pieces costs, which is about the time of 640 keys (3.5 us; batch 16, 8
  // kv heads, 1000 keys in two pieces 13.0, in one 10.6 us; one sequence of 2000 keys in four 12.1, in two
  // 14.4 us).
  const bool narrow = s.layout == kNarrow;
  const int waves = kLayoutWaves[s.layout], step = waves * kUnit;
  const int64_t have = slabs * s.tiles * waves, want = (narrow ? 8 : 4) * kComputeUnits;
  const int64_t most = rd::ceil_div(kv_len, (narrow ? 2 : 4) * step);
  int64_t pieces = have >= want ? 1 : want / have;  // (kWide: 1, it has 192 workgroups or more)
  pieces = pieces < most ? pieces : most;
  if ((int64_t)kv_len * (pieces - 1) < 640 * pieces) pieces = 1;
  s.piece = (int)(rd::ceil_div(rd::ceil_div((int64_t)kv_len + kUnit - 1, pieces), step) * step);
  s.max_pieces = (int)rd::ceil_div((int64_t)kv_len + kUnit - 1, s.piece);
  return s;
}

bool mfma_shape(int dtype, int head_dim) {
  return (dtype == RD_BF16 || dtype == RD_F16) && (head_dim == 64 || head_dim == 128);
}

template <typename T, int BITS, int D>
void launch(const QuantArgs& a, const Shape& s, hipStream_t stream) {
  const dim3 grid((unsigned)(a.Hkv * (int64_t)s.tiles), (unsigned)(a.B * (int64_t)s.max_pieces));
  rd::ScopedTiming rd_t("attn_quant_kernel", stream);
  const dim3 block(64 * kLayoutWaves[s.layout]);
  switch (s.layout) {
    case kNarrow: hipLaunchKernelGGL((attn_quant_kernel<T, BITS, D, 1, 1, 8>), grid, block, 0, stream, a); break;
    case kMiddle2: hipLaunchKernelGGL((attn_quant_kernel<T, BITS, D, 2, 1, 2>), grid, block, 0, stream, a); break;
    case kMiddle4: hipLaunchKernelGGL((attn_quant_kernel<T, BITS, D, 2, 1, 4>), grid, block, 0, stream, a); break;
    default: hipLaunchKernelGGL((attn_quant_kernel<T, BITS, D, 2, 8, 1>), grid, block, 0, stream, a); break;
  }
}

}  // namespace

extern "C" size_t rd_attn_spans_ints(int batch, int n_q) {
  return batch > 0 && n_q > 0 ? kSpanInts * (size_t)batch * rd::ceil_div(n_q, kSpanQueries) : 0;
}

extern "C" int rd_attn_spans(const uint64_t* bits, int batch, int n_q, int kv_len, int32_t* spans, void* stream) {
  RD_REQUIRE(batch > 0 && n_q > 0 && kv_len > 0, RD_EINVAL, "rd_attn_spans: bad sizes (batch %d n_q %d kv %d)", batch, n_q, kv_len);
  RD_REQUIRE(batch <= 65535, RD_ELIMIT, "rd_attn_spans: batch %d > 65535", batch);
  RD_REQUIRE(bits && spans, RD_EINVAL, "rd_attn_spans: null pointer");
  hipStream_t s = rd::as_stream(stream);
  {
    rd::ScopedTiming rd_t("attn_spans_kernel", s);
    hipLaunchKernelGGL(attn_spans_kernel, dim3((unsigned)rd::ceil_div(n_q, kSpanQueries), batch), dim3(kSpanThreads), 0, s,
                       bits, n_q, (kv_len + 63) / 64, kv_len, spans);
  }
  return rd::check_launch("rd_attn_spans");
}

extern "C" uint64_t rd_stream_capture_id(void* stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  // (the null stream is never captured, and asking it during another stream's capture is an error)
  if (stream == nullptr || hipStreamGetCaptureInfo(rd::as_stream(stream), &status, &id) != hipSuccess) return 0;
  return status == hipStreamCaptureStatusActive ? id + 1 : 0;
}

extern "C" size_t rd_verify_attention_quant_workspace_bytes(int dtype, int batch, int n_heads, int n_kv_heads, int n_q,
                                                            int kv_len, int head_dim) {
  if (batch <= 0 || n_heads <= 0 || n_kv_heads <= 0 || n_q <= 0 || kv_len <= 0 || n_heads % n_kv_heads != 0 ||
      !mfma_shape(dtype, head_dim)) return 0;
  const Shape s = shape_of(batch, n_heads, n_kv_heads, n_q, kv_len, head_dim);
  if (s.max_pieces == 1) return 0;
  const size_t rows = (size_t)batch * s.max_pieces * n_heads * n_q;
  return rd::align_up(rows * head_dim * sizeof(float), 256) + rd::align_up(rows * 2 * sizeof(float), 256);
}

extern "C" int rd_verify_attention_quant(const void* q, const int64_t* q_strides, const void* k_cache,
                                         const void* v_cache, const int64_t* cache_strides, int bits, int64_t max_len,
                                         void* out, const int64_t* o_strides, int dtype, int batch, int n_heads,
                                         int n_kv_heads, int n_q, int kv_len, int head_dim, float scale,
                                         const uint64_t* mask_bits, const int32_t* plan, const int32_t* spans,
                                         void* workspace, size_t workspace_bytes, int force_generic,
                                         const int32_t* row_start, void* stream) {
  const char* who = "rd_verify_attention_quant";
  RD_REQUIRE(batch > 0 && n_heads > 0 && n_kv_heads > 0 && n_q > 0 && kv_len > 0, RD_EINVAL,
             "%s: bad sizes (batch %d heads %d kv_heads %d n_q %d kv %d)", who, batch, n_heads, n_kv_heads, n_q, kv_len);
  RD_REQUIRE(n_heads % n_kv_heads == 0, RD_EINVAL, "%s: heads %d not a multiple of kv heads %d", who, n_heads, n_kv_heads);
  RD_REQUIRE(dtype == RD_BF16 || dtype == RD_F16 || dtype == RD_F32, RD_EINVAL, "%s: unknown dtype %d", who, dtype);
  RD_REQUIRE(known_bits(bits), RD_EINVAL, "%s: bits %d (4 or 8)", who, bits);
  RD_REQUIRE(known_dim(head_dim), RD_ELIMIT, "%s: head_dim %d must be a multiple of 32, at most %d", who, head_dim, kMaxDim);
  RD_REQUIRE(batch <= 65535 && n_heads <= 65535, RD_ELIMIT, "%s: batch/heads > 65535", who);
  RD_REQUIRE((int64_t)n_q * (n_heads / n_kv_heads) <= (1 << 30), RD_ELIMIT, "%s: too many query rows", who);
  RD_REQUIRE(kv_len <= (1 << 23), RD_ELIMIT, "%s: kv_len %d > 2^23", who, kv_len);
  RD_REQUIRE(q && k_cache && v_cache && out && mask_bits && plan && spans && q_strides && cache_strides && o_strides,
             RD_EINVAL, "%s: null pointer", who);
  RD_REQUIRE(max_len > 0, RD_EINVAL, "%s: empty cache", who);
  // (scores are held in log2 units)
  RD_REQUIRE(scale > 0.f && scale * 1.4426950408889634f <= 3.402823466e38f, RD_EINVAL,
             "%s: scale %g is not positive, or times log2(e) not finite", who, (double)scale);
  auto al = [](const void* p, int n) { return ((uintptr_t)p & (n - 1)) == 0; };
  RD_REQUIRE(al(k_cache, 16) && al(v_cache, 16) && al(spans, 16), RD_EINVAL, "%s: the cache and the spans must be 16-byte aligned", who);
  RD_REQUIRE(cache_strides[0] % 16 == 0 && cache_strides[1] % 16 == 0 && cache_strides[0] >= 0 && cache_strides[1] >= 0 &&
                 cache_strides[2] == record_bytes(bits, head_dim), RD_EINVAL,
             "%s: cache strides must be multiples of 16 bytes and rows %d bytes apart", who, record_bytes(bits, head_dim));
  QuantArgs a;
  a.q = q; a.q_sb = q_strides[0]; a.q_sh = q_strides[1]; a.q_ss = q_strides[2];
  a.k = reinterpret_cast<const char*>(k_cache); a.v = reinterpret_cast<const char*>(v_cache);
  a.c_sb = cache_strides[0]; a.c_sh = cache_strides[1];
  a.out = out; a.o_sb = o_strides[0]; a.o_sh = o_strides[1]; a.o_ss = o_strides[2];
  a.bits = mask_bits; a.plan = plan; a.spans = spans; a.row_start = row_start;
  a.part_o = nullptr; a.part_ml = nullptr;
  a.max_len = max_len;
  a.B = batch; a.H = n_heads; a.Hkv = n_kv_heads; a.group = n_heads / n_kv_heads; a.n_q = n_q; a.kv_len = kv_len;
  a.words = (kv_len + 63) / 64; a.D = head_dim; a.bits_per_code = bits;
  a.span_blocks = (int)rd::ceil_div(n_q, kSpanQueries);
  a.sorted = 0;
  a.max_pieces = 1; a.piece = (int)(rd::ceil_div((int64_t)kv_len + kUnit - 1, kUnit) * kUnit);
  a.scale = scale; a.inv_scale = 1.f; a.rise = 0.f;
  hipStream_t s = rd::as_stream(stream);
  auto whole = [](const int64_t* st, int m) { return st[0] % m == 0 && st[1] % m == 0 && st[2] % m == 0; };
  const bool mfma = !force_generic && mfma_shape(dtype, head_dim) && al(q, 16) && al(out, 8) && whole(q_strides, 8) && whole(o_strides, 4);
  if (mfma) {
    const Shape sh = shape_of(batch, n_heads, n_kv_heads, n_q, kv_len, head_dim);
    RD_REQUIRE((int64_t)batch * sh.max_pieces <= 65535 && (int64_t)n_kv_heads * sh.tiles <= 2147483647LL, RD_ELIMIT,
               "%s: grid too large", who);
    a.max_pieces = sh.max_pieces; a.piece = sh.piece;
    a.sorted = sh.sorted;
    a.scale = scale * 1.4426950408889634f;
    a.inv_scale = 1.f / a.scale;
    a.rise = 8.f / a.scale;
    if (!(a.rise <= 3.402823466e38f)) a.rise = 3.402823466e38f;  // (less than from no score at all, -infinity, to one)
    if (sh.max_pieces > 1) {
      const size_t need = rd_verify_attention_quant_workspace_bytes(dtype, batch, n_heads, n_kv_heads, n_q, kv_len, head_dim);
      RD_REQUIRE(workspace && workspace_bytes >= need, RD_EWORKSPACE, "%s: workspace %zu < %zu bytes", who, workspace_bytes, need);
      RD_REQUIRE(al(workspace, 256), RD_EINVAL, "%s: workspace not 256B aligned", who);
      a.part_o = reinterpret_cast<float*>(workspace);
      a.part_ml = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) +
                                           rd::align_up((size_t)batch * sh.max_pieces * n_heads * n_q * head_dim * sizeof(float), 256));
    }
    auto go = [&](auto zero) {
      using T = decltype(zero);
      if (bits == 4) { if (head_dim == 64) launch<T, 4, 64>(a, sh, s); else launch<T, 4, 128>(a, sh, s); }
      else { if (head_dim == 64) launch<T, 8, 64>(a, sh, s); else launch<T, 8, 128>(a, sh, s); }
      if (sh.max_pieces > 1) {
        rd::ScopedTiming rd_t("attn_quant_merge_kernel", s);
        const int parts = sh.max_pieces >= 16 ? kMergeMaxParts : (sh.max_pieces >= 8 ? 4 : 1);
        const int64_t per_wg = kMergeThreads / (head_dim / 4 * parts);
        hipLaunchKernelGGL(attn_quant_merge_kernel<T>, dim3((unsigned)rd::ceil_div((int64_t)n_q * a.group, per_wg), n_kv_heads, batch),
                           dim3(kMergeThreads), 0, s, a, sh.tile_rows, parts);
      }
    };
    if (dtype == RD_BF16) go(__hip_bfloat16{}); else go(__half{});
    return rd::check_launch(who);
  }
  const dim3 grid(n_q, n_heads, batch);
  {
    rd::ScopedTiming rd_t("attn_quant_generic_kernel", s);
    switch (dtype) {
      case RD_BF16: hipLaunchKernelGGL(attn_quant_generic_kernel<__hip_bfloat16>, grid, dim3(kGenThreads), 0, s, a); break;
      case RD_F16: hipLaunchKernelGGL(attn_quant_generic_kernel<__half>, grid, dim3(kGenThreads), 0, s, a); break;
      default: hipLaunchKernelGGL(attn_quant_generic_kernel<float>, grid, dim3(kGenThreads), 0, s, a); break;
    }
  }
  return rd::check_launch(who);
}
