// Masked attention over a KV cache held in 4 or 8 bits (gfx950; kv_quant.h has the row format).
//
//   O[b,q,h,:] = softmax_k( Q[b,h,q,:] . K[b,hk,k,:] * scale  masked by bits[b,q,k] ) V[b,hk,k,:]
//
// The mask bits and the row shifts are those of rd_verify_attention; a row that attends to nothing is
// written as zeros.  Two kernels behind one entry point:
//   attn_quant_kernel    bf16 and fp16, head_dim 64 and 128, on v_mfma_f32_16x16x32
//   attn_quant_generic_kernel  every other type and head size the cache has
//
// attn_quant_kernel.  The query heads of a kv head are folded into the rows (row = query * group +
// head in group), so that K and V are read once per kv head.  A workgroup owns 16 * RB rows and a
// piece of the keys; its waves take the 32-key units of the piece in turn, each with a running
// maximum, sum and accumulators of its own for all the rows, and are merged through LDS at the end.
// No tile passes through LDS and no wave waits for another inside the loop: a wave's loads land in
// the operand layout of the matrix instructions.
//   S^T = K Q^T  A operand: lane (key l % 16, chunk l / 16) needs 8 consecutive k-slots per step.  The
//                order of the dims in a dot product is free, so chunk c of the record is dims
//                [c D/4, (c+1) D/4): D/4 contiguous codes per lane, one block of 8 per step.
//   O^T = V^T P^T  A operand: lane (column l % 16, key group l / 16) needs 8 keys of one dim.  Column n
//                is the D/16 dims from n D/16 on, tile j of the output their j-th; the 8 keys are those
//                whose scores the lane already holds (16 t + 4 (l / 16) + i), so P^T goes from the
//                accumulators of the first product into the B operand of the second as it is.
//                Codes of two keys become two dims times two keys: two conversions (code pair x scale
//                to bf16, one instruction, exact) and two byte permutes.
// A query row lives in one column of the accumulators (l % 16), so rescaling is a lane scalar; the
// running maximum is lazy: raised only when some score exceeds it by 2^8, the row sum is kept per lane.
// Keys outside the piece and outside the row's attended span read as zeros through the range check of
// a buffer descriptor, without touching memory.
//
// V and masked keys: a probability of zero does not silence a NaN in V (0 * NaN).  Blocks of V that read
// back as NaN are taken out of the product, and the rows that attend to such a key get their NaN from a
// second product of the mask with the marks of those blocks.
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
  float scale;     // softmax scale; times log2 e for the MFMA kernel
  float inv_scale; // its reciprocal
};

__device__ inline float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

template <typename T> struct Ops;
template <> struct Ops<__hip_bfloat16> {
  using V8 = bf16x8;
  static constexpr bool kF16 = false;
  static constexpr uint32_t kOne = 0x3f80u;
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
};
__device__ inline Tile tile_of(const QuantArgs& a, int b, int row0, int rows_per_tile) {
  Tile t;
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
  t.lo = a.kv_len; t.hi = 0;
  if (row0 < t.rows) {
    const int end = row0 + rows_per_tile < t.rows ? row0 + rows_per_tile : t.rows;
    const int s0 = row0 / a.group / kSpanQueries, s1 = (end - 1) / a.group / kSpanQueries;
    for (int s = s0; s <= s1; ++s) {
      const int32_t* sp = a.spans + 2 * ((int64_t)b * a.span_blocks + s);
      t.lo = sp[0] < t.lo ? sp[0] : t.lo;
      t.hi = sp[1] > t.hi ? sp[1] : t.hi;
    }
  }
  t.begin = t.lo / kUnit * kUnit;
  t.n_pieces = t.hi > t.lo ? (t.hi - t.begin + a.piece - 1) / a.piece : 1;
  return t;
}

// the lanes l, l ^ 16, l ^ 32, l ^ 48 share a query row
__device__ inline float row_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}

// ---------------------------------------------------------------------------------------------
// MFMA kernel
// ---------------------------------------------------------------------------------------------
// A unit on its way: codes and scales of 32 keys and the rows' mask bits for them.
template <int BITS, int D, int RB>
struct Unit {
  static constexpr int kCw = D * BITS / 128;        // dwords of a lane's K chunk (D/4 codes)
  static constexpr int kVw = D * BITS / 512 > 0 ? D * BITS / 512 : 1;  // dwords of a lane's V column (D/16 codes)
  uint32_t k[2][kCw], ks[2];
  uint32_t v[8][kVw], vs[8];
  uint32_t mask[RB];
};

#ifndef WPE
#define WPE 2
#endif
template <typename T, int BITS, int D, int RB, int WAVES>
__global__ __launch_bounds__(WAVES * 64, WPE) void attn_quant_kernel(QuantArgs a) {
  using O = Ops<T>;
  using U = Unit<BITS, D, RB>;
  constexpr int kRec = record_bytes(BITS, D), kCodes = code_bytes(BITS, D);
  constexpr int kSteps = D / 32;                    // blocks of 8 dims in a K chunk
  constexpr int kCols = D / 16;                     // dims of a V column = tiles of the output
  constexpr int kColBytes = kCols * BITS / 8;
  constexpr int kRows = 16 * RB;
  constexpr int kPitch = D + 4;                     // floats of a merged row in LDS
  __shared__ __attribute__((aligned(16))) float s_o[WAVES * 16 * kPitch];
  __shared__ float s_ml[WAVES * 16 * 2];

  const int hk = blockIdx.x % a.Hkv, tile = blockIdx.x / a.Hkv;
  const int b = blockIdx.y / a.max_pieces, piece = blockIdx.y % a.max_pieces;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int row0 = tile * kRows;
  const Tile t = tile_of(a, b, row0, kRows);
  if (row0 >= t.rows || piece >= t.n_pieces) return;
  const int lo = t.begin + piece * a.piece;
  const int hi = t.hi < lo + a.piece ? t.hi : lo + a.piece;

  // K and V rows of the piece: offsets count from key lo, [first, hi) are read.  Rows from hi on read as
  // zeros through the descriptors' range check; keys of the first unit below `first` (which nobody
  // attends to and which may lie before the slab) read row `first` instead.
  const int shift = a.plan[RD_PLAN_HDR + 4 * b + 3];
  int first = lo > t.lo ? lo : t.lo;
  first = first > shift ? first : shift;            // (a shift is never followed out of the slab)
  int64_t end = hi < a.max_len + shift ? hi : a.max_len + shift;
  const bool any = end > first;
  const int64_t slab = (int64_t)b * a.c_sb + (int64_t)hk * a.c_sh + ((int64_t)lo - shift) * kRec;
  const int range = any ? (int)((end - lo) * kRec) : 0;
  const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(a.k) + slab, 0, range, 0x00020000);
  const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(a.v) + slab, 0, range, 0x00020000);
  const int q_first = row0 / a.group;               // first query of the tile
  const __amdgpu_buffer_rsrc_t mr = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint64_t*>(a.bits) + ((int64_t)b * a.n_q + q_first) * a.words, 0, 0x7fffffff, 0x00020000);

  // queries: B operand of the first product, lane (row l % 16, dims of chunk l / 16)
  u32x4 qf[RB][kSteps];
  int mask_off[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int r = row0 + 16 * rb + col;
    const int rc = r < t.rows ? r : t.rows - 1;     // behind the last row: that row again, not written
    const int qi = rc / a.group;
    mask_off[rb] = (qi - q_first) * a.words * 8;
    const int h = hk * a.group + (rc - qi * a.group);
    const T* qp = reinterpret_cast<const T*>(a.q) + t.q_off + (int64_t)h * a.q_sh + (int64_t)qi * a.q_ss + grp * (D / 4);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) qf[rb][s] = *reinterpret_cast<const u32x4*>(qp + 8 * s);
  }

  const int n_units = (hi - lo + kUnit - 1) / kUnit;
  const int i0 = (first - lo) / kUnit + wave;       // (0 + wave, unless a shift points in front of the slab)
  // Byte offsets of the lane's parts of unit i0.  They stay in registers and move by a unit stride per
  // turn, so that the rows inside a unit are constants in the loads' offset fields.
  uint32_t k_off = i0 * kUnit * kRec + col * kRec + D * BITS / 32 * grp, ks_off = i0 * kUnit * kRec + col * kRec + kCodes + kSteps * grp;
  uint32_t v_off = i0 * kUnit * kRec + 4 * grp * kRec + kColBytes * col, vs_off = i0 * kUnit * kRec + 4 * grp * kRec + kCodes + col * kCols / kBlock;
  constexpr uint32_t kStride = WAVES * kUnit * kRec;
  const int least = first - lo - i0 * kUnit;        // rows of the first unit that lie below `first`, if any
  auto fetch_k = [&](U& u, auto first_c) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t off = k_off, soff = ks_off;
      if constexpr (decltype(first_c)::value) {
        const int up = 16 * h + col < least ? (least - 16 * h - col) * kRec : 0;
        off += up; soff += up;
      }
      off += 16 * h * kRec; soff += 16 * h * kRec;
      if constexpr (U::kCw == 2) {
        const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(kr, off, 0, 0);
        u.k[h][0] = w[0]; u.k[h][1] = w[1];
      } else {
#pragma unroll
        for (int p = 0; p < U::kCw / 4; ++p) {
          const u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(kr, off + 16 * p, 0, 0);
#pragma unroll
          for (int e = 0; e < 4; ++e) u.k[h][4 * p + e] = w[e];
        }
      }
      if constexpr (kSteps == 4) u.ks[h] = __builtin_amdgcn_raw_buffer_load_b32(kr, soff, 0, 0);
      else u.ks[h] = __builtin_amdgcn_raw_buffer_load_b16(kr, soff, 0, 0);
    }
    k_off += kStride; ks_off += kStride;
    asm volatile("" : "+v"(k_off), "+v"(ks_off));
  };
  auto fetch_v = [&](U& u, auto first_c) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t off = v_off, soff = vs_off;
      const int row = 16 * (j / 4) + j % 4;
      if constexpr (decltype(first_c)::value) {
        const int up = row + 4 * grp < least ? (least - row - 4 * grp) * kRec : 0;
        off += up; soff += up;
      }
      off += row * kRec; soff += row * kRec;
      if constexpr (kColBytes == 2) u.v[j][0] = __builtin_amdgcn_raw_buffer_load_b16(vr, off, 0, 0);
      else if constexpr (kColBytes == 4) u.v[j][0] = __builtin_amdgcn_raw_buffer_load_b32(vr, off, 0, 0);
      else {
        const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(vr, off, 0, 0);
        u.v[j][0] = w[0]; u.v[j][1] = w[1];
      }
      u.vs[j] = __builtin_amdgcn_raw_buffer_load_b8(vr, soff, 0, 0);
    }
    v_off += kStride; vs_off += kStride;
    asm volatile("" : "+v"(v_off), "+v"(vs_off));
  };
  auto fetch_mask = [&](U& u, int i) __attribute__((always_inline)) {
    const int word = lo / kUnit + (i < n_units ? i : n_units - 1);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) u.mask[rb] = __builtin_amdgcn_raw_buffer_load_b32(mr, mask_off[rb], 4 * word, 0);
  };

  // o: output tiles, l: row sums (the product of P with ones: every element of a lane's l is its row's sum),
  // m: running maximum in log2 units, over: the score above which it is raised
  f32x4 o[RB][kCols], l[RB];
  float m[RB], over[RB];
  const u32x4 ones = {O::kOne * 0x10001u, O::kOne * 0x10001u, O::kOne * 0x10001u, O::kOne * 0x10001u};

  // Each part of a unit is requested again, for the wave's next unit, as soon as it has been used: one
  // set of registers, and the rest of the unit's work covers the trip.
  auto sweep = [&](auto check_c) __attribute__((always_inline)) {
    constexpr bool kCheck = decltype(check_c)::value;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      m[rb] = -INFINITY; over[rb] = -INFINITY; l[rb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < kCols; ++j) o[rb][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (!any || i0 >= n_units) return;
    U u;
    fetch_k(u, std::true_type{});
    fetch_mask(u, i0);
    fetch_v(u, std::true_type{});
    for (int i = i0; i < n_units; i += WAVES) {
      // scores: sc[rb][h] holds keys 16 h + 4 grp + e of row `col`
      f32x4 sc[RB][2];
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) sc[rb][0] = sc[rb][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        u32x4 kf[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // byte s of the scales in the exponent field (the conversion looks at nothing else)
          const uint32_t e = s == 0 ? u.ks[h] << 23 : (s == 1 ? u.ks[h] << 15 : (s == 2 ? u.ks[h] << 7 : u.ks[h] >> 1));
          uint32_t w[4];
          convert<T, BITS, 4>(&u.k[h][s * BITS / 4], __uint_as_float(e), w);
          kf[h] = u32x4{w[0], w[1], w[2], w[3]};
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          sc[rb][0] = O::mfma(kf[0], qf[rb][s], sc[rb][0]);
          sc[rb][1] = O::mfma(kf[1], qf[rb][s], sc[rb][1]);
        }
      }
      fetch_k(u, std::false_type{});
      if constexpr (kCheck) {
        // V blocks that read back as NaN (or that no append wrote: a scale beyond the type's range)
        constexpr uint32_t kCap = (uint32_t)scale_max(BITS, O::kF16);
        u32x4 bad;
#pragma unroll
        for (int j = 0; j < 8; j += 2)
          bad[j / 2] = (u.vs[j] > kCap ? O::kOne : 0u) | ((u.vs[j + 1] > kCap ? O::kOne : 0u) << 16);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool is_bad = u.vs[j] > kCap;
#pragma unroll
          for (int w = 0; w < U::kVw; ++w) u.v[j][w] = is_bad ? 0u : u.v[j][w];
          u.vs[j] = is_bad ? 127u : u.vs[j];
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          u32x4 on;
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            const uint32_t two = u.mask[rb] >> (16 * (j / 4) + 4 * grp + j % 4);
            on[j / 2] = ((two & 1) ? O::kOne : 0u) | ((two & 2) ? O::kOne << 16 : 0u);
          }
          const f32x4 count = O::mfma(bad, on, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float poison = count[e] > 0.f ? NAN : 0.f;
#pragma unroll
            for (int j = 0; j < kCols; ++j) o[rb][j][e] += poison;
          }
        }
      }
      // probabilities
      u32x4 pf[RB];
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const uint32_t w = u.mask[rb];
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = sc[rb][j / 4][j % 4];
        if (__ballot(w != 0xffffffffu) != 0) {
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = ((w >> (4 * grp)) >> (16 * (j / 4) + j % 4)) & 1 ? x[j] : -INFINITY;
        }
        const float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        if (__ballot(top > over[rb]) != 0) {
          const float up = fmaxf(m[rb], row_max(top) * a.scale);
          const float keep = up == -INFINITY ? 1.f : fast_exp2(m[rb] - up);
          m[rb] = up;
          over[rb] = (up + 8.f) * a.inv_scale;
          l[rb] *= keep;
#pragma unroll
          for (int j = 0; j < kCols; ++j) o[rb][j] *= keep;
        }
        const float m_use = fmaxf(m[rb], -3.4e38f);   // nothing attended yet: every p below is exp2(-inf)
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = fast_exp2(__builtin_fmaf(x[j], a.scale, -m_use));
        pf[rb] = u32x4{O::pack(p[0], p[1]), O::pack(p[2], p[3]), O::pack(p[4], p[5]), O::pack(p[6], p[7])};
      }
      fetch_mask(u, i + WAVES);
      // output tiles, two dims at a time: pairs of (dim, dim + 1) of one key -> pairs of keys of one dim
      uint32_t w[8][kCols / 2];
#pragma unroll
      for (int j = 0; j < 8; ++j) convert<T, BITS, kCols / 2>(u.v[j], __uint_as_float(u.vs[j] << 23), w[j]);
      fetch_v(u, std::false_type{});
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) l[rb] = O::mfma(ones, pf[rb], l[rb]);
#pragma unroll
      for (int d = 0; d < kCols / 2; ++d) {
        u32x4 even, odd;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          even[j] = __builtin_amdgcn_perm(w[2 * j + 1][d], w[2 * j][d], 0x05040100u);
          odd[j] = __builtin_amdgcn_perm(w[2 * j + 1][d], w[2 * j][d], 0x07060302u);
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          o[rb][2 * d] = O::mfma(even, pf[rb], o[rb][2 * d]);
          o[rb][2 * d + 1] = O::mfma(odd, pf[rb], o[rb][2 * d + 1]);
        }
      }
    }
  };
  const uint32_t k_start = k_off, ks_start = ks_off, v_start = v_off, vs_start = vs_off;
  sweep(std::false_type{});
  // A NaN in the output comes from one that somebody attends to, or from a NaN block of V under a masked
  // key (0 * NaN): the wave goes over its keys once more and keeps the two apart.
  bool odd_row = false;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int j = 0; j < kCols; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) odd_row = odd_row || o[rb][j][e] != o[rb][j][e];
  if (__builtin_expect(__ballot(odd_row) != 0, 0)) {
    k_off = k_start; ks_off = ks_start; v_off = v_start; vs_off = vs_start;
    sweep(std::true_type{});
  }

  // merge the waves, 16 rows at a time
  constexpr int kThreads = WAVES * 64, kQuads = D / 4;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const float lsum = l[rb][0];
    if (rb > 0) __syncthreads();
    float* dst = s_o + (wave * 16 + col) * kPitch + 4 * kCols * grp;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int j = 0; j < kCols; j += 4)
        *reinterpret_cast<f32x4*>(dst + kCols * i + j) = f32x4{o[rb][j][i], o[rb][j + 1][i], o[rb][j + 2][i], o[rb][j + 3][i]};
    }
    if (grp == 0) { s_ml[(wave * 16 + col) * 2] = m[rb]; s_ml[(wave * 16 + col) * 2 + 1] = lsum; }
    __syncthreads();
    for (int e = tid; e < 16 * kQuads; e += kThreads) {
      const int rr = e / kQuads, dq = (e - rr * kQuads) * 4;
      const int r = row0 + 16 * rb + rr;
      if (r >= t.rows) continue;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) top = fmaxf(top, s_ml[(w * 16 + rr) * 2]);
      const float m_use = fmaxf(top, -3.4e38f);
      float sum = 0.f;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const float f = fast_exp2(s_ml[(w * 16 + rr) * 2] - m_use);  // a wave without keys: exp2(-inf)
        sum += f * s_ml[(w * 16 + rr) * 2 + 1];
        acc += f * *reinterpret_cast<const f32x4*>(s_o + (w * 16 + rr) * kPitch + dq);
      }
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
    }
  }
}

// Joins the pieces of rows whose keys were cut: one thread per four dims of a row, pieces in order.
constexpr int kMergeThreads = 256;
template <typename T>
__global__ __launch_bounds__(kMergeThreads) void attn_quant_merge_kernel(QuantArgs a, int rows_per_tile) {
  using O = Ops<T>;
  const int hk = blockIdx.y, b = blockIdx.z;
  const int quads = a.D / 4;
  const int64_t e = (int64_t)blockIdx.x * kMergeThreads + threadIdx.x;
  const int64_t r64 = e / quads;
  const int dq = (int)(e - r64 * quads) * 4;
  if (r64 >= (int64_t)a.n_q * a.group) return;
  const int r = (int)r64;
  const Tile t = tile_of(a, b, r / rows_per_tile * rows_per_tile, rows_per_tile);
  if (r >= t.rows || t.n_pieces == 1) return;
  float top = -INFINITY, sum = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int p = 0; p < t.n_pieces; ++p) {
    const int64_t pr = (((int64_t)b * a.Hkv + hk) * a.max_pieces + p) * ((int64_t)a.n_q * a.group) + r;
    const float m = a.part_ml[2 * pr], l = a.part_ml[2 * pr + 1];
    const f32x4 o = *reinterpret_cast<const f32x4*>(a.part_o + pr * a.D + dq);
    const float up = fmaxf(top, m), m_use = fmaxf(up, -3.4e38f);
    const float f0 = fast_exp2(top - m_use), f1 = fast_exp2(m - m_use);
    sum = f0 * sum + f1 * l;
    acc = f0 * acc + f1 * o;
    top = up;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int qi = r / a.group, h = hk * a.group + (r - qi * a.group);
  T* op = reinterpret_cast<T*>(a.out) + t.o_off + (int64_t)h * a.o_sh + (int64_t)qi * a.o_ss + dq;
  const u32x2 w = {O::pack(acc[0] * inv, acc[1] * inv), O::pack(acc[2] * inv, acc[3] * inv)};
  *reinterpret_cast<u32x2*>(op) = w;
}

// ---------------------------------------------------------------------------------------------
// Generic kernel: one workgroup per (query, head, batch row); keys in chunks of 256.
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
constexpr int kSpanThreads = 256;
__global__ __launch_bounds__(kSpanThreads) void attn_spans_kernel(const uint64_t* __restrict__ bits, int n_q, int words,
                                                                  int kv_len, int32_t* __restrict__ spans) {
  __shared__ int s_lo[kSpanThreads / 64], s_hi[kSpanThreads / 64];
  const int b = blockIdx.y, q0 = blockIdx.x * kSpanQueries;
  const int nq = n_q - q0 < kSpanQueries ? n_q - q0 : kSpanQueries;
  const uint64_t* w = bits + ((int64_t)b * n_q + q0) * words;
  int lo = kv_len, hi = 0;
  for (int64_t i = threadIdx.x; i < (int64_t)nq * words; i += kSpanThreads) {
    const uint64_t x = w[i];
    if (x == 0) continue;
    const int key0 = (int)(i % words) * 64;
    const int f = key0 + __ffsll((unsigned long long)x) - 1, e = key0 + 64 - __clzll((long long)x);
    lo = f < lo ? f : lo;
    hi = e > hi ? e : hi;
  }
  for (int off = 32; off > 0; off >>= 1) {
    const int l2 = __shfl_xor(lo, off), h2 = __shfl_xor(hi, off);
    lo = l2 < lo ? l2 : lo;
    hi = h2 > hi ? h2 : hi;
  }
  if ((threadIdx.x & 63) == 0) { s_lo[threadIdx.x >> 6] = lo; s_hi[threadIdx.x >> 6] = hi; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kSpanThreads / 64; ++i) {
      lo = s_lo[i] < lo ? s_lo[i] : lo;
      hi = s_hi[i] > hi ? s_hi[i] : hi;
    }
    int32_t* out = spans + 2 * ((int64_t)b * gridDim.x + blockIdx.x);
    out[0] = lo;
    out[1] = hi < kv_len ? hi : kv_len;
  }
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
constexpr int kComputeUnits = 256;

// The launch of a shape: row blocks of a tile and how the keys are cut.
struct Shape { int row_blocks, tiles, piece, max_pieces; };
Shape shape_of(int batch, int n_heads, int n_kv_heads, int n_q, int kv_len) {
  Shape s;
  const int64_t rows = (int64_t)n_q * (n_heads / n_kv_heads);
  s.row_blocks = rows <= 16 ? 1 : 2;
  s.tiles = (int)rd::ceil_div(rows, 16 * s.row_blocks);
  const int waves = s.row_blocks == 1 ? 8 : 4;
  // enough pieces that every compute unit has two workgroups, none shorter than four units per wave
  const int64_t groups = (int64_t)batch * n_kv_heads * s.tiles;
  const int step = waves * kUnit;
  int64_t pieces = groups >= 2 * kComputeUnits ? 1 : 2 * kComputeUnits / groups;
  const int64_t most = rd::ceil_div(kv_len, 4 * step);
  if (pieces > most) pieces = most;
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
  switch (s.row_blocks) {
    case 1: hipLaunchKernelGGL((attn_quant_kernel<T, BITS, D, 1, 8>), grid, dim3(512), 0, stream, a); break;
    default: hipLaunchKernelGGL((attn_quant_kernel<T, BITS, D, 2, 4>), grid, dim3(256), 0, stream, a); break;
  }
}

}  // namespace

extern "C" size_t rd_attn_spans_ints(int batch, int n_q) {
  return batch > 0 && n_q > 0 ? 2 * (size_t)batch * rd::ceil_div(n_q, kSpanQueries) : 0;
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

extern "C" size_t rd_verify_attention_quant_workspace_bytes(int dtype, int batch, int n_heads, int n_kv_heads, int n_q,
                                                            int kv_len, int head_dim) {
  if (batch <= 0 || n_heads <= 0 || n_kv_heads <= 0 || n_q <= 0 || kv_len <= 0 || n_heads % n_kv_heads != 0 ||
      !mfma_shape(dtype, head_dim)) return 0;
  const Shape s = shape_of(batch, n_heads, n_kv_heads, n_q, kv_len);
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
  RD_REQUIRE(scale > 0.f && scale <= 3.402823466e38f, RD_EINVAL, "%s: scale %g is not a positive finite number", who, (double)scale);
  auto al = [](const void* p, int n) { return ((uintptr_t)p & (n - 1)) == 0; };
  RD_REQUIRE(al(k_cache, 16) && al(v_cache, 16), RD_EINVAL, "%s: the cache must be 16-byte aligned", who);
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
  a.max_pieces = 1; a.piece = (int)(rd::ceil_div((int64_t)kv_len + kUnit - 1, kUnit) * kUnit);
  a.scale = scale; a.inv_scale = 1.f;
  hipStream_t s = rd::as_stream(stream);
  auto whole = [](const int64_t* st, int m) { return st[0] % m == 0 && st[1] % m == 0 && st[2] % m == 0; };
  const bool mfma = !force_generic && mfma_shape(dtype, head_dim) && al(q, 16) && al(out, 8) && whole(q_strides, 8) && whole(o_strides, 4);
  if (mfma) {
    const Shape sh = shape_of(batch, n_heads, n_kv_heads, n_q, kv_len);
    RD_REQUIRE((int64_t)batch * sh.max_pieces <= 65535 && (int64_t)n_kv_heads * sh.tiles <= 2147483647LL, RD_ELIMIT,
               "%s: grid too large", who);
    a.max_pieces = sh.max_pieces; a.piece = sh.piece;
    a.scale = scale * 1.4426950408889634f;
    a.inv_scale = 1.f / a.scale;
    const int group_rows = 16 * sh.row_blocks;
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
        const int64_t n = (int64_t)n_q * a.group * (head_dim / 4);
        hipLaunchKernelGGL(attn_quant_merge_kernel<T>, dim3((unsigned)rd::ceil_div(n, kMergeThreads), n_kv_heads, batch),
                           dim3(kMergeThreads), 0, s, a, group_rows);
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
