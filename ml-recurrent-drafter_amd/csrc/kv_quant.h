// Rows of a KV cache held in 4 or 8 bits: the record of a row and the arithmetic of a block.
//
// A row of D values (D a multiple of 32) is cut into blocks of 8 consecutive values.  A block has
// one power of two 2^e and eight codes:
//   4 bits  e2m1 (0 .5 1 1.5 2 3 4 6 and negatives), value d in nibble d % 8 of the block's dword
//   8 bits  e4m3 without infinities (largest 448), value d in byte d % 8
// e is the smallest integer with max |x| <= top * 2^e (top = 7 / 464: what still rounds to the
// largest code), clamped to the range in which every code times 2^e is a number of the cache's type;
// a code is x / 2^e rounded to the nearest, ties to even, saturated.  Power-of-two scales make the
// value exact in bf16, fp16 and fp32, and gfx950 converts two codes and applies the scale in one
// instruction (v_cvt_scalef32_pk_*; the scale operand's sign and mantissa are ignored and the
// exponent field 255 gives NaN for every code: both checked on the machine for all codes).
// Scale byte = e + 127.  255 marks a block that held a NaN, an infinity or a number beyond the type's
// largest finite one; its eight values read back as NaN.
//
// Record of a row: D * bits / 8 code bytes, then D / 8 scale bytes, padded to a multiple of 16 bytes
// (rows stay whole 16-byte units for the row movement kernels).  D = 128: 80 and 144 bytes, where
// bf16 takes 256.  Blocks of 8 instead of 32 cost no bytes there (the scale bytes fill what would be
// padding) and gain 0.5 to 1.7 dB of signal to rounding noise at 4 bits; what they cost is the matrix instructions that
// apply one scale to 32 values, for which queries and weights would have to be rounded to 8 bits or fewer as well.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "attn_addr.h"  // RD_HD

namespace rd {
namespace kvq {

constexpr int kBlock = 8;          // values that share a scale
constexpr int kMaxDim = 256;
constexpr int kNanScale = 255;

RD_HD constexpr int code_bytes(int bits, int dim) { return dim * bits / 8; }
RD_HD constexpr int record_bytes(int bits, int dim) { return (code_bytes(bits, dim) + dim / kBlock + 15) / 16 * 16; }
inline bool known_bits(int bits) { return bits == 4 || bits == 8; }
inline bool known_dim(int dim) { return dim > 0 && dim <= kMaxDim && dim % 32 == 0; }

// largest and smallest biased exponent of a block's scale (f16: true for fp16, else bf16 or fp32)
RD_HD constexpr int scale_max(int bits, bool f16) { return (f16 ? 127 + 15 : 127 + 127) - (bits == 4 ? 2 : 8); }
RD_HD constexpr int scale_min(int bits, bool f16) { return f16 ? 127 - (bits == 4 ? 23 : 15) : 127 - 100; }

// Biased exponent of the scale of a block whose largest magnitude has these float bits: the exponent
// field minus the largest code's exponent, one more where the mantissa lies above top's (7 = 1.75 * 4,
// 464 = 1.8125 * 256): adding all mantissa values above it carries into the exponent.
RD_HD int scale_of(uint32_t amax_bits, int bits, bool f16) {
  const int e = (int)((amax_bits + (bits == 4 ? 0x1fffffu : 0x17ffffu)) >> 23) - (bits == 4 ? 2 : 8);
  const int lo = scale_min(bits, f16), hi = scale_max(bits, f16);
  return e < lo ? lo : (e > hi ? hi : e);
}

}  // namespace kvq
}  // namespace rd
