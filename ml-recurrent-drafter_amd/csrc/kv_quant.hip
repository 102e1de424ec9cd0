// Writing and reading the rows of a KV cache held in 4 or 8 bits (gfx950; kv_quant.h has the format).
//   rope_append_quant_kernel  rotation of the new q and k, rows of k and v into the cache's records
//   kv_quantize_kernel        rows into records, without a rotation
//   kv_dequantize_kernel      records back into rows of the model's type
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <type_traits>

#include "kv_quant.h"
#include "rd_common.h"

namespace {

using namespace rd::kvq;

constexpr int kThreads = 256;

typedef short i16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <typename T> struct Elem;
template <> struct Elem<float> {
  static constexpr bool kF16 = false;
  static constexpr float kMax = 3.402823466e38f;
  static __device__ float load(float v) { return v; }
  static __device__ float store(float v) { return v; }
};
template <> struct Elem<__hip_bfloat16> {
  static constexpr bool kF16 = false;
  static constexpr float kMax = 3.3895313892515355e38f;
  static __device__ float load(__hip_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __hip_bfloat16 store(float v) { return __float2bfloat16(v); }
};
template <> struct Elem<__half> {
  static constexpr bool kF16 = true;
  static constexpr float kMax = 65504.f;
  static __device__ float load(__half v) { return __half2float(v); }
  static __device__ __half store(float v) { return __float2half(v); }
};

// eight values of a row
template <typename T>
struct alignas(16) Vec8 {
  T v[kBlock];
};

// Float with the sticky last bit of x: exact values stay, others become the neighbour whose last
// bit is set.  Comparing it with, or rounding it to, anything of fewer bits decides as x itself
// would: a plain rounding to float could land on the border between two codes and take the wrong side.
__device__ inline float sticky_float(double x) {
  uint64_t u = __builtin_bit_cast(uint64_t, x);
  uint32_t lo = (uint32_t)u;
  const uint32_t rest = lo & 0x1fffffffu;  // the 29 bits a float has no room for
  lo = (lo & 0xe0000000u) | (rest != 0 ? 0x20000000u : 0u);
  u = (u & 0xffffffff00000000ull) | lo;
  return (float)__builtin_bit_cast(double, u);
}

// One block of eight values: its codes (one dword, or two) and its scale byte.
template <int BITS>
struct Block {
  uint32_t code[BITS / 4];
  uint32_t scale;
};

template <int BITS, typename T>
__device__ inline Block<BITS> encode(const float (&x)[kBlock]) {
  float amax = 0.f;
  bool ok = true;
#pragma unroll
  for (int i = 0; i < kBlock; ++i) {
    amax = fmaxf(amax, fabsf(x[i]));
    ok = ok && fabsf(x[i]) <= Elem<T>::kMax;  // (false for a NaN)
  }
  const int e = scale_of(__float_as_uint(amax), BITS, Elem<T>::kF16);
  const float s = __uint_as_float((uint32_t)e << 23);
  Block<BITS> b;
  if constexpr (BITS == 4) {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], s, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], s, 3);
    b.code[0] = ok ? c : 0u;
  } else {
    // (the conversion turns what rounds above 448 into NaN)
    const float top = 448.f * s;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = fminf(fmaxf(x[4 * i + j], -top), top);
      i16x2 c = {0, 0};
      c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, y[0], y[1], s, false);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, y[2], y[3], s, true);
      b.code[i] = ok ? __builtin_bit_cast(uint32_t, c) : 0u;
    }
  }
  b.scale = ok ? (uint32_t)e : (uint32_t)kNanScale;
  return b;
}

// block `blk` of the record at `rec`
template <int BITS>
__device__ inline void put_block(char* rec, int dim, int blk, const Block<BITS>& b) {
  if constexpr (BITS == 4) {
    *reinterpret_cast<uint32_t*>(rec + 4 * blk) = b.code[0];
  } else {
    const u32x2 c = {b.code[0], b.code[1]};
    *reinterpret_cast<u32x2*>(rec + 8 * blk) = c;
  }
  reinterpret_cast<uint8_t*>(rec)[code_bytes(BITS, dim) + blk] = (uint8_t)b.scale;
}

struct AppendArgs {
  const void* q; const void* k; const void* v;  // (B, n, heads, D), head_dim contiguous
  int64_t q_sb, q_st, k_sb, k_st, v_sb, v_st;   // element strides of batch and token; head stride D
  const void* cos; const void* sin;             // (table_rows, D)
  int64_t table_rows;
  const int64_t* position_ids; int64_t pos_sb;  // (B, n)
  void* q_out; int64_t qo_sb, qo_st;            // (B, n, heads, D); may be q itself
  char* k_cache; char* v_cache;                 // records, byte strides
  int64_t c_sb, c_sh, c_st;
  int64_t row0, max_len;
  const int32_t* kv_shift;                      // per batch row, or null (rd_rope_append has the same two)
  const int32_t* row_start;
  int n_new, n_heads, n_kv_heads, head_dim;
};

// One task per thread; grid (token, batch row, tasks of a token).  A rotation task covers one block of the
// first half of a head and its partner in the second half, a copy task one block of v.  Bound by memory: 920
// tokens of 32 heads of 128 (34 MB, 6.7 us at the rate of a large copy) 10.4 us, of which 3 are what one token
// takes; 10.9 us with a workgroup for all tasks of a token.
template <typename T, int BITS>
__global__ __launch_bounds__(kThreads) void rope_append_quant_kernel(AppendArgs a) {
#pragma clang fp contract(off)
  using V = Vec8<T>;
  const int t = blockIdx.x, b = blockIdx.y;
  const int D = a.head_dim, half = D / 2;
  const int per_head = half / kBlock;
  const int q_tasks = a.n_heads * per_head, k_tasks = a.n_kv_heads * per_head;
  const int v_tasks = a.n_kv_heads * (D / kBlock);
  int64_t pos = a.position_ids[b * a.pos_sb + t];
  pos = pos < 0 ? 0 : (pos >= a.table_rows ? a.table_rows - 1 : pos);  // never read outside the table
  const T* cos_row = reinterpret_cast<const T*>(a.cos) + pos * D;
  const T* sin_row = reinterpret_cast<const T*>(a.sin) + pos * D;
  int64_t tok = t, in_batch = b;  // token row within the batch row's rows, and which batch row
  if (a.row_start != nullptr) {
    const int r0 = a.row_start[b];
    if (t >= a.row_start[b + 1] - r0) return;
    tok = (int64_t)r0 + t;
    in_batch = 0;
  }
  const T* q_tok = reinterpret_cast<const T*>(a.q) + in_batch * a.q_sb + tok * a.q_st;
  const T* k_tok = reinterpret_cast<const T*>(a.k) + in_batch * a.k_sb + tok * a.k_st;
  const T* v_tok = reinterpret_cast<const T*>(a.v) + in_batch * a.v_sb + tok * a.v_st;
  T* qo_tok = reinterpret_cast<T*>(a.q_out) + in_batch * a.qo_sb + tok * a.qo_st;
  int64_t cache_row = a.row0 + t - (a.kv_shift ? a.kv_shift[b] : 0);
  // a shift that leaves the slab is never followed: q is still rotated, k and v are dropped
  const bool in_cache = cache_row >= 0 && cache_row < a.max_len;
  cache_row = in_cache ? cache_row : 0;
  char* kc = a.k_cache + b * a.c_sb + cache_row * a.c_st;
  char* vc = a.v_cache + b * a.c_sb + cache_row * a.c_st;
  const int n_tasks = in_cache ? q_tasks + k_tasks + v_tasks : q_tasks;

  const int task = blockIdx.z * kThreads + threadIdx.x;
  if (task < n_tasks) {
    if (task >= q_tasks + k_tasks) {
      const int c = task - q_tasks - k_tasks;
      const int h = c / (D / kBlock), blk = c % (D / kBlock);
      const V x = *reinterpret_cast<const V*>(v_tok + (int64_t)h * D + blk * kBlock);
      float f[kBlock];
#pragma unroll
      for (int e = 0; e < kBlock; ++e) f[e] = Elem<T>::load(x.v[e]);
      put_block<BITS>(vc + h * a.c_sh, D, blk, encode<BITS, T>(f));
      return;
    }
    const bool is_q = task < q_tasks;
    const int c = is_q ? task : task - q_tasks;
    const int h = c / per_head, blk = c % per_head, d = blk * kBlock;
    const T* src = (is_q ? q_tok : k_tok) + (int64_t)h * D;
    const V x1 = *reinterpret_cast<const V*>(src + d);
    const V x2 = *reinterpret_cast<const V*>(src + half + d);
    const V c1 = *reinterpret_cast<const V*>(cos_row + d), c2 = *reinterpret_cast<const V*>(cos_row + half + d);
    const V s1 = *reinterpret_cast<const V*>(sin_row + d), s2 = *reinterpret_cast<const V*>(sin_row + half + d);
    if (is_q) {
      // products of two 16-bit numbers are exact in fp32, so the sum is the only rounding before
      // the one to T
      V o1, o2;
#pragma unroll
      for (int e = 0; e < kBlock; ++e) {
        const float a1 = Elem<T>::load(x1.v[e]), a2 = Elem<T>::load(x2.v[e]);
        o1.v[e] = Elem<T>::store(a1 * Elem<T>::load(c1.v[e]) - a2 * Elem<T>::load(s1.v[e]));
        o2.v[e] = Elem<T>::store(a2 * Elem<T>::load(c2.v[e]) + a1 * Elem<T>::load(s2.v[e]));
      }
      T* dst = qo_tok + (int64_t)h * D;
      *reinterpret_cast<V*>(dst + d) = o1;
      *reinterpret_cast<V*>(dst + half + d) = o2;
    } else {
      // fp64, then a sticky bit: the codes are those of the rotated key as fp64 holds it.  The products are
      // exact; their sum is, too, unless the terms lie more than 2^37 (bf16; fp16: 2^31, fp32: 2^5) apart: it is then
      // rounded to 53 bits, and takes another code only where it lies within 2^-53 of a border beside it.  (The
      // sum's error by two-sum would settle that: 16 x 162 tokens of 40 heads 31.8 -> 38.5 us.  A key rounded to
      // T first, as a 16-bit cache would hold it, lands in another code about once in 2^6 values at 4 bits.)
      float o1[kBlock], o2[kBlock];
#pragma unroll
      for (int e = 0; e < kBlock; ++e) {
        const double a1 = Elem<T>::load(x1.v[e]), a2 = Elem<T>::load(x2.v[e]);
        o1[e] = sticky_float(a1 * (double)Elem<T>::load(c1.v[e]) - a2 * (double)Elem<T>::load(s1.v[e]));
        o2[e] = sticky_float(a2 * (double)Elem<T>::load(c2.v[e]) + a1 * (double)Elem<T>::load(s2.v[e]));
      }
      char* rec = kc + h * a.c_sh;
      put_block<BITS>(rec, D, blk, encode<BITS, T>(o1));
      put_block<BITS>(rec, D, blk + per_head, encode<BITS, T>(o2));
    }
  }
}

struct RowsArgs {
  const void* x; int64_t x_sb, x_sh, x_st;  // rows of the model's type, element strides {batch, head, row}
  char* cache; int64_t c_sb, c_sh, c_st;    // records, byte strides
  int64_t n_rows;
  int dim;
};

// One block per thread; grid (rows and blocks, head, batch row).  Values may lie on any element boundary, and
// are loaded one by one.  2548 rows of 8 x 32 heads of 128 into 4 bits (219 MB): 44.6 us with three sets of inputs in
// turn, 4.9 TB/s, near the rate of a large copy (33 us where part of the values is in the last-level cache); so is
// memory the bound here too.
template <typename T, int BITS>
__global__ __launch_bounds__(kThreads) void kv_quantize_kernel(RowsArgs a) {
  const int per_row = a.dim / kBlock;
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= a.n_rows * per_row) return;
  const int64_t row = i / per_row;
  const int blk = (int)(i - row * per_row);
  const T* src = reinterpret_cast<const T*>(a.x) + blockIdx.z * a.x_sb + blockIdx.y * a.x_sh + row * a.x_st;
  float f[kBlock];
#pragma unroll
  for (int e = 0; e < kBlock; ++e) f[e] = Elem<T>::load(src[blk * kBlock + e]);
  put_block<BITS>(a.cache + blockIdx.z * a.c_sb + blockIdx.y * a.c_sh + row * a.c_st, a.dim, blk, encode<BITS, T>(f));
}

// eight values of a block
template <typename T, int BITS>
__device__ inline Vec8<T> decode(const uint32_t (&code)[BITS / 4], uint32_t scale) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const float s = __uint_as_float(scale << 23);
  f32x2 p[4];
  if constexpr (BITS == 4) {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[0], s, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[0], s, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[0], s, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[0], s, 3);
  } else {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(code[0], s, false);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(code[0], s, true);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(code[1], s, false);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(code[1], s, true);
  }
  Vec8<T> out;
#pragma unroll
  for (int e = 0; e < kBlock; ++e) out.v[e] = Elem<T>::store(p[e / 2][e % 2]);
  return out;
}

// One block per thread, 16 bytes of 16-bit values at a time.  Bound by memory: 2548 rows of 8 x 32 heads of 128 from 4
// bits (219 MB) 42 us, 5.2 TB/s, the rate of a large copy.
template <typename T, int BITS>
__global__ __launch_bounds__(kThreads) void kv_dequantize_kernel(RowsArgs a) {
  const int per_row = a.dim / kBlock;
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= a.n_rows * per_row) return;
  const int64_t row = i / per_row;
  const int blk = (int)(i - row * per_row);
  const char* rec = a.cache + blockIdx.z * a.c_sb + blockIdx.y * a.c_sh + row * a.c_st;
  uint32_t code[BITS / 4];
#pragma unroll
  for (int w = 0; w < BITS / 4; ++w) code[w] = reinterpret_cast<const uint32_t*>(rec + BITS * blk)[w];
  const uint32_t scale = reinterpret_cast<const uint8_t*>(rec)[code_bytes(BITS, a.dim) + blk];
  T* dst = reinterpret_cast<T*>(const_cast<void*>(a.x)) + blockIdx.z * a.x_sb + blockIdx.y * a.x_sh + row * a.x_st;
  *reinterpret_cast<Vec8<T>*>(dst + blk * kBlock) = decode<T, BITS>(code, scale);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_format(const char* who, int dtype, int bits, int head_dim) {
  RD_REQUIRE(dtype == RD_F32 || dtype == RD_BF16 || dtype == RD_F16, RD_EINVAL, "%s: unknown dtype %d", who, dtype);
  RD_REQUIRE(known_bits(bits), RD_EINVAL, "%s: bits %d (4 or 8)", who, bits);
  RD_REQUIRE(known_dim(head_dim), RD_ELIMIT, "%s: head_dim %d must be a multiple of 32, at most %d", who, head_dim, kMaxDim);
  return RD_OK;
}
int check_cache_strides(const char* who, const int64_t* s, int bits, int head_dim) {
  RD_REQUIRE(s[0] % 16 == 0 && s[1] % 16 == 0 && s[2] % 16 == 0 && s[0] >= 0 && s[1] >= 0 &&
                 s[2] >= record_bytes(bits, head_dim), RD_EINVAL,
             "%s: cache strides must be multiples of 16 bytes, rows at least %d bytes apart", who,
             record_bytes(bits, head_dim));
  return RD_OK;
}

// f(T{}, std::integral_constant<int, BITS>) for the dtype and the bits
template <typename F>
void dispatch(int dtype, int bits, F&& f) {
  auto with_bits = [&](auto zero) {
    if (bits == 4) f(zero, std::integral_constant<int, 4>{});
    else f(zero, std::integral_constant<int, 8>{});
  };
  switch (dtype) {
    case RD_F32: with_bits(float{}); break;
    case RD_BF16: with_bits(__hip_bfloat16{}); break;
    default: with_bits(__half{}); break;
  }
}

}  // namespace

extern "C" size_t rd_kv_quant_row_bytes(int bits, int head_dim) {
  return known_bits(bits) && known_dim(head_dim) ? (size_t)record_bytes(bits, head_dim) : 0;
}

extern "C" int rd_rope_append_quant(const void* q, const int64_t* q_strides, const void* k,
                                    const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                    int dtype, int batch, int n_new, int n_heads, int n_kv_heads,
                                    int head_dim, const void* cos, const void* sin, int64_t table_rows,
                                    const int64_t* position_ids, int64_t pos_batch_stride, void* q_out,
                                    const int64_t* q_out_strides, void* k_cache, void* v_cache,
                                    const int64_t* cache_strides, int bits, int64_t row0, int64_t max_len,
                                    const int32_t* row_start, const int32_t* kv_row_shift, void* stream) {
  const char* who = "rd_rope_append_quant";
  RD_REQUIRE(batch > 0 && n_new > 0 && n_heads > 0 && n_kv_heads > 0, RD_EINVAL,
             "%s: bad sizes (batch %d n_new %d heads %d kv_heads %d)", who, batch, n_new, n_heads, n_kv_heads);
  RD_REQUIRE(batch <= 65535, RD_ELIMIT, "%s: batch %d > 65535", who, batch);
  if (const int rc = check_format(who, dtype, bits, head_dim)) return rc;
  const int64_t tasks = ((int64_t)n_heads + 3 * (int64_t)n_kv_heads) * (head_dim / kBlock / 2);
  RD_REQUIRE(tasks <= 65535LL * kThreads, RD_ELIMIT, "%s: too many heads (%d + 2 * %d)", who, n_heads, n_kv_heads);
  RD_REQUIRE(q && k && v && cos && sin && position_ids && q_out && k_cache && v_cache && q_strides && k_strides &&
                 v_strides && q_out_strides && cache_strides, RD_EINVAL, "%s: null pointer", who);
  RD_REQUIRE(table_rows > 0, RD_EINVAL, "%s: empty cos/sin table", who);
  RD_REQUIRE(row0 >= 0 && n_new <= max_len && row0 <= max_len - n_new, RD_EINVAL,
             "%s: %d rows from %lld do not fit max_len %lld", who, n_new, (long long)row0, (long long)max_len);
  RD_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(cos) && aligned16(sin) && aligned16(q_out) &&
                 aligned16(k_cache) && aligned16(v_cache), RD_EINVAL, "%s: pointers must be 16-byte aligned", who);
  for (const int64_t* s : {q_strides, k_strides, v_strides, q_out_strides})
    RD_REQUIRE(s[0] % kBlock == 0 && s[1] % kBlock == 0 && s[0] >= 0 && s[1] >= 0, RD_EINVAL,
               "%s: token and batch strides must be non-negative multiples of %d elements", who, kBlock);
  if (const int rc = check_cache_strides(who, cache_strides, bits, head_dim)) return rc;
  AppendArgs a;
  a.q = q; a.k = k; a.v = v;
  a.q_sb = q_strides[0]; a.q_st = q_strides[1];
  a.k_sb = k_strides[0]; a.k_st = k_strides[1];
  a.v_sb = v_strides[0]; a.v_st = v_strides[1];
  a.cos = cos; a.sin = sin; a.table_rows = table_rows;
  a.position_ids = position_ids; a.pos_sb = pos_batch_stride;
  a.q_out = q_out; a.qo_sb = q_out_strides[0]; a.qo_st = q_out_strides[1];
  a.k_cache = reinterpret_cast<char*>(k_cache); a.v_cache = reinterpret_cast<char*>(v_cache);
  a.c_sb = cache_strides[0]; a.c_sh = cache_strides[1]; a.c_st = cache_strides[2];
  a.row0 = row0; a.max_len = max_len;
  a.kv_shift = kv_row_shift; a.row_start = row_start;
  a.n_new = n_new; a.n_heads = n_heads; a.n_kv_heads = n_kv_heads; a.head_dim = head_dim;
  hipStream_t s = rd::as_stream(stream);
  {
    rd::ScopedTiming rd_t("rope_append_quant_kernel", s);
    dispatch(dtype, bits, [&](auto zero, auto bits_c) {
      using T = decltype(zero);
      hipLaunchKernelGGL((rope_append_quant_kernel<T, decltype(bits_c)::value>), dim3(n_new, batch, (unsigned)rd::ceil_div(tasks, kThreads)),
                         dim3(kThreads), 0, s, a);
    });
  }
  return rd::check_launch(who);
}

namespace {

// what rd_kv_quantize and rd_kv_dequantize have in common
int check_rows(const char* who, const void* x, const int64_t* x_strides, int dtype, int batch, int n_kv_heads,
               int64_t n_rows, int head_dim, int bits, const void* cache, const int64_t* cache_strides, int64_t row0,
               int64_t max_len, int x_align, RowsArgs* a, dim3* grid) {
  RD_REQUIRE(batch > 0 && n_kv_heads > 0 && n_rows > 0, RD_EINVAL, "%s: bad sizes (batch %d kv_heads %d rows %lld)",
             who, batch, n_kv_heads, (long long)n_rows);
  RD_REQUIRE(batch <= 65535 && n_kv_heads <= 65535, RD_ELIMIT, "%s: batch/kv_heads > 65535", who);
  if (const int rc = check_format(who, dtype, bits, head_dim)) return rc;
  RD_REQUIRE(x && x_strides && cache && cache_strides, RD_EINVAL, "%s: null pointer", who);
  RD_REQUIRE(row0 >= 0 && n_rows <= max_len && row0 <= max_len - n_rows, RD_EINVAL,
             "%s: %lld rows from %lld do not fit max_len %lld", who, (long long)n_rows, (long long)row0, (long long)max_len);
  RD_REQUIRE(aligned16(cache), RD_EINVAL, "%s: the cache must be 16-byte aligned", who);
  if (const int rc = check_cache_strides(who, cache_strides, bits, head_dim)) return rc;
  if (x_align > 1)
    RD_REQUIRE(aligned16(x) && x_strides[0] % x_align == 0 && x_strides[1] % x_align == 0 && x_strides[2] % x_align == 0,
               RD_EINVAL, "%s: rows must start on multiples of %d elements of a 16-byte aligned buffer", who, x_align);
  const int64_t blocks = n_rows * (head_dim / kBlock);
  RD_REQUIRE(rd::ceil_div(blocks, kThreads) <= 2147483647LL, RD_ELIMIT, "%s: %lld rows are too many", who, (long long)n_rows);
  *a = {x, x_strides[0], x_strides[1], x_strides[2],
        reinterpret_cast<char*>(const_cast<void*>(cache)) + row0 * cache_strides[2],
        cache_strides[0], cache_strides[1], cache_strides[2], n_rows, head_dim};
  *grid = dim3((unsigned)rd::ceil_div(blocks, kThreads), n_kv_heads, batch);
  return RD_OK;
}

}  // namespace

extern "C" int rd_kv_quantize(const void* x, const int64_t* x_strides, int dtype, int batch, int n_kv_heads,
                              int64_t n_rows, int head_dim, int bits, void* cache, const int64_t* cache_strides,
                              int64_t row0, int64_t max_len, void* stream) {
  RowsArgs a;
  dim3 grid;
  if (const int rc = check_rows("rd_kv_quantize", x, x_strides, dtype, batch, n_kv_heads, n_rows, head_dim, bits, cache,
                                cache_strides, row0, max_len, 1, &a, &grid)) return rc;
  hipStream_t s = rd::as_stream(stream);
  {
    rd::ScopedTiming rd_t("kv_quantize_kernel", s);
    dispatch(dtype, bits, [&](auto zero, auto bits_c) {
      hipLaunchKernelGGL((kv_quantize_kernel<decltype(zero), decltype(bits_c)::value>), grid, dim3(kThreads), 0, s, a);
    });
  }
  return rd::check_launch("rd_kv_quantize");
}

extern "C" int rd_kv_dequantize(const void* cache, const int64_t* cache_strides, int bits, int dtype, int batch,
                                int n_kv_heads, int64_t row0, int64_t n_rows, int head_dim, int64_t max_len, void* out,
                                const int64_t* out_strides, void* stream) {
  RowsArgs a;
  dim3 grid;
  if (const int rc = check_rows("rd_kv_dequantize", out, out_strides, dtype, batch, n_kv_heads, n_rows, head_dim, bits,
                                cache, cache_strides, row0, max_len, kBlock, &a, &grid)) return rc;
  hipStream_t s = rd::as_stream(stream);
  {
    rd::ScopedTiming rd_t("kv_dequantize_kernel", s);
    dispatch(dtype, bits, [&](auto zero, auto bits_c) {
      hipLaunchKernelGGL((kv_dequantize_kernel<decltype(zero), decltype(bits_c)::value>), grid, dim3(kThreads), 0, s, a);
    });
  }
  return rd::check_launch("rd_kv_dequantize");
}
