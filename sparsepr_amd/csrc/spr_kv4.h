// Layout of a 4-bit K/V cache page, shared by the kernels that write, read, attend and move pages.
//
// pages [num_pages, kv_heads, head_bytes] uint8.  One head's part of a page of S tokens:
//   K codes [S][D / 2], V codes [S][D / 2], K scales [S][D / 32], V scales [S][D / 32]
// A code is a 4-bit float e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), two to a byte, the even dim
// in the low half.  A scale byte b is the power of two 2^(b - 127) of 32 dims of one token, b in
// [2, 252]; a larger byte is a NaN (253 and 254 would pass bf16's range, with infinities that 0 * inf
// brings to rows that do not see the token).  code * scale has two significant bits, so bf16 holds it
// exactly, and one v_cvt_scalef32_pk_bf16_fp4 makes two of them.
#pragma once

#include "spr_common.h"

namespace spr {

constexpr int KV4_GROUP = 32;  // dims that share a scale
// Tokens a row of the block table may stand for: a token's place plus a chunk stays in 32 bits.
constexpr int64_t KV4_MOST_TOKENS = int64_t{1} << 30;

// Bytes of one head's part of a page.
__host__ __device__ __forceinline__ int64_t kv4_head_bytes(int32_t page_size, int32_t d) {
  return static_cast<int64_t>(page_size) * (d + d / 16);
}

inline bool kv4_page_size_ok(int32_t s) { return s >= 32 && s <= 256 && (s & (s - 1)) == 0; }

// Byte offsets inside one head's part, for a page of 1 << log_s tokens.
template <int D>
struct Kv4Part {
  static constexpr int CODE_ROW = D / 2;
  static constexpr int SCALE_ROW = D / KV4_GROUP;
  static __device__ __forceinline__ int32_t v_codes(int log_s) { return CODE_ROW << log_s; }
  static __device__ __forceinline__ int32_t k_scales(int log_s) { return D << log_s; }
  static __device__ __forceinline__ int32_t v_scales(int log_s) { return (D + SCALE_ROW) << log_s; }
};

typedef __bf16 kv4_bf16x2 __attribute__((ext_vector_type(2)));

// Two codes (byte SEL of w) times scale, as packed bf16: exact; a NaN scale gives NaN.
template <int SEL>
__device__ __forceinline__ uint32_t kv4_pair(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
}

// The eight values of a code word, times scale.
__device__ __forceinline__ u32x4 kv4_eight(uint32_t w, float scale) {
  return u32x4{kv4_pair<0>(w, scale), kv4_pair<1>(w, scale), kv4_pair<2>(w, scale), kv4_pair<3>(w, scale)};
}

// Whether a scale byte stands for no number.
__device__ __forceinline__ bool kv4_nan(uint32_t byte) { return byte > 252; }

// A scale byte as the float that the conversions take (exponent 255: not a number).
__device__ __forceinline__ float kv4_scale(uint32_t byte) { return __uint_as_float((kv4_nan(byte) ? 255 : byte) << 23); }

}  // namespace spr
