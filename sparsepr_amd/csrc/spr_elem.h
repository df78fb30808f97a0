// Elements of the three float types as the elementwise kernels take them: dtype codes 0 bfloat16,
// 1 float16, 2 float32, computed in fp32.
#pragma once

#include "spr_common.h"

namespace spr {

template <int DT>
struct Elem;
template <>
struct Elem<0> {  // bf16
  using S = uint16_t;
  __device__ static float to_f(S s) { return bf16_to_f32(s); }
  __device__ static S from_f(float f) { return f32_to_bf16(f); }
};
template <>
struct Elem<1> {  // fp16
  using S = uint16_t;
  __device__ static float to_f(S s) { return static_cast<float>(__builtin_bit_cast(_Float16, s)); }
  __device__ static S from_f(float f) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f)); }
};
template <>
struct Elem<2> {  // fp32
  using S = float;
  __device__ static float to_f(S s) { return s; }
  __device__ static S from_f(float f) { return f; }
};

// 8 consecutive elements <-> float[8] (16 bytes for 16-bit types, 32 for fp32).
template <int DT>
__device__ __forceinline__ void load8(const typename Elem<DT>::S* p, float (&x)[8]) {
  if constexpr (DT == 2) {
    const f32x4 a = reinterpret_cast<const f32x4*>(p)[0];
    const f32x4 b = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = a[e];
      x[e + 4] = b[e];
    }
  } else {
    const u32x4 r = *reinterpret_cast<const u32x4*>(p);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[2 * e] = Elem<DT>::to_f(static_cast<uint16_t>(w[e] & 0xFFFFu));
      x[2 * e + 1] = Elem<DT>::to_f(static_cast<uint16_t>(w[e] >> 16));
    }
  }
}
template <int DT>
__device__ __forceinline__ void store8(typename Elem<DT>::S* p, const float (&x)[8]) {
  if constexpr (DT == 2) {
    reinterpret_cast<f32x4*>(p)[0] = f32x4{x[0], x[1], x[2], x[3]};
    reinterpret_cast<f32x4*>(p)[1] = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = static_cast<uint32_t>(Elem<DT>::from_f(x[2 * e])) |
             (static_cast<uint32_t>(Elem<DT>::from_f(x[2 * e + 1])) << 16);
    }
    *reinterpret_cast<u32x4*>(p) = u32x4{w[0], w[1], w[2], w[3]};
  }
}
template <int DT>
__device__ __forceinline__ void copy8(const typename Elem<DT>::S* src, typename Elem<DT>::S* dst) {
  if constexpr (DT == 2) {
    reinterpret_cast<u32x4*>(dst)[0] = reinterpret_cast<const u32x4*>(src)[0];
    reinterpret_cast<u32x4*>(dst)[1] = reinterpret_cast<const u32x4*>(src)[1];
  } else {
    *reinterpret_cast<u32x4*>(dst) = *reinterpret_cast<const u32x4*>(src);
  }
}
template <int DT>
__device__ __forceinline__ float round_t(float x) {
  return Elem<DT>::to_f(Elem<DT>::from_f(x));
}

// The same from any address that an element may have (global memory takes a 16-byte access at any
// of them; a load that crosses a cache line costs two), and the first n of 8, zeros behind them.
struct Packed16 {
  uint32_t w[4];
};
template <int DT>
__device__ __forceinline__ void load8u(const typename Elem<DT>::S* p, float (&x)[8]) {
  if constexpr (DT == 2) {
    __builtin_memcpy(x, p, 32);
  } else {
    Packed16 r;
    __builtin_memcpy(&r, p, 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[2 * e] = Elem<DT>::to_f(static_cast<uint16_t>(r.w[e] & 0xFFFFu));
      x[2 * e + 1] = Elem<DT>::to_f(static_cast<uint16_t>(r.w[e] >> 16));
    }
  }
}
template <int DT>
__device__ __forceinline__ void load8n(const typename Elem<DT>::S* p, int n, float (&x)[8]) {
  if (n >= 8) {
    load8u<DT>(p, x);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = e < n ? Elem<DT>::to_f(p[e]) : 0.0f;
  }
}
template <int DT>
__device__ __forceinline__ void store8n(typename Elem<DT>::S* p, int n, const float (&x)[8]) {
  if (n >= 8) {
    if constexpr (DT == 2) {
      __builtin_memcpy(p, x, 32);
    } else {
      Packed16 r;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        r.w[e] = static_cast<uint32_t>(Elem<DT>::from_f(x[2 * e])) |
                 (static_cast<uint32_t>(Elem<DT>::from_f(x[2 * e + 1])) << 16);
      }
      __builtin_memcpy(p, &r, 16);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = Elem<DT>::from_f(x[e]);
  }
}

// The value at a dtype code known at run time only (one branch that all lanes take together).
__device__ __forceinline__ void load8n_any(const void* p, int dtype, int64_t at, int n, float (&x)[8]) {
  if (dtype == 0) load8n<0>(static_cast<const uint16_t*>(p) + at, n, x);
  else if (dtype == 1) load8n<1>(static_cast<const uint16_t*>(p) + at, n, x);
  else load8n<2>(static_cast<const float*>(p) + at, n, x);
}

// Sum and maximum over the 16 lanes of a DPP row, in every lane: rotations by 8, 4, 2 and 1.
template <int ROT>
__device__ __forceinline__ uint32_t row_rotate(uint32_t x) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int32_t>(x), 0x120 + ROT, 0xf, 0xf, false));
}
__device__ __forceinline__ float row_sum(float x) {
  x += __uint_as_float(row_rotate<8>(__float_as_uint(x)));
  x += __uint_as_float(row_rotate<4>(__float_as_uint(x)));
  x += __uint_as_float(row_rotate<2>(__float_as_uint(x)));
  x += __uint_as_float(row_rotate<1>(__float_as_uint(x)));
  return x;
}
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
  x = max(x, row_rotate<8>(x));
  x = max(x, row_rotate<4>(x));
  x = max(x, row_rotate<2>(x));
  x = max(x, row_rotate<1>(x));
  return x;
}

}  // namespace spr
