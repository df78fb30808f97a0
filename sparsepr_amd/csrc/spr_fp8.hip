// Rows to 8 bits and back (spr_fp8.h has the format): along the rows or along the columns, with a
// scale for 128 values or for 128 x 128, the codes laid out along the scaled direction.
//
// Bound by memory: values are read once, 8 a lane, and kept in registers while the group's maximum is
// found.  The transposed codes go through LDS, so that both sides move whole 128-byte lines.  A bf16 weight of
// 13,824 x 5120 to transposed codes (212 MB) takes 44 to 48 us, 4.5 TB/s where a copy has 5.1, and 34 us back;
// 20 x 32 tiles 10 us, a workgroup's load, maximum and store behind one another with 2.5 of them a CU.
#include "spr_fp8.h"

namespace {

using spr::Elem;
using spr::FP8_GROUP;
using spr::load8n;

constexpr int THREADS = 256;

// A scale for 128 values of a row: 16 lanes a group, VECS of them in turn.
template <int DT>
__global__ __launch_bounds__(THREADS) void quantise_rows_kernel(const typename Elem<DT>::S* __restrict__ x, int64_t ld,
                                                               uint32_t rows, int32_t width, uint32_t groups,
                                                               uint8_t* __restrict__ codes,
                                                               uint8_t* __restrict__ scales) {
  const uint64_t g = static_cast<uint64_t>(blockIdx.x) * (THREADS / 16) + threadIdx.x / 16;
  const uint32_t row = static_cast<uint32_t>(g / groups);
  if (row >= rows) return;
  const uint32_t at = static_cast<uint32_t>(g - static_cast<uint64_t>(row) * groups);
  const int c = static_cast<int>(at) * FP8_GROUP + static_cast<int>(threadIdx.x % 16) * 8;
  float v[8];
  load8n<DT>(x + row * ld + c, width - c, v);
  const uint32_t b = spr::fp8_scale_byte(spr::row_max(spr::magnitude_bits8(v)));
  const int64_t wide = spr::fp8_width(width);
  if (c < wide) *reinterpret_cast<uint64_t*>(codes + row * wide + c) = spr::fp8_codes8(v, spr::fp8_inverse_scale(b));
  if (threadIdx.x % 16 == 0) scales[static_cast<int64_t>(row) * groups + at] = static_cast<uint8_t>(b);
}

// One 128 x 128 tile a workgroup: thread t holds 8 columns from 8 (t % 16) of the 8 rows from 8 (t / 16).
// SQUARE: one scale for the tile, else (TRANSPOSE) one for each of its columns.
template <int DT, bool SQUARE, bool TRANSPOSE>
__global__ __launch_bounds__(THREADS) void quantise_tile_kernel(const typename Elem<DT>::S* __restrict__ x, int64_t ld,
                                                               int64_t rows, int32_t width, uint8_t* __restrict__ codes,
                                                               uint8_t* __restrict__ scales) {
  static_assert(SQUARE || TRANSPOSE, "rows of their own scales are quantise_rows_kernel's");
  __shared__ uint32_t tops[4][FP8_GROUP];
  __shared__ alignas(16) uint8_t tile[TRANSPOSE ? FP8_GROUP * FP8_GROUP : 16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int cv = threadIdx.x & 15, rv = threadIdx.x >> 4;
  const int32_t c0 = static_cast<int32_t>(blockIdx.x) * FP8_GROUP;
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * FP8_GROUP;
  const int c = c0 + 8 * cv;
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = r0 + 8 * rv + i;
    load8n<DT>(x + r * ld + c, r < rows ? width - c : 0, v[i]);
  }
  float inv[8];  // of this thread's columns
  if constexpr (SQUARE) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, spr::magnitude_bits8(v[i]));
    top = spr::row_max(top);
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16, 64)));
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32, 64)));
    if (lane == 0) tops[wave][0] = top;
    __syncthreads();
    const uint32_t b = spr::fp8_scale_byte(max(max(tops[0][0], tops[1][0]), max(tops[2][0], tops[3][0])));
    const float f = spr::fp8_inverse_scale(b);
#pragma unroll
    for (int e = 0; e < 8; ++e) inv[e] = f;
    if (threadIdx.x == 0) {
      const int64_t down = TRANSPOSE ? blockIdx.x : blockIdx.y, across = TRANSPOSE ? blockIdx.y : blockIdx.x;
      scales[down * (TRANSPOSE ? gridDim.y : gridDim.x) + across] = static_cast<uint8_t>(b);
    }
  } else {
    uint32_t top[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      top[e] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) top[e] = max(top[e], spr::magnitude_bits(v[i][e]));
      top[e] = max(top[e], static_cast<uint32_t>(__shfl_xor(static_cast<int>(top[e]), 16, 64)));
      top[e] = max(top[e], static_cast<uint32_t>(__shfl_xor(static_cast<int>(top[e]), 32, 64)));
    }
    if (lane < 16) {
#pragma unroll
      for (int e = 0; e < 8; ++e) tops[wave][8 * cv + e] = top[e];
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int j = 8 * cv + e;
      const uint32_t b = spr::fp8_scale_byte(max(max(tops[0][j], tops[1][j]), max(tops[2][j], tops[3][j])));
      inv[e] = spr::fp8_inverse_scale(b);
      if (rv == 0 && c + e < width)
        scales[static_cast<int64_t>(c + e) * gridDim.y + blockIdx.y] = static_cast<uint8_t>(b);
    }
  }
  if constexpr (!TRANSPOSE) {
    const int64_t wide = spr::fp8_width(width);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t r = r0 + 8 * rv + i;
      if (r < rows && c < wide) *reinterpret_cast<uint64_t*>(codes + r * wide + c) = spr::fp8_codes8(v[i], inv[0]);
    }
  } else {
    // a line of the tile is a column's 128 codes in 16 pieces of 8; piece p lies at p ^ (column / 8 % 16),
    // so that the 16 lanes that write one piece of columns 8 apart meet every bank once
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float line[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) line[i] = v[i][e];
      *reinterpret_cast<uint64_t*>(tile + (8 * cv + e) * FP8_GROUP + 8 * (rv ^ cv)) = spr::fp8_codes8(line, inv[e]);
    }
    __syncthreads();
    const int64_t wide = spr::fp8_width(rows);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = i * 32 + threadIdx.x / 8, p = threadIdx.x % 8, k = j / 8 % 16;
      const uint64_t* at = reinterpret_cast<const uint64_t*>(tile + j * FP8_GROUP);
      const uint64_t lo = at[(2 * p) ^ k], hi = at[(2 * p + 1) ^ k];
      const int64_t r = r0 + 16 * p;
      if (c0 + j < width && r < wide) {
        *reinterpret_cast<spr::u32x4*>(codes + (c0 + j) * wide + r) =
            spr::u32x4{static_cast<uint32_t>(lo), static_cast<uint32_t>(lo >> 32), static_cast<uint32_t>(hi),
                       static_cast<uint32_t>(hi >> 32)};
      }
    }
  }
}

// Values of codes: 16 a lane.  row_shift 7 where the scales are of 128 rows.
template <int DT>
__global__ __launch_bounds__(THREADS) void dequantise_kernel(const uint8_t* __restrict__ codes, int64_t ld,
                                                            const uint8_t* __restrict__ scales, int64_t scales_ld,
                                                            int32_t row_shift, uint32_t rows, uint32_t vecs,
                                                            typename Elem<DT>::S* __restrict__ out) {
  const uint64_t i = static_cast<uint64_t>(blockIdx.x) * THREADS + threadIdx.x;
  const uint32_t row = static_cast<uint32_t>(i / vecs);
  if (row >= rows) return;
  const uint32_t c = static_cast<uint32_t>(i - static_cast<uint64_t>(row) * vecs) * 16;
  const spr::u32x4 q = *reinterpret_cast<const spr::u32x4*>(codes + row * ld + c);
  const float s = spr::fp8_scale(scales[(row >> row_shift) * scales_ld + c / FP8_GROUP]);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  typename Elem<DT>::S* o = out + (static_cast<int64_t>(row) * vecs * 16 + c);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[2 * h + e]), false);
      const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[2 * h + e]), true);
      v[4 * e] = lo[0] * s, v[4 * e + 1] = lo[1] * s, v[4 * e + 2] = hi[0] * s, v[4 * e + 3] = hi[1] * s;
    }
    spr::store8<DT>(o + 8 * h, v);
  }
}

template <int DT>
int launch_quantise(const void* x, int64_t ld, int64_t rows, int32_t width, bool square, bool transpose, uint8_t* codes,
                    uint8_t* scales, hipStream_t stream) {
  const auto* xs = static_cast<const typename Elem<DT>::S*>(x);
  const uint32_t across = static_cast<uint32_t>(spr::fp8_groups(width));
  if (!square && !transpose) {
    const int64_t blocks = spr::ceil_div(rows * across, THREADS / 16);
    quantise_rows_kernel<DT><<<static_cast<uint32_t>(blocks), THREADS, 0, stream>>>(xs, ld, static_cast<uint32_t>(rows),
                                                                                   width, across, codes, scales);
    SPR_LAUNCHED("quantise_rows_kernel");
    return SPR_OK;
  }
  const dim3 grid(across, static_cast<uint32_t>(spr::fp8_groups(rows)));
  if (!transpose) quantise_tile_kernel<DT, true, false><<<grid, THREADS, 0, stream>>>(xs, ld, rows, width, codes, scales);
  else if (square) quantise_tile_kernel<DT, true, true><<<grid, THREADS, 0, stream>>>(xs, ld, rows, width, codes, scales);
  else quantise_tile_kernel<DT, false, true><<<grid, THREADS, 0, stream>>>(xs, ld, rows, width, codes, scales);
  SPR_LAUNCHED("quantise_tile_kernel");
  return SPR_OK;
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace

extern "C" int spr_fp8_quantize(const void* x, int64_t ld, int64_t rows, int32_t width, int32_t dtype, int32_t square,
                                int32_t transpose, uint8_t* codes, uint8_t* scales, hipStream_t stream) {
  SPR_REQUIRE(dtype >= 0 && dtype <= 2, "spr_fp8_quantize: dtype %d not in {0, 1, 2}", dtype);
  // (a launch of tiles has at most 65,535 of them one below the other)
  SPR_REQUIRE(rows >= 0 && rows < (int64_t(1) << 24) && (rows <= 65535 * int64_t(FP8_GROUP) || !(square || transpose)) &&
                  width >= 0 && width <= (1 << 30),
              "spr_fp8_quantize: %lld rows of %d", static_cast<long long>(rows), width);
  SPR_REQUIRE(rows * spr::fp8_groups(width) < (int64_t(1) << 28) - 64, "spr_fp8_quantize: too many groups");
  if (rows == 0 || width == 0) return SPR_OK;
  SPR_REQUIRE(x && codes && scales, "spr_fp8_quantize: null pointer");
  SPR_REQUIRE(ld >= 0, "spr_fp8_quantize: negative stride");
  SPR_REQUIRE(aligned(codes, 16), "spr_fp8_quantize: codes must be 16-byte aligned");
  switch (dtype) {
    case 0: return launch_quantise<0>(x, ld, rows, width, square != 0, transpose != 0, codes, scales, stream);
    case 1: return launch_quantise<1>(x, ld, rows, width, square != 0, transpose != 0, codes, scales, stream);
    default: return launch_quantise<2>(x, ld, rows, width, square != 0, transpose != 0, codes, scales, stream);
  }
}

extern "C" int spr_fp8_dequantize(const uint8_t* codes, int64_t ld, const uint8_t* scales, int64_t scales_ld,
                                  int32_t square, int64_t rows, int32_t width, int32_t dtype, void* out,
                                  hipStream_t stream) {
  SPR_REQUIRE(dtype >= 0 && dtype <= 2, "spr_fp8_dequantize: dtype %d not in {0, 1, 2}", dtype);
  SPR_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31) && width >= 0 && width % 16 == 0,
              "spr_fp8_dequantize: %lld rows of %d", static_cast<long long>(rows), width);
  if (rows == 0 || width == 0) return SPR_OK;
  SPR_REQUIRE(codes && scales && out, "spr_fp8_dequantize: null pointer");
  SPR_REQUIRE(ld >= 0 && ld % 16 == 0 && scales_ld >= 0, "spr_fp8_dequantize: strides %lld, %lld",
              static_cast<long long>(ld), static_cast<long long>(scales_ld));
  SPR_REQUIRE(aligned(codes, 16) && aligned(out, 16), "spr_fp8_dequantize: tensors must be 16-byte aligned");
  const uint32_t vecs = static_cast<uint32_t>(width / 16);
  const int64_t blocks = spr::ceil_div(rows * vecs, THREADS);
  SPR_REQUIRE(blocks < (int64_t(1) << 24), "spr_fp8_dequantize: too many values");
  const int32_t shift = square != 0 ? 7 : 0;
  const uint32_t n = static_cast<uint32_t>(rows);
#define SPR_DEQUANTISE(DT)                                                                          \
  dequantise_kernel<DT><<<static_cast<uint32_t>(blocks), THREADS, 0, stream>>>(                     \
      codes, ld, scales, scales_ld, shift, n, vecs, static_cast<typename Elem<DT>::S*>(out))
  if (dtype == 0) SPR_DEQUANTISE(0);
  else if (dtype == 1) SPR_DEQUANTISE(1);
  else SPR_DEQUANTISE(2);
#undef SPR_DEQUANTISE
  SPR_LAUNCHED("dequantise_kernel");
  return SPR_OK;
}
