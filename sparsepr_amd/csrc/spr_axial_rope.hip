// Rotary positions with several axes (time, height, width): Q and K turned in one launch, from the
// tokens' places instead of a table of angles.
//
//   turn_i = pos[axis_i] f_i / (2 pi), its nearest whole number taken off;  (c, s) = cos, sin(2 pi turn)
//   (a, b) -> (a c - b s, b c + a s)   on dims (2i, 2i + 1) or (i, i + R / 2); dims from R on are copied
// The inverse (the gradient of the rotation) has -s.
//
// The turn is 64 bits up to the part below one: at place 118,800 an angle in fp32 is off by 0.004.  Its
// sine and cosine are fp32 (sincospif of its first 24 digits, and what the next ones add, to first order: without it fp32
// outputs are off by 5.6e-8 of their norm instead of 4.1e-8), the rotation fp32 with one rounding at the end.
// Bound by memory (Q and K read and written once): Q and K of 32,760 x 40 x 128 in bf16 take 264 us, 5.1 TB/s, what a
// copy takes.  A lane holds 4 pairs of one token: it finds their angles once and turns the same pairs of several heads.
#include "spr_elem.h"

namespace {

using spr::Elem;

constexpr int THREADS = 256;

struct Side {  // Q or K, [batch, heads, tokens, D], and the output, contiguous
  const void* x;
  void* out;
  int64_t b, h, t;
  int32_t heads;
};

// N values, from any address that an element may have.
template <int DT, int N>
__device__ __forceinline__ void load(const typename Elem<DT>::S* p, float* x) {
  typename Elem<DT>::S r[N];
  __builtin_memcpy(r, p, sizeof(r));
#pragma unroll
  for (int e = 0; e < N; ++e) x[e] = Elem<DT>::to_f(r[e]);
}
template <int DT, int N>
__device__ __forceinline__ void store(typename Elem<DT>::S* p, const float* x) {
  typename Elem<DT>::S r[N];
#pragma unroll
  for (int e = 0; e < N; ++e) r[e] = Elem<DT>::from_f(x[e]);
  __builtin_memcpy(p, r, sizeof(r));
}

__device__ __forceinline__ double place_of(const void* positions, int32_t code, int64_t at) {
  switch (code) {
    case 0: return static_cast<double>(static_cast<const int32_t*>(positions)[at]);
    case 1: return static_cast<double>(static_cast<const int64_t*>(positions)[at]);
    case 2: return static_cast<double>(static_cast<const float*>(positions)[at]);
    default: return static_cast<const double*>(positions)[at];
  }
}

// cos and sin of pair i at a token's place; an axis that the positions do not have gives NaN.
__device__ __forceinline__ void angle_of(const void* positions, int32_t code, int64_t at, int32_t axes,
                                         const double* freqs, const int32_t* axis, int i, float sign, float& c,
                                         float& s) {
  const int32_t a = axis[i];
  if (a < 0 || a >= axes) {
    c = s = __uint_as_float(0x7fc00000u);
    return;
  }
  const double turn = place_of(positions, code, at + a) * (freqs[i] * 0.15915494309189533577);
  const double part = turn - __builtin_rint(turn);
  const float high = static_cast<float>(part);
  const float low = static_cast<float>((part - static_cast<double>(high)) * 6.283185307179586477);  // in radians
  float sn, cs;
  sincospif(2.0f * high, &sn, &cs);
  c = __builtin_fmaf(-sn, low, cs);
  s = sign * __builtin_fmaf(cs, low, sn);
}

// Units of a row: R / 2P of P pairs, then (D - R) / 2P of 2P dims to copy, a lane each.  A workgroup has as many
// tokens as its lanes hold rows, one behind the other, so that it writes one run of each head; its slot takes every
// `slots`-th head, AHEAD of them on their way at once.
template <int DT, bool HALVES, int P>
__global__ __launch_bounds__(THREADS) void rope_kernel(Side q, Side k, const void* __restrict__ positions,
                                                       int32_t position_code, int64_t position_b, int32_t axes,
                                                       const double* __restrict__ freqs,
                                                       const int32_t* __restrict__ axis, int64_t rows, int64_t tokens,
                                                       int32_t dim, int32_t rotated, int32_t slots, float sign) {
  using S = typename Elem<DT>::S;
  constexpr int AHEAD = 4;
  const int units = dim / (2 * P), per = THREADS / units;
  const int mine = threadIdx.x / units, unit = threadIdx.x - mine * units;
  if (mine >= per) return;
  const uint32_t group = blockIdx.x / static_cast<uint32_t>(slots);
  const int64_t row = static_cast<int64_t>(group) * per + mine;
  if (row >= rows) return;
  const int slot = static_cast<int>(blockIdx.x - group * static_cast<uint32_t>(slots));
  const int64_t b = row / tokens, t = row - b * tokens;
  const bool turned = unit * 2 * P < rotated;
  float c[P], s[P];
  if (turned) {
#pragma unroll
    for (int e = 0; e < P; ++e)
      angle_of(positions, position_code, b * position_b + t * axes, axes, freqs, axis, unit * P + e, sign, c[e], s[e]);
  }
  // the two groups of P dims of a unit: a pair's first and second dims, or (interleaved) one behind the other
  const int d0 = HALVES && turned ? unit * P : unit * 2 * P;
  const int d1 = HALVES && turned ? d0 + rotated / 2 : d0 + P;
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const Side& side = which == 0 ? q : k;
    const S* x = static_cast<const S*>(side.x) + b * side.b + t * side.t;
    S* o = static_cast<S*>(side.out) + (b * side.heads * tokens + t) * dim;
    for (int h0 = slot; h0 < side.heads; h0 += AHEAD * slots) {
      float u[AHEAD][2 * P];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int h = h0 + i * slots;
        if (h < side.heads) {
          const S* p = x + h * side.h;
          if constexpr (HALVES) {
            load<DT, P>(p + d0, u[i]);
            load<DT, P>(p + d1, u[i] + P);
          } else {
            load<DT, 2 * P>(p + d0, u[i]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int h = h0 + i * slots;
        if (h < side.heads) {
          if (turned) {
#pragma unroll
            for (int e = 0; e < P; ++e) {
              float& first = u[i][HALVES ? e : 2 * e];
              float& second = u[i][HALVES ? P + e : 2 * e + 1];
              const float f = __builtin_fmaf(first, c[e], -(second * s[e]));
              second = __builtin_fmaf(second, c[e], first * s[e]);
              first = f;
            }
          }
          S* p = o + static_cast<int64_t>(h) * tokens * dim;
          if constexpr (HALVES) {
            store<DT, P>(p + d0, u[i]);
            store<DT, P>(p + d1, u[i] + P);
          } else {
            store<DT, 2 * P>(p + d0, u[i]);
          }
        }
      }
    }
  }
}

// Slots of a token: a million lanes, as even a share of the heads as that allows, and two heads a slot at least where
// that still leaves half a million lanes, since an angle serves the heads that share its slot.  (32,760 tokens of 40
// heads: 264 us with three slots, 274 with two and one; 3 x 2311 tokens of 16 heads of 80 fp32 dims: 32 us with eight
// slots, 35 with sixteen, 40 with one.)
int32_t rope_slots(int64_t rows, int32_t units, int32_t heads) {
  const int64_t lanes = rows * units, wanted = spr::ceil_div(int64_t(1) << 20, lanes);
  const int64_t most = lanes * heads >= int64_t(1) << 20 ? spr::ceil_div(heads, 2) : heads;
  if (wanted >= most) return static_cast<int32_t>(most);
  return static_cast<int32_t>(spr::ceil_div(heads, spr::ceil_div(heads, wanted)));
}

template <int DT, bool HALVES, int P>
int launch_rope(const Side& q, const Side& k, const void* positions, int32_t code, int64_t position_b, int32_t axes,
                const double* freqs, const int32_t* axis, int64_t rows, int64_t tokens, int32_t dim, int32_t rotated,
                float sign, hipStream_t stream) {
  const int32_t units = dim / (2 * P), per = THREADS / units;
  const int32_t slots = rope_slots(rows, units, q.heads > k.heads ? q.heads : k.heads);
  const int64_t blocks = spr::ceil_div(rows, per) * slots;
  SPR_REQUIRE(blocks < (int64_t(1) << 24), "spr_axial_rope: too many rows");  // 2^32 threads of a launch
  rope_kernel<DT, HALVES, P><<<static_cast<uint32_t>(blocks), THREADS, 0, stream>>>(
      q, k, positions, code, position_b, axes, freqs, axis, rows, tokens, dim, rotated, slots, sign);
  SPR_LAUNCHED("rope_kernel");
  return SPR_OK;
}

}  // namespace

extern "C" int spr_axial_rope(const void* q, int64_t q_b, int64_t q_h, int64_t q_t, int32_t q_heads, const void* k,
                              int64_t k_b, int64_t k_h, int64_t k_t, int32_t k_heads, int32_t dtype, int64_t batch,
                              int64_t tokens, int32_t dim, int32_t rotated, const void* positions,
                              int32_t position_code, int64_t position_b, int32_t axes, const double* freqs,
                              const int32_t* axis, int32_t halves, int32_t inverse, void* q_out, void* k_out,
                              hipStream_t stream) {
  SPR_REQUIRE(dtype >= 0 && dtype <= 2, "spr_axial_rope: dtype %d not in {0, 1, 2}", dtype);
  SPR_REQUIRE(position_code >= 0 && position_code <= 3, "spr_axial_rope: position code %d not in {0, 1, 2, 3}",
              position_code);
  SPR_REQUIRE(dim >= 8 && dim <= 1024 && dim % 8 == 0, "spr_axial_rope: head dim %d not a multiple of 8 up to 1024", dim);
  SPR_REQUIRE(rotated >= 0 && rotated <= dim && rotated % 8 == 0, "spr_axial_rope: %d rotated dims of %d", rotated, dim);
  SPR_REQUIRE(axes >= 1 && axes <= 16, "spr_axial_rope: %d axes", axes);
  SPR_REQUIRE(batch >= 0 && tokens >= 0 && q_heads >= 0 && k_heads >= 0 && batch < (int64_t(1) << 31) &&
                  tokens < (int64_t(1) << 31) && q_heads < (1 << 20) && k_heads < (1 << 20),
              "spr_axial_rope: bad size");
  if (batch == 0 || tokens == 0 || q_heads + k_heads == 0) return SPR_OK;
  SPR_REQUIRE((q_heads == 0 || (q && q_out)) && (k_heads == 0 || (k && k_out)) && positions &&
                  (rotated == 0 || (freqs && axis)),
              "spr_axial_rope: null pointer");
  SPR_REQUIRE(batch < (int64_t(1) << 40) / tokens / (q_heads + k_heads), "spr_axial_rope: too many rows");
  const Side qs{q, q_out, q_b, q_h, q_t, q_heads}, ks{k, k_out, k_b, k_h, k_t, k_heads};
  const float sign = inverse != 0 ? -1.0f : 1.0f;
  // 16 bytes of a row a lane, or (halves) 8 and 8 in 16 bits: 16 and 16 took 2 % longer on 118,800 tokens
#define SPR_ROPE(DT, HALVES, P)                                                                                 \
  launch_rope<DT, HALVES, P>(qs, ks, positions, position_code, position_b, axes, freqs, axis, batch * tokens, tokens, \
                             dim, rotated, sign, stream)
  if (halves != 0) return dtype == 0 ? SPR_ROPE(0, true, 4) : dtype == 1 ? SPR_ROPE(1, true, 4) : SPR_ROPE(2, true, 4);
  return dtype == 0 ? SPR_ROPE(0, false, 4) : dtype == 1 ? SPR_ROPE(1, false, 4) : SPR_ROPE(2, false, 2);
#undef SPR_ROPE
}
