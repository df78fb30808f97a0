// Rotary positions with several axes (time, height, width): Q and K turned in one launch, from the
// tokens' places instead of a table of angles.
//
//   turn_i = pos[axis_i] f_i / (2 pi), its nearest whole number taken off;  (c, s) = cos, sin(2 pi turn)
//   (a, b) -> (a c - b s, b c + a s)   on dims (2i, 2i + 1) or (i, i + R / 2); dims from R on are copied
// The inverse (the gradient of the rotation) has -s.
//
// The turn is 64 bits up to the part below one: at place 118,800 an angle in fp32 is off by 0.004.  Its
// sine and cosine are fp32 (sincospif), the rotation fp32 with one rounding at the end.
// Bound by memory (Q and K read and written once).  A lane holds 4 pairs of one token: it finds their
// angles once and turns the same pairs of every PER-th head.
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

// Four values, from any address that an element may have.
template <int DT>
__device__ __forceinline__ void load4(const typename Elem<DT>::S* p, float (&x)[4]) {
  typename Elem<DT>::S r[4];
  __builtin_memcpy(r, p, sizeof(r));
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = Elem<DT>::to_f(r[e]);
}
template <int DT>
__device__ __forceinline__ void store4(typename Elem<DT>::S* p, const float (&x)[4]) {
  typename Elem<DT>::S r[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = Elem<DT>::from_f(x[e]);
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
  float sn;
  sincospif(2.0f * static_cast<float>(turn - __builtin_rint(turn)), &sn, &c);
  s = sign * sn;
}

// Units of a row: R / 8 of 4 pairs, then (D - R) / 8 of 8 dims to copy.  `units` of them a token, `per`
// tokens-and-head-slots (units lanes each) a workgroup; slots of one token take its heads in turn.
template <int DT, bool HALVES>
__global__ __launch_bounds__(THREADS) void rope_kernel(Side q, Side k, const void* __restrict__ positions,
                                                       int32_t position_code, int64_t position_b, int32_t axes,
                                                       const double* __restrict__ freqs,
                                                       const int32_t* __restrict__ axis, int64_t rows, int64_t tokens,
                                                       int32_t dim, int32_t rotated, int32_t units, int32_t slots,
                                                       float sign) {
  using S = typename Elem<DT>::S;
  const int per = THREADS / units;  // (token, slot) pairs of a workgroup
  const int mine = threadIdx.x / units, unit = threadIdx.x - mine * units;
  if (mine >= per) return;
  const int64_t job = static_cast<int64_t>(blockIdx.x) * per + mine;
  const int64_t row = job / slots;
  if (row >= rows) return;
  const int slot = static_cast<int>(job - row * slots);
  const int64_t b = row / tokens, t = row - b * tokens;
  const bool turned = unit * 8 < rotated;
  float c[4], s[4];
  if (turned) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      angle_of(positions, position_code, b * position_b + t * axes, axes, freqs, axis, unit * 4 + e, sign, c[e], s[e]);
  }
  // the two groups of 4 dims of a unit
  const int d0 = HALVES && turned ? unit * 4 : unit * 8;
  const int d1 = HALVES && turned ? d0 + rotated / 2 : d0 + 4;
  for (int h = slot; h < q.heads + k.heads; h += slots) {
    const bool is_k = h >= q.heads;
    const Side& side = is_k ? k : q;
    const int hh = is_k ? h - q.heads : h;
    const S* x = static_cast<const S*>(side.x) + b * side.b + hh * side.h + t * side.t;
    S* o = static_cast<S*>(side.out) + ((b * side.heads + hh) * tokens + t) * dim;
    float u[4], v[4];
    load4<DT>(x + d0, u);
    load4<DT>(x + d1, v);
    if (turned) {
      float p[4], r[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // pairs (2i, 2i + 1): the first two of a unit lie in u, the others in v
        const float a = HALVES ? u[e] : e < 2 ? u[2 * e] : v[2 * e - 4];
        const float w = HALVES ? v[e] : e < 2 ? u[2 * e + 1] : v[2 * e - 3];
        p[e] = __builtin_fmaf(a, c[e], -(w * s[e]));
        r[e] = __builtin_fmaf(w, c[e], a * s[e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        u[e] = HALVES ? p[e] : e % 2 == 0 ? p[e / 2] : r[e / 2];
        v[e] = HALVES ? r[e] : e % 2 == 0 ? p[2 + e / 2] : r[2 + e / 2];
      }
    }
    store4<DT>(o + d0, u);
    store4<DT>(o + d1, v);
  }
}

template <int DT>
int launch_rope(bool halves, const Side& q, const Side& k, const void* positions, int32_t code, int64_t position_b,
                 int32_t axes, const double* freqs, const int32_t* axis, int64_t rows, int64_t tokens, int32_t dim,
                 int32_t rotated, float sign, hipStream_t stream) {
  const int32_t units = dim / 8, per = THREADS / units, heads = q.heads + k.heads;
  // every head a slot of its own while that leaves CUs without work, else slots of 4 heads or more
  int32_t slots = heads;
  while (slots > 1 && rows * slots > 8192 * static_cast<int64_t>(per) && heads / slots < 8) slots = (slots + 1) / 2;
  const int64_t wanted = spr::ceil_div(rows * slots, per);
  SPR_REQUIRE(wanted < (int64_t(1) << 24), "spr_axial_rope: too many rows");  // 2^32 threads of a launch
  const uint32_t blocks = static_cast<uint32_t>(wanted);
#define SPR_ROPE(HALVES)                                                                                          \
  rope_kernel<DT, HALVES><<<blocks, THREADS, 0, stream>>>(q, k, positions, code, position_b, axes, freqs, axis, rows, \
                                                          tokens, dim, rotated, units, slots, sign)
  if (halves) SPR_ROPE(true);
  else SPR_ROPE(false);
#undef SPR_ROPE
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
#define SPR_ROPE(DT)                                                                                            \
  launch_rope<DT>(halves != 0, qs, ks, positions, position_code, position_b, axes, freqs, axis, batch * tokens, \
                  tokens, dim, rotated, sign, stream)
  if (dtype == 0) return SPR_ROPE(0);
  if (dtype == 1) return SPR_ROPE(1);
  return SPR_ROPE(2);
#undef SPR_ROPE
}
