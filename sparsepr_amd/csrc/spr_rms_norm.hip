// Root-mean-square norm of rows, with the residual's addition in front, 8-bit codes behind, and its gradient.
//
//   s = x + residual (rounded once, to the residual's type; s = x without one)
//   r = 1 / sqrt(mean(s^2) + eps),   y = s r w
//   out: y rounded to x's type, or e4m3 codes with a scale byte per 128 channels (spr_fp8.h)
// The norm reads the sum as it is stored, so that the gradient and a later call see the same one.
//
//   gradient, with g = dy w:   dx = r (g - s r^2 mean(g s)) + dsum,   dw = sum over rows of dy s r
//
// Sums are fp32, the norm's over more than 16 lanes 64 bits, in an order that depends on the sizes only.
// Bound by memory: every input is read once and kept in registers over the reduction, vectors of 8 channels a
// lane.  32,760 rows of 5120 in bf16 with residual and codes (1.18 GB) take 215 us one call behind the other, 5.5 TB/s
// where a copy has 5.1, and 241 to 265 between other kernels; the gradient of 8191 rows of 2560 (294 MB) 55 us, and
// 6 us for the weight's partial sums.  Outputs in bf16 (671 MB) take 139 to 146 us, with a residual (1.34 GB) 233 to 251.
// One row of 5120 takes 4.0 us.
#include "spr_fp8.h"

namespace {

using spr::Elem;
using spr::load8n;
using spr::load8n_any;
using spr::store8n;

constexpr int MAX_WIDTH = 16384;

// Rows of a [n0, n1, width] tensor with any strides of its first two dims.
struct Rows {
  const void* p;
  int64_t s0, s1;
  int32_t n1;
};
__device__ __forceinline__ int64_t row_at(const Rows& t, uint32_t row) {
  const uint32_t a = row / static_cast<uint32_t>(t.n1);
  return a * t.s0 + (row - a * static_cast<uint32_t>(t.n1)) * t.s1;
}

// The sums of N values over the threads of a row, in each of them: 16, or (0) the whole workgroup, whose waves meet
// in `red`, 16 N of T.  T double is for sums past 16 lanes in 64 bits: the roundings of those below average out.
template <int TPR, typename T, int N>
__device__ __forceinline__ void row_total(const float (&a)[N], T (&total)[N], T* red) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    total[i] = spr::row_sum(a[i]);
    if constexpr (TPR == 0) {
      total[i] += __shfl_xor(total[i], 16, 64);
      total[i] += __shfl_xor(total[i], 32, 64);
    }
  }
  if (TPR == 0 && blockDim.x > 64) {
    const int waves = blockDim.x >> 6;
    __syncthreads();  // earlier sums have been read
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) red[(threadIdx.x >> 6) * N + i] = total[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) total[i] = T(0);
    for (int w = 0; w < waves; ++w)
#pragma unroll
      for (int i = 0; i < N; ++i) total[i] += red[w * N + i];
  }
}

// Eight partial sums of a lane as a tree.
__device__ __forceinline__ float tree_sum(const float (&p)[8]) {
  return ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
}

// 1 / sqrt(ss / width + eps).  One step of Newton from the instruction's estimate.
__device__ __forceinline__ double inverse_rms(double ss, double inv_width, float eps) {
  const double v = ss * inv_width + static_cast<double>(eps);
  const double r = __builtin_amdgcn_rsq(v), e = __builtin_fma(-v * r, r, 1.0);
  return __builtin_isfinite(e) ? r + 0.5 * r * e : r;  // (of 0 and infinity as they are)
}

// s inv w with the roundings of the two products carried along, so rounded once to fp32: a value next to a border of its
// output's type then goes where the formula in more digits sends it (of 5 M bf16 outputs 2 to 12 go elsewhere, 16 to 35
// with two roundings; 305 instead of 301 us on 32,760 rows of 5120).  Where a product is 0, infinite or NaN it is as it is.
__device__ __forceinline__ float normed(float s, float inv, float inv_low, float w) {
  const float a = s * inv, y = a * w;
  const float low = __builtin_fmaf(s, inv_low, __builtin_fmaf(s, inv, -a));
  const float exact = __builtin_fmaf(a, w, low * w);
  return y != 0.0f && __builtin_isfinite(y) ? exact : y;
}

// TPR threads a row (0: the workgroup), NV vectors of 8 channels a thread.  RES: 0 no residual, 1 of x's type, 2 fp32.
template <int DT, int RES, bool FP8, int TPR, int NV>
__global__ __launch_bounds__(TPR == 0 ? 1024 : 256) void norm_kernel(
    Rows x, Rows residual, const void* __restrict__ weight, int32_t weight_dtype, uint32_t rows, int32_t width,
    double inv_width, float eps, void* __restrict__ out, uint8_t* __restrict__ scales, void* __restrict__ sum) {
  constexpr int SDT = RES == 2 ? 2 : DT;
  using S = typename Elem<DT>::S;
  using R = typename Elem<SDT>::S;
  __shared__ double red[16];
  const int lane = TPR == 0 ? threadIdx.x : threadIdx.x % TPR, step = TPR == 0 ? blockDim.x : TPR;
  const uint32_t row = TPR == 0 ? blockIdx.x : blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  if (TPR != 0 && row >= rows) return;
  const S* xr = static_cast<const S*>(x.p) + row_at(x, row);
  float s[NV][8];
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int c = (lane + u * step) * 8;
    load8n<DT>(xr + c, width - c, s[u]);
  }
  if constexpr (RES != 0) {
    const R* rr = static_cast<const R*>(residual.p) + row_at(residual, row);
    R* sr = static_cast<R*>(sum) + static_cast<int64_t>(row) * width;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int c = (lane + u * step) * 8;
      float t[8];
      load8n<SDT>(rr + c, width - c, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[u][e] = spr::round_t<SDT>(s[u][e] + t[e]);
      if (c < width) store8n<SDT>(sr + c, width - c, s[u]);
    }
  }
  float p[8] = {};
#pragma unroll
  for (int u = 0; u < NV; ++u)
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = __builtin_fmaf(s[u][e], s[u][e], p[e]);
  float ss[1] = {tree_sum(p)};
  double total[1];
  row_total<TPR>(ss, total, red);
  const double root = inverse_rms(total[0], inv_width, eps);
  const float inv = static_cast<float>(root);
  const float inv_low = __builtin_isfinite(inv) ? static_cast<float>(root - static_cast<double>(inv)) : 0.0f;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int c = (lane + u * step) * 8;
    float w[8];
    if (weight != nullptr) {
      load8n_any(weight, weight_dtype, c, width - c, w);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = 1.0f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s[u][e] = normed(s[u][e], inv, inv_low, w[e]);
    if constexpr (FP8) {
      // 16 lanes are a group of 128 channels; all of them come here
      if (c + 8 > width) {  // 0 * inf and 0 * NaN behind the row's end
#pragma unroll
        for (int e = 0; e < 8; ++e) s[u][e] = c + e < width ? s[u][e] : 0.0f;
      }
      const uint32_t b = spr::fp8_scale_byte(spr::row_max(spr::magnitude_bits8(s[u])));
      const int64_t wide = spr::fp8_width(width);
      if (c < wide) {
        const uint64_t codes = spr::fp8_codes8(s[u], spr::fp8_inverse_scale(b));
        *reinterpret_cast<uint64_t*>(static_cast<uint8_t*>(out) + row * wide + c) = codes;
        if (lane % 16 == 0) scales[row * spr::fp8_groups(width) + c / spr::FP8_GROUP] = static_cast<uint8_t>(b);
      }
    } else {
      if (c < width) store8n<DT>(static_cast<S*>(out) + static_cast<int64_t>(row) * width + c, width - c, s[u]);
    }
  }
}

// The gradient: workgroups take rows in turn, each thread keeps the weight's gradient of its channels
// over all of them, and the workgroups' parts are added by a second kernel in a fixed order.
template <int DT, int SDT, int TPR, int NV>
__global__ __launch_bounds__(TPR == 0 ? 1024 : 256) void norm_backward_kernel(
    Rows dy, Rows s_in, Rows dsum, const void* __restrict__ weight, int32_t weight_dtype, uint32_t rows, int32_t width,
    double inv_width, float eps, void* __restrict__ dx, float* __restrict__ parts) {
  constexpr int PER = TPR == 0 ? 1 : 256 / TPR;  // rows at a time
  using S = typename Elem<DT>::S;
  using R = typename Elem<SDT>::S;
  __shared__ float red[32];
  const int lane = TPR == 0 ? threadIdx.x : threadIdx.x % TPR, step = TPR == 0 ? blockDim.x : TPR;
  const int sub = TPR == 0 ? 0 : threadIdx.x / TPR;
  float w[NV][8], dw[NV][8];
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int c = (lane + u * step) * 8;
    if (weight != nullptr) {
      load8n_any(weight, weight_dtype, c, width - c, w[u]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[u][e] = 1.0f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[u][e] = 0.0f;
  }
  for (uint32_t row = blockIdx.x * PER + sub; row < rows; row += gridDim.x * PER) {
    const S* dyr = static_cast<const S*>(dy.p) + row_at(dy, row);
    const R* sr = static_cast<const R*>(s_in.p) + row_at(s_in, row);
    float g[NV][8], s[NV][8], d[NV][8];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int c = (lane + u * step) * 8;
      load8n<DT>(dyr + c, width - c, g[u]);
      load8n<SDT>(sr + c, width - c, s[u]);
    }
    if (dsum.p != nullptr) {
      const R* dr = static_cast<const R*>(dsum.p) + row_at(dsum, row);
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        const int c = (lane + u * step) * 8;
        load8n<SDT>(dr + c, width - c, d[u]);
      }
    } else {
#pragma unroll
      for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) d[u][e] = 0.0f;
    }
    float p[8] = {}, q[8] = {};
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = __builtin_fmaf(s[u][e], s[u][e], p[e]);
        q[e] = __builtin_fmaf(g[u][e] * w[u][e], s[u][e], q[e]);
      }
    float t[2] = {tree_sum(p), tree_sum(q)};  // of s^2 and of g s
    float total[2];  // (in 64 bits, as the norm's: 74 instead of 65 us on 8191 rows of 2560)
    row_total<TPR>(t, total, red);
    const float inv = static_cast<float>(inverse_rms(total[0], inv_width, eps));
    // (inv^2 by itself leaves fp32's range where rows below 2^-64 are normed with no epsilon)
    const float along = inv * (inv * (total[1] * static_cast<float>(inv_width)));
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int c = (lane + u * step) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        dw[u][e] = __builtin_fmaf(g[u][e], s[u][e] * inv, dw[u][e]);
        d[u][e] = __builtin_fmaf(inv, __builtin_fmaf(-s[u][e], along, g[u][e] * w[u][e]), d[u][e]);
      }
      if (c < width) store8n<SDT>(static_cast<R*>(dx) + static_cast<int64_t>(row) * width + c, width - c, d[u]);
    }
  }
  if (parts == nullptr) return;
  // the rows that a workgroup takes at a time, added in LDS; then one row of `parts` each
  if constexpr (PER > 1) {
    static_assert(NV == 1, "one vector a thread");
    __shared__ float add[PER * TPR * 8];
#pragma unroll
    for (int e = 0; e < 8; ++e) add[(sub * TPR + lane) * 8 + e] = dw[0][e];
    __syncthreads();
    for (int c = threadIdx.x; c < TPR * 8 && c < width; c += 256) {
      float t = 0.0f;
      for (int r = 0; r < PER; ++r) t += add[r * TPR * 8 + c];
      parts[static_cast<int64_t>(blockIdx.x) * width + c] = t;
    }
  } else {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int c = (lane + u * step) * 8;
      if (c < width) store8n<2>(parts + static_cast<int64_t>(blockIdx.x) * width + c, width - c, dw[u]);
    }
  }
}

// dw[c] = sum over the workgroups' parts: 32 channels a workgroup, 32 half waves over the parts.
__global__ __launch_bounds__(1024) void norm_weight_gradient_kernel(const float* __restrict__ parts, int32_t n,
                                                                   int32_t width, float* __restrict__ dw) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float t[4] = {};
  if (c < width) {
    int p = slice;
    for (; p + 96 < n; p += 128)
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] += parts[static_cast<int64_t>(p + 32 * i) * width + c];
    for (; p < n; p += 32) t[0] += parts[static_cast<int64_t>(p) * width + c];
  }
  red[slice][lane] = (t[0] + t[1]) + (t[2] + t[3]);
  __syncthreads();
  float sum = red[lane][slice];  // slice's channel, one part a lane
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 32);
  if (lane == 0 && blockIdx.x * 32 + slice < width) dw[blockIdx.x * 32 + slice] = sum;
}

// A row is a quarter wave's to 128 channels, a wave's to 512 and a workgroup's above.  The norm has one vector of 8
// channels a lane to 512 and two above: 160 M values of 5120 channels to 8 bits take 197 us with two (five waves),
// 250 with one (ten), 201 with four; 1024 and 8192 channels 183 and 192 with two, 187 and 204 with one.  The gradient
// has one to 8192: 21 M values of 2560 and 5120 channels take 41 and 40 us with one, 46 and 47 with two.
uint32_t norm_threads(int32_t width) {
  return width <= 128 ? 256 : width <= 512 ? 64 : 64 * static_cast<uint32_t>(spr::ceil_div(width, 1024));
}
uint32_t gradient_threads(int32_t width) {
  return width <= 128 ? 256 : 64 * static_cast<uint32_t>(spr::ceil_div(width, width <= 8192 ? 512 : 1024));
}
int32_t rows_at_a_time(int32_t width) { return width <= 128 ? 16 : 1; }

template <int DT, int RES, bool FP8>
void launch_norm(const Rows& x, const Rows& residual, const void* weight, int32_t weight_dtype, uint32_t rows,
                 int32_t width, float eps, void* out, uint8_t* scales, void* sum, hipStream_t stream) {
#define SPR_NORM(TPR, NV)                                                                                    \
  norm_kernel<DT, RES, FP8, TPR, NV>                                                                         \
      <<<static_cast<uint32_t>(spr::ceil_div(rows, rows_at_a_time(width))), norm_threads(width), 0, stream>>>( \
          x, residual, weight, weight_dtype, rows, width, 1.0 / width, eps, out, scales, sum)
  if (width <= 128) SPR_NORM(16, 1);
  else if (width <= 512) SPR_NORM(0, 1);
  else SPR_NORM(0, 2);
#undef SPR_NORM
}

template <int DT, int RES>
void launch_norm(bool fp8, const Rows& x, const Rows& residual, const void* weight, int32_t weight_dtype,
                 uint32_t rows, int32_t width, float eps, void* out, uint8_t* scales, void* sum, hipStream_t stream) {
  if (fp8) launch_norm<DT, RES, true>(x, residual, weight, weight_dtype, rows, width, eps, out, scales, sum, stream);
  else launch_norm<DT, RES, false>(x, residual, weight, weight_dtype, rows, width, eps, out, scales, sum, stream);
}

// Workgroups of the gradient: about 5120 waves, so that every SIMD has a few rows on their way and the parts of the
// weight's gradient stay small beside the rows (2560 channels: 43, 41 and 47 us with 512, 1024 and 2048 of them;
// 1024: 61, 44 and 42; 8192: 46 and 54 with 512 and 1024).
int32_t backward_groups(int64_t rows, int32_t width) {
  const int64_t waves = gradient_threads(width) / 64, most = 5120 / waves > 512 ? 5120 / waves : 512;
  const int64_t all = spr::ceil_div(rows, rows_at_a_time(width));
  return static_cast<int32_t>(all < most ? all : most);
}

template <int DT, int SDT>
void launch_backward(const Rows& dy, const Rows& s, const Rows& dsum, const void* weight, int32_t weight_dtype,
                     uint32_t rows, int32_t width, float eps, void* dx, float* parts, hipStream_t stream) {
  const uint32_t groups = static_cast<uint32_t>(backward_groups(rows, width));
#define SPR_NORM(TPR, NV)                                                                 \
  norm_backward_kernel<DT, SDT, TPR, NV><<<groups, gradient_threads(width), 0, stream>>>( \
      dy, s, dsum, weight, weight_dtype, rows, width, 1.0 / width, eps, dx, parts)
  if (width <= 128) SPR_NORM(16, 1);
  else if (width <= 8192) SPR_NORM(0, 1);
  else SPR_NORM(0, 2);
#undef SPR_NORM
}

// (a launch has fewer than 2^32 threads)
bool launch_fits(int64_t n0, int64_t n1, int32_t width) {
  const int64_t blocks = spr::ceil_div(n0 * n1, rows_at_a_time(width));
  return n0 * n1 < (int64_t(1) << 31) && blocks * norm_threads(width) < (int64_t(1) << 32);
}

bool rows_fit(int64_t n0, int64_t n1, int64_t s0, int64_t s1) {
  return n0 <= 1 || n1 <= 1 || (s0 >= 0 && s1 >= 0);
}

}  // namespace

extern "C" int spr_rms_norm(const void* x, int64_t x_s0, int64_t x_s1, const void* residual, int64_t res_s0,
                            int64_t res_s1, int32_t n0, int32_t n1, int32_t width, int32_t dtype,
                            int32_t residual_dtype, const void* weight, int32_t weight_dtype, float epsilon, void* out,
                            uint8_t* scales, void* sum, hipStream_t stream) {
  SPR_REQUIRE(dtype >= 0 && dtype <= 2, "spr_rms_norm: dtype %d not in {0, 1, 2}", dtype);
  SPR_REQUIRE(width >= 1 && width <= MAX_WIDTH, "spr_rms_norm: width %d not in 1 .. %d", width, MAX_WIDTH);
  SPR_REQUIRE(n0 >= 0 && n1 >= 0 && launch_fits(n0, n1, width), "spr_rms_norm: too many rows");
  SPR_REQUIRE(epsilon >= 0.0f && epsilon < __builtin_huge_valf(), "spr_rms_norm: epsilon must be finite and not negative");
  SPR_REQUIRE(weight == nullptr || weight_dtype == dtype || weight_dtype == 2,
              "spr_rms_norm: weights of dtype %d for rows of %d", weight_dtype, dtype);
  SPR_REQUIRE(residual == nullptr || residual_dtype == dtype || residual_dtype == 2,
              "spr_rms_norm: a residual of dtype %d for rows of %d", residual_dtype, dtype);
  if (n0 == 0 || n1 == 0) return SPR_OK;
  SPR_REQUIRE(x && out && (residual == nullptr || sum), "spr_rms_norm: null pointer");
  SPR_REQUIRE(rows_fit(n0, n1, x_s0, x_s1) && rows_fit(n0, n1, res_s0, res_s1), "spr_rms_norm: negative stride");
  SPR_REQUIRE(scales == nullptr || (reinterpret_cast<uintptr_t>(out) & 7) == 0, "spr_rms_norm: codes must be 8-byte aligned");
  const Rows xr{x, x_s0, x_s1, n1}, rr{residual, res_s0, res_s1, n1};
  const uint32_t rows = static_cast<uint32_t>(n0) * static_cast<uint32_t>(n1);
  const bool fp8 = scales != nullptr;
  const int res = residual == nullptr ? 0 : residual_dtype == dtype ? 1 : 2;
#define SPR_NORM(DT, RES) \
  launch_norm<DT, RES>(fp8, xr, rr, weight, weight_dtype, rows, width, epsilon, out, scales, sum, stream)
#define SPR_NORM_RES(DT)          \
  if (res == 0) SPR_NORM(DT, 0);  \
  else if (res == 1) SPR_NORM(DT, 1); \
  else SPR_NORM(DT, 2)
  if (dtype == 0) { SPR_NORM_RES(0); }
  else if (dtype == 1) { SPR_NORM_RES(1); }
  else if (res == 0) { SPR_NORM(2, 0); }
  else { SPR_NORM(2, 1); }
#undef SPR_NORM_RES
#undef SPR_NORM
  SPR_LAUNCHED("norm_kernel");
  return SPR_OK;
}

extern "C" size_t spr_rms_norm_backward_workspace(int64_t rows, int32_t width) {
  if (rows <= 0 || width < 1 || width > MAX_WIDTH) return 0;
  return sizeof(float) * static_cast<size_t>(width) * backward_groups(rows, width);
}

extern "C" int spr_rms_norm_backward(const void* dy, int64_t dy_s0, int64_t dy_s1, const void* s, int64_t s_s0,
                                     int64_t s_s1, const void* dsum, int64_t ds_s0, int64_t ds_s1, int32_t n0,
                                     int32_t n1, int32_t width, int32_t dtype, int32_t sum_dtype, const void* weight,
                                     int32_t weight_dtype, float epsilon, void* dx, float* dweight, void* workspace,
                                     size_t workspace_bytes, hipStream_t stream) {
  SPR_REQUIRE(dtype >= 0 && dtype <= 2, "spr_rms_norm_backward: dtype %d not in {0, 1, 2}", dtype);
  SPR_REQUIRE(sum_dtype == dtype || sum_dtype == 2, "spr_rms_norm_backward: a sum of dtype %d for gradients of %d",
              sum_dtype, dtype);
  SPR_REQUIRE(width >= 1 && width <= MAX_WIDTH, "spr_rms_norm_backward: width %d not in 1 .. %d", width, MAX_WIDTH);
  SPR_REQUIRE(n0 >= 0 && n1 >= 0 && launch_fits(n0, n1, width), "spr_rms_norm_backward: too many rows");
  SPR_REQUIRE(epsilon >= 0.0f && epsilon < __builtin_huge_valf(),
              "spr_rms_norm_backward: epsilon must be finite and not negative");
  SPR_REQUIRE(weight == nullptr || weight_dtype == dtype || weight_dtype == 2,
              "spr_rms_norm_backward: weights of dtype %d for gradients of %d", weight_dtype, dtype);
  const uint32_t rows = static_cast<uint32_t>(n0) * static_cast<uint32_t>(n1);
  const int32_t groups = rows == 0 ? 0 : backward_groups(rows, width);
  if (rows == 0) {
    if (dweight != nullptr) {
      norm_weight_gradient_kernel<<<static_cast<uint32_t>(spr::ceil_div(width, 32)), 1024, 0, stream>>>(nullptr, 0, width,
                                                                                                      dweight);
      SPR_LAUNCHED("norm_weight_gradient_kernel");
    }
    return SPR_OK;
  }
  SPR_REQUIRE(dy && s && dx, "spr_rms_norm_backward: null pointer");
  SPR_REQUIRE(rows_fit(n0, n1, dy_s0, dy_s1) && rows_fit(n0, n1, s_s0, s_s1) && rows_fit(n0, n1, ds_s0, ds_s1),
              "spr_rms_norm_backward: negative stride");
  if (dweight != nullptr) {
    const size_t need = spr_rms_norm_backward_workspace(rows, width);
    if (workspace == nullptr || workspace_bytes < need) {
      spr_set_error("spr_rms_norm_backward: workspace %zu < %zu bytes", workspace_bytes, need);
      return SPR_EWORKSPACE;
    }
    SPR_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "spr_rms_norm_backward: workspace not 16-byte aligned");
  }
  const Rows dyr{dy, dy_s0, dy_s1, n1}, sr{s, s_s0, s_s1, n1}, dsr{dsum, ds_s0, ds_s1, n1};
  float* parts = dweight != nullptr ? static_cast<float*>(workspace) : nullptr;
#define SPR_BACK(DT, SDT) \
  launch_backward<DT, SDT>(dyr, sr, dsr, weight, weight_dtype, rows, width, epsilon, dx, parts, stream)
  if (dtype == 2) SPR_BACK(2, 2);
  else if (dtype == 0 && sum_dtype == 0) SPR_BACK(0, 0);
  else if (dtype == 0) SPR_BACK(0, 2);
  else if (sum_dtype == 1) SPR_BACK(1, 1);
  else SPR_BACK(1, 2);
#undef SPR_BACK
  SPR_LAUNCHED("norm_backward_kernel");
  if (dweight != nullptr) {
    norm_weight_gradient_kernel<<<static_cast<uint32_t>(spr::ceil_div(width, 32)), 1024, 0, stream>>>(parts, groups, width,
                                                                                                    dweight);
    SPR_LAUNCHED("norm_weight_gradient_kernel");
  }
  return SPR_OK;
}
