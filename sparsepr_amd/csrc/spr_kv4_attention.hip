// Attention over a paged K/V cache held in 4 bits (layout: spr_kv4.h).
//
//   out[b, h, t] = softmax_j(scale * q[b, h, t] . K[j]) V[j],  lse = ln sum_j exp(scale * q . K[j])
//
// over the visible tokens j of sequence b's pages: all of them, or (causal) those up to the query's
// own, the last of the call's rows being the sequence's last token.  A row that sees nothing is 0
// with lse -inf.  The query heads of one kv head share its K and V: their rows, token-major, are one
// list of rows * group query rows.
//
// K and V values (code times scale) are exact in bf16, so the conversion to the MFMA's operand loses
// nothing; fp16 queries and probabilities go in as two bf16 terms (hi + lo) and lose at most 2^-16
// of themselves.  Scores, the running maximum and sum and the output are fp32; bf16 calls round each
// probability to bf16 once, relative to a maximum at most 2^8 below the row's own.
#include <algorithm>
#include <type_traits>

#include "spr_kv4.h"

namespace {

using spr::bf16x8;
using spr::f32x16;
using spr::f32x4;
using spr::u32x4;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float LOG2E = 1.44269504088896341f;
constexpr float LN2 = 0.693147180559945309f;
constexpr float NEG_INF = -__builtin_huge_valf();
// Growth of a row maximum (log2 units) that rescales the running output; below it p <= 2^8.
constexpr float RESCALE_SLACK = 8.0f;

struct AttnArgs {
  const uint16_t* q;
  const uint8_t* pages;
  const int32_t *table, *lengths, *counts, *seq_ids;
  uint16_t* out;
  float* lse;            // nullable
  float* part_o;         // [batch][kv_heads][nsplit][rows * group][D], unnormalised
  float* part_ml;        // the same rows' (maximum, sum)
  int64_t q_b, q_h, q_t;  // strides in elements
  int64_t page_stride;    // bytes
  int32_t batch, kv_heads, group, rows, sequences, wide, log_s, num_pages, nsplit, causal;
  float scale_log2;  // softmax scale * log2(e)
};

// What one sequence gives to attend.
struct Span {
  int32_t length;  // tokens, at most what the table's row can hold
  int32_t count;   // query rows in use
  int32_t seq;     // row of the table
  bool broken;     // no such sequence, or a length the table cannot hold: rows in use come out NaN
};

__device__ __forceinline__ Span span_of(const AttnArgs& a, int b) {
  Span s;
  s.seq = a.seq_ids != nullptr ? a.seq_ids[b] : b;
  s.broken = s.seq < 0 || s.seq >= a.sequences;
  if (s.broken) s.seq = 0;
  const int32_t room = a.wide << a.log_s;
  const int32_t len = a.lengths[s.seq];
  s.broken |= len < 0 || len > room;
  s.length = min(max(len, 0), room);
  s.count = a.counts != nullptr ? min(max(a.counts[b], 0), a.rows) : a.rows;
  return s;
}

// Tokens that query row t sees: keys [0, visible).
__device__ __forceinline__ int32_t visible_of(const AttnArgs& a, const Span& s, int t) {
  if (t >= s.count) return 0;
  return a.causal != 0 ? min(max(s.length - s.count + t + 1, 0), s.length) : s.length;
}

// Offset of a token block's page, and whether the table names one in the pool.
__device__ __forceinline__ int64_t page_offset(const AttnArgs& a, const int32_t* row, int32_t key, bool& ok) {
  const int32_t page = row[key >> a.log_s];
  ok = page >= 0 && page < a.num_pages;
  return (ok ? page : 0) * a.page_stride;
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// x over the four lane groups of 16 (lanes l, l ^ 16, l ^ 32, l ^ 48 end with the same value).
__device__ __forceinline__ float max_groups(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_groups(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(spr::as_bf16x8(a), spr::as_bf16x8(b), c, 0, 0, 0);
}

typedef __attribute__((__vector_size__(4 * sizeof(short)))) short v4i16;
typedef __attribute__((address_space(3))) v4i16 lds_v4i16;
// ds_read_b64_tr_b16: in each group of 16 lanes, output lane 4A + B gets element B of the reads of
// lanes A, A + 4, A + 8, A + 12.
__device__ __forceinline__ u32x2 lds_read_tr16(const uint8_t* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(p)));
}

// Eight values of a query row: bf16 as they are, fp16 as bf16 terms hi + lo (the 11 bits of an fp16
// split into 8 and 3: exact but for fp16 denormals below bf16's reach, none).
template <bool F16>
__device__ __forceinline__ void split8(u32x4 x, u32x4& hi, u32x4& lo) {
  if constexpr (!F16) {
    hi = x;
    lo = u32x4{0, 0, 0, 0};
  } else {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint32_t h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = spr::f16_to_f32(static_cast<uint16_t>(w[i])), b = spr::f16_to_f32(static_cast<uint16_t>(w[i] >> 16));
      h[i] = spr::pack_bf16x2(a, b);
      l[i] = spr::pack_bf16x2(a - spr::bf16_lo(h[i]), b - spr::bf16_hi(h[i]));
    }
    hi = u32x4{h[0], h[1], h[2], h[3]};
    lo = u32x4{l[0], l[1], l[2], l[3]};
  }
}

template <bool F16>
__device__ __forceinline__ uint32_t pack_out(float a, float b) {
  if constexpr (F16) return spr::f32_to_f16(a) | static_cast<uint32_t>(spr::f32_to_f16(b)) << 16;
  return spr::pack_bf16x2(a, b);
}

// ---------------------------------------------------------------------------- few rows

constexpr int FEW_WAVES = 4;
constexpr int FEW_KEYS = 32;  // keys a wave takes at a time

// What a wave holds of its next 32 keys: codes and scales, as they come from memory.
template <int D>
struct Held {
  static constexpr int WORDS = D / 32;  // code words a lane holds of one key: D / 4 dims
  uint32_t k[2][WORDS], v[2][WORDS];
  uint32_t ks[2], vs[2];
};

// Up to 16 * NT query rows of one kv head against a share of its keys.  Grid (nsplit, kv_heads * row
// tiles, batch); each wave walks 32-key blocks of its own with its own softmax, and the four are merged
// at the end.
//
// Scores: S^T[key, row] = K Q^T by 16x16x32 MFMA.  A lane holds a quarter of one key's dims (16 bytes
// of codes for D = 128, one load), of which MFMA step s takes the s-th eight: Q is held in the same
// order of dims, so the codes go from the load to the operand with nothing but the conversion.
// Output: O^T[d, row] += V^T P^T, P straight from the accumulator: lane group g holds the keys 4g + r
// of the two 16-key tiles, and V^T is read in that order.  V passes through LDS as bf16 rows of its
// own wave (no barrier) and comes back transposed (ds_read_b64_tr_b16).  A 32-byte unit u of row r sits
// at u ^ (r & 7) (D = 128; u ^ ((r >> 1) & 3) for D = 64), its halves swapped in rows 8 .. 15: the
// transposing read of eight rows meets every bank once, and so does the write of sixteen.
template <int D, int NT, bool F16>
__global__ __launch_bounds__(64 * FEW_WAVES) void kv4_few_kernel(AttnArgs a) {
  using Part = spr::Kv4Part<D>;
  constexpr int KS = D / 32;   // MFMA steps over the dims
  constexpr int VT = D / 16;   // 16-dim tiles of the output
  constexpr int ROW = 2 * D;   // bytes of a V row in LDS
  constexpr int WORDS = Held<D>::WORDS;
  __shared__ __align__(16) uint8_t lds[FEW_WAVES * FEW_KEYS * ROW];
  __shared__ float lds_ml[FEW_WAVES][2][16];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 15, g = lane >> 4;
  const int tiles = gridDim.y / a.kv_heads;
  const int hk = blockIdx.y / tiles, tile = blockIdx.y % tiles, b = blockIdx.z, split = blockIdx.x;
  const int total_rows = a.rows * a.group;
  const Span sp = span_of(a, b);
  const int32_t* row_table = a.table + static_cast<int64_t>(sp.seq) * a.wide;

  u32x4 qh[NT][KS], ql[NT][F16 ? KS : 1];
  int32_t seen[NT];  // keys this lane's query row sees
  int32_t least = sp.length, most = 0;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int rho = tile * 16 * NT + n * 16 + m;
    const bool in = rho < total_rows;
    const int t = in ? rho / a.group : 0, h = hk * a.group + (in ? rho % a.group : 0);
    seen[n] = in ? visible_of(a, sp, t) : 0;
    if (in && t < sp.count) least = min(least, seen[n]);
    most = max(most, seen[n]);
    const uint16_t* qp = a.q + b * a.q_b + h * a.q_h + t * a.q_t + g * (D / 4);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      u32x4 x = {0, 0, 0, 0}, lo;
      if (in && t < sp.count) x = *reinterpret_cast<const u32x4*>(qp + 8 * s);
      split8<F16>(x, qh[n][s], lo);
      if constexpr (F16) ql[n][s] = lo;
    }
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    least = min(least, __shfl_xor(least, o, 64));
    most = max(most, __shfl_xor(most, o, 64));
  }
  least = __builtin_amdgcn_readfirstlane(least);
  most = __builtin_amdgcn_readfirstlane(most);

  const int blocks = (most + FEW_KEYS - 1) / FEW_KEYS;
  const int per = (blocks + a.nsplit - 1) / a.nsplit;
  const int last = min(blocks, (split + 1) * per);

  f32x4 acc[NT][VT];
  float mx[NT], sum[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    mx[n] = NEG_INF;
    sum[n] = 0.0f;
#pragma unroll
    for (int v = 0; v < VT; ++v) acc[n][v] = f32x4{0, 0, 0, 0};
  }

  const int64_t head = static_cast<int64_t>(hk) * spr::kv4_head_bytes(1 << a.log_s, D);
  auto fetch = [&](int blk, Held<D>& x) {
    const int32_t key = blk * FEW_KEYS;
    bool ok;
    const uint8_t* part = a.pages + page_offset(a, row_table, key, ok) + head;
    const int32_t slot = key & ((1 << a.log_s) - 1);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const int32_t r = slot + kt * 16 + m;
      const uint8_t* kc = part + r * Part::CODE_ROW + g * (D / 8);
      const uint8_t* vc = kc + Part::v_codes(a.log_s);
      if constexpr (D == 128) {
        const u32x4 kw = *reinterpret_cast<const u32x4*>(kc), vw = *reinterpret_cast<const u32x4*>(vc);
        x.k[kt][0] = kw.x, x.k[kt][1] = kw.y, x.k[kt][2] = kw.z, x.k[kt][3] = kw.w;
        x.v[kt][0] = vw.x, x.v[kt][1] = vw.y, x.v[kt][2] = vw.z, x.v[kt][3] = vw.w;
      } else {
        const u32x2 kw = *reinterpret_cast<const u32x2*>(kc), vw = *reinterpret_cast<const u32x2*>(vc);
        x.k[kt][0] = kw[0], x.k[kt][1] = kw[1];
        x.v[kt][0] = vw[0], x.v[kt][1] = vw[1];
      }
      const int32_t sc = r * Part::SCALE_ROW + (g * (D / 4)) / spr::KV4_GROUP;
      x.ks[kt] = part[Part::k_scales(a.log_s) + sc];
      x.vs[kt] = part[Part::v_scales(a.log_s) + sc];
      if (!ok) x.ks[kt] = 255;
    }
  };

  uint8_t* mine = lds + wave * (FEW_KEYS * ROW);
  // byte of 16-byte piece p of V row r (see above); rows r and r + 16 differ by 16 rows only
  auto piece_at = [&](int r, int p) {
    const int unit = D == 128 ? (p >> 1) ^ (r & 7) : (p >> 1) ^ ((r >> 1) & 3);
    return r * ROW + unit * 32 + ((p & 1) ^ ((r >> 3) & 1)) * 16;
  };
  // this lane's part of the transposing reads: row 4g + (m >> 2) of a 16-key tile, dims 4 (m & 3) .. of
  // 16-dim tile v
  auto tr_at = [&](int v) { return piece_at(4 * g + (m >> 2), 2 * v + ((m & 3) >> 1)) + (m & 1) * 8; };

  auto step = [&](const Held<D>& x, int32_t key, auto masked) {
    constexpr bool MASKED = decltype(masked)::value;
    f32x4 s[NT][2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const float ks = spr::kv4_scale(x.ks[kt]);
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][kt] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < WORDS; ++w) {
        const u32x4 kf = spr::kv4_eight(x.k[kt][w], ks);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          s[n][kt] = mfma16(kf, qh[n][w], s[n][kt]);
          if constexpr (F16) s[n][kt] = mfma16(kf, ql[n][w], s[n][kt]);
        }
      }
      // in a masked block a NaN V scale is kept out of the product (0 * NaN) and put in below
      const float vs = spr::kv4_scale(MASKED && x.vs[kt] == 255 ? 127 : x.vs[kt]);
#pragma unroll
      for (int w = 0; w < WORDS; ++w) {
        *reinterpret_cast<u32x4*>(mine + piece_at(kt * 16 + m, g * WORDS + w)) = spr::kv4_eight(x.v[kt][w], vs);
      }
    }
    u32x4 ph[NT], pl[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float y[8];
      float top = NEG_INF;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = s[n][e >> 2][e & 3] * a.scale_log2;
        if (MASKED && key + (e >> 2) * 16 + 4 * g + (e & 3) >= seen[n]) y[e] = NEG_INF;
        top = fmaxf(top, y[e]);
      }
      top = max_groups(top);
      if (__ballot(top > mx[n] + RESCALE_SLACK || (mx[n] == NEG_INF && top > NEG_INF)) != 0) {
        const bool grown = top > mx[n] + RESCALE_SLACK || (mx[n] == NEG_INF && top > NEG_INF);
        const float f = grown ? exp2_hw(mx[n] - top) : 1.0f;
        if (grown) mx[n] = top;
        sum[n] *= f;
#pragma unroll
        for (int v = 0; v < VT; ++v) acc[n][v] *= f;
      }
      const float off = mx[n] == NEG_INF ? 0.0f : mx[n];
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = exp2_hw(y[e] - off);
        sum[n] += p[e];
      }
      ph[n] = u32x4{spr::pack_bf16x2(p[0], p[1]), spr::pack_bf16x2(p[2], p[3]), spr::pack_bf16x2(p[4], p[5]),
                    spr::pack_bf16x2(p[6], p[7])};
      if constexpr (F16) {
        const uint32_t w[4] = {ph[n].x, ph[n].y, ph[n].z, ph[n].w};
        uint32_t l[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          l[i] = spr::pack_bf16x2(p[2 * i] - spr::bf16_lo(w[i]), p[2 * i + 1] - spr::bf16_hi(w[i]));
        }
        pl[n] = u32x4{l[0], l[1], l[2], l[3]};
      }
    }
#pragma unroll
    for (int v = 0; v < VT; ++v) {
      const u32x2 r0 = lds_read_tr16(mine + tr_at(v)), r1 = lds_read_tr16(mine + 16 * ROW + tr_at(v));
      const u32x4 vf = {r0[0], r0[1], r1[0], r1[1]};
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        acc[n][v] = mfma16(vf, ph[n], acc[n][v]);
        if constexpr (F16) acc[n][v] = mfma16(vf, pl[n], acc[n][v]);
      }
    }
    if constexpr (MASKED) {
      // V scales that are NaN: their dims of every row that sees their key
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        uint64_t nan = __ballot(x.vs[kt] == 255);
        while (nan != 0) {
          const int l = __builtin_ctzll(nan);
          nan &= nan - 1;
          const int dim0 = (l >> 4) * (D / 4);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const bool sees = key + kt * 16 + (l & 15) < seen[n];
#pragma unroll
            for (int v = 0; v < VT; ++v) {
              const bool mine_too = v * 16 >= dim0 && v * 16 < dim0 + D / 4;
              if (sees && mine_too) acc[n][v] = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
            }
          }
        }
      }
    }
  };

  int blk = split * per + wave;
  if (blk < last) {
    Held<D> now, next;
    fetch(blk, now);
    while (true) {
      const int after = blk + FEW_WAVES;
      if (after < last) fetch(after, next);
      const int32_t key = blk * FEW_KEYS;
      if (key + FEW_KEYS <= least) step(now, key, std::false_type{});
      else step(now, key, std::true_type{});
      if (after >= last) break;
      now = next;
      blk = after;
    }
  }

  // merge the waves, one 16-row tile at a time, through the V rows
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float whole = sum_groups(sum[n]);
    __syncthreads();
    if (g == 0) {
      lds_ml[wave][0][m] = mx[n];
      lds_ml[wave][1][m] = whole;
    }
    // fp32 rows of D: 16-byte piece p of row m at p ^ m
#pragma unroll
    for (int v = 0; v < VT; ++v) {
      *reinterpret_cast<f32x4*>(mine + m * (4 * D) + (((4 * v + g) ^ m) & (D / 4 - 1)) * 16) = acc[n][v];
    }
    __syncthreads();
    constexpr int PIECES = D / 4;  // 16-byte pieces of a row
    for (int i = threadIdx.x; i < 16 * PIECES; i += 64 * FEW_WAVES) {
      const int r = i / PIECES, p = i % PIECES;
      const int rho = tile * 16 * NT + n * 16 + r;
      if (rho >= total_rows) continue;
      float top = lds_ml[0][0][r];
#pragma unroll
      for (int w = 1; w < FEW_WAVES; ++w) top = fmaxf(top, lds_ml[w][0][r]);
      float l = 0.0f;
      f32x4 o = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < FEW_WAVES; ++w) {
        const float mw = lds_ml[w][0][r];
        const float f = mw == NEG_INF ? 0.0f : exp2_hw(mw - top);
        const float lw = lds_ml[w][1][r];
        const f32x4 ow = *reinterpret_cast<const f32x4*>(lds + w * (FEW_KEYS * ROW) + r * (4 * D) + ((p ^ r) & (D / 4 - 1)) * 16);
        // a wave whose scores were all NaN keeps maximum -inf and a NaN sum
        l += mw == NEG_INF ? (lw == lw ? 0.0f : lw) : f * lw;
        o += mw == NEG_INF && lw == lw ? f32x4{0, 0, 0, 0} : (mw == NEG_INF ? ow : f * ow);
      }
      const int t = rho / a.group, h = hk * a.group + rho % a.group;
      if (a.nsplit > 1) {
        const int64_t at = ((static_cast<int64_t>(b) * a.kv_heads + hk) * a.nsplit + split) * total_rows + rho;
        reinterpret_cast<f32x4*>(a.part_o + at * D)[p] = o;
        if (p == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = float2{top, l};
      } else {
        // rows out of use went through unmasked blocks like the others: nothing of that is kept
        const bool used = t < sp.count;
        if (!used) l = 0.0f;
        if (sp.broken && used) l = __builtin_nanf("");
        o = l == 0.0f ? f32x4{0, 0, 0, 0} : o * (1.0f / l);
        const int64_t at = (static_cast<int64_t>(b) * a.kv_heads * a.group + h) * a.rows + t;
        *reinterpret_cast<u32x2*>(a.out + at * D + 4 * p) = u32x2{pack_out<F16>(o[0], o[1]), pack_out<F16>(o[2], o[3])};
        if (p == 0 && a.lse != nullptr) {
          a.lse[at] = l == 0.0f ? NEG_INF : (top + __builtin_amdgcn_logf(l)) * LN2;
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------- merge of key shares

// One workgroup a row: its waves take the shares in turn, each lane D / 64 dims.
template <int D, bool F16>
__global__ __launch_bounds__(256) void kv4_merge_kernel(AttnArgs a) {
  constexpr int E = D / 64;
  __shared__ float lds[4][D];
  __shared__ float lds_l[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int total_rows = a.rows * a.group;
  const int64_t bh = blockIdx.x / total_rows;
  const int rho = blockIdx.x % total_rows;
  const int b = static_cast<int>(bh / a.kv_heads), hk = static_cast<int>(bh % a.kv_heads);
  const Span sp = span_of(a, b);
  const int64_t first = bh * a.nsplit * total_rows + rho;
  float top = NEG_INF;
  for (int s = lane; s < a.nsplit; s += 64) top = fmaxf(top, a.part_ml[(first + static_cast<int64_t>(s) * total_rows) * 2]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  float l = 0.0f, acc[E] = {};
  for (int s = wave; s < a.nsplit; s += 4) {
    const int64_t at = first + static_cast<int64_t>(s) * total_rows;
    const float ms = a.part_ml[at * 2], ls = a.part_ml[at * 2 + 1];
    if (ms == NEG_INF && ls == ls) continue;  // saw nothing
    const float f = ms == NEG_INF ? 1.0f : exp2_hw(ms - top);
    l += f * ls;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] += f * a.part_o[at * D + lane * E + e];
  }
#pragma unroll
  for (int e = 0; e < E; ++e) lds[wave][lane * E + e] = acc[e];
  if (lane == 0) lds_l[wave] = l;
  __syncthreads();
  if (wave != 0) return;
  l = lds_l[0] + lds_l[1] + lds_l[2] + lds_l[3];
  const int t = rho / a.group, h = hk * a.group + rho % a.group;
  if (t >= sp.count) l = 0.0f;
  else if (sp.broken) l = __builtin_nanf("");
  const int64_t at = (static_cast<int64_t>(b) * a.kv_heads * a.group + h) * a.rows + t;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane * E + e;
    const float o = l == 0.0f ? 0.0f : (lds[0][d] + lds[1][d] + lds[2][d] + lds[3][d]) * (1.0f / l);
    a.out[at * D + d] = F16 ? spr::f32_to_f16(o) : spr::f32_to_bf16(o);
  }
  if (lane == 0 && a.lse != nullptr) a.lse[at] = l == 0.0f ? NEG_INF : (top + __builtin_amdgcn_logf(l)) * LN2;
}

// ---------------------------------------------------------------------------- host

// Key shares of the few-row kernel: about four workgroups for every CU, none of less than four blocks
// a wave.
int32_t few_splits(int64_t groups, int64_t max_length) {
  const int64_t fill = spr::ceil_div(1024, std::max<int64_t>(groups, 1));
  const int64_t most = std::max<int64_t>(1, max_length / (4 * FEW_WAVES * FEW_KEYS));
  return static_cast<int32_t>(std::min({fill, most, int64_t{256}}));
}

template <int D, bool F16>
void launch_few(const AttnArgs& a, int nt, hipStream_t stream) {
  const int tiles = static_cast<int>(spr::ceil_div(static_cast<int64_t>(a.rows) * a.group, 16 * nt));
  const dim3 grid(a.nsplit, a.kv_heads * tiles, a.batch);
  if (nt == 1) kv4_few_kernel<D, 1, F16><<<grid, 64 * FEW_WAVES, 0, stream>>>(a);
  else kv4_few_kernel<D, 2, F16><<<grid, 64 * FEW_WAVES, 0, stream>>>(a);
}

struct Shape {
  int32_t nt;      // 16-row tiles a workgroup
  int32_t nsplit;  // key shares
};

Shape shape_of(int32_t batch, int32_t kv_heads, int32_t group, int32_t rows, int64_t max_length) {
  const int64_t total = static_cast<int64_t>(rows) * group;
  Shape s;
  s.nt = total <= 16 ? 1 : 2;
  s.nsplit = few_splits(batch * kv_heads * spr::ceil_div(total, 16 * s.nt), max_length);
  return s;
}

}  // namespace

extern "C" size_t spr_kv4_attention_workspace(int32_t batch, int32_t heads, int32_t kv_heads, int32_t rows, int32_t d,
                                              int64_t max_length) {
  if (batch <= 0 || kv_heads <= 0 || rows <= 0 || heads % kv_heads != 0) return 0;
  const Shape s = shape_of(batch, kv_heads, heads / kv_heads, rows, max_length);
  if (s.nsplit <= 1) return 0;
  return static_cast<size_t>(batch) * heads * rows * s.nsplit * (d + 2) * sizeof(float);
}

extern "C" int spr_kv4_attention(const void* q, int64_t q_b, int64_t q_h, int64_t q_t, int32_t dtype, int32_t batch,
                                 int32_t heads, int32_t kv_heads, int32_t rows, int32_t d, const uint8_t* pages,
                                 int32_t num_pages, int32_t page_size, const int32_t* block_table, int32_t sequences,
                                 int32_t wide, const int32_t* lengths, const int32_t* counts, const int32_t* seq_ids,
                                 int32_t causal, float scale, int64_t max_length, void* out, float* lse,
                                 void* workspace, size_t workspace_bytes, hipStream_t stream) {
  const char* what = "spr_kv4_attention";
  SPR_REQUIRE(dtype == 0 || dtype == 1, "%s: dtype code %d (0 bf16, 1 fp16)", what, dtype);
  SPR_REQUIRE(d == 64 || d == 128, "%s: head dim %d not supported (64, 128)", what, d);
  SPR_REQUIRE(spr::kv4_page_size_ok(page_size), "%s: page size %d (32, 64, 128 or 256)", what, page_size);
  SPR_REQUIRE(num_pages >= 1 && sequences >= 1 && wide >= 1 && static_cast<int64_t>(wide) * page_size <= INT32_MAX,
              "%s: %d pages, a block table of %d x %d", what, num_pages, sequences, wide);
  SPR_REQUIRE(batch >= 0 && batch <= 65535 && rows >= 0 && kv_heads >= 1 && heads >= 1 && heads % kv_heads == 0,
              "%s: batch %d, rows %d, %d query heads on %d kv heads", what, batch, rows, heads, kv_heads);
  SPR_REQUIRE(scale > 0.0f && scale <= 3.402823466e38f, "%s: the scale must be positive and finite", what);
  SPR_REQUIRE(max_length >= 0, "%s: max_length %lld", what, static_cast<long long>(max_length));
  SPR_REQUIRE(q_b % 8 == 0 && q_h % 8 == 0 && q_t % 8 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(pages) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0,
              "%s: Q, pages and out must be 16-byte aligned, Q's strides multiples of 8", what);
  SPR_REQUIRE(static_cast<int64_t>(rows) * (heads / kv_heads) <= (1 << 20) &&
                  static_cast<int64_t>(batch) * heads * rows <= INT32_MAX / 2,
              "%s: %d rows of %d heads in %d sequences are too many for one call", what, rows, heads, batch);
  if (batch == 0 || rows == 0) return SPR_OK;
  const int32_t group = heads / kv_heads;
  const Shape s = shape_of(batch, kv_heads, group, rows, std::min<int64_t>(max_length, static_cast<int64_t>(wide) * page_size));
  const size_t part = static_cast<size_t>(batch) * heads * rows * s.nsplit;
  if (s.nsplit > 1 && (workspace == nullptr || workspace_bytes < part * (d + 2) * sizeof(float))) {
    spr_set_error("%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, part * (d + 2) * sizeof(float));
    return SPR_EWORKSPACE;
  }
  AttnArgs a;
  a.q = static_cast<const uint16_t*>(q);
  a.pages = pages;
  a.table = block_table, a.lengths = lengths, a.counts = counts, a.seq_ids = seq_ids;
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + part * d;
  a.q_b = q_b, a.q_h = q_h, a.q_t = q_t;
  a.page_stride = kv_heads * spr::kv4_head_bytes(page_size, d);
  a.batch = batch, a.kv_heads = kv_heads, a.group = group, a.rows = rows, a.sequences = sequences, a.wide = wide;
  a.log_s = 31 - __builtin_clz(static_cast<unsigned>(page_size));
  a.num_pages = num_pages, a.nsplit = s.nsplit, a.causal = causal;
  a.scale_log2 = scale * LOG2E;
  const bool f16 = dtype == 1;
  if (d == 128) {
    if (f16) launch_few<128, true>(a, s.nt, stream);
    else launch_few<128, false>(a, s.nt, stream);
  } else {
    if (f16) launch_few<64, true>(a, s.nt, stream);
    else launch_few<64, false>(a, s.nt, stream);
  }
  SPR_LAUNCHED(what);
  if (s.nsplit > 1) {
    const unsigned rows_all = static_cast<unsigned>(static_cast<int64_t>(batch) * heads * rows);
    if (d == 128) {
      if (f16) kv4_merge_kernel<128, true><<<rows_all, 256, 0, stream>>>(a);
      else kv4_merge_kernel<128, false><<<rows_all, 256, 0, stream>>>(a);
    } else {
      if (f16) kv4_merge_kernel<64, true><<<rows_all, 256, 0, stream>>>(a);
      else kv4_merge_kernel<64, false><<<rows_all, 256, 0, stream>>>(a);
    }
    SPR_LAUNCHED(what);
  }
  return SPR_OK;
}
