// Attention over a paged K/V cache held in 4 bits (layout: spr_kv4.h).
//
//   out[b, h, t] = softmax_j(scale * q[b, h, t] . K[j]) V[j],  lse = ln sum_j exp(scale * q . K[j])
//
// over the visible tokens j of sequence b's pages: all of them, or (causal) those up to the query's
// own, the last of the call's rows being the sequence's last token.  A row that sees nothing is 0
// with lse -inf, one that sees scores of -inf alone NaN.  The query heads of one kv head share its K
// and V: their rows, token-major, are one list of rows * group query rows.
//
// K and V values (code times scale) are exact in bf16, so the conversion to the MFMA's operand loses
// nothing; fp16 queries and probabilities go in as two bf16 terms (hi + lo) and lose at most 2^-14
// of themselves.  Scores, the running maximum and sum and the output are fp32.  bf16 calls of more than
// 8 rows round each probability to bf16 once, relative to a maximum at most 2^8 below the row's own: the
// output is off by 0.0023 of its norm where its own rounding leaves 0.0017, and a second term for the rest
// costs 25 to 38 % from 33 rows on (a frame 5.00 -> 6.90 ms).
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
  int32_t* share_out;    // the share that this call's lengths gave, for the merge
  int64_t q_b, q_h, q_t;  // strides in elements
  int64_t page_stride;    // bytes
  int32_t batch, kv_heads, group, rows, sequences, wide, log_s, num_pages, causal;
  int32_t nsplit, least_share;    // shares of the keys at most, blocks of one at least
  int32_t tile_rows, block_keys;  // query rows of a workgroup, keys of a block
  int32_t groups, chunk_cost;     // of split_cost
  int64_t merge_cost;
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

// What row t's sum of weights l stands for: rows out of use were computed beside the others, and nothing
// of that is kept (0); a row whose every score is -inf has no softmax, which only a row without keys may
// be 0 for.
__device__ __forceinline__ float sum_of(const AttnArgs& a, const Span& s, int t, float l) {
  if (t >= s.count) return 0.0f;
  return s.broken || (l == 0.0f && visible_of(a, s, t) > 0) ? __builtin_nanf("") : l;
}

// Keys that the rows [row0, row0 + tile_rows) see at most.  Rows are token-major: the last one in use
// sees most, the first one least.
__device__ __forceinline__ int32_t most_of(const AttnArgs& a, const Span& s, int row0) {
  const int32_t last = min((min(row0 + a.tile_rows, a.rows * a.group) - 1) / a.group, s.count - 1);
  return last < row0 / a.group ? 0 : visible_of(a, s, last);
}
__device__ __forceinline__ int32_t least_of(const AttnArgs& a, const Span& s, int row0) {
  return visible_of(a, s, min(row0 / a.group, max(s.count - 1, 0)));
}

// What a one-sequence call of the many-row kernel takes with its keys in n shares, in units of 50 ns.  One
// workgroup a CU, so it takes whole rounds of 256, each of them a share's chunks and two more; then the
// merge of the partial results.  Whole numbers: every workgroup has to come to the same n.
__host__ __device__ __forceinline__ uint64_t split_cost(int32_t groups, int32_t chunk_cost, int64_t merge_cost,
                                                        int32_t chunks, int32_t n) {
  const uint64_t rounds = static_cast<uint64_t>(groups * static_cast<int64_t>(n) + 255) / 256;
  const uint32_t all = static_cast<uint32_t>(chunk_cost) * static_cast<uint32_t>(chunks + 2 * n);
  const uint32_t each = all / static_cast<uint32_t>(n);
  return rounds * each + (n == 1 ? 0 : 120 + static_cast<uint64_t>(merge_cost) * n);
}
// A share has four chunks at least.
__host__ __device__ __forceinline__ bool split_fits(int32_t chunks, int32_t n) { return n == 1 || chunks >= 4 * n; }

// The largest of 64 lanes: within rows of 16 by rotations, then over the rows.
__device__ __forceinline__ uint32_t max_wave(uint32_t x) {
  auto turned = [](uint32_t v, auto ror) {
    const int w = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), decltype(ror)::value, 0xF, 0xF, false);
    return max(v, static_cast<uint32_t>(w));
  };
  x = turned(x, std::integral_constant<int, 0x128>{});
  x = turned(x, std::integral_constant<int, 0x124>{});
  x = turned(x, std::integral_constant<int, 0x122>{});
  x = turned(x, std::integral_constant<int, 0x121>{});
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return max(b[0], b[1]);
}

constexpr int32_t ONE_SHARE = 1 << 26;  // more blocks than any sequence has

// Blocks of a share of the keys, alike for all of a call's sequences, and how many the longest of them
// takes.  From the lengths as they are, not from the caller's bound, which may be the whole table: 24 heads
// on a table of 262,144, by the bound 3,600 tokens were one share of 24 workgroups, one row 31 us instead
// of 13, 128 rows 71 instead of 29, and against 20,000 tokens 74 instead of 21 and 204 instead of 55.
// COSTED: of one sequence the n <= nsplit that costs least, a lane each; else as many as there are.
// Uniform.
struct Share {
  int32_t blocks, count;
};
template <bool COSTED>
__device__ __forceinline__ Share share_of(const AttnArgs& a, int32_t length, int lane) {
  if (a.nsplit == 1) return {ONE_SHARE, 1};
  if (a.batch > 1) {
    for (int b = lane; b < a.batch; b += 64) length = max(length, span_of(a, b).length);
    length = static_cast<int32_t>(max_wave(length));
  }
  const int32_t blocks = (length + a.block_keys - 1) / a.block_keys;
  int32_t n = a.nsplit;
  if (COSTED && a.batch == 1) {
    uint32_t left = 0;  // to the most that 32 bits hold
    if (lane < a.nsplit && split_fits(blocks, lane + 1)) {
      const uint64_t cost = split_cost(a.groups, a.chunk_cost, a.merge_cost, blocks, lane + 1);
      left = cost < 0xffffffffu ? ~static_cast<uint32_t>(cost) : 1;
    }
    n = __builtin_ctzll(__ballot(left == max_wave(left))) + 1;
  }
  const int32_t share = __builtin_amdgcn_readfirstlane(max(a.least_share, (blocks + n - 1) / n));
  return {share, __builtin_amdgcn_readfirstlane(max(1, (blocks + share - 1) / share))};
}

// The keys of a tile in shares of `share` blocks: a short sequence takes one share, and that writes its
// rows straight to the output.
struct Deal {
  int32_t blocks, shares;
};
__device__ __forceinline__ Deal deal_of(const AttnArgs& a, int32_t share, int32_t keys) {
  Deal d;
  d.blocks = (keys + a.block_keys - 1) / a.block_keys;
  d.shares = max(1, (d.blocks + share - 1) / share);
  return d;
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

__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(spr::as_bf16x8(a), spr::as_bf16x8(b), c, 0, 0, 0);
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

// Up to 16 * NT query rows of one kv head against a share of its keys.  Grid (nsplit, kv_heads,
// batch); each wave walks 32-key blocks of its own with its own softmax, and the four are merged
// at the end.
//
// Scores: S^T[key, row] = K Q^T by 16x16x32 MFMA.  A lane holds a quarter of one key's dims (16 bytes
// of codes for D = 128, one load), of which MFMA step s takes the s-th eight: Q is held in the same
// order of dims, so the codes go from the load to the operand with nothing but the conversion.
// Output: O^T[d, row] += V^T P^T, P straight from the accumulator: lane group g holds the keys 4g + r
// of the two 16-key tiles, and V^T is read in that order.  V passes through LDS as bf16 rows of its
// own wave (no barrier) and comes back transposed (ds_read_b64_tr_b16).  A 32-byte unit u of row r sits
// at u ^ (r & 7) (D = 128; u ^ ((r >> 1) & 3) for D = 64), its halves swapped in rows 8 .. 15, so that
// the transposing read of eight rows meets every bank once (the writes take twice their least cycles;
// LDS is busy a third of the time).
//
// Bound by memory: one row of 24 heads against 118,800 tokens of 128 dims, 388 MB, takes 71 us, 5.5 TB/s
// (a large copy moves 4.9), and 5 us more for the merge of its 32 shares; 16 rows 74 us, 32 rows 118 (210
// registers, two waves a SIMD); 48 ragged sequences of up to 8,191 tokens, 32 heads on 8, 119 MB in 35 us; a
// short call of 301 tokens 6.2 us.  The next block's codes are in flight while one is computed, with three
// waves a SIMD (151 registers for D = 128).
//
// TWICE: at most 8 rows, each in two of the 16 columns (m and m + 8), one for the upper eight
// significant bits of its probabilities and one for the next eight, so P loses 2^-14 of itself instead of
// the 2^-8 of a rounding to bf16, for two VALU operations an element and no product more.  (As a second
// product of the remainders it cost 3 to 9 %.)
template <int D, int NT, bool F16, bool TWICE>
__global__ __launch_bounds__(64 * FEW_WAVES, NT == 1 ? 3 : 2) void kv4_few_kernel(AttnArgs a) {
  using Part = spr::Kv4Part<D>;
  constexpr int KS = D / 32;   // MFMA steps over the dims
  constexpr int VT = D / 16;   // 16-dim tiles of the output
  constexpr int ROW = 2 * D;   // bytes of a V row in LDS
  constexpr int WORDS = Held<D>::WORDS;
  __shared__ __align__(16) uint8_t lds[FEW_WAVES * FEW_KEYS * ROW];
  __shared__ float lds_ml[FEW_WAVES][2][16];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 15, g = lane >> 4;
  const int hk = blockIdx.y, b = blockIdx.z;
  // the shares turn from head to head: workgroup i runs on XCD i mod 8, so with 2, 4 or 8 shares every
  // short sequence's only one would be on the same XCDs (48 ragged sequences in 8 shares 67 us)
  const int split = (blockIdx.x + blockIdx.y + blockIdx.z) % a.nsplit;
  const int total_rows = a.rows * a.group;
  const Span sp = span_of(a, b);
  const int32_t share = share_of<false>(a, sp.length, lane).blocks;
  const Deal deal = deal_of(a, share, most_of(a, sp, 0));
  if (split >= deal.shares) return;
  const int32_t* row_table = a.table + static_cast<int64_t>(sp.seq) * a.wide;

  u32x4 qh[NT][KS], ql[NT][F16 ? KS : 1];
  int32_t seen[NT];  // keys this lane's query row sees
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int rho = TWICE ? (m & 7) : n * 16 + m;
    const bool in = rho < total_rows;
    const int t = in ? rho / a.group : 0, h = hk * a.group + (in ? rho % a.group : 0);
    seen[n] = in ? visible_of(a, sp, t) : 0;
    const uint16_t* qp = a.q + b * a.q_b + h * a.q_h + t * a.q_t + g * (D / 4);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      u32x4 x = {0, 0, 0, 0}, lo;
      if (in && t < sp.count) x = *reinterpret_cast<const u32x4*>(qp + 8 * s);
      split8<F16>(x, qh[n][s], lo);
      if constexpr (F16) ql[n][s] = lo;
    }
  }
  const int32_t least = least_of(a, sp, 0);
  const int32_t last = min(deal.blocks, (split + 1) * share);

  const uint32_t cut = TWICE && m >= 8 ? 0xffff0000u : 0u;
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
  auto fetch = [&](int blk, Held<D>& x) __attribute__((always_inline)) {
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

  auto step = [&](const Held<D>& x, int32_t key, auto masked) __attribute__((always_inline)) {
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
      // in a masked block a NaN V scale is kept out of the product (0 * NaN) and put in below; slots past
      // the sequence's end may hold any bytes
      const float vs = spr::kv4_scale(MASKED && spr::kv4_nan(x.vs[kt]) ? 127 : x.vs[kt]);
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
      if constexpr (TWICE) {
        // columns 0 .. 7 cut p to its upper bits, columns 8 .. 15 take what that leaves
        uint32_t x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = __float_as_uint(p[e] - __uint_as_float(__float_as_uint(p[e]) & cut));
        }
        ph[n] = u32x4{__builtin_amdgcn_perm(x[1], x[0], 0x07060302u), __builtin_amdgcn_perm(x[3], x[2], 0x07060302u),
                      __builtin_amdgcn_perm(x[5], x[4], 0x07060302u), __builtin_amdgcn_perm(x[7], x[6], 0x07060302u)};
        continue;
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
        if constexpr (F16 && !TWICE) acc[n][v] = mfma16(vf, pl[n], acc[n][v]);
      }
    }
    if constexpr (MASKED) {
      // V scales that are NaN: their dims of every row that sees their key
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        uint64_t nan = __ballot(spr::kv4_nan(x.vs[kt]));
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

  // blocks that every row sees whole, then the others: two loops, since one that takes either step holds
  // half as many registers again.  Two sets of registers in turn: copying the next block's to the current
  // one's cost 10 % on 48 sequences.  (Inlined by force: called, the steps keep them in scratch.)
  const int whole = min(last, least / FEW_KEYS);
  int blk = split * share + wave;
  if (blk < last) {
    Held<D> x0, x1;
    fetch(blk, x0);
    auto walk = [&](int end, auto masked) __attribute__((always_inline)) {
      while (blk < end) {
        if (blk + FEW_WAVES < last) fetch(blk + FEW_WAVES, x1);
        step(x0, blk * FEW_KEYS, masked);
        blk += FEW_WAVES;
        if (blk >= end) {
          x0 = x1;
          break;
        }
        if (blk + FEW_WAVES < last) fetch(blk + FEW_WAVES, x0);
        step(x1, blk * FEW_KEYS, masked);
        blk += FEW_WAVES;
      }
    };
    walk(whole, std::false_type{});
    walk(last, std::true_type{});
  }

  // (behind the walk: a store before it would keep the table's pages out of scalar loads, 76 -> 85 us)
  if (a.nsplit > 1 && blockIdx.x + blockIdx.y + blockIdx.z == 0 && threadIdx.x == 0) *a.share_out = share;
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
    for (int i = threadIdx.x; i < (TWICE ? 8 : 16) * PIECES; i += 64 * FEW_WAVES) {
      const int r = i / PIECES, p = i % PIECES;
      const int rho = n * 16 + r;
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
        auto row_of = [&](int c) {
          return *reinterpret_cast<const f32x4*>(lds + w * (FEW_KEYS * ROW) + c * (4 * D) + ((p ^ c) & (D / 4 - 1)) * 16);
        };
        f32x4 ow = row_of(r);
        if constexpr (TWICE) ow += row_of(r + 8);
        // a wave whose scores were all NaN keeps maximum -inf and a NaN sum
        l += mw == NEG_INF ? (lw == lw ? 0.0f : lw) : f * lw;
        o += mw == NEG_INF && lw == lw ? f32x4{0, 0, 0, 0} : (mw == NEG_INF ? ow : f * ow);
      }
      const int t = rho / a.group, h = hk * a.group + rho % a.group;
      if (deal.shares > 1) {
        const int64_t at = ((static_cast<int64_t>(b) * a.kv_heads + hk) * a.nsplit + split) * total_rows + rho;
        reinterpret_cast<f32x4*>(a.part_o + at * D)[p] = o;
        if (p == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = float2{top, l};
      } else {
        l = sum_of(a, sp, t, l);
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

// ---------------------------------------------------------------------------- many rows

constexpr int MANY_WAVES = 8;
constexpr int MANY_KEYS = 128;  // keys of a chunk
constexpr int RUN = 4;

__device__ __forceinline__ float max_xor32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_xor32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The batch entry that comes `at`-th: the longest sequences first, so that the call does not end with one
// of their shares alone on a CU (8 sequences to 9,000 tokens 215..240 -> 176 us, 5 fp16 prompts 76..87 ->
// 72..81).  Every wave ranks them itself, a lane each (more than 64 stay in order).
__device__ __forceinline__ int sequence_at(const AttnArgs& a, int at, int lane) {
  if (a.batch == 1 || a.batch > 64) return at;
  const int32_t mine = lane < a.batch ? span_of(a, lane).length : -1;
  int rank = 0;
  for (int k = 0; k < a.batch; ++k) {
    const int32_t other = __builtin_amdgcn_readlane(mine, k);
    rank += other > mine || (other == mine && k < lane) ? 1 : 0;
  }
  return __builtin_ctzll(__ballot(lane < a.batch && rank == at));
}

// 32 * RB query rows (RB 8, 4 or 2) of one kv head against a share of its keys.  One workgroup per CU,
// two waves per SIMD.  Wave w has row block w % RB and part w / RB of every chunk of 128 keys, all of
// it, 64 or 32 keys; the parts of a row block are merged at the end.
//
// A chunk is brought from its codes to bf16 once for all eight waves: a thread turns 32 values of one
// row (16 bytes of codes, one scale) into 64 bytes of a row-major LDS tile, 16 conversions and 4 writes.
// Two tiles each for K and V: the codes of chunk x + 3 are loaded and those of x + 1 written during
// chunk x, with one barrier a chunk.  Two chunks a turn of the loop, so that tiles and registers in
// flight are the same ones each time, by constant addresses (frame 5.13 -> 4.96 ms).
// Scores and output are S^T = K Q^T and O^T += V^T P^T by 32x32x16 MFMA with a lane owning one query
// row; V^T comes from the transposing read, P from the accumulator in the same order of keys.  S of the
// next 32 keys is computed beside the exponentials of the current ones.
//
// Tiles: 16-byte piece p of row r lies at p ^ (r & 15) in K and at p ^ (4 (r & 3) + (r >> 2 & 3)) in V
// (D = 128; within the eight pieces of a row for D = 64, p ^ (r >> 1 & 7) and p ^ (4 (r >> 1 & 1) +
// (r >> 2 & 3))): K's reads of 16 rows and V's transposing reads of four rows by 64 bytes each meet
// every bank once (the conversion's writes take 1.5 times their least cycles).
//
// Bound by neither unit alone: 3600 rows of 24 heads against 118,800 tokens of 128 dims, 5.26 TFLOP,
// take 5.0 to 5.2 ms, 1010 to 1050 TFLOP/s, where a library product of 8192^3 reaches 1129 on this card;
// the clock is down to 1.78 GHz, the MFMA pipe is busy half of the time, VALU issue as much.  128 rows take
// 0.225 to 0.245 ms (760 to 830 TFLOP/s): half the products to each conversion.  Row blocks by rows of the
// call, at 24 x 118,800 x 128: 33 to 64 rows 156 us with RB 2 and 200 with RB 4; 17 to 32 rows 150 us with RB 2
// and 118 with the few-row kernel.
template <int D, bool F16, int RB>
__global__ __launch_bounds__(64 * MANY_WAVES, 1) void kv4_many_kernel(AttnArgs a) {
  using Part = spr::Kv4Part<D>;
  constexpr int ROW = 2 * D;
  constexpr int TILE = MANY_KEYS * ROW;
  constexpr int KSTEPS = D / 16, DBLK = D / 32;
  constexpr int TROWS = 32 * RB;
  constexpr int PARTS = MANY_WAVES / RB;
  constexpr int HALVES = MANY_KEYS / 32 / PARTS;  // pieces of 32 keys a wave has of a chunk
  constexpr int GROUPS = D / spr::KV4_GROUP;      // scales of a row
  constexpr int ITEMS = D / 64;                   // D = 128: a thread converts K and V, D = 64: K or V
  constexpr int CONV = MANY_KEYS * GROUPS;        // items of K
  __shared__ __align__(1024) uint8_t tiles_lds[2][2][TILE];  // [K, V][chunk mod 2]
  __shared__ uint32_t v_bytes[2][MANY_KEYS];                 // the V scale bytes of every key
  __shared__ float merge_ml[MANY_WAVES][64][2];

  // runs of RUN consecutive tiles of one head and share on one XCD (workgroup b runs on XCD b mod 8):
  // they read the same codes, and shares of unlike length still spread over all XCDs
  const int total_rows = a.rows * a.group;
  const uint32_t tiles = (total_rows + TROWS - 1) / TROWS;
  const uint32_t heads = static_cast<uint32_t>(a.kv_heads) * a.batch;
  const uint32_t id = blockIdx.x / (8 * RUN) * (8 * RUN) + (blockIdx.x & 7) * RUN + (blockIdx.x >> 3) % RUN;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Share dealt = share_of<true>(a, a.batch == 1 ? span_of(a, 0).length : 0, lane);
  const int32_t share = dealt.blocks;
  // the shares that the lengths leave empty are the grid's last workgroups, not between the others (128
  // rows, 20,000 tokens on a table of 262,144: 90 -> 55 us)
  const uint32_t bhs = id / tiles, bh = bhs / dealt.count;
  const int tile = static_cast<int>(id - bhs * tiles);
  if (bh >= heads) return;
  // with few tiles a head the shares turn from head to head, as in the few-row kernel (4 sequences of 64
  // rows 59 -> 54 us); with many it would only bring some of the long ones late (13 tiles 81 -> 105 us)
  const int split = static_cast<int>((bhs + (tiles <= RUN ? bh : 0)) % dealt.count);
  const int hk = static_cast<int>(bh % a.kv_heads), b = sequence_at(a, static_cast<int>(bh / a.kv_heads), lane);

  const int col = lane & 31, half = lane >> 5;
  const int blk = wave % RB, part = wave / RB;
  const Span sp = span_of(a, b);
  const int row0 = tile * TROWS;
  const int32_t most = most_of(a, sp, row0), least = least_of(a, sp, row0);
  const Deal deal = deal_of(a, share, most);
  if (split >= deal.shares) return;
  const int32_t* row_table = a.table + static_cast<int64_t>(sp.seq) * a.wide;

  const int rho = row0 + blk * 32 + col;
  const bool in = rho < total_rows;
  const int t = in ? rho / a.group : 0, h = hk * a.group + (in ? rho % a.group : 0);
  const bool used = in && t < sp.count;
  const int32_t seen = used ? visible_of(a, sp, t) : 0;
  const int w0 = row0 + blk * 32;
  const bool wave_live = w0 < total_rows && w0 / a.group < sp.count;
  const int32_t wave_least = least_of(a, sp, w0);
  const int c0 = split * share, nch = min(deal.blocks, c0 + share) - c0;

  u32x4 qh[KSTEPS], ql[F16 ? KSTEPS : 1];
  const uint16_t* qp = a.q + b * a.q_b + h * a.q_h + t * a.q_t + half * 8;
#pragma unroll
  for (int s = 0; s < KSTEPS; ++s) {
    u32x4 lo;
    split8<F16>(used ? *reinterpret_cast<const u32x4*>(qp + 16 * s) : u32x4{0, 0, 0, 0}, qh[s], lo);
    if constexpr (F16) ql[s] = lo;
  }
  f32x16 o_acc[DBLK];
#pragma unroll
  for (int i = 0; i < DBLK; ++i) o_acc[i] = f32x16{};
  float m_run = NEG_INF, l_run = 0.0f, neg_m = 0.0f, m_thr = NEG_INF;

  // ---- codes to tiles
  const int64_t head = static_cast<int64_t>(hk) * spr::kv4_head_bytes(1 << a.log_s, D);
  const int ci = threadIdx.x & (CONV - 1);
  const int cr = (ci & 15) + 16 * (ci / (16 * GROUPS)), cg = (ci >> 4) & (GROUPS - 1);
  const int first_v = ITEMS == 1 ? threadIdx.x / CONV : 0;  // what item 0 is: K or V
  u32x4 codes[2][ITEMS];  // of the chunks mod 2 in flight
  uint32_t bytes[2][ITEMS];
  int32_t next_page = -1;
  auto look = [&](int c) {  // the page of this thread's row of chunk c
    const int32_t key = (c0 + c) * MANY_KEYS + cr;
    next_page = key < most ? row_table[key >> a.log_s] : -1;
  };
  auto fetch = [&](int c, auto par) {  // par: c mod 2
    auto& code = codes[decltype(par)::value];
    auto& byte = bytes[decltype(par)::value];
    const int32_t key = (c0 + c) * MANY_KEYS + cr;
    const bool ok = next_page >= 0 && next_page < a.num_pages;
    const uint8_t* from = a.pages + (ok ? next_page : 0) * a.page_stride + head;
    const int32_t r = key & ((1 << a.log_s) - 1);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const bool v = i + first_v != 0;
      code[i] = u32x4{0, 0, 0, 0};
      byte[i] = key < most ? 255 : 127;  // a page outside the pool is NaN; past the end nothing is read
      if (ok) {
        code[i] = *reinterpret_cast<const u32x4*>(from + (v ? Part::v_codes(a.log_s) : 0) + r * Part::CODE_ROW + cg * 16);
        byte[i] = from[(v ? Part::v_scales(a.log_s) : Part::k_scales(a.log_s)) + r * Part::SCALE_ROW + cg];
      }
    }
  };
  const int swz_k = D == 128 ? (cr & 15) : ((cr >> 1) & 7);
  const int swz_v = D == 128 ? 4 * (cr & 3) + ((cr >> 2) & 3) : 4 * ((cr >> 1) & 1) + ((cr >> 2) & 3);
  auto stash = [&](int c, auto par) {
    auto& code = codes[decltype(par)::value];
    auto& byte = bytes[decltype(par)::value];
    const int32_t end = (c0 + c + 1) * MANY_KEYS;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int v = i + first_v;
      uint8_t* to = tiles_lds[v][decltype(par)::value] + cr * ROW;
      const int x = v != 0 ? swz_v : swz_k;
      // a chunk that some row does not see whole keeps NaN V scales out of the products (0 * NaN); they
      // are put in row by row
      const float sc = spr::kv4_scale(v != 0 && spr::kv4_nan(byte[i]) && end > least ? 127 : byte[i]);
      const uint32_t w[4] = {code[i].x, code[i].y, code[i].z, code[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) *reinterpret_cast<u32x4*>(to + (((4 * cg + j) ^ x) << 4)) = spr::kv4_eight(w[j], sc);
      if (v != 0) reinterpret_cast<uint8_t*>(&v_bytes[decltype(par)::value][cr])[cg] = static_cast<uint8_t>(byte[i]);
    }
  };

  // ---- products
  const int k_x = D == 128 ? (half ^ (col & 15)) : (half ^ ((col >> 1) & 7));
  const int tr_a = lane & 3, tr_i = (lane >> 2) & 3, tr_g = (lane >> 4) & 1;
  const int v_lane = (4 * half + tr_i) * ROW + (tr_a & 1) * 8;
  const int v_piece = 2 * tr_g + (tr_a >> 1);
  const int v_x = (D == 128 ? 4 * tr_i : 4 * (tr_i >> 1)) + half;
  auto kfrag = [&](const uint8_t* kt, int hf, int s) {
    return *reinterpret_cast<const u32x4*>(kt + (hf * 32 + col) * ROW + (((2 * s) ^ k_x) << 4));
  };
  auto vfrag = [&](const uint8_t* vt, int hf, int f) {  // f = DBLK * key step + dim block
    const uint8_t* at = vt + 16 * (2 * hf + f / DBLK) * ROW + v_lane;
    const int p = 4 * (f % DBLK) + v_piece;
    const u32x2 r0 = lds_read_tr16(at + ((p ^ v_x) << 4));
    const u32x2 r1 = lds_read_tr16(at + 8 * ROW + ((p ^ v_x ^ 2) << 4));
    return u32x4{r0[0], r0[1], r1[0], r1[1]};
  };
  // mask, row maximum and lazy rescale of the 32 keys from `key` on
  auto row_max = [&](f32x16& acc, int32_t key) {
    if (key + 32 > wave_least) {
      const int lim = seen - key - 4 * half;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if (8 * (e / 4) + (e % 4) >= lim) acc[e] = NEG_INF;
      }
    }
    float mx = NEG_INF;
#pragma unroll
    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, acc[e]);
    const float mloc = max_xor32(mx) * a.scale_log2;
    const bool up = mloc > m_thr;
    if (__ballot(up) != 0) {
      // only the rows whose maximum grew move theirs: a row's result does not depend on its wave's
      const float m_new = up ? mloc : m_run;
      const float f = up ? exp2_hw(m_run - m_new) : 1.0f;
      l_run *= f;
#pragma unroll
      for (int i = 0; i < DBLK; ++i) o_acc[i] *= f;
      m_run = m_new;
      m_thr = m_new + RESCALE_SLACK;
      neg_m = m_new == NEG_INF ? 0.0f : -m_new;
    }
  };
  // S of 32 keys (piece hf_n of kt) into acc_next beside the exponentials of acc, as far as asked for;
  // then O += P V (piece hf of vt)
  auto step = [&](auto with_s, auto with_p, f32x16& acc_next, const uint8_t* kt, int hf_n, const f32x16& acc, const uint8_t* vt, int hf) {
    constexpr bool S = decltype(with_s)::value, P = decltype(with_p)::value;
    uint32_t ph[2][4], pl[2][4];
    float sum0 = 0.0f, sum1 = 0.0f;
    if constexpr (S) acc_next = f32x16{};
    constexpr int EACH = 16 / KSTEPS;  // elements of P beside each step of S
    u32x4 ka[3];
    if constexpr (S) {
      ka[0] = kfrag(kt, hf_n, 0);
      ka[1] = kfrag(kt, hf_n, 1);
    }
#pragma unroll
    for (int st = 0; st < KSTEPS; ++st) {
      if constexpr (S) {
        if (st + 2 < KSTEPS) ka[(st + 2) % 3] = kfrag(kt, hf_n, st + 2);
        acc_next = mfma32(ka[st % 3], qh[st], acc_next);
        if constexpr (F16) acc_next = mfma32(ka[st % 3], ql[st], acc_next);
      }
      if constexpr (P) {
#pragma unroll
        for (int e = EACH * st; e < EACH * (st + 1); e += 2) {
          const float p0 = exp2_hw(__builtin_fmaf(acc[e], a.scale_log2, neg_m));
          const float p1 = exp2_hw(__builtin_fmaf(acc[e + 1], a.scale_log2, neg_m));
          const uint32_t w = spr::pack_bf16x2(p0, p1);
          sum0 += p0;
          sum1 += p1;
          ph[e / 8][(e % 8) / 2] = w;
          if constexpr (F16) pl[e / 8][(e % 8) / 2] = spr::pack_bf16x2(p0 - spr::bf16_lo(w), p1 - spr::bf16_hi(w));
        }
      }
    }
    if constexpr (P) {
      l_run += sum0 + sum1;
      u32x4 va[3];
      va[0] = vfrag(vt, hf, 0);
      va[1] = vfrag(vt, hf, 1);
#pragma unroll
      for (int f = 0; f < 2 * DBLK; ++f) {
        if (f + 2 < 2 * DBLK) va[(f + 2) % 3] = vfrag(vt, hf, f + 2);
        const int k = f / DBLK;
        o_acc[f % DBLK] = mfma32(va[f % 3], u32x4{ph[k][0], ph[k][1], ph[k][2], ph[k][3]}, o_acc[f % DBLK]);
        if constexpr (F16) o_acc[f % DBLK] = mfma32(va[f % 3], u32x4{pl[k][0], pl[k][1], pl[k][2], pl[k][3]}, o_acc[f % DBLK]);
      }
    }
  };
  // NaN V scales of a chunk that some row does not see whole: their dims of the rows that see the key
  auto put_nan = [&](int c) {
    const int32_t first = (c0 + c) * MANY_KEYS;
    if (first + MANY_KEYS <= least) return;
#pragma unroll
    for (int k0 = 0; k0 < MANY_KEYS; k0 += 64) {
      const uint32_t w = v_bytes[c & 1][k0 + lane];
      uint32_t mine = 0;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) mine |= spr::kv4_nan((w >> (8 * g)) & 255) ? 1u << g : 0;
      uint64_t keys = __ballot(mine != 0);
      while (keys != 0) {
        const int k = __builtin_ctzll(keys);
        keys &= keys - 1;
        const uint32_t groups = __builtin_amdgcn_readlane(mine, k);
        if ((k0 + k) / (32 * HALVES) != part) continue;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          if (((groups >> g) & 1) != 0 && first + k0 + k < seen) {
#pragma unroll
            for (int e = 0; e < 16; ++e) o_acc[g][e] = __builtin_nanf("");
          }
        }
      }
    }
  };

  if (nch > 0) {
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    constexpr std::integral_constant<int, 0> even{};
    constexpr std::integral_constant<int, 1> odd{};
    look(0), fetch(0, even), look(1);
    fetch(1, odd), look(2);
    stash(0, even);
    fetch(2, even), look(3);
    // the two waves of a SIMD (w and w + 4) convert at opposite ends of a chunk: one's conversions run
    // beside the other's products (frame 5.30 -> 5.24 ms)
    auto refill = [&](int x, auto par) {  // par: (x + 1) mod 2
      if (x + 1 < nch) {
        stash(x + 1, par);
        fetch(x + 3, par);
        look(x + 4);
      }
    };
    f32x16 s[2];
    auto chunk = [&](int x, auto par) {  // par: (x + 1) mod 2
      spr::lds_barrier();  // chunk x is written; nobody reads chunk x - 1 any more
      constexpr int BUF = 1 - decltype(par)::value;
      const uint8_t *kt = tiles_lds[0][BUF], *vt = tiles_lds[1][BUF];
      const int32_t key = (c0 + x) * MANY_KEYS + part * (32 * HALVES);
      const int h0 = part * HALVES;
      if (wave >= 4) refill(x, par);
      if (wave_live) {
        step(yes, no, s[0], kt, h0, s[1], vt, h0);
#pragma unroll
        for (int i = 0; i < HALVES; ++i) {
          row_max(s[i & 1], key + 32 * i);
          if (i + 1 < HALVES) step(yes, yes, s[(i + 1) & 1], kt, h0 + i + 1, s[i & 1], vt, h0 + i);
          else step(no, yes, s[(i + 1) & 1], kt, h0, s[i & 1], vt, h0 + i);
        }
        put_nan(x);
      }
      if (wave < 4) refill(x, par);
    };
    for (int x = 0; x < nch; x += 2) {
      chunk(x, odd);
      if (x + 1 < nch) chunk(x + 1, even);
    }
  }

  if (a.nsplit > 1 && blockIdx.x == 0 && threadIdx.x == 0) *a.share_out = share;
  float l_tot = sum_xor32(l_run);
  if constexpr (PARTS > 1) {
    // the other parts hand (m, l, O) to part 0 through the tiles: 32 rows of D floats each
    __syncthreads();
    float* po = reinterpret_cast<float*>(&tiles_lds[0][0][0]);
    if (part > 0) {
      float* mine = po + (wave - RB) * (32 * D);
#pragma unroll
      for (int i = 0; i < DBLK; ++i) {
#pragma unroll
        for (int e = 0; e < 16; ++e) mine[(i * 16 + e) * 64 + lane] = o_acc[i][e];
      }
      merge_ml[wave][lane][0] = m_run;
      merge_ml[wave][lane][1] = l_tot;
    }
    __syncthreads();
    if (part > 0) return;
    float top = m_run;
#pragma unroll
    for (int p = 1; p < PARTS; ++p) top = fmaxf(top, merge_ml[wave + p * RB][lane][0]);
    // one without a maximum has no sum (or NaN)
    const float f0 = m_run == NEG_INF ? 1.0f : exp2_hw(m_run - top);
    l_tot *= f0;
#pragma unroll
    for (int i = 0; i < DBLK; ++i) o_acc[i] *= f0;
#pragma unroll
    for (int p = 1; p < PARTS; ++p) {
      const float m1 = merge_ml[wave + p * RB][lane][0], f1 = m1 == NEG_INF ? 1.0f : exp2_hw(m1 - top);
      const float* theirs = po + (wave + (p - 1) * RB) * (32 * D);
      l_tot += merge_ml[wave + p * RB][lane][1] * f1;
#pragma unroll
      for (int i = 0; i < DBLK; ++i) {
#pragma unroll
        for (int e = 0; e < 16; ++e) o_acc[i][e] += theirs[(i * 16 + e) * 64 + lane] * f1;
      }
    }
    m_run = top;
  }
  if (!in) return;
  if (deal.shares > 1) {
    const int64_t at = ((static_cast<int64_t>(b) * a.kv_heads + hk) * a.nsplit + split) * total_rows + rho;
#pragma unroll
    for (int i = 0; i < DBLK; ++i) {
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        *reinterpret_cast<f32x4*>(a.part_o + at * D + i * 32 + 2 * e + 4 * half) =
            f32x4{o_acc[i][e], o_acc[i][e + 1], o_acc[i][e + 2], o_acc[i][e + 3]};
      }
    }
    if (half == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = float2{m_run, l_tot};
    return;
  }
  l_tot = sum_of(a, sp, t, l_tot);
  const float inv = 1.0f / l_tot;
  const int64_t at = (static_cast<int64_t>(b) * a.kv_heads * a.group + h) * a.rows + t;
#pragma unroll
  for (int i = 0; i < DBLK; ++i) {
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      u32x2 w = {0, 0};
      if (l_tot != 0.0f) {
        w = u32x2{pack_out<F16>(o_acc[i][e] * inv, o_acc[i][e + 1] * inv),
                  pack_out<F16>(o_acc[i][e + 2] * inv, o_acc[i][e + 3] * inv)};
      }
      *reinterpret_cast<u32x2*>(a.out + at * D + i * 32 + 2 * e + 4 * half) = w;
    }
  }
  if (half == 0 && a.lse != nullptr) {
    a.lse[at] = l_tot == 0.0f ? NEG_INF : (m_run + __builtin_amdgcn_logf(l_tot)) * LN2;
  }
}

// ---------------------------------------------------------------------------- merge of key shares

// 16 lanes have all dims of a row, and P such teams share a row's shares; 16 / P rows a workgroup.
// Bound by latency where rows are few (24 rows of 32 shares 5 us), by the partial results' bytes where
// they are many (86,400 rows of 7 shares, 310 MB, 64 us).  The share is the attention kernel's.
template <int D, bool F16, int P>
__global__ __launch_bounds__(256) void kv4_merge_kernel(AttnArgs a, int64_t all_rows) {
  constexpr int E = D / 16;  // dims of a lane
  __shared__ float lds[P > 1 ? 16 : 1][D + 1];
  const int lane = threadIdx.x & 15, team = threadIdx.x >> 4;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (16 / P) + team / P;
  const int total_rows = a.rows * a.group;
  const bool in = row < all_rows;
  const int64_t bh = in ? row / total_rows : 0;
  const int rho = static_cast<int>(in ? row % total_rows : 0);
  const int b = static_cast<int>(bh / a.kv_heads), hk = static_cast<int>(bh % a.kv_heads);
  const Span sp = span_of(a, b);
  const int32_t shares = in ? deal_of(a, *a.share_out, most_of(a, sp, rho / a.tile_rows * a.tile_rows)).shares : 1;
  if (P == 1 && shares == 1) return;  // written already, or no row
  const int64_t first = bh * a.nsplit * total_rows + rho;
  float top = NEG_INF;
  float l = 0.0f, acc[E] = {};
  if (shares > 1) {
    for (int s = lane; s < shares; s += 16) top = fmaxf(top, a.part_ml[(first + static_cast<int64_t>(s) * total_rows) * 2]);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 16));
#pragma unroll 4
    for (int s = team % P; s < shares; s += P) {
      const int64_t at = first + static_cast<int64_t>(s) * total_rows;
      const float ms = a.part_ml[at * 2];
      // a share without a maximum saw nothing (or only NaN): its sums count as they are, zeros (or NaN)
      const float f = ms == NEG_INF ? 1.0f : exp2_hw(ms - top);
      l += f * a.part_ml[at * 2 + 1];
      const f32x4* o = reinterpret_cast<const f32x4*>(a.part_o + at * D + lane * E);
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        const f32x4 x = o[e / 4];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[e + i] += f * x[i];
      }
    }
  }
  if constexpr (P > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) lds[team][lane * E + e] = acc[e];
    if (lane == 0) lds[team][D] = l;
    __syncthreads();
    if (team % P != 0 || shares == 1) return;
#pragma unroll
    for (int w = 1; w < P; ++w) {
      l += lds[team + w][D];
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += lds[team + w][lane * E + e];
    }
  }
  const int t = rho / a.group, h = hk * a.group + rho % a.group;
  l = sum_of(a, sp, t, l);
  const int64_t at = (static_cast<int64_t>(b) * a.kv_heads * a.group + h) * a.rows + t;
  const float inv = 1.0f / l;
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    u32x2 w = {0, 0};
    if (l != 0.0f) w = u32x2{pack_out<F16>(acc[e] * inv, acc[e + 1] * inv), pack_out<F16>(acc[e + 2] * inv, acc[e + 3] * inv)};
    *reinterpret_cast<u32x2*>(a.out + at * D + lane * E + e) = w;
  }
  if (lane == 0 && a.lse != nullptr) a.lse[at] = l == 0.0f ? NEG_INF : (top + __builtin_amdgcn_logf(l)) * LN2;
}

// ---------------------------------------------------------------------------- host

// How a call is cut up: by the few-row kernel in 16 * nt rows, or by the many-row one in 64, 128 or 256
// rows, and the keys in at most nsplit shares.
struct Shape {
  int32_t nt;           // 0: the many-row kernel
  int32_t rb;           // its row blocks of 32
  int32_t fill;         // shares of a sequence of any length
  int32_t nsplit;       // and of one within max_length
  int32_t least_share;  // blocks of a share at least
  int64_t groups;       // workgroups to a share
  int32_t chunk_cost;   // of split_cost
  int64_t merge_cost;
};

Shape shape_of(int32_t batch, int32_t kv_heads, int32_t group, int32_t rows, int32_t d, bool f16, int64_t max_length) {
  max_length = std::min(max_length, spr::KV4_MOST_TOKENS);
  const int64_t total = static_cast<int64_t>(rows) * group, heads = static_cast<int64_t>(batch) * kv_heads;
  Shape s = {};
  auto within = [&](int64_t block_keys) {  // shares that sequences of max_length can take
    const int64_t shares = spr::ceil_div(std::max<int64_t>(max_length, 1), block_keys * s.least_share);
    return static_cast<int32_t>(std::min<int64_t>(s.fill, shares));
  };
  if (total <= 32) {
    s.nt = total <= 16 ? 1 : 2;
    s.groups = heads;
    // Three workgroups for every CU, in one round, where there is one sequence; two rounds where there are
    // several, whose lengths are not known here, so that long ones are dealt finer (48 ragged ones in one
    // round 55 us, in two 36; 16 alike 31 and 34).  None of less than four blocks a wave.
    s.fill = static_cast<int32_t>(std::min<int64_t>(std::max<int64_t>(1, (batch == 1 ? 768 : 1536) / s.groups), 256));
    s.least_share = 4 * FEW_WAVES;
    s.nsplit = within(FEW_KEYS);
    return s;
  }
  s.rb = total <= 64 ? 2 : total <= 128 ? 4 : 8;
  s.groups = heads * spr::ceil_div(total, 32 * s.rb);
  s.least_share = 4;
  if (batch > 1) {
    s.fill = static_cast<int32_t>(std::min<int64_t>(std::max<int64_t>(1, 1024 / s.groups), 64));
    s.nsplit = within(MANY_KEYS);
    return s;
  }
  // the shares that come out fastest, at what a chunk takes (256 workgroups on K and V of their own, 8,192
  // and 24,576 keys; units of 50 ns) and 4 TB/s for the partial results
  constexpr int32_t chunk[2][2][3] = {{{20, 30, 50}, {24, 41, 77}},  // [D 64, 128][bf16, fp16][RB 2, 4, 8]
                                      {{31, 47, 80}, {43, 74, 142}}};
  s.chunk_cost = chunk[d == 128 ? 1 : 0][f16 ? 1 : 0][s.rb == 8 ? 2 : s.rb == 4 ? 1 : 0];
  s.merge_cost = heads * total * d / 25000;
  const int32_t groups = static_cast<int32_t>(std::min<int64_t>(s.groups, INT32_MAX));
  auto best = [&](int64_t length) {
    const int32_t chunks = static_cast<int32_t>(std::max<int64_t>(1, spr::ceil_div(length, MANY_KEYS)));
    int32_t at = 1;
    uint64_t least = split_cost(groups, s.chunk_cost, s.merge_cost, chunks, 1);
    for (int32_t n = 2; n <= 64 && split_fits(chunks, n); ++n) {
      const uint64_t cost = split_cost(groups, s.chunk_cost, s.merge_cost, chunks, n);
      if (cost < least) least = cost, at = n;
    }
    return at;
  };
  s.fill = best(spr::KV4_MOST_TOKENS);
  s.nsplit = best(max_length);
  return s;
}

template <int D, bool F16>
void launch(const AttnArgs& a, const Shape& s, hipStream_t stream) {
  if (s.nt != 0) {
    const dim3 grid(a.nsplit, a.kv_heads, a.batch);
    const int64_t total = static_cast<int64_t>(a.rows) * a.group;
    if (total <= 8) kv4_few_kernel<D, 1, F16, true><<<grid, 64 * FEW_WAVES, 0, stream>>>(a);
    else if (s.nt == 1) kv4_few_kernel<D, 1, F16, false><<<grid, 64 * FEW_WAVES, 0, stream>>>(a);
    else kv4_few_kernel<D, 2, F16, false><<<grid, 64 * FEW_WAVES, 0, stream>>>(a);
  } else {
    const unsigned grid = static_cast<unsigned>(spr::ceil_div(s.groups * s.nsplit, 8 * RUN) * (8 * RUN));
    if (s.rb == 8) kv4_many_kernel<D, F16, 8><<<grid, 64 * MANY_WAVES, 0, stream>>>(a);
    else if (s.rb == 4) kv4_many_kernel<D, F16, 4><<<grid, 64 * MANY_WAVES, 0, stream>>>(a);
    else kv4_many_kernel<D, F16, 2><<<grid, 64 * MANY_WAVES, 0, stream>>>(a);
  }
  if (s.nsplit > 1) {
    const int64_t rows = static_cast<int64_t>(a.batch) * a.kv_heads * a.group * a.rows;
    // as many teams to a row as a long sequence has shares and there is room for on the card (200 rows of
    // 4 heads 37 us by teams of 16, 35 by 4; 72 rows of 30 shares 23 and 27)
    const unsigned all = static_cast<unsigned>(rows);
    if (s.fill >= 16 && rows <= 512) kv4_merge_kernel<D, F16, 16><<<all, 256, 0, stream>>>(a, rows);
    else if (s.fill >= 4 && rows <= 16384) kv4_merge_kernel<D, F16, 4><<<(all + 3) / 4, 256, 0, stream>>>(a, rows);
    else kv4_merge_kernel<D, F16, 1><<<(all + 15) / 16, 256, 0, stream>>>(a, rows);
  }
}

// `part` partial rows, their (maximum, sum) and the share.
size_t workspace_bytes_of(size_t part, int32_t d) { return part * (d + 2) * sizeof(float) + 16; }

}  // namespace

extern "C" size_t spr_kv4_attention_workspace(int32_t batch, int32_t heads, int32_t kv_heads, int32_t rows, int32_t d,
                                              int64_t max_length) {
  if (batch <= 0 || kv_heads <= 0 || rows <= 0 || heads % kv_heads != 0) return 0;
  int32_t nsplit = 1;  // of either type
  for (bool f16 : {false, true}) {
    nsplit = std::max(nsplit, shape_of(batch, kv_heads, heads / kv_heads, rows, d, f16, max_length).nsplit);
  }
  return nsplit == 1 ? 0 : workspace_bytes_of(static_cast<size_t>(batch) * heads * rows * nsplit, d);
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
  SPR_REQUIRE(num_pages >= 1 && sequences >= 1 && wide >= 1 && static_cast<int64_t>(wide) * page_size <= spr::KV4_MOST_TOKENS,
              "%s: %d pages, a block table of %d x %d", what, num_pages, sequences, wide);
  SPR_REQUIRE(batch >= 0 && batch <= 65535 && rows >= 0 && kv_heads >= 1 && kv_heads <= 65535 && heads >= 1 && heads % kv_heads == 0,
              "%s: batch %d, rows %d, %d query heads on %d kv heads", what, batch, rows, heads, kv_heads);
  SPR_REQUIRE(scale > 0.0f && scale <= 1e38f, "%s: the scale must be positive and at most 1e38", what);
  SPR_REQUIRE(max_length >= 0, "%s: max_length %lld", what, static_cast<long long>(max_length));
  SPR_REQUIRE(q_b % 8 == 0 && q_h % 8 == 0 && q_t % 8 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(pages) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0,
              "%s: Q, pages and out must be 16-byte aligned, Q's strides multiples of 8", what);
  SPR_REQUIRE(static_cast<int64_t>(rows) * (heads / kv_heads) <= (1 << 20) &&
                  static_cast<int64_t>(batch) * heads * rows <= INT32_MAX / 2,
              "%s: %d rows of %d heads in %d sequences are too many for one call", what, rows, heads, batch);
  if (batch == 0 || rows == 0) return SPR_OK;
  const int32_t group = heads / kv_heads;
  // as the workspace query, which does not know the table
  const Shape s = shape_of(batch, kv_heads, group, rows, d, dtype == 1, max_length);
  // a launch has fewer than 2^32 threads in x (8 * RUN workgroups of 512 spare: the grid is rounded up)
  SPR_REQUIRE(s.nt != 0 || s.groups * s.nsplit <= 0xffffffffll / (64 * MANY_WAVES) - 8 * RUN,
              "%s: %d rows of %d heads in %d sequences are too many for one call", what, rows, heads, batch);
  const size_t part = static_cast<size_t>(batch) * heads * rows * s.nsplit;
  if (s.nsplit > 1 && (workspace == nullptr || workspace_bytes < workspace_bytes_of(part, d))) {
    spr_set_error("%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, workspace_bytes_of(part, d));
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
  a.share_out = reinterpret_cast<int32_t*>(a.part_ml + part * 2);
  a.q_b = q_b, a.q_h = q_h, a.q_t = q_t;
  a.page_stride = kv_heads * spr::kv4_head_bytes(page_size, d);
  a.batch = batch, a.kv_heads = kv_heads, a.group = group, a.rows = rows, a.sequences = sequences, a.wide = wide;
  a.log_s = 31 - __builtin_clz(static_cast<unsigned>(page_size));
  a.num_pages = num_pages, a.causal = causal;
  a.nsplit = s.nsplit, a.least_share = s.least_share;
  a.groups = static_cast<int32_t>(std::min<int64_t>(s.groups, INT32_MAX));
  a.chunk_cost = s.chunk_cost, a.merge_cost = s.merge_cost;
  a.block_keys = s.nt != 0 ? FEW_KEYS : MANY_KEYS;
  a.tile_rows = s.nt != 0 ? 16 * s.nt : 32 * s.rb;
  a.scale_log2 = scale * LOG2E;
  if (d == 128) {
    if (dtype == 1) launch<128, true>(a, s, stream);
    else launch<128, false>(a, s, stream);
  } else {
    if (dtype == 1) launch<64, true>(a, s, stream);
    else launch<64, false>(a, s, stream);
  }
  SPR_LAUNCHED(what);
  return SPR_OK;
}
