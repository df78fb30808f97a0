// The product of two 8-bit matrices (spr_fp8.h), both with the summed dim along their rows:
//
//   out[m, n] = bias[n] + sum over blocks kb of 2^(sa[m, kb] + sb[n, kb] - 254) sum_{k in kb} a[m, k] b[n, k]
//
// Two ways of summing.  The codes become bf16 on their way from LDS, with their scale (the bf16 values that
// fp8_dequantize gives: exact but for scale bytes below 3 and above 246, whose values leave bf16's range), and run on
// the 16-bit matrix instruction, whose sums are fp32 throughout.  Or (fast sums, outputs in 16 bits) the scaled 8-bit
// matrix instruction (16 x 16, 128 deep) takes a block and its two scales at once, at twice the rate.  That one, like
// every instruction of this chip that multiplies 8-bit floats, adds eight neighbouring products at a time and keeps
// digits down to 2^-13 of the largest of the eight; the sums of the eights are fp32.  On normal rows the digits that it
// cuts are 5e-5 of the output's norm, a thirtieth of a bf16 output's own rounding and a quarter of an fp16 one's; an
// output whose large products cancel may lose all of it, so a caller asks for it.  32,760 x 5120 x 5120 to bf16 takes
// 1209 us with sums in fp32 and 676 with fast ones, 333 x 5000 x 4112 27 and 18, one row by 15,360 x 5120 18 and 14.
//
// Either way the sum over all blocks stays in one fp32 accumulator.  b's rows are the instruction's rows and a's its
// columns: a lane then holds four neighbours of an output row.  The order of k within a block is free as
// long as both sides have the same: lane group g (16 lanes) holds the 16-byte pieces g and g + 4.
#include "spr_elem.h"

namespace {

using spr::Elem;
using spr::f32x4;

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x8 __attribute__((ext_vector_type(8)));

constexpr int KB = 128;  // of the summed dim, one block
// An offset that no tile of a matrix reaches (256 rows of 2^22 bytes), nor with a tile's rows on it overflows.
constexpr int32_t OUTSIDE = 1 << 30;

struct Matrix {
  const uint8_t* codes;
  int64_t ld;
  const uint8_t* scales;
  int64_t scales_ld;
  int32_t shift;  // 7 where a scale is of 128 rows, else 0
  int32_t rows;
};

struct Output {
  void* out;
  const void* bias;
  int32_t bias_dtype;  // -1: none
  // Outputs that the 256 MB cache cannot hold are written past it (16 bits): 335 MB 674 instead of 684 us, but 50 MB
  // (5000 x 5000, K = 320) 42 instead of 26, with fast sums.
  bool past_caches;
};

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// A lane's 32 codes of a block, as the instruction takes them: as they are with their row's scale byte, or
// (WIDE) as four times eight bf16 values.
template <bool WIDE>
struct Operand;
template <>
struct Operand<false> {
  i32x4 v[2];
  int32_t scale;
  __device__ __forceinline__ void set(i32x4 lo, i32x4 hi, uint32_t byte) {
    v[0] = lo, v[1] = hi, scale = static_cast<int32_t>(byte);
  }
};
template <>
struct Operand<true> {
  spr::bf16x8 v[4];
  __device__ __forceinline__ void set(i32x4 lo, i32x4 hi, uint32_t byte) {
    // the conversion reads the exponent of its scale
    const float s = __uint_as_float((byte & 255u) << 23);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int32_t w0 = q < 2 ? lo[2 * q] : hi[2 * q - 4], w1 = q < 2 ? lo[2 * q + 1] : hi[2 * q - 3];
      const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, false);
      const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, true);
      const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, false);
      const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, true);
      v[q] = spr::bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
  }
};
__device__ __forceinline__ f32x4 product(const Operand<false>& n, const Operand<false>& m, f32x4 c) {
  const i32x8 a = __builtin_shufflevector(n.v[0], n.v[1], 0, 1, 2, 3, 4, 5, 6, 7);
  const i32x8 b = __builtin_shufflevector(m.v[0], m.v[1], 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, n.scale, 0, m.scale);
}
__device__ __forceinline__ f32x4 product(const Operand<true>& n, const Operand<true>& m, f32x4 c) {
#pragma unroll
  for (int q = 0; q < 4; ++q) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(n.v[q], m.v[q], c, 0, 0, 0);
  return c;
}

__device__ __forceinline__ float bias_at(const Output& o, int32_t n) {
  return o.bias_dtype == 0   ? Elem<0>::to_f(static_cast<const uint16_t*>(o.bias)[n])
         : o.bias_dtype == 1 ? Elem<1>::to_f(static_cast<const uint16_t*>(o.bias)[n])
                             : static_cast<const float*>(o.bias)[n];
}

// The bias of the four columns from n on, zeros without one and behind the last.
__device__ __forceinline__ f32x4 bias4(const Output& o, int32_t n, int32_t N) {
  f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  if (o.bias_dtype >= 0) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = n + e < N ? bias_at(o, n + e) : 0.0f;
  }
  return v;
}

// 64 columns of 16 rows: c[j] holds columns 16 j + 4 g .. + 3 of row r = lane % 16 in lane group g.  In 16 bits the
// groups first exchange them, so that a lane has 8 columns side by side and each store writes 64 bytes of a row.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
template <int DT>
__device__ __forceinline__ void put64(const Output& o, const f32x4 (&c)[4], int64_t m, bool in, int32_t n0, int32_t N,
                                      int lane) {
  using S = typename Elem<DT>::S;
  const int g = lane >> 4;
  if constexpr (DT == 2) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int32_t n = n0 + 16 * j + 4 * g;
      S* p = static_cast<S*>(o.out) + m * N + n;
      if (in && n + 4 <= N) {
        __builtin_memcpy(p, &c[j], 16);
      } else if (in) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < N) p[e] = c[j][e];
      }
    }
  } else {
    uint32_t w[4][2];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        w[j][h] = static_cast<uint32_t>(Elem<DT>::from_f(c[j][2 * h])) |
                  (static_cast<uint32_t>(Elem<DT>::from_f(c[j][2 * h + 1])) << 16);
    // groups 1, 3 of w[j] against 0, 2 of w[j + 1]: group g then has columns 8 (g / 2) + 16 (g % 2) .. + 7 of each 32
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const auto s = __builtin_amdgcn_permlane16_swap(w[j][h], w[j + 1][h], false, false);
        w[j][h] = s[0], w[j + 1][h] = s[1];
      }
    if (!in) return;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int32_t n = n0 + 32 * q + 8 * (g / 2) + 16 * (g % 2);
      S* p = static_cast<S*>(o.out) + m * N + n;
      const uint32_t v[4] = {w[2 * q][0], w[2 * q][1], w[2 * q + 1][0], w[2 * q + 1][1]};
      if (n + 8 <= N) {
        const u32x4_any all = {v[0], v[1], v[2], v[3]};
        if (o.past_caches) __builtin_nontemporal_store(all, reinterpret_cast<u32x4_any*>(p));
        else *reinterpret_cast<u32x4_any*>(p) = all;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (n + e < N) p[e] = static_cast<S>(v[e / 2] >> (e % 2 * 16));
      }
    }
  }
}

template <int DT>
__device__ __forceinline__ void put4(const Output& o, f32x4 v, int64_t m, int32_t n, int32_t N) {
  using S = typename Elem<DT>::S;
  S* p = static_cast<S*>(o.out) + m * N + n;
  const f32x4 x = v + bias4(o, n, N);
  if (n + 4 <= N) {
    S r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = Elem<DT>::from_f(x[e]);
    __builtin_memcpy(p, r, sizeof(r));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < N) p[e] = Elem<DT>::from_f(x[e]);
  }
}

// Workgroups come to the 8 XCDs in turn: each XCD gets a run of tiles, in groups of 8 tile rows, so that the
// tiles that are on it at once share their rows and columns in its L2.
template <int TM, int TN>
__device__ __forceinline__ void tile_of(int32_t tiles_m, int32_t tiles_n, int32_t& m0, int32_t& n0) {
  const int32_t tiles = tiles_m * tiles_n;
  const int32_t xcd = blockIdx.x % 8, each = tiles / 8, more = tiles % 8;
  const int32_t tile = xcd * each + (xcd < more ? xcd : more) + static_cast<int32_t>(blockIdx.x / 8);
  const int32_t group = tile / (8 * tiles_n), first = group * 8;
  const int32_t high = tiles_m - first < 8 ? tiles_m - first : 8;
  const int32_t in = tile - group * 8 * tiles_n;
  m0 = (first + in % high) * TM, n0 = in / high * TN;
}

// The scale bytes of a tile's rows for blocks kb .. kb + WIN - 1 into `win`, a dword for four blocks of a row, a
// row a thread; rows past the end as their last one.
template <int TM, int TN, int WIN, int THREADS>
__device__ __forceinline__ void fetch_scales(const Matrix& a, const Matrix& b, int32_t m0, int32_t n0, int32_t kb,
                                             int32_t blocks, uint32_t* win) {
  static_assert(WIN % 16 == 0, "16 bytes of a row at a time");
  for (int r = threadIdx.x; r < TM + TN; r += THREADS) {
    const bool is_a = r < TM;
    const int32_t row = is_a ? (m0 + r < a.rows ? m0 + r : a.rows - 1) >> a.shift
                             : (n0 + r - TM < b.rows ? n0 + r - TM : b.rows - 1) >> b.shift;
    const uint8_t* s = (is_a ? a.scales + row * a.scales_ld : b.scales + row * b.scales_ld) + kb;
    const int32_t left = blocks - kb;
    spr::Packed16 v[WIN / 16] = {};
#pragma unroll
    for (int c = 0; c < WIN / 16; ++c) {
      if (16 * c + 16 <= left) {
        __builtin_memcpy(&v[c], s + 16 * c, 16);
      } else if (16 * c < left) {  // (no branch for each byte: all in flight at once)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          v[c].w[e / 4] |= static_cast<uint32_t>(s[16 * c + e < left ? 16 * c + e : left - 1]) << (e % 4 * 8);
      }
    }
#pragma unroll
    for (int c = 0; c < WIN / 16; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) win[(4 * c + e) * (TM + TN) + r] = v[c].w[e];
  }
}

// ------------------------------------------------------------------ tiles
//
// TM x TN outputs a workgroup, WM x WN waves.  A block of both sides (128 bytes a row) goes by DMA into
// one of NBUF buffers in LDS while the products of an earlier one run; one barrier a block.  A row's 16-byte
// pieces lie at piece ^ (row % 8): eight rows' reads of one piece then meet every bank.  The scale bytes
// of the tile's rows lie in LDS for WIN blocks at a time, a dword for four blocks of a row.
//
// KG groups of such waves share one tile's blocks: a turn takes KG of them, each group one from buffers of its own,
// and the first adds the other's sums at the end.  For few tiles, where a block is a chain of its DMA, reads
// and products that one group alone leaves gaps in: 64 x 500 x 14,000 takes 25.7 us with two groups and 31.3 with one, with
// sums in fp32 42.6 and 54.8.  Where tiles are many it loses (512 x 5120 x 5120: 36 and 32, sums in fp32 54 and 50), since
// the groups wait for one another; four groups take 23.0 us on the first, but 21.4 instead of two's 19.0 on
// 300 x 1536 x 8960 (fast sums).
template <int DT, bool WIDE, int TM, int TN, int WM, int WN, int WIN, int NBUF, int KG>
__global__ __launch_bounds__(64 * WM * WN * KG) void product_kernel(Matrix a, Matrix b, int32_t K, int32_t tiles_m,
                                                              int32_t tiles_n, Output o) {
  constexpr int NW = WM * WN, THREADS = 64 * NW * KG;
  constexpr int MF = TM / WM / 16, NF = TN / WN / 16;
  constexpr int PA = TM / 8 / NW, PB = TN / 8 / NW;  // DMA instructions of a wave, 8 rows each
  static_assert(PA % 2 == 0 && PB % 2 == 0, "the DMA goes two by two");
  constexpr int BUF = (TM + TN) * KB;
  constexpr int SROWS = TM + TN;
  static_assert(KG == 1 || KG == 2, "a dword of scales is for four or two turns");
  __shared__ alignas(1024) uint8_t lds[KG * NBUF * BUF + SROWS * WIN];
  uint32_t* win = reinterpret_cast<uint32_t*>(lds + KG * NBUF * BUF);
  const int lane = threadIdx.x & 63, every = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = every / NW, wave = every % NW;
  const int wm = wave / WN, wn = wave % WN;

  int32_t m0, n0;
  tile_of<TM, TN>(tiles_m, tiles_n, m0, n0);

  const int32_t rows_m = a.rows - m0 < TM ? a.rows - m0 : TM, rows_n = b.rows - n0 < TN ? b.rows - n0 : TN;
  const auto desc_a = spr::buffer_desc(a.codes + m0 * a.ld, static_cast<int32_t>((rows_m - 1) * a.ld + K));
  const auto desc_b = spr::buffer_desc(b.codes + n0 * b.ld, static_cast<int32_t>((rows_n - 1) * b.ld + K));
  const int piece = ((lane & 7) ^ (lane >> 3)) * 16;
  const int32_t ld_a = static_cast<int32_t>(a.ld), ld_b = static_cast<int32_t>(b.ld);
  const int32_t off_a = (wave * PA * 8 + (lane >> 3)) * ld_a + piece;
  const int32_t off_b = (wave * PB * 8 + (lane >> 3)) * ld_b + piece;
  const int32_t blocks = (K + KB - 1) / KB;

  const int32_t base = spr::lds_base(lds);
  auto fetch = [&](int32_t turn, int32_t buf) {  // into buffer `buf` (an offset)
    const int32_t k = (turn * KG + kg) * KB;
    const bool in_row = k + piece < K;  // K is a multiple of 16: a piece is in or out, and what is out reads as zeros
    const int32_t va = in_row ? off_a + k : OUTSIDE, vb = in_row ? off_b + k : OUTSIDE;
#pragma unroll
    for (int i = 0; i < PA; i += 2) {
      const int32_t l = base + buf + (wave * PA + i) * 1024;
      spr::lds_dma16x2(desc_a, l, va + i * 8 * ld_a, desc_a, l + 1024, va + (i + 1) * 8 * ld_a);
    }
#pragma unroll
    for (int i = 0; i < PB; i += 2) {
      const int32_t l = base + buf + TM * KB + (wave * PB + i) * 1024;
      spr::lds_dma16x2(desc_b, l, vb + i * 8 * ld_b, desc_b, l + 1024, vb + (i + 1) * 8 * ld_b);
    }
  };

  f32x4 acc[MF][NF];
#pragma unroll
  for (int i = 0; i < MF; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  uint32_t sm[MF], sn[NF];

  // a lane's two pieces of a row: lane group g has pieces g and g + 4
  const int p0 = (lane & 15) * KB + (((lane >> 4) ^ (lane & 7)) * 16);
  const int p1 = (lane & 15) * KB + ((((lane >> 4) + 4) ^ (lane & 7)) * 16);

  Operand<WIDE> m[MF], n[NF];
  auto read = [&](int32_t turn, int32_t buf) {
    const uint8_t* at = lds + buf;
    if (turn * KG % 4 == 0) {
      const uint32_t* s = win + turn * KG % WIN / 4 * SROWS + (lane & 15);
#pragma unroll
      for (int i = 0; i < MF; ++i) sm[i] = s[wm * (TM / WM) + i * 16] >> (8 * kg);
#pragma unroll
      for (int j = 0; j < NF; ++j) sn[j] = s[TM + wn * (TN / WN) + j * 16] >> (8 * kg);
    } else {
#pragma unroll
      for (int i = 0; i < MF; ++i) sm[i] >>= 8 * KG;
#pragma unroll
      for (int j = 0; j < NF; ++j) sn[j] >>= 8 * KG;
    }
    const uint8_t* nt = at + TM * KB + wn * (TN / WN) * KB;
#pragma unroll
    for (int j = 0; j < NF; ++j)
      n[j].set(*reinterpret_cast<const i32x4*>(nt + j * 16 * KB + p0),
               *reinterpret_cast<const i32x4*>(nt + j * 16 * KB + p1), sn[j]);
    const uint8_t* mt = at + wm * (TM / WM) * KB;
#pragma unroll
    for (int i = 0; i < MF; ++i)
      m[i].set(*reinterpret_cast<const i32x4*>(mt + i * 16 * KB + p0),
               *reinterpret_cast<const i32x4*>(mt + i * 16 * KB + p1), sm[i]);
  };
  auto multiply = [&]() {
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
      for (int j = 0; j < NF; ++j) acc[i][j] = product(n[j], m[i], acc[i][j]);
  };

  const int32_t mine = kg * NBUF * BUF, turns = (blocks + KG - 1) / KG;
#pragma unroll
  for (int i = 0; i < NBUF - 1; ++i) fetch(i, mine + i * BUF);
  int32_t now = 0, next = (NBUF - 1) * BUF;  // the buffers of this turn and of the one NBUF - 1 later
  for (int32_t turn = 0; turn < turns; ++turn) {
    spr::wait_vm<(NBUF - 2) * (PA + PB)>();  // this turn's DMA has landed, those of the next NBUF - 2 may be on their way
    spr::lds_barrier();
    if (turn * KG % WIN == 0) {
      fetch_scales<TM, TN, WIN, THREADS>(a, b, m0, n0, turn * KG, blocks, win);
      spr::lds_barrier();
    }
    // the next DMA, into the buffer that all have read: with two buffers it cannot start too early (41 instead of 37 us
    // on 1024 x 5120 x 5120 behind the reads), with three the reads go first (19.0 instead of 20.6 us on 333 x 5000 x 4112;
    // both with fast sums)
    if (NBUF == 2) fetch(turn + NBUF - 1, mine + next);
    read(turn, mine + now);
    if (NBUF > 2) fetch(turn + NBUF - 1, mine + next);
    multiply();
    now = now == (NBUF - 1) * BUF ? 0 : now + BUF;
    next = next == (NBUF - 1) * BUF ? 0 : next + BUF;
  }
  spr::wait_vm<0>();  // of zeros behind the last block
  if constexpr (KG > 1) {  // the groups' sums, in their order
    static_assert((KG - 1) * MF * NF * NW * 1024 <= KG * NBUF * BUF, "the sums fit where the blocks were");
    spr::lds_barrier();
    f32x4* sums = reinterpret_cast<f32x4*>(lds) + wave * 64 + lane;
    if (kg > 0) {
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j) sums[(((kg - 1) * MF + i) * NF + j) * NW * 64] = acc[i][j];
    }
    spr::lds_barrier();
    if (kg > 0) return;
#pragma unroll
    for (int q = 0; q < KG - 1; ++q)
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j) acc[i][j] += sums[((q * MF + i) * NF + j) * NW * 64];
  }
  static_assert(NF == 4, "put64 takes 64 columns of a wave");
  const int32_t nw = n0 + wn * 64;
  f32x4 bias[NF];
#pragma unroll
  for (int j = 0; j < NF; ++j) bias[j] = bias4(o, nw + j * 16 + 4 * (lane >> 4), b.rows);
#pragma unroll
  for (int i = 0; i < MF; ++i) {
    const int32_t m = m0 + wm * (TM / WM) + i * 16 + (lane & 15);
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] += bias[j];
    put64<DT>(o, acc[i], m, m < a.rows, nw, b.rows, lane);
  }
}

// ------------------------------------------------------------------ large tiles, fast sums
//
// 256 x 256 outputs a workgroup of eight waves, 128 x 64 each, two waves a SIMD that take turns: while the
// first four read operands from LDS into registers, the other four multiply theirs, and the other way round,
// with a barrier at each change.  (With all waves in step the matrix units waited for LDS at the beginning of
// each block.)  Both groups run the same four turns a block, the second one turn later:
//   read b's rows and the first half of a's, multiply, read the second half of a's, multiply
// The first turn has twice the third one's reads, so it ends when b's are there; a's come in while the
// products begin.  A part of LDS is filled again as soon as both groups have read it: b's rows (kb + 2's) in the
// third turn, a's first half in the fourth, its second half (kb + 1's) in the first.  Each DMA has four or five
// turns to land.  (With three, and 32 x 32 x 64 instructions in half blocks, 32,760 x 5120 x 5120 took 834 us instead of 703.)
// That size takes 643 to 688 us, 2.5 to 2.7 PFLOP/s.  What bounds it is feeding the matrix units: they are busy for 63 % of
// the cycles, at the 1.9 GHz that real codes leave them (2.34 with constant ones).  Alone, the products take 400 us, with
// the LDS reads 511, with the DMA 641.  One wave a SIMD with 128 x 128 outputs, half the LDS reads, takes 761.
template <int DT>
__global__ __launch_bounds__(512) void turns_product_kernel(Matrix a, Matrix b, int32_t K, int32_t tiles_m,
                                                           int32_t tiles_n, Output o) {
  constexpr int T = 256, BUF = 2 * T * KB, SROWS = 2 * T, WIN = 64, NF = 4;
  __shared__ alignas(1024) uint8_t lds[2 * BUF + SROWS * WIN];
  uint32_t* win = reinterpret_cast<uint32_t*>(lds + 2 * BUF);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  int32_t m0, n0;
  tile_of<T, T>(tiles_m, tiles_n, m0, n0);

  const int32_t rows_m = a.rows - m0 < T ? a.rows - m0 : T, rows_n = b.rows - n0 < T ? b.rows - n0 : T;
  const auto desc_a = spr::buffer_desc(a.codes + m0 * a.ld, static_cast<int32_t>((rows_m - 1) * a.ld + K));
  const auto desc_b = spr::buffer_desc(b.codes + n0 * b.ld, static_cast<int32_t>((rows_n - 1) * b.ld + K));
  const int piece = ((lane & 7) ^ (lane >> 3)) * 16;
  const int32_t ld_a = static_cast<int32_t>(a.ld), ld_b = static_cast<int32_t>(b.ld);
  // of a's 128 rows that a half of the waves reads, the first turn takes 64 and the third 64: this wave's DMA
  // brings rows 16 (wave % 4) .. + 15 of them for wave / 4's half
  const int arow = wm * 128 + wn * 16, brow = wave * 32;
  const int32_t off_a = (arow + (lane >> 3)) * ld_a + piece, off_b = (brow + (lane >> 3)) * ld_b + piece;
  const int32_t blocks = (K + KB - 1) / KB;
  const int32_t base = spr::lds_base(lds);
  auto fetch_a = [&](int32_t kb, int half) {
    const int32_t k = kb * KB, to = base + (kb & 1) * BUF + (arow + 64 * half) * KB;
    const int32_t v = k + piece < K ? off_a + k : OUTSIDE;  // K is a multiple of 16: a piece is in or out, and
    const int32_t r = 64 * half * ld_a;                        // what is out reads as zeros
    spr::lds_dma16x2(desc_a, to, v + r, desc_a, to + 1024, v + r + 8 * ld_a);
  };
  auto fetch_b = [&](int32_t kb) {
    const int32_t k = kb * KB, to = base + (kb & 1) * BUF + (T + brow) * KB;
    const int32_t v = k + piece < K ? off_b + k : OUTSIDE;
#pragma unroll
    for (int i = 0; i < 4; i += 2)
      spr::lds_dma16x2(desc_b, to + i * 1024, v + i * 8 * ld_b, desc_b, to + (i + 1) * 1024, v + (i + 1) * 8 * ld_b);
  };

  f32x4 acc[8][NF];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  Operand<false> m[4], n[NF];
  uint32_t sm[8], sn[NF];
  const int p0 = (lane & 15) * KB + (((lane >> 4) ^ (lane & 7)) * 16);
  const int p1 = (lane & 15) * KB + ((((lane >> 4) + 4) ^ (lane & 7)) * 16);
  auto read_scales = [&](int32_t kb) {
    if (kb % 4 == 0) {
      const uint32_t* s = win + (kb % WIN) / 4 * SROWS + (lane & 15);
#pragma unroll
      for (int i = 0; i < 8; ++i) sm[i] = s[wm * 128 + i * 16];
#pragma unroll
      for (int j = 0; j < NF; ++j) sn[j] = s[T + wn * 64 + j * 16];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) sm[i] >>= 8;
#pragma unroll
      for (int j = 0; j < NF; ++j) sn[j] >>= 8;
    }
  };
  auto read_b = [&](int32_t kb) {
    const uint8_t* t = lds + (kb & 1) * BUF + (T + wn * 64) * KB;
#pragma unroll
    for (int j = 0; j < NF; ++j)
      n[j].set(*reinterpret_cast<const i32x4*>(t + j * 16 * KB + p0),
               *reinterpret_cast<const i32x4*>(t + j * 16 * KB + p1), sn[j]);
  };
  auto read_a = [&](int32_t kb, int half) {
    const uint8_t* t = lds + (kb & 1) * BUF + (wm * 128 + 64 * half) * KB;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      m[i].set(*reinterpret_cast<const i32x4*>(t + i * 16 * KB + p0),
               *reinterpret_cast<const i32x4*>(t + i * 16 * KB + p1), sm[4 * half + i]);
  };
  auto multiply = [&](int half) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < NF; ++j) acc[4 * half + i][j] = product(n[j], m[i], acc[4 * half + i][j]);
  };
  auto change = [&]() {  // nothing moves over a change of turns, the matrix instructions neither
    __builtin_amdgcn_sched_barrier(0);
    spr::lds_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };

  auto change_after_b = [&]() {  // the eight reads of a's first half may be on their way
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(8)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  fetch_scales<T, T, WIN, 512>(a, b, m0, n0, 0, blocks, win);
  fetch_b(0);
  fetch_a(0, 0);
  fetch_a(0, 1);
  fetch_b(1);
  fetch_a(1, 0);
  spr::wait_vm<8>();  // the first turn's rows
  change();
  if (wave >= 4) change();  // the second group is one turn behind
  for (int32_t k0 = 0; k0 < blocks; k0 += WIN) {
    const int32_t end = blocks - k0 < WIN ? blocks : k0 + WIN;
    if (k0 > 0) {  // (the scales in use are in registers; both groups have written before the first reads)
      fetch_scales<T, T, WIN, 512>(a, b, m0, n0, k0, blocks, win);
      change();
      change();
    }
    for (int32_t kb = k0; kb < end; ++kb) {
      fetch_a(kb + 1, 1);
      read_scales(kb);
      read_b(kb);
      __builtin_amdgcn_sched_barrier(0);
      read_a(kb, 0);
      spr::wait_vm<8>();  // a's second half of kb: behind it are kb + 1's b (4) and a's halves (2 and 2)
      change_after_b();
      multiply(0);
      change();
      fetch_b(kb + 2);
      read_a(kb, 1);
      spr::wait_vm<6>();  // kb + 1's b and a's first half: behind them are a's second (2) and kb + 2's b (4)
      change();
      fetch_a(kb + 2, 0);
      multiply(1);
      change();
    }
  }
  if (wave < 4) change();
  spr::wait_vm<0>();  // of zeros behind the last block

  const int32_t nw = n0 + wn * 64;
  f32x4 bias[NF];
#pragma unroll
  for (int j = 0; j < NF; ++j) bias[j] = bias4(o, nw + j * 16 + 4 * (lane >> 4), b.rows);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int32_t mm = m0 + wm * 128 + i * 16 + (lane & 15);
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] += bias[j];
    put64<DT>(o, acc[i], mm, mm < a.rows, nw, b.rows, lane);
  }
}

// ------------------------------------------------------------------ few rows
//
// Up to 16 MF rows of a: bound by b's bytes.  16 rows of b a workgroup, its WAVES waves take the blocks
// in turn and add their sums in LDS; both sides go straight from memory to the instruction's operands.
template <int DT, bool WIDE, int MF, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void few_rows_kernel(Matrix a, Matrix b, int32_t K, Output o) {
  constexpr int AHEAD = MF == 4 ? 2 : 4;  // blocks whose loads are in flight together
  __shared__ f32x4 part[WAVES][MF][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t n0 = blockIdx.x * 16, blocks = (K + KB - 1) / KB;
  const int32_t rows_n = b.rows - n0 < 16 ? b.rows - n0 : 16;
  const int g = lane >> 4, r = lane & 15;
  const auto desc_b = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(b.codes + n0 * b.ld), 0,
                                                        static_cast<int32_t>((rows_n - 1) * b.ld + K), 0x00020000);
  const auto desc_a = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.codes), 0,
                                                        static_cast<int32_t>((a.rows - 1) * a.ld + K), 0x00020000);
  const int32_t off_b = r * static_cast<int32_t>(b.ld) + g * 16;
  const uint8_t* sb = b.scales + ((n0 + (r < rows_n ? r : 0)) >> b.shift) * b.scales_ld;
  int32_t off_a[MF];
  const uint8_t* sa[MF];
#pragma unroll
  for (int i = 0; i < MF; ++i) {
    const int32_t m = i * 16 + r;
    off_a[i] = m * static_cast<int32_t>(a.ld) + g * 16;
    sa[i] = a.scales + ((m < a.rows ? m : 0) >> a.shift) * a.scales_ld;
  }
  f32x4 acc[MF];
#pragma unroll
  for (int i = 0; i < MF; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  // rows past the end and pieces past the summed dim read as zeros (K is a multiple of 16)
  auto load = [&](auto desc, int32_t off, int32_t k) {
    return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(desc, k < K - g * 16 ? off + k : OUTSIDE, 0, 0));
  };
  for (int32_t k0 = wave; k0 < blocks; k0 += WAVES * AHEAD) {
    i32x4 nv[AHEAD][2], mv[AHEAD][MF][2];
    uint32_t sn[AHEAD], sm[AHEAD][MF];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int32_t kb = k0 + u * WAVES, ks = kb < blocks ? kb : blocks - 1;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        nv[u][h] = load(desc_b, off_b, kb * KB + 64 * h);
#pragma unroll
        for (int i = 0; i < MF; ++i) mv[u][i][h] = load(desc_a, off_a[i], kb * KB + 64 * h);
      }
      sn[u] = sb[ks];
#pragma unroll
      for (int i = 0; i < MF; ++i) sm[u][i] = sa[i][ks];
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      Operand<WIDE> n, m;
      n.set(nv[u][0], nv[u][1], sn[u]);
#pragma unroll
      for (int i = 0; i < MF; ++i) {
        m.set(mv[u][i][0], mv[u][i][1], sm[u][i]);
        acc[i] = product(n, m, acc[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MF; ++i) part[wave][i][lane] = acc[i];
  __syncthreads();
  for (int i = wave; i < MF; i += WAVES) {
    f32x4 t = part[0][i][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) t += part[w][i][lane];
    const int32_t m = i * 16 + r, n = n0 + 4 * g;
    if (m < a.rows && n < b.rows) put4<DT>(o, t, m, n, b.rows);
  }
}

// Which kernel: by what the whole call takes, in hundredths of a microsecond, from measured times of a block
// of the summed dim while the chip is full of tiles (`full` of them), more than half full or less.  In us, outputs in
// bf16, sums in fp32 / fast, K = 5120 where none is given; of each pair the rule's pick is marked:
//                      256 x 256     128 x 128     64 x 128      64 x 64       two groups    few rows
//   1 x 5120                         43   / 26     29   / 18     22   / 13     18   / 11     10*  / 10*
//   1 x 15,360                       43   / 28     29   / 19     23   / 15*    19   / 15     19*  / 18
//   16 x 5120                        42   / 27     29   / 18     22   / 13     18   / 12*    14*  / 14
//   64 x 15,360        107  / 50     44   / 31     30   / 20     24   / 16*    20*  / 16     56
//   512 x 5120         109  / 53     47*  / 33     46   / 28*    50   / 32     54   / 36
//   1024 x 5120        108  / 53     71*  / 39*    68   / 44     77   / 50     87   / 59
//   2048 x 5120        110  / 55*    107* / 69     110  / 69     150  / 95     175  / 116
//   4096 x 5120        228  / 117    178* / 106*   226  / 140    294  / 181    346  / 230
//   32,760 x 5120      1209*/ 676*   1392 / 868    1708 / 1091   2280 / 1441   2748 / 1845
//   333 x 5000 x 4112  95   / 46     39   / 28     27*  / 18*    29   / 23     33   / 23
//   100 x 2560 x 2560  55   / 28     24   / 16     16   / 11     13   / 8      11*  / 8*
//   77 x 4096 x 4096   85   / 39     35   / 22     24   / 15     18   / 11     15*  / 10*
//   300 x 1536 x 8960  183  / 86     73   / 46     48   / 30     37   / 23     30*  / 19*
//   64 x 500 x 14,000  280  / 129    111  / 68     72   / 43     55   / 31     43   / 26*    32*
//   1000 x 1000 x 1008 27   / 16     12   / 9      9    / 7      8    / 6*     7*   / 6
//   4095 x 2560 x 2560 60   / 33*    57*  / 39     59   / 39     78   / 50     99   / 68
//   2560 x 2560 x 4096 88   / 44     56*  / 31*    68   / 38     81   / 48     94   / 60
// (fp32 outputs take up to 5 % longer than bf16 ones.)
constexpr int64_t MOST_TILES = int64_t(1) << 22;  // of a launch, below: 512 threads each, and their count is 32 bits
enum Kernel { LARGE, MIDDLE, SMALL, TINY, TINY2, FEW, NONE };
struct Cost {
  int32_t tm, tn, full, start, all, most, some;
};
Kernel pick_kernel(int64_t M, int64_t N, int32_t K, bool wide) {
  static const Cost costs[2][5] = {{{256, 256, 256, 600, 160, 130, 120},
                                    {128, 128, 512, 300, 95, 80, 70},
                                    {64, 128, 512, 200, 71, 57, 43},
                                    {64, 64, 512, 200, 55, 50, 30},
                                    {64, 64, 256, 300, 30, 29, 21}},
                                   {{256, 256, 256, 600, 287, 270, 257},
                                    {128, 128, 512, 300, 167, 169, 98},
                                    {64, 128, 512, 200, 105, 105, 70},
                                    {64, 64, 512, 200, 68, 80, 52},
                                    {64, 64, 256, 300, 38, 43, 38}}};
  const int64_t blocks = spr::ceil_div(K, KB);
  Kernel best = NONE;
  int64_t least = INT64_MAX;
  for (int i = 0; i < 5; ++i) {
    const Cost& c = costs[wide ? 1 : 0][i];
    const int64_t tiles = spr::ceil_div(M, c.tm) * spr::ceil_div(N, c.tn), rest = tiles % c.full;
    // (256 x 256 for 64 rows or columns is three quarters empty, and what no other tile takes is refused)
    if (tiles >= MOST_TILES || (i == LARGE && (M <= 64 || N <= 64))) continue;
    const int64_t cost = spr::ceil_div(tiles, c.full) * c.start +
                         blocks * (tiles / c.full * c.all + (rest == 0 ? 0 : 2 * rest > c.full ? c.most : c.some));
    if (cost < least) least = cost, best = static_cast<Kernel>(i);
  }
  // few rows: b's bytes once and a's for every 16 of b's rows, 0.15 us a MB, or the blocks that a wave takes in turn
  // (and 512 threads for 16 of b's rows, fewer than 2^32 in a launch; more than 32 rows pay beside two groups of waves only
  // where those convert to bf16: 64 x 500 x 14,000 in fp32 takes 32.0 us, with two groups 42.9)
  if (M <= (wide ? 64 : 32) && N <= (int64_t(1) << 26)) {
    const int64_t bytes = N * K / 1000 * (16 + M) / 16 * 15 / 1000;
    const int64_t turns = spr::ceil_div(blocks, 8) * (M <= 16 ? 80 : M <= 32 ? 120 : 200);
    if (400 + (bytes > turns ? bytes : turns) < least) best = FEW;
  }
  return best;
}

template <int DT, bool WIDE>
int launch_product(const Matrix& a, const Matrix& b, int32_t K, const Output& o, hipStream_t stream) {
  const int32_t M = a.rows, N = b.rows;
  const Kernel kernel = pick_kernel(M, N, K, WIDE);
  SPR_REQUIRE(kernel != NONE, "spr_fp8_matmul: too many outputs");
  if (kernel == FEW) {
    const uint32_t grid = static_cast<uint32_t>(spr::ceil_div(N, 16));
    if (M <= 16) few_rows_kernel<DT, WIDE, 1, 8><<<grid, 512, 0, stream>>>(a, b, K, o);
    else if (M <= 32) few_rows_kernel<DT, WIDE, 2, 8><<<grid, 512, 0, stream>>>(a, b, K, o);
    else if constexpr (WIDE) few_rows_kernel<DT, WIDE, 4, 8><<<grid, 512, 0, stream>>>(a, b, K, o);
    SPR_LAUNCHED("few_rows_kernel");
    return SPR_OK;
  }
  const int64_t tm = spr::ceil_div(M, kernel == LARGE ? 256 : kernel == MIDDLE ? 128 : 64);
  const int64_t tn = spr::ceil_div(N, kernel == LARGE ? 256 : kernel >= TINY ? 64 : 128);
  const uint32_t grid = static_cast<uint32_t>(tm * tn);
  const int32_t rows = static_cast<int32_t>(tm), columns = static_cast<int32_t>(tn);
  if (kernel == MIDDLE) {
    product_kernel<DT, WIDE, 128, 128, 2, 2, 32, 2, 1><<<grid, 256, 0, stream>>>(a, b, K, rows, columns, o);
  } else if (kernel == SMALL) {
    product_kernel<DT, WIDE, 64, 128, 2, 2, 32, 3, 1><<<grid, 256, 0, stream>>>(a, b, K, rows, columns, o);
  } else if (kernel == TINY) {
    product_kernel<DT, WIDE, 64, 64, 4, 1, 32, 4, 1><<<grid, 256, 0, stream>>>(a, b, K, rows, columns, o);
  } else if (kernel == TINY2) {
    product_kernel<DT, WIDE, 64, 64, 4, 1, 32, 3, 2><<<grid, 512, 0, stream>>>(a, b, K, rows, columns, o);
  } else {
    if constexpr (WIDE) product_kernel<DT, WIDE, 256, 256, 2, 4, 64, 2, 1><<<grid, 512, 0, stream>>>(a, b, K, rows, columns, o);
    else turns_product_kernel<DT><<<grid, 512, 0, stream>>>(a, b, K, rows, columns, o);
  }
  SPR_LAUNCHED("product_kernel");
  return SPR_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

extern "C" int spr_fp8_matmul_ex(const uint8_t* a, int64_t a_ld, const uint8_t* a_scales, int64_t a_scales_ld,
                                 int32_t a_square, const uint8_t* b, int64_t b_ld, const uint8_t* b_scales,
                                 int64_t b_scales_ld, int32_t b_square, int64_t M, int64_t N, int32_t K,
                                 const void* bias, int32_t bias_dtype, int32_t out_dtype, int32_t fast_sums, void* out,
                                 hipStream_t stream) {
  SPR_REQUIRE(out_dtype >= 0 && out_dtype <= 2, "spr_fp8_matmul: output dtype %d not in {0, 1, 2}", out_dtype);
  SPR_REQUIRE(fast_sums == 0 || out_dtype != 2, "spr_fp8_matmul: fast sums are for outputs in 16 bits");
  SPR_REQUIRE(bias == nullptr || (bias_dtype >= 0 && bias_dtype <= 2), "spr_fp8_matmul: bias dtype %d", bias_dtype);
  SPR_REQUIRE(M >= 0 && N >= 0 && M < (int64_t(1) << 31) - 256 && N < (int64_t(1) << 31) - 256 && K >= 0 &&
                  K % 16 == 0 && K <= (1 << 22),
              "spr_fp8_matmul: sizes %lld, %lld, %d", static_cast<long long>(M), static_cast<long long>(N), K);
  if (M == 0 || N == 0) return SPR_OK;
  SPR_REQUIRE(K > 0, "spr_fp8_matmul: nothing to sum over");
  SPR_REQUIRE(a && a_scales && b && b_scales && out, "spr_fp8_matmul: null pointer");
  SPR_REQUIRE(a_ld >= K && b_ld >= K && a_ld % 16 == 0 && b_ld % 16 == 0 && a_ld <= (1 << 22) && b_ld <= (1 << 22),
              "spr_fp8_matmul: row strides %lld, %lld", static_cast<long long>(a_ld), static_cast<long long>(b_ld));
  SPR_REQUIRE(a_scales_ld >= 0 && b_scales_ld >= 0, "spr_fp8_matmul: negative scale stride");
  SPR_REQUIRE(aligned16(a) && aligned16(b), "spr_fp8_matmul: codes must be 16-byte aligned");
  const Matrix am{a, a_ld, a_scales, a_scales_ld, a_square != 0 ? 7 : 0, static_cast<int32_t>(M)};
  const Matrix bm{b, b_ld, b_scales, b_scales_ld, b_square != 0 ? 7 : 0, static_cast<int32_t>(N)};
  const Output o{out, bias, bias == nullptr ? -1 : bias_dtype, M * N * (out_dtype == 2 ? 4 : 2) > (int64_t(256) << 20)};
  switch (out_dtype) {
    case 0: return fast_sums != 0 ? launch_product<0, false>(am, bm, K, o, stream) : launch_product<0, true>(am, bm, K, o, stream);
    case 1: return fast_sums != 0 ? launch_product<1, false>(am, bm, K, o, stream) : launch_product<1, true>(am, bm, K, o, stream);
    default: return launch_product<2, true>(am, bm, K, o, stream);
  }
}

extern "C" int spr_fp8_matmul(const uint8_t* a, int64_t a_ld, const uint8_t* a_scales, int64_t a_scales_ld,
                              int32_t a_square, const uint8_t* b, int64_t b_ld, const uint8_t* b_scales,
                              int64_t b_scales_ld, int32_t b_square, int64_t M, int64_t N, int32_t K, const void* bias,
                              int32_t bias_dtype, int32_t out_dtype, void* out, hipStream_t stream) {
  return spr_fp8_matmul_ex(a, a_ld, a_scales, a_scales_ld, a_square, b, b_ld, b_scales, b_scales_ld, b_square, M, N, K,
                           bias, bias_dtype, out_dtype, 0, out, stream);
}
