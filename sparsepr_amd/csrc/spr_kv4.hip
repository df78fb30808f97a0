// Pages of a 4-bit K/V cache (layout: spr_kv4.h): rows stored and loaded, pages reserved, freed,
// forked, copied and moved together.
//
// The page numbers live on the device: block_table int32 [sequences, wide] (-1: none), lengths int32
// [sequences] and ref_count int32 [pages] (the sequences that hold a page; 0 is free).  A call checks
// all it is asked for on the device before it changes anything, so it happens whole or not at all,
// with no host synchronisation; what was wrong is left in `status`.  New pages are the lowest free
// ones in ascending order, whatever the order of the free calls before: no free list, and the same
// calls give the same numbers.
#include <algorithm>
#include <type_traits>

#include "spr_kv4.h"

namespace {

using spr::u32x4;

// What a page call found wrong (status, kept until the caller clears it).
enum {
  KV4_OK = 0,
  KV4_BAD_SEQUENCE = 1,   // a sequence number outside the table
  KV4_REPEATED = 2,       // a sequence named twice
  KV4_BAD_COUNT = 3,      // a negative count or one past `most`, or a range outside the sequence's pages
  KV4_TABLE_FULL = 4,     // more tokens than a row of the table has pages for
  KV4_NO_PAGES = 5,       // not enough free pages
  KV4_NOT_EMPTY = 6,      // a fork onto a sequence that holds tokens
  KV4_BAD_LENGTH = 7,     // a length outside the table, or a table entry outside the pool
};

// ---------------------------------------------------------------------------- rows

// Where row t of batch entry b lies: the offset of its page, or -1.  The slot in the page goes to `slot`.
__device__ __forceinline__ int64_t page_of_row(const int32_t* table, const int32_t* seq_ids, const int32_t* starts,
                                               int b, int t, int32_t sequences, int32_t wide, int log_s,
                                               int32_t num_pages, int32_t& slot) {
  const int32_t seq = seq_ids != nullptr ? seq_ids[b] : b;
  const int32_t first = starts[b];
  const int64_t pos = static_cast<int64_t>(first) + t;
  slot = static_cast<int32_t>(pos & ((1 << log_s) - 1));
  if (seq < 0 || seq >= sequences || first < 0 || (pos >> log_s) >= wide) return -1;
  const int32_t page = table[static_cast<int64_t>(seq) * wide + (pos >> log_s)];
  return page >= 0 && page < num_pages ? page : -1;
}

struct RowArgs {
  const int32_t *table, *seq_ids, *starts, *counts;
  int32_t sequences, wide, log_s, num_pages, kv_heads, rows;
  int64_t page_stride;  // bytes
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const u32x4 a = reinterpret_cast<const u32x4*>(p)[0], b = reinterpret_cast<const u32x4*>(p)[1];
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
  } else {
    const u32x4 a = *reinterpret_cast<const u32x4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (__is_same(T, _Float16)) {
        x[2 * i] = spr::f16_to_f32(static_cast<uint16_t>(w[i]));
        x[2 * i + 1] = spr::f16_to_f32(static_cast<uint16_t>(w[i] >> 16));
      } else {
        x[2 * i] = spr::bf16_lo(w[i]);
        x[2 * i + 1] = spr::bf16_hi(w[i]);
      }
    }
  }
}

// The larger of v over the four lanes that hold one group of 32 dims (DPP quad permutes).
__device__ __forceinline__ uint32_t max_quad(uint32_t v) {
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0xB1, 0xF, 0xF, false)));
  return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x4E, 0xF, 0xF, false)));
}

// Eight values of a group to a code word and the group's scale byte.  The scale's exponent is that
// of the group's largest magnitude rounded to two significant bits (half up), less two: the largest
// value then lies in [3.5, 7) times the scale, so it is off by at most one unit of it, where the
// exponent of the unrounded magnitude would leave (7, 8) to be cut to 6.  Values round to the nearest
// code, of two equally near ones to the even one, in the conversion.  The byte stays in [2, 252],
// where every value is a normal finite bf16.  A group with an infinity or a NaN is NaN.
__device__ __forceinline__ uint32_t encode8(const float (&x)[8], uint32_t& byte) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  top = max_quad(top);
  byte = min(max(static_cast<int>((top + 0x200000u) >> 23) - 2, 2), 252);
  const float s = spr::kv4_scale(byte);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
  if (top >= 0x7f800000u) byte = 255, w = 0;
  return w;
}

constexpr int ROW_THREADS = 256;
constexpr int64_t MOST_BLOCKS = 0xffffffffll / ROW_THREADS;  // a launch has fewer than 2^32 threads in x

// D / 8 lanes a row, K and V of it: 16 bytes in and one code word out per lane and tensor.  Rows go
// by token inside a head, so a workgroup's codes fill neighbouring lines of one page.  Bound by memory:
// a frame of 3600 tokens of 24 heads of 128 dims, 56 MB, takes 11.8 us, 4.8 TB/s (a large copy: 4.9);
// 48 new tokens of 8 heads 3.2 us, a launch.
template <typename T, int D>
__global__ __launch_bounds__(ROW_THREADS) void kv4_store_kernel(RowArgs a, uint8_t* __restrict__ pages,
                                                                const T* __restrict__ k, const T* __restrict__ v,
                                                                int64_t k_b, int64_t k_h, int64_t k_t, int64_t v_b,
                                                                int64_t v_h, int64_t v_t) {
  using Part = spr::Kv4Part<D>;
  constexpr int LANES = D / 8;
  const int b = blockIdx.y;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * (ROW_THREADS / LANES) + threadIdx.x / LANES;
  const int lane = threadIdx.x % LANES;
  const int64_t h = r / a.rows;
  const int t = static_cast<int>(r - h * a.rows);
  if (h >= a.kv_heads || (a.counts != nullptr && t >= a.counts[b])) return;  // whole rows: quads stay together
  int32_t slot;
  const int64_t page = page_of_row(a.table, a.seq_ids, a.starts, b, t, a.sequences, a.wide, a.log_s, a.num_pages, slot);
  if (page < 0) return;
  float kx[8], vx[8];
  load8(k + b * k_b + h * k_h + t * k_t + lane * 8, kx);
  load8(v + b * v_b + h * v_h + t * v_t + lane * 8, vx);
  uint8_t* part = pages + page * a.page_stride + h * spr::kv4_head_bytes(1 << a.log_s, D);
  uint32_t kb, vb;
  const uint32_t kw = encode8(kx, kb), vw = encode8(vx, vb);
  reinterpret_cast<uint32_t*>(part + slot * Part::CODE_ROW)[lane] = kw;
  reinterpret_cast<uint32_t*>(part + Part::v_codes(a.log_s) + slot * Part::CODE_ROW)[lane] = vw;
  if (lane % 4 == 0) {
    part[Part::k_scales(a.log_s) + slot * Part::SCALE_ROW + lane / 4] = static_cast<uint8_t>(kb);
    part[Part::v_scales(a.log_s) + slot * Part::SCALE_ROW + lane / 4] = static_cast<uint8_t>(vb);
  }
}

template <typename T>
__device__ __forceinline__ void write8(T* p, u32x4 x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};  // bf16 pairs
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<u32x4*>(p)[0] = u32x4{w[0] << 16, w[0] & 0xffff0000u, w[1] << 16, w[1] & 0xffff0000u};
    reinterpret_cast<u32x4*>(p)[1] = u32x4{w[2] << 16, w[2] & 0xffff0000u, w[3] << 16, w[3] & 0xffff0000u};
  } else if constexpr (__is_same(T, _Float16)) {
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[i] = spr::f32_to_f16(spr::bf16_lo(w[i])) | static_cast<uint32_t>(spr::f32_to_f16(spr::bf16_hi(w[i]))) << 16;
    }
    *reinterpret_cast<u32x4*>(p) = u32x4{o[0], o[1], o[2], o[3]};
  } else {
    *reinterpret_cast<u32x4*>(p) = x;
  }
}

// The same walk the other way: out [b, kv_heads, rows, D].  Rows past the entry's count are zeros,
// rows with no page NaN.  11.6 us for the same frame.
template <typename T, int D>
__global__ __launch_bounds__(ROW_THREADS) void kv4_load_kernel(RowArgs a, const uint8_t* __restrict__ pages,
                                                               T* __restrict__ k, T* __restrict__ v) {
  using Part = spr::Kv4Part<D>;
  constexpr int LANES = D / 8;
  const int b = blockIdx.y;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * (ROW_THREADS / LANES) + threadIdx.x / LANES;
  const int lane = threadIdx.x % LANES;
  const int64_t h = r / a.rows;
  const int t = static_cast<int>(r - h * a.rows);
  if (h >= a.kv_heads) return;
  const int64_t at = ((b * static_cast<int64_t>(a.kv_heads) + h) * a.rows + t) * D + lane * 8;
  u32x4 kx = {0, 0, 0, 0}, vx = {0, 0, 0, 0};
  if (a.counts == nullptr || t < a.counts[b]) {
    int32_t slot;
    const int64_t page =
        page_of_row(a.table, a.seq_ids, a.starts, b, t, a.sequences, a.wide, a.log_s, a.num_pages, slot);
    uint32_t kw = 0, vw = 0, kb = 255, vb = 255;
    if (page >= 0) {
      const uint8_t* part = pages + page * a.page_stride + h * spr::kv4_head_bytes(1 << a.log_s, D);
      kw = reinterpret_cast<const uint32_t*>(part + slot * Part::CODE_ROW)[lane];
      vw = reinterpret_cast<const uint32_t*>(part + Part::v_codes(a.log_s) + slot * Part::CODE_ROW)[lane];
      kb = part[Part::k_scales(a.log_s) + slot * Part::SCALE_ROW + lane / 4];
      vb = part[Part::v_scales(a.log_s) + slot * Part::SCALE_ROW + lane / 4];
    }
    kx = spr::kv4_eight(kw, spr::kv4_scale(kb));
    vx = spr::kv4_eight(vw, spr::kv4_scale(vb));
  }
  write8(k + at, kx);
  write8(v + at, vx);
}

// ---------------------------------------------------------------------------- pages

constexpr int PLAN_THREADS = 1024;
constexpr int MAX_NAMED = 2048;  // sequences one call may name: their numbers and sums stay in LDS

// Header of a page call's workspace, written by its first kernel and read by its second.
struct PlanHeader {
  int32_t ok;     // the call may happen
  int32_t total;  // pages to take or move
  int32_t live;   // held pages
  int32_t pad[13];
};
constexpr int64_t HEADER_WORDS = sizeof(PlanHeader) / 4;

// Workspace: the header, `a` [pages] (new pages, or pages to move), `b` [pages] (their places, or the
// new page of every page), `sums` [MAX_NAMED + 1] (first new page of every named sequence).
__host__ __device__ inline int64_t plan_words(int64_t num_pages) { return HEADER_WORDS + 2 * num_pages + MAX_NAMED + 1; }

__device__ __forceinline__ int wave_scan(int v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int up = __shfl_up(v, o, 64);
    if (lane >= o) v += up;
  }
  return v;
}

// Exclusive scan of v over the workgroup; `all` is its sum.  scratch: PLAN_THREADS / 64 words of LDS.
__device__ __forceinline__ int block_scan(int v, int* scratch, int& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int incl = wave_scan(v, lane);
  __syncthreads();
  if (lane == 63) scratch[wave] = incl;
  __syncthreads();
  int before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < PLAN_THREADS / 64; ++w) {
    if (w < wave) before += scratch[w];
    all += scratch[w];
  }
  return before + incl - v;
}

// The lowest `want` pages with FREE (ref_count <= 0) or held (> 0) among [first, last), ascending, to
// `list`; returns how many there are (at most want).  Tiles of four pages a thread; stops at the tile
// that has the last one.
template <bool FREE>
__device__ int find_pages(const int32_t* refs, int first, int last, int want, int32_t* list, int* scratch) {
  int found = 0;
  for (int base = first; base < last && found < want; base += 4 * PLAN_THREADS) {
    const int p0 = base + 4 * threadIdx.x;
    bool hit[4];
    int n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      hit[i] = p0 + i < last && ((refs[p0 + i] <= 0) == FREE);
      n += hit[i] ? 1 : 0;
    }
    int all;
    int at = found + block_scan(n, scratch, all);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (hit[i]) {
        if (at < want) list[at] = p0 + i;
        ++at;
      }
    }
    found += all;
  }
  return min(found, want);
}

// The entry of sums [n + 1] (ascending, sums[0] = 0) that i < sums[n] falls into.
__device__ __forceinline__ int entry_of(const int32_t* sums, int n, int i) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (sums[mid] <= i) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// What the workgroup found wrong: every thread's findings (bit c for status c) together, and of them
// the lowest status.  `found` is a word of LDS that holds 0 before and after.
__device__ __forceinline__ int lowest_code(uint32_t mine, uint32_t* found) {
  if (mine != 0) atomicOr(found, mine);
  __syncthreads();
  const uint32_t all = *found;
  __syncthreads();
  if (threadIdx.x == 0) *found = 0;
  return all != 0 ? __builtin_ctz(all) : 0;
}

__device__ __forceinline__ void report(int32_t* status, int code) {
  if (status != nullptr && threadIdx.x == 0 && status[0] == 0) status[0] = code;
}

// Whether a[j] of [0, upto) is `id` (LDS).
__device__ __forceinline__ bool any_is(const int32_t* a, int upto, int32_t id) {
  bool is = false;
  for (int j = 0; j < upto; ++j) is |= a[j] == id;
  return is;
}

// Whether a page of one of the n sequences (ids in LDS) lies outside the pool: a wave a sequence.
__device__ __forceinline__ bool outside_pool(const int32_t* table, const int32_t* lengths, const int32_t* ids, int n,
                                             int32_t wide, int log_s, int32_t num_pages) {
  bool outside = false;
  for (int i = threadIdx.x >> 6; i < n; i += PLAN_THREADS / 64) {
    const int64_t held = (static_cast<int64_t>(lengths[ids[i]]) + (1 << log_s) - 1) >> log_s;
    for (int64_t j = threadIdx.x & 63; j < held; j += 64) {
      const int32_t p = table[static_cast<int64_t>(ids[i]) * wide + j];
      outside |= p < 0 || p >= num_pages;
    }
  }
  return outside;
}

// sums[i] = need[0] + .. + need[i - 1] over n entries in LDS, in place of need (n + 1 words); false if
// the sum passes `most` (it may pass 32 bits, so it is first taken in 64).
__device__ bool sum_needs(int32_t* need, int n, int64_t most, int* scratch, int& total) {
  __shared__ int64_t part[PLAN_THREADS / 64];
  int64_t s = 0;
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS) s += need[i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_down(s, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  s = 0;
#pragma unroll
  for (int w = 0; w < PLAN_THREADS / 64; ++w) s += part[w];
  if (s > most) return false;
  int carry = 0;
  for (int base = 0; base < n; base += PLAN_THREADS) {
    const int i = base + threadIdx.x;
    const int v = i < n ? need[i] : 0;
    int all;
    const int at = carry + block_scan(v, scratch, all);
    if (i < n) need[i] = at;
    carry += all;
  }
  if (threadIdx.x == 0) need[n] = carry;
  __syncthreads();
  total = carry;
  return true;
}

__device__ __forceinline__ int64_t pages_for(int64_t tokens, int log_s) { return (tokens + (1 << log_s) - 1) >> log_s; }

// Room for counts[b] more tokens in every named sequence, and the sequences' lengths with them.  One
// workgroup.  starts[b] is the first new token's place, or -1 for all when the call cannot happen.  No
// count may pass `most`.
__global__ __launch_bounds__(PLAN_THREADS) void kv4_reserve_kernel(int32_t* __restrict__ table, int32_t* lengths,
                                                                   int32_t* __restrict__ refs,
                                                                   const int32_t* counts, const int32_t* seq_ids,
                                                                   int32_t n, int32_t most, int32_t sequences, int32_t wide,
                                                                   int32_t log_s, int32_t num_pages,
                                                                   int32_t* __restrict__ starts,
                                                                   int32_t* __restrict__ status,
                                                                   int32_t* __restrict__ list) {
  __shared__ int32_t ids[MAX_NAMED], sums[MAX_NAMED + 1], olds[MAX_NAMED], news[MAX_NAMED];
  __shared__ int scratch[PLAN_THREADS / 64];
  __shared__ uint32_t found;
  const int64_t room = static_cast<int64_t>(wide) << log_s;
  if (threadIdx.x == 0) found = 0;
  uint32_t wrong = 0;
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
    const int32_t id = seq_ids != nullptr ? seq_ids[i] : i;
    ids[i] = id;
    olds[i] = 0;
    news[i] = 0;
    sums[i] = 0;
    if (id < 0 || id >= sequences) {
      wrong |= 1u << KV4_BAD_SEQUENCE;
      continue;
    }
    // all is read before anything is written: counts may be the lengths themselves
    const int32_t old = lengths[id], more = counts[i];
    if (more < 0 || more > most) wrong |= 1u << KV4_BAD_COUNT;
    if (old < 0 || old > room) wrong |= 1u << KV4_BAD_LENGTH;
    else if (static_cast<int64_t>(old) + more > room) wrong |= 1u << KV4_TABLE_FULL;
    olds[i] = old;
    news[i] = static_cast<int32_t>(min(static_cast<int64_t>(old) + more, room));
    sums[i] = static_cast<int32_t>(pages_for(static_cast<int64_t>(old) + more, log_s) - pages_for(old, log_s));
  }
  __syncthreads();
  if (seq_ids != nullptr) {
    for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
      if (any_is(ids, i, ids[i])) wrong |= 1u << KV4_REPEATED;
    }
  }
  int code = lowest_code(wrong, &found), total = 0;
  if (code != KV4_OK) {
  } else if (!sum_needs(sums, n, num_pages, scratch, total)) code = KV4_NO_PAGES;
  else if (find_pages<true>(refs, 0, num_pages, total, list, scratch) < total) code = KV4_NO_PAGES;
  if (code != KV4_OK) {
    report(status, code);
    for (int i = threadIdx.x; i < n; i += PLAN_THREADS) starts[i] = -1;
    return;
  }
  __syncthreads();  // the list is read by other threads than wrote it
  for (int i = threadIdx.x; i < total; i += PLAN_THREADS) {
    const int e = entry_of(sums, n, i);
    const int32_t page = list[i];
    table[static_cast<int64_t>(ids[e]) * wide + pages_for(olds[e], log_s) + (i - sums[e])] = page;
    refs[page] = 1;
  }
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
    starts[i] = olds[i];
    lengths[ids[i]] = news[i];
  }
}

// What a free call asks of entry i: `count` pages from `first` on, of `held`.
struct FreeRange {
  int64_t held, first, count;
};
__device__ __forceinline__ FreeRange free_range(int32_t len, const int32_t* firsts, const int32_t* page_counts, int i,
                                                int log_s) {
  FreeRange f;
  f.held = pages_for(len, log_s);
  f.first = firsts != nullptr ? firsts[i] : 0;
  f.count = page_counts != nullptr && page_counts[i] >= 0 ? page_counts[i] : f.held - f.first;
  return f;
}

// One wave: the freed pages of entry i lose a holder each, the entries behind them close up in ascending
// pieces of 64 (each read before it is written, and below every entry still to be read).
__device__ __forceinline__ void free_row(int32_t* table, int32_t* lengths, int32_t* refs, const int32_t* seq_ids,
                                         const int32_t* firsts, const int32_t* page_counts, int i, int32_t wide,
                                         int log_s) {
  const int lane = threadIdx.x & 63;
  const int32_t id = seq_ids[i];
  const int32_t len = lengths[id];
  const FreeRange f = free_range(len, firsts, page_counts, i, log_s);
  const int32_t held = static_cast<int32_t>(f.held), first = static_cast<int32_t>(f.first);
  const int32_t count = static_cast<int32_t>(f.count);
  if (count == 0) return;
  int32_t* row = table + static_cast<int64_t>(id) * wide;
  for (int32_t j = first + lane; j < first + count; j += 64) atomicSub(&refs[row[j]], 1);
  for (int32_t j0 = first; j0 < held; j0 += 64) {
    const int32_t j = j0 + lane;
    const int32_t p = j + count < held ? row[j + count] : -1;
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    if (j < held) row[j] = p;
  }
  if (lane == 0) {
    // the freed tokens: whole pages, but for the last page's
    const int64_t upto = min(static_cast<int64_t>(first + count) << log_s, static_cast<int64_t>(len));
    lengths[id] = static_cast<int32_t>(len - (upto - (static_cast<int64_t>(first) << log_s)));
  }
}

// Up to this many sequences are freed by the checking workgroup itself, four to a wave: one launch less
// (16 sequences of 63 pages 6.2 + 3.0 us as two).
constexpr int FREE_HERE = 4 * PLAN_THREADS / 64;

// Pages [first, first + count) of every named sequence are given back (count < 0: all from first on),
// the pages behind them close up, and the length loses the tokens that lay there.  This kernel checks.
__global__ __launch_bounds__(PLAN_THREADS) void kv4_free_check_kernel(int32_t* table, int32_t* lengths, int32_t* refs,
                                                                      const int32_t* __restrict__ seq_ids,
                                                                      const int32_t* __restrict__ firsts,
                                                                      const int32_t* __restrict__ page_counts,
                                                                      int32_t n, int32_t sequences, int32_t wide,
                                                                      int32_t log_s, int32_t num_pages,
                                                                      PlanHeader* __restrict__ plan,
                                                                      int32_t* __restrict__ status) {
  __shared__ int32_t ids[MAX_NAMED];
  __shared__ uint32_t found;
  const int64_t room = static_cast<int64_t>(wide) << log_s;
  if (threadIdx.x == 0) found = 0;
  uint32_t wrong = 0;
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
    const int32_t id = seq_ids[i];
    ids[i] = id;
    if (id < 0 || id >= sequences) {
      wrong |= 1u << KV4_BAD_SEQUENCE;
      continue;
    }
    const int32_t len = lengths[id];
    if (len < 0 || len > room) wrong |= 1u << KV4_BAD_LENGTH;
    const FreeRange f = free_range(len, firsts, page_counts, i, log_s);
    if (f.first < 0 || f.first > f.held || f.count < 0 || f.first + f.count > f.held) wrong |= 1u << KV4_BAD_COUNT;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
    if (any_is(ids, i, ids[i])) wrong |= 1u << KV4_REPEATED;
  }
  int code = lowest_code(wrong, &found);
  if (code == KV4_OK) {
    __syncthreads();  // `found` is 0 again
    code = lowest_code(outside_pool(table, lengths, ids, n, wide, log_s, num_pages) ? 1u << KV4_BAD_LENGTH : 0, &found);
  }
  if (plan != nullptr && threadIdx.x == 0) plan->ok = code == KV4_OK ? 1 : 0;
  report(status, code);
  if (n <= FREE_HERE && code == KV4_OK) {
    for (int i = threadIdx.x >> 6; i < n; i += PLAN_THREADS / 64) {
      free_row(table, lengths, refs, seq_ids, firsts, page_counts, i, wide, log_s);
    }
  }
}

__global__ __launch_bounds__(256) void kv4_free_apply_kernel(int32_t* table, int32_t* lengths, int32_t* refs,
                                                             const int32_t* __restrict__ seq_ids,
                                                             const int32_t* __restrict__ firsts,
                                                             const int32_t* __restrict__ page_counts, int32_t n,
                                                             int32_t wide, int32_t log_s,
                                                             const PlanHeader* __restrict__ plan) {
  const int i = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (plan->ok != 0 && i < n) free_row(table, lengths, refs, seq_ids, firsts, page_counts, i, wide, log_s);
}

// Sequence dst[i] becomes a copy of src[i]: with `share` its full pages are the same ones, and its last
// page, where that is not full, a new one with the same tokens; else all its pages are new.  This
// kernel checks and finds the new pages; `sums` says where each sequence's begin.
__global__ __launch_bounds__(PLAN_THREADS) void kv4_fork_plan_kernel(const int32_t* __restrict__ table,
                                                                     const int32_t* __restrict__ lengths,
                                                                     const int32_t* __restrict__ refs,
                                                                     const int32_t* __restrict__ src,
                                                                     const int32_t* __restrict__ dst, int32_t n,
                                                                     int32_t sequences, int32_t wide, int32_t log_s,
                                                                     int32_t num_pages, int32_t share,
                                                                     PlanHeader* __restrict__ plan,
                                                                     int32_t* __restrict__ list,
                                                                     int32_t* __restrict__ sums_out,
                                                                     int32_t* __restrict__ status) {
  __shared__ int32_t to[MAX_NAMED], from[MAX_NAMED], sums[MAX_NAMED + 1];
  __shared__ int scratch[PLAN_THREADS / 64];
  __shared__ uint32_t found;
  const int64_t room = static_cast<int64_t>(wide) << log_s;
  if (threadIdx.x == 0) found = 0;
  uint32_t wrong = 0;
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
    const int32_t s = src[i], d = dst[i];
    from[i] = s;
    to[i] = d;
    sums[i] = 0;
    if (s < 0 || s >= sequences || d < 0 || d >= sequences) {
      wrong |= 1u << KV4_BAD_SEQUENCE;
      continue;
    }
    const int32_t len = lengths[s];
    if (len < 0 || len > room) wrong |= 1u << KV4_BAD_LENGTH;
    if (lengths[d] != 0) wrong |= 1u << KV4_NOT_EMPTY;
    const int64_t every = pages_for(len, log_s), full = share != 0 ? (len >> log_s) : 0;
    sums[i] = static_cast<int32_t>(every - full);
  }
  __syncthreads();
  // one destination twice, or (an empty one: nothing else can be both) one that is a source too
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
    if (any_is(to, i, to[i]) || any_is(from, n, to[i])) wrong |= 1u << KV4_REPEATED;
  }
  int code = lowest_code(wrong, &found), total = 0;
  if (code == KV4_OK) {
    __syncthreads();  // `found` is 0 again
    code = lowest_code(outside_pool(table, lengths, from, n, wide, log_s, num_pages) ? 1u << KV4_BAD_LENGTH : 0, &found);
  }
  if (code != KV4_OK) {
  } else if (!sum_needs(sums, n, num_pages, scratch, total)) code = KV4_NO_PAGES;
  else if (find_pages<true>(refs, 0, num_pages, total, list, scratch) < total) code = KV4_NO_PAGES;
  if (code == KV4_OK) {
    for (int i = threadIdx.x; i <= n; i += PLAN_THREADS) sums_out[i] = sums[i];
  }
  if (threadIdx.x == 0) {
    plan->ok = code == KV4_OK ? 1 : 0;
    plan->total = total;
  }
  report(status, code);
}

// Pages are copied in pieces of 16 KB a workgroup, four 16-byte loads in flight a lane.  Bound by memory:
// 929 pages of 418 KB, 777 MB read and written, 139 us, 5.6 TB/s; 1,242 moved pages of 2 x 70 KB 67 to
// 81 us.  The plans are one workgroup's chain of dependent loads: 8 us for 16 sequences, 5 us for a
// compaction of 5,000 pages.
constexpr int COPY_THREADS = 256;
constexpr int COPY_PIECE = COPY_THREADS * 16 * 4;  // bytes a workgroup moves at a time

// bytes [at, at + COPY_PIECE) of one page to another, four 16-byte loads in flight a lane
__device__ __forceinline__ void copy_piece(const uint8_t* __restrict__ from, uint8_t* __restrict__ to, int64_t at,
                                           int64_t bytes) {
  typedef uint32_t words __attribute__((ext_vector_type(4)));
  words x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t o = at + (i * COPY_THREADS + threadIdx.x) * 16;
    x[i] = o < bytes ? *reinterpret_cast<const words*>(from + o) : words{0, 0, 0, 0};
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t o = at + (i * COPY_THREADS + threadIdx.x) * 16;
    if (o < bytes) *reinterpret_cast<words*>(to + o) = x[i];
  }
}

// The planned fork: table rows, holders, lengths, and the new pages' bytes in every layer.  A source
// page is never a new one (it is held), so copies do not meet.
__global__ __launch_bounds__(COPY_THREADS) void kv4_fork_apply_kernel(
    uint8_t* __restrict__ pages, int64_t page_bytes, int64_t layer_bytes, int32_t layers, int32_t* __restrict__ table,
    int32_t* __restrict__ lengths, int32_t* __restrict__ refs, const int32_t* __restrict__ src,
    const int32_t* __restrict__ dst, int32_t n, int32_t wide, int32_t log_s, int32_t share,
    const PlanHeader* __restrict__ plan, const int32_t* __restrict__ list, const int32_t* __restrict__ sums) {
  if (plan->ok == 0) return;
  const int32_t total = plan->total;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * COPY_THREADS + threadIdx.x; e < static_cast<int64_t>(n) * wide;
       e += static_cast<int64_t>(gridDim.x) * COPY_THREADS) {
    const int32_t i = static_cast<int32_t>(e / wide), j = static_cast<int32_t>(e - static_cast<int64_t>(i) * wide);
    const int32_t len = lengths[src[i]];
    const int32_t every = static_cast<int32_t>(pages_for(len, log_s)), full = share != 0 ? (len >> log_s) : 0;
    int32_t p = -1;
    if (j < full) {
      p = table[static_cast<int64_t>(src[i]) * wide + j];
      atomicAdd(&refs[p], 1);
    } else if (j < every) {
      p = list[sums[i] + j - full];
      refs[p] = 1;
    }
    table[static_cast<int64_t>(dst[i]) * wide + j] = p;
    if (j == 0) lengths[dst[i]] = len;
  }
  const int64_t pieces = spr::ceil_div(page_bytes, COPY_PIECE);
  for (int64_t w = blockIdx.x; w < total * layers * pieces; w += gridDim.x) {
    const int64_t piece = w % pieces, q = w / pieces;
    const int64_t layer = q % layers;
    const int32_t k = static_cast<int32_t>(q / layers);
    const int32_t i = entry_of(sums, n, k);
    const int32_t full = share != 0 ? (lengths[src[i]] >> log_s) : 0;
    const int64_t from = table[static_cast<int64_t>(src[i]) * wide + full + (k - sums[i])], to = list[k];
    uint8_t* base = pages + layer * layer_bytes;
    copy_piece(base + from * page_bytes, base + to * page_bytes, piece * COPY_PIECE, page_bytes);
  }
}

// live = the held pages; the i-th lowest held page at or above live goes to the i-th lowest free one
// below it.  a: the pages that move, b: where to.
__global__ __launch_bounds__(PLAN_THREADS) void kv4_compact_plan_kernel(const int32_t* __restrict__ refs,
                                                                        int32_t num_pages,
                                                                        PlanHeader* __restrict__ plan,
                                                                        int32_t* __restrict__ a,
                                                                        int32_t* __restrict__ b,
                                                                        int32_t* __restrict__ live_out) {
  __shared__ int scratch[PLAN_THREADS / 64];
  int n = 0;
  for (int p = threadIdx.x; p < num_pages; p += PLAN_THREADS) n += refs[p] > 0 ? 1 : 0;
  int live;
  block_scan(n, scratch, live);
  const int moving = find_pages<false>(refs, live, num_pages, num_pages, a, scratch);
  find_pages<true>(refs, 0, live, moving, b, scratch);
  if (threadIdx.x == 0) {
    plan->ok = 1;
    plan->total = moving;
    plan->live = live;
    live_out[0] = live;
  }
}

// Where page p of the table goes: its place in a (ascending) names its place in b.
__device__ __forceinline__ int32_t moved_to(const int32_t* a, const int32_t* b, int32_t total, int32_t p) {
  int lo = 0, hi = total;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] < p) lo = mid + 1;
    else hi = mid;
  }
  return lo < total && a[lo] == p ? b[lo] : p;
}

__global__ __launch_bounds__(COPY_THREADS) void kv4_compact_apply_kernel(
    uint8_t* __restrict__ pages, int64_t page_bytes, int64_t layer_bytes, int32_t layers, int32_t* __restrict__ table,
    int64_t entries, int32_t* __restrict__ refs, const PlanHeader* __restrict__ plan, const int32_t* __restrict__ a,
    const int32_t* __restrict__ b) {
  const int32_t total = plan->total, live = plan->live;
  if (total == 0) return;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * COPY_THREADS + threadIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * COPY_THREADS;
  for (int64_t e = first; e < entries; e += step) {
    const int32_t p = table[e];
    if (p >= live) table[e] = moved_to(a, b, total, p);
  }
  for (int64_t i = first; i < total; i += step) {
    refs[b[i]] = refs[a[i]];
    refs[a[i]] = 0;
  }
  const int64_t pieces = spr::ceil_div(page_bytes, COPY_PIECE);
  for (int64_t w = blockIdx.x; w < total * layers * pieces; w += gridDim.x) {
    const int64_t piece = w % pieces, q = w / pieces;
    const int64_t layer = q % layers;
    const int64_t k = q / layers;
    uint8_t* base = pages + layer * layer_bytes;
    copy_piece(base + a[k] * page_bytes, base + b[k] * page_bytes, piece * COPY_PIECE, page_bytes);
  }
}

// ---------------------------------------------------------------------------- host

int log2_of(int32_t s) { return 31 - __builtin_clz(static_cast<unsigned>(s)); }

int check_pool(const char* what, int32_t page_size, int32_t num_pages) {
  SPR_REQUIRE(spr::kv4_page_size_ok(page_size), "%s: page size %d (32, 64, 128 or 256)", what, page_size);
  SPR_REQUIRE(num_pages >= 1 && num_pages <= (1 << 28), "%s: %d pages", what, num_pages);
  return SPR_OK;
}

int check_table(const char* what, int32_t sequences, int32_t wide, int32_t page_size) {
  SPR_REQUIRE(sequences >= 1 && wide >= 1, "%s: a block table of %d x %d", what, sequences, wide);
  SPR_REQUIRE(static_cast<int64_t>(wide) * page_size <= spr::KV4_MOST_TOKENS,
              "%s: %d pages of %d tokens a sequence pass 2^30 tokens", what, wide, page_size);
  return SPR_OK;
}

// Pages of all layers are counted in 32 bits.
int check_layers(const char* what, const void* pages, int64_t page_bytes, int64_t layer_bytes, int32_t layers,
                 int32_t num_pages) {
  SPR_REQUIRE(page_bytes > 0 && page_bytes % 16 == 0 && layers >= 1 && layer_bytes % 16 == 0 &&
                  (layers == 1 || layer_bytes >= page_bytes * num_pages) && reinterpret_cast<uintptr_t>(pages) % 16 == 0 &&
                  static_cast<int64_t>(layers) * num_pages <= INT32_MAX,
              "%s: %d pages of %lld bytes, %d layers %lld bytes apart", what, num_pages,
              static_cast<long long>(page_bytes), layers, static_cast<long long>(layer_bytes));
  return SPR_OK;
}

int check_named(const char* what, int32_t n) {
  SPR_REQUIRE(n >= 0 && n <= MAX_NAMED, "%s: %d sequences in one call (at most %d)", what, n, MAX_NAMED);
  return SPR_OK;
}

int check_space(const char* what, const void* ws, size_t bytes, int32_t num_pages) {
  if (ws == nullptr || bytes < static_cast<size_t>(4 * plan_words(num_pages))) {
    spr_set_error("%s: workspace of %zu bytes, %lld needed", what, bytes,
                  static_cast<long long>(4 * plan_words(num_pages)));
    return SPR_EWORKSPACE;
  }
  return SPR_OK;
}

template <typename F>
int by_type(const char* what, int32_t dtype, int32_t d, F&& f) {
  SPR_REQUIRE(d == 64 || d == 128, "%s: head dim %d not supported (64, 128)", what, d);
  switch (dtype) {
    case 0: return d == 64 ? f(__bf16{}, std::integral_constant<int, 64>{}) : f(__bf16{}, std::integral_constant<int, 128>{});
    case 1: return d == 64 ? f(_Float16{}, std::integral_constant<int, 64>{}) : f(_Float16{}, std::integral_constant<int, 128>{});
    case 2: return d == 64 ? f(float{}, std::integral_constant<int, 64>{}) : f(float{}, std::integral_constant<int, 128>{});
  }
  spr_set_error("%s: dtype code %d (0 bf16, 1 fp16, 2 fp32)", what, dtype);
  return SPR_EINVAL;
}

int check_rows(const char* what, int32_t batch, int32_t kv_heads, int32_t rows) {
  SPR_REQUIRE(batch >= 0 && batch <= 65535 && kv_heads >= 1 && rows >= 0, "%s: batch %d, kv heads %d, rows %d", what,
              batch, kv_heads, rows);
  return SPR_OK;
}

// Workgroups for a page call's second kernel: enough for its table entries and pieces, at most two
// rounds of eight to a CU (the rest strides).
unsigned copy_blocks(int64_t entries, int64_t pieces) {
  const int64_t want = std::max(spr::ceil_div(entries, COPY_THREADS), pieces);
  return static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(want, 1), 4096));
}

}  // namespace

extern "C" int64_t spr_kv4_page_bytes(int32_t kv_heads, int32_t page_size, int32_t d) {
  return kv_heads * spr::kv4_head_bytes(page_size, d);
}

extern "C" size_t spr_kv4_pages_workspace(int32_t num_pages) {
  return static_cast<size_t>(4 * plan_words(num_pages > 0 ? num_pages : 0));
}

extern "C" int spr_kv4_store(uint8_t* pages, int32_t num_pages, int32_t kv_heads, int32_t page_size, int32_t d,
                             const int32_t* block_table, int32_t sequences, int32_t wide, const int32_t* seq_ids,
                             const int32_t* starts, const int32_t* counts, const void* k, const void* v, int32_t dtype,
                             int32_t batch, int32_t rows, int64_t k_b, int64_t k_h, int64_t k_t, int64_t v_b,
                             int64_t v_h, int64_t v_t, hipStream_t stream) {
  const char* what = "spr_kv4_store";
  if (int st = check_pool(what, page_size, num_pages)) return st;
  if (int st = check_table(what, sequences, wide, page_size)) return st;
  if (int st = check_rows(what, batch, kv_heads, rows)) return st;
  const RowArgs a = {block_table, seq_ids, starts, counts, sequences, wide, log2_of(page_size), num_pages,
                     kv_heads, rows, kv_heads * spr::kv4_head_bytes(page_size, d)};
  return by_type(what, dtype, d, [&](auto t, auto dim) -> int {
    using T = decltype(t);
    constexpr int D = decltype(dim)::value;
    constexpr int64_t step = 16 / sizeof(T);
    for (int64_t s : {k_b, k_h, k_t, v_b, v_h, v_t}) {
      SPR_REQUIRE(s % step == 0, "%s: strides must be multiples of 16 bytes", what);
    }
    SPR_REQUIRE(reinterpret_cast<uintptr_t>(k) % 16 == 0 && reinterpret_cast<uintptr_t>(v) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(pages) % 16 == 0,
                "%s: pages, K and V must be 16-byte aligned", what);
    if (batch == 0 || rows == 0) return SPR_OK;
    const int64_t blocks = spr::ceil_div(static_cast<int64_t>(kv_heads) * rows, ROW_THREADS / (D / 8));
    SPR_REQUIRE(blocks <= MOST_BLOCKS, "%s: %d rows of %d heads are too many for one call", what, rows, kv_heads);
    kv4_store_kernel<T, D><<<dim3(static_cast<unsigned>(blocks), batch), ROW_THREADS, 0, stream>>>(
        a, pages, static_cast<const T*>(k), static_cast<const T*>(v), k_b, k_h, k_t, v_b, v_h, v_t);
    SPR_LAUNCHED(what);
    return SPR_OK;
  });
}

extern "C" int spr_kv4_load(const uint8_t* pages, int32_t num_pages, int32_t kv_heads, int32_t page_size, int32_t d,
                            const int32_t* block_table, int32_t sequences, int32_t wide, const int32_t* seq_ids,
                            const int32_t* starts, const int32_t* counts, void* k, void* v, int32_t dtype,
                            int32_t batch, int32_t rows, hipStream_t stream) {
  const char* what = "spr_kv4_load";
  if (int st = check_pool(what, page_size, num_pages)) return st;
  if (int st = check_table(what, sequences, wide, page_size)) return st;
  if (int st = check_rows(what, batch, kv_heads, rows)) return st;
  const RowArgs a = {block_table, seq_ids, starts, counts, sequences, wide, log2_of(page_size), num_pages,
                     kv_heads, rows, kv_heads * spr::kv4_head_bytes(page_size, d)};
  return by_type(what, dtype, d, [&](auto t, auto dim) -> int {
    using T = decltype(t);
    constexpr int D = decltype(dim)::value;
    SPR_REQUIRE(reinterpret_cast<uintptr_t>(k) % 16 == 0 && reinterpret_cast<uintptr_t>(v) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(pages) % 16 == 0,
                "%s: pages, K and V must be 16-byte aligned", what);
    if (batch == 0 || rows == 0) return SPR_OK;
    const int64_t blocks = spr::ceil_div(static_cast<int64_t>(kv_heads) * rows, ROW_THREADS / (D / 8));
    SPR_REQUIRE(blocks <= MOST_BLOCKS, "%s: %d rows of %d heads are too many for one call", what, rows, kv_heads);
    kv4_load_kernel<T, D><<<dim3(static_cast<unsigned>(blocks), batch), ROW_THREADS, 0, stream>>>(
        a, pages, static_cast<T*>(k), static_cast<T*>(v));
    SPR_LAUNCHED(what);
    return SPR_OK;
  });
}

extern "C" int spr_kv4_reserve_ex(int32_t* block_table, int32_t* lengths, int32_t* ref_count, const int32_t* counts,
                                  const int32_t* seq_ids, int32_t n, int32_t most, int32_t sequences, int32_t wide,
                                  int32_t page_size, int32_t num_pages, int32_t* starts, int32_t* status,
                                  void* workspace, size_t workspace_bytes, hipStream_t stream) {
  const char* what = "spr_kv4_reserve";
  if (int st = check_pool(what, page_size, num_pages)) return st;
  if (int st = check_table(what, sequences, wide, page_size)) return st;
  if (int st = check_named(what, n)) return st;
  SPR_REQUIRE(seq_ids != nullptr || n <= sequences, "%s: %d counts for %d sequences", what, n, sequences);
  if (n == 0) return SPR_OK;
  if (int st = check_space(what, workspace, workspace_bytes, num_pages)) return st;
  kv4_reserve_kernel<<<1, PLAN_THREADS, 0, stream>>>(block_table, lengths, ref_count, counts, seq_ids, n, most,
                                                     sequences, wide, log2_of(page_size), num_pages, starts, status,
                                                     static_cast<int32_t*>(workspace) + HEADER_WORDS);
  SPR_LAUNCHED(what);
  return SPR_OK;
}

extern "C" int spr_kv4_reserve(int32_t* block_table, int32_t* lengths, int32_t* ref_count, const int32_t* counts,
                               const int32_t* seq_ids, int32_t n, int32_t sequences, int32_t wide, int32_t page_size,
                               int32_t num_pages, int32_t* starts, int32_t* status, void* workspace,
                               size_t workspace_bytes, hipStream_t stream) {
  return spr_kv4_reserve_ex(block_table, lengths, ref_count, counts, seq_ids, n, INT32_MAX, sequences, wide, page_size,
                            num_pages, starts, status, workspace, workspace_bytes, stream);
}

extern "C" int spr_kv4_free(int32_t* block_table, int32_t* lengths, int32_t* ref_count, const int32_t* seq_ids,
                            const int32_t* first_pages, const int32_t* page_counts, int32_t n, int32_t sequences,
                            int32_t wide, int32_t page_size, int32_t num_pages, int32_t* status, void* workspace,
                            size_t workspace_bytes, hipStream_t stream) {
  const char* what = "spr_kv4_free";
  if (int st = check_pool(what, page_size, num_pages)) return st;
  if (int st = check_table(what, sequences, wide, page_size)) return st;
  if (int st = check_named(what, n)) return st;
  if (n == 0) return SPR_OK;
  if (n > FREE_HERE) {
    if (int st = check_space(what, workspace, workspace_bytes, num_pages)) return st;
  }
  PlanHeader* plan = n > FREE_HERE ? static_cast<PlanHeader*>(workspace) : nullptr;
  const int log_s = log2_of(page_size);
  kv4_free_check_kernel<<<1, PLAN_THREADS, 0, stream>>>(block_table, lengths, ref_count, seq_ids, first_pages,
                                                        page_counts, n, sequences, wide, log_s, num_pages, plan,
                                                        status);
  SPR_LAUNCHED(what);
  if (n <= FREE_HERE) return SPR_OK;
  kv4_free_apply_kernel<<<static_cast<unsigned>(spr::ceil_div(n, 4)), 256, 0, stream>>>(
      block_table, lengths, ref_count, seq_ids, first_pages, page_counts, n, wide, log_s, plan);
  SPR_LAUNCHED(what);
  return SPR_OK;
}

extern "C" int spr_kv4_fork(uint8_t* pages, int64_t page_bytes, int64_t layer_bytes, int32_t layers,
                            int32_t* block_table, int32_t* lengths, int32_t* ref_count, const int32_t* src,
                            const int32_t* dst, int32_t n, int32_t sequences, int32_t wide, int32_t page_size,
                            int32_t num_pages, int32_t share, int32_t* status, void* workspace, size_t workspace_bytes,
                            hipStream_t stream) {
  const char* what = "spr_kv4_fork";
  if (int st = check_pool(what, page_size, num_pages)) return st;
  if (int st = check_table(what, sequences, wide, page_size)) return st;
  if (int st = check_named(what, n)) return st;
  if (int st = check_layers(what, pages, page_bytes, layer_bytes, layers, num_pages)) return st;
  if (n == 0) return SPR_OK;
  if (int st = check_space(what, workspace, workspace_bytes, num_pages)) return st;
  PlanHeader* plan = static_cast<PlanHeader*>(workspace);
  int32_t* list = static_cast<int32_t*>(workspace) + HEADER_WORDS;
  int32_t* sums = list + 2 * static_cast<int64_t>(num_pages);
  const int log_s = log2_of(page_size);
  kv4_fork_plan_kernel<<<1, PLAN_THREADS, 0, stream>>>(block_table, lengths, ref_count, src, dst, n, sequences, wide,
                                                       log_s, num_pages, share, plan, list, sums, status);
  SPR_LAUNCHED(what);
  const int64_t most = share != 0 ? n : std::min<int64_t>(static_cast<int64_t>(n) * wide, num_pages);
  const unsigned blocks = copy_blocks(static_cast<int64_t>(n) * wide, most * layers * spr::ceil_div(page_bytes, COPY_PIECE));
  kv4_fork_apply_kernel<<<blocks, COPY_THREADS, 0, stream>>>(pages, page_bytes, layer_bytes, layers, block_table,
                                                             lengths, ref_count, src, dst, n, wide, log_s, share, plan,
                                                             list, sums);
  SPR_LAUNCHED(what);
  return SPR_OK;
}

extern "C" int spr_kv4_compact(uint8_t* pages, int64_t page_bytes, int64_t layer_bytes, int32_t layers,
                               int32_t* block_table, int32_t* ref_count, int32_t sequences, int32_t wide,
                               int32_t num_pages, int32_t* live, void* workspace, size_t workspace_bytes,
                               hipStream_t stream) {
  const char* what = "spr_kv4_compact";
  if (int st = check_pool(what, 32, num_pages)) return st;
  if (int st = check_table(what, sequences, wide, 1)) return st;
  if (int st = check_layers(what, pages, page_bytes, layer_bytes, layers, num_pages)) return st;
  if (int st = check_space(what, workspace, workspace_bytes, num_pages)) return st;
  PlanHeader* plan = static_cast<PlanHeader*>(workspace);
  int32_t* a = static_cast<int32_t*>(workspace) + HEADER_WORDS;
  int32_t* b = a + num_pages;
  kv4_compact_plan_kernel<<<1, PLAN_THREADS, 0, stream>>>(ref_count, num_pages, plan, a, b, live);
  SPR_LAUNCHED(what);
  const int64_t entries = static_cast<int64_t>(sequences) * wide;
  const unsigned blocks =
      copy_blocks(entries, static_cast<int64_t>(num_pages / 2) * layers * spr::ceil_div(page_bytes, COPY_PIECE));
  kv4_compact_apply_kernel<<<blocks, COPY_THREADS, 0, stream>>>(pages, page_bytes, layer_bytes, layers, block_table,
                                                                entries, ref_count, plan, a, b);
  SPR_LAUNCHED(what);
  return SPR_OK;
}
