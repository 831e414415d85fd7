// Addresses in a paged key/value cache (internal; plain C++ on the host too).
//
// A cache is two tensors of pages; entry e of sequence s is slot e % page of
// page table[s][e / page].  New tokens of all sequences lie behind one another,
// sequence s in rows starts[s] .. starts[s + 1] - 1; lens[s] counts its entries
// with these, so its token i of n is entry lens[s] - n + i.  Tables, starts and
// lengths live on the device where the host cannot look at them: every value
// read from them is brought into range here before it forms an address, so
// that a wrong one gives a wrong result and never an access out of bounds.
#pragma once
#include <stdint.h>

#if defined(__HIPCC__)
#define ANN_HD __host__ __device__ __forceinline__
#else
#define ANN_HD inline
#endif

namespace ann {

struct PagedArgs {
  uint16_t* k;              // bf16 (pages, heads, page, head_dim) by the strides below
  uint16_t* v;
  long long kp, kh, ks;     // elements from page to page, head to head, slot to slot
  long long vp, vh, vs;
  const int32_t* table;     // (seqs, cols), row stride trow
  long long trow;
  const int32_t* starts;    // seqs + 1
  const int32_t* lens;      // seqs
  int pages, sh, heads, seqs, cols, rows;   // sh: log2 of the page size; rows: of new tokens
};

// Entries of a sequence: a length below zero is none, one past the table's
// last page ends there.
ANN_HD int pg_len(int len, int cols, int sh) {
  const long long cap = (long long)cols << sh;
  return len < 0 ? 0 : len > cap ? (int)cap : len;
}

struct PgRange {
  int first, n;   // row of the first new token, how many
};
// Rows of a sequence's new tokens from starts[s] and starts[s + 1].
ANN_HD PgRange pg_range(int a, int b, int rows) {
  if (a < 0) a = 0;
  if (a > rows) a = rows;
  if (b < a) b = a;
  if (b > rows) b = rows;
  return {a, b - a};
}

// A page to read from: an id that is no page reads page 0.
ANN_HD int pg_read(int id, int pages) { return (unsigned)id < (unsigned)pages ? id : 0; }
// Whether a page may be written.
ANN_HD bool pg_writable(int id, int pages) { return (unsigned)id < (unsigned)pages; }

// Offset of entry e's slot within its page.
ANN_HD long long pg_slot(int e, int sh, long long slot) {
  return (long long)(e & ((1 << sh) - 1)) * slot;
}

// n / d for 0 <= n < 2^31 by a product: m = ceil(2^s / d) with s = 31 + ceil(log2 d)
// is below 2^32 for d > 1, and n (m d - 2^s) < 2^31 d <= 2^s keeps the quotient.
struct FastDiv {
  uint32_t m;
  int s;   // 0: d is 1
  ANN_HD int div(int n) const { return s ? (int)(((uint64_t)(uint32_t)n * m) >> s) : n; }
  static inline FastDiv of(int d) {
    if (d <= 1) return {0, 0};
    int l = 0;
    while ((1LL << l) < d) ++l;
    const int s = 31 + l;
    return {(uint32_t)(((1ULL << s) + d - 1) / d), s};
  }
};

#if defined(__HIPCC__)
// The sequence whose new tokens row n belongs to, by a whole wave: the last s
// with starts[s] <= n, found among 64 of them at a time (two loads in a row up
// to 4096 sequences); -1 where there is none.  The caller checks the row
// against that sequence's range, so starts that do not rise find no entry.
__device__ __forceinline__ int pg_sequence(const int32_t* __restrict__ starts, int seqs, int n) {
  const int lane = threadIdx.x & 63;
  int lo = 0, span = seqs;
  while (span > 64) {
    const int step = (span + 63) / 64;
    const int i = lane * step;
    const unsigned long long le = __ballot(i < span && starts[lo + i] <= n);
    if (!le) return -1;
    const int at = (63 - __builtin_clzll(le)) * step;
    lo += at;
    span = span - at < step ? span - at : step;
  }
  const unsigned long long le = __ballot(lane < span && starts[lo + lane] <= n);
  return le ? lo + 63 - __builtin_clzll(le) : -1;
}

// The tile-th tile of br rows of the sequences with more than `few` rows (g rows
// for each new token), by a whole wave: its sequence and first row, the sequence's
// new tokens and length (read beside its rows); seq -1 where there are fewer tiles.
struct PgTile {
  int seq, row0;
  PgRange r;
  int len;
};
__device__ __forceinline__ PgTile pg_tile(const int32_t* __restrict__ starts,
                                          const int32_t* __restrict__ lens, int seqs, int rows,
                                          int g, int few, int br, int tile) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int s0 = 0; s0 < seqs; s0 += 64) {
    const int s = s0 + lane;
    int n = 0, len = 0;
    PgRange r = {0, 0};
    if (s < seqs) {
      len = lens[s];
      r = pg_range(starts[s], starts[s + 1], rows);
      n = r.n * g > few ? (r.n * g + br - 1) / br : 0;
    }
    int sum = n;   // of this lane's sequence and those before it
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(sum, o, 64);
      if (lane >= o) sum += v;
    }
    const unsigned long long past = __ballot(before + sum > tile);
    if (past) {
      const int at = __builtin_ctzll(past);
      return {s0 + at, (tile - before - __builtin_amdgcn_readlane(sum - n, at)) * br,
              {__builtin_amdgcn_readlane(r.first, at), __builtin_amdgcn_readlane(r.n, at)},
              __builtin_amdgcn_readlane(len, at)};
    }
    before += __shfl(sum, 63, 64);
  }
  return {-1, 0, {0, 0}, 0};
}

// The tile-th tile of br rows of groups of sequences (groups: ngroups + 1 of them,
// like starts), by a whole wave: seq is the group, r its rows.
__device__ __forceinline__ PgTile pg_group_tile(const int32_t* __restrict__ groups, int ngroups,
                                                const int32_t* __restrict__ starts, int seqs, int rows,
                                                int g, int br, int tile) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int g0 = 0; g0 < ngroups; g0 += 64) {
    const int i = g0 + lane;
    int n = 0;
    PgRange r = {0, 0};
    if (i < ngroups) {
      const PgRange s = pg_range(groups[i], groups[i + 1], seqs);
      r = pg_range(starts[s.first], starts[s.first + s.n], rows);
      n = (r.n * g + br - 1) / br;
    }
    int sum = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(sum, o, 64);
      if (lane >= o) sum += v;
    }
    const unsigned long long past = __ballot(before + sum > tile);
    if (past) {
      const int at = __builtin_ctzll(past);
      return {g0 + at, (tile - before - __builtin_amdgcn_readlane(sum - n, at)) * br,
              {__builtin_amdgcn_readlane(r.first, at), __builtin_amdgcn_readlane(r.n, at)}, 0};
    }
    before += __shfl(sum, 63, 64);
  }
  return {-1, 0, {0, 0}, 0};
}
#endif

}  // namespace ann
