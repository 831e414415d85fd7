// Pages of the cache given to sequences and taken back (paged_attn.hip reads
// them): block tables and row maps of a step from the requests' lengths.
//
// A page is free where its count refs[p] is not above zero.  With at = lens[s],
// n = new[s], a sequence needs the columns at / page <= c < ceil((at + n) / page)
// of its row that name no page.  It is served if at + n fits its row and the new
// rows and needed pages of all up to it that fit theirs are no more than there are
// (no page needed: rows only).  The i-th needed column of those served takes the i-th
// free page.  Whole numbers, no atomics: the same call gives the same tables.
//
// Three passes: needs, and the free pages as bits with the number in each chunk of
// 4096; running sums of both, which say who is served; tables and row maps, a
// work-group for each span of 4096 entries of a sequence, whose waves find 64 pages at a
// time among the bits of a chunk.  Up to 1024 sequences every work-group of the last
// pass forms the sums for itself, in the time of reading them: two launches; more are
// a work-group's between the two.  A call that one work-group gets through in their
// time is one launch.
//
// What bounds them is neither bytes nor operations but the passes that wait for each
// other: a launch that does next to nothing takes 3.4 us, two of them 12.0 us for 48
// sequences of 128 columns and 16384 rows (three 16.7) and 16.8 for 1000 of 512 over 512008
// pages (19.5; 8.3 MB, 1.6 us of copying), and the host 17 us to send them (three 21).
#include "common.h"
#include "launch.h"

namespace ann {

constexpr int PT_CHUNK = 64;   // words of 64 pages in a chunk
constexpr int PT_SPAN = 12;    // log2 of the entries that a work-group of k_table_fill has

struct PtArgs {
  TableArgs t;
  int same;                    // bit 0: the table is changed in place, 1: refs
  int spans, chunks;
  // of each sequence: its length, its new tokens (-1: they do not fit its row; then
  // of those served), pages needed, the rank of its first one (-1: not served)
  int32_t* at;
  int32_t* n;
  int32_t* need;
  int32_t* base;
  int32_t* before;             // (seqs, spans): pages it needs before a span that it touches
  unsigned long long* free_;   // a bit for each page
  int32_t* chunk;              // chunks + 1: free pages in a chunk, then before it
};

__device__ __forceinline__ bool pt_page_ok(int id, int pages) { return (unsigned)id < (unsigned)pages; }

// Columns [t0, t1) that n new entries from `at` on touch.
struct PtCols {
  int t0, t1;
};
__device__ __forceinline__ PtCols pt_cols(int at, int n, int sh) {
  if (n <= 0) return {0, 0};
  return {at >> sh, (int)(((long long)at + n - 1) >> sh) + 1};
}

// What sequence s asks for, by a whole wave.
__device__ __forceinline__ void pt_need(const PtArgs& a, int s) {
  const TableArgs& t = a.t;
  const int lane = threadIdx.x & 63, sh = t.sh;
  const int at = pg_len(t.lens[s], t.cols, sh), want = max(t.add[s], 0);
  const bool fits = (long long)at + want <= (long long)t.cols << sh;
  // more than there are rows is not served, and none behind it: its pages need no count
  const PtCols c = pt_cols(at, fits && want <= t.rows ? want : 0, sh);
  const int32_t* row = t.table + s * t.trow;
  const int spc = PT_SPAN - sh;   // log2 of a span's columns
  constexpr int D = 8;   // reads at once (131072 tokens of one sequence, pages of 16: the call 38.3 us with one, 24.9)
  int need = 0;
  for (int c0 = c.t0; c0 < c.t1;) {
    int from[D + 1];
    bool miss[D];
    from[0] = c0;
#pragma unroll
    for (int d = 0; d < D; ++d) {   // 64 columns at most, not past a span's end
      from[d + 1] = min(min(from[d] + 64, c.t1), ((from[d] >> spc) + 1) << spc);
      const int col = from[d] + lane;
      miss[d] = !pt_page_ok(row[min(col, c.t1 - 1)], t.pages) && col < from[d + 1];
    }
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (lane == 0 && from[d] < c.t1 && (from[d] == c.t0 || (from[d] & ((1 << spc) - 1)) == 0))
        a.before[(long long)s * a.spans + (from[d] >> spc)] = need;
      need += __popcll(__ballot(miss[d]));
    }
    c0 = from[D];
  }
  if (lane == 0) {
    a.at[s] = at;
    a.n[s] = fits ? want : -1;
    a.need[s] = need;
  }
}

// The word of 64 pages from 64 w on, by a whole wave; refs are copied.
__device__ __forceinline__ unsigned long long pt_word(const PtArgs& a, int w) {
  const TableArgs& t = a.t;
  const long long p = (long long)w * 64 + (threadIdx.x & 63);
  int r = 1;
  if (p < t.pages) {
    r = t.refs[p];
    if (!(a.same & 2)) t.refs_out[p] = r;
  }
  const unsigned long long m = __ballot(r <= 0);
  if ((threadIdx.x & 63) == 0) a.free_[w] = m;
  return m;
}

// Inclusive sums of x and y over a work-group of NT threads; tx, ty: over all.
template <int NT>
__device__ __forceinline__ void pt_scan(long long& x, long long& y, long long& tx, long long& ty,
                                        long long (*part)[2]) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long long u = __shfl_up(x, o, 64), v = __shfl_up(y, o, 64);
    if (lane >= o) {
      x += u;
      y += v;
    }
  }
  __syncthreads();
  if (lane == 63) {
    part[wv][0] = x;
    part[wv][1] = y;
  }
  __syncthreads();
  tx = ty = 0;
  long long bx = 0, by = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    if (w == wv) {
      bx = tx;
      by = ty;
    }
    tx += part[w][0];
    ty += part[w][1];
  }
  x += bx;
  y += by;
}

// What a sequence gets: its new tokens (0: not served), the rank of its first page, its
// first row; the free pages before each chunk; rows of all.
struct PtGrant {
  const int32_t* n;
  const int32_t* base;
  const int32_t* first;
  const int32_t* chunk;
  int rows;
};

// Free pages before each chunk, and who is served.
template <int NT>
__device__ __forceinline__ void pt_grant(const PtArgs& a, long long (*part)[2]) {
  const TableArgs& t = a.t;
  const int tid = threadIdx.x;
  long long free_pages = 0;
  for (int c0 = 0; c0 < a.chunks; c0 += NT) {
    const int c = c0 + tid;
    const int own = c < a.chunks ? a.chunk[c] : 0;
    long long x = own, y = 0, tx, ty;
    pt_scan<NT>(x, y, tx, ty, part);
    if (c < a.chunks) a.chunk[c] = (int)(free_pages + x - own);
    free_pages += tx;
  }
  long long need_all = 0, rows_all = 0, rank = 0, row = 0;
  for (int s0 = 0; s0 < t.seqs; s0 += NT) {
    const int s = s0 + tid;
    const bool real = s < t.seqs;
    const int n = real ? a.n[s] : -1, need = real && n >= 0 ? a.need[s] : 0;
    long long x = need, y = max(n, 0), tx, ty;
    pt_scan<NT>(x, y, tx, ty, part);
    const bool ok = n >= 0 && rows_all + y <= t.rows && (need == 0 || need_all + x <= free_pages);
    need_all += tx;
    rows_all += ty;
    const int gn = ok ? n : 0, gp = ok ? need : 0;
    x = gp;
    y = gn;
    pt_scan<NT>(x, y, tx, ty, part);
    if (real) {
      a.n[s] = gn;
      a.base[s] = ok ? (int)(rank + x - gp) : -1;
      t.starts[s] = (int)(row + y - gn);
      t.lens_out[s] = a.at[s] + gn;
    }
    rank += tx;
    row += ty;
  }
  if (tid == 0) t.starts[t.seqs] = (int)row;
}

// The k-th set bit of w.
__device__ __forceinline__ int pt_bit(unsigned long long w, int k) {
  int at = 0;
#pragma unroll
  for (int h = 32; h > 0; h >>= 1) {
    const int c = __popcll((w >> at) & ((1ull << h) - 1));
    if (k >= c) {
      k -= c;
      at += h;
    }
  }
  return at;
}

// The free page of rank `rank`, for the lanes with want; by a whole wave, whose
// lowest such rank is r0.  -1 past the last one.
__device__ __forceinline__ int pt_page(const unsigned long long* free_, const int32_t* chunk, int chunks, int pages,
                                       bool want, int rank, int r0) {
  const int lane = threadIdx.x & 63;
  const int words = (int)(((long long)pages + 63) / 64);
  int id = -1;
  for (int c = pg_sequence(chunk, chunks, r0); c >= 0 && c < chunks && __any(want); ++c) {
    const int w = c * PT_CHUNK + lane;
    const unsigned long long m = w < words ? free_[w] : 0;
    const int pop = __popcll(m);
    int sum = pop;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(sum, o, 64);
      if (lane >= o) sum += v;
    }
    const int total = __shfl(sum, 63, 64), k = rank - chunk[c];
    int at = 0;   // words that end at or before k
#pragma unroll
    for (int h = 32; h > 0; h >>= 1)
      if (__shfl(sum, at + h - 1, 64) <= k) at += h;
    at = min(at, 63);
    const unsigned long long mw = __shfl(m, at, 64);
    const int left = k - __shfl(sum - pop, at, 64);
    if (want && k < total) {
      id = (int)(((long long)c * PT_CHUNK + at) * 64 + pt_bit(mw, left));
      want = false;
    }
  }
  return id;
}

// Sums of x and y over the threads before this one; tx, ty: over all.  One barrier.
template <int NW>
__device__ __forceinline__ void pt_sums(uint32_t& x, uint32_t& y, uint32_t& tx, uint32_t& ty, uint32_t (*part)[NW]) {
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t ix = wave_scan(x), iy = wave_scan(y);
  if (lane == 63) {
    part[0][wv] = ix;
    part[1][wv] = iy;
  }
  __syncthreads();
  const uint32_t px = part[0][lane % NW], py = part[1][lane % NW];
  const uint32_t sx = wave_scan(lane < NW ? px : 0), sy = wave_scan(lane < NW ? py : 0);
  x = ix - x + lane_of(sx - px, wv);
  y = iy - y + lane_of(sy - py, wv);
  tx = lane_of(sx, NW - 1);
  ty = lane_of(sy, NW - 1);
}
// The same for up to PT_SUMS sequences and as many chunks as threads, by a work-group of 256
// for itself, to LDS: sums of what is asked for, at most one more than there is of each, in
// 32 bits.
constexpr int PT_SUMS = 1024;
constexpr int PT_SUM_PAGES = 256 * 64 * PT_CHUNK, PT_SUM_ROWS = 1 << 21;
struct PtSums {
  int32_t n[PT_SUMS], base[PT_SUMS], first[PT_SUMS], chunk[256];
  uint32_t part[3][2][4];
};
__device__ __forceinline__ int pt_sum_up(const PtArgs& a, PtSums& sh) {
  constexpr int PER = PT_SUMS / 256;
  const TableArgs& t = a.t;
  const int tid = threadIdx.x, s0 = tid * PER;
  const uint32_t own = tid < a.chunks ? (uint32_t)a.chunk[tid] : 0;
  int n[PER];
  uint32_t need[PER], x = 0, y = 0, tx, ty, free_pages;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int s = min(s0 + i, t.seqs - 1);
    n[i] = a.n[s];
    need[i] = (uint32_t)min(a.need[s], t.pages + 1);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (s0 + i >= t.seqs) n[i] = -1;
    if (n[i] < 0) need[i] = 0;
    x += need[i];
    y += (uint32_t)min(max(n[i], 0), t.rows + 1);
  }
  uint32_t c = own, none = 0;
  pt_sums<4>(c, none, free_pages, none, sh.part[0]);
  if (tid < a.chunks) sh.chunk[tid] = (int)c;
  pt_sums<4>(x, y, tx, ty, sh.part[1]);
  uint32_t px = 0, py = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    x += need[i];
    y += (uint32_t)min(max(n[i], 0), t.rows + 1);
    const bool ok = n[i] >= 0 && y <= (uint32_t)t.rows && (need[i] == 0 || x <= free_pages);
    n[i] = ok ? n[i] : 0;
    need[i] = ok ? need[i] : 0;
    px += need[i];
    py += (uint32_t)n[i];
  }
  pt_sums<4>(px, py, tx, ty, sh.part[2]);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int s = s0 + i;
    sh.n[s] = n[i];
    sh.base[s] = (int)px;
    sh.first[s] = (int)py;
    px += need[i];
    py += (uint32_t)n[i];
  }
  __syncthreads();
  return (int)ty;
}

// Columns and rows of one span of a sequence, by a work-group of 256 threads; page:
// 256 ids, cnt: 4 numbers, in LDS.
__device__ __forceinline__ void pt_fill(const PtArgs& a, const PtGrant& g, int s, int span, int* page, int* cnt) {
  const TableArgs& t = a.t;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int spc = PT_SPAN - t.sh;
  const int c0 = span << spc, c1 = min(t.cols, c0 + (1 << spc));
  const int at = a.at[s], n = g.n[s];
  const PtCols tc = pt_cols(at, n, t.sh);
  const bool touched = max(tc.t0, c0) < min(tc.t1, c1);
  if (!touched && (a.same & 1)) return;   // the same for all threads
  const int c = c0 + tid;
  int id = 0;
  bool take = false;
  if (c < c1) {
    id = t.table[s * t.trow + c];
    take = c >= tc.t0 && c < tc.t1 && !pt_page_ok(id, t.pages);
  }
  if (touched) {
    const unsigned long long m = __ballot(take);
    if (lane == 0) cnt[wv] = __popcll(m);
    __syncthreads();
    if (m) {   // of this wave
      int r0 = g.base[s] + a.before[(long long)s * a.spans + span];
      for (int w = 0; w < wv; ++w) r0 += cnt[w];
      const int got = pt_page(a.free_, g.chunk, a.chunks, t.pages, take, r0 + __popcll(m & ((1ull << lane) - 1)), r0);
      if (take) {
        id = got;
        if (got >= 0) t.refs_out[got] = 1;
      }
    }
    page[tid] = id;
  }
  if (c < c1 && (take || !(a.same & 1))) t.table_out[s * t.orow + c] = id;
  if (!touched) return;
  __syncthreads();
  const int lo = max(at, c0 << t.sh), hi = (int)min((long long)at + n, (long long)c1 << t.sh);
  const int row0 = g.first[s] - at;
  for (int e = lo + tid; e < hi; e += 256) {
    const int p = page[(e >> t.sh) - c0], r = row0 + e;
    t.seq[r] = s;
    t.pos[r] = e;
    t.slot[r] = pt_page_ok(p, t.pages) ? ((long long)p << t.sh) + (e & ((1 << t.sh) - 1)) : -1;
  }
  __syncthreads();   // page and cnt are used again
}

// Rows behind the last sequence's.
__device__ __forceinline__ void pt_behind(const TableArgs& t, int rows, int first, int step) {
  for (int r = rows + first; r < t.rows; r += step) {
    t.seq[r] = -1;
    t.pos[r] = -1;
    t.slot[r] = -1;
  }
}

__global__ __launch_bounds__(256) void k_table_need(PtArgs a, int seq_blocks) {
  __shared__ int cnt[4];
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if ((int)blockIdx.x < seq_blocks) {
    const int s = blockIdx.x * 4 + wv;
    if (s < a.t.seqs) pt_need(a, s);
    return;
  }
  const int c = blockIdx.x - seq_blocks;
  const int words = (int)(((long long)a.t.pages + 63) / 64);
  int n = 0;
#pragma unroll 4
  for (int i = wv; i < PT_CHUNK; i += 4) {
    const int w = c * PT_CHUNK + i;
    if (w < words) n += __popcll(pt_word(a, w));
  }
  if (lane == 0) cnt[wv] = n;
  __syncthreads();
  if (threadIdx.x == 0) a.chunk[c] = cnt[0] + cnt[1] + cnt[2] + cnt[3];
}

__global__ __launch_bounds__(1024) void k_table_grant(PtArgs a) {
  __shared__ long long part[16][2];
  pt_grant<1024>(a, part);
}

// SUMS: who is served is summed up here (k_table_grant's work).
template <bool SUMS>
__global__ __launch_bounds__(256) void k_table_fill(PtArgs a) {
  __shared__ int page[256], cnt[4];
  const TableArgs& t = a.t;
  const int tid = threadIdx.x;
  PtGrant g;
  if constexpr (SUMS) {
    __shared__ PtSums sh;
    g = {sh.n, sh.base, sh.first, sh.chunk, pt_sum_up(a, sh)};
    if (blockIdx.x == 0) {
      for (int s = tid; s < t.seqs; s += 256) {
        t.starts[s] = sh.first[s];
        t.lens_out[s] = a.at[s] + sh.n[s];
      }
      if (tid == 0) t.starts[t.seqs] = g.rows;
    }
  } else {
    g = {a.n, a.base, t.starts, a.chunk, t.starts[t.seqs]};
  }
  const long long all = (long long)t.seqs * a.spans;
  for (long long w = blockIdx.x; w < all; w += gridDim.x)
    pt_fill(a, g, (int)(w / a.spans), (int)(w % a.spans), page, cnt);
  pt_behind(t, g.rows, blockIdx.x * 256 + tid, gridDim.x * 256);
}

// All of it by one work-group, which reads everything at once: a wave takes up to PT_HELD
// pieces of 64 columns, whose ids it keeps.  Its time goes with the pieces and the pages;
// us on the device, and of a call among others (the host sends one launch in 13, two in 17),
// against those of two launches:
//   4 sequences of 64 columns, 512 pages      5.2 12.7    7.3 17.0
//   16, 1024 pages, 8192 rows                 7.2 12.9    8.1 18.5
//   32, 8192 pages                           10.3 12.7   10.7 16.9
//   64, 4096 pages                           13.8 13.6   10.7 17.0
//   64, 16384 pages                          17.5 17.2   10.9 16.9
//   1 of 256 columns, 8192 rows by 2 waves   11.1 12.7    8.6 17.1
// The rule is where a call stops being the shorter one (256 sequences, 16 pieces a wave:
// 46); more rows, which one wave may have to write, go with two.
constexpr int PT_HELD = 4, PT_SEQS = 16 * PT_HELD, PT_PAGES = 16384, PT_ROWS = 8192;
struct PtShared {
  int32_t at[PT_SEQS], n[PT_SEQS], base[PT_SEQS], first[PT_SEQS];
  int32_t need[16 * PT_HELD];             // of a piece
  unsigned long long free_[PT_PAGES / 64];
  int32_t chunk[PT_PAGES / (64 * PT_CHUNK)];
  uint32_t part[2][2][16];
  int rows;
};
__global__ __launch_bounds__(1024) void k_table_one(PtArgs a) {
  __shared__ PtShared sh;
  const TableArgs& t = a.t;
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int per = (t.cols + 63) / 64, pieces = t.seqs * per, words = (t.pages + 63) / 64;
  a.free_ = sh.free_;
  int ids[PT_HELD];
#pragma unroll
  for (int i = 0; i < PT_HELD; ++i) {
    const int q = wv + 16 * i;
    if (q < pieces) ids[i] = t.table[(q / per) * t.trow + min(q % per * 64 + lane, t.cols - 1)];
  }
  if (tid < t.seqs) {
    const int at = pg_len(t.lens[tid], t.cols, t.sh), want = max(t.add[tid], 0);
    sh.at[tid] = at;
    sh.n[tid] = (long long)at + want <= (long long)t.cols << t.sh ? want : -1;
  }
#pragma unroll 4
  for (int w = wv; w < words; w += 16) pt_word(a, w);
  __syncthreads();
  // what the pieces need, and the free pages of each chunk
#pragma unroll
  for (int i = 0; i < PT_HELD; ++i) {
    const int q = wv + 16 * i;
    if (q < pieces) {
      const int s = q / per, c = q % per * 64 + lane;
      const PtCols tc = pt_cols(sh.at[s], sh.n[s], t.sh);
      const unsigned long long m = __ballot(c >= tc.t0 && c < tc.t1 && !pt_page_ok(ids[i], t.pages));
      if (lane == 0) sh.need[q] = __popcll(m);
    }
  }
  for (int c = wv; c < a.chunks; c += 16) {
    const int w = c * PT_CHUNK + lane;
    const uint32_t n = wave_scan((uint32_t)(w < words ? __popcll(sh.free_[w]) : 0));
    if (lane == 63) sh.chunk[c] = (int)n;
  }
  __syncthreads();
  // who is served: sums of what is asked for, at most one more than there is of each, in 32
  // bits; the chunks' free pages, by every wave, a chunk a lane
  static_assert(PT_PAGES % (64 * PT_CHUNK) == 0 && PT_PAGES / (64 * PT_CHUNK) <= 64, "chunks: 4");
  const uint32_t own = lane < a.chunks ? (uint32_t)sh.chunk[lane] : 0, upto = wave_scan(own);
  const uint32_t free_pages = lane_of(upto, 63);
  const int n = tid < t.seqs ? sh.n[tid] : -1;
  int need = 0;
  if (n > 0)
    for (int i = 0; i < per; ++i) need += sh.need[tid * per + i];
  uint32_t x = (uint32_t)min(need, t.pages + 1), y = (uint32_t)min(max(n, 0), t.rows + 1), tx, ty;
  const uint32_t xi = x, yi = y;
  pt_sums<16>(x, y, tx, ty, sh.part[0]);   // behind its barrier the chunks' sums are read
  const bool ok = n >= 0 && y + yi <= (uint32_t)t.rows && (need == 0 || x + xi <= free_pages);
  x = ok ? (uint32_t)need : 0;
  y = ok ? (uint32_t)n : 0;
  pt_sums<16>(x, y, tx, ty, sh.part[1]);
  if (wv == 0 && lane < a.chunks) sh.chunk[lane] = (int)(upto - own);
  if (tid < t.seqs) {
    const int g = ok ? n : 0;
    sh.n[tid] = g;
    sh.base[tid] = (int)x;
    sh.first[tid] = (int)y;
    t.starts[tid] = (int)y;
    t.lens_out[tid] = sh.at[tid] + g;
  }
  if (tid == 0) {
    t.starts[t.seqs] = (int)ty;
    sh.rows = (int)ty;
  }
  __syncthreads();
  // tables and rows
#pragma unroll
  for (int i = 0; i < PT_HELD; ++i) {
    const int q = wv + 16 * i;
    if (q >= pieces) break;
    const int s = q / per, c0 = q % per * 64, c = c0 + lane, at = sh.at[s], n = sh.n[s];
    const PtCols tc = pt_cols(at, n, t.sh);
    int id = ids[i];
    const bool take = c >= tc.t0 && c < tc.t1 && !pt_page_ok(id, t.pages);
    const unsigned long long m = __ballot(take);
    if (m) {
      int rank = sh.base[s];
      for (int j = q - q % per; j < q; ++j) rank += sh.need[j];
      const int got = pt_page(sh.free_, sh.chunk, a.chunks, t.pages, take, rank + __popcll(m & ((1ull << lane) - 1)), rank);
      if (take) {
        id = got;
        if (got >= 0) t.refs_out[got] = 1;
      }
    }
    if (c < t.cols && (take || !(a.same & 1))) t.table_out[s * t.orow + c] = id;
    const int lo = max(at, c0 << t.sh), hi = (int)min((long long)at + n, (long long)(c0 + 64) << t.sh);
    const int row0 = sh.first[s] - at;
    for (int e0 = lo; e0 < hi; e0 += 64) {
      const int e = e0 + lane, p = __shfl(id, (e >> t.sh) - c0, 64);
      if (e < hi) {
        t.seq[row0 + e] = s;
        t.pos[row0 + e] = e;
        t.slot[row0 + e] = pt_page_ok(p, t.pages) ? ((long long)p << t.sh) + (e & ((1 << t.sh) - 1)) : -1;
      }
    }
  }
  for (int r = sh.rows + tid; r < t.rows; r += 1024) {
    t.seq[r] = -1;
    t.pos[r] = -1;
    t.slot[r] = -1;
  }
}

// ---- pages returned ---------------------------------------------------------------

__global__ __launch_bounds__(256) void k_refs_copy(const int32_t* __restrict__ in, int32_t* __restrict__ out,
                                                   int pages) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i < pages) out[i] = in[i];
}

// Columns behind a sequence's entries name no page any more; each one named counts
// one less.  Whole-number atomics: in any order the same counts.
__device__ __forceinline__ int pt_have(const TableArgs& t, int s) {   // columns that its entries touch
  return (int)(((long long)pg_len(t.lens[s], t.cols, t.sh) + (1 << t.sh) - 1) >> t.sh);
}
__global__ __launch_bounds__(256) void k_table_release(TableArgs t, int same) {
  const int tid = threadIdx.x, per = (t.cols + 63) / 64;   // waves a sequence
  for (long long w = (long long)blockIdx.x * 4 + (tid >> 6); w < (long long)t.seqs * per; w += (long long)gridDim.x * 4) {
    const int s = (int)(w / per), c = (int)(w % per) * 64 + (tid & 63);
    if (c >= t.cols) continue;
    const int id = t.table[s * t.trow + c];
    if (c >= pt_have(t, s)) {
      if (pt_page_ok(id, t.pages)) atomicSub(&t.refs_out[id], 1);
      if (id != -1 || !same) t.table_out[s * t.orow + c] = -1;
    } else if (!same) {
      t.table_out[s * t.orow + c] = id;
    }
  }
}
// The same by one work-group, which reads everything at once and counts in LDS.  64
// sequences of 64 columns, 12288 pages: 6.6 us, one call after another 7.1 (two launches
// 4.2, but 10.0, which is what the host takes); 256 of them 16.3 and 16.1.
constexpr int PT_COUNTS = 12288;
__global__ __launch_bounds__(1024) void k_table_release_one(TableArgs t, int same) {
  __shared__ int gone[PT_COUNTS];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int per = (t.cols + 63) / 64, pieces = t.seqs * per;
  int ids[PT_HELD], have[PT_HELD], refs[PT_COUNTS / 1024];
#pragma unroll
  for (int i = 0; i < PT_HELD; ++i) {
    const int q = wv + 16 * i;
    if (q < pieces) {
      ids[i] = t.table[(q / per) * t.trow + min(q % per * 64 + lane, t.cols - 1)];
      have[i] = t.lens[q / per];
    }
  }
#pragma unroll
  for (int i = 0; i < PT_COUNTS / 1024; ++i) {
    const int p = tid + 1024 * i;
    if (p < t.pages) refs[i] = t.refs[p];
    gone[p] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PT_HELD; ++i) {
    const int q = wv + 16 * i;
    if (q >= pieces) break;
    const int c = q % per * 64 + lane;
    if (c < t.cols) {
      int id = ids[i];
      const bool behind = c >= (int)(((long long)pg_len(have[i], t.cols, t.sh) + (1 << t.sh) - 1) >> t.sh);
      if (behind && pt_page_ok(id, t.pages)) atomicAdd(&gone[id], 1);
      if (behind ? id != -1 || !same : !same) t.table_out[(q / per) * t.orow + c] = behind ? -1 : id;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PT_COUNTS / 1024; ++i) {
    const int p = tid + 1024 * i;
    if (p < t.pages && (gone[p] || t.refs != t.refs_out)) t.refs_out[p] = refs[i] - gone[p];
  }
}

static int pt_spans(const TableArgs& t) {
  return (int)((((long long)t.cols << t.sh) + (1 << PT_SPAN) - 1) >> PT_SPAN);
}
static int pt_chunks(const TableArgs& t) { return (int)(((long long)t.pages + 64 * PT_CHUNK - 1) / (64 * PT_CHUNK)); }

static bool pt_held(const TableArgs& t) { return (long long)t.seqs * ((t.cols + 63) / 64) <= 16 * PT_HELD; }
static bool pt_one(const TableArgs& t) {
  return pt_held(t) && t.seqs <= PT_SEQS && t.pages <= PT_PAGES && t.rows <= PT_ROWS;
}

size_t table_assign_ws_bytes(const TableArgs& t) {
  if (pt_one(t)) return 0;
  const size_t words = ((size_t)t.pages + 63) / 64;
  return words * 8 + ((size_t)pt_chunks(t) + 1 + (size_t)t.seqs * (4 + (size_t)pt_spans(t))) * 4;
}

hipError_t table_assign(const TableArgs& t, void* ws, hipStream_t st) {
  PtArgs a{};
  a.t = t;
  a.same = (t.table == t.table_out) | (t.refs == t.refs_out) << 1;
  a.spans = pt_spans(t);
  a.chunks = pt_chunks(t);
  if (pt_one(t)) {
    hipLaunchKernelGGL(k_table_one, dim3(1), dim3(1024), 0, st, a);
    return hipGetLastError();
  }
  a.free_ = (unsigned long long*)ws;
  a.chunk = (int32_t*)(a.free_ + ((size_t)t.pages + 63) / 64);
  a.at = a.chunk + a.chunks + 1;
  a.n = a.at + t.seqs;
  a.need = a.n + t.seqs;
  a.base = a.need + t.seqs;
  a.before = a.base + t.seqs;
  const int sb = (t.seqs + 3) / 4;
  hipLaunchKernelGGL(k_table_need, dim3((unsigned)(sb + a.chunks)), dim3(256), 0, st, a, sb);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const long long all = (long long)t.seqs * a.spans, rows = ((long long)t.rows + 255) / 256;
  const long long most = all > rows ? all : rows;
  const dim3 grid((unsigned)(most < 1 ? 1 : most > 65536 ? 65536 : most));
  if (t.seqs >= 1 && t.seqs <= PT_SUMS && t.pages <= PT_SUM_PAGES && t.rows <= PT_SUM_ROWS) {
    hipLaunchKernelGGL(k_table_fill<true>, grid, dim3(256), 0, st, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(k_table_grant, dim3(1), dim3(1024), 0, st, a);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k_table_fill<false>, grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

hipError_t table_release(const TableArgs& t, hipStream_t st) {
  const int same = t.table == t.table_out;
  if (pt_held(t) && t.pages <= PT_COUNTS) {
    hipLaunchKernelGGL(k_table_release_one, dim3(1), dim3(1024), 0, st, t, same);
    return hipGetLastError();
  }
  if (t.refs != t.refs_out) {
    hipLaunchKernelGGL(k_refs_copy, dim3((unsigned)(((long long)t.pages + 255) / 256)), dim3(256), 0, st, t.refs,
                       t.refs_out, t.pages);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  const long long all = ((long long)t.seqs * ((t.cols + 63) / 64) + 3) / 4;
  if (all == 0) return hipSuccess;
  hipLaunchKernelGGL(k_table_release, dim3((unsigned)(all > 65536 ? 65536 : all)), dim3(256), 0, st, t, same);
  return hipGetLastError();
}

}  // namespace ann
