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
// Three launches, each a pass: needs, and the free pages as bits with the number in
// each chunk of 4096; one work-group's running sums of both, which say who is served;
// tables and row maps, a work-group for each span of 4096 entries of a sequence,
// whose waves find 64 pages at a time among the bits of a chunk.  A call that one
// work-group gets through in the time of a launch or two is one launch.
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
  const PtCols c = pt_cols(at, fits ? want : 0, sh);
  const int32_t* row = t.table + s * t.trow;
  const int spc = PT_SPAN - sh;   // log2 of a span's columns
  int need = 0;
  for (int c0 = c.t0; c0 < c.t1;) {
    // 64 columns at most, not past a span's end
    const int span = c0 >> spc, end = min(min(c0 + 64, c.t1), (span + 1) << spc);
    if (lane == 0 && (c0 == c.t0 || (c0 & ((1 << spc) - 1)) == 0))
      a.before[(long long)s * a.spans + span] = need;
    const int col = c0 + lane;
    need += __popcll(__ballot(col < end && !pt_page_ok(row[min(col, end - 1)], t.pages)));
    c0 = end;
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
__device__ __forceinline__ int pt_page(const PtArgs& a, bool want, int rank, int r0) {
  const int lane = threadIdx.x & 63;
  const int words = (int)(((long long)a.t.pages + 63) / 64);
  int id = -1;
  for (int c = pg_sequence(a.chunk, a.chunks, r0); c >= 0 && c < a.chunks && __any(want); ++c) {
    const int w = c * PT_CHUNK + lane;
    const unsigned long long m = w < words ? a.free_[w] : 0;
    const int pop = __popcll(m);
    int sum = pop;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(sum, o, 64);
      if (lane >= o) sum += v;
    }
    const int total = __shfl(sum, 63, 64), k = rank - a.chunk[c];
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

// Columns and rows of one span of a sequence, by a work-group of 256 threads at least
// (of which 256 have a column); page: 256 ids, cnt: 4 numbers, in LDS.
template <int NT>
__device__ __forceinline__ void pt_fill(const PtArgs& a, int s, int span, int* page, int* cnt) {
  const TableArgs& t = a.t;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int spc = PT_SPAN - t.sh;
  const int c0 = span << spc, c1 = min(t.cols, c0 + (1 << spc));
  const int at = a.at[s], n = a.n[s];
  const PtCols tc = pt_cols(at, n, t.sh);
  const bool touched = max(tc.t0, c0) < min(tc.t1, c1);
  if (!touched && (a.same & 1)) return;   // the same for all threads
  const int c = c0 + tid;
  int id = 0;
  bool take = false;
  if (tid < 256 && c < c1) {
    id = t.table[s * t.trow + c];
    take = c >= tc.t0 && c < tc.t1 && !pt_page_ok(id, t.pages);
  }
  if (touched) {
    const unsigned long long m = __ballot(take);
    if (wv < 4 && lane == 0) cnt[wv] = __popcll(m);
    __syncthreads();
    if (m) {   // of this wave
      int r0 = a.base[s] + a.before[(long long)s * a.spans + span];
      for (int w = 0; w < wv; ++w) r0 += cnt[w];
      const int got = pt_page(a, take, r0 + __popcll(m & ((1ull << lane) - 1)), r0);
      if (take) {
        id = got;
        if (got >= 0) t.refs_out[got] = 1;
      }
    }
    if (tid < 256) page[tid] = id;
  }
  if (tid < 256 && c < c1 && (take || !(a.same & 1))) t.table_out[s * t.orow + c] = id;
  if (!touched) return;
  __syncthreads();
  const int lo = max(at, c0 << t.sh), hi = (int)min((long long)at + n, (long long)c1 << t.sh);
  const int row0 = t.starts[s] - at;
  for (int e = lo + tid; e < hi; e += NT) {
    const int p = page[(e >> t.sh) - c0], r = row0 + e;
    t.seq[r] = s;
    t.pos[r] = e;
    t.slot[r] = pt_page_ok(p, t.pages) ? ((long long)p << t.sh) + (e & ((1 << t.sh) - 1)) : -1;
  }
  __syncthreads();   // page and cnt are used again
}

// Rows behind the last sequence's.
__device__ __forceinline__ void pt_behind(const TableArgs& t, int first, int step) {
  for (int r = t.starts[t.seqs] + first; r < t.rows; r += step) {
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

__global__ __launch_bounds__(256) void k_table_fill(PtArgs a) {
  __shared__ int page[256], cnt[4];
  const long long all = (long long)a.t.seqs * a.spans;
  for (long long w = blockIdx.x; w < all; w += gridDim.x)
    pt_fill<256>(a, (int)(w / a.spans), (int)(w % a.spans), page, cnt);
  pt_behind(a.t, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

// ---- pages returned ---------------------------------------------------------------

__global__ __launch_bounds__(256) void k_refs_copy(const int32_t* __restrict__ in, int32_t* __restrict__ out,
                                                   int pages) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i < pages) out[i] = in[i];
}

// Columns behind a sequence's entries name no page any more; each one named counts
// one less.  Whole-number atomics: in any order the same counts.
__global__ __launch_bounds__(256) void k_table_release(TableArgs t, int same) {
  const int tid = threadIdx.x;
  const int per = (t.cols + 255) / 256;   // work-groups a sequence
  for (long long w = blockIdx.x; w < (long long)t.seqs * per; w += gridDim.x) {
    const int s = (int)(w / per), c = (int)(w % per) * 256 + tid;
    if (c >= t.cols) continue;
    const int have = (int)(((long long)pg_len(t.lens[s], t.cols, t.sh) + (1 << t.sh) - 1) >> t.sh);
    int id = t.table[s * t.trow + c];
    if (c >= have) {
      if (pt_page_ok(id, t.pages)) atomicSub(&t.refs_out[id], 1);
      if (id != -1 || !same) t.table_out[s * t.orow + c] = -1;
    } else if (!same) {
      t.table_out[s * t.orow + c] = id;
    }
  }
}

static int pt_spans(const TableArgs& t) {
  return (int)((((long long)t.cols << t.sh) + (1 << PT_SPAN) - 1) >> PT_SPAN);
}
static int pt_chunks(const TableArgs& t) { return (int)(((long long)t.pages + 64 * PT_CHUNK - 1) / (64 * PT_CHUNK)); }

size_t table_assign_ws_bytes(const TableArgs& t) {
  const size_t words = ((size_t)t.pages + 63) / 64;
  return words * 8 + ((size_t)pt_chunks(t) + 1 + (size_t)t.seqs * (4 + (size_t)pt_spans(t))) * 4;
}

hipError_t table_assign(const TableArgs& t, void* ws, hipStream_t st) {
  PtArgs a{};
  a.t = t;
  a.same = (t.table == t.table_out) | (t.refs == t.refs_out) << 1;
  a.spans = pt_spans(t);
  a.chunks = pt_chunks(t);
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
  hipLaunchKernelGGL(k_table_grant, dim3(1), dim3(1024), 0, st, a);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  const long long all = (long long)t.seqs * a.spans, rows = ((long long)t.rows + 255) / 256;
  const long long grid = all > rows ? all : rows;
  hipLaunchKernelGGL(k_table_fill, dim3((unsigned)(grid < 1 ? 1 : grid > 65536 ? 65536 : grid)), dim3(256), 0, st, a);
  return hipGetLastError();
}

hipError_t table_release(const TableArgs& t, hipStream_t st) {
  if (t.refs != t.refs_out) {
    hipLaunchKernelGGL(k_refs_copy, dim3((unsigned)(((long long)t.pages + 255) / 256)), dim3(256), 0, st, t.refs,
                       t.refs_out, t.pages);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  const long long all = (long long)t.seqs * ((t.cols + 255) / 256);
  if (all == 0) return hipSuccess;
  hipLaunchKernelGGL(k_table_release, dim3((unsigned)(all > 65536 ? 65536 : all)), dim3(256), 0, st, t,
                     t.table == t.table_out);
  return hipGetLastError();
}

}  // namespace ann
