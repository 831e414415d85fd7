// Attention of new tokens over a paged key/value cache, and the weight that
// each entry receives from them.
//
// A token at entry e sees the entries j <= e and, with a window, e - j < window.
//   s_j = scale q.k_j,  lse = log sum_j exp(s_j),  o = sum_j exp(s_j - lse) v_j
//   w'_j = w_j + sum over the new tokens and heads of exp(s_j - lse)
// A token that sees nothing gets o = 0 and lse = -inf.
#include <math.h>
#include <type_traits>
#include "common.h"
#include "launch.h"

namespace ann {

// The kernels' window: INT_MAX for none, as for one past the largest table.
static int pa_window(int window) { return window > 0 && window <= 1 << 30 ? window : 0x7fffffff; }

constexpr float PA_LOG2E = 1.4426950408889634f, PA_LN2 = 0.6931471805599453f;

// One row (token, head) by one wave: 64 entries at a time, a lane for each
// entry's score, then DH / 64 dims of the sum for each lane.  lo .. hi - 1 are
// the entries it sees.
template <int DH>
__device__ __forceinline__ void pa_row(const PagedArgs& c, const int32_t* __restrict__ table,
                                       const bf16_t* __restrict__ q, int kvh, int lo, int hi,
                                       float sl2, float& m, float& l, float* o) {
  constexpr int DL = DH / 64;
  const int lane = threadIdx.x & 63;
  m = -INFINITY;
  l = 0.f;
#pragma unroll
  for (int d = 0; d < DL; ++d) o[d] = 0.f;
  for (int j0 = lo; j0 < hi; j0 += 64) {
    const int j = min(j0 + lane, hi - 1);
    const int id = pg_read(table[j >> c.sh], c.pages);
    const bf16_t* kr = c.k + id * c.kp + kvh * c.kh + pg_slot(j, c.sh, c.ks);
    float s = 0.f;
    for (int d = 0; d < DH; d += 8) {
      float x[8], y[8];
      unpack8(*(const uint4*)(kr + d), x);
      unpack8(*(const uint4*)(q + d), y);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += x[e] * y[e];
    }
    s = j0 + lane < hi ? s * sl2 : -INFINITY;
    const float mt = group_max<64>(s), mn = fmaxf(m, mt);
    const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
    const float p = j0 + lane < hi ? __builtin_amdgcn_exp2f(s - (mn == -INFINITY ? 0.f : mn)) : 0.f;
    m = mn;
    l = l * f + group_sum<64>(p);
#pragma unroll
    for (int d = 0; d < DL; ++d) o[d] *= f;
    const int nj = min(64, hi - j0);
    for (int i = 0; i < nj; ++i) {
      const int e = j0 + i;
      const float pi = __shfl(p, i, 64);
      const bf16_t* vr = c.v + pg_read(table[e >> c.sh], c.pages) * c.vp + kvh * c.vh +
                         pg_slot(e, c.sh, c.vs) + lane * DL;
#pragma unroll
      for (int d = 0; d < DL; ++d) o[d] += pi * bf2f(vr[d]);
    }
  }
}

// ---- tiles ------------------------------------------------------------------------
//
// Rows of a (sequence, cache head): G = heads / cache heads of them for each new
// token, row r being token r / G and head r % G of the group, so heads that share
// keys and values share their loads.  A tile of rows walks the entries that any of
// them sees in steps of 32 (64 at head dim 64):
//   S^T = K Q^T   (v_mfma_f32_16x16x32_bf16: 16 entries x 16 rows)
//   p = exp2(scale (s - m)), the sum of p
//   O^T += V^T P^T
// Rows are the columns of both products, so S^T leaves the matrix unit in the
// layout in which P^T enters it: k index g * 8 + e of a lane is entry 4 g + e (e <
// 4) or 16 + 4 g + e - 4.  V^T comes out of the row-major tile by ds_read_b64_tr_b16,
// as in the prefill attention (attn.hip).  m is a running maximum that is raised
// only where a score passes it by more than 2^8 in p: p stays at most 2^8, sums in
// fp32 far from their range, and the accumulators are seldom rescaled.  P is
// rounded to bf16 (relative 2^-8 of each weight, as the framework's attention
// rounds it); its sum is of the unrounded weights.  What that leaves of each weight as a
// second half, as few rows have it, takes the mean relative error from 0.0023 to 0.0017
// (the result's own rounding) and 230 us of 2048 tokens on 16384 entries to 285.
//
// Entries outside what a tile sees are not read: a lane past an end reads the
// nearest entry inside, masked.  What is masked for one row of a tile and seen by
// another is multiplied by zero, which keeps an infinity or a NaN; a row whose sum
// is not finite is therefore formed again, entry by entry, from what it sees alone.

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float floatx4_t __attribute__((ext_vector_type(4)));
typedef short pa_v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void pa_lds_void;
typedef __attribute__((address_space(3))) const unsigned char pa_lds_cchar;

// 16-byte chunk c of LDS row r is stored at chunk c ^ kswz(r) of a key tile and c
// ^ swz(r) of a value tile.  A fragment of keys is 16 rows of one chunk each,
// which the hardware reads 16 lanes at a time from two neighbouring chunks; one of
// values 8 rows of two chunks.  Measured with one wave, cycles for 1 KB of keys: 5
// with kswz, 8 with swz, 32 unswizzled; for 512 bytes of values 4.25 and 16 (with
// all waves 4.4 and 2.6, as for reads in a row).
template <int DH>
__device__ __forceinline__ int pa_kswz(int r) {
  return DH == 128 ? r & 15 : r & 7;
}
template <int DH>
__device__ __forceinline__ int pa_swz(int r) {
  return DH == 128 ? (((r & 7) << 1) | ((r >> 3) & 1)) : ((r >> 1) & 7);
}
template <int N>
__device__ __forceinline__ void pa_wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}
// LDS reads as inline assembly: the compiler would wait for every load into LDS
// in flight before each; the waits here are by hand (LDS reads return in order).
template <int OFF>
__device__ __forceinline__ bf16x8_t pa_rd_b128(pa_lds_cchar* p) {
  bf16x8_t v;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v) : "v"(p), "i"(OFF));
  return v;
}
template <int OFF>
__device__ __forceinline__ pa_v4i16 pa_rd_tr(pa_lds_cchar* p) {
  pa_v4i16 v;
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(v) : "v"(p), "i"(OFF));
  return v;
}
template <int N, typename X>
__device__ __forceinline__ void pa_wait_lgkm(X& x) {
  asm volatile("s_waitcnt lgkmcnt(%1)" : "+v"(x) : "i"(N));
}
template <int N, typename X>
__device__ __forceinline__ void pa_wait_lgkm2(X& x, X& y) {
  asm volatile("s_waitcnt lgkmcnt(%2)" : "+v"(x), "+v"(y) : "i"(N));
}
template <int I, int N, typename F>
__device__ __forceinline__ void pa_static_for(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    pa_static_for<I + 1, N>(f);
  }
}

// How a tile's entries [lo, hi) are shared out: n parts of `per` entries from lo
// rounded down to 32, per a multiple of 64.  As many as the call is split into, of
// 128 entries at least and 4096 at most where `most` parts allow it: a sequence far
// longer than the others does not keep one work-group.
struct PaSplit {
  int split, most;
};
struct PaParts {
  int begin, per, n;
};
__device__ __forceinline__ PaParts pa_parts(int lo, int hi, PaSplit sp) {
  PaParts p;
  p.begin = lo & ~31;
  const int total = hi - p.begin;
  if (hi <= lo) return {0, 64, 1};
  if (sp.most == 1) return {p.begin, (total + 63) & ~63, 1};
  const int n = min(sp.most, max(min(sp.split, (total + 127) / 128), (total + 4095) / 4096));
  p.per = ((total + n - 1) / n + 63) & ~63;
  p.n = (total + p.per - 1) / p.per;
  return p;
}

struct PaArgs {
  PagedArgs c;
  const bf16_t* q;
  long long qt, qh;
  int heads, window;   // window: none is INT_MAX
  int G;               // heads / cache heads
  FastDiv by;          // division by G
  float sl2, thr;      // |scale| log2(e); 8 / sl2, the rise of m's that is let pass
  float ssl2;          // scale log2(e)
  uint32_t keep, flip; // of the queries' words: the bits kept (scale 0: none, sl2 is 1) and turned (below 0: signs)
  bf16_t* out;
  float* lse;
  // parts of a row's sums (slots, most, DH), and (slots, most): m in log2 units, sum
  float* po_few;
  float* po_many;
  float2* ml_few;
  float2* ml_many;
  PaSplit sp_few, sp_many;
  int few;             // rows of a sequence up to which pa_few takes it
  int packed;          // slots of pa_few: 16 a (sequence, cache head), else as pa_many's, (rows, heads)
  int br;              // rows of pa_many's tiles
};

// One sequence's new tokens as a call sees them.
struct PaSeq {
  int first, n, len, rows, G, e0;   // e0: entry of token 0
  FastDiv by;                       // division by G
};
__device__ __forceinline__ PaSeq pa_seq(const PaArgs& a, PgRange r, int len) {
  PaSeq q;
  q.first = r.first;
  q.n = r.n;
  q.len = pg_len(len, a.c.cols, a.c.sh);
  q.G = a.G;
  q.by = a.by;
  q.rows = r.n * q.G;
  q.e0 = q.len - r.n;
  return q;
}
__device__ __forceinline__ PaSeq pa_seq(const PaArgs& a, int s) {
  return pa_seq(a, pg_range(a.c.starts[s], a.c.starts[s + 1], a.c.rows), a.c.lens[s]);
}
// The entries that rows row0 .. row0 + n - 1 see.
__device__ __forceinline__ void pa_span(const PaSeq& q, int row0, int n, int window, int& lo, int& hi) {
  const int el = q.e0 + q.by.div(row0), eh = q.e0 + q.by.div(row0 + n - 1);
  lo = el < window ? 0 : el - window + 1;
  hi = max(eh + 1, 0);
}

// A row of a tile: its token and head, and where the sums of its part go.
struct PaRow {
  int n, h;
  long long at;   // slot * most + part
};
template <bool FEW>
__device__ __forceinline__ PaRow pa_place(const PaArgs& a, const PaSeq& q, int s, int kvh, int row,
                                          int part) {
  PaRow r;
  const int tok = q.by.div(row);
  r.n = q.first + tok;
  r.h = kvh * q.G + row - tok * q.G;
  const long long slot = FEW && a.packed ? ((long long)s * a.c.heads + kvh) * 16 + row
                                         : (long long)r.n * a.heads + r.h;
  r.at = slot * (FEW ? a.sp_few.most : a.sp_many.most) + part;
  return r;
}

// Final (parts == 1) or partial result of a row: 4 dims from d on.
template <int DH, bool FEW>
__device__ __forceinline__ void pa_store4(const PaArgs& a, const PaRow& w, int parts, int d, float4 o,
                                          float m, float l) {
  const long long r = (long long)w.n * a.heads + w.h;
  if (parts == 1) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *(uint2*)(a.out + r * DH + d) =
        make_uint2(pack2(o.x * inv, o.y * inv), pack2(o.z * inv, o.w * inv));
    if (d == 0 && a.lse)
      a.lse[r] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * PA_LN2;
  } else {
    *(float4*)((FEW ? a.po_few : a.po_many) + w.at * DH + d) = o;
    if (d == 0) (FEW ? a.ml_few : a.ml_many)[w.at] = make_float2(m, l);
  }
}

// A row formed entry by entry, over the part [a0, b0) of what it sees.
template <int DH, bool FEW>
__device__ __forceinline__ void pa_again(const PaArgs& a, const PaSeq& q, int s,
                                         const int32_t* table, int kvh, int row, int a0, int b0,
                                         int part, int parts) {
  constexpr int DL = DH / 64;
  const int lane = threadIdx.x & 63;
  const PaRow w = pa_place<FEW>(a, q, s, kvh, row, part);
  const int e = q.e0 + q.by.div(row);
  const int lo = max(a0, e < a.window ? 0 : e - a.window + 1), hi = min(b0, e + 1);
  float m, l, o[DL];
  pa_row<DH>(a.c, table, a.q + w.n * a.qt + w.h * a.qh, kvh, lo, hi, a.ssl2, m, l, o);
  // lane i holds dims i DL ..: four lanes' (two's) values to the one that stores them
  float4 v;
  if constexpr (DL == 1) {
    v = make_float4(o[0], __shfl_down(o[0], 1, 64), __shfl_down(o[0], 2, 64), __shfl_down(o[0], 3, 64));
    if (lane % 4 == 0) pa_store4<DH, FEW>(a, w, parts, lane, v, m, l);
  } else {
    v = make_float4(o[0], o[1], __shfl_down(o[0], 1, 64), __shfl_down(o[1], 1, 64));
    if (lane % 2 == 0) pa_store4<DH, FEW>(a, w, parts, lane * 2, v, m, l);
  }
}

__device__ __forceinline__ bool pa_finite(const floatx4_t& v) {
  // 0 times a finite number is 0, times any other NaN
  const float z = v[0] * 0.f + v[1] * 0.f + v[2] * 0.f + v[3] * 0.f;
  return z == 0.f;
}

// The running maximum raised to the largest score, of which each of a row's four
// lanes knows its own: where one passes it by more than a.thr.
template <int NDB>
__device__ __forceinline__ void pa_raise(float lm, float sl2, float& m, float& msl, float& lsum,
                                         floatx4_t* o) {
  lm = fmaxf(lm, __shfl_xor(lm, 16, 64));
  lm = fmaxf(lm, __shfl_xor(lm, 32, 64));
  const float mn = fmaxf(m, lm);
  const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mn) * sl2);
  m = mn;
  msl = mn == -INFINITY ? 0.f : mn * sl2;
  lsum *= f;
#pragma unroll
  for (int i = 0; i < NDB; ++i) o[i] *= f;
}

// 8 values with the scale's sign: products are with |scale| then, whose largest
// score is the largest product.
__device__ __forceinline__ bf16x8_t pa_signed(const bf16_t* p, uint32_t keep, uint32_t flip) {
  uint4 w = *(const uint4*)p;
  w.x = (w.x & keep) ^ flip;
  w.y = (w.y & keep) ^ flip;
  w.z = (w.z & keep) ^ flip;
  w.w = (w.w & keep) ^ flip;
  return __builtin_bit_cast(bf16x8_t, w);
}

__device__ __forceinline__ bf16x8_t pa_join(pa_v4i16 a, pa_v4i16 b) {
  return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// ---- sequences of few rows ----------------------------------------------------------
//
// A work-group takes a part of a sequence's entries for one cache head and 16 rows
// (one row of a decoding sequence without shared heads).  Its NW waves
// take chunks of 32 entries in turn and meet only at the end: keys from memory
// straight into the fragments of the product, a chunk ahead; values into the
// wave's own ring of two LDS stages.  The products have time to spare here, and the
// weights enter as two bf16 halves (2^-17 of each).  Bound by memory on long caches
// (one token on 16 x 8192 entries of 6 heads of 128 in 5 parts: 59 us and 5 to join
// them, 290 MB, 4.5 TB/s of a copy's 5.2), by the wait for one read after another and
// a chunk's some 270 instructions a wave on short ones (777 entries: 11.7 us a call;
// 13.0 with the page ids read only behind the length, divisions by the group, every
// chunk's addresses formed from its page id and every chunk masked).
template <int DH, int NW>
constexpr size_t pa_few_lds() {
  // the rings; after them the waves' sums, their maxima and totals, rows to form again
  const size_t ring = (size_t)NW * 2 * 32 * DH * 2;
  const size_t sums = ((size_t)NW * 16 * (DH + 4) + 2 * NW * 16 + 16) * 4;
  return ring > sums ? ring : sums;
}
template <int DH, int NW>
__device__ __forceinline__ void pa_few(const PaArgs& a, int s, int row0, int kvh, int part,
                                       unsigned char* smem) {
  constexpr int RB = DH * 2, TB = 32 * RB;      // bytes of an LDS row, of a chunk's values
  constexpr int LPW = TB / 1024, RPL = 1024 / RB;   // loads of a chunk's values, rows of each
  constexpr int NKS = DH / 32, NDB = DH / 16, PW = DH + 4;
  float* sums = (float*)smem;
  float* s_m = sums + NW * 16 * PW;
  float* s_l = s_m + NW * 16;
  int* s_bad = (int*)(s_l + NW * 16);

  const int tid = threadIdx.x, lane = tid & 63;
  const int32_t* table = a.c.table + s * a.c.trow;
  // the first 64 page ids, on their way before the sequence's length is known
  const int first = a.c.cols ? table[min(lane, a.c.cols - 1)] : 0;
  const PaSeq q = pa_seq(a, s);
  if (row0 >= q.rows || q.rows > a.few) return;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, g4 = lane >> 4;
  const bf16_t* kh = a.c.k + kvh * a.c.kh;
  const bf16_t* vh = a.c.v + kvh * a.c.vh;
  unsigned char* ring = smem + wv * 2 * TB;
  const int trow = 4 * g4 + (r16 >> 2), tcol = 4 * (r16 & 3), vx = pa_swz<DH>(trow);

  const int nrow = min(16, q.rows - row0);
  int lo, hi;
  pa_span(q, row0, nrow, a.window, lo, hi);
  const PaParts pt = pa_parts(lo, hi, a.sp_few);
  if (part >= pt.n) return;
  const int a0 = max(pt.begin + part * pt.per, lo), b0 = min(pt.begin + (part + 1) * pt.per, hi);
  const int kb0 = pt.begin + part * pt.per;
  const int nch = b0 > a0 ? (b0 - kb0 + 31) / 32 : 0;
  const int nt = nch > wv ? (nch - wv + NW - 1) / NW : 0;   // chunks of this wave

  const int row = row0 + min(r16, nrow - 1), tok = q.by.div(row);
  // the entries that this lane's row sees of its part, from the lane's first one on
  const int e = q.e0 + tok;
  const int jl = max(a0, e < a.window ? 0 : e - a.window + 1) - 4 * g4, jh = min(b0 - 1, e) - 4 * g4;
  // and those that all rows see
  const int el = q.e0 + q.by.div(row0), eh = q.e0 + q.by.div(row0 + nrow - 1);
  const int seen0 = max(a0, eh < a.window ? 0 : eh - a.window + 1), seen1 = min(b0 - 1, el);
  const bf16_t* qr = a.q + (q.first + tok) * a.qt + (kvh * q.G + row - tok * q.G) * a.qh + g4 * 8;
  bf16x8_t qf[NKS];
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) qf[ks] = pa_signed(qr + ks * 32, a.keep, a.flip);

  floatx4_t o[NDB];
#pragma unroll
  for (int i = 0; i < NDB; ++i) o[i] = (floatx4_t){0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, msl = 0.f, lsum = 0.f;

  // Of chunks 32 b .. 32 b + 31 of this wave lane i has group i & 1 of chunk i >> 1:
  // its first entry (where all of it lies outside [a0, b0), the nearest group's), the
  // page id, and the offsets in bytes within a head that come of them.  The next 32
  // chunks' ids come ahead.
  auto place = [&](int b) {
    const int key = kb0 + 32 * (wv + NW * (32 * b + (lane >> 1))) + 16 * (lane & 1);
    return min(max(key, a0 & ~15), (b0 - 1) & ~15);
  };
  auto ids = [&](int b) {
    const int col = place(b) >> a.c.sh;
    return pg_read((b0 - 1) >> a.c.sh < 64 ? __shfl(first, col, 64) : table[col], a.c.pages);
  };
  int klo = 0, khi = 0, vlo = 0, vhi = 0, next = nt ? ids(0) : 0;
  auto turn = [&](int b) {
    const int k0 = place(b);
    const long long ko = (next * a.c.kp + pg_slot(k0, a.c.sh, a.c.ks)) * 2;
    const long long vo = (next * a.c.vp + pg_slot(k0, a.c.sh, a.c.vs)) * 2;
    klo = (int)ko;
    khi = (int)(ko >> 32);
    vlo = (int)vo;
    vhi = (int)(vo >> 32);
    if (32 * (b + 1) < nt) next = ids(b + 1);
  };
  const auto group = [&](const bf16_t* head, int lo, int hi, int i) {
    const unsigned l = __builtin_amdgcn_readlane(lo, i);
    return (const unsigned char*)head + (((long long)__builtin_amdgcn_readlane(hi, i) << 32) | l);
  };
  bf16x8_t kf[2][2][NKS];
  auto issue = [&](int t, int slot) {
    asm volatile("" ::: "memory");   // behind the reads of the stage it fills
    if (t % 32 == 0) turn(t / 32);
    const int kb = kb0 + 32 * (wv + NW * t), i = 2 * (t % 32);
    unsigned char* st = ring + (t & 1) * TB;
    const bool edge = kb < a0 || kb + 32 > b0;   // rows outside take the nearest inside
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const unsigned char* kp = group(kh, klo, khi, i + g);
      const unsigned char* vp = group(vh, vlo, vhi, i + g);
      int kr = r16, vr[LPW / 2];
#pragma unroll
      for (int u = 0; u < LPW / 2; ++u) vr[u] = u * RPL + lane / (RB / 16);   // row of the group
      if (edge) {
        const int k0 = min(max(kb + 16 * g, a0 & ~15), (b0 - 1) & ~15);
        const int rl = max(a0 - k0, 0), rh = min(b0 - 1 - k0, 15);
        kr = min(max(kr, rl), rh);
#pragma unroll
        for (int u = 0; u < LPW / 2; ++u) vr[u] = min(max(vr[u], rl), rh);
      }
      const unsigned ko = (unsigned)(kr * (int)a.c.ks * 2 + g4 * 16);
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) kf[slot][g][ks] = *(const bf16x8_t*)(kp + ko + ks * 64);
#pragma unroll
      for (int u = 0; u < LPW / 2; ++u) {
        const int r = u * RPL + lane / (RB / 16);
        const int col = ((lane % (RB / 16)) ^ pa_swz<DH>(r)) * 16;
        const unsigned char* src = vp + (unsigned)(vr[u] * (int)a.c.vs * 2 + col);
        __builtin_amdgcn_global_load_lds(src, (pa_lds_void*)(st + (g * LPW / 2 + u) * 1024), 16, 0, 0);
      }
    }
  };
  auto compute = [&](int t, int slot) {
    const int kb = kb0 + 32 * (wv + NW * t);
    floatx4_t sacc[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      sacc[g] = (floatx4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks)
        sacc[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[slot][g][ks], qf[ks], sacc[g], 0, 0, 0);
    }
    if (kb < seen0 || kb + 31 > seen1)   // what is masked scores -inf
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = kb + 16 * g + r;
          sacc[g][r] = j >= jl && j <= jh ? sacc[g][r] : -INFINITY;
        }
    float p[2][4], lm = sacc[0][0];
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int r = 0; r < 4; ++r) lm = fmaxf(lm, sacc[g][r]);
    if (__any(lm > m + a.thr)) pa_raise<NDB>(lm, a.sl2, m, msl, lsum, o);
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[g][r] = __builtin_amdgcn_exp2f(sacc[g][r] * a.sl2 - msl);
        lsum += p[g][r];
      }
    uint32_t pw[4], pl[4];   // the weights in bf16, and what that leaves of them
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float u = p[x >> 1][(x & 1) * 2], v = p[x >> 1][(x & 1) * 2 + 1];
      pw[x] = pack2(u, v);
      pl[x] = pack2(u - lo_f(pw[x]), v - hi_f(pw[x]));
    }
    const bf16x8_t pf = *(const bf16x8_t*)pw, pr = *(const bf16x8_t*)pl;
    pa_lds_cchar* vst = (pa_lds_cchar*)(ring + (t & 1) * TB) + trow * RB + (tcol & 7) * 2;
    pa_v4i16 v0[NDB], v1[NDB];
    pa_static_for<0, NDB>([&](auto dc) __attribute__((always_inline)) {
      constexpr int db = decltype(dc)::value;
      pa_lds_cchar* src = vst + (((2 * db + (tcol >> 3)) ^ vx) << 4);
      v0[db] = pa_rd_tr<0>(src);
      v1[db] = pa_rd_tr<16 * RB>(src);
    });
    pa_static_for<0, NDB>([&](auto dc) __attribute__((always_inline)) {
      constexpr int db = decltype(dc)::value;
      pa_wait_lgkm2<2 * (NDB - 1 - db)>(v0[db], v1[db]);
      const bf16x8_t vf = pa_join(v0[db], v1[db]);
      o[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf, o[db], 0, 0, 0);
      o[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pr, o[db], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  if (nt) issue(0, 0);
  for (int t = 0; t < nt; t += 2) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (t + u < nt) {
        if (t + u + 1 < nt) {
          issue(t + u + 1, (u + 1) & 1);
          pa_wait_vm<LPW + 2 * NKS>();   // all but the next chunk's
        } else {
          pa_wait_vm<0>();
        }
        compute(t + u, u);
      }
    }
  }

  // the four waves' sums, brought to their largest maximum, in wave order
  lsum += __shfl_xor(lsum, 16, 64);
  lsum += __shfl_xor(lsum, 32, 64);
  __syncthreads();   // every wave is done with the ring
  if (r16 < nrow) {
#pragma unroll
    for (int db = 0; db < NDB; ++db)
      *(floatx4_t*)(sums + (wv * 16 + r16) * PW + db * 16 + g4 * 4) = o[db];
    if (g4 == 0) {
      s_m[wv * 16 + r16] = m == -INFINITY ? -INFINITY : m * a.sl2;
      s_l[wv * 16 + r16] = lsum;
    }
  }
  if (tid < 16) s_bad[tid] = 0;
  __syncthreads();
  // a thread's four dims of up to NI rows; one row alone may see an infinity too,
  // which the halves of its weight, or the zeros behind a chunk's end, make a NaN
  constexpr int NI = (16 * (DH / 4) + 64 * NW - 1) / (64 * NW);
  floatx4_t v[NI];
  float M[NI], L[NI];
#pragma unroll
  for (int k = 0; k < NI; ++k) {
    const int i = tid + k * 64 * NW, r = i / (DH / 4), d = i % (DH / 4) * 4;
    if (r >= nrow) break;
    M[k] = s_m[r];
#pragma unroll
    for (int w = 1; w < NW; ++w) M[k] = fmaxf(M[k], s_m[w * 16 + r]);
    L[k] = 0.f;
    v[k] = (floatx4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = M[k] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(s_m[w * 16 + r] - M[k]);
      L[k] += s_l[w * 16 + r] * f;
      v[k] += *(const floatx4_t*)(sums + (w * 16 + r) * PW + d) * f;
    }
    if (!pa_finite(v[k])) s_bad[r] = 1;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < NI; ++k) {
    const int i = tid + k * 64 * NW, r = i / (DH / 4), d = i % (DH / 4) * 4;
    if (r >= nrow || s_bad[r]) continue;
    pa_store4<DH, true>(a, pa_place<true>(a, q, s, kvh, row0 + r, part), pt.n, d,
                        make_float4(v[k][0], v[k][1], v[k][2], v[k][3]), M[k], L[k]);
  }
  for (int r = wv; r < nrow; r += NW)
    if (s_bad[r]) pa_again<DH, true>(a, q, s, table, kvh, row0 + r, a0, b0, part, pt.n);
}

// Work-groups past the sequences' take the sixteens of rows behind a sequence's first:
// in the order of all the call's rows (token, head of the group), number x the one
// that begins among rows 16 x .. 16 x + 15, of which there is one at most, its
// sequence having begun at least 16 rows before.  A call with as many sequences as
// tokens may still bring most of them to one (a captured step of many slots): 512
// tokens on 2000 entries beside 511 empty sequences 42 us (one work-group for all of a
// sequence's rows: 619), where every sequence has one token nothing is lost.
template <int DH, int NW>
__global__ __launch_bounds__(64 * NW, 2) void k_paged_few(PaArgs a, int blocks) {
  extern __shared__ __attribute__((aligned(16))) unsigned char pa_smem[];
  const int i = blockIdx.z * gridDim.y + blockIdx.y;
  if (i >= blocks) return;
  int s = i, row0 = 0;
  if (i >= a.c.seqs) {
    const int at = 16 * (i - a.c.seqs + 1);
    s = __builtin_amdgcn_readfirstlane(pg_sequence(a.c.starts, a.c.seqs, a.by.div(at)));
    if (s < 0) return;
    row0 = (at - pg_range(a.c.starts[s], a.c.starts[s + 1], a.c.rows).first * a.G + 15) & ~15;
    if (row0 == 0) return;
  }
  pa_few<DH, NW>(a, s, row0, blockIdx.x % a.c.heads, blockIdx.x / a.c.heads, pa_smem);
}

// ---- sequences of many rows -----------------------------------------------------------
//
// A work-group takes BR = 64 QB rows (four waves of QB x 16) and a part of the
// entries, which pass through a ring of two LDS stages shared by its waves: loaded
// straight into LDS a step ahead, one barrier a step.  A key or value fragment
// read from LDS serves QB products.  Bound by three units that a step needs for about
// as long, in cycles for one wave on each SIMD: the matrix units 512, the vector units
// some 600 (an exponential takes four instructions' time), LDS 430 (300 of reads).  A
// model of the step without its LDS reads takes 196 ns a wave at 2.4 GHz, with them
// 317, with barrier and loads 358; here it is 440 at the 2.0 GHz that the card holds
// under real data, and 650 where a CU has one work-group alone.
// 2048 tokens of 12 heads of 128 on 16384 entries: 227 us, 193 GFLOP at 0.85 PFLOP/s
// (a large product of the same card: 1.38), matrix units busy 40% of the time, no bank
// conflicts; its 768 work-groups fill 512 places once and half again.  24 ragged
// sequences on a window of 384, 50 MB and 4 GFLOP, take 20.2 us: a dozen steps behind
// the search for the tile.  No faster: three steps ahead, higher priority of waves in
// the products (230 and 233), sums and maxima beside the products with P (228), the
// first key fragments read a step ahead (226, and 21.9 for the ragged ones), parts by
// thirds, fifths and sixths.
constexpr int PM_AHEAD = 1;   // steps that loads run ahead (odd: a step's parity is its stage's)
template <int LPW>
struct PaWalk {
  const unsigned char* head;
  long long page, slot;
  int lo, hi, next;    // lane i: offset of group i in bytes; page id of group i of the next batch
  unsigned off[LPW];   // this lane's row and column in the group of load u, bytes
};
template <int DH, int BK>
constexpr size_t pa_many_lds() { return (size_t)2 * (PM_AHEAD + 1) * BK * DH * 2; }
template <int DH, int BK, int QB>
__device__ __forceinline__ void pa_many(const PaArgs& a, int tile, int kvh, int part,
                                        unsigned char* smem) {
  constexpr int BR = 64 * QB, RB = DH * 2, TB = BK * RB;
  constexpr int LPW = TB / 1024 / 4, RPL = 1024 / RB;   // loads a wave makes of K (and of V), rows of each
  constexpr int NKS = DH / 32, NDB = DH / 16, NBLK = BK / 16, NI = BK / 32;
  constexpr int NS = PM_AHEAD + 1;   // stages of keys, and of values

  const PgTile pl = pg_tile(a.c.starts, a.c.lens, a.c.seqs, a.c.rows, a.G, a.few, BR, tile);
  if (pl.seq < 0) return;
  const int s = __builtin_amdgcn_readfirstlane(pl.seq), row0 = __builtin_amdgcn_readfirstlane(pl.row0);
  const PaSeq q = pa_seq(a, pl.r, pl.len);
  const int nrow = min(BR, q.rows - row0);
  int lo, hi;
  pa_span(q, row0, nrow, a.window, lo, hi);
  const PaParts pt = pa_parts(lo, hi, a.sp_many);
  if (part >= pt.n) return;
  const int kb0 = pt.begin + part * pt.per;
  const int a0 = max(kb0, lo), b0 = min(kb0 + pt.per, hi);
  const int nt = b0 > a0 ? (b0 - kb0 + BK - 1) / BK : 0;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, g4 = lane >> 4;
  const int32_t* table = a.c.table + s * a.c.trow;

  // this wave's rows, past the last one copies of it; their entries el .. eh
  const int wr0 = row0 + wv * 16 * QB, last = q.rows - 1;
  const bool some = wr0 <= last;
  const int el = q.e0 + q.by.div(min(wr0, last)), eh = q.e0 + q.by.div(min(wr0 + 16 * QB - 1, last));
  bf16x8_t qf[QB][NKS];
  int e[QB];
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    const int row = min(wr0 + 16 * b + r16, last), tok = q.by.div(row);
    e[b] = q.e0 + tok;
    const bf16_t* qr = a.q + (q.first + tok) * a.qt + (kvh * q.G + row - tok * q.G) * a.qh + g4 * 8;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) qf[b][ks] = pa_signed(qr + ks * 32, a.keep, a.flip);
  }
  floatx4_t o[QB][NDB];
  float m[QB], msl[QB], lsum[QB];
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    m[b] = -INFINITY;
    msl[b] = lsum[b] = 0.f;
#pragma unroll
    for (int i = 0; i < NDB; ++i) o[b][i] = (floatx4_t){0.f, 0.f, 0.f, 0.f};
  }

  // A wave's loads of a tile lie in one group of 16 entries, group gw.  Lane i
  // holds the offset in bytes within a head of that group of tile i of a batch of
  // 64, from one table entry each; the next batch's page ids come ahead.  Keys and
  // values walk apart by a tile.
  static_assert(LPW * RPL <= 16, "one group a wave");
  const int gw = wv * LPW * RPL / 16;
  auto slot0 = [&](int b) {
    return min(max(kb0 + BK * (64 * b + lane) + 16 * gw, a0 & ~15), (b0 - 1) & ~15);
  };
  PaWalk<LPW> wk, wx;
  wk.head = (const unsigned char*)(a.c.k + kvh * a.c.kh);
  wk.page = a.c.kp;
  wk.slot = a.c.ks;
  wx.head = (const unsigned char*)(a.c.v + kvh * a.c.vh);
  wx.page = a.c.vp;
  wx.slot = a.c.vs;
  int lrow[LPW], kcol[LPW], vcol[LPW];   // load u: this lane's row of its group, its columns in bytes
#pragma unroll
  for (int u = 0; u < LPW; ++u) {
    const int r = (wv * LPW + u) * RPL + lane / (RB / 16), ch = lane % (RB / 16);
    lrow[u] = r % 16;
    kcol[u] = (ch ^ pa_kswz<DH>(r)) * 16;
    vcol[u] = (ch ^ pa_swz<DH>(r)) * 16;
    wk.off[u] = (unsigned)(lrow[u] * (int)a.c.ks * 2 + kcol[u]);
    wx.off[u] = (unsigned)(lrow[u] * (int)a.c.vs * 2 + vcol[u]);
  }
  auto turn = [&](PaWalk<LPW>& w, int b) {   // to batch b, whose ids have arrived
    const long long off =
        (pg_read(w.next, a.c.pages) * w.page + pg_slot(slot0(b), a.c.sh, w.slot)) * 2;
    w.lo = (int)off;
    w.hi = (int)(off >> 32);
    if ((b + 1) * 64 < nt) w.next = table[slot0(b + 1) >> a.c.sh];
  };
  // tile t to stage st; edge: rows outside [a0, b0) take the nearest inside
  auto issue = [&](PaWalk<LPW>& w, const int* col, int t, unsigned char* st, bool edge)
                   __attribute__((always_inline)) {
    if (t % 64 == 0) turn(w, t / 64);
    const unsigned lo = __builtin_amdgcn_readlane(w.lo, t % 64);
    const unsigned char* base =
        w.head + (((long long)__builtin_amdgcn_readlane(w.hi, t % 64) << 32) | lo);
#pragma unroll
    for (int u = 0; u < LPW; ++u) {
      unsigned off = w.off[u];
      if (edge) {
        const int k0 = min(max(kb0 + BK * t + 16 * gw, a0 & ~15), (b0 - 1) & ~15);
        off = (unsigned)(min(max(lrow[u], a0 - k0), b0 - 1 - k0) * (int)w.slot * 2 + col[u]);
      }
      const unsigned char* src = base + off;
      __builtin_amdgcn_global_load_lds(src, (pa_lds_void*)(st + (wv * LPW + u) * 1024), 16, 0, 0);
    }
  };
  // fragment addresses of the first key and value stage
  const int trow = 4 * g4 + (r16 >> 2), tcol = 4 * (r16 & 3);
  pa_lds_cchar* kadr[NKS];
  pa_lds_cchar* vadr[NDB];
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks)
    kadr[ks] = (pa_lds_cchar*)smem + r16 * RB + (((ks * 4 + g4) ^ pa_kswz<DH>(r16)) << 4);
#pragma unroll
  for (int db = 0; db < NDB; ++db)
    vadr[db] = (pa_lds_cchar*)smem + NS * TB + trow * RB + (tcol & 7) * 2 +
               (((2 * db + (tcol >> 3)) ^ pa_swz<DH>(trow)) << 4);
  auto live = [&](int t) {   // whether this wave's rows see any of tile t
    const int kb = kb0 + BK * t;
    return some && t < nt && kb <= eh && el - (kb + BK - 1) < a.window;
  };

  // A step's scores were formed in the step before: its products with the next
  // keys run beside its exponentials, both in groups of one key fragment, and the
  // values' fragments arrive behind them for the products with P.  Steps f0 .. f1
  // - 1 are free of every edge: all their entries are seen by all rows, and what
  // they load ahead is there.
  constexpr int KG = NKS * NBLK, VG = NI * NDB, PG = NBLK * 4 / KG;   // PG weights a group and row block
  static_assert(KG == 8 && KG == VG && PG * KG == NBLK * 4, "one value fragment beside each key fragment");
  int f0 = max(a0 - kb0, eh < a.window ? 0 : eh - a.window + 1 - kb0);
  f0 = f0 > 0 ? (f0 + BK - 1) / BK : 0;
  const int f1 = some ? min((min(b0, el + 1) - kb0) / BK, (b0 - kb0) / BK - 1 - PM_AHEAD) : 0;
  floatx4_t sc[2][QB][NBLK];
  auto step = [&](int t, auto stage, auto free) __attribute__((always_inline)) {
    constexpr bool FREE = decltype(free)::value;
    constexpr int ST = decltype(stage)::value, P = ST & 1;   // t % NS, t % 2
    constexpr int KO = (ST + 1) % NS * TB, VO = ST * TB;
    // this wave's part of keys t + 1 and values t is in LDS: all but the last
    // PM_AHEAD - 1 steps' loads, or near the end all
    if (FREE || t + PM_AHEAD < nt) pa_wait_vm<(PM_AHEAD - 1) * 2 * LPW>();
    else pa_wait_vm<0>();
    __syncthreads();   // every wave's; keys t and values t - 1 are used up
    if (FREE || t + 1 + PM_AHEAD < nt) issue(wk, kcol, t + 1 + PM_AHEAD, smem + ST * TB, !FREE);
    if (FREE || t + PM_AHEAD < nt)
      issue(wx, vcol, t + PM_AHEAD, smem + (NS + (ST + NS - 1) % NS) * TB, !FREE);
    floatx4_t(&s0)[QB][NBLK] = sc[P];
    floatx4_t(&s1)[QB][NBLK] = sc[1 - P];
    if constexpr (!FREE) {
      const bool now = live(t);
      if (!now && !live(t + 1)) return;
      const int kb = kb0 + BK * t;
#pragma unroll
      for (int b = 0; b < QB; ++b) {   // what is masked scores -inf
        const int jl = max(a0, e[b] < a.window ? 0 : e[b] - a.window + 1) - kb - 4 * g4;
        const int jh = now ? min(b0 - 1, e[b]) - kb - 4 * g4 : -64;
#pragma unroll
        for (int i = 0; i < NBLK; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            s0[b][i][r] = 16 * i + r >= jl && 16 * i + r <= jh ? s0[b][i][r] : -INFINITY;
      }
    }
    float lm[QB];
    bool over = false;
#pragma unroll
    for (int b = 0; b < QB; ++b) {
      lm[b] = s0[b][0][0];
#pragma unroll
      for (int i = 0; i < NBLK; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) lm[b] = fmaxf(lm[b], s0[b][i][r]);
      over = over || lm[b] > m[b] + a.thr;
    }
    if (__any(over))
#pragma unroll
      for (int b = 0; b < QB; ++b) pa_raise<NDB>(lm[b], a.sl2, m[b], msl[b], lsum[b], o[b]);
    bf16x8_t kf[KG];
    pa_v4i16 v0[VG], v1[VG];
#pragma unroll
    for (int b = 0; b < QB; ++b)
#pragma unroll
      for (int i = 0; i < NBLK; ++i) s1[b][i] = (floatx4_t){0.f, 0.f, 0.f, 0.f};
    // four key fragments ahead; behind group x's the values' pair x, so that group x
    // waits for all but what was read after its own fragment
    pa_static_for<0, 4>([&](auto xc) __attribute__((always_inline)) {
      constexpr int x = decltype(xc)::value, ks = x / NBLK, i = x % NBLK;
      kf[x] = pa_rd_b128<KO + i * 16 * RB>(kadr[ks]);
    });
    uint32_t pw[QB][NBLK][2];
    pa_static_for<0, KG>([&](auto xc) __attribute__((always_inline)) {
      constexpr int x = decltype(xc)::value, ks = x / NBLK, i = x % NBLK, vi = x / NDB, db = x % NDB;
      pa_wait_lgkm<(x < 4 ? 3 + 2 * x : 15 - x)>(kf[x]);
#pragma unroll
      for (int b = 0; b < QB; ++b)
        s1[b][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[x], qf[b][ks], s1[b][i], 0, 0, 0);
      if constexpr (x + 4 < KG) {
        constexpr int y = x + 4;
        kf[y] = pa_rd_b128<KO + y % NBLK * 16 * RB>(kadr[y / NBLK]);
      }
      v0[x] = pa_rd_tr<VO + 32 * vi * RB>(vadr[db]);
      v1[x] = pa_rd_tr<VO + (32 * vi + 16) * RB>(vadr[db]);
#pragma unroll
      for (int b = 0; b < QB; ++b) {
#pragma unroll
        for (int g = 0; g < PG; ++g) {
          const int k = x * PG + g;
          const float v = __builtin_amdgcn_exp2f(s0[b][k / 4][k % 4] * a.sl2 - msl[b]);
          s0[b][k / 4][k % 4] = v;
          lsum[b] += v;
          if (k % 2 == 1) pw[b][k / 4][(k % 4) / 2] = pack2(s0[b][k / 4][k % 4 - 1], v);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    pa_static_for<0, VG>([&](auto xc) __attribute__((always_inline)) {
      constexpr int x = decltype(xc)::value, i = x / NDB, db = x % NDB;
      pa_wait_lgkm2<2 * (VG - 1 - x)>(v0[x], v1[x]);
      const bf16x8_t vf = pa_join(v0[x], v1[x]);
#pragma unroll
      for (int b = 0; b < QB; ++b) {
        const uint32_t w4[4] = {pw[b][2 * i][0], pw[b][2 * i][1], pw[b][2 * i + 1][0], pw[b][2 * i + 1][1]};
        o[b][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, *(const bf16x8_t*)w4, o[b][db], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  if (nt) {
    wk.next = wx.next = table[slot0(0) >> a.c.sh];
    issue(wk, kcol, 0, smem, true);
#pragma unroll
    for (int d = 0; d < PM_AHEAD; ++d) {
      if (d + 1 < nt) issue(wk, kcol, d + 1, smem + (d + 1) * TB, true);
      if (d < nt) issue(wx, vcol, d, smem + (NS + d) * TB, true);
    }
    if (PM_AHEAD < nt) pa_wait_vm<PM_AHEAD * 2 * LPW>();
    else pa_wait_vm<0>();
    __syncthreads();
    pa_static_for<0, KG>([&](auto xc) __attribute__((always_inline)) {
      constexpr int x = decltype(xc)::value, ks = x / NBLK, i = x % NBLK;
      bf16x8_t kf = pa_rd_b128<i * 16 * RB>(kadr[ks]);
      pa_wait_lgkm<0>(kf);
#pragma unroll
      for (int b = 0; b < QB; ++b)
        sc[0][b][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            kf, qf[b][ks], ks ? sc[0][b][i] : (floatx4_t){0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
    });
  }
  const auto steps = [&](int t, auto free) __attribute__((always_inline)) {
    pa_static_for<0, NS>([&](auto st) __attribute__((always_inline)) {
      constexpr int i = decltype(st)::value;
      if (decltype(free)::value || t + i < nt) step(t + i, st, free);
    });
  };
  int t = 0;
  for (; t < nt && (t < f0 || t + NS > f1); t += NS) steps(t, std::false_type{});
  for (; t + NS <= f1; t += NS) steps(t, std::true_type{});
  for (; t < nt; t += NS) steps(t, std::false_type{});
  pa_wait_vm<0>();
  if (!some) return;
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    const int row = wr0 + 16 * b + r16;
    const PaRow w = pa_place<false>(a, q, s, kvh, min(row, last), part);
    float l = lsum[b];
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    const float M = m[b] == -INFINITY ? -INFINITY : m[b] * a.sl2;
    bool fine = true;
#pragma unroll
    for (int db = 0; db < NDB; ++db) fine = fine && pa_finite(o[b][db]);
    unsigned long long bad = __ballot(!fine && row <= last);
    bad = (bad | bad >> 16 | bad >> 32 | bad >> 48) & 0xffff;
    if (row <= last && !((bad >> r16) & 1))
#pragma unroll
      for (int db = 0; db < NDB; ++db)
        pa_store4<DH, false>(a, w, pt.n, db * 16 + g4 * 4,
                             make_float4(o[b][db][0], o[b][db][1], o[b][db][2], o[b][db][3]), M, l);
    while (bad) {
      const int r = __builtin_ctzll(bad);
      bad &= bad - 1;
      pa_again<DH, false>(a, q, s, table, kvh, wr0 + 16 * b + r, a0, b0, part, pt.n);
    }
  }
}

// Tiles of many rows, then (where a call has both) sequences of few, each by a
// work-group of its own: the short ones fill the CUs that the long ones leave.
template <int DH, int QB>
__global__ __launch_bounds__(256, 2) void k_paged_many(PaArgs a, int tiles, int full, int blocks) {
  constexpr int BK = DH == 64 ? 64 : 32;
  extern __shared__ __attribute__((aligned(16))) unsigned char pa_smem[];
  const int L = blockIdx.x;
  if (L < blocks) {
    // Tiles of one (cache head, part) run together on one XCD and share its L2:
    // work-group L runs on XCD L % 8.  That many tiles as the rows fill go first; of
    // the others, one for each sequence, many are none, and among the first they
    // would leave CUs to them alone (64 rows on 16384 entries, 12 heads: 47 us).
    const int pairs = a.c.heads * a.sp_many.most, first = full * pairs;
    int tile, w = L;
    if (L < first) {
      if (first % 8 == 0) w = (L % 8) * (first / 8) + L / 8;
      tile = w % full;
      w /= full;
    } else {
      tile = full + (L - first) / pairs;
      w = (L - first) % pairs;
    }
    pa_many<DH, BK, QB>(a, tile, w % a.c.heads, w / a.c.heads, pa_smem);
  } else {
    const int w = L - blocks, i = w / a.c.heads;
    pa_few<DH, 4>(a, i % a.c.seqs, 0, w % a.c.heads, i / a.c.seqs, pa_smem);
  }
}

// The parts of each row joined, in part order.  A wave takes a token, its heads HPW
// at a time, W lanes of four dims each: GP such groups, whose parts' sums are on
// their way together, and then the next GP * step.  Of all tokens or (each) of the
// first ones of every sequence with few rows.
template <int DH, int GP>
__global__ __launch_bounds__(256) void k_paged_join(PaArgs a, int each, int groups, int waves) {
  constexpr int W = DH / 4, HPW = 64 / W, NP = 64 / W;   // NP: parts a lane weighs, 64 in all
  const int lane = threadIdx.x & 63, l = lane % W;
  const int wv = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int n = wv / waves;   // the token, or its place in its sequence
  int s = blockIdx.y;
  if (!each) {
    if (n >= a.c.rows) return;
    s = __builtin_amdgcn_readfirstlane(pg_sequence(a.c.starts, a.c.seqs, n));
    if (s < 0) return;
  }
  const PaSeq q = pa_seq(a, s);
  if (each) n += q.first;
  if (n - q.first >= q.n) return;
  const bool few = q.rows <= a.few;
  if (each && !few) return;
  const int br = few ? 16 : a.br;
  const PaSplit sp = few ? a.sp_few : a.sp_many;
  for (int g0 = wv % waves * GP; g0 < groups; g0 += waves * GP) {
    const float* po[GP];
    int np[GP], most = 0;
    float m[GP][NP], sum[GP], M[GP];
#pragma unroll
    for (int g = 0; g < GP; ++g) {
      const int h = (g0 + g) * HPW + lane / W, hc = min(h, a.heads - 1);
      const int kvh = q.by.div(hc), row = (n - q.first) * q.G + hc - kvh * q.G, row0 = row & ~(br - 1);
      int lo, hi;
      pa_span(q, row0, min(br, q.rows - row0), a.window, lo, hi);
      // heads of one token may lie in two tiles, of other numbers of parts
      np[g] = h < a.heads ? pa_parts(lo, hi, sp).n : 1;
      if (np[g] == 1) np[g] = 0;
      const long long at = few ? pa_place<true>(a, q, s, kvh, row, 0).at : pa_place<false>(a, q, s, kvh, row, 0).at;
      po[g] = (few ? a.po_few : a.po_many) + at * DH + l * 4;
      const float2* pml = (few ? a.ml_few : a.ml_many) + at;
      float f[NP];
      M[g] = -INFINITY;
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        const float2 ml = l + W * k < np[g] ? pml[l + W * k] : make_float2(-INFINITY, 0.f);
        m[g][k] = ml.x;
        f[k] = ml.y;
        M[g] = fmaxf(M[g], m[g][k]);
      }
      M[g] = group_max<W>(M[g]);
      const float base = M[g] == -INFINITY ? 0.f : M[g];
      sum[g] = 0.f;
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        m[g][k] = __builtin_amdgcn_exp2f(m[g][k] - base);
        sum[g] += f[k] * m[g][k];
      }
      sum[g] = group_sum<W>(sum[g]);
      most = max(most, np[g]);
    }
    floatx4_t o[GP];
#pragma unroll
    for (int g = 0; g < GP; ++g) o[g] = (floatx4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NP; ++k)
      for (int i0 = 0; i0 < W; i0 += 4) {
        if (!__any(W * k + i0 < most)) break;
        floatx4_t v[GP][4];
#pragma unroll
        for (int g = 0; g < GP; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i)   // of a row that came in one part: its slot, not added
            v[g][i] = *(const floatx4_t*)(po[g] + max(min(W * k + i0 + i, np[g] - 1), 0) * DH);
#pragma unroll
        for (int g = 0; g < GP; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float w = __shfl(m[g][k], i0 + i, W);
            if (W * k + i0 + i < np[g]) o[g] += v[g][i] * w;
          }
      }
#pragma unroll
    for (int g = 0; g < GP; ++g) {
      if (!np[g]) continue;
      const long long r = (long long)n * a.heads + (g0 + g) * HPW + lane / W;
      const float inv = sum[g] == 0.f ? 0.f : 1.f / sum[g];
      *(uint2*)(a.out + r * DH + l * 4) =
          make_uint2(pack2(o[g][0] * inv, o[g][1] * inv), pack2(o[g][2] * inv, o[g][3] * inv));
      if (a.lse && l == 0)
        a.lse[r] = sum[g] == 0.f ? -INFINITY : (M[g] + __builtin_amdgcn_logf(sum[g])) * PA_LN2;
    }
  }
}

// What a call launches, from what the host knows: rows and sequences, not how
// the rows are shared out among them.
struct PaPlan {
  int few;             // rows of a sequence up to which pa_few takes it
  bool many;           // pa_many takes the others
  int qb, tiles, full; // its row blocks, its tiles at most and where one sequence has all rows
  PaSplit sp_few, sp_many;
  bool wide;           // pa_few by eight waves
  bool packed;         // slots of pa_few: 16 a (sequence, cache head), else one a row
};
// Slots of the parts' sums of few rows.
static size_t pa_slots_few(const PagedArgs& c, int heads, bool packed) {
  return packed ? (size_t)c.seqs * c.heads * 16 : (size_t)c.rows * heads;
}
// Bytes that the parts of few rows, and those of many, may take: many times what fills
// the card's places (512 of 128 rows of 128 dims: 34 MB), and less than the table's
// width asks for where few of its sequences are long (1024 of up to 131072 entries, 8
// heads, 1535 rows: 2.2 GB by 16 slots a sequence and a part for every 4096).
constexpr size_t PA_WS_MAX = (size_t)1 << 28;
static PaPlan pa_plan(const PagedArgs& c, int heads, int Dh, int window) {
  static const int cus = device_cus();
  PaPlan p{};
  const int G = heads / c.heads;
  const long long rows = (long long)c.rows * G, pairs = (long long)c.seqs * c.heads;
  // entries that a tile of br rows sees at most
  const auto span = [&](long long br) {
    const long long all = (long long)c.cols << c.sh;
    return window > 0 && window + br < all ? window + br : all;
  };
  const auto clamp = [](long long v, long long hi) { return (int)(v < 1 ? 1 : v > hi ? hi : v); };
  p.many = rows > 16 && c.rows > c.seqs;
  p.few = !p.many ? 0x7fffffff : c.seqs == 1 ? 0 : 16;
  // Few rows: one part, and one launch, up to 1024 entries (us with parts and
  // without, 6 heads of 128: 1 sequence of 400 entries 18.8 / 14.3, of 1024 18.5 /
  // 15.4, of 2048 17.9 / 24.9; 64 of 400 23.8 / 18.5, of 1024 43.8 / 42.1) or with a
  // (sequence, head) for each CU (32 x 4096 of 8 heads of 64: 42.3 in one part, 46.6
  // in two), else what two work-groups a CU take at once (16 x 8192: 77.7 in 5 parts,
  // 480 work-groups, 87.3 in 6); by eight waves where there are CUs to spare (1024
  // entries, 1 sequence 15.4 against 16.7 by four, 64 of them 46.2 against 42.1).
  const bool one = p.few == 0 || span(16) <= 1024;
  p.sp_few.split = one || pairs >= cus ? 1 : clamp(2LL * cus / pairs, clamp((span(16) + 127) / 128, 64));
  p.sp_few.most = one ? 1 : clamp((span(16) + 4095) / 4096, 64);
  if (p.sp_few.most < p.sp_few.split) p.sp_few.most = p.sp_few.split;
  p.packed = p.many && pairs * 16 < (long long)c.rows * heads;
  const size_t part = (size_t)(Dh + 2) * sizeof(float);   // of a slot
  p.sp_few.most = clamp((long long)(PA_WS_MAX / (pa_slots_few(c, heads, p.packed) * part)), p.sp_few.most);
  if (p.sp_few.split > p.sp_few.most) p.sp_few.split = p.sp_few.most;
  p.wide = !p.many && p.sp_few.most == 1 && pairs <= cus;
  // Many rows: the tile and the number of parts that the figures below put
  // first.  A step of 32 entries takes a work-group of 64 rows 0.475 us, two on one
  // CU 0.68, of 128 rows 0.65 and 0.88 (of 64 entries at head dim 64 0.5, 0.86, 0.75
  // and 1.4); parts cost another launch and their sums' way to memory and back.  us
  // measured at 12 heads of 128, 2048 rows on 16384 entries: 64 rows 351 / 274 / 270
  // in 1 / 2 / 4 parts, 128 rows 350 / 240 / 230; 6 heads, 512 rows on 8192: 64 rows 122 / 71 / 43 / 35 / 39 in 1
  // .. 16 parts, 128 rows 160 / 91 / 54 / 38 / 36.
  p.sp_many = {1, 1};
  if (p.many) {
    const bool h = Dh == 64;
    const float alone[2] = {h ? 0.5f : 0.475f, h ? 0.75f : 0.65f};
    const float both[2] = {h ? 0.86f : 0.68f, h ? 1.4f : 0.88f};
    float best = 0.f;
    for (int qb = 1; qb <= 2; ++qb) {
      const int br = 64 * qb, step = Dh == 64 ? 64 : 32;
      const long long keys = span(br);
      const float tiles = (float)((rows + br - 1) / br) + 0.5f * (float)((c.seqs < c.rows ? c.seqs : c.rows) - 1);
      for (int ns = 1; ns <= 64 && (ns == 1 || (keys / ns >= 256 && (size_t)c.rows * heads * ns * part <= PA_WS_MAX));
           ns *= 2) {
        const int each = (int)ceilf(tiles * (float)(c.heads * ns) / (float)cus);   // of a CU's work-groups
        const float steps = (float)((keys + (long long)step * ns - 1) / ((long long)step * ns));
        float us = 4.f * (float)((each + 1) / 2) +   // to find the tile and its first entries
                   steps * ((float)(each / 2) * both[qb - 1] + (float)(each % 2) * alone[qb - 1]);
        if (ns > 1) us += 5.f + (float)c.rows * (float)heads * (float)ns * (float)(Dh + 4) * 8.f / 4e6f;
        if (best == 0.f || us < best) {
          best = us;
          p.qb = qb;
          p.sp_many = {ns, ns};
        }
      }
    }
    p.full = (int)(rows / (64 * p.qb));
    if (p.full < 1) p.full = 1;
    p.tiles = (int)(rows / (64 * p.qb) + (c.seqs < c.rows ? c.seqs : c.rows));
  }
  return p;
}
// Slots times parts: none where all rows come in one part.
struct PaSlots {
  size_t few, many;
};
static PaSlots pa_slots(const PagedArgs& c, int heads, const PaPlan& p) {
  PaSlots n = {0, 0};
  if (p.few && p.sp_few.most > 1)
    n.few = pa_slots_few(c, heads, p.packed) * p.sp_few.most;
  if (p.many && p.sp_many.most > 1) n.many = (size_t)c.rows * heads * p.sp_many.most;
  return n;
}

size_t paged_attention_ws_bytes(const PagedArgs& c, int heads, int Dh, int window) {
  if (c.rows == 0 || c.seqs == 0) return 0;
  const PaSlots n = pa_slots(c, heads, pa_plan(c, heads, Dh, window));
  return (n.few + n.many) * (Dh + 2) * sizeof(float);
}

template <int DH, int NW>
static hipError_t pa_launch_few(const PaArgs& a, hipStream_t st) {
  constexpr size_t lds = pa_few_lds<DH, NW>();
  if (lds > 64 * 1024) {
    static PerDevice limit;
    const hipError_t e = lds_limit(limit, (const void*)k_paged_few<DH, NW>, lds);
    if (e != hipSuccess) return e;
  }
  // the first sixteen rows of each sequence, and what may be behind them
  const long long blocks = a.c.seqs + ((long long)a.c.rows * a.G - 1) / 16;
  if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
  const unsigned z = (unsigned)((blocks + 65534) / 65535);
  const dim3 grid((unsigned)(a.c.heads * a.sp_few.most), (unsigned)((blocks + z - 1) / z), z);
  hipLaunchKernelGGL((k_paged_few<DH, NW>), grid, dim3(64 * NW), lds, st, a, (int)blocks);
  return hipGetLastError();
}

template <int DH>
static hipError_t pa_launch(const PaArgs& a, const PaPlan& p, hipStream_t st) {
  hipError_t e;
  if (p.many) {
    constexpr size_t m = pa_many_lds<DH, DH == 64 ? 64 : 32>(), f = pa_few_lds<DH, 4>();
    const long long blocks = (long long)p.tiles * a.c.heads * a.sp_many.most;
    const long long more = p.few ? (long long)a.c.seqs * a.c.heads * a.sp_few.most : 0;
    if (blocks + more >= 1LL << 24) return hipErrorInvalidConfiguration;   // 2^32 threads: a launch would be cut short
    const dim3 grid((unsigned)(blocks + more));
    const size_t lds = p.few && f > m ? f : m;
    if (p.qb == 2)
      hipLaunchKernelGGL((k_paged_many<DH, 2>), grid, dim3(256), lds, st, a, p.tiles, p.full, (int)blocks);
    else
      hipLaunchKernelGGL((k_paged_many<DH, 1>), grid, dim3(256), lds, st, a, p.tiles, p.full, (int)blocks);
    e = hipGetLastError();
  } else {
    e = p.wide ? pa_launch_few<DH, 8>(a, st) : pa_launch_few<DH, 4>(a, st);
  }
  if (e != hipSuccess || (a.sp_few.most == 1 && a.sp_many.most == 1)) return e;
  // only rows of sequences with few come in parts where the tiles do not
  const int G = a.G, groups = (a.heads * (DH / 4) + 63) / 64;
  const int each = p.many && a.sp_many.most == 1 ? (16 + G - 1) / G : 0;
  // a wave for each group of heads of few tokens, for all those of many (2048 tokens
  // of 12 heads in 4 parts: 18.3 and 15.4 us)
  const long long tokens = each ? (long long)each * a.c.seqs : a.c.rows;
  const bool wide = tokens * groups <= 4096;
  const int waves = wide ? groups : 1;
  const dim3 grid = each ? dim3((unsigned)((each * waves + 3) / 4), (unsigned)a.c.seqs)
                         : dim3((unsigned)(((long long)a.c.rows * waves + 3) / 4));
  if (wide) hipLaunchKernelGGL((k_paged_join<DH, 1>), grid, dim3(256), 0, st, a, each, groups, waves);
  else hipLaunchKernelGGL((k_paged_join<DH, 3>), grid, dim3(256), 0, st, a, each, groups, waves);
  return hipGetLastError();
}

hipError_t paged_attention(const PagedArgs& c, const bf16_t* q, long long qt, long long qh,
                           int heads, int Dh, float scale, int window, bf16_t* out, float* lse,
                           void* ws, hipStream_t st) {
  if (c.rows == 0 || c.seqs == 0) return hipSuccess;
  const PaPlan p = pa_plan(c, heads, Dh, window);
  PaArgs a{};
  a.c = c;
  a.q = q;
  a.qt = qt;
  a.qh = qh;
  a.heads = heads;
  a.G = heads / c.heads;
  a.by = FastDiv::of(a.G);
  a.window = pa_window(window);
  a.ssl2 = scale * PA_LOG2E;
  a.sl2 = scale == 0.f ? 1.f : fabsf(a.ssl2);
  a.thr = fminf(8.f / a.sl2, 3e38f);
  a.keep = scale == 0.f ? 0u : ~0u;
  a.flip = scale < 0.f ? 0x80008000u : 0u;
  a.out = out;
  a.lse = lse;
  a.sp_few = p.sp_few;
  a.sp_many = p.sp_many;
  a.few = p.few;
  a.packed = p.packed;
  a.br = 64 * p.qb;
  const PaSlots n = pa_slots(c, heads, p);
  a.po_few = (float*)ws;
  a.po_many = a.po_few + n.few * Dh;
  a.ml_few = (float2*)(a.po_many + n.many * Dh);
  a.ml_many = a.ml_few + n.few;
  if (Dh == 64) return pa_launch<64>(a, p, st);
  if (Dh == 128) return pa_launch<128>(a, p, st);
  return hipErrorInvalidValue;
}

// ---- weight of the entries -------------------------------------------------------
//
// A wave takes 16 NB entries of a sequence, `share` of a work-group's NW waves the
// same ones, and of the rows (token, head) that see any of them, in the order of
// the cache heads, an equal share each.  S = K Q^T, entries x rows, 16 x 16 a
// product: a lane adds the weights of its row's column for its four entries of
// each block, and only at the end are the 16 columns and the waves added, in a
// fixed order: the same call gives the same bits.  (How many waves share entries goes
// by the call's sequences, rows and table, so another call may add in another order.)
//
// FEW: calls of sixteen rows a head or so (decoding), where the keys change from
// head to head and the next head's are loaded ahead.  Otherwise the keys stay, and
// the next sixteen rows are.  FEW is bound by memory (one token on 16 x 4096 entries of
// 6 heads of 128: 17.4 us, 4.4 TB/s), the other by its vector instructions on the
// CUs whose sequences have the most rows (864 tokens of 8 heads of 64, 462 of them on
// one of four sequences of up to 4096 entries: 16.6 us; all CUs' vector units are busy
// 55% of 13 us).  No faster: rows three tiles ahead (16.4, but 30 to 34 us for 29 at
// head dim 128), 16 or 64 entries a wave (16.9 and 21.6), four or sixteen waves (22.7
// and 18.7), page ids ahead of the length (16.6).
template <int DH, bool FEW>
struct PwShape {
  static constexpr int NW = FEW ? 4 : 8, NB = 2, E = 16 * NB;
};
template <int DH, bool FEW>
__global__ __launch_bounds__(FEW ? 256 : 512, FEW ? 3 : 4) void k_paged_weight(
    PagedArgs c, const bf16_t* __restrict__ q, long long qt, long long qh, int heads, int G, FastDiv group,
    const float* __restrict__ lse, float sl2, int window, const float* w, long long wrow, float* out,
    long long orow, int cap, int share2, int tg2) {   // log2 of share, and of whole tokens a tile (or -1)
  constexpr int NW = PwShape<DH, FEW>::NW, NB = PwShape<DH, FEW>::NB, E = PwShape<DH, FEW>::E;
  constexpr int NKS = DH / 32;
  __shared__ float part[NW][E];
  extern __shared__ __attribute__((aligned(16))) unsigned char pw_smem[];   // NW * 2 * 16 rows
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g4 = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int share = 1 << share2, blocks = NW >> share2, s = blockIdx.y;
  const int j0 = (blockIdx.x * blocks + (wv >> share2)) * E;
  // the entry whose sum this thread writes
  const int j = blockIdx.x * blocks * E + tid;
  const bool mine = tid < blocks * E && j < cap;
  const float was = mine ? w[s * wrow + j] : 0.f;
  const int len = pg_len(c.lens[s], c.cols, c.sh);
  const PgRange r = pg_range(c.starts[s], c.starts[s + 1], c.rows);
  const int e0 = len - r.n, jl = min(j0 + E - 1, len - 1);
  // tokens t0 .. t1 - 1 see one of the entries j0 .. jl
  const int t0 = max(0, j0 - e0), t1 = jl - e0 < r.n - window ? jl - e0 + window : r.n;
  float acc[NB][4];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[b][i] = 0.f;
  if (j0 < len && t1 > t0) {
    const int hi = (t1 - t0) * G;   // rows, from token t0 on
    const int tiles = (hi + 15) / 16, all = tiles * c.heads, per = (all + share - 1) >> share2;
    const bf16_t* kr[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int k0 = min(j0 + 16 * b, jl & ~15);
      const int id = pg_read(c.table[s * c.trow + (k0 >> c.sh)], c.pages);
      kr[b] = c.k + id * c.kp + pg_slot(k0, c.sh, c.ks) + min(r16, jl - k0) * c.ks + g4 * 8;
    }
    const bf16_t* q0 = q + (r.first + t0) * qt;
    const float* l0 = lse + (long long)(r.first + t0) * heads;
    struct Rows {
      bf16x8_t q[NKS];
      float l2;
      int e;
    };
    auto keys = [&](bf16x8_t (&kf)[NB][NKS], int kvh) __attribute__((always_inline)) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) kf[b][ks] = *(const bf16x8_t*)(kr[b] + kvh * c.kh + ks * 32);
    };
    auto rows = [&](Rows& x, int kvh, int tile) __attribute__((always_inline)) {
      const unsigned char* qb = (const unsigned char*)(q0 + (long long)kvh * G * qh);
      const unsigned char* lb = (const unsigned char*)(l0 + kvh * G);
      const int at = tile * 16 + r16, row = min(at, hi - 1), t = group.div(row), h = row - t * G;
      const unsigned qx = (unsigned)(t * (int)qt + h * (int)qh + g4 * 8) * 2, lx = (unsigned)(t * heads + h) * 4;
      x.e = at < hi ? e0 + t0 + t : -1;   // a row past the last sees nothing
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) x.q[ks] = *(const bf16x8_t*)(qb + qx + ks * 64);
      x.l2 = *(const float*)(lb + lx);
    };
    auto add = [&](const bf16x8_t (&kf)[NB][NKS], const Rows& x, bool full) __attribute__((always_inline)) {
      floatx4_t sc[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) sc[b] = (floatx4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
        for (int b = 0; b < NB; ++b)
          sc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[b][ks], x.q[ks], sc[b], 0, 0, 0);
      const float base = x.l2 * PA_LOG2E;
      const int yl = x.e < window ? 0 : x.e - window + 1;   // entries yl .. x.e are seen
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int y = j0 + 16 * b + 4 * g4 + k;
          const float p = __builtin_amdgcn_exp2f(sc[b][k] * sl2 - base);
          acc[b][k] += full || (y <= x.e && y >= yl) ? p : 0.f;
        }
    };
    int u = (wv & (share - 1)) * per;
    const int end = min(u + per, all);
    bool done = false;
    if constexpr (FEW) {
      if (tiles == 1) {
        done = true;
        bf16x8_t kf[2][NB][NKS];
        Rows x[2];
        if (u < end) {
          rows(x[0], u, 0);
          keys(kf[0], u);
        }
        for (; u < end; u += 2)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (u + i >= end) break;
            if (u + i + 1 < end) {
              rows(x[1 - i], u + i + 1, 0);
              keys(kf[1 - i], u + i + 1);
            }
            add(kf[i], x[i], false);
          }
      }
    }
    // Sixteens of rows pass through the wave's own two LDS stages, loaded 1 KB at a
    // time: a fragment's lanes side by side belong to different rows, and read from
    // memory each is an access of its own (64 for 1 KB instead of 16).  Tiles f0 ..
    // f1 - 1 are of whole tokens that all see all the entries.
    constexpr int RB = DH * 2, LPT = 16 * RB / 1024, RPL = 1024 / RB;
    unsigned char* ring = pw_smem + wv * 2 * 16 * RB;
    int f0 = 0, f1 = 0;
    if (tg2 >= 0) {
      f0 = max(0, (j0 + E - 1 - e0 - t0 + (1 << tg2) - 1) >> tg2);
      f1 = min(hi / 16, window == 0x7fffffff ? 0x7fffffff : (window + j0 - e0 - t0) >> tg2);
    }
    unsigned qoff[LPT];
    int qrow[LPT], qcol[LPT];   // load u: this lane's row of the tile and column in bytes
#pragma unroll
    for (int k = 0; k < LPT; ++k) {
      qrow[k] = k * RPL + lane / (RB / 16);
      qcol[k] = ((lane % (RB / 16)) ^ pa_kswz<DH>(qrow[k])) * 16;
      const int t = group.div(qrow[k]);
      qoff[k] = (unsigned)(t * (int)qt + (qrow[k] - t * G) * (int)qh) * 2 + qcol[k];
    }
    auto issue = [&](int kvh, int tile, int stage, bool in) __attribute__((always_inline)) {
      const int tb = in ? tile << tg2 : group.div(tile * 16);
      const unsigned char* qb = (const unsigned char*)(q0 + (long long)kvh * G * qh + tb * qt);
#pragma unroll
      for (int k = 0; k < LPT; ++k) {
        unsigned off = qoff[k];
        if (!in) {
          const int row = min(tile * 16 + qrow[k], hi - 1), t = group.div(row);
          off = (unsigned)((t - tb) * (int)qt + (row - t * G) * (int)qh) * 2 + qcol[k];
        }
        const unsigned char* src = qb + off;
        __builtin_amdgcn_global_load_lds(src, (pa_lds_void*)(ring + stage * 16 * RB + k * 1024), 16, 0, 0);
      }
    };
    pa_lds_cchar* qadr[NKS];
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks)
      qadr[ks] = (pa_lds_cchar*)ring + r16 * RB + (((ks * 4 + g4) ^ pa_kswz<DH>(r16)) << 4);
    auto fetch = [&](Rows& x, auto stage) __attribute__((always_inline)) {   // a stage that has arrived
      constexpr int ST = decltype(stage)::value;
      pa_static_for<0, NKS>([&](auto kc) __attribute__((always_inline)) {
        x.q[decltype(kc)::value] = pa_rd_b128<ST * 16 * RB>(qadr[decltype(kc)::value]);
      });
      pa_static_for<0, NKS>([&](auto kc) __attribute__((always_inline)) {
        pa_wait_lgkm<NKS - 1 - decltype(kc)::value>(x.q[decltype(kc)::value]);
      });
      asm volatile("" ::: "memory");   // the stage's next load comes behind
    };
    // the log sums of 64 rows from `tile` on, a lane each
    auto sums = [&](int kvh, int tile) __attribute__((always_inline)) {
      const int row = min(tile * 16 + lane, hi - 1), t = group.div(row);
      return l0[(long long)t * heads + kvh * G + row - t * G];
    };
    while (!done && u < end) {   // the wave's rows of one cache head
      const int kvh = u / tiles, first = u - kvh * tiles, n = min(tiles - first, end - u);
      u += n;
      bf16x8_t kf[NB][NKS];
      keys(kf, kvh);
      int i = first;
      const int stop = first + n, g0 = min(max(f0, first), stop), g1 = min(f1, stop);
      Rows x;
      const auto some = [&](int to) __attribute__((always_inline)) {
        for (; i < to; ++i) {
          issue(kvh, i, 0, false);
          const int at = i * 16 + r16, t = group.div(min(at, hi - 1));
          x.e = at < hi ? e0 + t0 + t : -1;   // a row past the last sees nothing
          x.l2 = __shfl(sums(kvh, i), r16, 64);
          pa_wait_vm<0>();
          fetch(x, std::integral_constant<int, 0>{});
          add(kf, x, false);
        }
      };
      some(g0);
      if (i < g1) {
        issue(kvh, i, 0, true);
        float ls = sums(kvh, i), ln = 0.f;
        for (; i < g1; i += 4) {
          if (i + 4 < g1) ln = sums(kvh, i + 4);
          pa_static_for<0, 4>([&](auto kc) __attribute__((always_inline)) {
            constexpr int k = decltype(kc)::value;
            if (i + k >= g1) return;
            if (i + k + 1 < g1) {
              issue(kvh, i + k + 1, (k + 1) & 1, true);
              pa_wait_vm<LPT>();
            } else {
              pa_wait_vm<0>();
            }
            fetch(x, std::integral_constant<int, k & 1>{});
            x.l2 = __shfl(ls, 16 * k + r16, 64);
            add(kf, x, true);
          });
          ls = ln;
        }
        i = g1;
      }
      some(stop);
    }
  }
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v = group_sum<16>(acc[b][i]);
      if (r16 == 0) part[wv][16 * b + 4 * g4 + i] = v;
    }
  __syncthreads();
  if (!mine) return;
  if (j < len) {
    const int k0 = tid / E * share;
    float v = part[k0][tid % E];
    for (int k = 1; k < share; ++k) v += part[k0 + k][tid % E];
    out[s * orow + j] = was + v;
  } else if (out != w) {
    out[s * orow + j] = was;
  }
}

template <int DH, bool FEW>
static hipError_t pw_launch(const PagedArgs& c, const bf16_t* q, long long qt, long long qh,
                            int heads, const float* lse, float sl2, int window, const float* w,
                            long long wrow, float* out, long long orow, int cap, hipStream_t st) {
  using S = PwShape<DH, FEW>;
  static const int cus = device_cus();
  const long long blocks = (long long)c.seqs * ((cap + S::E - 1) / S::E);
  // waves that share their entries, while the call's stay below eight (sixteen)
  // for each CU: 864 tokens of 8 heads of 64 on 4 x 4096 entries 48.0 / 27.0 / 17.8
  // us with 2 / 4 / 8, one token each on 16 x 4096 (6 x 128) 17.9 / 19.8 / 20.8 with
  // 1 / 2 / 4
  int share2 = 0;
  while (1 << share2 < S::NW && blocks << (share2 + 1) <= (FEW ? 8LL : 16LL) * cus) ++share2;
  const int per = (S::NW >> share2) * S::E;
  const int G = heads / c.heads, tg2 = 16 % G ? -1 : __builtin_ctz(16 / G);
  const dim3 grid((unsigned)((cap + per - 1) / per), (unsigned)c.seqs);
  constexpr size_t lds = (size_t)S::NW * 2 * 16 * DH * 2;
  if (lds > 32 * 1024) {
    static PerDevice limit;
    const hipError_t e = lds_limit(limit, (const void*)k_paged_weight<DH, FEW>, lds);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((k_paged_weight<DH, FEW>), grid, dim3(64 * S::NW), lds, st, c, q, qt, qh, heads, G,
                     FastDiv::of(G), lse, sl2, window, w, wrow, out, orow, cap, share2, tg2);
  return hipGetLastError();
}

hipError_t paged_weight(const PagedArgs& c, const bf16_t* q, long long qt, long long qh, int heads,
                        int Dh, const float* lse, float scale, int window, const float* w,
                        long long wrow, float* out, long long orow, hipStream_t st) {
  const int cap = c.cols << c.sh;
  if (c.seqs == 0 || cap == 0) return hipSuccess;
  const int win = pa_window(window);
  const bool few = (long long)c.rows * (heads / c.heads) <= 16LL * c.seqs;
#define ANN_PW(D, F)                                                                             \
  return pw_launch<D, F>(c, q, qt, qh, heads, lse, scale * PA_LOG2E, win, w, wrow, out, orow, cap, st)
  if (Dh == 64) {
    if (few) ANN_PW(64, true); else ANN_PW(64, false);
  }
  if (Dh == 128) {
    if (few) ANN_PW(128, true); else ANN_PW(128, false);
  }
#undef ANN_PW
  return hipErrorInvalidValue;
}

}  // namespace ann
