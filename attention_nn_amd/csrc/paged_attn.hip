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
// rounds it); its sum is of the unrounded weights.
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

// 16-byte chunk c of LDS row r is stored at chunk c ^ swz(r): conflict-free for
// the fragment reads of the keys and the transposed ones of the values.
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
template <int I, int N, typename F>
__device__ __forceinline__ void pa_static_for(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    pa_static_for<I + 1, N>(f);
  }
}

// How a tile's entries [lo, hi) are shared out: n parts of `per` entries from lo
// rounded down to 32.  per is a multiple of 64; up to most parts, of 128 entries
// at least.
struct PaParts {
  int begin, per, n;
};
__device__ __forceinline__ PaParts pa_parts(int lo, int hi, int most) {
  PaParts p;
  p.begin = lo & ~31;
  const int total = hi - p.begin;
  if (hi <= lo) return {0, 64, 1};
  const int n = min(most, (total + 127) / 128);
  p.per = ((total + n - 1) / n + 63) & ~63;
  p.n = (total + p.per - 1) / p.per;
  return p;
}

struct PaArgs {
  PagedArgs c;
  const bf16_t* q;
  long long qt, qh;
  int heads, window;   // window: none is INT_MAX
  float sl2, thr;      // |scale| log2(e); 8 / sl2, the rise of m's that is let pass
  int neg;             // scale < 0: the queries enter negated
  bf16_t* out;
  float* lse;
  float* po;           // partial sums (rows, heads, parts, DH), or null: one part
  float2* pml;         // (rows, heads, parts): m in log2 units, sum
  int ns_few, ns_many; // most parts of a tile of each kind
  int nsmax;           // the larger, the stride of the partials
  int few;             // rows of a sequence up to which k_paged_few takes it
  int br;              // rows of k_paged_many's tiles
};

// One sequence's new tokens as a call sees them.
struct PaSeq {
  int first, n, len, rows, G, e0;   // e0: entry of token 0
};
__device__ __forceinline__ PaSeq pa_seq(const PaArgs& a, int s) {
  const PgRange r = pg_range(a.c.starts[s], a.c.starts[s + 1], a.c.rows);
  PaSeq q;
  q.first = r.first;
  q.n = r.n;
  q.len = pg_len(a.c.lens[s], a.c.cols, a.c.sh);
  q.G = a.heads / a.c.heads;
  q.rows = r.n * q.G;
  q.e0 = q.len - r.n;
  return q;
}
// The entries that rows row0 .. row0 + n - 1 see.
__device__ __forceinline__ void pa_span(const PaSeq& q, int row0, int n, int window, int& lo, int& hi) {
  const int el = q.e0 + row0 / q.G, eh = q.e0 + (row0 + n - 1) / q.G;
  lo = el < window ? 0 : el - window + 1;
  hi = max(eh + 1, 0);
}

// Final or partial result of one row (token, head) part: 4 dims from d on.
template <int DH>
__device__ __forceinline__ void pa_store4(const PaArgs& a, int n, int h, int part, int parts, int d,
                                          float4 o, float m, float l) {
  const long long r = (long long)n * a.heads + h;
  if (parts == 1) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *(uint2*)(a.out + r * DH + d) =
        make_uint2(pack2(o.x * inv, o.y * inv), pack2(o.z * inv, o.w * inv));
    if (d == 0 && a.lse)
      a.lse[r] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * PA_LN2;
  } else {
    const long long x = r * a.nsmax + part;
    *(float4*)(a.po + x * DH + d) = o;
    if (d == 0) a.pml[x] = make_float2(m, l);
  }
}

// A row formed entry by entry, over the part [a0, b0) of what it sees.
template <int DH>
__device__ __forceinline__ void pa_again(const PaArgs& a, const PaSeq& q, const int32_t* table,
                                         int kvh, int row, int a0, int b0, int part, int parts) {
  constexpr int DL = DH / 64;
  const int lane = threadIdx.x & 63;
  const int t = row / q.G, e = q.e0 + t, n = q.first + t, h = kvh * q.G + row % q.G;
  const int lo = max(a0, e < a.window ? 0 : e - a.window + 1), hi = min(b0, e + 1);
  float m, l, o[DL];
  pa_row<DH>(a.c, table, a.q + n * a.qt + h * a.qh, kvh, lo, hi, a.neg ? -a.sl2 : a.sl2, m, l, o);
  // lane i holds dims i DL ..: four lanes' (two's) values to the one that stores them
  float4 v;
  if constexpr (DL == 1) {
    v = make_float4(o[0], __shfl_down(o[0], 1, 64), __shfl_down(o[0], 2, 64), __shfl_down(o[0], 3, 64));
    if (lane % 4 == 0) pa_store4<DH>(a, n, h, part, parts, lane, v, m, l);
  } else {
    v = make_float4(o[0], o[1], __shfl_down(o[0], 1, 64), __shfl_down(o[1], 1, 64));
    if (lane % 2 == 0) pa_store4<DH>(a, n, h, part, parts, lane * 2, v, m, l);
  }
}

__device__ __forceinline__ bool pa_finite(const floatx4_t& v) {
  // 0 times a finite number is 0, times any other NaN
  const float z = v[0] * 0.f + v[1] * 0.f + v[2] * 0.f + v[3] * 0.f;
  return z == 0.f;
}

// The running maximum raised where a lane's largest score lm passes it by more
// than thr; the four lanes of a row agree on it.
template <int NDB>
__device__ __forceinline__ void pa_raise(float lm, float thr, float sl2, float& m, float& msl,
                                         float& lsum, floatx4_t* o) {
  if (!__any(lm > m + thr)) return;
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

__device__ __forceinline__ bf16x8_t pa_query(const bf16_t* p, int neg) {
  uint4 w = *(const uint4*)p;
  const uint32_t x = neg ? 0x80008000u : 0u;
  w.x ^= x;
  w.y ^= x;
  w.z ^= x;
  w.w ^= x;
  return __builtin_bit_cast(bf16x8_t, w);
}

__device__ __forceinline__ bf16x8_t pa_join(pa_v4i16 a, pa_v4i16 b) {
  return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// The 16 entries of a cache from entry k0 on (a multiple of 16): a uniform
// address, to which a lane adds its row's and column's 32 bits.
__device__ __forceinline__ const unsigned char* pa_group(const bf16_t* head, int id, long long page,
                                                         long long slot, int k0, int sh) {
  return (const unsigned char*)(head + id * page + pg_slot(k0, sh, slot));
}

// Page ids ahead of their use: lane i of a wave holds the id of its i-th group of
// 16 entries.
struct PaPages {
  int now, next;
};

// ---- sequences of few rows ----------------------------------------------------------
//
// A work-group takes a part of a sequence's entries for one cache head, 16 rows at
// a time (one row of a decoding sequence without shared heads).  Its four waves
// take chunks of 32 entries in turn and meet only at the end: keys from memory
// straight into the fragments of the product, two chunks ahead; values into the
// wave's own ring of LDS stages.
template <int DH>
__global__ __launch_bounds__(256, 2) void k_paged_few(PaArgs a) {
  constexpr int RB = DH * 2, TB = 32 * RB;      // bytes of an LDS row, of a chunk's values
  constexpr int LPW = TB / 1024, RPL = 1024 / RB;   // loads of a chunk's values, rows of each
  constexpr int NKS = DH / 32, NDB = DH / 16, PW = DH + 4;
  // the rings; after them the waves' sums, their maxima and totals, rows to form again
  constexpr int RING = 4 * 2 * TB, SUMS = 4 * 16 * PW * 4 + (2 * 64 + 16) * 4;
  __shared__ __attribute__((aligned(16))) unsigned char smem[RING > SUMS ? RING : SUMS];
  float* sums = (float*)smem;
  float* s_m = sums + 4 * 16 * PW;
  float* s_l = s_m + 64;
  int* s_bad = (int*)(s_l + 64);

  const int s = blockIdx.y, kvh = blockIdx.x % a.c.heads, part = blockIdx.x / a.c.heads;
  const PaSeq q = pa_seq(a, s);
  if (q.rows == 0 || q.rows > a.few) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, g4 = lane >> 4;
  const int32_t* table = a.c.table + s * a.c.trow;
  const bf16_t* kh = a.c.k + kvh * a.c.kh;
  const bf16_t* vh = a.c.v + kvh * a.c.vh;
  unsigned char* ring = smem + wv * 2 * TB;
  const int trow = 4 * g4 + (r16 >> 2), tcol = 4 * (r16 & 3), vx = pa_swz<DH>(trow);

  for (int row0 = 0; row0 < q.rows; row0 += 16) {
    const int nrow = min(16, q.rows - row0);
    int lo, hi;
    pa_span(q, row0, nrow, a.window, lo, hi);
    const PaParts pt = pa_parts(lo, hi, a.ns_few);
    if (part >= pt.n) continue;
    const int a0 = max(pt.begin + part * pt.per, lo), b0 = min(pt.begin + (part + 1) * pt.per, hi);
    const int kb0 = pt.begin + part * pt.per;
    const int nch = b0 > a0 ? (b0 - kb0 + 31) / 32 : 0;
    const int nt = nch > wv ? (nch - wv + 3) / 4 : 0;   // chunks of this wave

    const int row = row0 + min(r16, nrow - 1), tok = row / q.G;
    const int e = q.e0 + tok;
    const int el = q.e0 + row0 / q.G, eh = q.e0 + (row0 + nrow - 1) / q.G;
    const bf16_t* qr = a.q + (q.first + tok) * a.qt + (kvh * q.G + row % q.G) * a.qh + g4 * 8;
    bf16x8_t qf[NKS];
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) qf[ks] = pa_query(qr + ks * 32, a.neg);

    floatx4_t o[NDB];
#pragma unroll
    for (int i = 0; i < NDB; ++i) o[i] = (floatx4_t){0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, msl = 0.f, lsum = 0.f;

    // ids of chunks 32 b .. 32 b + 31 of this wave: lane i group i & 1 of chunk i >> 1
    auto ids = [&](int b) {
      const int key = kb0 + 32 * (wv + 4 * (32 * b + (lane >> 1))) + 16 * (lane & 1);
      return pg_read(table[min(max(key, a0), b0 - 1) >> a.c.sh], a.c.pages);
    };
    PaPages pg = {nt ? ids(0) : 0, nt > 32 ? ids(1) : 0};
    bf16x8_t kf[2][2][NKS];
    auto issue = [&](int t, int slot) {
      asm volatile("" ::: "memory");   // behind the reads of the stage it fills
      if (t && t % 32 == 0) {
        pg.now = pg.next;
        if (t + 32 < nt) pg.next = ids(t / 32 + 1);
      }
      const int kb = kb0 + 32 * (wv + 4 * t);
      unsigned char* st = ring + (t & 1) * TB;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int id = __builtin_amdgcn_readlane(pg.now, 2 * (t % 32) + g);
        // entries inside [a0, b0): where the whole group lies outside, the nearest one's page
        const int k0 = min(max(kb + 16 * g, a0 & ~15), (b0 - 1) & ~15);
        const int rl = max(a0 - k0, 0), rh = min(b0 - 1 - k0, 15);
        const unsigned char* kp = pa_group(kh, id, a.c.kp, a.c.ks, k0, a.c.sh);
        const unsigned char* vp = pa_group(vh, id, a.c.vp, a.c.vs, k0, a.c.sh);
        const unsigned ko = (unsigned)(min(max(r16, rl), rh) * (int)a.c.ks * 2 + g4 * 16);
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) kf[slot][g][ks] = *(const bf16x8_t*)(kp + ko + ks * 64);
#pragma unroll
        for (int u = 0; u < LPW / 2; ++u) {
          const int r = u * RPL + lane / (RB / 16);   // row of the group
          const int col = ((lane % (RB / 16)) ^ pa_swz<DH>(r)) * 16;
          const unsigned vo = (unsigned)(min(max(r, rl), rh) * (int)a.c.vs * 2 + col);
          __builtin_amdgcn_global_load_lds(vp + vo, (pa_lds_void*)(st + (g * LPW / 2 + u) * 1024), 16, 0, 0);
        }
      }
    };
    auto compute = [&](int t, int slot) {
      const int kb = kb0 + 32 * (wv + 4 * t);
      floatx4_t sacc[2];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        sacc[g] = (floatx4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks)
          sacc[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[slot][g][ks], qf[ks], sacc[g], 0, 0, 0);
      }
      const bool full = kb >= a0 && kb + 31 < b0 && kb + 31 <= el && eh - kb < a.window;
      float p[2][4], lm = -INFINITY;
      bool ok[2][4];
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = kb + 16 * g + 4 * g4 + r;
          ok[g][r] = full || (j >= a0 && j < b0 && j <= e && e - j < a.window);
          lm = fmaxf(lm, ok[g][r] ? sacc[g][r] : -INFINITY);
        }
      pa_raise<NDB>(lm, a.thr, a.sl2, m, msl, lsum, o);
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[g][r] = ok[g][r] ? __builtin_amdgcn_exp2f(sacc[g][r] * a.sl2 - msl) : 0.f;
          lsum += p[g][r];
        }
      uint32_t pw[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) pw[x] = pack2(p[x >> 1][(x & 1) * 2], p[x >> 1][(x & 1) * 2 + 1]);
      const bf16x8_t pf = *(const bf16x8_t*)pw;
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
        pa_wait_lgkm<2 * (NDB - 1 - db)>(v0[db]);
        pa_wait_lgkm<2 * (NDB - 1 - db)>(v1[db]);
        o[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pa_join(v0[db], v1[db]), pf, o[db], 0, 0, 0);
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
    auto joined = [&](int r, int d, float& M, float& L) {
      M = fmaxf(fmaxf(s_m[r], s_m[16 + r]), fmaxf(s_m[32 + r], s_m[48 + r]));
      L = 0.f;
      floatx4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = M == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(s_m[w * 16 + r] - M);
        L += s_l[w * 16 + r] * f;
        v += *(const floatx4_t*)(sums + (w * 16 + r) * PW + d) * f;
      }
      return v;
    };
    float M, L;
    if (nrow > 1) {   // one row alone sees all that its part reads
      for (int i = tid; i < nrow * (DH / 4); i += 256)
        if (!pa_finite(joined(i / (DH / 4), i % (DH / 4) * 4, M, L))) s_bad[i / (DH / 4)] = 1;
      __syncthreads();
    }
    for (int i = tid; i < nrow * (DH / 4); i += 256) {
      const int r = i / (DH / 4), d = i % (DH / 4) * 4, rr = row0 + r;
      if (s_bad[r]) continue;
      const floatx4_t v = joined(r, d, M, L);
      pa_store4<DH>(a, q.first + rr / q.G, kvh * q.G + rr % q.G, part, pt.n, d,
                    make_float4(v[0], v[1], v[2], v[3]), M, L);
    }
    for (int r = wv; r < nrow; r += 4)
      if (s_bad[r]) pa_again<DH>(a, q, table, kvh, row0 + r, a0, b0, part, pt.n);
    __syncthreads();   // the sums are read before the next rows' chunks arrive
  }
}

// ---- sequences of many rows -----------------------------------------------------------
//
// A work-group takes BR = 64 QB rows (four waves of QB x 16) and a part of the
// entries, which pass through a ring of two LDS stages shared by its waves: loaded
// straight into LDS a step ahead, one barrier a step.  A key or value fragment
// read from LDS serves QB products.
template <int DH, int BK, int QB>
__global__ __launch_bounds__(256, 2) void k_paged_many(PaArgs a, int tiles) {
  constexpr int BR = 64 * QB, RB = DH * 2, TB = BK * RB;
  constexpr int LPW = TB / 1024 / 4, RPL = 1024 / RB;   // loads a wave makes of K (and of V), rows of each
  constexpr int NKS = DH / 32, NDB = DH / 16, NBLK = BK / 16, NI = BK / 32, GPT = BK / 16;
  __shared__ __attribute__((aligned(16))) unsigned char smem[2 * 2 * TB];

  // tiles of one (cache head, part) run together on one XCD and share its L2:
  // work-group L runs on XCD L % 8
  const int total = gridDim.x, L = blockIdx.x;
  const int w = total % 8 == 0 ? (L % 8) * (total / 8) + L / 8 : L;
  const int tile = w % tiles, kvh = (w / tiles) % a.c.heads, part = w / tiles / a.c.heads;
  int s = 0, row0 = 0;
  if (!pg_tile(a.c.starts, a.c.seqs, a.c.rows, a.heads / a.c.heads, a.few, BR, tile, s, row0)) return;
  s = __builtin_amdgcn_readfirstlane(s);
  row0 = __builtin_amdgcn_readfirstlane(row0);
  const PaSeq q = pa_seq(a, s);
  const int nrow = min(BR, q.rows - row0);
  int lo, hi;
  pa_span(q, row0, nrow, a.window, lo, hi);
  const PaParts pt = pa_parts(lo, hi, a.ns_many);
  if (part >= pt.n) return;
  const int kb0 = pt.begin + part * pt.per;
  const int a0 = max(kb0, lo), b0 = min(kb0 + pt.per, hi);
  const int nt = b0 > a0 ? (b0 - kb0 + BK - 1) / BK : 0;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, g4 = lane >> 4;
  const int32_t* table = a.c.table + s * a.c.trow;
  const bf16_t* kh = a.c.k + kvh * a.c.kh;
  const bf16_t* vh = a.c.v + kvh * a.c.vh;

  // this wave's rows, past the last one copies of it; their entries el .. eh
  const int wr0 = row0 + wv * 16 * QB, last = q.rows - 1;
  const bool some = wr0 <= last;
  const int el = q.e0 + min(wr0, last) / q.G, eh = q.e0 + min(wr0 + 16 * QB - 1, last) / q.G;
  bf16x8_t qf[QB][NKS];
  int e[QB];
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    const int row = min(wr0 + 16 * b + r16, last), tok = row / q.G;
    e[b] = q.e0 + tok;
    const bf16_t* qr = a.q + (q.first + tok) * a.qt + (kvh * q.G + row % q.G) * a.qh + g4 * 8;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) qf[b][ks] = pa_query(qr + ks * 32, a.neg);
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

  constexpr int TPB = 64 / GPT;   // tiles whose page ids a wave holds
  auto ids = [&](int b) {
    const int key = kb0 + BK * TPB * b + 16 * lane;
    return pg_read(table[min(max(key, a0), b0 - 1) >> a.c.sh], a.c.pages);
  };
  PaPages pg = {nt ? ids(0) : 0, nt > TPB ? ids(1) : 0};
  // load x of a tile is rows x RPL .. of it: this lane's row of its group of 16 and column
  int lrow[LPW], lcol[LPW];
  unsigned koff[LPW], voff[LPW];
#pragma unroll
  for (int u = 0; u < LPW; ++u) {
    const int r = (wv * LPW + u) * RPL + lane / (RB / 16);
    lrow[u] = r % 16;
    lcol[u] = ((lane % (RB / 16)) ^ pa_swz<DH>(r)) * 16;
    koff[u] = (unsigned)(lrow[u] * (int)a.c.ks * 2 + lcol[u]);
    voff[u] = (unsigned)(lrow[u] * (int)a.c.vs * 2 + lcol[u]);
  }
  auto issue = [&](int t) {
    if (t && t % TPB == 0) {
      pg.now = pg.next;
      if (t + TPB < nt) pg.next = ids(t / TPB + 1);
    }
    const int kb = kb0 + BK * t;
    unsigned char* st = smem + (t & 1) * 2 * TB;
    const bool inside = kb >= a0 && kb + BK <= b0;
#pragma unroll
    for (int u = 0; u < LPW; ++u) {
      const int x = wv * LPW + u, g = x * RPL / 16;   // the load, and its group of 16 entries
      const int id = __builtin_amdgcn_readlane(pg.now, GPT * (t % TPB) + g);
      int k0 = kb + 16 * g;
      unsigned ko = koff[u], vo = voff[u];
      if (!inside) {   // rows outside [a0, b0) take the nearest inside
        k0 = min(max(k0, a0 & ~15), (b0 - 1) & ~15);
        const int rc = min(max(lrow[u], a0 - k0), b0 - 1 - k0);
        ko = (unsigned)(rc * (int)a.c.ks * 2 + lcol[u]);
        vo = (unsigned)(rc * (int)a.c.vs * 2 + lcol[u]);
      }
      __builtin_amdgcn_global_load_lds(pa_group(kh, id, a.c.kp, a.c.ks, k0, a.c.sh) + ko,
                                       (pa_lds_void*)(st + x * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds(pa_group(vh, id, a.c.vp, a.c.vs, k0, a.c.sh) + vo,
                                       (pa_lds_void*)(st + TB + x * 1024), 16, 0, 0);
    }
  };
  // fragment addresses of the first stage; the second lies 2 TB behind
  const int trow = 4 * g4 + (r16 >> 2), tcol = 4 * (r16 & 3);
  pa_lds_cchar* kadr[NKS];
  pa_lds_cchar* vadr[NDB];
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks)
    kadr[ks] = (pa_lds_cchar*)smem + r16 * RB + (((ks * 4 + g4) ^ pa_swz<DH>(r16)) << 4);
#pragma unroll
  for (int db = 0; db < NDB; ++db)
    vadr[db] = (pa_lds_cchar*)smem + TB + trow * RB + (tcol & 7) * 2 +
               (((2 * db + (tcol >> 3)) ^ pa_swz<DH>(trow)) << 4);

  auto step = [&](int t, auto stage) __attribute__((always_inline)) {
    constexpr int ST = decltype(stage)::value * 2 * TB;
    const int kb = kb0 + BK * t;
    pa_wait_vm<0>();   // this wave's part of tile t is in LDS
    __syncthreads();   // every wave's; the other stage is free
    if (t + 1 < nt) issue(t + 1);
    if (!(some && kb <= eh && el - (kb + BK - 1) < a.window)) return;   // nothing in it for this wave
    const bool full = kb >= a0 && kb + BK - 1 < b0 && kb + BK - 1 <= el && eh - kb < a.window;

    floatx4_t sacc[QB][NBLK];
#pragma unroll
    for (int b = 0; b < QB; ++b)
#pragma unroll
      for (int i = 0; i < NBLK; ++i) sacc[b][i] = (floatx4_t){0.f, 0.f, 0.f, 0.f};
    // key fragments: one k-step (NBLK reads) ahead of its products
    bf16x8_t kf[2][NBLK];
    pa_static_for<0, NBLK>([&](auto bc) __attribute__((always_inline)) {
      constexpr int i = decltype(bc)::value;
      kf[0][i] = pa_rd_b128<ST + i * 16 * RB>(kadr[0]);
    });
    pa_static_for<0, NKS>([&](auto kc) __attribute__((always_inline)) {
      constexpr int ks = decltype(kc)::value;
      if constexpr (ks + 1 < NKS) {
        pa_static_for<0, NBLK>([&](auto bc) __attribute__((always_inline)) {
          constexpr int i = decltype(bc)::value;
          kf[(ks + 1) & 1][i] = pa_rd_b128<ST + i * 16 * RB>(kadr[ks + 1]);
        });
      }
      constexpr int ahead = ks + 1 < NKS ? NBLK : 0;
      pa_static_for<0, NBLK>([&](auto bc) __attribute__((always_inline)) {
        constexpr int i = decltype(bc)::value;
        pa_wait_lgkm<ahead + NBLK - 1 - i>(kf[ks & 1][i]);
#pragma unroll
        for (int b = 0; b < QB; ++b)
          sacc[b][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[ks & 1][i], qf[b][ks], sacc[b][i], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      });
    });

    float p[QB][NBLK][4];
    if (full) {
#pragma unroll
      for (int b = 0; b < QB; ++b) {
        float lm = sacc[b][0][0];
#pragma unroll
        for (int i = 0; i < NBLK; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) lm = fmaxf(lm, sacc[b][i][r]);
        pa_raise<NDB>(lm, a.thr, a.sl2, m[b], msl[b], lsum[b], o[b]);
#pragma unroll
        for (int i = 0; i < NBLK; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            p[b][i][r] = __builtin_amdgcn_exp2f(sacc[b][i][r] * a.sl2 - msl[b]);
      }
    } else {
#pragma unroll
      for (int b = 0; b < QB; ++b) {
        // entries jl .. jh of this lane's four of each block; a masked one's score is -inf
        const int jl = max(a0, e[b] < a.window ? 0 : e[b] - a.window + 1) - kb - 4 * g4;
        const int jh = min(b0 - 1, e[b]) - kb - 4 * g4;
        float lm = -INFINITY;
#pragma unroll
        for (int i = 0; i < NBLK; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool ok = 16 * i + r >= jl && 16 * i + r <= jh;
            sacc[b][i][r] = ok ? sacc[b][i][r] : -INFINITY;
            lm = fmaxf(lm, sacc[b][i][r]);
          }
        pa_raise<NDB>(lm, a.thr, a.sl2, m[b], msl[b], lsum[b], o[b]);
#pragma unroll
        for (int i = 0; i < NBLK; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float v = __builtin_amdgcn_exp2f(sacc[b][i][r] * a.sl2 - msl[b]);
            const bool ok = 16 * i + r >= jl && 16 * i + r <= jh;
            p[b][i][r] = ok ? v : 0.f;
          }
      }
    }
#pragma unroll
    for (int b = 0; b < QB; ++b)
#pragma unroll
      for (int i = 0; i < NBLK; ++i)
        lsum[b] += (p[b][i][0] + p[b][i][1]) + (p[b][i][2] + p[b][i][3]);
    pa_static_for<0, NI>([&](auto ic) __attribute__((always_inline)) {
      constexpr int i = decltype(ic)::value;
      pa_v4i16 v0[NDB], v1[NDB];
      pa_static_for<0, NDB>([&](auto dc) __attribute__((always_inline)) {
        constexpr int db = decltype(dc)::value;
        v0[db] = pa_rd_tr<ST + 32 * i * RB>(vadr[db]);
        v1[db] = pa_rd_tr<ST + (32 * i + 16) * RB>(vadr[db]);
      });
      bf16x8_t pf[QB];
#pragma unroll
      for (int b = 0; b < QB; ++b) {
        uint32_t pw[4];
#pragma unroll
        for (int x = 0; x < 4; ++x)
          pw[x] = pack2(p[b][2 * i + (x >> 1)][(x & 1) * 2], p[b][2 * i + (x >> 1)][(x & 1) * 2 + 1]);
        pf[b] = *(const bf16x8_t*)pw;
      }
      pa_static_for<0, NDB>([&](auto dc) __attribute__((always_inline)) {
        constexpr int db = decltype(dc)::value;
        pa_wait_lgkm<2 * (NDB - 1 - db)>(v0[db]);
        pa_wait_lgkm<2 * (NDB - 1 - db)>(v1[db]);
        const bf16x8_t vf = pa_join(v0[db], v1[db]);
#pragma unroll
        for (int b = 0; b < QB; ++b)
          o[b][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[b], o[b][db], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      });
    });
  };
  if (nt) issue(0);
  for (int t = 0; t < nt; t += 2) {
    step(t, std::integral_constant<int, 0>{});
    if (t + 1 < nt) step(t + 1, std::integral_constant<int, 1>{});
  }
  pa_wait_vm<0>();
  if (!some) return;
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    const int row = wr0 + 16 * b + r16, tok = min(row, last) / q.G;
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
        pa_store4<DH>(a, q.first + tok, kvh * q.G + row % q.G, part, pt.n, db * 16 + g4 * 4,
                      make_float4(o[b][db][0], o[b][db][1], o[b][db][2], o[b][db][3]), M, l);
    while (bad) {
      const int r = __builtin_ctzll(bad);
      bad &= bad - 1;
      pa_again<DH>(a, q, table, kvh, wr0 + 16 * b + r, a0, b0, part, pt.n);
    }
  }
}

// The parts of each row joined, in part order: one wave for each (token, head).
template <int DH>
__global__ __launch_bounds__(256) void k_paged_join(PaArgs a) {
  constexpr int DL = DH / 64;
  const int lane = threadIdx.x & 63;
  const long long w = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = (int)(w / a.heads), h = (int)(w % a.heads);
  if (n >= a.c.rows) return;
  const int s = pg_sequence(a.c.starts, a.c.seqs, n);
  if (s < 0) return;
  const PaSeq q = pa_seq(a, s);
  if (n - q.first >= q.n) return;
  const bool few = q.rows <= a.few;
  const int br = few ? 16 : a.br;
  const int row0 = ((n - q.first) * q.G + h % q.G) / br * br;
  int lo, hi;
  pa_span(q, row0, min(br, q.rows - row0), a.window, lo, hi);
  const int np = pa_parts(lo, hi, few ? a.ns_few : a.ns_many).n;
  if (np == 1) return;
  const float2* ml = a.pml + w * a.nsmax;
  const float* po = a.po + w * a.nsmax * DH + lane * DL;
  float M = -INFINITY;
  for (int i = 0; i < np; ++i) M = fmaxf(M, ml[i].x);
  const float base = M == -INFINITY ? 0.f : M;
  float l = 0.f, o[DL] = {};
  for (int i = 0; i < np; ++i) {
    const float f = __builtin_amdgcn_exp2f(ml[i].x - base);
    l += ml[i].y * f;
#pragma unroll
    for (int d = 0; d < DL; ++d) o[d] += po[i * DH + d] * f;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int d = 0; d < DL; ++d) a.out[w * DH + lane * DL + d] = f2bf(o[d] * inv);
  if (a.lse && lane == 0) a.lse[w] = l == 0.f ? -INFINITY : (M + __builtin_amdgcn_logf(l)) * PA_LN2;
}

// What a call launches, from what the host knows: rows and sequences, not how
// the rows are shared out among them.
struct PaPlan {
  int few;             // rows of a sequence up to which k_paged_few takes it
  bool many;           // k_paged_many runs too
  int qb, tiles;       // its row blocks and (at most) its tiles
  int ns_few, ns_many;
};
static PaPlan pa_plan(const PagedArgs& c, int heads, int window) {
  static const int cus = device_cus();
  PaPlan p{};
  const int G = heads / c.heads;
  const long long rows = (long long)c.rows * G;
  long long keys = (long long)c.cols << c.sh;
  if (window > 0 && keys > window + 31LL) keys = window + 31LL;
  const auto clamp = [](long long v, long long hi) { return (int)(v < 1 ? 1 : v > hi ? hi : v); };
  const long long most = clamp((keys + 127) / 128, 64);
  p.many = rows > 16 && c.rows > c.seqs;
  p.few = !p.many ? 0x7fffffff : c.seqs == 1 ? 0 : 16;
  p.ns_few = clamp((2LL * cus + (long long)c.seqs * c.heads - 1) / ((long long)c.seqs * c.heads), most);
  if (p.many) {
    p.qb = rows >= 96LL * c.seqs ? 2 : 1;
    const int br = 64 * p.qb;
    const long long bands = c.seqs < c.rows ? c.seqs : c.rows;
    p.tiles = (int)(rows / br + bands);
    long long k2 = (long long)c.cols << c.sh;
    if (window > 0 && k2 > window + br + 31LL) k2 = window + br + 31LL;
    p.ns_many = clamp((2LL * cus) / ((long long)p.tiles * c.heads), clamp((k2 + 127) / 128, 16));
  } else {
    p.ns_many = 1;
  }
  return p;
}
static size_t pa_ws(const PagedArgs& c, int heads, int Dh, const PaPlan& p) {
  const int ns = p.ns_few > p.ns_many ? p.ns_few : p.ns_many;
  return ns == 1 ? 0 : (size_t)c.rows * heads * ns * (Dh + 2) * 4;
}

size_t paged_attention_ws_bytes(const PagedArgs& c, int heads, int Dh, int window) {
  return c.rows == 0 || c.seqs == 0 ? 0 : pa_ws(c, heads, Dh, pa_plan(c, heads, window));
}

hipError_t paged_attention(const PagedArgs& c, const bf16_t* q, long long qt, long long qh,
                           int heads, int Dh, float scale, int window, bf16_t* out, float* lse,
                           void* ws, hipStream_t st) {
  if (c.rows == 0 || c.seqs == 0) return hipSuccess;
  if (Dh != 64 && Dh != 128) return hipErrorInvalidValue;
  const PaPlan p = pa_plan(c, heads, window);
  PaArgs a{};
  a.c = c;
  a.q = q;
  a.qt = qt;
  a.qh = qh;
  a.heads = heads;
  a.window = window > 0 ? window : 0x7fffffff;
  a.sl2 = fabsf(scale) * PA_LOG2E;
  a.thr = fminf(8.f / a.sl2, 3e38f);
  a.neg = scale < 0.f;
  a.out = out;
  a.lse = lse;
  a.ns_few = p.ns_few;
  a.ns_many = p.ns_many;
  a.nsmax = p.ns_few > p.ns_many ? p.ns_few : p.ns_many;
  a.few = p.few;
  a.br = 64 * p.qb;
  a.po = (float*)ws;
  a.pml = (float2*)((float*)ws + (size_t)c.rows * heads * a.nsmax * Dh);
  const dim3 block(256);
  if (p.many) {
    const long long n = (long long)p.tiles * c.heads * p.ns_many;
    if (n > 0x7fffffffLL) return hipErrorInvalidValue;
    const dim3 grid((unsigned)n);
#define ANN_PM(D, BK, QB) \
  hipLaunchKernelGGL((k_paged_many<D, BK, QB>), grid, block, 0, st, a, p.tiles)
    if (Dh == 64) {
      if (p.qb == 2) ANN_PM(64, 64, 2); else ANN_PM(64, 64, 1);
    } else {
      if (p.qb == 2) ANN_PM(128, 32, 2); else ANN_PM(128, 32, 1);
    }
#undef ANN_PM
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (p.few > 0) {
    const dim3 grid((unsigned)(c.heads * p.ns_few), (unsigned)c.seqs);
    if (Dh == 64) hipLaunchKernelGGL(k_paged_few<64>, grid, block, 0, st, a);
    else hipLaunchKernelGGL(k_paged_few<128>, grid, block, 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (a.nsmax > 1) {
    const dim3 grid((unsigned)(((long long)c.rows * heads + 3) / 4));
    if (Dh == 64) hipLaunchKernelGGL(k_paged_join<64>, grid, block, 0, st, a);
    else hipLaunchKernelGGL(k_paged_join<128>, grid, block, 0, st, a);
  }
  return hipGetLastError();
}

// ---- weight of the entries -------------------------------------------------------
//
// A work-group takes WE entries of a sequence and all rows (token, head) that see
// any of them, its waves an equal share of them each: in the order of the cache
// heads, so that a wave's keys stay in registers from one 16 rows to the next.
// S = K Q^T, entries x rows, 16 x 16 a product: a lane adds the weights of its
// row's column for its four entries of each block, and only at the end are the 16
// columns and the waves added, in a fixed order, so a sum does not depend on what
// else is in the call.
constexpr int PW_E = 32;   // entries a work-group
template <int DH>
__global__ __launch_bounds__(512, 4) void k_paged_weight(PagedArgs c, const bf16_t* __restrict__ q,
                                                         long long qt, long long qh, int heads,
                                                         FastDiv group,
                                                         const float* __restrict__ lse, float sl2,
                                                         int neg, int window, const float* w,
                                                         long long wrow, float* out, long long orow,
                                                         int cap) {
  constexpr int NKS = DH / 32, NB = PW_E / 16;
  __shared__ float part[8][PW_E];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g4 = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int s = blockIdx.y, j0 = blockIdx.x * PW_E, j = j0 + tid;
  const int len = pg_len(c.lens[s], c.cols, c.sh);
  const PgRange r = pg_range(c.starts[s], c.starts[s + 1], c.rows);
  const float was = tid < PW_E && j < cap ? w[s * wrow + j] : 0.f;
  const int G = heads / c.heads, e0 = len - r.n, jl = min(j0 + PW_E - 1, len - 1);
  // tokens t0 .. t1 - 1 see one of the entries j0 .. jl
  const int t0 = max(0, j0 - e0), t1 = jl - e0 < r.n - window ? jl - e0 + window : r.n;
  float acc[NB][4];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[b][i] = 0.f;
  if (j0 < len && t1 > t0) {
    const int lo = t0 * G, hi = t1 * G;
    const int tiles = (hi - lo + 15) / 16, all = tiles * c.heads, per = (all + 7) / 8;
    const bf16_t* kr[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int k0 = min(j0 + 16 * b, jl & ~15);
      const int id = pg_read(c.table[s * c.trow + (k0 >> c.sh)], c.pages);
      kr[b] = c.k + id * c.kp + pg_slot(k0, c.sh, c.ks) + min(r16, jl - k0) * c.ks + g4 * 8;
    }
    int u = wv * per;
    const int end = min(u + per, all);
    while (u < end) {   // the wave's rows of one cache head
      const int kvh = u / tiles, first = u - kvh * tiles, n = min(tiles - first, end - u);
      u += n;
      bf16x8_t kf[NB][NKS], qf[NKS];
      const bf16_t* qb = q + r.first * qt + (long long)kvh * G * qh + g4 * 8;
      const float* lb = lse + (long long)r.first * heads + kvh * G;
      float l2;
      int e;
      auto load = [&](int tile) {
        const int at = lo + tile * 16 + r16, row = min(at, hi - 1), t = group.div(row), h = row - t * G;
        const bf16_t* qr = qb + t * qt + h * qh;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) qf[ks] = *(const bf16x8_t*)(qr + ks * 32);
        l2 = lb[(long long)t * heads + h];
        e = at < hi ? e0 + t : -1;   // a row past the last sees nothing
      };
      load(first);
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks)
          kf[b][ks] = pa_query(kr[b] + kvh * c.kh + ks * 32, neg);
      for (int i = 0; i < n; ++i) {
        floatx4_t sc[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) sc[b] = (floatx4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
          for (int b = 0; b < NB; ++b)
            sc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[b][ks], qf[ks], sc[b], 0, 0, 0);
        const float base = l2 * PA_LOG2E;
        const int at = e, row0 = lo + (first + i) * 16;
        if (i + 1 < n) load(first + i + 1);
        const bool full = row0 + 16 <= hi && e0 + group.div(row0) >= j0 + PW_E - 1 &&
                          e0 + group.div(row0 + 15) - j0 < window;
        if (full) {
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[b][k] += __builtin_amdgcn_exp2f(sc[b][k] * sl2 - base);
        } else {
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int x = j0 + 16 * b + 4 * g4 + k;
              acc[b][k] += x <= at && at - x < window ? __builtin_amdgcn_exp2f(sc[b][k] * sl2 - base) : 0.f;
            }
        }
      }
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
  if (tid >= PW_E || j >= cap) return;
  if (j < len) {
    float v = part[0][tid];
#pragma unroll
    for (int k = 1; k < 8; ++k) v += part[k][tid];
    out[s * orow + j] = was + v;
  } else if (out != w) {
    out[s * orow + j] = was;
  }
}

size_t paged_weight_ws_bytes(const PagedArgs&, int, int) { return 0; }

hipError_t paged_weight(const PagedArgs& c, const bf16_t* q, long long qt, long long qh, int heads,
                        int Dh, const float* lse, float scale, int window, const float* w,
                        long long wrow, float* out, long long orow, void* ws, hipStream_t st) {
  const int cap = c.cols << c.sh;
  if (c.seqs == 0 || cap == 0) return hipSuccess;
  (void)ws;
  const int win = window > 0 ? window : 0x7fffffff;
  const dim3 grid((unsigned)((cap + PW_E - 1) / PW_E), (unsigned)c.seqs), block(512);
#define ANN_PW(D)                                                                               \
  hipLaunchKernelGGL(k_paged_weight<D>, grid, block, 0, st, c, q, qt, qh, heads,                 \
                     FastDiv::of(heads / c.heads), lse,                                         \
                     fabsf(scale) * PA_LOG2E, (int)(scale < 0.f), win, w, wrow, out, orow, cap)
  if (Dh == 64) ANN_PW(64);
  else if (Dh == 128) ANN_PW(128);
  else return hipErrorInvalidValue;
#undef ANN_PW
  return hipGetLastError();
}

}  // namespace ann
