// A token of each row of logits, by given random numbers (sample.hip draws by its
// own, from the lm_head's candidates).
//
//   m = max x, w = exp((x - m) / T) where x is a number and that is at least
//   max(min_p, 2^-40), else 0; of these the x at or above the k-th largest; of these the x at
//   or above the largest t with sum_{x >= t} w >= top_p * sum w; the first index whose
//   running sum of the w left passes u times their sum.
//
// A draw next to a border has to fall to the same side whatever the order of the
// additions, so weights are formed in 64 bits (2^f by a polynomial, relative 2^-50)
// and added as whole numbers of 2^-F, F = 62 - log2 of the entries: exact sums, in
// any order, LDS atomics too.  2^-46 of the largest weight an entry at 50257 of them.
//
// A work-group has a row; its waves hold consecutive parts of it in registers (rows
// that do not fit are read again in each pass).  Forming all weights costs a CU as much
// time as reading the row, so entries that cannot be drawn go first: those below
// what min_p leaves, and below the k-th largest of the threads' maxima, under
// which the k-th largest of all does not lie.  What is left, if 4096 entries at most,
// is listed in LDS in the order of the indices, and thresholds and draw go over the
// list.  top_p alone has no such bound: the entries above the 896th largest
// maximum (some 2000) are listed and serve if their weight is enough of the whole
// row's.  Else (flat rows, many equal values, no limits) the passes go over the row.
// Thresholds by radix selection: sums in 2048 bins of the ordered 32-bit words,
// three rounds at most.
#include <math.h>
#include "common.h"
#include "launch.h"

namespace ann {

constexpr int SL_NT = 1024, SL_NW = SL_NT / 64;
constexpr int SL_BINS = 2048;
constexpr int SL_CAP = 4096;          // entries of the list
constexpr int SL_RANK = 896;          // threads' maxima that bound a k, or the list of a top_p
typedef unsigned long long sl_u64;

struct SlShared {
  sl_u64 hist[SL_BINS];
  float x[SL_CAP];
  int idx[SL_CAP];
  sl_u64 part[2][SL_NW];
  float fpart[2][SL_NW];
  sl_u64 pick[2];
  int at;
};

// Order-preserving word of a number (no NaN, no -0).
__device__ __forceinline__ uint32_t sl_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float sl_value(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
// A NaN is below every number; -0 is 0.
__device__ __forceinline__ float sl_number(float x) { return x == x ? x + 0.f : -INFINITY; }

// Sum over the work-group, and (ex) over the threads before this one.
__device__ __forceinline__ sl_u64 sl_scan(sl_u64 v, sl_u64& ex, SlShared& sh, int which) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  sl_u64 in = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const sl_u64 u = __shfl_up(in, o, 64);
    if (lane >= o) in += u;
  }
  __syncthreads();   // the part's last readers are done
  if (lane == 63) sh.part[which][wv] = in;
  __syncthreads();
  sl_u64 before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < SL_NW; ++w) {
    if (w == wv) before = all;
    all += sh.part[which][w];
  }
  ex = before + in - v;
  return all;
}

// The weights of a row.
struct SlWeight {
  float m;              // the largest entry
  float low;            // entries below have no weight (those above may have none either)
  double md, c, least;  // m, log2(e) / T, the least weight that counts
  double magic;         // 2^(52 - F): a sum's last F bits of fraction are the fixed-point weight
  sl_u64 one;           // 2^F
  __device__ __forceinline__ sl_u64 operator()(float x) const {
    if (!(x >= low)) return 0;
    if (x == m) return one;
    const double y = ((double)x - md) * c;
    if (!(y > -41.0)) return 0;
    const double n = rint(y), f = y - n;
    // (2^f - 1) / f on [-1/2, 1/2], interpolated at the Chebyshev nodes: relative 2^-50 of 2^f
    double q = 0x1.e5e9f548e5725p-28;
    q = fma(q, f, 0x1.b6571de2f2351p-24);
    q = fma(q, f, 0x1.62bfe46117445p-20);
    q = fma(q, f, 0x1.ffcb76789860fp-17);
    q = fma(q, f, 0x1.4309130378460p-13);
    q = fma(q, f, 0x1.5d87fe908f88ap-10);
    q = fma(q, f, 0x1.3b2ab6fba385fp-7);
    q = fma(q, f, 0x1.c6b08d7044119p-5);
    q = fma(q, f, 0x1.ebfbdff82c590p-3);
    q = fma(q, f, 0x1.62e42fefa39f7p-1);
    const double w = ldexp(fma(q, f, 1.0), (int)n);
    if (!(w >= least)) return 0;
    return (sl_u64)__double_as_longlong(w + magic) & ((one << 1) - 1);
  }
};

// The row as the work-group holds it: chunk c, 16 bytes, is entries c NE - shift on;
// group g is chunks 64 g + lane, and wave w has groups w J .. w J + J - 1.  NJ > 0: J <=
// NJ, in registers.
template <typename T, int NJ>
struct SlRow {
  static constexpr int NE = 16 / (int)sizeof(T);
  const unsigned char* base;   // 16-byte aligned
  int shift, n, chunks, J;
  int g0, lane;                // the wave's first group
  float held[NJ ? NJ : 1][NE];

  // Index of entry e of this lane's chunk of group g.
  __device__ __forceinline__ int index(int g, int e) const { return (g * 64 * NE + e - shift) + lane * NE; }
  // The first and last words may hold bytes of other rows, or before and behind the
  // tensor: within its allocation, which no aligned 16-byte word crosses the end of.
  __device__ __forceinline__ uint4 load(int g) const {
    return lane < chunks - g * 64 ? *(const uint4*)(base + (long long)g * 1024 + lane * 16) : make_uint4(0, 0, 0, 0);
  }
  // The entries of a chunk; -inf outside the row and for a NaN.
  __device__ __forceinline__ void values(const uint4& w, int g, float* v) const {
    if constexpr (sizeof(T) == 4) {
      v[0] = __uint_as_float(w.x);
      v[1] = __uint_as_float(w.y);
      v[2] = __uint_as_float(w.z);
      v[3] = __uint_as_float(w.w);
    } else {
      unpack8(w, v);
    }
#pragma unroll
    for (int e = 0; e < NE; ++e) v[e] = sl_number(v[e]);
    if (g == 0 || (g + 1) * 64 >= chunks) {   // the same for the wave
      const int i = index(g, 0);
#pragma unroll
      for (int e = 0; e < NE; ++e) v[e] = (unsigned)(i + e) < (unsigned)n ? v[e] : -INFINITY;
    }
  }
  __device__ __forceinline__ void open(const T* row, int cols) {
    const uintptr_t at = (uintptr_t)row;
    base = (const unsigned char*)(at & ~(uintptr_t)15);
    shift = (int)(at & 15) / (int)sizeof(T);
    n = cols;
    chunks = (cols + shift + NE - 1) / NE;
    J = (chunks + SL_NT - 1) / SL_NT;
    g0 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * J;
    lane = threadIdx.x & 63;
    if constexpr (NJ > 0) {
      uint4 w[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j) w[j] = j < J ? load(g0 + j) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        values(w[j], g0 + j, held[j]);
        if (j >= J)
#pragma unroll
          for (int e = 0; e < NE; ++e) held[j][e] = -INFINITY;
      }
    }
  }
  // f(values, group) for each chunk of the thread: a few instructions for each value, or
  // they are not held
  template <typename F>
  __device__ __forceinline__ void chunks_of(F&& f) const {
    if constexpr (NJ > 0) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) f(held[j], g0 + j);
    } else {
      walk(f);
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
    chunks_of([&](const float* v, int) {
#pragma unroll
      for (int e = 0; e < NE; ++e) f(v[e]);
    });
  }
  // The same from memory, a chunk ahead: where f is long.  52 copies of a weight's
  // instructions are 60 KB of code, and a row that was read is in the caches.
  template <typename F>
  __device__ __forceinline__ void walk(F&& f) const {
    uint4 next = load(g0);
#pragma unroll 1
    for (int j = 0; j < J; ++j) {
      const uint4 w = next;
      if (j + 1 < J) next = load(g0 + j + 1);
      float v[NE];
      values(w, g0 + j, v);
      f(v, g0 + j);
    }
  }
  template <typename F>
  __device__ __forceinline__ void heavy(F&& f) const {
    walk([&](const float* v, int) {
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        f(v[e]);
        __builtin_amdgcn_sched_barrier(0);   // one weight's temporaries at a time
      }
    });
  }
};

// Up to N numbers a thread.
template <int N>
struct SlFew {
  float v[N];
  template <typename F>
  __device__ __forceinline__ void heavy(F&& f) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      f(v[i]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// The largest word t in [lo, hi] such that the entries with words in [t, hi] count
// (MASS: weigh) `want` at least, lo where all of [lo, hi] does not.  MASS with
// share >= 0: want is that share of what [lo, hi] weighs.  once: after one round, a
// word at or below t (the lower end of its bin).
template <bool MASS, typename S>
__device__ __forceinline__ uint32_t sl_select(const S& src, const SlWeight& wt, uint32_t lo, uint32_t hi,
                                              sl_u64 want, double share, bool once, SlShared& sh) {
  const int tid = threadIdx.x;
  sl_u64 above = 0;   // of the entries above hi
  while (true) {
    const uint32_t range = hi - lo;
    const int bits = 32 - __clz((int)range);   // 0 for one word
    const int s = bits > 11 ? bits - 11 : 0;
    __syncthreads();
    sh.hist[tid] = 0;
    sh.hist[tid + SL_NT] = 0;
    if (tid == 0) sh.at = -1;
    __syncthreads();
    src.heavy([&](float x) {
      const uint32_t k = sl_key(x);
      if (k >= lo && k <= hi) {
        if constexpr (MASS) {
          const sl_u64 w = wt(x);
          if (w) atomicAdd(&sh.hist[(k - lo) >> s], w);
        } else {
          atomicAdd((unsigned*)&sh.hist[(k - lo) >> s], 1u);
        }
      }
    });
    __syncthreads();
    const int b = SL_BINS - 1 - 2 * tid;
    const sl_u64 v1 = sh.hist[b], v0 = sh.hist[b - 1];
    sl_u64 ex;
    const sl_u64 all = sl_scan(v1 + v0, ex, sh, 0);
    if (MASS && share >= 0.0) {
      want = (sl_u64)ceil(share * (double)all);
      if (want == 0) want = 1;
      if (want > all) want = all;
      share = -1.0;
    }
    ex += above;
    if (ex < want && want <= ex + v1) {
      sh.at = b;
      sh.pick[0] = ex;
    } else if (ex + v1 < want && want <= ex + v1 + v0) {
      sh.at = b - 1;
      sh.pick[0] = ex + v1;
    }
    __syncthreads();
    const int at = sh.at;
    if (at < 0) return lo;
    above = sh.pick[0];
    lo += (uint32_t)at << s;
    if (s == 0 || once) return lo;
    hi = min(hi, lo + ((1u << s) - 1));
  }
}

struct SlArgs {
  LogitRows r;
  int frac;   // F
};

template <typename T, int NJ>
__global__ __launch_bounds__(SL_NT) void k_sample_logits(SlArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char sl_smem[];
  SlShared& sh = *(SlShared*)sl_smem;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = blockIdx.x, V = a.r.cols;
  float u = a.r.u[r];
  const float temp = a.r.temperature ? a.r.temperature[r] : a.r.temperature_all;
  const int k = a.r.top_k ? a.r.top_k[r] : a.r.top_k_all;
  const float top_p = a.r.top_p ? a.r.top_p[r] : a.r.top_p_all;
  const float min_p = a.r.min_p ? a.r.min_p[r] : a.r.min_p_all;

  SlWeight wt;
  wt.c = 1.4426950408889634 / (double)temp;
  wt.least = fmin(fmax((double)min_p, 0x1p-40), 1.0);
  wt.magic = ldexp(1.0, 52 - a.frac);
  wt.one = 1ull << a.frac;
  const double reach = (log2(wt.least) - 1e-3) / wt.c;   // where weights end, less some
  SlRow<T, NJ> row;
  row.open((const T*)a.r.x + r * a.r.stride, V);

  // ---- the largest entry, and the smallest of the threads' largest
  float mine = -INFINITY;
  row.each([&](float x) { mine = fmaxf(mine, x); });
  float tmin;
  {
    const float hi = group_max<64>(mine), lo = -group_max<64>(mine > -INFINITY ? -mine : -INFINITY);
    if (lane == 0) {
      sh.fpart[0][wv] = hi;
      sh.fpart[1][wv] = lo;
    }
    __syncthreads();
    wt.m = sh.fpart[0][0];
    tmin = sh.fpart[1][0];
#pragma unroll
    for (int w = 1; w < SL_NW; ++w) {
      wt.m = fmaxf(wt.m, sh.fpart[0][w]);
      tmin = fminf(tmin, sh.fpart[1][w]);
    }
  }
  if (wt.m == -INFINITY) {   // nothing to draw
    if (tid == 0) {
      a.r.ids[r] = -1;
      if (a.r.logprob) a.r.logprob[r] = -INFINITY;
    }
    return;
  }
  if (!(temp > 0.f)) {   // the lowest index of the largest
    int at = 0x7fffffff;
    row.chunks_of([&](const float* v, int g) {
#pragma unroll
      for (int e = 0; e < SlRow<T, NJ>::NE; ++e)
        if (v[e] == wt.m) at = min(at, row.index(g, e));
    });
    if (tid == 0) sh.at = 0x7fffffff;
    __syncthreads();
    if (at != 0x7fffffff) atomicMin(&sh.at, at);
    __syncthreads();
    if (tid == 0) {
      a.r.ids[r] = sh.at;
      if (a.r.logprob) a.r.logprob[r] = 0.f;
    }
    return;
  }
  u = u >= 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;

  // ---- a bound below which no entry counts
  wt.md = (double)wt.m;
  {
    const double at = wt.md + reach;
    const float f = (float)(at - fabs(at) * 0x1p-22);
    wt.low = f > -3.4028235e38f ? f : -3.4028235e38f;
    if (!(wt.low <= wt.m)) wt.low = wt.m;
  }
  const uint32_t kmax = sl_key(wt.m), klow = sl_key(wt.low);
  const bool by_k = k > 0 && k < V, by_p = top_p < 1.f;
  const double share = by_p ? fmax((double)top_p, 0.0) : 1.0;

  uint32_t thr = klow;     // of the words that are kept so far
  bool ranked = !by_k;     // thr holds the k-th largest
  SlFew<1> top;
  top.v[0] = mine;
  const uint32_t tlow = max(klow, sl_key(tmin));
  const bool bound = by_k && k <= SL_RANK && V > SL_CAP;
  if (bound) thr = max(thr, sl_select<false>(top, wt, tlow, kmax, (sl_u64)k, -1.0, true, sh));

  const auto count = [&](uint32_t from, sl_u64& before) {   // entries from a word on
    const float x0 = sl_value(from);
    int n = 0;
    row.each([&](float x) { n += x >= x0; });
    return sl_scan((sl_u64)n, before, sh, 1);
  };
  sl_u64 before, total = 0;   // total: weight of all that min_p leaves, where known
  sl_u64 n = count(thr, before);
  uint32_t from = thr;        // the list's least word
  if (n > SL_CAP && by_k) {
    // many equal values, or many to keep: the k-th largest itself
    thr = max(thr, sl_select<false>(row, wt, thr, kmax, (sl_u64)k, -1.0, false, sh));
    ranked = true;
    from = thr;
    n = count(from, before);
  }
  if (n > SL_CAP && by_p && !by_k) {
    const uint32_t cut = max(thr, sl_select<false>(top, wt, tlow, kmax, (sl_u64)SL_RANK, -1.0, true, sh));
    const float x0 = sl_value(cut);
    int some = 0;
    sl_u64 all = 0, listed = 0, ex;
    row.heavy([&](float x) {
      const sl_u64 w = wt(x);
      all += w;
      if (x >= x0) {
        ++some;
        listed += w;
      }
    });
    total = sl_scan(all, ex, sh, 0);
    const sl_u64 got = sl_scan(listed, ex, sh, 1), few = sl_scan((sl_u64)some, before, sh, 0);
    if (few <= SL_CAP && (double)got >= share * (double)total) {
      from = cut;
      n = few;
    }
  }

  sl_u64 left, ex;       // what is kept weighs, and before this thread's
  double target;
  int id = -1;
  float drawn = 0.f;
  if (n <= SL_CAP) {
    // ---- the list, in the order of the indices: wave, chunk, lane, entry
    const float x0 = sl_value(from);
    constexpr int NE = SlRow<T, NJ>::NE;
    int at = __builtin_amdgcn_readfirstlane((int)before);   // of lane 0: before the wave
    row.chunks_of([&](const float* v, int g) {
      int some = 0;
#pragma unroll
      for (int e = 0; e < NE; ++e) some += v[e] >= x0;
      if (!__any(some)) return;
      int sum = some;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int w = __shfl_up(sum, o, 64);
        if (lane >= o) sum += w;
      }
      int p = at + sum - some;
#pragma unroll
      for (int e = 0; e < NE; ++e)
        if (v[e] >= x0) {
          sh.x[p] = v[e];
          sh.idx[p] = row.index(g, e);
          ++p;
        }
      at += __builtin_amdgcn_readlane(sum, 63);
    });
    __syncthreads();
    const int per = ((int)n + SL_NT - 1) / SL_NT;   // of a thread, in a row
    SlFew<SL_CAP / SL_NT> list;
#pragma unroll
    for (int i = 0; i < SL_CAP / SL_NT; ++i) {
      const int j = tid * per + i;
      list.v[i] = i < per && j < (int)n ? sh.x[j] : -INFINITY;
    }
    if (!ranked) thr = max(thr, sl_select<false>(list, wt, from, kmax, (sl_u64)k, -1.0, false, sh));
    if (by_p) {
      sl_u64 want = 0;
      double part = share;
      if (total) {   // of the whole row, as sl_select forms it
        want = (sl_u64)ceil(share * (double)total);
        if (want == 0) want = 1;
        part = -1.0;
      }
      thr = max(thr, sl_select<true>(list, wt, max(thr, from), kmax, want, part, false, sh));
    }
    sl_u64 w[SL_CAP / SL_NT], sum = 0;
#pragma unroll
    for (int i = 0; i < SL_CAP / SL_NT; ++i) {
      w[i] = sl_key(list.v[i]) >= thr ? wt(list.v[i]) : 0;
      sum += w[i];
      __builtin_amdgcn_sched_barrier(0);
    }
    left = sl_scan(sum, ex, sh, 1);
    target = (double)u * (double)left;
    if (sum && (double)ex <= target && target < (double)(ex + sum)) {
#pragma unroll
      for (int i = 0; i < SL_CAP / SL_NT; ++i) {
        ex += w[i];
        if (w[i] && id < 0 && target < (double)ex) {
          id = sh.idx[tid * per + i];
          drawn = list.v[i];
        }
      }
    }
  } else {
    // ---- the row itself
    if (by_p) thr = max(thr, sl_select<true>(row, wt, thr, kmax, 0, share, false, sh));
    const float x0 = sl_value(thr);
    sl_u64 sum = 0;
    row.heavy([&](float x) { sum += x >= x0 ? wt(x) : 0; });
    left = sl_scan(sum, ex, sh, 1);
    target = (double)u * (double)left;
    // the wave whose entries' weight holds the target walks them again, from memory
    sl_u64 start = 0, end = 0;
#pragma unroll
    for (int w = 0; w < SL_NW; ++w) {
      if (w < wv) start += sh.part[1][w];
      if (w <= wv) end += sh.part[1][w];
    }
    if ((double)start <= target && target < (double)end) {
      constexpr int NE = SlRow<T, NJ>::NE;
#pragma unroll 1
      for (int j = 0; j < row.J; ++j) {
        float v[NE];
        row.values(row.load(row.g0 + j), row.g0 + j, v);
        sl_u64 w[NE], mass = 0;
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          w[e] = v[e] >= x0 ? wt(v[e]) : 0;
          mass += w[e];
          __builtin_amdgcn_sched_barrier(0);
        }
        sl_u64 in = mass;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const sl_u64 b = __shfl_up(in, o, 64);
          if (lane >= o) in += b;
        }
        const sl_u64 all = __shfl(in, 63, 64);
        if (target < (double)(start + all)) {
          sl_u64 run = start + in - mass;
          if (mass && (double)run <= target && target < (double)(run + mass)) {
#pragma unroll
            for (int e = 0; e < NE; ++e) {
              run += w[e];
              if (w[e] && id < 0 && target < (double)run) {
                id = row.index(row.g0 + j, e);
                drawn = v[e];
              }
            }
          }
          break;
        }
        start += all;
      }
    }
  }
  if (id >= 0) {   // one thread's
    a.r.ids[r] = id;
    if (a.r.logprob) {
      const double y = drawn == wt.m ? 0.0 : ((double)drawn - wt.md) / (double)temp;
      a.r.logprob[r] = (float)(y - log((double)left * ldexp(1.0, -a.frac)));
    }
  }
}

template <typename T, int NJ>
static hipError_t sl_launch(const SlArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((k_sample_logits<T, NJ>), dim3((unsigned)a.r.rows), dim3(SL_NT), sizeof(SlShared), st, a);
  return hipGetLastError();
}

hipError_t sample_logits(const LogitRows& r, int dtype, hipStream_t st) {
  if (r.rows == 0) return hipSuccess;
  SlArgs a{r, 62};
  while (a.frac > 0 && (1LL << (62 - a.frac)) < r.cols) --a.frac;
  if (a.frac > 51) a.frac = 51;
  // chunks a thread has: with up to 15 bytes before the row
  const int ne = dtype == 0 ? 4 : 8, J = ((r.cols + ne - 1 + ne - 1) / ne + SL_NT - 1) / SL_NT;
  if (dtype == 0) return J <= 2 ? sl_launch<float, 2>(a, st) : J <= 13 ? sl_launch<float, 13>(a, st) : sl_launch<float, 0>(a, st);
  return J <= 1 ? sl_launch<bf16_t, 1>(a, st) : J <= 7 ? sl_launch<bf16_t, 7>(a, st) : sl_launch<bf16_t, 0>(a, st);
}

}  // namespace ann
