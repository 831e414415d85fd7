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
// A work-group of 16 waves has a row and a CU to itself: it holds up to 53248 fp32 or 57344
// bf16 entries in registers; longer rows are read from the caches in every pass.  Weights of
// 50257 entries cost a CU 11 us of its vector units, so entries that cannot be drawn go first: those below what
// min_p leaves, and below the k-th largest of the threads' maxima, under which
// the k-th largest of all does not lie.  What is left, if 8192 entries at most, is
// listed in LDS in the order of the indices, and thresholds and draw go over the
// list; 256 entries at most by one wave without a barrier.  top_p alone has no such
// bound: the weights of all entries, added up in bins, give one.  Else (flat rows,
// many equal values, no limits) the passes go over the row.
//
// 50257 entries: one row by top_k 50 10.9 us, of them 3 to read it; 64 rows, a setting each, 43.0,
// the longest by top_p alone: 14 for all weights into bins and 10 for those that stay, both bound by
// the CU's vector instructions (33 an entry), 10 for thresholds; 512 rows of bf16 by min_p 0.02 and
// top_p 0.9 38.9, two rounds of the CUs.  No faster: a threshold from 32-bit weights first, then
// one pass for all sums (42.4: 41 instructions an entry).
#include <math.h>
#include "common.h"
#include "launch.h"
#include "words.h"

namespace ann {

constexpr int SL_NT = 1024, SL_NW = SL_NT / 64;
constexpr int SL_BINS = 2048;
constexpr int SL_CAP = 8192;          // entries of the list
constexpr int SL_PER = SL_CAP / SL_NT;
constexpr int SL_WAVE = 256;          // entries of it that one wave goes over
constexpr int SL_PAIRS = 2;           // chunks that a thread reads again for others
constexpr int SL_RANK = 896;          // a k up to which the threads' largest entries bound it
typedef unsigned long long sl_u64;

struct SlShared {
  sl_u64 hist[SL_BINS];               // zero between two selections
  float2 list[SL_CAP];                // an entry and (its bits) its index
  uint32_t top[256];                  // of the threads' largest entries, by size
  sl_u64 part[2][SL_NW];
  uint32_t mm[3][SL_NW];
  int some[2][SL_NW];
  sl_u64 above[2];
  int at[2], low, bag[2];
  unsigned short hit[SL_NT];          // threads with an entry far up, and of each wave how many, and before it
  int hits[SL_NW], hits_before[SL_NW];
};

// Sum over the work-group, and (ex) over the threads before this one; one barrier.
// Calls take turns with `part` (which), and a barrier lies between two of one turn.
__device__ __forceinline__ sl_u64 sl_scan(sl_u64 v, sl_u64& ex, sl_u64* part) {
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const sl_u64 in = wave_scan(v);
  if (lane == 63) part[wv] = in;
  __syncthreads();
  const sl_u64 own = part[lane % SL_NW], sums = wave_scan(lane < SL_NW ? own : 0);
  ex = in - v + lane_of(sums - own, wv);
  return lane_of(sums, SL_NW - 1);
}

// The weights of a row, whole numbers of 2^-F.
struct SlWeight {
  double md, c, least;  // the largest entry, log2(e) / T, the least weight that counts
  double magic;         // 2^(52 - F): the last 52 bits of a sum with it are the other number's times 2^F
  float low;            // entries below have no weight (those above may have none either); a NaN has none
  double k[10], round;  // of the polynomial; 1.5 * 2^52: the last bits of a sum with it are the nearest integer
  __device__ __forceinline__ void open(float temp, float min_p, int frac) {
    c = fmax(1.4426950408889634 / (double)temp, 0x1p-1000);   // an infinite T: all alike
    least = fmin(fmax((double)min_p, 0x1p-40), 1.0);
    magic = ldexp(1.0, 52 - frac);
    // (2^f - 1) / f on [-1/2, 1/2], interpolated at the Chebyshev nodes: relative 2^-50 of 2^f
    const double q[10] = {0x1.e5e9f548e5725p-28, 0x1.b6571de2f2351p-24, 0x1.62bfe46117445p-20, 0x1.ffcb76789860fp-17,
                          0x1.4309130378460p-13, 0x1.5d87fe908f88ap-10, 0x1.3b2ab6fba385fp-7,  0x1.c6b08d7044119p-5,
                          0x1.ebfbdff82c590p-3,  0x1.62e42fefa39f7p-1};
#pragma unroll
    for (int i = 0; i < 10; ++i) {
      k[i] = q[i];
      if (i) asm volatile("" : "+s"(k[i]));   // scalar registers: else every use moves it to vector ones first
      else asm volatile("" : "+v"(k[i]));     // but for one of the first product's two
    }
    round = 0x1.8p52;
    asm volatile("" : "+s"(round));
  }
  // With reach = log2(least) / c less some: the bound `low` for a finite largest entry m.  No word
  // from there on is so far down that 2^n leaves the range below.
  __device__ __forceinline__ void bound(float m, double reach) {
    md = (double)m;
    const double at = (double)m + reach;
    low = fmaxf((float)(at - fabs(at) * 0x1p-22), -3.4028235e38f);
    if (!(low <= m)) low = m;
    // a few words, by which 2^-22 passes the bound
    for (int i = 0; i < 16 && low < m && ((double)low - md) * c < -60.0; ++i) low = word_value(word_of(low) + 1);
  }
  // Without a branch; additions and products only: the unit that converts and scales is slower.
  __device__ __forceinline__ sl_u64 operator()(float x) const {
    const double d = (double)x - md;
    const double t = fma(d, c, round), n = t - round, f = fma(d, c, -n);
    double q = k[0];
#pragma unroll
    for (int i = 1; i < 10; ++i) q = fma(q, f, k[i]);
    const double p = fma(q, f, 1.0);   // in [0.7, 1.42]: times 2^n, n >= -61, by its exponent
    const double w = __hiloint2double(__double2hiint(p) + (__double2loint(t) << 20), __double2loint(p));
    const sl_u64 bits = (sl_u64)__double_as_longlong(w + magic) & 0xfffffffffffffull;
    return x >= low && w >= least ? bits : 0;
  }
};

// A row as a work-group has it: chunk c, 16 bytes, is entries c NE - shift on; group g is
// chunks 64 g + lane, and wave w has groups w J .. w J + J - 1.  NJ > 0: J <= NJ, in registers;
// else it is read in every pass.  NaNs are as they are: no comparison takes one.
template <typename T, int NJ>
struct SlRow {
  static constexpr int NE = 16 / (int)sizeof(T);
  const unsigned char* base;   // 16-byte aligned
  int shift, n, chunks, J;
  int g0, lane;                // the wave's first group
  uint4 held[NJ ? NJ : 1];

  // Index of entry e of this lane's chunk of group g.
  __device__ __forceinline__ int index(int g, int e) const { return (g * 64 * NE + e - shift) + lane * NE; }
  // The first and last words may hold bytes of other rows, or before and behind the
  // tensor: within its allocation, which no aligned 16-byte word crosses the end of.
  // A chunk past the last one is that one.
  __device__ __forceinline__ uint4 chunk(int c) const {
    return *(const uint4*)(base + min((uint32_t)c, (uint32_t)chunks - 1) * 16u);
  }
  __device__ __forceinline__ uint4 load(int g) const { return chunk(g * 64 + lane); }
  __device__ __forceinline__ static void unpack(const uint4& w, float* v) {
    if constexpr (sizeof(T) == 4) {
      v[0] = __uint_as_float(w.x);
      v[1] = __uint_as_float(w.y);
      v[2] = __uint_as_float(w.z);
      v[3] = __uint_as_float(w.w);
    } else {
      unpack8(w, v);
    }
  }
  // What of a chunk lies outside the row is -inf.
  __device__ __forceinline__ uint4 inside(const uint4& w, int g) const {
    if (g != 0 && (g + 1) * 64 < chunks) return w;   // the same for the wave
    const int i = index(g, 0);
    uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < NE; ++e)
      if ((unsigned)(i + e) >= (unsigned)n) {
        if constexpr (sizeof(T) == 4) d[e] = 0xff800000u;
        else d[e / 2] = e % 2 ? (d[e / 2] & 0xffffu) | 0xff800000u : (d[e / 2] & 0xffff0000u) | 0xff80u;
      }
    return make_uint4(d[0], d[1], d[2], d[3]);
  }
  __device__ __forceinline__ void open(const T* row, int cols) {
    const int over = (int)((uintptr_t)row & 15);
    base = (const unsigned char*)row - over;
    shift = over / (int)sizeof(T);
    n = cols;
    chunks = (cols + shift + NE - 1) / NE;
    J = (chunks + SL_NT - 1) / SL_NT;
    g0 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * J;
    lane = threadIdx.x & 63;
    if constexpr (NJ > 0) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) held[j] = load(g0 + min(j, J - 1));
    }
  }
  // What open has sent for has arrived.
  __device__ __forceinline__ void arrived() {
    if constexpr (NJ > 0) {
#pragma unroll
      for (int j = 0; j < NJ; ++j)   // a group past the wave's last is all outside
        held[j] = j < J ? inside(held[j], g0 + j)
                        : sizeof(T) == 4 ? make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u)
                                         : make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
    }
  }
  // f(values, group) for each group of the wave.
  template <typename F>
  __device__ __forceinline__ void groups(F&& f) const {
    if constexpr (NJ > 0) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        // a copy that the compiler knows nothing of: it would keep what it forms of all of
        // them from one pass to the next
        uint4 w = held[j];
        asm volatile("" : "+v"(w.x), "+v"(w.y), "+v"(w.z), "+v"(w.w));
        float v[NE];
        unpack(w, v);
        f(v, g0 + j);
      }
    } else {
      constexpr int D = 4;   // loads at once
#pragma unroll 1
      for (int j0 = 0; j0 < J; j0 += D) {
        uint4 w[D];
#pragma unroll
        for (int d = 0; d < D; ++d) w[d] = load(g0 + min(j0 + d, J - 1));
#pragma unroll
        for (int d = 0; d < D; ++d)
          if (j0 + d < J) {
            float v[NE];
            unpack(inside(w[d], g0 + j0 + d), v);
            f(v, g0 + j0 + d);
          }
      }
    }
  }
  // f(values, group) for the groups of which in(values) holds for a lane.
  template <typename I, typename F>
  __device__ __forceinline__ void groups_with(I&& in, F&& f) const {
    if constexpr (NJ > 0) {   // all asked first: a branch on a vector's result waits for it
      uint32_t hit = 0;
      groups([&](const float* v, int g) { hit |= in(v) ? 1u << (g - g0) : 0; });
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) hit |= __shfl_xor(hit, o, 64);
      hit = __builtin_amdgcn_readfirstlane(hit);
      groups([&](const float* v, int g) {
        if (hit >> (g - g0) & 1) f(v, g);
      });
    } else {
      groups([&](const float* v, int g) {
        if (__any(in(v))) f(v, g);
      });
    }
  }
  // f(number, -) of each entry, two at a time: of long ones' temporaries
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
    groups([&](const float* v, int) {
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        f(v[e], 0);
        if (e % 2) __builtin_amdgcn_sched_barrier(0);
      }
    });
  }
};

// Up to N entries a thread, and their weights.
template <int N>
struct SlFew {
  float v[N];
  sl_u64 w[N];
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
#pragma unroll
    for (int i = 0; i < N; ++i) f(v[i], w[i]);
  }
};

// A threshold on its way: the largest word t of [lo, hi] such that the entries with words from t
// on count, or weigh, `want` at least; `above` of them lie above hi.
struct SlPart {
  uint32_t lo, hi;
  sl_u64 above, want;
  int turn;          // of the shared results
};

// What a round's bins hold: the one of them in which t lies (-1: none does, there are not
// `want`), p.above with what lies above it.  share >= 0: want is that share of all.
template <bool MASS>
__device__ __forceinline__ int sl_bin(SlPart& p, double share, SlShared& sh) {
  constexpr int PER = SL_BINS / SL_NT;
  const int tid = threadIdx.x, turn = p.turn ^= 1;
  if (tid == 0) sh.at[turn] = -1;
  __syncthreads();
  sl_u64 v[PER], sum = 0, ex;
#pragma unroll
  for (int i = 0; i < PER; ++i) {   // from the upper end down
    sl_u64* bin = &sh.hist[SL_BINS - 1 - PER * tid - i];
    sum += v[i] = *bin;
    *bin = 0;
  }
  const sl_u64 all = sl_scan(sum, ex, sh.part[turn]);
  if (MASS && share >= 0.0) {
    p.want = (sl_u64)ceil(share * (double)all);
    if (p.want == 0) p.want = 1;
    if (p.want > all) p.want = all;
  }
  ex += p.above;
  if (ex < p.want && p.want <= ex + sum) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (p.want <= ex + v[i]) {
        sh.at[turn] = SL_BINS - 1 - PER * tid - i;
        sh.above[turn] = ex;
        break;
      }
      ex += v[i];
    }
  }
  __syncthreads();
  p.above = sh.above[turn];
  return sh.at[turn];
}
// An entry's weight: formed here of a row's, at hand of a list's.
__device__ __forceinline__ sl_u64 sl_mass(const SlWeight& wt, float x, int) { return wt(x); }
__device__ __forceinline__ sl_u64 sl_mass(const SlWeight&, float, sl_u64 w) { return w; }
// To a bin where `in`; the weight is formed first, by all lanes.
template <bool MASS, typename W>
__device__ __forceinline__ void sl_add(const SlWeight& wt, float x, W w, bool in, int bin, SlShared& sh) {
  if constexpr (MASS) {
    const sl_u64 mass = sl_mass(wt, x, w);
    if (in && mass) atomicAdd(&sh.hist[bin], mass);
  } else {
    if (in) atomicAdd((unsigned*)&sh.hist[bin], 1u);
  }
}
// One round: [lo, hi] becomes the one of up to 2048 equal parts of it that holds t; false
// where none does.
template <bool MASS, typename S>
__device__ __forceinline__ bool sl_round(const S& src, const SlWeight& wt, SlPart& p, double share, SlShared& sh) {
  static_assert(SL_BINS == 2048, "parts of a range");
  const WordRange in = {p.lo, p.hi};
  const int s = in.shift();
  src.each([&](float x, auto w) {
    int bin;
    const bool inside = in.has(x, s, bin);
    sl_add<MASS>(wt, x, w, inside, bin, sh);
  });
  const int at = sl_bin<MASS>(p, share, sh);
  if (at < 0) return false;
  const WordRange to = in.part(at, s);
  p.lo = to.lo;
  p.hi = to.hi;
  return true;
}
// The first round over a whole row, whose largest entry is p.hi's: parts of equal difference
// instead, since half of all words are numbers below 1.  `floor`: about the least entry
// (what lies below goes to the lowest part).
template <bool MASS, typename S>
__device__ __forceinline__ bool sl_first(const S& src, const SlWeight& wt, SlPart& p, double share, float floor,
                                         SlShared& sh) {
  const float m = word_value(p.hi), least = fmaxf(word_value(p.lo), floor), c = SL_BINS / (m - least);
  if (!(c > 0.f && c < 1e30f)) return sl_round<MASS>(src, wt, p, share, sh);   // not finite, or one value
  const uint32_t lo = p.lo;
  const auto bin = [&](float x) { return SL_BINS - 1 - (int)fminf((m - x) * c, SL_BINS - 1.f); };   // rises with x
  const float x0 = word_value(lo);
  src.each([&](float x, auto w) {
    sl_add<MASS>(wt, x, w, x >= x0, bin(x), sh);
  });
  const int at = sl_bin<MASS>(p, share, sh);
  if (at < 0) return false;
  // the least words of that part and of the next, by 64 lanes at a time
  const int lane = threadIdx.x & 63;
  const auto least_in = [&](int b) {
    uint32_t a = lo, n = p.hi - lo + 1;   // it is one of the n words from a on, or the next
    while (n) {
      const uint32_t step = n / 64 + 1, at = lane * step;
      const unsigned long long in = __ballot(at < n && bin(word_value(a + at)) >= b);
      // the first lane that has reached the part; or all n words lie below
      const uint32_t first = in ? (uint32_t)__builtin_ctzll(in) : (n + step - 1) / step;
      if (first == 0) return a;
      const uint32_t past = (first - 1) * step + 1;   // the word behind the last one below
      a += past;
      n = in ? step - 1 : n - past;
    }
    return a;
  };
  const uint32_t a = least_in(at), b = least_in(at + 1);
  p.lo = a;
  p.hi = b - 1;
  return true;
}
// All rounds: the word, or lo where there are not `want`; where words no more than `grain`
// apart are one number, any of those.
template <bool MASS, typename S>
__device__ __forceinline__ uint32_t sl_select(const S& src, const SlWeight& wt, SlPart& p, double share, uint32_t grain, SlShared& sh) {
  const uint32_t none = p.lo;
  while (p.hi - p.lo > grain || share >= 0.0) {
    if (!sl_round<MASS>(src, wt, p, share, sh)) return none;
    share = -1.0;
  }
  return p.lo;
}

struct SlArgs {
  LogitRows r;
  int frac;   // F
};

template <typename T, int NJ>
__global__ __launch_bounds__(SL_NT, 4) void k_sample_logits(SlArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char sl_smem[];
  SlShared& sh = *(SlShared*)sl_smem;
  constexpr int NE = SlRow<T, NJ>::NE;
  constexpr uint32_t GRAIN = sizeof(T) == 4 ? 0 : 0xffff;   // words of bf16 lie 2^16 apart
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = blockIdx.x, V = a.r.cols;
  SlRow<T, NJ> row;
  row.open((const T*)a.r.x + r * a.r.stride, V);
  float u = a.r.u[r];
  const float temp = a.r.temperature ? a.r.temperature[r] : a.r.temperature_all;
  const int k = a.r.top_k ? a.r.top_k[r] : a.r.top_k_all;
  const float top_p = a.r.top_p ? a.r.top_p[r] : a.r.top_p_all;
  const float min_p = a.r.min_p ? a.r.min_p[r] : a.r.min_p_all;
  const bool by_k = k > 0 && k < V, by_p = top_p < 1.f;
#pragma unroll
  for (int b = 0; b < SL_BINS; b += SL_NT) sh.hist[b + tid] = 0;
  if (tid < 256) sh.top[tid] = 0;
  if (tid == 0) sh.low = 0x7fffffff;
  if (tid < 2) sh.bag[tid] = 0;

  SlWeight wt;
  wt.open(temp, min_p, a.frac);
  const double reach = (log2(wt.least) - 1e-3) / wt.c;   // while the row is on its way
  row.arrived();

  // ---- the largest entry, the least of the threads' largest, and the least of some entries
  float most = -INFINITY, few = INFINITY;
  row.groups([&](const float* v, int g) {
#pragma unroll
    for (int e = 0; e < NE; ++e) most = fmaxf(most, v[e]);
    if (g == row.g0)
#pragma unroll
      for (int e = 0; e < NE; ++e) few = fminf(few, v[e] > -INFINITY ? v[e] : INFINITY);
  });
  most += 0.f;   // 0 for -0
  const uint32_t key = word_of(most);
  {
    const uint32_t top = wave_max(key), low = wave_min(word_of(few + 0.f));
    const uint32_t least = wave_min(most > -INFINITY ? key : 0xffffffffu);
    if (lane == 0) {
      sh.mm[0][wv] = top;
      sh.mm[1][wv] = least;
      sh.mm[2][wv] = low;
    }
  }
  __syncthreads();
  const uint32_t kmax = wave_max(sh.mm[0][lane % SL_NW]);
  const float m = word_value(kmax);
  if (m == -INFINITY) {   // nothing to draw
    if (tid == 0) {
      a.r.ids[r] = -1;
      if (a.r.logprob) a.r.logprob[r] = -INFINITY;
    }
    return;
  }
  if (!(temp > 0.f)) {   // the lowest index of the largest
    int at = 0x7fffffff;
    if (most == m)
      row.groups([&](const float* v, int g) {
#pragma unroll
        for (int e = 0; e < NE; ++e)
          if (v[e] == m) at = min(at, row.index(g, e));
      });
    if (at != 0x7fffffff) atomicMin(&sh.low, at);
    __syncthreads();
    if (tid == 0) {
      a.r.ids[r] = sh.low;
      if (a.r.logprob) a.r.logprob[r] = 0.f;
    }
    return;
  }
  u = u >= 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;

  // Entries from a word on, and those of the waves before this one.
  int before = 0, turn = 0;
  const auto count = [&](uint32_t from) {
    const float x0 = word_value(from);
    uint32_t some = 0;
    row.groups([&](const float* v, int) {
#pragma unroll
      for (int e = 0; e < NE; ++e) some += v[e] >= x0;
    });
    const uint32_t all = lane_of(wave_scan(some), 63);
    turn ^= 1;
    if (lane == 0) sh.some[turn][wv] = (int)all;
    __syncthreads();
    const uint32_t own = (uint32_t)sh.some[turn][lane % SL_NW], in = wave_scan(lane < SL_NW ? own : 0);
    before = (int)lane_of(in - own, wv);
    return (int)lane_of(in, SL_NW - 1);
  };
  if (m == INFINITY) {   // the infinite entries weigh 1, all others nothing
    const int n = count(kmax), pick = (int)((double)u * n);
    int at = before;
    row.groups([&](const float* v, int g) {
      int p = at;   // behind the lower lanes' entries
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const unsigned long long in = __ballot(v[e] == m);
        p = __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, p));
        at += __popcll(in);
      }
#pragma unroll
      for (int e = 0; e < NE; ++e)
        if (v[e] == m && p++ == pick) {
          a.r.ids[r] = row.index(g, e);
          if (a.r.logprob) a.r.logprob[r] = (float)-log((double)n);
        }
    });
    return;
  }
  const uint32_t tmin = wave_min(sh.mm[1][lane % SL_NW]);
  const float floor = word_value(wave_min(sh.mm[2][lane % SL_NW]));

  // The threads' largest entries in 256 bins: k of them are at or above the lower end of the
  // bin that the k-th lies in, so the k-th largest of all is.
  uint32_t kth = 0;
  if (by_k && k <= SL_RANK && V > SL_CAP && kmax > tmin) {
    const int bits = 32 - __clz((int)(kmax - tmin)), s = bits > 8 ? bits - 8 : 0;
    if (key >= tmin) atomicAdd(&sh.top[(key - tmin) >> s], 1u);
    __syncthreads();
    const uint4 c = *(const uint4*)&sh.top[252 - 4 * lane];   // from the upper end down: w, z, y, x
    const uint32_t sum = c.x + c.y + c.z + c.w, in = wave_scan(sum), want = (uint32_t)k;
    const unsigned long long past = __ballot(in >= want);
    if (past) {
      const int at = __builtin_ctzll(past);
      uint32_t n = in - sum + c.w;
      int b = 255 - 4 * lane;
      if (n < want) n += c.z, --b;
      if (n < want) n += c.y, --b;
      if (n < want) --b;
      kth = tmin + (lane_of((uint32_t)b, at) << s);
    }
  }

  wt.bound(m, reach);
  const double share = by_p ? fmax((double)top_p, 0.0) : 1.0;
  uint32_t thr = max(word_of(wt.low), kth);   // the least word that is kept so far
  bool ranked = !by_k;                       // thr is the k-th largest, if there are as many
  SlPart sp{thr, kmax, 0, (sl_u64)k, 0};   // its turns are not those of count

  // The list of all from a word on, where few threads have an entry that far up: the chunks of
  // those, in the order of the indices (wave, group, lane), are shared out among all and
  // read again.  Its number, or -1 where they are too many.
  const auto few_of = [&](uint32_t from) {
    const float x0 = word_value(from);
    const unsigned long long mine = __ballot(most >= x0);
    if (lane == 0) sh.hits[wv] = __popcll(mine);
    __syncthreads();
    const uint32_t own = (uint32_t)sh.hits[lane % SL_NW], in = wave_scan(lane < SL_NW ? own : 0);
    const int hits = (int)lane_of(in, SL_NW - 1), pairs = hits * row.J;   // a hit for each thread at most
    if (pairs > SL_PAIRS * SL_NT) return -1;
    if (wv == 0 && lane < SL_NW) sh.hits_before[lane] = (int)(in - own);
    // by all lanes: inside the branch the lane that is asked may be off, and what it holds of
    // in - own not yet formed
    const uint32_t place = lane_of(in - own, wv) + __popcll(mine & ((1ull << lane) - 1));
    if (most >= x0) sh.hit[place] = (unsigned short)tid;
    __syncthreads();
    float v[SL_PAIRS][NE];
    int first[SL_PAIRS], some = 0;
    const int per = (pairs + SL_NT - 1) / SL_NT;
#pragma unroll
    for (int i = 0; i < SL_PAIRS; ++i) {
      const int pair = tid * per + i;
      const bool real = i < per && pair < pairs;
      // of the pairs of a wave's h hits the ones with group j are h in a row
      const int w = sh.hit[real ? pair / row.J : 0] >> 6, h = sh.hits[w], b = sh.hits_before[w];
      const int q = (real ? pair : b * row.J) - b * row.J, j = q / h, c = (w * row.J + j) * 64 + (sh.hit[b + q - j * h] & 63);
      first[i] = c * NE - row.shift;
      row.unpack(row.chunk(c), v[i]);
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        if (!real || (unsigned)(first[i] + e) >= (unsigned)V) v[i][e] = -INFINITY;
        some += v[i][e] >= x0;
      }
    }
    sl_u64 ex;
    sp.turn ^= 1;
    const int n = (int)sl_scan((sl_u64)some, ex, sh.part[sp.turn]);
    if (n > SL_CAP) return -1;
    int p = (int)ex;
#pragma unroll
    for (int i = 0; i < SL_PAIRS; ++i)
#pragma unroll
      for (int e = 0; e < NE; ++e)
        if (v[i][e] >= x0) {
          sh.list[p] = make_float2(v[i][e] + 0.f, __int_as_float(first[i] + e));
          ++p;
        }
    __syncthreads();
    return n;
  };
  // The entries with words of [from, to] in any order, without their indices: their number.
  const auto bag_of = [&](uint32_t from, uint32_t to) {
    const float x0 = word_value(from), x1 = word_most(to);
    turn ^= 1;
    if (tid == 0) sh.bag[turn ^ 1] = 0;
    // first the groups that may have one: within half the range of its middle and some more
    const float mid = 0.5f * x0 + 0.5f * x1, reach = (x1 - x0) * 0.5000002f + (fabsf(x0) + fabsf(x1)) * 1e-6f;
    const auto near = [&](const float* v) {
      float d = fabsf(v[0] - mid);
#pragma unroll
      for (int e = 1; e < NE; ++e) d = fminf(d, fabsf(v[e] - mid));
      return d <= reach;
    };
    const auto take = [&](const float* v) {
      int some = 0;
#pragma unroll
      for (int e = 0; e < NE; ++e) some += v[e] >= x0 && v[e] <= x1;
      if (some) {
        int p = atomicAdd(&sh.bag[turn], some);
#pragma unroll
        for (int e = 0; e < NE; ++e)
          if (v[e] >= x0 && v[e] <= x1) {
            if (p < SL_CAP) sh.list[p].x = v[e] + 0.f;
            ++p;
          }
      }
    };
    row.groups_with(near, [&](const float* v, int) { take(v); });
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(sh.bag[turn]);
  };

  uint32_t from = thr;                   // the list's least word
  int n = few_of(from);
  bool listed = n >= 0;
  if (!listed) n = count(from);
  double part = by_p ? share : -1.0;     // of the mass, while that is not known
  if (n > SL_CAP && by_k) {
    // many equal values, or many to keep: the k-th largest itself
    if (sl_first<false>(row, wt, sp, -1.0, floor, sh)) thr = max(thr, sl_select<false>(row, wt, sp, -1.0, GRAIN, sh));
    ranked = true;
    from = thr;
    n = count(from);
  }
  bool rest = n > SL_CAP;                // not all that is kept is listed
  if (rest && by_p) {
    // all weights in bins; then few threads have what is kept, or what one bin holds is listed
    sp = SlPart{thr, kmax, 0, 0, sp.turn};
    sl_first<true>(row, wt, sp, share, floor, sh);
    part = -1.0;
    from = sp.lo;
    n = few_of(from);
    listed = true;
    rest = n < 0;
    if (rest) {
      // none where one word is left.  Every round leaves a smaller range, or none and ends this.
      n = 0;
      while (sp.hi - sp.lo > GRAIN && (n = bag_of(sp.lo, sp.hi)) > SL_CAP && sl_round<true>(row, wt, sp, -1.0, sh)) {}
      if (sp.hi - sp.lo <= GRAIN || n > SL_CAP) n = 0;
    }
  } else if (rest) {
    n = 0;
  } else {
    sp = SlPart{thr, kmax, 0, 0, sp.turn};
  }

  // ---- the list, in the order of the indices: wave, group, lane, entry
  if (n && !listed) {
    const float x0 = word_value(from);
    int at = before;
    const auto write = [&](const float* v, int g) {
      unsigned long long in[NE];
      int p = at;   // behind the lower lanes' entries
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        in[e] = __ballot(v[e] >= x0);
        p = __builtin_amdgcn_mbcnt_hi((uint32_t)(in[e] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in[e], p));
        at += __popcll(in[e]);
      }
#pragma unroll
      for (int e = 0; e < NE; ++e)
        if (v[e] >= x0) {
          sh.list[p] = make_float2(v[e] + 0.f, __int_as_float(row.index(g, e)));
          ++p;
        }
    };
    // not asked first which groups have one: nearly all do (512 rows of bf16 41.2 -> 38.6 us)
    row.groups(write);
    __syncthreads();
  }

  sl_u64 left;           // weight of all that is kept
  int id = -1;
  float drawn = 0.f;
  if (!rest && n <= SL_WAVE) {
    // ---- one wave, thresholds by bisection
    if (wv) return;
    constexpr int N = SL_WAVE / 64;
    const int per = (n + 63) / 64;   // entries of a lane, in a row
    float x[N];
    uint32_t keys[N];
    sl_u64 w[N], sum = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int j = lane * per + i;
      const bool real = i < per && j < n;
      x[i] = real ? sh.list[j].x : -INFINITY;
      keys[i] = real ? word_of(x[i]) : 0;
    }
    if (!ranked && n >= k && per == 1) {   // an entry's rank by the others, one by one
      uint32_t rank = 0;
#pragma unroll 4
      for (int i = 0; i < n; ++i) rank += lane_of(keys[0], i) > keys[0];
      thr = max(thr, wave_min(lane < n && rank < (uint32_t)k ? keys[0] : 0xffffffffu));
    } else if (!ranked && n >= k) {   // else all of them are among the k
      uint32_t lo = from, hi = kmax;
      while (hi - lo > GRAIN) {
        const uint32_t mid = hi - ((hi - lo) >> 1);
        int c = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) c += __popcll(__ballot(keys[i] >= mid));
        if (c >= k) lo = mid;
        else hi = mid - 1;
      }
      thr = max(thr, lo);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      w[i] = keys[i] >= thr ? wt(x[i]) : 0;
      sum += w[i];
    }
    if (by_p) {
      sl_u64 want = sp.want;
      if (part >= 0.0) {
        want = (sl_u64)ceil(part * (double)lane_of(wave_scan(sum), 63));
        if (want == 0) want = 1;
      }
      uint32_t lo = thr, hi = kmax;
      if (per == 1) {   // what lies above an entry weighs
        sl_u64 above = 0;
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
          const sl_u64 wi = lane_of(w[0], i);
          above += lane_of(keys[0], i) > keys[0] ? wi : 0;
        }
        lo = hi = wave_min(w[0] && above < want ? keys[0] : 0xffffffffu);
      }
      while (hi - lo > GRAIN) {
        const uint32_t mid = hi - ((hi - lo) >> 1);
        sl_u64 c = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) c += keys[i] >= mid ? w[i] : 0;
        if (lane_of(wave_scan(c), 63) >= want) lo = mid;
        else hi = mid - 1;
      }
      sum = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (keys[i] < lo) w[i] = 0;
        sum += w[i];
      }
    }
    const sl_u64 in = wave_scan(sum);
    left = lane_of(in, 63);
    const double target = (double)u * (double)left;
    sl_u64 run = in - sum;
    if (sum && (double)run <= target && target < (double)in) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        run += w[i];
        if (w[i] && id < 0 && target < (double)run) {
          id = __float_as_int(sh.list[lane * per + i].y);
          drawn = x[i];
        }
      }
    }
  } else {
    if (n) {
      const int per = (n + SL_NT - 1) / SL_NT;   // of a thread, in a row
      SlFew<SL_PER> list;
#pragma unroll
      for (int i = 0; i < SL_PER; ++i) {
        const int j = tid * per + i;
        list.v[i] = i < per && j < n ? sh.list[j].x : -INFINITY;
        list.w[i] = i < per ? wt(list.v[i]) : 0;
        __builtin_amdgcn_sched_barrier(0);
      }
      if (!ranked) {
        SlPart q{from, kmax, 0, (sl_u64)k, sp.turn};
        thr = max(thr, sl_select<false>(list, wt, q, -1.0, GRAIN, sh));
        sp.turn = q.turn;
        sp.lo = max(sp.lo, thr);
      }
      if (by_p) thr = max(thr, sl_select<true>(list, wt, sp, part, GRAIN, sh));
      if (!rest) {
        // ---- the draw from the list
        sl_u64 sum = 0, ex;
#pragma unroll
        for (int i = 0; i < SL_PER; ++i) {
          if (word_of(list.v[i]) < thr) list.w[i] = 0;
          sum += list.w[i];
        }
        sp.turn ^= 1;
        left = sl_scan(sum, ex, sh.part[sp.turn]);
        const double target = (double)u * (double)left;
        if (sum && (double)ex <= target && target < (double)(ex + sum)) {
#pragma unroll
          for (int i = 0; i < SL_PER; ++i) {
            ex += list.w[i];
            if (list.w[i] && id < 0 && target < (double)ex) {
              id = __float_as_int(sh.list[tid * per + i].y);
              drawn = list.v[i];
            }
          }
        }
      }
    } else if (by_p) {
      thr = max(thr, sp.lo);
    }
    if (rest) {
      // ---- the draw from the row: the wave whose weight holds the target, by all waves its
      // groups, by the wave whose groups hold it the group, lane and entry
      const float x0 = word_value(thr);
      sl_u64 sum = 0;
      row.each([&](float x, int) {
        const sl_u64 w = wt(x);
        sum += x >= x0 ? w : 0;
      });
      sl_u64 ex;
      sp.turn ^= 1;
      left = sl_scan(sum, ex, sh.part[sp.turn]);
      const double target = (double)u * (double)left;
      const sl_u64 own = sh.part[sp.turn][lane % SL_NW], in = wave_scan(lane < SL_NW ? own : 0);
      const int at = __builtin_ctzll(__ballot(target < (double)in));   // target < left
      sl_u64 start = lane_of(in - own, at);
      const int per = (row.J + SL_NW - 1) / SL_NW, first = at * row.J;
      const int ga = first + min(wv * per, row.J), gb = first + min(wv * per + per, row.J);
      float v[NE];
      sl_u64 w[NE];
      const auto group = [&](int g) {
        SlRow<T, NJ>::unpack(row.inside(row.load(g), g), v);
        sl_u64 sum = 0;
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          w[e] = wt(v[e]);
          w[e] = v[e] >= x0 ? w[e] : 0;
          sum += w[e];
          if (e % 2) __builtin_amdgcn_sched_barrier(0);
        }
        return sum;
      };
      sl_u64 mass = 0;
#pragma unroll 1
      for (int g = ga; g < gb; ++g) mass += group(g);
      sp.turn ^= 1;
      sl_scan(mass, ex, sh.part[sp.turn]);
      for (int i = 0; i < wv; ++i) start += sh.part[sp.turn][i];
      if ((double)start <= target && target < (double)(start + sh.part[sp.turn][wv])) {
#pragma unroll 1
        for (int g = ga; g < gb; ++g) {
          if (gb - ga > 1) mass = group(g);
          const sl_u64 in = wave_scan(mass), all = lane_of(in, 63);
          if (target < (double)(start + all)) {
            sl_u64 run = start + in - mass;
            if (mass && (double)run <= target && target < (double)(run + mass)) {
#pragma unroll
              for (int e = 0; e < NE; ++e) {
                run += w[e];
                if (w[e] && id < 0 && target < (double)run) {
                  id = row.index(g, e);
                  drawn = v[e] + 0.f;
                }
              }
            }
            break;
          }
          start += all;
        }
      }
    }
  }
  if (id >= 0) {   // one thread's
    a.r.ids[r] = id;
    if (a.r.logprob) {
      const double y = drawn == m ? 0.0 : ((double)drawn - wt.md) / (double)temp;
      a.r.logprob[r] = (float)(y - log((double)left * ldexp(1.0, -a.frac)));
    }
  }
}

template <typename T, int NJ>
static hipError_t sl_launch(const SlArgs& a, hipStream_t st) {
  static PerDevice limit;
  const hipError_t e = lds_limit(limit, (const void*)k_sample_logits<T, NJ>, sizeof(SlShared));
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((k_sample_logits<T, NJ>), dim3((unsigned)a.r.rows), dim3(SL_NT), sizeof(SlShared), st, a);
  return hipGetLastError();
}

// Up to SL_ROWS rows: a launch holds less than 2^32 threads.
constexpr int SL_ROWS = 1 << 21;
static hipError_t sl_rows(const LogitRows& r, int dtype, hipStream_t st) {
  SlArgs a{r, 62};
  while (a.frac > 0 && (1LL << (62 - a.frac)) < r.cols) --a.frac;
  if (a.frac > 51) a.frac = 51;
  // groups a wave has, of rows that begin up to 15 bytes behind a chunk's begin
  const int ne = dtype == 0 ? 4 : 8, J = ((r.cols + 2 * ne - 2) / ne + SL_NT - 1) / SL_NT;
  // Every pass goes over NJ groups, full or not: 64 rows by top_p alone, of 12000 fp32 in 13 groups 40.2
  // us, in 4 23.5, of 32000 bf16 in 7 36.8, in 4 26.6.  (Left out by a branch on J: 24.7 and 27.1, but
  // 44.9 for 43.3 where all 13 are full.)
  if (dtype == 0)
    return J <= 2 ? sl_launch<float, 2>(a, st) : J <= 4 ? sl_launch<float, 4>(a, st) : J <= 8 ? sl_launch<float, 8>(a, st)
                  : J <= 13 ? sl_launch<float, 13>(a, st) : sl_launch<float, 0>(a, st);
  return J <= 1 ? sl_launch<bf16_t, 1>(a, st) : J <= 2 ? sl_launch<bf16_t, 2>(a, st) : J <= 4 ? sl_launch<bf16_t, 4>(a, st)
                : J <= 7 ? sl_launch<bf16_t, 7>(a, st) : sl_launch<bf16_t, 0>(a, st);
}

hipError_t sample_logits(const LogitRows& r, int dtype, hipStream_t st) {
  for (int r0 = 0; r0 < r.rows; r0 += min(SL_ROWS, r.rows - r0)) {
    LogitRows p = r;
    p.rows = min(SL_ROWS, r.rows - r0);
    p.x = (const char*)r.x + r0 * r.stride * (dtype == 0 ? 4 : 2);
    p.u += r0;
    if (p.temperature) p.temperature += r0;
    if (p.top_k) p.top_k += r0;
    if (p.top_p) p.top_p += r0;
    if (p.min_p) p.min_p += r0;
    p.ids += r0;
    if (p.logprob) p.logprob += r0;
    const hipError_t e = sl_rows(p, dtype, st);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace ann
