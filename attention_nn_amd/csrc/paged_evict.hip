// Eviction from a paged key/value cache by the weight its entries have
// gathered.  A sequence of L > keep entries is left with its last `recent` and,
// of the others, the keep - recent of the largest weight (of equal ones the
// lower entry); a NaN weighs less than any number.  What stays keeps its order
// and moves to entries 0 .. keep - 1.
#include "common.h"
#include "launch.h"

namespace ann {

// Weights as words that compare like them: NaN lowest, -0 equal to +0.
__device__ __forceinline__ uint32_t ev_key(float f) {
  if (f != f) return 0;
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

// One work-group for each sequence.  The smallest weight that stays is found a
// byte at a time, from the top: a count of the words by their next byte among
// those that agree with the bytes found so far.  Then what stays is written down
// in entry order, its places from the counts of each wave's ballots.  Up to SEG
// entries lie in registers throughout; longer sequences are read again, SEG at a
// time, for each of the five walks.  Bound by the latency of its some twenty
// barriers on one CU a sequence, not by the weights' bytes: 1,500 entries to 1,024
// 7.2 us, 16 x 8192 to 4096 13.5 us (0.5 MB in, 1 MB out).  Four copies of the counts,
// to spread the atomics of like weights, gained nothing.
constexpr int EV_T = 1024, EV_W = EV_T / 64;

// Exclusive prefix sums of the n <= 256 counts in cnt, and their total, by the
// first wave.
__device__ __forceinline__ void ev_scan(int* cnt, int n, int* total) {
  const int lane = threadIdx.x & 63;
  if (threadIdx.x < 64) {
    int v[4], own = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = 4 * lane + k < n ? cnt[4 * lane + k] : 0;
      own += v[k];
    }
    int sum = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(sum, o, 64);
      if (lane >= o) sum += x;
    }
    int at = sum - own;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (4 * lane + k < n) cnt[4 * lane + k] = at;
      at += v[k];
    }
    if (lane == 63) *total = sum;
  }
}

template <int NPT>
__global__ __launch_bounds__(EV_T) void k_evict_pick(const int32_t* lens, int cols, int sh,
                                                     const float* w, long long wrow, int keep,
                                                     int recent, int32_t* __restrict__ index,
                                                     int32_t* new_lens, float* out, long long orow,
                                                     int cap) {
  constexpr int SEG = EV_T * NPT;
  static_assert(NPT * EV_W <= 256, "counts of a segment");
  __shared__ unsigned hist[256];
  __shared__ unsigned s_prefix, s_want;
  __shared__ int s_cnt[256], s_total;
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int len = pg_len(lens[s], cols, sh);
  const float* ws = w + s * wrow;
  float* os = out + s * orow;
  int32_t* ix = index + (long long)s * keep;
  const int left = min(len, keep);
  const int last = min(recent, left);   // entries that stay whatever they weigh
  const int old = len - last;           // those that are ranked
  const int want = left - last;         // and how many of them stay
  const int segs = (old + SEG - 1) / SEG;
  // weight and word of entry seg * SEG + k * EV_T + tid, bit k of here: it is ranked
  float x[NPT];
  uint32_t u[NPT], here;
  auto load = [&](int seg) {
    here = 0;
#pragma unroll
    for (int k = 0; k < NPT; ++k) {
      const int i = seg * SEG + k * EV_T + tid;
      x[k] = ws[min(i, old - 1)];
      here |= (unsigned)(i < old) << k;
    }
#pragma unroll
    for (int k = 0; k < NPT; ++k) u[k] = ev_key(x[k]);
  };
  if (segs == 1) load(0);
  uint32_t edge = 0;                    // smallest word that stays
  int ties = 0;                         // how many of the words equal to it do
  if (want < old && want > 0) {
    if (tid == 0) {
      s_prefix = 0;
      s_want = want;
    }
    for (int byte = 3; byte >= 0; --byte) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      const uint32_t prefix = s_prefix, mask = byte == 3 ? 0u : ~0u << (8 * byte + 8);
      for (int seg = 0; seg < segs; ++seg) {
        if (segs > 1) load(seg);
#pragma unroll
        for (int k = 0; k < NPT; ++k) {
          if ((here >> k) & 1 && (u[k] & mask) == prefix)
            atomicAdd(&hist[(u[k] >> (8 * byte)) & 255], 1u);
        }
      }
      __syncthreads();
      if (wv == 0) {   // the byte at which the words above it no longer fill `want`
        const unsigned need = s_want;
        // lane l holds bytes 4 l .. 4 l + 3
        const unsigned own = hist[4 * lane] + hist[4 * lane + 1] + hist[4 * lane + 2] + hist[4 * lane + 3];
        unsigned suffix = own;   // words of this lane's bytes and those above
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const unsigned v = __shfl_down(suffix, o, 64);
          if (lane + o < 64) suffix += v;
        }
        // highest lane that reaches it
        const int at = 63 - __builtin_clzll(__ballot(suffix >= need));
        if (lane == at) {
          unsigned above = suffix - own;
          int b = 4 * lane + 3;
          for (; above + hist[b] < need; --b) above += hist[b];
          s_prefix = prefix | ((uint32_t)b << (8 * byte));
          s_want = need - above;
        }
      }
      __syncthreads();
    }
    edge = s_prefix;
    ties = (int)s_want;
  }
  const bool all = want >= old;   // nothing is ranked out
  __syncthreads();
  if (tid == 0) new_lens[s] = left;   // may be lens[s]: every thread has read it
  const unsigned long long below = lane ? ~0ull >> (64 - lane) : 0ull;
  int done = 0, tied = 0;
  for (int seg = 0; seg < segs && want > 0; ++seg) {
    if (segs > 1) load(seg);
    const int waves = min(NPT, (old - seg * SEG + EV_T - 1) / EV_T) * EV_W;   // counts in use
    unsigned long long be[NPT];
    if (!all) {   // ranks among the words equal to the edge
#pragma unroll
      for (int k = 0; k < NPT; ++k) {
        be[k] = __ballot((here >> k) & 1 && u[k] == edge);
        if (lane == 0) s_cnt[k * EV_W + wv] = __popcll(be[k]);
      }
      __syncthreads();
      ev_scan(s_cnt, waves, &s_total);
      __syncthreads();
    }
    unsigned stays = 0;
#pragma unroll
    for (int k = 0; k < NPT; ++k) {
      const bool in = (here >> k) & 1 &&
                      (all || u[k] > edge ||
                       (u[k] == edge && tied + s_cnt[k * EV_W + wv] + __popcll(be[k] & below) < ties));
      stays |= (unsigned)in << k;
    }
    if (!all) tied += s_total;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NPT; ++k) {
      be[k] = __ballot((stays >> k) & 1);
      if (lane == 0) s_cnt[k * EV_W + wv] = __popcll(be[k]);
    }
    __syncthreads();
    ev_scan(s_cnt, waves, &s_total);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NPT; ++k)
      if ((stays >> k) & 1) {   // its place p <= its entry: entries of later walks are never written
        const int p = done + s_cnt[k * EV_W + wv] + __popcll(be[k] & below);
        ix[p] = seg * SEG + k * EV_T + tid;
        os[p] = x[k];
      }
    done += s_total;
    __syncthreads();
  }
  // the last entries, in order too: out may be w
  for (int i0 = 0; i0 < last; i0 += EV_T) {
    const int i = i0 + tid;
    const float v = i < last ? ws[old + i] : 0.f;
    __syncthreads();
    if (i < last) {
      ix[want + i] = old + i;
      os[want + i] = v;
    }
    __syncthreads();
  }
  for (int i = left + tid; i < keep; i += EV_T) ix[i] = -1;
  for (int i = left + tid; i < cap; i += EV_T) os[i] = 0.f;
}

// The rows that stay, moved: keys or values of one head, 8 NT / W entries at a
// time (W lanes of 16 bytes a row).  Into other pages each work-group takes one
// such tile.  Into the same pages (their ids agree in some place) a sequence's
// first work-group takes all of them, in order: read, wait for all, write.  Entry i
// comes from index[i] >= i, and the ones read later lie above all that are written
// before; those before the first that moves stay untouched (16 x 4096 entries that all
// stay: 8.7 us a call, 94 with them copied onto themselves).  Bound by memory: rows of
// 256 bytes from where they lie (16 sequences of 8192 to 4096 entries, 6 heads of 128: 85 us
// for 400 MB, 4.7 TB/s, into other pages and in place alike; stores by way of the caches
// took 37 us more, their lines being fetched before they are written).  Eight rows a
// lane are on their way together.
template <int DH, int NT>
__global__ __launch_bounds__(NT) void k_evict_move(PagedArgs c, const int32_t* __restrict__ out_table,
                                                   long long orow, int out_cols,
                                                   const int32_t* __restrict__ index,
                                                   const int32_t* __restrict__ new_lens, int keep) {
  constexpr int W = DH / 8, RP = NT / W, ROWS = 8 * RP;   // rows a load, rows a tile
  __shared__ long long s_from[2][ROWS], s_to[2][ROWS];
  const int s = blockIdx.z, tid = threadIdx.x;
  const int left = new_lens[s];
  int i0 = blockIdx.x * ROWS;
  if (i0 >= left) return;
  const int h = blockIdx.y % c.heads;
  const bool isv = (int)blockIdx.y >= c.heads;
  const long long page = isv ? c.vp : c.kp, slot = isv ? c.vs : c.ks;
  bf16_t* base = (isv ? c.v + h * c.vh : c.k + h * c.kh) + (tid % W) * 8;
  const int32_t* from = c.table + s * c.trow;
  const int32_t* to = out_table + s * orow;
  bool same = from == to;
  if (!same) {
    const int n = min(((left - 1) >> c.sh) + 1, c.cols);
    int any = 0;
    for (int i = tid; i < n; i += NT) any |= from[i] == to[i];
    same = __syncthreads_or(any);
  }
  if (same && blockIdx.x) return;
  if (from == to) {   // what has not moved is a prefix, index[i] - i never falling: NT looks at a time
    const int32_t* ix = index + (long long)s * keep;
    for (int n = left;;) {   // it ends among entries i0 .. i0 + n
      const int step = (n + NT - 1) / NT, at = tid * step;
      const int still = __syncthreads_count(at < n && ix[i0 + at] == i0 + at);
      if (step == 1 || still == 0) {
        i0 += still;
        break;
      }
      i0 += (still - 1) * step;
      n = min(step, n - (still - 1) * step);
    }
    if (i0 >= left) return;
  }
  const int end = same ? left : min(left, i0 + ROWS);
  // where rows i .. i + ROWS - 1 come from and go to, -1: nowhere
  auto places = [&](int i, int b) {
    for (int k = tid; k < ROWS; k += NT) {
      long long f = 0, t = -1;
      if (i + k < end) {
        const int e = index[(long long)s * keep + i + k];
        const int id = to[(i + k) >> c.sh];
        f = pg_read(from[e >> c.sh], c.pages) * page + pg_slot(e, c.sh, slot);
        if (pg_writable(id, c.pages)) t = id * page + pg_slot(i + k, c.sh, slot);
      }
      s_from[b][k] = f;
      s_to[b][k] = t;
    }
  };
  places(i0, 0);
  __syncthreads();
  for (int b = 0; i0 < end; i0 += ROWS, b ^= 1) {
    uint4 w[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) w[u] = *(const uint4*)(base + s_from[b][u * RP + tid / W]);
    if (i0 + ROWS < end) places(i0 + ROWS, b ^ 1);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // every read of the wave has returned
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const long long t = s_to[b][u * RP + tid / W];
      if (t >= 0) st_once(base + t, w[u]);
    }
    if (i0 + ROWS < end) __syncthreads();   // s_to[b] is read before the next places take it
  }
}

template <int DH, int NT>
static void evict_move(const PagedArgs& c, const int32_t* out_table, long long out_row, int out_cols,
                       const int32_t* index, const int32_t* new_lens, int keep, hipStream_t st) {
  constexpr int ROWS = 8 * NT / (DH / 8);
  const dim3 grid(NT == 1024 ? 1u : (unsigned)((keep + ROWS - 1) / ROWS), (unsigned)(2 * c.heads),
                  (unsigned)c.seqs);
  hipLaunchKernelGGL((k_evict_move<DH, NT>), grid, dim3(NT), 0, st, c, out_table, out_row, out_cols,
                     index, new_lens, keep);
}

hipError_t paged_evict(const PagedArgs& c, int Dh, const int32_t* out_table, long long out_row,
                       int out_cols, const float* w, long long wrow, int keep, int recent,
                       int32_t* index, int32_t* new_lens, float* out, long long orow,
                       hipStream_t st) {
  if (c.seqs == 0) return hipSuccess;
  if (Dh != 64 && Dh != 128) return hipErrorInvalidValue;
  const int cap = c.cols << c.sh;
#define ANN_EP(N)                                                                                \
  hipLaunchKernelGGL(k_evict_pick<N>, dim3(c.seqs), dim3(EV_T), 0, st, c.lens, c.cols, c.sh, w,  \
                     wrow, keep, recent, index, new_lens, out, orow, cap)
  if (cap <= 2 * EV_T) ANN_EP(2);
  else if (cap <= 8 * EV_T) ANN_EP(8);
  else ANN_EP(16);
#undef ANN_EP
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  // in place a sequence's tiles follow one another: one large work-group
#define ANN_EM(D, NT) evict_move<D, NT>(c, out_table, out_row, out_cols, index, new_lens, keep, st)
  if (out_table == c.table && (out_row == c.trow || c.seqs == 1)) {
    if (Dh == 64) ANN_EM(64, 1024); else ANN_EM(128, 1024);
  } else {
    if (Dh == 64) ANN_EM(64, 256); else ANN_EM(128, 256);
  }
#undef ANN_EM
  return hipGetLastError();
}

}  // namespace ann
