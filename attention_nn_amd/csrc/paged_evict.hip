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
// those that agree with the bytes found so far.  Then one walk in entry order
// writes down what stays.
constexpr int EV_T = 1024;
__global__ __launch_bounds__(EV_T) void k_evict_pick(const int32_t* __restrict__ lens, int cols,
                                                     int sh, const float* w, long long wrow,
                                                     int keep, int recent, int32_t* __restrict__ index,
                                                     int32_t* __restrict__ new_lens, float* out,
                                                     long long orow, int cap) {
  __shared__ unsigned hist[256];
  __shared__ unsigned s_prefix, s_want;
  __shared__ int s_sum[EV_T / 64][2];
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int len = pg_len(lens[s], cols, sh);
  const float* ws = w + s * wrow;
  float* os = out + s * orow;
  int32_t* ix = index + (long long)s * keep;
  const int left = min(len, keep);
  const int last = min(recent, left);   // entries that stay whatever they weigh
  const int old = len - last;           // those that are ranked
  const int want = left - last;         // and how many of them stay
  uint32_t edge = 0;                    // smallest word that stays
  unsigned ties = 0;                    // how many of the words equal to it do
  if (want < old && want > 0) {
    if (tid == 0) {
      s_prefix = 0;
      s_want = want;
    }
    for (int byte = 3; byte >= 0; --byte) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      const uint32_t prefix = s_prefix, mask = byte == 3 ? 0u : ~0u << (8 * byte + 8);
      for (int i = tid; i < old; i += EV_T) {
        const uint32_t u = ev_key(ws[i]);
        if ((u & mask) == prefix) atomicAdd(&hist[(u >> (8 * byte)) & 255], 1u);
      }
      __syncthreads();
      if (wv == 0) {   // the byte at which the words above it no longer fill `want`
        unsigned need = s_want, above = 0;
        int b = 255;
        // lane l holds bytes 4 l .. 4 l + 3
        const unsigned own = hist[4 * lane] + hist[4 * lane + 1] + hist[4 * lane + 2] + hist[4 * lane + 3];
        unsigned suffix = own;   // words of this lane's bytes and those above
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const unsigned v = __shfl_down(suffix, o, 64);
          if (lane + o < 64) suffix += v;
        }
        const unsigned long long ok = __ballot(suffix >= need);
        const int at = 63 - __builtin_clzll(ok);   // highest lane that reaches it
        above = __shfl(suffix - own, at, 64);
        if (lane == at) {
          for (b = 4 * lane + 3; above + hist[b] < need; --b) above += hist[b];
          s_prefix = prefix | ((uint32_t)b << (8 * byte));
          s_want = need - above;
        }
      }
      __syncthreads();
    }
    edge = s_prefix;
    ties = s_want;
  }
  const bool all = want >= old;   // nothing is ranked out
  __syncthreads();
  if (tid == 0) new_lens[s] = left;   // may be lens[s]: every thread has read it
  // entry order: ranks among the equal words and among what stays, by ballots
  int done = 0, tied = 0;
  for (int i0 = 0; i0 < old && want > 0; i0 += EV_T) {
    const int i = i0 + tid;
    const float x = i < old ? ws[i] : 0.f;
    const uint32_t u = ev_key(x);
    const bool eq = i < old && !all && u == edge;
    const unsigned long long below = lane ? ~0ull >> (64 - lane) : 0ull;
    const unsigned long long be = __ballot(eq);
    if (lane == 0) s_sum[wv][0] = __popcll(be);
    __syncthreads();
    int t = tied, total = tied;
    for (int k = 0; k < EV_T / 64; ++k) {
      if (k < wv) t += s_sum[k][0];
      total += s_sum[k][0];
    }
    tied = total;
    const bool stays = i < old && (all || u > edge || (eq && t + __popcll(be & below) < (int)ties));
    const unsigned long long bs = __ballot(stays);
    if (lane == 0) s_sum[wv][1] = __popcll(bs);
    __syncthreads();
    int p = done;
    total = done;
    for (int k = 0; k < EV_T / 64; ++k) {
      if (k < wv) p += s_sum[k][1];
      total += s_sum[k][1];
    }
    done = total;
    p += __popcll(bs & below);
    if (stays) {   // p <= i: entries not read yet are never written
      ix[p] = i;
      os[p] = x;
    }
    __syncthreads();
  }
  // the last entries, in place order too
  for (int i0 = 0; i0 < last; i0 += EV_T) {
    const int i = i0 + tid;
    const float x = i < last ? ws[old + i] : 0.f;
    __syncthreads();
    if (i < last) {
      ix[want + i] = old + i;
      os[want + i] = x;
    }
    __syncthreads();
  }
  for (int i = left + tid; i < keep; i += EV_T) ix[i] = -1;
  for (int i = left + tid; i < cap; i += EV_T) os[i] = 0.f;
}

// The rows that stay, moved.  A work-group takes 128 bytes of one head's keys
// or values of a sequence and walks the entries in order, 256 at a time: read,
// wait for all, write.  Entry i comes from index[i] >= i, and the ones read
// later lie above all that are written before, so the pages may be the same.
constexpr int EM_ROWS = 256;
template <int DH>
__global__ __launch_bounds__(256) void k_evict_move(PagedArgs c, const int32_t* __restrict__ out_table,
                                                    long long orow, int out_cols,
                                                    const int32_t* __restrict__ index,
                                                    const int32_t* __restrict__ new_lens, int keep) {
  constexpr int PARTS = DH / 64;
  const int s = blockIdx.y, tid = threadIdx.x;
  const int part = blockIdx.x % PARTS, h = (blockIdx.x / PARTS) % c.heads;
  const bool isv = blockIdx.x / PARTS >= c.heads;
  const long long page = isv ? c.vp : c.kp, slot = isv ? c.vs : c.ks;
  bf16_t* base = (isv ? c.v + h * c.vh : c.k + h * c.kh) + part * 64 + (tid & 7) * 8;
  const int left = new_lens[s];
  for (int i0 = 0; i0 < left; i0 += EM_ROWS) {
    uint4 w[8];
    bf16_t* to[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = i0 + u * 32 + (tid >> 3);
      to[u] = nullptr;
      if (i < left) {
        const int e = index[(long long)s * keep + i];
        const int a = pg_read(c.table[s * c.trow + (e >> c.sh)], c.pages);
        const int b = out_table[s * orow + (i >> c.sh)];
        w[u] = *(const uint4*)(base + a * page + pg_slot(e, c.sh, slot));
        if (pg_writable(b, c.pages)) to[u] = base + b * page + pg_slot(i, c.sh, slot);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // every read of the wave has returned
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (to[u]) *(uint4*)to[u] = w[u];
    __syncthreads();
  }
}

hipError_t paged_evict(const PagedArgs& c, int Dh, const int32_t* out_table, long long out_row,
                       int out_cols, const float* w, long long wrow, int keep, int recent,
                       int32_t* index, int32_t* new_lens, float* out, long long orow,
                       hipStream_t st) {
  if (c.seqs == 0) return hipSuccess;
  hipLaunchKernelGGL(k_evict_pick, dim3(c.seqs), dim3(EV_T), 0, st, c.lens, c.cols, c.sh, w, wrow,
                     keep, recent, index, new_lens, out, orow, c.cols << c.sh);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const dim3 grid((unsigned)(2 * c.heads * (Dh / 64)), (unsigned)c.seqs), block(256);
  if (Dh == 64)
    hipLaunchKernelGGL(k_evict_move<64>, grid, block, 0, st, c, out_table, out_row, out_cols, index, new_lens, keep);
  else if (Dh == 128)
    hipLaunchKernelGGL(k_evict_move<128>, grid, block, 0, st, c, out_table, out_row, out_cols, index, new_lens, keep);
  else
    return hipErrorInvalidValue;
  return hipGetLastError();
}

}  // namespace ann
