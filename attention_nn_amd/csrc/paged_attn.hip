// Attention of new tokens over a paged key/value cache, and the weight that
// each entry receives from them.
//
// A token at entry e sees the entries j <= e and, with a window, e - j < window.
//   s_j = scale q.k_j,  lse = log sum_j exp(s_j),  o = sum_j exp(s_j - lse) v_j
//   w'_j = w_j + sum over the new tokens and heads of exp(s_j - lse)
// A token that sees nothing gets o = 0 and lse = -inf.
#include <math.h>
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

template <int DH>
__global__ __launch_bounds__(256) void k_paged_attn_row(PagedArgs c, const bf16_t* __restrict__ q,
                                                        long long qt, long long qh, int heads,
                                                        float scale, int window,
                                                        bf16_t* __restrict__ out,
                                                        float* __restrict__ lse) {
  constexpr int DL = DH / 64;
  const int lane = threadIdx.x & 63;
  const long long w = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = (int)(w / heads), h = (int)(w % heads);
  if (n >= c.rows) return;
  const int s = pg_sequence(c.starts, c.seqs, n);
  if (s < 0) return;
  const PgRange r = pg_range(c.starts[s], c.starts[s + 1], c.rows);
  if (n - r.first >= r.n) return;
  const int e = pg_len(c.lens[s], c.cols, c.sh) - r.n + (n - r.first);
  const int lo = max(0, e < window ? 0 : e - window + 1);
  float m, l, o[DL];
  pa_row<DH>(c, c.table + s * c.trow, q + n * qt + h * qh, h / (heads / c.heads), lo, e + 1,
             scale * PA_LOG2E, m, l, o);
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int d = 0; d < DL; ++d)
    out[((long long)n * heads + h) * DH + lane * DL + d] = f2bf(o[d] * inv);
  if (lse && lane == 0)
    lse[(long long)n * heads + h] =
        l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * PA_LN2;
}

size_t paged_attention_ws_bytes(const PagedArgs&, int, int) { return 0; }

hipError_t paged_attention(const PagedArgs& c, const bf16_t* q, long long qt, long long qh,
                           int heads, int Dh, float scale, int window, bf16_t* out, float* lse,
                           void* ws, hipStream_t st) {
  if (c.rows == 0 || c.seqs == 0) return hipSuccess;
  (void)ws;
  const int win = window > 0 ? window : 0x7fffffff;
  const dim3 grid((unsigned)(((long long)c.rows * heads + 3) / 4)), block(256);
  if (Dh == 64)
    hipLaunchKernelGGL(k_paged_attn_row<64>, grid, block, 0, st, c, q, qt, qh, heads, scale, win, out, lse);
  else if (Dh == 128)
    hipLaunchKernelGGL(k_paged_attn_row<128>, grid, block, 0, st, c, q, qt, qh, heads, scale, win, out, lse);
  else
    return hipErrorInvalidValue;
  return hipGetLastError();
}

// ---- weight of the entries -------------------------------------------------------
//
// A work-group takes 64 entries of a sequence, a lane for each entry, and its
// four waves every fourth (token, head): a lane's sum runs in row order and the
// four are added in wave order, so the result does not depend on the grid.
template <int DH>
__global__ __launch_bounds__(256) void k_paged_weight(PagedArgs c, const bf16_t* __restrict__ q,
                                                      long long qt, long long qh, int heads,
                                                      const float* __restrict__ lse, float scale,
                                                      int window, const float* __restrict__ w,
                                                      long long wrow, float* __restrict__ out,
                                                      long long orow, int cap) {
  __shared__ float part[4][64];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int s = blockIdx.y, j = blockIdx.x * 64 + lane;
  const int len = pg_len(c.lens[s], c.cols, c.sh);
  const PgRange r = pg_range(c.starts[s], c.starts[s + 1], c.rows);
  float sum = 0.f;
  if (blockIdx.x * 64 < len) {
    const int jr = min(j, len - 1);
    const int id = pg_read(c.table[s * c.trow + (jr >> c.sh)], c.pages);
    const bf16_t* kr = c.k + id * c.kp + pg_slot(jr, c.sh, c.ks);
    const int G = heads / c.heads, rows = r.n * heads;
    for (int x = wv; x < rows; x += 4) {
      const int i = x / heads, h = x % heads, n = r.first + i, e = len - r.n + i;
      const bf16_t* qr = q + n * qt + h * qh;
      const bf16_t* kk = kr + (h / G) * c.kh;
      float a = 0.f;
      for (int d = 0; d < DH; d += 8) {
        float f[8], g[8];
        unpack8(*(const uint4*)(kk + d), f);
        unpack8(*(const uint4*)(qr + d), g);
#pragma unroll
        for (int t = 0; t < 8; ++t) a += f[t] * g[t];
      }
      if (j <= e && e - j < window)
        sum += __builtin_amdgcn_exp2f((a * scale - lse[(long long)n * heads + h]) * PA_LOG2E);
    }
  }
  part[wv][lane] = sum;
  __syncthreads();
  if (wv || j >= cap) return;
  const float was = w[s * wrow + j];
  if (j < len)
    out[s * orow + j] = was + (((part[0][lane] + part[1][lane]) + part[2][lane]) + part[3][lane]);
  else if (out != w)
    out[s * orow + j] = was;
}

size_t paged_weight_ws_bytes(const PagedArgs&, int, int) { return 0; }

hipError_t paged_weight(const PagedArgs& c, const bf16_t* q, long long qt, long long qh, int heads,
                        int Dh, const float* lse, float scale, int window, const float* w,
                        long long wrow, float* out, long long orow, void* ws, hipStream_t st) {
  const int cap = c.cols << c.sh;
  if (c.seqs == 0 || cap == 0) return hipSuccess;
  (void)ws;
  const int win = window > 0 ? window : 0x7fffffff;
  const dim3 grid((unsigned)((cap + 63) / 64), (unsigned)c.seqs), block(256);
#define ANN_PW(D)                                                                              \
  hipLaunchKernelGGL(k_paged_weight<D>, grid, block, 0, st, c, q, qt, qh, heads, lse, scale, win, \
                     w, wrow, out, orow, cap)
  if (Dh == 64) ANN_PW(64);
  else if (Dh == 128) ANN_PW(128);
  else return hipErrorInvalidValue;
#undef ANN_PW
  return hipGetLastError();
}

}  // namespace ann
