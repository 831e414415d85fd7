// Queries and keys as the attention takes them (model.py:244-247): each head's
// row normalised, n = x / sqrt(mean(x^2) + eps), and its first half turned by
// the token's position, y0 = c n0 + s n1, y1 = c n1 - s n0 on the adjacent
// pairs p < D / 4; the other half as it is.  One pass, fp32 inside, rounded
// once (rope_ht(rms(x)) rounds twice).  The gradient of the same: g turned back,
// g' = (c g0 - s g1, c g1 + s g0), then dx = r (g' - x r^2 mean(x g')) with
// r = 1 / sqrt(mean(x^2) + eps).
#include "common.h"
#include "launch.h"

namespace ann {

__device__ __forceinline__ float qr_ld(const float* p) { return *p; }
__device__ __forceinline__ float qr_ld(const bf16_t* p) { return bf2f(*p); }
__device__ __forceinline__ void qr_st(float* p, float v) { *p = v; }
__device__ __forceinline__ void qr_st(bf16_t* p, float v) { *p = f2bf(v); }

// The row of head h (queries, then keys) of token (b, t): x, its gradient and
// its output.
template <typename T>
struct QkRow {
  const T* x;
  const T* g;
  T* y;
};
template <typename T, bool BWD>
__device__ __forceinline__ QkRow<T> qk_row(const QkRows& a, int b, int t, int h) {
  const bool k = h >= a.Hq;
  const int i = k ? h - a.Hq : h, H = k ? a.Hk : a.Hq;
  const long long* s = k ? a.ks : a.qs;
  QkRow<T> r;
  r.x = (const T*)(k ? a.k : a.q) + b * s[0] + t * s[1] + i * s[2];
  r.y = (T*)(k ? a.ko : a.qo) + (((long long)b * a.T + t) * H + i) * a.D;
  if constexpr (BWD) {
    const long long* gs = k ? a.gks : a.gqs;
    r.g = (const T*)(k ? a.gk : a.gq) + b * gs[0] + t * gs[1] + i * gs[2];
  }
  return r;
}

// The table row of token (b, t); a position the table does not have takes the
// nearest it has.  64 bits: a start may be any of 32, and t goes on from there.
__device__ __forceinline__ int qk_position(const QkRows& a, int b, int t) {
  long long p = (long long)a.pos0 + t;
  if (a.pos) p = a.pos_each ? a.pos[(long long)b * a.T + t] : (long long)a.pos[b] + t;
  return (int)min(max(p, 0LL), a.table_rows - 1LL);
}

// One wave for each row, any D that is a multiple of 4 and any alignment: a pair a
// lane, read twice.  Bound by its waves, not by memory: 32768 tokens of 6 heads of 20, 36 or
// 96 in bf16 63 us all alike, the gradient 86.
template <typename T, bool BWD>
__global__ __launch_bounds__(256) void k_qk_rope_any(QkRows a, long long first, long long n) {
  const long long w = first + (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= n) return;
  const int lane = threadIdx.x & 63;
  const int H = a.Hq + a.Hk, D = a.D, d4 = D / 4;
  const int h = (int)(w % H);
  const long long tok = w / H;
  const int b = (int)(tok / a.T), t = (int)(tok % a.T);
  const QkRow<T> r = qk_row<T, BWD>(a, b, t, h);
  const float* cs = a.cs + (long long)qk_position(a, b, t) * d4;
  const float* sn = a.sn + (long long)qk_position(a, b, t) * d4;
  auto turned = [&](int p, float& g0, float& g1) {   // pair p of the gradient, turned back
    g0 = qr_ld(r.g + 2 * p);
    g1 = qr_ld(r.g + 2 * p + 1);
    if (p < d4) {
      const float c = cs[p], s = sn[p], u = g0;
      g0 = c * u - s * g1;
      g1 = c * g1 + s * u;
    }
  };
  float ss = 0.f, sg = 0.f;
  for (int p = lane; p < D / 2; p += 64) {
    const float x0 = qr_ld(r.x + 2 * p), x1 = qr_ld(r.x + 2 * p + 1);
    ss += x0 * x0 + x1 * x1;
    if constexpr (BWD) {
      float g0, g1;
      turned(p, g0, g1);
      sg += x0 * g0 + x1 * g1;
    }
  }
  const float rr = rsqrtf(wave_sum(ss) / (float)D + a.eps);
  float f = 0.f;
  if constexpr (BWD) f = rr * rr * (wave_sum(sg) / (float)D);
  for (int p = lane; p < D / 2; p += 64) {
    const float x0 = qr_ld(r.x + 2 * p), x1 = qr_ld(r.x + 2 * p + 1);
    float y0, y1;
    if constexpr (BWD) {
      turned(p, y0, y1);
      y0 = rr * (y0 - x0 * f);
      y1 = rr * (y1 - x1 * f);
    } else {
      y0 = x0 * rr;
      y1 = x1 * rr;
      if (p < d4) {
        const float c = cs[p], s = sn[p], u = y0;
        y0 = c * u + s * y1;
        y1 = c * y1 - s * u;
      }
    }
    qr_st(r.y + 2 * p, y0);
    qr_st(r.y + 2 * p + 1, y1);
  }
}

// The same for head dims 64 and 128 of 16-byte aligned rows: one wave for each
// token, whose heads pass four (or so) at a time, W lanes of 16 bytes each, with
// the token's angles read once.  Bound by memory: a value is read (twice with its
// gradient) and written once, for 5 (10) operations.  U groups of heads are on
// their way together.  Measured: 64 x 512 tokens of 6 + 6 heads of 128 in bf16, of a
// fused projection, 32.6 us, 6.2 TB/s; the gradient at 16 x 1023 tokens of 8 + 8
// heads of 64 in fp32 36.3 us, 5.6 TB/s (a 1 GiB copy: 5.2 TB/s).  A wave for each
// row (above) takes 118 and 107 us there.
template <typename T>
struct QrWord;
template <>
struct QrWord<float> {
  static constexpr int NV = 4;
  static __device__ __forceinline__ void load(const float* p, float* f) {
    const float4 w = *(const float4*)p;
    f[0] = w.x; f[1] = w.y; f[2] = w.z; f[3] = w.w;
  }
  static __device__ __forceinline__ void store(float* p, const float* f) {
    st_once(p, __builtin_bit_cast(uint4, make_float4(f[0], f[1], f[2], f[3])));
  }
  static __device__ __forceinline__ void angles(const float* p, float* f) {
    const float2 w = *(const float2*)p;
    f[0] = w.x; f[1] = w.y;
  }
};
template <>
struct QrWord<bf16_t> {
  static constexpr int NV = 8;
  static __device__ __forceinline__ void load(const bf16_t* p, float* f) { unpack8(*(const uint4*)p, f); }
  static __device__ __forceinline__ void store(bf16_t* p, const float* f) {
    st_once(p, make_uint4(pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7])));
  }
  static __device__ __forceinline__ void angles(const float* p, float* f) {
    const float4 w = *(const float4*)p;
    f[0] = w.x; f[1] = w.y; f[2] = w.z; f[3] = w.w;
  }
};

template <typename T, int D, bool BWD>
__global__ __launch_bounds__(256) void k_qk_rope(QkRows a, int first, int tokens) {
  using V = QrWord<T>;
  constexpr int NV = V::NV, W = D / NV, HP = 64 / W, U = BWD ? 2 : 4;
  const int tok = first + blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (tok >= tokens) return;
  const int lane = threadIdx.x & 63, l = lane % W;
  const int b = a.B == 1 ? 0 : tok / a.T, t = tok - b * a.T;
  const int H = a.Hq + a.Hk;
  const bool turn = l < W / 2;
  const long long at = (long long)qk_position(a, b, t) * (D / 4) + (turn ? l : 0) * (NV / 2);
  float cs[NV / 2], sn[NV / 2];
  V::angles(a.cs + at, cs);
  V::angles(a.sn + at, sn);
  for (int h0 = 0; h0 < H; h0 += HP * U) {
    float x[U][NV], g[BWD ? U : 1][NV];
    QkRow<T> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = min(h0 + u * HP + lane / W, H - 1);   // past the last head: that one again
      r[u] = qk_row<T, BWD>(a, b, t, h);
      V::load(r[u].x + l * NV, x[u]);
      if constexpr (BWD) V::load(r[u].g + l * NV, g[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (h0 + u * HP >= H) break;
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) ss += x[u][j] * x[u][j];
      const float rr = rsqrtf(group_sum<W>(ss) / (float)D + a.eps);
      float y[NV];
      if constexpr (BWD) {
        float sg = 0.f;
#pragma unroll
        for (int j = 0; j < NV; j += 2) {
          const float u0 = g[u][j], u1 = g[u][j + 1];
          y[j] = turn ? cs[j / 2] * u0 - sn[j / 2] * u1 : u0;
          y[j + 1] = turn ? cs[j / 2] * u1 + sn[j / 2] * u0 : u1;
          sg += x[u][j] * y[j] + x[u][j + 1] * y[j + 1];
        }
        const float f = rr * rr * (group_sum<W>(sg) / (float)D);
#pragma unroll
        for (int j = 0; j < NV; ++j) y[j] = rr * (y[j] - x[u][j] * f);
      } else {
#pragma unroll
        for (int j = 0; j < NV; j += 2) {
          const float u0 = x[u][j] * rr, u1 = x[u][j + 1] * rr;
          y[j] = turn ? cs[j / 2] * u0 + sn[j / 2] * u1 : u0;
          y[j + 1] = turn ? cs[j / 2] * u1 - sn[j / 2] * u0 : u1;
        }
      }
      if (h0 + u * HP + lane / W < H) V::store(r[u].y + l * NV, y);
    }
  }
}

// Whether 16-byte words reach every row of the operands.
static bool qk_words(const QkRows& a, bool bwd, int size) {
  const auto fine = [&](const void* p, const long long* s) {
    const long long m = 16 / size - 1;
    return (((uintptr_t)p) & 15) == 0 && ((s[0] | s[1] | s[2]) & m) == 0;
  };
  return (a.D == 64 || a.D == 128) && fine(a.q, a.qs) && (!a.Hk || fine(a.k, a.ks)) &&
         (!bwd || (fine(a.gq, a.gqs) && (!a.Hk || fine(a.gk, a.gks)))) &&
         (((uintptr_t)a.qo | (uintptr_t)a.ko | (uintptr_t)a.cs | (uintptr_t)a.sn) & 15) == 0;
}

// Rows (a wave each, four a work-group) of one launch: a grid holds less than 2^32
// threads, and one of more is cut short without an error.
constexpr long long QK_ROWS = 1LL << 25;
static unsigned qk_blocks(long long rows) { return (unsigned)(((rows < QK_ROWS ? rows : QK_ROWS) + 3) / 4); }

hipError_t qk_norm_rope(const QkRows& a, bool bwd, int dtype, hipStream_t st) {
  const long long tokens = (long long)a.B * a.T, n = tokens * (a.Hq + a.Hk);
  if (n == 0) return hipSuccess;
  const dim3 block(256);
  if (qk_words(a, bwd, dtype == 0 ? 4 : 2) && tokens < (1LL << 31) - QK_ROWS) {
    for (long long first = 0; first < tokens; first += QK_ROWS) {
      const dim3 grid(qk_blocks(tokens - first));
#define ANN_QK(TY, D)                                                                                        \
  if (bwd) hipLaunchKernelGGL((k_qk_rope<TY, D, true>), grid, block, 0, st, a, (int)first, (int)tokens);   \
  else hipLaunchKernelGGL((k_qk_rope<TY, D, false>), grid, block, 0, st, a, (int)first, (int)tokens)
      if (dtype == 0) {
        if (a.D == 64) { ANN_QK(float, 64); } else { ANN_QK(float, 128); }
      } else {
        if (a.D == 64) { ANN_QK(bf16_t, 64); } else { ANN_QK(bf16_t, 128); }
      }
#undef ANN_QK
    }
    return hipGetLastError();
  }
  for (long long first = 0; first < n; first += QK_ROWS) {
    const dim3 grid(qk_blocks(n - first));
#define ANN_QK(TY)                                                                            \
  if (bwd) hipLaunchKernelGGL((k_qk_rope_any<TY, true>), grid, block, 0, st, a, first, n);   \
  else hipLaunchKernelGGL((k_qk_rope_any<TY, false>), grid, block, 0, st, a, first, n)
    if (dtype == 0) {
      ANN_QK(float);
    } else {
      ANN_QK(bf16_t);
    }
#undef ANN_QK
  }
  return hipGetLastError();
}

// ---- append to a paged cache ---------------------------------------------------
//
// One wave for each new token: its sequence is found once, then its heads
// (queries, keys, values) four or eight at a time, DH / 8 lanes of 16 bytes each.
// Queries and keys are normalised and turned; a key and a value go to their
// entry's slot, a query to its row of the output.  A token behind the last
// sequence's, an entry outside the table and a page that is none are left alone.
// Bound by memory where there is enough of it: 4,200 tokens of 3 x 12 heads of 128, 15.0 us,
// 5.2 TB/s; a decoding step of 64 sequences (0.6 MB) takes
// 6.2 us, a launch and three reads that wait for one another (starts, then length
// and table, beside the rows; then the angles).
template <int DH>
__global__ __launch_bounds__(256) void k_paged_append(PagedArgs c, QkRows a,
                                                      const bf16_t* __restrict__ v, long long vt,
                                                      long long vh, int first) {
  constexpr int W = DH / 8, HP = 64 / W, D4 = DH / 4;
  const int n = first + blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (n >= c.rows) return;
  const int lane = threadIdx.x & 63, l = lane % W;
  const int s = pg_sequence(c.starts, c.seqs, n);
  if (s < 0) return;
  const PgRange r = pg_range(c.starts[s], c.starts[s + 1], c.rows);
  const int i = n - r.first;
  if (i >= r.n) return;
  const int e = pg_len(c.lens[s], c.cols, c.sh) - r.n + i;
  const int id = e >= 0 ? c.table[s * c.trow + (e >> c.sh)] : -1;
  const bool store = pg_writable(id, c.pages);
  bf16_t* kd = c.k + (store ? id * c.kp + pg_slot(e, c.sh, c.ks) : 0) + l * 8;
  bf16_t* vd = c.v + (store ? id * c.vp + pg_slot(e, c.sh, c.vs) : 0) + l * 8;
  const int pos = min(max(a.pos ? a.pos[n] : e, 0), a.table_rows - 1);
  const bool turn = l < W / 2;   // this lane's 16 bytes are of the turned half
  float cs[4], sn[4];
  if (turn) {
    const float4 x = *(const float4*)(a.cs + (long long)pos * D4 + l * 4);
    const float4 y = *(const float4*)(a.sn + (long long)pos * D4 + l * 4);
    cs[0] = x.x; cs[1] = x.y; cs[2] = x.z; cs[3] = x.w;
    sn[0] = y.x; sn[1] = y.y; sn[2] = y.z; sn[3] = y.w;
  }
  const int H = a.Hq + 2 * a.Hk;
  for (int h0 = 0; h0 < H; h0 += HP) {
    const int h = h0 + lane / W;
    const bool on = h < H;
    const int i_ = h < a.Hq ? h : h < a.Hq + a.Hk ? h - a.Hq : h - a.Hq - a.Hk;
    const bool isv = h >= a.Hq + a.Hk, isk = !isv && h >= a.Hq;
    const bf16_t* src = isv ? v + n * vt + i_ * vh
                            : isk ? (const bf16_t*)a.k + n * a.ks[1] + i_ * a.ks[2]
                                  : (const bf16_t*)a.q + n * a.qs[1] + i_ * a.qs[2];
    uint4 w = make_uint4(0, 0, 0, 0);
    if (on) w = *(const uint4*)(src + l * 8);
    float x[8];
    unpack8(w, x);
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
    const float rr = rsqrtf(group_sum<W>(ss) / (float)DH + a.eps);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= rr;
    if (turn) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float u = x[2 * j];
        x[2 * j] = cs[j] * u + sn[j] * x[2 * j + 1];
        x[2 * j + 1] = cs[j] * x[2 * j + 1] - sn[j] * u;
      }
    }
    if (!isv) w = make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7]));
    if (!on) continue;
    if (isv) {
      if (store) st_once(vd + i_ * c.vh, w);
    } else if (isk) {
      if (store) st_once(kd + i_ * c.kh, w);
    } else {
      st_once((bf16_t*)a.qo + ((long long)n * a.Hq + i_) * DH + l * 8, w);
    }
  }
}

hipError_t paged_append(const PagedArgs& c, const QkRows& a, const bf16_t* v, long long vt,
                        long long vh, hipStream_t st) {
  if (c.rows == 0 || c.seqs == 0) return hipSuccess;
  if (a.D != 64 && a.D != 128) return hipErrorInvalidValue;
  for (long long first = 0; first < c.rows; first += QK_ROWS) {
    const dim3 grid(qk_blocks(c.rows - first)), block(256);
    if (a.D == 64) hipLaunchKernelGGL(k_paged_append<64>, grid, block, 0, st, c, a, v, vt, vh, (int)first);
    else hipLaunchKernelGGL(k_paged_append<128>, grid, block, 0, st, c, a, v, vt, vh, (int)first);
  }
  return hipGetLastError();
}

}  // namespace ann
