// Group normalisation with an activation, forward and backward, channels first [N][C][HW] or last [N][HW][C].
//
//   row (n, g): the D = C / groups * HW elements of image n whose channel lies in group g
//   mean = sum x / D;  var = sum (x - mean)^2 / D;  rstd = 1 / sqrt(var + eps);  xh = (x - mean) rstd
//   p = gamma[c] xh + beta[c];  y = f(p),  f = none, leaky ReLU (x >= 0 ? x : slope x) or SiLU (x / (1 + exp(-x)))
// Backward, with dp = dy f'(p) formed again from x:
//   dbeta[c] = sum dp;  dgamma[c] = sum dp xh;  both over n and pixels
//   s1 = sum over the row of gamma dp / D, s2 = sum of gamma dp xh / D;  dx = rstd (gamma dp - s1 - xh s2)
// Statistics, sums and all arithmetic are fp32; the variance is taken around the mean, never as a difference of
// squares.
#include <algorithm>

#include "keep8.hpp"

namespace lnn {

struct NormGeom {
  int N, C, HW, G, Cg, last, silu;
  int n0, nb;           // images of this launch
  float slope, eps, inv_d;
  uint32_t D, row0;   // row0: first row of this launch (a grid holds fewer than 2^32 threads)
};

// 1 / (1 + exp(-p)).  v_exp_f32 takes powers of two: -p log2(e) is rounded, and what the rounding lost goes back in to
// first order (without it the error grows with |p|).  Beyond 2^126 the sigmoid is 0 next to any p a row can hold.
__device__ __forceinline__ float sigmoid(float p) {
  constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
  const float t = fminf(-p * kLog2e, 126.0f);
  const float lo = fmaf(-p, kLog2e, -t);
  float e = __builtin_amdgcn_exp2f(t);
  e = fmaf(e, t < 126.0f ? lo * kLn2 : 0.0f, e);
  return __builtin_amdgcn_rcpf(1.0f + e);
}
// f of four values in place; no activation is a leaky ReLU of slope 1
__device__ __forceinline__ void act4(int silu, float slope, float* p) {
  if (silu) {
#pragma unroll
    for (int k = 0; k < 4; ++k) p[k] *= sigmoid(p[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) p[k] = p[k] >= 0.0f ? p[k] : slope * p[k];
  }
}
// d[k] *= f'(p[k])
__device__ __forceinline__ void slope4(int silu, float slope, const float* p, float* d) {
  if (silu) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float s = sigmoid(p[k]);
      d[k] *= s * fmaf(p[k], 1.0f - s, 1.0f);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) d[k] = p[k] >= 0.0f ? d[k] : slope * d[k];
  }
}

// ---- a whole row in registers (channels first, row contiguous) ------------------------------------------------------
//
// One workgroup per row reads it once: a lane holds V groups of four elements, and mean, variance and result come from
// registers.  The row is dealt out in units of 2^ul lanes, each unit inside one channel plane (4 * 2^ul elements of it),
// so gamma, beta and the channel sums of the backward pass belong to whole units and no element needs a division.
struct Units {
  int ul, per, total;   // log2 lanes of a unit; units of a plane; units of the row
  FastDiv dper;
};
struct UnitPos {
  uint32_t ch, at;   // channel of the group; element of the row
  int cnt;           // elements of this lane's four that exist
};
__device__ __forceinline__ UnitPos unit_pos(const NormGeom& q, const Units& un, uint32_t u, uint32_t lane) {
  UnitPos r;
  r.ch = un.per == 1 ? u : un.dper.div(u);
  const uint32_t pix = (((u - r.ch * un.per) << un.ul) + lane) * 4;
  r.at = r.ch * q.HW + pix;
  r.cnt = u < (uint32_t)un.total ? min(max(q.HW - (int)pix, 0), 4) : 0;
  return r;
}

template <int T>
__device__ __forceinline__ float sum_all(float v, float* sh) {   // over the T threads of the block; sh: T / 64 floats of its own
#pragma unroll
  for (int w = 32; w > 0; w >>= 1) v += __shfl_xor(v, w, 64);
  if (T == 64) return v;
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = sh[0];
#pragma unroll
  for (int w = 1; w < T / 64; ++w) s += sh[w];
  return s;
}

template <int T, int V, bool KEEP>
__global__ __launch_bounds__(T) void gn_fwd_res_kernel(NormGeom q, Units un, const float* x, const float* gamma, const float* beta,
                                                       float* y, float* mean, float* rstd, uint8_t* codes, uint8_t* bytes) {
  __shared__ float sh[2][T / 64];
  const uint32_t row = q.row0 + blockIdx.x, base = row * q.D, c0 = (row % q.G) * q.Cg;
  const uint32_t lane = threadIdx.x & ((1u << un.ul) - 1), u0 = threadIdx.x >> un.ul;
  const int step = T >> un.ul;
  float v[V][4];
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (i * step < un.total) {
      const UnitPos p = unit_pos(q, un, i * step + u0, lane);
      SrcF::load4(x, base + p.at, p.cnt, v[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (i * step < un.total) {
#pragma unroll
      for (int k = 0; k < 4; ++k) s += v[i][k];
    }
  }
  const float m = sum_all<T>(s, sh[0]) * q.inv_d;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (i * step < un.total) {
      const UnitPos p = unit_pos(q, un, i * step + u0, lane);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float d = k < p.cnt ? v[i][k] - m : 0.0f;
        s += d * d;
      }
    }
  }
  const float r = 1.0f / sqrtf(sum_all<T>(s, sh[1]) * q.inv_d + q.eps);
  if (threadIdx.x == 0) {
    mean[row] = m;
    rstd[row] = r;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (i * step < un.total) {
      const UnitPos p = unit_pos(q, un, i * step + u0, lane);
      if (KEEP) {   // planes are whole blocks of 32: the eight lanes of a block are all in or all out
        uint32_t byte;
        const uint32_t code = encode_lane4(v[i], &byte);
        if (p.cnt == 4) {
          reinterpret_cast<B4*>(codes + base + p.at)->v = code;
          if ((lane & 7) == 0) bytes[(base + p.at) >> 5] = (uint8_t)byte;
        }
      }
      if (p.cnt > 0) {
        const float ga = gamma ? gamma[c0 + p.ch] : 1.0f, be = beta ? beta[c0 + p.ch] : 0.0f;
        float o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = (v[i][k] - m) * r * ga + be;
        act4(q.silu, q.slope, o);
        store4(y, base + p.at, p.cnt, o);
      }
    }
  }
}

// Both sums of a unit are formed by lane exchanges and left in LDS; the channel sums are theirs in order, so nothing
// depends on which wavefront came first.  part (or null): [2][N][C], the channel sums of dp and of dp xh.
template <int T, int V, class SRC>
__global__ __launch_bounds__(T) void gn_bwd_res_kernel(NormGeom q, Units un, SRC x, const float* gamma, const float* beta,
                                                       const float* mean, const float* rstd, const float* dy, float* dx, int beta_dx,
                                                       float* part) {
  extern __shared__ float su[];   // [units][2]
  __shared__ float sh[2][T / 64];
  const uint32_t row = q.row0 + blockIdx.x, base = row * q.D, n = row / q.G, c0 = (row % q.G) * q.Cg;
  const uint32_t lane = threadIdx.x & ((1u << un.ul) - 1), u0 = threadIdx.x >> un.ul;
  const int step = T >> un.ul;
  const float m = mean[row], r = rstd[row];
  float xh[V][4], dp[V][4];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (i * step < un.total) {
      const UnitPos p = unit_pos(q, un, i * step + u0, lane);
      x.load(base + p.at, p.cnt, xh[i]);
      SrcF::load4(dy, base + p.at, p.cnt, dp[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (i * step < un.total) {
      const uint32_t u = i * step + u0;
      const UnitPos p = unit_pos(q, un, u, lane);
      float ga = 1.0f, be = 0.0f;
      if (p.cnt > 0) {
        if (gamma) ga = gamma[c0 + p.ch];
        if (beta) be = beta[c0 + p.ch];
      }
      float a = 0.0f, b = 0.0f, pre[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        xh[i][k] = k < p.cnt ? (xh[i][k] - m) * r : 0.0f;
        pre[k] = xh[i][k] * ga + be;
      }
      slope4(q.silu, q.slope, pre, dp[i]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        a += dp[i][k];
        b += dp[i][k] * xh[i][k];
        dp[i][k] *= ga;
      }
      for (int w = (1 << un.ul) >> 1; w > 0; w >>= 1) {
        a += __shfl_xor(a, w, 64);
        b += __shfl_xor(b, w, 64);
      }
      if (lane == 0 && u < (uint32_t)un.total) {
        su[2 * u] = a;
        su[2 * u + 1] = b;
      }
    }
  }
  __syncthreads();
  float s1 = 0.0f, s2 = 0.0f;
  for (int ch = threadIdx.x; ch < q.Cg; ch += T) {
    float a = 0.0f, b = 0.0f;
    for (int j = 0; j < un.per; ++j) {
      a += su[2 * (ch * un.per + j)];
      b += su[2 * (ch * un.per + j) + 1];
    }
    if (part) {
      part[n * q.C + c0 + ch] = a;
      part[(uint32_t)(q.N + n) * q.C + c0 + ch] = b;
    }
    const float ga = gamma ? gamma[c0 + ch] : 1.0f;
    s1 += ga * a;
    s2 += ga * b;
  }
  if (!dx) return;
  s1 = sum_all<T>(s1, sh[0]) * q.inv_d;
  s2 = sum_all<T>(s2, sh[1]) * q.inv_d;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (i * step < un.total) {
      const UnitPos p = unit_pos(q, un, i * step + u0, lane);
      if (p.cnt > 0) {
        float o[4];
        if (beta_dx) SrcF::load4(dx, base + p.at, p.cnt, o);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float e = r * (dp[i][k] - s1 - xh[i][k] * s2);
          o[k] = beta_dx ? o[k] + e : e;
        }
        store4(dx, base + p.at, p.cnt, o);
      }
    }
  }
}

// ---- rows of channels alone (HW = 1: behind a dense layer) ----------------------------------------------------------
//
// A row is C / groups neighbouring floats: L lanes hold it, V groups of four each, 256 / L rows to a workgroup.
template <int L>
__device__ __forceinline__ float sum_lanes(float v, float* sh) {
#pragma unroll
  for (int w = (L < 64 ? L : 64) / 2; w > 0; w >>= 1) v += __shfl_xor(v, w, 64);
  if (L <= 64) return v;
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return sh[0] + sh[1] + sh[2] + sh[3];
}

template <int L, int V, bool KEEP>
__global__ __launch_bounds__(256) void gn_fwd_rows_kernel(NormGeom q, const float* x, const float* gamma, const float* beta, float* y,
                                                          float* mean, float* rstd, uint8_t* codes, uint8_t* bytes) {
  __shared__ float sh[2][4];
  const uint32_t lane = threadIdx.x % L, row = blockIdx.x * (256 / L) + threadIdx.x / L, rows = (uint32_t)q.N * q.G;
  const uint32_t base = row * q.D, c0 = (row % q.G) * q.Cg;
  float v[V][4];
  int cnt[V];
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    cnt[i] = row < rows ? min(max(q.Cg - (int)(i * L + lane) * 4, 0), 4) : 0;
    SrcF::load4(x, base + (i * L + lane) * 4, cnt[i], v[i]);
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) s += v[i][k];
  const float m = sum_lanes<L>(s, sh[0]) * q.inv_d;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float d = k < cnt[i] ? v[i][k] - m : 0.0f;
      s += d * d;
    }
  const float r = 1.0f / sqrtf(sum_lanes<L>(s, sh[1]) * q.inv_d + q.eps);
  if (lane == 0 && row < rows) {
    mean[row] = m;
    rstd[row] = r;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const uint32_t at = base + (i * L + lane) * 4;
    if (KEEP) {   // rows are whole blocks of 32: the eight lanes of a block are all in or all out
      uint32_t byte;
      const uint32_t code = encode_lane4(v[i], &byte);
      if (cnt[i] == 4) {
        reinterpret_cast<B4*>(codes + at)->v = code;
        if ((lane & 7) == 0) bytes[at >> 5] = (uint8_t)byte;
      }
    }
    if (cnt[i] > 0) {
      float ga[4] = {1.0f, 1.0f, 1.0f, 1.0f}, be[4] = {0.0f, 0.0f, 0.0f, 0.0f}, o[4];
      if (gamma) SrcF::load4(gamma, c0 + (i * L + lane) * 4, cnt[i], ga);
      if (beta) SrcF::load4(beta, c0 + (i * L + lane) * 4, cnt[i], be);
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = (v[i][k] - m) * r * ga[k] + be[k];
      act4(q.silu, q.slope, o);
      store4(y, at, cnt[i], o);
    }
  }
}

// A workgroup stays with one group of channels and walks over a chunk of the rows, so a lane's channels are fixed: gamma,
// beta and the channel sums stay in registers, and the sums cross lanes once per workgroup.
// part (or null): [2][chunks][C].
template <int L, int V, class SRC>
__global__ __launch_bounds__(256) void gn_bwd_rows_kernel(NormGeom q, int chunks, SRC x, const float* gamma, const float* beta,
                                                          const float* mean, const float* rstd, const float* dy, float* dx, int beta_dx,
                                                          float* part) {
  constexpr int S = 256 / L;
  __shared__ float sh[2][4];
  __shared__ float tot[2][256 * 4];
  const uint32_t g = blockIdx.x % q.G, chunk = blockIdx.x / q.G, lane = threadIdx.x % L, slot = threadIdx.x / L;
  const int per = (q.N + chunks - 1) / chunks, n0 = (int)chunk * per, n1 = min(n0 + per, q.N);
  const uint32_t c0 = g * q.Cg;
  float ga[V][4], be[V][4], sa[V][4], sb[V][4];
  int cnt[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    cnt[i] = min(max(q.Cg - (int)(i * L + lane) * 4, 0), 4);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      ga[i][k] = 1.0f;
      be[i][k] = sa[i][k] = sb[i][k] = 0.0f;
    }
    if (gamma) SrcF::load4(gamma, c0 + (i * L + lane) * 4, cnt[i], ga[i]);
    if (beta) SrcF::load4(beta, c0 + (i * L + lane) * 4, cnt[i], be[i]);
  }
  for (int nn = n0; nn < n1; nn += S) {   // all lanes together: the row sums may cross wavefronts
    const int n = nn + (int)slot;
    const bool in = n < n1;
    const uint32_t row = (uint32_t)(in ? n : n0) * q.G + g, base = row * q.D;
    const float m = mean[row], r = rstd[row];
    float xh[V][4], dp[V][4], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x.load(base + (i * L + lane) * 4, in ? cnt[i] : 0, xh[i]);
      SrcF::load4(dy, base + (i * L + lane) * 4, in ? cnt[i] : 0, dp[i]);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float pre[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        xh[i][k] = in && k < cnt[i] ? (xh[i][k] - m) * r : 0.0f;
        pre[k] = xh[i][k] * ga[i][k] + be[i][k];
      }
      slope4(q.silu, q.slope, pre, dp[i]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        sa[i][k] += dp[i][k];
        sb[i][k] += dp[i][k] * xh[i][k];
        dp[i][k] *= ga[i][k];
        s1 += dp[i][k];
        s2 += dp[i][k] * xh[i][k];
      }
    }
    if (!dx) continue;
    if (L > 64) __syncthreads();   // sh is read no more
    s1 = sum_lanes<L>(s1, sh[0]) * q.inv_d;
    s2 = sum_lanes<L>(s2, sh[1]) * q.inv_d;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint32_t at = base + (i * L + lane) * 4;
      const int c = in ? cnt[i] : 0;
      if (c > 0) {
        float o[4];
        if (beta_dx) SrcF::load4(dx, at, c, o);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float e = r * (dp[i][k] - s1 - xh[i][k] * s2);
          o[k] = beta_dx ? o[k] + e : e;
        }
        store4(dx, at, c, o);
      }
    }
  }
  if (!part) return;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      tot[0][(slot * L + lane) * 4 + k] = sa[i][k];
      tot[1][(slot * L + lane) * 4 + k] = sb[i][k];
    }
    __syncthreads();
    for (int j = threadIdx.x; j < 4 * L; j += 256) {
      const int c = i * L * 4 + j;
      if (c < q.Cg) {
        float a = 0.0f, b = 0.0f;
        for (int t = 0; t < S; ++t) {
          a += tot[0][t * L * 4 + j];
          b += tot[1][t * L * 4 + j];
        }
        part[chunk * q.C + c0 + c] = a;
        part[(uint32_t)(chunks + chunk) * q.C + c0 + c] = b;
      }
    }
  }
}

// ---- rows too long for registers, and channels last -----------------------------------------------------------------
//
// Three launches: sums per channel and chunk of pixels, the rows' statistics from them, the result.  x is read twice;
// the host takes as many images at a time as stay in the memory-side cache between the two reads.
//
// Means and sums of squared distances of two sets join as
//   n = na + nb, d = mb - ma:  m = ma + d nb / n,  M = Ma + Mb + d^2 na nb / n
struct Stat {
  float n, m, M;
};
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b) {
  const float n = a.n + b.n;
  if (n == 0.0f) return a;
  const float f = b.n / n, d = b.m - a.m;
  // an empty side has weight 0 however far its m is: the weight goes in before the square
  return {n, a.m + d * f, a.M + b.M + d * (d * (a.n * f))};
}

// channels first: one wavefront per (plane, 4096 pixels of it), the pixels in registers
constexpr int kPlane = 4096;
struct PlanePos {
  uint32_t n, c, chunk, base;
  int count;   // pixels of this wavefront's chunk
  bool in;
};
__device__ __forceinline__ PlanePos plane_pos(const NormGeom& q, int chunks) {
  const uint32_t w = blockIdx.x * 4 + (threadIdx.x >> 6);
  PlanePos p;
  p.in = w < (uint32_t)q.nb * q.C * chunks;
  const uint32_t plane = w / chunks;
  p.chunk = w - plane * chunks;
  p.n = q.n0 + plane / q.C;
  p.c = plane % q.C;
  p.base = (p.n * q.C + p.c) * q.HW + p.chunk * kPlane;
  p.count = min(kPlane, q.HW - (int)p.chunk * kPlane);
  return p;
}

__global__ __launch_bounds__(256) void gn_stats_first_kernel(NormGeom q, int chunks, const float* x, float2* part) {
  const PlanePos p = plane_pos(q, chunks);
  if (!p.in) return;
  const int lane = threadIdx.x & 63;
  float v[16][4], s = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (i * 256 < p.count) SrcF::load4(x, p.base + i * 256 + lane * 4, min(max(p.count - i * 256 - lane * 4, 0), 4), v[i]);
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (i * 256 < p.count)
#pragma unroll
      for (int k = 0; k < 4; ++k) s += v[i][k];
  const float m = sum_all<64>(s, nullptr) / (float)p.count;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (i * 256 < p.count)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float d = i * 256 + lane * 4 + k < p.count ? v[i][k] - m : 0.0f;
        s += d * d;
      }
  s = sum_all<64>(s, nullptr);
  if (lane == 0) part[((p.n - q.n0) * chunks + p.chunk) * q.C + p.c] = make_float2(m, s);
}

template <bool KEEP>
__global__ __launch_bounds__(256) void gn_apply_first_kernel(NormGeom q, int chunks, const float* x, const float* gamma, const float* beta,
                                                             const float* mean, const float* rstd, float* y, uint8_t* codes,
                                                             uint8_t* bytes) {
  const PlanePos p = plane_pos(q, chunks);
  if (!p.in) return;
  const int lane = threadIdx.x & 63;
  const uint32_t row = p.n * q.G + p.c / q.Cg;
  const float m = mean[row], r = rstd[row], ga = gamma ? gamma[p.c] : 1.0f, be = beta ? beta[p.c] : 0.0f;
  for (int i0 = 0; i0 < p.count; i0 += 1024) {   // four loads in flight
    float v[4][4];
    int cnt[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      cnt[j] = min(max(p.count - i0 - j * 256 - lane * 4, 0), 4);
      SrcF::load4(x, p.base + i0 + j * 256 + lane * 4, cnt[j], v[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t at = p.base + i0 + j * 256 + lane * 4;
      if (KEEP) {   // planes are whole blocks of 32
        uint32_t byte;
        const uint32_t code = encode_lane4(v[j], &byte);
        if (cnt[j] == 4) {
          reinterpret_cast<B4*>(codes + at)->v = code;
          if ((lane & 7) == 0) bytes[at >> 5] = (uint8_t)byte;
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) v[j][k] = (v[j][k] - m) * r * ga + be;
      act4(q.silu, q.slope, v[j]);
      store4(y, at, cnt[j], v[j]);
    }
  }
}

template <class SRC>
__global__ __launch_bounds__(256) void gn_sums_first_kernel(NormGeom q, int chunks, SRC x, const float* gamma, const float* beta,
                                                            const float* mean, const float* rstd, const float* dy, float* pa, float* pb) {
  const PlanePos p = plane_pos(q, chunks);
  if (!p.in) return;
  const int lane = threadIdx.x & 63;
  const uint32_t row = p.n * q.G + p.c / q.Cg;
  const float m = mean[row], r = rstd[row], ga = gamma ? gamma[p.c] : 1.0f, be = beta ? beta[p.c] : 0.0f;
  float a = 0.0f, b = 0.0f;
#pragma unroll 4
  for (int i = 0; i < p.count; i += 256) {
    const int cnt = min(max(p.count - i - lane * 4, 0), 4);
    float v[4], d[4], pre[4];
    x.load(p.base + i + lane * 4, cnt, v);
    SrcF::load4(dy, p.base + i + lane * 4, cnt, d);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = k < cnt ? (v[k] - m) * r : 0.0f;
      pre[k] = v[k] * ga + be;
    }
    slope4(q.silu, q.slope, pre, d);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      a += d[k];
      b += d[k] * v[k];
    }
  }
  a = sum_all<64>(a, nullptr);
  b = sum_all<64>(b, nullptr);
  if (lane == 0) {
    const uint32_t at = (p.n * chunks + p.chunk) * q.C + p.c;
    pa[at] = a;
    pb[at] = b;
  }
}

template <class SRC>
__global__ __launch_bounds__(256) void gn_dx_first_kernel(NormGeom q, int chunks, SRC x, const float* gamma, const float* beta,
                                                          const float* mean, const float* rstd, const float* dy, const float2* s12,
                                                          float* dx, int beta_dx) {
  const PlanePos p = plane_pos(q, chunks);
  if (!p.in) return;
  const int lane = threadIdx.x & 63;
  const uint32_t row = p.n * q.G + p.c / q.Cg;
  const float m = mean[row], r = rstd[row], ga = gamma ? gamma[p.c] : 1.0f, be = beta ? beta[p.c] : 0.0f;
  const float2 s = s12[row];
#pragma unroll 4
  for (int i = 0; i < p.count; i += 256) {
    const int cnt = min(max(p.count - i - lane * 4, 0), 4);
    const uint32_t at = p.base + i + lane * 4;
    float v[4], d[4], pre[4], o[4];
    x.load(at, cnt, v);
    SrcF::load4(dy, at, cnt, d);
    if (beta_dx) SrcF::load4(dx, at, cnt, o);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = (v[k] - m) * r;
      pre[k] = v[k] * ga + be;
    }
    slope4(q.silu, q.slope, pre, d);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float e = r * (d[k] * ga - s.x - v[k] * s.y);
      o[k] = beta_dx ? o[k] + e : e;
    }
    store4(dx, at, cnt, o);
  }
}

// channels last: a lane keeps four channels and walks over pixels.  TX lanes side by side span the channels (256 groups
// of four at most; more channels make more workgroups), TY = 256 / TX of them walk together.
struct LastTile {
  int tx, ty, slabs, pix, chunks;   // pix: pixels of a workgroup
};
struct LastPos {
  uint32_t n, c, chunk;
  int x, y, p0, p1, cnt;   // lane's place; pixels; channels of this lane that exist (0: none)
};
__device__ __forceinline__ LastPos last_pos(const NormGeom& q, const LastTile& t) {
  LastPos p;
  const uint32_t slab = blockIdx.x % t.slabs, k = blockIdx.x / t.slabs;
  p.chunk = k % t.chunks;
  p.n = q.n0 + k / t.chunks;
  p.y = threadIdx.x / t.tx;
  p.x = threadIdx.x - p.y * t.tx;
  p.c = (slab * t.tx + p.x) * 4;
  p.cnt = p.y < t.ty ? min(max(q.C - (int)p.c, 0), 4) : 0;
  p.p0 = p.chunk * t.pix;
  p.p1 = min(p.p0 + t.pix, q.HW);
  return p;
}

__global__ __launch_bounds__(256) void gn_stats_last_kernel(NormGeom q, LastTile t, const float* x, float2* part) {
  __shared__ float sm[4][256], sM[4][256], sn[256];
  const LastPos p = last_pos(q, t);
  constexpr int B = 8;
  Stat st[4] = {};
  if (p.cnt > 0) {
    for (int q0 = p.p0 + p.y; q0 < p.p1; q0 += B * t.ty) {
      float v[B][4];
      int nv = 0;
#pragma unroll
      for (int i = 0; i < B; ++i) {
        const int pix = q0 + i * t.ty;
        const bool in = pix < p.p1;
        nv += in;
        SrcF::load4(x, (p.n * q.HW + pix) * q.C + p.c, in ? p.cnt : 0, v[i]);
      }
      const float inv = 1.0f / (float)nv;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float s = 0.0f, M = 0.0f;
#pragma unroll
        for (int i = 0; i < B; ++i) s += v[i][k];
        const float m = s * inv;
#pragma unroll
        for (int i = 0; i < B; ++i) {
          const float d = i < nv ? v[i][k] - m : 0.0f;
          M += d * d;
        }
        st[k] = join(st[k], Stat{(float)nv, m, M});
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    sm[k][threadIdx.x] = st[k].m;
    sM[k][threadIdx.x] = st[k].M;
  }
  sn[threadIdx.x] = st[0].n;
  for (int h = t.ty; h > 1;) {
    const int half = (h + 1) >> 1;
    __syncthreads();
    if (p.y + half < h) {
      const int o = threadIdx.x + half * t.tx;
      const float na = sn[threadIdx.x], nb = sn[o];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const Stat j = join(Stat{na, sm[k][threadIdx.x], sM[k][threadIdx.x]}, Stat{nb, sm[k][o], sM[k][o]});
        sm[k][threadIdx.x] = j.m;
        sM[k][threadIdx.x] = j.M;
      }
      sn[threadIdx.x] = na + nb;
    }
    h = half;
  }
  if (p.y == 0) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < p.cnt) part[((p.n - q.n0) * t.chunks + p.chunk) * q.C + p.c + k] = make_float2(sm[k][threadIdx.x], sM[k][threadIdx.x]);
  }
}

// Statistics of row (n, g) from those of its channels and chunks of `pix` pixels.
__global__ __launch_bounds__(256) void gn_finish_kernel(NormGeom q, int chunks, int pix, const float2* part, float* mean, float* rstd) {
  __shared__ Stat sh[256];
  const uint32_t n = blockIdx.x / q.G, g = blockIdx.x % q.G;   // n: image of the batch
  Stat s = {0.0f, 0.0f, 0.0f};
  for (int j = threadIdx.x; j < chunks * q.Cg; j += 256) {
    const int chunk = j / q.Cg, c = j - chunk * q.Cg;
    const float2 e = part[(n * chunks + chunk) * q.C + g * q.Cg + c];
    s = join(s, Stat{(float)min(pix, q.HW - chunk * pix), e.x, e.y});
  }
  sh[threadIdx.x] = s;
  for (int w = 128; w > 0; w >>= 1) {
    __syncthreads();
    if ((int)threadIdx.x < w) sh[threadIdx.x] = join(sh[threadIdx.x], sh[threadIdx.x + w]);
  }
  if (threadIdx.x == 0) {
    const uint32_t row = (q.n0 + n) * q.G + g;
    mean[row] = sh[0].m;
    rstd[row] = 1.0f / sqrtf(sh[0].M * q.inv_d + q.eps);
  }
}

// What a lane's four channels need of their rows: rstd, -mean rstd gamma..., one row each (four channels may span groups)
struct LaneRows {
  float m[4], r[4], ga[4], be[4];
};
__device__ __forceinline__ void lane_rows(const NormGeom& q, const LastPos& p, const float* gamma, const float* beta, const float* mean,
                                          const float* rstd, LaneRows* l) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const bool in = k < p.cnt;
    const uint32_t c = in ? p.c + k : 0, row = p.n * q.G + c / q.Cg;
    l->m[k] = in ? mean[row] : 0.0f;
    l->r[k] = in ? rstd[row] : 0.0f;
    l->ga[k] = gamma ? gamma[c] : 1.0f;
    l->be[k] = beta ? beta[c] : 0.0f;
  }
}

template <bool KEEP>
__global__ __launch_bounds__(256) void gn_apply_last_kernel(NormGeom q, LastTile t, const float* x, const float* gamma, const float* beta,
                                                            const float* mean, const float* rstd, float* y, uint8_t* codes, uint8_t* bytes) {
  const LastPos p = last_pos(q, t);
  LaneRows l;
  lane_rows(q, p, gamma, beta, mean, rstd, &l);
  for (int pix0 = p.p0 + p.y; pix0 < p.p1; pix0 += 4 * t.ty) {   // four loads in flight
    float v[4][4];
    int cnt[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int pix = pix0 + j * t.ty;
      cnt[j] = pix < p.p1 ? p.cnt : 0;
      SrcF::load4(x, (p.n * q.HW + pix) * q.C + p.c, cnt[j], v[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t at = (p.n * q.HW + pix0 + j * t.ty) * q.C + p.c;
      if (KEEP) {   // C is a multiple of 32: eight neighbouring lanes hold a block, all in or all out
        uint32_t byte;
        const uint32_t code = encode_lane4(v[j], &byte);
        if (cnt[j] == 4) {
          reinterpret_cast<B4*>(codes + at)->v = code;
          if ((p.x & 7) == 0) bytes[at >> 5] = (uint8_t)byte;
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) v[j][k] = (v[j][k] - l.m[k]) * l.r[k] * l.ga[k] + l.be[k];
      act4(q.silu, q.slope, v[j]);
      store4(y, at, cnt[j], v[j]);
    }
  }
}

template <class SRC>
__global__ __launch_bounds__(256) void gn_sums_last_kernel(NormGeom q, LastTile t, SRC x, const float* gamma, const float* beta,
                                                           const float* mean, const float* rstd, const float* dy, float* pa, float* pb) {
  __shared__ float sh[8][256];
  const LastPos p = last_pos(q, t);
  LaneRows l;
  lane_rows(q, p, gamma, beta, mean, rstd, &l);
  float a[4] = {}, b[4] = {};
#pragma unroll 4
  for (int pix = p.p0 + p.y; pix < p.p1; pix += t.ty) {
    const uint32_t at = (p.n * q.HW + pix) * q.C + p.c;
    float v[4], d[4], pre[4];
    x.load(at, p.cnt, v);
    SrcF::load4(dy, at, p.cnt, d);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = (v[k] - l.m[k]) * l.r[k];
      pre[k] = v[k] * l.ga[k] + l.be[k];
    }
    slope4(q.silu, q.slope, pre, d);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      a[k] += d[k];
      b[k] += d[k] * v[k];
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    sh[k][threadIdx.x] = a[k];
    sh[4 + k][threadIdx.x] = b[k];
  }
  for (int h = t.ty; h > 1;) {
    const int half = (h + 1) >> 1;
    __syncthreads();
    if (p.y + half < h) {
#pragma unroll
      for (int k = 0; k < 8; ++k) sh[k][threadIdx.x] += sh[k][threadIdx.x + half * t.tx];
    }
    h = half;
  }
  if (p.y == 0) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < p.cnt) {
        const uint32_t at = (p.n * t.chunks + p.chunk) * q.C + p.c + k;
        pa[at] = sh[k][threadIdx.x];
        pb[at] = sh[4 + k][threadIdx.x];
      }
  }
}

template <class SRC>
__global__ __launch_bounds__(256) void gn_dx_last_kernel(NormGeom q, LastTile t, SRC x, const float* gamma, const float* beta,
                                                         const float* mean, const float* rstd, const float* dy, const float2* s12,
                                                         float* dx, int beta_dx) {
  const LastPos p = last_pos(q, t);
  LaneRows l;
  lane_rows(q, p, gamma, beta, mean, rstd, &l);
  float s1[4], s2[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 s = s12[p.n * q.G + (k < p.cnt ? p.c + k : 0) / q.Cg];
    s1[k] = s.x;
    s2[k] = s.y;
  }
#pragma unroll 4
  for (int pix = p.p0 + p.y; pix < p.p1; pix += t.ty) {
    const uint32_t at = (p.n * q.HW + pix) * q.C + p.c;
    float v[4], d[4], pre[4], o[4];
    x.load(at, p.cnt, v);
    SrcF::load4(dy, at, p.cnt, d);
    if (beta_dx) SrcF::load4(dx, at, p.cnt, o);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = (v[k] - l.m[k]) * l.r[k];
      pre[k] = v[k] * l.ga[k] + l.be[k];
    }
    slope4(q.silu, q.slope, pre, d);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float e = l.r[k] * (d[k] * l.ga[k] - s1[k] - v[k] * s2[k]);
      o[k] = beta_dx ? o[k] + e : e;
    }
    store4(dx, at, p.cnt, o);
  }
}

// row (n, g): s1 and s2 from the sums of its channels and chunks
__global__ __launch_bounds__(256) void gn_finish_dx_kernel(NormGeom q, int chunks, const float* gamma, const float* pa, const float* pb,
                                                           float2* s12) {
  __shared__ float sh[2][4];
  const uint32_t n = q.n0 + blockIdx.x / q.G, g = blockIdx.x % q.G;
  float a = 0.0f, b = 0.0f;
  for (int j = threadIdx.x; j < chunks * q.Cg; j += 256) {
    const int chunk = j / q.Cg, c = g * q.Cg + (j - chunk * q.Cg);
    const float ga = gamma ? gamma[c] : 1.0f;
    a += ga * pa[(n * chunks + chunk) * q.C + c];
    b += ga * pb[(n * chunks + chunk) * q.C + c];
  }
  a = sum_all<256>(a, sh[0]);
  b = sum_all<256>(b, sh[1]);
  if (threadIdx.x == 0) s12[n * q.G + g] = make_float2(a * q.inv_d, b * q.inv_d);
}

// dbeta, dgamma: column sums of the K rows of pa and pb.  A workgroup takes 32 channels and the rows [y per, (y + 1) per):
// 8 lanes per channel walk over them, then add up in order.  With gridDim.y > 1 the sums are left as rows of outa / outb
// for a second launch.
__global__ __launch_bounds__(256) void gn_params_kernel(int K, int per, int C, const float* pa, const float* pb, float* outa, int beta_a,
                                                        float* outb, int beta_b) {
  __shared__ float sh[2][8][33];
  const int li = threadIdx.x & 31, lk = threadIdx.x >> 5, c = blockIdx.x * 32 + li;
  const int k0 = blockIdx.y * per, k1 = min(k0 + per, K);
  float a = 0.0f, b = 0.0f;
  if (c < C) {
#pragma unroll 4
    for (int k = k0 + lk; k < k1; k += 8) {
      a += pa[(uint32_t)k * C + c];
      b += pb[(uint32_t)k * C + c];
    }
  }
  sh[0][lk][li] = a;
  sh[1][lk][li] = b;
  __syncthreads();
  if (lk == 0 && c < C) {
#pragma unroll
    for (int k = 1; k < 8; ++k) {
      a += sh[0][k][li];
      b += sh[1][k][li];
    }
    const uint32_t at = blockIdx.y * (uint32_t)C + c;
    if (outa) outa[at] = beta_a ? outa[at] + a : a;
    if (outb) outb[at] = beta_b ? outb[at] + b : b;
  }
}

int launch_encode8(DeviceCtx*, uint64_t, const float*, void*);

static int make_geom(const lnn_group_norm_desc* d, NormGeom* q) {
  if (!d) return set_error(LNN_ERR_INVALID, "group_norm: null descriptor");
  if (d->N < 1 || d->C < 1 || d->HW < 1 || d->groups < 1) return set_error(LNN_ERR_INVALID, "group_norm: extents must be >= 1");
  if (d->C % d->groups != 0) return set_error(LNN_ERR_INVALID, "group_norm: groups must divide the channels");
  if (d->act != LNN_ACT_NONE && d->act != LNN_ACT_LEAKY_RELU && d->act != LNN_ACT_SILU)
    return set_error(LNN_ERR_INVALID, "group_norm: unknown activation");
  if (!(d->eps > 0.0f)) return set_error(LNN_ERR_INVALID, "group_norm: eps must be > 0");
  if ((uint64_t)d->N * d->C > kMaxTensorBytes / 4 || (uint64_t)d->N * d->C * d->HW > kMaxTensorBytes / 4)
    return set_error(LNN_ERR_UNSUPPORTED, "group_norm: tensor of 2 GiB or more");
  if (d->C > 1 << 22) return set_error(LNN_ERR_UNSUPPORTED, "group_norm: more than 4194304 channels");   // grids stay below 2^32 threads
  q->N = d->N;
  q->C = d->C;
  q->HW = d->HW;
  q->G = d->groups;
  q->Cg = d->C / d->groups;
  q->last = d->channels_last != 0 || d->HW == 1;   // with one pixel the two layouts are one
  q->n0 = 0;
  q->nb = d->N;
  q->silu = d->act == LNN_ACT_SILU;
  q->slope = d->act == LNN_ACT_NONE ? 1.0f : d->slope;
  q->eps = d->eps;
  q->row0 = 0;
  q->D = (uint32_t)q->Cg * (uint32_t)q->HW;
  q->inv_d = (float)(1.0 / (double)q->D);
  return LNN_OK;
}

// How a row is dealt out to a workgroup's lanes; false where it does not fit `most` groups of four per lane.
struct ResPlan {
  Units un;
  int T, V;
};
static bool res_plan(const DeviceCtx* ctx, const NormGeom& q, int most, ResPlan* p) {
  if (q.last) return false;
  // the shortest unit that holds a plane, or whole wavefronts
  p->un.ul = q.HW <= 4 ? 0 : q.HW <= 16 ? 2 : q.HW <= 64 ? 4 : 6;
  p->un.per = ((q.HW + 3) / 4 + (1 << p->un.ul) - 1) >> p->un.ul;
  const uint64_t lanes = ((uint64_t)q.Cg * p->un.per) << p->un.ul;
  p->un.total = q.Cg * p->un.per;
  if (lanes > 1024u * most || p->un.total > 7000) return false;   // 7000: the backward pass keeps two sums per unit in 64 KB
  p->un.dper = make_fastdiv((uint32_t)p->un.per);
  p->T = lanes <= 64 ? 64 : lanes <= 256u * most ? 256 : 1024;
  if (p->T == 256 && lanes >= 1024 && q.N * q.G <= 2 * ctx->cus) p->T = 1024;
  const uint64_t v = (lanes + p->T - 1) / p->T;
  p->V = v <= 1 ? 1 : v <= 2 ? 2 : v <= 4 ? 4 : v <= 8 ? 8 : 16;
  return true;
}

constexpr uint32_t kMaxRows = 1u << 21;   // of one launch

template <int T, int V>
static void fwd_res(DeviceCtx* ctx, const NormGeom& q, const Units& un, const float* x, const float* gamma, const float* beta, float* y,
                    float* mean, float* rstd, uint8_t* codes, uint8_t* bytes) {
  const unsigned rows = (unsigned)(q.N * q.G) - q.row0 < kMaxRows ? (unsigned)(q.N * q.G) - q.row0 : kMaxRows;
  if (codes)
    hipLaunchKernelGGL((gn_fwd_res_kernel<T, V, true>), dim3(rows), dim3(T), 0, ctx->stream, q, un, x, gamma, beta, y,
                       mean, rstd, codes, bytes);
  else
    hipLaunchKernelGGL((gn_fwd_res_kernel<T, V, false>), dim3(rows), dim3(T), 0, ctx->stream, q, un, x, gamma, beta, y,
                       mean, rstd, codes, bytes);
}
template <int T, int V>
static void bwd_res(DeviceCtx* ctx, const NormGeom& q, const Units& un, const float* x, const uint8_t* codes, const uint8_t* bytes,
                    const float* gamma, const float* beta, const float* mean, const float* rstd, const float* dy, float* dx, int beta_dx,
                    float* part) {
  const unsigned rows = (unsigned)(q.N * q.G) - q.row0 < kMaxRows ? (unsigned)(q.N * q.G) - q.row0 : kMaxRows;
  if (codes)
    hipLaunchKernelGGL((gn_bwd_res_kernel<T, V, Src8>), dim3(rows), dim3(T), (unsigned)un.total * 8, ctx->stream, q, un,
                       Src8{codes, bytes}, gamma, beta, mean, rstd, dy, dx, beta_dx, part);
  else
    hipLaunchKernelGGL((gn_bwd_res_kernel<T, V, SrcF>), dim3(rows), dim3(T), (unsigned)un.total * 8, ctx->stream, q, un,
                       SrcF{x}, gamma, beta, mean, rstd, dy, dx, beta_dx, part);
}
#define LNN_RES_CASES(p, F, ...)                                                        \
  switch ((p).T * 32 + (p).V) {                                                         \
    case 64 * 32 + 1: F<64, 1>(__VA_ARGS__); break;                                     \
    case 256 * 32 + 1: F<256, 1>(__VA_ARGS__); break;                                   \
    case 256 * 32 + 2: F<256, 2>(__VA_ARGS__); break;                                   \
    case 256 * 32 + 4: F<256, 4>(__VA_ARGS__); break;                                   \
    case 256 * 32 + 8: F<256, 8>(__VA_ARGS__); break;                                   \
    case 1024 * 32 + 1: F<1024, 1>(__VA_ARGS__); break;                                 \
    case 1024 * 32 + 2: F<1024, 2>(__VA_ARGS__); break;                                 \
    case 1024 * 32 + 4: F<1024, 4>(__VA_ARGS__); break;                                 \
    case 1024 * 32 + 8: F<1024, 8>(__VA_ARGS__); break;

// Lanes per row (L) and groups of four per lane (V) of the kernels for rows of channels alone; L = 0 where a row is longer.
struct RowPlan {
  int L, V;
};
static RowPlan row_plan(const NormGeom& q) {
  const int d = q.Cg;
  if (d <= 16) return {4, 1};
  if (d <= 64) return {16, 1};
  if (d <= 128) return {32, 1};
  if (d <= 256) return {64, 1};
  if (d <= 512) return {64, 2};
  if (d <= 1024) return {64, 4};
  if (d <= 2048) return {256, 2};
  if (d <= 4096) return {256, 4};
  if (d <= 8192) return {256, 8};
  return {0, 0};
}
#define LNN_ROW_CASES(p, F, ...)                                \
  switch ((p).L * 16 + (p).V) {                                 \
    case 4 * 16 + 1: F<4, 1>(__VA_ARGS__); break;               \
    case 16 * 16 + 1: F<16, 1>(__VA_ARGS__); break;             \
    case 32 * 16 + 1: F<32, 1>(__VA_ARGS__); break;             \
    case 64 * 16 + 1: F<64, 1>(__VA_ARGS__); break;             \
    case 64 * 16 + 2: F<64, 2>(__VA_ARGS__); break;             \
    case 64 * 16 + 4: F<64, 4>(__VA_ARGS__); break;             \
    case 256 * 16 + 2: F<256, 2>(__VA_ARGS__); break;           \
    case 256 * 16 + 4: F<256, 4>(__VA_ARGS__); break;           \
    default: F<256, 8>(__VA_ARGS__); break;                     \
  }
template <int L, int V>
static void fwd_rows(DeviceCtx* ctx, const NormGeom& q, const float* x, const float* gamma, const float* beta, float* y, float* mean,
                     float* rstd, uint8_t* codes, uint8_t* bytes) {
  const unsigned blocks = ((unsigned)(q.N * q.G) + 256 / L - 1) / (256 / L);   // a row has at least D / 4 lanes: below 2^24
  if (codes)
    hipLaunchKernelGGL((gn_fwd_rows_kernel<L, V, true>), dim3(blocks), dim3(256), 0, ctx->stream, q, x, gamma, beta, y, mean, rstd, codes, bytes);
  else
    hipLaunchKernelGGL((gn_fwd_rows_kernel<L, V, false>), dim3(blocks), dim3(256), 0, ctx->stream, q, x, gamma, beta, y, mean, rstd, codes, bytes);
}
template <int L, int V>
static void bwd_rows(DeviceCtx* ctx, const NormGeom& q, int chunks, const float* x, const uint8_t* codes, const uint8_t* bytes,
                     const float* gamma, const float* beta, const float* mean, const float* rstd, const float* dy, float* dx, int beta_dx,
                     float* part) {
  const unsigned blocks = (unsigned)chunks * q.G;
  if (codes)
    hipLaunchKernelGGL((gn_bwd_rows_kernel<L, V, Src8>), dim3(blocks), dim3(256), 0, ctx->stream, q, chunks, Src8{codes, bytes}, gamma, beta,
                       mean, rstd, dy, dx, beta_dx, part);
  else
    hipLaunchKernelGGL((gn_bwd_rows_kernel<L, V, SrcF>), dim3(blocks), dim3(256), 0, ctx->stream, q, chunks, SrcF{x}, gamma, beta, mean, rstd,
                       dy, dx, beta_dx, part);
}

// The tile of the channels-last kernels, and the chunks of either layout.
static LastTile last_tile(const DeviceCtx* ctx, const NormGeom& q) {
  LastTile t;
  const int cv = (q.C + 3) / 4;
  t.tx = cv < 256 ? cv : 256;
  t.slabs = (cv + 255) / 256;
  t.ty = 256 / t.tx;
  // a lane walks over 32 pixels, fewer where that leaves the chip short of workgroups
  int64_t per = 32;
  while (per > 4 && (int64_t)q.N * t.slabs * ((q.HW + t.ty * per - 1) / (t.ty * per)) < 4 * ctx->cus) per >>= 1;
  t.pix = (int)(t.ty * per);
  t.chunks = (q.HW + t.pix - 1) / t.pix;
  return t;
}
struct SplitPlan {
  LastTile t;
  int chunks, pix, images;   // images of one batch
  unsigned blocks;           // workgroups per image of the layout's kernels, in quarters of a workgroup channels first
};
static SplitPlan split_plan(const DeviceCtx* ctx, const NormGeom& q, int tensors) {
  SplitPlan s;
  s.t = last_tile(ctx, q);
  s.pix = q.last ? s.t.pix : kPlane;
  s.chunks = (q.HW + s.pix - 1) / s.pix;
  s.blocks = q.last ? (unsigned)s.t.slabs * s.chunks : (unsigned)q.C * s.chunks;
  // the tensors of one batch stay in the 256 MB memory-side cache until the second read; no grid reaches 2^32 threads
  const uint64_t image = (uint64_t)q.C * q.HW * 4 * tensors, cap = 160u << 20;
  uint64_t n = image >= cap ? 1 : cap / image;
  const uint64_t most = (1u << 23) / (s.blocks > (unsigned)q.G ? s.blocks : (unsigned)q.G);
  if (n > most) n = most > 0 ? most : 1;
  s.images = n < (uint64_t)q.N ? (int)n : q.N;
  return s;
}

int launch_group_norm_fwd(DeviceCtx* ctx, const lnn_group_norm_desc* d, const float* x, const float* gamma, const float* beta,
                          float* y, float* mean, float* rstd, void* x8) {
  NormGeom q;
  int st = make_geom(d, &q);
  if (st != LNN_OK) return st;
  const uint64_t n = (uint64_t)q.N * q.C * q.HW;
  // blocks of 32 lie inside a plane (channels first), a pixel's channels (last) or a row (one pixel): written on the way
  const bool whole = (!q.last ? q.HW : q.HW == 1 ? q.Cg : q.C) % 32 == 0;
  uint8_t* codes = x8 && whole ? static_cast<uint8_t*>(x8) : nullptr;
  uint8_t* bytes = codes ? codes + n : nullptr;
  ResPlan p;
  if (q.HW == 1 && row_plan(q).L) {
    LNN_ROW_CASES(row_plan(q), fwd_rows, ctx, q, x, gamma, beta, y, mean, rstd, codes, bytes)
  } else if (res_plan(ctx, q, 16, &p)) {
    for (; q.row0 < (uint32_t)(q.N * q.G); q.row0 += kMaxRows) {
      LNN_RES_CASES(p, fwd_res, ctx, q, p.un, x, gamma, beta, y, mean, rstd, codes, bytes)
        case 256 * 32 + 16: fwd_res<256, 16>(ctx, q, p.un, x, gamma, beta, y, mean, rstd, codes, bytes); break;
        default: fwd_res<1024, 16>(ctx, q, p.un, x, gamma, beta, y, mean, rstd, codes, bytes);
      }
    }
  } else {
    const SplitPlan s = split_plan(ctx, q, 2);
    st = ensure_workspace(ctx, (uint64_t)s.images * s.chunks * q.C * 8);
    if (st != LNN_OK) return st;
    float2* part = static_cast<float2*>(ctx->ws);
    for (; q.n0 < q.N; q.n0 += s.images) {
      q.nb = q.N - q.n0 < s.images ? q.N - q.n0 : s.images;
      const unsigned blocks = q.last ? q.nb * s.blocks : (q.nb * s.blocks + 3) / 4;
      if (q.last)
        hipLaunchKernelGGL(gn_stats_last_kernel, dim3(blocks), dim3(256), 0, ctx->stream, q, s.t, x, part);
      else
        hipLaunchKernelGGL(gn_stats_first_kernel, dim3(blocks), dim3(256), 0, ctx->stream, q, s.chunks, x, part);
      hipLaunchKernelGGL(gn_finish_kernel, dim3((unsigned)(q.nb * q.G)), dim3(256), 0, ctx->stream, q, s.chunks, s.pix, part, mean, rstd);
      if (q.last)
        hipLaunchKernelGGL(codes ? gn_apply_last_kernel<true> : gn_apply_last_kernel<false>, dim3(blocks), dim3(256), 0, ctx->stream, q, s.t, x,
                           gamma, beta, mean, rstd, y, codes, bytes);
      else
        hipLaunchKernelGGL(codes ? gn_apply_first_kernel<true> : gn_apply_first_kernel<false>, dim3(blocks), dim3(256), 0, ctx->stream, q,
                           s.chunks, x, gamma, beta, mean, rstd, y, codes, bytes);
    }
  }
  LNN_HIP(hipGetLastError());
  return x8 && !codes ? launch_encode8(ctx, n, x, x8) : LNN_OK;
}

template <class SRC>
static void bwd_split(DeviceCtx* ctx, NormGeom q, const SplitPlan& s, SRC x, const float* gamma, const float* beta, const float* mean,
                      const float* rstd, const float* dy, float* dx, int beta_dx, float* pa, float* pb, float2* s12) {
  for (; q.n0 < q.N; q.n0 += s.images) {
    q.nb = q.N - q.n0 < s.images ? q.N - q.n0 : s.images;
    const unsigned blocks = q.last ? q.nb * s.blocks : (q.nb * s.blocks + 3) / 4;
    if (q.last)
      hipLaunchKernelGGL((gn_sums_last_kernel<SRC>), dim3(blocks), dim3(256), 0, ctx->stream, q, s.t, x, gamma, beta, mean, rstd, dy, pa, pb);
    else
      hipLaunchKernelGGL((gn_sums_first_kernel<SRC>), dim3(blocks), dim3(256), 0, ctx->stream, q, s.chunks, x, gamma, beta, mean, rstd, dy, pa, pb);
    if (!dx) continue;
    hipLaunchKernelGGL(gn_finish_dx_kernel, dim3((unsigned)(q.nb * q.G)), dim3(256), 0, ctx->stream, q, s.chunks, gamma, pa, pb, s12);
    if (q.last)
      hipLaunchKernelGGL((gn_dx_last_kernel<SRC>), dim3(blocks), dim3(256), 0, ctx->stream, q, s.t, x, gamma, beta, mean, rstd, dy, s12, dx,
                         beta_dx);
    else
      hipLaunchKernelGGL((gn_dx_first_kernel<SRC>), dim3(blocks), dim3(256), 0, ctx->stream, q, s.chunks, x, gamma, beta, mean, rstd, dy, s12,
                         dx, beta_dx);
  }
}

int launch_group_norm_bwd(DeviceCtx* ctx, const lnn_group_norm_desc* d, const float* x, const void* x8, const float* gamma,
                          const float* beta, const float* mean, const float* rstd, const float* dy, float* dx, int beta_dx,
                          float* dgamma, int beta_dgamma, float* dbeta, int beta_dbeta) {
  NormGeom q;
  int st = make_geom(d, &q);
  if (st != LNN_OK) return st;
  if (!dx && !dgamma && !dbeta) return LNN_OK;
  const bool params = dgamma || dbeta;
  const uint8_t* codes = static_cast<const uint8_t*>(x8);
  const uint8_t* bytes = x8 ? codes + blocks8((uint64_t)q.N * q.C * q.HW) * 32 : nullptr;
  // K rows of channel sums, and room for the rows that many of them are first brought down to
  enum { kRows, kRes, kSplit } path;
  ResPlan p;
  SplitPlan s;
  uint64_t K;
  if (q.HW == 1 && row_plan(q).L) {
    path = kRows;
    const int slots = 256 / row_plan(q).L;   // four rows or more per slot, about eight workgroups per compute unit
    K = std::min<uint64_t>(((uint64_t)q.N + 4 * slots - 1) / (4 * slots), ((uint64_t)8 * ctx->cus + q.G - 1) / q.G);
  } else if (res_plan(ctx, q, 8, &p)) {
    path = kRes;
    K = q.N;
  } else {
    path = kSplit;
    s = split_plan(ctx, q, 3);
    K = (uint64_t)q.N * s.chunks;
  }
  const uint64_t per = std::max<uint64_t>(256, (K + 511) / 512), K2 = K > 512 ? (K + per - 1) / per : 0;
  const uint64_t sums = (params || path == kSplit) ? K * q.C : 0;
  st = ensure_workspace(ctx, (2 * sums + 2 * K2 * q.C + (path == kSplit ? 2 * (uint64_t)q.N * q.G : 0)) * 4 + 16);
  if (st != LNN_OK) return st;
  float* pa = sums ? static_cast<float*>(ctx->ws) : nullptr;
  float* pb = pa + sums;
  float* qa = pb + sums;
  float* qb = qa + K2 * q.C;
  float2* s12 = reinterpret_cast<float2*>(qb + K2 * q.C);   // an even number of floats behind the start
  if (path == kRows) {
    LNN_ROW_CASES(row_plan(q), bwd_rows, ctx, q, (int)K, x, codes, bytes, gamma, beta, mean, rstd, dy, dx, beta_dx, pa)
  } else if (path == kRes) {
    for (; q.row0 < (uint32_t)(q.N * q.G); q.row0 += kMaxRows) {
      LNN_RES_CASES(p, bwd_res, ctx, q, p.un, x, codes, bytes, gamma, beta, mean, rstd, dy, dx, beta_dx, pa)
      }
    }
  } else if (x8) {
    bwd_split(ctx, q, s, Src8{codes, bytes}, gamma, beta, mean, rstd, dy, dx, beta_dx, pa, pb, s12);
  } else {
    bwd_split(ctx, q, s, SrcF{x}, gamma, beta, mean, rstd, dy, dx, beta_dx, pa, pb, s12);
  }
  if (params) {
    const unsigned cols = (unsigned)((q.C + 31) / 32);
    if (K2) {
      hipLaunchKernelGGL(gn_params_kernel, dim3(cols, (unsigned)K2), dim3(256), 0, ctx->stream, (int)K, (int)per, q.C, pa, pb, qa, 0, qb, 0);
      pa = qa;
      pb = qb;
      K = K2;
    }
    hipLaunchKernelGGL(gn_params_kernel, dim3(cols, 1), dim3(256), 0, ctx->stream, (int)K, (int)K, q.C, pa, pb, dbeta, beta_dbeta, dgamma,
                       beta_dgamma);
  }
  LNN_HIP(hipGetLastError());
  return LNN_OK;
}

}  // namespace lnn
