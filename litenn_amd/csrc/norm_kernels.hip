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
#include <type_traits>

#include "keep8.hpp"

namespace lnn {

struct NormGeom {
  int N, C, HW, G, Cg, last, silu;
  int n0, nb;           // images of this launch
  float slope, eps;
  float d, inv_d;       // D and 1 / D
  uint32_t D, size;     // elements of a row and of the tensor
  uint32_t row0;        // first row of this launch (a grid holds fewer than 2^32 threads)
};

// 1 / (1 + exp(-p)) by the one-instruction power of two and reciprocal (one unit in the last place each).  Rounding
// -p log2(e) and the constant costs up to |p| (2^-24 + 2^-26) of exp(-p) besides: 3.7e-7 at |p| = 5, and where |p| is
// large the result is next to 0 or 1.
// The library's expf and a full division take five times the vector work, and these kernels then wait for it, not for memory.
__device__ __forceinline__ float sigmoid(float p) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(p * -1.44269504088896341f));
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
      d[k] *= fmaf(p[k] * s, 1.0f - s, s);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) d[k] = p[k] >= 0.0f ? d[k] : slope * d[k];
  }
}

// ---- a whole row in registers (channels first, row contiguous) ------------------------------------------------------
//
// One workgroup per row reads it once: a lane holds V groups of four elements, and mean, variance and result come from
// registers.  512 lanes: two rows or more to a compute unit, so that one is read while another is computed or written
// (32 x 256 x 56 x 56 from 8 bits, forward + backward: 116 us against 130 with 1024 lanes and one row); 1024 where there are
// fewer rows than compute units.  The loads of a row stand together, in front of everything that waits for them (67 -> 61 us).
// Bound: memory.  32 x 128 x 56 x 56 forward 22 us, 4.7 TB/s; forward + backward with SiLU 61 us, 4.2 TB/s.
//
// The row is dealt out in units of 2^ul lanes, each unit inside one channel plane (4 * 2^ul elements of it),
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
  r.ch = un.dper.div(u);
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

// Computes a value anew where it is used next, instead of holding it in a register until then.
__device__ __forceinline__ uint32_t anew(uint32_t v) {
  asm volatile("" : "+v"(v));
  return v;
}
// gamma and beta of a group in LDS (ones and zeros where there are none): the first T channels' are asked for before the
// row, so that waiting for them does not wait for it.
struct Affine {
  float g, b;
};
template <int T>
__device__ __forceinline__ Affine ask_affine(const NormGeom& q, uint32_t c0, const float* gamma, const float* beta) {
  const uint32_t ch = min((int)threadIdx.x, q.Cg - 1);
  return {gamma ? gamma[c0 + ch] : 1.0f, beta ? beta[c0 + ch] : 0.0f};
}
template <int T>
__device__ __forceinline__ void keep_affine(const NormGeom& q, uint32_t c0, const float* gamma, const float* beta, const Affine& a, float* lg) {
  if ((int)threadIdx.x < q.Cg) {
    lg[threadIdx.x] = a.g;
    lg[q.Cg + threadIdx.x] = a.b;
  }
  for (int ch = threadIdx.x + T; ch < q.Cg; ch += T) {
    lg[ch] = gamma ? gamma[c0 + ch] : 1.0f;
    lg[q.Cg + ch] = beta ? beta[c0 + ch] : 0.0f;
  }
}

template <int T, int V, int MODE, bool KEEP>
__global__ __launch_bounds__(T) void gn_fwd_res_kernel(NormGeom q, Units un, const float* x, const float* gamma, const float* beta,
                                                       float* y, float* mean, float* rstd, uint8_t* codes, uint8_t* bytes) {
  extern __shared__ float lg[];   // [2][Cg]
  __shared__ float sh[2][T / 64];
  const uint32_t row = q.row0 + blockIdx.x, base = row * q.D, c0 = (row % q.G) * q.Cg;
  const uint32_t lane = threadIdx.x & ((1u << un.ul) - 1), u0 = threadIdx.x >> un.ul;
  const int step = T >> un.ul;
  const Affine af = ask_affine<T>(q, c0, gamma, beta);
  float v[V][4];
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const UnitPos p = unit_pos(q, un, i * step + u0, lane);   // no test whether the units end: the loads stay together
    load4<MODE>(x, base + p.at, p.cnt, q.size, v[i]);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int k = 0; k < 4; ++k) s += v[i][k];
  }
  keep_affine<T>(q, c0, gamma, beta, af, lg);
  const float m = sum_all<T>(s, sh[0]) / q.d;
  s = 0.0f;
  const uint32_t u1 = anew(u0);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (i * step < un.total) {
      const UnitPos p = unit_pos(q, un, i * step + u1, lane);
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
  const uint32_t u2 = anew(u0);
  if (T == 64) __syncthreads();   // gamma and beta are in LDS: larger workgroups have passed a barrier since
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (i * step < un.total) {
      const UnitPos p = unit_pos(q, un, i * step + u2, lane);
      if (KEEP) {   // planes are whole blocks of 32: the eight lanes of a block are all in or all out
        uint32_t byte;
        const uint32_t code = encode_lane4(v[i], &byte);
        if (p.cnt == 4) {
          reinterpret_cast<B4*>(codes + base + p.at)->v = code;
          if ((lane & 7) == 0) bytes[(base + p.at) >> 5] = (uint8_t)byte;
        }
      }
      if (p.cnt > 0) {
        const float ga = lg[p.ch], be = lg[q.Cg + p.ch];
        float o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = (v[i][k] - m) * r * ga + be;
        act4(q.silu, q.slope, o);
        store4(y, base + p.at, p.cnt, o);
      }
    }
  }
}

// What a lane keeps of four elements of x between the two uses: the values, or where they lie in one block the codes and
// their step, which leaves room for twice the rows on a compute unit.
struct HoldF {
  float v[4];
  __device__ __forceinline__ float get(int k) const { return v[k]; }
};
struct Hold8 {
  uint32_t q;
  float s;
  __device__ __forceinline__ float get(int k) const { return code_at(q, k) * s; }
};
template <int MODE, class SRC>
__device__ __forceinline__ void hold4(const SRC& x, uint32_t at, int cnt, uint32_t size, HoldF* h) {
  x.template load<MODE>(at, cnt, size, h->v);
}
template <int MODE>
__device__ __forceinline__ void hold4(const Src8& x, uint32_t at, int cnt, uint32_t size, Hold8* h) {
  h->q = load_codes<MODE>(x.codes, at, cnt, size);
  h->s = step_of(x.bytes[cnt > 0 ? at >> 5 : 0u]);
}

// Both sums of a unit are formed by lane exchanges and left in LDS; the channel sums are theirs in order, so nothing
// depends on which wavefront came first.  part (or null): [2][N][C], the channel sums of dp and of dp xh.
template <int T, int V, int MODE, class SRC, class HOLD>
__global__ __launch_bounds__(T, T == 512 ? 4 : 1) void gn_bwd_res_kernel(NormGeom q, Units un, SRC x, const float* gamma, const float* beta,
                                                                         const float* mean, const float* rstd, const float* dy, float* dx,
                                                                         int beta_dx, float* part) {
  extern __shared__ float su[];   // [units][2], then gamma and beta [2][Cg]
  float* lg = su + 2 * un.total;
  __shared__ float sh[2][T / 64];
  const uint32_t row = q.row0 + blockIdx.x, base = row * q.D, n = row / q.G, c0 = (row % q.G) * q.Cg;
  const uint32_t lane = threadIdx.x & ((1u << un.ul) - 1), u0 = threadIdx.x >> un.ul;
  const int step = T >> un.ul;
  const float m = mean[row], r = rstd[row];
  const Affine af = ask_affine<T>(q, c0, gamma, beta);
  HOLD xv[V];
  float dp[V][4];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const UnitPos p = unit_pos(q, un, i * step + u0, lane);   // no test whether the units end: the loads stay together
    hold4<MODE>(x, base + p.at, p.cnt, q.size, &xv[i]);
    load4<MODE>(dy, base + p.at, p.cnt, q.size, dp[i]);
  }
  keep_affine<T>(q, c0, gamma, beta, af, lg);
  __syncthreads();
  const uint32_t u1 = anew(u0);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (i * step < un.total) {
      const uint32_t u = i * step + u1;
      const UnitPos p = unit_pos(q, un, u, lane);
      const uint32_t ch = min(p.ch, (uint32_t)q.Cg - 1);
      const float ga = lg[ch], be = lg[q.Cg + ch];
      float a = 0.0f, b = 0.0f, xh[4], pre[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        xh[k] = k < p.cnt ? (xv[i].get(k) - m) * r : 0.0f;
        pre[k] = xh[k] * ga + be;
      }
      slope4(q.silu, q.slope, pre, dp[i]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        a += dp[i][k];
        b += dp[i][k] * xh[k];
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
    const float ga = lg[ch];
    s1 += ga * a;
    s2 += ga * b;
  }
  if (!dx) return;
  s1 = sum_all<T>(s1, sh[0]) * q.inv_d;
  s2 = sum_all<T>(s2, sh[1]) * q.inv_d;
  const uint32_t u2 = anew(u0);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (i * step < un.total) {
      const UnitPos p = unit_pos(q, un, i * step + u2, lane);
      if (p.cnt > 0) {
        float o[4];
        if (beta_dx) load4<MODE>(dx, base + p.at, p.cnt, q.size, o);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float e = r * (dp[i][k] - s1 - (xv[i].get(k) - m) * r * s2);
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
// 8192 x 4096 in 32 groups, forward + backward: 142 us, 4.8 TB/s of the 5.0 that a large copy reaches.
template <int L>
__device__ __forceinline__ float sum_lanes(float v, float* sh) {
#pragma unroll
  for (int w = (L < 64 ? L : 64) / 2; w > 0; w >>= 1) v += __shfl_xor(v, w, 64);
  if (L <= 64) return v;
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return sh[0] + sh[1] + sh[2] + sh[3];
}

template <int L, int V, int MODE, bool KEEP>
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
    load4<MODE>(x, base + (i * L + lane) * 4, cnt[i], q.size, v[i]);
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) s += v[i][k];
  const float m = sum_lanes<L>(s, sh[0]) / q.d;
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
      if (gamma) load4<MODE>(gamma, c0 + (i * L + lane) * 4, cnt[i], q.C, ga);
      if (beta) load4<MODE>(beta, c0 + (i * L + lane) * 4, cnt[i], q.C, be);
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
template <int L, int V, int MODE, class SRC>
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
    if (gamma) load4<MODE>(gamma, c0 + (i * L + lane) * 4, cnt[i], q.C, ga[i]);
    if (beta) load4<MODE>(beta, c0 + (i * L + lane) * 4, cnt[i], q.C, be[i]);
  }
  for (int nn = n0; nn < n1; nn += S) {   // all lanes together: the row sums may cross wavefronts
    const int n = nn + (int)slot;
    const bool in = n < n1;
    const uint32_t row = (uint32_t)(in ? n : n0) * q.G + g, base = row * q.D;
    const float m = mean[row], r = rstd[row];
    float xh[V][4], dp[V][4], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x.template load<MODE>(base + (i * L + lane) * 4, in ? cnt[i] : 0, q.size, xh[i]);
      load4<MODE>(dy, base + (i * L + lane) * 4, in ? cnt[i] : 0, q.size, dp[i]);
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
        if (beta_dx) load4<MODE>(dx, at, c, q.size, o);
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

// ---- channels last, small problems ------------------------------------------------------------------------------------
//
// One workgroup per row again, element by element: a lane keeps one channel of the group and every PT-th pixel.  The row's
// pieces of Cg floats make poor use of memory lines, but one launch does it: for tensors up to a megaelement, which the
// caches hold, three launches (three more backward) take longer than their lines (3 x 37 x 41 x 60, step: 25 -> 20 us).
// Pixels per lane by the row's length: pixels that a lane does not have are read all the same (20 pixels x 160 channels, forward /
// backward kernel: four to a lane 4.0 / 4.0 us, eight 4.4 / 4.7).
template <int T, int V>
__global__ __launch_bounds__(T) void gn_fwd_gather_kernel(NormGeom q, int pt, const float* x, const float* gamma, const float* beta, float* y,
                                                          float* mean, float* rstd) {
  __shared__ float sh[2][T / 64];
  const uint32_t row = blockIdx.x, n = row / q.G, g = row % q.G;
  const int pl = threadIdx.x / q.Cg, c = g * q.Cg + ((int)threadIdx.x - pl * q.Cg);
  const int p0 = pl < pt ? pl : q.HW;   // lanes behind the last whole set of channels have no pixels
  float v[V], s = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = x[(n * q.HW + min(p0 + i * pt, q.HW - 1)) * q.C + c];
  const float ga = gamma ? gamma[c] : 1.0f, be = beta ? beta[c] : 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) s += p0 + i * pt < q.HW ? v[i] : 0.0f;
  const float m = sum_all<T>(s, sh[0]) / q.d;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float d = p0 + i * pt < q.HW ? v[i] - m : 0.0f;
    s += d * d;
  }
  const float r = 1.0f / sqrtf(sum_all<T>(s, sh[1]) * q.inv_d + q.eps);
  if (threadIdx.x == 0) {
    mean[row] = m;
    rstd[row] = r;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (p0 + i * pt < q.HW) {
      const float p = (v[i] - m) * r * ga + be;
      y[(n * q.HW + p0 + i * pt) * q.C + c] = q.silu ? p * sigmoid(p) : p >= 0.0f ? p : q.slope * p;
    }
  }
}

template <int T, int V, class SRC>
__global__ __launch_bounds__(T) void gn_bwd_gather_kernel(NormGeom q, int pt, SRC x, const float* gamma, const float* beta, const float* mean,
                                                          const float* rstd, const float* dy, float* dx, int beta_dx, float* part) {
  __shared__ float sh[2][T / 64], ch[2][T];
  const uint32_t row = blockIdx.x, n = row / q.G, g = row % q.G;
  const int pl = threadIdx.x / q.Cg, c = g * q.Cg + ((int)threadIdx.x - pl * q.Cg);
  const int p0 = pl < pt ? pl : q.HW;
  const float m = mean[row], r = rstd[row];
  float v[V], d[V], a = 0.0f, b = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const uint32_t at = (n * q.HW + min(p0 + i * pt, q.HW - 1)) * q.C + c;
    v[i] = x.at(at);
    d[i] = dy[at];
  }
  const float ga = gamma ? gamma[c] : 1.0f, be = beta ? beta[c] : 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const bool in = p0 + i * pt < q.HW;
    v[i] = (v[i] - m) * r;
    const float p = v[i] * ga + be;
    if (q.silu) {
      const float s = sigmoid(p);
      d[i] *= fmaf(p * s, 1.0f - s, s);
    } else {
      d[i] = p >= 0.0f ? d[i] : q.slope * d[i];
    }
    a += in ? d[i] : 0.0f;
    b += in ? d[i] * v[i] : 0.0f;
  }
  if (part) {   // over the pixel lanes of a channel, in halves
    ch[0][threadIdx.x] = a;
    ch[1][threadIdx.x] = b;
    for (int h = pt; h > 1;) {
      const int half = (h + 1) >> 1;
      __syncthreads();
      if (pl + half < h) {
        ch[0][threadIdx.x] += ch[0][threadIdx.x + half * q.Cg];
        ch[1][threadIdx.x] += ch[1][threadIdx.x + half * q.Cg];
      }
      h = half;
    }
    if (pl == 0) {
      part[n * q.C + c] = ch[0][threadIdx.x];
      part[(uint32_t)(q.N + n) * q.C + c] = ch[1][threadIdx.x];
    }
  }
  if (!dx) return;
  const float s1 = sum_all<T>(a * ga, sh[0]) * q.inv_d, s2 = sum_all<T>(b * ga, sh[1]) * q.inv_d;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (p0 + i * pt < q.HW) {
      float* o = dx + (n * q.HW + p0 + i * pt) * q.C + c;
      const float e = r * (d[i] * ga - s1 - v[i] * s2);
      *o = beta_dx ? *o + e : e;
    }
  }
}

// ---- rows too long for registers, and channels last -----------------------------------------------------------------
//
// Three launches: sums per channel and chunk of pixels, the rows' statistics from them, the result.  x is read twice; the
// second time from its end backwards, where what the first reading left in the 256 MB memory-side cache still is.
// Taking the images in batches that fit that cache was slower (16 x 128 x 128 x 256 forward: 276 us in batches of 96 MB, 208 of
// 160 MB, 166 in one): the cache saves less than each batch's three short launches cost.
// 16 x 128 x 128 x 256 forward 162 us = 824 MB at 5.1 TB/s; 8 x 64 x 64 x 320 step from 8 bits 85 us.
//
// Means and sums of squared distances of two sets join as
//   n = na + nb, d = mb - ma:  m = ma + d nb / n,  M = Ma + Mb + d^2 na nb / n
struct Stat {
  float n, m, M;
};
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b) {
  const float n = a.n + b.n;
  if (n == 0.0f) return a;
  const float f = b.n * __builtin_amdgcn_rcpf(n), d = b.m - a.m;
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
// back: last image first
__device__ __forceinline__ PlanePos plane_pos(const NormGeom& q, int chunks, bool back) {
  const uint32_t w = (back ? gridDim.x - 1 - blockIdx.x : blockIdx.x) * 4 + (threadIdx.x >> 6);
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

template <int MODE>
__global__ __launch_bounds__(256) void gn_stats_first_kernel(NormGeom q, int chunks, const float* x, float2* part) {
  const PlanePos p = plane_pos(q, chunks, false);
  if (!p.in) return;
  const int lane = threadIdx.x & 63;
  float v[16][4], s = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    load4<MODE>(x, p.base + i * 256 + lane * 4, min(max(p.count - i * 256 - lane * 4, 0), 4), q.size, v[i]);
#pragma unroll
  for (int i = 0; i < 16; ++i)
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

template <int MODE, bool KEEP>
__global__ __launch_bounds__(256) void gn_apply_first_kernel(NormGeom q, int chunks, const float* x, const float* gamma, const float* beta,
                                                             const float* mean, const float* rstd, float* y, uint8_t* codes,
                                                             uint8_t* bytes) {
  const PlanePos p = plane_pos(q, chunks, true);
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
      load4<MODE>(x, p.base + i0 + j * 256 + lane * 4, cnt[j], q.size, v[j]);
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

template <int MODE, class SRC>
__global__ __launch_bounds__(256) void gn_sums_first_kernel(NormGeom q, int chunks, SRC x, const float* gamma, const float* beta,
                                                            const float* mean, const float* rstd, const float* dy, float* pa, float* pb) {
  const PlanePos p = plane_pos(q, chunks, false);
  if (!p.in) return;
  const int lane = threadIdx.x & 63;
  const uint32_t row = p.n * q.G + p.c / q.Cg;
  const float m = mean[row], r = rstd[row], ga = gamma ? gamma[p.c] : 1.0f, be = beta ? beta[p.c] : 0.0f;
  float a = 0.0f, b = 0.0f;
  for (int i0 = 0; i0 < p.count; i0 += 1024) {   // four groups in flight
    float v[4][4], d[4][4], pre[4];
    int cnt[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      cnt[j] = min(max(p.count - i0 - j * 256 - lane * 4, 0), 4);
      x.template load<MODE>(p.base + i0 + j * 256 + lane * 4, cnt[j], q.size, v[j]);
      load4<MODE>(dy, p.base + i0 + j * 256 + lane * 4, cnt[j], q.size, d[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[j][k] = k < cnt[j] ? (v[j][k] - m) * r : 0.0f;
        pre[k] = v[j][k] * ga + be;
      }
      slope4(q.silu, q.slope, pre, d[j]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        a += d[j][k];
        b += d[j][k] * v[j][k];
      }
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

template <int MODE, class SRC>
__global__ __launch_bounds__(256) void gn_dx_first_kernel(NormGeom q, int chunks, SRC x, const float* gamma, const float* beta,
                                                          const float* mean, const float* rstd, const float* dy, const float2* s12,
                                                          float* dx, int beta_dx) {
  const PlanePos p = plane_pos(q, chunks, true);
  if (!p.in) return;
  const int lane = threadIdx.x & 63;
  const uint32_t row = p.n * q.G + p.c / q.Cg;
  const float m = mean[row], r = rstd[row], ga = gamma ? gamma[p.c] : 1.0f, be = beta ? beta[p.c] : 0.0f;
  const float2 s = s12[row];
  for (int i0 = 0; i0 < p.count; i0 += 1024) {
    float v[4][4], d[4][4], pre[4];
    int cnt[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      cnt[j] = min(max(p.count - i0 - j * 256 - lane * 4, 0), 4);
      x.template load<MODE>(p.base + i0 + j * 256 + lane * 4, cnt[j], q.size, v[j]);
      load4<MODE>(dy, p.base + i0 + j * 256 + lane * 4, cnt[j], q.size, d[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t at = p.base + i0 + j * 256 + lane * 4;
      float o[4];
      if (beta_dx) load4<MODE>(dx, at, cnt[j], q.size, o);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[j][k] = (v[j][k] - m) * r;
        pre[k] = v[j][k] * ga + be;
      }
      slope4(q.silu, q.slope, pre, d[j]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float e = r * (d[j][k] * ga - s.x - v[j][k] * s.y);
        o[k] = beta_dx ? o[k] + e : e;
      }
      store4(dx, at, cnt[j], o);
    }
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
__device__ __forceinline__ LastPos last_pos(const NormGeom& q, const LastTile& t, bool back) {
  LastPos p;
  const uint32_t w = back ? gridDim.x - 1 - blockIdx.x : blockIdx.x, slab = w % t.slabs, k = w / t.slabs;
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

template <int MODE>
__global__ __launch_bounds__(256) void gn_stats_last_kernel(NormGeom q, LastTile t, const float* x, float2* part) {
  __shared__ float sm[4][256], sM[4][256], sn[256];
  const LastPos p = last_pos(q, t, false);
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
        load4<MODE>(x, (p.n * q.HW + pix) * q.C + p.c, in ? p.cnt : 0, q.size, v[i]);
      }
      const float inv = __builtin_amdgcn_rcpf((float)nv);
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
// T lanes: 1024 where a row has more channel-chunks than one walk of 256 (2 x 22263 x 54 in one group, step: 99 -> 57 us)
template <int T>
__global__ __launch_bounds__(T) void gn_finish_kernel(NormGeom q, int chunks, int pix, const float2* part, float* mean, float* rstd) {
  __shared__ Stat sh[T / 64];
  const uint32_t n = blockIdx.x / q.G, g = blockIdx.x % q.G;   // n: image of the batch
  Stat s = {0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int j = threadIdx.x; j < chunks * q.Cg; j += T) {
    const int chunk = j / q.Cg, c = j - chunk * q.Cg;
    const float2 e = part[(n * chunks + chunk) * q.C + g * q.Cg + c];
    s = join(s, Stat{(float)min(pix, q.HW - chunk * pix), e.x, e.y});
  }
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) {
    const Stat o = {__shfl_down(s.n, w, 64), __shfl_down(s.m, w, 64), __shfl_down(s.M, w, 64)};
    s = join(s, o);   // lane 0's tree is the only one that counts
  }
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = sh[0];
#pragma unroll
    for (int w = 1; w < T / 64; ++w) s = join(s, sh[w]);
    const uint32_t row = (q.n0 + n) * q.G + g;
    mean[row] = s.m;
    rstd[row] = 1.0f / sqrtf(s.M * q.inv_d + q.eps);
  }
}

// What a lane's four channels need: their rows' mean and rstd (four channels may span groups), gamma and beta
struct LaneRows {
  float m[4], r[4], ga[4], be[4];
};
__device__ __forceinline__ void lane_rows(const NormGeom& q, const LastPos& p, const float* gamma, const float* beta, const float* mean,
                                          const float* rstd, LaneRows* l) {
  uint32_t c[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    c[k] = k < p.cnt ? p.c + k : 0;
    const uint32_t row = p.n * q.G + c[k] / q.Cg;
    l->m[k] = mean[row];
    l->r[k] = rstd[row];
    l->ga[k] = 1.0f;
    l->be[k] = 0.0f;
  }
  if (gamma) {
#pragma unroll
    for (int k = 0; k < 4; ++k) l->ga[k] = gamma[c[k]];
  }
  if (beta) {
#pragma unroll
    for (int k = 0; k < 4; ++k) l->be[k] = beta[c[k]];
  }
}

template <int MODE, bool KEEP>
__global__ __launch_bounds__(256) void gn_apply_last_kernel(NormGeom q, LastTile t, const float* x, const float* gamma, const float* beta,
                                                            const float* mean, const float* rstd, float* y, uint8_t* codes, uint8_t* bytes) {
  const LastPos p = last_pos(q, t, true);
  LaneRows l;
  lane_rows(q, p, gamma, beta, mean, rstd, &l);
  for (int pix0 = p.p0 + p.y; pix0 < p.p1; pix0 += 4 * t.ty) {   // four loads in flight
    float v[4][4];
    int cnt[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int pix = pix0 + j * t.ty;
      cnt[j] = pix < p.p1 ? p.cnt : 0;
      load4<MODE>(x, (p.n * q.HW + pix) * q.C + p.c, cnt[j], q.size, v[j]);
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

template <int MODE, class SRC>
__global__ __launch_bounds__(256) void gn_sums_last_kernel(NormGeom q, LastTile t, SRC x, const float* gamma, const float* beta,
                                                           const float* mean, const float* rstd, const float* dy, float* pa, float* pb) {
  __shared__ float sh[8][256];
  const LastPos p = last_pos(q, t, false);
  LaneRows l;
  lane_rows(q, p, gamma, beta, mean, rstd, &l);
  float a[4] = {}, b[4] = {};
  for (int pix0 = p.p0 + p.y; pix0 < p.p1; pix0 += 4 * t.ty) {   // four pixels in flight
    float v[4][4], d[4][4], pre[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int pix = pix0 + j * t.ty, cnt = pix < p.p1 ? p.cnt : 0;
      x.template load<MODE>((p.n * q.HW + pix) * q.C + p.c, cnt, q.size, v[j]);
      load4<MODE>(dy, (p.n * q.HW + pix) * q.C + p.c, cnt, q.size, d[j]);   // 0 where there is no pixel
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[j][k] = (v[j][k] - l.m[k]) * l.r[k];
        pre[k] = v[j][k] * l.ga[k] + l.be[k];
      }
      slope4(q.silu, q.slope, pre, d[j]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        a[k] += d[j][k];
        b[k] += d[j][k] * v[j][k];
      }
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

template <int MODE, class SRC>
__global__ __launch_bounds__(256) void gn_dx_last_kernel(NormGeom q, LastTile t, SRC x, const float* gamma, const float* beta,
                                                         const float* mean, const float* rstd, const float* dy, const float2* s12,
                                                         float* dx, int beta_dx) {
  const LastPos p = last_pos(q, t, true);
  LaneRows l;
  lane_rows(q, p, gamma, beta, mean, rstd, &l);
  float s1[4], s2[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 s = s12[p.n * q.G + (k < p.cnt ? p.c + k : 0) / q.Cg];
    s1[k] = s.x;
    s2[k] = s.y;
  }
  for (int pix0 = p.p0 + p.y; pix0 < p.p1; pix0 += 4 * t.ty) {
    float v[4][4], d[4][4], pre[4];
    int cnt[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int pix = pix0 + j * t.ty;
      cnt[j] = pix < p.p1 ? p.cnt : 0;
      x.template load<MODE>((p.n * q.HW + pix) * q.C + p.c, cnt[j], q.size, v[j]);
      load4<MODE>(dy, (p.n * q.HW + pix) * q.C + p.c, cnt[j], q.size, d[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t at = (p.n * q.HW + pix0 + j * t.ty) * q.C + p.c;
      float o[4];
      if (beta_dx) load4<MODE>(dx, at, cnt[j], q.size, o);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[j][k] = (v[j][k] - l.m[k]) * l.r[k];
        pre[k] = v[j][k] * l.ga[k] + l.be[k];
      }
      slope4(q.silu, q.slope, pre, d[j]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float e = l.r[k] * (d[j][k] * l.ga[k] - s1[k] - v[j][k] * s2[k]);
        o[k] = beta_dx ? o[k] + e : e;
      }
      store4(dx, at, cnt[j], o);
    }
  }
}

// Column sums of the K rows of pa and pb: a workgroup takes 32 channels and the rows [k0, k1), 8 lanes per channel walk over
// them, then add up in order: lanes behind the first 256 only pass the barrier, so the bits do not depend on the launch.
__device__ __forceinline__ void column_sums(uint32_t block, int k0, int k1, int C, const float* pa, const float* pb, float* outa, int beta_a,
                                            float* outb, int beta_b) {
  constexpr int S = 8;
  __shared__ float sh[2][S][33];
  const int li = threadIdx.x & 31, lk = threadIdx.x >> 5, c = block * 32 + li;
  float a = 0.0f, b = 0.0f;
  if (c < C && lk < S) {
#pragma unroll 4
    for (int k = k0 + lk; k < k1; k += S) {
      a += pa[(uint32_t)k * C + c];
      b += pb[(uint32_t)k * C + c];
    }
  }
  if (lk < S) {
    sh[0][lk][li] = a;
    sh[1][lk][li] = b;
  }
  __syncthreads();
  if (lk == 0 && c < C) {
#pragma unroll
    for (int k = 1; k < S; ++k) {
      a += sh[0][k][li];
      b += sh[1][k][li];
    }
    if (outa) outa[c] = beta_a ? outa[c] + a : a;
    if (outb) outb[c] = beta_b ? outb[c] + b : b;
  }
}

// row (n, g): s1 and s2 from the sums of its channels and chunks.  Workgroups behind the rows form dbeta and dgamma from the
// K rows of the same sums, in the launch that is there anyway.
template <int T>
__global__ __launch_bounds__(T) void gn_finish_dx_kernel(NormGeom q, int chunks, const float* gamma, const float* pa, const float* pb,
                                                           float2* s12, int K, float* dgamma, int beta_dgamma, float* dbeta, int beta_dbeta) {
  __shared__ float sh[2][T / 64];
  const uint32_t rows = (uint32_t)q.nb * q.G;
  if (blockIdx.x >= rows) {
    column_sums(blockIdx.x - rows, 0, K, q.C, pa, pb, dbeta, beta_dbeta, dgamma, beta_dgamma);
    return;
  }
  const uint32_t n = q.n0 + blockIdx.x / q.G, g = blockIdx.x % q.G;
  float a = 0.0f, b = 0.0f;
  for (int j = threadIdx.x; j < chunks * q.Cg; j += T) {
    const int chunk = j / q.Cg, c = g * q.Cg + (j - chunk * q.Cg);
    const float ga = gamma ? gamma[c] : 1.0f;
    a += ga * pa[(n * chunks + chunk) * q.C + c];
    b += ga * pb[(n * chunks + chunk) * q.C + c];
  }
  a = sum_all<T>(a, sh[0]);
  b = sum_all<T>(b, sh[1]);
  if (threadIdx.x == 0) s12[n * q.G + g] = make_float2(a * q.inv_d, b * q.inv_d);
}

// dbeta, dgamma; with gridDim.y > 1 the sums over `per` rows each, left as rows of outa / outb for a second launch
__global__ __launch_bounds__(256) void gn_params_kernel(int K, int per, int C, const float* pa, const float* pb, float* outa, int beta_a,
                                                        float* outb, int beta_b) {
  const int k0 = blockIdx.y * per;
  const uint64_t at = (uint64_t)blockIdx.y * C;
  column_sums(blockIdx.x, k0, min(k0 + per, K), C, pa, pb, outa ? outa + at : nullptr, beta_a, outb ? outb + at : nullptr, beta_b);
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
  q->last = (d->channels_last != 0 && d->C > 1) || d->HW == 1;   // with one channel or one pixel the two layouts are one
  q->n0 = 0;
  q->nb = d->N;
  q->silu = d->act == LNN_ACT_SILU;
  q->slope = d->act == LNN_ACT_NONE ? 1.0f : d->slope;
  q->eps = d->eps;
  q->row0 = 0;
  q->size = (uint32_t)((uint64_t)d->N * d->C * d->HW);
  q->D = (uint32_t)q->Cg * (uint32_t)q->HW;
  q->d = (float)q->D;
  q->inv_d = (float)(1.0 / (double)q->D);
  return LNN_OK;
}

// ---- which kernel runs ------------------------------------------------------------------------------------------------
//
// The variants that are built: lanes and groups of four per lane, for a gathered row pixels per lane.  Plans pick from these lists
// and launches switch over them, so that no plan can name a kernel that does not exist.
#define LNN_RES_BWD(X)                                                                                 \
  X(64, 1) X(256, 1) X(256, 2) X(256, 3) X(256, 4)                                                     \
  X(512, 3) X(512, 4) X(512, 5) X(512, 6) X(512, 7) X(512, 8) X(512, 10) X(512, 13)                    \
  X(1024, 2) X(1024, 3) X(1024, 4) X(1024, 5) X(1024, 6) X(1024, 7) X(1024, 8)
#define LNN_RES_FWD(X) LNN_RES_BWD(X) X(512, 16) X(1024, 10) X(1024, 13) X(1024, 16)
#define LNN_ROWS(X) X(4, 1) X(16, 1) X(32, 1) X(64, 1) X(64, 2) X(64, 4) X(256, 2) X(256, 4) X(256, 8)
#define LNN_GATHER(X) X(256, 1) X(256, 4) X(256, 8) X(256, 16) X(1024, 4) X(1024, 8) X(1024, 16)

struct Variant {
  int T, V;
};
#define LNN_VARIANT(T, V) {T, V},
static const Variant kResBwd[] = {LNN_RES_BWD(LNN_VARIANT)};
static const Variant kResFwd[] = {LNN_RES_FWD(LNN_VARIANT)};
static const Variant kRows[] = {LNN_ROWS(LNN_VARIANT)};
static const Variant kGather[] = {LNN_GATHER(LNN_VARIANT)};
#undef LNN_VARIANT

struct NormPlan {
  int path;    // LNN_NORM_PATH_*
  int T, V;    // of the path's list; 0 for the split kernels
  int pt;      // gathered rows: pixels that the lanes hold at a time
  Units un;    // rows in registers
};

// A row in registers; most, most512: groups per lane at 1024 and at 512 lanes.
template <int N>
static bool res_plan(const Variant (&list)[N], int cus, const NormGeom& q, int most, int most512, NormPlan* p) {
  if (q.last) return false;
  // the shortest unit that holds a plane, or whole wavefronts
  p->un.ul = q.HW <= 4 ? 0 : q.HW <= 16 ? 2 : q.HW <= 64 ? 4 : 6;
  p->un.per = ((q.HW + 3) / 4 + (1 << p->un.ul) - 1) >> p->un.ul;
  const uint64_t units = (uint64_t)q.Cg * p->un.per, lanes = units << p->un.ul;
  if (lanes > 1024u * most || units > 3500) return false;   // 3500: two sums per unit, gamma and beta in 64 KB of LDS
  p->un.total = (int)units;
  p->un.dper = make_fastdiv((uint32_t)p->un.per);
  int T = lanes <= 64 ? 64 : lanes <= 1024 ? 256 : lanes <= 512u * most512 ? 512 : 1024;
  if (lanes > 1024 && q.N * q.G <= cus) T = 1024;   // fewer rows than compute units: more lanes to each
  for (const Variant& v : list)
    if (v.T == T && lanes <= (uint64_t)v.T * v.V) {
      p->T = v.T;
      p->V = v.V;
      return true;
    }
  return false;
}

// kept: x is read from its 8-bit copy (backward)
static NormPlan norm_plan(int cus, const NormGeom& q, bool backward, bool kept) {
  NormPlan p = {};
  if (q.HW == 1) {
    for (const Variant& v : kRows)
      if (q.Cg <= 4 * v.T * v.V) {
        p.path = LNN_NORM_PATH_ROWS;
        p.T = v.T;
        p.V = v.V;
        return p;
      }
  }
  if (backward ? res_plan(kResBwd, cus, q, 8, q.HW % 4 != 0 ? 8 : kept ? 13 : 10, &p)
               : res_plan(kResFwd, cus, q, q.HW % 4 == 0 ? 16 : 13, 16, &p)) {
    p.path = LNN_NORM_PATH_ROW_IN_REGISTERS;
    return p;
  }
  if (q.last && q.HW > 1 && q.Cg <= 256 && q.size <= 1u << 20) {
    for (const Variant& v : kGather)
      if ((int64_t)(v.T / q.Cg) * v.V >= q.HW) {
        p.path = LNN_NORM_PATH_GATHERED_ROW;
        p.T = v.T;
        p.V = v.V;
        p.pt = v.T / q.Cg;
        return p;
      }
  }
  p.path = LNN_NORM_PATH_SPLIT;
  return p;
}

int group_norm_path(const lnn_group_norm_desc* d, int backward, int kept, int cus, int* path, int32_t* info) {
  if (!path || cus < 1) return set_error(LNN_ERR_INVALID, "group_norm_path: null pointer or no compute units");
  NormGeom q;
  const int st = make_geom(d, &q);
  if (st != LNN_OK) return st;
  const NormPlan p = norm_plan(cus, q, backward != 0, kept != 0);
  *path = p.path;
  if (info) {
    info[0] = p.T;
    info[1] = p.V;
  }
  return LNN_OK;
}

constexpr uint32_t kMaxRows = 1u << 21;   // of one launch

static unsigned rows_of_launch(const NormGeom& q) { return std::min((uint32_t)(q.N * q.G) - q.row0, kMaxRows); }

// Planes that are not whole groups of four take GANY, a tensor of fewer than four elements GTINY.  8-bit copies are written on
// the way (codes) only where planes are whole blocks of 32.
template <int T, int V>
static void fwd_res(DeviceCtx* ctx, const NormGeom& q, const Units& un, const float* x, const float* gamma, const float* beta, float* y,
                    float* mean, float* rstd, uint8_t* codes, uint8_t* bytes) {
  auto kernel = gn_fwd_res_kernel<T, V, GANY, false>;
  if (codes)
    kernel = gn_fwd_res_kernel<T, V, G4, true>;
  else if (q.HW % 4 == 0)
    kernel = gn_fwd_res_kernel<T, V, G4, false>;
  if constexpr (T == 64) {
    if (q.size < 4) kernel = gn_fwd_res_kernel<T, V, GTINY, false>;
  }
  hipLaunchKernelGGL(kernel, dim3(rows_of_launch(q)), dim3(T), (unsigned)q.Cg * 8, ctx->stream, q, un, x, gamma, beta, y, mean, rstd, codes,
                     bytes);
}
template <int T, int V, class SRC>
static void bwd_res_from(DeviceCtx* ctx, const NormGeom& q, const Units& un, SRC x, const float* gamma, const float* beta, const float* mean,
                         const float* rstd, const float* dy, float* dx, int beta_dx, float* part) {
  // groups of four lie in one block of a copy where planes are whole groups
  using Hold = std::conditional_t<std::is_same_v<SRC, Src8>, Hold8, HoldF>;
  auto kernel = gn_bwd_res_kernel<T, V, GANY, SRC, HoldF>;
  if (q.HW % 4 == 0) kernel = gn_bwd_res_kernel<T, V, G4, SRC, Hold>;
  if constexpr (T == 64) {
    if (q.size < 4) kernel = gn_bwd_res_kernel<T, V, GTINY, SRC, HoldF>;
  }
  hipLaunchKernelGGL(kernel, dim3(rows_of_launch(q)), dim3(T), (unsigned)(un.total + q.Cg) * 8, ctx->stream, q, un, x, gamma, beta, mean, rstd,
                     dy, dx, beta_dx, part);
}
template <int T, int V>
static void bwd_res(DeviceCtx* ctx, const NormGeom& q, const Units& un, const float* x, const uint8_t* codes, const uint8_t* bytes,
                    const float* gamma, const float* beta, const float* mean, const float* rstd, const float* dy, float* dx, int beta_dx,
                    float* part) {
  if (codes)
    bwd_res_from<T, V>(ctx, q, un, Src8{codes, bytes}, gamma, beta, mean, rstd, dy, dx, beta_dx, part);
  else
    bwd_res_from<T, V>(ctx, q, un, SrcF{x}, gamma, beta, mean, rstd, dy, dx, beta_dx, part);
}

template <int L, int V>
static void fwd_rows(DeviceCtx* ctx, const NormGeom& q, const float* x, const float* gamma, const float* beta, float* y, float* mean,
                     float* rstd, uint8_t* codes, uint8_t* bytes) {
  auto kernel = gn_fwd_rows_kernel<L, V, GANY, false>;
  if (codes)
    kernel = gn_fwd_rows_kernel<L, V, G4, true>;
  else if (q.Cg % 4 == 0)
    kernel = gn_fwd_rows_kernel<L, V, G4, false>;
  if constexpr (L == 4) {
    if (q.C < 4) kernel = gn_fwd_rows_kernel<L, V, GTINY, false>;
  }
  const unsigned blocks = ((unsigned)(q.N * q.G) + 256 / L - 1) / (256 / L);   // a row has at least D / 4 lanes: below 2^24
  hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, ctx->stream, q, x, gamma, beta, y, mean, rstd, codes, bytes);
}
template <int L, int V, class SRC>
static void bwd_rows_from(DeviceCtx* ctx, const NormGeom& q, int chunks, SRC x, const float* gamma, const float* beta, const float* mean,
                          const float* rstd, const float* dy, float* dx, int beta_dx, float* part) {
  auto kernel = gn_bwd_rows_kernel<L, V, GANY, SRC>;
  if (q.Cg % 4 == 0) kernel = gn_bwd_rows_kernel<L, V, G4, SRC>;
  if constexpr (L == 4) {
    if (q.C < 4) kernel = gn_bwd_rows_kernel<L, V, GTINY, SRC>;
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)chunks * q.G), dim3(256), 0, ctx->stream, q, chunks, x, gamma, beta, mean, rstd, dy, dx, beta_dx,
                     part);
}
template <int L, int V>
static void bwd_rows(DeviceCtx* ctx, const NormGeom& q, int chunks, const float* x, const uint8_t* codes, const uint8_t* bytes,
                     const float* gamma, const float* beta, const float* mean, const float* rstd, const float* dy, float* dx, int beta_dx,
                     float* part) {
  if (codes)
    bwd_rows_from<L, V>(ctx, q, chunks, Src8{codes, bytes}, gamma, beta, mean, rstd, dy, dx, beta_dx, part);
  else
    bwd_rows_from<L, V>(ctx, q, chunks, SrcF{x}, gamma, beta, mean, rstd, dy, dx, beta_dx, part);
}

template <int T, int V>
static void fwd_gather(DeviceCtx* ctx, const NormGeom& q, int pt, const float* x, const float* gamma, const float* beta, float* y, float* mean,
                       float* rstd) {
  hipLaunchKernelGGL((gn_fwd_gather_kernel<T, V>), dim3((unsigned)(q.N * q.G)), dim3(T), 0, ctx->stream, q, pt, x, gamma, beta, y, mean, rstd);
}
template <int T, int V>
static void bwd_gather(DeviceCtx* ctx, const NormGeom& q, int pt, const float* x, const uint8_t* codes, const uint8_t* bytes, const float* gamma,
                       const float* beta, const float* mean, const float* rstd, const float* dy, float* dx, int beta_dx, float* part) {
  const dim3 grid((unsigned)(q.N * q.G)), block(T);
  if (codes)
    hipLaunchKernelGGL((gn_bwd_gather_kernel<T, V, Src8>), grid, block, 0, ctx->stream, q, pt, Src8{codes, bytes}, gamma, beta, mean, rstd, dy,
                       dx, beta_dx, part);
  else
    hipLaunchKernelGGL((gn_bwd_gather_kernel<T, V, SrcF>), grid, block, 0, ctx->stream, q, pt, SrcF{x}, gamma, beta, mean, rstd, dy, dx,
                       beta_dx, part);
}

// The tile of the channels-last kernels, and the chunks of either layout.
static LastTile last_tile(const DeviceCtx* ctx, const NormGeom& q, int most) {
  LastTile t;
  const int cv = (q.C + 3) / 4;
  t.tx = cv < 256 ? cv : 256;
  t.slabs = (cv + 255) / 256;
  t.ty = 256 / t.tx;
  // a lane walks over `most` pixels, fewer where that leaves the chip short of workgroups
  int64_t per = most;
  while (per > 4 && (int64_t)q.N * t.slabs * ((q.HW + t.ty * per - 1) / (t.ty * per)) < 4 * ctx->cus) per >>= 1;
  t.pix = (int)(t.ty * per);
  t.chunks = (q.HW + t.pix - 1) / t.pix;
  return t;
}
struct SplitPlan {
  LastTile sum, out;         // channels last: tiles of the sums and of the result
  int chunks, pix, images;   // of the sums; images of one batch
  unsigned sum_blocks, out_blocks;   // workgroups per image (channels first: quarters of one)
};
static SplitPlan split_plan(const DeviceCtx* ctx, const NormGeom& q) {
  SplitPlan s;
  s.sum = last_tile(ctx, q, 32);
  s.out = last_tile(ctx, q, 8);
  s.pix = q.last ? s.sum.pix : kPlane;
  s.chunks = (q.HW + s.pix - 1) / s.pix;
  s.sum_blocks = q.last ? (unsigned)s.sum.slabs * s.chunks : (unsigned)q.C * s.chunks;
  s.out_blocks = q.last ? (unsigned)s.out.slabs * s.out.chunks : (unsigned)q.C * s.chunks;
  const uint64_t most = (1u << 21) / std::max({s.sum_blocks, s.out_blocks, (unsigned)q.G});   // no grid reaches 2^32 threads
  s.images = (int)std::max<uint64_t>(1, std::min<uint64_t>(q.N, most));
  return s;
}

static bool whole_fours(const NormGeom& q) { return (q.last ? q.C : q.HW) % 4 == 0; }
// The rows' sums are finished by 1024 lanes where a row has more channel-chunks than one walk of 256 lanes
static bool wide_finish(const NormGeom& q, const SplitPlan& s) { return s.chunks * q.Cg > 256; }
static unsigned split_blocks(const NormGeom& q, unsigned per_image) { return q.last ? q.nb * per_image : (q.nb * per_image + 3) / 4; }

// No tensor of fewer than four elements comes here.
static void fwd_split(DeviceCtx* ctx, NormGeom q, const SplitPlan& s, const float* x, const float* gamma, const float* beta, float* mean,
                      float* rstd, float* y, uint8_t* codes, uint8_t* bytes, float2* part) {
  const bool four = whole_fours(q), wide = wide_finish(q, s);
  auto finish = wide ? gn_finish_kernel<1024> : gn_finish_kernel<256>;
  for (; q.n0 < q.N; q.n0 += s.images) {
    q.nb = std::min(q.N - q.n0, s.images);
    const dim3 sums(split_blocks(q, s.sum_blocks)), results(split_blocks(q, s.out_blocks)), rows((unsigned)(q.nb * q.G)), block(256);
    if (q.last) {
      auto stats = four ? gn_stats_last_kernel<G4> : gn_stats_last_kernel<GANY>;
      hipLaunchKernelGGL(stats, sums, block, 0, ctx->stream, q, s.sum, x, part);
    } else {
      auto stats = four ? gn_stats_first_kernel<G4> : gn_stats_first_kernel<GANY>;
      hipLaunchKernelGGL(stats, sums, block, 0, ctx->stream, q, s.chunks, x, part);
    }
    hipLaunchKernelGGL(finish, rows, dim3(wide ? 1024 : 256), 0, ctx->stream, q, s.chunks, s.pix, part, mean, rstd);
    if (q.last) {
      auto apply = four ? gn_apply_last_kernel<G4, false> : gn_apply_last_kernel<GANY, false>;
      if (codes) apply = gn_apply_last_kernel<G4, true>;
      hipLaunchKernelGGL(apply, results, block, 0, ctx->stream, q, s.out, x, gamma, beta, mean, rstd, y, codes, bytes);
    } else {
      auto apply = four ? gn_apply_first_kernel<G4, false> : gn_apply_first_kernel<GANY, false>;
      if (codes) apply = gn_apply_first_kernel<G4, true>;
      hipLaunchKernelGGL(apply, results, block, 0, ctx->stream, q, s.chunks, x, gamma, beta, mean, rstd, y, codes, bytes);
    }
  }
}

int launch_group_norm_fwd(DeviceCtx* ctx, const lnn_group_norm_desc* d, const float* x, const float* gamma, const float* beta,
                          float* y, float* mean, float* rstd, void* x8) {
  NormGeom q;
  int st = make_geom(d, &q);
  if (st != LNN_OK) return st;
  const uint64_t n = (uint64_t)q.N * q.C * q.HW;
  const NormPlan p = norm_plan(ctx->cus, q, false, false);
  // blocks of 32 lie inside a plane (channels first), a pixel's channels (last) or a row (one pixel): written on the way
  const bool whole = p.path != LNN_NORM_PATH_GATHERED_ROW && (!q.last ? q.HW : q.HW == 1 ? q.Cg : q.C) % 32 == 0;
  uint8_t* codes = x8 && whole ? static_cast<uint8_t*>(x8) : nullptr;
  uint8_t* bytes = codes ? codes + n : nullptr;
  if (p.path == LNN_NORM_PATH_ROWS) {
#define LNN_LAUNCH(L, V) \
  case L * 32 + V: fwd_rows<L, V>(ctx, q, x, gamma, beta, y, mean, rstd, codes, bytes); break;
    switch (p.T * 32 + p.V) { LNN_ROWS(LNN_LAUNCH) }
#undef LNN_LAUNCH
  } else if (p.path == LNN_NORM_PATH_GATHERED_ROW) {
#define LNN_LAUNCH(T, V) \
  case T * 32 + V: fwd_gather<T, V>(ctx, q, p.pt, x, gamma, beta, y, mean, rstd); break;
    switch (p.T * 32 + p.V) { LNN_GATHER(LNN_LAUNCH) }
#undef LNN_LAUNCH
  } else if (p.path == LNN_NORM_PATH_ROW_IN_REGISTERS) {
#define LNN_LAUNCH(T, V) \
  case T * 32 + V: fwd_res<T, V>(ctx, q, p.un, x, gamma, beta, y, mean, rstd, codes, bytes); break;
    for (; q.row0 < (uint32_t)(q.N * q.G); q.row0 += kMaxRows) {
      switch (p.T * 32 + p.V) { LNN_RES_FWD(LNN_LAUNCH) }
    }
#undef LNN_LAUNCH
  } else {
    const SplitPlan s = split_plan(ctx, q);
    st = ensure_workspace(ctx, (uint64_t)s.images * s.chunks * q.C * 8);
    if (st != LNN_OK) return st;
    fwd_split(ctx, q, s, x, gamma, beta, mean, rstd, y, codes, bytes, static_cast<float2*>(ctx->ws));
  }
  LNN_HIP(hipGetLastError());
  return x8 && !codes ? launch_encode8(ctx, n, x, x8) : LNN_OK;
}

// Where the channel sums go: K rows of them are added up in the launch that finishes the rows' sums (0: in one of its own)
struct ChannelSums {
  int K;
  float* dgamma;
  int beta_dgamma;
  float* dbeta;
  int beta_dbeta;
};
template <class SRC>
static void bwd_split(DeviceCtx* ctx, NormGeom q, const SplitPlan& s, SRC x, const float* gamma, const float* beta, const float* mean,
                      const float* rstd, const float* dy, float* dx, int beta_dx, float* pa, float* pb, float2* s12, const ChannelSums& c) {
  const bool four = whole_fours(q), wide = wide_finish(q, s);
  auto finish = wide ? gn_finish_dx_kernel<1024> : gn_finish_dx_kernel<256>;
  for (; q.n0 < q.N; q.n0 += s.images) {
    q.nb = std::min(q.N - q.n0, s.images);
    const dim3 sums(split_blocks(q, s.sum_blocks)), results(split_blocks(q, s.out_blocks)), block(256);
    if (q.last) {
      auto kernel = four ? gn_sums_last_kernel<G4, SRC> : gn_sums_last_kernel<GANY, SRC>;
      hipLaunchKernelGGL(kernel, sums, block, 0, ctx->stream, q, s.sum, x, gamma, beta, mean, rstd, dy, pa, pb);
    } else {
      auto kernel = four ? gn_sums_first_kernel<G4, SRC> : gn_sums_first_kernel<GANY, SRC>;
      hipLaunchKernelGGL(kernel, sums, block, 0, ctx->stream, q, s.chunks, x, gamma, beta, mean, rstd, dy, pa, pb);
    }
    if (!dx) continue;
    const dim3 rows((unsigned)(q.nb * q.G + (c.K ? (q.C + 31) / 32 : 0)));
    hipLaunchKernelGGL(finish, rows, dim3(wide ? 1024 : 256), 0, ctx->stream, q, s.chunks, gamma, pa, pb, s12, c.K, c.dgamma, c.beta_dgamma,
                       c.dbeta, c.beta_dbeta);
    if (q.last) {
      auto kernel = four ? gn_dx_last_kernel<G4, SRC> : gn_dx_last_kernel<GANY, SRC>;
      hipLaunchKernelGGL(kernel, results, block, 0, ctx->stream, q, s.out, x, gamma, beta, mean, rstd, dy, s12, dx, beta_dx);
    } else {
      auto kernel = four ? gn_dx_first_kernel<G4, SRC> : gn_dx_first_kernel<GANY, SRC>;
      hipLaunchKernelGGL(kernel, results, block, 0, ctx->stream, q, s.chunks, x, gamma, beta, mean, rstd, dy, s12, dx, beta_dx);
    }
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
  const NormPlan p = norm_plan(ctx->cus, q, true, x8 != nullptr);
  const bool split = p.path == LNN_NORM_PATH_SPLIT;
  // K rows of channel sums, and room for the rows that many of them are first brought down to
  SplitPlan s;
  uint64_t K = q.N;
  if (p.path == LNN_NORM_PATH_ROWS) {
    const int slots = 256 / p.T;   // four rows or more per slot, about eight workgroups per compute unit
    K = std::min<uint64_t>(((uint64_t)q.N + 4 * slots - 1) / (4 * slots), ((uint64_t)8 * ctx->cus + q.G - 1) / q.G);
  } else if (split) {
    s = split_plan(ctx, q);
    K = (uint64_t)q.N * s.chunks;
  }
  const uint64_t per = std::max<uint64_t>(256, (K + 511) / 512), K2 = K > 512 ? (K + per - 1) / per : 0;
  const uint64_t sums = (params || split) ? K * q.C : 0;
  st = ensure_workspace(ctx, (2 * sums + 2 * K2 * q.C + (split ? 2 * (uint64_t)q.N * q.G : 0)) * 4 + 16);
  if (st != LNN_OK) return st;
  float* pa = sums ? static_cast<float*>(ctx->ws) : nullptr;
  float* pb = pa + sums;
  float* qa = pb + sums;
  float* qb = qa + K2 * q.C;
  float2* s12 = reinterpret_cast<float2*>(qb + K2 * q.C);   // an even number of floats behind the start
  // dgamma and dbeta in the launch that finishes the rows' sums, where there is one such launch
  const bool with = params && split && dx && K2 == 0 && s.images == q.N;
  if (p.path == LNN_NORM_PATH_ROWS) {
#define LNN_LAUNCH(L, V) \
  case L * 32 + V: bwd_rows<L, V>(ctx, q, (int)K, x, codes, bytes, gamma, beta, mean, rstd, dy, dx, beta_dx, pa); break;
    switch (p.T * 32 + p.V) { LNN_ROWS(LNN_LAUNCH) }
#undef LNN_LAUNCH
  } else if (p.path == LNN_NORM_PATH_ROW_IN_REGISTERS) {
#define LNN_LAUNCH(T, V) \
  case T * 32 + V: bwd_res<T, V>(ctx, q, p.un, x, codes, bytes, gamma, beta, mean, rstd, dy, dx, beta_dx, pa); break;
    for (; q.row0 < (uint32_t)(q.N * q.G); q.row0 += kMaxRows) {
      switch (p.T * 32 + p.V) { LNN_RES_BWD(LNN_LAUNCH) }
    }
#undef LNN_LAUNCH
  } else if (p.path == LNN_NORM_PATH_GATHERED_ROW) {
#define LNN_LAUNCH(T, V) \
  case T * 32 + V: bwd_gather<T, V>(ctx, q, p.pt, x, codes, bytes, gamma, beta, mean, rstd, dy, dx, beta_dx, pa); break;
    switch (p.T * 32 + p.V) { LNN_GATHER(LNN_LAUNCH) }
#undef LNN_LAUNCH
  } else {
    const ChannelSums c = {with ? (int)K : 0, dgamma, beta_dgamma, dbeta, beta_dbeta};
    if (x8)
      bwd_split(ctx, q, s, Src8{codes, bytes}, gamma, beta, mean, rstd, dy, dx, beta_dx, pa, pb, s12, c);
    else
      bwd_split(ctx, q, s, SrcF{x}, gamma, beta, mean, rstd, dy, dx, beta_dx, pa, pb, s12, c);
  }
  if (params && !with) {
    const unsigned cols = (unsigned)((q.C + 31) / 32);
    if (K2) {
      hipLaunchKernelGGL(gn_params_kernel, dim3(cols, (unsigned)K2), dim3(256), 0, ctx->stream, (int)K, (int)per, q.C, pa, pb, qa, 0, qb,
                         0);
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
