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
#include "keep8.hpp"

namespace lnn {

struct NormGeom {
  int N, C, HW, G, Cg, last, act;
  float slope, eps, inv_d;
  uint32_t D, row0;   // row0: first row of this launch (a grid holds fewer than 2^32 threads)
  FastDiv dHW, dCg;
};

__device__ __forceinline__ float act_f(int act, float slope, float p) {
  if (act == LNN_ACT_LEAKY_RELU) return p >= 0.0f ? p : slope * p;
  if (act == LNN_ACT_SILU) return p / (1.0f + expf(-p));
  return p;
}
__device__ __forceinline__ float act_df(int act, float slope, float p) {
  if (act == LNN_ACT_LEAKY_RELU) return p >= 0.0f ? 1.0f : slope;
  if (act == LNN_ACT_SILU) {
    const float s = 1.0f / (1.0f + expf(-p));
    return s * (1.0f + p * (1.0f - s));
  }
  return 1.0f;
}

// element i of row (n, g): its channel, and its place in memory
__device__ __forceinline__ uint32_t row_elem(const NormGeom& q, uint32_t n, uint32_t g, uint32_t i, uint32_t* c) {
  if (q.last) {
    const uint32_t p = q.dCg.div(i);
    *c = g * q.Cg + (i - p * q.Cg);
    return (n * q.HW + p) * q.C + *c;
  }
  const uint32_t k = q.dHW.div(i);
  *c = g * q.Cg + k;
  return (n * q.G + g) * q.D + i;
}

// a source of x: fp32, or its 8-bit copy
struct XSrc {
  const float* x;
  const uint8_t* codes;
  const uint8_t* bytes;
  __device__ __forceinline__ float at(uint32_t i) const {
    return x ? x[i] : (float)(int8_t)codes[i] * step_of(bytes[i >> 5]);
  }
};

__device__ __forceinline__ float block_sum(float v, float* sh) {
#pragma unroll
  for (int w = 32; w > 0; w >>= 1) v += __shfl_xor(v, w, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return sh[0] + sh[1] + sh[2] + sh[3];
}

__global__ __launch_bounds__(256) void gn_stats_kernel(NormGeom q, const float* x, float* mean, float* rstd) {
  __shared__ float sh[4];
  const uint32_t n = blockIdx.x / q.G, g = blockIdx.x % q.G;
  uint32_t c;
  float s = 0.0f;
  for (uint32_t i = threadIdx.x; i < q.D; i += 256) s += x[row_elem(q, n, g, i, &c)];
  const float m = block_sum(s, sh) * q.inv_d;
  s = 0.0f;
  for (uint32_t i = threadIdx.x; i < q.D; i += 256) {
    const float d = x[row_elem(q, n, g, i, &c)] - m;
    s += d * d;
  }
  const float var = block_sum(s, sh) * q.inv_d;
  if (threadIdx.x == 0) {
    mean[blockIdx.x] = m;
    rstd[blockIdx.x] = 1.0f / sqrtf(var + q.eps);
  }
}

__global__ __launch_bounds__(256) void gn_apply_kernel(NormGeom q, const float* x, const float* gamma, const float* beta,
                                                       const float* mean, const float* rstd, float* y) {
  const uint32_t row = blockIdx.x, n = row / q.G, g = row % q.G;
  const float m = mean[row], r = rstd[row];
  for (uint32_t i = blockIdx.y * 256 + threadIdx.x; i < q.D; i += gridDim.y * 256) {
    uint32_t c;
    const uint32_t at = row_elem(q, n, g, i, &c);
    const float p = (x[at] - m) * r * (gamma ? gamma[c] : 1.0f) + (beta ? beta[c] : 0.0f);
    y[at] = act_f(q.act, q.slope, p);
  }
}

// sums over the pixels of (n, c): part[0][n][c] = sum dp, part[1][n][c] = sum dp xh
__global__ __launch_bounds__(256) void gn_bwd_sums_kernel(NormGeom q, XSrc x, const float* gamma, const float* beta,
                                                          const float* mean, const float* rstd, const float* dy, float* part) {
  __shared__ float sh[4];
  const uint32_t n = blockIdx.x / q.C, c = blockIdx.x % q.C, row = n * q.G + c / q.Cg;
  const float m = mean[row], r = rstd[row], ga = gamma ? gamma[c] : 1.0f, be = beta ? beta[c] : 0.0f;
  float s0 = 0.0f, s1 = 0.0f;
  for (uint32_t p = threadIdx.x; p < (uint32_t)q.HW; p += 256) {
    const uint32_t at = q.last ? (n * q.HW + p) * q.C + c : (n * q.C + c) * q.HW + p;
    const float xh = (x.at(at) - m) * r;
    const float dp = dy[at] * act_df(q.act, q.slope, xh * ga + be);
    s0 += dp;
    s1 += dp * xh;
  }
  s0 = block_sum(s0, sh);
  s1 = block_sum(s1, sh);
  if (threadIdx.x == 0) {
    part[blockIdx.x] = s0;
    part[(uint32_t)q.N * q.C + blockIdx.x] = s1;
  }
}

// row (n, g): sums over its channels of gamma times the two sums
__global__ __launch_bounds__(64) void gn_bwd_rows_kernel(NormGeom q, const float* gamma, const float* part, float* s12) {
  const uint32_t row = blockIdx.x, n = row / q.G, g = row % q.G;
  float a = 0.0f, b = 0.0f;
  for (int k = threadIdx.x; k < q.Cg; k += 64) {
    const uint32_t c = g * q.Cg + k, at = n * q.C + c;
    const float ga = gamma ? gamma[c] : 1.0f;
    a += ga * part[at];
    b += ga * part[(uint32_t)q.N * q.C + at];
  }
#pragma unroll
  for (int w = 32; w > 0; w >>= 1) {
    a += __shfl_xor(a, w, 64);
    b += __shfl_xor(b, w, 64);
  }
  if (threadIdx.x == 0) {
    s12[2 * row] = a * q.inv_d;
    s12[2 * row + 1] = b * q.inv_d;
  }
}

__global__ __launch_bounds__(256) void gn_bwd_apply_kernel(NormGeom q, XSrc x, const float* gamma, const float* beta,
                                                           const float* mean, const float* rstd, const float* dy,
                                                           const float* s12, float* dx, int beta_dx) {
  const uint32_t row = blockIdx.x, n = row / q.G, g = row % q.G;
  const float m = mean[row], r = rstd[row], s1 = s12[2 * row], s2 = s12[2 * row + 1];
  for (uint32_t i = blockIdx.y * 256 + threadIdx.x; i < q.D; i += gridDim.y * 256) {
    uint32_t c;
    const uint32_t at = row_elem(q, n, g, i, &c);
    const float ga = gamma ? gamma[c] : 1.0f, be = beta ? beta[c] : 0.0f;
    const float xh = (x.at(at) - m) * r;
    const float gp = ga * dy[at] * act_df(q.act, q.slope, xh * ga + be);
    const float v = r * (gp - s1 - xh * s2);
    dx[at] = beta_dx ? dx[at] + v : v;
  }
}

// dgamma, dbeta: the sums of (n, c) over n, in order
__global__ __launch_bounds__(256) void gn_bwd_params_kernel(int N, int C, const float* part, float* dgamma, int beta_dgamma,
                                                            float* dbeta, int beta_dbeta) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  float a = 0.0f, b = 0.0f;
  for (int n = 0; n < N; ++n) {
    a += part[(uint32_t)n * C + c];
    b += part[(uint32_t)(N + n) * C + c];
  }
  if (dbeta) dbeta[c] = beta_dbeta ? dbeta[c] + a : a;
  if (dgamma) dgamma[c] = beta_dgamma ? dgamma[c] + b : b;
}

// Four elements of x (or fewer at the end of a plane: cnt), from fp32 memory or from the 8-bit copy.
struct SrcF {
  const float* x;
  __device__ __forceinline__ void load(uint32_t at, int cnt, float* v) const { load4(x, at, cnt, v); }
  static __device__ __forceinline__ void load4(const float* p, uint32_t at, int cnt, float* v) {
    if (cnt == 4) {
      const F4 f = *reinterpret_cast<const F4*>(p + at);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = f.v[k];
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = k < cnt ? p[at + k] : 0.0f;
    }
  }
};
struct Src8 {
  const uint8_t* codes;
  const uint8_t* bytes;
  __device__ __forceinline__ void load(uint32_t at, int cnt, float* v) const {
    uint32_t q = 0;
    if (cnt == 4) {
      q = reinterpret_cast<const B4*>(codes + at)->v;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) q |= k < cnt ? (uint32_t)codes[at + k] << (8 * k) : 0u;
    }
    if (cnt > 0) {   // four elements lie in one block, or in two
      const float s0 = step_of(bytes[at >> 5]), s1 = step_of(bytes[(at + cnt - 1) >> 5]);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = code_at(q, k) * (((at + k) >> 5) == (at >> 5) ? s0 : s1);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = 0.0f;
    }
  }
};
__device__ __forceinline__ void store4(float* p, uint32_t at, int cnt, const float* v) {
  if (cnt == 4) {
    F4 f;
#pragma unroll
    for (int k = 0; k < 4; ++k) f.v[k] = v[k];
    *reinterpret_cast<F4*>(p + at) = f;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < cnt) p[at + k] = v[k];
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
        for (int k = 0; k < 4; ++k) o[k] = act_f(q.act, q.slope, (v[i][k] - m) * r * ga + be);
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
      float a = 0.0f, b = 0.0f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float h = k < p.cnt ? (xh[i][k] - m) * r : 0.0f;
        const float d = dp[i][k] * act_df(q.act, q.slope, h * ga + be);
        a += d;
        b += d * h;
        xh[i][k] = h;
        dp[i][k] = d * ga;
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
  q->N = d->N;
  q->C = d->C;
  q->HW = d->HW;
  q->G = d->groups;
  q->Cg = d->C / d->groups;
  q->last = d->channels_last != 0;
  q->act = d->act;
  q->slope = d->slope;
  q->eps = d->eps;
  q->row0 = 0;
  q->D = (uint32_t)q->Cg * (uint32_t)q->HW;
  q->inv_d = (float)(1.0 / (double)q->D);
  q->dHW = make_fastdiv((uint32_t)q->HW);
  q->dCg = make_fastdiv((uint32_t)q->Cg);
  return LNN_OK;
}

static dim3 row_grid(const NormGeom& q) {
  uint32_t parts = (q.D + 2047) / 2048;
  if (parts > 64) parts = 64;
  return dim3((unsigned)(q.N * q.G), parts);
}

// How a row is dealt out to a workgroup's lanes; false where it does not fit `most` groups of four per lane.
struct ResPlan {
  Units un;
  int T, V;
};
static bool res_plan(const DeviceCtx* ctx, const NormGeom& q, int most, ResPlan* p) {
  if (q.last && q.HW > 1) return false;
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

int launch_group_norm_fwd(DeviceCtx* ctx, const lnn_group_norm_desc* d, const float* x, const float* gamma, const float* beta,
                          float* y, float* mean, float* rstd, void* x8) {
  NormGeom q;
  int st = make_geom(d, &q);
  if (st != LNN_OK) return st;
  ResPlan p;
  if (res_plan(ctx, q, 16, &p)) {
    uint8_t* codes = (x8 && q.HW % 32 == 0) ? static_cast<uint8_t*>(x8) : nullptr;
    uint8_t* bytes = codes ? codes + (uint64_t)q.N * q.C * q.HW : nullptr;
    for (; q.row0 < (uint32_t)(q.N * q.G); q.row0 += kMaxRows) {
    LNN_RES_CASES(p, fwd_res, ctx, q, p.un, x, gamma, beta, y, mean, rstd, codes, bytes)
    case 256 * 32 + 16: fwd_res<256, 16>(ctx, q, p.un, x, gamma, beta, y, mean, rstd, codes, bytes); break;
    default: fwd_res<1024, 16>(ctx, q, p.un, x, gamma, beta, y, mean, rstd, codes, bytes);
    }
    }
    LNN_HIP(hipGetLastError());
    return x8 && !codes ? launch_encode8(ctx, (uint64_t)q.N * q.C * q.HW, x, x8) : LNN_OK;
  }
  hipLaunchKernelGGL(gn_stats_kernel, dim3((unsigned)(q.N * q.G)), dim3(256), 0, ctx->stream, q, x, mean, rstd);
  hipLaunchKernelGGL(gn_apply_kernel, row_grid(q), dim3(256), 0, ctx->stream, q, x, gamma, beta, mean, rstd, y);
  LNN_HIP(hipGetLastError());
  return x8 ? launch_encode8(ctx, (uint64_t)q.N * q.C * q.HW, x, x8) : LNN_OK;
}

int launch_group_norm_bwd(DeviceCtx* ctx, const lnn_group_norm_desc* d, const float* x, const void* x8, const float* gamma,
                          const float* beta, const float* mean, const float* rstd, const float* dy, float* dx, int beta_dx,
                          float* dgamma, int beta_dgamma, float* dbeta, int beta_dbeta) {
  NormGeom q;
  int st = make_geom(d, &q);
  if (st != LNN_OK) return st;
  if (!dx && !dgamma && !dbeta) return LNN_OK;
  const uint64_t nc = (uint64_t)q.N * q.C;
  st = ensure_workspace(ctx, (2 * nc + 2 * (uint64_t)q.N * q.G) * 4);
  if (st != LNN_OK) return st;
  float* part = static_cast<float*>(ctx->ws);
  float* s12 = part + 2 * nc;
  XSrc src = {x, static_cast<const uint8_t*>(x8), nullptr};
  if (x8) src.bytes = src.codes + blocks8(nc * q.HW) * 32;
  ResPlan p;
  if (res_plan(ctx, q, 8, &p)) {
    float* sums = (dgamma || dbeta) ? part : nullptr;
    for (; q.row0 < (uint32_t)(q.N * q.G); q.row0 += kMaxRows) {
    LNN_RES_CASES(p, bwd_res, ctx, q, p.un, x, src.codes, src.bytes, gamma, beta, mean, rstd, dy, dx, beta_dx, sums)
    }
    }
    if (sums)
      hipLaunchKernelGGL(gn_bwd_params_kernel, dim3((unsigned)((q.C + 255) / 256)), dim3(256), 0, ctx->stream, q.N, q.C, part, dgamma,
                         beta_dgamma, dbeta, beta_dbeta);
    LNN_HIP(hipGetLastError());
    return LNN_OK;
  }
  hipLaunchKernelGGL(gn_bwd_sums_kernel, dim3((unsigned)nc), dim3(256), 0, ctx->stream, q, src, gamma, beta, mean, rstd, dy, part);
  if (dx) {
    hipLaunchKernelGGL(gn_bwd_rows_kernel, dim3((unsigned)(q.N * q.G)), dim3(64), 0, ctx->stream, q, gamma, part, s12);
    hipLaunchKernelGGL(gn_bwd_apply_kernel, row_grid(q), dim3(256), 0, ctx->stream, q, src, gamma, beta, mean, rstd, dy, s12, dx,
                       beta_dx);
  }
  if (dgamma || dbeta)
    hipLaunchKernelGGL(gn_bwd_params_kernel, dim3((unsigned)((q.C + 255) / 256)), dim3(256), 0, ctx->stream, q.N, q.C, part, dgamma,
                       beta_dgamma, dbeta, beta_dbeta);
  LNN_HIP(hipGetLastError());
  return LNN_OK;
}

}  // namespace lnn
