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
  uint32_t D;
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

int launch_group_norm_fwd(DeviceCtx* ctx, const lnn_group_norm_desc* d, const float* x, const float* gamma, const float* beta,
                          float* y, float* mean, float* rstd, void* x8) {
  NormGeom q;
  int st = make_geom(d, &q);
  if (st != LNN_OK) return st;
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
