// Activations kept in 8 bits: writing them, reading them back, and the weight gradient of a dense layer from its kept
// input.  The element format is in keep8.hpp.
#include "keep8.hpp"

namespace lnn {

// One lane holds four elements and eight lanes a block, so the block's largest magnitude is three lane exchanges away.
// Elements behind n count as zeros; the codes of the last block's padding are written too.
__global__ __launch_bounds__(256) void encode8_kernel(uint32_t n, uint32_t groups, const float* src, uint8_t* dst) {
  uint8_t* bytes = dst + (uint64_t)groups * 4;
  for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < groups; i += gridDim.x * 256) {
    float v[4];
    if (4 * i + 3 < n) {
      const F4 f = *reinterpret_cast<const F4*>(src + 4 * i);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = f.v[k];
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = 4 * i + k < n ? src[4 * i + k] : 0.0f;
    }
    uint32_t byte;
    const uint32_t q = encode_lane4(v, &byte);
    reinterpret_cast<B4*>(dst + (uint64_t)4 * i)->v = q;
    if ((i & 7) == 0) bytes[i >> 3] = (uint8_t)byte;
  }
}

__global__ __launch_bounds__(256) void decode8_kernel(uint32_t n, uint32_t groups, const uint8_t* src, float* dst) {
  const uint8_t* bytes = src + (uint64_t)groups * 4;
  for (uint32_t i = blockIdx.x * 256 + threadIdx.x; 4 * i < n; i += gridDim.x * 256) {
    const uint32_t q = reinterpret_cast<const B4*>(src + (uint64_t)4 * i)->v;
    const float s = step_of(bytes[i >> 3]);
    if (4 * i + 3 < n) {
      F4 f;
#pragma unroll
      for (int k = 0; k < 4; ++k) f.v[k] = code_at(q, k) * s;
      *reinterpret_cast<F4*>(dst + 4 * i) = f;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (4 * i + k < n) dst[4 * i + k] = code_at(q, k) * s;
    }
  }
}

static dim3 grid8(const DeviceCtx* ctx, uint64_t lanes) {
  const uint64_t blocks = (lanes + 255) / 256, cap = (uint64_t)ctx->cus * 16;
  return dim3((unsigned)(blocks < cap ? blocks : cap));
}

int launch_encode8(DeviceCtx* ctx, uint64_t n, const float* src, void* dst) {
  const uint64_t groups = blocks8(n) * 8;
  hipLaunchKernelGGL(encode8_kernel, grid8(ctx, groups), dim3(256), 0, ctx->stream, (uint32_t)n, (uint32_t)groups, src,
                     static_cast<uint8_t*>(dst));
  LNN_HIP(hipGetLastError());
  return LNN_OK;
}

int launch_decode8(DeviceCtx* ctx, uint64_t n, const void* src, float* dst) {
  const uint64_t groups = blocks8(n) * 8;
  hipLaunchKernelGGL(decode8_kernel, grid8(ctx, groups), dim3(256), 0, ctx->stream, (uint32_t)n, (uint32_t)groups,
                     static_cast<const uint8_t*>(src), dst);
  LNN_HIP(hipGetLastError());
  return LNN_OK;
}

// dW[b][k][m] (+)= sum over rows of X8[b][row][k] dO[b][row][m], 64 x 64 outputs per block, 4 x 4 per thread,
// 16 rows at a time through LDS.
__global__ __launch_bounds__(256) void wgrad8_kernel(int rows, int K, int M, uint32_t blocks, const uint8_t* x8, const float* dO,
                                                     float* dW, int beta) {
  __shared__ float xs[16][64], ds[16][64];
  const uint8_t* bytes = x8 + (uint64_t)blocks * 32;
  const int b = blockIdx.z, k0 = blockIdx.y * 64, m0 = blockIdx.x * 64, t = threadIdx.x;
  const uint32_t xbase = (uint32_t)b * rows * K;
  const float* d = dO + (uint64_t)b * rows * M;
  float acc[4][4] = {};
  for (int r0 = 0; r0 < rows; r0 += 16) {
    for (int i = t; i < 16 * 64; i += 256) {
      const int r = r0 + (i >> 6), c = i & 63;
      float xv = 0.0f, dv = 0.0f;
      if (r < rows && k0 + c < K) {
        const uint32_t at = xbase + (uint32_t)r * K + k0 + c;
        xv = (float)(int8_t)x8[at] * step_of(bytes[at >> 5]);
      }
      if (r < rows && m0 + c < M) dv = d[(uint64_t)r * M + m0 + c];
      xs[i >> 6][c] = xv;
      ds[i >> 6][c] = dv;
    }
    __syncthreads();
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += xs[r][(t >> 4) * 4 + i] * ds[r][(t & 15) * 4 + j];
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = k0 + (t >> 4) * 4 + i, m = m0 + (t & 15) * 4 + j;
      if (k < K && m < M) {
        float* o = dW + ((uint64_t)b * K + k) * M + m;
        *o = beta ? *o + acc[i][j] : acc[i][j];
      }
    }
}

int launch_wgrad8(DeviceCtx* ctx, int batch, int rows, int K, int M, const void* x8, const float* dO, float* dW, int beta) {
  const uint64_t blocks = blocks8((uint64_t)batch * rows * K);
  hipLaunchKernelGGL(wgrad8_kernel, dim3((M + 63) / 64, (K + 63) / 64, batch), dim3(256), 0, ctx->stream, rows, K, M,
                     (uint32_t)blocks, static_cast<const uint8_t*>(x8), dO, dW, beta);
  LNN_HIP(hipGetLastError());
  return LNN_OK;
}

}  // namespace lnn
