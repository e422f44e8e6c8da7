// Activations kept in 8 bits: writing them, reading them back, and the weight gradient of a dense layer from its kept
// input.  The element format is in keep8.hpp.
#include <algorithm>

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

// ---- weight gradient from a kept input -------------------------------------------------------------------------------
//
//   dW[k][m] = sum over rows of X8[row][k] dO[row][m]
//
// A kept value is exactly a bf16 number, and dO is exactly the sum of three: h holds the top 8 of its 24 bits, l the
// last 8, m those between (each cut off, so that all three have dO's sign).  So dW = X8^T h + X8^T m + X8^T l on the bf16 matrix
// pipe, every product exact and every sum fp32: what an fp32 product of the same values would give, at three times the
// bf16 work, which is a fifth of the fp32 pipe's time.  The pipe takes bf16 inputs below 2^-126 for 0: of a dO below 2^-110
// the parts under 2^-126 are lost.
//
// Measured: 8192 rows, 4096 x 4096: 0.67-0.69 ms = 1.2 PFLOP/s of bf16 work, 400 TFLOP/s of the product (the fp32 pipe's product of
// decoded values: 2.0 ms) in passes behind each other: main kernel 0.60, 1.4 PFLOP/s, as a library's bf16 product of that size
// runs here.  In the first dozen passes after a pause it takes 0.62 to 0.85 ms, until the clock has settled.
// Bound: the matrix pipe; the first pass, 444 MB of traffic in 75 us, is the rest.  Thin operands are laid out too: 16384 rows,
// 4 x 4096: 198 us, four times what decoding and an fp32 product take.
//
// First pass: both operands are laid out as the matrix instruction reads them, 1 KB per fragment of 32 columns x 16 rows
// (lane l holds column l % 32, rows 8 (l / 32) .. + 7), rows and columns padded with zeros to whole tiles.  The main kernel
// then copies fragments to LDS and reads them back without any index arithmetic, bank conflict or bounds check.
using bf16x8 = __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16;
using f32x16w = __attribute__((__vector_size__(16 * sizeof(float)))) float;
typedef __attribute__((address_space(3))) void* lds_void;
typedef const __attribute__((address_space(1))) void* glb_void;

struct W8 {
  int rows, K, M, batch;   // rows, batch: of this launch's part
  int b0, r0, all;         // its first batch item and row; rows of the whole operand
  int k0, m0, ldk, ldm;    // its first columns of X and dO (K and M of them); columns of the whole operands
  int steps;               // of 32 rows
  int ipan, jpan;    // panels of 32 columns of X and dO, whole tiles
  uint32_t xblocks, xsize;   // blocks of the 8-bit copy; elements of X
};

__device__ __forceinline__ uint32_t hi16(uint32_t lo, uint32_t hi) { return (lo >> 16) | (hi & 0xffff0000u); }   // two bf16 of two fp32

// A workgroup lays out 16 rows x 512 columns of X (the first xwgs pieces of 16 rows) or dO at a time.
//
// X: a thread takes 8 rows x 4 columns, words of four codes.
template <int MX>
__device__ __forceinline__ void w8_pack_x(const W8& w, int b, int r16, int pan0, const uint8_t* x8, uint4* ap) {
  const int pan = pan0 + threadIdx.x / 16, half = (threadIdx.x >> 3) & 1, quad = threadIdx.x & 7;
  if (pan >= w.ipan) return;
  const int c = pan * 32 + quad * 4, cnt = min(max(w.K - c, 0), 4), r0 = r16 * 16 + half * 8;
  const Src8 x = {x8, x8 + (uint64_t)w.xblocks * 32};
  float v[8][4];
#pragma unroll
  for (int r = 0; r < 8; ++r)
    x.load<MX>(((uint32_t)(w.b0 + b) * w.all + w.r0 + r0 + r) * w.ldk + w.k0 + c, r0 + r < w.rows ? cnt : 0, w.xsize, v[r]);
  uint4* o = ap + (((uint64_t)b * 2 * w.steps + r16) * w.ipan + pan) * 64 + half * 32 + quad * 4;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t h[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) h[r] = __float_as_uint(v[r][k]);
    o[k] = make_uint4(hi16(h[0], h[1]), hi16(h[2], h[3]), hi16(h[4], h[5]), hi16(h[6], h[7]));
  }
}
// dO: a thread takes 8 rows of one column, so that a wavefront stores each part of a fragment as one kilobyte (with 4 columns to a
// thread, stores of 16 bytes every 64: 146 us for this pass
// at 8192 x 4096 x 4096, 77 so)
__device__ __forceinline__ void w8_pack_o(const W8& w, int b, int r16, int pan0, const float* dO, uint4* bp) {
  const int half = (threadIdx.x >> 5) & 1, r0 = r16 * 16 + half * 8;
  float v[4][8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = (pan0 + j * 4 + (int)(threadIdx.x >> 6)) * 32 + (threadIdx.x & 31);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const bool in = c < w.M && r0 + r < w.rows;
      const float d = dO[in ? ((uint32_t)(w.b0 + b) * w.all + w.r0 + r0 + r) * w.ldm + w.m0 + c : 0u];
      v[j][r] = in ? d : 0.0f;
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int pan = pan0 + j * 4 + (int)(threadIdx.x >> 6);
    uint32_t h[8], m[8], l[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      h[r] = __float_as_uint(v[j][r]);
      const bool odd = (h[r] & 0x7f800000u) == 0x7f800000u;   // infinity and NaN have no rest
      const float rest = odd ? 0.0f : v[j][r] - __uint_as_float(h[r] & 0xffff0000u);
      if (odd && (h[r] & 0x7fffffu)) h[r] = 0x7fc00000u;
      m[r] = __float_as_uint(rest);
      l[r] = __float_as_uint(rest - __uint_as_float(m[r] & 0xffff0000u));
    }
    if (pan < w.jpan) {
      uint4* o = bp + (((uint64_t)b * 2 * w.steps + r16) * w.jpan + pan) * 192 + (threadIdx.x & 63);
      o[0] = make_uint4(hi16(h[0], h[1]), hi16(h[2], h[3]), hi16(h[4], h[5]), hi16(h[6], h[7]));
      o[64] = make_uint4(hi16(m[0], m[1]), hi16(m[2], m[3]), hi16(m[4], m[5]), hi16(m[6], m[7]));
      o[128] = make_uint4(hi16(l[0], l[1]), hi16(l[2], l[3]), hi16(l[4], l[5]), hi16(l[6], l[7]));
    }
  }
}

template <int MX>
__global__ __launch_bounds__(256) void w8_pack_kernel(W8 w, int xwgs, int owgs, const uint8_t* x8, const float* dO, uint4* ap, uint4* bp) {
  const uint32_t wgs = xwgs + owgs, pieces = (uint32_t)w.batch * 2 * w.steps * wgs;
  for (uint32_t u = blockIdx.x; u < pieces; u += gridDim.x) {
    const uint32_t k = u / wgs, y = u - k * wgs;
    if (y < (uint32_t)xwgs)
      w8_pack_x<MX>(w, k / (2 * w.steps), k % (2 * w.steps), y * 16, x8, ap);
    else
      w8_pack_o(w, k / (2 * w.steps), k % (2 * w.steps), (y - xwgs) * 16, dO, bp);
  }
}

// PI x PJ fragments per wavefront, WI x WJ wavefronts: a tile of 32 PI WI (columns of X) x 32 PJ WJ (columns of dO).  A step
// is 32 rows = two fragments deep; its fragments come into one half of LDS while the other half is multiplied.
// Output t of the launch's tiles x splits: splits outermost, then groups of eight tile rows, column by column, and the
// workgroups of one XCD (every eighth) take a contiguous run of t, so that its L2 serves each fragment to several tiles.
template <int PI, int PJ, int WI, int WJ>
__global__ __launch_bounds__(64 * WI * WJ) void w8_kernel(W8 w, int ti, int tj, int splits, int per, const uint4* ap, const uint4* bp,
                                                          float* out, int ldo, uint64_t bstride, int beta) {
  constexpr int NI = PI * WI, NJ = PJ * WJ, NW = WI * WJ, FR = 2 * (NI + 3 * NJ), LPW = FR / NW;
  static_assert(FR % NW == 0, "whole fragments per wavefront");
  __shared__ uint4 lds[2][FR][64];
  const int total = ti * tj * splits * w.batch;
  const int t = (int)(blockIdx.x & 7) * ((total + 7) / 8) + (int)(blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= (total + 7) / 8 || t >= total) return;
  const int tiles = ti * tj, tile = t % tiles, z = t / tiles, split = z % splits, b = z / splits;
  const int grp = tile / (8 * tj), rem = tile - grp * 8 * tj, gi = min(8, ti - grp * 8);
  const int it = grp * 8 + rem % gi, jt = rem / gi;
  const int s0 = split * per, s1 = min(s0 + per, w.steps);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, wi = wave / WJ, wj = wave % WJ;

  // this wavefront's fragments of a step: [depth][NI], then [depth][NJ][part]
  const uint4* src[LPW];
  uint32_t adv[LPW];
#pragma unroll
  for (int e = 0; e < LPW; ++e) {
    const int f = wave * LPW + e;
    if (f < 2 * NI) {
      const int d = f / NI, p = f % NI;
      src[e] = ap + (((uint64_t)(b * w.steps + s0) * 2 + d) * w.ipan + it * NI + p) * 64 + lane;
      adv[e] = 2u * w.ipan * 64;
    } else {
      const int g = f - 2 * NI, d = g / (3 * NJ), p = g % (3 * NJ);
      src[e] = bp + ((((uint64_t)(b * w.steps + s0) * 2 + d) * w.jpan + jt * NJ) * 3 + p) * 64 + lane;
      adv[e] = 6u * w.jpan * 64;
    }
  }
  auto request = [&](int half) {
#pragma unroll
    for (int e = 0; e < LPW; ++e) {
      __builtin_amdgcn_global_load_lds((glb_void)src[e], (lds_void)&lds[half][wave * LPW + e][0], 16, 0, 0);
      src[e] += adv[e];
    }
  };
  f32x16w acc[PI][PJ];
#pragma unroll
  for (int i = 0; i < PI; ++i)
#pragma unroll
    for (int j = 0; j < PJ; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

  if (s0 < s1) request(0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  for (int s = s0; s < s1; ++s) {
    const int half = (s - s0) & 1;
    if (s + 1 < s1) request(half ^ 1);
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      bf16x8 a[PI], v[PJ][3];
#pragma unroll
      for (int i = 0; i < PI; ++i) a[i] = __builtin_bit_cast(bf16x8, lds[half][d * NI + wi * PI + i][lane]);
#pragma unroll
      for (int j = 0; j < PJ; ++j)
#pragma unroll
        for (int p = 0; p < 3; ++p) v[j][p] = __builtin_bit_cast(bf16x8, lds[half][2 * NI + (d * NJ + wj * PJ + j) * 3 + p][lane]);
#pragma unroll
      for (int p = 2; p >= 0; --p)
#pragma unroll
        for (int j = 0; j < PJ; ++j)
#pragma unroll
          for (int i = 0; i < PI; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], v[j][p], acc[i][j], 0, 0, 0);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }
  float* o = out + (uint64_t)z * bstride;   // splits are one behind the other: z is b where there is one
#pragma unroll
  for (int i = 0; i < PI; ++i)
#pragma unroll
    for (int j = 0; j < PJ; ++j) {
      const int m = ((jt * WJ + wj) * PJ + j) * 32 + (lane & 31), k0 = ((it * WI + wi) * PI + i) * 32 + 4 * (lane >> 5);
      if (m < w.M) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int k = k0 + 8 * (e >> 2) + (e & 3);
          if (k < w.K) {
            float* at = o + (uint64_t)k * ldo + m;
            *at = beta ? *at + acc[i][j][e] : acc[i][j][e];
          }
        }
      }
    }
}

// dW (+)= the splits' partial results, in order
__global__ __launch_bounds__(256) void w8_join_kernel(uint32_t n, int splits, int batch, const float* part, float* dW, int beta) {
  for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < (uint64_t)n * batch; i += gridDim.x * 256ull) {
    const uint32_t b = (uint32_t)(i / n), e = (uint32_t)(i - (uint64_t)b * n);
    const float* p = part + (uint64_t)b * splits * n + e;
    float s = 0.0f;
#pragma unroll 4
    for (int k = 0; k < splits; ++k) s += p[(uint64_t)k * n];
    dW[i] = beta ? dW[i] + s : s;
  }
}

// need: where to leave the scratch bytes of this part instead of launching it, or null
static int wgrad8_part(DeviceCtx* ctx, W8 w, const uint8_t* codes, const float* dO, float* dW, int beta, uint64_t* need) {
  const int K = w.K, M = w.M, batch = w.batch;
  // 256 x 256 tiles once they alone give most compute units one, else 128 x 128 ones
  auto tiles = [&](int side) { return (int64_t)((K + side - 1) / side) * ((M + side - 1) / side) * batch; };
  const int side = tiles(256) * 4 >= 3 * ctx->cus ? 256 : 128;
  const int ti = (K + side - 1) / side, tj = (M + side - 1) / side;
  w.ipan = ti * side / 32;
  w.jpan = tj * side / 32;
  // rows split until every compute unit has a tile (128: two), two steps at least to a split; not in a run of columns, whose rows
  // of dW lie apart, and which has a tile's worth of rows at most
  const bool whole = K == w.ldk && M == w.ldm;
  const int64_t want = whole ? (int64_t)ctx->cus * (side == 256 ? 1 : 2) / tiles(side) : 1;
  int splits = (int)std::max<int64_t>(1, std::min<int64_t>(want, w.steps / 2));
  const int per = (w.steps + splits - 1) / splits;
  splits = (w.steps + per - 1) / per;
  const uint64_t afrag = (uint64_t)batch * 2 * w.steps * w.ipan, bfrag = (uint64_t)batch * 2 * w.steps * w.jpan * 3;
  const uint64_t part = splits > 1 ? (uint64_t)batch * splits * K * M * 4 : 0;
  if (need) {
    *need = (afrag + bfrag) * 1024 + part;
    return LNN_OK;
  }
  uint4* ap = static_cast<uint4*>(ctx->ws);
  uint4* bp = ap + afrag * 64;
  float* pp = reinterpret_cast<float*>(bp + bfrag * 64);
  const int xwgs = (w.ipan + 15) / 16, owgs = (w.jpan + 15) / 16;
  const uint64_t pieces = (uint64_t)batch * 2 * w.steps * (xwgs + owgs);
  const dim3 pgrid((unsigned)std::min<uint64_t>(pieces, 1u << 20));
  if (w.ldk % 4 == 0)   // rows of X are whole groups of four: no shifts
    hipLaunchKernelGGL((w8_pack_kernel<G4>), pgrid, dim3(256), 0, ctx->stream, w, xwgs, owgs, codes, dO, ap, bp);
  else
    hipLaunchKernelGGL((w8_pack_kernel<GANY>), pgrid, dim3(256), 0, ctx->stream, w, xwgs, owgs, codes, dO, ap, bp);
  const int64_t total = (int64_t)ti * tj * splits * batch;
  const dim3 grid((unsigned)((total + 7) / 8 * 8));
  // partial results are dense; dW's rows are ldm apart
  float* out = splits > 1 ? pp : dW;
  const int ldo = splits > 1 ? M : w.ldm, b0 = splits > 1 ? 0 : beta;
  const uint64_t bstride = splits > 1 ? (uint64_t)K * M : (uint64_t)w.ldk * w.ldm;
  if (side == 256)
    hipLaunchKernelGGL((w8_kernel<4, 2, 2, 4>), grid, dim3(512), 0, ctx->stream, w, ti, tj, splits, per, ap, bp, out, ldo, bstride, b0);
  else
    hipLaunchKernelGGL((w8_kernel<2, 2, 2, 2>), grid, dim3(256), 0, ctx->stream, w, ti, tj, splits, per, ap, bp, out, ldo, bstride, b0);
  if (splits > 1)
    hipLaunchKernelGGL(w8_join_kernel, grid8(ctx, (uint64_t)K * M * batch), dim3(256), 0, ctx->stream, (uint32_t)K * M, splits, batch, pp, dW, beta);
  LNN_HIP(hipGetLastError());
  return LNN_OK;
}

int launch_wgrad8(DeviceCtx* ctx, int batch, int rows, int K, int M, const void* x8, const float* dO, float* dW, int beta) {
  W8 w = {};
  w.all = rows;
  w.ldk = K;
  w.ldm = M;
  w.xsize = (uint32_t)batch * rows * K;
  w.xblocks = (uint32_t)blocks8(w.xsize);
  // The laid-out operands of one launch stay within a gigabyte: many small products go in groups, one product of very many rows
  // in runs of rows, each added to the one before, and one of very many columns in runs of 2^22 of them (16384 tiles at least).
  constexpr int kColumns = 1 << 22;
  const int kc = std::min(K, kColumns), mc = std::min(M, kColumns);
  const uint64_t step = ((uint64_t)((kc + 255) / 256) + 3 * (uint64_t)((mc + 255) / 256)) * 16384;   // bytes of 32 rows, at most
  const int64_t most = std::max<int64_t>(1, (int64_t)((1u << 30) / step));                           // steps of one launch
  const int64_t steps = ((int64_t)rows + 31) / 32;
  const int group = (int)std::min<int64_t>(batch, std::max<int64_t>(1, most / steps));
  const int run = (int)std::min<int64_t>(rows, most * 32);
  // Scratch for the largest part comes first: a call that runs out of memory has not written or added anything yet.
  uint64_t most_bytes = 0;
  for (int launch = 0; launch < 2; ++launch) {
    for (w.b0 = 0; w.b0 < batch; w.b0 += group)
      for (w.k0 = 0; w.k0 < K; w.k0 += kc)
        for (w.m0 = 0; w.m0 < M; w.m0 += mc)
          for (w.r0 = 0;; w.r0 += run) {
            w.batch = std::min(group, batch - w.b0);
            w.K = std::min(kc, K - w.k0);
            w.M = std::min(mc, M - w.m0);
            w.rows = std::min(run, rows - w.r0);
            w.steps = (w.rows + 31) / 32;
            float* out = dW + ((uint64_t)w.b0 * K + w.k0) * M + w.m0;
            uint64_t need = 0;
            int st = wgrad8_part(ctx, w, static_cast<const uint8_t*>(x8), dO, out, w.r0 > 0 ? 1 : beta, launch ? nullptr : &need);
            if (st != LNN_OK) return st;
            most_bytes = std::max(most_bytes, need);
            if (run >= rows - w.r0) break;
          }
    if (!launch) {
      int st = ensure_workspace(ctx, most_bytes);
      if (st != LNN_OK) return st;
    }
  }
  return LNN_OK;
}

}  // namespace lnn
