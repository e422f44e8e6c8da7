// Activations kept in 8 bits: the element format, shared by every kernel that writes or reads such a copy.
//
// Blocks of 32 elements, consecutive in memory, share a power of two.  With a = max |x| of a block:
//   k = floor(log2 a), e = k - 6 (k - 5 where a 2^-e >= 127.5 would round to 128), kept within [-126, 121];
//   q = x 2^-e rounded half to even, within +-127;  the value read back is q 2^e.
// 2^-e is a normal fp32 number and the product with it is exact (or far below half a step), so a code has exactly one
// right value, whichever kernel forms it, and every value read back is exactly a bf16 number (7 bits of magnitude).
// The error is at most half a step, 2^(e-1) <= a / 127.5 (2^-127 where e is held at -126; a whole step at the very top of the fp32
// range, where it is held at 121).
// Exponent byte: e + 127; 0 for a block of zeros; 255 for a block that holds an infinity or NaN.  Such a block's codes
// are 0 and read back as NaN (0 * inf): a diverged activation stays visible.
//
// Memory: the codes of ceil(n / 32) blocks (the last one padded with zeros), then the exponent bytes.
#pragma once
#include "common.hpp"

namespace lnn {

constexpr uint32_t kBlock8 = 32;
static inline uint64_t blocks8(uint64_t n) { return (n + kBlock8 - 1) / kBlock8; }
static inline uint64_t bytes8(uint64_t n) { return blocks8(n) * (kBlock8 + 1); }

// four bytes / floats at any 4-byte (floats) or 1-byte (codes) aligned address: global memory takes unaligned vectors
struct __attribute__((packed, aligned(4))) F4 { float v[4]; };
struct __attribute__((packed, aligned(1))) B4 { uint32_t v; };

// the bits of |x|: ordered like the magnitudes, infinity and NaN above every finite value
__device__ __forceinline__ uint32_t mag_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// exponent byte of a block from the bits of its largest magnitude
__device__ __forceinline__ uint32_t exp_byte(uint32_t amax) {
  if (amax >= 0x7f800000u) return 255u;
  if (amax == 0u) return 0u;
  // 127.5 = 64 * 1.9921875: fraction bits 0x7f0000
  const int b = (int)(amax >> 23) - 6 + ((amax & 0x7fffffu) >= 0x7f0000u ? 1 : 0);
  return (uint32_t)min(max(b, 1), 248);
}
// 2^-e of an exponent byte; 0 for blocks whose codes are all 0
__device__ __forceinline__ float inv_step(uint32_t byte) {
  return (byte == 0u || byte == 255u) ? 0.0f : __uint_as_float((254u - byte) << 23);
}
// 2^e: 0 for byte 0 and infinity for byte 255, whose codes are 0
__device__ __forceinline__ float step_of(uint32_t byte) { return __uint_as_float(byte << 23); }
__device__ __forceinline__ int code_of(float x, float inv) {
  return inv == 0.0f ? 0 : min(max((int)rintf(x * inv), -127), 127);   // |x 2^-e| < 128: the block is finite here
}
__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
  return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 | (uint32_t)d << 24;
}
__device__ __forceinline__ float code_at(uint32_t four, int i) { return (float)(int)(int8_t)(four >> (8 * i)); }

// four codes of a float4 whose block is spread over 8 neighbouring lanes (lane & 7 = position); byte = the block's
// exponent, the same in the eight lanes
__device__ __forceinline__ uint32_t encode_lane4(const float* v, uint32_t* byte) {
  uint32_t a = max(max(mag_bits(v[0]), mag_bits(v[1])), max(mag_bits(v[2]), mag_bits(v[3])));
  a = max(a, (uint32_t)__shfl_xor((int)a, 1, 64));
  a = max(a, (uint32_t)__shfl_xor((int)a, 2, 64));
  a = max(a, (uint32_t)__shfl_xor((int)a, 4, 64));
  *byte = exp_byte(a);
  const float inv = inv_step(*byte);
  return pack4(code_of(v[0], inv), code_of(v[1], inv), code_of(v[2], inv), code_of(v[3], inv));
}

// Four elements of a tensor at any place, of which the first cnt count; the others are set to 0.  No branch: behind one,
// the compiler waits for each load before it sends the next, and a kernel that holds a row in registers has nothing else
// to cover that latency (backward pass of 32 x 128 x 56 x 56: 39 us with branches).  Lanes without elements read the
// tensor's start; groups that hang over its end read its last four elements and shift.
//   G4      every group is whole (cnt 0 or 4)
//   GANY    any cnt, tensor of four elements or more
//   GTINY   any cnt, any tensor: element by element
// size: elements of the tensor.
enum { G4, GANY, GTINY };
template <int MODE>
__device__ __forceinline__ void load4(const float* p, uint32_t at, int cnt, uint32_t size, float* v) {
  if (MODE == GTINY) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = p[min(at + k, size - 1)];
  } else {
    const uint32_t from = cnt > 0 ? (MODE == GANY ? min(at, size - 4) : at) : 0u;
    const F4 f = *reinterpret_cast<const F4*>(p + from);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = f.v[k];
    if (MODE == GANY) {
      const uint32_t d = at - from;
      if (d & 1) { v[0] = v[1]; v[1] = v[2]; v[2] = v[3]; }
      if (d & 2) { v[0] = v[2]; v[1] = v[3]; }
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = k < cnt ? v[k] : 0.0f;
}
// The codes of four elements as one word (0 where there is none): the codes of a copy are padded to whole blocks.
template <int MODE>
__device__ __forceinline__ uint32_t load_codes(const uint8_t* p, uint32_t at, int cnt, uint32_t size) {
  if (MODE == G4) {
    const uint32_t q = reinterpret_cast<const B4*>(p + (cnt > 0 ? at : 0u))->v;
    return cnt > 0 ? q : 0u;
  }
  const uint32_t from = cnt > 0 ? min(at, ((size + 31) & ~31u) - 4) : 0u;
  const uint32_t q = reinterpret_cast<const B4*>(p + from)->v >> (cnt > 0 ? 8 * (at - from) : 0u);
  return cnt >= 4 ? q : q & ((1u << (8 * max(cnt, 0))) - 1);
}
// Sources of x: fp32 memory, or the 8-bit copy
struct SrcF {
  const float* x;
  __device__ __forceinline__ float at(uint32_t i) const { return x[i]; }
  template <int MODE>
  __device__ __forceinline__ void load(uint32_t at, int cnt, uint32_t size, float* v) const { load4<MODE>(x, at, cnt, size, v); }
};
struct Src8 {
  const uint8_t* codes;
  const uint8_t* bytes;
  __device__ __forceinline__ float at(uint32_t i) const { return (float)(int8_t)codes[i] * step_of(bytes[i >> 5]); }
  template <int MODE>
  __device__ __forceinline__ void load(uint32_t at, int cnt, uint32_t size, float* v) const {
    const uint32_t q = load_codes<MODE>(codes, at, cnt, size);
    const uint32_t b0 = cnt > 0 ? at >> 5 : 0u;
    // a lane without elements reads block 0, whose step may be infinite: 0 * inf is no 0
    const float first = step_of(bytes[b0]), s0 = cnt > 0 ? first : 0.0f;
    if (MODE == G4) {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = code_at(q, k) * s0;
    } else {   // four elements lie in one block, or in two
      const float s1 = step_of(bytes[cnt > 0 ? min(at + 3, size - 1) >> 5 : 0u]);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = k < cnt ? code_at(q, k) * (((at + k) >> 5) == b0 ? s0 : s1) : 0.0f;
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

}  // namespace lnn
