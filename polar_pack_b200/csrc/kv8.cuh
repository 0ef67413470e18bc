// The 8-bit KV cache of one layer (pp_kv8_cache), shared by its kernels.
//
// Positions of a sequence come in blocks of 64.  A stored key or value is
// (code - 128) * scale: uint8 codes [batch][kv head][capacity][head_dim], one
// FP32 scale per block and head.  The block that holds a sequence's last
// token is read from its FP16 rows (the tail, [batch][kv head][64][head_dim]);
// its codes are written by the call that completes it.
//   scale = max|x| / 127,  code = 128 + round(x / scale)   (ties to even)
// Every element's error is then at most scale / 2, and since a block is
// quantised once, from its FP16 rows, the cache does not depend on how its
// tokens were split into calls.
#pragma once

#include <cuda_fp16.h>
#include <math.h>

#include "pp_common.cuh"
#include "pp_host.h"

namespace pp {

constexpr int kKvBlock = 64;

struct Kv8Cache {
  uint8_t* codes[2];  // keys, values
  float* scales[2];
  __half* tail[2];
  int batch, nkv, cap, hd;

  __device__ __forceinline__ int64_t head(int b, int h) const { return (int64_t)b * nkv + h; }
  __device__ __forceinline__ uint8_t* code_row(int w, int b, int h, int t) const {
    return codes[w] + (head(b, h) * cap + t) * hd;
  }
  __device__ __forceinline__ float* scale(int w, int b, int h, int block) const {
    return scales[w] + head(b, h) * (cap / kKvBlock) + block;
  }
  __device__ __forceinline__ __half* tail_row(int w, int b, int h, int slot) const {
    return tail[w] + (head(b, h) * kKvBlock + slot) * hd;
  }
};

// The block read from FP16 rows: the one of the last of `len` tokens.
__host__ __device__ __forceinline__ int kv8_last_block(int len) { return len > 0 ? (len - 1) / kKvBlock : 0; }

// Rotary embedding of rows as they are read (cos == NULL: none).
struct Kv8Rope {
  const __half* cos;  // [len][hd], both halves
  const __half* sin;
  const int* pos;     // [batch] rotation position of the call's first row
  int len;
};

// Eight FP16 values of a row at dimension d0 (a multiple of 8), rotated at
// position t as the decoder step does it:
// x' = fp16(fp16(x cos) + fp16(rotate_half(x) sin)).
__device__ __forceinline__ uint4 kv8_load8(const __half* row, int d0, int hd, const Kv8Rope& rope, int t) {
  uint4 x = *reinterpret_cast<const uint4*>(row + d0);
  if (rope.cos == nullptr) return x;
  const int half = hd / 2;
  const uint4 y = *reinterpret_cast<const uint4*>(row + (d0 < half ? d0 + half : d0 - half));
  const uint4 c = *reinterpret_cast<const uint4*>(rope.cos + (int64_t)t * hd + d0);
  const uint4 s = *reinterpret_cast<const uint4*>(rope.sin + (int64_t)t * hd + d0);
  const uint32_t sign = d0 < half ? 0x80008000u : 0u;  // rotate_half: (-x2, x1)
  auto rot = [&](uint32_t a, uint32_t b, uint32_t cc, uint32_t ss) {
    return h2u(__hadd2_rn(__hmul2_rn(u2h(a), u2h(cc)), __hmul2_rn(u2h(b ^ sign), u2h(ss))));
  };
  return make_uint4(rot(x.x, y.x, c.x, s.x), rot(x.y, y.y, c.y, s.y), rot(x.z, y.z, c.z, s.z),
                    rot(x.w, y.w, c.w, s.w));
}

// The value that quantisation sees: NaN counts as 0, infinities as the
// largest finite FP16 number.
__device__ __forceinline__ float kv8_finite(float x) { return x != x ? 0.f : fminf(fmaxf(x, -65504.f), 65504.f); }

__device__ __forceinline__ float kv8_amax8(uint4 x) {
  float m = 0.f;
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(u2h(w[i]));
    m = fmaxf(m, fmaxf(fabsf(kv8_finite(f.x)), fabsf(kv8_finite(f.y))));
  }
  return m;
}

// Correctly rounded divisions, so that the codes follow from the definition.
__device__ __forceinline__ float kv8_scale(float amax) { return __fdiv_rn(amax, 127.f); }

__device__ __forceinline__ uint32_t kv8_code(float x, float scale) {
  return scale > 0.f ? (uint32_t)(128 + (int)rintf(__fdiv_rn(kv8_finite(x), scale))) : 128u;
}

__device__ __forceinline__ uint2 kv8_codes8(uint4 x, float scale) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t o[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(u2h(w[i]));
    o[i >> 1] |= (kv8_code(f.x, scale) | kv8_code(f.y, scale) << 8) << (16 * (i & 1));
  }
  return make_uint2(o[0], o[1]);
}

// fp16((code - 128) * scale) of eight codes.
__device__ __forceinline__ uint4 kv8_values8(uint2 c, float scale) {
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = (i < 2 ? c.x : c.y) >> (16 * (i & 1));
    r[i] = h2u(__floats2half2_rn(((int)(w & 255u) - 128) * scale, ((int)((w >> 8) & 255u) - 128) * scale));
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// Eight stored values of position t of a sequence of `len` tokens, FP16.
__device__ __forceinline__ uint4 kv8_read8(const Kv8Cache& c, int w, int b, int h, int t, int len, int d0) {
  if (t / kKvBlock == kv8_last_block(len))
    return *reinterpret_cast<const uint4*>(c.tail_row(w, b, h, t % kKvBlock) + d0);
  return kv8_values8(*reinterpret_cast<const uint2*>(c.code_row(w, b, h, t) + d0), *c.scale(w, b, h, t / kKvBlock));
}

// Checks a descriptor and fills the kernels' view of it.
int kv8_cache(const char* who, const pp_kv8_cache* c, Kv8Cache* out);
int kv8_rope(const char* who, const void* cos_t, const void* sin_t, const int* pos, int64_t len, Kv8Rope* out);

}  // namespace pp
