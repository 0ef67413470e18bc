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

// a[w] of a kernel parameter, without a copy of the array in local memory.
template <typename T>
__device__ __forceinline__ T pick(const T (&a)[2], int w) {
  return w ? a[1] : a[0];
}

struct Kv8Cache {
  uint8_t* codes[2];  // keys, values
  float* scales[2];
  __half* tail[2];
  int batch, nkv, cap, hd;

  __device__ __forceinline__ int64_t head(int b, int h) const { return (int64_t)b * nkv + h; }
  __device__ __forceinline__ uint8_t* code_row(int w, int b, int h, int t) const {
    return pick(codes, w) + (head(b, h) * cap + t) * hd;
  }
  __device__ __forceinline__ float* scale(int w, int b, int h, int block) const {
    return pick(scales, w) + head(b, h) * (cap / kKvBlock) + block;
  }
  __device__ __forceinline__ __half* tail_row(int w, int b, int h, int slot) const {
    return pick(tail, w) + (head(b, h) * kKvBlock + slot) * hd;
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

__device__ __forceinline__ uint32_t kv8_word(uint4 x, int i) { return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w; }

// Sets values of a word (two of them) that are infinite or NaN to zero; tells
// which, by all bits of theirs.  The value products take masked positions by a
// weight of 0, which such values would turn into NaN: the open block's go in
// without them, and the rows that attend them have them added afterwards (a
// softmax weight is positive, so it does not change them).
__device__ __forceinline__ uint32_t kv8_drop_odd(uint32_t& x) {
  const uint32_t odd = __vcmpeq2(x & 0x7c007c00u, 0x7c007c00u);
  x &= ~odd;
  return odd;
}
__device__ __forceinline__ uint32_t kv8_drop_odd(uint4& x) {
  return kv8_drop_odd(x.x) | kv8_drop_odd(x.y) | kv8_drop_odd(x.z) | kv8_drop_odd(x.w);
}

// Largest magnitude of eight values; not finite if one is not.
__device__ __forceinline__ float kv8_amax8(uint4 x) {
  __half2 m = __hmax2_nan(__hmax2_nan(__habs2(u2h(x.x)), __habs2(u2h(x.y))),
                          __hmax2_nan(__habs2(u2h(x.z)), __habs2(u2h(x.w))));
  const float2 f = __half22float2(m);
  return f.x <= 65504.f && f.y <= 65504.f ? fmaxf(f.x, f.y) : INFINITY;
}

// The same of the values that quantisation sees.
__device__ __forceinline__ float kv8_amax8_finite(uint4 x) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(u2h(kv8_word(x, i)));
    m = fmaxf(m, fmaxf(fabsf(kv8_finite(f.x)), fabsf(kv8_finite(f.y))));
  }
  return m;
}

// Correctly rounded divisions, so that the codes follow from the definition.
__device__ __forceinline__ float kv8_scale(float amax) { return __fdiv_rn(amax, 127.f); }

// Codes of eight values; finite: all of the block's values are.  The code is
// the low byte of x / scale + 1.5 * 2^23 + 128: the addition rounds to a whole
// number, ties to even.  x * (1 / scale) is within 2^-15 of the quotient (both
// below 128), so only within 4e-5 of a tie can it round otherwise: eight
// values with one there are divided.  Two values an instruction, one branch
// for eight.
__device__ __forceinline__ uint2 kv8_codes8(uint4 x, float scale, float per_scale, bool finite) {
  constexpr float kWhole = 12583040.f;
  const uint64_t whole = f32_pair(kWhole, kWhole), minus = f32_pair(-kWhole, -kWhole), per = f32_pair(per_scale, per_scale);
  float2 f[4];
  float y[8], off = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = __half22float2(u2h(kv8_word(x, i)));
    if (!finite) f[i] = make_float2(kv8_finite(f[i].x), kv8_finite(f[i].y));
    const uint64_t q = f32_mul2(f32_pair(f[i].x, f[i].y), per), r = f32_add2(q, whole), n = f32_fma2(f32_add2(r, minus), f32_pair(-1.f, -1.f), q);
    float n0, n1;
    f32_split(n, n0, n1);
    f32_split(r, y[2 * i], y[2 * i + 1]);
    off = fmaxf(off, fmaxf(fabsf(n0), fabsf(n1)));
  }
  if (off > 0.49996f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[2 * i] = __fdiv_rn(f[i].x, scale) + kWhole;
      y[2 * i + 1] = __fdiv_rn(f[i].y, scale) + kWhole;
    }
  }
  uint32_t o[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const auto c = [&](int i) { return __float_as_uint(y[4 * h + i]); };
    o[h] = __byte_perm(__byte_perm(c(0), c(1), 0x0040), __byte_perm(c(2), c(3), 0x0040), 0x5410);
  }
  return make_uint2(o[0], o[1]);
}

// fp16((code - 128) * scale) of eight codes: a byte in the low end of 2^23 is
// 2^23 + code, exactly.
__device__ __forceinline__ uint4 kv8_values8(uint2 c, float scale) {
  const uint64_t zero = f32_pair(-8388736.f, -8388736.f), by = f32_pair(scale, scale);
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = i < 2 ? c.x : c.y;
    const float a = __uint_as_float(__byte_perm(w, 0x4b000000u, i & 1 ? 0x7442 : 0x7440));
    const float b = __uint_as_float(__byte_perm(w, 0x4b000000u, i & 1 ? 0x7443 : 0x7441));
    float x, y;
    f32_split(f32_mul2(f32_add2(f32_pair(a, b), zero), by), x, y);
    r[i] = h2u(__floats2half2_rn(x, y));
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// A block's scale (0 where all values are: their quotient is then 0 too).  The
// smallest FP16 number / 127 still has a finite reciprocal.
struct Kv8Scale {
  float scale, per_scale;
  bool finite;  // all of the block's values are
};

__device__ __forceinline__ Kv8Scale kv8_make_scale(float amax, bool finite) {
  const float s = kv8_scale(amax);
  return Kv8Scale{s, s > 0.f ? __fdiv_rn(1.f, s) : 0.f, finite};
}

__device__ __forceinline__ uint2 kv8_codes8(uint4 x, const Kv8Scale& q) {
  return kv8_codes8(x, q.scale, q.per_scale, q.finite);
}

// Largest magnitudes over the CTA's threads and values v; where one is not
// finite they are counted again as quantisation sees them.  Every thread gets
// the result; red has a place for each warp.
template <int N, int THREADS>
__device__ __forceinline__ Kv8Scale kv8_block_scale(const uint4 (&v)[N], float* red) {
  auto all = [&](float m) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    m = red[0];
#pragma unroll
    for (int i = 1; i < THREADS / 32; ++i) m = fmaxf(m, red[i]);
    return m;
  };
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, kv8_amax8(v[i]));
  m = all(m);
  if (m <= 65504.f) return kv8_make_scale(m, true);
  m = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, kv8_amax8_finite(v[i]));
  return kv8_make_scale(all(m), false);
}

// One head's keys or values.
template <int HD>
struct Kv8Head {
  uint8_t* codes;  // [capacity][HD]
  float* scales;   // [capacity / 64]
  __half* tail;    // [64][HD]

  __device__ __forceinline__ Kv8Head(const Kv8Cache& c, int w, int b, int h)
      : codes(pick(c.codes, w) + c.head(b, h) * c.cap * HD),
        scales(pick(c.scales, w) + c.head(b, h) * (c.cap / kKvBlock)),
        tail(pick(c.tail, w) + c.head(b, h) * (kKvBlock * HD)) {}
  // Eight stored values of position t, FP16; last: the block in the tail.
  __device__ __forceinline__ uint4 read8(int t, int last, int d0) const {
    const int block = (unsigned)t / kKvBlock;
    if (block == last) return *reinterpret_cast<const uint4*>(tail + t % kKvBlock * HD + d0);
    return kv8_values8(*reinterpret_cast<const uint2*>(codes + ((int64_t)t * HD + d0)), scales[block]);
  }
};

// Checks a descriptor and fills the kernels' view of it.
int kv8_cache(const char* who, const pp_kv8_cache* c, Kv8Cache* out);
int kv8_rope(const char* who, const void* cos_t, const void* sin_t, const int* pos, int64_t len, Kv8Rope* out);

}  // namespace pp
