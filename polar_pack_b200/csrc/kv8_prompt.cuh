// Prompt attention over the 8-bit KV cache on the tcgen05 tensor cores: many
// query rows per kv head (kv8_attention.cu launches it).
//
// Mathematics as in kv8_decode.cuh, with the running maximum moved only when a
// row outgrows it by 2^4 and the block scale of the values folded into the
// weights: with f = s_v / v_ref, v_ref the power of two above the largest s_v of
// the range, the tensor core accumulates P' (c_v - 128) for
// P' = fp16(2^11 f exp(S - m)), and
// out = v_ref sum P' (c_v - 128) / (2^11 sum exp(S - m)).  The open block's rows
// are divided by v_ref instead (which is at least 2^-15 of their largest, so
// that they stay FP16 numbers).  2^11 leaves 2^4 for the lagging maximum below
// FP16's largest number, and keeps weights down to 2^-25 / f of the maximum at
// full precision.
//
// Bound: the matrix products; next to them the 16 exponentials a clock of an
// SM, which take about as long.  A CTA has 256 rows (query x head of the kv
// head's group) as two tiles of 128, so that one tile's softmax runs while the
// other's products do, and each block is unpacked once for both.  Roles:
//   warps 0-3, 4-7   softmax of tile 0, 1: a thread has one row; S from tensor
//                    memory, P over it, O rescaled in tensor memory when its
//                    row's maximum moved, the result at the end
//   warps 8-11       unpack a block's value codes (arrived by TMA) to FP16 tiles,
//   warps 12-15      its key codes
//   warp 16          issues S = Q K^T (M 128, N 64), two blocks ahead of
//   warp 18          which issues O += P V (M 128, N head_dim, P from tensor memory)
//   warp 17          the code boxes' TMA
// K and V tiles have the same layout, positions x dimensions in 128-byte
// swizzled rows: K-major for the first product, MN-major for the second.
// Every wait is bounded; tensor memory is released on every path.
//
// Measured: 4 prompts of 2048, 28 query heads on 4 kv heads of 128, causal: 185
// us, 649 TFLOP/s of the pairs that count; ragged chunks of 509 of 0, 2040, 2332
// and 4001, 16 heads on 2: 70 us (86 with the longest in one part).  A block
// takes 1.1 us of both tiles, where its products need 0.68.  Copies that left
// work out: without the unpacking, the exponentials or all but one step of
// either product hardly faster, without products and softmax together 0.65 us;
// so a block is bound by the softmax warps' own chain, one row to a thread, two
// such warps to a scheduler.  A single pass over the scores with the maximum so far,
// repeated where it grows, took 188 us where this took 182.  The unpacking roles
// keep some values in local memory (52 bytes at head_dim 128).
#pragma once

#include "kv8.cuh"
#include "kv8_decode.cuh"
#include "pp_tcgen05.cuh"

namespace pp {

constexpr int kPrRows = 256;                  // query rows of a CTA
constexpr int kPrTile = 128;                  // rows of one MMA
constexpr int kPrThreads = 20 * 32;           // the last warp has no role
constexpr int kPrCodeStages = 4;
constexpr float kPrLag = 4.f;                 // log2 growth of a maximum that rescales
constexpr float kPrLift = 11.f;               // log2 factor of the FP16 weights

struct Kv8PromptParams {
  Kv8Cache c;
  const __half* q;
  int64_t ldqb, ldqt, ldqh;
  __half* out;
  int64_t ldob, ldot, ldoh;
  const int* lens;
  const int* counts;
  int n, nq;
  float scale2;       // |scale| * log2(e)
  uint32_t q_sign;    // 0x80008000 for a negative scale
  Kv8Rope rope;
  int tiles, splits;  // row tiles per (sequence, kv head); parts of a tile's positions, at most
  int ctas;           // that run at a time
  float* part;        // splits > 1: [splits][batch][kv head][rows][hd] sums, then the same rows' (maximum, sum)
  int* part_blocks;   // splits > 1: blocks of a part, for the join
  int* status;
};

template <int HD>
struct Kv8PromptSmem {
  static constexpr int kHalves = HD / 64;                        // 64-dimension halves of a tile
  static constexpr int kQTile = kHalves * kPrTile * 128;
  static constexpr int kKv = kHalves * kKvBlock * 128;           // an FP16 tile of keys or values
  static constexpr int kCode = kKvBlock * HD;
  static constexpr int kQ = 0;
  static constexpr int kK = 2 * kQTile;                          // two buffers each
  static constexpr int kV = kK + 2 * kKv;
  static constexpr int kCodes = kV + 2 * kKv;
  static constexpr int kTail = kCodes + kPrCodeStages * 2 * kCode;  // the open block's values, plain rows
  static constexpr int kBar = kTail + kKvBlock * HD * 2;
  static constexpr int kBytes = kBar + 256;
};

// Blocks of a sequence of the call, and into how many parts they are split (a
// sequence without queries may be longer than all that count: at most `most`).
__device__ __forceinline__ int kv8_seq_blocks(int len, int cap) {
  return len > 0 && len <= cap ? (len + kKvBlock - 1) / kKvBlock : 0;
}
__device__ __forceinline__ int kv8_seq_parts(int blocks, int part_blocks, int most) {
  return min(most, max(1, (blocks + part_blocks - 1) / part_blocks));
}

// Blocks of a part (splits > 1), from the lengths: of 512 sizes up to the
// longest sequence's the one with which all tiles' parts, run `ctas` at a time,
// take the least time.  A CTA's start and end cost as much as 14 blocks (15 us),
// the join's start 4 and each of its parts 1/20 (its sums in FP32, written and
// read).
constexpr int kPrSplitBatch = 256;  // sequences of a call that may be split
constexpr int kPrMaxSplits = 256;

__device__ __forceinline__ int kv8_part_blocks(const Kv8PromptParams& p) {
  __shared__ int s_blocks[kPrSplitBatch], s_tiles[kPrSplitBatch], s_max;
  __shared__ unsigned s_best;
  const int tid = threadIdx.x, group = p.nq / p.c.nkv;
  if (tid == 0) {
    s_max = 1;
    s_best = ~0u;
  }
  __syncthreads();
  if (tid < p.c.batch) {
    const int cnt = p.counts ? min(max(p.counts[tid], 0), p.n) : p.n;
    const int blocks = kv8_seq_blocks(p.lens[tid], p.c.cap);
    s_blocks[tid] = blocks;
    s_tiles[tid] = (cnt * group + kPrRows - 1) / kPrRows;
    if (cnt > 0) atomicMax(&s_max, blocks);
  }
  __syncthreads();
  constexpr int kSizes = 512;
  auto size = [&](int i) { return (int)(((int64_t)s_max * (kSizes - i) + kSizes - 1) / kSizes); };
  if (tid < kSizes) {
    int n = 0, joined = 0;
    for (int b = 0; b < p.c.batch; ++b) {
      const int parts = kv8_seq_parts(s_blocks[b], size(tid), 0x7fffffff);
      n += s_tiles[b] * parts;
      if (parts > 1) joined += s_tiles[b] * parts;
    }
    const int64_t rounds = (n * p.c.nkv + p.ctas - 1) / p.ctas;
    const int64_t time = rounds * (14 + size(tid)) * 20 + (joined ? 80 + joined * p.c.nkv : 0);
    const bool fits = size(tid) * (int64_t)p.splits >= s_max;
    const unsigned best = __reduce_min_sync(0xffffffffu, fits ? (unsigned)min(time, (int64_t)0x3fffff) << 9 | tid : ~0u);
    if ((tid & 31) == 0) atomicMin(&s_best, best);
  }
  __syncthreads();
  return size((int)(s_best & 511));
}

// Row r of a call's n * group rows: query r / group, head r % group.
__device__ __forceinline__ int kv8_row_stop(int i, int len, int cnt) { return i < cnt ? len - cnt + i + 1 : 0; }

// Adds the values of the open block that are infinite or NaN to the results of
// this CTA's rows that attend them: to the output, or to the part's sums in
// FP32.  The softmax warps' threads come here, a row each; everything is worked
// out again, as the kernel has no registers to keep it in.
template <int HD>
__device__ __noinline__ void kv8_prompt_add_odd(const Kv8PromptParams& p, bool parts) {
  const int tile = p.tiles - 1 - blockIdx.y % p.tiles, split = blockIdx.y / p.tiles;
  const int kvh = blockIdx.x % p.c.nkv, b = blockIdx.x / p.c.nkv, group = p.nq / p.c.nkv, rows = p.n * group;
  const int r = tile * kPrRows + threadIdx.x, i = r / group, h = r - i * group;
  if (r >= rows) return;
  const int len = p.lens[b], cnt = p.counts ? min(max(p.counts[b], 0), p.n) : p.n;
  const int open = kv8_last_block(len) * kKvBlock, stop = kv8_row_stop(i, len, cnt);
  __half* out = p.out + b * p.ldob + i * p.ldot + (int64_t)(kvh * group + h) * p.ldoh;
  float* sums = p.part + ((((int64_t)split * p.c.batch + b) * p.c.nkv + kvh) * rows + r) * HD;
  for (int t = open; t < stop; ++t)
    for (int d = 0; d < HD; d += 2) {
      uint32_t v = *reinterpret_cast<const uint32_t*>(p.c.tail_row(1, b, kvh, t - open) + d), rest = v;
      v &= kv8_drop_odd(rest);
      if (v == 0) continue;
      const float2 f = __half22float2(u2h(v));
      if (parts) {
        sums[d] += f.x;
        sums[d + 1] += f.y;
      } else {
        __half2* o = reinterpret_cast<__half2*>(out + d);
        *o = __floats2half2_rn(__low2float(*o) + f.x, __high2float(*o) + f.y);
      }
    }
}

template <int HD>
__global__ void __launch_bounds__(kPrThreads, 1)
    kv8_prompt_kernel(const __grid_constant__ Kv8PromptParams p, const __grid_constant__ CUtensorMap tk,
                      const __grid_constant__ CUtensorMap tv) {
  using S = Kv8PromptSmem<HD>;
  __shared__ float s_red[8];
  __shared__ uint32_t s_tmem;
  __shared__ int s_odd;  // values of the open block are infinite or NaN
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = (uint32_t)__cvta_generic_to_shared(pp_smem);
  // long tiles first, of all heads: the last rows attend the most positions
  const int tile = p.tiles - 1 - blockIdx.y % p.tiles, split = blockIdx.y / p.tiles;
  const int kvh = blockIdx.x % p.c.nkv, b = blockIdx.x / p.c.nkv;
  int splits = 1;  // parts of this sequence's tiles; the CTAs past them have no work
  if (p.splits > 1) {
    pdl_launch_dependents();
    pdl_wait();
    const int size = kv8_part_blocks(p);
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) *p.part_blocks = size;
    splits = kv8_seq_parts(kv8_seq_blocks(p.lens[b], p.c.cap), size, p.splits);
    if (split >= splits) return;
  }
  const int group = p.nq / p.c.nkv, rows = p.n * group, row0 = tile * kPrRows;
  // barriers
  const uint32_t bar = base + S::kBar;
  const uint32_t code_full = bar, code_empty = bar + 32;           // [4]
  const uint32_t k_full = bar + 64, k_empty = bar + 80;            // [2]
  const uint32_t v_full = bar + 96, v_empty = bar + 112;           // [2]
  const uint32_t s_full = bar + 128;                               // [tile][2]
  const uint32_t p_full = bar + 160;                               // [tile][2]
  const uint32_t o_full = bar + 192;                               // [tile][2]
  const uint32_t done = bar + 224, q_full = bar + 232, tail_full = bar + 240;
  if (tid == 0) {
    for (int i = 0; i < kPrCodeStages; ++i) {
      mbar_init(code_full + 8 * i, 1);
      mbar_init(code_empty + 8 * i, 8);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(k_full + 8 * i, 4);
      mbar_init(k_empty + 8 * i, 1);
      mbar_init(v_full + 8 * i, 4);
      mbar_init(v_empty + 8 * i, 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(o_full + 8 * i, 1);
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_full + 8 * i, 4);
    }
    mbar_init(done, 1);
    mbar_init(q_full, 8);
    mbar_init(tail_full, 8);
    s_odd = 0;
    fence_mbar_init();
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
  }
  if (warp == 16) {
    tmem_alloc((uint32_t)__cvta_generic_to_shared(&s_tmem), 512);
    tmem_relinquish();
  }
  pdl_launch_dependents();
  pdl_wait();

  int len = p.lens[b];
  const int cnt = p.counts ? min(max(p.counts[b], 0), p.n) : p.n;
  bool ok = len <= p.c.cap;
  const int rot0 = p.rope.cos ? p.rope.pos[b] : 0;
  if (p.rope.cos && len > 0 && cnt > 0) ok = ok && rot0 >= 0 && rot0 <= p.rope.len - cnt;
  if (!ok && tid == 0) atomicExch(p.status, 5);
  len = ok ? max(len, 0) : 0;
  // blocks that this CTA's rows attend, and its part of them
  const int i_first = row0 / group, i_last = min((min(row0 + kPrRows, rows) - 1) / group, cnt - 1);
  const int max_stop = i_last >= i_first ? max(0, kv8_row_stop(i_last, len, cnt)) : 0;
  const int blocks = len > 0 ? (max_stop + kKvBlock - 1) / kKvBlock : 0;
  const int j0 = (int)((int64_t)blocks * split / splits), j1 = (int)((int64_t)blocks * (split + 1) / splits);
  const int J = j1 - j0;
  const int coded = kv8_last_block(len);  // the block after them is the tail
  const float *k_scale = p.c.scale(0, b, kvh, 0), *v_scale = p.c.scale(1, b, kvh, 0);

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  auto wait = [&](uint32_t b_, int parity) { return mbar_wait_warp(b_, parity, p.status); };

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");  // 256 x 144 + 384 x 64 = 640 x 96 registers
    // -------------------------------------------------------------- softmax
    // the query rows to their tiles, K-major, while the first blocks are on their
    // way: sixteen loads at a time; and the reference of the value scales
    float vref = 0.f;
    constexpr int kTailItems = kKvBlock * (HD / 8) / 256;
    uint4 open[kTailItems];
    if (J > 0) {
      constexpr int kItems = kPrRows * (HD / 8) / 256, kBatch = 16 < kItems ? 16 : kItems;
#pragma unroll 1
      for (int k0 = 0; k0 < kItems; k0 += kBatch) {
        uint4 x[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int e = (k0 + k) * 256 + tid, rr = e / (HD / 8), d0 = e % (HD / 8) * 8;
          const int qi = (row0 + rr) / group, qh = (row0 + rr) - qi * group;
          x[k] = make_uint4(0, 0, 0, 0);
          if (qi < cnt)
            x[k] = kv8_load8(p.q + b * p.ldqb + qi * p.ldqt + (int64_t)(kvh * group + qh) * p.ldqh, d0, HD, p.rope,
                             rot0 + qi);
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int e = (k0 + k) * 256 + tid, rr = e / (HD / 8), c = e % (HD / 8), tr = rr & (kPrTile - 1);
          *reinterpret_cast<uint4*>(pp_smem + S::kQ + rr / kPrTile * S::kQTile + c / 8 * (kPrTile * 128) + tr * 128 +
                                    (((c & 7) ^ (tr & 7)) << 4)) =
              make_uint4(x[k].x ^ p.q_sign, x[k].y ^ p.q_sign, x[k].z ^ p.q_sign, x[k].w ^ p.q_sign);
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      for (int j = j0 + tid; j < min(j1, coded); j += 256) vref = fmaxf(vref, v_scale[j]);
      if (j1 > coded) {  // the open block's values, zero past the end and where they are infinite or NaN
        uint32_t odd = 0;
#pragma unroll
        for (int k = 0; k < kTailItems; ++k) {
          const int e = k * 256 + tid, row = e / (HD / 8);
          open[k] = make_uint4(0, 0, 0, 0);
          if (coded * kKvBlock + row < len)
            open[k] = *reinterpret_cast<const uint4*>(p.c.tail_row(1, b, kvh, row) + e % (HD / 8) * 8);
        }
#pragma unroll
        for (int k = 0; k < kTailItems; ++k) {
          odd |= kv8_drop_odd(open[k]);
          vref = fmaxf(vref, kv8_amax8(open[k]) * 0x1p-15f);
        }
        if (odd) s_odd = 1;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) vref = fmaxf(vref, __shfl_xor_sync(0xffffffffu, vref, o));
    if (lane == 0) s_red[warp] = vref;
    asm volatile("bar.sync 1, 256;" ::: "memory");  // the eight softmax warps, all of which come here
    for (int k = 0; k < 8; ++k) vref = fmaxf(vref, s_red[k]);
    vref = __uint_as_float((__float_as_uint(vref) + 0x7fffffu) & 0xff800000u);
    if (!(vref > 0.f)) vref = 1.f;  // every value is zero
    const float per_vref = 1.f / vref;
    if (J > 0 && j1 > coded) {
#pragma unroll
      for (int k = 0; k < kTailItems; ++k) {
        uint32_t y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = __half22float2(u2h(kv8_word(open[k], i)));
          y[i] = h2u(__floats2half2_rn(f.x * per_vref, f.y * per_vref));
        }
        *reinterpret_cast<uint4*>(pp_smem + S::kTail + (k * 256 + tid) * 16) = make_uint4(y[0], y[1], y[2], y[3]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(tail_full);
    }
    const int t = warp >> 2, r = row0 + t * kPrTile + (warp & 3) * 32 + lane;
    const int i = r / group, h = r - i * group;
    const int stop = r < rows ? kv8_row_stop(i, len, cnt) : 0;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_cols = tmem + lanes + (uint32_t)(t * HD);
    float m = -INFINITY, l = 0.f;
    float ks = 1.f, vs = vref;  // of the next block
    if (J > 0 && j0 < coded) {
      ks = k_scale[j0];
      vs = v_scale[j0];
    }
    bool fine = true;
#pragma unroll 1
    for (int j = 0; j < J; ++j) {
      const int blk = j0 + j, buf = j & 1;
      const float k = fmaxf(ks * p.scale2, 1e-30f);  // positive: a masked score stays -inf
      const float log_f = vs == 0.f ? 0.f : __log2f(vs * per_vref);
      ks = 1.f;
      vs = vref;
      if (blk + 1 < min(j1, coded)) {
        ks = k_scale[blk + 1];
        vs = v_scale[blk + 1];
      }
      const int nv = min(max(stop - blk * kKvBlock, 0), kKvBlock);  // positions of the block that the row attends
      const bool masked = __any_sync(0xffffffffu, nv < kKvBlock);
      if (!(fine = wait(s_full + 8 * (2 * t + buf), (j >> 1) & 1))) break;
      tc_fence_after();
      const uint32_t s_cols = tmem + lanes + 256u + (uint32_t)((2 * t + buf) * kKvBlock);
      // the maximum first; the scores are read again for the weights, half a row
      // at a time (64 registers fewer)
      float mx[4];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t s[32];
        tc_ld32(s_cols + 32 * c, s);
        if (masked) {
#pragma unroll
          for (int u = 0; u < 32; ++u)
            if (32 * c + u >= nv) s[u] = 0xff800000u;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float x = __uint_as_float(s[16 * u]);
#pragma unroll
          for (int e = 1; e < 16; ++e) x = fmaxf(x, __uint_as_float(s[16 * u + e]));
          mx[2 * c + u] = x;
        }
      }
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * k;
      const bool grow = top > m + kPrLag;
      if (__any_sync(0xffffffffu, grow)) {
        const float to = grow ? top : m;
        const float g = m == to || m == -INFINITY ? 1.f : ex2(m - to);  // a row without a maximum has only zeros
        l *= g;
        m = to;
        if (j > 0 && __any_sync(0xffffffffu, g != 1.f)) {
          // the products up to the last block are in O
          if (!(fine = wait(o_full + 8 * (2 * t + (buf ^ 1)), ((j - 1) >> 1) & 1))) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < HD; c += 32) {
            uint32_t o[32];
            tc_ld32(o_cols + c, o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * g);
            tc_st32(o_cols + c, o);
          }
        }
      }
      const float shift = (m == -INFINITY ? 0.f : -m) + kPrLift + log_f;
      const uint64_t k2 = f32_pair(k, k), shift2 = f32_pair(shift, shift);
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t s[32], w[16];  // half a row's weights, over scores that have been read
        tc_ld32(s_cols + 32 * c, s);
        if (masked) {
#pragma unroll
          for (int u = 0; u < 32; ++u)
            if (32 * c + u >= nv) s[u] = 0xff800000u;
        }
#pragma unroll
        for (int u = 0; u < 32; u += 2) {
          float x, y;
          f32_split(f32_fma2(f32_pair(__uint_as_float(s[u]), __uint_as_float(s[u + 1])), k2, shift2), x, y);
          x = ex2(x);
          y = ex2(y);
          sum[u / 2 & 1] = f32_add2(sum[u / 2 & 1], f32_pair(x, y));
          w[u / 2] = h2u(__floats2half2_rn(x, y));
        }
        tc_st16(s_cols + 16 * c, w);
      }
      float sx, sy;
      f32_split(f32_add2(sum[0], sum[1]), sx, sy);
      l = fmaf(sx + sy, ex2(-log_f), l);
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + 8 * (2 * t + buf));
    }
    if (J > 0 && fine) fine = wait(done, 0);
    tc_fence_after();
    const bool empty = J == 0 || !fine;
    const float inv = empty || l == 0.f ? 0.f : vref / l;
    // The results leave by way of shared memory, which nothing else uses any
    // more, so that a row's bytes go out side by side (a thread has a whole row).
    const bool parts = splits > 1;
    char* mine = reinterpret_cast<char*>(pp_smem) + warp * (32 * HD * 4);  // this warp's 32 rows
    char* to = nullptr;  // where row `lane` goes
    if (r < rows)
      to = parts ? reinterpret_cast<char*>(p.part + ((((int64_t)split * p.c.batch + b) * p.c.nkv + kvh) * rows + r) * HD)
                 : reinterpret_cast<char*>(p.out + b * p.ldob + i * p.ldot + (int64_t)(kvh * group + h) * p.ldoh);
    const int row_bytes = parts ? HD * 4 : HD * 2;
#pragma unroll
    for (int c = 0; c < HD; c += 32) {
      uint32_t o[32];
      if (!empty) tc_ld32(o_cols + c, o);
      else {
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = 0;
      }
      if (parts) {
#pragma unroll
        for (int e = 0; e < 32; e += 4)
          *reinterpret_cast<float4*>(mine + lane * row_bytes + (((c + e) / 4 ^ (lane & 7)) << 4)) =
              make_float4(__uint_as_float(o[e]) * vref, __uint_as_float(o[e + 1]) * vref,
                          __uint_as_float(o[e + 2]) * vref, __uint_as_float(o[e + 3]) * vref);
      } else {
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          uint32_t x[4];
#pragma unroll
          for (int u = 0; u < 4; ++u)
            x[u] = h2u(__floats2half2_rn(__uint_as_float(o[e + 2 * u]) * inv, __uint_as_float(o[e + 2 * u + 1]) * inv));
          *reinterpret_cast<uint4*>(mine + lane * row_bytes + (((c + e) / 8 ^ (lane & 7)) << 4)) =
              make_uint4(x[0], x[1], x[2], x[3]);
        }
      }
    }
    __syncwarp();
    const int chunks = row_bytes / 16;  // 8, 16 or 32: a power of two
#pragma unroll 4
    for (int k = lane; k < 32 * chunks; k += 32) {
      const int rr = k / chunks, c = k % chunks;
      char* dst = reinterpret_cast<char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(to), rr));
      if (dst) *reinterpret_cast<uint4*>(dst + c * 16) = *reinterpret_cast<const uint4*>(mine + rr * row_bytes + ((c ^ (rr & 7)) << 4));
    }
    if (parts && r < rows)
      reinterpret_cast<float2*>(p.part + (int64_t)p.splits * p.c.batch * p.c.nkv * rows * HD)
          [(((int64_t)split * p.c.batch + b) * p.c.nkv + kvh) * rows + r] = make_float2(empty ? -INFINITY : m, empty ? 0.f : l);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp < 16) {
      // --------------------------------------------------------------- unpack
      // warps 8-11 values, 12-15 keys; rows 32 (w & 1) + lane, sixteen-dimension
      // chunks of parity w >> 1
      const int w = warp & 3, side = warp < 12 ? 1 : 0;
      const int r = (w & 1) * 32 + lane;
      constexpr int kChunks = HD / 32;
      const uint32_t full = side ? v_full : k_full, empty = side ? v_empty : k_empty;
      const uint32_t src = base + S::kCodes + side * S::kCode, dst = base + (side ? S::kV : S::kK) + r * 128;
#pragma unroll 1
      for (int j = 0; j < J; ++j) {
        const int st = j % kPrCodeStages, buf = j & 1;
        const bool is_tail = j0 + j >= coded;
        uint4 lo[kChunks], hi[kChunks];
        bool fine = true;
        if (!is_tail) {
          fine = wait(code_full + 8 * st, (j / kPrCodeStages) & 1);
          uint4 x[kChunks];
#pragma unroll
          for (int cc = 0; cc < kChunks; ++cc)
            x[cc] = lds128(src + 2 * st * S::kCode + tile_off<HD>(r, 2 * cc + (w >> 1)));
#pragma unroll
          for (int cc = 0; cc < kChunks; ++cc) {
            lo[cc] = make_uint4(codes2<0x4140>(x[cc].x), codes2<0x4342>(x[cc].x), codes2<0x4140>(x[cc].y),
                                codes2<0x4342>(x[cc].y));
            hi[cc] = make_uint4(codes2<0x4140>(x[cc].z), codes2<0x4342>(x[cc].z), codes2<0x4140>(x[cc].w),
                                codes2<0x4342>(x[cc].w));
          }
        } else {  // FP16 rows, zero past the end
          if (side) fine = wait(tail_full, 0);
          const __half* tail =
              side ? reinterpret_cast<const __half*>(pp_smem + S::kTail + r * HD * 2) : p.c.tail_row(0, b, kvh, r);
#pragma unroll
          for (int cc = 0; cc < kChunks; ++cc) {
            lo[cc] = hi[cc] = make_uint4(0, 0, 0, 0);
            if ((j0 + j) * kKvBlock + r < len) {
              const uint4* g = reinterpret_cast<const uint4*>(tail + 16 * (2 * cc + (w >> 1)));
              lo[cc] = g[0];
              hi[cc] = g[1];
            }
          }
        }
        if (j > 1) fine = fine && wait(empty + 8 * buf, ((j >> 1) - 1) & 1);
        if (!fine) break;
#pragma unroll
        for (int cc = 0; cc < kChunks; ++cc) {
          const int c = 2 * cc + (w >> 1), ch = 2 * (c & 3);
          const uint32_t to = dst + buf * S::kKv + c / 4 * (kKvBlock * 128);
          asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(to + ((ch ^ (r & 7)) << 4)), "r"(lo[cc].x),
                       "r"(lo[cc].y), "r"(lo[cc].z), "r"(lo[cc].w) : "memory");
          asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(to + (((ch + 1) ^ (r & 7)) << 4)), "r"(hi[cc].x),
                       "r"(hi[cc].y), "r"(hi[cc].z), "r"(hi[cc].w) : "memory");
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(full + 8 * buf);
          if (!is_tail) mbar_arrive(code_empty + 8 * st);
        }
      }
    } else if (warp == 16) {
      // ------------------------------------------------------------- S = Q K^T
      // Two blocks ahead of the second product, into the buffer whose weights it
      // has read.  Descriptors' offsets within a tile add to their address field.
      constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(kKvBlock >> 3) << 17) | ((uint32_t)(kPrTile >> 4) << 24);
      const uint64_t q_desc = sw128_desc(base + S::kQ, 16, 1024), k_desc = sw128_desc(base + S::kK, 16, 1024);
      bool fine = J == 0 || wait(q_full, 0);
#pragma unroll 1
      for (int j = 0; j < J && fine; ++j) {
        const int buf = j & 1;
        const uint64_t kd = k_desc + (uint32_t)(buf * (S::kKv >> 4));
        fine = wait(k_full + 8 * buf, (j >> 1) & 1);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (j > 1) fine = fine && wait(o_full + 8 * (2 * t + buf), ((j >> 1) - 1) & 1);
          if (!fine) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t qd = q_desc + (uint32_t)(t * (S::kQTile >> 4));
            const uint32_t dst = tmem + 256u + (uint32_t)((2 * t + buf) * kKvBlock);
#pragma unroll
            for (int d = 0; d < HD / 16; ++d)
              tc_mma(dst, qd + (d / 4 * (kPrTile * 128) + d % 4 * 32 >> 4),
                     kd + (d / 4 * (kKvBlock * 128) + d % 4 * 32 >> 4),
                     idesc, d > 0);
            tc_commit(s_full + 8 * (2 * t + buf));
            if (t == 1) tc_commit(k_empty + 8 * buf);
          }
          __syncwarp();
        }
      }
      if (J > 0) wait(done, 0);  // no product outlives the tensor memory
    } else if (warp == 18) {
      // --------------------------------------------------------------- O += P V
      constexpr uint32_t idesc =
          (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(kPrTile >> 4) << 24);
      const uint64_t v_desc = sw128_desc(base + S::kV, kKvBlock * 128, 1024);
      bool fine = true;
#pragma unroll 1
      for (int j = 0; j < J && fine; ++j) {
        const int buf = j & 1;
        const uint64_t vd = v_desc + (uint32_t)(buf * (S::kKv >> 4));
        fine = wait(v_full + 8 * buf, (j >> 1) & 1);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          fine = fine && wait(p_full + 8 * (2 * t + buf), (j >> 1) & 1);
          if (!fine) break;
          tc_fence_after();
          if (elect_one()) {
            const uint32_t pa = tmem + 256u + (uint32_t)((2 * t + buf) * kKvBlock);
#pragma unroll
            for (int x = 0; x < kKvBlock / 16; ++x)
              tc_mma_ta(tmem + (uint32_t)(t * HD), pa + 8 * x, vd + (x * 2048 >> 4), idesc, j > 0 || x > 0);
            tc_commit(o_full + 8 * (2 * t + buf));
            if (t == 1) tc_commit(v_empty + 8 * buf);
          }
          __syncwarp();
        }
      }
      if (elect_one()) tc_commit(done);
      __syncwarp();
      wait(done, 0);
    } else if (warp == 17 && lane == 0) {
      // ------------------------------------------------------------ code boxes
      const int n = min(j1, coded) - j0;
      int issued = 0;
      for (int j = 0; j < n; ++j, ++issued) {
        const int st = j % kPrCodeStages;
        if (j >= kPrCodeStages && !mbar_wait_bounded(code_empty + 8 * st, (j / kPrCodeStages - 1) & 1, p.status)) break;
        const int y = (int)(p.c.head(b, kvh) * p.c.cap) + (j0 + j) * kKvBlock;
        mbar_expect_tx(code_full + 8 * st, 2 * S::kCode);
        tma_load_2d(base + S::kCodes + 2 * st * S::kCode, &tk, 0, y, code_full + 8 * st);
        tma_load_2d(base + S::kCodes + (2 * st + 1) * S::kCode, &tv, 0, y, code_full + 8 * st);
      }
      for (int j = max(0, issued - kPrCodeStages); j < issued; ++j)  // none stays in flight
        mbar_wait_bounded(code_full + 8 * (j % kPrCodeStages), (j / kPrCodeStages) & 1, p.status);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid < kPrRows && s_odd) kv8_prompt_add_odd<HD>(p, splits > 1);  // the results are written
  if (warp == 16) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// The parts of a row (splits > 1) added up in order; a warp has one row.
struct Kv8JoinParams {
  const float* part;
  __half* out;
  int64_t ldob, ldot, ldoh;
  const int* lens;
  const int* part_blocks;
  int batch, nkv, n, nq, splits, cap;
};

template <int HD>
__global__ void __launch_bounds__(256) kv8_join_kernel(const Kv8JoinParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int group = p.nq / p.nkv, rows = p.n * group;
  const int64_t all = (int64_t)p.batch * p.nkv * rows;
  const int64_t at = blockIdx.x * (int64_t)8 + (threadIdx.x >> 5);
  if (at >= all) return;
  const int lane = threadIdx.x & 31, r = (int)(at % rows), kvh = (int)(at / rows % p.nkv), b = (int)(at / rows / p.nkv);
  const int splits = kv8_seq_parts(kv8_seq_blocks(p.lens[b], p.cap), *p.part_blocks, p.splits);
  if (splits == 1) return;  // written by its only part
  constexpr int kPer = HD / 32;
  const float2* ml = reinterpret_cast<const float2*>(p.part + (int64_t)p.splits * all * HD);
  float m = -INFINITY, l = 0.f, o[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) o[e] = 0.f;
  for (int s0 = 0; s0 < splits; s0 += 4) {  // four parts' loads at a time
    float2 v[4], x[4][kPer / 2];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      v[s] = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int e = 0; e < kPer / 2; ++e) x[s][e] = make_float2(0.f, 0.f);
      if (s0 + s < splits) {
        v[s] = ml[(s0 + s) * all + at];
#pragma unroll
        for (int e = 0; e < kPer / 2; ++e)
          x[s][e] = *reinterpret_cast<const float2*>(p.part + ((s0 + s) * all + at) * HD + lane * 2 + 64 * e);
      }
    }
    float to = m;
#pragma unroll
    for (int s = 0; s < 4; ++s) to = fmaxf(to, v[s].x);
    const float f0 = m == -INFINITY ? 1.f : ex2(m - to);
    l *= f0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[e] *= f0;
    m = to;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const float f = v[s].x == -INFINITY ? 1.f : ex2(v[s].x - m);
      l = fmaf(v[s].y, f, l);
#pragma unroll
      for (int e = 0; e < kPer / 2; ++e) {
        o[2 * e] = fmaf(x[s][e].x, f, o[2 * e]);
        o[2 * e + 1] = fmaf(x[s][e].y, f, o[2 * e + 1]);
      }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int i = r / group, h = r - i * group;
  __half* out = p.out + b * p.ldob + i * p.ldot + (int64_t)(kvh * group + h) * p.ldoh;
#pragma unroll
  for (int e = 0; e < kPer; e += 2)
    *reinterpret_cast<__half2*>(out + lane * 2 + 32 * e) = __floats2half2_rn(o[e] * inv, o[e + 1] * inv);  // e even: 64 halves apart
}

}  // namespace pp
