// Decode attention over the 8-bit KV cache: few query rows per kv head, any
// cache length (kv8_attention.cu launches it).
//
// Mathematics.  With S = scale * s_k (q . (c_k - 128)) for the codes c_k of a
// block, out = sum_blocks s_v (P (c_v - 128)) / sum P, P = exp(S - m): the
// codes enter the products as the exact FP16 integers -128..127 and the block
// scales are applied in FP32 beside them.  P is rounded to FP16 relative to its
// own unit's maximum m (2^-11 of values up to 1), everything else is FP32.
//
// Bound: the cache's bytes at long lengths, latency at short ones.  Work is
// counted in units, a block of codes or 16 FP16 rows of the tail, over all
// (sequence, kv head, row tile) segments in a row, and each CTA takes an equal
// share of them, so ragged batches balance; where the segments divide the GPU
// nearly evenly, no share spans two of them.  The shares come from the lengths
// in device memory.  A warp holds one block, keys and values apart, each
// arriving by a swizzled TMA box; the next block's keys are on their way while
// it works on the values, and the other way round.  Keys are the A operand of
// m16n8k16 (16 positions x 8 rows), read by ldmatrix with the four dimensions
// of a lane's word as its k elements, values by transposed ldmatrix, whose
// word holds two dimensions at two positions: both orders cost nothing, since
// the queries and the outputs take the same permutation.
//
// Measured: 4 sequences of 1024, 16 query heads on 2 kv heads of 128: 11 us, a
// chain of launch, lengths, boxes, products and join (13 us with two tokens each); 64 ragged sequences up
// to 8190, 28 heads on 4, 244 MB: 64 us, 3.8 TB/s, bound by the warps' chains
// of instructions (about 1200 a block; three warps to a scheduler keep 39% of
// its slots busy) and by the barriers where segments end.
#pragma once

#include "kv8.cuh"

namespace pp {

constexpr int kDecTailUnit = 16;  // FP16 rows of a tail unit; a coded unit is a block

// Warps of a CTA (one CTA per SM): 12 while a row tile is 8 rows, 8 warps with
// twice the accumulators for 16 rows.
constexpr int kv8_warps(int nt) { return nt == 1 ? 12 : 8; }

// Units that a CTA takes at least: with fewer than one to a warp, more SMs
// share a short cache and their warps do not compete for issue slots.
constexpr int kDecMinUnits = 4;

struct Kv8DecodeParams {
  Kv8Cache c;
  const __half* q;
  int64_t ldqb, ldqt, ldqh;
  __half* out;
  int64_t ldob, ldot, ldoh;
  const int* lens;
  int extra;                 // 1: the call's own token follows the lens[b] of the cache
  const int* counts;
  int n, nq, tiles;          // query tokens, query heads, row tiles per kv head
  float scale2;              // scale * log2(e)
  Kv8Rope rope;
  const __half* x[2];        // the token's key and value rows (extra == 1)
  int64_t ldxb[2], ldxh[2];
  int* cnt;                  // [ctas] arrivals at the segment whose units begin in that CTA, zero between launches
  float* part;               // [ctas][2] partial results
  float* lse;                // [batch][nq] log2 of the softmax sums (scores != NULL)
  float* scores;             // [batch][nq][cap] log2-scaled scores, or NULL
  int* status;
};

template <int NT, int HD>
struct Kv8DecodeSmem {
  static constexpr int kWarps = kv8_warps(NT);
  static constexpr int kSlot = kKvBlock * HD;                    // a block's keys or values
  static constexpr int kRounds = NT == 1 ? 2 : 1;                // the warps' results are added up in as many parts
  static constexpr int kPart = HD / 16 / kRounds * NT * 4;       // floats a lane contributes to one
  static constexpr int kMerge = kWarps * 2 * kSlot;
  static constexpr int kMl = kMerge + kWarps * kPart * 32 * 4;   // each warp's row maxima and sums
  static constexpr int kQ = kMl + kWarps * NT * 8 * 8;           // query rows, then the token's key and value
  static constexpr int kQRow = HD * 2 + 32;                      // conflict-free 8-byte reads of eight rows
  static constexpr int kNew = kQ + NT * 8 * kQRow;
  static constexpr int kBar = kNew + 2 * HD * 2;
  static constexpr int kLens = kBar + kWarps * 2 * 8;            // lengths, then unit prefix
  static constexpr int bytes(int batch) { return kLens + (2 * batch + 2) * 4; }
};

// Floats of one partial result: NT * 8 rows of HD sums, then maxima and sums.
__host__ __device__ constexpr int kv8_part_floats(int nt, int hd) { return nt * 8 * (hd + 2); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// D = A B + 0.
__device__ __forceinline__ void mma_16816_0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// Two codes of a word as FP16 integers code - 128: the byte in the low half of
// 0x6400 is 1024 + code, exactly.
template <int SEL>
__device__ __forceinline__ uint32_t codes2(uint32_t w) {
  return h2u(__hsub2(u2h(__byte_perm(w, 0x64646464u, SEL)), __float2half2_rn(1152.f)));
}

// Byte offset of 16-byte chunk c of row r in a swizzled tile (128-byte or
// 64-byte rows, as the tensor maps of launch_decode order them).  For an even
// k, chunk k + c (c = 0, 1) lies at the offset of chunk c xor 16 k.
template <int HD>
__device__ __forceinline__ uint32_t tile_off(int r, int c) {
  return HD == 128 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
}

// One warp's running result: NT tiles of 8 rows (the columns of its mma
// accumulators).  A lane holds rows 2 (lane & 3) + j of a tile; o[i][nt][j]
// and o[i][nt][2 + j] are dimensions 16 i + 2 (lane >> 2) and the next.
template <int NT, int HD>
struct Kv8Acc {
  float o[HD / 16][NT][4];
  float m[NT][2], l[NT][2];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < HD / 16; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][nt][e] = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        m[nt][j] = -INFINITY;
        l[nt][j] = 0.f;
      }
  }

  // Moves the reference of row (nt, j) to `to`.
  __device__ __forceinline__ void rebase(int nt, int j, float to) {
    const float f = m[nt][j] == -INFINITY ? 0.f : ex2(m[nt][j] - to);
    m[nt][j] = to;
    l[nt][j] *= f;
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) {
      o[i][nt][j] *= f;
      o[i][nt][2 + j] *= f;
    }
  }
};

// Scores s[mt] (16 positions each, log2-scaled, masked) to probabilities
// relative to the unit's maximum.  Gives each row's factor that brings the
// unit's sums to the running reference, which moves only when the maximum
// outgrows it by 2^8, so most units rescale nothing; and P^T as B operands.
template <int NT, int HD, int MT>
__device__ __forceinline__ void kv8_softmax(Kv8Acc<NT, HD>& a, float (&s)[MT][NT][4], float (&gain)[NT][2],
                                            uint32_t (&pb)[MT][NT][2]) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float mu[2];
    bool grow = false;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float m = s[0][nt][j];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) m = fmaxf(m, fmaxf(s[mt][nt][j], s[mt][nt][2 + j]));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
      mu[j] = m;
      grow |= m > a.m[nt][j] + 8.f;
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (mu[j] > a.m[nt][j] + 8.f) a.rebase(nt, j, mu[j]);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float base = mu[j] == -INFINITY ? 0.f : mu[j];
      gain[nt][j] = mu[j] == -INFINITY ? 0.f : ex2(mu[j] - a.m[nt][j]);
      float sum = 0.f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float e = ex2(s[mt][nt][2 * h + j] - base);
          s[mt][nt][2 * h + j] = e;
          sum += e;
        }
      a.l[nt][j] = fmaf(sum, gain[nt][j], a.l[nt][j]);
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        pb[mt][nt][h] = transpose8(h2u(__floats2half2_rn(s[mt][nt][2 * h], s[mt][nt][2 * h + 1])));
  }
}

// The first n rows of a tail unit's values, at v in shared memory, without those
// that are infinite or NaN (kv8_drop_odd); whether there were any.
template <int HD>
__device__ __forceinline__ bool kv8_drop_odd_rows(uint32_t v, int n) {
  const int lane = threadIdx.x & 31;
  __half2 top = __float2half2_rn(0.f);
#pragma unroll
  for (int k = 0; k < kDecTailUnit * HD / 8 / 32; ++k) {
    const int e = k * 32 + lane;
    const uint4 x = lds128(v + e * 16);
    const __half2 m = __hmax2_nan(__hmax2_nan(__habs2(u2h(x.x)), __habs2(u2h(x.y))),
                                  __hmax2_nan(__habs2(u2h(x.z)), __habs2(u2h(x.w))));
    if (e < n * (HD / 8)) top = __hmax2_nan(top, m);
  }
  const float2 f = __half22float2(top);
  if (__all_sync(0xffffffffu, f.x <= 65504.f && f.y <= 65504.f)) return false;
#pragma unroll 1
  for (int e = lane; e < n * (HD / 2); e += 32) {
    uint32_t x = lds_u32(v + e * 4);
    kv8_drop_odd(x);
    sts_u32(v + e * 4, x);
  }
  return true;
}

// What a CTA knows of the launch's work: effective lengths and unit counts.
// A segment counts kDecSegmentUnits more units than it has, at its end, for
// the time between two segments of a CTA (about 3 us, which at the memory's
// rate is eight blocks): shares with many short segments get fewer blocks.
constexpr int kDecSegmentUnits = 8;

struct Kv8Work {
  const int* len;   // [batch], 0 for sequences without work
  const int* pre;   // [batch + 1] counted units before each sequence, all heads and tiles
  int batch, per_seq;  // segments per sequence: kv heads x row tiles
  __device__ __forceinline__ static int units(int len) {
    if (len <= 0) return 0;
    const int last = kv8_last_block(len);
    return last + (len - last * kKvBlock + kDecTailUnit - 1) / kDecTailUnit;
  }
  __device__ __forceinline__ static int counted(int len) { return len > 0 ? units(len) + kDecSegmentUnits : 0; }
};

// Where a counted unit falls: sequence, segment of the sequence, unit.
struct Kv8Cursor {
  int b, seg, u, U;  // U: counted units of the segment
  __device__ __forceinline__ void seek(const Kv8Work& w, int idx) {
    int lo = 0, hi = w.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (w.pre[mid] <= idx) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
    U = Kv8Work::counted(w.len[b]);
    seg = (idx - w.pre[b]) / U;
    u = idx - w.pre[b] - seg * U;
  }
  // To the start of the next segment, which must exist.
  __device__ __forceinline__ void next(const Kv8Work& w) {
    u = 0;
    if (++seg < w.per_seq) return;
    seg = 0;
    do ++b;
    while (w.pre[b + 1] == w.pre[b]);
    U = Kv8Work::counted(w.len[b]);
  }
};

// The blocks of the cache that a token completes, and the token's own row in
// the tail: nothing that attends in this launch reads either.
template <int HD, int WARPS>
__device__ __forceinline__ void kv8_store_token(const Kv8DecodeParams& p, const int* s_len, float* red) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int items = p.c.batch * p.c.nkv * 2;
  const int cta = gridDim.x - 1 - blockIdx.x;  // idle CTAs of short launches come first
  auto row8 = [&](int w, int b, int h, int d0) {
    Kv8Rope r = w == 0 ? p.rope : Kv8Rope{};
    return kv8_load8(pick(p.x, w) + b * pick(p.ldxb, w) + h * pick(p.ldxh, w), d0, HD, r, r.cos ? r.pos[b] : 0);
  };
  for (int i = cta * WARPS + warp; i < items; i += gridDim.x * WARPS) {
    const int w = i & 1, h = (i >> 1) % p.c.nkv, b = (i >> 1) / p.c.nkv, len = s_len[b];
    if (len > 0 && lane < HD / 8)
      *reinterpret_cast<uint4*>(p.c.tail_row(w, b, h, (len - 1) % kKvBlock) + 8 * lane) = row8(w, b, h, 8 * lane);
  }
  constexpr int kThreads = WARPS * 32, kItems = kKvBlock * HD / 8, kVecs = (kItems + kThreads - 1) / kThreads;
  for (int i = cta; i < items; i += gridDim.x) {
    const int w = i & 1, h = (i >> 1) % p.c.nkv, b = (i >> 1) / p.c.nkv, len = s_len[b];
    if (len <= 0 || len % kKvBlock) continue;  // the same for the whole CTA
    uint4 v[kVecs];
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int e = k * kThreads + threadIdx.x, r = e / (HD / 8), d0 = e % (HD / 8) * 8;
      v[k] = e >= kItems ? make_uint4(0, 0, 0, 0)
             : r == kKvBlock - 1 ? row8(w, b, h, d0)
                                 : *reinterpret_cast<const uint4*>(p.c.tail_row(w, b, h, r) + d0);
    }
    const Kv8Scale q = kv8_block_scale<kVecs, kThreads>(v, red);
    const int block = len / kKvBlock - 1;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int e = k * kThreads + threadIdx.x, r = e / (HD / 8), d0 = e % (HD / 8) * 8;
      if (e < kItems) *reinterpret_cast<uint2*>(p.c.code_row(w, b, h, block * kKvBlock + r) + d0) = kv8_codes8(v[k], q);
    }
    if (threadIdx.x == 0) *p.c.scale(w, b, h, block) = q.scale;
  }
}

// A segment of which a CTA has only a part.
struct Kv8Part {
  int b, kvh, row0, rows, seg0, first, contrib, last;
};

// Adds the values of the tail rows u0 to u1 that are infinite or NaN to the
// results of the rows that attend them, in rec or (NULL) in the output.
template <int NT, int HD>
__device__ __noinline__ void kv8_add_odd(const Kv8DecodeParams& p, int b, int kvh, int row0, int rows, int cnt, int len,
                                         int u0, int u1, float* rec) {
  const int group = p.nq / p.c.nkv, t0 = kv8_last_block(len) * kKvBlock;
  for (int e = threadIdx.x; e < HD / 16 * NT * 2 * 32; e += kv8_warps(NT) * 32) {
    const int el = e & 31, r = (e >> 6) % NT * 8 + 2 * (el & 3) + ((e >> 5) & 1);
    const int d = 16 * ((e >> 6) / NT) + 2 * (el >> 2), i = (row0 + r) / group, h = row0 + r - i * group;
    if (r >= rows || i >= cnt) continue;
    float x = 0.f, y = 0.f;
    for (int t = u0; t < min(u1, len - cnt + i + 1 - t0); ++t) {
      uint32_t v = *reinterpret_cast<const uint32_t*>(p.c.tail_row(1, b, kvh, t) + d), rest = v;
      v &= kv8_drop_odd(rest);
      x += __low2float(u2h(v));
      y += __high2float(u2h(v));
    }
    if (x == 0.f && y == 0.f) continue;
    if (rec) {
      rec[r * HD + d] += x;
      rec[r * HD + d + 1] += y;
    } else {
      __half2* o = reinterpret_cast<__half2*>(p.out + b * p.ldob + i * p.ldot + (int64_t)(kvh * group + h) * p.ldoh + d);
      *o = __floats2half2_rn(__low2float(*o) + x, __high2float(*o) + y);
    }
  }
}

// MANY: the call has several query tokens (a single one attends all of the
// tail).  Its own kernel, as the other is 2 to 4% slower with its code.
template <int NT, int HD, bool MANY>
__global__ void __launch_bounds__(kv8_warps(NT) * 32, 1)
    kv8_decode_kernel(const __grid_constant__ Kv8DecodeParams p, const __grid_constant__ CUtensorMap tk,
                      const __grid_constant__ CUtensorMap tv) {
  using S = Kv8DecodeSmem<NT, HD>;
  constexpr int kWarps = S::kWarps, kThreads = kWarps * 32, kPartFloats = kv8_part_floats(NT, HD);
  __shared__ float red[kWarps];
  __shared__ int s_max;
  __shared__ int s_odd;  // the last segment with values in the tail that are infinite or NaN
  __shared__ Kv8Part s_part[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const uint32_t base = (uint32_t)__cvta_generic_to_shared(pp_smem);
  const uint32_t k_slot = base + warp * 2 * S::kSlot, v_slot = k_slot + S::kSlot;
  const uint32_t k_bar = base + S::kBar + warp * 16, v_bar = k_bar + 8;
  int* s_len = reinterpret_cast<int*>(pp_smem + S::kLens);
  int* s_pre = s_len + p.c.batch;
  if (tid == 0) s_odd = -1;
  if (lane == 0) {
    mbar_init(k_bar, 1);
    mbar_init(v_bar, 1);
    fence_mbar_init();
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
  }
  pdl_launch_dependents();
  pdl_wait();

  // Where the segments divide the CTAs, this CTA's segment does not depend on
  // the lengths: its rows are fetched together with them.
  const int group = p.nq / p.c.nkv, ctas = gridDim.x;
  const Kv8Work work{s_len, s_pre, p.c.batch, p.c.nkv * p.tiles};
  const int each = ctas / (p.c.batch * work.per_seq);  // CTAs per segment, if every one gets as many
  auto query_row8 = [&](int b, int kvh, int row0, int e) {  // item e of a tile's rows (padding rows are zero)
    const int r = e / (HD / 8), d0 = e % (HD / 8) * 8;
    const int i = p.n == 1 ? 0 : (row0 + r) / group, h = row0 + r - i * group;
    if (r >= NT * 8 || i >= p.n || h >= group) return make_uint4(0, 0, 0, 0);
    const int t0 = p.rope.cos ? p.rope.pos[b] : 0;
    if (p.rope.cos && (t0 < 0 || t0 >= p.rope.len - i)) return make_uint4(0, 0, 0, 0);
    return kv8_load8(p.q + b * p.ldqb + i * p.ldqt + (int64_t)(kvh * group + h) * p.ldqh, d0, HD, p.rope, t0 + i);
  };
  auto token_row8 = [&](int b, int kvh, int e) {  // the token's key, then its value
    const int w = e / (HD / 8), d0 = e % (HD / 8) * 8;
    Kv8Rope r = w == 0 ? p.rope : Kv8Rope{};
    const int t = r.cos ? r.pos[b] : 0;
    if (r.cos && (t < 0 || t >= r.len)) return make_uint4(0, 0, 0, 0);
    return kv8_load8(pick(p.x, w) + b * pick(p.ldxb, w) + kvh * pick(p.ldxh, w), d0, HD, r, t);
  };
  constexpr int kRowItems = NT * 8 * (HD / 8), kNewItems = 2 * (HD / 8);
  static_assert(kRowItems <= kThreads && kNewItems <= kThreads, "one item per thread");
  const bool is_new = p.extra && tid >= kThreads - kNewItems;
  auto fetch = [&](int b, int kvh, int row0, uint4& row, uint4& token) {
    if (tid < kRowItems) row = query_row8(b, kvh, row0, tid);
    if (is_new) token = token_row8(b, kvh, kThreads - 1 - tid);
  };
  uint4 row{}, token{};
  int have = -1;  // the segment whose rows these are
  if (each > 0 && (int)blockIdx.x / each < p.c.batch * work.per_seq) {
    have = blockIdx.x / each;
    const int s = have % work.per_seq;
    fetch(have / work.per_seq, s / p.tiles, s % p.tiles * NT * 8, row, token);
  }

  // lengths and the units before each sequence; every warp for itself while a
  // warp's lanes hold them all (all write the same), else the CTA together
  auto length = [&](int b) {
    const int held = p.lens[b];
    const int cnt = p.counts ? min(max(p.counts[b], 0), p.n) : p.n;
    bool ok = held <= p.c.cap - p.extra;  // held + extra may pass the type's end
    const int len = ok ? held + p.extra : 1;
    if (p.rope.cos && len > 0 && cnt > 0) {
      const int r = p.rope.pos[b];
      ok = ok && r >= 0 && r <= p.rope.len - cnt;
    }
    if (!ok && blockIdx.x == 0) atomicExch(p.status, 5);
    return ok && cnt > 0 ? max(len, 0) : 0;
  };
  const bool small = p.c.batch <= 32;
  if (!small) {
    for (int b = tid; b < p.c.batch; b += kThreads) s_len[b] = length(b);
    __syncthreads();
  }
  int max_units = 0;
  if (small || warp == 0) {
    int sum = 0;
    for (int b0 = 0; b0 < p.c.batch; b0 += 32) {
      const int b = b0 + lane;
      const int len = b >= p.c.batch ? 0 : small ? length(b) : s_len[b];
      const int u = Kv8Work::counted(len);
      max_units = max(max_units, u);
      int x = u * work.per_seq;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (b < p.c.batch) {
        if (small) s_len[b] = len;
        s_pre[b + 1] = sum + x;
      }
      sum += __shfl_sync(0xffffffffu, x, 31);
    }
    for (int o = 16; o > 0; o >>= 1) max_units = max(max_units, __shfl_xor_sync(0xffffffffu, max_units, o));
    if (lane == 0) {
      s_pre[0] = 0;
      if (!small) s_max = max_units;
    }
    __syncwarp();
  }
  if (!small) {
    __syncthreads();
    max_units = s_max;
  }

  // this CTA's share [a, z) of the units
  const int total = s_pre[p.c.batch];
  const int per = max(kDecMinUnits, (total + ctas - 1) / ctas);
  const bool aligned = each > 0 && (max_units + each - 1) / each <= per + per / 4;
  auto pieces = [&](int U) { return min(each, (U + kDecMinUnits - 1) / kDecMinUnits); };
  int a = 0, z = 0;
  if (aligned) {
    if (have >= 0) {
      const int b = have / work.per_seq, j = blockIdx.x - have * each;
      const int U = Kv8Work::units(s_len[b]), k = pieces(U);
      if (j < k) {
        const int s0 = s_pre[b] + (have - b * work.per_seq) * Kv8Work::counted(s_len[b]);
        a = s0 + (int)((uint32_t)U * j / k);
        z = s0 + (int)((uint32_t)U * (j + 1) / k);
      }
    }
  } else {
    a = min((int64_t)total, (int64_t)blockIdx.x * per);
    z = min((int64_t)total, (int64_t)a + per);
  }

  // Warp w takes units a + w, a + w + kWarps, ... of the share.  A block's
  // keys or values arrive as one tensor box, a tail unit's rows (without the
  // token, which is not in the tail yet) as one plain copy.
  bool fine = true;
  int idx = a + warp, phase = 0;
  Kv8Cursor seg{};
  if (a < z) seg.seek(work, a);
  int seg_head = 0, seg_coded = 0, seg_held = 0;  // sequence and head; blocks and tokens held as codes / in all
  auto load = [&](int w, int u) {
    if (lane != 0 || !fine) return;
    const uint32_t dst = w ? v_slot : k_slot, bar = w ? v_bar : k_bar;
    if (u < seg_coded) {
      mbar_expect_tx(bar, S::kSlot);
      tma_load_2d(dst, w ? &tv : &tk, 0, (seg_head * (p.c.cap / kKvBlock) + u) * kKvBlock, bar);
    } else {
      const int r = (u - seg_coded) * kDecTailUnit;
      const uint32_t bytes = min(kDecTailUnit, max(0, seg_held - seg_coded * kKvBlock - r)) * HD * 2;
      mbar_expect_tx(bar, bytes);
      if (bytes) bulk_load(dst, pick(p.c.tail, w) + ((int64_t)seg_head * kKvBlock + r) * HD, bytes, bar);
    }
  };
  auto enter = [&](int from) {  // starts the warp's first unit of the segment that begins at unit `from`
    const int len = s_len[seg.b], u = idx - from;
    seg_head = (int)p.c.head(seg.b, p.tiles == 1 ? seg.seg : seg.seg / p.tiles);
    seg_coded = kv8_last_block(len);
    seg_held = len - p.extra;
    if (idx < min(z, from + Kv8Work::units(len))) {
      load(0, u);
      load(1, u);
    }
  };

  // A copy that does not arrive in time sets status 1; nothing stays in flight.
  auto await_keys = [&]() {
    if (fine && !mbar_wait_bounded(k_bar, phase, p.status)) {
      fine = false;
      mbar_wait_bounded(k_bar, phase, p.status);
      mbar_wait_bounded(v_bar, phase, p.status);
    }
  };
  auto await_values = [&](bool more) {  // more: the next unit's keys are on their way
    if (fine && !mbar_wait_bounded(v_bar, phase, p.status)) {
      fine = false;
      if (more) mbar_wait_bounded(k_bar, phase ^ 1, p.status);
      mbar_wait_bounded(v_bar, phase, p.status);
    }
    phase ^= 1;
  };

  // rows without work
  for (int b = blockIdx.x; b < p.c.batch; b += gridDim.x)
    if (s_len[b] == 0)
      for (int e = tid; e < p.n * p.nq * (HD / 8); e += kThreads) {
        const int d0 = e % (HD / 8) * 8, h = e / (HD / 8) % p.nq, i = e / (HD / 8) / p.nq;
        *reinterpret_cast<uint4*>(p.out + b * p.ldob + i * p.ldot + h * p.ldoh + d0) = make_uint4(0, 0, 0, 0);
      }

  auto out_at = [&](int b, int kvh, int row0, int r, int d) {
    const int i = p.n == 1 ? 0 : (row0 + r) / group, h = row0 + r - i * group;
    return reinterpret_cast<__half2*>(p.out + b * p.ldob + i * p.ldot + (int64_t)(kvh * group + h) * p.ldoh + d);
  };
  const uint32_t lane_off = tile_off<HD>(lane & 15, lane >> 4);
  bool entered = false;
  int turn = 0, pending = 0;
  for (int at = a; at < z;) {
    const int b = seg.b, segment = seg.b * work.per_seq + seg.seg;
    const int kvh = p.tiles == 1 ? seg.seg : seg.seg / p.tiles, tile = p.tiles == 1 ? 0 : seg.seg % p.tiles;
    const int len = s_len[b], coded = kv8_last_block(len);
    const int seg0 = at - seg.u, seg1 = seg0 + seg.U, U = Kv8Work::units(len);
    const int real1 = seg0 + U, end = min(z, seg1), u_end = min(z, real1) - seg0;
    if (at >= real1) {  // only counted units of this segment fall here
      at = end;
      if (end < z) {
        seg.next(work);
        idx = at + warp;
      }
      continue;
    }
    const int cnt = p.counts ? min(max(p.counts[b], 0), p.n) : p.n;
    const int row0 = tile * NT * 8, rows = min(NT * 8, p.n * group - row0);

    // the tile's query rows and the token, fetched ahead of the segment's blocks
    if (segment != have) fetch(b, kvh, row0, row, token);
    have = -1;
    if (!entered) enter(seg0);
    if (tid < kRowItems) {
      uint2* dst = reinterpret_cast<uint2*>(pp_smem + S::kQ + tid / (HD / 8) * S::kQRow + tid % (HD / 8) * 16);
      dst[0] = make_uint2(row.x, row.y);
      dst[1] = make_uint2(row.z, row.w);
    }
    if (is_new) *reinterpret_cast<uint4*>(pp_smem + S::kNew + (kThreads - 1 - tid) * 16) = token;
    // first position that row (nt, j) does not attend
    int stop[NT][2];
    int min_stop = len;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = nt * 8 + 2 * t4 + j, i = (row0 + r) / group;
        stop[nt][j] = r >= rows ? len : i < cnt ? len - cnt + i + 1 : 0;  // padding rows are zero queries
        min_stop = min(min_stop, stop[nt][j]);
      }
    const float *k_scale = p.c.scale(0, b, kvh, 0), *v_scale = p.c.scale(1, b, kvh, 0);
    float ks = 0.f, vs = 0.f;  // of the warp's next block
    if (idx - seg0 < min(u_end, coded)) {
      ks = k_scale[idx - seg0];
      vs = v_scale[idx - seg0];
    }
    __syncthreads();
    uint32_t qb[NT][HD / 16][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        const uint2 v = lds_u2(base + S::kQ + (nt * 8 + g) * S::kQRow + (16 * k + 4 * t4) * 2);
        qb[nt][k][0] = v.x;
        qb[nt][k][1] = v.y;
      }

    Kv8Acc<NT, HD> acc;
    acc.clear();
    float* score_rows = p.scores ? p.scores + ((int64_t)b * p.nq + kvh * group) * p.c.cap : nullptr;
    int u = idx - seg0;
    const int coded_end = min(u_end, coded);
#pragma unroll 1
    for (; u < coded_end; u += kWarps) {
      constexpr int MT = kKvBlock / 16;
      const int t0 = u * kKvBlock;
      const bool more = u + kWarps < u_end;
      const float ks2 = ks * p.scale2, vs1 = vs;
      if (u + kWarps < coded_end) {
        ks = k_scale[u + kWarps];
        vs = v_scale[u + kWarps];
      }
      await_keys();
      float s[MT][NT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int k = 0; k < HD / 16; k += 2) {
          uint32_t r[4];
          ldsm4(r, (k_slot + mt * 16 * HD) + (lane_off ^ (k << 4)));
#pragma unroll
          for (int kk = 0; kk < 2; ++kk) {
            const uint32_t a0 = codes2<0x4140>(r[2 * kk]), a1 = codes2<0x4140>(r[2 * kk + 1]);
            const uint32_t a2 = codes2<0x4342>(r[2 * kk]), a3 = codes2<0x4342>(r[2 * kk + 1]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              if (k + kk == 0)
                mma_16816_0(s[mt][nt], a0, a1, a2, a3, qb[nt][0][0], qb[nt][0][1]);
              else
                mma_16816(s[mt][nt], a0, a1, a2, a3, qb[nt][k + kk][0], qb[nt][k + kk][1]);
          }
        }
      }
      __syncwarp();  // the keys are in registers: the next block's may come
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      if (more) load(0, u + kWarps);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[mt][nt][e] *= ks2;
      if (t0 + kKvBlock > min_stop) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (t0 + 16 * mt + g + 8 * (e >> 1) >= stop[nt][e & 1]) s[mt][nt][e] = -INFINITY;
      }
      if (score_rows) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int h = nt * 8 + 2 * t4 + j;
            float* row = score_rows + (int64_t)h * p.c.cap + t0 + g;
            if (h < rows) {
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                row[16 * mt] = s[mt][nt][j];
                row[16 * mt + 8] = s[mt][nt][2 + j];
              }
            }
          }
      }
      float gain[NT][2];
      uint32_t pb[MT][NT][2];
      kv8_softmax<NT, HD, MT>(acc, s, gain, pb);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) gain[nt][j] *= vs1;
      await_values(more);
#pragma unroll
      for (int i = 0; i < HD / 16; i += 2) {
        float x[2][NT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          uint32_t r[4];
          ldsm4_t(r, (v_slot + mt * 16 * HD) + (lane_off ^ (i << 4)));
#pragma unroll
          for (int ii = 0; ii < 2; ++ii) {
            const uint32_t a0 = codes2<0x4240>(r[2 * ii]), a1 = codes2<0x4341>(r[2 * ii]);
            const uint32_t a2 = codes2<0x4240>(r[2 * ii + 1]), a3 = codes2<0x4341>(r[2 * ii + 1]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              if (mt == 0)
                mma_16816_0(x[ii][nt], a0, a1, a2, a3, pb[mt][nt][0], pb[mt][nt][1]);
              else
                mma_16816(x[ii][nt], a0, a1, a2, a3, pb[mt][nt][0], pb[mt][nt][1]);
          }
        }
#pragma unroll
        for (int ii = 0; ii < 2; ++ii)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              acc.o[i + ii][nt][e] = fmaf(x[ii][nt][e], gain[nt][e & 1], acc.o[i + ii][nt][e]);
      }
      __syncwarp();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      if (more) load(1, u + kWarps);
    }
#pragma unroll 1
    for (; u < u_end; u += kWarps) {
      // 16 FP16 rows of the tail, the token's own from where it was put
      const int t0 = coded * kKvBlock + (u - coded) * kDecTailUnit;
      const bool more = u + kWarps < u_end;
      auto row = [&](int w, int r) {
        return p.extra && t0 + r == len - 1 ? base + S::kNew + w * HD * 2 : (w ? v_slot : k_slot) + r * HD * 2;
      };
      await_keys();
      float s[1][NT][4];
      {
        const uint32_t k0 = row(0, g) + 8 * t4, k1 = row(0, g + 8) + 8 * t4;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const uint2 x = lds_u2(k0 + 32 * k), y = lds_u2(k1 + 32 * k);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            if (k == 0)
              mma_16816_0(s[0][nt], x.x, y.x, x.y, y.y, qb[nt][k][0], qb[nt][k][1]);
            else
              mma_16816(s[0][nt], x.x, y.x, x.y, y.y, qb[nt][k][0], qb[nt][k][1]);
        }
      }
      __syncwarp();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      if (more) load(0, u + kWarps);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = t0 + g + 8 * (e >> 1), h = nt * 8 + 2 * t4 + (e & 1);
          s[0][nt][e] = t < stop[nt][e & 1] ? s[0][nt][e] * p.scale2 : -INFINITY;
          if (score_rows && h < rows && t < len) score_rows[(int64_t)h * p.c.cap + t] = s[0][nt][e];
        }
      float gain[NT][2];
      uint32_t pb[1][NT][2];
      kv8_softmax<NT, HD, 1>(acc, s, gain, pb);
      await_values(more);
      if (MANY && kv8_drop_odd_rows<HD>(v_slot, min(len - t0, kDecTailUnit))) {  // one query attends all rows
        __syncwarp();
        if (lane == 0) s_odd = segment;
      }
      const uint32_t v0 = row(1, 2 * t4) + 4 * g, v1 = row(1, 2 * t4 + 1) + 4 * g;
      const uint32_t v2 = row(1, 2 * t4 + 8) + 4 * g, v3 = row(1, 2 * t4 + 9) + 4 * g;
      const int left = len - t0 - 2 * t4;  // rows past the end count as zero: their contents may be anything
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        const uint32_t x0 = left > 0 ? lds_u32(v0 + 32 * i) : 0u, x1 = left > 1 ? lds_u32(v1 + 32 * i) : 0u;
        const uint32_t x2 = left > 8 ? lds_u32(v2 + 32 * i) : 0u, x3 = left > 9 ? lds_u32(v3 + 32 * i) : 0u;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float x[4];
          mma_16816_0(x, lo_pair(x0, x1), hi_pair(x0, x1), lo_pair(x2, x3), hi_pair(x2, x3), pb[0][nt][0], pb[0][nt][1]);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc.o[i][nt][e] = fmaf(x[e], gain[nt][e & 1], acc.o[i][nt][e]);
        }
      }
      __syncwarp();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      if (more) load(1, u + kWarps);
    }
    // the next segment's first units and rows travel while this one's results are added up
    turn = (turn + u_end - (at - seg0)) % kWarps;  // the warps go on in turn
    idx = end + (warp >= turn ? warp - turn : warp - turn + kWarps);
    entered = end < z;
    if (entered) {
      seg.next(work);
      enter(end);
      const int s = seg.seg;
      have = seg.b * work.per_seq + s;
      fetch(seg.b, p.tiles == 1 ? s : s / p.tiles, p.tiles == 1 ? 0 : s % p.tiles * NT * 8, row, token);
    }

    // the warps' results: every warp to the common reference, then added up by
    // all threads in warp order, two dimensions of a row each
    float2* ml = reinterpret_cast<float2*>(pp_smem + S::kMl);  // [warp][row]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float l = acc.l[nt][j];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        if (g == 0) ml[warp * NT * 8 + nt * 8 + 2 * t4 + j] = make_float2(acc.m[nt][j], l);
      }
    __syncthreads();
    float fa[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, ml[w * NT * 8 + nt * 8 + 2 * t4 + j].x);
        fa[nt][j] = acc.m[nt][j] == -INFINITY ? 1.f : ex2(acc.m[nt][j] - m);  // such a warp's sums are 0 (or NaN)
      }
    const bool whole = at == seg0 && z >= real1;
    float* rec = p.part + ((int64_t)blockIdx.x * 2 + (a >= seg0 ? 0 : 1)) * kPartFloats;
    constexpr int kI = HD / 16 / S::kRounds;  // dimension tiles of a round
#pragma unroll
    for (int round = 0; round < S::kRounds; ++round) {
      float* area = reinterpret_cast<float*>(pp_smem + S::kMerge);
      if (round) __syncthreads();
#pragma unroll
      for (int i = 0; i < kI; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            area[(warp * S::kPart + (i * NT + nt) * 4 + e) * 32 + lane] = acc.o[round * kI + i][nt][e] * fa[nt][e & 1];
      __syncthreads();
      for (int e = tid; e < kI * NT * 2 * 32; e += kThreads) {
        const int el = e & 31, j = (e >> 5) & 1, in = e >> 6, nt = in % NT, i = in / NT;
        const int r = nt * 8 + 2 * (el & 3) + j, d = 16 * (round * kI + i) + 2 * (el >> 2);
        if (r >= rows) continue;
        float m = -INFINITY, l = 0.f, x = 0.f, y = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, ml[w * NT * 8 + r].x);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float2 v = ml[w * NT * 8 + r];
          l = fmaf(v.y, v.x == -INFINITY ? 1.f : ex2(v.x - m), l);
          const float* f = area + (w * S::kPart + in * 4 + j) * 32 + el;
          x += f[0];
          y += f[64];
        }
        if (whole) {
          const float inv = l == 0.f ? 0.f : 1.f / l;
          *out_at(b, kvh, row0, r, d) = __floats2half2_rn(x * inv, y * inv);
          if (p.scores && d == 0) p.lse[b * p.nq + kvh * group + r] = m + log2f(l);
        } else {
          *reinterpret_cast<float2*>(rec + r * HD + d) = make_float2(x, y);
          if (d == 0) *reinterpret_cast<float2*>(rec + NT * 8 * HD + 2 * r) = make_float2(m, l);
        }
      }
    }

    if (MANY && s_odd == segment) {  // the same for all threads
      __syncthreads();               // the results are written
      kv8_add_odd<NT, HD>(p, b, kvh, row0, rows, cnt, len, (max(at - seg0, coded) - coded) * kDecTailUnit,
                          (u_end - coded) * kDecTailUnit, whole ? nullptr : rec);
    }
    if (!whole) {
      if (tid == 0) {
        const int first = aligned ? segment * each : seg0 / per;
        s_part[pending] = Kv8Part{b, kvh, row0, rows, seg0, first,
                                  aligned ? pieces(U) : (real1 - 1) / per - first + 1, 0};
      }
      ++pending;  // at most the share's first and last segment
    }
    at = end;
  }

  // segments that other CTAs have a part of: the last of them to arrive adds up
  // the parts in order
  if (pending) {
    __threadfence();
    __syncthreads();
    if (tid < pending) {
      Kv8Part& s = s_part[tid];
      s.last = atomicAdd(p.cnt + s.first, 1) == s.contrib - 1;  // at most one segment goes on past a CTA's share
      if (s.last) {
        p.cnt[s.first] = 0;
        __threadfence();
      }
    }
    __syncthreads();
    for (int i = 0; i < pending; ++i) {
      if (!s_part[i].last) continue;
      const int b = s_part[i].b, kvh = s_part[i].kvh, row0 = s_part[i].row0, rows = s_part[i].rows;
      const int seg0 = s_part[i].seg0, first = s_part[i].first, contrib = s_part[i].contrib;
      auto from = [&](int k) {
        return p.part +
               ((int64_t)(first + k) * 2 + (aligned || (first + k) * (int64_t)per >= seg0 ? 0 : 1)) * kPartFloats;
      };
      for (int e = tid; e < rows * (HD / 4); e += kThreads) {
        const int r = e / (HD / 4), d = e % (HD / 4) * 4;
        float m = -INFINITY, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k0 = 0; k0 < contrib; k0 += 8) {  // eight partials' loads at a time
          float2 v[8];
          float4 x[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            v[k] = make_float2(-INFINITY, 0.f);
            x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k0 + k < contrib) {
              v[k] = __ldcg(reinterpret_cast<const float2*>(from(k0 + k) + NT * 8 * HD + 2 * r));
              x[k] = __ldcg(reinterpret_cast<const float4*>(from(k0 + k) + r * HD + d));
            }
          }
          float to = m;
#pragma unroll
          for (int k = 0; k < 8; ++k) to = fmaxf(to, v[k].x);
          const float f0 = m == -INFINITY ? 1.f : ex2(m - to);
          l *= f0;
          o = make_float4(o.x * f0, o.y * f0, o.z * f0, o.w * f0);
          m = to;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float f = v[k].x == -INFINITY ? 1.f : ex2(v[k].x - m);
            l = fmaf(v[k].y, f, l);
            o.x = fmaf(x[k].x, f, o.x);
            o.y = fmaf(x[k].y, f, o.y);
            o.z = fmaf(x[k].z, f, o.z);
            o.w = fmaf(x[k].w, f, o.w);
          }
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        *out_at(b, kvh, row0, r, d) = __floats2half2_rn(o.x * inv, o.y * inv);
        *out_at(b, kvh, row0, r, d + 2) = __floats2half2_rn(o.z * inv, o.w * inv);
        if (p.scores && d == 0) p.lse[b * p.nq + kvh * group + r] = m + log2f(l);
      }
    }
  }
  if (p.extra) kv8_store_token<HD, kWarps>(p, s_len, red);
}

// weights[b][g][t] += sum of the group's exp2(score - lse).
struct Kv8WeightsParams {
  const float* scores;
  const float* lse;
  float* weights;
  const int* lens;
  const Kv8Rope rope;
  int extra, nq, nkv, cap;
};

__global__ void __launch_bounds__(256) kv8_weights_kernel(const Kv8WeightsParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.z, kvh = blockIdx.y, group = p.nq / p.nkv;
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= p.cap) return;
  // everything is read side by side, whatever the length turns out to be
  const float* s = p.scores + ((int64_t)b * p.nq + kvh * group) * p.cap + t;
  const float* l = p.lse + b * p.nq + kvh * group;
  float* out = p.weights + ((int64_t)b * p.nkv + kvh) * p.cap + t;
  constexpr int kChunk = 8;
  float x[kChunk], y[kChunk];
  auto load = [&](int h0) {
#pragma unroll
    for (int h = 0; h < kChunk; ++h) {
      const bool in = h0 + h < group;
      x[h] = in ? s[(int64_t)(h0 + h) * p.cap] : -INFINITY;
      y[h] = in ? l[h0 + h] : 0.f;
    }
  };
  load(0);
  const float before = *out;
  const int held = p.lens[b], rot = p.rope.cos ? p.rope.pos[b] : 0;
  if (held > p.cap - p.extra || t >= held + p.extra || (p.rope.cos && (rot < 0 || rot >= p.rope.len))) return;
  float w = 0.f;
  for (int h0 = 0;;) {
#pragma unroll
    for (int h = 0; h < kChunk; ++h) w += ex2(x[h] - y[h]);
    if ((h0 += kChunk) >= group) break;
    load(h0);
  }
  *out = before + w;
}

}  // namespace pp
