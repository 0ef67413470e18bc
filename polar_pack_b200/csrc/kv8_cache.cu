// Writing, reading back and evicting from the 8-bit KV cache (kv8.cuh).
#include <cooperative_groups.h>

#include "kv8.cuh"

namespace pp {

namespace cg = cooperative_groups;

int kv8_cache(const char* who, const pp_kv8_cache* c, Kv8Cache* out) {
  if (!c) {
    set_error("%s: no cache", who);
    return PP_ERR_INVALID;
  }
  if (c->batch < 1 || c->batch > PP_KV8_MAX_BATCH || c->kv_heads < 1 || c->kv_heads > 1024 || c->capacity < kKvBlock ||
      c->capacity % kKvBlock || c->capacity > INT32_MAX / 2 || (c->head_dim != 64 && c->head_dim != 128)) {
    set_error("%s: a cache has 1..%d sequences, 1..1024 heads, a capacity that is a multiple of %d, head_dim 64 or 128",
              who, PP_KV8_MAX_BATCH, kKvBlock);
    return PP_ERR_INVALID;
  }
  for (int w = 0; w < 2; ++w) {
    if (!c->codes[w] || !c->scales[w] || !c->tail[w] || !aligned(c->codes[w], 16) || !aligned(c->scales[w], 4) ||
        !aligned(c->tail[w], 16)) {
      set_error("%s: cache arrays are NULL or not 16-byte aligned", who);
      return PP_ERR_INVALID;
    }
    out->codes[w] = reinterpret_cast<uint8_t*>(c->codes[w]);
    out->scales[w] = c->scales[w];
    out->tail[w] = reinterpret_cast<__half*>(c->tail[w]);
  }
  out->batch = (int)c->batch;
  out->nkv = (int)c->kv_heads;
  out->cap = (int)c->capacity;
  out->hd = (int)c->head_dim;
  return PP_OK;
}

int kv8_rope(const char* who, const void* cos_t, const void* sin_t, const int* pos, int64_t len, Kv8Rope* out) {
  *out = Kv8Rope{};
  if (!cos_t && !sin_t && !pos) return PP_OK;
  if (!cos_t || !sin_t || !pos || len < 1 || len > INT32_MAX || !aligned(cos_t, 16) || !aligned(sin_t, 16)) {
    set_error("%s: a rotation needs both tables (16-byte aligned, at least one row) and positions", who);
    return PP_ERR_INVALID;
  }
  out->cos = reinterpret_cast<const __half*>(cos_t);
  out->sin = reinterpret_cast<const __half*>(sin_t);
  out->pos = pos;
  out->len = (int)len;
  return PP_OK;
}

namespace {

constexpr int kThreads = 256;

struct AppendParams {
  Kv8Cache c;
  const __half* x[2];  // keys, values: row (b, i, head) at b * ldb + i * ldt + head * ldh
  int64_t ldb[2], ldt[2], ldh[2];
  const int* pos;
  const int* counts;   // NULL: n new tokens for every sequence
  int n;
  Kv8Rope rope;        // of the keys
  int* status;
};

// CTA (j, head, sequence and side) makes block pos / 64 + j of one head's keys
// or values, each thread sixteen dimensions of HD / 64 rows in registers: one pass,
// rows read once, codes and tail written once.  The CTA of the first block
// also writes the tail rows of the last one: it alone reads the tail's old
// rows, so nothing overwrites them before they are read.  Bound: the rows'
// chain in a CTA, which has one block and nothing of another one under way.
// 16 ragged prompts, 17473 tokens of 4 heads of 128, 54 MB: 16 us, 3.4 TB/s.
template <int HD>
__global__ void __launch_bounds__(kThreads, 5) kv8_append_kernel(const AppendParams p) {
  constexpr int kRow = HD / 16, kItems = kKvBlock * kRow / kThreads;  // threads of a row, rows of a thread
  __shared__ float red[kThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.y, b = blockIdx.z >> 1, w = blockIdx.z & 1;
  const int pos = p.pos[b];
  int cnt = p.counts ? min(max(p.counts[b], 0), p.n) : p.n;
  if (pos < 0 || cnt == 0) return;
  bool ok = pos <= p.c.cap - cnt;
  Kv8Rope rope = w == 0 ? p.rope : Kv8Rope{};
  const int rot = rope.cos ? rope.pos[b] : 0;
  if (rope.cos && (rot < 0 || rot > rope.len - cnt)) ok = false;
  if (!ok) {
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, 5);
    return;
  }
  const int len = pos + cnt, last = kv8_last_block(len);
  const int block = pos / kKvBlock + blockIdx.x;
  if (block > last) return;
  const Kv8Head<HD> to(p.c, w, b, h);
  const int r0 = threadIdx.x / kRow, d0 = threadIdx.x % kRow * 16;
  const __half* x = pick(p.x, w) + b * pick(p.ldb, w) + h * pick(p.ldh, w);
  const int64_t ldt = pick(p.ldt, w);
  auto row = [&](int t, uint4 (&v)[2]) {  // 16 dimensions of a new token
    const __half* y = x + (int64_t)(t - pos) * ldt;
    v[0] = kv8_load8(y, d0, HD, rope, rot + t - pos);
    v[1] = kv8_load8(y, d0 + 8, HD, rope, rot + t - pos);
  };
  uint4 v[kItems][2];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int r = r0 + i * (kThreads / kRow), t = block * kKvBlock + r;
    v[i][0] = v[i][1] = make_uint4(0, 0, 0, 0);
    if (t < pos) {
      const uint4* y = reinterpret_cast<const uint4*>(to.tail + r * HD + d0);
      v[i][0] = y[0];
      v[i][1] = y[1];
    } else if (t < len) {
      row(t, v[i]);
    }
  }
  if ((block + 1) * kKvBlock <= len) {
    const Kv8Scale q = kv8_block_scale<2 * kItems, kThreads>(reinterpret_cast<const uint4(&)[2 * kItems]>(v), red);
    uint8_t* out = to.codes + ((int64_t)(block * kKvBlock + r0) * HD + d0);
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const uint2 lo = kv8_codes8(v[i][0], q), hi = kv8_codes8(v[i][1], q);
      *reinterpret_cast<uint4*>(out + i * (kThreads / kRow) * HD) = make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
    if (threadIdx.x == 0) to.scales[block] = q.scale;
  }
  if (blockIdx.x != 0) return;
  __syncthreads();  // the tail's old rows have been read
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int r = r0 + i * (kThreads / kRow), t = last * kKvBlock + r;
    if (t < pos || t >= len) continue;
    if (last != block) row(t, v[i]);
    uint4* y = reinterpret_cast<uint4*>(to.tail + r * HD + d0);
    y[0] = v[i][0];
    y[1] = v[i][1];
  }
}

struct RestoreParams {
  Kv8Cache c;
  const int* lens;
  const int* start;  // NULL: 0
  int count;
  __half* out[2];    // [batch][count][kv head][hd]
  int* status;
};

// CTA (64 positions, head, sequence and side): a thread restores kVecs vectors
// of eight dimensions, all read before the first is written.  Bound: the
// outputs' bytes.  8 x 4000 rows of 4 heads of 128, 25398 of them held, 92 MB: 18 us, 5.0 TB/s.
template <int HD>
__global__ void __launch_bounds__(kThreads) kv8_restore_kernel(const RestoreParams p) {
  constexpr int kVecs = kKvBlock * HD / 8 / kThreads;
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.y, b = blockIdx.z >> 1, w = blockIdx.z & 1;
  const int len = p.lens[b], first = p.start ? p.start[b] : 0;
  const bool ok = len <= p.c.cap;
  if (!ok && blockIdx.x == 0 && h == 0 && threadIdx.x == 0 && p.status) atomicExch(p.status, 5);
  const Kv8Head<HD> head(p.c, w, b, h);
  const int last = kv8_last_block(len), i0 = blockIdx.x * kKvBlock, n = min(kKvBlock, p.count - i0);
  uint4 v[kVecs];
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    const int e = k * kThreads + threadIdx.x, i = e / (HD / 8);
    const int64_t t = (int64_t)first + i0 + i;
    v[k] = make_uint4(0, 0, 0, 0);
    if (ok && i < n && t >= 0 && t < len) v[k] = head.read8((int)t, last, e % (HD / 8) * 8);
  }
  const int ld = p.c.nkv * HD;
  __half* out = pick(p.out, w) + ((int64_t)b * p.count + i0) * ld + h * HD;
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    const int e = k * kThreads + threadIdx.x, i = e / (HD / 8);
    if (i < n) *reinterpret_cast<uint4*>(out + i * ld + e % (HD / 8) * 8) = v[k];
  }
}

// ------------------------------------------------------------- eviction --
struct EvictParams {
  Kv8Cache c, to;
  const int* lens;
  const float* weights;   // [batch][kv head][c.cap]
  float* to_weights;      // [batch][kv head][to.cap]
  int* new_lens;          // [batch]
  int* kept;              // [batch][kv head][keep]
  int keep, sinks, recent;
  int* status;
};

// Weights as whole numbers of the same order; NaN above every number.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xfffffffeu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelThreads = 1024;
constexpr int kSelRounds = 16;         // of kSelThreads keys, whose kept ones are counted together
constexpr int kSelCached = 48 * 1024;  // keys that fit shared memory
constexpr int kSelParts = 8;           // CTAs of a cluster, at most

__host__ __device__ __forceinline__ int select_part(int len, int parts) {  // positions of a CTA
  return (int)(((int64_t)len + parts - 1) / parts + 31) & ~31;
}

// A cluster (head, sequence) finds the keep-th largest key by four passes over
// the keys' bytes: each CTA counts its stretch of positions (equal bytes of a
// warp at once), all add the cluster's counts up.  Then each writes its kept
// positions in order: those above the key, and as many equal to it, lowest
// first, as there is room.  The keys stay in shared memory where they fit
// (`cached` of a CTA's).  Bound: the chain of passes, four exchanges of a
// cluster among them.  8 sequences up to 16384, 70973 positions in all, of 4 heads:
// 21 us over clusters of eight; 38 us with one CTA to a head.
__global__ void __launch_bounds__(kSelThreads, 2) kv8_select_kernel(const EvictParams p, int cached) {
  __shared__ int hist[4][256];  // this CTA's counts, a pass each
  __shared__ int total[256];
  __shared__ int above_of[kSelRounds * 32 + 1], equal_of[kSelRounds * 32 + 1];  // kept before a round's warp
  __shared__ int digit[4], s_left, s_above;
  pdl_launch_dependents();
  pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  uint32_t* keys = reinterpret_cast<uint32_t*>(pp_smem);
  const int h = blockIdx.x / parts, b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int len = p.lens[b];
  const bool ok = len <= p.c.cap;
  if (!ok && tid == 0 && p.status) atomicExch(p.status, 5);
  len = ok ? max(len, 0) : 0;
  const int m = min(len, p.keep);
  if (blockIdx.x == 0 && tid == 0) p.new_lens[b] = m;
  const float* wt = p.weights + p.c.head(b, h) * p.c.cap;
  float* to_wt = p.to_weights + p.to.head(b, h) * p.to.cap;
  int* kept = p.kept + p.c.head(b, h) * p.keep;
  const int me = part * kSelThreads + tid, all = parts * kSelThreads;
  for (int t = m + me; t < p.keep; t += all) kept[t] = -1;
  for (int t = m + me; t < p.to.cap; t += all) to_wt[t] = 0.f;
  if (m == len) {
    for (int t = me; t < len; t += all) {
      kept[t] = t;
      to_wt[t] = wt[t];
    }
    return;
  }
  const int size = select_part(len, parts), lo = min(len, part * size), hi = min(len, lo + size);
  auto make_key = [&](int t) { return t < p.sinks || t >= len - p.recent ? 0xffffffffu : weight_key(wt[t]); };
  for (int i = tid; i < 4 * 256; i += kSelThreads) hist[i >> 8][i & 255] = 0;
  if (tid == 0) s_above = 0;
#pragma unroll 4
  for (int t = lo + tid; t < min(hi, lo + cached); t += kSelThreads) keys[t - lo] = make_key(t);
  auto key = [&](int t) { return t - lo < cached ? keys[t - lo] : make_key(t); };  // a thread reads its own
  auto meet = [&] {
    if (parts > 1) cluster.sync();
    else __syncthreads();
  };
  __syncthreads();
  uint32_t cut = 0;
  int left = m;  // kept positions among the keys that agree with `cut` so far
#pragma unroll 1
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
#pragma unroll 2
    for (int t0 = lo; t0 < hi; t0 += kSelThreads) {
      const int t = t0 + tid;
      const uint32_t k = t < hi ? key(t) : 0;
      const bool in = t < hi && (pass == 0 || (k >> (shift + 8)) == (cut >> (shift + 8)));
      const uint32_t d = in ? (k >> shift) & 255 : 256;
      if (__any_sync(0xffffffffu, in)) {
        const uint32_t same = __match_any_sync(0xffffffffu, d);
        if (in && lane == __ffs(same) - 1) atomicAdd(&hist[pass][d], __popc(same));
      }
    }
    meet();
    if (parts > 1) {
      if (tid < 256) {
        int n = 0;
        for (int c = 0; c < parts; ++c) n += *cluster.map_shared_rank(&hist[pass][tid], c);
        total[tid] = n;
      }
      __syncthreads();
    }
    if (warp == 0) {
      const int* count = parts > 1 ? total : hist[pass];
      // the digit at which the count from the top reaches `left`: lane l has digits 255 - 8 l and down
      int n[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += n[i] = count[255 - 8 * lane - i];
      int upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      int above = upto - sum;
      if (above < left && upto >= left) {
        int d = 255 - 8 * lane;
#pragma unroll
        for (int i = 0; i < 7; ++i)
          if (d == 255 - 8 * lane - i && above + n[i] < left) {
            above += n[i];
            --d;
          }
        digit[pass] = d;
        s_left = left - above;
      }
    }
    __syncthreads();
    cut |= (uint32_t)digit[pass] << shift;
    left = s_left;
  }
  int base_gt = 0, base_eq = 0;  // keys above / equal to the cut before these rounds
  if (parts > 1) {
    const int d = tid & 255, n = d > digit[tid >> 8] ? hist[tid >> 8][d] : 0;
    const int sum = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0 && sum) atomicAdd(&s_above, sum);
    cluster.sync();
    for (int c = 0; c < part; ++c) {
      base_gt += *cluster.map_shared_rank(&s_above, c);
      base_eq += *cluster.map_shared_rank(&hist[3][cut & 255], c);
    }
    cluster.sync();  // the others' counts have been read
  }
  for (int r0 = lo; r0 < hi; r0 += kSelRounds * kSelThreads) {
    const int rounds = min(kSelRounds, (hi - r0 + kSelThreads - 1) / kSelThreads);
    for (int i = 0; i < rounds; ++i) {
      const int t = r0 + i * kSelThreads + tid;
      const uint32_t k = t < hi ? key(t) : 0;
      const uint32_t bg = __ballot_sync(0xffffffffu, t < hi && k > cut), be = __ballot_sync(0xffffffffu, t < hi && k == cut);
      if (lane == 0) {
        above_of[i * 32 + warp] = __popc(bg);
        equal_of[i * 32 + warp] = __popc(be);
      }
    }
    __syncthreads();
    if (warp < 2) {  // exclusive sums over the rounds' warps
      int* a = warp == 0 ? above_of : equal_of;
      int sum = 0;
      for (int i = 0; i < rounds; ++i) {
        const int n = a[i * 32 + lane];
        int x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        a[i * 32 + lane] = sum + x - n;
        sum += __shfl_sync(0xffffffffu, x, 31);
      }
      if (lane == 0) a[kSelRounds * 32] = sum;
    }
    __syncthreads();
    for (int i = 0; i < rounds; ++i) {
      const int t = r0 + i * kSelThreads + tid;
      const uint32_t k = t < hi ? key(t) : 0;
      const bool gt = t < hi && k > cut, eq = t < hi && k == cut;
      const uint32_t bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq), below = (1u << lane) - 1;
      const int g = base_gt + above_of[i * 32 + warp] + __popc(bg & below);
      const int q = base_eq + equal_of[i * 32 + warp] + __popc(be & below);
      if (gt || (eq && q < left)) {
        const int at = g + min(q, left);
        kept[at] = t;
        to_wt[at] = wt[t];
      }
    }
    base_gt += above_of[kSelRounds * 32];
    base_eq += equal_of[kSelRounds * 32];
    __syncthreads();
  }
}

// CTA (block, head, sequence and side) gathers the kept rows of one block of
// the new cache and quantises them as an append would; a block that is one
// whole coded block of the old cache is copied, codes and scale, so that
// repeated evictions do not requantise what does not move apart.
// Bound: the instructions from codes to values and back.  8 x 4000 at most, 25398 kept tokens, of 4 heads of 128,
// 52 MB: 21 us.
template <int HD>
__global__ void __launch_bounds__(kThreads, 6) kv8_gather_kernel(const EvictParams p) {
  constexpr int kRow = HD / 16, kItems = kKvBlock * kRow / kThreads;  // threads of a row, rows of a thread
  __shared__ float red[kThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int block = blockIdx.x, h = blockIdx.y, b = blockIdx.z >> 1, w = blockIdx.z & 1;
  // the positions (-1 past the new length) are read beside the lengths, not after them
  const int* kept = p.kept + p.c.head(b, h) * p.keep + block * kKvBlock;
  const int room = p.keep - block * kKvBlock, r0 = threadIdx.x / kRow, d0 = threadIdx.x % kRow * 16;
  int src[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int r = r0 + i * (kThreads / kRow);
    src[i] = r < room ? kept[r] : -1;
  }
  const int f = kept[0], g = room >= kKvBlock ? kept[kKvBlock - 1] : -1;
  const int len = p.lens[b], m = p.new_lens[b], old_last = kv8_last_block(len);
  if (f < 0) return;
  const bool full = g >= 0;
  const Kv8Head<HD> from(p.c, w, b, h), to(p.to, w, b, h);
  uint4 v[2 * kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    v[2 * i] = v[2 * i + 1] = make_uint4(0, 0, 0, 0);
    if (src[i] < 0) continue;
    const int at = src[i] / kKvBlock;
    if (at == old_last) {
      const uint4* x = reinterpret_cast<const uint4*>(from.tail + src[i] % kKvBlock * HD + d0);
      v[2 * i] = x[0];
      v[2 * i + 1] = x[1];
    } else {
      const uint4 c = *reinterpret_cast<const uint4*>(from.codes + ((int64_t)src[i] * HD + d0));
      const float scale = from.scales[at];
      v[2 * i] = kv8_values8(make_uint2(c.x, c.y), scale);
      v[2 * i + 1] = kv8_values8(make_uint2(c.z, c.w), scale);
    }
  }
  if (block == kv8_last_block(m)) {
#pragma unroll
    for (int i = 0; i < kItems; ++i)
      if (src[i] >= 0) {
        uint4* x = reinterpret_cast<uint4*>(to.tail + (r0 + i * (kThreads / kRow)) * HD + d0);
        x[0] = v[2 * i];
        x[1] = v[2 * i + 1];
      }
  }
  if (!full) return;
  uint8_t* out = to.codes + ((int64_t)(block * kKvBlock + r0) * HD + d0);
  constexpr int kStep = kThreads / kRow * HD;
  if (f % kKvBlock == 0 && g - f == kKvBlock - 1 && f / kKvBlock != old_last) {
    const uint8_t* same = from.codes + ((int64_t)(f + r0) * HD + d0);
#pragma unroll
    for (int i = 0; i < kItems; ++i)
      *reinterpret_cast<uint4*>(out + i * kStep) = *reinterpret_cast<const uint4*>(same + i * kStep);
    if (threadIdx.x == 0) to.scales[block] = from.scales[f / kKvBlock];
    return;
  }
  const Kv8Scale q = kv8_block_scale<2 * kItems, kThreads>(v, red);
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const uint2 lo = kv8_codes8(v[2 * i], q), hi = kv8_codes8(v[2 * i + 1], q);
    *reinterpret_cast<uint4*>(out + i * kStep) = make_uint4(lo.x, lo.y, hi.x, hi.y);
  }
  if (threadIdx.x == 0) to.scales[block] = q.scale;
}

// Whether an array that an eviction writes shares bytes with another of its
// arrays: the kernels read the old cache while they write the new one.
bool evict_overlaps(const EvictParams& p, const int* lens, const float* weights, const float* to_weights,
                    const int* new_lens, const int* kept, int64_t keep) {
  struct Range {
    uintptr_t at;
    uint64_t bytes;
  } r[17];
  int n = 0;
  auto add = [&](const void* at, int64_t bytes) { r[n++] = Range{reinterpret_cast<uintptr_t>(at), (uint64_t)bytes}; };
  const int64_t heads = (int64_t)p.c.batch * p.c.nkv;
  auto cache = [&](const Kv8Cache& c) {
    for (int w = 0; w < 2; ++w) {
      add(c.codes[w], heads * c.cap * c.hd);
      add(c.scales[w], heads * (c.cap / kKvBlock) * (int64_t)sizeof(float));
      add(c.tail[w], heads * kKvBlock * c.hd * (int64_t)sizeof(__half));
    }
  };
  cache(p.to);
  add(to_weights, heads * p.to.cap * (int64_t)sizeof(float));
  add(new_lens, p.c.batch * (int64_t)sizeof(int));
  add(kept, heads * keep * (int64_t)sizeof(int));
  const int written = n;
  cache(p.c);
  add(weights, heads * p.c.cap * (int64_t)sizeof(float));
  add(lens, p.c.batch * (int64_t)sizeof(int));
  for (int i = 0; i < written; ++i)
    for (int j = i + 1; j < n; ++j)
      if (r[i].at < r[j].at + r[j].bytes && r[j].at < r[i].at + r[i].bytes) return true;
  return false;
}

bool g_select_attr[64];
int g_select_limit[64];

}  // namespace
}  // namespace pp

extern "C" {

int pp_kv8_append(const pp_kv8_cache* cache, const void* k, const int64_t k_strides[3], const void* v,
                  const int64_t v_strides[3], int64_t n, const int* pos, const int* counts, const void* cos_t,
                  const void* sin_t, const int* rope_pos, int64_t rope_len, int* status, void* stream) {
  pp::AppendParams p{};
  if (int rc = pp::kv8_cache("pp_kv8_append", cache, &p.c)) return rc;
  if (int rc = pp::kv8_rope("pp_kv8_append", cos_t, sin_t, rope_pos, rope_len, &p.rope)) return rc;
  if (n == 0) return PP_OK;
  if (!k || !v || !k_strides || !v_strides || !pos || n < 0 || n > INT32_MAX / 2) {
    pp::set_error("pp_kv8_append: keys, values, strides and positions are required");
    return PP_ERR_INVALID;
  }
  const void* x[2] = {k, v};
  const int64_t* st[2] = {k_strides, v_strides};
  for (int w = 0; w < 2; ++w) {
    if (!pp::aligned(x[w], 16) || st[w][0] % 8 || st[w][1] % 8 || st[w][2] % 8) {
      pp::set_error("pp_kv8_append: rows must be 16-byte aligned");
      return PP_ERR_INVALID;
    }
    p.x[w] = reinterpret_cast<const __half*>(x[w]);
    p.ldb[w] = st[w][0];
    p.ldt[w] = st[w][1];
    p.ldh[w] = st[w][2];
  }
  p.pos = pos;
  p.counts = counts;
  p.n = (int)n;
  p.status = status;
  const dim3 grid((unsigned)((n + pp::kKvBlock - 2) / pp::kKvBlock + 1), (unsigned)p.c.nkv, (unsigned)p.c.batch * 2);
  return pp::launch_kernel("kv8_append_kernel", pp::launch_overlap(),
                           p.c.hd == 128 ? pp::kv8_append_kernel<128> : pp::kv8_append_kernel<64>, grid,
                           dim3(pp::kThreads), 0, reinterpret_cast<cudaStream_t>(stream), p);
}

int pp_kv8_restore(const pp_kv8_cache* cache, const int* lens, const int* start, int64_t count, void* k, void* v,
                   int* status, void* stream) {
  pp::RestoreParams p{};
  if (int rc = pp::kv8_cache("pp_kv8_restore", cache, &p.c)) return rc;
  if (count == 0) return PP_OK;
  if (!lens || !k || !v || count < 0 || count > INT32_MAX / 2 || !pp::aligned(k, 16) || !pp::aligned(v, 16)) {
    pp::set_error("pp_kv8_restore: lengths and 16-byte aligned outputs are required");
    return PP_ERR_INVALID;
  }
  p.lens = lens;
  p.start = start;
  p.count = (int)count;
  p.out[0] = reinterpret_cast<__half*>(k);
  p.out[1] = reinterpret_cast<__half*>(v);
  p.status = status;
  return pp::launch_kernel("kv8_restore_kernel", pp::launch_overlap(),
                           p.c.hd == 128 ? pp::kv8_restore_kernel<128> : pp::kv8_restore_kernel<64>,
                           dim3((unsigned)pp::cdiv(count, pp::kKvBlock), (unsigned)p.c.nkv, (unsigned)p.c.batch * 2),
                           dim3(pp::kThreads), 0,
                           reinterpret_cast<cudaStream_t>(stream), p);
}

int pp_kv8_evict(const pp_kv8_cache* cache, const pp_kv8_cache* into, const int* lens, const float* weights,
                 float* into_weights, int* new_lens, int* kept, int64_t keep, int64_t sinks, int64_t recent, int* status,
                 void* stream) {
  pp::EvictParams p{};
  if (int rc = pp::kv8_cache("pp_kv8_evict", cache, &p.c)) return rc;
  if (int rc = pp::kv8_cache("pp_kv8_evict", into, &p.to)) return rc;
  if (p.c.batch != p.to.batch || p.c.nkv != p.to.nkv || p.c.hd != p.to.hd) {
    pp::set_error("pp_kv8_evict: the caches differ in sequences, heads or head_dim");
    return PP_ERR_INVALID;
  }
  if (!lens || !weights || !into_weights || !new_lens || !kept || keep < 1 || keep > p.to.cap || sinks < 0 ||
      recent < 0 || sinks > keep || recent > keep - sinks) {
    pp::set_error("pp_kv8_evict: lengths, weights and outputs are required, keep between 1 and the new capacity, "
                  "sinks + recent at most keep");
    return PP_ERR_INVALID;
  }
  if (pp::evict_overlaps(p, lens, weights, into_weights, new_lens, kept, keep)) {
    pp::set_error("pp_kv8_evict: the arrays that are written must not overlap the old cache, its weights and lengths "
                  "or one another");
    return PP_ERR_INVALID;
  }
  p.lens = lens;
  p.weights = weights;
  p.to_weights = into_weights;
  p.new_lens = new_lens;
  p.kept = kept;
  p.keep = (int)keep;
  p.sinks = (int)sinks;
  p.recent = (int)recent;
  p.status = status;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int lim = 0;
  if (int rc = pp::ensure_smem_attr(pp::kv8_select_kernel, pp::g_select_attr, pp::g_select_limit, &lim)) return rc;
  // long caches: as many CTAs to a head as find SMs of their own, each with two rounds of positions at least
  const int sms = pp::device_sm_count(pp::current_device());
  int parts = 1;
  while (parts < pp::kSelParts && (int64_t)p.c.nkv * p.c.batch * parts <= sms && p.c.cap >= parts * 4 * pp::kSelThreads)
    parts *= 2;
  int cached = pp::select_part(p.c.cap, parts);
  if (cached > pp::kSelCached) cached = pp::kSelCached;
  if (cached * 4 > lim) cached = lim / 4;
  if (int rc = pp::launch_clusters("kv8_select_kernel", pp::launch_overlap(), parts > 1 ? (unsigned)parts : 0u, pp::kv8_select_kernel,
                                   dim3((unsigned)(p.c.nkv * parts), (unsigned)p.c.batch), dim3(pp::kSelThreads),
                                   (size_t)cached * 4, s, p, cached))
    return rc;
  // started early whatever the overlap setting: it waits for the selection itself
  return pp::launch_kernel("kv8_gather_kernel", true,
                           p.c.hd == 128 ? pp::kv8_gather_kernel<128> : pp::kv8_gather_kernel<64>,
                           dim3((unsigned)pp::cdiv(keep, pp::kKvBlock), (unsigned)p.c.nkv, (unsigned)p.c.batch * 2),
                           dim3(pp::kThreads), 0, s, p);
}

}  // extern "C"
