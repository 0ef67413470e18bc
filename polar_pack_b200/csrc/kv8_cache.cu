// Writing, reading back and evicting from the 8-bit KV cache (kv8.cuh).
#include "kv8.cuh"

namespace pp {

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
// or values, each thread HD / 32 vectors of eight in registers: one pass,
// rows read once, codes and tail written once.  The CTA of the first block
// also writes the tail rows of the last one: it alone reads the tail's old
// rows, so nothing overwrites them before they are read.
template <int HD>
__global__ void __launch_bounds__(kThreads) kv8_append_kernel(const AppendParams p) {
  constexpr int kVecs = kKvBlock * HD / 8 / kThreads;
  __shared__ float red[kThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.y, b = blockIdx.z >> 1, w = blockIdx.z & 1;
  const int pos = p.pos[b];
  int cnt = p.counts ? min(max(p.counts[b], 0), p.n) : p.n;
  if (pos < 0 || cnt == 0) return;
  bool ok = pos <= p.c.cap - cnt;
  Kv8Rope rope = w == 0 ? p.rope : Kv8Rope{};
  const int r0 = rope.cos ? rope.pos[b] : 0;
  if (rope.cos && (r0 < 0 || r0 > rope.len - cnt)) ok = false;
  if (!ok) {
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, 5);
    return;
  }
  const int len = pos + cnt, last = kv8_last_block(len);
  const int block = pos / kKvBlock + blockIdx.x;
  if (block > last) return;
  const __half* x = pick(p.x, w) + b * pick(p.ldb, w) + h * pick(p.ldh, w);
  const int64_t ldt = pick(p.ldt, w);
  auto row8 = [&](int t, int d0) { return kv8_load8(x + (int64_t)(t - pos) * ldt, d0, HD, rope, r0 + t - pos); };
  uint4 v[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int e = i * kThreads + threadIdx.x, r = e / (HD / 8), d0 = e % (HD / 8) * 8;
    const int t = block * kKvBlock + r;
    v[i] = make_uint4(0, 0, 0, 0);
    if (t < pos)
      v[i] = *reinterpret_cast<const uint4*>(p.c.tail_row(w, b, h, r) + d0);
    else if (t < len)
      v[i] = row8(t, d0);
  }
  if ((block + 1) * kKvBlock <= len) {
    const Kv8Scale q = kv8_block_scale<kVecs, kThreads>(v, red);
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int e = i * kThreads + threadIdx.x, r = e / (HD / 8), d0 = e % (HD / 8) * 8;
      *reinterpret_cast<uint2*>(p.c.code_row(w, b, h, block * kKvBlock + r) + d0) = kv8_codes8(v[i], q);
    }
    if (threadIdx.x == 0) *p.c.scale(w, b, h, block) = q.scale;
  }
  if (blockIdx.x != 0) return;
  __syncthreads();  // the tail's old rows have been read
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int e = i * kThreads + threadIdx.x, r = e / (HD / 8), d0 = e % (HD / 8) * 8;
    const int t = last * kKvBlock + r;
    if (t >= pos && t < len)
      *reinterpret_cast<uint4*>(p.c.tail_row(w, b, h, r) + d0) = last == block ? v[i] : row8(t, d0);
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
// of eight dimensions, all read before the first is written.
template <int HD>
__global__ void __launch_bounds__(kThreads) kv8_restore_kernel(const RestoreParams p) {
  constexpr int kVecs = kKvBlock * HD / 8 / kThreads;
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.y, b = blockIdx.z >> 1, w = blockIdx.z & 1;
  const int len = p.lens[b], first = p.start ? p.start[b] : 0;
  const bool ok = len <= p.c.cap;
  if (!ok && blockIdx.x == 0 && h == 0 && threadIdx.x == 0 && p.status) atomicExch(p.status, 5);
  uint4 v[kVecs];
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    const int e = k * kThreads + threadIdx.x, i = blockIdx.x * kKvBlock + e / (HD / 8);
    const int64_t t = (int64_t)first + i;
    v[k] = make_uint4(0, 0, 0, 0);
    if (ok && i < p.count && t >= 0 && t < len) v[k] = kv8_read8(p.c, w, b, h, (int)t, len, e % (HD / 8) * 8);
  }
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    const int e = k * kThreads + threadIdx.x, i = blockIdx.x * kKvBlock + e / (HD / 8);
    if (i < p.count)
      *reinterpret_cast<uint4*>(pick(p.out, w) + (((int64_t)b * p.count + i) * p.c.nkv + h) * HD + e % (HD / 8) * 8) = v[k];
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
constexpr int kSelRounds = 32;            // of kSelThreads keys, whose kept ones are counted together
constexpr int kSelCached = 48 * 1024;     // keys that fit shared memory

// CTA (head, sequence) finds the keep-th largest key by four passes over the
// keys' bytes (a histogram each, equal bytes of a warp counted at once), then
// writes the kept positions in order: those above it, and as many equal to it,
// lowest first, as there is room.  The keys stay in shared memory where they
// fit (`cached` keys).
__global__ void __launch_bounds__(kSelThreads) kv8_select_kernel(const EvictParams p, int cached) {
  __shared__ int hist[256];
  __shared__ int above_of[kSelRounds * 32 + 1], equal_of[kSelRounds * 32 + 1];  // kept before a round's warp
  __shared__ int s_digit, s_left;
  pdl_launch_dependents();
  pdl_wait();
  uint32_t* keys = reinterpret_cast<uint32_t*>(pp_smem);
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int len = p.lens[b];
  const bool ok = len <= p.c.cap;
  if (!ok && tid == 0 && p.status) atomicExch(p.status, 5);
  len = ok ? max(len, 0) : 0;
  const int m = min(len, p.keep);
  if (h == 0 && tid == 0) p.new_lens[b] = m;
  const float* wt = p.weights + p.c.head(b, h) * p.c.cap;
  float* to_wt = p.to_weights + p.to.head(b, h) * p.to.cap;
  int* kept = p.kept + p.c.head(b, h) * p.keep;
  auto make_key = [&](int t) { return t < p.sinks || t >= len - p.recent ? 0xffffffffu : weight_key(wt[t]); };
  for (int t = m + tid; t < p.keep; t += kSelThreads) kept[t] = -1;
  for (int t = m + tid; t < p.to.cap; t += kSelThreads) to_wt[t] = 0.f;
  if (m == len) {
    for (int t = tid; t < len; t += kSelThreads) {
      kept[t] = t;
      to_wt[t] = wt[t];
    }
    return;
  }
#pragma unroll 4
  for (int t = tid; t < min(len, cached); t += kSelThreads) keys[t] = make_key(t);
  auto key = [&](int t) { return t < cached ? keys[t] : make_key(t); };  // a thread reads its own
  uint32_t cut = 0;
  int left = m;  // kept positions among the keys that agree with `cut` so far
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
#pragma unroll 2
    for (int t0 = 0; t0 < len; t0 += kSelThreads) {
      const int t = t0 + tid;
      const uint32_t k = t < len ? key(t) : 0;
      const bool in = t < len && (shift == 24 || (k >> (shift + 8)) == (cut >> (shift + 8)));
      const uint32_t d = in ? (k >> shift) & 255 : 256;
      if (__any_sync(0xffffffffu, in)) {
        const uint32_t same = __match_any_sync(0xffffffffu, d);
        if (in && lane == __ffs(same) - 1) atomicAdd(&hist[d], __popc(same));
      }
    }
    __syncthreads();
    if (warp == 0) {
      // the digit at which the count from the top reaches `left`: lane l has digits 255 - 8 l and down
      int n[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += n[i] = hist[255 - 8 * lane - i];
      int upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      int above = upto - sum;
      if (above < left && upto >= left) {
        int i = 0;
        while (above + n[i] < left) above += n[i++];
        s_digit = 255 - 8 * lane - i;
        s_left = left - above;
      }
    }
    __syncthreads();
    cut |= (uint32_t)s_digit << shift;
    left = s_left;
  }
  int base_gt = 0, base_eq = 0;  // kept above / equal before these rounds
  for (int r0 = 0; r0 < len; r0 += kSelRounds * kSelThreads) {
    const int rounds = min(kSelRounds, (len - r0 + kSelThreads - 1) / kSelThreads);
    for (int i = 0; i < rounds; ++i) {
      const int t = r0 + i * kSelThreads + tid;
      const uint32_t k = t < len ? key(t) : 0;
      const uint32_t bg = __ballot_sync(0xffffffffu, t < len && k > cut), be = __ballot_sync(0xffffffffu, t < len && k == cut);
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
      const uint32_t k = t < len ? key(t) : 0;
      const bool gt = t < len && k > cut, eq = t < len && k == cut;
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
template <int HD>
__global__ void __launch_bounds__(kThreads) kv8_gather_kernel(const EvictParams p) {
  constexpr int kVecs = kKvBlock * HD / 8 / kThreads;
  __shared__ float red[kThreads / 32];
  __shared__ int src[kKvBlock];
  pdl_launch_dependents();
  pdl_wait();
  const int block = blockIdx.x, h = blockIdx.y, b = blockIdx.z >> 1, w = blockIdx.z & 1;
  const int len = p.lens[b], m = p.new_lens[b];
  if (block * kKvBlock >= m) return;
  const bool full = (block + 1) * kKvBlock <= m, last = block == kv8_last_block(m);
  const int* kept = p.kept + p.c.head(b, h) * p.keep + block * kKvBlock;
  if (threadIdx.x < kKvBlock) src[threadIdx.x] = block * kKvBlock + threadIdx.x < m ? kept[threadIdx.x] : -1;
  __syncthreads();
  const int f = src[0];
  const bool whole = full && f % kKvBlock == 0 && src[kKvBlock - 1] - f == kKvBlock - 1 &&
                     f / kKvBlock != kv8_last_block(len);
  uint4 v[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int e = i * kThreads + threadIdx.x, r = e / (HD / 8), d0 = e % (HD / 8) * 8;
    v[i] = src[r] >= 0 ? kv8_read8(p.c, w, b, h, src[r], len, d0) : make_uint4(0, 0, 0, 0);
  }
  if (last) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int e = i * kThreads + threadIdx.x, r = e / (HD / 8), d0 = e % (HD / 8) * 8;
      if (src[r] >= 0) *reinterpret_cast<uint4*>(p.to.tail_row(w, b, h, r) + d0) = v[i];
    }
  }
  if (!full) return;
  const Kv8Scale q = kv8_block_scale<kVecs, kThreads>(v, red);
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int e = i * kThreads + threadIdx.x, r = e / (HD / 8), d0 = e % (HD / 8) * 8;
    const uint2 c = whole ? *reinterpret_cast<const uint2*>(p.c.code_row(w, b, h, f + r) + d0) : kv8_codes8(v[i], q);
    *reinterpret_cast<uint2*>(p.to.code_row(w, b, h, block * kKvBlock + r) + d0) = c;
  }
  if (threadIdx.x == 0) *p.to.scale(w, b, h, block) = whole ? *p.c.scale(w, b, h, f / kKvBlock) : q.scale;
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
  for (int w = 0; w < 2; ++w)
    for (int u = 0; u < 2; ++u)
      if (p.c.codes[w] == p.to.codes[u] || p.c.tail[w] == p.to.tail[u] || p.c.scales[w] == p.to.scales[u] ||
          weights == into_weights) {
        pp::set_error("pp_kv8_evict: the new cache must not be the old one");
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
  int cached = p.c.cap < pp::kSelCached ? p.c.cap : pp::kSelCached;
  if (cached * 4 > lim) cached = lim / 4;
  if (int rc = pp::launch_kernel("kv8_select_kernel", pp::launch_overlap(), pp::kv8_select_kernel,
                                 dim3((unsigned)p.c.nkv, (unsigned)p.c.batch), dim3(pp::kSelThreads), (size_t)cached * 4,
                                 s, p, cached))
    return rc;
  // started early whatever the overlap setting: it waits for the selection itself
  return pp::launch_kernel("kv8_gather_kernel", true,
                           p.c.hd == 128 ? pp::kv8_gather_kernel<128> : pp::kv8_gather_kernel<64>,
                           dim3((unsigned)pp::cdiv(keep, pp::kKvBlock), (unsigned)p.c.nkv, (unsigned)p.c.batch * 2),
                           dim3(pp::kThreads), 0, s, p);
}

}  // extern "C"
