// Log probabilities of given tokens, entropy and the likeliest alternatives
// of rows of logits.
//   m = max x,  Z = sum e^(x - m)
//   logprob = x_token - m - ln Z,  entropy = ln Z - sum e^(x - m) (x - m) / Z
// (both terms of the entropy are positive: no cancellation).
//
// Bound: the logits' bytes for many rows; next to them one exponential per
// logit, 16 a clock and SM, which at the measured memory rate are three
// quarters of the time for 2-byte logits.  Measured: 2048 rows of 151936 FP16
// with the 5 likeliest, 622 MB: 134 us back to back, 4.6 TB/s, about 9 instructions a logit
// (109 us without alternatives); 301 rows of 32003 FP32: 12 us, 3.2 TB/s; 4 rows
// with the 20 likeliest: 14 to 16 us, 6.7 without: the rest are the bound, the second
// look and the ranking at a row's end.  One pass: a thread keeps its own (maximum, Z, W = sum e^(x - m)
// (x - m)), moved to a new maximum when a batch of its logits exceeds it, and
// the place of its largest logit.  For the
// alternatives logits are whole numbers (value, then lower index), all
// different; the top-th largest of the best of 64 groups of threads is a bound
// that at least `top` logits reach, and only the logits of threads whose best
// reaches it, a few of the CTA, are gone through again (by all threads) for a
// list in shared memory, of which the `top` largest are ranked.  A row that lists
// more than there is room for goes through its logits batch by batch, with a
// bound that follows the list.  Few rows are spread over clusters of up to
// eight CTAs, whose results meet in the first one's shared memory.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include <type_traits>

#include "pp_common.cuh"
#include "pp_host.h"

namespace pp {
namespace {

namespace cg = cooperative_groups;

// Threads of a CTA, vectors of a thread in a batch, CTAs of an SM.  Many rows:
// small CTAs, whose row ends (a chain of barriers) hide behind the others'
// streams (2048 x 151936 FP16 with top 5: 134 us; 11% more with the other shape).
// Few rows: large ones, a row's chain being the time (4 rows, top 20: 15.2 us;
// 17.4 with the other shape).
struct ManyRows {
  static constexpr int kThreads = 256, kBatch = 4, kResident = 3;
};
struct FewRows {
  static constexpr int kThreads = 512, kBatch = 2, kResident = 2;
};
// Short rows: two warps, ten rows to an SM.  Which rows count as short
// (short_rows) by measurement of both (us, 256 threads against 64):
//   FP16 1001 x 31968, top 0 / 5 / 32    443 -> 96, 694 -> 211, 5113 -> 235
//   FP16 4001 x 7998                     75 -> 31, 142 -> 61, 159 -> 130
//   FP16 16001 x 1999                    26 -> 18, 45 -> 34, 61 -> 126
//   FP16 1001 x 200                      8.2 -> 5.3, 11 -> 8.2, 77 -> 10.5
//   FP16 4001 x 200                      6.1 -> 5.4, 9.5 -> 8.8, 10 -> 21
struct ShortRows {
  static constexpr int kThreads = 64, kBatch = 4, kResident = 10;
};
constexpr bool short_rows(int64_t rows, int64_t row_bytes, int top, int sms) {
  return row_bytes <= (rows < 8 * sms ? 4 << 10 : top > 8 ? 8 << 10 : 32 << 10);
}
constexpr int kMaxThreads = 512;
constexpr int kMaxCluster = 8;
constexpr int kGroups = 64;      // of threads, whose best logits give the first bound
constexpr int kList = 2048;      // keys that the list holds
constexpr float kLog2e = 1.44269504088896341f;

struct ScoreParams {
  const void* x;
  int64_t ldx;
  int64_t rows;
  int vocab;
  const int* tokens;
  int top;
  float* logprob;
  float* entropy;
  int* top_ids;
  float* top_logprobs;
  int* status;
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }

using Key = unsigned long long;

// Larger values first, NaN before all (-0 counts as 0).
__device__ __forceinline__ uint32_t order(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return x != x ? 0xffffffffu : u & 0x80000000u ? ~u : u | 0x80000000u;
}
// Equal values by the lower index: one whole number each.
__device__ __forceinline__ Key rank_key(float x, int i) {
  return (Key)order(x) << 32 | (uint32_t)(0x7fffffff - i);
}

__device__ __forceinline__ float ex2a(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Sums over e^(x - m), kept beside the maximum they refer to.
struct Stat {
  float m, z, w;  // maximum, sum e^(x-m), sum e^(x-m) (x-m)
  __device__ __forceinline__ void rescale(float to) {
    if (to == m) return;
    const float d = m - to, f = m == -INFINITY ? 0.f : ex2a(d * kLog2e);
    w = f == 0.f ? 0.f : f * fmaf(d, z, w);
    z = f == 0.f ? 0.f : f * z;
    m = to;
  }
  __device__ __forceinline__ void merge(Stat o) {
    const float t = fmaxf(m, o.m);
    rescale(t);
    o.rescale(t);
    z += o.z;
    w += o.w;
  }
};

// A thread's sums over pairs of logits, beside the maximum m.
struct PairSums {
  float m = -INFINITY;
  uint64_t z = 0, w = 0;
  __device__ __forceinline__ void raise(float top) {
    if (!(top > m)) return;
    const float d = m - top, f = m == -INFINITY ? 0.f : ex2a(d * kLog2e);
    float z0, z1, w0, w1;
    f32_split(z, z0, z1);
    f32_split(w, w0, w1);
    w = f == 0.f ? 0 : f32_pair(f * fmaf(d, z0, w0), f * fmaf(d, z1, w1));
    z = f == 0.f ? 0 : f32_pair(f * z0, f * z1);
    m = top;
  }
  // after raise: finite a, b
  __device__ __forceinline__ void add(float a, float b, uint64_t minus_m) {
    const uint64_t d = f32_add2(f32_pair(a, b), minus_m);
    float e0, e1;
    f32_split(f32_mul2(d, f32_pair(kLog2e, kLog2e)), e0, e1);
    const uint64_t e = f32_pair(ex2a(e0), ex2a(e1));
    z = f32_add2(z, e);
    w = f32_fma2(e, d, w);
  }
  // any a; -inf counts nothing
  __device__ __forceinline__ void add(float a) {
    const float d = fmaxf(a - m, -200.f);
    const uint64_t e = f32_pair(ex2a(d * kLog2e), 0.f);
    z = f32_add2(z, e);
    w = f32_fma2(e, f32_pair(d, 0.f), w);
  }
  __device__ __forceinline__ Stat stat() const {
    float z0, z1, w0, w1;
    f32_split(z, z0, z1);
    f32_split(w, w0, w1);
    return Stat{m, z0 + z1, w0 + w1};
  }
};

struct Shared {
  Key list[kList];
  Key kept[32];
  Key best[kGroups];
  uint16_t who[kMaxThreads];  // threads whose best logit reaches the bound
  int interested;
  Stat stat[kMaxThreads / 32];
  Key bound;  // keys below it are not among the row's top
  int count;       // listed keys
  int held;        // of them from earlier batches of a second passage
};

// A CTA's part of a row, read by the first CTA of the cluster.
struct Result {
  Stat stat;
  int nan, kept;
  Key keys[32];
};

// The `top` largest of the first n listed keys, in order, to s.kept.  Every
// thread of the CTA comes here.
template <int kThreads>
__device__ void rank_list(Shared& s, int n, int top) {
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const Key k = s.list[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) rank += s.list[j] > k;
    if (rank < top) s.kept[rank] = k;
  }
  __syncthreads();
}

// The list becomes its `top` largest, in order.
template <int kThreads>
__device__ void prune(Shared& s, int top) {
  const int n = min(s.count, kList);
  rank_list<kThreads>(s, n, top);
  const int left = min(n, top);
  if ((int)threadIdx.x < left) s.list[threadIdx.x] = s.kept[threadIdx.x];
  if (threadIdx.x == 0) {
    s.count = s.held = left;
    if (left == top) s.bound = s.kept[top - 1];
  }
  __syncthreads();
}

// 16 bytes of logits.
template <typename T>
struct Vec {
  static constexpr int kN = 16 / sizeof(T);
  uint4 v;
  __device__ __forceinline__ uint32_t word(int i) const { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(word(i));
    else if constexpr (std::is_same<T, __half>::value)
      return __half2float(__ushort_as_half((unsigned short)(word(i >> 1) >> (16 * (i & 1)))));
    else return __uint_as_float(i & 1 ? word(i >> 1) & 0xffff0000u : word(i >> 1) << 16);
  }
  // The larger of each pair of logits; NaN if one is.
  __device__ __forceinline__ Vec max(const Vec& o) const {
    Vec r{v};
    uint32_t* a = &r.v.x;
    const uint32_t* b = &o.v.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        float y = __uint_as_float(a[i]);
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(y) : "f"(__uint_as_float(b[i])));
        a[i] = __float_as_uint(y);
      } else if constexpr (std::is_same<T, __half>::value) {
        asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(a[i]) : "r"(b[i]));
      } else {
        asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(a[i]) : "r"(b[i]));
      }
    }
    return r;
  }
  // The largest; NaN if there is one.
  __device__ __forceinline__ float top() const {
    if constexpr (sizeof(T) == 4) {
      float m = get(0);
#pragma unroll
      for (int i = 1; i < 4; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(get(i)));
      return m;
    } else {
      uint32_t m = v.x;
#pragma unroll
      for (int i = 1; i < 4; ++i) {
        if constexpr (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(m) : "r"(word(i)));
        else asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(word(i)));
      }
      const Vec<T> r{make_uint4(m, 0, 0, 0)};
      float a = r.get(0);
      asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(r.get(1)));
      return a;
    }
  }
  static __device__ __forceinline__ Vec nothing() {  // -inf
    constexpr uint32_t w = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
    return Vec{make_uint4(w, w, w, w)};
  }
  // A finite number (a word of one or two) that takes the place of logits
  // below it, -inf above all: its e^(x - m) is 0, and x - m is finite.
  // -2^20 for positive m, else the type's lowest; `low` says that m is too
  // near to that.  NaN becomes it too.
  static __device__ __forceinline__ uint32_t lowest(float m) {
    if constexpr (sizeof(T) == 4) return m > 0.f ? 0xc9800000u : 0xff7fffffu;
    else if constexpr (std::is_same<T, __half>::value) return 0xfbfffbffu;
    else return m > 0.f ? 0xc980c980u : 0xff7fff7fu;
  }
  static __device__ __forceinline__ bool low(float m) {
    constexpr float lo = std::is_same<T, __half>::value ? -65504.f : sizeof(T) == 4 ? -3.40282347e38f : -3.38953139e38f;
    return !(m - lo > 200.f);
  }
  __device__ __forceinline__ Vec at_least(uint32_t lo) const {
    Vec r{v};
    uint32_t* a = &r.v.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) a[i] = __float_as_uint(fmaxf(__uint_as_float(a[i]), __uint_as_float(lo)));
      else if constexpr (std::is_same<T, __half>::value) asm("max.f16x2 %0, %0, %1;" : "+r"(a[i]) : "r"(lo));
      else asm("max.bf16x2 %0, %0, %1;" : "+r"(a[i]) : "r"(lo));
    }
    return r;
  }
};

template <typename T, bool TOP, typename S>
__global__ void __launch_bounds__(S::kThreads, S::kResident) token_logprobs_kernel(const ScoreParams p) {
  __shared__ Shared s;
  __shared__ Result mine;
  constexpr int N = Vec<T>::kN, kThreads = S::kThreads, kWarps = kThreads / 32, kBatch = S::kBatch;
  pdl_launch_dependents();
  pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int64_t r = blockIdx.x / parts; r < p.rows; r += gridDim.x / parts) {
    const T* x = reinterpret_cast<const T*>(p.x) + r * p.ldx;
    // 16-byte vectors between the ends of the row that are not aligned
    const int head = min(p.vocab, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T)));
    const int vecs = (p.vocab - head) / N;
    const int v0 = (int)((int64_t)vecs * part / parts), v1 = (int)((int64_t)vecs * (part + 1) / parts);
    const uint4* xv = reinterpret_cast<const uint4*>(x + head);
    if (TOP) {
      if (tid == 0) {
        s.bound = 0;
        s.count = s.held = s.interested = 0;
      }
      __syncthreads();
    }
    Stat st{-INFINITY, 0.f, 0.f};
    bool nan = false;
    auto raise = [&](float top) {  // top: a largest logit
      nan |= top != top;
      if (top > st.m) st.rescale(top);
    };
    auto add = [&](float v) {  // a logit, after raise; -inf counts nothing
      const float d = fmaxf(v - st.m, -200.f), e = ex2a(d * kLog2e);
      st.z += e;
      st.w = fmaf(e, d, st.w);
    };
    auto enlist = [&](float v, int i) {
      const Key k = rank_key(v, i);
      if (k >= s.bound) {
        const int at = atomicAdd(&s.count, 1);
        if (at < kList) s.list[at] = k;
      }
    };
    // this thread's logits of a batch whose vectors may hold listed ones
    auto scan = [&](int b0, auto&& use) {
#pragma unroll 1
      for (int k = 0; k < kBatch; ++k) {
        const int i = b0 + k * kThreads + tid;
        if (i >= v1) break;
        const Vec<T> v{xv[i]};
        if (order(v.top()) < (uint32_t)(s.bound >> 32)) continue;
#pragma unroll 1
        for (int e = 0; e < N; ++e) use(v.get(e), head + i * N + e);
      }
    };
    // the bound to the top-th largest of the groups' best keys, if that is higher
    auto bound_from = [&](Key best) {
#pragma unroll
      for (int o = 1; o < kThreads / kGroups; o <<= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
      if (tid % (kThreads / kGroups) == 0) s.best[tid / (kThreads / kGroups)] = best;
      __syncthreads();
      if (tid < kGroups) {
        const Key me = s.best[tid];
        int above = 0, equal = 0;
#pragma unroll 8
        for (int j = 0; j < kGroups; ++j) {
          above += s.best[j] > me;
          equal += s.best[j] == me;
        }
        if (above < p.top && above + equal >= p.top && me > s.bound) s.bound = me;  // all who write write the same
      }
      __syncthreads();
    };
    float best = -INFINITY;  // this thread's largest logit (a NaN counts as that), and its batch's first vector
    int best_at = -1;
    PairSums sums;
    // a batch is loaded while the one before it is summed
    auto load = [&](Vec<T> (&q)[kBatch], int b0) {
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int i = b0 + k * kThreads + tid;
        q[k] = Vec<T>::nothing();
        if (i < v1) q[k].v = ld_stream(xv + i);  // coherent: the logits may be new
      }
    };
    auto take = [&](const Vec<T> (&q)[kBatch], int b0) {
      Vec<T> m = q[0];
#pragma unroll
      for (int k = 1; k < kBatch; ++k) m = m.max(q[k]);
      const float top = m.top();
      nan |= top != top;
      sums.raise(top);
      if (Vec<T>::low(sums.m)) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
#pragma unroll 1
          for (int e = 0; e < N; ++e) sums.add(q[k].get(e));
        }
      } else {
        const uint64_t minus_m = f32_pair(-sums.m, -sums.m);
        const uint32_t lo = Vec<T>::lowest(sums.m);
        PairSums part{sums.m};  // a batch's sum first: equal terms would round the same way in a long one
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const Vec<T> v = q[k].at_least(lo);
#pragma unroll
          for (int e = 0; e < N; e += 2) part.add(v.get(e), v.get(e + 1), minus_m);
        }
        sums.z = f32_add2(sums.z, part.z);
        sums.w = f32_add2(sums.w, part.w);
      }
      if (TOP && b0 + tid < v1 && (best_at < 0 || !(top <= best)) && best == best) {
        best = top;
        best_at = b0 + tid;
      }
    };
    constexpr int kStep = kThreads * kBatch;
    Vec<T> q0[kBatch], q1[kBatch];
    load(q0, v0);
#pragma unroll 1
    for (int b0 = v0; b0 < v1; b0 += 2 * kStep) {
      load(q1, b0 + kStep);
      take(q0, b0);
      if (b0 + kStep >= v1) break;
      load(q0, b0 + 2 * kStep);
      take(q1, b0 + kStep);
    }
    st = sums.stat();
    if constexpr (TOP) {
      // the bound from the last logits of the best batches: none is above its batch's best
      bound_from(best_at < 0 ? 0 : rank_key(best, head + (best_at + kStep - kThreads) * N + N - 1));
      if (best_at >= 0 && rank_key(best, head + best_at * N) >= s.bound) s.who[atomicAdd(&s.interested, 1)] = tid;
      __syncthreads();
      const int per = (v1 - v0 + kThreads - 1) / kThreads, items = s.interested * per;
#pragma unroll 1
      for (int it0 = tid; it0 < items; it0 += kThreads * kBatch) {
        Vec<T> q[kBatch];
        int at[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int it = it0 + k * kThreads;
          at[k] = it < items ? v0 + it % per * kThreads + s.who[it / per] : v1;
          if (at[k] < v1) q[k].v = xv[at[k]];
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
          if (at[k] < v1 && order(q[k].top()) >= (uint32_t)(s.bound >> 32)) {
#pragma unroll 1
            for (int e = 0; e < N; ++e) enlist(q[k].get(e), head + at[k] * N + e);
          }
      }
    }
    if constexpr (TOP) {
      __syncthreads();
      const bool over = s.count > kList - 2 * N;  // the row's ends, not listed yet, need room too
      __syncthreads();  // everyone has read the count before it changes
      if (over) {
        // A second passage, batch by batch: the list holds the best so far, its
        // last the bound.  Equal logits of later batches rank below it.
        if (tid == 0) s.count = s.held = 0;
        __syncthreads();
        for (int b0 = v0; b0 < v1; b0 += kThreads * kBatch) {
          Key best = 0;
          scan(b0, [&](float v, int i) { best = max(best, rank_key(v, i)); });
          if (__syncthreads_count(best >= s.bound) == 0) continue;
          bound_from(best);
          for (;;) {
            if (best >= s.bound) scan(b0, enlist);
            __syncthreads();
            if (s.count <= kList) break;
            // too many: the top-th of those listed is a higher bound; list again
            rank_list<kThreads>(s, kList, p.top);
            if (tid == 0) {
              s.bound = max(s.bound, s.kept[p.top - 1]);
              s.count = s.held;
            }
            __syncthreads();
          }
          prune<kThreads>(s, p.top);
        }
      }
    }
    // the logits at the row's ends, by the last CTA's first threads: fewer than two vectors
    if (part == parts - 1) {
      const int tail = p.vocab - head - vecs * N;
      if (tid < head + tail) {
        const int i = tid < head ? tid : head + vecs * N + (tid - head);
        const float v = to_f(x[i]);
        raise(v);
        if (st.m > -INFINITY) add(v);
        if (TOP) enlist(v, i);
      }
    }
    // the CTA's sums
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Stat t{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.z, o),
                   __shfl_xor_sync(0xffffffffu, st.w, o)};
      st.merge(t);
    }
    if (lane == 0) s.stat[warp] = st;
    nan = __syncthreads_or(nan);
    if (TOP) prune<kThreads>(s, p.top);
    if (warp == 0) {
      st = lane < kWarps ? s.stat[lane] : Stat{-INFINITY, 0.f, 0.f};
#pragma unroll
      for (int o = kWarps / 2; o > 0; o >>= 1) {
        const Stat t{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.z, o),
                     __shfl_xor_sync(0xffffffffu, st.w, o)};
        st.merge(t);
      }
      st = Stat{__shfl_sync(0xffffffffu, st.m, 0), __shfl_sync(0xffffffffu, st.z, 0),
                __shfl_sync(0xffffffffu, st.w, 0)};
    }
    if (parts > 1) {
      if (tid == 0) {
        mine.stat = st;
        mine.nan = nan;
        mine.kept = TOP ? s.count : 0;
      }
      if (TOP && tid < s.count) mine.keys[tid] = s.list[tid];
      cluster.sync();
      if (part == 0) {
        if (warp == 0) {  // a lane reads one part's sums; merged in order
          const Result* o = cluster.map_shared_rank(&mine, lane < parts ? lane : 0);
          const Stat part_st = o->stat;
          nan = __any_sync(0xffffffffu, o->nan != 0);
          st = Stat{-INFINITY, 0.f, 0.f};
          for (int k = 0; k < parts; ++k)
            st.merge(Stat{__shfl_sync(0xffffffffu, part_st.m, k), __shfl_sync(0xffffffffu, part_st.z, k),
                          __shfl_sync(0xffffffffu, part_st.w, k)});
        }
        if (TOP) {
          // 32 places for each part's keys; empty ones rank last
          if (tid < parts * 32) {
            const Result* o = cluster.map_shared_rank(&mine, tid / 32);
            s.list[tid] = tid % 32 < o->kept ? o->keys[tid % 32] : 0;
          }
          __syncthreads();
          if (tid == 0) s.count = parts * 32;
          __syncthreads();
          prune<kThreads>(s, p.top);
        }
      }
      cluster.sync();  // the others' results have been read
    }
    if (part == 0 && warp == 0) {
      const float log_z = logf(st.z);
      float lse = st.m + log_z, ent = log_z - st.w / st.z;
      if (st.m == -INFINITY) lse = ent = 0.f;  // nothing but -inf
      if (nan || st.m == INFINITY) {
        lse = nan ? NAN : INFINITY;
        ent = NAN;
      }
      if (lane == 0) {
        const int t = p.tokens[r];
        p.logprob[r] = t < 0 ? 0.f : t < p.vocab ? to_f(x[t]) - lse : NAN;
        p.entropy[r] = ent;
        if (t >= p.vocab && p.status) atomicExch(p.status, 4);
      }
      if (TOP && lane < min(p.top, s.count)) {  // as many as `top` are always listed, unless the logits change meanwhile
        const int i = 0x7fffffff - (int)(uint32_t)s.list[lane];
        p.top_ids[r * p.top + lane] = i;
        p.top_logprobs[r * p.top + lane] = to_f(x[i]) - lse;
      }
    }
    __syncthreads();  // the warps' sums and the list have been read
  }
}

template <typename T, typename S>
int launch(const ScoreParams& p, int parts, cudaStream_t stream) {
  const int64_t rows = p.rows < (1 << 24) ? p.rows : (1 << 24);
  return launch_clusters("token_logprobs_kernel", launch_overlap(), (unsigned)parts,
                         p.top ? token_logprobs_kernel<T, true, S> : token_logprobs_kernel<T, false, S>,
                         dim3((unsigned)(rows * parts)), dim3(S::kThreads), 0, stream, p);
}

template <typename T>
int launch(const ScoreParams& p, cudaStream_t stream) {
  const int sms = device_sm_count(current_device());
  if (sms < 1) {
    set_error("pp_token_logprobs: no current CUDA device");
    return PP_ERR_CUDA;
  }
  // few rows: as many CTAs to each (a power of two) as keep them all on SMs of
  // their own, and 16 KB of logits to every CTA at least
  int parts = 1;
  while (parts < kMaxCluster && p.rows * parts * 2 <= sms &&
         (int64_t)p.vocab * (int)sizeof(T) >= (int64_t)parts * 2 * (16 << 10))
    parts *= 2;
  if (short_rows(p.rows, (int64_t)p.vocab * (int)sizeof(T), p.top, sms)) return launch<T, ShortRows>(p, 1, stream);
  return p.rows * kMaxCluster <= sms ? launch<T, FewRows>(p, parts, stream) : launch<T, ManyRows>(p, parts, stream);
}

}  // namespace
}  // namespace pp

extern "C" int pp_token_logprobs(const void* logits, int dtype, int64_t ldx, int64_t rows, int64_t vocab,
                                 const int* tokens, int64_t top, float* logprob, float* entropy, int* top_ids,
                                 float* top_logprobs, int* status, void* stream) {
  if (rows == 0) return PP_OK;
  const int size = dtype == PP_F32 ? 4 : 2;
  if (!logits || !tokens || !logprob || !entropy || rows < 0 || rows > INT32_MAX || vocab < 1 || vocab > INT32_MAX / 2 ||
      ldx < 0 || (dtype != PP_F16 && dtype != PP_BF16 && dtype != PP_F32) || !pp::aligned(logits, size) || top < 0 ||
      top > PP_LOGPROBS_MAX_TOP || top > vocab || (top && (!top_ids || !top_logprobs))) {
    pp::set_error("pp_token_logprobs: FP16, BF16 or FP32 logits, tokens and outputs are required, at most %d "
                  "alternatives and no more than the vocabulary has",
                  PP_LOGPROBS_MAX_TOP);
    return PP_ERR_INVALID;
  }
  const pp::ScoreParams p{logits, ldx, rows, (int)vocab, tokens, (int)top, logprob, entropy, top_ids, top_logprobs, status};
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == PP_F16 ? pp::launch<__half>(p, s) : dtype == PP_BF16 ? pp::launch<__nv_bfloat16>(p, s)
                                                                       : pp::launch<float>(p, s);
}
