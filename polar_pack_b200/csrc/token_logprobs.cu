// Log probabilities of given tokens, entropy and the likeliest alternatives
// of rows of logits.
//   m = max x,  Z = sum e^(x - m)
//   logprob = x_token - m - ln Z,  entropy = ln Z - sum e^(x - m) (x - m) / Z
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "pp_common.cuh"
#include "pp_host.h"

namespace pp {
namespace {

constexpr int kThreads = 512;

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

// Larger values first, NaN before all, equal values by the lower index.
__device__ __forceinline__ uint64_t rank_key(float x, int i) {
  uint32_t u = __float_as_uint(x + 0.f);
  u = x != x ? 0xffffffffu : u & 0x80000000u ? ~u : u | 0x80000000u;
  return (uint64_t)u << 32 | (uint32_t)(0x7fffffff - i);
}

// Sums over e^(x - m), kept beside the maximum they refer to.
struct Stat {
  float m, z, w;  // maximum, sum e^(x-m), sum e^(x-m) (x-m)
  __device__ __forceinline__ void rescale(float to) {
    if (to == m) return;
    const float d = m - to, f = m == -INFINITY ? 0.f : expf(d);
    w = f == 0.f ? 0.f : f * (w + d * z);
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

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const ScoreParams p) {
  __shared__ Stat st[kThreads / 32];
  __shared__ uint64_t best[kThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(p.x) + r * p.ldx;
    Stat s{-INFINITY, 0.f, 0.f};
    bool nan = false;
    for (int i = tid; i < p.vocab; i += kThreads) {
      const float v = to_f(x[i]);
      nan |= v != v;
      if (v > s.m) s.rescale(v);
      const float d = v - s.m, e = v == -INFINITY ? 0.f : expf(d);
      s.z += e;
      if (e > 0.f) s.w = fmaf(e, d, s.w);
    }
    for (int o = 16; o > 0; o >>= 1) {
      Stat t{__shfl_xor_sync(0xffffffffu, s.m, o), __shfl_xor_sync(0xffffffffu, s.z, o),
             __shfl_xor_sync(0xffffffffu, s.w, o)};
      s.merge(t);
    }
    if (lane == 0) st[warp] = s;
    nan = __syncthreads_or(nan);
    s = st[0];
    for (int i = 1; i < kThreads / 32; ++i) s.merge(st[i]);
    float lse = s.m + logf(s.z), ent = logf(s.z) - s.w / s.z;
    if (s.m == -INFINITY) {
      lse = 0.f;
      ent = 0.f;
    }
    if (nan || s.m == INFINITY) {
      lse = nan ? NAN : INFINITY;
      ent = NAN;
    }
    if (tid == 0) {
      const int t = p.tokens[r];
      p.logprob[r] = t < 0 ? 0.f : t < p.vocab ? to_f(x[t]) - lse : NAN;
      p.entropy[r] = ent;
      if (t >= p.vocab && p.status) atomicExch(p.status, 4);
    }
    uint64_t prev = ~0ull;
    for (int k = 0; k < p.top; ++k) {
      uint64_t b = 0;
      for (int i = tid; i < p.vocab; i += kThreads) {
        const uint64_t key = rank_key(to_f(x[i]), i);
        if ((k == 0 || key < prev) && key > b) b = key;
      }
      for (int o = 16; o > 0; o >>= 1) {
        const uint64_t c = __shfl_xor_sync(0xffffffffu, b, o);
        b = c > b ? c : b;
      }
      if (lane == 0) best[warp] = b;
      __syncthreads();
      b = best[0];
      for (int i = 1; i < kThreads / 32; ++i) b = best[i] > b ? best[i] : b;
      __syncthreads();
      prev = b;
      if (tid == 0) {
        const int i = 0x7fffffff - (int)(uint32_t)b;
        p.top_ids[r * p.top + k] = i;
        p.top_logprobs[r * p.top + k] = to_f(x[i]) - lse;
      }
    }
    __syncthreads();
  }
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
  pp::ScoreParams p{logits, ldx, rows, (int)vocab, tokens, (int)top, logprob, entropy, top_ids, top_logprobs, status};
  const unsigned grid = (unsigned)(rows < (1 << 20) ? rows : (1 << 20));
  auto kern = dtype == PP_F16 ? pp::token_logprobs_kernel<__half>
              : dtype == PP_BF16 ? pp::token_logprobs_kernel<__nv_bfloat16> : pp::token_logprobs_kernel<float>;
  return pp::launch_kernel("token_logprobs_kernel", pp::launch_overlap(), kern, dim3(grid), dim3(pp::kThreads), 0,
                           reinterpret_cast<cudaStream_t>(stream), p);
}
