// Attention over the 8-bit KV cache (kv8.cuh): one query row of one kv
// head's group per CTA.
//   s_t = scale * q . k_t,  p = softmax(s) over t <= the query's position,
//   out = sum_t p_t v_t     (FP32 throughout, rounded once)
#include "kv8.cuh"

namespace pp {
namespace {

constexpr int kTile = 128;    // positions per step, one thread each
constexpr int kMaxGroup = 16;

struct AttnParams {
  Kv8Cache c;
  const __half* q;
  int64_t ldqb, ldqt, ldqh;
  __half* out;
  int64_t ldob, ldot, ldoh;
  const int* lens;
  int extra;            // tokens beyond lens: 1 after a fused append, else 0
  const int* counts;
  int n, nq;
  float scale;
  Kv8Rope rope;
  float* weights;       // [batch][kv head][cap] += the group's probabilities (n == 1), or NULL
  int* status;
};

template <int HD>
__global__ void __launch_bounds__(kTile) kv8_attention_kernel(const AttnParams p) {
  __shared__ float qs[kMaxGroup][HD];
  __shared__ float ss[kMaxGroup][kTile];
  __shared__ float red[kTile / 32];
  __shared__ __align__(16) __half vrow[HD];
  pdl_launch_dependents();
  pdl_wait();
  const int i = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int group = p.nq / p.c.nkv;
  const int len = p.lens[b] + p.extra;
  const int cnt = p.counts ? min(max(p.counts[b], 0), p.n) : p.n;
  const int end = len - cnt + i + 1;  // positions attended
  bool ok = len <= p.c.cap;
  const int r = p.rope.cos ? p.rope.pos[b] + i : 0;
  if (p.rope.cos && len > 0 && i < cnt && (r < 0 || r >= p.rope.len)) ok = false;
  if (!ok && tid == 0 && p.status) atomicExch(p.status, 5);
  __half* out = p.out + b * p.ldob + i * p.ldot + (int64_t)kvh * group * p.ldoh;
  if (!ok || i >= cnt || end <= 0) {
    for (int e = tid; e < group * HD; e += kTile) out[e / HD * p.ldoh + e % HD] = __float2half(0.f);
    return;
  }
  const __half* q = p.q + b * p.ldqb + i * p.ldqt + (int64_t)kvh * group * p.ldqh;
  for (int e = tid; e < group * HD / 8; e += kTile) {
    const int h = e / (HD / 8), d0 = e % (HD / 8) * 8;
    const uint4 x = kv8_load8(q + h * p.ldqh, d0, HD, p.rope, r);
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(u2h(u[j]));
      qs[h][d0 + 2 * j] = f.x;
      qs[h][d0 + 2 * j + 1] = f.y;
    }
  }
  float mx[kMaxGroup], sum[kMaxGroup], acc[kMaxGroup];
#pragma unroll
  for (int h = 0; h < kMaxGroup; ++h) {
    mx[h] = -INFINITY;
    sum[h] = 0.f;
    acc[h] = 0.f;
  }
  __syncthreads();
  auto scores = [&](int t, float (&s)[kMaxGroup]) {
#pragma unroll
    for (int h = 0; h < kMaxGroup; ++h) s[h] = 0.f;
    for (int d0 = 0; d0 < HD; d0 += 8) {
      const bool tail = t / kKvBlock == kv8_last_block(len);
      float k[8];
      float mul = 1.f;
      if (tail) {
        const uint4 x = *reinterpret_cast<const uint4*>(p.c.tail_row(0, b, kvh, t % kKvBlock) + d0);
        const uint32_t u[4] = {x.x, x.y, x.z, x.w};
        for (int j = 0; j < 4; ++j) {
          const float2 f = __half22float2(u2h(u[j]));
          k[2 * j] = f.x;
          k[2 * j + 1] = f.y;
        }
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(p.c.code_row(0, b, kvh, t) + d0);
        for (int j = 0; j < 8; ++j) k[j] = (float)((int)((j < 4 ? x.x : x.y) >> (8 * (j & 3)) & 255u) - 128);
        mul = *p.c.scale(0, b, kvh, t / kKvBlock);
      }
      for (int h = 0; h < group; ++h) {
        float a = 0.f;
        for (int j = 0; j < 8; ++j) a = fmaf(qs[h][d0 + j], k[j], a);
        s[h] = fmaf(a, mul, s[h]);
      }
    }
  };
  for (int t0 = 0; t0 < end; t0 += kTile) {
    float s[kMaxGroup];
    const int t = t0 + tid;
    if (t < end) scores(t, s);
    for (int h = 0; h < group; ++h) ss[h][tid] = t < end ? s[h] * p.scale : -INFINITY;
    __syncthreads();
    const int rows = min(kTile, end - t0);
    for (int h = 0; h < group; ++h) {
      float m = mx[h];
      for (int j = 0; j < rows; ++j) m = fmaxf(m, ss[h][j]);
      const float c = mx[h] == -INFINITY ? 0.f : expf(mx[h] - m);
      sum[h] *= c;
      acc[h] *= c;
      mx[h] = m;
    }
    if (tid < HD)
      for (int j = 0; j < rows; ++j) {
        const int tt = t0 + j;
        float v;
        if (tt / kKvBlock == kv8_last_block(len))
          v = __half2float(p.c.tail_row(1, b, kvh, tt % kKvBlock)[tid]);
        else
          v = ((int)p.c.code_row(1, b, kvh, tt)[tid] - 128) * *p.c.scale(1, b, kvh, tt / kKvBlock);
        for (int h = 0; h < group; ++h) {
          const float e = expf(ss[h][j] - mx[h]);
          sum[h] += e;
          acc[h] = fmaf(e, v, acc[h]);
        }
      }
    else
      for (int j = 0; j < rows; ++j)
        for (int h = 0; h < group; ++h) sum[h] += expf(ss[h][j] - mx[h]);
    __syncthreads();
  }
  if (tid < HD)
    for (int h = 0; h < group; ++h) out[h * p.ldoh + tid] = __float2half_rn(acc[h] / sum[h]);
  if (p.weights) {
    for (int t = tid; t < end; t += kTile) {
      float s[kMaxGroup], w = 0.f;
      scores(t, s);
      for (int h = 0; h < group; ++h) w += expf(s[h] * p.scale - mx[h]) / sum[h];
      p.weights[p.c.head(b, kvh) * p.c.cap + t] += w;
    }
  }
}

}  // namespace
}  // namespace pp

extern "C" {

int pp_kv8_attention_workspace_bytes(const pp_kv8_cache* cache, int64_t n, int64_t nq, int weights, size_t* bytes) {
  pp::Kv8Cache c{};
  if (int rc = pp::kv8_cache("pp_kv8_attention_workspace_bytes", cache, &c)) return rc;
  if (!bytes || n < 0 || nq < 1) {
    pp::set_error("pp_kv8_attention_workspace_bytes: invalid arguments");
    return PP_ERR_INVALID;
  }
  *bytes = 0;
  return PP_OK;
}

static int kv8_run(const char* who, pp::AttnParams& p, const void* q, const int64_t* qs, int64_t n, int64_t nq,
                   const int* lens, float scale, void* out, const int64_t* os, void* stream) {
  const bool heads = nq >= 1 && nq % p.c.nkv == 0 && nq / p.c.nkv <= pp::kMaxGroup;
  if (n == 0 && heads) return PP_OK;
  if (!q || !qs || !lens || !out || !os || n < 0 || n > 65535 || !heads) {
    pp::set_error("%s: queries, lengths and outputs are required, at most 65535 tokens, query heads a multiple of the kv "
                  "heads (at most %d for each)", who, pp::kMaxGroup);
    return PP_ERR_INVALID;
  }
  for (int i = 0; i < 3; ++i)
    if (!pp::aligned(q, 16) || !pp::aligned(out, 16) || qs[i] % 8 || os[i] % 8) {
      pp::set_error("%s: query and output rows must be 16-byte aligned", who);
      return PP_ERR_INVALID;
    }
  p.q = reinterpret_cast<const __half*>(q);
  p.ldqb = qs[0];
  p.ldqt = qs[1];
  p.ldqh = qs[2];
  p.out = reinterpret_cast<__half*>(out);
  p.ldob = os[0];
  p.ldot = os[1];
  p.ldoh = os[2];
  p.lens = lens;
  p.n = (int)n;
  p.nq = (int)nq;
  p.scale = scale;
  return pp::launch_kernel("kv8_attention_kernel", pp::launch_overlap(),
                           p.c.hd == 128 ? pp::kv8_attention_kernel<128> : pp::kv8_attention_kernel<64>,
                           dim3((unsigned)n, (unsigned)p.c.nkv, (unsigned)p.c.batch), dim3(pp::kTile), 0,
                           reinterpret_cast<cudaStream_t>(stream), p);
}

int pp_kv8_attention(const pp_kv8_cache* cache, const void* q, const int64_t q_strides[3], int64_t n, int64_t nq,
                     const int* lens, const int* counts, float scale, void* out, const int64_t out_strides[3],
                     const void* cos_t, const void* sin_t, const int* rope_pos, int64_t rope_len, void* workspace,
                     size_t workspace_bytes, int* status, void* stream) {
  (void)workspace;
  (void)workspace_bytes;
  pp::AttnParams p{};
  if (int rc = pp::kv8_cache("pp_kv8_attention", cache, &p.c)) return rc;
  if (int rc = pp::kv8_rope("pp_kv8_attention", cos_t, sin_t, rope_pos, rope_len, &p.rope)) return rc;
  p.counts = counts;
  p.status = status;
  return kv8_run("pp_kv8_attention", p, q, q_strides, n, nq, lens, scale, out, out_strides, stream);
}

int pp_kv8_decode(const pp_kv8_cache* cache, const void* q, const int64_t q_strides[2], int64_t nq, const void* k,
                  const int64_t k_strides[2], const void* v, const int64_t v_strides[2], const int* pos, float scale,
                  float* weights, void* out, const int64_t out_strides[2], const void* cos_t, const void* sin_t,
                  const int* rope_pos, int64_t rope_len, void* workspace, size_t workspace_bytes, int* status,
                  void* stream) {
  (void)workspace;
  (void)workspace_bytes;
  pp::AttnParams p{};
  if (int rc = pp::kv8_cache("pp_kv8_decode", cache, &p.c)) return rc;
  if (int rc = pp::kv8_rope("pp_kv8_decode", cos_t, sin_t, rope_pos, rope_len, &p.rope)) return rc;
  if (!q_strides || !k_strides || !v_strides || !out_strides) {
    pp::set_error("pp_kv8_decode: strides are required");
    return PP_ERR_INVALID;
  }
  const int64_t ks[3] = {k_strides[0], 0, k_strides[1]}, vs[3] = {v_strides[0], 0, v_strides[1]};
  if (int rc = pp_kv8_append(cache, k, ks, v, vs, 1, pos, nullptr, cos_t, sin_t, rope_pos, rope_len, status, stream))
    return rc;
  p.extra = 1;
  p.weights = weights;
  p.status = status;
  const int64_t qs[3] = {q_strides[0], 0, q_strides[1]}, os[3] = {out_strides[0], 0, out_strides[1]};
  return kv8_run("pp_kv8_decode", p, q, qs, 1, nq, pos, scale, out, os, stream);
}

}  // extern "C"
