// Attention over the 8-bit KV cache (kv8.cuh): the choice between the kernel
// for few query rows per kv head (kv8_decode.cuh) and the one for many
// (kv8_prompt.cuh), their plans and the entry points.
#include "kv8.cuh"
#include "kv8_decode.cuh"
#include "kv8_prompt.cuh"

namespace pp {
namespace {

constexpr int kMaxGroup = 16;

// How a call with `rows` query rows per kv head runs on kv8_decode_kernel:
// tiles of 8 rows while one is enough, else of 16.
constexpr int kDecodeBatch = 512;  // sequences of a launch

struct DecodePlan {
  int nt, tiles, ctas;
  size_t cnt, part, lse, scores, bytes;  // workspace offsets
};

DecodePlan plan_decode(const Kv8Cache& c, int64_t n, int64_t nq, bool weights, int ctas) {
  DecodePlan d{};
  const int64_t rows = n * (nq / c.nkv);
  d.nt = rows <= 8 ? 1 : 2;
  d.tiles = (int)cdiv(rows, 8 * d.nt);
  d.ctas = ctas;
  d.part = align_up((size_t)ctas * sizeof(int), 256);  // the counters' place must not depend on the call
  d.lse = align_up(d.part + (size_t)ctas * 2 * kv8_part_floats(d.nt, c.hd) * sizeof(float), 256);
  d.scores = align_up(d.lse + (weights ? (size_t)c.batch * nq * sizeof(float) : 0), 256);
  d.bytes = d.scores + (weights ? (size_t)c.batch * nq * c.cap * sizeof(float) : 0);
  return d;
}

// More rows go to kv8_prompt_kernel.  With few tiles for the SMs, a tile's
// positions may be split into parts of at least eight blocks: as many of them
// here as the lengths, which are on the device, can make use of
// (kv8_part_blocks).
struct PromptPlan {
  int64_t base;  // tiles of all heads
  int tiles, splits;
  size_t join, part, bytes;  // of the workspace, after the other kernel's counters
};

PromptPlan plan_prompt(const Kv8Cache& c, int64_t n, int64_t nq, int ctas) {
  PromptPlan d{};
  const int64_t rows = n * (nq / c.nkv);
  d.tiles = (int)cdiv(rows, kPrRows);
  d.base = (int64_t)d.tiles * c.nkv * c.batch;
  int64_t s = c.batch <= kPrSplitBatch ? 2 * ctas / d.base : 1;
  if (s > c.cap / kKvBlock / 8) s = c.cap / kKvBlock / 8;
  if (s > kPrMaxSplits) s = kPrMaxSplits;
  d.splits = s > 1 ? (int)s : 1;
  d.join = align_up((size_t)ctas * sizeof(int), 256);
  d.part = d.join + 256;
  d.bytes = d.splits > 1 ? d.part + (size_t)d.splits * c.batch * c.nkv * rows * (c.hd + 2) * sizeof(float) : 0;
  return d;
}

// Whether kv8_decode_kernel takes a call: a single row tile always, more than
// 256 rows never.  Between, the times that the two kernels would take at full
// caches, in ns, as measured on 148 SMs (16 query heads on 2 kv heads of 128):
// decode 12 us and one for 300 blocks of 16 rows, a segment counting eight
// more; prompt 9 us, 1.45 for a CTA's block, 4 for joining parts.  The lengths
// are on the device, so the estimate is by the capacity.
//   sequences, positions, rows   decode  prompt (us)
//   1, 512, 256                  13.0    19.8
//   4, 4096, 96                  19.5    27.2
//   4, 4096, 128                 25.2    26.5 (taken, by 5% the slower)
//   32, 512, 32                  14.0    22.0
//   32, 512, 64                  34.4    22.1
//   32, 4096, 32                 32.6    63.7
//   32, 4096, 64                 64.8    65.1
bool decode_takes(const Kv8Cache& c, int64_t n, int64_t nq, int ctas) {
  const int64_t rows = n * (nq / c.nkv);
  if (rows <= 16 || rows > 256) return rows <= 16;
  const PromptPlan pr = plan_prompt(c, n, nq, ctas);
  const int64_t heads = (int64_t)c.nkv * c.batch, blocks = c.cap / kKvBlock;
  const int64_t decode = 12000 + heads * cdiv(rows, 16) * (blocks + 8) * 10 / 3;
  for (int64_t k = 1; k <= pr.splits; ++k)  // parts of a tile's positions
    if (decode > 9000 + 1450 * cdiv(blocks, k) * cdiv(pr.base * k, ctas) + (k > 1 ? 4000 : 0)) return false;
  return true;
}

bool g_attr[10][64];
int g_limit[10][64];

int encode_codes(const Kv8Cache& c, CUtensorMap (&tm)[2]) {
  const uint64_t rows = (uint64_t)c.batch * c.nkv * c.cap;
  for (int w = 0; w < 2; ++w)
    if (int rc = encode_tmap_2d(&tm[w], CU_TENSOR_MAP_DATA_TYPE_UINT8, c.codes[w], c.hd, rows, c.hd, c.hd, kKvBlock,
                                c.hd == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B))
      return rc;
  return PP_OK;
}

template <int NT, int HD, bool MANY>
int launch_decode(const Kv8DecodeParams& p, int ctas, cudaStream_t s) {
  constexpr int kv = (NT - 1) * 4 + MANY * 2 + (HD == 128);
  using S = Kv8DecodeSmem<NT, HD>;
  auto kern = kv8_decode_kernel<NT, HD, MANY>;
  int lim = 0;
  if (int rc = ensure_smem_attr(kern, g_attr[kv], g_limit[kv], &lim)) return rc;
  const int smem = S::bytes(p.c.batch);
  if (smem > lim) {
    set_error("kv8_decode_kernel: %d bytes of shared memory needed, %d available", smem, lim);
    return PP_ERR_CUDA;
  }
  CUtensorMap tm[2];
  if (int rc = encode_codes(p.c, tm)) return rc;
  return launch_kernel("kv8_decode_kernel", launch_overlap(), kern, dim3((unsigned)ctas), dim3(kv8_warps(NT) * 32),
                       (size_t)smem, s, p, tm[0], tm[1]);
}

template <bool MANY>
int launch_decode(const Kv8DecodeParams& p, int nt, int ctas, cudaStream_t s) {
  if (p.c.hd == 128) return nt == 1 ? launch_decode<1, 128, MANY>(p, ctas, s) : launch_decode<2, 128, MANY>(p, ctas, s);
  return nt == 1 ? launch_decode<1, 64, MANY>(p, ctas, s) : launch_decode<2, 64, MANY>(p, ctas, s);
}

template <int HD>
int launch_prompt(const Kv8PromptParams& p, cudaStream_t s) {
  using S = Kv8PromptSmem<HD>;
  constexpr int kv = 8 + (HD == 128);
  auto kern = kv8_prompt_kernel<HD>;
  int lim = 0;
  if (int rc = ensure_smem_attr(kern, g_attr[kv], g_limit[kv], &lim)) return rc;
  if (S::kBytes > lim) {
    set_error("kv8_prompt_kernel: %d bytes of shared memory needed, %d available", S::kBytes, lim);
    return PP_ERR_CUDA;
  }
  CUtensorMap tm[2];
  if (int rc = encode_codes(p.c, tm)) return rc;
  const dim3 grid((unsigned)(p.c.nkv * p.c.batch), (unsigned)(p.tiles * p.splits));
  if (int rc = launch_kernel("kv8_prompt_kernel", launch_overlap(), kern, grid, dim3(kPrThreads), (size_t)S::kBytes, s,
                             p, tm[0], tm[1]))
    return rc;
  if (p.splits == 1) return PP_OK;
  const Kv8JoinParams j{p.part, p.out, p.ldob, p.ldot, p.ldoh, p.lens, p.part_blocks, p.c.batch, p.c.nkv, p.n, p.nq,
                        p.splits, p.c.cap};
  const int64_t rows = (int64_t)p.c.batch * p.c.nkv * p.n * (p.nq / p.c.nkv);
  // started early whatever the overlap setting: it waits for the attention itself
  return launch_kernel("kv8_join_kernel", true, kv8_join_kernel<HD>, dim3((unsigned)cdiv(rows, 8)), dim3(256), 0, s, j);
}

// Query and output rows, heads and sizes, checked.  Sets *empty for a call
// without work.
int check_rows(const char* who, const Kv8Cache& c, const void* q, const int64_t* qs, int64_t n, int64_t nq,
               const int* lens, const void* out, const int64_t* os, const int* status, bool* empty) {
  const bool heads = nq >= 1 && nq % c.nkv == 0 && nq / c.nkv <= kMaxGroup;
  *empty = n == 0 && heads;
  if (*empty) return PP_OK;
  if (!q || !qs || !lens || !out || !os || !status || n < 0 || n > 65535 || !heads) {
    set_error("%s: queries, lengths, outputs and a status word are required, at most 65535 tokens, query heads a "
              "multiple of the kv heads (at most %d for each)", who, kMaxGroup);
    return PP_ERR_INVALID;
  }
  for (int i = 0; i < 3; ++i)
    if (!aligned(q, 16) || !aligned(out, 16) || qs[i] % 8 || os[i] % 8) {
      set_error("%s: query and output rows must be 16-byte aligned", who);
      return PP_ERR_INVALID;
    }
  if ((int64_t)c.batch * c.nkv * c.cap > INT32_MAX) {
    set_error("%s: sequences x heads x capacity must stay below 2^31", who);
    return PP_ERR_INVALID;
  }
  return PP_OK;
}

int run_decode(const char* who, Kv8DecodeParams& p, float* weights, void* workspace, size_t workspace_bytes,
               cudaStream_t s) {
  const int ctas = device_sm_count(current_device());
  if (ctas < 1) {
    set_error("%s: no current CUDA device", who);
    return PP_ERR_CUDA;
  }
  const DecodePlan d = plan_decode(p.c, p.n, p.nq, weights != nullptr, ctas);
  if (!workspace || workspace_bytes < d.bytes || !aligned(workspace, 256)) {
    set_error("%s: workspace of %zu bytes (256-byte aligned, zero-filled) required", who, d.bytes);
    return PP_ERR_WORKSPACE;
  }
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  p.tiles = d.tiles;
  p.cnt = reinterpret_cast<int*>(ws);
  p.part = reinterpret_cast<float*>(ws + d.part);
  if (weights) {
    p.lse = reinterpret_cast<float*>(ws + d.lse);
    p.scores = reinterpret_cast<float*>(ws + d.scores);
  }
  // a launch keeps its sequences' lengths in shared memory: larger batches go in parts
  const Kv8DecodeParams all = p;
  for (int b0 = 0; b0 < all.c.batch; b0 += kDecodeBatch) {
    const int64_t heads = (int64_t)b0 * all.c.nkv;
    p.c.batch = all.c.batch - b0 < kDecodeBatch ? all.c.batch - b0 : kDecodeBatch;
    for (int w = 0; w < 2; ++w) {
      p.c.codes[w] = all.c.codes[w] + heads * all.c.cap * all.c.hd;
      p.c.scales[w] = all.c.scales[w] + heads * (all.c.cap / kKvBlock);
      p.c.tail[w] = all.c.tail[w] + heads * kKvBlock * all.c.hd;
      p.x[w] = all.x[w] ? all.x[w] + b0 * all.ldxb[w] : nullptr;
    }
    p.q = all.q + b0 * all.ldqb;
    p.out = all.out + b0 * all.ldob;
    p.lens = all.lens + b0;
    p.counts = all.counts ? all.counts + b0 : nullptr;
    p.rope.pos = all.rope.pos ? all.rope.pos + b0 : nullptr;
    if (weights) {
      p.lse = all.lse + (int64_t)b0 * all.nq;
      p.scores = all.scores + (int64_t)b0 * all.nq * all.c.cap;
    }
    if (int rc = p.n > 1 ? launch_decode<true>(p, d.nt, ctas, s) : launch_decode<false>(p, d.nt, ctas, s)) return rc;
  }
  if (!weights) return PP_OK;
  const Kv8WeightsParams w{all.scores, all.lse, weights, all.lens, all.rope, all.extra, all.nq, all.c.nkv, all.c.cap};
  // started early whatever the overlap setting: it waits for the decode kernel itself
  return launch_kernel("kv8_weights_kernel", true, kv8_weights_kernel,
                       dim3((unsigned)cdiv(all.c.cap, 256), (unsigned)all.c.nkv, (unsigned)all.c.batch), dim3(256), 0, s,
                       w);
}

}  // namespace
}  // namespace pp

extern "C" {

int pp_kv8_attention_workspace_bytes(const pp_kv8_cache* cache, int64_t n, int64_t nq, int weights, size_t* bytes) {
  pp::Kv8Cache c{};
  if (int rc = pp::kv8_cache("pp_kv8_attention_workspace_bytes", cache, &c)) return rc;
  if (!bytes || n < 0 || nq < 1 || nq % c.nkv) {
    pp::set_error("pp_kv8_attention_workspace_bytes: invalid arguments");
    return PP_ERR_INVALID;
  }
  *bytes = 0;
  if (n == 0) return PP_OK;
  const int ctas = pp::device_sm_count(pp::current_device());
  if (ctas < 1) {
    pp::set_error("pp_kv8_attention_workspace_bytes: no current CUDA device");
    return PP_ERR_CUDA;
  }
  *bytes = pp::decode_takes(c, n, nq, ctas)
               ? pp::plan_decode(c, n, nq, weights != 0, ctas).bytes
               : pp::plan_prompt(c, n, nq, ctas).bytes;
  return PP_OK;
}

int pp_kv8_attention(const pp_kv8_cache* cache, const void* q, const int64_t q_strides[3], int64_t n, int64_t nq,
                     const int* lens, const int* counts, float scale, void* out, const int64_t out_strides[3],
                     const void* cos_t, const void* sin_t, const int* rope_pos, int64_t rope_len, void* workspace,
                     size_t workspace_bytes, int* status, void* stream) {
  pp::Kv8DecodeParams p{};
  if (int rc = pp::kv8_cache("pp_kv8_attention", cache, &p.c)) return rc;
  if (int rc = pp::kv8_rope("pp_kv8_attention", cos_t, sin_t, rope_pos, rope_len, &p.rope)) return rc;
  bool empty = false;
  if (int rc = pp::check_rows("pp_kv8_attention", p.c, q, q_strides, n, nq, lens, out, out_strides, status, &empty))
    return rc;
  if (empty) return PP_OK;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int ctas = pp::device_sm_count(pp::current_device());
  if (ctas < 1) {
    pp::set_error("pp_kv8_attention: no current CUDA device");
    return PP_ERR_CUDA;
  }
  if (pp::decode_takes(p.c, n, nq, ctas)) {
    p.q = reinterpret_cast<const __half*>(q);
    p.ldqb = q_strides[0];
    p.ldqt = q_strides[1];
    p.ldqh = q_strides[2];
    p.out = reinterpret_cast<__half*>(out);
    p.ldob = out_strides[0];
    p.ldot = out_strides[1];
    p.ldoh = out_strides[2];
    p.lens = lens;
    p.counts = counts;
    p.n = (int)n;
    p.nq = (int)nq;
    p.scale2 = scale * 1.44269504088896341f;
    p.status = status;
    return pp::run_decode("pp_kv8_attention", p, nullptr, workspace, workspace_bytes, s);
  }
  const pp::PromptPlan d = pp::plan_prompt(p.c, n, nq, ctas);
  if (d.bytes && (!workspace || workspace_bytes < d.bytes || !pp::aligned(workspace, 256))) {
    pp::set_error("pp_kv8_attention: workspace of %zu bytes (256-byte aligned) required", d.bytes);
    return PP_ERR_WORKSPACE;
  }
  pp::Kv8PromptParams a{};
  a.c = p.c;
  a.q = reinterpret_cast<const __half*>(q);
  a.ldqb = q_strides[0];
  a.ldqt = q_strides[1];
  a.ldqh = q_strides[2];
  a.out = reinterpret_cast<__half*>(out);
  a.ldob = out_strides[0];
  a.ldot = out_strides[1];
  a.ldoh = out_strides[2];
  a.lens = lens;
  a.counts = counts;
  a.n = (int)n;
  a.nq = (int)nq;
  a.scale2 = fabsf(scale) * 1.44269504088896341f;
  a.q_sign = scale < 0.f ? 0x80008000u : 0u;
  a.rope = p.rope;
  a.tiles = d.tiles;
  a.splits = d.splits;
  a.ctas = ctas;
  if (d.bytes) {
    a.part_blocks = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(workspace) + d.join);
    a.part = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(workspace) + d.part);
  }
  a.status = status;
  return p.c.hd == 128 ? pp::launch_prompt<128>(a, s) : pp::launch_prompt<64>(a, s);
}

int pp_kv8_decode(const pp_kv8_cache* cache, const void* q, const int64_t q_strides[2], int64_t nq, const void* k,
                  const int64_t k_strides[2], const void* v, const int64_t v_strides[2], const int* pos, float scale,
                  float* weights, void* out, const int64_t out_strides[2], const void* cos_t, const void* sin_t,
                  const int* rope_pos, int64_t rope_len, void* workspace, size_t workspace_bytes, int* status,
                  void* stream) {
  pp::Kv8DecodeParams p{};
  if (int rc = pp::kv8_cache("pp_kv8_decode", cache, &p.c)) return rc;
  if (int rc = pp::kv8_rope("pp_kv8_decode", cos_t, sin_t, rope_pos, rope_len, &p.rope)) return rc;
  if (!q_strides || !k || !k_strides || !v || !v_strides || !out_strides) {
    pp::set_error("pp_kv8_decode: keys, values and strides are required");
    return PP_ERR_INVALID;
  }
  const int64_t qs[3] = {q_strides[0], 0, q_strides[1]}, os[3] = {out_strides[0], 0, out_strides[1]};
  bool empty = false;
  if (int rc = pp::check_rows("pp_kv8_decode", p.c, q, qs, 1, nq, pos, out, os, status, &empty)) return rc;
  const void* x[2] = {k, v};
  const int64_t* st[2] = {k_strides, v_strides};
  for (int w = 0; w < 2; ++w) {
    if (!pp::aligned(x[w], 16) || st[w][0] % 8 || st[w][1] % 8) {
      pp::set_error("pp_kv8_decode: rows must be 16-byte aligned");
      return PP_ERR_INVALID;
    }
    p.x[w] = reinterpret_cast<const __half*>(x[w]);
    p.ldxb[w] = st[w][0];
    p.ldxh[w] = st[w][1];
  }
  p.q = reinterpret_cast<const __half*>(q);
  p.ldqb = qs[0];
  p.ldqh = qs[2];
  p.out = reinterpret_cast<__half*>(out);
  p.ldob = os[0];
  p.ldoh = os[2];
  p.lens = pos;
  p.extra = 1;
  p.n = 1;
  p.nq = (int)nq;
  p.scale2 = scale * 1.44269504088896341f;
  p.status = status;
  return pp::run_decode("pp_kv8_decode", p, weights, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
