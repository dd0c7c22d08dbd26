// Attention of one or a few query tokens per sequence over a KV cache held in
// 8 bits (kv8_append.cu writes it):
//   o[b, t, h] = sum_j softmax_j(scale * q[b, h, t] . k_j) v_j,  j <= start[b] + t,
// k_j = code * block scale, and the same for v.  A query with no position to
// see, or past its sequence's count, gives zeros.
//
// A CTA per query row: its warps take positions in turn, each with an online
// softmax (running maximum m, sum l, output o) in fp32, and merge at the end.
#include "kv8.cuh"

#include <cuda_fp8.h>

namespace ml {
namespace {

constexpr int kWarps = 8;

struct AttnArgs {
  const void* q;            // [B, Hq, T, D] at element strides
  int64_t sq[3];
  const uint8_t* codes[2];
  const float* scale[2];
  Kv8Span span;
  int q_heads, kv_heads, max_len, block;
  float qk_scale;
  void* out;                // [B, T, Hq, D]
};

template <int FMT>
__device__ __forceinline__ float decode(uint8_t c) {
  if (FMT == ML_KV8_INT8) return (float)(int8_t)c;
  __nv_fp8_e4m3 v;
  v.__x = c;
  return (float)v;
}

template <typename T, int FMT, int D>
__global__ void __launch_bounds__(32 * kWarps)
kv8_attention_simple(const __grid_constant__ AttnArgs a) {
  constexpr int E = D / 32;
  __shared__ float sm[kWarps], sl[kWarps], so[kWarps][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int kvh = h / (a.q_heads / a.kv_heads);
  const int64_t see = t < a.span.count(b) ? a.span.first(b) + t + 1 : 0;
  const int n = (int)(see < 0 ? 0 : see > a.max_len ? a.max_len : see);
  float q[E], o[E], m = -INFINITY, l = 0.f;
  const T* qp = static_cast<const T*>(a.q) + b * a.sq[0] + h * a.sq[1] + t * a.sq[2];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = to_f32(qp[lane * E + e]);
    o[e] = 0.f;
  }
  const int64_t bh = (int64_t)b * a.kv_heads + kvh;
  const int nblk = a.max_len / a.block;
  for (int j = warp; j < n; j += kWarps) {
    const uint8_t* kp = a.codes[0] + (bh * a.max_len + j) * D + lane * E;
    const uint8_t* vp = a.codes[1] + (bh * a.max_len + j) * D + lane * E;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], decode<FMT>(kp[e]), s);
    s = warp_sum(s) * (a.scale[0][bh * nblk + j / a.block] * a.qk_scale);
    const float vs = a.scale[1][bh * nblk + j / a.block];
    const float mn = s > m || s != s ? s : m;
    const float c = mn == -INFINITY ? 1.f : expf(m - mn);
    const float p = mn == -INFINITY ? 0.f : expf(s - mn);
    l = l * c + p;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * c + p * (vs * decode<FMT>(vp[e]));
    m = mn;
  }
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) so[warp][lane * E + e] = o[e];
  __syncthreads();
  T* out = static_cast<T*>(a.out) + (((int64_t)b * a.span.tokens + t) * a.q_heads + h) * D;
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float M = -INFINITY, L = 0.f, O = 0.f;
    for (int w = 0; w < kWarps; ++w) M = sl[w] > 0.f || sm[w] != sm[w] ? (sm[w] > M || sm[w] != sm[w] ? sm[w] : M) : M;
    for (int w = 0; w < kWarps; ++w) {
      if (sl[w] == 0.f) continue;
      const float c = expf(sm[w] - M);
      L += c * sl[w];
      O += c * so[w][d];
    }
    out[d] = from_f32<T>(L == 0.f ? 0.f : O / L);
  }
}

template <typename T, int FMT>
int launch(const AttnArgs& a, int64_t dim, dim3 grid, cudaStream_t st) {
  if (dim == 64) kv8_attention_simple<T, FMT, 64><<<grid, 32 * kWarps, 0, st>>>(a);
  else if (dim == 128) kv8_attention_simple<T, FMT, 128><<<grid, 32 * kWarps, 0, st>>>(a);
  else kv8_attention_simple<T, FMT, 256><<<grid, 32 * kWarps, 0, st>>>(a);
  ML_CHECK_LAUNCH("kv8_attention");
  return ML_OK;
}

}  // namespace
}  // namespace ml

using namespace ml;

extern "C" size_t ml_kv8_attention_workspace_bytes(const ml_kv8_cache* cache, int64_t q_heads,
                                                   int64_t tokens) {
  (void)cache;
  (void)q_heads;
  (void)tokens;
  return 0;
}

extern "C" int ml_kv8_attention(const ml_kv8_cache* cache, const void* q, const int64_t* q_strides,
                                int64_t q_heads, int64_t tokens, const int64_t* start,
                                int64_t start_stride, const int64_t* counts,
                                int64_t counts_stride, float scale, void* out, void* workspace,
                                size_t workspace_bytes, void* stream) {
  int rc = kv8_check("kv8_attention", cache);
  if (rc != ML_OK) return rc;
  ML_CHECK_ARG(tokens >= 0 && tokens < ((int64_t)1 << 20), "kv8_attention: bad token count");
  ML_CHECK_ARG(q_heads > 0 && q_heads <= 65535 && q_heads % cache->kv_heads == 0,
               "kv8_attention: %lld query heads for %lld kv heads", (long long)q_heads,
               (long long)cache->kv_heads);
  if (cache->batch == 0 || tokens == 0) return ML_OK;
  ML_CHECK_ARG(q && q_strides && start && out, "kv8_attention: null pointer");
  ML_CHECK_ARG((start_stride == 0 || start_stride == 1) &&
                   (counts_stride == 0 || counts_stride == 1),
               "kv8_attention: start / counts strides are 0 or 1");
  ML_CHECK_ARG(aligned16(q) && aligned16(out), "kv8_attention: q and out must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    ML_CHECK_ARG(q_strides[i] % 8 == 0, "kv8_attention: q strides must be multiples of 8 elements");
  AttnArgs a;
  a.q = q;
  for (int i = 0; i < 3; ++i) a.sq[i] = q_strides[i];
  a.codes[0] = static_cast<const uint8_t*>(cache->k_codes);
  a.codes[1] = static_cast<const uint8_t*>(cache->v_codes);
  a.scale[0] = cache->k_scale;
  a.scale[1] = cache->v_scale;
  a.span = {start, start_stride, counts, counts_stride, (int)tokens};
  a.q_heads = (int)q_heads;
  a.kv_heads = (int)cache->kv_heads;
  a.max_len = (int)cache->max_len;
  a.block = (int)cache->block;
  a.qk_scale = scale;
  a.out = out;
  const dim3 grid((unsigned)tokens, (unsigned)q_heads, (unsigned)cache->batch);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf = cache->dtype == ML_DTYPE_BF16;
  if (cache->format == ML_KV8_INT8)
    return bf ? launch<__nv_bfloat16, ML_KV8_INT8>(a, cache->head_dim, grid, st)
              : launch<__half, ML_KV8_INT8>(a, cache->head_dim, grid, st);
  return bf ? launch<__nv_bfloat16, ML_KV8_E4M3>(a, cache->head_dim, grid, st)
            : launch<__half, ML_KV8_E4M3>(a, cache->head_dim, grid, st);
}
