// Sampling a token from a row of logits with temperature, top-k, top-p and
// min-p, from a uniform number the caller gives.
//
// Definition, per row (logits x, temperature t, uniform u):
//   order the tokens by logit, largest first, equal logits by index;
//   w_i = exp((x_i - x_max) / t);
//   top-k: the first k;  top-p: of those, the shortest prefix whose weight is
//   at least p times theirs;  min-p: of those, the ones with w_i >= min_p;
//   never fewer than the first token;
//   id = the first kept index (in vocabulary order) at which the running sum
//   of kept weights exceeds u times their total;  logprob = log(w_id / total).
// t <= 0 (or NaN) takes the first token.  A NaN or -inf logit is masked (never
// taken); with +inf logits these share all weight; a row with nothing left
// gives id -1 and logprob -inf.
//
// A choice at a border must not depend on the order of a sum, so weights are
// summed as integers: W = round(2^43 exp(.)), which keeps V <= 2^20 of them
// below 2^63 and is exact in any order.
//
// The kept set is a prefix of the order, so it is found by selection, not by
// sorting: a radix descent over the logits' order-preserving 32-bit keys, 8
// bits at a time, counting (top-k) or adding weights (top-p) per digit.
#include "common.cuh"

namespace ml {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int64_t kMaxVocab = (int64_t)1 << 20;
constexpr double kOne = 8796093022208.0;  // 2^43

struct SampleArgs {
  const void* logits;  // [rows, V] at row pitch ld
  int64_t ld;
  int dtype;
  int V;
  const float* u;
  const float* temperature;  // null: the value
  const int64_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_v, top_p_v, min_p_v;
  int64_t top_k_v;
  int64_t* id;
  float* logprob;
};

// Unsigned order of the key = order of the logits, masked ones 0.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x > -INFINITY)) return 0;  // NaN and -inf
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 -> +0: equal logits, equal keys
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

__device__ __forceinline__ uint64_t weight(uint32_t key, double top, double inv_t) {
  if (key == 0) return 0;
  const float x = value_of(key);
  if (x == INFINITY) return (uint64_t)kOne;
  return (uint64_t)__double2ll_rn(exp(((double)x - top) * inv_t) * kOne);
}

struct Shared {
  uint64_t hist[256];
  uint64_t part[kWarps];
  uint32_t cut_key;   // the prefix keeps keys above it ...
  uint32_t cut_ties;  // ... and this many equal to it, lowest index first
  uint64_t above;
  int digit;
};

__device__ __forceinline__ uint64_t block_sum(uint64_t v, uint64_t* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  uint64_t s = 0;
  for (int i = 0; i < kWarps; ++i) s += part[i];
  return s;
}

__global__ void __launch_bounds__(kThreads) sample_simple(const __grid_constant__ SampleArgs a) {
  __shared__ Shared sh;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto key_at = [&](int i) { return key_of(load_as_f32(a.logits, row * a.ld + i, a.dtype)); };
  const float t = a.temperature ? a.temperature[row] : a.temperature_v;
  const int64_t k = a.top_k ? a.top_k[row] : a.top_k_v;
  const double p = a.top_p ? a.top_p[row] : a.top_p_v;
  const double least = a.min_p ? a.min_p[row] : a.min_p_v;

  // the first token of the order: largest key, lowest index
  uint64_t best = 0;
  for (int i = tid; i < a.V; i += kThreads) {
    const uint64_t c = ((uint64_t)key_at(i) << 32) | (uint32_t)~i;
    if (c > best) best = c;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t c = __shfl_xor_sync(0xffffffffu, best, o);
    if (c > best) best = c;
  }
  if (lane == 0) sh.part[warp] = best;
  __syncthreads();
  for (int i = 0; i < kWarps; ++i)
    if (sh.part[i] > best) best = sh.part[i];
  const uint32_t top_key = (uint32_t)(best >> 32);
  if (top_key == 0 || !(t > 0.f)) {
    if (tid == 0) {
      a.id[row] = top_key == 0 ? -1 : (int64_t)(uint32_t)~(uint32_t)best;
      a.logprob[row] = top_key == 0 ? -INFINITY : 0.f;
    }
    return;
  }
  const double top = value_of(top_key), inv_t = 1.0 / (double)t;

  // kept: key > cut_key, or the first cut_ties of the equal ones
  uint32_t cut_key = 0, cut_ties = 0;
  int tie_end = 0;  // first index whose equal key is no longer kept
  // pass 0: top-k by count, pass 1: top-p by weight among those
  for (int pass = 0; pass < 2; ++pass) {
    const bool on = pass == 0 ? (k > 0 && k < a.V) : p < 1.0;
    if (!on) continue;
    auto value = [&](int i, uint32_t key) -> uint64_t {
      const bool in = key > cut_key || (key == cut_key && i < tie_end && key != 0);
      if (!in) return 0;
      return pass == 0 ? 1 : weight(key, top, inv_t);
    };
    uint64_t need;  // the prefix ends where the running value reaches this
    uint64_t total = 0;
    for (int i = tid; i < a.V; i += kThreads) total += value(i, key_at(i));
    total = block_sum(total, sh.part);
    if (pass == 0) {
      need = (uint64_t)k;
      if (need >= total) continue;
    } else {
      const double f = p * (double)total;
      need = f <= 1.0 ? 1 : (uint64_t)ceil(f);
    }
    uint32_t prefix = 0;
    uint64_t above = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (tid < 256) sh.hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < a.V; i += kThreads) {
        const uint32_t key = key_at(i);
        if (shift < 24 && (key >> (shift + 8)) != (prefix >> (shift + 8))) continue;
        const uint64_t v = value(i, key);
        if (v) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.hist[(key >> shift) & 255]),
                         (unsigned long long)v);
      }
      __syncthreads();
      if (tid == 0) {
        uint64_t run = above;
        int d = 255;
        for (; d > 0; --d) {
          if (run + sh.hist[d] >= need) break;
          run += sh.hist[d];
        }
        sh.digit = d;
        sh.above = run;
      }
      __syncthreads();
      above = sh.above;
      prefix |= (uint32_t)sh.digit << shift;
    }
    const uint64_t each = pass == 0 ? 1 : weight(prefix, top, inv_t);
    const uint64_t left = need - above;
    cut_ties = (uint32_t)(each ? min((left + each - 1) / each, (uint64_t)a.V) : 1);
    // equal keys that an earlier cut kept in part stay bounded by it
    const int bound = prefix == cut_key ? tie_end : a.V;
    cut_key = prefix;
    // index of the cut_ties-th equal key: chunks of kThreads in index order
    int seen = 0, end = bound;
    for (int i0 = 0; i0 < a.V; i0 += kThreads) {
      const int i = i0 + tid;
      const bool eq = i < bound && key_at(i) == cut_key;
      const unsigned m = __ballot_sync(0xffffffffu, eq);
      __syncthreads();
      if (lane == 0) sh.part[warp] = __popc(m);
      __syncthreads();
      int before = seen, all = 0;
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += (int)sh.part[w];
        all += (int)sh.part[w];
      }
      before += __popc(m & ((1u << lane) - 1));
      if (eq && before == (int)cut_ties - 1) sh.digit = i + 1;
      __syncthreads();
      if (seen + all >= (int)cut_ties) {
        end = sh.digit;
        break;
      }
      seen += all;
    }
    tie_end = end;
  }

  // draw among the kept ones, in index order
  auto kept_weight = [&](int i) -> uint64_t {
    const uint32_t key = key_at(i);
    if (key == 0) return 0;
    if (!(key > cut_key || (key == cut_key && i < tie_end))) return 0;
    if (key != top_key && (key_of(INFINITY) == top_key ||
                           !(exp(((double)value_of(key) - top) * inv_t) >= least)))
      return 0;
    // at least the first token stays, whatever min_p
    if (key == top_key && least > 1.0) return i == (int)~(uint32_t)best ? (uint64_t)kOne : 0;
    return weight(key, top, inv_t);
  };
  uint64_t total = 0;
  for (int i = tid; i < a.V; i += kThreads) total += kept_weight(i);
  total = block_sum(total, sh.part);
  float uf = a.u[row];
  const double target = (uf > 0.f ? (double)uf : 0.0) * (double)total;
  uint64_t run = 0;
  __syncthreads();
  if (tid == 0) sh.digit = -1;
  int last = -1;
  for (int i0 = 0; i0 < a.V; i0 += kThreads) {
    const int i = i0 + tid;
    const uint64_t w = i < a.V ? kept_weight(i) : 0;
    uint64_t s = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t c = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += c;
    }
    __syncthreads();
    if (lane == 31) sh.part[warp] = s;
    __syncthreads();
    uint64_t before = run, all = 0;
    for (int v = 0; v < kWarps; ++v) {
      if (v < warp) before += sh.part[v];
      all += sh.part[v];
    }
    const uint64_t upto = before + s;
    if (w) {
      last = i;
      if ((double)upto > target && !((double)(upto - w) > target)) sh.digit = i;
    }
    __syncthreads();
    run += all;
    if (sh.digit >= 0) break;
  }
  __syncthreads();
  int id = sh.digit;
  if (id < 0) {  // u at or past 1: the last kept token
    const int top_last = (int)__reduce_max_sync(0xffffffffu, last);
    __syncthreads();
    if (lane == 0) sh.part[warp] = (uint64_t)(int64_t)top_last;
    __syncthreads();
    for (int i = 0; i < kWarps; ++i) id = max(id, (int)(int64_t)sh.part[i]);
  }
  if (tid == 0) {
    a.id[row] = id;
    const float x = value_of(key_at(id));
    const double z = x == INFINITY ? 0.0 : ((double)x - top) * inv_t;
    a.logprob[row] = (float)(z - log((double)total / kOne));
  }
}

}  // namespace
}  // namespace ml

using namespace ml;

extern "C" int ml_sample(const void* logits, int64_t ld, int logits_dtype, int64_t rows,
                         int64_t vocab, const float* uniform, const float* temperature,
                         float temperature_value, const int64_t* top_k, int64_t top_k_value,
                         const float* top_p, float top_p_value, const float* min_p,
                         float min_p_value, int64_t* id, float* logprob, void* stream) {
  ML_CHECK_ARG(rows >= 0 && vocab > 0, "sample: bad sizes");
  ML_CHECK_ARG(vocab <= kMaxVocab, "sample: a vocabulary of %lld (at most %lld)", (long long)vocab,
               (long long)kMaxVocab);
  ML_CHECK_ARG(logits_dtype >= 0 && logits_dtype <= 2, "sample: bad dtype code");
  if (rows == 0) return ML_OK;
  ML_CHECK_ARG(logits && uniform && id && logprob, "sample: null pointer");
  ML_CHECK_ARG(rows < ((int64_t)1 << 31), "sample: too many rows");
  SampleArgs a = {logits, ld, logits_dtype, (int)vocab, uniform, temperature, top_k, top_p, min_p,
                  temperature_value, top_p_value, min_p_value, top_k_value, id, logprob};
  sample_simple<<<(unsigned)rows, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  ML_CHECK_LAUNCH("sample");
  return ML_OK;
}
