// The 8-bit KV cache shared by its append (kv8_append.cu) and the attention
// over it (kv8_attention.cu): code formats, the checks of a cache's
// description, and which positions a sequence's new tokens take.
#pragma once

#include "common.cuh"

namespace ml {

// Positions per CTA-processed block and per scale.
inline bool kv8_block_ok(int64_t block) { return block == 32 || block == 64 || block == 128; }
inline bool kv8_dim_ok(int64_t dim) { return dim == 64 || dim == 128 || dim == 256; }

// The description every entry point checks before it enqueues anything.
inline int kv8_check(const char* who, const ml_kv8_cache* c) {
  ML_CHECK_ARG(c != nullptr, "%s: null cache", who);
  ML_CHECK_ARG(c->format == ML_KV8_INT8 || c->format == ML_KV8_E4M3, "%s: bad code format %d", who,
               c->format);
  ML_CHECK_ARG(c->dtype == ML_DTYPE_BF16 || c->dtype == ML_DTYPE_F16,
               "%s: dtype code %d is neither bf16 nor fp16", who, c->dtype);
  ML_CHECK_ARG(kv8_dim_ok(c->head_dim), "%s: head_dim %lld not in {64, 128, 256}", who,
               (long long)c->head_dim);
  ML_CHECK_ARG(kv8_block_ok(c->block), "%s: block %lld not in {32, 64, 128}", who,
               (long long)c->block);
  ML_CHECK_ARG(c->batch >= 0 && c->kv_heads > 0 && c->max_len > 0, "%s: bad sizes", who);
  ML_CHECK_ARG(c->max_len % c->block == 0, "%s: max_len %lld is not a multiple of block %lld", who,
               (long long)c->max_len, (long long)c->block);
  ML_CHECK_ARG(c->max_len < ((int64_t)1 << 30) && c->batch <= 65535 && c->kv_heads <= 32767,
               "%s: sizes out of range", who);
  if (c->batch == 0) return ML_OK;
  ML_CHECK_ARG(c->k_codes && c->v_codes && c->k_scale && c->v_scale, "%s: null pointer", who);
  ML_CHECK_ARG(aligned16(c->k_codes) && aligned16(c->v_codes),
               "%s: cache buffers must be 16-byte aligned", who);
  return ML_OK;
}

// Rows [0, tokens) of a call hold sequence b's new tokens; the first `n` are
// real and take positions start ... start + n - 1.
struct Kv8Span {
  const int64_t* start;   // [1] or [batch], device
  int64_t start_stride;   // 0 or 1
  const int64_t* counts;  // null: every row is real
  int64_t counts_stride;
  int tokens;

  __device__ __forceinline__ int64_t first(int b) const { return start[b * start_stride]; }
  __device__ __forceinline__ int count(int b) const {
    if (counts == nullptr) return tokens;
    const int64_t n = counts[b * counts_stride];
    return n < 0 ? 0 : n > tokens ? tokens : (int)n;
  }
};

}  // namespace ml
