// Appending K and V rows to a KV cache held in 8 bits.
//
// A block of `block` consecutive positions of one kv head has one fp32 scale.
// With a = max |x| over the block's live values x,
//   scale = a / qmax,   code = round(x * qmax / a)      (qmax: 127, or 448 for e4m3)
// rounded half to even to an integer, or to the nearest e4m3 value.  x has at
// most 11 significant bits and qmax 7, so x * qmax is exact in fp32, the
// quotient is correctly rounded, and so it is a tie exactly where the true one
// is (two such ratios that differ do so by more than 2^-22 of their size): every
// code is the one the formula gives in exact
// arithmetic.  A block without a non-zero value has scale 0 and codes 0; a
// block holding an infinity or NaN gets that as its scale and codes 0, so it
// reads back as NaN.
//
// Each block is quantised from the values themselves, never from codes: the
// rows of the last two blocks written are also kept unquantised (`tail`, slot
// block & 1), and a call that continues a partly filled block takes its older
// rows from there.  The cache after any sequence of calls is therefore the
// cache after one call with all the rows.  Two slots, not one, so that a
// sequence can be taken back across a block border.  `held` says which block a
// slot has (negative, or no `held`: the one that is asked for).  A sequence taken
// back into a block that its slot no longer has gets the block's older rows from
// their codes, code * scale rounded to the rows' type: off by what their first
// quantisation was, and quantised to the same codes while the block's largest
// value stands (the rounding is less than half a step of the codes).
//
// A CTA takes one block of one kv head, K or V: its rows (new ones from the
// call, older ones from the tail) go to registers as 16-byte vectors, one
// block-wide maximum of |bits| (for bf16 and fp16 the order of the magnitudes
// with inf and NaN on top), then the codes.  Rows past the last new one are
// left as they were.  2 bytes are read and 1 written per element; the quotients
// take about as long as the bytes do (SM throughput 77% at 76% of the copy rate).
//
// Measured: 8 prompts of 4096 rows, 8 heads of dim 128 (205 MB) 41.5 us, 4.9
// TB/s (60 us where blocks of new rows had row checks as well, 75 us with 512
// threads, 64 with 128); one row for each of 64 sequences 8.2 us: two loads that
// follow one another (start, then the rows, the tail's from L2), the open block's
// rows read and its codes written whole, and a launch (7.0 with 128 threads, which
// the prompts pay for).  With `held` 3 to 4% more; one kernel for both had cost
// the calls without it as much.
#include "kv8.cuh"

#include <cuda_fp8.h>

namespace ml {
namespace {

constexpr int kThreads = 256;

struct AppendArgs {
  const void* src[2];       // k, v [B, Hkv, T, D] at element strides
  int64_t stride[2][3];     // batch, head, token
  uint8_t* codes[2];        // [B, Hkv, L, D]
  float* scale[2];          // [B, Hkv, L / block]
  void* tail[2];            // [B, Hkv, 2, block, D]
  int32_t* held[2];         // [B, Hkv, 2]: the slots' blocks; null: not known
  Kv8Span span;
  int heads, max_len, block;
};

template <typename T>
__device__ __forceinline__ float unpack(uint32_t w, int half) {
  T v;
  const uint16_t u = (uint16_t)(half ? w >> 16 : w);
  memcpy(&v, &u, 2);
  return to_f32(v);
}

// What a block's codes are computed with: x * mul / top, mul = qmax, both times
// a power of two that keeps the product finite; inv = 1 / top, rounded.
struct Divisor {
  float mul, top, inv;
};
// p / top, correctly rounded: the product with the rounded reciprocal, corrected
// by its remainder, which a fused multiply-add gives exactly (Markstein 1990).
__device__ __forceinline__ float quotient(const Divisor& d, float x) {
  const float p = x * d.mul, q = p * d.inv;
  return fmaf(fmaf(-q, d.top, p), d.inv, q);
}

// Eight codes of a 16-byte vector.
template <typename T, int FMT, bool TINY>
__device__ __forceinline__ uint2 quantise8(const uint4& x, const Divisor& d) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = unpack<T>(w[i / 2], i & 1);
    q[i] = TINY ? __fdiv_rn(v * d.mul, d.top) : quotient(d, v);
  }
  uint32_t out[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (FMT == ML_KV8_INT8) {
      uint32_t b[4];  // the code in the low byte: steps of 1 at 1.5 * 2^23
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = __float_as_uint(q[4 * i + j] + 12582912.f);
      out[i] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    } else {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(q[4 * i], q[4 * i + 1]),
                                                   __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(q[4 * i + 2], q[4 * i + 3]),
                                                   __NV_SATFINITE, __NV_E4M3);
      out[i] = lo | (hi << 16);
    }
  }
  return make_uint2(out[0], out[1]);
}

// Eight values that codes stand for, in the rows' type.
template <typename T, int FMT>
__device__ __forceinline__ uint4 dequantise8(uint2 codes, float scale) {
  uint32_t out[4];
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint32_t w = (i < 4 ? codes.x : codes.y) >> (8 * (i & 3));
    float x[2];
    if (FMT == ML_KV8_INT8) {
      x[0] = (float)(int8_t)(w & 0xff);
      x[1] = (float)(int8_t)(w >> 8 & 0xff);
    } else {
      const __half2 h = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)w, __NV_E4M3));
      x[0] = __low2float(h);
      x[1] = __high2float(h);
    }
    const T two[2] = {from_f32<T>(x[0] * scale), from_f32<T>(x[1] * scale)};
    memcpy(&out[i / 2], two, 4);
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

// Block `blk` of (b, h): rows [start, end) are new, older ones of the block
// come from the tail or, `lost`, from their codes.  NV 16-byte vectors per thread
// cover the block.  HELD: a.held is there.
template <typename T, int FMT, int D, int NV, bool HELD>
__device__ __forceinline__ void append_block(const AppendArgs& a, int which, int b, int h,
                                             int64_t blk, int64_t start, int64_t end, bool keep,
                                             bool lost, uint32_t* red) {
  constexpr int VPR = D / 8;  // vectors per row
  const int64_t base = blk * a.block;
  const int live = (int)min((int64_t)a.block, end - base);
  const int64_t bh = (int64_t)b * a.heads + h;
  // row 0 of the block, in the call's rows (that far before them, where start
  // lies inside the block)
  const int64_t pitch = a.stride[which][2];
  const T* src = static_cast<const T*>(a.src[which]) + b * a.stride[which][0] +
                 h * a.stride[which][1] + (base - start) * pitch;
  int fresh = (int)(start > base ? start - base : 0);  // first new row
  T* tail = static_cast<T*>(a.tail[which]) + (bh * 2 + (blk & 1)) * a.block * D;
  // a thread's vectors lie kThreads / VPR rows apart
  const int row0 = threadIdx.x / VPR, col = threadIdx.x % VPR * 8;
  constexpr int kApart = kThreads / VPR;
  const bool full = live == a.block && fresh == 0;  // most blocks of a prompt
  uint4 x[NV];
  if (full) {
    const T* from = src + row0 * pitch + col;
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i] = __ldcs(reinterpret_cast<const uint4*>(from + i * kApart * pitch));
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int row = row0 + i * kApart;
      x[i] = make_uint4(0, 0, 0, 0);
      if (row < live)
        x[i] = *reinterpret_cast<const uint4*>(row < fresh ? tail + row * D + col
                                                           : src + row * pitch + col);
    }
    if (HELD && lost) {
      const uint8_t* codes = a.codes[which] + (bh * a.max_len + base + row0) * D + col;
      const float scale = a.scale[which][bh * (a.max_len / a.block) + blk];
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (row0 + i * kApart < fresh)
          x[i] = dequantise8<T, FMT>(*reinterpret_cast<const uint2*>(codes + i * kApart * D), scale);
      fresh = 0;  // the slot gets them all
    }
  }
  uint32_t top2 = 0;  // |bits| maxima of even and odd elements
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    top2 = __vmaxu2(top2, x[i].x & 0x7fff7fffu);
    top2 = __vmaxu2(top2, x[i].y & 0x7fff7fffu);
    top2 = __vmaxu2(top2, x[i].z & 0x7fff7fffu);
    top2 = __vmaxu2(top2, x[i].w & 0x7fff7fffu);
  }
  uint32_t top = max(top2 & 0xffffu, top2 >> 16);
  top = __reduce_max_sync(0xffffffffu, top);
  __syncthreads();  // `red` may still be read by an earlier block of this CTA
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) top = max(top, red[i]);
  constexpr float qmax = FMT == ML_KV8_INT8 ? 127.f : 448.f;
  const float amax = unpack<T>(top, 0);
  if (threadIdx.x == 0) {
    a.scale[which][bh * (a.max_len / a.block) + blk] = __fdiv_rn(amax, qmax);
    if (HELD && keep) a.held[which][bh * 2 + (blk & 1)] = (int32_t)blk;
  }
  const bool finite = amax <= 3.4028235e38f && amax > 0.f;
  // x * qmax has to stay finite: values near the top of bf16 are halved 16
  // times on both sides of the division first (exact)
  const float down = amax > 1e30f ? 1.52587890625e-5f : 1.f;
  Divisor d;
  d.mul = qmax * down;
  d.top = amax * down;
  d.inv = __frcp_rn(d.top);
  uint8_t* codes = a.codes[which] + (bh * a.max_len + base + row0) * D + col;
  if (full && finite && d.top >= 1e-20f) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      *reinterpret_cast<uint2*>(codes + i * kApart * D) = quantise8<T, FMT, false>(x[i], d);
  } else {
    const bool tiny = d.top < 1e-20f;  // so small that remainders would be rounded
#pragma unroll 1
    for (int i = 0; i < NV; ++i) {
      if (row0 + i * kApart >= live) break;
      uint4 y = x[0];
#pragma unroll
      for (int j = 1; j < NV; ++j)
        if (j == i) y = x[j];
      uint2 q = make_uint2(0, 0);
      if (finite) q = tiny ? quantise8<T, FMT, true>(y, d) : quantise8<T, FMT, false>(y, d);
      *reinterpret_cast<uint2*>(codes + i * kApart * D) = q;
    }
  }
  if (keep) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int row = row0 + i * kApart;
      if (row >= fresh && row < live) *reinterpret_cast<uint4*>(tail + row * D + col) = x[i];
    }
  }
}

// Grid ({K, V} x kv heads, blocks a call can touch, batch): heads next to one
// another, as the projections leave them in a token's row.
template <typename T, int FMT, int D, int NV, bool HELD>
__global__ void __launch_bounds__(kThreads, NV <= 4 ? 6 : NV == 8 ? 4 : 2)
kv8_append_kernel(const __grid_constant__ AppendArgs a) {
  __shared__ uint32_t red[kThreads / 32];
  pdl_wait();
  pdl_release();
  const int b = blockIdx.z, h = blockIdx.x >> 1, which = blockIdx.x & 1;
  // the slots' blocks: in a call of few rows asked for together with start, not
  // after it; where there are many only by the CTA that needs to know
  int2 held = make_int2(-1, -1);
  const bool few = gridDim.y <= 2;
  if (HELD && few)
    held = *reinterpret_cast<const int2*>(a.held[which] + ((int64_t)b * a.heads + h) * 2);
  const int64_t start = a.span.first(b);
  if (start < 0 || start >= a.max_len) return;
  const int64_t end = min((int64_t)a.max_len, start + a.span.count(b));
  const int64_t first = start / a.block, last = (end - 1) / a.block;
  const int64_t blk = first + blockIdx.y;
  if (end <= start || blk > last) return;
  // The block that replaces the tail slot the first block still reads (the
  // last or the one before, of the first one's parity) is done by the same
  // CTA after it.
  int64_t after = -1;
  if (start % a.block != 0 && last - first >= 2) after = (last - first) % 2 == 0 ? last : last - 1;
  if (blk == after) return;
  bool lost = false;
  if (HELD && start > blk * a.block) {
    const int has = few ? (blk & 1 ? held.y : held.x)
                        : a.held[which][((int64_t)b * a.heads + h) * 2 + (blk & 1)];
    lost = has >= 0 && has != (int)blk;
  }
  append_block<T, FMT, D, NV, HELD>(a, which, b, h, blk, start, end, blk >= last - 1, lost, red);
  if (blk == first && after >= 0) {
    __syncthreads();  // every thread has its tail rows
    append_block<T, FMT, D, NV, HELD>(a, which, b, h, after, start, end, true, false, red);
  }
}

template <typename T, int FMT, int D, bool HELD>
int launch_append(const AppendArgs& a, dim3 grid, cudaStream_t st) {
  switch (a.block * (D / 8) / kThreads) {
#define ML_KV8_NV(NV_) \
  case NV_:                                                                               \
    ML_CHECK_CUDA(launch_pdl(kv8_append_kernel<T, FMT, D, NV_, HELD>, grid, dim3(kThreads), 0, \
                             st, a),                                                      \
                  "kv8_append");                                                          \
    return ML_OK;
    ML_KV8_NV(1) ML_KV8_NV(2) ML_KV8_NV(4) ML_KV8_NV(8) ML_KV8_NV(16)
#undef ML_KV8_NV
    default: set_error("kv8_append: unsupported block size"); return ML_ERR_INVALID_ARG;
  }
}

template <typename T, int FMT, bool HELD>
int launch_append_dim(const AppendArgs& a, int64_t dim, dim3 grid, cudaStream_t st) {
  if (dim == 64) return launch_append<T, FMT, 64, HELD>(a, grid, st);
  if (dim == 128) return launch_append<T, FMT, 128, HELD>(a, grid, st);
  return launch_append<T, FMT, 256, HELD>(a, grid, st);
}

template <typename T, int FMT>
int launch_append_held(const AppendArgs& a, int64_t dim, dim3 grid, cudaStream_t st) {
  return a.held[0] ? launch_append_dim<T, FMT, true>(a, dim, grid, st)
                   : launch_append_dim<T, FMT, false>(a, dim, grid, st);
}

}  // namespace
}  // namespace ml

using namespace ml;

extern "C" int ml_kv8_append(const ml_kv8_cache* cache, const void* k, const int64_t* k_strides,
                             const void* v, const int64_t* v_strides, int64_t tokens,
                             const int64_t* start, int64_t start_stride, const int64_t* counts,
                             int64_t counts_stride, void* stream) {
  int rc = kv8_check("kv8_append", cache);
  if (rc != ML_OK) return rc;
  ML_CHECK_ARG(tokens >= 0 && tokens < ((int64_t)1 << 30), "kv8_append: bad token count");
  if (cache->batch == 0 || tokens == 0) return ML_OK;
  ML_CHECK_ARG(k && v && start && k_strides && v_strides && cache->k_tail && cache->v_tail,
               "kv8_append: null pointer");
  ML_CHECK_ARG((start_stride == 0 || start_stride == 1) &&
                   (counts_stride == 0 || counts_stride == 1),
               "kv8_append: start / counts strides are 0 or 1");
  ML_CHECK_ARG(aligned16(k) && aligned16(v) && aligned16(cache->k_tail) && aligned16(cache->v_tail),
               "kv8_append: k, v and tail must be 16-byte aligned");
  ML_CHECK_ARG((cache->k_held == nullptr) == (cache->v_held == nullptr) &&
                   reinterpret_cast<uintptr_t>(cache->k_held) % 8 == 0 &&
                   reinterpret_cast<uintptr_t>(cache->v_held) % 8 == 0,
               "kv8_append: k_held and v_held are both there or neither, 8-byte aligned");
  for (int i = 0; i < 3; ++i)
    ML_CHECK_ARG(k_strides[i] % 8 == 0 && v_strides[i] % 8 == 0,
                 "kv8_append: k and v strides must be multiples of 8 elements");
  AppendArgs a;
  a.src[0] = k;
  a.src[1] = v;
  for (int i = 0; i < 3; ++i) {
    a.stride[0][i] = k_strides[i];
    a.stride[1][i] = v_strides[i];
  }
  a.codes[0] = static_cast<uint8_t*>(cache->k_codes);
  a.codes[1] = static_cast<uint8_t*>(cache->v_codes);
  a.scale[0] = cache->k_scale;
  a.scale[1] = cache->v_scale;
  a.tail[0] = cache->k_tail;
  a.tail[1] = cache->v_tail;
  a.held[0] = cache->k_held;
  a.held[1] = cache->v_held;
  a.span = {start, start_stride, counts, counts_stride, (int)tokens};
  a.heads = (int)cache->kv_heads;
  a.max_len = (int)cache->max_len;
  a.block = (int)cache->block;
  // an unaligned start can touch one block more than the rows fill
  const int64_t nblk = (tokens + cache->block - 2) / cache->block + 1;
  const int64_t most = cache->max_len / cache->block;
  ML_CHECK_ARG(most <= 65535 || nblk <= 65535, "kv8_append: too many blocks in one call");
  const dim3 grid((unsigned)(2 * cache->kv_heads), (unsigned)(nblk < most ? nblk : most),
                  (unsigned)cache->batch);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf = cache->dtype == ML_DTYPE_BF16;
  if (cache->format == ML_KV8_INT8)
    return bf ? launch_append_held<__nv_bfloat16, ML_KV8_INT8>(a, cache->head_dim, grid, st)
              : launch_append_held<__half, ML_KV8_INT8>(a, cache->head_dim, grid, st);
  return bf ? launch_append_held<__nv_bfloat16, ML_KV8_E4M3>(a, cache->head_dim, grid, st)
            : launch_append_held<__half, ML_KV8_E4M3>(a, cache->head_dim, grid, st);
}
