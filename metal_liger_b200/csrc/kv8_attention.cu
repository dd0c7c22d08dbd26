// Attention of one or a few query tokens per sequence over a KV cache held in
// 8 bits (kv8_append.cu writes it):
//   o[b, t, h] = sum_j softmax_j(scale * q[b, h, t] . k_j) v_j,  j <= start[b] + t,
// k_j = code * block scale, and the same for v.  A query with no position to
// see, or past its sequence's count, gives zeros.
//
// The codes are read once and bound the time: 2 D bytes per position and kv
// head against 4 D flops per query head.  So a warp converts 32 positions of
// K and V to fp16 in registers (exact: codes have at most 8 bits) and lets
// mma.sync do both products for up to 8 NT query rows of the kv head at a
// time: it takes the operands from the registers that the conversion leaves them
// in, where tcgen05 (positions as M, query rows as N) would have them written to
// shared memory or TMEM first.  For one token that is no bound (long caches run at
// 87% of the copy rate).  Many query tokens convert the codes again for every 8 or
// 16 rows and get a tenth of the tensor rate: 4 sequences, 256 tokens of 32 heads
// over 4000 positions take 391 us, 172 TFLOP/s.
//   S^T = K Q^T:  A = 16 positions x 16 dims, B = 16 dims x 8 query rows
//   O^T = V^T P^T: A = 16 dims x 16 positions, B = 16 positions x 8 query rows
// Any order of the summed index serves as long as both operands agree on it,
// so a lane takes 16 consecutive bytes of a row for four k-steps of S^T, and
// 16 consecutive dims of four positions for eight m-tiles of O^T: neither
// operand is transposed in memory.  P^T needs one movmatrix per 8 x 8.
//
// Queries enter as fp16 scaled by a power of two per row (bf16 and fp16 fit
// exactly down to 2^-14 of the row's largest value, and to 2^-25 of it below).
// Sums, statistics and outputs are fp32.  The scale of a V block enters the
// exponent: the output keeps its own running reference Mo = max(s + log2
// vscale), so weights 2^(s + log2 vscale - Mo) stay in [0, 1] however far the
// block scales lie apart.  For the second product they are rounded to fp16
// (what mma.sync takes beside the codes), times 2^15, which the output is
// divided by: the largest is 2^15 and fp16's normal range ends at 2^-29 of it,
// its smallest step at 2^-39, so a long tail behind one dominant position
// keeps its weight (the denominator counts it in fp32).  With the largest at 1,
// outputs that are the tail behind a position with 0.9999 of the weight were 1.1%
// off (8192 positions, dim 256); the factor is one addition per tile, and its
// time does not show (64 sequences of up to 8192: 102.6 us, 103.2 before).
//
// Work is divided evenly whatever the lengths: all 32-position tiles of all
// (sequence, kv head, row tile) segments form one flat list, each CTA takes an
// equal run of it and each of its warps an equal run of that, with a cp.async
// ring of its own (no barrier in the loop).  Segments that end up whole in a
// warp are written out; pieces are joined in shared memory, and those that
// cross CTAs by a second kernel, always in position order, so the result does
// not vary from run to run.
#include "kv8.cuh"

#include <cuda_fp8.h>
#include <type_traits>

namespace ml {
namespace {

constexpr int kTile = 32;  // positions per warp step
constexpr float kUpLog2 = 15.f;       // of the weights in fp16 ...
constexpr float kDown = 0x1p-15f;     // ... and back

struct AttnArgs {
  const void* q;            // [B, Hq, T, D] at element strides
  int64_t sq[3];
  const uint8_t* codes[2];  // [B, Hkv, L, D]
  const float* scale[2];    // [B, Hkv, L / block]
  Kv8Span span;
  int batch, kv_heads, group, rows, row_tiles, max_len, block;
  int tiles_log2;           // tiles per block
  float qk_scale;           // scale * log2(e)
  void* out;                // [B, T, Hq, D]
  float* part;              // [2 * gridDim.x] pieces; null: a CTA per segment
  int ctas;                 // CTAs that share the flat list
  int split;                // the join: CTAs of a segment
};

// A segment counts as this many tiles more than it has when the list is cut
// into equal runs: reading its queries and writing its rows take a warp about
// as long as one or two tiles (2 against 0: 32 segments of 8000 positions 21.1
// us / 22.3, 8 of 65000 33.7 / 34.9).
constexpr int kPad = 2;

// NW warps, each with a ring of units of 32 positions of K or of V.
template <int D, int NT, int NW>
struct Config {
  static constexpr int kUnit = kTile * D;            // bytes
  static constexpr int kUnits = D * NT >= 256 ? 24 * 1024 / kUnit : 12 * 1024 / kUnit;
  static constexpr int MT = D / 16;                  // m-tiles of O^T
  static constexpr int kRows = 8 * NT;
  static constexpr int kImage = NT * MT * 4 * 32;    // floats of a piece: acc ...
  static constexpr int kStats = 3 * kRows;           // ... and m, l, mo of its rows
  static constexpr int kPiece = kImage + kStats;     // in the workspace
  static constexpr int kCtaPieces = 2 + NW;          // its first and last, its warps' first ones
  static constexpr size_t smem() { return (size_t)NW * kUnits * kUnit; }
};
// Warps of a CTA of the list (two CTAs to an SM) ...
constexpr int list_warps(int D, int NT) { return D * NT >= 256 ? 4 : 8; }
// ... and of a CTA that has a segment to itself.
constexpr int segment_warps(int D) { return 2 * list_warps(D, 1); }

// ---------------------------------------------------------------------------
// The flat list of tiles
// ---------------------------------------------------------------------------

// Positions that query t of sequence b sees.  (start and count are loaded
// together: the second does not wait for the first.)
__device__ __forceinline__ int visible(const AttnArgs& a, int b, int t) {
  const int64_t start = a.span.first(b);
  const int count = a.span.count(b);
  const int64_t n = start + t + 1;
  return t >= count || n <= 0 ? 0 : n > a.max_len ? a.max_len : (int)n;
}
// Tiles of each segment of sequence b: up to its last real query's position,
// at least one (which then writes the zeros).
__device__ __forceinline__ int tiles_of(const AttnArgs& a, int b) {
  const int64_t start = a.span.first(b);
  const int count = a.span.count(b);
  const int64_t n = count > 0 ? start + count : 0;
  return n <= 0 ? 1 : ((n > a.max_len ? a.max_len : (int)n) + kTile - 1) / kTile;
}
__device__ __forceinline__ int tiles_per_cta(int total, int ctas, int warps) {
  const int even = (int)(((unsigned)total + ctas - 1) / (unsigned)ctas);
  return even > warps ? even : warps;
}

// One warp: the length of the list.
__device__ __forceinline__ int total_tiles(const AttnArgs& a, int lane) {
  const int per = a.kv_heads * a.row_tiles;
  int total = 0;
  for (int b = lane; b < a.batch; b += 32) total += (kPad + tiles_of(a, b)) * per;
  return (int)__reduce_add_sync(0xffffffffu, (unsigned)total);
}
// One warp: the sequence that holds flat position `u` (below the total), and
// what comes before it.
__device__ __forceinline__ int find_sequence(const AttnArgs& a, int u, int lane, int* before) {
  const int per = a.kv_heads * a.row_tiles;
  int base = 0;
  for (int b0 = 0;; b0 += 32) {
    const int n = b0 + lane < a.batch ? (kPad + tiles_of(a, b0 + lane)) * per : 0;
    int run = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += v;
    }
    const unsigned in = __ballot_sync(0xffffffffu, u < base + run);
    if (in) {
      const int f = __ffs(in) - 1;
      *before = base + __shfl_sync(0xffffffffu, run - n, f);
      return b0 + f;
    }
    base += __shfl_sync(0xffffffffu, run, 31);
  }
}

// ---------------------------------------------------------------------------
// Codes to fp16 pairs
// ---------------------------------------------------------------------------

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t s) {
  return __byte_perm(a, b, s);
}
// int8: 0x64xx is 1024 + xx in fp16; with the sign bit flipped xx = code + 128.
__device__ __forceinline__ uint32_t minus1152(uint32_t x) {
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t x) {
  uint32_t r;
  asm("{.reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, lo;}" : "=r"(r) : "r"(x));
  return r;
}
// The fp16 pairs of bytes (0, 1) and (2, 3).
template <int FMT>
__device__ __forceinline__ void pairs(uint32_t w, uint32_t& a, uint32_t& b) {
  if (FMT == ML_KV8_INT8) {
    w ^= 0x80808080u;
    a = minus1152(prmt(w, 0x64646464u, 0x4140));
    b = minus1152(prmt(w, 0x64646464u, 0x4342));
  } else {
    a = e4m3_pair(w);
    b = e4m3_pair(w >> 16);
  }
}

__device__ __forceinline__ void mma(float* c, const uint32_t* a, const uint32_t* b) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// 2^(x - ref), 0 where there is no reference yet
__device__ __forceinline__ float rel2(float x, float ref) {
  return ex2(x - (ref == -INFINITY ? 0.f : ref));
}

// Where chunk c (16 bytes) of row r of a tile lies, in chunks of the row: lanes
// that read together (K: two rows, four chunks each; V: rows 2t, one chunk of
// two dims groups) meet different banks.
template <int D>
__device__ __forceinline__ int k_chunk(int r, int c) { return D == 64 ? c : c ^ ((r & 1) << 2); }
template <int D>
__device__ __forceinline__ int v_chunk(int r, int c) {
  return D == 64 ? c ^ ((r >> 1) & 3) : c ^ (((r >> 1) & 3) << 1);
}

// ---------------------------------------------------------------------------
// A warp's running state of one segment
// ---------------------------------------------------------------------------

// acc[n][j]: O^T of dims 16 g + 2 j (+ 1 in [2], [3]) of each 128 dims (8 g +
// ... of 64) and rows 8 n + 2 t, + 1.  m, l, mo belong to those two rows; l is
// this lane's part.
template <int D, int NT>
struct State {
  float acc[NT][D / 16][4];
  float m[NT][2], l[NT][2], mo[NT][2];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][j][e] = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        m[n][c] = mo[n][c] = -INFINITY;
        l[n][c] = 0.f;
      }
    }
  }
  __device__ __forceinline__ void sum_l() {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], o);
  }
  // As an image [register][lane], and m, l, mo by row
  __device__ __forceinline__ void save(float* image, float* stats, int lane) const {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) image[((n * (D / 16) + j) * 4 + e) * 32 + lane] = acc[n][j][e];
    if (lane < 4) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int r = n * 8 + 2 * lane + c;
          stats[r] = m[n][c];
          stats[8 * NT + r] = l[n][c];
          stats[16 * NT + r] = mo[n][c];
        }
    }
  }
  template <typename T>
  __device__ __forceinline__ void write(const AttnArgs& a, int b, int kvh, int rt, int lane) const {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = (rt * NT + n) * 8 + 2 * t + c;
        if (r >= a.rows) continue;
        const int tok = r / a.group, h = kvh * a.group + r % a.group;
        const bool none = visible(a, b, tok) == 0;
        const float f = rel2(mo[n][c], m[n][c]) / l[n][c];
        T* dst = static_cast<T*>(a.out) +
                 (((int64_t)b * a.span.tokens + tok) * (a.kv_heads * a.group) + h) * D;
        constexpr int PER = D == 64 ? 8 : 16;  // consecutive dims of a lane
#pragma unroll
        for (int p = 0; p < D / 8 / PER; ++p) {
          uint32_t w[PER / 2];
#pragma unroll
          for (int j = 0; j < PER / 2; ++j) {
            const float lo = none ? 0.f : acc[n][p * 8 + j][c] * kDown * f;
            const float hi = none ? 0.f : acc[n][p * 8 + j][2 + c] * kDown * f;
            T two[2] = {from_f32<T>(lo), from_f32<T>(hi)};
            memcpy(&w[j], two, 4);
          }
#pragma unroll
          for (int v = 0; v < PER / 8; ++v)
            *reinterpret_cast<uint4*>(dst + p * 128 + g * PER + v * 8) =
                make_uint4(w[4 * v], w[4 * v + 1], w[4 * v + 2], w[4 * v + 3]);
        }
      }
  }
};

// Query rows of a segment as B fragments, and what the scores of this lane's
// two columns are multiplied with and how far they see.
template <int D, int NT>
struct Query {
  uint32_t frag[NT][D / 16][2];
  float mul[NT][2];
  int lim[NT][2];
  int lim_min, lim_max;  // over the rows that see anything

  // The rows as they are, into `frag` ...
  template <typename T>
  __device__ __forceinline__ void fetch(const AttnArgs& a, int b, int seg, int lane) {
    const int g = lane >> 2, t = lane & 3;
    const int kvh = seg / a.row_tiles, rt = seg % a.row_tiles;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = (rt * NT + n) * 8 + g;
      const int tok = r / a.group, h = kvh * a.group + r % a.group;
      const T* src = static_cast<const T*>(a.q) + b * a.sq[0] + h * a.sq[1] + tok * a.sq[2];
#pragma unroll
      for (int i = 0; i < D / 64; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint4 x = r < a.rows
                              ? *reinterpret_cast<const uint4*>(src + i * 64 + t * 16 + u * 8)
                              : make_uint4(0, 0, 0, 0);
          // words of 2 dims: k-steps 4 i + 2 u and the next, two registers each
          frag[n][4 * i + 2 * u][0] = x.x;
          frag[n][4 * i + 2 * u][1] = x.y;
          frag[n][4 * i + 2 * u + 1][0] = x.z;
          frag[n][4 * i + 2 * u + 1][1] = x.w;
        }
    }
  }
  // ... and scaled to fp16.
  template <typename T>
  __device__ __forceinline__ void finish(const AttnArgs& a, int b, int seg, int lane) {
    const int t = lane & 3;
    const int rt = seg % a.row_tiles;
    lim_min = a.max_len;
    lim_max = 0;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        top = __vmaxu2(top, __vmaxu2(frag[n][i][0] & 0x7fff7fffu, frag[n][i][1] & 0x7fff7fffu));
      top = max(top & 0xffffu, top >> 16);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      T tv;
      const uint16_t tb = (uint16_t)top;
      memcpy(&tv, &tb, 2);
      const float amax = to_f32(tv);
      // 2^-e with 2^e the largest power of two <= amax; 1 for zero, inf and NaN
      // rows, and below 2^-100, where the scores are nothing anyway
      const uint32_t e = __float_as_uint(amax) & 0x7f800000u;
      const bool finite = amax <= 3.4028235e38f;
      const float down = !finite || e <= 0x0d800000u ? 1.f
                         : e < 0x7f000000u           ? __uint_as_float(0x7f000000u - e)
                                                     : 0x1p-127f;
      const float up = !finite || e <= 0x0d800000u ? 1.f : __uint_as_float(e);
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          T two[2];
          memcpy(two, &frag[n][i][k], 4);
          frag[n][i][k] = half2_bits(to_f32(two[0]) * down, to_f32(two[1]) * down);
        }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        mul[n][c] = __shfl_sync(0xffffffffu, up, (2 * t + c) * 4) * a.qk_scale;
        const int rc = (rt * NT + n) * 8 + 2 * t + c;
        lim[n][c] = rc < a.rows ? visible(a, b, rc / a.group) : 0;
        if (lim[n][c] > 0) {
          lim_min = min(lim_min, lim[n][c]);
          lim_max = max(lim_max, lim[n][c]);
        }
      }
    }
    lim_min = __reduce_min_sync(0xffffffffu, lim_min);
    lim_max = __reduce_max_sync(0xffffffffu, lim_max);
  }
};

// Scores and probabilities of one tile of 32 positions, the first of them
// `pos`, as B fragments of the second product.
template <int D, int NT, int FMT, bool MASK>
__device__ __forceinline__ void score_step(State<D, NT>& st, const Query<D, NT>& q,
                                           const uint8_t* ks, float k_scale, float v_scale,
                                           uint32_t (&p)[2][NT][2], int pos, int lane) {
  const int g = lane >> 2, t = lane & 3;
  float s[2][NT][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][n][e] = 0.f;
#pragma unroll
  for (int h = 0; h < D / 64; ++h) {
    uint4 k[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int r = i * 16 + u * 8 + g;
        k[i][u] = *reinterpret_cast<const uint4*>(ks + r * D + k_chunk<D>(r, h * 4 + t) * 16);
      }
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t f[4];
        const uint32_t lo = w == 0 ? k[i][0].x : w == 1 ? k[i][0].y : w == 2 ? k[i][0].z : k[i][0].w;
        const uint32_t hi = w == 0 ? k[i][1].x : w == 1 ? k[i][1].y : w == 2 ? k[i][1].z : k[i][1].w;
        pairs<FMT>(lo, f[0], f[2]);
        pairs<FMT>(hi, f[1], f[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma(s[i][n], f, q.frag[n][h * 4 + w]);
      }
  }
  const float lv = __log2f(v_scale);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float top[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float f = k_scale * q.mul[n][c];
      top[c] = -INFINITY;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float& x = s[i][n][2 * u + c];
          x *= f;
          if (MASK && pos + i * 16 + u * 8 + g >= q.lim[n][c]) x = -INFINITY;
          top[c] = fmaxf(top[c], x);
        }
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], o));
    }
    const bool more = top[0] > st.m[n][0] || top[1] > st.m[n][1] || top[0] + lv > st.mo[n][0] ||
                      top[1] + lv > st.mo[n][1];
    if (__any_sync(0xffffffffu, more)) {
      float ka[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float nm = fmaxf(st.m[n][c], top[c]), no = fmaxf(st.mo[n][c], top[c] + lv);
        st.l[n][c] *= rel2(st.m[n][c], nm);
        ka[c] = rel2(st.mo[n][c], no);
        st.m[n][c] = nm;
        st.mo[n][c] = no;
      }
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) st.acc[n][j][e] *= ka[e & 1];
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float m = st.m[n][c] == -INFINITY ? 0.f : st.m[n][c];
      const float o = lv + kUpLog2 - (st.mo[n][c] == -INFINITY ? 0.f : st.mo[n][c]);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float& x = s[i][n][2 * u + c];
          const bool off = MASK && x == -INFINITY;
          st.l[n][c] += off ? 0.f : ex2(x - m);
          x = off ? 0.f : ex2(x + o);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int u = 0; u < 2; ++u)
        p[i][n][u] = transpose8(half2_bits(s[i][n][2 * u], s[i][n][2 * u + 1]));
  }
}

// Adds the tile's V rows, weighted.  A lane holds 16 (8 of 64) consecutive dims
// of each 128.
template <int D, int NT, int FMT, bool MASK>
__device__ __forceinline__ void value_step(State<D, NT>& st, const Query<D, NT>& q,
                                           const uint8_t* vs, const uint32_t (&p)[2][NT][2],
                                           int pos, int lane) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int h = 0; h < (D + 127) / 128; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      constexpr int W = D == 64 ? 2 : 4;  // words
      uint32_t v[4][W];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int r = i * 16 + 2 * t + (u & 1) + (u >> 1) * 8;
        if (D == 64) {
          const uint2 x = *reinterpret_cast<const uint2*>(vs + r * D + v_chunk<D>(r, g >> 1) * 16 +
                                                          (g & 1) * 8);
          v[u][0] = x.x;
          v[u][1] = x.y;
        } else {
          const uint4 x = *reinterpret_cast<const uint4*>(vs + r * D + (v_chunk<D>(r, g) + h * 8) * 16);
          v[u][0] = x.x;
          v[u][1] = x.y;
          v[u][W - 2] = x.z;
          v[u][W - 1] = x.w;
        }
        // what lies past the last visible position may be any bytes
        if (MASK && pos + r >= q.lim_max) {
#pragma unroll
          for (int w = 0; w < W; ++w) v[u][w] = 0;
        }
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
        // tokens interleaved per dim: (dims 0, 1) and (2, 3) of the word
        uint32_t f[2][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t x = prmt(v[2 * half][w], v[2 * half + 1][w], 0x5140);
          const uint32_t y = prmt(v[2 * half][w], v[2 * half + 1][w], 0x7362);
          pairs<FMT>(x, f[0][2 * half], f[0][2 * half + 1]);
          pairs<FMT>(y, f[1][2 * half], f[1][2 * half + 1]);
        }
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int n = 0; n < NT; ++n) mma(st.acc[n][h * 8 + 2 * w + y], f[y], p[i][n]);
      }
    }
}

// Position `u` in the flat list: tile `tile` of `tiles` of segment `seg` (kv
// head x row tile) of sequence b.
struct Cursor {
  int u, b, seg, tile, tiles;

  // The first tile at or after u, which lies `offset` into sequence b_.
  __device__ __forceinline__ void set(const AttnArgs& a, int b_, int offset) {
    b = b_;
    tiles = tiles_of(a, b);
    const unsigned per = tiles + kPad;
    seg = (int)((unsigned)offset / per);
    const int x = offset - seg * (int)per;
    u += x < kPad ? kPad - x : 0;
    tile = x < kPad ? 0 : x - kPad;
  }
  // true where another segment begins
  __device__ __forceinline__ bool next(const AttnArgs& a) {
    ++u;
    if (++tile < tiles) return false;
    u += kPad;
    tile = 0;
    if (++seg == a.kv_heads * a.row_tiles) {
      seg = 0;
      if (++b < a.batch) tiles = tiles_of(a, b);
    }
    return true;
  }
};

// A cursor with this lane's place in the cache.
template <int D>
struct Loader {
  Cursor c;
  int64_t off;  // of its 16 bytes of the tile's first rows
  int scale;    // index of the segment's first block

  __device__ __forceinline__ void point(const AttnArgs& a, int lane) {
    const int bh = c.b * a.kv_heads + c.seg / a.row_tiles;
    off = ((int64_t)bh * a.max_len + (int64_t)c.tile * kTile) * D + lane * 16;
    scale = bh * (a.max_len / a.block);
  }
  __device__ __forceinline__ void next(const AttnArgs& a, int lane) {
    if (c.next(a)) {
      if (c.b < a.batch) point(a, lane);
    } else {
      off += kTile * D;
    }
  }
};

// The K unit of a tile brings the tile's two scales along.
template <int D, int WHICH>
__device__ __forceinline__ void load_unit(const AttnArgs& a, const Loader<D>& from, uint32_t dst,
                                          uint32_t scales, int lane) {
  constexpr int CPR = D / 16;
  constexpr int RPP = 32 / CPR;  // rows per pass of the warp
  const int r0 = lane / CPR, ch = lane % CPR;
  const uint8_t* src = a.codes[WHICH] + from.off;
#pragma unroll
  for (int i = 0; i < kTile / RPP; ++i) {
    const int r = r0 + i * RPP;
    const int at = WHICH == 0 ? k_chunk<D>(r, ch) : v_chunk<D>(r, ch);
    cp_async16(dst + r * D + at * 16, src + i * 512);
  }
  if (WHICH == 0 && lane < 2)
    cp_async4(scales + lane * 4,
              (lane ? a.scale[1] : a.scale[0]) + from.scale + (from.c.tile >> a.tiles_log2));
}

// A piece of a segment that its warp did not see whole.
struct Piece {
  int b, seg, lo, hi, tiles;  // tiles [lo, hi) of `tiles`; hi = 0: none
};

// Four values of a joined image, of one lane and m-tile: to the output ...
template <typename T, int D, int NT>
__device__ __forceinline__ void write_item(const AttnArgs& a, int b, int seg, int item,
                                           const float* o) {
  using C = Config<D, NT, 8>;
  const int l = item & 31, j = (item >> 5) % C::MT, n = (item >> 5) / C::MT;
  const int t = l & 3, g = l >> 2;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int r = (seg % a.row_tiles) * C::kRows + n * 8 + 2 * t + c;
    if (r >= a.rows) continue;
    const int tok = r / a.group, h = (seg / a.row_tiles) * a.group + r % a.group;
    constexpr int PER = D == 64 ? 8 : 16;  // consecutive dims of a lane
    T* dst = static_cast<T*>(a.out) +
             (((int64_t)b * a.span.tokens + tok) * (a.kv_heads * a.group) + h) * D +
             (j * 2 / PER) * 128 + g * PER + j * 2 % PER;
    T two[2] = {from_f32<T>(o[c] * kDown), from_f32<T>(o[2 + c] * kDown)};
    uint32_t w;
    memcpy(&w, two, 4);
    *reinterpret_cast<uint32_t*>(dst) = w;
  }
}
// ... from the images of every STEP-th piece of [from, to), each times its
// row's factor (negative: the row sees nothing, its images hold anything).
template <int D, int NT, int STEP, typename Image>
__device__ __forceinline__ void sum_item(int item, int from, int to, const Image& image,
                                         const float (*factor)[8 * NT], float* o) {
  using C = Config<D, NT, 8>;
  const int l = item & 31, n = (item >> 5) / C::MT, r = n * 8 + 2 * (l & 3);
  o[0] = o[1] = o[2] = o[3] = 0.f;
#pragma unroll 4
  for (int i = from; i < to; i += STEP) {
    const float* src = image(i) + (item >> 5) * 128 + l;
    const float2 k = *reinterpret_cast<const float2*>(&factor[i][r]);
    const float x[4] = {src[0], src[32], src[64], src[96]};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float f = e & 1 ? k.y : k.x;
      o[e] += f < 0.f ? 0.f : x[e] * f;  // a zero factor still passes NaN on
    }
  }
}

// A segment with pieces in this CTA: entries [from, to) of the list of pieces.
struct Run {
  int from, to, b, seg;
  bool whole;  // all of it is here
  bool begun;  // it began in an earlier CTA
};

template <typename T, int FMT, int D, int NT, int NW>
__global__ void __launch_bounds__(32 * NW, NW == list_warps(D, NT) ? 2 : 1)
kv8_attention_kernel(const __grid_constant__ AttnArgs a) {
  using C = Config<D, NT, NW>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Piece pieces[2 * NW];
  __shared__ float stats[2 * NW][C::kStats];
  __shared__ __align__(8) float factor[2 * NW][C::kRows];
  __shared__ Run runs[2 * NW];
  __shared__ int entry[2 * NW];  // of the list, by rank: 2 * warp + slot
  __shared__ float scales[NW][C::kUnits][2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint8_t* ring = smem + (size_t)warp * C::kUnits * C::kUnit;
  float* scratch = a.part + (int64_t)blockIdx.x * C::kCtaPieces * C::kPiece;

  pdl_wait();
  pdl_release();
  // this warp's run of the list: from `cur` up to `hi`
  int hi;
  Cursor cur;
  if (a.part == nullptr) {  // a CTA per segment
    const int segs = a.kv_heads * a.row_tiles;
    cur.b = blockIdx.x / segs;
    cur.seg = blockIdx.x % segs;
    cur.tiles = tiles_of(a, cur.b);
    const int sub = (cur.tiles + NW - 1) / NW;
    cur.u = cur.tile = min(warp * sub, cur.tiles);
    hi = min(cur.u + sub, cur.tiles);
  } else {
    const int total = total_tiles(a, lane);
    const int per_cta = tiles_per_cta(total, a.ctas, NW), sub = (per_cta + NW - 1) / NW;
    const int cta_lo = (int)min((int64_t)blockIdx.x * per_cta, (int64_t)total);
    const int cta_hi = min(total - cta_lo, per_cta) + cta_lo;
    cur.u = min(cta_lo + warp * sub, cta_hi);
    hi = min(cur.u + sub, cta_hi);
    if (cur.u < hi) {
      int before;
      const int b = find_sequence(a, cur.u, lane, &before);
      cur.set(a, b, cur.u - before);
    }
  }

  if (lane < 2) pieces[2 * warp + lane].hi = 0;
  __syncwarp();
  if (cur.u < hi) {
    const uint32_t ring_u = smem_u32_of(ring), scales_u = smem_u32_of(&scales[warp][0][0]);
    State<D, NT> st;
    Query<D, NT> q;
    // the queries first: behind the first units they would wait for those
    q.template fetch<T>(a, cur.b, cur.seg, lane);
    Loader<D> ahead;
    ahead.c = cur;
    ahead.point(a, lane);
    // units are K and V of the tiles in turn
    int to = 0;
    bool odd = false;
    auto load_next = [&] {
      if (ahead.c.u < hi) {
        if (odd) {
          load_unit<D, 1>(a, ahead, ring_u + to * C::kUnit, 0, lane);
          ahead.next(a, lane);
        } else {
          load_unit<D, 0>(a, ahead, ring_u + to * C::kUnit, scales_u + to * 8, lane);
        }
        odd = !odd;
        to = to == C::kUnits - 1 ? 0 : to + 1;
      }
      cp_commit();
    };
#pragma unroll 1
    for (int i = 0; i < C::kUnits - 1; ++i) load_next();
    int at = 0, piece_lo = cur.tile;
    q.template finish<T>(a, cur.b, cur.seg, lane);
    st.clear();
#pragma unroll 1
    while (true) {
      const int pos = cur.tile * kTile;
      const bool open = pos + kTile <= q.lim_min;
      uint32_t p[2][NT][2];
      cp_wait<C::kUnits - 2>();
      __syncwarp();
      load_next();  // into the unit read last, which every lane is done with
      const float k_scale = scales[warp][at][0], v_scale = scales[warp][at][1];
      if (open)
        score_step<D, NT, FMT, false>(st, q, ring + at * C::kUnit, k_scale, v_scale, p, pos, lane);
      else
        score_step<D, NT, FMT, true>(st, q, ring + at * C::kUnit, k_scale, v_scale, p, pos, lane);
      at = at == C::kUnits - 1 ? 0 : at + 1;
      cp_wait<C::kUnits - 2>();
      __syncwarp();
      load_next();
      if (open)
        value_step<D, NT, FMT, false>(st, q, ring + at * C::kUnit, p, pos, lane);
      else
        value_step<D, NT, FMT, true>(st, q, ring + at * C::kUnit, p, pos, lane);
      at = at == C::kUnits - 1 ? 0 : at + 1;

      const Cursor was = cur;
      const bool ends = cur.next(a), last = cur.u >= hi;
      if (!ends && !last) continue;
      st.sum_l();
      if (ends && piece_lo == 0) {
        st.template write<T>(a, was.b, was.seg / a.row_tiles, was.seg % a.row_tiles, lane);
      } else {
        // the run's last piece takes the ring, which nothing uses any more; a
        // first one before other segments goes to the workspace
        const int slot = last ? 1 : 0;
        if (last) {
          cp_wait<0>();
          __syncwarp();
        }
        st.save(last ? reinterpret_cast<float*>(ring) : scratch + (2 + warp) * C::kPiece,
                stats[2 * warp + slot], lane);
        if (lane == 0)
          pieces[2 * warp + slot] = {was.b, was.seg, piece_lo, was.tile + 1, was.tiles};
      }
      if (last) break;
      q.template fetch<T>(a, cur.b, cur.seg, lane);
      q.template finish<T>(a, cur.b, cur.seg, lane);
      st.clear();
      piece_lo = cur.tile;
    }
  }
  cp_wait<0>();
  __syncthreads();

  // Join the pieces: those of one segment follow one another.  A group of a
  // lane per entry finds the runs; then a group per row makes the entries'
  // factors with reductions inside the runs.
  constexpr int E = 2 * NW, kGroups = 32 / E;
  static_assert(E <= 32, "a lane per entry");
  const int e = lane % E, base = lane - e;
  constexpr unsigned kEntries = E == 32 ? 0xffffffffu : (1u << E) - 1;
  const Piece mine = pieces[e];
  const unsigned valid = __ballot_sync(0xffffffffu, mine.hi > 0) & kEntries;
  if (valid == 0) return;
  const unsigned below = (1u << e) - 1, upto = below | (1u << e);
  const int prev = base + ((valid & below) ? 31 - __clz(valid & below) : e);
  const int prev_b = __shfl_sync(0xffffffffu, mine.b, prev);
  const int prev_seg = __shfl_sync(0xffffffffu, mine.seg, prev);
  const bool on = mine.hi > 0;
  const bool starts = on && ((valid & below) == 0 || prev_b != mine.b || prev_seg != mine.seg);
  const unsigned head = __ballot_sync(0xffffffffu, starts) & kEntries;
  const int my_head = base + ((head & upto) ? 31 - __clz(head & upto) : e);
  const int end = (head & ~upto) ? __ffs(head & ~upto) - 1 : E;  // of this entry's run
  const unsigned in_run = valid & (end == 32 ? 0xffffffffu : (1u << end) - 1);
  const int head_lo = __shfl_sync(0xffffffffu, mine.lo, my_head);
  const int last_hi = __shfl_sync(0xffffffffu, mine.hi, base + (in_run ? 31 - __clz(in_run) : 0));
  const bool whole = head_lo == 0 && last_hi == mine.tiles;
  const int rank = __popc(valid & below);
  if (threadIdx.x < E && on) {
    entry[rank] = e;
    if (starts)
      runs[__popc(head & below)] = {rank, __popc(in_run), mine.b, mine.seg, whole, mine.lo > 0};
  }
#pragma unroll 1
  for (int r0 = warp * kGroups; r0 < C::kRows; r0 += NW * kGroups) {
    const int r = r0 + lane / E;
    const float m = on ? stats[e][r] : -INFINITY;
    const float l = on ? stats[e][C::kRows + r] : 0.f;
    const float mo = on ? stats[e][2 * C::kRows + r] : -INFINITY;
    float M = m, MO = mo;
#pragma unroll
    for (int o = 1; o < E; o <<= 1) {
      const float x = __shfl_down_sync(0xffffffffu, M, o), y = __shfl_down_sync(0xffffffffu, MO, o);
      if (e + o < end) {
        M = fmaxf(M, x);
        MO = fmaxf(MO, y);
      }
    }
    M = __shfl_sync(0xffffffffu, M, my_head);
    MO = __shfl_sync(0xffffffffu, MO, my_head);
    float L = on ? l * rel2(m, M) : 0.f;
#pragma unroll
    for (int o = 1; o < E; o <<= 1) {
      const float x = __shfl_down_sync(0xffffffffu, L, o);
      if (e + o < end) L += x;
    }
    L = __shfl_sync(0xffffffffu, L, my_head);
    if (on) {
      const int row = (mine.seg % a.row_tiles) * C::kRows + r;
      const bool sees = row < a.rows && visible(a, mine.b, row / a.group) > 0;
      factor[rank][r] = sees ? rel2(mo, MO) * (whole ? rel2(MO, M) / L : 1.f) : -1.f;
      if (starts && !whole) {
        // place 0 for a segment that began in an earlier CTA, 1 for one that
        // goes on in the next
        float* to = scratch + (mine.lo > 0 ? 0 : 1) * C::kPiece + C::kImage;
        to[r] = M;
        to[C::kRows + r] = L;
        to[2 * C::kRows + r] = MO;
      }
    }
  }
  __syncthreads();
  auto image = [&](int i) {
    const int e = entry[i];
    return e & 1 ? reinterpret_cast<const float*>(smem + (size_t)(e >> 1) * C::kUnits * C::kUnit)
                 : static_cast<const float*>(scratch + (2 + (e >> 1)) * C::kPiece);
  };
  constexpr int kItems = C::kImage / 4;
  for (int x = threadIdx.x; x < __popc(head) * kItems; x += 32 * NW) {
    const Run& run = runs[x / kItems];
    const int item = x % kItems;
    float o[4];
    sum_item<D, NT, 1>(item, run.from, run.to, image, factor, o);
    if (run.whole) {
      write_item<T, D, NT>(a, run.b, run.seg, item, o);
    } else {
      float* to = scratch + (run.begun ? 0 : 1) * C::kPiece + (item >> 5) * 128 + (item & 31);
#pragma unroll
      for (int e = 0; e < 4; ++e) to[e * 32] = o[e];
    }
  }
}

// Joins the segments that cross CTAs, `split` CTAs each.  The pieces' statistics
// become one factor per piece and row (a row per warp, lanes over the pieces);
// then the threads take the CTA's items (four values of every piece), in groups
// where there are fewer items than threads: a group takes every group-count-th
// piece, so that few loads follow one another, and the groups' sums are added in
// order.
constexpr int kJoinThreads = 256;
constexpr int kMaxCtas = 640;  // of the list

template <typename T, int D, int NT, int NW>
__global__ void __launch_bounds__(kJoinThreads)
kv8_attention_join(const __grid_constant__ AttnArgs a) {
  using C = Config<D, NT, NW>;
  __shared__ __align__(8) float factor[kMaxCtas][C::kRows];
  __shared__ float4 sums[kJoinThreads];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per_b = a.kv_heads * a.row_tiles;
  const int segment = blockIdx.x / a.split;
  const int b = segment / per_b, seg = segment % per_b;
  // start and counts may be read before the wait: this grid starts when the
  // first kernel's CTAs have passed theirs, and that kernel writes neither
  int before = 0, total = 0;  // of the list, before the segment's sequence and in all
  for (int i = lane; i < a.batch; i += 32) {
    const int n = (kPad + tiles_of(a, i)) * per_b;
    total += n;
    if (i < b) before += n;
  }
  before = (int)__reduce_add_sync(0xffffffffu, (unsigned)before);
  total = (int)__reduce_add_sync(0xffffffffu, (unsigned)total);
  const int per_cta = tiles_per_cta(total, a.ctas, NW);
  const int n = tiles_of(a, b);
  const int lo = before + seg * (n + kPad) + kPad;  // its first tile
  const int c0 = lo / per_cta;
  const int count = (lo + n - 1) / per_cta - c0 + 1;
  const int rt = seg % a.row_tiles;
  pdl_wait();
  pdl_release();
  if (count == 1) return;  // whole in one CTA, which wrote it
  auto piece = [&](int i) -> const float* {
    return a.part + ((int64_t)(c0 + i) * C::kCtaPieces + (i == 0 ? 1 : 0)) * C::kPiece;
  };
#pragma unroll
  for (int r = warp; r < C::kRows; r += kJoinThreads / 32) {
    const bool sees = rt * C::kRows + r < a.rows && visible(a, b, (rt * C::kRows + r) / a.group) > 0;
    float M = -INFINITY, MO = -INFINITY, L = 0.f;
    float m = -INFINITY, l = 0.f, mo = -INFINITY;  // of this lane's first piece
    if (lane < count) {
      const float* st = piece(lane) + C::kImage + r;
      m = st[0];
      l = st[C::kRows];
      mo = st[2 * C::kRows];
    }
    M = m;
    MO = mo;
    for (int i = lane + 32; i < count; i += 32) {
      const float* st = piece(i) + C::kImage + r;
      M = fmaxf(M, st[0]);
      MO = fmaxf(MO, st[2 * C::kRows]);
    }
    M = warp_max(M);
    MO = warp_max(MO);
    L = l * rel2(m, M);
    for (int i = lane + 32; i < count; i += 32) {
      const float* st = piece(i) + C::kImage + r;
      L += st[C::kRows] * rel2(st[0], M);
    }
    L = warp_sum(L);
    const float f = rel2(MO, M) / L;
    for (int i = lane; i < count; i += 32) {
      const float x = i == lane ? mo : piece(i)[C::kImage + 2 * C::kRows + r];
      factor[i][r] = sees ? rel2(x, MO) * f : -1.f;
    }
  }
  __syncthreads();
  const int items = C::kImage / 4 / a.split, first = (int)(blockIdx.x % a.split) * items;
  auto join = [&](auto groups) {
    constexpr int G = decltype(groups)::value;
    const int group = threadIdx.x / (kJoinThreads / G);
    for (int x = threadIdx.x % (kJoinThreads / G); x < items; x += kJoinThreads) {
      float o[4];
      sum_item<D, NT, G>(first + x, group, count, piece, factor, o);
      if constexpr (G > 1) {  // items = kJoinThreads / G: one round
        sums[threadIdx.x] = make_float4(o[0], o[1], o[2], o[3]);
        __syncthreads();
        if (group > 0) return;
#pragma unroll
        for (int i = 1; i < G; ++i) {
          const float4 y = sums[i * (kJoinThreads / G) + x];
          o[0] += y.x;
          o[1] += y.y;
          o[2] += y.z;
          o[3] += y.w;
        }
      }
      write_item<T, D, NT>(a, b, seg, first + x, o);
    }
  };
  if (items >= kJoinThreads) join(std::integral_constant<int, 1>());
  else if (items == kJoinThreads / 2) join(std::integral_constant<int, 2>());
  else if (items == kJoinThreads / 4) join(std::integral_constant<int, 4>());
  else join(std::integral_constant<int, 8>());  // 32: the least that the host's rule gives
}

// Query rows per tile: 8 NT.  Sixteen rows read the codes once instead of twice,
// eight leave room for twice the warps, which gives more where a warp has few
// tiles.  Eight against sixteen, 16 rows a kv head of dim 128: 4 x 8 heads of
// 1500 positions (3000 tiles of eight rows) 15.3 us / 17.8, 4 x 8 of 8000 (16000)
// 28.8 / 29.7, 16 x 8 of 8000 (64000) 87 / 78; dim 64, 16 x 8 of 8000 60 / 48.
inline int n_tiles(const ml_kv8_cache* c, int64_t rows) {
  const int64_t tiles = c->batch * c->kv_heads * ((rows + 7) / 8) * (c->max_len / kTile);
  return rows > 8 && c->head_dim != 256 && tiles >= 128 * (int64_t)num_sms() ? 2 : 1;
}

// Short caches go a CTA to a segment, in one launch, where these are one wave
// (one such CTA fills an SM).  One launch against the list, 64 segments: 250
// positions 7.3 us / 13.1, 1000 11.6 / 13.7, 2000 16.1 / 16.1; 8 segments: 1000
// 11.4 / 10.9, 2000 15.7 / 11.4; 256 segments: 250 14.5 / 14.5, 500 17.8 / 16.6.
// The rule goes by the capacity, since only the device knows how far a cache is
// filled: of 4096 positions, 250 of them filled, 64 segments take the list, 13.2
// us, where a cache of 256 takes one launch, 7.2 (8 segments 10.7, 6.8); 1000
// filled, 13.7 and 11.7 (10.9, 11.3).
constexpr int64_t kOneLaunchLen = 1024;

struct Plan {
  int nt, row_tiles, ctas;
  size_t workspace;  // 0: one launch
};
inline Plan plan_of(const ml_kv8_cache* c, int64_t rows) {
  Plan p;
  p.nt = n_tiles(c, rows);
  p.row_tiles = (int)((rows + 8 * p.nt - 1) / (8 * p.nt));
  p.ctas = 2 * num_sms() < kMaxCtas ? 2 * num_sms() : kMaxCtas;
  const int64_t segs = c->batch * c->kv_heads * p.row_tiles;
  if (p.nt == 1 && c->max_len <= kOneLaunchLen && segs <= num_sms()) {
    p.workspace = 0;
    return p;
  }
  const int warps = list_warps((int)c->head_dim, p.nt);
  const int64_t piece = p.nt * c->head_dim / 16 * 4 * 32 + 3 * 8 * p.nt;
  p.workspace = (size_t)p.ctas * (2 + warps) * piece * sizeof(float);
  return p;
}

template <typename T, int FMT, int D, int NT, int NW>
int launch_kernel(const AttnArgs& a, int64_t grid, cudaStream_t st) {
  using C = Config<D, NT, NW>;
  auto kernel = kv8_attention_kernel<T, FMT, D, NT, NW>;
  static PerDevice<cudaError_t> attr;
  ML_CHECK_CUDA(attr.get([&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)C::smem());
  }), "kv8_attention");
  ML_CHECK_CUDA(launch_pdl(kernel, dim3((unsigned)grid), dim3(32 * NW), C::smem(), st, a),
                "kv8_attention");
  return ML_OK;
}

template <typename T, int FMT, int D, int NT>
int launch(AttnArgs a, cudaStream_t st) {
  const int64_t segs = (int64_t)a.batch * a.kv_heads * a.row_tiles;
  // (below 2^31 by more than what a warp's `first tile + share` can pass the total
  // by: the CTAs' shares are rounded up to whole tiles, and so are the warps')
  ML_CHECK_ARG(segs * (a.max_len / kTile + kPad) < ((int64_t)1 << 31) - ((int64_t)1 << 17),
               "kv8_attention: too many query rows for this cache in one call");
  if constexpr (NT == 1) {
    if (a.part == nullptr) return launch_kernel<T, FMT, D, 1, segment_warps(D)>(a, segs, st);
  }
  constexpr int NW = list_warps(D, NT);
  const int rc = launch_kernel<T, FMT, D, NT, NW>(a, a.ctas, st);
  if (rc != ML_OK) return rc;
  // as many CTAs as four to an SM, each with 32 items or more.  Against all or
  // nothing (32 items a CTA, or a CTA to a segment): 64 segments of 4000 positions
  // 23.5 for 27 us, 8 of 65536 34.9 for 34.6
  a.split = 1;
  while (a.split * 2 <= Config<D, NT, NW>::kImage / 4 / 32 && segs * a.split * 2 <= 4 * num_sms())
    a.split *= 2;
  ML_CHECK_CUDA(launch_pdl(kv8_attention_join<T, D, NT, NW>, dim3((unsigned)(segs * a.split)),
                           dim3(kJoinThreads), 0, st, a),
                "kv8_attention(join)");
  return ML_OK;
}

template <typename T, int FMT>
int launch_dim(const AttnArgs& a, int64_t dim, int nt, cudaStream_t st) {
  if (dim == 64) return nt == 1 ? launch<T, FMT, 64, 1>(a, st) : launch<T, FMT, 64, 2>(a, st);
  if (dim == 128) return nt == 1 ? launch<T, FMT, 128, 1>(a, st) : launch<T, FMT, 128, 2>(a, st);
  return launch<T, FMT, 256, 1>(a, st);
}

}  // namespace
}  // namespace ml

using namespace ml;

extern "C" size_t ml_kv8_attention_workspace_bytes(const ml_kv8_cache* cache, int64_t q_heads,
                                                   int64_t tokens) {
  if (cache == nullptr || cache->kv_heads <= 0 || cache->batch <= 0 || tokens <= 0 || q_heads <= 0)
    return 0;
  return plan_of(cache, q_heads / cache->kv_heads * tokens).workspace;
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
  const int64_t rows = q_heads / cache->kv_heads * tokens;
  ML_CHECK_ARG(rows < ((int64_t)1 << 30), "kv8_attention: too many rows");
  const Plan plan = plan_of(cache, rows);
  ML_CHECK_ARG(plan.workspace == 0 ||
                   (workspace && aligned16(workspace) && workspace_bytes >= plan.workspace),
               "kv8_attention: workspace too small");
  AttnArgs a;
  a.q = q;
  for (int i = 0; i < 3; ++i) a.sq[i] = q_strides[i];
  a.codes[0] = static_cast<const uint8_t*>(cache->k_codes);
  a.codes[1] = static_cast<const uint8_t*>(cache->v_codes);
  a.scale[0] = cache->k_scale;
  a.scale[1] = cache->v_scale;
  a.span = {start, start_stride, counts, counts_stride, (int)tokens};
  a.batch = (int)cache->batch;
  a.kv_heads = (int)cache->kv_heads;
  a.group = (int)(q_heads / cache->kv_heads);
  a.rows = (int)rows;
  a.row_tiles = plan.row_tiles;
  a.max_len = (int)cache->max_len;
  a.block = (int)cache->block;
  a.tiles_log2 = a.block == 32 ? 0 : a.block == 64 ? 1 : 2;
  a.qk_scale = scale * 1.4426950408889634f;
  a.out = out;
  a.part = plan.workspace ? static_cast<float*>(workspace) : nullptr;
  a.ctas = plan.ctas;
  const int nt = plan.nt;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf = cache->dtype == ML_DTYPE_BF16;
  if (cache->format == ML_KV8_INT8)
    return bf ? launch_dim<__nv_bfloat16, ML_KV8_INT8>(a, cache->head_dim, nt, st)
              : launch_dim<__half, ML_KV8_INT8>(a, cache->head_dim, nt, st);
  return bf ? launch_dim<__nv_bfloat16, ML_KV8_E4M3>(a, cache->head_dim, nt, st)
            : launch_dim<__half, ML_KV8_E4M3>(a, cache->head_dim, nt, st);
}
