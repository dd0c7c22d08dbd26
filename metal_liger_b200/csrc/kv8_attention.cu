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
// time; with at most 16 rows to a tile a tcgen05 tile of 64 or 128 rows would
// be mostly padding, and its operands would have to go back through shared
// memory after the conversion.
//   S^T = K Q^T:  A = 16 positions x 16 dims, B = 16 dims x 8 query rows
//   O^T = V^T P^T: A = 16 dims x 16 positions, B = 16 positions x 8 query rows
// Any order of the summed index serves as long as both operands agree on it,
// so a lane takes 16 consecutive bytes of a row for four k-steps of S^T, and
// 16 consecutive dims of four positions for eight m-tiles of O^T: neither
// operand is transposed in memory.  P^T needs one movmatrix per 8 x 8.
//
// Queries enter as fp16 scaled by a power of two per row (bf16 and fp16 fit
// exactly down to 2^-14 of the row's largest value, and to 2^-25 of it below).
// Probabilities are fp16 in [0, 1], sums and outputs fp32.  The scale of a V
// block enters the exponent: the output keeps its own running reference
// Mo = max(s + log2 vscale), so weights 2^(s + log2 vscale - Mo) stay in
// [0, 1] however far the block scales lie apart.
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

namespace ml {
namespace {

constexpr int kTile = 32;  // positions per warp step

struct AttnArgs {
  const void* q;            // [B, Hq, T, D] at element strides
  int64_t sq[3];
  const uint8_t* codes[2];  // [B, Hkv, L, D]
  const float* scale[2];    // [B, Hkv, L / block]
  Kv8Span span;
  int batch, kv_heads, group, rows, row_tiles, max_len, block;
  float qk_scale;           // scale * log2(e)
  void* out;                // [B, T, Hq, D]
  float* part;              // [2 * gridDim.x] pieces; null: a CTA per segment
  int ctas;                 // CTAs that share the flat list
};

template <int D>
struct Shape {
  static constexpr int kWarps = D == 256 ? 4 : 8;
  static constexpr int kTileBytes = 2 * kTile * D;  // K and V
  static constexpr int MT = D / 16;                 // m-tiles of O^T
};

template <int D, int NT>
struct Config : Shape<D> {
  static constexpr int kStages = D == 64 ? 4 : NT == 1 ? 3 : 2;
  static constexpr int kImage = NT * Shape<D>::MT * 4 * 32;  // floats of a piece
  static constexpr int kStats = 3 * 8 * NT;
  static constexpr int kPiece = kImage + kStats;             // floats, in the workspace
  static constexpr size_t smem() {
    return (size_t)Shape<D>::kWarps * (kStages * Shape<D>::kTileBytes + kImage * 4);
  }
};

// ---------------------------------------------------------------------------
// The flat list of tiles
// ---------------------------------------------------------------------------

__device__ __forceinline__ int visible(const AttnArgs& a, int b, int t) {
  if (t >= a.span.count(b)) return 0;
  const int64_t n = a.span.first(b) + t + 1;
  return n <= 0 ? 0 : n > a.max_len ? a.max_len : (int)n;
}
// Tiles of each segment of sequence b: up to its last real query's position,
// at least one (which then writes the zeros).
__device__ __forceinline__ int tiles_of(const AttnArgs& a, int b) {
  const int c = a.span.count(b);
  const int n = c > 0 ? visible(a, b, c - 1) : 0;
  return n <= 0 ? 1 : (n + kTile - 1) / kTile;
}
__device__ __forceinline__ int64_t tiles_per_cta(int64_t total, int ctas, int warps) {
  const int64_t even = (total + ctas - 1) / ctas;
  return even > warps ? even : warps;
}

// Block-wide: the total number of tiles, and for each of `n` flat positions
// the sequence that holds it and the tiles before that sequence.
template <int THREADS>
__device__ int64_t locate(const AttnArgs& a, int64_t* scan, int warps, int* at_b,
                          int64_t* at_base, int64_t* per_cta) {
  const int per = (a.batch + THREADS - 1) / THREADS;
  const int64_t seg = (int64_t)a.kv_heads * a.row_tiles;
  const int b0 = threadIdx.x * per;
  int64_t mine = 0;
  for (int b = b0; b < min(b0 + per, a.batch); ++b) mine += tiles_of(a, b) * seg;
  // inclusive scan over the block
  int64_t run = mine;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += v;
  }
  if (lane == 31) scan[warp] = run;
  __syncthreads();
  int64_t total = 0, before = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += scan[w];
    total += scan[w];
  }
  int64_t lo = before + run - mine, hi = before + run;
  const int64_t cta = tiles_per_cta(total, a.ctas, warps);
  *per_cta = cta;
  const int64_t sub = (cta + warps - 1) / warps;
  for (int w = 0; w < warps; ++w) {
    const int64_t u = blockIdx.x * cta + min(w * sub, cta);
    if (u < lo || u >= hi) continue;
    int64_t base = lo;
    for (int b = b0;; ++b) {
      const int64_t n = tiles_of(a, b) * seg;
      if (u < base + n) {
        at_b[w] = b;
        at_base[w] = base;
        break;
      }
      base += n;
    }
  }
  __syncthreads();
  return total;
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
  // As an image [register][lane] and stats [3][8 NT]
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
  // Adds a saved piece (l summed over lanes in both).
  __device__ __forceinline__ void join(const float* image, const float* stats, int lane) {
    const int t = lane & 3;
    float ka[NT][2], kb[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = n * 8 + 2 * t + c;
        const float pm = stats[r], pl = stats[8 * NT + r], po = stats[16 * NT + r];
        const float nm = fmaxf(m[n][c], pm), no = fmaxf(mo[n][c], po);
        l[n][c] = l[n][c] * rel2(m[n][c], nm) + pl * rel2(pm, nm);
        ka[n][c] = rel2(mo[n][c], no);
        kb[n][c] = rel2(po, no);
        m[n][c] = nm;
        mo[n][c] = no;
      }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[n][j][e] = acc[n][j][e] * ka[n][e & 1] +
                         image[((n * (D / 16) + j) * 4 + e) * 32 + lane] * kb[n][e & 1];
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
        const float f = visible(a, b, tok) > 0 ? rel2(mo[n][c], m[n][c]) / l[n][c] : 0.f;
        const bool none = f == 0.f;  // no position, or all V blocks zero
        T* dst = static_cast<T*>(a.out) +
                 (((int64_t)b * a.span.tokens + tok) * (a.kv_heads * a.group) + h) * D;
        constexpr int PER = D == 64 ? 8 : 16;  // consecutive dims of a lane
#pragma unroll
        for (int p = 0; p < D / 8 / PER; ++p) {
          uint32_t w[PER / 2];
#pragma unroll
          for (int j = 0; j < PER / 2; ++j) {
            const float lo = none ? 0.f : acc[n][p * 8 + j][c] * f;
            const float hi = none ? 0.f : acc[n][p * 8 + j][2 + c] * f;
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

  template <typename T>
  __device__ __forceinline__ void load(const AttnArgs& a, int b, int kvh, int rt, int lane) {
    const int g = lane >> 2, t = lane & 3;
    lim_min = a.max_len;
    lim_max = 0;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = (rt * NT + n) * 8 + g;
      const int tok = r / a.group, h = kvh * a.group + r % a.group;
      const T* src = static_cast<const T*>(a.q) + b * a.sq[0] + h * a.sq[1] + tok * a.sq[2];
      uint4 raw[D / 32];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < D / 64; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint4& x = raw[2 * i + u];
          x = r < a.rows ? *reinterpret_cast<const uint4*>(src + i * 64 + t * 16 + u * 8)
                         : make_uint4(0, 0, 0, 0);
          top = __vmaxu2(top, __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu),
                                       __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu)));
        }
      top = max(top & 0xffffu, top >> 16);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      T tv;
      const uint16_t tb = (uint16_t)top;
      memcpy(&tv, &tb, 2);
      const float amax = to_f32(tv);
      // 2^-e with 2^e the largest power of two <= amax; 1 for zero, inf, NaN
      // rows and below 2^-100 (whose scores are nothing anyway)
      const uint32_t e = __float_as_uint(amax) & 0x7f800000u;
      const bool ok = e > 0x0d800000u && e < 0x7f000000u;
      const float down = ok ? __uint_as_float(0x7f000000u - e) : e >= 0x7f000000u && amax <= 3.4028235e38f ? 0x1p-127f : 1.f;
      const float up = ok ? __uint_as_float(e) : e >= 0x7f000000u && amax <= 3.4028235e38f ? 0x1p127f : 1.f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          T two[2];
          memcpy(two, &w[k], 4);
          // words of 2 dims: k-step 4 (i / 2) + 2 (i % 2) + k / 2, register k & 1
          frag[n][(i / 2) * 4 + (i % 2) * 2 + k / 2][k & 1] =
              half2_bits(to_f32(two[0]) * down, to_f32(two[1]) * down);
        }
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

// One tile of 32 positions, the first of them `pos`.
template <int D, int NT, int FMT, bool MASK>
__device__ __forceinline__ void tile_step(State<D, NT>& st, const Query<D, NT>& q,
                                          const uint8_t* ks, const uint8_t* vs, float k_scale,
                                          float v_scale, int pos, int lane) {
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
  const float lv = log2f(v_scale);
  uint32_t p[2][NT][2];
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
      const float o = lv - (st.mo[n][c] == -INFINITY ? 0.f : st.mo[n][c]);
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
  // dims: a lane's 16 (8 of 64) consecutive ones of each 128
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

// Position in the flat list: tile `tile` of `tiles` of segment `seg` (kv head x
// row tile) of sequence b.
struct Cursor {
  int b, seg, tile, tiles;

  __device__ __forceinline__ void set(const AttnArgs& a, int b_, int64_t offset) {
    b = b_;
    tiles = tiles_of(a, b);
    seg = (int)(offset / tiles);
    tile = (int)(offset - (int64_t)seg * tiles);
  }
  __device__ __forceinline__ void next(const AttnArgs& a) {
    if (++tile < tiles) return;
    tile = 0;
    if (++seg < a.kv_heads * a.row_tiles) return;
    seg = 0;
    if (++b < a.batch) tiles = tiles_of(a, b);
  }
};

template <int D>
__device__ __forceinline__ void load_tile(const AttnArgs& a, const Cursor& c, uint32_t dst,
                                          uint32_t scales, int lane) {
  const int64_t bh = (int64_t)c.b * a.kv_heads + c.seg / a.row_tiles;
  const int64_t off = (bh * a.max_len + (int64_t)c.tile * kTile) * D;
  constexpr int CPR = D / 16;
#pragma unroll
  for (int i = 0; i < kTile * CPR / 32; ++i) {
    const int x = i * 32 + lane;
    const int r = x / CPR, ch = x % CPR;
    cp_async16(dst + r * D + k_chunk<D>(r, ch) * 16, a.codes[0] + off + x * 16);
    cp_async16(dst + kTile * D + r * D + v_chunk<D>(r, ch) * 16, a.codes[1] + off + x * 16);
  }
  if (lane < 2)
    cp_async4(scales + lane * 4,
              a.scale[lane] + bh * (a.max_len / a.block) + (int64_t)c.tile * kTile / a.block);
}

// A piece of a segment that its warp did not see whole.
struct Piece {
  int b, seg, lo, hi, tiles;  // tiles [lo, hi) of `tiles`; hi = 0: none
};

template <typename T, int FMT, int D, int NT>
__global__ void __launch_bounds__(32 * Shape<D>::kWarps, 1)
kv8_attention_kernel(const __grid_constant__ AttnArgs a) {
  using C = Config<D, NT>;
  constexpr int NW = C::kWarps;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t scan[NW], at_base[NW];
  __shared__ int at_b[NW];
  __shared__ Piece pieces[2 * NW];
  __shared__ float stats[2 * NW][C::kStats];
  __shared__ float scales[NW][C::kStages][2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint8_t* ring = smem + (size_t)warp * C::kStages * C::kTileBytes;
  float* first_image = reinterpret_cast<float*>(smem + (size_t)NW * C::kStages * C::kTileBytes) +
                       (size_t)warp * C::kImage;

  pdl_wait();
  pdl_release();
  // this warp's run [lo, hi) of the list, and where it starts
  int64_t lo, hi, cta_lo = 0;
  Cursor cur;
  if (a.part == nullptr) {  // a CTA per segment
    const int seg = a.kv_heads * a.row_tiles;
    const int b = blockIdx.x / seg, s = blockIdx.x % seg;
    const int n = tiles_of(a, b), sub = (n + NW - 1) / NW;
    lo = min(warp * sub, n);
    hi = min(lo + sub, (int64_t)n);
    cur.b = b;
    cur.seg = s;
    cur.tiles = n;
    cur.tile = (int)lo;
  } else {
    int64_t per_cta;
    const int64_t total = locate<32 * NW>(a, scan, NW, at_b, at_base, &per_cta);
    cta_lo = blockIdx.x * per_cta;
    const int64_t cta_hi = min(total, cta_lo + per_cta), sub = (per_cta + NW - 1) / NW;
    lo = min(cta_lo + warp * sub, cta_hi);
    hi = min(lo + sub, cta_hi);
    if (lo < hi) cur.set(a, at_b[warp], lo - at_base[warp]);
  }

  if (lane < 2) pieces[2 * warp + lane].hi = 0;
  __syncwarp();
  if (lo < hi) {
    const uint32_t ring_u = smem_u32_of(ring), scales_u = smem_u32_of(&scales[warp][0][0]);
    Cursor ahead = cur;
    const int64_t n = hi - lo;
#pragma unroll
    for (int i = 0; i < C::kStages - 1; ++i) {
      if (i < n) {
        load_tile<D>(a, ahead, ring_u + i * C::kTileBytes, scales_u + i * 8, lane);
        ahead.next(a);
      }
      cp_commit();
    }
    State<D, NT> st;
    Query<D, NT> q;
    int stage = 0, piece_lo = 0;
    bool fresh = true;
    for (int64_t i = 0; i < n; ++i) {
      if (fresh) {
        q.template load<T>(a, cur.b, cur.seg / a.row_tiles, cur.seg % a.row_tiles, lane);
        st.clear();
        piece_lo = cur.tile;
        fresh = false;
      }
      cp_wait<C::kStages - 2>();
      __syncwarp();
      if (i + C::kStages - 1 < n) {
        const int to = stage == 0 ? C::kStages - 1 : stage - 1;
        load_tile<D>(a, ahead, ring_u + to * C::kTileBytes, scales_u + to * 8, lane);
        ahead.next(a);
      }
      cp_commit();
      const uint8_t* ks = ring + stage * C::kTileBytes;
      const int pos = cur.tile * kTile;
      const float k_scale = scales[warp][stage][0], v_scale = scales[warp][stage][1];
      if (pos + kTile <= q.lim_min)
        tile_step<D, NT, FMT, false>(st, q, ks, ks + kTile * D, k_scale, v_scale, pos, lane);
      else
        tile_step<D, NT, FMT, true>(st, q, ks, ks + kTile * D, k_scale, v_scale, pos, lane);
      stage = stage == C::kStages - 1 ? 0 : stage + 1;
      const bool ends = cur.tile + 1 == cur.tiles;
      if (ends || i + 1 == n) {
        st.sum_l();
        if (ends && piece_lo == 0) {
          st.template write<T>(a, cur.b, cur.seg / a.row_tiles, cur.seg % a.row_tiles, lane);
        } else {
          // the run's first piece has a place of its own, its last one takes
          // the ring, which nothing uses any more
          const int slot = i + 1 - (cur.tile + 1 - piece_lo) == 0 ? 0 : 1;
          if (slot == 1) {
            cp_wait<0>();
            __syncwarp();
          }
          st.save(slot == 0 ? first_image : reinterpret_cast<float*>(ring), stats[2 * warp + slot],
                  lane);
          if (lane == 0)
            pieces[2 * warp + slot] = {cur.b, cur.seg, piece_lo, cur.tile + 1, cur.tiles};
        }
        fresh = true;
      }
      cur.next(a);
    }
  }
  cp_wait<0>();
  __syncthreads();
  // Join the pieces of a segment: runs of consecutive entries, a warp per run.
  int run = 0;
  for (int e = 0; e < 2 * NW;) {
    const Piece p = pieces[e];
    if (p.hi == 0) {
      ++e;
      continue;
    }
    int last = e, f = e + 1;
    for (; f < 2 * NW; ++f) {
      const Piece& o = pieces[f];
      if (o.hi == 0) continue;
      if (o.b != p.b || o.seg != p.seg) break;
      last = f;
    }
    if (run++ % NW == warp) {
      State<D, NT> st;
      st.clear();
      for (int x = e; x <= last; ++x) {
        if (pieces[x].hi == 0) continue;
        const float* image =
            x & 1 ? reinterpret_cast<const float*>(smem + (size_t)(x >> 1) * C::kStages * C::kTileBytes)
                  : reinterpret_cast<const float*>(smem + (size_t)NW * C::kStages * C::kTileBytes) +
                        (size_t)(x >> 1) * C::kImage;
        st.join(image, stats[x], lane);
      }
      if (p.lo == 0 && pieces[last].hi == p.tiles) {
        st.template write<T>(a, p.b, p.seg / a.row_tiles, p.seg % a.row_tiles, lane);
      } else {
        // slot 0: the piece the CTA's run starts with
        const bool starts = e == 0;
        float* to = a.part + (int64_t)(2 * blockIdx.x + (starts ? 0 : 1)) * C::kPiece;
        st.save(to, to + C::kImage, lane);
      }
    }
    e = f;
  }
}

// Joins the segments that cross CTAs, a warp each.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(128) kv8_attention_join(const __grid_constant__ AttnArgs a) {
  using C = Config<D, NT>;
  __shared__ int64_t red[8];
  pdl_wait();
  pdl_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per_b = a.kv_heads * a.row_tiles;
  // the CTA's segments are of one sequence: tiles before it, and in all
  const int chunks = (per_b + 3) / 4;
  const int b = blockIdx.x / chunks;
  int64_t before = 0, total = 0;
  for (int i = threadIdx.x; i < a.batch; i += 128) {
    const int64_t n = (int64_t)tiles_of(a, i) * per_b;
    total += n;
    if (i < b) before += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  if (lane == 0) {
    red[warp] = before;
    red[4 + warp] = total;
  }
  __syncthreads();
  before = red[0] + red[1] + red[2] + red[3];
  total = red[4] + red[5] + red[6] + red[7];
  const int seg = (blockIdx.x % chunks) * 4 + warp;
  if (seg >= per_b) return;
  const int64_t per_cta = tiles_per_cta(total, a.ctas, C::kWarps);
  const int n = tiles_of(a, b);
  const int64_t lo = before + (int64_t)seg * n, hi = lo + n;
  const int64_t c0 = lo / per_cta, c1 = (hi - 1) / per_cta;
  if (c0 == c1) return;
  State<D, NT> st;
  st.clear();
  for (int64_t c = c0; c <= c1; ++c) {
    const float* p = a.part + (2 * c + (c == c0 && lo > c * per_cta ? 1 : 0)) * C::kPiece;
    st.join(p, p + C::kImage, lane);
  }
  st.template write<T>(a, b, seg / a.row_tiles, seg % a.row_tiles, lane);
}

// Query rows per tile: 8 NT.
inline int n_tiles(int64_t rows, int64_t dim) { return rows > 8 && dim != 256 ? 2 : 1; }

// Caches this short go a CTA to a segment, in one launch.
constexpr int64_t kOneLaunchLen = 512;

inline bool one_launch(const ml_kv8_cache* c) { return c->max_len <= kOneLaunchLen; }

template <typename T, int FMT, int D, int NT>
int launch(AttnArgs a, cudaStream_t st) {
  using C = Config<D, NT>;
  auto kernel = kv8_attention_kernel<T, FMT, D, NT>;
  static PerDevice<cudaError_t> attr;
  ML_CHECK_CUDA(attr.get([&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)C::smem());
  }), "kv8_attention");
  const int64_t segs = (int64_t)a.batch * a.kv_heads * a.row_tiles;
  ML_CHECK_ARG(segs < ((int64_t)1 << 31), "kv8_attention: too many rows");
  const dim3 grid((unsigned)(a.part ? a.ctas : segs));
  ML_CHECK_CUDA(launch_pdl(kernel, grid, dim3(32 * C::kWarps), C::smem(), st, a),
                "kv8_attention");
  if (a.part) {
    const int64_t chunks = ((int64_t)a.kv_heads * a.row_tiles + 3) / 4;
    ML_CHECK_CUDA(launch_pdl(kv8_attention_join<T, D, NT>, dim3((unsigned)(a.batch * chunks)),
                             dim3(128), 0, st, a),
                  "kv8_attention(join)");
  }
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
  if (cache == nullptr || cache->kv_heads <= 0 || cache->batch <= 0 || tokens <= 0 ||
      q_heads <= 0 || one_launch(cache))
    return 0;
  const int nt = n_tiles(q_heads / cache->kv_heads * tokens, cache->head_dim);
  const int64_t piece = nt * cache->head_dim / 16 * 4 * 32 + 3 * 8 * nt;
  return (size_t)num_sms() * 2 * piece * sizeof(float);
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
  const size_t need = ml_kv8_attention_workspace_bytes(cache, q_heads, tokens);
  ML_CHECK_ARG(need == 0 || (workspace && aligned16(workspace) && workspace_bytes >= need),
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
  const int64_t rows = a.group * tokens;
  ML_CHECK_ARG(rows < ((int64_t)1 << 30), "kv8_attention: too many rows");
  const int nt = n_tiles(rows, cache->head_dim);
  a.rows = (int)rows;
  a.row_tiles = (int)((rows + 8 * nt - 1) / (8 * nt));
  a.max_len = (int)cache->max_len;
  a.block = (int)cache->block;
  a.qk_scale = scale * 1.4426950408889634f;
  a.out = out;
  a.part = need ? static_cast<float*>(workspace) : nullptr;
  a.ctas = num_sms();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf = cache->dtype == ML_DTYPE_BF16;
  if (cache->format == ML_KV8_INT8)
    return bf ? launch_dim<__nv_bfloat16, ML_KV8_INT8>(a, cache->head_dim, nt, st)
              : launch_dim<__half, ML_KV8_INT8>(a, cache->head_dim, nt, st);
  return bf ? launch_dim<__nv_bfloat16, ML_KV8_E4M3>(a, cache->head_dim, nt, st)
            : launch_dim<__half, ML_KV8_E4M3>(a, cache->head_dim, nt, st);
}
