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
// summed as integers: W = round(2^43 w), of which V <= 2^20 come to 2^63 at most
// (64 bits, unsigned), exactly and in any order.  Where w < 2^-18 it comes from the fp32
// exponential, with what rounding took from its argument put back (off by
// 2^-22 of it, so by 2^-40 of the largest at most); above from fp64:
// 2^(i/64) from a table times Taylor's quintic in the rest, |r| <= 2^-7, whose
// first term left out is below 2^-54.
//
// A cluster of CTAs holds a row in shared memory where it fits (kMaxResident),
// so HBM is read once; longer ones are read again, from L2.  Every
// step is then a pass over the CTA's slice and an exchange of a few words
// through distributed shared memory.  The kept set is a prefix of the order and
// is found by selection, not by sorting: a histogram over the distance to the
// largest logit, of counts (top-k) or weights (top-p), gives the bin that the
// prefix ends in.  The tokens from there up are few as a rule; they go, in
// index order, to a list in the cluster's first CTA, which sorts it and draws.
// Otherwise the steps go on over the slices: histograms over the bin's keys
// narrow it to one key, and the draw adds up kept weights, and tokens equal to
// that key as long as they are kept, by CTA, warp and lane in index order.
//
// Tokens that need fp64 are rare in most rows and everywhere in flat ones: a
// warp queues them and weighs 32 at a time.
//
// Bound by instructions and by the steps that follow one another, not by
// memory.  Measured, 151936 tokens: one row, top-k and top-p, 15 us; 64 rows, top-p
// and min-p, 53 us (without the list 96, with top-p's end always searched for
// 68); 256 fp32 rows with nothing cut 105 us (1.5 TB/s).
#include "common.cuh"

#include <cooperative_groups.h>

namespace ml {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = kThreads;      // a thread per bin
constexpr int kMaxCluster = 16;
constexpr int kMaxSlice = 65536;     // tokens of a CTA: the histogram's 32-bit parts hold them
constexpr int64_t kMaxVocab = (int64_t)1 << 20;
constexpr double kOne = 8796093022208.0;  // 2^43
// A slice that leaves room for two CTAs on an SM is held; a larger one is read
// again from L2 (256 fp32 rows: 107 us, against 145 held by one CTA per SM).
constexpr size_t kMaxResident = 80 * 1024;
constexpr int kList = kThreads;      // tokens of the list
constexpr int kWarpList = kList / kWarps;  // of them from one warp
constexpr int kTable = 64;

struct SampleArgs {
  const void* logits;  // [rows, V] at row pitch ld
  int64_t ld;
  int V, slice;        // 16-byte vectors of a CTA
  bool resident;
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

// Unsigned order of the key = order of the logits, masked ones 0.  The low G
// bits of a widened 16-bit logit's key say nothing and are dropped.
template <int G>
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x > -INFINITY)) return 0;  // NaN and -inf
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 -> +0: equal logits, equal keys
  return (b & 0x80000000u ? ~b : b | 0x80000000u) >> G;
}
template <int G>
__device__ __forceinline__ float value_of(uint32_t key) {
  key <<= G;
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key & (0xffffffffu << G));
}
template <int G>
constexpr uint32_t kLowest = 0x00800000u >> G;  // of the lowest finite value, or just below
template <typename T> constexpr int kDropped = 0;
template <> constexpr int kDropped<__nv_bfloat16> = 16;
template <> constexpr int kDropped<__half> = 13;

// What the weights and bins of a row are computed with; G: of its keys.
//
// log2 w = (x - shift) rate + c, shift = 0 and c = -top rate as a rule.  With rate
// and c each in two parts, c_hi a multiple of 2^-11 under 2^12, the rest of it
// after the nearest integer n is one fused multiply-add, (x - shift) rate_f +
// (c_hi - n), whose addend is exact and whose result is under 1: off by 2^-25.
// Where |top| rate passes 2^12, the tokens with any weight are within 1% of the
// top: shift = top, x - top is exact and c = 0.
template <int G>
struct Row {
  static constexpr int kKey = G;
  float top, shift, floor;  // floor: its weight is 2^-60; nothing is smaller
  float rate_f, rate_lo, c_hi, c_lo;
  double inv_t, rate;
  const double* table;

  // Returns false where only tokens equal to the top have weight (it is +inf or
  // the lowest of all, or the temperature so small that the next one below has
  // none): the caller cuts the others.
  __device__ bool set(float top_, float t, const double* table_) {
    top = top_;
    table = table_;
    inv_t = 1.0 / (double)t;
    rate = inv_t * 1.4426950408889634;
    const double c = -(double)top * rate;
    shift = fabs(c) > 4096.0 ? top : 0.f;
    c_hi = fabs(c) > 4096.0 ? 0.f : (float)(rint(c * 2048.0) * (1.0 / 2048.0));
    c_lo = fabs(c) > 4096.0 ? 0.f : (float)(c - (double)c_hi);
    rate_f = (float)rate;
    rate_lo = (float)(rate - (double)rate_f);
    floor = fmaxf((float)((double)top - 60.0 / rate), -3.4028235e38f);
    while (((double)top - (double)floor) * rate < 50.0 && top < INFINITY)  // rounded up
      floor = value_of<0>(key_of<0>(floor) - 1);
    if (top < INFINITY && floor > -INFINITY && fabs(c) < 4294967296.0 && rate < 1e30) return true;
    // the top's log2 is 0 (or, of +inf, NaN: not small either)
    const bool inf = !(top < INFINITY);
    floor = -INFINITY;
    shift = inf ? 0.f : top;
    rate_f = inf ? 0.f : 1e30f;
    c_hi = rate_lo = c_lo = 0.f;
    return false;
  }
  __device__ __forceinline__ float log2_weight(float x) const {
    return fmaf(x - shift, rate_f, c_hi);
  }
  __device__ __forceinline__ static bool small(float z) { return z < -18.f; }
  // x >= floor.  43 is added to n on the way, for 2^43 w.
  __device__ __forceinline__ uint32_t small_weight(float x, float z) const {
    const float d = x - shift;
    const float shifted = z + 12582955.f;  // 1.5 * 2^23 + 43: its steps are 1
    const float n = shifted - 12582955.f;
    const float r = fmaf(d, rate_f, c_hi - n) + fmaf(d, rate_lo, c_lo);
    float w;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(r));
    w = __uint_as_float(__float_as_uint(w) + (__float_as_uint(shifted) << 23));
    return __float2uint_rn(w);
  }
  __device__ __forceinline__ uint64_t large_weight(float x) const {
    if (x == top) return (uint64_t)kOne;
    const double y = ((double)x - (double)top) * rate;
    const double magic = 105553116266496.0;  // 1.5 * 2^46: its steps are 2^-6
    const double shifted = y + magic;
    const int k = __double2loint(shifted);
    const double r = y - (shifted - magic);
    // 2^r - 1
    const double p = r * fma(r, fma(r, fma(r, fma(r, 0.0013333558146428443, 0.009618129107628477),
                                           0.05550410866482158), 0.24022650695910072),
                             0.6931471805599453);
    const double t = table[k & (kTable - 1)];
    double w = fma(t, p, t);
    w = __hiloint2double(__double2hiint(w) + ((k >> 6) << 20), __double2loint(w));
    const double i = fma(w, kOne, 4503599627370496.0);  // + 2^52: the integer in its low bits
    return (uint64_t)__double_as_longlong(i) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ uint64_t weight(float x) const {
    const float y = fmaxf(x, floor), z = log2_weight(y);
    return small(z) ? small_weight(y, z) : large_weight(x);
  }
  __device__ __forceinline__ double exact(float x) const {
    return x == top ? 1.0 : exp(((double)x - (double)top) * inv_t);
  }
};

// Which tokens are left: the ones with a logit above x, and the first `ties` of
// those equal to it.
struct Cut {
  static constexpr float kNone = -3.4028235e38f;  // (-inf and NaN never are)
  float x = kNone;
  uint64_t ties = ~(uint64_t)0;
  __device__ __forceinline__ bool has(float v) const { return v >= x; }  // but for the ties
};

struct Shared {
  double table[kTable];            // 2^(i / kTable)
  uint32_t hist[3][kBins];         // 15-bit parts of the sums
  uint64_t sums[2][kBins];         // this CTA's, for the others to read; two in turn
  uint64_t slot[5][kMaxCluster];   // one exchange each
  uint64_t part[kWarps], walk[kWarps];
  int ties[kWarps];
  uint64_t above, in_bin;
  int bin;
  uint32_t key[2];
  float queue[kWarps][64];
  float list_x[kList];
  int list_i[kList];
};

// A CTA's view of its slice: `get(v, x)` gives the N tokens of 16-byte vector v,
// the first of which has index `index(v)`; tokens outside the row read as -inf.
template <typename T>
struct Slice {
  static constexpr int N = 16 / sizeof(T);
  const T* row;
  int V, base, count;  // count: vectors
  const uint4* held;   // in shared memory, or null

  __device__ __forceinline__ Vec16<T> fetch(int v) const {
    const int i = base + v * N;
    if (i >= 0 && i + N <= V) return ld_vec_stream(row + i);
    Vec16<T> r;
#pragma unroll
    for (int e = 0; e < N; ++e)
      r.v[e] = i + e >= 0 && i + e < V ? row[i + e] : from_f32<T>(-INFINITY);
    return r;
  }
  __device__ __forceinline__ Vec16<T> load(int v) const {
    if (held == nullptr) return fetch(v);
    Vec16<T> r;
    *reinterpret_cast<uint4*>(&r) = held[v];
    return r;
  }
  __device__ __forceinline__ static void widen(const Vec16<T>& r, float* x) {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = to_f32(r.v[e]);
  }
  __device__ __forceinline__ void get(int v, float* x) const { widen(load(v), x); }
  __device__ __forceinline__ int index(int v) const { return base + v * N; }
  __device__ __forceinline__ float one(int v, int e) const {  // of a token of the row
    return to_f32(held ? reinterpret_cast<const T*>(held)[v * N + e] : row[index(v) + e]);
  }
};
// Calls f(x[N], v) for the vectors of this warp's share of the slice, all lanes
// together; lanes interleave, so a lane's tokens ascend.  fp32 rows, which are
// seldom held, are loaded a step ahead (256 of 151936: 111 for 115 us; 16-bit
// rows, held, would lose: 64 rows 54 for 52).
template <typename S, typename F>
__device__ __forceinline__ void each(const S& src, F&& f) {
  constexpr bool kAhead = S::N == 4;
  const int per = (src.count + kWarps - 1) / kWarps, warp = threadIdx.x >> 5;
  const int begin = warp * per, end = min(src.count, begin + per);
  const int lane = threadIdx.x & 31;
  decltype(src.load(0)) next;
  if (kAhead && begin + lane < end) next = src.load(begin + lane);
  for (int v0 = begin; v0 < end; v0 += 32) {
    const int v = v0 + lane;
    float x[S::N];
    if (v < end) {
      if (!kAhead) next = src.load(v);
      S::widen(next, x);
    } else {
#pragma unroll
      for (int e = 0; e < S::N; ++e) x[e] = -INFINITY;
    }
    if (kAhead && v + 32 < end) next = src.load(v + 32);
    f(x, v);
  }
}

// Tokens that few lanes have, handed on a warp at a time.
struct Queue {
  float* held;  // 64
  int at = 0, waiting = 0;

  // `mask`: of this lane's tokens x[N] of vector v; sink(x, valid).  Of four, one
  // is picked in registers; of eight, read again (64 rows of bf16: 52 for 54 us).
  template <typename S, typename F>
  __device__ __forceinline__ void push(const S& src, const float* x, int v, uint32_t mask,
                                       F&& sink) {
    constexpr int N = S::N;
    const int lane = threadIdx.x & 31;
    // one of each lane's at a time: they are few, or every lane has all
    while (__any_sync(0xffffffffu, mask != 0)) {
      const unsigned m = __ballot_sync(0xffffffffu, mask != 0);
      if (mask) {
        const int e = __ffs(mask) - 1;
        float one = x[0];
        if constexpr (N == 4) {
#pragma unroll
          for (int i = 1; i < N; ++i) one = e == i ? x[i] : one;
        } else {
          one = src.one(v, e);
        }
        held[(at + waiting + __popc(m & ((1u << lane) - 1))) & 63] = one;
        mask &= mask - 1;
      }
      waiting += __popc(m);
      if (waiting < 32) continue;
      __syncwarp();
      const float q = held[(at + lane) & 63];
      __syncwarp();
      at += 32;
      waiting -= 32;
      sink(q, true);
    }
  }
  template <typename F>
  __device__ __forceinline__ void flush(float none, F&& sink) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
    if (waiting) sink(lane < waiting ? held[(at + lane) & 63] : none, lane < waiting);
    __syncwarp();
  }
};

// each() for weights: sink(x, W, valid) gets the large ones, a warp at a time;
// the sum of this lane's small ones is returned.  OPEN: the cut has everything.
// TIES: this lane's tokens equal to the cut's x are counted.
template <bool OPEN, bool TIES, typename S, typename R, typename F>
__device__ __forceinline__ uint64_t each_weight(const S& src, const R& row, const Cut& cut,
                                                float* queue, int* ties, F&& sink) {
  uint64_t tail = 0;
  Queue waiting = {queue};
  auto weigh = [&](float x, bool valid) { sink(x, row.large_weight(x), valid); };
  each(src, [&](const float* x, int v) {
    uint32_t small = 0, large = 0;
#pragma unroll
    for (int e = 0; e < S::N; ++e) {
      // (-inf and NaN take the floor's place, which weighs nothing)
      const bool in = OPEN || cut.has(x[e]);
      if (TIES) *ties += x[e] == cut.x;
      const float y = fmaxf(x[e], row.floor), z = row.log2_weight(y);
      const uint32_t w = row.small_weight(y, z);
      if (!R::small(z)) large |= in ? 1u << e : 0;
      else small += in ? w : 0;
    }
    waiting.push(src, x, v, large, weigh);
    tail += small;
  });
  waiting.flush(row.top, weigh);
  return tail;
}

__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ uint64_t warp_scan64(uint64_t v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t c = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += c;
  }
  return v;
}

struct Cluster {
  int size, rank;
  __device__ __forceinline__ void sync() const {
    if (size == 1) __syncthreads();
    else cg::this_cluster().sync();
  }
  template <typename P>
  __device__ __forceinline__ P* of(P* p, int r) const {
    return size == 1 ? p : cg::this_cluster().map_shared_rank(p, r);
  }
  // Every CTA's value, in its own slot of every CTA.  The value is uniform.
  __device__ __forceinline__ void gather(Shared& sh, int step, uint64_t value) const {
    if ((int)threadIdx.x < size) of(&sh, threadIdx.x)->slot[step][rank] = value;
    sync();
  }
};

__device__ __forceinline__ void add_parts(uint32_t (*hist)[kBins], int bin, uint64_t v) {
  const uint32_t lo = (uint32_t)v & 0x7fff, mid = (uint32_t)(v >> 15) & 0x7fff,
                 hi = (uint32_t)(v >> 30);
  if (lo) atomicAdd(&hist[0][bin], lo);
  if (mid) atomicAdd(&hist[1][bin], mid);
  if (hi) atomicAdd(&hist[2][bin], hi);
}
// The same from a whole warp, which often has one bin (flat rows, the far end).
__device__ __forceinline__ void add_warp(uint32_t (*hist)[kBins], int bin, uint64_t v, bool valid) {
  const int b0 = __shfl_sync(0xffffffffu, bin, 0);
  if (__all_sync(0xffffffffu, !valid || bin == b0)) {
    v = warp_sum64(valid ? v : 0);
    if ((threadIdx.x & 31) == 0) add_parts(hist, b0, v);
  } else if (valid) {
    add_parts(hist, bin, v);
  }
}

// Where a selection stands: the prefix ends among the keys [lo, hi], after
// values of `above` before them; `need` in all.
struct Search {
  uint32_t lo, hi;
  uint64_t above, need;
  int round;        // histograms so far (of the two sums in turn)
  bool whole;       // nothing to cut
  bool beyond;      // the prefix ends in the last histogram's last bin
  uint64_t in_bin;  // sum of the bin that it ends in
};

// What a histogram's bins are: distances to the top, near or far, or keys.
// Near: counts in bins of 1/16 over 32, weights in bins of 1/28.5 over 18 log2s
// (the large weights: all small ones are in the last bin); far: twice as wide
// and long, from where the near ones end.
enum Bins { kNear, kFar, kKeys };

// One histogram of the tokens in `in` and [q.lo, q.hi]; q narrows to the bin
// that the prefix ends in.  WEIGHT: q.need, where 0, becomes p of the sum less
// `excess`, the weight of the last tokens in the order that are not in `in`.
template <bool WEIGHT, Bins BINS, typename S, typename R>
__device__ void narrow(const S& src, const Cluster& cl, Shared& sh, const R& row, const Cut& in,
                       Search& q, double p, uint64_t excess) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kFrom = BINS == kFar ? kBins / 2 : 0;
  const float per = (WEIGHT ? row.rate_f * 28.5f : 16.f) * (BINS == kFar ? 0.5f : 1.f);
  auto distance = [&](float x) {
    // (NaN, at the top where it or the rate is infinite, converts to 0)
    return max(0, min(__float2int_rz((row.top - x) * per) - kFrom, kBins - 1));
  };
  const int bits = 32 - __clz(q.hi - q.lo);
  const int shift = bits > 9 ? bits - 9 : 0;
#pragma unroll
  for (int i = 0; i < 3; ++i) sh.hist[i][tid] = 0;
  __syncthreads();
  if (tid == 0) sh.bin = kBins - 1;
  if (WEIGHT && BINS == kNear) {
    uint64_t tail = each_weight<false, false>(
        src, row, in, sh.queue[warp], nullptr,
        [&](float x, uint64_t w, bool valid) { add_warp(sh.hist, distance(x), w, valid); });
    tail = warp_sum64(tail);
    if (lane == 0) add_parts(sh.hist, kBins - 1, tail);
  } else {
    // in the keys' range by value: -0 has a key of its own, which no token has
    constexpr uint32_t kMinusZero = 0x7fffffffu >> R::kKey;
    const float x_lo = fmaxf(value_of<R::kKey>(q.lo == kMinusZero ? q.lo + 1 : q.lo), in.x);
    const float x_hi = value_of<R::kKey>(q.hi == kMinusZero ? q.hi - 1 : q.hi);
    auto bin_of = [&](float x) {
      return BINS == kKeys ? (int)((q.hi - key_of<R::kKey>(x)) >> shift) : distance(x);
    };
    Queue some = {sh.queue[warp]};
    auto weigh = [&](float x, bool valid) {
      if (valid) add_parts(sh.hist, bin_of(x), row.weight(x));
    };
    each(src, [&](const float* x, int v) {
      uint32_t mask = 0;
#pragma unroll
      for (int e = 0; e < S::N; ++e) {
        const bool in_range = x[e] >= x_lo && x[e] <= x_hi;
        if (WEIGHT) mask |= in_range ? 1u << e : 0;
        else if (in_range) atomicAdd(&sh.hist[0][bin_of(x[e])], 1u);
      }
      if (WEIGHT) some.push(src, x, v, mask, weigh);
    });
    if (WEIGHT) some.flush(row.top, weigh);
  }
  __syncthreads();
  uint64_t s = sh.hist[0][tid] + ((uint64_t)sh.hist[1][tid] << 15) + ((uint64_t)sh.hist[2][tid] << 30);
  if (cl.size > 1) {
    uint64_t* mine = &sh.sums[q.round & 1][tid];
    *mine = s;
    cl.sync();
    s = 0;
#pragma unroll 8
    for (int r = 0; r < cl.size; ++r) s += *cl.of(mine, r);
  }
  ++q.round;
  uint64_t incl = warp_scan64(s);
  if (lane == 31) sh.part[warp] = incl;
  __syncthreads();
  uint64_t total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) incl += sh.part[w];
    total += sh.part[w];
  }
  if (BINS == kNear) {
    total -= excess;
    if (WEIGHT && q.need == 0) {
      const double f = ceil(p * (double)total);
      q.need = f < 1.0 ? 1 : (uint64_t)f;
    }
    if (q.need >= total) {
      q.whole = true;
      return;
    }
  }
  if (q.above + incl >= q.need && q.above + incl - s < q.need) {
    sh.bin = tid;
    sh.above = q.above + incl - s;
    sh.in_bin = s;
  }
  __syncthreads();
  const int bin = sh.bin;
  q.above = sh.above;
  q.in_bin = sh.in_bin;
  q.beyond = bin == kBins - 1;
  if (BINS == kKeys) {
    const uint64_t down = (uint64_t)bin << shift;
    const uint32_t h = down <= q.hi - q.lo ? q.hi - (uint32_t)down : q.lo;
    const uint32_t span = (1u << shift) - 1;
    q.lo = h - q.lo > span ? h - span : q.lo;
    q.hi = h;
    return;
  }
  // The keys of a bin of distances are neighbours: find the first and last
  // (distances fall as keys grow), a warp for each: the smallest key with a
  // distance <= bin, and < bin.  By 32-way search, from around the bin's edge
  // where that holds the key.
  if (warp < 2) {
    auto holds = [&](uint64_t k) {
      const int d = distance(value_of<R::kKey>((uint32_t)k));
      return warp == 0 ? d <= bin : d < bin;
    };
    uint32_t a = q.lo, b = q.hi + 1;  // the answer lies in [a, b]
    const float edge = row.top - (float)(bin + kFrom + 1 - warp) / per;
    const float off = (fabsf(row.top) + fabsf(edge)) * 1e-6f;
    if (off < 1e30f) {
      const uint32_t ka = key_of<R::kKey>(edge - off), kb = key_of<R::kKey>(edge + off) + 1;
      const bool inside = ka > a && kb < b && ka < kb;
      if (__ballot_sync(0xffffffffu, inside && (lane == 0 ? !holds(ka - 1) : holds(kb))) ==
          0xffffffffu) {
        a = ka;
        b = kb;
      }
    }
    while (a < b) {
      const uint32_t step = (b - a + 31) / 32;
      const uint64_t k = (uint64_t)a + (uint64_t)step * lane;
      const bool ok = k >= b || holds(k);
      const unsigned m = __ballot_sync(0xffffffffu, ok);
      const int f = m ? __ffs(m) - 1 : 32;
      const uint64_t t = (uint64_t)a + (uint64_t)step * f;
      const uint32_t nb = t < b ? (uint32_t)t : b;
      a = f == 0 ? nb : (uint32_t)((uint64_t)a + (uint64_t)step * (f - 1) + 1);
      b = nb;
    }
    if (lane == 0) sh.key[warp] = a;
  }
  __syncthreads();
  q.lo = sh.key[0];
  q.hi = sh.key[1] - 1;
}

// The key of the smallest logit that min-p keeps, by 32-way search.
template <int G>
__device__ uint32_t least_key(Shared& sh, const Row<G>& row, float least, uint32_t top_key) {
  const int lane = threadIdx.x & 31;
  __syncthreads();
  if (threadIdx.x < 32) {
    uint32_t lo = kLowest<G>, hi = top_key;  // the answer lies in [lo, hi]: the largest qualifies
    while (lo < hi) {
      const uint32_t step = (hi - lo + 31) / 32;
      const uint64_t k = (uint64_t)lo + (uint64_t)step * lane;
      const bool ok = k >= hi || row.exact(value_of<G>((uint32_t)k)) >= (double)least;
      const unsigned m = __ballot_sync(0xffffffffu, ok);
      const int j = m ? __ffs(m) - 1 : 32;
      const uint64_t top_k = (uint64_t)lo + (uint64_t)step * j;
      const uint32_t nh = top_k < hi ? (uint32_t)top_k : hi;
      lo = j == 0 ? nh : (uint32_t)((uint64_t)lo + (uint64_t)step * (j - 1) + 1);
      hi = nh;
    }
    if (lane == 0) sh.key[0] = lo;
  }
  __syncthreads();
  return sh.key[0];
}

// Narrows to one key; as many of the tokens equal to it are left as still needed.
template <bool WEIGHT, typename S, typename R>
__device__ Cut finish(const S& src, const Cluster& cl, Shared& sh, const R& row, const Cut& in,
                      Search& q) {
  while (q.lo < q.hi) narrow<WEIGHT, kKeys>(src, cl, sh, row, in, q, 0.0, 0);
  Cut c;
  c.x = value_of<R::kKey>(q.lo);
  const uint64_t each_w = WEIGHT ? row.weight(c.x) : 1;
  c.ties = (q.need - q.above + each_w - 1) / each_w;
  return c;
}

// The tokens with a logit >= x, in index order, to the first CTA's list;
// returns their number there and everywhere, or -1 where they do not fit.
template <typename T>
__device__ int collect(const Slice<T>& sl, const Cluster& cl, Shared& sh, float x) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // each warp's go to a stretch of this CTA's own (idle) list space, the first
  // CTA's first warps' included: they are moved once all are counted
  int n = 0;
  constexpr int kHold = kWarpList;
  float* hx = sh.list_x + warp * kHold;
  int* hi = sh.list_i + warp * kHold;
  each(sl, [&](const float* f, int v) {
    unsigned mask = 0;
#pragma unroll
    for (int e = 0; e < Slice<T>::N; ++e)
      if (f[e] >= x) mask |= 1u << e;
    if (!__any_sync(0xffffffffu, mask != 0)) return;
    const int c = __popc(mask);
    int incl = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    int at = n + incl - c;
#pragma unroll
    for (int e = 0; e < Slice<T>::N; ++e)
      if (mask >> e & 1) {
        if (at < kHold) {
          hx[at] = f[e];
          hi[at] = sl.index(v) + e;
        }
        ++at;
      }
    n += __shfl_sync(0xffffffffu, incl, 31);
  });
  __syncthreads();
  if (lane == 0) sh.part[warp] = (uint64_t)n;
  __syncthreads();
  int here = 0, upto = 0;
  bool fits = true;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const int c = (int)sh.part[w];
    fits = fits && c <= kHold;
    if (w < warp) upto += c;
    here += c;
  }
  // this warp's tokens, in registers while the list is filled
  float kx[kHold / 32];
  int ki[kHold / 32];
#pragma unroll
  for (int j = 0; j < kHold / 32; ++j) {
    kx[j] = hx[j * 32 + lane];
    ki[j] = hi[j * 32 + lane];
  }
  cl.gather(sh, 4, fits ? (uint64_t)here : (uint64_t)kList + 1);
  int before = 0, total = 0;
  for (int r = 0; r < cl.size; ++r) {
    if (r < cl.rank) before += (int)sh.slot[4][r];
    total += (int)sh.slot[4][r];
  }
  if (total > kList) return -1;
  Shared* to = cl.of(&sh, 0);
#pragma unroll
  for (int j = 0; j < kHold / 32; ++j)
    if (j * 32 + lane < n) {
      to->list_x[before + upto + j * 32 + lane] = kx[j];
      to->list_i[before + upto + j * 32 + lane] = ki[j];
    }
  cl.sync();
  return total;
}

struct Filter {
  int64_t k;
  double p;
  float least, u;
};

// Inclusive sums over the CTA, and the whole.
__device__ __forceinline__ uint64_t block_scan(Shared& sh, uint64_t v, uint64_t* total,
                                               uint64_t* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_scan64(v);
  __syncthreads();
  if (lane == 31) part[warp] = v;
  __syncthreads();
  uint64_t all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) v += part[w];
    all += part[w];
  }
  *total = all;
  return v;
}

// u of the total, below it: the token is the first with a running weight above.
__device__ __forceinline__ uint64_t target_of(const Filter& f, uint64_t total) {
  const double t = (f.u > 0.f ? (double)f.u : 0.0) * (double)total;
  return t < (double)total ? min((uint64_t)t, total - 1) : total - 1;
}

// The list's n <= kThreads tokens, a thread each: sorted, cut by rank and running
// weight, put back in index order and drawn from.  need: the weight top-p asks
// for, 0 where it is p of the first k.
template <typename R, typename W>
__device__ void draw_sorted(Shared& sh, const R& row, const Filter& f, int n, uint64_t need,
                            W&& write) {
  const int tid = threadIdx.x;
  // largest first, then list (index) order; bitonic, by shuffles within a warp
  uint64_t mine =
      tid < n ? ((uint64_t)key_of<0>(sh.list_x[tid]) << 32) | ~(uint32_t)tid : (uint64_t)0;
  int size = 32;
  while (size < n) size *= 2;
  for (int k = 2; k <= size; k *= 2) {
    for (int j = k / 2; j > 0; j /= 2) {
      uint64_t other;
      if (j < 32) {
        other = __shfl_xor_sync(0xffffffffu, mine, j);
      } else {
        __syncthreads();
        sh.sums[0][tid] = mine;
        __syncthreads();
        other = sh.sums[0][tid ^ j];
      }
      const bool larger = ((tid & j) == 0) == ((tid & k) == 0);
      if ((mine < other) == larger) mine = other;
    }
  }
  const bool on = mine != 0 && tid < n;
  const int at = on ? (int)~(uint32_t)mine : 0;
  __syncthreads();
  sh.sums[0][tid] = 0;
  const float x = on ? value_of<0>((uint32_t)(mine >> 32)) : row.top;
  uint64_t w = on && (f.k <= 0 || tid < f.k) ? row.weight(x) : 0, total;
  const uint64_t upto = block_scan(sh, w, &total, sh.part);
  if (f.p < 1.0) {
    if (need == 0) {
      const double c = ceil(f.p * (double)total);
      need = c < 1.0 ? 1 : (uint64_t)c;
    }
    if (upto - w >= need) w = 0;
  }
  if (f.least > 0.f && tid > 0 && !(row.exact(x) >= (double)f.least)) w = 0;
  if (on) sh.sums[0][at] = w;
  __syncthreads();
  w = sh.sums[0][tid];
  const uint64_t run = block_scan(sh, w, &total, sh.part);
  const uint64_t target = target_of(f, total);
  if (run > target && run - w <= target) write(sh.list_i[tid], total);
}

// Draws from the slices' tokens in `cut`.
template <typename S, typename R, typename W>
__device__ void draw(const S& src, const Cluster& cl, Shared& sh, const R& row, const Filter& f,
                     const Cut& cut, W&& write) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t large = 0;
  int ties = 0;
  auto add = [&](float, uint64_t w, bool valid) { large += valid ? w : 0; };
  const bool some = cut.ties != ~(uint64_t)0;  // of the tokens equal to cut.x
  const uint64_t small =
      some ? each_weight<false, true>(src, row, cut, sh.queue[warp], &ties, add)
      : cut.x == Cut::kNone ? each_weight<true, false>(src, row, cut, sh.queue[warp], &ties, add)
                            : each_weight<false, false>(src, row, cut, sh.queue[warp], &ties, add);
  const uint64_t mine = warp_sum64(small + large);
  ties = (int)__reduce_add_sync(0xffffffffu, (unsigned)ties);
  const uint64_t each_w = some ? row.weight(cut.x) : 0;
  __syncthreads();
  if (lane == 0) {
    sh.part[warp] = mine;
    sh.ties[warp] = ties;
  }
  __syncthreads();
  uint64_t here = 0, here_ties = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    here += sh.part[w];
    here_ties += sh.ties[w];
  }
  if ((int)threadIdx.x < cl.size) {
    cl.of(&sh, threadIdx.x)->slot[2][cl.rank] = here;
    cl.of(&sh, threadIdx.x)->slot[3][cl.rank] = here_ties;
  }
  cl.sync();  // (nothing is exchanged any more: a CTA may leave)
  // the ties that are kept go to the first CTAs that have any
  uint64_t before = 0, total = 0, left = cut.ties, my_left = 0;
  for (int r = 0; r < cl.size; ++r) {
    const uint64_t n = sh.slot[3][r], kept = min(n, left);
    const uint64_t w = sh.slot[2][r] - (n - kept) * each_w;
    if (r < cl.rank) before += w;
    if (r == cl.rank) {
      here = w;
      my_left = left;
    }
    total += w;
    left -= kept;
  }
  const uint64_t target = target_of(f, total);
  if (target < before || target >= before + here) return;
  // this CTA: the warp whose share it is, then a thread per vector of that share
  uint64_t run = before;
  int w = 0;
  for (; w < kWarps - 1; ++w) {
    const uint64_t n = sh.ties[w], kept = min(n, my_left);
    const uint64_t c = sh.part[w] - (n - kept) * each_w;
    if (run + c > target) break;
    run += c;
    my_left -= kept;
  }
  const int per = (src.count + kWarps - 1) / kWarps, end = min(src.count, (w + 1) * per);
  for (int v0 = w * per; v0 < end && run <= target; v0 += kThreads) {
    const int v = v0 + threadIdx.x;
    float x[S::N];
    if (v < end) {
      src.get(v, x);
    } else {
#pragma unroll
      for (int e = 0; e < S::N; ++e) x[e] = -INFINITY;
    }
    uint64_t rank = 0, all_ties = 0;  // of this thread's first tie
    if (some) {
#pragma unroll
      for (int e = 0; e < S::N; ++e) rank += x[e] == cut.x;
      const uint64_t n = rank;
      rank = block_scan(sh, rank, &all_ties, sh.walk) - n;
    }
    uint64_t c[S::N], s = 0, all;
#pragma unroll
    for (int e = 0; e < S::N; ++e) {
      const bool tie = some && x[e] == cut.x;
      c[e] = cut.has(x[e]) && !(tie && rank >= my_left) ? row.weight(x[e]) : 0;
      rank += tie;
      s += c[e];
    }
    uint64_t at = run + block_scan(sh, s, &all, sh.walk) - s;
#pragma unroll
    for (int e = 0; e < S::N; ++e) {
      if (at <= target && target < at + c[e]) write(src.index(v) + e, total);
      at += c[e];
    }
    run += all;
    my_left -= min(my_left, all_ties);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ SampleArgs a) {
  extern __shared__ uint4 held[];
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Cluster cl;
  cl.size = (int)cg::this_cluster().num_blocks();
  cl.rank = (int)cg::this_cluster().block_rank();
  constexpr int G = kDropped<T>;
  const int64_t r = blockIdx.x / cl.size;
  // every CTA of the cluster has to run before another writes to its slots
  if (cl.size > 1) cg::this_cluster().barrier_arrive();

  // this CTA's slice of the row, in 16-byte vectors of aligned addresses
  Slice<T> sl;
  sl.row = static_cast<const T*>(a.logits) + r * a.ld;
  sl.V = a.V;
  const int skew = (int)(reinterpret_cast<uintptr_t>(sl.row) & 15) / (int)sizeof(T);
  const int vectors = (skew + a.V + Slice<T>::N - 1) / Slice<T>::N;
  const int v0 = min(cl.rank * a.slice, vectors);
  sl.count = min(a.slice, vectors - v0);
  sl.base = v0 * Slice<T>::N - skew;
  sl.held = nullptr;

  // hold it, and find the largest logit
  float top = -INFINITY;
#pragma unroll 4
  for (int v = tid; v < sl.count; v += kThreads) {
    const Vec16<T> x = sl.fetch(v);
    if (a.resident) held[v] = *reinterpret_cast<const uint4*>(&x);
#pragma unroll
    for (int e = 0; e < Slice<T>::N; ++e) top = fmaxf(top, to_f32(x.v[e]));  // (not NaN)
  }
  for (int i = tid; i < kTable; i += kThreads) sh.table[i] = exp2((double)i / kTable);
  if (a.resident) sl.held = held;
  const uint32_t mine = __reduce_max_sync(0xffffffffu, key_of<G>(top));
  if (lane == 0) sh.part[warp] = mine;
  __syncthreads();
  uint32_t top_key = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) top_key = max(top_key, (uint32_t)sh.part[i]);
  if (cl.size > 1) cg::this_cluster().barrier_wait();
  cl.gather(sh, 0, top_key);
  for (int i = 0; i < cl.size; ++i) top_key = max(top_key, (uint32_t)sh.slot[0][i]);

  float t = a.temperature ? a.temperature[r] : a.temperature_v;
  if (t > 1e30f) t = 1e30f;  // (all but uniform: floor stays finite)
  Filter f;
  f.k = a.top_k ? a.top_k[r] : a.top_k_v;
  const float p = a.top_p ? a.top_p[r] : a.top_p_v;
  f.p = p < 1.f ? (double)p : 1.0;  // NaN: off
  f.least = a.min_p ? a.min_p[r] : a.min_p_v;
  f.u = a.u[r];
  if (top_key == 0 || !(t > 0.f) || f.k == 1 || f.least > 1.f) {
    // the first token of the order: the lowest index with the largest logit
    int first = 0x7fffffff;
    const float x_top = top_key == 0 ? NAN : value_of<G>(top_key);
    each(sl, [&](const float* x, int v) {
#pragma unroll
      for (int e = 0; e < Slice<T>::N; ++e)
        if (x[e] == x_top) first = min(first, sl.index(v) + e);
    });
    first = __reduce_min_sync(0xffffffffu, first);
    __syncthreads();
    if (lane == 0) sh.part[warp] = (uint64_t)first;
    __syncthreads();
    for (int i = 0; i < kWarps; ++i) first = min(first, (int)sh.part[i]);
    cl.gather(sh, 1, (uint64_t)first);
    for (int i = 0; i < cl.size; ++i) first = min(first, (int)sh.slot[1][i]);
    if (cl.rank == 0 && tid == 0) {
      a.id[r] = top_key == 0 ? -1 : (int64_t)first;
      a.logprob[r] = top_key == 0 ? -INFINITY : 0.f;
    }
    return;  // every exchange is done
  }
  Row<G> row;
  Cut cut;
  if (!row.set(value_of<G>(top_key), t, sh.table)) cut.x = row.top;

  auto write = [&](int i, uint64_t total) {
    const float x = to_f32(sl.row[i]);
    const double z = x == row.top ? 0.0 : ((double)x - (double)row.top) * row.inv_t;
    a.id[r] = i;
    a.logprob[r] = (float)(z - log((double)total / kOne));
  };
  // Each cut's first histogram; what lies from the first one's bin up may fit the
  // list.
  auto listed = [&](float x, uint64_t need) {
    const int n = collect(sl, cl, sh, fmaxf(x, cut.x));
    if (n >= 0 && cl.rank == 0) draw_sorted(sh, row, f, n, need, write);
    return n >= 0;  // nothing of the other CTAs is needed any more
  };
  float x_least = Cut::kNone;  // of min-p; once it is known:
  auto cut_least = [&] {
    if (!(x_least > cut.x)) return;
    cut.x = x_least;
    cut.ties = ~(uint64_t)0;
  };
  Search q = {kLowest<G>, top_key, 0, 0, 0, false, false, 0};
  const bool by_count = f.k > 0 && f.k < a.V;
  uint64_t excess = 0;
  if (by_count) {
    q.need = (uint64_t)f.k;
    narrow<false, kNear>(sl, cl, sh, row, cut, q, 0.0, 0);
    if (!q.whole) {
      const bool near = !q.beyond;
      if (near && q.above + q.in_bin <= kList && listed(value_of<G>(q.lo), 0)) return;
      if (!near) narrow<false, kFar>(sl, cl, sh, row, cut, q, 0.0, 0);
      cut = finish<false>(sl, cl, sh, row, cut, q);
      excess = (q.in_bin - cut.ties) * row.weight(cut.x);
    }
  }
  if (f.p < 1.0) {
    q = {kLowest<G>, top_key, 0, 0, q.round, false, false, 0};
    narrow<true, kNear>(sl, cl, sh, row, cut, q, f.p, excess);
    if (!q.whole) {
      const bool near = !q.beyond;
      uint32_t least = 0;
      if (f.least > 0.f) {
        least = least_key<G>(sh, row, f.least, top_key);
        x_least = value_of<G>(least);
      }
      // The list is tried where it is likely to hold what is left.  Never, against
      // by these rules: the first, 64 peaked rows of 151936, top-p 0.95 and min-p 0.2,
      // 65.4 us / 60.7 (in vain, 37 flat rows of 32003, min-p 0.02, 28.4 / 29.6); the
      // second, one peaked row, top-p 0.9, 20.6 / 16.5, 64 at temperature 0.3 36.7 /
      // 28.8.  96 in place of 24 tries it in vain (64 flat rows, top-p 0.5, 105.6 /
      // 93.0), 6 takes the same times as 24.
      if (least > q.hi) {  // min-p ends before the bin that top-p ends in
        cut_least();
        if (!by_count && q.above <= (uint64_t)(kList * kOne * (double)f.least) &&
            listed(cut.x, q.need))
          return;
      } else {
        // (a bin of this width with some dozens of tokens has too many above it)
        if (!by_count && near && q.in_bin <= 24 * row.weight(value_of<G>(q.hi)) &&
            listed(value_of<G>(q.lo), q.need))
          return;
        if (!near) narrow<true, kFar>(sl, cl, sh, row, cut, q, f.p, excess);
        cut = finish<true>(sl, cl, sh, row, cut, q);
      }
    }
  }
  if (f.least > 0.f) {
    if (x_least == Cut::kNone) x_least = value_of<G>(least_key<G>(sh, row, f.least, top_key));
    cut_least();
  }
  draw(sl, cl, sh, row, f, cut, write);
}

// CTAs per row.  Few rows: sixteen or eight, so that a row's passes are short (a
// cluster is placed within a GPC, so more than 32 rows of eight would queue).
// More rows: four; with 256 rows of 151936 logits, four take 98 us (bf16, all
// tokens open) and 271 us (top-p 0.95), eight 121 and 314 us, one 114 and 481
// us.  At least 2048 tokens to a CTA, at most kMaxSlice.
template <typename T>
int launch(SampleArgs a, int64_t rows, cudaStream_t st) {
  constexpr int N = 16 / (int)sizeof(T);
  const int64_t vectors = ((int64_t)a.V + 2 * N - 2) / N;  // whatever the rows' skew
  const int most = rows <= 8 ? 16 : rows <= 32 ? 8 : 4;
  int size = 1;
  while (size < most && (int64_t)a.V >= 4096 * size) size *= 2;
  while (size < kMaxCluster && (vectors + size - 1) / size * N > kMaxSlice) size *= 2;
  a.slice = (int)((vectors + size - 1) / size);
  a.resident = (size_t)a.slice * 16 <= kMaxResident;
  const size_t smem = a.resident ? (size_t)a.slice * 16 : 0;
  auto kernel = sample_kernel<T>;
  static PerDevice<cudaError_t> attr;
  ML_CHECK_CUDA(attr.get([&] {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)kMaxResident);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    return e;
  }), "sample");
  ML_CHECK_ARG(rows * size < ((int64_t)1 << 31), "sample: too many rows");
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3((unsigned)(rows * size));
  lc.blockDim = dim3(kThreads);
  lc.dynamicSmemBytes = smem;
  lc.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)size;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  lc.attrs = at;
  lc.numAttrs = 1;
  ML_CHECK_CUDA(cudaLaunchKernelEx(&lc, kernel, a), "sample");
  return ML_OK;
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
  SampleArgs a = {};
  a.logits = logits;
  a.ld = ld;
  a.V = (int)vocab;
  a.u = uniform;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.temperature_v = temperature_value;
  a.top_p_v = top_p_value;
  a.min_p_v = min_p_value;
  a.top_k_v = top_k_value;
  a.id = id;
  a.logprob = logprob;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (logits_dtype == ML_DTYPE_F32) return launch<float>(a, rows, st);
  if (logits_dtype == ML_DTYPE_BF16) return launch<__nv_bfloat16>(a, rows, st);
  return launch<__half>(a, rows, st);
}
