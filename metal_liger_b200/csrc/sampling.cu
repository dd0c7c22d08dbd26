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
// summed as integers: W = round(2^43 w), which keeps V <= 2^20 of them below
// 2^63 and is exact in any order.  Where w < e^-17 it comes from the fp32
// exponential (off by under 2^-19 of it, which is 2^-43 of the largest), above
// from the fp64 one.
//
// A cluster of CTAs holds a row in shared memory, so HBM is read once; every
// step is then a pass over the CTA's slice and an exchange of a few words
// through distributed shared memory.  The kept set is a prefix of the order and
// is found by selection, not by sorting: a histogram over the distance to the
// largest logit, of counts (top-k) or weights (top-p), gives the bin that the
// prefix ends in, histograms over that bin's keys narrow it to one key (one or
// two more for 16-bit logits), and the tokens equal to that key are cut by
// index.  The draw adds up kept weights by CTA, warp and lane in index order.
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
constexpr size_t kMaxResident = 200 * 1024;

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

// Unsigned order of the key = order of the logits, masked ones 0.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x > -INFINITY)) return 0;  // NaN and -inf
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 -> +0: equal logits, equal keys
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t kLowest = 0x00800000u;  // of the lowest finite value
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// What the weights and bins of a row are computed with.
struct Row {
  uint32_t top_key;
  float top, inv_t_f;
  double inv_t;

  __device__ __forceinline__ double exact(float x) const {
    return x == top ? 1.0 : exp(((double)x - (double)top) * inv_t);
  }
  __device__ __forceinline__ uint64_t weight(float x) const {
    if (x == top) return (uint64_t)kOne;  // also where both are +inf
    const float z = (x - top) * inv_t_f;
    if (!(z >= -31.f)) return 0;  // under half of 2^-43 (or x far below a top of +inf)
    if (z < -17.f) return __float2uint_rn(__expf(z) * (float)kOne);
    return (uint64_t)__double2ll_rn(exact(x) * kOne);
  }
};

// Which tokens an earlier cut has left: key > cut, or equal and index < end.
struct Cut {
  uint32_t key = 0;
  int end = 0;
  __device__ __forceinline__ bool has(uint32_t k, int i) const {
    return k > key || (k == key && i < end && k != 0);
  }
};

struct Shared {
  uint32_t hist[2][3][kBins];      // 15-bit parts of the sums, two in turn
  uint64_t sums[kBins];            // over the cluster
  uint64_t slot[8][kMaxCluster];   // one exchange each
  uint64_t part[kWarps];
  uint64_t above;
  int bin, found;
  uint32_t key[2];
};

// A CTA's view of its slice: `vec(v)` is 16-byte vector v of the slice, whose
// first token has index `base + v * N`; tokens outside the row read as -inf.
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
  __device__ __forceinline__ Vec16<T> vec(int v) const {
    if (held == nullptr) return fetch(v);
    Vec16<T> r;
    *reinterpret_cast<uint4*>(&r) = held[v];
    return r;
  }
  // Calls f(x, key, index) for the tokens of this warp's share of the slice;
  // lanes interleave by vector, so a lane's tokens ascend.
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
    const int per = (count + kWarps - 1) / kWarps, warp = threadIdx.x >> 5;
    const int end = min(count, (warp + 1) * per);
    for (int v = warp * per + (threadIdx.x & 31); v < end; v += 32) {
      const Vec16<T> r = vec(v);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float x = to_f32(r.v[e]);
        f(x, key_of(x), base + v * N + e);
      }
    }
  }
};

__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
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

// Adds to one bin at a time, runs of equal bins in a register.
struct Adder {
  uint32_t (*hist)[kBins];
  int bin = -1;
  uint64_t sum = 0;

  __device__ __forceinline__ void flush() {
    if (bin < 0) return;
    const uint32_t lo = (uint32_t)sum & 0x7fff, mid = (uint32_t)(sum >> 15) & 0x7fff,
                   hi = (uint32_t)(sum >> 30);
    if (lo) atomicAdd(&hist[0][bin], lo);
    if (mid) atomicAdd(&hist[1][bin], mid);
    if (hi) atomicAdd(&hist[2][bin], hi);
  }
  __device__ __forceinline__ void add(int b, uint64_t v) {
    if (b == bin) {
      sum += v;
    } else {
      flush();
      bin = b;
      sum = v;
    }
  }
};

// The first index past the `want`-th token (in index order) of those that
// `value` counts, or past the first whose running sum exceeds `want` (OVER):
// by CTA, then warp, then lane.  Returns that token's index in every CTA; -1
// where the values do not reach that far.  `total`: the sum over the cluster.
template <bool OVER, typename T, typename F>
__device__ int locate(const Slice<T>& sl, const Cluster& cl, Shared& sh, int step, double want,
                      F&& value, uint64_t* total_out, double (*want_of)(uint64_t, double)) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t mine = 0;
  sl.each([&](float x, uint32_t key, int i) { mine += value(x, key, i); });
  mine = warp_sum64(mine);
  __syncthreads();
  if (lane == 0) sh.part[warp] = mine;
  if (threadIdx.x == 0) sh.found = -1;
  __syncthreads();
  uint64_t here = 0, upto = 0;  // of the CTA, before this warp
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) upto += sh.part[w];
    here += sh.part[w];
  }
  cl.gather(sh, step, here);
  uint64_t before = 0, total = 0;
  for (int r = 0; r < cl.size; ++r) {
    if (r < cl.rank) before += sh.slot[step][r];
    total += sh.slot[step][r];
  }
  *total_out = total;
  const double target = want_of(total, want);
  auto reached = [&](uint64_t s) { return OVER ? (double)s > target : (double)s >= target; };
  uint64_t run = before + upto;
  if (mine > 0 && !reached(run) && reached(run + mine)) {
    // one warp of the cluster: walk its share
    const int per = (sl.count + kWarps - 1) / kWarps, end = min(sl.count, (warp + 1) * per);
    for (int v0 = warp * per; v0 < end; v0 += 32) {
      const int v = v0 + lane;
      uint64_t w[Slice<T>::N], s = 0;
      Vec16<T> r;
      if (v < end) r = sl.vec(v);
#pragma unroll
      for (int e = 0; e < Slice<T>::N; ++e) {
        const float x = to_f32(r.v[e]);
        w[e] = v < end ? value(x, key_of(x), sl.base + v * Slice<T>::N + e) : 0;
        s += w[e];
      }
      uint64_t incl = s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t c = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += c;
      }
      uint64_t at = run + incl - s;
      const bool hit = s > 0 && !reached(at) && reached(at + s);
      if (hit) {
        for (int e = 0; e < Slice<T>::N; ++e) {
          if (w[e] > 0 && reached(at + w[e])) {
            sh.found = sl.base + v * Slice<T>::N + e;
            break;
          }
          at += w[e];
        }
      }
      if (__any_sync(0xffffffffu, hit)) break;
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  __syncthreads();
  return sh.found;
}

// The prefix of the tokens in `in` whose values (counts or weights) first
// reach `need` (WEIGHT: p of their sum), as a cut.
template <bool WEIGHT, typename T>
__device__ Cut select(const Slice<T>& sl, const Cluster& cl, Shared& sh, const Row& row,
                      const Cut& in, bool all, uint64_t need, double p, int step, int& round) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // counts: bins of 1/16 over 32; weights: of 1/32 over 16, in units of t
  const float per = WEIGHT ? row.inv_t_f * 32.f : 16.f;
  auto distance = [&](float x) { return min(__float2int_rz((row.top - x) * per), kBins - 1); };
  uint32_t lo = kLowest, hi = row.top_key;  // the keys still in question
  uint64_t above = 0;
  int shift = -1;                     // -1: bins of distance
  while (true) {
    uint32_t (*hist)[kBins] = sh.hist[round & 1];
    ++round;
#pragma unroll
    for (int i = 0; i < 3; ++i) hist[i][tid] = 0;
    __syncthreads();
    Adder add{hist};
    sl.each([&](float x, uint32_t key, int i) {
      if (key < lo || key > hi || !(all || in.has(key, i))) return;
      const uint64_t v = WEIGHT ? row.weight(x) : 1;
      if (v) add.add(shift < 0 ? distance(x) : (int)((hi - key) >> shift), v);
    });
    add.flush();
    cl.sync();
    {
      // a thread per bin of this CTA's share and CTA that counted it
      const int r = tid % cl.size, bin = cl.rank * (kBins / cl.size) + tid / cl.size;
      const Shared* o = cl.of(&sh, r);
      const uint32_t (*h)[kBins] = o->hist[(round - 1) & 1];
      uint64_t v = h[0][bin] + ((uint64_t)h[1][bin] << 15) + ((uint64_t)h[2][bin] << 30);
      for (int o2 = cl.size / 2; o2 > 0; o2 >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o2);
      cl.of(&sh, r)->sums[bin] = v;
    }
    if (tid == 0) sh.bin = -1;
    cl.sync();
    const uint64_t s = sh.sums[tid];
    uint64_t incl = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t c = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += c;
    }
    if (lane == 31) sh.part[warp] = incl;
    __syncthreads();
    uint64_t total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) incl += sh.part[w];
      total += sh.part[w];
    }
    if (shift < 0) {
      if (WEIGHT) {
        const double f = ceil(p * (double)total);
        need = f < 1.0 ? 1 : (uint64_t)f;
      }
      if (need >= total) {  // nothing to cut, or by rounding all of it
        Cut c = in;
        if (all) {
          c.key = 1;
          c.end = 0x7fffffff;
        }
        return c;
      }
    }
    if (above + incl >= need && above + incl - s < need) {
      sh.bin = tid;
      sh.above = above + incl - s;
    }
    __syncthreads();
    const int bin = sh.bin;
    above = sh.above;
    __syncthreads();
    if (shift < 0) {
      // The keys of a bin of distances are neighbours: find the first and last
      // (distances fall as keys grow) by 32-way search, a warp for each.
      if (warp < 2) {
        // smallest key in [lo, hi] with distance <= bin (warp 0) / < bin (warp 1)
        uint32_t a = lo, b = hi + 1;  // the answer lies in [a, b]
        while (a < b) {
          const uint32_t step_k = (b - a + 31) / 32;
          const uint64_t k = (uint64_t)a + (uint64_t)step_k * lane;
          bool ok = k >= b;
          if (!ok) {
            const int d = distance(value_of((uint32_t)k));
            ok = warp == 0 ? d <= bin : d < bin;
          }
          const unsigned m = __ballot_sync(0xffffffffu, ok);
          const int f = m ? __ffs(m) - 1 : 32;
          const uint64_t top_k = (uint64_t)a + (uint64_t)step_k * f;
          const uint32_t nb = top_k < b ? (uint32_t)top_k : b;
          const uint32_t na = f == 0 ? a : (uint32_t)((uint64_t)a + (uint64_t)step_k * (f - 1) + 1);
          a = f == 0 ? nb : na;
          b = nb;
        }
        if (lane == 0) sh.key[warp] = a;
      }
      __syncthreads();
      lo = sh.key[0];
      hi = sh.key[1] - 1;
      __syncthreads();
    } else {
      const uint32_t h = hi - ((uint32_t)bin << shift);
      const uint32_t span = (1u << shift) - 1;
      lo = h - lo > span ? h - span : lo;
      hi = h;
    }
    if (lo == hi) break;
    const int bits = 32 - __clz(hi - lo);
    shift = bits > 9 ? bits - 9 : 0;
  }
  // the tokens equal to the key: as many as are still needed, lowest index first
  const uint64_t each = WEIGHT ? row.weight(value_of(lo)) : 1;
  const uint64_t want = (need - above + each - 1) / each;
  uint64_t ties;
  const int at = locate<false>(
      sl, cl, sh, step, (double)want,
      [&](float, uint32_t key, int i) -> uint64_t { return key == lo && (all || in.has(key, i)); },
      &ties, [](uint64_t, double w) { return w; });
  // (every CTA learns it: only one found it)
  cl.gather(sh, step + 1, (uint64_t)(int64_t)at);
  Cut c;
  c.key = lo;
  c.end = 0;
  for (int r = 0; r < cl.size; ++r) c.end = max(c.end, (int)(int64_t)sh.slot[step + 1][r] + 1);
  return c;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ SampleArgs a) {
  extern __shared__ uint4 held[];
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Cluster cl;
  cl.size = (int)cg::this_cluster().num_blocks();
  cl.rank = (int)cg::this_cluster().block_rank();
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

  // hold it; the first token of the order: largest key, lowest index
  uint64_t best = 0;
#pragma unroll 4
  for (int v = tid; v < sl.count; v += kThreads) {
    const Vec16<T> x = sl.fetch(v);
    if (a.resident) held[v] = *reinterpret_cast<const uint4*>(&x);
#pragma unroll
    for (int e = 0; e < Slice<T>::N; ++e) {
      const uint32_t i = (uint32_t)(sl.base + v * Slice<T>::N + e);
      const uint64_t c = ((uint64_t)key_of(to_f32(x.v[e])) << 32) | ~i;
      if (c > best) best = c;
    }
  }
  if (a.resident) sl.held = held;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t c = __shfl_xor_sync(0xffffffffu, best, o);
    if (c > best) best = c;
  }
  if (lane == 0) sh.part[warp] = best;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i)
    if (sh.part[i] > best) best = sh.part[i];
  if (cl.size > 1) cg::this_cluster().barrier_wait();
  cl.gather(sh, 0, best);
  for (int i = 0; i < cl.size; ++i)
    if (sh.slot[0][i] > best) best = sh.slot[0][i];

  const float t = a.temperature ? a.temperature[r] : a.temperature_v;
  const int64_t k = a.top_k ? a.top_k[r] : a.top_k_v;
  const float p = a.top_p ? a.top_p[r] : a.top_p_v;
  const float least = a.min_p ? a.min_p[r] : a.min_p_v;
  Row row;
  row.top_key = (uint32_t)(best >> 32);
  const int first = (int)~(uint32_t)best;
  if (row.top_key == 0 || !(t > 0.f) || k == 1 || least > 1.f) {
    if (cl.rank == 0 && tid == 0) {
      a.id[r] = row.top_key == 0 ? -1 : first;
      a.logprob[r] = row.top_key == 0 ? -INFINITY : 0.f;
    }
    cl.sync();  // no CTA leaves while another may still write to its slots
    return;
  }
  row.top = value_of(row.top_key);
  row.inv_t = 1.0 / (double)t;
  row.inv_t_f = (float)row.inv_t;

  Cut cut;
  bool all = true;  // no cut yet
  int round = 0;
  if (k > 0 && k < a.V) {
    cut = select<false>(sl, cl, sh, row, cut, all, (uint64_t)k, 0.0, 1, round);
    all = false;
  }
  if (p < 1.f) {
    cut = select<true>(sl, cl, sh, row, cut, all, 0, (double)p, 3, round);
    all = false;
  }
  // min-p: the smallest key whose weight is large enough, by 32-way search
  uint32_t least_key = 1;
  if (least > 0.f) {
    if (warp == 0) {
      uint32_t lo = kLowest, hi = row.top_key;  // the answer lies in [lo, hi]: the largest qualifies
      while (lo < hi) {
        const uint32_t step = (hi - lo + 31) / 32;
        const uint64_t q = (uint64_t)lo + (uint64_t)step * lane;
        const bool ok = q >= hi || row.exact(value_of((uint32_t)q)) >= (double)least;
        const unsigned m = __ballot_sync(0xffffffffu, ok);
        const int f = m ? __ffs(m) - 1 : 32;
        const uint64_t top = (uint64_t)lo + (uint64_t)step * f;
        const uint32_t nh = top < hi ? (uint32_t)top : hi;
        lo = f == 0 ? nh : (uint32_t)((uint64_t)lo + (uint64_t)step * (f - 1) + 1);
        hi = nh;
      }
      if (lane == 0) sh.key[0] = lo;
    }
    __syncthreads();
    least_key = sh.key[0];
  }
  auto kept = [&](float x, uint32_t key, int i) -> uint64_t {
    return key >= least_key && (all || cut.has(key, i)) ? row.weight(x) : 0;
  };
  const float uf = a.u[r];
  uint64_t total;
  const int id = locate<true>(
      sl, cl, sh, 5, uf > 0.f ? (double)uf : 0.0, kept, &total,
      [](uint64_t sum, double u) { return u * (double)sum; });
  auto write = [&](int i) {
    const float x = to_f32(sl.row[i]);
    const double z = x == row.top ? 0.0 : ((double)x - (double)row.top) * row.inv_t;
    a.id[r] = i;
    a.logprob[r] = (float)(z - log((double)total / kOne));
  };
  if (id >= 0 && tid == 0) write(id);
  if (!(uf < 1.f) || (double)uf * (double)total >= (double)total) {
    // u at or past 1 (or rounded to it): the last kept token
    int last = -1;
    sl.each([&](float x, uint32_t key, int i) {
      if (key != 0 && kept(x, key, i) > 0) last = i;
    });
    last = __reduce_max_sync(0xffffffffu, last);
    __syncthreads();
    if (lane == 0) sh.part[warp] = (uint64_t)(int64_t)last;
    __syncthreads();
    for (int i = 0; i < kWarps; ++i) last = max(last, (int)(int64_t)sh.part[i]);
    cl.gather(sh, 6, (uint64_t)(int64_t)last);
    for (int i = 0; i < cl.size; ++i) last = max(last, (int)(int64_t)sh.slot[6][i]);
    if (cl.rank == 0 && tid == 0) write(last);
  }
  cl.sync();
}

// CTAs per row: enough for two per SM, each with at least 2048 tokens, at most
// kMaxSlice, and 16-byte vectors that fit shared memory twice per SM.
template <typename T>
int launch(SampleArgs a, int64_t rows, cudaStream_t st) {
  constexpr int N = 16 / (int)sizeof(T);
  const int64_t vectors = ((int64_t)a.V + 2 * N - 2) / N;  // whatever the rows' skew
  int size = 1;
  while (size < 8 && rows * size < 2 * num_sms() && (int64_t)a.V >= 4096 * size) size *= 2;
  while (size < 8 && (vectors + size - 1) / size * 16 > 100 * 1024) size *= 2;
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
