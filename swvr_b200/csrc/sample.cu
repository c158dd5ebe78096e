// Sampling of one token per row with temperature, top-k, top-p and min-p from given uniform numbers.
//
// Definition, in real arithmetic, for a row x of V scores and T > 0:  w_i = exp((x_i - max x) / T).  Order
// the tokens by falling x, equal ones by rising index.  top_k keeps the first k; top_p keeps a token while
// the weight before it is below p times the weight that top_k left; min_p keeps w_i >= m.  The token
// is the first, in index order over the kept ones, whose running weight exceeds u times the total.  T <= 0:
// the largest score, the lowest index among equals.  -inf and NaN scores have no weight.
//
// What makes the result that of 64 bits rather than of some summation order: weights are 64-bit fixed
// point, 2^44 for the largest (2^(62 - log2 V) where V is past 2^18), so sums are exact in any order, by any number of
// threads.
//
// A row is a cluster of 1 .. 8 CTAs, each with a contiguous share of the scores.  They are read from global memory in
// every pass: after the first they are in L2, and shared memory full of scores would leave one CTA an SM (256 rows of 128256
// bf16 then took 92 us; now 47).  What bounds it: at many rows the first pass (29 of the 47 us for 66 MB; FMAs in
// pairs, more loads in flight or loads ahead of the work did not shorten it) and the rows left open (below); at few rows the chain of cluster barriers and L2
// round trips, some 6 us a row whatever its length (1 row of 152064 fp32, top-k and top-p: 12 us; 16 rows, top-p 0.9: 20 us;
// 300 rows of 10007 with all three filters, one round of CTAs: 29 us).
//
// The usual filters leave few tokens, and those are found without a weight or a bin for every score:
//   1. the largest score, and each thread's largest; for a top-p without top-k, and where there is no filter, the weight of all;
//   2. a score that every token which may be kept reaches: for top-k, the k-th of the threads' largest scores (k tokens
//      are at least that large, and few more are, as long as k is well below the number of threads); for a top-p
//      without top-k, the one at which the threads' largest scores alone make up p of the row's weight (so what
//      is kept lies above); min-p knows its own;
//   3. the tokens that reach it are gathered in one CTA, ordered by (score, index), cut by prefix sums, and u is
//      looked up in the running weight by index.
// Otherwise (no filter, a wide nucleus, long runs of equal scores) thresholds come from a histogram over kBins
// bins below the largest score and from `boundary`, which splits the threshold's bin by the order of
// (score, index) until kList members are left; a last pass over all scores sums the kept weights per warp, in
// index order, and the warp whose range holds u rescans it.
//
// Sums over all scores (the row's weight for top-p, the last pass) are first taken with fp32 weights, a quarter of the
// instructions, and where a row needs the sums of all its scores they come out of the pass that finds the largest: weights
// are taken relative to a power of two, so a sum moves to a larger one exactly.  x / T in octaves is split
// into an integer and a rest |f| <= 0.55; 2^f is off by 0.6 2^-24 (roundings of f) + 4 2^-24 (ex2), sums of eight, in a tree, by 3 2^-24,
// and the fixed point itself (V weights of half a unit, V up to 2^20) by up to 2 2^-24, relatively: no partial sum is off by more than
// d = 10 2^-24 of the total (rough_error).  Where what is decided lies more than that from its border (2 d: both the
// running weight and the total may be off) the fixed-point sums would decide the same; otherwise, a row in a hundred,
// they are taken.
#include <cooperative_groups.h>

#include <cfloat>
#include <cmath>

#include "common.cuh"
#include "ptx.cuh"
#include "sample_sums.cuh"
#include "tc.cuh"

namespace swvr {
namespace sample {

namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 1024, kList = 1024;
constexpr int kBinsPer = kBins / kThreads;
constexpr float kReach = 31.5f;  // e^-31.2 2^44 = 1/2: weights further below the largest score than 31.5 T round to 0
constexpr int kRoughOne = 40;    // fp32 sums are kept in units of 2^-40 of a power of two near the largest weight

struct Setting {  // one value for all rows, or one per row
  const void* ptr;
  int dt;  // of ptr: a float dtype, or 32 / 64 for integers
  double value;
};

struct Params {
  int64_t N, V, ld;
  const void* x;
  int dt;
  Setting T, p, m;
  const void* k_ptr;
  int k_bits;
  int64_t k;
  const void* u;
  int u_dt;
  int64_t* token;
  float* logprob;
  int share;      // scores per CTA, a multiple of 32
  int lg_one;     // log2 of the fixed-point weight of the largest score: 44 or less
  bool aligned;   // rows start on 16-byte boundaries
  int64_t row0;   // first row of x among the rows of the settings, u and the outputs
  int stage;      // 0: all rows, to the end; 1: those that need fixed-point sums are left open; 2: the open ones
};
constexpr int64_t kOpen = -2;

__device__ __forceinline__ double setting(const Setting& s, int64_t row) { return s.ptr ? load_d(s.ptr, s.dt, row) : s.value; }

// The total order: larger is earlier.  Scores order as unsigned integers once negative ones are
// complemented; the index breaks ties, lowest first.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float score_of(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ u64 place_of(float x, uint32_t index) {
  return (static_cast<u64>(order_of(x)) << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ uint32_t index_of(u64 place) { return 0xffffffffu - static_cast<uint32_t>(place); }  // of the low half

template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 warp_max(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w > v ? w : v;
  }
  return v;
}
// Inclusive prefix sum over the warp.
__device__ __forceinline__ u64 warp_scan(u64 v) {
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  return v;
}

// Tokens at or ahead of a place.
struct Cut {
  float x;
  uint32_t index;
  __device__ __forceinline__ explicit Cut(u64 place) : x(place ? score_of(static_cast<uint32_t>(place >> 32)) : -INFINITY),
                                                       index(index_of(place)) {}
  __device__ __forceinline__ bool keeps(float v, uint32_t i) const { return v > x || (v == x && i <= index); }
};

struct Shared {
  u64 mass_all[kBins];
  uint32_t count_all[kBins];
  uint32_t count[kBins], mass_lo[kBins], mass_hi[kBins];
  u64 list[kList], list_w[kList];
  double root[64];        // 2^(j / 64 + lg_one)
  u64 part[kWarps];       // per-warp results of a block reduction or scan
  u64 slot[14];           // values other CTAs of the cluster read, each written once
  u64 found[3];           // boundary bin, and count or weight before it
  uint32_t n_list;        // read by the cluster's other CTAs
  uint32_t n_kept;        // by this CTA alone

  __device__ __forceinline__ void add_mass(int b, u64 w) {
    const uint32_t lo = static_cast<uint32_t>(w), old = atomicAdd(&mass_lo[b], lo);
    const uint32_t hi = static_cast<uint32_t>(w >> 32) + (old + lo < old ? 1u : 0u);
    if (hi) atomicAdd(&mass_hi[b], hi);
  }
  __device__ __forceinline__ u64 mass(int b) const { return (static_cast<u64>(mass_hi[b]) << 32) | mass_lo[b]; }
};

// A float as a double by its bits (a conversion runs at an eighth of the rate).  0 and subnormals become some 2^-127: off by
// less than 2^-126, for both scores of a difference.
__device__ __forceinline__ double widen(float x) {
  const uint32_t b = __float_as_uint(x);
  return __hiloint2double(static_cast<int>((((b >> 3) & 0x0fffffffu) + 0x38000000u) | (b & 0x80000000u)),
                          static_cast<int>(b << 29));
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ void set_lowest(float* v) { *v = -INFINITY; }
__device__ __forceinline__ void set_lowest(__nv_bfloat16* v) { *v = __ushort_as_bfloat16(0xff80); }
__device__ __forceinline__ void set_lowest(__half* v) { *v = __ushort_as_half(0xfc00); }
// NaN never wins; -0 equals +0
template <typename T>
__device__ __forceinline__ float to_score(T v) {
  const float f = to_float(v);
  return f != f ? -INFINITY : f + 0.f;
}

// fp32 weights: 2^(x c), c = log2(e) / T.
constexpr float kMagic = 12582912.f;  // 1.5 2^23: adding it rounds to an integer, which the low bits then hold
struct Octaves {
  float c, c_lo;  // c in two parts
  float low;      // -2^20 / c: scores below it (and -inf and NaN) count as it

  __device__ __forceinline__ explicit Octaves(double cd)
      : c(static_cast<float>(cd)), c_lo(static_cast<float>(cd - c)), low(-1048576.f / c) {}
  // the nearest integer to x c, plus kMagic's bits
  __device__ __forceinline__ int place(float x) const { return __float_as_int(fmaf(fmaxf(x, low), c, kMagic)); }
  // 2^(x c) over 2^(the integer of place `ref`), at least some 2^-125 and at most 2^64 for x up to 64 octaves above ref
  __device__ __forceinline__ float weight(float x, int ref) const {
    x = fmaxf(x, low);
    const float t = fmaf(x, c, kMagic);
    const float f = fmaf(x, c_lo, fmaf(x, c, kMagic - t));
    const int k = max(__float_as_int(t) - ref, -125);
    return __int_as_float(__float_as_int(ex2(f)) + k * (1 << 23));
  }
  // the sum over a pack of scores
  template <int VEC, typename P>
  __device__ __forceinline__ double pack(const P& p, int ref) const {
    float v[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = weight(to_float(p.e[e]), ref);
    return static_cast<double>(tree_sum<VEC>(v));
  }
};

struct Row {
  Octaves oct;
  int ref;        // fp32 weights are relative to 2^(the integer of this place: the largest score's)
  bool rough_ok;  // they are within their bound
  float top;      // the largest score
  double top_d, c64;  // top, and 64 log2(e) / T
  double invT;
  int lg_one;
  float reach;    // kReach T
  float floor;    // scores below have no weight; above -inf
  float per_bin;  // bins per unit of score
  const double* root;  // 2^(j / 64 + lg_one), j < 64

  __device__ __forceinline__ float rough(float x) const { return oct.weight(x, ref); }
  // 2^-40 of 2^(the integer of ref) in units of 2^-lg_one of the largest weight
  __device__ __forceinline__ double unit() const {
    return ldexp(exp2((ref - __float_as_int(kMagic)) - top_d * (c64 / 64)), lg_one - kRoughOne);
  }
  __device__ __forceinline__ bool live(float x) const { return x >= floor; }  // not NaN either
  // exp((x - top) / T) 2^lg_one, rounded.  With y = 64 log2(e) (x - top) / T = n + f, |f| <= 1/2:
  // 2^(y / 64) = 2^(n / 64) e^(f ln 2 / 64), the first factor from a table of 64, the second a polynomial of
  // degree 4 (remainder 2^-44.6), in doubles.  Adding 1.5 2^52 rounds y to n, adding 2^52 rounds the result.
  // No branch: several of a thread's scores are in flight at once.
  __device__ __forceinline__ u64 weight(float x) const {
    constexpr double kRound = 6755399441055744.0, a1 = 0.6931471805599453 / 64;
    const double dx = widen(x) - top_d;
    const double m = fma(dx, c64, kRound);
    const int n = __double2loint(m);
    const double f = fma(dx, c64, -(m - kRound));
    double q = fma(f, a1 * a1 * a1 * a1 / 24, a1 * a1 * a1 / 6);
    q = fma(f, q, a1 * a1 / 2);
    q = fma(f, q, a1);
    q = fma(f, q, 1.0);
    double v = root[n & 63] * q;
    v = __hiloint2double(__double2hiint(v) + ((n & ~63) << 14), __double2loint(v));  // n >> 6 added to the exponent
    const u64 w = static_cast<u64>(__double_as_longlong(v + 4503599627370496.0)) & 0xfffffffffffffull;
    return live(x) ? w : 0ull;
  }
  // a score d below the largest, or a little further; above -inf
  __device__ __forceinline__ float below(float d) const { return score_of(max(order_of(top - d), order_of(-INFINITY) + 3) - 2); }
  // rises as x falls: subtraction, product and conversion are all monotone
  __device__ __forceinline__ int bin(float x) const {
    return x == top ? 0 : min(kBins - 1, static_cast<int>((top - x) * per_bin));
  }
};

// This CTA's scores.
template <typename T>
struct Scores {
  static constexpr int VEC = 16 / sizeof(T);
  const T* x;      // this CTA's first score
  bool aligned;
  int n;
  uint32_t first;  // its index in the row

  struct alignas(16) Pack {
    T e[VEC];
  };
  // VEC scores from i on (i a multiple of VEC), as they are; -inf past `end`
  __device__ __forceinline__ Pack load(int i, int end) const {
    Pack p;
    if (aligned && i + VEC <= end) {
      p = *reinterpret_cast<const Pack*>(x + i);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        if (i + k < end) p.e[k] = x[i + k];
        else set_lowest(&p.e[k]);
      }
    }
    return p;
  }
  // f(pack, index) for the packs at i0, i0 + step, ... before end, U loads at a time (an L2 round trip is some 700
  // cycles; more than f has registers for costs more than it hides)
  template <int U, typename F>
  __device__ __forceinline__ void packs(int i0, int end, int step, F f) const {
    for (int i = i0; i < end; i += U * step) {
      Pack q[U];
#pragma unroll
      for (int j = 0; j < U; ++j) q[j] = load(i + j * step, end);
#pragma unroll
      for (int j = 0; j < U; ++j) f(q[j], i + j * step);
    }
  }
  // f(score, index within the CTA) for every score, in no order; NaN and -inf are left out, -0 is +0
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    packs<1>(threadIdx.x * VEC, n, kThreads * VEC, [&](const Pack& p, int i) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float v = to_score(p.e[k]);
        if (v != -INFINITY) f(v, i + k);
      }
    });
  }
};

// Sum / maximum over the block, to every thread.
__device__ __forceinline__ uint32_t block_max32(uint32_t v, Shared& s) {
  v = __reduce_max_sync(0xffffffffu, v);
  __syncthreads();
  if (threadIdx.x % 32 == 0) s.part[threadIdx.x / 32] = v;
  __syncthreads();
  const int lane = threadIdx.x % 32;
  return __reduce_max_sync(0xffffffffu, lane < kWarps ? static_cast<uint32_t>(s.part[lane]) : 0u);
}
__device__ __forceinline__ u64 block_max(u64 v, Shared& s) {
  v = warp_max(v);
  __syncthreads();
  if (threadIdx.x % 32 == 0) s.part[threadIdx.x / 32] = v;
  __syncthreads();
  u64 r = s.part[0];
  for (int i = 1; i < kWarps; ++i) r = s.part[i] > r ? s.part[i] : r;
  return r;
}
__device__ __forceinline__ u64 block_sum(u64 v, Shared& s) {
  v = warp_sum(v);
  __syncthreads();
  if (threadIdx.x % 32 == 0) s.part[threadIdx.x / 32] = v;
  __syncthreads();
  u64 r = 0;
  for (int i = 0; i < kWarps; ++i) r += s.part[i];
  return r;
}
// Exclusive prefix sum over the block's threads, in thread order.
__device__ __forceinline__ u64 block_scan(u64 v, Shared& s) {
  const u64 inc = warp_scan(v);
  __syncthreads();
  if (threadIdx.x % 32 == 31) s.part[threadIdx.x / 32] = inc;
  __syncthreads();
  u64 r = inc - v;
  for (int i = 0; i < static_cast<int>(threadIdx.x) / 32; ++i) r += s.part[i];
  return r;
}

constexpr int kMaxCluster = 8;

// One value of every CTA of the cluster: the loads are in flight together (a remote one takes some 600 cycles).
template <typename F>
__device__ __forceinline__ void read_all(cg::cluster_group& cl, u64 (&v)[kMaxCluster], F address) {
  const unsigned C = cl.num_blocks();
#pragma unroll
  for (unsigned c = 0; c < kMaxCluster; ++c) v[c] = c < C ? *address(c) : 0;
}

// A block's value made the cluster's, through slot `at` (each used once): the largest, or the sum.
template <bool kSum>
__device__ __forceinline__ u64 cluster_join(u64 v, int at, Shared& s, cg::cluster_group& cl) {
  if (cl.num_blocks() == 1) return v;
  if (threadIdx.x == 0) s.slot[at] = v;
  cl.sync();
  const unsigned lane = threadIdx.x % 32;
  const u64 o = lane < cl.num_blocks() ? *cl.map_shared_rank(&s.slot[at], lane) : 0;
  return kSum ? warp_sum(o) : warp_max(o);
}

__device__ __forceinline__ void clear_bins(bool masses, Shared& s) {
  for (int b = threadIdx.x; b < kBins; b += kThreads) {
    s.count[b] = 0;
    if (masses) s.mass_lo[b] = s.mass_hi[b] = 0;
  }
  __syncthreads();
}

// Adds up the CTAs' histograms: each CTA sums its share of the bins and hands the sums to all.
__device__ __forceinline__ void merge_bins(bool masses, Shared& s, cg::cluster_group& cl) {
  const unsigned C = cl.num_blocks(), me = cl.block_rank();
  cl.sync();  // every CTA's bins are complete, and nobody reads the sums of the pass before
  for (int b = me * (kBins / C) + threadIdx.x; b < static_cast<int>((me + 1) * (kBins / C)); b += kThreads) {
    u64 v[kMaxCluster];
    read_all(cl, v, [&](unsigned r) { return cl.map_shared_rank(&s.count[b], r); });
    u64 sum = 0;
#pragma unroll
    for (unsigned r = 0; r < kMaxCluster; ++r) sum += v[r];
    for (unsigned r = 0; r < C; ++r) *cl.map_shared_rank(&s.count_all[b], r) = static_cast<uint32_t>(sum);
    if (masses) {
      sum = 0;
      read_all(cl, v, [&](unsigned r) { return cl.map_shared_rank(&s.mass_lo[b], r); });
#pragma unroll
      for (unsigned r = 0; r < kMaxCluster; ++r) sum += v[r];
      read_all(cl, v, [&](unsigned r) { return cl.map_shared_rank(&s.mass_hi[b], r); });
#pragma unroll
      for (unsigned r = 0; r < kMaxCluster; ++r) sum += v[r] << 32;
      for (unsigned r = 0; r < C; ++r) *cl.map_shared_rank(&s.mass_all[b], r) = sum;
    }
  }
  cl.sync();
}

// The bin b with before(b) < goal <= before(b) + bin(b), before: the sum of the bins ahead of it.  By
// counts or by weights.  found[0] = kBins when the bins sum to less.
template <bool kByCount>
__device__ __forceinline__ void find_bin(u64 goal, Shared& s) {
  u64 v[kBinsPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kBinsPer; ++i) {
    v[i] = kByCount ? s.count_all[threadIdx.x * kBinsPer + i] : s.mass_all[threadIdx.x * kBinsPer + i];
    sum += v[i];
  }
  if (threadIdx.x == 0) s.found[0] = kBins;
  u64 before = block_scan(sum, s);
#pragma unroll
  for (int i = 0; i < kBinsPer; ++i) {
    if (before < goal && goal <= before + v[i]) {
      s.found[0] = threadIdx.x * kBinsPer + i;
      s.found[1] = before;
    }
    before += v[i];
  }
  __syncthreads();
}

// The weight, or the number, in the bins ahead of b.
template <bool kByCount>
__device__ __forceinline__ u64 ahead_of(int b, Shared& s) {
  u64 w = 0;
  for (int i = threadIdx.x; i < b; i += kThreads) w += kByCount ? s.count_all[i] : s.mass_all[i];
  return block_sum(w, s);
}

// What top-p compares running weights with: ceil(p total), at least 1 so that one token stays.
__device__ __forceinline__ u64 nucleus(double top_p, u64 total) {
  const double g = ceil(fmax(top_p, 0.0) * static_cast<double>(total));
  return g < 1.0 ? 1ull : min(static_cast<u64>(g), total);
}

// The running weight that the chosen token is the first to reach: floor(u total) + 1, at most total.
__device__ __forceinline__ u64 goal_of(double u, u64 total) {
  const double at = floor((u > 0.0 ? u : 0.0) * static_cast<double>(total));
  return at >= static_cast<double>(total) ? total : min(static_cast<u64>(at) + 1ull, total);
}

// Bitonic sort of the list's first n entries (a power of two), largest key first; weights move along.  A warp's
// 32 pairs span 64 entries while the stride is at most 32: only wider steps need the block's barrier.
__device__ __forceinline__ void sort_list(int n, Shared& s) {
  for (int size = 2; size <= n; size <<= 1)
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      for (int t = threadIdx.x; t < n / 2; t += kThreads) {
        const int i = 2 * t - (t & (stride - 1)), j = i + stride;
        const u64 a = s.list[i], b = s.list[j];
        if ((a < b) == ((i & size) == 0)) {
          s.list[i] = b;
          s.list[j] = a;
          const u64 w = s.list_w[i];
          s.list_w[i] = s.list_w[j];
          s.list_w[j] = w;
        }
      }
      // the next step's stride: half of this one, or this size's after stride 1
      if (stride > 32 || (stride == 1 ? size : stride / 2) > 32) __syncthreads();
      else __syncwarp();
    }
  __syncthreads();
}

// The token from a list of m places and weights that holds every token the filters may keep (one CTA).
// [total_lo, total_hi] holds the weight that top-p refers to (total_hi = 0: that of the first k).  False when tokens are kept
// or not depending on where in the range the total lies; the list is as it was.
// Up to 256 entries are ranked by comparing each with all others (512 / m threads an entry), more are sorted.
__device__ __forceinline__ bool choose_from_list(int m, bool by_k, u64 k, bool by_p, double top_p, u64 total_lo, u64 total_hi,
                                                 u64 cut, double u, int64_t* token, float* x_token, bool* mine, Shared& s) {
  if (m <= 256) {
    int G = 1;  // lanes that share an entry
    while (2 * G * m <= kThreads && G < 16) G *= 2;
    const int i = threadIdx.x / G, g = threadIdx.x % G;
    const bool have = i < m;
    const u64 pl = have ? s.list[i] : ~0ull;
    u64 w = have ? s.list_w[i] : 0, ahead = 0;
    uint32_t rank = 0;
    if (have) {
#pragma unroll 4
      for (int j = g; j < m; j += G) {
        const u64 o = s.list[j];
        if (by_p) {
          const u64 ow = s.list_w[j];
          ahead += o > pl ? ow : 0;
        }
        rank += o > pl;
      }
    }
    for (int o = 1; o < G; o <<= 1) {
      rank += __shfl_xor_sync(0xffffffffu, rank, o);
      if (by_p) ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
    }
    if (by_k && rank >= k) w = 0;  // what is ahead of the others is unchanged: it ranks behind them
    if (by_p) {
      const u64 sum = block_sum(g == 0 ? w : 0, s);
      const u64 lo = nucleus(top_p, total_hi ? total_lo : sum), hi = nucleus(top_p, total_hi ? total_hi : sum);
      if (lo != hi && __syncthreads_or(w != 0 && ahead >= lo && ahead < hi)) return false;
      if (ahead >= lo) w = 0;
    }
    if (pl < cut || g != 0) w = 0;
    if (threadIdx.x == 0) s.n_kept = 0;  // (other CTAs may still read n_list)
    const u64 goal = goal_of(u, block_sum(w, s));  // its barriers: the list has been read, the count is 0
    if (w != 0) {  // kept ones move together
      const uint32_t j = atomicAdd(&s.n_kept, 1u);
      s.list[j] = pl;
      s.list_w[j] = w;
    }
    __syncthreads();
    const uint32_t kept = s.n_kept;
    for (uint32_t e = threadIdx.x; e < kept; e += kThreads) {
      const u64 mine_pl = s.list[e];
      const uint32_t low = static_cast<uint32_t>(mine_pl);  // complemented index: a larger one comes first
      u64 run = 0;
#pragma unroll 4
      for (uint32_t j = 0; j < kept; ++j) {
        const u64 ow = s.list_w[j];
        run += static_cast<uint32_t>(s.list[j]) > low ? ow : 0;
      }
      if (run < goal && goal <= run + s.list_w[e]) {
        *token = index_of(mine_pl);
        *x_token = score_of(static_cast<uint32_t>(mine_pl >> 32));
        *mine = true;
      }
    }
    return true;
  }
  int n = 512;
  while (n < m) n <<= 1;
  for (int i = m + threadIdx.x; i < n; i += kThreads) s.list[i] = 0, s.list_w[i] = 0;
  __syncthreads();
  constexpr int PER = kList / kThreads;
  sort_list(n, s);
  // entries of this thread: consecutive ones, so that prefix sums follow the order
  u64 w[PER], sum = 0;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int i = threadIdx.x * PER + e;
    w[e] = i < n && !(by_k && static_cast<u64>(i) >= k) ? s.list_w[i] : 0;
    sum += w[e];
  }
  u64 ahead = block_scan(sum, s), goal_p = ~0ull;
  if (by_p) {
    const u64 listed = block_sum(sum, s);
    goal_p = nucleus(top_p, total_hi ? total_lo : listed);
    const u64 hi = nucleus(top_p, total_hi ? total_hi : listed);
    if (goal_p != hi) {
      bool unsure = false;
      u64 at = ahead;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        unsure |= w[e] != 0 && at >= goal_p && at < hi;
        at += w[e];
      }
      if (__syncthreads_or(unsure)) return false;
    }
  }
  // kept ones, by index: the place with its halves exchanged orders by (index, score)
  u64 key[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int i = threadIdx.x * PER + e;
    const u64 pl = i < n ? s.list[i] : 0;
    const bool keep = w[e] != 0 && ahead < goal_p && pl >= cut;
    ahead += w[e];
    key[e] = keep ? (pl << 32) | (pl >> 32) : 0;
    if (!keep) w[e] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int i = threadIdx.x * PER + e;
    if (i < n) s.list[i] = key[e], s.list_w[i] = w[e];
  }
  __syncthreads();
  sort_list(n, s);  // complemented indices, largest first: rising index
  sum = 0;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int i = threadIdx.x * PER + e;
    w[e] = i < n ? s.list_w[i] : 0;
    sum += w[e];
  }
  ahead = block_scan(sum, s);
  const u64 goal = goal_of(u, block_sum(sum, s));
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    if (ahead < goal && goal <= ahead + w[e]) {
      const u64 kx = s.list[threadIdx.x * PER + e];
      *token = index_of(kx >> 32);
      *x_token = score_of(static_cast<uint32_t>(kx));
      *mine = true;
    }
    ahead += w[e];
  }
  return true;
}

// Gathers in CTA 0 the places and weights of the scores that reach reach_x; returns their number, which may be over
// kList (then there is no list).  Each CTA lists its own first: a remote append per token would cost a round trip each.
// reach_x is above -inf; `also` narrows further.
template <typename T, typename F>
__device__ __forceinline__ uint32_t gather(const Scores<T>& sc, const Row& row, float reach_x, F also, Shared& s,
                                           cg::cluster_group& cl) {
  constexpr int VEC = Scores<T>::VEC;
  if (threadIdx.x == 0) s.n_list = 0;
  __syncthreads();
  sc.template packs<2>(threadIdx.x * VEC, sc.n, kThreads * VEC, [&](const typename Scores<T>::Pack& p, int i) {
    float most = to_float(p.e[0]);
#pragma unroll
    for (int k = 1; k < VEC; ++k) most = fmaxf(most, to_float(p.e[k]));
    if (!(most >= reach_x)) return;  // most packs
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const float v = to_float(p.e[k]) + 0.f;
      if (v >= reach_x && also(v, i + k)) {
        const uint32_t j = atomicAdd(&s.n_list, 1u);
        if (j < kList) s.list[j] = place_of(v, sc.first + i + k);
      }
    }
  });
  cl.sync();
  u64 n[kMaxCluster];
  read_all(cl, n, [&](unsigned c) { return cl.map_shared_rank(&s.n_list, c); });
  uint32_t m = 0, before = 0;  // before: of the CTAs ahead of the one this warp copies
  const unsigned warp = threadIdx.x / 32;
#pragma unroll
  for (unsigned c = 0; c < kMaxCluster; ++c) {
    if (c == warp) before = m;
    m += static_cast<uint32_t>(n[c]);
  }
  if (m <= kList && cl.block_rank() == 0) {
    if (warp > 0 && warp < cl.num_blocks()) {
      const Shared* o = cl.map_shared_rank(&s, warp);
      uint32_t count = 0;
#pragma unroll
      for (unsigned c = 0; c < kMaxCluster; ++c)
        if (c == warp) count = static_cast<uint32_t>(n[c]);
      for (uint32_t j = threadIdx.x % 32; j < count; j += 32) s.list[before + j] = o->list[j];
    }
    __syncthreads();
    for (uint32_t j = threadIdx.x; j < m; j += kThreads) s.list_w[j] = row.weight(score_of(static_cast<uint32_t>(s.list[j] >> 32)));
    __syncthreads();
  }
  return m;
}

// The lowest kept place when tokens are kept while what is ahead of them (their number, or their weight) is
// below goal; `bin` holds the boundary and `before` is ahead of it.
template <bool kByCount, typename T>
__device__ __noinline__ u64 boundary(const Scores<T>& sc, const Row& row, int bin, u64 before, u64 goal, Shared& s,
                                     cg::cluster_group& cl) {
  u64 lo = 0, hi = ~0ull;  // places of the members still in question
  Shared* s0 = cl.map_shared_rank(&s, 0);
  auto member = [&](float x, int i) {
    if (!row.live(x) || row.bin(x) != bin) return false;
    const u64 pl = place_of(x, sc.first + i);
    return pl >= lo && pl <= hi;
  };
  while (true) {
    const uint32_t m = gather(sc, row, row.floor, member, s, cl);
    if (m <= kList) {
      if (cl.block_rank() == 0) {
        u64 low = ~0ull;
        for (int i = threadIdx.x; i < static_cast<int>(m); i += kThreads) {
          const u64 mine = s.list[i];
          u64 ahead = before;
          for (uint32_t j = 0; j < m; ++j)
            if (s.list[j] > mine) ahead += kByCount ? 1 : s.list_w[j];
          if (ahead < goal) low = mine < low ? mine : low;
        }
        low = ~block_max(~low, s);
        if (threadIdx.x == 0) s.found[0] = low;
      }
      cl.sync();
      const u64 r = s0->found[0];
      cl.sync();  // found, and the lists, are written again only after everyone has read them
      return r;
    }
    // too many for the list: split [least, most] place of the members into kBins equal ranges
    u64 least = ~0ull, most = 0;
    sc.each([&](float x, int i) {
      if (!member(x, i)) return;
      const u64 pl = place_of(x, sc.first + i);
      least = pl < least ? pl : least;
      most = pl > most ? pl : most;
    });
    least = ~block_max(~least, s);
    most = block_max(most, s);
    cl.sync();
    if (threadIdx.x == 0) s.slot[10] = least, s.slot[13] = most;
    cl.sync();
    for (unsigned r = 0; r < cl.num_blocks(); ++r) {
      const u64 a = *cl.map_shared_rank(&s.slot[10], r), b = *cl.map_shared_rank(&s.slot[13], r);
      least = a < least ? a : least;
      most = b > most ? b : most;
    }
    int shift = 0;
    while (((most - least) >> shift) >= kBins) ++shift;
    clear_bins(!kByCount, s);
    sc.each([&](float x, int i) {
      if (!member(x, i)) return;
      const int b = static_cast<int>((most - place_of(x, sc.first + i)) >> shift);
      if (kByCount) atomicAdd(&s.count[b], 1u);
      else s.add_mass(b, row.weight(x));
    });
    merge_bins(!kByCount, s, cl);
    find_bin<kByCount>(goal - before, s);
    const int b = static_cast<int>(s.found[0]);
    before += s.found[1];
    hi = most - (static_cast<u64>(b) << shift);
    const u64 width = (1ull << shift) - 1;
    lo = hi >= width ? hi - width : 0;
  }
}

// The lowest kept place of top-k and top-p, whatever they leave.
template <typename T>
__device__ __forceinline__ u64 thresholds(const Scores<T>& sc, const Row& row, bool by_k, u64 k, bool by_p, double top_p,
                                       Shared& s, cg::cluster_group& cl) {
  u64 cut = 0;
  if (by_k) {
    clear_bins(false, s);
    sc.each([&](float x, int i) {
      if (row.live(x)) atomicAdd(&s.count[row.bin(x)], 1u);
    });
    merge_bins(false, s, cl);
    find_bin<true>(k, s);
    const int b = static_cast<int>(s.found[0]);
    const u64 before = s.found[1];
    if (b < kBins) cut = boundary<true>(sc, row, b, before, k, s, cl);  // else all that have weight fit
  }
  if (by_p) {
    clear_bins(true, s);
    const Cut first_k(cut);
    sc.each([&](float x, int i) {
      if (row.live(x) && first_k.keeps(x, sc.first + i)) s.add_mass(row.bin(x), row.weight(x));
    });
    merge_bins(true, s, cl);
    const u64 goal = nucleus(top_p, ahead_of<false>(kBins, s));
    find_bin<false>(goal, s);
    const int b = static_cast<int>(s.found[0]);
    const u64 before = s.found[1];
    if (b < kBins) {
      const u64 c = boundary<false>(sc, row, b, before, goal, s, cl);
      cut = c > cut ? c : cut;
    }
  }
  return cut;
}

// The weight of this CTA's scores, in units of 2^-lg_one of the largest.
// (By value: a reference to the caller's structs would keep them in local memory.)
template <typename T>
__device__ __noinline__ u64 exact_total(const Scores<T> sc, const Row row, Shared& s) {
  u64 w = 0;
  sc.template packs<1>(threadIdx.x * Scores<T>::VEC, sc.n, kThreads * Scores<T>::VEC, [&](const typename Scores<T>::Pack& p, int) {
#pragma unroll
    for (int e = 0; e < Scores<T>::VEC; ++e) w += row.weight(to_float(p.e[e]));
  });
  return block_sum(w, s);
}
__device__ __forceinline__ u64 rough_units(double w, int octaves = 0) { return static_cast<u64>(ldexp(w, kRoughOne + octaves)); }

// Scores per warp: each has a contiguous sixteenth of its CTA's share.
template <typename T>
__device__ __forceinline__ int warp_span(const Scores<T>& sc) {
  constexpr int STEP = 32 * Scores<T>::VEC;
  return (sc.n + STEP * kWarps - 1) / (STEP * kWarps) * STEP;
}

// This thread's largest score among its warp's, and with kSum the weight of those it reads, relative to 2^(the integer of ref).
// ref follows the largest score only once that is 64 octaves above it.
template <bool kSum, typename T>
__device__ __forceinline__ void first_pass(const Scores<T>& sc, const Octaves& oct, float* t_top, double* sum, int* ref) {
  constexpr int VEC = Scores<T>::VEC, STEP = 32 * VEC;
  const int span = warp_span(sc), i0 = min(sc.n, static_cast<int>(threadIdx.x) / 32 * span), i1 = min(sc.n, i0 + span);
  float top = -INFINITY;  // (fmaxf leaves NaN out)
  double w = 0;
  int r = 0;
  sc.template packs<kSum ? 2 : 4>(i0 + static_cast<int>(threadIdx.x) % 32 * VEC, i1, STEP, [&](const typename Scores<T>::Pack& p, int) {
    float m = to_float(p.e[0]);
#pragma unroll
    for (int e = 1; e < VEC; ++e) m = fmaxf(m, to_float(p.e[e]));
    top = fmaxf(top, m);
    if constexpr (kSum) {
      const int at = oct.place(m);
      if (at - r > 64) {
        w = ldexp(w, r - at);
        r = at;
      }
      w += oct.template pack<VEC>(p, r);
    }
  });
  *t_top = top + 0.f;
  *sum = w;
  *ref = r;
}

// Weights of the scores [i0, i1) of this CTA at or ahead of the cut, summed over the warp; i0 a multiple of VEC.
template <bool kExact, typename T>
__device__ __forceinline__ u64 span_weight(const Scores<T>& sc, const Row& row, const Cut& kept, bool cut, int i0, int i1) {
  constexpr int VEC = Scores<T>::VEC, STEP = 32 * VEC;
  const int lane = threadIdx.x % 32;
  using Pack = typename Scores<T>::Pack;
  if constexpr (kExact) {
    u64 w = 0;
    sc.template packs<1>(i0 + lane * VEC, i1, STEP, [&](const Pack& p, int i) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float x = to_float(p.e[e]);
        const u64 we = row.weight(x);
        w += !cut || kept.keeps(x, sc.first + i + e) ? we : 0ull;
      }
    });
    return warp_sum(w);
  } else {
    double r = 0;
    if (!cut) {
      sc.template packs<2>(i0 + lane * VEC, i1, STEP, [&](const Pack& p, int) { r += row.oct.template pack<VEC>(p, row.ref); });
    } else {
      sc.template packs<2>(i0 + lane * VEC, i1, STEP, [&](const Pack& p, int i) {
        float v[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float x = to_score(p.e[e]);
          v[e] = kept.keeps(x, sc.first + i + e) ? row.rough(x) : 0.f;
        }
        r += static_cast<double>(tree_sum<VEC>(v));
      });
    }
    return warp_sum(rough_units(r));
  }
}

// The token from all scores at or ahead of the cut, by sums in index order: of each warp's sixteenth of the share (w, or taken
// here where there is none); where the goal falls, of sixteenths of that; then of single scores.  Rough sums: false where
// the border is too near.
constexpr u64 kNone = ~0ull;
template <bool kExact, typename T>
__device__ __forceinline__ bool sweep(const Scores<T>& sc, const Row& row, u64 cut, double u, int slot, u64 w, int64_t* token,
                                      float* x_token, bool* mine, Shared& s, cg::cluster_group& cl) {
  constexpr int VEC = Scores<T>::VEC, STEP = 32 * VEC;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const unsigned me = cl.block_rank();
  const int span = warp_span(sc);
  const Cut kept(cut);
  if (w == kNone) w = span_weight<kExact>(sc, row, kept, cut != 0, min(sc.n, warp * span), min(sc.n, (warp + 1) * span));
  __syncthreads();
  if (lane == 0) s.part[warp] = w;
  __syncthreads();
  u64 own = 0;
  for (int i = 0; i < kWarps; ++i) own += s.part[i];
  if (threadIdx.x == 0) {
    s.slot[slot] = own;
    s.found[2] = 0;
  }
  cl.sync();
  u64 ahead = 0, total = 0, v[kMaxCluster];
  read_all(cl, v, [&](unsigned c) { return cl.map_shared_rank(&s.slot[slot], c); });
#pragma unroll
  for (unsigned c = 0; c < kMaxCluster; ++c) {
    if (c < me) ahead += v[c];
    total += v[c];
  }
  const u64 goal = goal_of(u, total), margin = kExact ? 0 : 2 * rough_error(total);
  if (ahead < goal && goal <= ahead + own) {  // this CTA's share holds it
    int part = 0;
    while (part < kWarps - 1 && ahead + s.part[part] < goal) ahead += s.part[part++];
    const int sub = (span + STEP * kWarps - 1) / (STEP * kWarps) * STEP, end = min(sc.n, (part + 1) * span);
    const int i0 = min(end, part * span + warp * sub), i1 = min(end, i0 + sub);
    w = span_weight<kExact>(sc, row, kept, cut != 0, i0, i1);
    __syncthreads();
    if (lane == 0) s.part[warp] = w;
    __syncthreads();
    for (int i = 0; i < warp; ++i) ahead += s.part[i];
    if (ahead < goal && goal <= ahead + s.part[warp]) {
      for (int i = i0 + lane * VEC; i - lane * VEC < i1; i += STEP) {
        const typename Scores<T>::Pack p = sc.load(i, i1);
        float x[VEC];
        u64 we[VEC], sum = 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          x[e] = to_score(p.e[e]);
          const u64 wx = kExact ? row.weight(x[e]) : static_cast<u64>(ldexpf(row.rough(x[e]), kRoughOne));
          we[e] = x[e] != -INFINITY && kept.keeps(x[e], sc.first + i + e) ? wx : 0;
          sum += we[e];
        }
        const u64 inc = warp_scan(sum);
        const uint32_t reached = __ballot_sync(0xffffffffu, ahead + inc >= goal);
        if (reached) {
          if (lane == __ffs(reached) - 1) {
            u64 at = ahead + inc - sum;
            bool found = false;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              if (!found && at + we[e] >= goal) {
                found = true;
                if (kExact || (at + margin < goal && goal + margin < at + we[e])) {
                  *mine = true;
                  *token = sc.first + i + e;
                  *x_token = x[e];
                  if (!kExact) *cl.map_shared_rank(&s.found[2], 0) = 1;
                }
              }
              at += we[e];
            }
          }
          break;
        }
        ahead += __shfl_sync(0xffffffffu, inc, 31);
      }
    }
  }
  if (kExact) return true;
  cl.sync();
  return *cl.map_shared_rank(&s.found[2], 0) != 0;
}

struct Choice {
  uint32_t token;
  float x;
  bool mine;  // this thread found it
};

// Thresholds of any width, and the sweeps: out of the way of the kernel that finds few tokens.
template <typename T>
__device__ __noinline__ Choice choose_among_many(const Scores<T> sc, const Row row, bool by_k, u64 k, bool by_p, double top_p, u64 cut,
                                                 double u, Shared& s) {
  cg::cluster_group cl = cg::this_cluster();
  if (by_k || by_p) {
    const u64 c = thresholds(sc, row, by_k, k, by_p, top_p, s, cl);
    cut = c > cut ? c : cut;
  }
  int64_t token = 0;
  float x = 0.f;
  bool mine = false;
  if (!row.rough_ok || !sweep<false>(sc, row, cut, u, 11, kNone, &token, &x, &mine, s, cl))
    sweep<true>(sc, row, cut, u, 5, kNone, &token, &x, &mine, s, cl);
  return {static_cast<uint32_t>(token), x, mine};
}

// kFilters: some row may have top-k, top-p or min-p; without, the kernel needs fewer registers.
template <typename T, bool kFilters>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const Params p) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Shared& s = *reinterpret_cast<Shared*>(smem_raw);
  cg::cluster_group cl = cg::this_cluster();
  const unsigned C = cl.num_blocks(), me = cl.block_rank();
  const int64_t r = blockIdx.x / C, row_id = p.row0 + r;
  const int tid = threadIdx.x;
  if (!kFilters && p.stage == 2 && p.token[row_id] != kOpen) return;  // the whole cluster: the token is written at the end
  const int64_t first = static_cast<int64_t>(me) * p.share;
  Scores<T> sc;
  sc.x = static_cast<const T*>(p.x) + r * p.ld + first;
  sc.aligned = p.aligned;
  sc.first = static_cast<uint32_t>(first);
  sc.n = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(p.share), p.V - first)));
  if (tid < 64) s.root[tid] = exp2(tid / 64.0 + p.lg_one);
  // settings, while the scores are on their way
  double temp = setting(p.T, row_id);
  const bool greedy = !(temp > 0.0);
  temp = greedy ? 1.0 : fmax(temp, 1e-300);
  const double top_p = setting(p.p, row_id), min_p = setting(p.m, row_id), u = load_d(p.u, p.u_dt, row_id);
  const int64_t k = p.k_ptr ? (p.k_bits == 64 ? static_cast<const int64_t*>(p.k_ptr)[row_id]
                                              : static_cast<int64_t>(static_cast<const int32_t*>(p.k_ptr)[row_id]))
                            : p.k;
  const bool by_k = kFilters && k > 0 && k < p.V, by_p = kFilters && top_p < 1.0, by_m = kFilters && min_p > 0.0;
  const double lm = by_m && !greedy ? log(min(min_p, 1.0)) : 0.0, invT = 1.0 / temp;

  // ---------------------------------------------------------------- the largest score, and the weight of all
  const Octaves oct(1.4426950408889634 * invT);
  float t_top;  // of this thread
  double t_sum;
  int t_ref;
  const bool by_all = !greedy && (kFilters ? by_p && !by_k : p.stage != 2);  // the weight of all scores is asked for
  if (by_all) first_pass<true>(sc, oct, &t_top, &t_sum, &t_ref);
  else first_pass<false>(sc, oct, &t_top, &t_sum, &t_ref);
  Row row{oct};
  row.top = score_of(static_cast<uint32_t>(cluster_join<false>(block_max32(order_of(t_top), s), 0, s, cl)));
  if (p.V == 0 || row.top == -INFINITY) {  // nothing to choose from
    if (me == 0 && tid == 0) {
      p.token[row_id] = -1;
      if (p.logprob) p.logprob[row_id] = -INFINITY;
    }
    cl.sync();
    return;
  }
  row.invT = invT;
  row.c64 = 64 * 1.4426950408889634 * row.invT;
  row.top_d = widen(row.top);
  row.lg_one = p.lg_one;
  row.reach = kReach * static_cast<float>(temp);
  row.floor = fmaxf(row.top - row.reach, -FLT_MAX);
  row.per_bin = static_cast<float>(kBins) / row.reach;
  row.root = s.root;
  row.ref = oct.place(row.top);
  row.rough_ok = p.V <= kRoughMost && oct.c > 1e-25f && oct.c < 1e25f && fabsf(row.top) * oct.c < 524288.f;
  const u64 weight = by_all && row.rough_ok ? rough_units(t_sum, t_ref - row.ref) : 0;  // of the scores that this thread read

  int64_t token = 0;
  float x_token = row.top;
  bool mine = false;  // the thread that writes the result
  if (greedy) {
    u64 pl = 0;
    sc.each([&](float x, int i) {
      if (x == row.top) pl = max(pl, place_of(x, sc.first + i));
    });
    token = index_of(cluster_join<false>(block_max(pl, s), 1, s, cl));
    mine = me == 0 && tid == 0;
  } else {
    u64 cut = 0;  // kept: place >= cut
    if (by_m) {
      // the lowest score with exp((x - top) / T) >= min_p: the nearest float to the root, or a neighbour
      const double top = row.top;
      auto keeps = [&](uint32_t o) { return (static_cast<double>(score_of(o)) - top) * row.invT >= lm || score_of(o) == row.top; };
      uint32_t o = order_of(static_cast<float>(top + temp * lm));
      const uint32_t o_top = order_of(row.top), o_low = order_of(-INFINITY) + 1;
      o = min(max(o, o_low), o_top);
      for (int i = 0; i < 8 && o > o_low && keeps(o - 1); ++i) --o;
      for (int i = 0; i < 8 && o < o_top && !keeps(o); ++i) ++o;
      cut = static_cast<u64>(o) << 32;
    }
    // -------------------------------------------------------------- few tokens left
    bool done = false;
    if (by_m || (by_k ? static_cast<u64>(k) <= min(kThreads * C / 2, kList / 2) : by_p)) {
      u64 lo = 0, hi = 0;  // the row's weight, for top-p without top-k
      bool exact = false, few = true;
      float reach_x = row.floor;  // a score that every token which may be kept reaches
      if (by_k || by_p) {
        clear_bins(!by_k, s);
        if (row.live(t_top)) {
          atomicAdd(&s.count[row.bin(t_top)], 1u);
          if (!by_k) s.add_mass(row.bin(t_top), row.weight(t_top));
        }
        if (!by_k) {
          if (row.rough_ok) {
            const u64 w = cluster_join<true>(block_sum(weight, s), 2, s, cl);
            const double unit = row.unit();
            lo = static_cast<u64>(static_cast<double>(w - rough_error(w)) * unit);
            hi = static_cast<u64>(static_cast<double>(w + rough_error(w)) * unit) + 1;
          } else {
            exact = true;
            lo = hi = cluster_join<true>(exact_total(sc, row, s), 2, s, cl);
          }
        }
        merge_bins(!by_k, s, cl);
        if (by_k) find_bin<true>(static_cast<u64>(k), s);
        else find_bin<false>(nucleus(top_p, hi), s);
        const int b = static_cast<int>(s.found[0]);
        few = b < kBins;  // else the threads' largest scores do not make it up
        // the lower end of that bin, less what rounding may have moved
        if (b < kBins - 1) reach_x = fmaxf(reach_x, row.below((b + 1) / row.per_bin * 1.000001f));
      }
      if (by_m && !(by_k && by_p)) reach_x = fmaxf(reach_x, Cut(cut).x);  // (top-p after top-k weighs the first k)
      if (few) {
        const uint32_t m = gather(sc, row, reach_x, [](float, int) { return true; }, s, cl);
        few = m <= kList;
        for (int slot = 3; few; ++slot) {
          bool sure = true;
          if (me == 0)
            sure = choose_from_list(static_cast<int>(m), by_k, static_cast<u64>(k), by_p, top_p, lo, hi, cut, u, &token,
                                    &x_token, &mine, s);
          done = true;
          if (by_k || !by_p || exact) break;
          if (tid == 0 && me == 0) s.slot[slot] = sure;
          cl.sync();
          if (*cl.map_shared_rank(&s.slot[slot], 0) != 0) break;
          exact = true;
          lo = hi = cluster_join<true>(exact_total(sc, row, s), 9, s, cl);
        }
      }
    }
    // -------------------------------------------------------------- many
    if (!done) {
      if constexpr (kFilters) {
        const Choice c = choose_among_many(sc, row, by_k, static_cast<u64>(k), by_p, top_p, cut, u, s);
        token = c.token;
        x_token = c.x;
        mine = c.mine;
      } else if (!row.rough_ok || p.stage == 2 || !sweep<false>(sc, row, 0, u, 11, warp_sum(weight), &token, &x_token, &mine, s, cl)) {
        if (p.stage == 1) {
          if (me == 0 && tid == 0) p.token[row_id] = kOpen;
          cl.sync();
          return;
        }
        sweep<true>(sc, row, 0, u, 5, kNone, &token, &x_token, &mine, s, cl);
      }
    }
  }
  if (mine) p.token[row_id] = token;
  if (p.logprob) {
    // log softmax(x / T) of the token over the whole row
    const u64 all = cluster_join<true>(exact_total(sc, row, s), 12, s, cl);
    if (mine)
      p.logprob[row_id] = static_cast<float>((x_token == row.top ? 0.0 : (static_cast<double>(x_token) - row.top) * row.invT) -
                                             log(ldexp(static_cast<double>(all), -row.lg_one)));
  }
  cl.sync();  // no CTA leaves while another may read its shared memory
}

// ------------------------------------------------------------------ host
template <typename T>
static cudaError_t launch_c(Params p, int C, bool filters, cudaStream_t st) {
  p.share = static_cast<int>(round_up(ceil_div(std::max<int64_t>(p.V, 1), C), 32));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(p.N * C), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = sizeof(Shared);
  cfg.stream = st;
  static_assert(sizeof(Shared) <= 48 * 1024, "more needs cudaFuncSetAttribute");
  ProfScope ps(kProfSample, st);
  return cudaLaunchKernelEx(&cfg, filters ? sample_kernel<T, true> : sample_kernel<T, false>, p);
}

template <typename T>
static cudaError_t launch_t(Params p, cudaStream_t st) {
  static_assert(kMaxCluster == 8, "cluster sizes below");
  const bool filters = p.k_ptr || p.k > 0 || p.p.ptr || p.p.value < 1.0 || p.m.ptr || p.m.value > 0.0;
  // Two CTAs fit an SM: one round of them (64 rows of 128256 fp32, top-k: 17 us with 256 CTAs, 32 with 512).  Rows that need
  // fixed-point sums would hold up the others where a row has few CTAs: without filters they are left to a second launch that
  // gives each of them as many as its length allows (256 rows of 128256 bf16: 53 us in one launch of 512 CTAs, 47 in two; 55 where a
  // few clusters look for the open rows and one may get two of them).
  int wide = 1;
  while (wide < kMaxCluster && p.V > 2048 * wide) wide *= 2;
  int C = wide;
  while (C > 1 && C * p.N > 2 * kNumSMsB200) C /= 2;
  p.aligned = (reinterpret_cast<uintptr_t>(p.x) & 15u) == 0 && (p.ld * sizeof(T)) % 16 == 0;
  p.lg_one = lg_one_of(p.V);
  p.stage = !filters && C < wide && p.V <= kRoughMost ? 1 : 0;
  cudaError_t e = launch_c<T>(p, C, filters, st);
  if (e != cudaSuccess || p.stage == 0) return e;
  p.stage = 2;
  return launch_c<T>(p, wide, false, st);
}

static cudaError_t launch(const Params& p, cudaStream_t st) {
  if (p.dt == SWVR_F32) return launch_t<float>(p, st);
  if (p.dt == SWVR_BF16) return launch_t<__nv_bfloat16>(p, st);
  return launch_t<__half>(p, st);
}

static bool float_dtype(int dt) { return dt >= SWVR_F32 && dt <= SWVR_F16; }

static int params(const swvr_sampling* o, int64_t N, int64_t V, Params* p) {
  if (!o) return fail(SWVR_ERR_INVALID_ARGUMENT, "sampling is NULL");
  if (N < 0 || V < 0) return fail(SWVR_ERR_INVALID_ARGUMENT, "negative size");
  if (V >= (1ll << 31) || N >= (1ll << 28)) return fail(SWVR_ERR_UNSUPPORTED, "sizes must be below 2^31 (rows 2^28)");
  if (N > 0 && (!o->u || !o->tokens)) return fail(SWVR_ERR_INVALID_ARGUMENT, "NULL pointer");
  if (!float_dtype(o->u_dtype) || (o->temperatures && !float_dtype(o->temperatures_dtype)) ||
      (o->top_ps && !float_dtype(o->top_ps_dtype)) || (o->min_ps && !float_dtype(o->min_ps_dtype)))
    return fail(SWVR_ERR_INVALID_ARGUMENT, "unknown dtype");
  if (o->top_ks && o->top_ks_bits != 32 && o->top_ks_bits != 64)
    return fail(SWVR_ERR_INVALID_ARGUMENT, "top_ks must be 32- or 64-bit integers");
  if ((!o->temperatures && !(o->temperature >= 0.0 && std::isfinite(o->temperature))) ||
      (!o->top_ps && !(o->top_p > 0.0 && o->top_p <= 1.0)) || (!o->min_ps && !(o->min_p >= 0.0 && o->min_p <= 1.0)) ||
      (!o->top_ks && o->top_k < 0))
    return fail(SWVR_ERR_INVALID_ARGUMENT, "temperature, top_k, top_p or min_p out of range");
  *p = Params{};
  p->N = N;
  p->V = V;
  p->T = {o->temperatures, o->temperatures_dtype, o->temperature};
  p->p = {o->top_ps, o->top_ps_dtype, o->top_p};
  p->m = {o->min_ps, o->min_ps_dtype, o->min_p};
  p->k_ptr = o->top_ks;
  p->k_bits = o->top_ks_bits;
  p->k = o->top_k;
  p->u = o->u;
  p->u_dt = o->u_dtype;
  p->token = o->tokens;
  p->logprob = o->logprobs;
  return SWVR_OK;
}

// Rows whose fp32 scores are held at a time: at most 256 MiB of them, at least one row, and no more than a launch of the
// fp32 product takes.
static int64_t head_rows(const swvr_problem& p) {
  const int64_t pitch = round_up(std::max<int64_t>(p.vocab, 1), 4) * 4;
  const int64_t most = is_tc(p.compute_dtype) ? p.n_tokens : std::min(p.n_tokens, simt::kMostRows);
  return std::max<int64_t>(1, std::min<int64_t>(most, (256ll << 20) / pitch));
}

static int check_head(const swvr_problem* p) {
  if (!p) return fail(SWVR_ERR_INVALID_ARGUMENT, "problem is NULL");
  if (p->n_tokens < 0 || p->hidden < 0 || p->vocab < 0) return fail(SWVR_ERR_INVALID_ARGUMENT, "negative size");
  // (a tile's last row index fits an int)
  if (p->n_tokens >= (1ll << 28) || p->vocab > (1ll << 31) - 512 || p->hidden > (1ll << 31) - 512)
    return fail(SWVR_ERR_UNSUPPORTED, "sizes must be at most 2^31 - 512 (rows below 2^28)");
  if (p->compute_dtype != SWVR_F32 && !is_tc(p->compute_dtype))
    return fail(SWVR_ERR_UNSUPPORTED, "sampling computes in bf16, fp16 or fp32");
  if (p->bias && !float_dtype(p->bias_dtype)) return fail(SWVR_ERR_INVALID_ARGUMENT, "unknown bias dtype %d", p->bias_dtype);
  if (p->ldh < p->hidden || p->ldw < p->hidden)
    return fail(SWVR_ERR_INVALID_ARGUMENT, "row stride smaller than the row length");
  if (p->n_tokens > 0 && p->hidden > 0 && (!p->h || (p->vocab > 0 && !p->W)))
    return fail(SWVR_ERR_INVALID_ARGUMENT, "NULL input pointer");
  if (is_tc(p->compute_dtype)) {
    if (p->hidden < 8 || (p->hidden % 8) != 0 || (p->ldh % 8) != 0 || (p->ldw % 8) != 0)
      return fail(SWVR_ERR_UNSUPPORTED, "tensor-core path needs K and row strides that are multiples of 8 elements");
    if ((reinterpret_cast<uintptr_t>(p->h) | reinterpret_cast<uintptr_t>(p->W)) & 15u)
      return fail(SWVR_ERR_UNSUPPORTED, "tensor-core path needs 16-byte aligned h and W");
  }
  return SWVR_OK;
}

__global__ void add_bias_rows(float* x, int64_t N, int64_t V, int64_t ld, const void* bias, int dt) {
  for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < N * V;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x)
    x[i / V * ld + i % V] += load_f(bias, dt, i % V);
}

// Scores of rows [n0, n0 + n) into `logits`.
static int head_scores(const swvr_problem& p, int64_t n0, int64_t n, float* logits, int64_t ld, cudaStream_t st) {
  if (!is_tc(p.compute_dtype)) {
    ProfScope ps(kProfSimt, st);
    SWVR_CUDA(simt::gemm<float>(st, n, p.vocab, p.hidden, static_cast<float>(p.logit_scale),
                                static_cast<const float*>(p.h) + n0 * p.ldh, p.ldh, 1, static_cast<const float*>(p.W), 1,
                                p.ldw, 0.f, logits, SWVR_F32, ld, 1));
    if (p.bias) {
      add_bias_rows<<<static_cast<unsigned>(std::min<int64_t>(ceil_div(n * p.vocab, 256), 8 * kNumSMsB200)), 256, 0, st>>>(
          logits, n, p.vocab, ld, p.bias, p.bias_dtype);
      SWVR_CUDA(cudaGetLastError());
    }
    return SWVR_OK;
  }
  const int BN = n <= 32 ? 32 : n <= 64 ? 64 : n <= 128 ? 128 : 256;
  const char* h = static_cast<const char*>(p.h) + n0 * p.ldh * 2;
  tc::HeadMaps maps;
  SWVR_TRY(make_map(&maps.a, p.W, p.compute_dtype, p.hidden, p.vocab, p.ldw * 2, 64, 128));
  SWVR_TRY(make_map(&maps.b, h, p.compute_dtype, p.hidden, n, p.ldh * 2, 64, BN / 2));
  tc::HeadParams q{};
  q.K = static_cast<int>(p.hidden);
  q.MT = static_cast<int>(ceil_div(p.vocab, 256));
  q.BT = static_cast<int>(ceil_div(n, BN));
  q.splits = 1;
  q.per = q.BT;
  q.units = q.MT;
  q.gm = 1;
  q.N = static_cast<int>(n);
  q.V = static_cast<int>(p.vocab);
  q.scale = static_cast<float>(p.logit_scale);
  q.bias = p.bias;
  q.bias_dt = p.bias_dtype;
  q.logits = logits;
  q.ld_logits = ld;
  ProfScope ps(kProfHead, st);
  const int pairs = std::max(1, num_sms() / 2);
  SWVR_CUDA(p.compute_dtype == SWVR_BF16 ? tc::launch_head_any<true>(tc::kHeadLogits, BN, maps, q, pairs, false, st)
                                         : tc::launch_head_any<false>(tc::kHeadLogits, BN, maps, q, pairs, false, st));
  return SWVR_OK;
}

}  // namespace sample
}  // namespace swvr

extern "C" {

int swvr_sample_logits(int64_t n_rows, int64_t vocab, const void* logits, int32_t dtype, int64_t ld,
                       const swvr_sampling* sampling, void* stream) {
  sample::Params p;
  SWVR_TRY(sample::params(sampling, n_rows, vocab, &p));
  if (dtype != SWVR_F32 && dtype != SWVR_BF16 && dtype != SWVR_F16)
    return fail(SWVR_ERR_UNSUPPORTED, "sampling takes bf16, fp16 or fp32 logits");
  if (ld < vocab) return fail(SWVR_ERR_INVALID_ARGUMENT, "row stride smaller than the row length");
  if (n_rows > 0 && vocab > 0 && !logits) return fail(SWVR_ERR_INVALID_ARGUMENT, "NULL input pointer");
  if (n_rows == 0) return SWVR_OK;
  p.x = logits;
  p.dt = dtype;
  p.ld = ld;
  SWVR_CUDA(sample::launch(p, static_cast<cudaStream_t>(stream)));
  return SWVR_OK;
}

int swvr_sample_workspace_size(const swvr_problem* p, size_t* bytes) {
  SWVR_TRY(sample::check_head(p));
  if (!bytes) return fail(SWVR_ERR_INVALID_ARGUMENT, "bytes is NULL");
  *bytes = static_cast<size_t>(sample::head_rows(*p)) * round_up(std::max<int64_t>(p->vocab, 1), 4) * 4;
  return SWVR_OK;
}

int swvr_sample(const swvr_problem* p, const swvr_sampling* sampling, void* workspace, size_t workspace_bytes,
                void* stream) {
  SWVR_TRY(sample::check_head(p));
  sample::Params q;
  SWVR_TRY(sample::params(sampling, p->n_tokens, p->vocab, &q));
  if (p->n_tokens == 0) return SWVR_OK;
  size_t need = 0;
  SWVR_TRY(swvr_sample_workspace_size(p, &need));
  if (workspace_bytes < need) return fail(SWVR_ERR_WORKSPACE, "workspace %zu < required %zu", workspace_bytes, need);
  if (!workspace) return fail(SWVR_ERR_INVALID_ARGUMENT, "NULL workspace");
  if (!aligned16(workspace)) return fail(SWVR_ERR_UNSUPPORTED, "workspace not 16-byte aligned");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t rows = sample::head_rows(*p), ld = round_up(std::max<int64_t>(p->vocab, 1), 4);
  q.x = workspace;
  q.dt = SWVR_F32;
  q.ld = ld;
  for (int64_t n0 = 0; n0 < p->n_tokens; n0 += rows) {
    const int64_t n = std::min(rows, p->n_tokens - n0);
    if (p->vocab > 0) SWVR_TRY(sample::head_scores(*p, n0, n, static_cast<float*>(workspace), ld, st));
    q.N = n;
    q.row0 = n0;
    SWVR_CUDA(sample::launch(q, st));
  }
  return SWVR_OK;
}

}  // extern "C"
