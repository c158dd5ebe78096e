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
// threads.  Weights below 2^-44 of the largest are 0 (30.5 T below the maximum).
//
// A row is a cluster of 1 .. 8 CTAs, each holding a contiguous share of the scores in shared memory, so
// the scores are read from global memory once; longer rows are read again in each pass.  Both thresholds are a
// selection: one histogram pass puts the scores into 2048 bins of equal width below the maximum (count for
// top-k, weight for top-p), the bin that holds the threshold is found by a scan, and its members
// (a few hundred) are gathered in one CTA and ranked against one another.  A bin with more than
// kList members (equal scores, mostly) is split again by the 64-bit order of (score, index) until it has
// no more.  A last pass sums the kept weights per warp, in index order, and the warp whose
// range holds u rescans its range.
#include <cooperative_groups.h>

#include <cmath>

#include "common.cuh"
#include "ptx.cuh"
#include "tc.cuh"

namespace swvr {
namespace sample {

namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2048, kList = 1024;
constexpr int kBinsPer = kBins / kThreads;
constexpr float kReach = 30.5f;  // e^-30.5 < 2^-44

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
  int share;      // scores per CTA
  double one;     // 2^44 or less: the fixed-point weight of the largest score
  int64_t row0;   // first row of x among the rows of the settings, u and the outputs
};

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

struct Shared {
  u64 mass[kBins], mass_all[kBins];
  uint32_t count[kBins], count_all[kBins];
  u64 list[kList], list_w[kList];
  u64 part[2 * kWarps];   // per-warp results of a block reduction or scan
  u64 slot[12];           // values other CTAs of the cluster read, each written once
  u64 found[3];           // boundary bin, and count and weight before it
  uint32_t n_list;
};

struct Row {
  float top;      // the largest score
  double invT, one;
  float reach;    // scores further below have no weight
  float per_bin;  // bins per unit of score

  __device__ __forceinline__ bool live(float x) const { return x == top || top - x < reach; }
  __device__ __forceinline__ u64 weight(float x) const {
    if (x == top) return static_cast<u64>(one);
    if (!(top - x < reach)) return 0;
    return static_cast<u64>(exp((static_cast<double>(x) - top) * invT) * one + 0.5);
  }
  // rises as x falls: subtraction, product and conversion are all monotone
  __device__ __forceinline__ int bin(float x) const {
    return x == top ? 0 : min(kBins - 1, static_cast<int>((top - x) * per_bin));
  }
};

template <bool kHeld>
struct Scores {
  const void* x;
  int dt;
  int64_t base;  // element of x that this CTA's first score is
  const float* held;
  int n;
  uint32_t first;  // its index in the row
  __device__ __forceinline__ float raw(int i) const {
    const float v = load_f(x, dt, base + i);
    return v != v ? -INFINITY : v + 0.f;  // NaN never wins; -0 equals +0
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (kHeld) return held[i];
    else return raw(i);
  }
};

// Sum / maximum over the block, to every thread.
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

// The cluster's maximum / sum of a block value, through slot `at` (each used once).
__device__ __forceinline__ u64 cluster_max(u64 v, int at, Shared& s, cg::cluster_group& cl) {
  if (threadIdx.x == 0) s.slot[at] = v;
  cl.sync();
  u64 r = 0;
  for (unsigned i = 0; i < cl.num_blocks(); ++i) {
    const u64 o = *cl.map_shared_rank(&s.slot[at], i);
    r = o > r ? o : r;
  }
  return r;
}

// Adds up the CTAs' histograms: each CTA sums its share of the bins and hands the sums to all.
__device__ __forceinline__ void merge_bins(bool counts, bool masses, Shared& s, cg::cluster_group& cl) {
  const unsigned C = cl.num_blocks(), me = cl.block_rank();
  cl.sync();  // every CTA's bins are complete, and nobody reads the sums of the pass before
  for (int b = me * (kBins / C) + threadIdx.x; b < static_cast<int>((me + 1) * (kBins / C)); b += kThreads) {
    uint32_t c = 0;
    u64 m = 0;
    for (unsigned r = 0; r < C; ++r) {
      if (counts) c += *cl.map_shared_rank(&s.count[b], r);
      if (masses) m += *cl.map_shared_rank(&s.mass[b], r);
    }
    for (unsigned r = 0; r < C; ++r) {
      if (counts) *cl.map_shared_rank(&s.count_all[b], r) = c;
      if (masses) *cl.map_shared_rank(&s.mass_all[b], r) = m;
    }
  }
  cl.sync();
}

// The bin b with before(b) < goal <= before(b) + bin(b), before: the sum of the bins ahead of it.  By
// counts or by weights.  found[0] = kBins when the bins sum to less.
template <bool kByCount>
__device__ __forceinline__ void find_bin(u64 goal, Shared& s) {
  const int t = threadIdx.x, lane = t % 32, warp = t / 32;
  u64 v[kBinsPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kBinsPer; ++i) {
    v[i] = kByCount ? s.count_all[t * kBinsPer + i] : s.mass_all[t * kBinsPer + i];
    sum += v[i];
  }
  u64 inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  __syncthreads();
  if (lane == 31) s.part[warp] = inc;
  if (t == 0) s.found[0] = kBins;
  __syncthreads();
  u64 before = inc - sum;
  for (int i = 0; i < warp; ++i) before += s.part[i];
#pragma unroll
  for (int i = 0; i < kBinsPer; ++i) {
    if (before < goal && goal <= before + v[i]) {
      s.found[0] = t * kBinsPer + i;
      s.found[1] = before;
    }
    before += v[i];
  }
  __syncthreads();
}

// The lowest kept place when tokens are kept while what is ahead of them (their number, or their weight) is
// below goal; `bin` holds the boundary and `before` is ahead of it.  *kept: the weight of all kept.
template <bool kHeld, bool kByCount>
__device__ u64 boundary(const Scores<kHeld>& sc, const Row& row, int bin, u64 before, u64 goal, bool masses,
                        u64 mass_before, u64* kept, Shared& s, cg::cluster_group& cl) {
  u64 lo = 0, hi = ~0ull;  // places of the members still in question
  Shared* s0 = cl.map_shared_rank(&s, 0);
  while (true) {
    if (threadIdx.x == 0) s.n_list = 0;
    cl.sync();
    for (int i = threadIdx.x; i < sc.n; i += kThreads) {
      const float x = sc.at(i);
      if (!row.live(x) || row.bin(x) != bin) continue;
      const u64 pl = place_of(x, sc.first + i);
      if (pl < lo || pl > hi) continue;
      const uint32_t j = atomicAdd(&s0->n_list, 1u);
      if (j < kList) {
        s0->list[j] = pl;
        s0->list_w[j] = kByCount && !masses ? 0 : row.weight(x);
      }
    }
    cl.sync();
    const uint32_t m = *cl.map_shared_rank(&s.n_list, 0);
    if (m <= kList) {
      if (cl.block_rank() == 0) {
        u64 low = ~0ull, w_kept = 0;
        for (int i = threadIdx.x; i < static_cast<int>(m); i += kThreads) {
          const u64 mine = s.list[i];
          u64 ahead = before;
          for (uint32_t j = 0; j < m; ++j)
            if (s.list[j] > mine) ahead += kByCount ? 1 : s.list_w[j];
          if (ahead < goal) {
            low = mine < low ? mine : low;
            w_kept += s.list_w[i];
          }
        }
        const u64 lowest = ~block_max(~low, s);
        const u64 w = block_sum(w_kept, s);
        if (threadIdx.x == 0) {
          s.found[0] = lowest;
          s.found[1] = mass_before + w;
        }
      }
      cl.sync();
      const u64 r = s0->found[0];
      *kept = s0->found[1];
      cl.sync();  // found is written again only after everyone has read it
      return r;
    }
    // too many for the list: split [least, greatest] place of the members into kBins equal ranges
    u64 least = ~0ull, most = 0;
    for (int i = threadIdx.x; i < sc.n; i += kThreads) {
      const float x = sc.at(i);
      if (!row.live(x) || row.bin(x) != bin) continue;
      const u64 pl = place_of(x, sc.first + i);
      if (pl < lo || pl > hi) continue;
      least = pl < least ? pl : least;
      most = pl > most ? pl : most;
    }
    least = ~block_max(~least, s);
    most = block_max(most, s);
    cl.sync();
    if (threadIdx.x == 0) s.slot[10] = least, s.slot[11] = most;
    cl.sync();
    for (unsigned r = 0; r < cl.num_blocks(); ++r) {
      const u64 a = *cl.map_shared_rank(&s.slot[10], r), b = *cl.map_shared_rank(&s.slot[11], r);
      least = a < least ? a : least;
      most = b > most ? b : most;
    }
    int shift = 0;
    while (((most - least) >> shift) >= kBins) ++shift;
    for (int b = threadIdx.x; b < kBins; b += kThreads) s.count[b] = 0, s.mass[b] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < sc.n; i += kThreads) {
      const float x = sc.at(i);
      if (!row.live(x) || row.bin(x) != bin) continue;
      const u64 pl = place_of(x, sc.first + i);
      if (pl < lo || pl > hi) continue;
      const int b = static_cast<int>((most - pl) >> shift);
      atomicAdd(&s.count[b], 1u);
      if (masses) atomicAdd(&s.mass[b], row.weight(x));
    }
    merge_bins(true, masses, s, cl);
    find_bin<kByCount>(goal - before, s);
    const int b = static_cast<int>(s.found[0]);
    before += s.found[1];
    if (masses) {
      u64 w = 0;
      for (int i = threadIdx.x; i < b; i += kThreads) w += s.mass_all[i];
      mass_before += block_sum(w, s);
    }
    hi = most - (static_cast<u64>(b) << shift);
    const u64 width = (1ull << shift) - 1;
    lo = hi >= width ? hi - width : 0;
  }
}

template <bool kHeld>
__global__ void __launch_bounds__(kThreads) sample_kernel(const Params p) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Shared& s = *reinterpret_cast<Shared*>(smem_raw);
  float* held = reinterpret_cast<float*>(smem_raw + sizeof(Shared));
  cg::cluster_group cl = cg::this_cluster();
  const unsigned C = cl.num_blocks(), me = cl.block_rank();
  const int64_t r = blockIdx.x / C, row_id = p.row0 + r;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  Scores<kHeld> sc;
  sc.x = p.x;
  sc.dt = p.dt;
  const int64_t first = static_cast<int64_t>(me) * p.share;
  sc.base = r * p.ld + first;
  sc.held = held;
  sc.first = static_cast<uint32_t>(first);
  sc.n = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(p.share), p.V - first)));

  // ---------------------------------------------------------------- scores in, the largest
  u64 best = 0;
  for (int i = tid; i < sc.n; i += kThreads) {
    const float x = sc.raw(i);
    if constexpr (kHeld) held[i] = x;
    const u64 pl = place_of(x, sc.first + i);
    best = pl > best ? pl : best;
  }
  best = cluster_max(block_max(best, s), 0, s, cl);
  Row row;
  row.top = score_of(static_cast<uint32_t>(best >> 32));
  const uint32_t arg = 0xffffffffu - static_cast<uint32_t>(best);
  if (p.V == 0 || row.top == -INFINITY) {  // nothing to choose from
    if (me == 0 && tid == 0) {
      p.token[row_id] = -1;
      if (p.logprob) p.logprob[row_id] = -INFINITY;
    }
    cl.sync();
    return;
  }
  double T = setting(p.T, row_id);
  const bool greedy = !(T > 0.0);
  if (greedy) T = 1.0;
  row.invT = 1.0 / T;
  row.one = p.one;
  row.reach = kReach * static_cast<float>(T);
  row.per_bin = static_cast<float>(kBins) / row.reach;

  int64_t token = arg;
  float x_token = row.top;
  bool mine = me == 0 && tid == 0;  // the thread that writes the result
  if (!greedy) {
    // -------------------------------------------------------------- thresholds
    const int64_t k = p.k_ptr ? (p.k_bits == 64 ? static_cast<const int64_t*>(p.k_ptr)[row_id]
                                                : static_cast<int64_t>(static_cast<const int32_t*>(p.k_ptr)[row_id]))
                              : p.k;
    const double top_p = setting(p.p, row_id), min_p = setting(p.m, row_id);
    const bool by_k = k > 0 && k < p.V, by_p = top_p < 1.0;
    u64 cut = 0;  // kept: place >= cut
    if (by_k || by_p) {
      for (int b = tid; b < kBins; b += kThreads) s.count[b] = 0, s.mass[b] = 0;
      __syncthreads();
      for (int i = tid; i < sc.n; i += kThreads) {
        const float x = sc.at(i);
        if (!row.live(x)) continue;
        const int b = row.bin(x);
        if (by_k) atomicAdd(&s.count[b], 1u);
        if (by_p) atomicAdd(&s.mass[b], row.weight(x));
      }
      merge_bins(by_k, by_p, s, cl);
      u64 total = 0;  // what top-k leaves
      bool have_total = false;
      if (by_k) {
        find_bin<true>(static_cast<u64>(k), s);
        const int b = static_cast<int>(s.found[0]);
        if (b < kBins) {
          const u64 before = s.found[1];
          u64 w = 0;
          if (by_p) {
            for (int i = tid; i < b; i += kThreads) w += s.mass_all[i];
            w = block_sum(w, s);
          }
          cut = boundary<kHeld, true>(sc, row, b, before, static_cast<u64>(k), by_p, w, &total, s, cl);
          have_total = true;
        }
      }
      if (by_p) {
        // boundary() may have used the bins for a split: the weights of a pass before are gone, so the
        // histogram is taken again, over what top-k left
        if (have_total) {
          for (int b = tid; b < kBins; b += kThreads) s.mass[b] = 0;
          __syncthreads();
          for (int i = tid; i < sc.n; i += kThreads) {
            const float x = sc.at(i);
            if (row.live(x) && place_of(x, sc.first + i) >= cut) atomicAdd(&s.mass[row.bin(x)], row.weight(x));
          }
          merge_bins(false, true, s, cl);
        } else {
          u64 w = 0;
          for (int i = tid; i < kBins; i += kThreads) w += s.mass_all[i];
          total = block_sum(w, s);
        }
        const double goal_r = ceil(fmax(top_p, 0.0) * static_cast<double>(total));
        const u64 goal = goal_r < 1.0 ? 1ull : min(static_cast<u64>(goal_r), total);
        find_bin<false>(goal, s);
        const int b = static_cast<int>(s.found[0]);
        if (b < kBins) {
          const u64 before = s.found[1];
          u64 ignored;
          const u64 c = boundary<kHeld, false>(sc, row, b, before, goal, true, before, &ignored, s, cl);
          cut = c > cut ? c : cut;
        }
      }
    }
    if (min_p > 0.0) {
      // the lowest score with exp((x - top) / T) >= min_p: the nearest float to the root, or a neighbour
      const double lm = log(min(min_p, 1.0));
      auto keeps = [&](uint32_t o) { return (static_cast<double>(score_of(o)) - row.top) * row.invT >= lm; };
      uint32_t o = order_of(static_cast<float>(static_cast<double>(row.top) + T * lm));
      const uint32_t o_top = order_of(row.top), o_low = order_of(-INFINITY) + 1;
      o = min(max(o, o_low), o_top);
      for (int i = 0; i < 8 && o > o_low && keeps(o - 1); ++i) --o;
      for (int i = 0; i < 8 && o < o_top && !keeps(o); ++i) ++o;
      const u64 c = static_cast<u64>(o) << 32;
      cut = c > cut ? c : cut;
    }
    // -------------------------------------------------------------- the token
    const int span = (sc.n + 32 * kWarps - 1) / (32 * kWarps) * 32;  // scores per warp, contiguous
    const int i0 = min(sc.n, warp * span), i1 = min(sc.n, i0 + span);
    u64 w = 0;
    for (int i = i0 + lane; i < i1; i += 32) {
      const float x = sc.at(i);
      if (place_of(x, sc.first + i) >= cut) w += row.weight(x);
    }
    w = warp_sum(w);
    __syncthreads();
    if (lane == 0) s.part[warp] = w;
    __syncthreads();
    u64 own = 0;
    for (int i = 0; i < kWarps; ++i) own += s.part[i];
    if (tid == 0) s.slot[1] = own;
    cl.sync();
    u64 ahead = 0, total = 0;
    for (unsigned c = 0; c < C; ++c) {
      const u64 o = *cl.map_shared_rank(&s.slot[1], c);
      if (c < me) ahead += o;
      total += o;
    }
    const double u = load_d(p.u, p.u_dt, row_id);
    const double at = floor((u > 0.0 ? u : 0.0) * static_cast<double>(total));
    const u64 goal = at >= static_cast<double>(total) ? total : min(static_cast<u64>(at) + 1ull, total);
    mine = false;
    for (int i = 0; i < warp; ++i) ahead += s.part[i];
    if (ahead < goal && goal <= ahead + s.part[warp]) {  // this warp's range holds it
      for (int i = i0 + lane; i - lane < i1; i += 32) {
        const float x = i < i1 ? sc.at(i) : -INFINITY;
        const u64 wi = i < i1 && place_of(x, sc.first + i) >= cut ? row.weight(x) : 0;
        u64 inc = wi;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 up = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += up;
        }
        const uint32_t reached = __ballot_sync(0xffffffffu, ahead + inc >= goal);
        if (reached) {
          if (lane == __ffs(reached) - 1) {
            mine = true;
            token = sc.first + i;
            x_token = x;
          }
          break;
        }
        ahead += __shfl_sync(0xffffffffu, inc, 31);
      }
    }
  }
  if (mine) p.token[row_id] = token;
  if (p.logprob) {
    // log softmax(x / T) of the token over the whole row
    u64 w = 0;
    for (int i = tid; i < sc.n; i += kThreads) w += row.weight(sc.at(i));
    w = block_sum(w, s);
    if (tid == 0) s.slot[2] = w;
    cl.sync();
    u64 all = 0;
    for (unsigned c = 0; c < C; ++c) all += *cl.map_shared_rank(&s.slot[2], c);
    if (mine)
      p.logprob[row_id] = static_cast<float>((x_token == row.top ? 0.0 : (static_cast<double>(x_token) - row.top) * row.invT) -
                                             log(static_cast<double>(all) / row.one));
  }
  cl.sync();  // no CTA leaves while another may read its shared memory
}

// ------------------------------------------------------------------ host
constexpr size_t kSmemMax = 227 * 1024;
constexpr int kHeldMax = static_cast<int>((kSmemMax - sizeof(Shared)) / 4 / 32 * 32);

static cudaError_t launch(Params p, cudaStream_t st) {
  // the smallest cluster whose CTAs hold the row; few rows take the largest, to spread over the SMs
  int C = 1;
  while (C < 8 && ((p.V + C - 1) / C > kHeldMax || p.N * C < kNumSMsB200 / 2) && p.V > 2048 * C) C *= 2;
  p.share = static_cast<int>(round_up(ceil_div(std::max<int64_t>(p.V, 1), C), 32));
  const bool held = p.share <= kHeldMax;
  int lg = 0;
  while ((1ll << lg) < p.V) ++lg;
  p.one = std::ldexp(1.0, std::min(44, 62 - lg));
  auto kern = held ? sample_kernel<true> : sample_kernel<false>;
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
  cfg.dynamicSmemBytes = sizeof(Shared) + (held ? static_cast<size_t>(p.share) * 4 : 0);
  cfg.stream = st;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemMax));
  if (e != cudaSuccess) return e;
  return cudaLaunchKernelEx(&cfg, kern, p);
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

// Rows whose fp32 scores are held at a time: at most 256 MiB of them, at least one row.
static int64_t head_rows(const swvr_problem& p) {
  const int64_t pitch = round_up(std::max<int64_t>(p.vocab, 1), 4) * 4;
  return std::max<int64_t>(1, std::min<int64_t>(p.n_tokens, (256ll << 20) / pitch));
}

static int check_head(const swvr_problem* p) {
  if (!p) return fail(SWVR_ERR_INVALID_ARGUMENT, "problem is NULL");
  if (p->n_tokens < 0 || p->hidden < 0 || p->vocab < 0) return fail(SWVR_ERR_INVALID_ARGUMENT, "negative size");
  if (p->n_tokens >= (1ll << 28) || p->vocab >= (1ll << 31) || p->hidden >= (1ll << 31))
    return fail(SWVR_ERR_UNSUPPORTED, "sizes must be below 2^31 (rows 2^28)");
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
  ProfScope ps(kProfSample, static_cast<cudaStream_t>(stream));
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
    ProfScope ps(kProfSample, st);
    SWVR_CUDA(sample::launch(q, st));
  }
  return SWVR_OK;
}

}  // extern "C"
