// Embedding lookup with scaling and its gradient by token:
//   out[n, :]  = scale * E[tokens[n], :]
//   dE[v, :]   = scale * sum over n with tokens[n] = v of g[n, :]     (row padding_idx: 0)
// The gradient is summed in a fixed order and without atomics on values: the (token, position)
// pairs are sorted stably by token, equal-length chunks of the sorted list are summed by the
// threads that own the columns, and the pieces of a token that spans several chunks are added in
// list order.  Sums run in fp32 (fp64 for fp64) and are rounded once.
//
// Tokens outside [0, V) read nothing: the row of the lookup is NaN, the gradient leaves them out,
// and the device error word is set.
#include <cmath>

#include "common.cuh"
#include "ptx.cuh"
#include "tc.cuh"

namespace swvr {
namespace embed {

template <typename T>
struct Acc {
  using type = float;
};
template <>
struct Acc<double> {
  using type = double;
};

__device__ __forceinline__ float to_acc(float v) { return v; }
__device__ __forceinline__ double to_acc(double v) { return v; }
__device__ __forceinline__ float to_acc(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_acc(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_acc(float v, float* d) { *d = v; }
__device__ __forceinline__ void from_acc(double v, double* d) { *d = v; }
__device__ __forceinline__ void from_acc(float v, __nv_bfloat16* d) { *d = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_acc(float v, __half* d) { *d = __float2half_rn(v); }

// VEC consecutive elements: 16 bytes, or one element where rows are not 16-byte aligned.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

__device__ __forceinline__ int64_t load_token(const void* tokens, int bits, int64_t i) {
  return bits == 64 ? static_cast<const int64_t*>(tokens)[i] : static_cast<int64_t>(static_cast<const int32_t*>(tokens)[i]);
}

// ------------------------------------------------------------------ lookup
// blockDim.x threads own packs of a row, blockDim.y rows share a block; ROWS rows a thread, loaded before any is
// stored.  Bound by HBM: 16384 rows of 2560 bf16 (168 MB in and out) in 23 us (27 us with one row a thread).
template <typename T, int VEC, int ROWS>
__global__ void __launch_bounds__(256) lookup_kernel(int64_t n, int packs, int64_t V, const void* __restrict__ tokens,
                                                     int bits, const T* __restrict__ E, int64_t lde,
                                                     typename Acc<T>::type scale, T* __restrict__ out) {
  using A = typename Acc<T>::type;
  using P = Pack<T, VEC>;
  const int pk = blockIdx.y * blockDim.x + threadIdx.x;
  if (pk >= packs) return;
  const int64_t c = static_cast<int64_t>(pk) * VEC, D = static_cast<int64_t>(packs) * VEC;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * (blockDim.y * ROWS) + threadIdx.y;
  int64_t tok[ROWS];
  P p[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int64_t i = row0 + r * static_cast<int>(blockDim.y);
    tok[r] = i < n ? load_token(tokens, bits, i) : -1;
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
    if (tok[r] >= 0 && tok[r] < V) p[r] = *reinterpret_cast<const P*>(E + tok[r] * lde + c);
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int64_t i = row0 + r * static_cast<int>(blockDim.y);
    if (i >= n) return;
    if (tok[r] >= 0 && tok[r] < V) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) from_acc(to_acc(p[r].v[k]) * scale, &p[r].v[k]);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) from_acc(static_cast<A>(NAN), &p[r].v[k]);
      atomicCAS(&g_device_error, 0u, kErrToken | 1u);
    }
    *reinterpret_cast<P*>(out + i * D + c) = p[r];
  }
}

// ------------------------------------------------------------------ stable sort by token
// Least-significant-digit radix sort of (key, position) pairs, 8 bits a pass.  Keys are tokens;
// the padding row and tokens out of range get key V, behind all others.  A tile is kSortTile
// consecutive pairs: the histogram kernel counts its digits, one block turns the counts
// [digit][tile] into output offsets, and the scatter kernel ranks each pair within its tile.
// Within a tile warp w owns pairs [w * 256, (w + 1) * 256) and takes them 32 at a time, so
// ranks follow the list order and each pass is stable.
constexpr int kSortThreads = 256, kSortItems = 8, kSortTile = kSortThreads * kSortItems;
constexpr int kSortWarps = kSortThreads / 32, kDigits = 256;

struct SortIn {
  const void* tokens;  // first pass: raw tokens
  int bits;
  int64_t V, padding;
  const uint32_t* key;  // later passes: the pairs of the pass before (null in the first pass)
  const uint32_t* pos;
};

__device__ __forceinline__ uint32_t sort_key(const SortIn& in, int64_t i) {
  if (in.key) return in.key[i];
  const int64_t t = load_token(in.tokens, in.bits, i);
  const bool ok = t >= 0 && t < in.V;
  if (!ok) atomicCAS(&g_device_error, 0u, kErrToken | 2u);
  return ok && t != in.padding ? static_cast<uint32_t>(t) : static_cast<uint32_t>(in.V);
}

// Lanes of the warp whose 8-bit digit equals this lane's, among the lanes of `active`.
__device__ __forceinline__ uint32_t match_digit(uint32_t digit, uint32_t active) {
  uint32_t m = active;
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const uint32_t ones = __ballot_sync(0xffffffffu, (digit >> b) & 1u);
    m &= ((digit >> b) & 1u) ? ones : ~ones;
  }
  return m;
}

__global__ void __launch_bounds__(kSortThreads) sort_hist_kernel(int64_t n, SortIn in, int shift, int tiles,
                                                                 uint32_t* counts) {
  __shared__ uint32_t hist[kDigits];
  hist[threadIdx.x] = 0;
  __syncthreads();
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kSortTile;
#pragma unroll
  for (int r = 0; r < kSortItems; ++r) {
    const int64_t i = base + r * kSortThreads + threadIdx.x;
    if (i < n) atomicAdd(&hist[(sort_key(in, i) >> shift) & 255u], 1u);
  }
  __syncthreads();
  counts[static_cast<int64_t>(threadIdx.x) * tiles + blockIdx.x] = hist[threadIdx.x];
}

// Exclusive prefix sum of counts[0, m) in place, one block of 1024 threads.
__global__ void __launch_bounds__(1024) sort_scan_kernel(int64_t m, uint32_t* counts) {
  __shared__ uint32_t warp_sum[32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  uint32_t carry = 0;
  for (int64_t base = 0; base < m; base += 4096) {
    const int64_t i = base + threadIdx.x * 4ll;
    uint32_t v[4], s = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = i + k < m ? counts[i + k] : 0u;
      s += v[k];
    }
    uint32_t inc = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 31) warp_sum[warp] = inc;
    __syncthreads();
    if (warp == 0) {
      uint32_t w = warp_sum[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += up;
      }
      warp_sum[lane] = w;
    }
    __syncthreads();
    uint32_t ex = carry + (warp ? warp_sum[warp - 1] : 0u) + inc - s;
    carry += warp_sum[31];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (i + k < m) counts[i + k] = ex;
      ex += v[k];
    }
  }
}

__global__ void __launch_bounds__(kSortThreads) sort_scatter_kernel(int64_t n, SortIn in, int shift, int tiles,
                                                                    const uint32_t* __restrict__ offsets,
                                                                    uint32_t* __restrict__ key_out,
                                                                    uint32_t* __restrict__ pos_out) {
  __shared__ uint32_t cnt[kSortWarps][kDigits];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
  for (int w = 0; w < kSortWarps; ++w) cnt[w][threadIdx.x] = 0;
  __syncthreads();
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kSortTile + warp * (32 * kSortItems);
  uint32_t key[kSortItems], rank[kSortItems];
#pragma unroll
  for (int r = 0; r < kSortItems; ++r) {
    const int64_t i = base + r * 32 + lane;
    const bool in_range = i < n;
    const uint32_t active = __ballot_sync(0xffffffffu, in_range);
    key[r] = in_range ? sort_key(in, i) : 0u;
    const uint32_t d = (key[r] >> shift) & 255u;
    const uint32_t same = match_digit(d, active);
    rank[r] = 0;
    if (in_range) rank[r] = cnt[warp][d] + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (in_range && (same >> lane) == 1u) cnt[warp][d] = rank[r] + 1u;  // the group's last lane
    __syncwarp();
  }
  __syncthreads();
  {
    uint32_t run = offsets[static_cast<int64_t>(threadIdx.x) * tiles + blockIdx.x];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t c = cnt[w][threadIdx.x];
      cnt[w][threadIdx.x] = run;
      run += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kSortItems; ++r) {
    const int64_t i = base + r * 32 + lane;
    if (i < n) {
      const uint32_t o = cnt[warp][(key[r] >> shift) & 255u] + rank[r];
      key_out[o] = key[r];
      pos_out[o] = in.pos ? in.pos[i] : static_cast<uint32_t>(i);
    }
  }
}

// Up to kSmallSort pairs: one block sorts them in shared memory while the other blocks of the launch clear dE, which takes
// longer where it matters (778 MB: 125 us; the sort of 16384 pairs with 18-bit keys: 39 us, of 8192: 21 us).  Pairs stay in
// registers, `digit` bits a pass; warp w owns items [w * 32 * ITEMS, ...), so ranks follow the list order as above.  The sorted list
// is put together in shared memory: scattered stores of it took 9 us more.
constexpr int kSmallThreads = 1024, kSmallSort = 16 * kSmallThreads, kSmallDigits = 512;

struct SmallSmem {
  uint16_t cnt[kSmallThreads / 32][kSmallDigits];  // pairs per warp and digit, then where each warp's go
  uint32_t warp_sum[kSmallThreads / 32];
};

template <int ITEMS>
__device__ __forceinline__ void small_sort(int n, const SortIn& in, int bits, int digit, unsigned char* smem, uint32_t* key_out,
                                           uint32_t* pos_out) {
  SmallSmem& s = *reinterpret_cast<SmallSmem*>(smem);
  uint32_t* sk = reinterpret_cast<uint32_t*>(smem + sizeof(SmallSmem));
  uint32_t* sp = sk + ITEMS * kSmallThreads;
  const int t = threadIdx.x, lane = t % 32, warp = t / 32, base = warp * 32 * ITEMS;
  const int digits = 1 << digit;
  uint32_t key[ITEMS], pos[ITEMS], rank[ITEMS];
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {
    const int i = base + r * 32 + lane;
    key[r] = i < n ? sort_key(in, i) : 0u;
    pos[r] = i;
  }
  for (int shift = 0;; shift += digit) {
    for (int i = t; i < (kSmallThreads / 32) * digits; i += kSmallThreads) s.cnt[i / digits][i % digits] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
      const bool have = base + r * 32 + lane < n;
      uint32_t same = __ballot_sync(0xffffffffu, have);
      const uint32_t d = (key[r] >> shift) & (digits - 1u);
      for (int b = 0; b < digit; ++b) {
        const uint32_t ones = __ballot_sync(0xffffffffu, (d >> b) & 1u);
        same &= ((d >> b) & 1u) ? ones : ~ones;
      }
      rank[r] = 0;
      if (have) rank[r] = s.cnt[warp][d] + __popc(same & ((1u << lane) - 1u));
      __syncwarp();
      if (have && (same >> lane) == 1u) s.cnt[warp][d] = static_cast<uint16_t>(rank[r] + 1u);  // the group's last lane
      __syncwarp();
    }
    __syncthreads();
    // digit t's total over the warps, its exclusive prefix over the digits, then each warp's start
    uint32_t total = 0;
    if (t < digits)
#pragma unroll 8
      for (int w = 0; w < kSmallThreads / 32; ++w) total += s.cnt[w][t];
    uint32_t inc = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 31) s.warp_sum[warp] = inc;
    __syncthreads();
    uint32_t run = inc - total;
    for (int w = 0; w < warp; ++w) run += s.warp_sum[w];
    if (t < digits)
#pragma unroll 8
      for (int w = 0; w < kSmallThreads / 32; ++w) {
        const uint32_t c = s.cnt[w][t];
        s.cnt[w][t] = static_cast<uint16_t>(run);  // below n, which fits
        run += c;
      }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
      if (base + r * 32 + lane < n) {
        const uint32_t o = s.cnt[warp][(key[r] >> shift) & (digits - 1u)] + rank[r];
        sk[o] = key[r];
        sp[o] = pos[r];
      }
    }
    __syncthreads();
    if (shift + digit >= bits) {
      for (int i = t; i < n; i += kSmallThreads) {
        key_out[i] = sk[i];
        pos_out[i] = sp[i];
      }
      return;
    }
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
      const int i = base + r * 32 + lane;
      if (i < n) {
        key[r] = sk[i];
        pos[r] = sp[i];
      }
    }
  }
}

// Block 0 sorts; the others clear `bytes` bytes from dE (16-byte aligned) on.
template <int ITEMS>
__global__ void __launch_bounds__(kSmallThreads)
    sort_fill_kernel(int n, SortIn in, int bits, int digit, uint32_t* key, uint32_t* pos, uint32_t* joins,
                     unsigned char* dE, int64_t bytes) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  if (blockIdx.x == 0) {
    if (threadIdx.x == 0) *joins = 0;
    small_sort<ITEMS>(n, in, bits, digit, smem_raw, key, pos);
    return;
  }
  const int64_t step = static_cast<int64_t>(gridDim.x - 1) * kSmallThreads;
  const int64_t at = static_cast<int64_t>(blockIdx.x - 1) * kSmallThreads + threadIdx.x;
  uint4* d = reinterpret_cast<uint4*>(dE);
  const int64_t vecs = bytes / 16;
#pragma unroll 4
  for (int64_t i = at; i < vecs; i += step) d[i] = make_uint4(0, 0, 0, 0);
  if (at < bytes % 16) dE[vecs * 16 + at] = 0;
}

// ------------------------------------------------------------------ sums by token
// A chunk is `len` consecutive sorted pairs.  TX threads own the packs of a row, TY chunks share a
// block.  A token that begins and ends inside a chunk is written to dE at once; the part of
// the chunk's first token that began earlier goes to part[chunk][0], the part of its last token
// that goes on (and began here) to part[chunk][1], and the chunk to the list of those that join_kernel starts from (in any
// order: each is joined by itself).  Four rows in flight a thread.  Bound by HBM and its latency: 16384 rows of 2560 bf16 in 30 us
// (84 MB read, some 50 written: 4.4 TB/s).
template <typename T, int VEC>
__global__ void __launch_bounds__(256) sum_kernel(int64_t n, int len, int chunks, int packs, uint32_t V,
                                                  const uint32_t* __restrict__ key, const uint32_t* __restrict__ pos,
                                                  const T* __restrict__ g, int64_t ldg,
                                                  typename Acc<T>::type scale, T* __restrict__ dE, int64_t lde,
                                                  typename Acc<T>::type* __restrict__ part, uint32_t* joins) {
  using A = typename Acc<T>::type;
  using P = Pack<T, VEC>;
  const int64_t chunk = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  const int pk = blockIdx.y * blockDim.x + threadIdx.x;
  if (chunk >= chunks || pk >= packs) return;
  const int64_t i0 = chunk * len, i1 = min(n, i0 + len);
  const int64_t c = static_cast<int64_t>(pk) * VEC, D = static_cast<int64_t>(packs) * VEC;
  A acc[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = A(0);
  uint32_t cur = key[i0];
  if (cur >= V) return;  // padding and invalid tokens are last
  bool first = i0 > 0 && key[i0 - 1] == cur;  // the current token began in an earlier chunk
  constexpr int U = 4;
  for (int64_t i = i0; i < i1; i += U) {
    P p[U];
    uint32_t kk[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      kk[u] = i + u < i1 ? key[i + u] : V;
      if (kk[u] < V) p[u] = *reinterpret_cast<const P*>(g + pos[i + u] * ldg + c);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u >= i1) break;
      if (kk[u] != cur) {  // the current token ends
        if (first) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) part[chunk * 2 * D + c + k] = acc[k];
        } else {
          P o;
#pragma unroll
          for (int k = 0; k < VEC; ++k) from_acc(acc[k] * scale, &o.v[k]);
          *reinterpret_cast<P*>(dE + static_cast<int64_t>(cur) * lde + c) = o;
        }
        first = false;
        cur = kk[u];
        if (cur >= V) return;
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] = A(0);
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] += to_acc(p[u].v[k]);
    }
  }
  const bool goes_on = i1 < n && key[i1] == cur;
  if (first || goes_on) {
    // a token that fills the whole chunk and goes on is a middle piece: slot 0
    if (goes_on && !first && pk == 0) joins[1 + atomicAdd(joins, 1u)] = static_cast<uint32_t>(chunk);
    A* dst = part + (chunk * 2 + (first ? 0 : 1)) * D + c;
#pragma unroll
    for (int k = 0; k < VEC; ++k) dst[k] = acc[k];
  } else {
    P o;
#pragma unroll
    for (int k = 0; k < VEC; ++k) from_acc(acc[k] * scale, &o.v[k]);
    *reinterpret_cast<P*>(dE + static_cast<int64_t>(cur) * lde + c) = o;
  }
}

// Adds the pieces of each token that spans chunks, in a fixed order: a block (32 packs wide) for each chunk in which
// such a token begins; 4 groups of threads take every 4th of the pieces that follow, four at a time, and the groups'
// sums are added in group order.  16384 tokens, some 300 spanning chunks and one of 82 pieces: 14 us; 38 us by one row of
// threads per chunk, 16 us with 16 groups (most tokens have a piece or two).
constexpr int kJoinGroups = 4;

template <typename T, int VEC>
__global__ void __launch_bounds__(32 * kJoinGroups)
    join_kernel(int len, int chunks, int packs, const uint32_t* __restrict__ key,
                typename Acc<T>::type scale, T* __restrict__ dE, int64_t lde,
                const typename Acc<T>::type* __restrict__ part, const uint32_t* __restrict__ joins) {
  using A = typename Acc<T>::type;
  using P = Pack<T, VEC>;
  __shared__ A sums[kJoinGroups][32][VEC + 1];
  const int64_t D = static_cast<int64_t>(packs) * VEC;
  const uint32_t wide = (packs + 31) / 32, work = joins[0] * wide;  // (chunk, 32 packs) pairs
  for (uint32_t u = blockIdx.x; u < work; u += gridDim.x) {
    const int64_t chunk = joins[1 + u / wide];
    const uint32_t cur = key[chunk * len + len - 1];  // it goes on, so the chunk is full
    const int pk = u % wide * 32 + threadIdx.x;
    const int64_t c = static_cast<int64_t>(pk) * VEC;
    A acc[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] = A(0);
    if (pk < packs) {
      if (threadIdx.y == 0)
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] = part[(chunk * 2 + 1) * D + c + k];
      constexpr int U = 4;  // pieces in flight: their keys, then their sums
      bool more = true;
      for (int64_t j0 = chunk + 1 + threadIdx.y; more; j0 += U * kJoinGroups) {
        bool is[U];
#pragma unroll
        for (int q = 0; q < U; ++q) {
          const int64_t j = j0 + q * kJoinGroups;
          is[q] = j < chunks && key[j * len] == cur;
        }
#pragma unroll
        for (int q = 0; q < U; ++q)
          if (is[q])
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[k] += part[(j0 + q * kJoinGroups) * 2 * D + c + k];
        more = is[U - 1];
      }
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) sums[threadIdx.y][threadIdx.x][k] = acc[k];
    __syncthreads();
    if (threadIdx.y == 0 && pk < packs) {
#pragma unroll
      for (int g = 1; g < kJoinGroups; ++g)
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] += sums[g][threadIdx.x][k];
      P o;
#pragma unroll
      for (int k = 0; k < VEC; ++k) from_acc(acc[k] * scale, &o.v[k]);
      *reinterpret_cast<P*>(dE + static_cast<int64_t>(cur) * lde + c) = o;
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ host
struct BwdPlan {
  int tiles, bits, passes, len, chunks;
  bool small;  // one block sorts
  size_t off_key[2], off_pos[2], off_counts, off_joins, off_part, bytes;
};

static BwdPlan plan_bwd(int64_t n, int64_t V, int64_t D, int dt) {
  BwdPlan b{};
  b.tiles = static_cast<int>(ceil_div(std::max<int64_t>(n, 1), kSortTile));
  b.bits = 1;
  while ((V >> b.bits) != 0) ++b.bits;  // keys 0 .. V
  b.passes = (b.bits + 7) / 8;
  b.small = n <= kSmallSort;
  // chunks of 16 pairs, longer where that gives more than 2048 of them
  b.len = static_cast<int>(std::min<int64_t>(512, std::max<int64_t>(16, ceil_div(n, 2048))));
  b.chunks = static_cast<int>(ceil_div(std::max<int64_t>(n, 1), b.len));
  size_t off = 0;
  for (int k = 0; k < 2; ++k) {
    b.off_key[k] = off;
    off += align_up(static_cast<size_t>(n) * 4, 256);
    b.off_pos[k] = off;
    off += align_up(static_cast<size_t>(n) * 4, 256);
  }
  b.off_counts = off;
  off += align_up(static_cast<size_t>(b.tiles) * kDigits * 4, 256);
  b.off_joins = off;
  off += align_up((static_cast<size_t>(b.chunks) + 1) * 4, 256);
  b.off_part = off;
  off += align_up(static_cast<size_t>(b.chunks) * 2 * D * (dt == SWVR_F64 ? 8 : 4), 256);
  b.bytes = off + 256;
  return b;
}

static bool rows16(const void* p, int64_t ld, int64_t D, size_t es) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (ld * es) % 16 == 0 && (D * es) % 16 == 0;
}

// Threads across a row: the widest of 256, 128, 64, 32 that leaves the fewest of them idle.
static int row_threads(int packs) {
  int best = 32;
  for (int tx : {64, 128, 256})
    if (round_up(packs, tx) <= round_up(packs, best)) best = tx;
  return best;
}

template <typename T, int VEC>
static cudaError_t lookup(int64_t n, int64_t V, int64_t D, const void* tokens, int bits, const void* E, int64_t lde,
                          double scale, void* out, cudaStream_t st) {
  using A = typename Acc<T>::type;
  const int packs = static_cast<int>(D / VEC), tx = row_threads(packs);
  const dim3 block(tx, 256 / tx);
  const unsigned gy = static_cast<unsigned>(ceil_div(packs, tx));
  // several rows a thread once one each would be over eight blocks an SM
  if (ceil_div(n, block.y) * gy > 8 * kNumSMsB200)
    lookup_kernel<T, VEC, 4><<<dim3(static_cast<unsigned>(ceil_div(n, block.y * 4)), gy), block, 0, st>>>(
        n, packs, V, tokens, bits, static_cast<const T*>(E), lde, static_cast<A>(scale), static_cast<T*>(out));
  else
    lookup_kernel<T, VEC, 1><<<dim3(static_cast<unsigned>(ceil_div(n, block.y)), gy), block, 0, st>>>(
        n, packs, V, tokens, bits, static_cast<const T*>(E), lde, static_cast<A>(scale), static_cast<T*>(out));
  return cudaGetLastError();
}

template <typename T>
static cudaError_t fwd(int64_t n, int64_t V, int64_t D, const void* tokens, int bits, const void* E, int64_t lde,
                       double scale, void* out, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(T);
  if (rows16(E, lde, D, sizeof(T)) && rows16(out, D, D, sizeof(T)))
    return lookup<T, VEC>(n, V, D, tokens, bits, E, lde, scale, out, st);
  return lookup<T, 1>(n, V, D, tokens, bits, E, lde, scale, out, st);
}

template <typename T, int VEC>
static cudaError_t sums(const BwdPlan& b, int64_t n, int64_t V, int64_t D, const uint32_t* key, const uint32_t* pos,
                        const void* g, int64_t ldg, double scale, void* dE, int64_t lde, void* part, uint32_t* joins,
                        cudaStream_t st) {
  using A = typename Acc<T>::type;
  const int packs = static_cast<int>(D / VEC), tx = row_threads(packs);
  const dim3 block(tx, 256 / tx);
  const dim3 grid(static_cast<unsigned>(ceil_div(b.chunks, block.y)), static_cast<unsigned>(ceil_div(packs, tx)));
  sum_kernel<T, VEC><<<grid, block, 0, st>>>(n, b.len, b.chunks, packs, static_cast<uint32_t>(V), key, pos,
                                             static_cast<const T*>(g), ldg, static_cast<A>(scale), static_cast<T*>(dE),
                                             lde, static_cast<A*>(part), joins);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int64_t work = ceil_div(packs, 32) * b.chunks;
  join_kernel<T, VEC><<<static_cast<unsigned>(std::min<int64_t>(work, 16 * kNumSMsB200)), dim3(32, kJoinGroups), 0, st>>>(
      b.len, b.chunks, packs, key, static_cast<A>(scale), static_cast<T*>(dE), lde, static_cast<const A*>(part), joins);
  return cudaGetLastError();
}

// One launch sorts and clears dE; otherwise three launches a pass, after a memset.
static bool one_block(const BwdPlan& b, int64_t n, int64_t D, const void* dE, int64_t lde) {
  return b.small && n > 0 && lde == D && (reinterpret_cast<uintptr_t>(dE) & 15u) == 0;
}

template <typename T>
static cudaError_t bwd(const BwdPlan& b, int64_t n, int64_t V, int64_t D, const void* tokens, int bits, const void* g,
                       int64_t ldg, double scale, int64_t padding, void* dE, int64_t lde, char* ws, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(T);
  cudaError_t e = cudaSuccess;
  SortIn in{tokens, bits, V, padding, nullptr, nullptr};
  uint32_t* joins = reinterpret_cast<uint32_t*>(ws + b.off_joins);
  uint32_t* key[2] = {reinterpret_cast<uint32_t*>(ws + b.off_key[0]), reinterpret_cast<uint32_t*>(ws + b.off_key[1])};
  uint32_t* pos[2] = {reinterpret_cast<uint32_t*>(ws + b.off_pos[0]), reinterpret_cast<uint32_t*>(ws + b.off_pos[1])};
  if (one_block(b, n, D, dE, lde)) {
    const int passes = (b.bits + 8) / 9, digit = (b.bits + passes - 1) / passes;  // at most 9 bits each
    const int64_t bytes = V * D * static_cast<int64_t>(sizeof(T));
    auto launch = [&](auto kern, int items) {
      const int smem = static_cast<int>(sizeof(SmallSmem)) + items * kSmallThreads * 8;
      const cudaError_t r = tc::allow_smem(reinterpret_cast<const void*>(kern), smem);
      if (r != cudaSuccess) return r;
      const int64_t fill = std::min<int64_t>(kNumSMsB200 - 1, ceil_div(bytes, 16 * kSmallThreads));
      kern<<<static_cast<unsigned>(1 + fill), kSmallThreads, smem, st>>>(static_cast<int>(n), in, b.bits, digit, key[0], pos[0], joins,
                                                                         static_cast<unsigned char*>(dE), bytes);
      return cudaGetLastError();
    };
    e = n <= 2 * kSmallThreads   ? launch(sort_fill_kernel<2>, 2)
        : n <= 8 * kSmallThreads ? launch(sort_fill_kernel<8>, 8)
                                 : launch(sort_fill_kernel<16>, 16);
    if (e != cudaSuccess) return e;
    in.key = key[0];
    in.pos = pos[0];
  } else {
    e = lde == D ? cudaMemsetAsync(dE, 0, sizeof(T) * V * D, st)
                 : cudaMemset2DAsync(dE, lde * sizeof(T), 0, D * sizeof(T), V, st);
    if (e != cudaSuccess || n == 0) return e;
    if ((e = cudaMemsetAsync(joins, 0, 4, st)) != cudaSuccess) return e;
    uint32_t* counts = reinterpret_cast<uint32_t*>(ws + b.off_counts);
    for (int p = 0; p < b.passes; ++p) {
      uint32_t *ko = key[p & 1], *po = pos[p & 1];
      sort_hist_kernel<<<b.tiles, kSortThreads, 0, st>>>(n, in, 8 * p, b.tiles, counts);
      sort_scan_kernel<<<1, 1024, 0, st>>>(static_cast<int64_t>(b.tiles) * kDigits, counts);
      sort_scatter_kernel<<<b.tiles, kSortThreads, 0, st>>>(n, in, 8 * p, b.tiles, counts, ko, po);
      if ((e = cudaGetLastError()) != cudaSuccess) return e;
      in.key = ko;
      in.pos = po;
    }
  }
  char* part = ws + b.off_part;
  if (rows16(g, ldg, D, sizeof(T)) && rows16(dE, lde, D, sizeof(T)))
    return sums<T, VEC>(b, n, V, D, in.key, in.pos, g, ldg, scale, dE, lde, part, joins, st);
  return sums<T, 1>(b, n, V, D, in.key, in.pos, g, ldg, scale, dE, lde, part, joins, st);
}

static int check_sizes(int64_t n, int64_t V, int64_t D, int bits, int dt, int64_t lde) {
  if (n < 0 || V < 0 || D < 0) return fail(SWVR_ERR_INVALID_ARGUMENT, "negative size");
  if (n >= (1ll << 31) || V >= (1ll << 31) - 1 || D >= (1ll << 31))
    return fail(SWVR_ERR_UNSUPPORTED, "sizes must be below 2^31");
  if (bits != 32 && bits != 64) return fail(SWVR_ERR_INVALID_ARGUMENT, "tokens must be 32- or 64-bit integers");
  if (dt < SWVR_F32 || dt > SWVR_F16) return fail(SWVR_ERR_INVALID_ARGUMENT, "unknown dtype %d", dt);
  if (lde < D) return fail(SWVR_ERR_INVALID_ARGUMENT, "row stride smaller than the row length");
  if (ceil_div(n, 8) * ceil_div(D, 32) >= (1ll << 40) || ceil_div(D, 32) > 65535) return fail(SWVR_ERR_UNSUPPORTED, "n_tokens x dim too large");
  return SWVR_OK;
}

}  // namespace embed
}  // namespace swvr

extern "C" {

int swvr_embed_fwd(int64_t n_tokens, int64_t vocab, int64_t dim, const void* tokens, int32_t token_bits, const void* E,
                   int32_t dtype, int64_t lde, double scale, void* out, void* stream) {
  SWVR_TRY(embed::check_sizes(n_tokens, vocab, dim, token_bits, dtype, lde));
  if (n_tokens == 0 || dim == 0) return SWVR_OK;
  if (!tokens || !out || (vocab > 0 && !E)) return fail(SWVR_ERR_INVALID_ARGUMENT, "NULL pointer");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  ProfScope ps(kProfEmbed, st);
  switch (dtype) {
    case SWVR_F32: SWVR_CUDA(embed::fwd<float>(n_tokens, vocab, dim, tokens, token_bits, E, lde, scale, out, st)); break;
    case SWVR_F64: SWVR_CUDA(embed::fwd<double>(n_tokens, vocab, dim, tokens, token_bits, E, lde, scale, out, st)); break;
    case SWVR_BF16:
      SWVR_CUDA(embed::fwd<__nv_bfloat16>(n_tokens, vocab, dim, tokens, token_bits, E, lde, scale, out, st));
      break;
    default: SWVR_CUDA(embed::fwd<__half>(n_tokens, vocab, dim, tokens, token_bits, E, lde, scale, out, st));
  }
  return SWVR_OK;
}

int swvr_embed_bwd_workspace_size(int64_t n_tokens, int64_t vocab, int64_t dim, int32_t dtype, size_t* bytes) {
  if (!bytes) return fail(SWVR_ERR_INVALID_ARGUMENT, "bytes is NULL");
  SWVR_TRY(embed::check_sizes(n_tokens, vocab, dim, 64, dtype, dim));
  *bytes = embed::plan_bwd(n_tokens, vocab, dim, dtype).bytes;
  return SWVR_OK;
}

int swvr_embed_bwd(int64_t n_tokens, int64_t vocab, int64_t dim, const void* tokens, int32_t token_bits,
                   const void* grad_out, int64_t ld_grad_out, double scale, int64_t padding_idx, void* grad_E,
                   int32_t dtype, int64_t ld_grad_E, void* workspace, size_t workspace_bytes, void* stream) {
  SWVR_TRY(embed::check_sizes(n_tokens, vocab, dim, token_bits, dtype, ld_grad_E));
  if (ld_grad_out < dim) return fail(SWVR_ERR_INVALID_ARGUMENT, "row stride smaller than the row length");
  if (vocab == 0 || dim == 0) return SWVR_OK;
  if (!grad_E || (n_tokens > 0 && (!tokens || !grad_out || !workspace)))
    return fail(SWVR_ERR_INVALID_ARGUMENT, "NULL pointer");
  if (!aligned16(workspace)) return fail(SWVR_ERR_UNSUPPORTED, "workspace not 16-byte aligned");
  const embed::BwdPlan b = embed::plan_bwd(n_tokens, vocab, dim, dtype);
  if (n_tokens > 0 && workspace_bytes < b.bytes)
    return fail(SWVR_ERR_WORKSPACE, "workspace %zu < required %zu", workspace_bytes, b.bytes);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  ProfScope ps(kProfEmbed, st, n_tokens == 0 ? 0 : (embed::one_block(b, n_tokens, dim, grad_E, ld_grad_E) ? 1 : 3 * b.passes) + 2);
  switch (dtype) {
    case SWVR_F32:
      SWVR_CUDA(embed::bwd<float>(b, n_tokens, vocab, dim, tokens, token_bits, grad_out, ld_grad_out, scale, padding_idx,
                                  grad_E, ld_grad_E, ws, st));
      break;
    case SWVR_F64:
      SWVR_CUDA(embed::bwd<double>(b, n_tokens, vocab, dim, tokens, token_bits, grad_out, ld_grad_out, scale,
                                   padding_idx, grad_E, ld_grad_E, ws, st));
      break;
    case SWVR_BF16:
      SWVR_CUDA(embed::bwd<__nv_bfloat16>(b, n_tokens, vocab, dim, tokens, token_bits, grad_out, ld_grad_out, scale,
                                          padding_idx, grad_E, ld_grad_E, ws, st));
      break;
    default:
      SWVR_CUDA(embed::bwd<__half>(b, n_tokens, vocab, dim, tokens, token_bits, grad_out, ld_grad_out, scale,
                                   padding_idx, grad_E, ld_grad_E, ws, st));
  }
  return SWVR_OK;
}

}  // extern "C"
