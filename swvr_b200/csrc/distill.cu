// Distillation of the head from a teacher's top logits:
//   z = (logit_scale * h W^T + bias) / T,   p = softmax(z) over the V rows of W,
//   q_k = exp(t_k / T - L_n)  over the K_t teacher entries of token n, L_n their logsumexp (or given),
//   each_n = T^2 * sum_k q_k (log q_k - z[id_k] + lse_n),   loss = none / sum / mean of w_n each_n,
//   dS[n, v] = g_n T (p_v * sum_k q_k - sum_{k: id_k = v} q_k),  dh = s dS W,  dW = s dS^T h,  db = sum_n dS.
// [N, V] is never kept: the forward (head_kernel, kHeadLse) leaves lse and the K_t scores of each token,
// the backward recomputes S a vocabulary chunk at a time (kHeadGrad) and runs the readout's dW / dh
// GEMMs.  kHeadGrad stores the dense part p * sum q; the entries of teacher tokens, p * sum q - q, come
// from the forward's fp32 scores and are written over it in one rounding (subtracting q from the
// 16-bit p would lose the difference where the student has learnt the teacher).
// The teacher's part of db is a sum over tokens in no fixed order: it is added in fixed point, where order does not matter, in
// two 64-bit words a row: what a contribution has below the first word's unit goes to the second.
#include <cfloat>
#include <climits>
#include <cmath>

#include "common.cuh"
#include "ptx.cuh"
#include "tc.cuh"

namespace swvr {
namespace distill {

template <typename A>
__device__ __forceinline__ A load_a(const void* p, int dt, int64_t i) {
  if constexpr (sizeof(A) == 8) return load_d(p, dt, i);
  else return load_f(p, dt, i);
}
// A teacher's logit: fp64 ones past fp32's range count as its ends there (a mask of the type's lowest value is no -inf).
template <typename A>
__device__ __forceinline__ A load_logit(const void* p, int dt, int64_t i) {
  if constexpr (sizeof(A) == 4) {
    if (dt == SWVR_F64) {
      const double d = static_cast<const double*>(p)[i];
      return static_cast<A>(isfinite(d) ? fmin(fmax(d, -static_cast<double>(FLT_MAX)), static_cast<double>(FLT_MAX)) : d);
    }
  }
  return load_a<A>(p, dt, i);
}
__device__ __forceinline__ float exp_a(float x) { return expf(x); }
__device__ __forceinline__ double exp_a(double x) { return exp(x); }
__device__ __forceinline__ float log_a(float x) { return logf(x); }
__device__ __forceinline__ double log_a(double x) { return log(x); }

template <typename A>
__device__ __forceinline__ A warp_sum(A v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <typename A>
__device__ __forceinline__ A warp_max(A v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const A u = __shfl_xor_sync(0xffffffffu, v, o);
    v = u > v ? u : v;
  }
  return v;
}

constexpr int kWarps = 4;          // tokens per block of the per-token kernels
constexpr int kMaxTeacher = 1024;  // entries per token: the sort's shared memory and its K_t^2 compares

// ------------------------------------------------------------------ teacher rows
// One warp per token: log q of each entry, their sum, and the entries sorted by id (each entry's rank
// is the number of entries before it, K_t^2 / 32 compares a lane: K_t is tens).  Entries with a negative id or a
// logit of -inf are left out (id INT_MAX, q = 0, sorted behind); an id >= V is an error: the token's
// loss and gradient are NaN.  8192 tokens of 64 entries: 20 us.
template <typename A>
__global__ void __launch_bounds__(32 * kWarps)
    teacher_kernel(int64_t N, int64_t V, int Kt, const void* __restrict__ ids, int bits, const void* __restrict__ t,
                   int t_dt, const A* __restrict__ t_lse, A inv_T, int32_t* sid, A* slogq, A* qsum, uint32_t* done) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  A* tv = reinterpret_cast<A*>(smem_raw) + warp * Kt;
  int32_t* id = reinterpret_cast<int32_t*>(reinterpret_cast<A*>(smem_raw) + kWarps * Kt) + warp * Kt;
  const int64_t n = blockIdx.x * static_cast<int64_t>(kWarps) + warp;
  if (blockIdx.x == 0 && threadIdx.x == 0) *done = 0;
  if (n >= N) return;
  A mx = -INFINITY;
  bool bad = false;
  for (int k = lane; k < Kt; k += 32) {
    const int64_t i = n * Kt + k;
    const int64_t v = bits == 64 ? static_cast<const int64_t*>(ids)[i] : static_cast<int64_t>(static_cast<const int32_t*>(ids)[i]);
    const A x = load_logit<A>(t, t_dt, i);
    const bool dead = v < 0 || x == -static_cast<A>(INFINITY);
    if (!dead && v >= V) bad = true;
    tv[k] = dead ? -static_cast<A>(INFINITY) : x;
    id[k] = dead || v >= V ? INT_MAX : static_cast<int32_t>(v);
    if (!dead) mx = x > mx ? x : mx;
  }
  __syncwarp();
  mx = warp_max(mx);
  A sum = 0;
  for (int k = lane; k < Kt; k += 32)
    if (id[k] != INT_MAX) sum += exp_a((tv[k] - mx) * inv_T);
  sum = warp_sum(sum);
  bad = __any_sync(0xffffffffu, bad);
  // log q from differences to the largest: the logsumexp itself would round at its own size, and t / T may be past the
  // type's range where the differences are not (entries at its lowest value, T below 1)
  const A lsum = log_a(sum);
  A qs = 0;
  for (int k = lane; k < Kt; k += 32) {
    const int32_t mine = id[k];
    int rank = 0;
    for (int j = 0; j < Kt; ++j) rank += id[j] < mine || (id[j] == mine && j < k);
    const A lq = mine == INT_MAX ? -static_cast<A>(INFINITY)
                 : t_lse         ? fma(tv[k], inv_T, -t_lse[n])
                                 : (tv[k] - mx) * inv_T - lsum;
    sid[n * Kt + rank] = mine;
    slogq[n * Kt + rank] = lq;
    if (mine != INT_MAX) qs += exp_a(lq);
  }
  qs = warp_sum(qs);
  if (lane == 0) {
    qsum[n] = bad ? static_cast<A>(NAN) : qs;
    if (bad) atomicCAS(&g_device_error, 0u, kErrToken | 3u);
  }
}

// ------------------------------------------------------------------ loss
template <typename A>
__device__ __forceinline__ A weighted(A w, A e) {
  return w == A(0) ? A(0) : w * e;  // a zero weight drops the token, whatever its loss
}

// Sum or mean over the tokens by one block in a fixed order, in double.  stats: loss, denominator.
template <typename A>
__device__ __forceinline__ void total_loss(int64_t N, bool mean, const A* each, const A* __restrict__ w, A* out, A* stats) {
  __shared__ double sh[2][32 * kWarps / 32];
  double s = 0, d = 0;
#pragma unroll 4
  for (int64_t n = threadIdx.x; n < N; n += blockDim.x) {
    const A wn = w ? w[n] : A(1);
    s += static_cast<double>(weighted(wn, __ldcg(each + n)));
    d += static_cast<double>(wn);
  }
  s = warp_sum(s);
  d = warp_sum(d);
  if (threadIdx.x % 32 == 0) sh[0][threadIdx.x / 32] = s, sh[1][threadIdx.x / 32] = d;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = d = 0;
    for (int i = 0; i < kWarps; ++i) s += sh[0][i], d += sh[1][i];
    if (!mean) d = 1.0;
    *out = static_cast<A>(s / d);
    stats[0] = static_cast<A>(s / d);
    stats[1] = static_cast<A>(d);
  }
}

// Sources of (m, l): `splits` partial slots of head_kernel in log2 units (slot (n / 256 * splits + s) * 256
// + n % 256), or one natural-unit pair per token (splits = 0).  The block that finishes last sums the tokens (all of
// them, in a fixed order); `done` counts finished blocks and is cleared by teacher_kernel.  2048 tokens of 64 entries: 5.3 us
// (a second launch for the sum would cost more than the last block's 2 us); 8192 tokens of 64: 37 us.
template <typename A>
__global__ void __launch_bounds__(32 * kWarps)
    each_kernel(int64_t N, int Kt, int splits, const A* __restrict__ m, const A* __restrict__ l,
                const int32_t* __restrict__ sid, const A* __restrict__ slogq, const A* __restrict__ z,
                const A* __restrict__ qsum, A T2, A* lse, A* lse_lo, A* each, int red, const A* __restrict__ w, A* out, A* stats,
                uint32_t* done) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t n = blockIdx.x * static_cast<int64_t>(kWarps) + warp;
  if (n < N) {
    double L;
    if (splits == 0) {
      L = static_cast<double>(m[n]) + log(static_cast<double>(l[n]));
    } else {
      const int64_t base = (n / 256) * splits * 256 + n % 256;
      A mx = -INFINITY;
      for (int s = lane; s < splits; s += 32) mx = m[base + s * 256ll] > mx ? m[base + s * 256ll] : mx;
      mx = warp_max(mx);
      double sum = 0;
      if (mx != -static_cast<A>(INFINITY))
        for (int s = lane; s < splits; s += 32) {
          const A w = exp2f(static_cast<float>(m[base + s * 256ll] - mx));
          sum += static_cast<double>(l[base + s * 256ll]) * w;
        }
      sum = warp_sum(sum);
      L = (static_cast<double>(mx) + log2(sum)) * 0.6931471805599453;
    }
    const A hi = static_cast<A>(L), lo = isfinite(L) ? static_cast<A>(L - static_cast<double>(hi)) : A(0);
    // (log q - z) + lse: z and lse are near each other, so the difference is taken first
    A s = 0;
    for (int k = lane; k < Kt; k += 32) {
      if (sid[n * Kt + k] == INT_MAX) continue;
      const A lq = slogq[n * Kt + k], q = exp_a(lq);
      if (q > 0) s += q * (lq - ((z[n * Kt + k] - hi) - lo));
      else if (q != q) s = q;
    }
    s = warp_sum(s);
    if (lane == 0) {
      const A e = qsum[n] != qsum[n] ? qsum[n] : T2 * s;
      lse[n] = hi;
      lse_lo[n] = lo;
      each[n] = e;
      if (red == SWVR_REDUCE_NONE) out[n] = w ? weighted(w[n], e) : e;
    }
  }
  if (red == SWVR_REDUCE_NONE) return;
  __shared__ bool last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(done, 1u) == gridDim.x - 1;
  __syncthreads();
  if (last) {
    __threadfence();
    total_loss(N, red == SWVR_REDUCE_MEAN, each, w, out, stats);
  }
}

// ------------------------------------------------------------------ backward
// One block.  Per token: gT = g_n T (g_n: upstream, weight and denominator), coef = gT sum q, and the weight's
// gradient.  Then the ranges, from the largest |gT| max(1, sum q), a:
// f[0] what dS is multiplied by when stored, f[1] its undoing (dh, dW), f[2] the binary exponent of the units of db's first
// word, f[3] how much finer those of its second are.  Both words have 59 - log2 N bits, 92 in all at 8192 tokens: a row whose
// contributions are 2^-60 of the largest still has them to fp32's accuracy.
// fp16 dS is scaled by a power of two that puts its largest value near 2^13, so that small gradients (1 / N of a
// mean) do not fall below fp16's range; bf16 has fp32's.  8192 tokens: 7.5 us; one block, so that the ranges need no second launch.
constexpr int kGradThreads = 1024;

template <typename A>
__global__ void __launch_bounds__(kGradThreads)
    token_grad_kernel(int64_t N, int red, A T, const A* __restrict__ gout, const A* __restrict__ w, const A* __restrict__ each,
                      const A* __restrict__ qsum, const A* __restrict__ stats, A* gT, A* coef, A* grad_w, float s, bool fp16,
                      float* f) {
  __shared__ float most[kGradThreads / 32];
  float a = 0.f;
#pragma unroll 4
  for (int64_t n = threadIdx.x; n < N; n += kGradThreads) {
    const A up = red == SWVR_REDUCE_NONE ? gout[n] : gout[0];
    const A den = red == SWVR_REDUCE_MEAN ? stats[1] : A(1);
    const A wn = w ? w[n] : A(1);
    const A q = qsum[n];
    // a row with no teacher left, and one of zero weight, take no part: 0, not 0 x inf
    const A g = wn == A(0) || q == A(0) ? A(0) : up * wn / den * T;
    gT[n] = g;
    coef[n] = g == A(0) ? A(0) : g * q;
    if (grad_w) grad_w[n] = red == SWVR_REDUCE_MEAN ? up * (each[n] - stats[0]) / den : up * each[n];
    const float b = fabsf(static_cast<float>(g)) * fmaxf(1.f, static_cast<float>(q));
    if (b < INFINITY) a = fmaxf(a, b);  // neither inf nor NaN
  }
  if (!f) return;
  a = warp_max(a);
  if (threadIdx.x % 32 == 0) most[threadIdx.x / 32] = a;
  __syncthreads();
  if (threadIdx.x < 32) {
    a = warp_max(most[threadIdx.x]);
    if (threadIdx.x == 0) {
      // a token adds less than 2^(bits + 1) to a word of a row, all of them less than 2^61
      const int bits = 60 - (64 - __clzll(N));
      int e = 0, x = 0;
      if (a > 0.f) {
        const float as = a * fabsf(s);
        if (fp16 && as > 0.f && as < INFINITY) e = max(-100, min(100, 13 - ilogbf(as)));
        x = max(-100, min(140, bits - ilogbf(a)));
      }
      f[0] = ldexpf(s, e);
      f[1] = ldexpf(1.f, -e);
      f[2] = static_cast<float>(x);
      f[3] = static_cast<float>(bits);
    }
  }
}

// The sum of q over the entries of sorted position j's id, when j is the first of them; -1 otherwise.
template <typename A>
__device__ __forceinline__ A merged_q(const int32_t* sid, const A* slogq, int j, int Kt) {
  const int32_t v = sid[j];
  if (j > 0 && sid[j - 1] == v) return A(-1);
  A q = exp_a(slogq[j]);
  for (int i = j + 1; i < Kt && sid[i] == v; ++i) q += exp_a(slogq[i]);
  return q;
}

// The teacher entries of vocabulary rows [v0, v1): written over the dense dS^T, and their part of db.  A thread an entry,
// bound by reading the ids and by scattered 2-byte stores: 8192 x 64 entries, 9 us a chunk.
template <bool kBF16>
__global__ void __launch_bounds__(256)
    entries_kernel(int64_t N, int Kt, int v0, int v1, const int32_t* __restrict__ sid, const float* __restrict__ slogq,
                   const float* __restrict__ z, const float* __restrict__ lse, const float* __restrict__ gT,
                   const float* __restrict__ coef, const float* __restrict__ f, void* ds, int64_t ld_ds,
                   unsigned long long* db) {
  const int64_t i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= N * Kt) return;
  const int32_t v = sid[i];
  if (v < v0 || v >= v1) return;
  const int64_t n = i / Kt;
  const float g = gT[n];
  if (g == 0.f) return;
  const float q = merged_q(sid + n * Kt, slogq + n * Kt, static_cast<int>(i - n * Kt), Kt);
  if (q < 0.f) return;
  if (ds) {
    const float p = expf(z[i] - lse[n]);
    const float o = (p * coef[n] - g * q) * f[0];
    const int64_t at = static_cast<int64_t>(v - v0) * ld_ds + n;
    if constexpr (kBF16) static_cast<__nv_bfloat16*>(ds)[at] = __float2bfloat16_rn(o);
    else static_cast<__half*>(ds)[at] = __float2half_rn(o);
  }
  if (db) {
    const double d = ldexp(-static_cast<double>(g) * q, static_cast<int>(f[2]));
    const long long hi = __double2ll_rn(d), lo = __double2ll_rn(ldexp(d - static_cast<double>(hi), static_cast<int>(f[3])));
    if (hi) atomicAdd(db + 2ll * v, static_cast<unsigned long long>(hi));
    if (lo) atomicAdd(db + 2ll * v + 1, static_cast<unsigned long long>(lo));
  }
}

// db[v] of a chunk: the token splits' partial sums in split order, and the teacher's part.
__global__ void db_kernel(int rows, int v0, int TS, const float* __restrict__ part, const unsigned long long* __restrict__ fix,
                          const float* __restrict__ f, void* gb, int gb_dt) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= rows) return;
  const float* p = part + static_cast<int64_t>(i / 256) * TS * 256 + i % 256;
  double s = 0;
  for (int t = 0; t < TS; ++t) s += static_cast<double>(p[t * 256]);
  const long long hi = static_cast<long long>(fix[2ll * (v0 + i)]), lo = static_cast<long long>(fix[2ll * (v0 + i) + 1]);
  s += ldexp(static_cast<double>(hi) + ldexp(static_cast<double>(lo), -static_cast<int>(f[3])), -static_cast<int>(f[2]));
  store_d(gb, gb_dt, v0 + i, s);
}

// dh from its slices of accumulators, added in slice order.  Bound by HBM: 8192 x 2560, one slice (126 MB): 26 us.
__global__ void cast_scaled_kernel(const float* __restrict__ src, int slices, int64_t slice, const float* __restrict__ f,
                                   void* dst, int dt, int64_t n) {
  const float k = f[1];
  for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    float v = src[i];
    for (int s = 1; s < slices; ++s) v += src[s * slice + i];
    store_f(dst, dt, i, v * k);
  }
}

// ------------------------------------------------------------------ exact path (fp32 / fp64)
template <typename A>
__global__ void scaled_bias_kernel(int64_t V, const void* bias, int dt, A inv_T, A* out) {
  const int64_t v = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
  if (v < V) out[v] = static_cast<A>(load_d(bias, dt, v)) * inv_T;
}

// One block per token: picks the teacher's scores of the chunk, then updates (m, l) with the row.  256 rows of 1000: 3.7 us.
template <typename A>
__global__ void __launch_bounds__(256)
    exact_update_kernel(const A* __restrict__ S, int64_t C, int64_t pitch, int v0, int Kt, const int32_t* __restrict__ sid, A* z, A* m,
                        A* l) {
  __shared__ A sh[32];
  const int64_t n = blockIdx.x;
  const A* row = S + n * pitch;
  for (int k = threadIdx.x; k < Kt; k += blockDim.x) {
    const int32_t v = sid[n * Kt + k];
    if (v >= v0 && v < v0 + C) z[n * Kt + k] = row[v - v0];
  }
  A mx = -INFINITY;
  for (int64_t c = threadIdx.x; c < C; c += blockDim.x) mx = row[c] > mx ? row[c] : mx;
  mx = simt::block_reduce<A>(mx, true, sh);
  const A m_old = v0 == 0 ? -static_cast<A>(INFINITY) : m[n], m_new = m_old > mx ? m_old : mx;
  const A shift = isinf(m_new) ? A(0) : m_new;
  A sum = 0;
  for (int64_t c = threadIdx.x; c < C; c += blockDim.x) sum += exp_a(row[c] - shift);
  sum = simt::block_reduce<A>(sum, false, sh);
  if (threadIdx.x == 0) {
    l[n] = (v0 == 0 ? A(0) : l[n] * exp_a(m_old - shift)) + sum;
    m[n] = m_new;
  }
}

// dS of a chunk in place of S: a block per token writes the dense row and zeros up to the pitch, then the teacher's
// entries over it.
template <typename A>
__global__ void __launch_bounds__(256)
    exact_grad_kernel(int64_t C, int64_t pitch, int Kt, int v0, const int32_t* __restrict__ sid, const A* __restrict__ slogq,
                      const A* __restrict__ z, const A* __restrict__ lse, const A* __restrict__ lse_lo,
                      const A* __restrict__ gT, const A* __restrict__ coef, A* S) {
  const int64_t n = blockIdx.x;
  const A c = coef[n], g = gT[n], hi = lse[n], lo = lse_lo[n];
  A* row = S + n * pitch;
  for (int64_t i = threadIdx.x; i < pitch; i += blockDim.x)
    row[i] = i >= C || c == A(0) ? A(0) : exp_a((row[i] - hi) - lo) * c;
  if (g == A(0)) return;
  __syncthreads();
  for (int j = threadIdx.x; j < Kt; j += blockDim.x) {
    const int32_t v = sid[n * Kt + j];
    if (v < v0 || v >= v0 + C) continue;
    const A q = merged_q(sid + n * Kt, slogq + n * Kt, j, Kt);
    if (q < A(0)) continue;
    row[v - v0] = exp_a((z[n * Kt + j] - hi) - lo) * c - g * q;
  }
}

// ------------------------------------------------------------------ host
// Shortest part of a split sum: a 32-deep step of the fp32 product takes 1.3 us, its reduction 3 us (N = 256, K = 64,
// V = 1000: dh 120 -> 19 us, dW 40 -> 16 us).
constexpr int64_t kLeastK = 64;

static int check(const swvr_distill* p) {
  if (!p) return fail(SWVR_ERR_INVALID_ARGUMENT, "problem is NULL");
  if (p->n_tokens < 0 || p->hidden < 0 || p->vocab < 0 || p->teacher < 0)
    return fail(SWVR_ERR_INVALID_ARGUMENT, "negative size");
  // (a tile's last row index fits an int)
  if (p->n_tokens > (1ll << 31) - 512 || p->vocab > (1ll << 31) - 512 || p->hidden > (1ll << 31) - 512)
    return fail(SWVR_ERR_UNSUPPORTED, "sizes must be at most 2^31 - 512");
  if (!is_tc(p->compute_dtype) && p->n_tokens > simt::kMostRows)
    return fail(SWVR_ERR_UNSUPPORTED, "at most %lld tokens in fp32 / fp64", (long long)simt::kMostRows);
  if (p->teacher > kMaxTeacher)
    return fail(SWVR_ERR_UNSUPPORTED, "at most %d teacher entries per token, got %lld", kMaxTeacher, (long long)p->teacher);
  if (p->compute_dtype < SWVR_F32 || p->compute_dtype > SWVR_F16)
    return fail(SWVR_ERR_INVALID_ARGUMENT, "unknown compute dtype %d", p->compute_dtype);
  if ((p->bias && (p->bias_dtype < SWVR_F32 || p->bias_dtype > SWVR_F16)) || p->teacher_dtype < SWVR_F32 ||
      p->teacher_dtype > SWVR_F16)
    return fail(SWVR_ERR_INVALID_ARGUMENT, "unknown bias or teacher dtype");
  if (p->id_bits != 32 && p->id_bits != 64) return fail(SWVR_ERR_INVALID_ARGUMENT, "ids must be 32- or 64-bit integers");
  if (p->chunk <= 0) return fail(SWVR_ERR_INVALID_ARGUMENT, "chunk must be positive, got %lld", (long long)p->chunk);
  if (!(p->temperature > 0.0) || !std::isfinite(p->temperature))
    return fail(SWVR_ERR_INVALID_ARGUMENT, "temperature must be positive and finite, got %g", p->temperature);
  if (p->reduction < SWVR_REDUCE_NONE || p->reduction > SWVR_REDUCE_MEAN)
    return fail(SWVR_ERR_INVALID_ARGUMENT, "unknown reduction %d", p->reduction);
  if (p->ldh < p->hidden || p->ldw < p->hidden)
    return fail(SWVR_ERR_INVALID_ARGUMENT, "row stride smaller than the row length");
  if (p->n_tokens > 0) {
    if (p->vocab == 0) return fail(SWVR_ERR_UNSUPPORTED, "empty vocabulary");
    if ((p->hidden > 0 && (!p->h || !p->W)) || !p->lse || !p->lse_lo || !p->qsum || !p->each ||
        (p->teacher > 0 && (!p->teacher_ids || !p->teacher_logits || !p->sid || !p->slogq || !p->z)))
      return fail(SWVR_ERR_INVALID_ARGUMENT, "NULL pointer");
  }
  if (p->reduction != SWVR_REDUCE_NONE && !p->stats) return fail(SWVR_ERR_INVALID_ARGUMENT, "SUM / MEAN need stats");
  if (is_tc(p->compute_dtype)) {
    if (p->hidden < 8 || (p->hidden % 8) != 0 || (p->ldh % 8) != 0 || (p->ldw % 8) != 0)
      return fail(SWVR_ERR_UNSUPPORTED, "tensor-core path needs K and row strides that are multiples of 8 elements");
    if ((reinterpret_cast<uintptr_t>(p->h) | reinterpret_cast<uintptr_t>(p->W)) & 15u)
      return fail(SWVR_ERR_UNSUPPORTED, "tensor-core path needs 16-byte aligned h and W");
  }
  return SWVR_OK;
}

struct LsePlan {
  int MT, BT, splits, per, units, pairs;
  size_t off_l, off_done, bytes;
};

// Splits of the vocabulary per 256-token tile: the rounds over the pairs times the tiles of a unit, least.
static LsePlan plan_lse(const swvr_distill& p) {
  LsePlan f{};
  f.pairs = std::max(1, num_sms() / 2);
  f.MT = static_cast<int>(ceil_div(p.n_tokens, 256));
  f.BT = static_cast<int>(ceil_div(p.vocab, 256));
  int best = 1;
  int64_t best_cost = -1;
  for (int s = 1; s <= std::min(std::max(f.BT, 1), 148); ++s) {
    const int64_t cost = ceil_div(static_cast<int64_t>(f.MT) * s, f.pairs) * ceil_div(f.BT, s);
    if (best_cost < 0 || cost < best_cost) best_cost = cost, best = s;
  }
  f.per = static_cast<int>(ceil_div(std::max(f.BT, 1), best));
  f.splits = static_cast<int>(ceil_div(std::max(f.BT, 1), f.per));
  f.units = f.MT * f.splits;
  const size_t rows = static_cast<size_t>(f.units) * 256;
  f.off_l = align_up(rows * 4, 256);
  f.off_done = f.off_l + align_up(rows * 4, 256);
  f.bytes = f.off_done + 256;
  return f;
}

static size_t acc_size(const swvr_distill& p) { return p.compute_dtype == SWVR_F64 ? 8 : 4; }

struct ExactPlan {
  int64_t C;
  size_t off_bias, off_m, off_l, off_done, off_dh, off_part, bytes;
};

static ExactPlan plan_exact(const swvr_distill& p, bool need_h, bool need_W) {
  ExactPlan e{};
  const size_t es = acc_size(p);
  e.C = std::min({p.chunk, std::max<int64_t>(p.vocab, 1), simt::kMostRows});  // a chunk's rows are those of its dW product
  size_t off = align_up(es * p.n_tokens * round_up(e.C, 4), 256);  // rows of a multiple of 4: 16-byte staging
  e.off_bias = off;
  off += align_up(es * p.vocab, 256);
  e.off_m = off;
  off += align_up(es * p.n_tokens, 256);
  e.off_l = off;
  off += align_up(es * p.n_tokens, 256);
  e.off_done = off;
  off += 256;
  e.off_dh = off;
  if (need_h) off += align_up(es * p.n_tokens * p.hidden, 256);
  // slices of dh and dW split along their sums, where 128 x 128 tiles would leave SMs idle (simt::gemm_split)
  e.off_part = off;
  if (es == 4)
    off += align_up(4 * std::max(need_h ? simt::splitk_floats(p.n_tokens, p.hidden) : 0,
                                 need_W ? simt::splitk_floats(e.C, p.hidden) : 0), 256);
  e.bytes = off + 256;
  return e;
}

struct GradPlan {
  int NT, C, pairs, max_units;
  int64_t Npad;
  bool need_h, need_W, need_b;
  int slices;     // of dh's accumulators
  size_t off_gT, off_coef, off_f, off_fix, off_dh, off_db, off_ds, clear, bytes;
};

static GradPlan plan_grad(const swvr_distill& p, const swvr_distill_grads& g) {
  GradPlan b{};
  b.pairs = std::max(1, num_sms() / 2);
  b.NT = static_cast<int>(ceil_div(p.n_tokens, 256));
  b.Npad = static_cast<int64_t>(b.NT) * 256;
  // equal chunks of at most 2 * chunk rows, as the readout's backward (plan_bwd in abi.cu)
  const int64_t cmax = round_up(2 * std::min<int64_t>(p.chunk, 1ll << 30), 256), V = std::max<int64_t>(p.vocab, 1);
  b.C = static_cast<int>(std::min<int64_t>(round_up(ceil_div(V, ceil_div(V, cmax)), 256), 1ll << 30));
  b.need_h = g.grad_h != nullptr;
  b.need_W = g.grad_W != nullptr;
  b.need_b = g.grad_bias != nullptr && p.bias != nullptr;
  b.max_units = 1;
  for (int64_t rows : {static_cast<int64_t>(b.C), p.vocab % b.C}) {
    if (rows <= 0) continue;
    const int VTc = static_cast<int>(ceil_div(rows, 256));
    int TS, per;
    choose_ts(VTc, b.NT, b.pairs, &TS, &per);
    b.max_units = std::max(b.max_units, VTc * TS);
  }
  size_t off = 0;
  b.off_gT = off;
  off += align_up(p.n_tokens * acc_size(p), 256);
  b.off_coef = off;
  off += align_up(p.n_tokens * acc_size(p), 256);
  b.off_f = off;
  off += 256;
  b.slices = 1;
  if (is_tc(p.compute_dtype)) {
    // few tokens: dh has few tiles and each sums over the whole chunk, so the sum is dealt over slices while that
    // fills pairs that would be idle (517 tokens, K = 512, V = 10007: the GEMMs 57 -> 22 us)
    const int64_t tiles = b.NT * ceil_div(p.hidden, 256), kblocks = b.C / 128;
    if (b.need_h && tiles > 0)
      b.slices = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({b.pairs / tiles, kblocks / 4, 16})));
    b.off_fix = off;
    if (b.need_b) off += align_up(p.vocab * 16, 256);
    b.off_dh = off;
    if (b.need_h) off += align_up(static_cast<size_t>(b.slices > 1 ? b.slices * b.Npad : p.n_tokens) * p.hidden * 4, 256);
    b.clear = off - b.off_fix;
    b.off_db = off;
    if (b.need_b) off += align_up(static_cast<size_t>(b.max_units) * 256 * 4, 256);
    b.off_ds = off;
    off += align_up(static_cast<size_t>(b.C) * b.Npad * 2, 256);
  }
  b.bytes = off + 256;
  return b;
}

template <typename A>
static cudaError_t teacher_rows(const swvr_distill& p, uint32_t* done, cudaStream_t st) {
  const size_t smem = static_cast<size_t>(kWarps) * p.teacher * (sizeof(A) + 4);
  auto kern = teacher_kernel<A>;
  const cudaError_t e = tc::allow_smem(reinterpret_cast<const void*>(kern), kWarps * kMaxTeacher * (static_cast<int>(sizeof(A)) + 4));
  if (e != cudaSuccess) return e;
  kern<<<static_cast<unsigned>(ceil_div(p.n_tokens, kWarps)), 32 * kWarps, smem, st>>>(
      p.n_tokens, p.vocab, static_cast<int>(p.teacher), p.teacher_ids, p.id_bits, p.teacher_logits, p.teacher_dtype,
      static_cast<const A*>(p.teacher_lse), static_cast<A>(1.0 / p.temperature), p.sid, static_cast<A*>(p.slogq),
      static_cast<A*>(p.qsum), done);
  return cudaGetLastError();
}

template <typename A>
__global__ void empty_kernel(bool mean, A* out, A* stats) {  // no tokens: a sum of 0, a mean of 0 / 0
  *out = stats[0] = mean ? static_cast<A>(NAN) : A(0);
  stats[1] = mean ? A(0) : A(1);
}

template <typename A>
static cudaError_t losses(const swvr_distill& p, int splits, const A* m, const A* l, void* out, uint32_t* done, cudaStream_t st) {
  const int64_t N = p.n_tokens;
  if (N > 0)
    each_kernel<A><<<static_cast<unsigned>(ceil_div(N, kWarps)), 32 * kWarps, 0, st>>>(
        N, static_cast<int>(p.teacher), splits, m, l, p.sid, static_cast<const A*>(p.slogq), static_cast<const A*>(p.z),
        static_cast<const A*>(p.qsum), static_cast<A>(p.temperature * p.temperature), static_cast<A*>(p.lse),
        static_cast<A*>(p.lse_lo), static_cast<A*>(p.each), p.reduction, static_cast<const A*>(p.weight),
        static_cast<A*>(out), static_cast<A*>(p.stats), done);
  else if (p.reduction != SWVR_REDUCE_NONE)
    empty_kernel<A><<<1, 1, 0, st>>>(p.reduction == SWVR_REDUCE_MEAN, static_cast<A*>(out), static_cast<A*>(p.stats));
  return cudaGetLastError();
}

static void head_scores(const swvr_distill& p, tc::HeadParams* h) {
  h->K = static_cast<int>(p.hidden);
  h->N = static_cast<int>(p.n_tokens);
  h->sc2 = static_cast<float>(p.logit_scale / p.temperature * 1.4426950408889634);
  h->bias2 = static_cast<float>(1.4426950408889634 / p.temperature);
  h->bias = p.bias;
  h->bias_dt = p.bias_dtype;
}

static int tc_fwd_distill(const swvr_distill& p, void* out, void* ws, size_t wsb, cudaStream_t st) {
  const LsePlan f = plan_lse(p);
  if (wsb < f.bytes) return fail(SWVR_ERR_WORKSPACE, "workspace %zu < required %zu", wsb, f.bytes);
  float* m2 = static_cast<float*>(ws);
  float* l = reinterpret_cast<float*>(static_cast<char*>(ws) + f.off_l);
  uint32_t* done = reinterpret_cast<uint32_t*>(static_cast<char*>(ws) + f.off_done);
  if (p.n_tokens > 0) {
    tc::HeadMaps maps;
    SWVR_TRY(make_map(&maps.a, p.h, p.compute_dtype, p.hidden, p.n_tokens, p.ldh * 2, 64, 128));
    SWVR_TRY(make_map(&maps.b, p.W, p.compute_dtype, p.hidden, p.vocab, p.ldw * 2, 64, 128));
    {
      ProfScope ps(kProfDistill, st);
      SWVR_CUDA(teacher_rows<float>(p, done, st));
    }
    tc::HeadParams h{};
    head_scores(p, &h);
    h.MT = f.MT;
    h.BT = f.BT;
    h.splits = f.splits;
    h.per = f.per;
    h.units = f.units;
    h.gm = fwd_group(f.MT);
    h.V = static_cast<int>(p.vocab);
    h.part_m2 = m2;
    h.part_l = l;
    h.ids = p.sid;
    h.z = static_cast<float*>(p.z);
    h.Kt = static_cast<int>(p.teacher);
    ProfScope ps(kProfHead, st);
    SWVR_CUDA(p.compute_dtype == SWVR_BF16
                  ? tc::launch_head_any<true>(tc::kHeadLse, 256, maps, h, f.pairs, false, st)
                  : tc::launch_head_any<false>(tc::kHeadLse, 256, maps, h, f.pairs, false, st));
  }
  ProfScope ps(kProfDistill, st);
  SWVR_CUDA(losses<float>(p, f.splits, m2, l, out, done, st));
  return SWVR_OK;
}

template <typename A>
static cudaError_t exact_scores(const swvr_distill& p, int64_t v0, int64_t c, A* S, const A* bias, cudaStream_t st) {
  const int adt = sizeof(A) == 8 ? SWVR_F64 : SWVR_F32;
  return simt::gemm_bias<A>(st, p.n_tokens, c, p.hidden, static_cast<A>(p.logit_scale / p.temperature),
                            static_cast<const A*>(p.h), p.ldh, 1, static_cast<const A*>(p.W) + v0 * p.ldw, 1, p.ldw, S,
                            adt, bias, adt, v0, round_up(c, 4));
}

template <typename A>
static cudaError_t exact_bias(const swvr_distill& p, A* out, cudaStream_t st) {
  scaled_bias_kernel<A><<<static_cast<unsigned>(ceil_div(p.vocab, 256)), 256, 0, st>>>(
      p.vocab, p.bias, p.bias_dtype, static_cast<A>(1.0 / p.temperature), out);
  return cudaGetLastError();
}

template <typename A>
static int exact_fwd(const swvr_distill& p, void* out, void* ws, size_t wsb, cudaStream_t st) {
  const ExactPlan x = plan_exact(p, false, false);
  if (wsb < x.bytes) return fail(SWVR_ERR_WORKSPACE, "workspace %zu < required %zu", wsb, x.bytes);
  char* w = static_cast<char*>(ws);
  A *S = reinterpret_cast<A*>(w), *bias = p.bias ? reinterpret_cast<A*>(w + x.off_bias) : nullptr;
  A *m = reinterpret_cast<A*>(w + x.off_m), *l = reinterpret_cast<A*>(w + x.off_l);
  const int64_t N = p.n_tokens;
  uint32_t* done = reinterpret_cast<uint32_t*>(w + x.off_done);
  ProfScope ps(kProfDistill, st);
  if (N > 0) {
    SWVR_CUDA(teacher_rows<A>(p, done, st));
    if (bias) SWVR_CUDA(exact_bias<A>(p, bias, st));
    for (int64_t v0 = 0; v0 < p.vocab; v0 += x.C) {
      const int64_t c = std::min(x.C, p.vocab - v0);
      SWVR_CUDA(exact_scores<A>(p, v0, c, S, bias, st));
      exact_update_kernel<A><<<static_cast<unsigned>(N), 256, 0, st>>>(
          S, c, round_up(c, 4), static_cast<int>(v0), static_cast<int>(p.teacher), p.sid, static_cast<A*>(p.z), m, l);
      SWVR_CUDA(cudaGetLastError());
    }
  }
  SWVR_CUDA(losses<A>(p, 0, m, l, out, done, st));
  return SWVR_OK;
}

template <typename A>
static cudaError_t token_grads(const swvr_distill& p, const swvr_distill_grads& g, A* gT, A* coef, float* f, cudaStream_t st) {
  token_grad_kernel<A><<<1, kGradThreads, 0, st>>>(
      p.n_tokens, p.reduction, static_cast<A>(p.temperature), static_cast<const A*>(g.grad_out),
      static_cast<const A*>(p.weight), static_cast<const A*>(p.each), static_cast<const A*>(p.qsum),
      static_cast<const A*>(p.stats), gT, coef, static_cast<A*>(g.grad_weight), static_cast<float>(p.logit_scale),
      p.compute_dtype == SWVR_F16, f);
  return cudaGetLastError();
}

static int tc_bwd_distill(const swvr_distill& p, const swvr_distill_grads& g, const GradPlan& b, char* w, cudaStream_t st) {
  const int64_t N = p.n_tokens, K = p.hidden, V = p.vocab;
  const bool bf16 = p.compute_dtype == SWVR_BF16;
  float *gT = reinterpret_cast<float*>(w + b.off_gT), *coef = reinterpret_cast<float*>(w + b.off_coef);
  float* f = reinterpret_cast<float*>(w + b.off_f);
  unsigned long long* fix = b.need_b ? reinterpret_cast<unsigned long long*>(w + b.off_fix) : nullptr;
  float* part_db = b.need_b ? reinterpret_cast<float*>(w + b.off_db) : nullptr;
  void* ds = w + b.off_ds;
  float* dh = b.need_h ? reinterpret_cast<float*>(w + b.off_dh) : nullptr;
  {
    ProfScope ps(kProfDistill, st);
    SWVR_CUDA(token_grads<float>(p, g, gT, coef, f, st));
  }
  if (!(b.need_h || b.need_W || b.need_b)) return SWVR_OK;
  if (b.clear) SWVR_CUDA(cudaMemsetAsync(w + b.off_fix, 0, b.clear, st));  // db's fixed point and dh, side by side
  tc::HeadMaps maps;
  SWVR_TRY(make_map(&maps.a, p.W, p.compute_dtype, K, V, p.ldw * 2, 64, 128));
  SWVR_TRY(make_map(&maps.b, p.h, p.compute_dtype, K, N, p.ldh * 2, 64, 128));
  tc::GemmMaps gm;
  SWVR_TRY(make_map(&gm.h_mn, p.h, p.compute_dtype, K, N, p.ldh * 2, 64, 64));
  SWVR_TRY(make_map(&gm.w_mn, p.W, p.compute_dtype, K, V, p.ldw * 2, 64, 64));
  gm.gw = gm.dh = gm.w_mn;  // unused unless set
  if (b.need_W) {
    if (g.grad_W_dtype == SWVR_F32)
      SWVR_TRY(make_map(&gm.gw, g.grad_W, SWVR_F32, K, V, g.ld_grad_W * 4, 32, 128));
    else
      SWVR_TRY(make_map(&gm.gw, g.grad_W, p.compute_dtype, K, V, g.ld_grad_W * 2, 64, 128));
  }
  if (dh) SWVR_TRY(make_map(&gm.dh, dh, SWVR_F32, K, b.slices > 1 ? b.slices * b.Npad : N, K * 4, 32, 128));
  for (int64_t v0 = 0; v0 < V; v0 += b.C) {
    const int64_t v1 = std::min<int64_t>(v0 + b.C, V);
    const int rows = static_cast<int>(v1 - v0), VTc = static_cast<int>(ceil_div(rows, 256));
    int TS, per;
    choose_ts(VTc, b.NT, b.pairs, &TS, &per);
    tc::HeadParams h{};
    head_scores(p, &h);
    h.a_base = static_cast<int>(v0);
    h.MT = VTc;
    h.BT = b.NT;
    h.splits = TS;
    h.per = per;
    h.units = VTc * TS;
    h.gm = bwd_group(VTc);
    h.V = static_cast<int>(v1);
    h.lse = static_cast<const float*>(p.lse);
    h.coef = coef;
    h.factor = f;
    h.ds = ds;
    h.ld_ds = b.Npad;
    h.part_db = part_db;
    {
      ProfScope ps(kProfHead, st);
      SWVR_CUDA(bf16 ? tc::launch_head_any<true>(tc::kHeadGrad, 256, maps, h, b.pairs, v0 > 0, st)
                     : tc::launch_head_any<false>(tc::kHeadGrad, 256, maps, h, b.pairs, v0 > 0, st));
    }
    if (p.teacher > 0) {
      ProfScope ps(kProfDistill, st);
      const unsigned blocks = static_cast<unsigned>(ceil_div(N * p.teacher, 256));
      auto kern = bf16 ? entries_kernel<true> : entries_kernel<false>;
      kern<<<blocks, 256, 0, st>>>(N, static_cast<int>(p.teacher), static_cast<int>(v0), static_cast<int>(v1), p.sid,
                                   static_cast<const float*>(p.slogq), static_cast<const float*>(p.z),
                                   static_cast<const float*>(p.lse), gT, coef, f, ds, b.Npad, fix);
      SWVR_CUDA(cudaGetLastError());
    }
    if (part_db) {
      ProfScope ps(kProfDistill, st);
      db_kernel<<<static_cast<unsigned>(ceil_div(rows, 256)), 256, 0, st>>>(rows, static_cast<int>(v0), TS, part_db, fix,
                                                                            f, g.grad_bias, g.grad_bias_dtype);
      SWVR_CUDA(cudaGetLastError());
    }
    if (b.need_h || b.need_W) {
      SWVR_TRY(make_map(&gm.ds_k, ds, p.compute_dtype, b.Npad, rows, b.Npad * 2, 64, 128));
      SWVR_TRY(make_map(&gm.ds_mn, ds, p.compute_dtype, b.Npad, rows, b.Npad * 2, 64, 64));
      tc::GemmParams gp{};
      const int nt = static_cast<int>(ceil_div(K, 256));
      gp.dw_mt = VTc;
      gp.dw_nt = nt;
      gp.dw_kb = static_cast<int>(b.Npad / 64);
      gp.dw_tiles = b.need_W ? gp.dw_mt * nt : 0;
      gp.dh_mt = b.NT;
      gp.dh_nt = nt;
      gp.dh_kb = static_cast<int>(ceil_div(rows, 64));
      gp.dh_splits = std::max(1, std::min<int>(b.slices, static_cast<int>(ceil_div(gp.dh_kb, 2))));
      gp.dh_splits = static_cast<int>(ceil_div(ceil_div(gp.dh_kb, 2), ceil_div(ceil_div(gp.dh_kb, 2), gp.dh_splits)));  // none empty
      gp.dh_slice_rows = static_cast<int>(b.Npad);
      gp.dh_tiles = dh ? gp.dh_mt * nt * gp.dh_splits : 0;
      gp.v_begin = static_cast<int>(v0);
      gp.gw_f32 = g.grad_W_dtype == SWVR_F32 ? 1 : 0;
      gp.gw_scale = bf16 ? nullptr : f + 1;
      ProfScope ps(kProfGemm, st);
      SWVR_CUDA(tc::launch_gemm_kernel(bf16, gm, gp, b.pairs, /*pdl=*/true, st));
    }
  }
  if (dh) {
    ProfScope ps(kProfCast, st);
    const int64_t n = N * K;
    cast_scaled_kernel<<<static_cast<unsigned>(std::min<int64_t>(ceil_div(n, 256), 8 * kNumSMsB200)), 256, 0, st>>>(
        dh, b.slices, b.Npad * K, f, g.grad_h, g.grad_h_dtype, n);
    SWVR_CUDA(cudaGetLastError());
  }
  return SWVR_OK;
}

template <typename A>
static int exact_bwd(const swvr_distill& p, const swvr_distill_grads& g, const GradPlan& b, char* w, cudaStream_t st) {
  const ExactPlan x = plan_exact(p, b.need_h, b.need_W);
  const int64_t N = p.n_tokens, K = p.hidden, V = p.vocab;
  const int adt = sizeof(A) == 8 ? SWVR_F64 : SWVR_F32;
  const A s = static_cast<A>(p.logit_scale);
  A *gT = reinterpret_cast<A*>(w + b.off_gT), *coef = reinterpret_cast<A*>(w + b.off_coef);
  w += b.bytes;
  A *S = reinterpret_cast<A*>(w), *bias = p.bias ? reinterpret_cast<A*>(w + x.off_bias) : nullptr;
  A* dh = reinterpret_cast<A*>(w + x.off_dh);
  float* part = sizeof(A) == 4 ? reinterpret_cast<float*>(w + x.off_part) : nullptr;
  ProfScope ps(kProfDistill, st);
  SWVR_CUDA(token_grads<A>(p, g, gT, coef, static_cast<float*>(nullptr), st));
  if (!(b.need_h || b.need_W || b.need_b)) return SWVR_OK;
  if (bias) SWVR_CUDA(exact_bias<A>(p, bias, st));
  const bool one = x.C >= V;  // one chunk: dh goes straight to its place
  for (int64_t v0 = 0; v0 < V; v0 += x.C) {
    const int64_t c = std::min(x.C, V - v0), ld = round_up(c, 4);
    SWVR_CUDA(exact_scores<A>(p, v0, c, S, bias, st));
    exact_grad_kernel<A><<<static_cast<unsigned>(N), 256, 0, st>>>(
        c, ld, static_cast<int>(p.teacher), static_cast<int>(v0), p.sid, static_cast<const A*>(p.slogq),
        static_cast<const A*>(p.z), static_cast<const A*>(p.lse), static_cast<const A*>(p.lse_lo), gT, coef, S);
    if (b.need_b)
      simt::colsum_kernel<A><<<static_cast<unsigned>(ceil_div(c, 32)), 256, 0, st>>>(S, N, c, ld, g.grad_bias,
                                                                                    g.grad_bias_dtype, v0);
    SWVR_CUDA(cudaGetLastError());
    if (b.need_h)
      SWVR_CUDA(simt::gemm_split<A>(st, N, K, c, s, S, ld, 1, static_cast<const A*>(p.W) + v0 * p.ldw, p.ldw, 1,
                                    A(v0 ? 1 : 0), one ? g.grad_h : dh, one ? g.grad_h_dtype : adt, K, 1, part, kLeastK, true));
    if (b.need_W)
      SWVR_CUDA(simt::gemm_split<A>(st, c, K, N, s, S, 1, ld, static_cast<const A*>(p.h), p.ldh, 1, A(0),
                                    static_cast<char*>(g.grad_W) + static_cast<size_t>(v0 * g.ld_grad_W) * dtype_size(g.grad_W_dtype),
                                    g.grad_W_dtype, g.ld_grad_W, 1, part, kLeastK, true));
  }
  if (b.need_h && !one) {
    simt::cast_kernel<A><<<simt::grid_for(N * K), 256, 0, st>>>(dh, g.grad_h, g.grad_h_dtype, N * K);
    SWVR_CUDA(cudaGetLastError());
  }
  return SWVR_OK;
}

static size_t bwd_bytes(const swvr_distill& p, const GradPlan& b) {
  return b.bytes + (is_tc(p.compute_dtype) ? 0 : plan_exact(p, b.need_h, b.need_W).bytes);
}

}  // namespace distill
}  // namespace swvr

extern "C" {

int swvr_distill_fwd_workspace_size(const swvr_distill* p, size_t* bytes) {
  SWVR_TRY(distill::check(p));
  if (!bytes) return fail(SWVR_ERR_INVALID_ARGUMENT, "bytes is NULL");
  *bytes = is_tc(p->compute_dtype) ? distill::plan_lse(*p).bytes : distill::plan_exact(*p, false, false).bytes;
  return SWVR_OK;
}

int swvr_distill_fwd(const swvr_distill* p, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  SWVR_TRY(distill::check(p));
  if (!out && (p->n_tokens > 0 || p->reduction != SWVR_REDUCE_NONE)) return fail(SWVR_ERR_INVALID_ARGUMENT, "NULL output");
  if (!workspace && p->n_tokens > 0) return fail(SWVR_ERR_INVALID_ARGUMENT, "NULL workspace");
  if (!aligned16(workspace)) return fail(SWVR_ERR_UNSUPPORTED, "workspace not 16-byte aligned");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (is_tc(p->compute_dtype)) return distill::tc_fwd_distill(*p, out, workspace, workspace_bytes, st);
  if (p->compute_dtype == SWVR_F64) return distill::exact_fwd<double>(*p, out, workspace, workspace_bytes, st);
  return distill::exact_fwd<float>(*p, out, workspace, workspace_bytes, st);
}

int swvr_distill_bwd_workspace_size(const swvr_distill* p, const swvr_distill_grads* g, size_t* bytes) {
  SWVR_TRY(distill::check(p));
  if (!g || !bytes) return fail(SWVR_ERR_INVALID_ARGUMENT, "NULL argument");
  *bytes = distill::bwd_bytes(*p, distill::plan_grad(*p, *g));
  return SWVR_OK;
}

int swvr_distill_bwd(const swvr_distill* p, const swvr_distill_grads* g, void* workspace, size_t workspace_bytes,
                     void* stream) {
  SWVR_TRY(distill::check(p));
  if (!g || !g->grad_out) return fail(SWVR_ERR_INVALID_ARGUMENT, "grads or grad_out is NULL");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t N = p->n_tokens, K = p->hidden, V = p->vocab;
  if ((g->grad_h && (g->grad_h_dtype < SWVR_F32 || g->grad_h_dtype > SWVR_F16)) ||
      (g->grad_W && (g->grad_W_dtype < SWVR_F32 || g->grad_W_dtype > SWVR_F16)) ||
      (g->grad_bias && (g->grad_bias_dtype < SWVR_F32 || g->grad_bias_dtype > SWVR_F16)))
    return fail(SWVR_ERR_INVALID_ARGUMENT, "unknown gradient dtype");
  if (g->grad_W && g->ld_grad_W < K) return fail(SWVR_ERR_INVALID_ARGUMENT, "row stride smaller than the row length");
  if (g->grad_weight && !p->weight) return fail(SWVR_ERR_INVALID_ARGUMENT, "grad_weight without weight");
  if (g->grad_W && is_tc(p->compute_dtype)) {
    if (g->grad_W_dtype != p->compute_dtype && g->grad_W_dtype != SWVR_F32)
      return fail(SWVR_ERR_UNSUPPORTED, "grad_W must be in the compute dtype or fp32");
    if ((reinterpret_cast<uintptr_t>(g->grad_W) & 15u) || (g->ld_grad_W * dtype_size(g->grad_W_dtype)) % 16)
      return fail(SWVR_ERR_UNSUPPORTED, "grad_W must be 16-byte aligned with a 16-byte multiple row pitch");
  }
  if (N == 0) {
    if (g->grad_W) SWVR_CUDA(small::zero_rows(g->grad_W, g->grad_W_dtype, V, K, g->ld_grad_W, st));
    if (g->grad_bias) SWVR_CUDA(small::zero_rows(g->grad_bias, g->grad_bias_dtype, 1, V, V, st));
    return SWVR_OK;
  }
  const distill::GradPlan b = distill::plan_grad(*p, *g);
  const size_t need = distill::bwd_bytes(*p, b);
  if (workspace_bytes < need) return fail(SWVR_ERR_WORKSPACE, "workspace %zu < required %zu", workspace_bytes, need);
  if (!workspace) return fail(SWVR_ERR_INVALID_ARGUMENT, "NULL workspace");
  if (!aligned16(workspace)) return fail(SWVR_ERR_UNSUPPORTED, "workspace not 16-byte aligned");
  char* w = static_cast<char*>(workspace);
  if (is_tc(p->compute_dtype)) return distill::tc_bwd_distill(*p, *g, b, w, st);
  if (p->compute_dtype == SWVR_F64) return distill::exact_bwd<double>(*p, *g, b, w, st);
  return distill::exact_bwd<float>(*p, *g, b, w, st);
}

}  // extern "C"
