// Tensor-core (tcgen05) products of the head that keep no readout: S = h . W^T tile by tile with
// an epilogue in place of the P.E product of tc_fwd.cu.
//
// One kernel, three epilogues (kHeadLse, kHeadGrad, kHeadLogits).  A CTA pair (cluster of 2) computes
// 256 x BN tiles with tcgen05.mma.cta_group::2: each CTA stages its own 128 rows of A and its own
// BN / 2 rows of B per 128-wide K block, both K-major.  A work unit is one 256-row A tile and a
// range of B tiles; the accumulator is double-buffered in TMEM (2 x BN columns), so a
// tile's epilogue runs under the next tile's MMAs.  Warp 0 issues TMA loads, warp 1 of the even CTA
// issues MMAs, warps 4-7 are the epilogue; one thread owns one A row.
//
//  kHeadLse     A = h, B = W (BN = 256): a thread owns a token.  Online softmax statistics of its row,
//               and the scores of its teacher tokens, whose ids come sorted: the thread walks the
//               list as the vocabulary goes by and picks each score out of its registers.  A
//               unit leaves (m, l) of its vocabulary range.  At 256 x 256 tiles the MMAs of a tile take K * 8
//               cycles and the epilogue about 4000, so from K = 512 on it is hidden.  Bound by the tensor cores:
//               8192 tokens, K = 2560, V = 152064 in 4.5 ms = 1.41 PFLOP/s (tensor pipe 94 % of active cycles).
//  kHeadGrad    A = W rows of a vocabulary chunk, B = h (BN = 256): a thread owns a vocabulary row.
//               dS^T = 2^(S - lse) * coef[token], stored in the 16-bit compute dtype for the dW / dh GEMMs
//               (tc_gemm.cu); the row sum of dS (bias gradient) goes to a partial slot.  Same size: 5.6 ms =
//               1.13 PFLOP/s (tensor pipe 93 %), with 2.5 GB of dS stored.
//  kHeadLogits  A = W, B = h with BN = 32 .. 256 tokens: logits[token, v] in fp32; W streams through once
//               per BN tokens.  W is the 256-row operand and the tokens the narrow one: the other way round a token would
//               cost a 256-row tile.  Bound by HBM: 1 token, K = 2560, V = 152064 (778 MB) in 129 us = 6.0 TB/s;
//               64 tokens, K = 4096, V = 128256 (1050 MB) in 177 us = 5.9 TB/s.
#include "ptx.cuh"
#include "tc.cuh"

namespace swvr {
namespace tc {

enum HeadMode { kHeadLse = 0, kHeadGrad, kHeadLogits };

struct HeadParams {
  int K;
  int a_base;                  // first row of A (the chunk's first vocabulary row)
  int MT, BT;                  // 256-row A tiles, BN-row B tiles
  int splits, per, units, gm;  // B splits per A tile, B tiles per split, MT * splits, unit order (fwd_unit)
  int N, V;                    // tokens; end of the vocabulary rows (of the chunk for kHeadGrad)
  float scale;                 // kHeadLogits: logit_scale
  float sc2, bias2;            // log2(e) * logit_scale / T, log2(e) / T
  const void* bias;
  int bias_dt;
  // kHeadLse
  float* part_m2;              // [units * 256]
  float* part_l;
  const int32_t* ids;          // [N, Kt] ascending, ids >= V behind the others
  float* z;                    // [N, Kt] scores / T of those ids, natural units
  int Kt;
  // kHeadGrad
  const float* lse;            // [N] natural units, at temperature T
  const float* coef;           // [N]
  const float* factor;         // [1] on the device: what dS is multiplied by when it is stored
  void* ds;                    // [rows of the chunk, ld_ds]
  int64_t ld_ds;
  float* part_db;              // [units * 256] or null
  // kHeadLogits
  float* logits;
  int64_t ld_logits;
};

struct HeadMaps {
  CUtensorMap a;  // box {64, 128}
  CUtensorMap b;  // box {64, BN / 2}
};

__device__ __forceinline__ void head_unit(const HeadParams& p, int u, int* mt, int* sp) {
  const int gsize = p.gm * p.splits;
  const int grp = u / gsize, r = u % gsize;
  const int rows = min(p.gm, p.MT - grp * p.gm);
  *sp = r / rows;
  *mt = grp * p.gm + r % rows;
}

template <int BN_, int NS>
struct HeadCfg {
  static constexpr int BN = BN_, KH = 2;
  static constexpr int BOXA = 128 * 128, BOXB = (BN / 2) * 128;
  static constexpr int A_BYTES = KH * BOXA, B_BYTES = KH * BOXB;
  static constexpr int SMEM_A = 0;
  static constexpr int SMEM_B = NS * A_BYTES;
  static constexpr int SMEM_ROW = SMEM_B + NS * B_BYTES;  // 2 x 2 x 256 floats: per-column values of a tile
  static constexpr int SMEM_BAR = SMEM_ROW + 4 * 256 * 4;
  static constexpr int NBAR = 2 * NS + 5;
  static constexpr int SMEM_ALLOC = SMEM_BAR + NBAR * 8 + 16 + 1024;
  static constexpr uint32_t TMEM_COLS = 2 * BN < 32 ? 32 : 2 * BN;
  static_assert(SMEM_ALLOC <= 232448, "shared memory budget");
  static_assert(BN == 32 || BN == 64 || BN == 128 || BN == 256, "column tile");
  static_assert(BOXB % 1024 == 0, "1024-byte alignment");
};

// x[i] for a run-time i: five levels of selects (a dynamic register index would go to local memory)
__device__ __forceinline__ float pick32(const float (&x)[32], int i) {
  float a[16], b[8], c[4];
#pragma unroll
  for (int k = 0; k < 16; ++k) a[k] = (i & 16) ? x[k + 16] : x[k];
#pragma unroll
  for (int k = 0; k < 8; ++k) b[k] = (i & 8) ? a[k + 8] : a[k];
#pragma unroll
  for (int k = 0; k < 4; ++k) c[k] = (i & 4) ? b[k + 4] : b[k];
  const float d0 = (i & 2) ? c[2] : c[0], d1 = (i & 2) ? c[3] : c[1];
  return (i & 1) ? d1 : d0;
}

template <bool kBF16, int MODE, int BN_, int NS>
__global__ void __launch_bounds__(256, 1)
    head_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const HeadParams p) {
  using Cfg = HeadCfg<BN_, NS>;
  constexpr int BN = BN_, KH = Cfg::KH;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::SMEM_BAR);
  uint64_t* full = bars;               // [NS] leader's copy counts both CTAs' bytes
  uint64_t* empty = bars + NS;         // [NS] both CTAs (multicast commit)
  uint64_t* acc_full = bars + 2 * NS;  // [2]  both CTAs (multicast commit)
  uint64_t* acc_empty = acc_full + 2;  // [2]  leader's copy: one arrival per CTA
  uint64_t* spare = acc_empty + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + Cfg::NBAR);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  float* row_s = reinterpret_cast<float*>(smem + Cfg::SMEM_ROW);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2);
    }
    mbar_init(spare, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tm_a);
    tma_prefetch_desc(&tm_b);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_holder, Cfg::TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // the peer's barriers are initialised before any remote arrive
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  if (threadIdx.x == 0) pdl_trigger();
  const int KB = (p.K + 64 * KH - 1) / (64 * KH);

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------------------ TMA producer (both CTAs)
      uint32_t stage = 0, sphase = 0;
      for (int u = pair; u < p.units; u += npairs) {
        int mt, sp;
        head_unit(p, u, &mt, &sp);
        const int t0 = sp * p.per, t1 = min(t0 + p.per, p.BT);
        const int arow = p.a_base + mt * 256 + static_cast<int>(rank) * 128;
        for (int t = t0; t < t1; ++t) {
          const int brow = t * BN + static_cast<int>(rank) * (BN / 2);
          for (int kb = 0; kb < KB; ++kb) {
            if (!mbar_wait(&empty[stage], sphase ^ 1u, abort_flag, kErrHead | 1)) goto done;
            if (leader) mbar_arrive_expect_tx(&full[stage], 2 * (Cfg::A_BYTES + Cfg::B_BYTES));
            const uint32_t fb = mapa_shared(smem_u32(&full[stage]), 0);
#pragma unroll
            for (int hk = 0; hk < KH; ++hk) {
              const int k0 = (kb * KH + hk) * 64;  // past K the boxes read zero fill
              tma_load_2d_pair(smem + Cfg::SMEM_A + stage * Cfg::A_BYTES + hk * Cfg::BOXA, &tm_a, fb, k0, arow);
              tma_load_2d_pair(smem + Cfg::SMEM_B + stage * Cfg::B_BYTES + hk * Cfg::BOXB, &tm_b, fb, k0, brow);
            }
            if (++stage == NS) {
              stage = 0;
              sphase ^= 1u;
            }
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      // ------------------------------------------------------------ MMA issuer (leader only)
      const uint32_t id = idesc_f16(kBF16, 256, BN, false, false);
      const uint64_t da0 = sdesc_sw128(smem_u32(smem + Cfg::SMEM_A), 16, 1024);
      const uint64_t db0 = sdesc_sw128(smem_u32(smem + Cfg::SMEM_B), 16, 1024);
      uint32_t stage = 0, sphase = 0, g = 0;
      for (int u = pair; u < p.units; u += npairs) {
        int mt, sp;
        head_unit(p, u, &mt, &sp);
        const int t0 = sp * p.per, t1 = min(t0 + p.per, p.BT);
        for (int t = t0; t < t1; ++t, ++g) {
          const uint32_t b = g & 1u;
          if (!mbar_wait(&acc_empty[b], ((g >> 1) & 1u) ^ 1u, abort_flag, kErrHead | 2)) goto done;
          tc_fence_after();
          for (int kb = 0; kb < KB; ++kb) {
            if (!mbar_wait(&full[stage], sphase, abort_flag, kErrHead | 3)) goto done;
            const uint64_t sa = static_cast<uint64_t>(stage * (Cfg::A_BYTES >> 4));
            const uint64_t sb = static_cast<uint64_t>(stage * (Cfg::B_BYTES >> 4));
#pragma unroll
            for (int k8 = 0; k8 < 4 * KH; ++k8)
              umma2_ss(tmem + b * BN, da0 + sa + (k8 >> 2) * (Cfg::BOXA >> 4) + (k8 & 3) * 2,
                       db0 + sb + (k8 >> 2) * (Cfg::BOXB >> 4) + (k8 & 3) * 2, id, (kb | k8) ? 1u : 0u);
            umma2_commit_mc(&empty[stage], 3);
            if (++stage == NS) {
              stage = 0;
              sphase ^= 1u;
            }
          }
          umma2_commit_mc(&acc_full[b], 3);
        }
      }
    }
  } else if (warp >= 4) {
    // -------------------------------------------------------------- epilogue warps (both CTAs)
    const int r = threadIdx.x - 128;
    const uint32_t trow = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t acc_empty_leader = mapa_shared(smem_u32(acc_empty), 0);
    const float2 sc2v = make_float2(p.sc2, p.sc2);
    uint32_t g = 0;
    if constexpr (MODE == kHeadGrad) pdl_wait();  // dS of the chunk before is still read until then
    for (int u = pair; u < p.units; u += npairs) {
      int mt, sp;
      head_unit(p, u, &mt, &sp);
      const int t0 = sp * p.per, t1 = min(t0 + p.per, p.BT);
      if (t1 <= t0) continue;
      const int arow = mt * 256 + static_cast<int>(rank) * 128 + r;  // token, or row within the chunk
      // state of the row over the unit
      float ref = -INFINITY, l = 0.f;          // kHeadLse
      int j = 0, nxt = INT_MAX;
      const int32_t* ids = nullptr;
      float2 db = make_float2(0.f, 0.f);       // kHeadGrad
      float brow = 0.f;                        // kHeadGrad, kHeadLogits: the row's bias
      const int vrow = p.a_base + arow;
      if constexpr (MODE == kHeadLse) {
        if (p.Kt > 0 && arow < p.N) {
          ids = p.ids + static_cast<int64_t>(arow) * p.Kt;
          int lo = 0, hi = p.Kt;  // first id of this unit's vocabulary range
          while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (ids[mid] < t0 * BN) lo = mid + 1;
            else hi = mid;
          }
          j = lo;
          nxt = j < p.Kt ? ids[j] : INT_MAX;
        }
      } else {
        if (p.bias != nullptr && vrow < p.V)
          brow = load_f(p.bias, p.bias_dt, vrow) * (MODE == kHeadGrad ? p.bias2 : 1.f);
      }
      const float fac = MODE == kHeadGrad ? *p.factor : 0.f;
      for (int t = t0; t < t1; ++t, ++g) {
        const uint32_t b = g & 1u;
        const int c0 = t * BN;  // first column: vocabulary row, or token
        float* rs = row_s + b * 512;
        if constexpr (MODE == kHeadLse) {
          // bias of the columns in log2 units; -inf past V masks them
          for (int c = r; c < BN; c += 128)
            rs[c] = c0 + c < p.V ? (p.bias ? load_f(p.bias, p.bias_dt, c0 + c) * p.bias2 : 0.f) : -INFINITY;
        } else if constexpr (MODE == kHeadGrad) {
          // tokens past N, and those whose gradient is zero, get p = 0 (whatever their lse is)
          for (int c = r; c < BN; c += 128) {
            const float cf = c0 + c < p.N ? p.coef[c0 + c] : 0.f;
            rs[c] = cf != 0.f ? -p.lse[c0 + c] * kLog2e : -INFINITY;
            rs[256 + c] = cf;
          }
        }
        if constexpr (MODE != kHeadLogits) named_bar_sync(1, 128);
        if (!warp_wait(&acc_full[b], (g >> 1) & 1u, abort_flag, kErrHead | 4)) goto done;
        tc_fence_after();
        const uint32_t sbase = trow + b * BN;
        float lt = 0.f;  // kHeadLse: the tile's sum
#pragma unroll 1
        for (int c = 0; c < BN / 32; ++c) {
          uint32_t x[32];
          tmem_ld32(sbase + c * 32, x);
          tmem_wait_ld();
          if constexpr (MODE == kHeadLse) {
            const float4* b4 = reinterpret_cast<const float4*>(rs + c * 32);
            float v[32];
            float mx = -INFINITY;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const float4 bb = b4[q];
              const float2 v0 = ffma2(make_float2(__uint_as_float(x[4 * q]), __uint_as_float(x[4 * q + 1])), sc2v,
                                      make_float2(bb.x, bb.y));
              const float2 v1 = ffma2(make_float2(__uint_as_float(x[4 * q + 2]), __uint_as_float(x[4 * q + 3])), sc2v,
                                      make_float2(bb.z, bb.w));
              v[4 * q] = v0.x, v[4 * q + 1] = v0.y, v[4 * q + 2] = v1.x, v[4 * q + 3] = v1.y;
              mx = fmaxf(mx, fmaxf(fmaxf(v0.x, v0.y), fmaxf(v1.x, v1.y)));
            }
            while (nxt < c0 + c * 32 + 32) {
              p.z[static_cast<int64_t>(arow) * p.Kt + j] = pick32(v, nxt & 31) * kLn2;
              ++j;
              nxt = j < p.Kt ? ids[j] : INT_MAX;
            }
            // sums stay finite and exact enough while no score is 2^64 above the reference
            if (mx > ref + 32.f) {
              const float alpha = ref == -INFINITY ? 0.f : ex2(ref - mx);
              l *= alpha;
              lt *= alpha;
              ref = mx;
            }
            const float nref = ref == -INFINITY ? 0.f : -ref;
            float2 s = make_float2(0.f, 0.f);
#pragma unroll
            for (int q = 0; q < 16; ++q) {
              const float2 e = fadd2(make_float2(v[2 * q], v[2 * q + 1]), make_float2(nref, nref));
              s = fadd2(s, make_float2(ex2(e.x), ex2(e.y)));
            }
            lt += s.x + s.y;
          } else if constexpr (MODE == kHeadGrad) {
            const float4* L4 = reinterpret_cast<const float4*>(rs + c * 32);
            const float4* C4 = reinterpret_cast<const float4*>(rs + 256 + c * 32);
            const float2 b2v = make_float2(brow, brow), facv = make_float2(fac, fac);
            uint32_t pk[16];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const float4 nl = L4[q], cf = C4[q];
#pragma unroll
              for (int hh = 0; hh < 2; ++hh) {
                const int i = 4 * q + 2 * hh;
                const float2 bl = fadd2(b2v, hh ? make_float2(nl.z, nl.w) : make_float2(nl.x, nl.y));
                const float2 e = ffma2(make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), sc2v, bl);
                const float2 d = fmul2(make_float2(ex2(e.x), ex2(e.y)),
                                       hh ? make_float2(cf.z, cf.w) : make_float2(cf.x, cf.y));
                db = fadd2(db, d);
                const float2 o = fmul2(d, facv);
                pk[i / 2] = pack2<kBF16>(o.x, o.y);
              }
            }
            if (vrow < p.V) {
              uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.ds) +
                                                    static_cast<int64_t>(arow) * p.ld_ds + c0 + c * 32);
#pragma unroll
              for (int k = 0; k < 4; ++k) dst[k] = make_uint4(pk[4 * k], pk[4 * k + 1], pk[4 * k + 2], pk[4 * k + 3]);
            }
          } else {
            if (vrow < p.V) {
              float* dst = p.logits + static_cast<int64_t>(c0 + c * 32) * p.ld_logits + vrow;
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (c0 + c * 32 + i < p.N)
                  dst[static_cast<int64_t>(i) * p.ld_logits] = fmaf(__uint_as_float(x[i]), p.scale, brow);
            }
          }
        }
        l += lt;
        // every thread of this CTA has read its accumulator rows: release them to the leader
        tc_fence_before();
        named_bar_sync(1, 128);
        if (r == 0) mbar_arrive_cluster_relaxed(acc_empty_leader + b * 8);
      }
      const int64_t slot = static_cast<int64_t>(mt * p.splits + sp) * 256 + static_cast<int>(rank) * 128 + r;
      if constexpr (MODE == kHeadLse) {
        p.part_m2[slot] = ref;
        p.part_l[slot] = l;
      }
      if constexpr (MODE == kHeadGrad) {
        if (p.part_db) p.part_db[slot] = db.x + db.y;
      }
    }
  }
done:
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) drain_after_abort_pair(warp == 1 && lane == 0 && leader, spare);
  cluster_sync_all();  // neither CTA releases TMEM / shared memory while its peer may use them
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, Cfg::TMEM_COLS);
  }
}

template <bool kBF16, int MODE, int BN, int NS>
static cudaError_t launch_head(const HeadMaps& m, const HeadParams& prm, int max_pairs, bool pdl, cudaStream_t st) {
  using Cfg = HeadCfg<BN, NS>;
  auto kern = head_kernel<kBF16, MODE, BN, NS>;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.blockDim = dim3(256, 1, 1);
  cfg.dynamicSmemBytes = Cfg::SMEM_ALLOC;
  cfg.stream = st;
  cfg.gridDim = dim3(2 * 74, 1, 1);
  static KnownClusters known;
  int clusters = 0;
  const cudaError_t e = resident_clusters(reinterpret_cast<const void*>(kern), cfg, known, &clusters);
  if (e != cudaSuccess) return e;
  int pairs = std::min(std::min(clusters, max_pairs), prm.units);
  if (pairs < 1) pairs = 1;
  cfg.gridDim = dim3(2 * pairs, 1, 1);
  if (pdl) {
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
  }
  return cudaLaunchKernelEx(&cfg, kern, m.a, m.b, prm);
}

template <bool kBF16>
static cudaError_t launch_head_any(int mode, int BN, const HeadMaps& m, const HeadParams& prm, int max_pairs, bool pdl,
                                   cudaStream_t st) {
  if (mode == kHeadLse) return launch_head<kBF16, kHeadLse, 256, 3>(m, prm, max_pairs, pdl, st);
  if (mode == kHeadGrad) return launch_head<kBF16, kHeadGrad, 256, 3>(m, prm, max_pairs, pdl, st);
  if (BN == 32) return launch_head<kBF16, kHeadLogits, 32, 6>(m, prm, max_pairs, pdl, st);
  if (BN == 64) return launch_head<kBF16, kHeadLogits, 64, 5>(m, prm, max_pairs, pdl, st);
  if (BN == 128) return launch_head<kBF16, kHeadLogits, 128, 4>(m, prm, max_pairs, pdl, st);
  return launch_head<kBF16, kHeadLogits, 256, 3>(m, prm, max_pairs, pdl, st);
}

}  // namespace tc
}  // namespace swvr
