// ffn_narrow_sm100.cu -- the products of the gated feed-forward block for few
// tokens (one to some hundreds), on tcgen05 (sm_100a).
//
// With few tokens a product reads every weight once and uses it a few times: it
// is bound by the weights' bytes (402 MB for one token at 4096 x 16384), and
// the work is to keep all SMs loading.  So the roles are swapped: a tile is 128
// features, whose weights are the MMA's A operand, by up to 128 tokens as its
// B operand (N = the tokens, rounded up to 16).  No weight row is loaded for a
// token that is not there, and the epilogue has a thread per feature instead of
// one per token.
//
// Tiles are few (4096 features: 32), so a cluster of 1 to 8 CTAs shares a
// tile: each takes a part of K, leaves its fp32 partial in its own shared
// memory, and after a cluster barrier the CTAs add the parts of a share of the
// tokens each, in rank order, and finish those (the sums do not depend on which
// CTA came first).  Roundings are those of ffn_sm100.cu: sums are exchanged and
// finished in fp32; h, dgate and dup are rounded to bf16 once, as operands of the
// next product.
//
// The kernel that follows another (the second product of a call) starts while
// that one ends: its weights do not depend on it, so the first stages are loaded
// before it waits for the other's output.
#include <algorithm>

#include "ffn_common.cuh"

namespace ltx {

namespace {

constexpr int kNThreads = 256;  // 8 warps: a producer, an MMA issuer, and then all for the epilogue
constexpr int kNRows = 128;     // features of a tile (UMMA M)
constexpr int kNMaxStages = 6;
constexpr int kNMaxCluster = 8;
constexpr int kNarrowColumns = 128;  // tokens of a tile at most
constexpr uint32_t kNATile = kNRows * kFfnK * 2;
constexpr uint32_t kNChunk = 64 * kFfnK * 2;  // MN-major: 64 features x 64 rows of K
constexpr uint32_t kNStageSpace = 108 * 1024;  // two CTAs to an SM
// full, empty per stage, acc_full
constexpr uint32_t kNOffBar = kNStageSpace;
constexpr uint32_t kNOffCtl = kNOffBar + (2 * kNMaxStages + 1) * 8;
constexpr uint32_t kNSmem = kNOffCtl + 16 + 1024;  // + alignment slack
static_assert(2 * (kNSmem + 1024) <= 228 * 1024, "two CTAs to an SM");
// Partial sums, [accumulator column][128 features] fp32, take the stages' place: of so many tokens at a time.
template <NarrowMode kMode>
constexpr int kExchange = kNStageSpace / (kNRows * 4) / (kMode == kNarrowProduct ? 2 : 1) / 8 * 8;

// bytes of the weights in a stage
template <NarrowMode kMode>
constexpr uint32_t kWeights = kMode == kNarrowProduct ? 2 * kNATile : kNATile;

// 4 floats at the address that `local` has in this CTA, of the CTA with that rank (of this one: without the
// way through the cluster's network, which gives some 10 bytes a cycle to an SM).
__device__ __forceinline__ float4 peer_load4(uint32_t local, uint32_t rank, uint32_t own) {
  float4 v;
  if (rank == own) {
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(local)
                 : "memory");
    return v;
  }
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(peer_address(local, rank))
               : "memory");
  return v;
}

// The cluster's parts of 4 features (from `feature`) of one accumulator column.
struct Parts {
  float4 part[kNMaxCluster];

  // all on their way at once: a read of another CTA's shared memory takes a few hundred ns
  __device__ __forceinline__ void load(uint32_t partial, int column, int feature, uint32_t ranks, uint32_t own) {
    const uint32_t at = partial + (column * kNRows + feature) * 4;
#pragma unroll
    for (uint32_t r = 0; r < kNMaxCluster; ++r)
      if (r < ranks) part[r] = peer_load4(at, r, own);
  }
  __device__ __forceinline__ void sum(uint32_t ranks, float (&v)[4]) const {
    v[0] = part[0].x, v[1] = part[0].y, v[2] = part[0].z, v[3] = part[0].w;
#pragma unroll
    for (uint32_t r = 1; r < kNMaxCluster; ++r)
      if (r < ranks) v[0] += part[r].x, v[1] += part[r].y, v[2] += part[r].z, v[3] += part[r].w;
  }
};

// 4 consecutive bf16 of a row (8-byte aligned).
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float (&v)[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}
__device__ __forceinline__ void unpack4(const uint2& w, float (&v)[4]) {
  v[0] = lo_f(w.x), v[1] = hi_f(w.x), v[2] = lo_f(w.y), v[3] = hi_f(w.y);
}

template <NarrowMode kMode>
__global__ void __launch_bounds__(kNThreads, 2) narrow_kernel(const __grid_constant__ NarrowParams p) {
  constexpr bool kDual = kMode == kNarrowProduct;
  constexpr bool kAMN = kMode == kNarrowSlopes || kMode == kNarrowStoreMN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = align1024(smem_raw);
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + kNOffBar);
  uint64_t* empty = full + kNMaxStages;
  uint64_t* acc_full = empty + kNMaxStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + kNOffCtl);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + kNOffCtl + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank(), ranks = cluster_size();
  const int tile = blockIdx.x / ranks;
  const int f0 = (tile / p.token_tiles) * kNRows;  // neighbours share weights
  const int t0 = (tile % p.token_tiles) * p.columns;
  const int kb0 = (int)((int64_t)p.kb * rank / ranks), kb1 = (int)((int64_t)p.kb * (rank + 1) / ranks);
  const int kb_n = kb1 - kb0;  // >= 1: there are no more ranks than K slices
  const uint32_t stage_bytes = kWeights<kMode> + p.columns * kFfnK * 2;
  const int stages = p.stages;
  constexpr uint32_t tmem_columns = (kDual ? 2 : 1) * kNarrowColumns;

  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, tmem_columns);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0 && lane == 0) {
    auto weights = [&](int i) {
      const int st = i % stages, kb = kb0 + i;
      uint8_t* sa = sm + st * stage_bytes;
      mbar_arrive_expect_tx(full + st, stage_bytes);
      const int part = kb >= p.kb_first;
      const int k0 = (part ? kb - p.kb_first : kb) * kFfnK;
      if (kAMN) {
#pragma unroll
        for (int c = 0; c < kNRows / 64; ++c) tma_load_2d(&p.a[part], full + st, sa + c * kNChunk, f0 + c * 64, k0);
      } else if (kDual) {
        tma_load_2d(&p.a[0], full + st, sa, k0, f0);
        tma_load_2d(&p.a[1], full + st, sa + kNATile, k0, f0);
      } else {
        tma_load_2d(&p.a[0], full + st, sa, k0, f0);
      }
    };
    auto tokens = [&](int i) {
      const int st = i % stages, kb = kb0 + i;
      const int part = kb >= p.kb_first;
      const int k0 = (part ? kb - p.kb_first : kb) * kFfnK;
      tma_load_2d(&p.b[part], full + st, sm + st * stage_bytes + kWeights<kMode>, k0, t0);
    };
    // The second product of a call need not wait for the first to load its weights, only to load its tokens.
    // The first one waits for whatever was before it in the stream, which may have written anything.
    const int first = min(stages, kb_n);
    // The kernel after this one may start once this wait is over in every CTA, so what came before this call is
    // complete when it loads its weights.
    if (!p.follows) grid_dep_wait();
    for (int i = 0; i < first; ++i) weights(i);
    if (p.follows) grid_dep_wait();
    grid_dep_launch_dependents();
    for (int i = 0; i < first; ++i) tokens(i);
    int i = first;
    for (; i < kb_n; ++i) {
      if (!mbar_wait(empty + i % stages, (i / stages - 1) & 1, abort_flag, p.err, 65)) break;
      weights(i);
      tokens(i);
    }
    // never leave the CTA with a bulk copy still writing its shared memory
    for (int j = i < stages ? 0 : i - stages; j < i; ++j) drain_wait(full + j % stages, (j / stages) & 1);
  } else if (warp == 1 && lane == 0) {
    grid_dep_wait();  // the limits of this kernel's waits count its own time, not that of the kernel before
    const uint32_t idesc = idesc_bf16_f32(kNRows, p.columns, kAMN, 0);
    const SDesc a0 = sdesc_split(smem_u32(sm), kAMN ? kNChunk : 16, 1024);
    const SDesc b0 = sdesc_split(smem_u32(sm) + kWeights<kMode>, 16, 1024);
    // 16 of K further along: 32 bytes of each row K-major, 16 rows of 128 bytes MN-major
    constexpr uint32_t a_step = kAMN ? 128 : 2;
    for (int i = 0; i < kb_n; ++i) {
      const int st = i % stages;
      if (!mbar_wait(full + st, (i / stages) & 1, abort_flag, p.err, 66)) break;
      tc_fence_after();
      const uint32_t alo = a0.lo + st * (stage_bytes >> 4), blo = b0.lo + st * (stage_bytes >> 4);
#pragma unroll
      for (int kk = 0; kk < kFfnK / 16; ++kk) {
        const uint32_t more = (i > 0 || kk > 0) ? 1u : 0u;
        umma_ss2(tmem, alo + kk * a_step, a0.hi, blo + kk * 2, b0.hi, idesc, more);
        if (kDual)
          umma_ss2(tmem + p.columns, alo + (kNATile >> 4) + kk * a_step, a0.hi, blo + kk * 2, b0.hi, idesc, more);
      }
      umma_commit(empty + st);  // the stage is free once these MMAs have read it
    }
    umma_commit(acc_full);
    drain_wait(acc_full, 0);  // no MMA still running when the CTA tears down
  }
  __syncwarp();

  // the partial sums go where the stages were: acc_full comes after the last MMA's reads, and every copy has
  // landed before an MMA that read it
  const uint32_t partial = smem_u32(sm);
  const int n_tokens = min(p.columns, p.tokens - t0);
  grid_dep_wait();  // for these threads too, what was written before is visible, and their wait starts here
  const bool have = warp_wait(acc_full, 0, abort_flag, p.err, 67);
  tc_fence_after();
  // TMEM is read 16 columns at a time: pieces start at multiples of 16, so that none reads past p.columns
  const int piece = n_tokens <= kExchange<kMode> ? kExchange<kMode> : kExchange<kMode> / 16 * 16;
  for (int c0 = 0; c0 < n_tokens; c0 += piece) {
    const int n = min(piece, n_tokens - c0);
    if (have) {
      const int quadrant = warp & 3, groups = (n + 15) / 16;
      float* row = reinterpret_cast<float*>(sm) + quadrant * 32 + lane;
      const uint32_t at = tmem + (static_cast<uint32_t>(quadrant * 32) << 16) + c0;
#pragma unroll 1
      for (int i = warp >> 2; i < (kDual ? 2 : 1) * groups; i += kNThreads / 128) {
        const int part = i >= groups, c = (part ? i - groups : i) * 16;
        __syncwarp();
        uint32_t r[16];
        tmem_ld16(at + part * p.columns + c, r);
        tmem_wait_ld();
        float* to = row + (part * kExchange<kMode> + c) * kNRows;
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (c + e < kExchange<kMode>) to[e * kNRows] = __uint_as_float(r[e]);
      }
    }
    cluster_barrier();
    // the cluster's CTAs share the tokens; a thread finishes 4 features of one
    const int first = (int)(n * rank / ranks), last = (int)(n * (rank + 1) / ranks);
    const int feature = lane * 4, col = f0 + feature;
    if (*abort_flag == 0 && col < p.features) {
      for (int t = first + warp; t < last; t += kNThreads / 32) {
        const int64_t token = t0 + c0 + t;
        uint2 gate, up;
        if (kMode == kNarrowSlopes) {
          gate = *reinterpret_cast<const uint2*>(p.gate + token * p.gate_stride + col);
          up = *reinterpret_cast<const uint2*>(p.up + token * p.up_stride + col);
        }
        Parts a, b;
        a.load(partial, t, feature, ranks, rank);
        if (kDual) b.load(partial, kExchange<kMode> + t, feature, ranks, rank);
        float v[4];
        a.sum(ranks, v);
        if (kDual) {
          float u[4];
          b.sum(ranks, u);
          if (p.gate != nullptr) {
            store4(p.gate + token * p.gate_stride + col, v);
            store4(p.up + token * p.up_stride + col, u);
          }
          with_activation(p.activation, [&](auto act) {
            float unused;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = activate<decltype(act)::value, false>(v[e], unused) * u[e];
          });
        }
        if (kMode == kNarrowSlopes) {
          float g[4], u[4], dg[4], du[4];
          unpack4(gate, g);
          unpack4(up, u);
          with_activation(p.activation, [&](auto act) {
#pragma unroll
            for (int e = 0; e < 4; ++e) slopes<decltype(act)::value>(g[e], u[e], v[e], dg[e], du[e], v[e]);
          });
          store4(p.dgate + token * p.dgate_stride + col, dg);
          store4(p.dup + token * p.dup_stride + col, du);
          if (p.out == nullptr) continue;  // h is wanted for dw_down alone
        }
        store4(p.out + token * p.out_stride + col, v);
      }
    }
    // No CTA writes the next tokens' sums, or leaves, while another reads these.  To leave takes no order on what was
    // written, and without one nothing waits for the stores: 1 us a product.
    if (c0 + piece < n_tokens)
      cluster_barrier();
    else
      cluster_barrier_after_reads();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_columns);
  }
}

constexpr int kMaxDev = 64;
std::mutex g_mu;

bool g_ready[kMaxDev][4];

template <NarrowMode kMode>
cudaError_t prepare() {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDev) return cudaErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(g_mu);
  if (g_ready[dev][kMode]) return cudaSuccess;
  e = cudaFuncSetAttribute(narrow_kernel<kMode>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kNSmem);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(narrow_kernel<kMode>, cudaFuncAttributePreferredSharedMemoryCarveout,
                             cudaSharedmemCarveoutMaxShared);
  g_ready[dev][kMode] = e == cudaSuccess;
  return e;
}

template <NarrowMode kMode>
int launch(NarrowParams& p, bool follows, const char* call, cudaStream_t st) {
  cudaError_t e = prepare<kMode>();
  if (e == cudaSuccess) {
    const int64_t tiles = div_up(p.features, kNRows) * p.token_tiles;
    const int cluster = p.cluster;
    if (tiles * cluster > 0x7fffffff) return fail_ffn(LTXATTN_ERR_UNSUPPORTED, "%s: too many output tiles", call);
    p.stages = std::min<int>(kNMaxStages, kNStageSpace / (kWeights<kMode> + p.columns * kFfnK * 2));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = (unsigned)(tiles * cluster);
    cfg.blockDim = kNThreads;
    cfg.dynamicSmemBytes = kNSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    p.follows = follows;
    e = cudaLaunchKernelEx(&cfg, narrow_kernel<kMode>, p);
  }
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail_ffn(LTXATTN_ERR_CUDA, "%s: %s", call, cudaGetErrorString(e));
  }
  return LTXATTN_OK;
}

}  // namespace

// How many CTAs of clusters of that size the GPU holds at once, two to an SM: clusters stay within a GPC, and leave
// some of the 296 places empty.
constexpr int kPlaces[kNMaxCluster + 1] = {0, 296, 296, 270, 264, 260, 264, 210, 240};

// What a cut takes, in microseconds: 1.5 a product and 3 a round of CTAs; an SM brings in 1 KB of a K slice per 10
// ns, and 1 KB of another CTA's sums per 28 ns, and finishes a token's 128 features in 50 ns (30 for a gradient, next to
// nothing for a plain store), for the one or two CTAs that it holds; and all weights come in at 6.4 TB/s, which takes
// the loads of 256 CTAs in flight (19 tokens at 2048 x 8192 with 128, 192 and 256 CTAs for the first product: 32.3, 29.1
// and 28.5 us for both).  Fitted to 2700 cuts of 128 products (96 to 1024 tokens, 1024 to 16384 features): the cut that
// it finds fastest is 0.8 us slower than the fastest one measured, on average.  The time to finish a token was fitted to
// 70 calls by both kernels (47 to 720 tokens).
double cut_us(NarrowMode mode, int tokens, int features, int kb, int columns, int cluster) {
  const int parts = mode == kNarrowProduct ? 2 : 1;
  const double finish = mode == kNarrowProduct ? 0.05 : mode == kNarrowSlopes ? 0.03 : 0.0;  // of a token
  const int64_t ctas = div_up(features, kNRows) * div_up(tokens, columns) * cluster;
  const int64_t rounds = ctas / kPlaces[cluster], rest = ctas - rounds * kPlaces[cluster];
  const double cta = 0.0103 * div_up(kb, cluster) * (parts * 16 + columns / 8.0) +
                     0.0285 * columns * parts * 0.5 * (cluster - 1) / cluster +
                     (cluster > 1 && columns * parts > 208 ? 1.5 : 0.0) +  // the exchange in two pieces
                     finish * columns / cluster;
  double us = 1.5 + rounds * (3.0 + 2 * cta);
  if (rest > 0) us += 3.0 + cta * (rest > 148 ? 2.0 : 1.0 + rest / 148.0);
  const double idle = std::max(0.0, (256.0 - ctas) / 128);
  return std::max(us, 4.5 + 2e-5 * features * parts * kb * (1 + 0.28 * idle * idle));
}

// The fastest cut: token tiles as few as fit (128 columns each) or up to three more, 1 to 8 CTAs to a tile with a
// K slice each.  More token tiles exchange less but load the weights more often from L2; more CTAs to a tile keep
// more loads in flight but exchange more.
NarrowPlan plan_narrow(NarrowMode mode, int tokens, int features, int kb) {
  const int64_t least = div_up(tokens, kNarrowColumns);
  NarrowPlan best{0, 0, 0};
  for (int64_t t = least; t <= least + 3; ++t) {
    const int columns = (int)div_up(div_up(tokens, t), 16) * 16;
    for (int s = 1; s <= std::min(kNMaxCluster, kb); ++s) {
      const double us = cut_us(mode, tokens, features, kb, columns, s);
      if (best.cluster == 0 || us < best.us) best = {columns, s, us};
    }
    if (columns == 16) break;
  }
  return best;
}

int launch_narrow(NarrowMode mode, NarrowParams& p, bool follows, const char* call, cudaStream_t st) {
  p.token_tiles = (int)div_up(p.tokens, p.columns);
  p.err = device_error_word();
  if (!p.err) return fail_ffn(LTXATTN_ERR_CUDA, "no device error word");
  switch (mode) {
    case kNarrowProduct: return launch<kNarrowProduct>(p, follows, call, st);
    case kNarrowStore: return launch<kNarrowStore>(p, follows, call, st);
    case kNarrowSlopes: return launch<kNarrowSlopes>(p, follows, call, st);
    default: return launch<kNarrowStoreMN>(p, follows, call, st);
  }
}

}  // namespace ltx
