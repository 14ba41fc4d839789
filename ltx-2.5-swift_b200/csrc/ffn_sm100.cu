// ffn_sm100.cu -- ltxattn_gated_ffn and ltxattn_gated_ffn_bwd: the gated
// feed-forward block and its gradient on tcgen05 (sm_100a).
//
//   forward:   h = act(x Wg^T) * (x Wu^T)           one GEMM over [Wg; Wu], the product in its epilogue
//              y = h Wd^T
//   backward:  dh = dy Wd, and from it in the epilogue, with the kept gate g and up u,
//              dg = dh u act'(g),  du = dh act(g),  h = act(g) u
//              dx = dg Wg + du Wu                   one GEMM whose K runs through both pairs
//              dWg = dg^T x,  dWu = du^T x,  dWd = dy^T h
//
// One persistent kernel, gemm_kernel<A major, B major, epilogue>, makes them
// all.  A pair of CTAs (a cluster, cta_group::2) walks over 256 x 256 output
// tiles: each holds 128 rows of A and 128 of B's 256 columns in its shared
// memory, and 128 rows of the result in its TMEM, so an SM loads 32 KB for the
// MMAs that one on its own would load 48 KB for.  In each CTA warps 0 and 2
// load 64-wide K slices of A and B with TMA into a ring of stages (128-byte
// swizzle) that the first CTA's barriers count; there warp 1 issues the MMAs for
// both; warps 4-11 turn the finished accumulator into the output while the next
// tile's MMAs fill the other half of TMEM.
//
// Operands that lie along the wrong axis (the weights of dh and dx, both
// operands of the weight gradients) are read as they lie: their tiles are
// staged as 64-element chunks of the row/column axis and the MMA takes them
// MN-major, so nothing is transposed through memory.
//
// Sizes that fill no tile need no case of their own: TMA reads zeros outside a
// tensor (also for the rest of K), and the epilogue stores only what exists.
//
// Roundings: accumulators are fp32.  h, dg and du are rounded to bf16 once,
// because the tensor cores take them as bf16 operands of the next product; the
// outputs are rounded once.
//
// Bound: the tensor cores (at 3120 x 4096 x 16384 the forward does 2770
// operations per byte it must move).  That forward takes 851 us on a cool GPU
// (1.48 PFLOP/s, 0.89 of the measured burst rate of a library GEMM) and 976 back
// to back under the power cap (0.93 of the measured sustained rate; the two bare
// products in the library: 802 and 942).  The backward takes 1829 and 2100 us
// (library products alone: 1619 and 1898); the difference is mostly dh's epilogue,
// which moves 640 KB through shared memory a tile and keeps the tensor pipe to 65%
// of its launch, where the other products' is busy for 88%.
#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <mutex>

#include "ffn_common.cuh"

namespace ltx {

int set_error_message(int status, const char* msg);

namespace {

constexpr int kGM = 128;          // rows of a CTA's part of a tile
constexpr int kGPairM = 2 * kGM;  // rows of a tile (UMMA M)
constexpr int kGN = 256;          // accumulator columns of a tile (UMMA N)
constexpr int kGHalfN = kGN / 2;  // of which a CTA holds the operand
constexpr int kGK = kFfnK;
constexpr int kGThreads = 384;    // 4 control warps, 8 epilogue warps
constexpr uint32_t kGA = kGM * kGK * 2;
constexpr uint32_t kGB = kGHalfN * kGK * 2;
constexpr uint32_t kGStage = kGA + kGB;
constexpr uint32_t kChunk = 64 * kGK * 2;  // MN-major: 64 columns x 64 rows of K
constexpr int kGEpilogueWarps = 8;

enum Epilogue { kProduct, kStore, kSlopes };

// The epilogue's warps pass their 32 rows through shared memory, 32 columns in bf16 at a time or 64, and TMA carries those
// pieces out (and the kept gate and up in): a thread finds a row in TMEM, and accesses of one row per thread take a
// line of memory each.  A piece is 32 rows of 64 bytes in the 64-byte swizzle, which lets eight rows' threads touch all
// banks; plain stores, which need no room for anything else, take 64 columns.
constexpr uint32_t kPiece = 32 * 64;

template <int kEpilogue>
struct GemmShape {
  // Pieces per warp.  Products go out through two in turn.  The gradient's epilogue has two of gate and up in turn, in
  // which dgate and dup take their place, and one of h.
  static constexpr int kPieces = kEpilogue == kSlopes ? 5 : 2;
  static constexpr uint32_t kPieceBytes = kEpilogue == kStore ? 2 * kPiece : kPiece;  // plain stores: 64 columns
  static constexpr int kStages = kEpilogue == kSlopes ? 4 : 5;
  static constexpr uint32_t kOffPieces = kStages * kGStage;
  // full[kStages] (the first CTA's counts for both), empty[kStages], acc_full[2], acc_empty[2] (the first CTA's), and
  // two for the gate and up of each warp
  static constexpr uint32_t kOffBar = kOffPieces + kGEpilogueWarps * kPieces * kPieceBytes;
  static constexpr uint32_t kOffCtl = kOffBar + (2 * kStages + 4 + 2 * kGEpilogueWarps) * 8;  // TMEM slot, abort flag
  static constexpr uint32_t kBytes = kOffCtl + 16 + 1024;                                     // + alignment slack
  static_assert(kBytes <= kMaxDynamicSmem, "shared memory of a CTA");
};

// One output of a launch (a launch of the weight gradients has up to three).
struct Gemm {
  CUtensorMap a[2], b[2];  // K slices beyond kb_first come from the second pair
  CUtensorMap out;         // in pieces of 32 x 32, plain stores of 32 x 64
  int M, N;                // rows and accumulator columns that exist (kProduct: columns of h)
  int kb, kb_first;        // 64-wide K slices in all, and those of the first pair
  int tiles_m, tiles_n;
};

struct GemmParams {
  Gemm g[3];
  int first_tile[4];  // tiles of g[i]: [first_tile[i], first_tile[i + 1])
  int count;
  int activation;
  // kProduct: gate and up to be kept (where `keep`).  kSlopes: the kept ones, and dgate and dup; h goes to out where
  // `keep`
  CUtensorMap gate, up, dgate, dup;
  int keep;
  int* err;
};

// ---------------------------------------------------------------------------

// Tiles are numbered down the rows first, in bands of kBand row blocks: the CTAs
// that run together then share a few column blocks of B and the band's rows of A.  4096 rows: of 3120 tokens the
// weights are then read once (bands of 1024, 2048 and 4096 rows: 1026, 993 and 979 us for the forward at 4096 x 16384,
// under the power cap).
constexpr int kBand = 16;

__device__ __forceinline__ void locate(const GemmParams& p, int tile, int& which, int& m0, int& tn) {
  which = 0;
  while (which + 1 < p.count && tile >= p.first_tile[which + 1]) ++which;
  const Gemm& g = p.g[which];
  const int i = tile - p.first_tile[which];
  const int band = i / (kBand * g.tiles_n);
  const int rows = min(kBand, g.tiles_m - band * kBand);
  const int j = i - band * kBand * g.tiles_n;
  m0 = (band * kBand + j % rows) * kGPairM;
  tn = j / rows;
}

// TMEM and MMAs of a CTA pair.  Both CTAs allocate and free; the first one issues.
__device__ __forceinline__ void pair_tmem_alloc(uint32_t* slot, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void pair_tmem_free(uint32_t tmem, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}
// Issued by the whole warp with the same operands, one elected lane doing it: they then stay in uniform registers, and
// the issue keeps up beside the epilogue warps that share the scheduler.
__device__ __forceinline__ void pair_mma(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                         uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\t"
      "setp.ne.b32 p, %6, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %5, p;\n\t}\n" ::"r"(d),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives at `bar` of both CTAs once every MMA issued so far is done (the whole warp; the same lane is elected).
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}\n" ::"r"(
          smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
// A load into this CTA's shared memory that is counted at a barrier of either CTA (its shared::cluster address).
__device__ __forceinline__ void pair_load(const CUtensorMap* map, uint32_t bar, void* dst, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void cluster_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void piece_store(const CUtensorMap* map, uint32_t piece, int col, int row) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(piece), "r"(col), "r"(row)
               : "memory");
}
// Waits until at most kPending of this thread's groups of stores still read their pieces.
template <int kPending>
__device__ __forceinline__ void piece_wait() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kPending) : "memory");
}
// 8 columns (16 bytes) of a row in a piece.
__device__ __forceinline__ uint4* in_piece(uint8_t* piece, int row, int q) {
  return reinterpret_cast<uint4*>(piece + row * 64 + ((q ^ ((row >> 1) & 3)) << 4));
}

// The two pieces that a warp's products go out through, in turn: 32 rows (one per lane) x 32 columns, or 64 in the
// 128-byte swizzle (all gradients of 1024 tokens at 4096 x 11008: 440 us in pieces of 32 columns, 424 in 64).  What is
// outside the tensor is left out.
template <int kCols>
struct Outgoing {
  uint8_t* pieces;
  int lane;
  uint8_t* piece = nullptr;
  int next = 0;

  __device__ __forceinline__ void start() {
    piece = pieces + next * (32 * kCols * 2);
    next ^= 1;
    if (lane == 0) piece_wait<1>();  // the one before the last has been read
    __syncwarp();
  }
  // 32 columns from `at` on
  __device__ __forceinline__ void put(const float (&v)[32], int at = 0) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint4* to = kCols == 32 ? in_piece(piece, lane, q)
                              : reinterpret_cast<uint4*>(piece + lane * 128 + (((at / 8 + q) ^ (lane & 7)) << 4));
      *to = pack8(v, 8 * q);
    }
  }
  __device__ __forceinline__ void send(const CUtensorMap* map, int col, int row) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      piece_store(map, smem_u32(piece), col, row);
      bulk_commit();
    }
  }
  __device__ __forceinline__ void send(const CUtensorMap* map, const float (&v)[32], int col, int row) {
    start();
    put(v);
    send(map, col, row);
  }
};

template <bool kAMN, bool kBMN, int kEpilogue>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGThreads, 1)
    gemm_kernel(const __grid_constant__ GemmParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = align1024(smem_raw);
  using S = GemmShape<kEpilogue>;
  constexpr int kGStages = S::kStages;
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + S::kOffBar);
  uint64_t* empty = full + kGStages;
  uint64_t* acc_full = empty + kGStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* kept_full = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + S::kOffCtl);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + S::kOffCtl + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank();
  const int tiles = p.first_tile[p.count];
  const int first = blockIdx.x / 2, step = gridDim.x / 2;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * kGStages; ++i) mbar_init(full + i, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full + i, 1);
      mbar_init(acc_empty + i, 2 * kGEpilogueWarps);
    }
    for (int i = 0; i < 2 * kGEpilogueWarps; ++i) mbar_init(kept_full + i, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncwarp();
  if (warp == 1) {
    pair_tmem_alloc(tmem_slot, 512);
    tc_fence_before();
  }
  __syncthreads();
  cluster_barrier();  // both CTAs' barriers are set up
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dep_wait();  // all that is read may have been written by the kernel before
  grid_dep_launch_dependents();

  // warp 0 loads A, warp 2 B: one thread takes about as long to issue both loads' copies as the MMAs of a stage run
  if ((warp == 0 || warp == 2) && lane == 0) {
    int it = 0;
    bool ok = true;
    for (int tile = first; tile < tiles && ok; tile += step) {
      int which, m0, tn;
      locate(p, tile, which, m0, tn);
      m0 += rank * kGM;
      const Gemm& g = p.g[which];
      for (int kb = 0; kb < g.kb; ++kb, ++it) {
        const int st = it % kGStages, u = it / kGStages;
        if (it >= kGStages && !mbar_wait(empty + st, (u - 1) & 1, abort_flag, p.err, 61)) {
          ok = false;
          break;
        }
        uint8_t* sa = sm + st * kGStage;
        uint8_t* sb = sa + kGA;
        const int part = kb >= g.kb_first;
        const int k0 = (part ? kb - g.kb_first : kb) * kGK;
        const uint32_t bar = peer_address(smem_u32(full + st), 0);
        if (warp == 0) {
          if (rank == 0) mbar_arrive_expect_tx(full + st, 2 * kGStage);
          if (kAMN) {
#pragma unroll
            for (int c = 0; c < kGM / 64; ++c) pair_load(&g.a[part], bar, sa + c * kChunk, m0 + c * 64, k0);
          } else {
            pair_load(&g.a[part], bar, sa, k0, m0);
          }
        } else if (kEpilogue == kProduct) {
          // the first CTA's half of B is the gate's weights, the second's the up projection's
          pair_load(&g.b[rank], bar, sb, k0, tn * kGHalfN);
        } else if (kBMN) {
#pragma unroll
          for (int c = 0; c < kGHalfN / 64; ++c)
            pair_load(&g.b[part], bar, sb + c * kChunk, tn * kGN + rank * kGHalfN + c * 64, k0);
        } else {
          pair_load(&g.b[part], bar, sb, k0, tn * kGN + rank * kGHalfN);
        }
      }
    }
    // never leave the CTA with a bulk copy still writing its shared memory: a stage is empty again once it was
    // full and has been read
    for (int i = it < kGStages ? 0 : it - kGStages; i < it; ++i) drain_wait(empty + i % kGStages, (i / kGStages) & 1);
  } else if (warp == 1 && rank == 0) {
    constexpr uint32_t idesc = idesc_bf16_f32(kGPairM, kGN, kAMN, kBMN);
    const SDesc a0 = sdesc_split(smem_u32(sm), kAMN ? kChunk : 16, 1024);
    const SDesc b0 = sdesc_split(smem_u32(sm) + kGA, kBMN ? kChunk : 16, 1024);
    // 16 of K further along: 32 bytes of each row K-major, 16 rows of 128 bytes MN-major
    constexpr uint32_t a_step = kAMN ? 128 : 2, b_step = kBMN ? 128 : 2;
    int it = 0, n = 0;
    bool ok = true;
    for (int tile = first; tile < tiles && ok; tile += step, ++n) {
      int which, m0, tn;
      locate(p, tile, which, m0, tn);
      const int kb_n = p.g[which].kb;
      const int buf = n & 1;
      if (n >= 2 && !warp_wait(acc_empty + buf, ((n >> 1) - 1) & 1, abort_flag, p.err, 62)) break;
      tc_fence_after();
      const uint32_t d = tmem + buf * kGN;
      for (int kb = 0; kb < kb_n; ++kb, ++it) {
        const int st = it % kGStages, u = it / kGStages;
        if (!warp_wait(full + st, u & 1, abort_flag, p.err, 63)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t alo = a0.lo + st * (kGStage >> 4), blo = b0.lo + st * (kGStage >> 4);
#pragma unroll
        for (int kk = 0; kk < kGK / 16; ++kk)
          pair_mma(d, alo + kk * a_step, a0.hi, blo + kk * b_step, b0.hi, idesc, (kb > 0 || kk > 0) ? 1u : 0u);
        pair_commit(empty + st);  // the stage is free, in both CTAs, once these MMAs have read it
      }
      pair_commit(acc_full + buf);
    }
    // no MMA still running when the CTA tears down: the last commits cover all of them
    for (int i = n < 2 ? 0 : n - 2; i < n; ++i) drain_wait(acc_full + (i & 1), (i >> 1) & 1);
  } else if (warp >= 4) {
    const int quadrant = warp & 3, half = (warp - 4) >> 2;
    const uint32_t lane_off = static_cast<uint32_t>(quadrant * 32) << 16;
    uint8_t* pieces = sm + S::kOffPieces + (warp - 4) * S::kPieces * S::kPieceBytes;
    Outgoing<S::kPieceBytes / 64> outgoing{pieces, lane};
    uint64_t* kept = kept_full + 2 * (warp - 4);
    int n = 0, turn = 0;  // turn: uses of the gate and up pieces
    for (int tile = first; tile < tiles; tile += step, ++n) {
      int which, m0, tn;
      locate(p, tile, which, m0, tn);
      const Gemm& g = p.g[which];
      const int buf = n & 1;
      const int row0 = m0 + rank * kGM + quadrant * 32;
      // kSlopes: the columns of gate and up for this warp's next turn, on their way
      auto fetch = [&](int c, int t) {
        const int col = tn * kGN + half * 128 + c;
        if (lane == 0 && c < 128 && col < g.N && row0 < g.M) {
          mbar_arrive_expect_tx(kept + (t & 1), 2 * kPiece);
          tma_load_2d(&p.gate, kept + (t & 1), pieces + (t & 1) * 2 * kPiece, col, row0);
          tma_load_2d(&p.up, kept + (t & 1), pieces + (t & 1) * 2 * kPiece + kPiece, col, row0);
        }
      };
      if (kEpilogue == kSlopes) {
        if (lane == 0) piece_wait<0>();
        fetch(0, turn);
      }
      if (!warp_wait(acc_full + buf, (n >> 1) & 1, abort_flag, p.err, 64)) {
        // never leave the CTA with a copy still writing its shared memory
        if (kEpilogue == kSlopes && lane == 0 && row0 < g.M && tn * kGN + half * 128 < g.N)
          drain_wait(kept + (turn & 1), (turn >> 1) & 1);
        break;
      }
      tc_fence_after();
      const uint32_t d = tmem + buf * kGN + lane_off;
      // The accumulator is free for the tile after the next once this warp has its last columns in registers.
      bool released = false;
      auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) cluster_arrive(peer_address(smem_u32(acc_empty + buf), 0));
        released = true;
      };
      if (row0 >= g.M) {
        // nothing of this warp's exists
      } else if (kEpilogue == kProduct) {
        // 64 columns of h per warp: accumulator columns c (gate) and 128 + c (up)
#pragma unroll 1
        for (int c = half * 64; c < half * 64 + 64; c += 32) {
          const int col = tn * kGHalfN + c;
          if (col >= g.N) break;  // warp-uniform
          __syncwarp();
          uint32_t rg[32], ru[32];
          tmem_ld32(d + c, rg);
          tmem_ld32(d + kGHalfN + c, ru);
          tmem_wait_ld();
          if (c + 32 == half * 64 + 64) release();
          float v[32];
          if (p.keep) {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(rg[e]);
            outgoing.send(&p.gate, v, col, row0);
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(ru[e]);
            outgoing.send(&p.up, v, col, row0);
          }
          with_activation(p.activation, [&](auto act) {
            float unused;
#pragma unroll
            for (int e = 0; e < 32; ++e)
              v[e] = activate<decltype(act)::value, false>(__uint_as_float(rg[e]), unused) * __uint_as_float(ru[e]);
          });
          outgoing.send(&g.out, v, col, row0);
        }
      } else if (kEpilogue == kStore) {
#pragma unroll 1
        for (int c = half * 128; c < half * 128 + 128; c += 64) {
          const int col = tn * kGN + c;
          if (col >= g.N) break;  // warp-uniform
          __syncwarp();
          uint32_t r[2][32];
          tmem_ld32(d + c, r[0]);
          tmem_ld32(d + c + 32, r[1]);
          tmem_wait_ld();
          if (c + 64 == half * 128 + 128) release();
          outgoing.start();
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float v[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(r[i][e]);
            outgoing.put(v, 32 * i);
          }
          outgoing.send(&g.out, col, row0);
        }
      } else {
#pragma unroll 1
        for (int c = 0; c < 128; c += 32, ++turn) {
          const int col = tn * kGN + half * 128 + c;
          if (col >= g.N) break;  // warp-uniform
          if (lane == 0) piece_wait<0>();  // the turn before has been read, its pieces are free
          fetch(c + 32, turn + 1);
          __syncwarp();
          uint32_t r[32];
          tmem_ld32(d + half * 128 + c, r);
          const bool here = warp_wait(kept + (turn & 1), (turn >> 1) & 1, abort_flag, p.err, 68);
          tmem_wait_ld();
          if (c + 32 == 128) release();
          if (!here) {
            // another wait gave up, or this one: never leave the CTA with a copy still writing its shared memory
            // (the next turn's is waited for in the next turn)
            if (lane == 0) drain_wait(kept + (turn & 1), (turn >> 1) & 1);
            continue;
          }
          uint8_t* gp = pieces + (turn & 1) * 2 * kPiece;
          uint8_t* hp = pieces + 4 * kPiece;
          with_activation(p.activation, [&](auto act) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint4 *gq = in_piece(gp, lane, q), *uq = in_piece(gp + kPiece, lane, q);
              float gv[8], uv[8], dgv[8], duv[8], hv[8];
              unpack8(*gq, gv);
              unpack8(*uq, uv);
#pragma unroll
              for (int e = 0; e < 8; ++e)
                slopes<decltype(act)::value>(gv[e], uv[e], __uint_as_float(r[8 * q + e]), dgv[e], duv[e], hv[e]);
              *gq = pack8(dgv);
              *uq = pack8(duv);
              *in_piece(hp, lane, q) = pack8(hv);
            }
          });
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            piece_store(&p.dgate, smem_u32(gp), col, row0);
            piece_store(&p.dup, smem_u32(gp + kPiece), col, row0);
            if (p.keep) piece_store(&g.out, smem_u32(hp), col, row0);
            bulk_commit();
          }
        }
      }
      if (!released) release();
    }
    if (lane == 0) piece_wait<0>();  // the CTA's shared memory must outlive the copies' reads
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_barrier();  // neither CTA leaves while the other's MMAs or arrivals reach it
  if (warp == 1) {
    tc_fence_after();
    pair_tmem_free(tmem, 512);
  }
}

// ---------------------------------------------------------------------------
// host side

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encoder() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(f);
    else
      (void)cudaGetLastError();
  });
  return fn;
}

}  // namespace

int fail_ffn(int status, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return set_error_message(status, buf);
}

int ffn_map(CUtensorMap* m, const void* ptr, int64_t rows, int64_t cols, int64_t stride, int box_rows,
            const char* name, int box_cols) {
  EncodeTiledFn enc = encoder();
  if (!enc) return fail_ffn(LTXATTN_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)stride * 2};
  cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE,
                         box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail_ffn(LTXATTN_ERR_ALIGN, "%s: cuTensorMapEncodeTiled rejected the view (CUresult %d)", name, (int)r);
  return LTXATTN_OK;
}

namespace {

// The pieces that an epilogue's warp stores and loads: boxes of 32 x 32, or of 32 x 64 for plain stores.
int piece_map(CUtensorMap* m, const void* ptr, int64_t rows, int64_t cols, int64_t stride, const char* name,
              int box_cols = 32) {
  return ffn_map(m, ptr, rows, cols, stride, 32, name, box_cols);
}

// A bf16 matrix argument.
struct Mat {
  const char* name;
  const void* data;
  int64_t stride;
  int64_t rows, cols;
};

int check_mat(const char* call, const Mat& m) {
  if (m.data == nullptr) return fail_ffn(LTXATTN_ERR_ARG, "%s: %s is required", call, m.name);
  if (m.stride < m.cols)
    return fail_ffn(LTXATTN_ERR_SHAPE, "%s: %s's row stride (%lld) is shorter than its row (%lld)", call, m.name,
                    (long long)m.stride, (long long)m.cols);
  if ((reinterpret_cast<uintptr_t>(m.data) & 15u) || m.stride % 8)
    return fail_ffn(LTXATTN_ERR_ALIGN, "%s: %s needs 16-byte aligned rows", call, m.name);
  if (m.stride > (int64_t(1) << 38))
    return fail_ffn(LTXATTN_ERR_UNSUPPORTED, "%s: %s's row stride is too large", call, m.name);
  return LTXATTN_OK;
}

// Refuses an output (from `first` on) that is another of the call's matrices.
int check_distinct(const char* call, const Mat* mats, int count, int first) {
  for (int i = first; i < count; ++i)
    for (int j = 0; j < i; ++j)
      if (mats[i].data != nullptr && mats[i].data == mats[j].data)
        return fail_ffn(LTXATTN_ERR_ARG, "%s: %s and %s are the same memory", call, mats[j].name, mats[i].name);
  return LTXATTN_OK;
}

// An epilogue waits for the whole sum of its tile, and a wait gives up after 2 s.  64 products of K take 0.33 us on every
// row and column of a tile: with K up to 2^27 (dx: twice inner) that is 0.7 s.
constexpr int kMaxWidth = 1 << 26;
constexpr int kMaxSummedTokens = 1 << 27;

int check_sizes(const char* call, int dtype, int activation, int m, int hidden, int inner, int out_dim) {
  if (dtype != LTXATTN_BF16) return fail_ffn(LTXATTN_ERR_DTYPE, "%s: bf16 only", call);
  if (activation < LTXATTN_SILU || activation > LTXATTN_GELU)
    return fail_ffn(LTXATTN_ERR_ARG, "%s: unknown activation %d", call, activation);
  if (m < 0 || hidden < 1 || inner < 1 || out_dim < 1)
    return fail_ffn(LTXATTN_ERR_SHAPE, "%s: m must be >= 0, hidden, inner and out_dim >= 1", call);
  if (hidden % 8 || inner % 8 || out_dim % 8)
    return fail_ffn(LTXATTN_ERR_UNSUPPORTED, "%s: hidden (%d), inner (%d) and out_dim (%d) must be multiples of 8", call,
                    hidden, inner, out_dim);
  if (std::max({hidden, inner, out_dim}) > kMaxWidth)
    return fail_ffn(LTXATTN_ERR_UNSUPPORTED, "%s: hidden (%d), inner (%d) or out_dim (%d) is above %d", call, hidden, inner,
                    out_dim, kMaxWidth);
  return LTXATTN_OK;
}

constexpr int kMaxDev = 64;
std::mutex g_mu;
bool g_attr_set[kMaxDev][8] = {};
int g_sms[kMaxDev] = {};

// The SM count, with the kernel's shared memory opted into once per device.
template <typename K>
cudaError_t prepare_kernel(K kernel, int slot, uint32_t smem, int* sms) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDev) return cudaErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(g_mu);
  if (!g_attr_set[dev][slot]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&g_sms[dev], cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    g_attr_set[dev][slot] = true;
  }
  *sms = g_sms[dev];
  return cudaSuccess;
}

template <bool kAMN, bool kBMN, int kEpilogue>
int launch_gemm(GemmParams& p, int slot, const char* call, cudaStream_t st) {
  const int width = kEpilogue == kProduct ? kGHalfN : kGN;
  int64_t tiles = 0;
  for (int i = 0; i < p.count; ++i) {
    Gemm& g = p.g[i];
    g.tiles_m = (int)div_up(g.M, kGPairM);
    g.tiles_n = (int)div_up(g.N, width);
    p.first_tile[i] = (int)tiles;
    tiles += (int64_t)g.tiles_m * g.tiles_n;
    if (tiles > 0x3fffffff) return fail_ffn(LTXATTN_ERR_UNSUPPORTED, "%s: too many output tiles", call);
  }
  p.first_tile[p.count] = (int)tiles;
  p.err = device_error_word();
  if (!p.err) return fail_ffn(LTXATTN_ERR_CUDA, "no device error word");
  int sms = 0;
  constexpr uint32_t smem = GemmShape<kEpilogue>::kBytes;
  cudaError_t e = prepare_kernel(gemm_kernel<kAMN, kBMN, kEpilogue>, slot, smem, &sms);
  if (e == cudaSuccess)
    e = launch_pdl(gemm_kernel<kAMN, kBMN, kEpilogue>, 2 * (unsigned)std::min<int64_t>(tiles, sms / 2), kGThreads, smem,
                   st, p);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail_ffn(LTXATTN_ERR_CUDA, "%s: %s", call, cudaGetErrorString(e));
  }
  return LTXATTN_OK;
}

// Whether a product runs feature by feature (ffn_narrow_sm100.cu), by what both kernels were measured to take.  The
// wide kernel pays for rounds of tiles over 74 CTA pairs (148 SMs), which few tokens leave mostly empty, and for the gradient's
// epilogue of the last round.  Over 120 calls (64 to 2000 tokens, 1024 to 16384 features, both directions) the choice was
// as fast as the best of both kernels for each product, to 0.3% on average; choosing by 128, 256 and 512 tokens alone
// was 23%, 12% and 8% slower.
bool few_tokens(int tokens, int features, int kb, NarrowMode mode, NarrowParams& p) {
  const NarrowPlan plan = plan_narrow(mode, tokens, features, kb);
  const int64_t tiles = div_up(tokens, kGPairM) * div_up(features, mode == kNarrowProduct ? kGHalfN : kGN);
  const double wide_us = (mode == kNarrowProduct ? 4.0 : mode == kNarrowSlopes ? 10.0 : 6.0) + (double)div_up(tiles, 74) * (0.33 * kb + 1.5);
  p.tokens = tokens;
  p.features = features;
  p.kb = p.kb_first = kb;
  p.columns = plan.columns;
  p.cluster = plan.cluster;
  return plan.us < wide_us;
}

size_t round256(size_t n) { return (n + 255) & ~size_t(255); }

// h, dgate and dup between the kernels: [m, inner] bf16 with contiguous rows.
size_t plane_bytes(int m, int inner) { return round256((size_t)m * inner * 2); }

int check_workspace(const char* call, const void* ws, size_t have, size_t need) {
  if (ws == nullptr || have < need)
    return fail_ffn(LTXATTN_ERR_WORKSPACE, "%s: the workspace has %zu bytes, %zu are needed", call, ws ? have : 0, need);
  if (reinterpret_cast<uintptr_t>(ws) & 255u)
    return fail_ffn(LTXATTN_ERR_ALIGN, "%s: the workspace must be 256-byte aligned", call);
  return LTXATTN_OK;
}

}  // namespace
}  // namespace ltx

using namespace ltx;

extern "C" {

size_t ltxattn_gated_ffn_workspace(const ltxattn_gated_ffn_args* a) {
  if (a == nullptr || a->m < 1 || a->inner < 1) return 0;
  return plane_bytes(a->m, a->inner);
}

int ltxattn_gated_ffn(const ltxattn_gated_ffn_args* a, void* stream) {
  const char* call = "ltxattn_gated_ffn";
  if (a == nullptr) return fail_ffn(LTXATTN_ERR_ARG, "args is NULL");
  if (int rc = check_sizes(call, a->dtype, a->activation, a->m, a->hidden, a->inner, a->out_dim)) return rc;
  if ((a->gate == nullptr) != (a->up == nullptr) && a->m > 0)
    return fail_ffn(LTXATTN_ERR_ARG, "%s: gate and up are kept together or not at all", call);
  if (a->m == 0) return LTXATTN_OK;
  const Mat mats[7] = {{"x", a->x, a->x_stride, a->m, a->hidden},
                       {"w_gate", a->w_gate, a->w_gate_stride, a->inner, a->hidden},
                       {"w_up", a->w_up, a->w_up_stride, a->inner, a->hidden},
                       {"w_down", a->w_down, a->w_down_stride, a->out_dim, a->inner},
                       {"out", a->out, a->out_stride, a->m, a->out_dim},
                       {"gate", a->gate, a->gate_stride, a->m, a->inner},
                       {"up", a->up, a->up_stride, a->m, a->inner}};
  for (int i = 0; i < (a->gate ? 7 : 5); ++i)
    if (int rc = check_mat(call, mats[i])) return rc;
  if (int rc = check_distinct(call, mats, 7, 4)) return rc;
  if (int rc = check_workspace(call, a->workspace, a->workspace_bytes, ltxattn_gated_ffn_workspace(a))) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  __nv_bfloat16* h = static_cast<__nv_bfloat16*>(a->workspace);

  const int kb_in = (int)div_up(a->hidden, kFfnK), kb_out = (int)div_up(a->inner, kFfnK);
  if (NarrowParams q{}; few_tokens(a->m, a->inner, kb_in, kNarrowProduct, q)) {
    q.activation = a->activation;
    q.out = h;
    q.out_stride = a->inner;
    q.gate = static_cast<__nv_bfloat16*>(a->gate);
    q.up = static_cast<__nv_bfloat16*>(a->up);
    q.gate_stride = a->gate_stride;
    q.up_stride = a->up_stride;
    const int box = narrow_box(kNarrowProduct);
    if (int rc = ffn_map(&q.a[0], a->w_gate, a->inner, a->hidden, a->w_gate_stride, box, "w_gate")) return rc;
    if (int rc = ffn_map(&q.a[1], a->w_up, a->inner, a->hidden, a->w_up_stride, box, "w_up")) return rc;
    if (int rc = ffn_map(&q.b[0], a->x, a->m, a->hidden, a->x_stride, q.columns, "x")) return rc;
    if (int rc = launch_narrow(kNarrowProduct, q, false, call, st)) return rc;
  } else {
    GemmParams p{};
    p.count = 1;
    p.activation = a->activation;
    Gemm& g = p.g[0];
    if (int rc = ffn_map(&g.a[0], a->x, a->m, a->hidden, a->x_stride, kGM, "x")) return rc;
    if (int rc = ffn_map(&g.b[0], a->w_gate, a->inner, a->hidden, a->w_gate_stride, kGHalfN, "w_gate")) return rc;
    if (int rc = ffn_map(&g.b[1], a->w_up, a->inner, a->hidden, a->w_up_stride, kGHalfN, "w_up")) return rc;
    g.M = a->m;
    g.N = a->inner;
    g.kb = g.kb_first = kb_in;
    if (int rc = piece_map(&g.out, h, a->m, a->inner, a->inner, "workspace")) return rc;
    p.keep = a->gate != nullptr;
    if (p.keep) {
      if (int rc = piece_map(&p.gate, a->gate, a->m, a->inner, a->gate_stride, "gate")) return rc;
      if (int rc = piece_map(&p.up, a->up, a->m, a->inner, a->up_stride, "up")) return rc;
    }
    if (int rc = launch_gemm<false, false, kProduct>(p, 0, call, st)) return rc;
  }
  if (NarrowParams q{}; few_tokens(a->m, a->out_dim, kb_out, kNarrowStore, q)) {
    q.out = static_cast<__nv_bfloat16*>(a->out);
    q.out_stride = a->out_stride;
    if (int rc = ffn_map(&q.a[0], a->w_down, a->out_dim, a->inner, a->w_down_stride, narrow_box(kNarrowStore), "w_down"))
      return rc;
    if (int rc = ffn_map(&q.b[0], h, a->m, a->inner, a->inner, q.columns, "workspace")) return rc;
    return launch_narrow(kNarrowStore, q, true, call, st);
  }
  GemmParams p{};
  p.count = 1;
  Gemm& g = p.g[0];
  if (int rc = ffn_map(&g.a[0], h, a->m, a->inner, a->inner, kGM, "workspace")) return rc;
  if (int rc = ffn_map(&g.b[0], a->w_down, a->out_dim, a->inner, a->w_down_stride, kGHalfN, "w_down")) return rc;
  g.M = a->m;
  g.N = a->out_dim;
  g.kb = g.kb_first = kb_out;
  if (int rc = piece_map(&g.out, a->out, a->m, a->out_dim, a->out_stride, "out", 64)) return rc;
  return launch_gemm<false, false, kStore>(p, 1, call, st);
}

int ltxattn_gated_ffn_plan(int32_t m, int32_t hidden, int32_t inner, int32_t out_dim, ltxattn_gated_ffn_plan_info* info) {
  const char* call = "ltxattn_gated_ffn_plan";
  if (info == nullptr) return fail_ffn(LTXATTN_ERR_ARG, "%s: info is NULL", call);
  if (int rc = check_sizes(call, LTXATTN_BF16, LTXATTN_SILU, m, hidden, inner, out_dim)) return rc;
  *info = {};
  if (m == 0) return LTXATTN_OK;
  auto product = [&](NarrowMode mode, int features, int64_t k, ltxattn_gated_ffn_product* to) {
    NarrowParams q{};
    if (few_tokens(m, features, (int)k, mode, q))
      *to = {2, q.columns, q.cluster};
    else
      *to = {1, 0, 0};
  };
  product(kNarrowProduct, inner, div_up(hidden, kFfnK), &info->inner);
  product(kNarrowStore, out_dim, div_up(inner, kFfnK), &info->out);
  product(kNarrowSlopes, inner, div_up(out_dim, kFfnK), &info->dinner);
  product(kNarrowStoreMN, hidden, 2 * div_up(inner, kFfnK), &info->dx);
  return LTXATTN_OK;
}

size_t ltxattn_gated_ffn_bwd_workspace(const ltxattn_gated_ffn_bwd_args* a) {
  if (a == nullptr || a->m < 1 || a->inner < 1) return 0;
  return 3 * plane_bytes(a->m, a->inner);
}

int ltxattn_gated_ffn_bwd(const ltxattn_gated_ffn_bwd_args* a, void* stream) {
  const char* call = "ltxattn_gated_ffn_bwd";
  if (a == nullptr) return fail_ffn(LTXATTN_ERR_ARG, "args is NULL");
  if (int rc = check_sizes(call, a->dtype, a->activation, a->m, a->hidden, a->inner, a->out_dim)) return rc;
  const bool dw_in = a->dw_gate != nullptr || a->dw_up != nullptr;
  const Mat outs[4] = {{"dx", a->dx, a->dx_stride, a->m, a->hidden},
                       {"dw_gate", a->dw_gate, a->dw_gate_stride, a->inner, a->hidden},
                       {"dw_up", a->dw_up, a->dw_up_stride, a->inner, a->hidden},
                       {"dw_down", a->dw_down, a->dw_down_stride, a->out_dim, a->inner}};
  bool any = false;
  for (int i = 0; i < 4; ++i) {
    if (outs[i].data == nullptr || (i == 0 && a->m == 0)) continue;
    any = true;
    if (int rc = check_mat(call, outs[i])) return rc;
  }
  if (!any) return LTXATTN_OK;
  if ((dw_in || a->dw_down != nullptr) && a->m > kMaxSummedTokens)
    return fail_ffn(LTXATTN_ERR_UNSUPPORTED, "%s: the weights' gradients of more than %d tokens", call, kMaxSummedTokens);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->m == 0) {  // no tokens: the weights' gradients are sums of nothing
    for (int i = 1; i < 4; ++i) {
      if (outs[i].data == nullptr) continue;
      const cudaError_t e = cudaMemset2DAsync(const_cast<void*>(outs[i].data), (size_t)outs[i].stride * 2, 0,
                                              (size_t)outs[i].cols * 2, (size_t)outs[i].rows, st);
      if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return fail_ffn(LTXATTN_ERR_CUDA, "%s: %s", call, cudaGetErrorString(e));
      }
    }
    return LTXATTN_OK;
  }
  const Mat ins[7] = {{"gate", a->gate, a->gate_stride, a->m, a->inner},
                      {"up", a->up, a->up_stride, a->m, a->inner},
                      {"dout", a->dout, a->dout_stride, a->m, a->out_dim},
                      {"w_down", a->w_down, a->w_down_stride, a->out_dim, a->inner},
                      {"w_gate", a->w_gate, a->w_gate_stride, a->inner, a->hidden},
                      {"w_up", a->w_up, a->w_up_stride, a->inner, a->hidden},
                      {"x", a->x, a->x_stride, a->m, a->hidden}};
  for (int i = 0; i < 7; ++i) {
    if ((i == 4 || i == 5) && a->dx == nullptr) continue;
    if (i == 6 && !dw_in) continue;
    if (int rc = check_mat(call, ins[i])) return rc;
  }
  Mat all[11];
  std::copy(ins, ins + 7, all);
  std::copy(outs, outs + 4, all + 7);
  if (int rc = check_distinct(call, all, 11, 7)) return rc;
  if (int rc = check_workspace(call, a->workspace, a->workspace_bytes, ltxattn_gated_ffn_bwd_workspace(a))) return rc;
  const size_t plane = plane_bytes(a->m, a->inner);
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  __nv_bfloat16* dgate = reinterpret_cast<__nv_bfloat16*>(ws);
  __nv_bfloat16* dup = reinterpret_cast<__nv_bfloat16*>(ws + plane);
  __nv_bfloat16* h = reinterpret_cast<__nv_bfloat16*>(ws + 2 * plane);

  __nv_bfloat16* gate = static_cast<__nv_bfloat16*>(const_cast<void*>(a->gate));
  __nv_bfloat16* up = static_cast<__nv_bfloat16*>(const_cast<void*>(a->up));
  const int kb_dh = (int)div_up(a->out_dim, kFfnK), kb_inner = (int)div_up(a->inner, kFfnK);
  // dh = dout w_down, and what follows from it element by element
  if (NarrowParams q{}; few_tokens(a->m, a->inner, kb_dh, kNarrowSlopes, q)) {
    q.activation = a->activation;
    q.out = a->dw_down != nullptr ? h : nullptr;
    q.out_stride = q.dgate_stride = q.dup_stride = a->inner;
    q.gate = gate;
    q.up = up;
    q.gate_stride = a->gate_stride;
    q.up_stride = a->up_stride;
    q.dgate = dgate;
    q.dup = dup;
    if (int rc = ffn_map(&q.a[0], a->w_down, a->out_dim, a->inner, a->w_down_stride, narrow_box(kNarrowSlopes), "w_down"))
      return rc;
    if (int rc = ffn_map(&q.b[0], a->dout, a->m, a->out_dim, a->dout_stride, q.columns, "dout")) return rc;
    if (int rc = launch_narrow(kNarrowSlopes, q, false, call, st)) return rc;
  } else {
    GemmParams p{};
    p.count = 1;
    p.activation = a->activation;
    Gemm& g = p.g[0];
    if (int rc = ffn_map(&g.a[0], a->dout, a->m, a->out_dim, a->dout_stride, kGM, "dout")) return rc;
    if (int rc = ffn_map(&g.b[0], a->w_down, a->out_dim, a->inner, a->w_down_stride, kGK, "w_down")) return rc;
    g.M = a->m;
    g.N = a->inner;
    g.kb = g.kb_first = kb_dh;
    p.keep = a->dw_down != nullptr;
    if (p.keep)
      if (int rc = piece_map(&g.out, h, a->m, a->inner, a->inner, "workspace")) return rc;
    if (int rc = piece_map(&p.gate, a->gate, a->m, a->inner, a->gate_stride, "gate")) return rc;
    if (int rc = piece_map(&p.up, a->up, a->m, a->inner, a->up_stride, "up")) return rc;
    if (int rc = piece_map(&p.dgate, dgate, a->m, a->inner, a->inner, "workspace")) return rc;
    if (int rc = piece_map(&p.dup, dup, a->m, a->inner, a->inner, "workspace")) return rc;
    if (int rc = launch_gemm<false, true, kSlopes>(p, 2, call, st)) return rc;
  }
  if (NarrowParams q{}; a->dx != nullptr && few_tokens(a->m, a->hidden, 2 * kb_inner, kNarrowStoreMN, q)) {
    q.kb_first = kb_inner;
    q.out = static_cast<__nv_bfloat16*>(a->dx);
    q.out_stride = a->dx_stride;
    const int box = narrow_box(kNarrowStoreMN);
    if (int rc = ffn_map(&q.a[0], a->w_gate, a->inner, a->hidden, a->w_gate_stride, box, "w_gate")) return rc;
    if (int rc = ffn_map(&q.a[1], a->w_up, a->inner, a->hidden, a->w_up_stride, box, "w_up")) return rc;
    if (int rc = ffn_map(&q.b[0], dgate, a->m, a->inner, a->inner, q.columns, "workspace")) return rc;
    if (int rc = ffn_map(&q.b[1], dup, a->m, a->inner, a->inner, q.columns, "workspace")) return rc;
    if (int rc = launch_narrow(kNarrowStoreMN, q, true, call, st)) return rc;
  } else if (a->dx != nullptr) {
    GemmParams p{};
    p.count = 1;
    Gemm& g = p.g[0];
    if (int rc = ffn_map(&g.a[0], dgate, a->m, a->inner, a->inner, kGM, "workspace")) return rc;
    if (int rc = ffn_map(&g.a[1], dup, a->m, a->inner, a->inner, kGM, "workspace")) return rc;
    if (int rc = ffn_map(&g.b[0], a->w_gate, a->inner, a->hidden, a->w_gate_stride, kGK, "w_gate")) return rc;
    if (int rc = ffn_map(&g.b[1], a->w_up, a->inner, a->hidden, a->w_up_stride, kGK, "w_up")) return rc;
    g.M = a->m;
    g.N = a->hidden;
    g.kb = 2 * kb_inner;
    g.kb_first = kb_inner;
    if (int rc = piece_map(&g.out, a->dx, a->m, a->hidden, a->dx_stride, "dx", 64)) return rc;
    if (int rc = launch_gemm<false, true, kStore>(p, 3, call, st)) return rc;
  }
  GemmParams p{};
  auto weight = [&](const void* at, int64_t at_stride, int rows, const void* b, int64_t b_stride, int cols, void* out,
                    int64_t out_stride, const char* an, const char* bn, const char* on) {
    if (out == nullptr) return (int)LTXATTN_OK;
    Gemm& g = p.g[p.count++];
    if (int rc = ffn_map(&g.a[0], at, a->m, rows, at_stride, kGK, an)) return rc;
    if (int rc = ffn_map(&g.b[0], b, a->m, cols, b_stride, kGK, bn)) return rc;
    g.M = rows;
    g.N = cols;
    g.kb = g.kb_first = (int)div_up(a->m, kGK);
    return piece_map(&g.out, out, rows, cols, out_stride, on, 64);
  };
  if (int rc = weight(dgate, a->inner, a->inner, a->x, a->x_stride, a->hidden, a->dw_gate, a->dw_gate_stride,
                      "workspace", "x", "dw_gate"))
    return rc;
  if (int rc = weight(dup, a->inner, a->inner, a->x, a->x_stride, a->hidden, a->dw_up, a->dw_up_stride, "workspace", "x",
                      "dw_up"))
    return rc;
  if (int rc = weight(a->dout, a->dout_stride, a->out_dim, h, a->inner, a->inner, a->dw_down, a->dw_down_stride, "dout",
                      "workspace", "dw_down"))
    return rc;
  if (p.count == 0) return LTXATTN_OK;
  return launch_gemm<true, true, kStore>(p, 4, call, st);
}

}  // extern "C"
