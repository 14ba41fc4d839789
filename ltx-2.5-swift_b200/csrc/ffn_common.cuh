// ffn_common.cuh -- what the two kernels of the gated feed-forward block share:
// the activations and the TMA maps.
#pragma once

#include <cstdio>
#include <mutex>
#include <type_traits>

#include "../../include/ltxattn.h"
#include "ltxattn_internal.h"
#include "sm100.cuh"

namespace ltx {

// ---------------------------------------------------------------------------
// activations (fp32)

// e^-|x| never overflows, and both signs keep its relative accuracy down to where fp32 ends (with 1 / (1 + e^-x) the fast
// division gives 0 for x < -87.3, where bf16 still holds the result).  The fast division is off by 2 units of 2^-24.
__device__ __forceinline__ float sigmoid(float x) {
  const float e = __expf(-fabsf(x));
  return __fdividef(x < 0.0f ? e : 1.0f, 1.0f + e);
}

// act(g), and with kSlope its derivative too.
template <int kAct, bool kSlope>
__device__ __forceinline__ float activate(float g, float& slope) {
  if constexpr (kAct == LTXATTN_SILU) {
    const float s = sigmoid(g);
    if (kSlope) slope = s * fmaf(g, 1.0f - s, 1.0f);
    return g * s;
  } else if constexpr (kAct == LTXATTN_GELU_TANH) {
    // (1 + tanh z) / 2 = sigmoid(2 z)
    constexpr float c2 = 1.5957691216057308f;  // 2 sqrt(2 / pi)
    const float g2 = g * g;
    const float s = sigmoid(c2 * g * fmaf(0.044715f, g2, 1.0f));
    if (kSlope) {
      const float t = g * s * (1.0f - s);  // 0 far out, where g2 may be infinite
      slope = t == 0.0f ? s : fmaf(t, c2 * fmaf(0.134145f, g2, 1.0f), s);
    }
    return g * s;
  } else {
    // erfc(x / sqrt 2) / 2 = e^(-x^2 / 2) P(1 / (1 + 0.26 x)) for x >= 0, P of degree 7 fitted by reweighted least squares
    // to the least relative error over [0, 14]: 3.8e-7 with the coefficients in fp32.  Far out on the left the exponential's error counts, relative to a
    // small result: under 2^-14 with its argument's.
    // The slope needs the exponential too.  With erfcf in its place the first product of 101 tokens at 2048 x 5464 took
    // 3.4 us longer where a round of tiles waits for its epilogue.
    const float x = fabsf(g), e = __expf(-0.5f * g * g), t = __fdividef(1.0f, fmaf(0.26f, x, 1.0f));
    float q = fmaf(t, -0.0772401318f, 0.246337339f);
    q = fmaf(t, q, -0.135466337f);
    q = fmaf(t, q, 0.192206472f);
    q = fmaf(t, q, 0.0602172539f);
    q = fmaf(t, q, 0.110970601f);
    q = fmaf(t, q, 0.102938913f);
    q = fmaf(t, q, 3.57263452e-05f) * e;
    const float s = g < 0.0f ? q : 1.0f - q;
    if (kSlope) slope = fmaf(g, 0.3989422804014327f * e, s);
    return g * s;
  }
}

// Calls f with the activation as a constant.  One branch for the many elements that f handles: with one in every
// element the gradient's epilogue took longer than its MMAs (47 thousand cycles a tile for 33).
template <typename F>
__device__ __forceinline__ void with_activation(int kind, F&& f) {
  if (kind == LTXATTN_SILU)
    f(std::integral_constant<int, LTXATTN_SILU>{});
  else if (kind == LTXATTN_GELU_TANH)
    f(std::integral_constant<int, LTXATTN_GELU_TANH>{});
  else
    f(std::integral_constant<int, LTXATTN_GELU>{});
}

__device__ __forceinline__ float lo_f(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float hi_f(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// The gradient through act(g) * u from dh: (dg, du), and the product itself.
template <int kAct>
__device__ __forceinline__ void slopes(float g, float u, float dh, float& dg, float& du, float& h) {
  float slope;
  const float a = activate<kAct, true>(g, slope);
  dg = dh * u * slope;
  du = dh * a;
  h = a * u;
}

// 8 of v, from `at` on, as bf16.
template <int kN>
__device__ __forceinline__ uint4 pack8(const float (&v)[kN], int at = 0) {
  return make_uint4(pack_bf16x2(v[at], v[at + 1]), pack_bf16x2(v[at + 2], v[at + 3]),
                    pack_bf16x2(v[at + 4], v[at + 5]), pack_bf16x2(v[at + 6], v[at + 7]));
}
__device__ __forceinline__ void unpack8(const uint4& w, float (&v)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[2 * e] = lo_f(u[e]);
    v[2 * e + 1] = hi_f(u[e]);
  }
}

// ---------------------------------------------------------------------------
// clusters

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

// Every thread of every CTA of the cluster comes here, whatever happened before:
// a CTA whose wait gave up still arrives.  Shared memory written before is
// visible to the cluster after.
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

// The same for CTAs that have read one another's shared memory and write nothing that another reads: the fence ends
// the reads before the arrival, without waiting for stores on their way to global memory.
__device__ __forceinline__ void cluster_barrier_after_reads() {
  asm volatile("fence.acq_rel.cta;" ::: "memory");
  asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  asm volatile("barrier.cluster.wait;" ::: "memory");
}

// The address that `local` has in this CTA, of the CTA with that rank (shared::cluster window).
__device__ __forceinline__ uint32_t peer_address(uint32_t local, uint32_t rank) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(local), "r"(rank));
  return at;
}

// ---------------------------------------------------------------------------
// host side

// Records the message and gives the status back.
int fail_ffn(int status, const char* fmt, ...);

// bf16 [rows, cols], `stride` elements between rows; boxes of box_cols columns (64 or 32: one row of the 128- or
// 64-byte swizzle) and box_rows rows.
int ffn_map(CUtensorMap* m, const void* ptr, int64_t rows, int64_t cols, int64_t stride, int box_rows, const char* name,
            int box_cols = 64);

constexpr int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int kFfnK = 64;  // K per pipeline stage: one 128-byte swizzle row of bf16

// One product of the block for few tokens (ffn_narrow_sm100.cu): the weights'
// rows or columns are the rows of the accumulator, the tokens its columns.
struct NarrowParams {
  CUtensorMap a[2];  // weights (kNarrowProduct: gate and up; else K slices from kb_first on come from the second pair)
  CUtensorMap b[2];  // tokens
  int tokens, features;
  int kb, kb_first;      // 64-wide K slices in all, and of the first pair
  int columns;           // tokens of a tile: a multiple of 16, the box of b
  int cluster;           // CTAs that share a tile
  int token_tiles;
  int stages;
  int follows;           // the kernel before it in the stream belongs to the same call
  int activation;
  __nv_bfloat16* out;    // [tokens, features]
  int64_t out_stride;
  __nv_bfloat16 *gate, *up, *dgate, *dup;  // as GemmParams
  int64_t gate_stride, up_stride, dgate_stride, dup_stride;
  int* err;
};

enum NarrowMode {
  kNarrowProduct,  // out = act(x Wg^T) * (x Wu^T), weights K-major
  kNarrowStore,    // out = h Wd^T, weights K-major
  kNarrowSlopes,   // dh = dout Wd and what follows from it, weights MN-major
  kNarrowStoreMN   // dx = dg Wg + du Wu, weights MN-major
};

// How such a product is cut: tokens of a tile, CTAs that share a tile, and what it is expected to take.
struct NarrowPlan {
  int columns, cluster;
  double us;
};
NarrowPlan plan_narrow(NarrowMode mode, int tokens, int features, int kb);
// Rows of the boxes of a[]: 128 features K-major, 64 of K MN-major.
inline int narrow_box(NarrowMode mode) { return mode == kNarrowProduct || mode == kNarrowStore ? 128 : kFfnK; }
// `follows`: the kernel before it in the stream belongs to the same call and does not write the weights.
int launch_narrow(NarrowMode mode, NarrowParams& p, bool follows, const char* call, cudaStream_t st);

}  // namespace ltx
