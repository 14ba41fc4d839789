// rotary_embed.cu -- ltxattn_rotary_embed and ltxattn_rotary_frequencies:
// rotary positions from token indices, for the queries and (grouped) keys of
// one attention in one launch, and their gradients.
//
//   (a, b) -> magnitude * (a cos w - b sin w,  b cos w + a sin w),  w = position * frequency
//
// for every pair of the leading rotary_dim elements of a head; the inverse call
// takes -w.  All heads of a token turn by the same angles, so a thread owns one
// slot of a token (kP pairs, or kP elements behind the rotary part) and walks
// over heads with cos and sin in registers.
//
// Angle: w reaches 1e6 radians at far positions, where fp32 is off by 0.03 of a
// radian.  The number of quarter turns is formed in fp64 and reduced there to
// [-1/2, 1/2] plus a count; only that remainder, as an angle rounded to fp32, goes
// through sin and cos, and the quarters are sign and swap selects.  Products are
// fp32; each element is rounded once.
//
// Bound: memory.  q and k are read once and written once, and nothing else has
// their size.
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "../../include/ltxattn.h"
#include "ltxattn_internal.h"
#include "sm100.cuh"

namespace ltx {

int set_error_message(int status, const char* msg);

namespace {

constexpr int kRThreads = 256;      // of a CTA at most
constexpr int kFewHeads = 16;        // q's and k's together
constexpr int kTargetThreads = 128;  // slots x head lanes, where the slots alone are fewer
constexpr int kMaxRotaryDim = 8192;
constexpr int kMaxHeads = 1 << 24;   // heads are counted in 32 bits, several steps ahead

struct RView {
  const void* x;
  void* y;
  int64_t x_sb, x_sh, x_st;
  int64_t y_sb, y_sh, y_st;
  int heads;
};

struct RotaryEmbedParams {
  RView v[2];  // q, k
  int T, pairs, head_dim;
  int rows;          // B * T
  int slots;         // slots of a token: turned ones, then copied ones
  int turn_slots;    // pairs / kP
  int slot_lanes, head_lanes, token_lanes;  // a CTA's threads
  int head_groups;
  int few_heads;     // the kernel for many tokens of few heads
  const double* freq;
  const void* positions;  // or null: token t stands at t
  int pos64;
  int64_t pos_sb, pos_st, offset;
  float magnitude;
  int inverse;
};

// A run of kN elements, moved in one access.  Every element is read once and
// written once, so the lines are marked to leave the caches first; at 29760
// tokens x 64 heads x 128 that took the half layout from 186 to 150 us.
template <typename T, int kN>
struct alignas(sizeof(T) * kN) Run {
  T e[kN];
};

template <typename R>
__device__ __forceinline__ R load_run(const void* p) {
  R r;
  if constexpr (sizeof(R) == 32) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p));
  } else if constexpr (sizeof(R) == 16) {
    *reinterpret_cast<uint4*>(&r) = __ldcs(static_cast<const uint4*>(p));
  } else if constexpr (sizeof(R) == 8) {
    *reinterpret_cast<uint2*>(&r) = __ldcs(static_cast<const uint2*>(p));
  } else if constexpr (sizeof(R) == 4) {
    *reinterpret_cast<uint32_t*>(&r) = __ldcs(static_cast<const uint32_t*>(p));
  } else {
    *reinterpret_cast<uint16_t*>(&r) = __ldcs(static_cast<const uint16_t*>(p));
  }
  return r;
}

template <typename R>
__device__ __forceinline__ void store_run(void* p, const R& r) {
  if constexpr (sizeof(R) == 32) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
    asm volatile("st.global.L1::no_allocate.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]),
                 "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else if constexpr (sizeof(R) == 16) {
    __stcs(static_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&r));
  } else if constexpr (sizeof(R) == 8) {
    __stcs(static_cast<uint2*>(p), *reinterpret_cast<const uint2*>(&r));
  } else if constexpr (sizeof(R) == 4) {
    __stcs(static_cast<uint32_t*>(p), *reinterpret_cast<const uint32_t*>(&r));
  } else {
    __stcs(static_cast<uint16_t*>(p), *reinterpret_cast<const uint16_t*>(&r));
  }
}

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f(float& d, float v) { d = v; }
__device__ __forceinline__ void from_f(__nv_bfloat16& d, float v) { d = __float2bfloat16_rn(v); }

// cos and sin of position * frequency (see the head of the file).  The number of
// quarter turns is rounded by adding 1.5 * 2^52, which leaves it in the low bits
// of the sum (for angles below 2^51 quarters).  The remainder is at most pi / 4,
// where the Taylor series to x^9 and x^10 are within 2^-28.5 of sin x and 2^-32 of
// cos x, relative to them; fp32 adds some 2^-23.
__device__ __forceinline__ void turn(double position, double frequency, float& c, float& s) {
  constexpr double kMagic = 6755399441055744.0, kQuarter = 1.57079632679489661923;
  const double quarters = position * frequency * 0.63661977236758134308;  // 2 / pi
  const double shifted = quarters + kMagic;
  const float x = static_cast<float>((quarters - (shifted - kMagic)) * kQuarter);
  const float x2 = x * x;
  float ps = fmaf(x2, 1.0f / 362880, -1.0f / 5040), pc = fmaf(x2, -1.0f / 3628800, 1.0f / 40320);
  ps = fmaf(x2, ps, 1.0f / 120);
  pc = fmaf(x2, pc, -1.0f / 720);
  ps = fmaf(x2, ps, -1.0f / 6);
  pc = fmaf(x2, pc, 1.0f / 24);
  const float sr = fmaf(x * x2, ps, x);
  pc = fmaf(x2, pc, -0.5f);
  const float cr = fmaf(x2, pc, 1.0f);
  const int q = __double2loint(shifted);
  const float c1 = (q & 1) ? sr : cr, s1 = (q & 1) ? cr : sr;
  c = ((q + 1) & 2) ? -c1 : c1;
  s = (q & 2) ? -s1 : s1;
}

__device__ __forceinline__ double place(const RotaryEmbedParams& p, int b, int t) {
  int64_t at = t;
  if (p.positions != nullptr) {
    const int64_t o = b * p.pos_sb + t * p.pos_st;
    at = p.pos64 ? static_cast<const int64_t*>(p.positions)[o] : static_cast<const int32_t*>(p.positions)[o];
  }
  return static_cast<double>(at + p.offset);
}

// How a slot lies in a head.  kP pairs per turned slot: two runs of kP elements,
// `pairs` apart, in the half layout, one run of 2 kP in the interleaved one (a
// single interleaved pair is two runs of one element: its row may start
// anywhere).  Copied slots are as many runs, side by side; where their number is odd the last slot moves its run
// twice.  With one run to a copied slot, 6242 fp32 tokens x 36 heads x 64, 24 of them turned, took 28 us for 22.
template <typename T, int kP, bool kInterleaved>
struct Slot {
  static constexpr bool kTwoRuns = !kInterleaved || kP == 1;
  static constexpr int kRun = kTwoRuns ? kP : 2 * kP;
  bool turned;
  int at, apart;  // the first run in a head, and from it to the second
  float c[kP], s[kP];

  __device__ __forceinline__ Slot(const RotaryEmbedParams& p, int slot)
      : turned(slot < p.turn_slots),
        at(turned ? (kInterleaved ? 2 * kP : kP) * slot
                  : 2 * p.pairs + (kTwoRuns ? 2 : 1) * kRun * (slot - p.turn_slots)),
        apart(turned && !kInterleaved ? p.pairs : at + 2 * kRun <= p.head_dim ? kRun : 0) {}

  // through the heads h, h + step, ... of a view's token; short runs take several heads at once, to have as many
  // bytes on their way as a long one
  __device__ __forceinline__ void walk(const RView& v, int b, int t, int h, int step) const {
    if (h >= v.heads) return;
    using R = Run<T, kRun>;
    constexpr int kAtOnce = sizeof(R) >= 16 ? 1 : sizeof(R) == 8 ? 2 : 4;
    const T* x = static_cast<const T*>(v.x) + b * v.x_sb + t * v.x_st + h * v.x_sh + at;
    T* y = static_cast<T*>(v.y) + b * v.y_sb + t * v.y_st + h * v.y_sh + at;
    const int64_t dx = step * v.x_sh, dy = step * v.y_sh;
#pragma unroll 1
    for (; h < v.heads; h += kAtOnce * step, x += kAtOnce * dx, y += kAtOnce * dy) {
      R r0[kAtOnce], r1[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        if (u > 0 && h + u * step >= v.heads) break;
        r0[u] = load_run<R>(x + u * dx);
        if (kTwoRuns) r1[u] = load_run<R>(x + u * dx + apart);
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        if (u > 0 && h + u * step >= v.heads) break;
        if (turned) {
#pragma unroll
          for (int e = 0; e < kP; ++e) {
            T& ea = kTwoRuns ? r0[u].e[e] : r0[u].e[(2 * e) % kRun];
            T& eb = kTwoRuns ? r1[u].e[e] : r0[u].e[(2 * e + 1) % kRun];
            const float fa = to_f(ea), fb = to_f(eb);
            from_f(ea, fmaf(fa, c[e], -(fb * s[e])));
            from_f(eb, fmaf(fb, c[e], fa * s[e]));
          }
        }
        if (kTwoRuns) store_run(y + u * dy + apart, r1[u]);
        store_run(y + u * dy, r0[u]);
      }
    }
  }
};

// A CTA takes token_lanes tokens (one, unless its heads are few) with all their
// heads.  Its threads first make the tokens' cos and sin, into shared memory;
// then thread (slot, head lane, token) keeps its slot's in registers and walks
// over every head_lanes-th head of q and of k (few tokens: the heads are shared
// by gridDim.y CTAs, each making the cos and sin again).  The heads of a token lie side by
// side in a projection's output, so a CTA streams whole rows of it.  Many small
// CTAs keep the memory busy better than more runs per thread: 128 threads at 48
// registers (for which seven of the instances spill 4 to 36 bytes) take 150 us for
// 29760 tokens x 64 heads x 128 in bf16 (6.5 TB/s, 0.99 of the measured copy);
// fetching a head ahead of the one that turns 158, four heads at once 257.
template <typename T, int kP, bool kInterleaved>
__global__ void __launch_bounds__(kRThreads, 5) rotary_embed_kernel(const __grid_constant__ RotaryEmbedParams p) {
  extern __shared__ float2 turns[];  // [token_lanes][pairs]: (cos, sin), with the magnitude
  grid_dep_wait();  // all that is read may have been written by the kernel before
  grid_dep_launch_dependents();
  const int row0 = blockIdx.x * p.token_lanes;
  const int n_rows = min(p.token_lanes, p.rows - row0);
  {
    const int pair_lanes = min(p.pairs, (int)blockDim.x), lanes = blockDim.x / pair_lanes;
    const int r0 = threadIdx.x / pair_lanes, j0 = threadIdx.x - r0 * pair_lanes;
    for (int r = r0; r < n_rows && r0 < lanes; r += lanes) {
      const int b = (row0 + r) / p.T, t = (row0 + r) - b * p.T;
      const double position = place(p, b, t);
      for (int j = j0; j < p.pairs; j += pair_lanes) {
        float c, s;
        turn(position, p.freq[j], c, s);
        turns[r * p.pairs + j] = make_float2(c * p.magnitude, s * (p.inverse ? -p.magnitude : p.magnitude));
      }
    }
  }
  __syncthreads();
  using S = Slot<T, kP, kInterleaved>;
  const int rest = threadIdx.x / p.slot_lanes, r = rest / p.head_lanes;
  const int h0 = blockIdx.y * p.head_lanes + rest - r * p.head_lanes, step = gridDim.y * p.head_lanes;
  if (r >= n_rows) return;
  const int b = (row0 + r) / p.T, t = (row0 + r) - b * p.T;
  for (int slot = threadIdx.x % p.slot_lanes; slot < p.slots; slot += p.slot_lanes) {
    S w(p, slot);
#pragma unroll
    for (int e = 0; e < kP; ++e) {
      const float2 cs = w.turned ? turns[r * p.pairs + slot * kP + e] : make_float2(1.f, 0.f);
      w.c[e] = cs.x;
      w.s[e] = cs.y;
    }
    w.walk(p.v[0], b, t, h0, step);
    w.walk(p.v[1], b, t, h0, step);
  }
}

// Many tokens of few heads: a thread takes one slot of one token through all
// heads and makes its own cos and sin.  Nothing is computed twice, and nothing
// passes through shared memory, which for a handful of heads costs more
// instructions than the rotation itself: 116 thousand tokens x 4 heads x 176 take
// 64 us (5.1 TB/s) against 98 above, 36 thousand x 12 x 128 45 against 49; at 24
// heads the two are even, at 64 this one is slower (185 us against 152).
template <typename T, int kP, bool kInterleaved>
__global__ void __launch_bounds__(kRThreads, 5) rotary_embed_few_heads_kernel(const __grid_constant__ RotaryEmbedParams p) {
  grid_dep_wait();  // all that is read may have been written by the kernel before
  grid_dep_launch_dependents();
  const unsigned i = blockIdx.x * kRThreads + threadIdx.x, row = i / p.slots, slot = i - row * p.slots;
  if (row >= (unsigned)p.rows) return;
  const int b = row / p.T, t = row - b * p.T;
  Slot<T, kP, kInterleaved> w(p, slot);
  if (w.turned) {
    const double position = place(p, b, t);
#pragma unroll
    for (int e = 0; e < kP; ++e) {
      turn(position, p.freq[slot * kP + e], w.c[e], w.s[e]);
      w.c[e] *= p.magnitude;
      w.s[e] *= p.inverse ? -p.magnitude : p.magnitude;
    }
  }
  w.walk(p.v[0], b, t, 0, 1);
  w.walk(p.v[1], b, t, 0, 1);
}

int fail_rotary(int status, const char* fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return set_error_message(status, buf);
}

template <typename T, int kP>
cudaError_t launch(const RotaryEmbedParams& p, bool interleaved, cudaStream_t st) {
  if (p.few_heads) {
    const unsigned grid = (unsigned)((int64_t(p.rows) * p.slots + kRThreads - 1) / kRThreads);
    return launch_pdl(interleaved ? rotary_embed_few_heads_kernel<T, kP, true> : rotary_embed_few_heads_kernel<T, kP, false>,
                      grid, kRThreads, 0, st, p);
  }
  const dim3 grid((unsigned)((p.rows + (int64_t)p.token_lanes - 1) / p.token_lanes), (unsigned)p.head_groups);
  const int threads = p.slot_lanes * p.head_lanes * p.token_lanes;
  return launch_pdl(interleaved ? rotary_embed_kernel<T, kP, true> : rotary_embed_kernel<T, kP, false>, grid, threads,
                    sizeof(float2) * p.token_lanes * p.pairs, st, p);
}

// Whether every row of the view starts on a multiple of `elements` elements.  The
// stride of an extent of 1 is never used.
bool rows_aligned(const ltxattn_tensor& v, int64_t B, int64_t H, int64_t T, int elements, int size) {
  return reinterpret_cast<uintptr_t>(v.data) % (elements * size) == 0 && (B == 1 || v.stride_b % elements == 0) &&
         (H == 1 || v.stride_h % elements == 0) && (T == 1 || v.stride_t % elements == 0);
}

// Checks one input and its output; 0 or the status that fail_rotary gave.
int check_view(const char* name, const ltxattn_tensor& x, const ltxattn_tensor& y, int64_t B, int64_t H, int64_t T,
               int D, int size) {
  if (x.data == nullptr || y.data == nullptr)
    return fail_rotary(LTXATTN_ERR_ARG, "ltxattn_rotary_embed: %s and its output are required", name);
  if (reinterpret_cast<uintptr_t>(x.data) % size || reinterpret_cast<uintptr_t>(y.data) % size)
    return fail_rotary(LTXATTN_ERR_ALIGN, "ltxattn_rotary_embed: %s is not aligned to its type", name);
  if (x.stride_b < 0 || x.stride_h < 0 || x.stride_t < 0 || y.stride_b < 0 || y.stride_h < 0 || y.stride_t < 0)
    return fail_rotary(LTXATTN_ERR_SHAPE, "ltxattn_rotary_embed: %s has a negative stride", name);
  if ((B > 1 && y.stride_b < D) || (H > 1 && y.stride_h < D) || (T > 1 && y.stride_t < D))
    return fail_rotary(LTXATTN_ERR_SHAPE, "ltxattn_rotary_embed: rows of %s's output overlap", name);
  if (x.data == y.data && ((B > 1 && x.stride_b != y.stride_b) || (H > 1 && x.stride_h != y.stride_h) ||
                           (T > 1 && x.stride_t != y.stride_t)))
    return fail_rotary(LTXATTN_ERR_ARG, "ltxattn_rotary_embed: %s in place needs the input's own strides", name);
  return LTXATTN_OK;
}

}  // namespace
}  // namespace ltx

extern "C" {

int ltxattn_rotary_frequencies(const ltxattn_rotary_frequency_args* a, double* frequencies, float* magnitude) {
  using namespace ltx;
  if (a == nullptr || frequencies == nullptr || magnitude == nullptr)
    return fail_rotary(LTXATTN_ERR_ARG, "ltxattn_rotary_frequencies: args, frequencies and magnitude are required");
  if (a->rotary_dim < 2 || a->rotary_dim % 2)
    return fail_rotary(LTXATTN_ERR_SHAPE, "ltxattn_rotary_frequencies: rotary_dim (%d) must be even and >= 2",
                       a->rotary_dim);
  if (a->scaling < LTXATTN_ROTARY_NONE || a->scaling > LTXATTN_ROTARY_BANDS)
    return fail_rotary(LTXATTN_ERR_ARG, "ltxattn_rotary_frequencies: unknown scaling %d", a->scaling);
  const bool bands = a->scaling == LTXATTN_ROTARY_YARN || a->scaling == LTXATTN_ROTARY_BANDS;
  if (!(a->theta > 0) || !std::isfinite(a->theta) || (a->scaling == LTXATTN_ROTARY_YARN && !(a->theta > 1)))
    return fail_rotary(LTXATTN_ERR_ARG, "ltxattn_rotary_frequencies: theta (%g) is out of range", a->theta);
  if (a->scaling != LTXATTN_ROTARY_NONE && (!(a->factor > 0) || !std::isfinite(a->factor)))
    return fail_rotary(LTXATTN_ERR_ARG, "ltxattn_rotary_frequencies: factor (%g) must be positive", a->factor);
  if (bands && (!(a->trained_length > 0) || !std::isfinite(a->trained_length) || !(a->slow > 0) ||
                !(a->fast > a->slow) || !std::isfinite(a->fast)))
    return fail_rotary(LTXATTN_ERR_ARG,
                       "ltxattn_rotary_frequencies: trained_length must be positive and fast > slow > 0");
  const int n = a->rotary_dim / 2;
  const double two_pi = 6.283185307179586476925;
  double theta = a->theta;
  if (a->scaling == LTXATTN_ROTARY_NTK && n > 1) theta *= std::pow(a->factor, (double)n / (n - 1));
  double low = 0, high = 0;
  if (a->scaling == LTXATTN_ROTARY_YARN) {
    // the pair that turns r times in L positions: theta^(-j / n) L = 2 pi r
    auto pair_of = [&](double r) { return n * std::log(a->trained_length / (r * two_pi)) / std::log(theta); };
    low = std::fmax(std::floor(pair_of(a->fast)), 0.0);
    high = std::fmin(std::ceil(pair_of(a->slow)), (double)(a->rotary_dim - 1));
  }
  for (int j = 0; j < n; ++j) {
    const double f = std::pow(theta, -(double)j / n);
    double stretched = 0;  // the share of f / s
    switch (a->scaling) {
      case LTXATTN_ROTARY_LINEAR: stretched = 1; break;
      case LTXATTN_ROTARY_YARN:
        // a ramp that ends at pair 0 or before it leaves none alone; one that starts behind the last pair is never met
        stretched = high <= 0 ? 1.0 : std::fmin(std::fmax((j - low) / std::fmax(high - low, 0.001), 0.0), 1.0);
        break;
      case LTXATTN_ROTARY_BANDS:
        stretched = 1 - std::fmin(std::fmax((a->trained_length * f / two_pi - a->slow) / (a->fast - a->slow), 0.0), 1.0);
        break;
      default: break;
    }
    frequencies[j] = stretched == 0 ? f : f / a->factor * stretched + f * (1 - stretched);
    if (!std::isfinite(frequencies[j]) || !std::isfinite(theta))
      return fail_rotary(LTXATTN_ERR_ARG,
                         "ltxattn_rotary_frequencies: theta (%g) with factor (%g) leaves the range of a double", a->theta,
                         a->factor);
  }
  *magnitude =
      a->scaling == LTXATTN_ROTARY_YARN && a->factor > 1 ? (float)(0.1 * std::log(a->factor) + 1.0) : 1.0f;
  return LTXATTN_OK;
}

int ltxattn_rotary_embed(const ltxattn_rotary_embed_args* a, void* stream) {
  using namespace ltx;
  if (a == nullptr) return fail_rotary(LTXATTN_ERR_ARG, "args is NULL");
  if (a->dtype != LTXATTN_BF16 && a->dtype != LTXATTN_F32)
    return fail_rotary(LTXATTN_ERR_DTYPE, "ltxattn_rotary_embed: dtype must be LTXATTN_BF16 or LTXATTN_F32");
  if (a->batch < 0 || a->tokens < 0 || a->heads < 0 || a->kv_heads < 0 || a->head_dim < 1)
    return fail_rotary(LTXATTN_ERR_SHAPE, "ltxattn_rotary_embed: a size is negative, or head_dim below 1");
  if (a->rotary_dim < 2 || a->rotary_dim % 2 || a->rotary_dim > a->head_dim)
    return fail_rotary(LTXATTN_ERR_SHAPE,
                       "ltxattn_rotary_embed: rotary_dim (%d) must be even, >= 2 and at most head_dim (%d)",
                       a->rotary_dim, a->head_dim);
  if (a->layout != LTXATTN_ROTARY_HALF && a->layout != LTXATTN_ROTARY_INTERLEAVED)
    return fail_rotary(LTXATTN_ERR_ARG, "ltxattn_rotary_embed: unknown layout %d", a->layout);
  if (!std::isfinite(a->magnitude))
    return fail_rotary(LTXATTN_ERR_ARG, "ltxattn_rotary_embed: magnitude (%g) must be finite in fp32", a->magnitude);
  if (a->positions != nullptr && a->position_bits != 64 && a->position_bits != 32)
    return fail_rotary(LTXATTN_ERR_DTYPE, "ltxattn_rotary_embed: positions must be 64- or 32-bit integers");
  const int64_t B = a->batch, T = a->tokens, H = a->heads, Hk = a->kv_heads;
  if (a->rotary_dim > kMaxRotaryDim)
    return fail_rotary(LTXATTN_ERR_UNSUPPORTED, "ltxattn_rotary_embed: rotary_dim (%d) is above %d", a->rotary_dim,
                       kMaxRotaryDim);
  if (H > kMaxHeads || Hk > kMaxHeads)
    return fail_rotary(LTXATTN_ERR_UNSUPPORTED, "ltxattn_rotary_embed: more than %d heads", kMaxHeads);
  if (B == 0 || T == 0 || H + Hk == 0) return LTXATTN_OK;
  if (a->frequencies == nullptr) return fail_rotary(LTXATTN_ERR_ARG, "ltxattn_rotary_embed: frequencies is required");
  if (reinterpret_cast<uintptr_t>(a->frequencies) % 8 ||
      reinterpret_cast<uintptr_t>(a->positions) % (a->position_bits == 64 ? 8 : 4))
    return fail_rotary(LTXATTN_ERR_ALIGN, "ltxattn_rotary_embed: frequencies or positions are not aligned to their type");
  if (a->positions != nullptr && (a->position_stride_b < 0 || a->position_stride_t < 0))
    return fail_rotary(LTXATTN_ERR_SHAPE, "ltxattn_rotary_embed: positions have a negative stride");
  const bool bf16 = a->dtype == LTXATTN_BF16;
  const int size = bf16 ? 2 : 4;
  if (H > 0)
    if (int rc = check_view("q", a->q, a->q_out, B, H, T, a->head_dim, size)) return rc;
  if (Hk > 0)
    if (int rc = check_view("k", a->k, a->k_out, B, Hk, T, a->head_dim, size)) return rc;

  if (H > 0 && Hk > 0 && (a->q_out.data == a->k_out.data || a->q_out.data == a->k.data || a->k_out.data == a->q.data))
    return fail_rotary(LTXATTN_ERR_ARG, "ltxattn_rotary_embed: an output of q or k is the other's memory");

  RotaryEmbedParams p{};
  p.pairs = a->rotary_dim / 2;
  // kP: as many pairs to a slot as give runs of 16 bytes (half) or 32 (interleaved) at most, of which the pairs, the
  // part behind them and every row are multiples
  const bool il = a->layout == LTXATTN_ROTARY_INTERLEAVED;
  int kp = bf16 ? 8 : 4;
  auto fits = [&](int n) {
    const int run = il ? 2 * n : n;  // n > 1: single pairs take single elements
    if (p.pairs % n || a->head_dim % run) return false;
    if (H > 0 && !(rows_aligned(a->q, B, H, T, run, size) && rows_aligned(a->q_out, B, H, T, run, size))) return false;
    return Hk == 0 || (rows_aligned(a->k, B, Hk, T, run, size) && rows_aligned(a->k_out, B, Hk, T, run, size));
  };
  while (kp > 1 && !fits(kp)) kp /= 2;
  const ltxattn_tensor* in[2] = {&a->q, &a->k};
  const ltxattn_tensor* out[2] = {&a->q_out, &a->k_out};
  bool in_place = true;
  for (int i = 0; i < 2; ++i) {
    const int heads = i == 0 ? a->heads : a->kv_heads;
    p.v[i] = {in[i]->data,     out[i]->data,     in[i]->stride_b,  in[i]->stride_h, in[i]->stride_t,
              out[i]->stride_b, out[i]->stride_h, out[i]->stride_t, heads};
    if (heads > 0) in_place = in_place && in[i]->data == out[i]->data;
  }
  p.T = (int)T;
  if (B * T > 0x7fffffff) return fail_rotary(LTXATTN_ERR_UNSUPPORTED, "ltxattn_rotary_embed: too many tokens for one call");
  p.rows = (int)(B * T);
  p.turn_slots = p.pairs / kp;
  p.head_dim = a->head_dim;
  p.slots = p.turn_slots + (in_place ? 0 : (a->head_dim - a->rotary_dim + 2 * kp - 1) / (2 * kp));
  p.freq = a->frequencies;
  p.positions = a->positions;
  p.pos64 = a->position_bits == 64;
  p.pos_sb = a->position_stride_b;
  p.pos_st = a->position_stride_t;
  p.offset = a->offset;
  p.magnitude = a->magnitude;
  p.inverse = a->inverse != 0;
  p.slot_lanes = std::min(p.slots, kRThreads);
  p.head_lanes = std::max(1, std::min((int)std::max(H, Hk), kTargetThreads / p.slot_lanes));
  const int64_t items = int64_t(p.rows) * p.slots;
  p.few_heads = H + Hk <= kFewHeads && items >= 148 * 1024 && items <= 0x7fffffff - kRThreads;
  // few tokens: as many CTAs to a token as fill the GPU (148 SMs), at a head to a thread at least
  const int64_t threads = std::min<int64_t>(int64_t(p.rows) * p.slot_lanes * p.head_lanes, 148 * 1024);
  p.head_groups = (int)std::min<int64_t>({148 * 1024 / threads, (std::max(H, Hk) + p.head_lanes - 1) / p.head_lanes, 65535});
  p.token_lanes = std::max(1, kTargetThreads / (p.slot_lanes * p.head_lanes));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (bf16) {
    switch (kp) {
      case 8: e = launch<__nv_bfloat16, 8>(p, il, st); break;
      case 4: e = launch<__nv_bfloat16, 4>(p, il, st); break;
      case 2: e = launch<__nv_bfloat16, 2>(p, il, st); break;
      default: e = launch<__nv_bfloat16, 1>(p, il, st); break;
    }
  } else {
    switch (kp) {
      case 4: e = launch<float, 4>(p, il, st); break;
      case 2: e = launch<float, 2>(p, il, st); break;
      default: e = launch<float, 1>(p, il, st); break;
    }
  }
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail_rotary(LTXATTN_ERR_CUDA, "ltxattn_rotary_embed: %s", cudaGetErrorString(e));
  }
  return LTXATTN_OK;
}

}  // extern "C"
