// Losses over the tied output table (include/mf_loss.h): softmax cross
// entropy over the whole vocabulary and distillation from a teacher's top
// logits, with their gradients.
//
// Forward, one pass: scores S = H E^T tile by tile on the tensor cores; each
// row keeps a running maximum m and sum l = sum exp(s - m) in registers while
// its pair of CTAs walks the vocabulary, and picks the wanted columns' scores
// out of the accumulator; a small kernel joins the walks.
// Backward: the scores again, a piece of the vocabulary at a time, turned into
// d = T g (p - q) in the epilogue and stored in 16 bits (a piece, never all of
// it; the tensor cores multiply 16-bit numbers, and a second 16 bits would double
// both products and d's traffic, which only up to 64 rows cost little), then two
// products on the piece: d E into FP32 sums of d_hidden and
// d^T H into d_embedding.  One launch makes piece i + 1 of d and the products
// of piece i, so the many small score tiles fill the SMs that the long product
// tiles leave idle; a last kernel joins and rounds d_hidden.
//
// All three products are one engine: tile = 256 rows (M) x up to 256 columns
// (N) on a pair of CTAs (tcgen05 cta_group::2), K in chunks of 64 through a
// ring of shared-memory stages filled by TMA, two accumulators in TMEM so that
// one drains while the next fills.  A persistent grid of one pair per two SMs;
// each pair works through fixed ranges of tiles chosen on the host.
//   S  = H E^T   A = hidden rows (K-major), B = table rows (K-major)
//   d E          A = d (K-major),           B = table piece (N-major)
//   d^T H        A = d (M-major),           B = scaled hidden copy (N-major)
// Every mbarrier wait is bounded; a pair whose wait runs out writes NaN into
// what is left of its tiles, drains its copies and returns.
//
// What bounds it (4,096 x 16,384 x 576, clocks counted in the kernel): the MMAs of
// a score tile's 64-K chunk take 668 clocks with neither copies nor an epilogue
// running (1.63 PFLOP/s at the clock seen), 708 with both; the epilogue warps are
// busy for half of a tile forward and two thirds of one backward.  Long runs
// are held by the power limit.  Measured (fp16, 8,192 x 49,152 x 576): a call alone
// after idling forward 342 to 370 us (1.25 to 1.36 PFLOP/s), backward 1,165 to 1,224
// us (1.14 to 1.19 PFLOP/s over its three products); in a run of two seconds, at
// 1,370 to 1,560 MHz under the power cap, 375 and 1,305 us, a step of both 1,676 us.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <initializer_list>
#include <mutex>

#include "common.cuh"
#include "mf_loss.h"
#include "tcgen05.cuh"

namespace mfb {
namespace loss {

constexpr int kBM = 128;       // rows of a tile per CTA (256 per pair)
constexpr int kBN = 256;       // columns of a score tile
constexpr int kBK = 64;        // K elements per chunk
constexpr int kMaxStages = 6;
constexpr int kChunkBytes = kBM * kBK * 2;    // 128 rows x 64 K: 16 KB
constexpr int kRingBytes = 14 * kChunkBytes;  // tiles in shared memory, per CTA
constexpr int kEpiWarps = 8;   // two per TMEM lane quadrant, each on half the columns
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr uint32_t kTmemCols = 512;
constexpr int kSetupThreads = 1024;
constexpr uint32_t kMaxPairs = 74;             // pairs of the persistent grid
constexpr uint64_t kPieceBytes = 128ull << 20; // one piece of d
constexpr uint32_t kHalvesRows = 64;           // up to these, d in two halves
constexpr float kLog2e = 1.4426950408889634f, kLog2eLow = (float)(1.4426950408889634 - (double)kLog2e);
constexpr float kLn2 = 0.6931471805599453f, kLn2Low = (float)(0.6931471805599453 - (double)kLn2);
// A maximum below this (units of ln 2) is that of masked columns: -inf, whose
// exponential relative to itself is NaN, or a score whose rounding is more than
// an exponential's range.  Their exponentials are taken as they are, that is 0.
constexpr float kMasked = -2147483648.f;

// kLostPerProduct: the tensor core's additions drop the bits that fall below the
// sum's last place, so a score of K products comes out too small, the more the
// products are of one sign and the more bits they have.  Measured over 16,384 rows
// for K from 192 to 2,048, relative to the score and per product, in 1e-9:
//   cosine of the two rows    0.1   0.3   0.5   0.7   0.8   0.9   1
//   fp16                      1.2   1.7   2.4   2.9   3.5   4.4   4.7 to 6.1
//   bfloat16                  0.9   1.1   1.2   1.2   1.3   1.6   1.7 to 3.0
// with a standard deviation of 1e-7 to 4e-7 of the score.  Scores are scaled by 1 + K
// times a number between those of the rows that a softmax is made of (0.5 and above).
template <typename T>
struct Type;
template <>
struct Type<__half> {
  static constexpr float kLostPerProduct = 3e-9f;
  // d / (largest weight) is at most 1: times 2^15 it uses fp16's whole range,
  // and keeps full precision down to 2^-29 of the largest weight
  static constexpr float kScale = 32768.f;
  static constexpr uint32_t kFormat = 0;  // of the instruction descriptor
  static constexpr CUtensorMapDataType kMap = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  static __device__ __forceinline__ float to(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half from(float x) { return __float2half_rn(x); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint32_t least(uint32_t a, uint32_t b) {  // NaN stays
    uint32_t d;
    asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
};
template <>
struct Type<__nv_bfloat16> {
  static constexpr float kLostPerProduct = 1.25e-9f;
  static constexpr float kScale = 1.f;
  static constexpr uint32_t kFormat = 1;
  static constexpr CUtensorMapDataType kMap = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  static __device__ __forceinline__ float to(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 from(float x) { return __float2bfloat16_rn(x); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint32_t least(uint32_t a, uint32_t b) {  // NaN stays
    uint32_t d;
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
};

// A teacher's distribution over its set: q = exp((t - top) / T) * share.  The
// largest logit and 1 / (sum of the exponentials) stay apart: in one FP32 number
// top / T + log sum, logits around 10,000 leave q's sum off by 5e-4.
struct Teacher {
  float top;       // of the logits; -inf: no entry that counts, NaN: invalid
  float share;
  float entropy;   // sum q log q
};

// What a row wants: one target, or a teacher's set.
struct Wanted {
  const uint32_t* targets;   // cross entropy
  const int32_t* offsets;    // distillation
  const int32_t* ids;
  const float* logits;
  float inv_t;               // 1 / temperature (1 for cross entropy)
  Teacher* stat;             // distillation
};

__device__ __forceinline__ bool stat_empty(const Teacher& s) { return s.top == -INFINITY; }
__device__ __forceinline__ bool stat_invalid(const Teacher& s) { return s.top != s.top; }

// Of one row over one walk through the vocabulary, half of every tile's
// columns: the largest score m in units of ln 2 and the sum of exp relative to
// it.  Distillation: the sum of q (s / T - m) and that of q; a loss is a small
// difference of the two where teacher and student are sure of the same id, so
// it is never made of numbers of the scores' size.  Cross entropy: the target's
// score as the tensor core gave it, and 0.
struct __align__(16) Partial {
  float m, l, dot, q;
};

// What a sum with the maximum m is relative to: masked columns have no part in it.
__device__ __forceinline__ float base_of(float m) { return m < kMasked ? 0.f : m; }

// lse = (m + log2 l) ln 2, rounded once: backward takes p from its distance to
// the scores.
__device__ __forceinline__ float lse_of(float m, float l) {
  const float g = log2f(l), z = m + g;
  if (!(fabsf(z) < INFINITY)) return z;
  const float low = fabsf(m) > fabsf(g) ? (m - z) + g : (g - z) + m;
  return fmaf(z, kLn2, fmaf(z, kLn2Low, low * kLn2));
}

// The same way back: lse in units of ln 2 and what that rounds off.
__device__ __forceinline__ float2 lse_units(float lse) {
  const float z = lse * kLog2e;
  return make_float2(z, fmaf(lse, kLog2e, -z) + lse * kLog2eLow);
}

// The teacher's distribution in row r, by one warp.
__device__ __forceinline__ Teacher teacher_stat(const Wanted& w, uint32_t r, uint32_t entries,
                                                uint32_t vocab) {
  const uint32_t lane = threadIdx.x & 31;
  const int32_t a = w.offsets[r], b = w.offsets[r + 1];
  bool bad = a < 0 || b < a || (uint32_t)b > entries;
  Teacher st{-INFINITY, 0.f, 0.f};
  if (!bad) {
    for (int32_t k = a + (int32_t)lane; k < b; k += 32) {
      const int32_t id = w.ids[k];
      const float t = w.logits[k];
      bad |= id < 0 || (uint32_t)id >= vocab || (k > a && w.ids[k - 1] >= id) || t != t ||
             t == INFINITY;
      st.top = fmaxf(st.top, t);
    }
  }
  bad = __any_sync(0xFFFFFFFFu, bad);
  for (int o = 16; o; o >>= 1) st.top = fmaxf(st.top, __shfl_xor_sync(0xFFFFFFFFu, st.top, o));
  if (bad) {
    st.top = __uint_as_float(0x7FC00000u);
  } else if (st.top > -INFINITY) {
    float l = 0.f;
    for (int32_t k = a + (int32_t)lane; k < b; k += 32) l += expf((w.logits[k] - st.top) * w.inv_t);
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
    st.share = 1.f / l;
    const float log_l = logf(l);
    for (int32_t k = a + (int32_t)lane; k < b; k += 32) {
      const float x = (w.logits[k] - st.top) * w.inv_t, q = expf(x) * st.share;
      if (q > 0.f) st.entropy += q * (x - log_l);
    }
    for (int o = 16; o; o >>= 1) st.entropy += __shfl_xor_sync(0xFFFFFFFFu, st.entropy, o);
  }
  return st;
}

__global__ void teacher_kernel(Wanted w, uint32_t rows, uint32_t entries, uint32_t vocab) {
  pdl_wait();
  pdl_trigger();
  for (uint32_t r = (blockIdx.x * blockDim.x + threadIdx.x) >> 5; r < rows;
       r += (gridDim.x * blockDim.x) >> 5) {
    const Teacher st = teacher_stat(w, r, entries, vocab);
    if ((threadIdx.x & 31) == 0) w.stat[r] = st;
  }
}

// First entry of row r's set with an id >= v.
__device__ __forceinline__ int32_t first_entry(const Wanted& w, uint32_t r, uint32_t v) {
  int32_t lo = w.offsets[r], hi = w.offsets[r + 1];
  while (lo < hi) {
    const int32_t mid = lo + (hi - lo) / 2;
    if ((uint32_t)w.ids[mid] < v) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// The same with seven probes in flight at a time, in entries [lo, hi): three waits
// for memory in place of nine for 300 entries.
__device__ __forceinline__ int32_t first_entry_of_8(const int32_t* ids, int32_t lo, int32_t hi,
                                                    uint32_t v) {
  while (lo < hi) {
    const int32_t step = (hi - lo + 7) / 8;
    int32_t below = 0;
#pragma unroll
    for (int32_t j = 1; j < 8; ++j) {
      const int64_t k = (int64_t)lo + (int64_t)step * j - 1;
      below += k < hi && (uint32_t)ids[k] < v;
    }
    lo += below * step;
    if (below < 7) hi = (int32_t)min((int64_t)hi, (int64_t)lo + step - 1);
  }
  return lo;
}

struct RowGrad {  // one row's factors of d
  float coef;     // d16 = (p - q) * coef
  float scale;    // d_hidden = (d16 . E) * scale
  float target;   // cross entropy: d16 at the target
};

__device__ __forceinline__ float row_weight(const Wanted& w, const float* grad, uint32_t r,
                                            uint32_t vocab) {
  if (w.targets) return w.targets[r] < vocab ? grad[r] : 0.f;
  const Teacher s = w.stat[r];
  return stat_empty(s) || stat_invalid(s) ? 0.f : grad[r] / w.inv_t;
}

__device__ __forceinline__ float min_nan(float a, float b) {  // NaN stays
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// hidden row . table row by one warp on the FP32 pipes, rounding to nearest.
template <typename T>
__device__ __forceinline__ float warp_score(const T* a, const T* b, uint32_t width) {
  float s0 = 0.f, s1 = 0.f;
  for (uint32_t c = (threadIdx.x & 31) * 8; c < width; c += 256) {
    const uint4 x = ld_v4(a + c), y = ld_v4(b + c);
    const T *xs = reinterpret_cast<const T*>(&x), *ys = reinterpret_cast<const T*>(&y);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      s0 = fmaf(Type<T>::to(xs[j]), Type<T>::to(ys[j]), s0);
      s1 = fmaf(Type<T>::to(xs[j + 1]), Type<T>::to(ys[j + 1]), s1);
    }
  }
  float s = s0 + s1;
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  return s;
}

// p - 1 of a row's target, by one warp.  lse holds the target's score as
// warp_score gives it (put_target), so that is the score here too: with the
// tensor core's, which loses up to 2e-6 of a score of 576 products, a target with
// 1 - p = 1e-5 at a score of 30 had a gradient several times too large, or none.
// What is left is lse's own rounding, 2^-24 |lse|.
template <typename T>
__device__ __forceinline__ float target_short(const T* hidden, const T* table, uint32_t r,
                                              uint32_t target, uint32_t width, float lse) {
  const float s = warp_score(hidden + (uint64_t)r * width, table + (uint64_t)target * width, width);
  return min_nan(expm1f(s - lse), 0.f);
}

// Row factors and the copy of the hidden rows that d_embedding is made of.
// Every block finds the largest weight by itself (8 bytes a row from L2, many
// in flight); then a warp per row.
template <typename T>
__global__ void __launch_bounds__(kSetupThreads, 1)
setup_kernel(Wanted w, const float* grad, const T* hidden, const T* table, const float* lse, T* scaled,
             RowGrad* rg, float* gmax_out, uint32_t rows, uint32_t width, uint32_t vocab,
             uint32_t halves) {
  __shared__ float s_max[kSetupThreads / 32];
  pdl_wait();
  pdl_trigger();
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float g = 0.f;
#pragma unroll 8
  for (uint32_t r = threadIdx.x; r < rows; r += kSetupThreads) {
    const float a = fabsf(row_weight(w, grad, r, vocab));
    g = fmaxf(g, a < INFINITY ? a : 0.f);  // an infinite weight spoils its own row only
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xFFFFFFFFu, g, o));
  if (lane == 0) s_max[warp] = g;
  __syncthreads();
  g = s_max[lane % (kSetupThreads / 32)];
#pragma unroll
  for (int o = 16; o; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xFFFFFFFFu, g, o));
  if (blockIdx.x == 0 && threadIdx.x == 0) *gmax_out = g;
  for (uint32_t r = blockIdx.x * (kSetupThreads / 32) + warp; r < rows;
       r += gridDim.x * (kSetupThreads / 32)) {
    const float wr = row_weight(w, grad, r, vocab);
    // |wr| / gmax = mant 2^e with mant in (1/2, 1]: d16 carries mant, the
    // hidden row 2^e, which is exact
    int e = 0;
    float mant = 0.f, two_e = 0.f;
    if (wr != 0.f) {
      mant = frexpf(wr / g, &e);
      if (fabsf(mant) == 0.5f) mant *= 2.f, e -= 1;
      two_e = ldexpf(1.f, e);
    }
    const float coef = mant * Type<T>::kScale;
    const float miss = w.targets && wr != 0.f
                           ? target_short(hidden, table, r, w.targets[r], width, lse[r]) : 0.f;
    if (lane == 0) rg[r] = RowGrad{coef, g * two_e / Type<T>::kScale, miss * coef};
    for (uint32_t c = lane * 8; c < width; c += 256) {
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (wr != 0.f) {
        x = ld_v4(hidden + (uint64_t)r * width + c);
        T* v = reinterpret_cast<T*>(&x);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = Type<T>::from(Type<T>::to(v[j]) * two_e);
      }
      for (uint32_t i = 0; i < halves; ++i)
        *reinterpret_cast<uint4*>(scaled + (uint64_t)(r + i * rows) * width + c) = x;
    }
  }
}

// ---- the tile engine ----------------------------------------------------

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 32 TMEM lanes x 32 consecutive f32 columns -> 32 registers per thread, valid
// after tmem_wait_ld.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Two FP32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

__device__ __forceinline__ void add_v4(float* p, const uint32_t* v) {
  asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1,%2,%3,%4};" ::"l"(p),
               "f"(__uint_as_float(v[0])), "f"(__uint_as_float(v[1])), "f"(__uint_as_float(v[2])),
               "f"(__uint_as_float(v[3]))
               : "memory");
}
__device__ __forceinline__ void store_v8(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// Shared-memory descriptor of an operand whose M or N index is contiguous:
// atoms of `atom_bytes` (128: SWIZZLE_128B, 64: SWIZZLE_64B) x 8 k, k groups
// 8 atom_bytes apart (SBO), atoms one 64-k box apart (LBO), version 1 (sm_100).
__device__ __forceinline__ uint64_t mn_desc(uint32_t addr, uint32_t atom_bytes) {
  uint64_t d = 0;
  d |= (uint64_t)((addr >> 4) & 0x3FFFu);
  d |= (uint64_t)((kBK * atom_bytes) >> 4) << 16;
  d |= (uint64_t)((8 * atom_bytes) >> 4) << 32;
  d |= 1ull << 46;
  d |= (atom_bytes == 128 ? 2ull : 4ull) << 61;
  return d;
}

__device__ __forceinline__ void mma_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc,
                                         uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void bar_arrive_relaxed_local(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// One CTA on its own: MMA, commit, load.
__device__ __forceinline__ void mma_one(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_commit_one(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   bar)
               : "memory");
}
__device__ __forceinline__ void tma_load_local(uint32_t dst, const CUtensorMap* map, int x, int y,
                                               uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

struct Maps {
  CUtensorMap hidden, table;   // K-major score operands, 64 x 128 boxes
  CUtensorMap d_k, table_n;    // d E: 64 x 128 and 32 x 64 boxes
  CUtensorMap d_m, scaled_n;   // d^T H: 64 x 64 and 32 x 64 boxes
};

enum : uint32_t { kHidden = 0, kTable = 1, kScore = 2 };  // in the order of a walk

struct Params {
  uint32_t rows, width, vocab;
  uint32_t m_tiles;             // 256-row tiles of the batch
  uint32_t w_chunks;            // ceil(width / 64)
  // score tiles: vocabulary rows [v0, v0 + cols)
  uint32_t v0, cols, n_tiles;
  uint32_t keep_hidden;         // the hidden tile stays in shared memory
  uint32_t s_ring, s_stages, s_stage_bytes;
  float score_scale;            // 1 + what the tensor core's additions lose
  uint32_t score_accs, seg_chunks;  // kHalves: accumulators of a score tile, chunks in the first
  Partial* partial;             // forward: [rows][slots]
  uint32_t slots;
  void* d;                      // backward: the piece being made
  uint32_t d_rows;              // its rows: the batch's, or twice them (high and low halves)
  uint32_t pitch;
  const float* lse;
  const RowGrad* rg;
  // product tiles: vocabulary rows [pv0, pv0 + pcols)
  uint32_t pv0, pcols, bn, bn_tiles;
  uint32_t blocks;               // 256-row blocks that share a tile's B
  uint32_t t_tiles;              // 256-row tiles of the piece
  uint32_t p_stages, p_stage_bytes;
  uint32_t p_chunks, per_split;  // d E: K chunks of the piece, and of one split
  float* planes;                 // this piece's: [splits][d_rows][width]
  uint32_t add;                  // they hold an earlier piece's sums
  uint32_t r_chunks;             // d^T H: K chunks of d_rows
  void* table_out;               // d_embedding + pv0 rows
  uint32_t wide_rows;            // its rows start on 32 bytes
  const float* gmax;
  // per pair: tile ranges of the three kinds
  uint32_t hidden_at[kMaxPairs + 1], table_at[kMaxPairs + 1], score_at[kMaxPairs + 1];
};

// Shared memory: one region that score tiles and product tiles lay out
// differently, each kind with barriers of its own (a pair does all its products
// before its scores, and drains between).
//   products  p_stages x (up to 16 KB of B, blocks x 16 KB of A)
//   scores    the hidden tile of 5 to 9 chunks of 16 KB and up to 6 x 16 KB of
//             table; for other widths 6 x (16 KB of table, 16 KB of hidden rows)
// Kept, a hidden tile crosses L2 -> SM once per row tile instead of once per score
// tile: 351 against 365 us for 8,192 x 49,152 forward, where power is the limit,
// and no difference for small batches.
struct Smem {
  static constexpr int bars = kRingBytes;
  // barriers: product full, empty, score full, empty [6 each],
  // acc_full[2], acc_empty[2], drain
  static constexpr int n_bars = 4 * kMaxStages + 5;
  static constexpr int tmem_slot = bars + n_bars * 8;
  static constexpr int abort_flag = tmem_slot + 4;
  // u32: product stages and score stages filled
  static constexpr int issued = abort_flag + 4;
  static constexpr int size = issued + 4 * 2;
};
constexpr size_t kSmemBytes = Smem::size + 1024;  // + alignment slack
static_assert(kSmemBytes <= 227 * 1024, "shared memory");

// Walks over the tiles of one pair, in order: d E, d^T H, scores.  Within a
// kind n runs fastest, then m, then (d E) the split.  Steps are additions: the
// MMA issuer has a few hundred clocks between tiles, and shares its scheduler
// with two busy warps.
struct Walk {
  uint32_t kind, left;             // tiles left of this kind, the current one among them
  uint32_t n, m, split;            // the current tile
  uint32_t blocks, k0, chunks;     // its row blocks of 256, first K chunk, chunks
  uint32_t n_end, m_end, m_step, pair;

  __device__ __forceinline__ Walk(const Params& p, uint32_t of_pair) : pair(of_pair) {
    kind = kHidden;
    start(p);
  }
  __device__ __forceinline__ bool done() const { return left == 0; }
  // The current kind's range, or the next one's that is not empty.
  __device__ __forceinline__ void start(const Params& p) {
    for (;;) {
      const uint32_t* at = kind == kHidden ? p.hidden_at : (kind == kTable ? p.table_at : p.score_at);
      uint32_t x = at[pair];
      left = at[pair + 1] - x;
      if (left > 0) {
        n_end = kind == kScore ? p.n_tiles : p.bn_tiles;
        m_end = kind == kTable ? p.t_tiles : p.m_tiles;
        m_step = kind == kScore ? 1u : p.blocks;
        n = x % n_end;
        x /= n_end;
        const uint32_t groups = (m_end + m_step - 1) / m_step;
        m = x % groups * m_step;
        split = x / groups;
        set(p);
        return;
      }
      if (kind == kScore) return;
      ++kind;
    }
  }
  __device__ __forceinline__ void set(const Params& p) {
    blocks = min(m_step, m_end - m);
    k0 = split * p.per_split;  // 0 but for d E
    chunks = kind == kHidden ? min(p.per_split, p.p_chunks - k0)
                             : (kind == kTable ? p.r_chunks : p.w_chunks);
  }
  __device__ __forceinline__ void next(const Params& p) {
    if (--left == 0) {
      if (kind == kScore) return;
      ++kind;
      start(p);
      return;
    }
    if (++n == n_end) {
      n = 0;
      m += m_step;
      if (m >= m_end) {
        m = 0;
        ++split;
      }
      set(p);
    }
  }
};

// A ring of stages: which one is next, and the parity of its barriers.
struct Ring {
  uint32_t n, at = 0, fills = 0;  // `fills`: earlier fills of stage `at`
  __device__ __forceinline__ explicit Ring(uint32_t stages) : n(stages) {}
  __device__ __forceinline__ void next() {
    if (++at == n) at = 0, ++fills;
  }
};

// The wanted columns of one row, ascending, through a window of four.
template <bool kDistill>
struct Cursor {
  uint32_t id[kDistill ? 4 : 1];
  float t[kDistill ? 4 : 1];
  int32_t at, end;

  __device__ __forceinline__ void none() {
    id[0] = 0xFFFFFFFFu;
    at = end = 0;
    if constexpr (kDistill) id[1] = id[2] = id[3] = 0xFFFFFFFFu;
  }
  // Row r from its first entry >= v on.
  __device__ __forceinline__ void start(const Wanted& w, uint32_t r, uint32_t v, bool live) {
    none();
    if (!live) return;
    if constexpr (kDistill) {
      at = first_entry(w, r, v);
      end = w.offsets[r + 1];
    } else {
      id[0] = w.targets[r];
    }
  }
  __device__ __forceinline__ void pop() {
    if constexpr (kDistill) {
#pragma unroll
      for (int i = 0; i < 3; ++i) id[i] = id[i + 1], t[i] = t[i + 1];
      id[3] = 0xFFFFFFFFu;
    } else {
      id[0] = 0xFFFFFFFFu;
    }
  }
  __device__ __forceinline__ void fill(const Wanted& w) {
    if constexpr (kDistill) {
      int n = 0;  // slots in use
#pragma unroll
      for (int i = 0; i < 4; ++i) n += id[i] != 0xFFFFFFFFu;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int32_t k = at + i - n;
        if (i >= n && k < end) id[i] = (uint32_t)w.ids[k], t[i] = w.logits[k];
      }
      at = min(end, at + 4 - n);
    }
  }
  // Takes the first entry off in the lanes that say so.  All lanes of the warp
  // call it: where one has used its window up, all top theirs up, so that a
  // tile waits for memory a few times and not once for every lane.
  __device__ __forceinline__ void drop(const Wanted& w, bool mine) {
    if (mine) pop();
    if constexpr (kDistill)
      if (__any_sync(0xFFFFFFFFu, id[0] == 0xFFFFFFFFu && at < end)) fill(w);
  }
  // Drops entries below v.
  __device__ __forceinline__ void skip_to(const Wanted& w, uint32_t v) {
    if constexpr (kDistill) {
      while (__any_sync(0xFFFFFFFFu, id[0] < v)) drop(w, id[0] < v);
    }
  }
  // The weight of the first entry; t2: 1 / T in units of ln 2.
  __device__ __forceinline__ float weight(float t2, float top, float share) const {
    if constexpr (kDistill) return exp2_approx((t[0] - top) * t2) * share;
    return 1.f;
  }
};

// r[i] for an index that differs from lane to lane (31 and 63 selects).
__device__ __forceinline__ float pick32(const uint32_t (&r)[32], uint32_t i) {
  uint32_t a[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) a[j] = (i & 16u) ? r[j + 16] : r[j];
#pragma unroll
  for (int s = 8; s > 0; s >>= 1)
#pragma unroll
    for (int j = 0; j < s; ++j) a[j] = (i & (uint32_t)s) ? a[j + s] : a[j];
  return __uint_as_float(a[0]);
}
__device__ __forceinline__ float pick64(const uint32_t (&r)[64], uint32_t i) {
  uint32_t a[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) a[j] = (i & 32u) ? r[j + 32] : r[j];
#pragma unroll
  for (int s = 16; s > 0; s >>= 1)
#pragma unroll
    for (int j = 0; j < s; ++j) a[j] = (i & (uint32_t)s) ? a[j + s] : a[j];
  return __uint_as_float(a[0]);
}

// kHalves (backward, up to 64 rows): d as the sum of two 16-bit numbers.  Both
// CTAs of a pair then hold the same rows' scores, and each takes half the columns;
// a score may be summed in two segments of its products, one in each accumulator,
// as the forward kernel of these rows sums it.
template <typename T, bool kForward, bool kDistill, bool kHalves>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
engine_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p, Wanted w) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(sm);
  const uint32_t bar0 = sbase + Smem::bars;
  auto p_full = [&](uint32_t st) { return bar0 + 8 * st; };
  auto p_empty = [&](uint32_t st) { return bar0 + 8 * (kMaxStages + st); };
  auto s_full = [&](uint32_t st) { return bar0 + 8 * (2 * kMaxStages + st); };
  auto s_empty = [&](uint32_t st) { return bar0 + 8 * (3 * kMaxStages + st); };
  auto acc_full = [&](uint32_t b) { return bar0 + 8 * (4 * kMaxStages + b); };
  auto acc_empty = [&](uint32_t b) { return bar0 + 8 * (4 * kMaxStages + 2 + b); };
  const uint32_t drain = bar0 + 8 * (4 * kMaxStages + 4);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(sm + Smem::abort_flag);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + Smem::tmem_slot);
  volatile uint32_t* issued = reinterpret_cast<volatile uint32_t*>(sm + Smem::issued);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t rank;  // 0 = leader (issues the MMAs), 1 = peer
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const bool leader = rank == 0;
  const uint32_t pair = blockIdx.x >> 1;

  if (threadIdx.x == 0) {
    for (uint32_t st = 0; st < 4 * kMaxStages; ++st) bar_init(bar0 + 8 * st, 1);
    issued[0] = issued[1] = 0u;
    for (int b = 0; b < 2; ++b) {
      bar_init(acc_full(b), 1);
      bar_init(acc_empty(b), 2 * kEpiWarps);  // leader's: one arrival per epilogue warp of the pair
    }
    bar_init(drain, 1);
    *abort_flag = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  fence_before();
  cluster_sync();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  Walk t(p, pair);
  pdl_wait();  // the previous kernel's results, before any bounded wait begins
  pdl_trigger();

  if (warp == 0) {
    // ---- producer: both CTAs load their halves; the copies complete on the
    // leader's barriers, whose expected byte counts cover both ----
    if (lane == 0) {
      Ring pr(p.p_stages), sr(p.s_stages);
      uint32_t held = 0xFFFFFFFFu;  // row tile of the kept hidden tile
      const uint32_t leader_p_full = mapa(p_full(0), 0), leader_s_full = mapa(s_full(0), 0);
      bool ok = true;
      for (bool scores = false; ok && !t.done() && !*abort_flag; t.next(p)) {
        const int arow = (int)(t.m * 2 * kBM + rank * kBM);
        if (t.kind == kScore) {
          const int hrow = kHalves ? 0 : arow;
          if (!scores) {  // every product stage read by its MMAs
            scores = true;
            for (uint32_t st = 0; ok && st < pr.n; ++st) {
              const uint32_t fills = pr.fills + (st < pr.at ? 1u : 0u);
              ok = bar_wait(p_empty(st), (fills & 1u) ^ 1u);
            }
            if (!ok) break;
          }
          const int brow = (int)(p.v0 + t.n * kBN + rank * (kBN / 2));
          const int k_end = (int)(t.chunks * kBK);
          // A kept hidden chunk may be replaced once the MMAs of the tile before
          // have read it: `chunks` fills ago, while the stage's own wait covers
          // all but the last s_stages <= chunks fills.
          const bool load_a = !p.keep_hidden || t.m != held;
          held = t.m;
          const uint32_t bytes = 2 * (load_a ? 2 * kChunkBytes : kChunkBytes);
          uint32_t a_at = sbase;
          for (int k = 0; k < k_end; k += kBK, a_at += kChunkBytes) {
            if (!bar_wait(s_empty(sr.at), (sr.fills & 1u) ^ 1u)) {
              ok = false;
              break;
            }
            const uint32_t bar = leader_s_full + 8 * sr.at;
            const uint32_t at = sbase + p.s_ring + sr.at * p.s_stage_bytes;
            if (leader) bar_expect_tx(s_full(sr.at), bytes);
            tma_load_2d(at, &maps.table, k, brow, bar);
            if (load_a) tma_load_2d(p.keep_hidden ? a_at : at + kChunkBytes, &maps.hidden, k, hrow, bar);
            sr.next();
          }
        } else if constexpr (!kForward) {
          const int bcol = (int)(t.n * p.bn + rank * (p.bn / 2));
          const uint32_t bytes = 2 * (t.blocks * kChunkBytes + p.bn * kBK);
          const uint32_t b_boxes = p.bn / 64;
          int k = (int)(t.k0 * kBK);
          const int k_end = k + (int)(t.chunks * kBK);
          for (; k < k_end; k += kBK) {
            if (!bar_wait(p_empty(pr.at), (pr.fills & 1u) ^ 1u)) {
              ok = false;
              break;
            }
            const uint32_t bar = leader_p_full + 8 * pr.at;
            uint32_t at = sbase + pr.at * p.p_stage_bytes;
            if (leader) bar_expect_tx(p_full(pr.at), bytes);
            if (t.kind == kHidden) {
              for (uint32_t j = 0; j < b_boxes; ++j, at += 4096)
                tma_load_2d(at, &maps.table_n, bcol + (int)(32 * j), (int)p.pv0 + k, bar);
              tma_load_2d(at, &maps.d_k, k, arow, bar);
              if (t.blocks > 1) tma_load_2d(at + kChunkBytes, &maps.d_k, k, arow + 2 * kBM, bar);
            } else {
              for (uint32_t j = 0; j < b_boxes; ++j, at += 4096)
                tma_load_2d(at, &maps.scaled_n, bcol + (int)(32 * j), k, bar);
              tma_load_2d(at, &maps.d_m, arow, k, bar);
              tma_load_2d(at + 8192, &maps.d_m, arow + 64, k, bar);
              if (t.blocks > 1) {
                tma_load_2d(at + kChunkBytes, &maps.d_m, arow + 2 * kBM, k, bar);
                tma_load_2d(at + kChunkBytes + 8192, &maps.d_m, arow + 2 * kBM + 64, k, bar);
              }
            }
            pr.next();
          }
        }
      }
      if (!ok) *abort_flag = 1u;
      // what is in flight, for the teardown after an abort
      issued[0] = pr.fills * pr.n + pr.at;
      issued[1] = sr.fills * sr.n + sr.at;
    }
  } else if (warp == 1) {
    // ---- MMA issuer (leader CTA only) ----
    if (lane == 0 && leader && !t.done()) {
      // F32 accumulator, A and B of type T, M = 256; bit 15 / 16: A / B not K-major
      constexpr uint32_t kIdesc = (1u << 4) | (Type<T>::kFormat << 7) | (Type<T>::kFormat << 10) |
                                  ((uint32_t)((2 * kBM) >> 4) << 24);
      bool ok = true;
      Ring pr(p.p_stages), sr(p.s_stages);
      uint32_t sub = 0;  // accumulators used so far: buffer sub & 1
      const uint64_t k_major = sw128_desc(sbase);  // + offset / 16: any place of the region
      const uint64_t m_major = mn_desc(sbase, 128), n_major = mn_desc(sbase, 64);
      for (; ok && !t.done() && !*abort_flag; t.next(p)) {
        const uint32_t accs = kHalves && t.kind == kScore ? p.score_accs : t.blocks;
        for (uint32_t j = 0; ok && j < accs; ++j)
          ok = bar_wait(acc_empty((sub + j) & 1u), (((sub + j) >> 1) & 1u) ^ 1u);
        if (!ok) break;
        fence_after();
        const uint32_t acc = tmem + (sub & 1u) * kBN;
        if (t.kind == kScore) {
          constexpr uint32_t idesc = kIdesc | ((uint32_t)(kBN >> 3) << 17);
          uint32_t to = acc, fresh = 0;  // the segment's accumulator and first chunk
          bool ready = bar_test(s_full(sr.at), sr.fills & 1u);
          for (uint32_t kc = 0; kc < t.chunks; ++kc) {
            if (!ready && !bar_wait(s_full(sr.at), sr.fills & 1u)) {
              ok = false;
              break;
            }
            const uint32_t at = sr.at;
            const uint64_t b = k_major + (p.s_ring + at * p.s_stage_bytes) / 16;
            const uint64_t a = p.keep_hidden ? k_major + kc * (kChunkBytes / 16)
                                             : b + kChunkBytes / 16;
            sr.next();
            // asked before the MMAs, whose issue takes as long as they do
            ready = bar_test(s_full(sr.at), sr.fills & 1u);
            if (kHalves && kc == p.seg_chunks) to = tmem + ((sub + 1) & 1u) * kBN, fresh = kc;
#pragma unroll
            for (int k4 = 0; k4 < kBK / 16; ++k4)
              mma_pair(to, a + 2 * k4, b + 2 * k4, idesc, kc != fresh || k4 != 0);
            mma_commit_pair(s_empty(at));  // frees the stage (both CTAs) once read
          }
        } else if constexpr (!kForward) {
          const uint32_t idesc = kIdesc | ((p.bn >> 3) << 17) |
                                 (t.kind == kTable ? 1u << 15 : 0u) | (1u << 16);
          const uint64_t a0 = (t.kind == kTable ? m_major : k_major) + p.bn * kBK / 16;
          const uint32_t a_step = t.kind == kTable ? 2048 / 16 : 2;
          const uint32_t stage = p.p_stage_bytes / 16;
          const uint32_t acc1 = tmem + ((sub + 1) & 1u) * kBN;
          bool ready = bar_test(p_full(pr.at), pr.fills & 1u);
          for (uint32_t kc = 0; kc < t.chunks; ++kc) {
            if (!ready && !bar_wait(p_full(pr.at), pr.fills & 1u)) {
              ok = false;
              break;
            }
            const uint32_t at = pr.at;
            const uint64_t b = n_major + at * stage, a = a0 + at * stage;
            pr.next();
            ready = bar_test(p_full(pr.at), pr.fills & 1u);
#pragma unroll
            for (int k4 = 0; k4 < kBK / 16; ++k4)
              mma_pair(acc, a + a_step * k4, b + 64 * k4, idesc, (kc | (uint32_t)k4) != 0u);
            if (t.blocks > 1) {
#pragma unroll
              for (int k4 = 0; k4 < kBK / 16; ++k4)
                mma_pair(acc1, a + kChunkBytes / 16 + a_step * k4, b + 64 * k4, idesc,
                         (kc | (uint32_t)k4) != 0u);
            }
            mma_commit_pair(p_empty(at));
          }
        }
        if (!ok) break;
        for (uint32_t j = 0; j < accs; ++j) mma_commit_pair(acc_full((sub + j) & 1u));
        sub += accs;
      }
      if (!ok) *abort_flag = 1u;
      mma_commit_local(drain);
      bar_wait(drain, 0);
    }
  } else {
    // ---- epilogue: warp w serves TMEM lanes 32 (w % 4) .. + 31 (one tile row
    // per thread) and column half (w - 2) / 4 ----
    const uint32_t quad = (uint32_t)(warp & 3);
    const uint32_t half = (uint32_t)(warp - 2) >> 2;
    const uint32_t tile_row = rank * kBM + quad * 32 + (uint32_t)lane;
    // this warp's columns of a score tile
    constexpr uint32_t kMine = kHalves ? kBN / 4 : kBN / 2;
    const uint32_t c_begin = (kHalves ? 2 * rank + half : half) * kMine;
    const uint32_t leader_acc_empty0 = mapa(acc_empty(0), 0);
    const uint32_t leader_acc_empty1 = mapa(acc_empty(1), 0);
    const float nan = __uint_as_float(0x7FC00000u);
    const float t2 = w.inv_t * kLog2e;  // of the teacher's logits
    const float c2 = w.inv_t * p.score_scale * kLog2e;
    const float scale = kForward || p.gmax == nullptr ? 1.f : *p.gmax / Type<T>::kScale;  // of d^T H
    bool dead = false;
    // state of the row this thread holds while it walks along score tiles
    uint32_t cur_m = 0xFFFFFFFFu, row = 0, slot = 0;
    bool live = false;
    float top = 0.f, share = 0.f;  // of the teacher
    float run_m = -INFINITY, run_l = 0.f, dot = 0.f, coef = 0.f;
    float run_q = 0.f;             // sum of the q seen
    float2 z2 = make_float2(0.f, 0.f);
    float at_target = 0.f;         // d of cross entropy there
    float e2 = 0.f;                // log2 |coef| - z2
    // of the packed pairs of d; p is at most 1, however far the errors of scores
    // of 1e6 lie beyond lse
    uint32_t most = 0, keep = 0, sign = 0;
    Cursor<kDistill> cur;
    cur.none();
    auto release = [&](uint32_t buf) {  // the accumulator has been read
      fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive_cluster_relaxed(buf ? leader_acc_empty1 : leader_acc_empty0);
    };
    auto flush = [&]() {
      if (kForward && cur_m != 0xFFFFFFFFu && row < p.rows)
        p.partial[(uint64_t)row * p.slots + slot] =
            Partial{dead ? nan : run_m, dead ? nan : run_l, dot, run_q};
    };
    uint32_t sub = 0;
    for (uint32_t block = 0; !t.done(); ++sub) {
      const uint32_t buf = sub & 1u;
      if (t.kind == kScore) {
        const uint32_t v = p.v0 + t.n * kBN + c_begin;
        if (t.m != cur_m) {  // (a score tile has one block)
          flush();
          cur_m = t.m;
          row = t.m * 2 * kBM + (kHalves ? tile_row - rank * kBM : tile_row);
          live = row < p.rows;
          if (kForward) {
            // slot: this pair's place among the pairs that walk row tile m
            const uint64_t x = (uint64_t)t.m * p.n_tiles;
            uint32_t lo = 0, hi = pair;  // first pair whose range reaches x
            while (lo < hi) {
              const uint32_t mid = (lo + hi) / 2;
              if (p.score_at[mid + 1] > x) hi = mid; else lo = mid + 1;
            }
            slot = 2 * (pair - lo) + half;
            run_m = -INFINITY;
            run_l = dot = run_q = 0.f;
          } else if (live) {
            coef = p.rg[row].coef;
            if (!kDistill) at_target = p.rg[row].target;
            z2 = lse_units(p.lse[row]);
            e2 = (log2f(fabsf(coef)) - z2.y) - z2.x;
            most = Type<T>::pack(fabsf(coef), fabsf(coef));
            keep = coef != 0.f ? 0xFFFFFFFFu : 0u;
            sign = coef < 0.f ? 0x80008000u : 0u;
            live = coef != 0.f;
          }
          if (kDistill && live) {
            const Teacher st = w.stat[row];
            live = !stat_empty(st) && !stat_invalid(st);
            top = st.top;
            share = st.share;
          }
          cur.start(w, row, v, live);
          cur.fill(w);
        }
      }
      const bool two = kHalves && t.kind == kScore && p.score_accs == 2;
      if (!dead && (*abort_flag || !bar_wait(acc_full(buf), (sub >> 1) & 1u) ||
                    (two && !bar_wait(acc_full(buf ^ 1u), ((sub + 1) >> 1) & 1u)))) {
        *abort_flag = 1u;
        dead = true;
      }
      fence_after();
      const uint32_t acc = tmem + ((quad * 32u) << 16) + buf * kBN;
      if (t.kind == kScore) {
        cur.skip_to(w, p.v0 + t.n * kBN + c_begin);
        const uint32_t c_end = p.cols - min(p.cols, t.n * kBN);  // columns of the tile that exist
        if constexpr (kHalves) {
#pragma unroll 1
          for (uint32_t c = c_begin; c < c_begin + kMine && c < c_end; c += 32) {
            uint32_t r[32];
            if (!dead) {
              tmem_ld32(acc + c, r);
              if (two) {
                uint32_t x[32];
                tmem_ld32(tmem + ((quad * 32u) << 16) + (buf ^ 1u) * kBN + c, x);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  r[j] = __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(x[j]));
              } else {
                tmem_wait_ld();
              }
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(nan);
            }
            const uint32_t col = p.v0 + t.n * kBN + c;
            T* out = static_cast<T*>(p.d) + (uint64_t)row * p.pitch + t.n * kBN + c;
            T* out_low = out + (uint64_t)p.rows * p.pitch;
            if (row < p.rows) {
              const float2 cc = make_float2(c2, c2), ee = make_float2(e2, e2);
              const float cap = fabsf(coef);
#pragma unroll
              for (int j = 0; j < 32; j += 16) {
                uint32_t v[8], lo[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  const float2 x = fma2(make_float2(__uint_as_float(r[j + 2 * e]),
                                                    __uint_as_float(r[j + 2 * e + 1])), cc, ee);
                  const float a = min_nan(exp2_approx(x.x), cap), b = min_nan(exp2_approx(x.y), cap);
                  v[e] = Type<T>::pack(a, b);
                  const T* h = reinterpret_cast<const T*>(&v[e]);
                  // (the high half of a finite weight is finite)
                  lo[e] = (Type<T>::pack(a - Type<T>::to(h[0]), b - Type<T>::to(h[1])) & keep) ^ sign;
                  v[e] = (v[e] & keep) ^ sign;
                }
                store_v8(out + j, v);
                store_v8(out_low + j, lo);
              }
            }
            // over the elements just stored
            while (__any_sync(0xFFFFFFFFu, cur.id[0] - col < 32u)) {
              const uint32_t i = cur.id[0] - col;
              float x = at_target;
              if constexpr (kDistill) {
                const float s = pick32(r, i);
                x = (min_nan(exp2_approx(fmaf(s, c2, -z2.x) - z2.y), 1.f) -
                     cur.weight(t2, top, share)) * coef;
              }
              if (dead) x = nan;
              const bool mine = i < 32u;
              if (mine) {
                out[i] = Type<T>::from(x);
                out_low[i] = Type<T>::from(x - Type<T>::to(Type<T>::from(x)));
              }
              cur.drop(w, mine);
            }
          }
        } else {
#pragma unroll 1
          for (uint32_t c = c_begin; c < c_begin + kMine; c += 64) {
            if (c >= c_end) break;
            uint32_t r[64];
            if (!dead) {
              tmem_ld64(acc + c, r);
            } else {
#pragma unroll
              for (int j = 0; j < 64; ++j) r[j] = __float_as_uint(nan);
            }
            const uint32_t col = p.v0 + t.n * kBN + c;  // vocabulary id of r[0]
            if constexpr (kForward) {
              if (c + 64 > c_end) {
#pragma unroll
                for (int j = 0; j < 64; ++j)
                  if (c + j >= c_end) r[j] = 0xFF800000u;  // -inf
              }
              float mx[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) mx[j] = __uint_as_float(r[j]);
#pragma unroll
              for (int j = 4; j < 64; j += 8)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (j + 4 + e < 64)
                    mx[e] = fmaxf(fmaxf(mx[e], __uint_as_float(r[j + e])),
                                  __uint_as_float(r[j + 4 + e]));
                  else
                    mx[e] = fmaxf(mx[e], __uint_as_float(r[j + e]));
              const float m =
                  fmaxf(run_m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c2);
              const float from = base_of(m);
              if (kDistill) dot = fmaf(run_q, base_of(run_m) - from, dot);
              float2 l[2] = {make_float2(run_l * exp2_approx(run_m - from), 0.f),
                             make_float2(0.f, 0.f)};
#pragma unroll
              for (int j = 0; j < 64; j += 2) {
                const float2 x = fma2(make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])),
                                      make_float2(c2, c2), make_float2(-from, -from));
                l[(j >> 1) & 1] =
                    add2(l[(j >> 1) & 1], make_float2(exp2_approx(x.x), exp2_approx(x.y)));
              }
              run_m = m;
              l[0] = add2(l[0], l[1]);
              run_l = l[0].x + l[0].y;
              while (__any_sync(0xFFFFFFFFu, cur.id[0] - col < 64u)) {
                const float s = pick64(r, cur.id[0] - col);
                const bool mine = cur.id[0] - col < 64u;
                if (mine) {
                  const float q = cur.weight(t2, top, share);
                  if (!kDistill) {
                    dot = s;
                  } else if (q > 0.f) {
                    dot = fmaf(q, fmaf(s, c2, -from), dot);
                    run_q += q;
                  }
                }
                cur.drop(w, mine);
              }
            } else {
              // |coef| goes into the exponent
              T* out = static_cast<T*>(p.d) + (uint64_t)row * p.pitch + t.n * kBN + c;
              const float2 cc = make_float2(c2, c2), ee = make_float2(e2, e2);
              if (row < p.rows) {
#pragma unroll
                for (int j = 0; j < 64; j += 16) {
                  uint32_t v[8];
#pragma unroll
                  for (int e = 0; e < 8; ++e) {
                    const float2 x = fma2(make_float2(__uint_as_float(r[j + 2 * e]),
                                                      __uint_as_float(r[j + 2 * e + 1])), cc, ee);
                    v[e] = (Type<T>::least(Type<T>::pack(exp2_approx(x.x), exp2_approx(x.y)), most) &
                            keep) ^ sign;
                  }
                  store_v8(out + j, v);
                }
              }
              if constexpr (!kDistill) {  // over the element just stored
                const bool mine = cur.id[0] - col < 64u;
                if (__any_sync(0xFFFFFFFFu, mine)) {
                  if (mine) out[cur.id[0] - col] = Type<T>::from(dead ? nan : at_target);
                  __syncwarp();
                }
              } else {
                while (__any_sync(0xFFFFFFFFu, cur.id[0] - col < 64u)) {
                  const float s = pick64(r, cur.id[0] - col);
                  const bool mine = cur.id[0] - col < 64u;
                  if (mine) {  // p - q in FP32
                    const float x = min_nan(exp2_approx(fmaf(s, c2, -z2.x) - z2.y), 1.f) -
                                    cur.weight(t2, top, share);
                    out[cur.id[0] - col] = Type<T>::from(x * coef);
                  }
                  cur.drop(w, mine);
                }
              }
            }
          }
        }
      } else if constexpr (!kForward) {
        const uint32_t c_half = p.bn / 2;
        const uint32_t m_row = (t.m + block) * 2 * kBM + tile_row;
        const bool mine = m_row < (t.kind == kHidden ? p.d_rows : p.pcols);
        const uint64_t at = ((uint64_t)(t.kind == kHidden ? t.split : 0u) * p.d_rows + m_row) * p.width;
#pragma unroll 1
        for (uint32_t c = 0; c < c_half; c += 64) {
          uint32_t r[2][32];
          const bool two = c + 32 < c_half;
          if (!dead) {
            tmem_ld32(acc + half * c_half + c, r[0]);
            if (two) tmem_ld32(acc + half * c_half + c + 32, r[1]);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) r[0][j] = r[1][j] = __float_as_uint(nan);
          }
          if (c + 64 >= c_half) release(buf);  // before the last stores
#pragma unroll
          for (uint32_t q = 0; q < 2; ++q) {
            const uint32_t col = t.n * p.bn + half * c_half + c + 32 * q;
            if ((q && !two) || !mine || col >= p.width) continue;
            const uint32_t n = min(4u, (p.width - col) / 8);  // groups of 8 that exist
            if (t.kind == kHidden) {
              float* out = p.planes + at + col;
              if (p.add) {  // one addition to each element a launch: the order is fixed
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j)
                  if (j < 2 * n) add_v4(out + 4 * j, r[q] + 4 * j);
              } else {
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j)
                  if (j < n) store_v8(out + 8 * j, r[q] + 8 * j);
              }
            } else {
              T* out = static_cast<T*>(p.table_out) + at + col;
              uint32_t v[16];
#pragma unroll
              for (int j = 0; j < 16; ++j)
                v[j] = Type<T>::pack(__uint_as_float(r[q][2 * j]) * scale,
                                     __uint_as_float(r[q][2 * j + 1]) * scale);
              if (p.wide_rows) {  // rows start on 32 bytes, and hold a multiple of that
#pragma unroll
                for (uint32_t j = 0; j < 4; j += 2)
                  if (j < n) store_v8(out + 8 * j, v + 4 * j);
              } else {
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j)
                  if (j < n)
                    *reinterpret_cast<uint4*>(out + 8 * j) =
                        make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
              }
            }
          }
        }
        if (++block == t.blocks) {
          block = 0;
          t.next(p);
        }
        continue;
      }
      release(buf);
      if (two) {
        release(buf ^ 1u);
        ++sub;
      }
      cur.fill(w);  // loads that the next tile waits for, not this one
      t.next(p);
    }
    flush();
  }

  // ---- teardown: drain the producers' copies, free TMEM ----
  __syncthreads();
  if (*abort_flag && threadIdx.x == 0) {
    if (leader) {  // wait (bounded) for the last copy issued into each stage
      for (uint32_t st = 0; st < kMaxStages; ++st) {
        if (issued[0] > st && st < p.p_stages)
          bar_wait(p_full(st), ((issued[0] - st - 1u) / p.p_stages) & 1u);
        if (issued[1] > st && st < p.s_stages)
          bar_wait(s_full(st), ((issued[1] - st - 1u) / p.s_stages) & 1u);
      }
    } else {
      // the peer's copies complete on the leader's barriers: give any still
      // in flight 1 ms (a copy of this GPU's memory takes microseconds)
      const uint64_t t0 = global_ns();
      while (global_ns() - t0 < 1000000ull) __nanosleep(10000);
    }
  }
  fence_before();
  cluster_sync();  // no CTA frees TMEM or exits while its pair may still touch it
  fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(kTmemCols)
                 : "memory");
}

// Joins the (m, l) of the lanes of a warp.
__device__ __forceinline__ void warp_join(float& m, float& l) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float om = __shfl_xor_sync(0xFFFFFFFFu, m, o), ol = __shfl_xor_sync(0xFFFFFFFFu, l, o);
    const float mn = fmaxf(m, om);
    l = l * (m == mn ? 1.f : exp2_approx(m - mn)) + ol * (om == mn ? 1.f : exp2_approx(om - mn));
    m = mn;
  }
}
__device__ __forceinline__ void join(float& m, float& l, float2 q) {
  const float mn = fmaxf(m, q.x);
  // a walk without a column has l = 0 at m = -inf
  l = l * (m == mn ? 1.f : exp2_approx(m - mn)) + q.y * (q.x == mn ? 1.f : exp2_approx(q.x - mn));
  m = mn;
}

// Joins a row's slots over the lanes of a warp; the loads of 160 slots (a call
// has at most 148 a row, but for few column tiles of many rows) are in flight
// together.  `local` (or NULL): the largest logit of each slot's entries, which
// its q are relative to.
__device__ __forceinline__ void join_slots(const Partial* part, const float* local, uint32_t slots,
                                           const Teacher& st, float inv_t, float& m, float& l,
                                           float& dot) {
  const uint32_t lane = threadIdx.x & 31;
  m = -INFINITY;
  l = dot = 0.f;
  float sum_q = 0.f;
  for (uint32_t s0 = lane; s0 < slots; s0 += 160) {
    float4 q[5];
    float t[5];
#pragma unroll
    for (uint32_t j = 0; j < 5; ++j) {
      const uint32_t i = s0 + 32 * j;
      q[j] = i < slots ? *reinterpret_cast<const float4*>(part + i)
                       : make_float4(-INFINITY, 0.f, 0.f, 0.f);
      t[j] = local && i < slots ? local[i] : -INFINITY;
    }
    if (local) {
#pragma unroll
      for (int j = 0; j < 5; ++j) {
        const float by = t[j] > -INFINITY ? expf((t[j] - st.top) * inv_t) * st.share : 0.f;
        q[j].z = by > 0.f ? q[j].z * by : 0.f;
        q[j].w *= by;
      }
    }
    float top = fmaxf(fmaxf(fmaxf(q[0].x, q[1].x), fmaxf(q[2].x, q[3].x)), q[4].x);
    top = fmaxf(top, m);
    // a walk without a column has l = 0 at m = -inf
    float sum = m == top ? l : l * exp2_approx(m - top);
    dot = fmaf(sum_q, base_of(m) - base_of(top), dot);
#pragma unroll
    for (int j = 0; j < 5; ++j) {
      sum += q[j].x == top ? q[j].y : q[j].y * exp2_approx(q[j].x - top);
      dot += fmaf(q[j].w, base_of(q[j].x) - base_of(top), q[j].z);
      sum_q += q[j].w;
    }
    m = top;
    l = sum;
  }
  const float mine = base_of(m);
  warp_join(m, l);
  dot = fmaf(sum_q, mine - base_of(m), dot);
#pragma unroll
  for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, o);
}

// T^2 (sum q log q + log l - dot): the scores' size cancels before it comes in.
__device__ __forceinline__ float set_loss(const Wanted& w, const Teacher& s, float l, float dot) {
  const float t = 1.f / w.inv_t;
  if (stat_empty(s)) return 0.f;
  if (stat_invalid(s) || !(l > 0.f)) return __uint_as_float(0x7FC00000u);
  return t * t * (s.entropy + (log2f(l) - dot) * kLn2);
}
// Of a row without a target: ignored or invalid.
__device__ __forceinline__ float no_target_loss(uint32_t target) {
  return target == kInvalid ? 0.f : __uint_as_float(0x7FC00000u);
}

// The target's score `dot` as it came from the tensor core (c2: its scale, in
// units of ln 2) leaves a row's sum (m, l), where it is exp2(dot c2 - m), and
// `score` from the FP32 pipes takes its place.  Returns
// the loss: ln of the sum over the target's term, which lse's rounding does not
// reach.  The two scores may lie further apart than an exponential's range
// (scores of 1e8).
__device__ __forceinline__ float put_target(float& m, float& l, float dot, float c2,
                                            float score) {
  if (m == -INFINITY) return __uint_as_float(0x7FC00000u);  // no score but -inf: lse stays so
  float rest = l - exp2_approx(fmaf(dot, c2, -m));
  if (rest < 0.f) rest = 0.f;  // rounding; a NaN stays
  const float above = fmaf(score, kLog2e, -m);
  if (above > 0.f || rest == 0.f) {  // the target is the largest
    l = 1.f + (rest == 0.f ? 0.f : rest * exp2_approx(-above));
    m += above;
    return log2f(l) * kLn2;
  }
  l = rest + exp2_approx(above);
  return (log2f(l) - above) * kLn2;
}

// A sure row's lse is score + loss, rounded once: the gradient takes p - 1 from
// the distance of the two.
__device__ __forceinline__ float row_lse(float m, float l, float score, float loss) {
  return loss < 1.f ? score + loss : lse_of(m, l);
}

// One warp per row joins the walks' partial sums.  Row tile m's n_tiles tiles
// lie in the ranges of a few consecutive pairs.  A target's score is computed
// again on the FP32 pipes and takes the place of the tensor core's in the sum:
// a loss is a difference of two numbers that a sure row has nearly equal.
template <typename T>
__global__ void merge_kernel(Wanted w, const T* hidden, const T* table, uint32_t width,
                             const Partial* part, uint32_t row_slots, uint32_t n_tiles,
                             uint32_t total, uint32_t pairs, uint32_t rows, uint32_t vocab,
                             float c2, float* losses, float* lse) {
  const uint32_t r = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  if (r >= rows) return;
  const uint32_t target = w.targets ? w.targets[r] : kInvalid;
  float score = 0.f;
  if (target < vocab)
    score = warp_score(hidden + (uint64_t)r * width, table + (uint64_t)target * width, width);
  pdl_wait();  // what came before was not written by the previous kernel
  pdl_trigger();
  const uint64_t x0 = (uint64_t)(r / (2 * kBM)) * n_tiles, x1 = x0 + n_tiles - 1;
  // range of pair i: [total i / pairs, total (i + 1) / pairs)
  const uint32_t first = (uint32_t)(((x0 + 1) * pairs - 1) / total);
  const uint32_t last = (uint32_t)(((x1 + 1) * pairs - 1) / total);
  const uint32_t slots = 2 * (last - first + 1);
  float m, l, dot;
  const Teacher st = w.targets ? Teacher{} : w.stat[r];
  join_slots(part + (uint64_t)r * row_slots, nullptr, slots, st, w.inv_t, m, l, dot);
  if (lane) return;
  float loss = no_target_loss(target);
  if (target < vocab) loss = put_target(m, l, dot, c2, score);
  lse[r] = target < vocab ? row_lse(m, l, score, loss) : lse_of(m, l);
  losses[r] = w.targets ? loss : set_loss(w, st, l, dot);
}

// ---- few rows ------------------------------------------------------------
//
// Up to 64 rows: reading the table bounds the call.  The table takes the M side:
// each CTA (one per SM) streams its own range of table rows once through a deep
// ring (128 rows x 64 K a stage, fetched 32 rows at a time so that ranges are
// even to 32 rows), against the hidden rows, which stay in shared memory (N =
// rows rounded up to 16).  All its scores fit in TMEM, so the softmax needs no
// running maximum: one pass for each row's maximum over the CTA's range, one
// for the sum.  TMEM that is left holds each score in up to three segments of its
// products, added in FP32 (distillation: as many as the gradients' kernel makes).
// Cross entropy: the target's score comes from the FP32 pipes in the join, in place
// of the tensor core's.  Distillation: the entries in the CTA's range are listed and
// weighed while the table streams; their scores are those of TMEM, the same numbers
// that lse and the gradients are made of, laid out in shared memory for any thread
// to read.
// Measured (49,152 x 576, fp16, table from DRAM): 13.9 us for 1 row (4.1 TB/s; a
// read of the table alone takes 8.6 us at 6.55 TB/s), against 24.6 us with the tile
// engine; the join adds 1.4 us.  Sets of 32 and 300 entries add 0.8 us for 1 row and
// 1 and 3 us for 64 (19.7).
constexpr uint32_t kFewRows = 64;
constexpr uint32_t kFewMaxStages = 12;
constexpr uint32_t kFewThreads = 192;  // producer, MMA issuer, 4 epilogue warps
constexpr uint32_t kFewSmem = 222 * 1024;
constexpr uint32_t kFewEntries = 2048;       // of a teacher's sets, listed at a time
constexpr uint32_t kFewListBytes = kFewEntries * 8;

struct FewParams {
  uint32_t rows, n;         // n: rows rounded up to 16
  uint32_t vocab, range;    // table rows per CTA, a multiple of 32
  uint32_t w_chunks, stages;
  uint32_t segments, seg_chunks;  // accumulators of a score, chunks in each
  float c2;                 // score scale / T in units of ln 2
  uint32_t entries;         // of the teacher's sets
  Partial* partial;         // [rows][CTA]; dot: the target's, where it is in the range
  float* local;             // distillation: [rows][CTA], what q in dot is relative to
};

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  tmem_wait_ld();
}

__device__ __forceinline__ float tmem_ld1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr));
  tmem_wait_ld();
  return __uint_as_float(r);
}

__device__ __forceinline__ float warp_max(float v) {
  float m;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}

template <typename T, bool kDistill>
__global__ void __launch_bounds__(kFewThreads, 1)
few_rows_kernel(const __grid_constant__ CUtensorMap tm_hidden,
                const __grid_constant__ CUtensorMap tm_table, const FewParams p, const Wanted w) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t bars[2 * kFewMaxStages + 2];
  __shared__ uint32_t tmem_at, abort_word, filled;
  __shared__ float2 part[4][kFewRows];
  __shared__ float s_dot[kFewRows];
  __shared__ int32_t s_at[kDistill ? 2 * kFewRows : 1];  // first entries in the range and behind it
  __shared__ uint32_t s_first[kDistill ? kFewRows + 1 : 1];  // their places in the list
  const uint32_t hid = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t hid_chunk = p.n * 128;
  const uint32_t ring = hid + ((p.w_chunks * hid_chunk + 1023u) & ~1023u);
  const uint32_t bar0 = smem_u32(bars);
  auto full = [&](uint32_t st) { return bar0 + 8 * st; };
  auto empty = [&](uint32_t st) { return bar0 + 8 * (kFewMaxStages + st); };
  const uint32_t h_full = bar0 + 8 * (2 * kFewMaxStages), done = h_full + 8;
  volatile uint32_t* abort_flag = &abort_word;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t v0 = blockIdx.x * p.range;
  const uint32_t count = min(p.range, p.vocab - v0);  // table rows of this CTA
  const uint32_t tiles = (count + 127) / 128;
  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < 2 * kFewMaxStages + 2; ++i) bar_init(bar0 + 8 * i, 1);
    abort_word = 0u;
    filled = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&tmem_at)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_at;
  pdl_wait();  // what the previous kernel wrote, before any bounded wait begins
  pdl_trigger();

  if (warp == 0) {
    if (lane == 0) {
      Ring rg(p.stages);
      bool ok = true;
      bar_expect_tx(h_full, p.w_chunks * hid_chunk);
      for (uint32_t kc = 0; kc < p.w_chunks; ++kc)
        tma_load_local(hid + kc * hid_chunk, &tm_hidden, (int)(kc * kBK), 0, h_full);
      for (uint32_t t = 0; ok && t < tiles; ++t) {
        const uint32_t boxes = min(4u, (count - t * 128 + 31) / 32);
        for (uint32_t kc = 0; kc < p.w_chunks; ++kc) {
          if (!bar_wait(empty(rg.at), (rg.fills & 1u) ^ 1u)) {
            ok = false;
            break;
          }
          bar_expect_tx(full(rg.at), boxes * 4096);
          for (uint32_t j = 0; j < boxes; ++j)
            tma_load_local(ring + rg.at * kChunkBytes + j * 4096, &tm_table, (int)(kc * kBK),
                           (int)(v0 + t * 128 + 32 * j), full(rg.at));
          rg.next();
        }
      }
      if (!ok) *abort_flag = 1u;
      filled = rg.fills * rg.n + rg.at;
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // F32 accumulator, A and B of type T, K-major, M = 128
      const uint32_t idesc = (1u << 4) | (Type<T>::kFormat << 7) | (Type<T>::kFormat << 10) |
                             ((p.n >> 3) << 17) | (8u << 24);
      Ring rg(p.stages);
      bool ok = bar_wait(h_full, 0);
      for (uint32_t t = 0; ok && t < tiles; ++t) {
        uint32_t acc = tmem + t * p.segments * p.n, seg_end = p.seg_chunks;
        for (uint32_t kc = 0; kc < p.w_chunks; ++kc) {
          if (!bar_wait(full(rg.at), rg.fills & 1u)) {
            ok = false;
            break;
          }
          fence_after();
          const uint64_t a = sw128_desc(ring + rg.at * kChunkBytes);
          const uint64_t b = sw128_desc(hid + kc * hid_chunk);
          if (kc == seg_end) acc += p.n, seg_end += p.seg_chunks;
          const bool add = kc + p.seg_chunks != seg_end;
#pragma unroll
          for (int k4 = 0; k4 < kBK / 16; ++k4)
            mma_one(acc, a + 2 * k4, b + 2 * k4, idesc, add || k4 != 0);
          mma_commit_one(empty(rg.at));
          rg.next();
        }
      }
      if (!ok) *abort_flag = 1u;
      mma_commit_one(done);  // everything issued, whether or not all of it was
      bar_wait(done, 0);
    }
  } else {
    const uint32_t quad = warp & 3, e = threadIdx.x - 64;
    auto together = [] {  // the epilogue warps
      __syncwarp();
      asm volatile("bar.sync 1, 128;" ::: "memory");
    };
    uint32_t target[2];  // of rows lane and lane + 32, from v0 on; the warp's own, if any
    uint32_t listed = 0;  // entries in the range, row after row
    // list of the entries in the range, row after row: place in the range, or
    // none; logit, then weight
    uint32_t* list = reinterpret_cast<uint32_t*>(smem_raw + (ring - smem_u32(smem_raw)) +
                                                 p.stages * kChunkBytes);
    float* list_t = reinterpret_cast<float*>(list + kFewEntries);
    auto fill = [&](uint32_t from) {
#pragma unroll 4
      for (uint32_t i = e; i < kFewEntries && from + i < listed; i += 128) {
        uint32_t r = 0;  // the last row that begins at or before the entry
#pragma unroll
        for (uint32_t step = kFewRows / 2; step > 0; step >>= 1)
          if (s_first[r + step] <= from + i) r += step;
        const int32_t k = s_at[r] + (int32_t)(from + i - s_first[r]);
        const uint32_t v = (uint32_t)w.ids[k] - v0;
        list[i] = v < count ? v : kInvalid;  // ids of an invalid set lie anywhere
        list_t[i] = v < count ? w.logits[k] : -INFINITY;
      }
    };
    // Distillation: 2 to 8 neighbouring threads share a row's entries.
    const uint32_t share = p.n <= 16 ? 8u : (p.n <= 32 ? 4u : 2u);
    const uint32_t r_mine = kDistill ? e / share : e, sub = kDistill ? e % share : 0u;
    const bool mine = r_mine < p.rows;
    float dot = 0.f, sum_q = 0.f, top = -INFINITY;  // weights relative to `top`
    uint32_t begin = 0, end = 0;                    // of the row, in the list
    // The listed logits of a row become weights.
    auto weigh = [&](uint32_t from) {
      begin = end = 0;
      if (mine) {
        begin = max(s_first[r_mine], from) - from + sub;
        end = min(max(s_first[r_mine + 1], from) - from, kFewEntries);
      }
      float most = top;
      for (uint32_t i = begin; i < end; i += share) most = fmaxf(most, list_t[i]);
      for (uint32_t o = 1; o < share; o <<= 1)
        most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
      if (most > top) {
        const float by = expf((top - most) * w.inv_t);
        sum_q *= by;
        dot = by > 0.f ? dot * by : 0.f;  // an infinite score that no longer counts
        top = most;
      }
      for (uint32_t i = begin; i < end; i += share) {
        const float t = list_t[i], q = t > -INFINITY ? expf((t - top) * w.inv_t) : 0.f;
        list_t[i] = q;
        sum_q += q;
      }
    };
    if constexpr (kDistill) {
      const uint32_t r = e & (kFewRows - 1);
      int32_t at = 0;
      if (r < p.rows) {
        const int32_t a = w.offsets[r], b = w.offsets[r + 1];
        if (a >= 0 && b >= a && (uint32_t)b <= p.entries)
          at = first_entry_of_8(w.ids, a, b, e < kFewRows ? v0 : v0 + count);
      }
      s_at[e] = at;
      together();
      if (warp == 2) {
        uint32_t n[2], sum[2];
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
          // an ascending set has at most one entry a table row; an invalid one is cut
          n[i] = min(count, (uint32_t)max(0, s_at[kFewRows + 32 * i + lane] - s_at[32 * i + lane]));
          sum[i] = n[i];
          for (uint32_t o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xFFFFFFFFu, sum[i], o);
            if (lane >= o) sum[i] += x;
          }
        }
        const uint32_t half = __shfl_sync(0xFFFFFFFFu, sum[0], 31);
        s_first[lane] = sum[0] - n[0];
        s_first[lane + 32] = half + sum[1] - n[1];
        if (lane == 31) s_first[kFewRows] = half + sum[1];
      }
      together();
      listed = s_first[kFewRows];
      fill(0);
      together();
      weigh(0);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t r = lane + 32 * i;
        target[i] = r < p.rows ? w.targets[r] - v0 : kInvalid;
        if (target[i] >= count || ((target[i] >> 5) & 3u) != quad) target[i] = kInvalid;
        if (warp == 2) s_dot[r] = 0.f;
      }
    }
    together();
    const bool ok = bar_wait(done, 0) && !*abort_flag;
    fence_after();
    const uint32_t acc = tmem + ((quad * 32u) << 16);
    auto scores = [&](uint32_t t, uint32_t c, uint32_t (&r)[16]) {  // the segments' sum
      tmem_ld16(acc + t * p.segments * p.n + c, r);
      for (uint32_t g = 1; g < p.segments; ++g) {
        uint32_t x[16];
        tmem_ld16(acc + (t * p.segments + g) * p.n + c, x);
#pragma unroll
        for (int j = 0; j < 16; ++j)
          r[j] = __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(x[j]));
      }
    };
    // Distillation: the ring, which nothing uses any more, takes the scores of as
    // many tiles as it holds, on the way of the sums; rows padded by one for the banks.
    float* dense = reinterpret_cast<float*>(smem_raw + (ring - smem_u32(smem_raw)));
    const uint32_t pitch = p.n + 1, held = p.stages * kChunkBytes / (512u * pitch);
    auto keep = [&](uint32_t t, uint32_t c, const uint32_t (&r)[16]) {
      float* at = dense + (t * 128 + quad * 32 + lane) * pitch + c;
#pragma unroll
      for (int j = 0; j < 16; ++j) at[j] = __uint_as_float(r[j]);
    };
    const uint32_t kept = listed > 0 ? held : 0;
    for (uint32_t c = 0; c < p.n; c += 16) {
      float mx[16], l[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) mx[j] = -INFINITY, l[j] = 0.f;
      for (uint32_t t = 0; t < tiles; ++t) {
        uint32_t r[16];
        scores(t, c, r);
        const bool in = t * 128 + quad * 32 + lane < count;
#pragma unroll
        for (int j = 0; j < 16; ++j) mx[j] = fmaxf(mx[j], in ? __uint_as_float(r[j]) : -INFINITY);
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        mx[j] = warp_max(mx[j]) * p.c2;
        l[j] = mx[j] < kMasked ? 0.f : mx[j];  // a warp without a table row sums zeros
      }
      float sum[16] = {};
      for (uint32_t t = 0; t < tiles; ++t) {
        uint32_t r[16];
        scores(t, c, r);
        if constexpr (kDistill)
          if (t < kept) keep(t, c, r);
        const bool in = t * 128 + quad * 32 + lane < count;
#pragma unroll
        for (int j = 0; j < 16; ++j)
          sum[j] += in ? exp2_approx(fmaf(__uint_as_float(r[j]), p.c2, -l[j])) : 0.f;
      }
      // add over the lanes, halving the columns a lane keeps: lane x ends with
      // column x / 2
#pragma unroll
      for (int h = 8, o = 16; h > 0; h >>= 1, o >>= 1) {
        const bool up = lane & (uint32_t)o;
#pragma unroll
        for (int j = 0; j < h; ++j) {
          const float give = up ? sum[j] : sum[j + h];
          const float keep = up ? sum[j + h] : sum[j];
          sum[j] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, o);
          mx[j] = up ? mx[j + h] : mx[j];
        }
      }
      sum[0] += __shfl_xor_sync(0xFFFFFFFFu, sum[0], 1);
      if ((lane & 1u) == 0)
        part[quad][c + lane / 2] = make_float2(mx[0], ok ? sum[0] : __uint_as_float(0x7FC00000u));
    }
    if constexpr (!kDistill) {
      // the targets' scores: of all rows' targets, few lie in one CTA's range
#pragma unroll
      for (uint32_t i = 0; i < 2; ++i)
        for (uint32_t todo = __ballot_sync(0xFFFFFFFFu, target[i] != kInvalid); todo; todo &= todo - 1) {
          const uint32_t from = __ffs(todo) - 1;
          const uint32_t v = __shfl_sync(0xFFFFFFFFu, target[i], from), c = from + 32 * i;
          float x = 0.f;
          for (uint32_t g = 0; g < p.segments; ++g)
            x += tmem_ld1(acc + ((v / 128) * p.segments + g) * p.n + c);
          if (lane == (v & 31u)) s_dot[c] = x;
        }
    }
    fence_before();
    together();
    float m = -INFINITY, l = 0.f;  // of the row
    if (mine)
#pragma unroll
      for (int q = 0; q < 4; ++q) join(m, l, part[q][r_mine]);
    if constexpr (!kDistill) {
      if (mine) dot = s_dot[r_mine];
    } else if (listed > 0) {
      const float base = base_of(m);
      for (uint32_t from = 0;;) {
        uint32_t i = begin;
        for (uint32_t t0 = 0; t0 < tiles; t0 += held) {
          if (held < tiles && (t0 > 0 || from > 0)) {
            together();
            for (uint32_t t = t0; t < min(tiles, t0 + held); ++t)
              for (uint32_t c = 0; c < p.n; c += 16) {
                uint32_t r[16];
                scores(t, c, r);
                keep(t - t0, c, r);
              }
            together();
          }
          // a valid set ascends; of an invalid one what lies elsewhere is left out
          for (; i < end; i += share) {
            const uint32_t v = list[i];
            if (v != kInvalid && v >= (t0 + held) * 128) break;
            const float q = list_t[i];
            if (q > 0.f && v >= t0 * 128)
              dot = fmaf(q, fmaf(dense[(v - t0 * 128) * pitch + r_mine], p.c2, -base), dot);
          }
        }
        if (listed - from <= kFewEntries) break;
        from += kFewEntries;
        together();
        fill(from);
        together();
        weigh(from);
      }
      for (uint32_t o = 1; o < share; o <<= 1) {
        dot += __shfl_xor_sync(0xFFFFFFFFu, dot, o);
        sum_q += __shfl_xor_sync(0xFFFFFFFFu, sum_q, o);
      }
    }
    if (mine && sub == 0) {
      const uint64_t at = (uint64_t)r_mine * gridDim.x + blockIdx.x;
      p.partial[at] = Partial{m, l, dot, sum_q};
      if (kDistill) p.local[at] = top;
    }
  }
  __syncthreads();
  if (abort_word != 0u && threadIdx.x == 0) {  // copies in flight, bounded
    bar_wait(h_full, 0);
    for (uint32_t st = 0; st < p.stages; ++st)
      if (filled > st) bar_wait(full(st), ((filled - st - 1u) / p.stages) & 1u);
  }
  __syncthreads();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(kTmemCols)
                 : "memory");
}

// Gradients for up to 32 rows, in one pass over the table: each CTA takes its
// range of table rows, 128 at a time.  The tile's rows stay in shared memory for
// both products that read them, and with so few rows each element of d is
// carried as a sum of two 16-bit numbers, which costs no memory traffic:
//   S^T = E H^T     [128, n]      A = table tile (K-major), B = hidden (K-major)
//   d^T in FP32 -> high and low halves, [128, 32 high | 32 low] in shared memory
//   d H^T += E^T d  [width, n]    A = table tile (M-major), B = d (N-major)
//   dE = d^T H      [128, width]  A = d (K-major), B = hidden (N-major)
// d H^T stays in TMEM over the CTA's tiles and leaves as one FP32 plane per CTA;
// dE leaves 128 columns at a time.  What bounds it is one read of the table and
// one write of its gradient: 17.4 us for 49,152 x 576 at 6.55 TB/s; measured 34
// us for 1 row and 42 us for 32 (66 us with the tile engine and its four
// launches), the rest being the chain of each of the three tiles of a CTA.
constexpr uint32_t kFewGradRows = 32;
constexpr uint32_t kFewGradChunks = 10;   // widths up to 640
constexpr uint32_t kFewGradThreads = 320;
constexpr uint32_t kDBytes = 128 * 128;   // d: 128 table rows x (32 high, 32 low)

struct FewGradParams {
  uint32_t rows, n;         // n: rows rounded up to 16
  uint32_t width, w_chunks;
  uint32_t vocab, range;    // table rows per CTA, a multiple of 32
  uint32_t segments, seg_chunks;  // as forward
  float c2;
  const void *hidden, *table;
  const float* grad;
  const float* lse;
  RowGrad* rg;
  float* planes;            // [CTA][rows][width], or NULL
  void* table_out;          // d_embedding, or NULL
  uint32_t wide_rows;
};

// Shared-memory descriptor, M or N contiguous, 128-byte swizzle: atoms of 64
// elements `lbo` bytes apart, groups of 8 K rows 1024 bytes apart.
__device__ __forceinline__ uint64_t mn128_desc(uint32_t addr, uint32_t lbo) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | (uint64_t)(lbo >> 4) << 16 |
         (uint64_t)(1024u >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
                 "=r"(r[7])
               : "r"(taddr));
  tmem_wait_ld();
}
__device__ __forceinline__ void bar_arrive_local(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void epilogue_sync() {  // the eight epilogue warps
  asm volatile("bar.sync 1, 256;" ::: "memory");
}

template <typename T, bool kDistill>
__global__ void __launch_bounds__(kFewGradThreads, 1)
few_rows_grad_kernel(const __grid_constant__ CUtensorMap tm_table, const FewGradParams p, Wanted w) {
  extern __shared__ unsigned char smem_raw[];
  // table chunks full, table free, scores full, d full, dE full / empty [2], dH done
  __shared__ uint64_t bars[kFewGradChunks + 8];
  __shared__ uint32_t tmem_at, abort_word, loads;
  __shared__ float s_coef[kFewGradRows];
  __shared__ float2 s_z2[kFewGradRows];
  __shared__ float s_top[kFewGradRows], s_share[kFewGradRows];
  __shared__ uint32_t s_target[kFewGradRows];
  __shared__ float s_short[kFewGradRows];  // p - 1 of the targets in the CTA's range
  __shared__ int32_t s_at[kFewGradRows], s_end[kFewGradRows];
  __shared__ float s_gmax;
  unsigned char* sm = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t tab = smem_u32(sm);
  const uint32_t hid_chunk = p.n * 128;
  const uint32_t hid = tab + p.w_chunks * kChunkBytes;
  const uint32_t dt = hid + p.w_chunks * hid_chunk;
  float* s_q = reinterpret_cast<float*>(sm + (dt - tab) + kDBytes);  // distillation: [n][128]
  const uint32_t bar0 = smem_u32(bars);
  auto e_full = [&](uint32_t kc) { return bar0 + 8 * kc; };
  const uint32_t e_free = bar0 + 8 * kFewGradChunks, s_full = e_free + 8, d_full = e_free + 16;
  auto de_full = [&](uint32_t b) { return e_free + 24 + 8 * b; };
  auto de_empty = [&](uint32_t b) { return e_free + 40 + 8 * b; };
  const uint32_t done = e_free + 56;
  volatile uint32_t* abort_flag = &abort_word;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t v0 = blockIdx.x * p.range;
  const uint32_t count = min(p.range, p.vocab - v0);
  const uint32_t tiles = (count + 127) / 128;
  const uint32_t passes = (p.w_chunks + 1) / 2;  // of 128 columns of dE
  const uint32_t blocks = (p.w_chunks + 1) / 2;  // of 128 rows of d H^T
  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < kFewGradChunks + 8; ++i)
      bar_init(bar0 + 8 * i, bar0 + 8 * i == d_full || bar0 + 8 * i == de_empty(0) ||
                                     bar0 + 8 * i == de_empty(1) ? 8u : 1u);
    abort_word = 0u;
    loads = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&tmem_at)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();
  pdl_trigger();
  __syncthreads();  // barriers initialised
  auto load_tile = [&](uint32_t t) {
    for (uint32_t kc = 0; kc < p.w_chunks; ++kc) {
      bar_expect_tx(e_full(kc), kChunkBytes);
      tma_load_local(tab + kc * kChunkBytes, &tm_table, (int)(kc * kBK), (int)(v0 + t * 128),
                     e_full(kc));
    }
    loads = t + 1;
  };
  if (threadIdx.x == 32) load_tile(0);  // under the set-up
  if (warp == 0) {  // row weights: |weight| / largest, all of it carried by d
    const float wr = lane < p.rows ? row_weight(w, p.grad, lane, p.vocab) : 0.f;
    const float a = fabsf(wr);
    const float g = warp_max(a < INFINITY ? a : 0.f);
    const float coef = wr != 0.f ? wr / g * Type<T>::kScale : 0.f;
    s_coef[lane] = coef;
    s_z2[lane] = lse_units(lane < p.rows ? p.lse[lane] : 0.f);
    s_target[lane] = w.targets && lane < p.rows && coef != 0.f ? w.targets[lane] : kInvalid;
    if (lane == 0) s_gmax = g;
    if (blockIdx.x == 0 && lane < p.rows) p.rg[lane] = RowGrad{coef, g / Type<T>::kScale, 0.f};
    if (kDistill) {
      s_at[lane] = s_end[lane] = 0;
      if (coef != 0.f) {
        s_top[lane] = w.stat[lane].top;
        s_share[lane] = w.stat[lane].share;
        s_at[lane] = first_entry(w, lane, v0);
        s_end[lane] = w.offsets[lane + 1];
      }
    }
  }
  __syncthreads();
  if (!kDistill) {
    for (uint32_t r = warp; r < p.rows; r += kFewGradThreads / 32) {
      if (s_target[r] - v0 >= count) continue;
      const float x = target_short(static_cast<const T*>(p.hidden), static_cast<const T*>(p.table), r,
                                   s_target[r], p.width, p.lse[r]);
      if (lane == 0) s_short[r] = x;
    }
  }
  // hidden rows as 64-wide chunks of 128-byte rows (128-byte swizzle); rows that
  // take no part are zero
  for (uint32_t i = threadIdx.x; i < p.w_chunks * p.n * 8; i += kFewGradThreads) {
    const uint32_t j = i & 7u, r = (i >> 3) % p.n, kc = (i >> 3) / p.n, c = kc * kBK + j * 8;
    uint4 x = make_uint4(0u, 0u, 0u, 0u);
    if (s_coef[r] != 0.f && c < p.width)
      x = ld_v4(static_cast<const T*>(p.hidden) + (uint64_t)r * p.width + c);
    *reinterpret_cast<uint4*>(sm + (hid - tab) + kc * hid_chunk + r * 128 + ((j ^ (r & 7u)) << 4)) = x;
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_at;
  // TMEM columns: d H^T [blocks x n], scores [segments x n], dE [2 x 128]
  const uint32_t acc_h = tmem, acc_s = tmem + blocks * p.n, acc_e = tmem + 256;

  if (warp == 0) {
    if (lane == 0) {
      for (uint32_t t = 1; t < tiles && !*abort_flag; ++t) {
        if (!bar_wait(e_free, (t & 1u) ^ 1u)) {
          *abort_flag = 1u;
          break;
        }
        load_tile(t);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t kIdesc = (1u << 4) | (Type<T>::kFormat << 7) | (Type<T>::kFormat << 10) |
                                  (8u << 24);  // F32 accumulator, type T, M = 128
      const uint32_t idesc_s = kIdesc | ((p.n >> 3) << 17);
      const uint32_t idesc_h = idesc_s | (1u << 15) | (1u << 16);
      const uint32_t idesc_e = kIdesc | ((128u >> 3) << 17) | (1u << 16);
      bool ok = true;
      uint32_t pass = 0;  // dE buffers used so far
      for (uint32_t t = 0; ok && t < tiles && !*abort_flag; ++t) {
        uint32_t acc = acc_s, seg_end = p.seg_chunks;
        for (uint32_t kc = 0; ok && kc < p.w_chunks; ++kc) {
          ok = bar_wait(e_full(kc), t & 1u);
          if (!ok) break;
          const uint64_t a = sw128_desc(tab + kc * kChunkBytes), b = sw128_desc(hid + kc * hid_chunk);
          if (kc == seg_end) acc += p.n, seg_end += p.seg_chunks;
          const bool add = kc + p.seg_chunks != seg_end;
#pragma unroll
          for (int k4 = 0; k4 < kBK / 16; ++k4)
            mma_one(acc, a + 2 * k4, b + 2 * k4, idesc_s, add || k4 != 0);
        }
        if (!ok) break;
        mma_commit_one(s_full);
        ok = bar_wait(d_full, t & 1u);
        if (!ok) break;
        fence_after();
        // two passes of dE first: the epilogue drains them under d H^T
        uint32_t j = 0;
        auto table_pass = [&]() {
          const uint32_t buf = pass & 1u;
          ok = bar_wait(de_empty(buf), ((pass >> 1) & 1u) ^ 1u);
          if (!ok) return;
          fence_after();
          for (uint32_t k = 0; k < p.n / 16; ++k) {
            const uint64_t b = mn128_desc(hid + 2 * j * hid_chunk + 2048 * k, hid_chunk);
            mma_one(acc_e + buf * 128, sw128_desc(dt + 32 * k), b, idesc_e, k != 0u);
            mma_one(acc_e + buf * 128, sw128_desc(dt + 64 + 32 * k), b, idesc_e, 1u);
          }
          mma_commit_one(de_full(buf));
          ++j;
          ++pass;
        };
        const uint32_t n_pass = p.table_out ? passes : 0;
        while (ok && j < 2 && j < n_pass) table_pass();
        if (!ok) break;
        if (p.planes) {
          for (uint32_t b = 0; b < blocks; ++b)
#pragma unroll 2
            for (uint32_t k = 0; k < 8; ++k) {  // 16 table rows
              const uint64_t a = mn128_desc(tab + 2 * b * kChunkBytes + 2048 * k, kChunkBytes);
              const uint32_t d = dt + 2048 * k;
              mma_one(acc_h + b * p.n, a, mn128_desc(d, 1024), idesc_h, (t | k) != 0u);
              mma_one(acc_h + b * p.n, a, mn128_desc(d + 64, 1024), idesc_h, 1u);
            }
        }
        mma_commit_one(e_free);  // the table tile has been read
        while (ok && j < n_pass) table_pass();
      }
      if (!ok) *abort_flag = 1u;
      mma_commit_one(done);
      bar_wait(done, 0);
    }
  } else {
    const uint32_t quad = warp & 3u, half = (warp - 2) >> 2;
    const uint32_t lanes = (quad * 32u) << 16;
    const uint32_t row = quad * 32 + lane;  // of the tile
    const float c2 = p.c2, t2 = w.inv_t * kLog2e;
    const float scale = s_gmax / Type<T>::kScale;
    const float nan = __uint_as_float(0x7FC00000u);
    bool dead = false;
    auto wait = [&](uint32_t bar, uint32_t parity) {
      if (!dead && (*abort_flag || !bar_wait(bar, parity))) {
        *abort_flag = 1u;
        dead = true;
      }
      fence_after();
    };
    uint32_t pass = 0;
    for (uint32_t t = 0; t < tiles; ++t) {
      const uint32_t v = v0 + t * 128 + row;
      const bool in = t * 128 + row < count;
      if (kDistill) {  // the tile's entries, dense
        epilogue_sync();  // the tile before has been read
        for (uint32_t i = threadIdx.x - 64; i < p.n * 128; i += 256) s_q[i] = 0.f;
        epilogue_sync();
        const uint32_t first = v0 + t * 128, n_in = min(128u, count - t * 128);
        for (uint32_t r = warp - 2; r < p.rows; r += 8) {
          int32_t k = s_at[r];
          const int32_t end = s_end[r];
          for (;;) {
            uint32_t id = 0xFFFFFFFFu;
            if (k + (int32_t)lane < end) id = (uint32_t)w.ids[k + lane];
            const bool mine = id - first < n_in;  // ascending: entries before `first` are behind k
            if (mine)
              s_q[r * 128 + (id - first)] = exp2_approx((w.logits[k + lane] - s_top[r]) * t2) * s_share[r];
            const uint32_t taken = __popc(__ballot_sync(0xFFFFFFFFu, mine));
            k += (int32_t)taken;
            if (taken < 32) break;
          }
          __syncwarp();
          if (lane == 0) s_at[r] = k;
        }
        epilogue_sync();
      }
      wait(s_full, t & 1u);
      for (uint32_t c = half * (p.n / 2); c < (half + 1) * (p.n / 2); c += 8) {
        uint32_t r[8];
        tmem_ld8(acc_s + lanes + c, r);
        for (uint32_t g = 1; g < p.segments; ++g) {
          uint32_t x[8];
          tmem_ld8(acc_s + lanes + g * p.n + c, x);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            r[j] = __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(x[j]));
        }
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          float x[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t n = c + j + e;
            const float coef = s_coef[n];
            const float2 z2 = s_z2[n];
            float d = min_nan(exp2_approx(fmaf(__uint_as_float(r[j + e]), c2, -z2.x) - z2.y), 1.f);
            if (kDistill) d -= s_q[n * 128 + row];
            else if (s_target[n] == v) d = s_short[n];
            x[e] = coef == 0.f || !in ? 0.f : (dead ? nan : d * coef);
          }
          hi[j / 2] = Type<T>::pack(x[0], x[1]);
          const T* h = reinterpret_cast<const T*>(&hi[j / 2]);
          // a high half beyond the type's range stays alone
          const float l0 = x[0] - Type<T>::to(h[0]), l1 = x[1] - Type<T>::to(h[1]);
          lo[j / 2] = Type<T>::pack(fabsf(l0) < INFINITY ? l0 : 0.f, fabsf(l1) < INFINITY ? l1 : 0.f);
        }
        unsigned char* at = sm + (dt - tab) + row * 128;
        *reinterpret_cast<uint4*>(at + (((c / 8) ^ (row & 7u)) << 4)) =
            make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(at + (((4 + c / 8) ^ (row & 7u)) << 4)) =
            make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive_local(d_full);
      for (uint32_t j = 0; p.table_out && j < passes; ++j, ++pass) {
        const uint32_t buf = pass & 1u;
        wait(de_full(buf), (pass >> 1) & 1u);
        uint32_t r[2][32];
        tmem_ld32(acc_e + lanes + buf * 128 + half * 64, r[0]);
        tmem_ld32(acc_e + lanes + buf * 128 + half * 64 + 32, r[1]);
        tmem_wait_ld();
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive_relaxed_local(de_empty(buf));
        if (!in) continue;
#pragma unroll
        for (uint32_t q = 0; q < 2; ++q) {
          const uint32_t col = j * 128 + half * 64 + 32 * q;
          if (col >= p.width) continue;
          const uint32_t groups = min(4u, (p.width - col) / 8);
          T* out = static_cast<T*>(p.table_out) + (uint64_t)v * p.width + col;
          const float by = dead ? nan : scale;
          uint32_t x[16];
#pragma unroll
          for (int i = 0; i < 16; ++i)
            x[i] = Type<T>::pack(__uint_as_float(r[q][2 * i]) * by,
                                 __uint_as_float(r[q][2 * i + 1]) * by);
          if (p.wide_rows) {
#pragma unroll
            for (uint32_t i = 0; i < 4; i += 2)
              if (i < groups) store_v8(out + 8 * i, x + 4 * i);
          } else {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
              if (i < groups)
                *reinterpret_cast<uint4*>(out + 8 * i) =
                    make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
          }
        }
      }
    }
    if (p.planes) {
      wait(done, 0);
      float* out = p.planes + (uint64_t)blockIdx.x * p.rows * p.width;
      for (uint32_t b = 0; b < blocks; ++b) {
        const uint32_t c = b * 128 + row;  // column of d_hidden
        for (uint32_t n = half * (p.n / 2); n < (half + 1) * (p.n / 2); n += 8) {
          uint32_t r[8];
          tmem_ld8(acc_h + lanes + b * p.n + n, r);
#pragma unroll
          for (uint32_t j = 0; j < 8; ++j)
            if (n + j < p.rows && c < p.width)
              out[(uint64_t)(n + j) * p.width + c] = dead ? nan : __uint_as_float(r[j]);
        }
      }
    }
    fence_before();
  }
  __syncthreads();
  if (abort_word != 0u && threadIdx.x == 0 && loads > 0u)  // copies in flight, bounded
    for (uint32_t kc = 0; kc < p.w_chunks; ++kc) bar_wait(e_full(kc), (loads - 1u) & 1u);
  __syncthreads();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(kTmemCols)
                 : "memory");
}

// One warp per row, a block each: the CTAs' sums, the target's score, the
// teacher's distribution.
template <typename T>
__global__ void __launch_bounds__(32)
few_rows_join_kernel(Wanted w, const T* hidden, const T* table, uint32_t width, const Partial* part,
                     const float* local, uint32_t slots, uint32_t entries, uint32_t vocab, float c2,
                     float* losses, float* lse) {
  const uint32_t r = blockIdx.x;
  const uint32_t target = w.targets ? w.targets[r] : kInvalid;
  Teacher st{};
  float score = 0.f;
  // The inputs were complete before this kernel could start: every kernel here
  // lets the next one start only after its own wait for the one before.
  if (target < vocab)
    score = warp_score(hidden + (uint64_t)r * width, table + (uint64_t)target * width, width);
  else if (w.offsets)
    st = teacher_stat(w, r, entries, vocab);
  pdl_wait();
  pdl_trigger();
  float m, l, dot;
  join_slots(part + (uint64_t)r * slots, w.offsets ? local + (uint64_t)r * slots : nullptr, slots, st,
             w.inv_t, m, l, dot);
  if (threadIdx.x) return;
  float loss = no_target_loss(target);
  if (target < vocab) loss = put_target(m, l, dot, c2, score);
  lse[r] = target < vocab ? row_lse(m, l, score, loss) : lse_of(m, l);
  losses[r] = w.targets ? loss : set_loss(w, st, l, dot);
}

// d_hidden: the splits' sums in a fixed order, scaled and rounded; four columns
// a thread, and with many splits eight threads for the same columns, each with
// every eighth split.
constexpr uint32_t kFinishThreads = 256;
template <typename T, uint32_t kGroups>
__global__ void __launch_bounds__(kFinishThreads)
finish_kernel(const float* planes, uint32_t splits, const RowGrad* rg, T* out, uint32_t rows,
              uint32_t width) {
  constexpr uint32_t kColumns = kFinishThreads / kGroups;
  __shared__ float4 part[kGroups][kColumns];
  const uint32_t c = threadIdx.x % kColumns, group = threadIdx.x / kColumns;
  const uint64_t i = ((uint64_t)blockIdx.x * kColumns + c) * 4;
  const uint64_t n = (uint64_t)rows * width;
  pdl_wait();
  pdl_trigger();
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (i < n) {
#pragma unroll 4
    for (uint32_t s = group; s < splits; s += kGroups) {
      const float4 a = __ldcg(reinterpret_cast<const float4*>(planes + s * n + i));
      v = make_float4(v.x + a.x, v.y + a.y, v.z + a.z, v.w + a.w);
    }
  }
  if (kGroups > 1) {
    part[group][c] = v;
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (uint32_t g = 1; g < kGroups; ++g) {
      const float4 a = part[g][c];
      v = make_float4(v.x + a.x, v.y + a.y, v.z + a.z, v.w + a.w);
    }
  }
  if (i >= n) return;
  const RowGrad g = rg[(uint32_t)(i / width)];
  const bool in = g.coef != 0.f;
  *reinterpret_cast<uint2*>(out + i) =
      make_uint2(Type<T>::pack(in ? v.x * g.scale : 0.f, in ? v.y * g.scale : 0.f),
                 Type<T>::pack(in ? v.z * g.scale : 0.f, in ? v.w * g.scale : 0.f));
}

// ---- host --------------------------------------------------------------

mf_status ok() { return mf_status{MF_OK, 0}; }
mf_status fail(int32_t code, uint32_t detail = 0) { return mf_status{code, detail}; }

uint64_t round_up(uint64_t x, uint64_t to) { return (x + to - 1) / to * to; }

struct Span {
  const void* p;
  uint64_t bytes;
};

// Whether one of `outs` overlaps another buffer (NULL buffers overlap nothing).
bool outputs_overlap(std::initializer_list<Span> outs, std::initializer_list<Span> ins) {
  auto hit = [](const Span& a, const Span& b) {
    if (a.p == nullptr || b.p == nullptr) return false;
    const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
    return x < y + b.bytes && y < x + a.bytes;
  };
  for (const Span* a = outs.begin(); a != outs.end(); ++a) {
    for (const Span* b = a + 1; b != outs.end(); ++b)
      if (hit(*a, *b)) return true;
    for (const Span& b : ins)
      if (hit(*a, b)) return true;
  }
  return false;
}

bool sizes_ok(uint64_t rows, uint64_t width, uint64_t vocab) {
  return rows != 0 && rows <= MF_LOSS_MAX_ROWS && width != 0 && width % 8 == 0 &&
         width <= MF_LOSS_MAX_HIDDEN && vocab != 0 && vocab <= MF_LOSS_MAX_VOCAB;
}

struct ForwardPlan {
  uint64_t m_tiles, n_tiles, slots, stat, partial, local, bytes;
  ForwardPlan(uint64_t rows, uint64_t vocab) {
    m_tiles = (rows + 2 * kBM - 1) / (2 * kBM);
    n_tiles = (vocab + kBN - 1) / kBN;
    // pairs that share a row tile: its n_tiles tiles lie in ranges of at least
    // floor(m n / pairs) tiles
    uint64_t per = m_tiles * n_tiles / kMaxPairs;
    if (per < 1) per = 1;
    slots = (n_tiles + per - 1) / per + 1;
    if (slots > n_tiles) slots = n_tiles;
    // the few-rows kernel: one slot per CTA
    if (rows <= kFewRows && slots < kMaxPairs) slots = kMaxPairs;
    stat = 0;
    partial = round_up(rows * sizeof(Teacher), 256);
    local = partial + 2 * slots * rows * sizeof(Partial);
    bytes = round_up(local + (rows <= kFewRows ? 2 * kMaxPairs * rows * sizeof(float) : 0), 256);
  }
};

struct BackwardPlan {
  uint64_t m_tiles, stat, rg, gmax, scaled, planes, piece[2], bytes;
  uint32_t halves;        // of d: 2 where both fit the one row tile
  uint32_t cols, pieces;  // vocabulary rows of one piece
  uint32_t bn, bn_tiles;  // product tiles along the hidden width
  uint32_t blocks;        // row blocks that share a product tile's B
  uint32_t splits, per_split;
  uint32_t sets;          // pieces with planes of their own
  BackwardPlan(uint64_t rows, uint64_t width, uint64_t vocab) {
    // decided by the number of row tiles, so that within one the bytes grow
    // with the rows
    m_tiles = (rows + 2 * kBM - 1) / (2 * kBM);
    const uint64_t all_rows = m_tiles * 2 * kBM;
    // Up to 64 rows d is carried as the sum of two 16-bit numbers, the low halves in
    // rows of their own of the one row tile (with the same hidden rows beside them,
    // and sums that the last kernel adds): gradients keep what their type holds. With
    // one 16-bit number a gradient is 1.4 times as far off as its own rounding makes
    // it, and with few rows, whose errors do not average, up to 2.3 times. 49,152 x
    // 576: 33 rows 57 and 63 us, 64 rows 58 and 65; 128 rows, where it is not done,
    // would take 73 in place of 62.
    halves = rows <= kHalvesRows ? 2 : 1;
    const uint64_t d_rows = rows * halves;
    uint64_t c = kPieceBytes / (2 * all_rows) / kBN * kBN;
    if (c < kBN) c = kBN;
    pieces = (uint32_t)((vocab + c - 1) / c);
    cols = (uint32_t)round_up((vocab + pieces - 1) / pieces, kBN);
    pieces = (uint32_t)((vocab + cols - 1) / cols);
    bn_tiles = (uint32_t)((width + kBN - 1) / kBN);
    bn = (uint32_t)round_up((width + bn_tiles - 1) / bn_tiles, 64);
    // d E is split along the piece so that no tile is longer than half a
    // pair's share of the two products, or the whole share where score tiles
    // fill the rest (a split costs a plane of sums: 4,096 x 49,152 x 576
    // backward 603 us with half, 558 with the whole, 580 with two)
    const uint64_t chunks = ((cols < vocab ? cols : vocab) + kBK - 1) / kBK;
    const uint64_t total = bn_tiles * (m_tiles * chunks + (cols + 2 * kBM - 1) / (2 * kBM) *
                                                              (all_rows / kBK));
    uint64_t most = total / kMaxPairs / (pieces > 1 ? 1 : 2);
    if (most < 4) most = 4;
    // Two 256-row blocks a tile read B once (backward, us, one block and two:
    // 2,000 x 49,152 x 576 350 and 322, 4,096 rows 717 and 608, 1,001 x 32,003 x
    // 328 100 and 91, 512 x 49,152 x 576 109 and 104), but leave no accumulator
    // to drain into, which short K does not repay, and waste half a tile of an
    // odd few (600 x 20,000 x 1,024, three row tiles: 95 and 114)
    blocks = all_rows >= 8 * kBK && most >= 32 && (m_tiles % 2 == 0 || m_tiles >= 8) ? 2 : 1;
    if (blocks == 2) most /= 2;
    splits = (uint32_t)((chunks + most - 1) / most);
    per_split = (uint32_t)((chunks + splits - 1) / splits);
    splits = (uint32_t)((chunks + per_split - 1) / per_split);
    // Sums kept apart cost a store a piece and are joined at the end; adding at
    // L2 from this layout (a row a thread) made a launch 25 us longer at 8,192 rows
    const uint64_t set = (uint64_t)splits * d_rows * width * 4;
    sets = (uint32_t)(kPieceBytes / ((uint64_t)splits * all_rows * width * 4));
    if (sets > pieces) sets = pieces;
    if (sets < 1) sets = 1;
    stat = 0;
    rg = round_up(stat + rows * sizeof(Teacher), 256);
    gmax = round_up(rg + rows * sizeof(RowGrad), 256);
    scaled = gmax + 256;
    planes = round_up(scaled + d_rows * width * 2, 256);
    uint64_t sums = sets * set;
    const uint64_t few = 2 * kMaxPairs * rows * width * 4;  // few_rows_grad_kernel's planes
    if (rows <= kFewGradRows && width <= kFewGradChunks * kBK && sums < few) sums = few;
    piece[0] = round_up(planes + sums, 256);
    const uint64_t one = round_up(d_rows * cols * 2, 256);
    piece[1] = piece[0] + (pieces > 1 ? one : 0);
    bytes = piece[1] + one;
  }
};

// What a batch of at most `rows` rows needs: the most that any needs.  Within a
// row tile, and up to each of `few` rows, a plan's bytes grow with the rows.
template <typename F>
uint64_t most_bytes(uint64_t rows, std::initializer_list<uint64_t> few, F bytes) {
  uint64_t most = bytes(rows);
  auto at = [&](uint64_t r) {
    if (r < rows && bytes(r) > most) most = bytes(r);
  };
  for (uint64_t r : few) at(r);
  for (uint64_t r = 2 * kBM; r < rows; r += 2 * kBM) at(r);
  return most;
}

// The checks that all calls share; `wanted` gives the rows' targets or sets.
mf_status check(uint64_t rows, uint64_t width, uint64_t vocab, void* stream, Span hidden,
                Span embedding, std::initializer_list<Span> row_f32, Span workspace,
                uint64_t needed, bool distill, Span targets, Span ids, Span logits,
                float temperature) {
  if (rows == 0 || width == 0 || vocab == 0 || stream == nullptr)
    return fail(MF_INVALID_ARGUMENT);
  if (distill) {
    const float inv = 1.f / temperature, sq = temperature * temperature;
    if (!(temperature > 0.f) || !std::isfinite(temperature) || !std::isfinite(inv) ||
        !std::isfinite(sq) || !(sq > 0.f))
      return fail(MF_INVALID_ARGUMENT);
  }
  if (!sizes_ok(rows, width, vocab)) return fail(MF_RESOURCE_LIMIT);
  if (hidden.p == nullptr || hidden.bytes != rows * width * 2 || embedding.p == nullptr ||
      embedding.bytes != vocab * width * 2 || workspace.p == nullptr || workspace.bytes < needed ||
      (uintptr_t)hidden.p % 16 != 0 || (uintptr_t)embedding.p % 16 != 0 ||
      (uintptr_t)workspace.p % 256 != 0)
    return fail(MF_INVALID_ARGUMENT);
  for (const Span& s : row_f32)
    if (s.p == nullptr || s.bytes != rows * 4 || (uintptr_t)s.p % 4 != 0)
      return fail(MF_INVALID_ARGUMENT);
  if (targets.p == nullptr || targets.bytes != (rows + (distill ? 1 : 0)) * 4 ||
      (uintptr_t)targets.p % 4 != 0)
    return fail(MF_INVALID_ARGUMENT);
  if (distill) {
    if (ids.bytes % 4 != 0 || ids.bytes != logits.bytes || (uintptr_t)ids.p % 4 != 0 ||
        (uintptr_t)logits.p % 4 != 0 || (ids.bytes != 0 && (ids.p == nullptr || logits.p == nullptr)))
      return fail(MF_INVALID_ARGUMENT);
    if (ids.bytes / 4 > MF_LOSS_MAX_ENTRIES) return fail(MF_RESOURCE_LIMIT);
  }
  return ok();
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static std::once_flag once;
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  });
  return fn;
}

// 2-D tensor map over 16-bit [rows, cols] with `pitch` columns from row to row,
// boxes of 64 columns (128-byte swizzle) or 32 (64-byte swizzle).
template <typename T>
bool make_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t pitch,
              uint32_t box_cols, uint32_t box_rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {cols, rows};
  const cuuint64_t strides[1] = {pitch * 2};
  const cuuint32_t box[2] = {box_cols, box_rows};
  const cuuint32_t elem[2] = {1, 1};
  return fn(map, Type<T>::kMap, 2, const_cast<void*>(base), dims, strides, box, elem,
            CU_TENSOR_MAP_INTERLEAVE_NONE,
            box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Sets the kernel's shared-memory limit (once per device) and returns how
// many CTA pairs can be resident at once, at most kMaxPairs.
template <typename T, bool kForward, bool kDistill, bool kHalves>
cudaError_t resident_pairs(uint32_t* pairs) {
  static std::mutex mu;
  static uint32_t cached[64] = {};
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lock(mu);
  uint32_t& c = cached[dev & 63];
  if (c == 0) {
    auto kernel = engine_kernel<T, kForward, kDistill, kHalves>;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(sms & ~1), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = kSmemBytes;
    int clusters = 0;
    e = cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg);
    if (e != cudaSuccess) return e;
    uint32_t n = clusters < 1 ? 1u : (uint32_t)clusters;
    if (n > (uint32_t)sms / 2) n = (uint32_t)sms / 2;
    c = n > kMaxPairs ? kMaxPairs : n;
  }
  *pairs = c;
  return cudaSuccess;
}

// A launch that may begin while the previous kernel on the stream drains: every
// kernel waits for it before it reads what it wrote or writes anything, and
// lets its own successor begin only after that wait.
template <typename... P, typename... A>
cudaError_t launch_after(void (*kernel)(P...), uint64_t blocks, unsigned threads, size_t smem,
                         cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// What both directions' engine launches share.
template <typename T>
Params base_params(uint64_t rows, uint64_t width, uint64_t vocab) {
  Params p = {};
  p.rows = (uint32_t)rows;
  p.width = (uint32_t)width;
  p.vocab = (uint32_t)vocab;
  p.m_tiles = (uint32_t)((rows + 2 * kBM - 1) / (2 * kBM));
  p.w_chunks = (uint32_t)((width + kBK - 1) / kBK);
  p.keep_hidden = p.w_chunks >= 5 && p.w_chunks <= 9;
  p.s_ring = p.keep_hidden ? p.w_chunks * kChunkBytes : 0;
  p.s_stage_bytes = (p.keep_hidden ? 1 : 2) * kChunkBytes;
  p.s_stages = (kRingBytes - p.s_ring) / p.s_stage_bytes;
  if (p.s_stages > kMaxStages) p.s_stages = kMaxStages;
  if (p.keep_hidden && p.s_stages > p.w_chunks) p.s_stages = p.w_chunks;
  p.p_stages = 1;
  p.score_scale = 1.f + (float)width * Type<T>::kLostPerProduct;
  return p;
}

// Deals n tiles of cost c to the pairs, each getting a contiguous range, so
// that the loads (which include earlier deals) come out level.
void deal(uint32_t n, double c, uint32_t pairs, double* load, uint32_t* at) {
  uint32_t count[kMaxPairs] = {}, order[kMaxPairs];
  double part[kMaxPairs] = {};
  double sum = n * c;
  for (uint32_t i = 0; i < pairs; ++i) sum += load[i];
  // the common level; pairs already above it get nothing
  bool out[kMaxPairs] = {};
  uint32_t in = pairs;
  for (bool again = n > 0; again;) {
    again = false;
    for (uint32_t i = 0; i < pairs; ++i)
      if (!out[i] && load[i] * in > sum && in > 1) {
        out[i] = again = true;
        sum -= load[i];
        --in;
      }
  }
  uint32_t dealt = 0, m = 0;
  for (uint32_t i = 0; i < pairs && n > 0; ++i) {
    if (out[i]) continue;
    part[i] = (sum / in - load[i]) / c;
    if (part[i] < 0) part[i] = 0;
    count[i] = (uint32_t)part[i];
    if (count[i] > n - dealt) count[i] = n - dealt;
    dealt += count[i];
    part[i] -= count[i];
    order[m++] = i;
  }
  // what rounding left over, one each
  std::sort(order, order + m, [&](uint32_t x, uint32_t y) {
    return part[x] != part[y] ? part[x] > part[y] : x < y;
  });
  for (uint32_t i = 0; dealt < n; i = i + 1 < m ? i + 1 : 0, ++dealt) ++count[order[i]];
  at[0] = 0;
  for (uint32_t i = 0; i < pairs; ++i) {
    at[i + 1] = at[i] + count[i];
    load[i] += count[i] * c;
  }
}

mf_status launched(cudaError_t e) {
  return e == cudaSuccess ? ok() : fail(MF_CUDA_BACKEND_FAILURE, (uint32_t)e);
}

cudaError_t teacher_launch(const Wanted& w, uint64_t rows, uint64_t entries, uint64_t vocab,
                           cudaStream_t s) {
  const uint64_t blocks = (rows + 7) / 8;
  return launch_after(teacher_kernel, blocks < 1184 ? blocks : 1184, 256, 0, s, w,
                      (uint32_t)rows, (uint32_t)entries, (uint32_t)vocab);
}

// SMs of the current device, at most twice kMaxPairs (the workspace's slots).
cudaError_t device_sms(uint32_t* sms) {
  static std::mutex mu;
  static uint32_t cached[64] = {};
  int dev = 0, n = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lock(mu);
  uint32_t& c = cached[dev & 63];
  if (c == 0) {
    e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    for (const void* k : {(const void*)few_rows_kernel<__half, false>,
                          (const void*)few_rows_kernel<__half, true>,
                          (const void*)few_rows_kernel<__nv_bfloat16, false>,
                          (const void*)few_rows_kernel<__nv_bfloat16, true>,
                          (const void*)few_rows_grad_kernel<__half, false>,
                          (const void*)few_rows_grad_kernel<__half, true>,
                          (const void*)few_rows_grad_kernel<__nv_bfloat16, false>,
                          (const void*)few_rows_grad_kernel<__nv_bfloat16, true>})
      if (e == cudaSuccess)
        e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kFewSmem);
    if (e != cudaSuccess) return e;
    c = (uint32_t)n < 2 * kMaxPairs ? (uint32_t)n : 2 * kMaxPairs;
  }
  *sms = c;
  return cudaSuccess;
}

// How the few-rows gradients take a call; smem 0: they do not.
struct FewGradPlan {
  uint32_t n, range, ctas, segments, seg_chunks;
  uint64_t smem = 0;
  FewGradPlan(uint64_t rows, uint64_t width, uint64_t vocab, uint64_t sms, bool distill) {
    const uint32_t chunks = (uint32_t)((width + kBK - 1) / kBK);
    if (rows > kFewGradRows || chunks > kFewGradChunks) return;
    n = (uint32_t)round_up(rows, 16);
    range = (uint32_t)round_up((vocab + sms - 1) / sms, 32);
    ctas = (uint32_t)((vocab + range - 1) / range);
    // as many segments of a score's products as TMEM holds here (beside d H^T, below
    // the 256 columns of dE) and in the forward kernel
    segments = (256 - (chunks + 1) / 2 * n) / n;
    const uint32_t forward = kTmemCols / ((range + 127) / 128 * n);
    if (segments > forward) segments = forward < 1 ? 1 : forward;
    if (segments > 3) segments = 3;
    seg_chunks = (chunks + segments - 1) / segments;
    segments = (chunks + seg_chunks - 1) / seg_chunks;
    const uint64_t bytes =
        chunks * (kChunkBytes + n * 128) + kDBytes + (distill ? n * 512 : 0) + 1024;
    if (bytes <= kFewSmem) smem = bytes;
  }
};

// How the few-rows forward kernel takes a call; stages 0: it does not.
struct FewPlan {
  uint32_t n, range, ctas, segments, seg_chunks, stages = 0;
  uint64_t smem;
  FewPlan(uint64_t rows, uint64_t width, uint64_t vocab, uint64_t sms, bool distill) {
    if (rows > kFewRows) return;
    n = (uint32_t)round_up(rows, 16);
    range = (uint32_t)round_up((vocab + sms - 1) / sms, 32);
    ctas = (uint32_t)((vocab + range - 1) / range);
    const uint32_t columns = (range + 127) / 128 * n;
    if (columns > kTmemCols) return;  // scores beyond TMEM
    const uint32_t chunks = (uint32_t)((width + kBK - 1) / kBK);
    // distillation: the scores that the gradients will have (two segments where the
    // tile engine makes them)
    const FewGradPlan grad(rows, width, vocab, sms, distill);
    segments = kTmemCols / columns < 3 ? kTmemCols / columns : 3;
    if (distill && grad.smem > 0) segments = grad.segments;
    else if (distill && segments > 2) segments = 2;
    seg_chunks = (chunks + segments - 1) / segments;
    segments = (chunks + seg_chunks - 1) / seg_chunks;
    const uint64_t hid = round_up((width + kBK - 1) / kBK * n * 128, 1024);
    const uint64_t rest = hid + 1024 + (distill ? kFewListBytes : 0);
    if (rest + 4 * kChunkBytes > kFewSmem) return;  // no room for a ring
    const uint64_t room = (kFewSmem - rest) / kChunkBytes;
    stages = (uint32_t)(room < kFewMaxStages ? room : kFewMaxStages);
    smem = rest + stages * kChunkBytes;
  }
};

// 1 / T and the correction of scores summed in segments, in units of ln 2.
template <typename T>
float few_scale(float inv_t, uint32_t segments, uint32_t seg_chunks, uint64_t width) {
  const uint64_t products = segments == 1 ? width : seg_chunks * kBK;
  return inv_t * (1.f + (float)products * Type<T>::kLostPerProduct) * kLog2e;
}

template <typename T, bool kDistill>
mf_status forward_few(const FewPlan& few, Wanted w, const T* hidden, const T* table, uint64_t entries,
                      void* partial, void* local, float* losses, float* lse, uint64_t rows,
                      uint64_t width, uint64_t vocab, cudaStream_t s) {
  CUtensorMap tm_h, tm_t;
  if (!make_map<T>(&tm_h, hidden, rows, width, width, kBK, few.n) ||
      !make_map<T>(&tm_t, table, vocab, width, width, kBK, 32))
    return fail(MF_CUDA_RUNTIME_FAILURE);
  FewParams p = {};
  p.rows = (uint32_t)rows;
  p.n = few.n;
  p.vocab = (uint32_t)vocab;
  p.range = few.range;
  p.w_chunks = (uint32_t)((width + kBK - 1) / kBK);
  p.stages = few.stages;
  p.segments = few.segments;
  p.seg_chunks = few.seg_chunks;
  p.c2 = few_scale<T>(w.inv_t, few.segments, few.seg_chunks, width);
  p.entries = (uint32_t)entries;
  p.partial = static_cast<Partial*>(partial);
  p.local = static_cast<float*>(local);
  cudaError_t e = launch_after(few_rows_kernel<T, kDistill>, few.ctas, kFewThreads, few.smem, s, tm_h,
                               tm_t, p, w);
  if (e == cudaSuccess)
    e = launch_after(few_rows_join_kernel<T>, rows, 32, 0, s, w, hidden, table, (uint32_t)width,
                     static_cast<const Partial*>(p.partial), static_cast<const float*>(p.local),
                     few.ctas, p.entries, p.vocab, p.c2, losses, lse);
  return launched(e);
}

template <typename T, bool kDistill>
mf_status forward(Span hidden, Span embedding, Span targets, Span ids, Span logits,
                  float temperature, Span losses, Span lse, Span workspace, uint64_t rows,
                  uint64_t width, uint64_t vocab, void* stream) {
  const uint64_t needed = sizes_ok(rows, width, vocab) ? ForwardPlan(rows, vocab).bytes : 0;
  mf_status st = check(rows, width, vocab, stream, hidden, embedding, {losses, lse}, workspace,
                       needed, kDistill, targets, ids, logits, temperature);
  if (st.code != MF_OK) return st;
  if (outputs_overlap({losses, lse, workspace}, {hidden, embedding, targets, ids, logits}))
    return fail(MF_INVALID_ARGUMENT);
  const ForwardPlan plan(rows, vocab);
  char* ws = static_cast<char*>(const_cast<void*>(workspace.p));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  Wanted w{};
  w.inv_t = kDistill ? 1.f / temperature : 1.f;
  if (kDistill) {
    w.offsets = static_cast<const int32_t*>(targets.p);
    w.ids = static_cast<const int32_t*>(ids.p);
    w.logits = static_cast<const float*>(logits.p);
    w.stat = reinterpret_cast<Teacher*>(ws + plan.stat);
  } else {
    w.targets = static_cast<const uint32_t*>(targets.p);
  }
  uint32_t sms = 0;
  cudaError_t e = device_sms(&sms);
  if (e != cudaSuccess) return fail(MF_CUDA_RUNTIME_FAILURE, (uint32_t)e);
  const FewPlan few(rows, width, vocab, sms, kDistill);
  if (few.stages > 0)
    return forward_few<T, kDistill>(few, w, static_cast<const T*>(hidden.p),
                          static_cast<const T*>(embedding.p), ids.bytes / 4, ws + plan.partial,
                          ws + plan.local,
                          static_cast<float*>(const_cast<void*>(losses.p)),
                          static_cast<float*>(const_cast<void*>(lse.p)), rows, width, vocab, s);
  uint32_t pairs = 0;
  e = resident_pairs<T, true, kDistill, false>(&pairs);
  if (e != cudaSuccess) return fail(MF_CUDA_RUNTIME_FAILURE, (uint32_t)e);
  Maps maps = {};
  if (!make_map<T>(&maps.hidden, hidden.p, rows, width, width, kBK, kBM) ||
      !make_map<T>(&maps.table, embedding.p, vocab, width, width, kBK, kBN / 2))
    return fail(MF_CUDA_RUNTIME_FAILURE);
  if (kDistill) {
    e = teacher_launch(w, rows, ids.bytes / 4, vocab, s);
    if (e != cudaSuccess) return launched(e);
  }
  const uint64_t total = plan.m_tiles * plan.n_tiles;
  if (pairs > total) pairs = (uint32_t)total;
  Params p = base_params<T>(rows, width, vocab);
  p.cols = (uint32_t)vocab;
  p.n_tiles = (uint32_t)plan.n_tiles;
  p.partial = reinterpret_cast<Partial*>(ws + plan.partial);
  p.slots = (uint32_t)(2 * plan.slots);
  for (uint32_t i = 0; i <= pairs; ++i) p.score_at[i] = (uint32_t)(total * i / pairs);
  e = launch_after(engine_kernel<T, true, kDistill, false>, 2 * pairs, kThreads, kSmemBytes, s,
                   maps, p, w);
  if (e != cudaSuccess) return launched(e);
  e = launch_after(merge_kernel<T>, (rows + 7) / 8, 256, 0, s, w,
                   static_cast<const T*>(hidden.p), static_cast<const T*>(embedding.p), p.width,
                   static_cast<const Partial*>(p.partial), p.slots, p.n_tiles, (uint32_t)total, pairs,
                   p.rows, p.vocab, w.inv_t * p.score_scale * kLog2e,
                   static_cast<float*>(const_cast<void*>(losses.p)),
                   static_cast<float*>(const_cast<void*>(lse.p)));
  return launched(e);
}

template <typename T>
cudaError_t finish_launch(const float* planes, uint32_t n_planes, const RowGrad* rg, T* out,
                          uint64_t rows, uint64_t width, cudaStream_t s) {
  const bool many = n_planes >= 8;
  const uint64_t columns = kFinishThreads / (many ? 8 : 1) * 4;
  return launch_after(many ? finish_kernel<T, 8> : finish_kernel<T, 1>,
                      (rows * width + columns - 1) / columns, kFinishThreads, 0, s, planes, n_planes,
                      rg, out, (uint32_t)rows, (uint32_t)width);
}

template <typename T, bool kDistill>
mf_status backward(Span hidden, Span embedding, Span targets, Span ids, Span logits,
                   float temperature, Span lse, Span grad, Span d_hidden, Span d_embedding,
                   Span workspace, uint64_t rows, uint64_t width, uint64_t vocab, void* stream) {
  const uint64_t needed = sizes_ok(rows, width, vocab) ? BackwardPlan(rows, width, vocab).bytes : 0;
  mf_status st = check(rows, width, vocab, stream, hidden, embedding, {lse, grad}, workspace,
                       needed, kDistill, targets, ids, logits, temperature);
  if (st.code != MF_OK) return st;
  if ((d_hidden.p == nullptr && d_embedding.p == nullptr) ||
      d_hidden.bytes != (d_hidden.p ? rows * width * 2 : 0) ||
      d_embedding.bytes != (d_embedding.p ? vocab * width * 2 : 0) ||
      (uintptr_t)d_hidden.p % 16 != 0 || (uintptr_t)d_embedding.p % 16 != 0 ||
      outputs_overlap({d_hidden, d_embedding, workspace},
                      {hidden, embedding, targets, ids, logits, lse, grad}))
    return fail(MF_INVALID_ARGUMENT);
  const BackwardPlan plan(rows, width, vocab);
  char* ws = static_cast<char*>(const_cast<void*>(workspace.p));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint32_t pairs = 0, sms = 0;
  cudaError_t err = device_sms(&sms);
  if (err == cudaSuccess) err = resident_pairs<T, false, false, false>(&pairs);
  if (err == cudaSuccess)
    err = plan.halves > 1 ? resident_pairs<T, false, kDistill, true>(&pairs)
                          : resident_pairs<T, false, kDistill, false>(&pairs);
  if (err != cudaSuccess) return fail(MF_CUDA_RUNTIME_FAILURE, (uint32_t)err);
  RowGrad* rg = reinterpret_cast<RowGrad*>(ws + plan.rg);
  float* gmax = reinterpret_cast<float*>(ws + plan.gmax);
  T* scaled = reinterpret_cast<T*>(ws + plan.scaled);
  float* planes = reinterpret_cast<float*>(ws + plan.planes);
  T* dh = static_cast<T*>(const_cast<void*>(d_hidden.p));
  T* de = static_cast<T*>(const_cast<void*>(d_embedding.p));
  Wanted w{};
  w.inv_t = kDistill ? 1.f / temperature : 1.f;
  if (kDistill) {
    w.offsets = static_cast<const int32_t*>(targets.p);
    w.ids = static_cast<const int32_t*>(ids.p);
    w.logits = static_cast<const float*>(logits.p);
    w.stat = reinterpret_cast<Teacher*>(ws + plan.stat);
    err = teacher_launch(w, rows, ids.bytes / 4, vocab, s);
    if (err != cudaSuccess) return launched(err);
  } else {
    w.targets = static_cast<const uint32_t*>(targets.p);
  }
  const FewGradPlan few(rows, width, vocab, sms, kDistill);
  if (few.smem > 0) {
    CUtensorMap tm_t;
    if (!make_map<T>(&tm_t, embedding.p, vocab, width, width, kBK, kBM))
      return fail(MF_CUDA_RUNTIME_FAILURE);
    FewGradParams f = {};
    f.rows = (uint32_t)rows;
    f.n = few.n;
    f.width = (uint32_t)width;
    f.w_chunks = (uint32_t)((width + kBK - 1) / kBK);
    f.vocab = (uint32_t)vocab;
    f.range = few.range;
    f.segments = few.segments;
    f.seg_chunks = few.seg_chunks;
    f.c2 = few_scale<T>(w.inv_t, few.segments, few.seg_chunks, width);
    f.hidden = hidden.p;
    f.table = embedding.p;
    f.grad = static_cast<const float*>(grad.p);
    f.lse = static_cast<const float*>(lse.p);
    f.rg = rg;
    f.planes = dh ? planes : nullptr;
    f.table_out = de;
    f.wide_rows = width % 16 == 0 && (uintptr_t)de % 32 == 0;
    err = launch_after(few_rows_grad_kernel<T, kDistill>, few.ctas, kFewGradThreads, few.smem, s,
                       tm_t, f, w);
    if (err == cudaSuccess && dh) err = finish_launch(planes, few.ctas, rg, dh, rows, width, s);
    return launched(err);
  }
  Maps maps = {};
  const uint64_t d_rows = rows * plan.halves;
  if (!make_map<T>(&maps.hidden, hidden.p, rows, width, width, kBK, kBM) ||
      !make_map<T>(&maps.table, embedding.p, vocab, width, width, kBK, kBN / 2) ||
      !make_map<T>(&maps.table_n, embedding.p, vocab, width, width, 32, kBK) ||
      !make_map<T>(&maps.scaled_n, scaled, d_rows, width, width, 32, kBK))
    return fail(MF_CUDA_RUNTIME_FAILURE);
  err = launch_after(setup_kernel<T>, rows < 32 * 148 ? (rows + 31) / 32 : 148, kSetupThreads, 0, s, w,
                     static_cast<const float*>(grad.p), static_cast<const T*>(hidden.p),
                     static_cast<const T*>(embedding.p), static_cast<const float*>(lse.p), scaled, rg,
                     gmax, (uint32_t)rows, (uint32_t)width, (uint32_t)vocab, plan.halves);
  if (err != cudaSuccess) return launched(err);

  Params p = base_params<T>(rows, width, vocab);
  p.lse = static_cast<const float*>(lse.p);
  p.rg = rg;
  p.bn = plan.bn;
  p.bn_tiles = plan.bn_tiles;
  p.blocks = plan.blocks;
  p.pitch = plan.cols;
  p.p_stage_bytes = p.blocks * kChunkBytes + p.bn * kBK;
  p.p_stages = kRingBytes / p.p_stage_bytes < kMaxStages ? kRingBytes / p.p_stage_bytes : kMaxStages;
  p.per_split = plan.per_split;
  p.d_rows = (uint32_t)d_rows;
  p.score_accs = 1;
  p.seg_chunks = p.w_chunks;
  if (kDistill && plan.halves > 1) {  // the scores that the forward call's lse is made of
    const FewPlan forward(rows, width, vocab, sms, true);
    const uint32_t first = (p.w_chunks + 1) / 2;
    if (forward.stages > 0 && forward.segments > 1 && p.w_chunks > 1) {
      p.score_accs = 2;
      p.seg_chunks = first;
      p.score_scale = 1.f + (float)(first * kBK) * Type<T>::kLostPerProduct;
    }
  }
  p.r_chunks = (uint32_t)((d_rows + kBK - 1) / kBK);
  p.gmax = gmax;
  p.wide_rows = width % 16 == 0 && (uintptr_t)de % 32 == 0;
  auto piece_cols = [&](uint32_t i) {
    const uint64_t left = vocab - (uint64_t)i * plan.cols;
    return (uint32_t)(left < plan.cols ? left : plan.cols);
  };
  uint32_t n_planes = 0;
  // launch i makes piece i of d and the products of piece i - 1
  for (uint32_t i = 0; i <= plan.pieces; ++i) {
    double load[kMaxPairs] = {};
    uint32_t n_hidden = 0, n_table = 0, n_score = 0;
    if (i > 0) {
      p.pv0 = (i - 1) * plan.cols;
      p.pcols = piece_cols(i - 1);
      p.p_chunks = (p.pcols + kBK - 1) / kBK;
      p.add = i > plan.sets;
      p.planes = planes + (uint64_t)((i - 1) % plan.sets) * plan.splits * d_rows * width;
      p.table_out = de ? de + (uint64_t)p.pv0 * width : nullptr;
      const void* d = ws + plan.piece[(i - 1) & 1];
      if (!make_map<T>(&maps.d_k, d, d_rows, p.pcols, plan.cols, kBK, kBM) ||
          !make_map<T>(&maps.d_m, d, d_rows, p.pcols, plan.cols, kBK, kBK))
        return fail(MF_CUDA_RUNTIME_FAILURE);
      const uint32_t splits = (p.p_chunks + p.per_split - 1) / p.per_split;
      // a short last piece fills the first splits of its set; a set that is
      // used again was filled by whole pieces before
      n_planes = i <= plan.sets ? (i - 1) * plan.splits + splits : plan.sets * plan.splits;
      p.t_tiles = (p.pcols + 2 * kBM - 1) / (2 * kBM);
      if (dh) n_hidden = splits * ((p.m_tiles + p.blocks - 1) / p.blocks) * p.bn_tiles;
      if (de) n_table = (p.t_tiles + p.blocks - 1) / p.blocks * p.bn_tiles;
    }
    if (i < plan.pieces) {
      p.v0 = i * plan.cols;
      p.cols = piece_cols(i);
      p.n_tiles = (p.cols + kBN - 1) / kBN;
      p.d = ws + plan.piece[i & 1];
      n_score = p.m_tiles * p.n_tiles;
    }
    // costs in columns x chunks, an epilogue taken as at least four chunks
    auto cost = [](uint32_t n, uint32_t chunks) { return (double)n * (chunks < 4 ? 4 : chunks) + 64; };
    deal(n_hidden, cost(p.blocks * p.bn, p.per_split), pairs, load, p.hidden_at);
    deal(n_table, cost(p.blocks * p.bn, p.r_chunks), pairs, load, p.table_at);
    // a score tile takes a tenth longer than its columns x chunks
    deal(n_score, 1.1 * cost(kBN, p.w_chunks), pairs, load, p.score_at);
    // products alone: the variant that needs the fewest registers
    auto kernel = i == plan.pieces ? engine_kernel<T, false, false, false>
                                   : (plan.halves > 1 ? engine_kernel<T, false, kDistill, true>
                                                      : engine_kernel<T, false, kDistill, false>);
    err = launch_after(kernel, 2 * pairs, kThreads, kSmemBytes, s, maps, p, w);
    if (err != cudaSuccess) return launched(err);
  }
  // a plane of two halves is two planes
  if (dh) err = finish_launch(planes, n_planes * plan.halves, rg, dh, rows, width, s);
  return launched(err);
}

}  // namespace loss
}  // namespace mfb

using namespace mfb;
using mfb::loss::Span;

extern "C" uint64_t mf_dense_loss_workspace_bytes(uint64_t rows, uint64_t hidden_size,
                                                  uint64_t vocab) {
  if (!loss::sizes_ok(rows, hidden_size, vocab)) return 0;
  return loss::most_bytes(rows, {loss::kFewRows},
                          [&](uint64_t r) { return loss::ForwardPlan(r, vocab).bytes; });
}

extern "C" uint64_t mf_dense_loss_backward_workspace_bytes(uint64_t rows, uint64_t hidden_size,
                                                           uint64_t vocab) {
  if (!loss::sizes_ok(rows, hidden_size, vocab)) return 0;
  return loss::most_bytes(rows, {loss::kFewGradRows, loss::kHalvesRows}, [&](uint64_t r) {
    return loss::BackwardPlan(r, hidden_size, vocab).bytes;
  });
}

#define MF_LOSS_ENTRY_POINTS(SUFFIX, TYPE)                                                         \
  extern "C" mf_status mf_dense_xent_##SUFFIX(                                                     \
      const void* hidden, uint64_t hidden_bytes, const void* embedding, uint64_t embedding_bytes,  \
      const void* targets, uint64_t targets_bytes, void* losses, uint64_t losses_bytes, void* lse, \
      uint64_t lse_bytes, void* workspace, uint64_t workspace_bytes, uint64_t rows,                \
      uint64_t hidden_size, uint64_t vocab, void* stream) {                                        \
    return loss::forward<TYPE, false>({hidden, hidden_bytes}, {embedding, embedding_bytes},        \
                               {targets, targets_bytes}, {}, {}, 1.f,                              \
                               {losses, losses_bytes}, {lse, lse_bytes},                           \
                               {workspace, workspace_bytes}, rows, hidden_size, vocab, stream);    \
  }                                                                                                \
  extern "C" mf_status mf_dense_xent_backward_##SUFFIX(                                            \
      const void* hidden, uint64_t hidden_bytes, const void* embedding, uint64_t embedding_bytes,  \
      const void* targets, uint64_t targets_bytes, const void* lse, uint64_t lse_bytes,            \
      const void* grad_losses, uint64_t grad_losses_bytes, void* d_hidden,                         \
      uint64_t d_hidden_bytes, void* d_embedding, uint64_t d_embedding_bytes, void* workspace,     \
      uint64_t workspace_bytes, uint64_t rows, uint64_t hidden_size, uint64_t vocab,               \
      void* stream) {                                                                              \
    return loss::backward<TYPE, false>({hidden, hidden_bytes}, {embedding, embedding_bytes},       \
                                {targets, targets_bytes}, {}, {}, 1.f, {lse, lse_bytes},           \
                                {grad_losses, grad_losses_bytes}, {d_hidden, d_hidden_bytes},      \
                                {d_embedding, d_embedding_bytes}, {workspace, workspace_bytes},    \
                                rows, hidden_size, vocab, stream);                                 \
  }                                                                                                \
  extern "C" mf_status mf_dense_distill_##SUFFIX(                                                  \
      const void* hidden, uint64_t hidden_bytes, const void* embedding, uint64_t embedding_bytes,  \
      const void* offsets, uint64_t offsets_bytes, const void* ids, uint64_t ids_bytes,            \
      const void* teacher_logits, uint64_t teacher_logits_bytes, float temperature, void* losses,  \
      uint64_t losses_bytes, void* lse, uint64_t lse_bytes, void* workspace,                       \
      uint64_t workspace_bytes, uint64_t rows, uint64_t hidden_size, uint64_t vocab,               \
      void* stream) {                                                                              \
    return loss::forward<TYPE, true>({hidden, hidden_bytes}, {embedding, embedding_bytes},         \
                               {offsets, offsets_bytes}, {ids, ids_bytes},                         \
                               {teacher_logits, teacher_logits_bytes}, temperature,                \
                               {losses, losses_bytes}, {lse, lse_bytes},                           \
                               {workspace, workspace_bytes}, rows, hidden_size, vocab, stream);    \
  }                                                                                                \
  extern "C" mf_status mf_dense_distill_backward_##SUFFIX(                                         \
      const void* hidden, uint64_t hidden_bytes, const void* embedding, uint64_t embedding_bytes,  \
      const void* offsets, uint64_t offsets_bytes, const void* ids, uint64_t ids_bytes,            \
      const void* teacher_logits, uint64_t teacher_logits_bytes, float temperature,                \
      const void* lse, uint64_t lse_bytes, const void* grad_losses, uint64_t grad_losses_bytes,    \
      void* d_hidden, uint64_t d_hidden_bytes, void* d_embedding, uint64_t d_embedding_bytes,      \
      void* workspace, uint64_t workspace_bytes, uint64_t rows, uint64_t hidden_size,              \
      uint64_t vocab, void* stream) {                                                              \
    return loss::backward<TYPE, true>({hidden, hidden_bytes}, {embedding, embedding_bytes},        \
                                {offsets, offsets_bytes}, {ids, ids_bytes},                        \
                                {teacher_logits, teacher_logits_bytes}, temperature,               \
                                {lse, lse_bytes}, {grad_losses, grad_losses_bytes},                \
                                {d_hidden, d_hidden_bytes}, {d_embedding, d_embedding_bytes},      \
                                {workspace, workspace_bytes}, rows, hidden_size, vocab, stream);   \
  }

MF_LOSS_ENTRY_POINTS(f16, __half)
MF_LOSS_ENTRY_POINTS(bf16, __nv_bfloat16)
