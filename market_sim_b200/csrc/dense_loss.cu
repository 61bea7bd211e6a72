// Losses over the tied output table (include/mf_loss.h): softmax cross
// entropy over the whole vocabulary and distillation from a teacher's top
// logits, with their gradients.
//
// Plain version: 64 x 64 tiles on the FP32 pipes.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <initializer_list>

#include "common.cuh"
#include "mf_loss.h"

namespace mfb {
namespace loss {

constexpr int kTile = 64;
constexpr int kStep = 16;
constexpr int kThreads = 256;
constexpr uint32_t kWorkers = 148;                 // forward: walks over the vocabulary
constexpr uint64_t kPieceBytes = 256ull << 20;     // one piece of d

template <typename T>
struct Type;
template <>
struct Type<__half> {
  // d / gmax is at most 1: times 2^15 it uses fp16's whole range, and keeps
  // full precision down to 2^-29 of the largest weight
  static constexpr float kScale = 32768.f;
  static __device__ __forceinline__ float to(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half from(float x) { return __float2half_rn(x); }
};
template <>
struct Type<__nv_bfloat16> {
  static constexpr float kScale = 1.f;
  static __device__ __forceinline__ float to(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 from(float x) { return __float2bfloat16_rn(x); }
};

// What a row wants: one target, or a teacher's set.
struct Wanted {
  const uint32_t* targets;   // cross entropy
  const int32_t* offsets;    // distillation
  const int32_t* ids;
  const float* logits;
  float inv_t;               // 1 / temperature (1 for cross entropy)
  float2* stat;              // distillation: {log sum exp of t / T, sum q log q}
};

// stat.x of a row without entries, and of an invalid row
__device__ __forceinline__ bool stat_empty(float2 s) { return s.x == -INFINITY; }
__device__ __forceinline__ bool stat_invalid(float2 s) { return s.x != s.x; }

struct Partial {  // of one row over one walk: running max, sum of exp, sum of q s
  float m, l, dot;
};

// One warp per row: the teacher's normaliser and entropy.
__global__ void teacher_kernel(Wanted w, uint32_t rows, uint32_t entries, uint32_t vocab) {
  const uint32_t lane = threadIdx.x & 31;
  for (uint32_t r = (blockIdx.x * blockDim.x + threadIdx.x) >> 5; r < rows;
       r += (gridDim.x * blockDim.x) >> 5) {
    const int32_t a = w.offsets[r], b = w.offsets[r + 1];
    bool bad = a < 0 || b < a || (uint32_t)b > entries;
    float m = -INFINITY;
    if (!bad) {
      for (int32_t k = a + (int32_t)lane; k < b; k += 32) {
        const int32_t id = w.ids[k];
        const float t = w.logits[k];
        bad |= id < 0 || (uint32_t)id >= vocab || (k > a && w.ids[k - 1] >= id) || t != t ||
               t == INFINITY;
        m = fmaxf(m, t * w.inv_t);
      }
    }
    bad = __any_sync(0xFFFFFFFFu, bad);
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    float2 st = make_float2(-INFINITY, 0.f);
    if (bad) {
      st.x = __uint_as_float(0x7FC00000u);
    } else if (m > -INFINITY) {
      float l = 0.f;
      for (int32_t k = a + (int32_t)lane; k < b; k += 32) l += expf(w.logits[k] * w.inv_t - m);
      for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
      st.x = m + logf(l);
      float ent = 0.f;
      for (int32_t k = a + (int32_t)lane; k < b; k += 32) {
        const float lq = w.logits[k] * w.inv_t - st.x, q = expf(lq);
        if (q > 0.f) ent += q * lq;
      }
      for (int o = 16; o; o >>= 1) ent += __shfl_xor_sync(0xFFFFFFFFu, ent, o);
      st.y = ent;
    }
    if (lane == 0) w.stat[r] = st;
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

// acc[i][j] = sum_k A(m0 + ty + 16 i, k) B(n0 + tx + 16 j, k); A(m, k) is
// a[m * am + k * ak], zero outside [0, M) x [0, K); B likewise.
template <typename T>
__device__ __forceinline__ void tile_product(float (&acc)[4][4], const T* a, uint64_t am,
                                             uint64_t ak, const T* b, uint64_t bn, uint64_t bk,
                                             uint32_t m0, uint32_t M, uint32_t n0, uint32_t N,
                                             uint32_t K, float (*sa)[kTile + 1],
                                             float (*sb)[kTile + 1]) {
  const uint32_t tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
  for (uint32_t k0 = 0; k0 < K; k0 += kStep) {
    for (uint32_t e = threadIdx.x; e < kTile * kStep; e += kThreads) {
      // neighbouring threads along whichever index is contiguous
      const uint32_t ia = ak == 1 ? e / kStep : e % kTile, ka = ak == 1 ? e % kStep : e / kTile;
      const uint32_t ib = bk == 1 ? e / kStep : e % kTile, kb = bk == 1 ? e % kStep : e / kTile;
      sa[ka][ia] = (m0 + ia < M && k0 + ka < K)
                       ? Type<T>::to(a[(uint64_t)(m0 + ia) * am + (uint64_t)(k0 + ka) * ak]) : 0.f;
      sb[kb][ib] = (n0 + ib < N && k0 + kb < K)
                       ? Type<T>::to(b[(uint64_t)(n0 + ib) * bn + (uint64_t)(k0 + kb) * bk]) : 0.f;
    }
    __syncthreads();
    for (int k = 0; k < kStep; ++k)
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j)
          acc[i][j] = fmaf(sa[k][ty + 16 * i], sb[k][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
}

// Forward: block (m, split) walks its share of the vocabulary tiles for 64 rows.
template <typename T>
__global__ void __launch_bounds__(kThreads) forward_kernel(const T* hidden, const T* emb, Wanted w,
                                                           Partial* out, uint32_t rows,
                                                           uint32_t width, uint32_t vocab,
                                                           uint32_t splits) {
  __shared__ float sa[kStep][kTile + 1], sb[kStep][kTile + 1], st[kTile][kTile + 1];
  const uint32_t m0 = blockIdx.x * kTile, split = blockIdx.y;
  const uint32_t tiles = (vocab + kTile - 1) / kTile;
  const uint32_t t0 = (uint32_t)((uint64_t)tiles * split / splits);
  const uint32_t t1 = (uint32_t)((uint64_t)tiles * (split + 1) / splits);
  const uint32_t tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const uint32_t r = m0 + threadIdx.x;
  const bool owner = threadIdx.x < kTile && r < rows;
  Partial p{-INFINITY, 0.f, 0.f};
  uint32_t target = kInvalid;
  int32_t at = 0, end = 0;
  float tlse = 0.f;
  if (owner && w.targets) target = w.targets[r];
  if (owner && w.offsets) {
    const float2 s = w.stat[r];
    if (!stat_empty(s) && !stat_invalid(s)) {
      at = first_entry(w, r, t0 * kTile);
      end = w.offsets[r + 1];
      tlse = s.x;
    }
  }
  for (uint32_t t = t0; t < t1; ++t) {
    float acc[4][4];
    tile_product(acc, hidden, width, 1, emb, width, 1, m0, rows, t * kTile, vocab, width, sa, sb);
    for (int i = 0; i < 4; ++i)
      for (int j = 0; j < 4; ++j) st[ty + 16 * i][tx + 16 * j] = acc[i][j] * w.inv_t;
    __syncthreads();
    if (owner) {
      const uint32_t n = min((uint32_t)kTile, vocab - t * kTile);
      float m = p.m;
      for (uint32_t c = 0; c < n; ++c) m = fmaxf(m, st[threadIdx.x][c]);
      float l = p.l * (p.m == m ? 1.f : expf(p.m - m));
      for (uint32_t c = 0; c < n; ++c) l += expf(st[threadIdx.x][c] - m);
      p.m = m;
      p.l = l;
      if (w.targets && target - t * kTile < n) p.dot = st[threadIdx.x][target - t * kTile];
      for (; at < end && (uint32_t)w.ids[at] < t * kTile + n; ++at) {
        const float q = expf(w.logits[at] * w.inv_t - tlse);
        if (q > 0.f) p.dot = fmaf(q, st[threadIdx.x][w.ids[at] - t * kTile], p.dot);
      }
    }
    __syncthreads();
  }
  if (owner) out[(uint64_t)r * splits + split] = p;
}

// One thread per row joins the walks' partial sums.
__global__ void merge_kernel(Wanted w, const Partial* part, uint32_t splits, uint32_t rows,
                             uint32_t vocab, float* losses, float* lse) {
  const uint32_t r = blockIdx.x * blockDim.x + threadIdx.x;
  if (r >= rows) return;
  float m = -INFINITY, l = 0.f, dot = 0.f;
  for (uint32_t s = 0; s < splits; ++s) m = fmaxf(m, part[(uint64_t)r * splits + s].m);
  for (uint32_t s = 0; s < splits; ++s) {
    const Partial p = part[(uint64_t)r * splits + s];
    l += p.l * (p.m == m ? 1.f : expf(p.m - m));
    dot += p.dot;
  }
  const float z = m + logf(l);
  lse[r] = z;
  float loss;
  if (w.targets) {
    const uint32_t t = w.targets[r];
    loss = t == kInvalid ? 0.f : (t >= vocab ? __uint_as_float(0x7FC00000u) : z - dot);
  } else {
    const float2 s = w.stat[r];
    const float t = 1.f / w.inv_t;
    loss = stat_empty(s) ? 0.f : (stat_invalid(s) ? s.x : t * t * (s.y + (z - dot)));
  }
  losses[r] = loss;
}

// ---- backward ----------------------------------------------------------

struct RowGrad {  // one row's factors of d
  float coef;     // d16 = (p - q) * coef
  float scale;    // d_hidden = (d16 . E) * scale
};

__device__ __forceinline__ float row_weight(const Wanted& w, const float* grad, uint32_t r,
                                            uint32_t vocab) {
  if (w.targets) return w.targets[r] < vocab ? grad[r] : 0.f;
  const float2 s = w.stat[r];
  return stat_empty(s) || stat_invalid(s) ? 0.f : grad[r] / w.inv_t;
}

// Row factors and the copy of the hidden rows that d_embedding is made of.
template <typename T>
__global__ void __launch_bounds__(kThreads) setup_kernel(Wanted w, const float* grad,
                                                         const T* hidden, T* scaled, RowGrad* rg,
                                                         float* gmax_out, uint32_t rows,
                                                         uint32_t width, uint32_t vocab) {
  __shared__ float s_max[kThreads / 32];
  float g = 0.f;
  for (uint32_t r = threadIdx.x; r < rows; r += kThreads) {
    const float a = fabsf(row_weight(w, grad, r, vocab));
    if (a < INFINITY) g = fmaxf(g, a);  // an infinite weight spoils its own row only
  }
  for (int o = 16; o; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xFFFFFFFFu, g, o));
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = g;
  __syncthreads();
  for (int i = 0; i < kThreads / 32; ++i) g = fmaxf(g, s_max[i]);
  if (blockIdx.x == 0 && threadIdx.x == 0) *gmax_out = g;
  for (uint32_t r = blockIdx.x; r < rows; r += gridDim.x) {
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
    if (threadIdx.x == 0)
      rg[r] = RowGrad{mant * Type<T>::kScale, g * two_e / Type<T>::kScale};
    for (uint32_t c = threadIdx.x; c < width; c += kThreads)
      scaled[(uint64_t)r * width + c] =
          wr == 0.f ? Type<T>::from(0.f)
                    : Type<T>::from(Type<T>::to(hidden[(uint64_t)r * width + c]) * two_e);
  }
}

// One piece of d: columns [v0, v0 + n_cols) for 64 rows x 64 columns a block.
template <typename T>
__global__ void __launch_bounds__(kThreads) piece_kernel(const T* hidden, const T* emb, Wanted w,
                                                         const float* lse, const RowGrad* rg, T* d,
                                                         uint32_t pitch, uint32_t rows,
                                                         uint32_t width, uint32_t v0,
                                                         uint32_t n_cols) {
  __shared__ float sa[kStep][kTile + 1], sb[kStep][kTile + 1], st[kTile][kTile + 1];
  const uint32_t m0 = blockIdx.x * kTile, n0 = blockIdx.y * kTile;
  const uint32_t tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const uint32_t r = m0 + threadIdx.x;
  float acc[4][4];
  tile_product(acc, hidden, width, 1, emb + (uint64_t)v0 * width, width, 1, m0, rows, n0, n_cols,
               width, sa, sb);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) st[ty + 16 * i][tx + 16 * j] = acc[i][j] * w.inv_t;
  __syncthreads();
  if (threadIdx.x >= kTile || r >= rows) return;
  const RowGrad g = rg[r];
  const uint32_t n = min((uint32_t)kTile, n_cols - n0);
  const uint32_t first = v0 + n0;
  int32_t at = 0, end = 0;
  float tlse = 0.f;
  if (w.offsets && g.coef != 0.f) {
    at = first_entry(w, r, first);
    end = w.offsets[r + 1];
    tlse = w.stat[r].x;
  }
  const float z = lse[r];
  for (uint32_t c = 0; c < n; ++c) {
    float p = expf(st[threadIdx.x][c] - z);
    if (w.targets) {
      if (w.targets[r] == first + c) p -= 1.f;
    } else if (at < end && (uint32_t)w.ids[at] == first + c) {
      p -= expf(w.logits[at] * w.inv_t - tlse);
      ++at;
    }
    d[(uint64_t)r * pitch + n0 + c] = Type<T>::from(g.coef == 0.f ? 0.f : p * g.coef);
  }
}

// d_hidden: adds one piece's part; the last piece scales and rounds.
template <typename T>
__global__ void __launch_bounds__(kThreads) hidden_kernel(const T* d, uint32_t pitch, const T* emb,
                                                          float* sum, T* out, const RowGrad* rg,
                                                          uint32_t rows, uint32_t width,
                                                          uint32_t n_cols, bool first, bool last) {
  __shared__ float sa[kStep][kTile + 1], sb[kStep][kTile + 1];
  const uint32_t m0 = blockIdx.x * kTile, n0 = blockIdx.y * kTile;
  float acc[4][4];
  tile_product(acc, d, pitch, 1, emb, 1, width, m0, rows, n0, width, n_cols, sa, sb);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const uint32_t r = m0 + (threadIdx.x >> 4) + 16 * i, c = n0 + (threadIdx.x & 15) + 16 * j;
      if (r >= rows || c >= width) continue;
      float v = acc[i][j];
      if (!first) v += sum[(uint64_t)r * width + c];
      if (last)
        out[(uint64_t)r * width + c] = Type<T>::from(rg[r].coef == 0.f ? 0.f : v * rg[r].scale);
      else
        sum[(uint64_t)r * width + c] = v;
    }
}

// d_embedding rows of one piece.
template <typename T>
__global__ void __launch_bounds__(kThreads) table_kernel(const T* d, uint32_t pitch,
                                                         const T* scaled, T* out,
                                                         const float* gmax, uint32_t rows,
                                                         uint32_t width, uint32_t n_cols) {
  __shared__ float sa[kStep][kTile + 1], sb[kStep][kTile + 1];
  const uint32_t m0 = blockIdx.x * kTile, n0 = blockIdx.y * kTile;
  float acc[4][4];
  tile_product(acc, d, 1, pitch, scaled, 1, width, m0, n_cols, n0, width, rows, sa, sb);
  const float scale = *gmax / Type<T>::kScale;
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const uint32_t v = m0 + (threadIdx.x >> 4) + 16 * i, c = n0 + (threadIdx.x & 15) + 16 * j;
      if (v < n_cols && c < width)
        out[(uint64_t)v * width + c] = Type<T>::from(acc[i][j] * scale);
    }
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

uint32_t forward_splits(uint64_t rows, uint64_t vocab) {
  const uint64_t m = (rows + kTile - 1) / kTile, n = (vocab + kTile - 1) / kTile;
  uint64_t s = (kWorkers + m - 1) / m;
  return (uint32_t)(s < n ? s : n);
}

struct ForwardPlan {
  uint64_t stat, partial, bytes;
  uint32_t splits;
  ForwardPlan(uint64_t rows, uint64_t vocab) {
    splits = forward_splits(rows, vocab);
    stat = 0;
    partial = round_up(rows * sizeof(float2), 256);
    bytes = round_up(partial + rows * splits * sizeof(Partial), 256);
  }
};

struct BackwardPlan {
  uint64_t stat, rg, gmax, scaled, sum, piece, bytes;
  uint32_t cols;  // vocabulary rows of one piece
  BackwardPlan(uint64_t rows, uint64_t width, uint64_t vocab) {
    uint64_t c = kPieceBytes / (2 * rows) / 256 * 256;
    if (c < 256) c = 256;
    const uint64_t all = round_up(vocab, 256);
    cols = (uint32_t)(c < all ? c : all);
    stat = 0;
    rg = round_up(stat + rows * sizeof(float2), 256);
    gmax = round_up(rg + rows * sizeof(RowGrad), 256);
    scaled = gmax + 256;
    sum = round_up(scaled + rows * width * 2, 256);
    piece = round_up(sum + (cols < vocab ? rows * width * 4 : 0), 256);
    bytes = round_up(piece + rows * cols * 2, 256);
  }
};

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
      (uintptr_t)workspace.p % 16 != 0)
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
    if (ids.bytes / 4 > (uint64_t)INT32_MAX) return fail(MF_RESOURCE_LIMIT);
  }
  return ok();
}

mf_status launched(cudaError_t e) {
  return e == cudaSuccess ? ok() : fail(MF_CUDA_BACKEND_FAILURE, (uint32_t)e);
}

void teacher_launch(const Wanted& w, uint64_t rows, uint64_t entries, uint64_t vocab,
                    cudaStream_t s) {
  const uint64_t blocks = (rows + 7) / 8;
  teacher_kernel<<<(unsigned)(blocks < 1184 ? blocks : 1184), 256, 0, s>>>(
      w, (uint32_t)rows, (uint32_t)entries, (uint32_t)vocab);
}

template <typename T>
mf_status forward(Span hidden, Span embedding, Span targets, Span ids, Span logits, bool distill,
                  float temperature, Span losses, Span lse, Span workspace, uint64_t rows,
                  uint64_t width, uint64_t vocab, void* stream) {
  const uint64_t needed = sizes_ok(rows, width, vocab) ? ForwardPlan(rows, vocab).bytes : 0;
  mf_status st = check(rows, width, vocab, stream, hidden, embedding, {losses, lse}, workspace,
                       needed, distill, targets, ids, logits, temperature);
  if (st.code != MF_OK) return st;
  if (outputs_overlap({losses, lse, workspace}, {hidden, embedding, targets, ids, logits}))
    return fail(MF_INVALID_ARGUMENT);
  const ForwardPlan plan(rows, vocab);
  char* ws = static_cast<char*>(const_cast<void*>(workspace.p));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  Wanted w{};
  w.inv_t = distill ? 1.f / temperature : 1.f;
  if (distill) {
    w.offsets = static_cast<const int32_t*>(targets.p);
    w.ids = static_cast<const int32_t*>(ids.p);
    w.logits = static_cast<const float*>(logits.p);
    w.stat = reinterpret_cast<float2*>(ws + plan.stat);
    teacher_launch(w, rows, ids.bytes / 4, vocab, s);
  } else {
    w.targets = static_cast<const uint32_t*>(targets.p);
  }
  Partial* part = reinterpret_cast<Partial*>(ws + plan.partial);
  forward_kernel<T><<<dim3((unsigned)((rows + kTile - 1) / kTile), plan.splits), kThreads, 0, s>>>(
      static_cast<const T*>(hidden.p), static_cast<const T*>(embedding.p), w, part,
      (uint32_t)rows, (uint32_t)width, (uint32_t)vocab, plan.splits);
  merge_kernel<<<(unsigned)((rows + 255) / 256), 256, 0, s>>>(
      w, part, plan.splits, (uint32_t)rows, (uint32_t)vocab,
      static_cast<float*>(const_cast<void*>(losses.p)), static_cast<float*>(const_cast<void*>(lse.p)));
  return launched(cudaGetLastError());
}

template <typename T>
mf_status backward(Span hidden, Span embedding, Span targets, Span ids, Span logits, bool distill,
                   float temperature, Span lse, Span grad, Span d_hidden, Span d_embedding,
                   Span workspace, uint64_t rows, uint64_t width, uint64_t vocab, void* stream) {
  const uint64_t needed = sizes_ok(rows, width, vocab) ? BackwardPlan(rows, width, vocab).bytes : 0;
  mf_status st = check(rows, width, vocab, stream, hidden, embedding, {lse, grad}, workspace,
                       needed, distill, targets, ids, logits, temperature);
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
  Wanted w{};
  w.inv_t = distill ? 1.f / temperature : 1.f;
  if (distill) {
    w.offsets = static_cast<const int32_t*>(targets.p);
    w.ids = static_cast<const int32_t*>(ids.p);
    w.logits = static_cast<const float*>(logits.p);
    w.stat = reinterpret_cast<float2*>(ws + plan.stat);
    teacher_launch(w, rows, ids.bytes / 4, vocab, s);
  } else {
    w.targets = static_cast<const uint32_t*>(targets.p);
  }
  RowGrad* rg = reinterpret_cast<RowGrad*>(ws + plan.rg);
  float* gmax = reinterpret_cast<float*>(ws + plan.gmax);
  T* scaled = reinterpret_cast<T*>(ws + plan.scaled);
  float* sum = reinterpret_cast<float*>(ws + plan.sum);
  T* d = reinterpret_cast<T*>(ws + plan.piece);
  const T* h = static_cast<const T*>(hidden.p);
  const T* e = static_cast<const T*>(embedding.p);
  T* dh = static_cast<T*>(const_cast<void*>(d_hidden.p));
  T* de = static_cast<T*>(const_cast<void*>(d_embedding.p));
  const float* z = static_cast<const float*>(lse.p);
  setup_kernel<T><<<(unsigned)(rows < 592 ? rows : 592), kThreads, 0, s>>>(
      w, static_cast<const float*>(grad.p), h, scaled, rg, gmax, (uint32_t)rows, (uint32_t)width,
      (uint32_t)vocab);
  const unsigned mt = (unsigned)((rows + kTile - 1) / kTile);
  const unsigned ht = (unsigned)((width + kTile - 1) / kTile);
  for (uint64_t v0 = 0; v0 < vocab; v0 += plan.cols) {
    const uint32_t n = (uint32_t)(vocab - v0 < plan.cols ? vocab - v0 : plan.cols);
    const unsigned nt = (n + kTile - 1) / kTile;
    piece_kernel<T><<<dim3(mt, nt), kThreads, 0, s>>>(h, e, w, z, rg, d, plan.cols, (uint32_t)rows,
                                                      (uint32_t)width, (uint32_t)v0, n);
    if (dh)
      hidden_kernel<T><<<dim3(mt, ht), kThreads, 0, s>>>(d, plan.cols, e + v0 * width, sum, dh, rg,
                                                         (uint32_t)rows, (uint32_t)width, n,
                                                         v0 == 0, v0 + n == vocab);
    if (de)
      table_kernel<T><<<dim3(nt, ht), kThreads, 0, s>>>(d, plan.cols, scaled, de + v0 * width, gmax,
                                                        (uint32_t)rows, (uint32_t)width, n);
  }
  return launched(cudaGetLastError());
}

}  // namespace loss
}  // namespace mfb

using namespace mfb;
using mfb::loss::Span;

extern "C" uint64_t mf_dense_loss_workspace_bytes(uint64_t rows, uint64_t hidden_size,
                                                  uint64_t vocab) {
  return loss::sizes_ok(rows, hidden_size, vocab) ? loss::ForwardPlan(rows, vocab).bytes : 0;
}

extern "C" uint64_t mf_dense_loss_backward_workspace_bytes(uint64_t rows, uint64_t hidden_size,
                                                           uint64_t vocab) {
  return loss::sizes_ok(rows, hidden_size, vocab)
             ? loss::BackwardPlan(rows, hidden_size, vocab).bytes : 0;
}

#define MF_LOSS_ENTRY_POINTS(SUFFIX, TYPE)                                                         \
  extern "C" mf_status mf_dense_xent_##SUFFIX(                                                     \
      const void* hidden, uint64_t hidden_bytes, const void* embedding, uint64_t embedding_bytes,  \
      const void* targets, uint64_t targets_bytes, void* losses, uint64_t losses_bytes, void* lse, \
      uint64_t lse_bytes, void* workspace, uint64_t workspace_bytes, uint64_t rows,                \
      uint64_t hidden_size, uint64_t vocab, void* stream) {                                        \
    return loss::forward<TYPE>({hidden, hidden_bytes}, {embedding, embedding_bytes},               \
                               {targets, targets_bytes}, {}, {}, false, 1.f,                       \
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
    return loss::backward<TYPE>({hidden, hidden_bytes}, {embedding, embedding_bytes},              \
                                {targets, targets_bytes}, {}, {}, false, 1.f, {lse, lse_bytes},    \
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
    return loss::forward<TYPE>({hidden, hidden_bytes}, {embedding, embedding_bytes},               \
                               {offsets, offsets_bytes}, {ids, ids_bytes},                         \
                               {teacher_logits, teacher_logits_bytes}, true, temperature,          \
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
    return loss::backward<TYPE>({hidden, hidden_bytes}, {embedding, embedding_bytes},              \
                                {offsets, offsets_bytes}, {ids, ids_bytes},                        \
                                {teacher_logits, teacher_logits_bytes}, true, temperature,         \
                                {lse, lse_bytes}, {grad_losses, grad_losses_bytes},                \
                                {d_hidden, d_hidden_bytes}, {d_embedding, d_embedding_bytes},      \
                                {workspace, workspace_bytes}, rows, hidden_size, vocab, stream);   \
  }

MF_LOSS_ENTRY_POINTS(f16, __half)
MF_LOSS_ENTRY_POINTS(bf16, __nv_bfloat16)
