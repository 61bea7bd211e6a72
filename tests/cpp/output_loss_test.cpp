// A C++ caller of the losses over the tied table (marketforge::cuda,
// include/marketforge/cuda/output_loss.hpp): small known answers in double
// precision on the host, both types, both directions, and refusals.  Prints
// "ALL PASSED" and exits 0 on success.  Built and run by tests/test_loss_cpp.py.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <type_traits>
#include <vector>

#include "marketforge/cuda/output_loss.hpp"

using marketforge::ErrorCode;
using namespace marketforge::cuda;

static int failures = 0;
#define CHECK(c)                                                 \
  do {                                                           \
    if (!(c)) {                                                  \
      std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #c); \
      ++failures;                                                \
    }                                                            \
  } while (0)

template <typename T>
static DeviceBuffer upload(const std::vector<T>& v, const CudaStream& s) {
  auto b = DeviceBuffer::allocate(v.size() * sizeof(T));
  CHECK(b.has_value());
  DeviceBuffer d = std::move(b).value();
  CHECK(d.copy_from_host_async(v.data(), v.size() * sizeof(T), 0, s.handle()).ok());
  return d;
}

static DeviceBuffer room(std::uint64_t bytes) {
  auto b = DeviceBuffer::allocate(bytes);
  CHECK(b.has_value());
  return std::move(b).value();
}

template <typename T>
static std::vector<T> download(const DeviceBuffer& d, std::size_t n, const CudaStream& s) {
  std::vector<T> v(n);
  CHECK(d.copy_to_host_async(v.data(), n * sizeof(T), 0, s.handle()).ok());
  CHECK(s.synchronize().ok());
  return v;
}

// Values that both 16-bit types hold exactly.
template <typename T>
static T value(int i, int j) {
  return T(float((i * 7 + j * 5) % 17 - 8) / 16.f);
}

template <typename T>
static void run(LossType type, const CudaStream& s, bool distill) {
  const std::uint64_t rows = 3, width = 16, vocab = 37;
  const double temperature = distill ? 2.0 : 1.0;
  std::vector<T> hidden, table;
  for (int r = 0; r < 3; ++r)
    for (int c = 0; c < 16; ++c) hidden.push_back(value<T>(r + 1, c));
  for (int v = 0; v < 37; ++v)
    for (int c = 0; c < 16; ++c) table.push_back(value<T>(v, 3 * c));
  // row 1 is ignored: no target, no set
  const std::vector<std::uint32_t> targets{5, 0xFFFFFFFFu, 36};
  const std::vector<std::int32_t> offsets{0, 2, 2, 4}, ids{3, 5, 0, 36};
  const std::vector<float> logits{0.5f, 2.f, -1.f, 1.f}, grad{1.f, 1.f, -0.5f};
  // the formulas in double precision
  std::vector<double> q(rows * vocab), loss(rows), lse(rows), dh(rows * width), de(vocab * width);
  for (std::uint64_t r = 0; r < rows; ++r) {
    if (r == 1) continue;
    if (!distill) {
      q[r * vocab + targets[r]] = 1.0;
    } else {
      double z = 0;
      for (int k = offsets[r]; k < offsets[r + 1]; ++k) z += std::exp(logits[k] / temperature);
      for (int k = offsets[r]; k < offsets[r + 1]; ++k)
        q[r * vocab + ids[k]] = std::exp(logits[k] / temperature) / z;
    }
  }
  for (std::uint64_t r = 0; r < rows; ++r) {
    std::vector<double> sc(vocab);
    double z = 0;
    for (std::uint64_t v = 0; v < vocab; ++v) {
      for (std::uint64_t c = 0; c < width; ++c)
        sc[v] += double(float(hidden[r * width + c])) * double(float(table[v * width + c]));
      sc[v] /= temperature;
      z += std::exp(sc[v]);
    }
    lse[r] = std::log(z);
    for (std::uint64_t v = 0; v < vocab; ++v) {
      const double qv = q[r * vocab + v], p = std::exp(sc[v] - lse[r]);
      if (qv > 0) loss[r] += temperature * temperature * qv * (std::log(qv) - sc[v] + lse[r]);
      const double d = r == 1 ? 0.0 : temperature * grad[r] * (p - qv);
      for (std::uint64_t c = 0; c < width; ++c) {
        dh[r * width + c] += d * float(table[v * width + c]);
        de[v * width + c] += d * float(hidden[r * width + c]);
      }
    }
  }
  DeviceBuffer h = upload(hidden, s), e = upload(table, s), t = upload(targets, s),
               o = upload(offsets, s), i = upload(ids, s), l = upload(logits, s),
               g = upload(grad, s), losses = room(rows * 4), z = room(rows * 4),
               d_h = room(rows * width * 2), d_e = room(vocab * width * 2);
  auto made = allocate_loss_workspace(rows, width, vocab, true);
  CHECK(made.has_value());
  DeviceBuffer ws = std::move(made).value();
  if (distill) {
    CHECK(dense_distillation(type, h, e, o, i, l, 2.f, losses, z, ws, rows, width, vocab,
                             s.handle()).ok());
    CHECK(dense_distillation_backward(type, h, e, o, i, l, 2.f, z, g, d_h, d_e, ws, rows, width,
                                      vocab, s.handle()).ok());
  } else {
    CHECK(dense_cross_entropy(type, h, e, t, losses, z, ws, rows, width, vocab, s.handle()).ok());
    CHECK(dense_cross_entropy_backward(type, h, e, t, z, g, d_h, d_e, ws, rows, width, vocab,
                                       s.handle()).ok());
  }
  const auto got_loss = download<float>(losses, rows, s), got_lse = download<float>(z, rows, s);
  for (std::uint64_t r = 0; r < rows; ++r) {
    // 16 exact products below 1/4 and 37 terms in FP32: far below 1e-5
    CHECK(std::fabs(got_lse[r] - lse[r]) < 1e-5 && std::fabs(got_loss[r] - loss[r]) < 4e-5);
  }
  // one rounding of the result (half a step, relative) on top of d's own,
  // smaller one: within a step, over a floor of 2^-14
  const double step = std::is_same_v<T, __half> ? 1.0 / 1024 : 1.0 / 128;
  const auto got_dh = download<T>(d_h, rows * width, s);
  const auto got_de = download<T>(d_e, vocab * width, s);
  for (std::size_t k = 0; k < got_dh.size(); ++k)
    CHECK(std::fabs(float(got_dh[k]) - dh[k]) <= step * (std::fabs(dh[k]) + 1.0 / 16));
  for (std::size_t k = 0; k < got_de.size(); ++k)
    CHECK(std::fabs(float(got_de[k]) - de[k]) <= step * (std::fabs(de[k]) + 1.0 / 16));
  for (std::uint64_t c = 0; c < width; ++c) CHECK(float(got_dh[width + c]) == 0.f);
  // one gradient alone
  DeviceBuffer none;
  if (!distill) {
    CHECK(dense_cross_entropy_backward(type, h, e, t, z, g, none, d_e, ws, rows, width, vocab,
                                       s.handle()).ok());
    CHECK(dense_cross_entropy_backward(type, h, e, t, z, g, d_h, none, ws, rows, width, vocab,
                                       s.handle()).ok());
    CHECK(dense_cross_entropy_backward(type, h, e, t, z, g, none, none, ws, rows, width, vocab,
                                       s.handle()).code == ErrorCode::invalid_argument);
    CHECK(dense_cross_entropy(type, h, e, t, losses, losses, ws, rows, width, vocab, s.handle())
              .code == ErrorCode::invalid_argument);
    CHECK(dense_cross_entropy(type, h, e, t, losses, z, ws, rows, width, vocab, StreamHandle{})
              .code == ErrorCode::invalid_argument);
  }
  CHECK(s.synchronize().ok());
}

int main() {
  CHECK(!allocate_loss_workspace(0, 16, 8, false).has_value());
  CHECK(!allocate_loss_workspace(4, 12, 8, true).has_value());
  auto made = CudaStream::create();
  if (!made.has_value()) {
    std::printf("no stream\n");
    return 1;
  }
  const CudaStream s = std::move(made).value();
  for (const bool distill : {false, true}) {
    run<__half>(LossType::f16, s, distill);
    run<__nv_bfloat16>(LossType::bf16, s, distill);
  }
  if (failures == 0) std::printf("ALL PASSED\n");
  return failures == 0 ? 0 : 1;
}
