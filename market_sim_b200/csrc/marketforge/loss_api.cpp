// marketforge::cuda losses over the C-ABI of include/mf_loss.h: the buffers'
// exact byte sizes are passed through, so validation happens in one place.
#include "marketforge/cuda/output_loss.hpp"
#include "mf_loss.h"

namespace marketforge::cuda {
namespace {

Status to_status(mf_status s) noexcept { return Status{static_cast<ErrorCode>(s.code), s.detail}; }
const void* ca(const DeviceBuffer& b) noexcept { return reinterpret_cast<const void*>(b.address().value); }
void* ma(DeviceBuffer& b) noexcept { return reinterpret_cast<void*>(b.address().value); }
void* st(StreamHandle h) noexcept { return reinterpret_cast<void*>(h.value); }

}  // namespace

Result<DeviceBuffer> allocate_loss_workspace(std::uint64_t rows, std::uint64_t hidden_size,
                                             std::uint64_t vocabulary_size,
                                             bool backward) noexcept {
  std::uint64_t bytes = mf_dense_loss_workspace_bytes(rows, hidden_size, vocabulary_size);
  if (backward && bytes != 0) {
    const std::uint64_t b = mf_dense_loss_backward_workspace_bytes(rows, hidden_size, vocabulary_size);
    if (b > bytes) bytes = b;
  }
  if (bytes == 0)
    return Result<DeviceBuffer>::failure(Status::failure(ErrorCode::resource_limit, 0));
  return DeviceBuffer::allocate(bytes);
}

Status dense_cross_entropy(LossType type, const DeviceBuffer& hidden,
                           const DeviceBuffer& embedding, const DeviceBuffer& targets,
                           DeviceBuffer& losses, DeviceBuffer& lse, DeviceBuffer& workspace,
                           std::uint64_t rows, std::uint64_t hidden_size,
                           std::uint64_t vocabulary_size, StreamHandle stream) noexcept {
  const auto f = type == LossType::f16 ? mf_dense_xent_f16 : mf_dense_xent_bf16;
  return to_status(f(ca(hidden), hidden.size_bytes(), ca(embedding), embedding.size_bytes(),
                     ca(targets), targets.size_bytes(), ma(losses), losses.size_bytes(), ma(lse),
                     lse.size_bytes(), ma(workspace), workspace.size_bytes(), rows, hidden_size,
                     vocabulary_size, st(stream)));
}

Status dense_cross_entropy_backward(LossType type, const DeviceBuffer& hidden,
                                    const DeviceBuffer& embedding, const DeviceBuffer& targets,
                                    const DeviceBuffer& lse, const DeviceBuffer& grad_losses,
                                    DeviceBuffer& d_hidden, DeviceBuffer& d_embedding,
                                    DeviceBuffer& workspace, std::uint64_t rows,
                                    std::uint64_t hidden_size, std::uint64_t vocabulary_size,
                                    StreamHandle stream) noexcept {
  const auto f = type == LossType::f16 ? mf_dense_xent_backward_f16 : mf_dense_xent_backward_bf16;
  return to_status(f(ca(hidden), hidden.size_bytes(), ca(embedding), embedding.size_bytes(),
                     ca(targets), targets.size_bytes(), ca(lse), lse.size_bytes(),
                     ca(grad_losses), grad_losses.size_bytes(), ma(d_hidden),
                     d_hidden.size_bytes(), ma(d_embedding), d_embedding.size_bytes(),
                     ma(workspace), workspace.size_bytes(), rows, hidden_size, vocabulary_size,
                     st(stream)));
}

Status dense_distillation(LossType type, const DeviceBuffer& hidden, const DeviceBuffer& embedding,
                          const DeviceBuffer& offsets, const DeviceBuffer& ids,
                          const DeviceBuffer& teacher_logits, float temperature,
                          DeviceBuffer& losses, DeviceBuffer& lse, DeviceBuffer& workspace,
                          std::uint64_t rows, std::uint64_t hidden_size,
                          std::uint64_t vocabulary_size, StreamHandle stream) noexcept {
  const auto f = type == LossType::f16 ? mf_dense_distill_f16 : mf_dense_distill_bf16;
  return to_status(f(ca(hidden), hidden.size_bytes(), ca(embedding), embedding.size_bytes(),
                     ca(offsets), offsets.size_bytes(), ca(ids), ids.size_bytes(),
                     ca(teacher_logits), teacher_logits.size_bytes(), temperature, ma(losses),
                     losses.size_bytes(), ma(lse), lse.size_bytes(), ma(workspace),
                     workspace.size_bytes(), rows, hidden_size, vocabulary_size, st(stream)));
}

Status dense_distillation_backward(LossType type, const DeviceBuffer& hidden,
                                   const DeviceBuffer& embedding, const DeviceBuffer& offsets,
                                   const DeviceBuffer& ids, const DeviceBuffer& teacher_logits,
                                   float temperature, const DeviceBuffer& lse,
                                   const DeviceBuffer& grad_losses, DeviceBuffer& d_hidden,
                                   DeviceBuffer& d_embedding, DeviceBuffer& workspace,
                                   std::uint64_t rows, std::uint64_t hidden_size,
                                   std::uint64_t vocabulary_size, StreamHandle stream) noexcept {
  const auto f =
      type == LossType::f16 ? mf_dense_distill_backward_f16 : mf_dense_distill_backward_bf16;
  return to_status(f(ca(hidden), hidden.size_bytes(), ca(embedding), embedding.size_bytes(),
                     ca(offsets), offsets.size_bytes(), ca(ids), ids.size_bytes(),
                     ca(teacher_logits), teacher_logits.size_bytes(), temperature, ca(lse),
                     lse.size_bytes(), ca(grad_losses), grad_losses.size_bytes(), ma(d_hidden),
                     d_hidden.size_bytes(), ma(d_embedding), d_embedding.size_bytes(),
                     ma(workspace), workspace.size_bytes(), rows, hidden_size, vocabulary_size,
                     st(stream)));
}

}  // namespace marketforge::cuda
