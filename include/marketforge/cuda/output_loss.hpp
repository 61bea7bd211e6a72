// Losses over the tied output table in the reference's style (no reference
// counterpart): cross entropy over the whole vocabulary and distillation from a
// teacher's top logits, with their gradients.  Contracts are those of
// include/mf_loss.h.  The workspace needs no initialisation.
#pragma once

#include <cstdint>

#include "marketforge/core/result.hpp"
#include "marketforge/core/status.hpp"
#include "marketforge/cuda/cuda_stream.hpp"
#include "marketforge/cuda/device_buffer.hpp"

namespace marketforge::cuda {

// The type of the hidden rows, the table and their gradients.
enum class LossType { f16, bf16 };

// A workspace for up to `rows` rows, for the forward calls or for both
// directions.  Sizes outside the limits give resource_limit.
[[nodiscard]] Result<DeviceBuffer> allocate_loss_workspace(std::uint64_t rows,
                                                           std::uint64_t hidden_size,
                                                           std::uint64_t vocabulary_size,
                                                           bool backward) noexcept;

// targets: u32 [rows] (restricted_greedy_invalid_token_id ignores a row);
// losses, lse: f32 [rows].
[[nodiscard]] Status dense_cross_entropy(LossType type, const DeviceBuffer& hidden,
                                         const DeviceBuffer& embedding,
                                         const DeviceBuffer& targets, DeviceBuffer& losses,
                                         DeviceBuffer& lse, DeviceBuffer& workspace,
                                         std::uint64_t rows, std::uint64_t hidden_size,
                                         std::uint64_t vocabulary_size,
                                         StreamHandle stream) noexcept;

// lse as the forward call wrote it; grad_losses: f32 [rows]; d_hidden [rows,
// hidden_size], d_embedding [vocabulary_size, hidden_size], one of them may be
// an empty buffer.
[[nodiscard]] Status dense_cross_entropy_backward(
    LossType type, const DeviceBuffer& hidden, const DeviceBuffer& embedding,
    const DeviceBuffer& targets, const DeviceBuffer& lse, const DeviceBuffer& grad_losses,
    DeviceBuffer& d_hidden, DeviceBuffer& d_embedding, DeviceBuffer& workspace, std::uint64_t rows,
    std::uint64_t hidden_size, std::uint64_t vocabulary_size, StreamHandle stream) noexcept;

// The teacher's sets as CSR: row r's entries are [offsets[r], offsets[r+1]) of
// ids (int32, ascending) and teacher_logits (f32).
[[nodiscard]] Status dense_distillation(LossType type, const DeviceBuffer& hidden,
                                        const DeviceBuffer& embedding,
                                        const DeviceBuffer& offsets, const DeviceBuffer& ids,
                                        const DeviceBuffer& teacher_logits, float temperature,
                                        DeviceBuffer& losses, DeviceBuffer& lse,
                                        DeviceBuffer& workspace, std::uint64_t rows,
                                        std::uint64_t hidden_size, std::uint64_t vocabulary_size,
                                        StreamHandle stream) noexcept;

[[nodiscard]] Status dense_distillation_backward(
    LossType type, const DeviceBuffer& hidden, const DeviceBuffer& embedding,
    const DeviceBuffer& offsets, const DeviceBuffer& ids, const DeviceBuffer& teacher_logits,
    float temperature, const DeviceBuffer& lse, const DeviceBuffer& grad_losses,
    DeviceBuffer& d_hidden, DeviceBuffer& d_embedding, DeviceBuffer& workspace, std::uint64_t rows,
    std::uint64_t hidden_size, std::uint64_t vocabulary_size, StreamHandle stream) noexcept;

}  // namespace marketforge::cuda
