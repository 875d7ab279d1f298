// float8 weights with block scales and the mixture-of-experts operators of the ttnn surface, beside the block-float linears. The reference has
// no counterpart (its 8-bit weights are bfloat8_b); arguments, checks and results follow the neighbouring operations (ops.hpp).
#pragma once
#include <optional>
#include <string>

#include "tensor.hpp"

namespace ttnn_b200 {

// Row-major codes [.., H, W] (FLOAT8_E4M3) and scales [.., ceil(H / block_rows), ceil(W / 128)] (FLOAT32).
struct Float8 {
    Tensor codes, scales;
};
Float8 quantize_float8(const Tensor &t, int block_rows);

// activation(x w^T + bias): w's codes are [N, K] and its scales [ceil(N / 128), ceil(K / 128)]; the result has x's layout.
Tensor linear_float8(const Tensor &x, const Float8 &w, const std::optional<Tensor> &bias, std::optional<DataType> dtype,
                     const std::optional<std::string> &activation);

// Row-major [.., rows, k]: weights (FLOAT32) and expert indexes (UINT32).
struct Routing {
    Tensor weights, experts;
};
Routing route_to_experts(const Tensor &logits, int k, const std::string &score, const std::optional<Tensor> &bias, int groups, int top_groups,
                         const std::string &group_score, bool renormalize, float scale);

// The experts' gated MLP, weighted and summed per token; the result has x's shape, layout and type.
Tensor experts_mlp_float8(const Tensor &x, const Tensor &experts, const Tensor &weights, const Float8 &gate, const Float8 &up, const Float8 &down,
                          const std::optional<std::string> &activation);

}  // namespace ttnn_b200
