#include "float8.hpp"

#include <algorithm>

namespace ttnn_b200 {
namespace {

int64_t blocks_of(int64_t n) { return (n + 127) / 128; }

void on_device(const char *op, const char *name, const Tensor &t) {
    if (t.storage_type() != StorageType::DEVICE) throw_error(std::string(op) + ": Tensor " + name + " must be on device!");
    if (!t.is_allocated()) throw_error(std::string(op) + ": Tensor " + name + " must be allocated!");
}
void same_device(const char *op, const Tensor &a, const Tensor &b) {
    if (a.device() != b.device()) throw_error(std::string(op) + ": operands must be on the same device");
}

// [outer, H, W] of an activation-like tensor (rank 2 to 4); only the last two dimensions may carry tile padding.
void activation_extents(const char *op, const char *name, const Tensor &t, int64_t &outer, int64_t &H, int64_t &W) {
    const Shape &s = t.shape();
    if (s.rank() < 2 || s.rank() > 4) throw_error(std::string(op) + ": Tensor " + name + " must be of rank 2, 3 or 4, but got " + std::to_string(s.rank()));
    if (t.layout() == Layout::ROW_MAJOR) {
        if (s.has_padding()) throw_error(std::string(op) + ": padded row-major tensors are not supported");
    } else if (!(s.padded() == Shape(s.dims()).tile_padded().padded())) {
        throw_error(std::string(op) + ": Tensor " + name + " must be padded to whole tiles in its last two dimensions only");
    }
    s.as_outer_hw(outer, H, W, false);
    if (outer <= 0 || H <= 0 || W <= 0) throw_error(std::string(op) + ": Tensor " + name + " must not be empty");
}

int activation_code(const char *op, const std::optional<std::string> &act) {
    if (!act) return TTB_ACT_NONE;
    if (*act == "relu") return TTB_ACT_RELU;
    if (*act == "gelu") return TTB_ACT_GELU;
    if (*act == "silu") return TTB_ACT_SILU;
    throw_error(std::string(op) + ": " + *act + " is not supported as activation function");
}

// A weight's codes [lead, N, K] and scales of 128 x 128 blocks; every dimension before the last two counts into lead.
void weight_extents(const char *op, const std::string &name, const Float8 &w, int64_t &lead, int64_t &N, int64_t &K) {
    on_device(op, (name + ".codes").c_str(), w.codes);
    on_device(op, (name + ".scales").c_str(), w.scales);
    same_device(op, w.codes, w.scales);
    if (w.codes.dtype() != DataType::FLOAT8_E4M3 || w.codes.layout() != Layout::ROW_MAJOR)
        throw_error(std::string(op) + ": " + name + ".codes must be a ROW_MAJOR_LAYOUT tensor of type float8_e4m3");
    if (w.scales.dtype() != DataType::FLOAT32 || w.scales.layout() != Layout::ROW_MAJOR)
        throw_error(std::string(op) + ": " + name + ".scales must be a ROW_MAJOR_LAYOUT tensor of type float32");
    const auto &c = w.codes.shape().dims(), &s = w.scales.shape().dims();
    if (c.size() < 2 || s.size() != c.size() || w.codes.shape().has_padding() || w.scales.shape().has_padding())
        throw_error(std::string(op) + ": " + name + ".codes and " + name + ".scales must have the same rank, 2 or more, and no padding");
    lead = 1;
    for (size_t i = 0; i + 2 < c.size(); ++i) {
        if (c[i] != s[i]) throw_error(std::string(op) + ": " + name + ".scales must have the leading dimensions of " + name + ".codes");
        lead *= c[i];
    }
    N = c[c.size() - 2];
    K = c[c.size() - 1];
    if (s[s.size() - 2] != blocks_of(N) || s[s.size() - 1] != blocks_of(K))
        throw_error(std::string(op) + ": " + name + ".scales must hold one scale for every 128 x 128 block of " + name + ".codes");
}

int layout_flags(const Tensor &t) { return t.layout() == Layout::ROW_MAJOR ? TTB_MM_A_ROW_MAJOR | TTB_MM_OUT_ROW_MAJOR : 0; }

}  // namespace

Float8 quantize_float8(const Tensor &t, int block_rows) {
    const char *op = "ttnn.quantize_float8";
    on_device(op, "input_tensor", t);
    if (t.dtype() != DataType::FLOAT32 && t.dtype() != DataType::BFLOAT16)
        throw_error(std::string(op) + ": Tensor input_tensor must be of type float32 or bfloat16, but got " + to_string(t.dtype()));
    if (block_rows != 1 && block_rows != 128) throw_error(std::string(op) + ": block_rows must be 1 or 128");
    int64_t outer, H, W;
    activation_extents(op, "input_tensor", t, outer, H, W);
    Device *dev = t.device();
    dev->make_current();
    std::vector<int64_t> sd = t.shape().dims();
    sd[sd.size() - 2] = (H + block_rows - 1) / block_rows;
    sd.back() = blocks_of(W);
    const Shape cs(t.shape().dims()), ss(sd);
    Float8 q{Tensor(allocate_device_buffer(dev, physical_bytes(cs, DataType::FLOAT8_E4M3, Layout::ROW_MAJOR)), cs, DataType::FLOAT8_E4M3, Layout::ROW_MAJOR),
             Tensor(allocate_device_buffer(dev, physical_bytes(ss, DataType::FLOAT32, Layout::ROW_MAJOR)), ss, DataType::FLOAT32, Layout::ROW_MAJOR)};
    check(ttb_quantize_float8(t.data(), static_cast<int>(t.dtype()), t.layout() == Layout::ROW_MAJOR, q.codes.data(), q.scales.data(), outer, H, W, block_rows, nullptr), op);
    return q;
}

Tensor linear_float8(const Tensor &x, const Float8 &w, const std::optional<Tensor> &bias, std::optional<DataType> dtype, const std::optional<std::string> &activation) {
    const char *op = "ttnn.linear_float8";
    on_device(op, "input_tensor", x);
    if (x.dtype() != DataType::BFLOAT16) throw_error(std::string(op) + ": Tensor input_tensor must be of type bfloat16, but got " + to_string(x.dtype()));
    int64_t outer, H, K, lead, N, Kw;
    activation_extents(op, "input_tensor", x, outer, H, K);
    weight_extents(op, "weight", w, lead, N, Kw);
    same_device(op, x, w.codes);
    if (lead != 1) throw_error(std::string(op) + ": the weight must be one matrix (leading dimensions of 1)");
    if (K != Kw) throw_error(std::string(op) + ": The width of the first tensor must be equal to the width of the weight's codes [N, K]");
    const DataType out_dtype = dtype.value_or(DataType::BFLOAT16);
    if (out_dtype != DataType::BFLOAT16 && out_dtype != DataType::FLOAT32) throw_error(std::string(op) + ": output dtype must be bfloat16 or float32");
    const int act = activation_code(op, activation);
    int flags = layout_flags(x);
    const void *bias_ptr = nullptr;
    if (bias) {
        on_device(op, "bias", *bias);
        same_device(op, x, *bias);
        const auto &bd = bias->shape().dims();
        if (bias->dtype() != DataType::BFLOAT16 || bias->shape().volume() != N || bd.empty() || bd.back() != N)
            throw_error(std::string(op) + ": bias must be a bfloat16 tensor of shape [1, N]");
        if (bias->layout() == Layout::ROW_MAJOR) {
            if (bias->shape().has_padding()) throw_error(std::string(op) + ": padded row-major tensors are not supported");
            flags |= TTB_MM_BIAS_ROW_MAJOR;
        } else if (bd.size() < 2 || bias->shape().padded_volume() != 32 * ((N + 31) / 32 * 32)) {
            throw_error(std::string(op) + ": bias must have shape [1, N] padded to one tile row");
        }
        bias_ptr = bias->data();
    }
    Device *dev = x.device();
    dev->make_current();
    std::vector<int64_t> od = x.shape().dims();
    od.back() = N;
    const Shape out_shape = x.layout() == Layout::TILE ? Shape(od).tile_padded() : Shape(od);
    const int64_t rows = outer * (x.layout() == Layout::TILE ? (H + 31) / 32 * 32 : H);
    auto outb = allocate_device_buffer(dev, physical_bytes(out_shape, out_dtype, x.layout()));
    const int64_t need = ttb_linear_float8_workspace_bytes(rows, K, N);
    void *ws = need > 0 ? dev->workspace(need) : nullptr;
    // Not TTB_MM_WEIGHTS_RESIDENT: the operation before may be the one that writes the codes (ttnn.quantize_float8, or whatever fills memory that this API only wraps),
    // and a kernel that starts early sees its stores only after waiting for it.
    check(ttb_linear_float8(x.data(), w.codes.data(), w.scales.data(), bias_ptr, outb->ptr, static_cast<int>(out_dtype), rows, K, N, act,
                            flags | TTB_MM_WORKSPACE_ZEROED, ws, need, nullptr),
          op);
    return Tensor(outb, out_shape, out_dtype, x.layout());
}

Routing route_to_experts(const Tensor &logits, int k, const std::string &score, const std::optional<Tensor> &bias, int groups, int top_groups,
                         const std::string &group_score, bool renormalize, float scale) {
    const char *op = "ttnn.route_to_experts";
    on_device(op, "logits", logits);
    if (logits.dtype() != DataType::FLOAT32 && logits.dtype() != DataType::BFLOAT16)
        throw_error(std::string(op) + ": Tensor logits must be of type float32 or bfloat16, but got " + to_string(logits.dtype()));
    if (score != "softmax" && score != "sigmoid") throw_error(std::string(op) + ": score must be \"softmax\" or \"sigmoid\"");
    if (group_score != "max" && group_score != "top2_sum") throw_error(std::string(op) + ": group_score must be \"max\" or \"top2_sum\"");
    int64_t outer, H, E;
    activation_extents(op, "logits", logits, outer, H, E);
    const void *bias_ptr = nullptr;
    if (bias) {
        on_device(op, "bias", *bias);
        same_device(op, logits, *bias);
        if (bias->dtype() != DataType::FLOAT32 || bias->layout() != Layout::ROW_MAJOR || bias->shape().has_padding() || bias->shape().volume() != E)
            throw_error(std::string(op) + ": bias must be a float32 ROW_MAJOR_LAYOUT tensor with one value for each expert");
        bias_ptr = bias->data();
    }
    Device *dev = logits.device();
    dev->make_current();
    std::vector<int64_t> od = logits.shape().dims();
    od.back() = std::clamp(k, 1, 32);   // (the call refuses others)
    const Shape shape(od);
    Routing r{Tensor(allocate_device_buffer(dev, physical_bytes(shape, DataType::FLOAT32, Layout::ROW_MAJOR)), shape, DataType::FLOAT32, Layout::ROW_MAJOR),
              Tensor(allocate_device_buffer(dev, physical_bytes(shape, DataType::UINT32, Layout::ROW_MAJOR)), shape, DataType::UINT32, Layout::ROW_MAJOR)};
    check(ttb_route_to_experts(logits.data(), static_cast<int>(logits.dtype()), bias_ptr, r.weights.data(), r.experts.data(), outer, H, E, k,
                               score == "sigmoid" ? TTB_SCORE_SIGMOID : TTB_SCORE_SOFTMAX, groups, top_groups,
                               group_score == "max" ? TTB_GROUP_MAX : TTB_GROUP_TOP2_SUM, renormalize, scale,
                               logits.layout() == Layout::ROW_MAJOR ? TTB_MM_A_ROW_MAJOR : 0, nullptr),
          op);
    return r;
}

Tensor experts_mlp_float8(const Tensor &x, const Tensor &experts, const Tensor &weights, const Float8 &gate, const Float8 &up, const Float8 &down,
                          const std::optional<std::string> &activation) {
    const char *op = "ttnn.experts_mlp_float8";
    on_device(op, "input_tensor", x);
    on_device(op, "experts", experts);
    on_device(op, "weights", weights);
    if (x.dtype() != DataType::BFLOAT16) throw_error(std::string(op) + ": Tensor input_tensor must be of type bfloat16, but got " + to_string(x.dtype()));
    int64_t outer, H, hidden;
    activation_extents(op, "input_tensor", x, outer, H, hidden);
    if (experts.dtype() != DataType::UINT32 || experts.layout() != Layout::ROW_MAJOR || weights.dtype() != DataType::FLOAT32 || weights.layout() != Layout::ROW_MAJOR)
        throw_error(std::string(op) + ": experts and weights must be ROW_MAJOR_LAYOUT tensors of type uint32 and float32");
    const auto &ed = experts.shape().dims();
    if (!(experts.shape() == weights.shape()) || experts.shape().has_padding() || ed.empty() || experts.shape().volume() != outer * H * ed.back())
        throw_error(std::string(op) + ": experts and weights must have shape [.., rows, k] with the rows of the input tensor");
    const int64_t k = ed.back();
    int64_t E, F, Kg, E2, F2, K2, E3, N3, K3;
    weight_extents(op, "gate", gate, E, F, Kg);
    weight_extents(op, "up", up, E2, F2, K2);
    weight_extents(op, "down", down, E3, N3, K3);
    for (const Tensor *t : {&experts, &weights, &gate.codes, &up.codes, &down.codes}) same_device(op, x, *t);
    if (E != E2 || F != F2 || Kg != K2) throw_error(std::string(op) + ": gate and up must have the same shape");
    if (E3 != E || N3 != hidden || K3 != F || Kg != hidden)
        throw_error(std::string(op) + ": gate and up must be [experts, ffn, hidden] and down [experts, hidden, ffn], hidden the width of the input tensor");
    if (k > 32) throw_error(std::string(op) + ": at most 32 experts for a row");
    const int act = activation_code(op, activation);
    Device *dev = x.device();
    dev->make_current();
    const int64_t need = ttb_experts_mlp_float8_workspace_bytes(outer * H, E, k, hidden, F);
    auto ws = need > 0 ? allocate_device_buffer(dev, need) : nullptr;
    auto outb = allocate_device_buffer(dev, physical_bytes(x.shape(), DataType::BFLOAT16, x.layout()));
    check(ttb_experts_mlp_float8(x.data(), experts.data(), weights.data(), gate.codes.data(), gate.scales.data(), up.codes.data(), up.scales.data(), down.codes.data(),
                                 down.scales.data(), outb->ptr, outer, H, E, (int32_t)k, hidden, F, act, layout_flags(x), ws ? ws->ptr : nullptr, need, nullptr),
          op);
    return Tensor(outb, x.shape(), DataType::BFLOAT16, x.layout());
}

}  // namespace ttnn_b200
