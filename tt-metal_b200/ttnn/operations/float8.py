"""float8 weights with block scales, the expert router and the experts' gated MLP: additions beside the block-float linears (the reference has no
counterpart; its 8-bit weights are bfloat8_b).

A Float8Tensor is two ordinary row-major tensors: codes [.., H, W] of type float8_e4m3 and float32 scales [.., ceil(H / block_rows), ceil(W / 128)];
value = code * scale of its block. Weights of linears are [N, K] (output columns first, K contiguous) with blocks of 128 x 128, which is how checkpoints
hold them: ttnn.Float8Tensor(ttnn.from_torch(codes, device=d), ttnn.from_torch(scales, device=d)) takes such a pair as it is, ttnn.quantize_float8 makes
one. Activations stay bfloat16 on this API; the operations quantise them themselves, one scale for 128 values of a row."""
from typing import NamedTuple, Optional

from .. import _ttnn
from .. import types as T
from ..multi_device import MultiDeviceTensor
from .core import _unwrap


class Float8Tensor(NamedTuple):
    codes: T.Tensor
    scales: T.Tensor


def _wrap(like, tensor):
    return MultiDeviceTensor(tensor, like.mesh) if isinstance(like, MultiDeviceTensor) else tensor


def _pair(op, name, w):
    if not isinstance(w, (tuple, list)) or len(w) != 2:
        raise RuntimeError(f"{op}: {name} must be a Float8Tensor (codes, scales)")
    return _unwrap(w[0]), _unwrap(w[1])


def quantize_float8(input_tensor, *, block_rows: int = 128) -> Float8Tensor:
    """A float32 or bfloat16 device tensor [.., H, W] as float8 codes with a scale for every block of block_rows x 128 values, block_rows 128 (weights) or 1
    (activations): scale = max(largest magnitude, 2^-100) / 448, code = x / scale rounded to the nearest e4m3 number (ties to even). A NaN becomes the NaN
    code and leaves the scale alone."""
    codes, scales = _ttnn.quantize_float8(_unwrap(input_tensor), block_rows)
    return Float8Tensor(_wrap(input_tensor, codes), _wrap(input_tensor, scales))


def linear_float8(input_tensor, weight: Float8Tensor, *, bias=None, activation: Optional[str] = None, dtype: Optional[T.DataType] = None):
    """activation(input_tensor @ weight^T + bias) on the float8 tensor cores: weight codes [N, K], scales of 128 x 128 blocks, K a multiple of 16. The bfloat16
    input (TILE or ROW_MAJOR layout, any row count) is quantised within the call, one scale for 128 values of a row; every 128 products are summed on the
    tensor cores and the sums scaled and added in float32. `bias` is bfloat16 [1, N]; the result has the input's layout and is bfloat16 or float32 (`dtype`)."""
    codes, scales = _pair("ttnn.linear_float8", "weight", weight)
    out = _ttnn.linear_float8(_unwrap(input_tensor), codes, scales, bias=_unwrap(bias) if bias is not None else None, dtype=dtype, activation=activation)
    return _wrap(input_tensor, out)


def route_to_experts(logits, k: int, *, score: str = "softmax", bias=None, groups: int = 1, top_groups: int = 1, group_score: str = "max",
                     renormalize: bool = True, scale: float = 1.0):
    """The router of a mixture of experts: for every row of `logits` [.., rows, E] (float32 or bfloat16) the k experts it goes to. Returns (weights, experts),
    row-major float32 and uint32 [.., rows, k], best first.

    Scores are the softmax or sigmoid of the logits. Experts are chosen by score + bias (`bias`: float32, one value an expert, for balance), ties to the
    lowest index; with groups > 1 only among the top_groups groups of E / groups neighbouring experts whose best expert (group_score "max") or two best
    together ("top2_sum") count most. Weights are the chosen experts' scores (without bias) times `scale`, divided by their sum under `renormalize`.
    Without bias and "top2_sum" the order is that of the logits, which is that of exact scores; with either it is that of 64-bit scores and sums, in which scores that
    only differ behind 64 bits (sigmoids of logits above about 37) are ties. An expert whose logit is -inf is never chosen; where a row has too few left, the remaining places hold the index E
    and the weight 0 (ttnn.experts_mlp_float8 skips them: a row of -inf gets no expert). The experts of a row with a NaN, or an infinity
    under softmax, have NaN weights; a NaN's own is never chosen."""
    weights, experts = _ttnn.route_to_experts(_unwrap(logits), k, score=score, bias=_unwrap(bias) if bias is not None else None, groups=groups,
                                              top_groups=top_groups, group_score=group_score, renormalize=renormalize, scale=scale)
    return _wrap(logits, weights), _wrap(logits, experts)


def experts_mlp_float8(input_tensor, experts, weights, gate: Float8Tensor, up: Float8Tensor, down: Float8Tensor, *, activation: Optional[str] = "silu"):
    """sum_j weights[t, j] * ((activation(x[t] @ gate[e]^T) * (x[t] @ up[e]^T)) @ down[e]^T) with e = experts[t, j]: the gated MLP (as ttnn.linear_gated
    followed by ttnn.linear) of every row's experts, as `route_to_experts` names and weights them. `gate` and `up` are Float8Tensors [E, ffn, hidden], `down`
    [E, hidden, ffn], with blocks of 128 x 128; hidden and ffn are multiples of 16. Inputs of both matmuls are quantised with a scale for 128 values of a row.
    An index outside [0, E) contributes nothing; a row without experts comes out as zeros. The result has the input's shape and layout, bfloat16."""
    op = "ttnn.experts_mlp_float8"
    pairs = _pair(op, "gate", gate) + _pair(op, "up", up) + _pair(op, "down", down)
    return _wrap(input_tensor, _ttnn.experts_mlp_float8(_unwrap(input_tensor), _unwrap(experts), _unwrap(weights), *pairs, activation))
