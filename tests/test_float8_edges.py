"""Limits of the float8 quantiser on the host (no GPU needed)."""
import pytest

import float8_ref as ref


@pytest.mark.parametrize("rows,outer,h,w", [(128, (1 << 31) - 1, 1, 129), (128, 1 << 30, 1, 300), (1, (1 << 31) - 1, 1, 129), (1, 1 << 23, 128, 256)])
def test_quantize_counts_the_blocks_of_the_call(rows, outer, h, w):
    """2^31 blocks and more are refused: 128 x 128 ones where the call has those (fewer than of single rows), 1 x 128 ones else."""
    assert outer * h * w <= 1 << 40 and outer * -(-h // rows) * -(-w // 128) >= 1 << 31
    c = ref.lib()
    assert c.ttb_quantize_float8(1 << 20, 1, 1, 1 << 20, 1 << 20, outer, h, w, rows, None) == -3 and b"too many" in c.ttb_last_error()


@pytest.mark.parametrize("rows,k", [(1 << 24, 1 << 24), (1 << 24, 128 * 128 + 16), (1 << 20, 1 << 18)])
def test_activations_of_too_many_blocks_are_refused(rows, k):
    """Blocks of activations are counted in 32 bits: refused before anything is launched."""
    assert rows * -(-k // 128) >= 1 << 31
    c = ref.lib()
    a = 1 << 20
    need = c.ttb_linear_float8_workspace_bytes(rows, k, 128)
    assert c.ttb_linear_float8(a, a, a, None, a, 0, rows, k, 128, 0, 3 | 8, a, need, None) == -3 and b"too many" in c.ttb_last_error()
    need = c.ttb_experts_mlp_float8_workspace_bytes(rows, 4, 1, k, 128)
    assert c.ttb_experts_mlp_float8(*[a] * 10, 1, rows, 4, 1, k, 128, 3, 3, a, need, None) == -3 and b"too many" in c.ttb_last_error()
