"""Limits of the float8 quantiser on the host (no GPU needed)."""
import pytest

import float8_ref as ref


@pytest.mark.parametrize("rows,outer,h,w", [(128, (1 << 31) - 1, 1, 129), (128, 1 << 30, 1, 300), (1, (1 << 31) - 1, 1, 129), (1, 1 << 23, 128, 256)])
def test_quantize_counts_the_blocks_of_the_call(rows, outer, h, w):
    """2^31 blocks and more are refused: 128 x 128 ones where the call has those (fewer than of single rows), 1 x 128 ones else."""
    assert outer * h * w <= 1 << 40 and outer * -(-h // rows) * -(-w // 128) >= 1 << 31
    c = ref.lib()
    assert c.ttb_quantize_float8(1 << 20, 1, 1, 1 << 20, 1 << 20, outer, h, w, rows, None) == -3 and b"too many" in c.ttb_last_error()
