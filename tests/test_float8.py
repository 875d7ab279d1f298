"""float8 and mixture-of-experts operators on the host: refusals of the C ABI and of the ttnn surface, row-major float8 tensors (no GPU needed)."""
import pytest
import torch

import float8_ref as ref
import ttnn

A = 1 << 20   # an aligned address that no refused call touches
INVALID, UNSUPPORTED, WORKSPACE = -1, -3, -4


def _says(lib, rc, code, text):
    assert rc == code and text.encode() in lib.ttb_last_error(), (rc, lib.ttb_last_error())


def test_float8_tensors_round_trip_without_a_gpu(tmp_path):
    codes = (torch.arange(6 * 40).reshape(2, 3, 40) - 100).float().to(torch.float8_e4m3fn)
    t = ttnn.from_torch(codes)
    assert t.dtype == ttnn.float8_e4m3 and t.layout == ttnn.ROW_MAJOR_LAYOUT and t.buffer_bytes() == 240
    assert torch.equal(ttnn.to_torch(t).view(torch.uint8), codes.view(torch.uint8))
    assert torch.equal(ttnn.to_torch(ttnn.from_torch(torch.tensor([[1.0, 300.0, 2.0 ** -9]]), dtype=ttnn.float8_e4m3)).float(), torch.tensor([[1.0, 288.0, 2.0 ** -9]]))
    ttnn.dump_tensor(tmp_path / "w.bin", t)
    assert torch.equal(ttnn.to_torch(ttnn.load_tensor(tmp_path / "w.bin")).view(torch.uint8), codes.view(torch.uint8))
    assert "FLOAT8_E4M3" in repr(t) and list(ttnn.reshape(t, [6, 40]).shape) == [6, 40]


def test_float8_tensors_are_row_major():
    codes = torch.zeros(32, 32).to(torch.float8_e4m3fn)
    with pytest.raises(RuntimeError, match="ROW_MAJOR"):
        ttnn.from_torch(codes, layout=ttnn.TILE_LAYOUT)
    t = ttnn.from_torch(codes)
    with pytest.raises(RuntimeError, match="row-major"):
        ttnn.to_layout(t, ttnn.TILE_LAYOUT)
    with pytest.raises(RuntimeError, match="not supported"):
        t.pad([64, 64], [0, 0], 0.0)
    with pytest.raises(RuntimeError, match="not supported"):
        t.unpad([0, 0], [3, 3])


def test_quantize_refusals():
    c = ref.lib()

    def call(src=A, dtype=1, codes=A, scales=A, outer=1, h=4, w=128, rows=128):
        return c.ttb_quantize_float8(src, dtype, 1, codes, scales, outer, h, w, rows, None)
    for kw in ({"src": None}, {"codes": None}, {"scales": None}):
        _says(c, call(**kw), INVALID, "null pointer")
    _says(c, call(dtype=2), UNSUPPORTED, "float32 or bfloat16")
    _says(c, call(rows=64), INVALID, "block_rows")
    for kw in ({"outer": 0}, {"h": 0}, {"w": -1}):
        _says(c, call(**kw), INVALID, "positive")
    for kw in ({"h": 1 << 41}, {"outer": 1 << 20, "h": 1 << 20, "w": 2}, {"outer": 1 << 62, "h": 4}, {"h": 1 << 31, "w": 1}, {"h": 1 << 31, "w": 1, "rows": 1},
               {"h": 1 << 30, "w": 300, "rows": 1}):
        _says(c, call(**kw), UNSUPPORTED, "too many")
    _says(c, call(src=A + 2), INVALID, "misaligned")
    _says(c, call(dtype=0, src=A + 1), INVALID, "misaligned")
    _says(c, call(scales=A + 2), INVALID, "misaligned")


def test_linear_refusals():
    c = ref.lib()

    def call(a=A, w=A, s=A, bias=None, out=A, dtype=0, rows=32, k=256, n=128, act=0, flags=3, ws=A, nbytes=1 << 30):
        return c.ttb_linear_float8(a, w, s, bias, out, dtype, rows, k, n, act, flags, ws, nbytes, None)
    for kw in ({"a": None}, {"w": None}, {"s": None}, {"out": None}):
        _says(c, call(**kw), INVALID, "null tensor")
    _says(c, call(dtype=3), UNSUPPORTED, "bfloat16 or float32")
    _says(c, call(act=4), INVALID, "activation")
    _says(c, call(act=-1), INVALID, "activation")
    _says(c, call(flags=4), INVALID, "flags")
    for kw in ({"rows": 0}, {"k": 0}, {"n": 0}, {"rows": -1}, {"n": (1 << 24) + 1}, {"k": 1 << 60}):
        _says(c, call(**kw), INVALID, "between 1 and 2^24")
    for k in (8, 100, 130):
        _says(c, call(k=k), INVALID, "multiple of 16")
    for flags in (0, 1, 2):
        _says(c, call(rows=33, flags=flags), INVALID, "multiple of 32 rows")
    for kw in ({"a": A + 8}, {"w": A + 1}, {"s": A + 2}, {"out": A + 1}, {"out": A + 2, "dtype": 1}, {"bias": A + 1}):
        _says(c, call(**kw), INVALID, "aligned")
    need = c.ttb_linear_float8_workspace_bytes(32, 256, 128)
    assert need > 0 and c.ttb_linear_float8_workspace_bytes(0, 256, 128) == -1
    for kw in ({"ws": None}, {"nbytes": need - 1}, {"ws": A + 16}):
        _says(c, call(**kw), WORKSPACE, "workspace")


def test_route_refusals():
    c = ref.lib()

    def call(x=A, dtype=1, bias=None, w=A, e=A, outer=1, h=4, n=64, k=8, score=0, groups=1, top=1, gs=0, flags=1):
        return c.ttb_route_to_experts(x, dtype, bias, w, e, outer, h, n, k, score, groups, top, gs, 1, 1.0, flags, None)
    for kw in ({"x": None}, {"w": None}, {"e": None}):
        _says(c, call(**kw), INVALID, "null tensor")
    _says(c, call(dtype=2), UNSUPPORTED, "float32 or bfloat16")
    _says(c, call(flags=2), INVALID, "flags")
    for kw in ({"outer": 0}, {"h": 0}, {"outer": 1 << 16, "h": 1 << 16}, {"h": 1 << 31}):
        _says(c, call(**kw), INVALID, "row count")
    for n in (0, 1025):
        _says(c, call(n=n, k=1), UNSUPPORTED, "experts")
    for kw in ({"k": 0}, {"k": 33}, {"n": 4, "k": 5}):
        _says(c, call(**kw), INVALID, "k must be")
    _says(c, call(score=2), INVALID, "score")
    for g in (0, 3, 64):
        _says(c, call(groups=g), INVALID, "groups of one size")
    for t in (0, 9):
        _says(c, call(groups=8, top=t), INVALID, "top_groups")
    _says(c, call(groups=16, top=1), INVALID, "have no 8 to choose")
    _says(c, call(groups=8, top=4, gs=2), INVALID, "group score")
    for kw in ({"x": A + 2}, {"bias": A + 1}, {"w": A + 2}, {"e": A + 1}):
        _says(c, call(**kw), INVALID, "misaligned")


def test_experts_refusals():
    c = ref.lib()

    def call(ptrs=None, outer=1, h=4, experts=8, k=2, hidden=256, ffn=128, act=3, flags=3, ws=A, nbytes=1 << 30):
        p = [A] * 10
        for i, v in (ptrs or {}).items():
            p[i] = v
        return c.ttb_experts_mlp_float8(*p, outer, h, experts, k, hidden, ffn, act, flags, ws, nbytes, None)
    for i in range(10):
        _says(c, call({i: None}), INVALID, "null tensor")
    for i in (0, 3, 5, 7, 9):
        _says(c, call({i: A + 8}), INVALID, "16-byte aligned")
    for i in (1, 2, 4, 6, 8):
        _says(c, call({i: A + 2}), INVALID, "misaligned")
    _says(c, call(flags=512), INVALID, "flags")
    _says(c, call(act=9), INVALID, "activation")
    for kw in ({"outer": 0}, {"h": 0}, {"h": 1 << 25}, {"outer": 1 << 62}):
        _says(c, call(**kw), INVALID, "rows must be")
    for kw in ({"experts": 0}, {"experts": 1025}, {"k": 0}, {"k": 33}, {"h": 1 << 24}, {"outer": 1 << 24, "h": 1 << 24}, {"hidden": 0}, {"ffn": 1 << 25}):
        _says(c, call(**kw), INVALID, "between 1 and 2^24 rows times k")
    for kw in ({"hidden": 100}, {"ffn": 72}):
        _says(c, call(**kw), INVALID, "multiples of 16")
    need = c.ttb_experts_mlp_float8_workspace_bytes(4, 8, 2, 256, 128)
    for kw in ({"ws": None}, {"nbytes": need - 1}, {"ws": A + 128}):
        _says(c, call(**kw), WORKSPACE, "workspace")


def test_surface_refuses_host_tensors():
    x = ttnn.from_torch(torch.zeros(4, 256, dtype=torch.bfloat16))
    w = ttnn.Float8Tensor(ttnn.from_torch(torch.zeros(128, 256).to(torch.float8_e4m3fn)), ttnn.from_torch(torch.ones(1, 2)))
    i, p = ttnn.from_torch(torch.zeros(4, 2, dtype=torch.int32)), ttnn.from_torch(torch.zeros(4, 2))
    for call in (lambda: ttnn.quantize_float8(x), lambda: ttnn.linear_float8(x, w), lambda: ttnn.route_to_experts(p, 1),
                 lambda: ttnn.experts_mlp_float8(x, i, p, w, w, w)):
        with pytest.raises(RuntimeError, match="must be on device"):
            call()
    with pytest.raises(RuntimeError, match="Float8Tensor"):
        ttnn.linear_float8(x, x)
