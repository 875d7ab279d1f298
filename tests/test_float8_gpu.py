"""float8 quantisation, linear, router and experts' MLP on the GPU against plain 64-bit implementations (float8_ref.py has the bounds)."""
import ctypes
import math

import pytest
import torch

import cabi
import float8_ref as ref
import ttnn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return ttnn.open_device(0)


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    assert cabi.load().check_status(None) == 0


def gen(*seed):
    return torch.Generator().manual_seed(hash(seed) % (1 << 31))


def put(t, dev, layout=ttnn.ROW_MAJOR_LAYOUT, dtype=None):
    return ttnn.from_torch(t, dtype=dtype, layout=layout, device=dev)


def pair(w, dev):
    return ttnn.Float8Tensor(put(w[0], dev), put(w[1], dev))


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


# ---- quantisation ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (5, 17), (3, 300), (130, 256), (2, 127, 136), (2, 2, 129, 144), (257, 4544)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", [ttnn.ROW_MAJOR_LAYOUT, ttnn.TILE_LAYOUT])
def test_quantize_equals_the_definition(dev, shape, rows, dtype, layout):
    g = gen(1, shape, rows)
    x = (torch.randn(*shape, generator=g) * torch.exp(3 * torch.randn(*shape[:-1], 1, generator=g))).to(dtype)
    q = ttnn.quantize_float8(put(x, dev, layout), block_rows=rows)
    codes, scales = ref.quantize(x, rows)
    assert list(q.codes.shape) == list(shape) and list(q.scales.shape) == list(scales.shape)
    assert same_bits(ttnn.to_torch(q.scales), scales)
    assert same_bits(ttnn.to_torch(q.codes), codes)


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_at_every_magnitude(dev, rows, dtype):
    """Quotients are those of a division from the smallest numbers to the largest, zeros of either sign among them, next to borders between two codes too."""
    exponents = torch.arange(-148, 127, 2, dtype=torch.float64)
    x = torch.randn(exponents.numel(), 128, 128, generator=gen(17), dtype=torch.float64).clamp(-3.9, 3.9) * torch.exp2(-10 * torch.rand(128, 128, generator=gen(18), dtype=torch.float64))
    x[:, 0, :] = torch.tensor([448.0, 17.0, 19.0, -21.0, 23.0, 25.0, 27.0, -29.0]).repeat(16) / 448 * 3.5
    x = (x * torch.exp2(exponents)[:, None, None]).float()
    x[:, 1] = torch.nextafter(x[:, 0], torch.tensor(math.inf))
    x[:, 2] = torch.nextafter(x[:, 0], torch.tensor(-math.inf))
    x[:, 3, ::2] = -0.0
    x = x.reshape(-1, 128).to(dtype)
    q = ttnn.quantize_float8(put(x, dev), block_rows=rows)
    codes, scales = ref.quantize(x, rows)
    assert same_bits(ttnn.to_torch(q.scales), scales)
    assert same_bits(ttnn.to_torch(q.codes), codes)


@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_of_special_values(dev, rows):
    x = torch.zeros(128, 6 * 128)
    x[:, 0:128] = 0.0
    x[:, 128:256] = 2.0 ** -140                       # below the least magnitude that counts, subnormal
    x[:, 256:384] = torch.arange(128) * 3.3e38 / 127
    x[3, 256] = -3.3e38
    x[:, 384:512] = 1.0
    x[5, 400] = math.nan
    x[:, 512:640] = 1.0
    x[7, 530] = -math.inf
    x[:, 640:768] = torch.tensor([448.0, 1.0625, 1.1875, 2.0 ** -10, 3 * 2.0 ** -10, -2.0 ** -9, 432.0, -464.0 / 448 * 400]).repeat(16)
    q = ttnn.quantize_float8(put(x, dev), block_rows=rows)
    codes, scales = ttnn.to_torch(q.codes).float(), ttnn.to_torch(q.scales)
    keep = torch.ones(6, dtype=torch.bool)
    keep[3:5] = False
    clean = x.clone()
    clean[:, 384:640] = 0
    wc, ws = ref.quantize(clean, rows)
    assert torch.equal(scales[:, keep], ws[:, keep])
    got, want = codes.view(128, 6, 128)[:, keep], wc.float().view(128, 6, 128)[:, keep]
    assert ((got == want) | (got.isnan() & want.isnan())).all()   # (the third block overflows to infinities from its third column on)
    # a NaN: its own code only, and no part in the scale
    assert torch.isnan(codes[5, 400]) and int(torch.isnan(codes[:, 384:512]).sum()) == 1
    assert (scales[:, 3] == torch.tensor(1.0) / torch.tensor(448.0)).all()
    # an infinity: its block's scale, its own code a NaN, the others zeros
    hit = scales[7 if rows == 1 else 0, 4]
    assert hit == math.inf and torch.isnan(codes[7, 530]) and (codes[7, 531:640] == 0).all()


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("layout", [ttnn.ROW_MAJOR_LAYOUT, ttnn.TILE_LAYOUT])
def test_quantize_bfloat16_rows_with_nan(dev, rows, layout):
    x = torch.randn(128, 384, generator=gen(19)).bfloat16()
    hole = torch.rand(128, 384, generator=gen(20)) < 0.3
    hole[:, 128:256] = True                           # nothing but NaN
    clean = x.masked_fill(hole, 0.0)
    x[hole] = math.nan
    q = ttnn.quantize_float8(put(x, dev, layout), block_rows=rows)
    codes, scales = ref.quantize(clean, rows)
    got = ttnn.to_torch(q.codes).float()
    assert same_bits(ttnn.to_torch(q.scales), scales)
    assert torch.equal(got.isnan(), hole) and torch.equal(got[~hole], codes.float()[~hole])


# ---- linear ----------------------------------------------------------------------------------------------------------------
LINEAR = [(1, 16, 1), (1, 128, 128), (1, 4096, 1024), (2, 144, 130), (7, 256, 8), (8, 400, 129), (9, 2048, 264), (31, 4544, 96), (33, 1024, 1000), (64, 512, 2048),
          (100, 8192, 136), (128, 128, 256), (129, 272, 257), (200, 1024, 512), (257, 640, 384), (350, 4544, 4672), (1025, 256, 520), (2500, 144, 130), (512, 2048, 2048)]


@pytest.mark.parametrize("rows,k,n", LINEAR)
@pytest.mark.parametrize("dtype,bias,act", [("bfloat16", False, None), ("float32", True, "gelu")])
def test_linear_row_major(dev, rows, k, n, dtype, bias, act):
    g = gen(2, rows, k, n)
    x, w = ref.rows_of(g, rows, k), ref.weight(g, n, k)
    b = torch.randn(1, n, generator=g).bfloat16() if bias else None
    y = ttnn.linear_float8(put(x, dev), pair(w, dev), bias=put(b, dev) if bias else None, activation=act, dtype=getattr(ttnn, dtype))
    assert y.layout == ttnn.ROW_MAJOR_LAYOUT and y.dtype == getattr(ttnn, dtype)
    got = ttnn.to_torch(y)
    want, tol = ref.linear(x.cuda(), w[0].cuda(), w[1].cuda(), b.cuda() if bias else None, act, getattr(torch, dtype))
    ref.assert_within(got, want, tol, (rows, k, n))


# one and two weight blocks a tile, tiles that several blocks share and whole ones, rings that go round, in each of the kernels' row ranges
KERNELS = [(1, 8192, 8192), (1, 640, 16384), (3, 18176, 1152), (8, 4544, 18176), (20, 2048, 28672), (32, 8192, 2048), (48, 28672, 512), (64, 1024, 28672), (60, 4096, 1000),
           (128, 18176, 512), (300, 8192, 640), (1500, 1024, 4096), (1280, 8192, 4096), (700, 256, 9000),
           (64, 18272, 6376), (126, 18272, 6376), (97, 9008, 2400)]


@pytest.mark.parametrize("rows,k,n", KERNELS)
@pytest.mark.parametrize("dtype,act", [("bfloat16", "silu"), ("float32", None)])
def test_linear_in_every_kernel(dev, rows, k, n, dtype, act):
    g = torch.Generator(device="cuda").manual_seed(rows + k + n)
    codes = (torch.randn(n, k, generator=g, device="cuda") * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = (torch.rand(ref.blocks(n), ref.blocks(k), generator=g, device="cuda") + 0.5) * (2.0 / 100 / k ** 0.5)
    x = torch.randn(rows, k, generator=g, device="cuda").bfloat16()
    b = torch.randn(1, n, generator=g, device="cuda").bfloat16()
    w = ttnn.Float8Tensor(put(codes.cpu(), dev), put(scales.cpu(), dev))
    xt, bt = put(x.cpu(), dev), put(b.cpu(), dev)
    want, tol = ref.linear(x, codes, scales, b, act, getattr(torch, dtype))
    first = None
    for _ in range(3):   # (what a launch leaves behind must not show in the next)
        y = ttnn.to_torch(ttnn.linear_float8(xt, w, bias=bt, activation=act, dtype=getattr(ttnn, dtype)))
        assert first is None or same_bits(first, y)
        first = y
    ref.assert_within(first, want, tol, (rows, k, n))


def test_linear_many_calls_behind_each_other():
    """Twelve launches of a graph that overlap, each with a weight of its own and more units a block than the ring has stages."""
    c = ref.lib()
    g = torch.Generator(device="cuda").manual_seed(30)
    n = k = 8192
    x = torch.randn(1, k, generator=g, device="cuda").bfloat16()
    ws = [((torch.randn(n, k, generator=g, device="cuda") * 100).clamp(-448, 448).to(torch.float8_e4m3fn), torch.rand(64, 64, generator=g, device="cuda") * 1e-3) for _ in range(4)]
    outs = [torch.empty(1, n, dtype=torch.float32, device="cuda") for _ in range(12)]
    need = c.ttb_linear_float8_workspace_bytes(1, k, n)
    space = torch.zeros(need, dtype=torch.uint8, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())

    def call(i):
        w = ws[i % 4]
        assert c.ttb_linear_float8(x.data_ptr(), w[0].data_ptr(), w[1].data_ptr(), None, outs[i].data_ptr(), 1, 1, k, n, 0, 3 | cabi.MM_WORKSPACE_ZEROED | cabi.MM_WEIGHTS_RESIDENT,
                                   space.data_ptr(), need, s.cuda_stream) == 0
    call(0)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        for i in range(12):
            call(i)
    for _ in range(20):
        graph.replay()
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        want, tol = ref.linear(x, *ws[i % 4], None, None, torch.float32)
        ref.assert_within(out, want, tol, i)
    assert int(space[:65536].count_nonzero()) == 0


def test_linear_between_block_float_linears(dev):
    """Both kinds share the device's scratch, whose counters each leaves at zero."""
    g = gen(31)
    x = ref.rows_of(g, 32, 2048)
    w8 = ref.weight(g, 1024, 2048)
    wb = torch.randn(2048, 4096, generator=g) * 0.02
    xt, f8, bf = put(x, dev, ttnn.TILE_LAYOUT), pair(w8, dev), put(wb, dev, ttnn.TILE_LAYOUT, ttnn.bfloat8_b)
    want, tol = ref.linear(x.cuda(), w8[0].cuda(), w8[1].cuda(), None, None, torch.bfloat16)
    exact = x.double() @ ttnn.to_torch(bf).double()
    near = (x.double().abs() @ wb.double().abs()) * 2.0 ** -7 + 1e-6
    for _ in range(4):
        a, b = ttnn.linear(xt, bf), ttnn.linear_float8(xt, f8)
        assert ((ttnn.to_torch(a).double() - exact).abs() <= near).all()
        ref.assert_within(ttnn.to_torch(b), want, tol)


def test_linear_with_offsets_behind_32_bits(dev):
    """A weight of more than 2^32 codes, and a result of more than 2^31 values."""
    c = ref.lib()
    g = torch.Generator(device="cuda").manual_seed(32)
    n, k = 140000, 32768
    codes = torch.empty(n, k, dtype=torch.float8_e4m3fn, device="cuda")
    for part in codes.split(8192):
        part.copy_((torch.randn(part.shape, generator=g, device="cuda") * 100).clamp_(-448, 448))
    scales = (torch.rand(ref.blocks(n), ref.blocks(k), generator=g, device="cuda") + 0.5) * (2.0 / 100 / k ** 0.5)
    pick = torch.tensor([0, 5, 65535, 131071, 131072, 131100, n - 1], device="cuda")
    for rows in (1, 40):
        x = torch.randn(rows, k, generator=g, device="cuda").bfloat16()
        out = torch.empty(rows, n, dtype=torch.float32, device="cuda")
        ws = _workspace(c.ttb_linear_float8_workspace_bytes(rows, k, n))
        _abi_linear(c, x, codes, scales, out, n, ws, dtype=1)
        w = codes[pick].double() * scales.double()[pick // 128].repeat_interleave(128, 1)
        want, tol = ref.sums(ref.requantized(x), w)
        ref.assert_within(out[:, pick], want, tol + want.abs() * 2.0 ** -23, rows)
    del codes, scales, out
    rows, k, n = 70000, 128, 32768
    x = torch.randn(rows, k, generator=g, device="cuda").bfloat16()
    w = [t.cuda() for t in ref.weight(gen(33), n, k)]
    out = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    _abi_linear(c, x, *w, out, n, _workspace(c.ttb_linear_float8_workspace_bytes(rows, k, n)))
    for r in (0, 32767, 65535, 65536, 69999):
        want, tol = ref.linear(x[r:r + 1], *w, None, None, torch.bfloat16)
        ref.assert_within(out[r:r + 1], want, tol, r)


@pytest.mark.parametrize("shape,n,act,dtype", [((1, 1, 5, 256), 160, None, "bfloat16"), ((2, 3, 33, 80), 70, "silu", "float32"), ((40, 4544), 4672, "relu", "bfloat16"),
                                               ((3, 32, 128), 128, "gelu", "float32"), ((1, 1, 150, 1040), 513, "silu", "bfloat16")])
def test_linear_tiled(dev, shape, n, act, dtype):
    """Tiled tensors of several matrices, row, K and N counts that end inside a tile; the tiles' padding holds NaN and must not show."""
    g = gen(3, shape, n)
    k = shape[-1]
    x, w = ref.rows_of(g, math.prod(shape[:-1]), k).reshape(shape), ref.weight(g, n, k)
    b = torch.randn(1, n, generator=g).bfloat16()
    h, hp, kp = shape[-2], -(-shape[-2] // 32) * 32, -(-k // 32) * 32
    wide = torch.full((*shape[:-2], hp, kp), math.nan, dtype=torch.bfloat16)
    wide[..., :h, :k] = x
    t = put(wide, dev, ttnn.TILE_LAYOUT).reshape(ttnn.Shape(list(shape), [*shape[:-2], hp, kp]))
    y = ttnn.linear_float8(t, pair(w, dev), bias=put(b, dev, ttnn.TILE_LAYOUT), activation=act, dtype=getattr(ttnn, dtype))
    assert list(y.shape) == [*shape[:-1], n] and y.layout == ttnn.TILE_LAYOUT
    got = ttnn.to_torch(y).reshape(-1, n)
    want, tol = ref.linear(x.reshape(-1, k).cuda(), w[0].cuda(), w[1].cuda(), b.cuda(), act, getattr(torch, dtype))
    ref.assert_within(got, want, tol, shape)
    if n % 32 and h % 32 == 0:
        full = ttnn.to_torch(y.reshape(ttnn.Shape(list(y.shape.padded))))
        assert (full[..., n:] == 0).all()


def test_linear_results_repeat_and_rows_are_independent(dev):
    g = gen(4)
    x, w = ref.rows_of(g, 70, 2048), pair(ref.weight(g, 1000, 2048), dev)
    a = ttnn.to_torch(ttnn.linear_float8(put(x, dev), w))
    b = ttnn.to_torch(ttnn.linear_float8(put(x, dev), w))
    assert same_bits(a, b)
    x[11, 5] = math.nan
    x[12, 700] = math.inf
    c = ttnn.to_torch(ttnn.linear_float8(put(x, dev), w))
    assert torch.isnan(c[11]).all() and torch.isnan(c[12]).all()
    keep = [i for i in range(70) if i not in (11, 12)]
    assert same_bits(a[keep], c[keep])


def test_linear_with_quantised_weight_is_near_the_unquantised_one(dev):
    """A chain as a user has it: weight quantised on the device, linear, linear. Each quantisation is off by at most 2^-4 of a value."""
    g = gen(5)
    x, w = torch.randn(64, 512, generator=g).bfloat16(), torch.randn(256, 512, generator=g) / 512 ** 0.5
    q = ttnn.quantize_float8(put(w, dev))
    y = ttnn.to_torch(ttnn.linear_float8(put(x, dev), q, dtype=ttnn.float32)).double()
    want, mag = x.double() @ w.double().T, x.double().abs() @ w.double().abs().T
    # (each factor's value is off by 2^-4 of it, or by half a step of the smallest numbers, 2^-10 of the scale's unit: at most 2^-10 / 448 of the block's largest)
    slack = (2 * 2.0 ** -4 + 2.0 ** -8) * mag + 2.0 ** -10 / 448 * 2 * 512 * x.double().abs().max() * w.double().abs().max()
    assert ((y - want).abs() <= slack).all()


def _abi_linear(c, x, codes, scales, out, n, ws, stream=None, dtype=0):
    rc = c.ttb_linear_float8(x.data_ptr(), codes.data_ptr(), scales.data_ptr(), None, out.data_ptr(), dtype, x.shape[0], x.shape[1], n, 0, 3, ws.data_ptr(), ws.numel(), stream)
    assert rc == 0, c.ttb_last_error()


def _workspace(nbytes):
    return torch.randint(0, 256, (nbytes,), dtype=torch.uint8, device="cuda")   # its contents do not matter


@pytest.mark.parametrize("rows,k,n", [(1, 4096, 1024), (5, 144, 130), (130, 1024, 257)])
def test_linear_leaves_the_memory_around_its_result_alone(rows, k, n):
    c = ref.lib()
    g = gen(6, rows)
    x, w = ref.rows_of(g, rows, k).cuda(), [t.cuda() for t in ref.weight(g, n, k)]
    buf = torch.full((rows * n + 512,), 7.0, dtype=torch.bfloat16, device="cuda")
    need = c.ttb_linear_float8_workspace_bytes(rows, k, n)
    ws = _workspace(need + 4096)
    tail = ws[need:].clone()
    _abi_linear(c, x, *w, buf[256:], n, ws[:need])
    torch.cuda.synchronize()
    assert (buf[:256] == 7).all() and (buf[256 + rows * n:] == 7).all() and torch.equal(ws[need:], tail)
    want, tol = ref.linear(x, *w, None, None, torch.bfloat16)
    ref.assert_within(buf[256:256 + rows * n].view(rows, n), want, tol)


def test_linear_with_an_oddly_aligned_result():
    c = ref.lib()
    g = gen(7)
    x, w = ref.rows_of(g, 40, 256).cuda(), [t.cuda() for t in ref.weight(g, 192, 256)]
    ws = _workspace(c.ttb_linear_float8_workspace_bytes(40, 256, 192))
    for dtype, t in ((0, torch.bfloat16), (1, torch.float32)):
        buf = torch.full((40 * 192 + 16,), 7.0, dtype=t, device="cuda")
        _abi_linear(c, x, *w, buf[1:], 192, ws, dtype=dtype)
        want, tol = ref.linear(x, *w, None, None, t)
        ref.assert_within(buf[1:1 + 40 * 192].view(40, 192), want, tol)
        assert buf[0] == 7 and (buf[1 + 40 * 192:] == 7).all()


def test_linear_on_another_stream_and_in_graphs():
    """Two captured calls with a workspace each, replayed on inputs that changed, and a call on a stream of its own between them."""
    c = ref.lib()
    g = gen(8)
    w = [t.cuda() for t in ref.weight(g, 512, 1024)]
    xs = [ref.rows_of(g, r, 1024).cuda() for r in (3, 200)]
    outs = [torch.empty(x.shape[0], 512, dtype=torch.bfloat16, device="cuda") for x in xs]
    wss = [_workspace(c.ttb_linear_float8_workspace_bytes(x.shape[0], 1024, 512)) for x in xs]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for x, o, ws in zip(xs, outs, wss):
        _abi_linear(c, x, *w, o, 512, ws, s.cuda_stream)   # (and sets the kernels up)
    s.synchronize()
    graphs = []
    for x, o, ws in zip(xs, outs, wss):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            _abi_linear(c, x, *w, o, 512, ws, s.cuda_stream)
    for turn in range(3):
        for x in xs:
            x.copy_(ref.rows_of(gen(9, turn, x.shape[0]), x.shape[0], 1024))
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for q in graphs:
            q.replay()
        torch.cuda.synchronize()
        for x, o in zip(xs, outs):
            want, tol = ref.linear(x, *w, None, None, torch.bfloat16)
            ref.assert_within(o, want, tol, turn)


# ---- router ----------------------------------------------------------------------------------------------------------------
ROUTE = [
    dict(rows=1, e=8, k=2), dict(rows=3, e=64, k=8), dict(rows=5, e=1, k=1), dict(rows=70, e=33, k=32), dict(rows=9, e=1024, k=32, renormalize=False),
    dict(rows=130, e=128, k=6, score="sigmoid"), dict(rows=65, e=60, k=4, score="sigmoid", bias=True, renormalize=False, scale=2.5),
    dict(rows=33, e=256, k=8, score="sigmoid", bias=True, groups=8, top_groups=4, group_score="top2_sum", scale=2.5),
    dict(rows=31, e=96, k=5, groups=32, top_groups=3, renormalize=False), dict(rows=17, e=120, k=3, groups=8, top_groups=2, group_score="top2_sum"),
    dict(rows=40, e=72, k=7, bias=True, groups=2, top_groups=1), dict(rows=12, e=300, k=10, bias=True), dict(rows=6, e=8, k=4, groups=8, top_groups=4, group_score="top2_sum"),
]


def _assert_route(got, want, k):
    w, e = (ttnn.to_torch(t).reshape(-1, k) for t in got)
    assert torch.equal(e, want[1])
    assert ((w.double() - want[0]).abs() <= want[0].abs() * 2.0 ** -23 + 1e-44).all()   # rounded once, what is left of 64 bits beside it


@pytest.mark.parametrize("case", ROUTE)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("masked", [False, True])
def test_route(dev, case, dtype, masked):
    case = dict(case)
    rows, e, k = case.pop("rows"), case.pop("e"), case["k"]
    g = gen(10, rows, e)
    x = (2 * torch.randn(rows, e, generator=g)).to(dtype)      # bfloat16 logits repeat within a row: ties
    if masked:
        x[torch.rand(rows, e, generator=g) < 0.6] = -math.inf
        x[0] = -math.inf
    bias = (torch.randn(e, generator=g) * 0.1) if case.pop("bias", False) else None
    got = ttnn.route_to_experts(put(x, dev), bias=put(bias, dev) if bias is not None else None, **case)
    _assert_route(got, ref.route(x, bias=bias.tolist() if bias is not None else None, **case), k)


def test_route_tiled_logits_of_a_batch(dev):
    g = gen(11)
    x = torch.randn(2, 3, 5, 40, generator=g)
    w, e = ttnn.route_to_experts(put(x, dev, ttnn.TILE_LAYOUT), 4, score="sigmoid")
    assert list(w.shape) == [2, 3, 5, 4] == list(e.shape)
    _assert_route((w, e), ref.route(x.reshape(-1, 40), 4, "sigmoid"), 4)


def test_route_ties_go_to_the_lowest_index(dev):
    x = torch.zeros(4, 64)
    x[1, 40:] = 1.0
    x[2, 5] = x[2, 63] = 3.0
    x[3] = 60.0                                  # sigmoid 1 in 32 bits for these and the next
    x[3, 50] = 61.0
    for score in ("softmax", "sigmoid"):
        e = ttnn.to_torch(ttnn.route_to_experts(put(x, dev), 3, score=score)[1])
        assert e.tolist() == [[0, 1, 2], [40, 41, 42], [5, 63, 0], [50, 0, 1]]
    e = ttnn.to_torch(ttnn.route_to_experts(put(x, dev), 2, groups=4, top_groups=2, group_score="top2_sum")[1])
    assert e.tolist() == [[0, 1], [40, 41], [5, 63], [50, 0]]


def test_route_choice_is_that_of_64_bits(dev):
    """Scores and biases whose sums agree in 32 bits and differ in 64."""
    e = 48
    x = torch.zeros(1, e)
    bias = torch.full((e,), 1.0)
    x[0, 30] = 1e-7                               # sigmoid 0.5 + 2.5e-8: next to 1.0 the step of 32 bits is 1.2e-7
    x[0, 20] = 0.5e-7
    w, i = ttnn.route_to_experts(put(x, dev), 2, score="sigmoid", bias=put(bias, dev))
    assert ttnn.to_torch(i).tolist() == [[30, 20]]


def test_route_of_not_a_number_and_infinity(dev):
    g = gen(12)
    x = torch.randn(6, 40, generator=g)
    x[1, 7] = math.nan
    x[2, :] = math.nan
    x[4, 9] = math.inf
    w, e = (ttnn.to_torch(t) for t in ttnn.route_to_experts(put(x, dev), 3))
    want = ref.route(x[[0, 3, 5]], 3)
    assert torch.equal(e[[0, 3, 5]], want[1]) and torch.allclose(w[[0, 3, 5]].double(), want[0], rtol=1e-6)
    y = x[1].clone()
    y[7] = -math.inf
    assert e[1].tolist() == ref.route(y[None], 3)[1][0].tolist() and torch.isnan(w[1]).all()
    assert e[2].tolist() == [40] * 3 and (w[2] == 0).all()
    assert e[4, 0] == 9 and torch.isnan(w[4]).any()
    bias = torch.zeros(40)
    bias[e[0, 0]] = -math.inf                     # an expert switched off
    e2 = ttnn.to_torch(ttnn.route_to_experts(put(x[:1], dev), 3, bias=put(bias, dev))[1])
    assert int(e[0, 0]) not in e2[0].tolist()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_of_infinity_by_score(dev, score):
    x = torch.randn(3, 40, generator=gen(13))
    x[0, 9] = x[0, 20] = x[2, 39] = math.inf
    w, e = (ttnn.to_torch(t) for t in ttnn.route_to_experts(put(x, dev), 3, score=score, bias=put(torch.zeros(40), dev)))
    assert e[0, :2].tolist() == [9, 20] and e[2, 0] == 39 and (e < 40).all()
    assert torch.isnan(w[[0, 2]]).all() == (score == "softmax") and torch.isfinite(w[1]).all()


def test_route_vanishing_scores(dev):
    x = torch.full((2, 16), -2000.0)
    x[1, 3] = 0.0
    w, e = (ttnn.to_torch(t) for t in ttnn.route_to_experts(put(x, dev), 2, score="sigmoid"))
    assert (w[0] == 0).all() and e[0].tolist() == [0, 1] and w[1].tolist() == [1.0, 0.0] and e[1].tolist() == [3, 0]


# ---- experts ---------------------------------------------------------------------------------------------------------------
def _expert_case(g, rows, e, k, hidden, ffn):
    x = ref.rows_of(g, rows, hidden)
    ws = ref.weight(g, ffn, hidden, (e,)), ref.weight(g, ffn, hidden, (e,)), ref.weight(g, hidden, ffn, (e,))
    logits = torch.randn(rows, e, generator=g) + torch.randn(e, generator=g)
    best, ids = logits.topk(k, -1)
    return x, ws, ids.int(), best.softmax(-1)


EXPERTS = [(1, 1, 1, 16, 16), (1, 8, 2, 256, 128), (1, 64, 8, 2048, 1024), (3, 4, 2, 128, 144), (7, 5, 3, 272, 400), (33, 8, 2, 512, 272), (64, 3, 2, 256, 1200),
           (100, 16, 4, 1040, 256), (130, 2, 1, 144, 384), (257, 4, 2, 640, 512), (300, 100, 8, 128, 128), (1000, 3, 2, 256, 256), (40, 1024, 3, 32, 48),
           (200, 1, 1, 8192, 384), (32, 2, 1, 4096, 512), (90, 2, 1, 512, 8192), (2000, 16, 8, 256, 384)]


@pytest.mark.parametrize("rows,e,k,hidden,ffn", EXPERTS)
def test_experts_mlp(dev, rows, e, k, hidden, ffn):
    x, ws, ids, p = _expert_case(gen(13, rows, e), rows, e, k, hidden, ffn)
    y = ttnn.experts_mlp_float8(put(x, dev), put(ids, dev), put(p, dev), *[pair(w, dev) for w in ws])
    assert y.dtype == ttnn.bfloat16 and list(y.shape) == [rows, hidden]
    want, tol = ref.experts(x.cuda(), ids.cuda(), p.cuda(), *[(a.cuda(), b.cuda()) for a, b in ws])
    ref.assert_within(ttnn.to_torch(y), want, tol, (rows, e))


@pytest.mark.parametrize("act", [None, "relu", "gelu"])
def test_experts_activations(dev, act):
    x, ws, ids, p = _expert_case(gen(14), 50, 4, 2, 256, 256)
    y = ttnn.experts_mlp_float8(put(x, dev), put(ids, dev), put(p, dev), *[pair(w, dev) for w in ws], activation=act)
    want, tol = ref.experts(x.cuda(), ids.cuda(), p.cuda(), *[(a.cuda(), b.cuda()) for a, b in ws], act=act)
    ref.assert_within(ttnn.to_torch(y), want, tol, act)


@pytest.mark.parametrize("kind", ["none", "one", "all_to_last", "twice", "outside", "negative_weights"])
def test_experts_with_unusual_routes(dev, kind):
    rows, e, k, hidden, ffn = 90, 6, 3, 256, 384
    x, ws, ids, p = _expert_case(gen(15, kind), rows, e, k, hidden, ffn)
    if kind == "none":
        ids[:] = e
    elif kind == "one":
        ids[:], ids[41, 1] = e, 2
    elif kind == "all_to_last":
        ids[:], ids[:, 0] = e, e - 1
    elif kind == "twice":
        ids[:, 1] = ids[:, 0]                    # the same expert in two places of a row counts twice
    elif kind == "outside":
        ids[::3] = -1
        ids[1::3, 0] = 1 << 30
        ids[5] = -(1 << 31)
    else:
        p = p - 0.5
    y = ttnn.to_torch(ttnn.experts_mlp_float8(put(x, dev), put(ids, dev), put(p, dev), *[pair(w, dev) for w in ws]))
    want, tol = ref.experts(x.cuda(), ids.cuda(), p.cuda(), *[(a.cuda(), b.cuda()) for a, b in ws])
    ref.assert_within(y, want, tol, kind)
    empty = ((ids < 0) | (ids >= e)).all(1)
    assert (y[empty] == 0).all()


def test_experts_tiled_batch(dev):
    """Tiled activations of several matrices; padding of the input's tiles holds NaN, that of the result's zeros."""
    shape, e, k, ffn = (2, 2, 5, 272), 4, 2, 144
    x, ws, ids, p = _expert_case(gen(16), 20, e, k, 272, ffn)
    wide = torch.full((2, 2, 32, 288), math.nan, dtype=torch.bfloat16)
    wide[..., :5, :272] = x.reshape(shape)
    t = put(wide, dev, ttnn.TILE_LAYOUT).reshape(ttnn.Shape(list(shape), [2, 2, 32, 288]))
    y = ttnn.experts_mlp_float8(t, put(ids.reshape(2, 2, 5, k), dev), put(p.reshape(2, 2, 5, k), dev), *[pair(w, dev) for w in ws])
    assert list(y.shape) == list(shape) and list(y.shape.padded) == [2, 2, 32, 288]
    want, tol = ref.experts(x.cuda(), ids.cuda(), p.cuda(), *[(a.cuda(), b.cuda()) for a, b in ws])
    ref.assert_within(ttnn.to_torch(y).reshape(20, 272), want, tol)
    full = ttnn.to_torch(y.reshape(ttnn.Shape([2, 2, 32, 288])))
    assert (full[..., 5:, :] == 0).all() and (full[..., 272:] == 0).all()


def test_experts_results_repeat_and_rows_are_independent(dev):
    x, ws, ids, p = _expert_case(gen(17), 120, 5, 2, 512, 256)
    args = [put(ids, dev), put(p, dev)] + [pair(w, dev) for w in ws]
    a = ttnn.to_torch(ttnn.experts_mlp_float8(put(x, dev), *args))
    b = ttnn.to_torch(ttnn.experts_mlp_float8(put(x, dev), *args))
    assert same_bits(a, b)
    x[33, 100] = math.nan
    c = ttnn.to_torch(ttnn.experts_mlp_float8(put(x, dev), *args))
    assert torch.isnan(c[33]).all()
    keep = [i for i in range(120) if i != 33]
    assert same_bits(a[keep], c[keep])


def test_experts_in_graphs_whose_routes_change():
    """Two captured calls with a workspace each; the expert indexes change between replays, so that every size of run occurs."""
    c = ref.lib()
    rows, e, k, hidden, ffn = 150, 7, 2, 256, 256
    x, ws, ids, p = _expert_case(gen(18), rows, e, k, hidden, ffn)
    ws = [(a.cuda(), b.cuda()) for a, b in ws]
    need = c.ttb_experts_mlp_float8_workspace_bytes(rows, e, k, hidden, ffn)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    calls = []
    for j in range(2):
        t = dict(x=x.cuda(), ids=ids.cuda(), p=p.cuda(), out=torch.empty(rows, hidden, dtype=torch.bfloat16, device="cuda"), ws=_workspace(need))

        def call(t=t):
            rc = c.ttb_experts_mlp_float8(t["x"].data_ptr(), t["ids"].data_ptr(), t["p"].data_ptr(), *[q.data_ptr() for w in ws for q in w], t["out"].data_ptr(), 1, rows, e, k,
                                          hidden, ffn, 3, 3, t["ws"].data_ptr(), need, s.cuda_stream)
            assert rc == 0, c.ttb_last_error()
        torch.cuda.synchronize()
        call()
        s.synchronize()
        t["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(t["graph"], stream=s):
            call()
        calls.append(t)
    for turn in range(4):
        g = gen(19, turn)
        for j, t in enumerate(calls):
            new = torch.randint(0, e + 1, (rows, k), generator=g) if turn != 2 else torch.full((rows, k), (turn + j) % e)
            t["ids"].copy_(new.int())
            t["x"].copy_(ref.rows_of(g, rows, hidden))
        torch.cuda.synchronize()
        for t in calls:
            t["graph"].replay()
        torch.cuda.synchronize()
        for t in calls:
            want, tol = ref.experts(t["x"], t["ids"], t["p"], *ws)
            ref.assert_within(t["out"], want, tol, turn)


def test_router_and_experts_together(dev):
    """A mixture-of-experts layer as a model runs it: router logits from a linear, routes, experts, with the last rows a batch's padding."""
    g = gen(20)
    rows, e, k, hidden, ffn = 75, 12, 3, 512, 384
    x, ws, _, _ = _expert_case(g, rows, e, k, hidden, ffn)
    router = (torch.randn(hidden, e, generator=g) / hidden ** 0.5).bfloat16()
    xt = put(x, dev, ttnn.TILE_LAYOUT)
    logits = ttnn.to_torch(ttnn.linear(xt, put(router, dev, ttnn.TILE_LAYOUT), dtype=ttnn.float32))
    logits[-5:] = -math.inf
    bias = torch.randn(e, generator=g) * 0.05
    p, ids = ttnn.route_to_experts(put(logits, dev, ttnn.TILE_LAYOUT), k, score="sigmoid", bias=put(bias, dev), groups=4, top_groups=2, group_score="top2_sum")
    y = ttnn.to_torch(ttnn.experts_mlp_float8(xt, ids, p, *[pair(w, dev) for w in ws]))
    wp, wi = ref.route(logits, k, "sigmoid", bias.tolist(), 4, 2, "top2_sum")
    assert torch.equal(ttnn.to_torch(ids), wi)
    want, tol = ref.experts(x.cuda(), wi.cuda(), wp.float().cuda(), *[(a.cuda(), b.cuda()) for a, b in ws])
    ref.assert_within(y, want, tol + want.abs() * 2.0 ** -22)
    assert (y[-5:] == 0).all()


def test_surface_refusals(dev):
    x = put(torch.zeros(4, 256).bfloat16(), dev)
    w = pair(ref.weight(gen(21), 128, 256), dev)
    f32 = put(torch.zeros(4, 256), dev)
    i, p = put(torch.zeros(4, 2, dtype=torch.int32), dev), put(torch.zeros(4, 2), dev)
    ew, dw = pair(ref.weight(gen(22), 128, 256, (3,)), dev), pair(ref.weight(gen(23), 256, 128, (3,)), dev)
    bad = [
        (lambda: ttnn.quantize_float8(i), "float32 or bfloat16"), (lambda: ttnn.quantize_float8(x, block_rows=32), "block_rows"),
        (lambda: ttnn.quantize_float8(put(torch.zeros(4).bfloat16(), dev)), "rank 2, 3 or 4"),
        (lambda: ttnn.linear_float8(f32, w), "bfloat16"), (lambda: ttnn.linear_float8(put(torch.zeros(4, 128).bfloat16(), dev), w), "width"),
        (lambda: ttnn.linear_float8(x, w, dtype=ttnn.bfloat8_b), "bfloat16 or float32"), (lambda: ttnn.linear_float8(x, w, activation="tanh"), "activation"),
        (lambda: ttnn.linear_float8(x, (w.scales, w.codes)), "float8_e4m3"), (lambda: ttnn.linear_float8(x, (w.codes, x)), "float32"),
        (lambda: ttnn.linear_float8(x, (w.codes, put(torch.ones(1, 3), dev))), "128 x 128"), (lambda: ttnn.linear_float8(x, (w.codes, put(torch.ones(2), dev))), "same rank"),
        (lambda: ttnn.linear_float8(x, w, bias=put(torch.zeros(1, 64).bfloat16(), dev)), "bias"), (lambda: ttnn.linear_float8(x, w, bias=put(torch.zeros(1, 128), dev)), "bias"),
        (lambda: ttnn.linear_float8(x, ew), "one matrix"), (lambda: ttnn.route_to_experts(i, 1), "float32 or bfloat16"),
        (lambda: ttnn.route_to_experts(p, 0), "k must be"), (lambda: ttnn.route_to_experts(p, 3), "k must be"), (lambda: ttnn.route_to_experts(p, 1, score="relu"), "score"),
        (lambda: ttnn.route_to_experts(p, 1, group_score="mean"), "group_score"), (lambda: ttnn.route_to_experts(p, 1, bias=put(torch.zeros(3), dev)), "bias"),
        (lambda: ttnn.experts_mlp_float8(x, p, p, ew, ew, dw), "uint32"), (lambda: ttnn.experts_mlp_float8(x, i, put(torch.zeros(4, 3), dev), ew, ew, dw), "rows, k"),
        (lambda: ttnn.experts_mlp_float8(x, put(torch.zeros(3, 2, dtype=torch.int32), dev), put(torch.zeros(3, 2), dev), ew, ew, dw), "rows, k"),
        (lambda: ttnn.experts_mlp_float8(x, i, p, ew, w, dw), "same shape"), (lambda: ttnn.experts_mlp_float8(x, i, p, ew, ew, ew), "hidden"),
        (lambda: ttnn.experts_mlp_float8(f32, i, p, ew, ew, dw), "bfloat16"), (lambda: ttnn.experts_mlp_float8(x, i, p, ew, ew, dw, activation="tanh"), "activation"),
    ]
    for call, text in bad:
        with pytest.raises(RuntimeError, match=text):
            call()
