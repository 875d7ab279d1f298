"""float8 operators where their contract is easy to miss: codes of the experts' inner quantisation, rows that are not finite under activations and in the
padding of tiled results, saturated router scores."""
import ctypes
import math

import pytest
import torch

import cabi
import float8_ref as ref
import ttnn
from test_matmul_gpu import make_case
from test_float8_gpu import dev, no_wait_ran_out, pair, put, same_bits  # noqa: F401  (fixtures among them)

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- the experts' inner quantisation ---------------------------------------------------------------------------------------
def _products():
    """Gate and up codes [256, 127] whose products are exact in 32 bits, and their quotients' codes by division and by a rounded reciprocal."""
    g = gen(1)
    gate, up = ((torch.randn(256, 127, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn) for _ in range(2))
    h = (gate.float() * up.float()).T.contiguous()
    codes, scales = ref.quantize(h, 1)
    by_reciprocal = (h * ref.spread(torch.ones_like(scales) / scales, 1, *h.shape)).clamp(-448, 448).to(torch.float8_e4m3fn)
    differ = (codes.view(torch.uint8) != by_reciprocal.view(torch.uint8)).any(1)
    order = torch.argsort(differ.int(), descending=True, stable=True)   # the rows that tell the two apart first
    return gate[:, order], up[:, order], h[order], int(differ.sum())


@pytest.mark.parametrize("rows", [3, 20, 50, 100])
@pytest.mark.parametrize("act", [None, "relu"])
def test_experts_inner_codes_are_those_of_the_quantiser(dev, rows, act):
    """Every number up to the quantisation is exact (a row of x picks a column of the weights), the down weight is a unit matrix: the result is code * scale."""
    gate, up, h, telling = _products()
    assert telling >= 3
    x = torch.zeros(rows, 256)
    x[torch.arange(rows), torch.arange(rows)] = 256.0   # a code of its own, as the row's scale is 1:
    x[:, 127] = 448.0
    wide = [torch.cat([w.view(torch.uint8), torch.zeros(256, 129, dtype=torch.uint8)], 1).view(torch.float8_e4m3fn)[None] for w in (gate, up)]
    scale = torch.full((1, 2, 2), 2.0 ** -8)
    down = torch.eye(256)[None].to(torch.float8_e4m3fn), torch.ones(1, 2, 2)
    ids, p = torch.zeros(rows, 1, dtype=torch.int32), torch.ones(rows, 1)
    y = ttnn.experts_mlp_float8(put(x.bfloat16(), dev), put(ids, dev), put(p, dev), pair((wide[0], scale), dev), pair((wide[1], scale), dev), pair(down, dev), activation=act)
    h = h[:rows] if act is None else torch.relu(gate.float().T[:rows]) * up.float().T[:rows]
    codes, scales = ref.quantize(h, 1)
    want = (codes.float() * ref.spread(scales, 1, *h.shape)).bfloat16()
    assert torch.equal(ttnn.to_torch(y).float(), want.float())


# ---- calls right behind the one that writes their weight -------------------------------------------------------------------
@pytest.mark.parametrize("rows", [1, 5, 40, 200])
def test_linear_right_behind_its_weights_quantiser(dev, rows):
    """Nothing between the two calls; the codes lie where another weight's were the call before."""
    g = gen(4)
    n, k = 2048, 4096
    x = ref.rows_of(g, rows, k)
    ws = [torch.randn(n, k, generator=g) * s for s in (0.02, 0.5, 0.001)]
    xt, wts = put(x, dev), [put(w, dev) for w in ws]
    want = [ref.linear(x.cuda(), *(t.cuda() for t in ref.quantize(w, 128)), None, None, torch.bfloat16) for w in ws]
    for turn in range(6):
        q = ttnn.quantize_float8(wts[turn % 3])
        y = ttnn.linear_float8(xt, q)
        del q
        ref.assert_within(ttnn.to_torch(y), *want[turn % 3], turn)


# ---- waits that are bounded ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,k,n", [(5120, 8192, 28672), (32, 8192, 148 * 15 * 256 + 50 * 256), (64, 8192, 148 * 15 * 256 + 50 * 256)])
def test_a_launch_longer_than_the_wait_limit_is_no_timeout(rows, k, n):
    """Rounds of whole tiles that take longer than the shortest limit, about half a millisecond, and then 40 to 50 tiles that several blocks share, most blocks two of
    them. The limit is for a step of a launch, not for all of it."""
    c = ref.lib()
    g = torch.Generator(device="cuda").manual_seed(5)
    codes = torch.empty(n, k, dtype=torch.float8_e4m3fn, device="cuda")
    for part in codes.split(16384):
        part.copy_((torch.randn(part.shape, generator=g, device="cuda") * 100).clamp_(-448, 448))
    scales = (torch.rand(ref.blocks(n), ref.blocks(k), generator=g, device="cuda") + 0.5) * (2.0 / 100 / k ** 0.5)
    x = torch.randn(rows, k, generator=g, device="cuda").bfloat16()
    out = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    need = c.ttb_linear_float8_workspace_bytes(rows, k, n)
    space = torch.zeros(need, dtype=torch.uint8, device="cuda")

    def call():
        assert c.ttb_linear_float8(x.data_ptr(), codes.data_ptr(), scales.data_ptr(), None, out.data_ptr(), 0, rows, k, n, 0, 3 | cabi.MM_WORKSPACE_ZEROED, space.data_ptr(), need,
                                   torch.cuda.current_stream().cuda_stream) == 0
    call()
    lib = cabi.load()
    lib.check(lib.set_wait_limit_cycles(1))
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    try:
        start.record()
        call()
        end.record()
        torch.cuda.synchronize()
    finally:
        lib.check(lib.set_wait_limit_cycles(0))
    assert lib.check_status(None) == 0
    assert start.elapsed_time(end) > 0.6
    pick = torch.cat([torch.arange(0, n, n // 37, device="cuda"), torch.arange(n - 130, n, device="cuda")])   # (the shared tiles come last)
    few = torch.arange(0, rows, max(1, rows // 40), device="cuda")
    w = codes[pick].double() * scales.double()[pick // 128].repeat_interleave(128, 1)
    want, tol = ref.sums(ref.requantized(x[few]), w)
    ref.assert_within(out[few][:, pick], want, tol + (want.abs() + tol) * 2.0 ** -8, (rows, n))
    assert int(space[:65536].count_nonzero()) == 0


# ---- rows that are not finite ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("rows,k,n", [(5, 256, 200), (30, 400, 130), (50, 8192, 256), (100, 256, 264), (90, 8192, 130)])
def test_linear_keeps_nan_under_every_activation(dev, act, rows, k, n):
    g = gen(2)
    x, w = ref.rows_of(g, rows, k), pair(ref.weight(g, n, k), dev)
    b = put(torch.randn(1, n, generator=g).bfloat16(), dev)
    clean = ttnn.to_torch(ttnn.linear_float8(put(x, dev), w, bias=b, activation=act))
    x[1, 7], x[4, k - 1] = math.nan, math.inf
    y = ttnn.to_torch(ttnn.linear_float8(put(x, dev), w, bias=b, activation=act))
    assert torch.isnan(y[[1, 4]]).all()
    keep = [i for i in range(rows) if i not in (1, 4)]
    assert same_bits(y[keep], clean[keep]) and torch.isfinite(clean).all()


@pytest.mark.parametrize("rows", [3, 20, 50, 100])
def test_experts_keep_nan_under_relu(dev, rows):
    g = gen(6)
    x = ref.rows_of(g, rows, 256)
    x[1, 7], x[2, 200] = math.nan, math.inf
    ws = [pair(ref.weight(g, 256, 256, (1,)), dev) for _ in range(3)]
    y = ttnn.to_torch(ttnn.experts_mlp_float8(put(x, dev), put(torch.zeros(rows, 1, dtype=torch.int32), dev), put(torch.ones(rows, 1), dev), *ws, activation="relu"))
    assert torch.isnan(y[[1, 2]]).all() and torch.isfinite(y[[i for i in range(rows) if i not in (1, 2)]]).all()


@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows,k,n", [(32, 256, 70), (32, 8192, 130), (64, 512, 513), (160, 1024, 150), (96, 8192, 257)])
def test_linear_columns_that_only_pad_are_zero(dev, rows, k, n, dtype, act):
    """... in rows of NaN and infinities too, whose products with the zeros behind the weight's last row are not zero."""
    g = gen(3)
    x, w = ref.rows_of(g, rows, k), pair(ref.weight(g, n, k), dev)
    x[1, 7], x[20, k - 1], x[31] = math.nan, math.inf, -math.inf
    for b in (None, put(torch.randn(1, n, generator=g).bfloat16(), dev, ttnn.TILE_LAYOUT)):
        y = ttnn.linear_float8(put(x, dev, ttnn.TILE_LAYOUT), w, bias=b, activation=act, dtype=getattr(ttnn, dtype))
        full = ttnn.to_torch(y.reshape(ttnn.Shape(list(y.shape.padded))))
        assert full.shape[-1] > n and (full[:, n:] == 0).all()
        assert torch.isfinite(full[[0, 2, 21, 30]]).all()


# ---- the router's order where scores saturate ------------------------------------------------------------------------------
@pytest.mark.parametrize("score,logits", [("sigmoid", [60.0, 62.0, 61.0, 62.0, 0.0, 59.0, 60.0, 63.0]), ("softmax", [0.0, -900.0, -800.0, -900.0, -1000.0, -800.0, -850.0, -950.0])])
def test_route_order_of_saturated_scores(dev, score, logits):
    """By the logits without bias and group sums, though the 64-bit scores of most of these are equal; else by the 64-bit scores, ties to the lowest index."""
    x = torch.tensor([logits], dtype=torch.double)
    s = torch.sigmoid(x) if score == "sigmoid" else torch.softmax(x, -1)
    by_logit, by_score = (sorted(range(8), key=lambda i: (-v[0, i].item(), i)) for v in (x, s))
    assert by_logit != by_score
    t = put(x.float(), dev)

    def ids(**kw):
        return ttnn.to_torch(ttnn.route_to_experts(t, 8, score=score, **kw)[1])[0].tolist()
    assert ids() == by_logit == ids(groups=2, top_groups=2)
    assert ids(bias=put(torch.zeros(8), dev)) == by_score == ids(groups=2, top_groups=2, group_score="top2_sum")


# ---- unusual routes, with inputs that are the same in every run ------------------------------------------------------------
@pytest.mark.parametrize("seed,kind", list(enumerate(["none", "one", "all_to_last", "twice", "outside", "negative_weights"])))
@pytest.mark.parametrize("rows", [5, 90, 400])
def test_experts_with_unusual_routes_of_fixed_seeds(dev, rows, seed, kind):
    g = gen(100 * rows + seed)
    e, k, hidden, ffn = 6, 3, 256, 384
    x, ws = ref.rows_of(g, rows, hidden), [ref.weight(g, *s, (e,)) for s in ((ffn, hidden), (ffn, hidden), (hidden, ffn))]
    best, ids = (torch.randn(rows, e, generator=g) + torch.randn(e, generator=g)).topk(k, -1)
    ids, p = ids.int(), best.softmax(-1)
    if kind == "none":
        ids[:] = e
    elif kind == "one":
        ids[:], ids[rows // 2, 1] = e, 2
    elif kind == "all_to_last":
        ids[:], ids[:, 0] = e, e - 1
    elif kind == "twice":
        ids[:, 1] = ids[:, 0]
    elif kind == "outside":
        ids[::3], ids[1::3, 0], ids[2] = -1, 1 << 30, -(1 << 31)
    else:
        p = p - 0.5
    y = ttnn.to_torch(ttnn.experts_mlp_float8(put(x, dev), put(ids, dev), put(p, dev), *[pair(w, dev) for w in ws]))
    want, tol = ref.experts(x.cuda(), ids.cuda(), p.cuda(), *[(a.cuda(), b.cuda()) for a, b in ws])
    ref.assert_within(y, want, tol, kind)
    assert (y[((ids < 0) | (ids >= e)).all(1)] == 0).all()


# ---- behind a wait that ran out --------------------------------------------------------------------------------------------
def _peer_matmul_that_waits_in_vain(lib, orc, workspace):
    """A block-float matmul whose activations other GPUs never deliver, on the workspace; it gives up at the limit of its launch."""
    x, w, _ = make_case(lib, orc, 18, 32, 4096, 512, cabi.BFLOAT8_B)
    a, out = lib.tilize(x.cuda(), 1, 32, 4096), torch.zeros(32 * 512, dtype=torch.bfloat16, device="cuda")
    counters = torch.zeros(64, dtype=torch.int32, device="cuda")
    counters[32] = 1
    torch.cuda.synchronize()
    wait = cabi.peer_wait(counters.data_ptr(), counters.data_ptr() + 128)

    def call():
        lib.check(lib.cdll.ttb_matmul_peer(a.data_ptr(), cabi.BFLOAT16, w.data_ptr(), cabi.BFLOAT8_B, None, out.data_ptr(), cabi.BFLOAT16, 1, 32, 4096, 512, 0,
                                           cabi.MM_WORKSPACE_ZEROED, workspace.data_ptr(), workspace.numel(), None, ctypes.byref(wait), None))
    call.keep = a, out, counters, w
    return call


@pytest.mark.parametrize("rows", [1, 40, 200])
def test_linear_behind_a_kernel_that_waits_for_peers(ttb, orc, rows):
    """The kernel in front waits 1.3 s and gives up; the float8 kernels, which start while it waits, do not count that time under their limit of about a second."""
    c = ref.lib()
    g = gen(7)
    x, w = ref.rows_of(g, rows, 2048).cuda(), [t.cuda() for t in ref.weight(g, 1000, 2048)]
    need = c.ttb_linear_float8_workspace_bytes(rows, 2048, 1000)
    spaces = [torch.zeros(max(need, 65536 + (48 << 20)), dtype=torch.uint8, device="cuda") for _ in range(2)]
    out = torch.zeros(rows, 1000, dtype=torch.float32, device="cuda")

    def linear(space, flags):
        assert c.ttb_linear_float8(x.data_ptr(), w[0].data_ptr(), w[1].data_ptr(), None, out.data_ptr(), 1, rows, 2048, 1000, 0, 3 | flags, space.data_ptr(), need, None) == 0
    linear(spaces[0], cabi.MM_WORKSPACE_ZEROED)
    assert ttb.check_status(None) == 0
    want, tol = ref.linear(x, *w, None, None, torch.float32)
    ref.assert_within(out, want, tol)
    out.zero_()
    wait = _peer_matmul_that_waits_in_vain(ttb, orc, spaces[1])
    ttb.check(ttb.set_wait_limit_cycles(2_600_000_000))
    try:
        wait()
    finally:
        ttb.check(ttb.set_wait_limit_cycles(0))
    linear(spaces[0], cabi.MM_WORKSPACE_ZEROED | cabi.MM_WEIGHTS_RESIDENT)
    assert ttb.check_status(None) == -5
    assert int(ttb.cdll.ttb_last_error().decode().split("wait site ")[1].rstrip(")")) < 40   # (the kernel in front)
    assert ttb.check_status(None) == 0
    ref.assert_within(out, want, tol)
    # the workspace that the matmul gave up on: trusted again once its head is clear, or by a call that clears the counters itself
    for flags in (0, cabi.MM_WORKSPACE_ZEROED):
        out.zero_()
        if flags:
            spaces[1][: 65536 + (16 << 20)].zero_()
        linear(spaces[1], flags)
        ref.assert_within(out, want, tol)
    assert ttb.check_status(None) == 0


def test_surface_linear_after_a_timeout(ttb, orc, dev):
    """The host layer raises once and clears its scratch; the next linear is right."""
    g = gen(8)
    x, w = ref.rows_of(g, 40, 8192), ref.weight(g, 1000, 8192)
    xt, wt = put(x, dev), pair(w, dev)
    want, tol = ref.linear(x.cuda(), w[0].cuda(), w[1].cuda(), None, None, torch.bfloat16)
    ref.assert_within(ttnn.to_torch(ttnn.linear_float8(xt, wt)), want, tol)
    space = torch.zeros(65536 + (48 << 20), dtype=torch.uint8, device="cuda")
    wait = _peer_matmul_that_waits_in_vain(ttb, orc, space)
    ttb.check(ttb.set_wait_limit_cycles(2_000_000))
    try:
        wait()
    finally:
        ttb.check(ttb.set_wait_limit_cycles(0))
    with pytest.raises(RuntimeError, match="ran out"):
        ttnn.synchronize_device(dev)
    for _ in range(2):
        ref.assert_within(ttnn.to_torch(ttnn.linear_float8(xt, wt)), want, tol)
