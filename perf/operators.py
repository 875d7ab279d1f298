"""The float8 and mixture-of-experts operators as a user's program runs them, beside their plain form in elementary torch operations.

listed() names the cases, draw() makes more of the same ranges, prepare() makes what a program holds before the call, run() is one pass, work() the bytes
and operations a pass cannot do without, exact() the results in 64 bits.

float8 numbers are e4m3 (largest value 448). A weight is codes [N, K], K contiguous, with one fp32 scale for every 128 x 128 block; activations are bfloat16
and are quantised within the call, with one scale for 128 values of a row."""
import math
import os
import sys

import torch

own = False
BLOCK, TOP, LEAST = 128, 448.0, 2.0 ** -100   # an all but empty block counts as one whose largest value is LEAST


def up(v, m):
    return (v + m - 1) // m * m


# ---- the cases -----------------------------------------------------------------------------------------------------------
def _linear(name, rows, k, n, bias=False, activation="", out="bfloat16", layout="row_major"):
    c = {"path": "linear", "rows": rows, "k": k, "n": n, "bias": bias, "activation": activation, "out": out, "layout": layout}
    return dict(c, name=name) if name else c


def _route(name, rows, experts, k, score, bias=False, groups=1, top_groups=1, group_score="max", renormalize=True, scale=1.0, masked=0, dtype="float32"):
    c = {"path": "route", "rows": rows, "experts": experts, "k": k, "score": score, "bias": bias, "groups": groups, "top_groups": top_groups,
         "group_score": group_score, "renormalize": renormalize, "scale": scale, "masked": masked, "dtype": dtype}
    return dict(c, name=name) if name else c


def _quantize(name, rows, cols, block_rows, dtype):
    c = {"path": "quantize", "rows": rows, "cols": cols, "block_rows": block_rows, "dtype": dtype}
    return dict(c, name=name) if name else c


def _experts(name, rows, experts, k, hidden, ffn, padding=0):
    c = {"path": "experts", "rows": rows, "experts": experts, "k": k, "hidden": hidden, "ffn": ffn, "padding": padding}
    return dict(c, name=name) if name else c


def listed():
    return [
        # The router of one token: latency only.
        _route("route_one_token", 1, 64, 8, "softmax"),
        # The router of a long prompt: sigmoid scores with a balance bias, groups of experts, some experts masked off.
        _route("route_prompt_8191", 8191, 128, 6, "sigmoid", bias=True, groups=8, top_groups=4, group_score="top2_sum", scale=2.0, masked=3),
        # A weight on its way to the device format, the tensor of the conversion benchmark.
        _quantize("quantize_weight_4096", 4096, 4096, 128, "float32"),
        # Activations on their way to 8 bits: ragged rows, Falcon-7B's width, whose last block holds 64 columns.
        _quantize("quantize_rows_350", 350, 4544, 1, "bfloat16"),
        # One token through a small projection: latency.
        _linear("linear_one_token", 1, 4096, 1024),
        # A decode batch of 32 through the Llama-2-70B gate projection: bound by the weight's bytes. Tiled, as it follows other linears.
        _linear("linear_decode_llama_mlp", 32, 8192, 28672, layout="tile"),
        # A short prompt through Falcon-7B's fused q/k/v projection: ragged rows, half a block at the end of both axes of the weight.
        _linear("linear_350_falcon_qkv", 350, 4544, 4672, bias=True, activation="gelu", out="float32"),
        # Prefill: the Llama-2-70B MLP shape of the benchmark, compute bound.
        _linear("linear_prefill_llama_mlp", 2048, 8192, 28672),
        # One token through eight of 64 small experts: latency.
        _experts("experts_one_token", 1, 64, 8, 2048, 1024),
        # A decode batch of 32 through eight experts of Mistral-7B's MLP size, two for a token: bound by the weights' bytes.
        _experts("experts_decode_mistral", 32, 8, 2, 4096, 14336),
        # A batch of ragged size whose last rows are padding (no expert), sixteen experts whose sizes end inside a block.
        _experts("experts_ragged_333", 333, 16, 4, 4544, 1200, padding=13),
        # A prompt through the same experts as the decode batch: compute bound.
        _experts("experts_prefill_mistral", 2048, 8, 2, 4096, 14336),
    ]


def _log(rng, low, high):
    return low * (high / low) ** rng.random()


def _size(rng, low, high, step):
    """Log-uniform; half of them whole blocks of 128, the others multiples of `step`."""
    s = rng.choice([128, step])
    return int(min(up(high, s), max(up(low, s), round(_log(rng, low, high) / s) * s)))


def draw(rng):
    path = rng.choice(["route", "quantize", "linear", "linear", "linear", "experts", "experts", "experts"])
    if path == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * rng.choice([4, 8, 15, 16, 32]) if groups > 1 else rng.randint(8, 256)
        bias = rng.random() < 0.5
        top = rng.randint(max(1, groups // 2), groups)
        k = rng.randint(1, min(8, max(1, experts * top // groups)))
        return _route(None, int(round(_log(rng, 1, 8192))), experts, k, rng.choice(["softmax", "sigmoid"]), bias, groups, top,
                      rng.choice(["max", "top2_sum"]), rng.random() < 0.7, rng.choice([1.0, 2.0]), rng.choice([0, 0, 3]), rng.choice(["float32", "bfloat16"]))
    if path == "quantize":
        return _quantize(None, int(round(_log(rng, 1, 8192))), _size(rng, 128, 8192, 16), rng.choice([1, 128]), rng.choice(["float32", "bfloat16"]))
    if path == "linear":
        while True:
            rows = int(round(_log(rng, 1, 2048)))
            k, n = _size(rng, 256, 28672, 16), _size(rng, 256, 28672, 8)
            layout = rng.choice(["row_major", "tile"]) if n % 32 == 0 and k % 32 == 0 else "row_major"
            if rows * k * n <= 2048 * 8192 * 28672 and k * n <= 8192 * 28672:
                return _linear(None, rows, k, n, rng.random() < 0.4, rng.choice(["", "", "relu", "gelu", "silu"]), rng.choice(["bfloat16"] * 4 + ["float32"]), layout)
    while True:
        experts = rng.choice([4, 8, 16, 32, 64, 128])
        rows, k = int(round(_log(rng, 1, 2048))), rng.randint(1, 8)
        hidden, ffn = _size(rng, 512, 8192, 16), _size(rng, 256, 14336, 16)
        # (the plain form takes every row through every expert)
        if k <= experts and rows * experts * hidden * ffn <= 2048 * 8 * 4096 * 14336 and experts * hidden * ffn <= 8 * 4096 * 14336 and rows * experts * ffn <= 1 << 28:
            return _experts(None, rows, experts, k, hidden, ffn, rng.choice([0, 0, min(rows // 2, 9)]))


# ---- inputs --------------------------------------------------------------------------------------------------------------
def _weight(g, n, k, lead=()):
    """Codes and scales as a checkpoint holds them: normal values whose largest one of a block is near 448."""
    codes = torch.empty(*lead, n, k, dtype=torch.float8_e4m3fn, device="cuda")
    for c in codes.view(-1, k).split(8192):
        c.copy_(torch.randn(c.shape, generator=g, device="cuda").mul_(100).clamp_(-TOP, TOP))
    scales = torch.rand(*lead, up(n, BLOCK) // BLOCK, up(k, BLOCK) // BLOCK, generator=g, device="cuda").add_(0.5).mul_(2.0 / 100 / math.sqrt(k))
    return codes, scales


def _activation(g, rows, k):
    """Rows of normal values with a few large columns, as the inputs of linears are."""
    x = torch.randn(rows, k, generator=g, device="cuda")
    return (x * (1 + 15 * (torch.rand(k, generator=g, device="cuda") < 0.01))).bfloat16()


def prepare(case, seed):
    torch.cuda.set_device(0)
    g = torch.Generator(device="cuda").manual_seed(seed)
    s, path = dict(case), case["path"]
    if path == "linear":
        x = _activation(g, case["rows"], case["k"])
        s["x"] = _tiled(x, up(case["rows"], 32)) if case["layout"] == "tile" else x
        s["w"] = _weight(g, case["n"], case["k"])
        s["b"] = torch.randn(case["n"], generator=g, device="cuda").bfloat16() if case["bias"] else None
    elif path == "route":
        x = torch.randn(case["rows"], case["experts"], generator=g, device="cuda").mul_(2)
        s["b"] = torch.randn(case["experts"], generator=g, device="cuda").mul_(0.1) if case["bias"] else None
        off = torch.randperm(case["experts"], generator=g, device="cuda")[:case["masked"]]
        x[:, off] = -math.inf
        s["x"] = x.bfloat16() if case["dtype"] == "bfloat16" else x
    elif path == "quantize":
        x = _activation(g, case["rows"], case["cols"])
        s["x"] = x if case["dtype"] == "bfloat16" else torch.randn(x.shape, generator=g, device="cuda").mul_(0.02)
    else:
        h, f, e = case["hidden"], case["ffn"], case["experts"]
        s["x"] = _activation(g, case["rows"], h)
        s["gate"], s["up"], s["down"] = _weight(g, f, h, (e,)), _weight(g, f, h, (e,)), _weight(g, h, f, (e,))
        # some experts are chosen more often than others
        logits = torch.randn(case["rows"], e, generator=g, device="cuda") + torch.randn(e, generator=g, device="cuda").mul_(0.5)
        best, ids = logits.topk(case["k"], -1)
        p, ids = best.softmax(-1), ids.int()
        if case["padding"]:
            p[-case["padding"]:], ids[-case["padding"]:] = 0, e
        s["p"], s["ids"] = p.contiguous(), ids.contiguous()
    torch.cuda.synchronize()
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------------
def run(s):
    return {"linear": _run_linear, "route": _run_route, "quantize": _run_quantize, "experts": _run_experts}[s["path"]](s)


def _run_linear(s):
    if own:
        ttnn = _ttnn()
        h = _handles(s)
        y = ttnn.linear_float8(h["x"], h["w"], bias=h["b"], activation=s["activation"] or None, dtype=getattr(ttnn, s["out"]))
        return _view(y, getattr(torch, s["out"]))
    tile = s["layout"] == "tile"
    x = _untiled(s["x"], up(s["rows"], 32), s["k"]) if tile else s["x"]
    y = torch.mm(_requantized(x.float()), _dequantized(*s["w"]).T)
    if s["b"] is not None:
        y = y + s["b"].float()
    y = _act(y, s["activation"]).to(getattr(torch, s["out"]))
    return _tiled(y, y.shape[0]) if tile else y


def _run_route(s):
    if own:
        ttnn = _ttnn()
        h = _handles(s)
        p, ids = ttnn.route_to_experts(h["x"], s["k"], score=s["score"], bias=h["b"], groups=s["groups"], top_groups=s["top_groups"],
                                       group_score=s["group_score"], renormalize=s["renormalize"], scale=s["scale"])
        return {"weights": _view(p, torch.float32), "experts": _view(ids, torch.int32)}
    # in 64 bits: two experts next to the border may differ by less than 32 bits show
    x = s["x"].double()
    off = x == -math.inf
    e = (x - x.amax(-1, keepdim=True)).exp()
    score = e / e.sum(-1, keepdim=True) if s["score"] == "softmax" else 1 / (1 + (-x).exp())
    choice = (score + s["b"].double() if s["b"] is not None else score).masked_fill(off, -math.inf)
    rows, n, G = x.shape[0], x.shape[1], s["groups"]
    if G > 1:
        best = choice.view(rows, G, n // G).sort(-1, descending=True)[0][..., :2]
        of_group = best[..., 0]
        if s["group_score"] == "top2_sum" and n // G > 1:
            of_group = of_group + best[..., 1].masked_fill(best[..., 1] == -math.inf, 0)
        order = of_group.sort(dim=-1, descending=True, stable=True)[1]
        kept = torch.zeros(rows, G, dtype=torch.bool, device=x.device).scatter_(1, order[:, :s["top_groups"]], True)
        choice = choice.masked_fill(~kept.repeat_interleave(n // G, 1), -math.inf)
    value, ids = (t[:, :s["k"]] for t in choice.sort(dim=-1, descending=True, stable=True))
    none = value == -math.inf
    p = score.gather(1, ids).masked_fill(none, 0)
    if s["renormalize"]:
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total == 0, torch.ones_like(total), total)
    return {"weights": (p * s["scale"]).float(), "experts": ids.masked_fill(none, n).int()}


def _run_quantize(s):
    if own:
        q = _ttnn().quantize_float8(_handles(s)["x"], block_rows=s["block_rows"])
        return {"codes": _view(q.codes, torch.float8_e4m3fn), "scales": _view(q.scales, torch.float32)}
    codes, scales = _quantized(s["x"].float(), s["block_rows"])
    return {"codes": codes, "scales": scales}


def _run_experts(s):
    if own:
        h = _handles(s)
        return _view(_ttnn().experts_mlp_float8(h["x"], h["ids"], h["p"], h["gate"], h["up"], h["down"], activation="silu"), torch.bfloat16)
    # every row through every expert, then weighted: 0 where the row does not go there
    x = _requantized(s["x"].float())
    gate, lin = (torch.matmul(x, _dequantized(*s[w]).mT) for w in ("gate", "up"))
    y = torch.matmul(_requantized(_act(gate, "silu") * lin), _dequantized(*s["down"]).mT)
    p = torch.zeros(s["rows"], s["experts"] + 1, device=x.device).scatter_add_(1, s["ids"].long(), s["p"])[:, :-1]
    return (y * p.T[..., None]).sum(0).bfloat16()


# ---- elementary parts of the plain form ----------------------------------------------------------------------------------
def _blocks(x, rows):
    """[..., H, W], padded with zeros to whole blocks of rows x 128, as [..., H / rows, rows, W / 128, 128]."""
    h, w = x.shape[-2:]
    x = torch.nn.functional.pad(x, (0, up(w, BLOCK) - w, 0, up(h, rows) - h))
    return x.reshape(*x.shape[:-2], x.shape[-2] // rows, rows, x.shape[-1] // BLOCK, BLOCK)


def _scale(b):
    """A correctly rounded quotient; a division by a number would be a multiplication by its rounded reciprocal."""
    most = b.abs().amax((-3, -1), keepdim=True).clamp(min=LEAST)
    return most / torch.full_like(most, TOP)


def _quantized(x, rows):
    b = _blocks(x, rows)
    scale = _scale(b)
    codes = (b / scale).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8).flatten(-2).flatten(-3, -2)[..., :x.shape[-2], :x.shape[-1]].contiguous().view(torch.float8_e4m3fn), scale[..., 0, :, 0]


def _requantized(x):
    """x after quantisation, one scale for 128 values of a row."""
    b = _blocks(x, 1)
    scale = _scale(b)
    return ((b / scale).clamp(-TOP, TOP).to(torch.float8_e4m3fn).float() * scale).flatten(-2).flatten(-3, -2)[..., :x.shape[-1]]


def _dequantized(codes, scales):
    n, k = codes.shape[-2:]
    return codes.float() * scales.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]


def _act(v, name):
    if name == "relu":
        return v.clamp(min=0)
    if name == "gelu":
        return v * 0.5 * (1 + torch.erf(v * math.sqrt(0.5)))
    return v / (1 + (-v).exp()) if name == "silu" else v


def _tiled(t, rows):
    """[r, c] padded to `rows` (both then multiples of 32) in the order of a tiled buffer: 32x32 tiles of four 16x16 faces."""
    t = torch.nn.functional.pad(t, (0, 0, 0, rows - t.shape[0])).view(rows // 32, 2, 16, t.shape[1] // 32, 2, 16)
    return t.permute(0, 3, 1, 4, 2, 5).reshape(-1)


def _untiled(t, rows, cols):
    return t.view(rows // 32, cols // 32, 2, 2, 16, 16).permute(0, 2, 4, 1, 3, 5).reshape(rows, cols)


# ---- the framework's side ------------------------------------------------------------------------------------------------
def _ttnn():
    package = os.path.join(os.getcwd(), "tt-metal_b200")   # imported with the repository's root as the working folder
    if package not in sys.path:
        sys.path.insert(0, package)
    import ttnn
    return ttnn


def _handles(s):
    """The tensors of a state under the framework's type, made on its first pass and kept as a program keeps them: views, nothing is copied or laid out."""
    if "handles" not in s:
        ttnn = _ttnn()
        device = ttnn.open_device(0)
        kinds = {torch.float32: ttnn.float32, torch.bfloat16: ttnn.bfloat16, torch.int32: ttnn.uint32, torch.float8_e4m3fn: ttnn.float8_e4m3}

        def wrap(t, shape=None, layout=ttnn.ROW_MAJOR_LAYOUT):
            return ttnn._ttnn.wrap_device_memory(t.data_ptr(), shape or ttnn.Shape(list(t.shape)), kinds[t.dtype], layout, device)

        h = {n: wrap(s[n]) for n in ("x", "p", "ids") if n in s}
        if s.get("layout") == "tile":
            h["x"] = wrap(s["x"], ttnn.Shape([s["rows"], s["k"]], [up(s["rows"], 32), s["k"]]), ttnn.TILE_LAYOUT)
        h.update({n: ttnn.Float8Tensor(wrap(s[n][0]), wrap(s[n][1])) for n in ("w", "gate", "up", "down") if n in s})
        h["b"] = wrap(s["b"].view(1, -1)) if s.get("b") is not None else None
        s["handles"] = h
    return s["handles"]


class _Buffer:
    """A ttnn tensor's device buffer under the CUDA array interface; keeps the tensor."""

    def __init__(self, t):
        self.tensor = t
        self.__cuda_array_interface__ = {"shape": (t.buffer_bytes(),), "typestr": "|u1", "data": (t.buffer_address(), False), "version": 2}


def _view(t, dtype):
    v = torch.as_tensor(_Buffer(t), device="cuda").view(dtype)
    return v if "TILE" in str(t.layout) else v.view(*t.shape)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------
def _weight_bytes(n, k):
    return n * k + 4 * (up(n, BLOCK) // BLOCK) * (up(k, BLOCK) // BLOCK)


def work(case):
    path = case["path"]
    if path == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": _weight_bytes(n, k) + 2 * m * k + m * n * (4 if case["out"] == "float32" else 2) + (2 * n if case["bias"] else 0), "flops": 2 * m * k * n}
    if path == "route":
        return {"bytes": case["rows"] * (case["experts"] * (4 if case["dtype"] == "float32" else 2) + 8 * case["k"]) + (4 * case["experts"] if case["bias"] else 0),
                "flops": case["rows"] * case["experts"]}
    if path == "quantize":
        blocks = up(case["rows"], case["block_rows"]) // case["block_rows"] * (up(case["cols"], BLOCK) // BLOCK)
        return {"bytes": case["rows"] * case["cols"] * (5 if case["dtype"] == "float32" else 3) + 4 * blocks, "flops": 2 * case["rows"] * case["cols"]}
    rows, e, k, h, f = case["rows"] - case["padding"], case["experts"], case["k"], case["hidden"], case["ffn"]
    hit = e * (1 - (1 - k / e) ** rows)   # experts that are chosen at all, were all as likely as each other
    return {"bytes": int(hit * (2 * _weight_bytes(f, h) + _weight_bytes(h, f))) + 4 * case["rows"] * h + 8 * case["rows"] * k, "flops": 6 * rows * k * h * f}


# ---- the same in 64 bits -------------------------------------------------------------------------------------------------
def _e4m3(v):
    """The nearest e4m3 values, ties to the even one: three bits of mantissa, steps of 2^-9 below 2^-6."""
    step = torch.ldexp(torch.ones_like(v), torch.frexp(v)[1].clamp(min=-5) - 4)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def _scales64(x, rows):
    """Scale of every element of x (they are held in 32 bits)."""
    h, w = x.shape
    of = torch.nn.functional.max_pool2d(torch.nn.functional.pad(x.abs(), (0, up(w, BLOCK) - w, 0, up(h, rows) - h))[None], (rows, BLOCK))[0]
    of = (of.clamp(min=LEAST) / TOP).float()
    return of, of.double().repeat_interleave(rows, 0)[:h].repeat_interleave(BLOCK, 1)[:, :w]


def _rounded64(x):
    each = _scales64(x, 1)[1]
    return _e4m3(_quotient(x, each)) * each


def _quotient(x, each):
    """In 32 bits by definition: quotients of short numbers lie on the border between two e4m3 values often, and what a scale's rounding leaves says nothing there."""
    return (x / each).float().double()


def _weight64(codes, scales):
    n, k = codes.shape
    at = lambda size: torch.arange(size, device=codes.device) // BLOCK  # noqa: E731
    return codes.double() * scales.double()[at(n)][:, at(k)]


def exact(case, seed):
    s, path = prepare(case, seed), case["path"]
    if path == "route":
        return _exact_route(s)
    if path == "quantize":
        x = s["x"].double()
        of, each = _scales64(x, case["block_rows"])
        return {"codes": _e4m3(_quotient(x, each)), "scales": of.double()}
    act = {"": lambda z: z, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}
    if path == "linear":
        x = s["x"]
        if case["layout"] == "tile":
            x = _untiled(x, up(case["rows"], 32), case["k"])
        y = _rounded64(x.double()) @ _weight64(*s["w"]).T
        y = act[case["activation"]](y + s["b"].double() if case["bias"] else y)
        return _tiled(y, y.shape[0]) if case["layout"] == "tile" else y
    x = _rounded64(s["x"].double())
    y = torch.zeros_like(x)
    for e in range(case["experts"]):
        row, slot = torch.nonzero(s["ids"] == e, as_tuple=True)
        if len(row):
            gate, lin, down = (_weight64(s[n][0][e], s[n][1][e]) for n in ("gate", "up", "down"))
            h = _rounded64(act["silu"](x[row] @ gate.T) * (x[row] @ lin.T))
            y.index_add_(0, row, (h @ down.T) * s["p"][row, slot].double()[:, None])
    return y


def _exact_route(s):
    """Expert after expert: the best that is left, as often as it takes."""
    x = s["x"].double()
    rows, n = x.shape
    score = torch.softmax(x, -1) if s["score"] == "softmax" else torch.sigmoid(x)
    left = torch.where(x == -math.inf, x, score if s["b"] is None else score + s["b"].double())
    size = n // s["groups"]
    if s["groups"] > 1:
        two = left.view(rows, -1, size).topk(min(2, size), -1)[0]
        two = torch.where((two == -math.inf) & (torch.arange(two.shape[-1], device=x.device) > 0), 0.0, two)
        of = two.sum(-1) if s["group_score"] == "top2_sum" else two[..., 0]
        taken = torch.zeros_like(of, dtype=torch.bool)
        for _ in range(s["top_groups"]):
            taken.scatter_(1, of.masked_fill(taken, -math.inf).argmax(1, keepdim=True), True)
        left = torch.where(taken[:, :, None].expand(-1, -1, size).reshape(rows, n), left, -math.inf)
    p = []
    for _ in range(s["k"]):
        value, at = left.max(1, keepdim=True)
        p.append(torch.where(value == -math.inf, 0.0, score.gather(1, at)))
        left = left.scatter(1, at, -math.inf)
    p = torch.cat(p, 1)
    if s["renormalize"]:
        p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
    return {"weights": p * s["scale"], "experts": None}
