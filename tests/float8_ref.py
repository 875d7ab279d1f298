"""float8 operators in 64 bits (plain torch), error bounds for the kernels' 32-bit sums, and the C-ABI signatures of their entry points.

Bounds. Sums: a block's 128 products are added on the tensor cores (at most 16 additions in a row are assumed for their tree), then scaled (two
roundings) and added in float32, one addition a block: off by at most (18 + blocks) * 2^-23 of the sum of magnitudes. A rounding to a type t is off by at
most finfo(t).eps / 2 of the value. Activations: exp and erf of the device are taken as right to 2^-20 of the result; their slopes are at most 1.13."""
import ctypes
import math

import torch

import cabi

BLOCK, TOP, LEAST = 128, 448.0, 2.0 ** -100
FLOAT8 = 16
BIAS_ROW_MAJOR = 512
SOFTMAX, SIGMOID, GROUP_MAX, GROUP_TOP2_SUM = 0, 1, 0, 1
ACTS = {None: lambda z: z, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}
ACT_CODES = {None: 0, "relu": 1, "gelu": 2, "silu": 3}

_p, _i, _l = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64
SIGS = {
    "ttb_quantize_float8": (_i, [_p, _i, _i, _p, _p, _l, _l, _l, _i, _p]),
    "ttb_linear_float8_workspace_bytes": (_l, [_l, _l, _l]),
    "ttb_linear_float8": (_i, [_p, _p, _p, _p, _p, _i, _l, _l, _l, _i, _i, _p, _l, _p]),
    "ttb_route_to_experts": (_i, [_p, _i, _p, _p, _p, _l, _l, _l, _i, _i, _i, _i, _i, _i, ctypes.c_float, _i, _p]),
    "ttb_experts_mlp_float8_workspace_bytes": (_l, [_l, _l, _l, _l, _l]),
    "ttb_experts_mlp_float8": (_i, [_p] * 10 + [_l, _l, _l, _i, _l, _l, _i, _i, _p, _l, _p]),
}


def lib():
    c = cabi.load().cdll
    for name, (res, args) in SIGS.items():
        fn = getattr(c, name)
        fn.restype, fn.argtypes = res, args
    return c


def blocks(n):
    return (n + BLOCK - 1) // BLOCK


def spread(s, rows, h, w):
    """A block's scale for each of its elements."""
    return s.repeat_interleave(rows, -2)[..., :h, :].repeat_interleave(BLOCK, -1)[..., :w]


def amax(x, rows):
    h, w = x.shape[-2:]
    p = torch.nn.functional.pad(x.abs(), (0, blocks(w) * BLOCK - w, 0, -h % rows))
    return p.reshape(*x.shape[:-2], p.shape[-2] // rows, rows, blocks(w), BLOCK).amax((-3, -1))


def quantize(x, rows):
    """Codes (float8) and scales of a float32 / bfloat16 tensor without NaN, on the CPU: divisions there are correctly rounded."""
    x = x.float().cpu()
    m = amax(x, rows).clamp(min=LEAST)
    s = m / torch.full_like(m, TOP)
    return (x / spread(s, rows, *x.shape[-2:])).clamp(-TOP, TOP).to(torch.float8_e4m3fn), s


def e4m3(v):
    """The nearest e4m3 number of 64-bit values, ties to even."""
    step = torch.ldexp(torch.ones_like(v), torch.frexp(v)[1].clamp(min=-5) - 4)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def dequantize(codes, scales, rows=BLOCK):
    return codes.double() * spread(scales.double(), rows, *codes.shape[-2:])


def requantized(x):
    """bfloat16 rows after quantisation with a scale for 128 values, in 64 bits, on x's device."""
    q, s = quantize(x, 1)
    return dequantize(q, s, 1).to(x.device)


def sums(x, w):
    """x w^T in 64 bits and how far a kernel's may be off."""
    return x @ w.mT, (x.abs() @ w.abs().mT) * (18 + blocks(x.shape[-1])) * 2.0 ** -23


def linear(x, codes, scales, bias, act, dtype):
    """Expected result and tolerance of linear_float8 (x bfloat16 [rows, K])."""
    y, tol = sums(requantized(x), dequantize(codes, scales))
    if bias is not None:
        y = y + bias.double()
        tol = tol + y.abs() * 2.0 ** -24
    tol = 1.13 * tol
    y = ACTS[act](y)
    if act in ("gelu", "silu"):
        tol = tol + y.abs() * 2.0 ** -20 + 2.0 ** -40
    return y, tol + (y.abs() + tol) * (torch.finfo(dtype).eps / 2) + 1e-38


def experts(x, ids, weights, gate, up, down, act="silu"):
    """Expected result and tolerance of experts_mlp_float8 (x bfloat16 [rows, hidden]; gate, up, down: (codes, scales))."""
    xq = requantized(x)
    y, tol = torch.zeros(x.shape, dtype=torch.double, device=x.device), torch.zeros(x.shape, dtype=torch.double, device=x.device)
    k = ids.shape[1]
    for e in range(gate[0].shape[0]):
        row, slot = torch.nonzero(ids == e, as_tuple=True)
        if not len(row):
            continue
        g, dg = sums(xq[row], dequantize(gate[0][e], gate[1][e]))
        u, du = sums(xq[row], dequantize(up[0][e], up[1][e]))
        a = ACTS[act](g)
        h = a * u
        dh = 1.13 * dg * (u.abs() + du) + a.abs() * du + h.abs() * 2.0 ** -20 + 2.0 ** -60
        # quantisation: the scale moves with the largest value; a quotient next to a border may go to either side
        m, dm = amax(h, 1).clamp(min=LEAST), amax(dh, 1)
        f = h.shape[-1]
        s, ds = spread(m / TOP, 1, len(row), f), spread((dm / m) + 2.0 ** -23, 1, len(row), f)
        q = h / s
        dq = dh / s + q.abs() * (ds + 2.0 ** -23)
        mid, low, high = e4m3(q), e4m3(q - dq), e4m3(q + dq)
        hq = mid * s
        dhq = torch.maximum((high - mid).abs(), (mid - low).abs()) * s + hq.abs() * ds
        w = dequantize(down[0][e], down[1][e])
        d, dd = sums(hq, w)
        dd = dd + dhq @ w.abs().mT
        p = weights[row, slot].double()[:, None]
        y.index_add_(0, row, d * p)
        tol.index_add_(0, row, dd * p.abs() + (d * p).abs() * k * 2.0 ** -23)
    return y, tol + (y.abs() + tol) * 2.0 ** -8 + 1e-38


def route(x, k, score="softmax", bias=None, groups=1, top_groups=1, group_score="max", renormalize=True, scale=1.0):
    """Weights (64 bits) and experts of rows of logits without NaN, one row and one expert after the other, in Python numbers."""
    out_w, out_e = [], []
    for row in x.double().tolist():
        n = len(row)
        most = max(row)
        if score == "softmax":
            e = [math.exp(v - most) if v > -math.inf else 0.0 for v in row]
            s = [v / math.fsum(e) if most > -math.inf else 0.0 for v in e]
        else:
            s = [1.0 / (1.0 + math.exp(-v)) if v > -700 else math.exp(max(v, -1e9)) for v in row]
        by_score = bias is not None or (groups > 1 and group_score == "top2_sum")
        c = [-math.inf if row[i] == -math.inf else (s[i] + (bias[i] if bias is not None else 0.0) if by_score else row[i]) for i in range(n)]
        size = n // groups
        if groups > 1:
            def of(g):
                two = sorted((v for v in c[g * size:(g + 1) * size] if v > -math.inf), reverse=True)[:2]
                return -math.inf if not two else sum(two) if group_score == "top2_sum" else two[0]
            kept = sorted(range(groups), key=lambda g: (-of(g), g))[:top_groups]
            c = [c[i] if i // size in kept else -math.inf for i in range(n)]
        ids = [i for i in sorted(range(n), key=lambda i: (-c[i], i))[:k] if c[i] > -math.inf]
        w = [s[i] for i in ids]
        if renormalize and math.fsum(w) > 0:
            w = [v / math.fsum(w) for v in w]
        out_e.append(ids + [n] * (k - len(ids)))
        out_w.append([v * scale for v in w] + [0.0] * (k - len(ids)))
    return torch.tensor(out_w, dtype=torch.double), torch.tensor(out_e, dtype=torch.int32)


def weight(g, n, k, lead=()):
    """A random weight as codes and scales (any positive scales, not those quantisation would give)."""
    codes = (torch.randn(*lead, n, k, generator=g) * 100).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
    return codes, (torch.rand(*lead, blocks(n), blocks(k), generator=g) + 0.5) * (2.0 / 100 / k ** 0.5)


def rows_of(g, rows, k):
    x = torch.randn(rows, k, generator=g)
    return (x * (1 + 15 * (torch.rand(k, generator=g) < 0.02))).bfloat16()


def assert_within(got, want, tol, what=""):
    got = got.double().to(want.device)
    off = (got - want).abs()
    assert torch.isfinite(got).all(), what
    worst = (off - tol).max().item()
    assert worst <= 0, f"{what}: {int((off > tol).sum())} of {off.numel()} outside, worst {(off / tol).max().item():.3g} of the tolerance"
