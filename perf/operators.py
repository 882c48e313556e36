"""The microscaled (MX) expert path: what its operators are measured on.

Four operators of the quantised mixture-of-experts layer, each in a plain form
(elementary torch operations in 32 bits) and as the framework's call:

  norm    residual add + RMSNorm with an 8-bit output: residual' = residual + hidden,
          normed = weight * rmsnorm(residual'), and normed again as MX rows (e4m3
          elements, one power-of-two scale for 32 of them)
  mx4     a matrix to 4-bit MX (e2m1 elements, one power-of-two scale for 32 of them)
          and back: what loading a checkpoint, and looking at its error, runs
  swiglu  act = silu(x Wg^T) * (x Wu^T) per expert, x MX 8-bit rows, W 4-bit MX, act MX
          8-bit rows
  down    y = act W^T per expert, act MX 8-bit rows, W 4-bit MX, y bf16

A block's scale is the smallest power of two (2^-127 at least) with which the block's
largest magnitude does not pass the element type's largest value (448 for e4m3, 6 for
e2m1); elements are rounded to the nearest, ties to even.
"""
import math

import torch

own = False

BLOCK = 32
E4M3_MAX, E2M1_MAX = 448.0, 6.0
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token of a decoding Qwen3-30B-A3B layer: the latency of one small launch
        dict(name="norm decode 1x2048", op="norm", tokens=1, hidden=2048, dtype="bf16", add=True, keep=True),
        # an odd fp32 batch without an add (first layer of a chunk)
        dict(name="norm fp32 257x1024", op="norm", tokens=257, hidden=1024, dtype="fp32", add=False, keep=False),
        # Mixtral-8x7B prefill, 8 x 2048 tokens
        dict(name="norm prefill 16384x4096", op="norm", tokens=16384, hidden=4096, dtype="bf16", add=True, keep=True),
        # the down projection of one Qwen3 expert, as a weight loader hands it over
        dict(name="mx4 2048x768", op="mx4", rows=2048, cols=768, dtype="bf16"),
        # the gate and up projections of two Mixtral experts
        dict(name="mx4 57344x4096", op="mx4", rows=57344, cols=4096, dtype="bf16"),
        # Qwen3 decode, one token: 8 of 128 experts with one row each
        dict(name="swiglu qwen3 decode 1", op="swiglu", tokens=1, top_k=8, experts=128, hidden=2048, inter=768, zipf=1.0),
        # Qwen3 decode, 64 tokens, skewed routing: most experts hit, a few rows each
        dict(name="swiglu qwen3 decode 64", op="swiglu", tokens=64, top_k=8, experts=128, hidden=2048, inter=768, zipf=1.0),
        # DeepSeek-V2-Lite, a short odd prompt: about 94 rows per expert, ragged tiles
        dict(name="swiglu dsv2lite 1001", op="swiglu", tokens=1001, top_k=6, experts=64, hidden=2048, inter=1408, zipf=0.0),
        # Mixtral-8x7B prefill: the layer's largest product
        dict(name="swiglu mixtral 16384", op="swiglu", tokens=16384, top_k=2, experts=8, hidden=4096, inter=14336, zipf=0.0),
        # Qwen3 decode, one token
        dict(name="down qwen3 decode 1", op="down", tokens=1, top_k=8, experts=128, hidden=2048, inter=768, zipf=1.0),
        # Qwen1.5-MoE decode, 128 tokens, skewed: some experts without a row
        dict(name="down qwen15 decode 128", op="down", tokens=128, top_k=4, experts=60, hidden=2048, inter=1408, zipf=1.0),
        # DeepSeek-V2-Lite prefill: 98304 rows
        dict(name="down dsv2lite 16384", op="down", tokens=16384, top_k=6, experts=64, hidden=2048, inter=1408, zipf=0.0),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["norm", "mx4", "swiglu", "down", "swiglu", "down"])
    if op == "norm":
        hidden = 128 * rng.randint(2, 32)
        return dict(op=op, tokens=log_int(1, 16384), hidden=hidden, dtype=rng.choice(["bf16", "bf16", "fp32"]),
                    add=rng.random() < 0.7, keep=rng.random() < 0.7)
    if op == "mx4":
        return dict(op=op, rows=log_int(1, 57344), cols=32 * rng.randint(1, 128), dtype=rng.choice(["bf16", "fp32"]))
    while True:
        experts = log_int(1, 128)
        case = dict(op=op, tokens=log_int(1, 16384), top_k=rng.randint(1, min(8, experts)), experts=experts,
                    hidden=128 * log_int(2, 32), inter=128 * log_int(1, 112), zipf=rng.choice([0.0, 0.6, 1.0, 1.4]))
        rows = case["tokens"] * case["top_k"]
        weights = experts * 2 * case["inter"] * case["hidden"]
        # skewed routing pads the plain form up to one expert with a row of every token
        padded = case["tokens"] * experts * max(case["hidden"], 2 * case["inter"])
        if (weights <= 8 * 28672 * 4096 and rows * 2 * case["inter"] * case["hidden"] <= 32768 * 28672 * 4096 // 4
                and padded <= 2 ** 31):
            return case


# ------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _row_bytes(k):
    return k + (k // BLOCK + 15) // 16 * 16


def _probabilities(case):
    p = torch.arange(1, case["experts"] + 1, dtype=torch.float64) ** -case["zipf"]
    return p / p.sum()


def _routing(case, g):
    """Rows per expert of a batch whose tokens draw top_k different experts each."""
    scores = _probabilities(case).log().cuda()[None, :]
    u = torch.rand(case["tokens"], case["experts"], generator=g, device="cuda", dtype=torch.float64)
    ids = (scores - (-(u.clamp_min(1e-300)).log()).log()).topk(case["top_k"], dim=1).indices
    place = torch.randperm(case["experts"], generator=g, device="cuda")  # hot experts sit anywhere
    counts = torch.bincount(place[ids].reshape(-1), minlength=case["experts"])
    offsets = torch.zeros(case["experts"] + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    return offsets, int(counts.max())


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "norm":
        dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        t, h = case["tokens"], case["hidden"]
        # a residual stream of spread 2 with a few loud channels, as deep layers have them
        loud = torch.where(torch.rand(h, generator=g, device="cuda") < 0.01, 12.0, 1.0)
        s = dict(residual=(2.0 * loud * torch.randn(t, h, generator=g, device="cuda")).to(dt), hidden=None,
                 weight=(1.0 + 0.2 * torch.randn(h, generator=g, device="cuda")).to(dt), eps=1e-6)
        if case["add"]:
            s["hidden"] = torch.randn(t, h, generator=g, device="cuda").to(dt)
        return dict(s, op=op, keep=case["keep"])
    if op == "mx4":
        dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        return dict(op=op, w=(0.02 * torch.randn(case["rows"], case["cols"], generator=g, device="cuda")).to(dt))
    offsets, most = _routing(case, g)
    rows, p = case["tokens"] * case["top_k"], case["experts"]
    n, k = (2 * case["inter"], case["hidden"]) if op == "swiglu" else (case["hidden"], case["inter"])
    x = torch.randn(rows, k, generator=g, device="cuda")
    if op == "down":  # what silu(gate) * up looks like
        x = x * torch.sigmoid(x) * torch.randn(rows, k, generator=g, device="cuda")
    values, scales = _quantize(x, E4M3_MAX)
    buf = torch.zeros(rows, _row_bytes(k), dtype=torch.uint8, device="cuda")
    buf[:, :k] = values.to(torch.float8_e4m3fn).view(torch.uint8)
    buf[:, k:k + k // BLOCK] = scales
    data = torch.empty(p, n, k // 2, dtype=torch.uint8, device="cuda")
    wscales = torch.empty(p, n, k // BLOCK, dtype=torch.uint8, device="cuda")
    for e in range(p):
        values, wscales[e] = _quantize(0.02 * torch.randn(n, k, generator=g, device="cuda"), E2M1_MAX)
        codes = _e2m1_codes(values)
        data[e] = codes[:, 0::2] | (codes[:, 1::2] << 4)
    s = dict(op=op, buf=buf, k=k, offsets=offsets, most=most, data=data, wscales=wscales)
    if own:  # weights are laid out once, when they are loaded
        from easyinfra_b200 import ops
        s["x"] = ops.MX8Rows(buf, k)
        s["w"] = ops.pack_mx4_weights(data, wscales, swiglu=op == "swiglu")
    return s


# ------------------------------------------------------------------------------ the plain form
def _quantize(x, largest):
    """(elements as values in 32 bits, scale bytes) of the last dimension's blocks."""
    b = x.float().unflatten(-1, (-1, BLOCK))
    m, e = torch.frexp(b.abs().amax(-1))          # amax = m 2^e, m in [0.5, 1)
    top, limit = (9, 0.875) if largest == E4M3_MAX else (3, 0.75)   # largest = limit 2^top
    e = (e - top + (m > limit)).clamp_min(-127)
    e = torch.where(m == 0, -127, e)
    v = torch.ldexp(b, -e[..., None])
    if largest == E4M3_MAX:
        v = v.to(torch.float8_e4m3fn).float()
    else:
        a = v.abs()
        step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
        v = torch.copysign((a / step).round() * step, v)
    return v.flatten(-2), (e + 127).to(torch.uint8)


def _scale_values(scales):
    return torch.ldexp(torch.ones((), device=scales.device), scales.int() - 127)


def _e2m1_codes(values):
    a = values.abs()
    code = torch.where(a < 2.0, a * 2.0, torch.where(a < 4.0, a + 2.0, a * 0.5 + 4.0)).to(torch.uint8)
    return code | (torch.signbit(values).to(torch.uint8) << 3)


def _rows32(buf, k):
    v = buf[:, :k].view(torch.float8_e4m3fn).float().unflatten(-1, (-1, BLOCK))
    return (v * _scale_values(buf[:, k:k + k // BLOCK])[..., None]).flatten(-2)


def _weights32(data, scales):
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=data.device)
    pairs = torch.stack([data & 15, data >> 4], -1).flatten(-2).int()
    return (table[pairs].unflatten(-1, (-1, BLOCK)) * _scale_values(scales)[..., None]).flatten(-2)


def _product(s):
    """x W^T of every row with its expert's weights, in 32 bits."""
    x, offsets = _rows32(s["buf"], s["k"]), s["offsets"].long()
    rows, p = x.shape[0], offsets.numel() - 1
    r = torch.arange(rows, device=x.device)
    slot = torch.searchsorted(offsets, r, right=True) - 1
    if rows <= p // 2:  # few rows: the weights of their experts alone
        return torch.matmul(_weights32(s["data"][slot], s["wscales"][slot]), x[:, :, None])[:, :, 0]
    pos = r - offsets[slot]
    padded = x.new_zeros(p, s["most"], s["k"])
    padded[slot, pos] = x
    return torch.bmm(padded, _weights32(s["data"], s["wscales"]).transpose(1, 2))[slot, pos]


def _plain(s):
    if s["op"] == "norm":
        dt = s["residual"].dtype
        r = s["residual"].float()
        if s["hidden"] is not None:
            r = (r + s["hidden"].float()).to(dt).float()
        inv = torch.rsqrt(r.double().square().mean(-1, keepdim=True) + s["eps"]).float()
        normed = ((r * inv).to(dt).float() * s["weight"].float()).to(dt)
        v, e = _quantize(normed, E4M3_MAX)
        return _norm_outputs(s, r.to(dt), normed, v.to(torch.float8_e4m3fn), e.view(torch.float8_e8m0fnu))
    if s["op"] == "mx4":
        v, e = _quantize(s["w"], E2M1_MAX)
        v = (v.unflatten(-1, (-1, BLOCK)) * _scale_values(e)[..., None]).flatten(-2)
        return dict(values=v.to(torch.bfloat16), scales=e.view(torch.float8_e8m0fnu))
    y = _product(s)
    if s["op"] == "down":
        return y.to(torch.bfloat16)
    gate, up = y.chunk(2, -1)
    v, e = _quantize(gate * torch.sigmoid(gate) * up, E4M3_MAX)
    return dict(data=v.to(torch.float8_e4m3fn), scales=e.view(torch.float8_e8m0fnu))


def _norm_outputs(s, residual, normed, data, scales):
    out = dict(residual=residual, data=data, scales=scales)
    return dict(out, normed=normed) if s["keep"] else out


# ------------------------------------------------------------------------------ one pass
def run(state):
    if not own:
        return _plain(state)
    from easyinfra_b200 import ops
    op = state["op"]
    if op == "norm":
        residual, normed, q = ops.add_rmsnorm_mx8(state["residual"], state["hidden"], state["weight"], state["eps"],
                                                  norm=state["keep"])
        return _norm_outputs(state, residual, normed, q.data, q.scales)
    if op == "mx4":
        data, scales = ops.quantize_mx4(state["w"])
        return dict(values=ops.dequantize_mx4(data, scales, torch.bfloat16), scales=scales.view(torch.float8_e8m0fnu))
    if op == "swiglu":
        act = ops.grouped_swiglu_mx4(state["x"], state["offsets"], state["w"])
        return dict(data=act.data, scales=act.scales)
    return ops.grouped_down_mx4(state["x"], state["offsets"], state["w"])


def work(case):
    op = case["op"]
    if op == "norm":
        t, h, eb = case["tokens"], case["hidden"], 2 if case["dtype"] == "bf16" else 4
        # residual read and written, hidden read, normed written, the 8-bit rows written, the weight read
        return dict(bytes=t * h * eb * (2 + case["add"] + case["keep"]) + t * (h + h // BLOCK) + h * eb, flops=6 * t * h)
    if op == "mx4":
        n, eb = case["rows"] * case["cols"], 2 if case["dtype"] == "bf16" else 4
        # read, packed written and read again, values written
        return dict(bytes=n * eb + 2 * (n // 2 + n // BLOCK) + 2 * n, flops=4 * n)
    rows = case["tokens"] * case["top_k"]
    # experts that have a row, on average: a token's experts differ, and beyond that a row misses expert j
    # with a probability of about 1 - p_j
    hit = max(case["top_k"], float((1 - (1 - _probabilities(case)) ** rows).sum()))
    h, i = case["hidden"], case["inter"]
    n, k = (2 * i, h) if op == "swiglu" else (h, i)
    out = rows * (i + i // BLOCK) if op == "swiglu" else rows * h * 2
    return dict(bytes=int(rows * (k + k // BLOCK) + hit * n * (k // 2 + k // BLOCK) + out), flops=2 * rows * n * k)


# ------------------------------------------------------------------------------ in 64 bits, written apart
def _exact_blocks(x, largest, grid):
    """Nearest grid values (ties to the even grid point) of x in 64 bits, and the scales."""
    rows = x.reshape(-1, BLOCK)
    amax = rows.abs().max(1).values
    e = torch.ceil(torch.log2(torch.where(amax > 0, amax, 1.0) / largest))
    # the logarithm may land one off next to a power of two
    e = torch.where(amax > largest * torch.exp2(e), e + 1, e)
    e = torch.where(amax <= largest * torch.exp2(e - 1), e - 1, e)
    scale = torch.exp2(torch.where(amax > 0, e.clamp(min=-127), torch.full_like(e, -127)))
    v = rows / scale[:, None]
    points = torch.tensor(grid, dtype=torch.float64, device=x.device)
    a = v.abs().contiguous()
    hi = torch.searchsorted(points, a).clamp(max=points.numel() - 1)
    lo = (hi - 1).clamp(min=0)
    up, down = points[hi] - a, a - points[lo]
    take = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    take = torch.where(points[hi] == a, hi, take)
    q = torch.where(v < 0, -points[take], points[take])
    return q.reshape(x.shape), scale.reshape(*x.shape[:-1], -1)


def _e4m3_grid():
    small = [m * 2.0 ** -9 for m in range(8)]
    return small + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8) if (e, m) != (15, 7)]


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "norm":
        # the operator rounds to its type after the add, after the normalisation and after the weight
        dt = s["residual"].dtype
        total = s["residual"].double() + (0 if s["hidden"] is None else s["hidden"].double())
        total = total.to(dt).double()
        unit = (total / torch.sqrt((total * total).sum(1, keepdim=True) / total.shape[1] + s["eps"])).to(dt).double()
        normed = (unit * s["weight"].double()).to(dt).double()
        q, scale = _exact_blocks(normed, E4M3_MAX, _e4m3_grid())
        return _norm_outputs(s, total, normed, q, scale)
    if s["op"] == "mx4":
        q, scale = _exact_blocks(s["w"].double(), E2M1_MAX, list(E2M1))
        return dict(values=(q.reshape(-1, BLOCK) * scale.reshape(-1, 1)).reshape(q.shape), scales=scale)
    k, offsets = s["k"], s["offsets"].tolist()
    x = s["buf"][:, :k].view(torch.float8_e4m3fn).double().reshape(-1, BLOCK)
    x = (x * torch.exp2(s["buf"][:, k:k + k // BLOCK].double() - 127).reshape(-1, 1)).reshape(-1, k)
    signed = torch.tensor([v for v in E2M1] + [-v for v in E2M1], dtype=torch.float64, device=x.device)
    parts = []
    for e in range(len(offsets) - 1):
        if offsets[e] == offsets[e + 1]:
            continue
        w = x.new_empty(s["data"].shape[1], k)
        w[:, 0::2] = signed[(s["data"][e] % 16).long()]
        w[:, 1::2] = signed[(s["data"][e] // 16).long()]
        w = (w.reshape(-1, BLOCK) * torch.exp2(s["wscales"][e].double() - 127).reshape(-1, 1)).reshape(-1, k)
        parts.append(x[offsets[e]:offsets[e + 1]] @ w.T)
    y = torch.cat(parts)
    if s["op"] == "down":
        return y
    half = y.shape[1] // 2
    q, scale = _exact_blocks(y[:, :half] / (1 + torch.exp(-y[:, :half])) * y[:, half:], E4M3_MAX, _e4m3_grid())
    return dict(data=q, scales=scale)
