"""Measured cases of the block-scaled 8-bit operators: the quantiser, the product (dense, batched, grouped over experts)
and the experts' layer for a few tokens, each in a plain form made of elementary torch operations and as a user calls the
library.

An 8-bit operand stands for q[r, c] * scale: one float32 scale for each group of 128 columns of a row ("rows") or for each
128 x 128 tile ("tiles").  Products contract the last index of both operands, A[m, k] and B[n, k].
"""
import math

import torch

own = False

BLOCK = 128
FLOOR = 2.0 ** -100  # magnitudes of a block count as at least this much
FORMATS = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
MANTISSA = {"e4m3": (3, -6), "e5m2": (2, -14)}  # stored bits, exponent of the smallest normal number
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases ------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token's activations in front of a product: latency alone
        dict(name="quantize one token", op="quantize", rows=1, cols=4096, block="rows", fmt="e4m3", src="bf16", both=False),
        # a training batch's activations, in both directions: for the product and for the weights' gradient
        dict(name="quantize batch both ways", op="quantize", rows=8192, cols=4096, block="rows", fmt="e4m3", src="bf16", both=True),
        # master weights after a step, odd sizes: the tiles and their transpose
        dict(name="quantize weights", op="quantize", rows=5001, cols=4104, block="tiles", fmt="e4m3", src="f32", both=True),
        # a linear layer for one token: the weights are read once
        dict(name="product one token", op="product", batch=1, m=1, n=4096, k=8192, a_block="rows", b_block="tiles", a_fmt="e4m3", out="bf16"),
        # odd sizes in every direction, a batch of three
        dict(name="product odd batched", op="product", batch=3, m=333, n=1500, k=2056, a_block="rows", b_block="tiles", a_fmt="e4m3", out="bf16"),
        # a linear layer for a prompt, or a training batch's forward pass
        dict(name="product prompt", op="product", batch=1, m=4096, n=8192, k=4096, a_block="rows", b_block="tiles", a_fmt="e4m3", out="bf16"),
        # the weights' gradient: both operands quantised along the tokens, the result's gradient in e5m2
        dict(name="product weight gradient", op="product", batch=1, m=4096, n=2048, k=16384, a_block="rows", b_block="rows", a_fmt="e5m2", out="f32"),
        # experts' products while generating: most experts see a row or two
        dict(name="grouped few rows", op="grouped", along="rows", experts=64, rows=96, n=2048, k=2048, out="bf16"),
        # experts' products for a long batch, ragged
        dict(name="grouped prompt", op="grouped", along="rows", experts=32, rows=16384, n=2048, k=4096, out="bf16"),
        # experts' weight gradients: the contracted index is ragged, padded to the block
        dict(name="grouped weight gradient", op="grouped", along="contracted", experts=16, rows=8192, n=1024, k=2048, out="f32"),
        # the experts' layer for one token
        dict(name="experts one token", op="experts", tokens=1, top=8, experts=64, hidden=2048, inner=1024),
        # and for a batch of sequences being generated
        dict(name="experts batch", op="experts", tokens=32, top=8, experts=64, hidden=4096, inner=1536),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "grouped", "experts"])
    if op == "quantize":
        rows, cols = _log(rng, 1, 16384), _log(rng, 16, 16384)
        while rows * cols > 8192 * 4096:
            rows, cols = (rows + 1) // 2, (cols + 1) // 2
        return dict(op=op, rows=rows, cols=cols, block=rng.choice(["rows", "tiles"]), fmt=rng.choice(["e4m3", "e4m3", "e5m2"]),
                    src=rng.choice(["bf16", "f32"]), both=rng.random() < 0.5)
    if op == "product":
        m, n, k = _log(rng, 1, 8192), _log(rng, 64, 8192), _log(rng, 64, 16384)
        while m * n * k > 4096 * 8192 * 4096:
            m, n, k = (m + 1) // 2, (n + 1) // 2, (k + 1) // 2
        if rng.random() < 0.7:  # most widths are multiples of 16
            n, k = -(-n // 16) * 16, -(-k // 16) * 16
        batch = rng.choice([1, 1, 1, 2, 5]) if m * n * k < 2 ** 33 else 1
        a_block, b_block = rng.choice([("rows", "tiles"), ("rows", "tiles"), ("rows", "rows"), ("tiles", "tiles"), ("tiles", "rows")])
        return dict(op=op, batch=batch, m=m, n=n, k=k, a_block=a_block, b_block=b_block, a_fmt=rng.choice(["e4m3", "e4m3", "e5m2"]),
                    out=rng.choice(["bf16", "f32"]))
    if op == "grouped":
        experts = rng.choice([4, 8, 16, 32, 60])
        along = rng.choice(["rows", "rows", "contracted"])
        n, k = 16 * _log(rng, 8, 160), 16 * _log(rng, 8, 160)
        if along == "rows":
            rows = _log(rng, 1, 16384)
            if rng.random() < 0.3:
                k += rng.randrange(16)
        else:
            rows = BLOCK * _log(rng, 2, 64)
        return dict(op=op, along=along, experts=experts, rows=rows, n=n, k=k, out=rng.choice(["bf16", "f32"]))
    return dict(op=op, tokens=_log(rng, 1, 48), top=rng.choice([1, 2, 4, 6, 8]), experts=rng.choice([8, 16, 40, 64]),
                hidden=16 * _log(rng, 16, 256), inner=16 * _log(rng, 8, 96))


# ---- the plain forms' parts -----------------------------------------------------------------------------------------
def _blocks(x, block):
    """x[..., r, c] in blocks of 128 columns (rows) or of 128 x 128 (tiles), padded with zeros: [..., br, 1 or 128, bc, 128]."""
    *lead, r, c = x.shape
    h = 1 if block == "rows" else BLOCK
    x = torch.nn.functional.pad(x, (0, -c % BLOCK, 0, -r % h))
    return x.reshape(*lead, -(-r // h), h, -(-c // BLOCK), BLOCK)


def _quantize(x, block, fmt):
    """(q, scale) of x in 32 bits; the scale's shape is (rows or tiles of rows, blocks of columns)."""
    *lead, r, c = x.shape
    b = _blocks(x.float(), block)
    mag = torch.where(b.isfinite(), b.abs(), torch.zeros_like(b))
    top = mag.amax(dim=(-3, -1)).clamp_min(FLOOR)
    largest = torch.full_like(top, LARGEST[fmt])
    q = (b * (largest / top)[..., :, None, :, None]).to(FORMATS[fmt])
    q = q.reshape(*lead, b.shape[-4] * b.shape[-3], b.shape[-2] * BLOCK)
    # narrow in bytes: not every torch operation knows the 8-bit types
    q = q.view(torch.uint8)[..., :r, :c].contiguous().view(FORMATS[fmt])
    return q, top / largest


def _spread(scale, rows, cols):
    """The scale of every element of a rows x cols operand."""
    if scale.shape[-2] != rows:
        scale = scale.repeat_interleave(BLOCK, -2)[..., :rows, :]
    return scale.repeat_interleave(BLOCK, -1)[..., :cols]


def _values(q, scale):
    return q.float() * _spread(scale.float(), q.shape[-2], q.shape[-1])


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)


def _activations(g, *shape):
    """Normal values; some channels are louder, as activations have it."""
    x = torch.randn(*shape, generator=g, device="cuda")
    loud = 1 + 8 * (torch.rand(shape[-1], generator=g, device="cuda") < 0.02)
    return x * loud


def _weights(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda") * 0.02


def _group_major(scale):
    """The same scales with the index of the rows fastest in memory, which is how the quantiser lays them out."""
    return scale.transpose(-1, -2).contiguous().transpose(-1, -2)


def _operand(x, block, fmt="e4m3"):
    q, s = _quantize(x, block, fmt)
    return q, _group_major(s)


# ---- inputs --------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = _generator(seed)
    s = dict(case)
    if case["op"] == "quantize":
        make = _weights if case["block"] == "tiles" else _activations
        s["x"] = make(g, case["rows"], case["cols"]).to(TYPES[case["src"]])
    elif case["op"] == "product":
        b, m, n, k = (case[i] for i in ("batch", "m", "n", "k"))
        lead = (b,) if b > 1 else ()
        s["a"], s["sa"] = _operand(_activations(g, *lead, m, k), case["a_block"], case["a_fmt"])
        s["b"], s["sb"] = _operand(_weights(g, *lead, n, k), case["b_block"])
    elif case["op"] == "grouped":
        e, r, n, k = (case[i] for i in ("experts", "rows", "n", "k"))
        # a router's shares: uneven, some experts may get nothing; whole blocks where the contracted index is ragged
        unit = 1 if case["along"] == "rows" else BLOCK
        share = torch.rand(e, generator=g, device="cuda") ** 2 + 1e-3
        to = torch.multinomial(share, r // unit, replacement=True, generator=g)
        count = torch.bincount(to, minlength=e) * unit
        s["offsets"] = torch.cat([count.new_zeros(1), count.cumsum(0)]).to(torch.int32)
        s["most"] = int(count.max())  # for the plain form's padding
        if case["along"] == "rows":
            s["a"], s["sa"] = _operand(_activations(g, r, k), "rows")
            s["b"], s["sb"] = _operand(_weights(g, e, n, k), "tiles")
        else:  # out[e] is k x n, both operands quantised along the tokens
            s["a"], s["sa"] = _operand(_activations(g, k, r), "rows")
            s["b"], s["sb"] = _operand(_activations(g, n, r), "rows")
    else:
        t, top, e, h, i = (case[x] for x in ("tokens", "top", "experts", "hidden", "inner"))
        s["x"] = _activations(g, t, h).to(torch.bfloat16)
        s["up"], s["s_up"] = _operand(_weights(g, e, 2 * i, h), "tiles")
        s["down"], s["s_down"] = _operand(_weights(g, e, h, i), "tiles")
        score = torch.randn(t, e, generator=g, device="cuda").softmax(-1)
        gate, pick = score.topk(top, -1)
        s["pick"], s["gate"] = pick.to(torch.int32), gate / gate.sum(-1, keepdim=True)
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------
def run(state):
    return {"quantize": _run_quantize, "product": _run_product, "grouped": _run_grouped, "experts": _run_experts}[state["op"]](state)


def _run_quantize(s):
    if own:
        import ctc_amd
        return ctc_amd.block_quantize(s["x"], s["block"], FORMATS[s["fmt"]], transposed="both" if s["both"] else False)
    q, scale = _quantize(s["x"], s["block"], s["fmt"])
    if not s["both"]:
        return q, scale
    qt, scale_t = _quantize(s["x"].t(), s["block"], s["fmt"])
    return q, scale, qt, scale_t


def _run_product(s):
    if own:
        import ctc_amd
        return ctc_amd.scaled_contract(s["a"], s["sa"], s["b"], s["sb"], dtype=TYPES[s["out"]])
    a, b = _values(s["a"], s["sa"]), _values(s["b"], s["sb"])
    return torch.matmul(a, b.transpose(-1, -2).contiguous()).to(TYPES[s["out"]])


def _run_grouped(s):
    if own:
        import ctc_amd
        return ctc_amd.scaled_grouped_contract(s["a"], s["sa"], s["b"], s["sb"], s["offsets"], along=s["along"], dtype=TYPES[s["out"]])
    off = s["offsets"].long()
    a, b = _values(s["a"], s["sa"]), _values(s["b"], s["sb"])
    # every group padded to the longest one: one batched product
    place = off[:-1, None] + torch.arange(s["most"], device=off.device)
    inside = place < off[1:, None]
    place = torch.where(inside, place, torch.zeros_like(place))
    if s["along"] == "rows":
        rows = a[place]  # [experts, most, k]
        full = torch.bmm(rows, b.transpose(-1, -2).contiguous())
        return full[inside].to(TYPES[s["out"]])  # group after group: the rows in their order
    pa = torch.where(inside[:, :, None], a.t()[place], torch.zeros((), device=a.device))  # [experts, most, m]
    pb = torch.where(inside[:, :, None], b.t()[place], torch.zeros((), device=a.device))
    return torch.bmm(pa.transpose(-1, -2).contiguous(), pb).to(TYPES[s["out"]])


def _run_experts(s):
    if own:
        import ctc_amd
        return ctc_amd.expert_layer(s["x"], s["up"], s["s_up"], s["down"], s["s_down"], s["pick"], s["gate"])
    x, pick, gate = s["x"].float(), s["pick"].long(), s["gate"].float()
    tokens, top = pick.shape
    inner = s["inner"]
    if tokens * top < s["experts"]:  # the picked experts' weights, pair by pair
        flat = pick.reshape(-1)
        up = _values(s["up"].view(torch.uint8)[flat].view(torch.float8_e4m3fn), s["s_up"][flat])
        down = _values(s["down"].view(torch.uint8)[flat].view(torch.float8_e4m3fn), s["s_down"][flat])
        xs = x.repeat_interleave(top, 0)
        h = torch.bmm(up, xs[:, :, None])[..., 0]
        h = torch.nn.functional.silu(h[:, :inner]) * h[:, inner:]
        y = torch.bmm(down, h[:, :, None])[..., 0].reshape(tokens, top, -1)
        return (y * gate[..., None]).sum(1).to(torch.bfloat16)
    # every expert for every token, and the router's weights afterwards
    up, down = _values(s["up"], s["s_up"]), _values(s["down"], s["s_down"])
    h = torch.matmul(x, up.transpose(-1, -2).contiguous())  # [experts, tokens, 2 inner]
    h = torch.nn.functional.silu(h[..., :inner]) * h[..., inner:]
    y = torch.bmm(h, down.transpose(-1, -2).contiguous())  # [experts, tokens, hidden]
    weight = torch.zeros(tokens, s["experts"], device=x.device).scatter_add_(1, pick, gate)
    return (y * weight.t()[..., None]).sum(0).to(torch.bfloat16)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    cdiv = lambda a, b: -(-a // b)  # noqa: E731
    scales = lambda r, c, block: 4 * (r if block == "rows" else cdiv(r, BLOCK)) * cdiv(c, BLOCK)  # noqa: E731
    if case["op"] == "quantize":
        r, c = case["rows"], case["cols"]
        out = r * c + scales(r, c, case["block"])
        if case["both"]:
            out += r * c + scales(c, r, case["block"])
        return {"bytes": r * c * (2 if case["src"] == "bf16" else 4) + out, "flops": 2 * r * c * (2 if case["both"] else 1)}
    if case["op"] == "product":
        b, m, n, k = (case[i] for i in ("batch", "m", "n", "k"))
        size = 2 if case["out"] == "bf16" else 4
        return {"bytes": b * (m * k + n * k + scales(m, k, case["a_block"]) + scales(n, k, case["b_block"]) + size * m * n), "flops": 2 * b * m * n * k}
    if case["op"] == "grouped":
        e, r, n, k = (case[i] for i in ("experts", "rows", "n", "k"))
        size = 2 if case["out"] == "bf16" else 4
        if case["along"] == "rows":
            seen = min(e, r)  # experts that may have a row
            return {"bytes": r * k + scales(r, k, "rows") + seen * (n * k + scales(n, k, "tiles")) + size * r * n + 4 * (e + 1), "flops": 2 * r * n * k}
        return {"bytes": (k + n) * r + scales(k, r, "rows") + scales(n, r, "rows") + size * e * k * n + 4 * (e + 1), "flops": 2 * r * n * k}
    t, top, e, h, i = (case[x] for x in ("tokens", "top", "experts", "hidden", "inner"))
    seen = e * (1 - (1 - top / e) ** t) if top < e else e  # experts that some token picks, in the mean
    return {"bytes": int(seen * (3 * h * i + 4 * 3 * cdiv(h, BLOCK) * cdiv(i, BLOCK))) + 4 * t * h + 8 * t * top, "flops": 2 * t * top * 3 * h * i}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------
def _exact_quantize(x, rows_per_block, fmt):
    """Column block after column block of x in 64 bits: (q, scale)."""
    x = x.double()
    r, c = x.shape
    bits, low = MANTISSA[fmt]
    q = torch.empty_like(x)
    scale = torch.empty(-(-r // rows_per_block), -(-c // BLOCK), dtype=torch.float64, device=x.device)
    owner = torch.arange(r, device=x.device) // rows_per_block
    for j in range(scale.shape[1]):
        part = x[:, j * BLOCK:(j + 1) * BLOCK]
        top = torch.full((scale.shape[0],), FLOOR, dtype=torch.float64, device=x.device)
        top = top.scatter_reduce(0, owner, part.abs().max(1).values, "amax")
        scale[:, j] = top / LARGEST[fmt]
        v = part * (LARGEST[fmt] / top)[owner][:, None]
        _, e = torch.frexp(v)
        step = torch.ldexp(torch.ones_like(v), (e - 1).clamp_min(low) - bits)
        q[:, j * BLOCK:(j + 1) * BLOCK] = torch.round(v / step) * step
    return q, scale


def _block_product(a, sa, b, sb, k0, k1):
    """sum over [k0, k1) of a[m, k] b[n, k], block of 128 after block, each times its two scales."""
    acc = torch.zeros(a.shape[0], b.shape[0], dtype=torch.float64, device=a.device)
    at = lambda s, rows: s.double() if s.shape[0] == rows else s.double()[torch.arange(rows, device=s.device) // BLOCK]  # noqa: E731
    sa, sb = at(sa, a.shape[0]), at(sb, b.shape[0])
    for k in range(k0 - k0 % BLOCK, k1, BLOCK):
        lo, hi = max(k, k0), min(k + BLOCK, k1)
        acc += (a[:, lo:hi].double() @ b[:, lo:hi].double().t()) * sa[:, k // BLOCK, None] * sb[None, :, k // BLOCK]
    return acc


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        h = 1 if case["block"] == "rows" else BLOCK
        out = _exact_quantize(s["x"], h, case["fmt"])
        return out + _exact_quantize(s["x"].t(), h, case["fmt"]) if case["both"] else out
    if case["op"] == "product":
        k = case["k"]
        if case["batch"] == 1:
            return _block_product(s["a"], s["sa"], s["b"], s["sb"], 0, k)
        return torch.stack([_block_product(s["a"][i], s["sa"][i], s["b"][i], s["sb"][i], 0, k) for i in range(case["batch"])])
    if case["op"] == "grouped":
        off = s["offsets"].tolist()
        pairs = list(zip(off[:-1], off[1:]))
        if case["along"] == "rows":
            return torch.cat([_block_product(s["a"][lo:hi], s["sa"][lo:hi], s["b"][e], s["sb"][e], 0, case["k"]) for e, (lo, hi) in enumerate(pairs) if hi > lo])
        return torch.stack([_block_product(s["a"], s["sa"], s["b"], s["sb"], lo, hi) for lo, hi in pairs])
    y = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device="cuda")
    one = torch.ones(case["tokens"], -(-case["hidden"] // BLOCK), dtype=torch.float64, device="cuda")
    inner_one = torch.ones(case["tokens"], -(-case["inner"] // BLOCK), dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        weight = (s["gate"].double() * (s["pick"] == e)).sum(1)
        h = _block_product(s["x"], one, s["up"][e], s["s_up"][e], 0, case["hidden"])
        gate, up = h[:, :case["inner"]], h[:, case["inner"]:]
        y += weight[:, None] * _block_product(gate / (1 + torch.exp(-gate)) * up, inner_one, s["down"][e], s["s_down"][e], 0, case["inner"])
    return y
