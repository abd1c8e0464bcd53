"""The microscaled row operators: what they compute, in plain torch, and the cases they are timed on.

Unit rows are laid out [num_units, B], one row of B samples per unit. A microscaled (MX) row holds blocks of 32
samples: one power-of-two scale byte (value 2^(byte - 127), 255 = not a number) and 32 codes of 8 bits (e4m3, e5m2)
or 4 bits (e2m1, two to a byte, the even sample in the low nibble). Weights are held in blocks of 32 in-edges of one
destination unit. `own` chooses between the plain form below and the framework's kernels.
"""

import math

import torch

own = False

DEVICE = "cuda"
BLOCK = 32

# name: (mantissa bits, exponent of the smallest normal number, largest value, bits of a code)
FORMATS = {"e4m3": (3, -6, 448.0, 8), "e5m2": (2, -14, 57344.0, 8), "e2m1": (1, 0, 6.0, 4)}
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the sparse MLP's batch of 256 (784-1000-1000-10 units) checkpointed for its backward pass: a latency case
        {"name": "quantize_mlp_e4m3", "op": "quantize", "units": 2794, "batch": 256, "fmt": "e4m3", "dtype": "f32",
         "keep": True, "by_sample": False},
        # a million-unit net's batch in 4 bits, from bfloat16, an odd batch
        {"name": "quantize_reservoir_e2m1", "op": "quantize", "units": 1 << 20, "batch": 250, "fmt": "e2m1",
         "dtype": "bf16", "keep": False, "by_sample": False},
        # reading a checkpoint of the unit-lifecycle net's slots back
        {"name": "dequantize_units_e4m3", "op": "dequantize", "units": 65536, "batch": 256, "fmt": "e4m3",
         "dtype": "f32"},
        # reading 4-bit rows back as bfloat16, at full width
        {"name": "dequantize_reservoir_e2m1", "op": "dequantize", "units": 1 << 20, "batch": 256, "fmt": "e2m1",
         "dtype": "bf16"},
        # the sparse MLP's ReLU derivative from the checkpoint
        {"name": "unit_grad_mlp", "op": "unit_grad", "units": 2794, "batch": 256, "fmt": "e4m3", "act": "relu",
         "seed_rows": False},
        # a wide tanh net's derivative with the loss rows added, an odd batch
        {"name": "unit_grad_units", "op": "unit_grad", "units": 65536, "batch": 509, "fmt": "e5m2", "act": "tanh",
         "seed_rows": True},
        # the sparse MLP's 1000 x 1000 level pair at a tenth density
        {"name": "edge_grad_mlp", "op": "edge_grad", "sources": 1000, "targets": 1000, "slots": 100000,
         "live": 100000, "batch": 256, "fmt": "e4m3", "grown": 0.0},
        # the same pair at half density, partly regrown (out of source order)
        {"name": "edge_grad_mlp50", "op": "edge_grad", "sources": 1000, "targets": 1000, "slots": 524288,
         "live": 500000, "batch": 256, "fmt": "e4m3", "grown": 0.05},
        # the unit-lifecycle arena (65,536 units, 2^22 slots, two thirds live)
        {"name": "edge_grad_units", "op": "edge_grad", "sources": 32768, "targets": 32768, "slots": 1 << 22,
         "live": 2796202, "batch": 128, "fmt": "e5m2", "grown": 0.1},
        # one sample through a trained arena: 4-bit weights, float32 activations
        {"name": "product_one_sample", "op": "product", "sources": 32768, "targets": 32768, "fan_in": 64, "batch": 1,
         "weights": "e2m1", "rows": "f32", "act": "tanh", "out": "f32"},
        # a batch through a 1000 x 1000 level pair, 4-bit weights and rows in and out
        {"name": "product_mlp", "op": "product", "sources": 1000, "targets": 1000, "fan_in": 100, "batch": 256,
         "weights": "e2m1", "rows": "e2m1", "act": "relu", "out": "e2m1"},
        # a ragged batch through the unit-lifecycle arena, 4-bit rows, float32 answers
        {"name": "product_units", "op": "product", "sources": 32768, "targets": 32768, "fan_in": 96, "batch": 100,
         "weights": "e2m1", "rows": "e2m1", "act": "identity", "out": "f32"},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "dequantize", "unit_grad", "edge_grad", "product"])
    if op in ("quantize", "dequantize", "unit_grad"):
        batch = _log(rng, 1, 1024)
        units = _log(rng, 1, min(1 << 20, (1 << 25 if op == "unit_grad" else 1 << 28) // batch))
        case = {"op": op, "units": units, "batch": batch, "fmt": rng.choice(sorted(FORMATS))}
        if op == "quantize":
            case |= {"dtype": rng.choice(sorted(DTYPES)), "keep": rng.random() < 0.5, "by_sample": rng.random() < 0.3}
        elif op == "dequantize":
            case |= {"dtype": rng.choice(sorted(DTYPES))}
        else:
            case |= {"fmt": rng.choice(["e4m3", "e5m2"]), "act": rng.choice(["identity", "tanh", "relu", "sigmoid"]),
                     "seed_rows": rng.random() < 0.5}
        return case
    sources, targets = _log(rng, 10, 32768), _log(rng, 1, 32768)
    if op == "edge_grad":
        batch = _log(rng, 1, 512)
        slots = _log(rng, 32, min(1 << 22, (1 << 28) // batch))
        return {"op": op, "sources": sources, "targets": targets, "slots": slots,
                "live": max(1, int(slots * rng.uniform(0.5, 1.0))), "batch": batch,
                "fmt": rng.choice(["e4m3", "e5m2"]), "grown": rng.choice([0.0, rng.uniform(0.0, 0.5)])}
    rows = rng.choice(["f32", "e2m1", "e4m3", "e5m2"])
    batch = _log(rng, 1, 32) if rows == "f32" else _log(rng, 1, 512)
    most = (32768 * 96 * 100) // (batch * targets)
    return {"op": op, "sources": sources, "targets": targets, "fan_in": _log(rng, 1, max(1, min(32768, most))),
            "batch": batch, "weights": rng.choice(["f32", "e2m1", "e4m3", "e5m2"]), "rows": rows,
            "act": rng.choice(["identity", "tanh", "relu", "sigmoid"]), "out": rng.choice(["f32", "f32", "e2m1", "e4m3"])}


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _act(kind, x):
    if kind == "tanh":
        return torch.tanh(x)
    if kind == "relu":
        return torch.clamp_min(x, 0.0)
    if kind == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-x))
    return x


def _act_prime(kind, a):
    if kind == "tanh":
        return 1.0 - a * a
    if kind == "relu":
        return (a > 0).to(a.dtype)
    if kind == "sigmoid":
        return a * (1.0 - a)
    return torch.ones_like(a)


def _pow2(e):
    """2^e in float32 for whole e of -127 to 127, from its bits."""
    e = e.to(torch.int32)
    return torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22)).view(torch.float32)


def _blocks(x):
    """[N, B] as [N, ceil(B / 32), 32], padded with zeros."""
    n, b = x.shape
    nb = -(-b // BLOCK)
    return torch.nn.functional.pad(x, (0, nb * BLOCK - b)).reshape(n, nb, BLOCK)


def _scale_exponent(amax, fmt):
    """The smallest e >= -127 with amax <= largest(fmt) * 2^e (-127 for a block of zeros)."""
    largest = FORMATS[fmt][2]
    m, e = torch.frexp(amax)  # amax = m * 2^e, 0.5 <= m < 1
    lm, le = math.frexp(largest)
    e = e - le + (m > lm).to(e.dtype)
    return torch.where(amax > 0, e, torch.full_like(e, -127)).clamp(min=-127)


def _round(x, fmt, keep):
    """[N, nb, 32] float32 -> (exponent of each block's scale, elements' values before the scale)."""
    mant, emin, largest, _ = FORMATS[fmt]
    e = _scale_exponent(x.abs().amax(dim=-1), fmt)
    y = x * _pow2(-e)[..., None]
    _, ye = torch.frexp(y)
    q = _pow2(torch.clamp(ye - 1, min=emin) - mant)
    r = (torch.round(y / q) * q).clamp(-largest, largest)
    if keep:
        tiny = torch.full_like(r, 2.0 ** (emin - mant))
        r = torch.where((x != 0) & (r == 0), torch.copysign(tiny, x), r)
    return e, r


def _encode(r, fmt):
    """Elements' values -> codes, one per byte."""
    mant, emin, _, bits = FORMATS[fmt]
    a = r.abs()
    _, e = torch.frexp(a)
    e = torch.clamp(e - 1, min=emin)
    k = (a * _pow2(mant - e)).to(torch.int32)  # the mantissa with its leading bit, if normal
    code = torch.where(k >= (1 << mant), ((e - emin) << mant) + k, k)
    return (code | (torch.signbit(r).to(torch.int32) << (bits - 1))).to(torch.uint8)


def _pack(code, fmt):
    n, nb, _ = code.shape
    if FORMATS[fmt][3] == 4:
        code = code[..., 0::2] | (code[..., 1::2] << 4)
    return code.reshape(n, nb * code.shape[2]).contiguous()


def _values(codes, scales, fmt, batch):
    """MX rows -> [N, batch] float32."""
    mant, emin, _, bits = FORMATS[fmt]
    c = codes.to(torch.int32)
    if bits == 4:
        c = torch.stack([c & 15, c >> 4], dim=-1)
    n, nb = scales.shape
    c = c.reshape(n, nb, BLOCK)
    field = (c & ((1 << (bits - 1)) - 1)) >> mant
    frac = (c & ((1 << mant) - 1)).to(torch.float32)
    a = torch.where(field > 0, (frac + (1 << mant)) * _pow2(field - 1 + emin - mant), frac * 2.0 ** (emin - mant))
    a = torch.where((c >> (bits - 1)) > 0, -a, a)
    return (a * _pow2(scales.to(torch.int32) - 127)[..., None]).reshape(n, nb * BLOCK)[:, :batch]


def _quantized_values(x, fmt, keep=False):
    """The values that [N, B] float32 rows have after quantisation (at most 4 significant bits: bfloat16 holds them)."""
    e, r = _round(_blocks(x), fmt, keep)
    return (r * _pow2(e)[..., None]).reshape(x.shape[0], -1)[:, :x.shape[1]]


def _quantize(x, fmt, keep=False):
    e, r = _round(_blocks(x), fmt, keep)
    return _pack(_encode(r, fmt), fmt), (e + 127).to(torch.uint8)


def _weight_values(s):
    """The in-edges' weights [E] float32 of a product's state, and each edge's destination position."""
    deg = s["offsets"][1:] - s["offsets"][:-1]
    pos = torch.repeat_interleave(torch.arange(deg.numel(), device=deg.device), deg)
    if s["weights"] == "f32":
        return s["weight"], pos
    lane = torch.arange(pos.numel(), device=pos.device) - s["offsets"][pos]
    flat = _values(s["wcodes"], s["wscales"][:, None], s["weights"], BLOCK).reshape(-1)
    return flat[s["block_offsets"][pos] * BLOCK + lane], pos


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _activations(g, n, b, act="relu"):
    """Rows as a layer leaves them: a spread of sizes from unit to unit, some units silent throughout."""
    x = torch.randn((n, b), generator=g, device=DEVICE)
    x *= torch.exp(torch.randn((n, 1), generator=g, device=DEVICE))
    x = torch.tanh(x) if act in ("tanh", "sigmoid") else torch.clamp_min(x, 0.0) if act == "relu" else x
    x *= (torch.rand((n, 1), generator=g, device=DEVICE) > 0.05)
    return x


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    op = case["op"]
    s = {"op": op, "fmt": case.get("fmt")}
    if op == "quantize":
        n, b = case["units"], case["batch"]
        x = _activations(g, n, b, "relu" if case["keep"] else "tanh").to(DTYPES[case["dtype"]])
        s |= {"x": x.t().contiguous().t() if case["by_sample"] else x, "keep": case["keep"]}
    elif op == "dequantize":
        n, b = case["units"], case["batch"]
        codes, scales = _quantize(_activations(g, n, b, "tanh"), case["fmt"])
        s |= {"codes": codes, "scales": scales, "batch": b, "dtype": DTYPES[case["dtype"]]}
    elif op == "unit_grad":
        n, b = case["units"], case["batch"]
        codes, scales = _quantize(_activations(g, n, b, case["act"]), case["fmt"], True)
        s |= {"codes": codes, "scales": scales, "batch": b, "act": case["act"],
              "acc": torch.randn((n, b), generator=g, device=DEVICE) * 0.1,
              "seed_rows": torch.randn((n, b), generator=g, device=DEVICE) if case["seed_rows"] else None,
              "out": torch.empty((n, b), device=DEVICE)}
    elif op == "edge_grad":
        ns, nt, slots, live, b = (case[k] for k in ("sources", "targets", "slots", "live", "batch"))
        n = ns + nt
        src = torch.randint(0, ns, (slots,), generator=g, device=DEVICE, dtype=torch.int32)
        grown = int(live * case["grown"])
        src[:live - grown] = src[:live - grown].sort().values  # built source-major, then regrown slots in any order
        dead = (torch.arange(slots, device=DEVICE) >= live).to(torch.uint8)
        if grown:  # pruned slots among the live ones
            dead[torch.randint(0, live, (grown,), generator=g, device=DEVICE)] = 1
        codes, scales = _quantize(_activations(g, n, b), case["fmt"], True)
        s |= {"bucket": {"from_id": src, "dead": dead, "to_id": torch.randint(
            ns, n, (slots,), generator=g, device=DEVICE, dtype=torch.int32)},
            "grad": torch.randn((n, b), generator=g, device=DEVICE) * 0.01, "codes": codes, "scales": scales,
            "batch": b}
    else:
        ns, nt, fan, b = (case[k] for k in ("sources", "targets", "fan_in", "batch"))
        n = ns + nt
        deg = torch.poisson(torch.full((nt,), float(fan), device=DEVICE), generator=g).to(torch.int64)
        zero = torch.zeros(1, dtype=torch.int64, device=DEVICE)
        s |= {"offsets": torch.cat([zero, deg.cumsum(0)]), "block_offsets": torch.cat([zero, ((deg + 31) // 32).cumsum(0)]),
              "units": torch.arange(ns, n, dtype=torch.int32, device=DEVICE), "weights": case["weights"],
              "act": case["act"], "rows": case["rows"], "out_fmt": case["out"], "batch": b, "num_units": n}
        edges = int(s["offsets"][-1])
        s["src"] = torch.randint(0, ns, (edges,), generator=g, device=DEVICE, dtype=torch.int32)
        w = torch.randn((edges,), generator=g, device=DEVICE) / math.sqrt(fan)
        if case["weights"] == "f32":
            s["weight"] = w
        else:
            blocks = torch.zeros((int(s["block_offsets"][-1]) * BLOCK,), device=DEVICE)
            pos = torch.repeat_interleave(torch.arange(nt, device=DEVICE), deg)
            blocks[s["block_offsets"][pos] * BLOCK + torch.arange(edges, device=DEVICE) - s["offsets"][pos]] = w
            codes, scales = _quantize(blocks.reshape(-1, BLOCK), case["weights"])
            s |= {"wcodes": codes, "wscales": scales.reshape(-1)}
        x = _activations(g, n, b)
        if case["rows"] == "f32":
            s["x"] = x
        else:
            s["codes"], s["scales"] = _quantize(x, case["rows"])
        if case["out"] == "f32":
            s["out"] = torch.zeros((n, b), device=DEVICE)
        else:
            nb = -(-b // BLOCK)
            s["out_codes"] = torch.zeros((n, nb * BLOCK * FORMATS[case["out"]][3] // 8), dtype=torch.uint8, device=DEVICE)
            s["out_scales"] = torch.zeros((n, nb), dtype=torch.uint8, device=DEVICE)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_plain(s):
    op = s["op"]
    if op == "quantize":
        return _quantized_values(s["x"].float(), s["fmt"], s["keep"]).to(torch.bfloat16)
    if op == "dequantize":
        return _values(s["codes"], s["scales"], s["fmt"], s["batch"]).to(s["dtype"])
    if op == "unit_grad":
        a = _values(s["codes"], s["scales"], s["fmt"], s["batch"])
        up = s["acc"] if s["seed_rows"] is None else s["acc"] + s["seed_rows"]
        return up * _act_prime(s["act"], a)
    if op == "edge_grad":
        a = _values(s["codes"], s["scales"], s["fmt"], s["batch"])
        b = s["bucket"]
        dw = (s["grad"][b["to_id"].long()] * a[b["from_id"].long()]).sum(dim=1) / s["batch"]
        return torch.where(b["dead"] == 0, dw, torch.zeros_like(dw))
    w, pos = _weight_values(s)
    x = s["x"] if s["rows"] == "f32" else _values(s["codes"], s["scales"], s["rows"], s["batch"])
    y = torch.zeros((s["units"].numel(), s["batch"]), device=DEVICE)
    y.index_add_(0, pos, w[:, None] * x[s["src"].long()])
    y = _act(s["act"], y)
    if s["out_fmt"] != "f32":
        y = _quantized_values(y, s["out_fmt"]).to(torch.bfloat16)
    out = torch.zeros((s["num_units"], s["batch"]), dtype=y.dtype, device=DEVICE)
    out[s["units"].long()] = y
    return out


def _run_own(s):
    import plastax_b200 as px

    op = s["op"]
    if op == "quantize":
        return px.mx_dequantize(px.mx_quantize(s["x"], s["fmt"], keep_nonzero=s["keep"]), dtype=torch.bfloat16)
    if op == "dequantize":
        return px.mx_dequantize(px.MxRows(s["codes"], s["scales"], s["fmt"], s["batch"]), dtype=s["dtype"])
    if op == "unit_grad":
        rows = px.MxRows(s["codes"], s["scales"], s["fmt"], s["batch"])
        return px.mx_unit_grad(s["acc"], rows, s["act"], seed=s["seed_rows"], out=s["out"])
    if op == "edge_grad":
        return px.mx_edge_grad(s["bucket"], s["grad"], px.MxRows(s["codes"], s["scales"], s["fmt"], s["batch"]))
    conns = px.MxConns(units=s["units"], offsets=s["offsets"], src=s["src"], weights=s["weights"],
                       weight=s.get("weight"), block_offsets=s["block_offsets"], codes=s.get("wcodes"),
                       scales=s.get("wscales"))
    x = s["x"] if s["rows"] == "f32" else px.MxRows(s["codes"], s["scales"], s["rows"], s["batch"])
    if s["out_fmt"] == "f32":
        return px.mx_product(conns, x, activation=s["act"], out=s["out"])
    out = px.MxRows(s["out_codes"], s["out_scales"], s["out_fmt"], s["batch"])
    return px.mx_dequantize(px.mx_product(conns, x, activation=s["act"], out=out), dtype=torch.bfloat16)


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without, and what it should give
# ---------------------------------------------------------------------------------------------------------------------
def _mx_bytes(n, b, fmt):
    return n * -(-b // BLOCK) * (BLOCK * FORMATS[fmt][3] // 8 + 1)


def work(case):
    op, b = case["op"], case["batch"]
    if op == "quantize":  # the rows are written narrow, and read back as bfloat16
        n = case["units"]
        return {"bytes": n * b * (DTYPES[case["dtype"]].itemsize + 2) + 2 * _mx_bytes(n, b, case["fmt"]),
                "flops": 4 * n * b}
    if op == "dequantize":
        n = case["units"]
        return {"bytes": n * b * DTYPES[case["dtype"]].itemsize + _mx_bytes(n, b, case["fmt"]), "flops": 2 * n * b}
    if op == "unit_grad":
        n = case["units"]
        return {"bytes": n * b * (12 if case["seed_rows"] else 8) + _mx_bytes(n, b, case["fmt"]), "flops": 4 * n * b}
    if op == "edge_grad":
        rows = case["targets"] * b * 4 + _mx_bytes(case["sources"], b, case["fmt"])
        return {"bytes": case["slots"] * 13 + rows, "flops": 2 * case["live"] * b}
    edges = case["targets"] * case["fan_in"]
    w = 4 if case["weights"] == "f32" else FORMATS[case["weights"]][3] / 8 + 1 / 32
    x = case["sources"] * b * 4 if case["rows"] == "f32" else _mx_bytes(case["sources"], b, case["rows"])
    y = case["targets"] * b * 4 if case["out"] == "f32" else _mx_bytes(case["targets"], b, case["out"])
    return {"bytes": int(edges * (4 + w)) + case["targets"] * 20 + x + y, "flops": 2 * edges * b}


def _table(fmt):
    """Every element's value, by its code."""
    mant, emin, _, bits = FORMATS[fmt]
    vals = []
    for c in range(1 << bits):
        sign = -1.0 if c >> (bits - 1) else 1.0
        field, frac = (c & ((1 << (bits - 1)) - 1)) >> mant, c & ((1 << mant) - 1)
        vals.append(sign * (math.ldexp(1 + frac / (1 << mant), field - 1 + emin) if field else
                            math.ldexp(frac / (1 << mant), emin)))
    return torch.tensor(vals, dtype=torch.float64, device=DEVICE)


def _powers():
    """2^(i - 127) at i."""
    return torch.tensor([math.ldexp(1.0, i - 127) for i in range(256)], dtype=torch.float64, device=DEVICE)


def _exact_values(codes, scales, fmt, batch):
    t = _table(fmt)
    idx = codes.long()
    if FORMATS[fmt][3] == 4:
        idx = torch.stack([idx % 16, idx // 16], dim=-1).flatten(1)
    s = _powers()[scales.long()]
    return (t[idx] * s.repeat_interleave(BLOCK, dim=1))[:, :batch]


def _exact_quantized(y, fmt, keep=False):
    """Nearest element of each block's grid, found in the sorted list of magnitudes; ties to the even code."""
    n, b = y.shape
    nb = -(-b // BLOCK)
    mags = _table(fmt)[:1 << (FORMATS[fmt][3] - 1)]
    mags = mags[mags <= FORMATS[fmt][2]]
    full = torch.zeros((n, nb * BLOCK), dtype=torch.float64, device=DEVICE)
    full[:, :b] = y
    blk = full.reshape(n, nb, BLOCK)
    top = blk.abs().amax(dim=2, keepdim=True)
    p = _powers()
    s = p[torch.searchsorted(p * mags[-1], top)]  # the first power that holds the block's largest
    z = (blk / s).abs()
    i = torch.searchsorted(mags, z).clamp(1, mags.numel() - 1)
    lo, hi = mags[i - 1], mags[i]
    up = (z - lo > hi - z) | ((z - lo == hi - z) & (i % 2 == 0))
    near = torch.where(up, hi, lo)
    if keep:
        near = near.clamp(min=mags[1])
    return (near * blk.sign() * s).reshape(n, -1)[:, :b]


def exact(case, seed):
    op = case["op"]
    s = prepare(case, seed)
    if op == "quantize":
        return _exact_quantized(s["x"].double(), s["fmt"], s["keep"])
    if op == "dequantize":
        return _exact_values(s["codes"], s["scales"], s["fmt"], s["batch"])
    if op == "unit_grad":
        a = _exact_values(s["codes"], s["scales"], s["fmt"], s["batch"])
        prime = {"tanh": lambda: 1 - a ** 2, "relu": lambda: (a > 0).double(), "sigmoid": lambda: a - a ** 2,
                 "identity": lambda: torch.ones_like(a)}[s["act"]]()
        seed_rows = 0.0 if s["seed_rows"] is None else s["seed_rows"].double()
        return (s["acc"].double() + seed_rows) * prime
    if op == "edge_grad":
        a = _exact_values(s["codes"], s["scales"], s["fmt"], s["batch"])
        g, b = s["grad"].double(), s["bucket"]
        out = torch.zeros(b["dead"].numel(), dtype=torch.float64, device=DEVICE)
        for part in torch.nonzero(b["dead"] == 0).flatten().split(1 << 19):
            f, t = b["from_id"][part].long(), b["to_id"][part].long()
            out[part] = torch.einsum("eb,eb->e", g[t], a[f]) / s["batch"]
        return out
    nt, b = s["units"].numel(), s["batch"]
    x = s["x"].double() if s["rows"] == "f32" else _exact_values(s["codes"], s["scales"], s["rows"], b)
    dst = torch.bucketize(torch.arange(s["src"].numel(), device=DEVICE), s["offsets"][1:], right=True)
    if s["weights"] == "f32":
        w = s["weight"].double()
    else:
        grid = _exact_values(s["wcodes"], s["wscales"].reshape(-1, 1), s["weights"], BLOCK)
        at = torch.arange(dst.numel(), device=DEVICE) - s["offsets"][:-1][dst]
        w = grid[s["block_offsets"][:-1][dst] + at // BLOCK, at % BLOCK]
    y = torch.zeros((nt, b), dtype=torch.float64, device=DEVICE)
    for part in torch.arange(dst.numel(), device=DEVICE).split(1 << 19):
        y.index_add_(0, dst[part], w[part, None] * x[s["src"][part].long()])
    y = {"tanh": torch.tanh, "relu": torch.relu, "sigmoid": torch.sigmoid, "identity": lambda v: v}[s["act"]](y)
    if s["out_fmt"] != "f32":
        y = _exact_quantized(y, s["out_fmt"])
    out = torch.zeros((s["num_units"], b), dtype=torch.float64, device=DEVICE)
    out[s["units"].long()] = y
    return out
