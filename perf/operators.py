"""Timed cases of the mixture-of-experts operators: microscaled 4-bit (MXFP4) quantisation and products, expert routing,
products grouped by expert, and the weighted sum of the experts' rows.

Kinds of case:

  quantize  rows to MXFP4 and back: the values that the codes stand for
  product   one MXFP4 matrix times fp32 rows ("x": "f32"), or times rows that the pass quantises first ("x": "mxfp4")
  route     router logits to experts, weights, and the rows sorted by expert
  experts   rows grouped by expert times their experts' matrices, (gate, up) pairs or plain ones
  combine   each token's sum of its experts' rows

Sizes are those of the 3B model that the benchmark uses (hidden 2560, MLP 6912, a quarter of it for an expert) or generic.
"""
import math

import numpy as np
import torch

own = False  # true: the framework's kernels; false: the plain forms

# Type codes as in a GGUF file.
CODES = {"f32": 0, "f16": 1, "bf16": 30, "mxfp4": 39}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # One decode step's activations, eight sequences: the smallest call, bound by launches.
        dict(name="quantize_step", kind="quantize", n=8, cols=2560, pad=0, dtype="f32"),
        # The MLP activations of a long prompt, rows of a wider buffer.
        dict(name="quantize_prompt", kind="quantize", n=8192, cols=6912, pad=64, dtype="bf16"),
        # A decode step of one sequence through an MXFP4 matrix.
        dict(name="product_row", kind="product", n=1, rows=6912, cols=2560, x="f32"),
        # A prompt, no multiple of any tile, at fp32 accuracy.
        dict(name="product_prompt", kind="product", n=1999, rows=6912, cols=2560, x="f32"),
        # A large batch of prompts with both operands in 4 bits: the largest case.
        dict(name="product_mx_prompt", kind="product", n=8192, rows=13824, cols=2560, x="mxfp4"),
        # Routing of a decode step.
        dict(name="route_step", kind="route", n=16, experts=64, k=4, over_all=False, dtype="f32", masked=0.0, padded=0.0),
        # Routing of a batch of prompts: half-precision logits, some experts masked for a token, padded tokens.
        dict(name="route_prompt", kind="route", n=16384, experts=128, k=8, over_all=True, dtype="bf16", masked=0.1,
             padded=0.05),
        # Decoding, 16 sequences: gate and up of the experts that their tokens chose, a few rows for each.
        dict(name="experts_step", kind="experts", n=16, k=4, experts=32, rows=1728, cols=2560, w="mxfp4", x="f32",
             gate=True, out="f32", skew=0.5),
        # A prompt through half-precision experts: the down products, rows already in expert order.
        dict(name="experts_bf16_prompt", kind="experts", n=2048, k=2, experts=8, rows=2560, cols=1728, w="bf16", x="bf16",
             gate=False, out="f32", skew=0.5),
        # Prompts through many small experts, both operands in 4 bits, an uneven load.
        dict(name="experts_mx_prompt", kind="experts", n=4096, k=4, experts=64, rows=1728, cols=2560, w="mxfp4", x="mxfp4",
             gate=True, out="bf16", skew=1.0),
        # The sum after a decode step.
        dict(name="combine_step", kind="combine", n=16, k=4, cols=2560, dtype="f32", out="f32", dropped=0.0),
        # The sum after a batch of prompts, half-precision rows, some slots without an expert.
        dict(name="combine_prompt", kind="combine", n=8192, k=8, cols=2560, dtype="bf16", out="bf16", dropped=0.05),
    ]


def _log(rng, low, high):
    """An integer in [low, high], even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["quantize", "product", "product", "route", "experts", "experts", "experts", "combine"])
    if kind == "quantize":
        return dict(kind=kind, n=_log(rng, 1, 8192), cols=32 * _log(rng, 1, 216), pad=rng.choice([0, 1, 64]),
                    dtype=rng.choice(["f32", "f16", "bf16"]))
    if kind == "product":
        return dict(kind=kind, n=_log(rng, 1, 4096), rows=_log(rng, 64, 8192), cols=32 * _log(rng, 2, 216),
                    x=rng.choice(["f32", "mxfp4"]))
    if kind == "route":
        experts = _log(rng, 4, 256)
        return dict(kind=kind, n=_log(rng, 1, 16384), experts=experts, k=rng.randint(1, min(8, experts)),
                    over_all=rng.random() < 0.5, dtype=rng.choice(["f32", "f16", "bf16"]),
                    masked=rng.choice([0.0, 0.2]), padded=rng.choice([0.0, 0.1]))
    if kind == "experts":
        experts = _log(rng, 4, 64)
        w, x = rng.choice([("mxfp4", "f32"), ("mxfp4", "f16"), ("mxfp4", "bf16"), ("mxfp4", "mxfp4"), ("mxfp4", "mxfp4"),
                           ("bf16", "f32"), ("bf16", "f16"), ("bf16", "bf16")])
        cols = 32 * _log(rng, 4, 96) if w == "mxfp4" else 8 * _log(rng, 16, 384) + rng.choice([0, 0, 3])
        return dict(kind=kind, n=_log(rng, 1, 4096), k=rng.randint(1, 4), experts=experts, rows=_log(rng, 64, 2048),
                    cols=cols, w=w, x=x, gate=rng.random() < 0.5, out=rng.choice(["f32", "f16", "bf16"]),
                    skew=rng.choice([0.0, 0.5, 1.5]))
    return dict(kind=kind, n=_log(rng, 1, 8192), k=rng.randint(1, 8), cols=_log(rng, 64, 4096),
                dtype=rng.choice(["f32", "f16", "bf16"]), out=rng.choice(["f32", "f16", "bf16"]),
                dropped=rng.choice([0.0, 0.1]))


# ------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _activations(g, n, cols, dtype):
    """Normal rows whose channels differ in size, as a residual stream's do."""
    return (_normal(g, n, cols) * (0.5 * _normal(g, cols)).exp()).to(TYPES[dtype])


def _blocks(g, *shape):
    """MXFP4 matrices as GGUF blocks on the GPU, uint8 [..., cols / 32, 17]: scale bytes about 2^-7, uniform codes."""
    *lead, cols = shape
    e = torch.randint(118, 123, (*lead, cols // 32, 1), generator=g, device="cuda", dtype=torch.uint8)
    q = torch.randint(0, 256, (*lead, cols // 32, 16), generator=g, device="cuda", dtype=torch.uint8)
    return torch.cat([e, q], -1)


def _groups(case, g):
    """(token of each row, rows of each expert): k different experts for each token, drawn by an uneven popularity."""
    n, k, experts = case["n"], case["k"], case["experts"]
    score = case["skew"] * _normal(g, experts) - (-_rand(g, n, experts).clamp_min(1e-12).log()).clamp_min(1e-12).log()
    ids = score.topk(k, -1).indices.reshape(-1)
    return (ids.sort(stable=True).indices // k).to(torch.int32), torch.bincount(ids, minlength=experts).tolist()


def _draw_experts(case, seed):
    """x, the matrices (raw, one or two of [experts][rows] each), the row index (None: rows in order) and the counts."""
    g = _gen(seed)
    tokens, counts = _groups(case, g)
    mats = []
    for _ in range(2 if case["gate"] else 1):
        if case["w"] == "mxfp4":
            mats.append(_blocks(g, case["experts"], case["rows"], case["cols"]))
        else:
            mats.append((_normal(g, case["experts"], case["rows"], case["cols"]) * 0.02).bfloat16())
    dtype = "bf16" if case["x"] == "mxfp4" else case["x"]
    x = _activations(g, case["n"] if case["gate"] else len(tokens), case["cols"], dtype)
    return x, mats, tokens if case["gate"] else None, counts


def _draw_route(case, seed):
    g = _gen(seed)
    n, experts = case["n"], case["experts"]
    x = _normal(g, n, experts) * 1.5 + 0.5 * _normal(g, experts)
    x = x.masked_fill(_rand(g, n, experts) < case["masked"], -math.inf)
    return x.masked_fill(_rand(g, n, 1) < case["padded"], -math.inf).to(TYPES[case["dtype"]])


def _draw_combine(case, seed):
    """Expert rows in sorted order, each slot's row (-1: none) and weight."""
    g = _gen(seed)
    n, k = case["n"], case["k"]
    y = _normal(g, n * k, case["cols"]).to(TYPES[case["dtype"]])
    positions = torch.randperm(n * k, generator=g, device="cuda").to(torch.int32).reshape(n, k)
    positions = positions.masked_fill(_rand(g, n, k) < case["dropped"], -1)
    weights = _normal(g, n, k).exp()
    return y, positions, weights / weights.sum(-1, keepdim=True)


_stream = []  # the one stream that the program runs its operators on


def _empty(*shape, dtype="f32"):
    return torch.empty(*shape, dtype=TYPES.get(dtype, dtype), device="cuda")


def prepare(case, seed):
    kind, s = case["kind"], dict(case=case)
    if kind == "quantize":
        wide = _activations(_gen(seed), case["n"], case["cols"] + case["pad"], case["dtype"])
        s.update(x=wide[:, :case["cols"]])
    elif kind == "product":
        g = _gen(seed)
        s.update(raw=_blocks(g, case["rows"], case["cols"]), x=_activations(g, case["n"], case["cols"], "f32"))
    elif kind == "route":
        s.update(logits=_draw_route(case, seed))
    elif kind == "experts":
        x, mats, index, counts = _draw_experts(case, seed)
        offsets = torch.tensor([0] + np.cumsum(counts).tolist(), dtype=torch.int32, device="cuda")
        s.update(x=x, mats=mats, index=index, counts=counts, offsets=offsets)
    else:
        y, positions, weights = _draw_combine(case, seed)
        s.update(y=y, positions=positions, weights=weights)
    if own:
        _prepare_own(case, s)
    torch.cuda.synchronize()
    return s


def _prepare_own(case, s):
    """The handles and buffers that a program keeps."""
    from tinyoai_amd import hip
    from tinyoai_amd import weights as W
    kind, n = case["kind"], case["n"]
    if not _stream:
        _stream.append(torch.cuda.Stream())
    s.update(hip=hip, stream=_stream[0].cuda_stream)
    if kind == "quantize":
        s.update(out=_empty(n, case["cols"], dtype="bf16" if case["dtype"] == "bf16" else "f32"))
    elif kind == "product":
        t = W.Tensor(CODES["mxfp4"], case["rows"], case["cols"], s["raw"].cpu().numpy().reshape(-1))
        s.update(w=hip.Weight(t), out=_empty(n, case["rows"]))
    elif kind == "route":
        slots, i32 = n * case["k"], torch.int32
        s.update(ids=_empty(n, case["k"], dtype=i32), weights=_empty(n, case["k"]),
                 offsets=_empty(case["experts"] + 1, dtype=i32), tokens=_empty(slots, dtype=i32),
                 positions=_empty(n, case["k"], dtype=i32))
    elif kind == "experts":
        mats = [m.view(torch.uint8).cpu().numpy().reshape(-1) for m in s["mats"]]
        s.update(e=hip.Experts(CODES[case["w"]], case["experts"], case["rows"], case["cols"], *mats),
                 out=_empty(n * case["k"], case["rows"], dtype=case["out"]))
    else:
        s.update(out=_empty(n, case["cols"], dtype=case["out"]))
    if kind == "quantize" or case.get("x") == "mxfp4":  # the rows' codes and scales, rows padded to 128 values
        m, units = len(s["x"]), -(-case["cols"] // 128)
        s.update(codes=_empty(m, 64 * units, dtype=torch.uint8), scales=_empty(m, 4 * units, dtype=torch.uint8))


# ------------------------------------------------------------ one pass
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    case, hip, stream = s["case"], s["hip"], s["stream"]
    kind, n = case["kind"], case["n"]
    if "codes" in s:
        x, codes, scales = s["x"], s["codes"].data_ptr(), s["scales"].data_ptr()
        dtype = next(CODES[name] for name, t in TYPES.items() if t == x.dtype)
        hip.quantize_mxfp4(dtype, x.data_ptr(), x.stride(0), len(x), case["cols"], codes, scales, stream)
    if kind == "quantize":
        out = s["out"]
        dtype = CODES["bf16" if case["dtype"] == "bf16" else "f32"]
        hip.dequantize_mxfp4(codes, scales, n, case["cols"], dtype, out.data_ptr(), case["cols"], stream)
        return out
    if kind == "product":
        if case["x"] == "mxfp4":
            s["w"].mul_mxfp4_device(codes, scales, n, s["out"].data_ptr(), stream)
        else:
            s["w"].mul_device(s["x"].data_ptr(), n, s["out"].data_ptr(), stream)
        return s["out"]
    if kind == "route":
        x = s["logits"]
        names = ("ids", "weights", "offsets", "tokens", "positions")
        hip.route(CODES[case["dtype"]], x.data_ptr(), x.stride(0), n, case["experts"], case["k"], case["over_all"],
                  *(s[name].data_ptr() for name in names), stream)
        return {name: s[name] for name in names}
    if kind == "experts":
        x, out = s["x"], s["out"]
        index = s["index"].data_ptr() if case["gate"] else 0
        data = (codes, scales) if case["x"] == "mxfp4" else (x.data_ptr(), 0)
        s["e"].mul_device(CODES[case["x"]], *data, case["cols"], len(x), s["offsets"].data_ptr(), index, len(out),
                          CODES[case["out"]], out.data_ptr(), case["rows"], stream)
        return out
    y, out = s["y"], s["out"]
    hip.combine(CODES[case["dtype"]], y.data_ptr(), case["cols"], len(y), s["positions"].data_ptr(),
                s["weights"].data_ptr(), n, case["k"], case["cols"], CODES[case["out"]], out.data_ptr(), case["cols"], stream)
    return out


def _values(raw, cols):
    """The fp32 values of GGUF MXFP4 blocks uint8 [..., cols / 32, 17]: byte j of a block's 16 holds values j and j + 16."""
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=raw.device)
    q = raw[..., 1:]
    scale = (raw[..., :1].int() << 23).view(torch.float32)  # 2^(e - 127); e is never 0 here
    return (table[torch.cat([q & 15, q >> 4], -1).int()] * scale).reshape(*raw.shape[:-2], cols)


def _rounded(x):
    """The values of x's MXFP4 form: blocks of 32 scaled by a power of two, to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6."""
    b = x.float().reshape(x.shape[0], -1, 32)
    e = (torch.frexp(b.abs().amax(-1, keepdim=True)).exponent - 3).clamp(-127, 127)
    y = b * ((127 - e) << 23).view(torch.float32)  # times 2^-e
    a = y.abs()
    a = torch.where(a < 2, (a * 2).round() / 2, torch.where(a < 4, a.round(), (a / 2).round() * 2)).clamp_max(6)
    scale = torch.where(e > -127, (e + 127) << 23, 1 << 22).view(torch.float32)
    return (a.copysign(y) * scale).reshape(x.shape)


def _run_plain(s):
    case = s["case"]
    kind, n = case["kind"], case["n"]
    if kind == "quantize":
        return _rounded(s["x"]).to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
    if kind == "route":
        return _route_plain(s["logits"].float(), case)
    if kind == "combine":
        pos = s["positions"].long()
        rows = s["y"].float()[pos.clamp_min(0)] * s["weights"][..., None]
        return torch.where((pos >= 0)[..., None], rows, 0.0).sum(1).to(TYPES[case["out"]])
    x = _rounded(s["x"]) if case["x"] == "mxfp4" else s["x"].float()
    if kind == "product":
        return x @ _values(s["raw"], case["cols"]).T
    out = _empty(n * case["k"], case["rows"], dtype=case["out"])
    row = 0
    for e, count in enumerate(s["counts"]):
        if not count:
            continue
        rows = slice(row, row + count)
        xe = x[s["index"][rows].long()] if case["gate"] else x[rows]
        y = [xe @ (_values(m[e], case["cols"]) if case["w"] == "mxfp4" else m[e].float()).T for m in s["mats"]]
        out[rows] = y[0] / (1 + (-y[0]).exp()) * y[1] if case["gate"] else y[0]
        row += count
    return out


def _route_plain(x, case):
    n, experts, k = case["n"], case["experts"], case["k"]
    x = torch.where(x > -math.inf, x, -math.inf)  # NaN too is never chosen
    top, ids = (t[:, :k] for t in x.sort(dim=-1, descending=True, stable=True))
    valid = top > -math.inf
    most = torch.where(valid[:, :1], top[:, :1], 0.0)
    weights = (top - most).exp()
    total = (x - most).exp().sum(-1, keepdim=True) if case["over_all"] else weights.sum(-1, keepdim=True)
    weights = torch.where(valid, weights / total, 0.0)
    ids = torch.where(valid, ids, -1).to(torch.int32)
    flat = torch.where(ids < 0, experts, ids).reshape(-1)
    order = flat.sort(stable=True).indices
    ends = (flat[:, None] == torch.arange(experts, device="cuda")).sum(0).cumsum(0)
    offsets = torch.cat([torch.zeros_like(ends[:1]), ends]).to(torch.int32)
    row = torch.arange(n * k, device="cuda", dtype=torch.int32)
    routed = row < offsets[-1]
    tokens = torch.where(routed, order // k, -1).to(torch.int32)
    positions = torch.empty_like(row)
    positions[order] = torch.where(routed, row, -1)
    return dict(ids=ids, weights=weights, offsets=offsets, tokens=tokens, positions=positions.reshape(n, k))


# ------------------------------------------------------------ what a pass costs
def _mx_bytes(values):
    return values * 17 // 32


def work(case):
    kind, n = case["kind"], case["n"]
    size = {name: t.itemsize for name, t in TYPES.items()}
    if kind == "quantize":  # the values in, codes and scales, the values that they stand for
        values = n * case["cols"]
        return {"bytes": values * (size[case["dtype"]] + (2 if case["dtype"] == "bf16" else 4)) + _mx_bytes(values),
                "flops": 3 * values}
    if kind == "product":
        rows, cols = case["rows"], case["cols"]
        return {"bytes": _mx_bytes(rows * cols) + 4 * n * (rows + cols), "flops": 2 * n * rows * cols}
    if kind == "route":
        values, slots = n * case["experts"], n * case["k"]
        return {"bytes": values * size[case["dtype"]] + 16 * slots + 4 * case["experts"] + 4,
                "flops": values * (case["k"] + 2)}
    slots = n * case["k"]
    if kind == "experts":  # the experts that some token chose, were the choice even
        rows, cols = case["rows"] * (2 if case["gate"] else 1), case["cols"]
        hit = case["experts"] * (1 - (1 - case["k"] / case["experts"]) ** n)
        matrix = _mx_bytes(rows * cols) if case["w"] == "mxfp4" else 2 * rows * cols
        x = (n if case["gate"] else slots) * cols * size["bf16" if case["x"] == "mxfp4" else case["x"]]
        return {"bytes": int(hit * matrix) + x + slots * case["rows"] * size[case["out"]] + 4 * slots,
                "flops": 2 * slots * rows * cols}
    return {"bytes": slots * (case["cols"] * size[case["dtype"]] + 8) + n * case["cols"] * size[case["out"]],
            "flops": 2 * slots * case["cols"]}


# ------------------------------------------------------------ 64 bits
def _mx64(x):
    """MXFP4 by its definition in 64 bits: the scale's exponent is that of the largest magnitude less 2 (that of 6, the
    largest code); a magnitude goes to the code whose interval of halfway points holds it, halfway ones to the even code."""
    b = x.double().unflatten(-1, (-1, 32))
    most = b.abs().amax(-1, keepdim=True)
    exponent = torch.where(most > 0, (torch.frexp(most).exponent - 1).double() - 2, -127.0).clamp(-127, 127)
    scale = torch.pow(torch.full_like(exponent, 2.0), exponent)
    m = b.abs() / scale
    code = torch.zeros_like(m, dtype=torch.long)
    for half, up in ((.25, False), (.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (m >= half) if up else (m > half)
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    return (grid[code] * b.sign() * scale).flatten(-2)


def _raw64(raw):
    """Blocks to float64: the code's sign, exponent and fraction bits taken apart."""
    q = torch.stack([raw[..., 1:] & 15, raw[..., 1:] >> 4], -2).long()  # values 0..15, 16..31
    e, f = (q >> 1) & 3, (q & 1).double()
    v = torch.where(e == 0, f * .5, (1 + f * .5) * (2.0 ** (e - 1).double())) * (1 - 2 * (q >> 3)).double()
    return (v.flatten(-2) * (2.0 ** (raw[..., :1].double() - 127))).flatten(-2)


def exact(case, seed):
    kind, n = case["kind"], case["n"]
    if kind == "quantize":
        return _mx64(_activations(_gen(seed), n, case["cols"] + case["pad"], case["dtype"])[:, :case["cols"]])
    if kind == "product":
        g = _gen(seed)
        w = _raw64(_blocks(g, case["rows"], case["cols"]))
        x = _activations(g, n, case["cols"], "f32")
        return (_mx64(x) if case["x"] == "mxfp4" else x.double()) @ w.T
    if kind == "route":
        return _route64(_draw_route(case, seed).double().cpu().numpy(), case["k"], case["over_all"])
    if kind == "experts":
        x, mats, index, counts = _draw_experts(case, seed)
        x = _mx64(x) if case["x"] == "mxfp4" else x.double()
        if index is not None:
            x = x.index_select(0, index.long())
        parts = []
        for e, xe in enumerate(x.split(counts)):
            y = [xe @ (_raw64(m[e]) if case["w"] == "mxfp4" else m[e].double()).T for m in mats]
            parts.append(y[0] * torch.sigmoid(y[0]) * y[1] if case["gate"] else y[0])
        return torch.cat(parts)
    y, positions, weights = _draw_combine(case, seed)
    out = torch.zeros(n, case["cols"], dtype=torch.float64, device="cuda")
    for j in range(case["k"]):
        t = (positions[:, j] >= 0).nonzero()[:, 0]
        out[t] += y[positions[t, j].long()].double() * weights[t, j, None].double()
    return out


def _route64(x, k, over_all):
    n, experts = x.shape
    ids = np.lexsort((np.broadcast_to(np.arange(experts), x.shape), -x), axis=-1)[:, :k]
    chosen = np.take_along_axis(x, ids, -1)
    ok = chosen > -np.inf
    top = np.where(ok[:, :1], chosen[:, :1], 0)
    weights = np.exp(chosen - top)
    with np.errstate(invalid="ignore"):
        weights = np.where(ok, weights / (np.exp(x - top) if over_all else weights).sum(-1, keepdims=True), 0)
    flat = np.where(ok, ids, experts).reshape(-1)
    total = int(ok.sum())
    order = np.argsort(flat, kind="stable")[:total]
    tokens = np.full(n * k, -1, np.int32)
    tokens[:total] = order // k
    positions = np.full(n * k, -1, np.int32)
    positions[order] = np.arange(total)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat, minlength=experts + 1)[:experts])])
    return dict(ids=np.where(ok, ids, -1).astype(np.int32), weights=weights, offsets=offsets.astype(np.int32),
                tokens=tokens, positions=positions.reshape(n, k))
