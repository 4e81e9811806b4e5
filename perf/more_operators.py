"""Timed cases of the attention operators that a serving program runs beside its weight products: rotary positions, the
paged key-value cache, the attention of new tokens over its pages, and the attention of packed prompts.

Kinds of case:

  rope    rows of query and key heads turned by their positions
  cache   rows of keys and values written to slots of a paged cache, quantised for 8-bit pages, and read back
  attend  one new token of each sequence over its pages
  prompt  packed sequences of queries over packed keys and values, causal or not

Head layouts are those of the repository's benchmark and tests (32 heads of 80, 22 of 128, 32 over 8 of 64, 8 over 4 of 8)
or generic.
"""
import math

import torch

own = False  # true: the framework's kernels; false: the plain forms

# Type codes as in a GGUF file.
CODES = {"f32": 0, "f16": 1, "q8_0": 8, "bf16": 30}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# Position scalings: (kind, factor, context of the training, low, high), low and high as the kind takes them.
SCALINGS = {"none": ("none", 1.0, 0, 0.0, 0.0), "linear": ("linear", 4.0, 0, 0.0, 0.0),
            "bands": ("bands", 8.0, 8192, 1.0, 4.0), "yarn": ("yarn", 16.0, 4096, 1.0, 32.0)}


def listed():
    return [
        # Queries and keys of a decode step of four chats, a quarter of each head turned: the smallest call.
        dict(name="rope_step", kind="rope", n=4, heads=64, hd=80, rot=20, layout="half", theta=1e4, scaling="none",
             pad=0, dtype="f32", out="f32", far=1000),
        # A batch of long documents, far positions, in the buffer of the fused projection (values follow the keys).
        dict(name="rope_prompt", kind="rope", n=8192, heads=40, hd=128, rot=128, layout="interleaved", theta=5e5,
             scaling="bands", pad=1024, dtype="bf16", out="bf16", far=130000),
        # The new keys and values of a decode step into 8-bit pages.
        dict(name="cache_step", kind="cache", n=16, kv_heads=8, hd=128, type="q8_0", page=64, pad=0, dtype="f32",
             dropped=0.0),
        # A batch of prompts into 8-bit pages, rows of the fused projection's buffer, some of them padding.
        dict(name="cache_prompt", kind="cache", n=8192, kv_heads=8, hd=128, type="q8_0", page=64, pad=5120, dtype="bf16",
             dropped=0.02),
        # One chat's next token: the 3B model's heads, half-precision pages.
        dict(name="attend_chat", kind="attend", n=1, heads=32, kv_heads=32, hd=80, type="f16", page=64, dtype="f32",
             longest=700, ragged=False),
        # A batch of requests of all lengths, some slots idle, small pages, grouped heads.
        dict(name="attend_batch", kind="attend", n=64, heads=32, kv_heads=8, hd=128, type="bf16", page=16, dtype="bf16",
             longest=4096, ragged=True),
        # A batch over 8-bit pages, a key head for each query head.
        dict(name="attend_q8", kind="attend", n=32, heads=22, kv_heads=22, hd=128, type="q8_0", page=128, dtype="f32",
             longest=2048, ragged=True),
        # Two very long contexts: few rows, the work lies along the cache.
        dict(name="attend_long", kind="attend", n=2, heads=32, kv_heads=8, hd=64, type="f16", page=256, dtype="f16",
             longest=131071, ragged=False),
        # A short turn after a resident prefix, fp32 rows as the products leave them.
        dict(name="prompt_turn", kind="prompt", q="19", k="449", heads=32, kv_heads=32, hd=80, dtype="f32", causal=True,
             pad=0),
        # A batch of prompts of all lengths, grouped heads.
        dict(name="prompt_packed", kind="prompt", q="1 2048 333 64 1201 17 2300 37",
             k="1 2048 333 64 1201 17 2300 37", heads=32, kv_heads=8, hd=128, dtype="bf16", causal=True, pad=0),
        # A whole document: the largest case.
        dict(name="prompt_long", kind="prompt", q="16381", k="16381", heads=32, kv_heads=32, hd=80, dtype="f16",
             causal=True, pad=0),
        # Chunks of two prompts behind what is cached of them, in the fused projection's buffer.
        dict(name="prompt_suffix", kind="prompt", q="200 96", k="8200 4000", heads=32, kv_heads=8, hd=128,
             dtype="bf16", causal=True, pad=64),
    ]


def _log(rng, low, high):
    """An integer in [low, high], even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _heads(rng):
    """(query heads, key heads, head width)"""
    kv = _log(rng, 1, 32)
    group = rng.choice([1, 1, 2, 3, 4, 8, 16] if kv <= 4 else [1, 2, 4] if kv <= 16 else [1])
    return kv * group, kv, rng.choice([8, 64, 64, 72, 80, 96, 128, 128, 256])


def draw(rng):
    kind = rng.choice(["rope", "cache", "attend", "attend", "prompt", "prompt"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    heads, kv, hd = _heads(rng)
    if kind == "rope":
        return dict(kind=kind, n=_log(rng, 1, 8192), heads=heads, hd=hd, rot=rng.choice([hd, hd, hd // 2, 2 * rng.randint(1, hd // 2)]),
                    layout=rng.choice(["half", "interleaved"]), theta=rng.choice([1e4, 5e5]),
                    scaling=rng.choice(sorted(SCALINGS)), pad=rng.choice([0, 1, 8, 512]), dtype=dtype,
                    out=rng.choice([dtype, "bf16", "f32"]), far=_log(rng, 10, 1000000))
    if kind == "cache":
        return dict(kind=kind, n=_log(rng, 1, 8192), kv_heads=kv, hd=hd, type=rng.choice(["f32", "f16", "bf16", "q8_0", "q8_0"]),
                    page=2 ** rng.randint(0, 8), pad=rng.choice([0, 1, 8, 512]), dtype=dtype,
                    dropped=rng.choice([0.0, 0.1]))
    if kind == "attend":
        n = _log(rng, 1, 96)
        longest = _log(rng, 1, max(1, min(131072, (1 << 28) // (n * kv * hd))))
        return dict(kind=kind, n=n, heads=heads, kv_heads=kv, hd=hd, type=rng.choice(["f32", "f16", "bf16", "q8_0"]),
                    page=2 ** rng.randint(3, 8), dtype=dtype, longest=longest, ragged=rng.random() < 0.6)
    sequences = _log(rng, 1, 12)
    causal = rng.random() < 0.8
    pairs = 10 ** 12 // (4 * hd * heads)  # no more of them than the largest listed case has work for
    total = _log(rng, sequences, min(8000 if dtype != "f32" else 3000, math.isqrt(pairs)))
    cuts = [rng.random() ** 2 + 1e-3 for _ in range(sequences)]
    q = [max(1, int(total * c / sum(cuts))) for c in cuts]
    before = _log(rng, 1, max(1, min(6000, pairs // total - total))) if rng.random() < 0.4 else 0  # cached keys in front
    k = [x + (rng.randint(0, before) if before else 0) for x in q]
    return dict(kind=kind, q=" ".join(map(str, q)), k=" ".join(map(str, k)), heads=heads, kv_heads=kv, hd=hd, dtype=dtype, causal=causal,
                pad=rng.choice([0, 0, 1, 8, 64]))


# ------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(g, n, heads, hd, pad, dtype):
    """[n][heads * hd + pad] head values: normal, channels of different size as keys have them, a wider buffer's padding."""
    x = torch.randn(n, heads * hd + pad, generator=g, device="cuda")
    x[:, :heads * hd] *= (0.4 * torch.randn(heads * hd, generator=g, device="cuda")).exp()
    return x.to(TYPES[dtype])


def _draw_rope(case, seed):
    g = _gen(seed)
    x = _rows(g, case["n"], case["heads"], case["hd"], case["pad"], case["dtype"])
    return x, torch.randint(0, case["far"], (case["n"],), generator=g, device="cuda", dtype=torch.int32)


def _pages(case):
    """Pages of the pool: a third more than the rows need."""
    return (case["n"] * 4 // 3 + case["page"]) // case["page"] + 1


def _draw_cache(case, seed):
    """Rows of keys and values, and the slot that each goes to (-1: padding)."""
    g = _gen(seed)
    k, v = (_rows(g, case["n"], case["kv_heads"], case["hd"], case["pad"], case["dtype"]) for _ in range(2))
    slots = torch.randperm(_pages(case) * case["page"], generator=g, device="cuda")[:case["n"]].to(torch.int32)
    gone = torch.rand(case["n"], generator=g, device="cuda") < case["dropped"]
    return k, v, slots.masked_fill(gone, -1)


def _width(case):
    return -(-case["longest"] // case["page"])


def _draw_attend(case, seed):
    """Queries, each sequence's length, the page table, and the keys and values of every slot of the pool."""
    g = _gen(seed)
    n, width, page = case["n"], _width(case), case["page"]
    q = _rows(g, n, case["heads"], case["hd"], 0, case["dtype"])
    longest = torch.full((n,), case["longest"], device="cuda")
    if case["ragged"]:  # from idle slots on
        u = torch.rand(n, generator=g, device="cuda")
        lengths = torch.where(u < 0.06, 0.0, ((u - 0.06) / 0.94 * math.log(case["longest"] + 1)).exp())
        lengths = torch.minimum(lengths, longest.float())
        lengths[0] = case["longest"]
    else:
        lengths = longest
    lengths = lengths.to(torch.int32)
    table = torch.randperm(n * width, generator=g, device="cuda").to(torch.int32).reshape(n, width)
    used = torch.arange(width, device="cuda")[None] * page < lengths[:, None]
    table = table.masked_fill(~used, -1)  # no page behind a sequence's last
    kind = "f32" if case["type"] == "q8_0" else case["type"]
    k, v = (_rows(g, n * width * page, case["kv_heads"], case["hd"], 0, kind) for _ in range(2))
    return q, lengths, table, k, v


def _lengths(case, name):
    """The sequences' numbers of queries ("q") or keys ("k")."""
    return [int(n) for n in case[name].split()]


def _draw_prompt(case, seed):
    g = _gen(seed)
    q = _rows(g, sum(_lengths(case, "q")), case["heads"], case["hd"], case["pad"], case["dtype"])
    k, v = (_rows(g, sum(_lengths(case, "k")), case["kv_heads"], case["hd"], case["pad"], case["dtype"]) for _ in range(2))
    return q, k, v


_stream = []  # the one stream that the program runs its operators on


def _empty(*shape, dtype="f32"):
    return torch.empty(*shape, dtype=TYPES.get(dtype, dtype), device="cuda")


def prepare(case, seed):
    kind, s = case["kind"], dict(case=case)
    if kind == "rope":
        x, positions = _draw_rope(case, seed)
        s.update(x=x, positions=positions)
    elif kind == "cache":
        k, v, slots = _draw_cache(case, seed)
        s.update(k=k, v=v, slots=slots)
    elif kind == "attend":
        q, lengths, table, k, v = _draw_attend(case, seed)
        s.update(q=q, lengths=lengths, table=table, k=k, v=v)
    else:
        q, k, v = _draw_prompt(case, seed)
        offsets = [torch.tensor([0] + _lengths(case, x), device="cuda").cumsum(0).to(torch.int32) for x in "qk"]
        s.update(q=q, k=k, v=v, q_offsets=offsets[0], k_offsets=offsets[1])
    if own:
        _prepare_own(case, s)
    elif kind == "rope":
        s.update(frequencies=_frequencies(case).cuda())
    elif kind == "cache":
        slots, heads, hd = _pages(case) * case["page"], case["kv_heads"], case["hd"]
        s.update(pool=[_pool(torch.zeros(slots, heads, hd, device="cuda"), case["type"]) for _ in "kv"])
    elif kind == "attend":
        shape = (-1, case["kv_heads"], case["hd"])
        s.update(pool=[_pool(s.pop(x).reshape(shape), case["type"]) for x in "kv"])
    torch.cuda.synchronize()
    return s


def _prepare_own(case, s):
    """The handles, their filled caches and the buffers that a program keeps."""
    from tinyoai_amd import hip
    kind = case["kind"]
    if not _stream:
        _stream.append(torch.cuda.Stream())
    stream = _stream[0].cuda_stream
    s.update(hip=hip, stream=stream)
    if kind == "rope":
        scaling, factor, context, low, high = SCALINGS[case["scaling"]]
        s.update(rope=hip.Rope(case["hd"], case["rot"], case["layout"], case["theta"], scaling, factor, context, low, high),
                 out=_empty(case["n"], case["heads"] * case["hd"], dtype=case["out"]))
    elif kind == "cache":
        width = case["kv_heads"] * case["hd"]
        s.update(pages=hip.KVPages(CODES[case["type"]], 1, case["kv_heads"], case["hd"], case["page"], _pages(case)),
                 ko=_empty(case["n"], width, dtype=case["dtype"]), vo=_empty(case["n"], width, dtype=case["dtype"]))
    elif kind == "attend":
        pages = hip.KVPages(CODES[case["type"]], 1, case["kv_heads"], case["hd"], case["page"], case["n"] * _width(case))
        k, v = s.pop("k"), s.pop("v")
        slots = torch.arange(len(k), dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        pages.write(0, _code(k), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), slots.data_ptr(), len(k), stream)
        torch.cuda.synchronize()
        s.update(pages=pages, out=_empty(case["n"], case["heads"] * case["hd"], dtype=case["dtype"]))
    else:
        s.update(out=_empty(len(s["q"]), case["heads"] * case["hd"], dtype=case["dtype"]))


def _code(x):
    return next(CODES[name] for name, t in TYPES.items() if t == x.dtype)


# ------------------------------------------------------------ one pass
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    case, stream = s["case"], s["stream"]
    kind, hd = case["kind"], case["hd"]
    if kind == "rope":
        x, out = s["x"], s["out"]
        s["rope"].rotate(_code(x), x.data_ptr(), x.stride(0), case["n"], case["heads"], s["positions"].data_ptr(),
                         _code(out), out.data_ptr(), out.stride(0), stream)
        return out
    if kind == "cache":
        k, v, ko, vo, slots = s["k"], s["v"], s["ko"], s["vo"], s["slots"].data_ptr()
        s["pages"].write(0, _code(k), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), slots, case["n"], stream)
        s["pages"].read(0, _code(ko), ko.data_ptr(), ko.stride(0), vo.data_ptr(), vo.stride(0), slots, case["n"], stream)
        return ko, vo
    q, out = s["q"], s["out"]
    if kind == "attend":
        s["pages"].attend(0, _code(q), q.data_ptr(), q.stride(0), case["heads"], hd ** -0.5, s["table"].data_ptr(), _width(case),
                          s["lengths"].data_ptr(), case["n"], out.data_ptr(), out.stride(0), stream)
        return out
    k, v = s["k"], s["v"]
    s["hip"].attention(_code(q), q.data_ptr(), q.stride(0), case["heads"], k.data_ptr(), k.stride(0), v.data_ptr(),
                       v.stride(0), case["kv_heads"], hd, hd ** -0.5, case["causal"], s["q_offsets"].data_ptr(),
                       s["k_offsets"].data_ptr(), len(s["q_offsets"]) - 1, len(q), len(k), out.data_ptr(), out.stride(0), stream)
    return out


def _frequencies(case):
    """The angle of each pair for a step of one position, in 64 bits."""
    kind, factor, context, low, high = SCALINGS[case["scaling"]]
    rot, theta = case["rot"], case["theta"]
    f = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if kind == "linear":
        return f / factor
    if kind == "bands":  # turns in the training's context: at least `high` keep, at most `low` are scaled
        keep = ((context * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        return f * keep + f / factor * (1 - keep)
    if kind == "yarn":  # by the pair's index, between those that turn `high` and `low` times
        at = [rot * math.log(context / (2 * math.pi * t)) / (2 * math.log(theta)) for t in (high, low)]
        first, last = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        ramp = ((torch.arange(rot // 2, dtype=torch.float64) - first) / max(last - first, 0.001)).clamp(0, 1)
        return f * (1 - ramp) + f / factor * ramp
    return f


def _magnitude(case):
    return 0.1 * math.log(SCALINGS[case["scaling"]][1]) + 1 if case["scaling"] == "yarn" else 1.0


def _pool(x, kind):
    """Rows [slots][heads][hd] as a cache holds them: (values, None), or 8-bit (codes, scales) of blocks of 32."""
    if kind != "q8_0":
        return x.to(TYPES[kind]), None
    hd = x.shape[-1]
    b = torch.nn.functional.pad(x.float(), (0, -hd % 32)).unflatten(-1, (-1, 32))
    d = (b.abs().amax(-1, keepdim=True) / 127).clamp_max(65504).half()
    codes = torch.where(d > 0, b / d.float(), 0.0).round().clamp(-127, 127).to(torch.int8)
    return codes.flatten(-2)[..., :hd].contiguous(), d[..., 0]


def _values(pool, index):
    """The fp32 values of a pool's slots [...]: [..., heads, hd]."""
    codes, d = pool[0][index], pool[1]
    if d is None:
        return codes.float()
    return codes.float() * d[index].float().repeat_interleave(32, -1)[..., :codes.shape[-1]]


def _run_plain(s):
    case = s["case"]
    kind, hd = case["kind"], case["hd"]
    if kind == "rope":
        return _rope_plain(s["x"], s["positions"], s["frequencies"], case)
    if kind == "cache":
        slots = s["slots"].long()
        ok = slots >= 0
        outs = []
        for x, pool in zip((s["k"], s["v"]), s["pool"]):
            rows = x[:, :case["kv_heads"] * hd].unflatten(1, (-1, hd))
            for old, new in zip(pool, _pool(rows, case["type"])):
                if old is not None:
                    old[slots[ok]] = new[ok]
            read = _values(pool, slots.clamp_min(0))
            outs.append(torch.where(ok[:, None, None], read, 0.0).flatten(1).to(TYPES[case["dtype"]]))
        return tuple(outs)
    if kind == "attend":
        return _attend_plain(s, case)
    q, k, v = (s[x][:, :h * hd].float().unflatten(1, (h, hd)) for x, h in
               (("q", case["heads"]), ("k", case["kv_heads"]), ("v", case["kv_heads"])))
    out = []
    for qs, ks, vs in zip(q.split(_lengths(case, "q")), k.split(_lengths(case, "k")), v.split(_lengths(case, "k"))):
        kt, vt = ks.permute(1, 2, 0).contiguous(), vs.transpose(0, 1).contiguous()  # [kv][hd][keys], [kv][keys][hd]
        shift = len(ks) - len(qs)
        for at in range(0, len(qs), 1024):  # as many scores as memory takes
            part = qs[at:at + 1024]
            rows = part.unflatten(1, (case["kv_heads"], -1)).permute(1, 2, 0, 3).flatten(1, 2).contiguous()
            score = torch.bmm(rows, kt).unflatten(1, (-1, len(part))) * hd ** -0.5  # [kv][group][query][key]
            if case["causal"]:
                last = torch.arange(at, at + len(part), device="cuda") + shift
                score.masked_fill_(torch.arange(len(ks), device="cuda") > last[:, None], -math.inf)
            most = score.amax(-1, keepdim=True)
            p = (score - torch.where(most > -math.inf, most, 0.0)).exp_()
            total = p.sum(-1, keepdim=True)
            o = torch.bmm(p.flatten(1, 2), vt).unflatten(1, (-1, len(part))) / torch.where(total > 0, total, 1.0)
            out.append(o.permute(2, 0, 1, 3).flatten(1))
    return torch.cat(out).to(TYPES[case["dtype"]])


def _rope_plain(x, positions, frequencies, case):
    rot, hd = case["rot"], case["hd"]
    angle = positions.double()[:, None, None] * frequencies  # [n][1][rot / 2]
    c, s = (angle.cos() * _magnitude(case)).float(), (angle.sin() * _magnitude(case)).float()
    x = x[:, :case["heads"] * hd].float().unflatten(1, (-1, hd))
    r = x[..., :rot]
    a, b = (r[..., :rot // 2], r[..., rot // 2:]) if case["layout"] == "half" else (r[..., ::2], r[..., 1::2])
    a, b = a * c - b * s, b * c + a * s
    r = torch.cat([a, b], -1) if case["layout"] == "half" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([r, x[..., rot:]], -1).flatten(1).to(TYPES[case["out"]])


def _attend_plain(s, case):
    n, page, kv, hd = case["n"], case["page"], case["kv_heads"], case["hd"]
    slots = (s["table"].long().clamp_min(0)[..., None] * page + torch.arange(page, device="cuda")).flatten(1)
    seen = torch.arange(slots.shape[1], device="cuda") < s["lengths"][:, None]
    q = s["q"].float().reshape(n * kv, -1, hd)
    k, v = (_values(pool, slots) for pool in s["pool"])  # [n][positions][kv][hd]
    score = torch.bmm(q, k.permute(0, 2, 3, 1).reshape(n * kv, hd, -1).contiguous()).unflatten(0, (n, kv)) * hd ** -0.5
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    most = score.amax(-1, keepdim=True)
    p = (score - torch.where(most > -math.inf, most, 0.0)).exp()
    total = p.sum(-1, keepdim=True)
    o = torch.bmm(p.flatten(0, 1), v.transpose(1, 2).reshape(n * kv, -1, hd).contiguous()).unflatten(0, (n, kv))
    return (o / torch.where(total > 0, total, 1.0)).reshape(n, -1).to(TYPES[case["dtype"]])


# ------------------------------------------------------------ what a pass costs
def work(case):
    kind, hd = case["kind"], case["hd"]
    size = {name: t.itemsize for name, t in TYPES.items()}
    if kind == "rope":
        values = case["n"] * case["heads"] * hd
        return {"bytes": values * (size[case["dtype"]] + size[case["out"]]) + 4 * case["n"],
                "flops": 3 * case["n"] * case["heads"] * case["rot"]}
    kv = case["kv_heads"]
    held = hd + 2 * -(-hd // 32) if case.get("type") == "q8_0" else hd * size.get(case.get("type"), 0)  # a head's row
    if kind == "cache":  # the rows in, what the pages hold out and in again, the values that it stands for
        rows = 2 * case["n"] * kv
        return {"bytes": int((1 - case["dropped"]) * rows * 2 * (hd * size[case["dtype"]] + held)) + 8 * case["n"],
                "flops": 4 * rows * hd}
    if kind == "attend":  # a ragged batch: the mean of its lengths
        n, longest = case["n"], case["longest"]
        total = n * longest if not case["ragged"] else longest + (n - 1) * 0.94 * longest / math.log(longest + 1)
        return {"bytes": int(total * 2 * kv * held) + 2 * n * case["heads"] * hd * size[case["dtype"]] + 4 * n,
                "flops": int(total * case["heads"] * 4 * hd)}
    pairs = 0
    for q, k in zip(_lengths(case, "q"), _lengths(case, "k")):
        pairs += q * k - (q * (q - 1) // 2 if case["causal"] else 0)
    rows = 2 * sum(_lengths(case, "q")) * case["heads"] + 2 * sum(_lengths(case, "k")) * kv
    return {"bytes": rows * hd * size[case["dtype"]] + 8 * len(_lengths(case, "q")), "flops": 4 * hd * case["heads"] * pairs}


# ------------------------------------------------------------ 64 bits
def _blocks64(x, kind):
    """What a cache of this type stands for, of rows [..., hd] in 64 bits. 8-bit: scale and quotient are fp32 by definition."""
    if kind != "q8_0":
        return x.to(TYPES[kind]).double()
    parts = []
    for b in x.double().split(32, -1):
        d = (b.abs().max(-1, keepdim=True).values / 127).float().clamp_max(65504).half().double()
        q = torch.div(b, torch.where(d == 0, 1.0, d)).float().double()
        parts.append(torch.where(d == 0, 0.0, torch.round(q).clamp(-127, 127) * d))
    return torch.cat(parts, -1)


def _softmax64(score, v):
    """softmax(score) v over rows that may see nothing."""
    w = torch.softmax(score, -1)
    return torch.matmul(torch.where(torch.isnan(w), 0.0, w), v)


def exact(case, seed):
    kind, hd = case["kind"], case["hd"]
    if kind == "rope":
        return _rope64(case, seed)
    kv = case["kv_heads"]
    if kind == "cache":
        k, v, slots = _draw_cache(case, seed)
        ok = (slots >= 0).double()[:, None, None]
        return tuple((_blocks64(x[:, :kv * hd].reshape(-1, kv, hd), case["type"]) * ok).reshape(len(x), -1) for x in (k, v))
    group = case["heads"] // kv
    if kind == "attend":
        q, lengths, table, k, v = _draw_attend(case, seed)
        out = torch.zeros(case["n"], case["heads"], hd, dtype=torch.float64, device="cuda")
        for i, length in enumerate(lengths.tolist()):
            if not length:
                continue
            pages = table[i, :-(-length // case["page"])].long()
            ks, vs = (_blocks64(x.reshape(-1, case["page"], kv, hd)[pages].flatten(0, 1)[:length], case["type"]) for x in (k, v))
            for h in range(kv):
                part = q[i].reshape(-1, hd)[h * group:(h + 1) * group].double()
                out[i, h * group:(h + 1) * group] = _softmax64(part @ ks[:, h].T.contiguous() / math.sqrt(hd), vs[:, h].contiguous())
        return out.reshape(case["n"], -1)
    q, k, v = _draw_prompt(case, seed)
    out = torch.zeros(len(q), case["heads"] * hd, dtype=torch.float64, device="cuda")
    at = [0, 0]
    for nq, nk in zip(_lengths(case, "q"), _lengths(case, "k")):
        for h in range(case["heads"]):
            cols, kcols = slice(h * hd, h * hd + hd), slice(h // group * hd, h // group * hd + hd)
            ks, vs = (x[at[1]:at[1] + nk, kcols].double() for x in (k, v))
            for r in range(0, nq, 4096):
                qs = q[at[0] + r:at[0] + min(nq, r + 4096), cols].double()
                score = qs @ ks.T.contiguous() / math.sqrt(hd)
                if case["causal"]:
                    hidden = torch.ones(len(qs), nk, dtype=torch.bool, device="cuda").triu(r + nk - nq + 1)
                    score = score.masked_fill(hidden, -math.inf)
                out[at[0] + r:at[0] + r + len(qs), cols] = _softmax64(score, vs.contiguous())
        at = [at[0] + nq, at[1] + nk]
    return out


def _rope64(case, seed):
    x, positions = _draw_rope(case, seed)
    rot, hd, heads = case["rot"], case["hd"], case["heads"]
    kind, factor, context, low, high = SCALINGS[case["scaling"]]
    out = x[:, :heads * hd].double().reshape(-1, heads, hd).clone()
    first = second = 0
    if kind == "yarn":
        turns = lambda t: rot / 2 * math.log(context / (t * math.tau), case["theta"])  # noqa: E731
        first, second = max(0, math.floor(turns(high))), min(rot - 1, math.ceil(turns(low)))
    for i in range(rot // 2):
        f = math.exp(-2 * i / rot * math.log(case["theta"]))
        if kind == "linear":
            f /= factor
        elif kind == "bands":
            wave = math.tau / f
            if wave > context / low:
                f /= factor
            elif wave > context / high:
                mix = (context / wave - low) / (high - low)
                f = mix * f + (1 - mix) * f / factor
        elif kind == "yarn":
            mix = min(1.0, max(0.0, (i - first) / max(0.001, second - first)))
            f = f * ((1 - mix) + mix / factor)
        turn = torch.polar(torch.full_like(positions.double(), _magnitude(case)), positions.double() * f)[:, None]
        a, b = (i, i + rot // 2) if case["layout"] == "half" else (2 * i, 2 * i + 1)
        z = torch.complex(out[..., a], out[..., b]) * turn
        out[..., a], out[..., b] = z.real, z.imag
    return out.reshape(len(x), -1)
