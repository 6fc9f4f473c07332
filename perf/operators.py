"""Cases of the decoder-step operators: RMS norm with the residual's addition (and an 8-bit output), rotary positions with the
write into a paged key-value cache, attention of one new token over that cache, and log-probabilities of given tokens.

``run`` computes them in a plain form (elementary torch operations in fp32, angles in fp64) or, where ``own`` is true, through
``docc_b200.ops``. ``exact`` restates each from its definition in fp64."""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
_E4M3_MAX = 448.0


# ---- cases --------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the norm in front of a layer while eight sequences decode, at the encoder block's width
        dict(name="rms step", op="rms", dtype="bf16", rows=8, cols=1024, residual=True, quant="none"),
        # the norm over a long prompt, handing the next product 8-bit activations with a scale per 128 columns
        dict(name="rms prompt 8-bit", op="rms", dtype="bf16", rows=8192, cols=4096, residual=True, quant="group"),
        # an odd width and an odd number of rows: no row but the first starts on a 16-byte boundary; one scale per row
        dict(name="rms odd 8-bit", op="rms", dtype="fp16", rows=1021, cols=5003, residual=False, quant="row"),
        # sixteen sequences decode: one token each is rotated and goes into the cache
        dict(name="rope step", op="rope", dtype="bf16", tokens=16, heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False,
             scaling="none", page=16, start=5000),
        # a chunk of a long context: interleaved pairs, half of each head, frequencies stretched, positions far out
        dict(name="rope prompt", op="rope", dtype="fp16", tokens=8192, heads=32, kv_heads=8, dim=128, rotary=64, interleaved=True,
             scaling="yarn", page=64, start=100000),
        # one user, a short conversation: latency
        dict(name="attention one", op="attention", dtype="bf16", batch=1, heads=32, kv_heads=8, dim=128, page=16, longest=1025,
             ragged=False, softcap=0.0, window=0),
        # a full server: sixty-four sequences of very different lengths
        dict(name="attention batch", op="attention", dtype="bf16", batch=64, heads=32, kv_heads=8, dim=128, page=16, longest=8192,
             ragged=True, softcap=0.0, window=0),
        # one very long context over two shared heads, capped scores: all parallelism comes from the cache's length
        dict(name="attention long", op="attention", dtype="fp16", batch=1, heads=16, kv_heads=2, dim=128, page=64, longest=131079,
             ragged=False, softcap=30.0, window=0),
        # fp32, every head with keys of its own, at the encoder block's head count and size
        dict(name="attention fp32", op="attention", dtype="fp32", batch=16, heads=16, kv_heads=16, dim=64, page=32, longest=2048,
             ragged=True, softcap=0.0, window=0),
        # four sequences have produced their logits: the chosen tokens' log-probabilities and five alternatives
        dict(name="logp step", op="logp", dtype="bf16", rows=4, vocab=32768, top=5),
        # a large batch over a large vocabulary with twenty alternatives
        dict(name="logp batch", op="logp", dtype="bf16", rows=256, vocab=128000, top=20),
        # scoring a prompt: every position's token, no alternatives, odd vocabulary in fp32
        dict(name="logp prompt", op="logp", dtype="fp32", rows=4096, vocab=50021, top=0),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread evenly over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rms", "rope", "attention", "logp"])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    if op == "rms":
        cols = _spread(rng, 64, 16384)
        if rng.random() < 0.6:
            cols = max(64, cols // 64 * 64)
        rows = _spread(rng, 1, max(1, min(16384, (1 << 24) // cols)))
        return dict(op=op, dtype=dtype, rows=rows, cols=cols, residual=rng.random() < 0.7, quant=rng.choice(["none", "row", "group"]))
    if op == "rope":
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
        dim = rng.choice([64, 80, 96, 128, 256])
        tokens = _spread(rng, 1, max(1, min(8192, (1 << 24) // (heads * dim))))
        return dict(op=op, dtype=dtype, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rotary=rng.choice([dim, dim, dim // 2]),
                    interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "ntk", "yarn"]), page=rng.choice([1, 16, 24, 64]),
                    start=_spread(rng, 1, 1000000))
    if op == "attention":
        kv_heads = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 3, 4, 7, 8, 16])
        dim = rng.choice([64, 80, 96, 128, 256])
        batch = _spread(rng, 1, 64)
        room = (1 << 27) // (batch * kv_heads * dim)
        longest = _spread(rng, 1, max(1, min(131072, room)))
        window = _spread(rng, 1, longest) if rng.random() < 0.25 else 0
        return dict(op=op, dtype=dtype, batch=batch, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=rng.choice([1, 8, 16, 24, 64, 128]),
                    longest=longest, ragged=rng.random() < 0.7, softcap=rng.choice([0.0, 0.0, 20.0, 50.0]), window=window)
    vocab = _spread(rng, 500, 200000)
    rows = _spread(rng, 1, max(1, min(4096, (1 << 26) // vocab)))
    return dict(op=op, dtype=dtype, rows=rows, vocab=vocab, top=rng.choice([0, 1, 5, 20, 32]))


def _lengths(case):
    """The cached lengths of the batch: a property of the case, so that its work is known. Ragged batches hold an empty sequence and
    one of a single token, as a server's do between two requests."""
    rng = random.Random(case["batch"] * 1000003 + case["longest"])
    if not case["ragged"]:
        return [case["longest"]] * case["batch"]
    lengths = [_spread(rng, 1, case["longest"]) if i % 2 else rng.randint(0, case["longest"]) for i in range(case["batch"])]
    lengths[0] = case["longest"]
    if case["batch"] > 2:
        lengths[1], lengths[2] = 0, 1
    rng.shuffle(lengths)
    return lengths


def _seen(case):
    """How many cached tokens each sequence's new token attends to."""
    return [min(n, case["window"]) if case["window"] else n for n in _lengths(case)]


def work(case):
    size = _SIZE[case["dtype"]]
    if case["op"] == "rms":
        n = case["rows"] * case["cols"]
        out = n * size if case["quant"] == "none" else n + 4 * case["rows"] * (1 if case["quant"] == "row" else -(-case["cols"] // 128))
        return {"bytes": n * size * (3 if case["residual"] else 1) + out + 4 * case["cols"], "flops": 6 * n}
    if case["op"] == "rope":
        n = case["tokens"] * (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * n * size + 16 * case["tokens"] + 4 * case["rotary"],
                "flops": 3 * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["rotary"]}
    if case["op"] == "attention":
        seen = sum(_seen(case))
        pages = sum(-(-n // case["page"]) for n in _seen(case))
        return {"bytes": 2 * seen * case["kv_heads"] * case["dim"] * size + 2 * case["batch"] * case["heads"] * case["dim"] * size
                + 4 * case["batch"] * (case["heads"] + 1) + 4 * pages,
                "flops": 4 * seen * case["heads"] * case["dim"]}
    return {"bytes": case["rows"] * (case["vocab"] * size + 16 + 12 * case["top"]), "flops": 5 * case["rows"] * case["vocab"]}


# ---- inputs -------------------------------------------------------------------------------------------------------------------
def _frequencies(case):
    """Radians per position of each pair (fp64) and the factor of cosine and sine."""
    rotary, base, factor, original = case["rotary"], 10000.0, 8.0, 4096
    i = torch.arange(rotary // 2, dtype=torch.float64)
    freq = base ** (-2.0 * i / rotary)
    if case["scaling"] == "linear":
        return freq / factor, 1.0
    if case["scaling"] == "ntk":
        return (base * factor ** (rotary / (rotary - 2.0))) ** (-2.0 * i / rotary), 1.0
    if case["scaling"] == "yarn":
        at = lambda turns: rotary * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rotary - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return freq / factor * ramp + freq * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return freq, 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    normal = lambda *shape, t=dtype: torch.randn(*shape, generator=g, device="cuda").to(t)  # noqa: E731
    s = {"case": case}
    if case["op"] == "rms":
        s["x"] = normal(case["rows"], case["cols"])
        s["residual"] = 3 * normal(case["rows"], case["cols"]) if case["residual"] else None
        s["gamma"] = 1 + 0.2 * normal(case["cols"], t=torch.float32)
    elif case["op"] == "rope":
        t, h, kv, d, page = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "page"))
        qkv = normal(t, (h + 2 * kv) * d)  # the packed projection output that the three are views of
        s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, d)) for x in qkv.split([h * d, kv * d, kv * d], dim=1))
        s["positions"] = case["start"] + torch.arange(t, device="cuda")
        pages = t // page + 3
        s["k_cache"], s["v_cache"] = normal(pages, kv, page, d), normal(pages, kv, page, d)
        s["slots"] = torch.randperm(pages * page, generator=g, device="cuda")[:t]
        freq, s["mscale"] = _frequencies(case)
        s["inv_freq"] = freq.cuda()
    elif case["op"] == "attention":
        lengths = _lengths(case)
        page, kv, d = case["page"], case["kv_heads"], case["dim"]
        need = [-(-n // page) for n in lengths]
        order = torch.randperm(sum(need) + 2, generator=g, device="cuda").int()
        most = max(1, max(need))
        start = [sum(need[:b]) for b in range(len(need))]
        at = torch.tensor([list(range(i, i + n)) + [sum(need)] * (most - n) for i, n in zip(start, need)], device="cuda")
        s["page_table"] = order[at].contiguous()
        s["k_cache"], s["v_cache"] = normal(sum(need) + 2, kv, page, d), normal(sum(need) + 2, kv, page, d)
        s["q"] = 2 * normal(case["batch"], case["heads"], d)
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    else:
        s["logits"] = 3 * normal(case["rows"], case["vocab"])
        s["ids"] = torch.randint(case["vocab"], (case["rows"],), generator=g, device="cuda")
    return s


# ---- the plain form -------------------------------------------------------------------------------------------------------------
def _plain_rms(s, case):
    x = s["x"].float()
    if s["residual"] is not None:
        x = x + s["residual"].float()
    y = x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + 1e-6) * s["gamma"]
    out = {"sum": x.to(s["x"].dtype)} if s["residual"] is not None else {}
    if case["quant"] == "none":
        return out | {"y": y.to(s["x"].dtype)}
    rows, cols = y.shape
    group = cols if case["quant"] == "row" else 128
    groups = -(-cols // group)
    y = torch.nn.functional.pad(y, (0, groups * group - cols)).view(rows, groups, group)
    scale = y.abs().amax(dim=2, keepdim=True) / _E4M3_MAX
    q = torch.where(scale > 0, y / scale, y).view(rows, groups * group)[:, :cols]
    return out | {"q": q.to(torch.float8_e4m3fn), "scale": scale.view(rows, groups)}


def _plain_rotate(x, cos, sin, case):
    turn, rest = x[..., : case["rotary"]], x[..., case["rotary"]:]
    if case["interleaved"]:
        u, v = turn[..., 0::2].float(), turn[..., 1::2].float()
        turn = torch.stack([u * cos - v * sin, v * cos + u * sin], dim=-1).flatten(-2)
    else:
        u, v = (t.float() for t in turn.chunk(2, dim=-1))
        turn = torch.cat([u * cos - v * sin, v * cos + u * sin], dim=-1)
    return torch.cat([turn.to(x.dtype), rest], dim=-1)


def _plain_rope(s, case):
    angle = s["positions"].double()[:, None] * s["inv_freq"]
    cos, sin = ((s["mscale"] * f(angle)).float()[:, None] for f in (torch.cos, torch.sin))
    place, within = s["slots"] // case["page"], s["slots"] % case["page"]
    s["k_cache"][place, :, within] = _plain_rotate(s["k"], cos, sin, case)
    s["v_cache"][place, :, within] = s["v"]
    return {"q": _plain_rotate(s["q"], cos, sin, case), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attention(s, case):
    batch, heads, kv, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    table = s["page_table"].long()
    k, v = (c[table].transpose(1, 2).reshape(batch, kv, -1, d).float() for c in (s["k_cache"], s["v_cache"]))
    q = s["q"].float().view(batch, kv, heads // kv, d)
    score = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    if case["softcap"]:
        score = case["softcap"] * torch.tanh(score / case["softcap"])
    at, length = torch.arange(k.shape[2], device="cuda"), s["lengths"].long()[:, None]
    seen = at < length
    if case["window"]:
        seen = seen & (at >= length - case["window"])
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(dim=3, keepdim=True).clamp(min=-1e30)
    p = torch.exp(score - top)
    total = p.sum(dim=3, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1)
    return {"out": out.view(batch, heads, d).to(s["q"].dtype), "lse": (top + torch.log(total)).view(batch, heads)}


def _plain_logp(s, case):
    x = s["logits"].float()
    top = x.amax(dim=1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(dim=1, keepdim=True)
    logp = x - (top + torch.log(total))
    out = {"logp": logp.gather(1, s["ids"][:, None])[:, 0], "entropy": -(e / total * logp).sum(dim=1)}
    if case["top"]:
        order = torch.sort(s["logits"], dim=1, descending=True, stable=True).indices[:, : case["top"]]
        out |= {"top_ids": order, "top_logp": logp.gather(1, order)}
    return out


# ---- the framework's form -------------------------------------------------------------------------------------------------------
_ops = None


def _framework():
    """The framework's operators, with their launches on torch's stream from the first call on."""
    global _ops
    if _ops is None:
        from docc_b200 import ops

        ops.init(torch.cuda.current_device())
        ops.set_stream(torch.cuda.current_stream().cuda_stream)
        _ops = ops
    return _ops


def _own(s, case):
    ops = _framework()
    if case["op"] == "rms":
        if case["quant"] == "none":
            r = ops.rmsnorm(s["x"], s["gamma"], residual=s["residual"], eps=1e-6)
            return {"sum": r[1], "y": r[0]} if case["residual"] else {"y": r}
        r = ops.rmsnorm_quant(s["x"], s["gamma"], residual=s["residual"], eps=1e-6, group=0 if case["quant"] == "row" else 128)
        return ({"sum": r[2]} if case["residual"] else {}) | {"q": r[0], "scale": r[1]}
    if case["op"] == "rope":
        q = ops.rope_append(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], s["k_cache"], s["v_cache"], s["slots"],
                            interleaved=case["interleaved"], mscale=s["mscale"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if case["op"] == "attention":
        out, lse = ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["lengths"], softcap=case["softcap"],
                                       window=case["window"], return_lse=True)
        return {"out": out, "lse": lse}
    logp, entropy, ids, top = ops.token_logprobs(s["logits"], s["ids"], k=case["top"])
    return {"logp": logp, "entropy": entropy} | ({"top_ids": ids, "top_logp": top} if case["top"] else {})


def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    return {"rms": _plain_rms, "rope": _plain_rope, "attention": _plain_attention, "logp": _plain_logp}[case["op"]](s, case)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------------
def _exact_rms(s, case):
    total = s["x"].double() + (s["residual"].double() if case["residual"] else 0.0)
    norm = total / (total.square().sum(dim=1, keepdim=True) / case["cols"] + 1e-6).sqrt()
    y = norm * s["gamma"].double()
    out = {"sum": total} if case["residual"] else {}
    if case["quant"] == "none":
        return out | {"y": y}
    width = case["cols"] if case["quant"] == "row" else 128
    parts = y.split(width, dim=1)
    scale = torch.stack([p.abs().max(dim=1).values / _E4M3_MAX for p in parts], dim=1)
    return out | {"q": torch.cat([p / scale[:, i, None] for i, p in enumerate(parts)], dim=1), "scale": scale}


def _exact_rope(s, case):
    half = case["rotary"] // 2
    i = torch.arange(half, device="cuda")
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
    turn = torch.polar(torch.full((case["tokens"], half), float(s["mscale"]), dtype=torch.float64, device="cuda"),
                       s["positions"].double()[:, None] * s["inv_freq"][None])

    def rotated(x):
        y = x.double().clone()
        z = torch.complex(y[..., first], y[..., second]) * turn[:, None, :]
        y[..., first], y[..., second] = z.real, z.imag
        return y

    out = {"q": rotated(s["q"])}
    page, within = torch.div(s["slots"], case["page"], rounding_mode="floor"), s["slots"].remainder(case["page"])
    for name, new in (("k_cache", rotated(s["k"])), ("v_cache", s["v"].double())):
        cache = s[name].double().permute(0, 2, 1, 3).contiguous()
        cache[page, within] = new
        out[name] = cache.permute(0, 2, 1, 3)
    return out


def _exact_attention(s, case):
    group = case["heads"] // case["kv_heads"]
    outs, lses = [], []
    for b, n in enumerate(_lengths(case)):
        low = max(0, n - case["window"]) if case["window"] else 0
        if n == 0:
            outs.append(torch.zeros(case["heads"], case["dim"], dtype=torch.float64, device="cuda"))
            lses.append(torch.full((case["heads"],), -math.inf, dtype=torch.float64, device="cuda"))
            continue
        j = torch.arange(low, n, device="cuda")
        pages = s["page_table"][b].long()[j // case["page"]]
        k, v = (s[c][pages, :, j % case["page"]].double().repeat_interleave(group, dim=1) for c in ("k_cache", "v_cache"))
        z = torch.einsum("hd,jhd->hj", s["q"][b].double(), k) / case["dim"] ** 0.5
        if case["softcap"]:
            z = torch.tanh(z / case["softcap"]) * case["softcap"]
        lse = torch.logsumexp(z, dim=1)
        outs.append(torch.einsum("hj,jhd->hd", torch.exp(z - lse[:, None]), v))
        lses.append(lse)
    return {"out": torch.stack(outs), "lse": torch.stack(lses)}


def _exact_logp(s, case):
    parts = []
    for x, ids in zip(s["logits"].split(512), s["ids"].split(512)):
        z = x.double()
        logp = z - torch.logsumexp(z, dim=1, keepdim=True)
        part = {"logp": logp[torch.arange(len(ids), device="cuda"), ids], "entropy": -torch.sum(torch.exp(logp) * logp, dim=1)}
        if case["top"]:
            values, order = torch.sort(logp, dim=1, descending=True, stable=True)
            part |= {"top_ids": order[:, : case["top"]], "top_logp": values[:, : case["top"]]}
        parts.append(part)
    return {name: torch.cat([p[name] for p in parts]) for name in parts[0]}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rms": _exact_rms, "rope": _exact_rope, "attention": _exact_attention, "logp": _exact_logp}[case["op"]](s, case)
