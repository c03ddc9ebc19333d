"""The operators of a decode step over a paged key-value cache: appending (norm of each head, position rotation, append), attention of one
new token per sequence, and sampling from the logits.

A program holds the cache's pages, its page table and the positions on the GPU, as torch tensors here that the backend's tensors wrap;
``run`` makes its calls, or computes the same from elementary operations where ``own`` is false.  A case is a dict of plain values;
sequence lengths follow from it alone, so that a case's work is known without its inputs.
"""
import math

import torch

own = False

_TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_DEV = "cuda"


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def _append(name, tokens, seqs, past, heads, kv_heads, dim, page, dtype, norm, fused):
    return {"name": name, "kind": "append", "tokens": tokens, "seqs": seqs, "past": past, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "dtype": dtype, "norm": norm, "fused": fused}


def _attention(name, batch, longest, ragged, heads, kv_heads, dim, page, dtype, softcap=0.0, window=0, slopes=False):
    return {"name": name, "kind": "attention", "batch": batch, "longest": longest, "ragged": ragged, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "dtype": dtype, "softcap": softcap, "window": window, "slopes": slopes}


def _sample(name, rows, vocab, dtype, top_k, top_p, min_p, spread):
    return {"name": name, "kind": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "top_k": top_k, "top_p": top_p, "min_p": min_p,
            "spread": spread}


def listed():
    return [
        # one new token of one sequence in a 0.6B-shaped model with normed heads: launch and host path count
        _append("append_one", 1, 1, 700, 16, 8, 128, 16, "f16", True, False),
        # one new token for each of sixty-four sequences, read from the rows of one fused q/k/v product
        _append("append_step_64", 64, 64, 1500, 32, 8, 128, 16, "bf16", True, True),
        # prompts of odd lengths, all their tokens at once, without norms
        _append("append_prompts", 8001, 5, 0, 32, 8, 128, 64, "bf16", False, False),
        # the smallest attention of a conversation that has just begun
        _attention("attention_short", 1, 45, False, 16, 8, 128, 16, "f16"),
        # eight sequences of about the same length, grouped query heads
        _attention("attention_batch_8", 8, 4000, False, 32, 8, 128, 16, "f16"),
        # a serving batch whose sequences are at very different places
        _attention("attention_ragged_64", 64, 8000, True, 32, 8, 128, 16, "bf16"),
        # one long document, few key-value heads
        _attention("attention_long", 1, 100_003, False, 16, 2, 128, 64, "bf16"),
        # capped scores over a sliding window, wide heads
        _attention("attention_capped", 16, 6000, True, 8, 4, 256, 32, "f16", softcap=50.0, window=4096),
        # f32 storage, the type torchlette's own frontend computes in by default, with a bias that falls with distance
        _attention("attention_f32", 4, 1500, True, 8, 8, 64, 16, "f32", slopes=True),
        # one token from a small vocabulary with the usual filters
        _sample("sample_one", 1, 32_000, "f32", 50, 0.9, 0.0, 2.5),
        # a batch over a large vocabulary, top-k and top-p
        _sample("sample_filtered_64", 64, 151_936, "f32", 50, 0.95, 0.0, 2.5),
        # f16 logits (many ties) with a nucleus alone, and flat enough that it is wide
        _sample("sample_nucleus_16", 16, 151_936, "f16", 0, 0.9, 0.02, 1.5),
    ]


def _between(rng, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "sample"])
    if kind == "sample":
        rows = _between(rng, 1, 64)
        vocab = _between(rng, 1000, 151_936)
        filters = rng.choice([(0, 1.0, 0.0), (rng.choice([1, 20, 50, 1000]), 1.0, 0.0), (0, round(rng.uniform(0.5, 0.99), 3), 0.0),
                              (rng.choice([40, 64, 200]), round(rng.uniform(0.5, 0.99), 3), 0.0), (0, 1.0, round(rng.uniform(0.01, 0.2), 3))])
        return _sample("", rows, vocab, rng.choice(["f32", "f32", "f16", "bf16"]), *filters, round(rng.uniform(1.0, 4.0), 2))
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (16, 8), (16, 2), (8, 8), (28, 4), (24, 1), (12, 2)])
    dim = rng.choice([64, 128, 128, 128, 256, 80])
    page = rng.choice([16, 16, 32, 64, 24, 256])
    dtype = rng.choice(["f16", "bf16", "bf16", "f32"])
    if kind == "append":
        norm, fused = rng.random() < 0.5, rng.random() < 0.5
        if rng.random() < 0.6:
            tokens = _between(rng, 1, 256)
            seqs, past = tokens, _between(rng, 1, 2000)
        else:
            tokens = _between(rng, 30, 8001 * 48 * 128 // ((heads + 2 * kv_heads) * dim * (2 if dtype == "f32" else 1)) // 2)
            seqs, past = min(tokens, rng.choice([1, 1, 3, 8])), rng.choice([0, 0, 500])
        return _append("", tokens, seqs, past, heads, kv_heads, dim, page, dtype, norm, fused)
    most = 64 * 8000 * 8 * 128 // (kv_heads * dim) // 8  # tokens in all
    batch = _between(rng, 1, 128)
    longest = _between(rng, 20, max(20, min(100_000, most // batch)))
    options = rng.choice([{}, {}, {}, {"softcap": round(rng.uniform(10, 60), 1)}, {"window": _between(rng, 16, 4096)}, {"slopes": True},
                          {"softcap": 30.0, "window": _between(rng, 16, 4096)}])
    return _attention("", batch, longest, rng.random() < 0.6, heads, kv_heads, dim, page, dtype, **options)


def _lengths(case):
    """Visible tokens of each sequence, the new one among them."""
    if case["kind"] == "attention":
        n, longest = case["batch"], case["longest"]
        if not case["ragged"]:
            return [longest - (7 * i) % max(1, longest // 20 + 1) for i in range(n)]
        return [1 + int((longest - 1) * ((0.61803398875 * i) % 1.0 - 1.0) ** 2) for i in range(n)]
    return [case["past"] + n for n in _shares(case)]


def _shares(case):
    """New tokens of each sequence: one each, or a prompt's, longer and shorter ones."""
    seqs, tokens = case["seqs"], case["tokens"]
    cuts = [tokens * i * (i + 1) // (seqs * (seqs + 1)) for i in range(seqs + 1)] if seqs < tokens else list(range(seqs + 1))
    return [b - a for a, b in zip(cuts, cuts[1:])]


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _normal(gen, shape, dtype="f32", scale=1.0):
    return (torch.randn(*shape, device=_DEV, generator=gen) * scale).to(_TORCH[dtype])


def _wrap(t, dtype):
    from torchlette_b200 import CudaTensor, getBackend
    return CudaTensor(getBackend(), list(t.shape), dtype, t.data_ptr(), t.numel() * t.element_size(), ownsBuffer=False)


def _cache(case, gen, lengths):
    """Pages in no order, as after some hours of serving, and what a table has behind a sequence's last page."""
    page, counts = case["page"], [-(-n // case["page"]) for n in lengths]
    widest = max(max(counts), 1)
    pages = sum(counts) + 3
    order = torch.randperm(pages, device=_DEV, generator=gen).to(torch.int32)
    used = torch.arange(widest, device=_DEV)[None, :] < torch.tensor(counts, device=_DEV)[:, None]
    table = torch.full((len(lengths), widest), -1, dtype=torch.int32, device=_DEV)
    table[used] = order[: sum(counts)]
    shape = (pages, case["kv_heads"], page, case["dim"])
    return _normal(gen, shape, case["dtype"]), _normal(gen, shape, case["dtype"]), table


def _prepare_append(case, gen):
    t, h, g, d, dtype = (case[f] for f in ("tokens", "heads", "kv_heads", "dim", "dtype"))
    shares, lengths = _shares(case), _lengths(case)
    k_pages, v_pages, table = _cache(case, gen, lengths)
    s = {"k_pages": k_pages, "v_pages": v_pages, "table": table,
         "seq": torch.repeat_interleave(torch.arange(len(shares)), torch.tensor(shares)).to(torch.int32).to(_DEV),
         "positions": torch.cat([torch.arange(n - new, n) for n, new in zip(lengths, shares)]).to(torch.int32).to(_DEV)}
    if case["fused"]:
        s["qkv"] = _normal(gen, (t, (h + 2 * g) * d), dtype)
    else:
        s["q"], s["k"], s["v"] = (_normal(gen, (t, n, d), dtype) for n in (h, g, g))
    if case["norm"]:
        s["q_norm"], s["k_norm"] = (1 + _normal(gen, (d,), scale=0.2) for _ in range(2))
    angle = torch.arange(max(lengths), dtype=torch.float64, device=_DEV).unsqueeze(1) / 1e6 ** (torch.arange(d // 2, dtype=torch.float64, device=_DEV) / (d // 2))
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    s["q_out"] = torch.empty(t, h, d, device=_DEV, dtype=_TORCH[dtype])
    return s


def _prepare_attention(case, gen):
    b, h, d, dtype = (case[f] for f in ("batch", "heads", "dim", "dtype"))
    lengths = _lengths(case)
    s = dict(zip(("k_pages", "v_pages", "table"), _cache(case, gen, lengths)))
    s["positions"] = (torch.tensor(lengths) - 1).to(torch.int32).to(_DEV)
    s["q"] = _normal(gen, (b, h, d), dtype)
    s["out"] = torch.empty(b, h * d, device=_DEV, dtype=_TORCH[dtype])
    if case["slopes"]:
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, h + 1, device=_DEV) / h)
    return s


def _prepare_sample(case, gen):
    rows, vocab = case["rows"], case["vocab"]
    # most of a vocabulary far behind a few tokens
    logits = torch.randn(rows, vocab, device=_DEV, generator=gen) * case["spread"]
    s = {"logits": logits.to(_TORCH[case["dtype"]]), "uniforms": torch.rand(rows, device=_DEV, generator=gen),
         "temperature": torch.empty(rows, device=_DEV).uniform_(0.6, 1.1, generator=gen),
         "tokens": torch.empty(rows, device=_DEV, dtype=torch.int32)}
    if rows > 4:
        s["temperature"][3::8] = 0.0  # requests that ask for the likeliest token
    for name, key, off in (("top_k", "top_k", 0), ("top_p", "top_p", 1.0), ("min_p", "min_p", 0.0)):
        if case[key] != off:
            s[name] = torch.full((rows,), case[key], device=_DEV, dtype=torch.int32 if key == "top_k" else torch.float32)
    return s


def prepare(case, seed):
    gen = torch.Generator(device=_DEV).manual_seed(int(seed))
    s = {"append": _prepare_append, "attention": _prepare_attention, "sample": _prepare_sample}[case["kind"]](case, gen)
    s["case"] = dict(case)
    if own:  # the handles that a program keeps of its own memory
        from torchlette_b200 import getBackend
        dtype = case["dtype"]
        kinds = {"table": "i32", "positions": "i32", "seq": "i32", "top_k": "i32", "tokens": "i32"}
        f32 = ("q_norm", "k_norm", "cos", "sin", "slopes", "uniforms", "temperature", "top_p", "min_p")
        s["own"] = {name: _wrap(t, kinds.get(name, "f32" if name in f32 else dtype)) for name, t in s.items() if isinstance(t, torch.Tensor)}
        if "table" in s:
            s["own"]["cache"] = getBackend().createPagedCache(s["own"]["k_pages"], s["own"]["v_pages"], s["own"]["table"])
    torch.cuda.synchronize()  # the backend has a stream of its own
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def _heads(s):
    """The new tokens' q, k and v as [tokens, heads, dim]."""
    if "q" in s:
        return s["q"], s["k"], s["v"]
    c = s["case"]
    return s["qkv"].view(c["tokens"], -1, c["dim"]).split([c["heads"], c["kv_heads"], c["kv_heads"]], 1)


def _turn(x, weight, cos, sin, eps=1e-6):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _run_append(s):
    c, pos = s["case"], s["positions"].long()
    q, k, v = _heads(s)
    cos, sin = s["cos"][pos].unsqueeze(1), s["sin"][pos].unsqueeze(1)
    page = s["table"][s["seq"].long(), pos // c["page"]].long()
    dtype = _TORCH[c["dtype"]]
    s["k_pages"][page, :, pos % c["page"]] = _turn(k, s.get("k_norm"), cos, sin).to(dtype)
    s["v_pages"][page, :, pos % c["page"]] = v
    return {"q": _turn(q, s.get("q_norm"), cos, sin).to(dtype), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _run_attention(s):
    c, b, g, d = s["case"], s["case"]["batch"], s["case"]["kv_heads"], s["case"]["dim"]
    rep = c["heads"] // g
    table = s["table"].long().clamp(min=0)
    keys, values = (p[table].transpose(1, 2).reshape(b, g, -1, d).float() for p in (s["k_pages"], s["v_pages"]))
    pos = s["positions"].long()[:, None]
    at = torch.arange(keys.shape[2], device=_DEV)[None, :]
    seen = at <= pos
    if c["window"]:
        seen &= pos - at < c["window"]
    x = torch.matmul(s["q"].float().view(b, g, rep, d), keys.transpose(2, 3)) * (1.0 / math.sqrt(d))
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    if c["slopes"]:
        x = x + s["slopes"].view(1, g, rep, 1) * (at - pos)[:, None, None, :]
    x = x.masked_fill(~seen[:, None, None, :], -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    out = torch.matmul(e, values) / e.sum(-1, keepdim=True)
    return out.reshape(b, c["heads"] * d).to(_TORCH[c["dtype"]])


def _run_sample(s):
    x = s["logits"].double()
    t = s["temperature"].double()[:, None]
    order = torch.sort(x, dim=1, descending=True, stable=True)
    size, index = order
    w = torch.exp((size - size[:, :1]) / torch.where(t > 0, t, 1.0))
    rank = torch.arange(x.shape[1], device=_DEV)[None, :]
    kept = (rank == 0) | (t > 0)
    if "top_k" in s:
        kept &= rank < s["top_k"].long()[:, None]
    if "top_p" in s:
        mass = torch.cumsum(w * kept, 1)
        kept &= (rank == 0) | (mass - w < s["top_p"].double()[:, None] * mass[:, -1:])
    if "min_p" in s:
        kept &= w >= s["min_p"].double()[:, None]
    mass = torch.cumsum(torch.zeros_like(w).scatter_(1, index, w * kept), 1)
    below = mass <= s["uniforms"].double()[:, None] * mass[:, -1:]
    return below.sum(1).to(torch.int32)


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"append": _run_append, "attention": _run_attention, "sample": _run_sample}[kind](s)
    from torchlette_b200 import getBackend
    c, o, ops = s["case"], s["own"], getBackend().ops
    if kind == "append":
        q, k, v = (o["qkv"], None, None) if c["fused"] else (o["q"], o["k"], o["v"])
        ops.pagedAppend(o["cache"], o["positions"], q, k, v, o["cos"], o["sin"], qNorm=o.get("q_norm"), kNorm=o.get("k_norm"), eps=1e-6,
                        tokenSeq=o["seq"], out=o["q_out"])
        return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if kind == "attention":
        ops.pagedAttention(o["cache"], o["positions"], o["q"], 1.0 / math.sqrt(c["dim"]), softcap=c["softcap"], window=c["window"],
                           slopes=o.get("slopes"), out=o["out"])
        return s["out"]
    ops.sample(o["logits"], o["uniforms"], temperature=o["temperature"], topK=o.get("top_k"), topP=o.get("top_p"), minP=o.get("min_p"),
               out=o["tokens"])
    return s["tokens"]


# ---------------------------------------------------------------------------
# What a pass cannot do without, and what it computes in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    size = _SIZE[case["dtype"]]
    if case["kind"] == "append":
        t, h, g, d = (case[f] for f in ("tokens", "heads", "kv_heads", "dim"))
        rows = len({p for n, new in zip(_lengths(case), _shares(case)) for p in range(n - new, n)})  # of the tables
        return {"bytes": 2 * t * (h + 2 * g) * d * size + 4 * rows * d + 12 * t + (8 * d if case["norm"] else 0),
                "flops": t * (h + g) * d * (7 if case["norm"] else 3)}
    if case["kind"] == "attention":
        b, h, g, d, page = (case[f] for f in ("batch", "heads", "kv_heads", "dim", "page"))
        lengths = _lengths(case)
        keys = sum(min(n, case["window"] or n) for n in lengths)
        return {"bytes": 2 * keys * g * d * size + 2 * b * h * d * size + 4 * sum(-(-n // page) for n in lengths) + 4 * b,
                "flops": 4 * h * d * keys}
    rows, vocab = case["rows"], case["vocab"]
    return {"bytes": rows * (vocab * size + 16), "flops": 4 * rows * vocab}


def _exact_append(s):
    c = s["case"]
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    q, k, v = (x.double() for x in _heads(s))
    half = c["dim"] // 2
    cos, sin = s["cos"].double(), s["sin"].double()
    for x, name in ((q, "q_norm"), (k, "k_norm")):
        if c["norm"]:
            x /= (x.square().sum(-1, keepdim=True) / c["dim"] + 1e-6).sqrt()
            x *= s[name].double()
    place = s["positions"].long()
    turned = []
    for x in (q, k):
        z = torch.complex(x[..., :half], x[..., half:]) * torch.complex(cos, sin)[place][:, None, :]
        turned.append(torch.cat([z.real, z.imag], -1))
    slot = s["table"].long().gather(1, (torch.arange(s["table"].shape[1] * c["page"], device=_DEV) // c["page"]).expand(s["table"].shape[0], -1))
    flat = slot[s["seq"].long(), place] * c["page"] + place % c["page"]
    for pages, new in ((k_pages, turned[1]), (v_pages, v)):
        rows = pages.transpose(1, 2).reshape(-1, c["kv_heads"], c["dim"])
        rows[flat] = new
        pages.copy_(rows.view(pages.shape[0], c["page"], c["kv_heads"], c["dim"]).transpose(1, 2))
    return {"q": turned[0], "k_pages": k_pages, "v_pages": v_pages}


def _exact_attention(s):
    c, out = s["case"], []
    rep, last = c["heads"] // c["kv_heads"], s["positions"].tolist()
    for i, p in enumerate(last):
        at = torch.arange(max(0, p + 1 - (c["window"] or p + 1)), p + 1, device=_DEV)
        page = s["table"][i, at // c["page"]].long()
        k, v = (x[page, :, at % c["page"]].double() for x in (s["k_pages"], s["v_pages"]))  # [keys, kv heads, dim]
        q = s["q"][i].double().view(c["kv_heads"], rep, c["dim"])
        x = torch.einsum("grd,jgd->grj", q, k) / math.sqrt(c["dim"])
        if c["softcap"]:
            x = torch.tanh(x / c["softcap"]) * c["softcap"]
        if c["slopes"]:
            x = x - s["slopes"].double().view(c["kv_heads"], rep, 1) * (p - at)
        out.append(torch.einsum("grj,jgd->grd", torch.softmax(x, -1), v).reshape(-1))
    return torch.stack(out)


def _exact_sample(s):
    """Row by row: a token's rank is found by counting, and the kept ones are walked in the order of the vocabulary."""
    out, x = [], s["logits"].double()
    for i in range(x.shape[0]):
        t = float(s["temperature"][i])
        if t <= 0:
            out.append(int((x[i] == x[i].max()).nonzero()[0]))
            continue
        w = torch.exp((x[i] - x[i].max()) / t)
        by_size = torch.argsort(x[i], descending=True, stable=True)
        keep = by_size[: int(s["top_k"][i])] if "top_k" in s else by_size
        if "top_p" in s:
            mass = w[keep].cumsum(0)
            keep = keep[: int((mass < float(s["top_p"][i]) * mass[-1]).sum()) + 1]
        if "min_p" in s:
            keep = keep[w[keep] >= float(s["min_p"][i])]
        keep = keep.sort().values
        mass = w[keep].cumsum(0)
        out.append(int(keep[int((mass <= float(s["uniforms"][i]) * mass[-1]).sum())]))
    return torch.tensor(out, dtype=torch.int32)


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "sample": _exact_sample}[case["kind"]](s)
