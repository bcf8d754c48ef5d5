"""The operators of a decode step over a paged key-value cache: what each computes, on which sizes.

A decode step appends the new token's rotated keys and its values to the sequence's pages
(`paged_append`), lets the token's query heads attend to those pages (`paged_attn`), and ends with
the adjustment of its logits (`adjust_logits`). `run` computes each of them either in its plain form
(elementary torch operations in fp32) or, where `own` is true, through `tread_b200.kernels`.
`exact` gives the same outputs from the definitions in 64 bits.

Head counts, head sizes and vocabularies are the 0.5B, 7B and 32B architectures' of
`tread_b200/configs.py`, lengths those of the benchmark's requests.
"""
import math

import torch

#: Whether `run` calls the framework's kernels instead of computing the plain forms.
own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
THETA = 1e6


# ---- the cases ----------------------------------------------------------------------------------


def _append(name, rows, seqs, hq, hkv, d, page, dtype, past, pad=0, source="rows", rotate="position"):
    """`rows` new tokens of `seqs` sequences with up to `past` tokens in their pages already; the last
    `pad` rows are padding. source "rows": columns of a fused projection [rows, (hq + 2 hkv) d];
    "planes": a dense cache [hkv, rows, d]. rotate: by each row's "position", by one "shift" for all
    rows of a sequence, or "none" (then there are no q heads)."""
    return dict(name=name, op="append", rows=rows, seqs=seqs, hq=hq, hkv=hkv, d=d, page=page, dtype=dtype, past=past,
                pad=pad, source=source, rotate=rotate)


def _attn(name, batch, lo, hi, hq, hkv, d, page, dtype, idle=0):
    """One new token of each of `batch` sequences, their lengths spread from `lo` to `hi` evenly over
    the logarithm; the last `idle` of them have no key at all (padding of a batch)."""
    return dict(name=name, op="attn", batch=batch, lo=lo, hi=hi, hq=hq, hkv=hkv, d=d, page=page, dtype=dtype,
                idle=idle)


def _logits(name, batch, vocab, dtype, prompt, output, bias, mask):
    """Logits of `batch` rows with histories of up to `prompt` + `output` tokens, `bias` biased
    tokens a row, and (mask) a grammar that allows a part of the vocabulary."""
    return dict(name=name, op="logits", batch=batch, vocab=vocab, dtype=dtype, prompt=prompt, output=output, bias=bias,
                mask=mask)


def listed():
    return [
        # the next token of the one request a server decodes (7B heads, 8256 tokens of prompt): latency
        _append("append one token", 1, 1, 28, 4, 128, 64, "bf16", 8256),
        # a decode batch of 64 clients, of which 61 are active
        _append("append batch 64", 64, 64, 28, 4, 128, 64, "bf16", 16640, pad=3),
        # the queries of a few requests prefilled into their pages together, fp32 parity model
        _append("append queries fp32", 250, 5, 14, 2, 64, 16, "fp32", 1000),
        # a whole 32B prompt of 16640 tokens, rotated into its pages
        _append("append prompt", 16640, 1, 40, 8, 128, 16, "bf16", 0),
        # a request cache of all 28 layers x 4 heads moved into pages, re-rotated to another offset
        _append("append request cache", 8256, 1, 0, 112, 128, 64, "bf16", 0, source="planes", rotate="shift"),
        # one request decoding after an 8256-token prompt: latency of the split and the join
        _attn("attend one request", 1, 8257, 8257, 28, 4, 128, 64, "bf16"),
        # 64 clients with prompts of 8 to 24 documents of 256 to 2048 tokens
        _attn("attend batch 64", 64, 2400, 16640, 28, 4, 128, 64, "bf16"),
        # the 32B heads in fp16 on small pages, two places of the batch idle
        _attn("attend 32B fp16", 18, 1000, 16640, 40, 8, 128, 16, "fp16", idle=2),
        # many short chats on the 0.5B heads, from the first token on
        _attn("attend short chats", 256, 1, 700, 14, 2, 64, 16, "bf16"),
        # the fp32 parity model after its request of 1048 tokens
        _attn("attend fp32", 4, 250, 1048, 14, 2, 64, 64, "fp32"),
        # one request's logits, a vocabulary that no vector divides
        _logits("adjust one row", 1, 151935, "bf16", 1048, 64, 20, True),
        # a decode batch's logits after long prompts
        _logits("adjust batch 64", 64, 152064, "bf16", 8256, 512, 100, True),
    ]


HEADS = [(28, 4, 128), (40, 8, 128), (14, 2, 64), (4, 2, 64), (8, 8, 128), (16, 2, 256), (16, 1, 128)]
PAGES = [16, 16, 32, 64, 64, 128, 8, 20, 1]


def _between(rng, lo, hi):
    """A whole number from lo to hi, evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "logits"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    hq, hkv, d = rng.choice(HEADS)
    page = rng.choice(PAGES)
    if op == "append":
        source = rng.choice(["rows", "rows", "planes"])
        rotate = rng.choice(["position", "position", "shift", "none"])
        rows = _between(rng, 1, 16000 if dtype != "fp32" else 8000)
        seqs = _between(rng, 1, min(rows, 256)) if source == "rows" else 1
        pad = rng.choice([0, 0, min(5, rows - 1)])
        past = _between(rng, 1, 20000)
        while seqs * (past // 2) * hkv * d * SIZE[dtype] > 400_000_000:
            past //= 2
        return {k: v for k, v in _append("", rows, seqs, hq if source == "rows" and rotate != "none" else 0, hkv, d, page, dtype, past,
                                         pad, source, rotate).items() if k != "name"}
    if op == "attn":
        batch = _between(rng, 1, 256)
        room = 900_000_000 // (batch * 2 * hkv * d * SIZE[dtype])
        hi = _between(rng, 1, max(1, min(32768, room)))
        lo = _between(rng, 1, hi)
        return {k: v for k, v in _attn("", batch, lo, hi, hq, hkv, d, page, dtype,
                                       idle=rng.choice([0, 0, min(3, batch - 1)])).items() if k != "name"}
    batch = _between(rng, 1, 64)
    return {k: v for k, v in _logits("", batch, _between(rng, 1000, 152064), dtype, _between(rng, 1, 8256),
                                     _between(rng, 1, 512), rng.choice([0, 1, 20, 100]),
                                     rng.random() < 0.5).items() if k != "name"}


# ---- what a user's program has in hand ----------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 11)


def _spread(case):
    """Lengths of an attention batch, without the idle places."""
    n = case["batch"] - case["idle"]
    lo, hi = case["lo"], case["hi"]
    return [int(round(lo * (hi / lo) ** ((i + 0.5) / n))) if n > 1 else hi for i in range(n)]


def _tables(pages, width, g):
    """Page tables of sequences that hold `pages[i]` pages each, drawn from a pool in random order
    with a few pages free; entries behind a sequence's last page are -1."""
    total = sum(pages)
    pool = total + 5
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    count = torch.tensor(pages, device="cuda")
    first = count.cumsum(0) - count
    col = torch.arange(width, device="cuda")
    table = order[(first[:, None] + col).clamp(max=pool - 1)]
    return torch.where(col < count[:, None], table, -1).to(torch.int32).contiguous(), pool


def _randn(shape, dtype, g):
    return torch.randn(shape, dtype=dtype, generator=g, device="cuda")


def _prepare_append(case, g):
    dt, hq, hkv, d, page = DTYPES[case["dtype"]], case["hq"], case["hkv"], case["d"], case["page"]
    rows, seqs, pad = case["rows"], case["seqs"], case["pad"]
    live = rows - pad
    counts = [live // seqs + (i < live % seqs) for i in range(seqs)]
    past = [case["past"] * (i + 1) // seqs for i in range(seqs)]
    perm = torch.randperm(seqs, generator=g, device="cuda").tolist()
    past = [past[i] for i in perm]
    pages = [-(-(a + n) // page) for a, n in zip(past, counts)]
    table, pool = _tables(pages, max(1, max(pages)), g)
    seq = torch.repeat_interleave(torch.arange(seqs), torch.tensor(counts))
    first = torch.tensor(counts).cumsum(0) - torch.tensor(counts)
    pos = torch.tensor(past)[seq] + torch.arange(live) - first[seq]
    seq = torch.cat([seq, torch.zeros(pad, dtype=torch.int64)]).to("cuda", torch.int32)
    pos = torch.cat([pos, torch.full((pad,), -1, dtype=torch.int64)]).to("cuda")
    st = dict(op="append", live=live, table=table, seq=seq, pos=pos, page=page,
              k_pages=_randn((pool, hkv, page, d), dt, g), v_pages=_randn((pool, hkv, page, d), dt, g), q=None)
    if case["source"] == "rows":
        qkv = _randn((rows, (hq + 2 * hkv) * d), dt, g)
        st["q"] = qkv[:, :hq * d].unflatten(1, (hq, d)) if hq else None
        st["k"] = qkv[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
        st["v"] = qkv[:, (hq + hkv) * d:].unflatten(1, (hkv, d))
    else:
        st["k"] = _randn((hkv, rows, d), dt, g).transpose(0, 1)
        st["v"] = _randn((hkv, rows, d), dt, g).transpose(0, 1)
    inv = (1.0 / THETA ** (torch.arange(0, d, 2, dtype=torch.float32) / d)).to("cuda")
    st["inv_freq"] = None if case["rotate"] == "none" else inv
    st["angle"] = pos
    if case["rotate"] == "shift":
        shift = torch.randint(-16384, 16385, (seqs,), generator=g, device="cuda")
        st["angle"] = shift[seq.long()]
    return st


def _prepare_attn(case, g):
    dt, hq, hkv, d, page = DTYPES[case["dtype"]], case["hq"], case["hkv"], case["d"], case["page"]
    lens = _spread(case) + [0] * case["idle"]
    perm = torch.randperm(len(lens), generator=g, device="cuda").tolist()
    lens = [lens[i] for i in perm]
    pages = [-(-n // page) for n in lens]
    table, pool = _tables(pages, max(1, max(pages)), g)
    return dict(op="attn", q=_randn((case["batch"], hq, d), dt, g), table=table, page=page,
                lens=torch.tensor(lens, dtype=torch.int64, device="cuda"),
                k_pages=_randn((pool, hkv, page, d), dt, g), v_pages=_randn((pool, hkv, page, d), dt, g))


def _prepare_logits(case, g):
    b, v = case["batch"], case["vocab"]
    width = case["prompt"] + case["output"]
    frac = torch.rand(b, 2, generator=g, device="cuda")
    prompt = (1 + frac[:, 0] * (case["prompt"] - 1)).round().long()
    lens = prompt + (1 + frac[:, 1] * (case["output"] - 1)).round().long()
    prompt[0], lens[0] = case["prompt"], width
    # the prompt from the whole vocabulary, the output with few distinct tokens, often repeated
    tokens = torch.randint(0, v, (b, width), generator=g, device="cuda")
    again = (torch.rand(b, width, generator=g, device="cuda") ** 4 * min(v, 300)).long()
    col = torch.arange(width, device="cuda")
    said = tokens[:, :1].clamp(max=v - 300 if v > 300 else 0) + again
    tokens = torch.where(col >= prompt[:, None], said, tokens)
    tokens = torch.where(col < lens[:, None], tokens, -1)
    rows = lambda lo, hi: lo + (hi - lo) * torch.rand(b, generator=g, device="cuda")  # noqa: E731
    st = dict(op="logits", logits=(3 * torch.randn(b, v, generator=g, device="cuda")).to(DTYPES[case["dtype"]]),
              tokens=tokens, lens=lens, prompt_lens=prompt, repetition=rows(1.0, 1.5), presence=rows(0.0, 1.0),
              frequency=rows(0.0, 0.5), bias_ids=None, bias=None, allowed=None)
    if case["bias"]:
        at = torch.arange(case["bias"], device="cuda") * (v // case["bias"])
        st["bias_ids"] = (at + torch.randint(0, v // case["bias"], (b, case["bias"]), generator=g, device="cuda"))
        st["bias"] = 4 * torch.randn(b, case["bias"], generator=g, device="cuda")
    if case["mask"]:
        words = (b, (v + 31) // 32)
        st["allowed"] = torch.randint(-2**31, 2**31, words, generator=g, device="cuda").to(torch.int32)
    return st


def prepare(case, seed):
    return {"append": _prepare_append, "attn": _prepare_attn, "logits": _prepare_logits}[case["op"]](
        case, _generator(seed))


# ---- one pass -----------------------------------------------------------------------------------


def _rotate(x, c, s):
    x1, x2 = x.float().chunk(2, -1)
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1)


def _plain_append(st):
    n, page = st["live"], st["page"]
    k, v = st["k"][:n], st["v"][:n]
    q_out = None
    if st["inv_freq"] is not None:
        angle = st["angle"].double()[:, None, None] * st["inv_freq"].double()
        c, s = angle.cos().float(), angle.sin().float()
        k = _rotate(k, c[:n], s[:n]).to(k.dtype)
    if st["q"] is not None:
        q_out = _rotate(st["q"], c, s).to(v.dtype) * (st["pos"] >= 0)[:, None, None]
    pos = st["pos"][:n]
    at = st["table"][st["seq"][:n].long(), pos // page].long()
    st["k_pages"][at, :, pos % page] = k
    st["v_pages"][at, :, pos % page] = v
    return q_out


def _plain_attn(st):
    q, table, lens = st["q"], st["table"], st["lens"]
    b, hq, d = q.shape
    hkv = st["k_pages"].shape[1]
    seen = (torch.arange(table.shape[1] * st["page"], device=q.device) < lens[:, None])[:, None, None]
    at = table.long().clamp(min=0)
    scores = torch.matmul(q.float().view(b, hkv, hq // hkv, d), _keys(st["k_pages"], at).transpose(2, 3)) * d ** -0.5
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weight = torch.exp(scores - top)
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, torch.where(seen.squeeze(2)[..., None], _keys(st["v_pages"], at), 0.0))
    return torch.where(total > 0, out / total, 0.0).view(b, hq, d).to(q.dtype)


def _keys(pages, at):
    """The pages of every sequence side by side, fp32 [batch, heads, tokens, d]."""
    return pages[at].float().transpose(1, 2).flatten(2, 3)


def _plain_logits(st):
    x, tokens, lens, prompt = st["logits"].float(), st["tokens"], st["lens"], st["prompt_lens"]
    b, v = x.shape
    col = torch.arange(tokens.shape[1], device=x.device)
    here = col < lens[:, None]
    new = here & (col >= prompt[:, None])
    one = torch.ones_like(tokens, dtype=torch.float32)
    seen = torch.zeros(b, v + 1, device=x.device).scatter_(1, torch.where(here, tokens, v), one)[:, :v] > 0
    count = torch.zeros(b, v + 1, device=x.device).scatter_add_(1, torch.where(new, tokens, v), one)[:, :v]
    rep = st["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - (st["frequency"][:, None] * count + st["presence"][:, None] * (count > 0))
    if st["bias"] is not None:
        x = x.scatter_add(1, st["bias_ids"], st["bias"])
    if st["allowed"] is not None:
        at = torch.arange(v, device=x.device)
        x = torch.where((st["allowed"][:, at // 32] >> (at % 32)) & 1 > 0, x, -math.inf)
    return x


def _own_append(st):
    from tread_b200 import kernels

    return kernels.paged_append(st["k"], st["v"], st["k_pages"], st["v_pages"], st["table"], st["pos"], seq=st["seq"],
                                inv_freq=st["inv_freq"], rope_pos=st["angle"], q=st["q"])


def _own_attn(st):
    from tread_b200 import kernels

    return kernels.paged_attn(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lens"])


def _own_logits(st):
    from tread_b200 import kernels

    return kernels.adjust_logits(st["logits"], tokens=st["tokens"], lens=st["lens"], prompt_lens=st["prompt_lens"],
                                 repetition=st["repetition"], presence=st["presence"], frequency=st["frequency"],
                                 bias_ids=st["bias_ids"], bias=st["bias"], allowed=st["allowed"])


def run(state):
    if state["op"] == "append":
        q = _own_append(state) if own else _plain_append(state)
        out = {"k_pages": state["k_pages"], "v_pages": state["v_pages"]}
        return out if q is None else {**out, "q": q}
    if state["op"] == "attn":
        return _own_attn(state) if own else _plain_attn(state)
    return _own_logits(state) if own else _plain_logits(state)


# ---- what a pass cannot do without --------------------------------------------------------------


def work(case):
    if case["op"] == "append":
        live, d, es = case["rows"] - case["pad"], case["d"], SIZE[case["dtype"]]
        row = (case["hq"] + 2 * case["hkv"]) * d * es
        turned = (case["hq"] + case["hkv"]) * d if case["rotate"] != "none" else 0
        return {"bytes": 2 * live * row + case["rows"] * 20 + case["pad"] * case["hq"] * d * es,
                "flops": 3 * live * turned}
    if case["op"] == "attn":
        keys, d, es = sum(_spread(case)), case["d"], SIZE[case["dtype"]]
        return {"bytes": 2 * keys * case["hkv"] * d * es + 2 * case["batch"] * case["hq"] * d * es
                + 4 * -(-keys // case["page"]) + 8 * case["batch"],
                "flops": 4 * keys * case["hq"] * d}
    b, v = case["batch"], case["vocab"]
    history = b * (case["prompt"] + case["output"]) // 2  # lengths are spread evenly up to the full ones
    return {"bytes": b * v * (SIZE[case["dtype"]] + 4) + 8 * history + 12 * b * case["bias"]
            + (4 * b * ((v + 31) // 32) if case["mask"] else 0), "flops": 4 * b * v}


# ---- the same from the definitions, in 64 bits ---------------------------------------------------


def _exact_append(st):
    """Pair (i, i + d/2) of a head as a complex number, turned by exp(i angle inv_freq)."""
    n, page = st["live"], st["page"]

    def turned(x):
        x = x.double()
        if st["inv_freq"] is None:
            return x
        half = x.shape[-1] // 2
        w = torch.outer(st["angle"][:x.shape[0]].double(), st["inv_freq"].double())
        z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous())
        z = z * torch.polar(torch.ones_like(w), w)[:, None]
        return torch.cat([z.real, z.imag], -1)

    out = {}
    flat = st["table"][st["seq"][:n].long(), st["pos"][:n] // page].long() * page + st["pos"][:n] % page
    for name, rows in (("k_pages", turned(st["k"][:n])), ("v_pages", st["v"][:n].double())):
        tokens = st[name].double().transpose(1, 2).flatten(0, 1)
        tokens[flat] = rows
        out[name] = tokens.unflatten(0, (-1, page)).transpose(1, 2).contiguous()
    if st["q"] is not None:
        q = turned(st["q"])
        q[n:] = 0
        out["q"] = q
    return out


def _exact_attn(st):
    q = st["q"].double()
    b, hq, d = q.shape
    hkv = st["k_pages"].shape[1]
    out = torch.zeros_like(q)
    for i, n in enumerate(st["lens"].tolist()):
        if n:
            at = st["table"][i, : -(-n // st["page"])].long()
            k, v = (st[p][at].double().permute(1, 0, 2, 3).reshape(hkv, -1, d)[:, :n] for p in ("k_pages", "v_pages"))
            s = torch.einsum("hgd,htd->hgt", q[i].view(hkv, -1, d), k) / math.sqrt(d)
            p = torch.softmax(s, -1)
            out[i] = torch.einsum("hgt,htd->hgd", p, v).reshape(hq, d)
    return out


def _exact_logits(st):
    out = st["logits"].double()
    b, v = out.shape
    for i in range(b):
        n, m = int(st["lens"][i]), int(st["prompt_lens"][i])
        x, rep = out[i], st["repetition"][i].double()
        ids, times = st["tokens"][i, m:n].unique(return_counts=True)
        every = st["tokens"][i, :n].unique()
        x[every] = torch.where(x[every] > 0, x[every] / rep, x[every] * rep)
        x[ids] -= st["frequency"][i].double() * times + st["presence"][i].double()
        if st["bias"] is not None:
            x.index_put_((st["bias_ids"][i],), st["bias"][i].double(), accumulate=True)
        if st["allowed"] is not None:
            word = st["allowed"][i].long() & 0xFFFFFFFF
            bits = (word[:, None] >> torch.arange(32, device=word.device)) & 1
            x[bits.flatten()[:v] == 0] = -math.inf
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attn": _exact_attn, "logits": _exact_logits}[case["op"]](st)
