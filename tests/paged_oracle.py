"""Test infrastructure of the decode-step operators: page tables and the operators' definitions in 64 bits."""
import torch

INV_THETA = 1e6


def make_table(lens, page, gen, spare=3, width=None, device="cuda"):
    """(int32 table [len(lens), width], pool size): every sequence's pages drawn from a shuffled pool;
    entries behind its last page name a page that does not exist."""
    counts = [-(-n // page) for n in lens]
    pool = sum(counts) + spare
    order = torch.randperm(pool, generator=gen, device=device).to(torch.int32)
    table = torch.full((len(lens), width or max(1, max(counts, default=1))), -7, dtype=torch.int32, device=device)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += c
    return table, pool


def inv_freq(D, device="cuda"):
    return (1.0 / INV_THETA ** (torch.arange(0, D, 2, dtype=torch.float32) / D)).to(device)


def rotate64(x, pos, inv):
    """x [R, H, D] rotated by pos [R], in 64 bits."""
    a = pos.double()[:, None, None] * inv.double()
    c, s = a.cos(), a.sin()
    x1, x2 = x.double().chunk(2, -1)
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1)


def rotate_bound(x, y, dtype):
    """How far the rounded rotation y (64 bits) of x may be off: half a step of the output's type, and in
    fp32 the cosine's error (its argument in half turns, at most 1, is rounded by 2^-25: pi 2^-25 <
    2^-23 rad; sincospif itself within 2^-23) and the three roundings of products and sum (3 x 2^-24):
    less than 2^-21 of |x1| + |x2|. Below the type's normal range half a step is half its smallest value."""
    f = torch.finfo(dtype)
    x1, x2 = x.double().abs().chunk(2, -1)
    size = torch.cat([x1 + x2, x1 + x2], -1)
    return f.eps / 2 * y.abs() + 1.01 * size * 2.0 ** -21 + f.smallest_normal * f.eps / 2


def attend64(q, k_pages, v_pages, table, lens, scale=None):
    """(out, weighted |v|, largest sum of |q k| scale) of one-token attention, in 64 bits."""
    B, Hq, D = q.shape
    Hkv, page = k_pages.shape[1], k_pages.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device=q.device)
    size, reach = torch.zeros_like(out), torch.zeros(B, Hq, 1, dtype=torch.float64, device=q.device)
    for b, n in enumerate(lens.tolist()):
        if n <= 0:
            continue
        at = table[b, : -(-n // page)].long()
        k, v = (p[at].double().transpose(0, 1).reshape(Hkv, -1, D)[:, :n] for p in (k_pages, v_pages))
        qb = q[b].double().view(Hkv, Hq // Hkv, D)
        w = torch.softmax(qb @ k.transpose(1, 2) * scale, -1)
        out[b] = (w @ v).view(Hq, D)
        size[b] = (w @ v.abs()).view(Hq, D)
        reach[b] = (qb.abs() @ k.abs().transpose(1, 2)).amax(-1).view(Hq, 1) * scale
    return out, size, reach


def attend_bound(out, size, reach, lens, D, dtype):
    """How far the kernel's output may be off the 64-bit one, with u = half a step of the type:
    u |out| for the last rounding; each weight off by a relative d, which moves the quotient by at most
    2 d (weighted |v|): fp32 scores summed over D products, (D + 2) 2^-24 reach, and the exponential,
    2^-20 (a scaled argument of up to 2^3 rounded by 2^-24 of it, exp2 within 2^-22); fp32 sums over
    the keys, n 2^-24; and 16-bit types round each weight once before it meets v: u (weighted |v|)."""
    f = torch.finfo(dtype)
    u = f.eps / 2
    n = lens.double().clamp(min=1)[:, None, None]
    d = (D + 2) * 2.0 ** -24 * reach + 2.0 ** -20 * (1 + reach / 8) + n * 2.0 ** -24
    return 1.01 * (u * out.abs() + (2 * d + (u if dtype != torch.float32 else 0)) * size) + f.smallest_normal * u


def adjust64(logits, tokens=None, lens=None, prompt_lens=None, repetition=1.0, presence=0.0, frequency=0.0,
             bias_ids=None, bias=None, allowed=None):
    """(adjusted logits, sum of the sizes of their terms) in 64 bits, row by row."""
    out = logits.double().cpu().clone()
    B, V = out.shape
    size = out.abs()
    value = lambda x, b: float(x[b]) if isinstance(x, torch.Tensor) else float(x)  # noqa: E731
    for b in range(B):
        x = out[b]
        if tokens is not None:
            n = tokens.shape[1] if lens is None else min(max(int(lens[b]), 0), tokens.shape[1])
            m = 0 if prompt_lens is None else int(prompt_lens[b])
            row = tokens[b, :n].cpu().tolist()
            for v in sorted(set(row)):
                if not 0 <= v < V:
                    continue
                r = value(repetition, b)
                x[v] = x[v] / r if x[v] > 0 else x[v] * r
                size[b, v] += abs(x[v])
                c = row[max(m, 0):].count(v)
                if c:
                    pen = value(frequency, b) * c + value(presence, b)
                    x[v] -= pen
                    size[b, v] += 3 * (abs(value(frequency, b)) * c + abs(value(presence, b)))
        if bias is not None:
            ids, val = (t if t.dim() == 1 else t[b] for t in (bias_ids, bias))
            for i, v in enumerate(ids.tolist()):
                if 0 <= v < V:
                    x[v] += float(val[i])
                    size[b, v] += 2 * len(ids) * abs(float(val[i]))
        if allowed is not None:
            words = (allowed if allowed.dim() == 1 else allowed[b]).cpu().long() & 0xFFFFFFFF
            bits = (words[:, None] >> torch.arange(32)) & 1
            x[bits.flatten()[:V] == 0] = -torch.inf
    return out.to(logits.device), size.to(logits.device)
