"""Paged caches for tests and the operators' definitions in 64 bits."""
import torch

CONFIGS = [(1, 1, 64), (12, 12, 64), (32, 4, 64), (4, 2, 64), (3, 1, 64), (24, 8, 128), (16, 1, 128), (6, 6, 128), (40, 2, 128)]


def make_cache(lengths, kv_heads, page, D, dtype, device, seed=0, spare=3, token_major=False, poison=True):
    """Pages in random order, table entries and slots behind the last token unusable: NaN slots, entries that name no page."""
    g = torch.Generator().manual_seed(seed)
    used = [(n + page - 1) // page for n in lengths]
    pages = sum(used) + spare
    order = torch.randperm(pages, generator=g).to(torch.int32)
    width = max(1, max(used)) + 1
    table = torch.full((len(lengths), width), 2 ** 30, dtype=torch.int32)
    shape = (pages, page, kv_heads, D) if token_major else (pages, kv_heads, page, D)
    k, v = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    if token_major:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    at = 0
    for s, (n, u) in enumerate(zip(lengths, used)):
        table[s, :u] = order[at:at + u]
        if poison and n % page:
            for t in (k, v):
                t[order[at + u - 1].long(), :, n % page:] = float("nan")
        at += u
    if poison:
        for t in (k, v):
            t[order[at:].long()] = float("nan")
    to = lambda t: t.to(device)
    if token_major:   # .to keeps the strides of dense tensors
        assert to(k).stride() == k.stride()
    return to(k), to(v), to(table), torch.tensor(lengths, dtype=torch.int32, device=device)


def tokens_of(pages, table, s, n):
    """Tokens 0 .. n - 1 of sequence s: ``[kv_heads, n, D]`` in 64 bits."""
    P = pages.shape[2]
    pos = torch.arange(n)
    ids = table.cpu()[s, pos // P].long().to(pages.device)
    return pages[ids, :, (pos % P).to(pages.device)].double().transpose(0, 1)


def attention_ref(q, k_pages, v_pages, table, lengths, offsets, scale):
    """``(o, bound)`` in 64 bits.  With u the half step of the type, P rounded to it costs u sum p |v| (fp16 below its normal
    range 2^-25 of a probability of at least 1 before the division by the sum), the result u |o|.  In fp32: scores are sums of D
    products (D 2^-23 of sum |q k| each way, twice: one score and the maximum), exponentials 2^-22, sums of up to 4096 terms
    in a chain 2^-23 a term."""
    hq, D = q.shape[1:]
    hkv = k_pages.shape[1]
    group = hq // hkv
    u = torch.finfo(q.dtype).eps / 2
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    out, bound = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lens = lengths.tolist()
    offs = list(range(len(lens) + 1)) if offsets is None else offsets.tolist()
    for s, n in enumerate(lens):
        a, b = offs[s], offs[s + 1]
        if n == 0 or a == b:
            continue
        k, v = (tokens_of(t, table, s, n).repeat_interleave(group, 0) for t in (k_pages, v_pages))
        qs = q[a:b].double().transpose(0, 1)
        seen = torch.arange(n, device=q.device)[None] <= torch.arange(n - (b - a), n, device=q.device)[:, None]
        z = (qs @ k.mT * scale).masked_fill(~seen, float("-inf"))
        za = (qs.abs() @ k.abs().mT * scale).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
        p = torch.softmax(z, -1)
        # 0 * NaN of a masked place has no part in the sum
        vz = torch.where(torch.isfinite(v), v, 0.0)
        o = p @ vz
        odd = ~torch.isfinite(v)
        if odd.any():
            for h, j, d in odd.nonzero().tolist():
                rows = seen[:, j]
                o[h, rows, d] += v[h, j, d]
        f = 2.2 * (D + 8) * 2.0 ** -23 * za + (min(n, 4096) + 16) * 2.0 ** -23
        spread = p @ vz.abs()
        out[a:b] = o.transpose(0, 1)
        bound[a:b] = ((u + f) * spread + u * o.abs() + tiny * vz.abs().sum(1, keepdim=True) + 1e-7).transpose(0, 1)
    return out, bound


def append_ref(x, lengths, offsets, n_rot, theta):
    """Rows ``[rows, heads, D]`` with the first ``n_rot`` heads turned to their positions, in 64 bits, and the positions."""
    x = x.double().cpu()
    D = x.shape[2]
    lens = lengths.tolist()
    offs = list(range(len(lens) + 1)) if offsets is None else offsets.tolist()
    pos = torch.full((x.shape[0],), -1, dtype=torch.long)
    for s, n in enumerate(lens):
        if offsets is None and n == 0:
            continue
        pos[offs[s]:offs[s + 1]] = torch.arange(n - (offs[s + 1] - offs[s]), n)
    if theta is not None:
        ang = pos.clamp(min=0).double()[:, None] * theta ** (-2.0 * torch.arange(D // 2).double() / D)
        cs, sn = ang.cos()[:, None], ang.sin()[:, None]
        a, b = x[:, :n_rot, :D // 2], x[:, :n_rot, D // 2:]
        x = torch.cat([torch.cat([a * cs - b * sn, b * cs + a * sn], -1), x[:, n_rot:]], 1)
    return x, pos
