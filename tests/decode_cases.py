"""Inputs and 64-bit references of the decode-step operators' tests."""
import math

import torch


def paged(lengths, page_size, kv_heads, dim, dtype, seed, layout="hnd", extra_pages=3, fill=None):
    """(k, v, block_table): a cache with the sequences' pages in random order.  fill: value of every unused slot."""
    g = torch.Generator("cuda").manual_seed(seed)
    need = [-(-max(n, 0) // page_size) for n in lengths]
    pages = sum(need) + extra_pages
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lengths), max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    shape = (pages, kv_heads, page_size, dim) if layout == "hnd" else (pages, page_size, kv_heads, dim)
    kv = [torch.randn(shape, device="cuda", generator=g).to(dtype) for _ in range(2)]
    kv = kv if layout == "hnd" else [t.transpose(1, 2) for t in kv]
    if fill is not None:
        used = torch.zeros(pages, page_size, dtype=torch.bool)
        for s, n in enumerate(lengths):
            for t in range(max(n, 0)):
                used[table[s, t // page_size], t % page_size] = True
        for t in kv:
            t.masked_fill_(~used.cuda()[:, None, :, None], fill)
    return kv[0], kv[1], table.cuda()


def attention_reference(q, k, v, positions, table, scale, seqs=None):
    """(o, bound): the operator in 64 bits, and how far a result of its precision may be off, element by element.

    bound: a score is a sum of D exact products in chains of D/32 tensor-core adds,
    each off by at most 2^-23 of the running sum of magnitudes (truncation), then 4
    rounding adds, with factors good to 2^-22: |ds| <= (D/32 + 8) 2^-23 A, A the sum
    of |q_i k_i| times scale, +2^-23 times |s| for scaling.  A weight's relative
    error is twice that (its own and the maximum's) and 4 units of exp2; weights and
    sums of n tokens add (n/64 + 24) roundings (64-token tiles, then warps and CTAs).
    """
    rows, heads, dim = q.shape
    kv_heads, page = k.shape[1], k.shape[2]
    group = heads // kv_heads
    o = torch.zeros(rows, heads, dim, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(o)
    u = 2.0 ** -23
    for r, p in enumerate(positions.tolist()):
        if p < 0:
            continue
        s = r if seqs is None else int(seqs[r])
        tok = torch.arange(p + 1, device=q.device)
        pg = table[s].long()[tok // page]
        kk = k[pg, :, tok % page].double().transpose(0, 1).repeat_interleave(group, 0)
        vv = v[pg, :, tok % page].double().transpose(0, 1).repeat_interleave(group, 0)
        qq = q[r].double()
        sc = torch.einsum("hd,htd->ht", qq, kk) * scale
        size = torch.einsum("hd,htd->ht", qq.abs(), kk.abs()) * scale
        w = torch.softmax(sc, -1)
        o[r] = torch.einsum("ht,htd->hd", w, vv)
        rel = 2 * (dim / 32 + 9) * u * size.amax(-1) + (4 + (p + 1) / 64 + 24) * u
        bound[r] = rel[:, None] * torch.einsum("ht,htd->hd", w, vv.abs()) + 1e-37
    return o, bound


def rope_reference(qkv, heads, kv_heads, dim, positions, rot, base, interleaved, q_norm, k_norm, eps, factors=None):
    """(q, k, v) in 64 bits and the pair magnitudes that bound their rounding."""
    rows = qkv.shape[0]
    x = qkv.double().view(rows, heads + 2 * kv_heads, dim)
    q, k, v = x.split([heads, kv_heads, kv_heads], 1)

    def norm(t, w):
        return t if w is None else t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps) * w.double()

    def turn(t):
        size = t.abs().clone()
        y = t.clone()
        if rot:
            i = torch.arange(rot // 2, dtype=torch.float64, device=t.device)
            f = torch.ones_like(i) if factors is None else torch.as_tensor(factors, dtype=torch.float64, device=t.device)
            a = positions.double()[:, None] * (math.log(base) * (-2 * i / rot)).exp() / f
            c, s = a.cos()[:, None], a.sin()[:, None]
            ia = (torch.arange(rot // 2) * 2 if interleaved else torch.arange(rot // 2)).to(t.device)
            ib = ia + 1 if interleaved else ia + rot // 2
            y[..., ia] = t[..., ia] * c - t[..., ib] * s
            y[..., ib] = t[..., ib] * c + t[..., ia] * s
            size[..., ia] = size[..., ib] = t[..., ia].abs() + t[..., ib].abs()
        return y, size

    return turn(norm(q, q_norm)), turn(norm(k, k_norm)), (v, v.abs())
