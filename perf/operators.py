"""Cases of the decode-step operators that stand between the quantized linear layers and after the head.

Three operators, each with a plain form in elementary torch operations and the
call a user makes of the framework's own kernel:

  rope       per-head norm of q and k, position rotation, k and v into the paged cache
  attention  attention of new tokens over the paged cache
  logits     penalties, biases and the grammar mask on the head's logits, and the greedy pick
"""
import math
import random

import numpy as np
import torch

own = False
_backend = None

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one user's next token, the shape of the 8B layer: nothing but latency
        {"name": "rope_1", "op": "rope", "rows": 1, "seqs": 1, "past": 700, "kv_heads": 8, "group": 4, "head_dim": 128,
         "rotated": 128, "interleaved": True, "norm": False, "base": 500000.0, "page": 16, "type": "bf16"},
        # a decode batch with head norms, seven query heads to a key head, an odd row count
        {"name": "rope_57", "op": "rope", "rows": 57, "seqs": 57, "past": 6000, "kv_heads": 4, "group": 7, "head_dim": 128,
         "rotated": 128, "interleaved": False, "norm": True, "base": 1000000.0, "page": 32, "type": "f16"},
        # the end of a very long prompt, far positions, half of each wide head rotated
        {"name": "rope_far_509", "op": "rope", "rows": 509, "seqs": 1, "past": 130000, "kv_heads": 2, "group": 5,
         "head_dim": 256, "rotated": 128, "interleaved": False, "norm": True, "base": 10000.0, "page": 24, "type": "bf16"},
        # prompts of several users in one prefill pass of the 8B layer
        {"name": "rope_8190", "op": "rope", "rows": 8190, "seqs": 9, "past": 1000, "kv_heads": 8, "group": 4, "head_dim": 128,
         "rotated": 128, "interleaved": False, "norm": True, "base": 500000.0, "page": 16, "type": "bf16"},
        # one user, a short conversation: latency
        {"name": "attention_1_short", "op": "attention", "rows": 1, "ahead": 1, "longest": 555, "shortest": 555, "empty": 0,
         "kv_heads": 8, "group": 4, "head_dim": 128, "page": 16, "type": "bf16"},
        # one user, a very long document: the length has to be split over the whole chip
        {"name": "attention_1_long", "op": "attention", "rows": 1, "ahead": 1, "longest": 131000, "shortest": 131000,
         "empty": 0, "kv_heads": 8, "group": 4, "head_dim": 128, "page": 16, "type": "bf16"},
        # a serving batch of the 8B layer, lengths from a greeting to a long chat
        {"name": "attention_64_ragged", "op": "attention", "rows": 64, "ahead": 1, "longest": 16000, "shortest": 70, "empty": 3,
         "kv_heads": 8, "group": 4, "head_dim": 128, "page": 16, "type": "bf16"},
        # many short chats, small heads, seven query heads to a key head, odd pages
        {"name": "attention_230_short", "op": "attention", "rows": 230, "ahead": 1, "longest": 900, "shortest": 5, "empty": 7,
         "kv_heads": 2, "group": 7, "head_dim": 64, "page": 20, "type": "f16"},
        # four drafted tokens of each of six users checked at once, wide heads of the 70B layer's grouping
        {"name": "attention_24_drafted", "op": "attention", "rows": 24, "ahead": 4, "longest": 6000, "shortest": 900, "empty": 0,
         "kv_heads": 4, "group": 8, "head_dim": 256, "page": 64, "type": "bf16"},
        # one user's logits, a few hundred tokens of history: latency
        {"name": "logits_1", "op": "logits", "rows": 1, "vocab": 128256, "longest": 600, "shortest": 600, "biases": 0,
         "mask": False, "greedy": True},
        # an odd vocabulary with biases and a grammar, in a small batch
        {"name": "logits_7_odd", "op": "logits", "rows": 7, "vocab": 32003, "longest": 1500, "shortest": 3, "biases": 300,
         "mask": True, "greedy": True},
        # a full serving batch with everything on
        {"name": "logits_190", "op": "logits", "rows": 190, "vocab": 151936, "longest": 8000, "shortest": 20, "biases": 40,
         "mask": True, "greedy": True},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rope", "attention", "attention", "logits"])
    if op == "logits":
        rows = _log(rng, 1, 180)
        longest = _log(rng, 1, 8000)
        return {"op": op, "rows": rows, "vocab": _log(rng, 1000, 151936), "longest": longest,
                "shortest": rng.randint(0, longest), "biases": rng.choice([0, 0, 3, 64, 300]), "mask": rng.random() < 0.5,
                "greedy": rng.random() < 0.7}
    kv, group, dim = rng.choice([1, 2, 3, 4, 8]), rng.randint(1, 10), rng.choice([64, 96, 128, 256])
    heads = {"kv_heads": kv, "group": group, "head_dim": dim, "page": rng.choice([1, 7, 16, 16, 32, 48, 64, 256]),
             "type": rng.choice(["bf16", "f16"])}
    if op == "rope":
        most = max(1, min(8190, (8190 * 48 * 128) // (kv * (group + 2) * dim)))
        rows = _log(rng, 1, most)
        seqs = rng.choice([1, max(1, rows // 50), rows])
        past = min(_log(rng, 1, 130000), 60_000_000 // (kv * dim * seqs))
        return {"op": op, "rows": rows, "seqs": seqs, "past": past, "rotated": rng.choice([dim, dim, dim // 2]),
                "interleaved": rng.random() < 0.5, "norm": rng.random() < 0.5, "base": rng.choice([10000.0, 500000.0, 1000000.0]),
                **heads}
    seqs = _log(rng, 1, 250)
    ahead = rng.choice([1, 1, 1, 2, 5])
    most = max(8, min(131000, 150_000_000 // (seqs * ahead * kv * dim)))
    longest = _log(rng, 4, most)
    return {"op": op, "rows": seqs * ahead, "ahead": ahead, "longest": max(ahead, longest),
            "shortest": rng.randint(ahead, max(ahead, longest)), "empty": rng.choice([0, 0, seqs // 9]), **heads}


def _spread(count, shortest, longest):
    """`count` lengths from the shortest to the longest, evenly over the logarithm: the same for every seed."""
    if count == 1:
        return [longest]
    a, b = math.log(shortest + 1), math.log(longest + 1)
    return [int(round(math.exp(a + (b - a) * i / (count - 1)))) - 1 for i in range(count)]


def _attention_lengths(case):
    """Cached tokens of each sequence, its new ones among them; the first `empty` sequences have none."""
    seqs = case["rows"] // case["ahead"]
    ls = _spread(seqs, case["shortest"], case["longest"])
    return [0] * case["empty"] + ls[case["empty"]:]


def _paged(r, lengths, page):
    """A block table with the pages of all sequences in random order; -1 where a sequence has no page."""
    need = [-(-n // page) for n in lengths]
    total, wide = sum(need) + 1, max(1, max(need))
    order = list(range(total))
    r.shuffle(order)
    table, at = np.full((len(lengths), wide), -1, np.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return torch.from_numpy(table).cuda(), total


def _framework():
    global _backend
    if _backend is None:
        from ocelotl_b200 import CudaKernelBackend
        _backend = CudaKernelBackend(0)
    return _backend


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    r = random.Random(seed)
    return {"rope": _prepare_rope, "attention": _prepare_attention, "logits": _prepare_logits}[case["op"]](case, g, r)


def _prepare_rope(case, g, r):
    rows, seqs, kv, dim, page = case["rows"], case["seqs"], case["kv_heads"], case["head_dim"], case["page"]
    heads = kv * case["group"]
    seq = [i * seqs // rows for i in range(rows)]
    first = [seq.index(s) for s in range(seqs)]
    start = [r.randint(case["past"] // 2, case["past"]) for _ in range(seqs)]
    pos = [start[s] + i - first[s] for i, s in enumerate(seq)]
    table, pages = _paged(r, [case["past"] + -(-rows // seqs)] * seqs, page)
    weights = [1 + 0.2 * torch.randn(dim, device="cuda", generator=g) for _ in range(2)]
    state = {
        "case": case, "table": table,
        "qkv": torch.randn(rows, (heads + 2 * kv) * dim, device="cuda", generator=g) * 1.7,
        "k": torch.zeros(pages, kv, page, dim, device="cuda", dtype=TYPES[case["type"]]),
        "v": torch.zeros(pages, kv, page, dim, device="cuda", dtype=TYPES[case["type"]]),
        "positions": torch.tensor(pos, dtype=torch.int32, device="cuda"),
        "seqs": None if seqs == rows else torch.tensor(seq, dtype=torch.int32, device="cuda"),
        "q_norm": weights[0] if case["norm"] else None, "k_norm": weights[1] if case["norm"] else None,
        "eps": 1e-6,
    }
    if own:
        b = _framework()
        state["cache"] = b.kv_cache_view(state["k"], state["v"])
        state["rope"] = b.rope_table(case["rotated"], case["base"], interleaved=case["interleaved"])
    return state


def _prepare_attention(case, g, r):
    kv, dim, ahead = case["kv_heads"], case["head_dim"], case["ahead"]
    lengths = _attention_lengths(case)
    r.shuffle(lengths)
    table, pages = _paged(r, lengths, case["page"])
    pos = [n - ahead + i if n else -1 for n in lengths for i in range(ahead)]
    seq = [s for s in range(len(lengths)) for _ in range(ahead)]
    shape, kind = (pages, kv, case["page"], dim), TYPES[case["type"]]
    state = {
        "case": case, "table": table,
        "k": torch.randn(shape, device="cuda", generator=g, dtype=kind),
        "v": torch.randn(shape, device="cuda", generator=g, dtype=kind),
        "q": torch.randn(case["rows"], kv * case["group"], dim, device="cuda", generator=g) * 1.5,
        "positions": torch.tensor(pos, dtype=torch.int32, device="cuda"),
        "seqs": None if ahead == 1 else torch.tensor(seq, dtype=torch.int32, device="cuda"),
        "scale": dim ** -0.5,
    }
    if own:
        state["cache"] = _framework().kv_cache_view(state["k"], state["v"])
    return state


def _prepare_logits(case, g, r):
    rows, vocab, longest = case["rows"], case["vocab"], max(1, case["longest"])
    lens = _spread(rows, case["shortest"], case["longest"])
    r.shuffle(lens)
    u = torch.rand(rows, longest, device="cuda", generator=g)
    state = {
        "case": case,
        "logits": torch.randn(rows, vocab, device="cuda", generator=g) * 3,
        "history": (u ** 3 * (vocab - 1)).round().to(torch.int32),  # a few tokens come often, most seldom
        "history_lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
        "prompt_lens": torch.tensor([r.randint(0, n) for n in lens], dtype=torch.int32, device="cuda"),
        "repetition": 1 + torch.rand(rows, device="cuda", generator=g) * 0.3,
        "frequency": torch.rand(rows, device="cuda", generator=g) * 0.4,
        "presence": torch.rand(rows, device="cuda", generator=g) * 0.4,
        "bias_ids": None, "bias_values": None, "allowed": None,
    }
    if case["biases"]:
        n = case["biases"]
        pick = torch.rand(rows, vocab, device="cuda", generator=g).topk(n, dim=1).indices.to(torch.int32)
        pick[torch.rand(rows, n, device="cuda", generator=g) < 0.1] = -1  # places that a request leaves unused
        state["bias_ids"] = pick
        state["bias_values"] = torch.randn(rows, n, device="cuda", generator=g) * 4
    if case["mask"]:
        words = (vocab + 31) // 32
        state["allowed"] = torch.randint(-2**31, 2**31, (rows, words), device="cuda", generator=g).to(torch.int32)
    if own:
        state["rules"] = _framework().logit_rules(**{k: state[k] for k in (
            "history", "history_lens", "prompt_lens", "repetition", "frequency", "presence", "bias_ids", "bias_values",
            "allowed")})
    return state


def run(state):
    case = state["case"]
    if own:
        b = _framework()
        if case["op"] == "rope":
            q = b.qk_norm_rope(state["qkv"], state["cache"], state["positions"], state["table"], state["rope"],
                               q_norm=state["q_norm"], k_norm=state["k_norm"], eps=state["eps"], seqs=state["seqs"])
            return {"q": q, "k": state["k"], "v": state["v"]}
        if case["op"] == "attention":
            return b.paged_attention(state["q"], state["cache"], state["positions"], state["table"], scale=state["scale"],
                                     seqs=state["seqs"])
        if case["greedy"]:
            ids = torch.empty(case["rows"], dtype=torch.int32, device="cuda")
            return {"logits": b.process_logits(state["logits"], state["rules"], ids=ids), "ids": ids}
        return {"logits": b.process_logits(state["logits"], state["rules"])}
    return {"rope": _plain_rope, "attention": _plain_attention, "logits": _plain_logits}[case["op"]](state)


def _row_seqs(state):
    rows = state["positions"].shape[0]
    return torch.arange(rows, device="cuda") if state["seqs"] is None else state["seqs"].long()


def _plain_norm(x, w, eps):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w


def _plain_rotate(x, cos, sin, rotated, interleaved):
    half = rotated // 2
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:rotated:2], x[..., 1:rotated:2]
        y[..., 0:rotated:2], y[..., 1:rotated:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :half], x[..., half:rotated]
        y[..., :half], y[..., half:rotated] = a * cos - b * sin, b * cos + a * sin
    return y


def _plain_rope(state):
    case = state["case"]
    rows, kv, dim, page = case["rows"], case["kv_heads"], case["head_dim"], case["page"]
    heads = kv * case["group"]
    q, k, v = state["qkv"].view(rows, heads + 2 * kv, dim).split([heads, kv, kv], dim=1)
    if state["q_norm"] is not None:
        q, k = _plain_norm(q, state["q_norm"], state["eps"]), _plain_norm(k, state["k_norm"], state["eps"])
    i = torch.arange(case["rotated"] // 2, device="cuda", dtype=torch.float64)
    angle = state["positions"].double()[:, None] * case["base"] ** (-2 * i / case["rotated"])
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q = _plain_rotate(q, cos, sin, case["rotated"], case["interleaved"])
    k = _plain_rotate(k, cos, sin, case["rotated"], case["interleaved"])
    pos = state["positions"].long()
    at = state["table"][_row_seqs(state), pos // page].long()
    state["k"][at, :, pos % page] = k.to(state["k"].dtype)
    state["v"][at, :, pos % page] = v.to(state["v"].dtype)
    return {"q": q, "k": state["k"], "v": state["v"]}


def _plain_attention(state):
    case = state["case"]
    rows, kv, dim, group, ahead = case["rows"], case["kv_heads"], case["head_dim"], case["group"], case["ahead"]
    pages = state["table"].clamp(min=0).long()
    seqs = pages.shape[0]
    k = state["k"][pages].transpose(1, 2).reshape(seqs, kv, -1, dim).float()
    v = state["v"][pages].transpose(1, 2).reshape(seqs, kv, -1, dim).float()
    q = state["q"].view(seqs, ahead, kv, group, dim).transpose(1, 2).reshape(seqs, kv, ahead * group, dim)
    s = (q @ k.transpose(-1, -2) * state["scale"]).view(seqs, kv, ahead, group, -1)
    hidden = torch.arange(s.shape[-1], device="cuda") > state["positions"].view(seqs, 1, ahead, 1, 1)
    s = s.masked_fill(hidden, -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp().masked_fill(hidden, 0.0)
    total = p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = (p.view(seqs, kv, ahead * group, -1) @ v).view(seqs, kv, ahead, group, dim) / total
    return o.transpose(1, 2).reshape(rows, kv * group, dim)


def _plain_logits(state):
    case = state["case"]
    rows, vocab = case["rows"], case["vocab"]
    at = torch.arange(state["history"].shape[1], device="cuda")[None]
    here = (at < state["history_lens"][:, None]).int()
    made = here * (at >= state["prompt_lens"][:, None])
    ids = state["history"].long()
    seen = torch.zeros(rows, vocab, dtype=torch.int32, device="cuda").scatter_add_(1, ids, here) > 0
    count = torch.zeros(rows, vocab, dtype=torch.int32, device="cuda").scatter_add_(1, ids, made)
    x, rep = state["logits"], state["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    y = (x - state["frequency"][:, None] * count.float()) - state["presence"][:, None]
    x = torch.where(count > 0, y, x)
    if state["bias_ids"] is not None:
        used = state["bias_ids"] >= 0
        x = x.scatter_add(1, state["bias_ids"].clamp(min=0).long(), state["bias_values"].masked_fill(~used, 0.0))
    if state["allowed"] is not None:
        bit = torch.arange(32, dtype=torch.int32, device="cuda")
        allowed = ((state["allowed"][:, :, None] >> bit) & 1).reshape(rows, -1)[:, :vocab].bool()
        x = x.masked_fill(~allowed, -math.inf)
    return {"logits": x, "ids": x.argmax(-1).to(torch.int32)} if case["greedy"] else {"logits": x}


def work(case):
    if case["op"] == "rope":
        kv, heads, dim = case["kv_heads"], case["kv_heads"] * case["group"], case["head_dim"]
        a_row = ((heads + 2 * kv) * 4 + heads * 4 + 2 * kv * 2) * dim + 8
        return {"bytes": case["rows"] * a_row, "flops": case["rows"] * (heads + kv) * dim * (7 if case["norm"] else 3)}
    if case["op"] == "attention":
        kv, heads, dim, ahead = case["kv_heads"], case["kv_heads"] * case["group"], case["head_dim"], case["ahead"]
        ls = _attention_lengths(case)
        seen = sum((n - ahead + 1 + i) for n in ls if n for i in range(ahead))
        return {"bytes": sum(ls) * kv * dim * 4 + case["rows"] * heads * dim * 8, "flops": 4 * seen * heads * dim}
    rows, vocab = case["rows"], case["vocab"]
    lens = _spread(rows, case["shortest"], case["longest"])
    return {"bytes": rows * vocab * (8 + (0.125 if case["mask"] else 0)) + 4 * sum(lens) + rows * 8 * case["biases"],
            "flops": 2 * rows * vocab}


def exact(case, seed):
    state = prepare(case, seed)
    return {"rope": _exact_rope, "attention": _exact_attention, "logits": _exact_logits}[case["op"]](case, state)


def _exact_rope(case, state):
    kv, dim, page, rot = case["kv_heads"], case["head_dim"], case["page"], case["rotated"]
    heads = kv * case["group"]
    x = state["qkv"].double().reshape(case["rows"], -1, dim)
    if case["norm"]:
        weight = torch.ones(heads + 2 * kv, dim, device="cuda", dtype=torch.float64)
        weight[:heads], weight[heads:heads + kv] = state["q_norm"].double(), state["k_norm"].double()
        size = torch.sqrt((x * x).sum(-1, keepdim=True) / dim + state["eps"])
        size[:, heads + kv:] = 1
        x = x / size * weight
    turn = torch.tensor([math.pow(case["base"], -2.0 * i / rot) for i in range(rot // 2)], device="cuda", dtype=torch.float64)
    turn = torch.polar(torch.ones_like(turn), torch.zeros_like(turn)) * torch.exp(
        1j * torch.outer(state["positions"].double(), turn))
    part = x[:, :heads + kv, :rot]
    if case["interleaved"]:
        z = torch.complex(part[..., 0::2].contiguous(), part[..., 1::2].contiguous()) * turn[:, None]
        y = torch.stack([z.real, z.imag], -1).flatten(-2)
    else:
        z = torch.complex(part[..., :rot // 2].contiguous(), part[..., rot // 2:].contiguous()) * turn[:, None]
        y = torch.cat([z.real, z.imag], -1)
    x = torch.cat([torch.cat([y, x[:, :heads + kv, rot:]], -1), x[:, heads + kv:]], 1)
    k, v = state["k"].double(), state["v"].double()
    seqs = range(case["rows"]) if state["seqs"] is None else state["seqs"].tolist()
    table = state["table"].tolist()
    pos = state["positions"].tolist()
    slot = torch.tensor([table[s][p // page] * page + p % page for s, p in zip(seqs, pos)], device="cuda")
    k.transpose(1, 2)[slot // page, slot % page] = x[:, heads:heads + kv]
    v.transpose(1, 2)[slot // page, slot % page] = x[:, heads + kv:]
    return {"q": x[:, :heads].contiguous(), "k": k, "v": v}


def _exact_attention(case, state):
    kv, dim, page, ahead = case["kv_heads"], case["head_dim"], case["page"], case["ahead"]
    out = torch.zeros(case["rows"], kv * case["group"], dim, dtype=torch.float64, device="cuda")
    for row, pos in enumerate(state["positions"].tolist()):
        if pos < 0:
            continue
        mine = state["table"][row // ahead, :pos // page + 1].long()
        keys = torch.cat(list(state["k"][mine].double()), 1)[:, :pos + 1]
        values = torch.cat(list(state["v"][mine].double()), 1)[:, :pos + 1]
        q = state["q"][row].double().view(kv, case["group"], dim)
        weight = torch.softmax(torch.bmm(q, keys.mT) * state["scale"], -1)
        out[row] = torch.bmm(weight, values).reshape(-1, dim)
    return out


def _exact_logits(case, state):
    out = state["logits"].double().cpu().numpy()
    hist, lens, prompts = (state[k].cpu().numpy() for k in ("history", "history_lens", "prompt_lens"))
    rep, freq, pres = (state[k].double().cpu().numpy() for k in ("repetition", "frequency", "presence"))
    ids, values = (None if state[k] is None else state[k].cpu().numpy() for k in ("bias_ids", "bias_values"))
    allowed = None if state["allowed"] is None else state["allowed"].cpu().numpy()
    for r in range(case["rows"]):
        x = out[r]
        seen = np.unique(hist[r, :lens[r]])
        x[seen] = np.where(x[seen] > 0, x[seen] / rep[r], x[seen] * rep[r])
        made, times = np.unique(hist[r, prompts[r]:lens[r]], return_counts=True)
        x[made] -= freq[r] * times + pres[r]
        if ids is not None:
            for t, b in zip(ids[r], values[r]):
                if t >= 0:
                    x[t] += float(b)
        if allowed is not None:
            bits = np.unpackbits(allowed[r].view(np.uint8), bitorder="little")[:case["vocab"]]
            x[bits == 0] = -np.inf
    return {"logits": out, "ids": None} if case["greedy"] else {"logits": out}
