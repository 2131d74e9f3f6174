"""Workloads of the KV-cache attention operators: what is timed, its plain form and its 64-bit definition.

Four operators over the decoder's f32 caches ``[batch][kv_heads][max_t][128]``:

* ``tree``    -- RoPE, cache append and attention of a tree of drafted tokens per sequence;
* ``weights`` -- causal attention (one token or a prompt chunk) that also adds every key's
  softmax weight to a per-key accumulator;
* ``evict``   -- keep the heaviest rows of a cache by that accumulator, in place, in order;
* ``blocks``  -- attention over the blocks of keys that a score against block means selects.

``own`` False runs the plain form (elementary torch operations), True the framework's calls.
"""
import math

import torch

own = False

D = 128
SCALE = float(torch.tensor(1.0 / math.sqrt(D), dtype=torch.float32))


def listed():
    return [
        # one sequence, a small draft after a short prompt (the decoder's default cache of 640 rows)
        {"name": "tree_short", "op": "tree", "batch": 1, "hq": 16, "hkv": 2, "n": 8, "pos": 200, "step": 0,
         "max_t": 640},
        # no grouping, a long history, a draft of 16: the cache is the work
        {"name": "tree_long_mha", "op": "tree", "batch": 1, "hq": 16, "hkv": 16, "n": 16, "pos": 16001, "step": 0,
         "max_t": 16384},
        # a ragged batch with odd sizes
        {"name": "tree_ragged", "op": "tree", "batch": 5, "hq": 16, "hkv": 2, "n": 33, "pos": 2001, "step": 333,
         "max_t": 2048},
        # a wide draft for a batch with long histories: 512 query rows share each kv head
        {"name": "tree_wide", "op": "tree", "batch": 8, "hq": 16, "hkv": 2, "n": 64, "pos": 8100, "step": 101,
         "max_t": 8192},
        # the decode step of one sequence with weight tracking
        {"name": "weights_token", "op": "weights", "batch": 1, "hq": 16, "hkv": 2, "t": 1, "pos": 500, "step": 0,
         "max_t": 640},
        # the decode step of a batch with long ragged histories
        {"name": "weights_tokens_long", "op": "weights", "batch": 8, "hq": 16, "hkv": 16, "t": 1, "pos": 8100,
         "step": 211, "max_t": 8192},
        # the decoder's prompt of 4 x 1024 tokens
        {"name": "weights_prompt", "op": "weights", "batch": 4, "hq": 16, "hkv": 2, "t": 1024, "pos": 0, "step": 0,
         "max_t": 1024},
        # shrinking the decoder's default cache to half
        {"name": "evict_short", "op": "evict", "batch": 1, "hkv": 2, "len": 640, "step": 0, "keep": 320, "sink": 4,
         "recent": 64, "max_t": 640},
        # a batch of long caches, no grouping
        {"name": "evict_long", "op": "evict", "batch": 4, "hkv": 16, "len": 8001, "step": 117, "keep": 4096,
         "sink": 16, "recent": 500, "max_t": 8192},
        # one token over a long history: 17 blocks of 64 keys instead of 32 K keys
        {"name": "blocks_token", "op": "blocks", "batch": 1, "hq": 16, "hkv": 2, "t": 1, "pos": 32001, "step": 0,
         "block": 64, "topk": 16, "max_t": 32768},
        # a batch of single tokens, no grouping
        {"name": "blocks_tokens", "op": "blocks", "batch": 8, "hq": 16, "hkv": 16, "t": 1, "pos": 16001, "step": 555,
         "block": 64, "topk": 16, "max_t": 16384},
        # a prompt chunk behind a long history, every row with blocks of its own
        {"name": "blocks_chunk", "op": "blocks", "batch": 1, "hq": 16, "hkv": 2, "t": 512, "pos": 16001, "step": 0,
         "block": 64, "topk": 16, "max_t": 16896},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "weights", "weights", "evict", "blocks"])
    hq, hkv = rng.choice([(16, 2), (16, 16), (16, 4), (8, 1), (12, 4), (32, 2)])
    batch = rng.randint(1, 6)
    step = rng.choice([0, 1, 37, 120])
    if op == "tree":
        n = _log_int(rng, 1, 96)
        pos = min(_log_int(rng, 16, 16000), int(8 * 16 * 64 * 8000 / (batch * hq * n)), 100000 // (batch * hkv))
        return {"op": op, "batch": batch, "hq": hq, "hkv": hkv, "n": n, "pos": pos, "step": step,
                "max_t": pos + n + rng.randint(0, 300)}
    if op == "weights" and rng.random() < 0.5:
        pos = min(_log_int(rng, 16, 16000), 400000 // (batch * hkv))
        return {"op": op, "batch": batch, "hq": hq, "hkv": hkv, "t": 1, "pos": pos, "step": step,
                "max_t": pos + 1 + rng.randint(0, 300)}
    if op == "weights":
        t = _log_int(rng, 2, 900)
        pos = rng.choice([0, rng.randint(1, 1000)])
        batch = max(1, min(batch, 1000000 // ((t + pos) * t)))
        return {"op": op, "batch": batch, "hq": hq, "hkv": hkv, "t": t, "pos": pos, "step": min(step, pos),
                "max_t": pos + t + rng.randint(0, 300)}
    if op == "evict":
        length = min(_log_int(rng, 64, 16000), 400000 // (batch * hkv))
        keep = rng.randint(length // 4, length - 1)
        return {"op": op, "batch": batch, "hkv": hkv, "len": length, "step": step, "keep": keep,
                "sink": rng.randint(0, keep // 8), "recent": rng.randint(0, keep // 4),
                "max_t": length + rng.randint(0, 300)}
    t = rng.choice([1, 1, _log_int(rng, 2, 300)])
    block = rng.choice([16, 32, 64, 128])
    topk = rng.randint(1, 512 // block + 4)
    pos = min(_log_int(rng, 16, 30000), 200000 // (batch * hkv))
    batch = max(1, min(batch, 8000 * 64 // (t * hkv * topk * block)))
    return {"op": op, "batch": batch, "hq": hq, "hkv": hkv, "t": t, "pos": pos, "step": step, "block": block,
            "topk": topk, "max_t": pos + t + rng.randint(0, 300)}


def _positions(case, key="pos"):
    """Per-sequence lengths: the case's, less `step` for each further sequence."""
    return [max(0, case[key] - b * case["step"]) for b in range(case["batch"])]


def _rope_tables(rows, device):
    freq = (10000.0 ** (-2.0 * torch.arange(D // 2, dtype=torch.float64) / D)).float()
    ang = torch.arange(rows, dtype=torch.float32)[:, None] * freq
    return ang.double().cos().float().to(device), ang.double().sin().float().to(device)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed * 7919 + 17)
    op, batch, hkv, max_t = case["op"], case["batch"], case["hkv"], case["max_t"]
    randn = lambda *s: torch.randn(s, generator=g, device=dev)
    st = {"case": dict(case), "op": op,
          # rows past a sequence's length hold an earlier sequence's keys and values
          "k": randn(batch, hkv, max_t, D), "v": randn(batch, hkv, max_t, D)}
    lens = _positions(case, "len" if op == "evict" else "pos")
    st["pos"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    if op == "tree":
        n = case["n"]
        st["qkv"] = randn(batch, n, (case["hq"] + 2 * hkv) * D)
        # a draft: each node continues one of the few nodes before it, or the context
        u = torch.rand((batch, n), generator=g, device=dev)
        i = torch.arange(n, device=dev)
        back = (u * torch.clamp(i + 1, max=6)).long()
        st["parents"] = torch.clamp(i - 1 - back, min=-1).to(torch.int32)
        st["cos"], st["sin"] = _rope_tables(max_t, dev)
    elif op == "weights":
        st["q"] = randn(batch, case["t"], case["hq"], D) * 1.5
        st["weight"] = torch.rand((batch, hkv, max_t), generator=g, device=dev)
    elif op == "evict":
        # accumulated weights span orders of magnitude; some rows were never looked at
        st["weight"] = torch.exp(2.0 * randn(batch, hkv, max_t)) * (torch.rand((batch, hkv, max_t), generator=g,
                                                                               device=dev) > 0.05)
        st["weight_out"] = torch.empty_like(st["weight"])
    else:
        st["q"] = randn(batch, case["t"], case["hq"], D) * 1.5
        nb = -(-max_t // case["block"])
        pad = torch.nn.functional.pad(st["k"], (0, 0, 0, nb * case["block"] - max_t))
        st["keys"] = pad.view(batch, hkv, nb, case["block"], D).mean(3).contiguous()
    if op != "evict":
        st["out"] = torch.empty((batch, case["n" if op == "tree" else "t"], case["hq"], D), device=dev)
    return st


def run(st):
    return (_own if own else _plain)[st["op"]](st)


# -- the framework's calls -----------------------------------------------------------------

def _own_tree(st):
    from talechime_b200 import attention

    attention.rope_attention_tree(st["qkv"], st["parents"], st["pos"], st["cos"], st["sin"], st["k"], st["v"],
                                  out=st["out"])
    return st["out"], st["k"], st["v"]


def _own_weights(st):
    from talechime_b200 import attention

    attention.attention_weights(st["q"], st["k"], st["v"], st["pos"], st["weight"], out=st["out"])
    return st["out"], st["weight"]


def _own_evict(st):
    from talechime_b200 import attention

    c = st["case"]
    index = attention.kv_evict(st["weight"], st["k"], st["v"], st["pos"], c["keep"], sink=c["sink"],
                               recent=c["recent"], weight_out=st["weight_out"])
    return index, st["k"], st["v"], st["weight_out"]


def _own_blocks(st):
    from talechime_b200 import attention

    c = st["case"]
    out, index = attention.attention_blocks(st["q"], st["k"], st["v"], st["keys"], st["pos"], c["block"], c["topk"],
                                            out=st["out"])
    return out, index


_own = {"tree": _own_tree, "weights": _own_weights, "evict": _own_evict, "blocks": _own_blocks}


# -- the plain forms -----------------------------------------------------------------------

def _ancestors(parents):
    """[batch][n][n]: j is i or an ancestor of i, by repeated squaring of (identity + parent)."""
    n = parents.shape[1]
    j = torch.arange(n, device=parents.device)
    m = ((parents.long()[:, :, None] == j) | (j[:, None] == j)).float()
    for _ in range(max(1, (n - 1).bit_length())):
        m = (torch.matmul(m, m) > 0).float()
    return m > 0


def _softmax(s):
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain_tree(st):
    c, k, v, pos = st["case"], st["k"], st["v"], st["pos"].long()
    b, n, hq, hkv = c["batch"], c["n"], c["hq"], c["hkv"]
    g, L = hq // hkv, c["pos"] + n
    anc = _ancestors(st["parents"])
    at = pos[:, None] + anc.sum(-1) - 1                       # RoPE position [b][n]
    cos, sin = (torch.cat([t[at], t[at]], -1)[:, :, None] for t in (st["cos"], st["sin"]))
    x = st["qkv"].view(b, n, hq + 2 * hkv, D)
    rot = x[:, :, :hq + hkv]
    rot = rot * cos + torch.cat([-rot[..., D // 2:], rot[..., :D // 2]], -1) * sin
    rows = pos[:, None] + torch.arange(n, device=k.device)    # cache row [b][n]
    seq = torch.arange(b, device=k.device)[:, None]
    k[seq, :, rows] = rot[:, :, hq:]
    v[seq, :, rows] = x[:, :, hq + hkv:]
    q = rot[:, :, :hq].reshape(b, n, hkv, g, D).permute(0, 2, 1, 3, 4).reshape(b, hkv, n * g, D)
    s = torch.matmul(q, k[:, :, :L].transpose(-1, -2)) * SCALE
    j = torch.arange(L, device=k.device) - pos[:, None]       # key's node number [b][L]
    node = j.clamp(0, n - 1)[:, None, :].expand(b, n, L)
    seen = (j < 0)[:, None, :] | (torch.gather(anc, 2, node) & (j < n)[:, None, :])
    s = s.view(b, hkv, n, g, L).masked_fill(~seen[:, None, :, None, :], -math.inf)
    o = torch.matmul(_softmax(s).view(b, hkv, n * g, L), v[:, :, :L])
    st["out"].copy_(o.view(b, hkv, n, g, D).permute(0, 2, 1, 3, 4).reshape(b, n, hq, D))
    return st["out"], k, v


def _plain_weights(st):
    c, k, v, pos = st["case"], st["k"], st["v"], st["pos"].long()
    b, t, hq, hkv = c["batch"], c["t"], c["hq"], c["hkv"]
    g, L = hq // hkv, c["pos"] + t
    q = st["q"].view(b, t, hkv, g, D).permute(0, 2, 1, 3, 4).reshape(b, hkv, t * g, D)
    s = torch.matmul(q, k[:, :, :L].transpose(-1, -2)) * SCALE
    last = pos[:, None] + torch.arange(t, device=k.device)    # last key of row [b][t]
    seen = torch.arange(L, device=k.device) <= last[:, :, None]
    s = s.view(b, hkv, t, g, L).masked_fill(~seen[:, None, :, None, :], -math.inf)
    p = _softmax(s).view(b, hkv, t * g, L)
    st["weight"][:, :, :L] += p.sum(2)
    st["out"].copy_(torch.matmul(p, v[:, :, :L]).view(b, hkv, t, g, D).permute(0, 2, 1, 3, 4).reshape(b, t, hq, D))
    return st["out"], st["weight"]


def _plain_evict(st):
    c, k, v, w = st["case"], st["k"], st["v"], st["weight"]
    length = st["pos"].long()[:, None, None]
    keep, max_t = c["keep"], c["max_t"]
    j = torch.arange(max_t, device=w.device)
    key = torch.where((j < c["sink"]) | (j >= length - c["recent"]), math.inf, w)
    key = torch.where(j < length, key, -math.inf)
    index = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]
    index = torch.where(index < length, index, max_t)          # a sequence shorter than keep
    index = torch.sort(index, dim=-1).values
    there = index < max_t
    at = index.clamp(max=max_t - 1)
    rows = at[..., None].expand(*at.shape, D)
    for cache in (k, v):
        cache[:, :, :keep] = torch.where(there[..., None], torch.gather(cache, 2, rows), cache[:, :, :keep])
    st["weight_out"].zero_()
    st["weight_out"][:, :, :keep] = torch.where(there, torch.gather(w, 2, at), 0.0)
    return torch.where(there, index, -1).to(torch.int32), k, v, st["weight_out"]


def _chosen(st):
    """Blocks [b][hkv][t][topk] in ascending order, -1 behind the last; scores in 64 bits, where a tie is a tie."""
    c = st["case"]
    b, t, hkv, topk = c["batch"], c["t"], c["hkv"], c["topk"]
    q = st["q"].double().view(b, t, hkv, c["hq"] // hkv, D).sum(3).permute(0, 2, 1, 3)
    s = torch.matmul(q, st["keys"].double().transpose(-1, -2))
    nb = s.shape[-1]
    block = (st["pos"].long()[:, None] + torch.arange(t, device=q.device)) // c["block"]  # a row's own [b][t]
    past = torch.arange(nb, device=q.device) < block[:, None, :, None]
    order = torch.sort(s.masked_fill(~past, -math.inf), dim=-1, descending=True, stable=True).indices
    best = torch.full((b, hkv, t, topk), nb, dtype=torch.long, device=q.device)
    m = min(topk, nb)
    best[..., :m] = torch.where(torch.gather(past.expand_as(s), 3, order[..., :m]), order[..., :m], nb)
    best = torch.sort(best, dim=-1).values
    return torch.where(best < nb, best, -1), block


def _plain_blocks(st):
    c, k, v = st["case"], st["k"], st["v"]
    b, t, hq, hkv, B = c["batch"], c["t"], c["hq"], c["hkv"], c["block"]
    g, max_t = hq // hkv, c["max_t"]
    best, block = _chosen(st)
    mine = block[:, None, :, None].expand(b, hkv, t, 1)
    rows = (torch.cat([best, mine], -1)[..., None] * B + torch.arange(B, device=k.device)).reshape(b, hkv, t, -1)
    last = (st["pos"].long()[:, None] + torch.arange(t, device=k.device))[:, None, :, None]
    seen = (rows >= 0) & (rows <= last)
    at = rows.clamp(0, max_t - 1)
    head = (torch.arange(b * hkv, device=k.device) * max_t).view(b, hkv, 1, 1)
    kk, vv = (cache.view(-1, D)[at + head] for cache in (k, v))  # [b][hkv][t][keys][D]
    q = st["q"].view(b, t, hkv, g, D).permute(0, 2, 1, 3, 4)
    s = torch.matmul(q, kk.transpose(-1, -2)) * SCALE
    p = _softmax(s.masked_fill(~seen[..., None, :], -math.inf))
    st["out"].copy_(torch.matmul(p, vv).permute(0, 2, 1, 3, 4).reshape(b, t, hq, D))
    return st["out"], best.permute(0, 2, 1, 3).to(torch.int32).contiguous()


_plain = {"tree": _plain_tree, "weights": _plain_weights, "evict": _plain_evict, "blocks": _plain_blocks}


# -- what a pass cannot do without ----------------------------------------------------------

def work(case):
    op, hkv = case["op"], case["hkv"]
    row = 2 * D * 4  # a key and a value
    if op == "evict":
        total = 0
        for n in _positions(case, "len"):
            kept = min(n, case["keep"])
            moved = max(0, kept - case["sink"]) if n > kept else 0
            total += hkv * (4 * n + 4 * case["keep"] + 4 * case["max_t"] + 2 * row * moved)
        return {"bytes": total, "flops": 0}
    hq, pos = case["hq"], _positions(case)
    if op == "tree":
        n = case["n"]
        keys = sum(p + n for p in pos)
        io = 4 * D * case["batch"] * n * (2 * hq + 4 * hkv)
        return {"bytes": row * hkv * keys + io, "flops": sum(4 * D * hq * n * (p + 1) for p in pos)}
    t = case["t"]
    io = 4 * D * case["batch"] * t * 2 * hq
    if op == "weights":
        keys = sum(p + t for p in pos)
        return {"bytes": (row + 8) * hkv * keys + io, "flops": sum(4 * D * hq * (t * p + t * (t + 1) // 2) for p in pos)}
    B, total, flops = case["block"], io, 0
    for p in pos:
        past = p // B
        picked = min(case["topk"], past)
        keys = min(p + t, t * (picked * B + B // 2))
        total += hkv * (row * keys + 4 * D * past + 4 * t * case["topk"])
        flops += 4 * D * hq * t * (picked * B + B // 2) + 2 * D * hkv * t * past
    return {"bytes": total, "flops": flops}


# -- the definition in 64 bits --------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    k, v = st["k"].double(), st["v"].double()
    lens = [int(x) for x in st["pos"].tolist()]
    if case["op"] == "evict":
        return [None, *_exact_evict(case, st, k, v, lens)]
    hq, hkv = case["hq"], case["hkv"]
    g = hq // hkv
    scale = 1.0 / math.sqrt(D)
    out = torch.zeros_like(st["out"], dtype=torch.float64)
    if case["op"] == "tree":
        n = case["n"]
        parents = st["parents"].tolist()
        cos, sin = st["cos"].double(), st["sin"].double()
        for b, p0 in enumerate(lens):
            paths = []
            for i in range(n):
                paths.append((paths[parents[b][i]] if parents[b][i] >= 0 else []) + [i])
            x = st["qkv"][b].double().view(n, hq + 2 * hkv, D)
            at = torch.tensor([p0 + len(path) - 1 for path in paths], device=k.device)
            lo, hi = x[:, :hq + hkv, :D // 2], x[:, :hq + hkv, D // 2:]
            co, si = cos[at][:, None], sin[at][:, None]
            rot = torch.cat([lo * co - hi * si, hi * co + lo * si], -1)
            k[b, :, p0:p0 + n] = rot[:, hq:].transpose(0, 1)
            v[b, :, p0:p0 + n] = x[:, hq + hkv:].transpose(0, 1)
            seen = torch.zeros((n, p0 + n), dtype=torch.bool)
            seen[:, :p0] = True
            for i, path in enumerate(paths):
                seen[i, [p0 + a for a in path]] = True
            seen = seen.to(k.device)
            for h in range(hq):
                s = (rot[:, h] @ k[b, h // g, :p0 + n].T) * scale
                out[b, :, h] = torch.softmax(s.masked_fill(~seen, -math.inf), -1) @ v[b, h // g, :p0 + n]
        return out, k, v
    q, t = st["q"].double(), case["t"]
    if case["op"] == "weights":
        weight = st["weight"].double()
        for b, p0 in enumerate(lens):
            hidden = torch.ones((t, p0 + t), dtype=torch.bool, device=k.device).triu(p0 + 1)
            for h in range(hq):
                s = (q[b, :, h] @ k[b, h // g, :p0 + t].T) * scale
                p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
                weight[b, h // g, :p0 + t] += p.sum(0)
                out[b, :, h] = p @ v[b, h // g, :p0 + t]
        return out, weight
    B, topk = case["block"], case["topk"]
    keys = st["keys"].double()
    for b, p0 in enumerate(lens):
        at = torch.arange(p0, p0 + t, device=k.device)
        own_block = at // B
        L = p0 + t
        j = torch.arange(L, device=k.device)
        for h in range(hkv):
            nb = keys.shape[2]
            s = sum(q[b, :, h * g + e] for e in range(g)) @ keys[b, h].T
            s = s.masked_fill(torch.arange(nb, device=k.device) >= own_block[:, None], -math.inf)
            m = min(topk, nb)
            top = torch.topk(s, m, dim=-1)
            chosen = torch.zeros((t, nb), dtype=torch.bool, device=k.device)
            chosen.scatter_(1, top.indices, top.values > -math.inf)
            chosen.scatter_(1, own_block[:, None], True)
            seen = chosen[:, j // B] & (j <= at[:, None])
            for e in range(g):
                s = (q[b, :, h * g + e] @ k[b, h, :L].T) * scale
                out[b, :, h * g + e] = torch.softmax(s.masked_fill(~seen, -math.inf), -1) @ v[b, h, :L]
    return out, None


def _exact_evict(case, st, k, v, lens):
    w = st["weight"].double()
    w_out = torch.zeros_like(w)
    for b, n in enumerate(lens):
        kept = min(n, case["keep"])
        first, last = min(case["sink"], kept), max(case["sink"], n - case["recent"])
        for h in range(case["hkv"]):
            if n <= case["keep"]:
                index = list(range(n))
            else:
                row = w[b, h].tolist()
                middle = sorted(range(first, last), key=lambda i: (-row[i], i))
                index = sorted(list(range(first)) + list(range(last, n)) + middle[:kept - first - (n - last)])
            at = torch.tensor(index, device=k.device, dtype=torch.long)
            k[b, h, :kept], v[b, h, :kept] = k[b, h, at], v[b, h, at]
            w_out[b, h, :kept] = w[b, h, at]
    return k, v, w_out
