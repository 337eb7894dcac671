"""Operators behind replies that share what they have read: beams of one request, several replies to one prompt, and
requests behind one common text.

* ``attention``  decode attention of a batch whose rows hold a long stretch of positions in the same pages of the cache;
* ``select``     the best continuations of every request over its beams and the vocabulary;
* ``states``     fixed-size states of sequences copied to other slots, which go on from there;
* ``pages``      pages of keys and values copied where a sequence has to write into one that others read too.

A case is a dict of plain values; ``prepare`` makes its data on the GPU from the seed, ``run`` is one pass.  With ``own``
false ``run`` computes the plain form from elementary torch operations, with ``own`` true it calls the library.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda:0"
PAGE = 64


# ---- the cases ----------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one request with four beams over a short prompt, at the 2B sizes: a call that is all latency
        dict(name="attention-4-beams", op="attention", groups=1, rows=4, shared=448, own_from=1, own_to=40, heads=8, kv_heads=4,
             head_dim=256, cap=50.0, window=0, dtype="bfloat16"),
        # eight beams over the longest prompt of the 2B sizes, some way into the reply
        dict(name="attention-8-beams-long", op="attention", groups=1, rows=8, shared=7936, own_from=100, own_to=190, heads=8,
             kv_heads=4, head_dim=256, cap=50.0, window=0, dtype="bfloat16"),
        # sixteen requests of four beams under a window that the sequences have outgrown (a ring), at the 9B sizes
        dict(name="attention-16x4-window", op="attention", groups=16, rows=4, shared=4544, own_from=33, own_to=290, heads=16,
             kv_heads=8, head_dim=256, cap=50.0, window=4096, dtype="bfloat16"),
        # 128 requests behind one long common text, each with a text and a reply of its own, at the 27B sizes
        dict(name="attention-128-requests", op="attention", groups=1, rows=128, shared=6144, own_from=40, own_to=1500, heads=32,
             kv_heads=16, head_dim=128, cap=50.0, window=0, dtype="bfloat16"),
        # the float32 path with a small model's heads, three requests of five beams
        dict(name="attention-float32", op="attention", groups=3, rows=5, shared=960, own_from=1, own_to=77, heads=6, kv_heads=1,
             head_dim=24, cap=0.0, window=0, dtype="float32"),
        # beams of one request of a small model
        dict(name="select-4-small", op="select", requests=1, beams=4, vocab=1000, take=8),
        # eight beams of one request at the vocabulary of the 2B sizes
        dict(name="select-8", op="select", requests=1, beams=8, vocab=256000, take=16),
        # a batch of requests with an odd number of beams and an odd vocabulary
        dict(name="select-16x5", op="select", requests=16, beams=5, vocab=255029, take=10),
        # four beams of a small recurrent model, one of which goes on from another
        dict(name="states-small", op="states", slots=4, pairs=1, lines=3, heads=2, dim=16, vdim=32, conv=96),
        # half of 64 sequences go on from the other half's states: the 2B sizes' matrix memories and convolutions
        dict(name="states-32", op="states", slots=64, pairs=32, lines=4, heads=9, dim=128, vdim=256, conv=2304),
        # eight beams of the 2B sizes: three go on from others and need the page they write into
        dict(name="pages-3", op="pages", lines=13, pages=160, pairs=3, kv_heads=4, head_dim=256, dtype="bfloat16"),
        # 64 replies leave the partly filled page of their common prompt at once
        dict(name="pages-63", op="pages", lines=13, pages=400, pairs=63, kv_heads=4, head_dim=256, dtype="bfloat16"),
    ]


MOST_BYTES = 750e6          # what the largest listed cases move, and compute
MOST_FLOPS = 13e9


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["attention", "attention", "attention", "select", "select", "states", "pages"])
        if op == "attention":
            small = rng.random() < 0.2
            kv = rng.choice([1, 2]) if small else rng.choice([1, 2, 4, 8, 16])
            case = dict(op=op, groups=_log_int(rng, 1, 16), rows=_log_int(rng, 2, 128), shared=PAGE * _log_int(rng, 1, 128),
                        own_from=_log_int(rng, 1, 40), heads=kv * rng.choice([1, 2, 4, 6, 8]), kv_heads=kv,
                        head_dim=rng.choice([16, 24, 64]) if small else rng.choice([64, 128, 256]),
                        cap=rng.choice([0.0, 50.0]), window=rng.choice([0, 0, 1024, 4096]),
                        dtype="float32" if small else "bfloat16")
            case["own_to"] = case["own_from"] + _log_int(rng, 1, 1500)
            if small:
                case["rows"] = min(case["rows"], 16)
            if case["window"]:                       # what a ring still holds: the sharers differ by less than their common range
                case["own_to"] = min(case["own_to"], case["own_from"] + case["window"] // 4)
        elif op == "select":
            beams = _log_int(rng, 2, 16)
            case = dict(op=op, requests=_log_int(rng, 1, 16), beams=beams, vocab=_log_int(rng, 300, 256000), take=2 * beams)
        elif op == "states":
            slots = _log_int(rng, 2, 64)
            case = dict(op=op, slots=slots, pairs=rng.randint(1, slots // 2), lines=rng.randint(1, 8), heads=rng.randint(1, 9),
                        dim=rng.choice([16, 40, 64, 128]), vdim=rng.choice([16, 40, 128, 256]), conv=rng.randint(8, 2400))
        else:
            pairs = _log_int(rng, 1, 64)
            case = dict(op=op, lines=rng.randint(1, 26), pages=2 * pairs + 8 + rng.randint(0, 100), pairs=pairs,
                        kv_heads=rng.choice([1, 2, 4, 8]), head_dim=rng.choice([24, 64, 128, 256]),
                        dtype=rng.choice(["bfloat16", "bfloat16", "float32"]))
            if case["lines"] * case["pages"] * case["kv_heads"] * case["head_dim"] > 13 * 400 * 4 * 256:
                continue                             # the pools, not the copies, would be out of range
        w = work(case)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS:
            return case


# ---- where the keys of a case stand -------------------------------------------------------------------------------------

def _rng_of(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _lengths(case):
    """Per row: its length; per group: (begin, end) of the shared positions."""
    rng = _rng_of(case)
    lengths, ranges = [], []
    W = case["window"]
    for _ in range(case["groups"]):
        s = case["shared"]
        if case["groups"] > 1:                       # requests differ: between half and all of the common length
            s = PAGE * max(1, rng.randint((s // PAGE + 1) // 2, s // PAGE))
        ns = [s + rng.randint(case["own_from"], case["own_to"]) for _ in range(case["rows"])]
        begin = 0
        if W:                                        # a ring of W positions: pages that every row still holds
            begin = max(0, -(-(max(ns) - W) // PAGE) * PAGE)
            begin = min(begin, s)
        lengths += ns
        ranges.append((begin, s))
    return lengths, ranges


def _pages(case):
    """The page table of every row, as page ids 1.. given out in a mixed order, and how many there are."""
    lengths, ranges = _lengths(case)
    W, R = case["window"], case["rows"]
    ring_pages = W // PAGE if W else 0
    width = ring_pages or max(-(-n // PAGE) for n in lengths)
    table, taken = [], 0
    for b, n in enumerate(lengths):
        begin, end = ranges[b // R]
        row = [0] * width
        last = (n - 1) // PAGE
        for g in range(max(0, last - ring_pages + 1) if W else 0, last + 1):
            at = g % ring_pages if W else g
            if begin <= g * PAGE and (g + 1) * PAGE <= end:
                if b % R:
                    row[at] = table[b - b % R][at]
                    continue
            taken += 1
            row[at] = taken
        table.append(row)
    ids = list(range(1, taken + 1))
    _rng_of(case).shuffle(ids)
    return [[ids[p - 1] if p else 0 for p in row] for row in table], taken + 1


# ---- inputs -------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device=DEVICE)  # noqa: E731
    st = dict(case=case)
    if case["op"] == "attention":
        dt = getattr(torch, case["dtype"])
        H, K, D, R = case["heads"], case["kv_heads"], case["head_dim"], case["rows"]
        lengths, ranges = _lengths(case)
        table, n_pages = _pages(case)
        B = len(lengths)
        st["k"] = torch.empty(n_pages, K, PAGE, D, dtype=dt, device=DEVICE)
        st["v"] = torch.empty(n_pages, K, PAGE, D, dtype=dt, device=DEVICE)
        for t in (st["k"], st["v"]):
            for i in range(0, n_pages, 4096):
                t[i:i + 4096] = randn(min(4096, n_pages - i), K, PAGE, D)
        st["qkv"] = randn(B, (H + 2 * K) * D).to(dt)           # the packed rows of a step: queries, then the new keys and values
        order = list(range(B))
        random.Random(seed).shuffle(order)                     # row b lives in slot order[b]
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)  # noqa: E731
        by_slot = [0] * B
        for b, s in enumerate(order):
            by_slot[s] = b
        st["table"] = i32([table[b] for b in by_slot])
        st["slot_len"] = i32([lengths[b] for b in by_slot])
        st["slots"] = i32(order)
        st["lengths"], st["ranges"] = lengths, ranges
        if own:
            from quicknn_b200.kernels import ops
            groups = [(i * R, R, a, e) for i, (a, e) in enumerate(ranges)]
            st["shared"] = ops.SharedKeys(i32(groups), i32([b // R for b in range(B)]), rows=R, keys=max(e - a for a, e in ranges),
                                          own=max(n - (e - a) for n, (a, e) in zip(lengths, (ranges[b // R] for b in range(B)))))
            st["plan"] = ops.shared_attention_plan(st["qkv"].dtype, B, H, K, D, st["shared"], case["window"])
            st["scratch"] = torch.empty(st["plan"].scratch_bytes, dtype=torch.uint8, device=DEVICE)
    elif case["op"] == "select":
        rows, V = case["requests"] * case["beams"], case["vocab"]
        x = 4.0 * randn(rows, V)
        x += 10.0 * (torch.rand(rows, V, generator=g, device=DEVICE) < 20.0 / V)    # a few words that fit well
        st["logits"] = 30.0 * torch.tanh(x / 30.0)
        s = -20.0 * torch.rand(case["requests"], case["beams"], generator=g, device=DEVICE)
        st["scores"] = s.sort(dim=1, descending=True).values.reshape(-1).contiguous()
        if own:
            from quicknn_b200.kernels import ops
            st["scratch"] = torch.empty(ops.beam_select_scratch_bytes(rows, V, case["take"]), dtype=torch.uint8, device=DEVICE)
    elif case["op"] == "states":
        n = case["slots"]
        st["tensors"] = ([randn(n, case["heads"], case["dim"], case["vdim"]) for _ in range(case["lines"])]
                         + [randn(n, 3, case["conv"]).to(torch.bfloat16) for _ in range(case["lines"])])
        ids = list(range(n))
        random.Random(seed).shuffle(ids)
        p = case["pairs"]
        st["dst"] = ids[:p]                                    # sequences that end, and those that go on twice or more
        st["src"] = [ids[p + random.Random(seed + i).randrange(n - p)] for i in range(p)]
    else:
        dt = getattr(torch, case["dtype"])
        shape = (case["lines"], case["pages"], case["kv_heads"], PAGE, case["head_dim"])
        st["k"], st["v"] = randn(*shape).to(dt), randn(*shape).to(dt)
        r = random.Random(seed)
        ids = list(range(1, case["pages"]))
        r.shuffle(ids)
        p = case["pairs"]
        st["dst"] = ids[:p]
        st["src"] = [r.choice(ids[p:]) for _ in range(p)]
        st["used"] = [r.randint(1, PAGE - 1) for _ in range(p)]
    return st


# ---- one pass -----------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if case["op"] == "attention":
        return _attention_own(state) if own else _attention_plain(state)
    if case["op"] == "select":
        return _select_own(state) if own else _select_plain(state)
    if case["op"] == "states":
        if own:
            from quicknn_b200.kernels import ops
            ops.copy_slots(state["tensors"], state["src"], state["dst"])
        else:
            src, dst = torch.tensor(state["src"], device=DEVICE), torch.tensor(state["dst"], device=DEVICE)
            for t in state["tensors"]:
                t[dst] = t[src]
        return state["tensors"]
    if own:
        from quicknn_b200.kernels import ops
        ops.copy_pages(state["k"], state["v"], state["src"], state["dst"], state["used"])
    else:
        for t in (state["k"], state["v"]):
            for s, d, u in zip(state["src"], state["dst"], state["used"]):
                t[:, d, :, :u] = t[:, s, :, :u]
    return [state["k"], state["v"]]


def _attention_own(st):
    from quicknn_b200.kernels import ops
    c = st["case"]
    return ops.attn_decode_shared(st["qkv"], c["heads"], c["kv_heads"], c["head_dim"], st["k"], st["v"], st["table"], PAGE,
                                  c["window"], st["slots"], st["slot_len"], st["shared"], c["head_dim"] ** -0.5, c["cap"] or None,
                                  c["window"] or None, st["plan"], st["scratch"])


def _gather(pool, table, positions, window):
    """Rows of a pool [pages, kv heads, PAGE, head size] at positions of sequences with these page tables."""
    at = positions % window if window else positions
    page = torch.gather(table.long(), 1, at // PAGE) if table.dim() == 2 else table.long()[at // PAGE]
    return pool.transpose(1, 2)[page, at % PAGE].float()       # [..., kv heads, head size]


def _attention_plain(st):
    c = st["case"]
    H, K, D, R, W = c["heads"], c["kv_heads"], c["head_dim"], c["rows"], c["window"]
    B = len(st["lengths"])
    q = st["qkv"][:, :H * D].float().view(B, K, H // K, D)
    out = torch.empty(B, H * D, dtype=st["qkv"].dtype, device=DEVICE)
    for i, (begin, end) in enumerate(st["ranges"]):
        rows = slice(i * R, (i + 1) * R)
        slots = st["slots"][rows].long()
        table, n = st["table"][slots], st["slot_len"][slots].long()
        first = (n - W).clamp(min=0) if W else torch.zeros_like(n)
        # the keys that all rows hold in the same pages, once; then every row's others
        common = torch.arange(begin, end, device=DEVICE)
        kc, vc = _gather(st["k"], table[0], common, W), _gather(st["v"], table[0], common, W)
        before = (begin - first).clamp(min=0)
        most = max(st["lengths"][rows]) - end + max(max(0, begin - max(0, m - W)) if W else 0 for m in st["lengths"][rows])
        j = torch.arange(most, device=DEVICE)[None, :]
        place = torch.where(j < before[:, None], first[:, None] + j, end + j - before[:, None])
        inside = place < n[:, None]
        place = torch.where(inside, place, end)
        ko, vo = _gather(st["k"], table, place, W), _gather(st["v"], table, place, W)
        s = torch.cat([torch.einsum("rkgd,skd->rkgs", q[rows], kc), torch.einsum("rkgd,rskd->rkgs", q[rows], ko)], dim=-1) * D ** -0.5
        if c["cap"]:
            s = c["cap"] * torch.tanh(s / c["cap"])
        seen = torch.cat([(common[None, :] >= first[:, None]) & (common[None, :] < n[:, None]), inside], dim=-1)
        s = torch.where(seen[:, None, None, :], s, float("-inf"))
        w = torch.exp(s - s.amax(dim=-1, keepdim=True))
        w = w / w.sum(dim=-1, keepdim=True)
        m = end - begin
        o = torch.einsum("rkgs,skd->rkgd", w[..., :m], vc) + torch.einsum("rkgs,rskd->rkgd", w[..., m:], vo)
        out[rows] = o.reshape(R, H * D).to(out.dtype)
    return out


def _select_own(st):
    from quicknn_b200.kernels import ops
    c = st["case"]
    return ops.beam_select(st["logits"], st["scores"], c["beams"], c["take"], st["scratch"])


def _select_plain(st):
    c = st["case"]
    # in 64 bits: sums over the vocabulary decide between beams whose candidates stand next to each other
    x = st["logits"].double()
    m = x.amax(dim=1, keepdim=True)
    logp = x - m - torch.log(torch.exp(x - m).sum(dim=1, keepdim=True))
    total = (st["scores"].double()[:, None] + logp).view(c["requests"], -1)
    best, flat = torch.sort(total, dim=1, descending=True, stable=True)
    best, flat = best[:, :c["take"]], flat[:, :c["take"]]
    return best.float(), (flat // c["vocab"]).int(), (flat % c["vocab"]).int()


# ---- what a pass cannot do without --------------------------------------------------------------------------------------

def work(case):
    if case["op"] == "attention":
        size = 4 if case["dtype"] == "float32" else 2
        H, K, D, W = case["heads"], case["kv_heads"], case["head_dim"], case["window"]
        lengths, ranges = _lengths(case)
        keys = seen = 0
        for i, (begin, end) in enumerate(ranges):
            ns = lengths[i * case["rows"]:(i + 1) * case["rows"]]
            firsts = [max(0, n - W) if W else 0 for n in ns]
            keys += end - max(begin, min(firsts))              # each shared key once
            for n, f in zip(ns, firsts):
                keys += n - f - (end - max(begin, min(f, end)))
                seen += n - f
        return {"bytes": size * (2 * keys * K * D + 2 * len(lengths) * H * D), "flops": 4 * seen * H * D}
    if case["op"] == "select":
        rows = case["requests"] * case["beams"]
        return {"bytes": 4 * rows * (case["vocab"] + 1) + 12 * case["requests"] * case["take"], "flops": 3 * rows * case["vocab"]}
    if case["op"] == "states":
        per = case["lines"] * (4 * case["heads"] * case["dim"] * case["vdim"] + 2 * 3 * case["conv"])
        return {"bytes": 2 * case["pairs"] * per, "flops": 0}
    size = 4 if case["dtype"] == "float32" else 2              # a page is half full on the average
    return {"bytes": 2 * 2 * case["pairs"] * case["lines"] * case["kv_heads"] * (PAGE // 2) * case["head_dim"] * size, "flops": 0}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] in ("states", "pages"):
        return None                                            # copies: nothing is computed
    st = prepare(case, seed)
    if case["op"] == "select":
        x = st["logits"].double()
        lse = torch.logsumexp(x, dim=1)
        tot = st["scores"].double() + x.T - lse                # [vocab, rows]
        best, parents, tokens = [], [], []
        V, W = case["vocab"], case["beams"]
        for r in range(case["requests"]):
            flat = tot[:, r * W:(r + 1) * W].T.reshape(-1)
            vals, ids = torch.topk(flat, min(case["take"] + 64, flat.numel()))
            pick = sorted(zip((-vals).tolist(), ids.tolist()))[:case["take"]]
            best.append([-v for v, _ in pick])
            parents.append([i // V for _, i in pick])
            tokens.append([i % V for _, i in pick])
        f = lambda v, t: torch.tensor(v, dtype=t, device=DEVICE)  # noqa: E731
        return f(best, torch.float64), f(parents, torch.int32), f(tokens, torch.int32)
    H, K, D, W, cap = case["heads"], case["kv_heads"], case["head_dim"], case["window"], case["cap"]
    out = torch.empty(len(st["lengths"]), H * D, dtype=torch.float64, device=DEVICE)
    for b, n in enumerate(st["lengths"]):
        slot = int(st["slots"][b])
        pos = torch.arange(max(0, n - W) if W else 0, n, device=DEVICE)
        cell = pos % W if W else pos
        page = st["table"][slot].long()[torch.div(cell, PAGE, rounding_mode="floor")]
        k = st["k"][page, :, cell % PAGE].double()             # [keys, kv heads, head size]
        v = st["v"][page, :, cell % PAGE].double()
        q = st["qkv"][b, :H * D].double().view(H, D)
        for h in range(K):
            mine = slice(h * (H // K), (h + 1) * (H // K))
            s = (q[mine] @ k[:, h].T) / math.sqrt(D)
            if cap:
                s = torch.tanh(s / cap) * cap
            out[b].view(H, D)[mine] = torch.softmax(s, dim=1) @ v[:, h]
    return out
