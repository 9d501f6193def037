"""The operators of a cache bounded by what is attended to, on their own: attention that adds up the weight each cached key
receives, the choice of the keys that a request keeps, and the moves that close the gaps.

A case is one call.  The sizes are those of the engine's own models (32 or 16 query heads over 8 KV heads of 128, pages of 256;
small models with pages of 8 and 16) and of what it serves: chat turns, batches of decoded tokens, long documents.

``run`` computes the formulas with elementary torch operations in 32 bits, or, where ``own`` is set, calls the engine's kernels.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
KEEP_FIRST = 4          # the first keys of a request, which every later token leans on


# ------------------------------------------------------------------------------------------------ the cases
def _attend(name, seqs, new, kv, heads, kv_heads, dim, page, dtype="bf16", cap=0.0, sinks=False, lens=0):
    return {"name": name, "op": "attend", "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "kv_lo": kv[0], "kv_hi": kv[1],
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "cap": cap, "sinks": sinks, "lens": lens}


def _evict(name, op, seqs, kv, budget, recent, kv_heads, dim, page, dtype="bf16", lens=0):
    return {"name": name, "op": op, "seqs": seqs, "kv_lo": kv[0], "kv_hi": kv[1], "budget": budget, "recent": recent,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "lens": lens}


def listed():
    return [
        # one token of one chat on the 0.6B-shaped model: latency is all there is
        _attend("attend_chat_1", 1, (1, 1), (517, 517), 16, 8, 128, 256),
        # a decode step of 64 requests on the 8B-shaped model, each held to about two thousand keys
        _attend("attend_decode_64", 64, (1, 1), (1200, 2304), 32, 8, 128, 256, lens=1),
        # three requests over long documents that have not been cut yet, eight query heads a KV head (32B-shaped)
        _attend("attend_decode_long", 3, (1, 1), (65000, 98304), 64, 8, 128, 256, lens=2),
        # drafted tokens being checked: five new tokens a request
        _attend("attend_drafts_12", 12, (5, 5), (2900, 9000), 32, 8, 128, 256, lens=3),
        # a whole prompt of 2,048 tokens
        _attend("attend_prompt_2048", 1, (2048, 2048), (2048, 2048), 32, 8, 128, 256),
        # a portion of 1,024 tokens behind 16 thousand cached ones
        _attend("attend_portion_17k", 1, (1024, 1024), (17407, 17407), 32, 8, 128, 256),
        # prompt portions beside single tokens on a small model: heads of 64 in groups of three, small pages, capped scores, sinks
        _attend("attend_mixed_capped", 20, (1, 200), (200, 1500), 24, 8, 64, 16, cap=30.0, sinks=True, lens=4),
        # the 32-bit path: prompts of some hundred tokens
        _attend("attend_float32", 5, (90, 400), (400, 777), 16, 8, 128, 64, dtype="f32", lens=5),
        # 64 decoding requests that are each a page over their budget: which keys go, and the moves
        _evict("choose_page_64", "choose", 64, (2304, 2304), 2048, 512, 8, 128, 256),
        _evict("move_page_64", "move", 64, (2304, 2304), 2048, 512, 8, 128, 256),
        # eight long prompts just read, each cut down to 4,096 keys
        _evict("choose_prompt_8", "choose", 8, (20000, 40000), 4096, 1024, 8, 128, 256, lens=6),
        _evict("move_prompt_8", "move", 8, (20000, 40000), 4096, 1024, 8, 128, 256, lens=6),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    if rng.random() < 0.4:
        op = rng.choice(("choose", "move"))
        kv_heads, dim, page = rng.choice((1, 2, 4, 8, 8)), rng.choice((32, 64, 96, 128, 128)), rng.choice((8, 16, 64, 256))
        hi = _log(rng, 200, 40000)
        budget = max(16, int(hi * rng.uniform(0.1, 0.95)))
        seqs = min(_log(rng, 1, 64), max(1, 150000 * 8 // (hi * kv_heads)))
        return _drawn(_evict("", op, seqs, (max(1, int(hi * rng.uniform(0.3, 1.0))), hi), budget, max(1, int(budget * rng.uniform(0.02, 0.6))),
                             kv_heads, dim, page, rng.choice(("bf16", "bf16", "bf16", "f32")), rng.randrange(1 << 20)))
    kv_heads = rng.choice((1, 2, 4, 8, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 4, 6, 8))
    dim, page = rng.choice((32, 64, 64, 80, 96, 128, 128, 128, 256)), rng.choice((8, 16, 32, 64, 256, 256))
    dtype = rng.choice(("bf16", "bf16", "bf16", "f32"))
    one = rng.random() < 0.4
    hi = _log(rng, 33, 65536 if one else 16384)
    new = 1 if one else min(_log(rng, 2, 2048), hi)
    # no dearer than the largest listed case: pairs of a query row and a key, and keys of the cache
    seqs = _log(rng, 1, 64)
    pairs, keys = (1 << 26 if dtype == "f32" else 1 << 28), 1 << 28
    while seqs > 1 and (seqs * new * heads * hi > pairs or seqs * hi * kv_heads * dim > keys):
        seqs //= 2
    while new > 2 and seqs * new * heads * hi > pairs:
        new //= 2
    while hi > max(new, 64) and seqs * new * heads * hi > pairs:
        hi = max(new, hi // 2)
    lo = new if rng.random() < 0.5 else max(1, new // 4)
    return _drawn(_attend("", seqs, (lo, new), (max(new, int(hi * rng.uniform(0.3, 1.0))), hi), heads, kv_heads, dim, page, dtype,
                          rng.choice((0.0, 0.0, 30.0)), rng.random() < 0.3, rng.randrange(1 << 20)))


def _drawn(case):
    del case["name"]
    return case


def _lengths(case):
    """Per request: new tokens and keys in the cache with them.  They belong to the case, not to the seed."""
    rng = random.Random(case["lens"])
    kv = [rng.randint(case["kv_lo"], case["kv_hi"]) for _ in range(case["seqs"])]
    if case["op"] != "attend":
        return [0] * len(kv), kv
    return [min(k, rng.randint(case["new_lo"], case["new_hi"])) for k in kv], kv


def work(case):
    new, kv = _lengths(case)
    item = 2 if case["dtype"] == "bf16" else 4
    h, d = case["kv_heads"], case["dim"]
    if case["op"] == "attend":
        rows = sum(new) * case["heads"] * d
        pairs = sum(n * k - n * (n - 1) // 2 for n, k in zip(new, kv)) * case["heads"]
        keys = sum(kv) * h
        # q and the output; keys and values; old scores in, new ones out; births of the new keys
        return {"bytes": 2 * rows * item + 2 * keys * d * item + 4 * (2 * keys - sum(new) * h) + 4 * sum(new) * h, "flops": 4 * d * pairs}
    moves = sum(_expected_moves(k, case["budget"], case["recent"]) for k in kv) * h
    if case["op"] == "choose":
        return {"bytes": 8 * sum(kv) * h + 8 * moves, "flops": 2 * sum(kv) * h}
    return {"bytes": moves * (4 * d * item + 16 + 8), "flops": 0}


def _expected_moves(kv, budget, recent):
    """Kept keys at or above the budget when scores are in no order: all recent ones there, and a fair share of the others."""
    if kv <= budget:
        return 0
    recent, tail = min(recent, kv), kv - budget
    late = min(recent, tail)
    others = tail - late
    return late + int(others * max(0, budget - recent) / max(1, kv - recent))


# ------------------------------------------------------------------------------------------------ what a program has in hand
def _tables(kv, page, rng):
    """A block table per request over pages in no order, -1 behind a request's last page; and how many pages there are."""
    counts = [-(-k // page) for k in kv]
    n_pages = sum(counts) + 3
    ids = list(range(n_pages))
    rng.shuffle(ids)
    table, at = np.full((len(kv), max(counts)), -1, dtype=np.int32), 0
    for s, c in enumerate(counts):
        table[s, :c] = ids[at:at + c]
        at += c
    return torch.from_numpy(table).cuda(), n_pages


def prepare(case, seed):
    rng, gen = random.Random(seed), torch.Generator(device="cuda")
    gen.manual_seed(seed)
    new, kv = _lengths(case)
    dt, h, d, page = DTYPES[case["dtype"]], case["kv_heads"], case["dim"], case["page"]
    table, n_pages = _tables(kv, page, rng)
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)      # noqa: E731
    pages = None
    if case["op"] != "choose":                                  # the choice looks at scores alone
        pages = torch.empty((n_pages, 2, h, page, d), dtype=dt, device="cuda")
        for p in range(0, n_pages, 256):
            pages[p:p + 256] = normal(*pages[p:p + 256].shape)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")      # noqa: E731
    # what keys have gathered so far: most next to nothing, a few a great deal, and some exactly nothing
    scores = normal(n_pages, h, page).mul_(1.5).exp_()
    scores[torch.rand(scores.shape, generator=gen, device="cuda") < 0.1] = 0.0
    if case["op"] == "attend":                                  # about what this step adds, so that both count in the sum
        scores *= sum(new) * case["heads"] / (h * sum(kv))
    state = {"case": case, "pages": pages, "scores": scores, "table": table, "kv_len": ints(kv), "kv": kv, "new": new}
    if case["op"] == "attend":
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        gone = [rng.randrange(0, 5000) for _ in kv]             # keys that were dropped before this step
        positions = [g + k - n + t for g, k, n in zip(gone, kv, new) for t in range(n)]
        state |= {"q": (normal(cu[-1], case["heads"] * d) * 1.5).to(dt), "cu_q": ints(cu), "positions": ints(positions),
                  "births": torch.zeros((n_pages, h, page), dtype=torch.int32, device="cuda"),
                  "scores_out": torch.zeros_like(scores),
                  "sinks": normal(case["heads"]) if case["sinks"] else None}
        return state
    # births: slots in order of arrival, as after a prompt; some early positions are already gone
    gone = 1000
    slots = torch.arange(table.shape[1] * page, device="cuda", dtype=torch.int32)
    births = torch.zeros((n_pages, h, page), dtype=torch.int32, device="cuda")
    at = torch.where(slots < KEEP_FIRST, slots, slots + gone)
    index = table.clamp(min=0).long()
    ok = (table >= 0)
    values = at.view(1, -1, 1, page).expand(len(kv), -1, h, -1)
    births[index[ok]] = values[ok]
    seen = [k + gone for k in kv]
    state |= {"births": births, "seen": ints(seen), "budgets": ints([case["budget"]] * len(kv)),
              "max_moves": max(1, min(case["budget"], max(kv) - case["budget"]))}
    if case["op"] == "move":
        state["sources"], state["targets"] = _choose(state)     # a program has them from the call before
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"attend": _attend_own, "choose": _choose_own, "move": _move_own}[op](state)
    if op == "attend":
        return _attend_plain(state)
    if op == "choose":
        sources, targets = _choose(state)
        return {"sources": sources, "targets": targets}
    return _move(state)


def _attend_own(state):
    from nanohybrid_vlm_b200.kernels import ops
    c = state["case"]
    out = torch.empty_like(state["q"])
    ops.attention_scored(out, state["q"], state["pages"], state["scores"], state["table"], state["cu_q"], state["kv_len"], c["seqs"],
                         min(state["new"]), max(state["new"]), max(state["kv"]), c["heads"], c["kv_heads"], c["dim"], c["dim"] ** -0.5,
                         births=state["births"], positions=state["positions"], sinks=state["sinks"], softcap=c["cap"] or None,
                         scores_out=state["scores_out"])
    return {"out": out, "scores": state["scores_out"], "births": state["births"]}


def _choose_own(state):
    from nanohybrid_vlm_b200.kernels import ops
    c = state["case"]
    sources = torch.empty((c["seqs"], c["kv_heads"], state["max_moves"]), dtype=torch.int32, device="cuda")
    targets = torch.empty_like(sources)
    ops.select_keys(sources, targets, state["scores"], state["births"], state["table"], state["kv_len"], state["seen"], state["budgets"],
                    c["seqs"], max(state["kv"]), KEEP_FIRST, c["recent"])
    return {"sources": sources, "targets": targets}


def _move_own(state):
    from nanohybrid_vlm_b200.kernels import ops
    ops.move_keys(state["pages"], state["scores"], state["births"], state["table"], state["sources"], state["targets"], state["case"]["seqs"])
    return {"pages": state["pages"], "scores": state["scores"], "births": state["births"]}


def _slots(state):
    """Per request and slot: its page, its place in the page, and whether the request has such a key."""
    page, table = state["case"]["page"], state["table"]
    slot = torch.arange(max(state["kv"]), device="cuda")
    where = table.clamp(min=0).long()[:, slot // page]
    return where, (slot % page).expand_as(where), slot[None] < state["kv_len"][:, None]


def _attend_plain(state):
    c, q, table = state["case"], state["q"], state["table"]
    S, H, G, d = c["seqs"], c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    where, offset, there = _slots(state)
    L, n = where.shape[1], max(state["new"])
    k = state["pages"][:, 0][where, :, offset].float().permute(0, 2, 3, 1)               # [S, H, d, L]
    v = state["pages"][:, 1][where, :, offset].float().permute(0, 2, 1, 3)               # [S, H, L, d]
    start, count = state["cu_q"][:-1].long(), (state["cu_q"][1:] - state["cu_q"][:-1]).long()
    t = torch.arange(n, device="cuda")
    real = t[None] < count[:, None]                                                      # [S, n]
    row = (start[:, None] + t[None]).clamp(max=q.shape[0] - 1)
    x = q[row].float().view(S, n, H, G, d).permute(0, 2, 3, 1, 4).reshape(S, H, G * n, d)
    s = (x @ k).view(S, H, G, n, L) * d ** -0.5
    if c["cap"]:
        s = torch.tanh(s / c["cap"]) * c["cap"]
    last = state["kv_len"].long()[:, None] - count[:, None] + t[None]                    # the newest key that a token sees
    seen = (torch.arange(L, device="cuda")[None, None] <= last[..., None]) & there[:, None] & real[..., None]
    s = s.masked_fill(~seen[:, None, None], -torch.inf)
    top = s.amax(-1, keepdim=True)
    if state["sinks"] is not None:
        sink = state["sinks"].view(1, H, G, 1, 1)
        top = torch.maximum(top, sink)
    top = torch.where(top == -torch.inf, 0.0, top)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    if state["sinks"] is not None:
        total = total + torch.exp(sink - top)
    p = p / torch.where(total == 0, 1.0, total)
    o = (p.view(S, H, G * n, L) @ v).view(S, H, G, n, d).permute(0, 3, 1, 2, 4).reshape(S, n, H * G * d)
    out = o[real].to(q.dtype)
    first_new = (state["kv_len"].long() - count)[:, None]
    slot = torch.arange(L, device="cuda")[None]
    old = torch.where((slot < first_new)[..., None], state["scores"][where, :, offset], 0.0)
    state["scores_out"][where[there], :, offset[there]] = (old + p.sum((2, 3)).permute(0, 2, 1))[there]
    fresh = there & (slot >= first_new)
    state["births"][where[fresh], :, offset[fresh]] = state["positions"][:, None].expand(-1, H)
    return {"out": out, "scores": state["scores_out"], "births": state["births"]}


def _choose(state):
    c, M = state["case"], state["max_moves"]
    where, offset, there = _slots(state)
    births = state["births"][where, :, offset].permute(0, 2, 1)                          # [S, H, L]
    scores = state["scores"][where, :, offset].permute(0, 2, 1)
    held = (births < KEEP_FIRST) | (births >= (state["seen"] - c["recent"])[:, None, None])
    scores = torch.where(held, torch.inf, scores).masked_fill(~there[:, None], -torch.inf)
    order = torch.sort(scores, dim=-1, descending=True, stable=True).indices             # ties: the lowest slot first
    slot = torch.arange(where.shape[1], device="cuda").expand_as(order)
    rank = torch.empty_like(order).scatter_(-1, order, slot)
    budget = state["budgets"].long()[:, None, None]
    kept = (rank < budget) & there[:, None]
    low = slot < budget

    def packed(mask):                                                                    # the mask's slots in order, then -1
        out = torch.full((*mask.shape[:-1], mask.shape[-1] + 1), -1, dtype=torch.int32, device="cuda")
        place = torch.where(mask, mask.cumsum(-1) - 1, mask.shape[-1])
        return out.scatter_(-1, place, torch.where(mask, slot, -1).int())[..., :-1]

    sources = packed(kept & ~low)
    targets = packed(~kept & low & there[:, None])
    # a request within its budget drops nothing; M places are enough for the others
    targets = torch.where(sources >= 0, targets, -1)
    fill = max(0, M - sources.shape[-1])
    sources, targets = (torch.nn.functional.pad(x, (0, fill), value=-1)[..., :M].contiguous() for x in (sources, targets))
    return sources, targets


def _move(state):
    c, table = state["case"], state["table"]
    request, head, i = torch.nonzero(state["sources"] >= 0, as_tuple=True)
    source, target = state["sources"][request, head, i].long(), state["targets"][request, head, i].long()
    a, b = table[request, source // c["page"]].long(), table[request, target // c["page"]].long()
    x, y = source % c["page"], target % c["page"]
    state["pages"][b, :, head, y] = state["pages"][a, :, head, x]
    state["scores"][b, head, y] = state["scores"][a, head, x]
    state["births"][b, head, y] = state["births"][a, head, x]
    return {"pages": state["pages"], "scores": state["scores"], "births": state["births"]}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The definitions in 64 bits, a request and a KV head at a time."""
    state = prepare(case, seed)
    new, kv = state["new"], state["kv"]
    page, d, H = case["page"], case["dim"], case["kv_heads"]
    pages, table = state["pages"], state["table"].cpu().tolist()
    if case["op"] == "choose":
        return None                                             # whole numbers: nothing to compute in 64 bits
    if case["op"] == "move":
        # copies: the values themselves, moved one head of one request at a time
        kv_rows, scores = pages.clone(), state["scores"].double()
        for s in range(len(kv)):
            for g in range(H):
                src, dst = state["sources"][s, g], state["targets"][s, g]
                src, dst = src[src >= 0].long(), dst[dst >= 0].long()
                at = lambda z: (state["table"][s].long()[z // page], z % page)      # noqa: E731
                (pa, xa), (pb, xb) = at(src), at(dst)
                kv_rows[pb, 0, g, xb] = pages[pa, 0, g, xa]
                kv_rows[pb, 1, g, xb] = pages[pa, 1, g, xa]
                scores[pb, g, xb] = state["scores"][pa, g, xa].double()
        return {"pages": kv_rows.double(), "scores": scores, "births": None}
    G = case["heads"] // H
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    scores_out = torch.zeros(state["scores"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for s, (n, L) in enumerate(zip(new, kv)):
        used = table[s][:-(-L // page)]
        old = state["scores"][used].permute(1, 0, 2).reshape(H, -1)[:, :L].double()
        for g in range(H):
            k = pages[used, 0, g].reshape(-1, d)[:L].double()
            v = pages[used, 1, g].reshape(-1, d)[:L].double()
            gained = old[g].clone()
            gained[L - n:] = 0
            for r in range(G):
                head = g * G + r
                x = state["q"][first:first + n, head * d:(head + 1) * d].double()
                z = x @ k.T / math.sqrt(d)
                if case["cap"]:
                    z = case["cap"] * torch.tanh(z / case["cap"])
                ahead = torch.ones(n, L, dtype=torch.bool, device="cuda").triu(L - n + 1)
                z[ahead] = -torch.inf
                norm = torch.logsumexp(z, 1, keepdim=True)
                if state["sinks"] is not None:
                    norm = torch.logaddexp(norm, state["sinks"][head].double())
                w = torch.exp(z - norm)
                out[first:first + n, head * d:(head + 1) * d] = w @ v
                gained += w.sum(0)
            full = torch.zeros(len(used) * page, dtype=torch.float64, device="cuda")
            full[:L] = gained
            scores_out[used, g] = full.view(-1, page)
        first += n
    return {"out": out, "scores": scores_out, "births": None}
