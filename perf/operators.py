"""Cases over which the paged-cache operators are measured: building the tables of a serving step, storing its keys and
values, and attention of a batch whose requests share a long prefix.

``run`` computes a case in its plain form (elementary torch operations, 32-bit arithmetic) or, with ``own`` set, through
the library's entry points; ``exact`` computes it from the definition in 64 bits."""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one decoding step of a handful of requests: latency
        {"name": "plan_step_8", "op": "plan", "B": 8, "P": 16, "width": 64, "prompt": 0},
        # a large step: decoding, prompts in chunks, finished requests
        {"name": "plan_step_1000", "op": "plan", "B": 1000, "P": 32, "width": 128, "prompt": 64},
        # admission of a whole queue of prompts
        {"name": "plan_admit_4096", "op": "plan", "B": 4096, "P": 16, "width": 256, "prompt": 250},
        # the new tokens of one decoding step
        {"name": "write_step_16", "op": "write", "T": 16, "Hkv": 8, "D": 128, "P": 16, "dtype": "bf16", "layout": "hnd"},
        # a chunk of a prompt, token-major pages, some rows are padding
        {"name": "write_chunk_2000", "op": "write", "T": 2000, "Hkv": 8, "D": 128, "P": 32, "dtype": "fp16", "layout": "nhd"},
        # the prompts of many requests at once
        {"name": "write_prompt_65536", "op": "write", "T": 65536, "Hkv": 8, "D": 128, "P": 64, "dtype": "fp16", "layout": "hnd"},
        # one request decoding behind a short system prompt: latency
        attend("decode_1", 1, 1, 32, 8, 128, 16, 512, 33, "fp16"),
        # chat: a batch behind one system prompt
        attend("decode_32", 32, 1, 32, 8, 128, 32, 4096, 1024, "bf16"),
        # many questions about one long document
        attend("decode_128_long", 128, 1, 64, 8, 128, 64, 32768, 2048, "fp16"),
        # a small model without shared heads; nothing a multiple of anything, token-major pages
        attend("decode_17_odd", 17, 1, 16, 16, 64, 16, 1001, 333, "fp16", "nhd"),
        # verification of drafted tokens, wide heads
        attend("verify_48", 48, 5, 16, 4, 256, 16, 2048, 500, "bf16"),
        # requests' own prompts, up to 1000 tokens each, behind a shared document
        attend("extend_8", 8, 1000, 32, 8, 128, 128, 8192, 2000, "bf16"),
    ]


def attend(name, B, n, Hq, Hkv, D, P, prefix, own_keys, dtype, layout="hnd"):
    """n: new tokens per request (1 .. n spread over the batch); own_keys: the longest request's keys behind the prefix,
    its new ones among them."""
    return {"name": name, "op": "attend", "B": B, "n": n, "Hq": Hq, "Hkv": Hkv, "D": D, "P": P, "prefix": prefix,
            "own_keys": own_keys, "dtype": dtype, "layout": layout}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "write", "attend", "attend"])
    if op == "plan":
        return {"op": op, "B": _log(rng, 1, 4096), "P": rng.choice([16, 32, 64, 128]), "width": rng.randint(40, 256),
                "prompt": rng.choice([0, 0, _log(rng, 2, 250)])}
    if op == "write":
        Hkv, D = rng.choice([1, 2, 3, 8, 16]), rng.choice([64, 128, 256])
        return {"op": op, "T": _log(rng, 1, 67108864 // (Hkv * D) // 2), "Hkv": Hkv, "D": D, "P": rng.choice([16, 32, 64, 128, 256]),
                "dtype": rng.choice(["fp16", "bf16"]), "layout": rng.choice(["hnd", "nhd"])}
    Hkv, g, D = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8, 16]), rng.choice([64, 128, 128, 256])
    if rng.random() < 0.7:  # single tokens, or a few drafted ones
        B, n = _log(rng, 1, 160), rng.choice([1, 1, 1, rng.randint(2, 8)])
    else:
        B, n = _log(rng, 1, 8), _log(rng, 16, 700)
    rows = B * ((n + 1) // 2 if n > 1 else 1) * g * Hkv * D
    prefix = _log(rng, 1, max(64, min(50000, 34359738368 // (2 * rows), 67108864 // (Hkv * D))))
    own_keys = n + _log(rng, 1, max(16, min(2048, 67108864 // (B * Hkv * D))))
    return {"op": op, "B": B, "n": n, "Hq": Hkv * g, "Hkv": Hkv, "D": D, "P": rng.choice([16, 16, 32, 64, 128]),
            "prefix": prefix, "own_keys": own_keys, "dtype": rng.choice(["fp16", "bf16"]), "layout": rng.choice(["hnd", "nhd"])}


# --------------------------------------------------------------------------------------------- inputs

def _spread(lo, hi, count, rng):
    """count whole numbers spread evenly over [lo, hi], in an order of the seed's: their sum does not depend on it."""
    v = [hi if count == 1 else lo + (hi - lo) * i // (count - 1) for i in range(count)]
    rng.shuffle(v)
    return v


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _plan_lengths(case, rng):
    """(keys held, keys added) of every request; nothing exceeds the table."""
    B, room = case["B"], case["P"] * case["width"]
    held = _spread(1, room - max(case["prompt"], 1), B, rng)
    new = []
    kinds = [(i % 16, 1 + (max(case["prompt"], 1) - 1) * i // B) for i in range(B)]
    rng.shuffle(kinds)
    for b, (kind, prompt) in enumerate(kinds):  # of 16 requests: one is finished, one idle, one drops drafted tokens, three bring prompts
        if kind == 15:
            new.append(-held[b])
        elif kind == 14:
            new.append(0)
        elif kind == 13:
            new.append(-min(held[b], 3))
        else:
            new.append(prompt if kind in (1, 5, 9) else 1)
    return held, new


def _cache(case, n_pages, gen):
    shape = (n_pages, case["Hkv"], case["P"], case["D"])
    if case["layout"] == "nhd":
        shape = (shape[0], shape[2], shape[1], shape[3])
    made = [torch.randn(shape, dtype=DTYPES[case["dtype"]], device="cuda", generator=gen) for _ in range(2)]
    return [t.permute(0, 2, 1, 3) if case["layout"] == "nhd" else t for t in made]


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    P = case["P"]
    if case["op"] == "plan":
        held, new = _plan_lengths(case, rng)
        pages = [-(-h // P) for h in held]
        tokens = sum(max(n, 0) for n in new)
        s["max_tokens"] = -(-max(tokens, 1) // 64) * 64  # the step's token buffers are padded
        free = min(sum(-(-(h + max(n, 0)) // P) - p for h, n, p in zip(held, new, pages)) + 5, case["B"] * case["width"] + 5 - sum(pages))
        pool = case["B"] * case["width"] + 5
        ids = torch.randperm(pool, generator=gen, device="cuda", dtype=torch.int32)
        table = torch.full((case["B"], case["width"]), -1, dtype=torch.int32, device="cuda")
        mask = torch.arange(case["width"], device="cuda")[None] < _ints(pages)[:, None]
        table[mask] = ids[: sum(pages)]
        s["free_pages"] = torch.full((pool,), -1, dtype=torch.int32, device="cuda")
        s["free_pages"][:free] = ids[sum(pages): sum(pages) + free]
        s |= {"k_len": _ints(held), "n_new": _ints(new), "block_table": table, "free_count": _ints([free])}
        s["tables"] = {"q_start": table.new_empty(case["B"] + 1), "k_len": table.new_empty(case["B"]),
                       "slots": table.new_empty(s["max_tokens"]), "counts": table.new_empty(2)}  # where the step's tables go
    elif case["op"] == "write":
        T = case["T"]
        n_pages = -(-T // P) + 3
        s["k_cache"], s["v_cache"] = _cache(case, n_pages, gen)
        s["k"], s["v"] = (torch.randn((T, case["Hkv"], case["D"]), dtype=DTYPES[case["dtype"]], device="cuda", generator=gen) for _ in range(2))
        # the tokens of a request follow one another inside pages that lie anywhere; the last sixteenth is padding
        page = torch.randperm(n_pages, generator=gen, device="cuda", dtype=torch.int32)
        t = torch.arange(T, device="cuda", dtype=torch.int32)
        s["slots"] = torch.where(t < T - T // 16, page[(t // P).long()] * P + t % P, torch.full_like(t, -1))
    else:
        B, Lp = case["B"], case["prefix"]
        new = _spread(1, case["n"], B, rng) if case["n"] > 8 else [case["n"]] * B
        past = _spread(0, case["own_keys"] - case["n"], B, rng)
        held = [a + b for a, b in zip(new, past)]
        pages, prefix_pages = [-(-h // P) for h in held], -(-Lp // P)
        ids = torch.randperm(sum(pages) + prefix_pages + 7, generator=gen, device="cuda", dtype=torch.int32)
        s["k_cache"], s["v_cache"] = _cache(case, ids.numel(), gen)
        table = torch.zeros((B, max(pages)), dtype=torch.int32, device="cuda")
        mask = torch.arange(max(pages), device="cuda")[None] < _ints(pages)[:, None]
        table[mask] = ids[prefix_pages: prefix_pages + sum(pages)]
        start = [0]
        for n in new:
            start.append(start[-1] + n)
        s["q"] = torch.randn((start[-1], case["Hq"], case["D"]), dtype=DTYPES[case["dtype"]], device="cuda", generator=gen)
        s["out"] = torch.empty_like(s["q"])
        s |= {"q_start": _ints(start), "k_len": _ints(held), "block_table": table, "prefix_table": ids[:prefix_pages].clone(),
              "max_new": max(new)}
    return s


def work(case):
    P, rng = case["P"], random.Random(0)
    if case["op"] == "plan":
        held, new = _plan_lengths(case, rng)
        tokens = sum(max(n, 0) for n in new)
        moved = sum(abs(-(-(h + n) // P) - -(-h // P)) for h, n in zip(held, new))
        return {"bytes": 16 * case["B"] + 8 * moved + 4 * tokens, "flops": 0}
    if case["op"] == "write":
        return {"bytes": 8 * (case["T"] - case["T"] // 16) * case["Hkv"] * case["D"] + 4 * case["T"], "flops": 0}
    B, n = case["B"], case["n"]
    new = _spread(1, n, B, rng) if n > 8 else [n] * B
    past = _spread(0, case["own_keys"] - n, B, rng)
    seen = sum(a * case["prefix"] + a * b + a * (a + 1) // 2 for a, b in zip(new, past))
    keys = case["prefix"] + sum(new) + sum(past)
    return {"bytes": 4 * case["D"] * (sum(new) * case["Hq"] + keys * case["Hkv"]), "flops": 4 * case["D"] * case["Hq"] * seen}


# --------------------------------------------------------------------------------------------- the operators

def _library():
    if "flash_attention_amd" not in sys.modules:
        sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
        import __graft_entry__

        __graft_entry__.load_package()
    return sys.modules["flash_attention_amd"]


def run(s):
    if own:
        fa = _library()
        if s["op"] == "plan":
            p = fa.cache_plan(s["k_len"], s["n_new"], s["block_table"], s["free_pages"], s["free_count"], s["P"],
                              out=fa.CachePlan(**s["tables"]))
            return {"q_start": p.q_start, "k_len": p.k_len, "slots": p.slots, "counts": p.counts,
                    "block_table": s["block_table"], "free_pages": s["free_pages"]}
        cache = s.get("cache") or s.setdefault("cache", fa.PagedCache(s["k_cache"], s["v_cache"]))  # a program has one for good
        if s["op"] == "write":
            fa.cache_write(s["k"], s["v"], cache, s["slots"])
            return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        return fa.attention_shared_prefix(s["q"], cache, s["q_start"], s["k_len"], s["block_table"],
                                          prefix_table=s["prefix_table"], prefix_len=s["prefix"], out=s["out"])
    return {"plan": _plan, "write": _write, "attend": _attend}[s["op"]](s)


def _plan(s):
    P, width, cap = s["P"], s["width"], s["free_pages"].numel()
    k, n, table = s["k_len"].long(), s["n_new"].long(), s["block_table"]
    have, want = (k + P - 1) // P, (k + n + P - 1) // P
    rel, need = (have - want).clamp_min(0), (want - have).clamp_min(0)
    rel_end, need_end = rel.cumsum(0), need.cumsum(0)
    q_start = torch.cat([n.new_zeros(1), n.clamp_min(0).cumsum(0)])
    c0 = s["free_count"].long()[0]
    top = c0 + rel_end[-1]
    fits = (need == 0) | (need_end <= top)
    taken = torch.where(fits, need_end, 0).amax()
    # the free list with the released pages on it, in request order
    i = torch.arange(cap, device=k.device)
    b = torch.searchsorted(rel_end, i - c0, right=True).clamp_max(k.numel() - 1)
    col = (want[b] + (i - c0) - (rel_end[b] - rel[b])).clamp(0, width - 1)
    stack = torch.where((i >= c0) & (i < top), table[b, col], s["free_pages"])
    s["free_pages"].copy_(stack)
    # the pages taken, into the table
    j = torch.arange(width, device=k.device)[None]
    new = (j >= have[:, None]) & (j < want[:, None]) & fits[:, None]
    at = (top - 1 - (need_end - need)[:, None] - (j - have[:, None])).clamp(0, cap - 1)
    table.copy_(torch.where(new, stack[at], table))
    t = torch.arange(s["max_tokens"], device=k.device)
    b = torch.searchsorted(q_start[1:], t, right=True).clamp_max(k.numel() - 1)
    pos = k[b] + t - q_start[b]
    slot = table[b, (pos // P).clamp(0, width - 1)] * P + pos % P
    slots = torch.where((t < q_start[-1]) & fits[b], slot, -1)
    counts = torch.stack([top - taken, (~fits).sum()])
    return {"q_start": q_start.int(), "k_len": torch.where(fits, k + n, k).int(), "slots": slots.int(), "counts": counts.int(),
            "block_table": table, "free_pages": s["free_pages"]}


def _write(s):
    live = s["slots"] >= 0
    slot = s["slots"][live].long()
    s["k_cache"][slot // s["P"], :, slot % s["P"]] = s["k"][live]
    s["v_cache"][slot // s["P"], :, slot % s["P"]] = s["v"][live]
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _piece(q, k, v, seen):
    """Rows q against keys k, of which `seen` are visible (all where None): sum of exp(score - m) v, the sum of
    exp(score - m), and m, the largest score."""
    scores = q @ k.transpose(-1, -2)
    if seen is not None:
        scores = torch.where(seen, scores, -math.inf)
    m = scores.amax(-1, keepdim=True).clamp_min(-1e30)
    p = torch.exp(scores - m)
    return p @ v, p.sum(-1, keepdim=True), m


def _attend(s):
    q, P, Hkv, D, Lp = s["q"], s["P"], s["Hkv"], s["D"], s["prefix"]
    T, B, g, n = q.shape[0], s["B"], s["Hq"] // s["Hkv"], s["max_new"]
    start = s["q_start"].long()
    rows = (q.float() / math.sqrt(D)).reshape(T, Hkv, g, D).transpose(0, 1)  # [Hkv, T, g, D]
    kp, vp = (c[s["prefix_table"].long()].transpose(0, 1).reshape(Hkv, -1, D)[:, :Lp].float() for c in (s["k_cache"], s["v_cache"]))
    o1, l1, m1 = (x.reshape(Hkv, T, g, -1) for x in _piece(rows.reshape(Hkv, T * g, D), kp, vp, None))
    # every request's own keys, padded to the longest; its rows padded to the most new tokens
    kb, vb = (c[s["block_table"].long()].transpose(1, 2).reshape(B, Hkv, -1, D).float() for c in (s["k_cache"], s["v_cache"]))
    i = torch.arange(n, device=q.device)
    count = start[1:] - start[:-1]
    padded = rows[:, (start[:-1, None] + i).clamp_max(T - 1)].permute(1, 0, 2, 3, 4).reshape(B, Hkv, n * g, D)
    last = (s["k_len"].long() - count)[:, None] + i  # the last key that new token i sees
    seen = torch.arange(kb.shape[2], device=q.device)[None, None] <= last[:, :, None]
    o2, l2, m2 = (x.reshape(B, Hkv, n, g, -1) for x in _piece(padded, kb, vb, seen.repeat_interleave(g, 1)[:, None]))
    t = torch.arange(T, device=q.device)
    b = torch.searchsorted(start[1:], t, right=True)
    o2, l2, m2 = (x[b, :, t - start[b]].transpose(0, 1) for x in (o2, l2, m2))
    m = torch.maximum(m1, m2)
    w1, w2 = torch.exp(m1 - m), torch.exp(m2 - m)
    o = (o1 * w1 + o2 * w2) / (l1 * w1 + l2 * w2)
    return o.transpose(0, 1).reshape(T, s["Hq"], D).to(q.dtype)


# --------------------------------------------------------------------------------------------- from the definition

def exact(case, seed):
    s = prepare(case, seed)
    P = case["P"]
    if case["op"] == "plan":
        held, new = s["k_len"].tolist(), s["n_new"].tolist()
        table, stack = s["block_table"].tolist(), s["free_pages"].tolist()[: s["free_count"].item()]
        after, slots, start, refused = [], [], [0], 0
        for b, (h, n) in enumerate(zip(held, new)):
            stack += table[b][-(-(h + n) // P): -(-h // P)]
        pages = stack + s["free_pages"].tolist()[len(stack):]  # what lies above the count stays where it was
        for b, (h, n) in enumerate(zip(held, new)):
            need = max(0, -(-(h + n) // P) - -(-h // P))
            ok = need <= len(stack) and (not refused or need == 0)
            refused += not ok
            for j in range(need if ok else 0):
                table[b][-(-h // P) + j] = stack.pop()
            slots += [table[b][p // P] * P + p % P if ok else -1 for p in range(h, h + n)]
            start.append(start[-1] + max(n, 0))
            after.append(h + n if ok else h)
        slots += [-1] * (s["max_tokens"] - len(slots))
        return {"q_start": _ints(start), "k_len": _ints(after), "slots": _ints(slots), "counts": _ints([len(stack), refused]),
                "block_table": _ints(table), "free_pages": _ints(pages)}
    if case["op"] == "write":
        got = {}
        t = (s["slots"] >= 0).nonzero()[:, 0]
        for name, rows in (("k_cache", s["k"]), ("v_cache", s["v"])):
            flat = s[name].transpose(1, 2).double().reshape(-1, case["Hkv"], case["D"]).contiguous()
            flat.index_copy_(0, s["slots"][t].long(), rows[t].double())
            got[name] = flat.reshape(-1, P, case["Hkv"], case["D"]).transpose(1, 2)
        return got
    g, start, out = case["Hq"] // case["Hkv"], s["q_start"].tolist(), torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, kl in enumerate(s["k_len"].tolist()):
        n, past = start[b + 1] - start[b], kl - (start[b + 1] - start[b])
        pages = s["block_table"][b, : -(-kl // P)].long()
        for h in range(case["Hkv"]):
            k, v = (torch.cat([c[s["prefix_table"].long(), h].reshape(-1, case["D"])[: case["prefix"]],
                               c[pages, h].reshape(-1, case["D"])[:kl]]).double() for c in (s["k_cache"], s["v_cache"]))
            rows = s["q"][start[b]: start[b + 1], h * g: (h + 1) * g].double().transpose(0, 1).reshape(g * n, -1)
            scores = (rows @ k.t() / case["D"] ** 0.5).reshape(g, n, -1)
            hidden = torch.arange(k.shape[0], device="cuda") > case["prefix"] + past + torch.arange(n, device="cuda")[:, None]
            p = scores.masked_fill(hidden, -math.inf).softmax(-1)
            out[start[b]: start[b + 1], h * g: (h + 1) * g] = (p.reshape(g * n, -1) @ v).reshape(g, n, -1).transpose(0, 1)
    return out
