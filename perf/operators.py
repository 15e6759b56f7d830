"""What the ragged operators are measured on: page tables, append and decode attention of
requests with different lengths that share one page pool.

``run`` makes one pass through an operator: in its plain form (elementary torch operations)
or, with ``own`` set, through the package.  ``exact`` is the attention in 64 bits.
"""

import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}

# Padded K elements of the largest attention case (8 requests x 32768 tokens x 8 heads x 128):
# drawn cases stay at or below it.
MOST_ELEMENTS = 8 * 32768 * 8 * 128


def listed():
    return [
        # a decode step's tables: each of 64 running requests grows by one token
        {"name": "tables step 64", "op": "tables", "requests": 64, "page": 16, "grow": 64,
         "admit": 0, "retire": 0, "prompt": 0, "context": 4096},
        # a busy server's step: decoding requests, 24 prompts of up to 8192 tokens, 40 leave
        {"name": "tables mixed 1024", "op": "tables", "requests": 1024, "page": 16, "grow": 960,
         "admit": 24, "retire": 40, "prompt": 8192, "context": 16384},
        # one layer's append of a decode step over 64 requests
        {"name": "append step 64 bf16", "op": "append", "dtype": "bf16", "tokens": 64,
         "kv_heads": 8, "dim": 128, "page": 16, "padding": 0},
        # one layer's append of a chunk of prompts, 32768 tokens
        {"name": "append prompts fp16", "op": "append", "dtype": "fp16", "tokens": 32768,
         "kv_heads": 8, "dim": 128, "page": 16, "padding": 0},
        # fp32, five-token pages, an odd count of tokens and a padded tail
        {"name": "append odd fp32", "op": "append", "dtype": "fp32", "tokens": 5001,
         "kv_heads": 3, "dim": 64, "page": 5, "padding": 119},
        # a single short request: nothing but latency
        {"name": "attend one short bf16", "op": "attend", "dtype": "bf16", "batch": 1,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "length": 77, "mix": 0,
         "window": 0},
        # the benchmark's batch: 8 requests of 32768 tokens, 4 query heads per kv head
        {"name": "attend 8x32768 bf16", "op": "attend", "dtype": "bf16", "batch": 8,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "length": 32768, "mix": 0,
         "window": 0},
        # one request of 131072 tokens, 7 query heads per kv head
        {"name": "attend 1x131072 bf16", "op": "attend", "dtype": "bf16", "batch": 1,
         "heads": 28, "kv_heads": 4, "dim": 128, "page": 16, "length": 131072, "mix": 0,
         "window": 0},
        # continuous batching: 64 requests from a token to 4093, one of them empty, 8 query
        # heads per kv head
        {"name": "attend 64 mixed fp16", "op": "attend", "dtype": "fp16", "batch": 64,
         "heads": 64, "kv_heads": 8, "dim": 128, "page": 32, "length": 4093, "mix": 1,
         "window": 0},
        # many short requests without head sharing
        {"name": "attend 255 short fp16", "op": "attend", "dtype": "fp16", "batch": 255,
         "heads": 16, "kv_heads": 16, "dim": 64, "page": 16, "length": 509, "mix": 2,
         "window": 0},
        # fp32, five-token pages, a sliding window over part of each request
        {"name": "attend odd window fp32", "op": "attend", "dtype": "fp32", "batch": 5,
         "heads": 12, "kv_heads": 4, "dim": 64, "page": 5, "length": 9001, "mix": 3,
         "window": 5000},
        # 16 query heads on each of 2 kv heads
        {"name": "attend 16 shared bf16", "op": "attend", "dtype": "bf16", "batch": 16,
         "heads": 32, "kv_heads": 2, "dim": 128, "page": 64, "length": 16384, "mix": 4,
         "window": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "append", "attend", "attend"])
    if op == "tables":
        requests = _log(rng, 1, 1024)
        admit = rng.randint(0, min(24, requests))
        retire = rng.randint(0, min(40, requests - admit))
        return {"op": op, "requests": requests, "page": rng.choice([5, 8, 16, 32, 64]),
                "grow": requests - admit - retire, "admit": admit, "retire": retire,
                "prompt": _log(rng, 1, 8192), "context": _log(rng, 2, 16384)}
    if op == "append":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        kv_heads, dim = rng.randint(1, 8), rng.choice([64, 128])
        most = 32768 * 8 * 128 * 2 // (kv_heads * dim * BYTES[dtype])
        tokens = _log(rng, 1, min(32768, most))
        return {"op": op, "dtype": dtype, "tokens": tokens, "kv_heads": kv_heads, "dim": dim,
                "page": rng.choice([5, 8, 16, 32, 64]),
                "padding": rng.choice([0, rng.randint(0, tokens)])}
    dtype = rng.choice(["bf16", "fp16", "bf16", "fp16", "fp32"])
    kv_heads, dim = rng.randint(1, 8), rng.choice([64, 128])
    batch = _log(rng, 1, 256)
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 16])
    if dtype == "fp32":
        group = min(group, 8)
    most = MOST_ELEMENTS // (batch * kv_heads * dim) // (2 if dtype == "fp32" else 1)
    length = _log(rng, 1, min(131072, most))
    window = rng.choice([0, 0, _log(rng, 1, length)])
    return {"op": op, "dtype": dtype, "batch": batch, "heads": kv_heads * group,
            "kv_heads": kv_heads, "dim": dim, "page": rng.choice([5, 8, 16, 32, 64]),
            "length": length, "mix": rng.randint(0, 1000), "window": window}


def _lengths(case):
    """Tokens of each request: all of them ``length`` where ``mix`` is 0, and otherwise spread
    over the logarithm of [1, length], with one request of ``length`` and, of four or more, an
    empty one."""
    batch, length = case["batch"], case["length"]
    if not case["mix"]:
        return [length] * batch
    rng = random.Random(case["mix"])
    lengths = [_log(rng, 1, length) for _ in range(batch)]
    lengths[rng.randrange(batch)] = length
    if batch >= 4:
        lengths[min(range(batch), key=lengths.__getitem__)] = 0
    return lengths


def _starts(case):
    """First attended token of each request: the last ``window`` ones (0: all of them)."""
    return [max(0, n - case["window"]) if case["window"] else 0 for n in _lengths(case)]


def _pages(n, page):
    return -(-n // page)


def _table_lengths(case):
    """(tokens cached, tokens wanted) of each request, in a mixed order."""
    rng = random.Random(case["requests"] * 131 + case["context"])
    pairs = []
    for _ in range(case["grow"]):
        n = _log(rng, 1, case["context"])
        pairs.append((n, n + 1))
    for i in range(case["admit"]):
        pairs.append((0, case["prompt"] if i == 0 else _log(rng, 1, case["prompt"])))
    for _ in range(case["retire"]):
        pairs.append((_log(rng, 1, case["context"]), 0))
    rng.shuffle(pairs)
    return pairs


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = torch.device("cuda")

    def ints(values):
        return torch.tensor(values, dtype=torch.int64, device=dev)

    def normal(*shape, dtype):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).to(dtype)

    if case["op"] == "tables":
        pairs, page = _table_lengths(case), case["page"]
        width = _pages(max(case["context"] + 1, case["prompt"], 1), page)
        held = [_pages(n, page) for n, _ in pairs]
        want = sum(max(0, _pages(m, page) - _pages(n, page)) for n, m in pairs)
        spare = want + 100
        slots = sum(held) + spare
        perm = torch.randperm(slots, generator=g, device=dev)
        table = torch.zeros(len(pairs), width, dtype=torch.int64, device=dev)
        at = torch.arange(width, device=dev)[None] < ints(held)[:, None]
        table[at] = perm[:sum(held)]
        ring = torch.zeros(slots, dtype=torch.int64, device=dev)
        head = slots - min(slots, spare // 2 + 1)     # the free part runs over the ring's end
        ring[(head + torch.arange(spare, device=dev)) % slots] = perm[sum(held):]
        return {"case": case, "lengths": ints([n for n, _ in pairs]),
                "new_lengths": ints([m for _, m in pairs]), "page_table": table,
                "ring": ring, "free": ints([head, spare, 0]),
                "most": sum(max(0, m - n) for n, m in pairs) + 3}
    dtype, page = DTYPES[case["dtype"]], case["page"]
    kv_heads, dim = case["kv_heads"], case["dim"]
    if case["op"] == "append":
        tokens = case["tokens"]
        slots = _pages(tokens, page) + 7
        slot_map = torch.randperm(slots * page, generator=g, device=dev)[:tokens]
        if tokens >= 64:    # prompts fill whole pages in order
            pages = torch.randperm(slots, generator=g, device=dev)
            t = torch.arange(tokens, device=dev)
            slot_map = pages[t // page] * page + t % page
        slot_map[max(1, tokens - case["padding"]):] = -1
        return {"case": case, "key": normal(tokens, kv_heads, dim, dtype=dtype),
                "value": normal(tokens, kv_heads, dim, dtype=dtype),
                "key_pool": normal(slots, kv_heads, page, dim, dtype=dtype),
                "value_pool": normal(slots, kv_heads, page, dim, dtype=dtype),
                "slot_map": slot_map}
    lengths = _lengths(case)
    held = [_pages(n, page) for n in lengths]
    width = max(1, max(held))
    slots = sum(held) + 5
    perm = torch.randperm(slots, generator=g, device=dev)
    table = torch.zeros(len(lengths), width, dtype=torch.int64, device=dev)
    table[torch.arange(width, device=dev)[None] < ints(held)[:, None]] = perm[:sum(held)]
    return {"case": case,
            # queries of different sharpness: logits of deviation 1 to 3
            "query": (normal(len(lengths), case["heads"], 1, dim, dtype=torch.float32)
                      * torch.linspace(1, 3, case["heads"], device=dev)[:, None, None]).to(dtype),
            "key_pool": normal(slots, kv_heads, page, dim, dtype=dtype),
            "value_pool": normal(slots, kv_heads, page, dim, dtype=dtype),
            "page_table": table, "lengths": ints(lengths),
            "starts": ints(_starts(case)) if case["window"] else None}


def run(state):
    op = state["case"]["op"]
    if own:
        import razorkv_b200
        if op == "tables":
            t = razorkv_b200.ragged_page_tables(
                state["lengths"], state["new_lengths"], state["page_table"], state["ring"],
                state["free"], state["case"]["page"], state["most"])
            return {"lengths": t.lengths, "slot_map": t.slot_map, "positions": t.positions,
                    "token_starts": t.token_starts, "free": t.free_state,
                    "page_table": state["page_table"], "ring": state["ring"]}
        if op == "append":
            razorkv_b200.ragged_append(state["key"], state["value"], state["key_pool"],
                                       state["value_pool"], state["slot_map"])
            return {"key_pool": state["key_pool"], "value_pool": state["value_pool"]}
        out, lse = razorkv_b200.ragged_decode_attention(
            state["query"], state["key_pool"], state["value_pool"], state["page_table"],
            state["lengths"], starts=state["starts"], return_lse=True)
        return {"out": out, "lse": lse}
    return {"tables": _plain_tables, "append": _plain_append, "attend": _plain_attend}[op](state)


def _plain_tables(state):
    n, m, table = state["lengths"], state["new_lengths"], state["page_table"]
    ring, free, page = state["ring"], state["free"], state["case"]["page"]
    have, want = (n + page - 1) // page, (m + page - 1) // page
    need, give, new = (want - have).clamp(min=0), (have - want).clamp(min=0), (m - n).clamp(min=0)
    starts = torch.cat([torch.zeros_like(n[:1]), new.cumsum(0)])
    j = torch.arange(table.shape[1], device=n.device)[None]
    taken = (j >= have[:, None]) & (j < want[:, None])
    rank = (need.cumsum(0) - need)[:, None] + j - have[:, None]
    given = (j >= want[:, None]) & (j < have[:, None])
    place = free[0] + free[1] + (give.cumsum(0) - give)[:, None] + j - want[:, None]
    size = ring.numel()
    # entries that are not given back go to a place behind the ring
    longer = torch.cat([ring, ring[:1]])
    longer[torch.where(given, place % size, size)] = table
    table.copy_(torch.where(taken, ring[(free[0] + rank) % size], table))
    ring.copy_(longer[:size])
    i = torch.arange(state["most"], device=n.device)
    r = (torch.searchsorted(starts, i, right=True) - 1).clamp(max=n.numel() - 1)
    used = i < starts[-1]
    position = torch.where(used, n[r] + i - starts[r], 0)
    slot = table[r, (position // page).clamp(max=table.shape[1] - 1)] * page + position % page
    after = torch.stack([(free[0] + need.sum()) % size, free[1] - need.sum() + give.sum(),
                         free[2]])
    return {"lengths": m.clone(), "slot_map": torch.where(used, slot, -1), "positions": position,
            "token_starts": starts, "free": after, "page_table": table, "ring": ring}


def _plain_append(state):
    slot, page = state["slot_map"], state["case"]["page"]
    # a row without a slot repeats the first row that has one
    valid = slot >= 0
    row = torch.where(valid, torch.arange(slot.numel(), device=slot.device),
                      valid.to(torch.int32).argmax())
    at = slot[row]
    state["key_pool"][at // page, :, at % page] = state["key"][row]
    state["value_pool"][at // page, :, at % page] = state["value"][row]
    return {"key_pool": state["key_pool"], "value_pool": state["value_pool"]}


def _plain_attend(state):
    q, table, lengths, starts = (state[k] for k in ("query", "page_table", "lengths", "starts"))
    b, heads, _, dim = q.shape
    kv_heads, page = state["key_pool"].shape[1:3]
    # pages of one request in order: [batch, kv heads, tokens, dim]
    k, v = (state[name][table].float().transpose(1, 2).reshape(b, kv_heads, -1, dim)
            for name in ("key_pool", "value_pool"))
    t = torch.arange(table.shape[1] * page, device=q.device)[None]
    inside = t < lengths[:, None]
    if starts is not None:
        inside = inside & (t >= starts[:, None])
    inside = inside[:, None, None]
    logits = q.float().reshape(b, kv_heads, -1, dim) @ k.transpose(2, 3) / math.sqrt(dim)
    logits = torch.where(inside, logits, -math.inf)
    top = logits.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(logits - top)
    total = p.sum(-1, keepdim=True)
    out = p @ torch.where(inside.transpose(2, 3), v, 0.0) / torch.where(total == 0, 1.0, total)
    return {"out": out.reshape(b, heads, 1, dim).to(q.dtype),
            "lse": (torch.log(total) + top).reshape(b, heads)}


def work(case):
    if case["op"] == "tables":
        pairs, page = _table_lengths(case), case["page"]
        moved = sum(abs(_pages(m, page) - _pages(n, page)) for n, m in pairs)
        part = sum(1 for n, m in pairs if m > n and n % page)
        new = sum(max(0, m - n) for n, m in pairs)
        # lengths in and out, starts, ring and table entries, slots and positions
        return {"bytes": 8 * (3 * len(pairs) + len(pairs) + 1 + 2 * moved + part + 2 * (new + 3)),
                "flops": 0}
    size = BYTES[case["dtype"]]
    if case["op"] == "append":
        rows = max(1, case["tokens"] - case["padding"])
        return {"bytes": 4 * rows * case["kv_heads"] * case["dim"] * size + 8 * case["tokens"],
                "flops": 0}
    lengths, starts = _lengths(case), _starts(case)
    tokens = sum(n - s for n, s in zip(lengths, starts))
    pages = sum(_pages(n, case["page"]) - s // case["page"] for n, s in zip(lengths, starts))
    ends = case["batch"] * case["heads"] * (2 * case["dim"] * size + 4)
    return {"bytes": 2 * tokens * case["kv_heads"] * case["dim"] * size + 8 * pages
            + 8 * case["batch"] + ends,
            "flops": 4 * tokens * case["heads"] * case["dim"]}


def exact(case, seed):
    if case["op"] == "tables":
        return None     # whole numbers
    state = prepare(case, seed)
    if case["op"] == "append":
        used = (state["slot_map"] >= 0).nonzero()[:, 0]
        slot, pools = state["slot_map"][used], {}
        for name in ("key", "value"):
            pool = state[name + "_pool"].double().transpose(1, 2).contiguous()
            pool.flatten(0, 1).index_copy_(0, slot, state[name][used].double())
            pools[name + "_pool"] = pool.transpose(1, 2)
        return pools
    q, table = state["query"].double(), state["page_table"]
    group = case["heads"] // case["kv_heads"]
    outs, sums = [], []
    for b, (n, s) in enumerate(zip(_lengths(case), _starts(case))):
        if n <= s:
            outs.append(torch.zeros_like(q[b, :, 0]))
            sums.append(torch.full_like(q[b, :, 0, 0], -math.inf))
            continue
        t = torch.arange(s, n, device=q.device)
        at, off = table[b, t // case["page"]], t % case["page"]
        one, two = [], []
        for h in range(case["kv_heads"]):
            k = state["key_pool"][at, h, off].double()
            v = state["value_pool"][at, h, off].double()
            logits = torch.einsum("gd,td->gt", q[b, h * group:(h + 1) * group, 0], k) * case["dim"] ** -0.5
            one.append(torch.einsum("gt,td->gd", torch.softmax(logits, 1), v))
            two.append(torch.logsumexp(logits, 1))
        outs.append(torch.cat(one))
        sums.append(torch.cat(two))
    return {"out": torch.stack(outs)[:, :, None], "lse": torch.stack(sums)}
