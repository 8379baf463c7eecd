"""The paged K/V cache's operators as timed cases: tables, appends and the two attentions that read pages.

A paged cache holds the K/V rows of many requests of different lengths in
blocks of ``block`` rows, ``[blocks, kv_heads, block, D]``; a request's block
table names its blocks in order.  Four kinds of case:

* ``tables``: one step's bookkeeping on the GPU (blocks taken from and given
  back to the ring of free blocks, block tables, slot map, query starts).
* ``append``: K/V rows of a step's tokens into their slots.
* ``window``: attention of each request's new tokens over its blocks, with an
  optional sliding window and first tokens that stay visible.
* ``prefix``: the same for requests that share one prefix's blocks.

With ``own`` false ``run`` computes them by elementary torch operations in 32
bits, on all requests at once (padded); with ``own`` true it calls the
framework.  Request lengths are a function of the case; values, block order
and slots are a function of the seed.
"""

import random

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------- cases

def listed():
    attn = dict(kind="window", block=16, dim=128, dtype="bf16", window=0, sinks=0, causal=True, ragged=False, pad=0,
                layout="heads")
    shared = dict(kind="prefix", block=16, dim=128, dtype="bf16", causal=True, ragged=False, pad=0, layout="heads")
    tables = dict(kind="tables", block=16, window=0, sinks=0, ended=0.0, ragged=False, pad=0)
    return [
        # One decode step of eight requests: the latency of the bookkeeping.
        dict(tables, name="tables_decode", requests=8, held=1000, new=1),
        # A large serving step: prompts arrive, decodes go on, a tenth of the
        # requests end, and blocks leave a sliding window.
        dict(tables, name="tables_prompts", requests=1000, held=4000, new=128, window=1024, sinks=21, ended=0.1,
             ragged=True, pad=500),
        # K/V of one token of each of 16 requests.
        dict(kind="append", name="append_decode", requests=16, held=500, new=1, kv_heads=8, dim=128, block=16,
             dtype="bf16", ragged=True, pad=0, layout="heads"),
        # K/V of the prompts of four requests, 16 heads, rows in another order.
        dict(kind="append", name="append_prompts", requests=4, held=0, new=4096, kv_heads=16, dim=128, block=32,
             dtype="bf16", ragged=False, pad=0, layout="tokens"),
        # Single tokens of a CFG pair with 16 heads over the 1024x1024 schedule's
        # prior rows: the smallest call.
        dict(attn, name="window_token_pair", requests=2, held=6424, new=1, heads=16, kv_heads=16),
        # Single tokens of many ragged requests, four query heads for each K/V head:
        # the bytes of a long cache.
        dict(attn, name="window_tokens_64", requests=64, held=16000, new=1, heads=32, kv_heads=8, ragged=True, pad=3),
        # The same with a window: only its rows and the first 21 are read.
        dict(attn, name="window_tokens_sinks", requests=48, held=30000, new=1, heads=32, kv_heads=8, window=4096,
             sinks=21, ragged=True, layout="tokens", block=64),
        # A long prompt, the largest product.
        dict(attn, name="window_prompt", requests=1, held=0, new=8192, heads=32, kv_heads=8),
        # Ragged prompts in fp16 with odd lengths, 64-wide heads, a window and sinks, behind held rows.
        dict(attn, name="window_prompts_odd", requests=7, held=1111, new=2047, heads=12, kv_heads=4, dim=64,
             dtype="fp16", window=777, sinks=5, ragged=True, pad=9),
        # A small batch behind a shared prompt of the first seven scales' 521 rows.
        dict(shared, name="prefix_tokens_small", requests=4, prefix=521, held=100, new=1, heads=16, kv_heads=16),
        # Many continuations of one long prompt.
        dict(shared, name="prefix_tokens_128", requests=128, prefix=16384, held=500, new=1, heads=32, kv_heads=8,
             ragged=True),
        # A scale of 256 tokens (every token sees the whole scale) of 8 images
        # that share 6425 prior rows.
        dict(shared, name="prefix_scale", requests=8, prefix=6425, held=256, new=256, heads=16, kv_heads=16,
             causal=False),
    ]


def draw(rng):
    log = lambda a, b: int(round(a * (b / a) ** rng.random()))  # noqa: E731
    kind = rng.choice(["tables", "append", "window", "window", "window", "prefix", "prefix"])
    case = dict(kind=kind, block=rng.choice([8, 16, 32, 64, 128]), ragged=rng.random() < 0.7,
                pad=rng.choice([0, 0, 1, 7, 64]))
    if kind == "tables":
        few = rng.random() < 0.5
        case.update(requests=log(1, 1000), held=log(1, 4000), new=1 if few else log(2, 128),
                    window=rng.choice([0, 300, 1024]), ended=rng.choice([0.0, 0.2]))
        case["sinks"] = rng.choice([0, 4, 21]) if case["window"] else 0
        return case
    group = rng.choice([1, 1, 2, 3, 4, 6, 8])
    case.update(dim=rng.choice([64, 128, 128]), dtype=rng.choice(["bf16", "bf16", "fp16"]),
                layout=rng.choice(["heads", "tokens"]), kv_heads=rng.choice([1, 2, 4, 5, 8]))
    if kind == "append":
        case.update(requests=log(1, 64), held=log(1, 500), new=rng.choice([1, log(2, 500)]))
        return case
    case.update(heads=case["kv_heads"] * group, causal=rng.random() < 0.75)
    if rng.random() < 0.5:  # single tokens, or a few
        case.update(requests=log(1, 96), held=log(1, 10000), new=rng.choice([1, 1, 1, 2, 5]))
    else:
        case.update(requests=log(1, 8), held=log(1, 2000), new=log(16, 2000))
    if kind == "prefix":
        case.update(prefix=log(64, 8000))
        case["held"] = min(case["held"], 1000)
    else:
        case.update(window=rng.choice([0, 0, 100, 1000, 4096]))
        case["sinks"] = rng.choice([0, 4, 21, 130]) if case["window"] else 0
    return case


def _lengths(case):
    """(rows held before the step, new tokens) of each request; -1 new: the request has ended."""
    rng = random.Random("%d %d %d" % (case["requests"], case["held"], case["new"]))
    got = []
    for _ in range(case["requests"]):
        held, new = case["held"], case["new"]
        if case["ragged"]:
            held = int(held * (0.05 + 0.95 * rng.random()))
            new = new if new == 1 else int(new * rng.random() ** 2) + (rng.random() < 0.9)
        if case.get("ended") and rng.random() < case["ended"]:
            new = -1
        got.append((held, new))
    if all(new <= 0 for _, new in got):
        got[0] = (got[0][0], case["new"])
    return got


def _blocks(rows, block):
    return -(-rows // block)


# ---------------------------------------------------------------- inputs

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    sizes = _lengths(case)
    block = case["block"]
    held, new = [h for h, _ in sizes], [max(n, 0) for _, n in sizes]
    total = [h + n for h, n in sizes] if case["kind"] != "tables" else [h + max(n, 0) for h, n in sizes]
    tokens = sum(new) + case["pad"]
    width = max(max(_blocks(t, block) for t in total), 1)
    s = {"case": case, "tokens": tokens}
    if case["kind"] == "tables":
        s.update(_tables_inputs(case, sizes, width, gen))
        return s
    shared = _blocks(case.get("prefix", 0), block)
    counts = [_blocks(t, block) for t in total]
    blocks = sum(counts) + shared + 5
    order = torch.randperm(blocks, generator=gen, device=DEVICE).to(torch.int32)
    first = torch.tensor([0] + counts, device=DEVICE).cumsum(0)[:-1] + shared
    at = first[:, None] + torch.arange(width, device=DEVICE)
    live = torch.arange(width, device=DEVICE) < torch.tensor(counts, device=DEVICE)[:, None]
    tables = torch.where(live, order[at.clamp(max=blocks - 1)], 0).contiguous()
    s["query_starts"] = _ints([0] + new).cumsum(0).to(torch.int32)
    s["lengths"] = _ints(total)
    s["block_tables"] = tables
    s["max_new"], s["max_total"] = max(new), max(max(total), 1)
    dtype = TYPES[case["dtype"]]

    def cache():
        if case["layout"] == "heads":
            shape = (blocks, case["kv_heads"], block, case["dim"])
            return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dtype)
        shape = (blocks, block, case["kv_heads"], case["dim"])
        return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dtype).transpose(1, 2)

    s["k_cache"], s["v_cache"] = cache(), cache()
    if case["kind"] == "append":
        rows = (tokens, case["kv_heads"], case["dim"])
        s["k"] = torch.randn(rows, generator=gen, device=DEVICE).to(dtype)
        s["v"] = torch.randn(rows, generator=gen, device=DEVICE).to(dtype)
        slots = torch.full((tokens,), -1, dtype=torch.int64, device=DEVICE)
        t = torch.arange(sum(new), device=DEVICE)
        r = torch.searchsorted(s["query_starts"][1:].contiguous(), t, right=True)
        pos = torch.tensor(held, device=DEVICE)[r] + t - s["query_starts"][r]
        slots[: sum(new)] = tables[r, pos // block].long() * block + pos % block
        s["slot_map"] = slots
        return s
    s["q"] = torch.randn((tokens, case["heads"], case["dim"]), generator=gen, device=DEVICE).to(dtype)
    s["scale"] = case["dim"] ** -0.5
    if case["kind"] == "prefix":
        s["prefix_blocks"] = order[:shared].contiguous()
    return s


def _tables_inputs(case, sizes, width, gen):
    """Tables of the rows held, and the other blocks in the ring of free ones."""
    block = case["block"]
    counts = [_blocks(h, block) for h, _ in sizes]
    spare = sum(_blocks(h + max(n, 0), block) for h, n in sizes) - sum(counts) + 10
    blocks = sum(counts) + spare
    order = torch.randperm(blocks, generator=gen, device=DEVICE).to(torch.int32)
    c = torch.tensor(counts, device=DEVICE)
    at = (c.cumsum(0) - c)[:, None] + torch.arange(width, device=DEVICE)
    live = torch.arange(width, device=DEVICE) < c[:, None]
    tables = torch.where(live, order[at.clamp(max=blocks - 1)], 0).contiguous()
    first = int(torch.randint(0, blocks, (1,), generator=gen, device=DEVICE))
    ring = torch.zeros(blocks, dtype=torch.int32, device=DEVICE)
    ring[(first + torch.arange(spare, device=DEVICE)) % blocks] = order[sum(counts):]
    return {"block_tables": tables, "lengths": _ints([h for h, _ in sizes]), "new_counts": _ints([n for _, n in sizes]),
            "free_blocks": ring, "free_range": _ints([first, spare])}


# ---------------------------------------------------------------- one pass

def run(s):
    case = s["case"]
    return {"tables": _tables, "append": _append, "window": _window, "prefix": _prefix}[case["kind"]](s, case)


def _tables(s, case):
    if own:
        from heatkv_amd import build_paged_tables
        step = build_paged_tables(
            block_tables=s["block_tables"], lengths=s["lengths"], new_counts=s["new_counts"],
            free_blocks=s["free_blocks"], free_range=s["free_range"], num_tokens=s["tokens"],
            block_size=case["block"], window=case["window"], sinks=case["sinks"])
        return {"tables": s["block_tables"], "free": s["free_blocks"], "slots": step.slot_map,
                "starts": step.query_starts, "lengths": step.lengths, "range": step.free_range,
                "status": step.status}
    block, N, M = case["block"], s["free_blocks"].numel(), s["block_tables"].shape[1]
    held, counts = s["lengths"].long(), s["new_counts"].long()
    first, free = s["free_range"].long().unbind()
    over = counts < 0
    n = counts.clamp(min=0)
    after = torch.where(over, 0, held + n)
    have, need = (held + block - 1) // block, (held + n + block - 1) // block
    take = need - have
    status = (take.sum() > free).int() + 2 * (need > M).any().int() + 4 * (n.sum() > s["tokens"]).int()
    fine = status == 0
    j = torch.arange(M, device=DEVICE)
    fresh = fine & (j >= have[:, None]) & (j < need[:, None])
    at = (first + (take.cumsum(0) - take)[:, None] + j - have[:, None]) % N
    tables = torch.where(fresh, s["free_blocks"][at], s["block_tables"])
    # blocks whose rows no later token sees go to the end of the ring
    kept = (case["sinks"] + block - 1) // block
    gone = lambda rows: ((rows - case["window"] + 1).clamp(min=0) // block).clamp(min=kept)  # noqa: E731
    live = j < have[:, None]
    if case["window"]:
        live = live & ((j < kept) | (j >= gone(held)[:, None]))
        leave = (j >= gone(held)[:, None]) & (j < gone(after)[:, None])
    else:
        leave = torch.zeros_like(live)
    back = fine & torch.where(over[:, None], live, leave)
    place = (first + free + back.flatten().cumsum(0) - 1) % N
    ring = torch.cat([s["free_blocks"], s["free_blocks"][:1]])
    ring.scatter_(0, torch.where(back.flatten(), place, N), tables.flatten())
    used = torch.where(fine, take.sum(), 0)
    starts = torch.cat([n[:1] * 0, n.cumsum(0)]) * fine
    t = torch.arange(s["tokens"], device=DEVICE)
    r = torch.searchsorted(starts[1:].contiguous(), t, right=True).clamp(max=n.numel() - 1)
    pos = held[r] + t - starts[r]
    slot = tables[r, (pos // block).clamp(max=M - 1)].long() * block + pos % block
    return {"tables": tables, "free": ring[:N].contiguous(), "slots": torch.where(t < starts[-1], slot, -1),
            "starts": starts.int(), "lengths": torch.where(fine, after, held).int(),
            "range": torch.stack([(first + used) % N, free - used + back.sum()]).int(), "status": status.view(1)}


def _append(s, case):
    if own:
        from heatkv_amd import append_paged_kv
        append_paged_kv(k=s["k"], v=s["v"], k_cache=s["k_cache"], v_cache=s["v_cache"], slot_map=s["slot_map"])
        return s["k_cache"], s["v_cache"]
    # tokens without a slot go to row 0's present value
    slot = s["slot_map"]
    b, row = slot.clamp(min=0) // case["block"], slot.clamp(min=0) % case["block"]
    at = torch.where(slot < 0, slot[0], slot)
    b, row = at // case["block"], at % case["block"]
    mine = (slot >= 0)[:, None, None]
    s["k_cache"][b, :, row] = torch.where(mine, s["k"], s["k"][:1])
    s["v_cache"][b, :, row] = torch.where(mine, s["v"], s["v"][:1])
    return s["k_cache"], s["v_cache"]


def _rows(cache, tables, rows):
    """The first `rows` cached rows of each table: [R, kv_heads, rows, D] in 32 bits."""
    got = cache[tables.long()].transpose(1, 2)
    return got.reshape(got.shape[0], got.shape[1], -1, got.shape[-1])[:, :, :rows].float()


def _queries(s, case):
    """Queries by request and K/V head, [R, kv_heads, group * max_new, D], their positions among the
    request's own rows [R, max_new] and which exist."""
    starts = s["query_starts"].long()
    i = torch.arange(s["max_new"], device=DEVICE)
    count = starts[1:] - starts[:-1]
    have = i < count[:, None]
    at = torch.where(have, starts[:-1, None] + i, 0)
    R, n, hk, d = at.shape[0], at.shape[1], case["kv_heads"], case["dim"]
    q = s["q"][at].float().view(R, n, hk, -1, d).permute(0, 2, 3, 1, 4).reshape(R, hk, -1, d)
    return q, s["lengths"].long()[:, None] - count[:, None] + i, have, at


def _scatter(s, case, out, lse, have, at):
    """Padded results back to their tokens; tokens behind the last request get zeros."""
    T, (R, n), hk, d = s["tokens"], at.shape, case["kv_heads"], case["dim"]
    out = out.view(R, hk, -1, n, d).permute(0, 3, 1, 2, 4).reshape(R * n, -1)
    lse = lse.view(R, hk, -1, n).permute(0, 3, 1, 2).reshape(R * n, -1)
    to = torch.where(have, at, T).flatten()
    o = torch.zeros((T + 1, out.shape[1]), device=DEVICE, dtype=TYPES[case["dtype"]])
    l = torch.full((T + 1, lse.shape[1]), -float("inf"), device=DEVICE)
    o[to] = out.to(o.dtype)
    l[to] = lse
    return o[:T], l[:T].t().contiguous()


def _softmax_parts(scores):
    """Maximum, exponentials and their sum along the last axis; rows without any key give 0."""
    m = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(m == -float("inf"), 0.0, m))
    return m, p, p.sum(-1, keepdim=True)


def _window(s, case):
    if own:
        from heatkv_amd import paged_window_attention
        return paged_window_attention(
            q=s["q"], k_cache=s["k_cache"], v_cache=s["v_cache"], block_tables=s["block_tables"],
            lengths=s["lengths"], query_starts=s["query_starts"], softmax_scale=s["scale"], window=case["window"],
            sinks=case["sinks"], causal=case["causal"], return_lse=True)
    q, pos, have, at = _queries(s, case)
    S = s["max_total"]
    scores = torch.matmul(q, _rows(s["k_cache"], s["block_tables"], S).transpose(2, 3).contiguous())
    scores = (scores * s["scale"]).view(*q.shape[:2], -1, pos.shape[1], S)
    j = torch.arange(S, device=DEVICE)
    seen = (j < s["lengths"].long()[:, None, None]) & (pos[:, :, None] >= 0)
    if case["causal"]:
        seen = seen & (j <= pos[:, :, None])
    if case["window"]:
        seen = seen & ((j > pos[:, :, None] - case["window"]) | (j < case["sinks"]))
    scores = torch.where(seen[:, None, None], scores, -float("inf"))
    m, p, total = _softmax_parts(scores.view(*q.shape[:3], S))
    out = torch.matmul(p, _rows(s["v_cache"], s["block_tables"], S)) / torch.where(total > 0, total, 1.0)
    return _scatter(s, case, out, (m + total.log()).squeeze(-1), have, at)


def _prefix(s, case):
    if own:
        from heatkv_amd import paged_shared_prefix_attention
        return paged_shared_prefix_attention(
            q=s["q"], k_cache=s["k_cache"], v_cache=s["v_cache"], prefix_blocks=s["prefix_blocks"],
            prefix_length=case["prefix"], block_tables=s["block_tables"], lengths=s["lengths"],
            query_starts=s["query_starts"], softmax_scale=s["scale"], causal=case["causal"], return_lse=True)
    q, pos, have, at = _queries(s, case)
    S, P = s["max_total"], case["prefix"]
    R, hk, rows, d = q.shape
    # the prefix once for all requests' queries, then each request's own rows
    every = q.transpose(0, 1).reshape(hk, R * rows, d)
    pk = _rows(s["k_cache"], s["prefix_blocks"][None], P)[0]
    shared = torch.matmul(every, pk.transpose(1, 2).contiguous()).view(hk, R, rows, P).transpose(0, 1)
    mine = torch.matmul(q, _rows(s["k_cache"], s["block_tables"], S).transpose(2, 3).contiguous())
    j = torch.arange(S, device=DEVICE)
    seen = (j < s["lengths"].long()[:, None, None]).expand(-1, pos.shape[1], -1)
    if case["causal"]:
        seen = seen & (j <= pos[:, :, None])
    mine = torch.where(seen[:, None, None], mine.view(R, hk, -1, pos.shape[1], S), -float("inf"))
    m, p, total = _softmax_parts(torch.cat([shared, mine.view(R, hk, rows, S)], -1) * s["scale"])
    out = torch.matmul(p[..., P:], _rows(s["v_cache"], s["block_tables"], S))
    front = p[..., :P].transpose(0, 1).reshape(hk, R * rows, P)
    front = torch.matmul(front, _rows(s["v_cache"], s["prefix_blocks"][None], P)[0])
    out = (out + front.view(hk, R, rows, d).transpose(0, 1)) / total
    return _scatter(s, case, out, (m + total.log()).squeeze(-1), have, at)


# ---------------------------------------------------------------- work

def work(case):
    sizes = _lengths(case)
    if case["kind"] == "tables":
        tokens = sum(max(n, 0) for _, n in sizes) + case["pad"]
        return {"bytes": 8 * tokens + 16 * len(sizes), "flops": 0}
    row = case["kv_heads"] * case["dim"] * 2
    tokens = sum(n for _, n in sizes)
    if case["kind"] == "append":
        return {"bytes": tokens * (4 * row + 8), "flops": 0}
    pairs = keys = 0
    for held, new in sizes:
        W = case.get("window") or held + new + 1
        for i in range(held, held + new):
            end = i + 1 if case["causal"] else held + new
            pairs += end - max(0, i + 1 - W) + min(case.get("sinks", 0), max(0, i + 1 - W))
        if new:
            low = max(0, held + 1 - W)
            keys += held + new - low + min(case.get("sinks", 0), low)
    keys += case.get("prefix", 0)
    pairs += tokens * case.get("prefix", 0)
    each = case["heads"] * case["dim"]
    return {"bytes": 2 * keys * row + tokens * (4 * each + 4 * case["heads"]), "flops": 4.0 * pairs * each}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    """The operators' definition in 64 bits, request by request and head by head."""
    if case["kind"] == "tables":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["kind"] == "append":
        k, v = s["k_cache"].double(), s["v_cache"].double()
        slots = s["slot_map"].tolist()
        keep = [t for t, slot in enumerate(slots) if slot >= 0]
        blocks = [slots[t] // case["block"] for t in keep]
        rows = [slots[t] % case["block"] for t in keep]
        k[blocks, :, rows] = s["k"].double()[keep]
        v[blocks, :, rows] = s["v"].double()[keep]
        return k, v
    T, H, hk, D, block = s["tokens"], case["heads"], case["kv_heads"], case["dim"], case["block"]
    out = torch.zeros((T, H, D), dtype=torch.float64, device=DEVICE)
    lse = torch.full((H, T), -float("inf"), dtype=torch.float64, device=DEVICE)
    starts, ends = s["query_starts"].tolist(), s["lengths"].tolist()
    P = case.get("prefix", 0)

    def rows_of(cache, blocks, count, head):
        return cache[blocks, head].reshape(-1, D)[:count].double()

    for r, n in enumerate(b - a for a, b in zip(starts, starts[1:])):
        if n == 0:
            continue
        total = ends[r]
        mine = s["block_tables"][r, : _blocks(total, block)].long()
        pos = torch.arange(total - n, total, device=DEVICE)[:, None]
        key = torch.arange(total, device=DEVICE)[None]
        hidden = torch.zeros((n, total), dtype=torch.bool, device=DEVICE)
        if case["causal"]:
            hidden |= key > pos
        if case.get("window"):
            hidden |= (pos - key >= case["window"]) & (key >= case["sinks"])
        if P:
            hidden = torch.cat([hidden.new_zeros((n, P)), hidden], 1)
        for g in range(hk):
            K, V = rows_of(s["k_cache"], mine, total, g), rows_of(s["v_cache"], mine, total, g)
            if P:
                front = s["prefix_blocks"].long()
                K = torch.cat([rows_of(s["k_cache"], front, P, g), K])
                V = torch.cat([rows_of(s["v_cache"], front, P, g), V])
            for h in range(g * (H // hk), (g + 1) * (H // hk)):
                q = s["q"][starts[r]:starts[r] + n, h].double()
                a = (q @ K.t() * D ** -0.5).masked_fill_(hidden, -float("inf"))
                total_lse = torch.logsumexp(a, 1)
                lse[h, starts[r]:starts[r] + n] = total_lse
                out[starts[r]:starts[r] + n, h] = torch.exp(a - total_lse[:, None]) @ V
    return out.reshape(T, H * D), lse
