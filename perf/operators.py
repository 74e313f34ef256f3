"""Cases of the serving-step operators: chunk attention over a paged cache, rotary append, page fork, page compaction.

One step of a paged-cache server runs them in this order: ``fork_pages`` gives every row of the batch its pages (shared
prefixes, a private copy of a partly filled last page, room for the new tokens), ``rotary_append`` rotates the new
tokens' queries and keys and writes keys and values into the cache, ``paged_chunk_attention`` attends from the new
tokens to everything cached, and ``compact_pages`` moves the live pages to the pool's start now and then.
"""
import math
import random

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}


# --- the cases ---------------------------------------------------------------------------------------------------
def _attend(name, rows, new, past, heads, kv_heads, dim, page, dtype, causal=True):
    return {"name": name, "op": "attend", "rows": rows, "new": new, "past": past, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "dtype": dtype, "causal": causal}


def _rotary(name, rows, new, past, heads, kv_heads, dim, rotary, interleaved, page, dtype):
    return {"name": name, "op": "rotary", "rows": rows, "new": new, "past": past, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "rotary": rotary, "interleaved": interleaved, "page": page, "dtype": dtype}


def _fork(name, rows, kept, past, layers, kv_heads, dim, page, dtype):
    return {"name": name, "op": "fork", "rows": rows, "kept": kept, "past": past, "layers": layers,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}


def _compact(name, rows, past, layers, moved, kv_heads, dim, page, dtype):
    return {"name": name, "op": "compact", "rows": rows, "past": past, "layers": layers, "moved": moved,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}


def listed():
    return [
        # a handful of chats generating: one new token each over short caches, where the call's latency counts
        _attend("attend_tokens_small", 8, 1, 1000, 32, 8, 128, 64, "bfloat16"),
        # a full decode batch over caches up to 8K tokens: the read of the cache is the whole cost
        _attend("attend_tokens_batch", 64, 1, 8192, 32, 8, 128, 16, "bfloat16"),
        # a mixed step: single tokens and prompt chunks together, a group of three heads, odd lengths
        _attend("attend_mixed", 16, 509, 4000, 24, 8, 64, 32, "float16"),
        # prompts with little cached before them, every head its own keys
        _attend("attend_prompts", 8, 1024, 100, 16, 16, 128, 128, "bfloat16"),
        # one 4096-token chunk of a long document, 28K tokens already cached
        _attend("attend_long_chunk", 1, 4096, 28672, 32, 8, 128, 128, "bfloat16"),
        # a few draft positions each over an encoder's paged states, unmasked, wide heads sharing one key head
        _attend("attend_wide_unmasked", 13, 7, 3001, 8, 1, 256, 48, "float16", causal=False),
        # the decode batch's rotation and append
        _rotary("rotary_tokens", 64, 1, 8192, 32, 8, 128, 128, False, 16, "bfloat16"),
        # 16K prompt tokens, half of each head rotated in adjacent pairs
        _rotary("rotary_prompts", 4, 4096, 12000, 32, 8, 128, 64, True, 64, "bfloat16"),
        # eight rows, two leave and two fork: one layer's pools
        _fork("fork_small", 8, 6, 700, 1, 8, 128, 64, "bfloat16"),
        # a beam step of 96 rows over 8 layers
        _fork("fork_beams", 96, 40, 4000, 8, 8, 128, 64, "bfloat16"),
        # a small pool after a few rows left
        _compact("compact_small", 8, 900, 1, 24, 4, 64, 16, "float16"),
        # a fragmented pool of four layers
        _compact("compact_layers", 64, 4000, 4, 700, 8, 128, 64, "bfloat16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "rotary", "fork", "compact"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    page = rng.choice([16, 32, 48, 64, 128, 256])
    dim = rng.choice([64, 128, 128, 128, 256, 16 * rng.randint(1, 16)])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8, 16] if kv_heads <= 2 else [1, 2, 3, 4, 5])
    while True:
        if op == "attend":
            new = rng.choice([1, 1, rng.randint(2, 16), _log(rng, 17, 4096)])
            case = _attend("", _log(rng, 1, 96), new, _log(rng, 1, 24000), heads, kv_heads, dim, page, dtype,
                           rng.random() < 0.8)
            scores = case["rows"] * heads * new * (new + case["past"])
            cache = case["rows"] * (new + case["past"]) * kv_heads * dim
            fits = scores <= 2 << 30 and cache * 2 <= 1 << 30 and scores * dim <= 4e11
        elif op == "rotary":
            new = rng.choice([1, _log(rng, 2, 4096)])
            half = rng.randint(1, dim // 2) if rng.random() < 0.5 else dim // 2
            case = _rotary("", _log(rng, 1, 256), new, _log(rng, 1, 16000), heads, kv_heads, dim,
                           2 * half, rng.random() < 0.5, page, dtype)
            fits = case["rows"] * new * (heads + 2 * kv_heads) * dim <= 16384 * 48 * 128
            fits = fits and case["rows"] * (new + case["past"]) * kv_heads * dim <= 64 * 8192 * 8 * 128
        else:
            layers, past, rows = rng.randint(1, 8), _log(rng, 20, 6000), _log(rng, 2, 96)
            if op == "fork":
                case = _fork("", rows, rng.randint(1, rows), past, layers, kv_heads, dim, page, dtype)
            else:
                moved = rng.randint(0, max(1, rows * past // (4 * page)))
                case = _compact("", rows, past, layers, moved, kv_heads, dim, page, dtype)
            fits = layers * rows * (past + page) * kv_heads * dim <= 8 * 64 * 4000 * 8 * 128
        if fits:
            del case["name"]
            return case


# --- inputs ------------------------------------------------------------------------------------------------------
def _lengths(case):
    """(new tokens, tokens in the cache with them) of every row, by the case's sizes alone. Row 0 has the full
    lengths; where rows have chunks, every third row has a single token."""
    rng = random.Random("%d %d %d" % (case["rows"], case.get("new", 0), case["past"]))
    new, held = [], []
    for b in range(case["rows"]):
        n = case.get("new", 0)
        if n > 1 and b:
            n = 1 if b % 3 == 0 else rng.randint(max(1, n // 4), n)
        new.append(n)
        held.append(n + (case["past"] if b == 0 else rng.randint(case["past"] // 8, case["past"])))
    return new, held


def _pages(length, page):
    return -(-length // page)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def _table(counts, width, ids):
    """[rows, width] page table: the first counts[b] entries of row b take the next of `ids`, the rest are -1."""
    counts = _int32(counts).long()
    column = torch.arange(width, device="cuda")
    first = torch.cumsum(counts, 0) - counts
    at = (first[:, None] + column).clamp_(max=max(0, ids.numel() - 1))
    return torch.where(column < counts[:, None], ids[at], -1).int().contiguous()


def prepare(case, seed):
    gen = _generator(seed)
    dtype, page = DTYPES[case["dtype"]], case["page"]
    new, held = _lengths(case)
    kv_heads, dim = case["kv_heads"], case["dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32 if math.prod(shape) < 1 << 28
                           else dtype).to(dtype)

    counts = [_pages(n, page) for n in held]
    state = {"case": case, "page": page, "max_held": max(held), "max_new": max(new)}
    if case["op"] in ("attend", "rotary"):
        width = max(counts) + 1
        pages = sum(counts) + 3
        state["table"] = _table(counts, width, torch.randperm(pages, generator=gen, device="cuda"))
        state["lens"] = _int32(held)
        state["cu"] = _int32(_offsets(new))
        tokens = sum(new)
        # queries, keys and values come as one product's output, as a fused projection leaves them
        wide = case["heads"] + 2 * kv_heads
        state["qkv"] = normal(tokens, wide, dim)
        state["k_cache"] = normal(pages * page, kv_heads, dim)
        state["v_cache"] = normal(pages * page, kv_heads, dim)
        if case["op"] == "rotary":
            # positions counted twice as dense as trained: linear scaling by two
            turn = torch.arange(case["rotary"] // 2, device="cuda", dtype=torch.float64) * (2.0 / case["rotary"])
            angle = torch.arange(max(held), device="cuda", dtype=torch.float64)[:, None] * (10000.0 ** -turn / 2.0)
            state["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()
        return state

    layers = case["layers"]
    if case["op"] == "fork":
        total = sum(counts) + 2 * case["rows"] + 5  # room for the copies and the new tokens' pages
        ids = torch.randperm(total, generator=gen, device="cuda")
        rng = random.Random(seed)
        winners = rng.sample(range(case["rows"]), case["kept"])
        parents = [b if b in winners else rng.choice(winners) for b in range(case["rows"])]
        parents[rng.randrange(case["rows"])] = -1 if case["rows"] > 2 else parents[0]
        state["parents"] = _int32(parents)
        # one more token each
        state["reserve"] = _int32([held[p] + 1 if p >= 0 else 0 for p in parents])
        width = max(counts) + 2
        state["held_of"] = held
    else:
        live = sum(counts)
        moved = min(case["moved"], live)
        total = live + 2 * moved + 7
        low = torch.randperm(live, generator=gen, device="cuda")[:live - moved]
        high = live + torch.randperm(total - live, generator=gen, device="cuda")[:moved]
        ids = torch.cat([low, high])
        ids = ids[torch.randperm(live, generator=gen, device="cuda")]
        width = max(counts) + 1
    state["pages"] = total
    state["table"] = _table(counts, width, ids)
    state["lens"] = _int32(held)
    state["store"] = normal(2 * layers, total * page, kv_heads, dim)
    state["pools"] = list(state["store"].unbind(0))
    return state


# --- one pass ----------------------------------------------------------------------------------------------------
def run(state):
    return _OPS[state["case"]["op"]][1 if own else 0](state)


def _split(state):
    """The queries, keys and values as views of the projection's output."""
    h, kv = state["case"]["heads"], state["case"]["kv_heads"]
    qkv = state["qkv"]
    return qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:]


def _attend_own(state):
    from fgw_b200.operators.mha.chunk_attention import paged_chunk_attention
    q, _, _ = _split(state)
    return paged_chunk_attention(q, state["k_cache"], state["v_cache"], state["table"], state["lens"], state["cu"],
                                 state["page"], is_causal=state["case"]["causal"])


def _attend_plain(state):
    case, page = state["case"], state["page"]
    q, _, _ = _split(state)
    cu, lens = state["cu"].long(), state["lens"].long()
    tokens, heads, dim = q.shape
    kv, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    n = cu[1:] - cu[:-1]
    i = torch.arange(state["max_new"], device="cuda")
    j = torch.arange(state["max_held"], device="cuda")
    row = (cu[:-1, None] + i).clamp(max=tokens - 1)                        # [B, N] token of each place
    place = state["table"].long()[:, j // page].clamp(min=0) * page + j % page  # [B, L] cache row of each position
    live = j < lens[:, None]
    k = torch.where(live[..., None, None], state["k_cache"][place].float(), 0.0)
    v = torch.where(live[..., None, None], state["v_cache"][place].float(), 0.0)
    qs = q[row].float().reshape(len(n), -1, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(len(n), kv, -1, dim)
    seen = lens[:, None].expand(-1, i.numel())
    if case["causal"]:
        seen = lens[:, None] - n[:, None] + i + 1                           # [B, N] keys each place sees
    hidden = j >= seen[..., None]                                            # [B, N, L]
    scores = torch.matmul(qs, k.permute(0, 2, 3, 1)).mul_(1.0 / math.sqrt(dim))
    by_place = scores.view(len(n), kv, group, i.numel(), j.numel())
    by_place.masked_fill_(hidden[:, None, None], -math.inf)
    top = by_place.amax(-1, keepdim=True)
    by_place.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = by_place.sum(-1, keepdim=True)
    out = torch.matmul(scores, v.permute(0, 2, 1, 3)).view(len(n), kv, group, i.numel(), dim)
    out = out / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(len(n), i.numel(), heads, dim)
    token = torch.arange(tokens, device="cuda")
    b = torch.searchsorted(cu, token, right=True) - 1
    return out[b, token - cu[b]].to(q.dtype)


def _rotary_own(state):
    from fgw_b200.operators.mha.rotary_append import rotary_append
    q, k, v = _split(state)
    out = rotary_append(q, k, v, state["k_cache"], state["v_cache"], state["table"], state["lens"], state["cu"],
                        state["cos_sin"], state["page"], interleaved=state["case"]["interleaved"])
    return out, state["k_cache"], state["v_cache"]


def _turn(x, cos, sin, rotary, interleaved):
    """Rotates the first `rotary` values of each head, in 32 bits, rounded once."""
    y = x.float()
    r, rest = y[..., :rotary], y[..., rotary:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rotary // 2], r[..., rotary // 2:])
    c, d = a * cos - b * sin, b * cos + a * sin
    r = torch.stack([c, d], -1).flatten(-2) if interleaved else torch.cat([c, d], -1)
    return torch.cat([r, rest], -1).to(x.dtype)


def _rotary_plain(state):
    case, page = state["case"], state["page"]
    q, k, v = _split(state)
    cu, lens = state["cu"].long(), state["lens"].long()
    token = torch.arange(q.shape[0], device="cuda")
    b = torch.searchsorted(cu, token, right=True) - 1
    at = lens[b] - cu[b + 1] + token
    place = state["table"].long()[b, at // page] * page + at % page
    half = case["rotary"] // 2
    cos, sin = state["cos_sin"][at, None, :half], state["cos_sin"][at, None, half:]
    state["k_cache"][place] = _turn(k, cos, sin, case["rotary"], case["interleaved"])
    state["v_cache"][place] = v
    return _turn(q, cos, sin, case["rotary"], case["interleaved"]), state["k_cache"], state["v_cache"]


def _fork_own(state):
    from fgw_b200.operators.mha.page_ops import fork_pages
    table, lens, status = fork_pages(state["pools"], state["table"], state["lens"], state["parents"], state["page"],
                                     reserve_seqlens=state["reserve"])
    return table, lens, status, state["store"]


def _fork_plain(state):
    table, page, pages = state["table"].long(), state["page"], state["pages"]
    parents = state["parents"].long()
    rows, width = table.shape
    row, column = torch.arange(rows, device="cuda"), torch.arange(width, device="cuda")
    kept = parents >= 0
    parent = parents.clamp(min=0)
    lens = torch.where(kept, state["lens"].long()[parent], 0)
    room = torch.where(kept, torch.maximum(state["reserve"].long(), lens), 0)
    full, held, want = lens // page, (lens + page - 1) // page, (room + page - 1) // page
    # of the rows with one parent the first keeps the partly filled page, the others copy it
    first = torch.full((rows,), rows, device="cuda").scatter_reduce(0, parent, torch.where(kept, row, rows), "amin")
    copies = kept & (lens % page > 0) & (first[parent] != row)
    source = table[parent]
    is_held = column < held[:, None]
    used = torch.zeros(pages + 1, dtype=torch.bool, device="cuda")
    used[torch.where(is_held, source, pages)] = True
    used = used[:pages]
    is_copy = copies[:, None] & (column == full[:, None])
    is_new = is_copy | ((column >= held[:, None]) & (column < want[:, None]))
    order = torch.cumsum(is_new.flatten(), 0).view(rows, width) - 1
    free = torch.argsort(used.int(), stable=True)
    needed, available = is_new.sum(), pages - used.sum()
    fits = needed <= available
    fresh = free[order.clamp(0, pages - 1)]
    after = torch.where(is_new, fresh, torch.where(is_held, source, -1))
    new_table = torch.where(fits, after, table).int()
    new_lens = torch.where(fits, lens, state["lens"].long()).int()
    # the filled rows of the copied pages, in every pool
    at = torch.nonzero(copies & fits)[:, 0]
    src, dst, rows_in = source[at, full[at]], after[at, full[at]], lens[at] % page
    pools = state["store"].view(state["store"].shape[0], pages, page, -1)
    filled = (torch.arange(page, device="cuda") < rows_in[:, None])[None, :, :, None]
    pools[:, dst] = torch.where(filled, pools[:, src], pools[:, dst])
    return new_table, new_lens, torch.stack([needed, available]).int(), state["store"]


def _compact_own(state):
    from fgw_b200.operators.mha.page_ops import compact_pages
    table, status = compact_pages(state["pools"], state["table"], state["lens"], state["page"])
    return table, status, state["store"]


def _compact_plain(state):
    table, page, pages = state["table"].long(), state["page"], state["pages"]
    column = torch.arange(table.shape[1], device="cuda")
    is_held = column < ((state["lens"].long() + page - 1) // page)[:, None]
    used = torch.zeros(pages + 1, dtype=torch.bool, device="cuda")
    used[torch.where(is_held, table, pages)] = True
    used = used[:pages]
    live = used.sum()
    at = torch.arange(pages, device="cuda")
    moves = used & (at >= live)
    # the k-th used page past the live count goes to the k-th free page below it
    free = torch.argsort((used | (at >= live)).int(), stable=True)
    to = torch.where(moves, free[(torch.cumsum(moves, 0) - 1).clamp(min=0)], at)
    new_table = torch.where(is_held, to[table.clamp(min=0)], -1).int()
    src = torch.nonzero(moves)[:, 0]
    pools = state["store"].view(state["store"].shape[0], pages, page, -1)
    pools[:, to[src]] = pools[:, src]
    return new_table, torch.stack([live, moves.sum()]).int(), state["store"]


_OPS = {"attend": (_attend_plain, _attend_own), "rotary": (_rotary_plain, _rotary_own),
        "fork": (_fork_plain, _fork_own), "compact": (_compact_plain, _compact_own)}


# --- what a pass cannot do without -------------------------------------------------------------------------------
def work(case):
    new, held = _lengths(case)
    kv, dim, page = case["kv_heads"], case["dim"], case["page"]
    token = kv * dim * 2  # bytes of one token's keys, or values, in the cache
    if case["op"] == "attend":
        pairs = sum(n * h - (n * (n - 1) // 2 if case["causal"] else 0) for n, h in zip(new, held))
        moved = sum(held) * 2 * token + 2 * sum(new) * case["heads"] * dim * 2
        return {"bytes": moved + sum(4 * _pages(h, page) + 8 for h in held), "flops": 4 * case["heads"] * dim * pairs}
    if case["op"] == "rotary":
        values = sum(new) * (case["heads"] + 2 * kv) * dim
        turned = sum(new) * (case["heads"] + kv) * case["rotary"]
        return {"bytes": 4 * values + 4 * sum(new) * case["rotary"], "flops": 3 * turned}
    entries = sum(_pages(h, page) for h in held)
    if case["op"] == "fork":
        # a copied page is on average filled as the rows' last pages are
        copied = max(0, case["rows"] - case["kept"] - 1) * sum(h % page for h in held) / len(held)
        return {"bytes": int(2 * copied * token * 2 * case["layers"]) + 8 * entries, "flops": 0}
    moved = min(case["moved"], entries)
    return {"bytes": 2 * moved * page * token * 2 * case["layers"] + 8 * entries, "flops": 0}


# --- the definitions, in 64 bits ---------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    new, held = _lengths(case)
    page, table = case["page"], state["table"].cpu().tolist()
    if case["op"] in ("fork", "compact"):
        return _exact_pages(case, state, held, table)
    q, k, v = _split(state)
    starts = _offsets(new)
    if case["op"] == "attend":
        group = case["heads"] // case["kv_heads"]
        out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        for b, (n, h) in enumerate(zip(new, held)):
            rows = torch.cat([torch.arange(p * page, p * page + page) for p in table[b][:_pages(h, page)]])[:h].cuda()
            hide = torch.ones(n, h, dtype=torch.bool, device="cuda").triu(h - n + 1) if case["causal"] else None
            for g in range(case["kv_heads"]):
                keys, values = state["k_cache"][rows, g].double(), state["v_cache"][rows, g].double()
                mine = q[starts[b]:starts[b + 1], g * group:(g + 1) * group].double()
                for head in range(group):
                    s = mine[:, head] @ keys.T / case["dim"] ** 0.5
                    if hide is not None:
                        s[hide] = -math.inf
                    out[starts[b]:starts[b + 1], g * group + head] = torch.softmax(s, -1) @ values
        return out
    half = case["rotary"] // 2
    dst = torch.tensor([table[b][p // page] * page + p % page for b, (n, h) in enumerate(zip(new, held))
                        for p in range(h - n, h)], device="cuda")
    where = torch.tensor([p for n, h in zip(new, held) for p in range(h - n, h)], device="cuda")
    turn = torch.complex(state["cos_sin"][where, :half].double(), state["cos_sin"][where, half:].double())[:, None]

    def turned(x):
        x = x.double()
        step = 2 if case["interleaved"] else 1
        one = torch.arange(half, device="cuda") * step
        two = one + (1 if case["interleaved"] else half)
        z = torch.complex(x[..., one], x[..., two]) * turn
        x[..., one], x[..., two] = z.real, z.imag
        return x

    keys, values = state["k_cache"].double(), state["v_cache"].double()
    keys[dst], values[dst] = turned(k), v.double()
    return turned(q), keys, values


def _exact_pages(case, state, held, table):
    """The page tables by plain lists, and the pools' values page by page (not of the large pools, whose copies have no
    other value in 64 bits)."""
    page, pages = case["page"], state["pages"]
    width = len(table[0])

    def stored(copies):
        if state["store"].numel() > 1 << 28:
            return None
        before = state["store"].double()
        after = before.clone()
        for src, dst, filled in copies:
            after[:, dst * page:dst * page + filled] = before[:, src * page:src * page + filled]
        return after

    if case["op"] == "compact":
        used = sorted({p for row, h in zip(table, held) for p in row[:_pages(h, page)]})
        holes = sorted(set(range(len(used))) - set(used))
        to = dict(zip([p for p in used if p >= len(used)], holes))
        after = [[to.get(p, p) for p in row[:_pages(h, page)]] for row, h in zip(table, held)]
        after = [row + [-1] * (width - len(row)) for row in after]
        return _int32(after), _int32([len(used), len(to)]), stored([(p, q, page) for p, q in to.items()])
    parents, reserve = state["parents"].tolist(), state["reserve"].tolist()
    lens = [held[p] if p >= 0 else 0 for p in parents]
    used = {e for p, h in zip(parents, lens) if p >= 0 for e in table[p][:_pages(h, page)]}
    free = [e for e in range(pages) if e not in used]
    after, given, seen, copies = [], 0, set(), []
    for p, h, room in zip(parents, lens, reserve):
        row = list(table[p][:_pages(h, page)]) if p >= 0 else []
        if h % page and p in seen:
            copies.append((row[-1], free[given], h % page))
            row[-1] = free[given]
            given += 1
        seen.add(p)
        while p >= 0 and len(row) < _pages(room, page):
            row.append(free[given])
            given += 1
        after.append(row + [-1] * (width - len(row)))
    return _int32(after), _int32(lens), _int32([given, len(free)]), stored(copies)
