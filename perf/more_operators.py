"""Performance cases of whole-prompt serving: prompts of different lengths packed
into one call, and the pages of the cache that they are written to.

  attention  ``packed_attention_hip``: causal attention over whole prompts, packed
  resize     ``paged_resize_hip``: every sequence gets the pages that its length
             needs, and gives up those that it does not
  fork       ``paged_fork_hip``: the next batch is made of copies of this one's
             sequences (samples of one prompt, beams), full pages shared
  compact    ``paged_compact_hip``: the pages in use move to the front of the pool

Rows are packed: sequence b's tokens are rows ``cu_rows[b]`` up to
``cu_rows[b + 1]``.  A pool is [layers, pages, kv_heads, page_size, head_dim];
``page_users[p]`` counts what names page p.  Shapes are Qwen2-1.5B's (12 query and
2 key/value heads of 128) or generic ones; ``draw`` spreads over the same ranges.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

_PACKAGE = Path(__file__).resolve().parents[1] / "qwen2-int4-systems_amd"
if str(_PACKAGE) not in sys.path:
    sys.path.insert(0, str(_PACKAGE))

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one short question of an interactive user: the smallest prompt
        {"name": "attention_1x37", "op": "attention", "batch": 1, "rows_lo": 37, "rows_hi": 37, "heads": 12,
         "kv_heads": 2, "dim": 128, "dtype": "bf16"},
        # the 512-token prompt of the end-to-end benchmark
        {"name": "attention_1x512", "op": "attention", "batch": 1, "rows_lo": 512, "rows_hi": 512, "heads": 12,
         "kv_heads": 2, "dim": 128, "dtype": "bf16"},
        # eight prompts of unequal length, packed: 8 K rows in all
        {"name": "attention_8x1000", "op": "attention", "batch": 8, "rows_lo": 37, "rows_hi": 2011, "heads": 12,
         "kv_heads": 2, "dim": 128, "dtype": "bf16"},
        # many short texts, down to one token; heads of 64, each with keys of its own
        {"name": "attention_96x60_d64", "op": "attention", "batch": 96, "rows_lo": 1, "rows_hi": 119, "heads": 16,
         "kv_heads": 16, "dim": 64, "dtype": "fp16"},
        # three documents of a larger head layout
        {"name": "attention_3x4001", "op": "attention", "batch": 3, "rows_lo": 1003, "rows_hi": 6999, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "fp16"},
        # one long document: the largest
        {"name": "attention_1x16384", "op": "attention", "batch": 1, "rows_lo": 16384, "rows_hi": 16384,
         "heads": 12, "kv_heads": 2, "dim": 128, "dtype": "bf16"},
        # a decode step's growth: 64 sequences with up to five new tokens each, few of them in need of a page
        {"name": "resize_64x2048", "op": "resize", "batch": 64, "width": 128, "pages": 8192, "page": 16,
         "shared": 3, "step": 5, "turnover": 0.05},
        # a large server's tables: contexts of up to 32 K, every third sequence ended, begun or cut back
        {"name": "resize_511x32768", "op": "resize", "batch": 511, "width": 2048, "pages": 600_000, "page": 16,
         "shared": 64, "step": 1000, "turnover": 0.33},
        # eight samples of one prompt: seven copies of its last page
        {"name": "fork_1to8", "op": "fork", "batch": 1, "alive": 1, "fan": 8, "past_lo": 575, "past_hi": 575,
         "width": 64, "pages": 256, "page": 16, "layers": 1, "kv_heads": 2, "dim": 128, "token_major": False,
         "dtype": "bf16"},
        # beam search over 64 requests: half of the beams end, the others have three continuations
        {"name": "fork_64to96", "op": "fork", "batch": 64, "alive": 32, "fan": 3, "past_lo": 100, "past_hi": 1003,
         "width": 129, "pages": 4000, "page": 16, "layers": 8, "kv_heads": 2, "dim": 128, "token_major": False,
         "dtype": "bf16"},
        # a small pool after a few requests ended
        {"name": "compact_250", "op": "compact", "batch": 8, "width": 32, "pages": 250, "live": 150, "page": 16,
         "layers": 1, "kv_heads": 2, "dim": 128, "token_major": False, "dtype": "bf16"},
        # a pool of eight layers whose load fell to less than half, before its end is given back
        {"name": "compact_4000", "op": "compact", "batch": 64, "width": 128, "pages": 4000, "live": 1700, "page": 16,
         "layers": 8, "kv_heads": 2, "dim": 128, "token_major": True, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "resize", "fork", "compact"])
    if op == "attention":
        heads, kv_heads = rng.choice([(12, 2), (12, 2), (14, 2), (16, 16), (16, 4), (32, 8), (8, 1), (9, 3)])
        batch = _log_int(rng, 1, 128)
        low = _log_int(rng, 1, 4096)
        case = {"op": op, "batch": batch, "rows_lo": low, "rows_hi": low * rng.choice([1, 2, 5]), "heads": heads,
                "kv_heads": kv_heads, "dim": rng.choice([128, 128, 64]), "dtype": rng.choice(["bf16", "bf16", "fp16"])}
        # (below the largest listed case's products, and what the plain form holds at once)
        fits = batch * heads * case["rows_hi"] ** 2 < 12 * 16384 ** 2 // 2
        return case if fits and batch * case["rows_hi"] < 40_000 else draw(rng)
    page = rng.choice([16, 16, 32, 64])
    batch = _log_int(rng, 1, 256)
    if op == "resize":
        width = _log_int(rng, 4, 1024)
        return {"op": op, "batch": batch, "width": width, "pages": batch * width + rng.randint(0, 3000), "page": page,
                "shared": rng.randint(0, width // 4), "step": _log_int(rng, 1, 4 * page * (1 + width // 16)),
                "turnover": rng.choice([0.0, 0.05, 0.4])}
    case = {"op": op, "page": page, "layers": rng.choice([1, 2, 4, 8]), "kv_heads": rng.choice([1, 2, 2, 8]),
            "dim": rng.choice([128, 128, 64]), "token_major": rng.random() < 0.3, "dtype": rng.choice(["bf16", "fp16"])}
    most = 60_000_000 // (case["layers"] * case["kv_heads"] * page * case["dim"])  # pages, of the pool's size
    if op == "fork":
        batch = _log_int(rng, 1, max(1, min(128, most // 8)))
        alive, fan = rng.randint(1, batch), rng.choice([1, 2, 2, 4])
        past = _log_int(rng, 1, max(1, (most - alive * fan) * page // (batch * 2)))
        width = -(-past // page) + rng.randint(0, 9)
        pages = batch * -(-past // page) + alive * fan + rng.randint(0, 40)
        case |= {"batch": batch, "alive": alive, "fan": fan, "past_lo": rng.randint(0, past), "past_hi": past,
                 "width": width, "pages": pages}
        return case if pages <= most + 40 else draw(rng)
    pages = _log_int(rng, 2, max(2, min(4000, most)))
    live = rng.randint(1, pages)
    batch = min(batch, live)
    case |= {"pages": pages, "live": live, "batch": batch, "width": -(-live // batch) + rng.randint(0, 9)}
    return case


def _spread(lo, hi, count):
    """`count` whole numbers from lo to hi, evenly apart."""
    return [lo + (hi - lo) * i // max(1, count - 1) for i in range(count)]


def _pool(case, gen):
    shape = (case["layers"], case["pages"], case["kv_heads"], case["page"], case["dim"])
    if case["token_major"]:
        shape = (shape[0], shape[1], shape[3], shape[2], shape[4])
    pool = torch.randn(shape, generator=gen, device="cuda", dtype=DTYPES[case["dtype"]])
    return pool.transpose(2, 3) if case["token_major"] else pool


def _table(case, held, free, shared=()):
    """Rows of `held[b]` pages each: the shared ones, then pages taken from `free`."""
    table = torch.full((len(held), case["width"]), -1, dtype=torch.int32)
    at, common = 0, len(shared)
    for b, count in enumerate(held):
        first = min(common, count)
        table[b, :first] = torch.as_tensor(shared[:first], dtype=torch.int32)
        table[b, first:count] = free[at:at + count - first]
        at += count - first
    return table


def _users(table, pages):
    return torch.bincount(table[table >= 0].long(), minlength=pages).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    state = {"case": case}
    if case["op"] == "attention":
        lengths = _spread(case["rows_lo"], case["rows_hi"], case["batch"])
        lengths = [lengths[i] for i in torch.randperm(case["batch"], generator=host).tolist()]
        state["cu_rows"] = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda()
        heads, kv_heads = case["heads"], case["kv_heads"]
        # the fused q|k|v projection's rows; its parts are views, the queries and keys rotated in place
        qkv = torch.randn((sum(lengths), heads + 2 * kv_heads, case["dim"]), generator=gen, device="cuda")
        qkv[:, :heads] *= 1.5
        state["q"], state["k"], state["v"] = qkv.to(DTYPES[case["dtype"]]).split((heads, kv_heads, kv_heads), dim=1)
        return state
    page, width, pages, batch = case["page"], case["width"], case["pages"], case["batch"]
    free = torch.randperm(pages, generator=host).to(torch.int32)
    if case["op"] == "resize":
        shared = case["shared"]
        reach = width * page
        before = torch.randint(shared * page, max(shared * page, reach - case["step"]) + 1, (batch,), generator=host)
        after = (before + torch.randint(1, case["step"] + 1, (batch,), generator=host)).clamp_max(reach)
        # sequences that end, that begin, that are cut back
        kind, share = torch.rand(batch, generator=host), case["turnover"] / 3
        after[kind < share] = 0
        before[(kind >= share) & (kind < 2 * share)] = 0
        cut = (kind >= 2 * share) & (kind < 3 * share)
        after[cut] = (before[cut].double() * torch.rand(int(cut.sum()), generator=host)).long()
        table = _table(case, ((before + page - 1) // page).tolist(), free[shared:], free[:shared].tolist())
        users = _users(table, pages)
        users[free[:shared].long()] += 1  # a prefix that stays cached without a sequence
        return state | {"table": table.cuda(), "lengths": after.to(torch.int32).cuda(), "users": users.cuda()}
    state["k_pages"], state["v_pages"] = _pool(case, gen), _pool(case, gen)
    if case["op"] == "fork":
        past = _spread(case["past_lo"], case["past_hi"], batch)
        row = torch.randperm(batch, generator=host)  # where each length's sequence lies
        lengths = torch.zeros(batch, dtype=torch.int64)
        lengths[row] = torch.tensor(past)
        table = _table(case, ((lengths + page - 1) // page).tolist(), free)
        # every second length lives on, then those between
        alive = torch.cat((row[::2], row[1::2]))[:case["alive"]].repeat(case["fan"])
        parents = alive[torch.randperm(len(alive), generator=host)].to(torch.int32)
        return state | {"table": table.cuda(), "lengths": lengths.to(torch.int32).cuda(), "parents": parents.cuda(),
                        "users": _users(table, pages).cuda()}
    live = case["live"]
    moving = _moving(case)
    # `moving` of the pool's first `live` pages are free, as many behind them in use
    kept = torch.randperm(live, generator=host)[moving:]
    behind = live + torch.randperm(pages - live, generator=host)[:moving]
    used = torch.cat((kept, behind))
    used = used[torch.randperm(live, generator=host)].to(torch.int32)
    held = [(live - b + batch - 1) // batch for b in range(batch)]
    table = _table(case, held, used)
    return state | {"table": table.cuda(), "users": _users(table, pages).cuda()}


def _moving(case):
    """Pages that a compaction moves, if those in use lie anywhere."""
    live, pages = case["live"], case["pages"]
    return min(live, pages - live, max(1, round(live * (pages - live) / pages)))


def _plain_attention(state):
    case, q = state["case"], state["q"]
    batch, heads, kv_heads, dim = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    longest = max(case["rows_lo"], case["rows_hi"])
    cu = state["cu_rows"].long()
    row = torch.arange(q.shape[0], device=q.device)
    seq = (row.view(-1, 1) >= cu[1:].view(1, -1)).sum(dim=1)
    place = row - cu[seq]

    def padded(x):  # [kv_heads, batch, heads of it * positions, dim], 32 bits
        full = torch.zeros((batch, longest, x.shape[1], dim), device=q.device)
        full[seq, place] = x.float()
        return full.view(batch, longest, kv_heads, -1, dim).permute(2, 0, 3, 1, 4).reshape(kv_heads, batch, -1, dim)

    scores = torch.matmul(padded(q) * dim ** -0.5, padded(state["k"]).transpose(2, 3).contiguous())
    key = torch.arange(longest, device=q.device)
    hidden = key.view(1, -1) > key.view(-1, 1)
    scores.view(kv_heads, batch, -1, longest, longest).masked_fill_(hidden, float("-inf"))
    weight = scores.sub_(scores.amax(dim=-1, keepdim=True)).exp_()
    out = torch.matmul(weight, padded(state["v"])) / weight.sum(dim=-1, keepdim=True)
    out = out.view(kv_heads, batch, -1, longest, dim).permute(1, 3, 0, 2, 4)[seq, place]
    return out.reshape(q.shape).to(q.dtype)


def _held(table, pages):
    """Entries of each row before its first that names no page."""
    return ((table >= 0) & (table < pages)).long().cumprod(dim=1).sum(dim=1)


def _free_pages(users):
    """The free pages from the lowest on, then -1."""
    pages = users.shape[0]
    free = users == 0
    order = torch.full((pages + 1,), -1, dtype=torch.int64, device=users.device)
    order.scatter_(0, torch.where(free, free.long().cumsum(0) - 1, pages), torch.arange(pages, device=users.device))
    order[pages:] = -1
    return order


def _add_users(users, table, valid, sign):
    # (entries that are not valid add nothing, each to a page of its own, so that they do not queue up at one)
    nothing = torch.arange(table.numel(), device=table.device).view(table.shape) % users.shape[0]
    return users.index_add(0, torch.where(valid, table, nothing).flatten(), sign * valid.flatten().to(users.dtype))


def _plain_resize(state):
    table, users, page = state["table"].long(), state["users"], state["case"]["page"]
    pages, width = users.shape[0], table.shape[1]
    column = torch.arange(width, device=table.device).view(1, -1)
    held = _held(table, pages)
    need = (state["lengths"].long().clamp_min(0) + page - 1) // page
    keep = torch.minimum(held, need)
    want = need.clamp_max(width) - keep
    kept = column < keep.view(-1, 1)
    new = ~kept & (column < need.view(-1, 1))
    rank = (want.cumsum(0) - want - keep).view(-1, 1) + column
    given = torch.where(new, _free_pages(users)[rank.clamp(0, pages)], -1)
    out = torch.where(kept, table, given)
    after = _add_users(users, table, ~kept & (column < held.view(-1, 1)), -1)
    after = _add_users(after, given, given >= 0, 1)
    return out.to(torch.int32), after, (need - (out >= 0).sum(dim=1)).to(torch.int32)


def _plain_fork(state):
    table, users, page = state["table"].long(), state["users"], state["case"]["page"]
    lengths, parents = state["lengths"].long().clamp_min(0), state["parents"].long()
    pages, (batch, width) = users.shape[0], table.shape
    column = torch.arange(width, device=table.device).view(1, -1)
    there = (parents >= 0) & (parents < batch)
    parent = parents.clamp(0, batch - 1)
    held = _held(table, pages)
    need = (lengths + page - 1) // page
    used = torch.minimum(held, need)
    out = torch.where(there.view(-1, 1) & (column < used[parent].view(-1, 1)), table[parent], -1)
    # the last page, not full: the first child takes it where nobody else names it, the others get a copy
    partial = (lengths % page != 0) & (held >= need)
    last = (need - 1).clamp_min(0)
    source = table.gather(1, last.view(-1, 1)).squeeze(1).clamp(0, pages - 1)
    earlier = (parents.view(-1, 1) == parents.view(1, -1)).tril(-1).any(dim=1)
    copies = there & partial[parent] & (earlier | (users[source] != 1)[parent])
    target = _free_pages(users)[(copies.long().cumsum(0) - 1).clamp(0, pages)]
    out = torch.where(copies.view(-1, 1) & (column == last[parent].view(-1, 1)), target.view(-1, 1), out)
    after = _add_users(users, table, column < held.view(-1, 1), -1)
    after = _add_users(after, out, out >= 0, 1)
    missing = copies & (target < 0)
    # rows that copy nothing repeat the first copy (or copy a page to itself, where there is none)
    does = copies & (target >= 0)
    which = torch.where(does, torch.arange(len(does), device=does.device), does.long().argmax())
    some = does.any()
    a = torch.where(some, source[parent][which], 0)
    b = torch.where(some, target[which], 0)
    count = (lengths % page)[parent][which]
    filled = torch.arange(page, device=table.device).view(1, 1, 1, -1, 1) < count.view(1, -1, 1, 1, 1)
    for pool in (state["k_pages"], state["v_pages"]):
        pool[:, b] = torch.where(filled, pool[:, a], pool[:, b])
    return (out.to(torch.int32), torch.where(there, lengths[parent], 0).to(torch.int32), after,
            missing.to(torch.int32), state["k_pages"], state["v_pages"])


def _plain_compact(state):
    table, users = state["table"].long(), state["users"]
    pages = users.shape[0]
    page = torch.arange(pages, device=table.device)
    live = users != 0
    count = live.sum()
    hole = ~live & (page < count)
    moves = live & (page >= count)
    holes = torch.full((pages + 1,), -1, dtype=torch.int64, device=table.device)
    holes.scatter_(0, torch.where(hole, hole.long().cumsum(0) - 1, pages), page)
    to = torch.where(live, torch.where(moves, holes[(moves.long().cumsum(0) - 1).clamp_min(0)], page), -1)
    # a hole takes the page that moves there, every other page keeps what it holds
    filled = torch.zeros((pages + 1,), dtype=torch.int64, device=table.device)
    filled.scatter_(0, torch.where(moves, to, pages), page)
    source = torch.where(hole, filled[:pages], page)
    named = (table >= 0) & (table < pages)
    out = torch.where(named, to[table.clamp(0, pages - 1)], -1)
    after = torch.where(page < count, users[source], 0)
    for pool in (state["k_pages"], state["v_pages"]):
        pool.copy_(pool[:, source])
    return out.to(torch.int32), after, to.to(torch.int32), state["k_pages"], state["v_pages"]


def run(state):
    op = state["case"]["op"]
    if op == "attention":
        if own:
            from qwen_int4_hip import packed_attention_hip

            return packed_attention_hip(state["q"], state["k"], state["v"], state["cu_rows"])
        return _plain_attention(state)
    if op == "resize":
        if own:
            from qwen_int4_hip import paged_resize_hip

            return paged_resize_hip(state["table"], state["lengths"], state["users"],
                                    page_size=state["case"]["page"])
        return _plain_resize(state)
    if op == "fork":
        if own:
            from qwen_int4_hip import paged_fork_hip

            return *paged_fork_hip(state["k_pages"], state["v_pages"], state["table"], state["lengths"],
                                   state["users"], state["parents"]), state["k_pages"], state["v_pages"]
        return _plain_fork(state)
    if own:
        from qwen_int4_hip import paged_compact_hip

        return *paged_compact_hip(state["k_pages"], state["v_pages"], state["table"], state["users"]), \
            state["k_pages"], state["v_pages"]
    return _plain_compact(state)


def work(case):
    if case["op"] == "attention":
        lengths = _spread(case["rows_lo"], case["rows_hi"], case["batch"])
        heads, kv_heads, dim, total = case["heads"], case["kv_heads"], case["dim"], sum(lengths)
        return {"bytes": 2 * total * (2 * heads + 2 * kv_heads) * dim + 4 * (case["batch"] + 1),
                "flops": 4 * sum(n * (n + 1) // 2 for n in lengths) * heads * dim}
    batch, width, pages = case["batch"], case["width"], case["pages"]
    if case["op"] == "resize":  # table and counts read and written
        return {"bytes": 8 * batch * width + 8 * pages + 8 * batch, "flops": batch * width + pages}
    position = 4 * case["layers"] * case["kv_heads"] * case["dim"]  # bytes of a key and a value, all layers
    if case["op"] == "fork":
        past, page, rows = _spread(case["past_lo"], case["past_hi"], batch), case["page"], case["alive"] * case["fan"]
        lasts = [n % page for n in (past[::2] + past[1::2])[:case["alive"]]]
        return {"bytes": 4 * (batch + rows) * width + 8 * pages + 4 * batch + 12 * rows
                + 2 * position * (case["fan"] - 1) * sum(lasts), "flops": rows * width + pages}
    return {"bytes": 8 * batch * width + 12 * pages + 2 * position * case["page"] * _moving(case),
            "flops": batch * width + pages}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "attention":
        cu, q = state["cu_rows"].tolist(), state["q"]
        group = case["heads"] // case["kv_heads"]
        out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        for first, end in zip(cu, cu[1:]):
            for head in range(case["heads"]):
                k, v = (state[name][first:end, head // group].double() for name in ("k", "v"))
                for at in range(first, end, 2048):  # rows at a time
                    upto = min(at + 2048, end)
                    logits = q[at:upto, head].double() @ k[:upto - first].T / math.sqrt(case["dim"])
                    later = torch.ones_like(logits, dtype=torch.bool).triu(at - first + 1)
                    out[at:upto, head] = torch.softmax(logits.masked_fill(later, -math.inf), dim=-1) @ v[:upto - first]
        return out

    users = state["users"].tolist()
    table = state["table"].tolist()
    width = case["width"]
    free = [p for p, n in enumerate(users) if n == 0]

    def answer(*values):
        return tuple(torch.tensor(v, dtype=torch.int32, device="cuda") for v in values)

    if case["op"] == "compact":
        live = [p for p, n in enumerate(users) if n]
        to = [-1] * len(users)
        holes = iter([p for p in free if p < len(live)])
        k_pages, v_pages = state["k_pages"].double(), state["v_pages"].double()
        for p in live:
            to[p] = p if p < len(live) else next(holes)
            if to[p] != p:
                for pool in (k_pages, v_pages):
                    pool[:, to[p]] = pool[:, p]
        after = [0] * len(users)
        for p in live:
            after[to[p]] = users[p]
        return *answer([[to[e] if e >= 0 else -1 for e in row] for row in table], after, to), k_pages, v_pages

    lengths, page = state["lengths"].tolist(), case["page"]
    free = iter(free)
    if case["op"] == "resize":
        missing = []
        for row, length in zip(table, lengths):
            need = -(-max(length, 0) // page)
            for c in range(width):
                if c >= need and row[c] >= 0:
                    users[row[c]] -= 1
                    row[c] = -1
                elif c < need and row[c] < 0:
                    row[c] = next(free, -1)
                    if row[c] >= 0:
                        users[row[c]] += 1
            missing.append(need - sum(e >= 0 for e in row))
        return answer(table, users, missing)

    k_pages, v_pages = state["k_pages"].double(), state["v_pages"].double()
    rows, sizes, missing, taken, after = [], [], [], set(), list(users)
    for row in table:
        for e in row:
            if e >= 0:
                after[e] -= 1
    for parent in state["parents"].tolist():
        length, row = lengths[parent], list(table[parent])
        at, rest = divmod(length, page)
        lacks = 0
        if rest:
            if parent in taken or users[row[at]] != 1:
                source, row[at] = row[at], next(free, -1)
                if row[at] >= 0:
                    for pool in (k_pages, v_pages):
                        pool[:, row[at], :, :rest] = pool[:, source, :, :rest]
                else:
                    lacks = 1
            taken.add(parent)
        for e in row:
            if e >= 0:
                after[e] += 1
        rows.append(row)
        sizes.append(length)
        missing.append(lacks)
    return *answer(rows, sizes, after, missing), k_pages, v_pages
