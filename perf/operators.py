"""Performance cases of the paged serving operators: a speculative serving
step over a paged key/value cache.

  append     ``paged_append_hip``: rotate the new rows' queries and keys, write
             keys and values into the cache's pages
  attention  ``paged_attention_hip``: attention of the new rows over pages, the
             leading ones common to the whole batch
  verify     ``verify_drafts_hip``: which drafted tokens stand, and the token
             that follows them

Rows are packed: sequence b's new positions are rows ``cu_rows[b]`` up to
``cu_rows[b + 1]``, and they are the last ones of its ``lengths[b]`` cached
positions.  Shapes are Qwen2-1.5B's (12 query and 2 key/value heads of 128,
vocabulary 151936) or generic ones; ``draw`` spreads over the same ranges.
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

VOCAB, THETA = 151936, 1_000_000.0
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one token of one interactive sequence: the smallest append of a decode loop
        {"name": "append_1row", "op": "append", "batch": 1, "rows_lo": 1, "rows_hi": 1, "past_lo": 575,
         "past_hi": 575, "heads": 12, "kv_heads": 2, "dim": 128, "rotary": 128, "interleaved": False, "page": 16,
         "token_major": False, "dtype": "bf16"},
        # 64 sequences with four drafted tokens each; interleaved pairs over half the head, token-major pages
        {"name": "append_64x5_interleaved", "op": "append", "batch": 64, "rows_lo": 5, "rows_hi": 5, "past_lo": 20,
         "past_hi": 500, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 64, "interleaved": True, "page": 32,
         "token_major": True, "dtype": "fp16"},
        # eight prompts of unequal length, packed: 8 K rows in all
        {"name": "append_prompts_8x1000", "op": "append", "batch": 8, "rows_lo": 37, "rows_hi": 2011, "past_lo": 0,
         "past_hi": 0, "heads": 12, "kv_heads": 2, "dim": 128, "rotary": 128, "interleaved": False, "page": 16,
         "token_major": False, "dtype": "bf16"},
        # one token of one sequence, nothing shared: the smallest attention call
        {"name": "attention_1x576", "op": "attention", "batch": 1, "rows_lo": 1, "rows_hi": 1, "past_lo": 575,
         "past_hi": 575, "shared": 0, "heads": 12, "kv_heads": 2, "dim": 128, "page": 16, "token_major": False,
         "dtype": "bf16"},
        # a serving batch of unequal contexts, one token each
        {"name": "attention_24x1000", "op": "attention", "batch": 24, "rows_lo": 1, "rows_hi": 1, "past_lo": 11,
         "past_hi": 2047, "shared": 0, "heads": 12, "kv_heads": 2, "dim": 128, "page": 16, "token_major": False,
         "dtype": "bf16"},
        # 32 requests that share a 4096-token system prompt, one token each
        {"name": "attention_shared_32x4096", "op": "attention", "batch": 32, "rows_lo": 1, "rows_hi": 1,
         "past_lo": 0, "past_hi": 511, "shared": 256, "heads": 12, "kv_heads": 2, "dim": 128, "page": 16,
         "token_major": False, "dtype": "bf16"},
        # heads of 64, each with keys of its own, 16 requests with up to five drafted tokens, token-major pages
        {"name": "attention_shared_16x2048_d64", "op": "attention", "batch": 16, "rows_lo": 1, "rows_hi": 6,
         "past_lo": 0, "past_hi": 777, "shared": 32, "heads": 16, "kv_heads": 16, "dim": 64, "page": 64,
         "token_major": True, "dtype": "fp16"},
        # prompts continued in pieces beside decoding sequences
        {"name": "attention_pieces_6x400", "op": "attention", "batch": 6, "rows_lo": 1, "rows_hi": 400,
         "past_lo": 0, "past_hi": 1501, "shared": 0, "heads": 12, "kv_heads": 2, "dim": 128, "page": 32,
         "token_major": False, "dtype": "bf16"},
        # 64 requests with four drafted tokens each over a common 16 K document: the largest
        {"name": "attention_shared_64x5x16384", "op": "attention", "batch": 64, "rows_lo": 5, "rows_hi": 5,
         "past_lo": 0, "past_hi": 1000, "shared": 256, "heads": 12, "kv_heads": 2, "dim": 128, "page": 64,
         "token_major": False, "dtype": "bf16"},
        # one sequence's four drafted tokens
        {"name": "verify_1x4", "op": "verify", "batch": 1, "drafts": 4, "vocab": VOCAB, "one_hot": False,
         "dtype": "fp32"},
        # a serving batch, probabilities of the draft model in hand
        {"name": "verify_64x4", "op": "verify", "batch": 64, "drafts": 4, "vocab": VOCAB, "one_hot": False,
         "dtype": "fp32"},
        # drafts copied from the prompt (no draft model), an odd vocabulary, 16-bit probabilities
        {"name": "verify_96x7_copied", "op": "verify", "batch": 96, "drafts": 7, "vocab": 50257, "one_hot": True,
         "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "attention", "verify"])
    if op == "verify":
        vocab = rng.choice([VOCAB, _log_int(rng, 500, VOCAB)])
        drafts = rng.randint(1, 8)
        return {"op": op, "batch": _log_int(rng, 1, max(1, min(256, 48_000_000 // (vocab * drafts)))),
                "drafts": drafts, "vocab": vocab, "one_hot": rng.random() < 0.3,
                "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"])}
    heads, kv_heads = rng.choice([(12, 2), (12, 2), (14, 2), (16, 16), (16, 4), (32, 8), (8, 1), (9, 3)])
    case = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": rng.choice([128, 128, 64]),
            "page": rng.choice([16, 16, 32, 64, 128]), "token_major": rng.random() < 0.3,
            "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    if op == "append":
        batch = _log_int(rng, 1, 64)
        low = _log_int(rng, 1, 8000 // batch)
        past = _log_int(rng, 1, 1000)
        case |= {"batch": batch, "rows_lo": low, "rows_hi": min(max(low, 8000 // batch), low * rng.randint(1, 3)),
                 "past_lo": rng.randint(0, past), "past_hi": past, "rotary": rng.choice([case["dim"], 32]),
                 "interleaved": rng.random() < 0.4}
        return case
    # below the largest listed cases' products and bytes
    batch = _log_int(rng, 1, 64)
    low = rng.choice([1, 1, 1, rng.randint(1, 8), _log_int(rng, 1, 256)])
    high = low * rng.choice([1, 1, 2])
    most = int(16e6 / (batch * high * heads)) + 64
    pages = max(1, min(16384, most) // case["page"])
    past = _log_int(rng, 16, max(16, min(4000, most, 7_500_000 // (batch * kv_heads * case["dim"]))))
    case |= {"batch": batch, "rows_lo": low, "rows_hi": high, "past_lo": rng.randint(0, past), "past_hi": past,
             "shared": rng.choice([0, _log_int(rng, 1, pages), _log_int(rng, max(1, pages // 16), pages)])}
    cost = work(case)
    return case if cost["flops"] < 2e10 and cost["bytes"] < 7.5e7 else draw(rng)


def _spread(lo, hi, count):
    """`count` whole numbers from lo to hi, evenly apart."""
    return [lo + (hi - lo) * i // max(1, count - 1) for i in range(count)]


def _sizes(case):
    """(new rows, own cached positions before them) of each sequence: the rows rise as the past falls, so that
    long pieces come early in a sequence's life and decoding rows late."""
    return (_spread(case["rows_lo"], case["rows_hi"], case["batch"]),
            _spread(case["past_lo"], case["past_hi"], case["batch"])[::-1])


def _cache(case, gen, pages, dtype):
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    if case["token_major"]:
        return torch.randn((pages, case["page"], case["kv_heads"], case["dim"]), generator=gen,
                           device="cuda").to(dtype).transpose(1, 2)
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if case["op"] == "verify":
        batch, drafts, vocab = case["batch"], case["drafts"], case["vocab"]
        logits = 2.5 * randn(batch, drafts + 1, vocab)
        target = torch.softmax(logits, dim=-1).to(dtype)
        # a draft model that agrees with the target about two times in three
        draft = torch.softmax(logits[:, :drafts] + 0.8 * randn(batch, drafts, vocab), dim=-1)
        tokens = torch.multinomial(draft.reshape(-1, vocab), 1, generator=gen).view(batch, drafts)
        if case["one_hot"]:  # copied tokens: often the likeliest ones
            likely = target[:, :drafts].argmax(dim=-1)
            tokens = torch.where(torch.rand((batch, drafts), generator=gen, device="cuda") < 0.7, likely, tokens)
        return {"case": case, "target": target, "draft": None if case["one_hot"] else draft.to(dtype),
                "tokens": tokens, "uniforms": torch.rand((batch, drafts + 1), generator=gen, device="cuda")}

    rows, past = _sizes(case)
    shared, page, batch = case.get("shared", 0), case["page"], case["batch"]
    order = torch.randperm(batch, generator=host).tolist()  # which sequence has which size
    rows, past = [rows[i] for i in order], [past[i] for i in order]
    needed = [-(-(n + p) // page) for n, p in zip(rows, past)]
    pages = shared + sum(needed)
    free = torch.randperm(pages, generator=host).to(torch.int32)  # pages lie anywhere
    table = torch.zeros((batch, shared + max(needed)), dtype=torch.int32)
    table[:, :shared] = free[:shared]
    at = shared
    for b, count in enumerate(needed):
        table[b, shared:shared + count] = free[at:at + count]
        at += count
    cu = torch.tensor([0] + rows).cumsum(0).to(torch.int32)
    lengths = torch.tensor([shared * page + n + p for n, p in zip(rows, past)], dtype=torch.int32)
    total = int(cu[-1])
    state = {"case": case, "cu_rows": cu.cuda(), "lengths": lengths.cuda(), "table": table.cuda(),
             "longest": max(rows), "k_pages": _cache(case, gen, pages, dtype),
             "v_pages": _cache(case, gen, pages, dtype)}
    if case["op"] == "attention":
        state["q"] = (1.5 * randn(total, case["heads"], case["dim"])).to(dtype)
        return state
    # the fused q|k|v projection's rows; its parts are views
    heads, kv_heads = case["heads"], case["kv_heads"]
    qkv = randn(total, heads + 2 * kv_heads, case["dim"]).to(dtype)
    state["q"], state["k"], state["v"] = qkv.split((heads, kv_heads, kv_heads), dim=1)
    exponent = torch.arange(0, case["rotary"], 2, dtype=torch.float32, device="cuda") / case["rotary"]
    state["inv_freq"] = 1.0 / (THETA ** exponent)
    return state


def _rows_of(state, total):
    """(sequence, place in it, cached position) of every packed row."""
    cu = state["cu_rows"].long()
    row = torch.arange(total, device=cu.device)
    seq = (row.view(-1, 1) >= cu[1:].view(1, -1)).sum(dim=1)
    place = row - cu[seq]
    return seq, place, state["lengths"].long()[seq] - (cu[seq + 1] - cu[seq]) + place


def _plain_append(state):
    case = state["case"]
    page, rotary = case["page"], case["rotary"]
    seq, _, position = _rows_of(state, state["q"].shape[0])
    angle = position.double().view(-1, 1, 1) * state["inv_freq"].double()
    cos, sin = angle.cos().float(), angle.sin().float()

    def rotate(x):
        y = x.float()
        if case["interleaved"]:
            a, b = y[..., 0:rotary:2], y[..., 1:rotary:2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
        else:
            a, b = y[..., :rotary // 2], y[..., rotary // 2:rotary]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
        return torch.cat((turned, y[..., rotary:]), dim=-1).to(x.dtype)

    where = state["table"].long()[seq, position // page]
    state["k_pages"][where, :, position % page] = rotate(state["k"])
    state["v_pages"][where, :, position % page] = state["v"]
    return rotate(state["q"])


def _plain_attention(state):
    case, q = state["case"], state["q"]
    page, shared, group = case["page"], case["shared"], case["heads"] // case["kv_heads"]
    batch, kv_heads, dim, longest = case["batch"], case["kv_heads"], case["dim"], state["longest"]
    seq, place, position = _rows_of(state, q.shape[0])
    # rows padded to the longest sequence's, query heads beside their key/value head
    x = torch.zeros((batch, longest, kv_heads, group, dim), device=q.device)
    x[seq, place] = q.float().view(-1, kv_heads, group, dim)
    at = torch.full((batch, longest), -1, dtype=torch.long, device=q.device)
    at[seq, place] = position
    x = x.permute(2, 0, 1, 3, 4).reshape(kv_heads, batch, longest * group, dim) * dim ** -0.5
    at = at.view(batch, longest, 1).expand(batch, longest, group).reshape(batch, longest * group, 1)

    def gathered(cache, table):  # [rows of the table, kv_heads, positions, dim], 32 bits
        part = cache[table.long()].float()
        return part.transpose(1, 2).reshape(table.shape[0], kv_heads, -1, dim)

    table = state["table"]
    kp, vp = (gathered(state[name], table[:1, :shared])[0] for name in ("k_pages", "v_pages"))
    ko, vo = (gathered(state[name], table[:, shared:]).transpose(0, 1) for name in ("k_pages", "v_pages"))
    scores = torch.cat((torch.matmul(x.reshape(kv_heads, -1, dim), kp.transpose(1, 2).contiguous()).view(
        kv_heads, batch, longest * group, -1), torch.matmul(x, ko.transpose(2, 3).contiguous())), dim=-1)
    key = torch.arange(scores.shape[-1], device=q.device)
    scores = scores.masked_fill(key > at, float("-inf"))
    top = scores.amax(dim=-1, keepdim=True)
    weight = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total = weight.sum(dim=-1, keepdim=True)
    split = shared * page
    # (rows that see less than the table's pages hold: what lies behind is a weight of zero over written values)
    out = torch.matmul(weight[..., :split].flatten(1, 2), vp).view(x.shape) + torch.matmul(
        weight[..., split:].contiguous(), vo)
    out = torch.where(total > 0, out / total, 0.0)
    out = out.view(kv_heads, batch, longest, group, dim).permute(1, 2, 0, 3, 4)[seq, place]
    return out.reshape(q.shape).to(q.dtype)


def _plain_verify(state):
    target, draft, tokens, uniforms = state["target"], state["draft"], state["tokens"], state["uniforms"]
    batch, drafts = tokens.shape
    row = torch.arange(batch, device=tokens.device)
    p = target[:, :drafts].gather(2, tokens.unsqueeze(-1)).squeeze(-1).double()
    q = torch.ones_like(p) if draft is None else draft.gather(2, tokens.unsqueeze(-1)).squeeze(-1).double()
    accepted = (uniforms[:, :drafts].double() * q < p).long().cumprod(dim=1).sum(dim=1)
    rejected = (accepted < drafts).view(-1, 1)
    first = accepted.clamp_max(drafts - 1)
    weight = target[row, accepted].double()
    if draft is None:
        less = torch.zeros_like(weight).scatter_(1, tokens[row, first].view(-1, 1), 1.0)
    else:
        less = draft[row, first].double()
    weight = torch.where(rejected, (weight - less).clamp_min(0), weight)
    running = weight.cumsum(dim=1)
    chosen = (running <= uniforms[:, drafts:].double() * running[:, -1:]).sum(dim=1)
    place = torch.arange(drafts + 1, device=tokens.device)
    padded = torch.cat((tokens, tokens[:, :1]), dim=1)
    out = torch.where(place < accepted.view(-1, 1), padded, torch.where(place == accepted.view(-1, 1),
                                                                        chosen.view(-1, 1), -1))
    return out, accepted.to(torch.int32)


def run(state):
    case = state["case"]
    if case["op"] == "append":
        if own:
            from qwen_int4_hip import paged_append_hip

            rotated = paged_append_hip(state["q"], state["k"], state["v"], state["k_pages"], state["v_pages"],
                                       state["table"], state["cu_rows"], state["lengths"], state["inv_freq"],
                                       interleaved=case["interleaved"])
        else:
            rotated = _plain_append(state)
        return rotated, state["k_pages"], state["v_pages"]
    if case["op"] == "attention":
        if own:
            from qwen_int4_hip import paged_attention_hip

            return paged_attention_hip(state["q"], state["k_pages"], state["v_pages"], state["table"],
                                       state["cu_rows"], state["lengths"], shared_pages=case["shared"])
        return _plain_attention(state)
    if own:
        from qwen_int4_hip import verify_drafts_hip

        return verify_drafts_hip(state["target"], state["tokens"], state["uniforms"], draft_probs=state["draft"])
    return _plain_verify(state)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "verify":
        # one target row per sequence, and one draft row where a draft was refused (all but a few sequences)
        rows = 1 if case["one_hot"] else 2
        return {"bytes": case["batch"] * rows * case["vocab"] * size + case["batch"] * (case["drafts"] + 1) * 28,
                "flops": 2 * case["batch"] * case["vocab"]}
    rows, past = _sizes(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    total = sum(rows)
    table = 4 * sum(-(-(n + p) // case["page"]) for n, p in zip(rows, past))
    if case["op"] == "append":
        return {"bytes": 2 * total * (heads + 2 * kv_heads) * dim * size + 8 * case["batch"] + table,
                "flops": 3 * total * (heads + kv_heads) * case["rotary"]}
    prefix = case["shared"] * case["page"]
    keys = prefix + sum(n + p for n, p in zip(rows, past))
    pairs = sum(n * (prefix + p) + n * (n + 1) // 2 for n, p in zip(rows, past))
    return {"bytes": 2 * keys * kv_heads * dim * size + 2 * total * heads * dim * size + 8 * case["batch"] + table
            + 4 * case["shared"], "flops": 4 * pairs * heads * dim}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "verify":
        target, draft, uniforms = state["target"], state["draft"], state["uniforms"].double()
        tokens = state["tokens"].tolist()
        out = torch.full((case["batch"], case["drafts"] + 1), -1, dtype=torch.int64, device="cuda")
        counts = torch.zeros(case["batch"], dtype=torch.int32, device="cuda")
        for b in range(case["batch"]):
            stood = 0
            for i, token in enumerate(tokens[b]):
                odds = 1.0 if draft is None else float(draft[b, i, token])
                if not float(uniforms[b, i]) * odds < float(target[b, i, token]):
                    break
                out[b, i] = token
                stood += 1
            left = target[b, stood].double()
            if stood < case["drafts"]:
                if draft is None:
                    left[tokens[b][stood]] -= 1.0
                else:
                    left -= draft[b, stood].double()
                left = torch.maximum(left, torch.zeros_like(left))
            heap = torch.cumsum(left, 0)
            out[b, stood] = torch.searchsorted(heap, uniforms[b, -1:] * heap[-1], right=True)[0]
            counts[b] = stood
        return out, counts

    cu, lengths, page = state["cu_rows"].tolist(), state["lengths"].tolist(), case["page"]
    dim = case["dim"]
    if case["op"] == "append":
        rotary = case["rotary"]
        if case["interleaved"]:
            one, two = torch.arange(0, rotary, 2), torch.arange(1, rotary, 2)
        else:
            one, two = torch.arange(rotary // 2), torch.arange(rotary // 2, rotary)
        one, two = one.cuda(), two.cuda()
        turned = state["q"].double()
        k_pages, v_pages = state["k_pages"].double(), state["v_pages"].double()
        keys = state["k"].double()
        for b in range(case["batch"]):
            new = cu[b + 1] - cu[b]
            position = torch.arange(lengths[b] - new, lengths[b], device="cuda")
            angle = torch.outer(position.double(), state["inv_freq"].double()).unsqueeze(1)
            turn = torch.polar(torch.ones_like(angle), angle)
            for x in (turned, keys):
                part = x[cu[b]:cu[b + 1]]
                pairs = torch.complex(part[..., one], part[..., two]) * turn
                part[..., one], part[..., two] = pairs.real, pairs.imag
            slot = state["table"][b].long()[position // page]
            k_pages[slot, :, position % page] = keys[cu[b]:cu[b + 1]]
            v_pages[slot, :, position % page] = state["v"][cu[b]:cu[b + 1]].double()
        return turned, k_pages, v_pages

    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        new, length = cu[b + 1] - cu[b], lengths[b]
        every = torch.arange(length, device="cuda")
        slot = state["table"][b].long()[every // page]
        hidden = every.view(1, 1, -1) > (length - new + torch.arange(new, device="cuda")).view(1, -1, 1)
        for head in range(case["kv_heads"]):
            k, v = (state[name][slot, head, every % page].double() for name in ("k_pages", "v_pages"))
            q = state["q"][cu[b]:cu[b + 1], head * group:(head + 1) * group].double().transpose(0, 1)
            logits = (q.reshape(-1, dim) @ k.T).view(group, new, length) / math.sqrt(dim)
            share = torch.softmax(logits.masked_fill(hidden, -math.inf), dim=-1)
            out[cu[b]:cu[b + 1], head * group:(head + 1) * group] = (
                share.view(-1, length) @ v).view(group, new, dim).transpose(0, 1)
    return out
