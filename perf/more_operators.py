"""The step around new tokens, measured: where they stand, what they attend to, and which token comes next.

Three operators on the fixed-point tensors of a quantised transformer (int32 at scale 2^16, products in 64 bits,
q = floor((y + s/2) / s), r = y - q*s), as a server calls them one after the other:

  pages    from the requests' lengths: the pages that new tokens need, taken from a ring of free ones, those that a sliding
           window has left behind given back, every new token's position and slot in the cache
  attend   attention of several new tokens a sequence (prompts, pieces of prompts, drafted tokens, single ones) over a paged
           cache: each sees what came before it, or a window of that and the first few tokens (sinks), through the
           exponential table; for a proof with every tensor that its lookups need, for an answer without
  next     penalties for repeated tokens, biases and a grammar's mask on the logits, and the token that is chosen; for a
           proof with counts, remainders and distances from the maximum

Sizes are those of the decoder layer that the witness generator makes elsewhere (model width 4096 as one head or as 32
heads of 128, sequences of 2048), longer caches, vocabularies of usual sizes, and odd ones.  Every result is a whole number.
"""
import math
import random

import numpy as np
import torch

own = False

SCALE = 1 << 16
BIT_SHIFT = INDEX_BITS = 20          # the exponential table: 2^20 entries, entry i stands for (i - (2^20 - 1)) / 2^16
SIGMA = 65536.0                      # activations of unit variance at scale 2^16
LOWEST = -(1 << 31)


# ------------------------------------------------------------------ cases
def _pages(name, seqs, longest, new, page, window, sinks, padding, ended):
    return {"name": name, "op": "pages", "seqs": seqs, "longest": longest, "new": new, "page": page, "window": window, "sinks": sinks,
            "padding": padding, "ended": ended}


def _attend(name, seqs, new, longest, lengths, heads, kv_heads, dim, page, window, sinks, proof):
    return {"name": name, "op": "attend", "seqs": seqs, "new": new, "longest": longest, "lengths": lengths, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "window": window, "sinks": sinks, "proof": proof}


def _next(name, seqs, vocab, history, bias, mask, proof):
    return {"name": name, "op": "next", "seqs": seqs, "vocab": vocab, "history": history, "bias": bias, "mask": mask, "proof": proof}


def listed():
    return [
        # one more token of each of a serving batch: latency counts
        _pages("pages_tokens", 64, 2048, 1, 16, 0, 0, 0, False),
        # prompts of a few thousand tokens and running answers in one step, rows padded
        _pages("pages_prompts", 200, 2048, 1000, 16, 0, 0, 500, True),
        # many conversations behind a sliding window, odd pages, some of them over
        _pages("pages_window", 1023, 60000, 70, 17, 1024, 4, 33, True),
        # a serving batch that sees a window and the first four tokens, single new tokens, every tensor of the proof
        _attend("attend_tokens_window", 24, 1, 5000, "ragged", 32, 8, 128, 16, 1024, 4, True),
        # five drafted tokens a sequence checked at once
        _attend("attend_drafts", 8, 5, 3000, "ragged", 32, 8, 128, 16, 0, 0, True),
        # a whole prompt, every tensor of the proof
        _attend("attend_prompt", 1, 2048, 2048, "full", 32, 8, 128, 16, 0, 0, True),
        # the witness generator's own layer: one head of 4096
        _attend("attend_prompt_one_head", 1, 2048, 2048, "full", 1, 1, 4096, 64, 0, 0, True),
        # the next piece of long documents behind a window, an answer without a proof, odd heads and pages
        _attend("attend_piece_window", 3, 1500, 7777, "ragged", 12, 4, 80, 17, 1024, 4, False),
        # the next token of one conversation
        _next("next_one", 1, 32000, 700, False, False, True),
        # a serving batch with a grammar each, every tensor of the proof
        _next("next_batch", 64, 32000, 2048, True, True, True),
        # a large batch with a large vocabulary, the answer's tokens alone
        _next("next_large_answer", 256, 131072, 4096, True, True, False),
        # an odd vocabulary, rows that no vector load fits
        _next("next_odd", 37, 50257, 1333, False, True, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["pages", "attend", "attend", "next"])
    if op == "pages":
        while True:
            seqs, longest, new, page = _log(rng, 1, 2000), _log(rng, 16, 60000), _log(rng, 1, 2000), rng.choice([8, 16, 16, 17, 32, 64, 100, 128])
            if seqs * new <= 1 << 18 and seqs * (longest + new) // page <= 1 << 22:
                break
        window = _log(rng, 16, 4096) if rng.random() < 0.4 else 0
        case = _pages("", seqs, longest, new, page, window, rng.choice([0, 1, 4, 64]) if window else 0, rng.choice([0, 0, 7, 100]), rng.random() < 0.5)
    elif op == "attend":
        dim = rng.choice([32, 48, 64, 64, 80, 96, 100, 128, 128, 128, 192, 256, 50])
        kv_heads = rng.choice([1, 2, 4, 5, 8, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 7, 8])
        if rng.random() < 0.1:
            dim, kv_heads, heads = rng.choice([1024, 2048, 4096]), 1, 1
        while True:
            seqs, new, longest = _log(rng, 1, 64), rng.choice([1, _log(rng, 1, 16), _log(rng, 1, 2048), _log(rng, 1, 2048)]), _log(rng, 1, 131072)
            longest = max(longest, new)
            pairs = seqs * new * longest * heads
            if pairs <= 1 << 27 and pairs * dim <= 1 << 34 and seqs * longest * kv_heads * dim <= 131072 * 8 * 128:
                break
        window = _log(rng, 16, 4096) if rng.random() < 0.4 else 0
        case = _attend("", seqs, new, longest, rng.choice(["full", "ragged"]), heads, kv_heads, dim, rng.choice([8, 16, 16, 17, 32, 64, 100, 128]),
                       window, rng.choice([0, 1, 4, 4, 64]) if window else 0, rng.random() < 0.7)
    else:
        while True:
            seqs, vocab, history = _log(rng, 1, 256), _log(rng, 1000, 262144), _log(rng, 1, 32768)
            if seqs * vocab <= 256 * 131072 and seqs * history <= 1 << 22:
                break
        if rng.random() < 0.5:
            vocab = vocab // 64 * 64
        case = _next("", seqs, vocab, history, rng.random() < 0.5, rng.random() < 0.6, rng.random() < 0.6)
    del case["name"]
    return case


def _pages_numbers(case):
    """Cached lengths and numbers of new tokens (-1: a request that is over) of the sequences."""
    r = random.Random(case["seqs"] * 1000 + case["longest"])
    lens = [r.randint(0, case["longest"]) for _ in range(case["seqs"])]
    new = [r.randint(1, case["new"]) if r.random() < 0.3 else 1 for _ in range(case["seqs"])]
    if case["ended"]:
        new = [-1 if r.random() < 0.05 else 0 if r.random() < 0.05 else n for n in new]
    return lens, new


def _attend_numbers(case):
    """Numbers of new tokens and lengths (with them) of the sequences."""
    seqs, longest, most = case["seqs"], case["longest"], case["new"]
    if case["lengths"] == "full":
        return [most] * seqs, [longest] * seqs
    r = random.Random(longest * 1000 + seqs)
    new = [0 if r.random() < 0.05 else r.randint(1, most) for _ in range(seqs)]
    new[r.randrange(seqs)] = most
    lens = [r.randint(n, longest) for n in new]
    lens[new.index(most)] = longest
    return new, lens


def _seen(pos, window, sinks):
    """How many positions the token at `pos` attends to."""
    if not window or pos < window:
        return pos + 1
    return window + min(sinks, pos + 1 - window)


def work(case):
    if case["op"] == "pages":
        lens, new = _pages_numbers(case)
        page, rows = case["page"], sum(max(n, 0) for n in new)
        taken = sum(-(-(a + max(n, 0)) // page) - -(-a // page) for a, n in zip(lens, new))
        return {"bytes": 16 * case["seqs"] + 12 * (rows + case["padding"]) + 8 * taken, "flops": 0}
    if case["op"] == "attend":
        new, lens = _attend_numbers(case)
        pairs = sum(_seen(p, case["window"], case["sinks"]) for n, a in zip(new, lens) for p in range(a - n, a)) * case["heads"]
        first = [max(0, a - n + 1 - case["window"]) if case["window"] else 0 for n, a in zip(new, lens)]
        live = sum(a - f + min(case["sinks"], f) for n, a, f in zip(new, lens, first) if n)
        rows = sum(new) * case["heads"]
        proof = (24 * pairs + 8 * rows) if case["proof"] else 0
        return {"bytes": 8 * live * case["kv_heads"] * case["dim"] + 4 * live // case["page"] + 12 * rows * case["dim"] + proof,
                "flops": 4 * pairs * case["dim"]}
    n = case["seqs"] * case["vocab"]
    return {"bytes": n * (4 + (16 if case["proof"] else 0)) + (4 * case["vocab"] if case["bias"] else 0) + (n // 8 if case["mask"] else 0)
            + 4 * case["seqs"] * case["history"] + 24 * case["seqs"], "flops": 4 * n}


# ------------------------------------------------------------------ inputs
def _gauss(g, shape, sigma=SIGMA):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(sigma).round_().to(torch.int32)


def _exp_table():
    x = torch.arange(1 << INDEX_BITS, dtype=torch.float64, device="cuda") - ((1 << BIT_SHIFT) - 1)
    return torch.round(torch.exp(x / SCALE) * SCALE).to(torch.int32)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 13)
    new_ = lambda *shape: torch.full(shape, -7, dtype=torch.int32, device="cuda")  # noqa: E731
    s = {"op": case["op"]}
    if case["op"] == "pages":
        lens, new = _pages_numbers(case)
        page, seqs, rows = case["page"], case["seqs"], sum(max(n, 0) for n in new) + case["padding"]
        held = _int32([-(-n // page) for n in lens]).long()
        width = max(-(-(a + max(n, 0)) // page) for a, n in zip(lens, new)) + 1
        total = int(held.sum())
        pages = total + sum(-(-(a + max(n, 0)) // page) - -(-a // page) for a, n in zip(lens, new)) + 17
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        at = torch.arange(width, device="cuda")[None, :]
        mine = at < held[:, None]
        s["block_table"] = torch.where(mine, order[(held.cumsum(0) - held)[:, None] + torch.where(mine, at, 0)], -1)
        # the free pages stand somewhere in their ring
        head, free = int(torch.randint(0, 2 * pages, (1,), generator=g, device="cuda")), pages - total
        s["free_pages"] = new_(2 * pages)
        s["free_pages"][(head + torch.arange(free, device="cuda")) % (2 * pages)] = order[total:]
        s["free_span"] = _int32([head, free])
        s["lens"], s["new"] = _int32(lens), _int32(new)
        s["page"], s["rows"], s["window"], s["sinks"] = page, rows, case["window"], case["sinks"]
        s["out"] = {"starts": new_(seqs + 1), "positions": new_(rows), "slots": new_(rows).long(), "lens": new_(seqs), "free_span": new_(2)}
        return s
    if case["op"] == "attend":
        b, h, hk, d, page, longest = (case[k] for k in ("seqs", "heads", "kv_heads", "dim", "page", "longest"))
        new, lens = _attend_numbers(case)
        rows = sum(new)
        each = -(-longest // page)
        used = [-(-n // page) for n in lens]
        pages = sum(used) + 2
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = np.full((b, each), -1, dtype=np.int64)  # where in `order` a sequence's pages stand
        at = 0
        for i, n in enumerate(used):
            table[i, :n] = np.arange(at, at + n)
            at += n
        table = torch.from_numpy(table).cuda()
        s["block_table"] = torch.where(table >= 0, order[table.clamp(min=0)], -1).to(torch.int32)
        s["starts"] = _int32([sum(new[:i]) for i in range(b + 1)])
        s["lens"], s["most"], s["longest"] = _int32(lens), case["new"], longest
        s["window"], s["sinks"] = case["window"], case["sinks"]
        s["q"] = _gauss(g, (rows, h, d))
        s["k_cache"], s["v_cache"] = _gauss(g, (pages, page, hk, d)), _gauss(g, (pages, page, hk, d))
        s["table"] = _exp_table()
        s["qk_scale"] = int(round(SCALE * math.sqrt(d)))
        s["out"] = {"qkv": new_(rows, h, d), "qkv_rem": new_(rows, h, d)}
        if case["proof"]:
            for name in ("scores", "scores_rem", "exp_input", "exp_output", "softmax_output", "softmax_lookup_query"):
                s["out"][name] = new_(rows, h, longest)
            s["out"]["max"], s["out"]["exp_sum"] = new_(rows, h), new_(rows, h)
        return s
    n, v, longest = case["seqs"], case["vocab"], case["history"]
    s["logits"] = _gauss(g, (n, v), 3 * SIGMA)
    # a text's tokens: few of them often, most of them seldom
    u = torch.rand((n, longest), generator=g, device="cuda", dtype=torch.float64)
    s["history"] = torch.exp(u * math.log(v)).floor_().clamp_(max=v - 1).to(torch.int32)
    lens = torch.randint(0, longest + 1, (n,), generator=g, device="cuda")
    lens[0] = longest
    s["history_lens"] = lens.to(torch.int32)
    one = lambda lo, hi: torch.randint(lo, hi, (n,), generator=g, device="cuda").to(torch.int32)  # noqa: E731
    s["repetition"], s["presence"], s["frequency"] = one(SCALE, 3 * SCALE // 2), one(0, SCALE // 2), one(0, SCALE // 4)
    s["bias"] = s["mask"] = None
    if case["bias"]:                     # of a few tokens, one of them forbidden
        s["bias"] = torch.where(torch.rand(v, generator=g, device="cuda") < 0.01, _gauss(g, (v,)), 0)
        s["bias"][v // 2] = LOWEST
    if case["mask"]:                     # what a grammar allows; in one row nothing
        s["mask"] = torch.randint(-(1 << 31), 1 << 31, (n, -(-v // 32)), generator=g, device="cuda").to(torch.int32)
        s["mask"][n // 2] = 0 if n > 1 else -1
    s["out"] = {"token": new_(n), "max": new_(n)}
    if case["proof"]:
        for name in ("logits", "rem", "count", "gap"):
            s["out"][name] = new_(n, v)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        from grape_amd import ops
        if s["op"] == "pages":
            return ops.wit_page_step(s["lens"], s["new"], s["block_table"], s["free_pages"], s["free_span"], s["page"], s["rows"],
                                     window=s["window"], sinks=s["sinks"], out=s["out"]), s["block_table"], s["free_pages"]
        if s["op"] == "attend":
            return ops.wit_window_attention(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["starts"], s["lens"], s["most"], s["longest"],
                                            s["table"], window=s["window"], sinks=s["sinks"], bit_shift=BIT_SHIFT, index_bits=INDEX_BITS,
                                            qk_scale=s["qk_scale"], prob_scale=SCALE, out_scale=SCALE, out=s["out"])
        return ops.wit_next_token(s["logits"], s["history"], s["history_lens"], repetition=s["repetition"], presence=s["presence"],
                                  frequency=s["frequency"], bias=s["bias"], mask=s["mask"], scale=SCALE, out=s["out"])
    if s["op"] == "pages":
        return _plain_pages(s)
    if s["op"] == "attend":
        return _plain_attend(s)
    return _plain_next(s)


def _plain_pages(s):
    lens, new, table, ring, page, window = s["lens"].long(), s["new"].long(), s["block_table"], s["free_pages"], s["page"], s["window"]
    room, rows = ring.numel(), s["rows"]
    ended, n = new < 0, new.clamp(min=0)
    up = lambda x: (x + page - 1) // page  # noqa: E731
    held = up(lens)
    want = up(lens + n) - held
    last, taken = n.cumsum(0), want.cumsum(0)
    head, count = s["free_span"][0].long(), s["free_span"][1].long()
    at = torch.arange(table.shape[1], device="cuda")[None, :]
    k = (taken - want)[:, None] + at - held[:, None]
    fresh = (k >= (taken - want)[:, None]) & (k < taken[:, None])
    table.copy_(torch.where(fresh, ring[(head + torch.where(fresh, k, 0)) % room], table))
    # what the window leaves behind, and everything of a request that is over
    keep = up(torch.tensor(s["sinks"], device="cuda"))
    gone = (lambda p: (p + 1 - window).clamp(min=0) // page) if window else (lambda p: torch.zeros_like(p))
    lo = torch.maximum(gone(lens), keep)[:, None]
    back = torch.where(ended[:, None], (at < held[:, None]) & ((at < keep) | (at >= lo)), (at >= lo) & (at < gone(lens + n)[:, None]))
    rank = back.flatten().cumsum(0).view(back.shape)
    to = torch.where(back, (head + count + rank - 1) % room, room)
    wider = torch.cat((ring, ring[:1]))
    wider.scatter_(0, to.flatten(), table.flatten())
    ring.copy_(wider[:room])
    row = torch.arange(rows, device="cuda")
    b = torch.searchsorted(last, row, right=True).clamp(max=len(lens) - 1)
    live = row < last[-1]
    pos = torch.where(live, lens[b] + row - (last - n)[b], 0)
    out = s["out"]
    out["starts"][0] = 0
    out["starts"][1:] = last
    out["positions"].copy_(pos)
    out["slots"].copy_(torch.where(live, table[b, pos // page].long() * page + pos % page, -1))
    out["lens"].copy_(torch.where(ended, 0, lens + n))
    out["free_span"][0] = (head + taken[-1]) % room
    out["free_span"][1] = count - taken[-1] + rank[-1, -1]
    return out, table, ring


def _rescale(y, scale):
    """(q, r) of 64-bit whole numbers, as 32-bit ones"""
    q = torch.div(y + scale // 2, scale, rounding_mode="floor")
    return q.to(torch.int32), (y - q * scale).to(torch.int32)


def _plain_attend(s):
    rows, h, d = s["q"].shape
    page, hk = s["k_cache"].shape[1:3]
    b, most, longest = len(s["lens"]), s["most"], s["longest"]
    at = torch.arange(longest, device="cuda")
    token = s["block_table"][:, at // page].clamp(min=0).long() * page + at % page             # [b][longest]
    starts, lens = s["starts"].long(), s["lens"].long()
    new = starts[1:] - starts[:-1]
    j = torch.arange(most, device="cuda")
    there = j < new[:, None]                                                                  # [b][most]
    row = torch.where(there, starts[:-1, None] + j, 0)
    pos = (lens - new)[:, None] + j
    live = (at <= pos[..., None]) & there[..., None]
    if s["window"]:
        live = live & ((at > pos[..., None] - s["window"]) | (at < s["sinks"]))
    live = live[:, None]                                                                      # [b][1][most][longest]
    # float64 products of whole numbers: every sum stays below 2^53 and is exact
    q = s["q"][row].permute(0, 2, 1, 3).contiguous().double().view(b, hk, -1, d)              # heads of a cache head, then tokens
    k = s["k_cache"].view(-1, hk, d)[token].permute(0, 2, 3, 1).contiguous().double()           # [b][hk][d][longest]
    scores, scores_rem = _rescale(torch.matmul(q, k).long().view(b, h, most, longest), s["qk_scale"])
    del k
    empty = ~live.any(-1)
    top = torch.where(live, scores, LOWEST).amax(-1)
    top = torch.where(empty, 0, top)
    x = scores.long() - top.long()[..., None]
    index = x + ((1 << BIT_SHIFT) - 1)
    e = s["table"][torch.where((index >= 0) & (index < 1 << INDEX_BITS), index, 0)].long()
    del index
    e = torch.where(live, e, 0)
    total = e.sum(-1)
    denominator = torch.where(empty, 1, total)[..., None]
    p = torch.div(e * SCALE + denominator // 2, denominator, rounding_mode="floor")
    query = e * (2 * SCALE) - denominator * (2 * p - 1)
    p = torch.where(live, p, 0)
    v = s["v_cache"].view(-1, hk, d)[token].permute(0, 2, 1, 3).contiguous().double()           # [b][hk][longest][d]
    y, y_rem = _rescale(torch.matmul(p.double().view(b, hk, -1, longest), v).long().view(b, h, most, d), SCALE)
    del v
    out, to = s["out"], row[there]
    put = lambda name, t: out[name].index_copy_(0, to, t.transpose(1, 2)[there].to(torch.int32))  # noqa: E731
    put("qkv", y), put("qkv_rem", y_rem)
    if "scores" in out:
        put("max", top), put("exp_sum", total)
        mask = live.expand(b, h, most, longest).transpose(1, 2)[there]
        keep = lambda name, t: out[name].index_copy_(0, to, torch.where(mask, t.transpose(1, 2)[there].to(torch.int32), out[name][to]))  # noqa: E731
        keep("scores", scores), keep("scores_rem", scores_rem), keep("exp_input", x), keep("exp_output", e)
        keep("softmax_output", p), keep("softmax_lookup_query", query)
    return out


def _plain_next(s):
    x, out = s["logits"].long(), s["out"]
    n, v = x.shape
    inside = torch.arange(s["history"].shape[1], device="cuda") < s["history_lens"][:, None]
    count = torch.zeros((n, v + 1), dtype=torch.int64, device="cuda")
    count.scatter_add_(1, torch.where(inside, s["history"].long(), v), torch.ones_like(inside, dtype=torch.int64))
    count = count[:, :v]
    allowed = x != LOWEST
    if s["bias"] is not None:
        allowed = allowed & (s["bias"] != LOWEST)
    if s["mask"] is not None:
        at = torch.arange(v, device="cuda")
        allowed = allowed & ((s["mask"][:, at // 32] >> (at % 32)) & 1).bool()
    repetition = s["repetition"].long()[:, None]
    y, divisor = torch.where(x > 0, x * SCALE, x * repetition), torch.where(x > 0, repetition, SCALE)
    q = torch.div(y + divisor // 2, divisor, rounding_mode="floor")
    repeated = (count > 0) & allowed
    rem = torch.where(repeated, y - q * divisor, 0)
    z = torch.where(repeated, q - s["presence"].long()[:, None] - s["frequency"].long()[:, None] * count, x)
    if s["bias"] is not None:
        z = z + s["bias"].long()
    z = torch.where(allowed, z.clamp(min=LOWEST + 1, max=(1 << 31) - 1), LOWEST)
    top = z.amax(-1)
    first = torch.where(z == top[:, None], torch.arange(v, device="cuda"), v).amin(-1)
    out["token"].copy_(torch.where(top == LOWEST, -1, first)), out["max"].copy_(top)
    if "logits" in out:
        out["logits"].copy_(z), out["rem"].copy_(rem), out["count"].copy_(count)
        out["gap"].copy_(torch.where(allowed, top[:, None] - z, 0))
    return out


# ------------------------------------------------------------------ the definition, in 64-bit whole numbers on the host
def _split(y, scale):
    q = (y + scale // 2) // scale
    return q, y - q * scale


def _host(t):
    return t.cpu().numpy().astype(np.int64)


def _exact_pages(case, s):
    table, ring, page, rows = _host(s["block_table"]), _host(s["free_pages"]), s["page"], s["rows"]
    head, count = (int(x) for x in _host(s["free_span"]))
    window, keep = s["window"], -(-s["sinks"] // s["page"])
    starts, positions, slots, lens, at, pushed = [0], [0] * rows, [-1] * rows, [], head, []
    for b, (have, n) in enumerate(zip(_host(s["lens"]).tolist(), _host(s["new"]).tolist())):
        held = -(-have // page)
        for i in range(held, -(-(have + max(n, 0)) // page)):
            table[b, i] = ring[at % len(ring)]
            at += 1
        for j in range(max(n, 0)):
            positions[starts[-1] + j] = have + j
            slots[starts[-1] + j] = int(table[b, (have + j) // page]) * page + (have + j) % page
        # a page is out of sight for the token at position p where its last position is at most p - window
        unseen = lambda i, p: window > 0 and i >= keep and (i + 1) * page - 1 <= p - window  # noqa: E731
        for i in range(-(-(have + max(n, 0)) // page)):
            if (n < 0 or unseen(i, have + n)) and not unseen(i, have):
                pushed.append(int(table[b, i]))
        starts.append(starts[-1] + max(n, 0))
        lens.append(0 if n < 0 else have + n)
    for i, p in enumerate(pushed):
        ring[(head + count + i) % len(ring)] = p
    out = {"starts": starts, "positions": positions, "slots": slots, "lens": lens, "free_span": [at % len(ring), count - (at - head) + len(pushed)]}
    return {k: np.array(v, dtype=np.int64 if k == "slots" else np.int32) for k, v in out.items()}, table.astype(np.int32), ring.astype(np.int32)


def _exact_attend(case, s):
    new, lens = _attend_numbers(case)
    out = {n: _host(t) for n, t in s["out"].items()}
    q, table, pages = _host(s["q"]), _host(s["table"]), _host(s["block_table"])
    each, page, row = case["heads"] // case["kv_heads"], case["page"], 0
    for b, (n, a) in enumerate(zip(new, lens)):
        at = np.arange(a)
        where = torch.from_numpy(pages[b][at // page] * page + at % page).cuda()
        shape = (-1, case["kv_heads"], case["dim"])
        keys, values = (_host(s[c].view(shape)[where]) for c in ("k_cache", "v_cache"))
        for pos in range(a - n, a):
            sees = at[: pos + 1]
            if case["window"]:
                sees = sees[(sees > pos - case["window"]) | (sees < case["sinks"])]
            for h in range(case["heads"]):
                kv = h // each
                score, rem = _split((keys[sees, kv] * q[row, h]).sum(1), s["qk_scale"])
                x = score - score.max()
                e = table[x + (1 << BIT_SHIFT) - 1]
                total = int(e.sum())
                p = (e * SCALE + total // 2) // total
                out["qkv"][row, h], out["qkv_rem"][row, h] = _split((values[sees, kv] * p[:, None]).sum(0), SCALE)
                if case["proof"]:
                    out["max"][row, h], out["exp_sum"][row, h] = score.max(), total
                    for name, t in (("scores", score), ("scores_rem", rem), ("exp_input", x), ("exp_output", e), ("softmax_output", p),
                                    ("softmax_lookup_query", 2 * SCALE * e - total * (2 * p - 1))):
                        out[name][row, h, sees] = t
            row += 1
    return {n: x.astype(np.int32) for n, x in out.items()}


def _exact_next(case, s):
    out = {n: _host(t) for n, t in s["out"].items()}
    x, history, lens = _host(s["logits"]), _host(s["history"]), _host(s["history_lens"])
    v, bias = case["vocab"], _host(s["bias"]) if case["bias"] else np.zeros(case["vocab"], dtype=np.int64)
    penalties = [_host(s[k]) for k in ("repetition", "presence", "frequency")]
    words = s["mask"].cpu().numpy().view(np.uint32) if case["mask"] else None
    for b in range(case["seqs"]):
        repetition, presence, frequency = (int(p[b]) for p in penalties)
        count = np.bincount(history[b, : lens[b]], minlength=v)
        z, rem, allowed = x[b].copy(), np.zeros(v, dtype=np.int64), (x[b] != LOWEST) & (bias != LOWEST)
        if words is not None:
            allowed &= np.unpackbits(words[b].view(np.uint8), bitorder="little")[:v].astype(bool)
        up, down = (count > 0) & (z > 0), (count > 0) & (z <= 0)
        z[up], rem[up] = _split(z[up] * SCALE, repetition)
        z[down], rem[down] = _split(z[down] * repetition, SCALE)
        z -= np.where(count > 0, presence + frequency * count, 0)
        z = np.where(allowed, np.clip(z + bias, LOWEST + 1, (1 << 31) - 1), LOWEST)
        out["max"][b] = z.max()
        out["token"][b] = z.argmax() if allowed.any() else -1
        if case["proof"]:
            out["logits"][b], out["rem"][b], out["count"][b], out["gap"][b] = z, np.where(allowed, rem, 0), count, np.where(allowed, z.max() - z, 0)
    return {n: t.astype(np.int32) for n, t in out.items()}


def exact(case, seed):
    w = work(case)
    if case["op"] == "attend" and w["flops"] > 1 << 32:        # minutes on the host
        return None
    s = prepare(case, seed)
    return {"pages": _exact_pages, "attend": _exact_attend, "next": _exact_next}[case["op"]](case, s)
