"""The witness of one new token, measured: what a user has computed who proves an answer as it is generated.

Three operators on the fixed-point tensors of a quantised transformer block (int32 at scale 2^16, products in 64 bits,
q = floor((y + s/2) / s), r = y - q*s):

  append   rotates the queries and keys of new tokens by their positions and appends keys and values to a paged cache
  attend   attention of one new token a sequence over the paged cache, through the exponential table; for a proof with
           every tensor that its lookups need, for an answer without
  q4       products of a few tokens with 4-bit weights and group scales, rescaled

Sizes are those of the decoder layer that the witness generator makes elsewhere (model width 4096 as one head or as 32
heads of 128, feed-forward width 11008, sequences of 2048), longer caches, and odd ones.  Every result is a whole number.
"""
import math
import random

import numpy as np
import torch

own = False

SCALE = 1 << 16
BIT_SHIFT = INDEX_BITS = 20          # the exponential table: 2^20 entries, entry i stands for (i - (2^20 - 1)) / 2^16
SIGMA = 65536.0                      # activations of unit variance at scale 2^16


# ------------------------------------------------------------------ cases
def _append(name, tokens, heads, kv_heads, dim, rot, interleaved, page, padding, at):
    return {"name": name, "op": "append", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
            "interleaved": interleaved, "page": page, "padding": padding, "at": at}


def _attend(name, seqs, longest, lengths, heads, kv_heads, dim, page, window, proof):
    return {"name": name, "op": "attend", "seqs": seqs, "longest": longest, "lengths": lengths, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "window": window, "proof": proof}


def _q4(name, tokens, outputs, inputs, group, zeros):
    return {"name": name, "op": "q4", "tokens": tokens, "outputs": outputs, "inputs": inputs, "group": group, "zeros": zeros}


def listed():
    return [
        # the next token of one conversation
        _append("append_one_token", 1, 32, 8, 128, 128, False, 16, 0, 1000),
        # the next tokens of a batch that was padded to 64
        _append("append_batch", 64, 32, 8, 128, 128, False, 16, 3, 700),
        # a whole prompt of the witness generator's own layer: one head of 4096, pairs side by side
        _append("append_prompt_one_head", 2048, 1, 1, 4096, 4096, True, 64, 0, 0),
        # a prompt that follows a cached one; heads of 80 of which 32 are rotated, pages of 17
        _append("append_prompt_odd", 1533, 12, 4, 80, 32, False, 17, 0, 515),
        # the first words of an answer: latency counts
        _attend("attend_short", 1, 37, "full", 32, 8, 128, 16, 0, True),
        # a serving batch, lengths from none to 2048, every tensor of the proof
        _attend("attend_batch", 64, 2048, "ragged", 32, 8, 128, 16, 0, True),
        # one long document
        _attend("attend_long", 1, 131072, "full", 32, 8, 128, 256, 0, True),
        # the witness generator's own layer, eight sequences of 2048
        _attend("attend_one_head", 8, 2048, "full", 1, 1, 4096, 64, 0, True),
        # an answer without a proof: sliding window, odd heads and pages
        _attend("attend_window", 24, 5000, "ragged", 12, 4, 80, 17, 1024, False),
        # one token through a square projection
        _q4("q4_square", 1, 4096, 4096, 128, False),
        # one token through the feed-forward projection, weights with zero points
        _q4("q4_up", 1, 11008, 4096, 64, True),
        # sixteen tokens through the projection back
        _q4("q4_down_batch", 16, 4096, 11008, 128, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "q4"])
    if op == "q4":
        group = rng.choice([32, 64, 128, 128, 256])
        while True:
            tokens, outputs, inputs = _log(rng, 1, 24), _log(rng, 64, 16384), _log(rng, 64, 16384)
            if tokens * outputs * inputs <= 16 * 4096 * 11008 and outputs * inputs <= 16384 * 8192:
                break
        if rng.random() < 0.7:
            inputs = max(group, inputs // group * group)         # else the last group is short
        case = _q4("", tokens, outputs, inputs, group, rng.random() < 0.5)
    else:
        dim = rng.choice([32, 48, 64, 64, 80, 96, 100, 128, 128, 128, 192, 256, 50])
        kv_heads = rng.choice([1, 2, 4, 5, 8, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 7, 8])
        if rng.random() < 0.15:
            dim, kv_heads, heads = rng.choice([1024, 2048, 4096]), 1, 1
        page = rng.choice([8, 16, 16, 17, 32, 64, 100, 128])
        if op == "append":
            most = min(4096, 2048 * 4096 // (heads * dim))
            tokens = _log(rng, 1, most)
            padding = rng.randint(1, tokens - 1) if tokens > 4 and tokens < 128 and rng.random() < 0.3 else 0
            rot = dim if rng.random() < 0.7 else dim // 4 * 2
            case = _append("", tokens, heads, kv_heads, dim, rot, rng.random() < 0.4, page, padding, _log(rng, 1, 4000))
        else:
            while True:
                seqs, longest = _log(rng, 1, 96), _log(rng, 1, 131072)
                if seqs * longest * kv_heads * dim <= 131072 * 8 * 128 and seqs * longest * heads <= 131072 * 32:
                    break
            window = _log(rng, 16, 4096) if rng.random() < 0.2 else 0
            case = _attend("", seqs, longest, rng.choice(["full", "ragged"]), heads, kv_heads, dim, page, window, rng.random() < 0.75)
    del case["name"]
    return case


def _lengths(case):
    """The sequences' lengths, and the first position that each of them attends to."""
    seqs, longest = case["seqs"], case["longest"]
    lens = [longest] * seqs
    if case["lengths"] == "ragged":
        r = random.Random(longest * 1000 + seqs)
        lens = [0 if r.random() < 0.05 else r.randint(1, longest) for _ in range(seqs)]
        lens[r.randrange(seqs)] = longest
    first = [max(0, n - case["window"]) if case["window"] else 0 for n in lens]
    return lens, first


def work(case):
    if case["op"] == "append":
        t, q, k = case["tokens"] - case["padding"], case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
        table = 2 * (case["rot"] // 2)
        return {"bytes": 4 * t * ((q + 2 * k) + 2 * q + 3 * k + table) + 12 * case["tokens"],
                "flops": 3 * t * case["rot"] * (case["heads"] + case["kv_heads"])}
    if case["op"] == "attend":
        lens, first = _lengths(case)
        live = sum(n - f for n, f in zip(lens, first))
        rows, d, kd = case["heads"], case["dim"], case["kv_heads"] * case["dim"]
        proof = (24 * live * rows + 8 * case["seqs"] * rows) if case["proof"] else 0
        return {"bytes": 8 * live * kd + 4 * live // case["page"] + 12 * case["seqs"] * rows * d + proof, "flops": 4 * live * rows * d}
    groups = -(-case["inputs"] // case["group"])
    return {"bytes": case["outputs"] * ((case["inputs"] + 1) // 2 + groups * (5 if case["zeros"] else 4))
            + case["tokens"] * (4 * case["inputs"] + 8 * case["outputs"]), "flops": 2 * case["tokens"] * case["outputs"] * case["inputs"]}


# ------------------------------------------------------------------ inputs
def _gauss(g, shape, sigma=SIGMA):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(sigma).round_().to(torch.int32)


def _exp_table():
    x = torch.arange(1 << INDEX_BITS, dtype=torch.float64, device="cuda") - ((1 << BIT_SHIFT) - 1)
    return torch.round(torch.exp(x / SCALE) * SCALE).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 13)
    new = lambda *shape: torch.full(shape, -7, dtype=torch.int32, device="cuda")  # noqa: E731
    s = {"op": case["op"]}
    if case["op"] == "append":
        t, h, hk, d, rot, page = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "rot", "page"))
        # one fused projection's output: the queries, keys and values of a token stand side by side
        qkv = _gauss(g, (t, (h + 2 * hk) * d))
        s["q"] = qkv[:, :h * d].view(t, h, d)
        s["k"] = qkv[:, h * d:(h + hk) * d].view(t, hk, d)
        s["v"] = qkv[:, (h + hk) * d:].view(t, hk, d)
        live = t - case["padding"]
        if t > 256:                                    # one prompt behind `at` cached tokens
            positions = case["at"] + torch.arange(t, device="cuda")
            pages = -(-(case["at"] + t) // page) + 3
            order = torch.randperm(pages, generator=g, device="cuda")
            slots = order[positions // page] * page + positions % page
        else:                                          # one token of each sequence, the last ones padding
            positions = torch.randint(0, case["at"] + 1, (t,), generator=g, device="cuda")
            pages = t + 5
            slots = torch.randperm(pages, generator=g, device="cuda")[:t] * page + positions % page
            slots[live:] = -1
        s["positions"], s["slots"] = positions.to(torch.int32), slots.to(torch.int64)
        angle = torch.arange(case["at"] + t + 1, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
            -torch.arange(rot // 2, dtype=torch.float64, device="cuda") * 2 / max(rot, 1))
        s["cos"], s["sin"] = (torch.round(f(angle) * SCALE).to(torch.int32) for f in (torch.cos, torch.sin))
        s["interleaved"] = case["interleaved"]
        s["k_cache"], s["v_cache"] = new(pages, page, hk, d), new(pages, page, hk, d)
        s["q_out"], s["q_rem"], s["k_rem"] = new(t, h, d), new(t, h, d), new(t, hk, d)
        return s
    if case["op"] == "attend":
        b, h, hk, d, page, longest = (case[k] for k in ("seqs", "heads", "kv_heads", "dim", "page", "longest"))
        lens, first = _lengths(case)
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
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["first"] = torch.tensor(first, dtype=torch.int32, device="cuda") if case["window"] else None
        s["q"] = _gauss(g, (b, h, d))
        s["k_cache"], s["v_cache"] = _gauss(g, (pages, page, hk, d)), _gauss(g, (pages, page, hk, d))
        s["table"], s["longest"] = _exp_table(), longest
        s["qk_scale"] = int(round(SCALE * math.sqrt(d)))
        s["out"] = {"qkv": new(b, h, d), "qkv_rem": new(b, h, d)}
        if case["proof"]:
            for name in ("scores", "scores_rem", "exp_input", "exp_output", "softmax_output", "softmax_lookup_query"):
                s["out"][name] = new(b, h, longest)
            s["out"]["max"], s["out"]["exp_sum"] = new(b, h), new(b, h)
        return s
    n, m, k, group = (case[x] for x in ("tokens", "outputs", "inputs", "group"))
    groups = -(-k // group)
    s["x"] = _gauss(g, (n, k))
    # weights of a trained layer, rounded to 16 steps about the zero point
    nibbles = (torch.randn((m, k + k % 2), generator=g, device="cuda") * 2.5 + 8).round_().clamp_(0, 15).to(torch.uint8)
    s["w"] = (nibbles[:, 0::2] | (nibbles[:, 1::2] << 4)).contiguous()      # the lower half holds the even input
    s["scales"] = (torch.rand((m, groups), generator=g, device="cuda") * 0.5 + 0.75).mul_(SCALE / (2.5 * math.sqrt(k))).round_().to(torch.int32)
    s["zeros"] = torch.randint(5, 12, (m, groups), generator=g, device="cuda").to(torch.uint8) if case["zeros"] else None
    s["group"] = group
    s["y"], s["y_rem"] = new(n, m), new(n, m)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        from grape_amd import ops
        if s["op"] == "append":
            ops.wit_rope_append(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["cos"], s["sin"], s["k_cache"], s["v_cache"],
                                s["q_out"], s["q_rem"], s["k_rem"], scale=SCALE, interleaved=s["interleaved"])
            return s["q_out"], s["q_rem"], s["k_rem"], s["k_cache"], s["v_cache"]
        if s["op"] == "attend":
            return ops.wit_paged_attention(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["lens"], s["longest"], s["table"],
                                           first=s["first"], bit_shift=BIT_SHIFT, index_bits=INDEX_BITS, qk_scale=s["qk_scale"],
                                           prob_scale=SCALE, out_scale=SCALE, out=s["out"])
        return ops.wit_matvec_q4(s["x"], s["w"], s["scales"], s["group"], zeros=s["zeros"], scale=SCALE, q=s["y"], r=s["y_rem"])
    if s["op"] == "append":
        return _plain_append(s)
    if s["op"] == "attend":
        return _plain_attend(s)
    return _plain_q4(s)


def _rescale(y, scale):
    """(q, r) of 64-bit whole numbers, as 32-bit ones"""
    q = torch.div(y + scale // 2, scale, rounding_mode="floor")
    return q.to(torch.int32), (y - q * scale).to(torch.int32)


def _plain_rotate(x, s, positions):
    rot = 2 * s["cos"].shape[1]
    y = x.to(torch.int64) * SCALE                      # what is not rotated keeps its value, with no remainder
    c, z = (s[n][positions].to(torch.int64)[:, None, :] for n in ("cos", "sin"))
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if s["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot))
    x0, x1 = x[..., a].to(torch.int64), x[..., b].to(torch.int64)
    y[..., a], y[..., b] = x0 * c - x1 * z, x0 * z + x1 * c
    return _rescale(y, SCALE)


def _plain_append(s):
    live = s["slots"] >= 0
    positions, slots = s["positions"][live].long(), s["slots"][live]
    s["q_out"][live], s["q_rem"][live] = _plain_rotate(s["q"][live], s, positions)
    k, s["k_rem"][live] = _plain_rotate(s["k"][live], s, positions)
    s["k_cache"].view(-1, *k.shape[1:])[slots] = k
    s["v_cache"].view(-1, *k.shape[1:])[slots] = s["v"][live]
    return s["q_out"], s["q_rem"], s["k_rem"], s["k_cache"], s["v_cache"]


def _plain_attend(s):
    b, h, d = s["q"].shape
    page, hk = s["k_cache"].shape[1:3]
    at = torch.arange(s["longest"], device="cuda")
    token = s["block_table"][:, at // page].clamp(min=0).long() * page + at % page             # [b][longest]
    live = at < s["lens"][:, None]
    if s["first"] is not None:
        live = live & (at >= s["first"][:, None])
    live = live[:, None, :]
    # float64 products of whole numbers: every sum stays below 2^53 and is exact
    q = s["q"].double().view(b, hk, h // hk, d)
    k = s["k_cache"].view(-1, hk, d)[token].permute(0, 2, 3, 1).contiguous().double()           # [b][hk][d][longest]
    scores, scores_rem = _rescale(torch.matmul(q, k).long().view(b, h, -1), s["qk_scale"])
    del k
    empty = ~live.any(-1)
    top = torch.where(live, scores, -(1 << 31)).amax(-1)
    top = torch.where(empty, 0, top)
    x = scores.long() - top.long()[..., None]
    index = x + ((1 << BIT_SHIFT) - 1)
    e = s["table"][torch.where((index >= 0) & (index < 1 << INDEX_BITS), index, 0)].long()
    e = torch.where(live, e, 0)
    total = e.sum(-1)
    denominator = torch.where(empty, 1, total)[..., None]
    p = torch.div(e * SCALE + denominator // 2, denominator, rounding_mode="floor")
    query = e * (2 * SCALE) - denominator * (2 * p - 1)
    p = torch.where(live, p, 0)
    v = s["v_cache"].view(-1, hk, d)[token].permute(0, 2, 1, 3).contiguous().double()           # [b][hk][longest][d]
    y, y_rem = _rescale(torch.matmul(p.double().view(b, hk, h // hk, -1), v).long().view(b, h, d), SCALE)
    del v
    out = s["out"]
    out["qkv"].copy_(y), out["qkv_rem"].copy_(y_rem)
    if "scores" in out:
        out["max"].copy_(top), out["exp_sum"].copy_(total)
        out["scores"].copy_(torch.where(live, scores, out["scores"]))
        out["scores_rem"].copy_(torch.where(live, scores_rem, out["scores_rem"]))
        out["exp_input"].copy_(torch.where(live, x, out["exp_input"].long()))
        out["exp_output"].copy_(torch.where(live, e, out["exp_output"].long()))
        out["softmax_output"].copy_(torch.where(live, p, out["softmax_output"].long()))
        out["softmax_lookup_query"].copy_(torch.where(live, query, out["softmax_lookup_query"].long()))
    return out


def _plain_q4(s):
    n, k = s["x"].shape
    m, group = s["w"].shape[0], s["group"]
    w = torch.stack((s["w"] & 15, s["w"] >> 4), dim=-1).view(m, -1)[:, :k].to(torch.int32)
    which = torch.arange(k, device="cuda") // group
    zeros = s["zeros"][:, which].to(torch.int32) if s["zeros"] is not None else 8
    w = (w - zeros) * s["scales"][:, which]
    # float64 products of whole numbers, exact below 2^53
    y, y_rem = _rescale(torch.matmul(s["x"].double(), w.double().t().contiguous()).long(), SCALE)
    s["y"].copy_(y), s["y_rem"].copy_(y_rem)
    return s["y"], s["y_rem"]


# ------------------------------------------------------------------ the definition, in 64-bit whole numbers on the host
def _split(y, scale):
    q = (y + scale // 2) // scale
    return q, y - q * scale


def _host(t):
    return t.cpu().numpy().astype(np.int64)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        rows = []
        for name in ("q", "k"):
            x, c, z = _host(s[name]), _host(s["cos"]), _host(s["sin"])
            y, half = x * SCALE, case["rot"] // 2
            for j in range(half):
                a, b = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + half)
                cj, zj = (t[_host(s["positions"]), j][:, None] for t in (c, z))
                y[:, :, a], y[:, :, b] = x[:, :, a] * cj - x[:, :, b] * zj, x[:, :, b] * cj + x[:, :, a] * zj
            rows.append(_split(y, SCALE))
        q_out, q_rem, k_rem, k_cache, v_cache = (_host(s[n]) for n in ("q_out", "q_rem", "k_rem", "k_cache", "v_cache"))
        v, page = _host(s["v"]), case["page"]
        for t, slot in enumerate(_host(s["slots"])):
            if slot >= 0:
                q_out[t], q_rem[t], k_rem[t] = rows[0][0][t], rows[0][1][t], rows[1][1][t]
                k_cache[slot // page, slot % page], v_cache[slot // page, slot % page] = rows[1][0][t], v[t]
        return tuple(x.astype(np.int32) for x in (q_out, q_rem, k_rem, k_cache, v_cache))
    if case["op"] == "attend":
        lens, first = _lengths(case)
        out = {n: _host(t) for n, t in s["out"].items()}
        q, table, pages = _host(s["q"]), _host(s["table"]), _host(s["block_table"])
        each, page = case["heads"] // case["kv_heads"], case["page"]
        for b, (n, f) in enumerate(zip(lens, first)):
            at = np.arange(f, n)
            where = torch.from_numpy(pages[b][at // page] * page + at % page).cuda()
            shape = (-1, case["kv_heads"], case["dim"])
            keys, values = (_host(s[c].view(shape)[where]) for c in ("k_cache", "v_cache"))
            for h in range(case["heads"]):
                kv = h // each
                got = {"qkv": 0, "qkv_rem": 0, "max": 0, "exp_sum": 0}
                if n > f:
                    score, rem = _split((keys[:, kv] * q[b, h]).sum(1), s["qk_scale"])
                    e = table[score - score.max() + (1 << BIT_SHIFT) - 1]
                    total = int(e.sum())
                    p = (e * SCALE + total // 2) // total
                    got["qkv"], got["qkv_rem"] = _split((values[:, kv] * p[:, None]).sum(0), SCALE)
                    got |= {"max": score.max(), "exp_sum": total, "scores": score, "scores_rem": rem, "exp_input": score - score.max(),
                            "exp_output": e, "softmax_output": p, "softmax_lookup_query": 2 * SCALE * e - total * (2 * p - 1)}
                for name, x in got.items():
                    if name in ("qkv", "qkv_rem", "max", "exp_sum"):
                        if name in out:
                            out[name][b, h] = x
                    elif name in out:
                        out[name][b, h, f:n] = x
        return {n: x.astype(np.int32) for n, x in out.items()}
    x, packed, scales = _host(s["x"]), _host(s["w"]), _host(s["scales"])
    zeros = _host(s["zeros"]) if case["zeros"] else np.full_like(scales, 8)
    y = np.zeros((case["tokens"], case["outputs"]), dtype=np.int64)
    for g in range(scales.shape[1]):
        lo, hi = g * case["group"], min((g + 1) * case["group"], case["inputs"])
        w = np.stack([(packed[:, k // 2] >> (4 * (k % 2))) & 15 for k in range(lo, hi)], axis=1)
        for n in range(case["tokens"]):
            y[n] += scales[:, g] * ((w - zeros[:, g:g + 1]) * x[n, lo:hi]).sum(1)
    return tuple(t.astype(np.int32) for t in _split(y, SCALE))
