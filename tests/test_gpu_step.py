"""GPU parity tests of the calls around a step of new tokens (its pages and slots, attention of several tokens a sequence behind a
window, the choice of the next token) against the numpy oracle.  Every result is a whole number and is compared exactly."""
import numpy as np
import pytest
import torch
from oracle import witness_oracle as wo
from test_gpu_tokens import PROOF, TOP, UNTOUCHED, dev, exp_table, filled, gauss, host, ops, paged  # noqa: F401  (ops, exp_table are fixtures)

pytestmark = pytest.mark.gpu

LOWEST = -(1 << 31)


# ------------------------------------------------------------------ pages and slots
def pages_case(rng, seqs, longest, most, page, spare=5, ended=True, zero=True):
    """lengths, new tokens, a block table with scattered pages and a ring with the free ones somewhere in it"""
    lens = rng.integers(0, longest + 1, seqs)
    new = rng.integers(1, most + 1, seqs)
    if ended:
        new[rng.random(seqs) < 0.2] = -1
    if zero:
        new[rng.random(seqs) < 0.2] = 0
        lens[rng.random(seqs) < 0.2] = 0
    held, after = -(-lens // page), -(-(lens + np.maximum(new, 0)) // page)
    width = int(after.max(initial=0)) + 2
    pages = int(after.sum()) + spare
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((seqs, width), -9, dtype=np.int32)
    at = 0
    for b in range(seqs):
        table[b, :held[b]] = order[at:at + held[b]]
        at += held[b]
    ring = np.full(2 * pages, -5, dtype=np.int32)
    head, count = int(rng.integers(0, 2 * pages)), pages - at
    ring[(head + np.arange(count)) % (2 * pages)] = order[at:]
    return {"lens": lens, "new": new, "table": table, "ring": ring, "span": [head, count], "page": page, "rows": int(np.maximum(new, 0).sum()) + 3}


def run_pages(ops, c, window=0, sinks=0, status=0):
    table, ring = c["table"].copy(), c["ring"].copy()
    want, short = wo.page_step(c["lens"], c["new"], table, ring, c["span"], c["page"], c["rows"], window, sinks)
    d = {x: dev(np.asarray(c[x])) for x in ("lens", "new", "table", "ring", "span")}
    got = ops.wit_page_step(d["lens"], d["new"], d["table"], d["ring"], d["span"], c["page"], c["rows"], window=window, sinks=sinks)
    assert got["slots"].dtype is torch.int64
    for x, t in want.items():
        assert host(got[x]).tolist() == list(t), x
    assert np.array_equal(host(d["table"]), table) and np.array_equal(host(d["ring"]), ring)
    assert ops.wit_status() == (32 if short else 0) | status
    return got, d


@pytest.mark.parametrize("seqs,longest,most,page", [(1, 0, 1, 1), (1, 100, 1, 16), (3, 5, 9, 1), (64, 300, 1, 16), (65, 50, 40, 17), (200, 3000, 30, 64), (257, 20, 3, 5),
                                                    (1025, 100, 7, 16), (4096, 40, 4, 7), (7, 4000, 5000, 100)])
def test_pages_and_slots(ops, seqs, longest, most, page):
    rng = np.random.default_rng(seqs + longest + page)
    c = pages_case(rng, seqs, longest, most, page)
    for window, sinks in ((0, 0), (1, 0), (20, 0), (20, 3), (20, page), (700, 33), (1 << 30, 5), (3, 1 << 30)):
        run_pages(ops, c, window, sinks)


def test_pages_that_run_out(ops):
    """rows, free pages or room in the ring that do not suffice, at every place of the batch"""
    rng = np.random.default_rng(2)
    c = pages_case(rng, 40, 100, 30, 8)
    need = int((-(-(c["lens"] + np.maximum(c["new"], 0)) // 8) - -(-c["lens"] // 8)).sum())
    for rows in (0, 1, 50, 100, c["rows"] - 4, c["rows"] - 3):
        run_pages(ops, {**c, "rows": rows}, 20, 3)
    for count in (0, 1, need // 2, need - 1, need):
        run_pages(ops, {**c, "span": [c["span"][0], count]}, 20, 3)
    # a ring that is full: what comes back has no room beyond what it had
    for size in (c["span"][1], c["span"][1] + 3):
        ring = np.concatenate((np.roll(c["ring"], -c["span"][0])[:c["span"][1]], np.full(3, -5, dtype=np.int32)))[:size]
        run_pages(ops, {**c, "ring": ring, "span": [0, c["span"][1]]}, 20, 3)


def test_pages_of_bad_numbers(ops):
    rng = np.random.default_rng(3)
    c = pages_case(rng, 9, 60, 10, 8, ended=False, zero=False)
    most = c["table"].shape[1] * 8
    for ln, new in ((-1, 2), (-(1 << 31), 0), (5, -2), (5, -(1 << 31)), (most, 1), (most + 1, 0), ((1 << 31) - 1, (1 << 31) - 1), (3, (1 << 31) - 1)):
        lens, news = c["lens"].copy(), c["new"].copy()
        lens[4], news[4] = ln, new
        run_pages(ops, {**c, "lens": lens, "new": news}, 16, 0, status=2)
    table = c["table"].copy()
    lens, news = np.full(9, 5), np.full(9, 2)
    table[:, 0] = np.arange(9)
    table[4, 0] = -1                                    # the last page that a sequence holds is none
    got, _ = run_pages(ops, {**c, "lens": lens, "new": news, "table": table}, status=2)
    assert host(got["slots"]).tolist()[8:10] == [-1, -1]
    for head, count in ((-1, 0), (len(c["ring"]), 0), (0, -1), (0, len(c["ring"]) + 1)):
        d = {x: dev(np.asarray(c[x])) for x in ("lens", "new", "table", "ring")}
        got = ops.wit_page_step(d["lens"], d["new"], d["table"], d["ring"], dev(np.array([head, count])), 8, c["rows"])
        assert ops.wit_status() & 2 and host(got["free_span"]).tolist() == [head, count] and np.array_equal(host(d["ring"]), c["ring"])


def test_pages_of_no_sequences_and_no_rows(ops):
    i32 = dict(dtype=torch.int32, device="cuda")
    got = ops.wit_page_step(torch.zeros(0, **i32), torch.zeros(0, **i32), torch.zeros((0, 4), **i32), torch.zeros(8, **i32), dev(np.array([3, 2])), 16, 5)
    assert host(got["starts"]).tolist() == [0] and host(got["slots"]).tolist() == [-1] * 5 and host(got["free_span"]).tolist() == [3, 2]
    got = ops.wit_page_step(dev(np.array([0])), dev(np.array([0])), torch.zeros((1, 0), **i32), torch.zeros(0, **i32), dev(np.array([0, 0])), 16, 0)
    assert host(got["starts"]).tolist() == [0, 0] and host(got["free_span"]).tolist() == [0, 0]
    assert ops.wit_status() == 0


def test_pages_of_a_conversation(ops):
    """steps of requests that come, grow behind a window and go: every page is in one place, and what a token sees stays where it is"""
    rng = np.random.default_rng(4)
    seqs, page, window, sinks, pages = 6, 4, 10, 5, 60
    ring = np.full(2 * pages, -1, dtype=np.int32)
    ring[:pages] = rng.permutation(pages)
    d = {"ring": dev(ring), "span": dev(np.array([0, pages])), "table": filled(seqs, 40), "lens": dev(np.zeros(seqs, dtype=np.int64))}
    owner = {}
    for step in range(40):
        lens = host(d["lens"])
        new = rng.integers(0, 4, seqs)
        new[lens > 100] = -1
        new[rng.random(seqs) < 0.05] = -1
        out = ops.wit_page_step(d["lens"], dev(new), d["table"], d["ring"], d["span"], page, 24, window=window, sinks=sinks)
        table, slots, pos, starts = host(d["table"]), host(out["slots"]), host(out["positions"]), host(out["starts"])
        for b in range(seqs):
            if new[b] < 0:
                owner = {k: v for k, v in owner.items() if k[0] != b}
            for r in range(starts[b], starts[b + 1]):
                owner[b, pos[r]] = slots[r]
                for t in range(pos[r] + 1):
                    if t > pos[r] - window or t < sinks:
                        assert owner[b, t] == table[b, t // page] * page + t % page
            live = {t: s for (x, t), s in owner.items() if x == b and (t > lens[b] + new[b] - window or t < sinks)}
            owner = {k: v for k, v in owner.items() if k[0] != b} | {(b, t): s for t, s in live.items()}
        assert len(set(owner.values())) == len(owner)
        d["lens"], d["span"] = out["lens"], out["free_span"]
        head, count = host(d["span"])
        free = host(d["ring"])[(head + np.arange(count)) % (2 * pages)]
        held = {s // page for s in owner.values()}
        assert len(set(free.tolist())) == count and not held & set(free.tolist()) and count >= pages - seqs * ((window + sinks) // page + 3)
    assert ops.wit_status() == 0


def test_drafted_tokens_are_taken_back(ops):
    """without a window: a shorter length, and the pages behind it at the ring's end by the caller's hand; every page stays in one place"""
    rng = np.random.default_rng(6)
    seqs, page, pages, width = 5, 4, 200, 40
    ring = np.full(2 * pages, -1, dtype=np.int32)
    ring[:pages] = rng.permutation(pages)
    ring, span, table, lens = dev(ring), dev(np.array([0, pages])), filled(seqs, width), dev(rng.integers(0, 1, seqs))
    at = torch.arange(width, device="cuda")
    for step in range(30):
        out = ops.wit_page_step(lens, dev(rng.integers(1, 12, seqs)), table, ring, span, page, 60)
        shorter = torch.maximum(lens, out["lens"] - dev(rng.integers(0, 9, seqs)))
        up = lambda n: ((n + page - 1) // page)[:, None]  # noqa: E731
        back = table[(at >= up(shorter)) & (at < up(out["lens"]))]
        head, count = host(out["free_span"]).tolist()
        ring[(head + count + torch.arange(len(back), device="cuda")) % (2 * pages)] = back
        span, lens = dev(np.array([head, count + len(back)])), shorter
        held = table[at < up(lens)]
        free = ring[(head + torch.arange(count + len(back), device="cuda")) % (2 * pages)]
        assert sorted(host(torch.cat((held, free))).tolist()) == list(range(pages)), step
        if bool((lens > 130).any()):
            break
    assert ops.wit_status() == 0


# ------------------------------------------------------------------ attention
def run_window(ops, q, kc, vc, table, starts, lens, exp_table, max_new, max_len, window=0, sinks=0, proof=True, keep=None, **kw):
    rows, H, D = q.shape
    shapes = {"qkv": (rows, H, D), "qkv_rem": (rows, H, D)}
    if proof:
        shapes |= {x: (rows, H, max_len) for x in PROOF} | {"max": (rows, H), "exp_sum": (rows, H)}
    if keep:
        shapes = {x: shapes[x] for x in keep}
    want = {x: np.full(s, UNTOUCHED, dtype=np.int32) for x, s in shapes.items()}
    wo.window_attention(q, kc, vc, table, starts, lens, window, sinks, exp_table, want, **kw)
    got = {x: filled(*s) for x, s in shapes.items()}
    res = ops.wit_window_attention(dev(q), dev(kc), dev(vc), dev(table), dev(np.asarray(starts)), dev(np.asarray(lens)), max_new, max_len, dev(exp_table), window=window,
                                   sinks=sinks, out=got, **kw)
    assert res is got
    for x in shapes:
        assert np.array_equal(host(got[x]), want[x]), (x, int((host(got[x]) != want[x]).sum()), np.argwhere(host(got[x]) != want[x])[:3].tolist())
    return got


def starts_of(new):
    return np.concatenate(([0], np.cumsum(new)))


WINDOWS = [
    # new tokens, lengths, heads, cache heads, dim, page, window, sinks
    ([1], [1], 1, 1, 1, 1, 0, 0), ([3], [3], 2, 1, 3, 2, 0, 0), ([5], [70], 4, 2, 64, 16, 0, 0), ([2, 0, 7], [2, 9, 40], 4, 2, 50, 7, 0, 0),
    ([64], [64], 1, 1, 32, 16, 0, 0), ([65, 1, 63], [65, 130, 64], 2, 2, 16, 16, 0, 0), ([30], [200], 12, 4, 80, 17, 50, 4), ([30], [200], 12, 4, 80, 17, 1, 0),
    ([20, 33], [300, 33], 7, 1, 20, 5, 64, 70), ([70], [70], 3, 1, 100, 16, 20, 1), ([9], [500], 8, 1, 96, 64, 100, 65), ([11], [333], 5, 5, 33, 8, 1000, 9),
    ([150], [260], 1, 1, 260, 32, 0, 0), ([17], [90], 1, 1, 1024, 16, 33, 2), ([4, 4, 4, 4, 4], [4, 100, 57, 1000, 8], 16, 2, 128, 16, 0, 0),
    ([1, 1, 1], [1, 70, 600], 8, 2, 64, 16, 30, 4), ([1] * 9, [9, 1, 300, 44, 45, 46, 47, 600, 599], 4, 1, 40, 16, 45, 1), ([2], [1400], 2, 1, 256, 100, 0, 0),
    ([100], [130], 65, 1, 8, 16, 0, 0), ([3], [5], 130, 2, 4, 3, 2, 1)]


@pytest.mark.parametrize("new,lens,H,HK,D,page,window,sinks", WINDOWS)
def test_window_attention_matches_the_oracle(ops, exp_table, new, lens, H, HK, D, page, window, sinks):
    rng = np.random.default_rng(sum(lens) + H + D)
    table, kc, vc = paged(rng, lens, page, HK, D)
    starts = starts_of(new) + 1                           # the first row and the last are of no sequence
    q = gauss(rng, (int(starts[-1]) + 2, H, D))
    scale = int(round(65536 * D ** 0.5)) if D > 4 else 1 << 17
    full = run_window(ops, q, kc, vc, table, starts, lens, exp_table, max(new), max(lens) + 3, window, sinks, qk_scale=scale)
    answer = run_window(ops, q, kc, vc, table, starts, lens, exp_table, max(new) + 2 if max(new) < max(lens) else max(new), max(lens), window, sinks, proof=False, qk_scale=1 << (22 if D >= 64 else 20))
    assert set(answer) == {"qkv", "qkv_rem"} and ops.wit_status() == 0
    # pages that nobody sees are not read
    if window:
        first = [max(0, n - m + 1 - window) for n, m in zip(lens, new)]
        for b in range(len(lens)):
            for i in range(table.shape[1]):
                if i * page >= sinks and (i + 1) * page <= first[b]:
                    table[b, i] = -3
        again = {x: filled(*t.shape) for x, t in full.items()}
        ops.wit_window_attention(dev(q), dev(kc), dev(vc), dev(table), dev(starts), dev(np.array(lens)), max(new), max(lens) + 3, dev(exp_table), window=window, sinks=sinks, out=again, qk_scale=scale)
        assert all(torch.equal(again[x], full[x]) for x in full) and ops.wit_status() == 0


def test_window_attention_of_many_sequences(ops, exp_table):
    rng = np.random.default_rng(20)
    for seqs, H, HK, D in ((65, 2, 1, 16), (200, 1, 1, 8), (4100, 1, 1, 4)):
        new = rng.integers(0, 4, seqs)
        lens = new + rng.integers(0, 20, seqs)
        table, kc, vc = paged(rng, lens.tolist(), 4, HK, D)
        q = gauss(rng, (int(new.sum()), H, D))
        run_window(ops, q, kc, vc, table, starts_of(new), lens, exp_table, 3, 23, 9, 2, qk_scale=1 << 18)
    assert ops.wit_status() == 0


def test_window_attention_is_the_single_tokens_one(ops, exp_table):
    """of one token a sequence, wit_paged_attention; of a prompt, its tokens one after the other"""
    rng = np.random.default_rng(21)
    lens = [300, 1, 77, 128]
    table, kc, vc = paged(rng, lens, 16, 2, 64)
    q = gauss(rng, (4, 8, 64))
    a = ops.wit_paged_attention(dev(q), dev(kc), dev(vc), dev(table), dev(np.array(lens)), 300, dev(exp_table), first=dev(np.maximum(np.array(lens) - 50, 0)), qk_scale=1 << 19)
    b = ops.wit_window_attention(dev(q), dev(kc), dev(vc), dev(table), dev(np.arange(5)), dev(np.array(lens)), 1, 300, dev(exp_table), window=50, qk_scale=1 << 19)
    c = ops.wit_window_attention(dev(q), dev(kc), dev(vc), dev(table), dev(np.arange(5)), dev(np.array(lens)), 2, 300, dev(exp_table), window=50, qk_scale=1 << 19)
    assert set(a) == set(b) == set(c) and all(torch.equal(a[x], b[x]) and torch.equal(a[x], c[x]) for x in a)
    n = 100
    q = gauss(rng, (n, 8, 64))
    prompt = ops.wit_window_attention(dev(q), dev(kc), dev(vc), dev(table[:1]), dev(np.array([0, n])), dev(np.array([300])), n, 300, dev(exp_table), qk_scale=1 << 19)
    alone = ops.wit_paged_attention(dev(q), dev(kc), dev(vc), dev(np.repeat(table[:1], n, 0)), dev(np.arange(201, 301)), 300, dev(exp_table), qk_scale=1 << 19)
    assert all(torch.equal(prompt[x], alone[x]) for x in prompt) and ops.wit_status() == 0


@pytest.mark.parametrize("prob_scale,out_scale", [(1 << 22, 1 << 22), (1 << 30, 1 << 31), (1, 1), (3000, 777), ((1 << 22) + 1, 1 << 20)])
def test_window_attention_over_its_scales(ops, exp_table, prob_scale, out_scale):
    rng = np.random.default_rng(prob_scale % 1000)
    table, kc, vc = paged(rng, [70, 300], 16, 2, 64, sigma=20000.0)
    run_window(ops, gauss(rng, (50, 8, 64)), kc, vc, table, [0, 40, 50], [70, 300], exp_table, 40, 300, 90, 3, qk_scale=100000, prob_scale=prob_scale, out_scale=out_scale)
    assert ops.wit_status() == 0


@pytest.mark.parametrize("where", ["queries", "keys", "values", "all"])
def test_window_attention_of_the_largest_values(ops, exp_table, where):
    """queries, keys and values at the ends of 32 bits, beside ordinary ones: the products fill 64 bits"""
    rng = np.random.default_rng(8)
    H, HK, D, page, new, lens = 4, 2, 64, 16, [40, 3], [150, 70]
    ends = np.array([-(1 << 31), (1 << 31) - 1, TOP, TOP + 1, -TOP - 1, 0x7F7F7F, 0x7F7F80, -0x808080, -0x808081, 0], dtype=np.int64)
    table, kc, vc = paged(rng, lens, page, HK, D)
    q = rng.integers(-3, 4, (43, H, D)).astype(np.int32)
    kc[:] = gauss(rng, kc.shape, 1000.0)
    kc[..., 2] = rng.integers(0, 1 << 19, kc.shape[:3])
    q[..., 0], q[..., 1], q[..., 2] = 1, -1, 1
    if where in ("keys", "all"):                        # the large parts of a key cancel in its score, the rest stays within the table
        kc[..., 0] = kc[..., 1] = rng.choice(ends, kc.shape[:3])
    if where in ("queries", "all"):                     # and those of a query
        q[..., 3] = q[..., 4] = rng.choice(ends, q.shape[:2])
        kc[..., 3] = rng.integers(-100, 100, kc.shape[:3])
        kc[..., 4] = -kc[..., 3]
    if where in ("values", "all"):
        vc[..., ::3] = rng.choice(ends, vc[..., ::3].shape)
    run_window(ops, q, kc, vc, table, starts_of(new), lens, exp_table, 40, 150, 60, 5, qk_scale=2)
    if where == "all":                                  # the largest queries and keys: scores next to the ends of 32 bits
        q[:] = 0
        q[:, :, 0] = rng.choice(np.array([(1 << 31) - 1, -(1 << 31)]), q.shape[:2])
        kc[..., 0] = rng.choice(np.array([TOP, TOP + 1, TOP + 7, TOP + 1000], dtype=np.int64), kc.shape[:3])
        run_window(ops, q, kc, vc, table, starts_of(new), lens, exp_table, 40, 150, qk_scale=1 << 31)
    assert ops.wit_status() == 0


@pytest.mark.parametrize("max_new", [1, 6])
def test_window_attention_reports_bad_sequences_and_pages(ops, exp_table, max_new):
    rng = np.random.default_rng(9)
    H, HK, D, page, L = 4, 2, 64, 16, 100
    new = [max_new, 1, 1]
    lens = [L, L - 1, 7]
    starts = starts_of(new)
    table, kc, vc = paged(rng, lens, page, HK, D)
    q = gauss(rng, (int(starts[-1]), H, D))
    for bad in (-1, kc.shape[0], (1 << 31) - 1, -(1 << 31)):
        t = table.copy()
        t[1, 1] = bad                                              # its keys and values count as zero
        run_window(ops, q, kc, vc, t, starts, lens, exp_table, max_new, L, qk_scale=65536 * 8)
        assert ops.wit_status() == 2
    good = run_window(ops, q, kc, vc, table, starts, lens, exp_table, max_new, L, 40, 2, qk_scale=65536 * 8)
    assert ops.wit_status() == 0
    s = starts
    for st, ln in (([0, s[1], s[2], s[3]], L + 1), ([0, s[1], s[2], s[3]], -1), ([0, s[1], s[2], s[3]], 0), ([0, s[1], s[2], s[3]], -(1 << 31)), ([0, s[1], s[2], s[3]], (1 << 31) - 1),
                   ([0, s[1], s[2], s[3]], table.shape[1] * page + 1)):
        got = {x: filled(*t.shape) for x, t in good.items()}
        ops.wit_window_attention(dev(q), dev(kc), dev(vc), dev(table), dev(np.array(st)), dev(np.array([L, ln, 7])), max_new, L, dev(exp_table), window=40, sinks=2, out=got, qk_scale=65536 * 8)
        assert ops.wit_status() == 2
        for x in good:
            want = good[x].clone()
            want[s[1]:s[2]] = UNTOUCHED
            assert torch.equal(got[x], want), (st, ln, x)
    # starts that lead anywhere: nothing but rows of the call is written, and the bit is set
    for st in ([0, -1, 2, 3], [-(1 << 31), 0, 1, 2], [0, 1, (1 << 31) - 1, 2], [5, 4, 3, 2], [0, 9, 9, 9], [0, 0, 0, 99], [0, max_new + 1, max_new + 1, max_new + 1], [7, 7, 0, 1]):
        q2 = dev(q)
        got = {x: filled(*t.shape) for x, t in good.items()}
        ops.wit_window_attention(q2, dev(kc), dev(vc), dev(table), dev(np.array(st)), dev(np.array(lens)), max_new, L, dev(exp_table), window=40, sinks=2, out=got, qk_scale=65536 * 8)
        assert ops.wit_status() & 2, st


@pytest.mark.parametrize("new,H,HK,D", [([128, 20, 12, 30], 2, 2, 64), ([300, 280, 260, 290], 16, 2, 128), ([2, 1, 3] * 30, 4, 1, 32), ([1] * 199 + [2], 2, 1, 16), ([1] * 100, 2, 1, 64)])
def test_window_attention_beside_starts_that_are_no_rows(ops, exp_table, new, H, HK, D):
    """a start that is no row of the call leaves the rows of the two sequences that it bounds as they were, and all others get theirs"""
    rng = np.random.default_rng(sum(new))
    lens, page = [n + int(x) for n, x in zip(new, rng.integers(0, 40, len(new)))], 16
    table, kc, vc = paged(rng, lens, page, HK, D)
    starts, L, n = starts_of(new), max(lens), len(new)
    q, k, v, lens = gauss(rng, (int(starts[-1]), H, D)), dev(kc), dev(vc), dev(np.array(lens))
    call = lambda st, **kw: ops.wit_window_attention(dev(q), k, v, dev(table), dev(st), lens, max(new), L, dev(exp_table), qk_scale=65536 * 11, **kw)  # noqa: E731
    shapes = {"qkv": q.shape, "qkv_rem": q.shape, "max": q.shape[:2], "exp_sum": q.shape[:2]} | {x: q.shape[:2] + (L,) for x in PROOF}
    want = call(starts, out={x: filled(*t) for x, t in shapes.items()})
    assert ops.wit_status() == 0
    for bad in ([n // 2], [1], [0], [n], [n - 1, n], list(range(n // 3, n)), [1, n // 2, n - 1], list(range(0, n, 3)), list(range(0, n + 1, 64))):
        st = starts.copy()
        st[bad] = rng.choice([-1, len(q) + 1, (1 << 31) - 1, -(1 << 31)], len(bad))
        out = call(st, out={x: filled(*t.shape) for x, t in want.items()})
        assert ops.wit_status() == 2
        gone = {b for i in bad for b in (i - 1, i)}
        there = torch.tensor([b not in gone for b in range(n) for _ in range(new[b])], device="cuda")
        for x in shapes:
            assert torch.equal(out[x][there], want[x][there]) and bool((out[x][~there] == UNTOUCHED).all()), (bad, x)


def test_window_attention_reports_its_table_and_sums(ops, exp_table):
    rng = np.random.default_rng(10)
    table, kc, vc = paged(rng, [200], 16, 1, 64)
    q = gauss(rng, (70, 2, 64))
    args = (dev(q), dev(kc), dev(vc), dev(table), dev(np.array([0, 70])), dev(np.array([200])), 70, 200)
    ops.wit_window_attention(*args, dev(exp_table), qk_scale=1 << 10)       # scores spread over far more than the table
    assert ops.wit_status() & 2
    got = ops.wit_window_attention(*args, torch.zeros(1 << 20, dtype=torch.int32, device="cuda"), qk_scale=1 << 19)
    assert ops.wit_status() == 4 and bool((got["exp_sum"] == 1).all()) and bool((got["qkv"] == 0).all())
    neg = exp_table.copy()
    neg[-1] = -5
    ops.wit_window_attention(*args, dev(neg), qk_scale=1 << 19)
    assert ops.wit_status() & 4
    ops.wit_window_attention(*args, dev(exp_table), qk_scale=1)
    assert ops.wit_status() & 1
    # other tables: of few entries, of another scale, with one entry that is off
    for bits, scale in ((10, 128.0), (16, 4096.0), (20, 60000.0)):
        other = np.rint(np.exp((np.arange(1 << bits) - ((1 << bits) - 1)) / scale) * 65536).astype(np.int32)
        run_window(ops, q, kc, vc, table, [0, 70], [200], other, 70, 200, 0, 0, qk_scale=1 << (39 - bits), bit_shift=bits, index_bits=bits)
    for at in (-1, -2, -1000, -65537, 0):
        other = exp_table.copy()
        other[at] += 1
        run_window(ops, q, kc, vc, table, [0, 70], [200], other, 70, 200, 0, 0, qk_scale=1 << 19)
    more = np.concatenate((exp_table[-(1 << 19):], np.arange(1 << 19, dtype=np.int32)))          # entries past that of the maximum
    run_window(ops, q, kc, vc, table, [0, 70], [200], more, 70, 200, 0, 0, qk_scale=1 << 20, bit_shift=19)
    assert ops.wit_status() == 0
    # sums beyond int32 are said to be
    equal = np.zeros((1, 1, 8), dtype=np.int32)
    heavy = np.full(1 << 20, 1 << 29, dtype=np.int32)
    t2, k2, v2 = paged(rng, [9], 16, 1, 8)
    ops.wit_window_attention(dev(np.repeat(equal, 2, 0)), dev(k2), dev(v2), dev(t2), dev(np.array([0, 2])), dev(np.array([9])), 2, 9, dev(heavy))
    assert ops.wit_status() == 16


def test_window_attention_of_strided_caches_and_queries(ops, exp_table):
    rng = np.random.default_rng(11)
    for new, lens, H, HK, D, page in (([20, 7], [33, 70], 6, 3, 64, 16), ([1, 1], [900, 130], 8, 2, 64, 16), ([9, 9], [40, 9], 2, 2, 30, 7)):
        table, kc, vc = paged(rng, lens, page, HK, D)
        starts = starts_of(new)
        q = gauss(rng, (int(starts[-1]), H, D))
        good = run_window(ops, q, kc, vc, table, starts, lens, exp_table, max(new), max(lens), 30, 2, qk_scale=65536 * 8)
        for pad, at in ((5, 1), (4, 4)):
            wide = torch.zeros((len(q), H * D + pad), dtype=torch.int32, device="cuda")
            wq = wide[:, at:at + H * D].view(len(q), H, D) if at + H * D <= wide.shape[1] else wide[:, :H * D].view(len(q), H, D)
            wq.copy_(dev(q))
            P = kc.shape[0]
            for make in (lambda: filled(HK, P, page, D).permute(1, 2, 0, 3), lambda: filled(P, page, HK, D + 3)[..., :D],
                         lambda: filled(P, HK, page, D).permute(0, 2, 1, 3), lambda: filled(P * page * HK * D + 1)[1:].view(P, page, HK, D)):
                a, b = make(), make()
                a.copy_(dev(kc)), b.copy_(dev(vc))
                got = ops.wit_window_attention(wq, a, b, dev(table), dev(starts), dev(np.array(lens)), max(new), max(lens), dev(exp_table), window=30, sinks=2, qk_scale=65536 * 8,
                                               out={x: filled(*t.shape) for x, t in good.items()})
                assert all(torch.equal(got[x], good[x]) for x in good)
    assert ops.wit_status() == 0


@pytest.mark.parametrize("new,lens", [([1, 1], [50, 700]), ([50, 20], [50, 100]), ([3, 2], [1500, 700])])
def test_window_attention_with_some_outputs_and_a_kept_workspace(ops, exp_table, new, lens):
    rng = np.random.default_rng(12)
    table, kc, vc = paged(rng, lens, 16, 2, 64)
    starts, L = starts_of(new), max(lens)
    q = gauss(rng, (int(starts[-1]), 4, 64))
    good = run_window(ops, q, kc, vc, table, starts, lens, exp_table, max(new), L, 300, 4, qk_scale=65536 * 8)
    size = ops.wit_window_attention_workspace(len(q), 2, 4, 2, 64, max(new), L, 300, 4)
    ws = torch.randint(-128, 127, (size,), device="cuda", dtype=torch.int8).view(torch.uint8)
    args = (dev(q), dev(kc), dev(vc), dev(table), dev(starts), dev(np.array(lens)), max(new), L, dev(exp_table))
    for keep in (("qkv",), ("qkv", "scores"), ("qkv", "exp_output", "max"), ("qkv", "softmax_output", "exp_sum"), ("qkv", "qkv_rem", "softmax_lookup_query"),
                 ("qkv", "exp_input", "scores_rem")):
        got = ops.wit_window_attention(*args, window=300, sinks=4, qk_scale=65536 * 8, out={x: filled(*good[x].shape) for x in keep}, workspace=ws)
        assert all(torch.equal(got[x], good[x]) for x in keep), keep
    fresh = ops.wit_window_attention(*args, window=300, sinks=4, qk_scale=65536 * 8)
    assert set(fresh) == set(good) and torch.equal(fresh["qkv"], good["qkv"]) and not bool((fresh["scores"] == UNTOUCHED).any())
    assert ops.wit_status() == 0


@pytest.mark.parametrize("lens,max_len,window,sinks", [([5000, 1, 1023, 1024, 1025, 1028, 1029, 3000, 0], 6000, 1024, 4), ([700, 300, 299, 257], 100000, 256, 0), ([900, 2000], 2000, 300, 900),
                                                       ([20, 60, 0, 400], 500, 40, 3), ([100000, 3], 100000, 5000, 70)])
def test_single_tokens_keep_what_they_see_and_no_more(ops, exp_table, lens, max_len, window, sinks):
    """scores and exponentials in a workspace of exactly its size, whose rows are as long as the window and the sinks: the answer, with or
    without some of a proof's rows, is that of the call for several tokens, and nothing stands behind the workspace"""
    rng = np.random.default_rng(sum(lens))
    H, HK, D, page = 8, 2, 64, 16
    new = [min(n, 1) for n in lens]
    table, kc, vc = paged(rng, lens, page, HK, D)
    starts = starts_of(new) + 1
    q = gauss(rng, (int(starts[-1]) + 1, H, D))
    args = (dev(q), dev(kc), dev(vc), dev(table), dev(starts), dev(np.array(lens)))
    kw = {"window": window, "sinks": sinks, "qk_scale": 1 << 19}
    shapes = {"qkv": (len(q), H, D), "qkv_rem": (len(q), H, D), "scores": (len(q), H, max_len), "exp_output": (len(q), H, max_len), "softmax_output": (len(q), H, max_len),
              "scores_rem": (len(q), H, max_len), "exp_sum": (len(q), H)}
    want = ops.wit_window_attention(*args, 2, max_len, dev(exp_table), out={x: filled(*t) for x, t in shapes.items()}, **kw)
    size = ops.wit_window_attention_workspace(len(q), len(lens), H, HK, D, 1, max_len, window, sinks)
    assert size < 4 * len(q) * H * (window + sinks) * 4 + len(q) * H * D * 8 * 40 + 4096
    for keep in (("qkv", "qkv_rem"), ("qkv", "scores"), ("qkv", "exp_output"), ("qkv", "softmax_output", "scores_rem", "exp_sum"), tuple(shapes)):
        space = torch.randint(-128, 127, (size + 4096,), device="cuda", dtype=torch.int8).view(torch.uint8)
        behind = space[size:].clone()
        got = ops.wit_window_attention(*args, 1, max_len, dev(exp_table), out={x: filled(*shapes[x]) for x in keep}, workspace=space[:size] if size else None, **kw)
        for x in keep:
            assert torch.equal(got[x], want[x]), (keep, x)
        assert torch.equal(space[size:], behind)
    assert ops.wit_status() == 0


# ---- calls with many rows, whose queries, keys and values are turned into digits once
def alone(ops, q, kc, vc, table, starts, lens, exp_table, max_len, window=0, sinks=0, **kw):
    """each token as a sequence of its own, one new token long"""
    new = np.diff(starts)
    seq = np.repeat(np.arange(len(new)), new)
    ends = np.concatenate([np.arange(n - m + 1, n + 1) for n, m in zip(lens, new)]).astype(np.int64)
    rows = slice(int(starts[0]), int(starts[-1]))
    return ops.wit_window_attention(dev(q[rows]), kc, vc, dev(table[seq]), dev(np.arange(len(seq) + 1)), dev(ends), 1, max_len, dev(exp_table), window=window, sinks=sinks, **kw)


MANY = [
    # new tokens, lengths, heads, cache heads, dim, page, window, sinks: 256 rows of a cache head and more for each sequence, 2^30 products and more
    ([300], [640], 8, 1, 1024, 16, 0, 0), ([520], [1000], 8, 2, 260, 17, 0, 0), ([400], [500], 2, 1, 4096, 7, 100, 70), ([300, 0, 261], [900, 5, 261], 16, 2, 128, 16, 0, 0),
    ([512], [2049], 16, 2, 64, 100, 0, 0), ([700], [1700], 16, 2, 128, 16, 700, 4), ([1100], [1100], 30, 10, 33, 16, 0, 0), ([600, 400], [700, 777], 8, 2, 183, 32, 640, 130),
    ([513], [513], 16, 16, 255, 16, 0, 0), ([300], [2000], 4, 1, 515, 64, 0, 0)]


@pytest.mark.parametrize("new,lens,H,HK,D,page,window,sinks", MANY)
def test_window_attention_of_many_rows(ops, exp_table, new, lens, H, HK, D, page, window, sinks):
    rng = np.random.default_rng(sum(lens) + H + D)
    table, kc, vc = paged(rng, lens, page, HK, D)
    starts, L, scale = starts_of(new), max(lens), int(round(65536 * D ** 0.5))
    q, k, v = gauss(rng, (int(starts[-1]), H, D)), dev(kc), dev(vc)
    args = (dev(q), k, v, dev(table), dev(starts), dev(np.array(lens)), max(new), L, dev(exp_table))
    want = alone(ops, q, k, v, table, starts, lens, exp_table, L, window, sinks, qk_scale=scale)
    got = ops.wit_window_attention(*args, window=window, sinks=sinks, qk_scale=scale)
    assert set(got) == set(want)
    for x in want:
        assert torch.equal(got[x], want[x]), x
    for keep in (("qkv",), ("qkv", "softmax_output"), ("qkv", "qkv_rem", "exp_output", "softmax_lookup_query")):
        some = ops.wit_window_attention(*args, window=window, sinks=sinks, qk_scale=scale, out={x: torch.zeros_like(want[x]) for x in keep})
        assert all(torch.equal(some[x], want[x]) for x in keep), keep
    assert ops.wit_status() == 0


def test_window_attention_of_many_rows_matches_the_oracle(ops, exp_table):
    rng = np.random.default_rng(30)
    table, kc, vc = paged(rng, [600], 16, 1, 2048)
    run_window(ops, gauss(rng, (129, 8, 2048)), kc, vc, table, [0, 129], [600], exp_table, 129, 600, 0, 0, qk_scale=65536 * 45)
    assert ops.wit_status() == 0


@pytest.mark.parametrize("where", ["queries", "keys", "values", "all", "one"])
def test_window_attention_of_many_rows_with_the_largest_values(ops, exp_table, where):
    rng = np.random.default_rng(31)
    H, HK, D, page, new, lens = 8, 1, 700, 16, [300], [640]
    ends = np.array([-(1 << 31), (1 << 31) - 1, TOP, TOP + 1, -TOP - 1, 0x7F7F7F, 0x7F7F80, -0x808080, -0x808081, 0], dtype=np.int64)
    table, kc, vc = paged(rng, lens, page, HK, D)
    q = rng.integers(-3, 4, (300, H, D)).astype(np.int32)
    kc[:] = gauss(rng, kc.shape, 1000.0)
    kc[..., 2] = rng.integers(0, 1 << 19, kc.shape[:3])
    q[..., 0], q[..., 1], q[..., 2] = 1, -1, 1
    if where in ("keys", "all"):
        kc[..., 0] = kc[..., 1] = rng.choice(ends, kc.shape[:3])
    if where in ("queries", "all"):
        q[..., 3] = q[..., 4] = rng.choice(ends, q.shape[:2])
        kc[..., 3] = rng.integers(-100, 100, kc.shape[:3])
        kc[..., 4] = -kc[..., 3]
    if where in ("values", "all"):
        vc[..., ::3] = rng.choice(ends, vc[..., ::3].shape)
    if where == "one":                                  # one element of one row, of the last key and of the first value
        q[299, 7, 699], kc[table[0, 639 // page], 639 % page, 0, 699], vc[table[0, 0], 0, 0, 0] = 1 << 23, 1, -(1 << 31)
    want = alone(ops, q, dev(kc), dev(vc), table, [0, 300], lens, exp_table, 640, 600, 5, qk_scale=2)
    # 2^23 times a key's element of about 1000 is beyond 2^31 after a rescaling by 2, and further from the maximum than the table is long
    status = 3 if where == "one" else 0
    assert ops.wit_status() == status
    got = ops.wit_window_attention(dev(q), dev(kc), dev(vc), dev(table), dev(np.array([0, 300])), dev(np.array(lens)), 300, 640, dev(exp_table), window=600, sinks=5, qk_scale=2)
    assert all(torch.equal(got[x], want[x]) for x in want) and ops.wit_status() == status


def test_window_attention_of_many_rows_reports(ops, exp_table):
    """a page outside the cache counts as zero, a sequence whose numbers do not fit is left out, and neither reaches another one's rows"""
    rng = np.random.default_rng(32)
    new, lens, H, HK, D, page = [300, 260, 280], [800, 700, 280], 16, 2, 128, 16
    table, kc, vc = paged(rng, lens, page, HK, D)
    starts, k, v = starts_of(new), dev(kc), dev(vc)
    q = gauss(rng, (int(starts[-1]), H, D))
    for bad in (-1, kc.shape[0], (1 << 31) - 1, -(1 << 31)):
        t = table.copy()
        t[0, 3], t[1, 40] = bad, bad
        want = alone(ops, q, k, v, t, starts, lens, exp_table, 800, qk_scale=65536 * 11)
        assert ops.wit_status() == 2
        got = ops.wit_window_attention(dev(q), k, v, dev(t), dev(starts), dev(np.array(lens)), 300, 800, dev(exp_table), qk_scale=65536 * 11)
        assert ops.wit_status() == 2 and all(torch.equal(got[x], want[x]) for x in want)
    want = alone(ops, q, k, v, table, starts, lens, exp_table, 800, 500, 3, qk_scale=65536 * 11)
    s = starts.tolist()
    for st, ln in ((s, [800, 801, 280]), (s, [800, -1, 280]), (s, [800, 259, 280]), (s, [800, (1 << 31) - 1, 280])):
        out = {x: filled(*t.shape) for x, t in want.items()}
        ops.wit_window_attention(dev(q), k, v, dev(table), dev(np.array(st)), dev(np.array(ln)), 300, 800, dev(exp_table), window=500, sinks=3, out=out, qk_scale=65536 * 11)
        assert ops.wit_status() == 2
        for x in ("qkv", "qkv_rem", "max", "exp_sum"):
            expected = want[x].clone()
            expected[s[1]:s[2]] = UNTOUCHED
            assert torch.equal(out[x], expected), (ln, x)
        for x in PROOF:
            assert bool((out[x][s[1]:s[2]] == UNTOUCHED).all())
    for st in ([0, -1, 300, 840], [-(1 << 31), 0, 1, 2], [0, 300, (1 << 31) - 1, 840], [840, 560, 300, 0], [0, 0, 0, 9999], [0, 301, 301, 301]):
        out = {x: filled(*t.shape) for x, t in want.items()}
        ops.wit_window_attention(dev(q), k, v, dev(table), dev(np.array(st)), dev(np.array(lens)), 300, 800, dev(exp_table), window=500, sinks=3, out=out, qk_scale=65536 * 11)
        assert ops.wit_status() & 2, st


@pytest.mark.parametrize("n,H,D", [(70, 2, 64), (720, 16, 128)])
def test_window_attention_of_wide_sums(ops, exp_table, n, H, D):
    """a table of large entries that is no exponential: sums beyond 2^28, probabilities of three digits"""
    rng = np.random.default_rng(33)
    table, kc, vc = paged(rng, [n], 16, 2, D)
    q = gauss(rng, (n, H, D))
    flat = np.full(1 << 20, 3 << 20, dtype=np.int32)
    flat[::7] = 1 << 16
    k, v = dev(kc), dev(vc)
    for prob_scale in (1 << 16, 1 << 22, 1 << 24):
        want = alone(ops, q, k, v, table, [0, n], [n], flat, n, qk_scale=65536 * 11, prob_scale=prob_scale, out_scale=prob_scale)
        got = ops.wit_window_attention(dev(q), k, v, dev(table), dev(np.array([0, n])), dev(np.array([n])), n, n, dev(flat), qk_scale=65536 * 11, prob_scale=prob_scale, out_scale=prob_scale)
        assert all(torch.equal(got[x], want[x]) for x in want)
        ops.wit_status()                                # queries beyond 32 bits where the probabilities are many
    run_window(ops, q[:40, :4], kc[:, :, :1], vc[:, :, :1], table, [0, 40], [n], flat, 40, n, 20, 2, qk_scale=65536 * 11)
    assert ops.wit_status() == 0


@pytest.mark.parametrize("prob_scale", [1 << 16, 1 << 22, 1 << 24])
def test_window_attention_of_rows_that_go_different_ways(ops, exp_table, prob_scale):
    """rows of one tile whose sums are below and above 2^28, and pages outside the cache that turn up between tiles that all rows see"""
    rng = np.random.default_rng(38)
    for new, n, H, HK, D in ((40, 2600, 4, 4, 64), (33, 2600, 2, 2, 33), (260, 2600, 16, 2, 128)):
        table, kc, vc = paged(rng, [n], 16, HK, D)
        q, k, v = gauss(rng, (new, H, D)), dev(kc), dev(vc)
        # all entries the same, so that a row's sum says how many positions it sees: 2^28 in the middle of the new tokens
        flat = np.full(1 << 20, (1 << 28) // (n - new // 2), dtype=np.int32)
        for bad in ([], [120], [64, 70, 128, 161], [1, 162]):
            t = table.copy()
            t[0, bad] = -1
            want = alone(ops, q, k, v, t, [0, new], [n], flat, n, qk_scale=65536 * 11, prob_scale=prob_scale, out_scale=prob_scale)
            status = ops.wit_status()
            assert (status & 2 != 0) == bool(bad) and int(want["exp_sum"].min()) < 1 << 28 <= int(want["exp_sum"].max())
            got = ops.wit_window_attention(dev(q), k, v, dev(t), dev(np.array([0, new])), dev(np.array([n])), new, n, dev(flat), qk_scale=65536 * 11, prob_scale=prob_scale, out_scale=prob_scale)
            assert ops.wit_status() == status
            for x in want:
                assert torch.equal(got[x], want[x]), (new, bad, x)


def test_window_attention_of_a_long_cache(ops):
    """131072 positions of the same score and value, whose digits' products would leave 32 bits if all were added up there"""
    n, new, H, D = 131072, 128, 16, 1024
    prob_scale, out_scale, e, x = 8064 * n, 1 << 31, 1000, -128 * 65536 + 127 * 256 - 128
    k = torch.zeros((n // 1024, 1024, 1, D), dtype=torch.int32, device="cuda")
    v = torch.full_like(k, x)
    table = torch.full((1 << 10,), e, dtype=torch.int32, device="cuda")
    got = ops.wit_window_attention(dev(np.ones((new, H, D), dtype=np.int32)), k, v, dev(np.arange(n // 1024)[None]), dev(np.array([0, new])), dev(np.array([n])), new, n, table,
                                   bit_shift=10, index_bits=10, prob_scale=prob_scale, out_scale=out_scale, proof=False)
    for j in range(new):
        seen = n - new + j + 1
        y = seen * ((e * prob_scale + seen * e // 2) // (seen * e)) * x
        want = (y + out_scale // 2) // out_scale
        assert bool((got["qkv"][j] == want).all()) and bool((got["qkv_rem"][j] == y - want * out_scale).all()), j
    assert ops.wit_status() == 0


def test_window_attention_looks_a_table_up_that_is_off_by_one(ops, exp_table):
    """wherever the entry stands that is not the exponential's"""
    rng = np.random.default_rng(34)
    n, H, D = 520, 16, 128
    table, kc, vc = paged(rng, [n], 16, 2, D)
    q, k, v = gauss(rng, (n, H, D)), dev(kc), dev(vc)
    for at in (-1, -2, -3, -1025, -40000, -200000, -(1 << 19)):
        other = exp_table.copy()
        other[at] += 1
        want = alone(ops, q, k, v, table, [0, n], [n], other, n, qk_scale=65536 * 11)
        got = ops.wit_window_attention(dev(q), k, v, dev(table), dev(np.array([0, n])), dev(np.array([n])), n, n, dev(other), qk_scale=65536 * 11)
        assert all(torch.equal(got[x], want[x]) for x in want), at
    assert ops.wit_status() == 0


def test_window_attention_of_many_sequences_with_long_heads(ops, exp_table):
    """the largest workgroups of the scores: eight steps of the queries' digits and offsets of 32 tiles; pages that sequences share"""
    rng = np.random.default_rng(35)
    for seqs, H, D, window in ((100, 8, 512, 0), (100, 8, 450, 1900), (40, 16, 130, 0)):
        kc, vc = gauss(rng, (130, 16, H, D)), gauss(rng, (130, 16, H, D))
        table = rng.integers(0, 130, (seqs, 129)).astype(np.int32)
        lens, starts = rng.integers(1900, 2060, seqs), np.arange(seqs + 1) * 2
        q, k, v = gauss(rng, (2 * seqs, H, D)), dev(kc), dev(vc)
        want = alone(ops, q, k, v, table, starts, lens, exp_table, 2060, window, 0, qk_scale=65536 * 22)
        got = ops.wit_window_attention(dev(q), k, v, dev(table), dev(starts), dev(lens), 2, 2060, dev(exp_table), window=window, qk_scale=65536 * 22)
        assert all(torch.equal(got[x], want[x]) for x in want) and ops.wit_status() == 0


def test_window_attention_of_offsets_beyond_32_bits(ops, exp_table):
    """pages 2^27 elements apart, and rows of a proof of more than 2^32 elements"""
    rng = np.random.default_rng(36)
    D, n = 512, 17 * 16
    far = torch.empty((16 << 27) + 16 * D, dtype=torch.int32, device="cuda").as_strided((17, 16, 1, D), (1 << 27, D, D, 1))
    near = dev(gauss(rng, (17, 16, 1, D)))
    far.copy_(near)
    table = rng.permutation(17)[None].astype(np.int32)
    for new, H in ((1, 4), (9, 4), (272, 32)):
        q = dev(gauss(rng, (new, H, D)))
        args = (dev(table), dev(np.array([0, new])), dev(np.array([n])), new, n, dev(exp_table))
        want, got = (ops.wit_window_attention(q, x, x, *args, qk_scale=65536 * 22) for x in (near, far))
        assert all(torch.equal(got[x], want[x]) for x in want)
    del far, want, got
    new, L, H, HK, D = 2048, 70000, 32, 8, 64
    kc, vc = gauss(rng, (9, 1000, HK, D)), gauss(rng, (9, 1000, HK, D))
    table = rng.integers(0, 9, (1, 70)).astype(np.int32)
    q, k, v = gauss(rng, (new, H, D)), dev(kc), dev(vc)
    got = {"qkv": filled(new, H, D), "softmax_output": torch.zeros((new, H, L), dtype=torch.int32, device="cuda")}
    ops.wit_window_attention(dev(q), k, v, dev(table), dev(np.array([0, new])), dev(np.array([L])), new, L, dev(exp_table), window=256, sinks=4, out=got, qk_scale=65536 * 8)
    want = alone(ops, q[-40:], k, v, table, [0, 40], [L], exp_table, L, 256, 4, qk_scale=65536 * 8, out={x: torch.zeros_like(t[-40:]) for x, t in got.items()})
    assert all(torch.equal(got[x][-40:], want[x]) for x in want) and ops.wit_status() == 0


def test_calls_with_many_rows_on_two_streams_and_replayed(ops, exp_table):
    rng = np.random.default_rng(37)
    cases = []
    for n, H, HK, D in ((520, 16, 2, 128), (300, 8, 1, 1024), (40, 4, 2, 64)):
        table, kc, vc = paged(rng, [n + 160], 16, HK, D)
        q = [dev(gauss(rng, (n, H, D))) for _ in range(3)]
        rest = (dev(kc), dev(vc), dev(table), dev(np.array([0, n])), dev(np.array([n + 160])), n, n + 160, dev(exp_table))
        cases.append((q, rest, [ops.wit_window_attention(x, *rest, qk_scale=65536 * 11) for x in q]))
    # the scores of 1024 products over 11 have a deviation of 2.9, and the table's 2^20 entries end 16 below the maximum: some are looked for outside
    status = ops.wit_status()
    assert status == 2
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    results = []
    for i in range(3):
        for (q, rest, _), s in zip(cases, streams):
            with torch.cuda.stream(s):
                results.append(ops.wit_window_attention(q[i], *rest, qk_scale=65536 * 11))
    torch.cuda.synchronize()
    for j, got in enumerate(results):
        want = cases[j % 3][2][j // 3]
        assert all(torch.equal(got[x], want[x]) for x in want)
    for q, rest, want in cases:
        x = q[0].clone()
        out = {name: torch.zeros_like(t) for name, t in want[0].items()}
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.wit_window_attention(x, *rest, qk_scale=65536 * 11, out=out)
        for i in (1, 0, 2, 1):
            x.copy_(q[i])
            graph.replay()
            again = ops.wit_window_attention(q[i], *rest, qk_scale=65536 * 11)
            torch.cuda.synchronize()
            assert all(torch.equal(out[name], want[i][name]) and torch.equal(again[name], want[i][name]) for name in want[i])
    assert ops.wit_status() == status


# ------------------------------------------------------------------ the next token
def next_case(rng, n, vocab, longest):
    logits = gauss(rng, (n, vocab), 200000.0)
    history = rng.integers(0, vocab, (n, longest)).astype(np.int32)
    history[:, ::3] = rng.integers(0, min(vocab, 5), history[:, ::3].shape)
    history[rng.random(history.shape) < 0.1] = -1
    lens = rng.integers(0, longest + 1, n)
    return {"logits": logits, "history": history, "history_lens": lens, "repetition": rng.integers(1, 200000, n), "presence": rng.integers(-50000, 50000, n),
            "frequency": rng.integers(-30000, 30000, n), "bias": gauss(rng, (n, vocab)), "mask": rng.integers(LOWEST, 1 << 31, (n, -(-vocab // 32))).astype(np.int32)}


def run_next(ops, c, status=0, scale=1 << 16, **kw):
    want, left = wo.next_token(**c, scale=scale)
    d = {x: None if t is None else dev(np.asarray(t)) for x, t in c.items()}
    got = ops.wit_next_token(**d, scale=scale, **kw)
    wide = bool((want["gap"] >= 1 << 31).any()) and "gap" in got
    for x, t in got.items():
        assert np.array_equal(host(t), want[x].astype(np.int32)), (x, np.argwhere(host(t) != want[x].astype(np.int32))[:4].tolist())
    assert ops.wit_status() == (1 if left else 0) | (16 if wide else 0) | status
    return got


@pytest.mark.parametrize("n,vocab,longest", [(1, 1, 1), (2, 3, 9), (1, 32, 5), (3, 31, 40), (2, 33, 0), (5, 1000, 100), (2, 1025, 300), (1, 8193, 70), (3, 4096, 1000), (260, 40, 6)])
def test_next_token(ops, n, vocab, longest):
    rng = np.random.default_rng(n + vocab)
    c = next_case(rng, n, vocab, longest)
    run_next(ops, c)
    run_next(ops, c, proof=False)
    run_next(ops, {**c, "bias": c["bias"][0], "mask": c["mask"][0]})
    run_next(ops, {**c, "mask": None, "bias": None}, scale=1000)
    run_next(ops, {**c, "history": None, "history_lens": None})
    for x in ("repetition", "presence", "frequency"):
        run_next(ops, {**c, x: None})
    run_next(ops, {"logits": c["logits"]})


def test_next_token_of_the_lowest_and_the_same(ops):
    rng = np.random.default_rng(1)
    c = next_case(rng, 6, 777, 50)
    c["logits"][0], c["logits"][1, ::2] = LOWEST, LOWEST
    c["mask"][2] = 0                                       # nothing left
    c["bias"][3] = LOWEST
    c["logits"][4], c["bias"][4], c["history_lens"][4] = 7, 0, 0          # the first of equal ones that the mask leaves
    got = run_next(ops, c)
    assert host(got["token"])[[0, 2, 3]].tolist() == [-1] * 3 and host(got["max"])[0] == LOWEST
    run_next(ops, {**c, "mask": None})
    # one token is left, at every place of a word and of the row's end
    for v in (0, 1, 31, 32, 63, 775, 776):
        m = np.zeros((6, 25), dtype=np.uint32)
        m[:, v // 32] = 1 << (v % 32)
        d = {**c, "mask": m.view(np.int32), "logits": gauss(rng, (6, 777)), "bias": None}
        assert host(run_next(ops, d)["token"]).tolist() == [v] * 6
    # bits behind the vocabulary's end choose nothing
    m = np.zeros((6, 25), dtype=np.uint32)
    m[:, 24] = 0xFFFFFFFF << (777 % 32) & 0xFFFFFFFF
    assert host(run_next(ops, {**c, "mask": m.view(np.int32)})["token"]).tolist() == [-1] * 6


def test_next_token_of_the_largest_numbers(ops):
    """quotients and logits that leave 32 bits, remainders by the largest divisors"""
    rng = np.random.default_rng(2)
    ends = np.array([LOWEST + 1, (1 << 31) - 1, 0, 1, -1, LOWEST])
    for scale in (1, 3, 1 << 16, 1 << 31):
        for rep in (1, 2, 65535, (1 << 31) - 1):
            c = next_case(rng, 3, 200, 400)
            c["logits"] = rng.choice(ends, (3, 200))
            c["repetition"][:] = rep
            c["presence"], c["frequency"] = rng.choice(ends, 3), rng.choice(ends, 3)
            c["bias"] = rng.choice(ends, (3, 200))
            run_next(ops, c, scale=scale)
            run_next(ops, {**c, "presence": None, "frequency": None, "bias": None}, scale=scale)


@pytest.mark.parametrize("x", [(1 << 31) - 1, -(1 << 31) + 1])
def test_next_token_of_penalties_that_cancel(ops, x):
    """a quotient beyond 2^53 that the penalty for 2^23 occurrences brings back into 32 bits: every bit of both counts"""
    n = (1 << 23) + 1
    for rep in (259, 275) if x > 0 else ((1 << 31) - 40, (1 << 31) - 33):
        scale = 1 << 31 if x > 0 else 300
        y, by = (x * scale, rep) if x > 0 else (x * rep, scale)
        y, rem = (y + by // 2) // by, y - (y + by // 2) // by * by
        assert abs(y) > 1 << 53 and y % 2
        frequency = y // n
        assert abs(frequency) < 1 << 31
        got = ops.wit_next_token(dev(np.array([[x, -5, 3]])), torch.zeros((1, n), dtype=torch.int32, device="cuda"), dev(np.array([n])), repetition=dev(np.array([rep])),
                                 presence=dev(np.array([77])), frequency=dev(np.array([frequency])), scale=scale)
        assert host(got["logits"])[0].tolist() == [y - frequency * n - 77, -5, 3] and host(got["rem"])[0].tolist() == [rem, 0, 0] and host(got["count"])[0].tolist() == [n, 0, 0]
    assert ops.wit_status() == 0


def test_next_token_reports_what_is_out_of_range(ops):
    rng = np.random.default_rng(3)
    c = next_case(rng, 4, 100, 30)
    c["history_lens"][:] = 30
    bad = {**c, "history": c["history"].copy()}
    bad["history"][1, 3] = 100
    run_next(ops, bad, status=2)
    bad["history"][1, 3] = (1 << 31) - 1
    run_next(ops, bad, status=2)
    d = {x: dev(np.asarray(t)) for x, t in c.items()}
    for lens, as_if in (([30, 31, 30, 30], [30] * 4), ([30, -1, 30, 30], [30, 0, 30, 30]), ([1 << 30, 30, 30, LOWEST], [30, 30, 30, 0])):
        got = ops.wit_next_token(**{**d, "history_lens": dev(np.array(lens))})
        assert ops.wit_status() == 2
        want = ops.wit_next_token(**{**d, "history_lens": dev(np.array(as_if))})
        assert ops.wit_status() == 0 and all(torch.equal(got[x], want[x]) for x in got)
    for rep in (0, -5, LOWEST):
        got = ops.wit_next_token(**{**d, "repetition": dev(np.array([rep] * 4))})
        assert ops.wit_status() == 2
        want = ops.wit_next_token(**{**d, "repetition": None})
        assert all(torch.equal(got[x], want[x]) for x in got)


def test_next_token_of_strided_rows_in_place_and_with_some_outputs(ops):
    rng = np.random.default_rng(4)
    for vocab in (1000, 1001):
        c = next_case(rng, 5, vocab, 60)
        good = run_next(ops, c)
        d = {x: dev(np.asarray(t)) for x, t in c.items()}
        for pad in (4, 3):
            wide = {x: torch.full((5, d[x].shape[1] + 2 * pad), UNTOUCHED, dtype=torch.int32, device="cuda") for x in ("logits", "history", "bias", "mask")}
            views = {x: t[:, pad:pad + d[x].shape[1]] for x, t in wide.items()}
            for x in views:
                views[x].copy_(d[x])
            got = ops.wit_next_token(**{**d, **views})
            assert all(torch.equal(got[x], good[x]) for x in good)
            assert all(bool((t[:, :pad] == UNTOUCHED).all()) and bool((t[:, -pad:] == UNTOUCHED).all()) for t in wide.values())
        # one row of biases and masks for all
        one = ops.wit_next_token(**{**d, "bias": d["bias"][:1].expand(5, vocab), "mask": d["mask"][:1].expand(5, -1)})
        want = ops.wit_next_token(**{**d, "bias": d["bias"][0].contiguous(), "mask": d["mask"][0].contiguous()})
        assert all(torch.equal(one[x], want[x]) for x in want)
        for keep in (("token",), ("token", "gap"), ("token", "max", "count"), ("token", "logits", "rem")):
            out = {x: filled(*good[x].shape) for x in keep}
            assert ops.wit_next_token(**d, out=out) is out and all(torch.equal(out[x], good[x]) for x in keep)
        place = d["logits"].clone()
        got = ops.wit_next_token(**{**d, "logits": place}, out={"token": filled(5), "logits": place, "gap": filled(5, vocab)})
        assert torch.equal(place, good["logits"]) and torch.equal(got["gap"], good["gap"])
    assert ops.wit_status() == 0


def test_next_token_appends_to_its_history(ops):
    """the token goes behind those it was chosen by, its logit where a penalty stood: both are written when all has been read"""
    rng = np.random.default_rng(5)
    for vocab in (50, 40000):
        c = next_case(rng, 1, vocab, 3000)
        history = dev(np.concatenate((c["history"], np.full((1, 50), -9, dtype=np.int32)), 1))
        for n in range(2990, 3010):
            d = {x: dev(np.asarray(t)) for x, t in c.items()} | {"history": history, "history_lens": dev(np.array([n]))}
            want = ops.wit_next_token(**{**d, "history": history.clone()})
            got = ops.wit_next_token(**d, out={"token": history[0, n:n + 1], "max": d["presence"]})
            assert torch.equal(history[0, n:n + 1], want["token"]) and torch.equal(got["max"], want["max"])
            c["logits"] = gauss(rng, (1, vocab), 200000.0)
    assert ops.wit_status() == 0


# ------------------------------------------------------------------ together
def test_a_step_after_the_other(ops, exp_table):
    """requests with prompts, then their answers token by token: pages, rotation and append, attention, a projection as the head, the next token -
    against the same with every sequence's keys and values in one piece"""
    rng = np.random.default_rng(30)
    seqs, H, HK, D, page, window, sinks, vocab, pages = 4, 4, 2, 32, 8, 24, 3, 500, 40
    width, scale = H * D, 1 << 16
    cos, sin = (np.rint(f(np.arange(200)[:, None] * 100.0 ** (-np.arange(D // 2) / 16)) * scale).astype(np.int32) for f in (np.cos, np.sin))
    emb = gauss(rng, (vocab, width))
    wq, wk, wv = (gauss(rng, (n, width), 5000.0) for n in (H * D, HK * D, HK * D))
    head_w, head_s = rng.integers(0, 256, (vocab, width // 2)).astype(np.uint8), rng.integers(200, 400, (vocab, width // 32)).astype(np.int32)
    ring = np.full(2 * pages, -1, dtype=np.int32)
    ring[:pages] = rng.permutation(pages)
    kc, vc, table = filled(pages, page, HK, D), filled(pages, page, HK, D), filled(seqs, 12)
    lens, span, ring = dev(np.zeros(seqs, dtype=np.int64)), dev(np.array([0, pages])), dev(ring)
    texts = [rng.integers(0, vocab, n).tolist() for n in (17, 1, 40, 9)]
    keys, values = [np.zeros((0, HK, D), dtype=np.int32)] * seqs, [np.zeros((0, HK, D), dtype=np.int32)] * seqs
    fresh = [list(t) for t in texts]
    for step in range(6):
        new, R = [len(t) for t in fresh], 70
        out = ops.wit_page_step(lens, dev(np.array(new)), table, ring, span, page, R, window=window, sinks=sinks)
        tokens = sum(fresh, [])
        x = np.zeros((R, width), dtype=np.int32)
        x[:len(tokens)] = emb[tokens]
        q, k, v = (ops.wit_matmul_rescale(dev(x), dev(w), scale)[0] for w in (wq, wk, wv))
        q = ops.wit_rope_append(q.view(R, H, D), k.view(R, HK, D), v.view(R, HK, D), out["positions"], out["slots"], dev(cos), dev(sin), kc, vc)
        got = ops.wit_window_attention(q, kc, vc, table, out["starts"], out["lens"], max(new), 96, dev(exp_table), window=window, sinks=sinks, qk_scale=370728)
        last = (out["starts"][1:] - 1).long()
        logits = ops.wit_matvec_q4(got["qkv"].view(R, width)[last], dev(head_w), dev(head_s), 32)[0]
        history = np.full((seqs, 60), -1, dtype=np.int32)
        for b, t in enumerate(texts):
            history[b, :len(t)] = t
        hl = np.array([len(t) for t in texts])
        pen = {"repetition": np.full(seqs, 90000), "presence": np.full(seqs, 1000), "frequency": np.full(seqs, 77)}
        chosen = ops.wit_next_token(logits, dev(history), dev(hl), **{n: dev(t) for n, t in pen.items()})
        # the same in one piece
        start, want_logits = host(out["starts"]), []
        for b in range(seqs):
            rows, at = slice(start[b], start[b + 1]), np.arange(len(keys[b]), len(keys[b]) + new[b])
            hq, hk, hv = (wo.rescale(wo.matmul_t(x[rows], w), scale)[0].reshape(new[b], -1, D) for w in (wq, wk, wv))
            hq, hk = (wo.rotate(t, at, cos, sin, False)[0] for t in (hq, hk))
            keys[b], values[b] = np.concatenate((keys[b], hk)), np.concatenate((values[b], hv))
            o = {"qkv": np.zeros((new[b], H, D), dtype=np.int32), "softmax_lookup_query": np.zeros((new[b], H, 96), dtype=np.int32)}
            wo.window_attention(hq, keys[b][:, None], values[b][:, None], np.arange(len(keys[b]))[None], [0, new[b]], [len(keys[b])], window, sinks, exp_table, o, qk_scale=370728)
            for name, t in o.items():
                assert np.array_equal(host(got[name])[rows], t), (step, b, name)
            want_logits.append(wo.matvec_q4(o["qkv"][-1].reshape(1, width), head_w, head_s, 32, None)[0][0])
        want, _ = wo.next_token(np.array(want_logits), history, hl, **pen)
        for name in chosen:
            assert np.array_equal(host(chosen[name]), want[name].astype(np.int32)), (step, name)
        fresh = [[int(t)] for t in host(chosen["token"])]
        texts = [t + f for t, f in zip(texts, fresh)]
        lens, span = out["lens"], out["free_span"]
    assert ops.wit_status() == 0


@pytest.mark.parametrize("new", [1, 5])
def test_captured_steps_are_replayed(ops, exp_table, new):
    """a step in a graph, replayed with other inputs, with eager calls between the replays; two streams at once"""
    rng = np.random.default_rng(40)
    seqs, H, HK, D, page, vocab = 3, 4, 2, 64, 16, 600
    rows, longest = seqs * new, 400
    cases = []
    for i in range(3):
        lens = [int(n) for n in rng.integers(new, longest - new, seqs)]
        table, kc, vc = paged(rng, [longest] * seqs, page, HK, D)
        cases.append({"lens": np.array(lens), "table": table, "k": kc, "v": vc, "q": gauss(rng, (rows, H, D)), **next_case(rng, seqs, vocab, 50)})
    names = ("lens", "table", "k", "v", "q", "logits", "history", "history_lens")
    fixed = {x: dev(cases[0][x]) for x in names}
    free, span, more, et = dev(np.arange(100)), dev(np.array([0, 50])), dev(np.full(seqs, new)), dev(exp_table)
    ws = torch.empty(ops.wit_window_attention_workspace(rows, seqs, H, HK, D, new, longest, 100, 4), dtype=torch.uint8, device="cuda")
    ns = torch.empty(ops.wit_next_token_workspace(seqs, vocab), dtype=torch.uint8, device="cuda")

    def step(t, out=None, workspace=None, next_space=None):
        p = ops.wit_page_step(t["lens"], more, t["table"], free.clone(), span, page, rows, out=None if out is None else out[0])
        a = ops.wit_window_attention(t["q"], t["k"], t["v"], t["table"], p["starts"], p["lens"], new, longest, et, window=100, sinks=4, qk_scale=1 << 19,
                                     out=None if out is None else out[1], workspace=workspace)
        return p, a, ops.wit_next_token(t["logits"], t["history"], t["history_lens"], out=None if out is None else out[2], workspace=next_space)

    want = [step({x: dev(c[x]) for x in names}) for c in cases]
    out = [{x: torch.zeros_like(t) for x, t in one.items()} for one in want[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(fixed, out, ws, ns)
    for i in (0, 1, 2, 1, 0):
        for x in names:
            fixed[x].copy_(dev(cases[i][x]))
        for x in out[1]:
            out[1][x].zero_()
        graph.replay()
        other = step({x: dev(cases[2 - i][x]) for x in names})
        torch.cuda.synchronize()
        for a, b in ((out, want[i]), (other, want[2 - i])):
            assert all(torch.equal(x[n], y[n]) for x, y in zip(a, b) for n in y), i
    with torch.cuda.stream(side):
        other = step({x: dev(cases[1][x]) for x in names})
    here = step({x: dev(cases[2][x]) for x in names})
    torch.cuda.synchronize()
    for a, b in ((other, want[1]), (here, want[2])):
        assert all(torch.equal(x[n], y[n]) for x, y in zip(a, b) for n in y)
    assert ops.wit_status() == 0
