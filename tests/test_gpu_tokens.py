"""GPU parity tests of the new tokens' kernels (rotation and append to a paged cache, attention of one token a sequence over
it, products with 4-bit weights) against the numpy oracle.  Every result is a whole number and is compared exactly."""
import numpy as np
import pytest
import torch
from oracle import witness_oracle as wo

pytestmark = pytest.mark.gpu

PROOF = ("scores", "scores_rem", "exp_input", "exp_output", "softmax_output", "softmax_lookup_query")
UNTOUCHED = -77
TOP = 0x7F7F7F7F          # the largest value that four signed bytes hold as balanced digits


@pytest.fixture(scope="module")
def ops():
    from grape_amd import ops as o
    o.init(0)
    o.wit_status()                          # start from a clean status word
    return o


@pytest.fixture(scope="module")
def exp_table():
    return wo.exp_table()


def dev(a):
    a = np.ascontiguousarray(a)
    return torch.from_numpy(a.astype(np.int32) if a.dtype == np.int64 else a).cuda()


def host(t):
    return t.cpu().numpy()


def gauss(rng, shape, sigma=65536.0):
    return np.rint(rng.normal(0.0, sigma, shape)).astype(np.int32)


def filled(*shape):
    return torch.full(shape, UNTOUCHED, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ rotation and append
def tables(rows, rot, scale):
    angle = np.arange(rows)[:, None] * 10000.0 ** (-2.0 * np.arange(rot // 2) / max(rot, 1))
    return (np.rint(f(angle) * scale).astype(np.int64).clip(-(1 << 31), (1 << 31) - 1).astype(np.int32) for f in (np.cos, np.sin))


def append_case(rng, T, H, HK, D, rot, page, scale=1 << 16, rows=300, pages=None, sigma=65536.0):
    cos, sin = tables(rows, rot, scale)
    pages = pages or T // page + 3
    return {"q": gauss(rng, (T, H, D), sigma), "k": gauss(rng, (T, HK, D), sigma), "v": gauss(rng, (T, HK, D), sigma),
            "positions": rng.integers(0, rows, T).astype(np.int32), "slots": rng.permutation(pages * page)[:T].astype(np.int64),
            "cos": cos, "sin": sin, "caches": (pages, page, HK, D)}


def run_append(ops, c, scale, interleaved, caches=None):
    """outputs of the kernel and of the oracle"""
    T, H, D = c["q"].shape
    HK = c["k"].shape[1]
    want = [np.full(s, UNTOUCHED, dtype=np.int32) for s in (c["caches"], c["caches"], (T, H, D), (T, H, D), (T, HK, D))]
    wo.rope_append(c["q"], c["k"], c["v"], c["positions"], c["slots"], c["cos"], c["sin"], want[0], want[1], want[2], want[3], want[4], interleaved, scale)
    kc, vc = caches or (filled(*c["caches"]), filled(*c["caches"]))
    got = [kc, vc, filled(T, H, D), filled(T, H, D), filled(T, HK, D)]
    ops.wit_rope_append(dev(c["q"]), dev(c["k"]), dev(c["v"]), dev(c["positions"]), torch.from_numpy(c["slots"]).cuda(), dev(c["cos"]),
                        dev(c["sin"]), got[0], got[1], got[2], got[3], got[4], scale=scale, interleaved=interleaved)
    return got, want


def same(got, want):
    for g, w in zip(got, want):
        assert np.array_equal(host(g), w)


APPENDS = [
    # tokens, heads, cache heads, dim, rot, page, scale
    (1, 32, 8, 128, 128, 16, 1 << 16), (1, 1, 1, 2, 2, 1, 1 << 16), (7, 3, 1, 5, 4, 3, 1000), (64, 4, 2, 80, 32, 17, 1 << 16),
    (33, 2, 2, 64, 0, 16, 1 << 16), (5, 1, 1, 4096, 4096, 64, 1 << 16), (19, 6, 3, 50, 50, 10, 1 << 14), (300, 2, 1, 16, 8, 16, 1 << 31),
    (257, 1, 1, 1, 0, 4, 1), (40, 5, 5, 100, 50, 8, 1 << 16), (1500, 8, 2, 32, 32, 32, 12345), (23, 2, 1, 12, 8, 5, 1 << 16)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,HK,D,rot,page,scale", APPENDS)
def test_append_matches_the_oracle(ops, T, H, HK, D, rot, page, scale, interleaved):
    rng = np.random.default_rng(T * 7 + D + rot)
    c = append_case(rng, T, H, HK, D, rot, page, scale)
    if T > 4:
        c["slots"][rng.permutation(T)[: T // 4]] = -1 - rng.integers(0, 5)         # padding anywhere
    same(*run_append(ops, c, scale, interleaved))
    assert ops.wit_status() == 0


def test_append_keeps_the_last_of_several_tokens_in_one_slot(ops):
    rng = np.random.default_rng(5)
    for T, page in ((9, 4), (700, 16)):
        c = append_case(rng, T, 2, 2, 64, 64, page)
        c["slots"][:] = rng.integers(0, 5, T)                   # the oracle writes token after token
        c["slots"][T // 2] = -1
        same(*run_append(ops, c, 1 << 16, False))
    # a later token that is out of range takes nothing away
    c = append_case(rng, 3, 1, 1, 64, 64, 4)
    c["slots"][:] = 2
    c["positions"][2] = 300
    got, _ = run_append(ops, {**c, "q": c["q"][:2], "k": c["k"][:2], "v": c["v"][:2], "positions": c["positions"][:2], "slots": c["slots"][:2]}, 1 << 16, False)
    all_three = [filled(*c["caches"]), filled(*c["caches"]), filled(3, 1, 64)]
    ops.wit_rope_append(dev(c["q"]), dev(c["k"]), dev(c["v"]), dev(c["positions"]), torch.from_numpy(c["slots"]).cuda(), dev(c["cos"]),
                        dev(c["sin"]), all_three[0], all_three[1], all_three[2])
    assert torch.equal(all_three[0], got[0]) and torch.equal(all_three[1], got[1]) and bool((all_three[2][2] == UNTOUCHED).all())
    assert ops.wit_status() == 2


def test_append_reports_and_skips_what_is_out_of_range(ops):
    rng = np.random.default_rng(6)
    for pos, slot in ((-1, 3), (300, 3), (5, 40), (5, 1 << 40)):
        c = append_case(rng, 6, 2, 1, 16, 16, 8, pages=5)
        c["positions"][4], c["slots"][4] = pos, slot
        ok = {**c, "slots": np.where(np.arange(6) == 4, -1, c["slots"]), "positions": np.where(np.arange(6) == 4, 0, c["positions"]).astype(np.int32)}
        _, want = run_append(ops, ok, 1 << 16, False)
        assert ops.wit_status() == 0
        got = [filled(*c["caches"]), filled(*c["caches"]), filled(6, 2, 16), filled(6, 2, 16), filled(6, 1, 16)]
        ops.wit_rope_append(dev(c["q"]), dev(c["k"]), dev(c["v"]), dev(c["positions"]), torch.from_numpy(c["slots"]).cuda(), dev(c["cos"]),
                            dev(c["sin"]), *got)
        same(got, want)
        assert ops.wit_status() == 2


def test_append_of_the_largest_values(ops):
    """quotients that leave 32 bits are reported; those at their ends are exact"""
    lo, hi = -(1 << 31), (1 << 31) - 1
    x = np.array([[[lo, hi, hi, lo]]], dtype=np.int64).astype(np.int32)
    cos, sin = np.full((1, 2), 1 << 16, dtype=np.int32), np.zeros((1, 2), dtype=np.int32)
    for inter in (False, True):
        kc, vc = filled(1, 2, 1, 4), filled(1, 2, 1, 4)
        out = ops.wit_rope_append(dev(x), dev(x), dev(x), dev(np.zeros(1, np.int32)), torch.zeros(1, dtype=torch.int64, device="cuda"), dev(cos), dev(sin),
                                  kc, vc, interleaved=inter)
        assert np.array_equal(host(out), x) and np.array_equal(host(kc)[0, 0], x[0]) and np.array_equal(host(vc)[0, 0], x[0])
        assert ops.wit_status() == 0
        ops.wit_rope_append(dev(x), dev(x), dev(x), dev(np.zeros(1, np.int32)), torch.zeros(1, dtype=torch.int64, device="cuda"), dev(cos + 5), dev(sin),
                            kc, vc, interleaved=inter)
        assert ops.wit_status() == 1


@pytest.mark.parametrize("D,rot", [(64, 64), (30, 20)])
def test_append_of_strided_tokens_in_place_and_without_queries(ops, D, rot):
    rng = np.random.default_rng(D)
    T, H, HK, page = 37, 4, 2, 16
    c = append_case(rng, T, H, HK, D, rot, page)
    base, want = run_append(ops, c, 1 << 16, False)
    # one fused projection's output, with some columns more
    fused = torch.zeros((T, (H + 2 * HK) * D + 4), dtype=torch.int32, device="cuda")
    q, k, v = (fused[:, a * D:b * D].view(T, -1, D) for a, b in ((0, H), (H, H + HK), (H + HK, H + 2 * HK)))
    q.copy_(dev(c["q"])), k.copy_(dev(c["k"])), v.copy_(dev(c["v"]))
    rest = (dev(c["positions"]), torch.from_numpy(c["slots"]).cuda(), dev(c["cos"]), dev(c["sin"]))
    got = [filled(*c["caches"]), filled(*c["caches"]), filled(T, H, D), filled(T, H, D), filled(T, HK, D)]
    ops.wit_rope_append(q, k, v, *rest, *got)
    same(got, want)
    # in place
    qq = dev(c["q"])
    assert ops.wit_rope_append(qq, k, v, *rest, got[0], got[1], q_out=qq) is qq
    assert np.array_equal(host(qq), want[2])
    # keys and values only, and no remainders
    got = [filled(*c["caches"]), filled(*c["caches"])]
    assert ops.wit_rope_append(None, k, v, *rest, *got) is None
    same(got, want[:2])
    # a cache whose heads stand before its pages, one with gaps, and one whose start is not 16-byte aligned
    pages = c["caches"][0]
    for make in (lambda: filled(HK, pages, page, D).permute(1, 2, 0, 3), lambda: filled(pages, page, HK, D + 3)[..., :D],
                 lambda: filled(pages, HK, page, D).permute(0, 2, 1, 3), lambda: filled(pages * page * HK * D + 1)[1:].view(pages, page, HK, D)):
        got = [make(), make()]
        ops.wit_rope_append(q, k, v, *rest, *got)
        same(got, want[:2])
    assert ops.wit_status() == 0


# ------------------------------------------------------------------ attention
def paged(rng, lens, page, HK, D, sigma=65536.0, spare=2):
    used = [-(-n // page) for n in lens]
    pages = sum(used) + spare
    order = rng.permutation(pages)
    table = np.full((len(lens), max(max(used), 1)), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    return table, gauss(rng, (pages, page, HK, D), sigma), gauss(rng, (pages, page, HK, D), sigma)


def run_attention(ops, q, kc, vc, table, lens, first, exp, max_len, proof=True, **kw):
    n, H, D = q.shape
    shapes = {"qkv": (n, H, D), "qkv_rem": (n, H, D)}
    if proof:
        shapes.update({x: (n, H, max_len) for x in PROOF})
        shapes.update({"max": (n, H), "exp_sum": (n, H)})
    got = {x: filled(*s) for x, s in shapes.items()}
    want = {x: np.full(s, UNTOUCHED, dtype=np.int32) for x, s in shapes.items()}
    wo.paged_attention(q, kc, vc, table, lens, first if first is not None else [0] * n, exp, want, **kw)
    res = ops.wit_paged_attention(dev(q), dev(kc), dev(vc), dev(table), dev(np.array(lens)), max_len, dev(exp),
                                  first=None if first is None else dev(np.array(first)), out=got, **kw)
    assert res is got
    for x in shapes:
        assert np.array_equal(host(got[x]), want[x]), (x, int((host(got[x]) != want[x]).sum()))
    return got


ATTENTIONS = [
    # lengths, first positions, heads, cache heads, dim, page
    ([1], None, 1, 1, 1, 1), ([1], None, 32, 8, 128, 16), ([37], None, 32, 8, 128, 16), ([2, 0, 5], None, 2, 1, 3, 2),
    ([0], None, 4, 2, 64, 16), ([64, 65, 63, 128, 129], None, 8, 2, 64, 16), ([300, 17, 255, 0, 1], [0, 16, 255, 0, 1], 12, 4, 80, 17),
    ([500, 20], [499, 30], 6, 2, 50, 33), ([700], None, 1, 1, 4096, 64), ([260, 3], [130, 0], 1, 1, 1024, 7), ([1030, 513], None, 16, 1, 96, 64),
    ([100, 90], None, 40, 2, 100, 16), ([2500, 1, 1024], [1, 0, 1000], 8, 8, 32, 100), ([5000], [37], 4, 1, 128, 128), ([90, 33], None, 34, 1, 33, 5)]


@pytest.mark.parametrize("lens,first,H,HK,D,page", ATTENTIONS)
def test_attention_matches_the_oracle(ops, exp_table, lens, first, H, HK, D, page):
    rng = np.random.default_rng(sum(lens) + H + D)
    table, kc, vc = paged(rng, lens, page, HK, D)
    q = gauss(rng, (len(lens), H, D))
    max_len = max(lens) + 3
    for scale in (int(round(65536 * D ** 0.5)), 1 << 22 if D >= 64 else 1 << 20):
        full = run_attention(ops, q, kc, vc, table, lens, first, exp_table, max_len, qk_scale=scale)
        answer = run_attention(ops, q, kc, vc, table, lens, first, exp_table, max_len, proof=False, qk_scale=scale)
        assert torch.equal(full["qkv"], answer["qkv"]) and torch.equal(full["qkv_rem"], answer["qkv_rem"])
        assert ops.wit_status() == 0


@pytest.mark.parametrize("seqs,longest,H,HK,D,page", [(7, 700, 4, 2, 64, 16), (8, 700, 4, 2, 64, 16), (63, 300, 2, 1, 40, 9), (64, 260, 2, 2, 32, 16), (65, 400, 3, 3, 16, 5),
                                                     (130, 300, 2, 1, 20, 16), (256, 290, 1, 1, 16, 8), (257, 290, 1, 1, 16, 8), (9, 500, 1, 1, 1024, 16), (200, 2, 1, 1, 300, 1)])
@pytest.mark.parametrize("windows", [False, True])
def test_attention_of_many_sequences(ops, exp_table, seqs, longest, H, HK, D, page, windows):
    """of every length, some of none, some refused"""
    rng = np.random.default_rng(seqs + longest)
    lens = [int(n) for n in rng.integers(0, longest + 1, seqs)]
    lens[0], lens[seqs // 2], lens[-1] = 0, longest, 0
    if seqs > 64:
        lens[60:64] = [0] * 4
    first = [int(rng.integers(0, n + 2)) for n in lens] if windows else None
    table, kc, vc = paged(rng, lens, page, HK, D)
    q = gauss(rng, (seqs, H, D))
    full = run_attention(ops, q, kc, vc, table, lens, first, exp_table, longest, qk_scale=1 << 20)
    assert ops.wit_status() == 0
    full = {x: host(t).copy() for x, t in full.items()}
    bad = np.array(lens)
    wrong = [1, seqs // 2 - 1, seqs - 2]
    bad[wrong] = [-1, longest + 1, -(1 << 31)]
    got = {x: filled(*t.shape) for x, t in full.items()}
    ops.wit_paged_attention(dev(q), dev(kc), dev(vc), dev(table), dev(bad), longest, dev(exp_table), first=None if first is None else dev(np.array(first)), out=got, qk_scale=1 << 20)
    assert ops.wit_status() == 2
    for x, t in full.items():
        t[wrong] = UNTOUCHED if t.ndim == 3 and t.shape[2] == longest and x in PROOF else 0
        assert np.array_equal(host(got[x]), t), x


@pytest.mark.parametrize("prob_scale,out_scale", [(1 << 22, 1 << 22), (1 << 30, 1 << 31), (1, 1), (3000, 777), ((1 << 22) + 1, 1 << 20)])
def test_attention_over_its_scales(ops, exp_table, prob_scale, out_scale):
    rng = np.random.default_rng(prob_scale % 1000)
    for lens, H, HK, D, page in (([70, 200], 8, 2, 64, 16), ([1500], 4, 2, 128, 32)):
        table, kc, vc = paged(rng, lens, page, HK, D, sigma=20000.0)
        run_attention(ops, gauss(rng, (len(lens), H, D)), kc, vc, table, lens, None, exp_table, max(lens), qk_scale=100000 * D // 64,
                      prob_scale=prob_scale, out_scale=out_scale)
        assert ops.wit_status() == 0


@pytest.mark.parametrize("L", [40, 1200])
def test_attention_of_the_largest_values(ops, exp_table, L):
    """keys, queries and values at the ends of 32 bits, beside ordinary ones: the products fill 64 bits"""
    rng = np.random.default_rng(8)
    H, HK, D, page = 4, 2, 64, 16
    table, kc, vc = paged(rng, [L, L], page, HK, D)
    ends = np.array([-(1 << 31), (1 << 31) - 1, TOP, TOP + 1, -TOP - 1, 0], dtype=np.int64)
    # the large parts of a key cancel in its score, the rest stays within the table
    q = rng.integers(-3, 4, (1, H, D)).astype(np.int32)
    q[..., 0], q[..., 1], q[..., 2] = 1, -1, 1
    kc[:] = gauss(rng, kc.shape, 1000.0)
    kc[..., 0] = kc[..., 1] = rng.choice(ends, kc.shape[:3])
    kc[..., 2] = rng.integers(0, 1 << 19, kc.shape[:3])
    vc[..., ::3] = rng.choice(ends, vc[..., ::3].shape)
    run_attention(ops, q, kc, vc, table[:1], [L], None, exp_table, L, qk_scale=2)
    # the largest queries and keys: scores next to the ends of 32 bits
    q = np.zeros((2, 2, D), dtype=np.int32)
    q[:, :, 0] = [(1 << 31) - 1, -(1 << 31)]
    kc[..., 0] = rng.choice(np.array([TOP, TOP + 1, TOP + 7, TOP + 1000], dtype=np.int64), kc.shape[:3])
    run_attention(ops, q, kc, vc, table, [L, L - 3], None, exp_table, L, qk_scale=1 << 31)
    assert ops.wit_status() == 0


def test_attention_reports_bad_lengths_and_pages(ops, exp_table):
    rng = np.random.default_rng(9)
    for H, HK, D, page, L in ((4, 2, 64, 16, 100), (2, 1, 6, 5, 40), (8, 1, 128, 16, 1000)):
        lens = [L, L - 1, 7]
        table, kc, vc = paged(rng, lens, page, HK, D)
        q = gauss(rng, (3, H, D))
        for bad in (-1, kc.shape[0], (1 << 31) - 1, -(1 << 31)):
            t = table.copy()
            t[1, 1] = bad                                              # its keys and values count as zero
            run_attention(ops, q, kc, vc, t, lens, None, exp_table, L, qk_scale=65536 * 8)
            assert ops.wit_status() == 2
        good = {x: t.clone() for x, t in run_attention(ops, q, kc, vc, table, [L, 0, 7], None, exp_table, L, qk_scale=65536 * 8).items()}
        assert ops.wit_status() == 0
        for ln, fs in ((L + 1, 0), (-1, 0), (L - 1, -1), (-(1 << 31), 0), ((1 << 31) - 1, 0), (table.shape[1] * page + 1, 0)):
            got = {x: torch.full_like(t, UNTOUCHED) for x, t in good.items()}
            ops.wit_paged_attention(dev(q), dev(kc), dev(vc), dev(table), dev(np.array([L, ln, 7])), L, dev(exp_table),
                                    first=dev(np.array([0, fs, 0])), out=got, qk_scale=65536 * 8)
            assert all(torch.equal(got[x], good[x]) for x in good)
            assert ops.wit_status() == 2
        # positions of the table that no sequence reaches may hold anything
        t = table.copy()
        t[2, 1:] = 1 << 30
        run_attention(ops, q, kc, vc, t, lens[:2] + [min(7, page)], None, exp_table, L, qk_scale=65536 * 8)
        assert ops.wit_status() == 0


@pytest.mark.parametrize("L", [50, 3000])
def test_attention_reports_its_table_and_sums(ops, exp_table, L):
    rng = np.random.default_rng(10)
    table, kc, vc = paged(rng, [L], 16, 1, 64)
    q = gauss(rng, (1, 2, 64))
    args = (dev(q), dev(kc), dev(vc), dev(table), dev(np.array([L])), L)
    ops.wit_paged_attention(*args, dev(exp_table), qk_scale=1 << 10)       # scores spread over far more than the table
    assert ops.wit_status() & 2
    got = ops.wit_paged_attention(*args, torch.zeros(1 << 20, dtype=torch.int32, device="cuda"), qk_scale=1 << 19)
    assert ops.wit_status() == 4 and bool((got["exp_sum"] == 1).all()) and bool((got["qkv"] == 0).all())
    neg = exp_table.copy()
    neg[-1] = -5
    ops.wit_paged_attention(*args, dev(neg), qk_scale=1 << 19)
    assert ops.wit_status() & 4
    ops.wit_paged_attention(*args, dev(exp_table), qk_scale=1)
    assert ops.wit_status() & 1


def test_attention_of_strided_caches_and_queries(ops, exp_table):
    rng = np.random.default_rng(11)
    for lens, H, HK, D, page in (([33, 70], 6, 3, 64, 16), ([900, 1300], 8, 2, 64, 16), ([40, 9], 2, 2, 30, 7)):
        table, kc, vc = paged(rng, lens, page, HK, D)
        q = gauss(rng, (len(lens), H, D))
        good = run_attention(ops, q, kc, vc, table, lens, None, exp_table, max(lens), qk_scale=65536 * 8)
        wide = torch.zeros((len(lens), H * D + 5), dtype=torch.int32, device="cuda")
        wq = wide[:, 1:1 + H * D].view(len(lens), H, D)
        wq.copy_(dev(q))
        P = kc.shape[0]
        for make in (lambda: filled(HK, P, page, D).permute(1, 2, 0, 3), lambda: filled(P, page, HK, D + 3)[..., :D],
                     lambda: filled(P, HK, page, D).permute(0, 2, 1, 3), lambda: filled(P * page * HK * D + 1)[1:].view(P, page, HK, D)):
            a, b = make(), make()
            a.copy_(dev(kc)), b.copy_(dev(vc))
            got = ops.wit_paged_attention(wq, a, b, dev(table), dev(np.array(lens)), max(lens), dev(exp_table), qk_scale=65536 * 8,
                                          out={x: filled(*t.shape) for x, t in good.items()})
            assert all(torch.equal(got[x], good[x]) for x in good)
    assert ops.wit_status() == 0


def test_attention_with_some_outputs_and_a_kept_workspace(ops, exp_table):
    rng = np.random.default_rng(12)
    for lens in ([50, 20], [1500, 700]):
        table, kc, vc = paged(rng, lens, 16, 2, 64)
        q, L = gauss(rng, (2, 4, 64)), max(lens)
        good = run_attention(ops, q, kc, vc, table, lens, None, exp_table, L, qk_scale=65536 * 8)
        ws = torch.randint(-128, 127, (ops.wit_paged_attention_workspace(2, 4, 2, 64, L),), device="cuda", dtype=torch.int8).view(torch.uint8)
        for keep in (("qkv",), ("qkv", "scores"), ("qkv", "exp_output", "max"), ("qkv", "softmax_output", "exp_sum"), ("qkv", "qkv_rem", "softmax_lookup_query"),
                     ("qkv", "exp_input", "scores_rem")):
            got = ops.wit_paged_attention(dev(q), dev(kc), dev(vc), dev(table), dev(np.array(lens)), L, dev(exp_table), qk_scale=65536 * 8,
                                          out={x: filled(*good[x].shape) for x in keep}, workspace=ws)
            assert all(torch.equal(got[x], good[x]) for x in keep)
    fresh = ops.wit_paged_attention(dev(q), dev(kc), dev(vc), dev(table), dev(np.array(lens)), L, dev(exp_table), qk_scale=65536 * 8)
    assert set(fresh) == set(good) and torch.equal(fresh["qkv"], good["qkv"])
    assert ops.wit_status() == 0


# ------------------------------------------------------------------ 4-bit weights
Q4 = [
    # tokens, outputs, inputs, group
    (1, 1, 1, 1), (1, 3, 2, 1), (2, 5, 7, 3), (1, 64, 64, 32), (1, 4096, 4096, 128), (3, 100, 200, 64), (5, 33, 1000, 128), (1, 257, 96, 32),
    (16, 130, 11008, 128), (17, 65, 512, 256), (4, 777, 1001, 100), (40, 31, 320, 64), (2, 16, 8200, 8200), (1, 20, 130, 4096), (9, 48, 288, 96),
    (7, 2049, 1024, 32), (24, 300, 160, 16),
    (2, 1040, 40000, 128), (3, 8200, 2600, 64), (4, 9000, 2050, 96), (2, 65, 33000, 32), (6, 8200, 520, 32), (12, 8200, 200, 128)]


def q4_case(rng, n, m, k, group, top=400):
    groups = -(-k // group)
    return (gauss(rng, (n, k)), rng.integers(0, 256, (m, (k + 1) // 2)).astype(np.uint8), rng.integers(-top, top + 1, (m, groups)).astype(np.int32),
            rng.integers(0, 16, (m, groups)).astype(np.uint8))


@pytest.mark.parametrize("n,m,k,group", Q4)
def test_q4_matches_the_oracle(ops, n, m, k, group):
    rng = np.random.default_rng(n + m + k)
    x, w, scales, zeros = q4_case(rng, n, m, k, group)
    for z, scale in ((None, 1 << 16), (zeros, 1 << 20), (zeros, 99999)):
        want = wo.matvec_q4(x, w, scales, group, z, scale)
        q, r = ops.wit_matvec_q4(dev(x), dev(w), dev(scales), group, zeros=None if z is None else dev(z), scale=scale)
        assert np.array_equal(host(q), want[0]) and np.array_equal(host(r), want[1])
    q2, r2 = ops.wit_matvec_q4(dev(x), dev(w), dev(scales), group, zeros=dev(zeros), scale=99999, want_r=False)
    assert r2 is None and torch.equal(q2, q)
    assert ops.wit_status() == 0


@pytest.mark.parametrize("n", [1, 3, 4, 5, 8, 9, 16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_q4_of_rows_that_end_anywhere(ops, n, group):
    rng = np.random.default_rng(n + group)
    for k in (1, 2, 7, 8, 9, 15, 31, 32, 33, 63, 65, 95, 127, 129, 160, 223, 255, 257, 500, 511, 513, 1000, 1025, 2047):
        # two to four tokens through that many rows have their digits made beforehand, as more tokens always have
        m = 16 * (40000 // (n * ((k + 127) // 128))) + 17 if 2 <= n <= 4 and k in (1000, 1025) else 17
        x, w, scales, zeros = q4_case(rng, n, m, k, group)
        want = wo.matvec_q4(x, w, scales, group, zeros)
        # rows that stand at any byte, between others that hold anything
        wide = dev(rng.integers(0, 256, (m, w.shape[1] + 5), dtype=np.uint8))
        rows = wide[:, 3:3 + w.shape[1]]
        rows.copy_(dev(w))
        got = ops.wit_matvec_q4(dev(x), rows, dev(scales), group, zeros=dev(zeros))
        assert np.array_equal(host(got[0]), want[0]) and np.array_equal(host(got[1]), want[1]), k
    assert ops.wit_status() == 0


def test_q4_equals_the_product_with_the_weights_written_out(ops):
    rng = np.random.default_rng(3)
    x, w, scales, zeros = q4_case(rng, 5, 300, 512, 64)
    full = wo.weights_q4(w, scales, 64, zeros, 512).astype(np.int32)
    a = ops.wit_matmul_rescale(dev(x), dev(full), 1 << 16)
    b = ops.wit_matvec_q4(dev(x), dev(w), dev(scales), 64, zeros=dev(zeros))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert ops.wit_status() == 0


@pytest.mark.parametrize("k,group", [(64, 32), (70, 7), (4096, 128)])
def test_q4_of_the_largest_values(ops, k, group):
    rng = np.random.default_rng(4)
    x, w, scales, zeros = q4_case(rng, 6, 50, k, group, top=3)
    ends = np.array([-(1 << 31), (1 << 31) - 1, TOP, TOP + 1, -TOP - 1], dtype=np.int64)
    x[:] = rng.choice(ends, x.shape)
    x[1:3] = gauss(rng, x[1:3].shape)
    x[2, k // 2] = TOP + 1
    x[3] = (1 << 31) - 1
    want = wo.matvec_q4(x, w, scales, group, zeros, 1 << 31)
    q, r = ops.wit_matvec_q4(dev(x), dev(w), dev(scales), group, zeros=dev(zeros), scale=1 << 31)
    assert np.array_equal(host(q), want[0]) and np.array_equal(host(r), want[1])
    # scales and zero points over their whole range
    scales[:] = rng.choice(np.array([-(1 << 31), (1 << 31) - 1, 1, 0]), scales.shape)
    zeros[:] = rng.choice(np.array([0, 15, 128, 255]), zeros.shape)
    x = rng.integers(-3, 4, x.shape).astype(np.int32)
    want = wo.matvec_q4(x, w, scales, group, zeros, 1 << 31)
    q, r = ops.wit_matvec_q4(dev(x), dev(w), dev(scales), group, zeros=dev(zeros), scale=1 << 31)
    assert np.array_equal(host(q), want[0]) and np.array_equal(host(r), want[1])
    assert ops.wit_status() == 0
    ops.wit_matvec_q4(dev(x), dev(w), dev(scales), group, zeros=dev(zeros), scale=1)
    assert ops.wit_status() == 1


def test_rescaling_by_any_scale_is_exact_over_64_bits(ops):
    """quotients far beyond 32 bits are reported; their low 32 bits and the remainders are those of the whole numbers"""
    rng = np.random.default_rng(14)
    m = 500
    x = np.array([[(1 << 31) - 1], [-(1 << 31)], [1], [1 << 20]], dtype=np.int64).astype(np.int32)
    w, zeros = rng.integers(0, 16, (m, 1)).astype(np.uint8), np.full((m, 1), 8, dtype=np.uint8)
    scales = rng.integers(-(1 << 28), 1 << 28, (m, 1)).astype(np.int32)
    scales[::3] = rng.integers(-50, 50, scales[::3].shape)
    y = [[int(a[0]) * int(s[0]) * ((int(b[0]) & 15) - 8) for b, s in zip(w, scales)] for a in x]
    for s in (3, 5, 7, 999, 999983, (1 << 31) - 1, 3 << 20):
        q, r = ops.wit_matvec_q4(dev(x), dev(w), dev(scales), 1, zeros=dev(zeros), scale=s)
        want = [[(v + s // 2) // s for v in row] for row in y]
        assert host(r).tolist() == [[v - k * s for v, k in zip(row, ks)] for row, ks in zip(y, want)]
        assert (host(q).astype(np.int64) % (1 << 32)).tolist() == [[k % (1 << 32) for k in ks] for ks in want]
        assert ops.wit_status() == (1 if any(not -(1 << 31) <= k < 1 << 31 for ks in want for k in ks) else 0)


def test_q4_of_strided_rows(ops):
    rng = np.random.default_rng(13)
    for n, m, k, group in ((3, 70, 256, 64), (2, 33, 77, 32), (1, 40, 1024, 128)):
        x, w, scales, zeros = q4_case(rng, n, m, k, group)
        good = ops.wit_matvec_q4(dev(x), dev(w), dev(scales), group, zeros=dev(zeros))
        wide, ww = torch.zeros((n, k + 3), dtype=torch.int32, device="cuda"), torch.zeros((m, w.shape[1] + 5), dtype=torch.uint8, device="cuda")
        wide[:, 1:1 + k] = dev(x)
        ww[:, 3:3 + w.shape[1]] = dev(w)
        got = ops.wit_matvec_q4(wide[:, 1:1 + k], ww[:, 3:3 + w.shape[1]], dev(scales), group, zeros=dev(zeros))
        assert torch.equal(got[0], good[0]) and torch.equal(got[1], good[1])
        one = ops.wit_matvec_q4(dev(x[:1]).expand(4, k), dev(w), dev(scales), group, zeros=dev(zeros))[0]     # the same token four times
        assert all(torch.equal(row, good[0][0]) for row in one)
    assert ops.wit_status() == 0


# ------------------------------------------------------------------ as they are used
def test_empty_calls_do_nothing(ops, exp_table):
    none = torch.zeros((0, 2, 8), dtype=torch.int32, device="cuda")
    kc, vc = filled(2, 4, 2, 8), filled(2, 4, 2, 8)
    tab = torch.zeros((4, 4), dtype=torch.int32, device="cuda")
    idx = torch.zeros(0, dtype=torch.int32, device="cuda")
    ops.wit_rope_append(none, none, none, idx, idx.long(), tab, tab, kc, vc)
    ops.wit_paged_attention(none, kc, vc, idx.view(0, 0), idx, 5, dev(exp_table))
    assert bool((kc == UNTOUCHED).all()) and bool((vc == UNTOUCHED).all())
    one = ops.wit_paged_attention(filled(1, 2, 8), kc, vc, torch.zeros((1, 0), dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), 0,
                                  dev(exp_table))                            # no position anywhere
    assert bool((one["qkv"] == 0).all()) and bool((one["max"] == 0).all())
    one = ops.wit_paged_attention(filled(2, 1, 300), filled(2, 4, 1, 300), filled(2, 4, 1, 300), torch.zeros((2, 0), dtype=torch.int32, device="cuda"),
                                  torch.zeros(2, dtype=torch.int32, device="cuda"), 0, dev(exp_table))
    assert bool((one["qkv"] == 0).all()) and bool((one["qkv_rem"] == 0).all()) and bool((one["exp_sum"] == 0).all())
    q, r = ops.wit_matvec_q4(filled(0, 16), torch.zeros((4, 8), dtype=torch.uint8, device="cuda"), filled(4, 1), 16)
    assert q.shape == (0, 4)
    q, r = ops.wit_matvec_q4(filled(2, 16), torch.zeros((0, 8), dtype=torch.uint8, device="cuda"), filled(0, 1), 16)
    assert q.shape == (2, 0)
    assert ops.wit_status() == 0


class Decoder:
    """one attention block of a model with 4-bit projections over a paged cache, token by token"""

    def __init__(self, ops, rng, seqs, H, HK, D, page, steps, exp):
        self.ops, self.seqs, self.H, self.HK, self.D, self.page, self.steps = ops, seqs, H, HK, D, page, steps
        width, group = H * D, 64
        self.group, out = group, (H + 2 * HK) * D
        self.w = {"qkv": q4_case(rng, 1, out, width, group, top=int(65536 / (4 * width ** 0.5)))[1:],
                  "o": q4_case(rng, 1, width, width, group, top=int(65536 / (4 * width ** 0.5)))[1:]}
        self.each = -(-steps // page)
        self.table = rng.permutation(seqs * self.each).astype(np.int32).reshape(seqs, self.each)
        self.cos, self.sin = tables(steps, D, 1 << 16)
        self.exp, self.scale = exp, int(round(65536 * D ** 0.5))
        self.x = gauss(rng, (steps, seqs, width))
        self.dw = {n: [dev(t) for t in ts] for n, ts in self.w.items()}
        self.dx, self.dcos, self.dsin, self.dexp, self.dtable = dev(self.x), dev(self.cos), dev(self.sin), dev(exp), dev(self.table)
        self.kc, self.vc = filled(seqs * self.each, page, HK, D), filled(seqs * self.each, page, HK, D)
        self.keep = {n: filled(*s) for n, s in (("qkv", (seqs, H, D)), ("qkv_rem", (seqs, H, D)), ("max", (seqs, H)), ("exp_sum", (seqs, H)))}
        self.keep.update({n: filled(seqs, H, steps) for n in PROOF})
        self.proj, self.proj_r, self.rot, self.rot_r = filled(seqs, out), filled(seqs, out), filled(seqs, H, D), filled(seqs, H, D)
        self.k_r, self.y, self.y_r = filled(seqs, HK, D), filled(seqs, width), filled(seqs, width)
        self.positions = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        self.slots = torch.zeros(seqs, dtype=torch.int64, device="cuda")
        self.cur = torch.zeros((seqs, width), dtype=torch.int32, device="cuda")

    def feed(self, t):
        """what the next step reads: the inputs, positions and slots of token t"""
        self.cur.copy_(self.dx[t])
        self.positions.fill_(t)
        self.lens.fill_(t + 1)
        self.slots.copy_(self.dtable[:, t // self.page].long() * self.page + t % self.page)

    def step(self):
        o, H, HK, D = self.ops, self.H, self.HK, self.D
        o.wit_matvec_q4(self.cur, *self.dw["qkv"][:2], self.group, zeros=self.dw["qkv"][2], q=self.proj, r=self.proj_r)
        q, k, v = (self.proj[:, a * D:b * D].view(self.seqs, -1, D) for a, b in ((0, H), (H, H + HK), (H + HK, H + 2 * HK)))
        o.wit_rope_append(q, k, v, self.positions, self.slots, self.dcos, self.dsin, self.kc, self.vc, self.rot, self.rot_r, self.k_r)
        o.wit_paged_attention(self.rot, self.kc, self.vc, self.dtable, self.lens, self.steps, self.dexp, qk_scale=self.scale, out=self.keep)
        o.wit_matvec_q4(self.keep["qkv"].view(self.seqs, H * D), *self.dw["o"][:2], self.group, zeros=self.dw["o"][2], q=self.y, r=self.y_r)

    def outputs(self):
        return [self.proj, self.proj_r, self.rot, self.rot_r, self.k_r, self.y, self.y_r, self.kc, self.vc] + [self.keep[n] for n in sorted(self.keep)]

    def oracle(self, upto):
        """outputs() after the steps 0..upto"""
        H, HK, D, n = self.H, self.HK, self.D, self.seqs
        kc, vc = (np.full(tuple(self.kc.shape), UNTOUCHED, dtype=np.int32) for _ in range(2))
        keep = {x: np.full(tuple(t.shape), UNTOUCHED, dtype=np.int32) for x, t in self.keep.items()}
        for t in range(upto + 1):
            proj = wo.matvec_q4(self.x[t], self.w["qkv"][0], self.w["qkv"][1], self.group, self.w["qkv"][2])
            q, k, v = (proj[0][:, a * D:b * D].reshape(n, -1, D) for a, b in ((0, H), (H, H + HK), (H + HK, H + 2 * HK)))
            rot, rot_r, k_r = np.zeros((n, H, D), np.int32), np.zeros((n, H, D), np.int32), np.zeros((n, HK, D), np.int32)
            slots = self.table[:, t // self.page].astype(np.int64) * self.page + t % self.page
            wo.rope_append(q, k, v, np.full(n, t), slots, self.cos, self.sin, kc, vc, rot, rot_r, k_r, False)
        wo.paged_attention(rot, kc, vc, self.table, [upto + 1] * n, [0] * n, self.exp, keep, qk_scale=self.scale)
        y = wo.matvec_q4(keep["qkv"].reshape(n, H * D), self.w["o"][0], self.w["o"][1], self.group, self.w["o"][2])
        return [proj[0], proj[1], rot, rot_r, k_r, y[0], y[1], kc, vc] + [keep[x] for x in sorted(keep)]


def test_a_block_token_by_token(ops, exp_table):
    d = Decoder(ops, np.random.default_rng(20), 3, 4, 2, 64, 16, 40, exp_table)
    for t in range(40):
        d.feed(t)
        d.step()
        if t in (0, 15, 16, 39):
            assert all(np.array_equal(host(g)[..., :t + 1] if g.shape[-1] == 40 else host(g), w[..., :t + 1] if w.shape[-1] == 40 else w)
                       for g, w in zip(d.outputs(), d.oracle(t)))
    assert ops.wit_status() == 0


def test_the_last_token_of_a_prompt_sees_what_the_whole_prompt_kernels_compute(ops, exp_table):
    """one head, nothing rotated: the last rows of the prompt's scores, softmax and products"""
    rng = np.random.default_rng(21)
    T, D, page = 200, 128, 16
    q, k, v = (gauss(rng, (T, 1, D)) for _ in range(3))
    order = rng.permutation(-(-T // page) + 1)
    kc, vc = filled(len(order), page, 1, D), filled(len(order), page, 1, D)
    slots = torch.from_numpy(order[np.arange(T) // page] * page + np.arange(T) % page).cuda()
    none = torch.zeros((1, 0), dtype=torch.int32, device="cuda")
    ops.wit_rope_append(None, dev(k), dev(v), torch.zeros(T, dtype=torch.int32, device="cuda"), slots, none, none, kc, vc)
    got = ops.wit_paged_attention(dev(q[-1:]), kc, vc, dev(order[None, :-1]), dev(np.array([T])), T, dev(exp_table), qk_scale=1 << 20)
    scores, rem = ops.wit_matmul_rescale(dev(q[:, 0]), dev(k[:, 0]), 1 << 20)
    soft = ops.wit_softmax(scores, dev(exp_table))
    qkv, qkv_rem = ops.wit_matmul_rescale(soft["softmax_output"], dev(np.ascontiguousarray(v[:, 0].T)), 1 << 16)
    for name, t in {"scores": scores, "scores_rem": rem, "qkv": qkv, "qkv_rem": qkv_rem, **soft}.items():
        assert torch.equal(got[name].reshape(-1), t[-1].reshape(-1)), name
    assert ops.wit_status() == 0


@pytest.mark.parametrize("seqs,steps", [(2, 24), (6, 300)])
def test_captured_steps_replay(ops, exp_table, seqs, steps):
    """one captured step a model, two models' graphs replayed at once on two streams, with eager work between; two sequences in the
    forms of one launch, six with workspaces"""
    a, b = (Decoder(ops, np.random.default_rng(s), seqs, 4, 2, 64, 16, steps, exp_table) for s in (30, 31))
    graphs = []
    for d in (a, b):
        d.feed(0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            d.step()                                                  # each shape once before it is captured
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            d.step()
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for t in range(6):
        for d in (a, b):
            d.feed(t)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for d in (a, b):
            assert all(np.array_equal(host(x)[..., :t + 1] if x.shape[-1] == steps else host(x), w[..., :t + 1] if w.shape[-1] == steps else w)
                       for x, w in zip(d.outputs(), d.oracle(t)))
        ops.wit_paged_attention(a.rot, a.kc, a.vc, a.dtable, a.lens, steps, a.dexp, qk_scale=a.scale)         # eager, its own workspace
    assert ops.wit_status() == 0


def test_attention_on_two_streams_at_once(ops, exp_table):
    rng = np.random.default_rng(40)
    lens = [1500, 900]
    cases, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in streams:
        table, kc, vc = paged(rng, lens, 16, 2, 64)
        cases.append([dev(gauss(rng, (2, 8, 64))), dev(kc), dev(vc), dev(table), dev(np.array(lens)), 1500, dev(exp_table)])
    good = [ops.wit_paged_attention(*c, qk_scale=65536 * 8) for c in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(ops.wit_paged_attention(*c, qk_scale=65536 * 8))
        torch.cuda.synchronize()
        for x, y in zip(got, good):
            assert all(torch.equal(x[n], y[n]) for n in y)
    assert ops.wit_status() == 0


FIRST_CALL_CAPTURED = """
import numpy as np, torch
from grape_amd import ops
from oracle import witness_oracle as wo
ops.init()
rng = np.random.default_rng(1)
x, w = rng.integers(-1000, 1000, (1, 100)).astype(np.int32), rng.integers(0, 256, (40, 50)).astype(np.uint8)
scales = rng.integers(-400, 400, (40, 4)).astype(np.int32)
dx, dw, ds = (torch.from_numpy(a).cuda() for a in (x, w, scales))
q, r = torch.zeros((1, 40), dtype=torch.int32, device="cuda"), torch.zeros((1, 40), dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    ops.wit_matvec_q4(dx, dw, ds, 32, q=q, r=r)
for _ in range(3):
    q.fill_(-1), r.fill_(-1)
    graph.replay()
    torch.cuda.synchronize()
    want = wo.matvec_q4(x, w, scales, 32, None)
    assert np.array_equal(q.cpu().numpy(), want[0]) and np.array_equal(r.cpu().numpy(), want[1])
assert ops.wit_status() == 0
print("captured")
"""


def test_the_first_call_of_a_process_may_be_captured():
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    res = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED], cwd=here, capture_output=True, text=True, timeout=100)
    assert res.returncode == 0 and "captured" in res.stdout, res.stderr
