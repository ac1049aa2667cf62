"""GPU tests of the new tokens' calls at their edges: rows of equal scores, sums next to and beyond 32 bits, forms of the
kernels that need large products, odd heads with fine probabilities, or long heads with the largest values.  The
helpers are those of test_gpu_tokens.py; every result is a whole number and is compared exactly with the numpy oracle."""
import numpy as np
import pytest
import torch
from oracle import witness_oracle as wo
from test_gpu_tokens import TOP, dev, exp_table, filled, gauss, host, ops, paged, q4_case, run_attention  # noqa: F401  (two of them are fixtures)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ one launch: a row's scores and exponentials in one place
@pytest.mark.parametrize("each", [1, 2, 4])
@pytest.mark.parametrize("score", [0, 3 << 20, -(3 << 20)])
def test_equal_scores_set_no_bit(ops, exp_table, each, score):
    """Every score of a row is the same, so that none of its exponentials - 2^16 each - would pass for a score: read in a score's
    place, the exponential's index is above the table with scores of 0 or less and below it with scores of 3 * 2^20.  One, two and four query
    heads a cache head give a row's positions to eight, four and two waves."""
    rng = np.random.default_rng(each)
    HK, D, page = 2, 64, 16
    q = np.zeros((3, each * HK, D), dtype=np.int32)
    q[:, :, 5] = score
    for n in (100, 129, 200, 255, 256):
        lens = [n, n - 1, 100]
        table, kc, vc = paged(rng, lens, page, HK, D)
        kc[..., 5] = 1
        got = run_attention(ops, q, kc, vc, table, lens, None, exp_table, n, qk_scale=1)
        assert ops.wit_status() == 0
        assert bool((got["scores"][0] == score).all()) and bool((got["exp_output"][0] == 1 << 16).all())
        assert ops.wit_status() == 0


# ------------------------------------------------------------------ sums and lookup queries that leave int32
ROWS = ("scores", "scores_rem", "exp_input", "exp_output", "softmax_output")          # of a proof, in 32 bits whatever the sum is
INT32 = range(-(1 << 31), 1 << 31)


def attend_flat(ops, lens, exp, out, H=2, HK=1, D=8, page=64, **kw):
    """rows of equal scores over caches of ordinary values; what the call gave, the oracle's outputs and the sums and queries as whole numbers"""
    rng = np.random.default_rng(sum(lens))
    table, kc, vc = paged(rng, lens, page, HK, D)
    q = np.zeros((len(lens), H, D), dtype=np.int32)
    shapes = {"qkv": (len(lens), H, D), "qkv_rem": (len(lens), H, D), "max": (len(lens), H), "exp_sum": (len(lens), H)}
    got = {x: filled(*shapes.get(x, (len(lens), H, max(lens)))) for x in out}
    want = {x: np.full(t.shape, -77, dtype=np.int32) for x, t in got.items()}
    wo.paged_attention(q, kc, vc, table, lens, [0] * len(lens), exp, want, **kw)
    ops.wit_paged_attention(dev(q), dev(kc), dev(vc), dev(table), dev(np.array(lens)), max(lens), dev(exp), out=got, **kw)
    e = int(exp[(1 << 20) - 1])
    sums = [n * e for n in lens if n]
    prob = kw.get("prob_scale", 1 << 16)
    queries = [2 * prob * e - s * (2 * ((e * prob + s // 2) // s) - 1) for s in sums]
    return got, want, sums, queries


@pytest.mark.parametrize("lens", [[16384], [32767], [32768], [65536, 100], [0, 40000, 3], [131072]])
def test_sums_and_queries_beyond_32_bits_are_reported(ops, exp_table, lens):
    """each entry is 2^16: a sum of 32768 and a query of some 16384 positions on leave int32, and 65536 positions' sum is 0 in 32 bits"""
    for names, of in ((ROWS + ("max",), ()), (("exp_sum",), ("sum",)), (("softmax_lookup_query",), ("query",)), (("exp_sum", "softmax_lookup_query"), ("sum", "query")), ((), ())):
        got, want, sums, queries = attend_flat(ops, lens, exp_table, ("qkv", "qkv_rem") + names)
        wide = ("sum" in of and any(s not in INT32 for s in sums)) or ("query" in of and any(s not in INT32 for s in queries))
        assert ops.wit_status() == (16 if wide else 0), (names, sums, queries)
        for x in got:                                                             # the answer is exact, the low 32 bits are stored
            assert np.array_equal(got[x].cpu().numpy(), want[x]), x


@pytest.mark.parametrize("lens", [[200], [250, 1, 0], [900, 300]])
@pytest.mark.parametrize("entry", [(1 << 31) // 250, (1 << 31) // 249, 1 << 30, (1 << 31) - 1])
def test_sums_of_large_entries_are_reported(ops, lens, entry):
    """the same up to 256 positions, where the call is one launch, with a table of larger entries"""
    table = np.full(1 << 20, entry, dtype=np.int32)
    for prob_scale in (1 << 16, 3000):
        got, want, sums, queries = attend_flat(ops, lens, table, ("qkv", "qkv_rem", "exp_sum", "softmax_lookup_query") + ROWS, H=3, HK=3, prob_scale=prob_scale)
        assert ops.wit_status() == (16 if any(s not in INT32 for s in sums + queries) else 0)
        got2, _, _, _ = attend_flat(ops, lens, table, ("qkv",), H=3, HK=3, prob_scale=prob_scale)
        assert ops.wit_status() == 0 and torch.equal(got2["qkv"], got["qkv"])
        for x in got:
            assert np.array_equal(got[x].cpu().numpy(), want[x]), x


# ------------------------------------------------------------------ forms that few sizes choose
@pytest.mark.parametrize("n,m,k,group", [(6, 8200, 520, 128), (8, 8161, 1030, 256), (12, 8200, 200, 64), (16, 8177, 300, 192), (20, 8200, 200, 128), (33, 4100, 130, 64), (37, 5000, 257, 128),
                                         (20, 8200, 160, 32)])
def test_q4_of_many_rows_and_tiles_of_tokens(ops, n, m, k, group):
    """two tiles of rows a workgroup, of five to sixteen tokens and of more than one tile of tokens, with inputs above the digits"""
    rng = np.random.default_rng(n * m + k)
    x, w, scales, zeros = q4_case(rng, n, m, k, group, top=200)
    x[n - 1, k - 1], x[0, 0] = TOP + 1, (1 << 31) - 1
    for z in (None, zeros):
        want = wo.matvec_q4(x, w, scales, group, z, 1 << 24)
        q, r = ops.wit_matvec_q4(dev(x), dev(w), dev(scales), group, zeros=None if z is None else dev(z), scale=1 << 24)
        assert np.array_equal(host(q), want[0]) and np.array_equal(host(r), want[1])
    assert ops.wit_status() == 0


@pytest.mark.parametrize("n,m,k,group", [(1, 4096, 11008, 128), (1, 70, 16384, 64), (1, 33, 40000, 32), (1, 16, 33001, 128), (2, 100, 9000, 128), (4, 33, 4900, 64)])
def test_q4_of_few_tokens_with_long_inputs(ops, n, m, k, group):
    """digits and turned weights of up to 124 KB a workgroup, inputs that go through in pieces"""
    rng = np.random.default_rng(m + k)
    x, w, scales, zeros = q4_case(rng, n, m, k, group, top=60)
    x[0, [0, k // 2, k - 1]] = TOP + 1, -(1 << 31), (1 << 31) - 1
    for z in (None, zeros):
        want = wo.matvec_q4(x, w, scales, group, z, 1 << 20)
        q, r = ops.wit_matvec_q4(dev(x), dev(w), dev(scales), group, zeros=None if z is None else dev(z), scale=1 << 20)
        assert np.array_equal(host(q), want[0]) and np.array_equal(host(r), want[1])
    assert ops.wit_status() == 0


@pytest.mark.parametrize("prob_scale,out_scale", [((1 << 22) + 1, 1 << 20), (1 << 30, 1 << 31)])
@pytest.mark.parametrize("lens,H,HK,D,page", [([70, 200], 6, 2, 30, 9), ([256, 1], 5, 5, 50, 16), ([1500, 800], 4, 2, 30, 32), ([700], 34, 2, 50, 7), ([300, 299], 2, 1, 257, 16)])
def test_fine_probabilities_of_heads_of_odd_sizes(ops, exp_table, lens, H, HK, D, page, prob_scale, out_scale):
    """four planes of a probability, elements that are not read four at a time"""
    rng = np.random.default_rng(D + len(lens))
    table, kc, vc = paged(rng, lens, page, HK, D, sigma=20000.0)
    for proof in (True, False):
        run_attention(ops, gauss(rng, (len(lens), H, D)), kc, vc, table, lens, None, exp_table, max(lens), proof=proof, qk_scale=200000, prob_scale=prob_scale, out_scale=out_scale)
    assert ops.wit_status() == 0


@pytest.mark.parametrize("D", [512, 576, 1000, 1024, 4096])
def test_long_heads_of_the_largest_values(ops, exp_table, D):
    """queries above four planes of digits where the waves of a workgroup share a head's elements, an odd number of 64s among them"""
    rng = np.random.default_rng(D)
    H, HK, page, L = 2, 1, 16, 300
    table, kc, vc = paged(rng, [L, L], page, HK, D, sigma=1000.0)
    ends = np.array([-(1 << 31), (1 << 31) - 1, TOP, TOP + 1, -TOP - 1, 0], dtype=np.int64)
    # products of the largest queries with the largest keys cancel, at both ends of a head and in its middle
    q = rng.integers(-3, 4, (2, H, D)).astype(np.int32)
    for a, b in ((0, 1), (D // 2, D // 2 + 1), (D - 2, D - 1)):
        q[..., a] = q[..., b] = rng.choice(np.array([(1 << 31) - 1, TOP + 1, TOP, -(1 << 31)]), (2, H))
        large = rng.integers(-(1 << 28), 1 << 28, kc.shape[:3])
        kc[..., a], kc[..., b] = large, -large
    vc[..., ::3] = rng.choice(ends, vc[..., ::3].shape)
    run_attention(ops, q, kc, vc, table, [L, L - 7], None, exp_table, L, qk_scale=8)
    # scores next to the ends of 32 bits
    q = np.zeros((2, H, D), dtype=np.int32)
    q[:, :, D - 1] = [(1 << 31) - 1, -(1 << 31)]
    q[:, :, 3] = TOP + 5
    kc[:] = 0
    kc[..., D - 1] = rng.choice(np.array([TOP, TOP + 1, TOP + 7, TOP + 1000], dtype=np.int64), kc.shape[:3])
    kc[..., 3] = rng.integers(-500, 500, kc.shape[:3])
    run_attention(ops, q, kc, vc, table, [L, L - 3], None, exp_table, L, qk_scale=1 << 31)
    assert ops.wit_status() == 0
