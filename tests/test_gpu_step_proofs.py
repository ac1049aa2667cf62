"""What a step of several new tokens writes, taken into proofs: the products with keys and values of a piece of a prompt behind a window,
the lookups of its exponentials, and the choice of the next token by lookups of how far the others are below it.  Transcripts are
compared with the CPU oracle's."""
import numpy as np
import pytest
import torch
import bigref as br
import orc
from gpuutil import assert_same, rand_fr
from test_gpu_host import gens, host  # noqa: F401  (fixtures)
from test_gpu_token_proofs import OUT, QK, SHIFT, evaluation, padded
from test_gpu_tokens import dev, gauss, ops, paged  # noqa: F401  (ops is a fixture)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def piece(ops):
    """the last 8 tokens of a sequence of 29, beside one of two tokens, behind a window of 11 and the first 3"""
    rng = np.random.default_rng(60)
    lens, starts, H, HK, D, page = [29, 2], [0, 8, 10], 4, 2, 16, 8
    table, kc, vc = paged(rng, lens, page, HK, D, sigma=180.0)
    exp = np.rint(np.exp((np.arange(1 << SHIFT) - ((1 << SHIFT) - 1)) / 128.0) * 65536).astype(np.int32)
    s = {"q": dev(gauss(rng, (10, H, D), 180.0)), "k": dev(kc), "v": dev(vc), "pages": dev(table), "exp": dev(exp), "page": page}
    s["out"] = ops.wit_window_attention(s["q"], s["k"], s["v"], s["pages"], dev(np.array(starts)), dev(np.array(lens)), 8, 32, s["exp"], window=11, sinks=3, bit_shift=SHIFT,
                                        index_bits=SHIFT, qk_scale=QK, out_scale=OUT)
    assert ops.wit_status() == 0
    pos, t = torch.arange(21, 29, device="cuda")[:, None], torch.arange(32, device="cuda")[None]
    s["sees"] = (t <= pos) & ((t > pos - 11) | (t < 3))
    return s


def test_the_products_of_a_piece_are_proved(ops, host, piece):
    """cache heads as layers, a token's query heads of a cache head as rows, token after token.  The scores that a token does not attend to belong to the
    product with the keys all the same, and come from the product of its own; the probabilities there are zero."""
    out, pages, page, n, rows, N = piece["out"], piece["pages"], piece["page"], 29, 8, 32
    H, HK, D = piece["q"].shape[1], piece["k"].shape[2], piece["q"].shape[2]
    each = H // HK
    t = torch.arange(n, device="cuda")
    keys, values = (torch.zeros((HK, N, D), dtype=torch.int32, device="cuda") for _ in range(2))
    keys[:, :n], values[:, :n] = (c[pages[0, t // page].long(), t % page].transpose(0, 1) for c in (piece["k"], piece["v"]))

    def by_cache_head(x):
        return x[:rows].reshape(rows, HK, each, -1).transpose(0, 1).reshape(HK, rows * each, -1).contiguous()
    queries, seen = by_cache_head(piece["q"]), by_cache_head(piece["sees"][:, None].expand(rows, H, N))
    scores, rem = by_cache_head(out["scores"]), by_cache_head(out["scores_rem"])
    for h in range(HK):
        q, r = ops.wit_matmul_rescale(queries[h].contiguous(), keys[h].contiguous(), QK)
        assert torch.equal(q[seen[h]], scores[h][seen[h]]) and torch.equal(r[seen[h]], rem[h][seen[h]])
        scores[h], rem[h] = q, r
    prob = by_cache_head(out["softmax_output"])
    assert not bool(prob[~seen].any())
    for A, B, M, K, q, r, scale in ((queries, keys, N, D, scores, rem, QK), (prob, values.transpose(1, 2).contiguous(), D, N, by_cache_head(out["qkv"]), by_cache_head(out["qkv_rem"]), OUT)):
        L, rows_all = HK, rows * each
        u, v = rand_fr(br.log2ceil(L * rows_all * M), 81), rand_fr(br.log2ceil(L * K), 82)
        claim = evaluation(host, ops, q, r, scale, u)
        Af, Bf = (x.reshape(-1).contiguous() for x in (A, B))
        st, wtr, wclaim, wac, wbc = orc.prove_matmul(orc.from_i32(Af.cpu().numpy()), orc.from_i32(Bf.cpu().numpy()), L, rows_all, M, K, u, v, claim)
        assert st == 0
        tr, end, ac, bc = host.prove_matmul(ops.fr_from_i32(Af), ops.fr_from_i32(Bf), L, rows_all, M, K, u, v, claim)
        assert_same(tr, wtr, "transcript")
        assert_same(end, wclaim, "final claim")
        assert_same(ac, wac, "A(v)")
        assert_same(bc, wbc, "B(v)")
        wrong = r.clone()
        wrong[0, 0, 0] += 1
        with pytest.raises(host.HostError, match="matmul_phase"):
            host.prove_matmul(ops.fr_from_i32(Af), ops.fr_from_i32(Bf), L, rows_all, M, K, u, v, evaluation(host, ops, q, wrong, scale, u))


def test_the_exponentials_of_a_piece_are_looked_up(ops, host, gens, piece):
    out, n, sees = piece["out"], 1 << SHIFT, piece["sees"][:, None].expand(8, 4, 32)
    x, y = out["exp_input"][:8][sees], out["exp_output"][:8][sees]
    assert x.numel() == 8 * 4 * 14
    x, y = padded(x, n, 0), padded(y, n, int(piece["exp"][-1]))
    exp, low = piece["exp"].cpu().numpy(), 1 - n
    alpha, r, u, v = rand_fr(1, 61), rand_fr(1, 62), rand_fr(SHIFT, 63), rand_fr(SHIFT, 64)
    beta = br.fr_pack([n])[0]
    T, B = orc.tlookup_init(low, n, beta, orc.from_i32(exp), r[0])
    xs, ys = x.cpu().numpy(), y.cpu().numpy()
    S = orc.vec2("orc_fr_vec_add", orc.vec_bcast("orc_fr_vec_bcast_mul", orc.from_i32(ys), r[0]), orc.from_i32(xs))
    st, wtr, wsc = orc.tlookup_prove(S, T, B, orc.tlookup_prep(orc.from_i32(xs), low, n), alpha[0], beta, u, v)
    assert st == 0
    table = ops.g1_table_gen(gens[1], 256)
    tr, sc = host.tlookup_mapping_prove(ops.fr_from_i32(x), ops.fr_from_i32(y), n, low, n, exp, alpha, r, u, v, table, 256, 1, 16)
    assert_same(tr, wtr, "transcript")
    assert_same(sc, wsc, "S(v)")


def test_the_choice_is_looked_up(ops, host, gens):
    """no logit is above the chosen one's: the gaps are in a range, and one that is negative is not"""
    rng = np.random.default_rng(61)
    n = 1 << 10
    got = ops.wit_next_token(dev(rng.integers(-300, 300, (4, 256))), dev(rng.integers(0, 256, (4, 20))), dev(np.full(4, 20)), dev(np.full(4, 90000)), dev(np.full(4, 7)), dev(np.full(4, 3)))
    assert ops.wit_status() == 0
    gap = got["gap"].reshape(-1)
    assert torch.equal(got["logits"] + got["gap"], got["max"][:, None].expand(4, 256)) and torch.equal(got["logits"].gather(1, got["token"][:, None].long())[:, 0], got["max"])
    table = ops.g1_table_gen(gens[1], 256)
    u, v, alpha = rand_fr(10, 71), rand_fr(10, 72), rand_fr(1, 73)
    beta = br.fr_pack([n])[0]
    S = orc.from_i32(gap.cpu().numpy())
    T, B = orc.tlookup_init(0, n, beta)
    st, wtr, wsc = orc.tlookup_prove(S, T, B, orc.tlookup_prep(S, 0, n), alpha[0], beta, u, v)
    assert st == 0
    res = host.tlookup_range_prove(ops.fr_from_i32(gap), n, 0, n, alpha, u, v, table, 256, 1, 16)
    assert_same(res["transcript"], wtr, "gap")
    assert_same(res["S_claim"], wsc, "gap")
