"""What the new tokens' attention writes, taken into proofs: the products with keys and values, and the lookups of the exponentials
and remainders, of sequences of different lengths (one of them empty).  Transcripts are compared with the CPU oracle's."""
import numpy as np
import pytest
import torch
import bigref as br
import orc
from gpuutil import assert_same, rand_fr
from test_gpu_host import gens, host  # noqa: F401  (fixtures)
from test_gpu_tokens import dev, gauss, ops, paged  # noqa: F401  (ops is a fixture)

pytestmark = pytest.mark.gpu

SHIFT = 10                                  # a table of 2^10 exponentials
QK = OUT = 1 << 10


@pytest.fixture(scope="module")
def step(ops):
    """an attention call of ragged sequences, with its inputs"""
    rng = np.random.default_rng(50)
    lens, H, HK, D, page = [21, 0, 32, 5], 4, 2, 16, 8
    table, kc, vc = paged(rng, lens, page, HK, D, sigma=180.0)
    exp = np.rint(np.exp((np.arange(1 << SHIFT) - ((1 << SHIFT) - 1)) / 128.0) * 65536).astype(np.int32)
    s = {"lens": dev(np.array(lens)), "q": dev(gauss(rng, (len(lens), H, D), 180.0)), "k": dev(kc), "v": dev(vc), "pages": dev(table), "exp": dev(exp), "page": page, "longest": 32}
    s["out"] = ops.wit_paged_attention(s["q"], s["k"], s["v"], s["pages"], s["lens"], 32, s["exp"], bit_shift=SHIFT, index_bits=SHIFT, qk_scale=QK, out_scale=OUT)
    assert ops.wit_status() == 0
    s["live"] = (torch.arange(32, device="cuda") < s["lens"][:, None])[:, None, :].expand(len(lens), H, 32)
    return s


def padded(x, n, value):
    return torch.cat((x, torch.full((n - x.numel(),), value, dtype=torch.int32, device="cuda")))


def test_the_exponentials_are_looked_up(ops, host, gens, step):
    """the entries of the sequences' positions, filled up with the pair of a score that is the maximum"""
    out, n = step["out"], 1 << SHIFT
    x, y = out["exp_input"][step["live"]], out["exp_output"][step["live"]]
    assert x.numel() == 4 * 58
    x, y = padded(x, n, 0), padded(y, n, int(step["exp"][-1]))
    exp, low = step["exp"].cpu().numpy(), 1 - n
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
    # the rows as they stand hold positions of no sequence, and their pairs of zeros are in no table
    whole, wy = out["exp_input"].reshape(-1)[:n // 2], out["exp_output"].reshape(-1)[:n // 2]
    with pytest.raises(host.HostError, match="tLookup_phase"):
        host.tlookup_mapping_prove(ops.fr_from_i32(padded(whole, n, 0)), ops.fr_from_i32(padded(wy, n, int(exp[-1]))), n, low, n, exp, alpha, r, u, v, table, 256, 1, 16)


def test_the_remainders_are_looked_up(ops, host, gens, step):
    """those of the scores and of the output: zeros, in the range, where there is none"""
    table = ops.g1_table_gen(gens[1], 256)
    for name, low, n in (("scores_rem", -QK // 2, QK), ("qkv_rem", -OUT // 2, OUT)):
        t = step["out"][name].reshape(-1)
        t = padded(t[: min(t.numel(), n)], n, 0)
        u, v, alpha = rand_fr(10, 71), rand_fr(10, 72), rand_fr(1, 73)
        beta = br.fr_pack([n])[0]
        S = orc.from_i32(t.cpu().numpy())
        T, B = orc.tlookup_init(low, n, beta)
        st, wtr, wsc = orc.tlookup_prove(S, T, B, orc.tlookup_prep(S, low, n), alpha[0], beta, u, v)
        assert st == 0
        res = host.tlookup_range_prove(ops.fr_from_i32(t), n, low, n, alpha, u, v, table, 256, 1, 16)
        assert_same(res["transcript"], wtr, name)
        assert_same(res["S_claim"], wsc, name)


def evaluation(host, ops, q, r, scale, u):
    """of q * scale + r, as a proof has it from the two tensors' openings"""
    at = [host.mle_eval(ops.fr_from_i32(t.reshape(-1).contiguous()), t.numel(), u) for t in (q, r)]
    return orc.fr_add(orc.fr_mul(at[0], br.fr_pack([scale])[0]), at[1])


@pytest.mark.parametrize("b", [0, 2, 3])
def test_the_products_are_proved(ops, host, step, b):
    """a sequence's products with its keys and with its values, which stand in pages: cache heads as layers, a cache head's query heads as
    rows, positions filled up with zeros"""
    out, pages, page, n = step["out"], step["pages"], step["page"], int(step["lens"][b])
    H, HK, D = step["q"].shape[1], step["k"].shape[2], step["q"].shape[2]
    each, N = H // HK, 1 << br.log2ceil(n)
    t = torch.arange(n, device="cuda")
    keys, values = (torch.zeros((HK, N, D), dtype=torch.int32, device="cuda") for _ in range(2))
    keys[:, :n], values[:, :n] = (c[pages[b, t // page].long(), t % page].transpose(0, 1) for c in (step["k"], step["v"]))
    rows = {}
    for name in ("scores", "scores_rem", "softmax_output"):
        rows[name] = torch.zeros((H, N), dtype=torch.int32, device="cuda")
        rows[name][:, :n] = out[name][b, :, :n]
    # scores * scale + remainder = queries . keys, and output * scale + remainder = probabilities . values
    for A, B, M, K, q, r, scale in ((step["q"][b], keys, N, D, rows["scores"], rows["scores_rem"], QK),
                                    (rows["softmax_output"], values.transpose(1, 2).contiguous(), D, N, out["qkv"][b], out["qkv_rem"][b], OUT)):
        u, v = rand_fr(br.log2ceil(H * M), 81), rand_fr(br.log2ceil(HK * K), 82)
        claim = evaluation(host, ops, q, r, scale, u)
        Af, Bf = (x.reshape(-1).contiguous() for x in (A, B))
        st, wtr, wclaim, wac, wbc = orc.prove_matmul(orc.from_i32(Af.cpu().numpy()), orc.from_i32(Bf.cpu().numpy()), HK, each, M, K, u, v, claim)
        assert st == 0
        tr, end, ac, bc = host.prove_matmul(ops.fr_from_i32(Af), ops.fr_from_i32(Bf), HK, each, M, K, u, v, claim)
        assert_same(tr, wtr, "transcript")
        assert_same(end, wclaim, "final claim")
        assert_same(ac, wac, "A(v)")
        assert_same(bc, wbc, "B(v)")
        wrong = r.clone()
        wrong[0, 0] += 1
        with pytest.raises(host.HostError, match="matmul_phase"):
            host.prove_matmul(ops.fr_from_i32(Af), ops.fr_from_i32(Bf), HK, each, M, K, u, v, evaluation(host, ops, q, wrong, scale, u))
