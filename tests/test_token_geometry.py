"""CPU checks of what the new tokens' entry points refuse, which positions and pages they touch, and how the Python helpers
check and pack their arguments (the expressions of grape_amd/csrc/token_geometry.hpp, in a host build)."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from grape_amd import ops

HERE = os.path.dirname(os.path.abspath(__file__))
SRC = os.path.join(HERE, "native", "token_geometry_host.cpp")
LIB = os.path.join(HERE, "native", "libtoken_geometry_host.so")
HDRS = (os.path.join(HERE, "..", "grape_amd", "csrc", "token_geometry.hpp"), os.path.join(HERE, "..", "include", "grape_hip.h"))


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(LIB) or any(os.path.getmtime(d) > os.path.getmtime(LIB) for d in (SRC,) + HDRS):
        subprocess.check_call(["g++", "-O1", "-std=c++17", "-Wall", "-fPIC", "-shared", "-o", LIB, SRC])
    l = ctypes.CDLL(LIB)
    p, u, i, q = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_int32, ctypes.c_int64
    for name in ("refuse_append", "refuse_attention", "refuse_q4"):
        getattr(l, name).restype = ctypes.c_char_p
    l.refuse_append.argtypes = l.refuse_attention.argtypes = [p, p]
    l.refuse_q4.argtypes = [p, p, q, p, q, p, u, u, u, u, q, p, ctypes.c_size_t]
    l.q4_workspace.argtypes, l.q4_workspace.restype = [u] * 4, ctypes.c_size_t
    l.struct_bytes.restype = l.workspace.restype = ctypes.c_size_t
    l.overlaps.argtypes = [p]
    l.span.argtypes = [i, i, u, u, u, p]
    l.offset_of.argtypes, l.offset_of.restype = [p, i, u], q
    l.kind.argtypes = [p, q, i, u, u]
    l.workspace.argtypes = [u] * 5
    l.append_fields.argtypes = l.attention_fields.argtypes = l.cache_fields.argtypes = [p, p]
    return l


CACHE = dict(k=16, v=32, pages=10, page=16, heads=4, dim=64, ps=16 * 4 * 64, ts=4 * 64, hs=64)
APPEND = dict(q=16, k=32, v=48, qs=512, ks=256, vs=256, pos=64, slots=80, cos=96, sin=112, qo=128, qr=0, kr=0, n=3, heads=8, rot=64, rows=100, scale=65536,
              inter=0, res=0)
ATTEND = dict(q=16, qs=512, table=32, lens=48, first=0, exp=64, s=0, sr=0, x=0, e=0, p=0, lq=0, mx=0, sm=0, o=80, r=0, ws=96, wb=1 << 30, qk=1 << 22, pr=1 << 16,
              os=1 << 16, n=2, heads=8, max_len=100, ts=10, shift=20, bits=20)


def cache(**kw):
    return ops._CACHE.pack(*{**CACHE, **kw}.values())


def append(**kw):
    return ops._APPEND.pack(*{**APPEND, **kw}.values())


def attend(**kw):
    return ops._ATTEND.pack(*{**ATTEND, **kw}.values())


def test_helpers_pack_the_structs_of_the_header(lib):
    for which, s, fields in ((0, ops._CACHE, lib.cache_fields), (1, ops._APPEND, lib.append_fields), (2, ops._ATTEND, lib.attention_fields)):
        assert lib.struct_bytes(which) == s.size
        n = len(s.unpack(bytes(s.size)))
        values = [i + 1 for i in range(n)]
        out = (ctypes.c_int64 * n)()
        fields(s.pack(*values), out)
        assert list(out) == values


@pytest.mark.parametrize("bad", [dict(k=0), dict(v=0), dict(pages=0), dict(page=0), dict(heads=0), dict(dim=0), dict(pages=1 << 27), dict(heads=65536),
                                 dict(dim=8193), dict(ps=-1), dict(ts=-1), dict(hs=-1), dict(ps=1 << 40), dict(hs=1 << 40)])
def test_bad_caches_are_refused(lib, bad):
    assert lib.refuse_append(append(), cache()) is None and lib.refuse_attention(attend(), cache()) is None
    assert lib.refuse_append(append(), cache(**bad)) and lib.refuse_attention(attend(), cache(**bad))
    assert lib.refuse_append(append(), None) and lib.refuse_attention(attend(), None)
    assert lib.refuse_append(None, cache()) and lib.refuse_attention(None, cache())


@pytest.mark.parametrize("bad", [dict(scale=0), dict(scale=-1), dict(scale=(1 << 31) + 1), dict(rot=63), dict(rot=66), dict(heads=65536), dict(qs=-1), dict(ks=-1),
                                 dict(vs=-1), dict(k=0), dict(v=0), dict(slots=0), dict(q=0), dict(qo=0), dict(pos=0), dict(cos=0), dict(sin=0), dict(rows=0),
                                 dict(n=(1 << 32) - 1)])
def test_bad_appends_are_refused(lib, bad):
    assert lib.refuse_append(append(**bad), cache())


def test_appends_that_are_taken(lib):
    for ok in (dict(heads=0, q=0, qo=0), dict(rot=0, pos=0, cos=0, sin=0, rows=0), dict(n=0, k=0, v=0, slots=0), dict(scale=1), dict(scale=1 << 31), dict(qs=0)):
        assert lib.refuse_append(append(**ok), cache()) is None


@pytest.mark.parametrize("bad", [dict(qk=0), dict(qk=(1 << 31) + 1), dict(pr=0), dict(pr=(1 << 30) + 1), dict(os=0), dict(os=(1 << 31) + 1), dict(shift=0), dict(shift=31),
                                 dict(bits=0), dict(bits=31), dict(heads=0), dict(heads=6), dict(heads=2), dict(heads=65536), dict(qs=-1), dict(n=65536), dict(max_len=1 << 31),
                                 dict(q=0), dict(lens=0), dict(exp=0), dict(o=0), dict(table=0), dict(ws=0, max_len=1000, ts=100), dict(wb=10, max_len=1000, ts=100), dict(ws=100, max_len=1000, ts=100), dict(n=60000, heads=60000)])
def test_bad_attentions_are_refused(lib, bad):
    assert lib.refuse_attention(attend(**bad), cache())


@pytest.mark.parametrize("bad", [dict(scale=0), dict(scale=(1 << 31) + 1), dict(k=0), dict(group=0), dict(k=(1 << 30) + 1), dict(xs=-1), dict(ws=-1), dict(q=0), dict(x=0), dict(w=0),
                                 dict(sc=0), dict(n=65536, sb=1 << 40), dict(m=(1 << 24) + 1), dict(group=(1 << 30) + 1), dict(n=5), dict(n=5, sp=64), dict(n=5, sp=72, sb=1 << 20)])
def test_bad_products_are_refused(lib, bad):
    good = dict(q=16, x=16, xs=64, w=16, ws=32, sc=16, n=2, m=8, k=64, group=32, scale=65536, sp=0, sb=0)
    assert lib.refuse_q4(*good.values()) is None
    assert lib.refuse_q4(*{**good, "n": 0, "q": 0}.values()) is None
    assert lib.refuse_q4(*{**good, "n": 5, "sp": 64, "sb": lib.q4_workspace(5, 8, 64, 32)}.values()) is None
    assert lib.refuse_q4(*{**good, "n": 5, "group": 20}.values()) is None               # no digits without the matrix cores
    assert lib.refuse_q4(*{**good, **bad}.values())


def test_calls_whose_time_grows_with_a_square_are_bounded(lib):
    """a workgroup of the append looks through all later slots, a product with an input above the digits through all of a row"""
    few = cache(heads=1, dim=1, hs=1, ts=1, ps=16)
    one = dict(heads=0, q=0, qo=0, rot=0, pos=0, cos=0, sin=0, rows=0)
    assert lib.refuse_append(append(n=1 << 24, **one), few) is None
    for n in ((1 << 24) + 1, 1 << 31, (1 << 32) - 200, (1 << 32) - 1):
        assert lib.refuse_append(append(n=n, **one), few)
    good = dict(q=16, x=16, xs=1 << 24, w=16, ws=1 << 23, sc=16, n=1, m=8, k=1 << 24, group=32, scale=65536, sp=0, sb=0)
    assert lib.refuse_q4(*good.values()) is None
    assert lib.refuse_q4(*{**good, "k": (1 << 24) + 1}.values()) and lib.q4_workspace(5, 8, (1 << 24) + 1, 32) == 0 < lib.q4_workspace(5, 8, 1 << 24, 32)


def test_overlapping_caches_are_found(lib):
    """against the elements themselves"""
    rng = np.random.default_rng(1)
    seen = set()
    for _ in range(3000):
        n = [int(x) for x in rng.integers(1, 5, 4)]
        st = [int(x) for x in rng.choice([0, 1, 2, 3, 4, 6, 8, 12, 16, 24, 48], 3)]
        at = (np.arange(n[0])[:, None, None, None] * st[0] + np.arange(n[1])[:, None, None] * st[1] + np.arange(n[2])[:, None] * st[2] + np.arange(n[3])).reshape(-1)
        found = bool(lib.overlaps(cache(pages=n[0], page=n[1], heads=n[2], dim=n[3], ps=st[0], ts=st[1], hs=st[2])))
        seen.add(found)
        if len(set(at.tolist())) < len(at):
            assert found, (n, st)                         # never missed
        if found:                                         # and nothing refused that is an ordinary tensor's layout in some order
            order = sorted((s, m) for s, m in zip(st, n) if m > 1)
            reach = n[3]
            ordinary = True
            for s, m in order:
                ordinary = ordinary and s >= reach
                reach = s * m if s >= reach else reach
            assert not ordinary, (n, st)
    assert seen == {False, True}


def test_spans_and_pages(lib):
    out = (ctypes.c_uint32 * 2)()
    for len_, first, max_len, stride, page, ok, want in ((5, 0, 10, 2, 8, 1, (0, 5)), (5, 5, 10, 2, 8, 1, (5, 5)), (5, 9, 10, 2, 8, 1, (5, 5)), (16, 3, 16, 2, 8, 1, (3, 16)),
                                                         (17, 0, 20, 2, 8, 0, (0, 0)), (11, 0, 10, 2, 8, 0, (0, 0)), (-1, 0, 10, 2, 8, 0, (0, 0)), (5, -1, 10, 2, 8, 0, (0, 0)),
                                                         (-(1 << 31), 0, 10, 2, 8, 0, (0, 0)), (0, 0, 0, 0, 8, 1, (0, 0)), (1, 0, 1, 0, 8, 0, (0, 0)),
                                                         ((1 << 31) - 1, 0, (1 << 31) - 1, 1 << 20, 1 << 20, 1, (0, (1 << 31) - 1))):
        assert lib.span(len_, first, max_len, stride, page, out) == ok and tuple(out) == want
    c = cache()
    assert lib.offset_of(c, 9, 15) == 9 * 4096 + 15 * 256
    assert lib.offset_of(c, 10, 0) == lib.offset_of(c, -1, 0) == lib.offset_of(c, (1 << 31) - 1, 3) == lib.offset_of(c, -(1 << 31), 3) == -1
    big = cache(pages=1 << 20, page=1 << 10, ps=1 << 30, ts=1 << 20)
    assert lib.offset_of(big, (1 << 20) - 1, 1023) == ((1 << 20) - 1 << 30) + (1023 << 20)             # offsets pass 32 bits
    for slot, pos, rot, want in ((0, 0, 64, 0), (159, 99, 64, 0), (160, 0, 64, 2), (1 << 62, 0, 64, 2), (-1, 500, 64, 1), (-(1 << 63), 0, 64, 1), (3, 100, 64, 2), (3, -1, 64, 2), (3, -1, 0, 0)):
        assert lib.kind(c, slot, pos, rot, 100) == want


def test_division_by_a_page_size(lib):
    rng = np.random.default_rng(2)
    lib.divided.restype = ctypes.c_uint32
    for d in [1, 2, 3, 5, 7, 16, 17, 100, 255, 256, 257, 1 << 16, (1 << 16) + 1, 1 << 30, (1 << 31) - 1] + [int(x) for x in rng.integers(1, 1 << 31, 200)]:
        for n in [0, 1, d - 1, d, d + 1, 2 * d - 1, 2 * d, (1 << 31) - 1, (1 << 31) // d * d, (1 << 31) // d * d - 1] + [int(x) for x in rng.integers(0, 1 << 31, 50)]:
            if n < 1 << 31:
                assert lib.divided(n, d) == n // d, (n, d)


def test_plans_cover_every_position_within_their_limits(lib):
    rng = np.random.default_rng(3)
    names = "dim64 rows tiles score_chunk score_chunks exp_chunk exp_chunks blocks groups value_chunk value_chunks at_scores at_exp at_max at_sum at_part bytes whole whole_lds".split()
    out = (ctypes.c_uint64 * len(names))()
    sizes = [(1, 32, 8, 128, 37), (1, 1, 1, 8192, 1 << 20), (64, 32, 8, 128, 2048), (1, 64, 1, 64, 131072), (65535, 1, 1, 1, 1), (1, 1, 1, 1, 0), (3, 48, 3, 192, 5000)]
    for _ in range(2000):
        hk = int(rng.integers(1, 20))
        sizes.append((int(2 ** rng.uniform(0, 12)), hk * int(2 ** rng.uniform(0, 6)), hk, int(2 ** rng.uniform(0, 13)), int(2 ** rng.uniform(0, 22))))
    taken = split = 0
    for s, h, hk, d, n in sizes:
        if not lib.plan_of(s, h, hk, d, n, out):
            continue
        taken += 1
        p = dict(zip(names, out))
        assert p["dim64"] * 64 >= d > (p["dim64"] - 1) * 64 and 1 <= p["rows"] <= 16 and p["rows"] * p["tiles"] >= h // hk > p["rows"] * (p["tiles"] - 1)
        assert p["blocks"] * p["groups"] * 32 >= d and p["blocks"] * (p["groups"] - 1) * 32 < d and p["blocks"] in (1, 2, 4)
        for kind, step in (("score", 16 if d > 448 else 64), ("exp", 1024), ("value", 64)):
            assert p[kind + "_chunk"] % step == 0 and p[kind + "_chunk"] * p[kind + "_chunks"] >= n and (p[kind + "_chunks"] == 0 or p[kind + "_chunk"] * (p[kind + "_chunks"] - 1) < n)
        assert p["value_chunk"] <= 1024                                         # what the 32-bit sums of the planes' products hold
        assert p["dim64"] * 64 * 5 * p["rows"] + 8 * p["score_chunk"] * (p["rows"] + 1) <= 61440          # LDS
        assert p["value_chunk"] * (p["rows"] * 4 + 8) <= 61440 and p["rows"] * p["blocks"] * 32 * 8 <= 61440
        assert hk * p["tiles"] * max(p["score_chunks"], p["value_chunks"] * p["groups"]) * 256 < 1 << 31
        rows = s * h
        need = [rows * n * 4, rows * n * 4, rows * p["score_chunks"] * 4, rows * p["exp_chunks"] * 8, rows * p["value_chunks"] * d * 8 if p["value_chunks"] > 1 else 0]
        if p["whole"]:
            assert p["bytes"] == 0 and n <= 256
            assert 73728 >= p["whole_lds"] >= 8 * 256 + 8 * p["rows"] * max(d, 256) + 4 * 256 * p["rows"] + p["rows"] * max(5 * 64 * p["dim64"], 4 * 256)
            assert lib.workspace(s, h, hk, d, n) == p["bytes"]
            continue
        split += 1
        at = [p[x] for x in ("at_scores", "at_exp", "at_max", "at_sum", "at_part", "bytes")]
        assert at[0] == 0 and all(x % 16 == 0 for x in at[:5]) and all(b - a >= k for a, b, k in zip(at, at[1:], need))
        assert lib.workspace(s, h, hk, d, n) == p["bytes"]
    assert taken > 1000 and split > 300


def test_counted_launches_fit_one_axis(lib):
    names = "dim64 rows tiles score_chunk score_chunks exp_chunk exp_chunks blocks groups value_chunk value_chunks".split()
    out = (ctypes.c_uint64 * 19)()
    seen = set()
    for s, h, hk, d, n in ((7, 8, 8, 64, 1000), (8, 8, 8, 64, 1000), (8, 8, 8, 64, 0), (256, 32, 8, 128, 2048), (257, 32, 8, 128, 2048), (256, 65535, 65535, 64, 64), (256, 512, 512, 128, 4096),
                           (8, 65535, 65535, 8, 1000), (250, 16, 1, 8192, 100000), (256, 1, 1, 8192, 1 << 20)):
        counted = lib.counted(s, h, hk, d, n)
        if counted == 1:
            lib.plan_of(s, h, hk, d, n, out)
            p = dict(zip(names, out))
            assert 8 <= s <= 256 and s * hk * p["tiles"] * max(p["score_chunks"], p["value_chunks"] * p["groups"], 1) * 256 < 1 << 31
        seen.add(counted)
    assert seen >= {0, 1} and lib.counted(64, 32, 8, 128, 2048) == 1 and lib.counted(1, 32, 8, 128, 131072) == 0


def test_workspace_sizes(lib):
    assert lib.q4_workspace(1, 1 << 20, 1 << 20, 128) == 0 and lib.q4_workspace(4, 4096, 4096, 128) == 0
    assert lib.q4_workspace(9, 64, 4096, 100) == 0 and lib.q4_workspace(9, 64, 0, 32) == 0 and lib.q4_workspace(9, 0, 64, 32) == 0
    for n, m, k in ((2, 16384, 8192), (4, 11008, 4096), (5, 1, 1), (8, 100, 128), (9, 1, 129), (16, 4096, 11008), (17, 5, 2049), (40, 3, 4095), (65535, 1, 1 << 16)):
        tile, units = 4 if n <= 4 else 8 if n <= 8 else 16, -(-k // 128)
        # a byte an input and plane, whole units and tiles of tokens, and a word a token and 2048 inputs
        assert lib.q4_workspace(n, m, k, 32) == -(-n // tile) * tile * 4 * units * 128 + 4 * n * -(-units // 16)
    assert lib.workspace(0, 8, 8, 64, 100) == 0 and lib.workspace(65536, 8, 8, 64, 100) == 0 and lib.workspace(60000, 60000, 1, 64, 100000) == 0
    assert lib.workspace(1, 8, 2, 64, 1000) >= 4 * 8 * 1000


# ------------------------------------------------------------------ the helpers' own checks


@pytest.fixture
def helpers(monkeypatch):
    """the helpers on host tensors, in front of a library that takes every call"""
    calls = []

    class Library:
        def __getattr__(self, name):
            def call(*args):
                calls.append((name, args))
                return 64 if name.endswith("_workspace") else 0
            return call
    monkeypatch.setattr(ops, "init", lambda *a: Library())
    monkeypatch.setattr(ops, "_place", lambda: -1)          # what get_device() says of host tensors
    monkeypatch.setattr(ops, "_stream", lambda dev: None)
    monkeypatch.setattr(ops, "_i32", lambda *s: torch.empty(s, dtype=torch.int32))
    return calls


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def append_args():
    return dict(q=i32(3, 8, 64), k=i32(3, 4, 64), v=i32(3, 4, 64), positions=i32(3), slots=torch.zeros(3, dtype=torch.int64), cos=i32(100, 32), sin=i32(100, 32),
                k_cache=i32(10, 16, 4, 64), v_cache=i32(10, 16, 4, 64), q_out=i32(3, 8, 64), q_rem=i32(3, 8, 64), k_rem=i32(3, 4, 64))


@pytest.mark.parametrize("bad", [dict(q=i32(3, 512)), dict(q=i32(2, 8, 64)), dict(q=i32(3, 8, 64).float()), dict(q=i32(3, 64, 8).transpose(1, 2)), dict(k=i32(3, 8, 64)),
                                 dict(v=i32(3, 4, 63)), dict(positions=i32(4)), dict(positions=torch.zeros(3, dtype=torch.int64)), dict(slots=i32(3)),
                                 dict(slots=torch.zeros(6, dtype=torch.int64)[::2]), dict(cos=i32(99, 32)), dict(sin=i32(100, 31)), dict(cos=i32(32, 100).t(), sin=i32(32, 100).t()),
                                 dict(k_cache=i32(10, 16, 256)), dict(v_cache=i32(11, 16, 4, 64)), dict(k_cache=i32(10, 16, 64, 4).transpose(2, 3), v_cache=i32(10, 16, 64, 4).transpose(2, 3)),
                                 dict(k_cache=i32(10, 16, 4, 64).long(), v_cache=i32(10, 16, 4, 64).long()), dict(q_out=i32(3, 8, 63)), dict(q_rem=i32(3, 4, 64)), dict(k_rem=i32(3, 8, 64)),
                                 dict(q=None)])
def test_append_helper_refuses(helpers, bad):
    ops.wit_rope_append(**append_args())
    with pytest.raises(ValueError):
        ops.wit_rope_append(**{**append_args(), **bad})
    assert len(helpers) == 1


def test_helpers_refuse_tensors_of_another_device(helpers, monkeypatch):
    monkeypatch.setattr(ops, "_place", lambda: 0)
    for call, args in ((ops.wit_rope_append, append_args()), (ops.wit_paged_attention, attend_args()),
                       (ops.wit_matvec_q4, dict(x=i32(2, 64), w=torch.zeros((8, 32), dtype=torch.uint8), scales=i32(8, 2), group=32))):
        with pytest.raises(ValueError):
            call(**args)
    assert not helpers


def attend_args():
    return dict(q=i32(2, 8, 64), k_cache=i32(10, 16, 4, 64), v_cache=i32(10, 16, 4, 64), block_table=i32(2, 5), lens=i32(2), max_len=70, exp_table=i32(1 << 20))


@pytest.mark.parametrize("bad", [dict(q=i32(2, 512)), dict(q=i32(2, 8, 60)), dict(block_table=i32(3, 5)), dict(block_table=i32(2, 10)[:, :5]), dict(block_table=i32(10)), dict(lens=i32(3)),
                                 dict(first=i32(3)), dict(first=torch.zeros(2)), dict(exp_table=i32(1000)), dict(index_bits=19), dict(max_len=-1), dict(out={}), dict(out={"max": i32(2, 8)}),
                                 dict(out={"qkv": i32(2, 8, 64), "score": i32(2, 8, 70)}), dict(out={"qkv": i32(2, 8, 64), "scores": i32(2, 8, 71)}), dict(out={"qkv": i32(2, 8, 64, 1)}),
                                 dict(workspace=i32(1000)), dict(v_cache=i32(10, 16, 64, 4).transpose(2, 3))])
def test_attention_helper_refuses(helpers, bad):
    got = ops.wit_paged_attention(**attend_args())
    assert got["scores"].shape == (2, 8, 70) and got["qkv"].shape == (2, 8, 64)
    n = len(helpers)
    with pytest.raises(ValueError):
        ops.wit_paged_attention(**{**attend_args(), **bad})
    assert not [c for c in helpers[n:] if not c[0].endswith("_workspace")]


@pytest.mark.parametrize("bad", [dict(x=i32(64)), dict(x=i32(2, 64).long()), dict(x=i32(64, 2).t()), dict(w=i32(8, 32)), dict(w=torch.zeros((8, 33), dtype=torch.uint8)), dict(scales=i32(8, 3)),
                                 dict(scales=i32(2, 8).t()), dict(zeros=i32(8, 2)), dict(group=0), dict(q=i32(2, 9)), dict(r=i32(3, 8)), dict(x=i32(2, 0), w=torch.zeros((8, 0), dtype=torch.uint8))])
def test_q4_helper_refuses(helpers, bad):
    good = dict(x=i32(2, 64), w=torch.zeros((8, 32), dtype=torch.uint8), scales=i32(8, 2), group=32)
    assert ops.wit_matvec_q4(**good)[0].shape == (2, 8)
    n = len(helpers)
    with pytest.raises(ValueError):
        ops.wit_matvec_q4(**{**good, **bad})
    assert not [c for c in helpers[n:] if not c[0].endswith("_workspace")]


def test_helpers_hand_over_strides(helpers):
    fused = i32(3, 16 * 64 + 4)
    q, k, v = (fused[:, a * 64:b * 64].view(3, -1, 64) for a, b in ((0, 8), (8, 12), (12, 16)))
    kc = i32(4, 10, 16, 70).permute(1, 2, 0, 3)[..., :64]
    ops.wit_rope_append(**{**append_args(), "q": q, "k": k, "v": v, "k_cache": kc, "v_cache": kc})
    args, c = helpers[0][1][:2]
    assert ops._APPEND.unpack(args)[3:6] == (fused.stride(0),) * 3 and ops._CACHE.unpack(c)[2:] == (10, 16, 4, 64, 16 * 70, 70, 160 * 70)
    x = i32(1, 64).expand(4, 64)
    ops.wit_matvec_q4(x, torch.zeros((8, 40), dtype=torch.uint8)[:, 3:35], i32(8, 2), 32)
    args = [c[1] for c in helpers if c[0] == "grape_wit_matvec_q4"][0]
    assert args[3] == 0 and args[5] == 40


@pytest.mark.parametrize("call, args, bad", [
    (ops.wit_rope_append, append_args, dict(scale=1 << 63)), (ops.wit_rope_append, append_args, dict(scale=0.5)),
    (ops.wit_paged_attention, attend_args, dict(max_len=1 << 32)), (ops.wit_paged_attention, attend_args, dict(qk_scale=1 << 64)),
    (ops.wit_paged_attention, attend_args, dict(bit_shift=-1)), (ops.wit_paged_attention, attend_args, dict(bit_shift=1 << 32)),
    (ops.wit_matvec_q4, lambda: dict(x=i32(2, 64), w=torch.zeros((8, 32), dtype=torch.uint8), scales=i32(8, 1), group=1 << 20), dict(group=(1 << 32) + 32)),
    (ops.wit_matvec_q4, lambda: dict(x=i32(2, 64), w=torch.zeros((8, 32), dtype=torch.uint8), scales=i32(8, 1), group=1 << 20), dict(scale=(1 << 64) + 65536)),
    (ops.wit_matvec_q4, lambda: dict(x=i32(2, 64), w=torch.zeros((8, 32), dtype=torch.uint8), scales=i32(8, 1), group=1 << 20), dict(x=i32(1, 64).expand((1 << 32) + 2, 64)))])
def test_numbers_that_the_call_would_cut_off_are_refused(helpers, call, args, bad):
    call(**args())
    n = len(helpers)
    with pytest.raises(ValueError):
        call(**{**args(), **bad})
    assert not [c for c in helpers[n:] if not c[0].endswith("_workspace")]


def test_no_workspace_for_sizes_beyond_the_abi(helpers):
    assert ops.wit_matvec_q4_workspace(2, (1 << 32) + 8, 64, 32) == 0 and ops.wit_paged_attention_workspace(1, 8, 8, 64, 1 << 32) == 0
    assert not helpers
