"""CPU checks of the calls around a step of new tokens: what they refuse, which pages a sequence takes and gives back, what tokens
see and how that is cut into tiles, what the plans cover, and how the Python helpers check and pack their arguments (the expressions of
grape_amd/csrc/step_geometry.hpp, in a host build)."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from grape_amd import ops
from test_token_geometry import cache, helpers, i32  # noqa: F401  (helpers is a fixture)

HERE = os.path.dirname(os.path.abspath(__file__))
SRC = os.path.join(HERE, "native", "step_geometry_host.cpp")
LIB = os.path.join(HERE, "native", "libstep_geometry_host.so")
HDRS = tuple(os.path.join(HERE, "..", *x) for x in (("grape_amd", "csrc", "token_geometry.hpp"), ("grape_amd", "csrc", "step_geometry.hpp"), ("include", "grape_hip.h")))
LARGE = 1 << 31


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(LIB) or any(os.path.getmtime(d) > os.path.getmtime(LIB) for d in (SRC,) + HDRS):
        subprocess.check_call(["g++", "-O1", "-std=c++17", "-Wall", "-fPIC", "-shared", "-o", LIB, SRC])
    l = ctypes.CDLL(LIB)
    p, u, i, q, z = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_int32, ctypes.c_uint64, ctypes.c_size_t
    for name, args, res in (("refuse_pages", [p], ctypes.c_char_p), ("refuse_window", [p, p], ctypes.c_char_p), ("refuse_next", [p], ctypes.c_char_p), ("struct_bytes", [ctypes.c_int], z),
                            ("window_workspace", [u] * 9, z), ("next_workspace", [u] * 2, z), ("next_of", [u, u, p], None), ("sequence", [i, i, q, u, u, u, p, u], ctypes.c_int),
                            ("new_tokens", [i, i, i, u, u, u, q, p], ctypes.c_int), ("sees", [u] * 4, ctypes.c_int), ("seen_tiles", [u] * 6 + [p] * 3, u), ("any", [u] * 5, ctypes.c_int),
                            ("window_of", [u] * 9 + [p], ctypes.c_int), ("tile_owners", [p, u, u, u, u, p], None), ("pages_fields", [p, p], None), ("window_fields", [p, p], None), ("next_fields", [p, p], None)):
        getattr(l, name).argtypes, getattr(l, name).restype = args, res
    return l


def test_helpers_pack_the_structs_of_the_header(lib):
    for which, s, fields in ((0, ops._PAGES, lib.pages_fields), (1, ops._WINDOW, lib.window_fields), (2, ops._NEXT, lib.next_fields)):
        assert lib.struct_bytes(which) == s.size
        n = len(s.unpack(bytes(s.size)))
        values = [i + 1 for i in range(n)]
        out = (ctypes.c_int64 * n)()
        fields(s.pack(*values), out)
        assert list(out) == values


# ------------------------------------------------------------------ pages and slots
PAGES = dict(lens=0x1000, new=0x2000, span=0x3000, table=0x10000, free=0x20000, starts=0x30000, pos=0x40000, slots=0x50000, lo=0x60000, so=0x70000, n=8, width=20, ring=100,
             rows=64, page=16, window=0, sinks=0, res=0)


def pages(**kw):
    return ops._PAGES.pack(*{**PAGES, **kw}.values())


@pytest.mark.parametrize("bad", [dict(n=4097), dict(page=0), dict(page=1 << 30), dict(width=1 << 28), dict(n=4096, width=1 << 20, page=1), dict(rows=LARGE), dict(ring=LARGE), dict(window=LARGE),
                                 dict(window=5, sinks=LARGE), dict(sinks=1), dict(span=0), dict(so=0), dict(starts=0), dict(lens=0), dict(new=0), dict(lo=0), dict(table=0), dict(free=0),
                                 dict(pos=0), dict(slots=0)])
def test_bad_page_steps_are_refused(lib, bad):
    assert lib.refuse_pages(pages()) is None and lib.refuse_pages(None)
    assert lib.refuse_pages(pages(**bad))


def test_page_steps_that_are_taken(lib):
    for ok in (dict(n=0, lens=0, new=0, lo=0, table=0), dict(width=0, table=0), dict(ring=0, free=0), dict(rows=0, pos=0, slots=0), dict(window=1, sinks=LARGE - 1), dict(window=LARGE - 1),
               dict(n=4096, lens=0x100000, new=0x200000, starts=0x300000, lo=0x400000, table=0x1000000)):
        assert lib.refuse_pages(pages(**ok)) is None, ok


def test_page_steps_in_place_are_refused(lib):
    """every workgroup reads the lengths, the new tokens and the ring's span, whatever another has written by then"""
    size = dict(lens=32, new=32, span=8, table=4 * 8 * 20, free=400, starts=36, pos=256, slots=512, lo=32, so=8)
    outputs = ("table", "free", "starts", "pos", "slots", "lo", "so")
    for a in size:
        for b in outputs:
            if a != b:
                assert lib.refuse_pages(pages(**{b: PAGES[a]})), (a, b)
                assert lib.refuse_pages(pages(**{b: PAGES[a] + size[a] - 4})) and lib.refuse_pages(pages(**{b: PAGES[a] - size[b] + 4})), (a, b)
                assert lib.refuse_pages(pages(**{b: PAGES[a] + size[a]})) is None and lib.refuse_pages(pages(**{b: PAGES[a] - size[b]})) is None, (a, b)


def test_pages_that_sequences_take_and_give_back(lib):
    """against the tokens themselves: a page is held from its first token on until no later token sees one of its own"""
    rng = np.random.default_rng(1)
    out = (ctypes.c_uint32 * 404)()
    for _ in range(4000):
        page = int(rng.choice([1, 2, 3, 5, 16, 17]))
        window, n, new = int(rng.choice([0, 0, 1, 2, 7, 16, 30, 200])), int(rng.integers(0, 150)), int(rng.integers(-1, 40))
        sinks = int(rng.choice([0, 1, 5, 16, 33, 500])) if window else 0
        most = int(rng.choice([n + max(new, 0), 400]))
        assert lib.sequence(n, new, most, page, window, sinks, out, 400) == 1
        tokens, after = max(new, 0), n + max(new, 0)
        held, taken = -(-n // page), -(-after // page) - -(-n // page)

        def gone(i, length):                               # no token from position `length` on sees page i, which has been full or held
            return window > 0 and i * page >= sinks and (i + 1) * page - 1 <= length - window
        before = {i for i in range(held + taken) if gone(i, n)}
        back = {i for i in range(held) if i not in before} if new == -1 else {i for i in range(held + taken) if gone(i, after)} - before
        assert list(out[:3]) == [tokens, held, taken]
        got = list(out[4:4 + out[3]])
        assert len(got) == len(set(got)) and set(got) == back, (page, window, sinks, n, new)
        assert lib.sequence(n, new, after - 1 if after else 0, page, window, sinks, out, 400) == (1 if after == 0 else 0)
    for n, new in ((-1, 1), (-LARGE, 0), (5, -2), (5, -LARGE), (LARGE - 1, 1), (LARGE - 1, LARGE - 1), (1, LARGE - 1)):
        assert lib.sequence(n, new, LARGE - 1, 16, 5, 0, out, 400) == 0 and list(out[:4]) == [0, 0, 0, 0]


# ------------------------------------------------------------------ attention
WINDOW = dict(q=16, qs=512, table=32, starts=40, lens=48, exp=64, s=0, sr=0, x=0, e=0, p=0, lq=0, mx=0, sm=0, o=80, r=0, ws=96, wb=1 << 30, qk=1 << 22, pr=1 << 16, os=1 << 16,
              rows=9, n=2, heads=8, new=5, max_len=100, ts=10, window=0, sinks=0, shift=20, bits=20)


def window(**kw):
    return ops._WINDOW.pack(*{**WINDOW, **kw}.values())


@pytest.mark.parametrize("bad", [dict(qk=0), dict(qk=LARGE + 1), dict(pr=0), dict(pr=(1 << 30) + 1), dict(os=0), dict(os=LARGE + 1), dict(shift=0), dict(shift=31), dict(bits=0), dict(bits=31),
                                 dict(heads=0), dict(heads=6), dict(heads=2), dict(heads=65536), dict(qs=-1), dict(n=65536), dict(max_len=LARGE), dict(max_len=4), dict(new=101), dict(q=0),
                                 dict(starts=0), dict(lens=0), dict(exp=0), dict(o=0), dict(table=0), dict(ws=0), dict(wb=10), dict(ws=100), dict(window=LARGE), dict(window=3, sinks=LARGE),
                                 dict(sinks=1), dict(rows=(1 << 24) + 1), dict(rows=1 << 24, heads=1 << 14, max_len=1 << 20), dict(new=1, rows=1 << 24, heads=1 << 14, max_len=1 << 20, ws=0),
                                 dict(new=1, max_len=1000, ws=0), dict(new=1, max_len=1000, wb=10), dict(new=1, max_len=1000, ws=100)])
def test_bad_attentions_are_refused(lib, bad):
    assert lib.refuse_window(window(), cache()) is None and lib.refuse_window(window(new=1), cache()) is None
    assert lib.refuse_window(None, cache()) and lib.refuse_window(window(), None) and lib.refuse_window(window(), cache(k=0)) and lib.refuse_window(window(), cache(dim=8193))
    assert lib.refuse_window(window(**bad), cache())


def test_attentions_that_are_taken(lib):
    nothing = dict(q=0, starts=0, lens=0, exp=0, table=0, o=0, ws=0, wb=0)
    for ok in (dict(n=0, **nothing), dict(rows=0, **nothing), dict(new=0, **nothing), dict(new=0, max_len=0, **nothing), dict(qs=0), dict(window=1), dict(window=LARGE - 1, sinks=LARGE - 1),
               dict(new=100), dict(rows=1, n=5), dict(qk=1, pr=1, os=1), dict(qk=LARGE, pr=1 << 30, os=LARGE, bits=1, shift=30)):
        assert lib.refuse_window(window(**ok), cache()) is None, ok


def test_new_tokens_of_a_sequence(lib):
    out = (ctypes.c_uint32 * 2)()
    for s, e, n, rows, new, longest, most, ok, want in ((0, 5, 9, 9, 5, 100, 160, 1, (5, 4)), (4, 9, 5, 9, 5, 100, 160, 1, (5, 0)), (3, 3, 0, 9, 5, 100, 160, 1, (0, 0)), (3, 3, 50, 9, 5, 100, 160, 1, (0, 50)),
                                                        (0, 6, 9, 9, 5, 100, 160, 0, (0, 0)), (5, 10, 9, 9, 5, 100, 160, 0, (0, 0)), (-1, 3, 9, 9, 5, 100, 160, 0, (0, 0)), (5, 4, 9, 9, 5, 100, 160, 0, (0, 0)),
                                                        (0, 5, 4, 9, 5, 100, 160, 0, (0, 0)), (0, 5, 101, 9, 5, 100, 160, 0, (0, 0)), (0, 5, 81, 9, 5, 100, 80, 0, (0, 0)), (0, 5, -1, 9, 5, 100, 160, 0, (0, 0)),
                                                        (-LARGE, LARGE - 1, 9, 9, 5, 100, 160, 0, (0, 0)), (LARGE - 1, -LARGE, 9, 9, 5, 100, 160, 0, (0, 0)), (0, 1, -LARGE, 9, 5, 100, 160, 0, (0, 0)),
                                                        (0, 1, LARGE - 1, 9, 5, LARGE - 1, LARGE - 1, 1, (1, LARGE - 2))):
        assert lib.new_tokens(s, e, n, rows, new, longest, most, out) == ok and tuple(out) == want, (s, e, n)


def test_what_tokens_see_in_tiles(lib):
    """every position that a token sees stands in one of its tile of rows' tiles, once, and a tile that is called full is seen by all"""
    rng = np.random.default_rng(2)
    tiles, numbers, full = (ctypes.c_uint32 * 200)(), (ctypes.c_uint32 * 200)(), (ctypes.c_uint32 * 2)()
    everything = (ctypes.c_uint32 * 200)()
    for _ in range(1500):
        pos0 = int(rng.integers(0, 1500))
        pos1 = pos0 + int(rng.integers(0, 32))
        w, v0, n = int(rng.choice([0, 1, 2, 31, 63, 64, 65, 128, 500, 3000])), int(rng.integers(0, 10)), int(rng.integers(1, 40))
        sinks = int(rng.choice([0, 1, 4, 63, 64, 65, 200, 5000])) if w else 0
        count = lib.seen_tiles(pos0, pos1, w, sinks, v0, n, tiles, numbers, full)
        listed = list(tiles[:count])
        assert len(set(listed)) == count and sorted(listed) == listed and list(numbers[:count]) == list(range(count))
        t = np.arange(pos1 + 70)
        seen = np.array([[bool(lib.sees(p, int(x), w, sinks)) for x in t] for p in (pos0, (pos0 + pos1) // 2, pos1)])
        for p, row in zip((pos0, (pos0 + pos1) // 2, pos1), seen):
            assert np.array_equal(row, (t <= p) & ((w == 0) | (t > p - w) | (t < sinks)))
        for x in t[seen.any(0)]:
            assert x // 64 in listed and lib.any(pos0, pos1, w, sinks, int(x))
        assert lib.any(pos0, pos1, w, sinks, pos1) and not lib.any(pos0, pos1, w, sinks, pos1 + 1) and listed[-1] == pos1 // 64
        assert 0 <= full[0] <= full[1] <= n
        for v in range(full[0], min(full[1], max(count - v0, 0))):
            assert seen[:, 64 * listed[v0 + v]:64 * listed[v0 + v] + 64].all()
        assert v0 + full[1] <= count or full[0] == full[1]
        # the tiles of a sequence's rows, all of them, contain those of some of its rows
        first, last = max(0, pos0 - int(rng.integers(0, 400))), pos1 + int(rng.integers(0, 400))
        of_all = list(everything[:lib.seen_tiles(first, last, w, sinks, 0, 1, everything, numbers, full)])
        assert set(listed) <= set(of_all)


NAMES = ("each dim64 tiles cols score_cols score_chunks exp_cols exp_chunks value_cols value_chunks groups packed steps all_cols splits at_scores at_exp at_max at_sum at_factors at_part "
         "at_keys at_values at_queries at_over at_query_over bytes").split()


def plan_of(lib, *sizes):
    out = (ctypes.c_uint64 * len(NAMES))()
    return dict(zip(NAMES, out)) if lib.window_of(*sizes, out) else None


def test_plans_cover_what_is_seen_within_their_limits(lib):
    rng = np.random.default_rng(3)
    sizes = [(2048, 1, 32, 8, 128, 2048, 2048, 0, 0), (2048, 1, 1, 1, 4096, 2048, 2048, 0, 0), (40, 8, 32, 8, 128, 5, 3000, 0, 0), (4500, 3, 12, 4, 80, 1500, 7777, 1024, 4),
             (1 << 20, 1, 1, 1, 64, 1 << 17, 1 << 17, 100, 0), (1 << 16, 1, 8, 1, 8192, 4096, 4096, 0, 0), (2, 2, 1, 1, 1, 2, 2, 0, 0)]
    for _ in range(3000):
        hk, longest = int(2 ** rng.uniform(0, 5)), int(2 ** rng.uniform(1, 18))
        w = int(rng.choice([0, 0, 1, 2 ** rng.uniform(0, 18)]))
        sizes.append((int(2 ** rng.uniform(0, 16)), int(2 ** rng.uniform(0, 12)), hk * int(2 ** rng.uniform(0, 5)), hk, int(2 ** rng.uniform(0, 13)), int(rng.integers(2, longest + 1)), longest,
                      w, int(rng.choice([0, 1, 5, 2 ** rng.uniform(0, 18)])) if w else 0))
    taken = packed = 0
    out, tiles, numbers = (ctypes.c_uint32 * 2)(), (ctypes.c_uint32 * 9000)(), (ctypes.c_uint32 * 9000)()
    for size in sizes:
        rows, seqs, h, hk, d, most, n, w, s = size
        p = plan_of(lib, *size)
        assert lib.window_workspace(*size) == (p["bytes"] if p else 0)
        if not p:
            continue
        taken += 1
        assert p["each"] * hk == h and p["dim64"] * 64 >= d > (p["dim64"] - 1) * 64 and p["groups"] * 128 >= d > (p["groups"] - 1) * 128
        for kind in ("score", "exp", "value"):
            assert p[kind + "_cols"] * p[kind + "_chunks"] >= p["cols"] > p[kind + "_cols"] * (p[kind + "_chunks"] - 1) and p[kind + "_chunks"] <= 65535
        assert p["value_chunks"] * p["groups"] <= 65535 and p["tiles"] * hk < 1 << 22 and p["tiles"] >= rows * p["each"] // 32 + seqs
        assert min(p["dim64"], 8) * 12 * 32 * 16 + p["score_cols"] * 64 * 8 <= 65536          # LDS
        assert 4 * 2 ** 14 * 64 * p["value_cols"] < 1 << 31                                   # what the 32-bit sums of the planes' products hold
        # whatever 32 rows see, and a sequence's all, has its place
        for pos0 in {0, max(0, n - 32), max(0, n // 2), max(0, min(n - 32, w))}:
            pos1 = min(pos0 + 31, n - 1)
            assert lib.seen_tiles(pos0, pos1, w, s, 0, 1, tiles, numbers, out) <= p["cols"]
            pos1 = min(pos0 + most, n) - 1
            if pos1 >= pos0:
                assert lib.seen_tiles(pos0, pos1, w, s, 0, 1, tiles, numbers, out) <= p["all_cols"]
        rows_all = rows * h
        need = [rows_all * p["cols"] * 64 * 4] * 2 + [rows_all * p["score_chunks"] * 4, rows_all * 8, 2 * 1024 * 8 + 64 * 4, rows_all * p["value_chunks"] * d * 8 if p["value_chunks"] > 1 else 0]
        if p["packed"]:
            packed += 1
            cache_tiles = seqs * p["all_cols"] * hk
            need += [cache_tiles * p["steps"] * 3 * 64 * 64, cache_tiles * p["dim64"] * 3 * 64 * 64, p["tiles"] * hk * p["steps"] * 3 * 32 * 64, cache_tiles * p["splits"] * 4, p["tiles"] * hk * p["splits"] * 4]
            assert sum(need[6:9]) <= 1 << 32 and (cache_tiles + p["tiles"] * hk) * p["splits"] < 1 << 22
            assert p["steps"] in (p["dim64"], p["dim64"] + 1) and (p["steps"] == 1 or p["steps"] % 2 == 0) and p["splits"] * 4 >= p["steps"]
            assert rows * p["each"] >= 256 * seqs and rows_all * p["cols"] * 64 * d >= 1 << 30
        else:
            need += [0] * 5
        at = [p[x] for x in NAMES[15:]]
        assert at[0] == 0 and all(x % 16 == 0 for x in at[:-1]) and all(b - a >= k for a, b, k in zip(at, at[1:], need)), size
    assert taken > 1500 and packed > 50


def test_launches_of_workgroups_without_work_are_bounded(lib):
    """many sequences, each of which might be long, and few rows: what is launched is not what is there"""
    assert plan_of(lib, 2, 60000, 64, 64, 64, 2, 65000 * 16 * 64, 0, 0) is None and plan_of(lib, 2, 60000, 64, 64, 64, 2, 131072, 0, 0) is None
    assert plan_of(lib, 2, 2, 64, 64, 64, 2, 65000 * 16 * 64, 0, 0) and plan_of(lib, 16384, 4096, 64, 8, 128, 4, 131072, 0, 0) and plan_of(lib, 1 << 20, 1, 1, 1, 64, 1 << 17, 1 << 17, 100, 0)
    rng = np.random.default_rng(5)
    for _ in range(2000):
        hk, n = int(2 ** rng.uniform(0, 8)), int(2 ** rng.uniform(1, 30))
        size = (int(2 ** rng.uniform(0, 16)), int(2 ** rng.uniform(0, 16)), hk, hk, int(2 ** rng.uniform(0, 13)), 2, n, 0, 0)
        p = plan_of(lib, *size)
        assert p is None or p["tiles"] * hk * max(p["score_chunks"], p["exp_chunks"], p["value_chunks"] * p["groups"]) < 1 << 27


def test_launches_that_join_are_bounded(lib):
    """a workgroup for 64 elements of four rows of every tile, of sequences without rows too"""
    assert plan_of(lib, 2, 65535, 8, 8, 8192, 2, 40000, 0, 0) is None
    assert plan_of(lib, 2, 16383 - 1, 8, 8, 8192, 2, 40000, 0, 0)["value_chunks"] == 2 and plan_of(lib, 2, 16384, 8, 8, 8192, 2, 40000, 0, 0) is None
    assert plan_of(lib, 2, 65535, 8, 8, 8192, 2, 30000, 0, 0)["value_chunks"] == 1          # nothing is joined
    rng = np.random.default_rng(8)
    joined = 0
    for _ in range(4000):
        hk, n, seqs = int(2 ** rng.uniform(0, 8)), int(2 ** rng.uniform(10, 20)), int(2 ** rng.uniform(0, 16))
        rows = int(rng.choice([seqs, 1 + seqs // 4, 2 ** rng.uniform(0, 10)]))
        size = (rows, seqs, hk, hk, int(2 ** rng.uniform(0, 13)), 2, n, 0, 0)
        p = plan_of(lib, *size)
        if p and p["value_chunks"] > 1:
            joined += 1
            assert p["tiles"] * hk * p["dim64"] * 8 < 1 << 27, size
    assert joined > 500


def test_tiles_of_rows_are_owned_by_one_sequence(lib):
    """numbered from starts[b] * each / 32 + b on: no number twice, none beyond the plan's"""
    rng = np.random.default_rng(4)
    for _ in range(500):
        each, seqs = int(rng.integers(1, 70)), int(rng.integers(1, 40))
        new = rng.integers(0, int(rng.choice([2, 40, 300])), seqs)
        starts = np.concatenate(([0], np.cumsum(new))) + int(rng.integers(0, 5))
        rows = int(starts[-1]) + int(rng.integers(0, 3))
        p = plan_of(lib, max(rows, 1), seqs, each, 1, 64, 300, 300, 0, 0)
        numbers = [int(starts[b]) * each // 32 + b + i for b in range(seqs) for i in range(-(-int(new[b]) * each // 32))]
        assert len(set(numbers)) == len(numbers) and max(numbers, default=0) < p["tiles"]


def owners_of(lib, starts, rows, each):
    """the sequence that each tile of rows is given to, and of those whose rows are some the one that it should be"""
    starts = np.asarray(starts, dtype=np.int32)
    seqs = len(starts) - 1
    tiles = rows * each // 32 + seqs
    got = np.zeros(tiles, dtype=np.uint32)
    lib.tile_owners(starts.ctypes.data, seqs, rows, each, tiles, got.ctypes.data)
    want = np.full(tiles, -1, dtype=np.int64)
    for b, (s, e) in enumerate(zip(starts.tolist(), starts[1:].tolist())):
        if 0 <= s <= e <= rows:
            want[s * each // 32 + b:s * each // 32 + b + -(-(e - s) * each // 32)] = b
    return got, want


def test_tiles_of_rows_find_their_sequence_beside_entries_that_are_no_rows(lib):
    """an entry of the starts that is no row of the call takes the two sequences that it bounds with it, and no other"""
    got, want = owners_of(lib, [0, 128, -1, 160], 160, 1)
    assert got[:4].tolist() == [0] * 4 and want[:4].tolist() == [0] * 4
    rng = np.random.default_rng(7)
    for _ in range(400):
        each, seqs = int(rng.integers(1, 40)), int(2 ** rng.uniform(0, 9))
        if rng.random() < 0.05:
            seqs = int(rng.integers(4000, 9000))
        starts = np.concatenate(([0], np.cumsum(rng.integers(0, int(rng.choice([2, 3, 30])), seqs)))) + int(rng.integers(0, 5))
        rows = int(starts[-1]) + int(rng.integers(0, 3))
        at = rng.random(seqs + 1) < rng.choice([0, 0.01, 0.1, 0.7])
        starts[at] = rng.choice([-1, -LARGE, LARGE - 1, rows + 1], int(at.sum()))
        if rng.random() < 0.3:                             # entries behind the last sequence that are not made
            starts[int(rng.integers(0, seqs + 1)):] = -1
        got, want = owners_of(lib, starts, rows, each)
        assert (got < seqs).all() and np.array_equal(got[want >= 0], want[want >= 0])


def test_workspace_of_refused_sizes(lib):
    good = (100, 2, 8, 2, 64, 50, 200, 0, 0)
    assert lib.window_workspace(*good) > 0 and lib.window_workspace(*good[:5], 1, *good[6:]) >= 0
    for i, x in ((0, 0), (0, (1 << 24) + 1), (1, 0), (1, 65536), (2, 0), (2, 65536), (2, 7), (3, 0), (3, 3), (4, 0), (4, 8193), (5, 0), (5, 201), (6, LARGE), (7, LARGE), (8, LARGE)):
        assert lib.window_workspace(*good[:i], x, *good[i + 1:]) == 0, (i, x)


def test_workspace_of_single_tokens_is_of_what_they_see(lib):
    """behind a window a row of scores is as long as the window and the sinks, whatever the sequences' lengths are"""
    rng = np.random.default_rng(6)
    for _ in range(2000):
        seqs, hk, longest, w = int(2 ** rng.uniform(0, 11)), int(2 ** rng.uniform(0, 4)), int(2 ** rng.uniform(0, 20)), int(2 ** rng.uniform(0, 14))
        sinks, h, d = int(rng.choice([0, 1, 4, 300])), hk * int(2 ** rng.uniform(0, 4)), int(2 ** rng.uniform(0, 9))
        got = lib.window_workspace(seqs, seqs, h, hk, d, 1, longest, w, sinks)
        assert got == lib.window_workspace(seqs, seqs, h, hk, d, 1, min(longest, w + sinks), 0, 0)
    size = (24, 24, 32, 8, 128, 1, 131072)
    row = 24 * 32 * 1028 * 4
    assert 2 * row < lib.window_workspace(*size, 1024, 4) < 4 * row and lib.window_workspace(*size, 0, 0) > 24 * 32 * 131072 * 8
    # a call that fits is not refused for the positions that nobody sees: 65535 sequences that may have 2^20
    assert lib.window_workspace(65535, 65535, 32, 8, 128, 1, 1 << 20, 1024, 4) > 0
    assert lib.refuse_window(window(n=65535, rows=65535, heads=32, new=1, max_len=1 << 20, window=1024, sinks=4, wb=1 << 50), cache(heads=8, dim=128)) is None


# ------------------------------------------------------------------ the next token
NEXT = dict(x=0x100000, h=0x200000, hl=0x300000, rep=0, pre=0, fre=0, b=0x400000, m=0x500000, o=0x600000, r=0x700000, c=0x800000, g=0x900000, t=0xa00000, mx=0xb00000, ws=0xc00000,
            wb=1 << 20, xs=1000, hs=50, bs=0, ms=0, scale=1 << 16, n=4, vocab=1000, history=50, res=0)


def following(**kw):
    return ops._NEXT.pack(*{**NEXT, **kw}.values())


@pytest.mark.parametrize("bad", [dict(n=65536), dict(vocab=0), dict(vocab=(1 << 24) + 1), dict(scale=0), dict(scale=-1), dict(scale=LARGE + 1), dict(history=LARGE), dict(history=(1 << 24) + 1), dict(xs=-1), dict(hs=-1), dict(bs=-1),
                                 dict(ms=-1), dict(xs=1 << 40), dict(hs=1 << 40), dict(bs=1 << 40), dict(ms=1 << 40), dict(x=0), dict(t=0), dict(h=0), dict(hl=0), dict(ws=0), dict(wb=10), dict(ws=0xc00008)])
def test_bad_choices_are_refused(lib, bad):
    assert lib.refuse_next(following()) is None and lib.refuse_next(None)
    assert lib.refuse_next(following(**bad))


def test_choices_that_are_taken(lib):
    for ok in (dict(n=0, x=0, t=0, ws=0, wb=0, h=0, hl=0), dict(history=0, h=0, hl=0), dict(b=0), dict(m=0), dict(o=0, r=0, c=0, g=0, mx=0), dict(scale=1), dict(scale=LARGE), dict(xs=0), dict(xs=5000),
               dict(o=0x100000), dict(o=0x100000, n=1, xs=7), dict(history=1 << 24)):
        assert lib.refuse_next(following(**ok)) is None, ok


def test_choices_whose_outputs_overlap_are_refused(lib):
    outs = dict(o=16000, r=16000, c=16000, g=16000, t=16, mx=16, ws=lib.next_workspace(4, 1000))
    for a in list(outs) + ["x", "b"]:
        size = outs.get(a, 16000 if a == "x" else 4000)
        for b in outs:
            if a == b or (a, b) == ("x", "o"):
                continue
            for at in (NEXT[a], NEXT[a] + size - 16, NEXT[a] + 16 - outs[b]):
                assert lib.refuse_next(following(**{b: at})), (a, b)
            assert lib.refuse_next(following(**{b: NEXT[a] + -(-size // 16) * 16})) is None and lib.refuse_next(following(**{b: NEXT[a] - -(-outs[b] // 16) * 16})) is None, (a, b)
    # in place only where every element is its own
    assert lib.refuse_next(following(o=0x100000, xs=1001)) and lib.refuse_next(following(o=0x100000 + 4000)) and lib.refuse_next(following(o=0x100004))


def test_choices_whose_rows_overlap_what_is_read_beside_the_logits_are_refused(lib):
    """another workgroup may read lengths, penalties and masks when one has written its part of the rows; the tokens are written behind all"""
    ins = dict(hl=16, rep=16, pre=16, fre=16, m=4 * (3 * 40 + 32))
    base = dict(rep=0xd00000, pre=0xe00000, fre=0xf00000, ms=40)
    at = {**NEXT, **base}
    outs = dict(o=16000, r=16000, c=16000, g=16000, ws=lib.next_workspace(4, 1000))
    assert lib.refuse_next(following(**base)) is None
    for a, size in ins.items():
        for b, n in outs.items():
            first = at[a] - n + 16
            for x in (at[a], at[a] + (size - 4) // 16 * 16, first - first % 16):
                assert lib.refuse_next(following(**{**base, b: x})), (a, b)
            assert lib.refuse_next(following(**{**base, b: at[a] + -(-size // 16) * 16})) is None and lib.refuse_next(following(**{**base, b: at[a] - -(-n // 16) * 16})) is None, (a, b)
        assert lib.refuse_next(following(**{**base, "t": at[a]})) is None and lib.refuse_next(following(**{**base, "mx": at[a]})) is None
    # rows of the mask that are the same, and lengths that are not read
    assert lib.refuse_next(following(**{**base, "ms": 0, "c": at["m"] + 128})) is None and lib.refuse_next(following(**{**base, "ms": 0, "c": at["m"] + 124}))
    assert lib.refuse_next(following(**{**base, "history": 0, "c": at["hl"]})) is None


def test_chunks_of_the_vocabulary(lib):
    out = (ctypes.c_uint32 * 2)()
    for n in (1, 2, 7, 64, 256, 1000, 65535):
        for vocab in (1, 2047, 2048, 2049, 32000, 131072, 1 << 24):
            lib.next_of(n, vocab, out)
            assert out[0] in (2048, 4096, 8192) and out[0] * out[1] >= vocab > out[0] * (out[1] - 1)
            assert lib.next_workspace(n, vocab) == 8 * n * out[1]
    assert lib.next_workspace(0, 5) == lib.next_workspace(5, 0) == lib.next_workspace(65536, 5) == lib.next_workspace(5, (1 << 24) + 1) == 0


# ------------------------------------------------------------------ the helpers' own checks
def page_args():
    return dict(lens=i32(3), new=i32(3), block_table=i32(3, 20), free_pages=i32(100), free_span=i32(2), page_size=16, rows=8)


def page_out():
    return {"starts": i32(4), "positions": i32(8), "slots": torch.zeros(8, dtype=torch.int64), "lens": i32(3), "free_span": i32(2)}


@pytest.mark.parametrize("bad", [dict(lens=i32(2)), dict(lens=i32(3).long()), dict(new=i32(4)), dict(new=i32(6)[::2]), dict(block_table=i32(2, 20)), dict(block_table=i32(60)),
                                 dict(block_table=i32(20, 3).t()), dict(free_pages=i32(10, 10)), dict(free_pages=i32(200)[::2]), dict(free_span=i32(3)), dict(free_span=torch.zeros(2)), dict(rows=-1),
                                 dict(rows=1 << 31), dict(page_size=-1), dict(window=-1), dict(window=1 << 32), dict(sinks=1 << 32), dict(out={}), dict(out={**page_out(), "slots": i32(8)}),
                                 dict(out={**page_out(), "starts": i32(3)}), dict(out={**page_out(), "max": i32(3)}), dict(out={k: v for k, v in page_out().items() if k != "lens"})])
def test_page_helper_refuses(helpers, monkeypatch, bad):
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: empty(*a, **{**kw, "device": "cpu"}))
    out = page_out()
    assert ops.wit_page_step(**page_args(), out=out) is out and set(ops.wit_page_step(**page_args())) == set(out)
    with pytest.raises(ValueError):
        ops.wit_page_step(**{**page_args(), **bad})
    assert len(helpers) == 2


def window_args():
    return dict(q=i32(9, 8, 64), k_cache=i32(10, 16, 4, 64), v_cache=i32(10, 16, 4, 64), block_table=i32(2, 5), starts=i32(3), lens=i32(2), max_new=5, max_len=70, exp_table=i32(1 << 20))


@pytest.mark.parametrize("bad", [dict(q=i32(9, 512)), dict(q=i32(9, 8, 60)), dict(q=i32(9, 8, 64).float()), dict(block_table=i32(3, 5)), dict(block_table=i32(2, 10)[:, :5]), dict(block_table=i32(10)),
                                 dict(lens=i32(3)), dict(starts=i32(2)), dict(starts=i32(6)[::2]), dict(starts=torch.zeros(3)), dict(exp_table=i32(1000)), dict(index_bits=19), dict(max_len=-1),
                                 dict(max_new=-1), dict(max_len=1 << 32), dict(max_new=1 << 31), dict(window=-1), dict(sinks=1 << 32), dict(qk_scale=1 << 64), dict(bit_shift=-1), dict(out={}),
                                 dict(out={"max": i32(9, 8)}), dict(out={"qkv": i32(9, 8, 64), "score": i32(9, 8, 70)}), dict(out={"qkv": i32(9, 8, 64), "scores": i32(9, 8, 71)}),
                                 dict(out={"qkv": i32(2, 8, 64)}), dict(workspace=i32(1000)), dict(v_cache=i32(10, 16, 64, 4).transpose(2, 3))])
def test_window_helper_refuses(helpers, bad):
    got = ops.wit_window_attention(**window_args())
    assert got["scores"].shape == (9, 8, 70) and got["qkv"].shape == (9, 8, 64) and not any(t.any() for t in got.values())
    assert set(ops.wit_window_attention(**window_args(), proof=False)) == {"qkv", "qkv_rem"}
    n = len(helpers)
    with pytest.raises(ValueError):
        ops.wit_window_attention(**{**window_args(), **bad})
    assert not [c for c in helpers[n:] if not c[0].endswith("_workspace")]


def next_args():
    return dict(logits=i32(3, 100), history=i32(3, 20), history_lens=i32(3), repetition=i32(3), presence=i32(3), frequency=i32(3), bias=i32(3, 100), mask=i32(3, 4))


@pytest.mark.parametrize("bad", [dict(logits=i32(300)), dict(logits=i32(3, 100).float()), dict(logits=i32(100, 3).t()), dict(history=i32(2, 20)), dict(history=i32(60)), dict(history=None),
                                 dict(history_lens=None), dict(history_lens=i32(2)), dict(repetition=i32(2)), dict(presence=i32(3, 1)), dict(frequency=torch.zeros(3)), dict(bias=i32(99)),
                                 dict(bias=i32(2, 100)), dict(mask=i32(3)), dict(mask=i32(3, 100)), dict(mask=torch.zeros((3, 4), dtype=torch.bool)), dict(scale=1 << 63), dict(scale=0.5), dict(out={}),
                                 dict(out={"max": i32(3)}), dict(out={"token": i32(3), "logits": i32(3, 99)}), dict(out={"token": i32(3), "scores": i32(3, 100)}), dict(out={"token": i32(4)}),
                                 dict(workspace=i32(1000))])
def test_next_helper_refuses(helpers, bad):
    got = ops.wit_next_token(**next_args())
    assert set(got) == {"token", "max", "logits", "rem", "count", "gap"} and got["gap"].shape == (3, 100)
    assert set(ops.wit_next_token(i32(3, 100), proof=False)) == {"token", "max"}
    n = len(helpers)
    with pytest.raises(ValueError):
        ops.wit_next_token(**{**next_args(), **bad})
    assert not [c for c in helpers[n:] if not c[0].endswith("_workspace")]


def test_helpers_hand_over_strides(helpers):
    ops.wit_next_token(i32(3, 130)[:, 5:105], i32(3, 64)[:, :20], i32(3), bias=i32(100), mask=i32(3, 7)[:, 1:5])
    args = [c[1] for c in helpers if c[0] == "grape_wit_next_token"][0]
    assert ops._NEXT.unpack(args[0])[16:20] == (130, 64, 0, 7)
    ops.wit_window_attention(**{**window_args(), "q": i32(9, 12 * 64)[:, 64:9 * 64].view(9, 8, 64)})
    args = [c[1] for c in helpers if c[0] == "grape_wit_window_attention"][0]
    assert ops._WINDOW.unpack(args[0])[1] == 12 * 64


def test_helpers_refuse_tensors_of_another_device(helpers, monkeypatch):
    monkeypatch.setattr(ops, "_place", lambda: 0)
    for call, args in ((ops.wit_page_step, {**page_args(), "out": page_out()}), (ops.wit_window_attention, window_args()), (ops.wit_next_token, next_args())):
        with pytest.raises(ValueError):
            call(**args)
    assert not helpers
