"""The 4-bit paged cache on the host: the page pool's forks, drops and compaction, what the C entries refuse, turns, tiles, and the plain restatement against itself."""
import ctypes as C
import random

import numpy as np
import pytest

import kv4_plain as P
from prima_cpp_amd import lib as L
from prima_cpp_amd import ops

SHAPE, ALIGN, RANGE, UNSUPPORTED, NOMEM = -2, -3, -4, -1, -11


@pytest.fixture
def pool():
    made = []

    def new(pages, seqs, limit):
        lib = L.load()
        lib.pm355_page_pool_new.restype = C.c_void_p
        lib.pm355_page_pool_free.argtypes = [C.c_void_p]
        for n, k in dict(open=0, close=1, grow=2, drop_before=2, drop=3, fork=2, page=2, free_pages=0, users=1).items():
            getattr(lib, "pm355_page_pool_" + n).argtypes = [C.c_void_p] + [C.c_int] * k
        lib.pm355_page_pool_own.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_int]
        lib.pm355_page_pool_compact.argtypes = [C.c_void_p, C.c_void_p, C.c_int]
        made.append(lib.pm355_page_pool_new(pages, seqs, limit))

        def call(name, *a):
            if name in ("own", "compact"):
                n = a[-1]
                buf = np.zeros((max(1, n), 2), np.int32)
                rc = getattr(lib, "pm355_page_pool_" + name)(made[-1], *a[:-1], buf.ctypes.data, n)
                return rc, buf[:max(0, rc)].tolist()
            return getattr(lib, "pm355_page_pool_" + name)(made[-1], *a)
        return call
    yield new
    for p in made:
        L.load().pm355_page_pool_free(p)


def test_fork_shares_and_own_copies(pool):
    p = pool(10, 4, 8)
    a = p("open")
    assert p("grow", a, 150) == 0 and p("free_pages") == 7
    b = p("fork", a, 150)
    assert b >= 0 and [p("page", b, i) for i in range(4)] == [p("page", a, i) for i in range(3)] + [-1] and p("free_pages") == 7
    assert [p("users", p("page", a, i)) for i in range(3)] == [2, 2, 2]
    last = p("page", a, 2)
    n, pairs = p("own", b, 150, 4)
    assert n == 1 and pairs == [[last, p("page", b, 2)]] and p("page", b, 2) != last and p("users", last) == 1 and p("free_pages") == 6
    assert p("own", a, 150, 4) == (0, [])                  # the other one holds its page alone now
    assert p("close", a) == 0 and p("free_pages") == 7     # the two shared pages stay
    assert p("close", b) == 0 and p("free_pages") == 10


def test_fork_of_a_part_and_refusals(pool):
    p = pool(4, 2, 8)
    a = p("open")
    assert p("grow", a, 200) == 0
    assert p("fork", a, 257) == RANGE and p("fork", a, -1) == RANGE and p("fork", 7, 0) == RANGE and p("fork", a, 2 ** 31 - 1) == RANGE
    b = p("fork", a, 64)
    assert p("page", b, 0) == p("page", a, 0) and p("page", b, 1) == -1
    assert p("fork", a, 64) == NOMEM                       # no sequence left
    assert p("own", b, 0, 4)[0] == NOMEM                   # no page left
    assert p("own", b, 0, 0)[0] == RANGE and p("own", b, -1, 4)[0] == RANGE and p("users", p("page", a, 0)) == 2
    assert p("grow", b, 65) == NOMEM and p("grow", b, 2 ** 31 - 1) == RANGE and p("users", 4) == RANGE


def test_drop_keeps_the_first_pages(pool):
    p = pool(10, 2, 10)
    a = p("open")
    assert p("grow", a, 640) == 0
    held = [p("page", a, i) for i in range(10)]
    assert p("drop", a, 4, 300) == 0                       # pages 1 .. 3 lie wholly in [4, 300)
    assert [p("page", a, i) for i in range(10)] == held[:1] + [-1] * 3 + held[4:] and p("free_pages") == 3
    assert p("drop", a, 4, 300) == 0 and p("free_pages") == 3
    assert p("drop", a, 300, 299) == RANGE and p("drop", a, -1, 64) == RANGE and p("drop", 9, 0, 64) == RANGE
    assert p("drop", a, 0, 64) == 0 and p("free_pages") == 4
    assert p("drop_before", a, 330) == 0 and p("free_pages") == 5
    assert p("drop", a, 0, 2 ** 31 - 1) == 0 and p("free_pages") == 10 and p("close", a) == 0 and p("free_pages") == 10


@pytest.mark.parametrize("seed", range(4))
def test_pool_against_plain_sets(pool, seed):
    """random opens, growths, forks, drops, owns, closes and compactions; contents move with the pairs, every sequence keeps reading what it wrote"""
    r = random.Random(seed)
    p, memory, want = pool(40, 6, 12), [None] * 40, {}
    for step in range(600):
        op = r.choice(["open", "grow", "grow", "fork", "write", "write", "drop", "close", "compact"])
        s = r.choice(list(want)) if want else None
        if op == "open" or s is None:
            s = p("open")
            assert s == NOMEM if len(want) == 6 else s not in want
            if s >= 0:
                want[s] = {}
        elif op == "grow":
            n = r.randint(0, 12 * 64)
            have = max(want[s], default=-1) + 1
            rc = p("grow", s, n)
            if rc == 0:
                for i in range(have, (n + 63) // 64):
                    want[s][i] = memory[p("page", s, i)] = (s, i, step)
        elif op == "fork":
            n = r.randint(0, (max(want[s], default=-1) + 1) * 64)
            t = p("fork", s, n)
            if t >= 0:
                want[t] = {i: c for i, c in want[s].items() if i < (n + 63) // 64}
        elif op == "write" and want[s]:
            i = r.choice(list(want[s]))
            n, pairs = p("own", s, i * 64, 12)
            if n >= 0:
                for a, b in pairs:
                    memory[b] = memory[a]
                if p("page", s, i) >= 0:
                    want[s][i] = memory[p("page", s, i)] = (s, i, step)
        elif op == "drop":
            a = r.randint(0, 700)
            b = a + r.randint(0, 400)
            assert p("drop", s, a, b) == 0
            want[s] = {i: (None if a <= 64 * i and 64 * i + 64 <= b else c) for i, c in want[s].items()}
        elif op == "close":
            assert p("close", s) == 0
            del want[s]
        elif op == "compact":
            n, pairs = p("compact", 40)
            used = 40 - p("free_pages")
            ends = [x for q in pairs for x in q]
            assert n >= 0 and len(set(ends)) == 2 * n and all(a >= used > b for a, b in pairs)
            for a, b in pairs:
                memory[b] = memory[a]
        held = {}
        for s, pages in want.items():
            for i, c in pages.items():
                at = p("page", s, i)
                assert (at < 0) == (c is None)
                if c is not None:
                    assert memory[at] == c
                    held[at] = held.get(at, 0) + 1
        assert p("free_pages") == 40 - len(held) and all(p("users", at) == n for at, n in held.items())


def test_rope_turns():
    import torch
    if not torch.cuda.is_available():
        ops_dev, ops._dev = ops._dev, lambda: torch.device("cpu")
    try:
        t, m = ops.rope_turns(128, freq_base=500000.0)
        assert m == 1.0 and np.allclose(t.cpu().numpy(), 500000.0 ** (-np.arange(64) / 64) / (2 * np.pi), rtol=1e-14, atol=0)
        ff = np.linspace(1, 8, 16).astype(np.float32)
        t, m = ops.rope_turns(32, freq_base=10000.0, freq_scale=0.25, attn_factor=1.5, freq_factors=ff)
        assert m == 1.5 and np.allclose(t.cpu().numpy(), 0.25 * 10000.0 ** (-np.arange(16) / 16) / ff / (2 * np.pi), rtol=1e-14, atol=0)
        # the ramp between scaled and unscaled pairs: rope_yarn in 64 bits
        n, base, orig, scale = 64, 10000.0, 4096, 0.125
        t, m = ops.rope_turns(n, n_ctx_orig=orig, freq_base=base, freq_scale=scale, ext_factor=1.0)
        dim = lambda rot: n * np.log(orig / (rot * 2 * np.pi)) / (2 * np.log(base))  # noqa: E731
        lo, hi = max(0, np.floor(dim(32))), min(n - 1, np.ceil(dim(1)))
        mix = 1 - np.clip((np.arange(n // 2) - lo) / max(0.001, hi - lo), 0, 1)
        assert np.allclose(t.cpu().numpy(), base ** (-2 * np.arange(n // 2) / n) / (2 * np.pi) * (scale * (1 - mix) + mix), rtol=1e-12, atol=0)
        assert abs(m - (1 + 0.1 * np.log(8))) < 1e-6 and 0 < lo < hi < n
        for bad in (dict(n_dims=0), dict(n_dims=7), dict(n_dims=8, freq_base=0.0), dict(n_dims=8, freq_factors=np.ones(3))):
            with pytest.raises(L.PM355Error):
                ops.rope_turns(**bad)
    finally:
        if not torch.cuda.is_available():
            ops._dev = ops_dev


def test_structures():
    assert (ops._KV4_CACHE.size, ops._KV4_APPEND.size, ops._ATTN_KV4.size) == tuple(C.sizeof(t) for t in (ops.KV4Cache, ops.KV4AppendArgs, ops.AttnKV4Args))


def test_tiles():
    t, n, keys = ops.kv4_tiles([(3, 10, 1), (0, 70, 1)], 32, 8)
    assert n == 4 and keys == 71 and t.tolist() == [[0, 1, 10, 3], [1, 1, 70, 0]]
    t, n, keys = ops.kv4_tiles([(1, 5, 40), (2, 0, 1), (0, 9, 33)], 32, 8)
    assert n == 32 and keys == 45 and t.tolist() == [[0, 32, 5, 1], [32, 8, 37, 1], [40, 1, 0, 2], [41, 32, 9, 0], [73, 1, 41, 0]]
    assert ops.kv4_tiles([(0, 0, 1)], 40, 1)[1] == 1 and ops.kv4_tiles([(0, 0, 3)], 28, 4)[1] == 18 and ops.kv4_tiles([(0, 0, 2)], 28, 4)[1] == 2
    assert ops.kv4_tiles([], 8, 8)[0].shape == (0, 4)


def test_page_bytes():
    assert [ops.kv4_page_bytes(1, d) for d in (64, 96, 128, 192, 256)] == [64 * 36 * n for n in (2, 3, 4, 6, 8)] and ops.kv4_page_bytes(8, 128) == 8 * 9216
    for G, d in ((1, 32), (1, 80), (1, 0), (0, 64), (-1, 64), (1, 512)):
        with pytest.raises(L.PM355Error):
            ops.kv4_page_bytes(G, d)


@pytest.mark.parametrize("d", [64, 96, 256])
def test_plain_round_trip(d):
    r = np.random.default_rng(d)
    page = r.integers(0, 256, 2 * P.slab(d)["bytes"], dtype=np.uint8)
    rows = {(h, s): (r.normal(size=d).astype(np.float32), r.normal(size=d).astype(np.float32)) for h in range(2) for s in (0, 1, 2, 3, 17, 63)}
    for (h, s), (k, v) in rows.items():
        P.store(page, h, d, s, k, v)
    ku, vu = P.unpack(page[None], 2, d)
    for (h, s), (k, v) in rows.items():
        a, b = P.load(page, h, d, s)
        assert np.array_equal(a, P.values(*P.quantize(k))) and np.array_equal(b, P.values(*P.quantize(v)))
        assert np.array_equal(ku[0, h, s], a) and np.array_equal(vu[0, h, s], b)
        # at most half a step of a scale that is within half a unit of M / 8, or a whole step at the value opposite to M
        step = np.abs(k.reshape(-1, 32)).max(1) / 8
        assert (np.abs(a.astype(np.float64) - k).reshape(-1, 32) <= step[:, None] * (1 + 2.0 ** -7)).all()


# ---- what the C entries refuse, before any device is asked ----
def cache(**kw):
    a = dict(n_head_kv=2, head_dim=64, n_pages=4, pages=4096, d_table=4096, table_ld=4, n_seq=2)
    a.update(kw)
    return ops.KV4Cache(**a)


def append(c=None, **kw):
    a = dict(type=L.F32, n_head=4, n_tokens=3, proj=4096, ld_proj=512, q=4096, ldq=256, norm=0, norm_q=None, norm_k=None, eps=1e-6, d_turns=None, n_rot=0, rope_neox=0, mscale=1.0, d_pos=4096,
             d_seq=4096)
    a.update(kw)
    f = L.declare("pm355_kv4_append", C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p])
    return f(C.byref(c or cache()), C.byref(ops.KV4AppendArgs(**a)), None)


def attend(c=None, **kw):
    a = dict(type=L.F32, n_head=4, q=4096, ldq=256, out=4096, ldo=256, scale=1.0, window=0, n_first=0, d_tiles=4096, n_tiles=2, tile_tokens=8, max_keys=10, n_tokens=9, work=None, work_floats=0)
    a.update(kw)
    f = L.declare("pm355_attn_kv4", C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p])
    return f(C.byref(c or cache()), C.byref(ops.AttnKV4Args(**a)), None)


CACHES = [(dict(pages=None), SHAPE), (dict(d_table=None), SHAPE), (dict(n_pages=0), SHAPE), (dict(n_seq=0), SHAPE), (dict(table_ld=0), SHAPE), (dict(table_ld=2 ** 30), SHAPE),
          (dict(n_head_kv=0), SHAPE), (dict(head_dim=80), SHAPE), (dict(head_dim=32), SHAPE), (dict(pages=4104), SHAPE)]


@pytest.mark.parametrize("bad,code", CACHES)
def test_caches_refused(bad, code):
    assert append(cache(**bad)) == code and attend(cache(**bad)) == code
    f = L.declare("pm355_kv4_load", C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p])
    assert f(C.byref(cache(**bad)), 4096, 4096, 1, 4096, 4096, None) == code


@pytest.mark.parametrize("bad,code", [
    (dict(type=L.F16), UNSUPPORTED), (dict(type=99), UNSUPPORTED), (dict(n_tokens=-1), SHAPE), (dict(n_head=3), SHAPE), (dict(n_head=0), SHAPE), (dict(proj=None), SHAPE), (dict(q=None), SHAPE),
    (dict(d_pos=None), SHAPE), (dict(d_seq=None), SHAPE), (dict(ld_proj=508), SHAPE), (dict(ldq=252), SHAPE), (dict(ld_proj=514), ALIGN), (dict(ldq=258), ALIGN), (dict(proj=4104), ALIGN),
    (dict(q=4100), ALIGN), (dict(d_turns=4096, n_rot=0), SHAPE), (dict(d_turns=4096, n_rot=12), SHAPE), (dict(d_turns=4096, n_rot=72), SHAPE), (dict(mscale=float("inf")), RANGE), (dict(eps=float("nan")), RANGE)])
def test_append_refused(bad, code):
    assert append(**bad) == code


@pytest.mark.parametrize("bad,code", [
    (dict(type=L.F16), UNSUPPORTED), (dict(n_tiles=-1), SHAPE), (dict(n_tokens=0), SHAPE), (dict(n_head=5), SHAPE), (dict(q=None), SHAPE), (dict(out=None), SHAPE), (dict(d_tiles=None), SHAPE),
    (dict(ldq=248), SHAPE), (dict(ldo=248), SHAPE), (dict(window=-1), SHAPE), (dict(n_first=-1), SHAPE), (dict(max_keys=-1), SHAPE), (dict(tile_tokens=0), SHAPE), (dict(tile_tokens=65), SHAPE),
    (dict(ldq=260), ALIGN), (dict(ldo=260), ALIGN), (dict(q=4104), ALIGN), (dict(out=4104), ALIGN), (dict(d_tiles=4100), ALIGN), (dict(work=4100, work_floats=9), ALIGN),
    (dict(n_tiles=2 ** 30, tile_tokens=4), SHAPE), (dict(scale=float("nan")), RANGE), (dict(scale=float("-inf")), RANGE)])
def test_attend_refused(bad, code):
    assert attend(**bad) == code


def test_nothing_to_do():
    assert append(n_tokens=0) == 0 and attend(n_tiles=0) == 0


@pytest.mark.parametrize("bad,code", [
    (dict(pairs=[(0, 4)]), RANGE), (dict(pairs=[(-1, 0)]), RANGE), (dict(pairs=[(0, 1), (2, 1)]), RANGE), (dict(pairs=[(0, 1), (1, 2)]), RANGE), (dict(pairs=[(2, 2)]), RANGE),
    (dict(page_bytes=24), ALIGN), (dict(page_bytes=0), SHAPE), (dict(layer_bytes=32 * 3), SHAPE), (dict(layer_bytes=32 * 4 + 8), ALIGN), (dict(pages=4104), ALIGN), (dict(pages=None), SHAPE),
    (dict(n_layers=0), SHAPE), (dict(n_pages=0), SHAPE), (dict(n_pairs=-1), SHAPE), (dict(n_pairs=5), SHAPE), (dict(n_pairs=1 << 30), SHAPE), (dict(n_pages=1 << 30), SHAPE)])
def test_pages_copy_refused(bad, code):
    a = dict(pages=4096, page_bytes=32, layer_bytes=128, n_layers=2, n_pages=4, pairs=[(0, 1)])
    a.update(bad)
    pairs = np.array(a["pairs"], np.int32)
    f = L.declare("pm355_pages_copy", C.c_int, [C.c_void_p, C.c_size_t, C.c_size_t, C.c_int, C.c_int, C.c_void_p, C.c_int, C.c_void_p])
    assert f(a["pages"], a["page_bytes"], a["layer_bytes"], a["n_layers"], a["n_pages"], pairs.ctypes.data, a.get("n_pairs", len(pairs)), None) == code
