"""The 4-bit paged cache on the device against the 64-bit restatement (tests/kv4_plain.py): append, load, attention, page copies, and all of them together.

Tolerances. A rounding to t is off by at most half a step, torch.finfo(t).eps / 2 of the value. Queries of append: one rounding, and 32-bit arithmetic of some ten operations on values up to
the head's largest. Attention: one rounding of the output; with bf16 rows probabilities are f16 (2^-11 of each, so 2^-11 of sum p |v|), with f32 rows pairs of f16 (2^-22), queries likewise
exact / 2^-22; scores are f32 sums of d products, each addition off by at most 2^-24 of sum |q k| scale =: B, so that a probability is off by 2 (d 2^-24 + 2^-22) B, and exp2 and the sums by
2^-18 at most of sum p |v|. A probability against the largest one also has the absolute step of f16: it is held times 2^8, so it is off by up to 2^-25 / 2^8 = 2^-33 however small it is,
each times its |v| (a value of 1e-71 in 64 bits is 0 here)."""
import numpy as np
import pytest
import torch

import kv4_plain as P
from prima_cpp_amd import lib as L
from prima_cpp_amd import ops

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
DIMS = [64, 96, 128, 192, 256]


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def tables(lengths, r, spare=3, ld=None):
    """page tables with pages in random order out of a pool that has `spare` more, padded with -1"""
    need = [(n + 63) // 64 for n in lengths]
    order, t, at = r.permutation(sum(need) + spare), np.full((len(need), ld or max(need + [1])), -1, np.int32), 0
    for s, n in enumerate(need):
        t[s, :n] = order[at:at + n]
        at += n
    return t, sum(need) + spare


def random_pages(n, G, d, r, spread=0.1):
    """pages of random codes, finite scales of either sign"""
    s = P.slab(d)
    p = r.integers(0, 256, (n, G, s["bytes"]), dtype=np.uint8)
    for a, b in ((s["ks"], s["v"]), (s["vs"], s["bytes"])):
        p[..., a:b] = (r.uniform(0.2, 1.0, (n, G, (b - a) // 2)) * r.choice([-spread, spread], (n, G, (b - a) // 2))).astype(np.float16).view(np.uint8).reshape(n, G, b - a)
    return p.reshape(n, -1)


# ---- append and load --------------------------------------------------------------------------------------------------------
APPENDS = [  # d, H, G, type, rot, neox, norm, weights, positions
    (128, 8, 2, "bf16", 128, True, True, True, "mixed"), (128, 4, 4, "f32", 128, False, True, True, "mixed"), (64, 14, 2, "bf16", 32, False, False, False, "one"),
    (64, 3, 1, "f32", 64, True, True, False, "far"), (96, 10, 5, "bf16", 96, True, True, True, "mixed"), (192, 6, 3, "bf16", 64, True, False, False, "mixed"), (192, 2, 1, "f32", 192, False, True, True, "far"),
    (256, 16, 1, "bf16", 256, True, True, True, "mixed"), (256, 5, 5, "f32", 8, False, True, True, "mixed"), (128, 40, 8, "bf16", 0, False, False, False, "prompt"), (96, 9, 9, "f32", 24, True, True, True, "prompt"),
    (128, 1, 1, "bf16", 128, False, True, True, "prompt"), (64, 71, 1, "bf16", 64, True, True, True, "mixed"),
]


def positions(kind, r):
    if kind == "one":
        return [(0, 0)]
    if kind == "far":
        return [(0, 1048575 - 64 * i) for i in range(4)] + [(1, 999_999), (1, 63), (1, 64)]
    if kind == "prompt":
        return [(1, i) for i in range(131)]
    return [(2, 5), (0, 63), (0, 64), (1, 0), (2, 6), (3, 200), (1, 1), (2, 127), (2, 128), (3, 201), (0, 1)]


@pytest.mark.parametrize("d,H,G,type,rot,neox,norm,weights,where", APPENDS)
def test_append(d, H, G, type, rot, neox, norm, weights, where):
    r = np.random.default_rng(d + H)
    at = positions(where, r)
    T = len(at)
    lengths = [1 + max([p for q, p in at if q == s], default=-1) for s in range(4)]
    if where == "far":                                      # (sparse: only the pages that are written exist)
        table = np.full((2, 16384), -1, np.int32)
        for i, page in enumerate(sorted({(s, p // 64) for s, p in at})):
            table[page] = i
        n_pages = len({(s, p // 64) for s, p in at}) + 1
    else:
        table, n_pages = tables(lengths, r)
    before = r.integers(0, 256, (n_pages, ops.kv4_page_bytes(G, d)), dtype=np.uint8)
    width = (H + 2 * G) * d
    proj = torch.from_numpy(r.normal(size=(T, width + 8)).astype(np.float32)).to(TYPES[type])
    wq, wk = (torch.from_numpy(r.uniform(0.5, 1.5, d).astype(np.float32)) if weights else None for _ in range(2))
    turns, mscale = ops.rope_turns(rot, freq_base=500000.0, attn_factor=1.25) if rot else (None, 1.0)
    pages = dev(before)
    pos, seq = dev(np.array([p for _, p in at], np.int32)), dev(np.array([s for s, _ in at], np.int32))
    q = torch.full((T, H * d + 16), 7.0, dtype=TYPES[type], device="cuda")
    args = (pages, dev(table), pos, seq)
    ops.kv4_append(proj.cuda()[:, :width], *args, H, G, d, q=q[:, :H * d], norm=norm, norm_q=None if wq is None else wq.cuda(), norm_k=None if wk is None else wk.cuda(), eps=1e-5, turns=turns,
                   mscale=mscale, neox=neox)
    k, v = (t.cpu().numpy() for t in ops.kv4_load(*args, G, d))
    got, x, tn = q.float().cpu().numpy(), proj.float().numpy(), None if turns is None else turns.cpu().numpy()
    assert (got[:, H * d:] == 7.0).all()
    want, half = before.copy(), torch.finfo(TYPES[type]).eps / 2
    for t, (s, p) in enumerate(at):
        row = lambda h, w: P.norm_rotate(x[t, h * d:(h + 1) * d], None if w is None else w.numpy(), norm, 1e-5, p, tn, mscale, neox)  # noqa: E731
        for h in range(H):
            e = row(h, wq)
            assert (np.abs(got[t, h * d:(h + 1) * d] - e) <= half * np.abs(e) + 2e-6 * np.abs(e).max()).all(), (t, h)
        for g in range(G):
            kr, vr = row(H + g, wk).astype(np.float32), x[t, (H + G + g) * d:(H + G + g + 1) * d]
            P.store(want[table[s, p // 64]], g, d, p % 64, kr, vr)
            assert np.array_equal(k[t, g], P.values(*P.quantize(kr))) and np.array_equal(v[t, g], P.values(*P.quantize(vr))), (t, g)
    assert np.array_equal(pages.cpu().numpy(), want)        # and nothing else in the pool changed


def test_append_rows_without_a_place():
    """padding rows, unknown sequences, positions without a page and beyond the table store nothing"""
    r = np.random.default_rng(0)
    G, H, d = 2, 4, 64
    before = r.integers(0, 256, (3, ops.kv4_page_bytes(G, d)), dtype=np.uint8)
    table = np.array([[0, -1, 1], [2, 99, -7]], np.int32)
    at = [(-1, 0), (5, -1), (5, 2), (64, 0), (192, 0), (70, 1), (130, 1), (2 ** 31 - 1, 0), (3, 0)]
    proj = r.normal(size=(len(at), (H + 2 * G) * d)).astype(np.float32)
    pages = dev(before)
    args = (pages, dev(table), dev(np.array([p for p, _ in at], np.int32)), dev(np.array([s for _, s in at], np.int32)))
    turns, _ = ops.rope_turns(64)
    q = ops.kv4_append(dev(proj), *args, H, G, d, turns=turns)
    want = before.copy()
    for g in range(G):
        P.store(want[0], g, d, 3, P.norm_rotate(proj[-1, (H + g) * d:(H + g + 1) * d], None, False, 0, 3, turns.cpu().numpy(), 1.0, False).astype(np.float32),
                proj[-1, (H + G + g) * d:(H + G + g + 1) * d])
    assert np.array_equal(pages.cpu().numpy(), want)
    k, v = ops.kv4_load(*args, G, d)
    assert not k[:-1].any() and not v[:-1].any() and k[-1].any()
    q = q.cpu().numpy()
    assert np.array_equal(q[0], proj[0, :H * d])            # position 0 for a padding row
    assert np.isfinite(q).all()


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("T", [1, 70])
def test_append_in_place(T, type):
    """queries over the front of their own projections"""
    G, H, d = 2, 12, 128
    proj = torch.randn(T, (H + 2 * G) * d, device="cuda").to(TYPES[type])
    table, turns = torch.arange(2, dtype=torch.int32, device="cuda")[None], ops.rope_turns(d)[0]
    pos, seq = torch.arange(T, dtype=torch.int32, device="cuda"), torch.zeros(T, dtype=torch.int32, device="cuda")
    a, b = (torch.zeros(2, ops.kv4_page_bytes(G, d), dtype=torch.uint8, device="cuda") for _ in range(2))
    q = ops.kv4_append(proj, a, table, pos, seq, H, G, d, norm=True, turns=turns, neox=True)
    x = proj.clone()
    ops.kv4_append(x, b, table, pos, seq, H, G, d, q=x[:, :H * d], norm=True, turns=turns, neox=True)
    assert torch.equal(x[:, :H * d], q) and torch.equal(x[:, H * d:], proj[:, H * d:]) and torch.equal(a, b)


@pytest.mark.parametrize("type", ["bf16", "f32"])
def test_append_borders(type):
    """zeros, both signs of the largest value, ties between codes, values that a 16-bit scale cannot hold, NaN and infinities"""
    G, H, d = 1, 1, 64
    r = np.random.default_rng(1)
    rows = np.zeros((12, d), np.float32)
    rows[1, :32], rows[1, 32:] = 1e-30, r.normal(size=32)
    rows[2, 3], rows[2, 40] = 5.0, -5.0
    rows[3, :4], rows[3, 32:36] = [8, -8, 1, 2], [-8, 8, 3, 4]
    rows[4, :16] = np.arange(16) * 0.5 - 8                  # ties at every half
    rows[5] = 3e38
    rows[6, ::2], rows[6, 1::2] = 65504.0, -70000.0
    rows[7] = r.normal(size=d) * 1e-7                       # scales among the denormals
    rows[8], rows[9], rows[10] = r.normal(size=(3, d))
    rows[8, 5], rows[9, 37], rows[10, 63] = np.nan, np.inf, -np.inf
    rows[11] = r.normal(size=d) * 1e4
    x = torch.from_numpy(rows).to(TYPES[type])
    proj = torch.cat([torch.zeros(12, d, dtype=x.dtype), x, x.flip(-1)], 1).cuda()
    pages = torch.zeros(1, ops.kv4_page_bytes(G, d), dtype=torch.uint8, device="cuda")
    args = (pages, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.arange(12, dtype=torch.int32, device="cuda"), torch.zeros(12, dtype=torch.int32, device="cuda"))
    ops.kv4_append(proj, *args, H, G, d)
    k, v = (t.cpu().numpy()[:, 0] for t in ops.kv4_load(*args, G, d))
    x = x.float().numpy()
    for t in range(12):
        assert np.array_equal(k[t], P.values(*P.quantize(x[t])), equal_nan=True) and np.array_equal(v[t], P.values(*P.quantize(x[t, ::-1])), equal_nan=True), t
    assert np.isnan(k[8:11]).all() and np.isfinite(k[:8]).all() and not k[0].any()


# ---- attention --------------------------------------------------------------------------------------------------------------
def attend_case(d, H, G, type, entries, window=0, first=0, seed=0, drop=(), spread=0.1, work=True, break_pages=None, gain=1.0, stride=0, scale=None):
    """entries (sequence, first new position, new tokens); compares every row with the restatement, returns the output"""
    r = np.random.default_rng(seed)
    n_seq = max(s for s, _, _ in entries) + 1
    lengths = [max([p + n for s, p, n in entries if s == q], default=0) for q in range(n_seq)]
    table, n_pages = tables(lengths, r)
    for s, i in drop:
        table[s, i] = -1
    raw = random_pages(n_pages, G, d, r, spread)
    if break_pages:
        break_pages(raw, table)
    T = sum(n for _, _, n in entries)
    q = torch.from_numpy((gain * r.normal(size=(T, H * d + stride))).astype(np.float32)).to(TYPES[type])
    tiles, tile, keys = ops.kv4_tiles(entries, H, G)
    out = torch.full((T + 1, H * d + stride), 5.0, dtype=TYPES[type], device="cuda")
    qd = torch.cat([q, q[:1]]).cuda()
    scale = d ** -0.5 if scale is None else scale
    w = ops.kv4_work(H, G, d) if work else None
    ops.attn_kv4(qd[:, :H * d], dev(raw), dev(table), dev(tiles), tile, keys, H, G, d, scale, window, first, out=out[:, :H * d], work=w)
    if work:                                                # a second call on the same scratch
        again = torch.full_like(out, 5.0)
        ops.attn_kv4(qd[:, :H * d], dev(raw), dev(table), dev(tiles), tile, keys, H, G, d, scale, window, first, out=again[:, :H * d], work=w)
        assert torch.equal(out.nan_to_num(9.0), again.nan_to_num(9.0))
    got = out.double().cpu().numpy()
    assert (got[T] == 5.0).all() and (got[:, H * d:] == 5.0).all()
    k, v = P.unpack(raw, G, d)
    half, pq = torch.finfo(TYPES[type]).eps / 2, (2.0 ** -11, 0.0) if type == "bf16" else (2.0 ** -21, 2.0 ** -22)
    row, R, worst = 0, H // G, 0.0
    for s, p0, n in entries:
        held = (p0 + n + 63) // 64
        ks, vs = (z[np.maximum(table[s, :held], 0)].transpose(1, 0, 2, 3).reshape(G, -1, d) for z in (k, v))
        there = np.repeat(table[s, :held] >= 0, 64)
        for i in (range(n) if n < 40 else sorted({0, 1, 2, 3, 31, 32, 33, 62, 63, 64, n // 2, n - 2, n - 1} & set(range(n)))):
            ok = P.seen(p0 + i, held * 64, window, first) & there
            for h in (range(H) if n < 12 else sorted({0, H // 2, H - 1})):
                g = h // R
                e, A, B = P.attend(q[row + i, h * d:(h + 1) * d].float().numpy(), ks[g], vs[g], ok, scale)
                o = got[row + i, h * d:(h + 1) * d]
                if np.isnan(e).any():
                    assert np.isnan(o).all() and np.isnan(e).all(), (s, i, h)
                    continue
                tol = half * np.abs(e) + (pq[0] + 2.0 ** -18 + 2 * (d * 2.0 ** -24 + pq[1]) * B) * A + 2.0 ** -33 * np.abs(vs[g][ok].astype(np.float64)).sum(0)
                bad = ~(np.abs(o - e) <= tol)
                assert not bad.any(), (s, i, h, o[bad][:3], e[bad][:3], tol[bad][:3])
                worst = max(worst, float((np.abs(o - e) / np.maximum(tol, 1e-30)).max()))
        row += n
    print("worst %.2f of the tolerance" % worst)
    return out


FEW = [(0, 0, 1), (1, 62, 1), (2, 63, 1), (3, 64, 1), (4, 700, 1)]


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("H,G", [(4, 4), (8, 2), (7, 1), (40, 2), (9, 3)])
def test_attend_one_token(d, H, G, type):
    attend_case(d, H, G, type, FEW)


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("d,H,G,entries", [
    (128, 8, 2, [(0, 0, 4), (1, 61, 3), (2, 126, 4), (3, 5, 1)]), (64, 2, 2, [(0, 0, 16), (1, 60, 9)]), (96, 7, 1, [(0, 300, 2), (1, 63, 2)]), (256, 16, 4, [(1, 127, 4), (0, 1, 2)])])
def test_attend_drafted_tokens(d, H, G, type, entries):
    attend_case(d, H, G, type, entries)
    attend_case(d, H, G, type, entries, window=33, first=3, seed=1)


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("d", DIMS)
def test_attend_prompts(d, type):
    attend_case(d, 8, 2, type, [(0, 0, 33), (1, 63, 1), (2, 0, 130), (3, 301, 70)])


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("H,G", [(2, 2), (5, 1), (7, 1), (12, 3), (40, 1), (128, 1)])
def test_attend_prompt_groups(H, G, type):
    attend_case(64, H, G, type, [(0, 0, 65), (1, 190, 129)])


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("window,first", [(1, 0), (1, 1), (7, 64), (64, 0), (65, 4), (100, 130), (500, 17), (5000, 3)])
@pytest.mark.parametrize("n", [1, 3, 90])
def test_attend_windows(window, first, n, type):
    attend_case(128, 8, 2, type, [(0, 700, n), (1, 0, n), (2, 64, n)], window, first)


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 70])
def test_attend_dropped_pages_and_empty_rows(n, type):
    """pages that are gone count as masked: behind the window, in the middle, all of a sequence's"""
    attend_case(128, 8, 2, type, [(0, 500, n), (1, 130, n), (2, 10, n)], drop=[(0, 1), (0, 2), (0, 5), (1, 2)] + [(2, i) for i in range(2 if n > 1 else 1)])
    attend_case(64, 4, 4, type, [(0, 900, n)], window=200, first=5, drop=[(0, i) for i in range(1, 10)])


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 2, 80])
def test_attend_garbage_in_masked_places(n, type):
    """slots that no query sees hold NaN, infinities and the largest scales: behind the last token, in front of the window, in a page that another sequence holds"""
    d, G = 128, 2
    s = P.slab(d)

    def spoil(pages, table):
        b = pages.reshape(len(pages), G, s["bytes"])
        ks, vs = b[..., s["ks"]:s["v"]].view(np.float16), b[..., s["vs"]:].view(np.float16)
        last = 300 + n - 1
        page, slot = table[0, last // 64], last % 64
        for bad, sl in zip((np.nan, np.inf, -np.inf, 65504.0), range(slot + 1, 64)):
            ks.reshape(len(pages), G, 64, -1)[page, :, sl] = bad
            vs.reshape(len(pages), G, -1, 64)[page, :, :, sl] = bad
        for j in range(200, 300 - 40):                      # outside the window of every query
            page, sl = table[0, j // 64], j % 64
            ks.reshape(len(pages), G, 64, -1)[page, :, sl] = np.nan
            vs.reshape(len(pages), G, -1, 64)[page, :, :, sl] = np.inf
        for p in set(range(len(pages))) - set(table.flat):
            ks[p], vs[p] = np.nan, np.nan

    out = attend_case(d, 8, 2, type, [(0, 300, n), (1, 20, n)], window=40, first=6, break_pages=spoil)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
def test_attend_garbage_two_pages_on(d, type):
    """tiles over three pages, none of which all of their queries see: what the last one's hidden slots hold is no matter of the first one's keys"""
    s, heads, entries = P.slab(d), 4, [(i, 40, 90) for i in range(24)]

    def spoil(pages, table):
        b = pages.reshape(len(pages), heads, s["bytes"])
        for part, order in (("ks", (64, -1)), ("vs", (-1, 64))):
            x = b[..., s[part]:s[part] + 128 * (d // 32)].view(np.float16).reshape(len(pages), heads, *order)
            x = x if part == "ks" else x.swapaxes(2, 3)
            x[table[:, 2], :, 2:] = np.nan

    out = attend_case(d, heads, heads, type, entries, break_pages=spoil)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("where", ["key", "value"])
@pytest.mark.parametrize("n", [3, 80])
def test_attend_nan_reaches_those_who_see_it(n, where, type):
    """a row that is not finite: NaN for the queries behind it, whose window reaches it, and for no other"""
    d, G = 64, 1
    s = P.slab(d)

    def spoil(pages, table):
        b = pages.reshape(len(pages), G, s["bytes"])
        ks, vs = b[..., s["ks"]:s["v"]].view(np.float16), b[..., s["vs"]:].view(np.float16)
        page, sl = table[0, 101 // 64], 101 % 64
        (ks.reshape(len(pages), G, 64, -1)[page, :, sl] if where == "key" else vs.reshape(len(pages), G, -1, 64)[page, :, :, sl])[...] = np.nan

    out = attend_case(d, 4, 1, type, [(0, 100, n)], window=30, break_pages=spoil).float().cpu().numpy()
    bad = np.isnan(out[:n, :4 * d]).all(1)
    assert [i for i in range(n) if bad[i]] == [i for i in range(n) if 1 <= i < 31]


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("gain,spread", [(40.0, 2.0), (1e-4, 1e-5), (3000.0, 0.01)])
def test_attend_ranges(gain, spread, type):
    """sharp and flat softmaxes, large and tiny queries and values"""
    attend_case(128, 8, 2, type, [(0, 333, 1), (1, 64, 1)], gain=gain, spread=spread)
    attend_case(128, 8, 2, type, [(0, 333, 40)], gain=gain, spread=spread)


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("entries", [[(0, 333, 1), (1, 64, 1)], [(0, 9000, 1)], [(0, 300, 7), (1, 64, 7)], [(0, 333, 33)], [(0, 9000, 40)]])
@pytest.mark.parametrize("gain", [1e6, 1e9, 1e18, 1e31, 1e37])
def test_attend_far_scores(gain, entries, type):
    """scores up to the largest that a query of its type can make: the value of the key with the largest one, whose probability (1, or any number of f16 steps over the sum of just that)
    is rounded once in the probabilities and once in the output. Rows whose two largest scores lie nearer to each other than the score sums' error are not compared."""
    H, G, d, r = 8, 2, 128, np.random.default_rng(len(entries))
    table, n = tables([p + m for _, p, m in entries], r)
    raw = random_pages(n, G, d, r)
    tiles, tile, keys = ops.kv4_tiles(entries, H, G)
    q = torch.from_numpy((gain * r.normal(size=(sum(m for *_, m in entries), H * d))).astype(np.float32)).to(TYPES[type])
    for scale in (0.088, -1.0):
        got = ops.attn_kv4(q.cuda(), dev(raw), dev(table), dev(tiles), tile, keys, H, G, d, scale, work=ops.kv4_work(H, G, d)).double().cpu().numpy()
        k, v = P.unpack(raw, G, d)
        row, compared, half = 0, 0, torch.finfo(TYPES[type]).eps / 2
        for s, p0, m in entries:
            held = (p0 + m + 63) // 64
            ks, vs = (z[table[s, :held]].transpose(1, 0, 2, 3).reshape(G, -1, d).astype(np.float64) for z in (k, v))
            for i in range(m):
                for h in range(H):
                    x = q[row + i, h * d:(h + 1) * d].double().numpy()
                    score = ks[h * G // H][:p0 + i + 1] @ x * scale
                    at = np.argsort(score)[-2:]
                    B = (np.abs(ks[h * G // H]) @ np.abs(x)).max() * abs(scale)
                    if score[at[1]] - score[at[0]] < max(40.0, 4 * (d + 2) * 2.0 ** -24 * B):
                        continue
                    want = vs[h * G // H][at[1]]
                    assert (np.abs(got[row + i, h * d:(h + 1) * d] - want) <= (half + 2.0 ** -11 + 2.0 ** -18) * np.abs(want)).all(), (s, i, h)
                    compared += 1
            row += m
        assert compared > row * H // 2


@pytest.mark.parametrize("type", ["bf16", "f32"])
def test_attend_strides_and_no_scratch(type):
    attend_case(128, 8, 2, type, [(0, 1000, 1), (1, 3, 1)], stride=24, work=False)
    attend_case(128, 8, 2, type, [(0, 1000, 50), (1, 3, 1)], stride=8, work=False)


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("entries", [[(0, 20000, 1)], [(0, 9000, 4)], [(0, 12345, 70), (1, 77, 5)], [(0, 3000, 1), (1, 8191, 1), (2, 64, 1)]])
def test_attend_split_keys(entries, type):
    attend_case(128, 8, 2, type, entries, gain=2.0)
    attend_case(128, 8, 2, type, entries, gain=2.0, window=2500, first=70)


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 192])
@pytest.mark.parametrize("entries", [[(0, 700, 18)] + [(s, 40 * s, 1) for s in range(1, 12)], [(0, 130, 17), (1, 0, 3), (2, 64, 2), (3, 900, 4), (4, 63, 5)]])
def test_attend_unequal_tiles(entries, d, type):
    """tiles whose columns are many more than those of the others, for which the launch is made"""
    attend_case(d, 14, 2, type, entries)
    attend_case(d, 14, 2, type, entries, window=90, first=5)


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [-0.08, 0.0, 3.0])
@pytest.mark.parametrize("n", [1, 40])
def test_attend_scales(n, scale, type):
    attend_case(128, 8, 2, type, [(0, 333, n), (1, 64, n)], scale=scale)


def test_attend_rows_nobody_names():
    """tiles of padded rows: position < 0 gives zeros, rows outside the tensors and empty tiles nothing"""
    r = np.random.default_rng(0)
    H, G, d = 4, 2, 64
    pages, table = dev(random_pages(4, G, d, r)), dev(np.array([[0, 1], [2, 3]], np.int32))
    q = torch.randn(6, H * d, device="cuda")
    for tile in (1, 8, 64):
        out = torch.full((6, H * d), 5.0, device="cuda")
        tiles = np.array([(0, 1, 20, 0), (2, 1, -1, 0), (3, 1, 5, 7), (4, 0, 9, 1), (-1, 1, 3, 0), (6, 1, 3, 0), (5, 1, 127, 1)], np.int32)
        ops.attn_kv4(q, pages, table, dev(tiles), tile, 128, H, G, d, 0.125, out=out)
        o = out.cpu()
        assert (o[[1, 4]] == 5.0).all() and not o[[2, 3]].any() and (o[[0, 5]] != 5.0).all()


@pytest.mark.parametrize("n", [1, 60])
@pytest.mark.parametrize("floats", [0, 64, 70_000, 1_000_000])
def test_scratch_of_any_size_and_contents(floats, n):
    """and the output over the queries"""
    H, G, d = 8, 2, 128
    r = np.random.default_rng(0)
    table, pages = tables([9000 + n, 70 + n], r)
    pages, table = dev(random_pages(pages, G, d, r)), dev(table)
    tiles, tile, keys = ops.kv4_tiles([(0, 9000, n), (1, 70, n)], H, G)
    q = torch.randn(2 * n, H * d, device="cuda")
    args = (pages, table, dev(tiles), tile, keys, H, G, d, 0.1)
    want = ops.attn_kv4(q, *args)
    work = torch.full((floats,), float("nan"), device="cuda")
    assert torch.allclose(ops.attn_kv4(q, *args, work=work), want, rtol=1e-5, atol=1e-5)
    x = q.clone()
    assert torch.equal(ops.attn_kv4(x, *args, out=x, work=work), ops.attn_kv4(q, *args, work=work)) and x.data_ptr() != q.data_ptr()


def test_far_offsets():
    """a pool beyond 4 GB, a position beyond 2^20"""
    H, G, d, n = 8, 8, 128, 60000
    r = np.random.default_rng(0)
    pages = torch.zeros(n, ops.kv4_page_bytes(G, d), dtype=torch.uint8, device="cuda")
    ids = [n - 1, n // 2 + 7, 3, n - 2]
    part = random_pages(4, G, d, r)
    pages[torch.tensor(ids, device="cuda")] = dev(part)
    table = np.full((1, 1 << 15), -1, np.int32)
    table[0, 16384 * 1:16384 + 4] = ids
    pos0 = 16384 * 64 + 200
    q = torch.randn(2, H * d, device="cuda")
    k, v = P.unpack(part, G, d)
    for most, w in ((1, 8192), (2, 8192), (2, 300), (16, 300)):
        tiles = dev(np.array([(0, 1, pos0, 0), (1, 1, pos0 + 1, 0)], np.int32))
        out = ops.attn_kv4(q, pages, dev(table), tiles, most, pos0 + 2, H, G, d, d ** -0.5, window=w, work=ops.kv4_work(H, G, d)).cpu().numpy()
        for i in range(2):
            for h in (0, 7):
                ok = np.arange(256) + 16384 * 64 <= pos0 + i
                e, A, B = P.attend(q[i, h * d:(h + 1) * d].cpu().numpy(), k[:, h].reshape(-1, d), v[:, h].reshape(-1, d), ok, d ** -0.5)
                assert (np.abs(out[i, h * d:(h + 1) * d] - e) <= 2.0 ** -24 * np.abs(e) + (2.0 ** -17 + 2 * (d * 2.0 ** -24 + 2.0 ** -22) * B) * A + 2.0 ** -33 * np.abs(v[:, h].reshape(-1, d)[ok]).astype(np.float64).sum(0)).all()
    pos, seq = dev(np.array([pos0, pos0 + 1], np.int32)), dev(np.zeros(2, np.int32))
    ops.kv4_append(torch.randn(2, (H + 2 * G) * d, device="cuda"), pages, dev(table), pos, seq, H, G, d)
    ops.pages_copy(pages, [(ids[3], ids[1])])
    assert torch.equal(pages[ids[1]], pages[ids[3]]) and ops.kv4_load(pages, dev(table), pos, seq, G, d)[0].any()


# ---- page copies ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("layers,n,size,pairs", [(1, 2, 16, 1), (3, 50, 4608, 20), (2, 1000, 2304, 500), (5, 9, 147456, 4), (1, 2000, 48, 1000), (70, 3, 9216, 1)])
def test_pages_copy(layers, n, size, pairs):
    r = np.random.default_rng(n)
    order = r.permutation(n)
    to, src = order[:pairs], r.choice(order[pairs:], pairs)  # (a source may stand more than once)
    p = torch.randint(0, 256, (layers, n, size), dtype=torch.uint8, device="cuda")
    want = p.clone()
    want[:, torch.from_numpy(to).cuda()] = p[:, torch.from_numpy(src).cuda()]
    ops.pages_copy(p, np.stack([src, to], 1))
    assert torch.equal(p, want)
    ops.pages_copy(p, [])
    wide = torch.randint(0, 256, (layers, n + 1, size), dtype=torch.uint8, device="cuda")          # layers further apart than their pages
    want = wide.clone()
    want[:, int(order[0])] = wide[:, int(order[-1])]
    ops.pages_copy(wide[:, :n], [(order[-1], order[0])])
    assert torch.equal(wide, want)


# ---- refusals ---------------------------------------------------------------------------------------------------------------
def test_refusals():
    H, G, d = 4, 2, 64
    z = lambda *n, t=torch.float32: torch.zeros(*n, dtype=t, device="cuda")  # noqa: E731
    i32 = torch.int32
    pages, table, pos = z(2, ops.kv4_page_bytes(G, d), t=torch.uint8), z(1, 2, t=i32), z(3, t=i32)
    proj, q, tiles = z(3, (H + 2 * G) * d), z(3, H * d), z(1, 4, t=i32)
    good = dict(proj=proj, pages=pages, table=table, pos=pos, seq=pos, n_head=H, n_head_kv=G, head_dim=d)
    for bad in (dict(proj=proj.half()), dict(proj=proj.cpu()), dict(proj=proj[:, :-1]), dict(proj=proj.t()), dict(proj=z(3, (H + 2 * G) * d + 2)[:, :-2]), dict(pages=pages[:, :-16]),
                dict(pages=pages.cpu()), dict(pages=z(4, ops.kv4_page_bytes(G, d), t=torch.uint8)[::2]), dict(table=table.long()), dict(table=table[0]), dict(table=z(2, 4, t=i32)[:, :2]), dict(pos=pos[:2]),
                dict(seq=pos.long()), dict(q=q.bfloat16()), dict(q=q[:2]), dict(q=z(3, H * d + 2)[:, :-2]), dict(norm_q=z(d)), dict(norm=True, norm_q=z(d + 1)), dict(turns=z(4)),
                dict(turns=z(6, t=torch.float64)), dict(turns=z(36, t=torch.float64)), dict(head_dim=80), dict(n_head=3), dict(n_head_kv=0)):
        with pytest.raises(L.PM355Error):
            ops.kv4_append(**{**good, **bad})
    good = dict(q=q, pages=pages, table=table, tiles=tiles, tile_tokens=1, max_keys=4, n_head=H, n_head_kv=G, head_dim=d, scale=1.0)
    for bad in (dict(q=q.half()), dict(q=q[:, :-8]), dict(q=z(3, H * d + 4)[:, :-4]), dict(tiles=tiles.long()), dict(tiles=z(1, 5, t=i32)), dict(tile_tokens=0), dict(tile_tokens=65), dict(window=-1),
                dict(n_first=-1), dict(out=q.bfloat16()), dict(out=q[:2]), dict(work=z(4, t=torch.float64)), dict(max_keys=-1), dict(n_head=5)):
        with pytest.raises(L.PM355Error):
            ops.attn_kv4(**{**good, **bad})
    for bad in ([(0, 2)], [(0, 0)], [(-1, 0)], [(0, 1), (1, 0)], [(0, 1 << 32)], [(0.0, 1.0)], [0, 1]):
        with pytest.raises(L.PM355Error):
            ops.pages_copy(pages, bad)
    with pytest.raises(L.PM355Error):
        ops.kv4_load(pages, table, pos, pos[:2], G, d)
    assert ops.kv4_append(proj[:0], pages, table, pos[:0], pos[:0], H, G, d).shape == (0, H * d) and ops.attn_kv4(**{**good, "tiles": tiles[:0]}).shape == (3, H * d)


@pytest.mark.parametrize("bad", [dict(window=1 << 32), dict(n_first=-1 << 40), dict(max_keys=1 << 31), dict(tile_tokens=1 << 31), dict(scale=1e39), dict(scale="1")])
def test_numbers_that_do_not_fit(bad):
    H, G, d = 4, 2, 64
    z = lambda *n, t=torch.float32: torch.zeros(*n, dtype=t, device="cuda")  # noqa: E731
    pages, table, tiles = z(2, ops.kv4_page_bytes(G, d), t=torch.uint8), z(1, 2, t=torch.int32), z(1, 4, t=torch.int32)
    with pytest.raises(L.PM355Error):
        ops.attn_kv4(**{**dict(q=z(3, H * d), pages=pages, table=table, tiles=tiles, tile_tokens=1, max_keys=4, n_head=H, n_head_kv=G, head_dim=d, scale=1.0), **bad})
    if "scale" in bad:
        with pytest.raises(L.PM355Error):
            ops.kv4_append(z(3, (H + 2 * G) * d), pages, table, z(3, t=torch.int32), z(3, t=torch.int32), H, G, d, mscale=bad["scale"])


# ---- together ---------------------------------------------------------------------------------------------------------------
class Serving:
    """a model's cache as a program keeps it: pool, tables, pages of all layers"""

    def __init__(self, H, G, d, layers, n_pages, n_seq, dtype):
        import ctypes as C
        self.H, self.G, self.d, self.layers, self.dtype = H, G, d, layers, dtype
        self.lib, self.n_seq, self.most = L.load(), n_seq, 40
        self.lib.pm355_page_pool_new.restype = C.c_void_p
        for n, k in dict(open=0, close=1, grow=2, drop=3, fork=2, page=2, free_pages=0).items():
            getattr(self.lib, "pm355_page_pool_" + n).argtypes = [C.c_void_p] + [C.c_int] * k
        self.lib.pm355_page_pool_own.argtypes, self.lib.pm355_page_pool_compact.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_int], [C.c_void_p, C.c_void_p, C.c_int]
        self.lib.pm355_page_pool_free.argtypes = [C.c_void_p]
        self.p = self.lib.pm355_page_pool_new(n_pages, n_seq, self.most)
        self.pages = torch.randint(0, 256, (layers, n_pages, ops.kv4_page_bytes(G, d)), dtype=torch.uint8, device="cuda")
        self.work, self.turns = ops.kv4_work(H, G, d), ops.rope_turns(d)[0]
        self.weights = [(torch.rand(d, device="cuda") + 0.5, torch.rand(d, device="cuda") + 0.5) for _ in range(layers)]

    def call(self, name, *a):
        return getattr(self.lib, "pm355_page_pool_" + name)(self.p, *a)

    def move(self, name, *a):
        pairs = np.zeros((self.pages.shape[1], 2), np.int32)
        n = getattr(self.lib, "pm355_page_pool_" + name)(self.p, *a, pairs.ctypes.data, len(pairs))
        assert n >= 0
        ops.pages_copy(self.pages, pairs[:n])
        return n

    def table(self):
        return np.array([[self.call("page", s, i) for i in range(self.most)] for s in range(self.n_seq)], np.int32)

    def step(self, entries, proj, window=0, first=0):
        """entries (sequence, first position, tokens) through every layer: queries, keys and values of layer l are proj[l]"""
        for s, p, n in entries:
            assert self.call("grow", s, p + n) == 0
            self.move("own", s, p)
        t, pos = dev(self.table()), dev(np.concatenate([p + np.arange(n) for _, p, n in entries]).astype(np.int32))
        seq = dev(np.concatenate([np.full(n, s) for s, _, n in entries]).astype(np.int32))
        tiles, tile, keys = ops.kv4_tiles(entries, self.H, self.G)
        out = []
        for l in range(self.layers):
            q = ops.kv4_append(proj[l], self.pages[l], t, pos, seq, self.H, self.G, self.d, norm=True, norm_q=self.weights[l][0], norm_k=self.weights[l][1], turns=self.turns)
            out.append(ops.attn_kv4(q, self.pages[l], t, dev(tiles), tile, keys, self.H, self.G, self.d, self.d ** -0.5, window, first, work=self.work))
        return torch.stack(out)

    def close(self):
        self.lib.pm355_page_pool_free(self.p)


@pytest.mark.parametrize("type", ["bf16", "f32"])
def test_serving_together(type):
    """a prompt, a fork that goes another way, drafted tokens, dropped pages, a compaction: every sequence reads what a sequence of its own, fed the same rows, reads"""
    H, G, d, layers = 8, 2, 128, 2
    g = torch.Generator("cuda").manual_seed(0)
    rows = lambda n: torch.randn(layers, n, (H + 2 * G) * d, generator=g, device="cuda").to(TYPES[type])  # noqa: E731
    a, alone = Serving(H, G, d, layers, 40, 4, type), Serving(H, G, d, layers, 40, 4, type)
    alone.weights = a.weights
    try:
        x, y0, y1, z = rows(150), rows(5), rows(70), rows(1)
        s0 = a.call("open")
        first = a.step([(s0, 0, 150)], x)
        s1 = a.call("fork", s0, 150)
        o = a.step([(s0, 150, 5), (s1, 150, 5)], torch.cat([y0, y1[:, :5]], 1))
        b = a.step([(s1, 155, 65)], y1[:, 5:])
        c = a.step([(s0, 155, 1)], z)
        t0, t1 = alone.call("open"), alone.call("open")
        assert torch.equal(first, alone.step([(t0, 0, 150)], x)) and torch.equal(first, alone.step([(t1, 0, 150)], x))
        assert torch.equal(o, alone.step([(t0, 150, 5), (t1, 150, 5)], torch.cat([y0, y1[:, :5]], 1)))
        assert torch.equal(b, alone.step([(t1, 155, 65)], y1[:, 5:])) and torch.equal(c, alone.step([(t0, 155, 1)], z))
        # the longer one goes on under a window: what it hides may go, then the pool is compacted
        w = rows(1)
        want = alone.step([(t1, 220, 1)], w, window=50, first=4)
        free = a.call("free_pages")
        assert a.call("drop", s1, 64, 220 - 50) == 0 and a.call("close", s0) == 0 and a.call("free_pages") > free
        filler = a.call("open")
        assert a.call("grow", filler, 64 * 8) == 0
        assert a.call("drop", filler, 64, 64 * 7) == 0
        a.move("compact")
        assert torch.equal(want, a.step([(s1, 220, 1)], w, window=50, first=4))
    finally:
        a.close()
        alone.close()


def test_captured_and_replayed():
    """append and attention of a decoded token in a graph, replayed with new rows and positions while eager calls run in between"""
    H, G, d, S = 8, 2, 128, 3
    r = np.random.default_rng(0)
    table, n = tables([5000] * S, r)
    start = dev(random_pages(n, G, d, r))
    pages, eager = start.clone(), start.clone()
    table = dev(table)
    proj, pos, seq = torch.zeros(S, (H + 2 * G) * d, device="cuda"), torch.zeros(S, dtype=torch.int32, device="cuda"), torch.arange(S, dtype=torch.int32, device="cuda")
    tiles = torch.zeros(S, 4, dtype=torch.int32, device="cuda")
    turns, work, work2 = ops.rope_turns(d)[0], ops.kv4_work(H, G, d), ops.kv4_work(H, G, d)

    def step(pages, work, out=None, q=None):
        q = ops.kv4_append(proj, pages, table, pos, seq, H, G, d, q=q, turns=turns)
        return ops.attn_kv4(q, pages, table, tiles, 1, 5000, H, G, d, d ** -0.5, out=out, work=work)

    def feed(i):
        p = np.array([4000 + i, 100 + i, 63 + i], np.int32)
        proj.copy_(dev(r.normal(size=proj.shape).astype(np.float32)))
        pos.copy_(dev(p))
        tiles.copy_(dev(np.stack([np.arange(S), np.ones(S), p, np.arange(S)], 1).astype(np.int32)))

    feed(0)
    step(pages, work)
    out, q = torch.zeros(S, H * d, device="cuda"), torch.zeros(S, H * d, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(pages, work, out, q)
    for i in range(6):
        feed(i)
        want = step(eager, work2)
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(out, want) and torch.equal(pages, eager), i


def test_other_streams():
    H, G, d = 8, 2, 64
    r = np.random.default_rng(0)
    table, n = tables([3000, 10], r)
    pages, table = dev(random_pages(n, G, d, r)), dev(table)
    q = torch.randn(2, H * d, device="cuda")
    tiles = dev(np.array([(0, 1, 2999, 0), (1, 1, 9, 1)], np.int32))
    want = ops.attn_kv4(q, pages, table, tiles, 1, 3000, H, G, d, 0.125, work=ops.kv4_work(H, G, d))
    torch.cuda.synchronize()
    got = []
    for _ in range(2):                                      # two calls at once, each with its scratch
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got.append(ops.attn_kv4(q, pages, table, tiles, 1, 3000, H, G, d, 0.125, work=ops.kv4_work(H, G, d)))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
