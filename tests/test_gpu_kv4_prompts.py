"""The kernel for prompts of attention over the 4-bit cache (workgroups of 128 columns) for every head size: all rows and heads against 64 bits. Every case here has to be one that takes this kernel,
which is asked of the launch plan (also on the host, tests/test_kv4_plan_cpu.py)."""
import numpy as np
import pytest
import torch

import kv4_check as A
import kv4_plain as P
from kv4_check import TYPES
from kv4_plan import plan
from prima_cpp_amd import ops
from test_gpu_kv4 import DIMS, dev, random_pages, tables

pytestmark = pytest.mark.gpu

# name: heads, KV heads, entries (sequence, first position, tokens)
CASES = {
    "portions": (16, 16, [(s, 37 * s, 58 + 7 * s) for s in range(9)]),       # tiles of one sequence each, unequal, the first one's first row sees one key
    "grouped": (8, 2, [(0, 300, 1100), (1, 0, 65)]),                         # tiles of 32 tokens, split keys
    "seven": (14, 2, [(0, 63, 700), (1, 64, 1), (2, 5, 100)]),               # 126 of 128 columns
    "forty": (40, 1, [(0, 190, 301)]),                                       # three tokens a tile
    "one": (1, 1, [(0, 0, 33000)]),                                          # a single head and many tiles
}
WINDOWS = [(0, 0), (1, 0), (7, 64), (64, 0), (100, 130), (200, 17)]


def make(case, d, type, seed=0, gain=2.0, stride=0, drop=()):
    H, G, entries = CASES[case]
    r = np.random.default_rng([seed, d])
    table, n = tables([p + m for _, p, m in entries], r)
    for s, i in drop:
        table[s, i] = -1
    q = torch.from_numpy((gain * r.standard_normal((sum(m for *_, m in entries), H * d + stride), dtype=np.float32))).to(TYPES[type]).cuda()
    return H, G, entries, table, random_pages(n, G, d, r), q


def attend(q, raw, table, entries, H, G, d, scale, window=0, first=0, work=True):
    """rows behind the batch's and values behind a row's heads are left as they are"""
    got = plan("bf16" if q.dtype == torch.bfloat16 else "f32", H, G, d, entries, window, first, work)
    assert got[0] == 128, got
    tiles, tile, keys = ops.kv4_tiles(entries, H, G)
    out = torch.full((len(q) + 1, q.shape[1]), 5.0, dtype=q.dtype, device="cuda")
    x = torch.cat([q, q[:1]])
    w = ops.kv4_work(H, G, d).fill_(float("nan")) if work else None
    ops.attn_kv4(x[:, :H * d], dev(raw), dev(table), dev(tiles), tile, keys, H, G, d, scale, window, first, out=out[:, :H * d], work=w)
    assert (out[-1] == 5.0).all() and (out[:, H * d:] == 5.0).all()
    return out[:-1, :H * d]


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("work", [True, False])
@pytest.mark.parametrize("window,first", WINDOWS)
@pytest.mark.parametrize("case", ["portions", "grouped", "seven", "forty"])
def test_prompts(case, window, first, work, d, type):
    H, G, entries, table, raw, q = make(case, d, type, stride=8)
    A.compare(attend(q, raw, table, entries, H, G, d, d ** -0.5, window, first, work), *A.expected(q[:, :H * d], raw, table, entries, H, G, d, d ** -0.5, window, first))


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 256])
def test_prompt_of_one_head(d, type):
    H, G, entries, table, raw, q = make("one", d, type)
    out = attend(q, raw, table, entries, H, G, d, d ** -0.5, 300, 9)
    # (the last 4000 rows as a portion of their own: the reference needs all keys of a portion for each of its rows)
    A.compare(out[-4000:], *A.expected(q[-4000:], raw, table, [(0, 29000, 4000)], H, G, d, d ** -0.5, 300, 9))


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("window,first", [(0, 0), (100, 5)])
def test_dropped_pages(window, first, d, type):
    """pages that are gone in front, in the middle and at the end; a sequence that has none left"""
    drop = [(0, 0), (3, 1), (4, 0), (4, 2), (5, 4)] + [(2, i) for i in range(3)] + [(8, i) for i in range(3)]
    H, G, entries, table, raw, q = make("portions", d, type, drop=drop)
    want, tol = A.expected(q, raw, table, entries, H, G, d, d ** -0.5, window, first)
    assert (want == 0).all(-1).any() and (want != 0).any()
    A.compare(attend(q, raw, table, entries, H, G, d, d ** -0.5, window, first), want, tol)


def spoil(raw, table, d, G, which, values):
    """keys (ks) or values (vs) of (sequence, position) get scales that are not finite"""
    s = P.slab(d)
    b = raw.reshape(len(raw), G, s["bytes"])
    ks, vs = b[..., s["ks"]:s["v"]].view(np.float16).reshape(len(raw), G, 64, -1), b[..., s["vs"]:].view(np.float16).reshape(len(raw), G, -1, 64)
    for i, (part, seq, pos) in enumerate(which):
        page, slot = table[seq, pos // 64], pos % 64
        if part == "ks":
            ks[page, :, slot] = values[i % len(values)]
        else:
            vs[page, :, :, slot] = values[i % len(values)]


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("window,first", [(0, 0), (40, 6)])
def test_nan_reaches_those_who_see_it(window, first, d, type):
    H, G, entries, table, raw, q = make("portions", d, type)
    spoil(raw, table, d, G, [("ks", 1, 60), ("vs", 3, 130), ("ks", 6, 64 * 4 + 3), ("vs", 8, 2), ("vs", 7, 299)], [np.nan])
    want, tol = A.expected(q, raw, table, entries, H, G, d, d ** -0.5, window, first)
    assert torch.isnan(want).any() and not torch.isnan(want[:58]).any()
    A.compare(attend(q, raw, table, entries, H, G, d, d ** -0.5, window, first), want, tol)


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("d", DIMS)
def test_garbage_in_masked_places(d, type):
    """slots behind the last token and in front of every window, pages that nobody holds"""
    H, G, entries, table, raw, q = make("portions", d, type)
    window, first, which = 30, 6, []
    for s, p, n in entries:
        which += [(part, s, x) for x in list(range(p + n, (p + n + 63) // 64 * 64)) + list(range(6, p - 30)) for part in ("ks", "vs")]
    spoil(raw, table, d, G, which, [np.nan, np.inf, -np.inf, 65504.0])
    raw[sorted(set(range(len(raw))) - set(table.flat))] = 0xff
    want, tol = A.expected(q, raw, table, entries, H, G, d, d ** -0.5, window, first)
    assert torch.isfinite(want).all()
    A.compare(attend(q, raw, table, entries, H, G, d, d ** -0.5, window, first), want, tol)


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("scale", [-0.08, 0.0, 3.0])
@pytest.mark.parametrize("case", ["portions", "grouped"])
def test_scales(case, scale, d, type):
    H, G, entries, table, raw, q = make(case, d, type)
    A.compare(attend(q, raw, table, entries, H, G, d, scale), *A.expected(q, raw, table, entries, H, G, d, scale))


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("case", ["portions", "grouped"])
@pytest.mark.parametrize("gain", [1e6, 1e9, 1e18, 1e31, 1e37])
def test_far_scores(gain, case, d, type):
    """scores up to the largest that a query can make: the value of the key with the largest one, rounded once as a probability's and once in the output (and what is left of the others). Head rows whose two largest scores lie nearer
    to each other than the score sums' error are not compared."""
    H, G, entries, table, raw, q = make(case, d, type, gain=gain)
    k, v = (torch.from_numpy(x).cuda().double() for x in P.unpack(raw, G, d))
    half = torch.finfo(TYPES[type]).eps / 2
    for scale in (0.088, -1.0):
        got, row, compared, of = attend(q, raw, table, entries, H, G, d, scale).double().view(-1, H, d), 0, 0, 0
        for s, p0, n in entries:
            ids = torch.from_numpy(table[s, :(p0 + n + 63) // 64].astype(np.int64)).cuda()
            ks, vs = (x[ids].transpose(0, 1).reshape(G, -1, d) for x in (k, v))
            x = q[row:row + n].double().view(n, G, H // G, d).permute(1, 2, 0, 3).reshape(G, -1, d)
            seen = (torch.arange(ks.shape[1], device="cuda") <= torch.arange(p0, p0 + n, device="cuda")[:, None]).repeat(H // G, 1)
            top, at = (torch.matmul(x, ks.transpose(1, 2).contiguous()) * scale).masked_fill(~seen, -torch.inf).topk(2, -1)
            B = torch.matmul(x.abs(), ks.abs().transpose(1, 2).contiguous()).amax(-1) * abs(scale)
            clear = top[..., 0] - top[..., 1] >= torch.clamp(4 * (d + 2) * 2.0 ** -24 * B, min=40.0)
            want = torch.gather(vs, 1, at[..., :1].expand(-1, -1, d))
            o = got[row:row + n].view(n, G, H // G, d).permute(1, 2, 0, 3).reshape(G, -1, d)
            # (the other keys: each score is off by (d + 2) 2^-24 B at most, so each of the n others weighs exp(-(gap - 2 (d + 2) 2^-24 B)) at the most, times the difference of two values)
            rest = ks.shape[1] * torch.exp(2 * (d + 2) * 2.0 ** -24 * B - (top[..., 0] - top[..., 1]))[..., None] * 2 * vs.abs().amax((1, 2))[:, None, None]
            assert ((o - want).abs() <= (half + 2.0 ** -11 + 2.0 ** -18) * want.abs() + rest)[clear].all(), (s, scale)
            compared, of, row = compared + int(clear.sum()), of + clear.numel(), row + n
        assert compared > of // 2
