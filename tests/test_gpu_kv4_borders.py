"""The 4-bit paged cache at the borders of its numbers: queries that are not finite, very small and very large ones, rows whose squares leave 32 bits."""
import numpy as np
import pytest
import torch

import kv4_check as A
import kv4_plain as P
from kv4_check import TYPES
from prima_cpp_amd import ops
from test_gpu_kv4 import dev, random_pages, tables

pytestmark = pytest.mark.gpu
# a decoded token each, one far behind (split keys), drafted tokens, short portions, and portions of so many sequences that they take the kernel for prompts
BATCHES = {"one": [(0, 0, 1), (1, 70, 1), (2, 130, 1)], "far": [(0, 9000, 1)], "drafted": [(0, 3, 4), (1, 60, 7)], "short": [(0, 10, 33), (1, 0, 40)], "prompt": [(s, 7 * s, 90) for s in range(9)]}


def run(q, raw, table, entries, H, G, d, scale, **kw):
    tiles, tile, keys = ops.kv4_tiles(entries, H, G)
    return ops.attn_kv4(q, dev(raw), dev(table), dev(tiles), tile, keys, H, G, d, scale, work=ops.kv4_work(H, G, d), **kw)


def rows(entries):
    return sum(n for *_, n in entries)


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("batch", list(BATCHES))
def test_queries_that_are_not_finite(batch, d, type):
    """NaN wherever such a query sees a key - also where all of its scores are -inf -, nothing else changes"""
    H = G = 16
    entries, r = BATCHES[batch], np.random.default_rng(d)
    table, n = tables([p + m for _, p, m in entries], r)
    raw = random_pages(n, G, d, r)
    b, s = raw.reshape(n, G, -1), P.slab(d)
    b[..., s["k"]:s["ks"]] = 0x33                          # key heads of one sign each: an infinity gives scores of one sign
    ks = b[..., s["ks"]:s["v"]].view(np.float16)
    ks[...] = np.abs(ks) * np.where(np.arange(G) % 2, 1, -1)[:, None]
    q = torch.from_numpy(r.normal(size=(rows(entries), H, d)).astype(np.float32))
    for i, (row, head, bad) in enumerate((x, h, v) for x in (0, rows(entries) // 2, rows(entries) - 1) for h, v in ((1, np.inf), (2, np.inf), (5, -np.inf), (6, -np.inf), (9, np.nan))):
        q[row, head, (5 * i) % d] = bad
    q = q.to(TYPES[type]).view(-1, H * d).cuda()
    A.compare(run(q, raw, table, entries, H, G, d, d ** -0.5), *A.expected(q, raw, table, entries, H, G, d, d ** -0.5))


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 40])
def test_queries_that_are_not_finite_and_see_nothing(n, type):
    H, G, d, r = 4, 2, 64, np.random.default_rng(0)
    q = torch.full((2 * n, H * d), float("inf"), device="cuda", dtype=TYPES[type])
    tiles = dev(np.array([(0, n, -n, 0), (n, n, 3, 9)], np.int32))
    assert not ops.attn_kv4(q, dev(random_pages(2, G, d, r)), dev(np.array([[0, 1]], np.int32)), tiles, n, 128, H, G, d, 1.0).any()


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("gain,scale", [(1e-36, 1e35), (3e-33, 3e38), (5e37, 2e-39), (1e-20, 9e18), (1e-38, 3e38), (1e-39, 3e38)])
@pytest.mark.parametrize("batch", list(BATCHES))
def test_queries_and_scales_of_any_size(batch, gain, scale, type):
    """the smallest and largest queries with the scale that makes ordinary scores of them: nothing of either is lost on the way"""
    H, G, d = 16, 16, 128
    entries, r = BATCHES[batch], np.random.default_rng(3)
    table, n = tables([p + m for _, p, m in entries], r)
    raw = random_pages(n, G, d, r)
    q = torch.from_numpy((gain * r.normal(size=(rows(entries), H * d))).astype(np.float32)).to(TYPES[type]).cuda()
    assert torch.isfinite(q).all()
    A.compare(run(q, raw, table, entries, H, G, d, scale), *A.expected(q, raw, table, entries, H, G, d, scale))


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("d,H,G,T", [(64, 5, 1, 9), (96, 4, 2, 9), (128, 12, 3, 9), (256, 8, 2, 9), (128, 12, 3, 700)])
@pytest.mark.parametrize("eps", [0.0, 1e-6])
def test_norms_of_any_size(eps, d, H, G, T, type):
    """queries and keys whose squares leave 32 bits at either end have norms like others; a row of zeros stays zeros where eps is not 0"""
    r = np.random.default_rng(d + T)
    sizes = np.array([1.0, 1e19, 3e25, 4e37, 1e-12, 1e-20, 1e-24, 1e-37, 0.0 if eps else 1e-30])[np.arange(T) % 9]
    x = r.normal(size=(T, H + 2 * G, d)) * sizes[:, None, None]
    x[T // 2, ::2] *= 1e-8                                   # heads of unlike sizes in one token
    proj = torch.from_numpy(x.reshape(T, -1).astype(np.float32)).to(TYPES[type])
    wq, wk = (torch.from_numpy(r.uniform(0.5, 1.5, d).astype(np.float32)) for _ in range(2))
    pages = torch.zeros(T // 64 + 1, ops.kv4_page_bytes(G, d), dtype=torch.uint8, device="cuda")
    args = (pages, torch.arange(T // 64 + 1, dtype=torch.int32, device="cuda")[None], torch.arange(T, dtype=torch.int32, device="cuda"), torch.zeros(T, dtype=torch.int32, device="cuda"))
    q = ops.kv4_append(proj.cuda(), *args, H, G, d, norm=True, norm_q=wq.cuda(), norm_k=wk.cuda(), eps=eps).float().cpu().numpy().reshape(T, H, d)
    k = ops.kv4_load(*args, G, d)[0].cpu().numpy()
    x, half, eps = proj.float().numpy().reshape(T, -1, d), torch.finfo(TYPES[type]).eps / 2, float(np.float32(eps))
    for t in range(T) if T < 10 else (0, 1, 2, 3, 6, 8, 66, T // 2, T - 1):
        for h in range(H):
            e = P.norm_rotate(x[t, h], wq.numpy(), True, eps, 0, None, 1.0, False)
            assert (np.abs(q[t, h] - e) <= half * np.abs(e) + 2e-6 * np.abs(e).max()).all(), (t, h, q[t, h, :4], e[:4])
        for g in range(G):
            assert np.array_equal(k[t, g], P.values(*P.quantize(P.norm_rotate(x[t, H + g], wk.numpy(), True, eps, 0, None, 1.0, False).astype(np.float32)))), (t, g)


@pytest.mark.parametrize("R", [1, 3, 5])
def test_tiles_without_tokens(R):
    """counts of 0, -1 and of numbers whose products with the heads of a KV head leave 32 bits: nothing is written, and the scratch behind the slots stays as it is"""
    G, d, r = 2, 64, np.random.default_rng(R)
    H, q = G * R, torch.randn(3, G * R * 64, device="cuda")
    table, n = tables([9000, 300], r)
    raw = random_pages(n, G, d, r)
    counts = [0, -1, -2 ** 31, -2 ** 30, -715827883, -858993460, -429496730, -1431655765]
    for tile in (1, 16 // R, 128 // R):
        tiles = dev(np.array([(1, c, 5, 1) for c in counts] + [(0, 1, 8999, 0)], np.int32))
        out, work = torch.full((3, H * d), 5.0, device="cuda"), torch.full((1 << 22,), 7.0, device="cuda")
        ops.attn_kv4(q, dev(raw), dev(table), tiles, tile, 9000, H, G, d, 0.125, out=out, work=work)
        A.compare(out[:1], *A.expected(q[:1], raw, table, [(0, 8999, 1)], H, G, d, 0.125))
        assert (out[1:] == 5.0).all() and (work[1 << 21:] == 7.0).all()


def test_very_many_tiles():
    """131073 rows of 8 KV heads, each a tile: more than 2^20 workgroups"""
    H = G = 8
    d, r = 64, np.random.default_rng(0)
    entries = [(s, 0, 200) for s in range(4)]
    table, n = tables([200] * 4, r)
    raw = random_pages(n, G, d, r)
    at = np.array([(i, 1, i % 200, i // 200) for i in range(800)], np.int32)
    q = torch.randn(800, H * d, device="cuda").bfloat16()
    few = ops.attn_kv4(q, dev(raw), dev(table), dev(at), 1, 200, H, G, d, 0.125)
    A.compare(few, *A.expected(q, raw, table, entries, H, G, d, 0.125))
    N = (1 << 17) + 1
    which = np.arange(N) % 800
    many = at[which]
    many[:, 0] = np.arange(N)
    rows = torch.from_numpy(which).cuda()
    out = ops.attn_kv4(q[rows], dev(raw), dev(table), dev(many), 1, 200, H, G, d, 0.125, work=ops.kv4_work(H, G, d))
    assert torch.equal(out, few[rows])
