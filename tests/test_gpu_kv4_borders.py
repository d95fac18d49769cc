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
