"""Partial sums of split keys joined: every head size, numbers of splits of all kinds, odd ones among them (the factors of the splits then end beside a multiple of 16 bytes)."""
import numpy as np
import pytest
import torch

import kv4_check as A
from kv4_check import TYPES
from prima_cpp_amd import ops
from test_gpu_kv4 import DIMS, dev, random_pages, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("H,G", [(8, 2), (3, 1), (16, 1)])
def test_numbers_of_splits(H, G, d, type):
    """4 k pages behind one token are split k times"""
    r = np.random.default_rng(d)
    work = ops.kv4_work(H, G, d)
    for k in (5, 8, 9, 12, 21, 35, 64, 127):
        entries = [(0, 256 * k - 1, 1)]
        table, n = tables([256 * k], r)
        raw = random_pages(n, G, d, r)
        q = torch.from_numpy(2 * r.normal(size=(1, H * d)).astype(np.float32)).to(TYPES[type]).cuda()
        tiles, tile, keys = ops.kv4_tiles(entries, H, G)
        work.fill_(float("nan"))
        A.compare(ops.attn_kv4(q, dev(raw), dev(table), dev(tiles), tile, keys, H, G, d, d ** -0.5, work=work), *A.expected(q, raw, table, entries, H, G, d, d ** -0.5))


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("window,first", [(0, 0), (2500, 70)])
@pytest.mark.parametrize("entries", [[(0, 9000, 4)], [(0, 9000, 70), (1, 77, 5)]])
def test_joined_portions(entries, window, first, d, type):
    H, G, r = 8, 2, np.random.default_rng(d)
    table, n = tables([p + m for _, p, m in entries], r)
    raw = random_pages(n, G, d, r)
    q = torch.from_numpy(2 * r.normal(size=(sum(m for *_, m in entries), H * d)).astype(np.float32)).to(TYPES[type]).cuda()
    tiles, tile, keys = ops.kv4_tiles(entries, H, G)
    out = ops.attn_kv4(q, dev(raw), dev(table), dev(tiles), tile, keys, H, G, d, d ** -0.5, window, first, work=ops.kv4_work(H, G, d))
    A.compare(out, *A.expected(q, raw, table, entries, H, G, d, d ** -0.5, window, first))
