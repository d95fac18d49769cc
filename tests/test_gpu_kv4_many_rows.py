"""Append of so many rows that a wave takes several groups of head rows, one behind another: 8192 / T waves per token, rounded down, where that is less than its groups (of 8, 4 or 2 head rows with
heads up to 64, 128, 256)."""
import numpy as np
import pytest
import torch

import kv4_plain as P
from kv4_check import TYPES
from prima_cpp_amd import ops
from test_gpu_kv4 import dev

pytestmark = pytest.mark.gpu

CASES = [  # tokens, d, H, G: one wave per token, then several with more groups than waves; heads that fill no last group
    (8193, 64, 20, 10), (8200, 96, 9, 3), (9001, 128, 10, 5), (8192, 192, 6, 3), (8193, 256, 3, 3), (4097, 128, 18, 6), (2700, 128, 46, 23), (1500, 128, 40, 8), (1500, 64, 71, 1), (1100, 256, 10, 5), (701, 96, 63, 21)]


def waves(T, d, H, G):
    rpw = 8 if d <= 64 else 4 if d <= 128 else 2
    return min(max(1, 8192 // T), 2 * -(-G // rpw) + -(-H // rpw)), 2 * -(-G // rpw) + -(-H // rpw)


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("neox,norm", [(True, True), (False, True), (False, False)])
@pytest.mark.parametrize("T,d,H,G", CASES)
def test_append_of_many_rows(T, d, H, G, neox, norm, type):
    """the same as in calls of 64 rows, whose waves take one group each; sampled rows against 64 bits; in place"""
    parts, groups = waves(T, d, H, G)
    assert 1 <= parts < groups and waves(64, d, H, G)[0] == groups
    r = np.random.default_rng(T)
    where = r.permutation(T)                                # rows of three sequences in any order, some without a place
    pos, seq = (where // 3).astype(np.int32), (where % 3).astype(np.int32)
    pos[::97], seq[::89] = -1, 7
    held = T // 3 // 64 + 1
    table = r.permutation(3 * held + 2)[:3 * held].reshape(3, held).astype(np.int32)
    table[1, held // 2] = -1
    g = torch.Generator("cuda").manual_seed(T)
    proj = torch.randn(T, (H + 2 * G) * d, generator=g, device="cuda").to(TYPES[type])
    start = torch.randint(0, 256, (3 * held + 2, ops.kv4_page_bytes(G, d)), generator=g, device="cuda", dtype=torch.uint8)
    wq, wk = (torch.rand(d, generator=g, device="cuda") + 0.5 for _ in range(2))
    turns, mscale = ops.rope_turns(d // 2 if neox else d, freq_base=500000.0, attn_factor=1.25)
    more = dict(norm=norm, norm_q=wq if norm else None, norm_k=wk if norm else None, turns=turns, mscale=mscale, neox=neox)
    table, p, s = dev(table), dev(pos), dev(seq)

    pages, parted = start.clone(), start.clone()
    q = ops.kv4_append(proj, pages, table, p, s, H, G, d, **more)
    small = torch.cat([ops.kv4_append(proj[i:i + 64], parted, table, p[i:i + 64], s[i:i + 64], H, G, d, **more) for i in range(0, T, 64)])
    assert torch.equal(pages, parted) and not torch.equal(pages, start) and torch.equal(q, small)

    x, again = proj.clone(), start.clone()
    ops.kv4_append(x, again, table, p, s, H, G, d, q=x[:, :H * d], **more)
    assert torch.equal(again, pages) and torch.equal(x[:, :H * d], q) and torch.equal(x[:, H * d:], proj[:, H * d:])

    k, v = (t.cpu().numpy() for t in ops.kv4_load(pages, table, p, s, G, d))
    half, tn, page_of = torch.finfo(TYPES[type]).eps / 2, turns.cpu().numpy(), table.cpu().numpy()
    for t in sorted({0, 1, 63, 64, 97, T // 2, T - 2, T - 1} | set(r.integers(0, T, 8).tolist())):
        a, at = proj[t].float().cpu().numpy().reshape(-1, d), max(0, int(pos[t]))
        for h in sorted({0, 1, H // 2, H - 1}):
            e = P.norm_rotate(a[h], wq.cpu().numpy() if norm else None, norm, 1e-6, at, tn, mscale, neox)
            assert (np.abs(q[t, h * d:(h + 1) * d].float().cpu().numpy() - e) <= half * np.abs(e) + 2e-6 * np.abs(e).max()).all(), (t, h)
        there = pos[t] >= 0 and seq[t] < 3 and page_of[seq[t], at // 64] >= 0
        for h in sorted({0, G // 2, G - 1}):
            e = P.norm_rotate(a[H + h], wk.cpu().numpy() if norm else None, norm, np.float32(1e-6), at, tn, mscale, neox).astype(np.float32)
            assert np.array_equal(k[t, h], P.values(*P.quantize(e)) if there else np.zeros(d)) and np.array_equal(v[t, h], P.values(*P.quantize(a[H + G + h])) if there else np.zeros(d)), (t, h)
