"""What a call of attn_kv4 launches (host arithmetic, no device): (columns per workgroup, workgroups side by side per tile, splits of the keys, workgroups) or the error code."""
import ctypes as C

import numpy as np

from prima_cpp_amd import lib as L
from prima_cpp_amd import ops


def raw_plan(type, H, G, d, n_tiles, tile_tokens, max_keys, n_tokens, window=0, first=0, floats=0):
    c = ops.KV4Cache(n_head_kv=G, head_dim=d, n_pages=1, pages=4096, d_table=4096, table_ld=1, n_seq=1)
    a = ops.AttnKV4Args(type=L.BF16 if type == "bf16" else L.F32, n_head=H, q=4096, ldq=H * d, out=4096, ldo=H * d, scale=1.0, window=window, n_first=first, d_tiles=4096, n_tiles=n_tiles,
                        tile_tokens=tile_tokens, max_keys=max_keys, n_tokens=n_tokens, work=4096 if floats else None, work_floats=floats)
    out = np.zeros(4, np.int32)
    rc = L.declare("pm355_attn_kv4_plan", C.c_int, [C.c_void_p] * 3)(C.byref(c), C.byref(a), out.ctypes.data)
    return rc or tuple(out.tolist())


def plan(type, H, G, d, entries, window=0, first=0, work=True):
    """of entries (sequence, first position, tokens) in the tiles that ops.kv4_tiles makes, with ops.kv4_work or no scratch"""
    tiles, tile, keys = ops.kv4_tiles(entries, H, G)
    floats = L.declare("pm355_attn_kv4_work_floats", C.c_size_t, [C.c_int] * 3)(H, G, d) if work else 0
    return raw_plan(type, H, G, d, len(tiles), tile, keys, sum(n for *_, n in entries), window, first, floats)
