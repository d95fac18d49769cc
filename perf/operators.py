"""Operators over a cache held in 4 bits, in pages of 64 tokens, and their plain forms.

kind "append": queries and keys normed per head and rotated, keys and values rounded to 4 bits and put into the pages, then read back as the values they stand for; "attend": attention
of new tokens over the pages (causal, optionally a sliding window and first tokens that stay visible); "pages": pages of all layers copied by (from, to) pairs.

A block is 32 values of a head row that share a 16-bit scale s; a value is the 16-bit rounding of s * (code - 8). A page holds, for each KV head of d = 32 * nb dimensions, one after another:
  key codes    [64 tokens][4 g][nb s][4 bytes]  the 8 dimensions from 32 s + 8 g on: byte b has dimension (0, 4, 1, 5)[b] in its low and that + 2 in its high half
  key scales   [64 tokens][nb]
  value codes  [16 quads of tokens][16 n][nb w][4 bytes]  byte b: token (0, 2, 1, 3)[b] of the quad, dimension 32 w + n in its low and 32 w + 16 + n in its high half
  value scales [nb][64 tokens]"""
import math

import numpy as np
import torch

own = False
PAGE = 64
MOST = 65504.0 / 8


def listed():
    return [
        # one token of one sequence on its way into the cache: latency alone
        dict(name="append_1", kind="append", H=32, G=8, d=128, rot=128, neox=False, norm=True, type="bf16", seqs=1, new=1, past=203),
        # a decoded token of 48 users far into their contexts, the head layout of the 70B / 72B windows
        dict(name="append_48", kind="append", H=64, G=8, d=128, rot=128, neox=True, norm=True, type="bf16", seqs=48, new=1, past=120000),
        # a long prompt read in one pass, odd length
        dict(name="append_6001", kind="append", H=32, G=8, d=128, rot=128, neox=True, norm=True, type="bf16", seqs=1, new=6001, past=0),
        # portions of unequal prompts in the 32-bit type, half of each head rotated, no norm
        dict(name="append_f32", kind="append", H=14, G=2, d=64, rot=32, neox=False, norm=False, type="f32", seqs=5, new=311, past=900),
        # chat: one user, short history
        dict(name="attend_1", kind="attend", H=32, G=8, d=128, type="bf16", seqs=1, new=1, past=203, window=0, first=0),
        # a decoded token of 48 users with unequal histories
        dict(name="attend_48", kind="attend", H=64, G=8, d=128, type="bf16", seqs=48, new=1, past=8203, window=0, first=0),
        # a book in the cache, one user
        dict(name="attend_long", kind="attend", H=32, G=8, d=128, type="bf16", seqs=1, new=1, past=131100, window=0, first=0),
        # four drafted tokens of 16 users verified at once, a window of 4096 tokens and the first four
        dict(name="attend_window", kind="attend", H=28, G=4, d=128, type="bf16", seqs=16, new=4, past=32768, window=4096, first=4),
        # a prompt portion of 4096 tokens behind 2011 cached ones
        dict(name="attend_4096", kind="attend", H=32, G=8, d=128, type="bf16", seqs=1, new=4096, past=2011, window=0, first=0),
        # unequal prompt portions in the 32-bit type under a window that ends inside pages
        dict(name="attend_f32", kind="attend", H=14, G=2, d=64, type="f32", seqs=6, new=201, past=900, window=500, first=17),
        # a conversation forked: the half-full last page of each of 16 layers gets a copy
        dict(name="fork", kind="pages", G=8, d=128, layers=16, pool=64, pairs=1),
        # a pool compacted: every page from the upper end moves into a hole below
        dict(name="compact", kind="pages", G=8, d=128, layers=8, pool=1200, pairs=501),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "pages"])
    G, R = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 4, 5, 7, 8])
    d = rng.choice([64, 96, 128, 128, 192, 256])
    if kind == "pages":
        layers = rng.choice([1, 2, 5, 8, 16])
        pairs = _log_uniform(rng, 1, 501 * 8 * 8 * 128 // (layers * G * d) if layers * G * d > 8 * 8 * 128 else 501)
        return dict(kind=kind, G=G, d=d, layers=layers, pool=2 * pairs + rng.randint(5, 60), pairs=pairs)
    c = dict(kind=kind, H=G * R, G=G, d=d, type=rng.choice(["bf16", "bf16", "f32"]), seqs=_log_uniform(rng, 1, 64))
    if kind == "append":
        most = 6001 * 48 * 128 // ((c["H"] + 2 * G) * d * c["seqs"]) // (2 if c["type"] == "f32" else 1)
        c["new"] = _log_uniform(rng, 1, max(1, min(6001, most)))
        return dict(c, rot=rng.choice([d, d, d // 2]), neox=rng.random() < 0.6, norm=rng.random() < 0.6, past=rng.choice([0, _log_uniform(rng, 1, 120000)]))
    c["new"] = rng.choice([1, 1, rng.randint(2, 8), _log_uniform(rng, 9, 4096)])
    room = min(48 * 8203 * 8 * 128 // (c["seqs"] * G * d), 4096 * 6107 * 32 // (c["seqs"] * c["H"] * c["new"])) - c["new"]
    c["new"] = min(c["new"], max(1, int((4096 * 6107 * 32 / (c["seqs"] * c["H"])) ** 0.5)))
    c["past"] = 0 if room < 2 else min(_log_uniform(rng, 1, 131100), room)
    window = rng.choice([0, 0, _log_uniform(rng, 16, 8192)])
    return dict(c, window=window, first=rng.choice([0, rng.randint(1, 130)]) if window else 0)


# sequences of a batch: tokens that are there, and new ones (unequal: down to about a half of what the case says)
def _lengths(case):
    r = np.random.default_rng([case["seqs"], case["new"], case["past"]])
    past = [case["past"]] + [int(case["past"] * r.uniform(0.4, 1.0)) for _ in range(case["seqs"] - 1)]
    new = [case["new"]] + [max(1, int(case["new"] * r.uniform(0.5, 1.0))) for _ in range(case["seqs"] - 1)]
    return past, new


def _rows(past, new):
    """int32 position, sequence and place in its portion of every new token"""
    pos = np.concatenate([p + np.arange(n) for p, n in zip(past, new)])
    seq = np.repeat(np.arange(len(new)), new)
    return pos.astype(np.int32), seq.astype(np.int32), np.concatenate([np.arange(n) for n in new])


def _tiles(past, new, most):
    """portions cut into tiles of up to `most` tokens: {row, tokens, position, sequence}"""
    out, row = [], 0
    for s, (p, n) in enumerate(zip(past, new)):
        out += [(row + i, min(most, n - i), p + i, s) for i in range(0, n, most)]
        row += n
    return np.array(out, np.int32)


def _table(lengths, r):
    """page tables of sequences of these lengths, in pages of a pool taken in random order"""
    need = [(n + PAGE - 1) // PAGE for n in lengths]
    order, t, at = r.permutation(sum(need)), np.full((len(need), max(need)), -1, np.int32), 0
    for s, n in enumerate(need):
        t[s, :n] = order[at:at + n]
        at += n
    return t, sum(need)


def page_bytes(G, d):
    return G * PAGE * 36 * (d // 32)


def _quantize(x):
    """scale [..] and codes [.., 32] of blocks x [.., 32] (32-bit values)"""
    hi, lo = x.amax(-1), x.amin(-1)
    s = (torch.where(hi >= -lo, hi, lo) / -8.0).clamp(-MOST, MOST).half()
    f = s.float()[..., None]
    return s, torch.where(f != 0, torch.round(x / torch.where(f != 0, f, torch.ones_like(f))), torch.zeros_like(x)).clamp(-8, 7) + 8


def _values(s, c):
    return (s.float()[..., None] * (c.float() - 8.0)).half()


def _pack(k, v):
    """pages of keys and values [pages, G, 64, d]"""
    n, G, _, d = k.shape
    nb = d // 32
    ks, kc = _quantize(k.view(n, G, PAGE, nb, 32))
    vs, vc = _quantize(v.view(n, G, PAGE, nb, 32))
    kc = kc.to(torch.uint8).view(n, G, PAGE, nb, 4, 8).transpose(3, 4)[..., [0, 2, 4, 6, 1, 3, 5, 7]].reshape(n, G, PAGE, 4, nb, 4, 2)
    vc = vc.to(torch.uint8).view(n, G, 16, 4, nb, 2, 16).permute(0, 1, 2, 6, 4, 3, 5)[..., [0, 2, 1, 3], :]
    parts = [kc[..., 0] | kc[..., 1] << 4, ks.contiguous().view(torch.uint8), vc[..., 0] | vc[..., 1] << 4, vs.transpose(2, 3).contiguous().view(torch.uint8)]
    return torch.cat([p.reshape(n, G, -1) for p in parts], -1).view(n, -1)


def _unpack(pages, G, d):
    """keys and values [pages, G, 64, d] (16 bits) that pages stand for"""
    n, nb = pages.shape[0], d // 32
    kc, ks, vc, vs = pages.view(n, G, -1).split([PAGE * 16 * nb, PAGE * 2 * nb, PAGE * 16 * nb, PAGE * 2 * nb], -1)
    kc, vc = (torch.stack([c & 15, c >> 4], -1) for c in (kc, vc))
    kc = kc.view(n, G, PAGE, 4, nb, 8)[..., [0, 4, 1, 5, 2, 6, 3, 7]].transpose(3, 4).reshape(n, G, PAGE, nb, 32)
    vc = vc.view(n, G, 16, 16, nb, 4, 2)[..., [0, 2, 1, 3], :].permute(0, 1, 2, 5, 4, 6, 3).reshape(n, G, PAGE, nb, 32)
    ks, vs = ks.contiguous().view(torch.float16).view(n, G, PAGE, nb), vs.contiguous().view(torch.float16).view(n, G, nb, PAGE).transpose(2, 3)
    return _values(ks, kc).reshape(n, G, PAGE, d), _values(vs, vc).reshape(n, G, PAGE, d)


def prepare(case, seed):
    r = np.random.default_rng(seed)
    gen = torch.Generator("cuda").manual_seed(seed)
    normal = lambda *n: torch.randn(*n, generator=gen, device="cuda")  # noqa: E731
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    G, d = case["G"], case["d"]
    if case["kind"] == "pages":
        n = case["pairs"]
        order = r.permutation(case["pool"])[:2 * n]
        pages = torch.randint(0, 256, (case["layers"], case["pool"], page_bytes(G, d)), generator=gen, device="cuda", dtype=torch.uint8)
        return dict(case=case, pages=pages, pairs=np.stack([order[:n], order[n:]], 1).astype(np.int32))
    H, dtype = case["H"], torch.bfloat16 if case["type"] == "bf16" else torch.float32
    past, new = _lengths(case)
    pos, seq, idx = _rows(past, new)
    table, n_pages = _table([p + n for p, n in zip(past, new)], r)
    st = dict(case=case, pos=dev(pos), seq=dev(seq), table=dev(table))
    if case["kind"] == "append":
        st["proj"] = normal(len(pos), (H + 2 * G) * d).to(dtype)
        st["pages"] = torch.zeros(n_pages, page_bytes(G, d), dtype=torch.uint8, device="cuda")
        st["norm_q"], st["norm_k"] = (1 + 0.1 * normal(d) if case["norm"] else None for _ in range(2))
        st["turns"] = dev(500000.0 ** (-2.0 * np.arange(case["rot"] // 2) / case["rot"]) / (2 * math.pi))
        return st
    st["q"] = (2 * normal(len(pos), H * d)).to(dtype)
    st["pages"] = torch.cat([_pack(normal(n, G, PAGE, d), normal(n, G, PAGE, d)) for n in [1024] * (n_pages // 1024) + [n_pages % 1024] if n])
    # up to 16 columns (tokens x query heads of a KV head) are one tile of the matrix cores, a prompt's tiles have up to 128
    st["most"] = max(1, (16 if max(new) * (H // G) <= 16 or max(new) == 1 else 128) // (H // G))
    st["tiles"] = dev(_tiles(past, new, st["most"]))
    st["keys"] = max(p + n for p, n in zip(past, new))
    st["work"] = torch.zeros(16 << 20, device="cuda")                       # partial sums of split keys
    st["starts"], st["new"], st["idx"] = dev(np.array(past, np.int64)), max(new), dev(idx)
    return st


def run(state):
    return globals()["_" + state["case"]["kind"]](state)


def _append(st):
    c = st["case"]
    if own:
        from prima_cpp_amd import ops
        q = ops.kv4_append(st["proj"], st["pages"], st["table"], st["pos"], st["seq"], c["H"], c["G"], c["d"], norm=c["norm"], norm_q=st["norm_q"], norm_k=st["norm_k"], eps=1e-6,
                           turns=st["turns"], neox=c["neox"])
        k, v = ops.kv4_load(st["pages"], st["table"], st["pos"], st["seq"], c["G"], c["d"])
        return dict(q=q, k=k, v=v)
    H, G, d = c["H"], c["G"], c["d"]
    T = st["proj"].shape[0]
    q, k, v = st["proj"].view(T, H + 2 * G, d).split([H, G, G], 1)
    angle = st["pos"].double()[:, None] * st["turns"]
    angle = 2 * math.pi * (angle - angle.floor())
    # keys in 64 bits: their codes depend on which side of a border a value lies
    q, k = _rotate(_norm(q.float(), st["norm_q"]), angle, c), _rotate(_norm(k.double(), st["norm_k"]), angle, c).float()
    k, v = (_values(*_quantize(x.reshape(T, G, d // 32, 32))).reshape(T, G, d) for x in (k, v.float()))
    return dict(q=q.reshape(T, H * d).to(st["proj"].dtype), k=k, v=v)


def _norm(x, w):
    return x if w is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w


def _rotate(x, angle, c):
    cos, sin = angle.cos().to(x.dtype)[:, None], angle.sin().to(x.dtype)[:, None]
    n = c["rot"]
    a, b = (x[..., :n // 2], x[..., n // 2:n]) if c["neox"] else (x[..., 0:n:2], x[..., 1:n:2])
    y = torch.stack([a * cos - b * sin, b * cos + a * sin], -2 if c["neox"] else -1).flatten(-2)
    return torch.cat([y, x[..., n:]], -1)


def _attend(st):
    c = st["case"]
    H, G, d = c["H"], c["G"], c["d"]
    if own:
        from prima_cpp_amd import ops
        return ops.attn_kv4(st["q"], st["pages"], st["table"], st["tiles"], st["most"], st["keys"], H, G, d, scale=d ** -0.5, window=c["window"], n_first=c["first"], work=st["work"])
    S, P = st["table"].shape
    R, N, L = H // G, st["new"], P * PAGE
    k, v = (x.view(S, P, G, PAGE, d).transpose(1, 2).reshape(S, G, L, d).float() for x in _unpack(st["pages"][st["table"].clamp(min=0).flatten().long()], G, d))
    q = torch.zeros(S, N, G, R, d, device="cuda")
    seq, idx = st["seq"].long(), st["idx"]
    q[seq, idx] = st["q"].float().view(-1, G, R, d)
    s = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(S, G, R * N, d), k.transpose(-1, -2)).view(S, G, R, N, L) * d ** -0.5
    i, j = (st["starts"][:, None] + torch.arange(N, device="cuda"))[:, :, None], torch.arange(L, device="cuda")
    seen = j <= i
    if c["window"]:
        seen &= (i - j < c["window"]) | (j < c["first"])
    s.masked_fill_(~seen[:, None, None], -math.inf)
    s = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(s.view(S, G, R * N, L), v).view(S, G, R, N, d) / s.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4)[seq, idx].reshape(-1, H * d).to(st["q"].dtype)


def _pages(st):
    if own:
        from prima_cpp_amd import ops
        ops.pages_copy(st["pages"], st["pairs"])
        return st["pages"]
    pairs = torch.from_numpy(st["pairs"]).cuda().long()
    st["pages"][:, pairs[:, 1]] = st["pages"][:, pairs[:, 0]]
    return st["pages"]


def _seen(case, past, new):
    """(pairs of query and key, keys that any of them sees) of one sequence's portion"""
    if not case["window"]:
        return new * past + new * (new + 1) // 2, past + new
    w, f = case["window"], case["first"]
    pairs = sum(min(i + 1, w) + min(f, max(0, i + 1 - w)) for i in range(past, past + new))
    lo = max(0, past + 1 - w)
    return pairs, past + new - lo + min(f, lo)


def work(case):
    G, d = case["G"], case["d"]
    row = G * 36 * (d // 32)                                                  # bytes of a token's keys and values
    if case["kind"] == "pages":
        return dict(bytes=2 * case["pairs"] * case["layers"] * PAGE * row, flops=0)
    H, es = case["H"], 2 if case["type"] == "bf16" else 4
    past, new = _lengths(case)
    T = sum(new)
    if case["kind"] == "append":
        return dict(bytes=T * ((2 * H + 2 * G) * d * es + row + 2 * G * d * 2), flops=T * (H + 2 * G) * d * 8)
    seen = [_seen(case, p, n) for p, n in zip(past, new)]
    return dict(bytes=sum(k for _, k in seen) * row + 2 * T * H * d * es, flops=4 * d * H * sum(p for p, _ in seen))


def exact(case, seed):
    if case["kind"] == "pages":
        return None
    st = prepare(case, seed)
    H, G, d = case["H"], case["G"], case["d"]
    T = len(st["pos"])
    if case["kind"] == "append":
        x = st["proj"].double().view(T, H + 2 * G, d)
        if case["norm"]:
            rms = x.pow(2).sum(-1, keepdim=True).div(d).add(1e-6).sqrt()
            x = torch.cat([x[:, :H] / rms[:, :H] * st["norm_q"].double(), x[:, H:H + G] / rms[:, H:H + G] * st["norm_k"].double(), x[:, H + G:]], 1)
        n, qk = case["rot"], x[:, :H + G]
        turn = torch.polar(torch.ones(T, 1, n // 2, dtype=torch.float64, device="cuda"), (st["pos"].double()[:, None] * st["turns"]).remainder(1.0)[:, None] * (2 * math.pi))
        if case["neox"]:
            z = torch.complex(qk[..., :n // 2].contiguous(), qk[..., n // 2:n].contiguous()) * turn
            y = torch.cat([z.real, z.imag], -1)
        else:
            y = torch.view_as_real(torch.view_as_complex(qk[..., :n].reshape(T, H + G, n // 2, 2).contiguous()) * turn).flatten(-2)
        qk = torch.cat([y, qk[..., n:]], -1)

        def rounded(z):
            z = z.reshape(T, G, d // 32, 32)
            hi, lo = z.amax(-1), z.amin(-1)
            s = (torch.where(z.abs().amax(-1) <= hi, hi, lo) / -8).clamp(-MOST, MOST).half().double()[..., None]
            return (torch.where(s == 0, torch.zeros_like(z), (z / s).round().clamp(-8, 7)) * s).reshape(T, G, d)
        return dict(q=qk[:, :H].reshape(T, H * d), k=rounded(qk[:, H:]), v=rounded(x[:, H + G:]))
    out, at, R = torch.empty(T, H * d, dtype=torch.float64, device="cuda"), 0, H // G
    past, new = _lengths(case)
    for s, (p, n) in enumerate(zip(past, new)):
        held = (p + n + PAGE - 1) // PAGE
        k, v = (x.transpose(0, 1).reshape(G, held * PAGE, d)[:, :p + n].double() for x in _unpack(st["pages"][st["table"][s, :held].long()], G, d))
        j = torch.arange(p + n, device="cuda")
        for a in range(0, n, 512):
            i = torch.arange(p + a, p + min(n, a + 512), device="cuda")[:, None]
            hidden = (j > i) | ((i - j >= case["window"]) & (j >= case["first"]) if case["window"] else False)
            for g in range(G):
                q = st["q"][at + a:at + a + len(i)].double().view(-1, G, R, d)[:, g].transpose(0, 1)
                w = (q @ k[g].T / math.sqrt(d)).masked_fill(hidden, -math.inf).softmax(-1)
                out[at + a:at + a + len(i)].view(-1, G, R, d)[:, g] = (w @ v[g]).transpose(0, 1)
        at += n
    return out
