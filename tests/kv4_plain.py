"""The 4-bit paged cache restated in 64 bits (numpy): page bytes, norm + rotation, attention over (sequence, position), one value at a time by the definition in include/prima_mi355.h."""
import numpy as np

PAGE = 64


def slab(d):
    nb = d // 32
    codes, scales = PAGE * 16 * nb, PAGE * 2 * nb
    return dict(k=0, ks=codes, v=codes + scales, vs=2 * codes + scales, bytes=2 * (codes + scales))


def quantize(row):
    """scales (f16) and codes of a head row [d] (f32)"""
    x = np.asarray(row, np.float32).reshape(-1, 32)
    if not np.isfinite(x).all():
        return np.full(len(x), np.nan, np.float16), np.full(x.shape, 8)
    hi, lo = x.max(1), x.min(1)
    s = np.clip(np.where(hi >= -lo, hi, lo) * np.float32(-0.125), -8188, 8188).astype(np.float16)
    f = s.astype(np.float32)[:, None]
    c = np.clip(np.rint(np.divide(x, f, out=np.zeros_like(x), where=f != 0)), -8, 7) + 8
    return s, c.astype(int)


def values(s, c):
    with np.errstate(invalid="ignore"):
        return (s.astype(np.float16)[..., None].astype(np.float32) * (np.asarray(c) - 8)).astype(np.float16).reshape(-1)


# place of each dimension of a row in the codes of a token: byte offset from the token's first, and whether the high half
def _k_places(d):
    nb, out = d // 32, []
    for x in range(d):
        s, g, e = x // 32, x % 32 // 8, x % 8
        out.append(((g * nb + s) * 4 + {0: 0, 2: 0, 4: 1, 6: 1, 1: 2, 3: 2, 5: 3, 7: 3}[e], e in (2, 3, 6, 7)))
    return out


def _v_places(d):
    nb = d // 32
    return [((x % 16) * nb + x // 32) * 4 for x in range(d)], [x // 16 % 2 for x in range(d)]


def _put(buf, at, high, code):
    buf[at] = (buf[at] & (0x0F if high else 0xF0)) | (code << (4 if high else 0))


def store(page, h, d, slot, k, v):
    """key and value rows (f32) of a token into a page (uint8, changed in place)"""
    s, nb = slab(d), d // 32
    b = page[h * s["bytes"]:(h + 1) * s["bytes"]]
    sc, c = quantize(k)
    for x, (at, high) in enumerate(_k_places(d)):
        _put(b, s["k"] + slot * 16 * nb + at, high, int(c.flat[x]))
    b[s["ks"] + slot * nb * 2:s["ks"] + (slot + 1) * nb * 2] = sc.view(np.uint8)
    sc, c = quantize(v)
    at, high = _v_places(d)
    for x in range(d):
        _put(b, s["v"] + slot // 4 * 64 * nb + at[x] + [0, 2, 1, 3][slot % 4], high[x], int(c.flat[x]))
    for w in range(nb):
        b[s["vs"] + (w * PAGE + slot) * 2:][:2] = sc[w:w + 1].view(np.uint8)


def load(page, h, d, slot):
    s, nb = slab(d), d // 32
    b = page[h * s["bytes"]:(h + 1) * s["bytes"]]
    kp, (vat, vhigh) = _k_places(d), _v_places(d)
    kc = [int(b[s["k"] + slot * 16 * nb + at]) >> (4 if high else 0) & 15 for at, high in kp]
    vc = [int(b[s["v"] + slot // 4 * 64 * nb + vat[x] + [0, 2, 1, 3][slot % 4]]) >> 4 * vhigh[x] & 15 for x in range(d)]
    ks = b[s["ks"] + slot * nb * 2:s["ks"] + (slot + 1) * nb * 2].copy().view(np.float16)
    vs = np.array([b[s["vs"] + (w * PAGE + slot) * 2:][:2].copy().view(np.float16)[0] for w in range(nb)])
    return values(ks, np.array(kc).reshape(nb, 32)), values(vs, np.array(vc).reshape(nb, 32))


def unpack(pages, G, d):
    """(k, v) f16 [pages, G, 64, d] of many pages at once, by the same places"""
    s, nb, n = slab(d), d // 32, len(pages)
    b = np.asarray(pages).reshape(n, G, s["bytes"])
    kat, khigh = (np.array(z) for z in zip(*_k_places(d)))
    vat, vhigh = (np.array(z) for z in _v_places(d))
    slot = np.arange(PAGE)
    kc = b[..., s["k"] + slot[:, None] * 16 * nb + kat] >> (4 * khigh).astype(np.uint8) & 15
    vc = b[..., s["v"] + (slot // 4 * 64 * nb + np.array([0, 2, 1, 3])[slot % 4])[:, None] + vat] >> (4 * vhigh).astype(np.uint8) & 15
    ks = np.ascontiguousarray(b[..., s["ks"]:s["v"]]).view(np.float16).reshape(n, G, PAGE, nb)
    vs = np.ascontiguousarray(b[..., s["vs"]:]).view(np.float16).reshape(n, G, nb, PAGE).transpose(0, 1, 3, 2)
    with np.errstate(invalid="ignore", over="ignore"):
        return tuple((np.repeat(sc.astype(np.float32), 32, -1) * (c.astype(np.float32) - 8)).astype(np.float16) for sc, c in ((ks, kc), (vs, vc)))


def norm_rotate(x, w, norm, eps, pos, turns, mscale, neox):
    """a head row in 64 bits"""
    x = np.asarray(x, np.float64)
    if norm:
        x = x / np.sqrt((x * x).mean() + eps) * (1.0 if w is None else np.asarray(w, np.float64))
    if turns is None:
        return x
    n = 2 * len(turns)
    a = 2 * np.pi * np.mod(pos * turns, 1.0)
    i = np.arange(n // 2)
    i, j = (i, i + n // 2) if neox else (2 * i, 2 * i + 1)
    y = x.copy()
    y[i] = (x[i] * np.cos(a) - x[j] * np.sin(a)) * mscale
    y[j] = (x[j] * np.cos(a) + x[i] * np.sin(a)) * mscale
    return y


def seen(pos, n_keys, window, first):
    j = np.arange(n_keys)
    ok = j <= pos
    if window:
        ok &= (pos - j < window) | (j < first)
    return ok


def attend(q, k, v, ok, scale):
    """one query row [d], keys and values [n, d] of which `ok` are seen: (o, sum of p |v|, sum of |q k| scale at most)"""
    if not ok.any():
        z = np.zeros(len(q))
        return z, z, 0.0
    k, v = k[ok].astype(np.float64), v[ok].astype(np.float64)
    q = np.asarray(q, np.float64)
    s = k @ q * scale
    with np.errstate(invalid="ignore"):
        p = np.exp(s - s.max())
    p /= p.sum()
    return p @ v, p @ np.abs(v), (np.abs(k) @ np.abs(q)).max() * abs(scale)
