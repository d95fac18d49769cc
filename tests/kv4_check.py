"""Attention over the 4-bit paged cache in 64 bits for all rows and heads of a batch at once (torch, on the device of the tensors that it gets), with the tolerance of every value.

The tolerance, from the roundings on the way (half a step of a type is torch.finfo(t).eps / 2 of the value): the output's one rounding; probabilities in f16 with bf16 rows (2^-11 of each) and in
pairs of f16 with f32 rows (2^-21), queries likewise exact and 2^-22; scores are f32 sums of d products, so a probability is off by 2 (d 2^-24 + 2^-22 or 0) B, B = scale sum |q k| at the most; exp2
and the sums 2^-18 of sum p |v|; and a probability has the absolute step of f16 too: held times 2^8 it is off by up to 2^-33, times its |v|."""
import numpy as np
import torch

import kv4_plain as P

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def expected(q, raw, table, entries, H, G, d, scale, window=0, first=0):
    """(values, tolerance), 64 bits [rows, H, d], for q [rows, H * d] (its type counts) and entries (sequence, first position, tokens) whose rows follow each other. NaN for a head row that sees a
    key or value that is not finite, or sees anything with a query that is not finite; 0 for one that sees nothing."""
    half, (pe, qe) = torch.finfo(q.dtype).eps / 2, (2.0 ** -11, 0.0) if q.dtype == torch.bfloat16 else (2.0 ** -21, 2.0 ** -22)
    k, v = (torch.from_numpy(x).to(q.device) for x in P.unpack(raw, G, d))
    want, tol, row, R = [], [], 0, H // G
    for s, p0, n in entries:
        held = (p0 + n + 63) // 64
        ids = torch.from_numpy(np.maximum(table[s, :held], 0).astype(np.int64)).to(q.device)
        ks, vs = (x[ids].transpose(0, 1).reshape(G, held * 64, d).double() for x in (k, v))
        there = torch.from_numpy(np.repeat(table[s, :held] >= 0, 64)).to(q.device)
        i, j = torch.arange(p0, p0 + n, device=q.device)[:, None], torch.arange(held * 64, device=q.device)
        ok = there & (j <= i)
        if window:
            ok &= (i - j < window) | (j < first)
        x = q[row:row + n].double().view(n, G, R, d).permute(1, 2, 0, 3)                                       # [G, R, n, d]
        odd_q, odd_kv = ~torch.isfinite(x).all(-1), ~(torch.isfinite(ks).all(-1) & torch.isfinite(vs).all(-1))   # [G, R, n], [G, keys]
        x = x.masked_fill(odd_q[..., None], 0).reshape(G, R * n, d)
        ks, vs = (t.masked_fill(odd_kv[..., None], 0) for t in (ks, vs))
        seen = ok.repeat(R, 1)                                                                                 # [R * n, keys]
        p = torch.matmul(x, ks.transpose(1, 2).contiguous()) * scale
        p = torch.exp(p.masked_fill(~seen, -torch.inf) - p.masked_fill(~seen, -torch.inf).amax(-1, keepdim=True).clamp(min=-1e300))
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
        B = (torch.matmul(x.abs(), ks.abs().transpose(1, 2).contiguous()).masked_fill(~seen, 0).amax(-1) * abs(scale))[..., None]
        o, A, total = torch.matmul(p, vs), torch.matmul(p, vs.abs()), torch.matmul(seen.double(), vs.abs())
        t = half * o.abs() + (pe + 2.0 ** -18 + 2 * (d * 2.0 ** -24 + qe) * B) * A + 2.0 ** -33 * total
        nan = (odd_q.reshape(G, R * n) & seen.any(-1)) | (odd_kv[:, None] & seen).any(-1)
        o = o.masked_fill(nan[..., None], torch.nan)
        want.append(o.view(G, R, n, d).permute(2, 0, 1, 3).reshape(n, H, d))
        tol.append(t.view(G, R, n, d).permute(2, 0, 1, 3).reshape(n, H, d))
        row += n
    return torch.cat(want), torch.cat(tol)


def compare(got, want, tol):
    got = got.double().reshape(want.shape)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), "NaN in the wrong places: %d, %d" % (int(torch.isnan(got).sum()), int(nan.sum()))
    off = ((got - want).abs() / tol.clamp(min=1e-300)).masked_fill(nan, 0)
    assert float(off.max()) <= 1.0, "row, head, value %s: %g for %g, %g of the tolerance" % (np.unravel_index(int(off.argmax()), tuple(off.shape)), float(got.flatten()[off.argmax()]),
                                                                                      float(want.flatten()[off.argmax()]), float(off.max()))
