"""Plain 64-bit models of the paged 8-bit operators, for the tests."""
from __future__ import annotations

import numpy as np
import torch

QMAX = {"fp8": 448.0, "int8": 127.0}
DT = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}


def e4m3_table():
    """Value of each of the 256 e4m3 codes (NaN at 0x7f and 0xff)."""
    v = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v[c] = np.nan if (c & 127) == 127 else (-x if c & 128 else x)
    return v


def scale_for(amax, fmt):
    """Smallest 2^e, e >= -126, with amax <= QMAX 2^e."""
    e = -126
    while amax > QMAX[fmt] * 2.0 ** e:
        e += 1
    return 2.0 ** e


def encode(x, fmt):
    """float64 array (in units of the scale) -> uint8 codes, nearest, ties to even; saturating."""
    x = np.asarray(x, np.float64)
    if fmt == "int8":
        return np.rint(np.clip(np.where(np.isnan(x), 0, x), -127, 127)).astype(np.int8).view(np.uint8)
    pos = e4m3_table()[:127]
    a = np.clip(np.abs(x), 0, 448)
    a = np.where(np.isnan(x), 0, a)
    hi = np.clip(np.searchsorted(pos, a), 1, 126)
    lo = hi - 1
    dl, dh = a - pos[lo], pos[hi] - a
    pick = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi))).astype(np.uint8)
    pick = pick | np.where(np.signbit(x), 128, 0).astype(np.uint8)
    return np.where(np.isnan(x), np.uint8(0x7F), pick).astype(np.uint8)


def decode(c, fmt):
    return c.view(np.int8).astype(np.float64) if fmt == "int8" else e4m3_table()[c]


class Model:
    """A pool in numpy with the append rule written out token by token."""

    def __init__(self, codes, scales, fmt):
        self.c, self.s, self.fmt = codes.copy(), scales.astype(np.float64).copy(), fmt
        self.page = codes.shape[3]

    def append(self, k, v, table, starts, first):
        x = np.stack([k, v], 1).astype(np.float64)            # [rows, 2, hk, d]
        for b in range(len(first)):
            rows = [(r, first[b] + r - starts[b]) for r in range(starts[b], starts[b + 1])]
            rows = [(r, p) for r, p in rows if p >= 0]
            for pg in sorted({p // self.page for _, p in rows}):
                here = [(r, p % self.page) for r, p in rows if p // self.page == pg]
                keep, page = here[0][1], table[b][pg]
                for kv in range(2):
                    for h in range(x.shape[2]):
                        new = np.stack([x[r, kv, h] for r, _ in here])
                        fin = np.abs(new[np.isfinite(new)])
                        sc = scale_for(fin.max() if fin.size else 0.0, self.fmt)
                        if keep:
                            old = self.s[page, kv, h]
                            sc = max(sc, old)
                            if sc != old:
                                held = decode(self.c[page, kv, h, :keep], self.fmt) * old
                                self.c[page, kv, h, :keep] = encode(held / sc, self.fmt)
                        self.s[page, kv, h] = sc
                        for (r, slot), val in zip(here, new):
                            self.c[page, kv, h, slot] = encode(val / sc, self.fmt)


def values(codes, scales, table_row, n, fmt):
    """Keys and values of a sequence's first n positions: float64 [n, 2, hk, d] (torch, CPU)."""
    page = codes.shape[3]
    ids = [int(i) for i in table_row[:-(-n // page)]]
    c = codes.view(torch.int8)[ids].cpu().numpy().view(np.uint8)
    x = decode(c, fmt) * scales[ids].cpu().double().numpy()[..., None, None]
    x = np.moveaxis(x, 3, 1).reshape(len(ids) * page, *x.shape[1:3], x.shape[4])
    return torch.from_numpy(x[:n])


def attend(q, kvs, starts, first, *, kv_lens=None, sm_scale=None, causal=True, window=0):
    """out, lse and the scale of rounding errors (sum p |v|, largest sum |q k|) of every row, in 64 bits."""
    rows, hq, d = q.shape
    out, lse = torch.zeros(rows, hq, d, dtype=torch.float64), torch.full((rows, hq), -np.inf, dtype=torch.float64)
    mag, dots = torch.zeros_like(out), torch.zeros_like(lse)
    sm_scale = d ** -0.5 if sm_scale is None else sm_scale
    q = q.detach().cpu().double()
    for b, kv in enumerate(kvs):
        r0, r1 = starts[b], starts[b + 1]
        length = first[b] + r1 - r0 if kv_lens is None else kv_lens[b]
        length = max(0, length)
        if r1 == r0:
            continue
        g = hq // kv.shape[2]
        k, v = (kv[:length, i].repeat_interleave(g, 1) for i in (0, 1))
        p = torch.arange(first[b], first[b] + r1 - r0)[:, None]
        j = torch.arange(length)[None]
        seen = (p >= 0) & (j >= 0)
        if causal:
            seen = seen & (j <= p)
        if window:
            seen = seen & (j > p - window)
        qk = torch.einsum("rhd,jhd->hrj", q[r0:r1], k) * sm_scale
        ab = torch.einsum("rhd,jhd->hrj", q[r0:r1].abs(), k.abs()) * sm_scale
        s = qk.masked_fill(~seen, -np.inf)
        if length:
            l = torch.logsumexp(s, 2)
            w = torch.exp(s - torch.where(torch.isinf(l), 0.0, l)[..., None])
            out[r0:r1] = torch.einsum("hrj,jhd->rhd", w, v)
            mag[r0:r1] = torch.einsum("hrj,jhd->rhd", w, v.abs())
            lse[r0:r1] = l.T
            dots[r0:r1] = ab.masked_fill(~seen, 0).amax(2).T
    return out, lse, mag, dots


FIX, FIXU = 36, 24


def fixed(p):
    p = np.asarray(p, np.float64)
    return np.rint(np.clip(np.where(p > 0, p, 0.0), 0, 1) * 2.0 ** FIX).astype(np.int64)


def verify(tokens, target, draft, uniforms, sample_u, starts):
    """The rule in Python's whole numbers."""
    out, acc = [], []
    vocab = target.shape[1]
    for b in range(len(starts) - 1):
        r0, n = starts[b], starts[b + 1] - starts[b]
        if n == 0:
            acc.append(0)
            continue
        a, weight = 0, None
        while a < n - 1:
            p, x = fixed(target[r0 + a]), int(tokens[r0 + a + 1])
            q = np.zeros_like(p)
            if draft is not None:
                q = fixed(draft[r0 + a])
            elif 0 <= x < vocab:
                q[x] = 1 << FIX
            u = int(np.floor(float(uniforms[r0 + a]) * 2.0 ** FIXU))
            if 0 <= x < vocab and u * int(q[x]) < int(p[x]) << FIXU:
                a += 1
                continue
            weight = np.maximum(p - q, 0)
            if weight.sum() == 0:
                weight = p
            break
        if weight is None:
            weight = fixed(target[r0 + a])
        total, token = int(weight.sum()), -1
        if total:
            bar = (int(np.floor(float(sample_u[b]) * 2.0 ** FIXU)) * total) >> FIXU
            token = int(np.searchsorted(np.cumsum(weight), bar, side="right"))
        out += [int(t) for t in tokens[r0 + 1:r0 + 1 + a]] + [token] + [-1] * (n - a - 1)
        acc.append(a)
    return out, acc
