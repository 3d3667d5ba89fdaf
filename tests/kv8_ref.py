"""Plain 64-bit statement of the 8-bit KV pages: quantisation and append token by token, attention row by row (CPU)."""
import math

import torch

PAGE = 16
LEVELS = torch.tensor(sorted(m * 2.0 ** (e - 10) if e else m * 2.0 ** -9 for e in range(16) for m in (range(8, 16) if e else range(8))),
                      dtype=torch.float64)[:-1]                       # 0 .. 448


def exponent(top):
    """smallest e in [-64, 56] with top <= 448 * 2^e"""
    e = -64
    while e < 56 and top > 448 * 2.0 ** e:
        e += 1
    return e


def round8(x, e):
    """float64 x to e4m3(code) * 2^e, nearest, ties to even"""
    a = (x.abs() * 2.0 ** -e).clamp_max(448.0)
    hi = torch.searchsorted(LEVELS, a).clamp(1, LEVELS.numel() - 1)
    dl, dh = a - LEVELS[hi - 1], LEVELS[hi] - a
    pick = torch.where((dh < dl) | ((dh == dl) & (hi % 2 == 0)), hi, hi - 1)
    return (LEVELS[pick] * 2.0 ** e).copysign(x)


def norm(x, w, eps):
    return x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()


def rotate(x, cos, sin, interleaved):
    """x [..., D] float64, cos / sin [..., D / 2]"""
    h = x.shape[-1] // 2
    i = torch.arange(h)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + h)
    y = torch.empty_like(x)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * cos.double() - b * sin.double(), a * sin.double() + b * cos.double()
    return y


class Pages:
    """vals float64 [blocks, H, 2, 16, D], exps [blocks, H, 2]"""

    def __init__(self, blocks, H, D):
        self.vals = torch.zeros(blocks, H, 2, PAGE, D, dtype=torch.float64)
        self.exps = torch.full((blocks, H, 2), -64, dtype=torch.int64)

    def append(self, K, V, slots):
        """K, V float64 [N, H, D] as they are to be stored"""
        goes = {}
        for i, s in enumerate(slots.tolist()):
            if 0 <= s < self.vals.shape[0] * PAGE:
                goes.setdefault(s // PAGE, {})[s % PAGE] = i             # (the last token of a slot)
        for page, rows in goes.items():
            r, tok = list(rows), list(rows.values())
            for kvi, X in enumerate((K, V)):
                for h in range(self.vals.shape[1]):
                    unit = self.vals[page, h, kvi]
                    new = X[tok, h]
                    fin = torch.where(new.isfinite(), new, torch.zeros_like(new))
                    e = exponent(float(fin.abs().max()))
                    if 0 in rows:
                        unit.zero_()
                    else:
                        e = max(e, int(self.exps[page, h, kvi]))
                    unit[r] = torch.where(new.isnan(), torch.zeros_like(new), new)
                    self.vals[page, h, kvi] = round8(unit, e)
                    self.exps[page, h, kvi] = e

    def dense(self):
        return self.vals[:, :, 0].transpose(1, 2), self.vals[:, :, 1].transpose(1, 2)


def attend(q, K, V, pos, scale, start=0, window=0):
    """q float64 [n, Hq, D] at positions pos (list) over K, V float64 [L, H, D] -> (out, sum p |v|, largest sum |q k| scale) per row"""
    n, Hq, D = q.shape
    L, H, _ = K.shape
    out, mag = torch.zeros_like(q), torch.zeros_like(q)
    wide = torch.zeros(n, Hq, dtype=torch.float64)
    for i, p in enumerate(pos):
        lo, hi = max(start, p - window + 1 if window else 0, 0), min(p + 1, L)
        if hi <= lo:
            continue
        for h in range(H):
            g = slice(h * (Hq // H), (h + 1) * (Hq // H))
            s = q[i, g] @ K[lo:hi, h].T * scale
            w = torch.softmax(s, -1)
            out[i, g], mag[i, g] = w @ V[lo:hi, h], w @ V[lo:hi, h].abs()
            wide[i, g] = (q[i, g].abs() @ K[lo:hi, h].abs().T).amax(-1) * scale
    return out, mag, wide


def allowed(out, mag, wide, keys, D):
    """how far a kernel's BF16 output may be from attend()'s: probabilities rounded to BF16 (2^-8 of each), the output rounded to BF16
    (2^-8), scores summed in fp32 over D products (each sum off by at most D 2^-24 of its absolute sum; twice, since the maximum is
    subtracted), the sum of the probabilities over `keys` (2^-24 each), the exponential's argument in base 2 (a rounding of the product
    with the scale and one of the difference) and itself (2^-21)"""
    rel = 2.0 ** -8 + 2 * (D + 4) * 2.0 ** -24 * wide[..., None] + keys * 2.0 ** -24 + 2.0 ** -21
    return mag * rel * 1.01 + 2.0 ** -8 * out.abs() + 1e-30
