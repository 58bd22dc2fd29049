"""The norm / rotation / block-scaled cache operators written from their
definitions in float64, for the tests."""

from __future__ import annotations

import numpy as np

E4M3_MAX = 448.0


def e4m3_values() -> np.ndarray:
    """The value of each of the 256 e4m3 codes (NaN for 0x7f and 0xff)."""
    c = np.arange(256)
    sign = np.where(c & 0x80, -1.0, 1.0)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m / 8.0 * 2.0 ** -6, (1 + m / 8.0) * 2.0 ** (e - 7.0))
    v = sign * v
    v[(c & 0x7F) == 0x7F] = np.nan
    return v


_VALUES = e4m3_values()


def from_e4m3(codes: np.ndarray) -> np.ndarray:
    return _VALUES[codes]


def to_e4m3(x: np.ndarray) -> np.ndarray:
    """Codes of x: nearest, ties to even, saturating at +-448; NaN -> 0x7f."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(x), E4M3_MAX)
    _, e = np.frexp(np.maximum(np.nan_to_num(a), 2.0 ** -6))  # a in [2^(e-1), 2^e)
    step = np.exp2(e - 4.0)
    q = np.rint(np.nan_to_num(a) / step) * step
    _, e = np.frexp(np.maximum(q, 2.0 ** -6))
    normal = q >= 2.0 ** -6
    m = np.where(normal, q / np.exp2(e - 4.0) - 8, q * 2.0 ** 9).astype(np.int64)
    code = np.where(normal, ((e - 1 + 7) << 3) | m, m)
    code = code | np.where(np.signbit(x), 0x80, 0)
    return np.where(np.isnan(x), 0x7F, code).astype(np.uint8)


def norm_rope(x, weight, cos_sin, positions, interleaved, eps):
    """x [T, H, D] -> float64 [T, H, D]."""
    y = np.asarray(x, np.float64).copy()
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    r = cos_sin.shape[1]
    row = np.asarray(cos_sin, np.float64)[positions][:, None, :]
    c, s = row[..., : r // 2], row[..., r // 2:]
    i = np.arange(r // 2)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
    a, b = y[..., ia].copy(), y[..., ib].copy()
    y[..., ia] = a * c - b * s
    y[..., ib] = b * c + a * s
    return y


def power_of_two(amax):
    """The smallest power of two s >= 2^-126 with amax <= 448 s; 0 for 0."""
    if amax == 0:
        return 0.0
    s = 2.0 ** -126
    while amax > E4M3_MAX * s:
        s *= 2
    return s


def append_block(x, cache, scales, slots, live=None):
    """One call's append of x [T, Hkv, D] (float64) into codes `cache` [N, Hkv,
    16, D] with `scales` [N, Hkv], both changed in place; slots outside the
    pool and tokens that are not `live` append nothing."""
    rows = {}
    for t, s in enumerate(slots):
        if 0 <= s < cache.shape[0] * 16 and (live is None or live[t]):
            rows[(s // 16, s % 16)] = t
    for b in sorted({k[0] for k in rows}):
        offs = {o: t for (bb, o), t in rows.items() if bb == b}
        for h in range(cache.shape[1]):
            new = {o: x[t, h] for o, t in offs.items()}
            amax = max((np.abs(v[np.isfinite(v)]).max(initial=0.0) for v in new.values()), default=0.0)
            need = power_of_two(np.float32(amax))
            old = float(scales[b, h])
            old = old if 0 < old < np.inf else 0.0
            s = need if 0 in offs else max(old, need)
            if 0 not in offs and s > old:
                for o in range(16):
                    if o not in new:
                        cache[b, h, o] = to_e4m3(np.float32(from_e4m3(cache[b, h, o]) * (old / s)))
            for o, v in new.items():
                cache[b, h, o] = to_e4m3(v / s if s > 0 else v)
            scales[b, h] = s


def attention(q, kc, vc, ks, vs, tables, lens, scale):
    """Decode attention over block-scaled codes; float64 [S, H, D]."""
    S, H, D = q.shape
    hkv = kc.shape[1]
    out = np.zeros((S, H, D))
    for s in range(S):
        n = int(lens[s])
        if n == 0:
            continue
        ids = tables[s, : (n + 15) // 16]
        k = (from_e4m3(kc[ids]) * ks[ids].astype(np.float64)[..., None, None]).transpose(1, 0, 2, 3)
        v = (from_e4m3(vc[ids]) * vs[ids].astype(np.float64)[..., None, None]).transpose(1, 0, 2, 3)
        k = k.reshape(hkv, -1, D)[:, :n]
        v = v.reshape(hkv, -1, D)[:, :n]
        qq = np.asarray(q[s], np.float64).reshape(hkv, H // hkv, D)
        logits = np.einsum("hgd,htd->hgt", qq, k) * scale
        p = np.exp(logits - logits.max(-1, keepdims=True))
        out[s] = (np.einsum("hgt,htd->hgd", p, v) / p.sum(-1, keepdims=True)).reshape(H, D)
    return out
