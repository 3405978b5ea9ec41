"""4-bit K/V pages and attention over them, in numpy and float64, one step after
the other from the definitions (the format: include/helm_b200.h)."""
from __future__ import annotations

import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def _e4m3_table() -> np.ndarray:
    """Values of the e4m3 codes 0x00 .. 0x7e."""
    c = np.arange(0x7F)
    e, m = c >> 3, c & 7
    return np.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * 2.0 ** (e.astype(float) - 7))


E4M3 = _e4m3_table()


def _nearest(x: np.ndarray, levels: np.ndarray) -> np.ndarray:
    """Index of the level nearest to x >= 0; of two at the same distance the even one."""
    hi = np.clip(np.searchsorted(levels, x), 0, len(levels) - 1)
    lo = np.maximum(hi - 1, 0)
    dl, dh = np.abs(x - levels[lo]), np.abs(levels[hi] - x)
    low = (dl < dh) | ((dl == dh) & (lo % 2 == 0))
    return np.where(low, lo, hi)


def e4m3_values(codes: np.ndarray) -> np.ndarray:
    mag = np.append(E4M3, np.nan)[codes & 0x7F]
    return np.where(codes & 0x80, -mag, mag)


def quantise(x: np.ndarray):
    """x [..., D] -> (codes [..., D], scale bytes [..., D / 16]), both uint8."""
    b = np.asarray(x, dtype=np.float64).reshape(*x.shape[:-1], -1, 16)
    nan = np.isnan(b).any(-1)
    amax = np.where(nan, 0.0, np.abs(np.where(np.isnan(b), 0.0, b)).max(-1))
    s8 = np.where(nan, 0x7F, _nearest(np.minimum(amax / 6.0, 448.0), E4M3)).astype(np.uint8)
    s = np.where(nan, 1.0, e4m3_values(s8))[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        r = np.where(s > 0, np.abs(b) / s, 0.0)
    c = _nearest(np.minimum(np.where(np.isnan(r), 0.0, r), 6.0), E2M1).astype(np.uint8)
    c = c | (np.signbit(b).astype(np.uint8) << 3)
    return c.reshape(x.shape), s8


def values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    v = np.where(codes & 8, -E2M1[codes & 7], E2M1[codes & 7])
    return (v.reshape(*scales.shape, 16) * e4m3_values(scales)[..., None]).reshape(codes.shape)


def tile_bytes(d: int, t: int):
    """Byte offsets in a tile of token t's K code bytes, V code bytes, K scales, V scales."""
    row = t ^ (((t >> 2) & 1) << 1 | (t >> 3) & 1)
    kc, vc, ks, vs = [], [], [], []
    for i in range(d // 2):
        j = i // 16
        if d == 256:
            j ^= 4 * (t & 1)
        kc.append(row * d // 2 + 16 * j + i % 16)
        u = i // (d // 16)
        if d == 128:
            u ^= 4 * ((t >> 2) & 1)
        elif d == 256:
            u ^= 2 * ((t >> 2) & 3)
        vc.append(8 * d + row * d // 2 + u * (d // 16) + i % (d // 16))
    for g in range(d // 16):
        # the lane that reads dims of block g, and the block's place among that lane's blocks
        if d == 64:
            c, k = g, 0
        elif d == 128:
            c, k = g // 2, g % 2
        else:
            c, k = (g % 8) // 2, g % 2 + 2 * (g // 8)
        pair = 2 * (t >> 2) + (t & 1)
        per = d // 64  # blocks of a lane
        ks.append(16 * d + (pair * 4 + c) * 2 * per + ((t >> 1) & 1) * per + k)
        vs.append(17 * d + 16 * g + t)
    return tuple(np.array(x) for x in (kc, vc, ks, vs))


def write_rows(pool: np.ndarray, rows, k: np.ndarray, v: np.ndarray, page_size: int) -> None:
    """Quantises k, v [N, Hkv, D] into pool rows (negative rows skipped)."""
    d = k.shape[-1]
    at = [tile_bytes(d, t) for t in range(16)]
    for x, ci, si in ((k, 0, 2), (v, 1, 3)):
        codes, scales = quantise(x)
        packed = codes[..., 0::2] | (codes[..., 1::2] << 4)
        for n, row in enumerate(rows):
            if row < 0:
                continue
            page, r = divmod(int(row), page_size)
            off = at[r % 16]
            for h in range(k.shape[1]):
                pool[page, h, r // 16][off[ci]] = packed[n, h]
                pool[page, h, r // 16][off[si]] = scales[n, h]


def read_rows(pool: np.ndarray, rows, page_size: int):
    """K, V float64 [N, Hkv, D] of pool rows (zeros for negative rows)."""
    d = pool.shape[-1] // 18
    at = [tile_bytes(d, t) for t in range(16)]
    out = []
    for ci, si in ((0, 2), (1, 3)):
        x = np.zeros((len(rows), pool.shape[1], d))
        for n, row in enumerate(rows):
            if row < 0:
                continue
            page, r = divmod(int(row), page_size)
            off = at[r % 16]
            packed = pool[page, :, r // 16][:, off[ci]]
            codes = np.stack([packed & 15, packed >> 4], -1).reshape(packed.shape[0], d)
            x[n] = values(codes, pool[page, :, r // 16][:, off[si]])
        out.append(x)
    return out


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float, softcap: float = 0.0,
              mask: np.ndarray | None = None):
    """q [Hq, D], k, v [T, Hkv, D], mask [T] or None -> (O [Hq, D], LSE [Hq], A [Hq, D]) with
    A = sum p |v| / l, the size of what O sums up.  Keys masked with -inf do not take part."""
    hq, d = q.shape
    hkv = k.shape[1]
    o, lse, size = np.zeros((hq, d)), np.full(hq, -np.inf), np.zeros((hq, d))
    use = np.ones(k.shape[0], bool) if mask is None else mask > -np.inf
    if not use.any():
        return o, lse, size
    for h in range(hq):
        kv = h // (hq // hkv)
        s = k[use, kv] @ q[h] * scale
        if softcap > 0:
            s = softcap * np.tanh(s / softcap)
        if mask is not None:
            s = s + mask[use]
        m = s.max()
        p = np.exp(s - m)
        o[h] = p @ v[use, kv] / p.sum()
        size[h] = p @ np.abs(v[use, kv]) / p.sum()
        lse[h] = m + np.log(p.sum())
    return o, lse, size
