"""The 4-bit format and its operators restated in numpy float64, for the tests of ``q4``.

Written from the format's definition (include/hla_s6.h), byte by byte: ``pack_row`` / ``unpack_cache`` place the
codes, ``quantize`` makes them, ``attention`` and ``rope`` are the operators.  Nothing here imports the package.
"""
import numpy as np

E4M3 = np.array([((b & 7) * 2.0 ** -9) if (b >> 3) & 15 == 0 else (1 + (b & 7) / 8) * 2.0 ** (((b >> 3) & 15) - 7)
                 for b in range(127)])       # bytes 0x00 .. 0x7e; 0x7f is NaN


def e4m3_byte(a):
    """Nearest e4m3 byte of nonnegative values, ties to the even byte, saturated at 448 (0x7e)."""
    a = np.minimum(np.asarray(a, dtype=np.float64), 448.0)
    hi = np.searchsorted(E4M3, a, side='left').clip(0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - E4M3[lo], E4M3[hi] - a
    return np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi).astype(np.uint8)


def bf16(x):
    """Round float64 / float32 to bf16 (ties to even), returned as float64."""
    x = np.asarray(x, dtype=np.float64)
    m, e = np.frexp(x)
    return np.ldexp(np.rint(m * 256), e - 8)


def quantize(x, ts):
    """``[..., C]`` -> codes 1..15 and scale bytes ``[..., C / 32]``."""
    g = np.asarray(x, dtype=np.float64).reshape(*x.shape[:-1], -1, 32)
    byte = e4m3_byte(np.abs(g).max(-1) / 7 / ts)
    step = E4M3[byte][..., None] * ts
    with np.errstate(divide='ignore', invalid='ignore'):
        q = np.where(step > 0, np.clip(np.rint(g / step), -7, 7), 0)
    return (q + 8).astype(np.int64).reshape(x.shape), byte


def stored(x, ts):
    """The values ``x`` is stored as."""
    n, byte = quantize(x, ts)
    return (n - 8) * np.repeat(E4M3[byte], 32, -1) * ts


def words(n):
    """codes ``[..., C]`` -> bytes ``[..., C / 2]`` (4 bytes per 8 columns: nibble i column 2i, i + 4 column 2i + 1)."""
    n = n.reshape(*n.shape[:-1], -1, 8)
    w = sum(n[..., 2 * i] << (4 * i) for i in range(4)) + sum(n[..., 2 * i + 1] << (16 + 4 * i) for i in range(4))
    return w.astype(np.uint32)[..., None].view(np.uint8).reshape(*n.shape[:-2], -1)


def codes(b):
    """The inverse of ``words``: bytes ``[..., 4 m]`` -> ``n - 8`` ``[..., 8 m]``."""
    w = np.ascontiguousarray(b).view(np.uint32).astype(np.int64)
    cols = [((w >> (4 * (c // 2) + 16 * (c % 2))) & 15) - 8 for c in range(8)]
    return np.stack(cols, -1).reshape(*w.shape[:-1], -1)


def tile_views(page_bytes, W):
    """Views of the tiles of pages ``[..., page * 17 W / 16]``: K codes, V codes, K scales, V scales."""
    G = W // 32
    t = page_bytes.reshape(-1, 17 * W)
    return (t[:, :8 * W].reshape(-1, G, 16, 16), t[:, 8 * W:16 * W].reshape(-1, W // 8, 16, 4),
            t[:, 16 * W:16 * W + 16 * G].reshape(-1, 16, G), t[:, 16 * W + 16 * G:].reshape(-1, G, 16))


def put_row(cache, W, page, slot, k, v, k_ts, v_ts):
    """Store row ``k, v`` (float64 [W]) at ``slot`` of ``cache`` uint8 [nb, 1, page, 17 W / 16] (in place)."""
    kn, kb = quantize(k, k_ts)
    vn, vb = quantize(v, v_ts)
    kc, vc, ks, vs = tile_views(cache[slot // page].reshape(-1), W)
    t, r = (slot % page) // 16, slot % 16
    kc[t, :, r] = words(kn).reshape(-1, 16)
    vc[t, :, r] = words(vn).reshape(-1, 4)
    ks[t, r] = kb
    vs[t, :, r] = vb


def random_cache(rng, nb, page, W):
    """Random codes 1..15 and random scales of ordinary size in every row; and the values (float64 [nb, page, W])."""
    cache = np.zeros((nb, 1, page, 17 * W // 16), dtype=np.uint8)
    kc, vc, ks, vs = tile_views(cache.reshape(-1), W)
    n = kc.shape[0]
    k, v = rng.integers(1, 16, (n, 16, W)), rng.integers(1, 16, (n, 16, W))
    kb, vb = rng.integers(24, 56, (n, 16, W // 32)), rng.integers(24, 56, (n, 16, W // 32))
    kc[:] = words(k).reshape(n, 16, -1, 16).transpose(0, 2, 1, 3)
    vc[:] = words(v).reshape(n, 16, -1, 4).transpose(0, 2, 1, 3)
    ks[:] = kb
    vs[:] = vb.transpose(0, 2, 1)
    val = lambda c, b: ((c - 8) * np.repeat(E4M3[b], 32, -1)).reshape(nb, page, W)
    return cache, val(k, kb), val(v, vb)


def unpack_cache(cache, W):
    """cache [nb, 1, page, 17 W / 16] -> K, V values without the tensor scales (float64 [nb, page, W])."""
    nb, _, page, _ = cache.shape
    kc, vc, ks, vs = tile_views(np.ascontiguousarray(cache).reshape(-1), W)
    n = kc.shape[0]
    scale = np.append(E4M3, np.nan)
    k = codes(kc.transpose(0, 2, 1, 3).reshape(n, 16, -1)) * np.repeat(scale[ks & 127], 32, -1)
    v = codes(vc.transpose(0, 2, 1, 3).reshape(n, 16, -1)) * np.repeat(scale[vs.transpose(0, 2, 1) & 127], 32, -1)
    return k.reshape(nb, page, W), v.reshape(nb, page, W)


def unpack_weight(packed, N, K):
    """packed [N / 16, K / 128, 1088] -> float64 [N, K] without the tensor scale."""
    n, k, _ = packed.shape
    c = codes(np.ascontiguousarray(packed[..., :1024]).reshape(n, k, 2, 8, 4, 16))
    s = E4M3[packed[..., 1024:].reshape(n, k, 8, 4, 2)].transpose(0, 1, 4, 2, 3)
    return (c * s[..., None]).reshape(n, k, 16, 128).transpose(0, 2, 1, 3).reshape(16 * n, 128 * k)[:N, :K]


def rope(x, table, pos):
    """The committed rotation of ``x [T, W]`` in the bf16 operation order."""
    half = x.shape[1] // 2
    c, s = table[pos][:, :half], table[pos][:, half:]
    a, b = x[:, :half], x[:, half:]
    return np.concatenate((bf16(bf16(a * c) + bf16(-b * s)), bf16(bf16(b * c) + bf16(a * s))), 1)


def attention(q, k, v, scale):
    """One row: q [H, W] over k, v [n, W] -> o [H, W], lse [H], and what the error bounds need: sum p |v| [H, W]
    and the largest sum |q k| scale [H]."""
    H, W = q.shape
    if k.shape[0] == 0:
        return np.zeros((H, W)), np.full(H, -np.inf), np.zeros((H, W)), np.zeros(H)
    s = q @ k.T * scale
    m = s.max(1, keepdims=True)
    p = np.exp(s - m)
    tot = p.sum(1, keepdims=True)
    return p @ v / tot, (m + np.log(tot))[:, 0], p @ np.abs(v) / tot, (np.abs(q) @ np.abs(k).T * abs(scale)).max(1)
