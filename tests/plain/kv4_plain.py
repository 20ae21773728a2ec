"""A key/value cache held in 4 bits, and attention over it, in numpy: quantising in the 32-bit steps that the format names,
everything else in float64.  Nothing of the package is used."""
import numpy as np

LARGEST, NAN_WORD = 2112.0, 0x7FE0


def place(i):
    return (6 + 4 * (i // 2) + 16 * (i % 2)) % 32


def row_bytes(dim):
    return dim // 2 + dim // 16


def scale_table():
    """Every scale there is, ascending: the half-precision numbers whose low five bits are zero, up to the largest."""
    bits = np.arange(0, 0x7C00, 32, dtype=np.uint16)
    values = bits.view(np.float16).astype(np.float64)
    return values[values <= LARGEST], bits[values <= LARGEST]


def quantise(x):
    """float32 [..., dims] -> (numbers int [..., dims], scale words int [..., dims / 32])."""
    g = np.asarray(x, dtype=np.float32).reshape(*x.shape[:-1], -1, 32)
    finite = np.isfinite(g).all(-1)
    g = np.where(finite[..., None], g, np.float32(0))
    lo, hi = np.minimum(g.min(-1), 0), np.maximum(g.max(-1), 0)
    with np.errstate(over="ignore"):
        want = np.minimum((hi - lo) / np.float32(15), np.float32(LARGEST))
    values, bits = scale_table()
    at = np.searchsorted(values, want.astype(np.float64))              # the smallest scale that is no less
    s = values[at].astype(np.float32)
    unit = np.where(s > 0, s, np.float32(1))
    z = np.clip(np.rint(-lo / unit), 0, 15)
    n = np.clip(np.rint(g / unit[..., None]) + z[..., None], 0, 15).astype(np.int64)
    words = np.where(finite, bits[at].astype(np.int64) | z.astype(np.int64), NAN_WORD)
    return n.reshape(x.shape), words


def values(numbers, words):
    words = np.asarray(words)
    s = (words & 0x7FE0).astype(np.uint16).view(np.float16).astype(np.float64)
    g = numbers.reshape(*numbers.shape[:-1], -1, 32).astype(np.float64)
    return (s[..., None] * (g - (words & 15)[..., None])).reshape(numbers.shape)


def put(buffer, at, number_index, number):
    """Store one number as `number_index` of the word at byte `at`, bit by bit."""
    for bit in range(4):
        b = (place(number_index) + bit) % 32
        byte = at + b // 8
        buffer[byte] = (int(buffer[byte]) & ~(1 << b % 8)) | (((int(number) >> bit) & 1) << b % 8)


class Cache:
    """Both caches, uint8 [pages, heads, page, row bytes], every byte `fill` where nothing is stored."""

    def __init__(self, pages, heads, page, dim, fill=255):
        self.shape, self.page, self.dim, self.heads = (pages, heads, page, row_bytes(dim)), page, dim, heads
        self.keys = np.full(self.shape, fill, dtype=np.uint8)
        self.values = np.full(self.shape, fill, dtype=np.uint8)

    def store(self, page_of, slot, k, v):
        """k, v float32 [heads, dim] into a slot."""
        dim, page = self.dim, self.page
        for h in range(self.heads):
            n, words = quantise(k[h][None])
            flat = self.keys[page_of, h].reshape(-1)
            for d in range(dim):
                put(flat, slot * dim // 2 + d // 8 * 4, d % 8, n[0, d])
            for g in range(dim // 32):
                flat[page * dim // 2 + 2 * (slot * (dim // 32) + g):][:2] = [words[0, g] & 255, words[0, g] >> 8]
            n, words = quantise(v[h][None])
            flat = self.values[page_of, h].reshape(-1)
            for d in range(dim):
                put(flat, (slot // 8 * dim + d) * 4, slot % 8, n[0, d])
            for g in range(dim // 32):
                flat[page * dim // 2 + 2 * ((slot // 8 * (dim // 32) + g) * 8 + slot % 8):][:2] = [words[0, g] & 255, words[0, g] >> 8]


def pages_of(rows, page, dim, keys):
    """Whole pages at once: float32 rows [pages, heads, page, dim] -> bytes [pages, heads, page, row bytes]."""
    n, words = quantise(rows)
    p, h = rows.shape[:2]
    if keys:
        eights = n.reshape(p, h, page * dim // 8, 8)
    else:
        eights = n.reshape(p, h, page // 8, 8, dim).swapaxes(3, 4).reshape(p, h, page * dim // 8, 8)
        words = words.reshape(p, h, page // 8, 8, dim // 32).swapaxes(3, 4)
    word = np.zeros(eights.shape[:-1], dtype=np.uint64)
    for i in range(8):
        at, e = np.uint64(place(i)), eights[..., i].astype(np.uint64)
        word |= ((e << at) | (e >> (np.uint64(32) - at))) & np.uint64(0xFFFFFFFF)
    packed = word.astype("<u4").view(np.uint8).reshape(p, h, -1)
    scales = np.ascontiguousarray(words.reshape(p, h, -1).astype("<u2")).view(np.uint8).reshape(p, h, -1)
    return np.concatenate([packed, scales], axis=-1).reshape(p, h, page, row_bytes(dim))


def attention(q, k, v, pos, window, scale):
    """One token: q [heads, dim], k and v [positions, kv heads, dim] float64, positions 0 .. pos.  Returns the output and, for
    bounds, sum p |v|, the largest sum_d |q_d k_d| scale of a seen position, a head, and sum |v|, the largest max |q| sum |k_d| scale."""
    nh, dim = q.shape
    nkv = k.shape[1]
    out, weight, score, size, spread = np.zeros((nh, dim)), np.zeros((nh, dim)), np.zeros((nh, 1)), np.zeros((nh, dim)), np.zeros((nh, 1))
    if pos < 0:
        return out, weight, score, size, spread
    lo = max(0, pos + 1 - window) if window else 0
    for h in range(nh):
        kh, vh = k[lo:pos + 1, h // (nh // nkv)], v[lo:pos + 1, h // (nh // nkv)]
        s = kh @ q[h] * scale
        e = np.exp(s - s.max())
        p = e / e.sum()
        out[h], weight[h], score[h] = p @ vh, p @ np.abs(vh), (np.abs(kh) @ np.abs(q[h])).max() * scale
        size[h], spread[h] = np.abs(vh).sum(0), np.abs(q[h]).max() * np.abs(kh).sum(-1).max() * scale
    return out, weight, score, size, spread
