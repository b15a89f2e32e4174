"""The 4-bit KV cache in 64 bits, from its definition (include/ribn_b200.h, ribn_b200/csrc/kvq4.cuh): quantiser, byte order, attention."""
import numpy as np

PAGE = 16


def scale_of(x):
    """x of the largest magnitude (the first) / -8 as binary16, to seven significant bits, half away from zero, at most 896."""
    s = np.float16(np.float64(x) / -8.0) if np.isfinite(x) else np.float16(-np.sign(x) * np.inf)
    bits = int(np.frombuffer(np.float16(s).tobytes(), np.uint16)[0])
    size = min(((bits & 0x7fff) + 8) & ~15, 0x6300)
    return float(np.frombuffer(np.uint16(size).tobytes(), np.float16)[0]) * (-1.0 if bits & 0x8000 else 1.0)


def quantise(rows):
    """rows [n][h][d] -> codes 0..15 [n][h][d], scales [n][h][d / 32], both of the definition's exact arithmetic."""
    x = np.nan_to_num(np.asarray(rows, np.float64), nan=0.0, posinf=np.inf, neginf=-np.inf)
    n, h, d = x.shape
    g = x.reshape(n, h, d // 32, 32)
    place = np.argmax(np.abs(g), axis=3)   # the first of the largest
    top = np.take_along_axis(g, place[..., None], axis=3)[..., 0]
    scales = np.vectorize(scale_of, otypes=[np.float64])(top)
    with np.errstate(invalid="ignore", divide="ignore"):
        q = np.floor(g / scales[..., None] + 0.5)
    q = np.where(scales[..., None] == 0, 0.0, np.clip(q, -8, 7))
    return (q + 8).astype(np.uint8).reshape(n, h, d), scales


def values(codes, scales):
    n, h, d = codes.shape
    return ((codes.astype(np.float64) - 8).reshape(n, h, d // 32, 32) * scales[..., None]).reshape(n, h, d)


class Arena:
    """The bytes of an arena and the values they stand for, one token at a time."""

    def __init__(self, pages, kv_heads, head_dim):
        self.bytes = np.zeros((pages, kv_heads, 18 * head_dim), np.uint8)
        self.k = np.zeros((pages * PAGE, kv_heads, head_dim))
        self.v = np.zeros_like(self.k)

    def put(self, slot, k_codes, k_scales, v_codes, v_scales):
        pages, heads, record = self.bytes.shape
        d, page, j = record // 18, slot // PAGE, slot % PAGE
        words = min(4, d // 32)
        self.k[slot], self.v[slot] = values(k_codes[None], k_scales[None])[0], values(v_codes[None], v_scales[None])[0]
        c, t, e = j // 8, j % 8 // 2, j % 2
        for h in range(heads):
            r = self.bytes[page, h]
            for G in range(d // 32):
                sub, w = divmod(G, words)
                for i in range(32):
                    # K: eight dimensions per word; V: the half word of dimension i % 8
                    at = sub * 256 * words + j * 16 * words + (i // 8) * 4 * words + w * 4 + i % 8 // 2
                    shift = 4 * (i % 2)
                    r[at] = r[at] & (0xF0 >> shift) | int(k_codes[h, 32 * G + i]) << shift
                    at = 8 * d + sub * 256 * words + c * 128 * words + (i % 8) * 16 * words + t * 4 * words + w * 4 + e * 2 + i // 16
                    shift = 4 * (i // 8 % 2)
                    r[at] = r[at] & (0xF0 >> shift) | int(v_codes[h, 32 * G + i]) << shift
                at = 16 * d + (j * (d // 32) + G) * 2
                r[at:at + 2] = np.frombuffer(np.float16(k_scales[h, G]).tobytes(), np.uint8)
                at = 17 * d + ((c * 4 + t) * (d // 32) + G) * 4 + e * 2
                r[at:at + 2] = np.frombuffer(np.float16(v_scales[h, G]).tobytes(), np.uint8)

    def append(self, k, v, slots):
        kc, ks = quantise(k)
        vc, vs = quantise(v)
        for i, s in enumerate(slots):
            if 0 <= s < self.k.shape[0]:
                self.put(int(s), kc[i], ks[i], vc[i], vs[i])


def attention(k, v, pages, q, tables, lengths, cu_rows, window, scale, out):
    """out with the rows of every sequence, and the sizes its error is measured by: sum p |v| and sum |v| per value, and the
    largest scale sum |q k| of a row.  k, v: [slots][kv_heads][d]; a page outside of the arena hides its keys."""
    q, out = np.asarray(q, np.float64), np.array(out, np.float64)
    weight, extent, reach = np.zeros_like(out), np.zeros_like(out), np.zeros(out.shape[:2])
    group = q.shape[1] // k.shape[1]
    for s in range(len(lengths)):
        n = cu_rows[s + 1] - cu_rows[s]
        for i in range(n):
            row, pos = cu_rows[s] + i, min(lengths[s], tables.shape[1] * PAGE) - n + i
            keys = np.arange(max(0, pos - window + 1) if window else 0, pos + 1)
            page = tables[s, keys // PAGE] if len(keys) else keys
            keys, page = keys[(page >= 0) & (page < pages)], page[(page >= 0) & (page < pages)]
            out[row] = 0.0
            if not len(keys):
                continue
            at = page * PAGE + keys % PAGE
            for h in range(q.shape[1]):
                kk, vv = k[at, h // group], v[at, h // group]
                with np.errstate(invalid="ignore"):
                    x = kk @ q[row, h] * scale
                p = np.exp(x - x.max())
                p /= p.sum()
                out[row, h], weight[row, h] = p @ vv, p @ np.abs(vv)
                extent[row, h] = np.abs(vv).sum(axis=0)
                with np.errstate(invalid="ignore"):
                    reach[row, h] = np.max(np.abs(kk) @ np.abs(q[row, h])) * abs(scale)
    return out, (weight, extent, reach)
