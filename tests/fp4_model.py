"""The cache in 4 bits by its definition, in numpy: what writing makes of a block, where a row keeps it, what the bytes stand for."""

import numpy as np

LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def row_bytes(h, d):
    return ((d + 1) // 2 + (h + 1) // 2 + -(-d // 32) + -(-h // 32) + 3) // 4 * 4


def quantise(x):
    """One block: (codes, scale byte)."""
    x = np.asarray(x, np.float64)
    if not np.isfinite(x).all():
        return np.zeros(len(x), np.uint8), 255
    most = np.abs(x).max()
    e = -125 if most == 0 else int(np.frexp(most)[1]) - 3
    if most > 7.25 * 2.0**e:
        e += 1
    e = min(max(e, -125), 125)
    y = np.abs(x) / 2.0**e
    codes = np.zeros(len(x), np.uint8)
    for i, halfway in enumerate((LEVELS[1:] + LEVELS[:-1]) / 2):
        codes += (y >= halfway) if i % 2 else (y > halfway)  # halves to the even code
    return codes | (np.signbit(x).astype(np.uint8) << 3), e + 127


def write_row(a, b):
    """Bytes of the row of a[h], b[d], those without a meaning -1."""
    h, d = len(a), len(b)
    row = np.full(row_bytes(h, d), -1, np.int64)
    at_codes, at_scale = 0, (d + 1) // 2 + (h + 1) // 2
    for part in (b, a):
        codes = []
        for first in range(0, len(part), 32):
            c, s = quantise(part[first : first + 32])
            codes += c.tolist()
            row[at_scale] = s
            at_scale += 1
        codes += [0] * (len(codes) % 2)
        row[at_codes : at_codes + len(codes) // 2] = np.array(codes[0::2], np.int64) + 16 * np.array(codes[1::2], np.int64)
        at_codes += len(codes) // 2
    return row


def read_rows(rows, h, d):
    """[.., bytes] -> (a[.., h], b[.., d]) in 64 bits."""
    rows = np.asarray(rows)

    def numbers(codes_at, scales_at, n):
        i = np.arange(n)
        codes = (rows[..., codes_at + i // 2].astype(np.int64) >> (4 * (i % 2))) & 15
        scale = rows[..., scales_at + i // 32].astype(np.float64)
        x = np.where(codes >= 8, -1.0, 1.0) * LEVELS[codes & 7] * 2.0 ** (np.minimum(scale, 254) - 127)
        return np.where(scale == 255, np.nan, x)

    at = (d + 1) // 2
    scales = at + (h + 1) // 2
    return numbers(at, scales + -(-d // 32), h), numbers(0, scales, d)


def random_rows(rng, shape, h, d, scales=(125, 130)):
    """Rows with random codes and scales near 1; the bytes without a meaning are random too."""
    rows = rng.integers(0, 256, (*shape, row_bytes(h, d)), dtype=np.uint8)
    at = (d + 1) // 2 + (h + 1) // 2
    n = -(-d // 32) + -(-h // 32)
    rows[..., at : at + n] = rng.integers(*scales, (*shape, n))
    return rows
