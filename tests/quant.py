"""4-bit rows for the matrix tests: random rows with finite scales, and their weights in 64 bits as the difference
of two nonnegative-scaled parts (Q4_K: d sc q and dmin mi; MXFP4: the weight and zero), written from the formats."""
import numpy as np

Q8_0, Q4_K, MXFP4 = 8, 12, 39
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])


def row_bytes(type_, n):
    return n // 256 * 144 if type_ == Q4_K else n // 32 * 17


def random_rows(type_, rows, n, rng, exponents=(112, 124)):
    """Any nibbles, any 6-bit scales; fp16 super scales of either sign up to 2^-6, or E8M0 exponents of a range."""
    raw = rng.integers(0, 256, (rows, row_bytes(type_, n))).astype(np.uint8)
    if type_ == Q4_K:
        b = raw.reshape(rows, -1, 144)
        s = (rng.standard_normal((rows, b.shape[1], 2)) * 2e-3).astype(np.float16)
        b[..., :4] = s.view(np.uint8).reshape(rows, -1, 4)
    else:
        raw.reshape(rows, -1, 17)[..., 0] = rng.integers(exponents[0], exponents[1], (rows, n // 32))
    return raw


def weights(type_, raw, n):
    """(w, a): the weights and the size of the terms they are sums of, float64 [rows][n]."""
    rows = raw.shape[0]
    if type_ == Q4_K:
        b = raw.reshape(rows, n // 256, 144)
        s = np.ascontiguousarray(b[..., :4]).view(np.float16).astype(np.float64)
        w = np.zeros((rows, n // 256, 8, 32))
        a = np.zeros_like(w)
        for g in range(8):
            if g < 4:
                sc, mi = b[..., 4 + g] & 63, b[..., 8 + g] & 63
            else:
                sc = b[..., 8 + g] & 15 | (b[..., g] >> 6) << 4
                mi = b[..., 8 + g] >> 4 | (b[..., 4 + g] >> 6) << 4
            q = b[..., 16 + g // 2 * 32:48 + g // 2 * 32] >> (4 * (g & 1)) & 15
            pos = (s[..., 0] * sc)[..., None] * q
            neg = (s[..., 1] * mi)[..., None]
            w[:, :, g], a[:, :, g] = pos - neg, np.abs(pos) + np.abs(neg)
        return w.reshape(rows, n), a.reshape(rows, n)
    b = raw.reshape(rows, n // 32, 17)
    code = np.concatenate([b[..., 1:] & 15, b[..., 1:] >> 4], -1)
    w = (E2M1[code] * np.exp2(b[..., :1].astype(np.float64) - 127)).reshape(rows, n)
    return w, np.abs(w)
