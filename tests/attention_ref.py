"""Plain implementations in 64 bits of the attention operators, and how far the kernels may be from them."""
import numpy as np

import mag_b200 as MB

U = 2.0 ** -24  # half an f32 step relative to the value
VALUES = MB.e4m3_values().astype(np.float64)


def turn(v, pos, freq, rot, pairs, mag=1.0, back=False):
    """v [rows][heads][dim] turned by its row's position (or its transpose), and the sizes that roundings act on."""
    v = np.asarray(v, np.float64)
    out, size = v.copy(), np.abs(v)
    if not rot:
        return out, size
    a = np.asarray(pos, np.float64)[:, None] * np.asarray(freq, np.float32).astype(np.float64)[None]
    c, s = (np.cos(a) * mag)[:, None], (np.sin(a) * mag)[:, None] * (-1.0 if back else 1.0)
    i, j = (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, rot // 2), slice(rot // 2, rot))
    x, y = v[..., i], v[..., j]
    out[..., i], out[..., j] = x * c - y * s, y * c + x * s
    size[..., i] = size[..., j] = (np.abs(x) + np.abs(y)) * abs(mag)
    return out, size


def norm(x, w, eps):
    x = np.asarray(x, np.float64)
    rstd = 1.0 / np.sqrt((x * x).mean(-1) + eps)
    return x * rstd[..., None] * np.asarray(w, np.float64), rstd


def attention(q, k, v, scale, n, length, window, ok=None):
    """q [n][q_heads][dim], k, v [length][heads][dim] in f64; ok [length]: the token's page exists.  Returns out, lse and
    how far the kernel's may be off."""
    group, dim = q.shape[1] // k.shape[1], q.shape[2]
    out, lse = np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
    tol, ltol = np.zeros(q.shape), np.zeros(q.shape[:2])
    j = np.arange(length)
    for t in range(n):
        p = length - n + t
        seen = (j <= p) & ((j > p - window) if window else True)
        if ok is not None:
            seen = seen & ok
        if not seen.any():
            continue
        ks, vs = k[seen], v[seen]
        for h in range(q.shape[1]):
            kk, vv = ks[:, h // group], vs[:, h // group]
            with np.errstate(invalid="ignore"):
                s = kk @ q[t, h] * scale
                m = s.max()
                e = np.exp(s - m)
                total = e.sum()
                out[t, h] = e @ vv / total
                lse[t, h] = m + np.log(total)
                # A logit: the query's two halves lose 2^-22 of each value; the tensor core adds 16 products at a time
                # to an f32 sum, dim / 8 instructions for both halves, each losing at most an f32 step (2 U) of the sum
                # of magnitudes; a few roundings for the scales and the exponent's argument.
                size = (np.abs(kk) @ np.abs(q[t, h]) * scale).max()
                ds = (dim / 8 + 12) * 2 * U * size
                # The output: both its sums move by the logits' error; the probabilities' halves lose 2^-22; the values
                # are added like the logits, 2 x 64 instructions between two flushes into f32 sums, one flush per 128 to
                # 1024 tokens and part; the exponential and the division take a few more.
                add = (2 * 64 + len(vv) / 128 + 40) * 2 * U
                # A weight is a sum of two f16, multiples of 2^-24 where the largest weight is 2^15 (few rows) or 2^9 (many): off by
                # up to 2^-25 / 2^9 = 2^-34 of the largest, times e4m3 values of up to 448 of a unit at most twice the largest
                # scale (2^10 scales, while the largest |v| may be as little as 2^6 of them): 2^-30 of the largest |v|.
                tol[t, h] = (np.abs(vv).T @ e) / total * (2 * ds + add) + 2.0 ** -30 * len(vv) * np.abs(vv).max() / total
                ltol[t, h] = ds + add + 2 * U * abs(lse[t, h])
    return out, lse, tol, ltol
