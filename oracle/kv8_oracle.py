"""The 8-bit key/value cache restated in numpy, 64 bits: e4m3 from its definition, the block scales, and softmax
attention over the dequantised rows.  Independent of the package and of torch's float8 type."""
import numpy as np

BLK, D = 64, 128
E_MIN, E_MAX = -120, 120


def _table():
    t = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = np.nan if (c & 127) == 127 else m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        t[c] = -v if c & 128 else v
    return t


TABLE = _table()


def decode(codes):
    """uint8 codes -> float64."""
    return TABLE[codes]


def encode(y):
    """float64 |y| <= 448 (or NaN) -> the code of the nearest e4m3 number, ties to the even code."""
    y = np.asarray(y, np.float64)
    a = np.abs(y)
    step = 2.0 ** (np.floor(np.log2(np.maximum(a, 2.0 ** -6))) - 3)
    r = np.rint(a / step) * step                        # the nearest multiple of the spacing, ties to even
    code = np.searchsorted(TABLE[:127], np.where(np.isnan(r), 0.0, r)).astype(np.uint8)
    assert np.array_equal(TABLE[code], np.where(np.isnan(r), 0.0, r))
    code = np.where(np.isnan(y), 127, code).astype(np.uint8)
    return (code | np.where(np.signbit(y) & ~np.isnan(y), 128, 0)).astype(np.uint8)


def scale_of(x):
    """2^e, e the smallest integer in [E_MIN, E_MAX] with every finite |x| <= 448 * 2^e."""
    x = np.abs(np.asarray(x, np.float64))
    top = x[np.isfinite(x)].max(initial=0.0)
    e = E_MIN
    if top > 0:
        e = int(np.clip(np.floor(np.log2(top / 448.0)) - 1, E_MIN, E_MAX))
        while e < E_MAX and top > 448.0 * 2.0 ** e:
            e += 1
    return 2.0 ** e


def write(rows, scales, K, V, start):
    """In place: rows uint8 [BH, cap, 2, 128], scales [BH, nblk, 2]; K, V [BH, T, 128]; start [BH] (negative:
    nothing; tokens past cap are dropped)."""
    for bh in range(rows.shape[0]):
        for w, X in enumerate((K, V)):
            s0 = int(start[bh])
            if s0 < 0:
                continue
            end = min(s0 + X.shape[1], rows.shape[1])
            for blk in range(s0 // BLK, -(-end // BLK)):
                a, b = max(s0, blk * BLK), min(end, (blk + 1) * BLK)
                if a >= b:
                    continue
                x = np.asarray(X[bh, a - s0:b - s0], np.float64)
                s = scale_of(x)
                if a > blk * BLK:
                    old = float(scales[bh, blk, w])
                    s = max(s, old)
                    if s > old:
                        r = rows[bh, blk * BLK:a, w]
                        nan = (r & 127) == 127
                        r[:] = np.where(nan, r, encode(np.where(nan, 0.0, decode(r)) * (old / s)))
                rows[bh, a:b, w] = encode(np.where(np.isfinite(x), x, np.nan) / s)
                scales[bh, blk, w] = s


def values(rows, scales):
    """float64 K, V [BH, cap, 128]."""
    v = decode(rows) * np.repeat(np.asarray(scales, np.float64), BLK, 1)[..., None]
    return v[:, :, 0], v[:, :, 1]


def softmax_rows(q, K, V):
    """q [R, 128], K, V [R or 1, n, 128] float64 -> (out [R, 128], sum of weight * |V| [R, 128]); n = 0 gives 0."""
    if K.shape[1] == 0:
        return np.zeros((len(q), D)), np.zeros((len(q), D))
    s = np.einsum("rd,rnd->rn", q, np.broadcast_to(K, (len(q),) + K.shape[1:])) / np.sqrt(D)
    w = np.exp(s - s.max(-1, keepdims=True))
    w /= w.sum(-1, keepdims=True)
    Vb = np.broadcast_to(V, (len(q),) + V.shape[1:])
    return np.einsum("rn,rnd->rd", w, Vb), np.einsum("rn,rnd->rd", w, np.abs(Vb))


def attend(q, rows, scales, end, Hkv):
    """q [B, Hq, T, 128]; end [B]: query t sees the keys [0, end - (T - 1 - t)).  (out, weighted |V|) float64."""
    q = np.asarray(q, np.float64)
    B, Hq, T, _ = q.shape
    K, V = values(rows, scales)
    out, mag = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        for h in range(Hq):
            bh = b * Hkv + h // (Hq // Hkv)
            for t in range(T):
                n = min(max(int(end[b]), 0), rows.shape[1]) - (T - 1 - t)
                if n > 0:
                    o, m = softmax_rows(q[b, h, t][None], K[bh, None, :n], V[bh, None, :n])
                    out[b, h, t], mag[b, h, t] = o[0], m[0]
    return out, mag


def attend_picks(q, idx, rows, scales, end):
    """q [BH, G, 128], idx [BH, G, k], end [BH]: picks outside [0, end) are left out."""
    q = np.asarray(q, np.float64)
    K, V = values(rows, scales)
    out, mag = np.zeros(q.shape), np.zeros(q.shape)
    for bh in range(q.shape[0]):
        for g in range(q.shape[1]):
            i = idx[bh, g]
            i = i[(i >= 0) & (i < min(int(end[bh]), rows.shape[1]))]
            if len(i):
                o, m = softmax_rows(q[bh, g][None], K[bh][i][None], V[bh][i][None])
                out[bh, g], mag[bh, g] = o[0], m[0]
    return out, mag
