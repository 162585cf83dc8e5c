"""The paged KV cache, attention over it, softmax and draft verification in plain
numpy: stored rows bit for bit, everything else in 64 bits."""
import numpy as np

F32, BF16, INT8, FP8 = 0, 1, 2, 3
DTYPE = {F32: np.float32, BF16: np.uint16, INT8: np.int8, FP8: np.uint8}


def e4m3_table():
    """Values of the 256 e4m3 codes (bias 7; 0x7f and 0xff are NaN)."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v[(c & 127) == 127] = np.nan
    return np.where(c < 128, v, -v)


E4M3 = e4m3_table()


def to_e4m3(y):
    """Codes of the nearest e4m3 values, halves to the even code; |y| <= 448."""
    pos = E4M3[:127]
    a = np.abs(y)
    i = np.clip(np.searchsorted(pos, a), 1, 126)
    lo, hi = pos[i - 1], pos[i]
    up = (a - lo > hi - a) | ((a - lo == hi - a) & ((i & 1) == 0))
    code = np.where(up, i, i - 1)
    return (code | np.where(np.signbit(y), 128, 0)).astype(np.uint8)


def to_bf16(x):
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), 0x7FC0, r).astype(np.uint16)


def store(x, fmt):
    """Rows [..][64] fp32 -> (stored values, scale or None)."""
    x = np.ascontiguousarray(x, np.float32)
    if fmt == F32:
        return x, None
    if fmt == BF16:
        return to_bf16(x), None
    fin = np.isfinite(x).all(-1)
    z = np.where(fin[..., None], x, 0).astype(np.float64)
    amax = np.abs(z).max(-1)
    if fmt == INT8:
        s = (amax / 127.0).astype(np.float32)  # no quotient of a 24-bit value by 127 lies near a midpoint
        q = np.round(z / np.where(s > 0, s, 1).astype(np.float64)[..., None])
        q = np.clip(np.where(s[..., None] > 0, q, 0), -127, 127).astype(np.int8)
    else:
        m, e = np.frexp(amax / 448.0)
        e = np.maximum(np.where(m == 0.5, e - 1, e), -126)
        s = np.ldexp(1.0, np.where(amax > 0, e, -126)).astype(np.float32)
        q = to_e4m3(z / s.astype(np.float64)[..., None])
        q = np.where(fin[..., None], q, 0).astype(np.uint8)
    return q, np.where(fin, s, np.float32(np.nan)).astype(np.float32)


def values(q, s, fmt):
    """The fp32 values that stored rows stand for."""
    if fmt == F32:
        return q
    if fmt == BF16:
        return (q.astype(np.uint32) << 16).view(np.float32)
    f = q.astype(np.float32) if fmt == INT8 else E4M3[q].astype(np.float32)
    return f * s[..., None]


def attention(q, k, v, visible):
    """q [64] per row [rows][64], k and v [keys][64], visible [rows][keys] -> (out, sum of p|v|,
    largest sum |q||k| / 8 of a row)."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    s = q @ k.T / 8.0
    s = np.where(visible, s, -np.inf)
    m = s.max(1, keepdims=True)
    p = np.where(visible, np.exp(s - np.where(np.isfinite(m), m, 0)), 0.0)
    t = p.sum(1, keepdims=True)
    p = p / np.where(t > 0, t, 1)
    return p @ v, p @ np.abs(v), (np.abs(q) @ np.abs(k).T / 8.0).max(1, initial=0.0)


def softmax(x, temperature):
    x = x.astype(np.float64)
    with np.errstate(invalid="ignore"):
        m = x.max(1, keepdims=True)
        e = np.exp((x - np.where(m == -np.inf, 0, m)) / np.float64(np.float32(temperature)))
    t = e.sum(1, keepdims=True)
    return e / np.where(t == 0, 1, t)


def draw(w, u):
    w = np.where(w > 0, w, 0.0)
    c = np.cumsum(w)
    above = np.nonzero(c > np.float64(u) * c[-1])[0]
    return int(above[0]) if len(above) else -1


def verify(target, draft, ids, u_accept, u_sample, n_valid):
    B, K1, V = target.shape
    K = K1 - 1
    t, d = target.astype(np.float64), None if K == 0 else draft.astype(np.float64)
    acc, tok = np.zeros(B, np.int32), np.full((B, K1), -1, np.int32)
    for b in range(B):
        n, a = min(max(int(n_valid[b]), 0), K), 0
        while a < n and 0 <= ids[b, a] < V and np.float64(u_accept[b, a]) * d[b, a, ids[b, a]] < t[b, a, ids[b, a]]:
            a += 1
        w = t[b, a]
        if a < n:
            r = w - d[b, a]
            r = np.where(r > 0, r, 0.0)
            w = r if r.sum() > 0 else w
        acc[b] = a
        if a:
            tok[b, :a] = ids[b, :a]
        tok[b, a] = draw(w, u_sample[b])
    return acc, tok
