"""A cache held in 4 bits, restated in numpy: the page layout and the rounding of include/b200seq.h (b200seq_kv4_*), and attention over it in 64 bits."""
import numpy as np

FIFTEENTH = np.float32(float.fromhex("0x1.11111p-4"))


def groups(D):
    return 1 if D <= 32 else 2 if D <= 64 else 4


def place(d, NG, key):
    """4-bit field of value d in a row of codes"""
    g, i = divmod(d, 32)
    return ((i // 8 * NG + g) * 8 + i % 8) if key else ((i // 4 * NG + g) * 4 + i % 4)


def quantise(x):
    """codes [.., D] and (s, m) [.., NG] float32 of rows x [.., D]"""
    x = np.nan_to_num(np.asarray(x, np.float32), nan=0.0, posinf=np.inf, neginf=-np.inf)
    x = np.clip(x, np.float32(-32000), np.float32(32000))
    D = x.shape[-1]
    NG = groups(D)
    codes, s, m = np.zeros(x.shape, np.int64), np.zeros(x.shape[:-1] + (NG,), np.float32), np.zeros(x.shape[:-1] + (NG,), np.float32)
    for g in range((D + 31) // 32):
        y = x[..., 32 * g:32 * g + 32]
        low = y.min(-1).astype(np.float16).astype(np.float32)
        step = np.maximum((y.max(-1) - low) * FIFTEENTH, np.float32(0))
        step = ((step.view(np.uint32) + np.uint32(0x1FFFF)) & np.uint32(0xFFFE0000)).view(np.float32)
        step = np.where(step < 2.0 ** -18, np.ceil(step * np.float32(2 ** 24)) * np.float32(2 ** -24), step).astype(np.float32)
        inv = np.divide(np.float32(1), step, out=np.zeros_like(step), where=step > 0)
        codes[..., 32 * g:32 * g + 32] = np.clip(np.rint((y - low[..., None]) * inv[..., None]), 0, 15).astype(np.int64)
        s[..., g], m[..., g] = step, low
    return codes, s, m


def held(x):
    """the values that rows stand for once they are in the cache (float32: codes times steps are exact, the sum is rounded once)"""
    codes, s, m = quantise(x)
    at = np.arange(codes.shape[-1]) // 32
    return (codes * s[..., at].astype(np.float64) + m[..., at]).astype(np.float32)


def row_bytes(x, key):
    """(codes, parameters) of one row as the bytes of its page"""
    codes, s, m = quantise(x)
    NG = groups(len(x))
    nib = np.zeros(32 * NG, np.int64)
    for d in range(len(x)):
        nib[place(d, NG, key)] = codes[d]
    par = np.stack([s, m], -1).astype(np.float16).reshape(-1).view(np.uint8)
    return (nib[0::2] | (nib[1::2] << 4)).astype(np.uint8), par


def row_at(pool, bs, page, o, g, NG):
    """(codes, parameters) of row o of head g of a page, views of the pool's bytes [pages, heads, segment]"""
    unit = 16 if bs % 16 == 0 else bs
    u, ru = divmod(o, unit)
    seg = pool[page, g, u * unit * NG * 20:(u + 1) * unit * NG * 20]
    return seg[ru * NG * 16:(ru + 1) * NG * 16], seg[unit * NG * 16 + ru * NG * 4:unit * NG * 16 + (ru + 1) * NG * 4]


def put_rows(pool, bs, slots, x, key):
    """rows x [n, G, D] into the pool at (page, place) slots"""
    NG = groups(x.shape[-1])
    for (page, o), row in zip(slots, x):
        for g in range(x.shape[1]):
            c, p = row_at(pool, bs, page, o, g, NG)
            c[:], p[:] = row_bytes(row[g], key)


def get_rows(pool, bs, slots, D, key):
    """float64 [n, G, D]: what the pool's bytes stand for"""
    G, NG = pool.shape[1], groups(D)
    out = np.zeros((len(slots), G, D))
    at = [place(d, NG, key) for d in range(D)]
    for i, (page, o) in enumerate(slots):
        for g in range(G):
            c, p = row_at(pool, bs, page, o, g, NG)
            nib = np.stack([c & 15, c >> 4], -1).reshape(-1)
            par = np.ascontiguousarray(p).view(np.float16).astype(np.float64).reshape(NG, 2)
            for d in range(D):
                out[i, g, d] = par[d // 32, 0] * nib[at[d]] + par[d // 32, 1]
    return out


def attend(q, k, v, pos, scale, chunk=0, window=0, keep_first=0, softcap=0.0, sink=None, head_scale=None, gate=None):
    """float64 [n, H, V]: q [n, H, D] at positions pos over keys k [L, G, D] and values v [L, Gv, V]; gate [n, H] or [n, H, V] logits"""
    n, H, D = q.shape
    L, G, Gv = k.shape[0], k.shape[1], v.shape[1]
    j, i = np.arange(L)[None], np.asarray(pos)[:, None]
    see = j <= i
    if chunk:
        see &= j // chunk == i // chunk
    if window:
        see &= (i - j < window) | (j < keep_first)
    out = np.zeros((n, H, v.shape[2]))
    for h in range(H):
        g = h // (H // G)
        z = q[:, h].astype(np.float64) @ k[:, g].T * scale * (1.0 if head_scale is None else float(head_scale[h]))
        if softcap:
            z = softcap * np.tanh(z / softcap)
        z = np.where(see, z, -np.inf)
        top = z.max(1, keepdims=True)
        if sink is not None:
            top = np.maximum(top, float(sink[h]))
        w = np.exp(z - top)
        den = w.sum(1, keepdims=True) + (np.exp(float(sink[h]) - top) if sink is not None else 0.0)
        out[:, h] = (w / den) @ v[:, g // (G // Gv)]
    if gate is not None:
        f = 1.0 / (1.0 + np.exp(-gate.astype(np.float64)))
        out *= f if f.ndim == 3 else f[:, :, None]
    return out
