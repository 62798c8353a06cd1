"""What lies between two steps of a serving loop, restated in numpy and 64 bits: drafts verified, the weight of cached keys, eviction (include/b200seq.h has the definitions)."""
import numpy as np


# ---- drafts ------------------------------------------------------------------------------------------------------------------------------
def probabilities(z, T, top_k=0, top_p=1.0):
    """f64 probabilities of a row of logits, or None where it leaves no choice; kept: which tokens"""
    z = np.asarray(z, np.float64)
    top = z.max()
    if not np.isfinite(top):        # (NaN among them too)
        return None
    if not T > 0:
        p = np.zeros(len(z))
        p[int(np.argmax(z))] = 1.0
        return p
    with np.errstate(over="ignore"):
        w = np.exp((z - top) / T)
    if top_k > 0 and top_k < len(z):
        w = np.where(z >= np.sort(z)[::-1][top_k - 1], w, 0.0)
    if top_p < 1:
        order = np.argsort(-z, kind="stable")
        before = np.cumsum(w[order]) - w[order]
        zs = z[order]
        first = np.searchsorted(-zs, -zs, side="left")          # of the equal ones
        keep = before[first] < top_p * w.sum()
        keep[0:1] = True
        keep |= zs == zs[0]
        w = np.where(np.isin(np.arange(len(z)), order[keep]), w, 0.0)
    return w / w.sum()


def choose(w, u):
    """(lowest index whose cumulated weight exceeds u * sum, how near another index is: of the sum)"""
    cum = np.cumsum(w)
    target = u * cum[-1]
    i = min(int(np.searchsorted(cum, target, side="right")), int(np.nonzero(w)[0][-1]))
    edges = cum[np.nonzero(w)[0]]
    edges = edges[:-1]
    return i, (np.abs(edges - target).min() / cum[-1] if len(edges) else 1.0)


def verify(logits, start, drafts, accept_u, sample_u, T, top_k=None, top_p=None, probs=None):
    """accepted [B], tokens [R], and for every entry how near it came to another answer (relative)"""
    V = logits.shape[1]
    B = len(T)
    accepted, tokens, margin = np.zeros(B, int), np.full(logits.shape[0], -1), np.ones(B)
    for e in range(B):
        s0, s1 = int(start[e]), int(start[e + 1])
        if s0 == s1:
            continue
        k, share = (0 if top_k is None else int(top_k[e])), (1.0 if top_p is None else float(top_p[e]))
        n = s1 - s0 - 1
        for i in range(n + 1):
            row = s0 + i
            p = probabilities(logits[row], float(T[e]), k, share)
            if p is None:
                tokens[row] = -1
                break
            x = int(drafts[row])
            if i < n:
                fine = False
                if 0 <= x < V:
                    if T[e] > 0:
                        q = 1.0 if probs is None else float(probs[row, x])
                        lhs = float(accept_u[row]) * q
                        fine = lhs < p[x]
                        margin[e] = min(margin[e], abs(lhs - p[x]) / max(lhs, p[x], 1e-300))
                    else:
                        fine = p[x] > 0
                if fine:
                    tokens[row] = x
                    accepted[e] += 1
                    continue
            if not T[e] > 0:
                tokens[row] = int(np.argmax(p))
                break
            w = p
            if i < n:
                q = np.zeros(V)
                if probs is not None:
                    q = probs[row].astype(np.float64)
                elif 0 <= x < V:
                    q[x] = 1.0
                rest = np.maximum(p - q, 0.0)
                if rest.sum() > 0:
                    w = rest
            tokens[row], near = choose(w, float(sample_u[e]))
            # (what is left of a distribution after another went off it is known to the roundings of the whole)
            margin[e] = min(margin[e], near * w.sum())
            break
    return accepted, tokens, margin


# ---- weights of cached keys ----------------------------------------------------------------------------------------------------------------
def key_weights(q, keys, pos0, lens, slots, acc, G, scale, last=0, window=0, chunk=0, keep_first=0, softcap=0.0, head_scale=None, sink=None):
    """acc [slots, G, room] after a step.  q: per entry [n, H, D]; keys: per entry [pos0 + n, G, D].  Also the largest sum |q k| scale that a score is made of."""
    acc, most = np.array(acc, np.float64), 0.0
    for e, n in enumerate(lens):
        if n == 0:
            continue
        H, total = q[e].shape[1], pos0[e] + n
        m = min(last, n) if last > 0 else n
        acc[slots[e], :, pos0[e]:total] = 0.0
        for i in range(n - m, n):
            p = pos0[e] + i
            lo = p // chunk * chunk if chunk > 0 else 0
            if window > 0:
                lo = max(lo, p - window + 1)
            j = np.arange(total)
            see = (j <= p) & ((j >= lo) | (j < (keep_first if window > 0 else 0)))
            for h in range(H):
                g = h * G // H
                f = scale * (1.0 if head_scale is None else float(head_scale[h]))
                kk, qq = keys[e][:, g].astype(np.float64), q[e][i, h].astype(np.float64)
                z = kk @ qq * f
                most = max(most, float((np.abs(kk[see]) @ np.abs(qq)).max() * abs(f)))
                if softcap > 0:
                    z = softcap * np.tanh(z / softcap)
                z = np.where(see, z, -np.inf)
                top = z.max() if sink is None else max(z.max(), float(sink[h]))
                if top == -np.inf:
                    continue
                w = np.exp(z - top)
                den = w.sum() + (0.0 if sink is None else np.exp(float(sink[h]) - top))
                acc[slots[e], g, :total] += w / den
    return acc, most


# ---- eviction ------------------------------------------------------------------------------------------------------------------------------
def stays(weights, n, keep, first, recent):
    """rows of n that stay, in order, by their weights [n] (NaN lowest, equal ones: the lower row)"""
    if n <= keep:
        return list(range(n))
    mid = np.asarray(weights[first:n - recent], np.float64)
    mid = np.where(np.isnan(mid), -np.inf, mid) + 0.0
    nan_last = np.where(np.isnan(np.asarray(weights[first:n - recent], np.float64)), 1, 0)
    order = np.lexsort((np.arange(len(mid)), nan_last, -mid))
    best = sorted(int(i) + first for i in order[:keep - first - recent])
    return list(range(first)) + best + list(range(n - recent, n))
