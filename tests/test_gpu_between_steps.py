"""Drafts verified (csrc/seq/seq_verify.cu), the weight of cached keys (seq_weigh*.cu) and eviction (seq_evict.cu) against 64 bits.

verify_drafts gives whole numbers.  Its weights are 2^(d c) with d c rounded twice (|d c| < 16 where a weight counts: 2^-20 of it) and 2 units of the function (2^-22): every weight is
within 2^-19 of itself, and so is every sum of them, whatever the share.  An entry is compared where the oracle's next other answer is further away than 2^-17 of what is compared
(two sums and their quotient).

key_weights: a score is a sum of f32 products of `chain` roundings, each 2^-24 of the sum of their magnitudes at most, and four more for factors and differences: scores are off by
(chain + 4) 2^-24 of sum |q k| scale (natural units), a weight by as much of itself, and its row's denominator too; the function adds 2^-21, sums of `rows` weights 2^-24 each."""
import ctypes as C

import numpy as np
import pytest
import torch

import between_oracle as oracle
import kv4_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NEAR = 2.0 ** -17


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from blazr_b200 import seqops
    seqops.lib()
    seqops.error_flags()
    return seqops


def up(x, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(x, dtype))).to(DEV)


# ---- drafts ----------------------------------------------------------------------------------------------------------------------------------
def run_verify(ops, z, start, drafts, ua, us, T, top_k=None, top_p=None, probs=None, **kw):
    o = lambda x, t: None if x is None else up(x, t)
    acc, tok = ops.verify_drafts(z if isinstance(z, torch.Tensor) else up(z, np.float32), up(start, np.int32), up(drafts, np.int32), up(ua, np.float32), up(us, np.float32),
                                 up(T, np.float32), top_k=o(top_k, np.int32), top_p=o(top_p, np.float32), draft_probs=probs if isinstance(probs, torch.Tensor) else o(probs, np.float32), **kw)
    return acc.cpu().numpy(), tok.cpu().numpy()


def same(got, want, start):
    """entries whose oracle is sure; how many those are"""
    sure = 0
    for e in range(len(start) - 1):
        if want[2][e] < NEAR:
            continue
        sure += 1
        assert got[0][e] == want[0][e], (e, got[0][e], want[0][e])
        np.testing.assert_array_equal(got[1][start[e]:start[e + 1]], want[1][start[e]:start[e + 1]], err_msg=f"entry {e}")
    return sure


@pytest.mark.parametrize("V", [1, 2, 5, 33, 1000, 4093, 16387, 50257, 131072])
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("ruled", [False, True])
def test_drafts_are_verified(ops, V, probs, ruled):
    rng = np.random.default_rng(V + 2 * probs + ruled)
    lens = [5, 1, 0, 3, 2, 1, 9, 4]
    start = np.concatenate([[0], np.cumsum(lens)])
    R, B = int(start[-1]), len(lens)
    z = (2.0 * rng.standard_normal((R, V))).astype(np.float32)
    T = np.array([1.0, 0.7, 1.0, 0.0, 1.5, 0.3, 1.0, 1.0], np.float32)
    q = None
    if probs:
        y = z + 0.3 * rng.standard_normal((R, V))
        q = np.exp(y - y.max(1, keepdims=True))
        q = (q / q.sum(1, keepdims=True)).astype(np.float32)
        drafts = np.array([rng.choice(V, p=r / r.sum()) for r in q.astype(np.float64)])
    else:
        drafts = np.where(rng.random(R) < 0.8, z.argmax(1), rng.integers(0, V, R))
    k = rng.choice([0, 1, 3, 50, V, V + 7], B) if ruled else None
    p = np.where(rng.random(B) < 0.3, 1.0, rng.random(B)).astype(np.float32) if ruled else None
    ua, us = rng.random(R).astype(np.float32), rng.random(B).astype(np.float32)
    want = oracle.verify(z, start, drafts, ua, us, T, k, p, q)
    got = run_verify(ops, z, start, drafts, ua, us, T, k, p, q)
    assert same(got, want, start) >= B // 2
    assert ops.error_flags() == 0


@pytest.mark.parametrize("V", [7, 5000, 70001])
def test_rows_of_another_stride_and_alignment(ops, V):
    """rows inside wider ones, from an odd place on: logits and draft probabilities apart"""
    rng = np.random.default_rng(V)
    R, start = 12, np.array([0, 4, 12])
    z = (2.0 * rng.standard_normal((R, V))).astype(np.float32)
    q = rng.random((R, V)).astype(np.float32)
    q /= q.sum(1, keepdims=True)
    drafts = rng.integers(0, V, R)
    ua, us, T = rng.random(R).astype(np.float32) * 0.2, rng.random(2).astype(np.float32), np.array([1.0, 0.8], np.float32)
    for off, wide in ((1, V + 3), (3, V + 8), (2, V + 5)):
        zz, qq = torch.full((R, wide + off), 9e9, device=DEV), torch.full((R, wide + 4), 9e9, device=DEV)
        zz[:, off:off + V] = up(z)
        qq[:, 1:V + 1] = up(q)
        got = run_verify(ops, zz[:, off:off + V], start, drafts, ua, us, T, None, None, qq[:, 1:V + 1])
        assert same(got, oracle.verify(z, start, drafts, ua, us, T, None, None, q), start) >= 1


def test_rows_without_a_choice(ops):
    """masks that leave nothing, infinities, NaN: -1, and nothing behind them; masks that leave one token"""
    V, inf = 6000, np.inf
    rng = np.random.default_rng(3)
    base = rng.standard_normal(V).astype(np.float32)
    none, nan, plus, one, low = (np.array(base) for _ in range(5))
    none[:] = -inf
    nan[V - 1] = np.nan
    plus[17] = inf
    one[:] = -inf
    one[5999] = -3.0
    low[:] = np.finfo(np.float32).min
    low[77] = 0.0
    for T in (0.0, 1.0):
        for k, p in ((None, None), ([3] * 9, [0.9] * 9)):
            rows = [none, base, nan, base, plus, base, one, one, low, base, none, nan, plus, one, low]
            start = np.array([0, 2, 4, 6, 8, 10, 11, 12, 13, 15])
            drafts = np.array([0, 0, 1, 0, 17, 0, 5999, 0, 77, 0, 0, 0, 0, 5999, 0])
            want = [0, 0, 0, 1, 1, 0, 0, 0, 1]
            got = run_verify(ops, np.stack(rows), start, drafts, [0.5] * 15, [0.3] * 9, [T] * 9, k, p)
            np.testing.assert_array_equal(got[0], want)
            for r in (0, 2, 4, 10, 11, 12):
                assert got[1][r] == -1
            assert list(got[1][[1, 3, 5]]) == [-1, -1, -1] and got[1][6] == 5999 and got[1][7] == 5999 and got[1][8] == 77 and got[1][13] == 5999 and got[1][14] == 77
    assert ops.error_flags() == 0


def test_equal_logits(ops):
    """the first maximum where the temperature is zero; top_k and top_p keep equal ones together; -0 and 0 are equal"""
    V = 3000
    z = np.zeros((1, V), np.float32)
    z[0, [5, 9, 2999]] = 1.0
    z[0, 7::2] = np.where(z[0, 7::2] == 0, -0.0, z[0, 7::2])
    go = lambda u, T, k, p: run_verify(ops, z, [0, 1], [0], [0.0], [u], [T], [k], [p])[1][0]
    assert go(0.9, 0.0, 0, 1.0) == 5
    for k in (1, 2, 3):
        assert [go(u, 1.0, k, 1.0) for u in (0.0, 0.3, 0.34, 0.66, 0.67, 0.999)] == [5, 5, 9, 9, 2999, 2999]
    assert [go(u, 1.0, 0, 1e-6) for u in (0.1, 0.5, 0.9)] == [5, 9, 2999]        # the largest ones alone
    assert go(0.5, 1.0, 4, 1.0) == oracle.verify(z, [0, 1], [0], [0], [0.5], [1.0], [4], [1.0])[1][0]       # the fourth is every zero
    assert go(0.0, 1.0, 4, 1.0) == 0
    share = 3 * np.e / (3 * np.e + V - 3)
    assert go(0.0, 1.0, 0, share * 0.999) == 5 and go(0.0, 1.0, 0, share * 1.001) == 0      # below the three's share they are all; above, every zero joins


def test_temperatures_and_numbers_at_their_ends(ops):
    V = 9000
    rng = np.random.default_rng(5)
    z = (3 * rng.standard_normal((1, V))).astype(np.float32)
    go = lambda u, T, **kw: int(run_verify(ops, z, [0, 1], [0], [0.0], [u], [T], **kw)[1][0])
    top = 1 - 2.0 ** -24
    best = int(z[0].argmax())
    for T in (1e-30, 1e-38, 1e-3):
        for u in (0.0, 0.5, top):
            assert go(u, T) == best
    assert go(0.0, 1.0) == 0 and go(top, 1.0) >= 0 and go(0.0, 1e30) == 0 and go(top, 1e30) == V - 1
    for u in (0.25, 0.5, 0.75):
        assert abs(go(u, 1e30) - u * V) <= 1
    for k in ([1], [2]):
        assert go(0.0, 1.0, top_k=k) in np.argsort(-z[0])[:k[0]]
    for p in (0.0, -1.0, 1e-30):
        assert go(top, 1.0, top_p=[p]) == best
    for p in (1.0, 2.0, float("nan")):
        assert go(0.37, 1.0, top_p=[p]) == go(0.37, 1.0)


@pytest.mark.parametrize("T", [0.0, 1e-30, 0.7, 3e29, 1e38])
def test_logits_at_the_ends_of_their_type(ops, T):
    """differences beyond the type, minus infinities in some slices, one equal maximum a slice, a NaN in the last place"""
    V, rng = 30011, np.random.default_rng(12)
    z = (2 * rng.standard_normal((6, V))).astype(np.float32)
    z[0, ::3] = -np.inf
    z[1, 100:20000] = -np.inf
    z[2, :] = -np.inf
    z[2, 17000:17003] = 0.5
    z[3, ::2], z[3, 1::2] = 3e38, -3e38
    z[4, [5, 9000, 29999]] = 50.0
    z[5, V - 1] = np.nan
    start, n = np.arange(7), 6
    us = np.array([0.1, 0.35, 0.5, 0.83, 0.6, 0.2], np.float32)
    got = run_verify(ops, z, start, np.zeros(n), np.zeros(n), us, np.full(n, T))
    want = oracle.verify(z, start, np.zeros(n, np.int32), np.zeros(n), us, np.full(n, T, np.float32))
    assert same(got, want, start) >= 3
    assert got[1][5] == -1


def test_what_is_drawn_has_the_target_s_distribution(ops):
    """drafts from q, verified against p: tokens as often as p says.  Random numbers from an even grid in both places: counts are off by the grid's steps alone"""
    V, n = 5, 64
    z = np.array([0.3, -1.0, 1.2, 0.1, -0.4], np.float32)
    q = np.array([0.35, 0.25, 0.05, 0.15, 0.2], np.float32)
    p = oracle.probabilities(z, 1.0)
    grid = ((np.arange(n) + 0.5) / n).astype(np.float32)
    x, ua, us = (a.reshape(-1) for a in np.meshgrid(np.arange(V), grid, grid, indexing="ij"))
    B = len(x)
    start = np.arange(0, 2 * B + 1, 2)
    two = lambda a, b: np.stack([a, b], 1).reshape(-1)
    out = run_verify(ops, np.tile(z, (2 * B, 1))[:, :], start, two(x, 0 * x), two(ua, 0 * ua), us, np.ones(B), None, None, np.tile(q, (2 * B, 1)))
    first = out[1][0::2]
    freq = np.array([(q[x] * (first == t)).sum() for t in range(V)]) / (n * n)
    assert abs(freq.sum() - 1) < 1e-5
    np.testing.assert_allclose(freq, p, atol=4.0 / n)          # a step of the grid in the acceptance, one at either end of a token's share of the draw
    assert ((out[0] == 1) == (first == x))[q[x] <= p[x]].all()


def test_drafts_that_are_none(ops):
    """ids outside the vocabulary are refused and flagged; probabilities that say more than the target leaves the target's own"""
    V = 100
    rng = np.random.default_rng(1)
    z = rng.standard_normal((6, V)).astype(np.float32)
    z[2, 3] = -np.inf
    q = np.zeros((6, V), np.float32)
    q[:, 3] = 1.0
    q[2] = oracle.probabilities(z[2], 1.0) * 1.01
    ops.error_flags()
    got = run_verify(ops, z, [0, 2, 4, 6], [-1, 0, 3, 0, V, 0], [0.0] * 6, [0.4] * 3, [1.0] * 3, None, None, q)
    assert ops.error_flags() == 16
    want = oracle.verify(z, [0, 2, 4, 6], [-1, 0, 3, 0, V, 0], [0.0] * 6, [0.4] * 3, [1.0] * 3, None, None, q)
    np.testing.assert_array_equal(got[0], [0, 0, 0])
    np.testing.assert_array_equal(got[1], want[1])
    got = run_verify(ops, z, [0, 3, 2, 7], [0] * 6, [0.0] * 6, [0.4] * 3, [1.0] * 3)       # starts that are none: the second and third entry
    assert ops.error_flags() == 16 and list(got[0][1:]) == [0, 0]


def test_many_entries(ops):
    """more entries than a block looks through at once, each of one row or two"""
    rng = np.random.default_rng(8)
    B, V = 1500, 64
    lens = rng.integers(0, 3, B)
    start = np.concatenate([[0], np.cumsum(lens)])
    R = int(start[-1])
    z = (2 * rng.standard_normal((R, V))).astype(np.float32)
    drafts, ua, us, T = rng.integers(0, V, R), rng.random(R).astype(np.float32), rng.random(B).astype(np.float32), rng.random(B).astype(np.float32) + 0.2
    want = oracle.verify(z, start, drafts, ua, us, T)
    assert same(run_verify(ops, z, start, drafts, ua, us, T), want, start) > B - 40


def test_no_rows_and_no_entries(ops):
    e = lambda n, t=torch.float32: torch.zeros(n, dtype=t, device=DEV)
    i32 = torch.int32
    acc, tok = ops.verify_drafts(torch.zeros(0, 50, device=DEV), e(4, i32), e(0, i32), e(0), e(3), torch.ones(3, device=DEV))
    assert acc.tolist() == [0, 0, 0] and tok.numel() == 0
    tok = torch.full((2,), 7, dtype=i32, device=DEV)
    acc, tok = ops.verify_drafts(torch.zeros(2, 50, device=DEV), e(1, i32), e(2, i32), e(2), e(0), e(0), tokens=tok)
    assert acc.numel() == 0 and tok.tolist() == [7, 7]
    acc, tok = ops.verify_drafts(torch.zeros(2, 50, device=DEV), torch.tensor([1, 2], dtype=i32, device=DEV), e(2, i32), e(2), e(1), e(1), tokens=tok)      # a row of nobody's
    assert acc.tolist() == [0] and tok.tolist() == [7, 0] and ops.error_flags() == 0


def captured(run):
    run()
    torch.cuda.synchronize()
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        run()
    return g


def test_two_captured_verifications(ops):
    """two graphs with work areas of their own, replayed one after the other on inputs that have changed"""
    rng = np.random.default_rng(9)
    V, start = 20000, np.array([0, 3, 6])
    made = []
    for i in range(2):
        t = dict(z=up(rng.standard_normal((6, V)), np.float32), s=up(start, np.int32), d=up(rng.integers(0, V, 6), np.int32), ua=up(rng.random(6), np.float32), us=up(rng.random(2), np.float32),
                 T=up([1.0, 0.5], np.float32), k=up([40, 0], np.int32), a=torch.empty(2, dtype=torch.int32, device=DEV), t=torch.empty(6, dtype=torch.int32, device=DEV))
        made.append((t, captured(lambda t=t: ops.verify_drafts(t["z"], t["s"], t["d"], t["ua"], t["us"], t["T"], top_k=t["k"], accepted=t["a"], tokens=t["t"]))))
    for i in range(3):
        for t, g in made:
            t["z"].copy_(up(3 * rng.standard_normal((6, V)), np.float32))
            t["us"].copy_(up(rng.random(2), np.float32))
            t["d"].copy_(t["z"].argmax(1).to(torch.int32))
        for t, g in made:
            g.replay()
        torch.cuda.synchronize()
        for t, g in made:
            n = {k: v.cpu().numpy() for k, v in t.items()}
            want = oracle.verify(n["z"], start, n["d"], n["ua"], n["us"], n["T"], n["k"])
            same((n["a"], n["t"]), want, start)


# ---- weights of cached keys --------------------------------------------------------------------------------------------------------------------
class Step:
    """a step over pages of random rows; places that hold no key are NaN (f32) or 0xFF (4 bits)"""

    def __init__(self, ops, rng, lens, past, H, G, D, bits=32, bs=16, extra=0, spare=2):
        self.lens, self.past, self.H, self.G, self.D, self.bits, self.bs = lens, past, H, G, D, bits, bs
        B, T = len(lens), sum(lens)
        need = [-(-(p + n) // bs) for p, n in zip(past, lens)]
        total = sum(need) + spare
        perm = list(rng.permutation(total))
        self.tables = [[int(perm.pop()) for _ in range(m)] for m in need]
        mb = max(max(need), 1) + extra
        bt = np.full((B, mb), -1 if extra == 0 else 0, np.int32)
        for e, t in enumerate(self.tables):
            bt[e, :len(t)] = t
        self.keys = [(rng.standard_normal((p + n, G, D)) + 0.5 * rng.standard_normal((G, D))).astype(np.float32) for p, n in zip(past, lens)]
        if bits == 4:
            self.keys = [kv4_oracle.held(k) for k in self.keys]
        self.q = [rng.standard_normal((n, H, D)).astype(np.float32) for n in lens]
        self.total = total
        self.slots = rng.permutation(B + 2)[:B].astype(np.int32)
        i32 = lambda x: up(x, np.int32)
        self.start = np.concatenate([[0], np.cumsum(lens)])
        self.t = dict(ent=i32(np.repeat(np.arange(B), lens)), pos=i32(np.concatenate([np.arange(p, p + n) for p, n in zip(past, lens)] + [np.zeros(0)])), start=i32(self.start), slot=i32(self.slots),
                      pos0=i32(past), bt=i32(bt))
        t = self.t
        self.desc = ops.StepDesc(t["ent"].data_ptr(), t["pos"].data_ptr(), t["start"].data_ptr(), t["slot"].data_ptr(), t["pos0"].data_ptr(), t["bt"].data_ptr(), T, B, mb, bs)
        if bits == 32:
            pool = np.full((total, bs, G, D), np.nan, np.float32)
            for tab, k in zip(self.tables, self.keys):
                for j in range(len(k)):
                    pool[tab[j // bs], j % bs] = k[j]
            self.kpool = up(pool)
        else:
            NG = kv4_oracle.groups(D)
            pool = np.full((total, G, bs * NG * 20), 0xFF, np.uint8)
            raw = self.keys
            for tab, k in zip(self.tables, raw):
                for j in range(len(k)):
                    for g in range(G):
                        c, p = kv4_oracle.row_at(pool, bs, tab[j // bs], j % bs, g, NG)
                        c[:], p[:] = kv4_oracle.row_bytes(k[j, g], True)
            self.kpool = up(pool)
            # what the pages hold is what their bytes stand for (a value put in a second time may move by a rounding)
            self.keys = [kv4_oracle.held(k) for k in raw]

    def proj(self, wide=0, col=0):
        T = sum(self.lens)
        x = torch.full((T, col + self.H * self.D + wide), float("nan"), device=DEV)
        x[:, col:col + self.H * self.D] = up(np.concatenate([q.reshape(len(q), self.H * self.D) for q in self.q]))
        return x


def weigh(ops, s, chain, *, last=0, wide=0, room=7, max_keys=0, **kw):
    """runs and compares; returns the largest error over its bound"""
    rng = np.random.default_rng(1)
    H, G, D = s.H, s.G, s.D
    names = dict(head_scale=kw.get("head_scale"), sink=kw.get("sink"))
    dev = {k: up(v, np.float32) for k, v in names.items() if v is not None}
    layer = ops.attn_desc(H, G, D, D, kw.get("scale", D ** -0.5), gated=False, window=kw.get("window", 0), chunk=kw.get("chunk", 0), keep_first=kw.get("keep_first", 0), softcap=kw.get("softcap", 0.0),
                          kv_shared=True, **dev)
    cap = max(p + n for p, n in zip(s.past, s.lens)) + room
    acc0 = rng.random((len(s.lens) + 2, G, cap)).astype(np.float32)
    acc = up(acc0)
    ops.key_weights(s.proj(wide), s.desc, layer, s.kpool, acc, last=last, max_keys=max_keys)
    got = acc.cpu().numpy()
    want, most = oracle.key_weights(s.q, s.keys, s.past, s.lens, s.slots, acc0, G, kw.get("scale", D ** -0.5), last=last, window=kw.get("window", 0), chunk=kw.get("chunk", 0),
                                    keep_first=kw.get("keep_first", 0), softcap=kw.get("softcap", 0.0), **names)
    touched = np.zeros(acc0.shape, bool)
    old = np.array(acc0, np.float64)
    for e, n in enumerate(s.lens):
        if n:
            touched[s.slots[e], :, :s.past[e] + n] = True
            old[s.slots[e], :, s.past[e]:s.past[e] + n] = 0.0
    assert np.array_equal(got[~touched].view(np.uint32), acc0[~touched].view(np.uint32))
    rows = max(s.lens) * H // G
    rel = 2 * ((chain + 4) * 2.0 ** -24 * max(most, 1.0) + 2.0 ** -21) + rows * 2.0 ** -24
    bound = rel * (want - old) + 2.0 ** -23 * np.abs(want) + 1e-30
    off = np.abs(got - want)
    assert not np.isnan(got[touched]).any()
    assert (off <= bound)[touched].all(), float((off / bound)[touched].max())
    assert ops.error_flags() == 0
    return float((off / bound)[touched].max())


FEW = [  # lens, past, H, G, D
    ([1], [0], 4, 2, 64), ([1], [500], 32, 8, 64), ([1, 1, 1], [127, 128, 129], 8, 2, 128), ([5, 1, 3], [0, 1000, 17], 8, 4, 80), ([4], [300], 16, 1, 32), ([2, 1], [40, 4000], 12, 4, 96),
    ([1], [2000], 64, 1, 128), ([1, 0, 1], [33, 5, 60], 8, 8, 16), ([1], [1100], 40, 8, 100), ([3], [9], 2, 2, 4)]


@pytest.mark.parametrize("case", FEW, ids=lambda c: f"{c[0]}-{c[1]}-{c[2:]}")
@pytest.mark.parametrize("bits", [32, 4])
def test_weights_of_few_rows(ops, case, bits):
    lens, past, H, G, D = case
    if bits == 4 and max(past) > 1200:
        past = [min(p, 700) for p in past]
    s = Step(ops, np.random.default_rng(D + bits), lens, past, H, G, D, bits)
    weigh(ops, s, 14, wide=8)


def test_rows_that_take_several_passes_over_a_short_last_block(ops):
    """48 rows an entry go in two passes over its keys; most warps run out of keys before the last block's end"""
    rng = np.random.default_rng(31)
    s = Step(ops, rng, [12] * 32, [int(k) for k in rng.integers(500, 620, 32)], 32, 8, 128)
    weigh(ops, s, 128 + 14)


@pytest.mark.parametrize("kw", [dict(window=50), dict(window=50, keep_first=4), dict(chunk=64), dict(softcap=5.0), dict(sink=True), dict(head_scale=True), dict(scale=-0.3), dict(window=1), dict(last=2),
                                dict(softcap=2.0, sink=True, head_scale=True, window=40, keep_first=3)], ids=str)
@pytest.mark.parametrize("bits", [32, 4])
@pytest.mark.parametrize("lens,past", [([3, 1], [100, 290]), ([40, 70], [100, 0])])
def test_weights_under_masks(ops, kw, bits, lens, past):
    rng = np.random.default_rng(7)
    kw = dict(kw)
    H, G, D = 8, 2, 64
    if kw.get("sink"):
        kw["sink"] = rng.standard_normal(H).astype(np.float32) * 2
    if kw.get("head_scale"):
        kw["head_scale"] = rng.standard_normal(H).astype(np.float32)
    s = Step(ops, rng, lens, past, H, G, D, bits)
    weigh(ops, s, D + 14, **kw)


MANY = [([70], [0], 8, 2, 64, 0), ([200], [130], 8, 2, 128, 0), ([129], [64], 4, 4, 32, 0), ([300, 20, 1], [0, 600, 90], 8, 2, 64, 0), ([257], [0], 12, 4, 96, 0), ([64], [700], 16, 2, 80, 17), ([513], [33], 8, 1, 48, 64),
        ([33], [0], 8, 8, 20, 0), ([90], [40], 4, 2, 160, 0), ([50], [10], 6, 3, 7, 0)]


@pytest.mark.parametrize("case", MANY, ids=lambda c: f"{c[0]}-{c[1]}-{c[2:]}")
@pytest.mark.parametrize("bits", [32, 4])
def test_weights_of_many_rows(ops, case, bits):
    lens, past, H, G, D, last = case
    if bits == 4 and D > 128:
        pytest.skip("4-bit pages hold heads of up to 128 values")
    s = Step(ops, np.random.default_rng(D), lens, past, H, G, D, bits)
    weigh(ops, s, D + 14, last=last, wide=5 if D == 7 else 0)


@pytest.mark.parametrize("bs,extra,max_keys", [(16, 0, 0), (5, 3, 0), (32, 40, 0), (16, 600, 260), (1, 0, 0), (16, 600, 2000)])
@pytest.mark.parametrize("bits,n", [(32, 2), (4, 2), (32, 60), (4, 60)])
def test_weights_over_pages_of_other_sizes(ops, bs, extra, max_keys, bits, n):
    """pages that end inside a tile, tables for many more keys than there are"""
    s = Step(ops, np.random.default_rng(bs), [n, 1], [150, 200], 8, 2, 64, bits, bs, extra)
    weigh(ops, s, 64 + 14, max_keys=max_keys)


def test_keys_and_queries_of_large_range(ops):
    """one key takes all the weight; keys far beyond and far below one"""
    rng = np.random.default_rng(2)
    for n in (1, 90):
        for mag in (1e-6, 30.0, 1e5):
            s = Step(ops, rng, [n], [140], 8, 2, 64)
            s.keys = [k * np.float32(mag) for k in s.keys]
            s.q = [q * np.float32(min(1.0, 30.0 / mag)) for q in s.q]
            s.kpool = s.kpool * np.float32(mag)
            weigh(ops, s, 64 + 14)


def test_infinities_and_nan_in_masked_places(ops):
    """keys that a token does not see may be anything; rows that see nothing but scores of minus infinity give nothing"""
    rng = np.random.default_rng(4)
    for n, past in ((1, 200), (70, 200)):
        s = Step(ops, rng, [n], [past], 8, 2, 64)
        row = lambda j: s.kpool[s.tables[0][j // 16], j % 16]
        for j, x in ((3, float("nan")), (40, float("inf")), (41, 3e38)):
            row(j)[:] = x
            s.keys[0][j] = 0.0          # (outside every window: the oracle's are not read either)
        weigh(ops, s, 64 + 14, window=100)
    s = Step(ops, rng, [1], [20], 2, 2, 64)
    s.kpool[:] = float("-inf")
    s.q = [np.abs(q) + 0.1 for q in s.q]
    acc = torch.ones(3, 2, 30, device=DEV)
    layer = ops.attn_desc(2, 2, 64, 64, 0.125, gated=False, kv_shared=True)
    ops.key_weights(s.proj(), s.desc, layer, s.kpool, acc)
    want = torch.ones(3, 2, 30, device=DEV)
    want[int(s.slots[0]), :, 20] = 0.0
    assert torch.equal(acc, want)


def test_entries_that_are_none(ops):
    """slots and keys without a place: flagged, and nothing is written for them"""
    rng = np.random.default_rng(6)
    layer = ops.attn_desc(4, 2, 64, 64, 0.125, gated=False, kv_shared=True)
    for n in (1, 80):
        for what in ("slot", "low", "room", "pos", "table", "keys"):
            s = Step(ops, rng, [n, 1], [30, 40], 4, 2, 64)
            acc = torch.ones(4, 2, 41 if what == "room" else 200, device=DEV)
            if what == "slot":
                s.t["slot"][0] = 4
            elif what == "low":
                s.t["slot"][0] = -1
            elif what == "pos":
                s.t["pos0"][0] = -5
            elif what == "table":
                s.t["pos0"][0] = 16 * s.desc.max_blocks - n + 1
            elif what == "room" and n == 1:
                s.t["pos0"][0] = 41
            elif what == "keys":
                s.t["pos0"][0] = 130
            keys = 128 if what == "keys" and n == 1 else 0
            if what == "keys" and n > 1:
                continue
            bad = int(s.t["slot"][0])
            s2 = int(s.t["slot"][1])
            ops.key_weights(s.proj(), s.desc, layer, s.kpool, acc, max_keys=keys)
            assert ops.error_flags() == 1, what
            others = [i for i in range(4) if i != s2]
            assert torch.equal(acc[others], torch.ones_like(acc[others])), what
            assert not torch.equal(acc[s2], torch.ones_like(acc[s2])), what


@pytest.mark.parametrize("n", [4, 80, 300])
def test_starts_out_of_order(ops, n):
    """entries of overlapping tokens: flagged, and nothing beyond the entries' own rows is written"""
    rng = np.random.default_rng(8)
    s = Step(ops, rng, [n, 0, 0, 0, 0], [60, 0, 0, 0, 0], 16, 2, 64)
    layer = ops.attn_desc(16, 2, 64, 64, 0.125, gated=False, kv_shared=True)
    s.t["start"].copy_(up([0, n, 0, n, 0, n], np.int32))
    s.t["bt"].copy_(s.t["bt"][:1].expand(5, -1).contiguous())
    s.t["pos0"].fill_(60)
    acc = torch.ones(7, 2, n + 80, device=DEV)
    ops.key_weights(s.proj(), s.desc, layer, s.kpool, acc)
    assert ops.error_flags() == 1
    assert torch.equal(acc[:, :, n + 60:], torch.ones_like(acc[:, :, n + 60:]))
    spare = [i for i in range(7) if i not in s.slots[[0, 2, 4]]]
    assert torch.equal(acc[spare], torch.ones_like(acc[spare]))


def test_weights_captured_and_on_another_stream(ops):
    rng = np.random.default_rng(11)
    layer = ops.attn_desc(8, 2, 64, 64, 0.125, gated=False, kv_shared=True)
    for n in (1, 40):
        a, b = Step(ops, rng, [n, 2], [100, 300], 8, 2, 64), Step(ops, rng, [1, n], [50, 170], 8, 2, 64)
        want = []
        for s in (a, b):
            acc = torch.zeros(4, 2, 400, device=DEV)
            for _ in range(3):
                ops.key_weights(s.proj(), s.desc, layer, s.kpool, acc)
            want.append(acc)
        accs, qs = [torch.zeros(4, 2, 400, device=DEV) for _ in range(2)], [s.proj() for s in (a, b)]
        graphs = [captured(lambda s=s, acc=acc, q=q: ops.key_weights(q, s.desc, layer, s.kpool, acc)) for s, acc, q in zip((a, b), accs, qs)]
        for _ in range(2):
            for g in graphs:
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(accs[0], want[0]) and torch.equal(accs[1], want[1])
        side, acc = torch.cuda.Stream(), torch.zeros(4, 2, 400, device=DEV)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(3):
                ops.key_weights(qs[0], a.desc, layer, a.kpool, acc)
        side.synchronize()
        assert torch.equal(acc, want[0])


@pytest.mark.parametrize("n,past,last,D", [(700, 0, 0, 128), (100, 6000, 60, 64), (3, 5000, 0, 128)])
def test_calls_behind_one_another(ops, n, past, last, D):
    """steps of other sequences before and after, with nothing waited for: bit by bit what a call alone gives"""
    g = torch.Generator(device=DEV)
    g.manual_seed(n)
    H, G, keys = 32, 8, past + n
    pages = -(-keys // 16)
    layer = ops.attn_desc(H, G, D, D, D ** -0.5, gated=False, kv_shared=True)
    i32 = lambda x: up(x, np.int32)
    t = dict(ent=i32(np.zeros(n)), pos=i32(np.arange(past, keys)), start=i32([0, n]), slot=i32([0]), pos0=i32([past]), bt=i32(np.arange(pages)[None]))
    st = ops.StepDesc(t["ent"].data_ptr(), t["pos"].data_ptr(), t["start"].data_ptr(), t["slot"].data_ptr(), t["pos0"].data_ptr(), t["bt"].data_ptr(), n, 1, pages, 16)
    sets = [(torch.randn(n, H * D, device=DEV, generator=g), torch.randn(pages, 16, G, D, device=DEV, generator=g)) for _ in range(3)]
    want = []
    for q, k in sets:
        acc = torch.zeros(1, G, keys, device=DEV)
        ops.key_weights(q, st, layer, k, acc, last=last)
        torch.cuda.synchronize()
        want.append(acc)
    rows = (min(last, n) if last else n) * H // G
    for acc in want:
        assert abs(float(acc.double().sum()) - rows * G) < 1e-4 * rows * G
    for _ in range(25):
        accs = [torch.zeros(1, G, keys, device=DEV) for _ in sets]
        for (q, k), acc in zip(sets, accs):
            ops.key_weights(q, st, layer, k, acc, last=last)
        assert all(torch.equal(a, b) for a, b in zip(accs, want))


# ---- eviction ------------------------------------------------------------------------------------------------------------------------------------
def bytes_of(pool, bits, bs, G, page, o, g):
    if bits == 32:
        return pool[page, o, g].copy()
    NG = pool.shape[2] // (20 * bs)
    return np.concatenate(kv4_oracle.row_at(pool, bs, page, o, g, NG))


def put_bytes(pool, bits, bs, G, page, o, g, x):
    if bits == 32:
        pool[page, o, g] = x
    else:
        NG = pool.shape[2] // (20 * bs)
        c, p = kv4_oracle.row_at(pool, bs, page, o, g, NG)
        c[:], p[:] = x[:16 * NG], x[16 * NG:]


def evict(ops, rng, rows, keep, first, recent, L=2, G=2, D=64, V=None, bits=32, bs=16, inplace=True, weights=None, odd=False):
    B, V = len(rows), V or D
    need = [-(-n // bs) for n in rows]
    mine = [-(-min(n, keep) // bs) for n in rows]
    total = sum(need) + (0 if inplace else sum(mine)) + 2
    perm = list(rng.permutation(total))
    tab = [[int(perm.pop()) for _ in range(m)] for m in need]
    to = tab if inplace else [[int(perm.pop()) for _ in range(m)] for m in mine]
    full = lambda ts, w: np.array([t + [-1] * (w - len(t)) for t in ts], np.int32)
    table, to_table = full(tab, max(max(need), 1)), full([t[:m] for t, m in zip(to, mine)], max(max(mine), 1))
    slots = rng.permutation(2 * B + 1).astype(np.int32)
    src, dst = slots[:B], (slots[:B] if inplace else slots[B:2 * B])
    cap = max(rows) + 3
    if bits == 32:
        make = lambda d: rng.standard_normal((total, bs, G, d)).astype(np.float32)
    else:
        make = lambda d: rng.integers(0, 256, (total, G, bs * kv4_oracle.groups(d) * 20), dtype=np.uint8)
    kp, vp = [make(D) for _ in range(L)], [make(V) for _ in range(L)]
    ac = [(rng.random((2 * B + 1, G, cap)) if weights is None else weights(rng, (2 * B + 1, G, cap))).astype(np.float32) for _ in range(L)]

    def dev(x):
        if not odd:
            return up(x)
        flat = torch.empty(x.size + 1, dtype=torch.from_numpy(x).dtype, device=DEV)      # from the second number on: rows that no 16-byte piece fits
        flat[1:] = up(x).reshape(-1)
        return flat[1:].view(x.shape)
    dk, dv, da = [dev(x) for x in kp], [dev(x) for x in vp], [up(x) for x in ac]
    kw = {} if inplace else dict(to_table=up(to_table), to_slots=up(dst))
    kept = ops.evict_keys(dk, dv, da, up(src), up(np.array(rows, np.int32)), up(table), keep, first=first, recent=recent, block_size=bs, **kw).cpu().numpy()
    wk, wv, wa = [x.copy() for x in kp], [x.copy() for x in vp], [x.copy() for x in ac]
    for l in range(L):
        for e, n in enumerate(rows):
            for g in range(G):
                st = oracle.stays(ac[l][src[e], g, :n], n, keep, first, recent)
                np.testing.assert_array_equal(kept[l, e, g], st + [-1] * (keep - len(st)), err_msg=f"layer {l} entry {e} head {g}")
                for i, j in enumerate(st):
                    for w, p in ((wk, kp), (wv, vp)):
                        put_bytes(w[l], bits, bs, G, to[e][i // bs], i % bs, g, bytes_of(p[l], bits, bs, G, tab[e][j // bs], j % bs, g))
                    wa[l][dst[e], g, i] = ac[l][src[e], g, j]
    for a, b in zip(dk + dv + da, wk + wv + wa):
        assert np.array_equal(a.cpu().numpy().view(np.uint8), b.view(np.uint8))
    assert ops.error_flags() == 0


@pytest.mark.parametrize("bits", [32, 4])
@pytest.mark.parametrize("inplace", [True, False])
@pytest.mark.parametrize("rows,keep,first,recent", [([100], 60, 4, 10), ([61, 60, 59, 1, 0], 60, 2, 5), ([300, 700], 256, 0, 0), ([90], 20, 10, 10), ([50], 1, 0, 0), ([50], 1, 1, 0), ([50], 1, 0, 1),
                                                    ([5000, 40], 33, 1, 7), ([4200], 4100, 0, 3)])
def test_sequences_are_cut_back(ops, bits, inplace, rows, keep, first, recent):
    evict(ops, np.random.default_rng(keep), rows, keep, first, recent, bits=bits, inplace=inplace, L=1 if max(rows) > 1000 else 2)


@pytest.mark.parametrize("kw", [dict(D=128, V=64), dict(D=20), dict(D=7, V=5), dict(D=64, odd=True), dict(D=80, bs=5), dict(D=32, bs=1), dict(G=1, D=256), dict(G=8, D=16, bs=48), dict(L=35, G=1, D=8),
                                dict(bits=4, D=128, V=32), dict(bits=4, D=20, bs=5), dict(bits=4, D=96, V=128, bs=32), dict(bits=4, L=33, G=1, D=32)], ids=str)
def test_pools_of_other_shapes(ops, kw):
    for inplace in (True, False):
        evict(ops, np.random.default_rng(3), [130, 70], 64, 3, 9, inplace=inplace, **kw)


@pytest.mark.parametrize("name,weights", [
    ("equal", lambda r, s: np.ones(s)), ("few values", lambda r, s: r.integers(0, 3, s)), ("zeros of either sign", lambda r, s: np.where(r.random(s) < 0.5, 0.0, -0.0)),
    ("negative", lambda r, s: -r.random(s)), ("infinite", lambda r, s: r.choice([np.inf, -np.inf, 0.0, 1.0], s)), ("nan", lambda r, s: np.where(r.random(s) < 0.6, np.nan, r.random(s))),
    ("tiny", lambda r, s: r.random(s) * 1e-44), ("neighbours", lambda r, s: 1 + r.integers(0, 50, s) * 2.0 ** -23)])
def test_ties_and_odd_weights(ops, name, weights):
    evict(ops, np.random.default_rng(5), [500, 333], 201, 3, 20, weights=weights, G=3, D=8)
    evict(ops, np.random.default_rng(6), [9000], 4500, 0, 0, weights=weights, G=1, D=4, L=1)


def test_entries_that_cannot_be_cut(ops):
    """no slot, more rows than there is room or pages for, negative pages: flagged, the others are cut"""
    G, bs = 2, 16
    for what in ("slot", "to", "room", "table", "negative", "page"):
        pools = [torch.randn(20, bs, G, 8, device=DEV) for _ in range(2)]
        acc = torch.rand(4, G, 120, device=DEV)
        table = torch.arange(16, dtype=torch.int32, device=DEV).reshape(2, 8).contiguous()
        slots, rows, to = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([1, 2], [100, 100], [1, 2]))
        if what == "slot":
            slots[0] = 4
        elif what == "to":
            to[0] = -1
        elif what == "room":
            rows[0] = 121
        elif what == "table":
            rows[0] = 115
            table = table[:, :7].contiguous()
        elif what == "negative":
            rows[0] = -3
        elif what == "page":
            table[0, 0] = -1
        before = [p.clone() for p in pools] + [acc.clone()]
        kept = ops.evict_keys(pools[:1], pools[1:], [acc], slots, rows, table, 50, recent=10, to_slots=to)
        assert ops.error_flags() == 1, what
        lo = 0 if what != "page" else None
        if lo is not None:
            assert (kept[0, 0] == -1).all(), what
            first_pages = table[0].long()
            assert all(torch.equal(p[first_pages], b[first_pages]) for p, b in zip(pools, before)), what
        assert (kept[0, 1] >= 0).all() and not torch.equal(pools[0][table[1].long()], before[0][table[1].long()])


def test_eviction_captured(ops):
    rng = np.random.default_rng(13)
    pools = [torch.randn(12, 16, 2, 64, device=DEV) for _ in range(4)]
    acc = [torch.rand(2, 2, 100, device=DEV) for _ in range(2)]
    table = torch.arange(12, dtype=torch.int32, device=DEV).reshape(2, 6).contiguous()
    slots, rows = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 1], [90, 80]))
    kept = torch.empty(2, 2, 2, 48, dtype=torch.int32, device=DEV)
    run = lambda p, a, k: ops.evict_keys(p[:2], p[2:], a, slots, rows, table, 48, first=2, recent=8, kept=k)
    mine, macc = [p.clone() for p in pools], [a.clone() for a in acc]
    g = captured(lambda: run(mine, macc, kept))
    for p, q in zip(mine + macc, pools + acc):
        p.copy_(q)
    g.replay()
    torch.cuda.synchronize()
    want = run(pools, acc, None)
    assert torch.equal(kept, want) and all(torch.equal(a, b) for a, b in zip(mine + macc, pools + acc))


def test_attended_weighed_and_cut_back(ops):
    """the three as they are used: a prompt's weights, the cache cut back by them, attention of the next token over what is left"""
    rng = np.random.default_rng(17)
    H, G, D, n, keep = 8, 2, 64, 120, 48
    s = Step(ops, rng, [n], [0], H, G, D)
    vals = rng.standard_normal((n, G, D)).astype(np.float32)
    vpool = torch.zeros_like(s.kpool)
    for j in range(n):
        vpool[s.tables[0][j // 16], j % 16] = up(vals[j])
    kpool = torch.nan_to_num(s.kpool)
    acc = torch.zeros(3, G, 200, device=DEV)
    layer = ops.attn_desc(H, G, D, D, D ** -0.5, gated=False, kv_shared=True)
    ops.key_weights(s.proj(), s.desc, layer, kpool, acc)
    w, _ = oracle.key_weights(s.q, s.keys, [0], [n], s.slots, np.zeros((3, G, 200)), G, D ** -0.5)
    slot = int(s.slots[0])
    kept = ops.evict_keys([kpool], [vpool], [acc], s.t["slot"], up([n], np.int32), s.t["bt"], keep, first=2, recent=8)[0, 0].cpu().numpy()
    # a query at row keep - 1 attends over the kept rows
    q = rng.standard_normal((1, H * D)).astype(np.float32)
    i32 = lambda x: up(x, np.int32)
    t = dict(e=i32([0]), p=i32([keep - 1]), s=i32([0, 1]), b=s.t["bt"])
    st = ops.StepDesc(t["e"].data_ptr(), t["p"].data_ptr(), t["s"].data_ptr(), s.t["slot"].data_ptr(), t["p"].data_ptr(), t["b"].data_ptr(), 1, 1, t["b"].shape[1], 16)
    out = torch.empty(1, H * D, device=DEV)
    ops.attn_ex(up(q), st, layer, kpool, vpool, out)
    for h in range(H):
        g = h // (H // G)
        assert sorted(kept[g]) == list(kept[g]) and list(kept[g][:2]) == [0, 1] and list(kept[g][-8:]) == list(range(n - 8, n))
        # the kept ones have the largest weights: none that went is above one that stayed by more than the sums are off
        mid = [j for j in kept[g] if 2 <= j < n - 8]
        gone = [j for j in range(2, n - 8) if j not in set(mid)]
        assert w[slot, g, gone].max() <= w[slot, g, mid].min() * (1 + 1e-4)
        k, v = s.keys[0][kept[g], g].astype(np.float64), vals[kept[g], g].astype(np.float64)
        z = k @ q[0, h * D:(h + 1) * D].astype(np.float64) * D ** -0.5
        p = np.exp(z - z.max())
        np.testing.assert_allclose(out[0, h * D:(h + 1) * D].cpu().numpy(), (p / p.sum()) @ v, atol=2e-5)
    assert ops.error_flags() == 0
