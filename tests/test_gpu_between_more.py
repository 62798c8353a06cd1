"""Drafts verified, the weight of cached keys and eviction at places that test_gpu_between_steps.py does not reach (its docstring has the roundings that the bounds count)."""
import numpy as np
import pytest
import torch

import between_oracle as oracle
from test_gpu_between_steps import DEV, Step, evict, ops, run_verify, up, weigh  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- drafts: shares near one ---------------------------------------------------------------------------------------------------------------
# A token that top_p keeps is accepted at accept_u = 0, one that it does not keep is not.  The mass before a token is known to the roundings of the tail's weights (2^-19 of the tail,
# in that mass and in the whole), to those of the whole numbers that masses are added up in (2^-43 a weight) and to the weights that are left out (2^-46 each).  Tokens whose
# mass before them is within that of the share may go either way.
TAILS = {
    "flat": lambda r, n: np.full(n, -23.0),
    "one bin": lambda r, n: -23.0 - r.random(n) / 80,
    "two units": lambda r, n: -22.0 - 2 * r.random(n),
    "two units, cold": lambda r, n: 0.25 * (-22.0 - 2 * r.random(n)),
    "far": lambda r, n: -24.5 - 4 * r.random(n),
}


@pytest.mark.parametrize("tail", TAILS)
@pytest.mark.parametrize("top_k", [0, 60000])
@pytest.mark.parametrize("V", [50257, 128256])
def test_shares_near_one_keep_their_tail(ops, tail, top_k, V):
    rng = np.random.default_rng(V)
    z = np.empty(V, np.float32)
    z[0] = 0.0
    z[1:] = TAILS[tail](rng, V - 1)
    T = 0.25 if "cold" in tail else 1.0
    w = np.exp(z.astype(np.float64) / T)
    if 0 < top_k < V:
        w[z < np.sort(z)[::-1][top_k - 1]] = 0.0
    total = w.sum()
    order = np.argsort(-z, kind="stable")
    before = np.cumsum(w[order]) - w[order]
    before = before[np.searchsorted(-z[order], -z[order], side="left")]        # (equal ones together)
    share = np.float32(1.0 - 0.3 * (1.0 - w[0] / total))
    x = order[np.unique(np.linspace(1, V - 1, 60).astype(int))]
    rank = np.argsort(order)[x]
    near = V * (2.0 ** -43 + 2.0 ** -46) + 2.0 ** -18 * (1.0 - w[0] / total)
    sure = np.abs(before[rank] - float(share) * total) > near * total
    keep = (before[rank] < float(share) * total) & (w[x] > 0)
    B = len(x)
    rows, two = up(z).expand(2 * B, V).contiguous(), lambda a: np.stack([a, 0 * a], 1).reshape(-1)
    got, _ = run_verify(ops, rows, np.arange(0, 2 * B + 1, 2), two(x), np.zeros(2 * B), np.full(B, 0.5), np.full(B, T), [top_k] * B if top_k else None, [share] * B)
    assert sure.sum() >= B // 2 and keep[sure].any()
    np.testing.assert_array_equal(got[sure], keep[sure].astype(int))
    assert ops.error_flags() == 0


# ---- drafts: draws beside the border of two tokens ---------------------------------------------------------------------------------------------
# sample_u is the f32 number next to the share of the weights up to some token, so that the target is 2^-25 of the whole from a border at most.  Weights are known to 2^-34 of themselves and so is
# their sum up to any token; where a draft's distribution is taken off them, to 2^-33 of the target's whole.  Entries nearer than 2^-32 of the whole may go either way.
@pytest.mark.parametrize("form", ["sampled", "certain draft", "drafted", "top_p"])
@pytest.mark.parametrize("V,T", [(128256, 1.0), (50257, 0.6), (131072, 3.0), (1000, 1.0)])
def test_draws_beside_a_border(ops, form, V, T):
    rng = np.random.default_rng(V)
    B, z = 120, (2 * rng.standard_normal(V)).astype(np.float32)
    p = oracle.probabilities(z, float(np.float32(T)), 0, float(np.float32(0.9)) if form == "top_p" else 1.0)      # (of the numbers that the call gets)
    n, q, x = (1 if "draft" in form else 0), None, int(z.argmin())
    w = np.array(p)
    if form == "certain draft":
        w[x] = 0.0
    elif form == "drafted":
        y = z / T + 0.5 * rng.standard_normal(V)
        y[x] += 12.0
        q = np.exp(y - y.max())
        q = (q / q.sum()).astype(np.float32)
        w = np.maximum(p - q, 0.0)
    cum = np.cumsum(w) / w.sum()
    some = np.nonzero(w)[0][:-1]
    us = cum[some[(np.arange(B) * (len(some) / B)).astype(int)]].astype(np.float32)
    R = B * (n + 1)
    start = np.arange(B + 1) * (n + 1)
    args = (start, np.full(R, x), np.full(R, 1 - 2.0 ** -24, np.float32), us, np.full(B, T, np.float32), None, np.full(B, 0.9, np.float32) if form == "top_p" else None)
    got = run_verify(ops, up(z).expand(R, V).contiguous(), *args, None if q is None else up(q).expand(R, V).contiguous())
    near = np.abs(cum[None, some] - us[:, None].astype(np.float64)).min(1) * w.sum()
    want = np.minimum(np.searchsorted(cum, us.astype(np.float64), side="right"), some[-1] + 1)
    sure = near > 2.0 ** -32
    assert sure.sum() >= B // 2 and (near < 2.0 ** -20).all()
    np.testing.assert_array_equal(got[0], 0)
    np.testing.assert_array_equal(got[1][::n + 1][sure], want[sure])


# ---- weights: heads whose sink is none -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kw", [dict(window=50), dict(chunk=64), dict(window=50, keep_first=3), dict(softcap=3.0, window=50), dict()], ids=str)
@pytest.mark.parametrize("lens,past,H,G", [([300], [700], 4, 4), ([3], [700], 4, 4), ([130, 1], [0, 400], 8, 2), ([40], [900], 8, 1)])
@pytest.mark.parametrize("bits", [32, 4])
def test_sinks_of_minus_infinity(ops, kw, lens, past, H, G, bits):
    """such a head has no sink: also where a part of the walk over the keys has none that the row sees"""
    s = Step(ops, np.random.default_rng(H), lens, past, H, G, 64, bits)
    sink = np.where(np.arange(H) % 2 == 0, -np.inf, 0.7).astype(np.float32)
    weigh(ops, s, 64 + 14, sink=sink, **kw)


@pytest.mark.parametrize("n", [1, 90])
@pytest.mark.parametrize("sink", [None, -np.inf, 0.5])
def test_rows_that_see_nothing_but_minus_infinity(ops, n, sink):
    s = Step(ops, np.random.default_rng(5), [n], [400], 2, 2, 64)
    s.kpool[:] = float("-inf")
    s.q = [np.abs(q) + 0.1 for q in s.q]
    acc = torch.ones(3, 2, 500, device=DEV)
    dev = None if sink is None else torch.full((2,), sink, device=DEV)
    ops.key_weights(s.proj(), s.desc, ops.attn_desc(2, 2, 64, 64, 0.125, gated=False, kv_shared=True, sink=dev), s.kpool, acc)
    want = torch.ones(3, 2, 500, device=DEV)
    want[int(s.slots[0]), :, 400:400 + n] = 0.0
    assert torch.equal(acc, want) and ops.error_flags() == 0


@pytest.mark.parametrize("B,n,past,G,D,bits,launches", [(4, 8, 500, 8, 128, 32, 2), (3, 8, 500, 8, 128, 32, 1), (9, 8, 240, 8, 128, 32, 2), (18, 8, 100, 8, 128, 32, 1), (6, 16, 250, 8, 128, 32, 2),
                                                        (4, 8, 500, 8, 64, 32, 1), (4, 8, 500, 8, 128, 4, 1), (4, 6, 500, 8, 128, 32, 1)])
def test_steps_are_joined_where_their_blocks_fit(ops, B, n, past, G, D, bits, launches):
    """four tiles of rows with f32 keys above 64 values: one block an SM instead of two, and one launch up to two waves of clusters"""
    s = Step(ops, np.random.default_rng(B), [n] * B, [past] * B, 4 * G, G, D, bits)
    before = ops.launch_count()
    weigh(ops, s, D + 14)
    assert ops.launch_count() - before == launches


# ---- eviction in place -------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kw", [dict(rows=[9000], keep=8000, L=1, G=4, D=128), dict(rows=[7000, 6500], keep=3000, L=2, G=2, D=80), dict(rows=[6000], keep=5990, L=1, G=1, D=600),
                                dict(rows=[5000] * 3, keep=4900, L=2, G=2, D=128, bits=4), dict(rows=[4000], keep=3999, L=1, G=3, D=7)], ids=str)
def test_long_sequences_are_cut_back_where_they_lie(ops, kw):
    """clusters of several blocks, many chunks each, rows that move by few places and by many"""
    kw = dict(kw)
    for seed in (1, 2):
        evict(ops, np.random.default_rng(seed), kw["rows"], kw["keep"], 4, 50, **{k: v for k, v in kw.items() if k not in ("rows", "keep")})
