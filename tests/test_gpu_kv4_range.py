"""Attention over 4-bit pages (csrc/seq/seq_attn4.cu, seq_attn4_tc.cu) at the ends of its range: groups as wide as the cache holds, rows that one key dominates.

Errors are bounded element by element.  With M_j the largest value that the group of value j can stand for (|m| + 15 s, larger than any of its parts) and w the soft-max weights
in 64 bits, roundings that are relative to a weight or to a sum's terms move a result by at most their size times sum w M.  f32 results: as in test_gpu_kv4.py, 4e-6 for weights,
powers and sums; scores: q is off by 2^-22 of a value, the products and sums of a score by 2^-22 of its terms, together 2^-21 of A = scale sum |q| (|m| + 15 s), which a weight and
the weights' sum each take in: 2^-20 A.  bf16 results: half a step is 2^-8 of a value, and q and the weights may be f16 numbers (2^-11 of a value each): 2^-7 and 2^-10 A.
Weights are f16 parts of the weight times 2^13 or more (bf16 results: 2^10 or more), whose spacing ends at 2^-24, half of which is 2^-25: each is off by up to 2^-38 (2^-35) of
the largest weight however small it is, together that much of sum M."""
import numpy as np
import pytest
import torch

import kv4_oracle as ref
import test_gpu_kv4 as base

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from blazr_b200 import seqops
    seqops.lib()
    seqops.error_flags()
    return seqops


def largest(x):
    """|m| + 15 s of the group of every value of rows x [.., D]"""
    _, s, m = ref.quantise(x)
    return (np.abs(m) + 15.0 * s)[..., np.arange(x.shape[-1]) // 32].astype(np.float64)


def check(ops, entries, q, k, v, scale, odt, bs=16, sink=None, softcap=0.0):
    """q [T, H, D], k and v: [positions, G, D] of every entry"""
    rng = np.random.default_rng(len(entries))
    H, D = q.shape[1:]
    G, V = k[0].shape[1], v[0].shape[2]
    st, keep, slots, pages = base.step(ops, entries, bs, rng)
    kp, vp = ops.kv4_pool(pages, bs, G, D, DEV), ops.kv4_pool(pages, bs, G, V, DEV)
    whole = [torch.from_numpy(np.concatenate(x).astype(np.int32)).to(DEV) for x in ([np.full(len(y), i) for i, y in enumerate(k)], [np.arange(len(y)) for y in k])]
    rows = ops.StepDesc(whole[0].data_ptr(), whole[1].data_ptr(), 0, 0, 0, keep["block_table"].data_ptr(), len(whole[0]), st.B, st.max_blocks, bs)
    dev = lambda x: torch.from_numpy(np.concatenate(x).reshape(len(whole[0]), -1)).to(DEV)
    ops.kv4_store(dev(k), dev(v), rows, kp, vp)
    dev_sink = torch.from_numpy(sink).to(DEV) if sink is not None else None
    d = ops.attn_desc(H, G, D, V, scale, gated=False, kv_shared=True, sink=dev_sink, softcap=softcap)
    out = torch.empty(st.T, H * V, device=DEV, dtype=odt)
    ops.attn_kv4(torch.from_numpy(q.reshape(st.T, H * D)).to(DEV), st, d, kp, vp, out)
    assert ops.error_flags() == 0
    out = out.double().cpu().numpy().reshape(st.T, H, V)
    tol, part, least, r0 = (4e-6, 2.0 ** -20, 2.0 ** -38, 0) if odt == F32 else (2.0 ** -7, 2.0 ** -10, 2.0 ** -35, 0)
    for e, (n, past) in enumerate(entries):
        pos, qe = np.arange(past, past + n), q[r0:r0 + n]
        M, K = largest(v[e]), largest(k[e])
        both = ref.attend(qe, ref.held(k[e]).astype(np.float64), np.concatenate([ref.held(v[e]), M], -1), pos, scale, softcap=softcap, sink=sink)
        want, near = both[..., :V], both[..., V:]
        top = np.maximum.accumulate(K, 0)[pos]                         # [n, G, D]: more than any key that a row sees
        A = np.stack([(np.abs(qe[:, h]) * top[:, h // (H // G)]).sum(1) for h in range(H)], 1) * abs(scale)
        far = np.cumsum(M, 0)[pos]
        far = np.stack([far[:, h // (H // G)] for h in range(H)], 1) * least
        err, bound = np.abs(out[r0:r0 + n] - want), near * (tol + part * A[..., None]) + far
        assert np.isfinite(out[r0:r0 + n]).all()
        assert (err <= bound).all(), (e, float((err / bound).max()), np.argwhere(err > bound)[:4].tolist())
        r0 += n


STEPS = [  # entries, H, G, D, V
    # few rows: single tokens, drafts, short prompts; the keys of one sequence dealt out
    ([(1, 70), (4, 37)], 8, 2, 64, 64), ([(1, 300)], 8, 2, 128, 128), ([(1, 40)], 4, 2, 32, 32), ([(3, 60)], 4, 2, 80, 48), ([(40, 30)], 8, 2, 64, 64), ([(1, 30000)], 8, 2, 64, 64),
    # many rows on the tensor cores: two row tiles a CTA, one; keys in parts
    ([(600, 0)], 64, 8, 64, 64), ([(600, 5)], 64, 16, 32, 32), ([(300, 200)], 32, 4, 128, 128), ([(200, 100)], 64, 2, 128, 104), ([(250, 1500)], 32, 4, 64, 64), ([(300, 2000)], 16, 2, 32, 24),
]


@pytest.mark.parametrize("entries,H,G,D,V", STEPS)
@pytest.mark.parametrize("odt", [F32, BF16])
@pytest.mark.parametrize("span", [13000.0, 14000.0, 60000.0])
@pytest.mark.parametrize("which", ["keys", "values"])
def test_groups_as_wide_as_the_cache_holds(ops, entries, H, G, D, V, odt, span, which):
    """one row of every sequence, among those that some of its tokens may not see where it has several, and the sequence's first one"""
    rng = np.random.default_rng(int(span) + D)
    f32 = lambda *s: rng.standard_normal(s).astype(np.float32)
    T = sum(n for n, _ in entries)
    k, v = [f32(n + p, G, D) for n, p in entries], [f32(n + p, G, V) for n, p in entries]
    for (n, p), x in zip(entries, k if which == "keys" else v):
        for at in (0, p + n // 2):
            x[at] = rng.uniform(-span / 2, span / 2, x[at].shape)
            x[at, :, 0], x[at, :, 1] = -span / 2, span / 2
    scale = 0.25 / D ** 0.5 / (span / 4 if which == "keys" else 1.0)
    check(ops, entries, f32(T, H, D), k, v, scale, odt)


@pytest.mark.parametrize("entries,H,G,D", [([(1, 5000)], 8, 2, 64), ([(1, 5000)], 8, 2, 128), ([(1, 2500)] * 20, 8, 2, 64), ([(4, 3000), (1, 700)], 8, 2, 128),
                                           ([(1, 30000)], 8, 2, 64),
                                           ([(600, 0)], 64, 8, 64), ([(300, 200)], 32, 4, 128), ([(300, 2000)], 16, 2, 32), ([(250, 1500)], 32, 4, 64), ([(150, 2500)], 32, 4, 128)])
@pytest.mark.parametrize("odt", [F32, BF16])
@pytest.mark.parametrize("gap", [12.0, 15.0, 18.0])
@pytest.mark.parametrize("first", [True, False])
def test_rows_that_one_key_dominates(ops, entries, H, G, D, odt, gap, first):
    """a key `gap` nats above the others, with a value of zeros: the rows are what the others leave"""
    rng = np.random.default_rng(int(gap) + D)
    f32 = lambda *s: rng.standard_normal(s).astype(np.float32)
    T = sum(n for n, _ in entries)
    e = np.ones(D, np.float32)
    q = (e + 0.1 * f32(T, H, D)).astype(np.float32)
    k, v = [0.3 * f32(n + p, G, D) for n, p in entries], [1 + 0.3 * f32(n + p, G, D) for n, p in entries]
    for (n, p), x, y in zip(entries, k, v):
        at = 0 if first else p // 2
        x[at], y[at] = gap, 0.0
    check(ops, entries, q, k, v, 1.0 / D, odt)


@pytest.mark.parametrize("entries,H,G,D", [([(1, 2000)], 8, 2, 128), ([(5, 900)], 8, 2, 64), ([(600, 0)], 64, 8, 64), ([(250, 1500)], 32, 4, 64), ([(150, 2500)], 32, 4, 128)])
@pytest.mark.parametrize("odt", [F32, BF16])
def test_dominated_rows_with_sinks_and_caps(ops, entries, H, G, D, odt):
    rng = np.random.default_rng(D)
    f32 = lambda *s: rng.standard_normal(s).astype(np.float32)
    T = sum(n for n, _ in entries)
    q = (1 + 0.1 * f32(T, H, D)).astype(np.float32)
    k, v = [0.3 * f32(n + p, G, D) for n, p in entries], [f32(n + p, G, D) for n, p in entries]
    check(ops, entries, q, k, v, 1.0 / D, odt, sink=np.linspace(-20, 20, H).astype(np.float32))
    for x, y in zip(k, v):
        x[3], y[3] = 14.0, 0.0
    check(ops, entries, q, k, v, 1.0 / D, odt, sink=np.linspace(-20, 20, H).astype(np.float32))
    check(ops, entries, q, k, v, 1.0 / D, odt, softcap=30.0)


@pytest.mark.parametrize("entries,H,G,D", [([(1, 400), (50, 30)], 8, 2, 64), ([(300, 200)], 32, 4, 128), ([(600, 0)], 64, 8, 64), ([(300, 2000)], 16, 2, 32)])
@pytest.mark.parametrize("odt", [F32, BF16])
def test_keys_around_different_places(ops, entries, H, G, D, odt):
    """minima of ten times the spread beside them, other ones for every key, so that a score's large parts are not common to all"""
    rng = np.random.default_rng(D + 1)
    f32 = lambda *s: rng.standard_normal(s).astype(np.float32)
    T = sum(n for n, _ in entries)
    k, v = [f32(n + p, G, D) + 10 * f32(n + p, G, 1) for n, p in entries], [f32(n + p, G, D) for n, p in entries]
    check(ops, entries, f32(T, H, D), k, v, 0.02, odt)


@pytest.mark.parametrize("entries,H,G,D", [([(1, 300)], 8, 2, 64), ([(1, 30000)], 8, 2, 64), ([(40, 30)], 8, 2, 128), ([(600, 0)], 64, 8, 64), ([(300, 200)], 32, 4, 128),
                                           ([(250, 1500)], 32, 4, 64), ([(300, 2000)], 16, 2, 32)])
@pytest.mark.parametrize("odt", [F32, BF16])
@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 23, 1.3 * 2.0 ** 24, 1.3 * 2.0 ** 25, 2.0 ** 26])
def test_scores_of_any_size(ops, entries, H, G, D, odt, size):
    """one key of every row scores `size` (base 2: 1.44 times that), the others a tenth of it: the row is that key's value, to the roundings of one weight and of the result.
    An f32 score of that size is a multiple of up to 8, and so is what the weight's exponent may be below 0: 2^-16 of the largest a weight can be has 11 bits and more in two
    parts, 2^-24 / 2^-16 / 2^13 of them the last (f32 results: 2^-21); in one part half of 2^-10 (bf16 results, beside the half step of the result of 2^-8)."""
    rng = np.random.default_rng(D)
    f32 = lambda *s: rng.standard_normal(s).astype(np.float32)
    (n, p), = entries
    q = (1 + 0.02 * f32(n, H, D)).astype(np.float32)
    k, v = 0.05 * f32(n + p, G, D), f32(n + p, G, D)
    k[0], k[n // 2 + p] = 8.0, 16.0                                    # rows see the first, the later ones the second too
    st, keep, slots, pages = base.step(ops, entries, 16, rng)
    kp, vp = (torch.from_numpy(np.zeros((pages, G, ops.kv4_page_bytes(16, 1, D)), np.uint8)).to(DEV) for _ in range(2))
    ent, pos = torch.zeros(n + p, dtype=torch.int32, device=DEV), torch.arange(n + p, dtype=torch.int32, device=DEV)
    rows = ops.StepDesc(ent.data_ptr(), pos.data_ptr(), 0, 0, 0, keep["block_table"].data_ptr(), n + p, 1, st.max_blocks, 16)
    ops.kv4_store(torch.from_numpy(k.reshape(n + p, -1)).to(DEV), torch.from_numpy(v.reshape(n + p, -1)).to(DEV), rows, kp, vp)
    d = ops.attn_desc(H, G, D, D, size / (16 * D), gated=False, kv_shared=True)
    out = torch.empty(n, H * D, device=DEV, dtype=odt)
    ops.attn_kv4(torch.from_numpy(q.reshape(n, -1)).to(DEV), st, d, kp, vp, out)
    got = out.double().cpu().numpy().reshape(n, G, H // G, D)
    first, later = (ref.held(v[i]).astype(np.float64) for i in (0, n // 2 + p))
    want = np.stack([later if i >= n // 2 else first for i in range(n)])[:, :, None]
    M = np.stack([largest(v[n // 2 + p]) if i >= n // 2 else largest(v[0]) for i in range(n)])[:, :, None]
    err = np.abs(got - want)
    assert np.isfinite(got).all() and (err <= M * (4e-6 if odt == F32 else 2.0 ** -7)).all(), float((err / M).max())
