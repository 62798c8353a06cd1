"""The KV cache held in 4 bits (csrc/seq/seq_kv4.cu, seq_attn4.cu): rows into and out of pages, and attention over them, against the restatement of
tests/kv4_oracle.py.

Stored bytes are exact: every step of the rounding is one f32 operation with one result.  Attention, f32 results: q and the weights enter as 22 bits (2^-22 of a
term each), a power is good to 2^-22, sums of at most a few hundred terms in f32 lose a few 2^-24 of their magnitude, a score of magnitude 2^4 carries 2^4 of its own
roundings into its power (2^-20): 4e-6 of the largest value.  bf16 results: half a step, 2^-9 of a value, is within 2^-8 of the largest."""
import numpy as np
import pytest
import torch

import kv4_oracle as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from blazr_b200 import seqops
    seqops.lib()
    seqops.error_flags()
    return seqops


def step(ops, entries, bs, rng, spare=2):
    """entries [(tokens, past)] -> (descriptor, arrays to keep, slots of every position of every entry, pages of the pool); pages in random order, `spare` unused"""
    from blazr_b200.batch import StepEntry, build_step
    need = [-(-(n + p) // bs) for n, p in entries]
    pages = sum(need) + spare
    perm = rng.permutation(pages).tolist()
    tables, at = [], 0
    for n in need:
        tables.append(perm[at:at + n])
        at += n
    sa = build_step([StepEntry([0] * n, p, i, tables[i]) for i, (n, p) in enumerate(entries)], bs)
    t = {k: torch.from_numpy(np.ascontiguousarray(getattr(sa, k))).to(DEV) for k in ("tok_ent", "tok_pos", "ent_start", "ent_slot", "ent_pos0", "block_table")}
    st = ops.StepDesc(*(t[k].data_ptr() for k in ("tok_ent", "tok_pos", "ent_start", "ent_slot", "ent_pos0", "block_table")), sa.T, sa.B, sa.block_table.shape[1], bs)
    slots = [[(tables[e][j // bs], j % bs) for j in range(n + p)] for e, (n, p) in enumerate(entries)]
    return st, t, slots, pages


# ---- rows into pages and back ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("D,V,bs", [(128, 128, 16), (64, 64, 16), (32, 32, 16), (80, 48, 32), (128, 64, 48), (1, 3, 16), (33, 31, 16), (97, 128, 5), (64, 20, 1), (128, 127, 7)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_are_stored_and_read_back(ops, D, V, bs, dtype):
    """every byte of a row's place, and no other byte of the pool; rows lie apart and start where nothing is aligned"""
    rng = np.random.default_rng(D * 131 + V + bs)
    G, Gv = 3, 2
    st, keep, slots, pages = step(ops, [(9, 0), (1, 13), (5, 2 * bs + 1)], bs, rng)
    x = lambda w: torch.from_numpy((rng.standard_normal((st.T, w + 5)) * np.exp(rng.standard_normal((st.T, 1)) * 2) + rng.standard_normal(w + 5) * 2).astype(np.float32)).to(dtype).to(DEV)
    k, v = x(G * D)[:, 1:1 + G * D], x(Gv * V)[:, 3:3 + Gv * V]
    before = [rng.integers(0, 256, (pages, h, ops.kv4_page_bytes(bs, 1, d)), dtype=np.uint8) for h, d in ((G, D), (Gv, V))]
    kp, vp = (torch.from_numpy(b).to(DEV) for b in before)
    ops.kv4_store(k, v, st, kp, vp)
    new = [s for (n, p), e in zip([(9, 0), (1, 13), (5, 2 * bs + 1)], slots) for s in e[p:]]
    for pool, want, rows, h, d, key in ((kp, before[0], k, G, D, True), (vp, before[1], v, Gv, V, False)):
        ref.put_rows(want, bs, new, rows.float().cpu().numpy().reshape(st.T, h, d), key)
        np.testing.assert_array_equal(pool.cpu().numpy(), want)
    ko, vo = torch.full((st.T, G * D + 3), 7.0, device=DEV), torch.full((st.T, Gv * V + 2), 7.0, device=DEV)
    ops.kv4_load(kp, vp, st, ko[:, 2:2 + G * D], vo[:, 1:1 + Gv * V])
    np.testing.assert_array_equal(ko[:, 2:2 + G * D].cpu().numpy(), ref.held(k.float().cpu().numpy().reshape(st.T, G, D)).reshape(st.T, -1))
    np.testing.assert_array_equal(vo[:, 1:1 + Gv * V].cpu().numpy(), ref.held(v.float().cpu().numpy().reshape(st.T, Gv, V)).reshape(st.T, -1))
    assert bool((ko[:, :2] == 7).all()) and bool((ko[:, -1] == 7).all()) and bool((vo[:, 0] == 7).all()) and ops.error_flags() == 0


def test_rows_of_every_size(ops):
    """ranges from none to the largest, far from zero and below the smallest f16"""
    rng = np.random.default_rng(3)
    rows = [np.full(32, 5.3), np.zeros(32), np.linspace(0, 15 * 0.25, 32), rng.uniform(-1e-6, 1e-6, 32), rng.uniform(-3e-8, 3e-8, 32), np.full(32, 1e-9), rng.uniform(-32000, 32000, 32),
            1000 + rng.uniform(0, 1e-2, 32), rng.uniform(2.0 ** -18, 2.0 ** -17, 32), np.r_[np.full(31, -31999.0), 31999.0], rng.uniform(-1e-40, 1e-40, 32)]
    x = np.stack(rows).astype(np.float32)
    st, keep, slots, pages = step(ops, [(len(x), 0)], 16, rng)
    kp, vp = ops.kv4_pool(pages, 16, 1, 32, DEV), ops.kv4_pool(pages, 16, 1, 32, DEV)
    d = torch.from_numpy(x).to(DEV)
    ops.kv4_store(d, -d, st, kp, vp)
    ko, vo = torch.empty_like(d), torch.empty_like(d)
    ops.kv4_load(kp, vp, st, ko, vo)
    np.testing.assert_array_equal(ko.cpu().numpy(), ref.held(x))
    np.testing.assert_array_equal(vo.cpu().numpy(), ref.held(-x))
    # a value is off by at most half a step of its group (a step: a fifteenth of the range and 2^-6 of that, at least 2^-24) and the minimum's rounding to f16
    span, low = x.max(1) - x.min(1), np.abs(x.min(1))
    bound = np.maximum(span / 15 * (1 + 2.0 ** -6), 2.0 ** -24) / 2 + low * 2.0 ** -11 * (1 + 1 / 15) + 2.0 ** -25
    assert (np.abs(ko.cpu().numpy().astype(np.float64) - x).max(1) <= bound * (1 + 1e-6)).all() and ops.error_flags() == 0


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), 32001.0, -1e30])
def test_what_the_cache_cannot_hold_is_flagged(ops, bad):
    """and the other groups of the row, and the other rows, are as ever"""
    rng = np.random.default_rng(5)
    st, keep, slots, pages = step(ops, [(4, 3)], 16, rng)
    x = rng.standard_normal((4, 2 * 64)).astype(np.float32)
    x[1, 70] = bad
    kp, vp = ops.kv4_pool(pages, 16, 2, 64, DEV), ops.kv4_pool(pages, 16, 2, 64, DEV)
    d = torch.from_numpy(x).to(DEV)
    ops.kv4_store(d, d, st, kp, vp)
    assert ops.error_flags() == 8
    ko, vo = torch.empty_like(d), torch.empty_like(d)
    ops.kv4_load(kp, vp, st, ko, vo)
    want = ref.held(x.reshape(4, 2, 64)).reshape(4, -1)
    assert np.isfinite(want).all() and ops.error_flags() == 0
    np.testing.assert_array_equal(ko.cpu().numpy(), want)
    np.testing.assert_array_equal(vo.cpu().numpy(), want)


def test_a_position_without_a_page_is_flagged(ops):
    rng = np.random.default_rng(6)
    st, keep, slots, pages = step(ops, [(3, 30)], 16, rng)
    st.max_blocks = 2                                          # positions 32 and 33 lie behind the table
    x = torch.randn(3, 32, device=DEV)
    kp, vp = ops.kv4_pool(pages, 16, 1, 32, DEV), ops.kv4_pool(pages, 16, 1, 32, DEV)
    ops.kv4_store(x[:, :32], x, st, kp, vp)
    assert ops.error_flags() == 1
    ko, vo = torch.full_like(x, 9.0), torch.full_like(x, 9.0)
    ops.kv4_load(kp, vp, st, ko, vo)
    assert ops.error_flags() == 1 and not bool((ko[:2] == 9).any()) and bool((ko[2] == 9).all()) and int((kp != 0).any(2).sum()) == 1
    d = ops.attn_desc(1, 1, 32, 32, 1.0, gated=False)
    out = torch.full((3, 32), 4.0, device=DEV)
    ops.attn_kv4(x, st, d, kp, vp, out)
    assert ops.error_flags() == 1


# ---- the prep step -------------------------------------------------------------------------------------------------------------------------
PREP = [
    dict(), dict(qk_eps=1e-5), dict(rot=64), dict(rot=32, rot_half=True), dict(qk_eps=1e-6, rot=64, rot_half=True, weights=True), dict(qk_eps=1e-6, weights=True, norm_full=True, rot=20),
    dict(in_bias=True, rot=64), dict(values_from_keys=True, qk_eps=1e-5, rot=64), dict(value_heads=1), dict(kv_shared=True, rot=64, qk_eps=1e-5, weights=True),
]


def prep_case(ops, o, H, G, D, V, bs, entries, spare):
    """rows that lie `spare` values further apart than they are long"""
    rng = np.random.default_rng(11)
    st, keep, slots, pages = step(ops, entries, bs, rng)
    t = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to(DEV)
    freq = torch.from_numpy((10000.0 ** (-np.arange(o["rot"] // 2) / 32)).astype(np.float32)).to(DEV) if "rot" in o else None
    full = o.get("norm_full", False)
    qw, kw = (t(H * D if full else D), t(G * D if full else D)) if o.get("weights") else (None, None)
    bias = t(8192) if o.get("in_bias") else None
    d = ops.attn_desc(H, G, D, V, 1.0, gated=False, qk_eps=o.get("qk_eps", -1.0), rot_freq=freq, rot_half=o.get("rot_half", False), rot_scale=1.1, q_norm_w=qw, k_norm_w=kw, norm_full=full,
                      in_bias=bias, values_from_keys=o.get("values_from_keys", False), value_heads=o.get("value_heads", 0), kv_shared=o.get("kv_shared", False))
    Gv = o.get("value_heads", 0) or G
    rows = t(st.T, d.width + spare)
    a, b = rows.clone(), rows.clone()
    kf, vf = torch.zeros(pages, bs, G, D, device=DEV), torch.zeros(pages, bs, Gv, V, device=DEV)
    k4, v4 = ops.kv4_pool(pages, bs, G, D, DEV), ops.kv4_pool(pages, bs, Gv, V, DEV)
    if o.get("values_from_keys") and (d.q_norm_w or d.rot_half):
        pytest.skip("no such layer")
    ops.attn_prep_ex(a, st, d, kf, vf)
    ops.attn_prep_kv4(b, st, d, k4, v4)
    assert (a - b).abs().max().item() <= 4e-6 * a.abs().max().item()
    if o.get("kv_shared"):
        assert not bool(k4.any()) and not bool(v4.any())
        return
    ko, vo = torch.empty(st.T, G * D, device=DEV), torch.empty(st.T, Gv * V, device=DEV)
    ops.kv4_load(k4, v4, st, ko, vo)
    new = [s for (n, p), e in zip(entries, slots) for s in e[p:]]
    for got, pool, h, w in ((ko, kf, G, D), (vo, vf, Gv, V)):
        x = np.stack([pool[pg, at].cpu().numpy() for pg, at in new])
        want, _, step_ = ref.held(x), *ref.quantise(x)[:2]
        off = np.abs(got.cpu().numpy().reshape(x.shape) - want)
        at = np.arange(w) // 32
        assert (off <= step_[..., at] * 1.05 + 1e-5).all() and (off > 1e-5).mean() < 0.01
    assert ops.error_flags() == 0


@pytest.mark.parametrize("o", PREP, ids=lambda o: "-".join(o) or "plain")
@pytest.mark.parametrize("D,bs", [(64, 16), (80, 16), (128, 5)])
def test_prep_is_that_of_the_f32_cache(ops, o, D, bs):
    """queries to f32 roundings, cached rows as what the f32 pool's rows become (a value that such a rounding moves over the middle between two codes may be a step off)"""
    prep_case(ops, o, 4, 2, D, D, bs, [(7, 0), (1, 40), (2, 15)], 3)


@pytest.mark.parametrize("o", PREP, ids=lambda o: "-".join(o) or "plain")
@pytest.mark.parametrize("H,G,D,V,bs,entries", [(4, 2, 64, 64, 16, [(7, 0), (1, 40), (2, 15)]), (5, 5, 80, 80, 16, [(1, 100)]), (6, 2, 128, 72, 5, [(3, 1), (1, 9)]),
                                                (8, 2, 64, 24, 16, [(600, 3), (700, 0)]), (32, 8, 128, 128, 16, [(1, 700)] * 33)])
def test_prep_of_rows_in_whole_pieces(ops, o, H, G, D, V, bs, entries):
    if o.get("values_from_keys") and D != V:
        pytest.skip("no such layer")
    prep_case(ops, o, H, G, D, V, bs, entries, 4)


def test_prep_of_small_heads_in_whole_pieces(ops):
    for o in (dict(), dict(qk_eps=1e-5, rot=16, rot_half=True, weights=True), dict(qk_eps=1e-5, rot=10)):
        prep_case(ops, o, 9, 3, 24, 8, 16, [(5, 0), (1, 31)], 0)
        prep_case(ops, o, 2, 1, 32, 128, 16, [(2, 14)], 8)


# ---- attention -------------------------------------------------------------------------------------------------------------------------------
def attend(ops, entries, H, G, D, V, o, odt, bs=16, plant=None, mean=0.0):
    """(results, float64 reference) over pools whose bytes outside the rows in use are random"""
    rng = np.random.default_rng(H * D + V + len(entries))
    st, keep, slots, pages = step(ops, entries, bs, rng)
    Gv = o.get("value_heads", 0) or G
    gated, elem = o.get("gated", False), o.get("gate_elem", False)
    f32 = lambda *s: rng.standard_normal(s).astype(np.float32)
    sink, hs = f32(H) if o.get("sink") else None, f32(H) if o.get("head_scale") else None
    dev = [torch.from_numpy(x).to(DEV) if x is not None else None for x in (sink, hs)]
    d = ops.attn_desc(H, G, D, V, o.get("scale", 2.0 * D ** -0.5), gated=gated, chunk=o.get("chunk", 0), window=o.get("window", 0), keep_first=o.get("keep_first", 0),
                      softcap=o.get("softcap", 0.0), sink=dev[0], head_scale=dev[1], gate_elem=elem, value_heads=o.get("value_heads", 0), kv_shared=True)
    rows = f32(st.T, d.width + o.get("pad", 0))
    pools = [rng.integers(0, 256, (pages, h, ops.kv4_page_bytes(bs, 1, w)), dtype=np.uint8) for h, w in ((G, D), (Gv, V))]
    for pool, h, w, key in ((pools[0], G, D, True), (pools[1], Gv, V, False)):
        centre = mean * f32(h, w) if key else 0.0
        for e in slots:
            ref.put_rows(pool, bs, e, f32(len(e), h, w) + centre, key)
    if plant is not None:
        plant(rows)
    want = np.zeros((st.T, H, V))
    r0 = 0
    for (n, past), e in zip(entries, slots):
        k, v = ref.get_rows(pools[0], bs, e, D, True), ref.get_rows(pools[1], bs, e, V, False)
        gl = None
        if gated:
            gl = rows[r0:r0 + n, d.gate_col:]
            gl = gl[:, :H * V].reshape(n, H, V) if elem else gl[:, :H]
        want[r0:r0 + n] = ref.attend(rows[r0:r0 + n, :H * D].reshape(n, H, D), k, v, np.arange(past, past + n), d.scale, d.chunk, d.window, d.keep_first, d.softcap, sink, hs, gl)
        r0 += n
    out = torch.full((st.T + 1, H * V), 3.0, device=DEV, dtype=odt)
    kp, vp = (torch.from_numpy(p).to(DEV) for p in pools)
    ops.attn_kv4(torch.from_numpy(rows).to(DEV), st, d, kp, vp, out[:st.T])
    assert bool((out[st.T] == 3.0).all()) and ops.error_flags() == 0
    np.testing.assert_array_equal(kp.cpu().numpy(), pools[0])
    return out[:st.T].double().cpu().numpy(), want.reshape(st.T, -1)


def close(out, want, odt):
    err = np.abs(out - want).max() / np.abs(want).max()
    assert err < (4e-6 if odt == torch.float32 else 2.0 ** -8), err


CASES = [
    # entries (tokens, past), H, G, D, V, options, block size
    ([(1, 0)], 1, 1, 32, 32, {}, 16),                                    # one key: the row is that value
    ([(1, 0), (1, 15), (1, 16), (1, 500)], 8, 2, 64, 64, {}, 16),        # the first key of a page, the last
    ([(1, 777)], 32, 8, 128, 128, {}, 16),
    ([(1, 300), (1, 2)], 6, 2, 128, 128, {}, 16),                        # three query heads to a key head
    ([(1, 300)], 16, 1, 64, 64, {}, 16),                                 # more query heads than a row tile has rows
    ([(1, 130)], 22, 2, 64, 64, dict(pad=2), 16),
    ([(5, 90), (3, 0), (1, 17)], 8, 4, 64, 64, {}, 16),                  # a few tokens each: their rows see different keys
    ([(17, 40)], 4, 4, 32, 128, {}, 16),
    ([(2, 40)], 4, 2, 128, 32, {}, 32),
    ([(3, 100)], 4, 2, 80, 48, dict(pad=1), 16),                         # sizes that are no whole groups, rows that are not aligned
    ([(3, 61)], 3, 1, 1, 3, {}, 16),
    ([(4, 50)], 4, 2, 33, 97, {}, 16),
    ([(1, 70), (6, 21)], 4, 2, 64, 64, {}, 5),                           # pages that end inside a tile
    ([(1, 70), (6, 21)], 4, 2, 128, 128, {}, 1),
    ([(2, 200)], 4, 2, 64, 64, {}, 48),
    ([(2, 200)], 4, 2, 128, 64, {}, 24),
    ([(1, 200), (4, 37), (3, 0)], 4, 2, 64, 64, dict(window=37), 16),
    ([(1, 200), (4, 37)], 4, 2, 64, 64, dict(window=1), 16),
    ([(1, 200), (4, 100), (1, 5)], 4, 2, 64, 64, dict(window=40, keep_first=3), 16),
    ([(1, 200), (4, 100), (1, 5)], 4, 2, 64, 64, dict(window=40, keep_first=50), 16),
    ([(1, 95), (1, 96), (4, 94)], 4, 2, 64, 64, dict(chunk=48), 16),
    ([(1, 200), (2, 30)], 4, 2, 64, 64, dict(softcap=3.0), 16),
    ([(1, 200), (2, 30)], 8, 2, 64, 64, dict(sink=True, head_scale=True), 16),
    ([(1, 200), (2, 30)], 8, 2, 64, 64, dict(gated=True, scale=-0.2), 16),
    ([(1, 200), (2, 30)], 8, 2, 64, 64, dict(gated=True, gate_elem=True, scale=0.0), 16),
    ([(1, 200), (2, 30)], 8, 4, 64, 128, dict(value_heads=2), 16),
    ([(1, 3000)], 8, 2, 128, 128, dict(scale=1.0), 16),                  # scores up to 40
    ([(40, 0), (20, 77)], 8, 2, 64, 64, {}, 16),                         # prompts
    ([(150, 0)], 4, 2, 128, 128, dict(window=33, sink=True), 16),
    ([(70, 300), (1, 5), (33, 0)], 16, 2, 64, 64, dict(gated=True, chunk=64), 16),
    ([(130, 10)], 6, 2, 80, 48, dict(softcap=5.0), 16),
    ([(100, 0)], 4, 1, 32, 64, {}, 5),
    ([(33, 1500)], 32, 8, 128, 128, {}, 16),
    # row tiles of 128 and of twice that on the tensor cores
    ([(600, 0)], 64, 8, 64, 64, dict(window=130), 16),
    ([(600, 5)], 64, 16, 32, 32, dict(chunk=128, sink=True), 32),
    ([(450, 30), (150, 0)], 64, 1, 64, 64, dict(softcap=4.0, gated=True), 16),
    ([(300, 0), (1, 70), (300, 17)], 64, 8, 40, 64, dict(window=64, keep_first=70, gated=True, gate_elem=True), 16),
    ([(200, 100)], 8, 2, 128, 104, dict(window=70, keep_first=5, head_scale=True), 24),
    ([(40, 700)], 8, 1, 32, 24, dict(scale=-0.3), 16),
    ([(65, 190)], 12, 2, 88, 127, dict(sink=True), 5),
    ([(40, 2000)], 8, 2, 64, 64, {}, 16),                                # keys dealt to several CTAs
    ([(40, 2000), (35, 10)], 4, 1, 128, 128, dict(sink=True, gated=True), 16),
    ([(20, 3000)], 96, 1, 64, 64, dict(softcap=6.0), 16),
    ([(17, 63), (17, 64), (17, 47)], 256, 2, 32, 32, {}, 16),
]


@pytest.mark.parametrize("entries,H,G,D,V,o,bs", CASES)
@pytest.mark.parametrize("odt", [torch.float32, torch.bfloat16])
def test_attention_against_float64(ops, entries, H, G, D, V, o, bs, odt):
    close(*attend(ops, entries, H, G, D, V, o, odt, bs), odt)


@pytest.mark.parametrize("B", [17, 64, 150])
def test_many_sequences(ops, B):
    close(*attend(ops, [(1, (37 * i) % 300) for i in range(B)], 8, 2, 64, 64, {}, torch.float32), torch.float32)


def test_keys_far_from_zero(ops):
    """minima that are ten times the spread of the values beside them: the score's large parts are common to all keys"""
    out, want = attend(ops, [(1, 400), (50, 30)], 8, 2, 64, 64, dict(scale=0.02), torch.float32, mean=10.0)
    assert np.abs(out - want).max() / np.abs(want).max() < 2e-5       # scores of up to 0.02 * 64 * 10 * 3 = 40, rounded to f32 in parts ten times as large: 400 * 2^-24


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e-4, 1e4, 1e12])
@pytest.mark.parametrize("tokens", [1, 60])
def test_queries_of_every_size(ops, size, tokens):
    """the f16 parts of a row are taken relative to its largest value"""
    out, want = attend(ops, [(tokens, 100)], 8, 2, 64, 64, dict(scale=0.25 / size), torch.float32, plant=lambda rows: rows[:, :512].__imul__(np.float32(size)))
    close(out, want, torch.float32)


@pytest.mark.parametrize("tokens", [2, 60])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_query_that_is_not_finite(ops, tokens, bad):
    """makes its own row NaN and no other"""
    out, want = attend(ops, [(tokens, 50)], 8, 2, 64, 64, dict(sink=True), torch.float32, plant=lambda rows: rows.__setitem__((1, 3 * 64 + 5), bad))
    out, want = out.reshape(tokens, 8, 64), want.reshape(tokens, 8, 64)
    assert np.isnan(out[1, 3]).all()
    out[1, 3] = want[1, 3] = 0
    close(out, want, torch.float32)


def test_tiny_values_keep_their_digits(ops):
    """steps below the smallest normal f16: what the cache holds is multiplied as it is"""
    rng = np.random.default_rng(8)
    st, keep, slots, pages = step(ops, [(1, 200)], 16, rng)
    x = [(rng.standard_normal((201, 1, 64)) * s).astype(np.float32) for s in (1.0, 1e-5)]
    pools = [np.zeros((pages, 1, 640), np.uint8) for _ in range(2)]
    for p, y, key in zip(pools, x, (True, False)):
        ref.put_rows(p, 16, slots[0], y, key)
    q = rng.standard_normal((1, 4 * 64)).astype(np.float32)
    want = ref.attend(q.reshape(1, 4, 64), ref.get_rows(pools[0], 16, slots[0], 64, True), ref.get_rows(pools[1], 16, slots[0], 64, False), [200], 0.125)
    out = torch.empty(1, 256, device=DEV)
    ops.attn_kv4(torch.from_numpy(q).to(DEV), st, ops.attn_desc(4, 1, 64, 64, 0.125, gated=False, kv_shared=True), *(torch.from_numpy(p).to(DEV) for p in pools), out)
    close(out.double().cpu().numpy(), want.reshape(1, -1), torch.float32)


def test_a_step_is_captured_and_replayed(ops):
    """store, attend and read back as one graph, replayed with other rows and other positions"""
    rng = np.random.default_rng(9)
    st, keep, slots, pages = step(ops, [(1, 60), (1, 33)], 16, rng)
    H, G, D = 8, 2, 64
    kp, vp = ops.kv4_pool(pages, 16, G, D, DEV), ops.kv4_pool(pages, 16, G, D, DEV)
    d = ops.attn_desc(H, G, D, D, 0.125, gated=False)
    rows, out = torch.randn(2, d.width, device=DEV), torch.empty(2, H * D, device=DEV)
    run = lambda: (ops.attn_prep_kv4(rows, st, d, kp, vp), ops.attn_kv4(rows, st, d, kp, vp, out))
    run()
    torch.cuda.synchronize()
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        run()
    for shift in (0, 1, 2):
        keep["tok_pos"].copy_(torch.tensor([60 - shift, 33 + shift], dtype=torch.int32))
        rows.copy_(torch.randn(2, d.width, device=DEV))
        g.replay()
        a = out.clone()
        run()
        assert torch.equal(a, out)
    assert ops.error_flags() == 0


def test_the_same_call_gives_the_same_bits(ops):
    for entries in ([(1, 5000)], [(1, 900)] * 40, [(300, 200)]):
        a = attend(ops, entries, 8, 2, 64, 64, {}, torch.float32)[0] if len(entries) > 1 else None
        rng = np.random.default_rng(1)
        st, keep, slots, pages = step(ops, entries, 16, rng)
        kp, vp = (torch.zeros((pages, 2, 640), dtype=torch.uint8, device=DEV) for _ in range(2))
        q = torch.randn(st.T, 8 * 64, device=DEV)
        d = ops.attn_desc(8, 2, 64, 64, 0.125, gated=False, kv_shared=True)
        T = 16 * pages
        i32 = dict(dtype=torch.int32, device=DEV)
        fill = [torch.zeros(T, **i32), torch.arange(T, **i32), torch.arange(pages, **i32)]
        all_ = ops.StepDesc(fill[0].data_ptr(), fill[1].data_ptr(), 0, 0, 0, fill[2].data_ptr(), T, 1, pages, 16)
        ops.kv4_store(torch.randn(T, 128, device=DEV), torch.randn(T, 128, device=DEV), all_, kp, vp)
        outs = [torch.empty(st.T, 512, device=DEV) for _ in range(3)]
        for o in outs:
            ops.attn_kv4(q, st, d, kp, vp, o)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2]) and (a is None or np.isfinite(a).all())


# ---- steps that hold more than tokens ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("entries,D", [([(2, 50), (1, 30), (1, 9)], 64), ([(1, 5000)], 128), ([(1, 40)] * 6, 64), ([(70, 3000)], 64), ([(70, 3000)], 128), ([(100, 0), (37, 900)], 64),
                                       ([(5, 700), (3, 0)], 128)])
@pytest.mark.parametrize("odt", [torch.float32, torch.bfloat16])
def test_entries_without_tokens_and_rows_behind_the_last(ops, entries, D, odt):
    """entries without tokens among the others, and rows behind the last entry's, change nothing of the others' results; the latter are left as they were, and so are those of
    positions without pages"""
    rng = np.random.default_rng(len(entries) + D)
    H, G = 8, 2
    st, keep, slots, pages = step(ops, entries, 16, rng)
    pools = [np.zeros((pages, G, ops.kv4_page_bytes(16, 1, D)), dtype=np.uint8) for _ in range(2)]
    for pool, key in zip(pools, (True, False)):
        for e in slots:
            ref.put_rows(pool, 16, e, rng.standard_normal((len(e), G, D)).astype(np.float32), key)
    kp, vp = (torch.from_numpy(p).to(DEV) for p in pools)
    d = ops.attn_desc(H, G, D, D, 0.125, gated=False, kv_shared=True)
    T, B = st.T, st.B
    q = torch.from_numpy(rng.standard_normal((T + 5, d.width)).astype(np.float32)).to(DEV)

    def run(tok_ent, tok_pos, ent_start, table, n, flags=0):
        dev = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (tok_ent, tok_pos, ent_start)] + [torch.tensor(table, dtype=torch.int32, device=DEV)]
        s = ops.StepDesc(dev[0].data_ptr(), dev[1].data_ptr(), dev[2].data_ptr(), dev[0].data_ptr(), dev[1].data_ptr(), dev[3].data_ptr(), n, len(ent_start) - 1, len(table[0]), 16)
        out = torch.full((T + 5, H * D), 3.0, device=DEV, dtype=odt)
        ops.attn_kv4(q, s, d, kp, vp, out)
        assert ops.error_flags() == flags
        return out

    ent, pos, start, table = (keep[k].cpu().tolist() for k in ("tok_ent", "tok_pos", "ent_start", "block_table"))
    plain = run(ent, pos, start, table, T)
    assert bool((plain[T:] == 3).all()) and not bool((plain[:T] == 3).all(1).any())
    same = lambda out: (out[:T].float() - plain[:T].float()).abs().max().item() <= (4e-6 if odt == torch.float32 else 2.0 ** -7) * plain[:T].float().abs().max().item()
    # entries without tokens: behind the first one, and at the end as many as make it as many entries as tokens (two where that is many)
    extra = max(T - B - 1, 0) if T <= 8 else 2
    at = [0] + [i + 2 for i in range(B - 1)]
    start2, table2 = [0, start[1]] + start[1:] + [T] * extra, [table[0], table[0]] + table[1:] + [table[0]] * extra
    out = run([at[e] for e in ent], pos, start2, table2, T)
    assert same(out) and bool((out[T:] == 3).all())
    # rows behind the last entry's
    out = run(ent + [0] * 5, pos + [0] * 5, start, table, T + 5)
    assert same(out) and bool((out[T:] == 3).all())
    if T <= 8:                                                 # (as many entries as rows)
        out = run(ent + [0] * 5, pos + [0] * 5, start + [T] * (T + 5 - B), table + [table[0]] * (T + 5 - B), T + 5)
        assert same(out) and bool((out[T:] == 3).all())
    # no page for the last positions of the longest
    w = len(table[0]) - 1
    out = run(ent, pos, start, [r[:w] for r in table], T, flags=1)
    assert bool((out[:T][torch.tensor([p >= 16 * w for p in pos], device=DEV)] == 3).all()) and bool((out[T:] == 3).all())


@pytest.mark.parametrize("entries,D,keys", [([(1, 5000)], 128, 5001), ([(1, 30)] * 3, 64, 31), ([(16, 0)], 64, 16), ([(70, 3000)], 64, 3070), ([(5, 700), (3, 0)], 128, 705),
                                            ([(300, 200)], 128, 500)])
def test_results_for_any_number_of_keys_named(ops, entries, D, keys):
    """the keys that a caller names share the work out and do no more: too few, as many as there are, too many"""
    rng = np.random.default_rng(D + keys)
    st, keep, slots, pages = step(ops, entries, 16, rng)
    kp, vp = ops.kv4_pool(pages, 16, 2, D, DEV), ops.kv4_pool(pages, 16, 2, D, DEV)
    fill, keep2, *_ = step(ops, [(16 * pages, 0)], 16, np.random.default_rng(0), spare=0)      # (every row of every page)
    ops.kv4_store(torch.randn(fill.T, 2 * D, device=DEV), torch.randn(fill.T, 2 * D, device=DEV), fill, kp, vp)
    d = ops.attn_desc(8, 2, D, D, 0.125, gated=False, kv_shared=True)
    q = torch.randn(st.T, d.width, device=DEV)
    outs = []
    for named in (0, keys, 1, 64, 1 << 20):
        out = torch.full((st.T, 8 * D), 3.0, device=DEV)
        ops.attn_kv4(q, st, d, kp, vp, out, max_keys=named)
        outs.append(out)
    for o in outs[1:]:
        assert (o - outs[0]).abs().max().item() <= 4e-6 * outs[0].abs().max().item()
    assert ops.error_flags() == 0


@pytest.mark.parametrize("bs", [16, 5])
@pytest.mark.parametrize("n", [1, 70])
def test_tables_with_negative_pages(ops, n, bs):
    """no page is written, nothing outside the pools is read, and the error flag says so"""
    st, keep, slots, pages = step(ops, [(n, 300)], bs, np.random.default_rng(n))
    keep["block_table"][:] = -1
    kp, vp = ops.kv4_pool(pages, bs, 2, 64, DEV), ops.kv4_pool(pages, bs, 2, 64, DEV)
    x = torch.randn(n, 128, device=DEV)
    ops.kv4_store(x, x, st, kp, vp)
    assert ops.error_flags() == 1
    out = torch.full((n, 128), 9.0, device=DEV)
    ops.kv4_load(kp, vp, st, out, out.clone())
    assert ops.error_flags() == 1 and bool((out == 9).all())
    d = ops.attn_desc(8, 2, 64, 64, 0.125, gated=False)
    rows = torch.randn(n, d.width, device=DEV)
    ops.attn_prep_kv4(rows, st, d, kp, vp)
    assert ops.error_flags() == 1 and not bool(kp.any()) and not bool(vp.any())
    ops.attn_kv4(rows, st, d, kp, vp, torch.empty(n, 512, device=DEV))
    assert ops.error_flags() == 1
