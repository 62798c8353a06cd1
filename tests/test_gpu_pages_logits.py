"""Page copies (csrc/seq/seq_pages.cu) byte by byte, and the sampling rules on logits (csrc/seq/seq_logits.cu) against float64.

Logits: five f32 operations a value, each off by half a step (2^-24) of its result, on values of up to 40: 5 * 2^-24 * 40 = 1.2e-5; divisions by a temperature
below one scale what came before with the value itself.  Held to 1e-6 of the row's largest result + 1e-5."""
import numpy as np
import pytest
import torch

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


# ---- pages -----------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shapes,pages,n", [
    ([(16, 2, 64)], 9, 1), ([(16, 2, 64)], 9, 4), ([(4, 1, 3), (7,), (16, 8, 128), (1,)], 40, 17), ([(333,)] * 3, 300, 56), ([(333,)] * 3, 300, 57), ([(8, 5)] * 40, 64, 30),
    ([(24,)], 4000, 1999), ([(16, 8, 80)] * 2, 5, 2), ([(70000,)], 6, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.uint8, torch.bfloat16])
def test_pages_are_copied(ops, shapes, pages, n, dtype):
    """pools of any page size beside one another; more pools, pairs and bytes than one launch's table holds"""
    rng = np.random.default_rng(n)
    perm = rng.permutation(pages)
    pairs = [(int(perm[i % max(1, n // 2)]) if i % 3 == 0 else int(perm[i]), int(perm[n + i])) for i in range(n)]
    pools = [torch.from_numpy(rng.integers(0, 256, (pages, int(np.prod(s)) * torch.empty(0, dtype=dtype).element_size()), dtype=np.uint8)).to(DEV).view(dtype).reshape(pages, *s) for s in shapes]
    want = [p.clone() for p in pools]
    for w, p in zip(want, pools):
        for a, b in pairs:
            w[b] = p[a]
    ops.copy_pages(pools, pairs)
    for w, p in zip(want, pools):
        assert torch.equal(w.view(torch.uint8) if w.dtype != torch.uint8 else w, p.view(torch.uint8) if p.dtype != torch.uint8 else p)


def test_pools_that_start_anywhere(ops):
    """a pool that is a part of another tensor, at an odd byte"""
    base = torch.randint(0, 256, (1 + 10 * 48,), dtype=torch.uint8, device=DEV)
    pool = base[1:].view(10, 48)
    want = base.clone()
    want[1 + 3 * 48:1 + 4 * 48] = base[1 + 7 * 48:1 + 8 * 48]
    ops.copy_pages([pool], [(7, 3)])
    assert torch.equal(base, want)
    ops.copy_pages([pool], [])
    ops.copy_pages([], [])
    assert torch.equal(base, want)


def test_a_refused_copy_changes_nothing(ops):
    pool = torch.randn(6, 32, device=DEV)
    want = pool.clone()
    for pairs in ([(0, 1), (2, 1)], [(0, 1), (1, 2)], [(3, 3)], [(0, 6)], [(-1, 2)], [(0, 1), (2, 0)]):
        with pytest.raises(ops.SeqError):
            ops.copy_pages([pool], pairs)
    with pytest.raises(ValueError):
        ops.copy_pages([pool, torch.randn(7, 32, device=DEV)], [(0, 1)])
    with pytest.raises(ValueError):
        ops.copy_pages([pool.t()], [(0, 1)])
    assert torch.equal(pool, want)


def test_copies_follow_the_stream(ops):
    """captured beside what writes the pages, replayed twice"""
    pool = torch.zeros(8, 4096, device=DEV)
    src = torch.randn(4096, device=DEV)
    run = lambda: (pool[2].copy_(src), ops.copy_pages([pool], [(2, 5), (2, 7)]), pool[2].zero_())
    run()
    torch.cuda.synchronize()
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        run()
    for _ in range(2):
        src.copy_(torch.randn(4096, device=DEV))
        g.replay()
        assert torch.equal(pool[5], src) and torch.equal(pool[7], src) and not bool(pool[2].any())


# ---- sampling rules ------------------------------------------------------------------------------------------------------------------------
def make(rng, R, V, hist, bias, mask, prompt=None):
    f32 = lambda *s: rng.standard_normal(s).astype(np.float32)
    a = dict(logits=4 * f32(R, V), rules=np.stack([1 + rng.random(R), rng.random(R), rng.random(R), 0.5 + rng.random(R)], 1).astype(np.float32))
    lens = rng.integers(0, hist + 1, R)
    a["hist_start"] = np.r_[0, np.cumsum(lens)].astype(np.int32)
    a["hist"] = (rng.random(a["hist_start"][-1]) ** 3 * V).astype(np.int32)
    a["hist_prompt"] = (lens // 2 if prompt is None else np.minimum(lens, prompt)).astype(np.int32)
    if bias:
        n = rng.integers(0, bias + 1, R)
        a["bias_start"] = np.r_[0, np.cumsum(n)].astype(np.int32)
        a["bias_ids"] = rng.integers(0, V, a["bias_start"][-1]).astype(np.int32)        # some of them twice
        a["bias_vals"] = f32(a["bias_start"][-1])
    if mask:
        a["mask"] = rng.integers(0, 2 ** 32, (R, -(-V // 32)), dtype=np.uint32).view(np.int32)
    return a


def rules64(a):
    x = a["logits"].astype(np.float64)
    for r in range(x.shape[0]):
        rep, pres, freq, temp = a["rules"][r].astype(np.float64)
        h = a["hist"][a["hist_start"][r]:a["hist_start"][r + 1]]
        for t in set(h.tolist()):
            x[r, t] = x[r, t] / rep if x[r, t] > 0 else x[r, t] * rep
        for t, n in zip(*np.unique(h[a["hist_prompt"][r]:], return_counts=True)):
            x[r, t] -= n * freq + pres
        if "bias_ids" in a:
            at = slice(a["bias_start"][r], a["bias_start"][r + 1])
            for t, v in dict(zip(a["bias_ids"][at].tolist(), a["bias_vals"][at].tolist())).items():
                x[r, t] += v
        if temp != 0:
            x[r] /= temp
        if "mask" in a:
            v = np.arange(x.shape[1])
            x[r, (a["mask"][r].view(np.uint32)[v // 32] >> (v % 32).astype(np.uint32)) & 1 == 0] = -np.inf
    return x


def run(ops, a, out=None):
    d = {k: torch.from_numpy(np.ascontiguousarray(v)).to(DEV) for k, v in a.items()}
    return ops.process_logits(d.pop("logits"), d.pop("rules"), out, **d)


def same(got, want):
    got = got.double().cpu().numpy()
    fine = np.isfinite(want)
    assert (np.isfinite(got) == fine).all() and (got[~fine] == want[~fine]).all()
    if fine.any():
        assert np.abs(got[fine] - want[fine]).max() <= 1e-6 * np.abs(want[fine]).max() + 1e-5


@pytest.mark.parametrize("R,V,hist,bias,mask", [
    (1, 1, 3, 2, True), (1, 33, 10, 5, True), (3, 1000, 0, 0, False), (3, 1000, 200, 0, False), (2, 1024, 50, 40, True), (5, 1027, 3000, 30, True), (1, 32000, 500, 0, False),
    (64, 16385, 700, 100, True), (2, 128256, 20000, 300, True), (70, 4100, 64, 10, False)])
def test_rules_against_float64(ops, R, V, hist, bias, mask):
    a = make(np.random.default_rng(R * V), R, V, hist, bias, mask)
    same(run(ops, a), rules64(a))
    assert ops.error_flags() == 0


def test_rows_that_are_apart_and_results_elsewhere(ops):
    """row strides, rows that start off any boundary, results beside the logits"""
    a = make(np.random.default_rng(1), 3, 501, 60, 9, True)
    x = torch.zeros(3, 600, device=DEV)
    x[:, 3:504] = torch.from_numpy(a["logits"]).to(DEV)
    out = torch.full((3, 520), 5.0, device=DEV)
    d = {k: torch.from_numpy(np.ascontiguousarray(v)).to(DEV) for k, v in a.items()}
    m = torch.zeros(3, 40, dtype=torch.int32, device=DEV)
    m[:, 2:18] = d.pop("mask")
    d.pop("logits")
    ops.process_logits(x[:, 3:504], d.pop("rules"), out[:, 1:502], mask=m[:, 2:18], **d)
    same(out[:, 1:502], rules64(a))
    assert bool((out[:, 0] == 5).all()) and bool((out[:, 502:] == 5).all()) and torch.equal(x[:, 3:504].cpu(), torch.from_numpy(a["logits"]))


def test_prompt_tokens_are_only_repetitions(ops):
    rng = np.random.default_rng(2)
    for prompt in (0, 10 ** 6):
        a = make(rng, 4, 200, 150, 0, False, prompt=prompt)
        same(run(ops, a), rules64(a))


def test_logits_that_are_not_finite(ops):
    """infinities stay, masked ones of any kind are -inf; a row whose mask leaves nothing is -inf throughout"""
    a = make(np.random.default_rng(3), 3, 300, 50, 0, True)
    a["logits"][0, :6] = [np.inf, -np.inf, np.nan, np.finfo(np.float32).max, -np.finfo(np.float32).max, 0]
    a["rules"][0] = [1, 0, 0, 1]
    a["mask"][0] = -1
    a["mask"][1] = 0
    a["logits"][1, 5] = np.nan
    a["logits"][2, 7] = np.nan
    a["mask"][2] &= ~np.int32(1 << 7)
    got = run(ops, a).cpu().numpy()
    np.testing.assert_array_equal(got[0, :6], a["logits"][0, :6])
    assert np.isneginf(got[1]).all() and np.isneginf(got[2, 7])


def test_temperature_zero_and_no_rules(ops):
    """rules of (1, 0, 0, 0) leave the logits, bit by bit, whatever the history"""
    a = make(np.random.default_rng(4), 2, 700, 90, 0, False)
    a["rules"][:] = [1, 0, 0, 0]
    a["logits"][0, :3] = 3e38, -3e38, 1e-44
    assert np.array_equal(run(ops, a).cpu().numpy(), a["logits"])
    for k in ("hist", "hist_start", "hist_prompt"):
        a.pop(k)
    assert np.array_equal(run(ops, a).cpu().numpy(), a["logits"])


@pytest.mark.parametrize("where", ["hist", "bias_ids"])
@pytest.mark.parametrize("bad", [-1, 300, 2 ** 31 - 1])
def test_a_token_outside_the_vocabulary_is_flagged(ops, where, bad):
    """and passed over"""
    a = make(np.random.default_rng(5), 2, 300, 40, 20, False)
    a[where] = a[where].copy()
    a[where][1] = bad
    got = run(ops, a)
    assert ops.error_flags() == 16 and torch.isfinite(got).all()


def test_empty_histories(ops):
    a = make(np.random.default_rng(6), 3, 100, 0, 0, False)
    assert a["hist"].size == 0
    same(run(ops, a), rules64(a))


@pytest.mark.parametrize("V", [100, 128256])
def test_temperatures_whose_reciprocal_is_no_number(ops, V):
    a = make(np.random.default_rng(7), 64, V, 20, 0, False)
    a["logits"][:, ::2] = 0
    a["hist_prompt"][:] = np.diff(a["hist_start"])            # (repetitions leave zeros zero)
    a["rules"][::2, 3] = 2.0 ** -140
    want = rules64(a).astype(np.float32)                       # (infinities: beyond f32)
    got = run(ops, a).cpu().numpy()
    assert np.array_equal(np.isinf(want), np.isinf(got)) and np.array_equal(got[::2, ::2], np.zeros_like(got[::2, ::2])) and np.array_equal(np.sign(want), np.sign(got))


@pytest.mark.parametrize("what,starts", [("hist_start", [0, 5, 99999]), ("hist_start", [-3, 5, 9]), ("hist_start", [0, 9, 5]), ("bias_start", [0, 5, 99999]), ("bias_start", [7, 5, 9])])
@pytest.mark.parametrize("V", [300, 128256])
def test_rows_whose_lists_are_none(ops, what, starts, V):
    """starts that are not in order within their ids raise the flag, and the row goes without; nothing behind the ids is read"""
    a = make(np.random.default_rng(8), 2, V, 0, 0, False)
    a.update(hist=np.arange(9, dtype=np.int32), hist_start=np.array([0, 5, 9], np.int32), hist_prompt=np.zeros(2, np.int32), bias_ids=np.arange(9, dtype=np.int32),
             bias_start=np.array([0, 5, 9], np.int32), bias_vals=np.ones(9, np.float32))
    got = {True: dict(a), False: dict(a)}
    got[True][what] = np.array(starts, np.int32)
    bad = [starts[0] < 0 or starts[0] > starts[1], starts[1] > starts[2] or starts[2] > 9]
    out = run(ops, got[True]).cpu().numpy()
    assert ops.error_flags() == 16
    plain = rules64({k: a[k] for k in ("logits", "rules")} | dict(hist=np.zeros(0, np.int32), hist_start=np.zeros(3, np.int32), hist_prompt=np.zeros(2, np.int32)))
    full = rules64(got[False])
    for r in range(2):
        if bad[r]:
            same(torch.from_numpy(out[r]), plain[r])
        elif starts[r:r + 2] == [0, 5, 9][r:r + 2]:
            same(torch.from_numpy(out[r]), full[r])
