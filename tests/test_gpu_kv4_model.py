"""Layer-list models over a KV cache held in 4 bits, with forks, samples and sampling rules, through the engine.

Bound of logits that are reached in two ways (a prompt at once or in portions, prepared tokens or decoded ones): the hidden states differ by f32 roundings, about 1e-6
of their size; a value that such a rounding moves over the middle between two codes, one in about 1e5, is a step (a fifteenth of its group's range) off in the cache.  One
key among n that is off by a step in one of D values moves a score by at most a fifteenth of its size / sqrt(D), a result by that over n: far below 2e-2 of the
logits' largest."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def models():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from blazr_b200 import layered_bench as lb, registry, seqops
    from blazr_b200.layered import LayeredModel
    dev = torch.device(DEV)
    made = {}

    def get(name, dtype="float32"):
        if (name, dtype) not in made:
            if name == "Fenorax":
                cfg = lb.fenorax_config(dict(width=256, heads=8, kv_heads=2, dim=32, ff=512, ssm_heads=8, ssm_vdim=32, state=48, ssm_groups=2, chunk=40, vocab=1000), streams=3)
                t = lb.random_tensors(cfg, dev)
            elif name == "Pafelorn":
                cfg = lb.pafelorn_config(dict(width=256, heads=8, kv_heads=2, dim=32, ff=512, chunk=48, vocab=1000), experts=8, identity=2, top=2)
                t = lb.random_tensors_pafelorn(cfg, dev)
            elif name == "Vodelix":
                cfg = lb.vodelix_config(dict(width=256, heads=8, kv_heads=2, dim=32, ff=512, vocab=1000), experts=8, top=2)
                t = lb.random_tensors_vodelix(cfg, dev, rank=16)
            elif name == "Zetunex":
                cfg = lb.zetunex_config(dict(width=256, heads=8, kv_heads=2, dim=32, ff=512, chunk=48, vocab=1000), experts=8, top=2)
                t = lb.random_tensors_zetunex(cfg, dev)
            elif name == "Gemosun":
                cfg = lb.gemosun_config(dict(width=256, heads=8, kv_heads=2, dim=32, ff=512, chunk=48, vocab=1000), experts=8, top=2)
                t = lb.random_tensors_gemosun(cfg, dev)
            else:
                cfg = lb.teselix_config(dict(width=256, heads=8, dim=32, ff=512, vocab=1000), experts=8, top=2, kv_rank=64)
                t = lb.random_tensors_teselix(cfg, dev)
            made[(name, dtype)] = LayeredModel(registry.LAYERED[name](cfg), t, DEV, dtype)
        return made[(name, dtype)]
    seqops.error_flags()
    return get


PLAIN = ["Fenorax", "Pafelorn", "Vodelix", "Zetunex"]


def engine(model, kv_bits=4, **kw):
    from blazr_b200.engine import Engine
    return Engine(model, max_tokens=kw.pop("max_tokens", 1024), max_seqs=kw.pop("max_seqs", 4), kv_bits=kv_bits, **kw)


def prompt(n, seed=0):
    return [int(t) for t in np.random.default_rng(seed).integers(1, 1000, n)]


def near(a, b, bound=2e-2):
    assert np.isfinite(a).all() and np.abs(a - b).max() < bound * np.abs(b).max()


@pytest.mark.parametrize("name", PLAIN)
@pytest.mark.parametrize("bs", [16, 5])
def test_portions_and_single_tokens_reach_the_same_logits(models, name, bs):
    from blazr_b200 import seqops
    m, toks = models(name), prompt(150)
    eng = engine(m, block_size=bs)
    whole = eng.run_entries([{"id": "a", "tokens": toks, "want": [99, 149]}], ["a"])
    eng = engine(m, block_size=bs)
    eng.run_entries([{"id": "x", "tokens": prompt(20, 1), "want": []}, {"id": "a", "tokens": toks[:70], "want": []}])
    part = [eng.run_entries([{"id": "a", "tokens": toks[70:100], "want": [29]}])[0]]
    eng.run_entries([{"id": "a", "tokens": toks[100:146], "want": []}], ["x"])
    for t in toks[146:149]:
        eng.run_entries([{"id": "a", "tokens": [t], "want": []}])
    part.append(eng.run_entries([{"id": "a", "tokens": [toks[149]], "want": [0]}])[0])
    near(part[0], whole[0])
    near(part[1], whole[1])
    assert seqops.error_flags() == 0


@pytest.mark.parametrize("name", PLAIN)
def test_the_cache_is_small_and_the_logits_those_of_the_model(models, name):
    """beside the f32 cache: less than a fifth of its paged bytes, logits that move by the cache's steps (a fifteenth of a group's range each) and no more"""
    m, toks = models(name), prompt(120)
    out, size = {}, {}
    for bits in (32, 4):
        eng = engine(m, kv_bits=bits)
        out[bits] = eng.run_entries([{"id": "a", "tokens": toks, "want": [119]}])[0]
        size[bits] = sum(L[k].nbytes for L in m.layers for k in ("kpool", "vpool") if k in L)
    assert size[4] * 6 < size[32] * 1.01 and m.cache_bytes() > size[4]
    a, b = out[4].astype(np.float64), out[32].astype(np.float64)
    assert np.isfinite(a).all() and a @ b / np.linalg.norm(a) / np.linalg.norm(b) > 0.9 and not np.array_equal(a, b)


@pytest.mark.parametrize("name", PLAIN)
@pytest.mark.parametrize("bits", [4, 32])
def test_forks_continue_where_they_were(models, name, bits):
    """the pages that two requests share, the copies of those they write, and the copied state of their slots"""
    m, toks = models(name), prompt(61)
    eng = engine(m, kv_bits=bits)
    eng.run_entries([{"id": "a", "tokens": toks, "want": []}])
    eng.fork("a", "b")
    one = eng.run_entries([{"id": "a", "tokens": [7], "want": [0]}, {"id": "b", "tokens": [7], "want": [0]}])
    np.testing.assert_array_equal(one[0], one[1])
    eng.run_entries([{"id": "a", "tokens": [9, 4, 3], "want": []}, {"id": "b", "tokens": [5], "want": []}])
    assert eng.compact() >= 0
    eng.fork("b", "c")
    two = eng.run_entries([{"id": "a", "tokens": [8], "want": [0]}, {"id": "b", "tokens": [8], "want": [0]}, {"id": "c", "tokens": [8], "want": [0]}], ["a", "b", "c"])
    np.testing.assert_array_equal(two[1], two[2])
    ref = engine(m, kv_bits=bits)
    ref.run_entries([{"id": "a", "tokens": toks, "want": []}, {"id": "b", "tokens": toks, "want": []}])
    near(ref.run_entries([{"id": "a", "tokens": [7], "want": [0]}, {"id": "b", "tokens": [7], "want": [0]}]), one)
    ref.run_entries([{"id": "a", "tokens": [9, 4, 3], "want": []}, {"id": "b", "tokens": [5], "want": []}])
    near(ref.run_entries([{"id": "a", "tokens": [8], "want": [0]}, {"id": "b", "tokens": [8], "want": [0]}]), two[:2])
    assert eng.cache.pages.free_blocks == eng.cache.pages.num_blocks


def test_a_model_of_pooled_blocks_forks_too(models):
    m, toks = models("Gemosun"), prompt(77)
    eng = engine(m, kv_bits=32)
    assert eng.cache.pooled
    eng.run_entries([{"id": "a", "tokens": toks, "want": []}])
    eng.fork("a", "b")
    rng = np.random.default_rng(5)
    for _ in range(40):
        a, b = (int(t) for t in rng.integers(1, 1000, 2))
        out = eng.run_entries([{"id": "a", "tokens": [a], "want": [0]}, {"id": "b", "tokens": [b], "want": [0]}])
    ref = engine(m, kv_bits=32)
    ref.run_entries([{"id": "a", "tokens": toks, "want": []}, {"id": "b", "tokens": toks, "want": []}])
    rng = np.random.default_rng(5)
    for _ in range(40):
        a, b = (int(t) for t in rng.integers(1, 1000, 2))
        want = ref.run_entries([{"id": "a", "tokens": [a], "want": [0]}, {"id": "b", "tokens": [b], "want": [0]}])
    near(out, want, 1e-4)


@pytest.mark.parametrize("name", ["Gemosun", "Teselix"])
def test_models_that_it_does_not_hold(models, name):
    with pytest.raises(ValueError):
        engine(models(name))
    with pytest.raises(ValueError):
        engine(models("Fenorax"), kv_bits=8)
    engine(models(name), kv_bits=32)


@pytest.mark.parametrize("name", ["Pafelorn", "Zetunex"])
def test_captured_steps_give_the_same_tokens(models, name):
    from blazr_b200 import seqops
    from blazr_b200.engine import SamplingParams
    m = models(name, "bfloat16")
    outs = []
    for graphs in (True, False):
        m.use_graphs = graphs
        outs.append(engine(m).generate([prompt(40), prompt(7, 2)], SamplingParams(max_new_tokens=20)))
    m.use_graphs = True
    assert outs[0] == outs[1] and seqops.error_flags() == 0


def test_samples_penalties_and_masks(models):
    """a run of all of it: a 4-bit cache, a prompt sampled three times, penalties, a bias and a grammar of two tokens"""
    from blazr_b200 import seqops
    from blazr_b200.engine import SamplingParams
    m = models("Pafelorn", "bfloat16")
    words = np.zeros(32, np.uint32)
    words[3] = 1 << 5 | 1 << 9                                           # tokens 101 and 105
    outs = engine(m).generate([prompt(40)], SamplingParams(max_new_tokens=12, temperature=0.9, top_p=0.95, seed=3, n=3, mask_fn=lambda o: words if len(o) % 2 else None,
                                                           repetition_penalty=1.2, frequency_penalty=0.1))[0]
    assert len(outs) == 3 and all(len(o) == 12 and all(t in (101, 105) for t in o[1::2]) for o in outs) and len({tuple(o) for o in outs}) > 1
    eng = engine(m)
    plain = eng.generate([prompt(40)], SamplingParams(max_new_tokens=12))[0]
    same = eng.generate([prompt(40)], SamplingParams(max_new_tokens=12, logit_bias={5: -0.0}))[0]
    assert same == plain                                                 # (a bias of nothing goes the other way to the same tokens)
    pushed = eng.generate([prompt(40)], SamplingParams(max_new_tokens=12, logit_bias={5: 1e4}, frequency_penalty=3e3))[0]
    assert pushed[:4] == [5] * 4 and pushed[4:].count(5) == 0            # 1e4 - 3e3 n: four times
    assert seqops.error_flags() == 0


def test_captured_steps_of_growing_sequences(models):
    """a captured step is made for so many keys; sequences that outgrow them go through another one"""
    m, toks = models("Vodelix"), prompt(270)
    got = []
    for graphs in (True, False):
        m.use_graphs = graphs
        eng = engine(m, max_tokens=4096)
        eng.run_entries([{"id": "a", "tokens": toks[:250], "want": []}, {"id": "b", "tokens": toks[:40], "want": []}])
        got.append(np.stack([eng.run_entries([{"id": "a", "tokens": [t], "want": [0]}, {"id": "b", "tokens": [t], "want": [0]}]) for t in toks[250:]]))
        if graphs:
            assert {k[2] for k in m._graphs} == {256, 512}
    m.use_graphs = True
    near(got[0], got[1])
