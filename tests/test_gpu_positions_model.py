"""Positions of requests whose cached rows have been cut back, through whole models: what a layer makes of tokens and positions alone, before any attention, is bit by bit what the same
steps make of it in a cache that keeps all rows."""
import pytest
import torch

from test_gpu_drafts_evict_model import DEV, engine, models, prompt  # noqa: F401

pytestmark = pytest.mark.gpu


def run(model, **kw):
    """portions, a step of two requests, single tokens (captured from the second on); returns the engine"""
    eng = engine(model, block_size=16, **kw)
    toks = prompt(150, 3)
    for i in range(0, 120, 40):
        eng.run_entries([{"id": "a", "tokens": toks[i:i + 40], "want": []}])
    eng.run_entries([{"id": "a", "tokens": toks[120:], "want": [29]}, {"id": "b", "tokens": toks[:11], "want": []}])
    for t in range(9):
        eng.run_entries([{"id": "a", "tokens": [t + 5], "want": [0]}, {"id": "b", "tokens": [t + 7], "want": [0]}])
    return eng


def rows(L, eng, rid, bits, first):
    """keys and values of the tokens from `first` on, as the pages hold them (4 bits: whole rows of a page's codes and parameters stand apart, so rows are read back as numbers)"""
    from blazr_b200 import seqops
    s = eng.cache.live[rid]
    n, lo = s.n_tokens - first, first - s.gone
    if bits == 32:
        return [torch.stack([p[s.blocks[(lo + i) // 16], (lo + i) % 16] for i in range(n)]).clone() for p in (L["kpool"], L["vpool"])]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    t = [i32([0] * n), i32(list(range(lo, lo + n))), i32([0, n]), i32([0]), i32([lo]), i32([s.blocks])]
    st = seqops.StepDesc(*[x.data_ptr() for x in t], n, 1, len(s.blocks), 16)
    out = [torch.empty(n, L["desc"].G * d, device=DEV) for d in (L["desc"].D, L["desc"].V)]
    seqops.kv4_load(L["kpool"], L["vpool"], st, *out)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("name", ["Gemosun", "Vodelix", "Zetunex"])
@pytest.mark.parametrize("bits", [32, 4])
def test_keys_of_later_tokens_stand_at_their_positions(models, name, bits):
    m = models(name)
    L = next(x for x in m.layers if "kpool" in x or x["spec"].kind in ("attention", "two_branch"))
    whole = run(m, kv_bits=bits)
    want = rows(L, whole, "a", bits, 143)
    eng = run(m, kv_bits=bits, max_keys=64, first_keys=2)
    s = eng.cache.live["a"]
    assert s.gone > 80 and s.whole_from <= 143 and s.n_tokens == 159
    got = rows(L, eng, "a", bits, 143)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(float(x.abs().sum()) > 0 for x in got)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_retention_turns_by_positions(models, layout):
    """linear attention with rotary positions in front of attention whose rows leave the cache"""
    from blazr_b200 import layered_bench as lb, registry
    from blazr_b200.layered import LayeredModel, RotarySpec
    cfg = lb.zetunex_config(dict(width=256, heads=8, kv_heads=2, dim=32, ff=512, chunk=48, vocab=1000), experts=8, top=2)
    two, lin = cfg["layers"][0], cfg["layers"][1]
    two["mixer"]["left"].pop("mask", None)
    cfg["layers"] = [lin, two, dict(two)]
    t = lb.random_tensors_zetunex(cfg, torch.device(DEV))
    parsed = registry.LAYERED["Zetunex"](cfg)
    assert parsed.layers[0].kind == "retention"
    parsed.layers[0].mixer.rot = RotarySpec(dims=16, base=10000.0, layout=layout)
    m = LayeredModel(parsed, t, DEV, "float32")
    state = lambda eng: [m.layers[0]["ret_state"][eng.cache.live[r].slot].clone() for r in "ab"]
    want = state(run(m))
    eng = run(m, max_keys=64, first_keys=2)
    assert eng.cache.live["a"].gone > 80
    assert all(torch.equal(a, b) for a, b in zip(state(eng), want)) and float(want[0].abs().sum()) > 0
