"""Drafts and a cache of bounded size through the engine, and positions that are not cached rows in the preparation of queries and keys.

A token's weights over the keys of one head add up to one (with a sink: to less): the weights that a slot has gathered add up to tokens times query heads of the key head,
each sum within its roundings, (keys + tokens) 2^-23 of itself."""
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
            sz = dict(width=256, heads=8, kv_heads=2, dim=32, ff=512, chunk=48, vocab=1000)
            if name == "Vodelix":
                cfg = lb.vodelix_config(sz, experts=8, top=2)
                t = lb.random_tensors_vodelix(cfg, dev, rank=16)
            elif name == "Zetunex":
                cfg = lb.zetunex_config(sz, experts=8, top=2)
                for lay in cfg["layers"]:
                    if "left" in lay["mixer"]:
                        lay["mixer"]["left"].pop("mask", None)
                t = lb.random_tensors_zetunex(cfg, dev)
            else:
                cfg = lb.gemosun_config(sz, experts=8, top=2)
                if name == "Gemosun":       # every position is seen; "windowed": as the benchmark has it
                    for lay in cfg["layers"]:
                        lay["mixer"].pop("mask", None)
                t = lb.random_tensors_gemosun(cfg, dev)
            made[(name, dtype)] = LayeredModel(registry.LAYERED["Gemosun" if name == "windowed" else name](cfg), t, DEV, dtype)
        return made[(name, dtype)]
    seqops.error_flags()
    return get


def engine(model, **kw):
    from blazr_b200.engine import Engine
    return Engine(model, max_tokens=kw.pop("max_tokens", 1024), max_seqs=kw.pop("max_seqs", 4), **kw)


def prompt(n, seed=0):
    return [int(t) for t in np.random.default_rng(seed).integers(1, 1000, n)]


def known(prompts, outs, n, wrong_every=0):
    """a draft_fn that guesses what is known to come (every wrong_every-th guess is another token)"""
    def f(tokens):
        for p, o in zip(prompts, outs):
            whole = p + o
            if tokens == whole[:len(tokens)]:
                return [(t + 1) % 1000 if wrong_every and (i + 1) % wrong_every == 0 else t for i, t in enumerate(whole[len(tokens):len(tokens) + n])]
        return []
    return f


@pytest.mark.parametrize("name", ["Gemosun", "windowed"])
@pytest.mark.parametrize("bits", [32, 4])
def test_greedy_tokens_do_not_change(models, name, bits):
    from blazr_b200 import seqops
    from blazr_b200.engine import SamplingParams
    if name == "windowed" and bits == 4:
        pytest.skip("pooled blocks are held in 32 bits")
    m = models(name)
    prompts = [prompt(90), prompt(33, 1), prompt(61, 2)]
    plain = engine(m, kv_bits=bits)
    want = plain.generate(prompts, SamplingParams(max_new_tokens=30))
    for n, wrong in ((5, 0), (5, 2), (3, 1)):
        eng = engine(m, kv_bits=bits)
        assert eng.generate(prompts, SamplingParams(max_new_tokens=30, draft_fn=known(prompts, want, n, wrong))) == want
        assert eng.steps < plain.steps if wrong != 1 else eng.steps >= plain.steps
        assert eng.cache.pages.free_blocks == eng.cache.pages.num_blocks
    assert seqops.error_flags() == 0


def test_sampled_tokens_with_drafts(models):
    """the distribution of a sampled token stays what the logits say: greedy requests beside sampled ones, drafts with probabilities, top_k and top_p"""
    from blazr_b200.engine import SamplingParams
    m = models("Gemosun")
    gen = torch.Generator(device=DEV)
    gen.manual_seed(5)

    def fn(tokens):
        p = torch.softmax(torch.randn(2, 1000, device=DEV, generator=gen), 1)
        return torch.multinomial(p, 1, generator=gen)[:, 0].tolist(), p
    eng = engine(m)
    rs = [eng.add_request(f"r{i}", prompt(20, i), SamplingParams(max_new_tokens=12, temperature=t, top_k=k, top_p=p, seed=i, draft_fn=f))
          for i, (t, k, p, f) in enumerate([(0.8, 0, 1.0, fn), (1.0, 1, 1.0, fn), (1.0, 0, 1e-6, lambda x: [5, 6]), (0.0, 0, 1.0, fn)])]
    while eng.has_work():
        eng.step()
    assert all(len(r.output) == 12 for r in rs)
    for r in rs[1:]:        # one token is left of what these may choose from
        first = engine(m).generate([r.prompt], SamplingParams(max_new_tokens=12))[0]
        assert r.output[1:] == engine(m).generate([r.prompt + r.output[:1]], SamplingParams(max_new_tokens=11))[0], (r.rid, first)


@pytest.mark.parametrize("name,dtype", [("Gemosun", "float32"), ("Gemosun", "bfloat16"), ("Vodelix", "float32"), ("Zetunex", "bfloat16")])
@pytest.mark.parametrize("bits", [32, 4])
def test_weights_are_gathered_as_steps_run(models, name, dtype, bits):
    """prompts in portions, mixed steps, captured single tokens: every token gives every key head a weight of one for each of its query heads"""
    from blazr_b200 import seqops
    m = models(name, dtype)
    eng = engine(m, kv_bits=bits, max_keys=400, max_step_tokens=200)
    toks = prompt(180)
    eng.run_entries([{"id": "a", "tokens": toks[:100], "want": []}])
    eng.run_entries([{"id": "a", "tokens": toks[100:], "want": []}, {"id": "b", "tokens": toks[:7], "want": []}])
    for t in range(5):
        eng.run_entries([{"id": "a", "tokens": [t + 1], "want": [0]}, {"id": "b", "tokens": [t + 1], "want": [0]}])
    a, b = eng.cache.live["a"], eng.cache.live["b"]
    for L in m.layers:
        if "key_weight" not in L:
            continue
        R = L["desc"].H // L["desc"].G
        for s, n, runs in ((a, 185, 1), (b, 12, 1)):
            got = L["key_weight"][s.slot, :, :n].double().sum(1).cpu().numpy()
            # (the last layer of a step that wants nothing runs its attention too; a sink takes its share)
            if L["desc"].sink:
                assert (got < n * R).all() and (got > 0).all()
            else:
                np.testing.assert_allclose(got, n * R, rtol=2 * (n + 200) * 2.0 ** -23)
    assert seqops.error_flags() == 0


@pytest.mark.parametrize("bits", [32, 4])
def test_requests_beyond_the_bound_go_on(models, bits):
    """rows leave while requests decode, fork and bring drafts; positions go on"""
    from blazr_b200 import seqops
    from blazr_b200.engine import SamplingParams
    m = models("Gemosun")
    eng = engine(m, kv_bits=bits, max_tokens=400, max_keys=64, first_keys=2, prefill_chunk=40)
    rs = [eng.add_request(f"r{i}", prompt(110 + i, i), SamplingParams(max_new_tokens=60, n=1 + (i == 1), draft_fn=(lambda x: x[-3:]) if i == 2 else None)) for i in range(3)]
    while eng.has_work():
        eng.step()
        assert all(s.rows <= 64 and s.n_tokens == s.rows + s.gone for s in eng.cache.live.values())
    assert all(len(q.output) == 60 for r in rs for q in [r] + r.siblings) and rs[1].output == rs[1].siblings[0].output
    assert eng.cache.pages.free_blocks == eng.cache.pages.num_blocks and seqops.error_flags() == 0


def test_what_leaves_is_what_was_attended_least(models):
    """the rows that stay are those of largest weight, in every layer and head; the next logits stay near those of the whole cache"""
    m = models("Gemosun")
    toks = prompt(128)
    eng = engine(m, max_keys=10 ** 4)
    whole = eng.run_entries([{"id": "a", "tokens": toks, "want": []}, ])
    weights = [L["key_weight"][eng.cache.live["a"].slot, :, :128].cpu().numpy() for L in m.layers]
    keys = [L["kpool"].clone() for L in m.layers]
    pages = list(eng.cache.live["a"].blocks)
    want = eng.run_entries([{"id": "a", "tokens": [9], "want": [0]}])[0]
    eng = engine(m, max_keys=126, first_keys=4, recent_keys=20)      # 111 stay
    eng.run_entries([{"id": "a", "tokens": toks, "want": []}])
    s = eng.cache.live["a"]
    assert s.rows == 111 and s.gone == 17 and whole is None
    import between_oracle as oracle
    for L, w, k in zip(m.layers, weights, keys):
        row = lambda pool, blocks, j, g: pool[blocks[j // 16], j % 16, g]
        for g in range(L["desc"].G):
            stay = oracle.stays(w[g], 128, 111, 4, 20)
            assert all(torch.equal(row(L["kpool"], s.blocks, i, g), row(k, pages, j, g)) for i, j in enumerate(stay))
            np.testing.assert_array_equal(L["key_weight"][s.slot, g, :111].cpu().numpy(), w[g][stay])
    got = eng.run_entries([{"id": "a", "tokens": [9], "want": [0]}])[0]
    a, b = got.astype(np.float64), want.astype(np.float64)
    assert a @ b / np.linalg.norm(a) / np.linalg.norm(b) > 0.9 and not np.array_equal(got, want)


def test_models_whose_rows_stay(models):
    with pytest.raises(ValueError):
        engine(models("windowed"), max_keys=64)
    from blazr_b200.engine import SamplingParams
    with pytest.raises(ValueError):
        engine(models("Vodelix")).add_request("a", [1, 2], SamplingParams(draft_fn=lambda t: [1]))
    engine(models("Gemosun")).run_entries([{"id": "a", "tokens": [1, 2, 3], "want": [2]}])       # (nothing is gathered)
    assert not any("key_weight" in L for L in models("Gemosun").layers)


@pytest.mark.parametrize("kw", [dict(), dict(rot_half=True), dict(norms=True), dict(rot_half=True, norms=True, D=80), dict(D=20), dict(D=48, rot_half=True)], ids=str)
@pytest.mark.parametrize("bits", [32, 4])
def test_queries_and_keys_turn_by_their_own_positions(models, kw, bits):
    """rows at places of their own, angles of another position: the same rows as a step whose positions are those"""
    from blazr_b200 import seqops as ops
    H, G, D, n, shift = 4, 2, kw.get("D", 64), 9, 37
    g = torch.Generator(device=DEV)
    g.manual_seed(D)
    freq = torch.rand(D // 4, device=DEV, generator=g)
    norms = dict(q_norm_w=torch.rand(D, device=DEV, generator=g), k_norm_w=torch.rand(D, device=DEV, generator=g), qk_eps=1e-5) if kw.get("norms") else {}
    d = ops.attn_desc(H, G, D, D, 1.0, gated=False, rot_freq=freq, rot_half=bool(kw.get("rot_half")), **norms)
    proj = torch.randn(n, d.width, device=DEV, generator=g)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    bt = i32([[3, 1, 4, 0, 2]])

    def step(p0):
        t = [i32([0] * n), i32(list(range(p0, p0 + n))), i32([0, n]), i32([0]), i32([p0])]
        return t, ops.StepDesc(t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr(), t[3].data_ptr(), t[4].data_ptr(), bt.data_ptr(), n, 1, 5, 16)
    out = []
    for p0, rot in ((5, i32(list(range(5 + shift, 5 + shift + n)))), (5 + shift, None)):
        t, st = step(p0)
        q = proj.clone()
        if bits == 32:
            pools = [torch.zeros(5, 16, G, D, device=DEV) for _ in range(2)]
            ops.attn_prep_ex(q, st, d, *pools, rot_pos=rot)
            rows = [torch.stack([p[bt[0, (p0 + i) // 16].item(), (p0 + i) % 16] for i in range(n)]) for p in pools]
        else:
            pools = [ops.kv4_pool(5, 16, G, D, DEV) for _ in range(2)]
            ops.attn_prep_kv4(q, st, d, *pools, rot_pos=rot)
            rows = [torch.empty(n, G * D, device=DEV) for _ in range(2)]
            ops.kv4_load(*pools, st, *rows)
        out.append([q[:, :H * D].clone()] + rows)
    for a, b in zip(*out):
        assert torch.equal(a, b)
    assert not torch.equal(out[0][0], proj[:, :H * D])
    with pytest.raises(ValueError):
        ops.attn_prep_ex(proj, step(5)[1], d, torch.zeros(5, 16, G, D, device=DEV), torch.zeros(5, 16, G, D, device=DEV), rot_pos=i32([1] * (n - 1)))
