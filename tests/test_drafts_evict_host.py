"""Drafts and a cache of bounded size in the serving engine, without a GPU: bookkeeping over stand-in models, the kernels' definitions in numpy."""
import numpy as np
import pytest
import torch

import between_oracle as oracle
from blazr_b200 import engine as engine_module
from blazr_b200.batch import StepEntry, build_step
from blazr_b200.cache import CacheFull, CacheManager
from blazr_b200.engine import Engine, SamplingParams, lookup_drafts
from test_fork_host import VOCAB, PagedModel

PROMPT = [3, 1, 4, 1, 5, 9, 2, 6]


class RowModel(PagedModel):
    """a model without state whose next token is a function of the rows it has cached; its rows may be evicted: those of odd tokens first"""

    def __init__(self, spread=False):
        super().__init__(state=False)
        self.weighed, self.spread, self.positions, self.cut = 0, spread, [], []

    def allocate(self, num_blocks, block_size, max_seqs, max_seq_tokens, weighed_rows=0):
        super().allocate(num_blocks, block_size, max_seqs, max_seq_tokens)
        self.weighed = weighed_rows

    def forward(self, sa, sample=False):
        nxt = []
        for e in range(sa.B):
            bt, p0 = sa.block_table[e], int(sa.ent_pos0[e])
            for i, t in enumerate(sa.tok_ids[sa.ent_start[e]:sa.ent_start[e + 1]]):
                row = int(sa.ent_start[e]) + i
                assert sa.tok_pos[row] == p0 + i
                self.pages[bt[(p0 + i) // self.bs], (p0 + i) % self.bs] = t
                self.positions.append(int(sa.tok_pos[row] if sa.tok_abs is None else sa.tok_abs[row]))
                if row in sa.want_rows:
                    seq = [int(self.pages[bt[j // self.bs], j % self.bs]) for j in range(p0 + i + 1)]
                    assert min(seq) >= 0
                    nxt.append((sum((j + 1) * x for j, x in enumerate(seq[-5:])) + 1) % VOCAB)
        self.last_ids = torch.tensor(nxt, dtype=torch.int32)
        hot = torch.nn.functional.one_hot(torch.tensor(nxt, dtype=torch.long), VOCAB).float() * 4.0
        return hot if self.spread else hot * 25.0

    def evict(self, slots, rows, tables, to_tables, keep, first, recent):
        assert len({s for s in slots}) == len(slots)
        for n, src, dst in zip(rows, tables, to_tables):
            assert len(dst) == -(-keep // self.bs) and n > keep
            have = [self.pages[src[j // self.bs], j % self.bs] for j in range(n)]
            stay = oracle.stays(np.array([1.0 - x % 2 for x in have]), n, keep, first, recent)
            for i, j in enumerate(stay):
                self.pages[dst[i // self.bs], i % self.bs] = have[j]
            self.cut.append((n, keep))


@pytest.fixture
def verified(monkeypatch):
    """verify_drafts by its definition; the calls' sizes"""
    calls = []

    def fake(logits, start, drafts, accept_u, sample_u, temperature, top_k=None, top_p=None, draft_probs=None):
        n = lambda t: None if t is None else t.numpy()
        calls.append((start.tolist(), draft_probs is not None))
        a, t, _ = oracle.verify(logits.numpy(), n(start), n(drafts), n(accept_u), n(sample_u), n(temperature), n(top_k), n(top_p), n(draft_probs))
        return torch.tensor(a, dtype=torch.int32), torch.tensor(t, dtype=torch.int32)
    monkeypatch.setattr(engine_module.seqops, "verify_drafts", fake)
    monkeypatch.setattr(engine_module.seqops, "error_flags", lambda: 0)
    return calls


@pytest.fixture(autouse=True)
def host_argmax(monkeypatch):
    monkeypatch.setattr(engine_module.seqops, "argmax", lambda z, ids: ids.copy_(z.argmax(1)))
    monkeypatch.setattr(engine_module.seqops, "error_flags", lambda: 0)


def alone(prompt, n, **kw):
    return Engine(RowModel(), max_tokens=400, max_seqs=1, block_size=4, **kw).generate([prompt], SamplingParams(max_new_tokens=n))[0]


# ---- drafts -------------------------------------------------------------------------------------------------------------------------------
def oracle_drafts(n, wrong_every=0):
    """guesses that are right (but every wrong_every-th)"""
    def f(tokens):
        out = []
        for i in range(n):
            seq = (tokens + out)[-5:]
            t = (sum((j + 1) * x for j, x in enumerate(seq)) + 1) % VOCAB
            out.append((t + 1) % VOCAB if wrong_every and (i + 1) % wrong_every == 0 else t)
        return out
    return f


@pytest.mark.parametrize("fn,steps", [(oracle_drafts(4), 5), (oracle_drafts(4, 3), 8), (oracle_drafts(4, 1), 21), (lambda t: [], 21), (lookup_drafts(3), None)])
@pytest.mark.parametrize("bs", [1, 4, 16])
def test_drafts_change_the_steps_not_the_tokens(verified, fn, steps, bs):
    eng = Engine(RowModel(), max_tokens=200, max_seqs=2, block_size=bs)
    r = eng.add_request("a", PROMPT, SamplingParams(max_new_tokens=21, draft_fn=fn))
    while eng.has_work():
        eng.step()
        if "a" in eng.cache.live:
            s = eng.cache.live["a"]
            assert s.n_tokens == len(PROMPT) + len(r.output) - 1 and len(s.blocks) == -(-s.n_tokens // bs) and s.last_token == (PROMPT + r.output)[-2]
    assert r.output == alone(PROMPT, 21)
    if steps is not None:
        assert eng.steps == steps
    assert eng.cache.pages.free_blocks == eng.cache.pages.num_blocks


def test_drafts_beside_other_requests(verified):
    """requests with drafts, without, sampled ones and prompts in one step; each gets what it gets alone"""
    eng = Engine(RowModel(), max_tokens=600, max_seqs=8, block_size=4, prefill_chunk=3)
    fn = oracle_drafts(3, 2)
    rs = [eng.add_request("a", PROMPT, SamplingParams(max_new_tokens=15, draft_fn=fn)), eng.add_request("b", PROMPT[:3], SamplingParams(max_new_tokens=9)),
          eng.add_request("c", PROMPT[2:], SamplingParams(max_new_tokens=12, draft_fn=fn, n=2)), eng.add_request("d", PROMPT * 3, SamplingParams(max_new_tokens=5, temperature=0.5)),
          eng.add_request("e", PROMPT[::-1], SamplingParams(max_new_tokens=7, draft_fn=fn, temperature=0.7, top_k=5, top_p=0.9, seed=3))]
    while eng.has_work():
        eng.step()
    for r, p, n in ((rs[0], PROMPT, 15), (rs[1], PROMPT[:3], 9), (rs[2], PROMPT[2:], 12), (rs[2].siblings[0], PROMPT[2:], 12), (rs[3], PROMPT * 3, 5), (rs[4], PROMPT[::-1], 7)):
        assert r.output == alone(p, n), r.rid
    assert eng.cache.pages.free_blocks == eng.cache.pages.num_blocks and eng.cache.slots.free_slots == 8


def test_drafts_with_probabilities(verified):
    """guesses drawn from a distribution, beside certain ones; a model that spreads its weight, so that some are rejected"""
    rng = np.random.default_rng(0)

    def fn(tokens):
        p = rng.random((3, VOCAB)).astype(np.float32)
        p /= p.sum(1, keepdims=True)
        return [int(rng.choice(VOCAB, p=x / x.sum())) for x in p.astype(np.float64)], torch.from_numpy(p)
    eng = Engine(RowModel(spread=True), max_tokens=400, max_seqs=3, block_size=4)
    rs = [eng.add_request(i, PROMPT, SamplingParams(max_new_tokens=20, temperature=1.0, seed=i, draft_fn=f)) for i, f in enumerate((fn, oracle_drafts(2), fn))]
    while eng.has_work():
        eng.step()
    assert all(len(r.output) == 20 and all(0 <= t < VOCAB for t in r.output) for r in rs)
    assert {known for _, known in verified} == {False, True}


def test_stop_tokens_among_drafts(verified):
    want = alone(PROMPT, 12)
    eng = Engine(RowModel(), max_tokens=100, max_seqs=1, block_size=4)
    stop = want[6]
    got = eng.generate([PROMPT], SamplingParams(max_new_tokens=12, draft_fn=oracle_drafts(8), stop_tokens=(stop,)))[0]
    assert got == want[:want.index(stop) + 1]


def test_few_pages_and_small_budgets_take_fewer_drafts(verified):
    for kw in (dict(max_tokens=8 + 12, max_step_tokens=3), dict(max_tokens=8 + 12, max_step_tokens=1, prefill_chunk=1), dict(max_tokens=8 + 12)):
        eng = Engine(RowModel(), max_seqs=1, block_size=4, **kw)
        assert eng.generate([PROMPT], SamplingParams(max_new_tokens=12, draft_fn=oracle_drafts(9)))[0] == alone(PROMPT, 12)


def test_drafts_that_are_refused(verified):
    eng = Engine(RowModel(), max_tokens=100, max_seqs=2, block_size=4)
    for kw in (dict(repetition_penalty=1.2), dict(logit_bias={1: 2.0}), dict(mask_fn=lambda o: None)):
        with pytest.raises(ValueError):
            eng.add_request("a", PROMPT, SamplingParams(draft_fn=oracle_drafts(2), **kw))
    with pytest.raises(ValueError):
        Engine(PagedModel(state=True), max_tokens=100, max_seqs=2).add_request("a", PROMPT, SamplingParams(draft_fn=oracle_drafts(2)))
    for bad in (lambda t: [VOCAB], lambda t: [-1], lambda t: ([1, 2], torch.zeros(1, VOCAB)), lambda t: ([1], torch.zeros(1, VOCAB + 1))):
        eng = Engine(RowModel(), max_tokens=100, max_seqs=2, block_size=4)
        r = eng.add_request("a", PROMPT, SamplingParams(max_new_tokens=4, draft_fn=bad))
        eng.step()
        with pytest.raises(ValueError):
            eng.step()
        assert eng.cache.live["a"].n_tokens == len(PROMPT) and r in eng.running      # the step left nothing
    with pytest.raises(ValueError):
        lookup_drafts(-1)


def test_a_row_without_a_choice_ends_its_request(verified):
    class Broken(RowModel):
        def forward(self, sa, sample=False):
            z = super().forward(sa)
            if sa.T == 3:
                z[1] = float("nan")
            return z
    eng = Engine(Broken(), max_tokens=100, max_seqs=2, block_size=4)
    r = eng.add_request("a", PROMPT, SamplingParams(max_new_tokens=9, draft_fn=oracle_drafts(2)))
    eng.step()
    with pytest.raises(RuntimeError):
        eng.step()
    assert r.finished and r.output == alone(PROMPT, 2) and not eng.cache.live


def test_looked_up_drafts():
    f = lookup_drafts(3, match=2)
    assert f([1, 2, 3, 4, 1, 2]) == [3, 4, 1] and f([5, 2, 9, 1, 2]) == [9, 1, 2] and f([1, 2, 3]) == [] and f([7]) == [] and f([4, 4]) == [4]
    assert lookup_drafts(0)([1, 1]) == []


# ---- a cache of bounded size --------------------------------------------------------------------------------------------------------------
def test_rows_leave_and_positions_stay():
    m = RowModel()
    eng = Engine(m, max_tokens=64, max_seqs=2, block_size=4, max_keys=16, first_keys=2, prefill_chunk=5)
    assert m.weighed == eng.cache.pages.num_blocks * 4
    r = eng.add_request("a", list(range(30)), SamplingParams(max_new_tokens=25))
    seen = []
    while eng.has_work():
        eng.step()
        if "a" in eng.cache.live:
            s = eng.cache.live["a"]
            seen.append(s.rows)
            assert s.rows <= 16 and len(s.blocks) == -(-s.rows // 4)
    assert len(r.output) == 25 and max(seen) > 12 and m.positions == list(range(54)) and m.cut and all(k == 14 and n > 16 for n, k in m.cut)
    assert eng.cache.pages.free_blocks == eng.cache.pages.num_blocks


def test_more_tokens_than_the_pool_holds():
    eng = Engine(RowModel(), max_tokens=24, max_seqs=1, block_size=4, max_keys=12, first_keys=1, prefill_chunk=6)
    assert len(eng.generate([[1] * 40], SamplingParams(max_new_tokens=30))[0]) == 30
    with pytest.raises(CacheFull):
        Engine(RowModel(), max_tokens=24, max_seqs=1, block_size=4, prefill_chunk=6).generate([[1] * 40], SamplingParams(max_new_tokens=30))


def test_forks_of_cut_requests_go_their_own_way():
    """shared pages are replaced where a request is cut back: the other one keeps its rows"""
    m = RowModel()
    eng = Engine(m, max_tokens=200, max_seqs=3, block_size=4, max_keys=32, first_keys=2)
    toks = list(np.random.default_rng(0).integers(0, VOCAB, 30))
    eng.run_entries([{"id": "a", "tokens": toks, "want": []}])
    eng.fork("a", "b")
    before = [m.pages[x].copy() for x in eng.cache.live["b"].blocks]
    eng.run_entries([{"id": "a", "tokens": [1, 2, 3, 4], "want": []}])
    a, b = eng.cache.live["a"], eng.cache.live["b"]
    assert a.rows == 28 and a.gone == 6 and a.n_tokens == 34 and b.rows == 30 and b.gone == 0 and not set(a.blocks) & set(b.blocks)
    assert all((m.pages[x] == y).all() for x, y in zip(b.blocks, before))
    eng.fork("a", "c")
    assert eng.cache.live["c"].gone == 6 and eng.cache.live["c"].rows == 28
    with pytest.raises(ValueError):
        eng.truncate("c", 20)                   # rows before its last eight are not all there
    eng.truncate("c", 30)
    assert eng.cache.live["c"].rows == 24
    eng.compact()
    eng.run_entries([{"id": "c", "tokens": [5], "want": [0]}], ["a", "b", "c"])
    assert eng.cache.pages.free_blocks == eng.cache.pages.num_blocks


def test_a_full_pool_leaves_a_request_as_it_is():
    """no free pages for shared ones: the request is cut back after a later step"""
    m = RowModel()
    eng = Engine(m, max_tokens=16, max_seqs=2, block_size=4, max_keys=8, first_keys=1)      # 6 pages
    eng.run_entries([{"id": "a", "tokens": [1] * 8, "want": []}])
    eng.fork("a", "b")
    eng.run_entries([{"id": "a", "tokens": [2] * 12, "want": []}])      # 2 shared, 3 more: one page is free, two are shared
    assert eng.cache.live["a"].rows == 20 and not m.cut
    eng.release("b")
    eng.run_entries([{"id": "a", "tokens": [3], "want": []}])
    assert eng.cache.live["a"].rows == 7 and m.cut == [(21, 7)]


def test_drafts_over_a_bounded_cache(verified):
    """both at once: rows that drafts brought leave with them, rows of little weight when there are too many"""
    m = RowModel()
    eng = Engine(m, max_tokens=64, max_seqs=2, block_size=4, max_keys=24, first_keys=2, prefill_chunk=7)
    r = eng.add_request("a", list(range(30)), SamplingParams(max_new_tokens=40, draft_fn=oracle_drafts(4, 3)))
    while eng.has_work():
        eng.step()
        if "a" in eng.cache.live:
            s = eng.cache.live["a"]
            assert s.rows <= 24 and s.n_tokens == (30 + len(r.output) - 1 if r.output else r.fed)
    assert r.output == Engine(RowModel(), max_tokens=200, max_seqs=1, block_size=4).generate([list(range(30))], SamplingParams(max_new_tokens=40))[0]      # (its tokens go by the last five rows)


def test_sizes_that_are_refused():
    for kw in (dict(max_keys=-1), dict(max_keys=16, first_keys=14), dict(max_keys=16, recent_keys=15), dict(max_keys=16, first_keys=-1), dict(max_keys=2, first_keys=0), dict(max_keys=16, weigh_last=-1)):
        with pytest.raises(ValueError):
            Engine(RowModel(), max_tokens=64, max_seqs=1, block_size=4, **kw)
    eng = Engine(RowModel(), max_tokens=400, max_seqs=1, block_size=4, max_keys=16, max_step_tokens=20)
    with pytest.raises(CacheFull):
        eng.run_entries([{"id": "a", "tokens": [1] * 40, "want": []}])
    assert not eng.cache.live


def test_steps_of_evicted_requests():
    e = [StepEntry(tokens=[5, 6], pos0=50, slot=1, block_table=[3, 4], row0=6), StepEntry(tokens=[7], pos0=2, slot=0, block_table=[1])]
    sa = build_step(e, 4)
    assert sa.tok_pos.tolist() == [6, 7, 2] and sa.tok_abs.tolist() == [50, 51, 2] and sa.ent_pos0.tolist() == [6, 2] and sa.block_table.tolist() == [[3, 4], [1, 0]]
    assert build_step(e[1:], 4).tok_abs is None
    c = CacheManager(64, 2, 4)
    s = c.admit("a")
    c.reserve(s, 20)
    s.n_tokens = 20
    had, to, n = c.evict("a", 9, 4)
    assert n == 20 and to == had[:3] and s.rows == 9 and s.gone == 11 and s.whole_from == 16 and c.pages_needed(s, 4) == 1
    c.evicted(had, to)
    assert c.pages.free_blocks == c.pages.num_blocks - 3


def test_options_of_the_command_line(verified, monkeypatch, capsys):
    import json

    from blazr_b200 import cli
    made = {}

    class Model(RowModel):
        def allocate(self, *a, weighed_rows=0):
            super().allocate(*a, weighed_rows)
            made.update(weighed=weighed_rows)
    monkeypatch.setattr(cli, "_load", lambda *a: Model())
    assert cli.main(["generate", "--model", "x", "--prompt", "3,1,4,1,5", "--max-new", "30", "--drafts", "3", "--max-keys", "24"]) == 0
    got = json.loads(capsys.readouterr().out)
    assert got["tokens"] == alone([3, 1, 4, 1, 5], 30) and made["weighed"] > 0
    assert cli.main(["generate", "--model", "x", "--prompt", "3,1,4,1,5", "--max-new", "30"]) == 0
    assert json.loads(capsys.readouterr().out) == got and made["weighed"] == 0
