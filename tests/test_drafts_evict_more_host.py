"""Requests of a bounded cache and of drafts beside one another, without a GPU (test_drafts_evict_host.py has the stand-in models)."""
import time

import numpy as np
import pytest
import torch

from blazr_b200.cache import CacheFull
from blazr_b200.engine import Engine, SamplingParams, lookup_drafts
from test_drafts_evict_host import PROMPT, VOCAB, RowModel, alone, host_argmax, oracle_drafts, verified  # noqa: F401


def test_requests_that_cannot_be_cut_back_do_not_stop_others():
    """two samples share pages that there are no free ones for: they wait when the room of their weights is full, others go on, and so do they when pages are given back"""
    eng = Engine(RowModel(), max_tokens=36, max_seqs=4, block_size=4, max_keys=16, first_keys=1, max_step_tokens=4)      # 13 pages
    eng.run_entries([{"id": "x", "tokens": [1] * 4, "want": []}])
    for _ in range(3):
        eng.run_entries([{"id": "x", "tokens": [1] * 4, "want": []}])
    a = eng.add_request("a", PROMPT + PROMPT[:7], SamplingParams(max_new_tokens=30, n=2))
    for _ in range(12):
        if eng.cache.live["a"].rows == 20 if "a" in eng.cache.live else False:
            break
        eng.step()
    assert eng.cache.live["a"].rows == eng.cache.live["a#1"].rows == eng.weighed_rows == 20 and eng.cache.pages.free_blocks == 2 and not eng.model.cut
    c = eng.add_request("c", PROMPT[:2], SamplingParams(max_new_tokens=6))
    while not c.finished:
        eng.step()
    assert c.output == alone(PROMPT[:2], 6) and len(a.output) == 6
    with pytest.raises(CacheFull):
        eng.step()
    eng.release("x")
    while eng.has_work():
        eng.step()
        assert all(s.rows <= 16 for s in eng.cache.live.values())
    want = alone(PROMPT + PROMPT[:7], 30)
    assert a.output == a.siblings[0].output == want and eng.model.cut
    assert eng.cache.pages.free_blocks == eng.cache.pages.num_blocks


def test_prompts_that_cannot_be_cut_back_do_not_stop_others():
    """a prompt and its fork share eight pages, of which a cut would have to replace seven; five are free"""
    eng = Engine(RowModel(), max_tokens=48, max_seqs=3, block_size=4, max_keys=32, first_keys=1, max_step_tokens=4)      # 15 pages
    r = eng.add_request("a", PROMPT * 8, SamplingParams(max_new_tokens=3))
    for _ in range(8):
        eng.step()
    q = eng.fork("a", "b")
    others = eng.cache.pages.alloc(2)
    assert eng.cache.pages.free_blocks == 5
    eng.step()
    eng.step()
    assert eng.cache.live["a"].rows == eng.cache.live["b"].rows == eng.weighed_rows == 36 and not eng.model.cut
    c = eng.add_request("c", PROMPT[:2], SamplingParams(max_new_tokens=2))
    while not c.finished:
        eng.step()
    assert c.output == alone(PROMPT[:2], 2)
    with pytest.raises(CacheFull):
        eng.step()
    eng.cache.pages.free(others)
    with pytest.raises(CacheFull):              # five are free and seven wanted
        eng.step()
    eng.cache.release("b")
    eng.running.remove(q)
    while eng.has_work():
        eng.step()
    assert r.output == alone(PROMPT * 8, 3)


def test_sharers_are_cut_back_in_one_step():
    """the first one takes free pages, the last one keeps those that they shared"""
    m = RowModel()
    eng = Engine(m, max_tokens=16, max_seqs=2, block_size=4, max_keys=8, first_keys=1)      # 6 pages
    eng.run_entries([{"id": "a", "tokens": [1, 2, 3, 4, 5, 6, 7, 8], "want": []}])
    eng.fork("a", "b")
    eng.run_entries([{"id": "a", "tokens": [2, 4, 6, 8], "want": []}, {"id": "b", "tokens": [4, 4, 6, 6], "want": []}])
    a, b = eng.cache.live["a"], eng.cache.live["b"]
    assert a.rows == b.rows == 7 and m.cut == [(12, 7), (12, 7)] and not set(a.blocks) & set(b.blocks) and eng.cache.pages.free_blocks == 2
    row = lambda s: [int(m.pages[s.blocks[i // 4], i % 4]) for i in range(7)]
    assert row(a) == [1, 2, 4, 6, 8, 6, 8] and row(b) == [1, 2, 4, 6, 8, 6, 6]


def test_a_request_is_cut_back_before_it_is_refused():
    m = RowModel()
    eng = Engine(m, max_tokens=16, max_seqs=2, block_size=4, max_keys=8, first_keys=1)      # 6 pages
    eng.run_entries([{"id": "a", "tokens": [1] * 8, "want": []}])
    eng.fork("a", "b")
    eng.run_entries([{"id": "a", "tokens": [2] * 12, "want": []}])
    with pytest.raises(CacheFull):
        eng.run_entries([{"id": "a", "tokens": [3] * 5, "want": []}])
    assert eng.cache.live["a"].rows == 20 and not m.cut
    eng.release("b")
    eng.run_entries([{"id": "a", "tokens": [3] * 5, "want": []}])
    assert eng.cache.live["a"].n_tokens == 25 and m.cut == [(20, 7), (12, 7)]


# ---- guesses take what is left --------------------------------------------------------------------------------------------------------------
def run_until(eng, done, most):
    for _ in range(most):
        if done():
            return
        eng.step()
    assert done()


@pytest.mark.parametrize("wrong", [0, 1])
def test_guesses_take_no_tokens_from_other_requests(verified, wrong):
    """a step of four tokens, a request that brings nine guesses: others decode in every step, and prompts go on"""
    eng = Engine(RowModel(), max_tokens=400, max_seqs=4, block_size=4, max_step_tokens=4)
    a = eng.add_request("a", PROMPT, SamplingParams(max_new_tokens=60, draft_fn=oracle_drafts(9, wrong)))
    b = eng.add_request("b", PROMPT[:3], SamplingParams(max_new_tokens=9))
    run_until(eng, lambda: len(a.output) > 2 and b.output, 8)
    n, m = eng.steps, len(b.output)
    run_until(eng, lambda: b.finished, 9)
    assert eng.steps - n == 9 - m and not a.finished
    c = eng.add_request("c", PROMPT[2:], SamplingParams(max_new_tokens=1))
    run_until(eng, lambda: c.finished, 3)
    assert not a.finished
    run_until(eng, lambda: a.finished, 60)
    assert (a.output, b.output, c.output) == (alone(PROMPT, 60), alone(PROMPT[:3], 9), alone(PROMPT[2:], 1))


def test_guesses_take_no_pages_from_other_requests(verified):
    """eleven pages of one token are left: the second request needs one in every step, the first one's guesses take the others"""
    eng = Engine(RowModel(), max_tokens=20, max_seqs=2, block_size=1)
    a = eng.add_request("a", PROMPT, SamplingParams(max_new_tokens=14, draft_fn=oracle_drafts(30, 1)))
    b = eng.add_request("b", PROMPT[:3], SamplingParams(max_new_tokens=4))
    run_until(eng, lambda: b.finished, 4)
    assert len(a.output) == 4 and not a.finished
    run_until(eng, lambda: a.finished, 10)
    assert (a.output, b.output) == (alone(PROMPT, 14), alone(PROMPT[:3], 4))


def test_guesses_in_other_containers(verified):
    """tuples of one, two and three guesses, arrays, tensors; with None for the probabilities of certain ones"""
    want = alone(PROMPT, 13)
    for make in (tuple, np.array, torch.tensor, lambda g: tuple(torch.tensor(g)), lambda g: (g, None), lambda g: (torch.tensor(g), None), lambda g: tuple(np.array(g))):
        for n in (1, 2, 3):
            fn = oracle_drafts(n)
            eng = Engine(RowModel(), max_tokens=100, max_seqs=1, block_size=4)
            assert eng.generate([PROMPT], SamplingParams(max_new_tokens=13, draft_fn=lambda t: make(fn(t))))[0] == want
            assert eng.steps == 1 + 12 // (n + 1)


@pytest.mark.parametrize("top_k,T", [(2 ** 31, 0.5), (10 ** 12, 0.0), (-5, 0.0), (-2 ** 40, 0.0), (VOCAB, 0.5)])
def test_drafts_with_a_top_k_of_any_size(verified, top_k, T):
    """numbers that 32 bits do not hold, and negative ones beside a temperature of zero, choose among all tokens, as without drafts"""
    kw = dict(max_new_tokens=10, temperature=T, seed=1)
    eng = Engine(RowModel(), max_tokens=100, max_seqs=1, block_size=4)
    assert eng.generate([PROMPT], SamplingParams(top_k=top_k, draft_fn=oracle_drafts(3), **kw))[0] == alone(PROMPT, 10)


def plain_lookup(tokens, most, match):
    for m in range(min(match, len(tokens) - 1), 0, -1):
        for i in range(len(tokens) - m - 1, -1, -1):
            if tokens[i:i + m] == tokens[-m:]:
                return tokens[i + m:i + m + most]
    return []


def test_lookups_in_long_texts():
    """the same guesses as one place after the other gives, without the time that takes (a text of 32000 tokens without a match: 20 ms, several steps of a model)"""
    rng = np.random.default_rng(0)
    for n in list(range(0, 12)) + [50, 300]:
        for vocab in (1, 2, 5, 40, 2 ** 40):
            for most, match in ((0, 3), (1, 1), (4, 3), (9, 7)):
                text = [int(x) for x in rng.integers(0, vocab, n)]
                assert lookup_drafts(most, match)(text) == plain_lookup(text, most, match)
    text = [int(x) for x in rng.integers(0, 1000, 32000)] + [5000]

    def least(f):
        times = []
        for _ in range(5):
            t = time.perf_counter()
            assert f(text) == []
            times.append(time.perf_counter() - t)
        return min(times)
    assert least(lookup_drafts(4)) < least(lambda x: plain_lookup(x, 4, 3)) / 4
