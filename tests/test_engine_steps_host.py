"""Steps of the serving engine that fail, ids and slots that are spoken for, rules that are no numbers, without a GPU: what is refused leaves the engine able to go on."""
import numpy as np
import pytest
import torch

from blazr_b200.cache import CacheFull
from blazr_b200.engine import Engine, SamplingParams
from test_fork_host import VOCAB, PagedModel, alone, fake_rules

PROMPT = [3, 1, 4, 1, 5]


def engine(max_seqs=3, **kw):
    return Engine(PagedModel(), max_tokens=400, max_seqs=max_seqs, **{"block_size": 16, **kw})


def finish(eng):
    while eng.has_work():
        eng.step()
    assert eng.cache.slots.free_slots == eng.cache.slots.n and eng.cache.pages.free_blocks == eng.cache.pages.num_blocks


# ---- steps that fail -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n", [1, 2, 3])
def test_a_refused_mask_leaves_the_request_waiting(monkeypatch, n):
    """also one whose samples take every slot"""
    fake_rules(monkeypatch)
    eng = engine()
    words = [[0, 0]]
    r = eng.add_request("x", PROMPT, SamplingParams(max_new_tokens=4, n=n, mask_fn=lambda out: words[0]))
    for _ in range(2):
        with pytest.raises(ValueError):
            eng.step()
    assert list(eng.waiting) == [r] and not eng.running and not eng.cache.live
    words[0] = None
    finish(eng)
    assert [q.output for q in [r] + r.siblings] == [alone(PROMPT, 4)] * n


@pytest.mark.parametrize("n", [1, 3])
@pytest.mark.parametrize("bad", [RuntimeError, CacheFull])
def test_a_forward_pass_that_fails_once(monkeypatch, n, bad):
    fake_rules(monkeypatch)
    eng = engine()
    m, fails = eng.model, [1]
    fwd = m.forward

    def forward(sa, sample=False):
        if fails[0]:
            fails[0] -= 1
            raise bad("once")
        return fwd(sa, sample)
    m.forward = forward
    r = eng.add_request("x", PROMPT, SamplingParams(max_new_tokens=4, n=n))
    with pytest.raises(bad):
        eng.step()
    assert not eng.cache.live and list(eng.waiting) == [r] and eng.cache.slots.free_slots == 3
    finish(eng)
    assert [q.output for q in [r] + r.siblings] == [alone(PROMPT, 4)] * n
    # the same for requests that run already: they stay where they are
    r = eng.add_request("y", PROMPT, SamplingParams(max_new_tokens=4))
    eng.step()
    s = eng.add_request("z", PROMPT, SamplingParams(max_new_tokens=4, n=2))
    fails[0] = 1
    with pytest.raises(bad):
        eng.step()
    assert list(eng.cache.live) == ["y"] and eng.running == [r] and list(eng.waiting) == [s]
    finish(eng)
    assert [q.output for q in [r, s] + s.siblings] == [alone(PROMPT, 4)] * 3


def test_an_external_step_that_fails_leaves_no_new_request():
    eng = Engine(PagedModel(), max_tokens=32, max_seqs=2, block_size=16)               # 4 pages
    eng.run_entries([{"id": "a", "tokens": list(range(20)), "want": []}])
    with pytest.raises(CacheFull):
        eng.run_entries([{"id": "b", "tokens": [1] * 10, "want": []}, {"id": "a", "tokens": [2] * 40, "want": []}])
    assert list(eng.cache.live) == ["a"] and eng.cache.slots.free_slots == 1
    out = eng.run_entries([{"id": "b", "tokens": [4, 5], "want": [1]}, {"id": "a", "tokens": [3], "want": [0]}])
    assert out[0].argmax() == alone([4, 5], 1)[0] and out[1].argmax() == alone(list(range(20)) + [3], 1)[0]


# ---- ids ---------------------------------------------------------------------------------------------------------------------------------
def test_ids_of_samples_to_come_are_taken(monkeypatch):
    fake_rules(monkeypatch)
    eng = engine(4, prefill_chunk=2)
    r = eng.add_request("a", PROMPT, SamplingParams(max_new_tokens=4, n=3))
    taken = lambda: [eng.add_request, lambda i, p: eng.run_entries([{"id": i, "tokens": p, "want": []}])]
    for _ in range(2):                                                 # while the prompt waits, and while it runs
        for i in ("a#1", "a#2"):
            for use in taken():
                with pytest.raises(ValueError):
                    use(i, [1, 2])
        with pytest.raises(ValueError):
            eng.add_request("a", [1])
        eng.step()
    for i in ("a#1", "a#2"):
        with pytest.raises(ValueError):
            eng.fork("a", i)
    b = eng.add_request("a#3", [2, 7], SamplingParams(max_new_tokens=3))    # (nobody's)
    finish(eng)
    assert [q.output for q in [r] + r.siblings] == [alone(PROMPT, 4)] * 3 and [q.rid for q in r.siblings] == ["a#1", "a#2"] and b.output == alone([2, 7], 3)
    with pytest.raises(ValueError):                                    # they are the finished samples' still
        eng.add_request("a#1", [1])


def test_samples_do_not_take_ids_in_use(monkeypatch):
    """of requests that wait, of external ones, of samples to come"""
    fake_rules(monkeypatch)
    eng = engine(4)
    eng.add_request("b#1", [2, 7], SamplingParams(max_new_tokens=3))
    eng.run_entries([{"id": "c#2", "tokens": [5], "want": []}])
    eng.add_request("d#1", [2, 7], SamplingParams(max_new_tokens=3, n=2))    # d#1#1 to come
    for i, n in (("b", 2), ("c", 3), ("d", 2)):
        with pytest.raises(ValueError):
            eng.add_request(i, PROMPT, SamplingParams(n=n))
    with pytest.raises(ValueError):
        eng.add_request("d#1#1", PROMPT)
    with pytest.raises(ValueError):
        eng.add_request("c#2", PROMPT)                                 # an external request has it
    with pytest.raises(ValueError):
        eng.add_request(7, PROMPT, SamplingParams(n=0))
    eng.add_request(7, PROMPT, SamplingParams(max_new_tokens=2))
    with pytest.raises(ValueError):
        eng.add_request("7", PROMPT)
    eng.run_entries([], ["c#2"])
    c = eng.add_request("c", PROMPT, SamplingParams(max_new_tokens=4, n=3))
    finish(eng)
    assert [q.output for q in [c] + c.siblings] == [alone(PROMPT, 4)] * 3 and eng.requests["b#1"].output == alone([2, 7], 3)


def test_external_steps_leave_the_schedulers_requests_alone(monkeypatch):
    fake_rules(monkeypatch)
    eng = engine()
    r = eng.add_request("a", PROMPT, SamplingParams(max_new_tokens=4))
    for _ in range(2):                                                 # one that waits, one that runs
        with pytest.raises(ValueError):
            eng.run_entries([{"id": "e", "tokens": [1], "want": []}, {"id": "a", "tokens": [1, 2], "want": []}])
        assert "e" not in eng.cache.live
        eng.step()
    finish(eng)
    assert r.output == alone(PROMPT, 4)
    out = eng.run_entries([{"id": "a", "tokens": [4, 5], "want": [1]}])     # its name is free for others when it is through
    assert out[0].argmax() == alone([4, 5], 1)[0] and eng.fork("a", "b") is None
    out = eng.run_entries([{"id": "b", "tokens": [6], "want": [0]}], ["a", "b"])
    assert out[0].argmax() == alone([4, 5, 6], 1)[0] and not eng.has_work()


# ---- slots ---------------------------------------------------------------------------------------------------------------------------------
def test_external_requests_leave_the_slots_of_samples_to_come(monkeypatch):
    fake_rules(monkeypatch)
    eng = engine(3, prefill_chunk=2)
    r = eng.add_request("a", PROMPT, SamplingParams(max_new_tokens=4, n=2))
    eng.step()
    eng.run_entries([{"id": "e", "tokens": [4], "want": []}])          # the third slot
    with pytest.raises(CacheFull):
        eng.run_entries([{"id": "e", "tokens": [5], "want": []}, {"id": "f", "tokens": [4], "want": []}])
    assert sorted(eng.cache.live) == ["a", "e"] and eng.cache.live["e"].n_tokens == 1
    out = eng.run_entries([{"id": "e", "tokens": [5], "want": [0]}], ["e"])
    assert out[0].argmax() == alone([4, 5], 1)[0]
    finish(eng)
    assert [q.output for q in [r] + r.siblings] == [alone(PROMPT, 4)] * 2


def test_as_many_external_requests_as_slots():
    eng = engine(2)
    eng.run_entries([{"id": "a", "tokens": [4], "want": []}, {"id": "b", "tokens": [4], "want": []}])
    with pytest.raises(CacheFull):
        eng.run_entries([{"id": "a", "tokens": [5], "want": []}, {"id": "c", "tokens": [4], "want": []}])
    out = eng.run_entries([{"id": "a", "tokens": [5], "want": [0]}], ["a", "b"])
    assert out[0].argmax() == alone([4, 5], 1)[0]
