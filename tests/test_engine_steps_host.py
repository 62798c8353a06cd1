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


# ---- rules and logits that are no numbers ----------------------------------------------------------------------------------------------------
NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("p", [
    dict(presence_penalty=NAN), dict(presence_penalty=INF), dict(frequency_penalty=-INF), dict(frequency_penalty=NAN), dict(frequency_penalty=1e39), dict(presence_penalty=-1e300),
    dict(repetition_penalty=INF), dict(repetition_penalty=1e39), dict(repetition_penalty=1e-40), dict(repetition_penalty=-1.0), dict(logit_bias={3: NAN}), dict(logit_bias={3: INF}),
    dict(logit_bias={3: 1e39}), dict(logit_bias={i: -INF for i in range(VOCAB)}), dict(logit_bias={i: -1e39 for i in range(VOCAB)}), dict(temperature=NAN),
    dict(temperature=INF, logit_bias={3: -INF}), dict(temperature=1e39, mask_fn=lambda out: None), dict(temperature=0.5, top_p=0.0), dict(temperature=0.5, top_p=NAN),
    dict(temperature=0.5, top_p=-1.0), dict(temperature=1e-40)])
def test_rules_that_are_no_numbers(p):
    eng = engine()
    with pytest.raises(ValueError):
        eng.add_request("x", PROMPT, SamplingParams(**p))
    assert not eng.requests and not eng.has_work()
    eng.add_request("x", PROMPT)
    eng.step()
    with pytest.raises(ValueError):
        eng.fork("x", "y", SamplingParams(**p))
    assert list(eng.cache.live) == ["x"]


def test_rules_at_the_ends_of_their_range(monkeypatch):
    fake_rules(monkeypatch)
    eng = engine()
    for i, p in enumerate((dict(logit_bias={3: -INF}), dict(logit_bias={3: -1e300, 4: 3e38}), dict(presence_penalty=3e38, frequency_penalty=-3e38), dict(repetition_penalty=3e38),
                           dict(repetition_penalty=1.2e-38), dict(top_p=0.0), dict(temperature=-1.0))):
        eng.add_request(i, PROMPT, SamplingParams(max_new_tokens=1, **p))
    with np.errstate(all="raise"):
        finish(eng)


def test_a_mask_of_forbidden_tokens(monkeypatch):
    """allowed by the mask are only tokens whose bias forbids them"""
    fake_rules(monkeypatch)
    eng = engine()
    words = [[0b11000, 0]]
    r = eng.add_request("x", PROMPT, SamplingParams(max_new_tokens=2, logit_bias={3: -INF, 4: -1e39, 5: -2.0}, mask_fn=lambda out: words[0]))
    with pytest.raises(ValueError):
        eng.step()
    assert list(eng.waiting) == [r]
    words[0] = [0b110000, 0]
    finish(eng)
    assert len(r.output) == 2


@pytest.mark.parametrize("bad", [NAN, INF, -INF, 3e38])
def test_logits_that_leave_no_choice(monkeypatch, bad):
    """the request ends without that token, the others go on, and nothing is sampled from probabilities that are none (3e38: not after the temperature)"""
    fake_rules(monkeypatch)
    monkeypatch.setattr("torch.multinomial", lambda p, n, generator=None: (_ for _ in ()).throw(AssertionError) if not bool((p >= 0).all()) or not float(p.sum()) > 0 else p.argmax(0, True))
    eng = engine()
    m, spoil = eng.model, [False]
    fwd = m.forward

    def forward(sa, sample=False):
        z = fwd(sa, sample) * 100
        if spoil[0]:
            z[0, :] = bad if bad == -INF else z[0]
            z[0, 7] = bad
        return z
    m.forward = forward
    sampled = SamplingParams(max_new_tokens=4, temperature=0.5)
    x, y = eng.add_request("x", PROMPT, sampled), eng.add_request("y", [2, 7], sampled)
    eng.step()
    spoil[0] = True
    with pytest.raises(RuntimeError, match="x"):
        eng.step()
    spoil[0] = False
    assert x.finished and len(x.output) == 1 and len(y.output) == 2 and list(eng.cache.live) == ["y"]
    finish(eng)
    assert y.output == alone([2, 7], 4)


# ---- generate ------------------------------------------------------------------------------------------------------------------------------------
def test_a_generate_that_fails_takes_its_requests_back(monkeypatch):
    fake_rules(monkeypatch)
    eng = engine()
    other = eng.add_request("other", PROMPT, SamplingParams(max_new_tokens=6))
    eng.step()
    masked = SamplingParams(max_new_tokens=4, n=2, mask_fn=lambda out: [0, 0] if len(out) == 2 else None)
    for _ in range(2):                                                 # (a refused mask in the middle of the output)
        with pytest.raises(ValueError):
            eng.generate([[2, 7], [3, 8]], masked)
        assert list(eng.requests) == ["other"] and not eng.waiting and eng.running in ([other], []) and eng.cache.slots.free_slots == 3 - len(eng.running)
    with pytest.raises(ValueError):
        eng.generate([[2, 7], []])
    with pytest.raises(ValueError):
        eng.generate([[2, 7]], SamplingParams(temperature=0.5, top_k=-1))
    assert not eng._sample_ids and list(eng.requests) == ["other"]
    assert eng.generate([[2, 7], [3, 8]], SamplingParams(max_new_tokens=4)) == [alone([2, 7], 4), alone([3, 8], 4)]
    finish(eng)
    assert other.output == alone(PROMPT, 6)


def test_requests_of_the_scheduler_are_not_released_from_outside(monkeypatch):
    fake_rules(monkeypatch)
    eng = engine()
    r = eng.add_request("a", PROMPT, SamplingParams(max_new_tokens=4, n=2))
    for _ in range(2):
        with pytest.raises(ValueError):
            eng.release("a")
        with pytest.raises(ValueError):
            eng.run_entries([{"id": "e", "tokens": [1], "want": []}], ["e", "a"])
        assert "e" not in eng.cache.live
        eng.step()
    finish(eng)
    eng.release("a")                                                   # (through: nothing to give back)
    eng.release("nobody")
    assert [q.output for q in [r] + r.siblings] == [alone(PROMPT, 4)] * 2
