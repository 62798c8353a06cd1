"""Shared pages, forks, compaction and sampling rules of the serving engine, without a GPU: bookkeeping over a stand-in model that keeps what it is fed in pages."""
import numpy as np
import pytest
import torch

from blazr_b200.cache import CacheFull, CacheManager, PagePool
from blazr_b200.engine import Engine, SamplingParams

VOCAB = 40


class PagedModel:
    """keeps every token in its page and a sum in its slot; its next token is a function of the whole sequence as its pages have it"""

    class cfg:
        vocab = VOCAB
        bigram = None

    def __init__(self, state=True, pooled=()):
        self.dev, self.state, self.pooled = torch.device("cpu"), state, pooled
        self.copies = 0

    def pooled_sizes(self):
        return self.pooled

    def has_state(self):
        return self.state

    def allocate(self, num_blocks, block_size, max_seqs, max_seq_tokens):
        self.pages, self.sums, self.bs = np.full((num_blocks, block_size), -1), np.zeros(max_seqs, np.int64), block_size

    def copy_pages(self, pairs):
        assert len({b for _, b in pairs}) == len(pairs) and not {a for a, _ in pairs} & {b for _, b in pairs}
        for a, b in pairs:
            self.pages[b] = self.pages[a]
        self.copies += len(pairs)

    def copy_slots(self, pairs):
        for a, b in pairs:
            self.sums[b] = self.sums[a]

    def forward(self, sa, sample=False):
        nxt = []
        written = {}
        for e in range(sa.B):
            toks = sa.tok_ids[sa.ent_start[e]:sa.ent_start[e + 1]]
            bt, p0, slot = sa.block_table[e], int(sa.ent_pos0[e]), sa.ent_slot[e]
            if p0 == 0:
                self.sums[slot] = 0
            for i, t in enumerate(toks):
                page, at = bt[(p0 + i) // self.bs], (p0 + i) % self.bs
                assert written.setdefault(page, e) == e, "two requests write into one page"
                self.pages[page, at] = t
                self.sums[slot] += t
                if sa.ent_start[e] + i in sa.want_rows:
                    seq = [self.pages[bt[j // self.bs], j % self.bs] for j in range(p0 + i + 1)]
                    assert sum(seq) == self.sums[slot]
                    nxt.append((sum((j + 1) * int(x) for j, x in enumerate(seq)) + 1) % VOCAB)
        self.last_ids = torch.tensor(nxt, dtype=torch.int32)
        return torch.nn.functional.one_hot(torch.tensor(nxt, dtype=torch.long), VOCAB).float()


def alone(prompt, n, **kw):
    """greedy continuation of a prompt by itself"""
    out = list(prompt)
    for _ in range(n):
        out.append((sum((j + 1) * x for j, x in enumerate(out)) + 1) % VOCAB)
    return out[len(prompt):]


def fake_rules(monkeypatch, seen=None):
    def process(logits, rules, out=None, **kw):
        if seen is not None:
            seen.append((logits.clone(), rules, kw))
        out.copy_(logits)
        if "mask" in kw:
            bits = np.unpackbits(kw["mask"].numpy().view(np.uint8), axis=1, bitorder="little")[:, :logits.shape[1]]
            out[torch.from_numpy(bits == 0)] = float("-inf")
        return out
    monkeypatch.setattr("blazr_b200.seqops.process_logits", process)
    monkeypatch.setattr("blazr_b200.seqops.argmax", lambda z, ids: ids.copy_(z.argmax(1).int()))
    monkeypatch.setattr("blazr_b200.seqops.error_flags", lambda: 0)


def test_pages_have_owners():
    p = PagePool(5, 16)
    a = p.alloc(2)
    p.share(a)
    p.free(a)
    assert p.free_blocks == 3 and p.owners(a[0]) == 1
    p.free([a[0]])
    assert p.free_blocks == 4 and p.alloc(1) == [a[0]]
    with pytest.raises(AssertionError):
        p.free([4])
    with pytest.raises(AssertionError):
        p.share([4])


def test_compaction_fills_the_front():
    p = PagePool(8, 16)
    a = p.alloc(7)
    p.share([6])
    p.free([0, 2, 3, 5])
    moves = p.compact()
    assert moves == {4: 0, 6: 2} and p.owners(2) == 2 and p.owners(0) == 1 and p.free_blocks == 5
    assert p.alloc(5) == [3, 4, 5, 6, 7] and p.compact() == {}


@pytest.mark.parametrize("n", [1, 15, 16, 17, 32, 40])
def test_a_fork_copies_what_it_writes(n):
    cm = CacheManager(200, 3, 16)
    a = cm.admit("a")
    assert cm.reserve(a, n) == []
    a.n_tokens = n
    free = cm.pages.free_blocks
    b = cm.fork("a", "b")
    assert cm.pages.free_blocks == free and b.blocks == a.blocks and b.slot != a.slot and b.n_tokens == n
    partly = n % 16 != 0
    assert cm.pages_needed(b, 1) == 1 and cm.pages_to_copy(b) == partly
    copies = cm.reserve(b, 1)
    assert copies == ([(a.blocks[-1], b.blocks[-1])] if partly else [])
    assert cm.reserve(a, 1) == [] or not partly                      # the other one has the page to itself now
    assert not set(a.blocks[n // 16:]) & set(b.blocks[n // 16:])
    cm.release("a")
    cm.release("b")
    assert cm.pages.free_blocks == cm.pages.num_blocks


def test_pooled_blocks_are_written_after_their_page():
    """a block of 24 positions that begins in a shared page has its mean written there when it is complete"""
    cm = CacheManager(200, 2, 16, pooled=(24,))
    a = cm.admit("a")
    cm.reserve(a, 32)
    a.n_tokens = 32                                                    # positions 24 .. 47 are not complete: the block begins in page 1
    b = cm.fork("a", "b")
    copies = cm.reserve(b, 1)
    assert copies == [(a.blocks[1], b.blocks[1])] and b.blocks[0] == a.blocks[0]


def test_pages_that_run_out_leave_a_fork_whole():
    cm = CacheManager(32, 2, 16)
    a = cm.admit("a")
    cm.reserve(a, 60)
    a.n_tokens = 60
    b = cm.fork("a", "b")
    before = list(b.blocks)
    with pytest.raises(CacheFull):
        cm.reserve(b, 1)
    assert b.blocks == before and cm.pages.owners(before[-1]) == 2
    with pytest.raises(CacheFull):
        cm.fork("a", "c")                                              # no slot: nothing is shared
    assert cm.pages.owners(before[0]) == 2


def test_truncated_requests_share_nothing_they_write():
    cm = CacheManager(200, 2, 16)
    a = cm.admit("a")
    cm.reserve(a, 40)
    a.n_tokens = 40
    b = cm.fork("a", "b")
    cm.truncate("b", 20, 7)
    assert len(b.blocks) == 2 and b.last_token == 7 and cm.pages.owners(a.blocks[2]) == 1
    assert cm.reserve(b, 1) == [(a.blocks[1], b.blocks[1])]
    with pytest.raises(ValueError):
        cm.truncate("b", 21, 0)
    cm.truncate("b", 0, -1)
    assert b.blocks == []


@pytest.mark.parametrize("bs", [1, 4, 16])
def test_forks_run_on_like_requests_of_their_own(monkeypatch, bs):
    fake_rules(monkeypatch)
    eng = Engine(PagedModel(), max_tokens=400, max_seqs=4, block_size=bs)
    eng.add_request("a", [3, 1, 4, 1, 5], SamplingParams(max_new_tokens=12))
    for _ in range(4):
        eng.step()
    b = eng.fork("a", "b", SamplingParams(max_new_tokens=20))
    eng.step()
    c = eng.fork("b", "c")
    with pytest.raises(ValueError):
        eng.fork("a", "c")
    with pytest.raises(ValueError):
        eng.fork("nobody", "d")
    a = eng.requests["a"]
    moved = 0
    while eng.has_work():
        eng.step()
        moved += eng.compact()
    assert a.output == alone([3, 1, 4, 1, 5], 12) and b.output == alone([3, 1, 4, 1, 5], 20) and c.output == alone([3, 1, 4, 1, 5], 20)
    assert eng.cache.pages.free_blocks == eng.cache.pages.num_blocks and eng.cache.slots.free_slots == 4


def test_a_fork_within_its_prompt(monkeypatch):
    fake_rules(monkeypatch)
    prompt = list(range(1, 38))
    eng = Engine(PagedModel(), max_tokens=400, max_seqs=2, block_size=16, prefill_chunk=10)
    eng.add_request("a", prompt, SamplingParams(max_new_tokens=5))
    eng.step()
    b = eng.fork("a", "b")
    while eng.has_work():
        eng.step()
    assert eng.requests["a"].output == b.output == alone(prompt, 5) and eng.model.copies == 1


def test_externally_scheduled_forks_and_truncation():
    m = PagedModel(state=False)
    eng = Engine(m, max_tokens=400, max_seqs=3, block_size=4)
    m.sums = np.zeros(3, np.int64)
    monk = m.forward

    def forward(sa, sample=False):                                     # the sums are no state here: made again from the pages
        for e in range(sa.B):
            m.sums[sa.ent_slot[e]] = sum(m.pages[sa.block_table[e][j // 4], j % 4] for j in range(sa.ent_pos0[e]))
        return monk(sa, sample)
    m.forward = forward
    eng.run_entries([{"id": "a", "tokens": [5, 6, 7, 8, 9, 1], "want": []}])
    assert eng.fork("a", "b") is None
    eng.run_entries([{"id": "a", "tokens": [2, 3], "want": []}, {"id": "b", "tokens": [9, 9, 9], "want": []}])
    eng.truncate("b", 5)
    out = eng.run_entries([{"id": "a", "tokens": [4], "want": [0]}, {"id": "b", "tokens": [4], "want": [0]}], ["a", "b"])
    assert out[0].argmax() == alone([5, 6, 7, 8, 9, 1, 2, 3, 4], 1)[0] and out[1].argmax() == alone([5, 6, 7, 8, 9, 4], 1)[0]
    assert eng.cache.pages.free_blocks == eng.cache.pages.num_blocks
    with pytest.raises(ValueError):
        eng.truncate("a", 1)
    eng2 = Engine(PagedModel(state=True), max_tokens=64, max_seqs=1)
    eng2.run_entries([{"id": "a", "tokens": [1, 2], "want": []}])
    with pytest.raises(ValueError):
        eng2.truncate("a", 1)


def test_pages_that_run_out_in_a_step_leave_copies_made():
    m = PagedModel()
    eng = Engine(m, max_tokens=32, max_seqs=2, block_size=16)          # 4 pages
    eng.run_entries([{"id": "a", "tokens": list(range(20)), "want": []}])
    eng.fork("a", "b")
    with pytest.raises(CacheFull):                                     # b's copy takes the third page, a wants two more
        eng.run_entries([{"id": "b", "tokens": [1], "want": []}, {"id": "a", "tokens": [2] * 29, "want": []}])
    out = eng.run_entries([{"id": "a", "tokens": [3], "want": [0]}, {"id": "b", "tokens": [4], "want": [0]}])
    assert out[0].argmax() == alone(list(range(20)) + [3], 1)[0] and out[1].argmax() == alone(list(range(20)) + [4], 1)[0]


def test_a_prompt_is_sampled_several_times(monkeypatch):
    fake_rules(monkeypatch)
    m = PagedModel()
    eng = Engine(m, max_tokens=400, max_seqs=3, block_size=16)
    steps = []
    fwd = m.forward
    m.forward = lambda sa, sample=False: (steps.append(sa.T), fwd(sa, sample))[1]
    outs = eng.generate([[3, 1, 4], [2, 7]], SamplingParams(max_new_tokens=6, n=3))
    assert outs == [[alone([3, 1, 4], 6)] * 3, [alone([2, 7], 6)] * 3]
    assert steps[0] == 3 and sum(steps) == 3 + 5 * 3 + 2 + 5 * 3       # each prompt once; the second waits for three slots
    assert not eng.requests and eng.cache.slots.free_slots == 3
    with pytest.raises(ValueError):
        eng.add_request("x", [1], SamplingParams(n=4))
    with pytest.raises(ValueError):
        eng.add_request("x", [1], SamplingParams(n=0))


def test_a_fork_leaves_the_slots_of_samples_to_come(monkeypatch):
    fake_rules(monkeypatch)
    eng = Engine(PagedModel(), max_tokens=400, max_seqs=3, block_size=16, prefill_chunk=2)
    eng.add_request("a", [3, 1, 4, 1, 5], SamplingParams(max_new_tokens=4, n=3))
    eng.step()
    with pytest.raises(CacheFull):
        eng.fork("a", "b")
    r = eng.requests["a"]
    while eng.has_work():
        eng.step()
    assert [q.output for q in [r] + r.siblings] == [alone([3, 1, 4, 1, 5], 4)] * 3


def test_rules_of_a_batch(monkeypatch):
    seen = []
    fake_rules(monkeypatch, seen)
    eng = Engine(PagedModel(), max_tokens=400, max_seqs=3, block_size=16)
    allow = np.zeros(2, np.uint32)
    allow[0] = 1 << 7
    eng.add_request("plain", [1, 2], SamplingParams(max_new_tokens=2))
    eng.add_request("pen", [3, 4, 5], SamplingParams(max_new_tokens=2, repetition_penalty=1.5, presence_penalty=0.25, logit_bias={4: 2.0, 9: -1.0}))
    eng.add_request("mask", [6], SamplingParams(max_new_tokens=2, mask_fn=lambda out: allow if not out else None))
    eng.step()
    logits, rules, kw = seen[0]
    assert rules.tolist() == [[1, 0, 0, 0], [1.5, 0.25, 0, 0], [1, 0, 0, 0]]
    assert kw["hist"].tolist() == [3, 4, 5] and kw["hist_start"].tolist() == [0, 0, 3, 3] and kw["hist_prompt"].tolist() == [0, 3, 0]
    assert kw["bias_ids"].tolist() == [4, 9] and kw["bias_vals"].tolist() == [2, -1] and kw["bias_start"].tolist() == [0, 0, 2, 2]
    assert kw["mask"].tolist() == [[-1, -1], [-1, -1], [128, 0]]
    assert eng.requests["mask"].output == [7] and eng.requests["plain"].output == alone([1, 2], 1)
    eng.step()
    first = eng.requests["pen"].output[0]
    assert seen[1][2]["hist"].tolist() == [3, 4, 5, first, 7] and seen[1][2]["hist_prompt"].tolist() == [0, 3, 0] and "mask" not in seen[1][2]
    assert not eng.has_work()


def test_rules_that_are_refused(monkeypatch):
    fake_rules(monkeypatch)
    eng = Engine(PagedModel(), max_tokens=100, max_seqs=2, block_size=16)
    for p in (SamplingParams(repetition_penalty=0.0), SamplingParams(repetition_penalty=float("nan")), SamplingParams(logit_bias={VOCAB: 1.0}), SamplingParams(logit_bias={-1: 1.0})):
        with pytest.raises(ValueError):
            eng.add_request("x", [1], p)
    assert not eng.requests and not eng.has_work()
    words = [[1, 2, 3]]
    eng.add_request("x", [1, 2], SamplingParams(max_new_tokens=3, mask_fn=lambda out: words[0]))
    for bad in ([1, 2, 3], [0, 0], [0, 1 << 20]):                      # wrong length, nothing, only tokens behind the vocabulary
        words[0] = bad
        with pytest.raises(ValueError):
            eng.step()
    words[0] = None                                                    # the request is as it was
    while eng.has_work():
        eng.step()
    assert eng.requests["x"].output == alone([1, 2], 3)


def test_the_command_line_has_them(monkeypatch, capsys):
    """options of `generate`: bits of the cache, samples, penalties, biases; a line a sample"""
    import json

    from blazr_b200 import cli
    seen, made = [], {}
    fake_rules(monkeypatch, seen)

    class Model(PagedModel):
        def allocate(self, *a, kv_bits=32):
            made.update(bits=kv_bits)
            super().allocate(*a)
    monkeypatch.setattr(cli, "_load", lambda *a: Model())
    assert cli.main(["generate", "--model", "x", "--prompt", "3,1,4", "--prompt", "2,7", "--max-new", "5", "--samples", "3", "--kv-bits", "4", "--repetition-penalty", "1.5",
                     "--presence-penalty", "0.25", "--frequency-penalty", "0.5", "--logit-bias", "7:-2.5,9:1"]) == 0
    lines = [json.loads(s) for s in capsys.readouterr().out.splitlines()]
    assert [x["prompt"] for x in lines] == [[3, 1, 4]] * 3 + [[2, 7]] * 3 and made == {"bits": 4}
    assert [x["tokens"] for x in lines] == [alone([3, 1, 4], 5)] * 3 + [alone([2, 7], 5)] * 3
    _, rules, kw = seen[0]
    assert rules[0].tolist() == [1.5, 0.25, 0.5, 0.0] and kw["bias_ids"][:2].tolist() == [7, 9] and kw["bias_vals"][:2].tolist() == [-2.5, 1.0]
    assert cli.main(["generate", "--model", "x", "--prompt", "2,7", "--max-new", "4"]) == 0 and made == {"bits": 32}
    assert json.loads(capsys.readouterr().out) == {"prompt": [2, 7], "tokens": alone([2, 7], 4)}
