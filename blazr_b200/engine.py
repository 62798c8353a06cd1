"""Serving engine of layer-list models: request queue, scheduler, cache / state manager, sampling.

One `Engine.step()` is one forward pass over a flat mixed batch: every running request contributes its one decoded token, and
prompts that are not yet in the cache contribute their next portion (chunked prefill under a token budget), as the reference's
batch engine does (src/engine/batch_engine.rs:172-272 chunked prefill, src/engine/batch_decode.rs:35-209 decode batches).
Requests take a state slot and KV pages from `CacheManager` (blazr_b200/cache.py) on admission / growth and give them back when
they finish; pages and slots are reused.

`Engine.run_entries()` is the same step with the batch given from outside (which request brings which tokens): trace replay and
the tests drive it; `step()` builds the same entries from its own queues.  Both go through `_forward`, the only place that
touches the model.

`fork()` lets a second request continue from where another is: KV pages are shared and copied when one of the two is about to write
into them, recurrent state is copied at once.  `SamplingParams.n` samples a prompt several times that way.  Penalties, biases and
masks of a request are applied to its logits on the GPU before its token is chosen (seqops.process_logits).

Drafts (`SamplingParams.draft_fn`): a decoded request brings its last token and guesses of the next ones in one step, and keeps those that the
model's own probabilities bear out (seqops.verify_drafts).  A cache of bounded size (`max_keys`): the weight that every cached key is given is added up as the
steps run (seqops.key_weights), and a request that holds more rows is cut back to those of largest weight (seqops.evict_keys).
"""
from __future__ import annotations

from array import array
from collections import deque
from dataclasses import dataclass, field, replace
from typing import Any, Callable, Deque, Dict, List, Optional, Sequence, Set, Tuple

import numpy as np
import torch

from . import seqops
from .batch import StepEntry, build_step
from .cache import CacheFull, CacheManager, SeqState
from .layered import LayeredModel

F32_MAX, F32_TINY = float(np.finfo(np.float32).max), float(np.finfo(np.float32).tiny)


@dataclass
class SamplingParams:
    """temperature 0 = greedy (arg-max kernel); otherwise soft-max sampling, optionally among the top_k / top_p tokens.
    repetition_penalty: the logits of tokens of the prompt and the output are divided by it (multiplied where negative); frequency_penalty times how often, and
    presence_penalty once if, a token stands in the output is subtracted; logit_bias: added per token; mask_fn(output so far) -> int32 words, bit v % 32 of word
    v / 32 set where token v is allowed, or None (all).  n: samples of the prompt, which is run once (Request.siblings holds the others).
    draft_fn(prompt and output so far) -> guesses of the next tokens, which one step verifies together, or (guesses, f32 [guesses, vocab] probabilities they were drawn from);
    what comes out has the distribution that temperature, top_k and top_p give without them (tokens of equal logits are kept or left out together)"""
    temperature: float = 0.0
    top_k: int = 0
    top_p: float = 1.0
    seed: Optional[int] = None
    max_new_tokens: int = 16
    stop_tokens: Tuple[int, ...] = ()
    repetition_penalty: float = 1.0
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0
    logit_bias: Optional[Dict[int, float]] = None
    mask_fn: Optional[Callable[[List[int]], Optional[Sequence[int]]]] = None
    n: int = 1
    draft_fn: Optional[Callable[[List[int]], Any]] = None

    def ruled(self) -> bool:
        """whether the logits are changed before the token is chosen"""
        return bool(self.repetition_penalty != 1.0 or self.presence_penalty or self.frequency_penalty or self.logit_bias or self.mask_fn)


def lookup_drafts(most: int, match: int = 3) -> Callable[[List[int]], List[int]]:
    """a draft_fn that looks the last `match` tokens (or fewer, down to one) up in the text before them and guesses the up to `most` tokens that followed there last"""
    if most < 0 or match < 1:
        raise ValueError(f"{most} drafts by {match} tokens")

    def drafts(tokens: List[int]) -> List[int]:
        text, hits = np.frombuffer(array("q", tokens), dtype=np.int64), None
        for m in range(min(match, len(tokens) - 1)):       # places whose last m + 1 tokens are the text's
            ends = np.nonzero(text[:-1] == text[-1])[0] if m == 0 else hits[hits >= m]
            ends = ends[text[ends - m] == text[-1 - m]]
            if not ends.size:
                break
            hits = ends
        return tokens[hits[-1] + 1:hits[-1] + 1 + most] if hits is not None else []
    return drafts


@dataclass
class Request:
    rid: str
    prompt: List[int]
    params: SamplingParams
    output: List[int] = field(default_factory=list)
    fed: int = 0                 # prompt tokens already in the cache
    finished: bool = False
    siblings: List["Request"] = field(default_factory=list)   # the other samples of params.n
    _gen: Optional[torch.Generator] = None
    _probs: Optional[torch.Tensor] = None    # of the drafts that the step verifies


class Engine:
    def __init__(self, model: LayeredModel, max_tokens: int, max_seqs: int = 4, block_size: int = 16, max_step_tokens: int = 2048,
                 prefill_chunk: int = 512, kv_bits: int = 32, max_keys: int = 0, first_keys: int = 4, recent_keys: int = 0, weigh_last: int = 0):
        """max_tokens: tokens all live requests may hold together (the KV pool is made for this many, rounded up to pages);
        max_seqs: state slots = most requests live at a time; kv_bits: bits of a cached key or value, 32 or 4.
        max_keys: > 0: a request that holds more cached rows between two steps is cut back to seven eighths of them: the first first_keys, the last recent_keys (0: a quarter of
        max_keys) and, in every layer and key head, those that were given the most attention since they came (by guesses that were rejected, too).  weigh_last: only the attention
        of that many last tokens of a step's portion counts (0: of all).  Beside the cache, steps of many tokens or long sequences take a work area for the weights of up to
        256 MB of scores or keys, and some for the tokens"""
        self.model = model
        self.cache = CacheManager(max_tokens, max_seqs, block_size, model.pooled_sizes() if hasattr(model, "pooled_sizes") else ())
        room = self.cache.pages.num_blocks * block_size
        self.max_keys, self.first_keys, self.recent_keys = max_keys, first_keys, recent_keys or max_keys // 4
        self.keep_keys = max_keys - max_keys // 8
        if max_keys < 0 or weigh_last < 0 or (max_keys > 0 and (first_keys < 0 or self.recent_keys < 1 or first_keys + self.recent_keys > self.keep_keys)):
            raise ValueError(f"the first {first_keys} and the last {self.recent_keys} of {self.keep_keys} rows to keep")
        # (a slot's weights have room for what a request may hold when a step ends)
        self.weighed_rows = min(room, max_keys + max_step_tokens) if max_keys > 0 else 0
        model.allocate(self.cache.pages.num_blocks, block_size, max_seqs, room, **({} if kv_bits == 32 else {"kv_bits": kv_bits}), **({"weighed_rows": self.weighed_rows} if max_keys > 0 else {}))
        if max_keys > 0:
            model.weigh_last = weigh_last
        self.max_step_tokens, self.prefill_chunk = max_step_tokens, prefill_chunk
        self.waiting: Deque[Request] = deque()
        self.running: List[Request] = []
        self.requests: Dict[str, Request] = {}
        self._sample_ids: Set[str] = set()       # of the samples that prompts which are not through will have
        self.steps = 0

    # ---- the one place that runs the model -----------------------------------------------------------------------------------
    def _forward(self, batch: Sequence[Tuple[str, Sequence[int], Sequence[int]]], sample: bool = False) -> torch.Tensor:
        """batch: (request id, next tokens, wanted places) per entry.  Admits unseen ids, reserves pages, runs the step, advances
        the token counts.  Returns the f32 logits [wanted, vocab] (device; valid until the next step).  Where it raises, the ids that it admitted are none again."""
        entries: List[StepEntry] = []
        copies: List[Tuple[int, int]] = []
        admitted: List[str] = []
        seen = set()
        for rid, _, _ in batch:
            if rid in seen:
                raise ValueError(f"request {rid} appears twice in one step")
            seen.add(rid)
        if self.max_keys > 0:       # (requests that could not be cut back when it was their turn)
            self._cut([rid for rid, toks, _ in batch if rid in self.cache.live and self.cache.live[rid].rows + len(toks) > self.weighed_rows])
        try:
            try:
                for rid, toks, want in batch:
                    seq = self.cache.live.get(rid)
                    if seq is None:
                        seq = self.cache.admit(rid)
                        admitted.append(rid)
                    if self.max_keys > 0 and seq.rows + len(toks) > self.weighed_rows:
                        raise CacheFull(f"request {rid} would hold {seq.rows + len(toks)} cached rows, {self.weighed_rows} have room for their weights")
                    copies += self.cache.reserve(seq, len(toks))
                    entries.append(StepEntry(tokens=toks, pos0=seq.n_tokens, slot=seq.slot, block_table=seq.blocks, want=want, prev=seq.last_token, row0=seq.rows))
            finally:
                if copies:      # also when the pages ran out on the way: these requests hold their copies already
                    self.model.copy_pages(copies)
            sa = build_step(entries, self.cache.block_size)
            logits = self.model.forward(sa, sample=sample)
        except BaseException:
            for rid in admitted:
                self.cache.release(rid)
            raise
        for rid, toks, _ in batch:
            self.cache.live[rid].n_tokens += len(toks)
            self.cache.live[rid].last_token = int(toks[-1])
        self.steps += 1
        return logits

    def release(self, rid: str) -> None:
        """gives an externally scheduled request's pages and slot back; of an id that holds none nothing"""
        if self._scheduled(rid):
            raise ValueError(f"request {rid} belongs to the scheduler")
        if rid in self.cache.live:
            self.cache.release(rid)

    def fork(self, rid: str, new_rid: str, params: Optional[SamplingParams] = None) -> Optional[Request]:
        """a second request that continues from where the live request `rid` is.  Of a request of the engine's own scheduler a Request (with the prompt and the
        output so far, and params or the same ones) that runs from the next step on; of an externally scheduled one None.  A sampled one draws from the beginning of its
        seed's numbers, not from where `rid` is in them: params of another seed make another continuation"""
        rid, new_rid = str(rid), str(new_rid)
        if self._in_use(new_rid):
            raise ValueError(f"request id {new_rid} is in use")
        if rid not in self.cache.live:
            raise ValueError(f"request {rid} holds nothing in the cache")
        if self.cache.slots.free_slots <= self._promised():
            raise CacheFull(f"no state slot for request {new_rid}: {self.cache.slots.free_slots} free, {self._promised()} kept for samples of running prompts")
        r = self._scheduled(rid)
        if r is not None:
            self._check(replace(params or r.params, n=1))
        self._fork_cache(rid, new_rid)
        if r is None:
            return None
        q = self._request(new_rid, r.prompt, replace(params or r.params, n=1))
        q.output, q.fed = list(r.output), r.fed
        self.running.append(q)
        return q

    def _in_use(self, rid: str) -> bool:
        return rid in self.requests or rid in self.cache.live or rid in self._sample_ids

    def _scheduled(self, rid: str) -> Optional[Request]:
        """the scheduler's request of that id; an id whose request is through may be an external one's"""
        r = self.requests.get(rid)
        return None if r is None or r.finished else r

    def _promised(self) -> int:
        """slots that running requests take when their prompt is through, for its other samples"""
        return sum(r.params.n - 1 for r in self.running if r.params.n > 1 and not r.output and not r.siblings)

    def _fork_cache(self, rid: str, new_rid: str) -> None:
        src, new = self.cache.live[rid], self.cache.fork(rid, new_rid)
        if hasattr(self.model, "copy_slots"):
            self.model.copy_slots([(src.slot, new.slot)])

    def truncate(self, rid: str, n_tokens: int) -> None:
        """takes back the tokens of an externally scheduled request from position n_tokens on (rejected drafts); models whose layers carry state cannot"""
        rid = str(rid)
        if self._scheduled(rid):
            raise ValueError(f"request {rid} belongs to the scheduler")
        if rid not in self.cache.live:
            raise ValueError(f"request {rid} holds nothing in the cache")
        if hasattr(self.model, "has_state") and self.model.has_state():
            raise ValueError("layers of this model carry state that cannot be taken back")
        if getattr(self.model, "cfg", None) is not None and getattr(self.model.cfg, "bigram", None) is not None:
            raise ValueError("this model's embedding reads the token before the next one, which a truncated request has lost")
        self.cache.truncate(rid, n_tokens, -1)

    def _cut(self, rids: Sequence[str]) -> None:
        """cuts those of the live requests back that hold more than max_keys cached rows (a request whose shared pages cannot be replaced yet: after a later step)"""
        while self.max_keys > 0:        # (a request that is cut back leaves pages, and pages that it shared to those that it shared them with)
            cut = []
            for rid in rids:
                s = self.cache.live.get(rid)
                if s is not None and s.rows > self.max_keys:
                    pages = self.cache.evict(rid, self.keep_keys, self.recent_keys)
                    if pages is not None:
                        cut.append((s.slot, pages))
            if not cut:
                return
            self.model.evict([s for s, _ in cut], [p[2] for _, p in cut], [p[0] for _, p in cut], [p[1] for _, p in cut], self.keep_keys, self.first_keys, self.recent_keys)
            for _, (had, to, _) in cut:
                self.cache.evicted(had, to)

    def compact(self) -> int:
        """moves the KV pages in use to the front of the pool; returns how many moved"""
        pairs = self.cache.compact()
        if pairs:
            self.model.copy_pages(pairs)
        return len(pairs)

    # ---- externally scheduled steps (trace replay) ----------------------------------------------------------------------------
    def run_entries(self, entries: Sequence[dict], end: Sequence[str] = ()) -> Optional[np.ndarray]:
        """entries: [{"id", "tokens", "want"}], of ids that are none of the scheduler's; end: requests whose pages and slot are given back after the step.
        Returns the logits of the wanted places as a host array, or None when nothing was wanted."""
        out = None
        entries = [e for e in entries if len(e.get("tokens", ()))]      # an entry that brings no token has nothing to run
        for rid in [str(e["id"]) for e in entries] + [str(i) for i in end]:
            if rid in self._sample_ids or self._scheduled(rid):
                raise ValueError(f"request {rid} belongs to the scheduler")
        new, free = len({str(e["id"]) for e in entries} - self.cache.live.keys()), self.cache.slots.free_slots
        if new and new > free - self._promised():
            raise CacheFull(f"{new} state slots wanted, {free} free, {self._promised()} of them kept for samples of running prompts")
        if entries:
            logits = self._forward([(str(e["id"]), list(e["tokens"]), list(e.get("want", ()))) for e in entries])
            if logits.shape[0]:
                out = logits.cpu().numpy()
        for rid in end:
            self.release(str(rid))
        self._cut([str(e["id"]) for e in entries])
        return out

    # ---- own scheduler ---------------------------------------------------------------------------------------------------------
    def add_request(self, rid: str, prompt: Sequence[int], params: Optional[SamplingParams] = None) -> Request:
        rid = str(rid)
        if self._in_use(rid):
            raise ValueError(f"request id {rid} is in use")
        if not len(prompt):
            raise ValueError("empty prompt")
        params = params or SamplingParams()
        self._check(params)
        samples = [f"{rid}#{i}" for i in range(1, params.n)]
        if any(self._in_use(i) for i in samples):
            raise ValueError(f"request ids {rid}#1 and on are in use")
        r = self._request(rid, [int(t) for t in prompt], params)
        self._sample_ids.update(samples)
        self.waiting.append(r)
        return r

    def _check(self, p: SamplingParams) -> None:
        if not 1 <= p.n <= self.cache.slots.n:
            raise ValueError(f"{p.n} samples of a prompt, of {self.cache.slots.n} requests that may live at a time")
        # (numbers as the kernels have them: of 32 bits)
        if not F32_TINY <= p.repetition_penalty <= F32_MAX:
            raise ValueError(f"a repetition penalty of {p.repetition_penalty}")
        if not (abs(p.presence_penalty) <= F32_MAX and abs(p.frequency_penalty) <= F32_MAX):
            raise ValueError(f"presence and frequency penalties of {p.presence_penalty} and {p.frequency_penalty}")
        if p.temperature != p.temperature or 0 < p.temperature < F32_TINY or (p.temperature > F32_MAX and p.ruled()):
            raise ValueError(f"a temperature of {p.temperature}")
        if p.temperature > 0 and not p.top_p > 0:
            raise ValueError(f"a top_p of {p.top_p}")
        if p.temperature > 0 and p.top_k < 0:
            raise ValueError(f"a top_k of {p.top_k}")
        if p.draft_fn is not None:
            if p.ruled():
                raise ValueError("drafts go with temperature, top_k and top_p: not with penalties, biases or masks")
            if hasattr(self.model, "has_state") and self.model.has_state():
                raise ValueError("layers of this model carry state that rejected drafts cannot be taken out of")
        vocab = getattr(getattr(self.model, "cfg", None), "vocab", None)
        for t in p.logit_bias or ():
            if int(t) != t or t < 0 or (vocab is not None and t >= vocab):
                raise ValueError(f"a bias on token {t} of {vocab}")
        for t, v in (p.logit_bias or {}).items():
            if not v <= F32_MAX:
                raise ValueError(f"a bias of {v} on token {t}")
        if vocab is not None and len(self._forbidden(p)) == vocab:
            raise ValueError("biases that leave no token")

    @staticmethod
    def _forbidden(p: SamplingParams) -> List[int]:
        """tokens that a bias of minus infinity (in 32 bits) takes out"""
        return [int(t) for t, v in (p.logit_bias or {}).items() if v < -F32_MAX]

    def _request(self, rid: str, prompt: List[int], params: SamplingParams, place: int = 0) -> Request:
        r = Request(rid, prompt, params)
        if params.temperature > 0:
            r._gen = torch.Generator(device=self.model.dev)
            r._gen.manual_seed((params.seed if params.seed is not None else 0) + place)
        self.requests[r.rid] = r
        return r

    def has_work(self) -> bool:
        return bool(self.waiting or self.running)

    def _schedule(self) -> List[Tuple[Request, List[int], List[int]]]:
        """decoded tokens of running requests first, then prompt portions while the token budget, the slots and the pages last, then guesses: no request waits for another's"""
        plan: List[Tuple[Request, List[int], List[int]]] = []
        guessing: List[int] = []       # places in the plan
        budget = self.max_step_tokens
        free_pages = self.cache.pages.free_blocks
        free_slots = self.cache.slots.free_slots - self._promised()
        for r in self.running:
            if r.fed < len(r.prompt):
                continue
            seq = self.cache.live[r.rid]
            if budget < 1 or self.cache.pages_needed(seq, 1) > free_pages or self._weight_room(seq) < 1:
                continue
            if r.params.draft_fn is not None:
                guessing.append(len(plan))
            plan.append((r, [r.output[-1]], [0]))
            budget -= 1
            free_pages -= self.cache.pages_needed(seq, 1)
        prefilling = [r for r in self.running if r.fed < len(r.prompt)]
        for r in prefilling + list(self.waiting):
            if budget < 1:
                break
            seq = self.cache.live.get(r.rid)
            if seq is None:
                if free_slots < r.params.n:
                    break
                free_slots -= r.params.n
            n = min(len(r.prompt) - r.fed, self.prefill_chunk, budget)
            have = len(seq.blocks) if seq else 0
            held = seq.rows if seq else 0
            own = self.cache.pages_to_copy(seq) if seq else 0       # shared pages that the portion would write into
            room = (have + free_pages - own) * self.cache.block_size - held if free_pages >= own else 0
            if seq is not None and self._weight_room(seq) < 1:
                continue                # (it waits to be cut back: nobody waits for it)
            n = min(n, room, self._weight_room(seq))
            if n < 1:
                if seq is None:
                    free_slots += r.params.n
                break
            need = max(0, -(-(held + n) // self.cache.block_size) - have)
            free_pages -= need + own
            budget -= n
            last = r.fed + n == len(r.prompt)
            plan.append((r, r.prompt[r.fed:r.fed + n], [n - 1] if last else []))
        for i in guessing:
            r, toks, _ = plan[i]
            seq = self.cache.live[r.rid]
            most = min(budget, r.params.max_new_tokens - len(r.output) - 1, self._weight_room(seq) - 1)
            guess = self._drafts(r, most) if most > 0 else []
            more = lambda n: self.cache.pages_needed(seq, 1 + n) - self.cache.pages_needed(seq, 1)
            while guess and more(len(guess)) > free_pages:
                guess = guess[:-1]
            plan[i] = (r, toks + guess, list(range(1 + len(guess))))
            budget -= len(guess)
            free_pages -= more(len(guess))
        return plan

    def _weight_room(self, seq: Optional[SeqState]) -> int:
        """rows that a request may still bring before it is cut back (what its weights have room for)"""
        return self.weighed_rows - (seq.rows if seq is not None else 0) if self.max_keys > 0 else self.max_step_tokens

    def step(self) -> List[Request]:
        """one forward pass over what the scheduler picked; returns the requests that finished in it.  A request whose logits leave no choice (sampled, and the
        largest over its temperature is no number) finishes without a token; when all others have theirs, RuntimeError says so"""
        plan = self._schedule()
        if not plan and self.max_keys > 0:      # (pages that were given back since the last step may let a request be cut back)
            self._cut([r.rid for r in self.running])
            plan = self._schedule()
        if not plan:
            if self.has_work():
                raise CacheFull("no request can make progress: the KV pool is too small for the live requests")
            return []
        masks = {r.rid: self._mask(r) for r, _, w in plan if w and r.params.mask_fn is not None}
        greedy = all(r.params.temperature <= 0 and not r.params.ruled() and r.params.n == 1 and r.params.draft_fn is None for r, _, w in plan if w)
        logits = self._forward([(r.rid, toks, want) for r, toks, want in plan], sample=greedy)
        for r, _, _ in plan:        # (requests run from here on: a mask that was refused, or a pass that failed, leaves them waiting)
            if r in self.waiting:
                self.waiting.remove(r)
                self.running.append(r)
        drafted, sampled, others, row = [], [], [], 0      # requests whose drafts are verified (request, tokens, first row of logits); requests that get one token, and their rows
        for r, toks, w in plan:
            if w and r.params.draft_fn is not None and r.output:
                drafted.append((r, toks, row))
            elif w:
                sampled.append(r)
                others.append(row)
            row += len(w)
        chosen = self._verify(logits, drafted) if drafted else []
        if drafted and sampled:
            logits = logits[torch.tensor(others, device=logits.device)]
        ids = self.model.last_ids.cpu().tolist() if (greedy and sampled) else None
        for r, toks, _ in plan:
            if r.fed < len(r.prompt):
                r.fed += len(toks)
        done: List[Request] = []
        rows = list(range(len(sampled)))
        if any(r.params.n > 1 and not r.output and not r.siblings for r in sampled):
            rows, sampled = self._fan_out(sampled)      # the other samples of a prompt choose from the same logits
            logits = logits[torch.tensor(rows, device=logits.device)]
            rows = list(range(len(sampled)))
        if ids is None and any(r.params.ruled() for r in sampled):
            logits = self._apply_rules(logits[:len(sampled)], sampled, masks)
        # largest logits of rows that are sampled: where one is no number there is nothing to choose by (and a multinomial of it would end the process)
        tops = logits[:len(sampled)].max(1).values.tolist() if any(r.params.temperature > 0 for r in sampled) else None
        lost: List[str] = []
        for (r, _, _), tokens in zip(drafted, chosen):
            if tokens[-1] < 0:
                lost.append(f"{r.rid} (a row of its logits has no largest number)")
                tokens.pop()
                r.finished = True
            for tok in tokens:
                r.output.append(tok)
                if len(r.output) >= r.params.max_new_tokens or tok in r.params.stop_tokens:
                    r.finished = True
                    break
            if r.finished:
                done.append(r)
        for row, r in zip(rows, sampled):
            if r.params.temperature > 0 and not abs(tops[row] / r.params.temperature) <= F32_MAX:
                lost.append(f"{r.rid} (its largest logit is {tops[row]}, its temperature {r.params.temperature})")
                r.finished = True
                done.append(r)
                continue
            tok = ids[row] if ids is not None else self._sample(logits[row], r)
            r.output.append(int(tok))
            if len(r.output) >= r.params.max_new_tokens or int(tok) in r.params.stop_tokens:
                r.finished = True
                done.append(r)
        for r in done:
            self.running.remove(r)
            self.release(r.rid)
        self._cut([r.rid for r in self.running])
        if lost:
            raise RuntimeError("no token can be chosen for request " + ", ".join(lost))
        return done

    def _drafts(self, r: Request, most: int) -> List[int]:
        """up to `most` guesses of the request's next tokens (and the probabilities they were drawn from, kept for the step)"""
        got = r.params.draft_fn(r.prompt + r.output)
        probs = None
        if isinstance(got, tuple) and len(got) == 2 and np.ndim(got[0]) > 0:      # (two guesses are a tuple of two, too)
            got, probs = got
        tokens = [int(t) for t in got][:max(0, most)]
        vocab = getattr(getattr(self.model, "cfg", None), "vocab", None)
        if any(t < 0 or (vocab is not None and t >= vocab) for t in tokens):
            raise ValueError(f"drafts of request {r.rid} outside the vocabulary: {tokens}")
        if probs is not None and (probs.dim() != 2 or probs.shape[0] < len(tokens) or (vocab is not None and probs.shape[1] != vocab)):
            raise ValueError(f"the draft probabilities of request {r.rid} are a row for each of {len(tokens)} drafts, not {tuple(probs.shape)}")
        r._probs = probs
        return tokens

    def _verify(self, logits: torch.Tensor, drafted: Sequence[Tuple[Request, List[int], int]]) -> List[List[int]]:
        """the tokens that come behind the last one of every request (-1: a row without a choice); rejected drafts leave the cache"""
        dev, out = logits.device, {}
        for known in (False, True):        # certain guesses, and guesses with the probabilities they were drawn from
            part = [d for d in drafted if (d[0]._probs is not None and len(d[1]) > 1) == known]
            if not part:
                continue
            lens = [len(toks) for _, toks, _ in part]
            start = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
            rows = np.concatenate([np.arange(row, row + n) for (_, _, row), n in zip(part, lens)])
            z = logits[int(rows[0]):int(rows[-1]) + 1] if (np.diff(rows) == 1).all() else logits[torch.from_numpy(rows).to(dev)]
            up = lambda x, dt: torch.from_numpy(np.asarray(x, dt)).to(dev)
            drafts = up(np.concatenate([toks[1:] + [0] for _, toks, _ in part]), np.int32)
            # a request draws as many numbers as it brought rows, and one more
            u = [torch.rand(n + 1, device=dev, generator=r._gen) if r._gen is not None else torch.zeros(n + 1, device=dev) for (r, _, _), n in zip(part, lens)]
            kw: Dict[str, torch.Tensor] = {}
            if any(r.params.top_k for r, _, _ in part):
                kw["top_k"] = up([min(max(r.params.top_k, 0), logits.shape[1]) for r, _, _ in part], np.int32)      # (as many as there are: all)
            if any(r.params.top_p < 1.0 for r, _, _ in part):
                kw["top_p"] = up([r.params.top_p for r, _, _ in part], np.float32)
            if known:
                q = torch.zeros((int(start[-1]), logits.shape[1]), dtype=torch.float32, device=dev)
                for (r, _, _), s, n in zip(part, start, lens):
                    q[int(s):int(s) + n - 1] = r._probs[:n - 1].to(dev, torch.float32)
                kw["draft_probs"] = q
            accepted, tokens = seqops.verify_drafts(z, up(start, np.int32), drafts, torch.cat([x[:-1] for x in u]), torch.stack([x[-1] for x in u]),
                                             up([max(r.params.temperature, 0.0) for r, _, _ in part], np.float32), **kw)
            both = torch.cat([accepted, tokens]).cpu().tolist()
            got = both[len(part):]
            for (r, _, _), s, a in zip(part, start, both):
                out[r.rid] = got[int(s):int(s) + a + 1]
        for r, toks, _ in drafted:
            a = len(out[r.rid]) - 1
            if a + 1 < len(toks):
                seq = self.cache.live[r.rid]
                self.cache.truncate(r.rid, seq.n_tokens - (len(toks) - 1 - a), toks[a])
        return [out[r.rid] for r, _, _ in drafted]

    def _fan_out(self, sampled: List[Request]) -> Tuple[List[int], List[Request]]:
        """forks requests whose prompt is through into their params.n samples; (row of the step's logits, request) of every sample, in order"""
        rows, out = [], []
        for row, r in enumerate(sampled):
            rows.append(row)
            out.append(r)
            if r.params.n > 1 and not r.output and not r.siblings:
                for i in range(1, r.params.n):
                    rid = f"{r.rid}#{i}"
                    self._sample_ids.discard(rid)
                    self._fork_cache(r.rid, rid)
                    q = self._request(rid, r.prompt, r.params, i)
                    q.fed = r.fed
                    q.siblings = [r]
                    r.siblings.append(q)
                    self.running.append(q)
                    rows.append(row)
                    out.append(q)
        return rows, out

    def _mask(self, r: Request) -> Optional[np.ndarray]:
        """the words of the tokens that may come next, asked for before the step runs: a mask that is refused leaves the request as it was"""
        words = r.params.mask_fn(list(r.output))
        if words is None:
            return None
        m = np.asarray(words).reshape(-1).astype(np.int64).astype(np.uint32)
        vocab = getattr(getattr(self.model, "cfg", None), "vocab", 32 * m.size)
        if m.size != (vocab + 31) // 32:
            raise ValueError(f"the mask of request {r.rid} has {m.size} words, not {(vocab + 31) // 32}")
        forbidden = [t for t in self._forbidden(r.params) if t < 32 * m.size]
        if forbidden:
            bits = np.unpackbits(m.astype("<u4").view(np.uint8), bitorder="little")
            bits[forbidden] = 0
            m = np.packbits(bits, bitorder="little").view("<u4").astype(np.uint32)
        last = m[-1] if vocab % 32 == 0 else m[-1] & np.uint32((1 << vocab % 32) - 1)
        if not (m[:-1].any() or last):
            raise ValueError(f"the mask of request {r.rid} leaves no token")
        return m.view(np.int32)

    def _apply_rules(self, logits: torch.Tensor, requests: Sequence[Request], masks: Dict[str, Optional[np.ndarray]]) -> torch.Tensor:
        """the requests' penalties, biases and masks on their rows of logits (requests without any: the rows stay, bit by bit)"""
        V, dev = logits.shape[1], logits.device
        words = (V + 31) // 32
        rules = np.tile(np.array([1.0, 0.0, 0.0, 0.0], np.float32), (len(requests), 1))
        hist, start, prompt, bias, bstart, mask = [], [0], [], [], [0], None
        for i, r in enumerate(requests):
            p = r.params
            if p.ruled():
                rules[i, :3] = p.repetition_penalty, p.presence_penalty, p.frequency_penalty
                if p.repetition_penalty != 1.0:
                    hist += r.prompt
                    prompt.append(len(r.prompt))
                else:
                    prompt.append(0)
                hist += r.output
                bias += [(t, v if v >= -F32_MAX else -np.inf) for t, v in (p.logit_bias or {}).items()]
                m = masks.get(r.rid if r.rid in masks or not r.siblings else r.siblings[0].rid)      # (a sample's first token: the mask of its prompt's request)
                if m is not None:
                    if mask is None:
                        mask = np.full((len(requests), words), -1, np.int32)
                    mask[i] = m
            else:
                prompt.append(0)
            start.append(len(hist))
            bstart.append(len(bias))
        up = lambda x, dt: torch.from_numpy(np.asarray(x, dt)).to(dev)
        kw = {}
        if hist:
            kw.update(hist=up(hist, np.int32), hist_start=up(start, np.int32), hist_prompt=up(prompt, np.int32))
        if bias:
            kw.update(bias_start=up(bstart, np.int32), bias_ids=up([t for t, _ in bias], np.int32), bias_vals=up([v for _, v in bias], np.float32))
        if mask is not None:
            kw.update(mask=torch.from_numpy(mask).to(dev))
        return seqops.process_logits(logits, up(rules, np.float32), torch.empty_like(logits), **kw)

    def _sample(self, logits: torch.Tensor, r: Request) -> int:
        p = r.params
        if p.temperature <= 0:
            ids = torch.empty(1, dtype=torch.int32, device=logits.device)
            seqops.argmax(logits.reshape(1, -1).contiguous(), ids)
            return int(ids.item())
        z = logits.float() / p.temperature
        if p.top_k and p.top_k < z.numel():
            kth = torch.topk(z, p.top_k).values[-1]
            z = torch.where(z < kth, torch.full_like(z, float("-inf")), z)
        pr = torch.softmax(z, 0)
        if p.top_p < 1.0:
            sp, si = torch.sort(pr, descending=True)
            keep = torch.cumsum(sp, 0) - sp < p.top_p
            pr = torch.zeros_like(pr).scatter(0, si[keep], sp[keep])
            pr = pr / pr.sum()
        return int(torch.multinomial(pr, 1, generator=r._gen).item())

    def generate(self, prompts: Sequence[Sequence[int]], params: Optional[SamplingParams] = None) -> List[List[int]]:
        """runs the prompts to completion through the scheduler (more prompts than slots queue up); returns the new tokens of each (params.n > 1: a list of
        its n samples)"""
        reqs: List[Request] = []
        try:
            for i, p in enumerate(prompts):
                reqs.append(self.add_request(f"g{self.steps}_{i}", p, params))
            while any(not q.finished for r in reqs for q in [r] + r.siblings):
                self.step()
            flags = seqops.error_flags()
            if flags:
                raise RuntimeError(f"device error flags {flags:#x} (1: KV position outside its block table, 2: a bounded wait ran out, 4: expert table entry out of range, "
                                   "8: a key or value beyond what a 4-bit cache holds, 16: a token id outside the vocabulary)")
        finally:                    # also what is left of them where a step fails
            for r in reqs:
                self._sample_ids.difference_update(f"{r.rid}#{i}" for i in range(1, r.params.n))
                for q in [r] + r.siblings:
                    if not q.finished:
                        (self.running if q in self.running else self.waiting).remove(q)
                        q.finished = True
                        self.release(q.rid)
                    del self.requests[q.rid]
        return [[q.output for q in [r] + r.siblings] if r.params.n > 1 else r.output for r in reqs]
